"""Where the serving operators' errors are reported: one word per device, for eager and captured calls on any stream."""

import ctypes
import subprocess
import sys
import threading

import pytest
import torch

import orthocache_gpu_b200 as oc
from orthocache_gpu_b200 import _lib

pytestmark = pytest.mark.gpu


def _decode(page=0, length=40):
    q = torch.randn(1, 2, 64, device="cuda", dtype=torch.float16)
    c = torch.randn(4, 1, 16, 64, device="cuda", dtype=torch.float16)
    table = torch.tensor([[0, 1, page]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([length], dtype=torch.int32, device="cuda")
    return (q, c, c, table, lens), lambda: oc.paged_decode_attention(q, c, c, table, lens)


def _clear():
    try:
        oc.check_status()
    except RuntimeError:
        pass


def test_a_replayed_graph_reports_to_the_word_that_is_checked():
    (q, c, _, table, lens), call = _decode()
    call()
    torch.cuda.synchronize()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):  # the first call on this stream
        out = oc.paged_decode_attention(q, c, c, table, lens)
    _clear()
    graph.replay()
    oc.check_status()
    assert torch.equal(out, call())
    table[0, 2] = 9
    graph.replay()
    table[0, 2] = 0
    graph.replay()  # a good replay does not take the report back
    with pytest.raises(RuntimeError, match="block-table entry"):
        oc.check_status()
    oc.check_status()


def test_a_captured_reserve_that_runs_out_of_pages_is_reported():
    c = oc.PagedKVCache(1, 4, 1, 8, max_seqs=2, max_tokens=64, block_size=4)
    one = torch.tensor([3, 0], dtype=torch.int32, device="cuda")
    c.reserve(one)
    c.seq_lens += one
    grow = torch.zeros(2, dtype=torch.int32, device="cuda")
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        c.reserve(grow, check=False)
    graph.replay()
    oc.check_status()
    grow[0] = 30
    graph.replay()
    with pytest.raises(RuntimeError, match="too few free pages"):
        oc.check_status()
    assert c.block_tables[0].tolist() == [0] + [-1] * 15


def test_the_very_first_call_may_be_captured():
    """In a process of its own: nothing is allocated or cleared inside the capture."""
    code = """
import torch, orthocache_gpu_b200 as oc
q = torch.randn(1, 2, 64, device="cuda", dtype=torch.float16)
c = torch.randn(4, 1, 16, 64, device="cuda", dtype=torch.float16)
table = torch.tensor([[0, 1, 9]], dtype=torch.int32, device="cuda")
lens = torch.tensor([40], dtype=torch.int32, device="cuda")
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = oc.paged_decode_attention(q, c, c, table, lens)
oc.check_status()
graph.replay()
table[0, 2] = 0
graph.replay()
try:
    oc.check_status()
    print("not reported")
except RuntimeError as e:
    print("reported" if "block-table entry" in str(e) else e)
oc.check_status()
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=240)
    assert r.stdout.strip() == "reported", r.stdout + r.stderr[-2000:]


def test_other_streams_report_to_the_same_word():
    side = torch.cuda.Stream()
    args, call = _decode(page=-1)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    side.synchronize()
    with pytest.raises(RuntimeError, match="block-table entry"):
        oc.check_status()


def test_first_calls_of_two_threads_on_one_stream(monkeypatch):
    """Whichever thread sets up what a stream needs, the report is found."""
    made, init = [], _lib._Workspace.__init__

    def slow(self, device):
        threading.Event().wait(0.2)
        made.append(self)
        init(self, device)

    monkeypatch.setattr(_lib._Workspace, "__init__", slow)
    side = torch.cuda.Stream()
    args, call = _decode(page=-1)
    torch.cuda.synchronize()

    def work():
        with torch.cuda.stream(side):
            call()

    threads = [threading.Thread(target=work) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    with torch.cuda.stream(side):
        with pytest.raises(RuntimeError, match="block-table entry"):
            oc.check_status()
        oc.check_status()
        call()  # what the threads set up is still what is checked
        with pytest.raises(RuntimeError, match="block-table entry"):
            oc.check_status()


def test_the_cabi_clears_the_bits_that_it_is_given():
    lib = _lib.load()
    word = _lib._device_word(torch.device("cuda", torch.cuda.current_device()))
    at = ctypes.c_void_p()
    assert lib.oc_device_status(ctypes.byref(at)) == 0 and at.value == word.data_ptr()
    assert lib.oc_device_status(None) == 1
    other = torch.tensor([29], dtype=torch.int32, device="cuda")
    assert lib.oc_clear_status(other.data_ptr(), 24, _lib.stream_ptr(other.device)) == 0
    assert other.item() == 5
    assert lib.oc_clear_status(None, 1, None) == 1
