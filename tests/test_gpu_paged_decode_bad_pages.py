"""Pages outside the cache: reported, and their keys and values count as zeros in every kernel."""

import pytest
import torch

import orthocache_gpu_b200 as oc
from serving_helpers import pages_for

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype, f8", [(torch.bfloat16, False), (torch.float16, True), (torch.float32, False)])
@pytest.mark.parametrize("D, block, lens, cols", [(64, 16, [40, 300], 0), (128, 4, [40, 300], 0), (256, 128, [200, 500], 0),
                                                  (64, 2, [33, 70], 0), (128, 16, [2500, 9000], 0), (64, 64, [100, 200], 500)])
def test_their_keys_and_values_are_zeros(dtype, f8, D, block, lens, cols):
    table, pages = pages_for(lens, block, "cuda", spare=1)
    if cols:
        table = torch.cat([table, torch.full((2, cols), -1, dtype=torch.int32, device="cuda")], 1)
    g = torch.Generator(device="cuda").manual_seed(D)
    q = torch.randn(2, 6, D, device="cuda", generator=g).to(dtype)
    kc, vc = (torch.randn(pages, 2, block, D, device="cuda", generator=g).to(dtype) for _ in range(2))
    (zero,) = set(range(pages)) - set(table[table >= 0].tolist())
    kc[zero], vc[zero] = 0, 0
    if f8:
        kc, vc = kc.to(torch.float8_e4m3fn), vc.to(torch.float8_e4m3fn)
    n = torch.tensor(lens, device="cuda")
    columns = [0, (lens[1] - 1) // block // 2, (lens[1] - 1) // block]
    for column in columns:
        good = table.clone()
        good[1, column] = zero
        want = oc.paged_decode_attention(q, kc, vc, good, n, return_lse=True)
        oc.check_status()
        for page in (-1, pages, 2 ** 31 - 1, -2 ** 31):
            bad = table.clone()
            bad[1, column] = page
            for _ in range(2):
                # another call's tiles lie in shared memory before
                oc.paged_decode_attention(q * 3, kc, vc, good.flip(0), n.flip(0))
                got = oc.paged_decode_attention(q, kc, vc, bad, n, return_lse=True)
                with pytest.raises(RuntimeError, match="block-table entry"):
                    oc.check_status()
                assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), (column, page)
