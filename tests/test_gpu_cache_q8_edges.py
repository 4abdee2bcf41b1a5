"""The 8-bit cache on the GPU at the edges of its ranges: borders between codes, rows that are no numbers, the largest values, ..."""

import math

import pytest
import torch

from shrike_b200.cache.quantised import QuantisedPages
from tests import cache_q8_oracle as oracle
from tests.gpu_common import cuda_ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def border_rows(count, dim, seed=0):
    """float32 rows of elements at and one step beside the borders between two codes, small codes above all, with the largest
    magnitude in front."""
    g = torch.Generator().manual_seed(seed)
    a = (1 + torch.rand(count, 1, generator=g)).float() * 2.0 ** torch.randint(-90, 91, (count, 1), generator=g).float()
    border = torch.where(torch.rand(count, dim, generator=g) < 0.5, torch.randint(0, 4, (count, dim), generator=g),
                         torch.randint(0, 127, (count, dim), generator=g))
    x = (a.double() * (2 * border + 1) / 254).float()
    beside = torch.randint(-1, 2, (count, dim), generator=g)
    x = torch.where(beside > 0, torch.nextafter(x, a), torch.where(beside < 0, torch.nextafter(x, torch.zeros(())), x))
    x = x * (1 - 2 * torch.randint(0, 2, (count, dim), generator=g))
    x[:, 0] = a[:, 0]
    x[0, 1], x[0, 0] = float.fromhex("0x1.1a3ba6p-8"), float.fromhex("0x1.18072ep+0")
    x[0, 2:] = 0
    return x.to(DEV)


@pytest.mark.parametrize("dim", [32, 128, 256])
@pytest.mark.parametrize("fused", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_codes_beside_the_borders(dim, fused, dtype):
    """Rows in 32 bits: those of the 32-bit store, and of a projection in either type."""
    if not fused and dtype == torch.bfloat16:
        pytest.skip("a store of bfloat16 rows has no such elements")
    ops = cuda_ops(dtype)
    n, heads, page = 300, 2, 16
    k, v = (border_rows(n * heads, dim, seed).view(n, heads * dim) for seed in (1, 2))
    keys, values = (QuantisedPages.zeros(20, page, heads, dim, DEV) for _ in range(2))
    slots = torch.randperm(20 * page, generator=torch.Generator().manual_seed(3))[:n].to(torch.int32).to(DEV)
    if fused:
        q = torch.zeros(n, heads * dim, device=DEV)
        ops.rope_kv_write(torch.cat([q, k, v], 1), None, slots, None, torch.empty(n, heads * dim, dtype=dtype, device=DEV), keys, values, slots,
                          heads, heads, dim)
    else:
        ops.kv_write(k, v, keys, values, slots)
    at = slots.long()
    for pool, x in ((keys, k), (values, v)):
        codes, scales = oracle.quantise(x.view(n, heads, dim))
        assert torch.equal(pool.codes[at // page, at % page], codes)
        assert torch.equal(pool.scales[at // page, :, at % page], scales)
