"""The 8-bit cache on the GPU at the edges of its ranges: borders between codes, rows that are no numbers, the largest values, ..."""

import math

import pytest
import torch

from shrike_b200.cache.quantised import QuantisedPages
from tests import cache_q8_oracle as oracle
from tests.gpu_common import cuda_ops
from tests.test_gpu_cache_q8 import FORMS, attend

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
@pytest.mark.parametrize("fused,dtype", [(False, torch.float32), (True, torch.float32), (True, torch.bfloat16)])
def test_codes_beside_the_borders(dim, fused, dtype):
    """Rows in 32 bits: those of the 32-bit store, and of a projection in either type."""
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


@pytest.mark.parametrize("dtype,dim,tensor_cores", FORMS)
@pytest.mark.parametrize("splits", [1, 3])
@pytest.mark.parametrize("few_rows", [False, True])
@pytest.mark.parametrize("options", [{}, {"window": 90}])
def test_a_value_that_is_no_number_reaches_every_row_that_sees_it(dtype, dim, tensor_cores, splits, few_rows, options):
    """However small its key's weight: 2^-300 of the others', zero in 32 bits."""
    heads, kv_heads, page = 4, 2, 16
    q_lens, ctx_lens, bad = [100, 1, 1, 70], [150, 700, 90, 400], [120, 655, 89, 340]
    ops = cuda_ops(dtype)
    ops.tensor_core_attention, ops.portion_splits, ops.q8_splits, ops.q8_few_rows = tensor_cores, splits, (splits, 1), few_rows
    case = oracle.pages_case(heads, kv_heads, dim, page, q_lens, ctx_lens, dtype, 9, DEV)
    case["q"].view(-1, dim)[:, 0] = 16.0
    for s, position in enumerate(bad):
        page_id, within = int(case["table"][s, position // page]), position % page
        case["codes_k"][page_id, within] = 0
        case["codes_k"][page_id, within, :, 0] = -127
        case["scales_k"][page_id, :, within] = 0.125 * dim ** 0.5   # a score of -254, against some units
        case["scales_v"][page_id, :, within] = math.nan
        case["sequences"][s][0][0][position] = case["codes_k"][page_id, within]
        case["sequences"][s][0][1][position] = 0.125 * dim ** 0.5
        case["sequences"][s][1][1][position] = 0.0
    got = attend(ops, case, heads, kv_heads, dim, q_lens, ctx_lens, **options)
    want, bound = oracle.attention(case["q"], case["sequences"], q_lens, ctx_lens, heads, kv_heads, dim, dim ** -0.5, **options)
    position = torch.cat([torch.arange(c - n, c) for n, c in zip(q_lens, ctx_lens)])
    spoilt = torch.repeat_interleave(torch.tensor(bad), torch.tensor(q_lens))
    sees = ((position >= spoilt) & (position < spoilt + options.get("window", 1 << 30))).to(DEV)
    assert torch.isnan(got[sees]).all()
    assert ((got.double() - want).abs() <= bound)[~sees].all()
    ops.check_status()


@pytest.mark.parametrize("dtype,dim,tensor_cores", FORMS)
@pytest.mark.parametrize("few_rows", [False, True])
def test_a_value_that_is_no_number_among_keys_of_no_weight(dtype, dim, tensor_cores, few_rows):
    """All keys of a share score 2^-300 of the others': the share has no weight, and its NaN still counts."""
    heads, kv_heads, page = 4, 2, 16
    q_lens, ctx_lens = [70, 1], [400, 400]
    ops = cuda_ops(dtype)
    ops.tensor_core_attention, ops.portion_splits, ops.q8_splits, ops.q8_few_rows = tensor_cores, 3, (4, 2), few_rows
    case = oracle.pages_case(heads, kv_heads, dim, page, q_lens, ctx_lens, dtype, 9, DEV)
    case["q"].view(-1, dim)[:, 0] = 16.0
    for s in range(2):
        ids = case["table"][s, : 192 // page].long()   # the first 192 keys: a share of any form, and more
        case["codes_k"][ids] = 0
        case["codes_k"][ids, :, :, 0] = -127
        case["scales_k"][ids] = 0.125 * dim ** 0.5
    fine = attend(ops, case, heads, kv_heads, dim, q_lens, ctx_lens)
    assert torch.isfinite(fine).all()
    case["scales_v"][int(case["table"][0, 40 // page]), 1, 40 % page] = math.nan   # heads 2 and 3 of the portion
    case["scales_v"][int(case["table"][1, 7 // page]), 0, 7] = math.nan             # heads 0 and 1 of the single token
    got = attend(ops, case, heads, kv_heads, dim, q_lens, ctx_lens)
    none = torch.isnan(got.view(71, 2, -1))
    assert none[:70, 1].all() and none[70, 0].all() and not none[:70, 0].any() and not none[70, 1].any()
    ops.check_status()


@pytest.mark.parametrize("dtype,dim,tensor_cores", FORMS)
@pytest.mark.parametrize("few_rows", [False, True])
@pytest.mark.parametrize("size", [1e34, 1e36, 3e38])
def test_the_largest_values(dtype, dim, tensor_cores, few_rows, size):
    """Values of up to about float32's largest number under scores that grow along the keys, so that a base which lagged would show."""
    heads, kv_heads, page = 4, 2, 16
    q_lens, ctx_lens = [150, 1, 1], [700, 900, 70]
    ops = cuda_ops(dtype)
    ops.tensor_core_attention, ops.portion_splits, ops.q8_splits, ops.q8_few_rows = tensor_cores, 1, (1, 1), few_rows
    case = oracle.pages_case(heads, kv_heads, dim, page, q_lens, ctx_lens, dtype, 21, DEV)
    case["q"].view(-1, dim)[:, 0] = 4.0
    for s, context in enumerate(ctx_lens):
        (key_codes, key_scales), (codes, scales) = case["sequences"][s]
        for j in range(context):   # the first element's part of the score: up to 4 more from the first key to the last
            key_codes[j, :, 0] = ((j + 1) * dim ** 0.5 / context / key_scales[j]).round().clamp(0, 127).to(torch.int8)
        scales.copy_(torch.where(torch.arange(context, device=DEV)[:, None] % 5 == 4, 1.0, size / 127))   # ordinary ones among them
        ids = case["table"][s].long()
        for j in range(context):
            at = ids[j // page], j % page
            case["codes_k"][at], case["scales_v"][at[0], :, at[1]] = key_codes[j], scales[j]
    got = attend(ops, case, heads, kv_heads, dim, q_lens, ctx_lens)
    want, bound = oracle.attention(case["q"], case["sequences"], q_lens, ctx_lens, heads, kv_heads, dim, dim ** -0.5)
    # under F = 107 what is below 2^-19 of the largest weight is below 2^-126, zero: that much of a key's value, and of a sum
    lost = torch.repeat_interleave(torch.tensor(ctx_lens), torch.tensor(q_lens)).double().to(DEV)[:, None] * 2.0 ** -18 * size
    assert torch.isfinite(got).all()
    assert ((got.double() - want).abs() <= bound + lost).all()
    ops.check_status()


@pytest.mark.parametrize("dtype,dim,tensor_cores", FORMS)
@pytest.mark.parametrize("few_rows", [False, True])
@pytest.mark.parametrize("splits", [1, 3])
@pytest.mark.parametrize("size", [1.0, 1e20, 1e36])
def test_keys_without_values_before_large_ones(dtype, dim, tensor_cores, few_rows, splits, size):
    """Keys whose values are zeros have their part in the sums, however large the values behind them (or beside them, in another
    share of the keys) are."""
    heads, kv_heads, page = 4, 2, 16
    q_lens, ctx_lens, zeros = [90, 1, 1, 40], [700, 900, 70, 300], [350, 800, 32, 64]
    ops = cuda_ops(dtype)
    ops.tensor_core_attention, ops.portion_splits, ops.q8_splits, ops.q8_few_rows = tensor_cores, splits, (4 * splits, 2 * splits), few_rows
    case = oracle.pages_case(heads, kv_heads, dim, page, q_lens, ctx_lens, dtype, 22, DEV)
    for s, context in enumerate(ctx_lens):
        scales = case["sequences"][s][1][1]
        scales.mul_(size)
        scales[: zeros[s]] = 0
        for j in range(context):
            case["scales_v"][int(case["table"][s, j // page]), :, j % page] = scales[j]
    got = attend(ops, case, heads, kv_heads, dim, q_lens, ctx_lens)
    want, bound = oracle.attention(case["q"], case["sequences"], q_lens, ctx_lens, heads, kv_heads, dim, dim ** -0.5)
    lost = torch.repeat_interleave(torch.tensor(ctx_lens), torch.tensor(q_lens)).double().to(DEV)[:, None] * 2.0 ** -18 * 40 * size if size > 1e30 else 0.0
    assert ((got.double() - want).abs() <= bound + lost).all()
    ops.check_status()


@pytest.mark.parametrize("few_rows", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_largest_queries(dtype, few_rows):
    """Queries of the type's largest number over keys as small as that: scores of some units."""
    heads, kv_heads, dim, page = 4, 2, 64, 16
    q_lens, ctx_lens = [70, 1], [200, 300]
    ops = cuda_ops(dtype)
    ops.q8_few_rows = few_rows
    case = oracle.pages_case(heads, kv_heads, dim, page, q_lens, ctx_lens, dtype, 23, DEV)
    top = torch.finfo(dtype).max
    q = case["q"].view(-1, dim)
    q.copy_(torch.where(q > 0, top, -top) * (torch.arange(dim, device=DEV) % 16 == 0))
    case["scales_k"].mul_(1.0 / 2.0 ** 127)
    for keys, _values in case["sequences"]:
        keys[1].mul_(1.0 / 2.0 ** 127)
    got = attend(ops, case, heads, kv_heads, dim, q_lens, ctx_lens)
    want, bound = oracle.attention(case["q"], case["sequences"], q_lens, ctx_lens, heads, kv_heads, dim, dim ** -0.5)
    assert ((got.double() - want).abs() <= bound).all()
    ops.check_status()


def test_a_captured_call_keeps_its_workspace_when_a_larger_one_is_needed():
    """A sequence captured over split rows is replayed after the workspace has grown and the memory has found other users."""
    heads, kv_heads, dim, page = 8, 1, 64, 16
    ops = cuda_ops(torch.bfloat16)
    ops.q8_splits = (64, 1)
    case = oracle.pages_case(heads, kv_heads, dim, page, [1], [4000], torch.bfloat16, 4, DEV)
    out = torch.empty_like(case["q"])

    def call():
        ops.paged_attention(case["q"], QuantisedPages(case["codes_k"], case["scales_k"]), QuantisedPages(case["codes_v"], case["scales_v"]),
                            case["table"], case["q_start"], case["ctx_len"], case["seq_of"], heads, kv_heads, dim, dim ** -0.5, None, out,
                            max_q_len=1, min_q_len=1)

    call()
    want = out.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    old, count = ops._q8_scratch, 200
    many = oracle.pages_case(heads, kv_heads, dim, page, [1] * count, [70] * count, torch.bfloat16, 5, DEV)
    ops.q8_plan(heads, kv_heads, dim, 4000, 20, page, 1, 1)   # as a batch of many sequences asks for
    assert ops._q8_scratch.numel() > old.numel() and any(x is old for x in ops._q8_kept)
    del old
    others = [torch.full((1 << 20,), 7.0, device=DEV) for _ in range(8)]
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want) and all((x == 7.0).all() for x in others)
    got = attend(ops, many, heads, kv_heads, dim, [1] * count, [70] * count)
    expected, bound = oracle.attention(many["q"], many["sequences"], [1] * count, [70] * count, heads, kv_heads, dim, dim ** -0.5)
    assert ((got.double() - expected).abs() <= bound).all()


def test_the_first_call_of_all_may_be_a_captured_one():
    """Its counters are there already: a call before the first replay counts from zero, and so does a second sequence."""
    heads, kv_heads, dim, page = 8, 1, 64, 16
    torch.randint(1, 1000, (1 << 16,), dtype=torch.int32, device=DEV)   # what fresh memory may hold
    ops = cuda_ops(torch.bfloat16)
    ops.q8_splits = (64, 8)
    cases = [oracle.pages_case(heads, kv_heads, dim, page, [1], [3000 + 500 * i], torch.bfloat16, i, DEV) for i in range(3)]
    outs = [torch.zeros_like(case["q"]) for case in cases]

    def call(i):
        case = cases[i]
        ops.paged_attention(case["q"], QuantisedPages(case["codes_k"], case["scales_k"]), QuantisedPages(case["codes_v"], case["scales_v"]),
                            case["table"], case["q_start"], case["ctx_len"], case["seq_of"], heads, kv_heads, dim, dim ** -0.5, None, outs[i],
                            max_q_len=1, min_q_len=1)

    ops._q8_lib(dim)   # compiled, if it has to be, before a capture
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for i, graph in enumerate(graphs):
        with torch.cuda.graph(graph):
            call(i)
    call(2)
    graphs[1].replay()
    graphs[0].replay()
    torch.cuda.synchronize()
    for i, case in enumerate(cases):
        want, bound = oracle.attention(case["q"], case["sequences"], [1], [3000 + 500 * i], heads, kv_heads, dim, dim ** -0.5)
        assert ((outs[i].double() - want).abs() <= bound).all()


@pytest.mark.parametrize("dtype,dim,tensor_cores", FORMS)
@pytest.mark.parametrize("few_rows", [False, True])
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("options", [{"window": 64}, {"chunk": 96}])
def test_a_context_that_no_table_holds(dtype, dim, tensor_cores, few_rows, new, options):
    """Keys near 2^31 have no page: the rows that see nothing else are zeros, and the other sequences' are what they are without."""
    heads, kv_heads, page = 4, 2, 16
    q_lens, ctx_lens = [new, new, 1], [300, new, 90]
    ops = cuda_ops(dtype)
    ops.tensor_core_attention, ops.portion_splits, ops.q8_splits, ops.q8_few_rows = tensor_cores, 2, (2, 2), few_rows
    case = oracle.pages_case(heads, kv_heads, dim, page, q_lens, ctx_lens, dtype, 24, DEV)
    plain = attend(ops, case, heads, kv_heads, dim, q_lens, ctx_lens, **options)
    case["ctx_len"][1] = 2 ** 31 - 1
    got = attend(ops, case, heads, kv_heads, dim, q_lens, ctx_lens, **options)
    torch.cuda.synchronize()
    assert (got[new: 2 * new] == 0).all()
    assert torch.equal(got[:new], plain[:new]) and torch.equal(got[2 * new:], plain[2 * new:])
    ops.check_status()
