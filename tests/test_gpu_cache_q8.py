"""The 8-bit cache on the GPU: what is stored, what is read back, and attention over it, against 64 bits."""

import math

import pytest
import torch

from shrike_b200.cache.quantised import QuantisedPages
from tests import cache_q8_oracle as oracle
from tests.gpu_common import cuda_ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.bfloat16, torch.float32]


def rnd(*shape, seed=0, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(DEV, dtype)


def empty_pages(pages, page, heads, dim):
    """Pages whose every place is marked, so that what is stored beside its slot shows."""
    return QuantisedPages(torch.full((pages, page, heads, dim), 77, dtype=torch.int8, device=DEV),
                          torch.full((pages, heads, page), 7.5, device=DEV))


def check_stored(pages, x, slots, heads, dim):
    page = pages.codes.shape[1]
    codes, scales = oracle.quantise(x.view(-1, heads, dim))
    want_codes, want_scales = torch.full_like(pages.codes, 77), torch.full_like(pages.scales, 7.5)
    for row, slot in enumerate(slots.tolist()):
        if 0 <= slot < pages.codes.shape[0] * page:
            want_codes[slot // page, slot % page] = codes[row]
            want_scales[slot // page, :, slot % page] = scales[row]
    assert torch.equal(pages.codes, want_codes)
    assert torch.equal(pages.scales.nan_to_num(nan=-1.0), want_scales.nan_to_num(nan=-1.0))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,heads,dim,page", [(1, 4, 128, 16), (7, 1, 16, 1), (33, 3, 32, 8), (70, 2, 48, 5), (130, 2, 64, 64),
                                              (9, 3, 80, 16), (5, 2, 192, 7), (600, 2, 256, 16), (2500, 8, 128, 32)])
def test_store_and_read_back(dtype, n, heads, dim, page):
    ops = cuda_ops(dtype)
    pages = -(-n // page) + 2
    g = torch.Generator().manual_seed(n)
    slots = torch.randperm(pages * page, generator=g)[:n].to(torch.int32)
    if n > 5:
        slots[2], slots[4] = -1, pages * page   # none of the pool's: left out
    slots = slots.to(DEV)
    k, v = rnd(n, heads * dim, seed=1, dtype=dtype), rnd(n, heads * dim, seed=2, dtype=dtype)
    k[0, :dim] = 0                                       # a row of zeros
    k[0, dim - 1] = 0.5
    v[n - 1, -dim:] = 0
    v[n // 2, :4] = torch.tensor([2.0, 1.0, -1.0, -2.0])   # halves of the largest lie between two codes
    v[n // 2, 4: dim] = v[n // 2, 4: dim].clamp(-2, 2)
    keys, values = empty_pages(pages, page, heads, dim), empty_pages(pages, page, heads, dim)
    ops.kv_write(k, v, keys, values, slots)
    check_stored(keys, k, slots, heads, dim)
    check_stored(values, v, slots, heads, dim)
    k_out, v_out = (torch.full((n, heads * dim), math.nan, dtype=dtype, device=DEV) for _ in range(2))
    ops.kv_read(keys, values, slots, k_out, v_out)
    good = ((slots >= 0) & (slots < pages * page))[:, None, None]
    for x, out in ((k, k_out), (v, v_out)):
        codes, scales = oracle.quantise(x.view(n, heads, dim))
        want = torch.where(good, codes.float() * scales[..., None], 0.0).to(dtype)   # a product of 32-bit numbers, rounded once more
        assert torch.equal(out.view(n, heads, dim), want)


@pytest.mark.parametrize("dtype", TYPES)
def test_store_takes_rows_of_a_wider_array_at_any_element(dtype):
    ops = cuda_ops(dtype)
    n, heads, dim, page = 19, 2, 64, 16
    for first in (0, 8, 3):
        wide = rnd(n, 2 * heads * dim + 12, seed=first, dtype=dtype)
        k, v = wide[:, first: first + heads * dim], wide[:, -heads * dim:]
        keys, values = empty_pages(2, page, heads, dim), empty_pages(2, page, heads, dim)
        slots = torch.arange(n, dtype=torch.int32, device=DEV).flip(0).contiguous()
        ops.kv_write(k, v, keys, values, slots)
        check_stored(keys, k.contiguous(), slots, heads, dim)
        check_stored(values, v.contiguous(), slots, heads, dim)


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_of_extreme_elements(dtype):
    """Tiny, denormal and huge rows keep the nearest codes; a row with an infinity or a NaN is read as NaN and harms nobody else."""
    ops = cuda_ops(dtype)
    heads, dim, page = 1, 32, 4
    base = rnd(12, dim, seed=5)
    factors = torch.tensor([1e-38, 1e-36, 1e-30, 1e-20, 1.0, 1e20, 1e30, 1e37, 0.0, 1.0, 1.0, 1.0], device=DEV)
    x = (base * factors[:, None]).to(dtype)
    x[0] = torch.where(x[0].abs() < 1e-44, torch.zeros_like(x[0]), x[0])
    x[9, 3], x[10, 31], x[11, 0] = math.inf, math.nan, -math.inf
    keys, values = empty_pages(3, page, heads, dim), empty_pages(3, page, heads, dim)
    slots = torch.arange(12, dtype=torch.int32, device=DEV)
    ops.kv_write(x, x, keys, values, slots)
    check_stored(keys, x, slots, heads, dim)
    k_out, v_out = torch.empty_like(x), torch.empty_like(x)
    ops.kv_read(keys, values, slots, k_out, v_out)
    assert torch.isnan(k_out[9:]).all() and torch.isfinite(k_out[:9]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,heads,kv_heads,dim,partials,with_bias,rotate", [
    (1, 28, 4, 128, 3, True, True), (5, 4, 2, 16, 1, True, True), (40, 14, 2, 64, 2, False, True), (300, 6, 3, 32, 1, True, False),
    (513, 12, 2, 128, 1, True, True), (3, 2, 2, 256, 5, False, True)])
def test_rotation_and_store(dtype, n, heads, kv_heads, dim, partials, with_bias, rotate):
    """Queries get the bits of the call over a cache in the engine's type; keys and values the codes of what that call would
    have kept in 32 bits."""
    ops, wide = cuda_ops(dtype), cuda_ops(torch.float32)
    width = (heads + 2 * kv_heads) * dim
    qkv = rnd(partials, n, width, seed=3) if partials > 1 else rnd(n, width, seed=3)
    bias = rnd(width, seed=4) if with_bias else None
    positions = torch.randint(0, 30000, (n,), generator=torch.Generator().manual_seed(1)).to(torch.int32).to(DEV)
    inv_freq = (10000.0 ** (-torch.arange(0, dim, 2).double() / dim)).float().to(DEV) if rotate else None
    page = 8
    pages = -(-n // page) + 1
    slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(2))[:n].to(torch.int32).to(DEV)
    if n > 4:
        slots[3] = -1
    q, q_same = (torch.empty(n, heads * dim, dtype=dtype, device=DEV) for _ in range(2))
    keys, values = empty_pages(pages, page, kv_heads, dim), empty_pages(pages, page, kv_heads, dim)
    ops.rope_kv_write(qkv, bias, positions, inv_freq, q, keys, values, slots, heads, kv_heads, dim)
    plain = [torch.zeros(pages, page, kv_heads, dim, dtype=dtype, device=DEV) for _ in range(2)]
    ops.rope_kv_write(qkv, bias, positions, inv_freq, q_same, *plain, slots, heads, kv_heads, dim)
    assert torch.equal(q, q_same)
    exact = [torch.zeros(pages, page, kv_heads, dim, device=DEV) for _ in range(2)]
    wide.rope_kv_write(qkv, bias, positions, inv_freq, torch.empty(n, heads * dim, device=DEV), *exact, slots, heads, kv_heads, dim)
    there = slots[slots >= 0].long()
    for pool, x in ((keys, exact[0]), (values, exact[1])):
        check_stored(pool, x.view(-1, kv_heads * dim)[there], there, kv_heads, dim)


def attend(ops, case, heads, kv_heads, dim, q_lens, ctx_lens, window=None, chunk=None, scale=None, known=True):
    out = torch.full_like(case["q"], math.nan)
    ops.paged_attention(case["q"], QuantisedPages(case["codes_k"], case["scales_k"]), QuantisedPages(case["codes_v"], case["scales_v"]),
                        case["table"], case["q_start"], case["ctx_len"], case["seq_of"], heads, kv_heads, dim,
                        dim ** -0.5 if scale is None else scale, window, out, max_q_len=max(q_lens), max_ctx_len=max(ctx_lens),
                        min_q_len=min(q_lens) if known else 0, q_lens=list(q_lens) if known else None, chunk=chunk)
    return out


def check_attention(dtype, heads, kv_heads, dim, page, q_lens, ctx_lens, seed=0, q_scale=1.0, splits=None, known=True, tensor_cores=True,
                    portion_splits=0, few_rows=False, **options):
    ops = cuda_ops(dtype)
    ops.q8_few_rows = few_rows
    ops.q8_splits, ops.tensor_core_attention, ops.portion_splits = splits, tensor_cores, portion_splits
    case = oracle.pages_case(heads, kv_heads, dim, page, q_lens, ctx_lens, dtype, seed, DEV, q_scale)
    got = attend(ops, case, heads, kv_heads, dim, q_lens, ctx_lens, known=known, **options)
    scale = options.pop("scale", None)
    want, bound = oracle.attention(case["q"], case["sequences"], q_lens, ctx_lens, heads, kv_heads, dim, dim ** -0.5 if scale is None else scale,
                                   **options)
    assert torch.isfinite(got).all()
    excess = ((got.double() - want).abs() - bound)
    assert excess.max().item() <= 0, f"off by {excess.max().item():.3e} more than the bound at {divmod(int(excess.argmax()), heads * dim)}"
    again = attend(ops, case, heads, kv_heads, dim, q_lens, ctx_lens, known=known, scale=scale, **options)
    assert torch.equal(got, again)   # no result depends on who comes first
    ops.check_status()


HEADS = [(7, 1, 128, 16), (14, 2, 64, 16), (6, 3, 32, 8), (4, 2, 16, 5), (40, 8, 128, 64), (17, 1, 48, 7), (2, 2, 256, 16), (33, 1, 80, 1)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,dim,page", HEADS)
def test_single_tokens(dtype, heads, kv_heads, dim, page):
    ctx_lens = [1, 2, 15, 31, 32, 33, 64, 65, 127, 128, 129, 300, 517]
    check_attention(dtype, heads, kv_heads, dim, page, [1] * len(ctx_lens), ctx_lens, seed=heads)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("splits", [(1, 1), (2, 1), (2, 2), (3, 1), (8, 8), (16, 8), (12, 4), (64, 1), (64, 8)])
@pytest.mark.parametrize("options", [{}, {"window": 40}, {"chunk": 48}])
def test_single_tokens_in_any_number_of_splits(dtype, splits, options):
    ctx_lens = [1, 33, 700, 1900]
    check_attention(dtype, 7, 1, 64, 16, [1] * 4, ctx_lens, splits=splits, **options)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,dim,page", HEADS)
@pytest.mark.parametrize("options", [{}, {"window": 40}, {"chunk": 48}])
def test_portions(dtype, heads, kv_heads, dim, page, options):
    q_lens, ctx_lens = [2, 5, 33, 64, 70, 130, 3], [2, 40, 33, 129, 300, 130, 517]
    check_attention(dtype, heads, kv_heads, dim, page, q_lens, ctx_lens, seed=dim, tensor_cores=False, **options)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,dim,page", HEADS)
@pytest.mark.parametrize("options", [{}, {"window": 40}, {"chunk": 48}])
@pytest.mark.parametrize("few_rows,splits", [(True, None), (True, (8, 4)), (None, None)])
def test_portions_as_few_rows_and_as_the_rule_has_them(dtype, heads, kv_heads, dim, page, options, few_rows, splits):
    check_attention(dtype, heads, kv_heads, dim, page, [40, 1, 0, 9, 2], [170, 60, 5, 9, 300], seed=8, few_rows=few_rows, splits=splits, **options)


def test_which_form_the_rule_takes():
    """Few tokens over any keys, and more over few: the form that splits keys for few rows; else tcgen05, or mma.sync."""
    for dtype, dim, many in ((torch.bfloat16, 128, "tcgen05"), (torch.float32, 128, "mma")):
        ops = cuda_ops(dtype)
        ops.q8_splits, ops.tensor_core_attention, ops.portion_splits, ops.q8_few_rows = None, True, 0, None
        for tokens, keys, few in ((2, 160, True), (4, 1008, True), (48, 320, True), (2000, 2000, False)):
            plan = ops.q8_plan(28, 4, dim, 1, keys // 16, 16, tokens, tokens, 0, tokens, [tokens], keys)
            assert plan.has_single == few and plan.tc_portions == (not few and many == "tcgen05")


@pytest.mark.parametrize("heads,kv_heads,dim,page", [(7, 1, 128, 16), (14, 2, 64, 8), (40, 8, 128, 64), (2, 2, 64, 32), (64, 1, 128, 16), (25, 1, 64, 16)])
@pytest.mark.parametrize("splits", [1, 2, 5])
@pytest.mark.parametrize("options", [{}, {"window": 40}, {"window": 300}, {"chunk": 48}])
def test_portions_on_tcgen05_in_any_number_of_splits(heads, kv_heads, dim, page, splits, options):
    q_lens, ctx_lens = [2, 40, 129, 300, 64, 17], [2, 600, 129, 420, 1111, 128]
    check_attention(torch.bfloat16, heads, kv_heads, dim, page, q_lens, ctx_lens, seed=dim, portion_splits=splits, **options)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("known", [True, False])
@pytest.mark.parametrize("options", [{}, {"window": 70}])
def test_portions_beside_single_tokens(dtype, dim, known, options):
    q_lens, ctx_lens = [1, 200, 1, 1, 37, 1], [700, 611, 1, 129, 37, 64]
    check_attention(dtype, 12, 2, dim, 16, q_lens, ctx_lens, known=known, **options)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,dim", [(6, 3, 32), (14, 2, 64), (7, 1, 128)])
@pytest.mark.parametrize("options", [{}, {"window": 70}, {"chunk": 48}])
@pytest.mark.parametrize("q_lens,ctx_lens,one", [([1, 20, 1, 50, 0, 1], [190, 90, 1, 70, 9, 33], True), ([30, 1], [31, 200], True),
                                                 ([9] + [1] * 200, [60] + [70] * 199 + [300], False)])
def test_single_tokens_in_the_portions_launch_or_in_their_own(dtype, heads, kv_heads, dim, options, q_lens, ctx_lens, one):
    """Few single tokens run beside the portions in one launch, many after them in their own."""
    ops = cuda_ops(dtype)
    ops.q8_splits, ops.tensor_core_attention, ops.portion_splits, ops.q8_few_rows = None, True, 0, False
    plan = ops.q8_plan(heads, kv_heads, dim, len(q_lens), -(-max(ctx_lens) // 16) + 2, 16, max(q_lens), 1, 0, sum(q_lens), q_lens, max(ctx_lens))
    assert (not one and not plan.tc_portions) or plan.has_single + plan.has_portions == (1 if one else 2)
    check_attention(dtype, heads, kv_heads, dim, 16, q_lens, ctx_lens, seed=6, **options)


@pytest.mark.parametrize("dtype", TYPES)
def test_large_scores(dtype):
    """Scores of some hundreds: one key takes all the weight."""
    check_attention(dtype, 4, 2, 64, 16, [1, 20, 1], [300, 90, 5], q_scale=60.0)


def pages_of(case):
    return QuantisedPages(case["codes_k"], case["scales_k"]), QuantisedPages(case["codes_v"], case["scales_v"])


FORMS = [(torch.bfloat16, 128, True), (torch.bfloat16, 64, True), (torch.bfloat16, 64, False), (torch.float32, 32, False)]


@pytest.mark.parametrize("dtype,dim,tensor_cores", FORMS)
@pytest.mark.parametrize("splits", [0, 3])
@pytest.mark.parametrize("few_rows", [False, True])
def test_rows_that_see_nothing_are_zeros(dtype, dim, tensor_cores, splits, few_rows):
    """A context shorter than the new tokens: the first of them lie before position 0.  An entry without tokens is left out, and
    rows behind the last sequence stay as they are."""
    heads, kv_heads, page = 6, 2, 16
    q_lens, ctx_lens = [5, 90, 0, 1, 1, 40], [3, 70, 9, 0, 4, 400]
    ops = cuda_ops(dtype)
    ops.tensor_core_attention, ops.portion_splits, ops.q8_splits, ops.q8_few_rows = tensor_cores, splits, (2, 2) if splits else None, few_rows
    case = oracle.pages_case(heads, kv_heads, dim, page, q_lens, ctx_lens, dtype, 3, DEV)
    more = 3
    q = torch.cat([case["q"], rnd(more, heads * dim, dtype=dtype)])
    out = torch.full_like(q, 9.0)
    owner = torch.cat([case["seq_of"], torch.full((more,), 5, dtype=torch.int32, device=DEV)])
    ops.paged_attention(q, *pages_of(case), case["table"], case["q_start"], case["ctx_len"], owner, heads, kv_heads, dim, dim ** -0.5, None, out,
                        max_q_len=90, min_q_len=0, q_lens=q_lens)
    want, bound = oracle.attention(case["q"], case["sequences"], q_lens, ctx_lens, heads, kv_heads, dim, dim ** -0.5)
    assert (out[-more:] == 9.0).all()
    got = out[:-more].double()
    assert ((got - want).abs() <= bound).all()
    assert (got[:2] == 0).all() and (got[5: 25] == 0).all() and (got[95] == 0).all()
    ops.check_status()


@pytest.mark.parametrize("dtype,dim,tensor_cores", FORMS)
@pytest.mark.parametrize("splits", [1, 3])
@pytest.mark.parametrize("ctx_lens", [[30, 700, 12], [1, 300, 60], [54, 90, 2]])
def test_whole_runs_of_rows_that_see_nothing(dtype, dim, tensor_cores, splits, ctx_lens):
    """Contexts so short that a kernel's first run of 18 tokens (128 rows of seven heads) sees nothing and its second does."""
    check_attention(dtype, 7, 1, dim, 16, [60, 37, 19], ctx_lens, seed=5, splits=(splits, 1), tensor_cores=tensor_cores, portion_splits=splits)


@pytest.mark.parametrize("dtype,dim,tensor_cores", FORMS)
@pytest.mark.parametrize("options", [{}, {"window": 30}])
@pytest.mark.parametrize("few_rows", [False, True])
def test_what_a_row_does_not_see_has_no_part_in_it(dtype, dim, tensor_cores, options, few_rows):
    """Keys and values stored from infinities, NaN and the largest numbers: rows before them are what they would be without,
    rows that see them are NaN, or large."""
    heads, kv_heads, page = 4, 2, 16
    q_lens, ctx_lens = [100, 1, 33], [150, 140, 33]
    ops = cuda_ops(dtype)
    ops.q8_few_rows = few_rows
    ops.tensor_core_attention = tensor_cores
    case = oracle.pages_case(heads, kv_heads, dim, page, q_lens, ctx_lens, dtype, 7, DEV)
    bad = {0: 120, 2: 20}   # sequence -> the position that is spoilt
    for value in (math.nan, 3e38):
        for kind in ("scales_k", "scales_v"):
            spoilt = dict(case, **{kind: case[kind].clone()})
            for s, position in bad.items():
                page_id = int(case["table"][s, position // page])
                spoilt[kind][page_id, :, position % page] = value if math.isnan(value) or kind == "scales_v" else 0.0
            got = attend(ops, spoilt, heads, kv_heads, dim, q_lens, ctx_lens, **options)
            for s, position in bad.items():
                first = int(case["q_start"][s])
                at = position - (ctx_lens[s] - q_lens[s])   # rows before this one do not see it
                rows = got[first: first + at]
                # a base that takes the spoilt key's place into account may round a weight otherwise, by no more than the bound says
                want, bound = oracle.attention(case["q"], case["sequences"], q_lens, ctx_lens, heads, kv_heads, dim, dim ** -0.5, **options)
                assert torch.isfinite(rows).all()
                assert ((rows.double() - want[first: first + at]).abs() <= bound[first: first + at]).all()
                after = got[first + at: first + min(q_lens[s], at + options.get("window", 1 << 30))]
                if math.isnan(value):
                    assert torch.isnan(after).all()
            assert torch.isfinite(got[100]).all()   # the sequence between them
    ops.check_status()


def test_values_of_uneven_sizes():
    """Value rows between 1e-6 and 1e6 of one another: every row's output is good to its own keys' sizes."""
    heads, kv_heads, dim, page = 4, 1, 64, 16
    q_lens, ctx_lens = [200, 1, 1], [300, 900, 40]
    for dtype in TYPES:
        ops = cuda_ops(dtype)
        case = oracle.pages_case(heads, kv_heads, dim, page, q_lens, ctx_lens, dtype, 11, DEV)
        factor = 10.0 ** torch.randint(-6, 7, case["scales_v"].shape, generator=torch.Generator().manual_seed(1)).float().to(DEV)
        case["scales_v"] = case["scales_v"] * factor
        for s, (keys, values) in enumerate(case["sequences"]):
            for j in range(ctx_lens[s]):
                values[1][j] = case["scales_v"][case["table"][s, j // page], :, j % page]
        got = attend(ops, case, heads, kv_heads, dim, q_lens, ctx_lens)
        want, bound = oracle.attention(case["q"], case["sequences"], q_lens, ctx_lens, heads, kv_heads, dim, dim ** -0.5)
        assert ((got.double() - want).abs() <= bound).all()


@pytest.mark.parametrize("scale", [0.0, -0.2, 3.0])
def test_scales_of_any_sign(scale):
    for dtype, dim, tensor_cores in FORMS:
        check_attention(dtype, 4, 2, dim, 16, [1, 70], [200, 180], scale=scale, tensor_cores=tensor_cores)


@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 128), (torch.bfloat16, 64), (torch.float32, 64)])
@pytest.mark.parametrize("few_rows", [False, True])
def test_pools_beyond_32_bit_offsets(dtype, dim, few_rows):
    """Pages whose codes lie more than 2^31 and 2^32 bytes into the pool: stored, read back and attended over."""
    heads, kv_heads, page = 16, 8, 64
    pages = (1 << 32) // (page * kv_heads * dim) + 40
    ops = cuda_ops(dtype)
    ops.q8_few_rows = few_rows
    keys, values = (QuantisedPages(torch.empty(pages, page, kv_heads, dim, dtype=torch.int8, device=DEV),
                                   torch.full((pages, kv_heads, page), math.nan, device=DEV)) for _ in range(2))
    ctx_lens, q_lens = [200, 333, 130], [1, 120, 1]
    ids = [[pages - 1 - 7 * s - b for b in range(-(-c // page))] for s, c in enumerate(ctx_lens)]
    ids[1][0], ids[1][2] = 3, pages // 2 + 1
    table = torch.full((3, 6), -1, dtype=torch.int32)
    for s, mine in enumerate(ids):
        table[s, : len(mine)] = torch.tensor(mine, dtype=torch.int32)
    table = table.to(DEV)
    sequences = []
    for s, context in enumerate(ctx_lens):
        pair = []
        x = [rnd(context, kv_heads * dim, seed=10 * s + i, dtype=dtype) for i in range(2)]
        slots = torch.tensor([ids[s][j // page] * page + j % page for j in range(context)], dtype=torch.int32, device=DEV)
        ops.kv_write(*x, keys, values, slots)
        back = [torch.empty_like(y) for y in x]
        ops.kv_read(keys, values, slots, *back)
        for y, z in zip(x, back):
            codes, scales = oracle.quantise(y.view(context, kv_heads, dim))
            assert torch.equal(z.view(context, kv_heads, dim), (codes.float() * scales[..., None]).to(dtype))
            pair.append((codes, scales))
        sequences.append(pair)
    q = rnd(sum(q_lens), heads * dim, seed=5, dtype=dtype)
    starts = torch.tensor([0, 1, 121, 122], dtype=torch.int32, device=DEV)
    owner = torch.repeat_interleave(torch.arange(3), torch.tensor(q_lens)).to(torch.int32).to(DEV)
    out = torch.empty_like(q)
    ops.paged_attention(q, keys, values, table, starts, torch.tensor(ctx_lens, dtype=torch.int32, device=DEV), owner, heads, kv_heads, dim,
                        dim ** -0.5, None, out, max_q_len=120, min_q_len=1, q_lens=q_lens)
    want, bound = oracle.attention(q, sequences, q_lens, ctx_lens, heads, kv_heads, dim, dim ** -0.5)
    assert ((out.double() - want).abs() <= bound).all()


@pytest.mark.parametrize("dtype,dim,tensor_cores", FORMS)
@pytest.mark.parametrize("few_rows", [False, True])
def test_a_layer_captured_and_replayed_and_on_another_stream(dtype, dim, tensor_cores, few_rows):
    """Rotation and store, then attention, as a layer has them: captured once, replayed with other positions, contexts and pages."""
    heads, kv_heads, page = 4, 2, 16
    q_lens, first = [40, 1, 1], [30, 200, 5]
    ops = cuda_ops(dtype)
    ops.q8_few_rows = few_rows
    ops.tensor_core_attention = tensor_cores
    n, width = sum(q_lens), (heads + 2 * kv_heads) * dim
    inv_freq = (10000.0 ** (-torch.arange(0, dim, 2).double() / dim)).float().to(DEV)
    keys, values = (QuantisedPages.zeros(80, page, kv_heads, dim, DEV) for _ in range(2))
    owner = torch.repeat_interleave(torch.arange(3), torch.tensor(q_lens)).to(torch.int32).to(DEV)
    starts = torch.tensor([0, 40, 41, 42], dtype=torch.int32, device=DEV)
    table = torch.randperm(80, generator=torch.Generator().manual_seed(0))[:48].view(3, 16).to(torch.int32).to(DEV)
    qkv, bias = rnd(n, width, seed=1), rnd(width, seed=2)
    positions, slots, ctx = (torch.zeros(k, dtype=torch.int32, device=DEV) for k in (n, n, 3))
    q, out = (torch.empty(n, heads * dim, dtype=dtype, device=DEV) for _ in range(2))

    def fill(before, seed):
        qkv.copy_(rnd(n, width, seed=seed))
        at = torch.cat([torch.arange(b, b + k) for b, k in zip(before, q_lens)])
        positions.copy_(at.to(torch.int32))
        ctx.copy_(torch.tensor([b + k for b, k in zip(before, q_lens)], dtype=torch.int32))
        rows = owner.cpu().long()
        slots.copy_(table.cpu()[rows, at // page] * page + at % page)

    def layer():
        ops.rope_kv_write(qkv, bias, positions, inv_freq, q, keys, values, slots, heads, kv_heads, dim)
        ops.paged_attention(q, keys, values, table, starts, ctx, owner, heads, kv_heads, dim, dim ** -0.5, None, out, max_q_len=40, min_q_len=1,
                            max_ctx_len=256, q_lens=q_lens)

    def expected():
        sequences, lens = [], ctx.tolist()
        for s, context in enumerate(lens):
            where = [(int(table[s, j // page]), j % page) for j in range(context)]
            pages_at, within = (torch.tensor(x, device=DEV) for x in zip(*where))
            sequences.append([(p.codes[pages_at, within], p.scales[pages_at, :, within]) for p in (keys, values)])
        return oracle.attention(q, sequences, q_lens, lens, heads, kv_heads, dim, dim ** -0.5)

    fill(first, 1)
    for p in (keys, values):   # what earlier steps stored
        codes, scales = oracle.quantise(rnd(80, page, kv_heads, dim, seed=3))
        p.codes.copy_(codes)
        p.scales.copy_(scales.transpose(1, 2))
    layer()
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph.capture_begin()
        layer()
        graph.capture_end()
    torch.cuda.current_stream().wait_stream(side)
    for seed, before in ((2, [30, 200, 5]), (3, [0, 0, 0]), (4, [100, 255, 17])):
        fill(before, seed)
        graph.replay()
        want, bound = expected()
        assert ((out.double() - want).abs() <= bound).all()
        replayed = out.clone()
        out.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            layer()
        torch.cuda.synchronize()
        assert torch.equal(out, replayed)
    ops.check_status()
