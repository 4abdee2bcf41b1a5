"""The 8-bit cache's host side, without a GPU: pages, pools, the engine's option, what the calls refuse and how they are cut."""

import math
import struct

import numpy as np
import pytest
import torch

import shrike_b200.models  # noqa: F401
from shrike_b200 import SamplingParams
from shrike_b200.cache import quantised
from shrike_b200.cache.quantised import QuantisedPages
from shrike_b200.cli import parse_args
from shrike_b200.config import parse_config
from shrike_b200.engine.batch import StepEntry
from shrike_b200.engine.llm_engine import LLMEngine
from shrike_b200.engine.runner import ModelRunner
from shrike_b200.ops import quantised_cache
from shrike_b200.ops.cuda_ops import CudaOps, KernelError
from shrike_b200.weights import random_tensors
from tests import cache_q8_oracle as oracle
from tests.emulated_ops import EmulatedOps
from tests.helpers import random_tokens
from tests.kavedra_configs import KAVEDRA
from tests.plain import plain_model as pm
from tests.tiny_configs import PAGE_SIZES, SEEDS, TINY, windows_of


class Int8Ops(EmulatedOps):
    """The stand-in with 8-bit pages: stored as the kernels store them, read back before the plain attention."""

    def kv_write(self, k_new, v_new, keys, values, slots):
        if not isinstance(keys, QuantisedPages):
            return super().kv_write(k_new, v_new, keys, values, slots)
        pages, page, heads, dim = keys.shape
        for pool, x in ((keys, k_new), (values, v_new)):
            codes, scales = oracle.quantise(x.reshape(-1, heads, dim))
            for row, slot in enumerate(slots.tolist()):
                if 0 <= slot < pages * page:
                    pool.codes[slot // page, slot % page] = codes[row]
                    pool.scales[slot // page, :, slot % page] = scales[row]

    def paged_attention(self, q, keys, values, *args, **options):
        if isinstance(keys, QuantisedPages):
            keys, values = (x.codes.float() * x.scales.transpose(1, 2)[..., None] for x in (keys, values))
        return super().paged_attention(q, keys, values, *args, **options)


def plain_quantised(monkeypatch):
    """The plain model with keys and values as the cache keeps them."""
    attention = pm.causal_attention

    def quantised_attention(q, k, v, window=None):
        k, v = ((codes.double() * scales.double()[..., None]).to(k.dtype) for codes, scales in (oracle.quantise(k), oracle.quantise(v)))
        return attention(q, k, v, window)

    monkeypatch.setattr(pm, "causal_attention", quantised_attention)


def engine_for(key, **kw):
    config = parse_config(TINY[key])
    weights = random_tensors(config, SEEDS[key])
    options = dict(block_size=PAGE_SIZES[key], dtype="float32", device="cpu", config=config, tensors=dict(weights), ops=Int8Ops(),
                   kv_cache="int8")
    options.update(kw)
    return LLMEngine(None, **options), weights


# How far logits may be from the plain model's over the same 8 bits.  Rounding moves every one of n elements by up to half a step
# (a twelfth of a squared step on average), which is what `effect`, the difference that the 8 bits make in the plain model, shows.
# Elements within d steps of a border fall the other way where the layers before differ by d: a share of 2 d of them moves by a
# whole step.  The two effects are as sqrt(2 d n) to sqrt(n / 12): sqrt(24 d).  A flipped code moves its layer's output by about
# 1 % of one key's share, below 1e-4 of a row's largest element, which is d = 127e-4 / 2 steps in the next layer at most: 0.4.
def tolerance(effect, usual=2e-5):
    return usual + 0.4 * effect


@pytest.mark.parametrize("key", ["A", "C"])
def test_step_function_over_an_int8_pool_matches_plain(key, monkeypatch):
    raw = TINY[key]
    config = parse_config(raw)
    weights = random_tensors(config, SEEDS[key])
    ids = random_tokens(raw["vocab_size"], 60, 5)
    plain = pm.forward(raw, weights, ids, windows=windows_of(raw)).numpy()
    plain_quantised(monkeypatch)
    want = pm.forward(raw, weights, ids, windows=windows_of(raw)).numpy()
    tol = tolerance(np.abs(want - plain).max())
    runner = ModelRunner(config, dict(weights), Int8Ops(), "cpu", "float32", page_size=16, num_pages=6, max_slots=2, kv_cache="int8")
    cache, pos, rows = runner.cache.open(), 0, []
    for n in [7, 2, 5, 3, 2, 15, 16, 8, 1, 1]:
        runner.cache.append(cache, pos, n)
        rows.append(runner.step([StepEntry(cache, ids[pos:pos + n], pos, list(range(n)))]).clone())
        pos += n
        runner.cache.advance(cache, pos)
    np.testing.assert_allclose(torch.cat(rows).numpy(), want, atol=tol)


def test_generate_over_an_int8_pool_with_preemption(monkeypatch):
    engine, weights = engine_for("B", max_tokens_per_step=24, max_running=4, num_blocks=20)
    prompts = [random_tokens(384, n, 40 + n) for n in (1, 9, 40, 64, 70)]
    outs = engine.generate(prompts, SamplingParams(max_new_tokens=12, ignore_eos=True))
    assert engine.scheduler.num_preemptions >= 1 and engine.block_manager.whole()
    plain = [pm.forward(TINY["B"], weights, prompt + out) for prompt, out in zip(prompts, outs)]
    plain_quantised(monkeypatch)
    for prompt, out, logits in zip(prompts, outs, plain):
        want, margins = pm.greedy_continue(TINY["B"], weights, prompt, 12)
        tol = tolerance((pm.forward(TINY["B"], weights, prompt + out) - logits).abs().max().item())
        for a, b, margin in zip(out, want, margins):
            if a != b:
                assert margin < 2 * tol
                break


def test_an_int8_pool_is_codes_and_scales():
    engine, _ = engine_for("B", num_blocks=7)
    storage, config = engine.runner.storage, engine.config
    spec = config.layers[0].mixer
    layers = len(config.layers)
    assert storage.kv[0].dtype is torch.int8 and tuple(storage.kv[0].shape) == (layers, 2, 7, 8, spec.num_kv_heads, spec.head_dim)
    assert storage.scales[0].dtype is torch.float32 and tuple(storage.scales[0].shape) == (layers, 2, 7, spec.num_kv_heads, 8)
    group, keys, values = storage.keys_values(1)
    assert group == 0 and isinstance(keys, QuantisedPages) and keys.codes.data_ptr() == storage.kv[0][1][0].data_ptr()
    assert values.scales.data_ptr() == storage.scales[0][1][1].data_ptr() and storage.keys_values(1)[1] is keys
    assert engine.runner.bytes_per_page == layers * 2 * 8 * spec.num_kv_heads * (spec.head_dim + 4)
    assert storage.bytes() == 7 * engine.runner.bytes_per_page
    plain, _ = engine_for("B", num_blocks=7, kv_cache=None, ops=EmulatedOps())
    assert plain.runner.storage.scales == [] and plain.runner.bytes_per_page == layers * 2 * 8 * spec.num_kv_heads * spec.head_dim * 4


def test_the_option_is_refused_where_it_cannot_be_served():
    with pytest.raises(ValueError, match="kv_cache 'int4'"):
        engine_for("A", kv_cache="int4")
    config = parse_config(KAVEDRA["A"])
    with pytest.raises(ValueError, match="keeps its cache in the engine's dtype only"):
        LLMEngine(None, dtype="float32", device="cpu", config=config, tensors={}, ops=Int8Ops(), kv_cache="int8")


def test_the_command_line_has_the_option():
    assert parse_args(["--kv-cache", "int8"]).kv_cache == "int8" and parse_args([]).kv_cache is None
    with pytest.raises(SystemExit):
        parse_args(["--kv-cache", "int4"])


def test_pages_say_what_is_wrong():
    codes, scales = torch.zeros(3, 16, 2, 64, dtype=torch.int8), torch.zeros(3, 2, 16)
    pages = QuantisedPages(codes, scales)
    assert pages.dims == (3, 16, 2, 64) and pages.shape == codes.shape and pages.bytes() == codes.numel() + 4 * scales.numel()
    for bad_codes, bad_scales in ((codes.float(), scales), (codes[0], scales), (codes[:, ::2], scales), (codes, scales.half()),
                                  (codes, scales[:2]), (codes, torch.zeros(3, 16, 2)), (codes, torch.zeros(3, 2, 32)[..., ::2])):
        with pytest.raises(ValueError, match="must be a contiguous"):
            QuantisedPages(bad_codes, bad_scales)
    with pytest.raises(ValueError, match="are on"):
        QuantisedPages(codes, scales.to("meta"))


def test_the_native_look_at_tensors_sees_what_the_plain_one_sees():
    look = quantised_cache._look()
    codes, scales = torch.zeros(3, 16, 2, 64, dtype=torch.int8), torch.zeros(3, 2, 16)
    pairs = [(codes, scales), (codes.float(), scales), (codes[0], scales), (codes[:, ::2], scales), (codes, scales.half()), (codes, scales[:2]),
             (codes, torch.zeros(3, 16, 2)), (codes, torch.zeros(3, 2, 32)[..., ::2]), (codes, scales.to("meta")), (codes[:0], scales[:0]),
             (codes.to("meta"), scales.to("meta"))]
    for pair in pairs:
        assert look.pages(*pair) == quantised._look_here(*pair)
    assert look.pages(codes, None) is None
    with pytest.raises(TypeError):
        look.pages(codes)


def test_a_store_s_arguments_as_the_launcher_gets_them():
    look = quantised_cache._look()
    keys, values = (QuantisedPages.zeros(5, 16, 3, 32, "cpu") for _ in range(2))
    wide, slots = torch.zeros(4, 300), torch.zeros(4, dtype=torch.int32)
    k, v = wide[:, 1: 97], wide[:, 100: 196]
    pools = (keys.codes, keys.scales, values.codes, values.scales)
    got = struct.unpack("=8Q2q6i", look.cache(k, v, *pools, slots, -1, 0, 77, 1))
    assert got == (k.data_ptr(), v.data_ptr(), keys.codes.data_ptr(), values.codes.data_ptr(), keys.scales.data_ptr(), values.scales.data_ptr(),
                   slots.data_ptr(), 77, 300, 300, 0, 4, 3, 32, 5, 16)
    assert look.cache(k, v, *pools, slots, -1, 0, 77, 0) is None            # read back: dense rows on 16 bytes
    assert look.cache(k[:0], v[:0], *pools, slots[:0], -1, 0, 77, 1) == b""
    for args in ((k, v, *pools, slots, 0, 0, 77, 1), (k, v, *pools, slots, -1, 1, 77, 1), (k.to("meta"), v, *pools, slots, -1, 0, 77, 1),
                 (k, v[:3], *pools, slots, -1, 0, 77, 1), (k, v, *pools, slots[1:], -1, 0, 77, 1), (k, None, *pools, slots, -1, 0, 77, 1)):
        assert look.cache(*args) is None
    with pytest.raises(TypeError):
        look.cache(k, v, *pools, slots, -1, 0, "stream", 1)


class Library:
    """Kernels that must not be launched."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def launcher(*args):
            self.calls.append(name)
            return {"shrike_attention_q8_tile_rows": 8, "shrike_attention_q8_resident_ctas": 592, "shrike_attention_q8_row_floats": 66,
                    "shrike_attention_q8_max_splits": 64, "shrike_attention_q8_tc_tokens": 32, "shrike_attention_q8_tc_splits": 3, "shrike_attention_q8_portion_rows": 64,
                    "shrike_attention_q8_resident_portions": 444, "shrike_attention_q8_tc_time": 0}.get(name, 0)
        return launcher


@pytest.fixture
def calls(monkeypatch):
    """The package's kernels with a library that only counts, on tensors of the CPU (whose device number is -1)."""
    monkeypatch.setattr(quantised_cache, "_device", lambda: -1)
    monkeypatch.setattr(quantised_cache, "_raw_stream", lambda device: 0)
    ops = CudaOps.__new__(CudaOps)
    lib = Library()
    ops.dtype, ops.code, ops.device, ops.core = torch.bfloat16, 1, torch.device("cpu"), lib
    ops.launches = ops.generation = ops.portion_splits = 0
    ops._held_stream, ops.tensor_core_attention, ops.status = None, True, torch.zeros(4, dtype=torch.int32)
    ops._q8_libs, ops._q8_plans = {64: lib}, {}
    ops._q8_scratch = ops._q8_arrivals = ops._q8_portion_scratch = ops.q8_splits = None
    ops.q8_few_rows = False
    return ops, lib


def arguments(dim=64, heads=4, kv_heads=2, page=16, tokens=3):
    pool = [QuantisedPages.zeros(4, page, kv_heads, dim, "cpu") for _ in range(2)]
    rows = [torch.zeros(tokens, kv_heads * dim, dtype=torch.bfloat16) for _ in range(2)]
    q, out = (torch.zeros(tokens, heads * dim, dtype=torch.bfloat16) for _ in range(2))
    index = torch.arange(tokens + 1, dtype=torch.int32)
    return pool, rows, q, out, index


def test_store_and_reading_back_refuse_what_does_not_fit(calls):
    ops, lib = calls
    (keys, values), (k, v), _q, _out, index = arguments()
    slots = index[:3]
    ops.kv_write(k, v, keys, values, slots)
    ops.kv_read(keys, values, slots, k, v)
    assert lib.calls == ["shrike_kv_write_q8", "shrike_kv_read_q8"] and ops.launches == 2
    tensor = torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16)
    wide = torch.zeros(3, 128 * 2 + 8, dtype=torch.bfloat16)
    ops.kv_write(wide[:, 3:131], wide[:, 131:259], keys, values, slots)   # rows of a wider array
    shifted = torch.zeros(3 * 128 + 1, dtype=torch.bfloat16)[1:].view(3, 128)
    other = QuantisedPages.zeros(5, 16, 2, 64, "cpu")
    refused = [
        lambda: ops.kv_write(k, v, keys, tensor, slots), lambda: ops.kv_write(k, v, tensor, values, slots),
        lambda: ops.kv_write(k.float(), v, keys, values, slots), lambda: ops.kv_write(k, v[:, :64], keys, values, slots),
        lambda: ops.kv_write(k, v[:2], keys, values, slots), lambda: ops.kv_write(k.t().contiguous().t(), v, keys, values, slots),
        lambda: ops.kv_write(k, v, keys, values, slots.long()), lambda: ops.kv_write(k, v, keys, values, index),
        lambda: ops.kv_write(k, v, keys, other, slots),
        lambda: ops.kv_read(tensor, tensor, slots, k, v), lambda: ops.kv_read(keys, values, slots, k.float(), v),
        lambda: ops.kv_read(keys, values, slots, k, v[:2]), lambda: ops.kv_read(keys, values, slots, shifted, v),
        lambda: ops.kv_read(keys, values, slots, wide[:, :128], v), lambda: ops.kv_read(keys, values, slots.float(), k, v),
    ]
    for call in refused:
        with pytest.raises(KernelError):
            call()
    for dim in (8, 40, 272):
        narrow = [QuantisedPages.zeros(4, 16, 1, dim, "cpu") for _ in range(2)]
        row = torch.zeros(3, dim, dtype=torch.bfloat16)
        with pytest.raises(KernelError, match="is not served"):
            ops.kv_write(row, row, *narrow, slots)
    assert len(lib.calls) == 3
    ops.kv_write(k[:0], v[:0], keys, values, slots[:0])   # nothing to do
    assert len(lib.calls) == 3


def test_tensors_on_another_device_than_the_current_one_are_refused(calls, monkeypatch):
    ops, lib = calls
    monkeypatch.setattr(quantised_cache, "_device", lambda: 1)
    (keys, values), (k, v), q, out, index = arguments()
    for call in (lambda: ops.kv_write(k, v, keys, values, index[:3]), lambda: ops.kv_read(keys, values, index[:3], k, v),
                 lambda: ops.rope_kv_write(torch.zeros(3, 512), None, index[:3], None, q, keys, values, index[:3], 4, 2, 64),
                 lambda: ops.paged_attention(q, keys, values, torch.zeros(3, 2, dtype=torch.int32), index, index[1:], index[:3], 4, 2, 64,
                                             0.1, None, out, max_q_len=1)):
        with pytest.raises(KernelError, match="current device cuda:1"):
            call()
    assert lib.calls == []


def test_rotation_and_store_refuses_what_does_not_fit(calls):
    ops, lib = calls
    (keys, values), (k, v), q, _out, index = arguments()
    qkv, slots = torch.zeros(3, 8 * 64), index[:3]
    positions, inv_freq, bias = index[:3], torch.zeros(32), torch.zeros(512)
    ops.rope_kv_write(qkv, bias, positions, inv_freq, q, keys, values, slots, 4, 2, 64)
    ops.rope_kv_write(torch.zeros(2, 3, 512), None, positions, None, q, keys, values, slots, 4, 2, 64)
    assert lib.calls == ["shrike_rope_kv_write_q8"] * 2
    for args in ((qkv.double(), bias, positions, inv_freq, q, keys, values, slots, 4, 2, 64),
                 (qkv[:, :500], bias, positions, inv_freq, q, keys, values, slots, 4, 2, 64),
                 (qkv, bias[:500], positions, inv_freq, q, keys, values, slots, 4, 2, 64),
                 (qkv, bias, positions.long(), inv_freq, q, keys, values, slots, 4, 2, 64),
                 (qkv, bias, positions, inv_freq[:16], q, keys, values, slots, 4, 2, 64),
                 (qkv, bias, positions, inv_freq, q.float(), keys, values, slots, 4, 2, 64),
                 (qkv, bias, positions, inv_freq, q[:2], keys, values, slots, 4, 2, 64),
                 (qkv, bias, positions, inv_freq, q, keys, values, index, 4, 2, 64),
                 (qkv, bias, positions, inv_freq, q, keys, values, slots, 6, 1, 64)):
        with pytest.raises(KernelError):
            ops.rope_kv_write(*args)
    with pytest.raises(KernelError, match="not to both"):
        ops.rope_kv_write(qkv, bias, positions, inv_freq, q, keys, values, slots, 4, 2, 64, k_out=k, v_out=v)
    assert len(lib.calls) == 2


def test_attention_refuses_what_does_not_fit(calls):
    ops, lib = calls
    (keys, values), _rows, q, out, index = arguments()
    table, ctx = torch.zeros(3, 8, dtype=torch.int32), index[1:]

    def attend(q=q, keys=keys, values=values, table=table, starts=index, ctx=ctx, owner=index[:3], heads=4, kv_heads=2, dim=64, out=out,
               max_q_len=1, min_q_len=1, **options):
        ops.paged_attention(q, keys, values, table, starts, ctx, owner, heads, kv_heads, dim, 0.125, options.pop("window", None), out,
                            max_q_len=max_q_len, min_q_len=min_q_len, **options)

    attend()
    attend(window=7)
    attend(chunk=9)
    launched = lib.calls.count("shrike_paged_attention_q8")
    assert launched == 3
    attend(max_q_len=2, q_lens=[2, 1, 0])   # longer entries beside single tokens: both kernels
    assert lib.calls.count("shrike_paged_attention_q8_tc") == 1 and lib.calls.count("shrike_paged_attention_q8") == 4
    attend(max_q_len=2, q_lens=[2, 1, 0], max_ctx_len=64)   # few keys: one launcher for both
    assert lib.calls.count("shrike_paged_attention_q8_tc") == 1 and lib.calls.count("shrike_paged_attention_q8") == 5
    shifted = torch.zeros(3 * 256 + 1, dtype=torch.bfloat16)[1:].view(3, 256)
    for options in (dict(softcap=3.0), dict(slopes=torch.zeros(4)), dict(sinks=torch.zeros(4)), dict(window=4, keep_first=2),
                    dict(window=4, chunk=4), dict(max_q_len=0), dict(heads=5), dict(heads=2), dict(kv_heads=4), dict(dim=32),
                    dict(q=q.float()), dict(out=out[:2]), dict(out=shifted), dict(q=shifted), dict(table=table.long()),
                    dict(starts=index[:3]), dict(ctx=index), dict(values=QuantisedPages.zeros(4, 8, 2, 64, "cpu")),
                    dict(values=torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16)), dict(max_q_len=2, owner=index)):
        with pytest.raises(KernelError):
            attend(**options)
    assert lib.calls.count("shrike_paged_attention_q8") == 5


@pytest.mark.parametrize("resident", [148, 592])
def test_splits_of_few_rows(resident):
    """Never more CTAs than there are steps to share, never past the kernel's limits, in whole clusters of at most eight."""
    for keys in (1, 31, 64, 65, 128, 129, 500, 1000, 5000, 65536, 1 << 20):
        for pairs in (1, 2, 7, 40, 148, 512, 5000):
            splits, cluster = CudaOps.q8_few_row_splits(keys, pairs, resident)
            assert 1 <= splits <= 64 and 1 <= cluster <= 8 and splits % cluster == 0
            assert splits <= max(1, math.ceil(keys / 64))
    assert CudaOps.q8_few_row_splits(64, 1, resident) == (1, 1)
    assert CudaOps.q8_few_row_splits(1 << 20, 1, resident)[0] == 64


def test_plans_are_kept_by_shape_until_the_scratch_moves(calls):
    ops, _lib = calls
    first = ops.q8_plan(4, 2, 64, 3, 64, 16, 1, 1)
    assert first.has_single and not first.has_portions and first.splits > 1 and first.launches == 1
    assert ops.q8_plan(4, 2, 64, 3, 64, 16, 1, 1) is first
    mixed = ops.q8_plan(4, 2, 64, 3, 64, 16, 40, 1, 0, 42, [40, 1, 1])
    assert mixed.has_single and mixed.tc_portions and mixed.tiles == 2 and mixed.portion_splits == 3 and mixed.launches == 3
    assert mixed.portion_scratch is not None and ops.generation > 0
    unknown = ops.q8_plan(4, 2, 64, 3, 64, 16, 40, 0, 0, 42, None)
    assert unknown.tiles == 42 // 32 + 3   # at most
    assert ops.q8_plan(4, 2, 64, 3, 64, 16, 1, 1) is not first   # the scratch has moved: a plan of its own
    assert not ops.q8_plan(4, 2, 64, 3, 64, 5, 40, 1, 0, 42, [40, 1, 1]).tc_portions   # pages of five tokens: the other kernel


def test_plans_of_unknown_lengths_differ_by_the_longest(calls):
    """The form for few rows has a place for the longest entry's rows in every entry, in its grid and in its scratch."""
    ops, _lib = calls
    ops.q8_few_rows, ops.q8_splits = True, (64, 8)
    ops.tensor_core_attention = False
    needs = []
    for longest in (2, 4000, 2):
        plan = ops.q8_plan(4, 2, 64, 3, 1024, 16, longest, 1, 0, 4002)
        assert plan.has_single and not plan.has_portions
        pairs = 3 * 2 * -(-2 * longest // 8)
        assert plan.splits % plan.cluster == 0
        if plan.splits > plan.cluster:
            assert plan.scratch.numel() >= plan.splits // plan.cluster * 8 * 66 * pairs and plan.arrivals.numel() >= pairs
        needs.append(pairs)
    assert needs[1] > needs[0]


def test_codes_of_bfloat16_elements_fall_on_the_right_side_of_every_border():
    """The store's shorter form for bfloat16 (a 32-bit product, and halves of the largest element apart), for every pair of
    significands, against integers: 127 x / a to the nearest, halves to even."""
    significands = np.arange(128, 256, dtype=np.int64)
    for shift in range(10):
        for a in significands:
            x = significands if shift else significands[significands <= a]
            in_32 = x.astype(np.float32) / np.float32(2 ** shift)
            code = np.rint(in_32 * (np.float32(127) / np.float32(a))).astype(np.int64)
            code = np.where(2 * in_32 == np.float32(a), 64, code)
            whole, left = np.divmod(127 * x, a << shift)
            exact = whole + (2 * left > (a << shift)) + ((2 * left == (a << shift)) & (whole % 2 == 1))
            assert (code == exact).all()
