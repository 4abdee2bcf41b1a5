"""The 8-bit cache on the GPU at head sizes between the usual ones, in launches of either number, and in batches with padding rows."""

import pytest
import torch

from shrike_b200 import SamplingParams
from shrike_b200.cache import quantised
from shrike_b200.engine.llm_engine import LLMEngine
from shrike_b200.ops import quantised_cache
from tests.gpu_common import TOL, cuda_ops
from tests.helpers import make_model_folder, random_tokens
from tests.plain import plain_model as pm
from tests.test_gpu_cache_q8 import TYPES, check_attention, test_store_and_read_back
from tests.test_gpu_kv_cache_int8 import POINTS, weights_of
from tests.test_kv_cache_int8_host import plain_quantised, tolerance
from tests.tiny_configs import PAGE_SIZES, TINY, windows_of

pytestmark = pytest.mark.gpu
check_store_and_read_back = test_store_and_read_back
del test_store_and_read_back   # run there


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [96, 112, 144, 240])
def test_head_sizes_between_the_usual_ones(dtype, dim):
    """The elements of a head are not whole runs of 32 or 64, and 16-byte pieces of a step's keys not whole turns of a warp's."""
    check_store_and_read_back(dtype, 40, 2, dim, 16)
    ctx_lens = [1, 2, 31, 33, 64, 129, 517]
    check_attention(dtype, 6, 2, dim, 16, [1] * len(ctx_lens), ctx_lens, seed=dim)
    for few_rows, splits in ((False, None), (True, (4, 2)), (None, None)):
        for options in ({}, {"window": 40}):
            check_attention(dtype, 12, 1, dim, 7, [40, 1, 70, 2], [170, 60, 70, 300], seed=dim, few_rows=few_rows, splits=splits, **options)


@pytest.mark.parametrize("dtype,heads,kv_heads,dim", [(torch.float32, 6, 3, 32), (torch.float32, 14, 2, 64), (torch.float32, 7, 1, 128),
                                                      (torch.bfloat16, 6, 3, 32), (torch.bfloat16, 14, 2, 64), (torch.bfloat16, 7, 1, 128)])
@pytest.mark.parametrize("q_lens,ctx_lens,launches", [([1, 20, 1, 50, 0, 1], [190, 90, 1, 70, 9, 33], 1), ([30, 1], [31, 200], 1),
                                                      ([9] + [1] * 200, [60] + [70] * 199 + [300], 2)])
def test_how_many_launches_the_form_for_many_rows_takes(dtype, heads, kv_heads, dim, q_lens, ctx_lens, launches):
    """On mma.sync: one where the tables hold up to 256 keys and the CTAs find room, two behind tables of 336 keys and a portion of nine."""
    ops = cuda_ops(dtype)
    ops.tensor_core_attention, ops.q8_few_rows = False, False
    plan = ops.q8_plan(heads, kv_heads, dim, len(q_lens), -(-max(ctx_lens) // 16) + 2, 16, max(q_lens), 1, 0, sum(q_lens), q_lens, max(ctx_lens))
    assert not plan.tc_portions and plan.has_portions and plan.has_single + plan.has_portions == launches


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("key,count", [("A", 11), ("B", 21), ("C", 9)])
def test_batches_with_padding_rows(tmp_path, monkeypatch, dtype, key, count):
    """More than eight sequences are padded to a batch size: rows with slot and page -1, eagerly and in captured steps."""
    folder = make_model_folder(tmp_path, key)
    engine = LLMEngine(str(folder), block_size=PAGE_SIZES[key], num_blocks=16 * count, max_tokens_per_step=64, dtype=dtype, kv_cache="int8")
    raw, new = TINY[key], 6
    prompts = [random_tokens(raw["vocab_size"], 2 + 3 * i % 31, 70 + i) for i in range(count)]
    outs = engine.generate(prompts, SamplingParams(max_new_tokens=new, ignore_eos=True))
    assert engine.block_manager.whole()
    assert engine.generate(prompts, SamplingParams(max_new_tokens=new, ignore_eos=True)) == outs
    weights = weights_of(folder, dtype == "bfloat16")
    given = dict(rounding=POINTS if dtype == "bfloat16" else (), windows=windows_of(raw))
    plain = [pm.forward(raw, weights, prompt + out, **given) for prompt, out in zip(prompts, outs)]
    plain_quantised(monkeypatch)
    for prompt, out, logits in zip(prompts, outs, plain):
        tol = tolerance((pm.forward(raw, weights, prompt + out, **given) - logits).abs().max().item(), TOL[dtype])
        want, margins = pm.greedy_continue(raw, weights, prompt, new, **given)
        for position, (a, b, margin) in enumerate(zip(out, want, margins)):
            if a != b:
                assert margin < 2 * tol, f"token {position}: engine {a}, plain {b}, gap {margin}"
                break
    engine._check_kernels()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("key", ["A", "B", "C"])
def test_what_a_pool_held_before_has_no_part_in_it(tmp_path, dtype, key):
    """Places that nobody has written hold any codes and scales of NaN: the same tokens as from an empty pool."""
    folder = make_model_folder(tmp_path, key)
    prompts = [random_tokens(TINY[key]["vocab_size"], n, 90 + n) for n in (1, 17, 40, 5)]
    outs = []
    for poison in (False, True):
        engine = LLMEngine(str(folder), block_size=PAGE_SIZES[key], num_blocks=64, max_tokens_per_step=24, dtype=dtype, kv_cache="int8")
        if poison:
            for codes, scales in zip(engine.runner.storage.kv, engine.runner.storage.scales):
                codes.random_(-127, 128)
                scales.fill_(float("nan"))
        outs.append(engine.generate(prompts, SamplingParams(max_new_tokens=8, ignore_eos=True)))
        engine._check_kernels()
    assert outs[0] == outs[1]


@pytest.mark.parametrize("dtype", TYPES)
def test_the_calls_without_the_native_module(monkeypatch, dtype):
    """The same launches where what a call asks of its tensors is asked from Python."""
    monkeypatch.setattr(quantised_cache, "_look", lambda: quantised_cache.PlainLook)
    monkeypatch.setattr(quantised, "look_pages", None)
    check_store_and_read_back(dtype, 33, 3, 32, 8)
    check_attention(dtype, 7, 1, 128, 16, [1, 1, 1], [1, 300, 517])
    check_attention(dtype, 14, 2, 64, 16, [70, 1, 2], [300, 40, 129], window=40)
