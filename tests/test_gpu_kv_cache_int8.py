"""The engine over a cache of 8-bit pages, on the GPU: generation, captured steps, mixed batches, beside an engine of the usual kind."""

import pytest
import torch

from shrike_b200 import SamplingParams
from shrike_b200.engine.batch import StepEntry
from shrike_b200.engine.llm_engine import LLMEngine
from tests.gpu_common import TOL
from tests.helpers import make_model_folder, random_tokens, read_weights
from tests.plain import plain_model as pm
from tests.test_kv_cache_int8_host import plain_quantised, tolerance
from tests.tiny_configs import PAGE_SIZES, TINY, windows_of

pytestmark = pytest.mark.gpu


def weights_of(folder, bf16):
    weights = read_weights(folder)
    return {k: (v.to(torch.bfloat16) if bf16 and v.dim() >= 2 else v) for k, v in weights.items()}


# keys and values are quantised from 32 bits: no rounding to bfloat16 before
POINTS = [p for p in pm.ROUNDING_POINTS if p not in ("k", "v", "kv")]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("key,lengths,new", [("A", (5, 17, 33), 8), ("B", (1, 9, 40, 64, 70), 6), ("C", (3, 40, 29), 8)])
def test_generation_over_an_int8_cache_matches_plain(tmp_path, monkeypatch, key, lengths, new, dtype):
    folder = make_model_folder(tmp_path, key)
    engine = LLMEngine(str(folder), block_size=PAGE_SIZES[key], num_blocks=64, max_tokens_per_step=24, dtype=dtype, kv_cache="int8")
    assert engine.runner.storage.kv[0].dtype is torch.int8
    raw = TINY[key]
    prompts = [random_tokens(raw["vocab_size"], n, 30 + n) for n in lengths]
    outs = engine.generate(prompts, SamplingParams(max_new_tokens=new, ignore_eos=True))
    assert engine.block_manager.whole()
    again = engine.generate(prompts, SamplingParams(max_new_tokens=new, ignore_eos=True))   # by now on captured steps
    assert again == outs
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


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_logits_do_not_depend_on_how_a_request_is_cut(tmp_path, monkeypatch, dtype):
    """Whole, token by token, in portions beside another request's tokens: the plain model's logits within the tolerance."""
    folder = make_model_folder(tmp_path, "B")
    ids, other = random_tokens(384, 60, 3), random_tokens(384, 60, 4)
    given = weights_of(folder, dtype == "bfloat16"), ids, torch.float64, POINTS if dtype == "bfloat16" else ()
    plain = pm.forward(TINY["B"], *given)
    plain_quantised(monkeypatch)
    want = pm.forward(TINY["B"], *given)
    tol = tolerance((want - plain).abs().max().item(), TOL[dtype])
    runner = LLMEngine(str(folder), block_size=8, num_blocks=40, dtype=dtype, kv_cache="int8").runner
    for cuts in ([60], [1] * 60, [7, 1, 30, 1, 1, 20], [33, 27]):
        mine, theirs = runner.cache.open(), runner.cache.open()
        at, rows = 0, []
        for n in cuts:
            m = min(n, 5)
            for cache, count in ((mine, n), (theirs, m)):
                runner.cache.append(cache, at, count)
            rows.append(runner.step([StepEntry(mine, ids[at: at + n], at, list(range(n))), StepEntry(theirs, other[at: at + m], at, [0])])[:n].clone())
            at += n
            runner.cache.advance(mine, at)
            runner.cache.append(theirs, at - n + m, n - m) if n > m else None
            runner.cache.advance(theirs, at)
        runner.cache.free(mine)
        runner.cache.free(theirs)
        got = torch.cat(rows).cpu()
        assert torch.isfinite(got).all()
        assert (got.double() - want).abs().max().item() <= tol, cuts
        runner.ops.check_status()


def test_an_int8_pool_takes_about_half_the_memory_and_stands_beside_the_usual_one(tmp_path):
    folder = make_model_folder(tmp_path, "B")
    engines = [LLMEngine(str(folder), block_size=16, num_blocks=20, dtype="bfloat16", kv_cache=cache) for cache in (None, "int8", None)]
    small, usual = engines[1].runner.bytes_per_page, engines[0].runner.bytes_per_page
    assert small * 64 == usual * 36   # 32 codes and a scale of four bytes for 32 elements of two
    prompts = [random_tokens(384, n, 60 + n) for n in (3, 19, 41)]
    params = SamplingParams(max_new_tokens=6, ignore_eos=True)
    outs = [engine.generate(prompts, params) for engine in engines]
    assert outs[0] == outs[2]
    assert engines[1].runner.model.has_one_kernel is False


def test_warm_up_and_sampling_over_an_int8_cache(tmp_path):
    folder = make_model_folder(tmp_path, "B")
    engine = LLMEngine(str(folder), block_size=8, num_blocks=64, dtype="bfloat16", kv_cache="int8")
    engine.warm_up((1, 16, 64))
    prompts = [random_tokens(384, n, 40 + n) for n in (1, 9, 40)]
    params = [SamplingParams(max_new_tokens=12, temperature=0.8, top_p=0.9, ignore_eos=True, seed=500 + i) for i in range(3)]
    outs = engine.generate(prompts, params)
    assert [len(o) for o in outs] == [12] * 3 and engine.generate(prompts, params) == outs
    engine._check_kernels()
