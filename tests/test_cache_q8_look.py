"""What the calls over 8-bit pages ask of their tensors: natively, and from Python where the native module cannot be built."""

import sysconfig

import pytest
import torch

import tests.test_kv_cache_int8_host as host
from shrike_b200.cache import quantised
from shrike_b200.cache.quantised import QuantisedPages
from shrike_b200.ops import build, quantised_cache
from shrike_b200.ops.quantised_cache import PlainLook
from tests.test_kv_cache_int8_host import calls  # noqa: F401  (a fixture)


def native():
    module = build.tensor_look()
    if module is None:
        pytest.skip("no headers to build the native module with")
    return module


def test_both_say_the_same_of_stores_and_readings():
    keys, values = (QuantisedPages.zeros(5, 16, 3, 32, "cpu") for _ in range(2))
    pools = (keys.codes, keys.scales, values.codes, values.scales)
    wide, slots = torch.zeros(4, 300), torch.zeros(4, dtype=torch.int32)
    k, v = wide[:, 1: 97], wide[:, 100: 196]
    dense, odd = torch.zeros(4, 96), torch.zeros(4 * 96 + 1)[1:].view(4, 96)
    other = QuantisedPages.zeros(6, 16, 3, 32, "cpu")
    narrow = QuantisedPages.zeros(5, 16, 3, 24, "cpu")
    shifted = torch.zeros(5 * 16 * 3 * 32 + 1, dtype=torch.int8)[1:].view(5, 16, 3, 32)
    cases = []
    for stores in (0, 1):
        cases += [(x, y, *pools, slots, device, code, stream, stores) for x, y in ((k, v), (dense, dense), (dense, odd), (odd, dense), (dense[:0], dense[:0]),
                                                                                  (dense[:1], k[:1]), (dense, dense[:3]), (dense, None), (dense.view(2, 2, 96), dense),
                                                                                  (dense.bfloat16(), dense.bfloat16()), (dense.to("meta"), dense),
                                                                                  (dense.t().contiguous().t(), dense), (dense[:, :95], dense), (dense.double(), dense))
                  for device, code, stream in ((-1, 0, 77), (0, 0, 77), (-1, 1, 2 ** 63 + 5))]
        cases += [(dense, dense, *pools, ints, -1, 0, 7, stores) for ints in (slots.long(), slots[:3], slots[:0], torch.zeros(8, dtype=torch.int32)[::2], slots.view(2, 2))]
        cases += [(dense, dense, a.codes, a.scales, b.codes, b.scales, slots, -1, 0, 7, stores) for a, b in ((keys, other), (other, other), (narrow, narrow))]
        cases += [(dense, dense, shifted, keys.scales, values.codes, values.scales, slots, -1, 0, 7, stores), (dense, dense, *pools, slots[:0], -1, 0, 7, stores)]
    found = [(PlainLook.cache(*case), native().cache(*case)) for case in cases]
    assert all(plain == other for plain, other in found)
    assert sum(plain is not None for plain, _ in found) > 10 and sum(plain is None for plain, _ in found) > 10


def test_both_say_the_same_of_attention():
    keys, values = (QuantisedPages.zeros(5, 16, 2, 64, "cpu") for _ in range(2))
    q, out = torch.zeros(3, 256, dtype=torch.bfloat16), torch.zeros(3, 256, dtype=torch.bfloat16)
    table, starts, context = torch.zeros(3, 8, dtype=torch.int32), torch.zeros(4, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    usual = dict(q=q, out=out, kc=keys.codes, ks=keys.scales, vc=values.codes, vs=values.scales, table=table, starts=starts, context=context, device=-1, code=1,
                 heads=4, kv_heads=2, dim=64)
    odd = torch.zeros(3 * 256 + 1, dtype=torch.bfloat16)[1:].view(3, 256)
    changes = [{}, dict(q=q.float()), dict(q=odd), dict(out=odd), dict(out=out[:2]), dict(q=q[0]), dict(q=None), dict(table=table.long()), dict(table=table[:, ::2]),
               dict(table=table[0]), dict(table=table[:, :0]), dict(table=table[:0], starts=starts[:1], context=context[:0]), dict(starts=starts[:3]),
               dict(context=starts), dict(device=0), dict(code=0), dict(heads=5), dict(heads=0), dict(kv_heads=4), dict(kv_heads=0), dict(dim=32), dict(heads=2),
               dict(vc=values.codes[:4]), dict(q=q.to("meta")), dict(context=context.to("meta")), dict(q=q[:0], out=out[:0])]
    found = [(PlainLook.attention(*{**usual, **change}.values()), native().attention(*{**usual, **change}.values())) for change in changes]
    assert all(plain == other for plain, other in found)
    assert found[0][0] is not None and sum(plain is None for plain, _ in found) > 15


def test_both_say_the_same_of_pages():
    codes, scales = torch.zeros(3, 16, 2, 64, dtype=torch.int8), torch.zeros(3, 2, 16)
    for pair in ((codes, scales), (codes.float(), scales), (codes[0], scales), (codes, scales[:2]), (codes, None), (codes[:0], scales[:0])):
        assert PlainLook.pages(*pair) == native().pages(*pair)


@pytest.fixture
def without_headers(monkeypatch, tmp_path):
    monkeypatch.setattr(sysconfig, "get_paths", lambda: {"include": str(tmp_path)})
    monkeypatch.setattr(quantised, "look_pages", None)
    for held in (build.tensor_look, quantised_cache._look):
        held.cache_clear()
    yield
    monkeypatch.undo()
    for held in (build.tensor_look, quantised_cache._look):
        held.cache_clear()


def test_the_calls_do_without_the_native_module(without_headers, calls):  # noqa: F811
    assert build.tensor_look() is None and quantised_cache._look() is PlainLook
    host.test_store_and_reading_back_refuse_what_does_not_fit(calls)
    calls[1].calls.clear()
    host.test_attention_refuses_what_does_not_fit(calls)


def test_everything_else_is_built_without_the_headers(without_headers, monkeypatch):
    built = []
    monkeypatch.setattr(build, "compile_library", lambda name, *args, **options: built.append(name))
    build.build_all((64,))
    assert "shrike_core" in built and "shrike_attention_q8_d64" in built and "shrike_tensor_look" not in built


def test_the_calls_are_packed_as_the_launchers_declare_them():
    assert quantised_cache._CACHE_CALL.size == 104 and quantised_cache._ATTENTION_CALL.size == 14 * 8 + 17 * 4   # asserted beside the structures too
