"""Plans and workspaces of the calls over 8-bit pages, without a GPU."""

import weakref

import pytest
import torch

from shrike_b200.ops import quantised_cache
from shrike_b200.ops.cuda_ops import CudaOps, KernelError
from tests.test_kv_cache_int8_host import Library, arguments, calls  # noqa: F401  (a fixture)


@pytest.fixture
def ops(calls):  # noqa: F811
    return calls[0]


def portions(ops, tokens):
    return ops.q8_plan(4, 2, 64, 1, 1 << 16, 16, tokens, tokens, 0, tokens, [tokens])


def test_a_buffer_that_has_grown_is_given_back(ops):
    first = portions(ops, 40_000)
    held, size, generation = weakref.ref(first.portion_scratch), first.portion_scratch.numel(), ops.generation
    for tokens in (39_999, 39_998, 20):   # plans of their own, over the same buffer
        assert portions(ops, tokens).portion_scratch is first.portion_scratch
    assert ops.generation == generation
    del first
    more = portions(ops, 40_100)
    assert held() is None and ops.generation == generation + 1
    # to twice its size, or the most there may be: the next ones do not move it
    assert more.portion_scratch.numel() == min(2 * size, ops.PORTION_SCRATCH_FLOATS)
    generation = ops.generation
    portions(ops, 41_000)
    assert ops.generation == generation
    few = ops.q8_plan(4, 2, 64, 1, 4096, 16, 1, 1)   # the other buffers
    assert few.scratch is ops._q8_scratch and few.arrivals is ops._q8_arrivals and not few.arrivals.any()


def test_a_buffer_that_a_capture_has_seen_is_kept(ops, monkeypatch):
    monkeypatch.setattr(quantised_cache, "_raw_stream", lambda device: 5)
    capturing = False
    monkeypatch.setattr(quantised_cache, "_capturing", lambda: capturing)
    (keys, values), _rows, _q, _out, _index = arguments()
    tokens = 40_000
    q, out = (torch.zeros(tokens, 4 * 64, dtype=torch.bfloat16) for _ in range(2))
    table, owner = torch.zeros(1, 1 << 16, dtype=torch.int32), torch.zeros(tokens, dtype=torch.int32)

    def attend(count):
        ops.paged_attention(q[:count], keys, values, table, torch.tensor([0, count], dtype=torch.int32), torch.tensor([count], dtype=torch.int32),
                            owner[:count], 4, 2, 64, 0.125, None, out[:count], max_q_len=count, min_q_len=count, q_lens=[count])

    attend(22_000)
    before = weakref.ref(ops._q8_portion_scratch)
    capturing = True
    attend(22_000)
    capturing = False
    ops._q8_portion_scratch, keep = ops._q8_portion_scratch[:22_000], before   # as if it had been made for less
    small = ops._q8_portion_scratch
    ops._q8_plans.clear()
    attend(tokens)
    assert any(x is small for x in ops._q8_kept) and ops._q8_portion_scratch is not small and keep() is not None
    second = weakref.ref(ops._q8_portion_scratch)
    ops._q8_portion_scratch = ops._q8_portion_scratch[:10].clone()
    ops._q8_plans.clear()
    assert second() is None
    third = weakref.ref(ops._q8_portion_scratch)
    attend(tokens)   # no capture has seen this one
    assert third() is None and len(ops._q8_kept) == 1


def test_counters_are_not_made_while_a_call_is_captured(ops, monkeypatch):
    """Their zeros would be written when the sequence is replayed, and calls before that would count from anything."""
    monkeypatch.setattr(quantised_cache, "_raw_stream", lambda device: 5)
    monkeypatch.setattr(quantised_cache, "_capturing", lambda: True)
    ops.q8_splits = (64, 1)
    ops._q8_arrivals = torch.zeros(4096, dtype=torch.int32)
    assert ops.q8_plan(4, 2, 64, 2000, 64, 16, 1, 1).arrivals is ops._q8_arrivals
    with pytest.raises(KernelError, match="once before it is captured"):
        ops.q8_plan(4, 2, 64, 2100, 64, 16, 1, 1)
    monkeypatch.setattr(quantised_cache, "_capturing", lambda: False)
    assert ops.q8_plan(4, 2, 64, 2100, 64, 16, 1, 1).arrivals.numel() >= 4200


@pytest.mark.parametrize("resident", [148, 296, 592])
def test_the_counters_made_at_first_are_enough_for_the_rule(resident):
    for keys in (600, 1024, 5000, 65536, 1 << 20):
        for pairs in range(1, 8192):
            splits, cluster = CudaOps.q8_few_row_splits(keys, pairs, resident)
            assert splits == cluster or pairs <= 4096


def test_attention_on_another_device_than_the_object_s_is_refused(ops, monkeypatch):
    """Tensors and current device agree, but the workspaces and the status word are on the first device."""
    (keys, values), _rows, q, out, index = arguments()
    table = torch.zeros(3, 8, dtype=torch.int32)
    args = q, keys, values, table, index, index[1:], index[:3], 4, 2, 64, 0.125, None, out
    ops.paged_attention(*args, max_q_len=1, min_q_len=1)
    launches = ops.launches

    class Elsewhere:
        device = torch.device("cuda:1")

        def get_device(self):
            return 1

        def data_ptr(self):
            return 0

    ops.status = Elsewhere()
    with pytest.raises(KernelError, match="made for cuda:1"):
        ops.paged_attention(*args, max_q_len=1, min_q_len=1)
    assert ops.launches == launches


class Weighing(Library):
    """A library that keeps what it was asked to weigh."""

    def __init__(self, **answers):
        super().__init__()
        self.asked, self.answers = [], answers

    def __getattr__(self, name):
        plain = super().__getattr__(name)

        def launcher(*args):
            self.asked.append((name.replace("shrike_attention_q8_", ""), args))
            return self.answers.get(name.replace("shrike_attention_q8_", ""), plain(*args))
        return launcher

    def keys(self, name):
        return [args[-2] if name == "one_launch" else args[-1] for asked, args in self.asked if asked == name]


@pytest.mark.parametrize("window", [200, -200])
def test_windowed_portions_are_weighed_by_the_keys_that_they_see(ops, window):
    """Not by those of the block tables: 64 tokens behind a window of 200 over 8,192 keys are no reason for many splits."""
    lib = ops._q8_libs[64] = Weighing(tc_one_launch=0, one_launch=0, resident_ctas=592)
    ops.q8_few_rows = None
    q_lens = [64, 1, 1]
    seen = 200 + 32 - 1 + 63   # a query tile of the stand-in has 32 tokens, a key tile 64 keys
    ops.q8_plan(4, 2, 64, 3, 512, 16, 64, 1, window, 66, q_lens)
    ops.q8_few_rows = False
    ops.q8_plan(4, 2, 64, 3, 512, 16, 64, 1, window, 66, q_lens)
    for name in ("tc_one_launch", "tc_time", "tc_splits"):
        assert lib.keys(name) and set(lib.keys(name)) == {seen}, name
    short = ops.q8_plan(4, 2, 64, 3, 512, 16, 5, 1, window, 7, [5, 1, 1])   # a tile has no more tokens than the longest entry
    assert short.tc_portions and lib.keys("tc_splits")[-1] == 200 + 5 - 1 + 63
    ops.tensor_core_attention = False
    ops.q8_plan(4, 2, 64, 3, 512, 16, 64, 1, window, 66, q_lens)
    assert lib.keys("one_launch") == [200 + 33 - 1]   # 64 rows of two heads: up to 33 tokens
    ops.tensor_core_attention = True
    ops.q8_plan(4, 2, 64, 3, 512, 16, 64, 1, 0, 66, q_lens)
    ops.q8_plan(4, 2, 64, 3, 512, 16, 64, 1, 9000, 66, q_lens)
    assert lib.keys("tc_splits")[-2:] == [8192, 8192] and lib.keys("tc_one_launch")[-2:] == [8192, 8192]


def test_few_rows_behind_a_window_are_split_by_the_keys_that_they_see(ops):
    ops._q8_libs[64] = Weighing(resident_ctas=592)
    ops.q8_few_rows = True
    for tokens in (1, 100):   # eight rows of two heads: up to five tokens
        plan = ops.q8_plan(4, 2, 64, 1, 4096, 16, tokens, tokens, 64, tokens, [tokens])
        assert plan.has_single and plan.splits <= 2


def test_more_query_tiles_than_a_grid_takes_go_to_the_other_form(ops):
    """The stand-in's tiles have 32 tokens: 65,535 of them are served, one more would be refused."""
    most = 65535 * 32
    for tokens, tc in ((most, True), (most + 1, False)):
        for q_lens in ([tokens], [tokens, 1]):
            plan = ops.q8_plan(4, 2, 64, len(q_lens), 1 << 18, 16, tokens, min(q_lens), 0, sum(q_lens), q_lens)
            assert plan.tc_portions == tc and plan.has_portions
    assert not ops.q8_plan(4, 2, 64, 2, 1 << 18, 16, most, 1, 0, most + 1, None).tc_portions   # what unknown lengths may make
    ops._q8_libs[64] = Weighing(tc_tokens=256)
    assert not ops.q8_plan(256, 256, 64, 1, 1 << 20, 16, 1 << 23, 1 << 23, 0, 1 << 23, [1 << 23]).tc_portions   # 2^31 rows
