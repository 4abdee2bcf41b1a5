"""The kernels over 8-bit cache pages, as a part of `CudaOps`.

The public calls are those of the cache in the engine's type: `CudaOps.rope_kv_write`, `kv_write` and `paged_attention` come
here when they are given `QuantisedPages`; `kv_read` is this cache's own.  An engine object's calls share its scratch, so they
belong on one stream at a time, captured launch sequences included.
"""

from __future__ import annotations

import ctypes
import functools
import struct
from dataclasses import dataclass

import torch

from ..cache import quantised as quantised_pages
from ..cache.quantised import MOST_HEAD_DIM, QuantisedPages
from . import build

_c = ctypes
_P, _I, _F, _LL = _c.c_void_p, _c.c_int, _c.c_float, _c.c_longlong
DTYPE_CODE = {torch.float32: 0, torch.bfloat16: 1}
# The launchers take their arguments as one packed structure (ShrikeCacheQ8, ShrikeAttentionQ8): a call of thirty arguments takes
# ctypes two microseconds, this a third of one.
_ATTENTION_CALL = struct.Struct("=14Q16if")
_pack_attention = _ATTENTION_CALL.pack
_CACHE_CALL = struct.Struct("=8Q2q6i")
_INT32 = torch.int32
_DTYPES = {code: dtype for dtype, code in DTYPE_CODE.items()}
_device = getattr(torch._C, "_cuda_getDevice", None)          # the current device's number, and its current stream's handle:
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)   # asking torch for the objects costs more than a launch
_capturing = getattr(torch._C, "_cuda_isCurrentStreamCapturing", None)


@dataclass(frozen=True, slots=True)
class QuantisedPlan:
    """How a batch's attention over 8-bit pages is cut."""

    has_single: bool      # the form for few rows runs: single tokens, or every entry where has_portions is False
    has_portions: bool    # a form for many rows runs: longer entries, or every entry where has_single is False
    tc_portions: bool     # which is the tcgen05 kernel, else the mma.sync one
    splits: int           # CTAs that share the keys of a row tile of the former
    cluster: int          # how many of them form a thread-block cluster
    scratch: torch.Tensor | None
    arrivals: torch.Tensor | None
    tiles: int = 0        # query tiles that the tcgen05 kernel's portions make
    portion_splits: int = 1   # CTAs that share the keys of one
    portion_scratch: torch.Tensor | None = None
    lib: object = None
    launches: int = 0


class PlainLook:
    """What `tensor_look.cpp` answers, asked from Python: for where that cannot be built (no headers of Python or torch)."""

    @staticmethod
    def _tensors(*tensors) -> bool:
        return all(isinstance(x, torch.Tensor) for x in tensors)

    @staticmethod
    def _ints(tensor, count, device) -> bool:
        return tensor.get_device() == device and not tensor.is_meta and tensor.dtype is _INT32 and tensor.numel() == count and tensor.is_contiguous()

    @staticmethod
    def _both_fit(keys, values, device) -> bool:
        if keys.dim() != 4 or keys.shape != values.shape or any(x.get_device() != device or x.is_meta or x.data_ptr() % 16 for x in (keys, values)):
            return False
        pages, page_size, _heads, dim = keys.shape
        return dim % 16 == 0 and 16 <= dim <= MOST_HEAD_DIM and pages * page_size <= 0x7FFFFFFF

    @staticmethod
    def _rows(x, dtype, n, width, device) -> bool:
        return (x.shape == (n, width) and x.dtype is dtype and x.get_device() == device and not x.is_meta and (width <= 1 or x.stride(1) == 1)
                and (n <= 1 or x.stride(0) >= 0))

    @classmethod
    def pages(cls, codes, scales):
        return quantised_pages._look_here(codes, scales) if cls._tensors(codes, scales) else None

    @classmethod
    def cache(cls, k, v, key_codes, key_scales, value_codes, value_scales, slots, device, code, stream, stores):
        """The launcher's arguments (`ShrikeCacheQ8`), empty for no rows."""
        if (not cls._tensors(k, v, key_codes, key_scales, value_codes, value_scales, slots)
                or not cls._both_fit(key_codes, value_codes, device) or k.dim() != 2):
            return None
        pages, page_size, heads, dim = key_codes.shape
        n, width, dtype = k.shape[0] if stores else slots.numel(), heads * dim, _DTYPES[code]
        if not cls._ints(slots, n, device) or not all(cls._rows(x, dtype, n, width, device) for x in (k, v)) or n > 0x7FFFFFFF:
            return None
        if not stores and not all(x.is_contiguous() and x.data_ptr() % 16 == 0 for x in (k, v)):
            return None
        if n == 0:
            return b""
        return _CACHE_CALL.pack(*(x.data_ptr() for x in (k, v, key_codes, value_codes, key_scales, value_scales, slots)), stream,
                                *(x.stride(0) if n > 1 else width for x in (k, v)), code, n, heads, dim, pages, page_size)

    @classmethod
    def attention(cls, q, out, key_codes, key_scales, value_codes, value_scales, table, starts, context, device, code, heads, kv_heads, dim):
        """(tokens, sequences, blocks a sequence, out's address, (the addresses that a launch begins with))."""
        if not cls._tensors(q, out, key_codes, key_scales, value_codes, value_scales, table, starts, context):
            return None
        if (not cls._both_fit(key_codes, value_codes, device) or key_codes.shape[2:] != (kv_heads, dim) or kv_heads <= 0 or heads <= 0
                or heads % kv_heads or q.dim() != 2 or q.shape[1] != heads * dim or q.shape != out.shape or table.dim() != 2):
            return None
        if any(x.dtype is not _DTYPES[code] or x.get_device() != device or x.is_meta or not x.is_contiguous() or x.data_ptr() % 16 for x in (q, out)):
            return None
        sequences = table.shape[0]
        if not (cls._ints(table, table.numel(), device) and cls._ints(starts, sequences + 1, device) and cls._ints(context, sequences, device)):
            return None
        return (q.shape[0], sequences, table.shape[1], out.data_ptr(),
                tuple(x.data_ptr() for x in (q, key_codes, key_scales, value_codes, value_scales, table, starts, context)))


@functools.lru_cache(maxsize=None)
def _look():
    """The native module, which pages made from now on use too."""
    module = build.tensor_look()
    if module is None:
        return PlainLook
    quantised_pages.look_pages = module.pages
    return module


def _error(text):
    from .cuda_ops import KernelError

    return KernelError(text)


def _failed(code: int, what: str):
    from .cuda_ops import _check

    _check(code, what)


def quantised(keys, values) -> bool:
    """Whether a layer's cache is of 8-bit pages; both tensors of a layer have to be of one form."""
    if (type(keys) is QuantisedPages) != (type(values) is QuantisedPages):
        raise _error("keys and values must both be 8-bit pages, or neither")
    return type(keys) is QuantisedPages


class QuantisedCacheOps:
    """Mixed into `CudaOps`."""

    Q8_SCRATCH_FLOATS = 64 << 20   # at most 256 MiB for the shares of split rows: fewer splits beyond that
    _q8_captured = frozenset()     # names of the buffers that a capture has seen,
    _q8_kept = ()                  # and such buffers that are no longer in use

    def _declare_q8_core(self, lib):
        lib.shrike_kv_write_q8.argtypes = lib.shrike_kv_read_q8.argtypes = [_c.c_char_p]
        lib.shrike_rope_kv_write_q8.argtypes = [_P] * 10 + [_I] * 6 + [_LL, _I, _LL, _P]
        for name in ("shrike_kv_write_q8", "shrike_rope_kv_write_q8", "shrike_kv_read_q8"):
            getattr(lib, name).restype = _I
        self._q8_libs, self._q8_plans = {}, {}
        self._q8_scratch = self._q8_portion_scratch = None
        self._q8_arrivals = torch.zeros(4096, dtype=_INT32, device=self.device)   # more than the rule for splits ever asks for
        torch.cuda.current_stream(self.device).synchronize()   # zeros before the first call, whichever stream that is on
        self.q8_few_rows = None   # None: the rule of `_few_rows_serve`; whether the form for few rows takes portions (tests)
        self.q8_splits = None   # None: the rule of `q8_few_row_splits`; (splits, cluster) for few rows (tests)

    def _q8_lib(self, head_dim: int):
        lib = self._q8_libs.get(head_dim)
        if lib is None:
            if head_dim % 16 or not 16 <= head_dim <= MOST_HEAD_DIM:
                raise _error(f"head size {head_dim} is not served: 8-bit pages take multiples of 16 from 16 to {MOST_HEAD_DIM}")
            lib = build.attention_q8_library(head_dim)
            lib.shrike_paged_attention_q8.argtypes = lib.shrike_paged_attention_q8_tc.argtypes = [_c.c_char_p]
            lib.shrike_paged_attention_q8.restype = _I
            lib.shrike_attention_q8_tc_tokens.argtypes = [_I]
            lib.shrike_attention_q8_tc_splits.argtypes = [_I, _I, _LL]
            lib.shrike_attention_q8_tc_one_launch.argtypes = [_I, _I, _I, _LL]
            lib.shrike_attention_q8_tc_time.argtypes, lib.shrike_attention_q8_tc_time.restype = [_I, _I, _LL], _I
            lib.shrike_attention_q8_one_launch.argtypes = [_I, _LL, _LL, _LL]
            for name in ("shrike_paged_attention_q8_tc", "shrike_attention_q8_tc_tokens", "shrike_attention_q8_tc_splits",
                         "shrike_attention_q8_tc_one_launch", "shrike_attention_q8_one_launch"):
                getattr(lib, name).restype = _I
            lib.shrike_attention_q8_resident_portions.argtypes, lib.shrike_attention_q8_resident_portions.restype = [_I], _I
            for name in ("row_floats", "max_splits", "portion_rows"):
                getattr(lib, f"shrike_attention_q8_{name}").argtypes = []
                getattr(lib, f"shrike_attention_q8_{name}").restype = _I
            lib.shrike_attention_q8_resident_ctas.argtypes = [_I, _I]
            lib.shrike_attention_q8_tile_rows.argtypes = [_I]
            lib.shrike_attention_q8_resident_ctas.restype = lib.shrike_attention_q8_tile_rows.restype = _I
            self._q8_libs[head_dim] = lib
        return lib

    def _q8_buffer(self, name: str, need: int, least: int, most: int) -> torch.Tensor:
        """The object's buffer `name` with at least `need` elements, float32, or int32 zeros for the arrivals.  It grows to twice its
        size (up to `most`): few calls move it, and each move makes captured launch sequences stale (`generation`).  The old one is
        given back, unless a capture has seen it: whoever holds that sequence may replay it, and what its kernels write has to stay
        theirs.  With the doubling those that are kept are no larger than the one in use, all together."""
        held = getattr(self, name)
        if held is not None and held.numel() >= need:
            return held
        size = max(need, least, min(2 * held.numel() if held is not None else 0, most))
        if name == "_q8_arrivals" and self._q8_stream()[1] and _capturing():   # its zeros would be written by the replay, not now
            raise _error(f"attention over 8-bit pages needs {size} counters that are zero: make such a call once before it is captured")
        if name in self._q8_captured:
            self._q8_kept = (*self._q8_kept, held)
            self._q8_captured -= {name}
        self._q8_plans.clear()   # plans hold the buffers that they were made with
        held = None
        setattr(self, name, None)
        make, dtype = (torch.zeros, _INT32) if name == "_q8_arrivals" else (torch.empty, torch.float32)
        setattr(self, name, make(size, dtype=dtype, device=self.device))
        self.generation += 1
        return getattr(self, name)

    # ---- checks
    # A call takes longer on the host than its kernel takes for few tokens, so its tensors are looked at in one native call
    # (`tensor_look.cpp`: 0.3 us where the same questions from here take 2.5); what did not fit is looked up only then.
    def _q8_stream(self):
        """The current device and the handle of its current stream (or of the one that is held)."""
        device = _device()
        return device, _raw_stream(device) if self._held_stream is None else self._held_stream

    @staticmethod
    def _q8_refuse(device, named, ints=(), pages=None):
        """Says what is wrong: `named` (tensor, dtype, what), each dense; `ints` (tensor, count, what); `pages` (keys, values, kv
        heads, head size)."""
        if pages is not None:
            keys, values, num_kv_heads, head_dim = pages
            count, page_size, heads, dim = keys.shape
            if keys.shape != values.shape:
                raise _error(f"key pages {list(keys.shape)} and value pages {list(values.shape)} differ")
            if (num_kv_heads is not None and heads != num_kv_heads) or (head_dim is not None and dim != head_dim):
                raise _error(f"key cache {tuple(keys.shape)} does not fit {num_kv_heads} heads of {head_dim}")
            if dim % 16 or not 16 <= dim <= MOST_HEAD_DIM:
                raise _error(f"head size {dim} is not served: 8-bit pages take multiples of 16 from 16 to {MOST_HEAD_DIM}")
            if count * page_size > 0x7FFFFFFF:
                raise _error(f"{count} pages of {page_size} tokens: slots are 32-bit numbers")
            named = [*named, (keys.codes, torch.int8, "key codes"), (values.codes, torch.int8, "value codes")]
        for tensor, dtype, what in named:
            if tensor.get_device() != device:
                raise _error(f"{what} must be on the current device cuda:{device}, is on {tensor.device}")
            if tensor.dtype != dtype:
                raise _error(f"{what} must be {dtype}, is {tensor.dtype}")
            if not tensor.is_contiguous():
                raise _error(f"{what} must be contiguous")
            if tensor.data_ptr() % 16 and not dtype == torch.int32:
                raise _error(f"{what} must begin on 16 bytes")
        for tensor, count, what in ints:
            if tensor.get_device() != device:
                raise _error(f"{what} must be on the current device cuda:{device}, is on {tensor.device}")
            if tensor.dtype != torch.int32 or not tensor.is_contiguous() or tensor.numel() != count:
                raise _error(f"{what} must be {count} contiguous int32, is {tensor.dtype} {list(tensor.shape)}")

    @staticmethod
    def _q8_ints_fit(device, tensor, count) -> bool:
        return tensor.get_device() == device and tensor.dtype is _INT32 and tensor.numel() == count and tensor.is_contiguous()

    def _q8_rows(self, device, x, n, width, what):
        """The distance of x's rows in elements; a row's elements lie side by side."""
        if (x.get_device() != device or x.dtype is not self.dtype or x.shape != (n, width) or (width > 1 and x.stride(1) != 1)
                or (n > 1 and x.stride(0) < 0)):
            raise _error(f"{what} must be {self.dtype} [{n}, {width}] with adjacent columns on cuda:{device}, is {x.dtype} "
                         f"{list(x.shape)} on {x.device}")
        return x.stride(0) if n > 1 else width

    # ---- the cache
    def _kv_write_q8(self, k_new, v_new, keys, values, slots):
        device = _device()
        stream = _raw_stream(device) if self._held_stream is None else self._held_stream
        call = _look().cache(k_new, v_new, keys.codes, keys.scales, values.codes, values.scales, slots, device, self.code, stream, 1)
        if call is None:
            n, (_pages, _page_size, heads, dim) = k_new.shape[0], keys.dims
            self._q8_refuse(device, (), [(slots, n, "slots")], (keys, values, None, None))
            self._q8_rows(device, k_new, n, heads * dim, "new keys")
            self._q8_rows(device, v_new, n, heads * dim, "new values")
            raise _error("kv_write: the tensors do not fit 8-bit pages")
        if not call:   # no rows
            return
        self.launches += 1
        code = self.core.shrike_kv_write_q8(call)
        if code:
            _failed(code, "kv_write_q8")

    def _rope_kv_write_q8(self, qkv, bias, positions, inv_freq, q_out, keys, values, slots, num_heads, num_kv_heads, head_dim):
        from .cuda_ops import _check, _ptr

        device, stream = self._q8_stream()
        pages, page_size, _heads, _dim = keys.dims
        partials, stride = self._stack(qkv)
        n, width = qkv.shape[-2], (num_heads + 2 * num_kv_heads) * head_dim
        self._q8_refuse(device, [(q_out, self.dtype, "q")] + [(x, torch.float32, what) for x, what in (
            (bias, "bias"), (inv_freq, "inverse frequencies")) if x is not None],
            [(positions, n, "positions"), (slots, n, "slots")], (keys, values, num_kv_heads, head_dim))
        if (qkv.get_device() != device or qkv.dtype != torch.float32 or qkv.shape[-1] != width or qkv.stride(-1) != 1
                or (n > 1 and qkv.stride(-2) != width)):
            raise _error(f"qkv must be float32 rows of {width} on cuda:{device}, is {qkv.dtype} {list(qkv.shape)} on {qkv.device}")
        if q_out.numel() != n * num_heads * head_dim:
            raise _error(f"q {list(q_out.shape)} does not fit {n} tokens of {num_heads} heads of {head_dim}")
        if bias is not None and bias.numel() != width:
            raise _error(f"a bias of {bias.numel()} for rows of {width}")
        if inv_freq is not None and inv_freq.numel() != head_dim // 2:
            raise _error(f"{inv_freq.numel()} inverse frequencies for heads of {head_dim}")
        if n == 0:
            return
        self.launches += 1
        _check(self.core.shrike_rope_kv_write_q8(
            _ptr(qkv), _ptr(bias), _ptr(positions), _ptr(inv_freq), _ptr(q_out), _ptr(keys.codes), _ptr(keys.scales),
            _ptr(values.codes), _ptr(values.scales), _ptr(slots), self.code, n, num_heads, num_kv_heads, head_dim, page_size,
            pages * page_size, partials, stride, stream), "rope_kv_write_q8")

    def kv_read(self, keys, values, slots, k_out, v_out):
        """Reads tokens back from 8-bit pages: row n of `k_out` and `v_out` ([N, kv heads * head size], contiguous, in the engine's
        type) is what `slots[n]` (int32 [N]) holds, codes times scale in 32 bits rounded once; zeros for a slot that is none of
        the pool's (a negative one, say).  A row stored from an infinity or a NaN comes back as NaN."""
        if not quantised(keys, values):
            raise _error("kv_read reads 8-bit pages; a cache in the engine's type is indexed as it is")
        device = _device()
        stream = _raw_stream(device) if self._held_stream is None else self._held_stream
        call = _look().cache(k_out, v_out, keys.codes, keys.scales, values.codes, values.scales, slots, device, self.code, stream, 0)
        if call is None:
            n, (_pages, _page_size, heads, dim) = slots.numel(), keys.dims
            self._q8_refuse(device, [(k_out, self.dtype, "keys read"), (v_out, self.dtype, "values read")], [(slots, n, "slots")],
                            (keys, values, None, None))
            raise _error(f"keys and values read must be [{n}, {heads * dim}], are {list(k_out.shape)} and {list(v_out.shape)}")
        if not call:
            return
        self.launches += 1
        code = self.core.shrike_kv_read_q8(call)
        if code:
            _failed(code, "kv_read_q8")

    # ---- attention
    def q8_plan(self, num_heads, num_kv_heads, head_dim, num_seqs, max_blocks, page_size, max_q_len, min_q_len, window=0, num_tokens=0,
                q_lens=None, max_ctx_len=0) -> QuantisedPlan:
        """How a batch over 8-bit pages is cut: a function of its shape alone, so that a captured launch sequence serves every
        batch of that shape (and of its `context_class`).  `q_lens`: every entry's length, if they are known; `max_ctx_len`: the
        longest context, or 0."""
        short = 0 < max_ctx_len <= self.SHORT_CONTEXT
        shape = (num_tokens, short, max_q_len, tuple(q_lens) if q_lens is not None else None) if max_q_len > 1 else None
        key = (num_heads, num_kv_heads, head_dim, num_seqs, max_blocks, page_size, min_q_len <= 1, window, shape, self.q8_splits,
               self.tensor_core_attention, self.portion_splits, self.q8_few_rows)
        held = self._q8_plans.get(key)
        if held is not None and held[0] == self.generation:   # the scratch has not moved since
            return held[1]
        lib = self._q8_lib(head_dim)
        has_single, has_portions = min_q_len <= 1, max_q_len > 1
        # Up to 64 keys the mma.sync kernel is done before the other has set up (us, 28 heads of 128, mma.sync and tcgen05: one
        # portion of 16 tokens 5.6 and 7.4, of 64 7.3 and 9.1, four of 64 7.8 and 9.2; one of 5 tokens over 100 keys 8.9 and 8.3,
        # of 256 over 256 17.1 and 13.8, of 16 over 600 27.9 and 12.5).
        group, cta_rows = num_heads // num_kv_heads, lib.shrike_attention_q8_portion_rows()
        tile_tokens, table_keys = lib.shrike_attention_q8_tc_tokens(group), max_blocks * page_size
        tc_keys = self._keys_of_tile(table_keys, window, tile_tokens, max_q_len, 64)   # key tiles are 64 keys each, wherever a window begins
        tc_portions = bool(has_portions and tile_tokens and self.tensor_core_attention and self.dtype == torch.bfloat16
                           and page_size in (8, 16, 32, 64) and num_tokens > 0 and not short and table_keys > self.SHORT_CONTEXT)
        if tc_portions:   # no more query tiles than a grid takes, and rows that 32 bits count: the other form has no such limits
            tiles = num_tokens // tile_tokens + num_seqs if q_lens is None else sum(-(-q // tile_tokens) for q in q_lens if q > 1 or not has_single)
            tc_portions = tiles <= 65535 and num_tokens * num_heads <= 0x7FFFFFFF
        if has_single and has_portions and q_lens is not None:   # single tokens as portions, one launch for all
            if tc_portions:
                tiles = sum(-(-q // tile_tokens) for q in q_lens)
                has_single = not lib.shrike_attention_q8_tc_one_launch(tiles, sum(-(-q // tile_tokens) for q in q_lens if q > 1), num_kv_heads, tc_keys)
            else:
                ctas = num_kv_heads * sum(-(-q * group // cta_rows) for q in q_lens)
                has_single = not lib.shrike_attention_q8_one_launch(
                    self.code, ctas, self._keys_of_tile(table_keys, window, self._tokens_of_rows(cta_rows, group), max_q_len), max_q_len)
        splits, cluster, scratch, arrivals, few_tokens = 1, 1, None, None, 1
        rows = lib.shrike_attention_q8_tile_rows(group)
        if has_portions and self._few_rows_serve(lib, num_heads, num_kv_heads, table_keys, window, num_seqs, num_tokens, max_q_len, q_lens,
                                                 tile_tokens if tc_portions else 0, tc_keys, has_single):
            has_single, has_portions, tc_portions, few_tokens = True, False, False, max_q_len
        if has_single:
            pairs = num_seqs * num_kv_heads * -(-group * few_tokens // rows)
            keys = self._keys_of_tile(table_keys, window, self._tokens_of_rows(rows, group), few_tokens)
            most = lib.shrike_attention_q8_max_splits()
            splits, cluster = self.q8_splits or self.q8_few_row_splits(keys, pairs, lib.shrike_attention_q8_resident_ctas(self.code, group))
            share = rows * lib.shrike_attention_q8_row_floats() * pairs
            if splits > most or splits // cluster * share > self.Q8_SCRATCH_FLOATS:
                splits = cluster * max(1, min(most // cluster, self.Q8_SCRATCH_FLOATS // share))
            if splits > cluster:
                scratch = self._q8_buffer("_q8_scratch", splits // cluster * share, 1 << 20, self.Q8_SCRATCH_FLOATS)
                arrivals = self._q8_buffer("_q8_arrivals", pairs, 4096, 1 << 20)
        tiles, portion_splits, portion_scratch = 0, 1, None
        if tc_portions:
            if q_lens is not None:
                tiles = sum(-(-q // tile_tokens) for q in q_lens if q > 1 or not has_single)
            else:   # lengths that are not known: what the tokens can make at most
                tiles = num_tokens // tile_tokens + num_seqs
            portion_splits = self.portion_splits or lib.shrike_attention_q8_tc_splits(tiles, num_kv_heads, tc_keys)
            each = num_tokens * num_heads * (head_dim + 2)
            portion_splits = max(1, min(portion_splits, 32, self.PORTION_SCRATCH_FLOATS // each)) if num_tokens <= 8 * 65535 else 1
            if portion_splits > 1:
                portion_scratch = self._q8_buffer("_q8_portion_scratch", portion_splits * each, 1 << 22, self.PORTION_SCRATCH_FLOATS)
        plan = QuantisedPlan(has_single, has_portions, tc_portions, splits, cluster, scratch, arrivals, tiles, portion_splits, portion_scratch, lib,
                             int(has_single) + int(has_portions) + (portion_splits > 1))
        if len(self._q8_plans) >= 4096:
            self._q8_plans.clear()
        self._q8_plans[key] = (self.generation, plan)
        return plan

    @staticmethod
    def _tokens_of_rows(rows: int, group: int) -> int:
        """The tokens that `rows` rows belong to at most, `group` rows a token."""
        return (rows + group - 2) // group + 1

    @staticmethod
    def _keys_of_tile(table_keys: int, window: int, tokens: int, max_q_len: int, step: int = 1) -> int:
        """The keys that a tile of `tokens` tokens (of entries of up to `max_q_len`) can see of those that the block tables hold, in
        steps of `step` keys: what its CTAs walk, and what is worth dealing to several of them."""
        return table_keys if not window else min(table_keys, abs(window) + min(tokens, max_q_len) - 1 + step - 1)

    # In keys of the form for few rows, which a CTA's four warps share with 8 rows each: a key of the mma.sync form for many, which
    # all of them walk with 16 rows each; the tcgen05 kernel's unit of time; the least that a launch of the single tokens' own after it takes; a CTA
    # that finds nothing to do.
    Q8_MANY_ROWS_KEY, Q8_TC_UNIT, Q8_OWN_LAUNCH, Q8_EMPTY_KEYS = 5.6, 55, 400, 90

    def _few_rows_serve(self, lib, num_heads, num_kv_heads, table_keys, window, num_seqs, num_tokens, max_q_len, q_lens, tile_tokens,
                        tc_keys, own_launch) -> bool:
        """Whether the form for few rows, which splits the keys, serves a batch with portions sooner than the tcgen05 kernel (query
        tiles of `tile_tokens` tokens, which see `tc_keys` keys) or, where that does not serve (0), the mma.sync form for many rows, which walks the keys
        once for 64 rows.  The grid has a place for the longest entry's row tiles in every entry: the empty ones' CTAs take some
        time too.
        Measured, us, tcgen05 and few rows (28 heads of 128): 2 tokens over 100 keys 7.9 and 4.6, over 16,000 19.8 and 18.0; 5 over
        16,000 20.0 and 28.9; 16 over 1,000 11.2 and 10.2, over 4,000 14.5 and 18.5; 48 over 300 14.2 and 8.5, over 1,000 13.7 and
        18.1; 8 portions of 4 tokens over 4,000 32.5 and 17.7.  mma.sync and few rows (float32, 28 heads of 128): 2 tokens over 40
        keys 7.0 and 4.7, over 8,000 375 and 14; 128 over 136 12.8 and 12.0; 400 over 408 31.5 and 36.5; 3 portions of up to 64
        beside 9 single tokens over 72 keys 10.5 and 15.6, over 500 46 and 26."""
        group = num_heads // num_kv_heads
        rows = lib.shrike_attention_q8_tile_rows(group)
        grid = num_kv_heads * -(-max_q_len * group // rows)
        if grid > 65535 or grid * num_seqs > 1 << 20 or num_seqs > 65535:
            return False
        if self.q8_few_rows is not None:
            return self.q8_few_rows
        lens = q_lens if q_lens is not None else [max_q_len] * num_seqs
        keys = self._keys_of_tile(table_keys, window, self._tokens_of_rows(rows, group), max_q_len)
        pairs = num_kv_heads * sum(-(-q * group // rows) for q in lens)
        resident = lib.shrike_attention_q8_resident_ctas(self.code, group)
        few, splits = self.q8_few_row_time(keys, pairs, resident)
        few += self.Q8_EMPTY_KEYS * splits * (grid * num_seqs - pairs) / resident
        if tile_tokens:
            tiles = num_tokens // tile_tokens + num_seqs if q_lens is None else sum(-(-q // tile_tokens) for q in q_lens if q > 1 or not own_launch)
            many = lib.shrike_attention_q8_tc_time(tiles, num_kv_heads, tc_keys) * self.Q8_TC_UNIT
            if own_launch:
                singles = num_kv_heads * -(-group // rows) * sum(q == 1 for q in lens)
                many += max(self.Q8_OWN_LAUNCH, self.q8_few_row_time(keys, singles, resident)[0])
            return few < many
        cta_rows = lib.shrike_attention_q8_portion_rows()
        ctas = num_kv_heads * sum(-(-q * group // cta_rows) for q in lens)
        many_keys = self._keys_of_tile(table_keys, window, self._tokens_of_rows(cta_rows, group), max_q_len)
        return few < max(1.0, ctas / lib.shrike_attention_q8_resident_portions(self.code)) * (many_keys * self.Q8_MANY_ROWS_KEY + self.Q8_START_KEYS)

    # What a CTA costs beside its keys, in keys: its start alone, with its share's way through a cluster's shared memory, and
    # with the clusters' way through global memory.
    Q8_START_KEYS, Q8_CLUSTER_KEYS, Q8_GLOBAL_KEYS = 160, 320, 640

    @classmethod
    def q8_few_row_splits(cls, keys: int, pairs: int, resident: int):
        """(splits, cluster) of `q8_few_row_time`."""
        best = cls.q8_few_row_time(keys, pairs, resident)[1]
        return best, min(best, 8)

    @classmethod
    def q8_few_row_time(cls, keys: int, pairs: int, resident: int):
        """(time in keys, splits): CTAs that share the `keys` of each of `pairs` (entry, kv head, row tile) where the device holds
        `resident` at once, and how many of them form a cluster (all up to eight: a cluster adds up in shared memory, 2 us
        sooner than through global memory).  The count with the least time: no less than a CTA's own, and about that of all
        CTAs' work, whose contexts are of uneven lengths (three quarters of the longest, say), with half a CTA's at the end.
        Measured, us: 64 sequences of up to 4,096 keys, 8 kv heads: 94 unsplit, 87 with 2, 92 with 4, 106 with 8; one of 65,521
        keys: 65 with 16, 51 with 32, 42 with 48, 36 with 64; 8 of 1,024 keys, 4 kv heads: 9.7 with 2, 9.3 with 4, 8.9 with 8."""
        best, least = 1, None
        for splits in (1, 2, 4, 8, 16, 24, 32, 40, 48, 56, 64):
            if splits > max(1, -(-keys // 64)):
                break
            extra = cls.Q8_START_KEYS if splits == 1 else cls.Q8_CLUSTER_KEYS if splits <= 8 else cls.Q8_GLOBAL_KEYS
            each = -(-keys // (128 * splits)) * 128 + extra   # a CTA's four warps take 32 keys each at a time
            time = max(each, 0.75 * pairs * splits * each / resident + 0.5 * each)
            if least is None or time < least:
                best, least = splits, time
        return least, best

    def _paged_attention_q8(self, q, keys, values, block_table, q_start, ctx_len, seq_of_token, num_heads, num_kv_heads, head_dim,
                            scale, window, out, max_q_len, min_q_len, q_lens, max_ctx_len):
        device = _device()
        stream = _raw_stream(device) if self._held_stream is None else self._held_stream
        if device != self.status.get_device():   # workspaces are on the object's device: another one's kernels may not reach them
            raise _error(f"these kernels were made for {self.status.device}: they are called on the current device cuda:{device}")
        found = _look().attention(q, out, keys.codes, keys.scales, values.codes, values.scales, block_table, q_start, ctx_len, device,
                                  self.code, num_heads, num_kv_heads, head_dim)
        if found is None or max_q_len < 1:
            num_seqs, max_blocks = block_table.shape
            self._q8_refuse(device, [(q, self.dtype, "q"), (out, self.dtype, "attention output")], [
                (block_table, num_seqs * max_blocks, "block table"), (q_start, num_seqs + 1, "query starts"),
                (ctx_len, num_seqs, "context lengths")], (keys, values, num_kv_heads, head_dim))
            if num_heads % num_kv_heads:
                raise _error(f"{num_heads} heads do not share {num_kv_heads} kv heads evenly")
            if max_q_len < 1:
                raise _error("paged_attention over 8-bit pages needs max_q_len, the longest entry of the batch")
            raise _error(f"q {list(q.shape)} and output {list(out.shape)} must be [tokens, {num_heads * head_dim}]")
        n, num_seqs, max_blocks, out_at, at = found
        if n == 0 or num_seqs == 0:
            return
        pages, page_size, _heads, _dim = keys.dims
        window = window or 0
        plan = self.q8_plan(num_heads, num_kv_heads, head_dim, num_seqs, max_blocks, page_size, max_q_len, min_q_len, window, n, q_lens, max_ctx_len)
        tc, has_portions = plan.tc_portions, plan.has_portions
        if stream and (plan.scratch is not None or plan.portion_scratch is not None) and _capturing():   # the default stream never is
            self._q8_captured |= {"_q8_" + name for name in ("scratch", "arrivals", "portion_scratch") if getattr(plan, name) is not None}
        if tc and not self._q8_ints_fit(device, seq_of_token, n):
            self._q8_refuse(device, (), [(seq_of_token, n, "sequences of tokens")])
        sizes = (max_blocks, self.code, n, num_seqs, num_heads, num_kv_heads, page_size, pages, window, plan.has_single)
        self.launches += plan.launches
        if tc:
            scratch = plan.portion_scratch
            code = plan.lib.shrike_paged_attention_q8_tc(_pack_attention(
                *at, seq_of_token.data_ptr(), out_at, 0 if scratch is None else scratch.data_ptr(), 0, self.status.data_ptr(), stream,
                *sizes, 1, max_q_len, 0, plan.portion_splits, 1, plan.tiles, scale))
            if code:
                _failed(code, "paged_attention_q8_tc")
            has_portions = False
            if not plan.has_single:
                return
        scratch, arrivals = plan.scratch, plan.arrivals
        code = plan.lib.shrike_paged_attention_q8(_pack_attention(
            *at, 0, out_at, 0 if scratch is None else scratch.data_ptr(), 0 if arrivals is None else arrivals.data_ptr(), 0, stream,
            *sizes, has_portions, max_q_len, tc, plan.splits, plan.cluster, 0, scale))
        if code:
            _failed(code, "paged_attention_q8")
