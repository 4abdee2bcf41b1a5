"""The kernels over 8-bit cache pages, as a part of `CudaOps`.

The public calls are those of the cache in the engine's type: `CudaOps.rope_kv_write`, `kv_write` and `paged_attention` come
here when they are given `QuantisedPages`; `kv_read` is this cache's own.  An engine object's calls share its scratch, so they
belong on one stream at a time, captured launch sequences included.
"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass

import torch

from ..cache.quantised import QuantisedPages
from . import build

_c = ctypes
_P, _I, _F, _LL = _c.c_void_p, _c.c_int, _c.c_float, _c.c_longlong
DTYPE_CODE = {torch.float32: 0, torch.bfloat16: 1}
MOST_HEAD_DIM = 256   # of the kernels over 8-bit pages


@dataclass(frozen=True)
class QuantisedPlan:
    """How a batch's attention over 8-bit pages is cut."""

    has_single: bool      # entries of one token run on the form for few rows
    has_portions: bool    # longer ones on the form for many
    splits: int           # CTAs that share the keys of a row tile of the former
    scratch: torch.Tensor | None
    arrivals: torch.Tensor | None


def _error(text):
    from .cuda_ops import KernelError

    return KernelError(text)


def quantised(keys, values) -> bool:
    """Whether a layer's cache is of 8-bit pages; both tensors of a layer have to be of one form."""
    forms = (isinstance(keys, QuantisedPages), isinstance(values, QuantisedPages))
    if forms[0] != forms[1]:
        raise _error("keys and values must both be 8-bit pages, or neither")
    return forms[0]


class QuantisedCacheOps:
    """Mixed into `CudaOps`."""

    Q8_SCRATCH_FLOATS = 64 << 20   # at most 256 MiB for the shares of split rows: fewer splits beyond that

    def _declare_q8_core(self, lib):
        lib.shrike_kv_write_q8.argtypes = [_P, _P, _LL, _LL, _P, _P, _P, _P, _P] + [_I] * 5 + [_LL, _P]
        lib.shrike_rope_kv_write_q8.argtypes = [_P] * 10 + [_I] * 6 + [_LL, _I, _LL, _P]
        lib.shrike_kv_read_q8.argtypes = [_P] * 7 + [_I] * 5 + [_LL, _P]
        for name in ("shrike_kv_write_q8", "shrike_rope_kv_write_q8", "shrike_kv_read_q8"):
            getattr(lib, name).restype = _I
        self._q8_libs = {}
        self._q8_scratch = self._q8_arrivals = None
        self.q8_splits = 0   # 0: the rule of `q8_plan`; n: that many splits for few rows (tests)

    def _q8_lib(self, head_dim: int):
        lib = self._q8_libs.get(head_dim)
        if lib is None:
            if head_dim % 16 or not 16 <= head_dim <= MOST_HEAD_DIM:
                raise _error(f"head size {head_dim} is not served: 8-bit pages take multiples of 16 from 16 to {MOST_HEAD_DIM}")
            lib = build.attention_q8_library(head_dim)
            lib.shrike_paged_attention_q8.argtypes = [_P] * 6 + [_I, _P, _P] + [_I] * 6 + [_F, _I, _P] + [_I] * 4 + [_P, _P, _P]
            lib.shrike_paged_attention_q8.restype = _I
            for name in ("share_floats", "max_splits"):
                getattr(lib, f"shrike_attention_q8_{name}").argtypes = []
                getattr(lib, f"shrike_attention_q8_{name}").restype = _I
            lib.shrike_attention_q8_resident_ctas.argtypes = [_I]
            lib.shrike_attention_q8_resident_ctas.restype = _I
            self._q8_libs[head_dim] = lib
        return lib

    # ---- checks
    def _q8_here(self, *tensors):
        """Every tensor on the GPU that this call launches on."""
        current = torch.cuda.current_device()
        for tensor in tensors:
            if tensor is not None and (tensor.device.type != "cuda" or tensor.device.index != current):
                raise _error(f"a tensor is on {tensor.device}, the current device is cuda:{current}")

    def _q8_pages(self, keys, values, num_kv_heads=None, head_dim=None):
        if keys.shape != values.shape:
            raise _error(f"key pages {list(keys.shape)} and value pages {list(values.shape)} differ")
        pages, page_size, heads, dim = keys.shape
        if (num_kv_heads is not None and heads != num_kv_heads) or (head_dim is not None and dim != head_dim):
            raise _error(f"key cache {tuple(keys.shape)} does not fit {num_kv_heads} heads of {head_dim}")
        if dim % 16 or not 16 <= dim <= MOST_HEAD_DIM:
            raise _error(f"head size {dim} is not served: 8-bit pages take multiples of 16 from 16 to {MOST_HEAD_DIM}")
        if pages * page_size > 0x7FFFFFFF:
            raise _error(f"{pages} pages of {page_size} tokens: slots are 32-bit numbers")
        self._q8_here(keys.codes, keys.scales, values.codes, values.scales)
        return pages, page_size, heads, dim

    @staticmethod
    def _q8_ints(tensor, count, what):
        if tensor.dtype != torch.int32 or not tensor.is_contiguous() or tensor.numel() != count:
            raise _error(f"{what} must be {count} contiguous int32, is {tensor.dtype} {list(tensor.shape)}")

    def _q8_rows(self, x, n, width, what):
        """The distance of x's rows in elements; a row's elements lie side by side."""
        if x.dtype != self.dtype or tuple(x.shape) != (n, width) or (width > 1 and x.stride(1) != 1) or (n > 1 and x.stride(0) < 0):
            raise _error(f"{what} must be {self.dtype} [{n}, {width}] with adjacent columns, is {x.dtype} {list(x.shape)}")
        return x.stride(0) if n > 1 else width

    # ---- the cache
    def _kv_write_q8(self, k_new, v_new, keys, values, slots):
        from .cuda_ops import _check, _ptr

        pages, page_size, heads, dim = self._q8_pages(keys, values)
        n = k_new.shape[0]
        strides = [self._q8_rows(x, n, heads * dim, what) for x, what in ((k_new, "new keys"), (v_new, "new values"))]
        self._q8_ints(slots, n, "slots")
        self._q8_here(k_new, v_new, slots)
        if n == 0:
            return
        self.launches += 1
        _check(self.core.shrike_kv_write_q8(
            _ptr(k_new), _ptr(v_new), *strides, _ptr(keys.codes), _ptr(keys.scales), _ptr(values.codes), _ptr(values.scales),
            _ptr(slots), self.code, n, heads, dim, page_size, pages * page_size, self._stream()), "kv_write_q8")

    def _rope_kv_write_q8(self, qkv, bias, positions, inv_freq, q_out, keys, values, slots, num_heads, num_kv_heads, head_dim):
        from .cuda_ops import _check, _dense, _ptr

        pages, page_size, _heads, _dim = self._q8_pages(keys, values, num_kv_heads, head_dim)
        _dense(q_out, self.dtype, "q")
        partials, stride = self._stack(qkv)
        n, width = qkv.shape[-2], (num_heads + 2 * num_kv_heads) * head_dim
        if qkv.dtype != torch.float32 or qkv.shape[-1] != width or qkv.stride(-1) != 1 or (n > 1 and qkv.stride(-2) != width):
            raise _error(f"qkv must be float32 rows of {width}, is {qkv.dtype} {list(qkv.shape)}")
        if q_out.numel() != n * num_heads * head_dim:
            raise _error(f"q {list(q_out.shape)} does not fit {n} tokens of {num_heads} heads of {head_dim}")
        if bias is not None:
            _dense(bias, torch.float32, "bias")
            if bias.numel() != width:
                raise _error(f"a bias of {bias.numel()} for rows of {width}")
        if inv_freq is not None:
            _dense(inv_freq, torch.float32, "inverse frequencies")
            if inv_freq.numel() != head_dim // 2:
                raise _error(f"{inv_freq.numel()} inverse frequencies for heads of {head_dim}")
        self._q8_ints(positions, n, "positions")
        self._q8_ints(slots, n, "slots")
        self._q8_here(qkv, bias, positions, inv_freq, q_out, slots)
        if n == 0:
            return
        self.launches += 1
        _check(self.core.shrike_rope_kv_write_q8(
            _ptr(qkv), _ptr(bias), _ptr(positions), _ptr(inv_freq), _ptr(q_out), _ptr(keys.codes), _ptr(keys.scales),
            _ptr(values.codes), _ptr(values.scales), _ptr(slots), self.code, n, num_heads, num_kv_heads, head_dim, page_size,
            pages * page_size, partials, stride, self._stream()), "rope_kv_write_q8")

    def kv_read(self, keys, values, slots, k_out, v_out):
        """Reads tokens back from 8-bit pages: row n of `k_out` and `v_out` ([N, kv heads * head size], contiguous, in the engine's
        type) is what `slots[n]` (int32 [N]) holds, codes times scale in 32 bits rounded once; zeros for a slot that is none of
        the pool's (a negative one, say).  A row stored from an infinity or a NaN comes back as NaN."""
        from .cuda_ops import _check, _dense, _ptr

        if not quantised(keys, values):
            raise _error("kv_read reads 8-bit pages; a cache in the engine's type is indexed as it is")
        pages, page_size, heads, dim = self._q8_pages(keys, values)
        n = slots.numel()
        self._q8_ints(slots, n, "slots")
        for x, what in ((k_out, "keys read"), (v_out, "values read")):
            _dense(x, self.dtype, what)
            if tuple(x.shape) != (n, heads * dim):
                raise _error(f"{what} must be [{n}, {heads * dim}], are {list(x.shape)}")
            if x.data_ptr() % 16:
                raise _error(f"{what} must begin on 16 bytes")
        self._q8_here(slots, k_out, v_out)
        if n == 0:
            return
        self.launches += 1
        _check(self.core.shrike_kv_read_q8(
            _ptr(keys.codes), _ptr(keys.scales), _ptr(values.codes), _ptr(values.scales), _ptr(slots), _ptr(k_out), _ptr(v_out),
            self.code, n, heads, dim, page_size, pages * page_size, self._stream()), "kv_read_q8")

    # ---- attention
    def q8_plan(self, num_heads, num_kv_heads, head_dim, num_seqs, max_blocks, page_size, max_q_len, min_q_len, window=0) -> QuantisedPlan:
        """How a batch over 8-bit pages is cut: a function of its shape alone, so that a captured launch sequence serves every
        batch of that shape."""
        lib = self._q8_lib(head_dim)
        has_single, has_portions = min_q_len <= 1, max_q_len > 1
        splits, scratch, arrivals = 1, None, None
        if has_single:
            tiles = -(-(num_heads // num_kv_heads) // 16)
            pairs = num_seqs * num_kv_heads * tiles
            keys = max_blocks * page_size
            if window > 0:
                keys = min(keys, window)
            elif window < 0:
                keys = min(keys, -window)
            splits = self.q8_splits or self.q8_few_row_splits(keys, pairs, lib.shrike_attention_q8_resident_ctas(self.code))
            share = lib.shrike_attention_q8_share_floats()
            splits = max(1, min(splits, lib.shrike_attention_q8_max_splits(), self.Q8_SCRATCH_FLOATS // (share * pairs)))
            if splits > 1:
                need = pairs * splits * share
                if self._q8_scratch is None or self._q8_scratch.numel() < need:
                    self._q8_scratch = torch.empty(max(need, 1 << 20), dtype=torch.float32, device=self.device)
                    self.generation += 1
                if self._q8_arrivals is None or self._q8_arrivals.numel() < pairs:
                    self._q8_arrivals = torch.zeros(max(pairs, 4096), dtype=torch.int32, device=self.device)
                    self.generation += 1
                scratch, arrivals = self._q8_scratch, self._q8_arrivals
        return QuantisedPlan(has_single, has_portions, splits, scratch, arrivals)

    @staticmethod
    def q8_few_row_splits(keys: int, pairs: int, resident: int) -> int:
        """CTAs that share the `keys` of each of `pairs` (entry, kv head, row tile) where the device holds `resident` at once: as
        many as fill it, each with at least two steps of 32 keys for its four warps."""
        return max(1, min(resident // pairs, keys // 256))

    def _paged_attention_q8(self, q, keys, values, block_table, q_start, ctx_len, seq_of_token, num_heads, num_kv_heads, head_dim,
                            scale, window, out, max_q_len, min_q_len):
        from .cuda_ops import _check, _dense, _ptr

        pages, page_size, _heads, _dim = self._q8_pages(keys, values, num_kv_heads, head_dim)
        _dense(q, self.dtype, "q")
        _dense(out, self.dtype, "attention output")
        _dense(block_table, torch.int32, "block table")
        n = q.shape[0]
        if num_kv_heads < 1 or num_heads % num_kv_heads:
            raise _error(f"{num_heads} heads do not share {num_kv_heads} kv heads evenly")
        if tuple(q.shape) != (n, num_heads * head_dim) or out.shape != q.shape:
            raise _error(f"q {list(q.shape)} and output {list(out.shape)} must be [tokens, {num_heads * head_dim}]")
        num_seqs, max_blocks = block_table.shape
        self._q8_ints(q_start, num_seqs + 1, "query starts")
        self._q8_ints(ctx_len, num_seqs, "context lengths")
        self._q8_here(q, out, block_table, q_start, ctx_len)
        if q.data_ptr() % 16 or out.data_ptr() % 16:
            raise _error("q and the attention output must begin on 16 bytes")
        if n == 0 or num_seqs == 0:
            return
        if max_q_len < 1:
            raise _error("paged_attention over 8-bit pages needs max_q_len, the longest entry of the batch")
        plan = self.q8_plan(num_heads, num_kv_heads, head_dim, num_seqs, max_blocks, page_size, max_q_len, min_q_len, window or 0)
        self.launches += plan.has_single + plan.has_portions
        _check(self._q8_lib(head_dim).shrike_paged_attention_q8(
            _ptr(q), _ptr(keys.codes), _ptr(keys.scales), _ptr(values.codes), _ptr(values.scales), _ptr(block_table), max_blocks,
            _ptr(q_start), _ptr(ctx_len), self.code, num_seqs, num_heads, num_kv_heads, page_size, pages, scale, window or 0,
            _ptr(out), int(plan.has_single), int(plan.has_portions), max_q_len, plan.splits, _ptr(plan.scratch),
            _ptr(plan.arrivals), self._stream()), "paged_attention_q8")
