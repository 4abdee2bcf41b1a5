"""Cache pages in 8 bits: codes with one scale per token and kv head.

A head's row x of a token is kept as codes c = round(127 x / a), a = max |x|, and the float32 scale a / 127; it is read as
c * scale (`csrc/cache_q8.cu` writes and reads them, `csrc/attention_q8*.cu` attends over them).  A `QuantisedPages` stands
wherever the kernels take a layer's keys or values: `rope_kv_write`, `kv_write`, `kv_read` and `paged_attention`.
Azimml/shrike's pool has one form, the model's dtype (shrike/engine/model_runner.py:52-60).
"""

from __future__ import annotations

import torch

MOST_HEAD_DIM = 256   # of the kernels over 8-bit pages
_INT8, _FLOAT32 = torch.int8, torch.float32
look_pages = None   # the same questions as `_look_here`, natively, once the kernels are loaded (`ops/quantised_cache.py`)


def _look_here(codes, scales):
    """The codes' sizes; None: not a pool's codes and scales."""
    dims = codes.shape
    if not (len(dims) == 4 and codes.dtype is _INT8 and scales.dtype is _FLOAT32 and scales.shape == (dims[0], dims[2], dims[1])
            and codes.is_contiguous() and scales.is_contiguous() and codes.device == scales.device):
        return None
    return tuple(dims)


class QuantisedPages:
    """`codes` int8 [pages, page_size, kv heads, head size], `scales` float32 [pages, kv heads, page_size], on one device."""

    __slots__ = ("codes", "scales", "dims")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor):
        dims = (look_pages or _look_here)(codes, scales)
        if dims is None:
            self._refuse(codes, scales)
        self.codes, self.scales, self.dims = codes, scales, dims   # (pages, page_size, kv heads, head size)

    @staticmethod
    def _refuse(codes, scales):
        if codes.dtype != torch.int8 or codes.dim() != 4 or not codes.is_contiguous():
            raise ValueError("codes must be a contiguous int8 [pages, page_size, kv heads, head size]")
        pages, page_size, heads, _dim = codes.shape
        if scales.dtype != torch.float32 or tuple(scales.shape) != (pages, heads, page_size) or not scales.is_contiguous():
            raise ValueError(f"scales must be a contiguous float32 [{pages}, {heads}, {page_size}], are "
                             f"{scales.dtype} {list(scales.shape)}")
        raise ValueError(f"codes are on {codes.device}, scales on {scales.device}")

    @classmethod
    def zeros(cls, pages: int, page_size: int, kv_heads: int, head_dim: int, device) -> "QuantisedPages":
        return cls(torch.zeros(pages, page_size, kv_heads, head_dim, dtype=torch.int8, device=device),
                   torch.zeros(pages, kv_heads, page_size, dtype=torch.float32, device=device))

    @property
    def shape(self) -> torch.Size:
        """That of the codes: [pages, page_size, kv heads, head size], as a pool in the engine's type has it."""
        return self.codes.shape

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def bytes(self) -> int:
        return self.codes.numel() + 4 * self.scales.numel()
