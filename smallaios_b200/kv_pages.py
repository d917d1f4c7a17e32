"""A pool of pages of the compressed KV cache, for sequences of different lengths.

Where ``GpuKvCache`` holds a batch of sequences with one position, ``GpuKvPages`` holds pages of 64 tokens, and
every call names the pages (``page_table``) and lengths (``seq_lens``) of its rows by device tensors.  Pages hold
the same codes, scales and zero points.  Who owns which page is the caller's business: the pool allocates none.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass

import torch

from . import _lib, ops
from ._lib import check, lib
from .kv_cache import DEFAULT_SEED, _view


@dataclass
class PagesView:
    """One layer's pages as torch tensors (zero-copy, strided: a page's arrays lie side by side)."""

    k_codes: torch.Tensor  # uint8 (P, H, 64, CB)
    v_codes: torch.Tensor  # uint8 (P, H, 4, CB/4, 4, 4, 4): 16-token blocks, see v_codes_tokens
    k_meta: torch.Tensor   # f32 (P, H, 64, 2) {scale, zero_point}
    v_meta: torch.Tensor   # f32 (P, H, 64, 2)
    signs: torch.Tensor    # f32 (H, D) +-1
    wht_scale: float
    bits: int
    code_bytes: int

    def v_codes_tokens(self) -> torch.Tensor:
        """V codes in per-token pack_bits order (P, H, 64, CB), as LayerView.v_codes_tokens."""
        p, h, nblk, c4, g, jj, tt = self.v_codes.shape
        return self.v_codes.permute(0, 1, 2, 4, 6, 3, 5).reshape(p, h, nblk * g * tt, c4 * jj)


class GpuKvPages:
    """Pages of every layer's K/V, quantized as ``GpuKvCache`` quantizes them, on one GPU.

    ``num_pages`` pages of 64 tokens per layer; page p of a row's table is page p in all layers.
    ``kv_head_begin/kv_head_count`` select a shard of the KV heads.  bits 4 or 8, head_dim 64 or 128.
    """

    def __init__(self, num_layers: int, num_kv_heads: int, head_dim: int, num_pages: int, *,
                 num_heads: int | None = None, bits: int = 4, seed: int = DEFAULT_SEED, kv_head_begin: int = 0,
                 kv_head_count: int | None = None, device=None):
        self._handle = ctypes.c_void_p()
        self.device = torch.device(device if device is not None else "cuda")
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        cfg = _lib.KvPagesConfig()
        cfg.num_layers = num_layers
        cfg.num_pages = num_pages
        cfg.num_heads = num_heads if num_heads is not None else num_kv_heads
        cfg.num_kv_heads = num_kv_heads
        cfg.kv_head_begin = kv_head_begin
        cfg.kv_head_count = kv_head_count if kv_head_count is not None else num_kv_heads - kv_head_begin
        cfg.head_dim = head_dim
        cfg.bits = bits
        cfg.seed = seed & (2**64 - 1)
        for name, n in (("num_layers", num_layers), ("num_pages", num_pages), ("num_heads", num_heads or 0),
                        ("num_kv_heads", num_kv_heads), ("kv_head_begin", kv_head_begin),
                        ("kv_head_count", kv_head_count or 0), ("head_dim", head_dim), ("bits", bits)):
            ops._fits("kv_pages_create", name, n)
        with torch.cuda.device(self.device):
            check(lib.sa_kv_pages_create(ctypes.byref(cfg), ctypes.byref(self._handle)))
        self.config = cfg
        self.kv_width = cfg.kv_head_count * head_dim
        self.half_dim = head_dim // 2
        self.query_width = cfg.num_heads // cfg.num_kv_heads * self.kv_width
        self._workspace_bytes: dict = {}

    @property
    def handle(self) -> int:
        if not self._handle:
            raise RuntimeError("GpuKvPages used after close()")
        return self._handle.value

    def append(self, layer: int, key: torch.Tensor, value: torch.Tensor, page_table: torch.Tensor,
               seq_lens: torch.Tensor, *, counts: torch.Tensor | None = None, cos_cache=None, sin_cache=None,
               do_rotary: bool = False, rotary_interleaved: bool = False, stream=None) -> None:
        """Quantize-on-append of (B, S, H*D) K/V, both of the same strides: token s of row b goes to position
        seq_lens[b] + s (sa_kv_pages_append).

        ``page_table`` int32 (B, pages), ``seq_lens`` int32 (B), on the device: the row's pages, and its tokens
        before these; a length below 0 leaves a row out.  ``counts`` int32 (B): only the first counts[b] of the S
        tokens exist.  K is rotated to its position with ``do_rotary``.  ``seq_lens`` is not changed.  Tokens that
        have no page, or no row in the tables, are left out and reported by ``device_status``.
        """
        index = self.device.index
        b, s, *strides = ops._token_rows("kv_pages_append", key, self.kv_width, index, "key")
        if not isinstance(value, torch.Tensor) or value.shape != key.shape:
            raise ops.ShapeMismatch("kv_pages_append: key and value must be (B, S, H*D) with equal shapes")
        if value.dtype != key.dtype:
            raise ops.UnsupportedOp("kv_pages_append: key and value dtypes differ")
        if ops._token_rows("kv_pages_append", value, self.kv_width, index, "value") != (b, s, *strides):
            raise ValueError("key and value must have the same strides")
        table = ops._page_rows("kv_pages_append", page_table, seq_lens, counts, b, index)
        rope = ops._page_rope("kv_pages_append", cos_cache, sin_cache, self.half_dim, index)
        rc = lib.sa_kv_pages_append(self.handle, ops._fits("kv_pages_append", "layer_idx", layer), key.data_ptr(),
                                    value.data_ptr(), *strides, ops._dtype_code(key), b, s, *table, *rope,
                                    int(bool(do_rotary)), int(bool(rotary_interleaved)), ops._stream_handle(stream, self.device))
        ops._raise_op(rc, "kv_pages_append")

    def reorder_beams(self, page_table: torch.Tensor, seq_lens: torch.Tensor, parents: torch.Tensor, *,
                      out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
        """The beams' new page table, and copies of the pages that several of them go on filling, in every layer
        (sa_kv_pages_reorder).

        ``parents`` int32 (B, K): beam i of group b (row b*K + i) goes on as beam parents[b, i] was; -1: it stays.
        ``page_table`` int32 (B*K, pages), ``seq_lens`` int32 (B*K), equal within a group.  Full pages may be shared
        by rows; a row's page in use and the pages behind it must be its own.  ``out`` must share no element
        with ``page_table``.
        """
        index = self.device.index
        ops._on(parents, index, "parents")
        if not parents.is_contiguous():
            raise ValueError("parents must be contiguous")
        shape = parents.shape
        if len(shape) != 2:
            raise ops.ShapeMismatch("reorder_beams: parents must be (B, K)")
        if parents.dtype != torch.int32:
            raise ops.UnsupportedOp("reorder_beams: parents must be int32")
        b, k = shape
        if b >= 2**31 or not 1 <= k <= _lib.SA_MAX_BEAMS:
            raise ops.InvalidAttribute(f"reorder_beams: {b} groups of {k} beams (1..{_lib.SA_MAX_BEAMS})")
        table, stride, width, lens, _ = ops._page_rows("reorder_beams", page_table, seq_lens, None, b * k, index)
        if out is None:
            out = ops._empty(page_table.shape, torch.int32, page_table.device, stream)
            new, new_stride = out.data_ptr(), width
        else:
            if not isinstance(out, torch.Tensor) or out.shape != page_table.shape:
                raise ops.ShapeMismatch("reorder_beams: out must have page_table's shape")
            new, new_stride, _ = ops._page_table("reorder_beams", out, b * k, index, "out")
        rc = lib.sa_kv_pages_reorder(self.handle, table, stride, new, new_stride, width, lens, parents.data_ptr(), b, k,
                                     ops._stream_handle(stream, self.device))
        ops._raise_op(rc, "reorder_beams")
        return out

    def set_precision(self, full: bool) -> None:
        """Bits of queries and weights in ``gqa_paged_attend`` for f16 and bf16 callers (sa_kv_pages_set_precision): 24
        with ``full``, as f32 callers and the decode path over ``GpuKvCache`` have; else 16, the default."""
        check(lib.sa_kv_pages_set_precision(self.handle, int(bool(full))))
        self._workspace_bytes.clear()

    def workspace_bytes(self, batch: int, seq_len: int, dtype_code: int) -> int:
        """sa_gqa_paged_workspace_bytes, which a pool's configuration and precision fix."""
        key = (batch, seq_len, dtype_code)
        n = self._workspace_bytes.get(key)
        if n is None:
            n = self._workspace_bytes[key] = lib.sa_gqa_paged_workspace_bytes(self.handle, batch, seq_len, dtype_code)
        return n

    def view(self, layer: int) -> PagesView:
        """The layer's arrays.  The tensors keep the pool alive; ``close()`` ends them all the same."""
        v = _lib.KvPagesView()
        check(lib.sa_kv_pages_layer_view(self.handle, ops._fits("kv_pages_layer_view", "layer_idx", layer), ctypes.byref(v)))
        p, h, cb, d = v.num_pages, v.kv_heads, v.code_bytes, v.head_dim
        raw = _view(v.records, (p, h, v.record_bytes), "|u1", self)

        def piece(offset, end):
            return raw[:, :, offset:end]

        return PagesView(k_codes=piece(0, v.k_meta_offset).unflatten(-1, (64, cb)),
                         v_codes=piece(v.v_codes_offset, v.record_bytes).unflatten(-1, (4, cb // 4, 4, 4, 4)),
                         k_meta=piece(v.k_meta_offset, v.v_meta_offset).view(torch.float32).unflatten(-1, (64, 2)),
                         v_meta=piece(v.v_meta_offset, v.v_codes_offset).view(torch.float32).unflatten(-1, (64, 2)),
                         signs=_view(v.signs, (h, d), "<f4", self), wht_scale=v.wht_scale, bits=v.bits, code_bytes=cb)

    def device_status(self, clear: bool = False) -> int:
        """Bits of what kernels on this pool met (sa_kv_pages_device_status): 1 a bounded wait gave up, 2 a page
        outside the pool or the table, 4 a position outside the cos/sin tables, 8 beams that do not match.
        Synchronises."""
        st = ctypes.c_int32()
        check(lib.sa_kv_pages_device_status(self.handle, ctypes.byref(st), int(bool(clear))))
        return st.value

    def close(self) -> None:
        if self._handle:
            with torch.cuda.device(self.device):
                lib.sa_kv_pages_destroy(self._handle.value)
            self._handle = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
