"""The paged cache in 8 bits: the part of :class:`~fastgen_b200.csrc.ops.Ops` that writes it and reads it.

Pages hold e4m3 codes, keys as ``[pages, kv heads, page, size]``, values as ``[pages, kv heads, page / 4, size, 4]``, with
one power of two for each page and head (float32 ``[pages, kv heads]``); an entry stands for its code times that.
"""

from __future__ import annotations

import threading
from ctypes import c_float, c_int, c_void_p
from typing import Optional

import torch

from . import build

_P, _I, _F = c_void_p, c_int, c_float
_BF16, _F32, _E4M3 = torch.bfloat16, torch.float32, torch.float8_e4m3fn
_KV8_PAGES = (16, 32, 64, 128, 256)  # tokens a page

SIGNATURES = {
    "fg_kv8_write": [_P, _I, _P, _P, _I, _P, _I, _P, _P, _P, _P, _P, _P, _P, _P, _P, _I, _I, _I, _I, _I, _I, _I, _P,
                     _P, _P, _P, _I, _F, _I, _P],
    "fg_kv8_values": [_P, _P, _P, _P, _P, _I, _P, _P, _I, _I, _I, _I, _P, _P],
    "fg_kv8_expand": [_P, _P, _P, _P, _P, _I, _P, _P, _P, _I, _P, _P, _I, _I, _I, _I, _I, _P, _P],
    "fg_kv8_attention_decode": [_P, _I, _P, _I, _P, _P, _I, _P, _P, _P, _I, _I, _I, _P, _P, _P, _I, _I, _I, _I, _I, _F, _F, _P,
                                _I, _P, _I, _P, _P, _P, _P],
    "fg_kv8_decode_scratch_floats": [],
}
_libraries = {}
_capturing = torch.cuda.is_current_stream_capturing


def kv8(head_dim: int):
    """The library of the paged cache in 8 bits for this head size."""
    lib = _libraries.get(head_dim)
    if lib is None:
        lib = build.kv8_library(head_dim)
        _ops._declare(lib, SIGNATURES)
        _libraries[head_dim] = lib
    return lib


class _PromptsOnly:
    """A step's context without its single tokens."""

    def __init__(self, ctx) -> None:
        self._ctx = ctx

    def __getattr__(self, name):
        return getattr(self._ctx, name)

    def single_tokens(self):
        return _NO_SINGLES


class _NoSingles:
    n = 0


_NO_SINGLES = _NoSingles()


class Kv8Ops:
    """See the module; mixed into :class:`~fastgen_b200.csrc.ops.Ops`."""

    def _init_kv8(self) -> None:
        # ((pages, kv heads, page, head size), stream) -> pages in bfloat16 of caches in 8 bits that have none of their own; the
        # stream of captured calls is None (see kv8_expanded)
        self._expanded = {}
        self._expanding = threading.Lock()  # from the filling of such a pool to the launch that reads it
        # (head size, stream) -> partials and counters of the single-token attention over a cache in 8 bits; the stream of
        # captured calls is None
        self._kv8_buffers = {}
        self._growing = threading.Lock()
        self._kv8_retired = []

    def _clear_kv8(self) -> None:
        for counters in [*self._kv8_retired, *(count for _scratch, count in self._kv8_buffers.values())]:
            counters.zero_()

    @staticmethod
    def kv8_supported(head_dim: int, page_size: int) -> Optional[str]:
        """``None``, or why a cache of these sizes cannot be held in 8 bits."""
        if head_dim not in build.KV8_HEAD_DIMS:
            return f"head size {head_dim} is not one of {build.KV8_HEAD_DIMS}"
        if page_size not in _KV8_PAGES:
            return f"pages of {page_size} tokens are not a power of two from 16 to 256"
        return None

    def _check_kv8(self, memory, n_kv_heads: int, head_dim: int) -> None:
        """Raise unless ``memory`` is a cache in 8 bits of these sizes."""
        k, v, ks, vs, page = memory.k_pages, memory.v_pages, memory.k_scales, memory.v_scales, memory.page_size
        n_pages = k.shape[0]
        shape, scales = (n_pages, n_kv_heads, page, head_dim), (n_pages, n_kv_heads)
        if (k.shape == shape and v.shape == (n_pages, n_kv_heads, page // 4, head_dim, 4) and ks.shape == scales == vs.shape
                and k.dtype is v.dtype is _E4M3 and ks.dtype is vs.dtype is _F32 and k.is_contiguous() and v.is_contiguous()
                and ks.is_contiguous() and vs.is_contiguous() and head_dim in build.KV8_HEAD_DIMS and page in _KV8_PAGES
                and self.act_dtype is _BF16 and k.device == v.device == ks.device == vs.device == memory.block_table.device
                and k.is_cuda):
            return
        why = self.kv8_supported(head_dim, page)
        if why is not None:
            raise ValueError(f"a cache in 8 bits: {why}")
        if self.act_dtype != torch.bfloat16:
            raise ValueError("a cache in 8 bits serves bfloat16 models")
        for t, dtype in ((k, _E4M3), (v, _E4M3), (ks, _F32), (vs, _F32)):
            if t.dtype != dtype or not t.is_contiguous():
                raise ValueError(f"a cache in 8 bits: contiguous {dtype} wanted, got {t.dtype} {tuple(t.shape)}")
        if not all(t.is_cuda and t.device == k.device for t in (k, v, ks, vs, memory.block_table)):
            raise ValueError("a cache in 8 bits: its pages, scales and block table are on one GPU")
        raise ValueError(f"a cache in 8 bits of {n_kv_heads} heads of {head_dim}: keys {shape}, values "
                         f"{(n_pages, n_kv_heads, page // 4, head_dim, 4)} and scales {scales} wanted, got {tuple(k.shape)}, "
                         f"{tuple(v.shape)}, {tuple(ks.shape)} and {tuple(vs.shape)}")

    def make_kv8_tensor_maps(self, k_pool, v_pool):
        """Tensor maps of the pools of a cache in 8 bits: codes ``[layers, pages, kv heads, page, head size]`` of keys and
        ``[layers, pages, kv heads, page / 4, head size, 4]`` of values."""
        n_layers, n_pages, n_kv_heads, page, head_dim = k_pool.shape
        why = self.kv8_supported(head_dim, page)
        if why is not None:
            raise ValueError(f"a cache in 8 bits: {why}")
        assert v_pool.shape == (n_layers, n_pages, n_kv_heads, page // 4, head_dim, 4)
        maps = []
        for pool in (k_pool, v_pool):
            assert pool.dtype == torch.float8_e4m3fn and pool.is_contiguous()
            tm = _ops.TensorMap()
            _ops._check(self.lib, self.lib.fg_make_kv8_tensor_map(
                tm.ptr, _ops._ptr(pool), n_layers, n_pages, n_kv_heads, page, head_dim, min(page, _ops.DECODE_SPLIT)))
            _ops.Ops.launches -= 1  # not a kernel
            maps.append(tm)
        return tuple(maps)

    def rope_kv8_write(self, q, k, v, pos, req, freqs, memory, n_heads: int, n_kv_heads: int, head_dim: int,
                       v_freqs=None, qk_norm=None, magnitude: float = 1.0, rot_pairs: int = 0) -> torch.Tensor:
        """:meth:`rope_kv_write` for a cache in 8 bits: returns the rotated queries [T, heads * head size] and writes
        rotated keys and values to their pages as e4m3 codes with one power of two a (page, head), the smallest ``2^e``
        (``e >= -100``) at which every magnitude is at most ``448 * 2^e``.  Tokens that begin a page choose it; tokens
        behind cached ones never lower it, and where they raise it the cached codes are rounded again.  A sequence's
        tokens are neighbours in the step and in ascending order.  Entries that are not finite are stored as NaN.
        Queries, keys and values are bfloat16; the rotated numbers are rounded once, to the
        codes nearest to their values in 64 bits (of the float32 angle position * frequency)."""
        self._check_kv8(memory, n_kv_heads, head_dim)
        t = q.shape[0]
        kv_shape = (t, n_kv_heads * head_dim)
        if not (q.shape == (t, n_heads * head_dim) and k.shape == kv_shape == v.shape and q.dtype is k.dtype is v.dtype is _BF16
                and q.stride(1) == k.stride(1) == v.stride(1) == 1 and n_heads % n_kv_heads == 0
                and q.device == k.device == v.device == memory.k_pages.device):
            raise ValueError(f"rope_kv8_write takes bfloat16 rows of {n_heads} and twice {n_kv_heads} heads of {head_dim}, got "
                             f"{q.dtype} {tuple(q.shape)}, {k.dtype} {tuple(k.shape)} and {v.dtype} {tuple(v.shape)} on {q.device}")
        table = memory.block_table
        assert pos.dtype is req.dtype is table.dtype is torch.int32 and pos.numel() == req.numel() == t and table.is_contiguous()
        assert freqs is None or (freqs.dtype is _F32 and freqs.numel() == head_dim // 2 and freqs.is_contiguous())
        assert v_freqs is None or (v_freqs.dtype is _F32 and v_freqs.numel() == head_dim // 2 and v_freqs.is_contiguous())
        rstd = qn_w = kn_w = None
        rstd_heads = 0
        if qk_norm is not None:
            rstd, qn_w, kn_w = qk_norm
            assert rstd.dtype == torch.float32 and rstd.is_contiguous() and rstd.shape[0] == t
            rstd_heads = 0 if rstd.shape[1] == 2 else rstd.shape[1]
            assert rstd_heads in (0, n_heads + n_kv_heads)
            assert qn_w is None or (qn_w.dtype == torch.float32 and qn_w.numel() == n_heads * head_dim and qn_w.is_contiguous())
            assert kn_w is None or (kn_w.dtype == torch.float32 and kn_w.numel() == n_kv_heads * head_dim and kn_w.is_contiguous())
        out = torch.empty((t, n_heads * head_dim), dtype=_BF16, device=q.device)
        lib = kv8(head_dim)
        _ops._check(lib, lib.fg_kv8_write(
            q.data_ptr(), q.stride(0), out.data_ptr(), k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0), pos.data_ptr(),
            req.data_ptr(), _ops._ptr(freqs), _ops._ptr(v_freqs), memory.k_pages.data_ptr(), memory.v_pages.data_ptr(),
            memory.k_scales.data_ptr(), memory.v_scales.data_ptr(), table.data_ptr(), table.shape[1], memory.page_size,
            memory.k_pages.shape[0], t, n_heads, n_kv_heads, head_dim, self.status.data_ptr(), _ops._ptr(rstd), _ops._ptr(qn_w), _ops._ptr(kn_w), rstd_heads, float(magnitude), int(rot_pairs), _ops._stream()))
        return out

    def kv8_values(self, memory, pages):
        """What the pages ``pages`` (int32, on the device) of a cache in 8 bits stand for: keys and values in bfloat16
        ``[n, kv heads, page, head size]``, every slot of the pages, also those that hold no token."""
        n_pages, n_kv_heads, page, head_dim = memory.k_pages.shape
        self._check_kv8(memory, n_kv_heads, head_dim)
        assert pages.dtype is torch.int32 and pages.is_contiguous() and pages.device == memory.k_pages.device
        n = pages.numel()
        k = torch.empty((n, n_kv_heads, page, head_dim), dtype=_BF16, device=pages.device)
        v = torch.empty_like(k)
        lib = kv8(head_dim)
        _ops._check(lib, lib.fg_kv8_values(
            memory.k_pages.data_ptr(), memory.v_pages.data_ptr(), memory.k_scales.data_ptr(), memory.v_scales.data_ptr(),
            pages.data_ptr(), n, k.data_ptr(), v.data_ptr(), page, n_pages, n_kv_heads, head_dim, self.status.data_ptr(), _ops._stream()))
        return k, v

    def make_kv8_expanded(self, shape):
        """Pages in bfloat16 for a cache in 8 bits of ``shape`` (pages, kv heads, page, head size): keys, values and their
        tensor maps.  Prompt portions read such pages; all layers of a shape fill the same ones in turn."""
        k = torch.zeros(shape, dtype=torch.bfloat16, device=self.device)
        v = torch.zeros_like(k)
        return k, v, self.make_kv_tensor_maps(k[None], v[None], shape[2])

    def kv8_expanded(self, memory, stream: Optional[int] = None):
        """What :meth:`make_kv8_expanded` made for ``memory``'s cache: the pool in ``memory.expanded``, as an engine's memories
        have it, which belongs to the cache's one stream.  For a memory without one, a pool for each shape and stream, made at the
        first call (not inside a graph capture; captured calls take the first stream's) and kept as long as this object."""
        shape = tuple(memory.k_pages.shape)
        if memory.expanded is not None:
            if tuple(memory.expanded[0].shape) != shape or memory.expanded[0].device != memory.k_pages.device:
                raise ValueError(f"a cache in 8 bits of {shape} on {memory.k_pages.device} comes with the expanded pages of "
                                 f"{tuple(memory.expanded[0].shape)} on {memory.expanded[0].device}")
            return memory.expanded
        if _capturing():
            got = self._expanded.get((shape, None))
            if got is None:
                raise RuntimeError("the first prompt portion over a cache in 8 bits cannot be inside a graph capture")
            return got
        key = shape, _ops._stream() if stream is None else stream
        got = self._expanded.get(key)
        if got is None:
            got = self._expanded[key] = self.make_kv8_expanded(shape)
            self._expanded.setdefault((shape, None), got)
        return got

    def _kv8_work(self, lib, head_dim: int, counters: int, stream: int):
        """Scratch and zeroed counters of the single-token attention over a cache in 8 bits: of the stream, or of all
        captured graphs, which are replayed one after the other.  They grow outside graph captures only; the graphs' ones that were
        outgrown stay alive, since graphs hold their addresses."""
        if _capturing():
            got = self._kv8_buffers.get((head_dim, None))
            if got is None or got[1].numel() < counters:
                raise RuntimeError("the first single-token attention of a size over a cache in 8 bits cannot be inside a graph capture")
            return got
        got = self._kv8_buffers.get((head_dim, stream))
        if got is None or got[1].numel() < counters:
            n = max(1024, 1 << (counters - 1).bit_length())
            with self._growing:
                for key in ((head_dim, stream), (head_dim, None)):
                    old = self._kv8_buffers.get(key)
                    if old is not None and old[1].numel() >= n:
                        continue
                    scratch = old[0] if old is not None else torch.empty(lib.fg_kv8_decode_scratch_floats(), dtype=torch.float32,
                                                                         device=self.device)
                    if old is not None:
                        self._kv8_retired.append(old[1])
                    self._kv8_buffers[key] = (scratch, torch.zeros(n, dtype=torch.int32, device=self.device))
                torch.cuda.current_stream(self.device).synchronize()  # graphs are replayed on any stream
                got = self._kv8_buffers[head_dim, stream]
        return got

    def _attention_kv8(self, q, out, memory, ctx, n_heads, n_kv_heads, head_dim, window, scale, out_freqs, keep_first,
                       softcap, sinks, chunk) -> bool:
        self._check_kv8(memory, n_kv_heads, head_dim)
        assert q.dtype is out.dtype is _BF16 and q.stride(1) == 1 == out.stride(1) and q.device == out.device == memory.k_pages.device
        assert q.shape == out.shape and q.shape[1] == n_heads * head_dim and not (window and chunk)
        assert sinks is None or (sinks.dtype is _F32 and sinks.numel() == n_heads and sinks.is_contiguous())
        if window and keep_first:
            raise ValueError("a cache in 8 bits knows no window that keeps first positions")
        table = memory.block_table
        lib = kv8(head_dim)
        signed_window = -int(chunk) if chunk else int(window or 0)
        n_pages, page = memory.k_pages.shape[0], memory.page_size
        singles, stream = ctx.single_tokens(), _ops._stream()
        longest = getattr(ctx, "longest", None)
        prompts = longest != 1 and ctx.attention_tiles(_ops.attention_tiling(n_heads, n_kv_heads, _ops.PREFILL_TMA_ROWS), 2).n > 0
        if prompts:
            with self._expanding:
                k, v, maps = self.kv8_expanded(memory, stream)
                _ops._check(lib, lib.fg_kv8_expand(
                    _ops._ptr(memory.k_pages), _ops._ptr(memory.v_pages), _ops._ptr(memory.k_scales), _ops._ptr(memory.v_scales), _ops._ptr(table),
                    table.shape[1], _ops._ptr(ctx.seq_slot), _ops._ptr(ctx.seq_start), _ops._ptr(ctx.seq_cached), ctx.n_seqs, _ops._ptr(k), _ops._ptr(v), page,
                    n_pages, n_kv_heads, head_dim, signed_window, _ops._ptr(self.status), stream))
                expanded = type(memory)(k_pages=k, v_pages=v, block_table=table, page_size=page, tensor_maps=maps)
                self.attention(q, out, expanded, _PromptsOnly(ctx), n_heads, n_kv_heads, head_dim, window, scale,
                               softcap=softcap, sinks=sinks, chunk=chunk)
        fused = out_freqs is not None and not prompts and singles.n > 0
        if singles.n:
            # a counter for every sequence and slice of up to eight heads of a group
            slices = n_kv_heads * -(-n_heads // n_kv_heads // 8)
            scratch, counters = self._kv8_work(lib, head_dim, singles.n * slices, stream)
            maps = memory.tensor_maps
            _ops._check(lib, lib.fg_kv8_attention_decode(
                q.data_ptr(), q.stride(0), out.data_ptr(), out.stride(0), maps[0].ptr, maps[1].ptr, memory.layer_index,
                memory.k_scales.data_ptr(), memory.v_scales.data_ptr(), table.data_ptr(), table.shape[1], page, n_pages,
                ctx.pos.data_ptr(), singles.req.data_ptr(), singles.tok.data_ptr(), singles.n, n_heads, n_kv_heads, head_dim,
                signed_window, float(scale), float(softcap or 0.0), scratch.data_ptr(), scratch.numel(), counters.data_ptr(),
                counters.numel(), _ops._ptr(out_freqs) if fused else None, _ops._ptr(sinks), self.status.data_ptr(), stream))
        return fused


# (last, since that module takes its part from this one)
from . import ops as _ops  # noqa: E402
