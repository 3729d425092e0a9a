"""A paged K/V cache in 8 bits for batches of sequences of different lengths, and the operators on it.

``PagedKV`` holds the pages of all layers; page tables (device int32 [sequences, entries]) hand them out.  A decode step
is ``append`` (rotate the new keys and queries, round K / V to 8 bits into their pages) and ``attend`` per layer; both also
take many new tokens per sequence (prompts, chunks, drafted tokens).  ``read`` brings rows back to the dense tensors of
``ops.attn_decode`` / ``ops.attn_prefill``; ``reorder`` follows a beam search's choice (``ops.beam_select``).

Batches of new tokens are packed: ``q_start`` (device int32 [B + 1]) names the rows [q_start[b], q_start[b + 1]) of
sequence b; None: one row per sequence.  Everything is ordered on the current stream of the tensors' device and can be
captured into a graph (outputs then are the caller's, or live in the graph's pool).  Lengths, positions and tables are
read on the device, so a captured step follows what they hold at replay.  Device values that make no sense (a page id
outside the cache, lengths past the table) are not errors: see include/vault_amd.h for what each operator does with them.
"""
from __future__ import annotations

import ctypes as C
import functools
from typing import Optional, Tuple

import torch

from . import _lib as L
from .ops import KV_DTYPES, TICKETS, Workspace, _on, _ptr, _stream

I8, E4M3 = L.I8, L.E4M3
PAGES = (16, 32, 64, 128, 256)


class PagedKV:
    """Pages of 8-bit K / V codes with one scale per (layer, page, kv head).

    k: uint8 [layers, pages, G, page, D]; v: uint8 [layers, pages, G, D, page] (tokens contiguous); k_scale / v_scale:
    fp32 [layers, pages, G], not negative.  ``fmt``: I8 (value = (byte - 128) * scale) or E4M3 (float8_e4m3fn * scale).
    D 64 or 128, page 16 .. 256 (a power of two).  Layers may lie apart; all else must be contiguous."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor, fmt: int):
        if fmt not in (I8, E4M3):
            raise ValueError("fmt must be I8 or E4M3")
        if k.dim() != 5:
            raise ValueError("k must be [layers, pages, G, page, D]")
        n, pages, G, P, D = k.shape
        if min(k.shape) < 1 or D not in (64, 128) or P not in PAGES:
            raise ValueError(f"head dim 64 or 128 and pages of {PAGES} tokens, got {D} and {P}")
        if v.shape != (n, pages, G, D, P):
            raise ValueError("v must be [layers, pages, G, D, page]")
        if k_scale.shape != (n, pages, G) or v_scale.shape != k_scale.shape:
            raise ValueError("scales must be [layers, pages, G]")
        for t, dt, name in ((k, torch.uint8, "k"), (v, torch.uint8, "v"), (k_scale, torch.float32, "k_scale"),
                            (v_scale, torch.float32, "v_scale")):
            if not t.is_cuda:
                raise ValueError(f"{name} must be a device tensor")
            if t.dtype != dt:
                raise ValueError(f"{name} must be {dt}, got {t.dtype}")
            if t.device != k.device:
                raise ValueError("the cache must be on one device")
            if not t[0].is_contiguous():
                raise ValueError(f"{name}: a layer must be contiguous")
        if n > 1 and (v.stride(0) != k.stride(0) or v_scale.stride(0) != k_scale.stride(0)):
            raise ValueError("k and v, and their scales, need equal layer strides")
        self.k, self.v, self.k_scale, self.v_scale, self.fmt = k, v, k_scale, v_scale, fmt
        self.n_layers, self.n_pages, self.G, self.page, self.D = n, pages, G, P, D
        self.device = k.device
        self._c = L.PagedKV(fmt, k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), n, pages, G, P, D,
                            k.stride(0) if n > 1 else pages * G * P * D, k_scale.stride(0) if n > 1 else pages * G)
        self.ref = C.addressof(self._c)
        self.index = k.get_device()
        self.lib = L.load()

    @classmethod
    def empty(cls, n_layers: int, n_pages: int, G: int, D: int, device, page: int = 64, fmt: int = I8) -> "PagedKV":
        """Pages of zeros."""
        shape = (n_layers, n_pages, G)
        zero = 128 if fmt == I8 else 0
        full = lambda *tail: torch.full((*shape, *tail), zero, dtype=torch.uint8, device=device)  # noqa: E731
        return cls(full(page, D), full(D, page), torch.zeros(shape, device=device), torch.zeros(shape, device=device),
                   fmt)


# A decode step makes these calls per layer and token, so the checks below are as cheap as Python allows: devices are
# compared by index, and the launch context, the stream and the workspace's size cost no more than a dictionary look-up.

def _words(t: torch.Tensor, n: int, kv: PagedKV, name: str) -> None:
    if t.dtype is not torch.int32 or t.get_device() != kv.index:
        raise ValueError(f"{name} must be an int32 tensor on the cache's device")
    if t.dim() != 1 or t.shape[0] != n:
        raise ValueError(f"{name} must be [{n}], got {tuple(t.shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _table(t: torch.Tensor, kv: PagedKV, name: str = "table") -> Tuple[int, int, int]:
    """(sequences, entries, row stride)."""
    if t.dtype is not torch.int32 or t.get_device() != kv.index or t.dim() != 2:
        raise ValueError(f"{name} must be int32 [sequences, entries] on the cache's device")
    B, n = t.shape
    if n < 1:
        raise ValueError(f"{name} must have entries")
    if t.is_contiguous():
        return B, n, n
    ld = t.stride(0) if B > 1 else n
    if t.stride(1) != 1 or ld < n:
        raise ValueError(f"{name} rows must be contiguous and apart")
    return B, n, ld


def _stride(t: torch.Tensor, N: int, H: int, D: int) -> int:
    """The row stride of t [N, H, D] if its heads are contiguous and its rows 16-byte aligned, else 0."""
    if t.data_ptr() % 16:
        return 0
    if t.is_contiguous():
        return H * D
    st = t.stride()
    if st[2] != 1 or (H > 1 and st[1] != D):
        return 0
    if N == 1:
        return H * D
    return st[0] if st[0] * t.element_size() % 16 == 0 and st[0] >= H * D else 0


def _rows(t: torch.Tensor, heads: int, dtype, kv: PagedKV, name: str) -> Tuple[torch.Tensor, int, int, int]:
    """t [N, heads, D] (any number of heads where ``heads`` is 0) with contiguous heads and 16-byte aligned rows, a copy
    where the view is not; its row stride, N and heads."""
    shape = t.shape
    if len(shape) != 3 or shape[2] != kv.D or shape[1] < 1 or (heads and shape[1] != heads):
        raise ValueError(f"{name} must be [N, {heads or 'H'}, {kv.D}], got {tuple(shape)}")
    if t.dtype is not dtype or t.get_device() != kv.index:
        raise ValueError(f"{name} must be {dtype} on the cache's device")
    N, H, D = shape
    ld = _stride(t, N, H, D)
    if not ld:
        t, ld = t.clone(memory_format=torch.contiguous_format), H * D
    return t, ld, N, H


def _dest(t: torch.Tensor, N: int, H: int, dtype, kv: PagedKV, name: str) -> int:
    """The row stride of an output that rows are written into, in place."""
    if t.shape != (N, H, kv.D) or t.dtype is not dtype or t.get_device() != kv.index:
        raise ValueError(f"{name} must be {(N, H, kv.D)} {dtype} on the cache's device")
    ld = _stride(t, N, H, kv.D)
    if not ld:
        raise ValueError(f"{name} needs contiguous heads and 16-byte aligned rows")
    return ld


def _batch(q_start: Optional[torch.Tensor], B: int, N: int, kv: PagedKV) -> None:
    if q_start is None:
        if N != B:
            raise ValueError(f"without q_start every sequence has one row: {N} rows for {B} sequences")
    else:
        _words(q_start, B + 1, kv, "q_start")


def _layer(kv: PagedKV, layer: int) -> None:
    if not 0 <= layer < kv.n_layers:
        raise ValueError(f"layer {layer} of {kv.n_layers}")


@functools.lru_cache(maxsize=1024)
def _attn_bytes(*sizes: int) -> int:
    need = int(L.load().vgx_paged_attn_workspace_bytes(*sizes))
    L.check(min(need, 0), "vgx_paged_attn_workspace_bytes")
    return need


def append(kv: PagedKV, layer: int, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, start: torch.Tensor, *,
           rope: Optional[torch.Tensor] = None, q: Optional[torch.Tensor] = None, q_out: Optional[torch.Tensor] = None,
           q_start: Optional[torch.Tensor] = None, max_new: Optional[int] = None) -> Optional[torch.Tensor]:
    """New tokens into the pages of ``layer`` (vgx_paged_append).

    k, v [N, G, D] fp32 or bf16; sequence b's rows take the positions start[b], start[b] + 1, ... (start int32 [B]: the
    tokens that it holds already).  ``rope`` fp32 [positions, D], rows [cos | sin]: keys are rotated by their position's
    row.  With q [N, H, D] (dtype of k) the queries are rotated too, into ``q_out`` (may be q; a new tensor by default),
    which is returned.  A sequence's pages must be in its table row; a page that is written must be in one entry only.
    ``max_new`` is not needed and only accepted for symmetry with ``attend``."""
    D = kv.D
    _layer(kv, layer)
    B, cols, ldt = _table(table, kv)
    dt = KV_DTYPES.get(k.dtype)
    if dt is None:
        raise ValueError("k must be fp32 or bf16")
    dtype = k.dtype
    k, ldk, N, _ = _rows(k, kv.G, dtype, kv, "k")
    v, ldv, n, _ = _rows(v, kv.G, dtype, kv, "v")
    if n != N:
        raise ValueError("k and v must have the same rows")
    _batch(q_start, B, N, kv)
    _words(start, B, kv, "start")
    rope_ld = rope_rows = H = ldq = ldqo = 0
    if rope is not None:
        if rope.dtype is not torch.float32 or rope.get_device() != kv.index or rope.dim() != 2 or rope.shape[1] != D:
            raise ValueError("rope must be fp32 [positions, D] on the cache's device")
        rope_ld, rope_rows = rope.stride(0), rope.shape[0]
        if rope.stride(1) != 1 or rope_ld % 4 or rope_ld < D or rope.data_ptr() % 16:
            raise ValueError("rope rows must be contiguous, apart and 16-byte aligned")
    src = None
    if q is not None:
        src, ldq, n, H = _rows(q, 0, dtype, kv, "q")
        if n != N:
            raise ValueError("q must have the rows of k")
        if q_out is None:
            q_out, ldqo = torch.empty(N, H, D, dtype=dtype, device=kv.device), H * D
        else:
            ldqo = _dest(q_out, N, H, dtype, kv, "q_out")
    elif q_out is not None:
        raise ValueError("q_out without q")
    with _on(kv.device):
        rc = kv.lib.vgx_paged_append(kv.ref, layer, dt, k.data_ptr(), ldk, v.data_ptr(), ldv, N, table.data_ptr(), ldt,
                                     cols, start.data_ptr(), _ptr(q_start), B, _ptr(rope), rope_ld, rope_rows, _ptr(src), ldq,
                                     _ptr(q_out), ldqo, H, _stream(kv.device))
    if rc:
        L.check(rc, "vgx_paged_append")
    return q_out


def attend(kv: PagedKV, layer: int, q: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, *,
           q_start: Optional[torch.Tensor] = None, max_new: Optional[int] = None, max_keys: Optional[int] = None,
           window: int = 0, n_sink: int = 0, scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
           ws: Optional[Workspace] = None) -> torch.Tensor:
    """Attention over the pages of ``layer`` (vgx_paged_attn).

    q [N, H, D] fp32 or bf16, rotated; lens int32 [B]: tokens that sequence b holds, its queries being its last ones (so
    after an append, lens = start + new tokens).  Every query sees the keys up to its own position, with ``window`` > 0
    only the last ``window`` of them and the first ``n_sink`` tokens.  Returns [N, H, D] in q's dtype; a query that sees
    nothing gets zeros, rows behind the last sequence stay as they were.  ``out`` may be q.  ``max_new`` / ``max_keys``: the most rows and
    keys of one sequence, hints for the split of the work (by default what the shapes allow).  ``ws``: a Workspace of this
    stream; without it scratch is allocated."""
    D = kv.D
    _layer(kv, layer)
    B, cols, ldt = _table(table, kv)
    dt = KV_DTYPES.get(q.dtype)
    if dt is None:
        raise ValueError("q must be fp32 or bf16")
    dtype = q.dtype
    q, ldq, N, H = _rows(q, 0, dtype, kv, "q")
    if H % kv.G:
        raise ValueError(f"{H} query heads for {kv.G} kv heads")
    _batch(q_start, B, N, kv)
    _words(lens, B, kv, "lens")
    if window < 0 or n_sink < 0:
        raise ValueError("window and n_sink must not be negative")
    if out is None:
        out, ldo = torch.empty(N, H, D, dtype=dtype, device=kv.device), H * D
    else:
        ldo = _dest(out, N, H, dtype, kv, "out")
    most = 1 if q_start is None else N if max_new is None else max_new
    keys = cols * kv.page
    keys = keys if max_keys is None else min(max_keys, keys)
    if most < 0 or keys < 0:
        raise ValueError("max_new and max_keys must not be negative")
    need = _attn_bytes(N, B, H, kv.G, D, most, keys, window, n_sink)
    buf = None
    if need > 0:
        buf = ws.get(need) if ws is not None else torch.empty(need, dtype=torch.uint8, device=kv.device)
        if buf.get_device() != kv.index:
            raise ValueError("the workspace must be on the cache's device")
        need = buf.numel()
    marks = ws.tickets() if buf is not None and ws is not None else None
    with _on(kv.device):
        rc = kv.lib.vgx_paged_attn_tickets(kv.ref, layer, dt, q.data_ptr(), ldq, out.data_ptr(), ldo, N, H,
                                           table.data_ptr(), ldt, cols, lens.data_ptr(), _ptr(q_start), B, most, keys, window,
                                           n_sink, D ** -0.5 if scale is None else scale, _ptr(buf), need, _ptr(marks),
                                           0 if marks is None else TICKETS, _stream(kv.device))
    if rc:
        L.check(rc, "vgx_paged_attn_tickets")
    return out


def read(kv: PagedKV, table: torch.Tensor, first: torch.Tensor, n: int, lens: torch.Tensor,
         dtype: torch.dtype = torch.float32) -> Tuple[torch.Tensor, torch.Tensor]:
    """Dequantized rows of all layers (vgx_paged_read): (k, v), each [layers, B, G, n, D] fp32 or bf16, row i of sequence
    b being position first[b] + i; zeros at positions below 0 or at or past lens[b], and where the table has no page.
    Keys come back rotated as they were stored."""
    B, cols, ldt = _table(table, kv)
    _words(first, B, kv, "first")
    _words(lens, B, kv, "lens")
    dt = KV_DTYPES.get(dtype)
    if dt is None:
        raise ValueError("dtype must be fp32 or bf16")
    if n < 0:
        raise ValueError("n must not be negative")
    k = torch.empty(kv.n_layers, B, kv.G, n, kv.D, dtype=dtype, device=kv.device)
    v = torch.empty_like(k)
    with _on(kv.device):
        rc = kv.lib.vgx_paged_read(kv.ref, dt, table.data_ptr(), ldt, cols, first.data_ptr(), lens.data_ptr(), B, n,
                                   k.data_ptr(), v.data_ptr(), _stream(kv.device))
    if rc:
        L.check(rc, "vgx_paged_read")
    return k, v


def reorder(kv: PagedKV, table: torch.Tensor, lens: torch.Tensor, parents: torch.Tensor, table_out: torch.Tensor,
            lens_out: torch.Tensor) -> None:
    """After a beam search's choice: beam i of group b continues beam parents[b, i] (vgx_paged_reorder).

    table [B * K, entries] and lens [B * K] are the beams' before, table_out / lens_out (other tensors) after.  Full pages
    become shared; the page that the next token goes to is owned by one beam before and after (give every beam its own
    before the call): the first child takes its parent's over, further children get copies in the pages of beams that
    nothing continues.  Entries past that page stay the row's own.  A page stays in use until no table names it."""
    if parents.dim() != 2 or parents.dtype is not torch.int32 or parents.get_device() != kv.index or \
            not parents.is_contiguous():
        raise ValueError("parents must be contiguous int32 [groups, K] on the cache's device")
    B, K = parents.shape
    n, cols, ldt = _table(table, kv)
    _, cols_out, ldo = _table(table_out, kv, "table_out")
    if n != B * K or table_out.shape[0] != n or cols_out != cols:
        raise ValueError("table and table_out must have a row per beam")
    _words(lens, n, kv, "lens")
    _words(lens_out, n, kv, "lens_out")
    if table_out.data_ptr() == table.data_ptr() or lens_out.data_ptr() == lens.data_ptr():
        raise ValueError("table_out and lens_out must be other tensors than table and lens")
    with _on(kv.device):
        rc = kv.lib.vgx_paged_reorder(kv.ref, table.data_ptr(), ldt, cols, lens.data_ptr(), parents.data_ptr(), B, K,
                                      table_out.data_ptr(), ldo, lens_out.data_ptr(), _stream(kv.device))
    if rc:
        L.check(rc, "vgx_paged_reorder")
