"""A paged KV cache for requests that come and go (see ``csrc/ixb_paged.cuh``, ``csrc/ixb_attn_paged.cuh``): thin wrappers
over the C ABI.

The reference's batched generator keeps one static cache row per sequence (ixrun/batching.py:88-234).  Here the cache is a
pool of pages, [pages, page, kv heads, head_dim] each for keys and values, and a request holds as many as its tokens need.
A step of a batch is: ``page_step`` (where every new token goes), then per layer ``rope_kv_paged`` and ``AttnPaged``.
Every call is launches on the current stream that can be captured in a CUDA graph: lengths, tables and positions are device
tensors, and nothing is allocated when the outputs are passed in.
"""
from __future__ import annotations

from collections import namedtuple

import torch

from . import _lib
from ._lib import host as _host
from .glue import _bf16, _rows_view

__all__ = ["PageStep", "page_step", "page_release", "PageTables", "rope_kv_paged", "AttnPaged"]

PAGES = (16, 32, 64, 128, 256)
MAX_REQUESTS = 4096


class PageStep(namedtuple("PageStep", "cu_rows length n_free slot pos owner status")):
    """What ``page_step`` says about a step of R requests in a batch of `rows` rows (int32 device tensors): cu_rows [R + 1]
    first row of every request; length [R] tokens with the new ones; n_free [1] pages left; slot, pos, owner [rows] the
    pool row, position and request of every batch row (-1, 0, -1 behind the last token); status [2]: 0 or why the step does
    not fit (1 pages, 2 rows, 4 table), and the pages that it needs."""

    __slots__ = ()

    @classmethod
    def empty(cls, requests: int, rows: int, device, length=None, n_free=None):
        """Tensors for a step; length and n_free: existing ones to be updated in place."""
        device = torch.device(device)
        if device.type != "cuda":
            raise ValueError("expected a CUDA device")
        index = torch.cuda.current_device() if device.index is None else device.index
        cu_rows, new_length, new_n_free, slot, pos, owner, status = _host().empty(
            index, (requests + 1, "i"), (0 if length is not None else requests, "i"), (0 if n_free is not None else 1, "i"), (rows, "i"), (rows, "i"),
            (rows, "i"), (2, "i"))
        return cls(cu_rows, new_length if length is None else length, new_n_free if n_free is None else n_free, slot, pos, owner, status)


def _ints(device, **tensors):
    """contiguous int32 tensors on one CUDA device"""
    for name, t in tensors.items():
        if t.dtype != torch.int32 or not t.is_cuda or not t.is_contiguous():
            raise ValueError(f"{name}: a contiguous int32 CUDA tensor expected")
        if t.get_device() != device:
            raise ValueError(f"{name} is on another device")


def _page(page: int):
    if page not in PAGES:
        raise ValueError(f"a page holds {', '.join(map(str, PAGES))} positions, not {page}")


def page_step(q_len, length, table, free, n_free, page: int, rows: int, out: PageStep | None = None) -> PageStep:
    """Places for q_len [R] new tokens behind the length [R] that every request has: pages from the top of the stack free [pages]
    (its first n_free entries) into table [R, width], in the order of requests and positions.  rows: rows of the batch that
    the new tokens are packed into, at least as many as there are (a captured step has a fixed number).  out: tensors to
    write (``PageStep.empty``); out.length may be length and out.n_free n_free (updated in place).  All int32.
    A step that does not fit (out.status[0] != 0) takes no page and is empty: cu_rows is zero."""
    if out is not None and _host().page_step(q_len, length, table, free, n_free, page, rows, *out):
        return out
    _page(page)
    dev, r = q_len.get_device(), q_len.numel()
    _ints(dev, q_len=q_len, length=length, table=table, free=free, n_free=n_free)
    if r < 1 or r > MAX_REQUESTS or length.numel() != r or table.dim() != 2 or table.shape[0] != r or n_free.numel() != 1 or free.numel() < 1 or table.shape[1] < 1:
        raise ValueError(f"q_len and length [R], table [R, width], free [pages], n_free [1] with R of 1..{MAX_REQUESTS}")
    rows = int(rows)
    if rows < 0:
        raise ValueError("rows must not be negative")
    if out is None:
        out = PageStep.empty(r, rows, q_len.device)
    else:
        _ints(dev, **out._asdict())
        if out.cu_rows.numel() != r + 1 or out.length.numel() != r or out.n_free.numel() != 1 or out.status.numel() != 2 or any(
                t.numel() != rows for t in (out.slot, out.pos, out.owner)):
            raise ValueError("out does not have the sizes of this step")
    with _lib.on_device(dev) as st:
        _lib.check(_lib.lib().ixb_page_step(q_len.data_ptr(), length.data_ptr(), table.data_ptr(), free.data_ptr(), n_free.data_ptr(), r,
                                            table.shape[1], free.numel(), page, rows, out.cu_rows.data_ptr(), out.length.data_ptr(),
                                            out.n_free.data_ptr(), out.slot.data_ptr(), out.pos.data_ptr(), out.owner.data_ptr(),
                                            out.status.data_ptr(), st))
    return out


def page_release(done, length, table, free, n_free, page: int, status=None):
    """The pages of the requests with done [R] (bool or uint8) go back onto the stack, their lengths become 0 (in place).
    Returns status int32 [2]: 0, or 4 if the stack cannot take them (nothing is done then), and their number."""
    _page(page)
    dev, r = length.get_device(), length.numel()
    _ints(dev, length=length, table=table, free=free, n_free=n_free)
    if done.dtype not in (torch.bool, torch.uint8) or done.get_device() != dev or not done.is_contiguous() or done.numel() != r:
        raise ValueError("done: a contiguous bool or uint8 tensor [R] on the device of length")
    if r < 1 or r > MAX_REQUESTS or table.dim() != 2 or table.shape[0] != r or n_free.numel() != 1 or free.numel() < 1 or table.shape[1] < 1:
        raise ValueError(f"length [R], table [R, width], free [pages], n_free [1] with R of 1..{MAX_REQUESTS}")
    if status is None:
        status = torch.empty(2, dtype=torch.int32, device=length.device)
    _ints(dev, status=status)
    if status.numel() != 2:
        raise ValueError("status is [2]")
    with _lib.on_device(dev) as st:
        _lib.check(_lib.lib().ixb_page_release(done.data_ptr(), length.data_ptr(), table.data_ptr(), free.data_ptr(), n_free.data_ptr(), r,
                                               table.shape[1], free.numel(), page, status.data_ptr(), st))
    return status


class PageTables:
    """Block tables of up to `requests` requests over a pool of n_pages pages of `page` positions each, with the stack of free
    pages; a request has at most width * page tokens."""

    def __init__(self, requests: int, n_pages: int, page: int, width: int, device):
        _page(page)
        if not 1 <= requests <= MAX_REQUESTS or n_pages < 1 or width < 1 or n_pages * page > 2**31 - 1:
            raise ValueError(f"1..{MAX_REQUESTS} requests, and pages that hold less than 2^31 positions")
        self.requests, self.n_pages, self.page, self.width = int(requests), int(n_pages), int(page), int(width)
        self.table = torch.full((requests, width), -1, dtype=torch.int32, device=device)
        self.free = torch.arange(n_pages - 1, -1, -1, dtype=torch.int32, device=device)        # page 0 on top
        self.n_free = torch.full((1,), n_pages, dtype=torch.int32, device=device)
        self.length = torch.zeros(requests, dtype=torch.int32, device=device)
        if self.table.is_cuda and not torch.cuda.is_current_stream_capturing():
            torch.cuda.current_stream(self.table.device).synchronize()         # complete for a first call on any stream

    def new_step(self, rows: int) -> PageStep:
        """Tensors for steps of `rows` rows that update this table's lengths and stack."""
        return PageStep.empty(self.requests, rows, self.table.device, length=self.length, n_free=self.n_free)

    def step(self, q_len, rows: int, out: PageStep | None = None) -> PageStep:
        """``page_step`` on this table, in place."""
        return page_step(q_len, self.length, self.table, self.free, self.n_free, self.page, rows, out=out or self.new_step(rows))

    def release(self, done, status=None):
        """``page_release`` on this table."""
        return page_release(done, self.length, self.table, self.free, self.n_free, self.page, status=status)


def _pool(t, hkv: int, head_dim: int, what: str):
    """(pages, page, page pitch) of a pool [pages, page, hkv, head_dim] whose pages are contiguous and may lie apart"""
    if t.dtype != torch.bfloat16 or not t.is_cuda or t.dim() != 4 or t.shape[2:] != (hkv, head_dim) or t.shape[0] < 1:
        raise ValueError(f"{what}: a bf16 CUDA tensor [pages, page, hkv, head_dim] expected")
    _page(t.shape[1])
    if not t[0].is_contiguous():
        raise ValueError(f"{what}: every page must be contiguous")
    pitch = t.stride(0) if t.shape[0] > 1 else t[0].numel()
    if pitch < t[0].numel() or pitch % 8:
        raise ValueError(f"{what}: pages must not overlap and must lie a multiple of 8 elements apart")
    return t.shape[0], t.shape[1], pitch


def rope_kv_paged(q, k, v, pos, slot, k_pages, v_pages, cos, sin, hq: int, hkv: int, head_dim: int, rot_dim: int | None = None, q_norm=None,
                  k_norm=None, eps: float = 1e-6, out=None):
    """``glue.rope_kv`` for a paged cache: q [rows, >= hq*head_dim] rotated (in place, or into out [rows, hq*head_dim]); k, v [rows,
    hkv*head_dim] into the pools at slot [rows]; pos, slot: int32 [rows] as ``page_step`` gives them.  Column slices are allowed.  A
    row whose slot is outside the pools is left alone; a position outside the tables is rotated as the nearest one in them.  Between the
    norm and the result nothing is rounded."""
    if _host().rope_paged(q, k, v, pos, slot, k_pages, v_pages, cos, sin, hq, hkv, head_dim, rot_dim or head_dim, q_norm, k_norm, eps, q if out is None else out):
        return q if out is None else out
    _bf16(q_norm, k_norm)
    rows, qcols, q_pitch = _rows_view(q, "q")
    _, kcols, kv_pitch = _rows_view(k, "k")
    if _rows_view(v, "v") != (rows, kcols, kv_pitch) or _rows_view(k, "k")[0] != rows or kcols != hkv * head_dim or qcols < hq * head_dim:
        raise ValueError("q is [rows, >= hq*head_dim], k and v are [rows, hkv*head_dim] with the same row pitch")
    n_pages, page, k_pitch = _pool(k_pages, hkv, head_dim, "k_pages")
    if _pool(v_pages, hkv, head_dim, "v_pages")[:2] != (n_pages, page):
        raise ValueError("k_pages and v_pages must have the same shape")
    dev = q.get_device()
    _ints(dev, pos=pos, slot=slot)
    if pos.numel() < rows or slot.numel() < rows:
        raise ValueError("a position and a slot for every row")
    rot = rot_dim or head_dim
    for t in (cos, sin):
        if t.dtype != torch.float32 or not t.is_cuda or not t.is_contiguous() or t.dim() != 2 or t.shape[1] != rot // 2 or t.shape != cos.shape or not t.shape[0]:
            raise ValueError("cos and sin: contiguous fp32 CUDA tensors [max_seq, rot_dim / 2]")
    for t in (q_norm, k_norm):
        if t is not None and t.numel() != head_dim:
            raise ValueError("norm weights are [head_dim]")
    o, o_pitch = q, q_pitch
    if out is not None:
        if _rows_view(out, "out")[:2] != (rows, hq * head_dim):
            raise ValueError("out is [rows, hq*head_dim]")
        o, o_pitch = out, _rows_view(out, "out")[2]
    for t in (k, v, k_pages, v_pages, cos, sin, q_norm, k_norm, o):
        if t is not None and t.get_device() != dev:
            raise ValueError("all tensors must be on one device")
    if rows == 0:
        return o
    with _lib.on_device(dev) as st:
        _lib.check(_lib.lib().ixb_rope_paged(q.data_ptr(), k.data_ptr(), v.data_ptr(), pos.data_ptr(), slot.data_ptr(), k_pages.data_ptr(),
                                             v_pages.data_ptr(), None if q_norm is None else q_norm.data_ptr(),
                                             None if k_norm is None else k_norm.data_ptr(), cos.data_ptr(), sin.data_ptr(), o.data_ptr(), rows, hq,
                                             hkv, head_dim, rot, float(eps), q_pitch, kv_pitch, o_pitch, cos.shape[0], n_pages, page, k_pitch,
                                             _pool(v_pages, hkv, head_dim, "v_pages")[2], st))
    return o


class AttnPaged:
    """Causal grouped-query attention of the new tokens of a batch of requests over their pages; one token, a few or a chunk of a
    prompt per request, mixed as they come.  Owns the scratch of pairs that are cut over several CTAs: launches that may overlap
    (different streams without ordering) need separate objects."""

    def __init__(self, hq: int, hkv: int, head_dim: int, device):
        if hkv < 1 or hq < 1 or hq % hkv:
            raise ValueError("query heads must be a multiple of the KV heads")
        if head_dim not in (64, 128, 256):
            raise ValueError("head_dim must be 64, 128 or 256")
        self.hq, self.hkv, self.d = int(hq), int(hkv), int(head_dim)
        device = torch.device(device)
        if device.type != "cuda":
            raise ValueError("expected a CUDA device")
        if device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        with _lib.on_device(device.index):
            self.scratch = torch.zeros(_lib.lib().ixb_attn_paged_scratch_bytes(self.d), dtype=torch.uint8, device=device)
        if not torch.cuda.is_current_stream_capturing():
            torch.cuda.current_stream(device).synchronize()                    # zero for a first call on any stream

    def __call__(self, q, k_pages, v_pages, table, length, cu_rows, max_q: int | None = None, out=None, scale: float | None = None):
        """q [rows, >= hq*head_dim] (column slices allowed): rows cu_rows[r] .. cu_rows[r+1] - 1 are the newest tokens of request r, which
        has length[r] tokens (these among them) on the pages table [R, width] of the pools [pages, page, hkv, head_dim]; length [R],
        cu_rows [R+1], table: int32.  Every row attends to the positions up to its own, of those that the table has an entry for.
        max_q: the most new tokens that a request has (1 for a step of single tokens), by which the kernels are chosen.  Returns
        out [rows, hq*head_dim]; rows of no request are left as they are (undefined without `out`), rows that see no position are
        zero.

        Scores and sums are held in 32 bits.  Probabilities are multiplied with the values in 17 bits where a request has few rows (new
        tokens times query heads of a KV head: up to 16, up to 8 with heads of 256) or max_q says so of all, in 8 bits (bf16) where it
        has more (one request alone: by max_q): a token of a longer draft agrees with the same token alone to bf16 noise, not to the bit.  A row's last bits also depend
        on the other requests of the call, whose lengths say where the work is cut; the same call gives the same bits."""
        done = _host().attn_paged(self.hq, self.hkv, self.d, self.scratch, q, k_pages, v_pages, table, length, cu_rows, max_q, out, scale)
        if done is not None:
            return done
        rows, cols, pitch = _rows_view(q, "q")
        n_pages, page, k_pitch = _pool(k_pages, self.hkv, self.d, "k_pages")
        vn, vp, v_pitch = _pool(v_pages, self.hkv, self.d, "v_pages")
        dev, r = q.get_device(), length.numel()
        _ints(dev, table=table, length=length, cu_rows=cu_rows)
        if (vn, vp) != (n_pages, page) or cols < self.hq * self.d:
            raise ValueError("q is [rows, >= hq*head_dim], the pools have one shape")
        if r < 1 or r > MAX_REQUESTS or cu_rows.numel() != r + 1 or table.dim() != 2 or table.shape[0] != r or table.shape[1] < 1:
            raise ValueError(f"length [R], cu_rows [R+1], table [R, width] with R of 1..{MAX_REQUESTS}")
        if max_q is not None and max_q < 1:
            raise ValueError("max_q must be positive")
        if scale is not None and not 0.0 < scale < float("inf"):
            raise ValueError("scale must be positive")
        if out is None:
            out = torch.empty(rows, self.hq * self.d, dtype=torch.bfloat16, device=q.device)
        elif out.numel() != rows * self.hq * self.d:
            raise ValueError("out must be [rows, hq*head_dim]")
        _bf16(out)
        for t in (k_pages, v_pages, out, self.scratch):
            if t.get_device() != dev:
                raise ValueError("all tensors and this object must be on one device")
        if rows == 0:
            return out
        with _lib.on_device(dev) as st:
            _lib.check(_lib.lib().ixb_attn_paged(q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), table.data_ptr(), length.data_ptr(),
                                                 cu_rows.data_ptr(), out.data_ptr(), r, table.shape[1], rows, min(rows, max_q or rows), self.hq,
                                                 self.hkv, self.d, n_pages, page, pitch, k_pitch, v_pitch,
                                                 float(scale if scale is not None else self.d ** -0.5), self.scratch.data_ptr(),
                                                 self.scratch.numel(), st))
        return out
