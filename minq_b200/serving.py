"""The operators of one serving step over a paged 4-bit K/V cache, on CUDA
tensors (the C ABI's minq_pages_*, minq_kv4_* and minq_sample_rows):

    step = pages_extend(lens, new, table, free_pages, n_free, page_size, max_tokens)
    per layer: kv4_write(k, v, step.slots, k_pages, v_pages)
               kv4_attend(q, step.q_start, step.lens, table, k_pages, v_pages)
    sample_rows(logits, uniforms, temperature, top_k, top_p, min_p)

A pool is a uint8 tensor [n_pages, n_kv, page_size, head_dim / 32 * 20] of
Q4_0 blocks (`kv4_pool`). Every call runs on torch's current stream of the
tensors' device, without a host synchronisation, and may be captured into a
CUDA graph. Tensors of another dtype, device or layout are refused, never
converted.
"""
from __future__ import annotations

import functools
import math
from typing import NamedTuple

from . import _lib
from ._lib import MinqError, check, lib
from .minq_format import BLOCK_BYTES, BLOCK_SIZE, TAG_Q4_0

__all__ = ["PageStep", "PageTrim", "PAGES_SHORT", "PAGES_ROW_FULL", "PAGES_TOO_MANY_TOKENS",
           "PAGES_BAD_LENGTH", "PAGES_BAD_PAGE", "pages_extend", "pages_trim", "kv4_pool",
           "kv4_write", "kv4_read", "kv4_attend", "sample_rows"]

# info[0] of a pages call
PAGES_SHORT, PAGES_ROW_FULL, PAGES_TOO_MANY_TOKENS, PAGES_BAD_LENGTH, PAGES_BAD_PAGE = (
    1, 2, 4, 8, 16)

_Q4 = BLOCK_BYTES[TAG_Q4_0]


class PageStep(NamedTuple):
    """What pages_extend gives: lengths and free count after the step, the
    tokens' start per request, their slots and positions, and info (flags,
    missing pages)."""
    lens: object
    n_free: object
    q_start: object
    slots: object
    positions: object
    info: object


class PageTrim(NamedTuple):
    """What pages_trim gives: lengths and free count afterwards, and info."""
    lens: object
    n_free: object
    info: object


class _Bound:
    """torch and the library's functions, looked up once (importing this module
    loads neither)."""

    def __getattr__(self, name):  # the first use of a name
        import torch
        self.torch, self.i32, self.i64 = torch, torch.int32, torch.int64
        self.f32, self.u8 = torch.float32, torch.uint8
        self.stream, self.device = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice
        for fn in ("pages_extend", "pages_trim", "kv4_write", "kv4_read", "kv4_attend",
                   "sample_rows"):
            setattr(self, fn, getattr(lib(), "minq_" + fn))
        return self.__dict__[name]


_b = _Bound()


def _arg(msg: str) -> MinqError:
    return MinqError(_lib.ERR_ARG, msg)


def _shape(msg: str) -> MinqError:
    return MinqError(_lib.ERR_SHAPE, msg)


def _refuse(name, t, dtype, dev, shape):
    """Why a tensor argument is not taken."""
    if not getattr(t, "is_cuda", False):
        raise MinqError(_lib.ERR_CUDA, f"{name} must be a CUDA tensor (there is no CPU path)")
    if t.dtype is not dtype:
        raise _arg(f"{name} must be {dtype}, got {t.dtype}")
    if t.get_device() != dev:
        raise _arg(f"{name} is on {t.device}, expected cuda:{dev}")
    if shape is not None and t.shape != shape:
        raise _shape(f"{name} must have shape {list(shape)}, got {list(t.shape)}")
    raise _arg(f"{name} must be contiguous")


def _take(name, t, dtype, dev, shape=None):
    """Address of a contiguous tensor argument on CUDA device `dev`, checked."""
    if (t.dtype is not dtype or t.get_device() != dev or not t.is_contiguous()
            or (shape is not None and t.shape != shape)):
        _refuse(name, t, dtype, dev, shape)
    return t.data_ptr()


def _cuda(name, t) -> int:
    """Index of the CUDA device that a tensor is on."""
    if not getattr(t, "is_cuda", False):
        raise MinqError(_lib.ERR_CUDA, f"{name} must be a CUDA tensor (there is no CPU path)")
    return t.get_device()


def _run(dev: int, fn, *args) -> None:
    """Call a library function on the current stream of device `dev`, with that
    device current."""
    if _b.device() == dev:
        st = fn(*args, _b.stream(dev))
    else:
        with _b.torch.cuda.device(dev):
            st = fn(*args, _b.stream(dev))
    if st:
        check(st)


def _table(table, dev, n_req):
    if table.dim() != 2 or table.shape[0] != n_req:
        raise _shape(f"table must have shape [{n_req}, width], got {list(table.shape)}")
    return _take("table", table, _b.i32, dev)


def pages_extend(lens, new_tokens, table, free_pages, n_free, page_size: int, max_tokens: int,
                 out: PageStep | None = None) -> PageStep:
    """Grow every request by its new tokens: `table` [n_req, width] gets the
    new pages, taken from the top of `free_pages[:n_free]`; returns the step
    (slots and positions have max_tokens entries, the unused ones -1 and 0).
    All int32 except slots (int64). `out` reuses a step's tensors; its lens and
    n_free may be the inputs themselves. A step that does not fit (info) leaves
    everything as it was and has no tokens."""
    dev, i32 = _cuda("lens", lens), _b.i32
    n, one = lens.numel(), (lens.numel(),)
    lp = _take("lens", lens, i32, dev, one)
    ap = _take("new_tokens", new_tokens, i32, dev, one)
    tp = _table(table, dev, n)
    n_pages = free_pages.numel()
    fp = _take("free_pages", free_pages, i32, dev, (n_pages,))
    np_ = _take("n_free", n_free, i32, dev, (1,))
    if max_tokens < 0:
        raise _shape("max_tokens must not be negative")
    if out is None:
        # one allocation for the 32-bit outputs
        buf = lens.new_empty(2 * n + 4 + max_tokens)
        slots = lens.new_empty(max_tokens, dtype=_b.i64)
        lo, nf, qs, info, pos = buf.split_with_sizes((n, 1, n + 1, 2, max_tokens))
        out = PageStep(lo, nf, qs, slots, pos, info)
        b = buf.data_ptr()
        o = (b, b + 4 * n, b + 4 * n + 4, slots.data_ptr(), b + 8 * n + 16, b + 8 * n + 8)
    else:
        o = (_take("out.lens", out.lens, i32, dev, one),
             _take("out.n_free", out.n_free, i32, dev, (1,)),
             _take("out.q_start", out.q_start, i32, dev, (n + 1,)),
             _take("out.slots", out.slots, _b.i64, dev, (max_tokens,)),
             _take("out.positions", out.positions, i32, dev, (max_tokens,)),
             _take("out.info", out.info, i32, dev, (2,)))
    _run(dev, _b.pages_extend, lp, ap, n, page_size, tp, table.shape[1], fp, n_pages, np_,
         max_tokens, *o)
    return out


def pages_trim(lens, keep, table, free_pages, n_free, page_size: int,
               out: PageTrim | None = None) -> PageTrim:
    """Cut every request to at most keep[r] positions (0 ends it; a larger
    value keeps it whole) and put its pages back on `free_pages`."""
    dev, i32 = _cuda("lens", lens), _b.i32
    n, one = lens.numel(), (lens.numel(),)
    lp = _take("lens", lens, i32, dev, one)
    kp = _take("keep", keep, i32, dev, one)
    tp = _table(table, dev, n)
    n_pages = free_pages.numel()
    fp = _take("free_pages", free_pages, i32, dev, (n_pages,))
    np_ = _take("n_free", n_free, i32, dev, (1,))
    if out is None:
        buf = lens.new_empty(n + 3)
        out = PageTrim(*buf.split_with_sizes((n, 1, 2)))
        b = buf.data_ptr()
        o = (b, b + 4 * n, b + 4 * n + 4)
    else:
        o = (_take("out.lens", out.lens, i32, dev, one),
             _take("out.n_free", out.n_free, i32, dev, (1,)),
             _take("out.info", out.info, i32, dev, (2,)))
    _run(dev, _b.pages_trim, lp, kp, n, page_size, tp, table.shape[1], fp, n_pages, np_, *o)
    return out


def kv4_pool(n_pages: int, n_kv: int, page_size: int, head_dim: int, device="cuda"):
    """A zeroed pool of pages for the keys (or the values) of one layer."""
    if head_dim % BLOCK_SIZE:
        raise _shape(f"head_dim must be a multiple of {BLOCK_SIZE}, got {head_dim}")
    return _b.torch.zeros(n_pages, n_kv, page_size, head_dim // BLOCK_SIZE * _Q4, dtype=_b.u8,
                          device=device)


def _pools(k_pages, v_pages):
    """(n_pages, n_kv, page_size, head_dim, addresses) of a pair of pools."""
    dev = _cuda("k_pages", k_pages)
    if k_pages.dim() != 4 or k_pages.shape[3] % _Q4:
        raise _shape("a pool must have shape [n_pages, n_kv, page_size, head_dim / 32 * 20], got "
                     f"{list(k_pages.shape)}")
    kp = _take("k_pages", k_pages, _b.u8, dev)
    n, nkv, page, nb = shape = k_pages.shape
    vp = _take("v_pages", v_pages, _b.u8, dev, shape)
    return n, nkv, page, nb // _Q4 * BLOCK_SIZE, kp, vp, dev


def _rows(name, x, n_heads, hd, dev):
    """Address and token stride of [tokens, heads, head_dim] rows (the tokens
    may be strided, as slices of a projection are)."""
    if x.dtype is not _b.f32 or x.get_device() != dev:
        _refuse(name, x, _b.f32, dev, None)
    shape, st = x.shape, x.stride()
    if len(shape) != 3 or shape[1] != n_heads or shape[2] != hd:
        raise _shape(f"{name} must have shape [tokens, {n_heads}, {hd}], got {list(shape)}")
    if st[2] != 1 or (n_heads > 1 and st[1] != hd):
        raise _arg(f"{name}: a token's heads must be contiguous")
    return x.data_ptr(), st[0] if shape[0] > 1 else n_heads * hd


def kv4_write(k, v, slots, k_pages, v_pages) -> None:
    """Quantise k, v [tokens, n_kv, head_dim] into the pools at `slots` (int64;
    negative or outside the pool: skipped; the others distinct)."""
    n, nkv, page, hd, kp, vp, dev = _pools(k_pages, v_pages)
    a, sa = _rows("k", k, nkv, hd, dev)
    b, sb = _rows("v", v, nkv, hd, dev)
    T = k.shape[0]
    if v.shape[0] != T:
        raise _shape("k and v must hold the same tokens")
    s = _take("slots", slots, _b.i64, dev, (T,))
    _run(dev, _b.kv4_write, a, b, sa, sb, s, T, nkv, hd, kp, vp, n, page)


def kv4_read(slots, k_pages, v_pages, out=None):
    """(k, v) [tokens, n_kv, head_dim]: the values that the rows at `slots`
    stand for (zeros outside the pool)."""
    n, nkv, page, hd, kp, vp, dev = _pools(k_pages, v_pages)
    T = slots.numel()
    s = _take("slots", slots, _b.i64, dev, (T,))
    if out is None:
        out = slots.new_empty((2, T, nkv, hd), dtype=_b.f32).unbind(0)
        a, b, sa, sb = out[0].data_ptr(), out[1].data_ptr(), nkv * hd, nkv * hd
    else:
        a, sa = _rows("out[0]", out[0], nkv, hd, dev)
        b, sb = _rows("out[1]", out[1], nkv, hd, dev)
        if out[0].shape[0] != T or out[1].shape[0] != T:
            raise _shape(f"out must hold {T} tokens")
    _run(dev, _b.kv4_read, kp, vp, n, page, s, T, nkv, hd, a, b, sa, sb)
    return out


@functools.lru_cache(1024)
def _workspace(dev, n_req, n_tokens, n_heads, n_kv, hd) -> int:
    with _b.torch.cuda.device(dev):
        return lib().minq_kv4_attend_workspace_bytes(n_req, n_tokens, n_heads, n_kv, hd)


def kv4_attend(q, q_start, lens, table, k_pages, v_pages, scale: float | None = None, out=None,
               workspace=None):
    """Causal attention of the step's tokens q [tokens, n_heads, head_dim] over
    the pages of their requests; `lens` are the lengths with the step's tokens
    (PageStep.lens), whose rows are already written. Returns out [tokens,
    n_heads, head_dim]; rows behind q_start[-1] are left as they were (a fresh
    `out` holds nothing defined there). `scale`: 1 / sqrt(head_dim) unless given."""
    n, nkv, page, hd, kp, vp, dev = _pools(k_pages, v_pages)
    if q.dim() != 3:
        raise _shape(f"q must have shape [tokens, heads, {hd}], got {list(q.shape)}")
    T, nh = q.shape[0], q.shape[1]
    qp, qs = _rows("q", q, nh, hd, dev)
    R = lens.numel()
    lp = _take("lens", lens, _b.i32, dev, (R,))
    sp = _take("q_start", q_start, _b.i32, dev, (R + 1,))
    tp = _table(table, dev, R)
    if out is None:
        out = q.new_empty((T, nh, hd))
        op, os_ = out.data_ptr(), nh * hd
    else:
        op, os_ = _rows("out", out, nh, hd, dev)
        if out.shape[0] != T:
            raise _shape(f"out must hold {T} tokens")
    need = _workspace(dev, R, T, nh, nkv, hd)
    if workspace is None:
        workspace = q.new_empty(need, dtype=_b.u8)
    wp = _take("workspace", workspace, _b.u8, dev)
    _run(dev, _b.kv4_attend, qp, qs, sp, T, lp, R, tp, table.shape[1], kp, vp, n, page, nh, nkv,
         hd, 1.0 / math.sqrt(hd) if scale is None else scale, op, os_, wp, workspace.numel())
    return out


def sample_rows(logits, uniforms, temperature=None, top_k=None, top_p=None, min_p=None, out=None):
    """One token (int32) per row of logits [rows, n] from the row's uniform;
    temperature, top_p, min_p (f32) and top_k (int32) hold one value per row,
    None switches them off (see minq_sample_rows)."""
    dev = _cuda("logits", logits)
    if logits.dim() != 2:
        raise _shape(f"logits must have shape [rows, n], got {list(logits.shape)}")
    rows, n = logits.shape
    f32, i32, one = _b.f32, _b.i32, (rows,)
    stride, step = logits.stride()
    if logits.dtype is not f32:
        _refuse("logits", logits, f32, dev, None)
    if step != 1 and n > 1:
        raise _arg("logits: a row must be contiguous")
    if out is None:
        out = logits.new_empty(rows, dtype=i32)
        op = out.data_ptr()
    else:
        op = _take("out", out, i32, dev, one)
    _run(dev, _b.sample_rows, logits.data_ptr(), stride if rows > 1 else n, rows, n,
         None if temperature is None else _take("temperature", temperature, f32, dev, one),
         None if top_k is None else _take("top_k", top_k, i32, dev, one),
         None if top_p is None else _take("top_p", top_p, f32, dev, one),
         None if min_p is None else _take("min_p", min_p, f32, dev, one),
         _take("uniforms", uniforms, f32, dev, one), op)
    return out
