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


@functools.cache
def _torch():
    import torch
    return torch


@functools.cache
def _call(name):
    """The library's function of that name."""
    return getattr(lib(), name)


def _arg(msg: str) -> MinqError:
    return MinqError(_lib.ERR_ARG, msg)


def _shape(msg: str) -> MinqError:
    return MinqError(_lib.ERR_SHAPE, msg)


def _take(name, t, dtype, dev, shape=None, contiguous=True):
    """Check a tensor argument on CUDA device `dev`; returns its address."""
    if t.dtype is not dtype:
        raise _arg(f"{name} must be {dtype}, got {t.dtype}")
    if t.get_device() != dev:
        raise _arg(f"{name} is on {t.device}, expected cuda:{dev}")
    if shape is not None and t.shape != shape:
        raise _shape(f"{name} must have shape {list(shape)}, got {list(t.shape)}")
    if contiguous and not t.is_contiguous():
        raise _arg(f"{name} must be contiguous")
    return t.data_ptr()


def _cuda(name, t) -> int:
    """Index of the CUDA device that a tensor is on."""
    if not getattr(t, "is_cuda", False):
        raise MinqError(_lib.ERR_CUDA, f"{name} must be a CUDA tensor (there is no CPU path)")
    return t.get_device()


@functools.cache
def _on(dev: int):
    return _torch().device("cuda", dev)


def _run(dev: int, name: str, *args) -> None:
    """Call the library on the current stream of device `dev`, with that device
    current."""
    cuda = _torch()._C
    stream = cuda._cuda_getCurrentRawStream(dev)
    if cuda._cuda_getDevice() == dev:
        check(_call(name)(*args, stream))
    else:
        with _torch().cuda.device(dev):
            check(_call(name)(*args, stream))


def _table(table, dev, n_req):
    torch = _torch()
    if table.dim() != 2 or table.shape[0] != n_req:
        raise _shape(f"table must have shape [{n_req}, width], got {list(table.shape)}")
    return _take("table", table, torch.int32, dev)


def pages_extend(lens, new_tokens, table, free_pages, n_free, page_size: int, max_tokens: int,
                 out: PageStep | None = None) -> PageStep:
    """Grow every request by its new tokens: `table` [n_req, width] gets the
    new pages, taken from the top of `free_pages[:n_free]`; returns the step
    (slots and positions have max_tokens entries, the unused ones -1 and 0).
    All int32 except slots (int64). `out` reuses a step's tensors; its lens and
    n_free may be the inputs themselves. A step that does not fit (info) leaves
    everything as it was and has no tokens."""
    torch = _torch()
    dev = _cuda("lens", lens)
    n = lens.numel()
    a = [_take("lens", lens, torch.int32, dev, (n,)),
         _take("new_tokens", new_tokens, torch.int32, dev, (n,))]
    tp = _table(table, dev, n)
    fp = _take("free_pages", free_pages, torch.int32, dev, (free_pages.numel(),))
    np_ = _take("n_free", n_free, torch.int32, dev, (1,))
    if max_tokens < 0:
        raise _shape("max_tokens must not be negative")
    i32 = torch.int32
    if out is None:
        # one allocation for the 32-bit outputs
        buf = torch.empty(2 * n + 4 + max_tokens, dtype=i32, device=_on(dev))
        slots = torch.empty(max_tokens, dtype=torch.int64, device=_on(dev))
        lo, nf, qs, info, pos = buf.split_with_sizes([n, 1, n + 1, 2, max_tokens])
        out = PageStep(lo, nf, qs, slots, pos, info)
        b = buf.data_ptr()
        o = (b, b + 4 * n, b + 4 * n + 4, slots.data_ptr(), b + 8 * n + 16, b + 8 * n + 8)
    else:
        o = (_take("out.lens", out.lens, i32, dev, (n,)),
             _take("out.n_free", out.n_free, i32, dev, (1,)),
             _take("out.q_start", out.q_start, i32, dev, (n + 1,)),
             _take("out.slots", out.slots, torch.int64, dev, (max_tokens,)),
             _take("out.positions", out.positions, i32, dev, (max_tokens,)),
             _take("out.info", out.info, i32, dev, (2,)))
    _run(dev, "minq_pages_extend", a[0], a[1], n, page_size, tp, table.shape[1], fp,
         free_pages.numel(), np_, max_tokens, *o)
    return out


def pages_trim(lens, keep, table, free_pages, n_free, page_size: int,
               out: PageTrim | None = None) -> PageTrim:
    """Cut every request to at most keep[r] positions (0 ends it; a larger
    value keeps it whole) and put its pages back on `free_pages`."""
    torch = _torch()
    dev = _cuda("lens", lens)
    n, i32 = lens.numel(), torch.int32
    a = [_take("lens", lens, i32, dev, (n,)), _take("keep", keep, i32, dev, (n,))]
    tp = _table(table, dev, n)
    fp = _take("free_pages", free_pages, i32, dev, (free_pages.numel(),))
    np_ = _take("n_free", n_free, i32, dev, (1,))
    if out is None:
        buf = torch.empty(n + 3, dtype=i32, device=_on(dev))
        out = PageTrim(*buf.split_with_sizes([n, 1, 2]))
        b = buf.data_ptr()
        o = (b, b + 4 * n, b + 4 * n + 4)
    else:
        o = (_take("out.lens", out.lens, i32, dev, (n,)),
             _take("out.n_free", out.n_free, i32, dev, (1,)),
             _take("out.info", out.info, i32, dev, (2,)))
    _run(dev, "minq_pages_trim", a[0], a[1], n, page_size, tp, table.shape[1], fp,
         free_pages.numel(), np_, *o)
    return out


def kv4_pool(n_pages: int, n_kv: int, page_size: int, head_dim: int, device="cuda"):
    """A zeroed pool of pages for the keys (or the values) of one layer."""
    if head_dim % BLOCK_SIZE:
        raise _shape(f"head_dim must be a multiple of {BLOCK_SIZE}, got {head_dim}")
    torch = _torch()
    return torch.zeros(n_pages, n_kv, page_size, head_dim // BLOCK_SIZE * _Q4, dtype=torch.uint8,
                       device=device)


def _pools(k_pages, v_pages):
    """(n_pages, n_kv, page_size, head_dim, addresses) of a pair of pools."""
    torch = _torch()
    dev = _cuda("k_pages", k_pages)
    if k_pages.dim() != 4 or k_pages.shape[3] % _Q4:
        raise _shape("a pool must have shape [n_pages, n_kv, page_size, head_dim / 32 * 20], got "
                     f"{list(k_pages.shape)}")
    kp = _take("k_pages", k_pages, torch.uint8, dev)
    vp = _take("v_pages", v_pages, torch.uint8, dev, k_pages.shape)
    n, nkv, page, nb = k_pages.shape
    return n, nkv, page, nb // _Q4 * BLOCK_SIZE, kp, vp, dev


def _rows(name, x, n_heads, hd, dev):
    """Address and token stride of [tokens, heads, head_dim] rows (the tokens
    may be strided, as slices of a projection are)."""
    torch = _torch()
    if x.dim() != 3 or x.shape[1] != n_heads or x.shape[2] != hd:
        raise _shape(f"{name} must have shape [tokens, {n_heads}, {hd}], got {list(x.shape)}")
    p = _take(name, x, torch.float32, dev, contiguous=False)
    st = x.stride()
    if st[2] != 1 or (n_heads > 1 and st[1] != hd):
        raise _arg(f"{name}: a token's heads must be contiguous")
    return p, st[0] if x.shape[0] > 1 else n_heads * hd


def kv4_write(k, v, slots, k_pages, v_pages) -> None:
    """Quantise k, v [tokens, n_kv, head_dim] into the pools at `slots` (int64;
    negative or outside the pool: skipped; the others distinct)."""
    torch = _torch()
    n, nkv, page, hd, kp, vp, dev = _pools(k_pages, v_pages)
    a, sa = _rows("k", k, nkv, hd, dev)
    b, sb = _rows("v", v, nkv, hd, dev)
    T = k.shape[0]
    if v.shape[0] != T:
        raise _shape("k and v must hold the same tokens")
    s = _take("slots", slots, torch.int64, dev, (T,))
    _run(dev, "minq_kv4_write", a, b, sa, sb, s, T, nkv, hd, kp, vp, n, page)


def kv4_read(slots, k_pages, v_pages, out=None):
    """(k, v) [tokens, n_kv, head_dim]: the values that the rows at `slots`
    stand for (zeros outside the pool)."""
    torch = _torch()
    n, nkv, page, hd, kp, vp, dev = _pools(k_pages, v_pages)
    T = slots.numel()
    s = _take("slots", slots, torch.int64, dev, (T,))
    if out is None:
        out = torch.empty(2, T, nkv, hd, dtype=torch.float32, device=_on(dev)).unbind(0)
        a, b, sa, sb = out[0].data_ptr(), out[1].data_ptr(), nkv * hd, nkv * hd
    else:
        a, sa = _rows("out[0]", out[0], nkv, hd, dev)
        b, sb = _rows("out[1]", out[1], nkv, hd, dev)
        if out[0].shape[0] != T or out[1].shape[0] != T:
            raise _shape(f"out must hold {T} tokens")
    _run(dev, "minq_kv4_read", kp, vp, n, page, s, T, nkv, hd, a, b, sa, sb)
    return out


@functools.lru_cache(1024)
def _workspace(dev, n_req, n_tokens, n_heads, n_kv, hd) -> int:
    with _torch().cuda.device(dev):
        return lib().minq_kv4_attend_workspace_bytes(n_req, n_tokens, n_heads, n_kv, hd)


def kv4_attend(q, q_start, lens, table, k_pages, v_pages, scale: float | None = None, out=None,
               workspace=None):
    """Causal attention of the step's tokens q [tokens, n_heads, head_dim] over
    the pages of their requests; `lens` are the lengths with the step's tokens
    (PageStep.lens), whose rows are already written. Returns out [tokens,
    n_heads, head_dim]; rows behind q_start[-1] are left as they were (a fresh
    `out` holds nothing defined there). `scale`: 1 / sqrt(head_dim) unless given."""
    torch = _torch()
    n, nkv, page, hd, kp, vp, dev = _pools(k_pages, v_pages)
    if q.dim() != 3:
        raise _shape(f"q must have shape [tokens, heads, {hd}], got {list(q.shape)}")
    T, nh = q.shape[0], q.shape[1]
    qp, qs = _rows("q", q, nh, hd, dev)
    R = lens.numel()
    lp = _take("lens", lens, torch.int32, dev, (R,))
    sp = _take("q_start", q_start, torch.int32, dev, (R + 1,))
    tp = _table(table, dev, R)
    if out is None:
        out = torch.empty(T, nh, hd, dtype=torch.float32, device=_on(dev))
        op, os_ = out.data_ptr(), nh * hd
    else:
        op, os_ = _rows("out", out, nh, hd, dev)
        if out.shape[0] != T:
            raise _shape(f"out must hold {T} tokens")
    need = _workspace(dev, R, T, nh, nkv, hd)
    if workspace is None:
        workspace = torch.empty(need, dtype=torch.uint8, device=_on(dev))
    wp = _take("workspace", workspace, torch.uint8, dev)
    _run(dev, "minq_kv4_attend", qp, qs, sp, T, lp, R, tp, table.shape[1], kp, vp, n, page, nh, nkv,
         hd, 1.0 / math.sqrt(hd) if scale is None else scale, op, os_, wp, workspace.numel())
    return out


def sample_rows(logits, uniforms, temperature=None, top_k=None, top_p=None, min_p=None, out=None):
    """One token (int32) per row of logits [rows, n] from the row's uniform;
    temperature, top_p, min_p (f32) and top_k (int32) hold one value per row,
    None switches them off (see minq_sample_rows)."""
    torch = _torch()
    dev = _cuda("logits", logits)
    if logits.dim() != 2:
        raise _shape(f"logits must have shape [rows, n], got {list(logits.shape)}")
    rows, n = logits.shape
    f32 = torch.float32
    lp = _take("logits", logits, f32, dev, contiguous=False)
    if logits.stride(1) != 1 and n > 1:
        raise _arg("logits: a row must be contiguous")
    if out is None:
        out = torch.empty(rows, dtype=torch.int32, device=_on(dev))
    one = (rows,)
    _run(dev, "minq_sample_rows", lp, logits.stride(0) if rows > 1 else n, rows, n,
         None if temperature is None else _take("temperature", temperature, f32, dev, one),
         None if top_k is None else _take("top_k", top_k, torch.int32, dev, one),
         None if top_p is None else _take("top_p", top_p, f32, dev, one),
         None if min_p is None else _take("min_p", min_p, f32, dev, one),
         _take("uniforms", uniforms, f32, dev, one), _take("out", out, torch.int32, dev, one))
    return out
