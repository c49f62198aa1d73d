"""The serving-step operators (page tables, the paged 4-bit cache, attention
over it, row sampling) against plain implementations in 64 bits.

Tolerances. Page tables, slots, codes and tokens are exact. Attention, per
output element, from the arithmetic of an f32 evaluation with unit roundoff
e = 2^-24: a score is a sum of head_dim products and has an error of at most
(head_dim + 8) e sum_d |scale q_d k_d| =: ds (8 for the scales, the scaling and
the softmax's argument); a weight p_j is off by the factor exp(2 ds) and a few
e of the exponential (counted as 16 e); the sums over n positions run in
partial sums of at most n / 16 + 64 terms. So
    |out - ref| <= (2 ds + (80 + n / 16) e) sum_j p_j |v_j| + n 2^-35 a.
The last term is the smallest step of a weight's low half. The kernel holds
p_j d_j (d: V's scales) in units of vref / 2^10 with vref <= max d, as two f16
values whose smallest step is 2^-24: off by at most 2^-25 2^-10 max d, times a
code of at most 8. The weights are relative to a maximum that one position
has, so their sum is at least 1, and a position adds at most 2^-35 (8 max d);
a = 8 max d <= 8/7 max |v|, because a block's largest code is -8 or 7.
"""
import ctypes as C
import random

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

E = 2.0 ** -24


@pytest.fixture(scope="module")
def torch():
    import torch as _t
    return _t


def dev(torch, v, dtype=None):
    return torch.tensor(v, dtype=dtype or torch.int32, device="cuda")


# ---- page tables ----------------------------------------------------------------

class Book:
    """Page tables kept with Python lists."""

    def __init__(self, n_req, page, width, n_pages, seed):
        rng = random.Random(seed)
        self.page, self.width = page, width
        self.free = list(range(n_pages))
        rng.shuffle(self.free)
        self.n_pages = n_pages
        self.lens = [0] * n_req
        self.table = [[-1] * width for _ in range(n_req)]

    def extend(self, new):
        slots, pos = [], []
        for r, n in enumerate(new):
            for _ in range(n):
                i = self.lens[r]
                if i % self.page == 0:
                    self.table[r][i // self.page] = self.free.pop()
                slots.append(self.table[r][i // self.page] * self.page + i % self.page)
                pos.append(i)
                self.lens[r] += 1
        return slots, pos

    def trim(self, keep):
        back = []
        for r, k in enumerate(keep):
            k = min(k, self.lens[r])
            back += self.table[r][-(-k // self.page):-(-self.lens[r] // self.page)]
            self.lens[r] = k
        self.free += back[::-1]


class Pages:
    """The same state on the GPU."""

    def __init__(self, torch, book):
        self.t = torch
        self.lens = dev(torch, book.lens)
        self.table = dev(torch, book.table).reshape(len(book.lens), book.width)
        self.free = torch.full((book.n_pages,), -1, dtype=torch.int32, device="cuda")
        self.free[:len(book.free)] = dev(torch, book.free)
        self.n_free = dev(torch, [len(book.free)])

    def same(self, book, skip_table=()):
        assert self.lens.tolist() == book.lens
        n = int(self.n_free)
        assert n == len(book.free) and self.free[:n].tolist() == book.free
        got = self.table.tolist()
        for r, row in enumerate(book.table):
            k = -(-book.lens[r] // book.page)
            assert got[r][:k] == row[:k], r


@pytest.mark.parametrize("n_req,page,width,steps", [
    (1, 16, 4, [[1], [15], [1], [0], [47]]),
    (3, 16, 8, [[0, 0, 0], [16, 17, 0], [1, 1, 1]]),
    (5, 1024, 2, [[1024, 1, 0, 2048, 3], [0, 1023, 1, 0, 1]]),
    (64, 32, 64, "random"),
    (1500, 16, 12, "random"),
    (8192, 16, 2, "random"),
])
def test_extend_and_trim_follow_the_list(mq, torch, n_req, page, width, steps):
    book = Book(n_req, page, width, n_req * width + 3, n_req)
    gpu = Pages(torch, book)
    rng = random.Random(page)
    if steps == "random":
        steps = [[rng.choice([0, 1, rng.randint(0, page * width // 3)]) for _ in range(n_req)]
                 for _ in range(3)]
    for new in steps:
        total = sum(new)
        step = mq.pages_extend(gpu.lens, dev(torch, new), gpu.table, gpu.free, gpu.n_free, page,
                               total + 5,
                               out=mq.PageStep(gpu.lens, gpu.n_free,  # in place
                                               torch.empty(n_req + 1, dtype=torch.int32, device="cuda"),
                                               torch.empty(total + 5, dtype=torch.int64, device="cuda"),
                                               torch.empty(total + 5, dtype=torch.int32, device="cuda"),
                                               torch.empty(2, dtype=torch.int32, device="cuda")))
        slots, pos = book.extend(new)
        assert step.info.tolist() == [0, 0]
        assert step.slots.tolist() == slots + [-1] * 5
        assert step.positions.tolist() == pos + [0] * 5
        assert step.q_start.tolist() == [0] + np.cumsum(new).tolist()
        gpu.same(book)
        keep = [rng.choice([0, n, n + 9, rng.randint(0, n)]) for n in book.lens]
        cut = mq.pages_trim(gpu.lens, dev(torch, keep), gpu.table, gpu.free, gpu.n_free, page)
        assert cut.info.tolist() == [0, 0]
        gpu.lens, gpu.n_free = cut.lens, cut.n_free
        book.trim(keep)
        gpu.same(book)


def test_steps_of_nothing(mq, torch):
    """No requests, no tokens, no room for tokens, no free pages."""
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    free, n_free = dev(torch, [2, 0, 1]), dev(torch, [3])
    s = mq.pages_extend(none, none, none.reshape(0, 4), free, n_free, 16, 3)
    assert s.slots.tolist() == [-1] * 3 and s.positions.tolist() == [0] * 3
    assert s.q_start.tolist() == [0] and s.n_free.tolist() == [3] and s.info.tolist() == [0, 0]
    t = mq.pages_trim(none, none, none.reshape(0, 4), free, n_free, 16)
    assert t.n_free.tolist() == [3] and t.info.tolist() == [0, 0] and free.tolist() == [2, 0, 1]
    lens, table = dev(torch, [5, 0]), dev(torch, [[2, -1], [-1, -1]])
    s = mq.pages_extend(lens, dev(torch, [0, 0]), table, free, n_free, 16, 0)
    assert s.lens.tolist() == [5, 0] and s.q_start.tolist() == [0, 0, 0] and s.info.tolist() == [0, 0]
    s = mq.pages_extend(lens, dev(torch, [11, 0]), table, free, dev(torch, [0]), 16, 11)
    assert s.info.tolist() == [0, 0] and s.slots.tolist() == [2 * 16 + 5 + i for i in range(11)]
    kp, vp = (mq.kv4_pool(3, 2, 16, 64) for _ in range(2))
    rows = torch.empty(0, 2, 64, device="cuda")
    empty = torch.empty(0, dtype=torch.int64, device="cuda")
    mq.kv4_write(rows, rows, empty, kp, vp)
    assert mq.kv4_read(empty, kp, vp)[0].shape == (0, 2, 64)
    out = mq.kv4_attend(rows, dev(torch, [0]), none, none.reshape(0, 1), kp, vp)
    assert out.shape == (0, 2, 64)
    assert mq.sample_rows(torch.empty(0, 7, device="cuda"), torch.empty(0, device="cuda")).shape == (0,)


def test_trim_undoes_extend(mq, torch):
    book = Book(7, 16, 9, 70, 3)
    gpu = Pages(torch, book)
    free0 = gpu.free.clone()
    first = [3, 40, 0, 16, 1, 33, 90]
    a = mq.pages_extend(gpu.lens, dev(torch, first), gpu.table, gpu.free, gpu.n_free, 16, 200)
    b = mq.pages_extend(a.lens, dev(torch, [20, 5, 60, 0, 15, 1, 1]), gpu.table, gpu.free, a.n_free,
                        16, 200)
    back = mq.pages_trim(b.lens, a.lens, gpu.table, gpu.free, b.n_free, 16)
    assert back.lens.tolist() == first and int(back.n_free) == int(a.n_free)
    assert torch.equal(gpu.free, free0)


@pytest.mark.parametrize("what,flag", [("short", 1), ("row", 2), ("tokens", 4), ("neg_new", 8),
                                       ("neg_len", 8), ("bad_free", 16), ("bad_count", 16),
                                       ("over_count", 16)])
def test_extend_that_does_not_fit_changes_nothing(mq, torch, what, flag):
    book = Book(40, 16, 6, 190 if what == "short" else 200, 1)
    book.extend([17] * 40)  # two pages each
    gpu = Pages(torch, book)
    new, most = [20] * 40, 3000
    if what == "short":
        new = [60] * 40  # three more pages each: 120 of 110 free
    elif what == "row":
        new[31] = 80
    elif what == "tokens":
        most = 799
    elif what == "neg_new":
        new[3] = -1
    elif what == "neg_len":
        gpu.lens[39] = -5
    elif what == "bad_free":
        gpu.free[int(gpu.n_free) - 30] = 200
    elif what == "bad_count":
        gpu.n_free[0] = -3
    elif what == "over_count":
        gpu.n_free[0] = 201
    before = [t.clone() for t in (gpu.lens, gpu.table, gpu.free, gpu.n_free)]
    s = mq.pages_extend(gpu.lens, dev(torch, new), gpu.table, gpu.free, gpu.n_free, 16, most)
    assert int(s.info[0]) & flag
    if what == "short":
        assert s.info.tolist() == [1, 10]
    assert all(torch.equal(a, b) for a, b in zip(before, (gpu.lens, gpu.table, gpu.free, gpu.n_free)))
    assert torch.equal(s.lens, gpu.lens) and torch.equal(s.n_free, gpu.n_free)
    assert s.q_start.tolist() == [0] * 41
    assert (s.slots == -1).all() and (s.positions == 0).all()


def test_extend_reports_the_missing_pages(mq, torch):
    book = Book(4, 16, 64, 10, 1)
    gpu = Pages(torch, book)
    s = mq.pages_extend(gpu.lens, dev(torch, [100, 1, 0, 64]), gpu.table, gpu.free, gpu.n_free, 16,
                        300)
    assert s.info.tolist() == [mq.PAGES_SHORT, 7 + 1 + 4 - 10]


@pytest.mark.parametrize("what,flag", [("neg", 8), ("bad_page", 16), ("full", 16), ("len", 2)])
def test_trim_that_does_not_fit_changes_nothing(mq, torch, what, flag):
    book = Book(6, 16, 4, 24, 2)
    book.extend([60, 3, 17, 0, 32, 64])
    gpu = Pages(torch, book)
    keep = [1, 0, 0, 0, 0, 20]
    if what == "neg":
        keep[2] = -1
    elif what == "bad_page":
        gpu.table[5, 3] = 24
    elif what == "full":
        gpu.n_free[0] = 20
    elif what == "len":
        gpu.lens[3] = 65
    before = [t.clone() for t in (gpu.lens, gpu.table, gpu.free, gpu.n_free)]
    s = mq.pages_trim(gpu.lens, dev(torch, keep), gpu.table, gpu.free, gpu.n_free, 16)
    assert int(s.info[0]) & flag
    n = int(gpu.n_free)  # what lies above is no part of the list
    before[2], gpu.free = before[2][:n], gpu.free[:n]
    assert all(torch.equal(a, b) for a, b in zip(before, (gpu.lens, gpu.table, gpu.free, gpu.n_free)))
    assert torch.equal(s.lens, gpu.lens) and torch.equal(s.n_free, gpu.n_free)


# ---- the cache's rows ---------------------------------------------------------------

def _pool_rows(torch, pool, slots):
    n, nkv, page, nb = pool.shape
    s = torch.as_tensor(slots, device="cuda")
    h = torch.arange(nkv, device="cuda")[None]
    return pool[(s // page)[:, None], h, (s % page)[:, None]]


@pytest.mark.parametrize("T,nkv,hd,page", [(1, 1, 32, 16), (3, 2, 64, 16), (17, 8, 128, 16),
                                           (33, 3, 96, 32), (64, 1, 256, 1024), (700, 2, 128, 64)])
def test_write_is_the_quantiser_and_read_the_dequantiser(mq, torch, T, nkv, hd, page):
    g = torch.Generator(device="cuda").manual_seed(T)
    n_pages = -(-T // page) + 2
    # keys and values as slices of one projection, rows of very different size
    qkv = torch.randn(T, 3 * nkv, hd, generator=g, device="cuda")
    qkv *= torch.exp(4 * torch.randn(T, 3 * nkv, 1, generator=g, device="cuda"))
    qkv[0, nkv] = 0.0
    k, v = qkv[:, nkv:2 * nkv], qkv[:, 2 * nkv:]
    slots = torch.randperm(n_pages * page, generator=g, device="cuda")[:T]
    kp, vp = mq.kv4_pool(n_pages, nkv, page, hd), mq.kv4_pool(n_pages, nkv, page, hd)
    kp.fill_(0xAB), vp.fill_(0xCD)
    mq.kv4_write(k, v, slots, kp, vp)
    other = torch.ones(n_pages * page, dtype=torch.bool, device="cuda")
    other[slots] = False
    for x, pool, mark in ((k, kp, 0xAB), (v, vp, 0xCD)):
        want = mq.quantize_q4_0(x.contiguous().cpu().numpy())
        got = _pool_rows(torch, pool, slots)
        assert np.array_equal(got.cpu().numpy().reshape(-1), want)
        rest = pool.permute(0, 2, 1, 3).reshape(n_pages * page, -1)[other]
        assert (rest == mark).all()  # nothing else is touched
    back = mq.kv4_read(slots, kp, vp)
    for x, y in ((k, back[0]), (v, back[1])):
        want = mq.dequantize_q4_0(mq.quantize_q4_0(x.contiguous().cpu().numpy()))
        assert np.array_equal(y.cpu().numpy().reshape(-1).view(np.uint32), want.view(np.uint32))


def test_write_of_nonfinite_values_matches_the_quantiser(mq, torch):
    x = torch.randn(6, 2, 64, device="cuda")
    x[0, 0, 3], x[1, 1, 40], x[2, 0, 0], x[3, 1] = float("nan"), float("inf"), -float("inf"), 0.0
    x[4, 0] = float("nan")
    x[5] *= 1e-42  # denormal scales
    kp, vp = mq.kv4_pool(1, 2, 16, 64), mq.kv4_pool(1, 2, 16, 64)
    mq.kv4_write(x, x, torch.arange(6, device="cuda"), kp, vp)
    want = mq.quantize_q4_0(x.cpu().numpy())
    for pool in (kp, vp):
        assert np.array_equal(_pool_rows(torch, pool, range(6)).cpu().numpy().reshape(-1), want)


def test_slots_outside_the_pool_are_skipped_and_read_as_zero(mq, torch):
    x = torch.randn(5, 2, 64, device="cuda")
    kp, vp = mq.kv4_pool(2, 2, 16, 64), mq.kv4_pool(2, 2, 16, 64)
    slots = torch.tensor([-1, 5, 32, 2**62, -2**63], dtype=torch.int64, device="cuda")
    mq.kv4_write(x, x, slots, kp, vp)
    used = kp.permute(0, 2, 1, 3).reshape(32, -1).any(1)
    assert used.nonzero().flatten().tolist() == [5]
    k, v = mq.kv4_read(slots, kp, vp)
    assert not k[[0, 2, 3, 4]].any() and not v[[0, 2, 3, 4]].any()
    assert k[1].any()


def test_rows_at_odd_addresses(mq, torch):
    """Rows that do not start on 16 bytes take the scalar loads and stores."""
    T, nkv, hd = 9, 2, 64
    base = torch.randn(T * 131 + 8, device="cuda")
    x = torch.as_strided(base, (T, nkv, hd), (131, hd, 1), 3)
    kp, vp = mq.kv4_pool(2, nkv, 16, hd), mq.kv4_pool(2, nkv, 16, hd)
    slots = torch.arange(20, 20 + T, device="cuda")
    mq.kv4_write(x, x, slots, kp, vp)
    want = mq.quantize_q4_0(x.contiguous().cpu().numpy())
    assert np.array_equal(_pool_rows(torch, kp, slots).cpu().numpy().reshape(-1), want)
    assert torch.equal(kp, vp)
    room = torch.full((T * 131 + 8,), 7.0, device="cuda")
    o = torch.as_strided(room, (T, nkv, hd), (131, hd, 1), 1)
    mq.kv4_read(slots, kp, vp, out=(o, torch.empty(T, nkv, hd, device="cuda")))
    assert np.array_equal(o.cpu().numpy().reshape(-1), mq.dequantize_q4_0(want))
    gaps = torch.as_strided(room, (T, 3), (131, 1), 1 + nkv * hd)
    assert (gaps == 7.0).all() and room[0] == 7.0


# ---- attention ------------------------------------------------------------------------

def _fill(mq, torch, seed, lens, nkv, hd, page, width=None, extra=2, gain=1.0):
    """Pools, table and the values in them (f64, [request][kv head][pos][hd])."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    used = [-(-max(n, 0) // page) for n in lens]
    n_pages = sum(used) + extra
    order = torch.randperm(n_pages, generator=g, device="cuda").int()
    width = width or max(1, max(used))
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for r, u in enumerate(used):
        table[r, :u] = order[at:at + u]
        at += u
    pools, vals = [], []
    for side in range(2):
        x = torch.randn(n_pages, nkv, page, hd, generator=g, device="cuda")
        x *= torch.exp(0.5 * torch.randn(n_pages, nkv, page, 1, generator=g, device="cuda"))
        x *= gain if side == 0 else 1.0
        pool = mq.kv4_pool(n_pages, nkv, page, hd)
        slots = torch.arange(n_pages * page, device="cuda")
        rows = x.permute(0, 2, 1, 3).reshape(n_pages * page, nkv, hd)
        spare = mq.kv4_pool(n_pages, nkv, page, hd)
        mq.kv4_write(rows, rows, slots, pool, spare)
        pools.append(pool)
        vals.append(mq.kv4_read(slots, pool, pool)[0].double())  # [slot][kv head][hd]
    return pools[0], pools[1], table, vals[0], vals[1]


def _reference(torch, q, start, lens, table, page, kv, vv, scale, seen=None):
    """f64 outputs and the bound on each element; rows outside stay NaN."""
    T, nh, hd = q.shape
    nkv = kv.shape[1]
    G = nh // nkv
    out = torch.full((T, nh, hd), float("nan"), dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(out)
    tab = table.long()
    for r in range(len(lens)):
        n = min(max(lens[r], 0), table.shape[1] * page)
        i = torch.arange(n, device="cuda")
        pg = tab[r, i // page]
        ok = (pg >= 0) & (pg < kv.shape[0] // page)
        slot = torch.where(ok, pg * page + i % page, 0)
        for t in range(start[r], start[r + 1]):
            pos = lens[r] - (start[r + 1] - t)
            m = ok & (i <= pos)
            if not m.any():
                out[t] = 0.0
                continue
            k = kv[slot[m]].repeat_interleave(G, 1)  # [n][nh][hd]
            v = vv[slot[m]].repeat_interleave(G, 1)
            s = (q[t].double()[None] * k).sum(-1) * scale
            ds = ((q[t].double().abs()[None] * k.abs()).sum(-1) * abs(scale)).amax(0) * (hd + 8) * E
            p = torch.softmax(s, 0)
            out[t] = (p[..., None] * v).sum(0)
            spread = (p[..., None] * v.abs()).sum(0)
            step = int(m.sum()) * 2.0 ** -35 * 8 / 7 * v.abs().amax((0, 2))
            tol[t] = (2 * ds[:, None] + (80 + int(m.sum()) / 16) * E) * spread + step[:, None]
    return out, tol


def _check(torch, got, want, tol):
    rows = ~torch.isnan(want).any(-1).any(-1)
    err = (got.double() - want)[rows].abs()
    assert torch.isfinite(got[rows]).all()
    bad = err > tol[rows] + 1e-30
    assert not bad.any(), (int(bad.sum()), float((err / (tol[rows] + 1e-30)).max()))


HEADS = [(32, 8, 128), (14, 2, 64), (8, 8, 64), (4, 4, 128), (16, 1, 128), (40, 1, 64), (9, 1, 128),
         (6, 2, 32), (4, 2, 96), (4, 1, 256)]


@pytest.mark.parametrize("nh,nkv,hd", HEADS)
@pytest.mark.parametrize("page,lens,new", [
    (16, [1], [1]),
    (16, [700, 16, 17, 1, 250], [1, 1, 1, 1, 1]),
    (64, [333, 0, 40, 129], [5, 0, 40, 1]),
    (128, [1500], [65]),
])
def test_attend_matches_the_formula(mq, torch, nh, nkv, hd, page, lens, new):
    kp, vp, table, kv, vv = _fill(mq, torch, nh + hd + len(lens), lens, nkv, hd, page, width=14 * 128 // page)
    start = [0] + np.cumsum(new).tolist()
    g = torch.Generator(device="cuda").manual_seed(5)
    q = torch.randn(start[-1], nh, hd, generator=g, device="cuda") * 2
    scale = hd ** -0.5
    got = mq.kv4_attend(q, dev(torch, start), dev(torch, lens), table, kp, vp)
    want, tol = _reference(torch, q, start, lens, table, page, kv, vv, scale)
    _check(torch, got, want, tol)


@pytest.mark.parametrize("nh,nkv,hd", [(32, 8, 128), (14, 2, 64), (4, 2, 96)])
def test_attend_peaked_scores_and_large_values(mq, torch, nh, nkv, hd):
    """Scores in the hundreds (the running maximum moves late) and value rows
    whose scales differ by orders of magnitude."""
    lens, page = [900, 77], 32
    kp, vp, table, kv, vv = _fill(mq, torch, 3, lens, nkv, hd, page, gain=6.0)
    rows = vv * torch.exp(3 * torch.randn(vv.shape[0], 1, 1, device="cuda")).double()
    slots = torch.arange(vv.shape[0], device="cuda")
    mq.kv4_write(rows.float(), rows.float(), slots, vp, mq.kv4_pool(*vp.shape[:3], hd))
    vv = mq.kv4_read(slots, kp, vp)[1].double()
    start = [0, 3, 4]
    q = torch.randn(4, nh, hd, device="cuda") * 8
    got = mq.kv4_attend(q, dev(torch, start), dev(torch, lens), table, kp, vp, scale=0.3)
    want, tol = _reference(torch, q, start, lens, table, page, kv, vv, 0.3)
    _check(torch, got, want, tol)


@pytest.mark.parametrize("nh,nkv,hd", [(32, 8, 128), (14, 2, 64), (4, 2, 96)])
def test_attend_ignores_what_no_token_may_see(mq, torch, nh, nkv, hd):
    """NaN and infinite scales behind the last position, in pages of no
    request and under bad ids change nothing; rows that see nothing are zero
    and rows behind the last sequence stay as they were."""
    page, lens = 16, [37, 0, 50, 20, 64]
    new = [2, 0, 1, 1, 3]
    kp, vp, table, kv, vv = _fill(mq, torch, 9, lens, nkv, hd, page, width=5, extra=3)
    n_pages = kp.shape[0]
    seen = torch.zeros(n_pages, page, dtype=torch.bool, device="cuda")
    table[2, 1] = n_pages  # a bad page in the middle of a request
    table[3] = -1          # and a request of nothing but bad pages
    table[4, 3] = -2**31
    for r, n in enumerate(lens):
        for i in range(n):
            pg = int(table[r, i // page])
            if 0 <= pg < n_pages:
                seen[pg, i % page] = True
    for pool, bad in ((kp, float("nan")), (vp, float("inf"))):
        blocks = pool.view(n_pages, nkv, page, hd // 32, 20)
        mark = torch.tensor([bad], device="cuda").view(torch.uint8)
        hide = ~seen[:, None, :, None].expand(n_pages, nkv, page, hd // 32)
        blocks[..., :4] = torch.where(hide[..., None], mark, blocks[..., :4])
    start = [0] + np.cumsum(new).tolist()
    T = start[-1] + 4
    q = torch.randn(T, nh, hd, device="cuda")
    q[start[-1]:] = float("nan")
    out = torch.full((T, nh, hd), 5.0, device="cuda")
    mq.kv4_attend(q, dev(torch, start), dev(torch, lens), table, kp, vp, out=out)
    want, tol = _reference(torch, q, start, lens, table, page, kv, vv, hd ** -0.5)
    assert not out[3].any()  # the request of bad pages
    assert (out[start[-1]:] == 5.0).all()
    _check(torch, out[:start[-1]], want[:start[-1]], tol[:start[-1]])


def test_attend_lengths_that_contradict_the_starts(mq, torch):
    """More new tokens than positions: the tokens before the start see
    nothing. A length past the table row sees the row."""
    nh, nkv, hd, page = 8, 2, 64, 16
    lens, start = [3, 40], [0, 5, 6]
    kp, vp, table, kv, vv = _fill(mq, torch, 2, [16, 32], nkv, hd, page)
    q = torch.randn(6, nh, hd, device="cuda")
    got = mq.kv4_attend(q, dev(torch, start), dev(torch, lens), table, kp, vp)
    want, tol = _reference(torch, q, start, lens, table, page, kv, vv, hd ** -0.5)
    assert not got[:2].any()
    _check(torch, got, want, tol)
    # starts outside the tokens: those requests have none
    out = torch.full_like(got, 3.0)
    mq.kv4_attend(q, dev(torch, [-2, 1, 99]), dev(torch, lens), table, kp, vp, out=out)
    assert torch.isfinite(out).all()


def test_attend_strided_rows_and_odd_addresses(mq, torch):
    nh, nkv, hd, page, lens, start = 16, 4, 64, 32, [100, 31], [0, 3, 4]
    kp, vp, table, kv, vv = _fill(mq, torch, 4, lens, nkv, hd, page)
    base = torch.randn(4 * 1500 + 8, device="cuda")
    q = torch.as_strided(base, (4, nh, hd), (1499, hd, 1), 1)
    room = torch.full((4 * 1100 + 8,), 9.0, device="cuda")
    out = torch.as_strided(room, (4, nh, hd), (1099, hd, 1), 3)
    mq.kv4_attend(q, dev(torch, start), dev(torch, lens), table, kp, vp, out=out)
    want, tol = _reference(torch, q, start, lens, table, page, kv, vv, hd ** -0.5)
    _check(torch, out, want, tol)
    gaps = torch.as_strided(room, (3, 1099 - nh * hd), (1099, 1), 3 + nh * hd)
    assert (gaps == 9.0).all() and (room[:3] == 9.0).all()


def test_attend_repeats_bit_for_bit_and_in_a_graph(mq, torch):
    """The same bits on every call, on a side stream, and from a captured graph
    replayed over changed lengths."""
    nh, nkv, hd, page = 32, 8, 128, 16
    lens, new = [3000, 17, 801], [1, 1, 1]
    kp, vp, table, kv, vv = _fill(mq, torch, 8, lens, nkv, hd, page)
    start = dev(torch, [0, 1, 2, 3])
    ld = dev(torch, lens)
    q = torch.randn(3, nh, hd, device="cuda")
    a = mq.kv4_attend(q, start, ld, table, kp, vp)
    b = mq.kv4_attend(q, start, ld, table, kp, vp)
    assert torch.equal(a, b)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        c = mq.kv4_attend(q, start, ld, table, kp, vp)
    s.synchronize()
    assert torch.equal(a, c)
    out = torch.empty_like(a)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mq.kv4_attend(q, start, ld, table, kp, vp, out=out)
    for lens2 in (lens, [2048, 1, 16], [1, 17, 800]):
        ld.copy_(dev(torch, lens2))
        graph.replay()
        want, tol = _reference(torch, q, [0, 1, 2, 3], lens2, table, page, kv, vv, hd ** -0.5)
        _check(torch, out, want, tol)
    ld.copy_(dev(torch, lens))
    graph.replay()
    assert torch.equal(out, a)


# Prompt chunks (64 and more rows of a kv head) have a kernel of their own, whose
# arithmetic keeps the bound above: K and V as two f16 parts are off by 2^-23 of
# each value; a score's 3 head_dim / 16 tensor-core steps truncate at 2 e each,
# 48 e at head_dim 128, inside (head_dim + 8) e; a tile's 12 steps of P V 24 e,
# inside 80 e, and the tiles' sums are n / 64 f32 additions. The smallest steps
# of the parts of P and V are 2^-34 and 2^-36 of the largest weight and value.

CHUNK_HEADS = [(32, 8, 128), (14, 2, 64), (4, 4, 128), (16, 1, 128), (160, 1, 64), (129, 1, 128)]


@pytest.mark.parametrize("nh,nkv,hd", CHUNK_HEADS)
@pytest.mark.parametrize("page,lens,new", [
    (16, [64], [64]),                             # no history
    (16, [130, 700, 5, 0, 64], [129, 64, 1, 0, 63]),  # ends inside a tile, with single tokens
    (1024, [1100, 321], [70, 200]),               # one page holds whole tiles
])
def test_attend_chunks_match_the_formula(mq, torch, nh, nkv, hd, page, lens, new):
    kp, vp, table, kv, vv = _fill(mq, torch, nh + hd, lens, nkv, hd, page)
    start = [0] + np.cumsum(new).tolist()
    g = torch.Generator(device="cuda").manual_seed(6)
    q = torch.randn(start[-1], nh, hd, generator=g, device="cuda") * 2
    got = mq.kv4_attend(q, dev(torch, start), dev(torch, lens), table, kp, vp)
    want, tol = _reference(torch, q, start, lens, table, page, kv, vv, hd ** -0.5)
    _check(torch, got, want, tol)
    assert torch.equal(got, mq.kv4_attend(q, dev(torch, start), dev(torch, lens), table, kp, vp))


@pytest.mark.parametrize("scale", [0.0, -0.09, 0.4])
@pytest.mark.parametrize("nh,nkv,hd", [(32, 8, 128), (14, 2, 64)])
def test_attend_chunks_any_scale_and_large_values(mq, torch, nh, nkv, hd, scale):
    """Even weights, the reverse order, scores in the hundreds; value rows whose
    scales differ by orders of magnitude."""
    lens, page, new = [900, 77], 32, [65, 70]
    kp, vp, table, kv, vv = _fill(mq, torch, 3, lens, nkv, hd, page, gain=6.0)
    rows = vv * torch.exp(3 * torch.randn(vv.shape[0], 1, 1, device="cuda")).double()
    slots = torch.arange(vv.shape[0], device="cuda")
    mq.kv4_write(rows.float(), rows.float(), slots, vp, mq.kv4_pool(*vp.shape[:3], hd))
    vv = mq.kv4_read(slots, kp, vp)[1].double()
    start = [0, 65, 135]
    q = torch.randn(135, nh, hd, device="cuda") * 8
    got = mq.kv4_attend(q, dev(torch, start), dev(torch, lens), table, kp, vp, scale=scale)
    want, tol = _reference(torch, q, start, lens, table, page, kv, vv, scale)
    _check(torch, got, want, tol)


@pytest.mark.parametrize("nh,nkv,hd", [(32, 8, 128), (14, 2, 64)])
def test_attend_chunks_ignore_what_a_token_may_not_see(mq, torch, nh, nkv, hd):
    """Bad pages at the start, in the middle and throughout; NaN and infinite
    scales in all that no token sees; a value scale that is not finite reaches
    the tokens behind it, in its block, and no other."""
    page, lens, new = 16, [200, 100, 150], [70, 65, 66]
    kp, vp, table, kv, vv = _fill(mq, torch, 9, lens, nkv, hd, page, width=14, extra=3)
    n_pages, nb = kp.shape[0], hd // 32
    table[0, 0], table[0, 6], table[0, 9] = -1, n_pages, -2**31
    table[1] = -1
    seen = torch.zeros(n_pages, page, dtype=torch.bool, device="cuda")
    for r, n in enumerate(lens):
        for i in range(n):
            pg = int(table[r, i // page])
            if 0 <= pg < n_pages:
                seen[pg, i % page] = True
    blocks = [p.view(n_pages, nkv, page, nb, 20) for p in (kp, vp)]
    for b, bad in zip(blocks, (float("nan"), float("inf"))):
        mark = torch.tensor([bad], device="cuda").view(torch.uint8)
        hide = ~seen[:, None, :, None].expand(n_pages, nkv, page, nb)
        b[..., :4] = torch.where(hide[..., None], mark, b[..., :4])
    start = [0] + np.cumsum(new).tolist()
    T = start[-1] + 3
    q = torch.randn(T, nh, hd, device="cuda")
    q[start[-1]:] = float("nan")
    out = torch.full((T, nh, hd), 5.0, device="cuda")
    args = (q, dev(torch, start), dev(torch, lens), table, kp, vp)
    mq.kv4_attend(*args, out=out)
    want, tol = _reference(torch, q[:start[-1]], start, lens, table, page, kv, vv, hd ** -0.5)
    assert not out[start[1]:start[2]].any()
    assert (out[start[-1]:] == 5.0).all()
    _check(torch, out[:start[-1]], want, tol)
    # position 120 of request 2 (its tokens are 84 .. 149), kv head 1, block 1 of V
    pg = int(table[2, 120 // page])
    for bad in (float("inf"), float("nan")):
        blocks[1][pg, 1, 120 % page, 1, :4] = torch.tensor([bad], device="cuda").view(torch.uint8)
        got = mq.kv4_attend(*args)[:start[-1]]
        hit = torch.zeros_like(got, dtype=torch.bool)
        G = nh // nkv
        hit[start[2] + 36:start[3], G:2 * G, 32:64] = True
        assert not torch.isfinite(got[hit]).any()
        assert torch.equal(got[~hit], out[:start[-1]][~hit])
    # a key scale that is not finite: the tokens before it do not notice
    blocks[1][pg, 1, 120 % page, 1, :4] = torch.tensor([0.0], device="cuda").view(torch.uint8)
    blocks[0][pg, 1, 120 % page, 0, :4] = torch.tensor([float("nan")], device="cuda").view(torch.uint8)
    got = mq.kv4_attend(*args)[:start[-1]]
    assert not torch.isfinite(got[start[2] + 36:start[3], G:2 * G]).any()
    assert torch.equal(got[:start[2] + 36], out[:start[2] + 36])


def test_attend_many_requests(mq, torch):
    """More requests than a CTA has threads, decoding ones between chunks."""
    rng = random.Random(4)
    nh, nkv, hd, page = 8, 2, 64, 16
    lens = [rng.choice([0, 1, 16, rng.randint(1, 90)]) for _ in range(900)]
    new = [min(n, rng.choice([0, 1, 1, 1, 1, 1, 3])) for n in lens]
    for r in (0, 333, 700, 899):
        lens[r], new[r] = 150, 40
    kp, vp, table, kv, vv = _fill(mq, torch, 1, lens, nkv, hd, page)
    start = [0] + np.cumsum(new).tolist()
    q = torch.randn(start[-1], nh, hd, device="cuda")
    got = mq.kv4_attend(q, dev(torch, start), dev(torch, lens), table, kp, vp)
    want, tol = _reference(torch, q, start, lens, table, page, kv, vv, hd ** -0.5)
    _check(torch, got, want, tol)
    # the same requests with one token each (many more of them than a CTA's threads)
    one = [min(n, 1) for n in lens]
    start = [0] + np.cumsum(one).tolist()
    q = torch.randn(start[-1], nh, hd, device="cuda")
    got = mq.kv4_attend(q, dev(torch, start), dev(torch, lens), table, kp, vp)
    want, tol = _reference(torch, q, start, lens, table, page, kv, vv, hd ** -0.5)
    _check(torch, got, want, tol)


def test_attend_two_streams_and_a_chunk_in_a_graph(mq, torch):
    """Calls that overlap on two streams, and a captured mixed step replayed over
    other lengths (chunks that become single tokens and the other way round)."""
    nh, nkv, hd, page = 32, 8, 128, 32
    lens, new = [900, 400, 33], [64, 1, 30]
    kp, vp, table, kv, vv = _fill(mq, torch, 5, lens, nkv, hd, page)
    start = [0] + np.cumsum(new).tolist()
    sd, ld = dev(torch, start), dev(torch, lens)
    qs = [torch.randn(start[-1], nh, hd, device="cuda") for _ in range(2)]
    alone = [mq.kv4_attend(q, sd, ld, table, kp, vp) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(mq.kv4_attend(qs[i], sd, ld, table, kp, vp))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, alone[i]) for g in got[i])
    out = torch.empty_like(qs[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mq.kv4_attend(qs[0], sd, ld, table, kp, vp, out=out)
    graph.replay()
    assert torch.equal(out, alone[0])
    for lens2, new2 in (([700, 399, 31], [1, 80, 14]), ([20, 1, 33], [0, 1, 33]), (lens, new)):
        start2 = [0] + np.cumsum(new2).tolist()
        sd.copy_(dev(torch, start2))
        ld.copy_(dev(torch, lens2))
        out.fill_(7.0)
        graph.replay()
        want, tol = _reference(torch, qs[0], start2, lens2, table, page, kv, vv, hd ** -0.5)
        _check(torch, out[:start2[-1]], want[:start2[-1]], tol[:start2[-1]])
        assert (out[start2[-1]:] == 7.0).all()
    assert torch.equal(out, alone[0])


FIRST_CALL = """
import torch, minq_b200 as mq
kp, vp = (mq.kv4_pool(4, 8, 16, 128) for _ in range(2))
i32 = dict(dtype=torch.int32, device="cuda")
lens, table = torch.tensor([20], **i32), torch.tensor([[1, 3]], **i32)
start, q = torch.tensor([0, 20], **i32), torch.randn(20, 32, 128, device="cuda")
slots = torch.tensor([16 + i if i < 16 else 48 + i - 16 for i in range(20)], device="cuda")
k, v = (torch.randn(20, 8, 128, device="cuda") for _ in range(2))
logits, u = torch.randn(3, 5000, device="cuda"), torch.rand(3, device="cuda")
new, free, n_free = torch.tensor([5], **i32), torch.tensor([0, 2], **i32), torch.tensor([2], **i32)
torch.cuda.synchronize()
def step():
    mq.kv4_write(k, v, slots, kp, vp)
    return (*mq.kv4_read(slots, kp, vp), mq.kv4_attend(q, start, lens, table, kp, vp),
            mq.sample_rows(logits, u), mq.pages_extend(lens, new, table.clone(), free, n_free, 16, 8).slots)
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):  # the first call of everything
    got = step()
graph.replay()
torch.cuda.synchronize()
want = step()
assert all(torch.equal(a, b) for a, b in zip(got, want))
mq._lib.check(mq._lib.lib().minq_device_status())
print("same")
"""


def test_first_call_inside_a_capture(mq, torch):
    import subprocess
    import sys
    r = subprocess.run([sys.executable, "-c", FIRST_CALL], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip().endswith("same"), r.stderr[-2000:]


def test_attend_pages_past_four_gigabytes(mq, torch):
    """Byte offsets beyond 32 bits: the pages lie at the end of a 5 GB pool."""
    nh, nkv, hd, page = 8, 8, 128, 64
    n_pages = 5 * 2**30 // (nkv * page * 80)
    kp = torch.empty(n_pages, nkv, page, 80, dtype=torch.uint8, device="cuda")
    vp = torch.empty_like(kp)
    lens = [200]
    ids = [n_pages - 1, 5, n_pages - 2, n_pages // 2]
    table = dev(torch, [ids])
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(2, 200, nkv, hd, generator=g, device="cuda")
    slots = torch.tensor([ids[i // page] * page + i % page for i in range(200)], device="cuda")
    assert int(slots.max()) * nkv * 80 > 2**32
    mq.kv4_write(x[0], x[1], slots, kp, vp)
    k, v = mq.kv4_read(slots, kp, vp)
    q = torch.randn(2, nh, hd, generator=g, device="cuda")
    got = mq.kv4_attend(q, dev(torch, [0, 2]), dev(torch, lens), table, kp, vp)
    own = dev(torch, [[0, 1, 2, 3]])
    full = torch.zeros(256, nkv, hd, dtype=torch.float64, device="cuda")
    kv, vv = full.clone(), full.clone()
    kv[:200], vv[:200] = k.double(), v.double()
    want, tol = _reference(torch, q, [0, 2], lens, own, page, kv, vv, hd ** -0.5)
    _check(torch, got, want, tol)


@pytest.mark.parametrize("tokens,hd", [(100, 128), (100, 64), (3, 96)])
def test_attend_kernels_past_four_gigabytes(mq, torch, tokens, hd):
    """The same for a chunk's kernel and for the plain one."""
    nh, nkv, page, n = 4, 4, 32, 150
    n_pages = 2**32 // (nkv * page * (hd // 32 * 20)) + 100
    kp = torch.empty(n_pages, nkv, page, hd // 32 * 20, dtype=torch.uint8, device="cuda")
    vp = torch.empty_like(kp)
    ids = [n_pages - 1, 5, n_pages - 2, n_pages // 2, n_pages - 9]
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(2, n, nkv, hd, generator=g, device="cuda")
    slots = torch.tensor([ids[i // page] * page + i % page for i in range(n)], device="cuda")
    mq.kv4_write(x[0], x[1], slots, kp, vp)
    k, v = mq.kv4_read(slots, kp, vp)
    q = torch.randn(tokens, nh, hd, generator=g, device="cuda")
    got = mq.kv4_attend(q, dev(torch, [0, tokens]), dev(torch, [n]), dev(torch, [ids]), kp, vp)
    full = torch.zeros(5 * page, nkv, hd, dtype=torch.float64, device="cuda")
    kv, vv = full.clone(), full.clone()
    kv[:n], vv[:n] = k.double(), v.double()
    want, tol = _reference(torch, q, [0, tokens], [n], dev(torch, [[0, 1, 2, 3, 4]]), page, kv, vv,
                           hd ** -0.5)
    _check(torch, got, want, tol)


@pytest.mark.parametrize("nh,nkv,hd,new", [(4, 1, 64, 20), (4, 1, 64, 3), (2, 1, 128, 64)])
def test_attend_few_rows_of_a_long_history(mq, torch, nh, nkv, hd, new):
    """More pieces of an item than one warp joins."""
    lens, page = [70001], 64
    kp, vp, table, kv, vv = _fill(mq, torch, 12, lens, nkv, hd, page)
    q = torch.randn(new, nh, hd, device="cuda")
    got = mq.kv4_attend(q, dev(torch, [0, new]), dev(torch, lens), table, kp, vp)
    want, tol = _reference(torch, q, [0, new], lens, table, page, kv, vv, hd ** -0.5)
    _check(torch, got, want, tol)


def test_attend_equals_the_f32_cache_attention(mq, torch):
    """Next to minq_attend over the values that the cache stands for."""
    from minq_b200 import _lib
    nh, nkv, hd, page, n = 32, 8, 128, 16, 1000
    kp, vp, table, kv, vv = _fill(mq, torch, 6, [n], nkv, hd, page)
    i = torch.arange(n, device="cuda")
    slot = table[0].long()[i // page] * page + i % page
    k, v = kv[slot].float().contiguous(), vv[slot].float().contiguous()
    q = torch.randn(1, nh, hd, device="cuda")
    got = mq.kv4_attend(q, dev(torch, [0, 1]), dev(torch, [n]), table, kp, vp)
    L = _lib.lib()
    out = torch.empty_like(q)
    wb = L.minq_attn_workspace_bytes(1, nh, n)
    ws = torch.empty(wb, dtype=torch.uint8, device="cuda")
    P = lambda t: C.c_void_p(t.data_ptr())  # noqa: E731
    _lib.check(L.minq_attend(P(q), P(k), P(v), n, nh, nkv, hd, P(out), P(ws), wb, None))
    torch.cuda.synchronize()
    want, tol = _reference(torch, q, [0, 1], [n], table, page, kv, vv, hd ** -0.5)
    _check(torch, got, want, tol)
    assert ((got - out).double().abs() <= 2 * tol).all()


# ---- sampling -----------------------------------------------------------------------------

def _draw(x, u, t=1.0, k=0, p=1.0, mp=0.0):
    """One row in f64 numpy, from the definition."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    n = len(x)
    rank = np.lexsort((np.arange(n), -x))
    if not t > 0 or k == 1:
        return int(rank[0])
    top = x[rank[0]]
    if top == -np.inf:
        return 0
    with np.errstate(invalid="ignore"):
        w = np.where(x == top, 1.0, np.exp((x - top) / t))
    w[x == -np.inf] = 0.0
    if not ((0 < k < n) or p < 1 or mp > 0):
        c = np.cumsum(w)
        return int(np.flatnonzero((c >= u * c[-1]) & (w > 0))[0])
    wr = w[rank]
    c = np.cumsum(wr)
    keep = n
    if 0 < k < n:
        keep = k
    if p < 1:
        keep = min(keep, int(np.searchsorted(c, float(p) * c[-1])) + 1)
    if mp > 0:
        keep = min(keep, max(1, int((wr >= float(mp)).sum())))
    c = np.cumsum(wr[:max(1, keep)])
    return int(rank[np.flatnonzero((c >= u * c[-1]) & (wr[:len(c)] > 0))[0]])


def _settings(rng, n):
    return (rng.choice([0.0, 0.3, 0.8, 1.0, 1.0, 2.5, 50.0]),
            rng.choice([0, 0, 1, 2, 5, 40, 1000, n, n + 7, -3]),
            rng.choice([1.0, 1.0, 0.1, 0.5, 0.9, 0.99, 0.0, 1.5]),
            rng.choice([0.0, 0.0, 0.01, 0.2, 1.0, 2.0, -1.0]))


@pytest.mark.parametrize("n", [1, 2, 31, 100, 1023, 4097, 32000, 50257])
@pytest.mark.parametrize("kind", ["normal", "flat", "ties", "masked", "peaked"])
def test_sample_rows_follows_the_definition(mq, torch, n, kind):
    rng = random.Random(n * 7 + len(kind))
    g = np.random.default_rng(n + len(kind))
    rows = 40 if n < 5000 else 24
    x = g.standard_normal((rows, n)).astype(np.float32) * 2
    if kind == "flat":
        x *= 1e-4
    elif kind == "ties":
        x = np.round(x)
    elif kind == "masked":
        x[g.random((rows, n)) < 0.8] = -np.inf
        x[:, -1] = np.where(np.isinf(x[:, -1]), 0.5, x[:, -1])
        x[0] = -np.inf  # nothing left
        x[1] = np.finfo(np.float32).min
        x[2, ::2] = np.finfo(np.float32).min
        x[3, 0] = np.nan
        x[4] = np.nan
    elif kind == "peaked":
        x[np.arange(rows), g.integers(0, n, rows)] += 30
    s = [_settings(rng, n) for _ in range(rows)]
    if kind == "masked":  # NaN orders above all in a greedy row: a test of its own
        s[3], s[4] = (1.0, 0, 1.0, 0.0), (0.7, 5, 0.9, 0.0)
    u = g.random(rows).astype(np.float32)
    u = np.minimum(u, np.float32(1 - 2**-24))
    u[-1] = 0.0
    f = lambda i, t=torch.float32: torch.tensor([v[i] for v in s], dtype=t, device="cuda")  # noqa: E731
    got = mq.sample_rows(torch.from_numpy(x).cuda(), torch.from_numpy(u).cuda(), temperature=f(0),
                         top_k=f(1, torch.int32), top_p=f(2), min_p=f(3)).tolist()
    s32 = [(np.float32(a), b, np.float32(c), np.float32(d)) for a, b, c, d in s]
    want = [_draw(x[r], np.float64(u[r]), np.float64(s32[r][0]), s32[r][1], np.float64(s32[r][2]),
                  np.float64(s32[r][3])) for r in range(rows)]
    assert got == want, [(r, a, b, s[r]) for r, (a, b) in enumerate(zip(got, want)) if a != b][:5]


@pytest.mark.parametrize("n", [128257, 151936, 400001])
def test_sample_rows_large_vocabulary(mq, torch, n):
    rng = random.Random(n)
    g = np.random.default_rng(n)
    rows = 10
    x = g.standard_normal((rows, n)).astype(np.float32) * 2.5
    x[5] = 0.25  # one value throughout: every token ties
    x[6] *= 1e-3
    s = [(1.0, 0, 1.0, 0.0), (0.8, 50, 0.95, 0.0), (1.0, 0, 0.9, 0.0), (1.0, 20000, 1.0, 0.0),
         (1.3, 0, 0.99, 0.01), (1.0, 0, 0.7, 0.0), (1.0, 0, 0.5, 0.0), (0.0, 0, 1.0, 0.0),
         (5.0, 0, 0.999, 0.0), (1.0, n - 1, 1.0, 0.0)]
    u = g.random(rows).astype(np.float32)
    f = lambda i, t=torch.float32: torch.tensor([v[i] for v in s], dtype=t, device="cuda")  # noqa: E731
    got = mq.sample_rows(torch.from_numpy(x).cuda(), torch.from_numpy(u).cuda(), temperature=f(0),
                         top_k=f(1, torch.int32), top_p=f(2), min_p=f(3)).tolist()
    want = [_draw(x[r], np.float64(u[r]), np.float64(np.float32(s[r][0])), s[r][1],
                  np.float64(np.float32(s[r][2])), np.float64(np.float32(s[r][3])))
            for r in range(rows)]
    assert got == want, [(r, a, b, s[r]) for r, (a, b) in enumerate(zip(got, want)) if a != b]


@pytest.mark.parametrize("n", [1500001, 4194304])
def test_sample_rows_longer_than_shared_memory(mq, torch, n):
    g = np.random.default_rng(n)
    x = g.standard_normal((5, n)).astype(np.float32) * 3
    x[1] = -1.5  # every token ties
    x[2, ::2] = -np.inf
    x[3] *= 1e-2
    s = [(1.0, 0, 0.9, 0.0), (1.0, 0, 0.6, 0.0), (0.7, 0, 1.0, 0.0), (1.0, n // 2, 0.999, 0.0),
         (1.0, 50, 0.95, 0.01)]
    u = g.random(5).astype(np.float32)
    f = lambda i, t=torch.float32: torch.tensor([v[i] for v in s], dtype=t, device="cuda")  # noqa: E731
    got = mq.sample_rows(torch.from_numpy(x).cuda(), torch.from_numpy(u).cuda(), temperature=f(0),
                         top_k=f(1, torch.int32), top_p=f(2), min_p=f(3)).tolist()
    want = [_draw(x[r], np.float64(u[r]), np.float64(np.float32(s[r][0])), s[r][1],
                  np.float64(np.float32(s[r][2])), np.float64(np.float32(s[r][3]))) for r in range(5)]
    assert got == want


def test_sample_rows_edges(mq, torch):
    x = torch.tensor([[1.0, 3.0, 3.0, -1.0], [float("inf"), 0.0, float("inf"), 5.0],
                      [float("-inf"), 2.0, 1.0, float("-inf")]], device="cuda")
    cu = lambda *v: torch.tensor(v, device="cuda")  # noqa: E731
    # no settings at all; a uniform at the ends and beyond, and NaN
    assert mq.sample_rows(x, cu(0.0, 0.75, 0.0)).tolist() == [0, 2, 1]
    assert mq.sample_rows(x, cu(1.0, 2.0, 1.0)).tolist() == [3, 2, 2]
    assert mq.sample_rows(x, cu(-1.0, float("nan"), -5.0)).tolist() == [0, 0, 1]
    # greedy rows take minq_argmax's token (total order: NaN above all, +0 above -0)
    y = torch.tensor([[1.0, float("nan"), 2.0], [-0.0, 0.0, -1.0]], device="cuda")
    got = mq.sample_rows(y, cu(0.5, 0.5), temperature=cu(0.0, -1.0)).tolist()
    assert got == [mq.argmax(y[0]), mq.argmax(y[1])]
    # a temperature that is not a number is greedy; an infinite one is uniform
    z = torch.tensor([[0.0, 5.0, 1.0, 2.0]] * 2, device="cuda")
    got = mq.sample_rows(z, cu(0.1, 0.1), temperature=cu(float("nan"), float("inf"))).tolist()
    assert got == [1, 0]
    # strided rows
    wide = torch.zeros(2, 10, device="cuda")
    wide[:, 1:5] = z
    wide[:, 5:] = 50.0
    assert mq.sample_rows(wide[:, 1:5], cu(0.5, 0.5), temperature=cu(0.0, 0.0)).tolist() == [1, 1]


def test_sample_rows_equals_the_sampler(mq, orc, torch):
    """The draws of Sampler.sample with the same uniforms (its sums are f32
    steps over at most 40 tokens: one draw in 64 may sit on a border)."""
    n, draws = 151936, 64
    g = np.random.default_rng(3)
    x = (g.random(n, dtype=np.float32) * 12).astype(np.float32)
    want = mq.Sampler(0.8, 40, 0.9, 77)
    one = [want.sample(x) for _ in range(draws)]
    u = (orc.Sampler(0.8, 40, 0.9, 77).rng_u32(draws) >> 8).astype(np.float32) * np.float32(2**-24)
    d = lambda v, t=torch.float32: torch.full((draws,), v, dtype=t, device="cuda")  # noqa: E731
    rows = torch.from_numpy(x).cuda().expand(draws, n).contiguous()
    got = mq.sample_rows(rows, torch.from_numpy(u).cuda(), temperature=d(0.8),
                         top_k=d(40, torch.int32), top_p=d(0.9)).tolist()
    assert sum(a != b for a, b in zip(got, one)) <= 1


# ---- a step ---------------------------------------------------------------------------------

def test_serving_steps_end_to_end(mq, torch):
    """Three requests through a prompt step and decode steps, one of them ending:
    tables, cache rows, attention and draws against the plain computation kept
    beside them; the decode step is one captured graph, replayed."""
    nh, nkv, hd, page, n_pages, width, vocab = 8, 2, 64, 16, 40, 12, 500
    R, scale = 3, 64 ** -0.5
    g = torch.Generator(device="cuda").manual_seed(0)
    kp, vp = mq.kv4_pool(n_pages, nkv, page, hd), mq.kv4_pool(n_pages, nkv, page, hd)
    book = Book(R, page, width, n_pages, 4)
    gpu = Pages(torch, book)
    head = torch.randn(nh * hd, vocab, generator=g, device="cuda") / 8
    past = [[[], []] for _ in range(R)]  # values as the cache stands for them

    def plain(new, k, v, q):
        at = 0
        rows = []
        for r, n in enumerate(new):
            for x, side in ((k, 0), (v, 1)):
                b = x[at:at + n].contiguous().cpu().numpy()
                past[r][side] += list(mq.dequantize_q4_0(mq.quantize_q4_0(b)).reshape(n, nkv, hd)) if n else []
            for i in range(n):
                m = len(past[r][0]) - n + i + 1
                K = np.stack(past[r][0][:m]).astype(np.float64).repeat(nh // nkv, 1)
                V = np.stack(past[r][1][:m]).astype(np.float64).repeat(nh // nkv, 1)
                z = (K * q[at + i].double().cpu().numpy()[None]).sum(-1) * scale
                p = np.exp(z - z.max(0))
                rows.append(((p / p.sum(0))[..., None] * V).sum(0))
            at += n
        return np.stack(rows)

    def step(new, T):
        k, v = (torch.randn(T, nkv, hd, generator=g, device="cuda") for _ in range(2))
        q = torch.randn(T, nh, hd, generator=g, device="cuda")
        return k, v, q

    new = [20, 1, 37]
    k, v, q = step(new, 60)
    s = mq.pages_extend(gpu.lens, dev(torch, new), gpu.table, gpu.free, gpu.n_free, page, 60)
    mq.kv4_write(k, v, s.slots, kp, vp)
    o = mq.kv4_attend(q, s.q_start, s.lens, gpu.table, kp, vp)
    book.extend(new)
    gpu.lens, gpu.n_free = s.lens, s.n_free
    gpu.same(book)
    want = plain(new, k, v, q)
    assert np.abs(o[:58].cpu().numpy() - want).max() <= 1e-5 * np.abs(want).max()
    # decode: one graph, replayed over new rows
    k, v, q = step(None, R)
    one = dev(torch, [1, 1, 1])
    u = torch.rand(R, generator=g, device="cuda")
    temp = torch.full((R,), 0.9, device="cuda")
    tk = dev(torch, [0, 20, 1])
    tp = torch.tensor([0.9, 1.0, 1.0], device="cuda")
    lens, n_free = gpu.lens.clone(), gpu.n_free.clone()
    bufs = mq.PageStep(lens, n_free, *(torch.empty(*a, device="cuda") for a in (
        (R + 1,), (R,), (R,), (2,))))
    bufs = mq.PageStep(lens, n_free, bufs.q_start.int(), bufs.slots.long(), bufs.positions.int(),
                       bufs.info.int())
    o = torch.empty(R, nh, hd, device="cuda")
    tok = torch.empty(R, dtype=torch.int32, device="cuda")

    def decode():
        mq.pages_extend(lens, one, gpu.table, gpu.free, n_free, page, R, out=bufs)
        mq.kv4_write(k, v, bufs.slots, kp, vp)
        mq.kv4_attend(q, bufs.q_start, bufs.lens, gpu.table, kp, vp, out=o)
        mq.sample_rows(o.reshape(R, -1) @ head, u, temperature=temp, top_k=tk, top_p=tp, out=tok)

    (o.reshape(R, -1) @ head)  # the library's handle exists before the capture
    keep = [t.clone() for t in (lens, n_free)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        decode()
    for t, c in zip((lens, n_free), keep):
        t.copy_(c)
    for _ in range(18):  # over a page's border
        for x, y in zip((k, v, q), step(None, R)):
            x.copy_(y)
        u.copy_(torch.rand(R, generator=g, device="cuda"))
        graph.replay()
        book.extend([1, 1, 1])
        gpu.lens, gpu.n_free = lens, n_free
        gpu.same(book)
        assert bufs.info.tolist() == [0, 0]
        want = plain([1, 1, 1], k, v, q)
        assert np.abs(o.cpu().numpy() - want).max() <= 1e-5 * np.abs(want).max()
        x = (o.reshape(R, -1) @ head).cpu().numpy()
        for r in range(R):
            assert int(tok[r]) == _draw(x[r], float(u[r]), float(np.float32(0.9)), int(tk[r]),
                                        float(tp[r]))
    # the second request ends
    cut = mq.pages_trim(lens, dev(torch, [99, 0, 99]), gpu.table, gpu.free, n_free, page)
    book.trim([99, 0, 99])
    gpu.lens, gpu.n_free = cut.lens, cut.n_free
    gpu.same(book)


def test_no_bounded_wait_gave_up(mq):
    """After all of the above: no kernel left a mark in the status words."""
    mq._lib.check(mq._lib.lib().minq_device_status())
