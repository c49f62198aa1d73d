"""Serving-step operators where they had failed: ranges of sizes, borders and
inputs on which a call was refused, answered wrongly or read too early."""
import numpy as np
import pytest

from test_gpu_serving import _check, _draw, _fill, _reference, dev, torch  # noqa: F401

pytestmark = pytest.mark.gpu


# ---- page tables ----------------------------------------------------------------

@pytest.mark.parametrize("bad", [-1, 24, 2**31 - 1, -2**31])
def test_extend_into_a_page_outside_the_pool_changes_nothing(mq, torch, bad):
    """New tokens that go on in a partly filled page whose id is bad: the step is
    refused (their keys and values would be lost). A bad id that no new token
    reaches is none of the step's."""
    def state():
        return (dev(torch, [20, 32, 5, 0]),
                dev(torch, [[3, 4, -1, -1], [bad, 6, -1, -1], [8, -1, -1, -1], [-1] * 4]),
                dev(torch, [0, 1, 2, 10, 11, 12] + [-1] * 18), dev(torch, [6]))
    for n, r in ((1, 0), (12, 0), (13, 2), (1, 2)):
        lens, table, free, n_free = state()
        table[r, int(lens[r]) // 16] = bad
        new = [1, 1, 0, 3]
        new[r] = n
        before = [t.clone() for t in (lens, table, free, n_free)]
        s = mq.pages_extend(lens, dev(torch, new), table, free, n_free, 16, 30)
        assert s.info.tolist() == [mq.PAGES_BAD_PAGE, 0]
        assert all(torch.equal(a, b) for a, b in zip(before, (lens, table, free, n_free)))
        assert torch.equal(s.lens, lens) and torch.equal(s.n_free, n_free)
        assert (s.slots == -1).all() and s.q_start.tolist() == [0] * 5
        new[r] = 0  # the others' tokens alone
        s = mq.pages_extend(lens, dev(torch, new), table, free, n_free, 16, 30)
        assert s.info.tolist() == [0, 0] and (s.slots[:sum(new)] >= 0).all()
    # full pages before the new tokens are not looked at
    lens, table, free, n_free = state()
    s = mq.pages_extend(lens, dev(torch, [0, 2, 0, 0]), table, free, n_free, 16, 2)
    assert s.info.tolist() == [0, 0] and s.slots.tolist() == [12 * 16, 12 * 16 + 1]


# ---- attention ------------------------------------------------------------------

@pytest.mark.parametrize("nh,nkv,hd", [(8, 2, 64), (8, 2, 128), (4, 2, 96), (4, 1, 32)])
@pytest.mark.parametrize("T,starts,rows", [
    (6, [-2, 1, 99], []), (6, [-1, 6, 7], []), (6, [0, 3, 99], [0, 1, 2]), (6, [5, 2, 4], [2, 3]),
    (200, [-2, 100, 999], []), (200, [0, 100, 201], range(100)), (200, [-90, 100, 200], range(100, 200)),
])
def test_attend_requests_outside_the_tokens_have_none(mq, torch, nh, nkv, hd, T, starts, rows):
    """A request whose run of tokens is not inside them is left out as a whole,
    by every kernel alike; its rows stay as they were."""
    lens, page = [120, 130], 16
    kp, vp, table, kv, vv = _fill(mq, torch, 2, lens, nkv, hd, page)
    q = torch.randn(T, nh, hd, device="cuda")
    out = torch.full((T, nh, hd), 3.0, device="cuda")
    mq.kv4_attend(q, dev(torch, starts), dev(torch, lens), table, kp, vp, out=out)
    on = torch.zeros(T, dtype=torch.bool, device="cuda")
    on[list(rows)] = True
    assert (out[~on] == 3.0).all()
    valid = [r for r in range(2) if 0 <= starts[r] < starts[r + 1] <= T]
    for r in valid:
        want, tol = _reference(torch, q, [starts[r], starts[r + 1]], [lens[r]], table[r:r + 1], page,
                               kv, vv, hd ** -0.5)
        _check(torch, out[starts[r]:starts[r + 1]], want[starts[r]:starts[r + 1]],
               tol[starts[r]:starts[r + 1]])


@pytest.mark.parametrize("nh,nkv,hd", [(8, 2, 64), (8, 2, 128), (4, 2, 96), (4, 1, 32), (2, 1, 256)])
@pytest.mark.parametrize("lens,new", [([1, 40], [1, 1]), ([70, 300], [2, 1]), ([130, 90], [100, 70])])
def test_attend_keeps_what_is_not_a_number(mq, torch, nh, nkv, hd, lens, new):
    """A query row that holds NaN gives NaN, not the zeros of a row that sees
    nothing; so do keys whose scales are NaN. Other rows do not notice."""
    page = 16
    kp, vp, table, kv, vv = _fill(mq, torch, 7, lens, nkv, hd, page)
    start = [0, new[0], sum(new)]
    q = torch.randn(start[-1], nh, hd, device="cuda")
    args = (dev(torch, start), dev(torch, lens), table, kp, vp)
    clean = mq.kv4_attend(q, *args)
    assert torch.isfinite(clean).all()
    bad = q.clone()
    bad[0, 1, hd // 2] = float("nan")
    bad[start[-1] - 1, 0] = float("nan")
    got = mq.kv4_attend(bad, *args)
    hit = torch.zeros_like(got, dtype=torch.bool)
    hit[0, 1], hit[start[-1] - 1, 0] = True, True
    assert torch.isnan(got[hit]).all()
    want, tol = _reference(torch, q, start, lens, table, page, kv, vv, hd ** -0.5)
    want[hit.any(-1).any(-1)] = float("nan")  # (their other heads: below)
    _check(torch, torch.where(hit, 0.0, got), want, tol)
    assert torch.isfinite(got[~hit]).all()
    # every key of request 0
    blocks = kp.view(kp.shape[0], nkv, page, hd // 32, 20)
    blocks[table[0, :-(-lens[0] // page)].long(), :, :, 0, :4] = torch.tensor(
        [float("nan")], device="cuda").view(torch.uint8)
    got = mq.kv4_attend(q, *args)
    assert torch.isnan(got[:start[1]]).all() and torch.isfinite(got[start[1]:]).all()


@pytest.mark.parametrize("nh,nkv,hd,new", [(8, 2, 64, 1), (8, 2, 128, 3), (16, 1, 128, 1), (8, 2, 128, 70),
                                           (4, 2, 96, 2)])
@pytest.mark.parametrize("kg,qg,vg", [(1.0, 1.0, 1e-17), (1.0, 1.0, 1e28), (1e-20, 1e20, 1.0),
                                      (1e18, 1e-18, 1e-10), (1e-30, 1.0, 1.0)])
def test_attend_over_the_range_of_sizes(mq, torch, nh, nkv, hd, new, kg, qg, vg):
    """Keys, queries and values far from 1: the bound is relative to them."""
    lens, page = [90, 700], 16
    kp, vp, table, kv, vv = _fill(mq, torch, 5, lens, nkv, hd, page)
    every = torch.arange(kv.shape[0], device="cuda")
    mq.kv4_write((kv * kg).float(), (vv * vg).float(), every, kp, vp)
    k, v = mq.kv4_read(every, kp, vp)
    start = [0, new, 2 * new]
    q = torch.randn(2 * new, nh, hd, device="cuda") * qg
    got = mq.kv4_attend(q, dev(torch, start), dev(torch, lens), table, kp, vp)
    want, tol = _reference(torch, q, start, lens, table, page, k.double(), v.double(), hd ** -0.5)
    _check(torch, got / vg, want / vg, tol / vg)


@pytest.mark.parametrize("nh,nkv,hd", [(32, 8, 128), (14, 2, 64)])
@pytest.mark.parametrize("page", [16, 64])
def test_attend_chunks_whose_maximum_moves_within_a_tile(mq, torch, nh, nkv, hd, page):
    """Scores that grow in steps of 6 to 40 log2 units at every step of 16 columns
    of a tile (the columns' positions are 2 x, 2 x + 1 mod 8), in some tiles over
    several tiles: the weights stored before are read back and scaled each time."""
    lens, new = [515, 200], [70, 130]
    kp, vp, table, kv, vv = _fill(mq, torch, 4, lens, nkv, hd, page)
    n_pages = kp.shape[0]
    g = torch.Generator(device="cuda").manual_seed(2)
    u = torch.nn.functional.normalize(torch.randn(nkv, hd, generator=g, device="cuda"), dim=-1)
    pos = torch.zeros(n_pages * page, device="cuda")  # position of a slot
    for r, n in enumerate(lens):
        i = torch.arange(n, device="cuda")
        pos[table[r].long()[i // page] * page + i % page] = i.float()
    step, tile = (pos.int() % 8) // 2, pos.int() // 64
    rise = torch.tensor([6.0, 11.0, 40.0], device="cuda")[tile.long() % 3]
    level = (step * rise + torch.where(tile % 4 == 3, 130.0, 0.0) + 0.3 * torch.randn(
        pos.shape, generator=g, device="cuda")) * 0.6931472 + torch.where(tile % 2 == 1, -20.0, 0.0)
    k = (level[:, None, None] * u).contiguous()
    mq.kv4_write(k, k, torch.arange(n_pages * page, device="cuda"), kp, mq.kv4_pool(*kp.shape[:3], hd))
    kv = mq.kv4_read(torch.arange(n_pages * page, device="cuda"), kp, vp)[0].double()
    start = [0, new[0], sum(new)]
    q = u.repeat_interleave(nh // nkv, 0)[None] * (1 + 0.1 * torch.rand(
        start[-1], nh, 1, generator=g, device="cuda"))
    q = q.contiguous()
    got = mq.kv4_attend(q, dev(torch, start), dev(torch, lens), table, kp, vp, scale=1.0)
    want, tol = _reference(torch, q, start, lens, table, page, kv, vv, 1.0)
    _check(torch, got, want, tol)
    assert torch.equal(got, mq.kv4_attend(q, dev(torch, start), dev(torch, lens), table, kp, vp, scale=1.0))


@pytest.mark.parametrize("nh,nkv,hd", [(16, 4, 128), (8, 2, 64)])
def test_attend_chunks_of_every_number_of_tiles(mq, torch, nh, nkv, hd):
    """Chunks of one to thirteen tiles one behind the other in a CTA: the places of
    scores, weights, outputs and their barriers' phases go on from item to item."""
    page = 32
    lens = [64 * t + d for t in range(1, 14) for d in (-3, 0, 17)]
    new = [61 if n < 64 else 64 for n in lens]
    kp, vp, table, kv, vv = _fill(mq, torch, 11, lens, nkv, hd, page)
    start = [0] + np.cumsum(new).tolist()
    q = torch.randn(start[-1], nh, hd, device="cuda")
    args = (q, dev(torch, start), dev(torch, lens), table, kp, vp)
    got = mq.kv4_attend(*args)
    want, tol = _reference(torch, q, start, lens, table, page, kv, vv, hd ** -0.5)
    _check(torch, got, want, tol)
    assert all(torch.equal(got, mq.kv4_attend(*args)) for _ in range(20))


@pytest.mark.parametrize("nh,nkv,hd", [(16, 4, 64), (8, 2, 128)])
@pytest.mark.parametrize("qs,qo,os_,oo", [(1, 1, 1, 3), (0, 0, 2, 0), (3, 0, 0, 2)])
def test_attend_chunk_rows_off_sixteen_bytes(mq, torch, nh, nkv, hd, qs, qo, os_, oo):
    """Queries and outputs of a chunk whose rows do not start on 16 bytes, whole
    items and pieces of one alike; nothing beside the rows is touched."""
    page, lens, new = 32, [100, 9000, 64], [70, 65, 1]
    start = [0] + np.cumsum(new).tolist()
    T, w = start[-1], nh * hd
    kp, vp, table, kv, vv = _fill(mq, torch, 4, lens, nkv, hd, page)
    base = torch.randn(T * (w + qs) + 8, device="cuda")
    q = torch.as_strided(base, (T, nh, hd), (w + qs, hd, 1), qo)
    room = torch.full((T * (w + 64 + os_) + 8,), 9.0, device="cuda")
    out = torch.as_strided(room, (T, nh, hd), (w + 64 + os_, hd, 1), oo)
    mq.kv4_attend(q, dev(torch, start), dev(torch, lens), table, kp, vp, out=out)
    want, tol = _reference(torch, q, start, lens, table, page, kv, vv, hd ** -0.5)
    _check(torch, out, want, tol)
    gaps = torch.as_strided(room, (T, 64 + os_), (w + 64 + os_, 1), oo + w)
    assert (gaps == 9.0).all() and (room[:oo] == 9.0).all()


# ---- sampling -------------------------------------------------------------------

def _rows(mq, torch, x, u, s):
    f = lambda i, t=torch.float32: torch.tensor([v[i] for v in s], dtype=t, device="cuda")  # noqa: E731
    got = mq.sample_rows(torch.from_numpy(x).cuda(), torch.from_numpy(u).cuda(), temperature=f(0),
                         top_k=f(1, torch.int32), top_p=f(2), min_p=f(3)).tolist()
    want = [_draw(x[r], np.float64(u[r]), np.float64(np.float32(s[r][0])), s[r][1],
                  np.float64(np.float32(s[r][2])), np.float64(np.float32(s[r][3])))
            for r in range(len(s))]
    assert got == want, [(r, a, b, s[r]) for r, (a, b) in enumerate(zip(got, want)) if a != b]


@pytest.mark.parametrize("n", [390784, 390785, 393184, 393185])
def test_sample_rows_around_what_shared_memory_holds(mq, torch, n):
    """The longest rows that eight CTAs hold in shared memory, and the next ones."""
    g = np.random.default_rng(n)
    s = [(1.0, 0, 1.0, 0.0), (0.8, 50, 0.95, 0.0), (1.2, 0, 0.9, 0.0), (0.0, 0, 1.0, 0.0),
         (1.0, 3000, 1.0, 0.01)]
    x = g.standard_normal((len(s), n)).astype(np.float32) * 2.5
    x[3, -1] = 40.0  # the greedy row's token is its last
    _rows(mq, torch, x, g.random(len(s)).astype(np.float32), s)


@pytest.mark.parametrize("n", [2, 100, 5000, 151936, 400001])
@pytest.mark.parametrize("low", [-1e9, float(np.finfo(np.float32).min)])
def test_sample_rows_never_draws_a_masked_token(mq, torch, n, low):
    """A uniform of 0 takes the first token that weighs anything: masks of a very
    low value count like -infinity, small weights do not."""
    g = np.random.default_rng(n)
    x = np.clip(g.standard_normal((4, n)), -4, 4).astype(np.float32)
    x[0, :n // 2] = low
    x[1] = low           # masks alone: they all weigh the same
    x[2, :-1] = low
    x[3, 0] = -200.0     # exp(-200) is a weight
    u = np.zeros(4, np.float32)
    _rows(mq, torch, x, u, [(1.0, 0, 1.0, 0.0)] * 4)
    # at the lowest temperature: what a double still holds, and what it does not
    y = np.full((2, n), 3.0, np.float32)
    y[0, 0], y[1, 0] = 3.0 - 0.3 * 740, 3.0 - 0.3 * 750
    _rows(mq, torch, y, u[:2], [(0.3, 0, 1.0, 0.0)] * 2)
