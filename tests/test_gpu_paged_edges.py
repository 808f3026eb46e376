"""The paged int8 KV cache operators where they can go wrong: warps whose lanes part, values that
are not finite or far from one another in size, padded batches.  Tolerances as in
test_gpu_paged.py unless a test derives its own."""
import pytest
import torch

import paged_ref as ref
import tabinfer_b200 as tb

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _ints(a):
    return torch.tensor(a, dtype=torch.int32, device="cuda")


def _evict(c, lens, w, budget, sinks, recent, choose=ref.evict):
    """An eviction into pools of its own, every output compared with the definition's."""
    keep = -(-budget // c.page)
    dst = [torch.full((c.B * keep, c.page, t.shape[-1]), 9, dtype=t.dtype, device="cuda")
           for t in (c.Kq, c.Ks, c.Vq, c.Vs)]
    fresh = torch.randperm(c.B * keep, generator=c.g).to(torch.int32).reshape(c.B, keep).contiguous()
    kept, new_lens, new_w = (t.cpu() for t in tb.kv_evict_paged_q8(
        c.dev(), c.table.cuda(), _ints(lens), w.cuda(), fresh.cuda(), budget, sinks, recent, c.nKv, c.hd, kv_out=dst))
    dst = [t.cpu().reshape(-1, t.shape[-1]) for t in dst]
    for b, n in enumerate(lens):
        want = choose(w[b], n, budget, sinks, recent)
        assert int(new_lens[b]) == len(want)
        assert kept[b].tolist() == want + [-1] * (budget - len(want))
        moved = w[b][:, want]
        assert torch.equal(new_w[b, :, :len(want)].nan_to_num(7.5), moved.nan_to_num(7.5))
        assert torch.equal(new_w[b, :, :len(want)].isnan(), moved.isnan())
        assert (new_w[b, :, len(want):] == 0).all()
        at = torch.arange(keep * c.page)
        to = fresh[b, at // c.page].long() * c.page + at % c.page
        rows = c.rows(b, torch.tensor(want, dtype=torch.long))
        for src, d in zip((c.Kq, c.Ks, c.Vq, c.Vs), dst):
            assert torch.equal(d[to[:len(want)]], src.reshape(-1, src.shape[-1])[rows])
            assert (d[to[len(want):]] == 9).all()


@pytest.mark.parametrize("n", [131072 + 16384 + 13, 17 * 1024 + 5])
def test_evict_lanes_with_other_counts(cuda, n):
    """rows beyond those in registers, the last warp's lanes with one more or one less of them"""
    c = ref.Cache(43, 1, -(-n // 256), 256, 1, 64, fill=False)
    w = torch.randn(1, 1, c.cap, generator=c.g).abs()
    _evict(c, [n], w, 900, 3, 7)
    _evict(c, [n], w.round(), 900, 0, 0)


@pytest.mark.parametrize("nHq,nKv,hd,page", [(16, 8, 128, 16), (8, 1, 64, 32), (4, 2, 64, 16), (2, 2, 128, 64)])
def test_decode_masks_of_many_tiles(cuda, nHq, nKv, hd, page):
    """another set of left-out keys in every tile (pages outside the pool here and there): a tile is
    read with its own mask"""
    n = 1500
    c = ref.Cache(44, 1, -(-n // page), page, nKv, hd)
    gone = torch.rand(c.table.shape[1], generator=c.g) < 0.4
    table = c.table.clone()
    table[0, gone] = -1
    q = torch.randn(1, nHq * hd, generator=c.g) * 1.5
    w = torch.zeros(1, nKv, c.cap, device="cuda")
    got = tb.attention_decode_paged_q8(q.cuda(), c.dev(), table.cuda(), _ints([n]), nHq, nKv, hd, weights=w).cpu()
    assert tb.default_context(0).device_error() == 0x6c01
    ok = ~gone.repeat_interleave(page)[:n]
    grp = nHq // nKv
    for h in range(nKv):
        k, v = c.head(0, n, h)
        total = torch.zeros(n, dtype=torch.float64)
        for g in range(grp):
            x = q.double().reshape(nHq, hd)[h * grp + g]
            p = torch.softmax(k[ok] @ x * hd ** -0.5, 0)
            total[ok] += p
            mag = float((k[ok].abs() @ x.abs()).max()) * hd ** -0.5
            rel = 2 * (hd + 8) * U * mag + (n + 16) * U
            err = (got.double().reshape(nHq, hd)[h * grp + g] - p @ v[ok]).abs().max()
            assert float(err) <= rel * float(v[ok].abs().max())
        assert (w[0, h, :n].cpu()[~ok] == 0).all()
        assert float((w[0, h, :n].cpu().double() - total).abs().max()) <= grp * rel + 4 * U * float(total.max())


def _prefill(c, q, ts, lens, nHq, window=0, sinks=0, tail=0):
    """(outputs f64 [T, nHq, hd], cu) of packed chunks; rows behind the last stay as they were"""
    cu = [sum(ts[:b]) for b in range(c.B + 1)]
    out = torch.full((cu[-1] + tail, nHq * c.hd), 7.0, dtype=torch.bfloat16, device="cuda")
    got = tb.attention_prefill_paged_q8(q.cuda(), c.dev(), c.table.cuda(), _ints(cu), _ints(lens), nHq, c.nKv, c.hd,
                                        window=window, sinks=sinks, out=out).cpu().double()
    assert (got[cu[-1]:] == 7).all()
    return got.reshape(-1, nHq, c.hd), cu


def _prefill_rows(c, q, ts, lens, nHq, window=0, sinks=0, tail=0):
    got, cu = _prefill(c, q, ts, lens, nHq, window, sinks, tail)
    for b, (n, t) in enumerate(zip(lens, ts)):
        for i in range(t):
            o, _, mag, big = ref.attend(c, b, q[cu[b] + i], n - t + i, nHq, window, sinks)
            tol = big * (2.0 ** -9 * mag + 2.0 ** -9) + 2.0 ** -8 * o.abs()
            assert ((got[cu[b] + i] - o).abs() <= tol).all(), (b, i)


@pytest.mark.parametrize("nHq,nKv,hd", [(2, 2, 128), (6, 3, 64), (4, 1, 128), (8, 1, 64)])
def test_prefill_rows_that_end_inside_a_warp(cuda, nHq, nKv, hd):
    """chunks of 1 to 9 and some 33 rows: a warp of rows with and without a query"""
    ts = [1, 2, 3, 5, 7, 9, 33, 17]
    lens = [t + 40 * (i % 3) for i, t in enumerate(ts)]
    c = ref.Cache(45, len(ts), 8, 16, nKv, hd)
    q = torch.randn(sum(ts) + 3, nHq * hd, generator=c.g) * 1.5
    _prefill_rows(c, q, ts, lens, nHq, tail=3)
    _prefill_rows(c, q, ts, lens, nHq, window=20, sinks=2, tail=3)


@pytest.mark.parametrize("hd,nKv,nHq", [(128, 2, 4), (64, 1, 4)])
@pytest.mark.parametrize("n,ts", [([300], [140]), ([6001, 90], [7, 60])])
@pytest.mark.parametrize("what", [float("inf"), float("nan")])
def test_prefill_rows_of_no_number_stay_with_those_who_see_them(cuda, hd, nKv, nHq, n, ts, what):
    """A scale of infinity or NaN in one 32-group of one key: queries before the key, or whose window has left
    it, are what they are without it; those that see V's have no number in the group's 32 dimensions alone;
    those that see K's have none in the heads that read it.  (Whole items, and items in parts.)"""
    window, sinks, grp, G = 90, 3, nHq // nKv, hd // 32 - 1
    c = ref.Cache(46, len(n), -(-max(n) // 16) + 1, 16, nKv, hd)
    q = torch.randn(sum(ts), nHq * hd, generator=c.g) * 1.5
    for b, w in ((0, 0), (0, window), (len(n) - 1, 0)):
        j = n[b] - ts[b] // 2 - 1 if w == 0 else n[b] - ts[b] - window // 2
        r = int(c.rows(b, j))
        for key in (False, True):
            pool = (c.Ks if key else c.Vs).view(-1, nKv, hd // 32)
            was = pool[r, 0, G].clone()
            pool[r, 0, G] = what
            got, cu = _prefill(c, q, ts, n, nHq, w, sinks)
            pool[r, 0, G] = was
            for s in range(len(n)):
                for i in range(ts[s]):
                    pos = n[s] - ts[s] + i
                    o, _, mag, big = ref.attend(c, s, q[cu[s] + i], pos, nHq, w, sinks)
                    tol = big * (2.0 ** -9 * mag + 2.0 ** -9) + 2.0 ** -8 * o.abs()
                    hit = torch.zeros(nHq, hd, dtype=torch.bool)
                    if s == b and bool(ref.seen(n[s], pos, w, sinks)[j]):
                        hit[:grp, slice(None) if key else slice(32 * G, 32 * G + 32)] = True
                    x = got[cu[s] + i]
                    assert not x[hit].isfinite().any(), (s, i)
                    assert ((x - o).abs() <= tol)[~hit].all(), (s, i)


def test_decode_rows_of_no_number(cuda):
    """the same of a new token: V's group alone, K's heads alone, and no trace of a row that is not seen"""
    nKv, hd, nHq, n = 2, 128, 4, 400
    c = ref.Cache(47, 1, 26, 16, nKv, hd)
    q = torch.randn(1, nHq * hd, generator=c.g) * 1.5
    o, _, mag, big = ref.attend(c, 0, q[0], n - 1, nHq, 200, 2)
    rel = 2 * (hd + 8) * U * mag + (n + 16) * U
    for j in (100, 300):
        r = int(c.rows(0, j))
        for key in (False, True):
            pool = (c.Ks if key else c.Vs).view(-1, nKv, hd // 32)
            was = pool[r, 0, 2].clone()
            pool[r, 0, 2] = float("inf")
            x = tb.attention_decode_paged_q8(q.cuda(), c.dev(), c.table.cuda(), _ints([n]), nHq, nKv, hd, window=200,
                                             sinks=2).cpu().double().reshape(nHq, hd)
            pool[r, 0, 2] = was
            hit = torch.zeros(nHq, hd, dtype=torch.bool)
            if j >= n - 200:
                hit[:2, slice(None) if key else slice(64, 96)] = True
            assert not x[hit].isfinite().any()
            assert float((x - o).abs()[~hit].max()) <= rel * big


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("bits", [0, 6, 10, 14, 15])
def test_prefill_scores_of_any_size(cuda, hd, bits):
    """Scores up to some 2^28, where the last bit of a score is larger than 1: the keys with the largest score
    share the weight.  Products and sums are exact: q = +-2^bits in one element of a head, K = byte / 128 *
    2^bits in it, with bytes 10 apart; V's bytes are exact in f16.  (Tolerance as in the test of rising scores:
    P's and a part's 2^-11 each, f32, the output's bf16.)"""
    n, t, nKv, nHq = 700, 130, 1, 2
    c = ref.Cache(56, 1, 45, 16, nKv, hd)
    c.Kq[:] = 0
    c.Ks[:] = 127.0 / 128 * 2.0 ** bits
    c.Vs[:] = 127.0 / 64
    rows = c.rows(0, torch.arange(n))
    place = torch.randperm(n, generator=c.g)
    q = torch.zeros(t, nHq, hd)
    q[:, 0, 0], q[:, 1, 0] = 2.0 ** bits, -2.0 ** bits
    order = torch.randint(-11, 11, (n,), generator=c.g)
    order[place[:2]] = torch.tensor([12, -12])                      # the largest for either head
    c.Kq.view(-1, hd)[rows, 0] = (order * 10).to(torch.int8)
    got, _ = _prefill(c, q.reshape(t, -1), [t], [n], nHq)
    for i in list(range(0, t, 9)) + [t - 1]:
        o, _, _, big = ref.attend(c, 0, q[i].reshape(-1), n - t + i, nHq)
        assert ((got[i] - o).abs() <= 2.0 ** -8 * o.abs() + big * (2.0 ** -10 + 2.0 ** -14)).all(), (bits, i)


@pytest.mark.parametrize("hd,nKv,nHq", [(64, 2, 4), (128, 1, 2)])
@pytest.mark.parametrize("kscale", [1.0, 1e-7, 1e8])
@pytest.mark.parametrize("vscale", [1e-11, 1e-7, 1e-4, 1.0, 1e4, 1e9, 1e30])
def test_prefill_of_small_and_large_numbers(cuda, hd, nKv, nHq, kscale, vscale):
    """K and V of any size (and q of the size that keeps the scores): errors relative to what is seen"""
    ts, lens = [20, 150], [700, 150]
    c = ref.Cache(52, 2, 45, 16, nKv, hd)
    c.Ks *= kscale
    c.Vs *= vscale
    q = torch.randn(sum(ts), nHq * hd, generator=c.g) * (1.5 / kscale)
    got, cu = _prefill(c, q, ts, lens, nHq)
    for b, (n, t) in enumerate(zip(lens, ts)):
        for i in range(0, t, 7):
            o, _, mag, big = ref.attend(c, b, q[cu[b] + i], n - t + i, nHq)
            tol = big * (2.0 ** -9 * mag + 2.0 ** -9) + 2.0 ** -8 * o.abs()
            assert ((got[cu[b] + i] - o).abs() <= tol).all(), (b, i)
            assert float((got[cu[b] + i] - o).norm() / o.norm()) < 2.0 ** -7


@pytest.mark.parametrize("hd,nKv,nHq", [(64, 1, 4), (128, 2, 4)])
@pytest.mark.parametrize("slope", [-0.2, 0.2])
@pytest.mark.parametrize("window,sinks", [(0, 0), (60, 3)])
def test_prefill_of_numbers_that_grow_along_the_cache(cuda, hd, nKv, nHq, slope, window, sinks):
    """V's size changes by 2^slope from row to row, in all by 2^120: a query's output is right relative to
    the rows that it sees, whatever the others hold"""
    ts, lens = [4, 300], [601, 300]
    c = ref.Cache(53, 2, 40, 16, nKv, hd)
    for b, n in enumerate(lens):
        size = 2.0 ** torch.clamp(slope * (torch.arange(n) - n // 2), -38, 60).float()
        c.Vs.view(-1, nKv * hd // 32)[c.rows(b, torch.arange(n))] *= size[:, None]
    q = torch.randn(sum(ts), nHq * hd, generator=c.g) * 1.5
    got, cu = _prefill(c, q, ts, lens, nHq, window, sinks)
    for b, (n, t) in enumerate(zip(lens, ts)):
        for i in range(0, t, 5 if t > 9 else 1):
            o, _, mag, big = ref.attend(c, b, q[cu[b] + i], n - t + i, nHq, window, sinks)
            tol = big * (2.0 ** -9 * mag + 2.0 ** -9) + 2.0 ** -8 * o.abs()
            assert ((got[cu[b] + i] - o).abs() <= tol).all(), (b, i)


@pytest.mark.parametrize("hd", [64, 128])
def test_prefill_rows_of_q_of_any_size(cuda, hd):
    """a query's size is its own: tiny, huge and ordinary ones side by side"""
    nKv, nHq, t = 2, 8, 40
    c = ref.Cache(54, 1, 10, 16, nKv, hd)
    size = 10.0 ** torch.randint(-12, 13, (t, nHq, 1), generator=c.g).float()
    q = (torch.randn(t, nHq, hd, generator=c.g) * size).reshape(t, nHq * hd)
    got, _ = _prefill(c, q, [t], [150], nHq)
    for i in range(t):
        for h in range(nHq):
            one = q[i].clone().view(nHq, hd)
            one[torch.arange(nHq) != h] = 0
            o, _, mag, big = ref.attend(c, 0, one.view(-1), 150 - t + i, nHq)
            # where the scores are large the best key's lead decides, and a rounding of them may be more than it
            if mag < 100:
                tol = big * (2.0 ** -9 * mag + 2.0 ** -9) + 2.0 ** -8 * o[h].abs()
                assert ((got[i, h] - o[h]).abs() <= tol).all(), (i, h)
            assert got[i, h].isfinite().all() and float(got[i, h].abs().max()) <= big * (1 + 2.0 ** -7)


@pytest.mark.parametrize("hd", [64, 128])
def test_prefill_small_outputs_of_parts(cuda, hd):
    """V = +-1 that all but cancels (one key more of one sign): an item in parts keeps the small output's digits.
    All scores are zero, so weights and products are exact and sums of them too; what is left is 1/l and the
    join (f32, 2^-20 of the parts' outputs, which are at most 2^-8 here) and bf16's 2^-8 (twice the half step)."""
    n, t, nHq = 4097, 2, 2
    c = ref.Cache(50, 1, n // 32 + 1, 32, 1, hd)
    c.Kq[:] = 0
    c.Vs[:] = 127.0
    sign = torch.ones(c.cap, dtype=torch.int8)
    sign[1::2] = -1
    c.Vq.view(-1, hd)[c.rows(0, torch.arange(c.cap))] = sign[:, None]
    q = torch.randn(t, nHq * hd, generator=c.g)
    got, _ = _prefill(c, q, [t], [n], nHq)
    o = ref.attend(c, 0, q[1], n - 1, nHq)[0]
    assert torch.allclose(o, torch.full_like(o, 1.0 / n), rtol=1e-9)
    assert float((got[1] / o - 1).abs().max()) <= 2.0 ** -7


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n,t", [(8193, 3), (300, 290)])
@pytest.mark.parametrize("gap", [6.0, 14.0, 20.0, 22.0, 24.5])
def test_prefill_light_weights_beside_a_heavy_one(cuda, hd, n, t, gap):
    """One first key with nearly all of the weight and V = 0, so the output is what the light keys, 2^-gap of
    it each, give.  q and K's elements are multiples of 1/64 below 16 and exact in f16, V's are too, so what is
    left is a weight's rounding: 2^-11 of itself where 2^(8 - gap) is normal in f16, and 2^-25 of 2^(8 - gap)
    below (the exponential 2^-22); a part's output 2^-11, bf16 2^-8 (twice the half steps)."""
    nKv, nHq, page = 1, 2, 16
    c = ref.Cache(49, 1, n // page + 1, page, nKv, hd)
    c.Ks[:] = 127.0 / 64
    c.Vs[:] = 127.0 / 64
    c.Kq[:] = 0
    c.Vq[:] = (torch.arange(c.Vq.numel()).view(c.Vq.shape) % 50 + 60).to(torch.int8)
    first = int(c.rows(0, 0))
    c.Vq.view(-1, hd)[first] = 0
    # score of the first key: 16 x k q_0 / sqrt(hd) = gap ln 2, to the nearest step of q in 1/64
    c.Kq.view(-1, hd)[first, :16] = 64
    q = torch.zeros(t, nHq * hd)
    q.view(t, nHq, hd)[:, :, :16] = round(gap * 0.6931471805599453 * hd ** 0.5 / 16 * 64) / 64
    got, _ = _prefill(c, q, [t], [n], nHq)
    for i in sorted({1, t // 2, t - 1}):
        o, _, _, _ = ref.attend(c, 0, q[i], n - t + i, nHq)
        x = float(q[i, 0]) * 16 * hd ** -0.5 / 0.6931471805599453        # the gap as it is
        tol = 2.0 ** -8 + 2.0 ** -10 + 2.0 ** -11 + max(0.0, 2.0 ** (x - 33))
        assert float(((got[i] - o) / o).abs().max()) <= tol, i


def test_decode_weights_of_no_number(cuda):
    """a sequence whose scores hold no number (a query's NaN, a key's scale) has no weights either: every row
    it sees becomes NaN, those outside its window and the other sequences' stay numbers"""
    nKv, hd, nHq, lens, window, sinks = 2, 64, 4, [300, 77, 120], 100, 2
    c = ref.Cache(48, 3, 20, 16, nKv, hd)
    c.Ks.view(-1, nKv, 2)[int(c.rows(1, 40)), 0, 1] = float("nan")
    q = torch.randn(3, nHq * hd, generator=c.g)
    q.view(3, nHq, hd)[0, 1, 5] = float("nan")
    w = torch.ones(3, nKv, c.cap, device="cuda")
    tb.attention_decode_paged_q8(q.cuda(), c.dev(), c.table.cuda(), _ints(lens), nHq, nKv, hd, window=window,
                                 sinks=sinks, weights=w)
    for b, n in enumerate(lens):
        ok = torch.zeros(c.cap, dtype=torch.bool)
        ok[:n] = ref.seen(n, n - 1, window, sinks)
        none = torch.zeros(nKv, c.cap, dtype=torch.bool)
        if b < 2:
            none[0] = ok
        assert torch.equal(w[b].cpu().isnan(), none), b
        assert (w[b].cpu()[:, ~ok] == 1).all()


@pytest.mark.parametrize("hd,T", [(128, 3), (64, 3), (128, 900)])
def test_prep_keeps_what_is_not_a_number(cuda, hd, T):
    """NaN in v: its 32-group's scale is NaN, so that every reader meets it; infinity in v: an infinite scale;
    NaN in k: the head has no number after its norm, and every scale of it is NaN; infinity in k: x / sqrt(mean
    x^2) is inf / inf in its place, so the rotation makes it and its partner hd / 2 away NaN, and 0 elsewhere.
    Other groups, heads and rows are what they are without it."""
    nKv, nHq, page = 3, 3, 16
    c = ref.Cache(55, 1, T // page + 1, page, nKv, hd, fill=False)
    g = torch.Generator().manual_seed(7)
    q, k, v = (torch.randn(T, 3 * hd, generator=g) for _ in range(3))
    w = torch.ones(hd, dtype=torch.float16, device="cuda")
    at = torch.arange(T, dtype=torch.int32).cuda()

    def run(k, v):
        kv = c.dev()
        tb.attn_prep_paged_q8(q.cuda(), k.cuda(), v.cuda(), w, w, kv, c.table.cuda(), torch.zeros_like(at), at, at, nHq,
                              nKv, hd, 1e6, 1e-6)
        r = c.rows(0, torch.arange(T))
        return [t.cpu().view(-1, nKv, t.shape[-1] // nKv)[r] for t in kv]
    clean = run(k, v)
    k2, v2 = k.clone(), v.clone()
    v2.view(T, nKv, hd)[1, 0, 40] = float("nan")
    v2.view(T, nKv, hd)[T - 1, 2, 3] = float("-inf")
    k2.view(T, nKv, hd)[0, 1, 5] = float("nan")
    k2.view(T, nKv, hd)[T - 1, 0, 33] = float("inf")
    Kq, Ks, Vq, Vs = run(k2, v2)
    Kn = torch.zeros(T, nKv, hd // 32, dtype=torch.bool)
    Kn[0, 1] = True
    Kn[T - 1, 0, 1] = Kn[T - 1, 0, (33 + hd // 2) % hd // 32] = True
    assert torch.equal(Ks.isnan(), Kn)
    rest = ~Kn[T - 1, 0]
    assert (Ks[T - 1, 0][rest] == 1e-12).all() and (Kq[T - 1, 0][rest.repeat_interleave(32)] == 0).all()
    Kn[T - 1, 0] = True
    Vn = torch.zeros(T, nKv, hd // 32, dtype=torch.bool)
    Vn[1, 0, 1] = True
    assert torch.equal(Vs.isnan(), Vn) and Vs[T - 1, 2, 0] == float("inf") and int(Vs.isinf().sum()) == 1
    Vn[T - 1, 2, 0] = True
    for bad, now, was in ((Kn, (Kq, Ks), clean[:2]), (Vn, (Vq, Vs), clean[2:])):
        assert torch.equal(now[1][~bad], was[1][~bad])
        ok = ~bad.repeat_interleave(32, 2)
        assert torch.equal(now[0][ok], was[0][ok])


def test_prep_refuses_norm_weights_of_other_types(cuda):
    """bf16 has as many bits as f16 and another meaning"""
    c = ref.Cache(81, 2, 4, 16, 2, 64)
    kv, table = c.dev(), c.table.cuda()
    q = torch.randn(2, 256, device="cuda")
    w, i = torch.ones(64, dtype=torch.float16, device="cuda"), _ints([0, 1])
    kr = q[:, :128].contiguous()

    def prep(qw, kw):
        return tb.attn_prep_paged_q8(q, kr, kr, qw, kw, kv, table, i, i, i, 4, 2, 64, 1e6, 1e-6)
    want = prep(w, w)
    assert torch.equal(prep(w.view(torch.int16), w.view(torch.uint16)), want)      # the patterns of f16
    for a, b in ((w.bfloat16(), w), (w, w.bfloat16()), (w.float(), w), (w, w.float())):
        with pytest.raises(tb.TabInferError):
            prep(a, b)


def test_evict_refuses_a_budget_before_it_allocates(cuda):
    c = ref.Cache(82, 2, 4, 16, 2, 64)
    kv, weights = c.dev(), torch.zeros(2, 2, 64, device="cuda")
    for budget in (17, 1 << 31, 1 << 45):
        with pytest.raises(tb.TabInferError):
            tb.kv_evict_paged_q8(kv, c.table.cuda(), _ints([10, 20]), weights, _ints([[8], [9]]), budget, 2, 3, 2, 64)
    assert torch.cuda.memory_allocated() < 1 << 30


def _choose(w, n, budget, sinks, recent):
    """ref.evict where scores may be NaN: those come before every number, the lower row first"""
    if n <= budget:
        return list(range(n))
    score = w.double().sum(0)
    rank = [(0, 0.0, j) if score[j].isnan() else (1, -float(score[j]), j) for j in range(sinks, n - recent)]
    mid = [r[2] for r in sorted(rank)][:budget - sinks - recent]
    return sorted(list(range(sinks)) + mid + list(range(n - recent, n)))


@pytest.mark.parametrize("nKv,hd,lens,budget,page", [(2, 64, [300, 90, 40], 50, 16), (8, 128, [700, 1100], 300, 32),
                                                      (8, 128, [20000], 5000, 256), (3, 64, [2500], 40, 16)])
@pytest.mark.parametrize("few", [True, False])
def test_evict_weights_of_no_number(cuda, nKv, hd, lens, budget, page, few):
    """NaN of either sign, and NaN that is infinity less infinity over the heads, count as the largest score,
    beside infinities; few of them, or more than the budget holds"""
    c = ref.Cache(57, len(lens), -(-max(lens) // page), page, nKv, hd)
    w = torch.exp(2 * torch.randn(c.B, nKv, c.cap, generator=c.g))
    step = 29 if few else 3
    w[:, 0, 1::step] = float("nan")
    w[:, 1, 5::step] = -float("nan")
    w[:, 0, 9::step], w[:, 1, 9::step] = float("inf"), float("-inf")
    w[:, 1, 2::17] = float("inf")
    _evict(c, lens, w, budget, 3, 6, _choose)


def test_evict_more_heads_than_ctas(cuda):
    """more (sequence, kv head) pairs than CTAs copy weights, and more kept rows than warps"""
    B = 170
    lens = [1 + (37 * b) % 96 for b in range(B)]
    c = ref.Cache(58, B, 6, 16, 8, 128)
    w = torch.rand(B, 8, c.cap, generator=c.g)
    _evict(c, lens, w, 33, 2, 5)
