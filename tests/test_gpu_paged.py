"""Paged int8 KV cache operators (attn_prep_paged_q8, attention_decode_paged_q8,
attention_prefill_paged_q8, kv_evict_paged_q8) against plain 64-bit forms (paged_ref.py).

Tolerances.  u = 2^-24.  Decode: a score is a sum of hd exact or once-rounded products in
f32, so it is off by at most (hd + 8) u sum|q_i k_i| / sqrt(hd) =: d; every weight is then
off by at most a factor 1 + 2 d + (S + 16) u, and an output by that times the largest |v|
seen.  Prefill: q, a key's scale and their product with its byte are rounded to f16 (2^-11
each), which could put a score off by 1.5 * 2^-10 of sum|q_i k_i| / sqrt(hd) if every rounding
of a sum had the same sign; d := 2^-10 of it is asked for.  A weight is then off by a factor
1 + 2 d; p, v (scale and product) and a joined part's output add 2^-11 each, 2^-9 of the
largest |v| together, and the bf16 output 2^-8 of itself.  The sums are taken from the
reference.  Prep: rows formed in 64 bits, so bytes and scales are
those of the reference and qr is within half a step of f32."""
import pytest
import torch

import paged_ref as ref
import tabinfer_b200 as tb

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _ints(a):
    return torch.tensor(a, dtype=torch.int32, device="cuda")


def _decode_check(c, lens, nHq, window=0, sinks=0, weights=False, seed=1, kv=None, out=None):
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(c.B, nHq * c.hd, generator=g) * 1.5
    acc = torch.rand(c.B, c.nKv, c.cap, generator=g) if weights else None
    ad = acc.cuda() if weights else None
    got = tb.attention_decode_paged_q8(q.cuda(), kv or c.dev(), c.table.cuda(), _ints(lens), nHq, c.nKv, c.hd,
                                       window=window, sinks=sinks, weights=ad, out=out).cpu().double()
    for b, n in enumerate(lens):
        o, w, mag, big = ref.attend(c, b, q[b], n - 1, nHq, window, sinks)
        rel = 2 * (c.hd + 8) * U * mag + (n + 16) * U
        err = (got[b].reshape(nHq, c.hd) - o).abs().max()
        assert float(err) <= rel * big, (b, n, float(err), rel * big)
        if weights:
            want = acc[b].double()
            want[:, :max(n, 0)] += w
            werr = (ad[b].cpu().double() - want).abs().max()
            assert float(werr) <= (nHq // c.nKv) * rel + 4 * U * float(want.max()), (b, n, float(werr))
    return got


@pytest.mark.parametrize("nHq,nKv,hd,page,lens,window,sinks", [
    (16, 8, 128, 64, [1], 0, 0),
    (16, 8, 128, 16, [0, 1, 2, 31, 32, 33, 127, 128, 129, 160], 0, 0),
    (8, 8, 64, 32, [96, 95, 1, 0], 0, 0),
    (32, 8, 64, 16, [700, 3, 255, 513], 100, 4),
    (8, 1, 128, 128, [1000, 129], 0, 0),
    (8, 1, 64, 256, [600], 33, 1),
    (16, 4, 128, 32, [333, 64, 65], 64, 40),
    (4, 2, 64, 16, [50, 49, 17], 1, 0),
    (2, 2, 128, 64, [130, 5], 16, 100),
    (3, 3, 64, 16, [77, 16, 400], 0, 0),
    (1, 1, 64, 16, [2000], 1500, 17),
])
@pytest.mark.parametrize("weights", [False, True])
def test_decode(cuda, nHq, nKv, hd, page, lens, window, sinks, weights):
    c = ref.Cache(len(lens) * 7 + page, len(lens), -(-max(lens) // page) + 1, page, nKv, hd)
    _decode_check(c, lens, nHq, window, sinks, weights)


def test_decode_long_split(cuda):
    """one long sequence beside short ones: parts of a pair over many CTAs"""
    lens = [20011, 1, 700, 0, 4097]
    c = ref.Cache(5, 5, 20011 // 64 + 1, 64, 2, 128)
    _decode_check(c, lens, 4, weights=True)


def test_decode_many_sequences(cuda):
    """more sequences than a CTA has threads"""
    lens = [(37 * i) % 90 for i in range(300)]
    c = ref.Cache(6, 300, 6, 16, 1, 64)
    _decode_check(c, lens, 2, window=40, sinks=3)


def test_decode_unseen_rows_are_not_used(cuda):
    """NaN, infinities and the lowest byte in rows behind the length and outside the window"""
    c = ref.Cache(8, 2, 20, 16, 2, 64)
    lens, window, sinks = [250, 100], 40, 3
    for b, n in enumerate(lens):
        ok = ref.seen(n, n - 1, window, sinks)
        c.poison_rows(b, [j for j in range(c.cap) if j >= n or not ok[j]])
    _decode_check(c, lens, 4, window, sinks, weights=True)


def test_decode_shared_pages(cuda):
    """two sequences with a common first page (a shared prompt)"""
    c = ref.Cache(9, 3, 4, 32, 2, 128)
    c.table[1, 0] = c.table[0, 0]
    c.table[2, :2] = c.table[0, :2]
    _decode_check(c, [100, 60, 65], 4, weights=True)


def test_decode_large_scores(cuda):
    """scores of some hundreds: the running maximum has to carry them"""
    c = ref.Cache(10, 1, 40, 16, 1, 64)
    c.Ks *= 40
    _decode_check(c, [600], 4)


def test_decode_far_pages(cuda):
    """pool offsets past 2^31 bytes (and rows past 2^31 / 1024)"""
    nKv, hd, page = 8, 128, 256
    n = (1 << 31) // (page * nKv * hd) + 8
    small = ref.Cache(11, 1, 4, page, nKv, hd, spare=0)
    far = torch.tensor([[n - 1, n - 5, 0, n - 2]], dtype=torch.int32)
    kv = []
    for t in (small.Kq, small.Ks, small.Vq, small.Vs):
        big = torch.empty((n,) + tuple(t.shape[1:]), dtype=t.dtype, device="cuda")
        big[far[0].long().cuda()] = t[small.table[0].long()].cuda()
        kv.append(big)
    g = torch.Generator().manual_seed(3)
    q = torch.randn(1, 16 * hd, generator=g) * 1.5
    got = tb.attention_decode_paged_q8(q.cuda(), tuple(kv), far.cuda(), _ints([1000]), 16, nKv, hd).cpu()
    near = tb.attention_decode_paged_q8(q.cuda(), small.dev(), small.table.cuda(), _ints([1000]), 16, nKv, hd).cpu()
    assert torch.equal(got, near)
    pq = torch.randn(5, 16 * hd, generator=g)
    args = (_ints([0, 5]), _ints([1000]), 16, nKv, hd)
    a = tb.attention_prefill_paged_q8(pq.cuda(), tuple(kv), far.cuda(), *args)
    b = tb.attention_prefill_paged_q8(pq.cuda(), small.dev(), small.table.cuda(), *args)
    assert torch.equal(a, b)


@pytest.mark.parametrize("hd", [64, 128])
def test_nan_in_a_query_stays_in_its_head(cuda, hd):
    c = ref.Cache(51, 2, 20, 16, 2, hd)
    lens = [300, 9]
    q = torch.randn(2, 8 * hd, generator=c.g)
    bad = q.clone()
    bad.view(2, 8, hd)[1, 5, 3] = float("nan")
    kv, table = c.dev(), c.table.cuda()
    hit = torch.zeros(2, 8, dtype=torch.bool)
    hit[1, 5] = True
    for run in (lambda x: tb.attention_decode_paged_q8(x.cuda(), kv, table, _ints(lens), 8, 2, hd),
                lambda x: tb.attention_prefill_paged_q8(x.cuda(), kv, table, _ints([0, 1, 2]), _ints(lens), 8, 2, hd)):
        a, b = run(q).cpu().view(2, 8, hd), run(bad).cpu().view(2, 8, hd)
        assert b[hit].isnan().all() and torch.equal(a[~hit], b[~hit])


def test_decode_same_bits_every_time(cuda):
    c = ref.Cache(12, 3, 60, 32, 4, 128)
    a = _decode_check(c, [1900, 77, 1000], 16, weights=True)
    b = _decode_check(c, [1900, 77, 1000], 16, weights=True)
    assert torch.equal(a, b)


def test_contiguous_cache_is_one_page_table(cuda):
    """the contiguous cache read as pages in order: the contiguous operator's result"""
    c = ref.Cache(13, 1, 8, 32, 8, 128)
    c.table = torch.arange(8, dtype=torch.int32)[None].contiguous()
    q = torch.randn(1, 16 * 128, generator=c.g).cuda()
    kv = c.dev()
    a = tb.attention_decode_paged_q8(q, kv, c.table.cuda(), _ints([250]), 16, 8, 128)
    flat = tuple(t.reshape(-1, t.shape[-1]) for t in kv)
    b = tb.attention_decode_q8(q.reshape(-1), flat, 250, 16, 8, 128)
    assert float((a.reshape(-1) - b).abs().max()) < 1e-4 * float(b.abs().max())   # tb_attn_decode_q8's own bar


def _prefill_check(c, lens, ts, nHq, window=0, sinks=0, seed=2, lead=0, tail=0, only=None):
    g = torch.Generator().manual_seed(seed)
    cu = [lead + sum(ts[:b]) for b in range(c.B + 1)]
    T = cu[-1] + tail
    q = torch.randn(T, nHq * c.hd, generator=g) * 1.5
    out = torch.full((T, nHq * c.hd), 7.0, dtype=torch.bfloat16, device="cuda")
    got = tb.attention_prefill_paged_q8(q.cuda(), c.dev(), c.table.cuda(), _ints(cu), _ints(lens), nHq, c.nKv, c.hd,
                                        window=window, sinks=sinks, out=out).cpu().double()
    assert (got[:lead] == 7).all() and (got[cu[-1]:] == 7).all()
    for b, (n, t) in enumerate(zip(lens, ts)):
        for i in range(t):
            if only is not None and i not in only:
                continue
            o, _, mag, big = ref.attend(c, b, q[cu[b] + i], n - t + i, nHq, window, sinks)
            d = 2.0 ** -10 * mag
            x = got[cu[b] + i].reshape(nHq, c.hd)
            tol = big * (2 * d + 2.0 ** -9) + 2.0 ** -8 * o.abs()
            assert ((x - o).abs() <= tol).all(), (b, i, float((x - o).abs().max()))
            # the roundings are independent: the row as a whole is far nearer than the bound of each element
            rel = float((x - o).norm() / o.norm())
            assert rel < 2.0 ** -7, (b, i, rel)
    return got


@pytest.mark.parametrize("nHq,nKv,hd,page,lens,ts,window,sinks", [
    (16, 8, 128, 64, [1], [1], 0, 0),
    (16, 8, 128, 16, [130], [130], 0, 0),
    (4, 2, 64, 16, [40, 0, 7, 300], [5, 0, 7, 129], 0, 0),
    (32, 8, 64, 32, [200, 77], [70, 77], 50, 4),
    (8, 1, 128, 128, [513], [40], 0, 0),
    (8, 1, 64, 256, [600, 1], [33, 1], 100, 1),
    (16, 4, 128, 32, [260, 64], [65, 64], 64, 40),
    (2, 2, 128, 64, [150, 129], [150, 1], 16, 300),
    (3, 3, 64, 16, [77, 128], [77, 128], 1, 0),
    (1, 1, 64, 16, [257], [257], 0, 0),
])
def test_prefill(cuda, nHq, nKv, hd, page, lens, ts, window, sinks):
    c = ref.Cache(len(lens) * 5 + page, len(lens), -(-max(lens) // page) + 1, page, nKv, hd)
    _prefill_check(c, lens, ts, nHq, window, sinks, lead=3, tail=5)


def test_prefill_long_history(cuda):
    """few rows behind a long history (split over the length), and a long prompt, sampled"""
    c = ref.Cache(21, 2, 10000 // 64 + 1, 64, 2, 128)
    _prefill_check(c, [10000, 9001], [9, 2], 4)
    c = ref.Cache(22, 1, 3001 // 128 + 1, 128, 1, 128)
    _prefill_check(c, [3001], [3001], 2, only=set(range(0, 3001, 149)) | {127, 128, 255, 256, 3000})
    _prefill_check(c, [3001], [3001], 2, window=700, sinks=5, only=set(range(0, 3001, 211)) | {699, 700, 701, 3000})


def test_prefill_unseen_rows_are_not_used(cuda):
    c = ref.Cache(23, 2, 24, 16, 2, 64)
    lens, ts, window, sinks = [300, 100], [20, 100], 40, 3
    for b, (n, t) in enumerate(zip(lens, ts)):
        first = max(0, n - t - window + 1)
        c.poison_rows(b, [j for j in range(c.cap) if j >= n or (j < first and j >= sinks)])
    _prefill_check(c, lens, ts, 4, window, sinks)


def test_freed_pages_are_not_looked_up(cuda):
    """table entries of pages that no row under the window sees may be anything (their pages were freed)"""
    c = ref.Cache(25, 2, 40, 16, 2, 64)
    lens, window, sinks = [600, 333], 100, 5
    whole = c.table.clone()
    for b, n in enumerate(lens):
        c.table[b, 1:(n - window) // 16] = -1
        c.table[b, -(-n // 16):] = 2 ** 31 - 1
    q = torch.randn(2, 4 * 64, generator=c.g).cuda()
    a = tb.attention_decode_paged_q8(q, c.dev(), c.table.cuda(), _ints(lens), 4, 2, 64, window=window, sinks=sinks)
    b = tb.attention_decode_paged_q8(q, c.dev(), whole.cuda(), _ints(lens), 4, 2, 64, window=window, sinks=sinks)
    assert torch.equal(a, b)
    args = (_ints([0, 1, 2]), _ints(lens), 4, 2, 64)
    a = tb.attention_prefill_paged_q8(q, c.dev(), c.table.cuda(), *args, window=window, sinks=sinks)
    b = tb.attention_prefill_paged_q8(q, c.dev(), whole.cuda(), *args, window=window, sinks=sinks)
    assert torch.equal(a, b)
    assert tb.default_context(0).device_error() == 0


def test_prefill_many_sequences(cuda):
    """more sequences than the plan has threads, most of them short, some without new rows"""
    lens = [(37 * i) % 90 + 1 for i in range(600)]
    ts = [min(n, (11 * i) % 7) for i, n in enumerate(lens)]
    c = ref.Cache(26, 600, 6, 16, 1, 64)
    _prefill_check(c, lens, ts, 8, window=50, sinks=2)


@pytest.mark.parametrize("hd,slope", [(64, 1.0), (128, 1.0), (128, -1.0), (64, 0.3)])
def test_prefill_rising_scores(cuda, hd, slope):
    """scores that climb (or fall) by hundreds over the keys, so the running reference has to be raised again
    and again.  K = byte / 64, V likewise and q in eighths are exact in f16, so scores are exact; what is left
    is P's and a joined part's rounding (2^-11 each, relative), f32 and bf16's 2^-8 of the output."""
    n, t, nKv, nHq = 900, 140, 2, 4
    c = ref.Cache(27, 1, 60, 16, nKv, hd)
    c.Ks[:] = 127.0 / 64
    c.Vs[:] = 127.0 / 64
    ramp = (slope * 127.0 * torch.arange(n) / n).round().to(torch.int8)
    rows = c.rows(0, torch.arange(n))
    c.Kq.view(-1, nKv, hd)[rows, :, 0] = ramp[:, None]
    q = (torch.randint(-8, 9, (t, nHq * hd), generator=c.g).float() / 8)
    q.view(t, nHq, hd)[:, :, 0] = 1600.0
    got = tb.attention_prefill_paged_q8(q.cuda(), c.dev(), c.table.cuda(), _ints([0, t]), _ints([n]), nHq, nKv,
                                        hd).cpu().double()
    for i in list(range(0, t, 13)) + [t - 1]:
        o, _, _, big = ref.attend(c, 0, q[i], n - t + i, nHq)
        tol = 2.0 ** -8 * o.abs() + big * (2.0 ** -10 + 2.0 ** -14)
        assert ((got[i].reshape(nHq, hd) - o).abs() <= tol).all(), i
    dec = tb.attention_decode_paged_q8(q[-1:].cuda(), c.dev(), c.table.cuda(), _ints([n]), nHq, nKv, hd).cpu().double()
    o, _, mag, big = ref.attend(c, 0, q[-1], n - 1, nHq)
    assert float((dec[0].reshape(nHq, hd) - o).abs().max()) <= (2 * (hd + 8) * U * mag + (n + 16) * U) * big


def test_prefill_last_row_is_decode(cuda):
    c = ref.Cache(24, 1, 20, 32, 4, 128)
    q = torch.randn(50, 8 * 128, generator=c.g).cuda()
    kv, table = c.dev(), c.table.cuda()
    a = tb.attention_prefill_paged_q8(q, kv, table, _ints([0, 50]), _ints([600]), 8, 4, 128, window=90, sinks=2)
    b = tb.attention_decode_paged_q8(q[-1:].contiguous(), kv, table, _ints([600]), 8, 4, 128, window=90, sinks=2)
    assert float((a[-1].float() - b[0]).norm() / b.norm()) < 2.0 ** -7


@pytest.mark.parametrize("nHq,nKv,hd,page,T", [(16, 8, 128, 64, 1), (16, 8, 128, 16, 37), (32, 8, 64, 32, 300),
                                               (8, 1, 64, 256, 5), (3, 3, 64, 16, 9), (6, 2, 128, 128, 700)])
def test_prep(cuda, nHq, nKv, hd, page, T):
    B = 3
    c = ref.Cache(31, B, max(4, -(-T // page) + 1), page, nKv, hd, fill=False)
    g = torch.Generator().manual_seed(T)
    q, k, v = (torch.randn(T, h * hd, generator=g) * 2 for h in (nHq, nKv, nKv))
    qw, kw = ((1 + 0.2 * torch.randn(hd, generator=g)).to(torch.float16) for _ in range(2))
    flat = torch.randperm(B * c.cap, generator=g)[:T]          # distinct (sequence, row) pairs, in no order
    seq, slot = (flat // c.cap).to(torch.int32), (flat % c.cap).to(torch.int32)
    pos = torch.randint(0, 200000, (T,), generator=g).to(torch.int32)
    if T > 4:
        seq[2] = -1                                            # a padding row
        k[4, :32] = 0                                          # a zero head group keeps a zero row
    kv = c.dev()
    qr = torch.full((T, nHq * hd), 5.0, device="cuda")
    tb.attn_prep_paged_q8(q.cuda(), k.cuda(), v.cuda(), qw.cuda(), kw.cuda(), kv, c.table.cuda(), seq.cuda(),
                          slot.cuda(), pos.cuda(), nHq, nKv, hd, 1e6, 1e-6, qr=qr)
    live = seq >= 0
    want = ref.norm_rope(q, qw, pos, nHq, hd, 1e6, 1e-6)
    got = qr.cpu()
    assert (got[~live] == 5).all()
    # half a step of f32, and the 64-bit rows behind it: an angle is pos * theta^-x, whose power two
    # libraries may round one step (2^-52 of it) apart and whose product rounds once more, so it is off by
    # at most 2^-51 * 200000 = 8.9e-11; a rotated pair is off by that times its length, below 2 sqrt(hd)
    assert ((got[live].double() - want[live]).abs() <= want[live].abs() * U + 8.9e-11 * 2 * hd ** 0.5).all()
    Kq, Ks, Vq, Vs = c.Kq.clone(), c.Ks.clone(), c.Vq.clone(), c.Vs.clone()
    k8, km = ref.quantize(ref.norm_rope(k, kw, pos, nKv, hd, 1e6, 1e-6).float())
    v8, vm = ref.quantize(v)
    for t in range(T):
        if not live[t]:
            continue
        r = c.rows(int(seq[t]), int(slot[t]))
        w = nKv * hd
        Kq.view(-1, w)[r], Ks.view(-1, w // 32)[r] = k8[t], km[t]
        Vq.view(-1, w)[r], Vs.view(-1, w // 32)[r] = v8[t], vm[t]
    for have, need in zip(kv, (Kq, Ks, Vq, Vs)):              # rows that no call names stay as they were
        assert torch.equal(have.cpu(), need)


@pytest.mark.parametrize("nHq,nKv,hd,page,T", [(6, 2, 128, 128, 803), (5, 3, 64, 64, 1001)])
def test_prep_many_rows(cuda, nHq, nKv, hd, page, T):
    """enough rows for four of them a CTA, the last CTA's not all there"""
    test_prep(cuda, nHq, nKv, hd, page, T)


@pytest.mark.parametrize("lens,budget,sinks,recent,page,new_page", [
    ([300, 40, 41, 0, 1], 40, 4, 8, 16, 16),
    ([5000, 3000], 700, 0, 0, 64, 64),
    ([200], 17, 17, 0, 32, 16),
    ([200], 30, 0, 30, 32, 256),
    ([130, 129], 128, 3, 100, 16, 16),
    ([64, 7], 1, 0, 0, 16, 16),
    ([4100], 4099, 1, 1, 128, 128),
])
@pytest.mark.parametrize("kind", ["random", "ties", "strange"])
def test_evict(cuda, lens, budget, sinks, recent, page, new_page, kind):
    nKv, hd, B = 2, 64, len(lens)
    c = ref.Cache(41, B, -(-max(lens) // page) + 1, page, nKv, hd)
    g = torch.Generator().manual_seed(4)
    w = torch.exp(2 * torch.randn(B, nKv, c.cap, generator=g))
    if kind == "ties":
        w = torch.randint(0, 3, w.shape, generator=g).float()
    if kind == "strange":
        w[:, :, ::5] = 0
        w[:, 0, 1::7] = float("inf")
        w[:, :, 2::9] = 1e-42
        w[:, :, 3::11] = -1.0
    keep = -(-budget // new_page)
    n_new = B * keep
    dst = [torch.full((n_new, new_page, t.shape[-1]), 9, dtype=t.dtype, device="cuda")
           for t in (c.Kq, c.Ks, c.Vq, c.Vs)]
    new_table = torch.randperm(n_new, generator=g).to(torch.int32).reshape(B, keep).contiguous()
    kv = c.dev()
    kept, new_lens, new_w = tb.kv_evict_paged_q8(kv, c.table.cuda(), _ints(lens), w.cuda(), new_table.cuda(), budget,
                                                 sinks, recent, nKv, hd, kv_out=dst)
    kept, new_lens, new_w = kept.cpu(), new_lens.cpu(), new_w.cpu()
    dst = [t.cpu() for t in dst]
    for b, n in enumerate(lens):
        want = ref.evict(w[b], n, budget, sinks, recent)
        assert int(new_lens[b]) == len(want)
        assert kept[b].tolist() == want + [-1] * (budget - len(want))
        assert torch.equal(new_w[b, :, :len(want)], w[b][:, want])
        assert (new_w[b, :, len(want):] == 0).all()
        r0 = c.rows(b, torch.tensor(want, dtype=torch.long))
        at = torch.arange(keep * new_page)
        r1 = new_table[b, at // new_page].long() * new_page + at % new_page
        for src, d in zip((c.Kq, c.Ks, c.Vq, c.Vs), dst):
            d = d.reshape(-1, d.shape[-1])
            assert torch.equal(d[r1[:len(want)]], src.reshape(-1, src.shape[-1])[r0])
            assert (d[r1[len(want):]] == 9).all()              # the rest of the new pages stays as it was
    for have, need in zip(kv, (c.Kq, c.Ks, c.Vq, c.Vs)):
        assert torch.equal(have.cpu(), need)


def test_evict_more_rows_than_registers(cuda):
    """a cache beyond the rows that the selecting threads hold in registers, with ties"""
    n, budget, page = 150001, 20000, 256
    c = ref.Cache(42, 1, n // page + 1, page, 1, 64, fill=False)
    g = torch.Generator().manual_seed(6)
    for w in (torch.randn(1, 1, c.cap, generator=g).abs(), torch.randint(0, 5, (1, 1, c.cap), generator=g).float(),
              torch.ones(1, 1, c.cap)):
        fresh = torch.arange(-(-budget // page), dtype=torch.int32)[None]
        dst = [torch.zeros(fresh.numel(), page, t.shape[-1], dtype=t.dtype, device="cuda") for t in c.dev()]
        kept, nl, nw = tb.kv_evict_paged_q8(c.dev(), c.table.cuda(), _ints([n]), w.cuda(), fresh.cuda(), budget, 4, 100,
                                            1, 64, kv_out=dst)
        want = ref.evict(w[0], n, budget, 4, 100)
        assert kept[0].tolist() == want and int(nl) == budget
        assert torch.equal(nw[0, 0, :budget].cpu(), w[0, 0][want])


def test_run_of_all(cuda):
    """two requests served: a prompt each (prep, prefill), decode steps that add up the weights, an
    eviction to a quarter, and decode steps on the shrunk cache whose rotary positions go on"""
    nHq, nKv, hd, page, B = 8, 4, 128, 16, 2
    c = ref.Cache(51, B, 12, page, nKv, hd, spare=8, fill=False)
    kv, table = c.dev(), c.table.cuda()
    g = torch.Generator().manual_seed(5)
    qw, kw = ((1 + 0.2 * torch.randn(hd, generator=g)).to(torch.float16) for _ in range(2))
    lens = [150, 90]

    def rows(T):
        return [torch.randn(T, h * hd, generator=g) for h in (nHq, nKv, nKv)]

    def prep(x, seq, slot, pos):
        return tb.attn_prep_paged_q8(*[t.cuda() for t in x], qw.cuda(), kw.cuda(), kv, table, _ints(seq), _ints(slot),
                                     _ints(pos), nHq, nKv, hd, 1e6, 1e-6)

    def sync_ref():
        c.Kq, c.Ks, c.Vq, c.Vs = (t.cpu() for t in kv)
        c.table = table.cpu()
        c.cap = c.table.shape[1] * page

    seq = [0] * 150 + [1] * 90
    slot = list(range(150)) + list(range(90))
    qr = prep(rows(240), seq, slot, slot)
    out = tb.attention_prefill_paged_q8(qr, kv, table, _ints([0, 150, 240]), _ints(lens), nHq, nKv, hd).cpu().double()
    sync_ref()
    for t in (0, 77, 149, 150, 239):
        b, pos = seq[t], slot[t]
        o = ref.attend(c, b, qr[t].cpu(), pos, nHq)[0]
        assert float((out[t].reshape(nHq, hd) - o).norm() / o.norm()) < 2.0 ** -7
    weights = torch.zeros(B, nKv, 12 * page, device="cuda")
    total = weights.cpu().double()
    pos = list(lens)

    def steps(n):
        for _ in range(n):
            qr = prep(rows(B), [0, 1], lens, pos)
            for b in range(B):
                lens[b] += 1
                pos[b] += 1
            got = tb.attention_decode_paged_q8(qr, kv, table, _ints(lens), nHq, nKv, hd, weights=weights).cpu().double()
            sync_ref()
            for b in range(B):
                o, w, mag, big = ref.attend(c, b, qr[b].cpu(), lens[b] - 1, nHq)
                rel = 2 * (hd + 8) * U * mag + (lens[b] + 16) * U
                assert float((got[b].reshape(nHq, hd) - o).abs().max()) <= rel * big
                total[b, :, :lens[b]] += w
    steps(4)
    assert float((weights.cpu().double() - total).abs().max()) < 1e-4 * float(total.max())
    new_table = torch.arange(c.table.max() + 1, dtype=torch.int32)
    free = [p for p in range(c.Kq.shape[0]) if p not in set(c.table.flatten().tolist())][:6]
    new_table = _ints([free[:3], free[3:]])
    kept, nl, weights = tb.kv_evict_paged_q8(kv, table, _ints(lens), weights, new_table, 40, 2, 8, nKv, hd)
    kept = kept.cpu()
    assert nl.tolist() == [40, 40]
    total = torch.stack([total[b][:, kept[b].long()] for b in range(B)])
    total = torch.cat([total, torch.zeros(B, nKv, 8, dtype=torch.float64)], 2)
    table = new_table
    lens[:] = [40, 40]
    steps(3)
    assert float((weights.cpu().double() - total).abs().max()) < 1e-4 * float(total.max())


def test_other_stream_and_graphs(cuda):
    """another stream; a captured call replayed on new contents; two captured calls side by side"""
    c = ref.Cache(61, 2, 30, 32, 2, 128)
    kv, table, lens = c.dev(), c.table.cuda(), _ints([900, 500])
    q = torch.randn(2, 4 * 128, generator=c.g).cuda()
    pq = torch.randn(40, 4 * 128, generator=c.g).cuda()
    cu = _ints([0, 25, 40])
    fresh = torch.arange(60, 62, dtype=torch.int32).reshape(2, 1).cuda()
    w = torch.rand(2, 2, 960, generator=c.g).cuda()
    out_kv = [torch.zeros(62, *t.shape[1:], dtype=t.dtype, device="cuda") for t in kv]

    def calls():
        return (tb.attention_decode_paged_q8(q, kv, table, lens, 4, 2, 128),
                tb.attention_prefill_paged_q8(pq, kv, table, cu, lens, 4, 2, 128, window=200, sinks=4),
                *tb.kv_evict_paged_q8(kv, table, lens, w, fresh, 30, 2, 4, 2, 128, kv_out=out_kv))

    want = [t.clone() for t in calls()]
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = calls()
    s.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a, b)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o = calls()
        graphs.append((g, o))
    q.mul_(2.0)
    want = [t.clone() for t in calls()]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for (g, _), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for _, o in graphs:
        for a, b in zip(want, o):
            assert torch.equal(a, b)


def test_context_scratch(cuda):
    """the C entry without a workspace takes the context's scratch"""
    import ctypes
    from tabinfer_b200._lib import LIB, PagedKV
    c = ref.Cache(62, 1, 30, 32, 2, 128)
    kv, table, lens = c.dev(), c.table.cuda(), _ints([900])
    q = torch.randn(1, 4 * 128, generator=c.g).cuda()
    want = tb.attention_decode_paged_q8(q, kv, table, lens, 4, 2, 128)
    out = torch.empty_like(want)
    ctx = tb.default_context(0)
    s = PagedKV(*[t.data_ptr() for t in kv], table.data_ptr(), kv[0].shape[0], 32, 1, 30, 2, 128)
    ctx.check(LIB.tb_attn_decode_paged_q8(ctx.h, ctypes.byref(s), out.data_ptr(), q.data_ptr(), lens.data_ptr(), 4, 0,
                                          0, None, None, 0), "decode")
    assert torch.equal(out, want)
    n = ctypes.c_size_t()
    ctx.check(LIB.tb_attn_decode_paged_ws(ctx.h, ctypes.byref(s), 4, 0, ctypes.byref(n)), "ws")
    small = torch.empty(256, dtype=torch.uint8, device="cuda")
    assert LIB.tb_attn_decode_paged_q8(ctx.h, ctypes.byref(s), out.data_ptr(), q.data_ptr(), lens.data_ptr(), 4, 0, 0,
                                       None, small.data_ptr(), n.value - 1) == 1


def test_device_checks(cuda):
    """bad pages, lengths, rows: the error word, and nothing out of the pool is touched"""
    ctx = tb.default_context(0)

    def word():
        return ctx.device_error()
    c = ref.Cache(71, 2, 8, 16, 2, 64)
    kv = c.dev()
    q = torch.randn(2, 4 * 64, generator=c.g)
    for bad in (-1, c.Kq.shape[0], 2 ** 31 - 1, -2 ** 31):
        table = c.table.clone()
        table[0, 3] = bad
        out = tb.attention_decode_paged_q8(q.cuda(), kv, table.cuda(), _ints([100, 50]), 4, 2, 64).cpu()
        assert word() == 0x6c01
        # the sequence beside it is whole, and the bad page's rows are left out
        o = ref.attend(c, 1, q[1], 49, 4)[0]
        assert float((out[1].double().reshape(4, 64) - o).norm() / o.norm()) < 1e-5
        j = torch.arange(100)
        ok = (j < 48) | (j >= 64)
        k, v = c.head(0, 100, 0)
        p = torch.softmax(k[ok] @ q[0].double()[:64] * 64 ** -0.5, 0)
        assert float((out[0].double()[:64] - p @ v[ok]).norm() / (p @ v[ok]).norm()) < 1e-5
        pq = torch.randn(8, 4 * 64, generator=c.g).cuda()
        got = tb.attention_prefill_paged_q8(pq, kv, table.cuda(), _ints([0, 4, 8]), _ints([100, 50]), 4, 2, 64).cpu()
        assert word() == 0x6c01
        p = torch.softmax(k[:97][ok[:97]] @ pq[0].cpu().double()[:64] * 64 ** -0.5, 0) @ v[:97][ok[:97]]
        assert float((got[0].double()[:64] - p).norm() / p.norm()) < 2.0 ** -7
        new = torch.full((4, 16, 128), 9, dtype=torch.int8, device="cuda")
        dst = (new, torch.zeros(4, 16, 4, device="cuda"), new.clone(), torch.zeros(4, 16, 4, device="cuda"))
        tb.kv_evict_paged_q8(kv, table.cuda(), _ints([100, 50]), torch.ones(2, 2, 128, device="cuda"),
                             _ints([[0, bad], [1, 2]]), 32, 0, 32, 2, 64, kv_out=dst)
        assert word() == 0x6c01
        assert (new[3] == 9).all()
    # a table entry behind the last row is not read
    table = c.table.clone()
    table[:, 7] = -5
    tb.attention_decode_paged_q8(q.cuda(), kv, table.cuda(), _ints([112, 50]), 4, 2, 64)
    assert word() == 0
    for bad in (-1, 129, 2 ** 31 - 1):
        out = tb.attention_decode_paged_q8(q.cuda(), kv, c.table.cuda(), _ints([bad, 50]), 4, 2, 64).cpu()
        assert word() == 0x6c02 and (out[0] == 0).all() and out[1].abs().max() > 0
        got = tb.attention_prefill_paged_q8(q.cuda(), kv, c.table.cuda(), _ints([0, 1, 2]), _ints([bad, 50]), 4, 2, 64)
        assert word() == 0x6c02 and (got[0] == 0).all()
    # a chunk longer than its sequence: the rows before its start are empty
    got = tb.attention_prefill_paged_q8(torch.randn(6, 256, device="cuda"), kv, c.table.cuda(), _ints([0, 5, 6]),
                                        _ints([3, 1]), 4, 2, 64)
    assert word() == 0x6c02 and (got[:2] == 0).all() and got[2].abs().max() > 0
    x = [torch.randn(3, n, device="cuda") for n in (256, 128, 128)]
    w = torch.ones(64, dtype=torch.float16, device="cuda")
    before = [t.clone() for t in kv]
    qr = torch.full((3, 256), 5.0, device="cuda")
    tb.attn_prep_paged_q8(*x, w, w, kv, c.table.cuda(), _ints([2, 0, 1]), _ints([0, 128, -1]), _ints([0, 0, 0]), 4, 2,
                          64, 1e6, 1e-6, qr=qr)
    assert word() == 0x6c02 and (qr == 5).all()
    assert all(torch.equal(a, b) for a, b in zip(kv, before))


def test_refusals(cuda):
    c = ref.Cache(81, 2, 4, 16, 2, 64)
    kv, table, lens = c.dev(), c.table.cuda(), _ints([10, 20])
    q = torch.randn(2, 256, device="cuda")
    ok = dict(qr=q, kv=kv, table=table, lens=lens, nHq=4, nKv=2, hd=64)

    def refuse(f, base, **kw):
        with pytest.raises(tb.TabInferError):
            f(**{**base, **kw})
    dec = tb.attention_decode_paged_q8
    dec(**ok)
    refuse(dec, ok, window=-1)
    refuse(dec, ok, sinks=-1)
    refuse(dec, ok, nHq=6, qr=torch.randn(2, 384, device="cuda"))           # a group of three
    refuse(dec, ok, nHq=8)                                                   # q too narrow
    refuse(dec, ok, hd=32, nKv=4)                                            # head_dim 32
    refuse(dec, ok, qr=q.cpu())
    refuse(dec, ok, qr=q.double())
    refuse(dec, ok, qr=torch.randn(256, 2, device="cuda").T)                 # strided
    refuse(dec, ok, lens=lens.long())
    refuse(dec, ok, lens=lens[:1])
    refuse(dec, ok, table=table.long())
    refuse(dec, ok, weights=torch.zeros(2, 2, 63, device="cuda"))
    refuse(dec, ok, kv=(kv[0][:, :15].contiguous(),) + kv[1:])
    refuse(dec, ok, kv=(kv[0].reshape(-1, 128),) + kv[1:])
    odd = tuple(t[:, :12].contiguous() for t in kv)                          # 12 rows a page
    refuse(dec, ok, kv=odd)
    flat = torch.zeros(kv[0].numel() + 1, dtype=torch.int8, device="cuda")[1:].reshape(kv[0].shape)
    refuse(dec, ok, kv=(flat,) + kv[1:])                                     # not 16-byte aligned
    pre = tb.attention_prefill_paged_q8
    ok = dict(q=q, kv=kv, table=table, cu=_ints([0, 1, 2]), lens=lens, nHq=4, nKv=2, hd=64)
    pre(**ok)
    refuse(pre, ok, cu=_ints([0, 2]))
    refuse(pre, ok, window=-1)
    refuse(pre, ok, out=torch.zeros(2, 256, device="cuda"))                  # f32 out
    refuse(pre, ok, q=q[:, :128].contiguous())
    assert pre(**{**ok, "q": q[:0], "cu": _ints([0, 0, 0])}).shape == (0, 256)
    ev = tb.kv_evict_paged_q8
    ok = dict(kv=kv, table=table, lens=lens, weights=torch.zeros(2, 2, 64, device="cuda"), new_table=_ints([[8], [9]]),
              budget=16, sinks=2, recent=3, nKv=2, hd=64)
    ev(**ok)
    refuse(ev, ok, budget=17)                                                # more than the new table holds
    refuse(ev, ok, budget=0, sinks=0, recent=0)
    refuse(ev, ok, budget=-1)
    refuse(ev, ok, sinks=14)                                                 # sinks + recent over the budget
    refuse(ev, ok, recent=-1)
    refuse(ev, ok, new_table=_ints([[8]]))
    prep = tb.attn_prep_paged_q8
    w = torch.ones(64, dtype=torch.float16, device="cuda")
    i = _ints([0, 1])
    ok = dict(q=q, k=q[:, :128].contiguous(), v=q[:, :128].contiguous(), qw16=w, kw16=w, kv=kv, table=table, seq=i,
              slot=i, pos=i, nHq=4, nKv=2, hd=64, theta=1e6, eps=1e-6)
    prep(**ok)
    refuse(prep, ok, seq=i.long())
    refuse(prep, ok, pos=i[:1])
    refuse(prep, ok, qw16=w[:32])
    refuse(prep, ok, theta=0.0)
    refuse(prep, ok, v=q)
    assert prep(**{**ok, "q": q[:0], "k": q[:0, :128], "v": q[:0, :128], "seq": i[:0], "slot": i[:0], "pos": i[:0]}).shape == (0, 256)
