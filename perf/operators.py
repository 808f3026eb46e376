"""Cases of the paged int8 KV cache operators: their inputs, their plain forms and the framework's calls.

The operators share one cache format: pools Kq / Vq int8 [pages][page][hk*hd] with one f32 scale per 32
elements in Ks / Vs [pages][page][hk*hd/32]; an element stands for q / 127 * scale.  Row r of sequence b is
line r % page of pool page table[b][r // page].

  prep     head norm and rotary embedding of q and k, k and v quantized into the cache's pages
  decode   one new token a sequence over its pages (window, sinks, accumulated attention weights)
  prefill  packed prompts or chunks of prompts over their pages (causal, window, sinks)
  evict    keeps a sequence's heaviest rows by accumulated weight and compacts them into other pages
"""
import math

import torch

own = False

THETA = 1e6
EPS = 1e-6


# --------------------------------------------------------------------------
# cases
# --------------------------------------------------------------------------

def _case(name, op, **kw):
    c = dict(name=name, op=op, B=1, T=0, S=1, hq=16, hk=8, hd=128, page=64, window=0, sinks=0, acc=False, budget=0,
             recent=0)
    c.update(kw)
    return c


def listed():
    return [
        # the prep of one decode step of a 16/8-head model (the smallest call: latency)
        _case("prep_one_row", "prep", T=1, S=4096),
        # the prep of four 2048-token prompts at once
        _case("prep_prompt_rows", "prep", B=4, T=2048, S=2048),
        # a single user's decode step at 4096 rows (the framework's own decode benchmark)
        _case("decode_one_4096", "decode", S=4096),
        # a serving batch of ragged lengths that tracks the weights for a later eviction
        _case("decode_batch_ragged", "decode", B=32, S=8192, page=32, acc=True),
        # one very long, odd-length context
        _case("decode_long", "decode", S=131001, page=128),
        # a batch of long chats under a sliding window with first tokens kept, 64-wide heads, small pages
        _case("decode_window_sinks", "decode", B=16, S=32768, hq=32, hk=8, hd=64, page=16, window=4096, sinks=4),
        # a short chunk of a prompt behind a long history (few rows: the length has to be split)
        _case("prefill_short_chunk", "prefill", T=77, S=8192, page=16),
        # the framework's own prefill benchmark length
        _case("prefill_2048", "prefill", T=2048, S=2048),
        # a long prompt
        _case("prefill_8192", "prefill", T=8192, S=8192, page=128),
        # three packed chunks with histories under a window with sinks, 64-wide heads in groups of four
        _case("prefill_window_ragged", "prefill", B=3, T=2001, S=6000, hq=32, hk=8, hd=64, page=32, window=1024,
              sinks=4),
        # a serving batch shrunk to a quarter
        _case("evict_batch", "evict", B=16, S=8192, page=32, budget=2048, sinks=4, recent=128),
        # one long context shrunk to an eighth
        _case("evict_long", "evict", S=131072, page=128, budget=16384, sinks=4, recent=512),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["prep", "decode", "prefill", "evict"])
    hq, hk, hd = rng.choice([(16, 8, 128), (32, 8, 64), (8, 8, 64), (8, 1, 128), (16, 4, 128), (32, 8, 128), (4, 2, 64)])
    c = _case("", op, hq=hq, hk=hk, hd=hd, page=rng.choice([16, 32, 64, 128]))
    del c["name"]
    if op == "prep":
        T = _log(rng, 1, 4096)
        c.update(T=T, B=_log(rng, 1, max(1, 4096 // T)), S=T + _log(rng, 1, 4096))
    elif op == "decode":
        S = _log(rng, 1, 131072)
        c.update(S=S, B=_log(rng, 1, max(1, min(64, 131072 // S))), acc=rng.random() < 0.5)
        if rng.random() < 0.5:
            c.update(window=_log(rng, 1, S + 100), sinks=rng.randint(0, 40))
    elif op == "prefill":
        T = _log(rng, 1, 4096)
        S = T + (_log(rng, 1, 8192) if rng.random() < 0.5 else 0)
        S = max(T, min(S, (1 << 29) // (T * hq)))
        c.update(T=T, S=S, B=_log(rng, 1, max(1, min(8, (1 << 29) // (T * S * hq)))))
        if rng.random() < 0.5:
            c.update(window=_log(rng, 1, S + 100), sinks=rng.randint(0, 40))
    else:
        S = _log(rng, 64, 131072)
        budget = _log(rng, 16, S)
        sinks = rng.randint(0, 8)
        c.update(S=S, B=_log(rng, 1, max(1, min(32, 131072 // S))), budget=budget, sinks=sinks,
                 recent=rng.randint(0, budget - sinks))
    return c


def _lens(c):
    """Cached rows of each sequence: S, and for a batch a spread of lengths below it."""
    return [max(1, c["S"] - (c["S"] * b) // (c["B"] + 1) - 7 * (b % 3) * (b > 0)) for b in range(c["B"])]


def _chunks(c):
    """New rows of each sequence (the last ones of its cache)."""
    return [max(1, min(n, c["T"] - (c["T"] * b) // (2 * c["B"]))) for b, n in enumerate(_lens(c))]


def _visible(pos, window, sinks):
    """Keys that the query at row `pos` sees."""
    return pos + 1 if not window or window > pos else window + min(sinks, pos + 1 - window)


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------

def _quantized(x):
    g = x.reshape(x.shape[0], -1, 32)
    m = g.abs().amax(-1).clamp_min(1e-12)
    return torch.floor(0.5 + 127.0 * (g / m[..., None])).to(torch.int8).reshape(x.shape), m


def prepare(case, seed):
    c = case
    d = torch.device("cuda")
    g = torch.Generator(device=d)
    g.manual_seed(seed)
    B, P, hq, hk, hd = c["B"], c["page"], c["hq"], c["hk"], c["hd"]
    lens = _lens(c)
    pages = -(-c["S"] // P)                            # pages a sequence's table holds
    keep = -(-c["budget"] // P) if c["op"] == "evict" else 0
    pool = B * (pages + keep) + 3                      # some pages belong to nobody
    order = torch.randperm(pool, device=d, generator=g).to(torch.int32)
    s = dict(c)
    s["table"] = order[:B * pages].reshape(B, pages).contiguous()
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device=d)
    fill = c["op"] != "prep"

    def cache():
        if fill:
            x = torch.randn(pool * P, hk * hd, device=d, generator=g)
            q, m = _quantized(x)
        else:
            q = torch.zeros(pool * P, hk * hd, dtype=torch.int8, device=d)
            m = torch.zeros(pool * P, hk * hd // 32, device=d)
        return q.reshape(pool, P, hk * hd), m.reshape(pool, P, hk * hd // 32).contiguous()

    kq, ks = cache()
    vq, vs = cache()
    s["kv"] = (kq, ks, vq, vs)
    if c["op"] == "prep":
        rows = [(b, n - t + i) for b, (n, t) in enumerate(zip(lens, _chunks(c))) for i in range(t)]
        idx = torch.tensor(rows, dtype=torch.int32)
        s["seq"], s["slot"] = idx[:, 0].contiguous().to(d), idx[:, 1].contiguous().to(d)
        # rotary positions: the rows' own, and far ones (a cache that was evicted keeps counting)
        s["pos"] = s["slot"] + torch.randint(0, 100000, (1,), device=d, generator=g).to(torch.int32)
        n = len(rows)
        s["q"] = torch.randn(n, hq * hd, device=d, generator=g) * 2
        s["k"] = torch.randn(n, hk * hd, device=d, generator=g) * 2
        s["v"] = torch.randn(n, hk * hd, device=d, generator=g)
        s["qw"] = (1 + 0.2 * torch.randn(hd, device=d, generator=g)).to(torch.float16)
        s["kw"] = (1 + 0.2 * torch.randn(hd, device=d, generator=g)).to(torch.float16)
    elif c["op"] == "decode":
        s["q"] = torch.randn(B, hq * hd, device=d, generator=g) * 1.5
        s["weights"] = torch.rand(B, hk, pages * P, device=d, generator=g) if c["acc"] else None
    elif c["op"] == "prefill":
        ts = _chunks(c)
        cu = [sum(ts[:b]) for b in range(B + 1)]
        s["cu"] = torch.tensor(cu, dtype=torch.int32, device=d)
        s["most"] = max(ts)
        s["q"] = torch.randn(cu[-1], hq * hd, device=d, generator=g) * 1.5
    else:
        s["new_table"] = order[B * pages:B * (pages + keep)].reshape(B, keep).contiguous()
        # accumulated weights are heavy-tailed: a few rows hold most of them
        s["weights"] = torch.exp(2 * torch.randn(B, hk, pages * P, device=d, generator=g))
    return s


# --------------------------------------------------------------------------
# plain forms
# --------------------------------------------------------------------------

def _rows(table, slots, page):
    """Pool rows of cache rows `slots` [B, n]."""
    return torch.gather(table.long(), 1, slots // page) * page + slots % page


def _dequantized(q, m, rows, hk, hd):
    """f32 [B, n, hk, hd] of the pool rows [B, n]."""
    x = q.reshape(-1, hk, hd // 32, 32)[rows].float() * (m.reshape(-1, hk, hd // 32, 1)[rows] / 127.0)
    return x.reshape(*rows.shape, hk, hd)


def _seen(key, pos, window, sinks):
    """Whether the query at row `pos` sees row `key`."""
    ok = key <= pos
    return ok & ((pos - key < window) | (key < sinks)) if window else ok


def _softmax(x, ok):
    x = torch.where(ok, x, torch.full_like(x, -torch.inf))
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(top == -torch.inf, torch.zeros_like(top), top))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total == 0, torch.ones_like(total), total)


def _cache_of(s):
    cap = s["table"].shape[1] * s["page"]
    slots = torch.arange(cap, device=s["table"].device).expand(s["B"], cap)
    rows = _rows(s["table"], slots, s["page"])
    kq, ks, vq, vs = s["kv"]
    k = _dequantized(kq, ks, rows, s["hk"], s["hd"]).permute(0, 2, 3, 1)     # [B, hk, hd, cap]
    v = _dequantized(vq, vs, rows, s["hk"], s["hd"]).permute(0, 2, 1, 3)     # [B, hk, cap, hd]
    return slots, k, v


def _norm_rotate(x, w, pos, heads, hd):
    """Head norm and rotation in 64 bits (angles of far positions; cache bytes next to a border), f32 out."""
    x = x.double().reshape(-1, heads, hd)
    eps = float(torch.tensor(EPS, dtype=torch.float32))
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
    f = torch.arange(hd // 2, dtype=torch.float64, device=x.device)
    a = (pos.double()[:, None] * THETA ** (-2.0 * f / hd))[:, None, :]
    lo, hi = y[..., :hd // 2], y[..., hd // 2:]
    y = torch.cat([lo * torch.cos(a) - hi * torch.sin(a), hi * torch.cos(a) + lo * torch.sin(a)], -1)
    return y.float().reshape(y.shape[0], heads * hd)


def _plain_prep(s):
    hq, hk, hd, P = s["hq"], s["hk"], s["hd"], s["page"]
    qr = _norm_rotate(s["q"], s["qw"], s["pos"], hq, hd)
    kr = _norm_rotate(s["k"], s["kw"], s["pos"], hk, hd)
    slot = s["slot"].long()
    rows = s["table"][s["seq"].long(), slot // P].long() * P + slot % P
    kq, ks, vq, vs = s["kv"]
    k8, km = _quantized(kr)
    v8, vm = _quantized(s["v"])
    kq.view(-1, hk * hd)[rows] = k8
    ks.view(-1, hk * hd // 32)[rows] = km
    vq.view(-1, hk * hd)[rows] = v8
    vs.view(-1, hk * hd // 32)[rows] = vm
    return qr


def _plain_decode(s):
    B, hq, hk, hd = s["B"], s["hq"], s["hk"], s["hd"]
    slots, k, v = _cache_of(s)
    ok = _seen(slots, s["lens"].long()[:, None] - 1, s["window"], s["sinks"])[:, None, None, :]
    p = _softmax(torch.matmul(s["q"].reshape(B, hk, hq // hk, hd), k) / math.sqrt(hd), ok)
    if s["weights"] is not None:
        s["weights"] += p.sum(2)
    return torch.matmul(p, v).reshape(B, hq * hd)


def _plain_prefill(s):
    B, hq, hk, hd, T = s["B"], s["hq"], s["hk"], s["hd"], s["most"]
    slots, k, v = _cache_of(s)
    cu = s["cu"].long()
    n = cu[1:] - cu[:-1]
    i = torch.arange(T, device=cu.device)
    q = s["q"][torch.clamp(cu[:-1, None] + i, max=s["q"].shape[0] - 1)]                     # [B, T, hq*hd]
    q = q.reshape(B, T, hk, hq // hk, hd).permute(0, 2, 3, 1, 4).reshape(B, hk, -1, hd)     # head, then query
    pos = (s["lens"].long() - n)[:, None] + i
    ok = _seen(slots[:, None, :], pos[:, :, None], s["window"], s["sinks"])                 # [B, T, cap]
    ok = ok[:, None, None].expand(B, 1, hq // hk, T, ok.shape[-1]).reshape(B, 1, -1, ok.shape[-1])
    p = _softmax(torch.matmul(q, k) / math.sqrt(hd), ok)
    o = torch.matmul(p, v).reshape(B, hk, hq // hk, T, hd).permute(0, 3, 1, 2, 4).reshape(B, T, hq * hd)
    t = torch.arange(s["q"].shape[0], device=cu.device)
    b = torch.searchsorted(cu, t, right=True) - 1
    return o[b, t - cu[b]].to(torch.bfloat16)


def _plain_evict(s):
    B, hk, P, budget = s["B"], s["hk"], s["page"], s["budget"]
    table, fresh, weights = s["table"], s["new_table"], s["weights"]
    cap, new_cap = table.shape[1] * P, fresh.shape[1] * P
    d = table.device
    n = s["lens"].long()[:, None]
    slots = torch.arange(cap, device=d).expand(B, cap)
    score = weights.double().sum(1)
    score = torch.where((slots < s["sinks"]) | (slots >= n - s["recent"]), torch.full_like(score, torch.inf), score)
    score = torch.where(slots < n, score, torch.full_like(score, -torch.inf))
    best = torch.sort(score, dim=1, descending=True, stable=True).indices[:, :budget]
    left = torch.clamp(n, max=budget)                                                     # rows that stay
    at = torch.arange(best.shape[1], device=d).expand(B, -1)
    best = torch.sort(torch.where(at < left, best, torch.full_like(best, cap)), dim=1).values
    kept = torch.full((B, budget), -1, dtype=torch.int32, device=d)
    kept[:, :best.shape[1]] = torch.where(at < left, best, torch.full_like(best, -1)).to(torch.int32)
    dst = _rows(fresh, at, P)
    src = torch.where(at < left, _rows(table, torch.clamp(best, max=cap - 1), P), dst)    # past the end: itself
    kq, ks, vq, vs = (x.view(-1, x.shape[-1]) for x in s["kv"])
    kq[dst], ks[dst], vq[dst], vs[dst] = kq[src], ks[src], vq[src], vs[src]
    moved = torch.gather(weights, 2, torch.clamp(best, max=cap - 1)[:, None].expand(B, hk, best.shape[1]))
    out = torch.zeros(B, hk, new_cap, device=d)
    out[:, :, :best.shape[1]] = torch.where((at < left)[:, None], moved, torch.zeros_like(moved))
    return kept, left[:, 0].to(torch.int32), out


# --------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------

def run(state):
    s = state
    kq, ks, vq, vs = s["kv"]
    if s["op"] == "prep":
        if own:
            import tabinfer_b200 as tb
            qr = tb.attn_prep_paged_q8(s["q"], s["k"], s["v"], s["qw"], s["kw"], s["kv"], s["table"], s["seq"],
                                       s["slot"], s["pos"], s["hq"], s["hk"], s["hd"], THETA, EPS)
        else:
            qr = _plain_prep(s)
        # the cache's bytes and scales: the rows are formed in 64 bits before they are rounded, so a byte is
        # defined by the operator and has to be equal
        return {"qr": qr, "Kq": kq, "Ks": ks, "Vq": vq, "Vs": vs}
    if s["op"] == "decode":
        if own:
            import tabinfer_b200 as tb
            out = tb.attention_decode_paged_q8(s["q"], s["kv"], s["table"], s["lens"], s["hq"], s["hk"], s["hd"],
                                               window=s["window"], sinks=s["sinks"], weights=s["weights"])
        else:
            out = _plain_decode(s)
        return {"out": out, "weights": s["weights"]}
    if s["op"] == "prefill":
        if own:
            import tabinfer_b200 as tb
            return tb.attention_prefill_paged_q8(s["q"], s["kv"], s["table"], s["cu"], s["lens"], s["hq"], s["hk"],
                                                 s["hd"], window=s["window"], sinks=s["sinks"])
        return _plain_prefill(s)
    if own:
        import tabinfer_b200 as tb
        kept, lens, weights = tb.kv_evict_paged_q8(s["kv"], s["table"], s["lens"], s["weights"], s["new_table"],
                                                   s["budget"], s["sinks"], s["recent"], s["hk"], s["hd"])
    else:
        kept, lens, weights = _plain_evict(s)
    return {"kept": kept, "lens": lens, "weights": weights, "Kq": kq, "Ks": ks, "Vq": vq, "Vs": vs}


def work(case):
    c = case
    hq, hk, hd = c["hq"], c["hk"], c["hd"]
    row = 2 * hk * hd * (1 + 4 / 32)                   # K and V bytes of one cache row
    if c["op"] == "prep":
        n = sum(_chunks(c))
        return {"bytes": n * (4 * (2 * hq + 2 * hk) * hd + row + 12) + 4 * hd, "flops": n * (8 * (hq + hk) + 4 * 2 * hk) * hd}
    if c["op"] == "decode":
        seen = sum(_visible(n - 1, c["window"], c["sinks"]) for n in _lens(c))
        return {"bytes": seen * (row + (8 * hk if c["acc"] else 0)) + c["B"] * 8 * hq * hd, "flops": 4 * hd * hq * seen}
    if c["op"] == "prefill":
        w, k = c["window"], c["sinks"]
        pairs = keys = 0
        for n, t in zip(_lens(c), _chunks(c)):
            pairs += sum(_visible(p, w, k) for p in range(n - t, n))
            first = max(0, n - t - w + 1) if w else 0  # the first key that the chunk's window reaches
            keys += n - first + min(k, first)
        return {"bytes": keys * row + sum(_chunks(c)) * hq * hd * (4 + 2), "flops": 4 * hd * hq * pairs}
    kept = sum(min(n, c["budget"]) for n in _lens(c))
    return {"bytes": sum(_lens(c)) * 4 * hk + kept * (2 * row + 4 * hk + 4), "flops": sum(_lens(c)) * hk}


# --------------------------------------------------------------------------
# the definitions in 64 bits, one row, head or sequence at a time
# --------------------------------------------------------------------------

def _exact_rows(q, m, page_ids, page, n, h, hd):
    """f64 [n, hd] of head h of the first n rows of a sequence whose pages are page_ids."""
    x = q[page_ids].reshape(-1, q.shape[-1])[:n, h * hd:(h + 1) * hd].double()
    sc = m[page_ids].reshape(-1, m.shape[-1])[:n, h * hd // 32:(h + 1) * hd // 32].double()
    return x * sc.repeat_interleave(32, dim=1) / 127.0


def exact(case, seed):
    c = case
    s = prepare(case, seed)
    B, P, hq, hk, hd, W, sinks = c["B"], c["page"], c["hq"], c["hk"], c["hd"], c["window"], c["sinks"]
    lens = _lens(c)
    kq, ks, vq, vs = s["kv"]
    if c["op"] == "prep":
        freq = torch.exp(-torch.arange(hd // 2, device="cuda").double() * (2.0 * math.log(THETA) / hd))
        angle = s["pos"].double().unsqueeze(1) * freq
        turn = torch.complex(torch.cos(angle), torch.sin(angle))

        def rotated(x, w, heads):
            x = x.double().view(-1, heads, hd)
            x = x * (x.square().sum(-1, keepdim=True) / hd + float(torch.tensor(EPS, dtype=torch.float32))).rsqrt()
            x = x * w.double()
            z = torch.complex(x[..., :hd // 2].contiguous(), x[..., hd // 2:].contiguous()) * turn.unsqueeze(1)
            return torch.cat((z.real, z.imag), dim=-1).reshape(-1, heads * hd)

        where = [int(p) * P for p in s["table"].flatten().tolist()]
        per = s["table"].shape[1]
        rows = torch.tensor([where[b * per + r // P] + r % P for b, r in zip(s["seq"].tolist(), s["slot"].tolist())],
                            device="cuda")
        kr = rotated(s["k"], s["kw"], hk)
        out = {"qr": rotated(s["q"], s["qw"], hq), "Kq": None, "Vq": None}
        for name, pool, x in (("Ks", ks, kr), ("Vs", vs, s["v"].double())):
            m = pool.double().view(-1, hk * hd // 32)
            m[rows] = x.abs().view(len(rows), -1, 32).max(-1).values
            out[name] = m.view(pool.shape)
        return out
    if c["op"] == "evict":
        return None                                     # a choice and copies: nothing is computed in floating point
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    weights = s["weights"].double() if c["op"] == "decode" and c["acc"] else None
    ts = _chunks(c) if c["op"] == "prefill" else [1] * B
    first = 0
    for b in range(B):
        n, t = lens[b], ts[b]
        ids = s["table"][b].long()
        pos = torch.arange(n - t, n, device="cuda")
        key = torch.arange(n, device="cuda")
        hidden = key[None, :] > pos[:, None]
        if W:
            hidden |= (pos[:, None] - key[None, :] >= W) & (key[None, :] >= sinks)
        for h in range(hk):
            k = _exact_rows(kq, ks, ids, P, n, h, hd)
            v = _exact_rows(vq, vs, ids, P, n, h, hd)
            for j in range(h * (hq // hk), (h + 1) * (hq // hk)):
                x = s["q"][first:first + t, j * hd:(j + 1) * hd].double() @ k.T * hd ** -0.5
                p = torch.softmax(x.masked_fill_(hidden, -torch.inf), dim=-1)
                out[first:first + t, j * hd:(j + 1) * hd] = p @ v
                if weights is not None:
                    weights[b, h, :n] += p[0]
        first += t
    return out if c["op"] == "prefill" else {"out": out, "weights": weights}
