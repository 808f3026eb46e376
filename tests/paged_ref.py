"""Plain 64-bit forms of the paged int8 KV cache operators, one sequence and head at a
time (test infrastructure; torch CPU tensors)."""
import torch


def quantize(x):
    """f32 [n, w] -> (int8, f32 scale a 32-group): the cache's bytes."""
    g = x.reshape(x.shape[0], -1, 32)
    m = g.abs().amax(-1).clamp_min(1e-12)
    return torch.floor(0.5 + 127.0 * (g / m[..., None])).to(torch.int8).reshape(x.shape), m


class Cache:
    """A random paged cache on the CPU and its copy on the device."""

    def __init__(self, seed, batch, max_pages, page, nKv, hd, spare=3, fill=True, poison=False):
        g = torch.Generator().manual_seed(seed)
        self.g, self.B, self.page, self.nKv, self.hd = g, batch, page, nKv, hd
        n = batch * max_pages + spare
        w = nKv * hd
        self.cap = max_pages * page

        def pool():
            q, m = quantize(torch.randn(n * page, w, generator=g) if fill else torch.zeros(n * page, w))
            return q.reshape(n, page, w), m.reshape(n, page, w // 32)
        (self.Kq, self.Ks), (self.Vq, self.Vs) = pool(), pool()
        order = torch.randperm(n, generator=g).to(torch.int32)
        self.table = order[:batch * max_pages].reshape(batch, max_pages).contiguous()
        self.free = order[batch * max_pages:]

    def rows(self, b, slots):
        """pool rows of cache rows"""
        slots = torch.as_tensor(slots)
        return self.table[b, slots // self.page].long() * self.page + slots % self.page

    def poison_rows(self, b, slots):
        """what may stand in rows that nobody sees: NaN and infinite scales, the lowest byte"""
        r = self.rows(b, slots)
        w = self.nKv * self.hd
        self.Ks.view(-1, w // 32)[r] = float("nan")
        self.Vs.view(-1, w // 32)[r] = float("inf")
        self.Kq.view(-1, w)[r] = -128
        self.Vq.view(-1, w)[r] = -128

    def dev(self):
        return tuple(t.cuda() for t in (self.Kq, self.Ks, self.Vq, self.Vs))

    def head(self, b, n, h):
        """(k, v) f64 [n, hd] of one head"""
        r = self.rows(b, torch.arange(n))
        out = []
        for q, m in ((self.Kq, self.Ks), (self.Vq, self.Vs)):
            x = q.view(-1, self.nKv, self.hd)[r, h].double()
            s = m.view(-1, self.nKv, self.hd // 32)[r, h].double()
            out.append(x * s.repeat_interleave(32, 1) / 127.0)
        return out


def seen(n, pos, window, sinks):
    j = torch.arange(n)
    ok = j <= pos
    return ok & ((pos - j < window) | (j < sinks)) if window else ok


def attend(c, b, q, pos, nHq, window=0, sinks=0):
    """One query (f32 [nHq*hd]) at row pos: (out f64 [nHq, hd], weights f64 [nKv, pos+1],
    the largest sum |q_i k_i| / sqrt(hd) of a seen key, the largest |v| seen)."""
    hd, grp, n = c.hd, nHq // c.nKv, pos + 1
    out = torch.zeros(nHq, hd, dtype=torch.float64)
    w = torch.zeros(c.nKv, max(n, 0), dtype=torch.float64)
    mag, big = 0.0, 0.0
    if n <= 0:
        return out, w, mag, big
    ok = seen(n, pos, window, sinks)
    for h in range(c.nKv):
        k, v = c.head(b, n, h)
        k, v = k[ok], v[ok]
        big = max(big, float(v.abs().max()))
        for g in range(grp):
            x = q.double().reshape(nHq, hd)[h * grp + g]
            p = torch.softmax(k @ x * hd ** -0.5, 0)
            mag = max(mag, float((k.abs() @ x.abs()).max()) * hd ** -0.5)
            out[h * grp + g] = p @ v
            w[h, ok] += p
    return out, w, mag, big


def norm_rope(x, w16, pos, heads, hd, theta, eps):
    """f32 [T, heads*hd] -> the f64 rows before rounding"""
    x = x.double().reshape(-1, heads, hd)
    e = float(torch.tensor(eps, dtype=torch.float32))
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + e) * w16.double()
    f = torch.arange(hd // 2, dtype=torch.float64)
    a = (pos.double()[:, None] * theta ** (-2.0 * f / hd))[:, None, :]
    lo, hi = y[..., :hd // 2], y[..., hd // 2:]
    return torch.cat([lo * a.cos() - hi * a.sin(), hi * a.cos() + lo * a.sin()], -1).reshape(-1, heads * hd)


def evict(weights, n, budget, sinks, recent):
    """Rows of one sequence that stay (ascending); weights f32 [nKv, cap]."""
    if n <= budget:
        return list(range(n))
    score = weights.double().sum(0)
    mid = sorted(range(sinks, n - recent), key=lambda j: (-float(score[j]), j))[:budget - sinks - recent]
    return sorted(list(range(sinks)) + mid + list(range(n - recent, n)))
