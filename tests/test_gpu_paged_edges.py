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
