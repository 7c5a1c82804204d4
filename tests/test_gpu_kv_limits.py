"""The paged cache's operators at the ends of their ranges: logits past fp32, long chunks and many
heads, against the definitions in 64 bits. Tolerances as in tests/test_gpu_kv_more.py."""
import numpy as np
import pytest

from conftest import assert_bitexact
from test_gpu_kv_cache import F, HD
from test_gpu_kv_more import More, _weights

pytestmark = pytest.mark.gpu


# ---- counted weights: logits past fp32's range ----

def _counted(c, q, w, heads, causal, scale=None):
    tw, out = c.t(w), c.torch.zeros((c.T, heads * HD), device=c.dev)
    c.sdq.kv_attention_weights(c.cache, c.batch, tw, c.t(q), out, heads, causal=causal, scale=scale)
    return tw.cpu().numpy(), out.cpu().numpy()


@pytest.mark.parametrize("new,L", [(12, 40), (200, 700), (1100, 1100)])
@pytest.mark.parametrize("causal", [True, False])
def test_weights_of_overflowing_rows(sdq_dev, new, L, causal):
    """Finite rows whose logits are past fp32's range have no softmax and add nothing, whichever form
    counts; the other rows add what they add beside rows of NaN, bit for bit."""
    c = More(sdq_dev, [new], [L], 1, 16, seed=40)
    q, w = c.queries(2), c.rng.uniform(0, 0.1, (c.pages, 1, 16)).astype(F)
    lost = np.zeros((new, 2), bool)
    lost[[0, new // 2, new - 1], [0, 1, 0]] = True
    lost[new // 3] = True
    first = c.k[c.table[0, 0], 0, 0]  # a key that every row sees
    for r, j in np.argwhere(lost):
        q[r, j * HD:(j + 1) * HD] = F(3e38) * np.where(first < 0, -1, 1)
    got, out = _counted(c, q, w, 2, causal)
    assert np.isnan(out.reshape(new, 2, HD)[lost]).all()
    bad = q.reshape(new, 2, HD).copy()
    bad[lost] = np.nan
    bad = bad.reshape(new, 2 * HD)
    assert_bitexact(got, _counted(c, bad, w, 2, causal)[0], "beside rows of NaN")
    c.close(got, *c.weights64(w, bad, 2, HD**-0.5, causal))


@pytest.mark.parametrize("new", [5, 45, 90])
def test_weights_of_a_huge_scale(sdq_dev, new):
    """A key's scale times the softmax's passes fp32's range, the rows' logits do not (their queries
    are next to nothing): every key gets the same. Rows that fill a tile up add nothing."""
    c = More(sdq_dev, [new], [700], 1, 16, seed=41)
    c.ks[c.table[0, 3], 0, 5] = F(3e37)
    c.up()
    q = np.full((new, 2 * HD), F(1e-45))
    got, _ = _counted(c, q, np.zeros((c.pages, 1, 16), F), 2, False, scale=10.0)
    p = np.arange(700)
    got = got[c.table[0, p // 16], 0, p % 16]
    want = 2 * new / 700
    # logits within 1e-45 * 127 * 128 * 3e37 * 10 * log2(e) < 0.01 of 0, the others' exactly 0 here
    assert (np.abs(got - want) <= 0.01 * want).all(), (got.min(), got.max(), want)


# ---- eviction: chunks of more tokens than a workgroup's registers, and many heads ----

@pytest.mark.parametrize("kind", ["spread", "ties", "odd"])
def test_evict_longer_chunks(sdq_dev, kind):
    """A table of 2^22 tokens, most of it unused: chunks of 65536, read in several rounds."""
    c = More(sdq_dev, [0] * 3, [150001, 65536, 70000], 2, 256, seed=47)
    table = np.full((3, 1 << 14), -1, np.int32)
    table[:, :c.most] = c.table
    c.table, c.most = table, 1 << 14
    c.up()
    c.check_evict(_weights(c, kind), 20000, 3, 100)


class Sparse(More):
    def evict64(self, w, keep, first, last):
        """More.evict64 where few tokens have a page."""
        kept = np.full((len(self.lens), self.kvh, keep), -1, np.int32)
        lens = np.zeros(len(self.lens), np.int32)
        for s, L in enumerate(self.lens):
            pages = np.flatnonzero((self.table[s] >= 0) & (self.table[s] < self.pages))
            p = (pages[:, None] * self.page + np.arange(self.page)).ravel()
            p = p[p < L]
            lens[s] = min(keep, len(p))
            must = (p < first) | (p >= L - last)
            x = w[self.table[s, p // self.page], :, p % self.page].astype(np.float64)
            for h in range(self.kvh):
                order = np.lexsort((p, np.where(must, 0, -x[:, h]), ~must))[:keep]
                kept[s, h, :len(order)] = np.sort(p[order])
        return kept, lens


def test_evict_many_heads(sdq_dev):
    """1024 cached heads over a table of 2^20 tokens: fewer and longer chunks, and scratch of no more
    than 256 MiB."""
    import torch

    c = Sparse(sdq_dev, [0, 0], [90, 40], 1024, 16, seed=48)
    table = np.full((2, 1 << 16), -1, np.int32)
    for s, at in ((0, [0, 1, 1023, 1024, 9000, 20001]), (1, [0, 7168, 14336])):  # tokens far apart
        table[s, at] = c.table[s, :len(at)]
    c.table, c.most, c.lens = table, 1 << 16, [20001 * 16 + 10, 14336 * 16 + 3]
    c.up()
    w = _weights(c, "ties")
    with torch.cuda.stream(torch.cuda.Stream()):  # a workspace of its own
        torch.cuda.synchronize()
        before = torch.cuda.mem_get_info()[0] + torch.cuda.memory_reserved()
        c.check_evict(w, 33, 2, 15)
        torch.cuda.synchronize()
        used = before - torch.cuda.mem_get_info()[0] - torch.cuda.memory_reserved()
    assert used <= 2**28 + 2**24, used
