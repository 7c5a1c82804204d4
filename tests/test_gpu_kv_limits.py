"""The paged cache's operators at the ends of their ranges: logits past fp32, long chunks and many
heads, and calls that the host cuts into several launches (cached heads, sequences or rows at a time), against
the definitions in 64 bits. Tolerances as in tests/test_gpu_kv_more.py."""
import numpy as np
import pytest

from conftest import assert_bitexact
from test_gpu_kv_cache import F, HD
from test_gpu_kv_more import More, _weights, soft

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


# ---- keys whose scale is no number ----

@pytest.mark.parametrize("new", [1, 40, 300])
@pytest.mark.parametrize("where", ["own", "part"])
@pytest.mark.parametrize("scale", [np.nan, np.inf])
def test_shared_bad_scale(sdq_dev, new, where, scale):
    """A key whose scale is NaN makes the rows NaN that see it, be it alone in its part or among the
    rows' own keys: as kv_attention of the same tokens through one table. An infinite one does where the
    logit is not -infinity."""
    c = More(sdq_dev, [new, new], [new if where == "part" else 1, new + 3], 2, 16, seed=49)
    c.share([0, 1, 2], [16, 16])
    if where == "own":
        c.table[0, 1:] = -1
        c.ks[c.table[0, 0], :, 0] = scale
    else:  # alone: the other fifteen have no page
        c.s_lens[0] = 1
        c.ks[c.s_table[0, 0], :, 0] = scale
    c.up_shared()
    q = c.queries(4)
    key = (c.k[c.table[0, 0], :, 0] if where == "own" else c.k[c.s_table[0, 0], :, 0]).astype(np.float64)
    got, same = (c.torch.full((c.T, 512), -3.0, device=c.dev) for _ in range(2))
    c.sdq.kv_attention_shared(c.cache, c.shared, c.batch, c.t(q), got, 4)
    got = got.cpu().numpy().reshape(-1, 4, HD)
    for r in range(new):
        placed = c.lens[0] - new + r >= 0
        for h in range(4):
            dot = q[r, h * HD:(h + 1) * HD].astype(np.float64) @ key[h // 2]
            lost = placed and (np.isnan(scale) or dot >= 0)
            assert np.isnan(got[r, h]).all() if lost else np.isfinite(got[r, h]).all(), (r, h, dot)
    c.s_lens[0] = 0 if where == "part" else 16
    c.ks[~np.isfinite(c.ks)] = F(0.01)
    c.up_shared()
    c.sdq.kv_attention_shared(c.cache, c.shared, c.batch, c.t(q), same, 4)
    assert_bitexact(got.reshape(-1, 512)[new:], same.cpu().numpy()[new:], "the other sequence")


@pytest.mark.parametrize("new", [1, 40, 70, 300, 1100])
def test_bad_row_over_an_infinite_scale(sdq_dev, new):
    """A row of NaN that sees a single key is NaN, also where that key's scale is infinite and what is
    left of the row would have a logit of -infinity."""
    c = More(sdq_dev, [new], [1], 1, 16, seed=50)
    c.share([0, 1], [0])
    key = c.k[c.table[0, 0], 0, 0]
    c.ks[c.table[0, 0], 0, 0] = np.inf
    c.up_shared()
    q = np.repeat(np.where(key > 0, -1, 1)[None], new, 0).astype(F)
    q[-1, 5] = np.nan
    for call in (lambda o: c.sdq.kv_attention(c.cache, c.batch, c.t(q), o, 1),
                 lambda o: c.sdq.kv_cross_attention(c.cache, c.batch, c.t(q), o, 1),
                 lambda o: c.sdq.kv_attention_shared(c.cache, c.shared, c.batch, c.t(q), o, 1)):
        out = c.torch.full((new, HD), -3.0, device=c.dev)
        call(out)
        got = out.cpu().numpy()
        assert np.isnan(got[-1]).all() and (got[:-1] == 0).all()


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


# ---- calls of several launches ----

def _shared_case(dev, new, lens, kvh, s_start, parts, seed):
    c = More(dev, new, lens, kvh, 16, seed=seed, first=1, behind=1)
    c.share(s_start, parts)
    return c


def _check_shared_rows(c, heads, places):
    """kv_attention_shared, causal, at (sequence, its row, query head)."""
    import torch

    g = torch.Generator(device=c.dev).manual_seed(c.T)
    q = torch.randn((c.T, heads * HD), generator=g, device=c.dev).mul_(1.5)
    out = torch.full((c.T, heads * HD), -3.0, device=c.dev)
    c.sdq.kv_attention_shared(c.cache, c.shared, c.batch, q, out, heads)
    assert (out[0] == -3).all() and (out[-1] == -3).all()
    assert bool(torch.isfinite(out).all())
    for s, r, h in places:
        kh, n = h // (heads // c.kvh), c.new[s]
        k, v, ok = c.values(s, kh)
        pk, pv, pok = c.part(s, kh)
        see = np.concatenate([pok, ok & (np.arange(len(k)) <= len(k) - n + r)])[None]
        at = c.start[s] + r, slice(h * HD, (h + 1) * HD)
        want, tol, _, _ = soft(q[at].cpu().numpy()[None], np.concatenate([pk, k]),
                               np.concatenate([pv, v]), see, HD**-0.5)
        c.close(out[at].cpu().numpy()[None], want, tol)


@pytest.mark.parametrize("nseq,new,parts", [(2, 8500, [300, 4099]), (1000, 17, [2050, 0, 33])])
def test_shared_heads_at_a_time(sdq_dev, nseq, new, parts):
    """More rows than 512 MiB of shares hold for all heads: seven of eight cached heads, then one."""
    rng = np.random.default_rng(nseq)
    rows = [new] * nseq if nseq < 3 else list(rng.integers(new - 3, new + 4, nseq))
    lens = [int(n + rng.integers(0, 60)) for n in rows]
    s_start = [0, 1, 2] if nseq < 3 else [0, 500, 600, 990]
    c = _shared_case(sdq_dev, rows, lens, 8, s_start, parts, seed=42)
    assert 7 * sum(rows) * 4 * 2 * 520 <= 2**29 < 8 * sum(rows) * 4 * 2 * 520
    places = [(s, r, h) for s in (0, nseq // 2, nseq - 1) for r in (0, rows[s] // 2, rows[s] - 1)
              for h in (0, 1, 26, 27, 28, 31)]
    _check_shared_rows(c, 32, places)


def test_shared_rows_of_one_head(sdq_dev):
    """Query heads of one cached head, more than 2^22 rows: the join takes several launches."""
    rng = np.random.default_rng(3)
    rows = list(rng.integers(60, 141, 1400))
    c = _shared_case(sdq_dev, rows, [int(n + rng.integers(0, 20)) for n in rows], 1, [0, 700, 1390],
                     [60, 17], seed=43)
    assert sum(rows) * 32 > 2**22
    places = [(s, r, h) for s in (0, 699, 700, 1300, 1395, 1399) for r in (0, rows[s] - 1) for h in (0, 31)]
    _check_shared_rows(c, 32, places)


def test_weights_sequences_at_a_time(sdq_dev):
    """More pairs of a sequence and cached head than a grid takes: 512 sequences of 64 heads, then the
    others, long ones (whose rows are cut into ranges) on both sides."""
    import torch

    nseq, kvh, G = 516, 64, 2
    new = [64] * nseq
    for s in (0, 511, 512, 515):
        new[s] = 1100
    new[514] = 0
    lens = [n + 9 if s % 2 else n for s, n in enumerate(new)]
    need = [-(-n // 32) for n in lens]
    pages = sum(need) + 1
    g = torch.Generator(device=sdq_dev).manual_seed(44)
    codes = lambda: torch.randint(-127, 128, (pages, kvh, 32, HD), generator=g, device=sdq_dev,  # noqa: E731
                                  dtype=torch.int8)
    rand = lambda *s: torch.rand(s, generator=g, device=sdq_dev)  # noqa: E731
    c = More(sdq_dev, [1], [1], 1, 16)  # the definitions' home
    cache = c.sdq.KvCache(codes(), 0.012 * (0.5 + rand(pages, kvh, 32)), codes(),
                          0.02 * (0.5 + rand(pages, kvh, 32)))
    table = np.full((nseq, max(need)), -1, np.int32)
    ids = np.random.default_rng(44).permutation(pages)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = ids[at:at + n]
        at += n
    start = np.concatenate([[0], np.cumsum(new)])
    T = int(start[-1])
    batch = c.sdq.KvBatch(c.t(start.astype(np.int32)), c.t(np.array(lens, np.int32)), c.t(table))
    q = torch.randn((T, kvh * G * HD), generator=g, device=sdq_dev).mul_(1.5)
    w = rand(pages, kvh, 32)
    before = w.clone()
    out = torch.empty_like(q)
    c.sdq.kv_attention_weights(cache, batch, w, q, out, kvh * G)
    assert bool(torch.isfinite(w).all())
    assert torch.equal(w[ids[-1]], before[ids[-1]])  # no sequence's page
    same = torch.empty_like(q)
    c.sdq.kv_attention(cache, batch, q, same, kvh * G)
    assert torch.equal(out, same)
    for s in (0, 1, 300, 511, 512, 513, 515):
        n, L = new[s], lens[s]
        p = np.arange(L)
        see = p[None] <= (L - n + np.arange(n))[:, None]
        for h in (0, 31, 63):
            pg, slot = torch.from_numpy(table[s, p // 32].astype(np.int64)), torch.from_numpy(p % 32)
            host = lambda t: t[pg.to(sdq_dev), h, slot.to(sdq_dev)].cpu().numpy().astype(np.float64)  # noqa: E731
            k, v = host(cache.k) * host(cache.ks)[:, None], host(cache.v) * host(cache.vs)[:, None]
            total, off = np.zeros(L), np.zeros(L)
            for j in range(G * h, G * h + G):
                x = q[start[s]:start[s + 1], j * HD:(j + 1) * HD].cpu().numpy()
                _, _, wt, rel = soft(x, k, v, see, HD**-0.5)
                total += wt.sum(0)
                off += (wt * rel).sum(0)
            total += np.where(p < L - n, host(before), 0)
            c.close(host(w), total, off + (n * G / 16 + 16) * 2.0**-24 * total + 1e-37)


def test_evict_long_sequences_at_a_time(sdq_dev):
    """Tables of 2^20 tokens, nearly all unused, of 64 heads: two sequences of three at a time."""
    c = More(sdq_dev, [0] * 3, [3000, 17000, 700], 64, 256, seed=45)
    table = np.full((3, 4096), -1, np.int32)
    table[:, :c.most] = c.table
    c.table, c.most = table, 4096
    c.up()
    w = np.exp(2 * c.rng.standard_normal((c.pages, 64, 256))).astype(F)
    c.check_evict(w, 500, 3, 40)


def test_evict_sequences_at_a_time(sdq_dev):
    """33000 sequences of 64 heads, the same few pages' tokens: 32768 of them, then the others."""
    import torch

    nseq, kvh, keep = 33000, 64, 6
    c = More(sdq_dev, [0] * 5, [16, 9, 0, 31, 6], kvh, 16, seed=46)
    w = c.rng.integers(0, 4, (c.pages, kvh, 16)).astype(F)
    want, want_lens = c.evict64(w, keep, 1, 2)
    which = np.random.default_rng(46).integers(0, 5, nseq)
    i32 = lambda a: c.t(np.asarray(a, np.int32))  # noqa: E731
    batch = c.sdq.KvBatch(i32(np.zeros(nseq + 1)), i32(np.array(c.lens)[which]), i32(c.table[which]))
    free = 10
    shape = (c.pages + free, kvh, 16)
    pool = c.sdq.KvCache.empty(shape[0], 16, kvh)
    for name in ("k", "v", "ks", "vs"):
        getattr(pool, name).zero_()
        getattr(pool, name)[:c.pages] = getattr(c.cache, name)
    tw = torch.zeros(shape, device=sdq_dev)
    tw[:c.pages] = c.t(w)
    # most go nowhere; ten sequences on either side of the launches' border have a page
    live = [0, 1, 2, 32766, 32767, 32768, 32769, 32770, 32998, 32999]
    to = np.full((nseq, 1), -1, np.int32)
    to[live, 0] = c.pages + np.arange(free)
    lens = torch.full((nseq,), -9, dtype=torch.int32, device=sdq_dev)
    kept = torch.full((nseq, kvh, keep), -9, dtype=torch.int32, device=sdq_dev)
    c.sdq.kv_evict(pool, batch, tw, i32(to), lens, kept, first=1, last=2)
    assert_bitexact(lens.cpu().numpy(), want_lens[which], "lens")
    assert_bitexact(kept.cpu().numpy(), want[which], "kept")
    for i, s in enumerate(live):
        n, src = want_lens[which[s]], which[s]
        for h in (0, 63):
            pos = want[src, h, :n]
            at = c.table[src, pos // 16], h, pos % 16
            for got, x in ((pool.k, c.k), (pool.vs, c.vs), (tw, w)):
                assert_bitexact(got[c.pages + i, h, :n].cpu().numpy(), x[at])
    assert torch.equal(tw[:c.pages], c.t(w))
