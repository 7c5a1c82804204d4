"""The paged cache's operators beyond a sequence's own tokens: cross attention, shared
beginnings, counted weights and eviction, against their definitions in 64 bits over the values
that the cache holds.

Tolerances: of outputs as in tests/test_gpu_kv_cache.py (a logit's error from its products'
magnitudes, the sums over n keys). Of a key's summed weights: each weight is off by its own logit's
error, exp2's and the parts' 2^-20, and its row's denominator's error; the sum over n rows by one
rounding a step, of which a lane makes n / 16, and 16 that stand for the joins and the old sum's."""
import numpy as np
import pytest

from conftest import assert_bitexact
from test_gpu_kv_cache import F, HD, Case

pytestmark = pytest.mark.gpu


def soft(x, k, v, see, scale):
    """Softmax attention of rows x over keys k in 64 bits: output, its tolerance, weights,
    and the weights' relative tolerance."""
    x = x.astype(np.float64)
    t = x @ k.T * scale
    size = np.abs(x) @ np.abs(k).T * abs(scale)
    t = np.where(see, t, -np.inf)
    top = t.max(1, initial=-np.inf, keepdims=True)
    top = np.where(np.isinf(top), 0, top)
    w = np.exp(t - top) * see
    z = w.sum(1, keepdims=True)
    w = w / np.where(z == 0, 1, z)
    err = ((2.0**-22 + 136 * 2.0**-24) * size + 2.0**-21 * np.abs(np.where(see, t, 0))
           + 2.0**-21 * np.abs(top))
    rel = (w * (err + 2.0**-20)).sum(1, keepdims=True) + (len(k) / 8 + 64) * 2.0**-24
    seen = see.any(0)
    return (w @ np.where(seen[:, None], v, 0), 2 * rel * np.abs(v[seen]).max(initial=0), w,
            err + 2.0**-20 + rel)


class More(Case):
    def rows(self, s):
        return slice(self.start[s], self.start[s + 1])

    def own(self, s, h, causal, free=False):
        """Keys and values of sequence s, cached head h, and which of its rows see which."""
        k, v, ok = self.values(s, h)
        n = self.new[s]
        pos = len(k) - n + np.arange(n)
        see = np.broadcast_to(ok[None], (n, len(k))).copy()
        if not free:
            see &= (pos[:, None] >= 0)
            if causal:
                see &= np.arange(len(k))[None] <= pos[:, None]
        return k, v, see

    def close(self, got, want, tol):
        bad = ~(np.abs(got - want) <= tol)
        assert not bad.any(), (np.argwhere(bad)[:3], got[bad][:3], want[bad][:3], tol[bad][:3])

    def queries(self, heads, std=1.5):
        return (self.rng.standard_normal((self.T, heads * HD)) * std).astype(F)

    # ---- cross ----

    def cross64(self, q, heads, scale, fill):
        out = np.full((self.T, heads * HD), fill)
        tol = np.zeros_like(out)
        for s in range(len(self.new)):
            for h in range(heads):
                k, v, see = self.own(s, h // (heads // self.kvh), False, free=True)
                at = self.rows(s), slice(h * HD, (h + 1) * HD)
                out[at], tol[at], _, _ = soft(q[at], k, v, see, scale)
        return out, tol

    def check_cross(self, heads, scale=None, q=None, fill=-3.0):
        q = self.queries(heads) if q is None else q
        out = self.torch.full((self.T, heads * HD), fill, device=self.dev)
        self.sdq.kv_cross_attention(self.cache, self.batch, self.t(q), out, heads, scale=scale)
        got = out.cpu().numpy()
        self.close(got, *self.cross64(q, heads, HD**-0.5 if scale is None else scale, fill))
        return got

    # ---- shared ----

    def share(self, s_start, lens):
        """Parts of their own pages (the pool grows by them)."""
        need = [-(-max(n, 0) // self.page) for n in lens]
        add = sum(need) + 1
        shape = (add, self.kvh, self.page)
        self.k = np.concatenate([self.k, self.rng.integers(-127, 128, shape + (HD,)).astype(np.int8)])
        self.v = np.concatenate([self.v, self.rng.integers(-127, 128, shape + (HD,)).astype(np.int8)])
        self.ks = np.concatenate([self.ks, (0.012 * self.rng.uniform(0.5, 1.5, shape)).astype(F)])
        self.vs = np.concatenate([self.vs, (0.02 * self.rng.uniform(0.5, 1.5, shape)).astype(F)])
        ids = self.pages + self.rng.permutation(add)
        self.pages += add
        self.s_start, self.s_lens = np.array(s_start, np.int32), np.array(lens, np.int32)
        self.s_table = np.full((len(lens), max(need + [1])), -1, np.int32)
        at = 0
        for g, n in enumerate(need):
            self.s_table[g, :n] = ids[at:at + n]
            at += n
        self.up_shared()

    def up_shared(self):
        self.up()
        self.shared = self.sdq.KvShared(self.t(self.s_start), self.t(self.s_lens),
                                        self.t(self.s_table))

    def part(self, s, h):
        """Keys and values of the part that sequence s begins with, and which are there."""
        for g in range(len(self.s_lens)):
            if self.s_start[g] <= s < self.s_start[g + 1]:
                n = max(0, min(self.s_lens[g], self.s_table.shape[1] * self.page))
                p = np.arange(n)
                page = self.s_table[g, p // self.page]
                ok = (page >= 0) & (page < self.pages)
                at = np.where(ok, page, 0), h, p % self.page
                return (self.k[at] * self.ks[at].astype(np.float64)[:, None],
                        self.v[at] * self.vs[at].astype(np.float64)[:, None], ok)
        return np.zeros((0, HD)), np.zeros((0, HD)), np.zeros(0, bool)

    def shared64(self, q, heads, scale, causal, fill):
        out = np.full((self.T, heads * HD), fill)
        tol = np.zeros_like(out)
        for s, n in enumerate(self.new):
            for h in range(heads):
                kh = h // (heads // self.kvh)
                k, v, see = self.own(s, kh, causal)
                pk, pv, ok = self.part(s, kh)
                placed = len(k) - n + np.arange(n) >= 0
                see = np.concatenate([ok[None] & placed[:, None], see], 1)
                at = self.rows(s), slice(h * HD, (h + 1) * HD)
                out[at], tol[at], _, _ = soft(q[at], np.concatenate([pk, k]),
                                              np.concatenate([pv, v]), see, scale)
        return out, tol

    def check_shared(self, heads, causal=True, scale=None, q=None, fill=-3.0):
        q = self.queries(heads) if q is None else q
        out = self.torch.full((self.T, heads * HD), fill, device=self.dev)
        self.sdq.kv_attention_shared(self.cache, self.shared, self.batch, self.t(q), out, heads,
                                     causal=causal, scale=scale)
        got = out.cpu().numpy()
        self.close(got, *self.shared64(q, heads, HD**-0.5 if scale is None else scale, causal, fill))
        return got

    # ---- weights ----

    def weights64(self, w, q, heads, scale, causal):
        """The pool of sums after the call, and its tolerance (0: the same bits)."""
        got, tol = w.astype(np.float64), np.zeros(w.shape)
        G = heads // self.kvh
        for s, n in enumerate(self.new):
            L = max(0, min(self.lens[s], self.most * self.page))
            p = np.arange(L)
            page = self.table[s, p // self.page]
            live = (page >= 0) & (page < self.pages)
            if not n:
                continue
            for h in range(self.kvh):
                k, v, see = self.own(s, h, causal)
                total, off = np.zeros(L), np.zeros(L)
                for j in range(h * G, (h + 1) * G):
                    x = q[self.rows(s), j * HD:(j + 1) * HD]
                    fine = np.isfinite(x).all(1)
                    _, _, wt, rel = soft(np.where(fine[:, None], x, 0), k, v, see, scale)
                    total += (wt * fine[:, None]).sum(0)
                    off += (wt * rel * fine[:, None]).sum(0)
                at = page[live], h, (p % self.page)[live]
                old = np.where(p < L - n, 1.0, 0.0)[live] * w[at]
                got[at] = old + total[live]
                tol[at] = off[live] + (n * G / 16 + 16) * 2.0**-24 * (old + total[live]) + 1e-37
        return got, tol

    def check_weights(self, heads, causal=True, scale=None, q=None, calls=1):
        q = self.queries(heads) if q is None else q
        w = self.rng.uniform(0, 0.1, (self.pages, self.kvh, self.page)).astype(F)
        tw, tq = self.t(w), self.t(q)
        out = self.torch.full((self.T, heads * HD), -3.0, device=self.dev)
        same = out.clone()
        for _ in range(calls):
            w = tw.cpu().numpy()
            self.sdq.kv_attention_weights(self.cache, self.batch, tw, tq, out, heads, causal=causal,
                                          scale=scale)
            got = tw.cpu().numpy()
            self.close(got, *self.weights64(w, q, heads, HD**-0.5 if scale is None else scale, causal))
        self.sdq.kv_attention(self.cache, self.batch, tq, same, heads, causal=causal, scale=scale)
        assert_bitexact(out.cpu().numpy(), same.cpu().numpy(), "out")
        return got

    # ---- eviction ----

    def evict64(self, w, keep, first, last):
        """Kept positions [nseq, kv_heads, keep] and lengths."""
        kept = np.full((len(self.lens), self.kvh, keep), -1, np.int32)
        lens = np.zeros(len(self.lens), np.int32)
        for s in range(len(self.lens)):
            L = max(0, min(self.lens[s], self.most * self.page))
            p = np.arange(L)
            page = self.table[s, p // self.page]
            live = (page >= 0) & (page < self.pages)
            lens[s] = min(keep, live.sum())
            for h in range(self.kvh):
                x = w[np.where(live, page, 0), h, p % self.page].astype(np.float64)
                must = (p < first) | (p >= L - last)
                # groups in order: must, numbers by weight, NaN; then by position
                group = np.where(must, 0, np.where(np.isnan(x), 2, 1))
                x = np.where(group == 1, x, 0)
                order = np.lexsort((p, -x, group))
                order = order[live[order]][:keep]
                kept[s, h, :len(order)] = np.sort(order)
        return kept, lens

    def check_evict(self, w, keep, first=0, last=0, table=None):
        """The whole pool, weights, kept and lens against the definition, exact."""
        torch = self.torch
        nseq = len(self.lens)
        need = -(-keep // self.page)
        if table is None:  # pages behind the present ones
            add = nseq * need + 1
            for name in ("k", "v", "ks", "vs"):
                a = getattr(self, name)
                setattr(self, name, np.concatenate([a, np.zeros((add,) + a.shape[1:], a.dtype) + 1]))
            w = np.concatenate([w, np.full((add,) + w.shape[1:], -5, F)])
            table = (self.pages + self.rng.permutation(nseq * need).astype(np.int32)).reshape(nseq, need)
            self.pages += add
            self.up()
        tw = self.t(w)
        lens = torch.full((nseq,), -9, dtype=torch.int32, device=self.dev)
        kept = torch.full((nseq, self.kvh, keep), -9, dtype=torch.int32, device=self.dev)
        self.sdq.kv_evict(self.cache, self.batch, tw, self.t(table.astype(np.int32)), lens, kept,
                          first=first, last=last)
        want, want_lens = self.evict64(w, keep, first, last)
        assert_bitexact(kept.cpu().numpy(), want, "kept")
        assert_bitexact(lens.cpu().numpy(), want_lens, "lens")
        pools = [self.k.copy(), self.v.copy(), self.ks.copy(), self.vs.copy(), w.copy()]
        for s in range(nseq):
            for h in range(self.kvh):
                n = want_lens[s]
                to, src = np.arange(n), want[s, h, :n]
                page = table[s, to // self.page]
                ok = (page >= 0) & (page < self.pages)
                a = self.table[s, src // self.page], h, src % self.page
                b = page[ok], h, (to % self.page)[ok]
                for pool in pools:
                    pool[b] = pool[a][ok]
        for got, x, name in zip((self.cache.k, self.cache.v, self.cache.ks, self.cache.vs, tw), pools,
                                ("k", "v", "ks", "vs", "weights")):
            assert_bitexact(got.cpu().numpy(), x, name)
        return table, want_lens, tw


# ---- cross attention ----

@pytest.mark.parametrize("rows,lens", [
    ([1], [1]), ([1], [512]), ([7], [3]), ([1] * 8, [512, 0, 77, 1, 16, 300, 33, 511]), ([40], [1]),
    ([300], [17]), ([3, 0, 50, 1], [0, 9, 130, 2]), ([65, 129], [1000, 4099]), ([700], [512]),
    ([257, 1, 0, 300], [2050, 31, 64, 0])])
@pytest.mark.parametrize("heads,kvh", [(2, 2), (4, 1), (5, 1)])
def test_cross(sdq_dev, rows, lens, heads, kvh):
    """Any number of rows over any number of keys, none among them; rows before the first and
    behind the last sequence."""
    c = More(sdq_dev, rows, lens, kvh, (16, 64, 32)[len(rows) % 3], seed=sum(rows), first=1, behind=2)
    c.check_cross(heads)


@pytest.mark.parametrize("rows,lens", [([1100], [1]), ([1024], [64]), ([2500], [577]),
                                       ([1030, 2000, 900], [300, 0, 4099]), ([3000, 1100], [65, 127])])
@pytest.mark.parametrize("heads,kvh", [(2, 2), (3, 1)])
def test_cross_of_thousands(sdq_dev, rows, lens, heads, kvh):
    """Rows enough for keys that are turned to operands once; their first rows alone, which take
    the other form beside a table of more keys, have the same bits."""
    import torch

    c = More(sdq_dev, rows, lens, kvh, (16, 64, 32)[len(rows) % 3], seed=sum(rows), first=1, behind=2)
    c.vs[c.table[0, 0], :, 0] *= F(2.0**14)  # the others' exponents far below the first one's
    c.up()
    q = c.queries(heads)
    got = c.check_cross(heads, q=q)
    if len(rows) == 1:
        table = np.full((1, 800 // c.page + 1), -1, np.int32)
        table[:, :c.table.shape[1]] = c.table
        few = c.sdq.KvBatch(c.t(np.array([0, 700], np.int32)), c.batch.lens, c.t(table))
        out = torch.zeros((700, heads * HD), device=sdq_dev)
        c.sdq.kv_cross_attention(c.cache, few, c.t(q[1:701]), out, heads)
        assert_bitexact(out.cpu().numpy(), got[1:701])


@pytest.mark.parametrize("rows", [1, 40, 300])
def test_cross_scale_strides_missing_pages(sdq_dev, rows):
    import torch

    c = More(sdq_dev, [rows, rows], [333, 90], 2, 16, seed=3)
    c.table[0, 3] = c.pages
    c.table[1] = -1  # a sequence whose pages are all missing: 0
    c.up()
    c.check_cross(4, scale=0.3)
    c.check_cross(4, scale=-0.05)
    wide = torch.full((2 * rows, 1536), -2.0, device=sdq_dev)
    q = c.queries(4)
    wide[:, 256:768] = c.t(q)
    c.sdq.kv_cross_attention(c.cache, c.batch, wide[:, 256:768], wide[:, 896:1408], 4)
    got = wide.cpu().numpy()
    c.close(got[:, 896:1408], *c.cross64(q, 4, HD**-0.5, 0.0))
    assert (got[rows:, 896:1408] == 0).all()
    assert (got[:, :256] == -2).all() and (got[:, 768:896] == -2).all() and (got[:, 1408:] == -2).all()


@pytest.mark.parametrize("rows,lens", [([110] * 5, [900, 0, 1500, 33, 800]), ([100] * 20, [90, 700] * 10),
                                       ([300] * 8, [500, 1, 64, 127] * 2)])
@pytest.mark.parametrize("heads", [8, 16])
def test_cross_of_many_sequences(sdq_dev, rows, lens, heads):
    """Work enough for the taller tiles."""
    c = More(sdq_dev, rows, lens, 8, 32, seed=len(rows) + heads, first=1, behind=2)
    c.check_cross(heads)


@pytest.mark.parametrize("n", [1, 16, 600])
def test_cross_of_as_many_rows(sdq_dev, n):
    """As many rows as keys: the bits of kv_attention without its causal mask, where both take tiles
    of the same height."""
    import torch

    c = More(sdq_dev, [n, n], [n, n], 2, 32, seed=n)
    q = c.t(c.queries(4))
    a, b = torch.zeros((c.T, 512), device=sdq_dev), torch.zeros((c.T, 512), device=sdq_dev)
    c.sdq.kv_cross_attention(c.cache, c.batch, q, a, 4)
    c.sdq.kv_attention(c.cache, c.batch, q, b, 4, causal=False)
    assert_bitexact(a.cpu().numpy(), b.cpu().numpy())


@pytest.mark.parametrize("rows", [1, 100])
def test_cross_nan(sdq_dev, rows):
    """NaN behind the end changes nothing; a NaN row is its own affair, 0 without keys."""
    c = More(sdq_dev, [rows, rows, rows], [50, 75, 0], 1, 16, seed=6)
    q = c.queries(2)
    first = c.check_cross(2, q=q)
    for s in range(2):
        end = c.lens[s]
        c.ks[c.table[s, end // 16], :, end % 16:] = np.nan
        c.vs[c.table[s, end // 16], :, end % 16:] = np.inf
    c.up()
    assert_bitexact(c.check_cross(2, q=q), first, "masked NaN")
    bad = q.copy()
    bad[0, 3] = np.nan
    bad[2 * rows:] = np.inf
    out = c.torch.zeros((c.T, 256), device=sdq_dev)
    c.sdq.kv_cross_attention(c.cache, c.batch, c.t(bad), out, 2)
    got = out.cpu().numpy()
    assert np.isnan(got[0, :HD]).all() and (got[2 * rows:] == 0).all()
    assert_bitexact(got[0, HD:], first[0, HD:])
    assert_bitexact(got[1:2 * rows], first[1:2 * rows])


# ---- shared beginnings ----

@pytest.mark.parametrize("new,lens,s_start,parts", [
    ([1], [1], [0, 1], [1]), ([1] * 5, [3, 1, 17, 40, 2], [0, 5], [500]),
    ([1] * 7, [1, 20, 5, 3, 0, 9, 64], [1, 3, 3, 6], [129, 40, 2050]),
    ([3, 0, 20, 5], [3, 9, 40, 100], [0, 2, 4], [31, 0]),
    ([40, 70], [50, 70], [0, 2], [1000]), ([130, 300], [200, 301], [0, 1, 2], [77, 4099]),
    ([2, 5], [2, 3], [0, 2], [33])])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads,kvh", [(2, 2), (4, 1)])
def test_shared(sdq_dev, new, lens, s_start, parts, causal, heads, kvh):
    """Parts that end inside a page, empty parts, parts of no sequence, sequences without one, rows
    without a position."""
    c = More(sdq_dev, new, lens, kvh, (32, 16, 64)[len(new) % 3], seed=len(new) + sum(parts), first=1,
             behind=2)
    c.share(s_start, parts)
    c.check_shared(heads, causal)


@pytest.mark.parametrize("new", [1, 30, 100])
def test_shared_is_attention_over_both(sdq_dev, new):
    """Against kv_attention of the same tokens through one table (the part ends with a page)."""
    c = More(sdq_dev, [new] * 3, [new + 5, new + 40, new], 2, 16, seed=9)
    c.share([0, 3], [320])
    q = c.queries(4)
    got = c.check_shared(4, q=q)
    c.table = np.concatenate([np.repeat(c.s_table, 3, 0), c.table], 1)
    c.most = c.table.shape[1]
    c.lens = [320 + n for n in c.lens]
    c.up()
    want = c.check(4, True, q=q)
    _, tol = c.attend(q, 4, HD**-0.5, True)
    assert (np.abs(got - want) <= 2 * tol).all()


@pytest.mark.parametrize("new", [1, 90])
def test_shared_missing_pages_and_nan(sdq_dev, new):
    """Pages outside the pool leave their tokens out; NaN where no token is changes nothing."""
    c = More(sdq_dev, [new] * 3, [new + 20] * 3, 2, 16, seed=10)
    c.share([0, 2], [100])
    c.s_table[0, 2] = c.pages + 3
    c.table[1, 0] = -4
    c.up_shared()
    q = c.queries(4)
    first = c.check_shared(4, q=q)
    c.ks[c.s_table[0, 6], :, 4:] = np.nan
    c.vs[c.s_table[0, 6], :, 4:] = np.inf
    c.up_shared()
    assert_bitexact(c.check_shared(4, q=q), first, "masked NaN")
    # scratch that other calls filled with NaN
    bad = c.t(q)
    bad[2 * new:] = float("nan")
    out = c.torch.zeros((c.T, 512), device=sdq_dev)
    c.sdq.kv_attention_shared(c.cache, c.shared, c.batch, bad, out, 4)
    got = out.cpu().numpy()
    assert np.isnan(got[2 * new:]).all()
    assert_bitexact(got[:2 * new], first[:2 * new], "the other sequences")
    assert_bitexact(c.check_shared(4, q=q), first, "after it")
    c.s_lens[:] = 10**6  # past the table: as long as the table
    c.ks[c.s_table[0, 6], :, 4:] = F(0.01)
    c.vs[c.s_table[0, 6], :, 4:] = F(0.02)
    c.up_shared()
    c.check_shared(4, q=q)
    c.s_lens[:] = -5
    c.up_shared()
    assert_bitexact(c.check_shared(4, q=q)[2 * new:], first[2 * new:])


@pytest.mark.parametrize("new", [1, 90])
@pytest.mark.parametrize("ratio", [2.0**-50, 2.0**-20, 2.0**20, 2.0**50])
def test_shared_value_scales(sdq_dev, new, ratio):
    """Own values of far larger or smaller scales than the shared ones: to their range of 2^60."""
    c = More(sdq_dev, [new, new], [new + 30, new], 1, 16, seed=11)
    c.share([0, 1], [200])
    c.vs[c.table[c.table >= 0]] *= F(ratio)
    c.up_shared()
    c.check_shared(2)


def test_shared_without_parts(sdq_dev):
    """No parts: kv_attention, bit for bit; parts that no sequence has: close to it."""
    import torch

    c = More(sdq_dev, [1, 40], [30, 50], 1, 16, seed=12)
    c.share([0, 0], [40])
    q = c.queries(2)
    c.check_shared(2, q=q)
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device=sdq_dev)  # noqa: E731
    c.shared = c.sdq.KvShared(i32(1), i32(0), i32(0, 3))
    assert_bitexact(c.check_shared(2, q=q), c.check(2, True, q=q))


@pytest.mark.parametrize("nseq,n", [(64, 3), (70, 66), (300, 130)])
def test_shared_many_sequences(sdq_dev, nseq, n):
    rng = np.random.default_rng(nseq)
    new = rng.integers(0, 4, nseq)
    c = More(sdq_dev, new, new + rng.integers(0, 30, nseq), 1, 16, seed=13, first=2, behind=1)
    c.share(np.sort(rng.integers(0, nseq + 1, n + 1)), rng.integers(0, 90, n))
    c.check_shared(3)


@pytest.mark.parametrize("new,parts", [(20, 6), (50, 3), (140, 2)])
@pytest.mark.parametrize("heads", [8, 16])
def test_shared_of_many_rows(sdq_dev, new, parts, heads):
    """Work enough for the parts' taller tiles."""
    rng = np.random.default_rng(new)
    nseq = 18 // parts * parts // (1 if new < 50 else 2)
    rows = rng.integers(new - 10, new + 1, nseq)
    c = More(sdq_dev, rows, rows + rng.integers(0, 70, nseq), 8, 16, seed=15, first=1, behind=1)
    c.share([nseq * g // parts for g in range(parts + 1)], rng.integers(100, 900, parts))
    c.check_shared(heads)


# ---- counted weights ----

@pytest.mark.parametrize("new,lens", [
    ([1], [1]), ([1], [257]), ([1] * 6, [3, 0, 700, 64, 129, 2050]), ([2], [2]), ([17], [40]),
    ([33, 0, 1], [100, 50, 16]), ([130], [131]), ([300, 7], [300, 2000]), ([31, 1, 128], [0, 1, 500]),
    ([64, 65], [64, 1000]), ([1100], [1100]), ([600, 500], [700, 4099])])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads,kvh", [(2, 2), (4, 1), (6, 2)])
def test_weights(sdq_dev, new, lens, causal, heads, kvh):
    """Sums of the weights by key: new tokens start anew, older ones add up, others keep every bit;
    the output is kv_attention's."""
    c = More(sdq_dev, new, lens, kvh, (16, 32, 128)[len(new) % 3], seed=sum(new) + 1, first=1, behind=2)
    c.check_weights(heads, causal)


@pytest.mark.parametrize("new,L", [(1, 30011), (20, 20000), (700, 5000)])
def test_weights_long(sdq_dev, new, L):
    c = More(sdq_dev, [new], [L], 2, 256, seed=7)
    c.check_weights(4, True, calls=2)
    c.check_weights(2, False, scale=0.2)


@pytest.mark.parametrize("new", [1, 20, 200])
def test_weights_bad_rows_and_pages(sdq_dev, new):
    """Rows of NaN or infinities add nothing; missing pages and NaN behind the end stay out; rows of
    shared heads beside a bad one count. The same bits twice."""
    c = More(sdq_dev, [new, new], [new + 50, new + 7], 2, 16, seed=14)
    c.table[0, 1] = c.pages
    end = c.lens[1]
    c.ks[c.table[1, end // 16], :, end % 16:] = np.nan
    c.up()
    q = c.queries(4)
    q[0, 3] = np.nan
    q[-1, 200] = np.inf
    tq = c.t(q)
    w = c.rng.uniform(0, 0.1, (c.pages, 2, 16)).astype(F)
    out = c.torch.zeros((c.T, 512), device=sdq_dev)
    runs = []
    for _ in range(2):
        tw = c.t(w)
        c.sdq.kv_attention_weights(c.cache, c.batch, tw, tq, out, 4)
        runs.append(tw.cpu().numpy())
    c.close(runs[0], *c.weights64(w, q, 4, HD**-0.5, True))
    assert_bitexact(runs[1], runs[0], "twice")


@pytest.mark.parametrize("scale", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("new,L", [(12, 40), (90, 700), (1100, 1100)])
def test_weights_bad_scale(sdq_dev, new, L, scale):
    """A key whose scale is no number: rows whose logit of it is NaN or infinity add nothing, the
    others what they add without it, and itself gets nothing."""
    c = More(sdq_dev, [new], [L], 1, 16, seed=21)
    key = L - new // 2
    at = c.table[0, key // 16], 0, key % 16
    q, w = c.queries(2), c.rng.uniform(0, 0.1, (c.pages, 1, 16)).astype(F)
    k, v, see = c.own(0, 0, True)
    want, tol = np.zeros(L), np.zeros(L)
    for j in range(2):
        x = q[:, j * HD:(j + 1) * HD]
        dot = (x.astype(np.float64) @ k[key]) * scale
        lost = see[:, key] & ~(dot < 0)
        rest = see.copy()
        rest[:, key] = False
        _, _, wt, rel = soft(x, k, v, rest, HD**-0.5)
        want += (wt * ~lost[:, None]).sum(0)
        tol += (wt * rel * ~lost[:, None]).sum(0)
    p = np.arange(L)
    place = c.table[0, p // 16], 0, p % 16
    want += np.where(p < L - new, w[place], 0)
    c.ks[at] = scale
    c.up()
    tw, out = c.t(w), c.torch.zeros((c.T, 256), device=sdq_dev)
    c.sdq.kv_attention_weights(c.cache, c.batch, tw, c.t(q), out, 2)
    c.close(tw.cpu().numpy()[place], want, tol + (new / 8 + 16) * 2.0**-24 * want + 1e-37)


@pytest.mark.parametrize("new", [1, 100])
def test_weights_range(sdq_dev, new):
    """Value scales 2^60 apart do not enter the weights; sharp and huge logits."""
    c = More(sdq_dev, [new], [new + 100], 1, 16, seed=15)
    c.vs[:] = F(2.0) ** c.rng.integers(-40, 40, c.vs.shape)
    c.up()
    c.check_weights(2)
    c = More(sdq_dev, [new], [new + 600], 1, 64, seed=16, kscale=0.4)
    c.check_weights(2)
    w = c.t(np.zeros((c.pages, 1, 64), F))
    q = c.t(c.queries(2) * F(1e30))
    out = c.torch.zeros((c.T, 256), device=sdq_dev)
    c.sdq.kv_attention_weights(c.cache, c.batch, w, q, out, 2, causal=False)
    w = w.cpu().numpy()
    # a one for each row and head
    assert np.isfinite(w).all() and abs(w.sum() - 2 * new) <= 2 * new * 2.0**-20


def test_weights_at_any_float(sdq_dev):
    """Sums that begin one to three floats past a 16-byte boundary."""
    c = More(sdq_dev, [20], [400], 2, 32, seed=17)
    q, out = c.t(c.queries(4)), c.torch.zeros((20, 512), device=sdq_dev)
    runs = []
    for off in range(4):
        wide = c.torch.zeros(c.pages * 64 + 4, device=sdq_dev)
        w = wide[off:off + c.pages * 64].view(c.pages, 2, 32)
        c.sdq.kv_attention_weights(c.cache, c.batch, w, q, out, 4)
        runs.append(w.cpu().numpy())
        assert (wide[:off] == 0).all() and (wide[off + c.pages * 64:] == 0).all()
        assert_bitexact(runs[-1], runs[0])


@pytest.mark.parametrize("new", [1, 5])
def test_weights_of_a_wide_table(sdq_dev, new):
    """A table of 2^27 tokens, nearly all of it unused: the form that keeps no logits."""
    c = More(sdq_dev, [new, new], [300, 4000], 1, 16, seed=18)
    table = np.full((2, 1 << 23), -1, np.int32)
    table[:, :c.most] = c.table
    c.table, c.most = table, 1 << 23
    c.up()
    c.check_weights(2)
    c.check_weights(2, causal=False)


# ---- eviction ----

def _weights(c, kind):
    shape = (c.pages, c.kvh, c.page)
    w = np.exp(2 * c.rng.standard_normal(shape)).astype(F)
    if kind == "ties":
        w = c.rng.integers(0, 3, shape).astype(F)
    elif kind == "odd":
        w *= np.where(c.rng.random(shape) < 0.5, -1, 1)
        for x in (np.nan, -np.nan, np.inf, -np.inf, 0.0, -0.0, 1e-42, -1e-42):
            w[c.rng.random(shape) < 0.06] = x
    elif kind == "equal":
        w[:] = 0.25
    return w


@pytest.mark.parametrize("lens,keep,first,last", [
    ([1], 1, 0, 0), ([17], 16, 0, 0), ([40], 64, 3, 5), ([100, 0, 3, 64], 32, 4, 8),
    ([1000, 999, 33], 200, 200, 0), ([2111], 2048, 4, 512), ([500], 33, 0, 33), ([300], 7, 2, 4),
    ([5000, 16384, 16385], 1000, 1, 77), ([40000, 20], 16, 0, 1)])
@pytest.mark.parametrize("kind", ["spread", "ties", "odd", "equal"])
def test_evict(sdq_dev, lens, keep, first, last, kind):
    c = More(sdq_dev, [0] * len(lens), lens, 2, (16, 64, 32)[len(lens) % 3], seed=len(lens) + keep)
    c.check_evict(_weights(c, kind), keep, first, last)


@pytest.mark.parametrize("kind", ["spread", "ties", "odd", "equal"])
@pytest.mark.parametrize("lens,keep,first,last", [
    ([150001], 30000, 64, 4096), ([70000, 0, 16384, 16385, 33000], 5000, 3, 100),
    ([66000, 65999], 65999, 0, 1), ([100000], 1, 0, 0), ([65552, 1], 65552, 7, 9)])
def test_evict_long(sdq_dev, lens, keep, first, last, kind):
    """Tables of more tokens than a workgroup's registers hold."""
    c = More(sdq_dev, [0] * len(lens), lens, 2, 256, seed=20)
    c.check_evict(_weights(c, kind), keep, first, last)


@pytest.mark.parametrize("kind", ["spread", "odd"])
def test_evict_missing_pages(sdq_dev, kind):
    """Tokens without a page are not kept, first and last or not; tokens for a page outside the
    pool are lost and nothing else is."""
    c = More(sdq_dev, [0] * 3, [200, 70, 90], 2, 16, seed=21)
    c.table[0, 0] = -1
    c.table[0, 5] = c.pages + 40
    c.table[1, 4] = -7
    c.table[2] = -1
    c.up()
    w = _weights(c, kind)
    free = c.pages + np.arange(12, dtype=np.int32)
    for name in ("k", "v", "ks", "vs"):
        a = getattr(c, name)
        setattr(c, name, np.concatenate([a, np.zeros((12,) + a.shape[1:], a.dtype)]))
    w = np.concatenate([w, np.zeros((12,) + w.shape[1:], F)])
    c.pages += 12
    c.up()
    to = free.reshape(3, 4).copy()
    to[0, 1] = -1
    to[1, 2] = c.pages
    c.check_evict(w, 60, 3, 20, table=to)


def test_evict_lengths_past_the_table(sdq_dev):
    c = More(sdq_dev, [0, 0, 0], [100, 30, 60], 1, 16, seed=22)
    c.lens = [10**6, -4, 60]
    c.up()
    c.table[0, -1] = c.table[0, -1]
    c.check_evict(_weights(c, "spread"), 20, 1, 2)


# ---- together ----

def test_prompt_evicted_and_continued(sdq_dev):
    """A prompt written and attended with its weights counted, evicted, continued by single tokens
    behind a shared beginning, over another context by cross attention: each step against its
    definition on what the cache then holds."""
    import torch

    c = More(sdq_dev, [150, 90], [150, 90], 2, 16, seed=30)
    c.share([0, 2], [75])
    kv = c.rng.standard_normal((c.T, 512)).astype(F)
    c.sdq.kv_write(c.cache, c.batch, c.t(kv[:, :256]), c.t(kv[:, 256:]))
    pull = lambda: [setattr(c, n, getattr(c.cache, n).cpu().numpy()) for n in ("k", "v", "ks", "vs")]  # noqa: E731
    pull()
    q = c.queries(4)
    w = torch.zeros((c.pages, 2, 16), device=sdq_dev)
    out = torch.zeros((c.T, 512), device=sdq_dev)
    c.sdq.kv_attention_weights(c.cache, c.batch, w, c.t(q), out, 4)
    c.close(out.cpu().numpy(), *c.attend(q, 4, HD**-0.5, True))
    c.close(w.cpu().numpy(), *c.weights64(np.zeros(w.shape, F), q, 4, HD**-0.5, True))
    table, lens, tw = c.check_evict(w.cpu().numpy(), 50, 4, 16)
    pull()
    # single tokens behind what is left, counted again, behind the shared beginning, and across
    c.table = np.concatenate([table, np.full((2, 1), -1, np.int32)], 1)
    c.most = c.table.shape[1]
    c.new, c.lens, c.T = [1, 1], [int(n) + 1 for n in lens], 2
    c.start = np.array([0, 1, 2], np.int32)
    c.up_shared()
    kv = c.rng.standard_normal((2, 512)).astype(F)
    c.sdq.kv_write(c.cache, c.batch, c.t(kv[:, :256]), c.t(kv[:, 256:]))
    pull()
    c.check_shared(4)
    c.check_weights(4)
    c.check_cross(4)
    again = tw.clone()
    q = c.queries(4)
    c.sdq.kv_attention_weights(c.cache, c.batch, again, c.t(q), torch.zeros((2, 512), device=sdq_dev), 4)
    c.close(again.cpu().numpy(), *c.weights64(tw.cpu().numpy(), q, 4, HD**-0.5, True))


@pytest.mark.parametrize("new", [1, 70])
def test_captured(sdq_dev, new):
    """A step of all four, captured after one eager call, replayed with other lengths and inputs, eager
    calls between the replays; each replay equals the eager step."""
    import torch

    c = More(sdq_dev, [new, new], [new + 900, new + 800], 2, 16, seed=31)
    c.share([0, 2], [600])
    keep, need = 64, 4
    to = torch.arange(2 * need, dtype=torch.int32, device=sdq_dev).view(2, need) + c.pages
    grown = [np.concatenate([a, np.ones((2 * need,) + a.shape[1:], a.dtype)]) for a in (c.k, c.v, c.ks, c.vs)]
    c.k, c.v, c.ks, c.vs = grown
    c.pages += 2 * need
    c.up_shared()
    q = torch.empty((c.T, 512), device=sdq_dev)
    w0 = torch.rand((c.pages, 2, 16), device=sdq_dev)

    def outputs():
        return [torch.zeros((c.T, 512), device=sdq_dev) for _ in range(3)] + [
            torch.zeros_like(w0), torch.zeros(2, dtype=torch.int32, device=sdq_dev),
            torch.zeros((2, 2, keep), dtype=torch.int32, device=sdq_dev)]

    def step(o):
        c.sdq.kv_cross_attention(c.cache, c.batch, q, o[0], 4)
        c.sdq.kv_attention_shared(c.cache, c.shared, c.batch, q, o[1], 4)
        o[3].copy_(w0)
        c.sdq.kv_attention_weights(c.cache, c.batch, o[3], q, o[2], 4)
        c.sdq.kv_evict(c.cache, c.batch, o[3], to, o[4], o[5], first=2, last=9)

    side = torch.cuda.Stream()
    q.normal_()
    got, want = outputs(), outputs()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        step(got)
    side.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        step(got)
    for i in range(4):
        c.batch.lens.copy_(torch.tensor([new + 900 - 50 * i, new + 17 * i], dtype=torch.int32))
        c.shared.lens.copy_(torch.tensor([600 - 77 * i], dtype=torch.int32))
        q.normal_()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            g.replay()
        torch.cuda.synchronize()
        step(want)
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b), i
        for a in got + want:
            a.zero_()


def test_two_streams_and_threads(sdq_dev):
    """The same calls on two streams at once, and by threads that share one: each as alone."""
    import threading

    import torch

    import sdq

    c = More(sdq_dev, [1] * 4, [3000, 2000, 50, 700], 2, 64, seed=32)
    c.share([0, 4], [5000])
    q = c.t(c.queries(4))
    w = torch.rand((c.pages, 2, 64), device=sdq_dev)

    def cross(s):
        return c.sdq.kv_cross_attention(c.cache, c.batch, q, torch.zeros_like(q), 4, stream=s)

    def shared(s):
        return c.sdq.kv_attention_shared(c.cache, c.shared, c.batch, q, torch.zeros_like(q), 4, stream=s)

    def counted(s, o=None):
        o = w.clone() if o is None else o
        c.sdq.kv_attention_weights(c.cache, c.batch, o, q, torch.zeros_like(q), 4, stream=s)
        return o

    calls = [cross, shared, counted]
    want = [f(None) for f in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                outs += [(i, f(None)) for i, f in enumerate(calls)]
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i, o in outs)

    own = torch.cuda.Stream()
    fresh = [[torch.zeros_like(q) for _ in range(8)] for _ in range(2)] + [[w.clone() for _ in range(8)]]
    idle = torch.zeros_like(q)
    torch.cuda.synchronize()
    go = threading.Barrier(3)

    def run(i):
        sdq.init(0)
        go.wait()
        for o in fresh[i]:
            if i == 0:
                sdq.kv_cross_attention(c.cache, c.batch, q, o, 4, stream=own)
            elif i == 1:
                sdq.kv_attention_shared(c.cache, c.shared, c.batch, q, o, 4, stream=own)
            else:
                sdq.kv_attention_weights(c.cache, c.batch, o, q, idle, 4, stream=own)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    own.synchronize()
    for i in range(3):
        assert all(torch.equal(o, want[i]) for o in fresh[i]), i


def test_empty_calls(sdq_dev):
    import torch

    c = More(sdq_dev, [1], [0], 2, 16)
    c.share([0, 1], [0])
    assert (c.check_cross(2) == 0).all() and (c.check_shared(2) == 0).all()
    c.check_weights(2)
    none = torch.empty((0, 256), device=sdq_dev)
    w = torch.zeros((c.pages, 2, 16), device=sdq_dev)
    c.sdq.kv_cross_attention(c.cache, c.batch, none, none, 2)
    c.sdq.kv_attention_shared(c.cache, c.shared, c.batch, none, none, 2)
    c.sdq.kv_attention_weights(c.cache, c.batch, w, none, none, 2)
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device=sdq_dev)  # noqa: E731
    empty = c.sdq.KvBatch(i32(1), i32(0), i32(0, 1))
    x, o = (torch.full((2, 256), 3.0, device=sdq_dev) for _ in range(2))
    c.sdq.kv_cross_attention(c.cache, empty, x, o, 2)
    c.sdq.kv_attention_shared(c.cache, c.shared, empty, x, o, 2)
    c.sdq.kv_attention_weights(c.cache, empty, w, x, o, 2)
    c.sdq.kv_evict(c.cache, empty, w, i32(0, 1), i32(0), i32(0, 2, 5))
    assert (o == 3).all() and (w == 0).all()


@pytest.mark.parametrize("rows", [([3, 60]), ([1100, 90])])
def test_far_pages(sdq_dev, rows):
    """Pages behind 4 GiB of codes: the bits of the same pages at the pool's beginning."""
    import torch

    c = More(sdq_dev, rows, [n + 700 for n in rows], 8, 256, seed=33, extra=4)
    c.share([0, 2], [600])
    n, far = c.pages, 20000
    pool = c.sdq.KvCache.empty(far, 256, 8)
    for name in ("k", "v", "ks", "vs"):
        getattr(pool, name)[far - n:] = getattr(c.cache, name)
    move = lambda t: c.t(np.where(t >= 0, t + far - n, -1).astype(np.int32))  # noqa: E731
    there = (pool, c.sdq.KvBatch(c.batch.q_start, c.batch.lens, move(c.table)),
             c.sdq.KvShared(c.shared.s_start, c.shared.lens, move(c.s_table)), move)
    to, q = c.free[:2].reshape(2, 1), c.t(c.queries(16))
    w = c.t(c.rng.uniform(0, 0.1, (n, 8, 256)).astype(F))

    def step(cache, batch, shared, place):
        outs = [torch.zeros((c.T, 2048), device=sdq_dev) for _ in range(3)]
        ws = torch.zeros((cache.pages, 8, 256), device=sdq_dev)
        ws[-n:] = w
        lens = torch.zeros(2, dtype=torch.int32, device=sdq_dev)
        kept = torch.zeros((2, 8, 200), dtype=torch.int32, device=sdq_dev)
        c.sdq.kv_cross_attention(cache, batch, q, outs[0], 16)
        c.sdq.kv_attention_shared(cache, shared, batch, q, outs[1], 16)
        c.sdq.kv_attention_weights(cache, batch, ws, q, outs[2], 16)
        c.sdq.kv_evict(cache, batch, ws, place(to), lens, kept, first=3, last=20)
        return [x.cpu().numpy() for x in outs + [ws[-n:], lens, kept, cache.k[-n:], cache.v[-n:]]]

    for got, want in zip(step(*there), step(c.cache, c.batch, c.shared, lambda t: c.t(t))):
        assert_bitexact(got, want)


def test_pool_without_pages(sdq_dev):
    """Tables that name pages of an empty pool: rows see nothing, nothing is kept."""
    import torch

    c = More(sdq_dev, [2, 40], [20, 40], 2, 16, seed=34)
    c.share([0, 2], [30])
    cache = c.sdq.KvCache.empty(0, 16, 2)
    w, q = torch.zeros((0, 2, 16), device=sdq_dev), c.t(c.queries(4))
    for call in (lambda o: c.sdq.kv_cross_attention(cache, c.batch, q, o, 4),
                 lambda o: c.sdq.kv_attention_shared(cache, c.shared, c.batch, q, o, 4),
                 lambda o: c.sdq.kv_attention_weights(cache, c.batch, w, q, o, 4)):
        out = torch.full((c.T, 512), 3.0, device=sdq_dev)
        call(out)
        assert (out == 0).all()
    lens = torch.full((2,), 9, dtype=torch.int32, device=sdq_dev)
    kept = torch.full((2, 2, 16), 9, dtype=torch.int32, device=sdq_dev)
    c.sdq.kv_evict(cache, c.batch, w, c.t(c.table[:, :1]), lens, kept)
    assert (lens == 0).all() and (kept == -1).all()


def test_captured_large(sdq_dev):
    """Keys as operands, rows counted by their parts and a table of many chunks in one graph, replayed
    over other weights with eager calls between."""
    import torch

    c = More(sdq_dev, [1100], [1200], 2, 16, seed=35)
    wide = np.full((1, 20000 // 16), -1, np.int32)
    wide[:, :c.table.shape[1]] = c.table
    long = c.sdq.KvBatch(c.batch.q_start, c.batch.lens, c.t(wide))
    q = c.t(c.queries(4))
    to = c.t(np.full((1, 4), c.pages, np.int32))  # nowhere: only what is kept counts
    w = torch.zeros((c.pages, 2, 16), device=sdq_dev)
    outs = [torch.zeros((c.T, 512), device=sdq_dev) for _ in range(2)]
    lens = torch.zeros(1, dtype=torch.int32, device=sdq_dev)
    kept = torch.zeros((1, 2, 64), dtype=torch.int32, device=sdq_dev)

    def step():
        c.sdq.kv_cross_attention(c.cache, c.batch, q, outs[0], 4)
        c.sdq.kv_attention_weights(c.cache, c.batch, w, q, outs[1], 4)
        c.sdq.kv_evict(c.cache, long, w, to, lens, kept, first=2, last=5)
        return outs + [w, lens, kept]

    def fresh(seed):
        g = torch.Generator(device=sdq_dev).manual_seed(seed)
        q.copy_(torch.randn(q.shape, generator=g, device=sdq_dev))
        w.copy_(torch.rand(w.shape, generator=g, device=sdq_dev))

    side = torch.cuda.Stream()
    fresh(0)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step()
    for seed in (1, 2, 3):
        fresh(seed)
        want = [x.cpu().numpy() for x in step()]
        fresh(seed)
        for x in outs + [lens, kept]:
            x.fill_(-1)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graph.replay()
        torch.cuda.synchronize()
        for got, x in zip(outs + [w, lens, kept], want):
            assert_bitexact(got.cpu().numpy(), x)
