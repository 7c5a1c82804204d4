"""The paged int8 cache: sdq_kv_write / sdq_kv_read against the quantizer's steps
(exact), sdq_kv_attention against the softmax in 64 bits over the values that the
cache holds.

Attention's tolerance, per row, from its arithmetic: a logit (in units of log2)
is off by the q parts and the fp32 roundings of the sum of |q k| products (128, and 8
more that stand for the parts' 2^-21), plus two roundings of itself and of the running
maximum; a weight by its logit's error times ln 2, exp2's 2^-22 and the parts' 2^-21; the sums over n keys by
(n / 8 + 64) 2^-24. Numerator and denominator each, so twice that, of max |v|."""
import numpy as np
import pytest

from conftest import assert_bitexact
from test_gpu_rmsnorm_quant import codes_of

pytestmark = pytest.mark.gpu

F = np.float32
HD = 128


class Case:
    """A pool of shuffled pages and a ragged batch over it, host and device."""

    def __init__(self, dev, new, lens, kv_heads, page, seed=0, extra=2, first=0, behind=0,
                 kscale=0.012, vscale=0.02):
        import torch

        import sdq

        rng = np.random.default_rng(seed)
        self.new, self.lens, self.kvh, self.page = list(new), list(lens), kv_heads, page
        need = [-(-max(n, 0) // page) for n in lens]
        self.pages = sum(need) + extra
        ids = rng.permutation(self.pages).astype(np.int32)
        self.most = max(need + [1])
        self.table = np.full((len(lens), self.most), -1, np.int32)
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = ids[at:at + n]
            at += n
        self.free = ids[at:]
        shape = (self.pages, kv_heads, page)
        self.k = rng.integers(-127, 128, shape + (HD,)).astype(np.int8)
        self.v = rng.integers(-127, 128, shape + (HD,)).astype(np.int8)
        self.ks = (kscale * rng.uniform(0.5, 1.5, shape)).astype(F)
        self.vs = (vscale * rng.uniform(0.5, 1.5, shape)).astype(F)
        self.start = first + np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        self.T = int(self.start[-1]) + behind
        self.dev, self.rng = dev, rng
        self.sdq, self.torch = sdq, torch
        self.up()

    def t(self, a):
        return self.torch.from_numpy(np.ascontiguousarray(a)).to(self.dev)

    def up(self):
        self.cache = self.sdq.KvCache(self.t(self.k), self.t(self.ks), self.t(self.v),
                                      self.t(self.vs))
        self.batch = self.sdq.KvBatch(self.t(self.start), self.t(np.array(self.lens, np.int32)),
                                      self.t(self.table))

    def values(self, s, h):
        """K and V of sequence s, head h in 64 bits, and which tokens have a page."""
        p = np.arange(max(0, min(self.lens[s], self.most * self.page)))
        page = self.table[s, p // self.page]
        ok = (page >= 0) & (page < self.pages)
        at = np.where(ok, page, 0), h, p % self.page
        f = lambda c, sc: c[at].astype(np.float64) * sc[at].astype(np.float64)[:, None]  # noqa: E731
        with np.errstate(invalid="ignore"):
            return f(self.k, self.ks), f(self.v, self.vs), ok

    def attend(self, q, heads, scale, causal, fill=0.0):
        """The definition in 64 bits, and the tolerance of each row and head."""
        out = np.full((self.T, heads * HD), fill)
        tol = np.zeros((self.T, heads * HD))
        G = heads // self.kvh
        for s, n in enumerate(self.new):
            L = max(0, min(self.lens[s], self.most * self.page))
            pos = L - n + np.arange(n)
            for h in range(heads):
                k, v, ok = self.values(s, h // G)
                x = q[self.start[s]:self.start[s + 1], h * HD:(h + 1) * HD].astype(np.float64)
                t = x @ k.T * scale
                size = np.abs(x) @ np.abs(k).T * abs(scale)
                see = ok[None] & (pos[:, None] >= 0) & np.ones((n, len(k)), bool)
                if causal:
                    see &= np.arange(len(k))[None] <= pos[:, None]
                t = np.where(see, t, -np.inf)
                top = t.max(1, initial=-np.inf, keepdims=True)
                w = np.exp(t - np.where(np.isinf(top), 0, top)) * see
                z = w.sum(1, keepdims=True)
                w = w / np.where(z == 0, 1, z)
                rows = slice(self.start[s], self.start[s + 1]), slice(h * HD, (h + 1) * HD)
                out[rows] = w @ np.where(ok[:, None], v, 0)
                # of a key far below the maximum the weight itself bounds the error
                err = ((2.0**-22 + 136 * 2.0**-24) * size + 2.0**-21 * np.abs(np.where(see, t, 0))
                       + 2.0**-21 * np.abs(np.where(np.isinf(top), 0, top)))
                rel = (w * (err + 2.0**-20)).sum(1, keepdims=True) + (len(k) / 8 + 64) * 2.0**-24
                tol[rows] = 2 * rel * np.abs(v[ok]).max(initial=0)
        return out, tol

    def check(self, heads, causal, scale=None, q=None, fill=-3.0, slack=1.0):
        q = self.rng.standard_normal((self.T, heads * HD)).astype(F) * F(1.5) if q is None else q
        out = self.torch.full((self.T, heads * HD), fill, device=self.dev)
        self.sdq.kv_attention(self.cache, self.batch, self.t(q), out, heads, causal=causal,
                              scale=scale)
        got = out.cpu().numpy()
        want, tol = self.attend(q, heads, HD**-0.5 if scale is None else scale, causal, fill)
        bad = ~(np.abs(got - want) <= tol * slack)
        assert not bad.any(), (np.argwhere(bad)[:3], got[bad][:3], want[bad][:3], tol[bad][:3])
        return got


# ---- writes and reads ----

@pytest.mark.parametrize("new,lens,kvh,page", [
    ([1], [1], 1, 16), ([1, 1, 1], [40, 1, 17], 3, 16), ([5, 0, 33, 1], [5, 9, 70, 256], 2, 32),
    ([300], [300], 24, 256), ([17, 16, 15], [17, 48, 1000], 5, 64)])
@pytest.mark.parametrize("strided", [False, True])
def test_write_and_read(sdq_dev, new, lens, kvh, page, strided):
    import torch

    c = Case(sdq_dev, new, lens, kvh, page, first=2, behind=3)
    C = kvh * HD
    kv = c.rng.standard_normal((c.T, 2 * C)).astype(F) * 3
    kv[0, :HD] = 0
    kv[2, 5] = np.nan
    kv[3 if c.T > 3 else 2, C + 7] = np.inf
    kv[2 + sum(new) - 1, C:C + HD] = 0
    t = c.t(kv)
    k, v = (t[:, :C], t[:, C:]) if strided else (t[:, :C].contiguous(), t[:, C:].contiguous())
    before = [a.copy() for a in (c.k, c.ks, c.v, c.vs)]
    c.sdq.kv_write(c.cache, c.batch, k, v)
    want = before
    for s, n in enumerate(new):
        for i in range(n):
            p = lens[s] - n + i
            at = c.table[s, p // page], slice(None), p % page
            for x, codes, scales in ((kv[c.start[s] + i, :C], want[0], want[1]),
                                     (kv[c.start[s] + i, C:], want[2], want[3])):
                codes[at], scales[at] = codes_of(x.reshape(kvh, HD))
    for got, w, name in zip((c.cache.k, c.cache.ks, c.cache.v, c.cache.vs), want,
                            ("k", "ks", "v", "vs")):
        assert_bitexact(got.cpu().numpy(), w, name)  # the whole pool: nothing else moved
    o = torch.full((c.T, 2 * C), -9.0, device=sdq_dev)
    c.sdq.kv_read(c.cache, c.batch, o[:, :C], o[:, C:])
    got = o.cpu().numpy()
    assert (got[:2] == -9).all() and (got[2 + sum(new):] == -9).all()
    for s, n in enumerate(new):
        for i in range(n):
            p = lens[s] - n + i
            at = c.table[s, p // page], slice(None), p % page
            with np.errstate(invalid="ignore"):
                y = np.concatenate([(want[0][at] * want[1][at][:, None]).ravel(),
                                    (want[2][at] * want[3][at][:, None]).ravel()])
            np.testing.assert_array_equal(got[c.start[s] + i], y)


def test_rows_without_a_place(sdq_dev):
    """Page ids outside the pool, lengths past the table and below the rows: nothing
    is written there, reads give 0, and attention leaves the tokens out."""
    import torch

    c = Case(sdq_dev, [4, 6, 3], [40, 4, 30], 2, 16, behind=1)
    c.table[0, 2] = c.pages  # tokens 32..39 of the first sequence have no page
    c.table[2, 1] = -7
    c.up()
    x = c.t(c.rng.standard_normal((c.T, 256)).astype(F))
    pool = [a.clone() for a in (c.cache.k, c.cache.v, c.cache.ks, c.cache.vs)]
    c.sdq.kv_write(c.cache, c.batch, x, x)
    k, v = torch.full((c.T, 256), 5.0, device=sdq_dev), torch.full((c.T, 256), 5.0, device=sdq_dev)
    c.sdq.kv_read(c.cache, c.batch, k, v)
    rows = k.cpu().numpy()
    assert (rows[:4] == 0).all() and (rows[4:6] == 0).all() and (rows[6:10] != 0).any(1).all()
    assert (rows[10:13] == 0).all() and (rows[13] == 5).all()
    for a, b in zip(pool, (c.cache.k, c.cache.v, c.cache.ks, c.cache.vs)):
        a[c.table[1, 0]] = b[c.table[1, 0]]
        assert torch.equal(a, b)
    c.k, c.v = c.cache.k.cpu().numpy(), c.cache.v.cpu().numpy()
    c.ks, c.vs = c.cache.ks.cpu().numpy(), c.cache.vs.cpu().numpy()
    for causal in (False, True):
        c.check(4, causal)
    c.lens[0] = 10**6  # past the table: as long as the table
    c.up()
    c.check(2, True)


# ---- attention ----

@pytest.mark.parametrize("lens", [[1], [2], [15], [16], [17], [31], [33], [64], [65], [127], [500],
                                  [1025], [4099], [3, 0, 700, 64, 1, 129, 0, 2050]])
@pytest.mark.parametrize("heads,kvh", [(1, 1), (6, 2), (8, 1), (20, 1), (3, 3)])
def test_single_tokens(sdq_dev, lens, heads, kvh):
    c = Case(sdq_dev, [1] * len(lens), lens, kvh, 16 if len(lens) > 1 else 64, seed=len(lens))
    c.check(heads, True)


@pytest.mark.parametrize("new,lens", [([2], [2]), ([16], [16]), ([17], [40]), ([33], [100]),
                                      ([64], [64]), ([65], [1000]), ([130], [131]), ([257], [700]),
                                      ([5, 40, 0, 100], [5, 300, 50, 99]), ([300, 7], [300, 2000]),
                                      ([31, 1, 128, 2], [0, 1, 500, 77])])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("heads,kvh", [(2, 2), (4, 1), (5, 1)])
def test_chunks(sdq_dev, new, lens, causal, heads, kvh):
    """Ragged chunks; new tokens beyond the cache's length (rows without a
    position: 0) and empty sequences among them."""
    c = Case(sdq_dev, new, lens, kvh, (16, 32, 128)[len(new) % 3], seed=sum(new), first=1, behind=2)
    c.check(heads, causal)


@pytest.mark.parametrize("new,L,heads,kvh", [(1, 30011, 4, 1), (1, 9000, 3, 3), (40, 20000, 2, 1),
                                             (700, 5000, 2, 2)])
def test_long(sdq_dev, new, L, heads, kvh):
    c = Case(sdq_dev, [new], [L], kvh, 256, seed=7)
    c.check(heads, True)
    c.check(heads, False)


@pytest.mark.parametrize("new", [1, 40, 300])
def test_scale_and_strides(sdq_dev, new):
    import torch

    c = Case(sdq_dev, [new], [333], 2, 32, seed=3)
    c.check(4, True, scale=0.3)
    c.check(4, False, scale=-0.05)
    c.check(4, True, scale=0.0)
    # columns of wider rows, in and out; the columns beside them stay
    wide = torch.full((new, 1536), -2.0, device=sdq_dev)
    q = c.rng.standard_normal((new, 512)).astype(F)
    wide[:, 256:768] = c.t(q)
    c.sdq.kv_attention(c.cache, c.batch, wide[:, 256:768], wide[:, 896:1408], 4, causal=True)
    want, tol = c.attend(q, 4, HD**-0.5, True)
    got = wide.cpu().numpy()
    assert (np.abs(got[:, 896:1408] - want) <= tol).all()
    assert (got[:, :256] == -2).all() and (got[:, 768:896] == -2).all() and (got[:, 1408:] == -2).all()
    assert_bitexact(got[:, 256:768], q, "q")


@pytest.mark.parametrize("new", [1, 20, 100])
def test_scales_at_any_float(sdq_dev, new):
    """Scales that begin one, two or three floats past a 16-byte boundary: the same bits."""
    c = Case(sdq_dev, [new, new], [new + 300, new + 77], 2, 32, seed=27)
    q = c.rng.standard_normal((c.T, 512)).astype(F)
    first = c.check(4, True, q=q)
    for off in (1, 2, 3):
        moved = []
        for t in (c.cache.ks, c.cache.vs):
            wide = c.torch.zeros(t.numel() + 4, device=sdq_dev)
            moved.append(wide[off:off + t.numel()].view(t.shape))
            moved[-1].copy_(t)
            assert moved[-1].data_ptr() % 16 == 4 * off
        c.cache = c.sdq.KvCache(c.cache.k, moved[0], c.cache.v, moved[1])
        assert_bitexact(c.check(4, True, q=q), first, f"offset {off}")
        c.sdq.kv_write(c.cache, c.batch, c.t(q[:, :256]), c.t(q[:, 256:]))
        k, v = (c.torch.zeros((c.T, 256), device=sdq_dev) for _ in range(2))
        c.sdq.kv_read(c.cache, c.batch, k, v)
        assert (k - c.t(q[:, :256])).abs().max() < 0.05
        c.up()


@pytest.mark.parametrize("new", [1, 100])
def test_sharp_and_far_apart(sdq_dev, new):
    """Logits of hundreds; scales of keys and values far apart, weights the other
    way round, so that small values of heavy keys stand beside large ones of light
    keys: each output to its own scale."""
    c = Case(sdq_dev, [new], [600], 1, 64, seed=4, kscale=0.4)
    c.check(2, True)
    c = Case(sdq_dev, [new], [600], 1, 64, seed=5)
    p = c.table[0, np.arange(600) // 64], 0, np.arange(600) % 64
    heavy = np.arange(600) % 50 == 3
    c.vs[p] = np.where(heavy, F(2.0**-24), F(1.0))
    c.ks[p] = np.where(heavy, F(0.02), F(1e-6))
    q = np.zeros((new, HD), F)
    k0 = c.k[p][3].astype(F)
    q[:] = k0 / np.linalg.norm(k0) * 60
    for i in np.arange(600)[heavy]:
        c.k[c.table[0, i // 64], 0, i % 64] = c.k[p][3]
    c.up()
    c.check(1, False, q=q)
    c.vs[p] = F(2.0) ** c.rng.integers(-40, 40, 600)
    c.ks[p] = F(0.05) * F(2.0) ** c.rng.integers(-20, 2, 600)
    c.up()
    c.check(2, True)


@pytest.mark.parametrize("new", [1, 100])
def test_nan_stays_where_it_is(sdq_dev, new):
    """NaN and infinite scales behind a sequence's end, in pages that are not its
    own, and in another sequence change nothing; a NaN query its own row only."""
    c = Case(sdq_dev, [new, new], [new + 37, new + 90], 2, 16, seed=6)
    clean = c.check(4, True)
    q = c.rng.standard_normal((c.T, 512)).astype(F)
    first = c.check(4, True, q=q)
    for f in c.free:
        c.ks[f], c.vs[f] = np.nan, np.inf
    for s in range(2):
        end = c.lens[s]
        if end % 16:
            c.ks[c.table[s, end // 16], :, end % 16:] = np.nan
            c.vs[c.table[s, end // 16], :, end % 16:] = np.inf
    c.up()
    assert_bitexact(c.check(4, True, q=q), first, "masked NaN")
    bad = q.copy()
    bad[0, 3] = np.nan
    bad[new, 130] = np.inf
    out = c.torch.zeros((c.T, 512), device=sdq_dev)
    c.sdq.kv_attention(c.cache, c.batch, c.t(bad), out, 4, causal=True)
    got = out.cpu().numpy()
    assert np.isnan(got[0, :HD]).all() and not np.isfinite(got[new, HD:2 * HD]).all()
    want, tol = c.attend(q, 4, HD**-0.5, True)
    keep = np.ones((c.T, 512), bool)
    keep[0, :HD] = keep[new, HD:2 * HD] = False
    assert (np.abs(got - want) <= tol)[keep].all()
    c.vs[c.table[1, 0]] = np.nan
    c.up()
    out.zero_()
    c.sdq.kv_attention(c.cache, c.batch, c.t(q), out, 4, causal=True)
    got = out.cpu().numpy()
    assert_bitexact(got[:new], first[:new], "the other sequence")
    assert np.isnan(got[new:]).all() and np.isfinite(clean).all()


@pytest.mark.parametrize("new", [1, 40, 100, 300])
def test_nan_queries_that_see_no_key(sdq_dev, new):
    """Rows of padding, whatever they hold, whose sequence has no page or no keys are 0."""
    c = Case(sdq_dev, [new, new, new], [new + 40, new + 90, 0], 1, 16, seed=24)
    c.table[0] = -1
    c.up()
    q = c.rng.standard_normal((c.T, 2 * HD)).astype(F)
    want = c.check(2, True, q=q)
    for bad in (np.nan, np.inf):
        q[:new] = bad
        q[2 * new:, 5] = bad
        for causal in (True, False):
            out = c.torch.full((c.T, 2 * HD), 4.0, device=sdq_dev)
            c.sdq.kv_attention(c.cache, c.batch, c.t(q), out, 2, causal=causal)
            got = out.cpu().numpy()
            assert (got[:new] == 0).all() and (got[2 * new:] == 0).all()
            if causal:
                assert_bitexact(got[new:2 * new], want[new:2 * new], "the other sequence")
    # the first half of the pages is missing: rows that see none of the others
    c.table[1, :c.lens[1] // 32] = -1
    c.up()
    q = c.rng.standard_normal((c.T, 2 * HD)).astype(F)
    c.check(2, True, q=q)
    c.check(2, False, q=q)


@pytest.mark.parametrize("nseq,most", [(63, 3), (64, 2), (65, 40), (200, 9), (4100, 2)])
def test_many_sequences(sdq_dev, nseq, most):
    """Ragged batches around the search's widths, empty sequences among them, rows
    before the first and behind the last."""
    rng = np.random.default_rng(nseq)
    new = rng.integers(0, most + 1, nseq)
    lens = new + rng.integers(0, 30, nseq)
    c = Case(sdq_dev, new, lens, 1, 16, seed=18, first=3, behind=2)
    c.check(3, True)


@pytest.mark.parametrize("new", [1, 100])
def test_a_huge_row_takes_nothing_from_others(sdq_dev, new):
    """A head of a token holds 1e30: the rows beside it, of its own tile among
    them, keep every bit."""
    c = Case(sdq_dev, [new], [new + 300], 1, 32, seed=12)
    q = c.rng.standard_normal((c.T, 3 * HD)).astype(F)
    first = c.check(3, True, q=q)
    big = q.copy()
    big[-1, HD:2 * HD] = F(1e30)
    out = c.torch.zeros((c.T, 3 * HD), device=sdq_dev)
    c.sdq.kv_attention(c.cache, c.batch, c.t(big), out, 3, causal=True)
    got = out.cpu().numpy()
    keep = np.ones(first.shape, bool)
    keep[-1, HD:2 * HD] = False
    assert_bitexact(got[keep], first[keep], "the other rows")


@pytest.mark.parametrize("new", [1, 20, 100, 300])
@pytest.mark.parametrize("size", [1e30, 3e35, 1e36])
def test_large_queries(sdq_dev, new, size):
    """Queries whose products with the codes alone pass fp32's range, with the key's scale they do
    not: one key's logit is far above all others, and its value is the result (its code times its
    scale: the weight's parts and three roundings)."""
    L = new + 200
    c = Case(sdq_dev, [new], [L], 1, 32, seed=22)
    sign = np.where(np.arange(HD) % 3, 1, -1)
    c.k[c.table[0, 1], 0, 7] = 127 * sign  # token 39
    c.ks[c.table[0, 1], 0, 7] = F(0.018)
    c.up()
    q = np.repeat((size * sign).astype(F)[None], new, 0)
    q = np.concatenate([q, q * F(0.5)], 1)
    out = c.torch.zeros((new, 2 * HD), device=sdq_dev)
    c.sdq.kv_attention(c.cache, c.batch, c.t(q), out, 2, causal=True)
    want = np.tile(c.values(0, 0)[1][39], 2)[None]
    assert (np.abs(out.cpu().numpy() - want) <= 2.0**-20 * np.abs(want)).all()


@pytest.mark.parametrize("new", [1, 100])
def test_range_of_value_scales(sdq_dev, new):
    """A first value of next to nothing leaves the others their precision; scales
    2^60 past the first one's are refused the only way a kernel can: NaN in the rows
    that see them, and in those alone."""
    c = Case(sdq_dev, [new], [new + 100], 1, 16, seed=13)
    at = lambda p: (c.table[0, p // 16], 0, p % 16)  # noqa: E731
    for tiny in (2.0**-40, 2.0**-90, 2.0**-130):
        c.vs[at(0)] = F(tiny)
        c.up()
        q = c.rng.standard_normal((c.T, 2 * HD)).astype(F)
        got = c.check(2, True, q=q)
    c.vs[at(0)] = F(0.75)  # its exponent is 0
    c.vs[at(new + 90)] = F(2.0**59 * 1.99)
    c.up()
    c.check(2, True, q=q)
    c.vs[at(new + 90)] = F(2.0**60)
    c.up()
    out = c.torch.zeros((c.T, 2 * HD), device=sdq_dev)
    c.sdq.kv_attention(c.cache, c.batch, c.t(q), out, 2, causal=True)
    got = out.cpu().numpy()
    sees = 100 + np.arange(new) >= new + 90
    assert np.isnan(got[sees]).all() and np.isfinite(got[~sees]).all()


@pytest.mark.parametrize("new,L", [(1, 200), (1, 1500), (1, 4200), (100, 200), (100, 4200),
                                   (300, 700), (300, 4200)])
@pytest.mark.parametrize("where", ["early", "late"])
def test_both_ends_of_the_value_scales(sdq_dev, new, L, where):
    """One value of scale nearly 2^60 times the first, all others of nearly 2^-60 of it, and
    eight octaves less weight: its logit and exponent put the others' weights under the
    smallest float, and they still own most of the denominator. The large value before and
    behind them, in the same wave's keys and in other shares.

    A small key's exponent is a difference of numbers up to 2^8: three roundings of at most
    2^-17, 2^-16 of its weight; the same relative to the result, beside check()'s terms."""
    c = Case(sdq_dev, [new], [L], 1, 64, seed=21)
    at = lambda p: (c.table[0, p // 64], 0, p % 64)  # noqa: E731
    big = 3 if where == "early" else L - new - 1
    keys = np.arange(1, L)
    c.vs[at(keys)] = F(0.75 * 2.0**-60)
    c.vs[at(0)], c.vs[at(big)] = F(0.75), F(2.0**59 * 1.9)
    c.ks[at(np.arange(L))] = F(0.01)
    c.k[at(np.arange(L))] = c.rng.integers(-3, 4, (L, HD))
    for p in range(L):
        c.k[c.table[0, p // 64], 0, p % 64, 0] = 100 if p == big else 0
    c.v[at(0)] = 0
    c.up()
    q = np.zeros((c.T, HD), F)
    q[:, 0] = 8 * np.log(2) * HD**0.5
    out = c.torch.zeros((c.T, HD), device=sdq_dev)
    for causal in (True, False):
        c.sdq.kv_attention(c.cache, c.batch, c.t(q), out, 1, causal=causal)
        want, tol = c.attend(q, 1, HD**-0.5, causal)
        got = out.cpu().numpy()
        bad = ~(np.abs(got - want) <= tol + 2.0**-16 * 2 * np.abs(want))
        assert not bad.any(), (causal, np.argwhere(bad)[:3], got[bad][:3], want[bad][:3])


@pytest.mark.parametrize("nseq,new", [(800, 1), (1100, 100), (1, 1 << 17)])
def test_many_light_keys(sdq_dev, nseq, new):
    """2^17 keys of equal weight, 22 octaves under that of the first, whose value is zero, seen
    by so many rows that their keys are not cut: each light weight is rounded to the parts'
    smallest step, all of them the same way, and the sum keeps them.

    Of max |v|: the weights' second part is off by at most 2^-25 where the largest weight is 2^9
    (2^-34 a key, 2^-17 of all), the parts otherwise and the query's by 2^-21 of a share of 2^-5; the
    logits' roundings 2^-19 of it. A lane adds up the denominator of a block of 32 keys at a time, and
    every addition of an equal share to a sum near 1 can be off the same way by 2^-24: n / 32 of
    them, 2^-12 of the denominator, of which the result is a share of 2^-5."""
    n = 1 << 17
    L = n + 1
    c = Case(sdq_dev, [1], [L], 1, 1024, seed=23)
    p = np.arange(L)
    at = c.table[0, p // 1024], 0, p % 1024
    c.vs[at] = F(0.0199)
    c.ks[at] = F(0.01)
    k = np.zeros((L, HD), np.int8)
    k[0, 0] = 100
    v = np.full((L, HD), 127, np.int8)
    v[0] = 0
    c.k[at], c.v[at] = k, v
    c.table = np.repeat(c.table, nseq, 0)  # shared pages
    c.lens, c.start, c.T = [L] * nseq, new * np.arange(nseq + 1, dtype=np.int32), nseq * new
    c.up()
    tol = (2.0**-17 + 2.0**-5 * (2.0**-21 + 2.0**-19 + 2.0**-12)) * 127 * 0.0199
    out = c.torch.zeros((c.T, HD), device=sdq_dev)
    for octaves in (22.0, 22.17, 22.31, 22.5, 22.63, 22.9):
        q = c.torch.zeros((c.T, HD), device=sdq_dev)
        q[:, 0] = octaves * np.log(2) * HD**0.5
        c.sdq.kv_attention(c.cache, c.batch, q, out, 1, causal=False)
        w = np.exp2(-float(q[0, 0]) * 100 * float(F(0.01)) * HD**-0.5 / np.log(2))
        want = n * w / (1 + n * w) * 127 * float(F(0.0199))
        err = (out.double() - want).abs().max().item()
        assert err <= tol, (octaves, err / tol)


def test_shared_pages_and_independence(sdq_dev):
    """Two sequences that share their first pages; a batch's rows do not depend on
    who else is in it, bit for bit where the call's sizes are the same."""
    c = Case(sdq_dev, [3, 3], [50, 60], 2, 16, seed=8)
    c.table[1, :2] = c.table[0, :2]
    c.up()
    q = c.rng.standard_normal((c.T, 256)).astype(F)
    both = c.check(2, True, q=q)
    c.k[c.table[1, 3]] = 5
    c.up()
    assert_bitexact(c.check(2, True, q=q)[:3], both[:3], "first sequence")


def test_empty_calls(sdq_dev):
    import torch

    c = Case(sdq_dev, [1], [0], 2, 16)
    got = c.check(2, True)
    assert (got == 0).all()
    none = torch.empty((0, 256), device=sdq_dev)
    c.sdq.kv_attention(c.cache, c.batch, none, none, 2)
    c.sdq.kv_write(c.cache, c.batch, none, none)
    empty = c.sdq.KvBatch(torch.zeros(1, dtype=torch.int32, device=sdq_dev),
                          torch.zeros(0, dtype=torch.int32, device=sdq_dev),
                          torch.zeros((0, 1), dtype=torch.int32, device=sdq_dev))
    x = torch.full((2, 256), 3.0, device=sdq_dev)
    o = torch.full((2, 256), 3.0, device=sdq_dev)
    c.sdq.kv_attention(c.cache, empty, x, o, 2)
    assert (o == 3).all()


@pytest.mark.parametrize("new", [1, 70])
def test_captured_and_two_streams(sdq_dev, new):
    """Write and attention captured (after one eager call) and replayed with growing
    sequences; two batches at once on two streams."""
    import torch

    c = Case(sdq_dev, [new, new], [new, new], 2, 16, seed=9)
    most = 6 * new + 400
    need = -(-most // 16)
    c.pages = 2 * need
    c.table = np.arange(2 * need, dtype=np.int32)[::-1].reshape(2, need).copy()
    c.most = need
    shape = (c.pages, 2, 16)
    c.k, c.v = np.zeros(shape + (HD,), np.int8), np.zeros(shape + (HD,), np.int8)
    c.ks, c.vs = np.ones(shape, F), np.ones(shape, F)
    c.up()
    qkv = torch.empty((c.T, 512 + 512), device=sdq_dev)
    out = torch.empty((c.T, 512), device=sdq_dev)

    def step(o):
        c.sdq.kv_write(c.cache, c.batch, qkv[:, 512:768], qkv[:, 768:])
        c.sdq.kv_attention(c.cache, c.batch, qkv[:, :512], o, 4)

    side = torch.cuda.Stream()
    qkv.normal_()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        step(out)
    side.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        step(out)
    for i in range(4):
        c.lens = [new * (i + 1), new * (i + 1) + 100 * i]
        c.batch.lens.copy_(torch.tensor(c.lens, dtype=torch.int32))
        qkv.copy_(torch.from_numpy(np.random.default_rng(i).standard_normal((c.T, 1024)).astype(F)))
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            g.replay()
        torch.cuda.synchronize()
        got = out.clone()
        again = torch.empty_like(out)
        step(again)
        torch.cuda.synchronize()
        assert torch.equal(got, again), i
        c.k, c.v = c.cache.k.cpu().numpy(), c.cache.v.cpu().numpy()
        c.ks, c.vs = c.cache.ks.cpu().numpy(), c.cache.vs.cpu().numpy()
        want, tol = c.attend(qkv[:, :512].cpu().numpy(), 4, HD**-0.5, True)
        assert (np.abs(got.cpu().numpy() - want) <= tol).all(), i
    others = [torch.cuda.Stream() for _ in range(2)]
    outs = [torch.empty_like(out) for _ in others]
    for _ in range(3):
        for st, o in zip(others, outs):
            with torch.cuda.stream(st):
                c.sdq.kv_attention(c.cache, c.batch, qkv[:, :512], o, 4)
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o, again)


def test_growth_under_capture_is_refused(sdq_dev):
    """A call whose scratch the stream does not have yet raises under capture and leaves the
    capture usable; after one eager call it captures. (torch hands out pooled streams:
    the first one that other tests have not grown is taken.)"""
    import torch

    c = Case(sdq_dev, [250], [40000], 8, 64, seed=14)
    q = torch.randn((250, 8 * HD), device=sdq_dev)
    out, want = torch.zeros_like(q), torch.zeros_like(q)
    torch.cuda.synchronize()
    for _ in range(64):
        side = torch.cuda.Stream()
        g = torch.cuda.CUDAGraph()
        try:
            with torch.cuda.graph(g, stream=side):
                c.sdq.kv_attention(c.cache, c.batch, q, out, 8)
        except c.sdq.SdqError as e:
            assert "captures a graph" in str(e)
            break
    else:
        pytest.fail("every stream has the scratch")
    del g
    with torch.cuda.stream(side):
        c.sdq.kv_attention(c.cache, c.batch, q, want, 8)
    side.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        c.sdq.kv_attention(c.cache, c.batch, q, out, 8)
    for _ in range(3):
        out.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_threads_on_one_stream(sdq_dev):
    """Four threads on one stream, the calls' scratch the same memory: attention with its keys
    cut, 4-bit Linears, and the packed attention: each result equals the call alone."""
    import threading

    import torch

    import sdq
    import test_gpu_q4linear as q4

    cases = [Case(sdq_dev, [1, 1], [9000, 70], 2, 64, seed=15),
             Case(sdq_dev, [200], [9000], 2, 32, seed=16)]
    qs = [torch.randn((c.T, 4 * HD), device=sdq_dev) for c in cases]
    u, scale, zero = q4.make(512, 4096, 64, True, 3)
    w = sdq.Weight4.from_host(u, scale, zero, group=64)
    x = torch.randn((20, 4096), device=sdq_dev)
    kv = torch.randn((1500, 2 * 384), device=sdq_dev)
    calls = [(lambda o, s, i=i: sdq.kv_attention(cases[i].cache, cases[i].batch, qs[i], o, 4, stream=s),
              qs[i].shape) for i in range(2)]
    calls.append((lambda o, s: sdq.q4linear(w, x, o, stream=s), (20, 512)))
    calls.append((lambda o, s: sdq.sdpa(kv, kv, kv, o, 3, qcol=0, kcol=0, vcol=384, stream=s),
                  (1500, 384)))
    own = torch.cuda.Stream()
    outs = [[torch.zeros(shape, device=sdq_dev) for _ in range(9)] for _, shape in calls]
    torch.cuda.synchronize()
    go = threading.Barrier(len(calls))

    def run(i):
        sdq.init(0)
        go.wait()
        for o in outs[i][1:]:
            calls[i][0](o, own)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(len(calls))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for i, (call, _) in enumerate(calls):
        call(outs[i][0], own)
        own.synchronize()
        assert outs[i][0].abs().sum() > 0
        for o in outs[i][1:]:
            assert torch.equal(o, outs[i][0]), i


def test_a_thread_that_ends_waits_for_its_stream(sdq_dev):
    """Calls queued on a thread's own stream are done when the thread is: nothing can wait
    for them afterwards, and the next thread's calls may use the same scratch."""
    import threading

    import torch

    import sdq

    cases = [Case(sdq_dev, [1, 1], [20000, 9000], 2, 64, seed=17 + i) for i in range(2)]
    qs = [torch.randn((c.T, 4 * HD), device=sdq_dev) for c in cases]
    want = [sdq.kv_attention(c.cache, c.batch, q, torch.zeros_like(q), 4) for c, q in zip(cases, qs)]
    outs = [[torch.zeros_like(q) for _ in range(40)] for q in qs]
    torch.cuda.synchronize()

    def run(i):
        sdq.init(0)
        for o in outs[i]:
            sdq.kv_attention(cases[i].cache, cases[i].batch, qs[i], o, 4, stream=2)

    for i in range(2):
        t = threading.Thread(target=run, args=(i,))
        t.start()
        t.join()
    for w, os_ in zip(want, outs):
        for o in os_:
            assert torch.equal(o, w)


@pytest.mark.parametrize("what", ["write", "read", "attention", "norm", "dequant", "linear"])
def test_a_thread_that_ends_waits_for_calls_without_scratch(sdq_dev, what):
    """The same for calls that ask the stream's workspace for nothing: what a thread queued is
    there when it has ended."""
    import threading

    import torch

    import sdq
    import test_gpu_q4linear as q4

    n = 20000
    c = Case(sdq_dev, [n], [n], 2, 64, seed=25)
    x, y = (torch.randn((n, 256), device=sdq_dev) for _ in range(2))
    u, scale, _ = q4.make(8192, 4096, 128, False, 3)
    w = sdq.Weight4.from_host(u, scale, group=128)
    one = torch.randn((1, 4096), device=sdq_dev)
    codes = torch.empty((n, 256), dtype=torch.int8, device=sdq_dev)
    scales = torch.empty(n, device=sdq_dev)
    sdq.act_quant(x, codes, scales)
    fresh = lambda *like: [torch.zeros_like(t) for t in like]  # noqa: E731
    pool = lambda: sdq.KvCache(*fresh(c.cache.k, c.cache.ks, c.cache.v, c.cache.vs))  # noqa: E731
    few = Case(sdq_dev, [1] * 400, [200] * 400, 2, 64, seed=26)  # too few keys to be cut
    q = torch.randn((400, 512), device=sdq_dev)

    def make():  # outputs, and the call that fills them
        if what == "write":
            p = pool()
            return [p.k, p.ks, p.v, p.vs], lambda s: sdq.kv_write(p, c.batch, x, y, stream=s)
        if what == "read":
            o = fresh(x, y)
            return o, lambda s: sdq.kv_read(c.cache, c.batch, *o, stream=s)
        if what == "attention":
            o = fresh(q)
            return o, lambda s: sdq.kv_attention(few.cache, few.batch, q, o[0], 4, stream=s)
        if what == "norm":
            o = fresh(codes, scales, x)
            return o, lambda s: sdq.rmsnorm_quant(x, *o[:2], delta=y, sum_out=o[2], stream=s)
        if what == "dequant":
            o = fresh(x)
            return o, lambda s: sdq.dequant(codes, scales, o[0], stream=s)
        o = [torch.zeros((1, 8192), device=sdq_dev)]
        return o, lambda s: sdq.q4linear(w, one, o[0], stream=s)

    want, call = make()
    call(None)
    assert all(t.float().abs().sum() > 0 for t in want)
    made = [make() for _ in range(24)]
    torch.cuda.synchronize()

    def run():
        sdq.init(0)
        for _ in range(5):
            for _, call in made:
                call(2)  # hipStreamPerThread

    t = threading.Thread(target=run)
    t.start()
    t.join()
    for got, _ in made:
        for a, b in zip(got, want):
            assert torch.equal(a, b)


# ---- a serving step out of all of them ----

def test_serving_step(sdq_dev, oracle):
    """Residual + norm + codes -> q|k|v -> cache -> attention -> 4-bit output Linear
    into the residual, over a prompt and three single tokens, against the same
    steps in 64 bits on the GPU's own codes and cache."""
    import torch

    import sdq
    from test_gpu_q4linear import expected, make

    D, H = 512, 4
    rng = np.random.default_rng(12)
    qw, qs = oracle.quant_rows((rng.standard_normal((3 * D, D)) * 0.04).astype(F))
    wqkv = sdq.Weight.from_host(qw, qs)
    u, sc, z = make(D, D, 64, True, 13)
    sc *= F(0.1)
    wo = sdq.Weight4.from_host(u, sc, z, group=64)
    nw = (1 + 0.1 * rng.standard_normal(D)).astype(F)
    cache = sdq.KvCache.empty(8, 16, H, sdq_dev)
    table = torch.tensor([[5, 2, 7, 0]], dtype=torch.int32, device=sdq_dev)
    total = 0
    for n in (21, 1, 1, 1):
        total += n
        batch = sdq.KvBatch(torch.tensor([0, n], dtype=torch.int32, device=sdq_dev),
                            torch.tensor([total], dtype=torch.int32, device=sdq_dev), table)
        x, d = (rng.standard_normal((n, D)).astype(F) for _ in range(2))
        tx, td = (torch.from_numpy(a).to(sdq_dev) for a in (x, d))
        aq = torch.empty((n, D), dtype=torch.int8, device=sdq_dev)
        asc = torch.empty(n, device=sdq_dev)
        qkv, att = torch.empty((n, 3 * D), device=sdq_dev), torch.empty((n, D), device=sdq_dev)
        sdq.rmsnorm_quant(tx, aq, asc, w=torch.from_numpy(nw).to(sdq_dev), delta=td, sum_out=tx)
        sdq.qlinear_codes(wqkv, aq, asc, qkv)
        sdq.kv_write(cache, batch, qkv[:, D:2 * D], qkv[:, 2 * D:])
        sdq.kv_attention(cache, batch, qkv[:, :D], att, H)
        h = tx.clone()
        sdq.q4linear(wo, att, tx, kind="resid", resid=tx)
        torch.cuda.synchronize()
        want_h, want_q, want_s = __import__("test_gpu_rmsnorm_quant").oracle_norm(x, d, nw, 1e-6)
        assert_bitexact(h.cpu().numpy(), want_h, "sum")
        assert_bitexact(aq.cpu().numpy(), want_q, "codes")
        acc = want_q.astype(np.int64) @ qw.astype(np.int64).T
        y = acc.astype(F) * (want_s[:, None] * qs[None]).astype(F)
        assert_bitexact(qkv.cpu().numpy(), y, "q|k|v")
        c = Case.__new__(Case)
        c.new, c.lens, c.kvh, c.page, c.most, c.pages = [n], [total], H, 16, 4, 8
        c.table, c.start, c.T = table.cpu().numpy(), np.array([0, n]), n
        c.k, c.v = cache.k.cpu().numpy(), cache.v.cpu().numpy()
        c.ks, c.vs = cache.ks.cpu().numpy(), cache.vs.cpu().numpy()
        place = c.table[0, (total - n + np.arange(n)) // 16], slice(None), (total - n + np.arange(n)) % 16
        for got, cols in ((c.k, slice(D, 2 * D)), (c.v, slice(2 * D, 3 * D))):
            codes, _ = codes_of(y[:, cols].reshape(n * H, HD))
            assert_bitexact(got[place], codes.reshape(n, H, HD), "cache")
        want, tol = c.attend(y[:, :D], H, HD**-0.5, True)
        a = att.cpu().numpy()
        assert (np.abs(a - want) <= tol).all()
        o, tol = expected(a, u, sc, z, 64)
        o = want_h + o
        assert (np.abs(tx.cpu().numpy() - o) <= tol + 2.0**-24 * np.abs(o)).all()
