"""sdq_rmsnorm_quant, sdq_dequant and sdq_qlinear_codes against the definition in
64 bits. Codes, scales and sums are compared exactly: the kernel's 64-bit norm
and the test's differ by about 1e-16, and would have to lie that near to a
rounding edge of the fp32 value to tell (a chance of ~1e-9 a value)."""
import numpy as np
import pytest

from conftest import assert_bitexact

pytestmark = pytest.mark.gpu

F = np.float32


def codes_of(y):
    """The row quantizer's steps (sdq.h) on fp32 rows, NaN and overflow included."""
    with np.errstate(all="ignore"):
        a = np.where(np.isnan(y), F(0), np.abs(y))
        sc = (a.max(1) / F(127)).astype(F)
        sc[sc == 0] = 1
        t = np.rint((y * (F(1) / sc)[:, None]).astype(F))
        ok = (t >= F(-2147483648)) & (t < F(2147483648))
        return np.where(ok, np.clip(np.where(ok, t, 0), -127, 127), -127).astype(np.int8), sc


def oracle_norm(x, d, w, eps):
    with np.errstate(all="ignore"):
        h = x if d is None else (x + d).astype(F)
        u = h.astype(np.float64)
        inv = 1 / np.sqrt((u * u).sum(1) / x.shape[1] + np.float64(F(eps)))
        y = (u * inv[:, None] * (1.0 if w is None else w.astype(np.float64))).astype(F)
    return (h,) + codes_of(y)


def rows(M, K, seed):
    rng = np.random.default_rng(seed)
    x = (rng.standard_normal((M, K)) * rng.uniform(0.05, 20, (M, 1))).astype(F)
    x[:, rng.random(K) < 0.01] *= 40
    return x


def run(sdq_dev, x, d, w, eps, pad=0, sum_out=None, offset=0):
    """The call on device copies; pad: extra columns behind every row of x and d;
    offset: floats past a 16-byte boundary."""
    import torch

    import sdq

    M, K = x.shape

    def put(a):
        if a is None:
            return None
        t = torch.full((M * (K + pad) + offset,), 7.0, device=sdq_dev)[offset:].view(M, K + pad)[:, :K]
        t.copy_(torch.from_numpy(a))
        return t

    tx, td = put(x), put(d)
    tw = None if w is None else torch.from_numpy(w).to(sdq_dev)
    s = {"x": tx, "d": td, "new": torch.empty((M, K), device=sdq_dev), None: None}[sum_out]
    aq = torch.full((M, K), 99, dtype=torch.int8, device=sdq_dev)
    asc = torch.full((M,), -1.0, device=sdq_dev)
    sdq.rmsnorm_quant(tx, aq, asc, w=tw, delta=td, sum_out=s, eps=eps)
    torch.cuda.synchronize()
    return (None if s is None else s.cpu().numpy()), aq.cpu().numpy(), asc.cpu().numpy(), tx, td


# every register form (64 / 256 / 1024 threads a row, each number of groups), its
# edges, odd lengths, and the re-reading form past 16384
@pytest.mark.parametrize("M,K", [(1, 1), (3, 7), (5, 64), (9, 256), (6, 257), (7, 512), (4, 513),
                                 (33, 1024), (2, 1027), (600, 2048), (530, 2052), (1, 4096),
                                 (700, 4096), (521, 4100), (3, 5120), (1030, 5120), (515, 6148),
                                 (2, 8192), (513, 8192), (3, 8196), (2, 16384), (2, 16387),
                                 (3, 20000)])
@pytest.mark.parametrize("delta", [False, True])
def test_norm_codes(sdq_dev, M, K, delta):
    x = rows(M, K, M + K)
    d = rows(M, K, M + K + 1) if delta else None
    w = (1 + 0.1 * np.random.default_rng(3).standard_normal(K)).astype(F)
    h, q, s = oracle_norm(x, d, w, 1e-6)
    gh, gq, gs, _, _ = run(sdq_dev, x, d, w, 1e-6, sum_out="new")
    assert_bitexact(gh, h, "sum")
    assert_bitexact(gs, s, "scales")
    assert_bitexact(gq, q, "codes")


@pytest.mark.parametrize("K", [300, 1024, 4096, 20001])
@pytest.mark.parametrize("sum_out", [None, "x", "d"])
@pytest.mark.parametrize("pad,offset", [(0, 0), (4, 0), (3, 1)])
def test_strides_aliases_and_alignment(sdq_dev, K, sum_out, pad, offset):
    x, d = rows(5, K, 1), rows(5, K, 2)
    h, q, s = oracle_norm(x, d, None, 1e-5)
    gh, gq, gs, tx, td = run(sdq_dev, x, d, None, 1e-5, pad=pad, sum_out=sum_out, offset=offset)
    assert_bitexact(gq, q, "codes")
    assert_bitexact(gs, s, "scales")
    assert_bitexact(tx.cpu().numpy(), h if sum_out == "x" else x, "x")
    assert_bitexact(td.cpu().numpy(), h if sum_out == "d" else d, "delta")
    if pad:  # what lies behind the rows stays
        assert (tx.as_strided((4, pad), (K + pad, 1), tx.storage_offset() + K) == 7).all()


@pytest.mark.parametrize("M,K", [(1, 300), (5, 300), (7, 4096), (600, 1024)])
def test_column_blocks_of_one_array(sdq_dev, M, K):
    """x, delta and sum side by side in one array, in any order, and what stands beside them."""
    import torch

    import sdq

    x, d = rows(M, K, 41), rows(M, K, 42)
    w = np.ones(K, F)
    h, q, s = oracle_norm(x, d, w, 1e-6)
    for order in ((0, 1, 2), (2, 1, 0), (1, 2, 0)):
        wide = torch.full((M, 3 * K + 4), 7.0, device=sdq_dev)
        tx, td, th = (wide[:, i * K:(i + 1) * K] for i in order)
        tx.copy_(torch.from_numpy(x)), td.copy_(torch.from_numpy(d))
        aq = torch.empty((M, K), dtype=torch.int8, device=sdq_dev)
        asc = torch.empty(M, device=sdq_dev)
        sdq.rmsnorm_quant(tx, aq, asc, w=torch.from_numpy(w).to(sdq_dev), delta=td, sum_out=th)
        assert_bitexact(th.cpu().numpy(), h, "sum")
        assert_bitexact(aq.cpu().numpy(), q, "codes")
        assert_bitexact(asc.cpu().numpy(), s, "scales")
        assert_bitexact(tx.cpu().numpy(), x, "x")
        assert_bitexact(td.cpu().numpy(), d, "delta")
        assert (wide[:, 3 * K:] == 7).all()


@pytest.mark.parametrize("K", [64, 1000, 4096, 17000])
def test_special_rows(sdq_dev, K):
    """Zero, constant, tiny, huge, infinite and NaN rows; eps 0."""
    x = rows(8, K, 5)
    x[0] = 0
    x[1] = -1.5
    x[2] *= F(1e-30)
    x[3] *= F(1e18)
    x[4, 3] = np.nan
    x[5, 2] = np.inf
    x[6] = 0
    x[6, K - 1] = 3
    w = np.ones(K, F)
    for eps in (1e-6, 0.0):
        h, q, s = oracle_norm(x, None, w, eps)
        gh, gq, gs, _, _ = run(sdq_dev, x, None, w, eps, sum_out="new")
        assert_bitexact(gs, s, "scales")
        assert_bitexact(gq, q, "codes")


def test_dequant(sdq_dev):
    import torch

    import sdq

    rng = np.random.default_rng(9)
    for M, K in ((1, 1), (3, 5), (70, 1024), (1000, 4099)):
        q = rng.integers(-128, 128, (M, K)).astype(np.int8)
        s = rng.standard_normal(M).astype(F)
        y = torch.empty((M, K), device=sdq_dev)
        sdq.dequant(torch.from_numpy(q).to(sdq_dev), torch.from_numpy(s).to(sdq_dev), y)
        assert_bitexact(y.cpu().numpy(), q.astype(F) * s[:, None], "dequant")


@pytest.mark.parametrize("M,K,N", [(1, 512, 256), (3, 1000, 130), (64, 4096, 512), (300, 998, 516),
                                   (513, 14336, 384), (2100, 512, 2048)])
def test_qlinear_codes_equals_qlinear(sdq_dev, oracle, M, K, N):
    """Codes of act_quant through every GEMM form: qlinear's own bits."""
    import torch

    import sdq

    q, s = oracle.quant_rows(rows(N, K, 11) * F(0.02))
    w = sdq.Weight.from_host(q, s)
    A = torch.from_numpy(rows(M, K, 12)).to(sdq_dev)
    aq = torch.empty((M, K), dtype=torch.int8, device=sdq_dev)
    asc = torch.empty(M, device=sdq_dev)
    sdq.act_quant(A, aq, asc)
    bias, gate = torch.randn(N, device=sdq_dev), torch.randn(N, device=sdq_dev)
    resid = torch.randn((M, N), device=sdq_dev)
    for kind in ("none", "gelu", "gated", "resid"):
        kw = dict(kind=kind, bias=bias, gate=gate if kind == "gated" else None,
                  resid=resid if kind in ("gated", "resid") else None)
        a, b = torch.empty((M, N), device=sdq_dev), torch.empty((M, N), device=sdq_dev)
        sdq.qlinear(w, A, a, **kw)
        sdq.qlinear_codes(w, aq, asc, b, **kw)
        assert_bitexact(b.cpu().numpy(), a.cpu().numpy(), kind)
    if oracle:
        acc = torch.empty((M, N), dtype=torch.int32, device=sdq_dev)
        sdq.qlinear_codes(w, aq, asc, acc, kind="acc")
        got = aq.cpu().numpy()[:2].astype(np.int64) @ q.astype(np.int64).T
        assert (acc.cpu().numpy()[:2] == got).all()


def test_norm_then_linears_captured(sdq_dev, oracle):
    """Norm and codes once, two Linears on them; captured and replayed with new
    inputs, eager work between: the eager bits every time."""
    import torch

    import sdq

    M, K = 70, 1024
    ws = []
    for i, N in enumerate((512, 384)):
        q, s = oracle.quant_rows(rows(N, K, 20 + i) * F(0.02))
        ws.append(sdq.Weight.from_host(q, s))
    x, d = (torch.empty((M, K), device=sdq_dev) for _ in range(2))
    w = torch.rand(K, device=sdq_dev) + 0.5
    aq, asc = torch.empty((M, K), dtype=torch.int8, device=sdq_dev), torch.empty(M, device=sdq_dev)
    outs = [torch.empty((M, wt.N), device=sdq_dev) for wt in ws]

    def step():
        sdq.rmsnorm_quant(x, aq, asc, w=w, delta=d, sum_out=x)
        for wt, o in zip(ws, outs):
            sdq.qlinear_codes(wt, aq, asc, o)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        step()
    for seed in range(4):
        a, b = (torch.from_numpy(rows(M, K, 30 + seed + 9 * i)).to(sdq_dev) for i in range(2))
        x.copy_(a), d.copy_(b)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            g.replay()
        torch.cuda.synchronize()
        got = [x.clone(), aq.clone(), asc.clone()] + [o.clone() for o in outs]
        x.copy_(a)
        step()
        torch.cuda.synchronize()
        for i, (p, r) in enumerate(zip(got, [x, aq, asc] + outs)):
            assert torch.equal(p, r), (seed, i)
