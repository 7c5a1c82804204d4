"""sdq_q4linear (4-bit weights with group scales and zero points) against the
product in 64 bits.

Tolerance, from the kernels' arithmetic, the larger of their two forms'. As bytes
(up to five rows): every x enters its group as a multiple of 2^(E - 22), 2^E <=
max|x| of the group, so it is off by at most 2^-23 of that maximum; sums inside a
group are exact. As fp16 parts, scaled so that the largest value of a row's range
lies in [2^14, 2^15): two roundings by at most 2^-11 of what they round, 2^-22 of
every value, or half of fp16's smallest step, 2^-25, which is 2^-39 of the largest;
a group's sum is 2 * group / 32 MFMAs of 32 exact products, of which each is
counted with 8 roundings to fp32 of 2^-24. Both: three roundings a group and at
most G + 40 over the G groups, where waves, parts and ranges join."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

F = np.float32


def make(N, K, group, zeros, seed):
    rng = np.random.default_rng(seed)
    u = rng.integers(0, 256, (N, (K + 1) // 2), dtype=np.uint8)  # odd K: the last half is noise
    G = -(-K // group)
    scale = (0.01 * rng.uniform(0.2, 2, (N, G))).astype(F)
    zero = rng.integers(0, 16, (N, G), dtype=np.uint8) if zeros else None
    return u, scale, zero


def weights64(u, scale, zero, K, group):
    c = np.stack([u & 15, u >> 4], -1).reshape(u.shape[0], -1)[:, :K].astype(np.float64)
    at = np.arange(K) // group
    z = 8.0 if zero is None else zero.astype(np.float64)[:, at]
    return (c - z), scale.astype(np.float64)[:, at]


def expected(x, u, scale, zero, group):
    """The product and its tolerance."""
    M, K = x.shape
    c, s = weights64(u, scale, zero, K, group)
    x = x.astype(np.float64)
    G = -(-K // group)
    y, size, coarse = 0.0, 0.0, 0.0
    for g in range(G):
        k = slice(g * group, min(K, (g + 1) * group))
        part = x[:, k] @ (c[:, k] * s[:, k]).T
        y = y + part
        size = size + np.abs(part)
        coarse = coarse + np.abs(x[:, k]).max(1)[:, None] * np.abs(c[:, k] * s[:, k]).sum(1)[None]
    products = np.abs(x) @ np.abs(c * s).T
    parts = ((2.0**-22 + 2 * group / 32 * 8 * 2.0**-24) * products
             + 2.0**-39 * np.abs(x).max(1)[:, None] * np.abs(c * s).sum(1)[None])
    return y, np.maximum(parts, 2.0**-23 * coarse) + (G + 43) * 2.0**-24 * size


def gelu(y):
    return y / (1 + np.exp(-2 * np.sqrt(2 / np.pi) * (y + 0.044715 * y**3)))


def call(sdq_dev, u, scale, zero, group, x, host=True, **kw):
    import torch

    import sdq

    K = x.shape[1]
    t = lambda a: None if a is None else torch.from_numpy(a).to(sdq_dev)  # noqa: E731
    w = (sdq.Weight4.from_host(u, scale, zero, k=K, group=group) if host else
         sdq.Weight4.from_device(t(u), t(scale), t(zero), k=K, group=group))
    out = torch.full((x.shape[0], u.shape[0]), 7.0, device=sdq_dev)
    sdq.q4linear(w, t(x), out, **{k: t(v) if isinstance(v, np.ndarray) else v
                                  for k, v in kw.items()})
    return out.cpu().numpy()


@pytest.mark.parametrize("M", [1, 2, 5, 6, 13, 16, 17, 32, 33, 70])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
def test_rows_groups_zeros(sdq_dev, M, group, zeros):
    N, K = 200, 1296  # an odd number of 16-wide blocks; K ends inside a unit and a group
    u, scale, zero = make(N, K, group, zeros, M)
    x = np.random.default_rng(M + 1).standard_normal((M, K)).astype(F)
    want, tol = expected(x, u, scale, zero, group)
    got = call(sdq_dev, u, scale, zero, group, x)
    assert (np.abs(got - want) <= tol).all(), np.max(np.abs(got - want) / tol)


@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 15, 31), (2, 17, 33), (1, 16, 128), (3, 1, 129),
                                   (1, 67, 65), (7, 33, 4099), (1, 4096, 14336), (20, 301, 14336),
                                   (1, 18432, 512), (5, 70, 16390), (32, 2050, 515), (1, 40, 70001),
                                   (9, 24, 70001)])
@pytest.mark.parametrize("zeros", [False, True])
def test_sizes(sdq_dev, M, N, K, zeros):
    group = (32, 64, 128)[(M + N + K) % 3]
    u, scale, zero = make(N, K, group, zeros, K)
    x = np.random.default_rng(N).standard_normal((M, K)).astype(F)
    x[:, ::97] *= 50  # a few channels far above the others
    want, tol = expected(x, u, scale, zero, group)
    got = call(sdq_dev, u, scale, zero, group, x, host=False)
    assert (np.abs(got - want) <= tol).all(), np.max(np.abs(got - want) / tol)


@pytest.mark.parametrize("M", [1, 4, 12, 31])
@pytest.mark.parametrize("kind,gate_fma", [("none", True), ("gelu", True), ("gated", True),
                                           ("gated", False), ("resid", True)])
@pytest.mark.parametrize("bias", [False, True])
def test_epilogues(sdq_dev, M, kind, gate_fma, bias):
    N, K = 130, 640
    u, scale, zero = make(N, K, 64, True, 3)
    rng = np.random.default_rng(4)
    x = rng.standard_normal((M, K)).astype(F)
    b = rng.standard_normal(N).astype(F) if bias else None
    gate = rng.standard_normal(N).astype(F)
    resid = rng.standard_normal((M, N)).astype(F)
    y, tol = expected(x, u, scale, zero, 64)
    if bias:
        y = y + b
        tol = tol + 2.0**-24 * np.abs(y)
    kw = {"bias": b}
    if kind == "gelu":  # slope at most 1.13; the hardware's exp2 and reciprocal: sdq_qlinear's 1e-6
        want, tol = gelu(y), 1.13 * tol + 1e-6 * (1 + np.abs(y))
    elif kind == "gated":
        want = resid + y * gate
        tol = np.abs(gate) * tol + 2.0**-24 * (np.abs(want) + np.abs(y * gate))
        kw.update(gate=gate, resid=resid, gate_fma=gate_fma)
    elif kind == "resid":
        want = resid + y
        tol = tol + 2.0**-24 * np.abs(want)
        kw.update(resid=resid)
    else:
        want = y
    got = call(sdq_dev, u, scale, zero, 64, x, kind=kind, **kw)
    assert (np.abs(got - want) <= tol).all(), np.max(np.abs(got - want) / tol)


@pytest.mark.parametrize("M", [1, 3, 8, 32])
def test_special_values(sdq_dev, M):
    """Zero rows and groups, tiny, huge and denormal values; a NaN or an infinity
    makes its own row NaN and no other."""
    N, K, group = 48, 512, 32
    u, scale, zero = make(N, K, group, True, 8)
    rng = np.random.default_rng(9)
    for factor in (0.0, 1e-38, 1e-30, 1e30):
        x = (rng.standard_normal((M, K)) * factor).astype(F)
        x[:, 64:96] = 0
        want, tol = expected(x, u, scale, zero, group)
        got = call(sdq_dev, u, scale, zero, group, x)
        # results below the normal range are off by a denormal's spacing a step
        assert (np.abs(got - want) <= tol + 64 * 2.0**-149).all(), factor
    for bad in (np.nan, np.inf, -np.inf):
        x = rng.standard_normal((M, K)).astype(F)
        x[M - 1, 77] = bad
        got = call(sdq_dev, u, scale, zero, group, x)
        assert np.isnan(got[M - 1]).all()
        if M > 1:
            want, tol = expected(x[:M - 1], u, scale, zero, group)
            assert (np.abs(got[:M - 1] - want) <= tol).all()


@pytest.mark.parametrize("M", [1, 3, 5, 6, 17, 32])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_rows_near_the_largest_float(sdq_dev, M, group):
    """Values up to fp32's largest whose results are finite: dense rows of one sign, where a
    group's sum with the codes alone passes fp32's range, rows of both signs, and one such value
    beside ordinary ones."""
    N, K = 70, 1024
    u, scale, zero = make(N, K, group, True, 31)
    rng = np.random.default_rng(32)
    top = float(np.finfo(F).max)
    for size, sc in ((1e36, 1e-3), (top, 2e-6), (top, 1e-30)):
        one = np.full((M, K), size)
        two = size * rng.uniform(-1, 1, (M, K))
        few = rng.standard_normal((M, K))
        few[:, 300] = size
        for x in (one, two, few):
            x = x.astype(F)
            s = (scale * (sc / 0.02)).astype(F)
            codes = np.where(u & 1, u | 0x77, u)  # more of one sign
            want, tol = expected(x, codes, s, zero, group)
            assert (np.abs(want) < top / 4).all()
            got = call(sdq_dev, codes, s, zero, group, x)
            bad = ~(np.abs(got - want) <= tol + 64 * 2.0**-149)
            assert not bad.any(), (size, sc, np.argwhere(bad)[:3], got[bad][:3], want[bad][:3])


@pytest.mark.parametrize("M", [1, 5, 6, 32])
@pytest.mark.parametrize("group", [32, 128])
def test_range_of_weight_scales(sdq_dev, M, group):
    """Weight scales up to 2^100 of either sign, and as small, with values the other way round."""
    N, K = 70, 640
    u, scale, zero = make(N, K, group, True, 33)
    rng = np.random.default_rng(34)
    for e in (-120, -60, 60, 99):
        s = (scale / F(0.02) * F(2.0)**e * rng.choice([-1, 1], scale.shape)).astype(F)
        x = (rng.standard_normal((M, K)) * 2.0**-e).astype(F)
        want, tol = expected(x, u, s, zero, group)
        got = call(sdq_dev, u, s, zero, group, x)
        assert (np.abs(got - want) <= tol).all(), e


def test_in_place_residual_and_two_streams(sdq_dev):
    """resid is Y; two calls of different sizes at once on two streams."""
    import torch

    import sdq

    todo = []
    for i, (M, N, K) in enumerate(((1, 4096, 5120), (16, 1024, 2048))):
        u, scale, zero = make(N, K, 128, i == 0, i)
        rng = np.random.default_rng(20 + i)
        x, r = rng.standard_normal((M, K)).astype(F), rng.standard_normal((M, N)).astype(F)
        todo.append((sdq.Weight4.from_host(u, scale, zero, group=128),
                     torch.from_numpy(x).to(sdq_dev), r, expected(x, u, scale, zero, 128),
                     torch.cuda.Stream()))
    torch.cuda.synchronize()
    outs = [torch.from_numpy(r).to(sdq_dev) for _, _, r, _, _ in todo]
    torch.cuda.synchronize()
    for _ in range(3):
        for o, (w, x, r, _, st) in zip(outs, todo):
            with torch.cuda.stream(st):
                o.copy_(torch.from_numpy(r), non_blocking=False)
                sdq.q4linear(w, x, o, kind="resid", resid=o)
    torch.cuda.synchronize()
    for o, (_, _, r, (y, tol), _) in zip(outs, todo):
        want = r + y
        assert (np.abs(o.cpu().numpy() - want) <= tol + 2.0**-24 * np.abs(want)).all()


@pytest.mark.parametrize("M", [1, 12, 32])
def test_captured(sdq_dev, M):
    """One eager call, then a capture; replays with new inputs give the eager bits,
    and running again gives the same bits."""
    import torch

    import sdq

    N, K = 1024, 4096
    u, scale, zero = make(N, K, 64, True, 5)
    w = sdq.Weight4.from_host(u, scale, zero, group=64)
    x, out = torch.empty((M, K), device=sdq_dev), torch.empty((M, N), device=sdq_dev)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        sdq.q4linear(w, x.zero_(), out)
    side.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        sdq.q4linear(w, x, out)
    for seed in range(4):
        x.copy_(torch.from_numpy(np.random.default_rng(seed).standard_normal((M, K)).astype(F)))
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            g.replay()
        torch.cuda.synchronize()
        got = out.clone()
        again = torch.empty_like(out)
        sdq.q4linear(w, x, again)
        torch.cuda.synchronize()
        assert torch.equal(got, again), seed
