"""The paged cache's operators at the ends of their ranges: logits past fp32, against the
definitions in 64 bits. Tolerances as in tests/test_gpu_kv_more.py."""
import numpy as np
import pytest

from conftest import assert_bitexact
from test_gpu_kv_cache import F, HD
from test_gpu_kv_more import More

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
