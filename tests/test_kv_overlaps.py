"""Refusals of the paged attentions and of eviction where an output meets another array (CPU: nothing
is launched). Without a device a call that passes its checks ends with another error."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

import sdq  # noqa: E402
from test_serving_checks import P, _kv, _refused  # noqa: E402

# pages 4, page 16, heads 2: codes of 16 KiB, scales of 512 bytes; nseq 2, most 4
AT = dict(k=P, ks=P << 1, v=P << 2, vs=P << 3, q_start=P << 4, lens=P << 5, table=P << 6)
SIZE = dict(k=16384, ks=512, v=16384, vs=512, q_start=12, lens=8, table=32)
S = dict(s_start=P << 7, s_lens=P << 8, s_table=P << 9)
S_SIZE = dict(s_start=16, s_lens=12, s_table=60)
Q, O, W, TO, L, K = (P << n for n in range(10, 16))
ROW = 1024  # 2 heads of 128 floats

pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="what passes would run")


def _call(fn, w=W, q=Q, out=O, ldo=256, T=3):
    c, b = _kv(**AT)
    shared = ctypes.byref(sdq.KvSharedView(S["s_start"], S["s_lens"], S["s_table"], 3, 5))
    rows = (q, 256, out, ldo, T, 2, 0.1)
    return {"sdq_kv_attention": (c, b) + rows + (1, None),
            "sdq_kv_cross_attention": (c, b) + rows + (None,),
            "sdq_kv_attention_shared": (c, shared, b) + rows + (1, None),
            "sdq_kv_attention_weights": (c, b, w) + rows + (1, None)}[fn]


def _passes(fn, *args):
    rc = getattr(sdq.load_library(), fn)(*args)
    assert rc != sdq.ERR_INVALID, sdq.load_library().sdq_last_error().decode()


FNS = ["sdq_kv_attention", "sdq_kv_cross_attention", "sdq_kv_attention_shared",
       "sdq_kv_attention_weights"]


def _edges(at, size, n):
    """Addresses of an output of n bytes that meets an array's first and last bytes, and of one
    that ends and begins beside it (rows are 16-byte aligned)."""
    up = -(-size // 16) * 16
    return (at - n + 16, at, at + (size - 1) // 16 * 16), (at - n, at + up)


@pytest.mark.parametrize("fn", FNS)
def test_out(fn):
    arrays = {**AT, **(S if fn.endswith("shared") else {})}
    sizes = {**SIZE, **S_SIZE}
    for name, at in arrays.items():
        bad, good = _edges(at, sizes[name], 3 * ROW)
        for out in bad:
            _refused("out overlaps", fn, *_call(fn, out=out))
        for out in good:
            _passes(fn, *_call(fn, out=out))


@pytest.mark.parametrize("fn", FNS)
def test_out_rows_apart(fn):
    """An array between two rows of out meets neither; one byte further it does."""
    ldo = 256 + 16
    for i in (1, 2):
        at = AT["table"] - (i * ldo * 4 - 64)  # the gap before row i begins with the table
        _passes(fn, *_call(fn, out=at, ldo=ldo))
        _refused("out overlaps", fn, *_call(fn, out=at - 48, ldo=ldo))
        _refused("out overlaps", fn, *_call(fn, out=at + 16, ldo=ldo))
    _passes(fn, *_call(fn, out=AT["table"] - 3 * ldo * 4 + 64, ldo=ldo))  # behind the last row


def test_weights():
    fn = "sdq_kv_attention_weights"
    for name in AT:
        for w in (AT[name] - 508, AT[name] + SIZE[name] - 4):
            _refused("weights overlaps", fn, *_call(fn, w=w))
        for w in (AT[name] - 512, AT[name] + SIZE[name]):
            _passes(fn, *_call(fn, w=w))
    for at in (Q, O):
        for w in (at - 508, at + 3 * ROW - 4):
            _refused("weights overlaps", fn, *_call(fn, w=w))
        for w in (at - 512, at + 3 * ROW):
            _passes(fn, *_call(fn, w=w))
    _passes(fn, *_call(fn, w=O + ROW, ldo=256 + 128))  # between two rows
    _refused("weights overlaps", fn, *_call(fn, w=O + ROW + 4, ldo=256 + 128))


def _evict(w=W, to=TO, to_lens=L, kept=K, **at):
    c, b = _kv(**{**AT, **at})
    return "sdq_kv_evict", c, b, w, 0, 0, 16, to, 1, to_lens, kept, None


def test_evict():
    """Targets: 8 bytes of to_table and to_lens, 256 of kept, 512 of weights."""
    _passes(*_evict())
    _passes(*_evict(to_lens=AT["q_start"]))  # not read
    reads = {"lens": 8, "table": 32}
    for name, n in reads.items():
        for kw, size in (("w", 512), ("to_lens", 8), ("kept", 256)):
            for at in (AT[name] - size + 4, AT[name] + n - 4):
                _refused("overlaps", *_evict(**{kw: at}))
            for at in (AT[name] - size, AT[name] + n):
                _passes(*_evict(**{kw: at}))
        for pool in ("k", "ks", "v", "vs"):  # the cache is written too
            _refused("overlaps", *_evict(**{name: AT[pool] + SIZE[pool] - 4}))
            _passes(*_evict(**{name: AT[pool] + SIZE[pool]}))
    for kw, size in (("w", 512), ("to_lens", 8), ("kept", 256)):
        _refused("overlaps", *_evict(**{kw: TO + 4}))
        _refused("overlaps", *_evict(**{kw: TO - size + 4}))
        _passes(*_evict(**{kw: TO + 8}))
        for pool in ("k", "ks", "v", "vs"):
            _refused("overlaps", *_evict(**{kw: AT[pool] + SIZE[pool] - 4}))
    for pool in ("k", "ks", "v", "vs"):
        _refused("overlaps", *_evict(to=AT[pool] + SIZE[pool] - 4))
    _refused("overlaps", *_evict(to_lens=W + 508))
    _refused("overlaps", *_evict(kept=W - 252))
    _refused("overlaps", *_evict(kept=L - 252))
