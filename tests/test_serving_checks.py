"""Refusals of the quantized serving operators (CPU: nothing is launched): the C
ABI's own checks, the binding's checks of tensors, and the layout of the structs
that cross between them."""
import ctypes
import os
import re
import shutil
import subprocess

import pytest

torch = pytest.importorskip("torch")

import sdq  # noqa: E402
from conftest import PKG, ROOT  # noqa: E402

P = 0x10000  # an address that is never read: the checks come first


def _refused(match, fn, *args):
    rc = getattr(sdq.load_library(), fn)(*args)
    msg = sdq.load_library().sdq_last_error().decode()
    assert rc == sdq.ERR_INVALID and match in msg, (rc, msg)


def _norm(M=4, K=64, x=P, ldx=64, d=None, ldd=0, w=None, eps=1e-6, s=None, lds=0, aq=P << 8,
          as_=P << 9):
    return x, ldx, d, ldd, M, K, w, eps, s, lds, aq, as_, None


@pytest.mark.parametrize("match,kw", [
    ("negative M", dict(M=-1)), ("K < 1", dict(K=0)), ("at most 2^30", dict(M=2**30 + 1)),
    ("2^22", dict(K=2**22 + 1, ldx=2**23)), ("eps", dict(eps=-1.0)), ("eps", dict(eps=float("nan"))),
    ("eps", dict(eps=float("inf"))), ("null pointer", dict(x=None)), ("null pointer", dict(aq=None)),
    ("null pointer", dict(as_=None)), ("row strides", dict(ldx=63)),
    ("row strides", dict(d=P << 10, ldd=63)), ("row strides", dict(s=P << 10, lds=0)),
    ("overlaps", dict(s=P + 4, lds=64)), ("overlaps", dict(s=P, lds=65)),
    ("overlaps", dict(aq=P + 16)), ("overlaps", dict(as_=P + 1020)),
    ("overlaps", dict(as_=(P << 8) + 8)), ("overlaps", dict(w=P << 10, s=(P << 10) + 128, lds=64))])
def test_rmsnorm_quant(match, kw):
    _refused(match, "sdq_rmsnorm_quant", *_norm(**kw))


def test_dequant_and_codes():
    _refused("negative", "sdq_dequant", P, P, -1, 4, P, None)
    _refused("2^30", "sdq_dequant", P, P, 2**30 + 1, 4, P, None)
    _refused("null", "sdq_dequant", P, None, 2, 4, P << 8, None)
    _refused("overlaps", "sdq_dequant", P, P << 8, 2, 16, P + 16, None)
    _refused("null weight", "sdq_qlinear_codes", None, P, P, 2, 4, None, P << 8, None)
    assert sdq.load_library().sdq_rmsnorm_quant(*_norm(M=0)) == sdq.OK
    assert sdq.load_library().sdq_dequant(None, None, 0, 4, None, None) == sdq.OK


@pytest.mark.parametrize("fn", ["sdq_weight4_upload", "sdq_weight4_upload_device"])
def test_weight4(fn):
    out = ctypes.c_void_p()
    ref = ctypes.byref(out)
    for match, args in (("N 1", (P, P, None, 0, 4, 32)), ("K 1", (P, P, None, 4, 0, 32)),
                        ("2^20", (P, P, None, 2**20 + 1, 4, 32)),
                        ("2^22", (P, P, None, 4, 2**22 + 1, 32)), ("group", (P, P, None, 4, 64, 16)),
                        ("group", (P, P, None, 4, 64, 0)), ("null", (None, P, None, 4, 64, 32)),
                        ("null", (P, None, None, 4, 64, 32))):
        _refused(match, fn, *args, None, ref)
        assert out.value is None
    _refused("null out", fn, P, P, None, 4, 64, 32, None, None)
    lib = sdq.load_library()
    assert lib.sdq_weight4_free(None) == sdq.OK
    _refused("null weight", "sdq_weight4_dims", None, None, None, None)
    _refused("null weight", "sdq_q4linear", None, P, 1, 4, None, P, None)


def _kv(pages=4, page=16, heads=2, k=P, ks=P, v=P, vs=P, q_start=P, lens=P, table=P, nseq=2,
        most=4):
    return (ctypes.byref(sdq.KvCacheView(k, ks, v, vs, pages, page, heads)),
            ctypes.byref(sdq.KvBatchView(q_start, lens, table, nseq, most)))


@pytest.mark.parametrize("match,kw", [
    ("page_size", dict(page=8)), ("page_size", dict(page=24)), ("page_size", dict(page=65536)),
    ("page_size", dict(page=0)), ("page_size", dict(page=-16)), ("kv_heads", dict(heads=0)),
    ("kv_heads", dict(heads=65536)), ("pages", dict(pages=-1)), ("pages", dict(pages=2**31 + 1)),
    ("nseq", dict(nseq=-1)), ("nseq", dict(nseq=65536)), ("max_pages", dict(most=-1)),
    ("max_pages", dict(most=2**26 + 1)), ("null cache", dict(k=None)), ("null cache", dict(vs=None)),
    ("16-byte", dict(v=P + 8)), ("null batch", dict(q_start=None)), ("null batch", dict(lens=None)),
    ("null batch", dict(table=None))])
def test_kv_batches(match, kw):
    c, b = _kv(**kw)
    Q, O = P << 10, P << 12
    _refused(match, "sdq_kv_write", c, b, Q, 256, O, 256, 3, None)
    _refused(match, "sdq_kv_read", c, b, Q, 256, O, 256, 3, None)
    _refused(match, "sdq_kv_attention", c, b, Q, 256, O, 256, 3, 2, 0.1, 1, None)


def test_kv_rows():
    lib = sdq.load_library()
    c, b = _kv()
    Q, O = P << 10, P << 12
    nan = float("nan")
    for fn in ("sdq_kv_write", "sdq_kv_read"):
        _refused("null cache or batch", fn, None, b, Q, 256, O, 256, 3, None)
        _refused("null cache or batch", fn, c, None, Q, 256, O, 256, 3, None)
        _refused("T must", fn, c, b, Q, 256, O, 256, -1, None)
        _refused("T must", fn, c, b, Q, 256, O, 256, 2**30 + 1, None)
        _refused("null k", fn, c, b, None, 256, O, 256, 3, None)
        _refused("null v", fn, c, b, Q, 256, None, 256, 3, None)
        _refused("row stride of k", fn, c, b, Q, 255, O, 256, 3, None)
        _refused("row stride of v", fn, c, b, Q, 256, O, 2**32 + 4, 3, None)
        _refused("16-byte", fn, c, b, Q + 4, 256, O, 256, 3, None)
        _refused("16-byte", fn, c, b, Q, 256, O, 257, 3, None)
    _refused("k and v overlap", "sdq_kv_read", c, b, Q, 256, Q + 512, 256, 3, None)
    _refused("k and v overlap", "sdq_kv_read", c, b, Q, 512, Q + 512, 256, 3, None)
    for match, args in (("multiple of", (Q, 512, O, 512, 3, 3, 0.1)),
                        ("multiple of", (Q, 512, O, 512, 3, 0, 0.1)),
                        ("65535", (Q, 512, O, 512, 3, 65536, 0.1)),
                        ("finite", (Q, 512, O, 512, 3, 4, nan)),
                        ("finite", (Q, 512, O, 512, 3, 4, float("inf"))),
                        ("null q", (None, 512, O, 512, 3, 4, 0.1)),
                        ("null out", (Q, 512, None, 512, 3, 4, 0.1)),
                        ("row stride of q", (Q, 508, O, 512, 3, 4, 0.1)),
                        ("16-byte", (Q, 512, O + 8, 512, 3, 4, 0.1)),
                        ("overlaps", (Q, 512, Q, 512, 3, 4, 0.1)),
                        ("overlaps", (Q, 1024, Q + 1024, 1024, 3, 4, 0.1))):
        _refused(match, "sdq_kv_attention", c, b, *args, 1, None)
    assert lib.sdq_kv_attention(c, b, None, 0, None, 0, 0, 2, 0.1, 1, None) == sdq.OK
    c2, b2 = _kv(heads=1024)
    _refused("T * kv_heads", "sdq_kv_write", c2, b2, Q, 2**17, O, 2**17, 2**24, None)


def test_binding_structs_match_the_header(tmp_path):
    src = tmp_path / "layout.cpp"
    structs = {"sdq_kv_cache": sdq.KvCacheView, "sdq_kv_batch": sdq.KvBatchView}
    lines = ['#include <cstddef>', '#include <cstdio>', '#include "sdq.h"', "int main() {"]
    for c, py in structs.items():
        lines.append(f'printf("%zu\\n", sizeof({c}));')
        lines += [f'printf("%zu\\n", offsetof({c}, {n}));' for n, _ in py._fields_]
    src.write_text("\n".join(lines + ["}"]))
    exe = tmp_path / "layout"
    subprocess.run([shutil.which("g++"), "-I", os.path.join(ROOT, "include"), str(src), "-o",
                    str(exe)], check=True)
    got = [int(n) for n in subprocess.run([str(exe)], capture_output=True, text=True,
                                          check=True).stdout.split()]
    want = []
    for py in structs.values():
        want.append(ctypes.sizeof(py))
        want += [getattr(py, n).offset for n, _ in py._fields_]
    assert got == want


def _raises(match, fn, *a, **k):
    with pytest.raises(sdq.SdqError, match=match) as e:
        fn(*a, **k)
    assert e.value.code == sdq.ERR_INVALID


def test_binding_tensors():
    f, i8, u8 = torch.zeros, lambda *s: torch.zeros(*s, dtype=torch.int8), lambda *s: torch.zeros(
        *s, dtype=torch.uint8)
    x, aq, s = f(4, 64), i8(4, 64), f(4)
    _raises("on the GPU", sdq.rmsnorm_quant, x, aq, s)
    _raises("delta: shape", sdq.rmsnorm_quant, x, aq, s, delta=f(4, 63))
    _raises("sum_out: dtype", sdq.rmsnorm_quant, x, aq, s, sum_out=x.double())
    _raises("w: shape", sdq.rmsnorm_quant, x, aq, s, w=f(63))
    _raises("aq: shape", sdq.rmsnorm_quant, x, i8(3, 64), s)
    _raises("as: shape", sdq.rmsnorm_quant, x, aq, f(5))
    _raises("x: must be 2-D", sdq.rmsnorm_quant, f(64, 4).t(), aq, s)
    _raises("y: shape", sdq.dequant, aq, s, f(4, 63))
    _raises("group", sdq.Weight4.from_host, u8(4, 8).numpy(), f(4, 1).numpy(), group=16)
    _raises("k: 17", sdq.Weight4.from_host, u8(4, 8).numpy(), f(4, 1).numpy(), k=17, group=32)
    _raises("scale: shape", sdq.Weight4.from_host, u8(4, 32).numpy(), f(4, 1).numpy(), group=32)
    _raises("zero: shape", sdq.Weight4.from_host, u8(4, 8).numpy(), f(4, 1).numpy(),
            u8(4, 2).numpy(), group=32)
    _raises("on the GPU", sdq.Weight4.from_device, u8(4, 8), f(4, 1), group=32)
    _raises("not a live Weight4", sdq.q4linear, None, x, x)
    w4 = sdq.Weight4(None, 8, 64, 32)
    _raises("not a live Weight4", sdq.q4linear, w4, x, x)
    _raises("page_size", sdq.KvCache.empty, 2, 24, 1, "cpu")
    cache = sdq.KvCache.empty(2, 16, 1, "cpu")
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    batch = sdq.KvBatch(i32(2), i32(1), i32(1, 3))
    kv = f(4, 128)
    _raises("on the GPU", sdq.kv_write, cache, batch, kv, kv)
    _raises("v: shape", sdq.kv_write, cache, batch, kv, f(3, 128))
    _raises("k: shape", sdq.kv_read, cache, batch, f(4, 127), kv)
    _raises("q: shape", sdq.kv_attention, cache, batch, kv, kv, 2)
    _raises("q_start: shape", sdq.KvBatch, i32(3), i32(1), i32(1, 3))
    _raises("lens: dtype", sdq.KvBatch, i32(2), f(1), i32(1, 3))
    _raises("expected a KvCache and a KvBatch", sdq.kv_attention, cache, None, kv, kv, 1)
    with pytest.raises(AttributeError):
        batch.lens = i32(1)
    _raises("KvCache", sdq.kv_attention, None, batch, kv, kv, 1)
    _raises("cache.ks: shape", sdq.KvCache, cache.k, f(2, 1, 15), cache.v, cache.vs)
    _raises("cache.v: must be contiguous", sdq.KvCache, cache.k, cache.ks,
            torch.zeros(2, 1, 128, 16, dtype=torch.int8).transpose(2, 3), cache.vs)


def test_every_stream_argument_is_known_to_its_thread():
    """A thread waits as it ends for what it queued on its hipStreamPerThread: each entry point's
    stream passes stream_of, which notes the thread, or goes to an entry point that does so."""
    with open(os.path.join(PKG, "csrc", "sdq_api.hip")) as f:
        text = f.read()
    with open(os.path.join(ROOT, "include", "sdq.h")) as f:
        header = f.read()
    names = [m.group(1) for m in re.finditer(r"^int (sdq_\w+)\(([^;{]*)\);", header, re.M)
             if re.search(r"void ?\* ?(stream|waiter)", m.group(2))]
    assert len(names) >= 30 and "sdq_kv_write" in names and "sdq_stream_wait" in names
    for name in names:
        body = re.search(r"^int %s\([^{;]*\) \{\n(.*?)^\}" % name, text, re.M | re.S).group(1)
        assert "stream_of(" in body or re.search(r"\bsdq_\w+\([^;]*\bstream\b", body), name
    assert text.count("static_cast<hipStream_t>") == 1  # stream_of's own


def test_column_blocks_that_share_a_column():
    """A sum beside x in one array may not reach into its columns, nor have another stride."""
    for s in (P + 63 * 4, P + 129 * 4, P + (192 + 63) * 4):
        _refused("overlaps", "sdq_rmsnorm_quant", *_norm(x=P, ldx=192, s=s, lds=192))
        _refused("overlaps", "sdq_rmsnorm_quant", *_norm(d=P << 10, ldd=192, s=s - P + (P << 10),
                                                         lds=192))
    _refused("overlaps", "sdq_rmsnorm_quant", *_norm(x=P, ldx=192, s=P + 64 * 4, lds=193))
