"""Refusals of the paged cache's cross attention, shared beginnings, counted weights and
eviction (CPU: nothing is launched), the layout of the struct that is new, the work plan over
shared parts, and the hazard scans over the kernels."""
import ctypes
import os
import shutil
import subprocess

import pytest

torch = pytest.importorskip("torch")

import sdq  # noqa: E402
from conftest import PKG, ROOT  # noqa: E402
from test_mfma_hazards import scan, scan_c  # noqa: E402
from test_serving_checks import P, _kv, _raises, _refused  # noqa: E402
from test_store_hazards import CSRC, HIPCC, _scan, _scan_sgpr  # noqa: E402

Q, O, W = P << 10, P << 12, P << 14


def _shared(s_start=P, lens=P, table=P, n=1, most=4):
    return ctypes.byref(sdq.KvSharedView(s_start, lens, table, n, most))


def _calls(c, b, rows=(Q, 256, O, 256, 3, 2, 0.1)):
    return (("sdq_kv_cross_attention", (c, b) + rows + (None,)),
            ("sdq_kv_attention_shared", (c, _shared(), b) + rows + (1, None)),
            ("sdq_kv_attention_weights", (c, b, W) + rows + (1, None)))


@pytest.mark.parametrize("match,kw", [
    ("page_size", dict(page=8)), ("page_size", dict(page=24)), ("kv_heads", dict(heads=0)),
    ("pages", dict(pages=-1)), ("nseq", dict(nseq=65536)), ("max_pages", dict(most=2**26 + 1)),
    ("null cache", dict(k=None)), ("null cache", dict(vs=None)), ("16-byte", dict(v=P + 8)),
    ("null batch", dict(lens=None)), ("null batch", dict(table=None))])
def test_batches(match, kw):
    c, b = _kv(**kw)
    for fn, args in _calls(c, b):
        _refused(match, fn, *args)
    _refused(match, "sdq_kv_evict", c, b, W, 0, 0, 16, Q, 1, O, O << 1, None)


def test_rows():
    c, b = _kv()
    nan = float("nan")
    for match, rows in (("multiple of", (Q, 512, O, 512, 3, 3, 0.1)),
                        ("multiple of", (Q, 512, O, 512, 3, 0, 0.1)),
                        ("65535", (Q, 512, O, 512, 3, 65536, 0.1)),
                        ("finite", (Q, 512, O, 512, 3, 4, nan)),
                        ("null q", (None, 512, O, 512, 3, 4, 0.1)),
                        ("null out", (Q, 512, None, 512, 3, 4, 0.1)),
                        ("row stride of q", (Q, 508, O, 512, 3, 4, 0.1)),
                        ("16-byte", (Q, 512, O + 8, 512, 3, 4, 0.1)),
                        ("overlaps", (Q, 512, Q, 512, 3, 4, 0.1)),
                        ("T must", (Q, 512, O, 512, -1, 4, 0.1)),
                        ("T must", (Q, 512, O, 512, 2**30 + 1, 4, 0.1))):
        for fn, args in _calls(c, b, rows):
            _refused(match, fn, *args)
    for fn, args in _calls(None, b) + _calls(c, None):
        _refused("null cache or batch", fn, *args)
    lib = sdq.load_library()
    for fn, args in _calls(c, b, (None, 0, None, 0, 0, 2, 0.1)):
        assert getattr(lib, fn)(*args) == sdq.OK


def test_shared_parts():
    c, b = _kv()
    rows = (b, Q, 256, O, 256, 3, 2, 0.1, 1, None)
    for match, kw in (("n must", dict(n=-1)), ("n must", dict(n=65536)),
                      ("max_pages", dict(most=-1)), ("max_pages", dict(most=2**26 + 1)),
                      ("null arrays", dict(s_start=None)), ("null arrays", dict(lens=None)),
                      ("null arrays", dict(table=None))):
        _refused(match, "sdq_kv_attention_shared", c, _shared(**kw), *rows)
    _refused("null shared", "sdq_kv_attention_shared", c, None, *rows)


def test_weights():
    c, b = _kv()
    rows = (Q, 256, O, 256, 3, 2, 0.1, 1, None)
    _refused("null weights", "sdq_kv_attention_weights", c, b, None, *rows)
    for w in (Q, Q + 512, O - 64, P):
        _refused("overlaps", "sdq_kv_attention_weights", c, b, w, *rows)
    c, b = _kv(k=P, ks=P << 1, v=P << 2, vs=P << 3)
    for w in (P, P << 1, P << 2, P << 3, (P << 2) + 4096):
        _refused("overlaps", "sdq_kv_attention_weights", c, b, w, *rows)


def test_evict():
    c, b = _kv(k=P, ks=P << 1, v=P << 2, vs=P << 3, lens=P << 4, table=P << 5)
    TO, L, K = P << 15, P << 16, P << 17

    def call(w=W, first=0, last=0, keep=16, to=TO, most=1, lens=L, kept=K):
        return c, b, w, first, last, keep, to, most, lens, kept, None

    for match, kw in (("keep must", dict(keep=0)), ("keep must", dict(keep=2**30 + 1)),
                      ("keep must", dict(first=-1)), ("keep must", dict(last=-1)),
                      ("keep must", dict(first=9, last=8)), ("keep must", dict(first=17)),
                      ("keep must", dict(last=2**62, first=2)),
                      ("to_max_pages", dict(keep=17)), ("to_max_pages", dict(most=-1)),
                      ("to_max_pages", dict(most=2**26 + 1)), ("to_max_pages", dict(most=0)),
                      ("null", dict(w=None)), ("null", dict(to=None)), ("null", dict(lens=None)),
                      ("null", dict(kept=None)), ("overlaps", dict(lens=P << 4)),
                      ("overlaps", dict(lens=(P << 5) + 28)), ("overlaps", dict(kept=TO - 4)),
                      ("overlaps", dict(lens=K + 16)), ("overlaps", dict(kept=W - 4)),
                      ("overlaps", dict(w=P << 1)), ("overlaps", dict(w=(P << 3) + 64)),
                      ("overlaps", dict(w=P)), ("overlaps", dict(lens=P << 3)),
                      ("overlaps", dict(kept=P << 2))):
        _refused(match, "sdq_kv_evict", *call(**kw))
    _refused("null cache or batch", "sdq_kv_evict", None, *call()[1:])
    _refused("null cache or batch", "sdq_kv_evict", c, None, *call()[2:])
    big, many = _kv(nseq=65535, heads=2)[0], _kv(nseq=65535)[1]
    _refused("2^33", "sdq_kv_evict", big, many, W, 0, 0, 2**17, TO, 2**13, L, K, None)
    none = _kv(nseq=0)[1]
    assert sdq.load_library().sdq_kv_evict(c, none, None, 0, 0, 16, None, 1, None, None, None) == sdq.OK


def test_binding():
    f = torch.zeros
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    cache, batch = sdq.KvCache.empty(2, 16, 1, "cpu"), sdq.KvBatch(i32(2), i32(1), i32(1, 3))
    shared = sdq.KvShared(i32(2), i32(1), i32(1, 2))
    x, w = f(4, 128), f(2, 1, 16)
    for fn, head in ((sdq.kv_cross_attention, (cache, batch)),
                     (sdq.kv_attention_shared, (cache, shared, batch)),
                     (sdq.kv_attention_weights, (cache, batch, w))):
        _raises("on the GPU", fn, *head, x, x, 1)
        _raises("q: shape", fn, *head, x, x, 2)
        _raises("out: shape", fn, *head, x, f(3, 128), 1)
        _raises("KvCache", fn, None, *head[1:], x, x, 1)
    _raises("KvShared", sdq.kv_attention_shared, cache, None, batch, x, x, 1)
    _raises("KvBatch", sdq.kv_attention_shared, cache, shared, None, x, x, 1)
    _raises("s_start: shape", sdq.KvShared, i32(3), i32(1), i32(1, 2))
    _raises("lens: dtype", sdq.KvShared, i32(2), f(1), i32(1, 2))
    with pytest.raises(AttributeError):
        shared.table = i32(1, 2)
    _raises("weights: shape", sdq.kv_attention_weights, cache, batch, f(2, 1, 15), x, x, 1)
    _raises("weights: dtype", sdq.kv_attention_weights, cache, batch, w.double(), x, x, 1)
    to, lens, kept = i32(1, 2), i32(1), i32(1, 1, 20)
    _raises("on the GPU", sdq.kv_evict, cache, batch, w, to, lens, kept)
    _raises("to_table: shape", sdq.kv_evict, cache, batch, w, i32(2, 2), lens, kept)
    _raises("to_lens: dtype", sdq.kv_evict, cache, batch, w, to, f(1), kept)
    _raises("kept: shape", sdq.kv_evict, cache, batch, w, to, lens, i32(1, 2, 20))
    _raises("KvBatch", sdq.kv_evict, cache, None, w, to, lens, kept)
    _raises("weights: must be contiguous", sdq.kv_evict, cache, batch, f(2, 1, 32)[:, :, ::2], to, lens,
            kept)


def test_struct_matches_the_header(tmp_path):
    src = tmp_path / "layout.cpp"
    names = [n for n, _ in sdq.KvSharedView._fields_]
    src.write_text("\n".join(
        ['#include <cstddef>', '#include <cstdio>', '#include "sdq.h"', "int main() {",
         'printf("%zu\\n", sizeof(sdq_kv_shared));']
        + [f'printf("%zu\\n", offsetof(sdq_kv_shared, {n}));' for n in names] + ["}"]))
    exe = tmp_path / "layout"
    subprocess.run([shutil.which("g++"), "-I", os.path.join(ROOT, "include"), str(src), "-o",
                    str(exe)], check=True)
    got = [int(n) for n in subprocess.run([str(exe)], capture_output=True, text=True,
                                          check=True).stdout.split()]
    assert got == [ctypes.sizeof(sdq.KvSharedView)] + [getattr(sdq.KvSharedView, n).offset
                                                       for n in names]


def test_every_shared_plan_fits(tmp_path):
    exe = str(tmp_path / "shared_plan")
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Wextra", "-I" + os.path.join(PKG, "csrc"),
                    os.path.join(ROOT, "tests", "cpp", "shared_plan.cpp"), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr


@pytest.mark.slow
@pytest.mark.parametrize("src", ["sdq_kv_packed.hip", "sdq_kv_weights.hip", "sdq_kv_evict.hip"])
def test_no_hazard(tmp_path, src):
    if not os.path.exists(HIPCC):
        pytest.skip("hipcc not available")
    out = tmp_path / (src + ".s")
    r = subprocess.run(
        [HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17", "-ffp-contract=off",
         "-fno-gpu-flush-denormals-to-zero", "-fhip-fp32-correctly-rounded-divide-sqrt",
         "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
         "-I" + os.path.join(ROOT, "include"), "--cuda-device-only", "-S", os.path.join(CSRC, src),
         "-o", str(out)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    text = out.read_text()
    bad = _scan(text) + _scan_sgpr(text) + scan(text) + scan_c(text)
    assert not bad, f"{len(bad)} hazards:\n" + "\n".join(map(str, bad[:10]))
    assert not [op for op in ("v_pk_add_f32", "v_pk_mul_f32", "v_pk_fma_f32") if op in text]
