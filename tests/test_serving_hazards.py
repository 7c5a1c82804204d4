"""The scans of tests/test_store_hazards.py over the serving operators' kernels."""
import os
import subprocess

import pytest

from test_store_hazards import CSRC, HIPCC, ROOT, _scan, _scan_sgpr


@pytest.mark.slow
@pytest.mark.parametrize("src", ["sdq_kv.hip", "sdq_kv_attn.hip", "sdq_rmsq.hip", "sdq_w4.hip"])
def test_no_store_or_sgpr_hazard(tmp_path, src):
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
    bad = _scan(text) + _scan_sgpr(text)
    assert not bad, f"{len(bad)} hazards:\n" + "\n".join(bad[:10])
    # packed fp32 operations stay out
    assert not [op for op in ("v_pk_add_f32", "v_pk_mul_f32", "v_pk_fma_f32") if op in text]
