"""The int8 scale of the rotating append is the IEEE quotient absmax / 127 whichever kernel writes it: the fma-corrected quotient
(hn_common.cuh: quot_const) equals it for every positive finite fp32 absmax. CPU only, some seconds."""
import os
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))


def test_int8_scale_of_any_fp32_peak(tmp_path):
    exe = os.path.join(tmp_path, "check")
    subprocess.check_call(["gcc", "-O2", "-march=native", "-ffp-contract=off", "-fopenmp", "-o", exe,
                           os.path.join(HERE, "scale_quotient_check.c"), "-lm"])
    r = subprocess.run([exe], capture_output=True, text=True, timeout=900)
    assert r.returncode == 0 and "2139095039 values, mismatches 0" in r.stdout, r.stdout + r.stderr
