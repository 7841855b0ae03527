"""How an attention call with sinks and shared prefixes is cut into parts and workgroups
(secure_infer_amd/csrc/si_attend_plan.h), checked as compiled host code over seeded calls up to the longest
tables and the most rows a call may have (tests/csrc/attend_more_plan_check.hip)."""
import subprocess

from tests.test_codec_math import CSRC, ROOT, _hipcc


def test_parts_fit_their_places(tmp_path):
    exe = tmp_path / "attend_more_plan_check"
    subprocess.run([_hipcc(), "--cuda-host-only", "-x", "hip", "-O2", "-std=c++17", "-I", str(ROOT / "include"),
                    "-I", str(CSRC), str(ROOT / "tests" / "csrc" / "attend_more_plan_check.hip"), "-o", str(exe)],
                   check=True, capture_output=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stdout + out.stderr
    fields = out.stdout.split()
    stats = dict(zip(fields[0::2], map(int, fields[1::2])))
    assert stats["bad"] == 0 and stats["cases"] > 500_000
