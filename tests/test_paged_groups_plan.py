"""How attention calls with groups of many sequences are cut (secure_infer_amd/csrc/si_attend_plan.h), checked
as compiled host code against the same calls without groups (tests/csrc/attend_groups_plan_check.hip)."""
import subprocess

from tests.test_codec_math import CSRC, ROOT, _hipcc


def test_long_sequences_keep_their_parts(tmp_path):
    exe = tmp_path / "attend_groups_plan_check"
    subprocess.run([_hipcc(), "--cuda-host-only", "-x", "hip", "-O2", "-std=c++17", "-I", str(ROOT / "include"),
                    "-I", str(CSRC), str(ROOT / "tests" / "csrc" / "attend_groups_plan_check.hip"), "-o", str(exe)],
                   check=True, capture_output=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stdout + out.stderr
    fields = out.stdout.split()
    stats = dict(zip(fields[0::2], map(int, fields[1::2])))
    assert stats["bad"] == 0 and stats["cases"] > 50_000
