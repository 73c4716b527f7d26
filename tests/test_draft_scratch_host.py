"""What hxm_tree_attention launches and keeps against the pieces that any batch makes, under
AddressSanitizer and UndefinedBehaviorSanitizer (tests/sanitize/draft_scratch_check.cpp)."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_draft_scratch_under_asan_and_ubsan(tmp_path):
    exe = tmp_path / "draft_scratch_check"
    src = os.path.join(ROOT, "tests", "sanitize", "draft_scratch_check.cpp")
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-fno-omit-frame-pointer",
                    "-fsanitize=address,undefined", "-fno-sanitize-recover=all",
                    "-Wall", "-Werror", src, "-o", str(exe)], check=True, timeout=300)
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=1:abort_on_error=0",
               UBSAN_OPTIONS="print_stacktrace=1:halt_on_error=1")
    env.pop("LD_PRELOAD", None)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300, env=env)
    assert r.returncode == 0 and "draft scratch ok" in r.stdout, r.stdout + r.stderr
