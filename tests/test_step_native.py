"""The training-step operators' native side without a GPU: the header serves a
plain C11 caller, and the host code runs clean under AddressSanitizer and
UndefinedBehaviorSanitizer on the refusals and workspaces of the C ABI."""
import os
import shutil
import subprocess
import sys
from pathlib import Path

import pytest

from suika_amd import _lib

ROOT = Path(__file__).resolve().parents[1]


def test_c_caller(tmp_path):
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("no C compiler on this host")
    exe = tmp_path / "abi_step_calls"
    cmd = [gcc, "-std=c11", "-Wall", "-Wextra", "-Werror", "-D__HIP_PLATFORM_AMD__", f"-I{ROOT / 'include'}",
           "-I/opt/rocm/include", str(ROOT / "tests" / "c" / "abi_step_calls.c"), f"-L{_lib.LIB_PATH.parent}",
           "-lsuika_reshard", f"-Wl,-rpath,{_lib.LIB_PATH.parent}", "-o", str(exe)]
    res = subprocess.run(cmd, capture_output=True, text=True)
    assert res.returncode == 0, res.stderr[-3000:]
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert out.returncode == 0, out.stdout + out.stderr
    assert out.stdout.splitlines() == [
        "sum 0 1",
        f"dtype {_lib.SR_EDTYPE}",
        "embedding 0 1",
        "logprob 0",
        f"top {_lib.SR_EINVAL}",
        f"step {_lib.SR_EINVAL} 1",
    ], out.stdout


@pytest.mark.slow
def test_host_code_is_clean_under_asan_and_ubsan():
    from suika_amd import build
    libs = [build.SANITIZE_DIR / "libsuika_reshard.so", build.SANITIZE_DIR / "_suika_host.so"]
    sources = [*build.SOURCES, *build.HOST_SOURCES, *(ROOT / "include").glob("*.h"),
               *(ROOT / "suika_amd" / "csrc").glob("*.h")]
    if not all(p.exists() for p in libs) or \
            min(p.stat().st_mtime for p in libs) < max(p.stat().st_mtime for p in sources):
        build.build_sanitized()
    env = dict(os.environ, LD_PRELOAD=str(build.sanitizer_runtime()),
               ASAN_OPTIONS="detect_leaks=0:abort_on_error=1", UBSAN_OPTIONS="print_stacktrace=1:halt_on_error=1",
               SUIKA_RESHARD_LIB=str(libs[0]), SUIKA_HOST_LIB=str(libs[1]))
    res = subprocess.run([sys.executable, "-m", "pytest", "tests/test_step_optim.py", "tests/test_step_vocab.py", "-q",
                          "-m", "not gpu", "-p", "no:cacheprovider"],
                         cwd=ROOT, env=env, capture_output=True, text=True, timeout=900)
    out = res.stdout + res.stderr
    reports = [l for l in out.splitlines() if "runtime error:" in l or "AddressSanitizer" in l]
    assert res.returncode == 0 and not reports, "\n".join(reports[:20]) + "\n" + out[-4000:]
    assert " passed" in out.splitlines()[-1], out[-2000:]
