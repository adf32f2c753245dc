"""The batch attention entry points' refusals again, with the library's host code under
AddressSanitizer and UndefinedBehaviorSanitizer (libsimp_hip_san.so), on the CPU."""
import glob
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_serve_refusals_under_sanitizers():
    san = os.path.join(ROOT, "simplang_amd", "libsimp_hip_san.so")
    if not os.path.exists(san):
        pytest.skip("libsimp_hip_san.so not built (make -C simplang_amd/runtime sanitize)")
    rt = sorted(glob.glob("/opt/rocm/lib/llvm/lib/clang/*/lib/linux/libclang_rt.asan-x86_64.so"))
    if not rt:
        pytest.skip("the compiler's ASan runtime is not installed")
    env = dict(os.environ, SIMP_HIP_LIB=san, LD_PRELOAD=rt[-1],
               ASAN_OPTIONS="halt_on_error=1:abort_on_error=0:detect_leaks=0",
               UBSAN_OPTIONS="halt_on_error=1:print_stacktrace=1")
    r = subprocess.run([sys.executable, "-m", "pytest", "-q", "-x", "-m", "not gpu", "-p", "no:cacheprovider",
                        os.path.join(ROOT, "tests", "test_serve_args.py")],
                       env=env, cwd=ROOT, capture_output=True, text=True, timeout=600)
    out = r.stdout + r.stderr
    assert r.returncode == 0, out[-4000:]
    assert " passed" in r.stdout and "AddressSanitizer" not in out and "runtime error" not in out


def test_serve_limits_under_sanitizers():
    """The refusals at the edge of the sizes, strides and shared memory, the same way."""
    san = os.path.join(ROOT, "simplang_amd", "libsimp_hip_san.so")
    rt = sorted(glob.glob("/opt/rocm/lib/llvm/lib/clang/*/lib/linux/libclang_rt.asan-x86_64.so"))
    if not os.path.exists(san) or not rt:
        pytest.skip("libsimp_hip_san.so or the compiler's ASan runtime is not there")
    env = dict(os.environ, SIMP_HIP_LIB=san, LD_PRELOAD=rt[-1],
               ASAN_OPTIONS="halt_on_error=1:abort_on_error=0:detect_leaks=0",
               UBSAN_OPTIONS="halt_on_error=1:print_stacktrace=1")
    r = subprocess.run([sys.executable, "-m", "pytest", "-q", "-x", "-m", "not gpu", "-p", "no:cacheprovider",
                        os.path.join(ROOT, "tests", "test_serve_limits.py")],
                       env=env, cwd=ROOT, capture_output=True, text=True, timeout=600)
    out = r.stdout + r.stderr
    assert r.returncode == 0, out[-4000:]
    assert " passed" in r.stdout and "AddressSanitizer" not in out and "runtime error" not in out
