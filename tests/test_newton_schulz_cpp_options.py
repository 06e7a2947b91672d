"""Builds and runs the C++ test of newton_schulz's options.  On CPU only the build is checked."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CUDA = os.environ.get("CUDA_HOME", "/usr/local/cuda")
SRC = os.path.join(ROOT, "tests", "cpp", "newton_schulz_options_tests.cc")
EXE = os.path.join(ROOT, "tests", "cpp", "newton_schulz_options_tests.bin")


def build_exe():
    headers = [os.path.join(ROOT, "include", f) for f in ("batchlas_b200.hh", "blb200.h")]
    libdir = os.path.join(ROOT, "batchlas_b200")
    if not os.path.exists(EXE) or os.path.getmtime(EXE) < max(os.path.getmtime(f) for f in [SRC, *headers]):
        gxx = shutil.which("g++") or "/opt/gcc/bin/g++"
        subprocess.check_call([gxx, "-std=c++20", "-O1", "-I", os.path.join(ROOT, "include"), "-I",
                               os.path.join(CUDA, "include"), SRC, "-o", EXE, "-L", libdir, "-lbatchlas_b200",
                               "-L", os.path.join(CUDA, "lib64"), "-lcudart", f"-Wl,-rpath,{libdir}",
                               f"-Wl,-rpath,{os.path.join(CUDA, 'lib64')}"])
    return EXE


def test_newton_schulz_options_compile(lib):
    out = subprocess.run([build_exe(), "--compile-only-check"], capture_output=True, text=True, timeout=60)
    assert out.returncode == 0 and "overload set resolves" in out.stdout


@pytest.mark.gpu
def test_newton_schulz_options_on_gpu(lib):
    out = subprocess.run([build_exe()], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and " 0 failed" in out.stdout, out.stdout[-4000:] + out.stderr[-2000:]
