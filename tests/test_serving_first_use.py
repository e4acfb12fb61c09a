"""The serving entries' first calls from several threads, under ThreadSanitizer on
the CPU: what they look up once per device is published in order. tests/
serving_first_use.cpp stands in for the CUDA runtime; nothing is launched."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC, INC = os.path.join(ROOT, "isa-lm_b200", "csrc"), os.path.join(ROOT, "include")


def test_first_calls_do_not_race(tmp_path):
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc) or not shutil.which("setarch"):
        pytest.skip("nvcc or setarch not found")
    plain = tmp_path / "plain.cpp"
    plain.write_text("int main() { return 0; }\n")
    if subprocess.run(["g++", "-fsanitize=thread", str(plain), "-o", str(tmp_path / "plain")], capture_output=True).returncode or \
            subprocess.run(["setarch", "-R", str(tmp_path / "plain")], capture_output=True).returncode:
        pytest.skip("no ThreadSanitizer")
    obj, exe = str(tmp_path / "serve.o"), str(tmp_path / "first_use")
    # (the device code is not run: made without optimization, as PTX)
    subprocess.run([nvcc, "-gencode", "arch=compute_100a,code=compute_100a", "-Xcicc", "-O0", "-std=c++17", "-Xcompiler",
                    "-fPIC,-fsanitize=thread,-ffp-contract=off,-g", "--expt-relaxed-constexpr", "-I", INC, "-I", CSRC, "-c",
                    os.path.join(CSRC, "kc_serve.cu"), "-o", obj], check=True, capture_output=True)
    cuda = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(nvcc))), "include")
    subprocess.run(["g++", "-fsanitize=thread", "-g", "-std=c++17", "-I", cuda, "-I", INC,
                    os.path.join(ROOT, "tests", "serving_first_use.cpp"), obj, "-o", exe, "-lpthread"], check=True, capture_output=True)
    r = subprocess.run(["setarch", "-R", exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout == "ok\n" and "data race" not in r.stderr, r.stdout + r.stderr[:4000]
