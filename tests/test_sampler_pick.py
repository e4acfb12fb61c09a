"""The device sampler's walk over probabilities, on the CPU: which token a coin
falls on where a mask or a bias bars tokens, the last of the vocabulary among
them. tests/sampler_pick_check.cu compiles kc_sampler.cuh for the host (nothing
is launched) and tries the coins where the sums' roundings tell."""
import os
import shutil
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def checker(tmp_path_factory):
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        pytest.skip("nvcc not found")
    exe = str(tmp_path_factory.mktemp("pick") / "sampler_pick_check")
    subprocess.run([nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-O1", "-std=c++17", "-Xcompiler", "-ffp-contract=off",
                    "--expt-relaxed-constexpr", "-I", os.path.join(ROOT, "isa-lm_b200", "csrc"),
                    "-I", os.path.join(ROOT, "include"), os.path.join(ROOT, "tests", "sampler_pick_check.cu"),
                    "-o", exe], check=True, capture_output=True)
    return exe


def probabilities(kind, n):
    rng = np.random.default_rng(n)
    z = rng.normal(0, {"flat": 0.5, "normal": 2.0, "peaked": 0.5}[kind], n)
    p = np.exp(z)
    if kind == "peaked":
        p[n // 3] = 0
        p *= 2e-4 / p.sum()
        p[n // 3] = 1 - 2e-4
    p[-1] = 0.0                                       # barred: the last token, a run of them, and one in ten
    p[n // 2:n // 2 + n // 10] = 0.0
    p[rng.random(n) < 0.1] = 0.0
    return (p / p.sum()).astype(np.float32)


@pytest.mark.parametrize("kind", ["flat", "normal", "peaked"])
@pytest.mark.parametrize("n", [1000, 1025, 32000, 128256])
def test_no_barred_token_is_drawn(checker, kind, n):
    p = probabilities(kind, n)
    r = subprocess.run([checker], input=f"{n} 1\n" + " ".join(map(repr, p.tolist())), capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr
    tried, zero, far = map(int, r.stdout.split())
    assert tried > 20000 and zero == 0 and far == 0


def test_checker_sees_the_last_token(checker):
    """A control: by the reference's rule, which holds where nothing is barred, coins that end without a hit take the
    last token whatever its probability."""
    p = probabilities("peaked", 32000)
    r = subprocess.run([checker], input="32000 0\n" + " ".join(map(repr, p.tolist())), capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and int(r.stdout.split()[1]) > 100
