"""CPU: the limit of shared memory that the experts' down product asks of the runtime does not depend on which of two
host threads, with different numbers of tokens, came first (tests/consumer/moe_threads.cpp, on a runtime that runs
nothing)."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def binary(tmp_path_factory):
    out = tmp_path_factory.mktemp("moe_threads") / "moe_threads"
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    r = subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror", f"-I{ROOT}/include", f"-I{cuda}/include",
                        os.path.join(ROOT, "tests", "consumer", "moe_threads.cpp"), "-o", str(out), f"-L{ROOT}/lib", "-lpopcorn",
                        "-lpthread", "-ldl", "-Wl,--unresolved-symbols=ignore-all"], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
    return out


@pytest.mark.parametrize("hidden, many, few", [
    (2560, 10, 5), (2560, 40, 20),  # 18 channels a tile: one kernel with four stages, one with three
    (2048, 16, 5), (2048, 64, 20),  # 14 channels: six and four stages
    (4096, 8, 5), (4096, 40, 16),   # 28 channels: three and two stages
])
def test_threads_with_different_numbers_of_tokens(binary, hidden, many, few):
    # (The limit of the down product is the one above 150 KB; the up product's is 144 KB.)
    r = subprocess.run([str(binary), str(hidden), str(many), str(few), str(150 * 1024), "2"], capture_output=True, text=True,
                       timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr
