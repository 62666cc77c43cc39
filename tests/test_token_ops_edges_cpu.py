"""Host-side parts of the token-model operators that need no GPU."""
import os
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "..", "idash26-track3_b200", "csrc")
INCLUDE = os.path.join(HERE, "..", "include")


def host_build(tmp_path, name, *flags):
    """tests/<name>.cpp compiled with the host C++ compiler against csrc/"""
    cxx = shutil.which("g++") or shutil.which("c++")
    cuda = next((d for d in (os.environ.get("CUDA_HOME", ""), "/usr/local/cuda")
                 if d and os.path.exists(os.path.join(d, "include", "cuda_runtime.h"))), None)
    if cxx is None or cuda is None:
        pytest.skip("needs a host C++ compiler and the CUDA headers")
    exe = str(tmp_path / name)
    r = subprocess.run([cxx, "-std=c++17", "-O1", "-g", *flags, "-I", CSRC, "-I", INCLUDE, "-I",
                        os.path.join(cuda, "include"), os.path.join(HERE, name + ".cpp"), "-o", exe, "-pthread"],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    return exe


def test_first_tensor_maps_of_two_threads_do_not_race(tmp_path):
    """Two parties of one process make their first tensor map at the same time, under the thread sanitizer."""
    cxx = shutil.which("g++") or shutil.which("c++")
    empty = tmp_path / "empty.cpp"
    empty.write_text("int main() { return 0; }")
    if cxx is None or subprocess.run([cxx, "-fsanitize=thread", str(empty), "-o", str(tmp_path / "empty")],
                                     capture_output=True).returncode or \
            subprocess.run([str(tmp_path / "empty")], capture_output=True).returncode:
        pytest.skip("no working thread sanitizer")
    exe = host_build(tmp_path, "tma_map_check", "-fsanitize=thread")
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr


@pytest.fixture(scope="module")
def q4_plan(tmp_path_factory):
    """(bw, M, K, N) tuples -> (tile, CTAs along K), the choice of csrc/q4_plan.cuh"""
    exe = host_build(tmp_path_factory.mktemp("plan"), "q4_plan_check")

    def plan(sizes):
        r = subprocess.run([exe], input="".join(f"{bw // 8} {M} {K} {N}\n" for bw, M, K, N in sizes),
                           capture_output=True, text=True, timeout=60)
        return [tuple(int(v) for v in line.split()) for line in r.stdout.splitlines()]

    return plan


def test_gpu_tests_take_every_4_bit_kernel(q4_plan):
    """The sizes of tests/test_token_ops_edges_gpu.py reach each kernel and split of K that the choice can make."""
    from tests.test_token_ops_edges_gpu import FC_LONGEST, FC_TILES

    every = {(-2, 1), (5, 1)} | {(t, s) for t in range(5) for s in (1, 2, 4, 8)}
    for bw, cases in FC_TILES.items():
        assert set(cases) == every
        assert q4_plan([(bw, *mkn) for mkn in cases.values()]) == list(cases)
        longest = q4_plan([(bw, *mkn) for mkn in FC_LONGEST])
        assert all(t >= 0 and K == s * 32768 for (t, s), (_, K, _) in zip(longest, FC_LONGEST))
        assert {t for t, _ in longest} >= {0, 5}


def test_4_bit_choice_over_its_range(q4_plan):
    """Every size that the calls accept finds a kernel, whose grid and sums are within their limits."""
    sizes = [(bw, M, K, N) for bw in (32, 64) for M in (1, 2, 3, 17, 64, 1000, 65535 * 2048 // bw)
             for K in (1, 31, 500, 32768, 32769, 131073, 262144) for N in (1, 128, 5000, 2**31 - 1)]
    rows = (4, 8, 16, 32, 64, 64)
    for (bw, M, K, _), (tile, split) in zip(sizes, q4_plan(sizes)):
        assert tile == -2 and M <= 2 or tile >= 0 and -(-M // (rows[tile] * 32 // bw)) <= 65535
        assert tile == -2 or split in (1, 2, 4, 8) and -(-K // split) <= 32768
    assert q4_plan([(32, 4, 0, 5)]) == [(-3, 1)]
    assert q4_plan([(32, 4, (1 << 18) + 1, 5)])[0][0] == -1
