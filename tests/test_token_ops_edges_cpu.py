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
