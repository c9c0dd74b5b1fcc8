"""Memory that a stream capture takes from the pool is its graph's until that is gone: the pool's bookkeeping, with made-up memory and captures."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_blocks_of_a_capture_stay_its_graphs(tmp_path):
    program = str(tmp_path / "pool")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-o", program, os.path.join(ROOT, "tests", "captured_pool.cc"), os.path.join(ROOT, "sage_b200", "csrc", "runtime", "allocator.cc"),
                    "-pthread"], check=True)
    found = subprocess.run([program], capture_output=True, text=True, timeout=60)
    assert found.returncode == 0 and found.stdout == "fine\n", found.stdout + found.stderr
