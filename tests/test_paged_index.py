"""The paged attention's index arithmetic on the host (tests/native/paged_index_cases.cpp)."""
import os
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))


def test_paged_index(tmp_path):
    exe = str(tmp_path / "paged_index_cases")
    subprocess.run(["g++", "-std=c++20", "-O2", "-Wall", "-Werror",
                    os.path.join(HERE, "native", "paged_index_cases.cpp"), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout.startswith("ok "), r.stdout
