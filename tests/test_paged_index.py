"""The paged attention's index arithmetic and the batched generation's steps on the host
(tests/native/paged_index_cases.cpp, batch_schedule_cases.cpp)."""
import os
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.mark.parametrize("name", ("paged_index_cases", "batch_schedule_cases"))
def test_native_cases(tmp_path, name):
    exe = str(tmp_path / name)
    subprocess.run(["g++", "-std=c++20", "-O2", "-Wall", "-Werror", os.path.join(HERE, "native", name + ".cpp"),
                    "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.startswith("ok"), r.stdout
