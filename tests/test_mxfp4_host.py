"""Products of 4-bit floats on the host side: launch arithmetic. No device is needed."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_every_tile_is_made_once_whatever_the_number_of_cus(tmp_path):
    exe = str(tmp_path / "tile_quarters_test")
    subprocess.check_call(["g++", "-std=c++17", "-I" + os.path.join(ROOT, "ruy_amd", "csrc"),
                           os.path.join(ROOT, "tests", "cpp", "tile_quarters_test.cc"), "-o", exe])
    assert "all passed" in subprocess.check_output([exe]).decode()
