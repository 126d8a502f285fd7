"""Where the product in eight bits reads its weights' scales, without a GPU."""
import os
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))


def test_scales_are_read_inside_their_buffer(tmp_path):
    from telmo_amd import build

    exe = str(tmp_path / "scales")
    subprocess.run([build.HIPCC, "-x", "hip", "--cuda-host-only", "-std=c++17", "-O2", os.path.join(HERE, "e4m3_scales.cpp"), "-o", exe],
                   check=True, capture_output=True)
    assert subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split() == ["0", "0", "1"]
