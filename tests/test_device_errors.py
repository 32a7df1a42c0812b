"""What a check makes of the device's error words, with a fake in their place (no GPU)."""
import os
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))


def test_all_words_are_reported_at_once_and_cleared(tmp_path):
    exe = str(tmp_path / "device_errors_test")
    r = subprocess.run(["g++", "-std=c++17", "-Wall", "-Wextra", "-Werror", "-o", exe, os.path.join(HERE, "device_errors_test.cpp")],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and "device errors ok" in r.stdout, r.stdout + r.stderr
