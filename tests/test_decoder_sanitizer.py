"""CPU sanitizer build of the decoder's GPU-free host code (qvl_decoder_meta.cpp), run by
tests/host_sanitizer/decoder_driver.cpp on random and malformed sequences with exactly-sized buffers."""
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]


def test_decoder_host_code_under_asan_ubsan(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    exe, csrc = tmp_path / "qvl_decoder_asan", ROOT / "qwen3-vl-jax_amd" / "csrc"
    cmd = [gxx, "-std=c++17", "-O1", "-g", "-fno-omit-frame-pointer", "-fsanitize=address,undefined",
           "-fno-sanitize-recover=undefined", "-I", str(ROOT / "include"), "-I", str(csrc),
           str(ROOT / "tests" / "host_sanitizer" / "decoder_driver.cpp"), str(csrc / "qvl_decoder_meta.cpp"),
           str(csrc / "qvl_meta.cpp"), "-o", str(exe)]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0 and "asan" in r.stderr.lower() and "cannot find" in r.stderr.lower():
        pytest.skip("the sanitizer runtime is not installed")
    assert r.returncode == 0, r.stderr[-4000:]
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300,
                         env={"ASAN_OPTIONS": "detect_leaks=1:abort_on_error=0", "PATH": "/usr/bin:/bin"})
    assert run.returncode == 0, (run.stdout[-2000:], run.stderr[-4000:])
    assert "0 failures" in run.stdout
