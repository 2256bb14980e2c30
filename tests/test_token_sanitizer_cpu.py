"""The image decoder's steps for models of tokens under AddressSanitizer, signed overflow trapped
(tests/token_sanitizer_driver.py in a child process with the ASan runtime preloaded)."""
import os
import subprocess
import sys
from pathlib import Path

import pytest

HERE = Path(__file__).resolve().parent


def test_images_of_token_models_are_decoded_cleanly(tmp_path, monkeypatch):
    from tests import asan_build
    try:
        runtime = asan_build.asan_runtime()
    except FileNotFoundError as e:
        pytest.skip(str(e))
    monkeypatch.setattr(asan_build, "OUT", tmp_path)
    monkeypatch.setattr(asan_build, "LIB", tmp_path / "libsynaptik_hip_sanitized.so")
    monkeypatch.setattr(asan_build, "ASAN", asan_build.ASAN + [
        "-Xarch_host", "-fsanitize=signed-integer-overflow",
        "-Xarch_host", "-fsanitize-trap=signed-integer-overflow"])
    lib = asan_build.build()
    env = dict(os.environ, LD_PRELOAD=runtime,
               ASAN_OPTIONS="detect_leaks=0:halt_on_error=1:abort_on_error=0:exitcode=99",
               PYTHONPATH=str(HERE.parent))
    res = subprocess.run([sys.executable, str(HERE / "token_sanitizer_driver.py"), str(lib)], env=env,
                         capture_output=True, text=True, timeout=600)
    assert "AddressSanitizer" not in res.stderr, res.stderr[-4000:]
    assert res.returncode == 0, (res.returncode, res.stderr[-4000:])
    assert "images of token models ok" in res.stdout
