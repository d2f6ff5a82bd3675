"""The 8-bit operators' host side where there is no GPU, no torch, or no device that answers (no GPU is needed)."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def python(code, **env):
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, env={**os.environ, **env}, capture_output=True, text=True,
                       timeout=600)
    assert r.returncode == 0, r.stdout + r.stderr[-3000:]
    return r.stdout


def test_a_device_that_cannot_be_asked_is_an_error():
    pytest.importorskip("torch")
    assert "reported" in python("""
import qwen_asr_b200 as Q
assert Q.lib().qwen_asr_ops_error(-1) < 0 and Q.lib().qwen_asr_ops_error(0) < 0
from qwen_asr_b200 import ops
try:
    ops.check('cuda:0')
except RuntimeError as e:
    assert 'timed out' not in str(e), e
    print('reported')
""", CUDA_VISIBLE_DEVICES="")


def test_the_build_does_without_torch():
    """What is left of the build where torch is missing is the library (its own compilation, which needs none, is
    left out here: this process has it loaded)."""
    assert "built" in python("""
import sys
sys.modules['torch'] = None  # an import of it fails
from oracle import ref_decode
from qwen_asr_b200 import build
called = []
build.build = lambda *a, **k: called.append('library')
ref_decode.build = lambda *a, **k: called.append('oracle')
import __graft_entry__
__graft_entry__.build()
assert called == ['library', 'oracle'] and build.build_binding() is None
print('built')
""")
