"""The range-checking build (liblf_sm100_dbg.so) on the rotating append, the gather and the decode of a 4-bit cache: the
same tests pass, with a status word of zero where they ask for one. The library is chosen when it is loaded, so
they run in a child process with LF_DEBUG_BOUNDS=1."""
import os
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent


@pytest.mark.gpu
def test_rotary_and_4bit_entry_points_stay_in_range():
    from loopfuse_b200.build import DBG_LIB_PATH, build_native
    if not DBG_LIB_PATH.exists():
        build_native(debug_bounds=True)
    env = dict(os.environ, LF_DEBUG_BOUNDS="1")
    code = ("import sys, pytest; sys.path.insert(0, '.'); from loopfuse_b200 import _native; "
            "assert _native.load().lf_debug_bounds() == 1; "
            "sys.exit(pytest.main(['-q', '-x', '-m', 'gpu', '-p', 'no:cacheprovider', '-k', "
            "'append or gather or rotation_bits or test_decode or few_short or window or sense or serving', "
            "'tests/test_gpu_rotary.py', 'tests/test_gpu_decode4.py']))")
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and " passed" in r.stdout, r.stdout[-3000:] + r.stderr[-2000:]


@pytest.mark.gpu
def test_long_runs_and_normed_appends_stay_in_range():
    from loopfuse_b200.build import DBG_LIB_PATH, build_native
    if not DBG_LIB_PATH.exists():
        build_native(debug_bounds=True)
    env = dict(os.environ, LF_DEBUG_BOUNDS="1")
    code = ("import sys, pytest; sys.path.insert(0, '.'); from loopfuse_b200 import _native; "
            "assert _native.load().lf_debug_bounds() == 1; "
            "sys.exit(pytest.main(['-q', '-x', '-m', 'gpu', '-p', 'no:cacheprovider', "
            "'tests/test_gpu_decode4_runs.py', 'tests/test_gpu_rotary_norm.py']))")
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and " passed" in r.stdout, r.stdout[-3000:] + r.stderr[-2000:]
