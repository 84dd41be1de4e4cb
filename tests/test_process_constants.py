"""The per-read constants that go through the C library are formed by the PROCESS's own log / exp / logf (csrc/np_constants.h), on a CPU:
the library's host entry points in a child process whose functions are one unit in the last place off for half of all arguments
(tests/libm_skew.c, LD_PRELOAD) still equal the oracle's C port, which calls the same functions -- a table of some C library's values
inside the product would not follow."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CHECK = r"""
import ctypes as C
import numpy as np
from nanopolish_amd import api, lib as _l
from oracle import Oracle
L = _l.load_library(); orc = Oracle()
rng = np.random.default_rng(29)
plain = C.CDLL(None); plain.log.restype = C.c_double; plain.log.argtypes = [C.c_double]
for e in np.concatenate([rng.uniform(0.0, 6.0, 6000), [0.0, 1.25, 5.0, 50.0, 400.0, 1e9]]):
    assert np.array_equal(api.calculate_transitions(float(e)), orc.calculate_transitions(float(e), 1.0), equal_nan=True), e
out = np.zeros(4); rd = _l.ReadDev()
for ne in list(range(1, 30000, 37)) + [0, 1 << 31]:
    for nk in (1, 97, 5445):
        want = orc.aligner_constants(ne, nk)
        L.np_aligner_constants(ne, nk, out.ctypes.data_as(_l.c_f64p))
        assert tuple(out) == want, (ne, nk)
        L.np_fill_read_host(C.byref(rd), 0.0, 1.0, 1.3, 0, ne, 0, nk)
        assert (rd.lp_skip, rd.lp_stay, rd.lp_step, rd.lp_trim) == want, (ne, nk)
x = np.exp(rng.uniform(-20, 20, 4000)); ol = np.zeros_like(x); oe = np.zeros_like(x)
L.np_restated_log_exp(x.ctypes.data_as(_l.c_f64p), len(x), ol.ctypes.data_as(_l.c_f64p), oe.ctypes.data_as(_l.c_f64p))
assert np.array_equal(ol, [plain.log(float(v)) for v in x])
print("constants follow the process")
"""


def _child(env_extra):
    return subprocess.run([sys.executable, "-c", CHECK], cwd=ROOT, env=dict(os.environ, PYTHONPATH=ROOT, **env_extra), capture_output=True, text=True, timeout=300)


def test_host_constants_follow_the_process(tmp_path):
    out = str(tmp_path / "libm_skew.so")
    cc = subprocess.run(["gcc", "-O1", "-shared", "-fPIC", "-fno-builtin", os.path.join(ROOT, "tests", "libm_skew.c"), "-o", out, "-ldl", "-lm"],
                        capture_output=True, text=True)
    if cc.returncode != 0:
        pytest.skip("no C compiler for the skewed library here: " + cc.stderr[-300:])
    normal, skewed = _child({}), _child({"LD_PRELOAD": out})
    for r in (normal, skewed):
        assert r.returncode == 0 and "constants follow the process" in r.stdout, r.stdout[-500:] + r.stderr[-2000:]


def test_device_formed_constants_are_refused():
    """NP_HOST_CONSTANTS=0 asked for constants formed on the device; there is no such form, and np_create says so before it looks for a device."""
    code = ("from nanopolish_amd import lib as _l\n"
            "L = _l.load_library()\n"
            "assert not L.np_create(0, None)\n"
            "print(L.np_last_error(None).decode())\n")
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, env=dict(os.environ, PYTHONPATH=ROOT, NP_HOST_CONSTANTS="0"), capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "NP_HOST_CONSTANTS=0" in r.stdout, r.stdout + r.stderr[-1000:]
