"""Dynamic LDS beyond 64 KiB has to be granted to every kernel that is launched with it.  The host code of the score attention entries runs
here against a stand-in for the runtime (tests/native/recording_hip.cpp) that writes down grants and launches."""
import os
import shutil
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CHILD = r"""
import ctypes as C, sys
fake = C.CDLL(sys.argv[1], mode=C.RTLD_GLOBAL)          # in front of the runtime for every library loaded from here on
from transfusion_amd import _lib as L
lib = C.CDLL(L.LIB_PATH)
for f in ("tf_score_attn_work", "tf_score_attn_bwd_work"):
    getattr(lib, f).restype = C.c_size_t
PTR = 1 << 20                                           # nothing reads it: no kernel runs

def call(entry, D, f32, Sq, doc):
    n = 16 * D
    a = L.TfScoreAttnArgs(q=PTR, k=PTR, v=PTR, out=PTR, lse=PTR, dout=PTR, dq=PTR, dk=PTR, dv=PTR, delta=PTR, B=1, Sq=Sq, Sk=Sq, H=2, Hk=2, D=D, is_f32=f32,
                          scale=0.1, q_ss=n, k_ss=n, v_ss=n, do_ss=n, q_sh=D, k_sh=D, v_sh=D, do_sh=D, work=PTR, work_bytes=1 << 40,
                          q_doc=PTR if doc else 0, k_doc=PTR if doc else 0)
    return getattr(lib, entry)(C.byref(a), None)

fake.refuse_grants(1)
assert call("tf_score_attn_fwd", 128, 0, 200, False) != 0       # a refused grant is an error, and asked for again by the next call
for D in (32, 64, 96, 128, 192, 256):
    for f32 in (0, 1):
        for doc in (False, True):
            for again in range(2):
                assert call("tf_score_attn_fwd", D, f32, 3, doc) == 0       # few rows
                assert call("tf_score_attn_fwd", D, f32, 200, doc) == 0
                assert call("tf_score_attn_bwd", D, f32, 200, doc) == 0
"""


def test_every_kernel_is_granted_the_lds_it_is_launched_with(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("needs g++")
    from transfusion_amd import _lib, build
    if not os.path.exists(_lib.LIB_PATH):
        build.build_lib(verbose=False)
    fake = str(tmp_path / "recording_hip.so")
    subprocess.run([gxx, "-shared", "-fPIC", "-O1", os.path.join(ROOT, "tests", "native", "recording_hip.cpp"), "-o", fake], check=True)
    r = subprocess.run([sys.executable, "-c", CHILD, fake], capture_output=True, text=True, cwd=ROOT, timeout=120)
    assert r.returncode == 0, r.stderr
    granted, launched, asked = {}, {}, 0
    for line in r.stdout.splitlines():
        what, kernel, n = line.split()
        if what == "attr":
            asked += 1
            granted[kernel] = max(int(n), granted.get(kernel, 0))
        else:
            launched[kernel] = max(int(n), launched.get(kernel, 0))
            if int(n) > 65536:
                assert granted.get(kernel, 0) >= int(n), f"{kernel}: launched with {n} bytes, granted {granted.get(kernel, 0)}"
    large = [k for k, n in launched.items() if n > 65536]
    assert len(large) >= 40, len(large)
    assert asked == len(granted)                         # once a kernel, not once a launch
