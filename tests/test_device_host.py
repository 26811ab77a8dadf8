"""CPU suite: a call on a context of another device than the caller's leaves the caller's device current.  The library's host side
runs on a stand-in for the HIP runtime with two devices (tests/host/fake_hip.cpp), in a process of its own."""
import os
import shutil
import subprocess
import sys

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)

CHILD = r'''
import ctypes as C, sys, types
fake = C.CDLL(sys.argv[1], mode=C.RTLD_GLOBAL)
sys.modules['torch'] = types.ModuleType('torch')          # the binding names it; the real one would bring the real runtime along
sys.path.insert(0, sys.argv[2])
from trebi_amd import _lib
lib = _lib.lib()
where = lambda: (fake.hipGetDevice(C.byref(now)), now.value)[1]
now = C.c_int()
seen = []
def call(name, *a, want=0):
    rc = getattr(lib, name)(*a)
    assert rc == want, (name, rc, lib.trebi_last_error())
    seen.append(name)
    assert where() == 0, f'{name} left device {now.value} current'

ctx, h = C.c_void_p(), C.c_void_p()
call('trebi_ctx_create', 1, C.byref(ctx))
d = _lib.TrainDesc()
d.horizon, d.observation_dim, d.action_dim, d.n_timesteps, d.dim, d.n_mults = 8, 3, 2, 20, 32, 2
d.dim_mults[0], d.dim_mults[1] = 1, 2
d.n_cond = 1
call('trebi_trainer_create', ctx, C.byref(d), 4, C.byref(h))
n = lib.trebi_trainer_param_count(h)
buf = lambda k: C.c_void_p((lambda b: (keep.append(b), (C.addressof(b) + 255) // 256 * 256)[1])((C.c_float * (k + 64))()))
f = lambda k: C.cast(buf(k), _lib.c_float_p)
keep = []
call('trebi_trainer_bind', h, buf(n), buf(n), buf(n), buf(n), buf(n), f(40), f(20), f(20))
x, t, g = buf(160), buf(64), buf(160)
call('trebi_trainer_repack', h, None)
call('trebi_trainer_forward', h, x, t, g, 4, None)
call('trebi_trainer_backward', h, x, t, g, 4, None)
cond = (C.c_void_p * 1)(buf(12).value)
call('trebi_trainer_accumulate', h, x, cond, t, g, 4, 1.0, buf(2), None)
call('trebi_trainer_step', h, 1, 1e-3, 0.9, 0.999, 1e-8, 0, 0.0, None)
call('trebi_trainer_step_clipped', h, 2, 1e-3, 0.9, 0.999, 1e-8, 0, 0.0, 1.0, buf(1), None)
call('trebi_trainer_set_precision', h, 1, 0)
call('trebi_trainer_set_precision', h, 0, 0)
tok = _lib.TokenDesc(4, 10, 0, None, None, None, 0, 1)
pol = _lib.PolicyLossDesc(0, x, None, None, 10, 1, 0, 0, 0, 0, x, 1, 0, g, g, 0.2, 0.2, 0.0, 0.0, 3, 0, 0.0, 1.0)
call('trebi_policy_loss', ctx, C.byref(tok), C.byref(pol), None, 0, None)
call('trebi_policy_loss', ctx, C.byref(tok), C.byref(_lib.PolicyLossDesc()), None, 0, None, want=-1)
call('trebi_trainer_forward', h, x, t, g, 5, None, want=-2)
print('calls', len(seen))
'''


@pytest.mark.skipif(shutil.which('g++') is None, reason='needs g++')
def test_calls_put_the_caller_s_device_back(tmp_path):
    so = str(tmp_path / 'libfake_hip.so')
    subprocess.run(['g++', '-shared', '-fPIC', '-O1', '-w', '-D__HIP_PLATFORM_AMD__', '-I/opt/rocm/include',
                    os.path.join(HERE, 'host', 'fake_hip.cpp'), '-o', so], check=True)
    r = subprocess.run([sys.executable, '-c', CHILD, so, os.path.join(ROOT, 'safe-offline-rl-with-diffusion-model_amd')],
                       capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and 'calls 14' in r.stdout, r.stdout + r.stderr
