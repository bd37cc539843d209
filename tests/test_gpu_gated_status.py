"""Waits that run out, told apart: an env's own flag, the device's flag of the other gated calls, and the trainer that stops on
either.  The waits are bounded ones on barriers that nothing arrives at; nothing faults or hangs."""
import ctypes
import os
import subprocess
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _lib():
    import g1env
    lib = g1env.load_library()
    lib.g1_gated_ff_test_wait.argtypes = [ctypes.c_uint, ctypes.c_void_p]
    lib.g1_env_test_wait_timeout.argtypes = [ctypes.c_void_p, ctypes.c_uint]
    return lib


def _rollout(env, hidden):
    import g1env
    z = lambda *s: torch.zeros(*s, device="cuda")
    N, H = env.N, 2
    env.set_policy(hidden, "swiglu", precision="bf16")
    env.reset()
    ac = g1env.init_policy_normal(g1env.AC(100, 29, hidden, "swiglu").cuda(), seed=2)
    out = z(H, N, 100), z(H, N, 29), z(H, N), z(H, N), z(H, N), z(H, N), z(N)
    env.rollout(H, g1env.pack_weights(ac).detach(), z(100), torch.ones(100, device="cuda"), *out)
    return out


def test_flags_belong_to_their_callers():
    import g1env
    lib = _lib()
    a, b = g1env.G1Env(300, 10, 8, seed=1), g1env.G1Env(40, 10, 8, seed=2)
    for env in (a, b):
        _rollout(env, (64, 32))
    assert a.tc_status() == b.tc_status() == g1env.gated_ff_status() == 0
    # a call outside the envs: theirs do not report it, nor do they clear it
    assert lib.g1_gated_ff_test_wait(4096, None) == 0
    torch.cuda.synchronize()
    assert a.tc_status() == b.tc_status() == 0
    assert g1env.gated_ff_status(torch.device("cuda", 0)) == 1 and g1env.gated_ff_status() == 0
    # one env
    assert lib.g1_env_test_wait_timeout(a.h, 4096) == 0
    assert b.tc_status() == 0 and g1env.gated_ff_status() == 0
    assert a.tc_status() == 2 and a.tc_status() == 0
    for env in (a, b):
        assert all(bool(torch.isfinite(t).all()) for t in _rollout(env, (64, 32))) and env.tc_status() == 0
        env.close()


def test_status_waits_for_other_streams():
    """A wait that runs out later, on streams that do not wait for the default one."""
    import g1env
    lib = _lib()
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        torch.cuda._sleep(100_000_000)  # some 50 ms
        assert lib.g1_gated_ff_test_wait(4096, s.cuda_stream) == 0
    assert g1env.gated_ff_status() == 1 and g1env.gated_ff_status() == 0
    env = g1env.G1Env(40, 10, 8, seed=2)
    env.set_stream(s)
    with torch.cuda.stream(s):
        _rollout(env, (64, 32))
        assert lib.g1_env_test_wait_timeout(env.h, 4096) == 0
    assert env.tc_status() == 2 and env.tc_status() == 0
    env.set_stream(None)
    env.close()


TRAINER = """
import ctypes, sys
sys.path.insert(0, sys.argv[1])
import ppo_fused, g1env
lib = g1env.load_library()
lib.g1_gated_ff_test_wait.argtypes = [ctypes.c_uint, ctypes.c_void_p]
update = ppo_fused.ppo_update
def lost(*args):
    loss = update(*args)
    assert lib.g1_gated_ff_test_wait(4096, None) == 0
    return loss
ppo_fused.ppo_update = lost
saved = []
ppo_fused.torch.save = lambda *args: saved.append(args)
sys.argv = ["ppo_fused.py", "2", "64", "--smoke", "--gated", "--fused-opt", "--tag=lost_wait_test"]
try:
    ppo_fused.main()
except g1env.G1Error as e:
    assert "gated layer ran out" in str(e) and not saved, (e, saved)
    print("STOPPED")
"""


def test_the_trainer_stops():
    r = subprocess.run([sys.executable, "-c", TRAINER, os.path.join(ROOT, "g1.cu_b200")], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "STOPPED" in r.stdout and "SMOKE OK" not in r.stdout, r.stdout + r.stderr
