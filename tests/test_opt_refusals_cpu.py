"""Arguments that the gradient-norm and Adam entry points refuse before any GPU work (no GPU here)."""
import ctypes
import os

import pytest

vp = ctypes.c_void_p


@pytest.fixture(scope="module")
def lib():
    import g1env
    if not os.path.exists(g1env.LIB):
        from build import build  # g1.cu_b200/build.py
        build()
    return g1env.load_library()


WS = ctypes.create_string_buffer(1 << 16)
WS_PTR = (ctypes.addressof(WS) + 15) & ~15
NORM = ctypes.c_float()


def _clip(lib, ptrs, types, counts, max_norm=1.0, norm=ctypes.addressof(NORM), ws=WS_PTR, size=1 << 15, n=None):
    k = len(ptrs)
    rc = lib.g1_clip_grad_norm(k if n is None else n, (vp * k)(*ptrs), (ctypes.c_int * k)(*types),
                               (ctypes.c_longlong * k)(*counts), max_norm, norm, ws, size, None)
    msg = lib.g1_env_last_error()
    lib.g1_env_clear_error()
    return rc, msg


def test_clip_refuses(lib):
    ok = dict(ptrs=[4096, 8192], types=[0, 1], counts=[10, 10])
    bad = [dict(ok, n=-1), dict(ok, max_norm=-1.0), dict(ok, max_norm=float("nan")), dict(ok, norm=None),
           dict(ok, ws=None), dict(ok, ws=WS_PTR + 8), dict(ok, size=100), dict(ok, types=[0, 3]), dict(ok, types=[-1, 0]),
           dict(ok, counts=[10, -1]), dict(ok, counts=[10, 1 << 50]), dict(ok, ptrs=[4096, None]),
           dict(ok, ptrs=[4097, 8192]), dict(ok, ptrs=[4098, 8192]), dict(ok, ptrs=[4096, 8193]),
           dict(ok, ptrs=[4096, 4096]), dict(ok, ptrs=[4096, 4096 + 36]), dict(ok, ptrs=[8192 + 18, 8192])]
    for kw in bad:
        rc, msg = _clip(lib, **kw)
        assert rc == -22 and msg and b"g1_clip_grad_norm" in msg, kw


def _adam(lib, g=(4096,), t=(0,), p=(1 << 16,), m=(1 << 17,), v=(1 << 18,), counts=(100,), steps=1 << 19, lr=1e-3,
          lr_dev=None, b1=0.9, b2=0.999, eps=1e-8, wd=0.0):
    n = len(g)
    arr = lambda x: (vp * n)(*x)
    rc = lib.g1_clip_adam(n, arr(g), (ctypes.c_int * n)(*t), arr(p), arr(m), arr(v), (ctypes.c_longlong * n)(*counts),
                          steps, 1.0, lr, lr_dev, b1, b2, eps, wd, ctypes.addressof(NORM), WS_PTR, 1 << 15, None)
    msg = lib.g1_env_last_error()
    lib.g1_env_clear_error()
    return rc, msg


def test_adam_refuses(lib):
    nan = float("nan")
    bad = [dict(lr=-1.0), dict(lr=nan), dict(b1=1.0), dict(b1=-0.1), dict(b2=nan), dict(eps=-1.0), dict(wd=-1.0),
           dict(lr_dev=4098), dict(steps=None), dict(steps=4), dict(p=(None,)), dict(m=(1 << 17 | 2,)),
           dict(p=(4096,)), dict(m=(1 << 16,)), dict(v=((1 << 17) + 396,)), dict(g=(None,))]
    for kw in bad:
        rc, msg = _adam(lib, **kw)
        assert rc == -22 and msg and b"g1_clip_adam" in msg, kw


def test_workspace_size(lib):
    assert lib.g1_opt_workspace(-1) == 0
    assert lib.g1_opt_workspace(100) > lib.g1_opt_workspace(0) > 0


def test_python_refuses_cpu_tensors():
    import torch

    import g1env
    if torch.cuda.is_available():
        pytest.skip("GPU present")
    with pytest.raises(g1env.G1Error):
        g1env.clip_grad_norm_device([torch.zeros(3)], 1.0)
    with pytest.raises(g1env.G1Error):
        g1env.ClipAdam([torch.zeros(3)])
