"""Host side of gated policies without a GPU: packing, initialisation, and what the entry points refuse."""
import ctypes
import os

import pytest
import torch

vp = ctypes.c_void_p


@pytest.fixture(scope="module")
def lib():
    import g1env
    if not os.path.exists(g1env.LIB):
        from build import build  # g1.cu_b200/build.py
        build()
    return g1env.load_library()


def test_pack_and_init():
    import g1env
    ac = g1env.init_policy_normal(g1env.AC(100, 29, (64, 40), "swiglu", value_hidden=(16,)), seed=3)
    w = g1env.pack_weights(ac)
    n = 2 * 64 * 100 + 2 * 64 + 2 * 40 * 64 + 2 * 40 + 29 * 40 + 29 + 29 + 2 * 16 * 100 + 2 * 16 + 16 + 1
    assert w.numel() == n
    assert torch.equal(w[:2 * 64 * 100].view(128, 100), ac.body[0].weight)
    assert torch.equal(w[2 * 64 * 100:2 * 64 * 100 + 128], torch.zeros(128))
    assert abs(ac.body[0].weight.std().item() * 10 - 1) < 0.05
    assert [p.dtype for p in ac.parameters()] == [torch.float32] * len(list(ac.parameters()))
    with pytest.raises(g1env.G1Error):
        ac(torch.zeros(2, 100))


def test_plain_actor_critic_is_as_it_was():
    import g1env
    torch.manual_seed(0)
    ac = g1env.AC(100, 29)
    torch.manual_seed(0)
    body = torch.nn.Sequential(torch.nn.Linear(100, 256), torch.nn.Tanh(), torch.nn.Linear(256, 256), torch.nn.Tanh())
    mu, v = torch.nn.Linear(256, 29), torch.nn.Linear(256, 1)
    x = torch.randn(7, 100)
    a, _, b = ac(x)
    assert torch.equal(a, mu(body(x))) and torch.equal(b, v(body(x)).squeeze(-1))


A, B, C, D, W = 1 << 12, 1 << 14, 1 << 16, 1 << 18, 1 << 20


def _fwd(lib, M=5, K=16, F=8, type=1, act=2, x=A, ldx=16, w=B, ldw=16, b=C, h=D, ws=W, size=1 << 20):
    rc = lib.g1_gated_ff(M, K, F, type, act, x, ldx, w, ldw, b, h, ws, size, None)
    msg = lib.g1_env_last_error()
    lib.g1_env_clear_error()
    return rc, msg


BAD = [dict(M=-1), dict(K=0), dict(F=0), dict(M=(1 << 30) + 1), dict(K=(1 << 20) + 1), dict(type=0), dict(type=3), dict(act=-1),
       dict(act=4), dict(ldx=15), dict(ldw=15), dict(ldx=1 << 40), dict(x=None), dict(x=A + 1), dict(w=None), dict(w=B + 1),
       dict(b=C + 2)]


@pytest.mark.parametrize("kw", BAD, ids=str)
def test_refuses(lib, kw):
    rc, msg = _fwd(lib, **kw)
    assert rc == -22 and b"g1_gated_ff" in msg


def test_tile_count_bound(lib):
    assert _fwd(lib, M=1 << 30, K=1 << 20, F=1 << 20, ldx=1 << 20, ldw=1 << 20)[0] == -22
    assert lib.g1_gated_ff_workspace(1 << 30, 1 << 20, 1 << 20, A, 1 << 20, B, 1 << 20, 1) == 0


def test_workspace(lib):
    ws = lib.g1_gated_ff_workspace
    assert ws(100, 64, 32, A, 64, B, 64, 0) == 0                          # rows on 16-byte boundaries: no copies
    assert ws(100, 60, 32, A, 60, B, 60, 0) == 100 * 64 * 2 + 64 * 64 * 2
    assert ws(100, 60, 32, A, 64, B, 60, 0) == 64 * 64 * 2
    assert ws(100, 64, 32, A + 2, 64, B, 64, 0) == 100 * 64 * 2
    assert ws(4, 60, 32, A, 60, B, 60, 0) == 0                            # a few rows: single numbers are read
    assert ws(100, 64, 32, A, 64, B, 64, 1) > 100 * 64 * 2
    assert ws(-1, 64, 32, A, 64, B, 64, 1) == 0
