"""How many numbers a packed policy has, for every kind of policy an env takes, and that a rollout refuses fewer."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hidden,act,prec,value", [((256, 256), "tanh", "fp32", None), ((100,), "elu", "fp32-ffma", None),
                                                   ((64, 32), "elu", "bf16", None), ((64, 32), "swiglu", "bf16", None),
                                                   ((64, 32), "elu", "bf16", (16, 24)), ((64, 32), "geglu", "bf16", (16, 24))])
def test_count(hidden, act, prec, value):
    import g1env
    lib = g1env.load_library()
    env = g1env.G1Env(3, 10, 8, seed=1)
    ac = g1env.AC(100, 29)
    assert lib.g1_env_weight_count(env.h) == g1env.pack_weights(ac).numel()   # before any policy is set
    env.set_policy(hidden, act, precision=prec)
    env.set_value_net(value or ())
    env.reset()
    W = g1env.pack_weights(g1env.init_policy_normal(g1env.AC(100, 29, hidden, act, value_hidden=value).cuda())).detach()
    assert lib.g1_env_weight_count(env.h) == W.numel()
    z = lambda *s: torch.zeros(*s, device="cuda")
    H, N = 1, 3
    bufs = z(H, N, 100), z(H, N, 29), z(H, N), z(H, N), z(H, N), z(H, N), z(N)
    mean, var = z(100), torch.ones(100, device="cuda")
    with pytest.raises(g1env.G1Error, match="packed weights"):
        env.rollout(H, W[:-1], mean, var, *bufs)
    with pytest.raises(g1env.G1Error, match="packed weights"):
        env.rollout(H, W.bfloat16(), mean, var, *bufs)
    env.rollout(H, W, mean, var, *bufs)
    torch.cuda.synchronize()
    assert all(bool(torch.isfinite(b).all()) for b in bufs)
    # an env that was made gated, and weights that were not
    if act == "elu" and prec == "bf16":
        env.set_policy(hidden, "swiglu", precision=prec)
        with pytest.raises(g1env.G1Error, match="packed weights"):
            env.rollout(H, W, mean, var, *bufs)
    env.close()
