"""Gated policies through the framework's own paths: the bf16 rollout (g1_rollout with gated layers), the actor-critic with
its gradients, the update with the clipped Adam step, and the trainer's command.

Tolerances: the rollout rounds weights, observations and each layer's output to bf16 where the reference here does, sums in
fp32, and only the sums' order differs: a value on a rounding border moves by one bf16 step, 2^-7 of it; such moves are rare
and average out over the next layer's inputs: 1e-2 of the outputs' norm, as for the plain wide policy.  Gradients of the
actor-critic against the same network in fp64 from the fp32 weights: every bf16 rounding (inputs, weights, layer
outputs, dz: about 4 a layer and direction, 2^-9 each on the average) adds up as the root of their number, 2 layers: 2^-9
sqrt(16) = 8e-3 of the norm; 3e-2 allowed."""
import os
import subprocess
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _act(name, g):
    return g * torch.sigmoid(g) if name == "swiglu" else g * 0.5 * (1 + torch.erf(g / 2 ** 0.5))


def _bf(t):
    return t.to(torch.bfloat16).float()


def _mlp(seq, x, name):
    h = _bf(x)
    for m in seq:
        z = h @ _bf(m.weight).T + m.bias
        f = z.shape[-1] // 2
        h = _bf(_act(name, z[..., :f]) * z[..., f:])
    return h


@pytest.mark.parametrize("name,hidden,value_hidden,N", [("swiglu", (128, 64), None, 300), ("geglu", (256, 1024, 512), (64, 40), 1000),
                                                        ("swiglu", (16,), None, 1), ("geglu", (24, 8), (8,), 3)])
def test_rollout(name, hidden, value_hidden, N):
    import g1env
    H = 2
    env = g1env.G1Env(N, 10, 8, seed=13)
    # another policy first: the buffers it leaves are smaller in biases, larger in weights
    env.set_policy((1024,), "elu", precision="bf16")
    z = lambda *s: torch.zeros(*s, device="cuda")
    mk = lambda: (z(H, N, 100), z(H, N, 29), z(H, N), z(H, N), z(H, N), z(H, N), z(N))
    mean, var = torch.zeros(100, device="cuda"), torch.ones(100, device="cuda")
    env.reset()
    plain = g1env.init_policy_normal(g1env.AC(100, 29, (1024,), "elu").cuda(), seed=1)
    env.rollout(H, g1env.pack_weights(plain).detach(), mean, var, *mk())
    env.set_policy(hidden, name, precision="bf16")
    env.set_value_net(value_hidden or ())
    env.reset()
    ac = g1env.init_policy_normal(g1env.AC(100, 29, hidden, name, value_hidden=value_hidden).cuda(), seed=2)
    g = torch.Generator(device="cuda").manual_seed(1)
    with torch.no_grad():
        ac.log_std.fill_(-20.0)
        for m in ac.modules():
            if isinstance(m, (torch.nn.Linear, g1env.GatedLinear)):
                m.bias.copy_(torch.randn(m.bias.shape, device="cuda", generator=g) * 0.2)
    O, A, LP, V, R, D, Vl = mk()
    env.rollout(H, g1env.pack_weights(ac).detach(), mean, var, O, A, LP, V, R, D, Vl)
    torch.cuda.synchronize()
    assert env.tc_status() == 0
    with torch.no_grad():
        for t in range(H):
            x = torch.clamp((O[t] - mean) / torch.sqrt(var + 1e-8), -10, 10)
            h = _mlp(ac.body, x, name)
            mu = h @ _bf(ac.mu.weight).T + ac.mu.bias
            hv = _mlp(ac.v_body, x, name) if value_hidden else h
            v = (hv @ _bf(ac.v.weight).T + ac.v.bias).squeeze(-1)
            assert ((A[t] - mu).norm() / mu.norm()).item() <= 1e-2
            assert ((V[t] - v).norm() / v.norm()).item() <= 1e-2
            # the actor-critic itself, whose heads are fp32
            mu2, _, v2 = ac(x)
            assert ((A[t] - mu2).norm() / mu2.norm()).item() <= 2e-2
    assert torch.isfinite(LP).all()
    env.close()


def test_gated_layers_need_the_bf16_path():
    import g1env
    env = g1env.G1Env(4, 10, 8, seed=1)
    for prec in ("fp32", "fp32-ffma"):
        with pytest.raises(g1env.G1Error):
            env.set_policy((64, 64), "swiglu", precision=prec)
    with pytest.raises(g1env.G1Error):
        env.set_policy((60,), "swiglu", precision="bf16")
    env.close()


@pytest.mark.parametrize("name", ["swiglu", "geglu"])
def test_actor_critic_gradients(name):
    import g1env
    torch.manual_seed(0)
    ac = g1env.AC(100, 29, (96, 40), name).cuda()
    x = torch.randn(500, 100, device="cuda")
    cm, cv = torch.randn(500, 29, device="cuda") / 500, torch.randn(500, device="cuda") / 500
    mu, _, v = ac(x)
    ((mu * cm).sum() + (v * cv).sum()).backward()
    got = {n: p.grad.double() for n, p in ac.named_parameters() if p.grad is not None}
    ps = {n: p.detach().double().requires_grad_() for n, p in ac.named_parameters()}
    h = x.double()
    for i in range(2):
        zz = h @ ps[f"body.{i}.weight"].T + ps[f"body.{i}.bias"]
        f = zz.shape[-1] // 2
        h = _act(name, zz[:, :f]) * zz[:, f:]
    mu = h @ ps["mu.weight"].T + ps["mu.bias"]
    v = (h @ ps["v.weight"].T + ps["v.bias"]).squeeze(-1)
    ((mu * cm).sum() + (v * cv).sum()).backward()
    for n, g in got.items():
        if n == "log_std":
            continue
        want = ps[n].grad
        assert ((g - want).norm() / want.norm()).item() <= 3e-2, n


def test_update_with_clipped_adam():
    """One PPO update of a gated actor-critic, gradients through the gated layers and the step by ClipAdam, beside the same
    update with torch's clipping and Adam.  The gradients are the same bits in the first step; its result differs by
    the step's roundings; further steps start from parameters that differ so little that bf16 hides it except on
    rounding borders: after the whole update the parameters agree to 5 % of what the update moved them by."""
    import g1env
    from ppo_fused import ppo_update
    outs = []
    for fused in (False, True):
        torch.manual_seed(5)
        ac = g1env.AC(100, 29, (64, 64), "swiglu").cuda()
        start = [p.detach().clone() for p in ac.parameters()]
        opt = g1env.ClipAdam(ac.parameters(), lr=3e-4, max_norm=0.5) if fused else torch.optim.Adam(ac.parameters(), lr=3e-4)
        g = torch.Generator(device="cuda").manual_seed(1)
        n = lambda *s: torch.randn(*s, device="cuda", generator=g)
        o, a, adv, ret = n(512, 100), n(512, 29), n(512), n(512)
        torch.manual_seed(6)
        ppo_update(ac, opt, o, a, n(512) - 40.0, adv, ret, epochs=2, mb=4)
        outs.append((start, [p.detach() for p in ac.parameters()]))
    moved = sum(float((p - s).square().sum()) for s, p in zip(*outs[0])) ** 0.5
    apart = sum(float((p - q).square().sum()) for p, q in zip(outs[0][1], outs[1][1])) ** 0.5
    assert moved > 0 and apart <= 0.05 * moved


@pytest.mark.parametrize("flags", [["--gated", "--fused-opt"], ["--fused-opt"], ["--config4", "--gated", "--no-eval"]])
def test_trainer_command(flags):
    r = subprocess.run([sys.executable, os.path.join(ROOT, "g1.cu_b200", "ppo_fused.py"), "2", "64", "--smoke", "--tag=gated_test"]
                       + flags, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "SMOKE OK" in r.stdout, r.stdout + r.stderr
    assert "nan" not in r.stdout.split("rew/step")[-1].split("sps")[0]
