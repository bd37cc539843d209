"""The operators of a policy's update and of gated policies, as cases to be measured.

ff_fwd    one gated feed-forward layer, h = act(X Wg^T + bg) * (X Wu^T + bu), as a rollout or an
          evaluation calls it
ff_train  the same layer forward and backward, as the update calls it: h, dX, dW, db
clip      the global gradient norm over all tensors of a network, and the gradients scaled in place
adam      the norm, the clipping and the Adam step of a network's parameters

`own` false: the plain form in elementary torch operations, in 32 bits (64 for the long sums of the norm),
rounded once at the end; true: the framework's operators.
"""
import math
import os
import sys

import torch

own = False

MAX_NORM = 0.5          # the trainer's clip threshold
LR, BETAS, EPS = 3e-4, (0.9, 0.999), 1e-8
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
ACTS = ("tanh", "elu", "silu", "gelu")

# parameter shapes of the trainer's networks: the default 100-256-256 actor-critic, and the wide policy
# 100-1024-1024-512-29 with its separate 100-512-512-512-1 value network
DEFAULT_AC = [29, 256 * 100, 256, 256 * 256, 256, 29 * 256, 29, 256, 1]
WIDE_AC = [29, 1024 * 100, 1024, 1024 * 1024, 1024, 512 * 1024, 512, 29 * 512, 29, 512 * 100, 512, 512 * 512, 512,
           512 * 512, 512, 512, 1]


def listed():
    return [
        # one world asks for its next action: the weights' bytes and the call's latency are all there is
        dict(name="ff_fwd_one_world", op="ff_fwd", m=1, k=1024, f=1024, act="silu", type="bf16", bias=True),
        # an evaluation of a few hundred worlds on the raw 100 observations, odd width, no bias
        dict(name="ff_fwd_eval_odd", op="ff_fwd", m=333, k=100, f=257, act="gelu", type="fp16", bias=False),
        # a hidden layer of the wide policy in a rollout of 32768 worlds
        dict(name="ff_fwd_rollout", op="ff_fwd", m=32768, k=1024, f=1024, act="silu", type="bf16", bias=True),
        # the first layer in a smoke run's minibatch
        dict(name="ff_train_smoke", op="ff_train", m=1024, k=100, f=256, act="elu", type="bf16", bias=True),
        # a ragged minibatch and widths that fill no tile
        dict(name="ff_train_ragged", op="ff_train", m=10007, k=264, f=501, act="gelu", type="fp16", bias=True),
        # the 1024-to-512 layer in the update of 65536 worlds: a quarter of 32 x 65536 samples
        dict(name="ff_train_minibatch", op="ff_train", m=524288, k=1024, f=512, act="silu", type="bf16", bias=True),
        # the default network's gradients: nine tensors, 99387 numbers, latency
        dict(name="clip_default", op="clip", sizes="default", type="fp32", scale=1.0),
        # many tensors of all lengths, single numbers and odd lengths among them, 16-bit gradients
        dict(name="clip_many", op="clip", sizes="spread", count=300, total=3000000, type="bf16", scale=1.0),
        # a gradient far beyond the caches
        dict(name="clip_large", op="clip", sizes="spread", count=40, total=268435456, type="fp32", scale=0.01),
        # the update's last step for the default network, and for the wide one
        dict(name="adam_default", op="adam", sizes="default", type="fp32", scale=0.01),
        dict(name="adam_wide", op="adam", sizes="wide", type="fp32", scale=0.01),
        # a network far beyond the caches, 16-bit gradients for 32-bit parameters
        dict(name="adam_large", op="adam", sizes="spread", count=60, total=67108864, type="bf16", scale=0.01),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("ff_fwd", "ff_train", "clip", "adam"))
    if op in ("ff_fwd", "ff_train"):
        k, f = _log_int(rng, 8, 2048), _log_int(rng, 8, 2048)
        most = 524288 * 1024 * 512 if op == "ff_train" else 32768 * 1024 * 1024
        m = _log_int(rng, 1, max(1, min(524288, most // (k * f))))
        return dict(op=op, m=m, k=k, f=f, act=rng.choice(ACTS), type=rng.choice(("bf16", "fp16")),
                    bias=rng.random() < 0.7)
    count = _log_int(rng, 1, 400)
    total = _log_int(rng, max(count, 1000), 134217728 if op == "clip" else 33554432)
    return dict(op=op, sizes="spread", count=count, total=total, type=rng.choice(("fp32", "bf16")),
                scale=10.0 ** rng.uniform(-4, 1))


def _sizes(case):
    """Lengths of the tensors: a network of the trainer, or `count` lengths spread over their logarithm that add
    up to `total` (the first takes what is left)."""
    if case["sizes"] == "default":
        return list(DEFAULT_AC)
    if case["sizes"] == "wide":
        return list(WIDE_AC)
    count, total = case["count"], case["total"]
    w = [math.exp(math.log(1e6) * ((i * 0.6180339887498949) % 1.0)) for i in range(count)]
    s = sum(w)
    out = [max(1, int(total * x / s)) for x in w]
    big = max(range(count), key=lambda i: out[i])
    out[big] += total - sum(out)
    return out


def _tensors(case, flat, sizes):
    """The numbers of `flat` as tensors of those lengths, and what holds them: the trainer's networks have
    tensors of their own, the others are views of one flat buffer, as a flat all-reduce bucket leaves them."""
    parts = list(torch.split(flat, sizes))
    if case["sizes"] == "spread":
        return parts, [flat]
    parts = [t.clone() for t in parts]
    return parts, parts


def _own():
    here = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "g1.cu_b200")
    if here not in sys.path:
        sys.path.insert(0, here)
    import g1env
    return g1env


def _inputs(case, seed):
    """The inputs of a case, from the seed alone."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = TYPES[case["type"]]
    n = lambda *s: torch.randn(*s, device="cuda", generator=g)
    if case["op"] in ("ff_fwd", "ff_train"):
        m, k, f = case["m"], case["k"], case["f"]
        d = dict(x=n(m, k).clamp_(-10.0, 10.0).to(t), w=(n(2 * f, k) / math.sqrt(k)).to(t),
                 b=n(2 * f) * 0.1 if case["bias"] else None)
        if case["op"] == "ff_train":
            # the loss is a mean over the rows; 16-bit floats with a short exponent carry a loss scale
            d["dh"] = (n(m, f) * (1.0 if case["type"] == "fp16" else 1.0 / math.sqrt(m))).to(t)
        return d
    sizes = _sizes(case)
    total = sum(sizes)
    # gradients of different layers differ in size by orders of magnitude
    mag = torch.exp(torch.randn(len(sizes), device="cuda", generator=g))
    grad = n(total) * case["scale"]
    grad *= torch.repeat_interleave(mag, torch.tensor(sizes, device="cuda"), output_size=total)
    bufs = dict(g=grad.to(t))
    if case["op"] == "adam":
        bufs["p"] = n(total) * 0.05
        bufs["m"] = n(total) * (0.1 * case["scale"])
        bufs["v"] = n(total).square_() * (case["scale"] ** 2)
    d = {}
    for name, flat in bufs.items():
        d[name], d["held_" + name] = _tensors(case, flat, sizes)
    d["t"] = 1 + seed % 1000           # steps taken before this one
    return d


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = dict(case)
    if own:
        s["g1env"] = g1env = _own()
        if case["op"] == "ff_train":
            for name in ("x", "w", "b"):
                if s[name] is not None:
                    s[name].requires_grad_(True)
        if case["op"] == "adam":
            params = [torch.nn.Parameter(p) for p in s["p"]]
            s["opt"] = g1env.ClipAdam(params, lr=LR, betas=BETAS, eps=EPS, max_norm=MAX_NORM,
                                      moments=(s["m"], s["v"]), steps=s["t"])
            if case["type"] == "fp32":
                for p, g in zip(params, s["g"]):
                    p.grad = g
    return s


# ------------------------------------------------------------------------------ plain forms
def _act(name, g):
    if name == "tanh":
        return torch.tanh(g)
    if name == "elu":
        return torch.where(g > 0, g, torch.expm1(g))
    if name == "silu":
        return g / (1.0 + torch.exp(-g))
    return g * 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))


def _act_grad(name, g):
    if name == "tanh":
        return 1.0 - torch.tanh(g).square()
    if name == "elu":
        return torch.where(g > 0, torch.ones_like(g), torch.exp(g))
    if name == "silu":
        s = 1.0 / (1.0 + torch.exp(-g))
        return s * (1.0 + g * (1.0 - s))
    return 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5))) + g * torch.exp(-0.5 * g * g) * (1.0 / math.sqrt(2.0 * math.pi))


def _plain_ff(s):
    c = s["case"]
    t, f = TYPES[c["type"]], c["f"]
    x, w = s["x"].float(), s["w"].float()
    z = x @ w.T
    if s["b"] is not None:
        z = z + s["b"]
    g, u = z[:, :f], z[:, f:]
    a = _act(c["act"], g)
    h = (a * u).to(t)
    if c["op"] == "ff_fwd":
        return h
    dh = s["dh"].float()
    dz = torch.cat([dh * u * _act_grad(c["act"], g), dh * a], 1)
    out = [h, (dz @ w).to(t), (dz.T @ x).to(t)]
    return out + [dz.sum(0)] if s["b"] is not None else out


def _plain_norm(grads):
    total = torch.zeros((), dtype=torch.float64, device="cuda")
    for g in grads:
        total = total + g.double().square().sum()
    norm = total.sqrt()
    return norm, torch.clamp(MAX_NORM / (norm + 1e-6), max=1.0)


def _plain_clip(s):
    norm, coef = _plain_norm(s["g"])
    coef = coef.float()
    for g in s["g"]:
        g.copy_(g.float() * coef)
    return [norm.float()] + s["held_g"]


def _plain_adam(s):
    norm, coef = _plain_norm(s["g"])
    coef = coef.float()
    s["t"] += 1
    bc1, bc2 = 1.0 - BETAS[0] ** s["t"], 1.0 - BETAS[1] ** s["t"]
    for p, g, m, v in zip(s["p"], s["g"], s["m"], s["v"]):
        c = g.float() * coef
        m.copy_(BETAS[0] * m + (1.0 - BETAS[0]) * c)
        v.copy_(BETAS[1] * v + (1.0 - BETAS[1]) * c * c)
        p.sub_((LR / bc1) * m / (v.sqrt() / math.sqrt(bc2) + EPS))
    return [norm.float()] + s["held_p"] + s["held_m"] + s["held_v"]


# ------------------------------------------------------------------------------ one pass
def run(state):
    s, op = state, state["case"]["op"]
    if not own:
        return {"ff_fwd": _plain_ff, "ff_train": _plain_ff, "clip": _plain_clip, "adam": _plain_adam}[op](s)
    g1env = s["g1env"]
    if op == "ff_fwd":
        return g1env.gated_ff_device(s["x"], s["w"], s["b"], s["case"]["act"])
    if op == "ff_train":
        h = g1env.gated_ff(s["x"], s["w"], s["b"], s["case"]["act"])
        leaves = [s[n] for n in ("x", "w", "b") if s[n] is not None]
        return [h.detach()] + list(torch.autograd.grad(h, leaves, s["dh"]))
    if op == "clip":
        return [g1env.clip_grad_norm_device(s["g"], MAX_NORM)] + s["held_g"]
    # 16-bit gradients of 32-bit parameters do not fit in .grad and are handed over as a list
    norm = s["opt"].step() if s["case"]["type"] == "fp32" else s["opt"].step(s["g"])
    return [norm] + s["held_p"] + s["held_m"] + s["held_v"]


def work(case):
    if case["op"] in ("ff_fwd", "ff_train"):
        m, k, f = case["m"], case["k"], case["f"]
        nb = 2 * f if case["bias"] else 0
        fwd = dict(bytes=2 * (m * k + 2 * f * k + m * f) + 4 * nb, flops=4 * m * k * f)
        if case["op"] == "ff_fwd":
            return fwd
        # X, W, b and dh in, h, dX, dW and db out; two products forward, four backward
        return dict(bytes=2 * (2 * m * k + 4 * f * k + 2 * m * f) + 8 * nb, flops=12 * m * k * f)
    n = sum(_sizes(case))
    e = 4 if case["type"] == "fp32" else 2
    if case["op"] == "clip":
        return dict(bytes=2 * e * n + 4, flops=3 * n)
    return dict(bytes=(e + 24) * n + 4, flops=16 * n)


# ------------------------------------------------------------------------------ in 64 bits
def _held(case, parts):
    """Tensors as they are returned: the buffer that holds them, or each by itself."""
    return [torch.cat(parts)] if case["sizes"] == "spread" else parts


def exact(case, seed):
    d = _inputs(case, seed)
    if case["op"] in ("ff_fwd", "ff_train"):
        f = case["f"]
        x, wg, wu = d["x"].double(), d["w"][:f].double(), d["w"][f:].double()
        gate, up = torch.mm(x, wg.t()), torch.mm(x, wu.t())
        if d["b"] is not None:
            gate += d["b"][:f].double()
            up += d["b"][f:].double()
        if case["act"] == "tanh":
            val = torch.tanh(gate)
            slope = 1.0 - val * val
        elif case["act"] == "elu":
            slope = torch.exp(torch.clamp(gate, max=0.0))
            val = torch.clamp(gate, min=0.0) + torch.expm1(torch.clamp(gate, max=0.0))
        elif case["act"] == "silu":
            sig = torch.sigmoid(gate)
            val = gate * sig
            slope = sig + val * (1.0 - sig)
        else:
            cdf = 0.5 * torch.erfc(-gate / math.sqrt(2.0))
            val = gate * cdf
            slope = cdf + gate * torch.exp(-gate * gate / 2.0) / math.sqrt(2.0 * math.pi)
        h = val * up
        if case["op"] == "ff_fwd":
            return h
        dh = d["dh"].double()
        dgate, dup = dh * up * slope, dh * val
        del val, slope, gate, up
        out = [h, torch.mm(dgate, wg) + torch.mm(dup, wu),
               torch.cat([torch.mm(dgate.t(), x), torch.mm(dup.t(), x)])]
        if d["b"] is not None:
            out.append(torch.cat([dgate.sum(0), dup.sum(0)]))
        return out
    grads = [g.double() for g in d["g"]]
    norm = torch.stack([torch.linalg.vector_norm(g) for g in grads]).square().sum().sqrt()
    coef = torch.clamp(MAX_NORM / (norm + 1e-6), max=1.0)
    if case["op"] == "clip":
        return [norm] + _held(case, [g * coef for g in grads])
    t = d["t"] + 1
    ps, ms, vs = [], [], []
    for p, g, m, v in zip(d["p"], grads, d["m"], d["v"]):
        g = g * coef
        m1 = m.double() + (1.0 - BETAS[0]) * (g - m.double())
        v1 = v.double() + (1.0 - BETAS[1]) * (g * g - v.double())
        mhat, vhat = m1 / (1.0 - BETAS[0] ** t), v1 / (1.0 - BETAS[1] ** t)
        ps.append(p.double() - LR * mhat / (vhat.sqrt() + EPS))
        ms.append(m1)
        vs.append(v1)
    return [norm] + _held(case, ps) + _held(case, ms) + _held(case, vs)
