"""The gated layer h = act(x Wg^T + bg) * (x Wu^T + bu), forward and backward, against the formulas in 64 bits.

Tolerances, element by element (U = 2^-24; HALF = half a step of the type, relative to the value: 2^-8 / 2^-11):
* a product of n 16-bit terms: each of the n/16 tensor-core steps and 16 additions within one may lose a step of fp32,
  2U, of the running sum, which is at most the sum of the terms' sizes: (n/16 + 16) 2U sum |x||w|.
* activations: |act'|, |act''| <= 1.2 for all four; act and act' themselves are good to 2^-20 of 1 + |g|.
* h: what g and u are off by, through the product, + HALF |h|.
* dg, du: likewise, times |dh|, + HALF of their value (they are rounded to the type between the products).
* dx, dw: the sum over the terms of what dz is off by times the other operand, + the product's own error,
  + HALF (fp32 dw: U) of the result.
* db: the sum over rows of what dz is off by before its rounding, + M/32 + 40 additions in fp32.
As worst cases these are loose for long sums, so the 2-norm of the whole error is held as well: terms rounded
by at most HALF, independently, and the result once more: sqrt(2) HALF / sqrt(3) of its norm, twice that allowed.
fp16 results below the type's normal range round absolutely, by 2^-25 (dz: each term).
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
B16, F16 = torch.bfloat16, torch.float16
HALF = {B16: 2.0 ** -8, F16: 2.0 ** -11, torch.float32: U}
SUB = {B16: 2.0 ** -134, F16: 2.0 ** -25, torch.float32: 2.0 ** -150}
ACTS = ("tanh", "elu", "silu", "gelu")


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _make(M, K, F, t, bias, seed, dh_scale=1.0):
    g = _gen(seed)
    n = lambda *s: torch.randn(*s, device="cuda", generator=g)
    return (n(M, K).to(t), (n(2 * F, K) / math.sqrt(K)).to(t), n(2 * F) * 0.3 if bias else None, (n(M, F) * dh_scale).to(t))


def _act64(name, g):
    if name == "tanh":
        a = torch.tanh(g)
        return a, 1 - a * a
    if name == "elu":
        return torch.where(g > 0, g, torch.expm1(g)), torch.where(g > 0, torch.ones_like(g), torch.exp(g))
    if name == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    c = 0.5 * torch.erfc(-g / math.sqrt(2.0))
    return g * c, c + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)


def _oracle(x, w, b, dh, act):
    """Values and worst-case errors of h, dx, dw, db."""
    t, F = x.dtype, w.shape[0] // 2
    x, w, dh = x.double(), w.double(), dh.double()
    z, s = x @ w.T, x.abs() @ w.abs().T
    if b is not None:
        z, s = z + b.double(), s + b.double().abs()
    e = (x.shape[1] / 16 + 18) * 2 * U * s
    g, u, eg, eu = z[:, :F], z[:, F:], e[:, :F], e[:, F:]
    a, d = _act64(act, g)
    ea = 1.2 * eg + 2.0 ** -20 * (1 + g.abs())
    ed = 1.2 * eg + 2.0 ** -20 * (1 + g.abs())
    h = a * u
    eh = ea * (u.abs() + eu) + a.abs() * eu
    dz = torch.cat([dh * u * d, dh * a], 1)
    edz = torch.cat([dh.abs() * (ed * (u.abs() + eu) + d.abs() * eu), dh.abs() * ea], 1) + 4 * U * dz.abs()
    er = edz + HALF[t] * (dz.abs() + edz) + SUB[t]
    dx, dw = dz @ w, dz.T @ x
    edx = er @ w.abs() + (2 * F / 16 + 16) * 2 * U * ((dz.abs() + er) @ w.abs())
    edw = er.T @ x.abs() + (x.shape[0] / 16 + 400) * 2 * U * ((dz.abs() + er).T @ x.abs())
    db = dz.sum(0)
    edb = edz.sum(0) + (x.shape[0] / 32 + 40) * 2 * U * dz.abs().sum(0)
    return (h, eh), (dx, edx), (dw, edw), (db, edb)


def _check(name, got, want, norm_only=False):
    val, err = want
    t = got.dtype
    assert got.shape == val.shape, name
    off = (got.double() - val).abs()
    lim = err + HALF[t] * (val.abs() + err) + SUB[t]
    assert bool(torch.isfinite(got).all()) and bool((off <= lim).all()), (name, (off - lim).max().item())
    return off


def _check_norm(name, got, want, half, floor):
    """the whole error against twice sqrt(2/3) HALF of the whole result; floor: absolute roundings of tiny terms"""
    rel = (got.double() - want[0]).norm().item()
    assert rel <= 2 * math.sqrt(2 / 3) * half * want[0].norm().item() + floor, (name, rel, want[0].norm().item())


SHAPES = [(1, 1, 1), (1, 8, 8), (3, 17, 5), (128, 64, 128), (129, 65, 129), (2, 300, 2), (127, 100, 257), (300, 104, 1024),
          (64, 1024, 1024), (1000, 1024, 64), (2, 2048, 300), (5000, 40, 24), (777, 264, 501), (20000, 128, 136),
          (8200, 130, 700), (200, 2048, 2048),
          # sums of dx cut over CTAs (few rows, many outputs), on 64 and 128 columns; dw in two passes with cut sums
          (70, 40, 2500), (100, 104, 2600), (129, 129, 3001), (19000, 2048, 2048),
          # narrow matrices on pairs of CTAs
          (13000, 100, 60), (13001, 520, 40)]


@pytest.mark.parametrize("t", [B16, F16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("M,K,F", SHAPES)
def test_forward_backward(M, K, F, t):
    import g1env
    act = ACTS[(M + K + F) % 4]
    bias = (M + F) % 3 != 0
    x, w, b, dh = _make(M, K, F, t, bias, seed=M + 7 * K + 13 * F)
    h64, dx64, dw64, db64 = _oracle(x, w, b, dh, act)
    h = g1env.gated_ff_device(x, w, b, act)
    _check("h", h, h64)
    dx, dw, db = g1env.gated_ff_backward_device(dh, x, w, b, act)
    assert g1env.gated_ff_status() == 0
    _check("dx", dx, dx64)
    _check("dw", dw, dw64)
    _check("db", db, db64)
    if M * F >= 1000 and K * F >= 1000:
        _check_norm("h", h, h64, HALF[t], 0.0)
        _check_norm("dx", dx, dx64, HALF[t], SUB[t] * math.sqrt(2 * F * M * K))
        _check_norm("dw", dw, dw64, HALF[t], SUB[t] * math.sqrt(2 * F * M * K) * 3)
    dw32 = g1env.gated_ff_backward_device(dh, x, w, b, act, (False, True, False), torch.float32)
    assert dw32[0] is None and dw32[2] is None and torch.equal(dw32[1].to(t), dw)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("t", [B16, F16], ids=["bf16", "fp16"])
def test_activations_over_their_range(act, t):
    """x = one number, Wg = a ladder from -40 to 40: act and act' by themselves, far tails included."""
    import g1env
    F = 4001
    x = torch.ones(1, 1, device="cuda", dtype=t)
    w = torch.cat([torch.linspace(-40, 40, F, device="cuda"), torch.full((F,), 1.0, device="cuda")])[:, None].to(t)
    dh = torch.ones(1, F, device="cuda", dtype=t)
    h64, dx64, dw64, db64 = _oracle(x, w, None, dh, act)
    _check("h", g1env.gated_ff_device(x, w, None, act), h64)
    dx, dw, db = g1env.gated_ff_backward_device(dh, x, w, None, act)
    _check("dw", dw, dw64)
    _check("db", db, db64)
    # the tails keep their relative size where the formula does: silu and gelu of -10 are not zero
    if act == "silu" and t is B16:
        g = w[:F, 0].double()
        far = (g < -5) & (g > -30)
        got = g1env.gated_ff_device(x, w, None, act)[0, far].double()
        want = (g * torch.sigmoid(g))[far]
        assert bool(((got - want).abs() <= (HALF[t] + 2.0 ** -18) * want.abs()).all())


def test_gradient_against_differences():
    """db (fp32, from unrounded terms) against central differences of the formula in fp64 with the kernel's inputs; the
    difference quotient is off by about 1e-9."""
    import g1env
    M, K, F, eps = 40, 24, 16, 1e-4
    for act in ACTS:
        x, w, b, dh = _make(M, K, F, B16, True, seed=3)
        db = g1env.gated_ff_backward_device(dh, x, w, b, act)[2].double()
        f = lambda bb: ((lambda z: _act64(act, z[:, :F])[0] * z[:, F:])(x.double() @ w.double().T + bb) * dh.double()).sum()
        for j in (0, 5, F - 1, F, 2 * F - 1):
            step = torch.zeros(2 * F, device="cuda", dtype=torch.float64)
            step[j] = eps
            num = (f(b.double() + step) - f(b.double() - step)) / (2 * eps)
            # ELU's slope has a kink at 0: no value of g lies within eps of it here
            assert abs(num.item() - db[j].item()) <= 1e-5 * (1 + dh.double().abs().sum().item() / F)


def test_strided_and_misaligned_rows():
    import g1env
    g = _gen(1)
    big = torch.randn(300, 400, device="cuda", generator=g).to(B16)
    w = torch.randn(2 * 70, 64, device="cuda", generator=g).to(B16)
    wide = torch.randn(300, 70, device="cuda", generator=g).to(B16)
    for x in (big[:, :64], big[:, 8:72], big[:, 3:67], big[::2, 16:80], big[:, :128:2], big[:64].t()[:300], big[:1, :64],
              big[:5, :64].expand(5, 64), big[0, :64].expand(7, 64)):
        want = g1env.gated_ff_device(x.contiguous(), w)
        assert torch.equal(g1env.gated_ff_device(x, w), want)
        a = g1env.gated_ff_backward_device(wide[:x.shape[0]], x, w)
        c = g1env.gated_ff_backward_device(wide[:x.shape[0]], x.contiguous(), w)
        assert all(torch.equal(p, q) for p, q in zip(a, c))
    flat = torch.randn(2 * 70 * 64 + 1, device="cuda", generator=g).to(B16)
    w1 = flat[1:].view(140, 64)                                # weights off their 16-byte boundary
    assert torch.equal(g1env.gated_ff_device(big[:, :64], w1), g1env.gated_ff_device(big[:, :64], w1.clone()))
    # leading axes, and a gradient that is not laid out row by row
    x = big[:, :64].reshape(3, 100, 64)
    h = g1env.gated_ff_device(x, w)
    assert h.shape == (3, 100, 70) and torch.equal(h.view(300, 70), g1env.gated_ff_device(big[:, :64], w))
    dh = torch.ones((), device="cuda", dtype=B16).expand(3, 100, 70)
    a = g1env.gated_ff_backward_device(dh, x, w)
    c = g1env.gated_ff_backward_device(dh.contiguous(), x, w)
    assert all(torch.equal(p, q) for p, q in zip(a, c)) and a[0].shape == x.shape


def test_no_rows():
    import g1env
    w = torch.randn(20, 8, device="cuda").to(B16)
    x = torch.empty(0, 8, device="cuda", dtype=B16)
    assert g1env.gated_ff_device(x, w).shape == (0, 10)
    dx, dw, db = g1env.gated_ff_backward_device(torch.empty(0, 10, device="cuda", dtype=B16), x, w)
    assert dx.shape == (0, 8) and not dw.any() and not db.any()


def test_rows_do_not_touch_each_other():
    """A row of NaN, one of infinities: the other rows' bits stay; and a row's result does not depend on the row count."""
    import g1env
    for F in (40, 41):
        x, w, b, dh = _make(300, 72, F, B16, True, seed=9)
        h, dx = g1env.gated_ff_device(x, w, b), g1env.gated_ff_backward_device(dh, x, w, b)[0]
        y = x.clone()
        y[5], y[200] = float("nan"), float("inf")
        h2, dx2 = g1env.gated_ff_device(y, w, b), g1env.gated_ff_backward_device(dh, y, w, b)[0]
        keep = torch.ones(300, dtype=torch.bool, device="cuda")
        keep[5] = keep[200] = False
        assert torch.equal(h[keep], h2[keep]) and torch.equal(dx[keep], dx2[keep])
        assert bool(torch.isnan(h2[5]).all()) and not bool(torch.isfinite(dx2[5]).any())


def test_memory_around_the_outputs_stays():
    import ctypes
    import g1env
    lib = g1env.load_library()
    vp = lambda t: ctypes.c_void_p(t.data_ptr())
    for M, K, F in ((5, 24, 9), (130, 20, 33), (257, 64, 40)):
        x, w, b, dh = _make(M, K, F, F16, True, seed=2)
        bufs = {k: torch.full((n + 64,), 7.0, device="cuda", dtype=t) for k, n, t in
                (("h", M * F, F16), ("dx", M * K, F16), ("dw", 2 * F * K, F16), ("db", 2 * F, torch.float32))}
        n = lib.g1_gated_ff_workspace(M, K, F, vp(x), K, vp(w), K, 1)
        ws = torch.empty(n, dtype=torch.uint8, device="cuda")
        s = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
        assert lib.g1_gated_ff(M, K, F, 2, 2, vp(x), K, vp(w), K, vp(b), vp(bufs["h"]), vp(ws), n, s) == 0
        assert lib.g1_gated_ff_backward(M, K, F, 2, 2, vp(dh), vp(x), K, vp(w), K, vp(b), vp(bufs["dx"]), vp(bufs["dw"]), 2,
                                        vp(bufs["db"]), vp(ws), n, s) == 0
        want = [g1env.gated_ff_device(x, w, b), *g1env.gated_ff_backward_device(dh, x, w, b)]
        for k, y in zip(("h", "dx", "dw", "db"), want):
            assert torch.equal(bufs[k][:y.numel()], y.reshape(-1)) and bool((bufs[k][y.numel():] == 7.0).all()), k


def test_same_inputs_same_bits():
    import g1env
    x, w, b, dh = _make(30000, 200, 300, B16, True, seed=4)
    first = [g1env.gated_ff_device(x, w, b), *g1env.gated_ff_backward_device(dh, x, w, b)]
    for _ in range(3):
        again = [g1env.gated_ff_device(x, w, b), *g1env.gated_ff_backward_device(dh, x, w, b)]
        assert all(torch.equal(p, q) for p, q in zip(first, again))


def test_autograd_shared_weights_and_master_weights():
    import g1env
    x, w, b, dh = _make(150, 48, 48, B16, True, seed=6)
    master = w.float()
    leaves = [x.clone().requires_grad_(), master.clone().requires_grad_(), b.clone().requires_grad_()]
    h1 = g1env.gated_ff(leaves[0], leaves[1], leaves[2], "gelu")
    h2 = g1env.gated_ff(h1, leaves[1], leaves[2], "gelu")       # the same weights twice: gradients add up
    h2.backward(dh)
    want1 = g1env.gated_ff_device(x, w, b, "gelu")
    d2 = g1env.gated_ff_backward_device(dh, want1, w, b, "gelu", dw_dtype=torch.float32)
    d1 = g1env.gated_ff_backward_device(d2[0], x, w, b, "gelu", dw_dtype=torch.float32)
    assert torch.equal(h1, want1) and torch.equal(leaves[0].grad, d1[0])
    assert torch.equal(leaves[1].grad, d1[1] + d2[1]) and leaves[1].grad.dtype == torch.float32
    assert torch.equal(leaves[2].grad, d1[2] + d2[2])
    # gradients are only made for what asks for them, and twice differentiable it is not
    y = g1env.gated_ff(x, leaves[1], None)
    (gw,) = torch.autograd.grad(y, leaves[1], dh, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(gw.sum(), leaves[1])


@pytest.mark.parametrize("K,off", [(48, 0), (45, 0), (48, 1)])
def test_saved_tensors_go_through_hooks(K, off):
    """What the forward pass saves is what the backward pass works on: copies that a hook made (of which the originals may
    change), or those that a checkpoint makes again; and it is let go once the backward pass has been through."""
    import g1env
    from torch.utils.checkpoint import checkpoint
    x, w, b, dh = _make(150, K, 48, B16, True, seed=16)
    at = torch.empty(150 * K + off, dtype=B16, device="cuda")[off:].view(150, K)  # off 1: not on 16-byte boundaries
    want = g1env.gated_ff_backward_device(dh, x, w, b)
    for kind in ("copies", "host", "checkpoint"):
        wl, bl = w.clone().requires_grad_(), b.clone().requires_grad_()
        xl = at.copy_(x).detach().requires_grad_()
        if kind == "checkpoint":
            h = checkpoint(g1env.gated_ff, xl, wl, bl, use_reentrant=False)
        else:
            hooks = (torch.autograd.graph.save_on_cpu(pin_memory=True) if kind == "host"
                     else torch.autograd.graph.saved_tensors_hooks(torch.clone, lambda t: t))
            with hooks:
                h = g1env.gated_ff(xl, wl, bl)
            torch.cuda.synchronize()
            with torch.no_grad():
                at.fill_(float("nan"))
                wl.fill_(float("nan"))
                bl.fill_(float("nan"))
        h.backward(dh)
        for leaf, g in zip((xl, wl, bl), want):
            assert torch.equal(leaf.grad, g), kind
    # a layer's rows between two layers: freed by its backward pass, not with the graph's last name
    rows = 1 << 16
    x, w, b, dh = _make(rows, 64, 64, B16, True, seed=17)
    wl = w.clone().requires_grad_()
    h = x
    for _ in range(8):
        h = g1env.gated_ff(h, wl)
    mem = torch.cuda.memory_allocated()
    h.backward(dh)
    wl.grad = None
    assert torch.cuda.memory_allocated() <= mem - 7 * rows * 64 * 2


def test_streams_and_graphs():
    """Two captured calls with workspaces of their own, replayed in turn on new inputs, and a call on another stream."""
    import g1env
    shapes = ((300, 100, 60), (2000, 96, 200))
    data = [_make(*s, B16, True, seed=i) for i, s in enumerate(shapes)]
    graphs, outs = [], []
    for x, w, b, dh in data:
        g1env.gated_ff_device(x, w, b), g1env.gated_ff_backward_device(dh, x, w, b)
    torch.cuda.synchronize()
    for x, w, b, dh in data:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append([g1env.gated_ff_device(x, w, b), *g1env.gated_ff_backward_device(dh, x, w, b)])
        graphs.append(graph)
    for k in range(4):
        for (x, w, b, dh), s in zip(data, shapes):
            x.copy_(_make(*s, B16, True, seed=10 + k)[0])
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for (x, w, b, dh), out in zip(data, outs):
            want = [g1env.gated_ff_device(x, w, b), *g1env.gated_ff_backward_device(dh, x, w, b)]
            assert all(torch.equal(p, q) for p, q in zip(out, want))
    s = torch.cuda.Stream()
    x, w, b, dh = data[1]
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        h = g1env.gated_ff_device(x, w, b)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(h, g1env.gated_ff_device(x, w, b))


FIRST = """
import sys
sys.path.insert(0, sys.argv[1])
import torch, g1env
x = torch.randn(300, 100, device="cuda").bfloat16()
w = torch.randn(80, 100, device="cuda").bfloat16()
dh = torch.randn(300, 40, device="cuda").bfloat16()
p = torch.nn.Parameter(torch.randn(700000, device="cuda"))
q = torch.nn.Parameter(torch.randn(70, device="cuda"))
opt, small = g1env.ClipAdam([p], max_norm=0.5), g1env.ClipAdam([q], max_norm=0.5)
gp, gq = torch.randn_like(p), torch.randn_like(q)
graph = torch.cuda.CUDAGraph()
torch.cuda.synchronize()
with torch.cuda.graph(graph):
    h = g1env.gated_ff_device(x, w)
    one = g1env.gated_ff_device(x[:1], w)
    d = g1env.gated_ff_backward_device(dh, x, w)
    opt.step([gp]), small.step([gq])
    n = g1env.clip_grad_norm_device([gp.clone()], 0.5)
graph.replay()
torch.cuda.synchronize()
assert torch.equal(h, g1env.gated_ff_device(x, w)) and torch.equal(one, g1env.gated_ff_device(x[:1], w))
assert all(torch.equal(a, b) for a, b in zip(d, g1env.gated_ff_backward_device(dh, x, w)))
assert opt.steps.item() == small.steps.item() == 1 and abs(n.item() - gp.double().norm().item()) < 1e-3
print("FIRST OK")
"""


def test_first_calls_of_a_process_inside_a_capture():
    import os
    import subprocess
    import sys
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "g1.cu_b200")
    r = subprocess.run([sys.executable, "-c", FIRST, pkg], capture_output=True, text=True, timeout=200)
    assert r.returncode == 0 and "FIRST OK" in r.stdout, r.stdout + r.stderr


def test_a_wait_that_runs_out_is_reported():
    """Failure detection without a GPU fault: a bounded wait on a barrier that nothing arrives at."""
    import ctypes

    import g1env
    lib = g1env.load_library()
    lib.g1_gated_ff_test_wait.argtypes = [ctypes.c_uint, ctypes.c_void_p]
    assert g1env.gated_ff_status() == 0
    assert lib.g1_gated_ff_test_wait(4096, None) == 0
    assert g1env.gated_ff_status() == 1 and g1env.gated_ff_status() == 0
    x, w, b, dh = _make(300, 64, 40, B16, True, seed=8)
    first = g1env.gated_ff_device(x, w, b)
    assert torch.equal(first, g1env.gated_ff_device(x, w, b)) and g1env.gated_ff_status() == 0


def test_two_threads_at_once():
    """Two host threads, each on a stream of its own: the same bits as one after the other."""
    import threading

    import g1env
    data = [_make(700 + 300 * i, 96 + 8 * i, 120, B16, True, seed=20 + i) for i in range(2)]
    want = [[g1env.gated_ff_device(x, w, b), *g1env.gated_ff_backward_device(dh, x, w, b)] for x, w, b, dh in data]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        x, w, b, dh = data[i]
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(20):
                got = [g1env.gated_ff_device(x, w, b), *g1env.gated_ff_backward_device(dh, x, w, b)]
                if not all(torch.equal(p, q) for p, q in zip(got, want[i])):
                    bad.append(i)
        s.synchronize()

    ts = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in ts]
    [t.join() for t in ts]
    assert not bad


def test_offsets_beyond_32_bits():
    """More than 2^31 numbers in x, h and z: the last rows are where they belong."""
    import g1env
    M, K, F = 2_200_000, 1024, 1000
    free, _ = torch.cuda.mem_get_info()
    if free < 60e9:
        pytest.skip("needs 60 GB")
    g = _gen(1)
    w = (torch.randn(2 * F, K, device="cuda", generator=g) / 32).to(B16)
    rows = torch.randn(256, K, device="cuda", generator=g).to(B16)
    dr = torch.randn(256, F, device="cuda", generator=g).to(B16)
    x = torch.zeros(M, K, device="cuda", dtype=B16)
    dh = torch.zeros(M, F, device="cuda", dtype=B16)
    x[-256:] = rows
    dh[-256:] = dr
    h = g1env.gated_ff_device(x, w)
    assert torch.equal(h[-256:], g1env.gated_ff_device(rows, w)) and not h[:-256].any()
    dx, dw, db = g1env.gated_ff_backward_device(dh, x, w)
    a, bw, c = g1env.gated_ff_backward_device(dr, rows, w)
    assert torch.equal(dx[-256:], a) and not dx[:-256].any()
    # the same terms, added up in other groups
    assert bool(((dw.double() - bw.double()).abs() <= 2 * HALF[B16] * bw.double().abs() + 1e-3).all())
    assert bool(((db - c).abs() <= 1e-4 * (1 + c.abs())).all())


def test_refusals():
    import g1env
    x, w, b, dh = _make(4, 16, 8, B16, True, seed=1)
    f, bw = g1env.gated_ff_device, g1env.gated_ff_backward_device
    for args in ((x.cpu(), w, b), (x, w.cpu(), b), (x, w, b.cpu()), (x.float(), w.float(), b), (x, w.half(), b),
                 (x, w[:15], b), (x, w[:, :15], b), (x, w, b[:15]), (x, w[:0], None), (x, w, b, "relu"),
                 (x, w.view(-1), b), (x, w, b.int())):
        with pytest.raises(g1env.G1Error):
            f(*args)
    for args in ((dh.float(), x, w, b), (dh[:3], x, w, b), (dh.cpu(), x, w, b), (dh[:, :7], x, w, b)):
        with pytest.raises(g1env.G1Error):
            bw(*args)
    with pytest.raises(g1env.G1Error):
        bw(dh, x, w, b, dw_dtype=F16)
    with pytest.raises(g1env.G1Error):
        g1env.gated_ff(x, w.double(), b)
    with pytest.raises(g1env.G1Error):
        g1env.GatedLinear(16, 8)(torch.zeros(3, 16))
