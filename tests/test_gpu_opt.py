"""Gradient norm, clipping and the clipped Adam step on the GPU against the formulas in 64 bits.

Tolerances (u = 2^-24 is fp32's rounding, relative to the value; 2^-8 bf16's, 2^-11 fp16's):
* norm: an fp64 sum rounded once to fp32: 2u.
* clipped gradient g c: c is rounded to fp32 and so is the product, then the result's own type rounds once: 2u, + the
  type's half step (for fp32 the product is the result).  Results below the type's normal range round
  absolutely, by half its smallest number.
* moments: m + (1-b1)(g' - m) with g' = g c: g' carries 2u, the difference and the fused add 1u each, (1-b1) 1u: 5u of
  |m| + |g'|.  v: sums of positive terms with at most 6 roundings: 8u of v.
* parameters: the update a m / (sqrt(v) rb + eps) carries the moments' 5u (scaled by the terms) + 4u + 8u for the root,
  the two corrections, the product, the sum and the quotient, and the result one rounding of p: u |p| + u |p'| +
  20u a (|m| + |g'|) / denominator.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
HALF = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _tensors(sizes, types, seed, scale=1.0):
    g = _gen(seed)
    return [(torch.randn(n, device="cuda", generator=g) * scale).to(t) for n, t in zip(sizes, types)]


def _norm64(ts):
    return math.sqrt(sum(float(t.double().square().sum()) for t in ts))


def _close(got, want, rel, floor=0.0):
    err = (got.double() - want).abs()
    lim = rel * want.abs() + floor
    assert bool((err <= lim).all()), (err - lim).max().item()


F, B, H = torch.float32, torch.bfloat16, torch.float16
LISTS = [
    ([1], [F]),
    ([0, 5, 0], [F, F, B]),
    ([256 * 100, 256, 65536, 256, 29 * 256, 29, 256, 1, 29], [F] * 9),
    ([1, 2, 3, 7, 8, 9, 2047, 2048, 2049, 4099], [B, H, F] * 3 + [B]),
    ([1 << 18], [F]),                       # the largest of the one-cluster path
    ([(1 << 18) + 1], [H]),                 # the smallest beyond it
    ([13] * 48 + [400000], [B] * 49),       # a table in the workspace
    ([5] * 60 + [0], [B, H, F, H] * 15 + [F]),  # one for the one-cluster path
    (list(range(1, 1101)), [F, B, H] * 366 + [F, B]),  # three table launches
    ([30000001, 5], [B, F]),                # long chunks
]


@pytest.mark.parametrize("sizes,types", LISTS, ids=lambda x: f"{len(x)}" if isinstance(x, list) else None)
@pytest.mark.parametrize("max_norm", [0.5, 1e9])
def test_clip(sizes, types, max_norm):
    import g1env
    ts = _tensors(sizes, types, seed=len(sizes))
    before = [t.clone() for t in ts]
    want = _norm64(before)
    norm = g1env.clip_grad_norm_device(ts, max_norm)
    assert abs(norm.item() - want) <= 2 * U * want
    c = min(1.0, max_norm / (want + 1e-6))
    for t, b in zip(ts, before):
        if c == 1.0:
            assert torch.equal(t, b)
        else:
            _close(t, b.double() * c, 2 * U + HALF[t.dtype], TINY[t.dtype] / 2)


def test_clip_views_of_one_buffer_and_neighbours():
    """Tensors at every offset of one buffer: the gaps between them stay as they were."""
    import g1env
    for t in (F, B, H):
        flat = torch.randn(5000, device="cuda", generator=_gen(1)).to(t)
        keep = flat.clone()
        views, used, o = [], torch.zeros(5000, dtype=torch.bool, device="cuda"), 0
        for n in (1, 2, 3, 5, 17, 33, 600, 1500):
            o += 1 + n % 3
            views.append(flat[o:o + n])
            used[o:o + n] = True
            o += n
        want = _norm64(views)
        g1env.clip_grad_norm_device(views, 0.25)
        assert torch.equal(flat[~used], keep[~used])
        _close(flat[used], keep[used].double() * (0.25 / (want + 1e-6)), 2 * U + HALF[t], TINY[t] / 2)


def test_clip_extreme_values():
    """Squares beyond fp32's range at both ends."""
    import g1env
    for s in (1e30, 1e-30):
        t = torch.full((1000,), s, device="cuda")
        want = _norm64([t])
        assert abs(g1env.clip_grad_norm_device([t], 1e9 if s < 1 else 1.0).item() - want) <= 2 * U * want
        if s > 1:
            _close(t, torch.full((1000,), s, device="cuda", dtype=torch.float64) / want, 3 * U)
    z = torch.zeros(10, device="cuda")
    assert g1env.clip_grad_norm_device([z], 0.5).item() == 0.0 and not z.any()
    assert g1env.clip_grad_norm_device([], 0.5).item() == 0.0
    t = torch.ones(10, device="cuda")
    g1env.clip_grad_norm_device(t, 0.0)
    assert not t.any()


@pytest.mark.parametrize("value", [float("inf"), float("nan")])
@pytest.mark.parametrize("n", [1000, 400000])
def test_clip_non_finite_as_torch(value, n):
    import g1env
    a = torch.randn(n, device="cuda", generator=_gen(2))
    a[17] = value
    p = torch.nn.Parameter(torch.zeros(n, device="cuda"))
    p.grad = a.clone()
    want = torch.nn.utils.clip_grad_norm_([p], 0.5)
    got = g1env.clip_grad_norm_device([a], 0.5)
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.isinf(got), torch.isinf(want))
    assert torch.equal(torch.isnan(a), torch.isnan(p.grad))
    assert not torch.nan_to_num(a).any() and not torch.nan_to_num(p.grad).any()


def test_no_limit_with_infinite_gradients():
    """max_norm inf clips nothing: an infinite gradient stays its own tensor's trouble, as in Adam without clipping."""
    import g1env
    a = torch.tensor([1.0, float("inf"), 2.0], device="cuda")
    keep = a.clone()
    assert g1env.clip_grad_norm_device([a], float("inf")).item() == float("inf") and torch.equal(a, keep)
    p = torch.nn.Parameter(torch.ones(3, device="cuda"))
    g1env.ClipAdam([p], lr=0.1).step([a])
    assert torch.isfinite(p.detach()).tolist() == [True, False, True]


def test_clip_deterministic():
    import g1env
    for n in (100000, 5000000):
        t = torch.randn(n, device="cuda", generator=_gen(3))
        norms = {g1env.clip_grad_norm_device([t.clone()], 0.5).item() for _ in range(5)}
        assert len(norms) == 1


def _adam64(p, g, m, v, t, c, lr, b1, b2, eps, wd):
    g = g.double() * c
    m1 = m.double() + (1 - b1) * (g - m.double())
    v1 = b2 * v.double() + (1 - b2) * g * g
    den = v1.sqrt() / math.sqrt(1 - b2 ** t) + eps
    a = lr / (1 - b1 ** t)
    return p.double() * (1 - lr * wd) - a * m1 / den, m1, v1, a * (m.abs().double() + g.abs()) / den, m.abs() + g.abs()


@pytest.mark.parametrize("sizes,types", LISTS, ids=lambda x: f"{len(x)}" if isinstance(x, list) else None)
@pytest.mark.parametrize("max_norm,wd,lr_tensor", [(0.5, 0.0, False), (float("inf"), 0.01, True)])
def test_adam_steps(sizes, types, max_norm, wd, lr_tensor):
    """Three steps, each against the formula from the state before it."""
    import g1env
    ps = [torch.nn.Parameter(t) for t in _tensors(sizes, [F] * len(sizes), seed=5)]
    lr = 1e-2
    opt = g1env.ClipAdam(ps, lr=torch.full((), lr, device="cuda") if lr_tensor else lr, betas=(0.9, 0.95), eps=1e-6,
                         max_norm=max_norm, weight_decay=wd)
    for t in range(1, 4):
        gs = _tensors(sizes, types, seed=10 + t, scale=0.1)
        old = [[x.detach().clone() for x in xs] for xs in (ps, opt.exp_avg, opt.exp_avg_sq, gs)]
        norm = opt.step(gs)
        want = _norm64(gs)
        assert abs(norm.item() - want) <= 2 * U * want
        c = min(1.0, max_norm / (want + 1e-6))
        for i in range(len(ps)):
            assert torch.equal(gs[i], old[3][i])
            p64, m64, v64, dp, dm = _adam64(old[0][i], gs[i], old[1][i], old[2][i], t, c, lr, 0.9, 0.95, 1e-6, wd)
            assert bool(((opt.exp_avg[i].double() - m64).abs() <= 5 * U * dm).all())
            _close(opt.exp_avg_sq[i], v64, 8 * U, 2.0 ** -149)
            lim = U * (old[0][i].abs() * 3 + p64.abs()) + 20 * U * dp
            assert bool(((ps[i].detach().double() - p64).abs() <= lim).all())
    assert opt.steps.tolist() == [0 if n == 0 else 3 for n in sizes]


def test_adam_tensors_without_gradient_and_grad_attribute():
    import g1env
    ps = [torch.nn.Parameter(torch.randn(50, 3, device="cuda", generator=_gen(i))) for i in range(3)]
    opt = g1env.ClipAdam(ps, lr=0.1, max_norm=1.0)
    keep = ps[1].detach().clone()
    for _ in range(2):
        opt.zero_grad()
        (ps[0].square().sum() + ps[2].sum()).backward()
        opt.step()
    assert torch.equal(ps[1].detach(), keep) and not opt.exp_avg[1].any()
    assert opt.steps.tolist() == [2, 0, 2]
    ps[0].grad = None
    ps[1].grad = torch.ones_like(ps[1])
    opt.step()
    assert opt.steps.tolist() == [2, 1, 3]
    # the first step of Adam is lr times the gradient's sign
    _close(ps[1].detach(), keep.double() - 0.1, 4 * U, 1e-6)


def test_adam_against_torch_clip_and_adam():
    """Ten steps of a small network beside torch's clip_grad_norm_ and Adam; both round in fp32, so each step adds a few
    roundings of the parameter (3 U |p|) and of an update of size lr.  The gradients, taken in fp64, differ by their
    rounding and by what the parameters differ by, some 10 U of their usual size; an element whose gradients
    were 40 times smaller than usual in all steps would see 400 U of its update, a chance of (1/40)^10.  Twice
    10 (3 U |p| + 400 U lr)."""
    import g1env
    a = torch.nn.Linear(37, 11).cuda()
    b = torch.nn.Linear(37, 11).cuda()
    b.load_state_dict(a.state_dict())
    oa = torch.optim.Adam(a.parameters(), lr=3e-4)
    ob = g1env.ClipAdam(b.parameters(), lr=3e-4, max_norm=0.5)
    for k in range(10):
        x = torch.randn(64, 37, device="cuda", generator=_gen(k)).double()
        for net, opt in ((a, oa), (b, ob)):
            opt.zero_grad()
            y = x @ net.weight.double().T + net.bias.double()
            y.square().mean().backward()
        torch.nn.utils.clip_grad_norm_(a.parameters(), 0.5)
        oa.step()
        ob.step()
    for p, q in zip(a.parameters(), b.parameters()):
        lim = 2 * 10 * (3 * U * p.detach().abs() + 400 * U * 3e-4)
        assert bool(((p - q).detach().abs() <= lim).all())


def test_adam_strided_gradients_and_parameters():
    import g1env
    p = torch.nn.Parameter(torch.randn(20, 30, device="cuda", generator=_gen(1)).t())   # dense, transposed
    q = torch.nn.Parameter(p.detach().contiguous())
    g = torch.randn(30, 20, device="cuda", generator=_gen(2))
    a, b = g1env.ClipAdam([p], lr=0.1, max_norm=0.1), g1env.ClipAdam([q], lr=0.1, max_norm=0.1)
    a.step([g])
    b.step([g])
    assert torch.equal(p.detach(), q.detach())
    wide = torch.randn(30, 40, device="cuda", generator=_gen(3))
    a.step([wide[:, ::2]])
    b.step([wide[:, ::2].contiguous()])
    assert torch.equal(p.detach(), q.detach())


def test_adam_graph_counts_on():
    """A captured step replayed: the same as the eager steps, bit for bit, and two graphs with workspaces of their own."""
    import g1env
    for n in (5000, 600000):
        g = torch.randn(n, device="cuda", generator=_gen(1))
        ps = [torch.nn.Parameter(torch.ones(n, device="cuda")) for _ in range(2)]
        opts = [g1env.ClipAdam([p], lr=1e-2, max_norm=0.5) for p in ps]
        opts[0].step([g])
        opts[1].step([g])
        graphs = []
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                norm = opts[1].step([g])
            graphs.append(graph)
        for k in range(4):
            opts[0].step([g])
            graphs[k % 2].replay()
        torch.cuda.synchronize()
        assert opts[1].steps.item() == 5 and torch.equal(ps[0].detach(), ps[1].detach())
        assert torch.equal(opts[0].exp_avg_sq[0], opts[1].exp_avg_sq[0])


def test_state_dict_round_trip():
    import g1env
    p = torch.nn.Parameter(torch.randn(100, device="cuda", generator=_gen(1)))
    a = g1env.ClipAdam([p], lr=0.1, max_norm=1.0)
    gs = [torch.randn(100, device="cuda", generator=_gen(i)) for i in range(4)]
    a.step([gs[0]])
    sd, q = a.state_dict(), torch.nn.Parameter(p.detach().clone())
    b = g1env.ClipAdam([q])
    b.load_state_dict(sd)
    for g in gs[1:]:
        a.step([g])
        b.step([g])
    assert torch.equal(p.detach(), q.detach())


def test_streams_and_versions():
    import g1env
    s = torch.cuda.Stream()
    t = torch.randn(1000000, device="cuda", generator=_gen(1))
    want = _norm64([t])
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        n = g1env.clip_grad_norm_device([t], 0.5)
    torch.cuda.current_stream().wait_stream(s)
    assert abs(n.item() - want) <= 2 * U * want
    # a tensor saved for a backward pass and then changed is noticed by torch
    p = torch.nn.Parameter(torch.ones(10, device="cuda"))
    y = p.square().sum()
    g1env.ClipAdam([p]).step([torch.ones(10, device="cuda")])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_refusals():
    import g1env
    c = lambda *s, **k: torch.zeros(*s, device="cuda", **k)
    t = c(10)
    for bad in ([torch.zeros(3)], [c(3).double()], [c(3, 4)[:, :2]], [t, t], [t[:6], t[5:]]):
        with pytest.raises(g1env.G1Error):
            g1env.clip_grad_norm_device(bad, 1.0)
    with pytest.raises(g1env.G1Error, match="parameters"):
        g1env.clip_grad_norm_device([torch.nn.Parameter(c(4))], 1.0)
    for norm in (-1.0, float("nan")):
        with pytest.raises(g1env.G1Error):
            g1env.clip_grad_norm_device([t], norm)
    p = torch.nn.Parameter(c(10))
    for kw in (dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(eps=-1.0), dict(weight_decay=-0.1), dict(max_norm=float("nan"))):
        with pytest.raises(g1env.G1Error):
            g1env.ClipAdam([p], **kw).step([t])
    with pytest.raises(g1env.G1Error):
        g1env.ClipAdam([p, p]).step([t, c(10)])
    with pytest.raises(g1env.G1Error):
        g1env.ClipAdam([p]).step([c(11)])
    with pytest.raises(g1env.G1Error):
        g1env.ClipAdam([p]).step([t, t])
    with pytest.raises(g1env.G1Error):
        g1env.ClipAdam([torch.nn.Parameter(torch.zeros(3))])
    with pytest.raises(g1env.G1Error):
        g1env.ClipAdam([torch.nn.Parameter(c(3).half())])
    with pytest.raises(g1env.G1Error):
        g1env.ClipAdam([])
    with pytest.raises(g1env.G1Error):
        g1env.ClipAdam([p], moments=([c(9)], [c(10)]))
