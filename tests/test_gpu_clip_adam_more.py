"""ClipAdam with norms that are infinite or NaN under a finite limit, and gradients that only share strides and lengths with their
parameters."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("n", [100, 400000])
@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_non_finite_norm_as_torch(value, n, t):
    """As clip_grad_norm_ and Adam have it: an infinite norm clips all to 0 and leaves NaN where the infinity was, a NaN norm
    leaves NaN everywhere.  Before it and beside it: the same finite numbers, up to the steps' few roundings of 2^-24."""
    import g1env
    gen = torch.Generator(device="cuda").manual_seed(n)
    start, other = torch.randn(n, device="cuda", generator=gen), torch.randn(50, device="cuda", generator=gen)
    ours = [torch.nn.Parameter(start.clone()), torch.nn.Parameter(other.clone())]
    theirs = [torch.nn.Parameter(start.clone()), torch.nn.Parameter(other.clone())]
    a, b = g1env.ClipAdam(ours, lr=1e-2, max_norm=0.5), torch.optim.Adam(theirs, lr=1e-2)
    for step in range(2):
        gs = [torch.randn(n, device="cuda", generator=gen).to(t), torch.randn(50, device="cuda", generator=gen).to(t)]
        if step == 1:
            gs[0][17] = value
        keep = [g.clone() for g in gs]
        norm = a.step(gs)
        assert all(torch.equal(torch.nan_to_num(g, nan=7.0), torch.nan_to_num(k, nan=7.0)) for g, k in zip(gs, keep))
        for p, g in zip(theirs, gs):
            p.grad = g.float()
        want = torch.nn.utils.clip_grad_norm_(theirs, 0.5)
        b.step()
        assert torch.isnan(norm).item() == torch.isnan(want).item() and torch.isinf(norm).item() == torch.isinf(want).item()
        for p, q in zip(ours, theirs):
            assert torch.equal(torch.isnan(p), torch.isnan(q))
            off = torch.nan_to_num(p.detach() - q.detach()).abs()
            # a parameter of size up to 6 and an update of 1e-2: a few roundings of either
            assert off.max().item() <= 20 * 2.0 ** -24 * 6
    assert a.steps.tolist() == [2, 2]


def test_gradients_of_other_shapes_are_refused():
    import g1env
    c = lambda *s: torch.zeros(*s, device="cuda")
    for shape, g in (((2, 3), c(3, 3)[:, :2]), ((2, 3), c(6, 3)[:, :1]), ((4, 3), c(9).as_strided((2, 6), (3, 1))), ((2, 3), c(6))):
        p = torch.nn.Parameter(torch.ones(shape, device="cuda"))
        opt = g1env.ClipAdam([p])
        with pytest.raises(g1env.G1Error, match="shapes"):
            opt.step([g])
        assert bool((p == 1).all()) and opt.steps.item() == 0
        p.grad = torch.ones_like(p)
        opt.step()
        assert opt.steps.item() == 1
