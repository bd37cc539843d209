"""Hooks on the gated layer's saved tensors that bring them back with other strides (the same gradients, bit for bit) or left on
the host (refused before anything is launched)."""
import pytest
import torch
from test_gpu_gated import B16, _make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("K,off", [(48, 0), (45, 0), (48, 1)])
def test_other_strides(K, off):
    import g1env
    x, w, b, dh = _make(150, K, 48, B16, True, seed=16)
    x = torch.empty(150 * K + off, dtype=B16, device="cuda")[off:].view(150, K).copy_(x)
    want = g1env.gated_ff_backward_device(dh, x, w, b)
    gaps = lambda t: torch.stack([t, torch.full_like(t, 7)], -1)[..., 0]          # every second number
    turned = lambda t: t.t().contiguous().t() if t.dim() == 2 else t
    for back in (gaps, turned):
        leaves = [t.clone().requires_grad_() if t is not x else x.detach().requires_grad_() for t in (x, w, b)]
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, back):
            h = g1env.gated_ff(*leaves)
        h.backward(dh)
        for leaf, g in zip(leaves, want):
            assert torch.equal(leaf.grad, g)


def test_left_on_the_host():
    import g1env
    x, w, b, dh = _make(150, 48, 48, B16, True, seed=16)
    for back in (lambda t: t, lambda t: t.cuda().half(), lambda t: t.cuda()[:-1]):
        wl = w.clone().requires_grad_()
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), back):
            h = g1env.gated_ff(x, wl, b)
        with pytest.raises(g1env.G1Error, match="saved tensors"):
            h.backward(dh)
        assert wl.grad is None


def test_no_rows_and_other_bias_types():
    import g1env
    w, b = (torch.randn(20, 8, device="cuda") / 3).to(B16).requires_grad_(), torch.randn(20, device="cuda").to(B16).requires_grad_()
    x = torch.empty(0, 8, device="cuda", dtype=B16, requires_grad=True)
    h = g1env.gated_ff(x, w, b)
    h.sum().backward()
    assert h.shape == (0, 10) and x.grad.shape == (0, 8) and not w.grad.any() and not b.grad.any() and b.grad.dtype == B16
    x, w, b, dh = _make(30, 24, 16, B16, True, seed=3)
    want = g1env.gated_ff_backward_device(dh, x, w, b.to(B16))[2]
    for t in (B16, torch.float16, torch.float64):
        bl = b.to(B16).to(t).requires_grad_()
        g1env.gated_ff(x, w, bl).backward(dh)
        assert bl.grad.dtype == t and torch.equal(bl.grad, want.to(t))
