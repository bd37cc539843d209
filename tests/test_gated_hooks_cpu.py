"""What the gated layer's backward pass takes back from hooks on saved tensors, without a GPU: the library is a fake that keeps the
calls, and CPU tensors pass for CUDA ones."""
import contextlib

import pytest
import torch


class _Fake:
    def __init__(self):
        self.calls = []

    def g1_gated_ff(self, *args):
        self.calls.append("forward")
        return 0

    def g1_gated_ff_workspace(self, *args):
        return 256

    def g1_gated_ff_backward(self, *args):
        self.calls.append("backward")
        return 0


@pytest.mark.parametrize("K", [16, 15])
@pytest.mark.parametrize("back,good", [(lambda t: t, True), (torch.clone, True), (lambda t: t.t().contiguous().t(), True),
                                       (lambda t: t.float().double(), False), (lambda t: t[:1], False),
                                       (lambda t: torch.cat([t, t]), False), (lambda t: t.to("meta"), False)],
                         ids=["same", "clone", "strided", "type", "shorter", "longer", "device"])
def test_saved_tensors_come_back_as_they_went(monkeypatch, K, back, good):
    import g1env
    fake = _Fake()
    monkeypatch.setattr(g1env, "load_library", lambda: fake)
    monkeypatch.setattr(g1env, "_on", lambda dev: contextlib.nullcontext())
    monkeypatch.setattr(g1env, "_stream_of", lambda dev: 0)
    x = torch.zeros(9, K, dtype=torch.bfloat16, requires_grad=True)
    w, b = torch.zeros(8, K, dtype=torch.bfloat16, requires_grad=True), torch.zeros(8, requires_grad=True)
    monkeypatch.setattr(torch.Tensor, "is_cuda", True, raising=False)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, back):
        h = g1env.gated_ff(x, w, b)
    if good:
        h.backward(torch.zeros_like(h))
        assert fake.calls == ["forward", "backward"]
    else:
        with pytest.raises(g1env.G1Error, match="saved tensors"):
            h.backward(torch.zeros_like(h))
        assert fake.calls == ["forward"]
