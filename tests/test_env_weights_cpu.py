"""A rollout takes packed weights only where they hold all that the env's policy reads (no GPU: the library is a fake that keeps
the calls, the tensors pass for CUDA ones)."""
import pytest
import torch


class _Fake:
    def __init__(self):
        self.calls = 0

    def g1_env_weight_count(self, h):
        return 1000

    def g1_rollout(self, *args):
        self.calls += 1

    def g1_env_last_error_code(self):
        return 0


class _Cuda(torch.Tensor):
    is_cuda = True


def test_weights_that_are_too_few_are_refused(monkeypatch):
    import g1env
    fake = _Fake()
    monkeypatch.setattr(g1env, "_lib", fake)
    env = object.__new__(g1env.G1Env)
    env.h = None
    go = lambda W: env.rollout(2, W, *[None] * 9)
    cuda = lambda *s, **k: torch.zeros(*s, **k).as_subclass(_Cuda)
    for bad in (cuda(999), cuda(1000, dtype=torch.bfloat16), cuda(2000)[::2], torch.zeros(1000), cuda(0)):
        with pytest.raises(g1env.G1Error, match="packed weights"):
            go(bad)
    assert fake.calls == 0
    go(cuda(1000))
    go(cuda(1200))
    assert fake.calls == 2
