"""The trainer's check for waits that ran out, without a GPU: it asks the env and, for gated networks, the device."""
import pytest


class _Env:
    def __init__(self, status):
        self.status = status

    def tc_status(self):
        return self.status


@pytest.mark.parametrize("env,layers,gated,bad", [(0, 0, True, False), (2, 0, True, True), (0, 1, True, True), (-1, 0, False, True),
                                                  (0, -1, True, True), (0, 1, False, False)])
def test_check_waits(monkeypatch, env, layers, gated, bad):
    import g1env
    import ppo_fused
    asked = []
    monkeypatch.setattr(ppo_fused, "gated_ff_status", lambda dev: asked.append(dev) or layers)
    if bad:
        with pytest.raises(g1env.G1Error, match="wait"):
            ppo_fused.check_waits(_Env(env), "cuda:3", gated)
    else:
        ppo_fused.check_waits(_Env(env), "cuda:3", gated)
    assert asked == (["cuda:3"] if gated and env == 0 else [])
