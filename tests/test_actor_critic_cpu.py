"""The plain actor-critic under autocast: its heads take what the last hidden layer makes, with no cast between."""
import pytest
import torch


@pytest.mark.parametrize("value_hidden", [None, (16,)])
@pytest.mark.parametrize("activation", ["tanh", "elu"])
def test_heads_take_the_hidden_layers_type(activation, value_hidden):
    import g1env
    torch.manual_seed(0)
    ac = g1env.AC(100, 29, (32, 24), activation, value_hidden=value_hidden)
    seen = []
    for head in (ac.mu, ac.v):
        head.register_forward_pre_hook(lambda m, args: seen.append(args[0].dtype))
    x = torch.randn(5, 100)
    with torch.autocast("cpu", torch.bfloat16):
        ac(x)
    assert seen == [torch.bfloat16] * 2
    seen.clear()
    ac(x)
    assert seen == [torch.float32] * 2
