"""The host side of ClipAdam and clip_grad_norm_device without a GPU: which gradients reach the library.  The library is a fake that keeps the calls; the
tensors are on the CPU, so only the checks of device are out of the way."""
import contextlib

import pytest
import torch


class _Fake:
    def __init__(self):
        self.calls = []

    def g1_opt_workspace(self, n):
        return 64

    def g1_clip_adam(self, n, *args):
        self.calls.append((n,) + args)
        return 0


@pytest.fixture
def make(monkeypatch):
    import g1env
    fake = _Fake()
    monkeypatch.setattr(g1env, "_lib", fake)
    monkeypatch.setattr(g1env, "_require_gpu", lambda: None)
    monkeypatch.setattr(g1env, "load_library", lambda: fake)
    monkeypatch.setattr(g1env, "_cuda_list", lambda ts, what, types: (torch.device("cpu"), {t.dtype for t in ts}))
    monkeypatch.setattr(g1env, "_on", lambda dev: contextlib.nullcontext())
    monkeypatch.setattr(g1env, "_stream_of", lambda dev: 0)

    def build(params, **kw):
        opt = g1env.ClipAdam(params, **kw)
        opt._where = {-1}  # where get_device() says that CPU tensors are
        return opt, fake
    return build


# shapes of parameter and gradient, and the gradient: equal strides and lengths do not make equal shapes
def _cases():
    z = torch.zeros
    return [((2, 3), z(3, 3)[:, :2]),                             # [3, 2], strides (3, 1)
            ((2, 3), z(6, 3)[:, :1]),                             # [6, 1], strides (3, 1)
            ((4, 3), z(9).as_strided((2, 6), (3, 1))),            # overlaps itself: 9 numbers where 12 would be read
            ((2, 3), z(6)), ((2, 3), z(3, 2)), ((6,), z(2, 3))]


@pytest.mark.parametrize("i", range(6))
def test_gradients_of_other_shapes_are_refused(make, i):
    import g1env
    shape, g = _cases()[i]
    opt, fake = make([torch.nn.Parameter(torch.zeros(shape))])
    with pytest.raises(g1env.G1Error, match="shapes"):
        opt.step([g])
    assert not fake.calls
    opt.step([torch.zeros(shape)])
    assert len(fake.calls) == 1 and fake.calls[0][0] == 1


def test_parameter_of_another_shape_is_noticed(make):
    import g1env
    p = torch.nn.Parameter(torch.zeros(2, 3))
    opt, fake = make([p])
    p.data = torch.zeros(3, 3)[:, :2]
    with pytest.raises(g1env.G1Error, match="laid out"):
        opt.step([torch.zeros(2, 3)])
    assert not fake.calls


def _state(opt):
    return [opt.lr] + [t.clone() for t in (*opt.exp_avg, *opt.exp_avg_sq, opt.steps)]


@pytest.mark.parametrize("change", [dict(exp_avg=lambda d: d[:1]), dict(exp_avg_sq=lambda d: d[:1]),
                                    dict(exp_avg_sq=lambda d: [d[0], d[1][:1]]), dict(exp_avg_sq=lambda d: d + d),
                                    dict(steps=lambda s: s[:1]), dict(steps=lambda s: torch.tensor(3)),
                                    dict(steps=lambda s: s - 5), dict(steps=lambda s: s.float()),
                                    dict(lr=lambda x: torch.ones(2))], ids=lambda c: next(iter(c)))
def test_a_state_that_does_not_fit_changes_nothing(make, change):
    """Among them those that broadcasting or a shorter list would have let through."""
    import g1env
    ps = lambda: [torch.nn.Parameter(torch.zeros(2, 3)), torch.nn.Parameter(torch.zeros(4))]
    src, dst = make(ps(), lr=0.5, steps=2)[0], make(ps(), lr=0.1)[0]
    for t in src.exp_avg + src.exp_avg_sq:
        t.fill_(1.0)
    d = src.state_dict()
    (key, f), = change.items()
    before = _state(dst)
    with pytest.raises(g1env.G1Error, match="state"):
        dst.load_state_dict(dict(d, **{key: f(d[key])}))
    assert all(torch.equal(a, b) if isinstance(a, torch.Tensor) else a == b for a, b in zip(before, _state(dst)))
    dst.load_state_dict(d)
    assert dst.lr == 0.5 and dst.steps.tolist() == [2, 2] and all(bool((t == 1).all()) for t in dst.exp_avg + dst.exp_avg_sq)


def test_negative_step_counts_are_refused(make):
    import g1env
    with pytest.raises(g1env.G1Error, match="steps"):
        make([torch.nn.Parameter(torch.zeros(3))], steps=-1)


@pytest.mark.parametrize("grads", [[None], [torch.zeros(3), None], ["weight"], {"a": torch.zeros(3)}])
def test_clipping_says_that_gradients_are_missing(monkeypatch, grads):
    """A parameter's .grad may be None."""
    import g1env
    monkeypatch.setattr(g1env, "load_library", lambda: _Fake())
    with pytest.raises(g1env.G1Error, match="must be tensors"):
        g1env.clip_grad_norm_device(grads, 1.0)


@pytest.mark.parametrize("params", [torch.nn.Parameter(torch.zeros(2, 3)), [{"params": [torch.zeros(3)]}],
                                    [("w", torch.zeros(3))], [None]], ids=["tensor", "groups", "names", "none"])
def test_parameters_must_be_a_list_of_tensors(make, params):
    """One tensor would be taken for the list of its rows, views that nobody else holds."""
    import g1env
    with pytest.raises(g1env.G1Error, match="parameters must be"):
        make(params)


def test_the_states_tensors_stay(make):
    """Other tensors in their places (offloaded, of other lengths) would be written to without a check."""
    opt, fake = make([torch.nn.Parameter(torch.zeros(2, 3))])
    was = [opt.exp_avg[0], opt.exp_avg_sq[0], opt.steps]
    for name in ("exp_avg", "exp_avg_sq", "steps"):
        with pytest.raises(AttributeError):
            setattr(opt, name, [torch.zeros(1)])
    for ms in (opt.exp_avg, opt.exp_avg_sq):
        with pytest.raises(TypeError):
            ms[0] = torch.zeros(1)
    opt.exp_avg[0].fill_(2.0)
    opt.step([torch.zeros(2, 3)])
    # n, gradients, types, p, m, v, counts, steps
    assert fake.calls[0][7] == was[2].data_ptr() and opt.exp_avg[0] is was[0] and opt.exp_avg_sq[0] is was[1]
