"""What the gated layer's outputs hold beyond the rounding of the 16-bit ones, against the formulas in 64 bits: the fp32 sums of db,
the fp32 dW, gradients far from 1 in fp16, far tails and non-finite gates.

Tolerances (U = 2^-24; HALF, SUB and the elementwise bounds as in test_gpu_gated.py, whose oracle is used):
* dz before its rounding, relative to its norm, E(K): a product of K terms loses at most a step of fp32, 2U, of the running sum
  at each of its K/16 steps and at 18 additions; act and act' carry that on, times 1.2 at most, for g and once for u: allow
  4U (K/16 + 18) together; act and act' by themselves are good to 2^-20 of 1 + |g|, |g| mostly below 1: 2^-19.
* db, 2-norm: E(K), and M/32 + 40 additions in fp32 that round to nearest, independently: 2U sqrt(M/32 + 40).  (Summed from dz
  rounded to 16 bits it would be off by 1.6e-3 in bf16 and 2e-4 in fp16: 42 and 5 times what is allowed at least.)
* fp32 dW against products of the oracle's dz rounded to 16 bits: the kernel's dz lands on the other side of a rounding border where
  it is off by more than the distance to it: a share of at most 2 E(K) / (2^-8 or 2^-11, the smallest step relative to the value)
  of them, each off by one step, at most 2 HALF; their errors are independent: 2 HALF sqrt(share) of the norm; the sum's own
  steps, 2U (M/16 + 400) at most.
* tails of act: silu HALF + 2^-18; gelu's erf polynomial (Abramowitz and Stegun 7.1.26) is off by 4.7e-4 of 1 - erf at g = -4
  and 3.7e-2 at g = -13 (computed in 64 bits from the polynomial), so 4e-2 over the whole range.
"""
import math

import pytest
import torch
from test_gpu_gated import ACTS, B16, F16, HALF, U, _act64, _check, _make, _oracle

pytestmark = pytest.mark.gpu
TYPES = pytest.mark.parametrize("t", [B16, F16], ids=["bf16", "fp16"])


def _dz_error(K):
    return 4 * U * (K / 16 + 18) + 2.0 ** -19


def _dz64(x, w, b, dh, act):
    F = w.shape[0] // 2
    z = x.double() @ w.double().T
    if b is not None:
        z = z + b.double()
    a, d = _act64(act, z[:, :F])
    return torch.cat([dh.double() * z[:, F:] * d, dh.double() * a], 1)


def _rel(got, want):
    return ((got.double() - want).norm() / want.norm()).item()


@TYPES
@pytest.mark.parametrize("M,K,F", [(20000, 128, 136), (8200, 130, 700), (10007, 264, 501), (30000, 100, 256), (4096, 1024, 512),
                                   (777, 2048, 300), (700, 2048, 301), (65000, 16, 24)])
def test_db_is_summed_before_the_rounding(M, K, F, t):
    import g1env
    act = ACTS[(M + K + F) % 4]
    x, w, b, dh = _make(M, K, F, t, True, seed=M + K + F)
    want = _dz64(x, w, b, dh, act).sum(0)
    db = g1env.gated_ff_backward_device(dh, x, w, b, act)[2]
    assert _rel(db, want) <= _dz_error(K) + 2 * U * math.sqrt(M / 32 + 40)
    # and so it is whatever else is asked for
    for need in ((False, False, True), (True, False, True), (False, True, True)):
        assert torch.equal(g1env.gated_ff_backward_device(dh, x, w, b, act, need)[2], db)


@TYPES
@pytest.mark.parametrize("K", [512, 1024, 2048])
def test_long_sums_keep_their_size(K, t):
    """The tensor cores truncate at each of K/16 steps, which makes sums smaller on the average: half a step of fp32 (0.36 of 2^-23 of
    the sum, its mantissa being anywhere in [1, 2)) of a sum that is half there on the average, 0.18 of 2^-23 a step at most.  Put
    back are 2^-26 a step; of what is left, 2^-27 a step is allowed.  One row, dh = 1, ELU and gates above 1/2, where act is
    g itself: db holds u, then g.  32768 numbers: the mean's own spread is below 2^-27."""
    import g1env
    F = 16384
    g = torch.Generator(device="cuda").manual_seed(K)
    x = torch.randn(1, K, device="cuda", generator=g).to(t)
    w = (torch.randn(2 * F, K, device="cuda", generator=g) / math.sqrt(K)).to(t)
    db = g1env.gated_ff_backward_device(torch.ones(1, F, device="cuda", dtype=t), x, w, None, "elu", (False, False, True))[2].double()
    z = x[0].double() @ w.double().T
    far = (z[:F] > 0.5).nonzero()[:, 0]
    want = torch.cat([z[F:][far], z[:F][far]])
    off = torch.cat([db[:F][far], db[F:][far]]) - want
    assert abs((off @ want / (want @ want)).item()) <= 2.0 ** -27 * K / 16


@TYPES
@pytest.mark.parametrize("M,K,F", [(300, 104, 1024), (5000, 40, 24), (10007, 264, 501), (4096, 1024, 512), (130, 60, 33), (64, 1024, 1024)])
def test_fp32_dw_is_not_rounded_again(M, K, F, t):
    import g1env
    act = ACTS[(M + F) % 4]
    x, w, b, dh = _make(M, K, F, t, True, seed=M + K)
    dw = g1env.gated_ff_backward_device(dh, x, w, b, act, (False, True, False), torch.float32)[1]
    want = _dz64(x, w, b, dh, act).to(t).double().T @ x.double()
    share = min(1.0, 2 * _dz_error(K) / (HALF[t]))
    assert _rel(dw, want) <= 2 * HALF[t] * math.sqrt(share) + 2 * U * (M / 16 + 400)
    # the lower half of its bits is in use: a number that the 16-bit type holds too comes up by chance only, 2^-13 at most
    assert (dw.to(t).float() == dw).float().mean().item() < 0.01


@TYPES
@pytest.mark.parametrize("scale", [1e-4, 1e3])
@pytest.mark.parametrize("act", ACTS)
def test_gradients_far_from_one(act, scale, t):
    """dh a little above fp16's smallest normal number, where terms of dX and dW round absolutely, and large ones."""
    import g1env
    x, w, b, dh = _make(40, 64, 56, t, True, seed=7, dh_scale=scale)
    h64, dx64, dw64, db64 = _oracle(x, w, b, dh, act)
    dx, dw, db = g1env.gated_ff_backward_device(dh, x, w, b, act)
    for name, got, want in (("dx", dx, dx64), ("dw", dw, dw64), ("db", db, db64)):
        _check(name, got, want)
    _check("dw32", g1env.gated_ff_backward_device(dh, x, w, b, act, (False, True, False), torch.float32)[1], dw64)


@pytest.mark.parametrize("rows", [1, 8])
def test_tails_keep_their_relative_size(rows):
    """silu and gelu of far negative gates, by the kernel for a few rows and by the tiles."""
    import g1env
    F = 2001
    for act, t, lo, hi, rel in (("silu", B16, -30, -5, 2.0 ** -18), ("silu", F16, -9, -5, 2.0 ** -18), ("gelu", B16, -12.9, -4, 4e-2)):
        x = torch.ones(rows, 1, device="cuda", dtype=t)
        w = torch.cat([torch.linspace(lo, hi, F, device="cuda"), torch.ones(F, device="cuda")])[:, None].to(t)
        got = g1env.gated_ff_device(x, w, None, act).double()
        want = _act64(act, w[:F, 0].double())[0].expand(rows, F)
        assert bool(((got - want).abs() <= (HALF[t] + rel) * want.abs()).all()), (act, t)


@TYPES
@pytest.mark.parametrize("rows", [2, 6])
@pytest.mark.parametrize("act", ACTS)
def test_infinite_and_nan_gates(act, rows, t):
    """h of gates that are +-inf or NaN is what the formula gives, and the gates beside them are what they were."""
    import g1env
    inf = float("inf")
    gates = [1.0, inf, 0.5, -inf, -2.0, float("nan"), 3.0]
    F = len(gates)
    w = torch.cat([torch.tensor(gates), torch.full((F,), 0.75)])[:, None].to(t).cuda()
    x = torch.ones(rows, 1, device="cuda", dtype=t)
    h = g1env.gated_ff_device(x, w, None, act).float().cpu()
    for r in range(rows):
        assert h[r, 1].item() == (0.75 if act == "tanh" else inf)
        # -inf times 0 in silu and gelu, as torch has it
        assert h[r, 3].item() == -0.75 if act in ("tanh", "elu") else math.isnan(h[r, 3].item())
        assert math.isnan(h[r, 5].item())
    keep = [0, 2, 4, 6]
    plain = g1env.gated_ff_device(x, torch.cat([w[keep], w[[F + i for i in keep]]]), None, act).float().cpu()
    assert torch.equal(h[:, keep], plain)


@pytest.mark.parametrize("act", ["tanh", "elu", "gelu"])
@pytest.mark.parametrize("F", [40, 41])
def test_rows_of_nan_and_infinity_stay_by_themselves(act, F):
    import g1env
    x, w, b, dh = _make(300, 72, F, B16, True, seed=9)
    y = x.clone()
    y[5], y[200] = float("nan"), float("inf")
    keep = torch.ones(300, dtype=torch.bool, device="cuda")
    keep[5] = keep[200] = False
    h, dx = g1env.gated_ff_device(x, w, b, act), g1env.gated_ff_backward_device(dh, x, w, b, act)[0]
    h2, dx2 = g1env.gated_ff_device(y, w, b, act), g1env.gated_ff_backward_device(dh, y, w, b, act)[0]
    assert torch.equal(h[keep], h2[keep]) and torch.equal(dx[keep], dx2[keep])
    assert bool(torch.isnan(h2[5]).all()) and not bool(torch.isfinite(dx2[5]).any())
