"""Launches that follow one another without a wait between: each reads what the one before it has just written, from
addresses that earlier ones have been read at.  The same bits as with the device waited for after every call."""
import pytest
import torch

pytestmark = pytest.mark.gpu
B16 = torch.bfloat16


def _randn(seed, *s):
    return torch.randn(*s, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))


@pytest.mark.parametrize("M", [1, 2, 3, 4, 5, 40, 300])
@pytest.mark.parametrize("K", [64, 50])
def test_layers_read_what_the_last_one_wrote(M, K):
    """A hundred layers between two buffers, on the rows that the one before has written."""
    import g1env
    ws = [(_randn(i, 2 * K, K) * (0.7 / K ** 0.5)).to(B16) for i in range(4)]
    bs = [_randn(10 + i, 2 * K) for i in range(4)]
    lib = g1env.load_library()
    outs = []
    for wait in (True, False):
        bufs = [_randn(20, M, K).to(B16), torch.zeros(M, K, device="cuda", dtype=B16)]
        n = [lib.g1_gated_ff_workspace(M, K, K, bufs[i].data_ptr(), K, ws[0].data_ptr(), K, 0) for i in range(2)]
        space = torch.empty(max(n) + 256, dtype=torch.uint8, device="cuda")
        stream = torch.cuda.current_stream().cuda_stream
        torch.cuda.synchronize()
        for i in range(100):
            a, b = bufs[i % 2], bufs[1 - i % 2]
            assert lib.g1_gated_ff(M, K, K, 1, 0, a.data_ptr(), K, ws[i % 4].data_ptr(), K, bs[i % 4].data_ptr(), b.data_ptr(),
                                   space.data_ptr(), max(n), stream) == 0
            if wait:
                torch.cuda.synchronize()
        torch.cuda.synchronize()
        outs.append([t.clone() for t in bufs])
    assert all(torch.equal(p, q) for p, q in zip(*outs)) and bool(torch.isfinite(outs[0][0]).all())


@pytest.mark.parametrize("M", [1, 3, 4, 40])
def test_weights_and_biases_that_the_last_call_wrote(M):
    """The gradients of a call are the next one's weights and bias (both written by launches of the same kind)."""
    import g1env
    K = F = 96
    x, dh = _randn(1, M, K).to(B16), _randn(2, M, F).to(B16)
    outs = []
    for wait in (True, False):
        w, b, got = (_randn(3, 2 * F, K) / K ** 0.5).to(B16), _randn(4, 2 * F), []
        for _ in range(30):
            _, w, b = g1env.gated_ff_backward_device(dh, x, w, b, "tanh", (False, True, True))
            if wait:
                torch.cuda.synchronize()
            got.append(g1env.gated_ff_device(x, w, b, "tanh"))
            if wait:
                torch.cuda.synchronize()
            w, b = (w.float() / w.float().norm() * 14).to(B16), b / b.norm()
        outs.append(got)
    assert all(torch.equal(p, q) for p, q in zip(*outs))


def test_optimiser_reads_what_the_last_launch_wrote():
    """The gradients that a backward pass is still writing, its bias's among them, clipped and stepped on at once."""
    import g1env
    for M, K, F in ((40, 64, 48), (3000, 256, 320)):
        x, dh = _randn(1, M, K).to(B16), _randn(2, M, F).to(B16)
        outs = []
        for wait in (True, False):
            w, b = torch.nn.Parameter(_randn(3, 2 * F, K) / K ** 0.5), torch.nn.Parameter(_randn(4, 2 * F))
            opt = g1env.ClipAdam([w, b], lr=1e-2, max_norm=0.5)
            norms = []
            for _ in range(20):
                _, dw, db = g1env.gated_ff_backward_device(dh, x, w.detach().to(B16), b.detach(), dw_dtype=torch.float32)
                if wait:
                    torch.cuda.synchronize()
                norms.append(opt.step([dw, db]))
                if wait:
                    torch.cuda.synchronize()
                norms.append(g1env.clip_grad_norm_device([dw, db], 0.1))
            outs.append([w.detach(), b.detach(), dw, db] + norms)
        assert all(torch.equal(p, q) for p, q in zip(*outs))
