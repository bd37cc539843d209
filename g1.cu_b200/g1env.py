"""Python host side of the B200 G1 rollout: the ctypes binding of libg1env.so plus the
trainer-facing classes, under the names the reference's scripts use
(scripts/ppo.py:24-125: the ctypes binding, G1Env, RunNorm, AC, evaluate;
scripts/ppo_fused.py:27-44: the g1_rollout binding and pack_weights).

The CUDA library is required: importing works on a CPU-only machine, but creating an env
or calling a kernel entry point raises if libg1env.so is missing or no GPU is visible --
there is no CPU fallback.
"""
import contextlib
import ctypes
import os
from array import array

import numpy as np
import torch
import torch.nn as nn

HERE = os.path.dirname(os.path.abspath(__file__))
LIB = os.path.join(HERE, "libg1env.so")
OBS_DIM, ACT_DIM, NQ, NV = 100, 29, 36, 35

_fp = ctypes.POINTER(ctypes.c_float)
_vp = ctypes.c_void_p
_lib = None

# exported symbols and their ctypes signatures (include/g1env.h)
SIGNATURES = {
    "g1_env_create": (_vp, [ctypes.c_int, ctypes.c_int, ctypes.c_int, ctypes.c_ulong]),
    "g1_env_create_ex": (_vp, [ctypes.c_int, ctypes.c_int, ctypes.c_int, ctypes.c_ulong, ctypes.c_int, ctypes.c_uint,
                               ctypes.c_float]),
    "g1_env_destroy": (None, [_vp]),
    "g1_env_reset": (None, [_vp, _fp]),
    "g1_env_step": (None, [_vp, _fp, _fp, _fp, _fp]),
    "g1_env_step_device": (None, [_vp] + [_vp] * 4),
    "g1_rollout": (None, [_vp, ctypes.c_int] + [_vp] * 10),
    "g1_rollout_noalloc": (None, [_vp, ctypes.c_int] + [_vp] * 10),
    "g1_env_bench_phys": (None, [_vp, ctypes.c_int]),
    "g1_env_phys_async": (None, [_vp, ctypes.c_int]),
    "g1_env_phys_actions": (None, [_vp, ctypes.c_int, _vp]),
    "g1_env_qpos": (None, [_vp, _fp]),
    "g1_env_qpos_all": (None, [_vp, _fp]),
    "g1_env_obs_dim": (ctypes.c_int, []),
    "g1_env_act_dim": (ctypes.c_int, []),
    "g1_occupancy_report": (None, []),
    "g1_env_last_error": (ctypes.c_char_p, []),
    "g1_env_last_error_code": (ctypes.c_int, []),
    "g1_env_clear_error": (None, []),
    "g1_env_set_stream": (None, [_vp, _vp]),
    "g1_env_set_policy": (ctypes.c_int, [_vp, ctypes.c_int, _vp, ctypes.c_int]),
    "g1_env_set_friction": (None, [_vp, ctypes.c_float]),
    "g1_env_set_policy_ex": (ctypes.c_int, [_vp, ctypes.c_int, _vp, ctypes.c_int, ctypes.c_int]),
    "g1_env_tc_status": (ctypes.c_int, [_vp]),
    "g1_env_weight_count": (ctypes.c_longlong, [_vp]),
    "g1_env_set_value_net": (ctypes.c_int, [_vp, ctypes.c_int, _vp]),
    "g1_env_get_state": (None, [_vp, _vp, _vp, _vp, _vp, _vp]),
    "g1_env_set_state": (None, [_vp, _vp, _vp, _vp, _vp, ctypes.c_ulonglong]),
    "g1_env_ncon_hist": (None, [_vp, ctypes.c_int, _vp]),
    "g1_gemm_bf16_tc": (ctypes.c_int, [ctypes.c_int, ctypes.c_int, ctypes.c_int, _vp, ctypes.c_int, _vp, _vp, ctypes.c_int,
                                       _vp]),
    "g1_dense_bf16x3": (ctypes.c_int, [ctypes.c_int] * 3 + [_vp] * 3 + [ctypes.c_int, _vp]),
    "g1_gae": (ctypes.c_int, [ctypes.c_int, ctypes.c_int] + [_vp] * 4 + [ctypes.c_double, ctypes.c_double] + [_vp] * 4),
    "g1_obs_prep": (ctypes.c_int, [ctypes.c_longlong, ctypes.c_int] + [_vp] * 6),
    "g1_adv_normalize": (ctypes.c_int, [ctypes.c_longlong, _vp, _vp, _vp]),
    "g1_runnorm_update": (ctypes.c_int, [ctypes.c_int, _vp, _vp, ctypes.c_double, _vp, _vp]),
    "g1_gated_ff_workspace": (ctypes.c_longlong, [ctypes.c_int] * 3 + [_vp, ctypes.c_longlong, _vp, ctypes.c_longlong,
                                                                     ctypes.c_int]),
    "g1_gated_ff": (ctypes.c_int, [ctypes.c_int] * 5 + [_vp, ctypes.c_longlong] * 2 + [_vp] * 3 + [ctypes.c_longlong, _vp]),
    "g1_gated_ff_backward": (ctypes.c_int, [ctypes.c_int] * 5 + [_vp] + [_vp, ctypes.c_longlong] * 2 + [_vp] * 3
                             + [ctypes.c_int, _vp, _vp, ctypes.c_longlong, _vp]),
    "g1_gated_ff_status": (ctypes.c_int, []),
    "g1_opt_workspace": (ctypes.c_longlong, [ctypes.c_int]),
    "g1_clip_grad_norm": (ctypes.c_int, [ctypes.c_int, _vp, _vp, _vp, ctypes.c_double, _vp, _vp, ctypes.c_longlong, _vp]),
    "g1_clip_adam": (ctypes.c_int, [ctypes.c_int] + [_vp] * 7 + [ctypes.c_double, ctypes.c_double, _vp]
                     + [ctypes.c_double] * 4 + [_vp, _vp, ctypes.c_longlong, _vp]),
    "g1_qacc_batch": (ctypes.c_int, [ctypes.c_int] + [_vp] * 4 + [ctypes.c_int, ctypes.c_float] + [_vp] * 5),
}


class G1Error(RuntimeError):
    pass


def load_library(path=LIB):
    """Load libg1env.so and bind every exported symbol (raises if it is missing)."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(path):
        raise G1Error(f"{path} not built: run `python g1.cu_b200/build.py` (nvcc, sm_100a); "
                      "there is no CPU fallback")
    lib = ctypes.CDLL(path)
    for name, (res, args) in SIGNATURES.items():
        f = getattr(lib, name)
        f.restype = res
        f.argtypes = args
    _lib = lib
    return lib


def _check():
    code = _lib.g1_env_last_error_code()
    if code:
        msg = _lib.g1_env_last_error()
        _lib.g1_env_clear_error()
        raise G1Error(f"libg1env: {msg.decode() if msg else code}")


def _p(a):
    return a.ctypes.data_as(_fp)


def _dp(t):
    """device (or host numpy) pointer as c_void_p (ppo_fused.py:31-32)"""
    if t is None:
        return None
    if isinstance(t, np.ndarray):
        return t.ctypes.data_as(_vp)
    return ctypes.c_void_p(t.data_ptr())


def _require_gpu():
    if not torch.cuda.is_available():
        raise G1Error("no CUDA device visible: the G1 rollout runs only on the GPU (no CPU fallback)")


class G1Env:
    """Batched G1 env on one GPU (ppo.py:39-60).  All N worlds stay resident on the device."""

    def __init__(self, n_worlds, substeps=10, pgs_iters=2000, seed=0, device=None, world0=0, mu=0.6):
        _require_gpu()
        lib = load_library()
        self.N = n_worlds
        self.obs_dim = lib.g1_env_obs_dim()
        self.act_dim = lib.g1_env_act_dim()
        dev = torch.cuda.current_device() if device is None else int(device)
        self.device = dev
        self.h = lib.g1_env_create_ex(n_worlds, substeps, pgs_iters, seed, dev, world0, mu)
        if not self.h:
            _check()
            raise G1Error("g1_env_create failed")
        self._obs = np.zeros((n_worlds, self.obs_dim), np.float32)
        self._rew = np.zeros(n_worlds, np.float32)
        self._done = np.zeros(n_worlds, np.float32)

    def reset(self):
        _lib.g1_env_reset(self.h, _p(self._obs)); _check()
        return self._obs.copy()

    def step(self, act):
        act = np.ascontiguousarray(act, np.float32)
        _lib.g1_env_step(self.h, _p(act), _p(self._obs), _p(self._rew), _p(self._done)); _check()
        return self._obs.copy(), self._rew.copy(), self._done.copy()

    def step_device(self, act, obs, rew, done):
        """g1_env_step_device: one control step on CUDA tensors (act [N, 29] -> obs [N, 100],
        rew [N], done [N]), asynchronous on the env's stream."""
        _lib.g1_env_step_device(self.h, _dp(act), _dp(obs), _dp(rew), _dp(done)); _check()

    def set_stream(self, stream):
        _lib.g1_env_set_stream(self.h, ctypes.c_void_p(stream.cuda_stream if stream is not None else 0))

    def set_policy(self, hidden=(256, 256), activation="tanh", precision="fp32"):
        """precision "fp32": the in-kernel fp32-accurate policy (split-bf16 on the tensor cores when
        every hidden width is a multiple of 16 up to 256, else FFMA); "fp32-ffma": always FFMA;
        "bf16": tensor-core policy for wide MLPs; with activation "swiglu" or "geglu"
        of gated layers (AC of the same activation)."""
        hid = np.ascontiguousarray(hidden, np.int32)
        code = {"fp32": 0, "bf16": 1, "fp32-ffma": 2}[precision]
        act = {"tanh": 0, "swiglu": 2, "geglu": 3}.get(activation, 1)
        rc = _lib.g1_env_set_policy_ex(self.h, len(hidden), _dp(hid), act, code)
        if rc:
            _check()

    def tc_status(self):
        """Nonzero if a wait of this env's tensor-core policy ran out since the last call (waits for the env's stream; clears)."""
        return _lib.g1_env_tc_status(self.h)

    def set_value_net(self, hidden=()):
        """Separate value network for the bf16 tensor-core policy path;
        () returns to the shared trunk's value head."""
        hid = np.ascontiguousarray(hidden if len(hidden) else [0], np.int32)
        if _lib.g1_env_set_value_net(self.h, len(hidden), _dp(hid)):
            _check()

    def set_friction(self, mu):
        _lib.g1_env_set_friction(self.h, float(mu))

    def _weights(self, W):
        """W's address, once it is known to hold all that the env's policy reads (a gated layer's weights are twice a plain
        one's)."""
        need = _lib.g1_env_weight_count(self.h)
        if not W.is_cuda or W.dtype != torch.float32 or not W.is_contiguous():
            raise G1Error("packed weights must be a contiguous fp32 CUDA tensor")
        if W.numel() < need:
            raise G1Error(f"packed weights hold {W.numel()} numbers, the env's policy has {need} (set_policy, set_value_net)")
        return _dp(W)

    def rollout(self, H, W, mean, var, O, A, LP, V, R, D, Vlast):
        """g1_rollout on torch-owned device tensors (ppo_fused.py:101-102)."""
        _lib.g1_rollout(self.h, H, self._weights(W), _dp(mean), _dp(var), _dp(O), _dp(A), _dp(LP), _dp(V), _dp(R), _dp(D),
                        _dp(Vlast))
        _check()

    def rollout_noalloc(self, H, W, mean, var, O, A, LP, V, R, D, Vlast):
        """g1_rollout_noalloc: the same rollout without any device allocation (weights repacked
        into the library's fixed device area)."""
        _lib.g1_rollout_noalloc(self.h, H, _dp(W), _dp(mean), _dp(var), _dp(O), _dp(A), _dp(LP), _dp(V), _dp(R),
                                _dp(D), _dp(Vlast))
        _check()

    def bench_phys(self, K):
        _lib.g1_env_bench_phys(self.h, K); _check()

    def phys_async(self, K):
        _lib.g1_env_phys_async(self.h, K); _check()

    def phys_actions(self, K, act=None):
        """g1_env_phys_actions: K control steps of physics with a constant action per world
        (act: CUDA tensor [N, 29], None = zero), asynchronous."""
        _lib.g1_env_phys_actions(self.h, K, _dp(act.contiguous() if act is not None else None)); _check()

    def get_state(self):
        N = self.N
        qp = np.zeros((N, NQ), np.float32); qv = np.zeros((N, NV), np.float32); pa = np.zeros((N, ACT_DIM), np.float32)
        st = np.zeros(N, np.int32); tick = np.zeros(1, np.uint64)
        _lib.g1_env_get_state(self.h, _dp(qp), _dp(qv), _dp(pa), _dp(st), _dp(tick)); _check()
        return qp, qv, pa, st, int(tick[0])

    def set_state(self, qp, qv, pa, steps, tick=0):
        N = self.N
        a = [np.ascontiguousarray(qp, np.float32).reshape(N, NQ), np.ascontiguousarray(qv, np.float32).reshape(N, NV),
             np.ascontiguousarray(pa, np.float32).reshape(N, ACT_DIM), np.ascontiguousarray(steps, np.int32).reshape(N)]
        _lib.g1_env_set_state(self.h, *[_dp(x) for x in a], int(tick)); _check()

    def qpos(self):
        out = np.zeros(NQ, np.float32)
        _lib.g1_env_qpos(self.h, _p(out)); _check()
        return out

    def qpos_all(self):
        out = np.zeros((self.N, NQ), np.float32)
        _lib.g1_env_qpos_all(self.h, _p(out)); _check()
        return out

    def ncon_hist(self, enable=True):
        out = np.zeros(9, np.uint64)
        _lib.g1_env_ncon_hist(self.h, 1 if enable else 0, _dp(out)); _check()
        return out

    def close(self):
        if getattr(self, "h", None):
            _lib.g1_env_destroy(self.h)
            self.h = None


def qacc_batch(qpos, qvel, tau=None, bdt=None, pgs_iters=8, mu=0.6):
    """Per-state FK + generalized acceleration on the GPU (g1_qacc_batch).  Takes CUDA
    tensors; returns dict of CUDA tensors qacc, qacc_smooth, bias [n,35], f [n,32], ncon [n]."""
    _require_gpu()
    lib = load_library()
    n = qpos.shape[0]
    dev = qpos.device
    f32 = dict(dtype=torch.float32, device=dev)
    out = dict(qacc=torch.zeros(n, NV, **f32), qacc_smooth=torch.zeros(n, NV, **f32), bias=torch.zeros(n, NV, **f32),
               f=torch.zeros(n, 32, **f32), ncon=torch.zeros(n, dtype=torch.int32, device=dev))
    qpos = qpos.contiguous().float(); qvel = qvel.contiguous().float()
    tau = None if tau is None else tau.contiguous().float()
    bdt = None if bdt is None else bdt.expand(n, NV).contiguous().float()
    rc = lib.g1_qacc_batch(n, _dp(qpos), _dp(qvel), _dp(tau), _dp(bdt), pgs_iters, float(mu),
                           *[_dp(out[k]) for k in ("qacc", "qacc_smooth", "bias", "f", "ncon")])
    if rc:
        _check()
    return out


def gemm_bf16_tc(X, W, bias=None, act=-1):
    """out = act(X W^T + b) on the tensor cores (tcgen05).  X [M,K], W [N,K] bf16 CUDA tensors."""
    _require_gpu()
    lib = load_library()
    M, K = X.shape
    N = W.shape[0]
    out = torch.empty(M, N, dtype=torch.float32, device=X.device)
    X = X.contiguous(); W = W.contiguous()
    b = None if bias is None else bias.float().contiguous()
    rc = lib.g1_gemm_bf16_tc(M, N, K, _dp(X), K, _dp(W), _dp(b), act, _dp(out))
    if rc:
        _check()
    return out


def dense_bf16x3(X, W, bias=None, act=-1):
    """out = act(X W^T + b) with the rollout kernel's split-bf16 tensor-core layer (rows <= 64)."""
    _require_gpu()
    lib = load_library()
    X = X.float().contiguous(); W = W.float().contiguous()
    rows, K = X.shape
    N = W.shape[0]
    out = torch.empty(rows, N, dtype=torch.float32, device=X.device)
    b = None if bias is None else bias.float().contiguous()
    if lib.g1_dense_bf16x3(rows, K, N, _dp(X), _dp(W), _dp(b), act, _dp(out)):
        _check()
    return out


# ---------------- gated layers ----------------
_ACT = {"tanh": 0, "elu": 1, "silu": 2, "gelu": 3}
_FF_TYPE = {torch.bfloat16: 1, torch.float16: 2}
_FF_ROWS = 4  # rows up to which the forward pass makes no copies (g1_gated.cuh ROWS_MAX)


_HERE = contextlib.nullcontext()


def _on(dev):
    """Makes `dev` the current device for the calls within."""
    return _HERE if torch.cuda.current_device() == dev.index else torch.cuda.device(dev)


def _stream_of(dev):
    """torch's current stream on `dev`, as the number that the C-ABI takes"""
    return torch._C._cuda_getCurrentRawStream(dev.index)


def _rows(t):
    """The last axis as the columns of a matrix whose rows do not overlap; a copy only where there is no such view."""
    m = t if t.dim() == 2 else t.reshape(-1, t.shape[-1])
    if m.is_contiguous():
        return m
    if (m.stride(1) != 1 and m.shape[1] > 1) or (m.shape[0] > 1 and m.stride(0) < m.shape[1]):
        return m.contiguous()
    return m


def _ff_args(x, w, b, act):
    """Checked operands of a gated layer: rows [M, K] of x, w [2F, K] in x's type, b [2F] fp32 or None, F, and the codes of
    type and activation."""
    if not x.is_cuda:
        raise G1Error("a gated layer takes CUDA tensors (no CPU fallback)")
    t, code, shape = _FF_TYPE.get(x.dtype), _ACT.get(act), w.shape
    if t is None:
        raise G1Error(f"a gated layer takes bf16 or fp16 rows, not {str(x.dtype)[6:]}")
    if w.dtype != x.dtype:
        raise G1Error("the weights must be of the rows' type")
    if code is None:
        raise G1Error(f"unknown activation {act!r} (one of {', '.join(_ACT)})")
    if len(shape) != 2 or shape[0] % 2 or not shape[0] or not shape[1] or not x.dim() or x.shape[-1] != shape[1]:
        raise G1Error("a gated layer takes x [..., K] and w [2F, K]")
    where = x.get_device()
    if w.get_device() != where or (b is not None and b.get_device() != where):
        raise G1Error("a gated layer's tensors must be on one device")
    if b is not None:
        if b.shape != shape[:1] or not b.is_floating_point():
            raise G1Error("the bias must be [2F]")
        if b.dtype != torch.float32:
            b = b.float()
        b = b.contiguous()
    return _rows(x), _rows(w), b, shape[0] // 2, t, code


def _ff_operands(x, w):
    """(M, K, address and row stride of x, of w)"""
    M, K = x.shape
    if M > 1 << 30:
        raise G1Error("too many rows")
    return M, K, x.data_ptr(), x.stride(0) if M > 1 else (K + 7) & ~7, w.data_ptr(), w.stride(0)


def _bytes(x, n):
    """A workspace of n bytes beside x (16-bit numbers)"""
    return x.new_empty((n + 1) // 2) if n else None


def _ff_forward(lib, dev, x, x2, w, b, F, t, code):
    """h, and where rows are not aligned the workspace with their copies and how many bytes of it are x's and w's."""
    M, K, px, ldx, pw, ldw = _ff_operands(x2, w)
    nx = nw = n = 0
    ws = None
    if M > _FF_ROWS and ((px | pw) & 15 or (ldx | ldw) & 7):
        k8 = (K + 7) & ~7
        nx = (M * k8 * 2 + 255) & ~255 if px & 15 or ldx & 7 else 0
        nw = (F * k8 * 4 + 255) & ~255 if pw & 15 or ldw & 7 else 0
        n = nx + nw
        ws = _bytes(x, n)
    h = x.new_empty(x.shape[:-1] + (F,))
    if lib.g1_gated_ff(M, K, F, t, code, px, ldx, pw, ldw, _addr(b), h.data_ptr(), _addr(ws), n, _stream_of(dev)):
        _check()
    return h, ws, nx, nw


def _ff_backward(lib, dev, dh, x, shape, b, F, t, code, operands, need, dw_dtype):
    M, K, px, ldx, pw, ldw = operands
    n = lib.g1_gated_ff_workspace(M, K, F, px, ldx, pw, ldw, 1)
    ws = _bytes(x, n)
    dh = dh.contiguous()
    dx = x.new_empty(shape) if need[0] else None
    dw = x.new_empty((2 * F, K), dtype=dw_dtype) if need[1] else None
    db = x.new_empty(2 * F, dtype=torch.float32) if need[2] else None
    if lib.g1_gated_ff_backward(M, K, F, t, code, dh.data_ptr(), px, ldx, pw, ldw, _addr(b), _addr(dx), _addr(dw),
                                _FF_TYPE.get(dw_dtype, 0), _addr(db), _addr(ws), n, _stream_of(dev)):
        _check()
    return dx, dw, db


def _addr(t):
    return None if t is None else t.data_ptr()


def gated_ff_device(x, w, b=None, act="silu"):
    """One gated layer, h = act(x Wg^T + bg) * (x Wu^T + bu) (g1_gated_ff): x [..., K] bf16 or fp16, w [2F, K] of the
    same type (the F gate rows, then the F up rows), b [2F] or None, act "tanh", "elu", "silu" or "gelu" (erf).
    Returns h [..., F] in x's type, on torch's current stream.  Rows may be strided; rows or weights that do
    not start on 16-byte boundaries (a row stride that is no multiple of 8) are copied first."""
    lib = load_library()
    x2, w, b, F, t, code = _ff_args(x, w, b, act)
    dev = x2.device
    with _on(dev):
        return _ff_forward(lib, dev, x, x2, w, b, F, t, code)[0]


def gated_ff_backward_device(dh, x, w, b=None, act="silu", need=(True, True, True), dw_dtype=None):
    """The gradients of gated_ff_device for dh [..., F] (g1_gated_ff_backward): dx like x, dw [2F, K] (dw_dtype: x's type
    or fp32), db [2F] fp32; None where `need` (dx, dw, db) says so.  Nothing of the forward pass but its inputs
    is needed.  dg and du are rounded to x's type before the products with W and x, but not in db: dx and dw, an fp32 dw
    too, carry that rounding of their terms (1.7e-3 of the norm in bf16, 2.1e-4 in fp16).  In fp16 dg and du overflow above
    65504 and lose digits below 6e-5: scale the loss so that dh lies between."""
    lib = load_library()
    x2, w, b, F, t, code = _ff_args(x, w, b, act)
    dev = x2.device
    if dw_dtype is None:
        dw_dtype = x.dtype
    elif dw_dtype not in (x.dtype, torch.float32):
        raise G1Error("dw is fp32 or of the rows' type")
    if dh.device != dev or dh.dtype != x.dtype or dh.shape != x.shape[:-1] + (F,):
        raise G1Error("dh must be [..., F] on x's device and of its type")
    with _on(dev):
        return _ff_backward(lib, dev, dh, x, x.shape, b, F, t, code, _ff_operands(x2, w), need, dw_dtype)


def gated_ff_status(device=None):
    """Nonzero if a wait inside a gated layer's kernels ran out on `device` (default: the current one) since the last call, in
    whatever call but an env's rollout (env.tc_status says that); what they wrote is then garbage.  Waits for all work of
    the device, so not while a graph is captured; clears."""
    lib = load_library()
    with torch.cuda.device(device):
        return lib.g1_gated_ff_status()


def _vector(t, n, dtype, at):
    return t is None or (t.shape == (n,) and t.dtype == dtype and t.device == at)


class _GatedFF(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, b, act):
        lib = load_library()
        w16 = w if w.dtype == x.dtype else w.to(x.dtype)
        x2, w2, b2, F, t, code = _ff_args(x, w16, b, act)
        dev = x2.device
        with _on(dev):
            h, ws, nx, nw = _ff_forward(lib, dev, x, x2, w2, b2, F, t, code)
        ctx.save_for_backward(x2, w2, b2, ws)
        ctx.call = (lib, dev, F, t, code, nx, nw, x.shape, w.dtype, None if b is None else b.dtype, x2.shape, w2.shape)
        return h

    @staticmethod
    def backward(ctx, dh):
        # once_differentiable costs 6 us a call; only a backward pass that is itself recorded needs it
        return _gated_ff_once(ctx, dh) if torch.is_grad_enabled() else _gated_ff_back(ctx, dh)


def _gated_ff_back(ctx, dh):
    # notices a change made since; a hook may have put other tensors in their place
    x2, w2, b2, ws = ctx.saved_tensors
    lib, dev, F, t, code, nx, nw, shape, w_dtype, b_dtype, rows, cols = ctx.call
    at, kind = dh.device, dh.dtype  # as the layer's rows had
    if (x2.shape != rows or w2.shape != cols or x2.dtype != kind or w2.dtype != kind or x2.device != at or w2.device != at
            or not _vector(b2, 2 * F, torch.float32, at) or not _vector(ws, (nx + nw) // 2, kind, at)):
        raise G1Error("a hook brought a gated layer's saved tensors back with another shape or type, or on another device")
    x2, w2 = _rows(x2), _rows(w2)
    if b2 is not None and not b2.is_contiguous():
        b2 = b2.contiguous()
    operands = _ff_operands(x2, w2)
    if ws is not None:  # the forward pass's copies of unaligned rows
        ws = ws.contiguous()
        M, K, px, ldx, pw, ldw = operands
        at, k8 = ws.data_ptr(), (K + 7) & ~7
        operands = (M, K, at if nx else px, k8 if nx else ldx, at + nx if nw else pw, k8 if nw else ldw)
    with _on(dev):
        dx, dw, db = _ff_backward(lib, dev, dh, x2, shape, b2, F, t, code, operands, ctx.needs_input_grad, w_dtype)
    return dx, dw, db if db is None or b_dtype == torch.float32 else db.to(b_dtype), None


_gated_ff_once = torch.autograd.function.once_differentiable(_gated_ff_back)


def gated_ff(x, w, b=None, act="silu"):
    """gated_ff_device with gradients.  w may be fp32 beside 16-bit rows: it is rounded to their type for the
    products, and its gradient comes back in fp32, summed from terms that are rounded to x's type
    (gated_ff_backward_device).  The forward pass keeps only its inputs as the products take them (w
    rounded; copies of those whose rows are not on 16-byte boundaries), as saved tensors that hooks and checkpoints see.
    In a captured backward pass the graphs of eager passes over the same leaves have to be gone first, as for any torch
    operator; gated_ff_backward_device has no such tie."""
    if w.dtype not in (x.dtype, torch.float32):
        raise G1Error("the weights must be fp32 or of the rows' type")
    return _GatedFF.apply(x, w, b, act)


class GatedLinear(nn.Module):
    """A gated layer with fp32 parameters, weight [2F, K] (gate rows, then up rows) and bias [2F], on rows that are taken
    to `dtype`.  Initialised as nn.Linear(K, 2F).  The weight's gradient is fp32 with terms rounded to `dtype` (gated_ff); with
    torch.float16 the loss wants a scale."""

    def __init__(self, in_features, out_features, act="silu", bias=True, dtype=torch.bfloat16):
        super().__init__()
        lin = nn.Linear(in_features, 2 * out_features, bias=bias)
        self.weight, self.bias = lin.weight, lin.bias
        self.in_features, self.out_features, self.act, self.dtype = in_features, out_features, act, dtype

    def forward(self, x):
        return gated_ff(x.to(self.dtype), self.weight, self.bias, self.act)

    def extra_repr(self):
        return f"{self.in_features}, {self.out_features}, act={self.act}"


# ---------------- trainer batch preparation (ppo_fused.py:104-119, ppo.py:71-79) ----------------
def _stream():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def gae_device(R, V, D, Vlast, gamma=0.99, lam=0.95):
    """adv, ret [H,N] and the fp64 advantage moments [count, sum, sumsq] (g1_gae), on torch's
    current stream.  adv/ret are bit-identical to the reference's torch GAE loop."""
    _require_gpu()
    lib = load_library()
    H, N = R.shape
    adv, ret = torch.empty_like(R), torch.empty_like(R)
    mom = torch.empty(3, dtype=torch.float64, device=R.device)
    Rc, Vc, Dc, Lc = (t.contiguous() for t in (R, V, D, Vlast))
    if lib.g1_gae(H, N, _dp(Rc), _dp(Vc), _dp(Dc), _dp(Lc), gamma, lam, _dp(adv), _dp(ret), _dp(mom), _stream()):
        _check()
    return adv, ret, mom


def obs_prep_device(O, fmean, fvar):
    """nobs = clamp((O - fmean)/sqrt(fvar + 1e-8), -10, 10) and the fp64 raw-observation
    moments [rows, sum[dim], sumsq[dim]] in one pass (g1_obs_prep)."""
    _require_gpu()
    lib = load_library()
    dim = O.shape[-1]
    Oc = O.contiguous()
    rows = Oc.numel() // dim
    nobs = torch.empty_like(Oc)
    mom = torch.empty(1 + 2 * dim, dtype=torch.float64, device=O.device)
    fm, fv = fmean.float().contiguous(), fvar.float().contiguous()
    if lib.g1_obs_prep(rows, dim, _dp(Oc), _dp(fm), _dp(fv), _dp(nobs), _dp(mom), _stream()):
        _check()
    return nobs, mom


def adv_normalize_device(adv, adv_mom):
    """In place: adv = (adv - mean)/(std + 1e-8) from (possibly all-reduced) moments."""
    lib = load_library()
    assert adv.is_contiguous()
    if lib.g1_adv_normalize(adv.numel(), _dp(adv), _dp(adv_mom), _stream()):
        _check()
    return adv


def runnorm_update_device(norm, obs_mom, rows_total):
    """RunNorm.update (ppo.py:71-79) on the device from (possibly all-reduced) moments;
    rows_total = obs_mom[0], known on the host so nothing synchronises."""
    lib = load_library()
    assert norm.mean.is_contiguous() and norm.var.is_contiguous()
    if lib.g1_runnorm_update(norm.mean.numel(), _dp(norm.mean), _dp(norm.var), float(norm.count), _dp(obs_mom),
                             _stream()):
        _check()
    norm.count = norm.count + rows_total


# ---------------- gradient norm, clipping and the clipped Adam step ----------------
_GRAD_TYPE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _dense(t):
    """Whether t fills its memory without gaps, in whatever order of its axes."""
    if t.is_contiguous():
        return True
    order = sorted(range(t.dim()), key=t.stride, reverse=True)
    return t.permute(order).is_contiguous()


_T = torch.Tensor


def _cuda_list(tensors, what, types):
    """Checks a list of dense CUDA tensors of those types on one device; their device (None for an empty list) and types."""
    where = set(map(_T.get_device, tensors))
    if -1 in where:
        raise G1Error(f"{what} must be CUDA tensors")
    if len(where) > 1:
        raise G1Error(f"{what} must be on one device")
    kinds = {t.dtype for t in tensors}
    for t in kinds:
        if t not in types:
            raise G1Error(f"{what} must be {' / '.join(str(x)[6:] for x in types)}, not {str(t)[6:]}")
    if not all(map(_T.is_contiguous, tensors)) and not all(map(_dense, tensors)):
        raise G1Error(f"{what} must fill their memory without gaps (use .contiguous())")
    return (tensors[0].device if tensors else None), kinds


def _ptrs(tensors):
    return array("Q", map(_T.data_ptr, tensors))


def _types(grads, kinds):
    if len(kinds) == 1:
        return array("i", [_GRAD_TYPE[t] for t in kinds]) * len(grads)
    return array("i", [_GRAD_TYPE[g.dtype] for g in grads])


def _at(a):
    """where an array's values lie: NULL for an empty one; the array has to live as long as the address is used"""
    return a.buffer_info()[0] if a else None


def clip_grad_norm_device(grads, max_norm):
    """The global 2-norm over all tensors of `grads` (a tensor or an iterable of fp32 / bf16 / fp16 CUDA tensors; the
    types may differ), and grads *= min(1, max_norm / (norm + 1e-6)) in place (g1_clip_grad_norm), on torch's
    current stream.  Returns the norm before clipping as a CUDA fp32 scalar; nothing synchronises.  The
    squares are summed in fp64 in a fixed order.  max_norm inf: nothing is scaled; otherwise a norm that is NaN or
    infinite scales as in torch.nn.utils.clip_grad_norm_.  It takes gradients, not the parameters that hold
    them.  Tensors of one call may not share memory."""
    lib = load_library()
    grads = [grads] if isinstance(grads, torch.Tensor) else list(grads)
    kinds = set(map(type, grads))
    if nn.Parameter in kinds:
        raise G1Error("clip_grad_norm_device takes the gradients, not the parameters")
    if not all(issubclass(t, torch.Tensor) for t in kinds):
        raise G1Error("gradients must be tensors (leave out those of parameters that have none)")
    dev, kinds = _cuda_list(grads, "gradients", _GRAD_TYPE)
    if dev is None:
        _require_gpu()
        dev = torch.device("cuda", torch.cuda.current_device())
    n = len(grads)
    norm = torch.empty((), dtype=torch.float32, device=dev)
    size = lib.g1_opt_workspace(n)
    ws = torch.empty(size, dtype=torch.uint8, device=dev)
    ptrs, types, counts = _ptrs(grads), _types(grads, kinds), array("q", map(_T.numel, grads))
    with _on(dev):
        rc = lib.g1_clip_grad_norm(n, _at(ptrs), _at(types), _at(counts), max_norm, norm.data_ptr(), ws.data_ptr(), size,
                                   _stream_of(dev))
    if rc:
        _check()
    torch.autograd.graph.increment_version(grads)
    return norm


class ClipAdam:
    """Adam with the clipping of the global gradient norm taken into its step (g1_clip_adam): one pass over
    gradients, parameters and moments in place of clip_grad_norm_ followed by torch.optim.Adam.step.

    params: fp32 CUDA tensors on one device.  max_norm: the clip threshold (inf: none).  weight_decay is
    decoupled (p *= 1 - lr * weight_decay).  lr may be a one-element fp32 CUDA tensor, read by the kernel.
    moments: (first, second), lists of fp32 tensors laid out like the parameters, to be used in place
    (made, zero, by default); steps: steps taken before.  Each parameter counts its own steps on the
    device; one without a gradient is left alone, its count too, as in torch.

    step() reads each parameter's .grad, step(grads) a list of fp32 / bf16 / fp16 gradients (None: left alone).
    It returns the norm before clipping as a CUDA scalar; the gradients keep their values.  Nothing
    synchronises, and a step captured into a CUDA graph counts on at each replay.  lr, betas, eps, max_norm and
    weight_decay are plain attributes, read at each step (at capture, for a captured one; a tensor lr at each replay)."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, max_norm=float("inf"), weight_decay=0.0,
                 moments=None, steps=0):
        _require_gpu()
        load_library()
        if isinstance(params, torch.Tensor):
            raise G1Error("parameters must be a list of tensors")
        self.params = list(params)
        if not self.params:
            raise G1Error("no parameters")
        if not all(isinstance(p, torch.Tensor) for p in self.params):
            raise G1Error("parameters must be tensors (no groups of them, no names)")
        self.device = _cuda_list(self.params, "parameters", (torch.float32,))[0]
        self.lr, self.betas, self.eps = lr, (float(betas[0]), float(betas[1])), float(eps)
        self.max_norm, self.weight_decay = float(max_norm), float(weight_decay)
        like = lambda: [torch.zeros_like(p, requires_grad=False) for p in self.params]
        self._m, self._v = (tuple(x) for x in (moments if moments is not None else (like(), like())))
        for ms in (self._m, self._v):
            if len(ms) != len(self.params):
                raise G1Error("moments must be one tensor a parameter")
            _cuda_list([*ms, *self.params[:1]], "moments", (torch.float32,))
            for m, p in zip(ms, self.params):
                if m.shape != p.shape or m.stride() != p.stride():
                    raise G1Error("moments must be laid out like their parameters")
        if int(steps) < 0:
            raise G1Error("steps must be >= 0")
        self._steps = torch.full((len(self.params),), int(steps), dtype=torch.int64, device=self.device)
        self._counts = [p.numel() for p in self.params]
        self._shapes = [p.shape for p in self.params]
        self._strides = [p.stride() for p in self.params]
        self._flat = all(p.is_contiguous() for p in self.params)
        self._where = {self.device.index}
        self._state = [*self._m, *self._v, self._steps]

    # the kernel writes to these: their numbers may be changed, the tensors stay
    exp_avg = property(lambda self: self._m)
    exp_avg_sq = property(lambda self: self._v)
    steps = property(lambda self: self._steps)

    def zero_grad(self, set_to_none=True):
        for p in self.params:
            if set_to_none:
                p.grad = None
            elif p.grad is not None:
                p.grad.zero_()

    def _like(self, ts):
        """Whether these lie in memory as the parameters did.  Strides and lengths alone do not say so: [6, 1] and [2, 3] may share
        strides (3, 1), and only one of them has no gaps."""
        if [t.shape for t in ts] != self._shapes:
            return False
        return all(map(_T.is_contiguous, ts)) if self._flat else list(map(_T.stride, ts)) == self._strides

    def step(self, grads=None):
        params, n, dev = self.params, len(self.params), self.device
        grads = [p.grad for p in params] if grads is None else list(grads)
        if len(grads) != n:
            raise G1Error("step takes one gradient (or None) a parameter")
        lib = _lib
        if (not self._like(params) or set(map(_T.get_device, params)) != self._where
                or {p.dtype for p in params} != {torch.float32}):
            raise G1Error("a parameter is no longer laid out as it was when the optimiser was made")
        if any(g is None for g in grads):
            have = [i for i, g in enumerate(grads) if g is not None]
        else:
            have = range(n)
            if self._like(grads):
                have = ()  # nothing to look at one by one
        for i in have:
            g, p = grads[i], params[i]
            if g.shape != p.shape:
                raise G1Error("gradients must have their parameters' shapes")
            if g.stride() != self._strides[i]:
                if not g.is_cuda:
                    raise G1Error("gradients must be CUDA tensors")
                grads[i] = torch.empty_like(p, dtype=g.dtype, requires_grad=False).copy_(g.detach())
        there = grads if have == () else [g for g in grads if g is not None]
        kinds = {g.dtype for g in there}
        if not set(map(_T.get_device, there)) <= self._where or not kinds <= _GRAD_TYPE.keys():
            raise G1Error("gradients must be fp32, bf16 or fp16 on their parameters' device")
        if len(there) == n:
            ptrs, types, counts, moved = _ptrs(grads), _types(grads, kinds), array("q", self._counts), params
        else:
            ptrs = array("Q", [0 if g is None else g.data_ptr() for g in grads])
            types = array("i", [0 if g is None else _GRAD_TYPE[g.dtype] for g in grads])
            counts = array("q", [0 if g is None else c for g, c in zip(grads, self._counts)])
            moved = [p for p, g in zip(params, grads) if g is not None]
        norm = torch.empty((), dtype=torch.float32, device=dev)
        size = lib.g1_opt_workspace(n)
        ws = torch.empty(size, dtype=torch.uint8, device=dev)
        lr, lr_dev = self.lr, None
        if isinstance(lr, torch.Tensor):
            if not (lr.device == dev and lr.dtype == torch.float32 and lr.numel() == 1):
                raise G1Error("a tensor lr must be one fp32 number on the parameters' device")
            lr, lr_dev = 0.0, lr.data_ptr()
        p, m, v = _ptrs(params), _ptrs(self._m), _ptrs(self._v)
        with _on(dev):
            rc = lib.g1_clip_adam(n, _at(ptrs), _at(types), _at(p), _at(m), _at(v), _at(counts), self._steps.data_ptr(),
                                  self.max_norm, lr, lr_dev, self.betas[0], self.betas[1], self.eps, self.weight_decay,
                                  norm.data_ptr(), ws.data_ptr(), size, _stream_of(dev))
        if rc:
            _check()
        torch.autograd.graph.increment_version(moved + self._state)
        return norm

    def state_dict(self):
        lr = self.lr.detach().clone() if isinstance(self.lr, torch.Tensor) else self.lr
        return dict(lr=lr, betas=self.betas, eps=self.eps, max_norm=self.max_norm, weight_decay=self.weight_decay,
                    exp_avg=[m.clone() for m in self.exp_avg], exp_avg_sq=[v.clone() for v in self.exp_avg_sq],
                    steps=self.steps.clone())

    @torch.no_grad()
    def load_state_dict(self, d):
        """Takes the state of another ClipAdam over parameters of the same shapes; one that does not fit changes nothing."""
        for name in ("exp_avg", "exp_avg_sq"):
            if [tuple(m.shape) for m in d[name]] != [tuple(p.shape) for p in self.params]:
                raise G1Error("the state's moments do not have the parameters' shapes")
        steps = torch.as_tensor(d["steps"])
        if steps.shape != self.steps.shape or steps.dtype != torch.int64 or bool((steps < 0).any()):
            raise G1Error("the state's steps must be one count a parameter")
        if torch.as_tensor(d["lr"]).numel() != 1:
            raise G1Error("the state's lr must be one number")
        if isinstance(self.lr, torch.Tensor):
            self.lr.copy_(torch.as_tensor(d["lr"]).reshape(self.lr.shape))
        else:
            self.lr = float(d["lr"])
        self.betas, self.eps = tuple(d["betas"]), d["eps"]
        self.max_norm, self.weight_decay = d["max_norm"], d["weight_decay"]
        for ours, theirs in ((self.exp_avg, d["exp_avg"]), (self.exp_avg_sq, d["exp_avg_sq"])):
            for a, b in zip(ours, theirs):
                a.copy_(b)
        self.steps.copy_(steps)


# ---------------- running obs normalizer (the state of ppo.py:63-81) ----------------
class RunNorm:
    """Running mean / variance of the raw observations and the clipped normalisation
    z = clamp((o - mean) / sqrt(var + 1e-8), +-10) that the rollout kernel applies.

    The state (mean, var, count) and its merge rule are the reference's (a batch of b rows
    with moments (m_b, v_b) merged into (mean, var, count) by the parallel-variance formula).
    Batches are reduced here in fp64 -- the same moments the device batch preparation
    (g1_obs_prep + g1_runnorm_update) accumulates -- so a host update and a device update of
    the same rows agree to fp32 rounding."""

    def __init__(self, dim, dev):
        self.mean = torch.zeros(dim, device=dev)
        self.var = torch.ones(dim, device=dev)
        self.count = 1e-4

    def merge(self, m_b, v_b, b):
        """Merge a batch of b rows with per-dimension mean m_b and (biased) variance v_b."""
        n0, n = float(self.count), float(b)
        tot = n0 + n
        m0, v0 = self.mean.double(), self.var.double()
        d = m_b.double() - m0
        self.mean = (m0 + d * (n / tot)).float()
        self.var = ((v0 * n0 + v_b.double() * n + d * d * (n0 * n / tot)) / tot).float()
        self.count = tot

    def update(self, x):
        """Merge the rows of x [B, dim] (fp64 moments)."""
        xd = x.detach().double()
        m_b = xd.mean(0)
        self.merge(m_b, (xd * xd).mean(0) - m_b * m_b, x.shape[0])

    def norm(self, x):
        return torch.clamp((x - self.mean) / torch.sqrt(self.var + 1e-8), -10.0, 10.0)


# ---------------- actor-critic (ppo.py:85-99) ----------------
class AC(nn.Module):
    """The reference's actor-critic (shared trunk, value head on the last hidden layer).
    value_hidden: a separate value network of those widths instead.
    activation "swiglu" or "geglu": the hidden layers are GatedLinear, in bf16 on the tensor cores (CUDA only)."""

    def __init__(self, obs_dim, act_dim, hidden=(256, 256), activation="tanh", value_hidden=None):
        super().__init__()
        act = (lambda: nn.Tanh()) if activation == "tanh" else (lambda: nn.ELU())
        gate = {"swiglu": "silu", "geglu": "gelu"}.get(activation)
        layer = (lambda i, o: [GatedLinear(i, o, gate)]) if gate else (lambda i, o: [nn.Linear(i, o), act()])
        layers, d = [], obs_dim
        for h in hidden:
            layers += layer(d, h)
            d = h
        self.hidden = tuple(hidden)
        self.activation = activation
        self.value_hidden = tuple(value_hidden) if value_hidden else None
        self.body = nn.Sequential(*layers)
        self.mu = nn.Linear(d, act_dim)
        if self.value_hidden:
            vl, dv = [], obs_dim
            for h in self.value_hidden:
                vl += layer(dv, h)
                dv = h
            self.v_body = nn.Sequential(*vl)
            self.v = nn.Linear(dv, 1)
        else:
            self.v = nn.Linear(d, 1)
        self.log_std = nn.Parameter(-0.5 * torch.ones(act_dim))

    def forward(self, x):
        # gated layers answer in bf16, where the heads are fp32; other layers hand on what they make
        head = (lambda z: z.to(self.mu.weight.dtype)) if self.activation in ("swiglu", "geglu") else (lambda z: z)
        z = head(self.body(x))
        v = self.v(head(self.v_body(x))) if self.value_hidden else self.v(z)
        return self.mu(z), self.log_std.exp(), v.squeeze(-1)


def pack_weights(ac):
    """Flatten AC params in the order the kernel unpacks (ppo_fused.py:35-44): per hidden
    layer W,b; then Wmu,bmu, Wv,bv, log_std.  nn.Linear weight is [out,in] row-major.
    With a separate value network (g1_env_set_value_net): per policy hidden layer W,b; Wmu,
    bmu, log_std; per value hidden layer W,b; Wv, bv.  A gated layer's W is [2h,in], its b [2h]."""
    lin = lambda seq: [t for m in seq if isinstance(m, (nn.Linear, GatedLinear)) for t in (m.weight.reshape(-1), m.bias)]
    parts = lin(ac.body)
    if getattr(ac, "value_hidden", None):
        parts += [ac.mu.weight.reshape(-1), ac.mu.bias, ac.log_std] + lin(ac.v_body) + [ac.v.weight.reshape(-1), ac.v.bias]
    else:
        parts += [ac.mu.weight.reshape(-1), ac.mu.bias, ac.v.weight.reshape(-1), ac.v.bias, ac.log_std]
    return torch.cat(parts).contiguous()


def init_policy_normal(ac, seed=0):
    """Config-2 style random init: N(0, 1/fan_in) weights, zero bias, log_std = -0.5."""
    g = torch.Generator(device="cpu").manual_seed(seed)
    with torch.no_grad():
        for m in ac.modules():
            if isinstance(m, (nn.Linear, GatedLinear)):
                m.weight.copy_(torch.randn(m.weight.shape, generator=g) / np.sqrt(m.weight.shape[1]))
                m.bias.zero_()
        ac.log_std.fill_(-0.5)
    return ac


@torch.no_grad()
def evaluate(env, ac, norm, dev, steps=200):
    """Deterministic (mean-action) evaluation on the device-resident host-loop step path
    (g1_env_step_device), reporting the metrics of the reference trainer's evaluate
    (ppo.py:103-125): distance walked (base forward velocity, obs[:, 0], integrated over
    the 0.02 s control step) until the first episode end, its mean and max over worlds, the
    mean number of live steps, the fraction of worlds that ended an episode, and the mean
    forward velocity while live.  Everything stays on the GPU; one host sync at the end."""
    N, ctrl_dt = env.N, 0.02
    obs = torch.as_tensor(env.reset(), device=dev)
    rew = torch.zeros(N, device=dev)
    done = torch.zeros(N, device=dev)
    live = torch.ones(N, device=dev)
    dist = torch.zeros(N, device=dev)
    vsum = torch.zeros(N, device=dev)
    nlive = torch.zeros(N, device=dev)
    for _ in range(steps):
        mu = ac(norm.norm(obs))[0].contiguous()
        env.step_device(mu, obs, rew, done)
        vx = obs[:, 0]
        dist += live * vx * ctrl_dt
        vsum += live * vx
        nlive += live
        live = live * (done == 0).float()
    fallen = 1.0 - live
    out = torch.stack([dist.mean(), dist.max(), nlive.mean(), fallen.mean(),
                       (vsum / nlive.clamp_min(1.0)).mean()]).tolist()
    return dict(zip(("fwd_mean", "fwd_max", "ep_len_mean", "fall_rate", "vx_mean"), out))
