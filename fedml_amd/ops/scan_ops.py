"""Gated linear recurrence over long sequences (``csrc/scan_kernels.hip``): per sequence and feature

    f_t = σ(gate_t),   h_t = f_t·h_{t−1} + (1 − f_t)·x_t,   y_t = h_t

The recurrence is linear in the state, so unlike an LSTM's (:mod:`.rnn_ops`) it needs no product with a weight per step
and a whole sequence is one launch each way, two where few features cut the time into segments. Layout of the recurrent
models: ``[C, T, B, H]`` (client, time, sequence, feature); any strides with dense features, so token-major rows go in as
``x.view(C, B, T, H).transpose(1, 2)``.

CUDA tensors run the HIP kernels (bf16 or fp32 storage; states, maps and sums fp32), CPU tensors the same recurrence in
plain PyTorch (fp64 for fp64 inputs), the tests' oracle. Results are the same bit for bit from call to call. Everything
is enqueued on the current stream of the tensors' device and may be captured into a HIP graph."""
import ctypes as _c
import functools

import torch
from torch.autograd.function import once_differentiable

from ._launch import MAX_THREADS, launch, ptr, ptr_read
from .fl_ops import use_native

_TILE = 32                # steps between two kept states
# A call of fewer than _FULL workgroups cuts the time into segments, up to _WANT workgroups: x and gate are then read
# twice. Forward + backward in us, whole / cut, at 64 workgroups (16384 steps): 1330 / 346; at 256: 361 / 353; at 384
# (4096 steps): 495 / 541; more than 512 workgroups gain nothing.
_FULL, _WANT = 256, 1024
_I32 = 2 ** 31 - 1


class _Args(_c.Structure):
    _fields_ = [(n, _c.c_void_p) for n in ("x", "gate", "dy", "y", "dx", "dgate", "h0", "dh", "hT", "dh0", "ckpt",
                                           "agg", "mask")] + \
               [(n, _c.c_int64 * 3) for n in ("xs", "gs", "dys", "ys", "ms")] + \
               [(n, _c.c_int) for n in ("C", "T", "B", "H", "nseg", "tps")]


def _dense(t):
    """Dense features; nothing else is asked of the strides."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _like(x):
    """An empty [C, T, B, H] laid out in x's order of time and sequence."""
    C, T, B, H = x.shape
    if x.stride(2) > x.stride(1):
        return torch.empty(C, B, T, H, dtype=x.dtype, device=x.device).transpose(1, 2)
    return torch.empty(C, T, B, H, dtype=x.dtype, device=x.device)


@functools.lru_cache(maxsize=512)
def _plan(shape, xs, gs, ys, dys, ms, aligned):
    """(what the kernels' arguments hold for all calls of these sizes and strides, features a lane takes at a time)"""
    C, T, B, H = shape
    a = _Args(C=C, T=T, B=B, H=H)
    a.xs[:], a.gs[:], a.ys[:] = xs[:3], gs[:3], ys[:3]
    odd = H
    for st in (xs, gs, ys, dys or ()):
        for s in st[:3]:
            odd |= s
    if dys is not None:
        a.dys[:] = dys[:3]
    if ms is not None:
        a.ms[:] = ms
    vec = 2 if aligned and not odd & 1 else 1       # two where every row starts at a multiple of two features
    wgs, ntile = C * B * -(-H // (32 * vec)), -(-T // _TILE)
    nseg = 1 if wgs >= _FULL else min(ntile, -(-_WANT // wgs), 64)
    a.tps = -(-ntile // (2 * nseg)) * 2             # pairs of tiles
    a.nseg = -(-ntile // a.tps)
    if 256 * wgs * a.nseg > MAX_THREADS:
        raise ValueError(f"gated_scan: {C} clients · {B} sequences · {H} features are too many for one call")
    return a, vec


def _run(x, gate, mask, y, h0, hT, ckpt, dy=None, dh=None, dx=None, dgate=None, dh0=None):
    bwd = dx is not None
    out = dx if bwd else y
    at = x.data_ptr() | gate.data_ptr() | out.data_ptr() | (dgate.data_ptr() | dy.data_ptr() if bwd else 0)
    plan, vec = _plan(x.shape, x.stride(), gate.stride(), out.stride(), dy.stride() if bwd else None,
                      None if mask is None else mask.stride(), at % (2 * x.element_size()) == 0)
    a = _Args.from_buffer_copy(plan)
    a.x, a.gate, a.mask, a.ckpt = ptr_read(x), ptr_read(gate), ptr_read(mask), ptr_read(ckpt) if bwd else ptr(ckpt)
    if bwd:
        a.dy, a.dh, a.dx, a.dgate, a.dh0 = ptr_read(dy), ptr_read(dh), ptr(dx), ptr(dgate), ptr(dh0)
    else:
        a.y, a.hT, a.h0 = ptr(y), ptr(hT), ptr_read(h0)
    if a.nseg > 1:
        agg = torch.empty(a.C * a.B * a.nseg * 2 * a.H, dtype=torch.float32, device=x.device)
        a.agg = ptr(agg)
    launch("fa_gated_scan", a, (x.dtype == torch.bfloat16, vec, bwd), x.device)


def _forward(x, gate, h0, mask, keep):
    C, T, B, H = x.shape
    y = _like(x)
    hT = torch.empty(C, B, H, dtype=torch.float32, device=x.device)
    ckpt = torch.empty(C, -(-T // _TILE), B, H, dtype=torch.float32, device=x.device) if keep else None
    if C * B:
        _run(x, gate, mask, y, h0, hT, ckpt)
    return y, hT, ckpt


class _GatedScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, h0, mask):
        x, gate = _dense(x), _dense(gate)
        y, hT, ckpt = _forward(x, gate, None if h0 is None else h0.contiguous(), mask, True)
        ctx.save_for_backward(x, gate, mask, ckpt)
        ctx.set_materialize_grads(False)
        return y, hT

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dh):
        x, gate, mask, ckpt = ctx.saved_tensors
        if dy is None and dh is None:
            return None, None, None, None
        C, T, B, H = x.shape
        dy = torch.zeros_like(x) if dy is None else _dense(dy.to(x.dtype))
        dh = None if dh is None else dh.contiguous()
        dx, dgate = _like(x), _like(x)          # of one layout
        dh0 = torch.empty(C, B, H, dtype=torch.float32, device=x.device) if ctx.needs_input_grad[2] else None
        if C * B:
            _run(x, gate, mask, None, None, None, ckpt, dy, dh, dx, dgate, dh0)
        return dx, dgate, dh0, None


def _scan_ref(x, gate, h0, mask):
    ct = torch.float64 if x.dtype == torch.float64 else torch.float32
    C, T, B, H = x.shape
    g, b = gate.to(ct), x.to(ct)
    real = None if mask is None else (mask != 0).unsqueeze(-1)
    zero = torch.zeros((), dtype=ct, device=x.device)
    if real is not None:      # selected before any product: what padding holds reaches nothing
        g, b = torch.where(real, g, zero), torch.where(real, b, zero)
    ls = torch.nn.functional.logsigmoid       # f and 1 − f by their logarithms: neither they nor their slopes cancel
    f, b = ls(g).exp(), ls(-g).exp() * b
    if real is not None:
        f = torch.where(real, f, zero + 1)
    h = torch.zeros(C, B, H, dtype=ct, device=x.device) if h0 is None else h0.to(ct)
    ys = []
    for t in range(T):
        h = f[:, t] * h + b[:, t]
        ys.append(h if real is None else torch.where(real[:, t], h, zero))
    return torch.stack(ys, 1).to(x.dtype), h


def gated_scan(x: torch.Tensor, gate: torch.Tensor, h0: torch.Tensor = None, mask: torch.Tensor = None):
    """(y, h_T) of the recurrence above for ``x`` and ``gate`` [C, T, B, H] from the state ``h0`` [C, B, H] (fp32; zero
    if not given): y [C, T, B, H] at x's type, in x's order of time and sequence, and the state after the last step
    h_T [C, B, H], fp32 — the ``h0`` of the next call. T = 1 is the step of a program that answers token by token.

    ``mask`` [C, T, B] (bool or integer, nonzero = a step): a step that is padding leaves the state as it is, its y is
    zero, and what x, gate and the gradient of y hold there (NaN included) reaches nothing. Gradients: x, gate (at their
    type) and h0 (fp32)."""
    if x.dim() != 4 or gate.shape != x.shape:
        raise ValueError(f"gated_scan: x and gate [C, T, B, H] expected, got {tuple(x.shape)} and {tuple(gate.shape)}")
    if x.dtype not in (torch.bfloat16, torch.float32) and (x.is_cuda or x.dtype != torch.float64):
        raise TypeError(f"gated_scan: bf16 or fp32 expected, got {x.dtype}")
    if gate.dtype != x.dtype or gate.device != x.device:
        raise TypeError(f"gated_scan: gate is {gate.dtype} on {gate.device}, x {x.dtype} on {x.device}")
    C, T, B, H = x.shape
    if T < 1 or H < 1:
        raise ValueError(f"gated_scan: at least one step and one feature expected, got {tuple(x.shape)}")
    if T > _I32 - 2 * _TILE:
        raise ValueError(f"gated_scan: {T} steps are too many for one call")
    state = torch.float64 if x.dtype == torch.float64 else torch.float32
    if h0 is not None and (h0.shape != (C, B, H) or h0.dtype != state or h0.device != x.device):
        raise ValueError(f"gated_scan: h0 {state} [{C}, {B}, {H}] on {x.device} expected, got {h0.dtype} "
                         f"{tuple(h0.shape)} on {h0.device}")
    if mask is not None and (mask.shape != (C, T, B) or mask.dtype.is_floating_point or mask.dtype.is_complex or
                             mask.device != x.device):
        raise ValueError(f"gated_scan: mask bool or integer [{C}, {T}, {B}] on {x.device} expected, got {mask.dtype} "
                         f"{tuple(mask.shape)} on {mask.device}")
    if not use_native(x):
        return _scan_ref(x, gate, h0, mask)
    if mask is not None:
        mask = (mask if mask.dtype == torch.bool else mask != 0).view(torch.uint8)
    if (x.requires_grad or gate.requires_grad or (h0 is not None and h0.requires_grad)) and torch.is_grad_enabled():
        return _GatedScan.apply(x, gate, h0, mask)
    y, hT, _ = _forward(_dense(x), _dense(gate), None if h0 is None else h0.contiguous(), mask, False)
    return y, hT
