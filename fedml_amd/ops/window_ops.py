"""Causal sliding-window attention with sinks and a bucketed relative position bias, for long text
(``csrc/window_kernels.hip``).

* :func:`window_attention` — forward and backward over whole sequences of any length: token i sees the ``window`` last
  tokens up to itself and the first ``sinks`` tokens; ``kv_heads`` ≤ H shared key/value heads; a token mask; a learned
  bias per head and distance bucket (``bias``), with its gradient.
* :func:`window_attention_step` — the same for ONE new token per sequence over a ring cache of ``sinks + window``
  slots, which it updates; :func:`window_cache_fill` puts a prompt's keys and values there.
* :func:`relative_bucket_starts` — the first distance of every bucket.

Rows are token-major ``[sequences · S, heads · D]``, head h at columns ``[h·D, (h+1)·D)``, D = 64 or 128, bf16 or fp32
(row strides may exceed heads · D: column slices of a fused projection are read in place). CUDA tensors run the HIP
kernels at the storage precision with fp32 sums and statistics; CPU tensors run the plain-PyTorch form of the same
mathematics (fp64 for fp64 inputs), which is also the tests' oracle. All results are the same bit for bit from call to
call: no atomics. (With a bias and bf16 the output's bits differ between calls with and without a gradient of the bias:
before one, the probabilities go into it unrounded.) Everything is enqueued on the current stream of the tensors' device
and may be captured into a HIP graph, forward and backward in the same one, on leaves that no living eager graph holds;
scratch memory is allocated per call."""
import ctypes as _c
import functools
import math

import torch
from torch.autograd.function import once_differentiable

from ._launch import MAX_THREADS, launch, ptr, ptr_read
from .fl_ops import _check, _fn, _i64, _p, _pr, _stream, use_native

MAX_SINKS = 64
MAX_BUCKETS = 128
MAX_DISTANCE = 1024
_I32 = 2 ** 31 - 1
_ROWS_IN_CACHE = -1              # fa_window_step launched nothing: its rows lie in a cache that it writes


class _Args(_c.Structure):
    _fields_ = [(n, _c.c_void_p) for n in ("q", "k", "v", "dout", "o", "dq", "dk", "dv", "o32", "lse", "dsum", "part",
                                           "bpart", "dbias", "mask", "bias")] + \
               [(n, _c.c_int64) for n in ("ldq", "ldk", "ldv", "lddo")] + \
               [(n, _c.c_int) for n in ("N", "S", "H", "KV", "C", "W", "sinks", "NB", "maxd", "nchunk", "qchunk", "nslot",
                                        "exact", "tile", "ktile")] + \
               [("scale", _c.c_float), ("start", _c.c_int * MAX_BUCKETS)]


class _StepArgs(_c.Structure):
    _fields_ = [(n, _c.c_void_p) for n in ("q", "k", "v", "kc", "vc", "o", "pos", "bias", "pacc", "pml")] + \
               [(n, _c.c_int64) for n in ("ldq", "ldk", "ldv")] + \
               [(n, _c.c_int) for n in ("B", "H", "KV", "C", "W", "sinks", "NB", "maxd", "splits", "per")] + \
               [("scale", _c.c_float), ("start", _c.c_int * MAX_BUCKETS)]


@functools.lru_cache(maxsize=None)
def relative_bucket_starts(buckets: int, max_distance: int):
    """First distance of every bucket: one distance each below E = buckets // 2, then evenly over the logarithm up to
    ``max_distance``; the last bucket has no end. bucket(d) = d for d < E, else
    min(buckets − 1, E + ⌊n·log(d/E) / log(max_distance/E)⌋) with n = buckets − E, decided in whole numbers
    (d^n ≥ max_distance^j · E^(n−j)), so that no rounding moves a border."""
    buckets, M = int(buckets), int(max_distance)
    if not 2 <= buckets <= MAX_BUCKETS:
        raise ValueError(f"relative bias: 2 to {MAX_BUCKETS} buckets, got {buckets}")
    E = buckets // 2
    n = buckets - E
    if not E < M <= MAX_DISTANCE:
        raise ValueError(f"relative bias: max_distance in ({E}, {MAX_DISTANCE}] for {buckets} buckets, got {M}")
    starts, d = list(range(E + 1)), E
    for j in range(1, n):
        while d ** n < M ** j * E ** (n - j):
            d += 1
        starts.append(d)
    return tuple(starts)


def relative_bucket(distance: torch.Tensor, buckets: int, max_distance: int) -> torch.Tensor:
    """Bucket of every (whole, ≥ 0) distance."""
    starts = torch.tensor(relative_bucket_starts(buckets, max_distance), device=distance.device)
    return torch.bucketize(distance, starts, right=True) - 1


# ------------------------------------------------------------------------------------------------- argument checks
def _rows(t, heads, name, rows=None, dtype=None, device=None):
    """(D, rows) of a token-major operand."""
    if t.dim() != 2 or heads < 1 or t.shape[1] % heads:
        raise ValueError(f"{name}: [rows, heads · D] with {heads} heads expected, got {tuple(t.shape)}")
    if t.dtype not in (torch.bfloat16, torch.float32) and (t.is_cuda or t.dtype != torch.float64):
        raise TypeError(f"{name}: bf16 or fp32 expected, got {t.dtype}")
    if dtype is not None and t.dtype != dtype:
        raise TypeError(f"{name}: {dtype} expected, got {t.dtype}")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, q on {device}")
    if rows is not None and t.shape[0] != rows:
        raise ValueError(f"{name}: {rows} rows expected, got {t.shape[0]}")
    return t.shape[1] // heads


def _common(q, k, v, H, kv_heads, window, sinks):
    H, KV = int(H), int(H if kv_heads is None else kv_heads)
    if H < 1 or KV < 1 or H % KV:
        raise ValueError(f"H = {H} query heads over {KV} key/value heads")
    D = _rows(q, H, "q")
    if D not in (64, 128):
        raise ValueError(f"head dim 64 or 128 expected, got {D}")
    if q.shape[1] > _I32:                        # the kernels' offsets inside a row are 32 bits wide
        raise ValueError(f"{H} heads of dim {D}: at most 2^31 − 1 elements a row")
    for t, n in ((k, "k"), (v, "v")):
        if _rows(t, KV, n, q.shape[0], q.dtype, q.device) != D:
            raise ValueError(f"{n}: {KV} heads of dim {D} expected, got {tuple(t.shape)}")
    if not 1 <= int(window) <= _I32:
        raise ValueError(f"window ≥ 1 expected, got {window}")
    if not 0 <= int(sinks) <= MAX_SINKS:
        raise ValueError(f"sinks in [0, {MAX_SINKS}] expected, got {sinks}")
    return D, H, KV, int(window), int(sinks)


def _bias(bias, sequences, H, max_distance, device):
    """The table as [C, H, buckets]."""
    if bias is None:
        return None
    if bias.dim() not in (2, 3) or bias.shape[-2] != H:
        raise ValueError(f"bias: [H, buckets] or [C, H, buckets] with H = {H} expected, got {tuple(bias.shape)}")
    if bias.device != device:
        raise ValueError(f"bias is on {bias.device}, q on {device}")
    if bias.dtype != torch.float32 and (bias.is_cuda or bias.dtype != torch.float64):
        raise TypeError(f"bias: fp32 expected, got {bias.dtype}")
    if bias.dim() == 2:
        bias = bias.unsqueeze(0)
    C = bias.shape[0]
    if C < 1 or sequences % C:
        raise ValueError(f"bias of {C} clients for {sequences} sequences")
    relative_bucket_starts(bias.shape[-1], max_distance)      # its own refusals
    return bias


def _scale(scale, D):
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if not 2.0 ** -126 <= scale <= 2.0 ** 127:      # in fp32, and with log2 e, neither zero nor infinite
        raise ValueError(f"scale in [2^-126, 2^127] expected, got {scale}")
    return scale


def _aligned(t):
    """16-byte rows for the kernels: the tensor itself where its rows are, else a dense copy."""
    e = 16 // t.element_size()
    if (t.stride(1) == 1 or t.shape[1] == 1) and t.stride(0) % e == 0 and t.stride(0) >= t.shape[1] and \
            t.data_ptr() % 16 == 0:
        return t
    return t.clone(memory_format=torch.contiguous_format)


# ------------------------------------------------------------------------------------------------------- reference
def _ct(t):
    return torch.float64 if t.dtype == torch.float64 else torch.float32


def _bias_of(bias, distance, sequences, max_distance, ct):
    """[sequences, H, ·] bias of whole distances (negative ones: any value)."""
    b = relative_bucket(distance.clamp_min(0), bias.shape[-1], max_distance)
    return bias.to(ct)[..., b].repeat_interleave(sequences // bias.shape[0], 0)


def _window_ref(q, k, v, S, H, KV, W, sinks, mask, bias, max_distance, scale):
    N, D, ct = q.shape[0] // S, q.shape[1] // H, _ct(q)
    real = torch.ones(N, S, dtype=torch.bool, device=q.device) if mask is None else mask.bool()

    def heads(t, h):     # what is no token is zero, whatever it holds
        return torch.where(real.view(N, S, 1, 1), t.to(ct).view(N, S, h, D), torch.zeros((), dtype=ct, device=q.device)
                           ).transpose(1, 2)

    qh, kh, vh = heads(q, H), *(heads(t, KV).repeat_interleave(H // KV, 1) for t in (k, v))
    i = torch.arange(S, device=q.device)
    d = i.view(S, 1) - i
    see = (d >= 0) & ((d < W) | (i < sinks))
    see = (see & real.view(N, 1, S) & real.view(N, S, 1)).unsqueeze(1)
    s = qh @ kh.transpose(-1, -2) * scale
    if bias is not None:
        s = s + _bias_of(bias, d, N, max_distance, ct)
    s = s.masked_fill(~see, float("-inf"))
    p = torch.softmax(s.masked_fill(~see.any(-1, keepdim=True), 0.0), -1)
    p = torch.where(see, p, torch.zeros((), dtype=ct, device=q.device))
    o = torch.where(real.view(N, 1, S, 1), p @ vh, torch.zeros((), dtype=ct, device=q.device))
    return o.transpose(1, 2).reshape(N * S, H * D).to(q.dtype)


# --------------------------------------------------------------------------------------------------------- training
@functools.lru_cache(maxsize=256)
def _plan(D, N, S, H, KV, W, sinks, scale, fp32, C, buckets, max_distance, train):
    """What the kernels' arguments hold for all calls of these sizes (train: with a backward pass)."""
    a = _Args(N=N, S=S, H=H, KV=KV, C=C, W=W, sinks=sinks, NB=buckets, scale=scale)
    if buckets:
        a.maxd = max_distance
        a.start[:buckets] = relative_bucket_starts(buckets, max_distance)
    # Queries of a workgroup, forward and dq: one wave's 32 for short sequences, and at fp32, where products are 16 times
    # as long, wherever no more than 1024 such waves are there (a wave then walks its own keys, not its workgroup's).
    # us forward + backward, 128 / 32 queries, at windows of 32, 128 and 512:
    #   fp32 [80·80, 4 heads] 81 / 67, 86 / 80; [16·256, 4] 61 / 44, 94 / 78, 102 / 107; [2·1000, 8] 63 / 45, 96 / 80,
    #   220 / 215; [4·256, 8, D 128] 123 / 88, 183 / 151, 185 / 188; more waves: [64·128, 12] W 32 152 / 138, W 512
    #   173 / 192; [8·1024, 8] W 32 118 / 99, W 512 413 / 416;
    #   bf16 [64·20, 4] 15 / 15; [16·256, 4] 28 / 24, 33 / 32, 33 / 38; [2·2048, 8] 32 / 30, 38 / 39, 62 / 72.
    # Windows up to 64 gain from 32 queries on the other side of the rule too; the rule does not look at them.
    a.tile = 32 if S <= 64 or (fp32 and N * H * -(-S // 32) <= 1024) else 128
    # Keys of a workgroup, dk and dv: 64 for short sequences and at fp32, but 128 at fp32 and 128 dims, where two waves
    # would spill. us forward + backward, 128 / 64 keys, W 512: fp32 [8·2048, 8 heads] 862 / 829, [2·2048, 8] 239 / 237,
    # [16·256, 4] 108 / 106; bf16 [8·2048, 8] 162 / 162, [2·2048, 8] 64 / 69, [16·256, 4] 33 / 33, [4·4096, 8 over 2,
    # D 128, W 1024] 426 / 495.
    a.ktile = 64 if (S <= 64 or fp32) and not (fp32 and D == 128) else 128
    # The sinks' gradients from behind their window: up to 512 queries are walked by the sinks' own keys, more by a pass
    # of its own in chunks about as long as a window's walk. us forward + backward with the pass / without, for 128, 256,
    # 512 and 1024 such queries: bf16 [2 sequences, 8 heads, W 64] 29 / 27, 33 / 36, 36 / 44, 38 / 62; [16, 12 heads,
    # W 256] 79 / 74, 97 / 102, 139 / 150, 219 / 245; [2, 16 over 4, D 128, W 256] 113 / 114, 118 / 142, 121 / 193,
    # 138 / 302; fp32 [16, 12 heads, W 256] 293 / 290, 417 / 471, 618 / 727, 1013 / 1273. It pays from 256 queries on.
    if sinks and S - W > 512:
        a.qchunk = max(512, -(-(W + 128) // 128) * 128)
        a.nchunk = -(-(S - W) // a.qchunk)
        a.nslot = 1 + a.nchunk * (1 if fp32 else 2)      # a tile is 32 queries at fp32, two waves' 32 at bf16
    # a wave for 32 queries or keys of a head; finish_kernel: a thread for 4 columns of a sink's two gradients
    threads = [2 * N * H * -(-S // a.tile) * a.tile]
    if train:
        threads += [2 * N * KV * (a.nchunk + -(-S // a.ktile)) * a.ktile,
                    256 * C * H + (N * KV * sinks * D // 2 + 255 if a.nchunk else 0)]
    if max(threads) > MAX_THREADS:
        raise ValueError(f"{N} sequences · {H} heads · {S} tokens are too many for one call")
    return a


def _args(q, k, v, mask, bias, cfg):
    a = _Args.from_buffer_copy(_plan(*cfg))
    a.q, a.k, a.v, a.mask, a.bias = ptr_read(q), ptr_read(k), ptr_read(v), ptr_read(mask), ptr_read(bias)
    a.ldq, a.ldk, a.ldv = q.stride(0), k.stride(0), v.stride(0)
    return a


def _forward(q, k, v, mask, bias, cfg, keep, exact):
    """(o, o before its rounding, log-sum-exp); keep: for a backward pass, exact: with a gradient of the bias."""
    D, N, S, H = cfg[:4]
    bf16, dev = q.dtype == torch.bfloat16, q.device
    o = torch.empty(N * S, H * D, dtype=q.dtype, device=dev)
    o32 = lse = None
    if keep:
        o32 = torch.empty(N * S, H * D, dtype=torch.float32, device=dev) if bf16 else o
        # log-sum-exp; with a bias the maximum and the logarithm of the sum
        lse = torch.empty(1 if bias is None else 2, N, H, S, dtype=torch.float32, device=dev)
    if N:
        a = _args(q, k, v, mask, bias, cfg)
        a.o, a.o32, a.lse, a.exact = ptr(o), ptr(o32), ptr(lse), exact
        launch("fa_window_fwd", a, (bf16, D), dev)
    return o, o32, lse


class _WindowAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, bias, mask, cfg):
        q, k, v = _aligned(q), _aligned(k), _aligned(v)
        tab = None if bias is None else bias.contiguous()
        o, o32, lse = _forward(q, k, v, mask, tab, cfg, True, bias is not None and ctx.needs_input_grad[3])
        ctx.save_for_backward(q, k, v, tab, mask, o32, lse)
        ctx.cfg = cfg
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx, do):
        q, k, v, bias, mask, o32, lse = ctx.saved_tensors
        D, N, S, H, KV = ctx.cfg[:5]
        dev, dt, f32 = q.device, q.dtype, torch.float32
        do = _aligned(do if do.dtype == dt else do.to(dt))
        dq = torch.empty(N * S, H * D, dtype=dt, device=dev)
        dk = torch.empty(N * S, KV * D, dtype=dt, device=dev)
        dv = torch.empty(N * S, KV * D, dtype=dt, device=dev)
        dbias = None
        if bias is not None and ctx.needs_input_grad[3]:
            dbias = torch.empty(bias.shape, dtype=f32, device=dev) if N else torch.zeros_like(bias)
        if N:
            a = _args(q, k, v, mask, bias, ctx.cfg)
            dsum = torch.empty(N, H, S, dtype=f32, device=dev)
            part = bpart = None
            if a.nchunk:
                part = torch.empty(N, KV, a.nslot, 2, a.sinks, D, dtype=f32, device=dev)
            if dbias is not None:
                bpart = torch.empty(N, H, -(-S // a.tile), bias.shape[-1], dtype=f32, device=dev)
            a.dout, a.lddo, a.lse, a.o32 = ptr_read(do), do.stride(0), ptr_read(lse), ptr_read(o32)
            a.dq, a.dk, a.dv, a.dsum = ptr(dq), ptr(dk), ptr(dv), ptr(dsum)
            a.part, a.bpart, a.dbias = ptr(part), ptr(bpart), ptr(dbias)
            launch("fa_window_bwd", a, (dt == torch.bfloat16, D), dev)
        return dq, dk, dv, dbias, None, None


def window_attention(q, k, v, S: int, H: int, window: int, sinks: int = 0, kv_heads: int = None,
                     mask: torch.Tensor = None, bias: torch.Tensor = None, max_distance: int = 128,
                     scale: float = None):
    """Causal attention of ``q`` [N·S, H·D] over ``k`` / ``v`` [N·S, kv_heads·D], N sequences of S tokens: token i sees
    token j ≤ i if i − j < ``window`` or j < ``sinks`` (≤ 64). Query head h reads key/value head h // (H / kv_heads).

    ``mask`` [N, S] (bool or integer, nonzero = a token): what is no token is neither a key nor a query — its output row
    is zero, its gradients are zero, and what its rows hold (NaN included) reaches nothing. Distances and sinks count
    positions, so pad on the right. ``bias`` [H, buckets] or per-client [C, H, buckets] (fp32; sequences [c·N/C,
    (c+1)·N/C) are client c's) is added to the scaled scores by :func:`relative_bucket_starts`' bucket of i − j.
    ``scale``: 1/√D unless given. Gradients: q, k, v (at their type) and bias (fp32).

    Biases beyond ±2.08e38 count as one. A bias of −inf takes its bucket away; a row all of whose scores are −inf has no
    softmax: it is NaN, and so are the gradients of what it sees. A non-finite value in a real token's rows reaches
    every row that sees the token, and may reach others near it."""
    D, H, KV, W, sinks = _common(q, k, v, H, kv_heads, window, sinks)
    S = int(S)
    if S < 1 or q.shape[0] % S:
        raise ValueError(f"{q.shape[0]} rows are no whole sequences of {S} tokens")
    N = q.shape[0] // S
    if N * H * S > _I32 or S > 2 ** 30:
        raise ValueError(f"{N} sequences · {H} heads · {S} tokens: at most 2^31 − 1 in all, 2^30 a sequence")
    if mask is not None:
        if mask.shape != (N, S) or mask.dtype.is_floating_point or mask.dtype.is_complex or mask.device != q.device:
            raise ValueError(f"mask: bool or integer [{N}, {S}] on {q.device} expected, got {mask.dtype} "
                             f"{tuple(mask.shape)} on {mask.device}")
    table = _bias(bias, N, H, max_distance, q.device)
    scale = _scale(scale, D)
    if not use_native(q):
        return _window_ref(q, k, v, S, H, KV, W, sinks, mask, table, max_distance, scale)
    if mask is not None:
        mask = (mask if mask.dtype == torch.bool else mask != 0).contiguous().view(torch.uint8)
    train = torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or
                                         (table is not None and table.requires_grad))
    cfg = (D, N, S, H, KV, min(W, S), min(sinks, S), scale, q.dtype == torch.float32,
           *((0, 0, 0) if table is None else (table.shape[0], table.shape[2], int(max_distance))), train)
    if train:
        return _WindowAttention.apply(q, k, v, table, mask, cfg)
    tab = None if table is None else table.contiguous()
    return _forward(_aligned(q), _aligned(k), _aligned(v), mask, tab, cfg, False, False)[0]


# ---------------------------------------------------------------------------------------------------------- serving
def _cache(k_cache, v_cache, B, KV, D, slots, dtype, device):
    for t, n in ((k_cache, "k_cache"), (v_cache, "v_cache")):
        if tuple(t.shape) != (B, slots, KV * D) or t.dtype != dtype or t.device != device:
            raise ValueError(f"{n}: {dtype} [{B}, {slots}, {KV * D}] on {device} expected, got {t.dtype} "
                             f"{tuple(t.shape)} on {t.device}")
        if not t.is_contiguous() or t.data_ptr() % 16:
            raise ValueError(f"{n}: contiguous, 16-byte aligned memory expected (it is updated in place)")
        if t.requires_grad:
            raise ValueError(f"{n} takes no gradient")
    size = k_cache.numel() * k_cache.element_size()
    if abs(k_cache.data_ptr() - v_cache.data_ptr()) < size:
        raise ValueError("k_cache and v_cache are the same memory")
    return k_cache.data_ptr(), v_cache.data_ptr(), size


def _apart(t, caches):
    """The rows, or a copy of rows that lie in a cache, which the call writes while it reads them."""
    p = t.data_ptr()
    span = ((t.shape[0] - 1) * t.stride(0) + (t.shape[1] - 1) * t.stride(1) + 1) * t.element_size()
    k, v, size = caches
    return t.clone() if -span < p - k < size or -span < p - v < size else t


def _pos(pos, B, device, name):
    if pos.shape != (B,) or pos.dtype != torch.int32 or pos.device != device:
        raise ValueError(f"{name}: int32 [{B}] on {device} expected, got {pos.dtype} {tuple(pos.shape)} on {pos.device}")
    return pos.contiguous()


def _slot_tokens(pos, slots, window, sinks):
    """The token in every slot once token ``pos`` [B] is there, −1 where there is none: [B, slots]."""
    pos = pos.long().view(-1, 1)
    s = torch.arange(slots, device=pos.device).view(1, -1)
    ring = pos - (pos - s) % window
    ring = torch.where((pos >= sinks) & (ring >= sinks), ring, -1)
    return torch.where(s < sinks, torch.where(s <= pos, s, -1), ring)


def _step_ref(q, k, v, kc, vc, pos, H, KV, W, sinks, bias, max_distance, scale):
    B, n, D, ct = q.shape[0], kc.shape[1], q.shape[1] // H, _ct(q)
    tok = _slot_tokens(pos, n, W, sinks)
    p = pos.long().view(-1, 1)
    here = (tok == p) & (p >= 0)
    kc.copy_(torch.where(here.unsqueeze(-1), k.unsqueeze(1), kc))
    vc.copy_(torch.where(here.unsqueeze(-1), v.unsqueeze(1), vc))
    see = (tok >= 0) & (p >= 0)
    zero = torch.zeros((), dtype=ct, device=q.device)
    kh, vh = (torch.where(see.view(B, n, 1, 1), t.to(ct).view(B, n, KV, D), zero).transpose(1, 2)
              .repeat_interleave(H // KV, 1) for t in (kc, vc))
    s = (q.to(ct).view(B, H, 1, D) @ kh.transpose(-1, -2)).squeeze(2) * scale
    if bias is not None:
        b = relative_bucket((p - tok).clamp_min(0), bias.shape[-1], max_distance)                     # [B, n]
        tab = bias.to(ct).repeat_interleave(B // bias.shape[0], 0)
        s = s + tab.gather(2, b.unsqueeze(1).expand(B, H, n))
    s = s.masked_fill(~see.unsqueeze(1), float("-inf")).masked_fill(~see.any(1).view(B, 1, 1), 0.0)
    w = torch.where(see.unsqueeze(1), torch.softmax(s, -1), zero)
    return (w.unsqueeze(2) @ vh).reshape(B, H * D).to(q.dtype)


@functools.lru_cache(maxsize=256)
def _step_plan(B, H, KV, W, sinks, scale, threads, C, buckets, max_distance):
    # enough workgroups for 256 CUs, of at least one 32-slot tile a wave
    n, wgs = W + sinks, B * KV * -(-(H // KV) // 32)
    tiles = -(-n // 128)
    splits = max(1, min(tiles, -(-512 // wgs)))
    per = -(-tiles // splits) * 128
    splits = -(-n // per)
    if threads * wgs * splits > MAX_THREADS or B * H > _I32 or n > 2 ** 30:
        raise ValueError(f"{B} sequences of {H} heads and {n} slots are too many for one call")
    a = _StepArgs(B=B, H=H, KV=KV, C=C, W=W, sinks=sinks, NB=buckets, splits=splits, per=per, scale=scale)
    if buckets:
        a.maxd = max_distance
        a.start[:buckets] = relative_bucket_starts(buckets, max_distance)
    return a


def window_attention_step(q, k, v, k_cache, v_cache, pos, H: int, window: int, sinks: int = 0, kv_heads: int = None,
                          bias: torch.Tensor = None, max_distance: int = 128, scale: float = None):
    """:func:`window_attention` of one new token per sequence: ``q`` [B, H·D], ``k`` / ``v`` [B, kv_heads·D] are its
    rows, ``pos`` int32 [B] its position (the number of tokens before it). ``k_cache`` / ``v_cache`` [B, sinks + window,
    kv_heads·D] hold token t < sinks in slot t and token t in slot sinks + (t − sinks) % window: the new token's rows are
    written there (over the token that leaves the window) and the output [B, H·D] is returned. A sequence with
    ``pos`` < 0 is idle: its cache stays as it is and its output is zero. Slots that hold no token yet are not read. The
    caller counts ``pos`` on, once per token for all layers; no gradient."""
    D, H, KV, W, sinks = _common(q, k, v, H, kv_heads, window, sinks)
    B, n = q.shape[0], W + sinks
    caches = _cache(k_cache, v_cache, B, KV, D, n, q.dtype, q.device)
    pos = _pos(pos, B, q.device, "pos")
    table = _bias(bias, B, H, max_distance, q.device)
    scale = _scale(scale, D)
    if (q.requires_grad or k.requires_grad or v.requires_grad or (bias is not None and bias.requires_grad)) and \
            torch.is_grad_enabled():
        raise ValueError("window_attention_step computes no gradient: call it under torch.no_grad()")
    if B == 0:
        return torch.empty(B, H * D, dtype=q.dtype, device=q.device)
    if not use_native(q):
        q, k, v = (_apart(t, caches) for t in (q, k, v))
        return _step_ref(q, k, v, k_cache, v_cache, pos, H, KV, W, sinks, table, max_distance, scale)
    o = torch.empty(B, H * D, dtype=q.dtype, device=q.device)
    q, k, v = _aligned(q), _aligned(k), _aligned(v)
    tab = None if table is None else table.contiguous()
    threads = 128 if D == 128 and q.dtype == torch.float32 else 256
    plan = _step_plan(B, H, KV, W, sinks, scale, threads, *((1, 0, 0) if tab is None else
                                                   (tab.shape[0], tab.shape[2], int(max_distance))))
    a = _StepArgs.from_buffer_copy(plan)
    a.q, a.k, a.v, a.kc, a.vc = ptr_read(q), ptr_read(k), ptr_read(v), ptr(k_cache), ptr(v_cache)
    a.o, a.pos, a.bias = ptr(o), ptr_read(pos), ptr_read(tab)
    a.ldq, a.ldk, a.ldv = q.stride(0), k.stride(0), v.stride(0)
    if a.splits > 1:
        part = torch.empty(B * H * a.splits * (D + 2), dtype=torch.float32, device=q.device)
        a.pacc = ptr(part)
        a.pml = a.pacc + 4 * B * H * a.splits * D
    if not launch("fa_window_step", a, (q.dtype == torch.bfloat16, D), q.device, _ROWS_IN_CACHE):
        q, k, v = q.clone(), k.clone(), v.clone()
        a.q, a.k, a.v = ptr_read(q), ptr_read(k), ptr_read(v)
        a.ldq, a.ldk, a.ldv = q.stride(0), k.stride(0), v.stride(0)
        launch("fa_window_step", a, (q.dtype == torch.bfloat16, D), q.device)
    return o


def window_cache_fill(k, v, S: int, k_cache, v_cache, window: int, sinks: int = 0, lengths: torch.Tensor = None):
    """Puts a prompt's rows ``k`` / ``v`` [B·S, kv_heads·D] into the caches of :func:`window_attention_step`, as its
    steps would have left them after token ``lengths[b]`` − 1 (int32 [B], within [0, S]; all S tokens if not given).
    Slots that hold none of these tokens stay as they were."""
    if k_cache.dim() != 3:
        raise ValueError(f"k_cache: [B, sinks + window, kv_heads · D] expected, got {tuple(k_cache.shape)}")
    B, S, W, sinks, width = k_cache.shape[0], int(S), int(window), int(sinks), k_cache.shape[2]
    if not 1 <= W <= _I32 or not 0 <= sinks <= MAX_SINKS or S < 1:
        raise ValueError(f"window ≥ 1, sinks in [0, {MAX_SINKS}] and S ≥ 1 expected, got {window}, {sinks}, {S}")
    for t, n in ((k, "k"), (v, "v")):
        _rows(t, 1, n, B * S, k_cache.dtype, k_cache.device)
        if t.shape[1] != width or width % 64:
            raise ValueError(f"{n}: rows of the cache's {width} columns expected, got {t.shape[1]}")
    caches = _cache(k_cache, v_cache, B, 1, width, W + sinks, k.dtype, k.device)
    if lengths is not None:
        lengths = _pos(lengths, B, k.device, "lengths")
    if B == 0:
        return
    with torch.no_grad():
        k, v = _apart(k, caches), _apart(v, caches)
        if not use_native(k):
            last = (torch.full((B,), S, device=k.device) if lengths is None else lengths.clamp(0, S)) - 1
            tok = _slot_tokens(last, W + sinks, W, sinks)
            at = tok.clamp_min(0) + torch.arange(B, device=k.device).view(B, 1) * S
            for t, c in ((k, k_cache), (v, v_cache)):
                c.copy_(torch.where((tok >= 0).unsqueeze(-1), t[at], c))
            return
        k, v = _aligned(k), _aligned(v)
        e = 16 // k.element_size()
        with torch.cuda.device(k.device):
            rc = _fn("fa_window_fill")(_pr(k), _pr(v), _i64(k.stride(0) // e), _i64(v.stride(0) // e), _p(k_cache),
                                       _p(v_cache), _pr(lengths), _c.c_int(B), _c.c_int(S), _c.c_int(W),
                                       _c.c_int(sinks), _c.c_int(width // e), _stream(k))
            _check(rc, "fa_window_fill")
