"""Window attention kernels (``csrc/window_kernels.hip``) against the definition in 64 bits, element by element, within
bounds counted from the roundings that the kernels make — worst cases, from the absolute values of the same inputs:

u = 2^-24 (fp32 sums), r = half a step of the storage type (2^-8 for bf16, 0 for fp32 beyond u).
* a score of D products: (D + 4) u Σ|q||k| scale, and 8 u of the largest |score| of the row for its scaling, the bias,
  the subtraction of the maximum and the exponential (twice that much for the saved log-sum-exp of the backward);
* a probability: its score's error and the row's largest (through the sum), n + 8 roundings of the sum of n terms;
* o: those times |v|, the rounding r of the probabilities, n + 2 sums, the rounding of the result;
* D = dO·o inherits o's error as stored (with a gradient of the bias r²: the roundings' leftovers are kept);
* dS = p (dP − D): the errors of the three, 4 u; dq, dk, dv: their factors' errors, r for the rounding of the
  probabilities or dS to the storage type, n sums, the rounding of the result; dbias: 256 u for its sums."""
import math

import pytest
import torch

from fedml_amd import ops
from fedml_amd.ops import window_ops as W

pytestmark = pytest.mark.gpu
dev = "cuda"
U = 2.0 ** -24


def half(dtype):
    return torch.finfo(dtype).eps / 2


def _oracle(q, k, v, do, S, H, KV, window, sinks, mask, bias, M, scale, dtype, frozen=False):
    """[(value, bound)] of o, dq, dk, dv(, dbias), token-major, in 64 bits on the CPU."""
    N, D, G = q.shape[0] // S, q.shape[1] // H, H // KV
    r = half(dtype) if dtype == torch.bfloat16 else 0.0
    rs = half(dtype)                                       # storing the result
    real = torch.ones(N, S, dtype=torch.bool) if mask is None else mask.cpu().bool()
    z = torch.zeros((), dtype=torch.float64)

    def heads(t, h):
        t = t.detach().cpu().double().view(N, S, h, D)
        return torch.where(real.view(N, S, 1, 1), t, z).transpose(1, 2)

    qh, gh = heads(q, H), heads(do, H)
    kh, vh = (heads(t, KV).repeat_interleave(G, 1) for t in (k, v))
    i = torch.arange(S)
    d = i.view(S, 1) - i
    see = (((d >= 0) & ((d < window) | (i < sinks))) & real.view(N, 1, S) & real.view(N, S, 1)).unsqueeze(1)
    s, a = qh @ kh.mT * scale, qh.abs() @ kh.abs().mT * abs(scale)
    if bias is not None:
        C, NB = bias.shape[0], bias.shape[-1]
        of = W.relative_bucket(d.clamp_min(0), NB, M)
        s = s + bias.detach().cpu().double()[..., of].repeat_interleave(N // C, 0)
    s = torch.where(see, s, z - math.inf)
    n = see.sum(-1, keepdim=True)
    top = torch.where(n > 0, s.amax(-1, keepdim=True), z)
    p = torch.where(see, (s - top).exp(), z)
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-300)
    big = torch.where(see, s.abs(), z).amax(-1, keepdim=True)
    es = torch.where(see, (D + 4) * U * a + 16 * U * (big + 1), z)
    rp = es + es.amax(-1, keepdim=True) + (n + 8) * U
    o = p @ vh
    exact = bias is not None and not frozen
    ro = r * r if exact else r
    eo = (p * (rp + ro)) @ vh.abs() + (n + 2) * U * (p @ vh.abs())
    dp, dpa = gh @ vh.mT, gh.abs() @ vh.abs().mT
    dd = (gh * o).sum(-1, keepdim=True)
    ed = (gh.abs() * (eo + (r * r if exact else rs) * o.abs())).sum(-1, keepdim=True) + \
        (2 * D + 2) * U * (gh.abs() * o.abs()).sum(-1, keepdim=True)
    ds = p * (dp - dd)
    eds = ds.abs() * rp + p * ((D + 2) * U * dpa + ed) * (1 + rp) + 4 * U * p * (dp.abs() + dd.abs())
    eds = torch.where(see, eds, z)
    dq = ds @ kh * scale
    edq = ((eds + r * ds.abs() + (n + 2) * U * ds.abs()) @ kh.abs()) * abs(scale)
    m = see.sum(-2).unsqueeze(-1) * G + 2
    dk = ds.mT @ qh * scale
    edk = ((eds + r * ds.abs()).mT @ qh.abs() + m * U * (ds.abs().mT @ qh.abs())) * abs(scale)
    dv = p.mT @ gh
    edv = (p * (rp + r)).mT @ gh.abs() + m * U * (p.mT @ gh.abs())

    def rows(t, h):
        return t.transpose(1, 2).reshape(N * S, h * D)

    def shared(t):
        return t.view(N, KV, G, S, D).sum(2)

    def out(t, e, h):
        return rows(t, h), rows(e, h) + rs * (rows(t, h).abs() + rows(e, h)) + 1e-30

    res = [out(o, eo, H), out(dq, edq, H), out(shared(dk), shared(edk), KV), out(shared(dv), shared(edv), KV)]
    if bias is not None:
        def buckets(t):
            return torch.stack([torch.where(of == b, t, z).sum((-1, -2)) for b in range(NB)], -1) \
                .view(C, N // C, H, NB).sum(1)
        db, e = buckets(ds), buckets(eds + 256 * U * ds.abs())
        res.append((db, e + U * db.abs() + 1e-30))
    return res


def _within(got, want, what):
    value, bound = want
    assert got.shape == value.shape, what
    err = (got.detach().cpu().double() - value).abs()
    assert torch.isfinite(got).all(), what
    worst = (err / bound).max().item() if err.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.3g} of the bound"


def _data(N, S, H, KV, D, dtype, seed=0, spread=1.5):
    gen = torch.Generator(device=dev).manual_seed(seed)

    def normal(h, s=1.0):
        return (torch.randn(N * S, h * D, generator=gen, device=dev) * s).to(dtype)

    return normal(H, spread), normal(KV), normal(KV), normal(H)


def _mask(kind, N, S):
    if kind is None:
        return None
    gen = torch.Generator().manual_seed(11)
    if kind == "right":
        n = torch.randint(0, S + 1, (N,), generator=gen)
        n[0] = S
        m = torch.arange(S) < n.view(N, 1)
    else:                                                  # holes anywhere, the sinks and whole tiles among them
        m = torch.rand(N, S, generator=gen) > 0.3
        m[N // 2, : S // 2] = False
    return m.to(dev)


CASES = [  # N, S, H, KV, D, window, sinks, mask, C, NB, M
    (1, 1, 1, 1, 64, 1, 0, None, 0, 0, 0), (2, 2, 2, 1, 64, 1, 1, None, 0, 0, 0), (2, 31, 2, 2, 64, 8, 0, "holes", 0, 0, 0),
    (3, 33, 2, 1, 128, 5, 2, None, 3, 8, 16), (2, 64, 4, 2, 64, 100, 0, "right", 0, 0, 0),
    (2, 65, 1, 1, 64, 64, 64, None, 0, 0, 0), (1, 96, 3, 1, 128, 33, 33, "holes", 0, 0, 0),
    (2, 127, 2, 2, 64, 32, 1, "right", 2, 16, 64), (1, 129, 6, 2, 64, 16, 4, None, 1, 32, 128),
    (2, 200, 2, 1, 128, 1, 3, "right", 0, 0, 0), (1, 300, 2, 1, 64, 300, 0, None, 1, 2, 1024),
    (1, 300, 2, 2, 64, 47, 64, None, 1, 128, 300), (4, 61, 2, 1, 64, 9, 40, "right", 4, 5, 9),
    (1, 257, 8, 1, 128, 64, 0, None, 1, 8, 32), (2, 300, 2, 1, 64, 31, 31, "holes", 2, 3, 500),
    # enough heads for workgroups of 128 queries at fp32 too
    (40, 130, 8, 4, 64, 48, 3, "right", 2, 16, 64), (30, 140, 8, 2, 128, 33, 64, "holes", 0, 0, 0),
    (26, 150, 9, 3, 128, 150, 0, None, 1, 32, 128)]


def _call(ops_args, q, k, v, bias, do):
    S, H, window, sinks, KV, mask, M, scale = ops_args
    leaves = [t.detach().requires_grad_() for t in (q, k, v)] + ([bias.detach().requires_grad_()] if bias is not None else [])
    o = ops.window_attention(*leaves[:3], S, H, window, sinks, kv_heads=KV, mask=mask,
                             bias=leaves[3] if bias is not None else None, max_distance=M, scale=scale)
    return [o, *torch.autograd.grad(o, leaves, do)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
def test_forward_and_gradients(case, dtype):
    N, S, H, KV, D, window, sinks, kind, C, NB, M = case
    q, k, v, do = _data(N, S, H, KV, D, dtype)
    mask = _mask(kind, N, S)
    bias = torch.randn(C, H, NB, generator=torch.Generator().manual_seed(3)).to(dev) if C else None
    scale = 0.11 if D == 64 else None
    got = _call((S, H, window, sinks, KV, mask, M, scale), q, k, v, bias, do)
    want = _oracle(q, k, v, do, S, H, KV, window, sinks, mask, bias, M, scale or D ** -0.5, dtype)
    for g, w, name in zip(got, want, ("o", "dq", "dk", "dv", "dbias")):
        _within(g, w, name)
    with torch.no_grad():                                  # without a graph: the same bits
        o = ops.window_attention(q, k, v, S, H, window, sinks, kv_heads=KV, mask=mask, bias=bias, max_distance=M,
                                 scale=scale)
    if bias is None or dtype == torch.float32:
        assert torch.equal(o, got[0])
    else:
        _within(o, (want[0][0], want[0][1] + half(dtype) * (want[0][0].abs() + 4)), "o")
    again = _call((S, H, window, sinks, KV, mask, M, scale), q, k, v, bias, do)
    for g, a, name in zip(got, again, ("o", "dq", "dk", "dv", "dbias")):
        assert torch.equal(g, a), f"{name} differs from call to call"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("N,S,H,KV,D,window,sinks,kind,C", [
    (1, 2900, 2, 1, 64, 40, 3, None, 1), (1, 1100, 2, 2, 128, 70, 64, "right", 0), (2, 1400, 14, 7, 64, 100, 33, "right", 2),
    (1, 1200, 30, 10, 128, 129, 1, "holes", 0)])
def test_long_rows_against_short_windows(N, S, H, KV, D, window, sinks, kind, C, dtype):
    """Many more tokens than the window: the sinks' gradients come from chunks of queries."""
    q, k, v, do = _data(N, S, H, KV, D, dtype, 5)
    bias = torch.randn(C, H, 16, generator=torch.Generator().manual_seed(3)).to(dev) if C else None
    mask = _mask(kind, N, S)
    got = _call((S, H, window, sinks, KV, mask, 100, None), q, k, v, bias, do)
    want = _oracle(q, k, v, do, S, H, KV, window, sinks, mask, bias, 100, D ** -0.5, dtype)
    for g, w, name in zip(got, want, ("o", "dq", "dk", "dv", "dbias")):
        _within(g, w, name)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_padding_reaches_nothing(dtype):
    N, S, H, KV, D = 3, 150, 2, 1, 64
    q, k, v, do = _data(N, S, H, KV, D, dtype, 6)
    mask = torch.arange(S, device=dev) < torch.tensor([[150], [77], [0]], device=dev)
    args = (S, H, 50, 4, KV, mask, 16, None)
    bias = torch.randn(3, H, 8, generator=torch.Generator().manual_seed(3)).to(dev)
    want = _call(args, q, k, v, bias, do)
    for fill in (float("nan"), float("inf")):
        bad = [t.clone() for t in (q, k, v, do)]
        for t in bad:
            t.view(N, S, -1)[~mask] = fill
        got = _call(args, *bad[:3], bias, bad[3])
        for g, w in zip(got, want):
            assert torch.equal(g, w)
    for g in got[:4]:
        assert not g.view(N, S, -1)[~mask].any()
    assert not got[4][2].any()                             # a client of no tokens


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_layouts(dtype):
    """Column slices of a fused projection, rows off their alignment, other strides, one row for all, another stream."""
    N, S, H, KV, D = 2, 70, 2, 1, 64
    q, k, v, do = _data(N, S, H, KV, D, dtype, 7)
    args = (S, H, 20, 2, KV, None, 128, None)
    want = _call(args, q, k, v, None, do)
    fused = torch.cat([q, k, v], 1)
    odd = torch.zeros(N * S, 4 * D + 3, dtype=dtype, device=dev)
    odd[:, 1:1 + 4 * D] = fused
    for f in (fused, odd[:, 1:1 + 4 * D]):
        got = _call(args, f[:, :2 * D], f[:, 2 * D:3 * D], f[:, 3 * D:], None, do)
        assert all(torch.equal(g, w) for g, w in zip(got, want))
    t = [x.t().contiguous().t() for x in (q, k, v)]        # columns first
    got = _call(args, *t, None, do.t().contiguous().t())
    assert all(torch.equal(g, w) for g, w in zip(got, want))
    one = q[:1].expand(N * S, -1)
    got = _call(args, one, k, v, None, do[:1].expand(N * S, -1))
    ref = _call(args, one.contiguous(), k, v, None, do[:1].repeat(N * S, 1))
    assert all(torch.equal(g, w) for g, w in zip(got, ref))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _call(args, q, k, v, None, do)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(g, w) for g, w in zip(got, want))
    m = torch.ones(N, 2 * S, dtype=torch.int64, device=dev)[:, ::2] * 5        # a mask of whole numbers, strided
    got = _call((S, H, 20, 2, KV, m, 128, None), q, k, v, None, do)
    assert all(torch.equal(g, w) for g, w in zip(got, want))


def test_shared_bias_and_shared_inputs():
    """One table for all clients, and one tensor as q, k and v: gradients add up."""
    N, S, H, D = 4, 40, 2, 64
    q, _, _, do = _data(N, S, H, H, D, torch.float32, 8)
    table = torch.randn(H, 8, generator=torch.Generator().manual_seed(3)).to(dev).requires_grad_()
    x = q.clone().requires_grad_()
    o = ops.window_attention(x, x, x, S, H, 11, 1, bias=table, max_distance=20)
    gx, gt = torch.autograd.grad(o, (x, table), do)
    parts = _call((S, H, 11, 1, H, None, 20, None), q, q, q, table.detach().expand(N, H, 8).contiguous(), do)
    assert torch.equal(o, parts[0])
    assert torch.allclose(gx, parts[1] + parts[2] + parts[3], rtol=0, atol=4 * U * 64)       # three sums of O(10)
    assert torch.allclose(gt, parts[4].sum(0), rtol=0, atol=float(parts[4].abs().sum(0).max()) * 16 * U)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("N,S", [(1, 40), (2, 150), (40, 130)])
def test_frozen_bias_still_counts(N, S, dtype):
    """A bias that takes no gradient is in the probabilities of every gradient; and a bias alone gets its own."""
    H, D, window, sinks, M = 8, 64, 30, 2, 16
    q, k, v, do = _data(N, S, H, H, D, dtype, 12)
    bias = 2 * torch.randn(1, H, 8, generator=torch.Generator().manual_seed(3)).to(dev)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    o = ops.window_attention(*leaves, S, H, window, sinks, bias=bias, max_distance=M)
    got = [o, *torch.autograd.grad(o, leaves, do)]
    want = _oracle(q, k, v, do, S, H, H, window, sinks, None, bias, M, D ** -0.5, dtype, frozen=True)
    for g, w, name in zip(got, want, ("o", "dq", "dk", "dv")):
        _within(g, w, name)
    table = bias.clone().requires_grad_()
    o = ops.window_attention(q, k, v, S, H, window, sinks, bias=table, max_distance=M)
    want = _oracle(q, k, v, do, S, H, H, window, sinks, None, bias, M, D ** -0.5, dtype)
    _within(torch.autograd.grad(o, table, do)[0], want[4], "dbias")


def test_what_a_masked_query_would_have_met():
    """An infinite value of a real token: rows that are no token stay zero, forward and backward."""
    N, S, H, D = 1, 70, 1, 64
    q, k, v, do = _data(N, S, H, H, D, torch.float32, 13)
    v[3, 5] = float("inf")
    mask = torch.ones(N, S, dtype=torch.bool, device=dev)
    mask[0, 40:] = False
    got = _call((S, H, 100, 0, H, mask, 128, None), q, k, v, None, do)
    for g in got:
        assert not g[40:].any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("N,S,H,KV,D,window,sinks,whole", [
    (2, 40, 2, 1, 64, 9, 0, False), (1, 300, 2, 2, 128, 70, 3, False), (1, 700, 4, 2, 64, 33, 2, True),
    (40, 130, 8, 4, 64, 48, 0, True)])
def test_rows_of_minus_infinity(N, S, H, KV, D, window, sinks, whole, dtype):
    """A bias of −inf takes a bucket (or all of a head's) away. A row that keeps a key has the bits that e^−10000 gives,
    which is 0 in 32 bits; a row that keeps none is 0 / 0, as in the CPU form, and so is all that it sees."""
    q, k, v, do = _data(N, S, H, KV, D, dtype, 14)
    bias = torch.randn(1, H, 8, generator=torch.Generator().manual_seed(3))
    bias[0, 0, 0] = bias[0, H - 1, 2] = -math.inf
    if whole:
        bias[0, 1] = -math.inf
    args = (S, H, window, sinks, KV, None, 32, None)
    got = _call(args, q, k, v, bias.to(dev), do)
    ref = _call(args, *(t.cpu().double() for t in (q, k, v)), bias.double(), do.cpu().double())
    near = _call(args, q, k, v, bias.clamp_min(-1e4).to(dev), do)
    for g, r, f, name in zip(got, ref, near, ("o", "dq", "dk", "dv", "dbias")):
        nan = torch.isnan(r)
        assert nan.any() and torch.equal(torch.isnan(g).cpu(), nan), name
        assert torch.equal(g[~nan.to(dev)], f[~nan.to(dev)]), name
    with torch.no_grad():
        o = ops.window_attention(q, k, v, S, H, window, sinks, kv_heads=KV, bias=bias.to(dev), max_distance=32)
    assert torch.equal(torch.isnan(o).cpu(), torch.isnan(ref[0]))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("B,window,sinks", [(3, 9, 2), (2, 700, 4), (600, 40, 0)])
def test_step_of_minus_infinity(B, window, sinks, dtype):
    """The same for one token: a head whose table is all −inf gives NaN, an idle sequence's zeros stay zeros."""
    H, D, n = 2, 64, window + sinks
    gen = torch.Generator(device=dev).manual_seed(4)
    q, k, v, kc, vc = (torch.randn(*s, generator=gen, device=dev).to(dtype)
                       for s in (3 * [(B, H * D)] + 2 * [(B, n, H * D)]))
    bias = torch.randn(H, 8, generator=gen, device=dev)
    bias[1] = -math.inf
    pos = torch.full((B,), n + 5, dtype=torch.int32, device=dev)
    pos[0], pos[1] = -1, 3
    o = ops.window_attention_step(q, k, v, kc, vc, pos, H, window, sinks, bias=bias, max_distance=32).view(B, H, D)
    assert not o[0].any() and torch.isnan(o[1:, 1]).all() and torch.isfinite(o[1:, 0]).all()


def _apart(N, S, H, KV, D, dtype, seed):
    """Inputs whose scores are all exactly zero: queries and keys share no dim."""
    q, k, v, do = _data(N, S, H, KV, D, dtype, seed)
    q.view(N * S, H, D)[..., D // 2:] = 0
    k.view(N * S, KV, D)[..., :D // 2] = 0
    return q, k, v, do


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("N,S,H,KV,D,window,sinks,maxd", [
    (2, 40, 2, 1, 64, 9, 0, 32), (1, 300, 3, 3, 128, 70, 3, 32), (1, 700, 4, 2, 64, 33, 2, 16),
    (40, 130, 8, 4, 64, 48, 0, 32)])
def test_bias_of_the_lowest_and_highest_value(N, S, H, KV, D, window, sinks, maxd, dtype):
    """A table with the type's lowest value: a row that sees nothing else is shared out evenly, forward and backward (a
    score's few units are nothing to it: here they are zero). −200 is the same in 64 bits, up to e^−200. The highest
    value, in a bucket of the third head, takes all of a row that sees it, as 200 does."""
    q, k, v, do = _apart(N, S, H, KV, D, dtype, 15)
    low = torch.zeros(1, H, 8)
    low[0, 0, :3] = low[0, 1] = -200.0
    if H > 2:
        low[0, 2, 3] = 200.0
    top = torch.finfo(torch.float32).max
    bias = torch.where(low < 0, -top, torch.where(low > 0, top, 0.0))
    got = _call((S, H, window, sinks, KV, None, maxd, None), q, k, v, bias.to(dev), do)
    want = _oracle(q, k, v, do, S, H, KV, window, sinks, None, low, maxd, D ** -0.5, dtype)
    for g, w, name in zip(got, want, ("o", "dq", "dk", "dv", "dbias")):
        _within(g, w, name)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("B,window,sinks", [(3, 9, 2), (2, 700, 4), (600, 40, 0)])
def test_step_bias_of_the_lowest_value(B, window, sinks, dtype):
    H, D, n = 2, 64, window + sinks
    q, k, v, _ = _apart(B, 1, H, H, D, dtype, 16)
    kc, vc = (t.view(B, n, H * D) for t in _apart(B, n, H, H, D, dtype, 17)[1:3])
    low = torch.zeros(H, 8, device=dev)
    low[0, :3] = low[1] = -200.0
    pos = (torch.arange(B, device=dev) * 7 % (2 * n)).to(torch.int32)
    o = ops.window_attention_step(q, k, v, kc, vc, pos, H, window, sinks, max_distance=32,
                                  bias=torch.where(low < 0, torch.finfo(torch.float32).min, low))
    _within(o, _step_bound(q, kc, vc, pos, H, H, window, sinks, low.unsqueeze(0), 32, D ** -0.5, dtype), "o")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("S,window,sinks", [(60, 60, 0), (150, 100, 4), (1200, 90, 3)])
def test_buckets_that_only_padding_reaches(S, window, sinks, dtype):
    """What a table holds for distances that no two tokens are apart reaches no gradient, as it reaches no output."""
    N, H, KV, D = 3, 4, 2, 64
    q, k, v, do = _data(N, S, H, KV, D, dtype, 18)
    mask = torch.arange(S, device=dev) < torch.tensor([[15], [9], [0]], device=dev)
    bias = torch.randn(1, H, 8, generator=torch.Generator().manual_seed(3)).to(dev)
    assert ops.relative_bucket_starts(8, 64)[6] > 14       # buckets 6 and 7 begin behind the longest sequence
    bias[..., 6:] = 0.0
    want = _call((S, H, window, sinks, KV, mask, 64, None), q, k, v, bias, do)
    for fill in (float("nan"), float("inf")):
        bias[..., 6:] = fill
        got = _call((S, H, window, sinks, KV, mask, 64, None), q, k, v, bias, do)
        for g, w, name in zip(got, want, ("o", "dq", "dk", "dv", "dbias")):
            assert torch.equal(g, w), name


def test_empty_batch():
    e = torch.zeros(0, 128, device=dev, requires_grad=True)
    b = torch.zeros(1, 2, 8, device=dev, requires_grad=True)
    o = ops.window_attention(e, e, e, 5, 2, 3, 1, bias=b)
    assert o.shape == (0, 128)
    g = torch.autograd.grad(o, (e, b), torch.zeros_like(o))
    assert g[0].shape == (0, 128) and not g[1].any()
    c = torch.zeros(0, 4, 128, device=dev)
    assert ops.window_attention_step(*(x.detach() for x in (e, e, e)), c, c.clone(),
                                     torch.zeros(0, dtype=torch.int32, device=dev), 2, 3, 1).shape == (0, 128)


def test_offsets_past_32_bits():
    """Rows of a fused buffer of more than 2^31 elements."""
    S, wide, D = 180000, 12288, 64
    buf = torch.empty(S, wide, dtype=torch.bfloat16, device=dev)
    assert buf.numel() > 2 ** 31
    q, k, v, do = _data(1, S, 1, 1, D, torch.bfloat16, 9)
    at = (wide - 3 * D, wide - 2 * D, wide - D)
    for t, c in zip((q, k, v), at):
        buf[:, c:c + D] = t
    args = (S, 1, 70, 4, 1, None, 128, None)
    got = _call(args, *(buf[:, c:c + D] for c in at), None, do)
    want = _call(args, q, k, v, None, do)
    assert all(torch.equal(g, w) for g, w in zip(got, want))


def test_captured_training_step_replays():
    N, S, H, KV, D = 2, 150, 4, 2, 64
    q, k, v, do = _data(N, S, H, KV, D, torch.bfloat16, 10)
    bias = torch.randn(2, H, 8, generator=torch.Generator().manual_seed(3)).to(dev)
    mask = _mask("right", N, S)
    args = (S, H, 40, 4, KV, mask, 32, None)
    static = [t.clone() for t in (q, k, v, bias, do)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _call(args, *static)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _call(args, *static)
    for seed in (20, 21, 22):
        new = (*_data(N, S, H, KV, D, torch.bfloat16, seed),)
        for t, x in zip(static, (*new[:3], bias * seed / 20, new[3])):
            t.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        want = _call(args, *(t.clone() for t in static))
        assert all(torch.equal(g, w) for g, w in zip(out, want))


# ---------------------------------------------------------------------------------------------------- one new token
def _step_bound(q, kc, vc, pos, H, KV, window, sinks, bias, M, scale, dtype):
    """(value, bound) of the output over the caches as they are after the step; bounds as above, with n + 64 sums."""
    B, n, D = q.shape[0], kc.shape[1], q.shape[1] // H
    r, rs = (half(dtype) if dtype == torch.bfloat16 else 0.0), half(dtype)
    tok = W._slot_tokens(pos.cpu(), n, window, sinks)
    p_ = pos.cpu().long().view(B, 1)
    see = ((tok >= 0) & (p_ >= 0)).view(B, 1, n)
    z = torch.zeros((), dtype=torch.float64)
    kh, vh = (torch.where(see.view(B, n, 1, 1), t.cpu().double().view(B, n, KV, D), z).transpose(1, 2)
              .repeat_interleave(H // KV, 1) for t in (kc, vc))
    qh = q.cpu().double().view(B, H, 1, D)
    s, a = (qh @ kh.mT).squeeze(2) * scale, (qh.abs() @ kh.abs().mT).squeeze(2) * scale
    if bias is not None:
        b = W.relative_bucket((p_ - tok).clamp_min(0), bias.shape[-1], M)
        s = s + bias.cpu().double().repeat_interleave(B // bias.shape[0], 0).gather(2, b.unsqueeze(1).expand(B, H, n))
    s = torch.where(see, s, z - math.inf)
    top = torch.where(see.any(-1, keepdim=True), s.amax(-1, keepdim=True), z)
    p = torch.where(see, (s - top).exp(), z)
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-300)
    es = torch.where(see, (D + 4) * U * a + 8 * U * (torch.where(see, s.abs(), z).amax(-1, keepdim=True) + 1), z)
    cnt = see.sum(-1, keepdim=True)
    rp = es + es.amax(-1, keepdim=True) + (cnt + 64) * U
    o = (p.unsqueeze(2) @ vh).reshape(B, H * D)
    e = ((p * (rp + r + (cnt + 64) * U)).unsqueeze(2) @ vh.abs()).reshape(B, H * D)
    return o, e + rs * (o.abs() + e) + 1e-30


STEPS = [  # B, H, KV, D, window, sinks, C, NB, M
    (1, 1, 1, 64, 1, 0, 0, 0, 0), (3, 2, 1, 64, 5, 2, 0, 0, 0), (9, 4, 4, 128, 64, 4, 3, 8, 16),
    (2, 40, 1, 64, 131, 64, 1, 32, 128), (5, 8, 2, 128, 700, 1, 5, 128, 1024), (40, 12, 12, 64, 260, 4, 0, 0, 0),
    (1, 70, 2, 128, 2049, 33, 1, 16, 64), (300, 4, 2, 64, 33, 0, 0, 0, 0)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("case", STEPS, ids=lambda c: "-".join(map(str, c)))
def test_step(case, dtype):
    B, H, KV, D, window, sinks, C, NB, M = case
    n = window + sinks
    gen = torch.Generator(device=dev).manual_seed(1)

    def normal(*s):
        return torch.randn(*s, generator=gen, device=dev).to(dtype)

    q, k, v, kc, vc = normal(B, H * D), normal(B, KV * D), normal(B, KV * D), normal(B, n, KV * D), normal(B, n, KV * D)
    bias = torch.randn(C, H, NB, generator=gen, device=dev) if C else None
    some = torch.randint(0, 3 * n, (B,), generator=gen, device=dev)
    for name, pos in (("first", 0), ("filling", n // 2), ("last sink", max(sinks - 1, 0)), ("full", n - 1),
                      ("round", n), ("idle", -1), ("far", 2 ** 31 - 1), ("mixed", some)):
        pos = torch.zeros(B, dtype=torch.int32, device=dev) + pos
        pos = pos.to(torch.int32)
        tok = W._slot_tokens(pos, n, window, sinks)
        a, b = (torch.where((tok >= 0).unsqueeze(-1), c, float("nan")).to(dtype) for c in (kc, vc))   # empty slots: NaN
        want_a, want_b = a.clone(), b.clone()
        o = ops.window_attention_step(q, k, v, a, b, pos, H, window, sinks, kv_heads=KV, bias=bias, max_distance=M)
        here = ((tok == pos.long().view(B, 1)) & (pos >= 0).view(B, 1)).unsqueeze(-1)
        for got, want, new in ((a, want_a, k), (b, want_b, v)):
            want = torch.where(here, new.unsqueeze(1), want)
            assert torch.equal(torch.nan_to_num(got, nan=777.0), torch.nan_to_num(want, nan=777.0)), name
        _within(o, _step_bound(q, a, b, pos, H, KV, window, sinks, bias, M, D ** -0.5, dtype), name)
        if name == "idle":
            assert not o.any()
        assert torch.equal(o, ops.window_attention_step(q, k, v, a, b, pos, H, window, sinks, kv_heads=KV, bias=bias,
                                                        max_distance=M)), name


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("S,window,sinks", [(1, 3, 0), (5, 8, 2), (50, 8, 2), (50, 64, 4), (200, 33, 64)])
def test_fill(S, window, sinks, dtype):
    B, width, n = 3, 192, window + sinks
    gen = torch.Generator(device=dev).manual_seed(2)
    k, v = (torch.randn(B * S, width, generator=gen, device=dev).to(dtype) for _ in range(2))
    for lengths in (None, torch.tensor([0, S, (S + 1) // 2], dtype=torch.int32, device=dev),
                    torch.tensor([-3, S + 9, 1], dtype=torch.int32, device=dev)):
        caches = [torch.full((B, n, width), 7.0, dtype=dtype, device=dev) for _ in range(2)]
        want = [c.cpu() for c in caches]
        ops.window_cache_fill(k, v, S, *caches, window, sinks, lengths)
        ops.window_cache_fill(k.cpu(), v.cpu(), S, *want, window, sinks, None if lengths is None else lengths.cpu())
        assert all(torch.equal(c.cpu(), w) for c, w in zip(caches, want))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_rows_that_lie_in_a_cache(dtype):
    """Rows of the caches as arguments: what they held before the call counts."""
    B, n, H, D = 40, 69, 2, 64
    both = torch.randn(2, B, n, H * D, generator=torch.Generator(device=dev).manual_seed(9), device=dev).to(dtype)
    pos = (torch.arange(B, device=dev) * 31 % (3 * n)).to(torch.int32)
    mine, ref = both.clone(), both.clone()
    o = ops.window_attention_step(mine[1, :, 3], mine[0, :, 5], mine[0, :, 7], *mine, pos, H, 64, 5)
    want = ops.window_attention_step(both[1, :, 3].clone(), both[0, :, 5].clone(), both[0, :, 7].clone(), *ref, pos, H,
                                     64, 5)
    assert torch.equal(o, want) and torch.equal(mine, ref)
    mine, ref = both.clone(), both.clone()
    ops.window_cache_fill(mine[1].view(B * n, -1), mine[0].view(B * n, -1), n, *mine, 64, 5)
    ops.window_cache_fill(both[1].view(B * n, -1).clone(), both[0].view(B * n, -1).clone(), n, *ref, 64, 5)
    assert torch.equal(mine, ref)


def test_cache_past_32_bits():
    """A cache of more than 2^31 elements: the last sequence's last slots are read and written."""
    B, KV, D, window = 2, 8, 128, 1_060_000
    kc, vc = (torch.zeros(B, window, KV * D, dtype=torch.bfloat16, device=dev) for _ in range(2))
    assert kc.numel() > 2 ** 31
    q = torch.ones(B, KV * D, dtype=torch.bfloat16, device=dev)
    v = torch.randn(B, KV * D, generator=torch.Generator(device=dev).manual_seed(1), device=dev).to(torch.bfloat16)
    kc[1, window - 2] = 8.0
    vc[1, window - 2] = 3.0
    pos = torch.tensor([window - 1, window - 1], dtype=torch.int32, device=dev)
    o = ops.window_attention_step(q, q * 8, v, kc, vc, pos, KV, window, kv_heads=KV)
    # scores 8·√128 = 90.5 at the two slots against 0 elsewhere: 10^6 e^-90 is nothing
    assert torch.equal(kc[:, window - 1], q * 8) and torch.equal(vc[:, window - 1], v)
    assert torch.equal(o[0], v[0])
    want = (v[1].double() + 3) / 2                          # probabilities of a half are exact
    assert ((o[1].double() - want).abs() <= half(torch.bfloat16) * want.abs() + 4 * U).all()


def test_step_in_a_graph_counts_on():
    B, H, D, window, sinks = 4, 2, 64, 9, 2
    gen = torch.Generator(device=dev).manual_seed(4)
    rows = [torch.randn(B, H * D, generator=gen, device=dev) for _ in range(3)]
    caches = [torch.zeros(B, window + sinks, H * D, device=dev) for _ in range(2)]
    pos = torch.zeros(B, dtype=torch.int32, device=dev)

    def step():
        o = ops.window_attention_step(*rows, *caches, pos, H, window, sinks)
        pos.add_(1)
        return o

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    pos.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    mine = [torch.zeros_like(c) for c in caches]
    for t in range(25):
        for i, r in enumerate(rows):
            r.copy_(torch.randn(B, H * D, generator=gen, device=dev))
        graph.replay()
        torch.cuda.synchronize()
        want = ops.window_attention_step(*rows, *mine, torch.full((B,), t, dtype=torch.int32, device=dev), H, window,
                                         sinks)
        assert torch.equal(out, want) and all(torch.equal(a, b) for a, b in zip(caches, mine)), t
