"""Window attention with sinks and bucketed bias on the CPU path: the plain-PyTorch form (the GPU tests' oracle) against
loops over tokens written from the definition, its gradients against differences, the form for one token against the
whole sequence, and every refusal."""
import math

import pytest
import torch

from fedml_amd import ops
from fedml_amd.ops import window_ops as W


def _bucket(d, NB, M):
    """The definition, by its inequality in whole numbers."""
    E = NB // 2
    n = NB - E
    return d if d < E else E + max(j for j in range(n) if d ** n >= M ** j * E ** (n - j))


def _loops(q, k, v, S, H, KV, window, sinks, mask, bias, M, scale):
    """The definition, token by token, in Python floats over fp64 rows."""
    N, D = q.shape[0] // S, q.shape[1] // H
    o = torch.zeros_like(q)
    for n in range(N):
        for h in range(H):
            kv = h // (H // KV)
            for i in range(S):
                if mask is not None and not mask[n, i]:
                    continue
                see = [j for j in range(i + 1) if (i - j < window or j < sinks) and (mask is None or mask[n, j])]
                row = q[n * S + i, h * D:(h + 1) * D]
                s = []
                for j in see:
                    x = scale * float(row @ k[n * S + j, kv * D:(kv + 1) * D])
                    if bias is not None:
                        x += float(bias[n // (N // bias.shape[0]), h, _bucket(i - j, bias.shape[-1], M)])
                    s.append(x)
                top = max(s)
                e = [math.exp(x - top) for x in s]
                for j, p in zip(see, e):
                    o[n * S + i, h * D:(h + 1) * D] += p / sum(e) * v[n * S + j, kv * D:(kv + 1) * D]
    return o


def _inputs(N, S, H, KV, D, seed=0, dtype=torch.float64):
    gen = torch.Generator().manual_seed(seed)
    return [torch.randn(N * S, h * D, generator=gen, dtype=torch.float64).to(dtype) for h in (H, KV, KV)]


@pytest.mark.parametrize("S,H,KV,window,sinks,holes,C,NB,M", [
    (1, 1, 1, 1, 0, False, 0, 0, 0), (9, 2, 1, 3, 2, False, 0, 0, 0), (12, 2, 2, 4, 1, True, 2, 8, 16),
    (40, 2, 1, 100, 64, False, 1, 4, 8), (40, 2, 1, 7, 5, True, 0, 0, 0)])
def test_reference_is_the_definition(S, H, KV, window, sinks, holes, C, NB, M):
    q, k, v = _inputs(2, S, H, KV, 64)
    mask = None
    if holes:
        mask = torch.rand(2, S, generator=torch.Generator().manual_seed(1)) > 0.4
        mask[1, S // 2:] = False
    bias = torch.randn(C, H, NB, generator=torch.Generator().manual_seed(2), dtype=torch.float64) if C else None
    o = ops.window_attention(q, k, v, S, H, window, sinks, kv_heads=KV, mask=mask, bias=bias, max_distance=M, scale=0.2)
    ref = _loops(q, k, v, S, H, KV, window, sinks, mask, bias, M, 0.2)
    assert torch.allclose(o, ref, rtol=0, atol=1e-12)          # 64 bits: sums of < 2^7 terms of order 1, 2^-53 each


def test_reference_gradients_are_differences():
    S, H, KV = 7, 2, 1
    q, k, v = (t.requires_grad_() for t in _inputs(2, S, H, KV, 64, 3))
    bias = torch.randn(2, H, 4, generator=torch.Generator().manual_seed(4), dtype=torch.float64).requires_grad_()
    mask = torch.ones(2, S, dtype=torch.bool)
    mask[1, 5:] = False
    assert torch.autograd.gradcheck(
        lambda *a: ops.window_attention(*a[:3], S, H, 3, 1, kv_heads=KV, mask=mask, bias=a[3], max_distance=6),
        (q, k, v, bias), fast_mode=True)
    shared = torch.zeros(H, 4, dtype=torch.float64, requires_grad=True)    # one table for all sequences
    assert torch.autograd.gradcheck(
        lambda b: ops.window_attention(q.detach(), k.detach(), v.detach(), S, H, 3, 1, kv_heads=KV, bias=b,
                                       max_distance=6), (shared,), fast_mode=True)


@pytest.mark.parametrize("NB,M", [(2, 2), (3, 9), (8, 16), (32, 128), (32, 256), (64, 512), (128, 1024), (5, 1000)])
def test_bucket_borders(NB, M):
    starts = ops.relative_bucket_starts(NB, M)
    assert len(starts) == NB and starts[0] == 0 and all(a <= b for a, b in zip(starts, starts[1:])) and starts[-1] <= M
    d = torch.arange(M + 50)
    got = W.relative_bucket(d, NB, M).tolist()
    assert got == [_bucket(x, NB, M) for x in d.tolist()]
    E = NB // 2
    for x in range(E + 1, M):      # and the formula in real numbers, away from its borders
        real = E + (NB - E) * math.log(x / E) / math.log(M / E)
        if abs(real - round(real)) > 1e-9:
            assert got[x] == min(NB - 1, math.floor(real))


def test_padding_reaches_nothing():
    S, H = 10, 2
    q, k, v = _inputs(2, S, H, H, 64, 5)
    mask = torch.ones(2, S, dtype=torch.bool)
    mask[0, 6:] = False
    mask[1] = False                                            # a sequence of no tokens
    bad = [t.clone() for t in (q, k, v)]
    for t in bad:
        t.view(2, S, -1)[~mask] = float("nan")
        t.requires_grad_()
    o = ops.window_attention(*bad, S, H, 4, 1, mask=mask)
    assert torch.equal(o.view(2, S, -1)[~mask], torch.zeros(S + 4, 2 * 64, dtype=torch.float64))
    alone = ops.window_attention(*(t[:6] for t in (q, k, v)), 6, H, 4, 1)
    assert torch.allclose(o[:6], alone, rtol=0, atol=1e-14)
    g = torch.ones_like(o)
    g.view(2, S, -1)[~mask] = float("nan")
    for t in torch.autograd.grad(o, bad, g):
        assert torch.isfinite(t).all() and not t.view(2, S, -1)[~mask].any()


@pytest.mark.parametrize("window,sinks,KV", [(4, 2, 1), (1, 0, 2), (5, 0, 2), (64, 3, 1), (3, 30, 2)])
def test_steps_are_the_rows_of_the_whole(window, sinks, KV):
    S, H, D, M = 20, 2, 64, 8
    q, k, v = _inputs(2, S, H, KV, D, 6)
    bias = torch.randn(2, H, 6, generator=torch.Generator().manual_seed(7), dtype=torch.float64)
    whole = ops.window_attention(q, k, v, S, H, window, sinks, kv_heads=KV, bias=bias, max_distance=M).view(2, S, -1)
    rows = [t.view(2, S, -1) for t in (q, k, v)]
    for prompt in (0, 1, 9):
        kc, vc = (torch.full((2, sinks + window, KV * D), float("nan"), dtype=torch.float64) for _ in range(2))
        if prompt:
            ops.window_cache_fill(k, v, S, kc, vc, window, sinks, torch.full((2,), prompt, dtype=torch.int32))
        pos = torch.full((2,), prompt, dtype=torch.int32)
        for t in range(prompt, S):
            o = ops.window_attention_step(*(r[:, t].contiguous() for r in rows), kc, vc, pos, H, window, sinks,
                                          kv_heads=KV, bias=bias, max_distance=M)
            assert torch.allclose(o, whole[:, t], rtol=0, atol=1e-13), (prompt, t)
            pos += 1


def test_rows_of_minus_infinity_have_no_softmax():
    """A bias of −inf takes a bucket away; a row whose every score is −inf is 0 / 0, and only it and what it sees are."""
    S, H, M = 6, 2, 8
    q, k, v = (t.requires_grad_() for t in _inputs(1, S, H, H, 64, 8))
    bias = torch.zeros(H, 4, dtype=torch.float64)
    bias[0, 0] = -math.inf                                     # no token sees itself: token 0 of head 0 sees nothing
    bias.requires_grad_()
    o = ops.window_attention(q, k, v, S, H, 3, bias=bias, max_distance=M)
    assert torch.isnan(o[0, :64]).all() and torch.isfinite(o[1:]).all() and torch.isfinite(o[:, 64:]).all()
    far = bias.detach().clone()
    far[0, 0] = -1e4                                           # e^−10000 is 0 in 64 bits
    assert torch.equal(o[1:], ops.window_attention(q, k, v, S, H, 3, bias=far, max_distance=M)[1:])
    for g in torch.autograd.grad(o, (q, k, v), torch.ones_like(o)):
        assert torch.isnan(g[0, :64]).all() and torch.isfinite(g[1:]).all() and torch.isfinite(g[:, 64:]).all()
    kc, vc = torch.randn(2, 4, 128, dtype=torch.float64), torch.randn(2, 4, 128, dtype=torch.float64)
    rows = [t.detach()[:2] for t in (q, k, v)]
    all_gone = torch.full((H, 4), -math.inf, dtype=torch.float64)
    o = ops.window_attention_step(*rows, kc, vc, torch.tensor([5, -1], dtype=torch.int32), H, 4, bias=all_gone,
                                  max_distance=M)
    assert torch.isnan(o[0]).all() and not o[1].any()          # an idle sequence has no row


def test_idle_sequences_stay_as_they_are():
    kc, vc = torch.randn(3, 6, 64), torch.randn(3, 6, 64)
    before = kc.clone(), vc.clone()
    x = torch.full((3, 64), float("nan"))
    x[1] = 1.0
    o = ops.window_attention_step(x, x, x, kc, vc, torch.tensor([-1, 0, -7], dtype=torch.int32), 1, 4, 2)
    assert not o[0].any() and not o[2].any() and torch.equal(o[1], x[1])
    for c, b in zip((kc, vc), before):
        b[1, 0] = 1.0
        assert torch.equal(c, b)
    ops.window_cache_fill(torch.ones(6, 64), torch.ones(6, 64), 2, kc, vc, 4, 2,
                          torch.tensor([0, 1, 2], dtype=torch.int32))
    before[0][1, :1] = 1.0
    before[0][2, :2] = 1.0
    assert torch.equal(kc, before[0])


def _t(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("error,match,kw", [
    (ValueError, "head dim", dict(q=_t(8, 96), k=_t(8, 96), v=_t(8, 96), H=1)),
    (ValueError, "rows, heads", dict(q=_t(2, 4, 128))), (ValueError, "rows, heads", dict(H=3)),
    (ValueError, "query heads over", dict(kv_heads=3)), (ValueError, "query heads over", dict(H=0)),
    (ValueError, "heads of dim", dict(kv_heads=1)), (ValueError, "rows expected", dict(k=_t(4, 128))),
    (TypeError, "expected", dict(v=_t(8, 128, dtype=torch.bfloat16))),
    (TypeError, "bf16 or fp32", dict(q=_t(8, 128, dtype=torch.float16))),
    (ValueError, "whole sequences", dict(S=3)), (ValueError, "whole sequences", dict(S=0)),
    (ValueError, "window", dict(window=0)), (ValueError, "sinks", dict(sinks=-1)), (ValueError, "sinks", dict(sinks=65)),
    (ValueError, "scale", dict(scale=0.0)), (ValueError, "scale", dict(scale=float("nan"))),
    (ValueError, "mask", dict(mask=_t(2, 4))), (ValueError, "mask", dict(mask=torch.ones(2, 3, dtype=torch.bool))),
    (ValueError, "bias", dict(bias=_t(3, 8))), (TypeError, "bias", dict(bias=_t(2, 8, dtype=torch.bfloat16))),
    (ValueError, "clients", dict(bias=_t(3, 2, 8))), (ValueError, "buckets", dict(bias=_t(2, 1))),
    (ValueError, "buckets", dict(bias=_t(2, 129), max_distance=1000)),
    (ValueError, "max_distance", dict(bias=_t(2, 8), max_distance=4)),
    (ValueError, "max_distance", dict(bias=_t(2, 8), max_distance=1025))])
def test_refusals(error, match, kw):
    a = dict(q=_t(8, 128), k=_t(8, 128), v=_t(8, 128), S=4, H=2, window=3)
    a.update(kw)
    with pytest.raises(error, match=match):
        ops.window_attention(**a)


def test_caches_that_overlap_are_refused():
    buf = _t(3, 5, 128)
    row, pos = _t(2, 128), torch.zeros(2, dtype=torch.int32)
    for a, b in ((buf[:2], buf[1:]), (buf[1:], buf[:2]), (buf[:2], buf[:2])):
        with pytest.raises(ValueError, match="same memory"):
            ops.window_attention_step(row, row, row, a, b, pos, 2, 4, 1)
        with pytest.raises(ValueError, match="same memory"):
            ops.window_cache_fill(_t(6, 128), _t(6, 128), 3, a, b, 4, 1)
    both = _t(4, 5, 128)                                       # two caches of one piece of memory
    ops.window_attention_step(row, row, row, both[:2], both[2:], pos, 2, 4, 1)


def test_rows_that_lie_in_a_cache():
    """Rows of the caches as arguments: what they held before the call counts."""
    both = torch.randn(2, 2, 5, 128, generator=torch.Generator().manual_seed(9))
    pos = torch.tensor([3, 8], dtype=torch.int32)              # slots 3 and 4
    for pick in (lambda c: (c[0, :, 3], c[1, :, 3], c[0, :, 4]), lambda c: (c[1, :, 4], c[1, :, 3], c[0, :, 3])):
        mine, ref = both.clone(), both.clone()
        o = ops.window_attention_step(*pick(mine), *mine, pos, 2, 4, 1)
        want = ops.window_attention_step(*(t.clone() for t in pick(both)), *ref, pos, 2, 4, 1)
        assert torch.equal(o, want) and torch.equal(mine, ref)
    mine, ref = both.clone(), both.clone()
    ops.window_cache_fill(mine[1].view(10, 128), mine[0].view(10, 128), 5, *mine, 4, 1)
    ops.window_cache_fill(both[1].reshape(10, 128).clone(), both[0].reshape(10, 128).clone(), 5, *ref, 4, 1)
    assert torch.equal(mine, ref)


@pytest.mark.parametrize("scale", [1e-60, 2.0 ** -127, 2.0 ** 128, 3e38, 1e300, math.inf, -0.1])
def test_scales_that_32_bits_do_not_hold_are_refused(scale):
    q = torch.ones(4, 64)
    with pytest.raises(ValueError, match="scale"):
        ops.window_attention(q, q, q, 4, 1, 3, scale=scale)
    with pytest.raises(ValueError, match="scale"):
        ops.window_attention_step(q, q, q, _t(4, 3, 64), _t(4, 3, 64), torch.zeros(4, dtype=torch.int32), 1, 3,
                                  scale=scale)
    for fine in (2.0 ** -126, 2.0 ** 127):
        ops.window_attention(q * 0, q, q, 4, 1, 3, scale=fine)


def test_rows_past_32_bits_are_refused():
    H = 2 ** 31 // 64
    row = torch.zeros(1, 1).expand(1, H * 64)                  # no memory behind it
    for KV in (1, H):
        kv = row[:, :KV * 64]
        with pytest.raises(ValueError, match="elements a row"):
            ops.window_attention(row, kv, kv, 1, H, 1, kv_heads=KV)
        with pytest.raises(ValueError, match="elements a row"):
            ops.window_attention_step(row, kv, kv, *(torch.zeros(1).expand(1, 1, KV * 64) for _ in range(2)),
                                      torch.zeros(1, dtype=torch.int32), H, 1, kv_heads=KV)


@pytest.mark.parametrize("N,S,H,KV,sinks,train,ok", [
    (2 ** 26 - 1, 1, 1, 1, 0, False, True), (2 ** 26, 1, 1, 1, 0, False, False),      # 64 threads a row of one token
    (2 ** 25 - 1, 1, 1, 1, 0, True, True), (2 ** 25, 1, 1, 1, 0, True, False),        # dk/dv: 128
    (2 ** 25, 1, 2, 1, 0, False, False), (2 ** 24 - 1, 65, 1, 1, 0, False, True), (2 ** 24, 65, 1, 1, 0, False, False),
    (2 ** 20, 64, 1, 1, 64, True, True), (2 ** 21, 1000, 1, 1, 64, True, False)])
def test_calls_that_no_launch_holds_are_refused(N, S, H, KV, sinks, train, ok):
    """A launch has fewer than 2^32 threads."""
    def plan():
        return W._plan(64, N, S, H, KV, min(64, S), min(sinks, S), 0.125, False, 0, 0, 0, train)
    if not ok:
        with pytest.raises(ValueError, match="too many"):
            plan()
        return
    a = plan()
    assert 2 * a.tile * N * H * -(-S // a.tile) < 2 ** 32
    assert not train or 2 * a.ktile * N * KV * (a.nchunk + -(-S // a.ktile)) < 2 ** 32


def test_steps_that_no_launch_holds_are_refused():
    for threads in (128, 256):
        most = (2 ** 32 - 1) // threads
        assert W._step_plan(most, 1, 1, 5, 1, 0.125, threads, 1, 0, 0).splits == 1
        with pytest.raises(ValueError, match="too many"):
            W._step_plan(most + 1, 1, 1, 5, 1, 0.125, threads, 1, 0, 0)


@pytest.mark.parametrize("error,match,kw", [
    (ValueError, "k_cache", dict(k_cache=_t(2, 4, 128))), (ValueError, "v_cache", dict(v_cache=_t(2, 5, 64))),
    (ValueError, "v_cache", dict(v_cache=_t(2, 5, 128, dtype=torch.bfloat16))),
    (ValueError, "contiguous", dict(k_cache=_t(2, 5, 256)[..., :128])),
    (ValueError, "pos", dict(pos=torch.zeros(2, dtype=torch.int64))),
    (ValueError, "pos", dict(pos=torch.zeros(3, dtype=torch.int32))),
    (ValueError, "no gradient", dict(q=_t(2, 128).requires_grad_())),
    (ValueError, "takes no gradient", dict(k_cache=_t(2, 5, 128).requires_grad_())),
    (ValueError, "window", dict(window=0)), (ValueError, "clients", dict(bias=_t(3, 2, 8)))])
def test_step_refusals(error, match, kw):
    a = dict(q=_t(2, 128), k=_t(2, 128), v=_t(2, 128), k_cache=_t(2, 5, 128), v_cache=_t(2, 5, 128),
             pos=torch.zeros(2, dtype=torch.int32), H=2, window=4, sinks=1)
    a.update(kw)
    with pytest.raises(error, match=match):
        ops.window_attention_step(**a)
    with pytest.raises(ValueError, match="same memory"):
        c = _t(2, 5, 128)
        ops.window_attention_step(_t(2, 128), _t(2, 128), _t(2, 128), c, c, torch.zeros(2, dtype=torch.int32), 2, 4, 1)


@pytest.mark.parametrize("error,match,kw", [
    (ValueError, "k_cache", dict(k_cache=_t(2, 640))), (ValueError, "k_cache", dict(window=5)),
    (ValueError, "rows", dict(k=_t(5, 128))), (ValueError, "columns", dict(v=_t(6, 64))),
    (TypeError, "expected", dict(k=_t(6, 128, dtype=torch.bfloat16))), (ValueError, "S ≥ 1", dict(S=0)),
    (ValueError, "lengths", dict(lengths=torch.zeros(2, dtype=torch.int64)))])
def test_fill_refusals(error, match, kw):
    a = dict(k=_t(6, 128), v=_t(6, 128), S=3, k_cache=_t(2, 5, 128), v_cache=_t(2, 5, 128), window=4, sinks=1)
    a.update(kw)
    with pytest.raises(error, match=match):
        ops.window_cache_fill(**a)
