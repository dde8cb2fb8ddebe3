"""Gated linear recurrence kernels (``csrc/scan_kernels.hip``) against the CPU form in 64 bits, and a block of recurrence
and biased window attention, trained and then answered with token by token.

Bounds, counted from the roundings (u = 2^-24; r = half a step of the storage type): σ and 1 − σ are off by at most
8 u relative (the argument's scaling: |gate| ≤ 20 here gives 20·2 u through e^−g where it matters less than 1 does, the
two hardware approximations 2 u each), a step makes 3 roundings, and a state is a sum of terms that each passed up to T
factors: with the convex weights f and 1 − f its error is at most the sum over the steps of 24 u times what the step
keeps, so 24 u·min(T, reach) of the largest |h| — a reach is 1 / (1 − f) steps. The same recurrence with absolute
values gives that bound per element: E_t = f E_{t−1} + 24 u (f|h_{t−1}| + (1 − f)|x_t|). Composing maps in another
order adds at most as much again (products of up to 64 factors): doubled. The backward is the same recurrence over
|δ|; dgate has the state's error times f (1 − f)|δ| besides."""
import pytest
import torch

from fedml_amd import ops

pytestmark = pytest.mark.gpu
dev = "cuda"
U = 2.0 ** -24


def _oracle(x, gate, h0, mask, dy, dh, dtype):
    x, gate, dy = (t.detach().cpu().double() for t in (x, gate, dy))
    C, T, B, H = x.shape
    real = torch.ones(C, T, B, 1, dtype=torch.bool) if mask is None else mask.cpu().bool().unsqueeze(-1)
    z = torch.zeros((), dtype=torch.float64)
    x, gate, dy = (torch.where(real, t, z) for t in (x, gate, dy))
    f, keep = torch.where(real, torch.sigmoid(gate), z + 1), torch.where(real, torch.sigmoid(-gate), z)
    rel = (24 + 4 * gate.abs()) * U * 2
    h = torch.zeros(C, B, H, dtype=torch.float64) if h0 is None else h0.detach().cpu().double()
    e = torch.zeros_like(h)
    hs, es = [h], [e]
    for t in range(T):
        e = f[:, t] * e + rel[:, t] * (f[:, t] * h.abs() + keep[:, t] * x[:, t].abs())
        h = f[:, t] * h + keep[:, t] * x[:, t]
        hs.append(h)
        es.append(e)
    y, ey = torch.stack(hs[1:], 1) * real, torch.stack(es[1:], 1) * real
    g = torch.zeros(C, B, H, dtype=torch.float64) if dh is None else dh.detach().cpu().double()
    eg = torch.zeros_like(g)
    dx, dg, ex, edg = (torch.zeros_like(x) for _ in range(4))
    for t in range(T - 1, -1, -1):
        d, ed = dy[:, t] + g, eg + 4 * U * (dy[:, t].abs() + g.abs())
        dx[:, t], ex[:, t] = keep[:, t] * d, keep[:, t] * (ed + rel[:, t] * d.abs())
        w = f[:, t] * keep[:, t]
        a = hs[t] - x[:, t]
        dg[:, t] = d * a * w
        edg[:, t] = w * (ed * a.abs() + d.abs() * (es[t] + (2 * rel[:, t] + 4 * U) * (hs[t].abs() + x[:, t].abs())))
        g, eg = f[:, t] * d, f[:, t] * (ed + rel[:, t] * d.abs())
    r = torch.finfo(dtype).eps / 2

    def stored(v, e):
        return v, e + r * (v.abs() + e) + 1e-30

    return [stored(y, ey), (h, es[-1] + 1e-30), stored(dx, ex * real), stored(dg, edg * real), (g, eg + 1e-30)]


def _within(got, want, what):
    value, bound = want
    assert got.shape == value.shape and torch.isfinite(got).all(), what
    err = (got.detach().cpu().double() - value).abs()
    worst = (err / bound).max().item() if err.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.3g} of the bound"


def _data(C, T, B, H, dtype, seed=0):
    gen = torch.Generator(device=dev).manual_seed(seed)

    def normal(*s, scale=1.0, shift=0.0, d=dtype):
        return (torch.randn(*s, generator=gen, device=dev) * scale + shift).to(d)

    return (normal(C, T, B, H), normal(C, T, B, H, scale=3.0, shift=2.0), normal(C, B, H, d=torch.float32),
            normal(C, T, B, H), normal(C, B, H, d=torch.float32))


def _call(x, gate, h0, mask, dy, dh):
    leaves = [t.detach().requires_grad_() for t in (x, gate, h0)]
    y, hT = ops.gated_scan(*leaves, mask=mask)
    return [y, hT, *torch.autograd.grad((y, hT), leaves, (dy, dh))]


def _mask(kind, C, T, B):
    if kind is None:
        return None
    gen = torch.Generator().manual_seed(3)
    if kind == "right":
        m = torch.arange(T).view(1, T, 1) < torch.randint(0, T + 1, (C, 1, B), generator=gen)
    else:
        m = torch.rand(C, T, B, generator=gen) > 0.3
    return m.to(dev)


NAMES = ("y", "hT", "dx", "dgate", "dh0")
CASES = [  # C, T, B, H, mask
    (1, 1, 1, 1, None), (2, 1, 3, 40, None), (1, 7, 2, 65, "holes"), (2, 8, 1, 64, None), (1, 9, 1, 33, "right"),
    (1, 63, 2, 66, None), (3, 64, 2, 32, "right"), (1, 65, 3, 31, "holes"), (2, 130, 1, 670, "right"),
    (1, 513, 2, 64, None), (1, 2000, 1, 96, "right"), (1, 4500, 1, 34, None), (40, 70, 8, 256, None)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
def test_forward_and_gradients(case, dtype):
    C, T, B, H, kind = case
    x, gate, h0, dy, dh = _data(C, T, B, H, dtype)
    mask = _mask(kind, C, T, B)
    got = _call(x, gate, h0, mask, dy, dh)
    for g, w, name in zip(got, _oracle(x, gate, h0, mask, dy, dh, dtype), NAMES):
        _within(g, w, name)
    assert all(torch.equal(a, b) for a, b in zip(got, _call(x, gate, h0, mask, dy, dh)))
    with torch.no_grad():
        y, hT = ops.gated_scan(x, gate, h0, mask=mask)
    assert torch.equal(y, got[0]) and torch.equal(hT, got[1])


def test_gates_at_their_ends():
    """Gates far out: what is kept or replaced whole, without NaN; a state that lasts thousands of steps."""
    T = 3000
    x, gate, h0, dy, dh = _data(1, T, 1, 64, torch.float32, 4)
    gate[..., :8], gate[..., 8:16], gate[..., 16:24], gate[..., 24:32] = 200.0, -200.0, float("inf"), -float("inf")
    gate[..., 32:48] = 12.0
    got = _call(x, gate, h0, None, dy, dh)
    y = got[0][0, :, 0]
    assert torch.equal(y[:, :8], h0[0, :, :8].expand(T, 8)) and torch.equal(y[:, 16:24], h0[0, :, 16:24].expand(T, 8))
    for s in (slice(8, 16), slice(24, 32)):                  # 1 − f is 1 up to two hardware approximations of 2 u
        assert ((y - x[0, :, 0])[:, s].abs() <= 4 * U * x[0, :, 0, s].abs() + 1e-30).all()
    assert all(torch.isfinite(t).all() for t in got)
    s = slice(32, 64)
    want = _oracle(x[..., s], gate[..., s], h0[..., s], None, dy[..., s], dh[..., s], torch.float32)
    for g, w, name in zip(got, want, NAMES):
        _within(g[..., s].contiguous(), w, name)
    gate[0, 5, 0, 0] = float("nan")                          # a NaN goes where the formula takes it
    y = ops.gated_scan(x, gate, h0)[0][0, :, 0]
    assert torch.isnan(y[5:, 0]).all() and torch.isfinite(y[:5, 0]).all() and torch.isfinite(y[:, 1:]).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_padding_reaches_nothing(dtype):
    x, gate, h0, dy, dh = _data(2, 100, 3, 40, dtype, 5)
    mask = _mask("right", 2, 100, 3)
    mask[0, :, 0] = False
    want = _call(x, gate, h0, mask, dy, dh)
    for fill in (float("nan"), float("inf")):
        bad = [t.masked_fill(~mask.unsqueeze(-1), fill) for t in (x, gate, dy)]
        got = _call(bad[0], bad[1], h0, mask, bad[2], dh)
        assert all(torch.equal(g, w) for g, w in zip(got, want))
    assert torch.equal(got[1][0, 0], h0[0, 0]) and torch.equal(got[4][0, 0], dh[0, 0])


def test_layouts():
    """Halves of a fused projection, token-major rows, odd offsets, strided features, shared inputs, other streams."""
    C, T, B, H = 2, 70, 3, 40
    x, gate, h0, dy, dh = _data(C, T, B, H, torch.bfloat16, 6)
    mask = _mask("right", C, T, B)
    want = _call(x, gate, h0, mask, dy, dh)
    fused = torch.cat([x, gate], -1)
    odd = torch.zeros(C, T, B, 2 * H + 1, dtype=x.dtype, device=dev)
    odd[..., 1:] = fused
    rows = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (x, gate, dy)]
    wide = [t.repeat_interleave(2, -1)[..., ::2] for t in (x, gate, dy)]
    m8 = mask.to(torch.int32).transpose(1, 2).contiguous().transpose(1, 2)
    for a, b, c, m in ((fused[..., :H], fused[..., H:], dy, mask), (odd[..., 1:H + 1], odd[..., H + 1:], dy, m8),
                       (*rows, mask), (*wide, m8)):
        got = _call(a, b, h0, m, c, dh)
        assert all(torch.equal(g, w) for g, w in zip(got, want))
    got = _call(*rows[:2], h0, mask, rows[2], dh)
    assert got[0].stride() == rows[0].stride()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _call(x, gate, h0, mask, dy, dh)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(g, w) for g, w in zip(got, want))
    one = x[:, :1].expand(C, T, B, H).detach().requires_grad_()                  # the same input at every step
    y, _ = ops.gated_scan(one, gate)
    y2, _ = ops.gated_scan(one.detach().contiguous(), gate)
    assert torch.equal(y, y2)
    leaf = x.detach().requires_grad_()                                           # one of the two outputs alone
    for k in (0, 1):
        out = ops.gated_scan(leaf, gate, h0, mask=mask)
        part = torch.autograd.grad(out[k], leaf, (dy, dh)[k])[0]
        full = _call(x, gate, h0, mask, *((dy, torch.zeros_like(dh)) if k == 0 else (torch.zeros_like(dy), dh)))[2]
        assert torch.equal(part, full)


def test_empty_batch():
    e = torch.zeros(2, 5, 0, 8, device=dev, requires_grad=True)
    y, hT = ops.gated_scan(e, e)
    assert y.shape == e.shape and hT.shape == (2, 0, 8)
    assert torch.autograd.grad(y, e, torch.zeros_like(y))[0].shape == e.shape


def test_offsets_past_32_bits():
    T, wide, H = 70000, 32768, 64
    buf = torch.empty(1, T, 1, wide, dtype=torch.bfloat16, device=dev)
    assert buf.numel() > 2 ** 31
    x, gate, h0, dy, dh = _data(1, T, 1, H, torch.bfloat16, 7)
    buf[..., -H:], buf[..., -2 * H:-H], buf[..., -3 * H:-2 * H] = x, gate, dy
    got = _call(buf[..., -H:], buf[..., -2 * H:-H], h0, None, buf[..., -3 * H:-2 * H], dh)
    assert all(torch.equal(g, w) for g, w in zip(got, _call(x, gate, h0, None, dy, dh)))


def test_captured_training_step_replays():
    static = list(_data(1, 700, 2, 64, torch.bfloat16, 8))
    mask = _mask("right", 1, 700, 2)

    def call(x, gate, h0, dy, dh):
        return _call(x, gate, h0, mask, dy, dh)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(*static)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(*static)
    for seed in (20, 21, 22):
        for t, n in zip(static, _data(1, 700, 2, 64, torch.bfloat16, seed)):
            t.copy_(n)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(g, w) for g, w in zip(out, call(*(t.clone() for t in static))))


# ------------------------------------------------------------------------------------------------ used together
def _block(x, w, S, C, B, H, KV, D, window, sinks, M, mask=None):
    """A token mixer for long text: a gated recurrence for what lies behind the window, then biased window attention."""
    dm = H * D
    z = (x @ w["in"]).view(C, B, S, 2 * dm).transpose(1, 2)
    y, _ = ops.gated_scan(z[..., :dm], z[..., dm:], mask=None if mask is None else mask.view(C, B, S).transpose(1, 2))
    h = y.transpose(1, 2).reshape(C * B * S, dm) + x
    qkv = h @ w["qkv"]
    o = ops.window_attention(qkv[:, :dm], qkv[:, dm:dm + KV * D], qkv[:, dm + KV * D:], S, H, window, sinks,
                             kv_heads=KV, mask=mask, bias=w["bias"], max_distance=M)
    return h + o @ w["out"]


def test_block_trains_and_answers():
    C, B, S, H, KV, D, window, sinks, M = 2, 2, 90, 2, 1, 64, 24, 2, 32
    dm = H * D
    gen = torch.Generator().manual_seed(5)
    w64 = {"in": torch.randn(dm, 2 * dm, generator=gen, dtype=torch.float64) / dm ** 0.5,
           "qkv": torch.randn(dm, dm + 2 * KV * D, generator=gen, dtype=torch.float64) / dm ** 0.5,
           "out": torch.randn(dm, dm, generator=gen, dtype=torch.float64) / dm ** 0.5,
           "bias": torch.randn(C, H, 8, generator=gen, dtype=torch.float64)}
    x64 = torch.randn(C * B * S, dm, generator=gen, dtype=torch.float64)
    mask = torch.arange(S) < torch.tensor([[90], [50], [90], [31]])
    g64 = torch.randn(C * B * S, dm, generator=gen, dtype=torch.float64) * mask.view(-1, 1)
    w = {k: t.float().to(dev).requires_grad_() for k, t in w64.items()}
    w64 = {k: t.detach().cpu().double().requires_grad_() for k, t in w.items()}
    x = x64.float().to(dev).requires_grad_()
    x64 = x.detach().cpu().double().requires_grad_()
    cfg = (S, C, B, H, KV, D, window, sinks, M)
    out, want = _block(x, w, *cfg, mask=mask.to(dev)), _block(x64, w64, *cfg, mask=mask)
    got = torch.autograd.grad(out, [x, *w.values()], g64.float().to(dev))
    ref = torch.autograd.grad(want, [x64, *w64.values()], g64.float().double())
    # four products of length 128 and the two operators in a row, fp32: some 10^3 roundings of 2^-24 at most, in the norm
    for a, b in zip((out, *got), (want, *ref)):
        assert (a.detach().cpu().double() - b).norm() <= 2 ** 10 * U * b.norm()
    # token by token over the cache, from the 20th on: the same rows
    with torch.no_grad():
        whole = _block(x, w, *cfg).view(C * B, S, dm)
        xs, n = x.view(C * B, S, dm), 20
        z = (xs[:, :n].reshape(-1, dm) @ w["in"]).view(C, B, n, 2 * dm).transpose(1, 2)
        y, state = ops.gated_scan(z[..., :dm], z[..., dm:])
        h = y.transpose(1, 2).reshape(C * B * n, dm) + xs[:, :n].reshape(-1, dm)
        qkv = h @ w["qkv"]
        caches = [torch.zeros(C * B, sinks + window, KV * D, device=dev) for _ in range(2)]
        ops.window_cache_fill(qkv[:, dm:dm + KV * D], qkv[:, dm + KV * D:], n, *caches, window, sinks)
        pos = torch.full((C * B,), n, dtype=torch.int32, device=dev)
        for t in range(n, S):
            z = (xs[:, t] @ w["in"]).view(C, 1, B, 2 * dm)
            y, state = ops.gated_scan(z[..., :dm], z[..., dm:], state)
            h = y.reshape(C * B, dm) + xs[:, t]
            qkv = h @ w["qkv"]
            o = ops.window_attention_step(qkv[:, :dm], qkv[:, dm:dm + KV * D], qkv[:, dm + KV * D:], *caches, pos, H,
                                          window, sinks, kv_heads=KV, bias=w["bias"].detach(), max_distance=M)
            pos += 1
            row = h + o @ w["out"]
            assert (row - whole[:, t]).norm() <= 2 ** 10 * U * whole[:, t].norm(), t
