"""What is measured of the long-text operators: causal sliding-window attention with sinks (``window_attention``), its
learned relative position bias by buckets, its form for one new token over a ring cache (``window_attention_step``) and
the gated linear recurrence (``gated_scan``).

``own`` selects the side: the framework's kernels, or the plain form of the same operators in elementary torch
operations. ``exact`` states the operators once more, from their definitions, in 64 bits."""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
DEV = "cuda"


# ------------------------------------------------------------------------------------------------------------ cases
def _attn(name, dtype, train, C, B, S, H, KV, D, W, sinks, NB=0, M=0, padded=False):
    return {"name": name, "op": "attention", "dtype": dtype, "train": train, "C": C, "B": B, "S": S, "H": H, "KV": KV,
            "D": D, "window": W, "sinks": sinks, "buckets": NB, "max_distance": M, "padded": padded}


def _step(name, dtype, B, H, KV, D, W, sinks, NB=0, M=0):
    return {"name": name, "op": "step", "dtype": dtype, "B": B, "H": H, "KV": KV, "D": D, "window": W, "sinks": sinks,
            "buckets": NB, "max_distance": M}


def _scan(name, dtype, train, C, T, B, H, padded=False):
    return {"name": name, "op": "scan", "dtype": dtype, "train": train, "C": C, "T": T, "B": B, "H": H,
            "padded": padded}


def listed():
    return [
        # ten clients' local step on 80-character lines (the Shakespeare length), fp32 as the reference trains
        _attn("chars_attn_fp32", "fp32", True, 10, 8, 80, 4, 4, 64, 32, 1),
        # four clients' padded documents of odd length, DistilBERT's heads
        _attn("docs_attn_bf16", "bf16", True, 4, 4, 1999, 12, 12, 64, 256, 4, padded=True),
        # a training step on long text with shared key/value heads
        _attn("long_attn_bf16", "bf16", True, 1, 2, 16384, 16, 4, 128, 1024, 4),
        # reading one long prompt before answering: forward alone
        _attn("prompt_attn_bf16", "bf16", False, 1, 1, 32768, 32, 8, 128, 1024, 4),
        # next-word prediction on 20-word lines (the StackOverflow length), the window wider than the line, biased
        _attn("words_bias_fp32", "fp32", True, 4, 16, 20, 4, 4, 64, 32, 0, 8, 16, padded=True),
        # biased training step of four clients, each with a table of its own
        _attn("docs_bias_bf16", "bf16", True, 4, 2, 2047, 12, 12, 64, 512, 0, 32, 128),
        # one user's next token: latency
        _step("one_step_bf16", "bf16", 1, 12, 12, 64, 1024, 4),
        # the next token of a full batch over long caches, biased: bandwidth
        _step("batch_step_bf16", "bf16", 64, 32, 8, 128, 4096, 4, 32, 128),
        # ten clients' 80-character lines through one recurrent layer as wide as the framework's character LSTM
        _scan("chars_scan_fp32", "fp32", True, 10, 80, 64, 256),
        # a long text at a small batch: few channels, a long axis
        _scan("long_scan_bf16", "bf16", True, 1, 16384, 4, 1024),
        # eight clients' padded documents at the word LSTM's odd width
        _scan("docs_scan_bf16", "bf16", True, 8, 2048, 16, 670, padded=True),
        # the next token of a batch
        _scan("step_scan_bf16", "bf16", False, 1, 1, 64, 1024),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def draw(rng):
    most = {}
    for c in listed():
        most[c["op"]] = max(most.get(c["op"], 0), _cost(c))
    while True:
        op = rng.choice(("attention", "attention", "attention", "step", "scan", "scan"))
        dtype = rng.choice(("bf16", "bf16", "fp32"))
        KV = rng.choice((1, 2, 4, 8, 12))
        H = KV * rng.choice((1, 1, 2, 3, 4))
        D = rng.choice((64, 128))
        bias = rng.random() < 0.5
        NB = rng.choice((8, 16, 32, 64)) if bias else 0
        M = NB * rng.choice((2, 4, 8)) if bias else 0
        if op == "attention":
            c = _attn("", dtype, rng.random() < 0.75, rng.choice((1, 2, 4)), _log(rng, 1, 32), _log(rng, 17, 16384), H, KV,
                      D, _log(rng, 16, 2048), rng.choice((0, 1, 4, 33, 64)), NB, M, rng.random() < 0.4)
        elif op == "step":
            c = _step("", dtype, _log(rng, 1, 96), H, KV, D, _log(rng, 32, 8192), rng.choice((0, 1, 4, 64)), NB, M)
        else:
            c = _scan("", dtype, rng.random() < 0.75, rng.choice((1, 3, 8)), _log(rng, 1, 16384), _log(rng, 1, 64),
                      _log(rng, 32, 2048), rng.random() < 0.4)
        del c["name"]
        # the plain attention is a band of whole windows: a small window over a long text still costs it little
        if _cost(c) <= (most[op] if dtype == "bf16" or op != "attention" else most[op] / 8):
            return c


def _pairs(S, W, sinks):
    """Visible (query, key) pairs of one sequence."""
    W = min(W, S)
    n = W * (W + 1) // 2 + (S - W) * W
    return n + sum(max(0, S - W - j) for j in range(min(sinks, S)))


def work(case):
    e = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "attention":
        N, S, H, KV, D = case["C"] * case["B"], case["S"], case["H"], case["KV"], case["D"]
        real = 0.75 if case["padded"] else 1.0            # lengths run evenly from S/2 to S
        q, kv = N * S * H * D * e, N * S * KV * D * e
        pairs = real * N * H * _pairs(S, case["window"], case["sinks"])
        table = 4 * case["C"] * H * case["buckets"]
        if not case["train"]:
            return {"bytes": 2 * q + 2 * kv + table, "flops": 4 * D * pairs}
        return {"bytes": 4 * q + 4 * kv + 2 * table, "flops": 12 * D * pairs}   # q, o, dO, dq; k, v, dk, dv
    if case["op"] == "step":
        n = case["sinks"] + case["window"]
        rows = case["B"] * case["KV"] * case["D"] * e
        return {"bytes": 2 * rows * n + 4 * rows + 2 * case["B"] * case["H"] * case["D"] * e,
                "flops": 4 * case["B"] * case["H"] * case["D"] * n}
    n = case["C"] * case["T"] * case["B"] * case["H"]
    state = 4 * case["C"] * case["B"] * case["H"]
    if not case["train"]:
        return {"bytes": 3 * n * e + 2 * state, "flops": 8 * n}
    return {"bytes": 6 * n * e + 4 * state, "flops": 24 * n}                    # x, gate, y, dy, dx, dgate


# ----------------------------------------------------------------------------------------------------------- inputs
def _lengths(gen, n, S):
    return torch.randint((S + 1) // 2, S + 1, (n,), generator=gen, device=DEV)


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    dt = TYPES[case["dtype"]]

    def normal(*shape, scale=1.0, shift=0.0, dtype=None):
        return (torch.randn(*shape, generator=gen, device=DEV) * scale + shift).to(dtype or dt)

    st = {"case": case}
    if case["op"] == "scan":
        C, T, B, H = case["C"], case["T"], case["B"], case["H"]
        st.update(x=normal(C, T, B, H), gate=normal(C, T, B, H, scale=1.5, shift=2.0),
                  h0=normal(C, B, H, scale=0.5, dtype=torch.float32))
        st["mask"] = None
        if case["padded"]:
            n = _lengths(gen, C * B, T).view(C, 1, B)
            st["mask"] = torch.arange(T, device=DEV).view(1, T, 1) < n
        if case["train"]:
            st.update(dy=normal(C, T, B, H), dh=normal(C, B, H, dtype=torch.float32))
            for k in ("x", "gate", "h0"):
                st[k].requires_grad_()
        return st
    H, KV, D = case["H"], case["KV"], case["D"]
    if case["op"] == "step":
        B, n = case["B"], case["sinks"] + case["window"]
        st.update(q=normal(B, H * D, scale=1.5), k=normal(B, KV * D), v=normal(B, KV * D),
                  k_cache=normal(B, n, KV * D), v_cache=normal(B, n, KV * D), table=None)
        # sequences somewhere in a long answer, a few of them still shorter than the window
        pos = torch.randint(0, 4 * n, (B,), generator=gen, device=DEV)
        short = torch.randint(0, n, (B,), generator=gen, device=DEV)
        at = torch.arange(B, device=DEV) % 8 == 7
        st["pos"] = torch.where(at, short, pos + n).to(torch.int32)
        if case["buckets"]:
            st["table"] = normal(H, case["buckets"], dtype=torch.float32)
        return st
    C, N, S = case["C"], case["C"] * case["B"], case["S"]
    st.update(q=normal(N * S, H * D, scale=1.5), k=normal(N * S, KV * D), v=normal(N * S, KV * D), mask=None, table=None)
    if case["padded"]:
        st["mask"] = torch.arange(S, device=DEV).view(1, S) < _lengths(gen, N, S).view(N, 1)
    if case["buckets"]:
        st["table"] = normal(C, H, case["buckets"], dtype=torch.float32)
    if case["train"]:
        st["do"] = normal(N * S, H * D)
        for k in ("q", "k", "v", "table"):
            if st[k] is not None:
                st[k].requires_grad_()
    return st


# ------------------------------------------------------------------------------------------------------------- runs
def run(state):
    case = state["case"]
    if own:
        return _run_own(case, state)
    with torch.no_grad():
        return {"attention": _plain_attention, "step": _plain_step, "scan": _plain_scan}[case["op"]](case, state)


def _run_own(case, st):
    from fedml_amd import ops
    if case["op"] == "scan":
        y, h = ops.gated_scan(st["x"], st["gate"], st["h0"], mask=st["mask"])
        if not case["train"]:
            return y, h
        return (y, h, *torch.autograd.grad((y, h), (st["x"], st["gate"], st["h0"]), (st["dy"], st["dh"])))
    if case["op"] == "step":
        o = ops.window_attention_step(st["q"], st["k"], st["v"], st["k_cache"], st["v_cache"], st["pos"], case["H"],
                                      case["window"], case["sinks"], kv_heads=case["KV"], bias=st["table"],
                                      max_distance=case["max_distance"])
        return o, st["k_cache"], st["v_cache"]
    o = ops.window_attention(st["q"], st["k"], st["v"], case["S"], case["H"], case["window"], case["sinks"],
                             kv_heads=case["KV"], mask=st["mask"], bias=st["table"], max_distance=case["max_distance"])
    if not case["train"]:
        return o
    leaves = [st[k] for k in ("q", "k", "v", "table") if st[k] is not None]
    return (o, *torch.autograd.grad(o, leaves, st["do"]))


# ------------------------------------------------------------------------------------------------------ plain forms
def _starts(NB, M):
    """First distance of every bucket: whole numbers up to NB // 2, evenly spread over the logarithm up to M after."""
    E = NB // 2
    n = NB - E
    starts, d = list(range(E + 1)), E
    for j in range(1, n):
        while d ** n < M ** j * E ** (n - j):
            d += 1
        starts.append(d)
    return starts


def _bucket(distance, NB, M):
    starts = torch.tensor(_starts(NB, M), device=distance.device)
    return (distance.clamp_min(0).unsqueeze(-1) >= starts).sum(-1) - 1


def _band(t, w):
    """[N, KV, n·w, D] → the rows of each block of w with those of the block before it: [N, KV, n, 2w, D]."""
    N, KV, L, D = t.shape
    b = t.reshape(N, KV, L // w, w, D)
    before = torch.cat([torch.zeros_like(b[:, :, :1]), b[:, :, :-1]], 2)
    return torch.cat([before, b], 3)


def _unband(g, w):
    """The sum over both blocks that hold a row: _band's adjoint."""
    before, b = g[..., :w, :], g[..., w:, :]
    out = b.clone()
    out[:, :, :-1] += before[:, :, 1:]
    return out.flatten(2, 3)


def _plain_attention(case, st):
    C, N, S, H, KV, D = case["C"], case["C"] * case["B"], case["S"], case["H"], case["KV"], case["D"]
    G, w = H // KV, min(case["window"], S)
    n = -(-S // w)
    L, sinks, dt = n * w, min(case["sinks"], S), st["q"].dtype
    scale = 1.0 / math.sqrt(D)
    real = torch.ones(N, S, dtype=torch.bool, device=DEV) if st["mask"] is None else st["mask"]
    real = torch.nn.functional.pad(real, (0, L - S))

    def heads(t, h):      # [N·S, h·D] → [N, h, L, D], what is no token set to zero
        t = torch.nn.functional.pad(t.detach().float().view(N, S, h, D), (0, 0, 0, 0, 0, L - S))
        return torch.where(real.view(N, L, 1, 1), t, torch.zeros_like(t)).transpose(1, 2)

    def blocks(t):        # [N, H, L, D] → [N, KV, n, G·w, D]: the queries that share a block of keys
        return t.reshape(N, KV, G, n, w, D).transpose(2, 3).reshape(N, KV, n, G * w, D)

    def back(t, h):       # and back to the layout of the inputs
        return t[:, :, :S].transpose(1, 2).reshape(N * S, h * D).to(dt)

    def unblock(t):
        return t.view(N, KV, n, G, w, D).transpose(2, 3).reshape(N, H, L, D)

    q, kh, vh = blocks(heads(st["q"], H)), heads(st["k"], KV), heads(st["v"], KV)
    ks, vs = (t[:, :, None, :sinks].expand(N, KV, n, sinks, D) for t in (kh, vh))
    kc, vc = torch.cat([ks, _band(kh, w)], 3), torch.cat([vs, _band(vh, w)], 3)       # [N, KV, n, sinks + 2w, D]
    i = torch.arange(L, device=DEV).view(n, w, 1)
    at = torch.arange(2 * w, device=DEV) - w + torch.arange(0, L, w, device=DEV).view(n, 1, 1)
    first = torch.arange(sinks, device=DEV).expand(n, 1, sinks)
    see = torch.cat([(i - first) >= w, (at >= 0) & (at <= i) & (i - at < w)], -1)     # [n, w, sinks + 2w]
    j = torch.cat([first, at.clamp_min(0)], -1)
    see = see & real[:, j] & real.view(N, n, w, 1)                                    # [N, n, w, sinks + 2w]
    see = see.view(N, 1, n, 1, w, -1)
    s = (q @ kc.transpose(-1, -2)).view(N, KV, n, G, w, -1).mul_(scale)
    if st["table"] is not None:
        # a block's distances are the same in every block, but for those to the sinks
        table = st["table"].detach().view(C, KV, 1, G, -1)
        of = _bucket((torch.arange(w, device=DEV).view(w, 1) + w - torch.arange(2 * w, device=DEV)),
                     case["buckets"], case["max_distance"])
        to = _bucket(i - first, case["buckets"], case["max_distance"])
        s = s.view(C, case["B"], KV, n, G, w, -1)
        s[..., sinks:] += table[..., of].unsqueeze(1)
        s[..., :sinks] += table[:, :, 0][..., to].permute(0, 1, 3, 2, 4, 5).unsqueeze(1)
        s = s.view(N, KV, n, G, w, -1)
    s.masked_fill_(~see, float("-inf"))
    top = s.amax(-1, keepdim=True).clamp_min(-1e30)
    p = s.sub_(top).exp_()
    p /= p.sum(-1, keepdim=True).clamp_min(1e-30)
    o = p.flatten(3, 4) @ vc
    if not case["train"]:
        return back(unblock(o), H)
    do = blocks(heads(st["do"], H))
    g = (do @ vc.transpose(-1, -2)).view_as(p)
    gv = p.flatten(3, 4).transpose(-1, -2) @ do
    ds = p * (g - (p * g).sum(-1, keepdim=True))
    gq = ds.flatten(3, 4) @ kc * scale
    gk = ds.flatten(3, 4).transpose(-1, -2) @ q * scale

    def keys(t):          # the sinks' gradients come from every block
        out = _unband(t[..., sinks:, :], w)
        out[:, :, :sinks] += t[..., :sinks, :].sum(2)
        return out

    out = [back(unblock(o), H), back(unblock(gq), H), back(keys(gk), KV), back(keys(gv), KV)]
    if st["table"] is not None:
        ds = ds.view(C, case["B"], KV, n, G, w, -1)
        near = ds[..., sinks:].sum(3).sum(1, dtype=torch.float64)        # [C, KV, G, w, 2w]
        # rows one longer than they are shift each row by one more: a column then holds one distance, 2w − it
        near = torch.nn.functional.pad(near, (w, 0)).flatten(-2)
        near = torch.nn.functional.pad(near, (0, w)).view(C, H, w, 3 * w + 1).sum(2)
        near_of = _bucket(2 * w - torch.arange(3 * w + 1, device=DEV), case["buckets"], case["max_distance"])
        far = ds[..., :sinks].sum(1, dtype=torch.float64).transpose(2, 3).reshape(C, H, -1)
        ids = torch.arange(case["buckets"], device=DEV)
        gt = near @ (near_of.view(-1, 1) == ids).double() + far @ (to.reshape(-1, 1) == ids).double()
        out.append(gt.float())
    return tuple(out)


def _plain_step(case, st):
    B, H, KV, D, W, sinks = case["B"], case["H"], case["KV"], case["D"], case["window"], case["sinks"]
    n, pos = W + sinks, st["pos"].long()
    slot = torch.where(pos < sinks, pos, sinks + (pos - sinks) % W)
    row = torch.arange(B, device=DEV)
    st["k_cache"][row, slot], st["v_cache"][row, slot] = st["k"], st["v"]
    # the position of the token in every slot, −1 where there is none; a ring slot holds the last one that goes there
    s, last = torch.arange(n, device=DEV).view(1, n), pos.view(-1, 1)
    ring = last - (last - s) % W
    holds = torch.where(s < sinks, torch.where(s <= last, s, -1), torch.where(ring >= sinks, ring, -1))
    q = st["q"].float().view(B, KV, H // KV, D)
    kc, vc = (st[c].float().view(B, n, KV, D).transpose(1, 2) for c in ("k_cache", "v_cache"))
    sc = (q @ kc.transpose(-1, -2)) / math.sqrt(D)
    if st["table"] is not None:
        b = _bucket(pos.view(-1, 1) - holds, case["buckets"], case["max_distance"])
        sc = sc + st["table"].view(KV, H // KV, -1)[..., b].permute(2, 0, 1, 3)
    sc = sc.masked_fill(holds.view(B, 1, 1, n) < 0, float("-inf"))
    p = (sc - sc.amax(-1, keepdim=True)).exp()
    p = p / p.sum(-1, keepdim=True)
    return (p @ vc).reshape(B, H * D).to(st["q"].dtype), st["k_cache"], st["v_cache"]


def _recur(a, b):
    """h_t = a_t h_{t−1} + b_t over dim 1 from h = 0, by doubling the reach of each step."""
    reach, T = 1, a.shape[1]
    while reach < T:
        b = torch.cat([b[:, :reach], b[:, reach:] + a[:, reach:] * b[:, :-reach]], 1)
        a = torch.cat([a[:, :reach], a[:, reach:] * a[:, :-reach]], 1)
        reach *= 2
    return b


def _plain_scan(case, st):
    x, gate, h0 = st["x"].detach().float(), st["gate"].detach().float(), st["h0"].detach()
    f, keep = 1 / (1 + (-gate).exp()), 1 / (1 + gate.exp())              # 1 − f without its cancellation
    real = None if st["mask"] is None else st["mask"].unsqueeze(-1)
    if real is not None:
        f, keep = torch.where(real, f, 1.0), torch.where(real, keep, 0.0)
    b = keep * x
    b[:, 0] += f[:, 0] * h0
    h = _recur(f, b)
    y = h if real is None else torch.where(real, h, 0.0)
    y, last = y.to(st["x"].dtype), h[:, -1].clone()
    if not case["train"]:
        return y, last
    g = st["dy"].float()
    g = g.clone() if real is None else torch.where(real, g, 0.0)
    g[:, -1] += st["dh"]
    a = torch.cat([f[:, 1:], torch.zeros_like(f[:, :1])], 1)             # what a step's state gives to the next one
    g = _recur(a.flip(1), g.flip(1)).flip(1)
    before = torch.cat([h0.unsqueeze(1), h[:, :-1]], 1)
    dgate = g * (before - x) * f * keep
    return y, last, (g * keep).to(st["x"].dtype), dgate.to(st["x"].dtype), g[:, 0] * f[:, 0]


# ------------------------------------------------------------------------------------------------------------ exact
def _bucket_by_definition(d, NB, M):
    """Bucket of a whole distance, by the definition's inequality alone."""
    E = NB // 2
    if d < E:
        return d
    n = NB - E
    return E + max(j for j in range(n) if d ** n >= M ** j * E ** (n - j))


def _by_distance(case, most):
    """Bucket of the distances 0 … most (the last bucket from max_distance on)."""
    M, NB = case["max_distance"], case["buckets"]
    table = [_bucket_by_definition(d, NB, M) for d in range(min(most, M) + 1)]
    return torch.tensor(table + [NB - 1] * (most + 1 - len(table)), device=DEV)


def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        return {"attention": _exact_attention, "step": _exact_step, "scan": _exact_scan}[case["op"]](case, st)


def _exact_attention(case, st):
    C, N, S, H, KV, D = case["C"], case["C"] * case["B"], case["S"], case["H"], case["KV"], case["D"]
    W, sinks, G = case["window"], case["sinks"], case["H"] // case["KV"]
    real = torch.ones(N, S, dtype=torch.bool, device=DEV) if st["mask"] is None else st["mask"]

    def heads(t, h):
        return t.detach().double().view(N, S, h, D).permute(0, 2, 1, 3).contiguous()

    q, k, v = heads(st["q"], H).view(N, KV, G, S, D), heads(st["k"], KV), heads(st["v"], KV)
    o = torch.zeros_like(q)
    table = None if st["table"] is None else st["table"].detach().double().view(C, KV, G, -1)
    of = None if table is None else _by_distance(case, S)
    if case["train"]:
        do, dq, dk, dv = heads(st["do"], H).view_as(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
        dt = None if table is None else torch.zeros_like(table)
    for i0 in range(0, S, 256):
        i1 = min(S, i0 + 256)
        lo = max(0, i0 - W + 1)
        j = torch.cat([torch.arange(min(sinks, lo), device=DEV), torch.arange(lo, i1, device=DEV)])
        i = torch.arange(i0, i1, device=DEV)
        dist = i.view(-1, 1) - j
        see = (dist >= 0) & ((dist < W) | (j < sinks))
        see = see & real[:, None, j] & real[:, i0:i1, None]
        kj, vj = k[:, :, j], v[:, :, j]
        s = torch.einsum("nkgid,nkjd->nkgij", q[:, :, :, i0:i1], kj) / math.sqrt(D)
        if table is not None:
            b = of[dist.clamp_min(0)]
            s = s + table[..., b].repeat_interleave(case["B"], 0)
        s = torch.where(see[:, None, None], s, -math.inf)
        p = torch.softmax(s, -1).nan_to_num(0.0)
        o[:, :, :, i0:i1] = torch.einsum("nkgij,nkjd->nkgid", p, vj)
        if not case["train"]:
            continue
        g = torch.where(real[:, None, None, i0:i1, None], do[:, :, :, i0:i1], 0.0)
        dp = torch.einsum("nkgid,nkjd->nkgij", g, vj)
        ds = p * (dp - (o[:, :, :, i0:i1] * g).sum(-1, keepdim=True))
        dv[:, :, j] += torch.einsum("nkgij,nkgid->nkjd", p, g)
        dk[:, :, j] += torch.einsum("nkgij,nkgid->nkjd", ds, q[:, :, :, i0:i1]) / math.sqrt(D)
        dq[:, :, :, i0:i1] = torch.einsum("nkgij,nkjd->nkgid", ds, kj) / math.sqrt(D)
        if dt is not None:
            per = ds.view(C, case["B"], KV, G, *b.shape).sum(1)
            dt += torch.stack([(per * (b == m)).sum((-1, -2)) for m in range(case["buckets"])], -1)

    def rows(t, h):
        return t.reshape(N, h, S, D).permute(0, 2, 1, 3).reshape(N * S, h * D)

    if not case["train"]:
        return rows(o, H)
    out = [rows(o, H), rows(dq, H), rows(dk, KV), rows(dv, KV)]
    return tuple(out if dt is None else out + [dt.view(C, H, -1)])


def _exact_step(case, st):
    B, H, KV, D, W, sinks = case["B"], case["H"], case["KV"], case["D"], case["window"], case["sinks"]
    k, v = st["k_cache"].double(), st["v_cache"].double()
    out = torch.zeros(B, H, D, dtype=torch.float64, device=DEV)
    of = None if st["table"] is None else _by_distance(case, case["max_distance"])
    for b, pos in enumerate(st["pos"].tolist()):
        at = pos if pos < sinks else sinks + (pos - sinks) % W
        k[b, at], v[b, at] = st["k"][b].double(), st["v"][b].double()
        near = list(range(max(sinks, pos - W + 1), pos + 1))
        tokens = torch.tensor(list(range(min(sinks, pos + 1))) + near, device=DEV)
        slots = torch.where(tokens < sinks, tokens, sinks + (tokens - sinks) % W)
        kb, vb = (t[b, slots].view(-1, KV, D).repeat_interleave(H // KV, 1) for t in (k, v))
        s = torch.einsum("hd,nhd->hn", st["q"][b].double().view(H, D), kb) / math.sqrt(D)
        if of is not None:
            s = s + st["table"].double()[:, of[(pos - tokens).clamp_max(case["max_distance"])]]
        out[b] = torch.einsum("hn,nhd->hd", torch.softmax(s, -1), vb)
    return out.view(B, H * D), k, v


def _exact_scan(case, st):
    x, gate, h0 = (st[k].detach().double() for k in ("x", "gate", "h0"))
    C, T, B, H = x.shape
    f, keep = torch.sigmoid(gate), torch.sigmoid(-gate)
    real = torch.ones(C, T, B, 1, dtype=torch.bool, device=DEV) if st["mask"] is None else st["mask"].unsqueeze(-1)
    states, h = [h0], h0
    y = torch.zeros_like(x)
    for t in range(T):
        h = torch.where(real[:, t], torch.lerp(x[:, t], h, f[:, t]), h)
        states.append(h)
        y[:, t] = torch.where(real[:, t], h, 0.0)
    if not case["train"]:
        return y, h
    dy, g = st["dy"].double(), st["dh"].double()
    dx, dgate = torch.zeros_like(x), torch.zeros_like(x)
    for t in range(T - 1, -1, -1):
        r = real[:, t]
        e = torch.where(r, g + dy[:, t], 0.0)
        dx[:, t] = e * keep[:, t]
        dgate[:, t] = e * (states[t] - x[:, t]) * f[:, t] * keep[:, t]
        g = torch.where(r, e * f[:, t], g)
    return y, h, dx, dgate, g
