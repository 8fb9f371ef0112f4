"""Performance cases of the delta rule's attention and of the dense products of
the layers around it.

Sequence models on this package mix tokens with a state that fades and that
every token corrects before it adds to it, and project to and from that state's
heads.  Four groups of operators of ``catfuse_amd.kernels``:

delta   delta_attention on whole prompts (packed sequences or equal rows), with
        the states it leaves behind
step    delta_attention_step: one token of every running sequence against a
        pool of states
linear  linear: a product with its bias, activation and residual
gated   gated_linear: both projections of a gated feed-forward block, the
        activation of one and its product with the other

``own`` picks between the package's calls and the plain forms, which compute
the same from elementary torch operations in 32 bits (sums of a chunk's log
decays in 64).
"""
from __future__ import annotations

import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CHUNK = 64                       # tokens per block of the plain attention


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # One image's tokens at the repository's transformer width: the
        # smallest prompt, where latency counts.
        dict(name="delta_image", kind="delta", type="f32", form="rows", B=1, N=196, heads=12,
             kv_heads=12, dk=32, dv=32, state=False),
        # fp32 rows with head sizes off every tile, continued from states.
        dict(name="delta_odd", kind="delta", type="f32", form="rows", B=3, N=1237, heads=8,
             kv_heads=8, dk=80, dv=72, state=True),
        # Prompts of a serving batch, packed, of very different lengths, two
        # query heads on each key head.
        dict(name="delta_packed", kind="delta", type="bf16", form="packed", B=24, N=24011,
             heads=16, kv_heads=8, dk=128, dv=128, state=True),
        # One very long document.
        dict(name="delta_long", kind="delta", type="bf16", form="packed", B=1, N=65536, heads=32,
             kv_heads=16, dk=128, dv=128, state=False),
        # The next token of one sequence: latency.
        dict(name="delta_step_one", kind="step", type="f32", B=1, pool=1, heads=12, kv_heads=12,
             dk=32, dv=32),
        # A full serving batch, its states spread over a larger pool.
        dict(name="delta_step_batch", kind="step", type="bf16", B=256, pool=320, heads=32,
             kv_heads=16, dk=128, dv=128),
        # The output projection of one token, added to the stream.
        dict(name="linear_token", kind="linear", type="bf16", M=1, K=4096, N=4096, bias=False,
             activation=None, residual=True),
        # The class head of the benchmark's network over a batch of 32.
        dict(name="linear_head", kind="linear", type="f32", M=32, K=512, N=1000, bias=True,
             activation=None, residual=False),
        # The first layer of the repository's transformer MLP, 4 steps x 32
        # images of 196 tokens.
        dict(name="linear_tokens", kind="linear", type="f16", M=25088, K=384, N=1536, bias=True,
             activation="gelu", residual=False),
        # The output projection of a prompt.
        dict(name="linear_prompt", kind="linear", type="bf16", M=16384, K=4096, N=4096, bias=False,
             activation=None, residual=True),
        # The feed-forward block of a small decoding batch, widths off every
        # tile.
        dict(name="gated_tokens", kind="gated", type="f16", M=7, K=1000, N=2731, bias=True,
             activation="gelu_tanh"),
        # The feed-forward block of a prompt.
        dict(name="gated_prompt", kind="gated", type="bf16", M=8192, K=4096, N=11264, bias=False,
             activation="silu"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _head(rng):
    d = _log(rng, 16, 256)
    return rng.choice([d, 8 * max(2, round(d / 8)), min((32, 64, 128, 256), key=lambda s: abs(s - d))])


def _width(rng, lo, hi):
    d = _log(rng, lo, hi)
    return rng.choice([d, max(lo, d // 8 * 8), max(lo, 2 ** round(math.log2(d)))])


def _head_counts(rng, most):
    kv = _log(rng, 1, most)
    group = rng.choice([1, 1, 2, 4])
    while kv * group > most:
        kv = max(1, kv // 2)
        group = min(group, most)
    return kv * group, kv


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 100)


def draw(rng):
    """One more case of the listed kinds: 1 to 65536 tokens, 1 to 32 heads of
    16 to 256 channels, packed or equal rows; products of 1 to 25088 rows and
    widths of 16 to 16384; every type."""
    kind = rng.choice(["delta", "delta", "delta", "step", "linear", "linear", "gated"])
    t = rng.choice(["bf16", "bf16", "f16", "f32"])
    most = {n: max(_cost(c) for c in listed() if c["kind"] == n) for n in
            ("delta", "step", "linear", "gated")}[kind]
    if kind in ("linear", "gated"):
        c = dict(kind=kind, type=t, M=_log(rng, 1, 25088), K=_width(rng, 16, 8192),
                 N=_width(rng, 16, 16384), bias=rng.random() < 0.5)
        c["activation"] = rng.choice([None, "relu", "silu", "gelu", "gelu_tanh"] if kind == "linear"
                                     else ["silu", "gelu", "gelu_tanh"])
        if kind == "linear":
            c["residual"] = rng.random() < 0.5
        while _cost(c) > most or (t == "f32" and work(c)["flops"] > 3e11):
            c["M"] = (c["M"] + 1) // 2
        return c
    heads, kv = _head_counts(rng, 32)
    dk = _head(rng)
    dv = dk if rng.random() < 0.5 else _head(rng)
    if kind == "delta":
        form = rng.choice(["packed", "rows"])
        B = _log(rng, 1, 64)
        total = max(B, _log(rng, 1, 65536))
        c = dict(kind=kind, type=t, form=form, B=B, N=total if form == "packed" else
                 max(1, total // B), heads=heads, kv_heads=kv, dk=dk, dv=dv,
                 state=rng.random() < 0.5)
        least = B if form == "packed" else 1
        while c["N"] > least and _cost(c) > most:
            c["N"] = max(least, c["N"] // 2)
        return c
    B = _log(rng, 1, 256)
    c = dict(kind=kind, type=t, B=B, pool=B + rng.randint(0, 64), heads=heads, kv_heads=kv, dk=dk,
             dv=dv)
    while c["B"] > 1 and (_cost(c) > most or c["pool"] * heads * dk * dv * 4 > 671088640):
        c["B"] = (c["B"] + 1) // 2
        c["pool"] = c["B"] + min(c["pool"] - c["B"], c["B"])
    return c


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _lengths(case, seed):
    """Lengths of the packed sequences: random shares, one of a single token
    where there are several."""
    B, N = case["B"], case["N"]
    if B == 1:
        return [N]
    g = torch.Generator().manual_seed(7 * seed + B + N)
    w = torch.rand(B, generator=g, dtype=torch.float64) + 0.02
    cut = torch.floor(torch.cumsum(w, 0) / w.sum() * (N - B)).to(torch.int64)
    cut[-1] = N - B
    lens = (torch.diff(cut, prepend=torch.zeros(1, dtype=torch.int64)) + 1).tolist()
    spare = lens[0] - 1                      # the first one gives up all but one token
    lens[0], lens[-1] = 1, lens[-1] + spare
    return lens


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(5 * seed + 2)
    t = TYPES[case["type"]]
    kind = case["kind"]

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    s = {"case": case}
    if kind in ("linear", "gated"):
        M, K, N = case["M"], case["K"], case["N"]
        s["x"] = normal(M, K).to(t)
        names = [("w", "bias")] if kind == "linear" else [("w_gate", "bias_gate"), ("w_up", "bias_up")]
        for w, b in names:
            s[w] = (normal(N, K) * K ** -0.5).to(t)
            s[b] = (0.5 * normal(N)).to(t) if case["bias"] else None
        if kind == "linear":
            s["residual"] = normal(M, N).to(t) if case["residual"] else None
        return s
    H, Hk, dk, dv, B = (case[n] for n in ("heads", "kv_heads", "dk", "dv", "B"))
    if kind == "step":
        lead = (B,)
    else:
        lead = (case["N"],) if case["form"] == "packed" else (B, case["N"])
    # heads as the projections and their norms leave them: keys of length one
    s["q"] = normal(*lead, H, dk).to(t)
    k = normal(*lead, Hk, dk)
    s["k"] = (k / k.norm(dim=-1, keepdim=True)).to(t)
    s["v"] = normal(*lead, Hk, dv).to(t)
    s["beta"] = torch.sigmoid(normal(*lead, H)).to(t)
    # horizons of about 16 to 4096 tokens, each token's own by a factor of e^normal
    e = 4.0 + 8.0 * torch.arange(H, dtype=torch.float64, device="cuda") / H
    s["log_decay"] = (torch.log1p(-torch.exp2(-e)) * torch.exp(0.5 * normal(*lead, H).double())).float()
    s["scale"] = dk ** -0.5
    if kind == "step":
        s["state"] = normal(case["pool"], H, dk, dv)
        s["slots"] = torch.randperm(case["pool"], generator=g, device="cuda")[:B].to(torch.int32)
        return s
    s["cu"], s["longest"] = None, case["N"]
    if case["form"] == "packed":
        lens = _lengths(case, seed)
        s["cu"] = torch.tensor([0] + lens, device="cuda").cumsum(0).to(torch.int32)
        s["longest"] = max(lens)
    s["state"] = normal(B, H, dk, dv) if case["state"] else None
    return s


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------

def _delta_plain(q, k, v, beta, log_decay, scale, state, cu, longest):
    """Blocks of CHUNK tokens.  Within a block the corrections u of its tokens
    solve (I + L) u = beta (v - decayed k S), L the strictly lower part of
    beta decay (k k^T); one product with the inverse of I + L takes the blocks'
    own parts, and a loop over the blocks carries the state."""
    dtype, H, dk, dv = q.dtype, q.shape[-2], q.shape[-1], v.shape[-1]
    dev = q.device
    nc = -(-longest // CHUNK)
    n = torch.arange(nc * CHUNK, device=dev)
    if cu is None:
        B, N = q.shape[:2]
        lens = torch.full((B,), N, device=dev)
        start = torch.arange(B, device=dev) * N
    else:
        start, lens = cu[:-1].long(), torch.diff(cu).long()
        B = lens.shape[0]
    tokens = q.numel() // (H * dk)
    inside = n[None, :] < lens[:, None]                                 # [B, nc*CHUNK]
    at = (start[:, None] + n[None, :]).clamp(max=tokens - 1)

    def blocks(x):
        """[B, H, nc, CHUNK, d], zeros behind a sequence's end."""
        x = x.reshape(tokens, x.shape[-2], x.shape[-1])[at].float() * inside[..., None, None]
        x = x.unflatten(1, (nc, CHUNK)).permute(0, 3, 1, 2, 4)
        return x.repeat_interleave(H // x.shape[1], 1)

    q, k, v, beta = blocks(q) * scale, blocks(k), blocks(v), blocks(beta[..., None])
    fall = torch.cumsum(blocks(log_decay[..., None])[..., 0].double(), -1)      # [B, H, nc, CHUNK]
    i = torch.arange(CHUNK, device=dev)
    upto = i[:, None] >= i[None, :]
    gap = torch.where(upto, fall[..., :, None] - fall[..., None, :], -math.inf)
    fade = torch.exp(gap).float()                                       # 0 above the diagonal
    kt = k.transpose(-1, -2)
    low = beta * fade * (k @ kt) * (i[:, None] > i[None, :])
    inverse = torch.eye(CHUNK, device=dev).expand_as(low)
    size = 1
    while size < CHUNK:          # blocks of `size` are inverted: join them in pairs
        pair = (i[:, None] // size == i[None, :] // size + 1) & (i[:, None] // size % 2 == 1)
        inverse = inverse - inverse @ (low * pair) @ inverse
        size *= 2
    since = torch.exp(fall).float()[..., None]                          # from the block's start
    left = torch.exp(fall[..., -1:] - fall).float()[..., None]          # to the block's end
    own_u, w = inverse @ (beta * v), inverse @ (beta * since * k)
    kt_end = (k * left).transpose(-1, -2)
    whole = since[:, :, :, -1:]
    s = torch.zeros(B, H, dk, dv, device=dev) if state is None else state.float()
    before, us = [], []
    for c in range(nc):
        before.append(s)
        us.append(own_u[:, :, c] - w[:, :, c] @ s)
        s = whole[:, :, c] * s + kt_end[:, :, c] @ us[-1]
    out = (q * since) @ torch.stack(before, 2) + (fade * (q @ kt)) @ torch.stack(us, 2)
    out = out.flatten(2, 3).transpose(1, 2)                             # [B, nc*CHUNK, H, dv]
    if cu is None:
        return out[:, :longest].to(dtype), s
    t = torch.arange(tokens, device=dev)
    b = torch.searchsorted(cu[1:].long(), t, right=True)
    return out[b, t - start[b]].to(dtype), s


def _step_plain(q, k, v, beta, log_decay, scale, state, slots):
    H, slots = q.shape[1], slots.long()
    kf = k.float().repeat_interleave(H // k.shape[1], 1)
    vf = v.float().repeat_interleave(H // v.shape[1], 1)
    s = state[slots] * torch.exp(log_decay)[:, :, None, None]
    u = beta.float()[..., None] * (vf - (kf[:, :, None, :] @ s)[:, :, 0])
    new = s + kf[..., :, None] * u[..., None, :]
    state[slots] = new
    return ((q.float() * scale)[:, :, None, :] @ new)[:, :, 0].to(q.dtype)


def _activate(z, activation):
    if activation == "relu":
        return torch.where(z < 0, 0.0, z)
    if activation == "silu":
        return z / (1 + torch.exp(-z))
    if activation == "gelu":
        return 0.5 * z * (1 + torch.erf(z * 0.5 ** 0.5))
    if activation == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh((2 / math.pi) ** 0.5 * (z + 0.044715 * z * z * z)))
    return z


def _linear_plain(x, w, bias):
    z = x.float() @ w.float().t()
    return z if bias is None else z + bias.float()


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(s):
    case = s["case"]
    kind, act = case["kind"], case.get("activation")
    if own:
        from catfuse_amd import kernels
        if kind == "delta":
            return kernels.delta_attention(s["q"], s["k"], s["v"], s["beta"], s["log_decay"],
                                           scale=s["scale"], state=s["state"], cu_seqlens=s["cu"])
        if kind == "step":
            o = kernels.delta_attention_step(s["q"], s["k"], s["v"], s["beta"], s["log_decay"],
                                             s["state"], slots=s["slots"], scale=s["scale"])
            return o, s["state"]
        if kind == "linear":
            return kernels.linear(s["x"], s["w"], s["bias"], activation=act,
                                  residual=s["residual"])
        return kernels.gated_linear(s["x"], s["w_gate"], s["w_up"], bias_gate=s["bias_gate"],
                                    bias_up=s["bias_up"], activation=act)
    if kind == "delta":
        return _delta_plain(s["q"], s["k"], s["v"], s["beta"], s["log_decay"], s["scale"],
                            s["state"], s["cu"], s["longest"])
    if kind == "step":
        o = _step_plain(s["q"], s["k"], s["v"], s["beta"], s["log_decay"], s["scale"], s["state"],
                        s["slots"])
        return o, s["state"]
    if kind == "linear":
        y = _activate(_linear_plain(s["x"], s["w"], s["bias"]), act)
        return (y if s["residual"] is None else y + s["residual"].float()).to(s["x"].dtype)
    gate = _activate(_linear_plain(s["x"], s["w_gate"], s["bias_gate"]), act)
    return (gate * _linear_plain(s["x"], s["w_up"], s["bias_up"])).to(s["x"].dtype)


# ---------------------------------------------------------------------------
# work, and the definitions in 64 bits
# ---------------------------------------------------------------------------

def work(case):
    e, kind = TYPES[case["type"]].itemsize, case["kind"]
    if kind in ("linear", "gated"):
        M, K, N, n = case["M"], case["K"], case["N"], 1 if kind == "linear" else 2
        out = M * N * (2 if case.get("residual") else 1)
        return {"bytes": e * (M * K + n * N * K + out + n * N * case["bias"]),
                "flops": 2 * n * M * N * K}
    H, Hk, dk, dv, B = (case[n] for n in ("heads", "kv_heads", "dk", "dv", "B"))
    tokens = B if kind == "step" else case["N"] * (1 if case["form"] == "packed" else B)
    states = 2 if kind == "step" else 1 + bool(case["state"])
    return {"bytes": tokens * (e * (H + Hk) * (dk + dv) + (4 + e) * H) + 4 * states * B * H * dk * dv,
            "flops": 6 * tokens * H * dk * dv}


def _delta_exact(s):
    """Token by token, all sequences and heads at once."""
    q, cu, H, dk, dv = s["q"], s["cu"], s["q"].shape[-2], s["q"].shape[-1], s["v"].shape[-1]
    if cu is None:
        B, L = q.shape[:2]
        ends = [(b * L, b * L + L) for b in range(B)]
    else:
        at = cu.tolist()
        ends = list(zip(at, at[1:]))
        B = len(ends)
    L = max(j - i for i, j in ends)
    group = H // s["k"].shape[-2]

    def lay(x, d):
        """[L, B * heads, d] in 64 bits, zeros behind a sequence's end."""
        x = x.reshape(-1, x.shape[-1] if d == 1 else x.shape[-2], d)
        y = torch.zeros(L, B, x.shape[1], d, dtype=torch.float64, device=x.device)
        for b, (i, j) in enumerate(ends):
            y[:j - i, b] = x[i:j].double()
        return y

    def spread(x):                  # key heads to the heads that read them
        return x[:, :, :, None].expand(-1, -1, -1, group, -1).flatten(2, 3).flatten(1, 2)

    q, beta = lay(q, dk).flatten(1, 2)[:, :, None], lay(s["beta"], 1).flatten(1, 2)[:, :, None]
    keep = torch.exp(lay(s["log_decay"], 1)).flatten(1, 2)[:, :, None]
    k, v = spread(lay(s["k"], dk))[:, :, :, None], spread(lay(s["v"], dv))[:, :, None]
    S = torch.zeros(B * H, dk, dv, dtype=torch.float64, device=q.device)
    if s["state"] is not None:
        S += s["state"].flatten(0, 1).double()
    o = torch.empty(L, B * H, 1, dv, dtype=torch.float64, device=q.device)
    for t in range(L):
        S *= keep[t]
        u = (v[t] - torch.bmm(k[t].transpose(1, 2), S)) * beta[t]
        S += k[t] * u
        torch.bmm(q[t], S, out=o[t])
    o = o.unflatten(1, (B, H))[:, :, :, 0] * s["scale"]
    out = [o[:j - i, b] for b, (i, j) in enumerate(ends)]
    return (torch.stack(out) if cu is None else torch.cat(out)), S.unflatten(0, (B, H))


def _step_exact(s):
    state = s["state"].double()
    q, group, slots = s["q"], s["q"].shape[1] // s["k"].shape[1], s["slots"].long()
    out = torch.zeros(q.shape[:2] + (s["v"].shape[-1],), dtype=torch.float64, device=state.device)
    for h in range(q.shape[1]):
        k, v = s["k"][:, h // group].double(), s["v"][:, h // group].double()
        old = state[slots, h] * torch.exp(s["log_decay"][:, h].double())[:, None, None]
        u = s["beta"][:, h].double()[:, None] * (v - (k[:, :, None] * old).sum(1))
        state[slots, h] = old + k[:, :, None] * u[:, None, :]
        out[:, h] = (q[:, h].double()[:, :, None] * state[slots, h]).sum(1) * s["scale"]
    return out, state


def _curve(z, activation):
    """The activations by their own formulas: z times a distribution's value."""
    if activation is None:
        return z
    if activation == "relu":
        return z.clamp(min=0)
    if activation == "silu":
        return z * torch.sigmoid(z)
    if activation == "gelu":
        return z * torch.special.ndtr(z)
    return z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "delta":
        return _delta_exact(s)
    if case["kind"] == "step":
        return _step_exact(s)

    def product(w, bias):
        z = torch.nn.functional.linear(s["x"].double(), s[w].double())
        return z if s[bias] is None else z + s[bias].double()

    if case["kind"] == "linear":
        y = _curve(product("w", "bias"), case["activation"])
        return y if s["residual"] is None else y + s["residual"].double()
    return _curve(product("w_gate", "bias_gate"), case["activation"]) * product("w_up", "bias_up")
