"""Performance cases of the decayed attention and of what prepares its heads.

Sequence models on this package mix tokens with softmax-free attention whose
past fades by a factor of its own for each head.  Three groups of operators of
``catfuse_amd.kernels``:

attn    decay_attention on whole prompts (packed sequences or equal rows),
        with the states it leaves behind
step    decay_attention_step: one token of every running sequence against a
        pool of states
qknorm  qk_norm_rotary: the norms of the query and key heads and their
        position rotation in one pass
rotary  rotary: the rotation alone, positions of one to three axes (time,
        height, width)

``own`` picks between the package's calls and the plain forms, which compute
the same from elementary torch operations in 32 bits (angles in 64).
"""
from __future__ import annotations

import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CHUNK = 128                      # tokens per block of the plain attention


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # One image's tokens at the repository's transformer width: the
        # smallest prompt, where latency counts.
        dict(name="attn_image", kind="attn", type="f32", form="rows", B=1, N=196, heads=12,
             kv_heads=12, dk=32, dv=32, spikes=False, state=False),
        # The benchmark's transformer block: 4 steps x 32 images of 196 spike
        # tokens in the fp16 storage of the fused layers.
        dict(name="attn_spikes", kind="attn", type="f16", form="rows", B=128, N=196, heads=12,
             kv_heads=12, dk=32, dv=32, spikes=True, state=False),
        # fp32 rows with head sizes off every tile, continued from states.
        dict(name="attn_odd", kind="attn", type="f32", form="rows", B=3, N=1237, heads=8,
             kv_heads=8, dk=80, dv=72, spikes=False, state=True),
        # Prompts of a serving batch, packed, of very different lengths, with
        # four query heads on each key head.
        dict(name="attn_packed", kind="attn", type="bf16", form="packed", B=24, N=24011, heads=16,
             kv_heads=4, dk=128, dv=128, spikes=False, state=True),
        # One very long document.
        dict(name="attn_long", kind="attn", type="bf16", form="packed", B=1, N=65536, heads=32,
             kv_heads=8, dk=128, dv=128, spikes=False, state=False),
        # The next token of one sequence: latency.
        dict(name="step_one", kind="step", type="f32", B=1, pool=1, heads=12, kv_heads=12, dk=32,
             dv=32),
        # An odd number of sequences and head sizes.
        dict(name="step_odd", kind="step", type="f16", B=37, pool=50, heads=12, kv_heads=6, dk=80,
             dv=72),
        # A full serving batch, its states spread over a larger pool.
        dict(name="step_batch", kind="step", type="bf16", B=256, pool=320, heads=32, kv_heads=8,
             dk=128, dv=128),
        # A few tokens of a decoding batch.
        dict(name="qknorm_tokens", kind="qknorm", type="f16", N=7, heads=12, kv_heads=12, d=32,
             rot=32, axes=1, fused=True),
        # A prompt, its heads lying in one fused projection.
        dict(name="qknorm_prompt", kind="qknorm", type="bf16", N=16384, heads=32, kv_heads=8,
             d=128, rot=128, axes=1, fused=True),
        # A batch of images: rows and columns of 14 x 14 patches.
        dict(name="rotary_image", kind="rotary", type="f32", N=6272, heads=12, d=32, rot=32,
             axes=2, fused=False),
        # A video clip: 8 frames of 45 x 80 patches.
        dict(name="rotary_video", kind="rotary", type="bf16", N=28800, heads=16, d=128, rot=128,
             axes=3, fused=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _head(rng):
    d = _log(rng, 16, 256)
    return rng.choice([d, 8 * max(2, round(d / 8)), min((32, 64, 128, 256), key=lambda s: abs(s - d))])


def _head_counts(rng, most):
    kv = _log(rng, 1, most)
    group = rng.choice([1, 1, 2, 4, 8])
    while kv * group > most:
        kv = max(1, kv // 2)
        group = min(group, most)
    return kv * group, kv


def draw(rng):
    """One more case of the listed kinds: 1 to 65536 tokens, 1 to 32 heads of
    16 to 256 channels, every type, packed or equal rows, one to three axes."""
    kind = rng.choice(["attn", "attn", "attn", "step", "step", "qknorm", "rotary"])
    t = rng.choice(["bf16", "bf16", "f16", "f32"])
    heads, kv = _head_counts(rng, 32)
    if kind == "attn":
        form = rng.choice(["packed", "rows"])
        c = dict(kind=kind, type=t, form=form, B=_log(rng, 1, 64), N=0, heads=heads, kv_heads=kv,
                 dk=_head(rng), dv=_head(rng), spikes=rng.random() < 0.2,
                 state=rng.random() < 0.5)
        if rng.random() < 0.5:
            c["dv"] = c["dk"]
        total = max(c["B"], _log(rng, 1, 65536))
        c["N"] = total if form == "packed" else max(1, total // c["B"])
        big = work(listed()[4])["bytes"]
        while c["N"] > 1 and max(work(c)["bytes"], work(c)["flops"] / 100) > big:
            c["N"] = c["N"] // 2
        c["N"] = max(c["N"], c["B"]) if form == "packed" else c["N"]
        return c
    if kind == "step":
        B = _log(rng, 1, 256)
        c = dict(kind=kind, type=t, B=B, pool=B + rng.randint(0, 64), heads=heads, kv_heads=kv,
                 dk=_head(rng), dv=_head(rng))
        while c["pool"] * c["heads"] * c["dk"] * c["dv"] * 4 > 671088640:
            c["B"] = (c["B"] + 1) // 2
            c["pool"] = c["B"] + min(c["pool"] - c["B"], c["B"])
            if c["B"] == 1:
                break
        return c
    axes = rng.choice([1, 2, 3])
    d = max(8, _head(rng) // 2 * 2)
    rot = d if rng.random() < 0.7 else max(2 * axes, d // 4 * 2)
    c = dict(kind=kind, type=t, N=_log(rng, 1, 30000), heads=heads, d=d, rot=rot, axes=axes,
             fused=rng.random() < 0.5)
    if kind == "qknorm":
        c["kv_heads"] = kv
    return c


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _lengths(case, seed):
    """Lengths of the packed sequences: about 1 to twice the mean, one of a
    single token where there are several."""
    B, N = case["B"], case["N"]
    g = torch.Generator().manual_seed(7 * seed + B + N)
    if B == 1:
        return [N]
    w = torch.rand(B, generator=g, dtype=torch.float64) + 0.02
    cut = torch.floor(torch.cumsum(w, 0) / w.sum() * (N - B)).to(torch.int64)
    cut[-1] = N - B
    lens = (torch.diff(cut, prepend=torch.zeros(1, dtype=torch.int64)) + 1).tolist()
    spare = lens[0] - 1                      # the first one gives up all but one token
    lens[0], lens[-1] = 1, lens[-1] + spare
    return lens


def _sections(pairs, axes):
    """Pairs of channels for each axis: the first gets the smallest part."""
    if axes == 1:
        return None
    rest = pairs * 3 // 8 if axes == 3 else pairs // 2
    return (pairs - (axes - 1) * rest,) + (rest,) * (axes - 1)


def _log_decay(heads):
    """log(1 - 2^-(4 + 8 h / heads)): horizons of 16 to 4096 tokens."""
    e = 4.0 + 8.0 * torch.arange(heads, dtype=torch.float64, device="cuda") / heads
    return torch.log1p(-torch.exp2(-e)).float()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(3 * seed + 1)
    t = TYPES[case["type"]]
    kind = case["kind"]

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda").to(t)

    s = {"case": case}
    if kind == "attn":
        H, Hk, dk, dv, N, B = (case[n] for n in ("heads", "kv_heads", "dk", "dv", "N", "B"))
        lead = (N,) if case["form"] == "packed" else (B, N)
        if case["spikes"]:          # firing rates of live layers
            for n, h, d in (("q", H, dk), ("k", Hk, dk), ("v", Hk, dv)):
                s[n] = (torch.rand(lead + (h, d), generator=g, device="cuda") < 0.25).to(t)
        else:
            s |= {"q": normal(*lead, H, dk), "k": normal(*lead, Hk, dk),
                  "v": normal(*lead, Hk, dv)}
        s["scale"] = 0.125 if case["spikes"] else dk ** -0.5
        s["cu"], s["longest"] = None, N
        if case["form"] == "packed":
            lens = _lengths(case, seed)
            s["cu"] = torch.tensor([0] + lens, device="cuda").cumsum(0).to(torch.int32)
            s["longest"] = max(lens)
        s["state"] = torch.randn((B, H, dk, dv), generator=g, device="cuda") if case["state"] \
            else None
        s["log_decay"] = _log_decay(H)
        return s
    if kind == "step":
        H, Hk, dk, dv, B = (case[n] for n in ("heads", "kv_heads", "dk", "dv", "B"))
        s |= {"q": normal(B, H, dk), "k": normal(B, Hk, dk), "v": normal(B, Hk, dv)}
        s["state"] = torch.randn((case["pool"], H, dk, dv), generator=g, device="cuda")
        s["slots"] = torch.randperm(case["pool"], generator=g, device="cuda")[:B].to(torch.int32)
        s["log_decay"], s["scale"] = _log_decay(H), dk ** -0.5
        return s
    N, H, d, pairs, axes = case["N"], case["heads"], case["d"], case["rot"] // 2, case["axes"]
    Hk = case.get("kv_heads", 0)
    if case["fused"]:               # heads of one projection that holds more than is rotated
        x = normal(N, (H + 2 * max(Hk, 1)) * d)
        s["q"] = x[:, :H * d].unflatten(1, (H, d))
        s["k"] = x[:, H * d:(H + Hk) * d].unflatten(1, (Hk, d)) if Hk else None
    else:
        s["q"], s["k"] = normal(N, H, d), normal(N, Hk, d) if Hk else None
    if kind == "qknorm":
        s["q_weight"] = 1 + 0.1 * torch.randn(d, generator=g, device="cuda")
        s["k_weight"] = 1 + 0.1 * torch.randn(d, generator=g, device="cuda")
    s["sections"] = _sections(pairs, axes)
    n = torch.arange(N, device="cuda", dtype=torch.int64)
    if axes == 1:                   # a prompt somewhere in a long context
        first = torch.randint(0, 1 << 20, (1,), generator=g, device="cuda")
        s["positions"] = n + first
    else:                           # rows, columns (and frames) of a grid of patches
        h, w = (14, 14) if axes == 2 else (45, 80)
        first = torch.randint(0, 64, (axes, 1), generator=g, device="cuda")
        grid = torch.stack([n // (h * w), n // w % h, n % w][3 - axes:])
        s["positions"] = grid + first
    s["freqs"] = 10000.0 ** (-torch.arange(pairs, dtype=torch.float64, device="cuda") / pairs)
    return s


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------

def _attention_plain(q, k, v, log_decay, scale, state, cu, longest):
    """Blocks of CHUNK tokens: within a block all pairs, before it the block
    states, joined by one product over the blocks."""
    dtype, H, dk, dv = q.dtype, q.shape[-2], q.shape[-1], v.shape[-1]
    dev, f = q.device, log_decay.float()
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

    def blocks(x, heads):
        x = x.reshape(tokens, x.shape[-2], x.shape[-1])[at].float() * inside[..., None, None]
        x = x.unflatten(1, (nc, CHUNK)).permute(0, 3, 1, 2, 4)
        return x.repeat_interleave(heads // x.shape[1], 1)              # [B, H, nc, CHUNK, d]

    q, k, v = blocks(q, H) * scale, blocks(k, H), blocks(v, H)
    i = torch.arange(CHUNK, device=dev)
    back = (i[:, None] - i[None, :]).float()
    fade = torch.where(back >= 0, torch.exp(f[:, None, None] * back.clamp(min=0)), 0.0)
    out = ((q @ k.transpose(-1, -2)) * fade[:, None]) @ v
    to_end = torch.exp(f[:, None] * (CHUNK - 1 - i).float())            # [H, CHUNK]
    kv = (k * to_end[:, None, :, None]).transpose(-1, -2) @ v           # [B, H, nc, dk, dv]
    c = torch.arange(nc, device=dev)
    gap = (c[:, None] - c[None, :] - 1).float() * CHUNK
    join = torch.where(gap >= 0, torch.exp(f[:, None, None] * gap.clamp(min=0)), 0.0)
    before = (join @ kv.flatten(3)).unflatten(3, (dk, dv))
    if state is not None:
        first = torch.exp(f[:, None] * (c * CHUNK).float())
        before = before + first[:, :, None, None] * state.float()[:, :, None]
    out = out + ((q * torch.exp(f[:, None] * (i + 1).float())[:, None, :, None]) @ before)
    left = (lens[:, None] - 1 - n[None, :]).clamp(min=0).float()
    left = torch.exp(f[None, :, None] * left[:, None, :])               # [B, H, nc*CHUNK]
    last = (k.flatten(2, 3) * left[..., None]).transpose(-1, -2) @ v.flatten(2, 3)
    if state is not None:
        last = last + torch.exp(f[None, :] * lens[:, None].float())[..., None, None] * state
    out = out.flatten(2, 3).transpose(1, 2)                             # [B, nc*CHUNK, H, dv]
    if cu is None:
        return out[:, :longest].to(dtype), last
    t = torch.arange(tokens, device=dev)
    b = torch.searchsorted(cu[1:].long(), t, right=True)
    return out[b, t - start[b]].to(dtype), last


def _step_plain(q, k, v, log_decay, scale, state, slots):
    H, slots = q.shape[1], slots.long()
    kf = k.float().repeat_interleave(H // k.shape[1], 1)
    vf = v.float().repeat_interleave(H // v.shape[1], 1)
    new = state[slots] * torch.exp(log_decay)[:, None, None] + kf[..., :, None] * vf[..., None, :]
    state[slots] = new
    return ((q.float() * scale)[:, :, None, :] @ new)[:, :, 0].to(q.dtype)


def _turn_plain(x, positions, freqs, sections):
    """The first 2 * len(freqs) channels, channel i with channel i + pairs."""
    pairs = freqs.shape[0]
    if sections is None:
        angle = positions.double()[:, None] * freqs
    else:
        axis = torch.repeat_interleave(torch.arange(len(sections), device=x.device),
                                       torch.tensor(sections, device=x.device),
                                       output_size=pairs)
        angle = positions.double()[axis].t() * freqs
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    a, b, rest = x[..., :pairs], x[..., pairs:2 * pairs], x[..., 2 * pairs:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)


def _norm_plain(x, weight, eps):
    x = x.float()
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * weight


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

EPS = 1e-6


def run(s):
    kind = s["case"]["kind"]
    if own:
        from catfuse_amd import kernels
        if kind == "attn":
            return kernels.decay_attention(s["q"], s["k"], s["v"], s["log_decay"],
                                           scale=s["scale"], state=s["state"],
                                           cu_seqlens=s["cu"])
        if kind == "step":
            o = kernels.decay_attention_step(s["q"], s["k"], s["v"], s["log_decay"], s["state"],
                                             slots=s["slots"], scale=s["scale"])
            return o, s["state"]
        if kind == "qknorm":
            return kernels.qk_norm_rotary(s["q"], s["k"], s["positions"], s["freqs"],
                                          q_weight=s["q_weight"], k_weight=s["k_weight"],
                                          eps=EPS, sections=s["sections"])
        return kernels.rotary(s["q"], s["positions"], s["freqs"], sections=s["sections"])
    if kind == "attn":
        return _attention_plain(s["q"], s["k"], s["v"], s["log_decay"], s["scale"], s["state"],
                                s["cu"], s["longest"])
    if kind == "step":
        o = _step_plain(s["q"], s["k"], s["v"], s["log_decay"], s["scale"], s["state"],
                        s["slots"])
        return o, s["state"]
    if kind == "qknorm":
        return tuple(_turn_plain(_norm_plain(x, w, EPS), s["positions"], s["freqs"],
                                 s["sections"]).to(x.dtype)
                     for x, w in ((s["q"], s["q_weight"]), (s["k"], s["k_weight"])))
    return _turn_plain(s["q"].float(), s["positions"], s["freqs"],
                       s["sections"]).to(s["q"].dtype)


# ---------------------------------------------------------------------------
# work, and the definitions in 64 bits
# ---------------------------------------------------------------------------

def work(case):
    e = TYPES[case["type"]].itemsize
    H, kind = case["heads"], case["kind"]
    if kind in ("attn", "step"):
        Hk, dk, dv, B = (case[n] for n in ("kv_heads", "dk", "dv", "B"))
        tokens = B if kind == "step" else case["N"] * (1 if case["form"] == "packed" else B)
        states = 2 if kind == "step" else 1 + bool(case["state"])
        return {"bytes": tokens * e * (H * (dk + dv) + Hk * (dk + dv)) + 4 * states * B * H * dk * dv,
                "flops": 4 * tokens * H * dk * dv}
    n = case["N"] * (H + case.get("kv_heads", 0)) * case["d"]
    return {"bytes": 2 * n * e + 8 * case["axes"] * case["N"],
            "flops": (7 if kind == "qknorm" else 3) * n}


def _attention_exact(s):
    """sum over s <= t of decay^(t - s) (q_t . k_s) v_s, pair by pair, and
    decay^(t + 1) q_t S_0."""
    q, k, v, cu = s["q"], s["k"], s["v"], s["cu"]
    H, group = q.shape[-2], q.shape[-2] // k.shape[-2]
    if cu is None:
        spans = [(b, q[b], k[b], v[b]) for b in range(q.shape[0])]
    else:
        ends = cu.tolist()
        spans = [(b, q[i:j], k[i:j], v[i:j]) for b, (i, j) in enumerate(zip(ends, ends[1:]))]
    outs, states = [], []
    for b, qs, ks, vs in spans:
        L = qs.shape[0]
        pos = torch.arange(L, dtype=torch.float64, device=q.device)
        o = torch.zeros(L, H, v.shape[-1], dtype=torch.float64, device=q.device)
        left = torch.zeros(H, q.shape[-1], v.shape[-1], dtype=torch.float64, device=q.device)
        for h in range(H):
            f = s["log_decay"][h].double()
            qh, kh, vh = (x[:, i].double() for x, i in ((qs, h), (ks, h // group), (vs, h // group)))
            kt = kh.t().contiguous()
            for i in range(0, L, 2048):
                j = min(i + 2048, L)
                gap = pos[i:j, None] - pos[None, :j]
                w = torch.where(gap >= 0, torch.exp(f * gap.clamp(min=0)), 0.0)
                o[i:j, h] = ((qh[i:j] @ kt[:, :j]) * w) @ vh[:j]
            left[h] = (kt * torch.exp(f * (L - 1 - pos))) @ vh
            if s["state"] is not None:
                s0 = s["state"][b, h].double()
                o[:, h] += torch.exp(f * (pos + 1))[:, None] * (qh @ s0)
                left[h] += torch.exp(f * L) * s0
        outs.append(o * s["scale"])
        states.append(left)
    return (torch.stack(outs) if cu is None else torch.cat(outs)), torch.stack(states)


def _step_exact(s):
    state = s["state"].double()
    out = torch.zeros(s["q"].shape[:2] + (s["v"].shape[-1],), dtype=torch.float64,
                      device=state.device)
    group = s["q"].shape[1] // s["k"].shape[1]
    for h in range(s["q"].shape[1]):
        q, k, v = s["q"][:, h].double(), s["k"][:, h // group].double(), s["v"][:, h // group].double()
        slots = s["slots"].long()
        new = state[slots, h] * math.exp(float(s["log_decay"][h])) + k[:, :, None] * v[:, None, :]
        state[slots, h] = new
        out[:, h] = (q[:, :, None] * new).sum(1) * s["scale"]
    return out, state


def _turn_exact(x, s):
    """Each pair of channels as a complex number times exp(i position freq)."""
    pairs = s["freqs"].shape[0]
    pos = s["positions"].double().reshape(-1, x.shape[0])
    parts, at = [], 0
    for a, n in enumerate(s["sections"] or (pairs,)):
        parts.append(pos[a][:, None] * s["freqs"][at:at + n][None])
        at += n
    angle = torch.cat(parts, 1)
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]
    z = torch.complex(x[..., :pairs].contiguous(), x[..., pairs:2 * pairs].contiguous()) * turn
    return torch.cat([z.real, z.imag, x[..., 2 * pairs:]], -1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "attn":
        return _attention_exact(s)
    if case["kind"] == "step":
        return _step_exact(s)
    if case["kind"] == "rotary":
        return _turn_exact(s["q"].double(), s)
    out = []
    for x, w in ((s["q"].double(), s["q_weight"]), (s["k"].double(), s["k_weight"])):
        x = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS) * w.double()
        out.append(_turn_exact(x, s))
    return tuple(out)
