"""Sequence operators: attention whose past fades by head, and its heads.

The spiking self-attention core (`runtime.spike_attention_lif`) multiplies
Q, K and V of one image without a softmax and without an order.  These are its
relatives for ordered tokens: causal, with a decay for each head, over whole
prompts (`decay_attention`) and one token at a time (`decay_attention_step`),
and what its heads go through before: the norm of each head and the rotation
by the token's position on one to three axes (`qk_norm_rotary`, `rotary`).

Inference only, like the rest of the package: an input that requires a
gradient is refused while gradients are recorded.  Everything runs on the
current stream of the inputs' device and neither waits for the GPU nor reads
values back, so calls can be captured into a HIP graph; what is wrong with
values in device memory (offsets, slots) is handled on the device, as each
function says.  No counterpart in the reference.
"""
from __future__ import annotations

from typing import Optional, Sequence

import torch
# Tensors that a kernel writes count as changed, as after an in-place operation
# of torch: the package's copies of a fused output and autograd's saved tensors
# go by that count.
from torch.autograd.graph import increment_version as _changed

from catfuse_amd import _hip
from catfuse_amd._hip import check, ptr
from catfuse_amd.runtime import _t0, _t1

# element types: the `dtype` of the argument blocks
_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_POSITIONS = {torch.int32: 0, torch.int64: 1, torch.float32: 2}

MAX_HEADS = 4096            # CF_SEQ_MAX_HEADS
MAX_KEY_DIM = 256           # CF_DECAY_MAX_DK
MAX_VALUE_DIM = 1024        # CF_DECAY_MAX_DV
MAX_SEQUENCES = 65535       # CF_DECAY_MAX_SEQS
MAX_TOKENS = 2000000000     # CF_DECAY_MAX_TOKENS
CHUNK = 64                  # CF_DECAY_CHUNK
SPAN_BYTES = 48             # CF_DECAY_SPAN_BYTES
MAX_TOKEN_STRIDE = 8000000  # CF_DECAY_MAX_TOKEN_STRIDE
MAX_ROTARY_DIM = 512        # CF_ROTARY_MAX_DIM
MAX_AXES = 3                # CF_ROTARY_MAX_AXES


# Launch plans: the checked, packed static arguments of a call by what its
# tensors look like (shapes, strides, types, devices), so that a repeated call
# skips the checks; addresses are taken anew for each call.
_PLANS: dict = {}
_Tensor = torch.Tensor


def _looks(t):
    """What a plan depends on of a tensor (or of None)."""
    return None if t is None else (t.shape, t.stride(), t.dtype, t.device, t.requires_grad)


def _keep(key, plan):
    if len(_PLANS) >= 512:
        _PLANS.clear()
    _PLANS[key] = plan
    return plan


def _at(t) -> int:
    return 0 if t is None else t.data_ptr() if type(t) is _Tensor else ptr(t)


# ---------------------------------------------------------------------------
# checks
# ---------------------------------------------------------------------------

def _require(t, name: str, dtype, dev=None) -> None:
    """A tensor of one of the dtypes, on `dev`, without a gradient."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.dtype not in dtype:
        raise TypeError(f"{name} must be {' or '.join(str(d) for d in dtype)}, got {t.dtype}")
    if dev is not None and t.device != dev:
        raise RuntimeError(f"{name} is on {t.device}, the first input on {dev}")
    if t.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{name} requires a gradient: this operator is for inference (call it "
                           "under torch.no_grad() or detach the input)")


def _require_gpu(t, name: str) -> None:
    """Last of the checks: what is wrong with a call is said without a GPU."""
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a GPU tensor (catfuse_amd has no CPU path)")


def _require_rows(t, name: str) -> None:
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        raise ValueError(f"the last dimension of {name} must be contiguous")


def _span(t):
    """Bytes [first, last) that a tensor's elements lie in."""
    if t.numel() == 0:
        return 0, 0
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def _between_rows(a, b) -> bool:
    """Whether two tensors lie side by side in the same rows (heads of one
    fused projection): rows of equal strides, the heads of one between the
    ends of the other's."""
    if a.ndim != b.ndim or a.ndim < 3 or a.dtype != b.dtype:
        return False
    steps = {(s, t) for n, m, s, t in zip(a.shape, b.shape, a.stride()[:-2], b.stride()[:-2])
             if n > 1 or m > 1}
    if not steps or any(s != t or s <= 0 for s, t in steps):
        return False
    row = min(s for s, _ in steps)
    if any(s % row for s, _ in steps):
        return False
    wide = [sum((n - 1) * s for n, s in zip(t.shape[-2:], t.stride()[-2:])) + 1 for t in (a, b)]
    off, part = divmod(b.data_ptr() - a.data_ptr(), a.element_size())
    return part == 0 and off % row >= wide[0] and off % row + wide[1] <= row


def _require_apart(out, name: str, inputs) -> None:
    a, b = _span(out)
    for other in inputs:
        if other is not None:
            c, d = _span(other)
            if a < d and c < b and not _between_rows(out, other):
                raise ValueError(f"{name} overlaps the memory of an input")


def _require_distinct(t, name: str) -> None:
    """No two elements of an output in one place (an expanded tensor, rows
    that overlap)."""
    reach = 0
    for n, s in sorted(((n, s) for n, s in zip(t.shape, t.stride()) if n > 1),
                       key=lambda p: p[1]):
        if s <= reach:
            raise ValueError(f"elements of {name} overlap each other")
        reach += (n - 1) * s


def _require_output(out, name: str, shape, like) -> None:
    if out is None:
        return
    _require(out, name, (like.dtype,), like.device)
    if tuple(out.shape) != tuple(shape):
        raise ValueError(f"{name} has shape {tuple(out.shape)}, expected {tuple(shape)}")
    _require_rows(out, name)
    _require_distinct(out, name)


def _require_attention(q, k, v, log_decay, ndims):
    """Checks of what both forms of the attention share; the device."""
    _require(q, "q", _DTYPES)
    dev = q.device
    _require(k, "k", (q.dtype,), dev)
    _require(v, "v", (q.dtype,), dev)
    _require(log_decay, "log_decay", (torch.float32,), dev)
    if q.ndim not in ndims or k.ndim != q.ndim or v.ndim != q.ndim:
        raise ValueError(f"q, k and v must have {' or '.join(str(n) for n in ndims)} dimensions, "
                         f"got {q.ndim}, {k.ndim} and {v.ndim}")
    H, Hk, dk, dv = q.shape[-2], k.shape[-2], q.shape[-1], v.shape[-1]
    if k.shape[:-2] != q.shape[:-2] or v.shape[:-1] != k.shape[:-1] or k.shape[-1] != dk:
        raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not "
                         "belong together")
    if Hk < 1 or H < 1 or H % Hk or H > MAX_HEADS:
        raise ValueError(f"{H} query heads over {Hk} key heads (at most {MAX_HEADS}, a multiple)")
    if not 1 <= dk <= MAX_KEY_DIM or not 1 <= dv <= MAX_VALUE_DIM:
        raise ValueError(f"head sizes {dk} and {dv}: at most {MAX_KEY_DIM} and {MAX_VALUE_DIM}")
    if log_decay.shape != (H,) or not log_decay.is_contiguous():
        raise ValueError(f"log_decay must be a contiguous tensor of {H} values")
    for t, name in ((q, "q"), (k, "k"), (v, "v")):
        _require_rows(t, name)
    return dev


def _require_index(t, name: str, n: int, dev) -> None:
    _require(t, name, (torch.int32, torch.int64), dev)
    if t.shape != (n,) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous tensor of {n} values")


def _call(fn, what: str, dev, args) -> None:
    """One launch on the current stream of `dev`, which is made the current
    device for it."""
    if dev.index == torch.cuda.current_device():
        check(fn(args), what)
    else:
        with torch.cuda.device(dev):
            check(fn(args), what)


# ---------------------------------------------------------------------------
# attention with a decay for each head
# ---------------------------------------------------------------------------

def _segment(seqs: int, tokens: int, packed: bool, heads: int, dk: int, dv: int):
    """(tokens a segment, segments in all); (0, 0): whole sequences.

    A workgroup takes a segment of one head and `width` columns; the segments'
    own states cost a further pass over k and v (about half of the outputs'
    time), so sequences are split where they leave most of the card idle, into
    about as many workgroups as run at once.  Measured (us, bf16, heads of
    128): one sequence of 65536 tokens, 32 heads: segments of 2048 tokens 777,
    4096 766, 8192 852; 24 packed ones of 24011 tokens, 16 heads: whole 205,
    384 187, 512 179, 768 173, 1024 177; fp32, 3 sequences of 1237, 8 heads of 80: whole
    212, 64 42, 128 45, 192 58; one of 196, 12 heads of 32: whole 22, 64 18.
    (Where splitting ends, 4 at_once workgroups of packed sequences and an eighth
    of that of equal rows, is not measured.)"""
    width = 32 if dk <= 32 else 64 if dk <= 64 else 128
    columns = heads * -(-dv // width)          # workgroups of one segment
    at_once = 2048 if dk <= 32 else 1024 if dk <= 64 else 512 if dk <= 128 else 256
    if tokens <= 2 * CHUNK or seqs * columns * (1 if packed else 8) > 4 * at_once:
        return 0, 0
    total = tokens if packed else seqs * tokens
    segment = max(1, -(-total * columns // (at_once * CHUNK))) * CHUNK
    if segment >= tokens:
        return 0, 0
    return segment, tokens // segment + seqs if packed else seqs * -(-tokens // segment)


def decay_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor, *,
                    scale: Optional[float] = None, state: Optional[torch.Tensor] = None,
                    cu_seqlens: Optional[torch.Tensor] = None,
                    out: Optional[torch.Tensor] = None, return_state: bool = True):
    """Causal attention without a softmax, the past fading by exp(log_decay)
    a token:

        S_t = exp(log_decay[h]) S_{t-1} + k_t v_t^T,    out_t = scale q_t S_t

    for each sequence and head, over whole prompts.

    q [B, N, H, dk], k [B, N, Hk, dk], v [B, N, Hk, dv]: B sequences of N
    tokens; or, with cu_seqlens, [tokens, H, dk] and so on: packed sequences,
    number b the rows cu_seqlens[b] .. cu_seqlens[b + 1] - 1.  Query head h
    reads key head h // (H // Hk).  fp32, fp16 or bf16, all of one type; the
    last dimension contiguous, other strides free (tokens of a sequence at most
    8,000,000 elements apart).  dk <= 256, dv <= 1024.
    log_decay fp32 [H]: 0 keeps everything, -inf only the token itself; above 0
    the past grows (exp(64 log_decay), scale times it too, has to be a number of
    fp32: log_decay up to 1.38).
    scale: dk ** -0.5 if None.
    state: fp32 [sequences, H, dk, dv], S before the first token (None: zeros).
    cu_seqlens: int32 or int64 [sequences + 1], in device memory and therefore
    not checked: offsets are clamped to 0 .. tokens, one below its predecessor
    counts as that.  Rows of no sequence are zero in a new output and
    stay as they are in one given as `out`.
    out: a tensor for the output, apart from the inputs.

    Returns (out [.., H, dv], state after the last token), or out alone
    without return_state.  Sums and states are fp32, products exact to 2^-24 of
    their factors for every type; a token that holds an infinity or NaN does not
    reach the tokens before it, and what an infinity (or an overflow) does reach
    may be NaN where the formula gives an infinity.
    Long sequences of a small batch are computed in segments side by side, with
    a workspace of a state [H, dk, dv] for each, from torch's allocator (32 heads
    of 128: 36 MB for one prompt of 65536 tokens, 168 MB for 64 packed ones)."""
    scale = None if scale is None else float(scale)
    try:
        key = (decay_attention, _looks(q), _looks(k), _looks(v), _looks(log_decay), _looks(state),
               _looks(cu_seqlens), _looks(out), scale, return_state, torch.is_grad_enabled())
        plan = _PLANS.get(key)
    except (AttributeError, TypeError):      # not tensors: the checks say which
        key = plan = None
    if plan is None:
        plan = _attention_plan(q, k, v, log_decay, scale, state, cu_seqlens, out)
        if key is not None:
            _keep(key, plan)
    dev, shape, state_shape, ws_bytes, tail = plan
    given = out is not None
    if given:
        _require_apart(out, "out", (q, k, v, log_decay, state, cu_seqlens))
    else:
        out = torch.empty(shape, dtype=q.dtype, device=dev)
    _require_gpu(q, "q")
    left = torch.empty(state_shape, dtype=torch.float32, device=dev) if return_state else None
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev) if ws_bytes else None
    if state_shape[0] == 0:                  # no sequences: no row belongs to one
        if not given:
            out.zero_()
        return (out, left) if return_state else out
    ev = _t0()
    args = _hip.DECAY_ATTENTION_ARGS[0].pack(
        _at(q), _at(k), _at(v), _at(log_decay), _at(state), _at(left), _at(out), _at(cu_seqlens),
        _at(ws), _hip.stream(dev)) + tail
    _call(_hip.lib().cf_decay_attention, "cf_decay_attention", dev, args)
    if given:
        _changed(out)
    if ev is not None:
        H, Hk, dk, dv = q.shape[-2], k.shape[-2], q.shape[-1], v.shape[-1]
        rows = q.numel() // (H * dk)
        _t1("decay_attention", ev, flops=4 * rows * H * dk * dv,
            nbytes=q.element_size() * rows * (H + Hk) * (dk + dv) +
            4 * state_shape[0] * H * dk * dv * ((state is not None) + return_state))
    return (out, left) if return_state else out


def _attention_plan(q, k, v, log_decay, scale, state, cu_seqlens, out):
    """(device, shapes of the output and of the states, workspace bytes, packed
    arguments) of a checked call."""
    dev = _require_attention(q, k, v, log_decay, (4,) if cu_seqlens is None else (3,))
    H, Hk, dk, dv = q.shape[-2], k.shape[-2], q.shape[-1], v.shape[-1]
    packed = cu_seqlens is not None
    if packed:
        if not isinstance(cu_seqlens, torch.Tensor) or cu_seqlens.ndim != 1 or \
                cu_seqlens.shape[0] < 1:
            raise ValueError("cu_seqlens must be a one-dimensional tensor of offsets")
        B, N = cu_seqlens.shape[0] - 1, q.shape[0]
        _require_index(cu_seqlens, "cu_seqlens", B + 1, dev)
    else:
        B, N = q.shape[:2]
    if B > MAX_SEQUENCES:
        raise ValueError(f"{B} sequences (at most {MAX_SEQUENCES})")
    if state is not None:
        _require(state, "state", (torch.float32,), dev)
        if state.shape != (B, H, dk, dv) or not state.is_contiguous():
            raise ValueError(f"state must be contiguous [{B}, {H}, {dk}, {dv}]")
    shape = tuple(q.shape[:-1]) + (dv,)
    _require_output(out, "out", shape, q)
    for t, name in ((q, "q"), (k, "k"), (v, "v"), (out, "out")):
        if t is not None and t.stride(-3) > MAX_TOKEN_STRIDE and t.shape[-3] > 1:
            raise ValueError(f"tokens of {name} lie {t.stride(-3)} elements apart (at most "
                             f"{MAX_TOKEN_STRIDE})")
    if N > MAX_TOKENS:
        raise ValueError(f"{N} tokens (at most {MAX_TOKENS})")

    def steps(t):
        # (a dimension of one element may have any stride: a plain one)
        return (t.stride(0) if not packed and B > 1 else 0,
                t.stride(-3) if N > 1 else t.shape[-1],
                t.stride(-2) if t.shape[-2] > 1 else 0)
    # a new output is contiguous
    o = steps(out) if out is not None else (0 if packed else N * H * dv, H * dv, dv)
    segment, segments = _segment(B, N, packed, H, dk, dv)
    ws_bytes = segments * (4 * H * dk * dv + SPAN_BYTES)
    tail = _hip.DECAY_ATTENTION_ARGS[1].pack(
        packed and cu_seqlens.dtype == torch.int64, out is None, _DTYPES[q.dtype], B, N, H, Hk, dk,
        dv, *steps(q), *steps(k), *steps(v), *o, segment, ws_bytes,
        float(dk ** -0.5 if scale is None else scale))
    return dev, shape, (B, H, dk, dv), ws_bytes, tail


def decay_attention_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                         log_decay: torch.Tensor, state: torch.Tensor, *,
                         slots: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                         out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """`decay_attention` for one token of each running sequence, against a
    pool of states that is updated in place:

        S = exp(log_decay[h]) S + k v^T,    out = scale q S

    q [rows, H, dk], k [rows, Hk, dk], v [rows, Hk, dv] as there.
    state: fp32 [pool, H, dk, dv], each [H, dk, dv] contiguous (the slots may
    lie further apart, as in a pool of all layers' states).
    slots: int32 or int64 [rows], row i's place in the pool (None: its own
    number; the pool then has one place for each row).  They are in device
    memory and not checked there: a slot outside the pool (-1, say, for rows
    that pad a batch) gives a row of zeros and touches no state, and rows of
    the same slot are taken as consecutive tokens of one sequence.

    Returns out [rows, H, dv]."""
    scale = None if scale is None else float(scale)
    try:
        key = (decay_attention_step, _looks(q), _looks(k), _looks(v), _looks(log_decay),
               _looks(state), _looks(slots), _looks(out), scale, torch.is_grad_enabled())
        plan = _PLANS.get(key)
    except (AttributeError, TypeError):      # not tensors: the checks say which
        key = plan = None
    if plan is None:
        plan = _step_plan(q, k, v, log_decay, state, slots, scale, out)
        if key is not None:
            _keep(key, plan)
    dev, shape, spans, tail = plan
    first = state.data_ptr()
    last = first + spans[0]
    for t, n in zip((q, k, v, log_decay, slots), spans[1:]):
        if n and t.data_ptr() < last and first < t.data_ptr() + n:
            raise ValueError("state overlaps the memory of an input")
    written = (state,) if out is None else (state, out)
    if out is None:
        out = torch.empty(shape, dtype=q.dtype, device=dev)
    else:
        _require_apart(out, "out", (q, k, v, log_decay, slots, state))
    _require_gpu(q, "q")
    if shape[0] == 0:
        return out
    ev = _t0()
    args = _hip.DECAY_STEP_ARGS[0].pack(_at(q), _at(k), _at(v), _at(log_decay), _at(state), _at(out),
                                        _at(slots), _hip.stream(dev)) + tail
    _call(_hip.lib().cf_decay_attention_step, "cf_decay_attention_step", dev, args)
    _changed(written)
    if ev is not None:
        (rows, H, dk), Hk, dv = q.shape, k.shape[1], v.shape[2]
        _t1("decay_attention_step", ev, flops=4 * rows * H * dk * dv,
            nbytes=8 * rows * H * dk * dv + q.element_size() * rows * (H + Hk) * (dk + dv))
    return out


def _step_plan(q, k, v, log_decay, state, slots, scale, out):
    """(device, output shape, bytes that state and the inputs lie over, packed
    arguments) of a checked call."""
    dev = _require_attention(q, k, v, log_decay, (3,))
    rows, H, dk = q.shape
    dv = v.shape[-1]
    _require(state, "state", (torch.float32,), dev)
    if state.ndim != 4 or state.shape[1:] != (H, dk, dv) or \
            (state.numel() and not state[0].is_contiguous()):
        raise ValueError(f"state must be [pool, {H}, {dk}, {dv}], each slot contiguous")
    if state.shape[0] > 1 and state.stride(0) < H * dk * dv:
        raise ValueError("slots of state overlap each other")
    if slots is not None:
        _require_index(slots, "slots", rows, dev)
    elif state.shape[0] != rows:
        raise ValueError(f"{rows} rows but {state.shape[0]} states: slots are needed")
    if rows > MAX_SEQUENCES:
        raise ValueError(f"{rows} rows (at most {MAX_SEQUENCES})")
    shape = (rows, H, dv)
    _require_output(out, "out", shape, q)
    o = (H * dv, dv) if out is None else (out.stride(0), out.stride(1))
    spans = []
    for t in (state, q, k, v, log_decay, slots):
        a, b = (0, 0) if t is None else _span(t)
        spans.append(b - a)
    tail = _hip.DECAY_STEP_ARGS[1].pack(
        slots is not None and slots.dtype == torch.int64, _DTYPES[q.dtype], rows, H, k.shape[1],
        dk, dv, state.shape[0], state.stride(0), q.stride(0), q.stride(1), k.stride(0),
        k.stride(1), v.stride(0), v.stride(1), *o, float(dk ** -0.5 if scale is None else scale))
    return dev, shape, tuple(spans), tail


# ---------------------------------------------------------------------------
# norms and rotation of heads
# ---------------------------------------------------------------------------

def rotary_freqs(pairs: int, base: float = 10000.0, sections: Optional[Sequence[int]] = None,
                 device=None) -> torch.Tensor:
    """fp64 [pairs]: the angle that a pair of channels turns by for each
    position, base ** (-i / pairs).  With sections (pairs of each axis) the
    axes have frequencies of their own, each from 1 down."""
    parts = [pairs] if sections is None else [int(n) for n in sections]
    if sum(parts) != pairs or any(n < 0 for n in parts):
        raise ValueError(f"sections {tuple(parts)} do not make {pairs} pairs")
    return torch.cat([float(base) ** (-torch.arange(n, dtype=torch.float64) / max(n, 1))
                      for n in parts]).to(device)


def _split_tokens(shape, tensors):
    """(outer, inner) counts of the token dimensions and each tensor's strides
    for them: the first split of the dimensions at which every tensor steps
    evenly through both parts."""
    def step(sizes, strides):
        """Stride of dimensions taken as one, None if they have none."""
        got, need = 0, None
        for n, s in reversed(list(zip(sizes, strides))):
            if n == 1:
                continue
            if need is None:
                got = s
            elif s != need:
                return None
            need = s * n
        return got

    n = len(shape)
    for cut in range(n + 1):
        found = [(step(shape[:cut], t[:cut]), step(shape[cut:], t[cut:])) for t in tensors]
        if all(a is not None and b is not None for a, b in found):
            outer = 1
            for s in shape[:cut]:
                outer *= s
            inner = 1
            for s in shape[cut:]:
                inner *= s
            return outer, inner, found
    raise ValueError("the token dimensions do not reduce to two strides: make the inputs "
                     "contiguous")


def _weight(w, name, x):
    """(fp32?, stride between heads) of the norm weights of x's heads."""
    if w is None:
        return 1, 0
    _require(w, name, (torch.float32, x.dtype), x.device)
    H, d = x.shape[-2:]
    if w.shape not in ((d,), (H, d)) or not w.is_contiguous():
        raise ValueError(f"{name} must be contiguous [{d}] or [{H}, {d}]")
    return w.dtype == torch.float32, d if w.ndim == 2 else 0


def _rotate(x, k, positions, freqs, sections, interleaved, inverse, norm, eps, weights, outs,
            names):
    sections = None if sections is None else tuple(int(n) for n in sections)
    interleaved, inverse = bool(interleaved), bool(inverse)
    try:
        key = (_rotate, _looks(x), _looks(k), _looks(positions), _looks(freqs), sections,
               interleaved, inverse, norm, eps, _looks(weights[0]), _looks(weights[1]),
               _looks(outs[0]), _looks(outs[1]), torch.is_grad_enabled())
        plan = _PLANS.get(key)
    except (AttributeError, TypeError):      # not tensors: the checks say which
        key = plan = None
    if plan is None:
        plan = _rotary_plan(x, k, positions, freqs, sections, interleaved, inverse, norm, eps,
                            weights, outs, names)
        if key is not None:
            _keep(key, plan)
    dev, tail = plan
    ys = []
    for i, (t, out) in enumerate(zip((x, k), outs)):
        if t is None:
            ys.append(None)
        elif out is None:
            ys.append(torch.empty(t.shape, dtype=t.dtype, device=dev))
        else:
            in_place = out.data_ptr() == t.data_ptr() and out.stride() == t.stride()
            others = (positions, freqs, k if i == 0 else x) + weights
            _require_apart(out, "out", others if in_place else others + (t,))
            ys.append(out)
    if outs[0] is not None and outs[1] is not None:
        _require_apart(ys[0], "out", (ys[1],))
    _require_gpu(x, names[0])
    if x.numel() == 0:
        return ys
    ev = _t0()
    args = _hip.ROTARY_ARGS[0].pack(_at(x), _at(ys[0]), _at(weights[0]), _at(k), _at(ys[1]),
                                    _at(weights[1]), _at(positions), _at(freqs),
                                    _hip.stream(dev)) + tail
    _call(_hip.lib().cf_rotary, "cf_rotary", dev, args)
    for out in outs:
        if out is not None:
            _changed(out)
    if ev is not None:
        m = x.numel() + (0 if k is None else k.numel())
        _t1("qk_norm_rotary" if norm else "rotary", ev, nbytes=2 * m * x.element_size())
    return ys


def _rotary_plan(x, k, positions, freqs, sections, interleaved, inverse, norm, eps, weights, outs,
                 names):
    """(device, packed arguments) of a checked call."""
    _require(x, names[0], _DTYPES)
    dev = x.device
    xs = (x,) if k is None else (x, k)
    if k is not None:
        _require(k, names[1], (x.dtype,), dev)
    for t, name in zip(xs, names):
        if t.ndim < 3:
            raise ValueError(f"{name} must be [tokens.., heads, d]")
        if t.shape[:-2] != x.shape[:-2] or t.shape[-1] != x.shape[-1]:
            raise ValueError(f"{names[0]} {tuple(x.shape)} and {name} {tuple(t.shape)} do not "
                             "belong together")
        if not 1 <= t.shape[-2] <= MAX_HEADS:
            raise ValueError(f"{t.shape[-2]} heads in {name} (1 to {MAX_HEADS})")
        _require_rows(t, name)
    d, lead = x.shape[-1], tuple(x.shape[:-2])
    _require(freqs, "freqs", (torch.float64,), dev)
    if freqs.ndim != 1 or not freqs.is_contiguous():
        raise ValueError("freqs must be a contiguous tensor of one frequency a pair")
    pairs = freqs.shape[0]
    if not 1 <= d <= MAX_ROTARY_DIM or not 1 <= pairs or 2 * pairs > d:
        raise ValueError(f"{pairs} pairs in heads of {d} channels (at most {MAX_ROTARY_DIM})")
    parts = (pairs,) if sections is None else sections
    axes = len(parts)
    if not 1 <= axes <= MAX_AXES or sum(parts) != pairs or min(parts) < 0:
        raise ValueError(f"sections {parts} do not make {pairs} pairs of up to {MAX_AXES} axes")
    _require(positions, "positions", _POSITIONS, dev)
    if positions.ndim == len(lead):        # one position for all axes
        positions = positions.unsqueeze(0)
    if positions.ndim != len(lead) + 1:
        raise ValueError(f"positions must be {lead} or {(axes,) + lead}")
    try:
        positions = positions.expand((axes,) + lead)
    except RuntimeError:
        raise ValueError(f"positions {tuple(positions.shape)} do not fit {(axes,) + lead}") from None
    if not (eps >= 0):
        raise ValueError(f"eps {eps} is negative")
    ws = [_weight(w, n + "_weight", t) for t, w, n in zip(xs, weights, names)]
    for t, out in zip(xs, outs):
        _require_output(out, "out", t.shape, t)

    def contiguous(t):                       # strides of a new output
        got, n = [], 1
        for m in reversed(t.shape):
            got.insert(0, n)
            n *= m
        return tuple(got)
    out_strides = [contiguous(t) if out is None else out.stride() for t, out in zip(xs, outs)]
    strides = [t.stride()[:-2] for t in xs] + [st[:-2] for st in out_strides] + \
        [positions.stride()[1:]]
    outer, inner, at = _split_tokens(lead, strides)
    n = len(xs)
    second = (0, 0, 0, 0, 0, 0) if k is None else \
        at[1] + (k.stride(-2),) + at[3] + (out_strides[1][-2],)
    wk = (1, 0) if k is None else ws[1]
    tail = _hip.ROTARY_ARGS[1].pack(
        *ws[0], *wk, _POSITIONS[positions.dtype], _DTYPES[x.dtype], outer, inner, x.shape[-2],
        0 if k is None else k.shape[-2], d, pairs, axes, parts[0] if axes > 1 else 0,
        parts[0] + parts[1] if axes > 2 else 0, interleaved, norm, inverse,
        positions.stride(0), *at[2 * n], *at[0], x.stride(-2), *at[n], out_strides[0][-2], *second,
        float(eps))
    return dev, tail


def rotary(x: torch.Tensor, positions: torch.Tensor, freqs: torch.Tensor, *,
           sections: Optional[Sequence[int]] = None, interleaved: bool = False,
           inverse: bool = False, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Turns pairs of channels of every head by position * frequency.

    x [tokens.., H, d] (one or more token dimensions; fp32, fp16 or bf16; d <=
    512).  freqs: fp64 [pairs], radians a position (`rotary_freqs`); the first
    2 * pairs channels are turned, channel i with channel i + pairs, or
    2 i with 2 i + 1 where interleaved; the others are passed on.
    positions: int32, int64 or fp32, [tokens..], or [axes, tokens..] with
    sections, the number of pairs that go by each axis (time, height, width:
    up to three, in the order of the pairs).  Positions may be broadcast.
    Angles are taken in 64 bits, so far positions keep their precision.
    inverse turns back.  out: a tensor for the output, x itself to turn in
    place."""
    return _rotate(x, None, positions, freqs, sections, interleaved, inverse, False, 0.0,
                   (None, None), (out, None), ("x",))[0]


def qk_norm_rotary(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor,
                   freqs: torch.Tensor, *, q_weight: Optional[torch.Tensor] = None,
                   k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
                   sections: Optional[Sequence[int]] = None, interleaved: bool = False,
                   out=None):
    """Norm of every query and key head, then `rotary`, in one pass:

        y = x / sqrt(mean(x^2) + eps) * weight

    over the d channels of a head.  q [tokens.., H, d], k [tokens.., Hk, d] of
    one type; weights [d], shared by the heads, or [H, d] (fp32 or of q's
    type; None: ones).  out: a pair of tensors, each of which may be its own
    input.  Statistics and rotation are fp32, each value is rounded once.
    Returns (q, k)."""
    if k is None:
        raise TypeError("k must be a torch.Tensor")
    outs = (None, None) if out is None else tuple(out)
    if len(outs) != 2:
        raise ValueError("out must be a pair of tensors")
    return tuple(_rotate(q, k, positions, freqs, sections, interleaved, False, True, float(eps),
                         (q_weight, k_weight), outs, ("q", "k")))


__all__ = ["decay_attention", "decay_attention_step", "rotary_freqs", "rotary",
           "qk_norm_rotary"]
