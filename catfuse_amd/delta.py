"""The delta rule's attention: states that fade and correct themselves.

The relatives of `decay_attention` and `decay_attention_step`
(`catfuse_amd.sequence`) whose tokens first take out of the state what it
already answers to their key, with a strength and a decay of each token's own:
whole prompts (`delta_attention`) and one token at a time
(`delta_attention_step`), against the same states and pools of states.

Inference only, on the current stream of the inputs' device, without waiting for
the GPU or reading values back, like the operators there.  No counterpart in the
reference.
"""
from __future__ import annotations

import math
from typing import Optional

import torch
from torch.autograd.graph import increment_version as _changed

from catfuse_amd import _hip
from catfuse_amd.runtime import _t0, _t1
from catfuse_amd.sequence import (_DTYPES, _at, _call, _keep, _looks, _planned, _require,
                                  _require_apart, _require_gpu, _require_index, _require_output,
                                  _require_rows, _span, CHUNK, MAX_HEADS, MAX_KEY_DIM, MAX_SEQUENCES,
                                  MAX_TOKEN_STRIDE, MAX_TOKENS, MAX_VALUE_DIM)

MAX_SEGMENTS = 65535        # of a call (the grid of the launch that joins them)


def _require_delta(q, k, v, beta, log_decay, ndims):
    """Checks of what both forms share; (device, heads)."""
    _require(q, "q", _DTYPES)
    dev = q.device
    _require(k, "k", (q.dtype,), dev)
    _require(v, "v", (q.dtype,), dev)
    _require(beta, "beta", (torch.float32, q.dtype), dev)
    if log_decay is not None:
        _require(log_decay, "log_decay", (torch.float32, q.dtype), dev)
    if q.ndim not in ndims or k.ndim != q.ndim or v.ndim != q.ndim:
        raise ValueError(f"q, k and v must have {' or '.join(str(n) for n in ndims)} dimensions, "
                         f"got {q.ndim}, {k.ndim} and {v.ndim}")
    dk, dv, lead = q.shape[-1], v.shape[-1], q.shape[:-2]
    if k.shape[:-2] != lead or v.shape[:-2] != lead or k.shape[-1] != dk:
        raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not "
                         "belong together")
    if beta.ndim != q.ndim - 1 or beta.shape[:-1] != lead:
        raise ValueError(f"beta must be {tuple(lead) + ('heads',)}, got {tuple(beta.shape)}")
    if log_decay is not None and log_decay.shape != beta.shape:
        raise ValueError(f"log_decay must have beta's shape {tuple(beta.shape)}, got "
                         f"{tuple(log_decay.shape)}")
    H = beta.shape[-1]
    if not 1 <= H <= MAX_HEADS or any(t.shape[-2] < 1 or H % t.shape[-2] for t in (q, k, v)):
        raise ValueError(f"{q.shape[-2]}, {k.shape[-2]} and {v.shape[-2]} heads of q, k and v: each "
                         f"has to divide the {H} of beta (at most {MAX_HEADS})")
    if not 1 <= dk <= MAX_KEY_DIM or not 1 <= dv <= MAX_VALUE_DIM:
        raise ValueError(f"head sizes {dk} and {dv}: at most {MAX_KEY_DIM} and {MAX_VALUE_DIM}")
    for t, name in ((q, "q"), (k, "k"), (v, "v")):
        _require_rows(t, name)
    return dev, H


def _kinds(q, beta, log_decay):
    """Whether beta and log_decay are fp32."""
    return beta.dtype == torch.float32, log_decay is not None and log_decay.dtype == torch.float32


def _segment(seqs: int, tokens: int, packed: bool, heads: int, dk: int, dv: int) -> int:
    """Tokens a segment; 0: whole sequences."""
    # The walks along a segment get shorter with it, the walk over the segments'
    # states longer: least near a constant times the root of the length, 3.5 for wide
    # keys and 3 for narrow ones (us; one sequence of 1024 tokens and 8 heads of 128
    # channels: 64 tokens a segment 76, 128 65, 192 69, whole 138; 4096 tokens: 192 128,
    # 320 120, 448 136, whole 529; 16384 of 64 channels: 192 179, 448 167, 704 181).
    # No shorter than it takes to have all segments at work at once (16384 tokens, 32
    # heads: 576 750, 2048 698), by half as many for equal sequences of 65 to 128
    # channels (two of 8192 tokens and 16 heads: 576 393, 1088 373; four of 4096: 367 and
    # 372; but packed 20000, 10000 and 30000, which end some early: 3776 2197, 8192
    # 2434).  An odd number of chunks: with an even one all segments may read the same
    # channels of memory at a time (4096 tokens, 16 heads: 256 168, 320 140; 8192: 512
    # 244, 576 220; 5000 of 4 heads of 256 channels: 256 311, 320 265; where they do not,
    # the even number is better by 2 to 10 %: 5000 of 8 heads of 32: 71 and 76), which
    # counts once they are many and as long as they drift little.  Whole sequences if
    # they give workgroups enough (eight of 4096, 32 heads: whole 784, 2112 979; four of
    # 2048: 329 and 341) or are short (160 tokens, 8 heads: whole 36, 64 37; 196 43 and
    # 39; 300 51 and 43; of 256 channels 76 and 87).  Packed ones, whose lengths are not
    # known here, then are cut where they are longer than most: a little over the mean
    # (16 heads of 128: sixteen of 50 to 3000 tokens whole 419, cut 273; 24 of 20 to 2000
    # whole 405 to 553, cut 457 to 478; sixteen of 1000 whole 203, cut 219), until they
    # fill the card by themselves.
    width = 32 if dk <= 32 else 64 if dk <= 64 else 128
    columns = heads * -(-dv // width)          # workgroups of one segment
    at_once = 2048 if dk <= 32 else 1024 if dk <= 64 else 512 if dk <= 128 else 256
    total = tokens if packed else seqs * tokens
    short = (3 if dk <= 128 else 8) * CHUNK
    if total <= short * seqs or seqs * columns * (1 if packed else 4) > at_once:
        return 0
    if not packed and 64 < dk <= 128:
        at_once //= 2
    chunks = math.ceil(math.sqrt(tokens) * (3.0 if dk <= 64 else 3.5) / CHUNK)
    chunks = max(chunks, -(-total * columns // (at_once * CHUNK)))
    if packed and seqs * columns * 4 > at_once:    # what is longer than most
        chunks = max(chunks, -(-total * 21 // (seqs * CHUNK * 20)))
    if chunks < 32 and (chunks > 2 or total * columns >= chunks * at_once * CHUNK):
        chunks |= 1
    segment = chunks * CHUNK
    segments = tokens // segment + seqs if packed else seqs * -(-tokens // segment)
    return segment if segment < tokens and segments <= MAX_SEGMENTS else 0


def delta_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, beta: torch.Tensor,
                    log_decay: Optional[torch.Tensor] = None, *, scale: Optional[float] = None,
                    state: Optional[torch.Tensor] = None,
                    cu_seqlens: Optional[torch.Tensor] = None,
                    out: Optional[torch.Tensor] = None, return_state: bool = True):
    """Causal attention without a softmax by the delta rule: a token takes out
    of the state what it answers to the token's key, puts in the token's value
    instead, by as much as beta says, and the past fades by exp(log_decay):

        S_t = w_t S_{t-1} + k_t u_t^T,    u_t = beta_t (v_t - w_t S_{t-1}^T k_t)
        out_t = scale q_t S_t,            w_t = exp(log_decay_t)

    for each sequence and head, over whole prompts.

    q [B, N, Hq, dk], k [B, N, Hk, dk], v [B, N, Hv, dv]: B sequences of N
    tokens; or, with cu_seqlens, [tokens, Hq, dk] and so on: packed sequences,
    number b the rows cu_seqlens[b] .. cu_seqlens[b + 1] - 1.  fp32, fp16 or
    bf16, all of one type; the last dimension contiguous, other strides free
    (tokens of a sequence at most 8,000,000 elements apart).  dk <= 256,
    dv <= 1024.
    beta, log_decay [B, N, H] or [tokens, H], fp32 or of q's type, any strides:
    each head's own.  H is a multiple of Hq, Hk and Hv: head h reads head
    h // (H // Hq) of q, and so on.  log_decay None: nothing fades; -inf: only the
    token itself is kept; 0 or less as a rule (a sum over 64 tokens has to be the
    logarithm of a number of fp32).
    scale: dk ** -0.5 if None.
    state: fp32 [sequences, H, dk, dv], S before the first token (None: zeros).
    cu_seqlens: int32 or int64 [sequences + 1], in device memory and therefore
    not checked: offsets are clamped to 0 .. tokens, one below its predecessor
    counts as that.  Rows of no sequence are zero in a new output and stay as
    they are in one given as `out`.
    out: a tensor for the output, apart from the inputs.

    Returns (out [.., H, dv], state after the last token), or out alone without
    return_state.  Sums and states are fp32, products exact to 2^-24 of their
    factors for every type, powers of the decays to 2^-22 (from token to token within
    a chunk, to 2^-22 of one).  With keys of a length of at most 1 and beta in 0 .. 1
    (or keys of length 1 and beta in 0 .. 2) a step does not make errors grow; keys
    that are longer (|k|^2 beta > 2) let the state itself and its errors grow from
    token to token, and where |k|^2 beta itself is beyond fp32 the results may be NaN.
    Numbers of a state and u_t are computed so between 2^-100 and 2^100.  A token that
    holds an infinity or NaN, or whose u_t is beyond fp32, does not reach the tokens
    before it; what it does reach may be NaN where the formula gives an infinity.
    The workspace, from torch's allocator, is 300 bytes a token and head (bf16
    heads of 65 to 128 channels, whose sequences count as whole multiples of 64
    tokens; others 204 and 32), and for long sequences of a small batch, which are
    walked in segments side by side, [dk, dv + dk] fp32 a segment and head.  Many
    short sequences are computed in groups, so that the former is at most three
    times what the tokens themselves take, and 1 GiB."""
    scale = None if scale is None else float(scale)
    try:
        key = (delta_attention, _looks(q), _looks(k), _looks(v), _looks(beta), _looks(log_decay),
               _looks(state), _looks(cu_seqlens), _looks(out), scale, return_state,
               torch.is_grad_enabled())
        plan = _planned(key)
    except (AttributeError, TypeError):      # not tensors: the checks say which
        key = plan = None
    if plan is None:
        plan = _attention_plan(q, k, v, beta, log_decay, scale, state, cu_seqlens, out)
        if key is not None:
            _keep(key, plan)
    dev, shape, state_shape, ws_bytes, tail = plan
    given = out is not None
    if given:
        _require_apart(out, "out", (q, k, v, beta, log_decay, state, cu_seqlens))
    else:
        out = torch.empty(shape, dtype=q.dtype, device=dev)
    _require_gpu(q, "q")
    left = torch.empty(state_shape, dtype=torch.float32, device=dev) if return_state else None
    if state_shape[0] == 0:                  # no sequences: no row belongs to one
        if not given:
            out.zero_()
        return (out, left) if return_state else out
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev) if ws_bytes else None
    ev = _t0()
    args = _hip.DELTA_ATTENTION_ARGS[0].pack(
        _at(q), _at(k), _at(v), _at(beta), _at(log_decay), _at(state), _at(left), _at(out),
        _at(cu_seqlens), _at(ws), _hip.stream(dev)) + tail
    _call(_hip.lib().cf_delta_attention, "cf_delta_attention", dev, args)
    if given:
        _changed(out)
    if ev is not None:
        H, dk, dv = state_shape[1:]
        rows = out.numel() // (H * dv)
        _t1("delta_attention", ev, flops=6 * rows * H * dk * dv,
            nbytes=q.element_size() * (q.numel() + k.numel() + v.numel() + out.numel()) +
            4 * state_shape[0] * H * dk * dv * ((state is not None) + return_state))
    return (out, left) if return_state else out


def _attention_plan(q, k, v, beta, log_decay, scale, state, cu_seqlens, out):
    """(device, shapes of the output and of the states, workspace bytes, packed
    arguments) of a checked call."""
    dev, H = _require_delta(q, k, v, beta, log_decay, (4,) if cu_seqlens is None else (3,))
    dk, dv = q.shape[-1], v.shape[-1]
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
    shape = tuple(q.shape[:-2]) + (H, dv)
    _require_output(out, "out", shape, q)
    for t, name in ((q, "q"), (k, "k"), (v, "v"), (out, "out")):
        if t is not None and t.stride(-3) > MAX_TOKEN_STRIDE and t.shape[-3] > 1:
            raise ValueError(f"tokens of {name} lie {t.stride(-3)} elements apart (at most "
                             f"{MAX_TOKEN_STRIDE})")
    if N > MAX_TOKENS:
        raise ValueError(f"{N} tokens (at most {MAX_TOKENS})")

    def steps(t, i):
        # (a dimension of one element may have any stride: a plain one)
        return (t.stride(0) if not packed and B > 1 else 0,
                t.stride(i) if N > 1 else t.shape[-1],
                t.stride(i + 1) if t.shape[i + 1] > 1 else 0)
    # a new output is contiguous
    o = steps(out, -3) if out is not None else (0 if packed else N * H * dv, H * dv, dv)
    decay = (0, 0, 0) if log_decay is None else steps(log_decay, -2)
    kinds = _kinds(q, beta, log_decay)

    def tail(ws_bytes):
        return _hip.DELTA_ATTENTION_ARGS[1].pack(
            packed and cu_seqlens.dtype == torch.int64, out is None, _DTYPES[q.dtype], *kinds, B, N,
            H, q.shape[-2], k.shape[-2], v.shape[-2], dk, dv, *steps(q, -3), *steps(k, -3),
            *steps(v, -3), *steps(beta, -2), *decay, *o,
            _segment(B, N, packed, H, dk, dv), ws_bytes,
            float(dk ** -0.5 if scale is None else scale))
    # (the workspace's size goes by cu_seqlens being there, not by its address)
    pointers = _hip.DELTA_ATTENTION_ARGS[0].pack(*[int(packed) if i == 8 else 0 for i in range(11)])
    ws_bytes = _hip.lib().cf_delta_workspace(pointers + tail(0))
    return dev, shape, (B, H, dk, dv), ws_bytes, tail(ws_bytes)


def delta_attention_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, beta: torch.Tensor,
                         log_decay: Optional[torch.Tensor], state: torch.Tensor, *,
                         slots: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                         out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """`delta_attention` for one token of each running sequence, against a pool
    of states that is updated in place.

    q [rows, Hq, dk], k [rows, Hk, dk], v [rows, Hv, dv], beta and log_decay
    [rows, H] as there (log_decay None: nothing fades).
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
        key = (delta_attention_step, _looks(q), _looks(k), _looks(v), _looks(beta),
               _looks(log_decay), _looks(state), _looks(slots), _looks(out), scale,
               torch.is_grad_enabled())
        plan = _planned(key)
    except (AttributeError, TypeError):      # not tensors: the checks say which
        key = plan = None
    if plan is None:
        plan = _step_plan(q, k, v, beta, log_decay, state, slots, scale, out)
        if key is not None:
            _keep(key, plan)
    dev, shape, spans, tail = plan
    first = state.data_ptr()
    last = first + spans[0]
    for t, n in zip((q, k, v, beta, log_decay, slots), spans[1:]):
        if n and t.data_ptr() < last and first < t.data_ptr() + n:
            raise ValueError("state overlaps the memory of an input")
    written = (state,) if out is None else (state, out)
    if out is None:
        out = torch.empty(shape, dtype=q.dtype, device=dev)
    else:
        _require_apart(out, "out", (q, k, v, beta, log_decay, slots, state))
    _require_gpu(q, "q")
    if shape[0] == 0:
        return out
    ev = _t0()
    args = _hip.DELTA_STEP_ARGS[0].pack(_at(q), _at(k), _at(v), _at(beta), _at(log_decay),
                                        _at(state), _at(out), _at(slots), _hip.stream(dev)) + tail
    _call(_hip.lib().cf_delta_attention_step, "cf_delta_attention_step", dev, args)
    _changed(written)
    if ev is not None:
        rows, H, dv = shape
        dk = q.shape[2]
        _t1("delta_attention_step", ev, flops=6 * rows * H * dk * dv,
            nbytes=8 * rows * H * dk * dv +
            q.element_size() * (q.numel() + k.numel() + v.numel() + out.numel()))
    return out


def _step_plan(q, k, v, beta, log_decay, state, slots, scale, out):
    """(device, output shape, bytes that state and the inputs lie over, packed
    arguments) of a checked call."""
    dev, H = _require_delta(q, k, v, beta, log_decay, (3,))
    rows, dk, dv = q.shape[0], q.shape[-1], v.shape[-1]
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
    for t in (state, q, k, v, beta, log_decay, slots):
        a, b = (0, 0) if t is None else _span(t)
        spans.append(b - a)
    decay = (0, 0) if log_decay is None else log_decay.stride()
    tail = _hip.DELTA_STEP_ARGS[1].pack(
        slots is not None and slots.dtype == torch.int64, _DTYPES[q.dtype],
        *_kinds(q, beta, log_decay), rows, H, q.shape[1], k.shape[1], v.shape[1], dk, dv,
        state.shape[0], state.stride(0), q.stride(0), q.stride(1), k.stride(0), k.stride(1),
        v.stride(0), v.stride(1), *beta.stride(), *decay, *o,
        float(dk ** -0.5 if scale is None else scale))
    return dev, shape, tuple(spans), tail


__all__ = ["delta_attention", "delta_attention_step"]
