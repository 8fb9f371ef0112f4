"""Dense products with their epilogue: the projections of layers of real values.

The spiking layers' Linear -> BN -> LIF takes spikes (`kernels.linear_lif`,
`transformer.FusedLinearBNLIF`); these take real values, as the layers around
`delta_attention` and `decay_attention` have them: a product with its bias,
activation and residual (`linear`), and the two products of a gated feed-forward
block (`gated_linear`), each in one kernel that reads x once and writes only the
result.

Inference only, on the current stream of the inputs' device, without waiting for
the GPU or reading values back, like the sequence operators.  No counterpart in
the reference.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch.autograd.graph import increment_version as _changed

from catfuse_amd import _hip
from catfuse_amd.runtime import _t0, _t1
from catfuse_amd.sequence import (_DTYPES, _at, _call, _keep, _looks, _planned, _require,
                                  _require_apart, _require_gpu, _require_output, _require_rows)

ACTIVATIONS = {None: 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}   # CF_ACT_*
MAX_ROWS = 1000000000       # CF_LINEAR_MAX_ROWS
MAX_WIDTH = 16000000        # CF_LINEAR_MAX_WIDTH


def _row_stride(t, name: str) -> int:
    """The stride between rows, all dimensions but the last taken as one."""
    got, need = t.shape[-1], None
    for n, s in reversed(list(zip(t.shape[:-1], t.stride()[:-1]))):
        if n == 1:
            continue
        if need is None:
            got = s
        elif s != need:
            raise ValueError(f"the rows of {name} are not evenly apart: make it contiguous")
        need = s * n
    return got


def _apart(out, inputs) -> None:
    """As rows of one head, so that columns beside each other in the same rows
    count as apart."""
    _require_apart(out.unsqueeze(-2), "out",
                   [t.unsqueeze(-2) if t is not None and t.ndim > 1 else t for t in inputs])


def _plan(x, ws, biases, activation, residual, out):
    """(device, output shape, workspace bytes, packed arguments) of a checked call."""
    _require(x, "x", _DTYPES)
    dev = x.device
    if x.ndim < 1:
        raise ValueError("x must be [.., inner]")
    K = x.shape[-1]
    names = ("w",) if len(ws) == 1 else ("w_gate", "w_up")
    N = None
    for w, name in zip(ws, names):
        _require(w, name, (x.dtype,), dev)
        if w.ndim != 2 or w.shape[1] != K or (N is not None and w.shape[0] != N):
            raise ValueError(f"{name} {tuple(w.shape)} does not belong to x {tuple(x.shape)}" +
                             ("" if N is None else f" and w_gate {tuple(ws[0].shape)}"))
        N = w.shape[0]
    if not 1 <= N <= MAX_WIDTH or K > MAX_WIDTH:
        raise ValueError(f"widths {K} and {N}: at most {MAX_WIDTH}, outputs at least 1")
    kinds = set()
    for b, name in zip(biases, ("bias",) if len(ws) == 1 else ("bias_gate", "bias_up")):
        if b is not None:
            _require(b, name, (torch.float32, x.dtype), dev)
            if b.shape != (N,) or not b.is_contiguous():
                raise ValueError(f"{name} must be a contiguous tensor of {N} values")
            kinds.add(b.dtype)
    if len(kinds) > 1:
        raise TypeError("bias_gate and bias_up must be of one type")
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation {activation!r}: one of "
                         f"{', '.join(repr(n) for n in ACTIVATIONS)}")
    rows = 1
    for n in x.shape[:-1]:
        rows *= n
    if rows > MAX_ROWS:
        raise ValueError(f"{rows} rows (at most {MAX_ROWS})")
    shape = tuple(x.shape[:-1]) + (N,)
    if residual is not None:
        _require(residual, "residual", (x.dtype,), dev)
        if tuple(residual.shape) != shape:
            raise ValueError(f"residual has shape {tuple(residual.shape)}, expected {shape}")
        _require_rows(residual, "residual")
    for t, name in ((x, "x"),) + tuple(zip(ws, names)):
        _require_rows(t, name)
    _require_output(out, "out", shape, x)
    empty = rows == 0
    strides = [0 if t is None or empty else _row_stride(t, name) for t, name in
               ((x, "x"), (ws[0], names[0]), (ws[1] if len(ws) > 1 else None, names[-1]),
                (residual, "residual"))]
    o = N if out is None or empty else _row_stride(out, "out")

    def tail(ws_bytes):
        return _hip.LINEAR_ARGS[1].pack(_DTYPES[x.dtype], torch.float32 in kinds,
                                        ACTIVATIONS[activation], rows, K, N, *strides, o, ws_bytes)
    # (the workspace's size goes by w2 being there, not by its address)
    pointers = _hip.LINEAR_ARGS[0].pack(0, 0, len(ws) - 1, 0, 0, 0, 0, 0, 0)
    ws_bytes = _hip.lib().cf_linear_workspace(pointers + tail(0))
    return dev, shape, ws_bytes, tail(ws_bytes)


def _product(what, x, w, w2, bias, bias2, activation, residual, out):
    try:
        key = (what, activation, torch.is_grad_enabled(), _looks(x), _looks(w), _looks(w2),
               _looks(bias), _looks(bias2), _looks(residual), _looks(out))
        plan = _planned(key)
    except (AttributeError, TypeError):      # not tensors: the checks say which
        key = plan = None
    if plan is None:
        if what == "linear":
            plan = _plan(x, (w,), (bias,), activation, residual, out)
        else:
            plan = _plan(x, (w, w2), (bias, bias2), activation, residual, out)
        if key is not None:
            _keep(key, plan)
    dev, shape, ws_bytes, tail = plan
    given = out is not None
    if given:
        in_place = residual is not None and out.data_ptr() == residual.data_ptr() and \
            out.stride() == residual.stride()
        _apart(out, (x, w, w2, bias, bias2) + (() if in_place else (residual,)))
    else:
        out = torch.empty(shape, dtype=x.dtype, device=dev)
    _require_gpu(x, "x")
    if out.numel() == 0:
        return out
    work = torch.empty(ws_bytes, dtype=torch.uint8, device=dev) if ws_bytes else None
    ev = _t0()
    # (a second w of no elements has no address, and is there all the same: any one does)
    second = 0 if w2 is None else _at(w2) or _at(out)
    args = _hip.LINEAR_ARGS[0].pack(_at(x), _at(w), second, _at(bias), _at(bias2), _at(residual),
                                    _at(out), _at(work), _hip.stream(dev)) + tail
    _call(_hip.lib().cf_linear, "cf_linear", dev, args)
    if given:
        _changed(out)
    if ev is not None:
        rows, K, N = out.numel() // shape[-1], x.shape[-1], shape[-1]
        n = 1 if w2 is None else 2
        _t1(what, ev, flops=2 * n * rows * K * N,
            nbytes=x.element_size() * (rows * K + n * N * K + rows * N *
                                       (1 + (residual is not None))))
    return out


def linear(x: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
           activation: Optional[str] = None, residual: Optional[torch.Tensor] = None,
           out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """act(x w^T + bias) + residual, [.., cols].

    x [.., inner], w [cols, inner], residual [.., cols]: fp32, fp16 or bf16, all
    of one type; the last dimension contiguous, rows evenly apart (any distance,
    0 too).  bias [cols], fp32 or of x's type.
    activation: None, "relu", "silu" (z / (1 + e^-z)), "gelu" (by the error
    function: to 2^-20 of its value, for outputs of 16 bits to 2.6e-7 of |z|) or
    "gelu_tanh" (its approximation by tanh).
    out: a tensor for the output, apart from the inputs; it may be the residual
    itself, which is then added to in place.

    Sums and the epilogue are fp32, each output is rounded once.  Products of a
    small result and a long inner dimension are split along it, with a workspace
    of the splits' sums (fp32) from torch's allocator; large products of 16-bit
    rows that are not whole pieces of 16 bytes (an inner dimension or a stride that
    8 does not divide) take one of as many bytes as those rows have, laid out so."""
    return _product("linear", x, w, None, bias, None, activation, residual, out)


def gated_linear(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, *,
                 bias_gate: Optional[torch.Tensor] = None, bias_up: Optional[torch.Tensor] = None,
                 activation: Optional[str] = "silu",
                 out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """act(x w_gate^T + bias_gate) * (x w_up^T + bias_up), [.., cols]: the first
    half of a gated feed-forward block in one pass over x (`linear` with the
    residual is the other half).  Arguments as of `linear`; both biases of one
    type."""
    return _product("gated_linear", x, w_gate, w_up, bias_gate, bias_up, activation, None, out)


__all__ = ["linear", "gated_linear"]
