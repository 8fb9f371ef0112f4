"""Edges of the sequence operators: precision where terms cancel.

Tolerances as in test_gpu_sequence: an output's own rounding plus 72 * 2^-24
(a sum's depth and the roundings of its terms) of the definition evaluated
with absolute values, for outputs of 16 bits too; where a test needs another
one it stands there with its reason.
"""
import pytest
import torch

from catfuse_amd import kernels
from test_gpu_sequence import BF16, F16, F32, U32, _close, _definition

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------
# precision where terms cancel
# ---------------------------------------------------------------------------

def _check(cuda, q, k, v, state, dtype, scale=1.0):
    """Without a decay, against the definition; factors of 16-bit outputs too
    in 24 bits."""
    f = torch.zeros(1)
    out, left = kernels.decay_attention(
        q.to(dtype).to(cuda), k.to(dtype).to(cuda), v.to(dtype).to(cuda), f.to(cuda), scale=scale,
        state=None if state is None else state.to(cuda))
    a = [x[0].to(dtype).double() for x in (q, k, v)]
    s0 = None if state is None else state[0].double()
    want, s = _definition(*a, f.double(), scale, s0)
    big, sbig = _definition(*(x.abs() for x in a), f.double(), scale, s0)
    _close(out[0], want, big, dtype, 72 * U32)
    _close(left[0], s, sbig, F32, 72 * U32)
    return out, left


# Two numbers of 24 bits whose difference is 2^-22, on either side of the
# middle between two numbers of 16 bits: rounded to those they differ by 2^-15.
LOW, HIGH = 1 + 2.0 ** -8 + 2.0 ** -16 - 2.0 ** -23, 1 + 2.0 ** -8 + 2.0 ** -16 + 2.0 ** -23


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("dk", [32, 64, 128, 256])
def test_attention_reads_states_in_full(cuda, dtype, dk):
    """out = scale q S of channels that cancel: S keeps its 24 bits on the way
    to the output.  Every product is exact; rounded to 16 bits the states would
    be off by 2^-15 dk / 2, three times the tolerance."""
    N, dv = 70, 40
    q = torch.ones(1, N, 1, dk)
    q[..., 1::2] = -1
    state = torch.full((1, 1, dk, dv), LOW)
    state[:, :, 1::2] = HIGH
    zero = torch.zeros(1, N, 1, dk), torch.zeros(1, N, 1, dv)
    out, left = _check(cuda, q, *zero, state, dtype)
    assert torch.equal(left.cpu(), state)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("dk", [32, 64, 128, 256])
def test_attention_keeps_scores_in_full(cuda, dtype, dk):
    """Scores LOW and HIGH by turns on values 1 and -1."""
    N, dv = 128, 32
    q, k = torch.zeros(1, N, 1, dk), torch.zeros(1, N, 1, dk)
    q[..., :4] = torch.tensor([1.0, 2.0 ** -8, 2.0 ** -16, 2.0 ** -23]) * 2.0 ** 10
    k[..., :4] = 1
    k[:, ::2, :, 3] = -1
    v = torch.ones(1, N, 1, dv)
    v[:, 1::2] = -1
    _check(cuda, q, k, v, None, dtype, 2.0 ** -10)


def test_attention_keeps_products_of_second_parts(cuda):
    """fp16 heads: a state and keys with and without bits past the eighth,
    queries with three of them, terms that cancel but for the products of
    those."""
    x = 1 + 7 / 1024
    q = torch.full((1, 70, 1, 128), x)
    q[..., 1::2] = -x
    state = torch.ones(1, 1, 128, 32)
    state[:, :, ::2] = 1 + 2.0 ** -8
    zero = torch.zeros(1, 70, 1, 128), torch.zeros(1, 70, 1, 32)
    _check(cuda, q, *zero, state, F16)
    q = torch.zeros(1, 64, 1, 32)
    k = torch.zeros(1, 64, 1, 32)
    q[..., 0], q[..., 1] = x, 1.0
    k[:, ::2, :, 0] = x                       # scores x^2
    k[:, 1::2, :, 0] = 1
    k[:, 1::2, :, 1] = (torch.tensor(7 / 1024 * x).half()).float()    # and what fp16 has next to it
    v = torch.ones(1, 64, 1, 32)
    v[:, 1::2] = -1
    _check(cuda, q, k, v, None, F16)
