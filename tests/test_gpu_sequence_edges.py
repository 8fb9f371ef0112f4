"""Edges of the sequence operators: precision where terms cancel, tensors that
other parts of the package or autograd keep track of, decays that grow, many
chunks and workgroups in a row.

Tolerances as in test_gpu_sequence: an output's own rounding plus 72 * 2^-24
(a sum's depth and the roundings of its terms) of the definition evaluated
with absolute values, for outputs of 16 bits too; where a test needs another
one it stands there with its reason.
"""
import math

import pytest
import torch

from catfuse_amd import kernels, sequence
from test_gpu_sequence import (BF16, F16, F32, U32, _check_attention, _close, _decays, _definition,
                               _inputs)

pytestmark = pytest.mark.gpu


@pytest.fixture
def segments(monkeypatch):
    """Makes the calls that follow split sequences into segments of so many
    tokens (0: whole sequences), whatever the rule on sizes says."""
    def force(tokens):
        def split(seqs, n, packed, heads, dk, dv):
            if tokens == 0 or tokens >= n:
                return 0, 0
            return tokens, n // tokens + seqs if packed else seqs * -(-n // tokens)
        monkeypatch.setattr(sequence, "_segment", split)
        monkeypatch.setattr(sequence, "_PLANS", {})
    return force


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


# ---------------------------------------------------------------------------
# tensors that others keep track of
# ---------------------------------------------------------------------------

def test_written_tensors_change_versions(cuda):
    """Outputs that are given and states in place count as changed, inputs and
    other outputs do not; tensors of inference mode have no count."""
    q, k, v = (torch.randn(3, n, 16, device=cuda) for n in (4, 2, 2))
    f, pos = _decays(4).to(cuda), torch.arange(3, device=cuda)
    freqs = kernels.rotary_freqs(8, device=cuda)
    pool, out = torch.zeros(3, 4, 16, 16, device=cuda), torch.empty(3, 4, 16, device=cuda)
    cu = torch.tensor([0, 3], dtype=torch.int32, device=cuda)

    def changed(call, written):
        every = [q, k, v, f, pos, freqs, pool, out, cu]
        before = [t._version for t in every]
        call()
        assert [t._version > n for t, n in zip(every, before)] == \
            [any(t is w for w in written) for t in every]
    for _ in range(2):                                   # planned anew, and again
        changed(lambda: kernels.decay_attention(q, k, v, f, cu_seqlens=cu), [])
        changed(lambda: kernels.decay_attention(q, k, v, f, cu_seqlens=cu, out=out), [out])
        changed(lambda: kernels.decay_attention(q, k, v, f, cu_seqlens=cu, out=out,
                                                return_state=False), [out])
        changed(lambda: kernels.decay_attention_step(q, k, v, f, pool), [pool])
        changed(lambda: kernels.decay_attention_step(q, k, v, f, pool[:], slots=pos, out=out),
                [pool, out])
        changed(lambda: kernels.rotary(q, pos, freqs), [])
        changed(lambda: kernels.rotary(q, pos, freqs, out=out), [out])
        changed(lambda: kernels.rotary(q[:, :2], pos, freqs, out=q[:, :2]), [q])
        changed(lambda: kernels.qk_norm_rotary(q, k, pos, freqs, out=(None, k)), [k])
        changed(lambda: kernels.qk_norm_rotary(q, k, pos, freqs, out=(q, k)), [q, k])
    with torch.inference_mode():
        x = torch.randn(3, 4, 16, device=cuda)
        want = kernels.rotary(x, pos, freqs)
        assert torch.equal(kernels.rotary(x, pos, freqs, out=x), want)


def test_saved_activation_turned_in_place(cuda):
    """A head that autograd has saved, turned in place through a detached view:
    the backward pass refuses it, as after any change in place."""
    x = torch.randn(5, 2, 8, device=cuda)
    w = torch.randn(8, device=cuda, requires_grad=True)
    y = (x * w).sum()                                    # saves x for w's gradient
    kernels.rotary(x.detach(), torch.arange(5, device=cuda), kernels.rotary_freqs(4, device=cuda),
                   out=x.detach())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_fused_output_turned_in_place(cuda):
    """The output of a fused token layer, turned in place through a view of its
    heads: the next fused layer reads the turned values, not the copy that the
    first one left for it.  A quarter turn: spikes stay numbers that the fused
    layers take exactly."""
    import catfuse_amd
    from catfuse_amd.transformer import FusedLinearBNLIF
    from test_gpu_transformer import _triple
    first, second = (FusedLinearBNLIF.from_sj_modules(*_triple(64, 64, s)).to(cuda) for s in (3, 4))
    x = (torch.rand(2, 2, 49, 64, generator=torch.Generator().manual_seed(5)) < 0.3).float().to(cuda)
    pos = torch.ones(1, 1, 49, dtype=torch.int64, device=cuda)
    freqs = torch.full((16,), math.pi / 2, dtype=torch.float64, device=cuda)
    with torch.no_grad():
        y = first(x)
        plain = second(y).clone()
        heads = y.unflatten(-1, (2, 32))
        turned = kernels.rotary(heads, pos, freqs).flatten(-2)
        assert torch.equal(turned.abs().unflatten(-1, (2, 32)), heads.roll(16, -1))
        kernels.rotary(heads, pos, freqs, out=heads)
        assert torch.equal(y, turned)
        second.reset()
        got = second(y).clone()
        second.reset()
        want = second(turned).clone()
    assert torch.equal(got, want) and not torch.equal(got, plain)
    catfuse_amd.check_status()


# ---------------------------------------------------------------------------
# decays that grow
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("dk", [16, 40])
@pytest.mark.parametrize("segment", [0, 64, 256, 448])
def test_attention_growth_past_a_segment(cuda, segments, dtype, dk, segment):
    """Decays above 0 whose powers leave the range of fp32 (and of fp64) within
    a segment, on heads that are silent at first: the definition's zeros and
    what grows out of the first token that is not silent (by up to exp(69): with
    a scale that brings it into the range of fp16 there)."""
    segments(segment)
    N, start, scale = 700, 650, 2.0 ** -100 if dtype == F16 else None
    q, k, v = _inputs((1, N, 3, dk), (1, N, 3, dk), 24, dtype, dk)
    k[:, :start] = 0
    f = torch.tensor([1.0, 0.35, 1.38])                 # exp(64 * 1.38) = 2e38
    _check_attention(cuda, q, k, v, f, scale, None, None, dtype)
    out, left = _check_attention(cuda, q, torch.zeros_like(k), v, f, scale, None, None,
                                 dtype)
    assert bool((out == 0).all()) and bool((left == 0).all())


@pytest.mark.parametrize("segment", [0, 64, 256])
def test_attention_growth_of_a_small_state(cuda, segments, segment):
    """A state of 1e-20 times a power past 3.4e38 is a number of fp32 again."""
    segments(segment)
    N, f = 300, torch.tensor([0.35])                    # exp(0.35 * 256) = 8e38
    q, k, v = _inputs((1, N, 1, 32), (1, N, 1, 32), 32, F32, 1)
    state = 1e-20 * torch.randn(1, 1, 32, 32, generator=torch.Generator().manual_seed(6))
    out, left = _check_attention(cuda, q, torch.zeros_like(k), v, f, None, state, None, F32)
    assert bool(left.isfinite().all()) and bool((left != 0).any())


def test_attention_growth_in_the_segments_of_a_long_batch(cuda):
    """The same at a size that the rule splits by itself."""
    N, H = 8192, 32
    tokens, _ = sequence._segment(1, N, False, H, 8, 8)
    assert tokens > 64
    f = torch.full((H,), 90.0 / tokens, device=cuda)    # its power: past 3.4e38
    q, k, v = (torch.randn(1, N, H, 8, device=cuda) for _ in range(3))
    out, left = kernels.decay_attention(q, torch.zeros_like(k), v, f)
    assert bool((out == 0).all()) and bool((left == 0).all())


# ---------------------------------------------------------------------------
# many chunks and segments in a row
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("dk,dv", [(32, 32), (64, 40), (128, 128), (160, 64)])
@pytest.mark.parametrize("segment", [0, 64, 512, 1024])
def test_attention_chunks_in_a_row(cuda, segments, dtype, dk, dv, segment):
    """Whole sequences of 33 (bf16) and 66 chunks, and segments of 1 to 32, over
    states, no decay, a slow one and a fast one.

    A sum of N terms without a decay: the matrix cores add 16 products to a
    state at a time, N / 16 times one after another, each time rounded (the sum
    of the 16 and the sum with the state: 2 u of what is there)."""
    segments(segment)
    N = 2100
    q, k, v = _inputs((1, N, 3, dk), (1, N, 1, dk), dv, dtype, dk + segment)
    f = torch.tensor([0.0, -2.0 ** -12, -2.0 ** -5])
    state = torch.randn(1, 3, dk, dv, generator=torch.Generator().manual_seed(2))
    out, left = kernels.decay_attention(q.to(cuda), k.to(cuda), v.to(cuda), f.to(cuda),
                                        state=state.to(cuda))
    a = [x[0].double() for x in (q, k, v)]
    want, s = _definition(*a, f.double(), dk ** -0.5, state[0].double())
    big, sbig = _definition(*(x.abs() for x in a), f.double(), dk ** -0.5, state[0].double().abs())
    depth = (N / 8 + 72) * U32
    _close(out[0], want, big, dtype, depth)
    _close(left[0], s, sbig, F32, depth)


@pytest.mark.parametrize("lens", [[1000, 0, 1, 640, 63, 1025], [700] * 4])
@pytest.mark.parametrize("segment", [0, 128, 512])
def test_attention_packed_in_segments(cuda, segments, lens, segment):
    """Full segments, ends of every length and sequences without any, in one
    launch."""
    segments(segment)
    N, dk = sum(lens), 64
    q, k, v = _inputs((N, 2, dk), (N, 1, dk), dk, BF16, segment)
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32)
    state = torch.randn(len(lens), 2, dk, dk, generator=torch.Generator().manual_seed(3))
    f = torch.tensor([-2.0 ** -9, -2.0 ** -3])
    out, left = kernels.decay_attention(q.to(cuda), k.to(cuda), v.to(cuda), f.to(cuda),
                                        state=state.to(cuda), cu_seqlens=cu.to(cuda))
    for b, (i, j) in enumerate(zip(cu.tolist(), cu.tolist()[1:])):
        a = [x[i:j].double() for x in (q, k, v)]
        want, s = _definition(*a, f.double(), dk ** -0.5, state[b].double())
        big, sbig = _definition(*(x.abs() for x in a), f.double(), dk ** -0.5,
                                state[b].double().abs())
        depth = (1025 / 8 + 72) * U32
        _close(out[i:j], want, big, BF16, depth)
        _close(left[b], s, sbig, F32, depth)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("segment", [0, 512])
def test_attention_decay_does_not_drift(cuda, segments, dtype, segment):
    """65536 tokens of nothing: the state fades by w^65536 and no rounding of
    w^64 or w^32 adds up over the chunks.

    M chunks each multiply a state by a power, rounded (u of it at most, of
    either sign): errors with a deviation of at most u / sqrt(3) that are
    unrelated between the 4096 elements of a head, so their mean has one of
    sqrt(M / 3 / 4096) u; six of those, and 2 u for the powers' product and the
    joins.  Powers that were all off the same way would be off by M times their
    error; here by a half u and by a twentieth of it."""
    segments(segment)
    N, H, d = 65536, 4, 64
    chunk = 64 if dtype == BF16 else 32
    n = (segment or N) // chunk
    near = -2.0 ** -14 * (1 + torch.arange(4096) / 8192)
    power = torch.exp(chunk * near.double())
    off = (power.float().double() - power) / power
    at = torch.stack([off.argmin(), off.argmax(), (off - U32 / 20).abs().argmin(),
                      (off + U32 / 20).abs().argmin()])
    f, off = near[at], off[at]
    tol = (6 * math.sqrt(N // chunk / 3 / d ** 2) + 2) * U32
    assert segment or bool((n * off.abs() > 10 * tol).all())
    q, k, v = (torch.zeros(1, N, H, d, dtype=dtype, device=cuda) for _ in range(3))
    state = 1 + torch.rand(1, H, d, d, generator=torch.Generator().manual_seed(9))
    out, left = kernels.decay_attention(q, k, v, f.to(cuda), state=state.to(cuda))
    want = state[0].double() * torch.exp(N * f.double())[:, None, None]
    rel = ((left[0].double().cpu() - want) / want).mean((-2, -1))
    assert bool((rel.abs() <= tol).all()), (rel / U32, tol / U32)


@pytest.mark.parametrize("B,H,wide", [(5000, 2, False), (3000, 4, True)])
def test_attention_many_whole_sequences(cuda, B, H, wide):
    """Whole packed sequences whose first rows are found over many offsets,
    some of them decreasing, negative and past the tokens."""
    N, d = 9000, 16
    assert sequence._segment(B, N, True, H, d, d) == (0, 0)
    g = torch.Generator().manual_seed(B)
    q, k, v = _inputs((N, H, d), (N, 1, d), d, F32, B)
    f = _decays(H)
    cu = torch.randint(0, N + 1, (B + 1,), generator=g).sort()[0]
    cu[B // 2], cu[B // 3], cu[70], cu[130] = -7, 5, 3, cu[125]
    cu[-4], cu[-2], cu[-1] = N + 100, 12, N - 3
    ends = cu.clamp(0, N).cummax(0)[0].tolist()
    out, left = kernels.decay_attention(
        q.to(cuda), k.to(cuda), v.to(cuda), f.to(cuda),
        cu_seqlens=cu.to(torch.int64 if wide else torch.int32).to(cuda))
    want, big = (torch.zeros(N, H, d, dtype=torch.float64) for _ in range(2))
    s, sbig = (torch.zeros(B, H, d, d, dtype=torch.float64) for _ in range(2))
    for b, (i, j) in enumerate(zip(ends, ends[1:])):
        if j > i:
            a = [x[i:j].double() for x in (q, k, v)]
            want[i:j], s[b] = _definition(*a, f.double(), d ** -0.5, None)
            big[i:j], sbig[b] = _definition(*(x.abs() for x in a), f.double(), d ** -0.5, None)
    _close(out, want, big, F32, 72 * U32)
    _close(left, s, sbig, F32, 72 * U32)
    assert bool((out[:ends[0]] == 0).all())



def test_attention_more_workgroups_than_a_launch(cuda):
    """As many sequences as are allowed, of one token, on 1025 heads: more than
    2^32 threads.  Small integers: every value is exact."""
    B, H = 65535, 1025
    g = torch.Generator(device=cuda).manual_seed(1)
    q = torch.randint(-8, 9, (B, 1, H, 1), generator=g, device=cuda).to(BF16)
    k, v = (torch.randint(-3, 4, (B, 1, 1, 1), generator=g, device=cuda).to(BF16) for _ in range(2))
    out, left = kernels.decay_attention(q, k, v, torch.zeros(H, device=cuda), scale=1.0)
    assert torch.equal(out, q * (k * v))
    assert torch.equal(left, (k * v).float().expand(B, H, 1, 1))
