"""The sequence operators against their definitions in 64 bits.

Tolerances.  Inputs are exact in both.  An output of type t is rounded once:
at most u(t) = eps(t) / 2 of its own value.  Before that everything is in (at
least) the precision of fp32, u = 2^-24, over sums of n terms a_i: an error of
at most about (n_rounded + 8) u sum |a_i|, where a term takes a few roundings
of its own (the power of the decay, products, the scale) and n_rounded is the
depth of the sum.  A depth of 64 covers sums by blocks of up to 64 terms and
the joins of the blocks; decays fade longer ones.  So

    |got - want| <= u(t) |want| + 72 * 2^-24 * bound,

bound the definition evaluated with absolute values; and a rounded value below
the smallest normal number n(t) of its type is off by half the spacing of the
subnormal ones, n(t) eps(t) / 2, not of its own.  Outputs of 16 bits may
hold factors of products in 16 significant bits (two 8-bit parts), 2^-16 of
each term: their second summand is 2^-15 * bound.
"""
import math

import pytest
import torch

from catfuse_amd import kernels

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
U32 = 2.0 ** -24


def _close(got, want, bound, dtype, factors):
    """The tolerance above; `factors`: relative error of the terms."""
    i = torch.finfo(dtype)
    tol = i.eps / 2 * want.abs().clamp(min=i.smallest_normal) + factors * bound
    off = (got.double().cpu() - want).abs()
    worst = (off - tol).max().item() if off.numel() else 0.0
    assert bool((off <= tol).all()), f"off by {off.max().item()}, {worst} over the tolerance"


def _definition(q, k, v, f, scale, state):
    """One sequence, [N, H, d] in fp64 on the CPU: (out, state)."""
    N, H, dk = q.shape
    g = H // k.shape[1]
    k, v = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
    w = torch.exp(f)
    s = torch.zeros(H, dk, v.shape[2], dtype=torch.float64) if state is None else state.clone()
    out = torch.empty(N, H, v.shape[2], dtype=torch.float64)
    for t in range(N):
        s = s * w[:, None, None] + k[t][:, :, None] * v[t][:, None, :]
        out[t] = (q[t][:, None, :] @ s)[:, 0] * scale
    return out, s


def _inputs(shape_q, shape_k, dv, dtype, seed, spikes=False):
    g = torch.Generator().manual_seed(seed)
    def make(*shape):
        if spikes:
            return (torch.rand(shape, generator=g) < 0.3).to(dtype)
        return torch.randn(shape, generator=g).to(dtype)
    return make(*shape_q), make(*shape_k), make(*shape_k[:-1], dv)


def _factors(dtype):
    return 72 * U32 if dtype == F32 else 2.0 ** -15


def _decays(H):
    """From no decay at all to one that keeps only the last tokens."""
    f = torch.log1p(-torch.exp2(-(1.0 + 10.0 * torch.arange(H) / max(H, 1))))
    f[0] = 0.0
    return f


def _check_attention(cuda, q, k, v, f, scale, state, cu, dtype):
    """q [B, N, H, d] or packed with offsets; one call against the definition."""
    out, left = kernels.decay_attention(
        q.to(cuda), k.to(cuda), v.to(cuda), f.to(cuda), scale=scale,
        state=None if state is None else state.to(cuda), cu_seqlens=cu if cu is None else cu.to(cuda))
    assert out.dtype == dtype and left.dtype == F32
    if cu is None:
        spans = [(q[b], k[b], v[b], out[b]) for b in range(q.shape[0])]
    else:
        spans = [(q[i:j], k[i:j], v[i:j], out[i:j]) for i, j in zip(cu.tolist(), cu.tolist()[1:])]
    for b, (qs, ks, vs, o) in enumerate(spans):
        s0 = None if state is None else state[b].double()
        a = [x.double() for x in (qs, ks, vs)]
        sc = q.shape[-1] ** -0.5 if scale is None else scale
        want, s = _definition(*a, f.double(), sc, s0)
        big, sbig = _definition(*(x.abs() for x in a), f.double(), abs(sc),
                                None if s0 is None else s0.abs())
        _close(o, want, big, dtype, _factors(dtype))
        _close(left[b], s, sbig, F32, 72 * U32)
    return out, left


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("N", [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 200])
def test_attention_lengths(cuda, dtype, N):
    q, k, v = _inputs((2, N, 3, 32), (2, N, 3, 32), 32, dtype, N)
    state = torch.randn(2, 3, 32, 32, generator=torch.Generator().manual_seed(1))
    _check_attention(cuda, q, k, v, _decays(3), None, state if N % 2 else None, None, dtype)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("dk,dv", [(1, 1), (8, 24), (16, 64), (31, 33), (32, 128), (64, 64),
                                   (72, 80), (100, 160), (128, 128), (129, 65), (256, 256),
                                   (200, 300)])
def test_attention_head_sizes(cuda, dtype, dk, dv):
    q, k, v = _inputs((1, 150, 4, dk), (1, 150, 2, dk), dv, dtype, dk + dv)
    state = torch.randn(1, 4, dk, dv, generator=torch.Generator().manual_seed(2))
    _check_attention(cuda, q, k, v, _decays(4), 0.3, state, None, dtype)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("lens", [[0, 1, 0], [1], [300, 0, 1, 63, 65, 2], [64, 64, 128, 1],
                                  [0], [5, 700]])
@pytest.mark.parametrize("wide", [False, True])
def test_attention_packed(cuda, dtype, lens, wide):
    q, k, v = _inputs((sum(lens), 4, 64), (sum(lens), 1, 64), 40, dtype, len(lens))
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int64 if wide else torch.int32)
    state = torch.randn(len(lens), 4, 64, 40, generator=torch.Generator().manual_seed(3))
    _check_attention(cuda, q, k, v, _decays(4), None, None if wide else state, cu, dtype)


@pytest.mark.parametrize("dtype,dk", [(F32, 64), (BF16, 128), (F16, 32)])
@pytest.mark.parametrize("N", [1500, 4099])
def test_attention_long(cuda, dtype, dk, N):
    """Long enough for every way of splitting a sequence."""
    q, k, v = _inputs((1, N, 2, dk), (1, N, 1, dk), dk, dtype, N)
    _check_attention(cuda, q, k, v, torch.tensor([-2.0 ** -10, -2.0 ** -4]), None, None, None,
                     dtype)


def test_attention_rest_rows(cuda):
    """Rows before, between and behind the sequences: zero in a new output,
    untouched in one given; offsets that are out of range or decrease."""
    q, k, v = (x.to(cuda) for x in _inputs((90, 2, 32), (90, 2, 32), 32, BF16, 5))
    f = _decays(2).to(cuda)
    cu = torch.tensor([7, 20, 70], dtype=torch.int32, device=cuda)
    out, left = kernels.decay_attention(q, k, v, f, cu_seqlens=cu)
    assert bool((out[:7] == 0).all()) and bool((out[70:] == 0).all())
    given = torch.full_like(out, 3.0)
    got, left2 = kernels.decay_attention(q, k, v, f, cu_seqlens=cu, out=given)
    assert got.data_ptr() == given.data_ptr()
    assert bool((got[:7] == 3).all()) and bool((got[70:] == 3).all())
    assert torch.equal(got[7:70], out[7:70]) and torch.equal(left, left2)
    for i, (a, b) in enumerate(((7, 20), (20, 70))):
        o, s = kernels.decay_attention(q[None, a:b], k[None, a:b], v[None, a:b], f)
        assert torch.equal(o[0], out[a:b]) and torch.equal(s[0], left[i])
    bad = torch.tensor([-5, 20, 10, 400], dtype=torch.int32, device=cuda)
    out, left = kernels.decay_attention(q, k, v, f, cu_seqlens=bad)
    o, s = kernels.decay_attention(q[None, :20], k[None, :20], v[None, :20], f)
    assert torch.equal(s[0], left[0]) and bool((left[1] == 0).all())
    o, s = kernels.decay_attention(q[None, 20:], k[None, 20:], v[None, 20:], f)
    assert torch.equal(o[0], out[20:]) and torch.equal(s[0], left[2])


@pytest.mark.parametrize("B,N,H", [(3000, 9000, 2), (1500, 9000, 1), (130, 70000, 2)])
def test_attention_many_sequences(cuda, B, N, H):
    """Offsets beyond one scan of a wave, whole sequences and split ones (of any
    length, many empty), some out of order: each as by itself."""
    g = torch.Generator().manual_seed(B)
    q, k, v = (x.to(cuda) for x in _inputs((N, H, 16), (N, 1, 16), 16, F32, B))
    f = _decays(H).to(cuda)
    cu = torch.randint(0, N + 1, (B + 1,), generator=g).sort()[0]
    cu[0], cu[-1] = 0, N
    want = cu.clone()
    cu[B // 2], cu[B // 3] = -7, 5                   # count as their predecessors
    want[B // 2], want[B // 3] = want[B // 2 - 1], want[B // 3 - 1]
    out, left = kernels.decay_attention(q, k, v, f, cu_seqlens=cu.to(cuda))
    for b in [0, 1, 63, 64, 65, B // 3 - 1, B // 3, B // 2 - 1, B // 2, B - 2, B - 1]:
        i, j = int(want[b]), int(want[b + 1])
        o, s = kernels.decay_attention(q[None, i:j], k[None, i:j], v[None, i:j], f)
        # (split in other places: both within the tolerance of the definition's bound)
        big, sbig = kernels.decay_attention(q[None, i:j].abs(), k[None, i:j].abs(),
                                            v[None, i:j].abs(), f)
        assert bool(((out[i:j] - o[0]).abs() <= 150 * U32 * big[0]).all())
        assert bool(((left[b] - s[0]).abs() <= 150 * U32 * sbig[0]).all())


def test_attention_scale(cuda):
    """A scale of another value in the same tensor is another scale."""
    q, k, v = (x.to(cuda) for x in _inputs((1, 40, 2, 16), (1, 40, 2, 16), 16, F32, 1))
    f, scale = _decays(2).to(cuda), torch.tensor(0.5)
    a, _ = kernels.decay_attention(q, k, v, f, scale=scale)
    scale *= 4
    b, _ = kernels.decay_attention(q, k, v, f, scale=scale)
    assert torch.equal(b, 4 * a) and bool((a != 0).any())


def test_attention_strides(cuda):
    """Heads of one fused projection, transposed heads, expanded keys, an
    output among other columns, misaligned rows: all the values of contiguous
    inputs."""
    g = torch.Generator().manual_seed(9)
    f = _decays(4).to(cuda)
    for dtype in (F32, BF16):
        x = torch.randn(2, 70, 8 * 40, generator=g).to(dtype).to(cuda)
        q = x[..., :160].unflatten(2, (4, 40))
        k = x[..., 160:240].unflatten(2, (2, 40))
        v = x[..., 240:].unflatten(2, (2, 40))
        want, s = kernels.decay_attention(q.contiguous(), k.contiguous(), v.contiguous(), f)
        wide = torch.full((2, 70, 4, 50), 7.0, dtype=dtype, device=cuda)
        out, left = kernels.decay_attention(q, k, v, f, out=wide[..., 3:43])
        assert torch.equal(out, want) and torch.equal(left, s)
        assert bool((wide[..., :3] == 7).all()) and bool((wide[..., 43:] == 7).all())
        qt = q.transpose(1, 2).contiguous().transpose(1, 2)
        flat = torch.empty(2 * 70 * 160 + 1, dtype=dtype, device=cuda)[1:].view(2, 70, 4, 40)
        flat.copy_(q)
        for other in (qt, flat):
            out, left = kernels.decay_attention(other, k, v, f)
            assert torch.equal(out, want) and torch.equal(left, s)
        twice = k.as_strided(k.shape, (k.stride(0), 8, 16, 1))     # rows that overlap
        want, s = kernels.decay_attention(q, twice.contiguous(), v, f)
        out, left = kernels.decay_attention(q, twice, v, f)
        assert torch.equal(out, want) and torch.equal(left, s)
        row = q[:1, :1].contiguous()          # one token: its strides mean nothing
        odd = row.as_strided(row.shape, (7, 0, 40, 1))
        a = kernels.decay_attention(row, k[:1, :1].contiguous(), v[:1, :1].contiguous(), f)
        b = kernels.decay_attention(odd, k[:1, :1], v[:1, :1], f)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        one = k[:, :1].expand(2, 70, 2, 40)
        want, s = kernels.decay_attention(q, one.contiguous(), v, f)
        out, left = kernels.decay_attention(q, one, v, f)
        assert torch.equal(out, want) and torch.equal(left, s)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("which", ["q", "k", "v"])
def test_attention_keeps_later_values_from_earlier_tokens(cuda, dtype, bad, which):
    """A value that is not finite in token 70 of sequence 0: the tokens before
    it and the other sequence have the bits that they have without it."""
    x = dict(zip("qkv", (t.to(cuda) for t in _inputs((2, 140, 2, 64), (2, 140, 2, 64), 64, dtype,
                                                     3))))
    f = _decays(2).to(cuda)
    want, left = kernels.decay_attention(*x.values(), f)
    x[which][0, 70, 1, 5] = bad
    out, s = kernels.decay_attention(*x.values(), f)
    assert torch.equal(out[1], want[1]) and torch.equal(s[1], left[1])
    assert torch.equal(out[0, :, 0], want[0, :, 0]) and torch.equal(s[0, 0], left[0, 0])
    assert torch.equal(out[0, :70, 1], want[0, :70, 1])
    if which == "q":
        assert not bool(out[0, 70, 1].isfinite().any())
        assert torch.equal(out[0, 71:, 1], want[0, 71:, 1]) and torch.equal(s, left)
    elif which == "k":      # its row of the state, and through it every later output
        assert not bool(out[0, 70:, 1].isfinite().any())
        assert not bool(s[0, 1, 5].isfinite().any())
        assert bool(s[0, 1, :5].isfinite().all()) and bool(s[0, 1, 6:].isfinite().all())
    else:                   # its column
        assert not bool(out[0, 70:, 1, 5].isfinite().any())
        assert not bool(s[0, 1, :, 5].isfinite().any())
        rest = [c for c in range(64) if c != 5]
        assert torch.equal(out[0, :, 1, rest], want[0, :, 1, rest])
        assert torch.equal(s[0, 1][:, rest], left[0, 1][:, rest])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_attention_decay_ends(cuda, dtype):
    """log_decay -inf (only the token itself), 0 (everything), above 0 (the
    past grows) and one so low that its powers vanish."""
    for N, growth in ((100, 0.02), (900, 0.002)):
        q, k, v = _inputs((1, N, 4, 32), (1, N, 4, 32), 32, dtype, 8)
        f = torch.tensor([-math.inf, 0.0, growth, -50.0])
        state = torch.randn(1, 4, 32, 32, generator=torch.Generator().manual_seed(4))
        _check_attention(cuda, q, k, v, f, None, state, None, dtype)


def test_attention_large_values(cuda):
    """fp16 heads whose products pass the range of fp16 (their fp32 sums do
    not) and values far below it."""
    for big, small in ((300.0, 2.0 ** -10), (2.0 ** -8, 2.0 ** -8)):
        q, k, v = _inputs((1, 90, 1, 128), (1, 90, 1, 128), 64, F16, 6)
        q, k, v = (q * big).half(), (k * big).half(), (v * small).half()
        _check_attention(cuda, q, k, v, torch.tensor([-0.05]), 2.0 ** -12, None, None, F16)


def test_attention_spikes_are_exact(cuda):
    """Spikes without a decay: every sum is an integer below 2^24."""
    q, k, v = _inputs((3, 196, 4, 32), (3, 196, 4, 32), 32, F16, 2, spikes=True)
    f = torch.zeros(4)
    out, left = kernels.decay_attention(q.to(cuda), k.to(cuda), v.to(cuda), f.to(cuda), scale=1.0)
    for b in range(3):
        want, s = _definition(*(x[b].double() for x in (q, k, v)), f.double(), 1.0, None)
        assert torch.equal(left[b].cpu().double(), s)
        assert torch.equal(out[b].cpu(), want.to(F16))


def test_attention_empty(cuda):
    f = torch.zeros(2, device=cuda)
    def z(*s):
        return torch.zeros(s, device=cuda)
    out, s = kernels.decay_attention(z(0, 5, 2, 8), z(0, 5, 2, 8), z(0, 5, 2, 8), f)
    assert out.shape == (0, 5, 2, 8) and s.shape == (0, 2, 8, 8)
    first = torch.randn(3, 2, 8, 8, device=cuda)
    out, s = kernels.decay_attention(z(3, 0, 2, 8), z(3, 0, 2, 8), z(3, 0, 2, 8), f, state=first)
    assert out.shape == (3, 0, 2, 8) and torch.equal(s, first)
    out, s = kernels.decay_attention(z(4, 2, 8) + 1, z(4, 2, 8), z(4, 2, 8), f,
                                     cu_seqlens=torch.zeros(1, dtype=torch.int32, device=cuda))
    assert bool((out == 0).all()) and s.shape == (0, 2, 8, 8)
    only = kernels.decay_attention(z(1, 4, 2, 8), z(1, 4, 2, 8), z(1, 4, 2, 8), f,
                                   return_state=False)
    assert isinstance(only, torch.Tensor) and only.shape == (1, 4, 2, 8)


def test_attention_parts_join(cuda):
    """A prompt in pieces through the states, and the rest of it token by
    token: the whole prompt's output."""
    q, k, v = (x.to(cuda) for x in _inputs((2, 301, 4, 64), (2, 301, 2, 64), 32, F32, 12))
    f = _decays(4).to(cuda)
    want, last = kernels.decay_attention(q, k, v, f)
    s, outs = None, []
    for a, b in ((0, 100), (100, 101), (101, 280)):
        o, s = kernels.decay_attention(q[:, a:b], k[:, a:b], v[:, a:b], f, state=s)
        outs.append(o)
    for t in range(280, 301):
        outs.append(kernels.decay_attention_step(q[:, t], k[:, t], v[:, t], f, s)[:, None])
    got = torch.cat(outs, 1)
    # both within 72 u of the definition's bound
    bound, sb = kernels.decay_attention(q.abs(), k.abs(), v.abs(), f)
    assert bool(((got - want).abs() <= 150 * U32 * bound).all())
    assert bool(((s - last).abs() <= 150 * U32 * sb).all())


# ---------------------------------------------------------------------------
# one token
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,H,Hk,dk,dv", [(1, 1, 1, 1, 1), (1, 12, 12, 32, 32), (5, 4, 1, 64, 64),
                                             (3, 4, 2, 80, 72), (2, 2, 2, 33, 31), (7, 8, 2, 128, 128),
                                             (2, 2, 1, 256, 256), (2, 1, 1, 200, 300)])
def test_step(cuda, dtype, rows, H, Hk, dk, dv):
    q, k, v = _inputs((rows, H, dk), (rows, Hk, dk), dv, dtype, rows + dk)
    g = torch.Generator().manual_seed(7)
    pool = torch.randn(rows + 3, H, dk, dv, generator=g)
    slots = torch.randperm(rows + 3, generator=g)[:rows]
    f = _decays(H)
    for wide in (False, True):
        state = pool.to(cuda)
        out = kernels.decay_attention_step(q.to(cuda), k.to(cuda), v.to(cuda), f.to(cuda), state,
                                           slots=slots.to(torch.int64 if wide else torch.int32)
                                           .to(cuda))
        for i in range(rows):
            a = [x[i:i + 1].double() for x in (q, k, v)]
            want, s = _definition(*a, f.double(), dk ** -0.5, pool[slots[i]].double())
            big, sbig = _definition(*(x.abs() for x in a), f.double(), dk ** -0.5,
                                    pool[slots[i]].double().abs())
            # a sum of dk terms: depth of at most dk
            _close(out[i:i + 1], want, big, dtype, (dk + 8) * U32)
            _close(state[slots[i]], s, sbig, F32, 4 * U32)
        rest = [i for i in range(rows + 3) if i not in slots.tolist()]
        assert torch.equal(state[rest].cpu(), pool[rest])


def test_step_slots(cuda):
    """Padding rows, slots outside the pool, no slots, and rows of one slot as
    consecutive tokens."""
    q, k, v = (x.to(cuda) for x in _inputs((9, 4, 64), (9, 2, 64), 64, BF16, 1))
    f = _decays(4).to(cuda)
    pool = torch.randn(4, 4, 64, 64, device=cuda)
    slots = torch.tensor([2, -1, 0, 2, 4, 1 << 30, 2, 0, -(1 << 31)], dtype=torch.int32, device=cuda)
    state = pool.clone()
    out = kernels.decay_attention_step(q, k, v, f, state, slots=slots)
    want = pool.clone()
    for i, s in enumerate(slots.tolist()):
        if 0 <= s < 4:
            o = kernels.decay_attention_step(q[i:i + 1], k[i:i + 1], v[i:i + 1], f, want[s:s + 1])
            assert torch.equal(o[0], out[i])
        else:
            assert bool((out[i] == 0).all())
    assert torch.equal(state, want)
    same = pool.clone()
    o = kernels.decay_attention_step(q[:4], k[:4], v[:4], f, same)
    other = pool.clone()
    o2 = kernels.decay_attention_step(q[:4], k[:4], v[:4], f, other,
                                      slots=torch.arange(4, device=cuda))
    assert torch.equal(o, o2) and torch.equal(same, other)


def test_step_many_rows(cuda):
    """More rows than a workgroup scans at once, every second one a repeat."""
    rows, slots = 700, torch.arange(700) // 2
    q, k, v = (x.to(cuda) for x in _inputs((rows, 1, 16), (rows, 1, 16), 8, F32, 4))
    f = torch.tensor([-0.1], device=cuda)
    pool = torch.randn(350, 1, 16, 8, device=cuda)
    state = pool.clone()
    out = kernels.decay_attention_step(q, k, v, f, state, slots=slots.to(cuda))
    a = kernels.decay_attention_step(q[::2], k[::2], v[::2], f, pool)
    b = kernels.decay_attention_step(q[1::2], k[1::2], v[1::2], f, pool)
    assert torch.equal(out[::2], a) and torch.equal(out[1::2], b) and torch.equal(state, pool)


def test_step_many_tokens(cuda):
    """4096 tokens, one after another: the rounding of the decay does not add up."""
    f = torch.tensor([-2.0 ** -12, -2.0 ** -5])
    g = torch.Generator().manual_seed(3)
    N = 4096
    k, v = torch.randn(N, 2, 16, generator=g), torch.randn(N, 2, 8, generator=g)
    state = torch.zeros(1, 2, 16, 8, device=cuda)
    kg, vg, fg = k.to(cuda), v.to(cuda), f.to(cuda)
    for t in range(N):
        kernels.decay_attention_step(kg[t:t + 1], kg[t:t + 1], vg[t:t + 1], fg, state)
    left = torch.exp(f.double() * (N - 1 - torch.arange(N, dtype=torch.float64))[:, None])
    def total(k, v):
        return torch.einsum("th,thi,thj->hij", left, k, v)
    want, big = total(k.double(), v.double()), total(k.double().abs(), v.double().abs())
    # two roundings a token of a state that fades: at most 2 u sum_t |S_t| w^(N-1-t);
    # |S_t| is bound by big (1 - w^t) / (1 - w^N), so the sum by big times the
    # horizon 1 / (1 - w), of random signs by its root: 64, and six deviations
    _close(state[0], want, big, F32, 2 * 6 * 64 * U32)


def test_step_strides(cuda):
    """States of one layer among others, heads of a fused projection, an
    output among other columns, misaligned states."""
    x = torch.randn(5, 8 * 40, device=cuda).bfloat16()
    q, k, v = (t.unflatten(1, (-1, 40)) for t in (x[:, :160], x[:, 160:240], x[:, 240:]))
    f = _decays(4).to(cuda)
    layers = torch.randn(6, 3, 4, 40, 40, device=cuda)
    keep = layers.clone()
    slots = torch.tensor([5, 0, 3, 1, 2], dtype=torch.int32, device=cuda)
    plain = layers[:, 1].contiguous()
    want = kernels.decay_attention_step(q.contiguous(), k.contiguous(), v.contiguous(), f, plain,
                                        slots=slots)
    wide = torch.full((5, 4, 50), 7.0, dtype=BF16, device=cuda)
    out = kernels.decay_attention_step(q, k, v, f, layers[:, 1], slots=slots, out=wide[..., 5:45])
    assert torch.equal(out, want) and torch.equal(layers[:, 1], plain)
    assert torch.equal(layers[:, 0], keep[:, 0]) and torch.equal(layers[:, 2], keep[:, 2])
    assert bool((wide[..., :5] == 7).all()) and bool((wide[..., 45:] == 7).all())
    off = torch.empty(6 * 4 * 40 * 40 + 1, device=cuda)[1:].view(6, 4, 40, 40)
    off.copy_(keep[:, 1])
    out = kernels.decay_attention_step(q, k, v, f, off, slots=slots)
    assert torch.equal(off, plain)
    bound = 48 * U32 * (q.float().abs().sum(-1, keepdim=True) * 200)
    assert bool(((out.float() - want.float()).abs() <= bound + want.float().abs() * 2.0 ** -7).all())


# ---------------------------------------------------------------------------
# norms and rotation
# ---------------------------------------------------------------------------

def _turned(x, pos, freqs, sections, interleaved=False, inverse=False, weight=None, eps=None):
    """(values, bound) in fp64 on the CPU; pos [axes, tokens]."""
    x = x.double()
    if eps is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)
        if weight is not None:
            x = x * weight.double()
    pairs = freqs.shape[0]
    axis = torch.repeat_interleave(torch.arange(len(sections)), torch.tensor(sections))
    angle = pos.double()[axis].t() * freqs
    if inverse:
        angle = -angle
    c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    head = x[..., :2 * pairs]
    a, b = (head[..., 0::2], head[..., 1::2]) if interleaved else (head[..., :pairs],
                                                                  head[..., pairs:])
    ya, yb, size = a * c - b * s, b * c + a * s, a.abs() + b.abs()
    if interleaved:
        y, m = torch.stack([ya, yb], -1).flatten(-2), torch.stack([size, size], -1).flatten(-2)
    else:
        y, m = torch.cat([ya, yb], -1), torch.cat([size, size], -1)
    rest = x[..., 2 * pairs:]
    return torch.cat([y, rest], -1), torch.cat([m, rest.abs()], -1)


# Roundings of a term of the rotation: the angle's rounding to fp32 turns
# (half a unit of at most 1/2 turn: 2^-26 turns, 2 pi 2^-26 < 2 u), the sine
# (a few units: 4 u), a product and the sum (2 u), the reduced angle in fp64
# (2^-52 of the turns: below u for positions under 2^28); with a norm the sum
# of d squares (at most (d / lanes + 16) u under a root, so half of it), the
# root, the quotient and two products.
TURN = 10 * U32


def _norm(d):
    return TURN + (d / 2 + 16) * U32


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("d,rot", [(2, 2), (8, 4), (8, 8), (16, 16), (32, 32), (64, 64), (80, 80), (128, 128),
                                   (128, 32), (256, 256), (96, 48), (70, 70), (100, 36), (33, 32),
                                   (512, 512), (512, 2), (511, 16), (256, 16)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_sizes(cuda, dtype, d, rot, interleaved):
    g = torch.Generator().manual_seed(d + rot)
    x = torch.randn(19, 3, d, generator=g).to(dtype)
    pos = torch.randint(0, 100000, (19,), generator=g)
    freqs = kernels.rotary_freqs(rot // 2)
    y = kernels.rotary(x.to(cuda), pos.to(cuda), freqs.to(cuda), interleaved=interleaved)
    want, size = _turned(x, pos[None], freqs, (rot // 2,), interleaved)
    _close(y, want, size, dtype, TURN)
    assert torch.equal(y[..., rot:].cpu(), x[..., rot:])
    many = x.repeat(97, 1, 1)[:, :1].to(cuda)         # more tokens than a workgroup takes, one head
    z = kernels.rotary(many, pos.repeat(97).to(cuda), freqs.to(cuda), interleaved=interleaved)
    assert torch.equal(z, y[:, :1].repeat(97, 1, 1))
    back = kernels.rotary(y, pos.to(cuda), freqs.to(cuda), interleaved=interleaved, inverse=True)
    want, size = _turned(y.cpu(), pos[None], freqs, (rot // 2,), interleaved, inverse=True)
    _close(back, want, size, dtype, TURN)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("sections", [(16,), (6, 10), (4, 6, 6), (0, 16, 0), (1, 14, 1)])
@pytest.mark.parametrize("kind", [torch.int32, torch.int64, torch.float32])
def test_rotary_axes(cuda, dtype, sections, kind):
    g = torch.Generator().manual_seed(len(sections))
    x = torch.randn(2, 3, 5, 2, 40, generator=g).to(dtype)
    pos = torch.randint(-50, 1 << 20, (len(sections), 2, 3, 5), generator=g).to(kind)
    if kind == torch.float32:
        pos = pos / 8
    freqs = kernels.rotary_freqs(16, sections=sections)
    y = kernels.rotary(x.to(cuda), pos.to(cuda), freqs.to(cuda), sections=sections)
    want, size = _turned(x.flatten(0, 2), pos.flatten(1), freqs, sections)
    _close(y.flatten(0, 2), want, size, dtype, TURN)
    # one position for all axes; positions broadcast over the first dimension
    y = kernels.rotary(x.to(cuda), pos[0].to(cuda), freqs.to(cuda), sections=sections)
    want, size = _turned(x.flatten(0, 2), pos[:1].expand_as(pos).flatten(1), freqs, sections)
    _close(y.flatten(0, 2), want, size, dtype, TURN)
    y = kernels.rotary(x.to(cuda), pos[:, :1].to(cuda), freqs.to(cuda), sections=sections)
    want, size = _turned(x.flatten(0, 2), pos[:, :1].expand_as(pos).flatten(1), freqs, sections)
    _close(y.flatten(0, 2), want, size, dtype, TURN)


def test_rotary_large(cuda):
    """More output than the caches hold (streaming stores): the bits of the same
    rows in small launches."""
    N = 13000
    x = torch.randn(N, 32, 128, device=cuda).bfloat16()
    pos, freqs = torch.arange(N, device=cuda), kernels.rotary_freqs(64, device=cuda)
    y = kernels.rotary(x, pos, freqs)
    for i in range(0, N, 4001):
        assert torch.equal(y[i:i + 4001], kernels.rotary(x[i:i + 4001], pos[i:i + 4001], freqs))


def test_rotary_far_positions(cuda):
    """Positions of up to 2^31 keep an angle within 2^-52 of the turns."""
    x = torch.ones(4, 1, 8, device=cuda)
    pos = torch.tensor([0, 1 << 20, (1 << 31) - 1, -(1 << 31)], dtype=torch.int32, device=cuda)
    freqs = kernels.rotary_freqs(4)
    y = kernels.rotary(x, pos, freqs.to(cuda))
    want, size = _turned(x.cpu(), pos.cpu()[None], freqs, (4,))
    # fp64 products on both sides: 2^31 radians times 2^-52, twice
    _close(y, want, size, F32, TURN + 2.0 ** -20)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("d,rot,H,Hk,N", [(32, 32, 12, 12, 7), (128, 128, 32, 8, 5), (64, 32, 4, 1, 1),
                                          (80, 80, 3, 3, 65), (72, 70, 2, 1, 9), (256, 256, 1, 1, 300),
                                          (512, 6, 1, 1, 3)])
@pytest.mark.parametrize("weights", ["none", "shared", "heads"])
def test_qk_norm_rotary(cuda, dtype, d, rot, H, Hk, N, weights):
    g = torch.Generator().manual_seed(d + N)
    q, k = (torch.randn(N, n, d, generator=g).to(dtype) for n in (H, Hk))
    q[0] = 0                              # a silent head: its norm is sqrt(eps)
    w = [None, None]
    if weights == "shared":
        w = [torch.randn(d, generator=g) for _ in range(2)]
    elif weights == "heads":
        w = [torch.randn(n, d, generator=g).to(dtype) for n in (H, Hk)]
    pos = torch.randint(0, 5000, (N,), generator=g)
    freqs = kernels.rotary_freqs(rot // 2)
    got = kernels.qk_norm_rotary(q.to(cuda), k.to(cuda), pos.to(cuda), freqs.to(cuda),
                                 q_weight=None if w[0] is None else w[0].to(cuda),
                                 k_weight=None if w[1] is None else w[1].to(cuda), eps=1e-5)
    for x, y, wt in zip((q, k), got, w):
        want, size = _turned(x, pos[None], freqs, (rot // 2,), weight=wt, eps=1e-5)
        _close(y, want, size, dtype, _norm(d))


def test_rotary_strides_and_in_place(cuda):
    """Heads of a fused projection, in place or not, an output among other
    columns, misaligned rows: the bits of contiguous inputs."""
    for dtype in (F32, BF16):
        x = torch.randn(2, 9, 10 * 64, device=cuda).to(dtype)
        q, k = x[..., :256].unflatten(2, (4, 64)), x[..., 256:384].unflatten(2, (2, 64))
        pos, freqs = torch.arange(9, device=cuda), kernels.rotary_freqs(32, device=cuda)
        want = kernels.qk_norm_rotary(q.contiguous(), k.contiguous(), pos[None], freqs)
        got = kernels.qk_norm_rotary(q, k, pos[None], freqs)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        wide = torch.full((2, 9, 4, 80), 7.0, dtype=dtype, device=cuda)
        got = kernels.qk_norm_rotary(q, k, pos[None], freqs, out=(wide[..., 8:72], None))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        assert bool((wide[..., :8] == 7).all()) and bool((wide[..., 72:] == 7).all())
        tail = x[..., 384:].clone()
        got = kernels.qk_norm_rotary(q, k, pos[None], freqs, out=(q, k))
        assert got[0].data_ptr() == q.data_ptr()
        assert torch.equal(q, want[0]) and torch.equal(k, want[1])
        assert torch.equal(x[..., 384:], tail)
        y = torch.randn(11, 3, 64, device=cuda).to(dtype)
        off = torch.empty(11 * 3 * 64 + 1, dtype=dtype, device=cuda)[1:].view(11, 3, 64)
        off.copy_(y)
        args = (torch.arange(11, device=cuda), freqs)
        a, b = kernels.rotary(y, *args), kernels.rotary(off, *args)
        assert torch.equal(a, b)
        t = y.transpose(0, 1).contiguous().transpose(0, 1)
        assert torch.equal(kernels.rotary(t, *args), a)
    z = torch.zeros(0, 3, 64, device=cuda)
    assert kernels.rotary(z, torch.zeros(0, dtype=torch.int64, device=cuda), freqs).shape == z.shape


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------

def test_prompt_then_tokens(cuda):
    """A projection's heads normed and turned in place, a packed prompt, then
    tokens from a pool, the outputs driving a LIF over the steps: against the
    same in fp64, spikes compared where the potential is not at its threshold."""
    from catfuse_amd.runtime import lif_multistep
    H, Hk, d, lens, new = 4, 2, 32, [37, 0, 90], 6
    N = sum(lens)
    g = torch.Generator().manual_seed(11)
    x = torch.randn(N + new * 3, (H + 2 * Hk) * d, generator=g)
    pos = torch.cat([torch.arange(n) for n in lens] +
                    [torch.tensor(lens) + t for t in range(new)])
    freqs, f = kernels.rotary_freqs(d // 2), _decays(H)
    y = x.to(cuda)
    q, k, v = (y[:, a * d:b * d].unflatten(1, (b - a, d))
               for a, b in ((0, H), (H, H + Hk), (H + Hk, H + 2 * Hk)))
    kernels.qk_norm_rotary(q, k, pos.to(cuda), freqs.to(cuda), out=(q, k))
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32).to(cuda)
    fg = f.to(cuda)
    out, state = kernels.decay_attention(q[:N], k[:N], v[:N], fg, cu_seqlens=cu)
    pool = torch.empty(5, H, d, d, device=cuda)
    slots = torch.tensor([4, 0, 2], device=cuda)
    pool[slots] = state
    outs = []
    for t in range(new):
        r = slice(N + 3 * t, N + 3 * t + 3)
        outs.append(kernels.decay_attention_step(q[r], k[r], v[r], fg, pool, slots=slots))
    tokens = torch.stack(outs)                          # [new, 3, H, d]
    spikes, _ = lif_multistep(tokens, v_threshold=0.2)

    xd = x.double()
    a = [t.unflatten(1, (-1, d)) for t in (xd[:, :H * d], xd[:, H * d:(H + Hk) * d],
                                           xd[:, (H + Hk) * d:])]
    qd = _turned(a[0], pos[None], freqs, (d // 2,), eps=1e-6)[0]
    kd = _turned(a[1], pos[None], freqs, (d // 2,), eps=1e-6)[0]
    at = [0] + torch.tensor(lens).cumsum(0).tolist()
    steps = []
    for b in range(3):
        rows = list(range(at[b], at[b + 1])) + [N + 3 * t + b for t in range(new)]
        o, s = _definition(qd[rows], kd[rows], a[2][rows], f.double(), d ** -0.5, None)
        big, sbig = _definition(qd[rows].abs(), kd[rows].abs(), a[2][rows].abs(), f.double(),
                                d ** -0.5, None)
        tol = 72 * U32 + 2 * _norm(d)                   # the heads' own errors, of q and of k
        _close(out[at[b]:at[b + 1]], o[:lens[b]], big[:lens[b]], F32, tol)
        _close(tokens[:, b], o[lens[b]:], big[lens[b]:], F32, tol)
        _close(pool[slots[b]], s, sbig, F32, tol)
        steps.append(o[lens[b]:])
    z, pot = torch.stack(steps, 1), torch.zeros(3, H, d, dtype=torch.float64)
    alive = torch.ones_like(pot, dtype=torch.bool)      # potentials that never were at the threshold
    for t in range(new):
        pot = pot + (z[t] - pot) / 2
        alive &= (pot - 0.2).abs() > 1e-3
        fire = pot >= 0.2
        assert torch.equal(spikes[t].cpu()[alive], fire.float()[alive])
        pot = torch.where(fire, torch.zeros_like(pot), pot)
    assert alive.float().mean() > 0.9


def test_graph_and_streams(cuda):
    """Captured calls replay with new inputs; two graphs share nothing; calls
    on another stream give the same bits."""
    def data(seed):
        return [t.to(cuda) for t in _inputs((1, 700, 4, 64), (1, 700, 2, 64), 64, BF16, seed)]
    f = _decays(4).to(cuda)
    pos, freqs = torch.arange(700, device=cuda), kernels.rotary_freqs(32, device=cuda)

    def once(q, k, v, pool):
        q, k = kernels.qk_norm_rotary(q, k, pos[None], freqs)
        o, s = kernels.decay_attention(q, k, v, f)
        p = kernels.decay_attention_step(q[:, -1], k[:, -1], v[:, -1], f, pool)
        return o, s, p
    graphs = []
    for seed in (1, 2):
        x, pool = data(seed), torch.zeros(1, 4, 64, 64, device=cuda)
        once(*x, pool)
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            got = once(*x, pool)
        graphs.append((gr, x, pool, got))
    for rep in range(3):
        wants = []
        for n, (gr, x, pool, got) in enumerate(graphs):
            for a, b in zip(x, data(10 * rep + n)):
                a.copy_(b)
            pool.fill_(0.5)
            wants.append(once(*x, pool.clone()))
        torch.cuda.synchronize()
        for gr, *_ in graphs:
            gr.replay()
        torch.cuda.synchronize()
        for (gr, x, pool, got), want in zip(graphs, wants):
            assert all(torch.equal(a, b) for a, b in zip(got, want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    x = data(5)
    want = once(*x, torch.ones(1, 4, 64, 64, device=cuda))
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = once(*x, torch.ones(1, 4, 64, 64, device=cuda))
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
