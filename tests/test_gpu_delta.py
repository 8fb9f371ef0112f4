"""The delta rule's attention against its definition in 64 bits.

Tolerances.  Inputs are exact in both.  With A_t = w_t (I - beta_t k_t k_t^T) and
rho_t = w_t max(1, |1 - beta_t |k_t|^2|) its norm, an error in a column of the
state goes on by at most rho_t a token.  What is added to it: the roundings of the
sums that make u_t and the state, each a depth times u = 2^-24 of the sum's terms.
Per token |k_t| |u_t| twice (u_t itself, its product with k_t) and
beta_t |k_t| |v_t|; the state's own rounding, and that of k_t^T S through u, once a
chunk of at least 32 tokens, w_t |S_{t-1}| (1 + beta_t |k_t|^2) / 32 a token.  With

    n_t = rho_t n_{t-1} + 2 |k_t| |u_t| + beta_t |k_t| |v_t|
          + w_t |S_{t-1}| (1 + beta_t |k_t|^2) / 32,          n_0 = |S_0|

(column by column, 2-norms) the state is within depth u n_t of its definition and
the output within depth u scale |q_t| n_t, besides the half unit that its type
rounds off.  The depth: 72 as for sums by blocks of up to 64 terms and their joins,
times what the inverse of a chunk's I + L adds, at most the norm of |T| |I + L|
(rows of T times the terms of the sums they replace), taken from the definition.
"""
import math

import pytest
import torch

from catfuse_amd import kernels

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
U32 = 2.0 ** -24


def _close(got, want, dtype, tol):
    """tol: the tolerance before the rounding to dtype."""
    i = torch.finfo(dtype)
    tol = tol + i.eps / 2 * want.abs().clamp(min=i.smallest_normal)
    off = (got.double().cpu() - want).abs()
    worst = (off - tol).max().item() if off.numel() else 0.0
    assert bool((off <= tol).all()), f"off by {off.max().item()}, {worst} over the tolerance"


def _spread(x, H):
    """[N, heads, d] with the heads that H heads read."""
    return x.repeat_interleave(H // x.shape[-2], -2)


def _definition(q, k, v, beta, f, scale, state):
    """One sequence in fp64 on the CPU, q, k, v [N, heads, d], beta and f [N, H]:
    (out, state, bounds n of every token's output and of the state)."""
    N, H = beta.shape
    q, k, v = (_spread(x, H) for x in (q, k, v))
    dk, dv = k.shape[2], v.shape[2]
    s = torch.zeros(H, dk, dv, dtype=torch.float64) if state is None else state.clone()
    n = s.norm(dim=1)
    out, bound = torch.empty(N, H, dv, dtype=torch.float64), torch.empty(N, H, dv, dtype=torch.float64)
    for t in range(N):
        w, b, kt = torch.exp(f[t])[:, None], beta[t][:, None], k[t]
        kk = (kt * kt).sum(1, keepdim=True)
        mass = w * s.norm(dim=1) * (1 + b.abs() * kk) / 32
        s = s * w[:, :, None]
        u = b * (v[t] - (kt[:, None, :] @ s)[:, 0])
        s = s + kt[:, :, None] * u[:, None, :]
        out[t] = (q[t][:, None, :] @ s)[:, 0] * scale
        n = w * torch.clamp((1 - b * kk).abs(), min=1) * n + mass + \
            kk.sqrt() * (2 * u.abs() + b.abs() * v[t].abs())
        bound[t] = abs(scale) * q[t].norm(dim=1)[:, None] * n
    return out, s, bound, n


def _solve_norm(k, beta, f, H, C=64):
    """The largest norm of |T| |I + L| over the chunks of one sequence."""
    k, N, most = _spread(k, H), k.shape[0], 1.0
    for a in range(0, N, C):
        kc = k[a:a + C].transpose(0, 1)
        g = f[a:a + C].clamp(min=-1e4).cumsum(0).t()
        low = (beta[a:a + C].t()[:, :, None] * torch.exp((g[:, :, None] - g[:, None, :]).clamp(max=700)) *
               (kc @ kc.transpose(1, 2))).tril(-1)
        eye = torch.eye(low.shape[1], dtype=torch.float64)
        inv = torch.linalg.solve_triangular(eye + low, eye.expand_as(low), upper=False)
        most = max(most, (inv.abs() @ (eye + low.abs())).sum(2).max().item())
    return most


def _inputs(lead, heads, dk, dv, dtype, seed, H=None, unit=True):
    """q, k, v with heads = (Hq, Hk, Hv); beta in 0 .. 1 and log decays."""
    g = torch.Generator().manual_seed(seed)
    H = max(heads) if H is None else H
    def normal(*shape):
        return torch.randn(shape, generator=g)
    q, k, v = normal(*lead, heads[0], dk), normal(*lead, heads[1], dk), normal(*lead, heads[2], dv)
    if unit:
        k = k / k.norm(dim=-1, keepdim=True)
    beta = torch.sigmoid(normal(*lead, H))
    f = -torch.exp2(-1.0 - 9.0 * torch.arange(H) / H) * torch.exp(normal(*lead, H))
    return q.to(dtype), k.to(dtype), v.to(dtype), beta, f


def _check(cuda, x, scale=None, state=None, cu=None, **more):
    """One call of x = (q, k, v, beta, log_decay), rows or packed, against the
    definition."""
    q, k, v, beta, f = x
    dtype, H = q.dtype, beta.shape[-1]
    out, left = kernels.delta_attention(*(None if t is None else t.to(cuda) for t in x), scale=scale,
                                        state=None if state is None else state.to(cuda),
                                        cu_seqlens=None if cu is None else cu.to(cuda), **more)
    assert out.dtype == dtype and left.dtype == F32
    f = torch.zeros(beta.shape) if f is None else f
    if cu is None:
        spans = [([t[b] for t in (q, k, v, beta, f)], out[b]) for b in range(q.shape[0])]
    else:
        at = cu.tolist()
        spans = [([t[i:j] for t in (q, k, v, beta, f)], out[i:j]) for i, j in zip(at, at[1:])]
    for b, (a, o) in enumerate(spans):
        a = [t.double() for t in a]
        sc = q.shape[-1] ** -0.5 if scale is None else scale
        s0 = None if state is None else state[b].double()
        want, s, bound, n = _definition(*a, sc, s0)
        depth = 72 * _solve_norm(a[1], a[3], a[4], H)
        _close(o, want, dtype, depth * U32 * bound)
        _close(left[b], s, F32, (depth * U32 * n)[:, None, :])
    return out, left


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("N", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200])
@pytest.mark.parametrize("d", [32, 128])
def test_lengths(cuda, dtype, N, d):
    x = _inputs((2, N), (3, 3, 3), d, d, dtype, N)
    state = torch.randn(2, 3, d, d, generator=torch.Generator().manual_seed(1))
    _check(cuda, x, state=state if N % 2 else None)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("dk,dv", [(1, 1), (8, 24), (16, 64), (31, 33), (32, 128), (64, 64),
                                   (72, 80), (100, 160), (128, 128), (129, 65), (256, 256),
                                   (200, 300)])
def test_head_sizes(cuda, dtype, dk, dv):
    x = _inputs((1, 150), (4, 2, 2), dk, dv, dtype, dk + dv)
    state = torch.randn(1, 4, dk, dv, generator=torch.Generator().manual_seed(2))
    _check(cuda, x, scale=0.3, state=state)


@pytest.mark.parametrize("heads,H", [((1, 1, 1), 1), ((4, 4, 4), 4), ((2, 2, 6), 6), ((6, 3, 2), 6),
                                     ((1, 2, 1), 4), ((2, 1, 4), 8)])
def test_head_groups(cuda, heads, H):
    for dtype in (F32, BF16):
        _check(cuda, _inputs((2, 90), heads, 64, 48, dtype, H, H=H))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("lens", [[0, 1, 0], [1], [300, 0, 1, 63, 65, 2], [64, 64, 128, 1],
                                  [0], [5, 700], [31, 33, 0, 0, 97]])
@pytest.mark.parametrize("d", [64, 128])
def test_packed(cuda, dtype, lens, d):
    x = _inputs((sum(lens),), (4, 1, 2), d, 40, dtype, len(lens))
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int64 if d == 64 else torch.int32)
    state = torch.randn(len(lens), 4, d, 40, generator=torch.Generator().manual_seed(3))
    _check(cuda, x, state=None if len(lens) % 2 else state, cu=cu)


@pytest.mark.parametrize("dtype,d", [(F32, 64), (BF16, 128), (F16, 32), (BF16, 256)])
@pytest.mark.parametrize("N", [1500, 4099])
def test_long(cuda, dtype, d, N):
    """Long enough for every way of splitting a sequence."""
    state = torch.randn(1, 2, d, d, generator=torch.Generator().manual_seed(N))
    _check(cuda, _inputs((1, N), (2, 1, 2), d, d, dtype, N), state=state)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("dk,dv", [(20, 24), (30, 31), (61, 33), (72, 64), (101, 99), (129, 65),
                                   (160, 147), (250, 30)])
def test_long_heads(cuda, dtype, dk, dv):
    """Segments joined for heads that fill no tile, rows off 16 bytes, three heads."""
    state = torch.randn(1, 3, dk, dv, generator=torch.Generator().manual_seed(dk))
    x = _inputs((1, 1000), (3, 1, 3), dk, dv, dtype, dv)
    first, _ = _check(cuda, x, state=state)
    # the same bits from rows with other strides and addresses, others not finite around them
    def among(t):
        wide = torch.full((t.shape[0], t.shape[1] + 1, t.shape[2] + 1, t.shape[3] + 3), math.nan, dtype=t.dtype)
        wide[:, 1:, 1:, 1:-2] = t
        return wide.to(cuda)[:, 1:, 1:, 1:-2]
    y = [among(t) for t in x[:3]] + [t.to(cuda) for t in x[3:]]
    out = kernels.delta_attention(*y, state=state.to(cuda), return_state=False)
    if dk % 8 or dv % 8:
        assert torch.equal(out, first)
    else:
        assert bool(((out - first).abs() <= torch.finfo(dtype).eps * (first.abs() + 1)).all())


def test_long_packed(cuda):
    lens = [1, 2100, 0, 700, 64, 3]
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32)
    for dtype, d in ((F32, 32), (BF16, 128)):
        state = torch.randn(len(lens), 2, d, 40, generator=torch.Generator().manual_seed(6))
        _check(cuda, _inputs((sum(lens),), (2, 2, 2), d, 40, dtype, d), state=state, cu=cu)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_decays_and_betas(cuda, dtype):
    """No decay; -inf at some tokens; sums so low that their powers vanish next to
    slow ones; a past that grows; betas of 0, 1 and 2; both of q's type."""
    for d, N in ((32, 100), (128, 900)):
        q, k, v, beta, f = _inputs((1, N), (4, 4, 4), d, d, dtype, 8)
        state = torch.randn(1, 4, d, d, generator=torch.Generator().manual_seed(4))
        _check(cuda, (q, k, v, beta, None), state=state)
        f[0, ::37, 0] = -math.inf
        f[0, 3::41, 1] = -300.0
        f[0, :, 2] = 0.004
        f[0, 10::50, 3] = -20000.0
        beta[0, ::3] = 0.0
        beta[0, 1::3] = 1.0
        _check(cuda, (q, k, v, beta, f), state=state)
        _check(cuda, (q, k, v, (2 * beta).to(dtype), f.to(dtype)), state=state)


def test_powers_of_the_decays(cuda):
    """A state that only fades, asked channel by channel, and values written last,
    one key each: each number is one product with exp of a sum of log decays.

    Roundings in units of u = 2^-24 of it: the power of two 2 (an ulp), what its
    argument's rounding is put back with 1, the scale 1, the product with the state or
    with u 1; the state's fading 2 in each of at most 5 chunks before (a product with a
    sum of two floats), 2 more for 2^G' behind the last.  Products with a number of a
    single part, others zeros, lose none: 15 for outputs, 14 for a state that fades, 6
    for what the last chunk wrote."""
    N, H = 190, 8
    g = torch.Generator().manual_seed(11)
    rate = torch.tensor([0.01, 0.05, 0.07, 0.085, 0.1, 0.11, 0.2, 0.4])
    f = -rate * (0.5 + torch.rand(1, N, H, generator=g))
    f[0, 100:130, 0] = -1.3                  # a fall of 56 powers of two within a chunk
    fall = f[0].double().cumsum(0)
    for dtype, d in ((F32, 16), (F32, 128), (F16, 64), (BF16, 16), (BF16, 128)):
        state = torch.randn(1, H, d, d, generator=g)
        t = torch.arange(N)
        q = torch.zeros(1, N, H, d)
        q[0, t, :, t % d] = 1.0
        zero, v = torch.zeros_like(q), torch.randn(1, N, H, d, generator=g).to(dtype)
        q = q.to(dtype)
        out, left = kernels.delta_attention(*(x.to(cuda) for x in (q, zero.to(dtype), v, 0 * f, f)),
                                            scale=1.0, state=state.to(cuda))
        want = torch.exp(fall)[:, :, None] * state[0].double()[:, t % d].transpose(0, 1)
        _close(out[0], want, dtype, 15 * U32 * want.abs())
        want = torch.exp(fall[-1])[:, None, None] * state[0].double()
        _close(left[0], want, F32, 14 * U32 * want.abs())
        # sixteen of the last tokens write
        k, beta = zero.clone(), torch.zeros_like(f)
        wrote = torch.arange(N - 20, N - 4)
        k[0, wrote, :, wrote - wrote[0]] = 1.0
        beta[0, wrote] = 1.0
        _, left = kernels.delta_attention(*(x.to(cuda) for x in (q, k.to(dtype), v, beta, f)))
        want = torch.exp(fall[-1] - fall[wrote])[:, :, None] * v[0, wrote].double()
        _close(left[0, :, :16].transpose(0, 1), want, F32, 6 * U32 * want.abs())
        assert not bool(left[0, :, 16:].any())


def test_one_key(cuda):
    """Every token has the same key: the state holds the last value alone."""
    for dtype in (F32, F16, BF16):
        q, k, v, beta, _ = _inputs((1, 200), (2, 2, 2), 64, 64, dtype, 5)
        k = torch.zeros_like(k)
        k[..., 3] = 1.0
        out, left = _check(cuda, (q, k, v, torch.ones_like(beta), None), scale=1.0)
        # S = (v_1 - 0) + (v_2 - v_1) + ..: each chunk's sum and T's difference round
        # values of at most 2 max |v|, a depth of 72 of them
        off = (left[0, :, 3].cpu() - v[0, -1].float()).abs().max()
        assert float(off) <= 72 * U32 * 2 * float(v.abs().max())


def test_scale_and_plain_keys(cuda):
    """Keys of other lengths than one."""
    for dtype in (F32, F16, BF16):
        q, k, v, beta, f = _inputs((1, 150), (2, 2, 2), 64, 64, dtype, 7, unit=False)
        _check(cuda, (q, (0.3 * k).to(dtype), v, 0.2 * beta, f - 0.05), scale=-2.0)


def test_rest_rows(cuda):
    """Rows before, between and behind the sequences: zero in a new output,
    untouched in one given; offsets that are out of range or decrease."""
    x = [t.to(cuda) for t in _inputs((90,), (2, 2, 2), 32, 32, BF16, 5)]
    cu = torch.tensor([7, 20, 70], dtype=torch.int32, device=cuda)
    out, left = kernels.delta_attention(*x, cu_seqlens=cu)
    assert bool((out[:7] == 0).all()) and bool((out[70:] == 0).all())
    given = torch.full_like(out, 3.0)
    got, left2 = kernels.delta_attention(*x, cu_seqlens=cu, out=given)
    assert got.data_ptr() == given.data_ptr()
    assert bool((got[:7] == 3).all()) and bool((got[70:] == 3).all())
    assert torch.equal(got[7:70], out[7:70]) and torch.equal(left, left2)
    for i, (a, b) in enumerate(((7, 20), (20, 70))):
        o, s = kernels.delta_attention(*(t[None, a:b] for t in x))
        assert torch.equal(o[0], out[a:b]) and torch.equal(s[0], left[i])
    bad = torch.tensor([-5, 20, 10, 400], dtype=torch.int32, device=cuda)
    out, left = kernels.delta_attention(*x, cu_seqlens=bad)
    o, s = kernels.delta_attention(*(t[None, :20] for t in x))
    assert torch.equal(s[0], left[0]) and bool((left[1] == 0).all())
    o, s = kernels.delta_attention(*(t[None, 20:] for t in x))
    assert torch.equal(o[0], out[20:]) and torch.equal(s[0], left[2])


@pytest.mark.parametrize("dtype,H,d", [(BF16, 3, 64), (F16, 2, 13), (F32, 5, 32), (BF16, 2, 100)])
@pytest.mark.parametrize("cu", [[0, 100, 130], [20000, 20007], [3, 3], [5, 5] + [9] * 80 + [40, 30000],
                                [30000, 30000], [-4, 50000]])
def test_mostly_rest_rows(cuda, dtype, H, d, cu):
    """Few tokens in many rows: all others zero in a new output, on whatever memory,
    and none touched in one given."""
    N = 30000
    q, k, v, beta, f = (t.to(cuda) for t in _inputs((N,), (H, 1, H), d, d, dtype, 4, H=H))
    offsets = torch.tensor(cu, device=cuda)
    used = torch.full((N, H, d), 7.0, dtype=dtype, device=cuda)
    del used                                 # (its memory may be the output's)
    out = kernels.delta_attention(q, k, v, beta, f, cu_seqlens=offsets, return_state=False)
    first, end = max(cu[0], 0), min(max(cu), N)
    assert not bool(out[:first].any()) and not bool(out[end:].any())
    given = torch.full((N, H, d), 7.0, dtype=dtype, device=cuda)
    kernels.delta_attention(q, k, v, beta, f, cu_seqlens=offsets, return_state=False, out=given)
    assert torch.equal(given[first:end], out[first:end])
    assert bool((given[:first] == 7).all()) and bool((given[end:] == 7).all())
    if end > first:
        assert bool(out[first:end].any(2).any(1).all())


@pytest.mark.parametrize("B,N,H", [(3000, 9000, 2), (1025, 9000, 1), (130, 70000, 2)])
def test_many_sequences(cuda, B, N, H):
    """More sequences than one scan or one search takes, many empty, some offsets
    out of order: each as its definition (a call with it alone may split it in other
    places, which are other sums)."""
    g = torch.Generator().manual_seed(B)
    x = [t.to(cuda) for t in _inputs((N,), (H, 1, 1), 16, 16, F32, B, H=H)]
    cu = torch.randint(0, N + 1, (B + 1,), generator=g).sort()[0]
    cu[0], cu[-1] = 0, N
    want = cu.clone()
    cu[B // 2], cu[B // 3] = -7, 5                   # count as their predecessors
    want[B // 2], want[B // 3] = want[B // 2 - 1], want[B // 3 - 1]
    out, left = kernels.delta_attention(*x, cu_seqlens=cu.to(cuda))
    for b in [0, 1, 63, 64, 65, B // 3 - 1, B // 3, B // 2 - 1, B // 2, B - 2, B - 1]:
        i, j = int(want[b]), int(want[b + 1])
        a = [t[i:j].double().cpu() for t in x]
        o, s, bound, n = _definition(*a, 16 ** -0.5, None)
        depth = 72 * _solve_norm(a[1], a[3], a[4], H)
        _close(out[i:j], o, F32, depth * U32 * bound)
        _close(left[b], s, F32, (depth * U32 * n)[:, None, :])


@pytest.mark.parametrize("dtype,d", [(F32, 16), (BF16, 16), (BF16, 72)])
@pytest.mark.parametrize("packed", [False, True])
def test_workspace_of_many_short_sequences(cuda, dtype, d, packed):
    """Tens of thousands of prompts of no, one or a few tokens: each as its definition,
    in a workspace that is bound by the tokens."""
    g = torch.Generator().manual_seed(5)
    B, H, dv = 30000 if d < 32 else 12000, 8, 8
    if packed:
        lens = torch.randint(0, 3, (B,), generator=g)
        lens[7], lens[B // 2], lens[-1] = 90, 200, 65
        at = torch.cat([torch.zeros(1, dtype=torch.int64), lens.cumsum(0)]) + 3
        lead, given = (int(at[-1]) + 5,), at.clone()
        given[B // 3] = 0                    # counts as its predecessor
        at[B // 3] = at[B // 3 - 1]
    else:
        lead, given = (B, 2), None
    q, k, v, beta, f = _inputs(lead, (H, 1, H), d, dv, dtype, 3, H=H)
    state = torch.randn(B, H, d, dv, generator=g)
    x = [t.to(cuda) for t in (q, k, v, beta, f)]
    state_in = state.to(cuda)
    more = dict(state=state_in, cu_seqlens=None if given is None else given.to(cuda))
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    held = torch.cuda.memory_allocated()
    out, left = kernels.delta_attention(*x, **more)
    torch.cuda.synchronize()
    took = torch.cuda.max_memory_allocated() - held
    tokens = math.prod(lead)
    a_token = 300 if dtype == BF16 and d > 64 else 204
    took -= out.numel() * out.element_size() + left.numel() * 4 + 32 * (B + 1) + 4096
    assert took <= (1 << 30) + 3 * a_token * tokens * H
    if packed:
        assert not bool(out[:3].any()) and not bool(out[-5:].any())
    picks = [0, 1, 7, 8, B // 3 - 1, B // 3, B // 3 + 1, B // 2, B - 2, B - 1]
    picks += torch.randint(0, B, (40,), generator=g).tolist()
    for b in picks:
        i, j = (int(at[b]), int(at[b + 1])) if packed else (0, 2)
        a = [(t[i:j] if packed else t[b]).double() for t in (q, k, v, beta, f)]
        want, s, bound, n = _definition(*a, d ** -0.5, state[b].double())
        depth = 72 * _solve_norm(a[1], a[3], a[4], H)
        _close(out[i:j] if packed else out[b], want, dtype, depth * U32 * bound)
        _close(left[b], s, F32, (depth * U32 * n)[:, None, :])


def test_strides(cuda):
    """Heads of one fused projection, transposed and expanded ones, betas among
    other columns, an output among other columns, misaligned rows: the values of
    contiguous inputs."""
    g = torch.Generator().manual_seed(9)
    for dtype in (F32, BF16):
        for d, N in ((40, 70), (128, 70)):
            p = torch.randn(2, N, 8 * d + 8, generator=g).to(dtype).to(cuda)
            q = p[..., :4 * d].unflatten(2, (4, d))
            k = p[..., 4 * d:6 * d].unflatten(2, (2, d)) / d ** 0.5
            p[..., 4 * d:6 * d] = k.flatten(2)
            k = p[..., 4 * d:6 * d].unflatten(2, (2, d))
            v = p[..., 6 * d:8 * d].unflatten(2, (2, d))
            p[..., 8 * d:] = torch.sigmoid(p[..., 8 * d:].float()).to(dtype)
            beta, f = p[..., 8 * d:8 * d + 4], -p[..., 8 * d + 4:]
            want, s = kernels.delta_attention(q.contiguous(), k.contiguous(), v.contiguous(),
                                              beta.contiguous(), f.contiguous())
            wide = torch.full((2, N, 4, d + 10), 7.0, dtype=dtype, device=cuda)
            out, left = kernels.delta_attention(q, k, v, beta, f, out=wide[..., 3:d + 3])
            assert torch.equal(out, want) and torch.equal(left, s)
            assert bool((wide[..., :3] == 7).all()) and bool((wide[..., d + 3:] == 7).all())
            flat = torch.empty(q.numel() + 1, dtype=dtype, device=cuda)[1:].view(2, N, 4, d)
            flat.copy_(q)
            turned = q.transpose(1, 2).contiguous().transpose(1, 2)
            for other in (flat, turned):
                out, left = kernels.delta_attention(other, k, v, beta.transpose(0, 1).contiguous()
                                                    .transpose(0, 1), f)
                assert torch.equal(out, want) and torch.equal(left, s)
            one = beta[:, :1].expand(2, N, 4)
            want, s = kernels.delta_attention(q, k[:, :1].expand(2, N, 2, d).contiguous(), v,
                                              one.contiguous(), f)
            out, left = kernels.delta_attention(q, k[:, :1].expand(2, N, 2, d), v, one, f)
            assert torch.equal(out, want) and torch.equal(left, s)


@pytest.mark.parametrize("dtype,d", [(F32, 64), (F16, 64), (BF16, 64), (BF16, 128)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("which", ["q", "k", "v", "beta", "log_decay"])
def test_keeps_later_values_from_earlier_tokens(cuda, dtype, d, bad, which):
    """A value that is not finite in token 70 of sequence 0: the tokens before
    it, the other head and the other sequence have the bits that they have
    without it.  (A log decay of -inf is an ordinary one.)"""
    if which == "log_decay" and bad < 0:
        pytest.skip("an ordinary value")
    x = dict(zip(("q", "k", "v", "beta", "log_decay"),
                 (t.to(cuda) for t in _inputs((2, 140), (2, 2, 2), d, 64, dtype, 3))))
    want, left = kernels.delta_attention(*x.values())
    if which in "qkv":
        x[which][0, 70, 1, 5] = bad
    else:
        x[which][0, 70, 1] = bad
    out, s = kernels.delta_attention(*x.values())
    assert torch.equal(out[1], want[1]) and torch.equal(s[1], left[1])
    assert torch.equal(out[0, :, 0], want[0, :, 0]) and torch.equal(s[0, 0], left[0, 0])
    assert torch.equal(out[0, :70, 1], want[0, :70, 1])
    if which == "q":
        assert not bool(out[0, 70, 1].isfinite().any())
        assert torch.equal(out[0, 71:, 1], want[0, 71:, 1]) and torch.equal(s, left)
    elif which == "v":      # its column
        assert not bool(out[0, 70:, 1, 5].isfinite().any())
        assert not bool(s[0, 1, :, 5].isfinite().any())
        rest = [c for c in range(64) if c != 5]
        assert torch.equal(out[0, :, 1, rest], want[0, :, 1, rest])
        assert torch.equal(s[0, 1][:, rest], left[0, 1][:, rest])
    else:                   # everything from the token on
        assert not bool(out[0, 70:, 1].isfinite().any()) and not bool(s[0, 1].isfinite().any())


@pytest.mark.parametrize("dtype,d", [(F32, 32), (F32, 128), (BF16, 64), (BF16, 128), (BF16, 256)])
@pytest.mark.parametrize("what", ["keys", "chain", "long chain", "values"])
def test_overflow_does_not_reach_earlier_tokens(cuda, dtype, d, what):
    """Finite numbers whose correction is beyond fp32: a product of two keys, of
    corrections one after another, or the difference of two values of one key."""
    x = dict(zip(("q", "k", "v", "beta", "log_decay"),
                 (t.to(cuda) for t in _inputs((1, 150), (2, 2, 2), d, d, dtype, 3))))
    at = {"keys": (70, 75), "chain": (66, 72, 84), "long chain": (66, 84, 104), "values": (70, 75)}[what]
    end = at[-1]
    x["q"] *= 0.01
    x["k"][..., 5] = 0.0
    x["log_decay"].zero_()
    x["beta"][0, list(at)] = 1.0
    x["v"][0, at[0], 1] = 20.0
    if what == "values":
        x["k"][0, list(at), 1] = 0.0
        x["k"][0, list(at), 1, 5] = 1.0
        x["v"][0, at[0], 1, 7] = 2e38
        x["v"][0, end, 1, 7] = -3e38
    else:
        x["k"][0, list(at), 1, 5] = 3e19 if what == "keys" else 1e10
    want, _ = kernels.delta_attention(*(t[:, :end].contiguous() for t in x.values()))
    out, s = kernels.delta_attention(*x.values())
    assert bool(want.isfinite().all())
    assert torch.equal(out[:, :end], want)
    assert bool(out[0, :, 0].isfinite().all()) and bool(s[0, 0].isfinite().all())
    columns = [7] if what == "values" else list(range(d))
    assert not bool(out[0, end:, 1][:, columns].isfinite().any())
    rest = [c for c in range(d) if c not in columns]
    assert bool(out[0, :, 1, rest].isfinite().all()) and bool(s[0, 1][:, rest].isfinite().all())


def test_state_that_is_not_finite(cuda):
    """An infinity in a column of the state: the other columns keep their bits."""
    x = [t.to(cuda) for t in _inputs((1, 100), (2, 2, 2), 64, 64, BF16, 3)]
    state = torch.randn(1, 2, 64, 64, device=cuda)
    want, left = kernels.delta_attention(*x, state=state)
    state[0, 1, 7, 9] = math.inf
    out, s = kernels.delta_attention(*x, state=state)
    rest = [c for c in range(64) if c != 9]
    assert torch.equal(out[0, :, 0], want[0, :, 0]) and torch.equal(s[0, 0], left[0, 0])
    assert torch.equal(out[0, :, 1, rest], want[0, :, 1, rest])
    assert not bool(out[0, :, 1, 9].isfinite().any()) and not bool(s[0, 1, :, 9].isfinite().any())


def test_empty(cuda):
    def z(*s):
        return torch.zeros(s, device=cuda)
    out, s = kernels.delta_attention(z(0, 5, 2, 8), z(0, 5, 2, 8), z(0, 5, 2, 8), z(0, 5, 2), z(0, 5, 2))
    assert out.shape == (0, 5, 2, 8) and s.shape == (0, 2, 8, 8)
    first = torch.randn(3, 2, 8, 8, device=cuda)
    out, s = kernels.delta_attention(z(3, 0, 2, 8), z(3, 0, 2, 8), z(3, 0, 2, 8), z(3, 0, 2), state=first)
    assert out.shape == (3, 0, 2, 8) and torch.equal(s, first)
    out, s = kernels.delta_attention(z(4, 2, 8) + 1, z(4, 2, 8), z(4, 2, 8), z(4, 2),
                                     cu_seqlens=torch.zeros(1, dtype=torch.int32, device=cuda))
    assert bool((out == 0).all()) and s.shape == (0, 2, 8, 8)
    only = kernels.delta_attention(z(1, 4, 2, 8), z(1, 4, 2, 8), z(1, 4, 2, 8), z(1, 4, 2),
                                   return_state=False)
    assert isinstance(only, torch.Tensor) and only.shape == (1, 4, 2, 8)


# ---------------------------------------------------------------------------
# one token
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,heads,H,dk,dv", [
    (1, (1, 1, 1), 1, 1, 1), (1, (12, 12, 12), 12, 32, 32), (5, (4, 1, 2), 4, 64, 64),
    (3, (4, 2, 2), 4, 80, 72), (2, (2, 2, 2), 2, 33, 31), (70, (4, 2, 8), 8, 128, 128),
    (2, (2, 1, 1), 2, 256, 256), (2, (1, 1, 1), 2, 200, 300), (300, (2, 2, 2), 2, 240, 130)])
def test_step(cuda, dtype, rows, heads, H, dk, dv):
    q, k, v, beta, f = _inputs((rows,), heads, dk, dv, dtype, rows + dk, H=H)
    g = torch.Generator().manual_seed(7)
    pool = torch.randn(rows + 3, H, dk, dv, generator=g)
    slots = torch.randperm(rows + 3, generator=g)[:rows]
    for wide in (False, True):
        state = pool.to(cuda)
        b, d = (beta.to(dtype), f.to(dtype)) if wide else (beta, f)
        out = kernels.delta_attention_step(
            *(t.to(cuda) for t in (q, k, v, b, d)), state,
            slots=slots.to(torch.int64 if wide else torch.int32).to(cuda))
        out, state = out.cpu(), state.cpu()
        for i in range(0, rows, 1 + rows // 8):
            a = [t[i:i + 1].double() for t in (q, k, v, b, d)]
            want, s, bound, n = _definition(*a, dk ** -0.5, pool[slots[i]].double())
            # k^T S and q^T S: sums of dk terms each; (q . k) u
            _close(out[i:i + 1], want, dtype, (2 * dk + 8) * U32 * bound)
            _close(state[slots[i]], s, F32, ((dk + 8) * U32 * n)[:, None, :])
        rest = [i for i in range(rows + 3) if i not in slots.tolist()]
        assert torch.equal(state[rest], pool[rest])


def test_step_slots(cuda):
    """Padding rows, slots outside the pool, no slots, and rows of one slot as
    consecutive tokens."""
    x = [t.to(cuda) for t in _inputs((9,), (4, 2, 2), 64, 64, BF16, 1)]
    pool = torch.randn(4, 4, 64, 64, device=cuda)
    slots = torch.tensor([2, -1, 0, 2, 4, 1 << 30, 2, 0, -(1 << 31)], dtype=torch.int32, device=cuda)
    state = pool.clone()
    out = kernels.delta_attention_step(*x, state, slots=slots)
    want = pool.clone()
    for i, s in enumerate(slots.tolist()):
        if 0 <= s < 4:
            o = kernels.delta_attention_step(*(t[i:i + 1] for t in x), want[s:s + 1])
            assert torch.equal(o[0], out[i])
        else:
            assert bool((out[i] == 0).all())
    assert torch.equal(state, want)
    same = pool.clone()
    o = kernels.delta_attention_step(*(t[:4] for t in x), same)
    other = pool.clone()
    o2 = kernels.delta_attention_step(*(t[:4] for t in x), other, slots=torch.arange(4, device=cuda))
    assert torch.equal(o, o2) and torch.equal(same, other)


def test_step_without_decay(cuda):
    q, k, v, beta, f = (t.to(cuda) for t in _inputs((3,), (2, 2, 2), 32, 32, F32, 1))
    state = torch.randn(3, 2, 32, 32, device=cuda)
    a, b = state.clone(), state.clone()
    o = kernels.delta_attention_step(q, k, v, beta, None, a)
    assert torch.equal(o, kernels.delta_attention_step(q, k, v, beta, torch.zeros_like(f), b))
    assert torch.equal(a, b)


def test_step_many_rows(cuda):
    """More rows than a workgroup scans at once, every second one a repeat."""
    rows, slots = 700, torch.arange(700) // 2
    x = [t.to(cuda) for t in _inputs((rows,), (1, 1, 1), 16, 8, F32, 4)]
    pool = torch.randn(350, 1, 16, 8, device=cuda)
    state = pool.clone()
    out = kernels.delta_attention_step(*x, state, slots=slots.to(cuda))
    a = kernels.delta_attention_step(*(t[::2] for t in x), pool)
    b = kernels.delta_attention_step(*(t[1::2] for t in x), pool)
    assert torch.equal(out[::2], a) and torch.equal(out[1::2], b) and torch.equal(state, pool)


def test_step_strides(cuda):
    """States of one layer among others, heads of a fused projection, betas among
    other columns, an output among other columns, misaligned states."""
    p = torch.randn(5, 8 * 40 + 8, device=cuda).bfloat16()
    q, k, v = (t.unflatten(1, (-1, 40)) for t in (p[:, :160], p[:, 160:240], p[:, 240:320]))
    beta, f = p[:, 320:324], p[:, 324:].float().abs().neg()
    pool = torch.randn(6, 3, 4, 40, 40, device=cuda) * 0.1
    slots = torch.tensor([5, 0, 2, 1, 4], device=cuda)
    want_s = pool[:, 1].contiguous()
    want = kernels.delta_attention_step(q.contiguous(), k.contiguous(), v.contiguous(),
                                        beta.contiguous(), f, want_s, slots=slots)
    layers = pool.clone()
    wide = torch.full((5, 4, 50), 7.0, dtype=torch.bfloat16, device=cuda)
    out = kernels.delta_attention_step(q, k, v, beta, f, layers[:, 1], slots=slots,
                                       out=wide[..., 5:45])
    assert torch.equal(out, want) and torch.equal(layers[:, 1], want_s)
    assert torch.equal(layers[:, 0], pool[:, 0]) and torch.equal(layers[:, 2], pool[:, 2])
    assert bool((wide[..., :5] == 7).all()) and bool((wide[..., 45:] == 7).all())
    odd = torch.empty(6 * 4 * 40 * 40 + 1, device=cuda)[1:].view(6, 4, 40, 40)
    odd.copy_(pool[:, 1])
    out = kernels.delta_attention_step(q, k, v, beta, f, odd, slots=slots)
    # (single columns a thread: sums in another order)
    assert bool(((out.float() - want.float()).abs() <= 2.0 ** -7 * want.float().abs() + 1e-4).all())
    assert bool(((odd - want_s).abs() <= 1e-5 * (1 + want_s.abs())).all())


@pytest.mark.parametrize("more", [0, 70])
def test_packed_offsets_either_way(cuda, more):
    """Sequences few enough to be found without a launch, and the same ones with
    empty ones between them: the same rows and states, cut into segments or not,
    offsets that fall or lie outside among them."""
    for lens in ([5, 0, 64, 130], [900, 0, 1, 2500, 70, 0]):
        N = sum(lens)
        x = [t.to(cuda) for t in _inputs((N,), (2, 2, 2), 64, 64, BF16, 31)]
        cu = [0]
        for n in lens:
            cu.append(cu[-1] + n)
        odd = cu[:2] + [cu[1] - 3] + cu[2:-1] + [N + 1000]
        spread = cu[:2] + [cu[1]] * more + cu[2:] + [N] * more
        def run(o):
            return kernels.delta_attention(*x, cu_seqlens=torch.tensor(o, device=cuda))
        want, states = run(cu)
        got, left = run(odd)
        assert torch.equal(got, want)
        assert torch.equal(left[[0] + list(range(2, len(lens) + 1))], states) and not bool(left[1].any())
        got, left = run(spread)
        a = [b.double().cpu() for b in x]
        for i, n in enumerate(lens):
            rows = slice(cu[i], cu[i] + n)
            w, ws, bound, m = _definition(*(t[rows] for t in a), 64 ** -0.5, None) if n else (None,) * 4
            at = i if i < 1 else i + more
            if n == 0:
                assert not bool(left[at].any())
                continue
            depth = 72 * _solve_norm(a[1][rows], a[3][rows], a[4][rows], 2)
            for o, s in ((want, states[i]), (got, left[at])):
                _close(o[rows], w, BF16, depth * U32 * bound)
                _close(s, ws, F32, (depth * U32 * m)[:, None, :])


def test_pieces_join(cuda):
    """A prompt in pieces through the states, and the rest of it token by token:
    the whole prompt's output."""
    q, k, v, beta, f = x = [t.to(cuda) for t in _inputs((2, 301), (4, 2, 2), 64, 32, F32, 12)]
    want, last = kernels.delta_attention(*x)
    s, outs = None, []
    for a, b in ((0, 100), (100, 101), (101, 280)):
        o, s = kernels.delta_attention(*(t[:, a:b] for t in x), state=s)
        outs.append(o)
    for t in range(280, 301):
        outs.append(kernels.delta_attention_step(*(y[:, t] for y in x), s)[:, None])
    got = torch.cat(outs, 1)
    for b in range(2):
        a = [t[b].double().cpu() for t in x]
        w, ws, bound, n = _definition(*a, 64 ** -0.5, None)
        depth = 136 * _solve_norm(a[1], a[3], a[4], 4)     # (a step's sums: 2 x 64 + 8 deep)
        for o, left in ((want, last), (got, s)):
            _close(o[b], w, F32, depth * U32 * bound)
            _close(left[b], ws, F32, (depth * U32 * n)[:, None, :])


def test_a_layer_of_a_serving_batch(cuda):
    """Heads normalised and rotated, prompts, states into a pool, single tokens,
    as a serving program runs them: captured as a graph, replayed with other
    inputs, on another stream; every replay has the eager calls' bits."""
    g = torch.Generator().manual_seed(21)
    H, Hk, d, N = 4, 2, 64, 150
    freqs = kernels.rotary_freqs(32, device=cuda)
    pos = torch.arange(N, device=cuda)
    cu = torch.tensor([0, 40, 41, 150], dtype=torch.int32, device=cuda)
    slots = torch.tensor([3, 0, 4], device=cuda)
    unit = torch.full((d,), d ** -0.5, device=cuda)
    proj = torch.randn(N, (H + 2 * Hk) * d, generator=g).bfloat16().to(cuda)
    gate = torch.randn(N, 2 * H, generator=g).to(cuda)
    token, tgate = proj[:3].clone(), gate[:3].clone()

    def heads(p, pos):
        q = p[:, :H * d].unflatten(1, (H, d))
        k = p[:, H * d:(H + Hk) * d].unflatten(1, (Hk, d))
        q, k = kernels.qk_norm_rotary(q, k, pos, freqs, q_weight=unit, k_weight=unit)
        return q, k, p[:, (H + Hk) * d:].unflatten(1, (Hk, d))

    def layer(pool):
        beta, f = torch.sigmoid(gate[:, :H]), -torch.nn.functional.softplus(gate[:, H:])
        out, s = kernels.delta_attention(*heads(proj, pos), beta, f, cu_seqlens=cu)
        pool[slots] = s
        beta, f = torch.sigmoid(tgate[:, :H]), -torch.nn.functional.softplus(tgate[:, H:])
        return out, kernels.delta_attention_step(*heads(token, pos[:3] + N), beta, f, pool, slots=slots)

    pool = torch.zeros(5, H, d, d, device=cuda)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        layer(pool)
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, one = layer(pool)
    for i in range(4):
        proj.copy_(torch.randn(proj.shape, generator=g))
        gate.copy_(torch.randn(gate.shape, generator=g))
        token.copy_(torch.randn(token.shape, generator=g))
        eager = torch.zeros_like(pool)
        a, b = layer(eager)
        torch.cuda.synchronize()
        pool.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, a) and torch.equal(one, b) and torch.equal(pool, eager)


def test_two_streams(cuda):
    """Calls on two streams at once have workspaces of their own."""
    a = [t.to(cuda) for t in _inputs((1, 3000), (2, 2, 2), 128, 128, BF16, 1)]
    b = [t.to(cuda) for t in _inputs((1, 3000), (2, 2, 2), 128, 128, BF16, 2)]
    wa, wb = kernels.delta_attention(*a), kernels.delta_attention(*b)
    torch.cuda.synchronize()
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(3):
        with torch.cuda.stream(sa):
            ga = kernels.delta_attention(*a)
        with torch.cuda.stream(sb):
            gb = kernels.delta_attention(*b)
        got.append((ga, gb))
    torch.cuda.synchronize()
    for ga, gb in got:
        assert all(torch.equal(x, y) for x, y in zip(ga + gb, wa + wb))
