"""The dense products against their definitions in 64 bits.

Tolerances.  Inputs are exact in both.  A sum z of K products in fp32 is off by at
most its depth times u = 2^-24 of S = sum |x w| + |bias|: the products are taken in
runs (a lane's numbers, then steps, then splits), whose depths add up to at most
K / 4 + 64; roundings of random signs make a random walk, so six deviations of it,
6 sqrt(K + 64) u S.  (A product of 16-bit numbers is exact in fp32; one of fp32
numbers is rounded once, which the same allowance holds.)  The activations have
slopes of at most 1.2 and are evaluated to 8 u of |z| themselves, the residual's
and the gate's sums round once more.  The output is rounded to its type once: half
a unit, eps / 2 of its value, or of the smallest normal number below it.
"""
import math

import pytest
import torch

from catfuse_amd import kernels

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
U32 = 2.0 ** -24
ACTS = [None, "relu", "silu", "gelu", "gelu_tanh"]


def _act(z, kind):
    if kind == "relu":
        return z.clamp(min=0)
    if kind == "silu":
        return z * torch.sigmoid(z)
    if kind == "gelu":
        return z * torch.special.ndtr(z)
    if kind == "gelu_tanh":
        return z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
    return z


def _sum(x, w, b):
    """(z, its tolerance) in 64 bits on the GPU."""
    x, w = x.double(), w.double()
    z, s = x @ w.t(), x.abs() @ w.abs().t()
    if b is not None:
        z, s = z + b.double(), s + b.double().abs()
    return z, 6 * math.sqrt(x.shape[-1] + 64) * U32 * s


def _check(got, x, ws, bs, act, residual=None):
    z, tol = _sum(x, ws[0], bs[0])
    want = _act(z, act)
    tol = 1.2 * tol + 8 * U32 * z.abs()
    if len(ws) == 2:
        up, tup = _sum(x, ws[1], bs[1])
        tol = tol * (up.abs() + tup) + want.abs() * tup + 2 * U32 * (want * up).abs()
        want = want * up
    if residual is not None:
        want = want + residual.double()
        tol = tol + U32 * want.abs()
    i = torch.finfo(got.dtype)
    tol = tol + i.eps / 2 * (want.abs() + tol).clamp(min=i.smallest_normal)
    off = (got.double() - want).abs()
    assert got.shape == want.shape
    assert bool((off <= tol).all()), f"off by {off.max().item()}, {(off - tol).max().item()} over"


def _make(cuda, M, K, N, dtype, seed, gated=False, bias=None, residual=False):
    g = torch.Generator(device=cuda).manual_seed(seed)
    def normal(*shape):
        return torch.randn(shape, generator=g, device=cuda)
    x = normal(M, K).to(dtype)
    n = 2 if gated else 1
    ws = tuple((normal(N, K) * max(K, 1) ** -0.5).to(dtype) for _ in range(n))
    bs = tuple(None if bias is None else normal(N).to(bias) for _ in range(n))
    return x, ws, bs, normal(M, N).to(dtype) if residual else None


def _run(x, ws, bs, act, residual=None, **more):
    if len(ws) == 2:
        return kernels.gated_linear(x, *ws, bias_gate=bs[0], bias_up=bs[1], activation=act, **more)
    return kernels.linear(x, *ws, *bs, activation=act, residual=residual, **more)


# rows: the few-rows kernel's halves and ends, tiles' ends; odd, short and long widths
SHAPES = [(1, 1, 1), (1, 64, 16), (2, 7, 5), (3, 1000, 2731 // 8), (1, 4096, 100), (15, 33, 17),
          (16, 128, 48), (17, 96, 33), (31, 513, 65), (32, 512, 1000), (33, 64, 64), (33, 1, 3),
          (64, 100, 40), (65, 129, 130), (100, 2048, 72), (127, 8, 257), (129, 1000, 129),
          (300, 389, 301), (1000, 72, 8), (70, 5000, 66)]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("M,K,N", SHAPES)
@pytest.mark.parametrize("gated", [False, True])
def test_shapes(cuda, dtype, M, K, N, gated):
    act = ACTS[(M + K + N) % 5]
    bias = (None, F32, dtype)[(M + N) % 3]
    x, ws, bs, r = _make(cuda, M, K, N, dtype, M + K, gated, bias, residual=not gated and K % 2 == 0)
    _check(_run(x, ws, bs, act, r), x, ws, bs, act, r)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("M,K,N", [(2000, 600, 1100), (4100, 256, 2050), (513, 4096, 520),
                                   (4100, 328, 4200), (8200, 72, 2056)])
@pytest.mark.parametrize("gated", [False, True])
def test_large(cuda, dtype, M, K, N, gated):
    x, ws, bs, r = _make(cuda, M, K, N, dtype, M, gated, dtype, residual=not gated)
    _check(_run(x, ws, bs, "silu", r), x, ws, bs, "silu", r)


# more than half a tile of 128 x 128 a CU, with fewer steps than stages and with more,
# whole and not; few rows of many columns; long rows split in steps, the last shorter
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("M,K,N", [(1030, 64, 2100), (1100, 136, 2304), (1024, 320, 2048), (17000, 200, 24),
                                   (40, 72, 17000), (600, 201, 6000), (10, 264, 16500), (32, 1032, 6200),
                                   (24, 1029, 6200), (64, 4096, 200), (100, 4200, 160), (40, 1607, 200)])
@pytest.mark.parametrize("gated", [False, True])
def test_tiles(cuda, dtype, M, K, N, gated):
    x, ws, bs, r = _make(cuda, M, K, N, dtype, M, gated, dtype, residual=not gated)
    _check(_run(x, ws, bs, "gelu", r), x, ws, bs, "gelu", r)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("M,K,N", [(1100, 1101, 900), (50, 4101, 120), (300, 4100, 500), (1100, 2050, 2000)])
@pytest.mark.parametrize("gated", [False, True])
def test_rows_off_pieces(cuda, dtype, M, K, N, gated):
    """Rows that no 16 bytes divide, between others that are not finite."""
    x, ws, bs, r = _make(cuda, M, K, N, dtype, 7, gated, dtype, residual=not gated)
    def among(t):
        wide = torch.full((t.shape[0] + 2, t.shape[1] + 6), math.nan, dtype=dtype, device=cuda)
        wide[1:-1, 3:-3] = t
        return wide[1:-1, 3:-3]
    want = _run(x, ws, bs, "silu", r)
    _check(want, x, ws, bs, "silu", r)
    _check(_run(among(x), tuple(map(among, ws)), bs, "silu", r), x, ws, bs, "silu", r)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("M,N", [(1100, 900), (300, 2000)])
def test_one_operand_off_pieces(cuda, dtype, M, N):
    """x, w or the second w alone: the product of whole rows, to the bit where its
    tiles are the same ones."""
    K = 4096
    x, ws, bs, _ = _make(cuda, M, K, N, dtype, 8, True, F32)
    want = _run(x, ws, bs, "silu")
    _check(want, x, ws, bs, "silu")
    def off(t):
        wide = torch.full((t.shape[0], K + 5), math.inf, dtype=dtype, device=cuda)
        wide[:, 2:K + 2] = t
        return wide[:, 2:K + 2]
    assert torch.equal(_run(off(x), ws, bs, "silu"), want)
    assert torch.equal(_run(x, (off(ws[0]), ws[1]), bs, "silu"), want)
    assert torch.equal(_run(x, (ws[0], off(ws[1])), bs, "silu"), want)
    # whole rows from an address that is not: read as they lie
    flat = torch.empty(M * K + 1, dtype=dtype, device=cuda)
    y = flat[1:].view(M, K)
    y.copy_(x)
    _check(_run(y, ws, bs, "silu"), x, ws, bs, "silu")
    _check(_run(y, (off(ws[0]), ws[1]), bs, "silu"), x, ws, bs, "silu")


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("M", [1, 2, 16, 30])
@pytest.mark.parametrize("K", [1, 31, 33, 127, 1001])
def test_few_rows_inside_words(cuda, dtype, M, K):
    x, ws, bs, r = _make(cuda, M, K, 50, dtype, 9, False, dtype, residual=True)
    flat = torch.full((50 * K + 3,), math.nan, dtype=dtype, device=cuda)
    w = flat[1:50 * K + 1].view(50, K)
    w.copy_(ws[0])
    _check(_run(x, (w,), bs, None, r), x, ws, bs, None, r)
    _check(_run(x, ws, bs, None, r), x, ws, bs, None, r)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M", [5, 200])
def test_activations(cuda, act, M):
    """Over their whole range: sums from -200 to 200, and an infinity."""
    for dtype in (F32, BF16):
        x = torch.linspace(-200, 200, M * 64, device=cuda).view(M, 64)[:, :1].to(dtype)
        w = torch.linspace(-1, 1, 81, device=cuda)[:, None].to(dtype)
        _check(kernels.linear(x, w, activation=act), x, (w,), (None,), act)
        _check(kernels.gated_linear(x, w, w.flip(0).contiguous(), activation=act), x,
               (w, w.flip(0)), (None, None), act)
        x[1] = math.inf
        y = kernels.linear(x, w[1:2] + 2, activation=act)      # a positive weight
        assert bool((y[1] == math.inf).all()) and bool(y[[0, 2, 3]].isfinite().all())


@pytest.mark.parametrize("M", [20, 400])
def test_gelu_of_small_values(cuda, M):
    """fp32: relative to the result, also where it is nearly all cancelled.  Units of
    u = 2^-24: the reciprocal 2 (an ulp) and its argument 1, of which the tail has at
    most 1.3 times as much; the polynomial 3 (in a model of it, its fit among them);
    the power 4, products 3, the sum 1: 16."""
    x = torch.linspace(-12.5, 6, 40 * M, device=cuda).view(M, 40)[:, :1].contiguous()
    w = torch.ones(1, 1, device=cuda)
    for z in (x, x * 0.2, x.abs() * -1e-20):
        want = z.double() * torch.special.erfc(z.double() * -0.5 ** 0.5) / 2   # (1 + erf cancels)
        got = kernels.linear(z, w, activation="gelu").double()
        off = ((got - want).abs() / want.abs().clamp(min=2.0 ** -126)).max().item()
        assert off <= 16 * U32
    bad = torch.tensor([[math.nan], [math.inf], [-math.inf], [0.0]], device=cuda)
    y = kernels.linear(bad, w, activation="gelu")[:, 0]
    assert bool(y[0].isnan()) and y[1:].tolist() == [math.inf, 0.0, 0.0]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("M", [20, 400])
def test_sigmoids_of_small_values(cuda, dtype, M):
    """silu and gelu_tanh relative to the result, down to the smallest normal numbers.
    Units of u = 2^-24: the power 4, the sum 1, the reciprocal 2, products 2: 9; t of
    gelu_tanh is off by 3 u of itself, and the power by |t| times that.  For bf16 the
    power's argument is rounded, |t| u, and the output to half a unit."""
    w = torch.ones(1, 1, dtype=dtype, device=cuda)
    for act, low in (("silu", -88.5), ("gelu_tanh", -9.5)):
        z = torch.linspace(low, 3, 40 * M, device=cuda).view(M, 40)[:, :1].to(dtype)
        x = z.double()
        t = x if act == "silu" else 2 * math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3)
        want = x / (1 + torch.exp(-t))
        got = kernels.linear(z.contiguous(), w, activation=act).double()
        tol = (9 + 4 * t.abs() * ((act != "silu") + (dtype != F32))) * U32 * want.abs()
        i = torch.finfo(dtype)
        tol = tol + (i.eps / 2 * want.abs() if dtype != F32 else 0)
        ok = want.abs() >= i.smallest_normal
        assert int(ok.sum()) > 0.9 * M
        assert bool(((got - want).abs() <= tol)[ok].all())


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("M", [1, 20, 150])
def test_strides(cuda, dtype, M):
    """Rows of wider ones, misaligned, broadcast and overlapping rows, columns of
    one buffer beside each other: the bits of contiguous inputs, or (rows that
    cannot be copied in whole pieces take another path of the same sums) of them."""
    K, N = 160, 72
    x, (w,), (b,), r = _make(cuda, M, K, N, dtype, 3, bias=F32, residual=True)
    want = kernels.linear(x, w, b, residual=r)
    wide = torch.randn(M, K + N + 2 * N + 5, device=cuda).to(dtype)
    for off in (0, 3, 8):
        xs = wide[:, off:off + K]
        xs.copy_(x)
        ws = torch.empty(N, K + 24, dtype=dtype, device=cuda)[:, off:off + K]
        ws.copy_(w)
        assert torch.equal(kernels.linear(xs, ws, b, residual=r), want)
        out = wide[:, K + 8:K + 8 + N]
        rs = wide[:, K + 8 + N:K + 8 + 2 * N] if M > 1 else r
        rs.copy_(r)
        keep = wide.clone()
        got = kernels.linear(xs, ws, b, residual=rs, out=out)
        assert got.data_ptr() == out.data_ptr() and torch.equal(out, want)
        keep[:, K + 8:K + 8 + N] = out
        assert torch.equal(wide, keep)
    one = x[:1].expand(M, K)
    assert torch.equal(kernels.linear(one, w, b), kernels.linear(one.contiguous(), w, b))
    rolling = x.flatten().as_strided((M, 8), (1, 1))
    w8 = w[:, :8]
    assert torch.equal(kernels.linear(rolling, w8), kernels.linear(rolling.contiguous(), w8.contiguous()))
    assert torch.equal(kernels.linear(x, w, residual=r[:1].expand(M, N)),
                       kernels.linear(x, w, residual=r[:1].repeat(M, 1)))
    x4 = x.view(1, M, 1, K)
    assert torch.equal(kernels.linear(x4, w, b, residual=r.view(1, M, 1, N)).view(M, N), want)
    if M == 1:
        assert torch.equal(kernels.linear(x[0], w, b, residual=r[0]), want[0])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("M,K", [(7, 200), (150, 200), (150, 4096)])
def test_in_place_residual(cuda, dtype, M, K):
    x, (w,), _, r = _make(cuda, M, K, 130, dtype, 4, residual=True)
    want = kernels.linear(x, w, residual=r)
    version = r._version
    got = kernels.linear(x, w, residual=r, out=r)
    assert got is r and torch.equal(r, want) and r._version > version


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("M,K", [(9, 100), (90, 101), (90, 4096), (260, 128)])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_values_that_are_not_finite(cuda, dtype, M, K, bad):
    """In x they reach their row, in w their column, the inner dimension's end and
    rows and columns that pad a tile none."""
    x, (w,), _, _ = _make(cuda, M, K, 70, dtype, 5)
    want = kernels.linear(x, w)
    y = x.clone()
    y[M // 2, K - 1] = bad
    got = kernels.linear(y, w)
    rest = [i for i in range(M) if i != M // 2]
    assert torch.equal(got[rest], want[rest]) and not bool(got[M // 2].isfinite().any())
    w2 = w.clone()
    w2[69, K - 1] = bad
    got = kernels.linear(x, w2)
    assert torch.equal(got[:, :69], want[:, :69]) and not bool(got[:, 69].isfinite().any())
    # behind the last column and the last row
    wide = torch.full((M + 1, K + 8), bad, dtype=dtype, device=cuda)
    wide[:M, :K] = x
    ww = torch.full((71, K + 8), bad, dtype=dtype, device=cuda)
    ww[:70, :K] = w
    assert torch.equal(kernels.linear(wide[:M, :K], ww[:70, :K]), want)


def test_empty(cuda):
    def z(*s):
        return torch.zeros(s, device=cuda)
    assert kernels.linear(z(0, 5), z(7, 5)).shape == (0, 7)
    assert kernels.linear(z(3, 0, 5), z(7, 5)).shape == (3, 0, 7)
    b = torch.arange(7.0, device=cuda)
    for M in (2, 100):                               # an empty sum
        out = kernels.linear(z(M, 0), z(7, 0), b, activation="relu", residual=z(M, 7) + 1)
        assert torch.equal(out, (b + 1).expand(M, 7))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("M", [3, 40, 300])
def test_gated_without_an_inner_dimension(cuda, dtype, M):
    """Empty sums on both sides: the activated bias times the other."""
    def z(*s):
        return torch.zeros(s, dtype=dtype, device=cuda)
    bg, bu = torch.linspace(-2, 2, 40, device=cuda), torch.linspace(3, -1, 40, device=cuda)
    for act in ACTS:
        got = kernels.gated_linear(z(M, 0), z(40, 0), z(40, 0), bias_gate=bg, bias_up=bu, activation=act)
        _check(got, z(M, 0), (z(40, 0), z(40, 0)), (bg, bu), act)
        assert not bool(kernels.gated_linear(z(M, 0), z(40, 0), z(40, 0), bias_gate=bg,
                                             activation=act).any())


def test_more_than_32_bits(cuda):
    """An x and an output of more than 2^31 elements, rows more than 2^31 apart."""
    K, N = 64, 96
    M = (1 << 31) // K + 300
    g = torch.Generator(device=cuda).manual_seed(1)
    x = torch.empty(M, K, dtype=BF16, device=cuda)
    pick = torch.tensor([0, 1, 77, M // 2, (1 << 30) // K, M - 300, M - 2, M - 1], device=cuda)
    x.zero_()
    x[pick] = torch.randn(len(pick), K, generator=g, device=cuda).to(BF16)
    w = torch.randn(N, K, generator=g, device=cuda).to(BF16)
    out = kernels.linear(x, w)
    _check(out[pick], x[pick], (w,), (None,), None)
    assert int((out != 0).any(1).sum()) == len(pick)
    del out
    far = x.view(-1).as_strided((3, K), ((1 << 30) - 64, 1))
    _check(kernels.linear(far, w), far.contiguous(), (w,), (None,), None)
    rows = x.view(-1).as_strided((70, K), (30_000_000, 1))
    _check(kernels.linear(rows, w), rows.contiguous(), (w,), (None,), None)


def test_more_tiles_than_a_launch_takes(cuda):
    """Rows of one number and columns that just begin a second tile: 8.4 million tiles
    of 512 threads and more."""
    M, N = 540_000_001, 65
    x = torch.zeros(M, 1, dtype=BF16, device=cuda)
    pick = torch.tensor([0, 1, 129, M // 3, M // 2, 536_870_911, 536_870_912, M - 130, M - 1], device=cuda)
    x[pick, 0] = torch.arange(1, len(pick) + 1, device=cuda).to(BF16)
    g = torch.Generator(device=cuda).manual_seed(1)
    w, w2 = (torch.randn(N, 1, generator=g, device=cuda).to(BF16) for _ in range(2))
    out = kernels.gated_linear(x, w, w2)
    _check(out[pick], x[pick], (w, w2), (None, None), "silu")
    some = torch.arange(0, M, 10007, device=cuda)
    some = some[~torch.isin(some, pick)]
    assert not bool(out[some].any())
    del out, x, some
    torch.cuda.empty_cache()


def test_rows_too_long_to_lie_near(cuda):
    """256 rows reach over 2^31 bytes, and no 16 bytes divide one."""
    M, K, N = 40, 4_200_001, 24
    g = torch.Generator(device=cuda).manual_seed(3)
    x = torch.randn(M, K, generator=g, device=cuda).to(BF16)
    w = torch.randn(N, K, generator=g, device=cuda).to(BF16)
    _check(kernels.linear(x, w), x, (w,), (None,), None)


def test_a_block_of_a_serving_batch(cuda):
    """The projections around the delta rule's attention and its feed-forward
    block, as a serving program runs them: prompts, then single tokens; captured as
    a graph and replayed with other inputs.  Every replay has the eager calls'
    bits."""
    g = torch.Generator().manual_seed(2)
    D, H, Hk, d, F = 256, 4, 2, 64, 700
    def weight(n, k):
        return (torch.randn(n, k, generator=g) * k ** -0.5).bfloat16().to(cuda)
    w_in, w_gates, w_out = weight((H + 2 * Hk) * d, D), weight(2 * H, D), weight(D, H * d)
    w_gate, w_up, w_down = weight(F, D), weight(F, D), weight(D, F)
    freqs = kernels.rotary_freqs(d // 2, device=cuda)
    unit = torch.full((d,), d ** -0.5, device=cuda)

    def block(x, pos, attend):
        p, gates = kernels.linear(x, w_in), kernels.linear(x, w_gates)
        q = p[:, :H * d].unflatten(1, (H, d))
        k = p[:, H * d:(H + Hk) * d].unflatten(1, (Hk, d))
        q, k = kernels.qk_norm_rotary(q, k, pos, freqs, q_weight=unit, k_weight=unit)
        v = p[:, (H + Hk) * d:].unflatten(1, (Hk, d))
        beta, f = torch.sigmoid(gates[:, :H]), -torch.nn.functional.softplus(gates[:, H:].float())
        o = attend(q, k, v, beta, f)
        x = kernels.linear(o.flatten(1), w_out, residual=x)
        return kernels.linear(kernels.gated_linear(x, w_gate, w_up), w_down, residual=x)

    cu = torch.tensor([0, 30, 31, 130], dtype=torch.int32, device=cuda)
    slots = torch.tensor([2, 0, 3], device=cuda)
    prompt, token = torch.randn(130, D, generator=g).bfloat16().to(cuda), \
        torch.randn(3, D, generator=g).bfloat16().to(cuda)
    pos = torch.arange(130, device=cuda)

    def program(pool):
        def prompts(*a):
            o, s = kernels.delta_attention(*a, cu_seqlens=cu)
            pool[slots] = s
            return o
        a = block(prompt, pos, prompts)
        return a, block(token, pos[:3], lambda *t: kernels.delta_attention_step(*t, pool, slots=slots))

    pool = torch.zeros(5, H, d, d, device=cuda)
    program(pool)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = program(pool)
    for _ in range(3):
        prompt.copy_(torch.randn(130, D, generator=g))
        token.copy_(torch.randn(3, D, generator=g))
        eager = torch.zeros_like(pool)
        want = program(eager)
        torch.cuda.synchronize()
        pool.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want)) and torch.equal(pool, eager)
        # the first block's parts against the same formulas in 64 bits
        p = kernels.linear(prompt, w_in)
        _check(p, prompt, (w_in,), (None,), None)
        h = kernels.gated_linear(prompt, w_gate, w_up)
        _check(h, prompt, (w_gate, w_up), (None, None), "silu")
        _check(kernels.linear(h, w_down, residual=prompt), h, (w_down,), (None,), None, prompt)
