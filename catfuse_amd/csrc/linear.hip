// Dense products with an epilogue:
//   out = act(x w^T + bias) + residual                     (linear)
//   out = act(x w^T + bias) * (x w2^T + bias2)             (gated)
// x [rows][inner], w and w2 [cols][inner], out [rows][cols]; fp32, fp16 or bf16
// with fp32 sums, each output rounded once.
//
// Both operands lie with the inner dimension on end, which is how the matrix
// cores' operands want them: a lane takes 16 bytes of one row.  Products of
// fp32 numbers run on the fp32 matrix instructions (their products and sums, an
// infinity stays one), those of 16-bit ones on theirs.
//
// No counterpart in the reference.
#include "cf_seq.h"

namespace {

struct LinearArgs {
  const void* x;
  const void* w[2];
  const void* bias[2];
  const void* residual;
  void* out;
  float* parts;              // sums of the splits [split][product][rows][cols], or null
  int bias_f32, activation;
  int64_t rows;
  int inner, cols;
  int64_t xr, wr[2], rr, orow;
  int splits, split_steps;   // along the inner dimension; steps of a split
  int row_tiles, col_tiles;
};

typedef float f4v __attribute__((ext_vector_type(4)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));

// Products of 16 bytes of a row of either operand (`a`: rows of the result,
// `b`: its columns): 8 numbers of 16 bits, or 4 of 32 taken one at a time (the
// same ones of both operands, in whatever order).
template <typename T>
__device__ __forceinline__ f4v mfma(u32x4 a, u32x4 b, f4v c) {
  if constexpr (sizeof(T) == 4) {
    const f4v x = __builtin_bit_cast(f4v, a), y = __builtin_bit_cast(f4v, b);
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[j], y[j], c, 0, 0, 0);
    return c;
  } else if constexpr (__is_same(T, bf16_t)) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, a),
                                                   __builtin_bit_cast(bf8, b), c, 0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a),
                                                  __builtin_bit_cast(h8, b), c, 0, 0, 0);
  }
}

// 16 bytes from wherever they begin (a multiple of the type's size).
template <typename T>
__device__ __forceinline__ u32x4 load16(const T* p) {
  u32x4 r;
  __builtin_memcpy(&r, p, 16);
  return r;
}
// The same, read by words: of 16 bits where they may begin inside one, the five they
// lie in (the fifth only where it holds some of them).
struct Words { u32x4 w; uint32_t rest, shift; };
template <typename T>
__device__ __forceinline__ Words words_at(const T* p) {
  const char* const a = (const char*)((uintptr_t)p & ~(uintptr_t)3);
  Words r;
  r.shift = (uint32_t)((uintptr_t)p & 2);
  r.w = load16(reinterpret_cast<const uint32_t*>(a));
  r.rest = *reinterpret_cast<const uint32_t*>(a + (r.shift ? 16 : 12));
  return r;
}
__device__ __forceinline__ u32x4 whole_of(const Words& r) {
  u32x4 x;
#pragma unroll
  for (int j = 0; j < 4; ++j) x[j] = __builtin_amdgcn_alignbyte(j < 3 ? r.w[j + 1] : r.rest, r.w[j], r.shift);
  return x;
}
__device__ __forceinline__ u32x4 whole_of(const u32x4& x) { return x; }
// The first n of the numbers there, zeros behind.
template <typename T>
__device__ __forceinline__ u32x4 load_some(const T* p, int n) {
  constexpr int PER = 16 / sizeof(T);
  if (n >= PER) return load16(p);
  Vec<T, PER> v;
#pragma unroll
  for (int i = 0; i < PER; ++i) v.v[i] = i < n ? p[i] : from_f<T>(0.0f);
  return __builtin_bit_cast(u32x4, v);
}

// e^x to about an ulp: the rounding of x log2(e) is put back.
__device__ __forceinline__ float exp_f(float x) {
  const float y = x * 1.44269502f;
  const float low = __builtin_fmaf(x, 1.44269502f, -y) + x * 1.92596299e-8f;
  const float e = __builtin_amdgcn_exp2f(y);
  // (an infinite or vanished power stays one)
  return __builtin_fabsf(y) < 127.9f ? __builtin_fmaf(e, low * 0.693147182f, e) : e;
}
// z / (1 + e^-t).  For outputs of 16 bits the power of two alone will do: rounding its
// argument moves it, and so the result, by |t| 2^-24 of itself, 5e-6 where fp32 ends;
// the output is then rounded by 2.4e-4 of itself (fp16) or more.
template <typename T>
__device__ __forceinline__ float sigmoid_times(float z, float t) {
  const float e = sizeof(T) == 4 ? exp_f(-t) : __builtin_amdgcn_exp2f(t * -1.44269502f);
  if (__is_same(T, _Float16)) return z * __builtin_amdgcn_rcpf(1.0f + e);
  // (the reciprocal of what is beyond 2^126 would be lost, z times it not: t to -88)
  const float s = e > 0x1p64f ? 0x1p-64f : 1.0f;
  return (z * s) * __builtin_amdgcn_rcpf(__builtin_fmaf(e, s, s));
}
// x (1 + erf(x / sqrt(2))) / 2 = max(x, 0) - |x| Q(|x|), Q(y) = (1 - erf(y / sqrt(2))) / 2.
template <typename T>
__device__ __forceinline__ float gelu(float x) {
  const float a = __builtin_fabsf(x);
  if constexpr (sizeof(T) == 4) {
    // Q(y) e^(y^2 / 2) as a polynomial in 1 / (1 + 0.345 y), fitted here to 2.4e-8 of
    // itself from 0 to 14.5 (least squares, weights by the errors until they are even);
    // what rounding y^2 loses is put into the power.  To 16 x 2^-24 of the result,
    // however small (5 measured); 4000 x 384 x 1536 takes 59.0 us with it, 55.6 with
    // the formula below.  Beyond 20 Q is none (a NaN stays).
    const float y = a > 20.0f ? 20.0f : a, t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.345f, y, 1.0f));
    float p = __builtin_fmaf(-0.0281517822f, t, 0.14423351f);
    p = __builtin_fmaf(p, t, -0.269153401f);
    p = __builtin_fmaf(p, t, 0.185054465f);
    p = __builtin_fmaf(p, t, -0.0362378173f);
    p = __builtin_fmaf(p, t, 0.111267676f);
    p = __builtin_fmaf(p, t, 0.117362f);
    p = __builtin_fmaf(p, t, 0.138005239f);
    p = __builtin_fmaf(p, t, 0.137620113f) * t;
    const float s = y * y, low = __builtin_fmaf(y, y, -s);
    const float e = exp_f(-0.5f * s);
    return __builtin_fmaf(-y, p * __builtin_fmaf(e, -0.5f * low, e), __builtin_fmaxf(x, 0.0f));
  }
  // For 16 bits Q by Abramowitz and Stegun's formula 7.1.26, to 2.6e-7 of one: 1e-4 of
  // the result at -3, 1e-3 at -4, which is what rounding 1 + erf to fp32 leaves there.
  const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.231641888f, a, 1.0f));
  float p = __builtin_fmaf(0.530702715f, t, -0.726576014f);
  p = __builtin_fmaf(p, t, 0.710706871f);
  p = __builtin_fmaf(p, t, -0.142248368f);
  p = __builtin_fmaf(p, t, 0.127414796f) * t;
  const float tail = p * __builtin_amdgcn_exp2f(x * x * -0.721347520f);
  // (beyond 20 the tail is none, and infinity takes none of it)
  return __builtin_fmaf(-__builtin_fminf(a, 20.0f), tail, __builtin_fmaxf(x, 0.0f));
}
template <typename T, int N>
__device__ __forceinline__ void activate(float* z, int kind) {
  if (kind == CF_ACT_RELU) {
#pragma unroll
    for (int j = 0; j < N; ++j) z[j] = z[j] < 0.0f ? 0.0f : z[j];
  } else if (kind == CF_ACT_SILU) {
#pragma unroll
    for (int j = 0; j < N; ++j) z[j] = sigmoid_times<T>(z[j], z[j]);
  } else if (kind == CF_ACT_GELU) {
#pragma unroll
    for (int j = 0; j < N; ++j) z[j] = gelu<T>(z[j]);
  } else if (kind == CF_ACT_GELU_TANH) {     // 1 + tanh(t) = 2 / (1 + e^(-2 t))
#pragma unroll
    for (int j = 0; j < N; ++j)
      z[j] = sigmoid_times<T>(z[j], z[j] * __builtin_fmaf(0.0713548163f * z[j], z[j], 1.59576912f));
  }
}

template <typename T>
__device__ __forceinline__ float bias_of(const LinearArgs& a, int op, int n) {
  if (a.bias[op] == nullptr) return 0.0f;
  return a.bias_f32 ? reinterpret_cast<const float*>(a.bias[op])[n]
                    : to_f(reinterpret_cast<const T*>(a.bias[op])[n]);
}

// Outputs of a row, columns n .. n + 7 (COUNT of them), from the sums and the
// biases of each product; those from cols on are left alone.  wide: eight on end,
// from a multiple of eight, are aligned and whole.  given: the residual, if the
// caller has it.
template <typename T, int OPS, int COUNT>
__device__ __forceinline__ void finish(const LinearArgs& a, int64_t m, int n, const float (*s)[COUNT],
                                       const float (*b)[COUNT], const Vec<T, COUNT>& given, bool have, bool wide) {
  float y[COUNT], r[COUNT];
  constexpr int PER = COUNT * sizeof(T) > 16 ? 16 / sizeof(T) : COUNT;   // of an access
  T* const to = (T*)a.out + m * a.orow + n;
#pragma unroll
  for (int j = 0; j < COUNT; ++j) r[j] = 0.0f;
  if (OPS == 1 && a.residual != nullptr) {
    const T* const from = (const T*)a.residual + m * a.rr + n;
    if (have) {
#pragma unroll
      for (int j = 0; j < COUNT; ++j) r[j] = to_f(given.v[j]);
    } else if (wide) {
#pragma unroll
      for (int i = 0; i < COUNT; i += PER) {
        const Vec<T, PER> v = *reinterpret_cast<const Vec<T, PER>*>(from + i);
#pragma unroll
        for (int j = 0; j < PER; ++j) r[i + j] = to_f(v.v[j]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < COUNT; ++j)
        if (n + j < a.cols) r[j] = to_f(from[j]);
    }
  }
#pragma unroll
  for (int j = 0; j < COUNT; ++j) y[j] = s[0][j] + b[0][j];
  activate<T, COUNT>(y, a.activation);
  if constexpr (OPS == 2) {
#pragma unroll
    for (int j = 0; j < COUNT; ++j) y[j] *= s[1][j] + b[1][j];
  } else if (a.residual != nullptr) {
#pragma unroll
    for (int j = 0; j < COUNT; ++j) y[j] += r[j];
  }
  if (wide) {
#pragma unroll
    for (int i = 0; i < COUNT; i += PER) {
      Vec<T, PER> v;
#pragma unroll
      for (int j = 0; j < PER; ++j) v.v[j] = from_f<T>(y[i + j]);
      *reinterpret_cast<Vec<T, PER>*>(to + i) = v;
    }
  } else {
#pragma unroll
    for (int j = 0; j < COUNT; ++j)
      if (n + j < a.cols) to[j] = from_f<T>(y[j]);
  }
}

// The same of eight, or the sums themselves to the workspace.
template <typename T, int OPS>
__device__ __forceinline__ void finish8(const LinearArgs& a, int64_t m, int n, int split,
                                        const float (*s)[8], const float (*b)[8],
                                        const Vec<T, 8>& given, bool have, bool wide) {
  if (a.parts == nullptr) {
    finish<T, OPS, 8>(a, m, n, s, b, given, have, wide);
    return;
  }
#pragma unroll
  for (int o = 0; o < OPS; ++o) {
    float* const to = a.parts + (((int64_t)split * OPS + o) * a.rows + m) * a.cols + n;
    if (a.cols % 8 == 0) {
#pragma unroll
      for (int e = 0; e < 8; e += 4) {
        const Vec<float, 4> v = {s[o][e], s[o][e + 1], s[o][e + 2], s[o][e + 3]};
        *reinterpret_cast<Vec<float, 4>*>(to + e) = v;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (n + e < a.cols) to[e] = s[o][e];
    }
  }
}

// Whether eight columns on end, from a multiple of eight, are aligned (to 16
// bytes; four of 16 bits to 8) and whole.
template <typename T>
__device__ __forceinline__ bool wide_columns(const LinearArgs& a) {
  constexpr int PER = 16 / sizeof(T);
  return a.cols % 8 == 0 && a.orow % PER == 0 && ((uintptr_t)a.out & 15) == 0 &&
         (a.residual == nullptr || (a.rr % PER == 0 && ((uintptr_t)a.residual & 15) == 0));
}

// Few rows of x: bound by the bytes of w, each read once.  A workgroup takes 16
// columns (rows of w) and all rows of x, eight waves a part of the inner dimension
// each, joined in LDS (four took as long within 2 %, however many columns).  A lane of
// a product takes 16 bytes of w's row lane % 16, piece lane / 16 of four; U products'
// loads are in flight.  1 row of 4096 x 4096 and its residual: 8.9 us, 3.8 TB/s.
// ODD: rows of 16 bits that begin inside a word, read as the five words they lie in
// (6 gated rows of 2233 x 4821: 19 us; as 16 bytes from their own address 31, of 2232
// 14).
template <typename T, int MT, int OPS, bool ODD>
__global__ __launch_bounds__(512) void linear_few_kernel(LinearArgs a) {
  constexpr int NW = 8, PER = 16 / sizeof(T), STEP = 4 * PER, U = MT * OPS <= 2 && !ODD ? 8 : 4;
  __shared__ float part[NW][OPS * MT][4][64];
  const int tid = threadIdx.x, lane = tid & 63, row = lane & 15, quarter = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n0 = blockIdx.x * 16;
  const int steps = (a.inner + STEP - 1) / STEP, each = (steps + NW - 1) / NW;
  const int first = wave * each, whole = a.inner / STEP;
  const int last = first + each < steps ? first + each : steps;
  const T *wp[OPS], *xp[MT];
#pragma unroll
  for (int o = 0; o < OPS; ++o)
    wp[o] = (const T*)a.w[o] + (n0 + row < a.cols ? n0 + row : a.cols - 1) * a.wr[o] + quarter * PER;
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    const int64_t m = 16 * t + row;
    xp[t] = (const T*)a.x + (m < a.rows ? m : a.rows - 1) * a.xr + quarter * PER;
  }
  f4v acc[OPS][MT];
#pragma unroll
  for (int o = 0; o < OPS; ++o)
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[o][t] = f4v{};
  const int full = last < whole ? last : whole;
  auto take = [](const T* p) {
    if constexpr (ODD) return words_at(p);
    else return load16(p);
  };
  using Piece = decltype(take(nullptr));
  for (int s = first; s < full; s += U) {    // (conditions on s: the same in every lane)
    Piece wv[U][OPS], xv[U][MT];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (s + u < full) {
#pragma unroll
        for (int o = 0; o < OPS; ++o) wv[u][o] = take(wp[o] + (int64_t)(s + u) * STEP);
#pragma unroll
        for (int t = 0; t < MT; ++t) xv[u][t] = take(xp[t] + (int64_t)(s + u) * STEP);
      }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (s + u < full)
#pragma unroll
        for (int o = 0; o < OPS; ++o)
#pragma unroll
          for (int t = 0; t < MT; ++t) acc[o][t] = mfma<T>(whole_of(wv[u][o]), whole_of(xv[u][t]), acc[o][t]);
  }
  if (first <= whole && last > whole) {       // the inner dimension's end: zeros behind it
    const int left = a.inner - whole * STEP - quarter * PER;
    u32x4 wv[OPS], xv[MT];
#pragma unroll
    for (int o = 0; o < OPS; ++o) wv[o] = load_some(wp[o] + (int64_t)whole * STEP, left);
#pragma unroll
    for (int t = 0; t < MT; ++t) xv[t] = load_some(xp[t] + (int64_t)whole * STEP, left);
#pragma unroll
    for (int o = 0; o < OPS; ++o)
#pragma unroll
      for (int t = 0; t < MT; ++t) acc[o][t] = mfma<T>(wv[o], xv[t], acc[o][t]);
  }
#pragma unroll
  for (int o = 0; o < OPS; ++o)
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int j = 0; j < 4; ++j) part[wave][o * MT + t][j][lane] = acc[o][t][j];
  __syncthreads();
  const bool wide = wide_columns<T>(a);
  for (int t = wave; t < MT; t += NW) {
    float y[OPS][4];
#pragma unroll
    for (int o = 0; o < OPS; ++o)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float z = 0.0f;
#pragma unroll
        for (int i = 0; i < NW; ++i) z += part[i][o * MT + t][j][lane];
        y[o][j] = z;
      }
    const int64_t m = 16 * t + row;
    const int n = n0 + 4 * quarter;
    if (m < a.rows && n < a.cols) {
      float b[OPS][4];
#pragma unroll
      for (int o = 0; o < OPS; ++o)
#pragma unroll
        for (int j = 0; j < 4; ++j) b[o][j] = bias_of<T>(a, o, n + j < a.cols ? n + j : a.cols - 1);
      finish<T, OPS, 4>(a, m, n, y, b, {}, false, wide);
    }
  }
}

template <int N> struct Count { static constexpr int value = N; };

// Many rows.  A workgroup takes BM rows of x and BN columns, in steps of 128
// bytes of the inner dimension (whole lines: half as many a step, four stages,
// took 642 us where 570 were taken otherwise, 16384 x 4096 x 4096 bf16), two stages
// of LDS.  Waves WM x WN, each BM / WM rows and BN / WN columns of each product:
// results as accumulators of 16 columns (their rows) by 16 rows of x (their
// columns).  Bound by the card's power rather than by its matrix cores' cycles
// (63 % of them at 1.6 GHz): products of 16 x 16 x 32, which move half the sums of
// those of 32 x 32 x 16, took 1107 us where the latter took 1219 (gated, 8192 x 4096
// x 11264 bf16), and eight waves of 128 x 64 less than four of 128 x 128 (487).
//
// A step has two parts (64 bytes of a row).  A part's operands are read from LDS
// between the products of the part before; before a step's last products the waves
// meet, when all its operands are in registers and the next stage's copies have
// landed: the last products then cover the first reads of that stage and the start
// of the copies into the stage just read.
//
// LDS rows of 128 bytes, their eight pieces exchanged by row (piece ^ row / 2 % 8):
// sixteen rows on end then spread over all 64 banks.
//
// VEC: rows in pieces of 16 bytes, aligned and whole, not overlapping, copied
// straight to LDS; else through registers, element by element at the inner
// dimension's end.
template <typename T, int BM, int BN, int WM, int WN, int NST, int OPS, bool VEC>
__global__ __launch_bounds__(64 * WM * WN, 2) void linear_tile_kernel(LinearArgs a) {
  constexpr int NW = WM * WN, PER = 16 / sizeof(T), STEP = 8 * PER;
  constexpr int ROWS = BM + OPS * BN, STAGE = ROWS * 128;
  constexpr int TM = BM / WM / 16, TN = BN / WN / 16, WIDE = OPS * TN * 16;
  static_assert(ROWS % (8 * NW) == 0 && BM % 8 == 0 && BN % 8 == 0 && NW % 2 == 0, "whole copies");
  // the epilogue turns 32 rows of a wave's results at a time
  constexpr int PITCH = WIDE + 4, TURN = 32 * PITCH * 4;
  constexpr int LDS = NST * STAGE > NW * TURN ? NST * STAGE : NW * TURN;
  __shared__ __attribute__((aligned(1024))) char lds[LDS];
  const int tid = threadIdx.x, lane = tid & 63, quarter = lane >> 4, col = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave % WM, wn = wave / WM;

  // Tiles in bands of eight rows of them, a band column by column; each XCD
  // (workgroup number mod 8) takes a run of them, so that its L2 holds what its
  // tiles share.
  const int tiles = a.row_tiles * a.col_tiles;
  int tile = blockIdx.x;
  {
    const int each = tiles / 8, rest = tiles % 8, xcd = tile % 8, i = tile / 8;
    tile = xcd * each + (xcd < rest ? xcd : rest) + i;
  }
  const int band = tile / (8 * a.col_tiles), in_band = tile % (8 * a.col_tiles);
  const int band_rows = a.row_tiles - 8 * band < 8 ? a.row_tiles - 8 * band : 8;
  const int64_t m0 = (int64_t)(8 * band + in_band % band_rows) * BM;
  const int n0 = in_band / band_rows * BN;

  const int steps_all = (a.inner + STEP - 1) / STEP, split = blockIdx.y;
  const int from = split * a.split_steps;
  const int steps = steps_all - from < a.split_steps ? steps_all - from : a.split_steps;

  // What this thread copies: rows 8 wave + lane / 8 + 8 NW i of the stage (a
  // copy's eight rows are all of one operand), place lane % 8.
  const int piece = (lane & 7) ^ (((8 * wave + (lane >> 3)) >> 1) & 7);
  constexpr int COPIES = ROWS / (8 * NW);
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
  i32x4 xb, wb[OPS];
  uint32_t at[VEC ? COPIES : 1];             // rows beyond x's and w's: out of the buffers' ranges
  if constexpr (VEC) {
    const int64_t rn = a.rows - m0 < BM ? a.rows - m0 : BM, cn = a.cols - n0 < BN ? a.cols - n0 : BN;
    xb = buffer_of((const T*)a.x + m0 * a.xr, (uint32_t)(((rn - 1) * a.xr + a.inner) * sizeof(T)));
#pragma unroll
    for (int o = 0; o < OPS; ++o)
      wb[o] = buffer_of((const T*)a.w[o] + n0 * a.wr[o],
                        (uint32_t)(((cn - 1) * a.wr[o] + a.inner) * sizeof(T)));
#pragma unroll
    for (int i = 0; i < COPIES; ++i) {
      const int base = 8 * wave + 8 * NW * i;
      const int o = OPS == 2 && base >= BM + BN ? 1 : 0;
      const int row = base + (lane >> 3) - (base < BM ? 0 : BM + o * BN);
      at[i] = (uint32_t)(row * (int)(base < BM ? a.xr : a.wr[o]) * (int)sizeof(T) + piece * 16);
    }
  }
  u32x4 regs[VEC ? 1 : COPIES];
  auto fetch = [&](int stage, int step, int i) {
    const int base = 8 * wave + 8 * NW * i, k = (from + step) * STEP + piece * PER;
    const int o = OPS == 2 && base >= BM + BN ? 1 : 0;
    if constexpr (VEC) {
      copy16(base < BM ? xb : wb[o], k < a.inner && step < steps ? at[i] : 0x80000000u, (uint32_t)((from + step) * 128),
             lds0 + stage * STAGE + base * 128);
    } else {
      const int r = base + (lane >> 3);
      int64_t row = base < BM ? m0 + r : n0 + r - BM - o * BN;
      const int64_t end = base < BM ? a.rows : a.cols;
      row = row < end ? row : end - 1;       // (its results are not stored)
      const T* const p = (base < BM ? (const T*)a.x + row * a.xr : (const T*)a.w[o] + row * a.wr[o]) + k;
      regs[i] = k + PER <= a.inner ? load16(p) : load_some(p, a.inner - k);
    }
  };
  auto fetch_all = [&](int stage, int step) {
#pragma unroll
    for (int i = 0; i < COPIES; ++i) fetch(stage, step, i);
  };
  auto deposit = [&](int stage) {
    if constexpr (!VEC) {
#pragma unroll
      for (int i = 0; i < COPIES; ++i)
        *reinterpret_cast<u32x4*>(lds + stage * STAGE + (8 * wave + 8 * NW * i) * 128 + lane * 16) = regs[i];
    }
  };
  // The next step's copies have landed (as many as later steps' may be on their
  // way), reads are done.
  auto meet = [&](auto later) {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(decltype(later)::value * COPIES) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };

  f4v acc[OPS * TN][TM];
#pragma unroll
  for (int i = 0; i < OPS * TN; ++i)
#pragma unroll
    for (int j = 0; j < TM; ++j) acc[i][j] = f4v{};

  const char* const xs = lds + (wm * (BM / WM) + col) * 128;
  const char* const ws = lds + (BM + wn * (BN / WN) + col) * 128;
  constexpr int READS = TM + OPS * TN, PRODUCTS = TM * OPS * TN;
  u32x4 xv[2][TM], wv[2][OPS * TN];
  auto read = [&](int stage, int s, int i) {
    const int off = stage * STAGE + (((4 * s + quarter) ^ (col >> 1)) << 4);
    if (i < TM) xv[s & 1][i] = *reinterpret_cast<const u32x4*>(xs + i * 16 * 128 + off);
    else wv[s & 1][i - TM] =
        *reinterpret_cast<const u32x4*>(ws + ((i - TM) / TN * BN + (i - TM) % TN * 16) * 128 + off);
  };

  // Results: 32 rows at a time turned through LDS, each wave for itself, so that
  // eight columns on end of a row are a lane's and a row's lanes lie on end.  The
  // residual's first rows are loaded here, the others a turn before they are added:
  // with one workgroup a CU nothing else would cover their way.
  float* const turn = reinterpret_cast<float*>(lds + wave * TURN);
  constexpr int LANES = TN * 2, PARTS = 32 * LANES / 64;      // LANES of a row
  const int nc = lane % LANES * 8, n = n0 + wn * (BN / WN) + nc;
  const int64_t mt = m0 + wm * (BM / WM) + lane / LANES;
  const bool wide = wide_columns<T>(a);
  const bool early = OPS == 1 && wide && a.residual != nullptr && a.parts == nullptr;
  auto residual_at = [&](int t) {
    const int64_t m = mt + t * (64 / LANES);
    return *reinterpret_cast<const Vec<T, 8>*>((const T*)a.residual + (m < a.rows ? m : a.rows - 1) * a.rr +
                                               (n < a.cols ? n : 0));
  };

  if (steps > 0) {
    fetch_all(0, 0);
    deposit(0);
    if constexpr (NST > 2) {
#pragma unroll
      for (int i = 1; i < NST; ++i) fetch_all(i, i);
      meet(Count<NST - 1>());
    } else {
      meet(Count<0>());
      if (steps > 1) fetch_all(1, 1);
    }
#pragma unroll
    for (int i = 0; i < READS; ++i) read(0, 0, i);
  }
  for (int step = 0; step < steps; ++step) {
    const int stage = step % NST, next = (step + 1) % NST;
    const bool more = step + 1 < steps, copies = NST > 2 || step + NST < steps;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      if (s == 1) {
        if (more) deposit(next);
        meet(Count<NST - 2>());
        __builtin_amdgcn_s_setprio(1);
      }
      if (s == 0) __builtin_amdgcn_s_setprio(0);
#pragma unroll
      for (int p = 0; p < PRODUCTS; ++p) {
        const int i = p / TM, j = p % TM;
        acc[i][j] = mfma<T>(wv[s & 1][i], xv[s & 1][j], acc[i][j]);
        // spread over the products: the next part's reads, and in the last part
        // the copies of the stage that takes this one's place
#pragma unroll
        for (int r = p * READS / PRODUCTS; r < (p + 1) * READS / PRODUCTS; ++r) {
          if (s == 0) read(stage, 1, r);
          else if (more) read(next, 0, r);
        }
        if (s == 1 && copies)
#pragma unroll
          for (int c = p * COPIES / PRODUCTS; c < (p + 1) * COPIES / PRODUCTS; ++c)
            fetch(stage, step + NST, c);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
  meet(Count<0>());                     // LDS is free for the results
  Vec<T, 8> ahead[PARTS];
  if (early) {
#pragma unroll
    for (int q = 0; q < PARTS; ++q) ahead[q] = residual_at(q);
  }
  float b[OPS][8];
#pragma unroll
  for (int o = 0; o < OPS; ++o)
#pragma unroll
    for (int e = 0; e < 8; ++e) b[o][e] = bias_of<T>(a, o, n + e < a.cols ? n + e : a.cols - 1);
#pragma unroll 1
  for (int j = 0; j < TM / 2; ++j) {
#pragma unroll
    for (int c = 0; c < TM; ++c)
      if (j == c / 2) {
#pragma unroll
        for (int i = 0; i < OPS * TN; ++i) {
          const Vec<float, 4> y = {acc[i][c][0], acc[i][c][1], acc[i][c][2], acc[i][c][3]};
          *reinterpret_cast<Vec<float, 4>*>(turn + (16 * (c & 1) + col) * PITCH + 16 * i + 4 * quarter) = y;
        }
      }
    Vec<T, 8> now[PARTS];
#pragma unroll
    for (int q = 0; q < PARTS; ++q) now[q] = ahead[q];
    if (early && j + 1 < TM / 2) {
#pragma unroll
      for (int q = 0; q < PARTS; ++q) ahead[q] = residual_at((j + 1) * PARTS + q);
    }
#pragma unroll
    for (int q = 0; q < PARTS; ++q) {
      const int r = q * (64 / LANES) + lane / LANES;
      const int64_t m = mt + (j * PARTS + q) * (64 / LANES);
      float y[OPS][8];
#pragma unroll
      for (int o = 0; o < OPS; ++o)
#pragma unroll
        for (int e = 0; e < 8; e += 4) {
          const Vec<float, 4> v =
              *reinterpret_cast<const Vec<float, 4>*>(turn + r * PITCH + o * TN * 16 + nc + e);
#pragma unroll
          for (int f = 0; f < 4; ++f) y[o][e + f] = v.v[f];
        }
      if (m < a.rows && n < a.cols) finish8<T, OPS>(a, m, n, split, y, b, now[q], early, wide);
    }
  }
}

// Rows of 16-bit numbers, whatever they are, on 128 bytes with zeros behind their last
// ones, for tiles that are read in whole pieces: 16 bytes a thread.  Bound by the
// bytes, read and written once at 4 TB/s.
__global__ __launch_bounds__(256) void linear_rows_kernel(const _Float16* from, _Float16* to, int64_t rows,
                                                          int inner, int64_t stride, int to_stride) {
  const int units = (inner + 7) / 8;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= rows * units) return;
  const int64_t row = i / units;
  const int k = (int)(i % units) * 8;
  const _Float16* const p = from + row * stride + k;
  *reinterpret_cast<u32x4*>(to + row * to_stride + k) =
      k + 8 > inner ? load_some(p, inner - k) : whole_of(words_at(p));
}

// The sums of the splits, in their order, and the epilogue: four columns a thread.
template <typename T, int OPS>
__global__ __launch_bounds__(256) void linear_join_kernel(LinearArgs a) {
  const int quads = (a.cols + 3) / 4;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= a.rows * quads) return;
  const int64_t m = i / quads;
  const int n = (int)(i % quads) * 4;
  float y[OPS][4];
#pragma unroll
  for (int o = 0; o < OPS; ++o)
#pragma unroll
    for (int e = 0; e < 4; ++e) y[o][e] = 0.0f;
  for (int s = 0; s < a.splits; ++s)
#pragma unroll
    for (int o = 0; o < OPS; ++o) {
      const float* const from = a.parts + (((int64_t)s * OPS + o) * a.rows + m) * a.cols + n;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n + e < a.cols) y[o][e] += from[e];
    }
  float b[OPS][4];
#pragma unroll
  for (int o = 0; o < OPS; ++o)
#pragma unroll
    for (int e = 0; e < 4; ++e) b[o][e] = bias_of<T>(a, o, n + e < a.cols ? n + e : a.cols - 1);
  finish<T, OPS, 4>(a, m, n, y, b, {}, false, wide_columns<T>(a));
}

// Which kernel, in what pieces.  The times are of bf16.
//   rows <= 32, and <= 8 or few columns: few rows (1 gated row of 4096 x 11264 37.0 us,
//     tiles 39.4, 8 rows 42.2 and 39.9; 8 rows of 4096 x 4096 9.8 and 19.7, 32 of 512 x
//     1000 4.6 and 5.9).  Else tiles read w no slower and x less often (32 gated rows
//     of 4096 x 11264: 39 us, few rows 59; 32 of 4096 x 4096 13.4 and 14.7).
//   256: most work a byte read from L2, one workgroup a CU.  Taken if its rounds of
//     the card are no longer than those of 128, four of whose tiles (at two a CU) take
//     as long as one of it, or 1.2 times as long where the inner dimension is long and
//     the start and the epilogue, which nothing covers here, count little (25088 x
//     4096 x 1536, 588 tiles: 289 us, 128 324; 25088 x 384 x 1536 55 and 51; 304 tiles,
//     4864 x 4096 x 4096: 177 and 167; 160, 2560 x 4096 x 4096: 88 and 104).  Not for 32-bit
//     numbers, whose matrix instructions bound every tile alike.
//   128, two stages and two workgroups a CU: more than a tile a CU (384 tiles, 1500 x
//     4096 x 4096: 57 to 60 us, four stages 67).
//   128, four stages: more than half a tile a CU (256 tiles, 1024 x 4096 x 4096: 37 us,
//     two stages 44, 64 53; 192 tiles 33 and 64 45; 128 tiles 32 and 64 29).
//   64: four stages, two workgroups a CU.  Of long rows that give less than a tile a CU
//     the inner dimension is split, 16 steps and more a split (64 x 4096 x 4096: 19.8
//     us whole, 14.5 in four; 256 x 2048 x 2048 would be 13.8 in two, and takes 12.1).
// Rows of 16 bits that are not in whole pieces of 16 bytes are first laid out so in the
// workspace (pack) if that takes less than it saves: a read and a write of all rows at
// 4.5 TB/s and 4 us for the launches, against 0.75 of the product's time or 0.55 us a
// step, whichever is more (9506 x 1121 x 8192: 193 us, read as they lie 310; 300 x 4097 x
// 4096 42 and 70; 64 x 1121 x 8192, 18773 x 1137 x 137: not).  Those of 32 bits lose too
// little (2673 x 3321 x 536: 150, 2672 x 3320 x 536 109).
struct Plan {
  bool few;                                // the few-rows kernel
  int size, splits, split_steps;
  bool pack[3];                            // x, w, w2
};

constexpr int FEW_ROWS = 32;
constexpr int CUS = 256;

// Whether rows are whole pieces of 16 bytes, aligned from the first on if it is,
// and do not overlap.
inline bool whole_rows(const CfLinearArgs& x, int64_t stride) {
  const int per = x.dtype == SEQ_F32 ? 4 : 8;
  return x.inner % per == 0 && stride % per == 0 && stride >= x.inner;
}

// How x and w are read: in whole pieces of 16 bytes, 256 rows of them within 2^31
// bytes.  `addresses`: look at those, too.
inline bool whole_pieces(const CfLinearArgs& x, const Plan& p, bool addresses) {
  const int size = x.dtype == SEQ_F32 ? 4 : 2;
  auto whole = [&](const void* base, int64_t stride, bool packed) {
    return packed || (whole_rows(x, stride) && stride * size * 256 < 0x7fffffffll &&
                      (!addresses || (uintptr_t)base % 16 == 0));
  };
  return whole(x.x, x.x_row, p.pack[0]) && whole(x.w, x.w_row, p.pack[1]) &&
         (!x.w2 || whole(x.w2, x.w2_row, p.pack[2]));
}

inline int64_t packed_row(const CfLinearArgs& x) {         // of 16 bits: whole lines
  return (x.inner + 63) / 64 * 64;
}

// The plan does not look at addresses, so that a workspace can be asked for without
// them.
inline Plan plan_of(const CfLinearArgs& x, bool gated) {
  Plan p = {false, 0, 1, 0, {false, false, false}};
  const bool f32 = x.dtype == SEQ_F32;
  const int64_t step = f32 ? 32 : 64, steps = (x.inner + step - 1) / step;
  const int half = gated ? 2 : 1;
  auto tiles = [&](int64_t bm, int64_t bn) {
    return ((x.rows + bm - 1) / bm) * ((x.cols + bn / half - 1) / (bn / half));
  };
  bool vec = whole_pieces(x, p, false);
  if (x.rows <= FEW_ROWS && (!vec || x.rows <= 8 || x.rows * tiles(64, 64) < 8 * CUS)) {
    p.few = true;
    return p;
  }
  // (laid out rows have to be near each other, too, and one launch's work)
  const int64_t longest = x.rows > x.cols ? x.rows : x.cols;
  if (!vec && !f32 && 2 * 256 * packed_row(x) < 0x7fffffffll && longest * packed_row(x) < 1ll << 34) {
    const double columns = (double)half * x.cols, bytes = 4.0 * (x.rows + columns) * x.inner;
    const double product = 2.0 * x.rows * columns * x.inner / 1.15e9;      // us
    const double saved = 0.75 * product > 0.55 * steps ? 0.75 * product : 0.55 * steps;
    if (saved > bytes / 4.5e6 + 4.0) {
      p.pack[0] = !whole_rows(x, x.x_row);
      p.pack[1] = !whole_rows(x, x.w_row);
      p.pack[2] = gated && !whole_rows(x, x.w2_row);
      vec = whole_pieces(x, p, false);
    }
  }
  const int64_t rounds256 = (tiles(256, 256) + CUS - 1) / CUS, rounds128 = (tiles(128, 128) + 2 * CUS - 1) / (2 * CUS);
  const bool most = vec && !f32 && 10 * rounds256 <= (steps < 16 ? 5 : 6) * rounds128;
  p.size = most ? 256 : 2 * tiles(128, 128) > CUS ? 128 : 64;
  p.split_steps = (int)steps;
  const int64_t n = tiles(64, 64), least = f32 ? 8 : 16;   // (a step of 32 bits takes twice as long)
  if (p.size == 64 && n < CUS && steps >= 3 * least) {
    int64_t splits = CUS / n;
    if (splits > steps / least) splits = steps / least;
    if (splits > 1) {
      p.split_steps = (int)((steps + splits - 1) / splits);
      p.splits = (int)((steps + p.split_steps - 1) / p.split_steps);
    }
  }
  return p;
}

inline int64_t parts_bytes(const CfLinearArgs& x, const Plan& p, bool gated) {
  return p.few || p.splits < 2 ? 0 : (4 * (gated ? 2 : 1) * p.splits * x.rows * x.cols + 255) / 256 * 256;
}

inline int64_t workspace_of(const CfLinearArgs& x, const Plan& p, bool gated) {
  const int64_t rows = (p.pack[0] ? x.rows : 0) + (p.pack[1] ? x.cols : 0) + (p.pack[2] ? x.cols : 0);
  return parts_bytes(x, p, gated) + 2 * rows * packed_row(x);
}

template <typename T, int OPS, bool ODD>
hipError_t launch_rows(const LinearArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)((a.cols + 15) / 16));
  if (a.rows <= 16) hipLaunchKernelGGL((linear_few_kernel<T, 1, OPS, ODD>), grid, dim3(512), 0, st, a);
  else hipLaunchKernelGGL((linear_few_kernel<T, 2, OPS, ODD>), grid, dim3(512), 0, st, a);
  return hipGetLastError();
}

template <typename T, int OPS>
hipError_t launch_few(const LinearArgs& a, hipStream_t st) {
  if constexpr (sizeof(T) == 2) {
    auto odd = [](const void* base, int64_t stride) { return (uintptr_t)base % 4 != 0 || stride % 2 != 0; };
    if (odd(a.x, a.rows > 1 ? a.xr : 0) || odd(a.w[0], a.wr[0]) || (OPS == 2 && odd(a.w[1], a.wr[1])))
      return launch_rows<T, OPS, true>(a, st);
  }
  return launch_rows<T, OPS, false>(a, st);
}

template <typename T, int BM, int BN, int WM, int WN, int NST, int OPS, bool VEC>
hipError_t launch_tiles(const LinearArgs& a, hipStream_t st) {
  const int64_t ct = (a.cols + BN - 1) / BN;
  // a launch has fewer than 2^32 threads: more tiles take several, of whole bands
  const int64_t most = 0xffffffffll / (64 * WM * WN) / ct / 8 * 8 * BM;
  for (int64_t m = 0; m < a.rows; m += most) {
    LinearArgs b = a;
    b.x = (const T*)a.x + m * a.xr;
    b.out = (T*)a.out + m * a.orow;
    if (a.residual) b.residual = (const T*)a.residual + m * a.rr;
    b.rows = a.rows - m < most ? a.rows - m : most;
    b.row_tiles = (int)((b.rows + BM - 1) / BM);
    b.col_tiles = (int)ct;
    hipLaunchKernelGGL((linear_tile_kernel<T, BM, BN, WM, WN, NST, OPS, VEC>),
                       dim3((unsigned)(b.row_tiles * ct), (unsigned)a.splits), dim3(64 * WM * WN), 0, st, b);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  if (a.parts == nullptr) return hipSuccess;
  const int64_t n = a.rows * ((a.cols + 3) / 4);   // (splits have fewer tiles than the card CUs)
  hipLaunchKernelGGL((linear_join_kernel<T, OPS>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, a);
  return hipGetLastError();
}

template <typename T, int OPS, bool VEC>
hipError_t launch_sizes(const LinearArgs& a, const Plan& p, hipStream_t st) {
  constexpr int N = OPS == 2 ? 2 : 1;
  if constexpr (VEC && sizeof(T) == 2)
    if (p.size == 256) return launch_tiles<T, 256, 256 / N, 2, 4, 2, OPS, true>(a, st);
  if (p.size == 128) {
    if constexpr (VEC)
      if (((a.rows + 127) / 128) * ((a.cols + 128 / N - 1) / (128 / N)) <= CUS)
        return launch_tiles<T, 128, 128 / N, 2, 4, 4, OPS, true>(a, st);
    return launch_tiles<T, 128, 128 / N, 2, 4, 2, OPS, VEC>(a, st);
  }
  return launch_tiles<T, 64, 64 / N, 2, 2, VEC ? 4 : 2, OPS, VEC>(a, st);
}

template <typename T, int OPS>
hipError_t launch_linear(const LinearArgs& a, const Plan& p, bool vec, hipStream_t st) {
  if (p.few) return launch_few<T, OPS>(a, st);
  return vec ? launch_sizes<T, OPS, true>(a, p, st) : launch_sizes<T, OPS, false>(a, p, st);
}

// The rows that the plan says into the workspace, from `at` on; a reads them there.
inline hipError_t pack_rows(const CfLinearArgs& x, const Plan& p, int64_t at, LinearArgs& a, hipStream_t st) {
  const int64_t stride = packed_row(x), units = (x.inner + 7) / 8;
  auto pack = [&](const void*& base, int64_t& row, int64_t rows) {
    _Float16* const to = (_Float16*)((char*)x.workspace + at);
    const int64_t blocks = (rows * units + 255) / 256;
    if (blocks > 0xffffffffll / 256) return hipErrorInvalidValue;
    hipLaunchKernelGGL(linear_rows_kernel, dim3((unsigned)blocks), dim3(256), 0, st,
                       (const _Float16*)base, to, rows, (int)x.inner, row, (int)stride);
    at += 2 * rows * stride;
    base = to;
    row = stride;
    return hipGetLastError();
  };
  hipError_t e = hipSuccess;
  if (p.pack[0]) e = pack(a.x, a.xr, x.rows);
  if (e == hipSuccess && p.pack[1]) e = pack(a.w[0], a.wr[0], x.cols);
  if (e == hipSuccess && p.pack[2]) e = pack(a.w[1], a.wr[1], x.cols);
  if (e == hipSuccess) a.inner = (int)(8 * units);
  return e;
}

template <typename T>
hipError_t launch_ops(const LinearArgs& a, const Plan& p, bool vec, hipStream_t st) {
  return a.w[1] ? launch_linear<T, 2>(a, p, vec, st) : launch_linear<T, 1>(a, p, vec, st);
}

inline bool sizes_make_sense(const CfLinearArgs& x) {
  return x.dtype >= 0 && x.dtype <= 2 && x.rows >= 0 && x.rows <= CF_LINEAR_MAX_ROWS && x.inner >= 0 &&
         x.inner <= CF_LINEAR_MAX_WIDTH && x.cols >= 1 && x.cols <= CF_LINEAR_MAX_WIDTH;
}

}  // namespace

CF_API int64_t cf_linear_workspace(const CfLinearArgs* p) {
  if (!p || !sizes_make_sense(*p)) return -1;
  const bool gated = p->w2 != nullptr;
  return workspace_of(*p, plan_of(*p, gated), gated);
}

CF_API int cf_linear(const CfLinearArgs* p) {
  if (!p) return (int)hipErrorInvalidValue;
  const CfLinearArgs& x = *p;
  if (!sizes_make_sense(x) || x.activation < 0 || x.activation > CF_ACT_GELU_TANH || x.x_row < 0 ||
      x.w_row < 0 || x.w2_row < 0 || x.residual_row < 0 || x.out_row < x.cols || x.workspace_bytes < 0)
    return (int)hipErrorInvalidValue;
  if (x.rows == 0) return 0;
  const bool gated = x.w2 != nullptr;
  if (!x.out || (x.inner > 0 && (!x.x || !x.w)) || (gated && x.residual))
    return (int)hipErrorInvalidValue;
  Plan plan = plan_of(x, gated);
  const int64_t need = workspace_of(x, plan, gated);
  if (need > 0 && (!x.workspace || (uintptr_t)x.workspace % 16 != 0 || x.workspace_bytes < need))
    return (int)hipErrorInvalidValue;
  LinearArgs a;
  a.x = x.x;
  a.w[0] = x.w; a.w[1] = x.w2;
  a.bias[0] = x.bias; a.bias[1] = x.bias2;
  a.residual = x.residual;
  a.out = x.out;
  a.parts = plan.splits > 1 ? (float*)x.workspace : nullptr;
  a.bias_f32 = x.bias_f32 != 0;
  a.activation = (int)x.activation;
  a.rows = x.rows; a.inner = (int)x.inner; a.cols = (int)x.cols;
  a.xr = x.x_row; a.wr[0] = x.w_row; a.wr[1] = x.w2_row; a.rr = x.residual_row; a.orow = x.out_row;
  a.splits = plan.splits; a.split_steps = plan.split_steps;
  const bool v = whole_pieces(x, plan, true);
  if (!v && plan.size == 256) plan.size = 128;              // (an address that is no multiple of 16)
  a.row_tiles = a.col_tiles = 0;
  hipStream_t st = (hipStream_t)x.stream;
  hipError_t e;
  if (v && (plan.pack[0] || plan.pack[1] || plan.pack[2])) {
    e = pack_rows(x, plan, parts_bytes(x, plan, gated), a, st);
    if (e != hipSuccess) return (int)e;
  }
  if (x.dtype == SEQ_F32) e = launch_ops<float>(a, plan, v, st);
  else if (x.dtype == SEQ_F16) e = launch_ops<_Float16>(a, plan, v, st);
  else e = launch_ops<bf16_t>(a, plan, v, st);
  return (int)e;
}
