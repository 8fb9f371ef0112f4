// Position rotation of attention heads, with or without the norm of each head
// in the same pass, for one or two tensors (queries and keys) a launch.
//
//   y = x / sqrt(mean_d x^2 + eps) * weight                      (normed form)
//   (y_a, y_b) <- (y_a cos - y_b sin, y_b cos + y_a sin),  angle = pos f_i
// for the pairs i < pairs of a head: channels (i, i + pairs), or (2 i, 2 i + 1)
// interleaved; channels past 2 pairs are not turned.  Pair i takes the
// position of axis a where sec[a] <= i < sec[a + 1] (time, height, width), and
// inverse turns by -angle.
//
// The angle is taken in 64 bits as a number of turns, pos * f / (2 pi), whose
// whole part is dropped before rounding to fp32: a position of 2^31 keeps an
// angle within 1e-6, where an fp32 product is wrong from a few thousand on.
// Everything else is fp32; each output is rounded once.
//
// No counterpart in the reference.
#include "cf_seq.h"

namespace {

struct RotaryTensor {
  const void* x;
  void* y;
  const void* weight;          // [d] or [heads][d], or null
  int weight_f32;              // else of the tensor's type
  int64_t weight_head;         // elements from one head's weights to the next (0: shared)
  int64_t xo, xi, xh, yo, yi, yh;
  int heads;
};

struct RotaryArgs {
  RotaryTensor t[2];
  const void* pos;
  int pos_kind;                // 0 int32, 1 int64, 2 float32
  int64_t pa, po, pi;          // element strides: axis, outer, inner token
  const double* freqs;
  int sec[CF_ROTARY_MAX_AXES + 1];
  int axes;
  int64_t outer, inner;
  int d, pairs;
  int interleaved, norm;
  float eps, sign;
};

__device__ __forceinline__ double rotary_pos(const RotaryArgs& a, int64_t i) {
  if (a.pos_kind == 0) return (double)reinterpret_cast<const int32_t*>(a.pos)[i];
  if (a.pos_kind == 1) return (double)reinterpret_cast<const int64_t*>(a.pos)[i];
  return (double)reinterpret_cast<const float*>(a.pos)[i];
}

constexpr double INV_TWO_PI = 0.15915494309189533577;

// cos and sin of pos * freq.
__device__ __forceinline__ float2 rotary_angle(double pos, double freq) {
  const double turns = pos * freq * INV_TWO_PI;
  const float part = (float)(turns - rint(turns));   // within half a turn
  float sn, cs;
  sincospif(2.0f * part, &sn, &cs);
  return make_float2(cs, sn);
}

// Output stores: past the caches where the launch writes more than what the next
// one could find there.  Measured (us, plain / streaming): 16384 tokens x 40
// heads x 128 bf16 85.4 / 73.5, 28800 x 16 x 128 44.8 / 38.3; followed by
// decay_attention, 268 MB of outputs 335 / 328, but 67 MB 102.5 / 105.
constexpr int64_t STREAM_BYTES = 96 << 20;
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
template <bool STREAM, typename T, int VE>
__device__ __forceinline__ void put(T* p, const Vec<T, VE>& v) {
  if constexpr (STREAM)
    __builtin_nontemporal_store(__builtin_bit_cast(u32x4, v), reinterpret_cast<u32x4*>(p));
  else
    *reinterpret_cast<Vec<T, VE>*>(p) = v;
}

// Rows (a token's head) of LG lanes; a lane holds PU pair units (VE pairs: two
// vectors of VE elements) and RU vectors of channels that are not turned.
// A workgroup takes TT tokens: their angles first, one a thread, into LDS, so
// that the sines are computed once for all heads; also there where each token's
// heads lie (64-bit divisions) and the weights that the heads share, as fp32.
// Bound by HBM where it is large: with the norm 16384 tokens x 40 heads x 128
// bf16 74 us (4.6 TB/s), without it 28800 x 16 x 128 38 us (6.2 TB/s, inputs
// partly in the last-level cache).
template <typename T, int VE, int PU, int RU, bool STREAM>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a, int lg, int tt, int head_split) {
  extern __shared__ __attribute__((aligned(32))) char lds[];
  const int tid = threadIdx.x, shared_d = (a.d + 7) / 8 * 8;
  int64_t* const at_sh = reinterpret_cast<int64_t*>(lds);              // [tt][4]: x, y, k, k's y
  float2* const cs_sh = reinterpret_cast<float2*>(at_sh + 4 * tt);     // [tt][pairs]
  float* const w_sh = reinterpret_cast<float*>(cs_sh + (tt * a.pairs + 3) / 4 * 4);  // [2][shared_d]
  const int64_t tokens = a.outer * a.inner, tok0 = (int64_t)blockIdx.x * tt;
  const int ntok = (int)(tokens - tok0 < tt ? tokens - tok0 : tt);
  for (int i = tid; i < ntok * a.pairs; i += 256) {
    const int t = i / a.pairs, p = i % a.pairs;
    int axis = 0;
    while (axis + 1 < a.axes && p >= a.sec[axis + 1]) ++axis;
    const int64_t tok = tok0 + t, o = a.outer == 1 ? 0 : tok / a.inner, n = tok - o * a.inner;
    float2 cs = rotary_angle(rotary_pos(a, axis * a.pa + o * a.po + n * a.pi), a.freqs[p]);
    cs.y *= a.sign;
    cs_sh[i] = cs;
  }
  for (int i = tid; i < ntok; i += 256) {
    const int64_t tok = tok0 + i, o = a.outer == 1 ? 0 : tok / a.inner, n = tok - o * a.inner;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      at_sh[4 * i + 2 * j] = o * a.t[j].xo + n * a.t[j].xi;
      at_sh[4 * i + 2 * j + 1] = o * a.t[j].yo + n * a.t[j].yi;
    }
  }
  if (a.norm) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const RotaryTensor& r = a.t[j];
      if (r.weight == nullptr || r.weight_head == 0)
        for (int i = tid; i < a.d; i += 256)
          w_sh[j * shared_d + i] =
              r.weight == nullptr ? 1.0f
              : r.weight_f32      ? reinterpret_cast<const float*>(r.weight)[i]
                                  : to_f(reinterpret_cast<const T*>(r.weight)[i]);
    }
  }
  __syncthreads();
  const int lane = tid % lg, heads = a.t[0].heads + a.t[1].heads;
  const int upairs = a.pairs / VE, urest = (a.d - 2 * a.pairs) / VE;
  const int step = 256 / lg * head_split;
  int t = 0, head = tid / lg + 256 / lg * (int)blockIdx.y;   // the row: token and head of both
  for (;; head += step) {
    while (head >= heads) {
      head -= heads;
      ++t;
    }
    if (t >= ntok) break;
    const int second = head >= a.t[0].heads ? 1 : 0, h = head - (second ? a.t[0].heads : 0);
    const RotaryTensor& r = a.t[second];
    const T* const x = (const T*)r.x + at_sh[4 * t + 2 * second] + h * r.xh;
    T* const y = (T*)r.y + at_sh[4 * t + 2 * second + 1] + h * r.yh;
    float va[PU][VE], vb[PU][VE], vr[RU > 0 ? RU : 1][VE];
    float sum = 0.0f;
#pragma unroll
    for (int u = 0; u < PU; ++u) {
      const int unit = lane + u * lg;
      Vec<T, VE> xa{}, xb{};
      if (unit < upairs) {
        const int ca = a.interleaved ? 2 * unit * VE : unit * VE;
        const int cb = a.interleaved ? ca + VE : a.pairs + unit * VE;
        xa = *reinterpret_cast<const Vec<T, VE>*>(x + ca);
        xb = *reinterpret_cast<const Vec<T, VE>*>(x + cb);
      }
#pragma unroll
      for (int i = 0; i < VE; ++i) {
        va[u][i] = to_f(xa.v[i]);
        vb[u][i] = to_f(xb.v[i]);
        sum = __builtin_fmaf(va[u][i], va[u][i], sum);
        sum = __builtin_fmaf(vb[u][i], vb[u][i], sum);
      }
    }
#pragma unroll
    for (int u = 0; u < RU; ++u) {
      const int unit = lane + u * lg;
      Vec<T, VE> xr{};
      if (unit < urest) xr = *reinterpret_cast<const Vec<T, VE>*>(x + 2 * a.pairs + unit * VE);
#pragma unroll
      for (int i = 0; i < VE; ++i) {
        vr[u][i] = to_f(xr.v[i]);
        sum = __builtin_fmaf(vr[u][i], vr[u][i], sum);
      }
    }
    if (a.norm) {
      // (the lanes of a row run together: rows are whole groups of lg lanes)
      for (int m = lg >> 1; m > 0; m >>= 1) sum += __shfl_xor(sum, m, 64);
      const float inv = 1.0f / __builtin_sqrtf(sum / (float)a.d + a.eps);
      // the weights of VE channels from c on, times the norm
      auto scale = [&](float* v, int c) {
        if (r.weight == nullptr || r.weight_head == 0) {
          const Vec<float, VE> w =
              *reinterpret_cast<const Vec<float, VE>*>(w_sh + second * shared_d + c);
#pragma unroll
          for (int i = 0; i < VE; ++i) v[i] = v[i] * inv * w.v[i];
        } else {
          const int64_t from = h * r.weight_head + c;
#pragma unroll
          for (int i = 0; i < VE; ++i)
            v[i] = v[i] * inv * (r.weight_f32 ? reinterpret_cast<const float*>(r.weight)[from + i]
                                              : to_f(reinterpret_cast<const T*>(r.weight)[from + i]));
        }
      };
#pragma unroll
      for (int u = 0; u < PU; ++u) {
        const int unit = lane + u * lg;
        if (unit < upairs) {
          const int ca = a.interleaved ? 2 * unit * VE : unit * VE;
          scale(va[u], ca);
          scale(vb[u], a.interleaved ? ca + VE : a.pairs + unit * VE);
        }
      }
#pragma unroll
      for (int u = 0; u < RU; ++u) {
        const int unit = lane + u * lg;
        if (unit < urest) scale(vr[u], 2 * a.pairs + unit * VE);
      }
    }
#pragma unroll
    for (int u = 0; u < PU; ++u) {
      const int unit = lane + u * lg;
      if (unit >= upairs) break;
      const float2* const cs = cs_sh + t * a.pairs + unit * VE;
      const int ca = a.interleaved ? 2 * unit * VE : unit * VE;
      const int cb = a.interleaved ? ca + VE : a.pairs + unit * VE;
      Vec<T, VE> ya, yb;
      if (a.interleaved) {
        // vector a holds pairs 0 .. VE / 2 - 1 of the unit, vector b the rest
        // (VE == 1: the pair is (a, b) itself)
        if constexpr (VE == 1) {
          ya.v[0] = from_f<T>(va[u][0] * cs[0].x - vb[u][0] * cs[0].y);
          yb.v[0] = from_f<T>(vb[u][0] * cs[0].x + va[u][0] * cs[0].y);
        } else {
#pragma unroll
          for (int i = 0; i < VE; i += 2) {
            const float2 ea = cs[i / 2], eb = cs[VE / 2 + i / 2];
            ya.v[i] = from_f<T>(va[u][i] * ea.x - va[u][i + 1] * ea.y);
            ya.v[i + 1] = from_f<T>(va[u][i + 1] * ea.x + va[u][i] * ea.y);
            yb.v[i] = from_f<T>(vb[u][i] * eb.x - vb[u][i + 1] * eb.y);
            yb.v[i + 1] = from_f<T>(vb[u][i + 1] * eb.x + vb[u][i] * eb.y);
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < VE; ++i) {
          ya.v[i] = from_f<T>(va[u][i] * cs[i].x - vb[u][i] * cs[i].y);
          yb.v[i] = from_f<T>(vb[u][i] * cs[i].x + va[u][i] * cs[i].y);
        }
      }
      put<STREAM>(y + ca, ya);
      put<STREAM>(y + cb, yb);
    }
#pragma unroll
    for (int u = 0; u < RU; ++u) {
      const int unit = lane + u * lg;
      if (unit >= urest) break;
      Vec<T, VE> yr;
#pragma unroll
      for (int i = 0; i < VE; ++i) yr.v[i] = from_f<T>(vr[u][i]);
      put<STREAM>(y + 2 * a.pairs + unit * VE, yr);
    }
  }
}

constexpr int ROTARY_LDS = 32768;   // bytes of angles a workgroup holds at most
constexpr int ROTARY_TOKENS = 256;  // tokens of a workgroup at most (32 bytes of LDS each)

template <typename T, int VE, int PU, int RU, bool STREAM>
hipError_t launch_rotary_v(const RotaryArgs& a, int lg, hipStream_t st) {
  const int64_t tokens = a.outer * a.inner;
  const int heads = a.t[0].heads + a.t[1].heads;
  // tokens a workgroup: about four rounds of rows, as far as their angles fit
  int tt = (4 * (256 / lg) + heads - 1) / heads;
  const int fit = a.pairs > 0 ? ROTARY_LDS / (8 * a.pairs) : tt;
  if (tt > fit) tt = fit;
  if (tt > ROTARY_TOKENS) tt = ROTARY_TOKENS;
  if (tt < 1) tt = 1;
  // few tokens: their rows over several workgroups
  const int64_t groups = (tokens + tt - 1) / tt;
  int split = 1;
  while (split < 16 && groups * split < 256 && split * (256 / lg) < tt * heads) split *= 2;
  if (groups > 0x7fffffff) return hipErrorInvalidValue;
  hipLaunchKernelGGL((rotary_kernel<T, VE, PU, RU, STREAM>), dim3((unsigned)groups, (unsigned)split),
                     dim3(256), (size_t)tt * 32 + (tt * a.pairs + 3) / 4 * 32 + (a.d + 7) / 8 * 64, st,
                     a, lg, tt, split);
  return hipGetLastError();
}

int pow2_at_least(int n) {
  int p = 1;
  while (p < n) p *= 2;
  return p;
}

// The widest vectors that the channels, strides and addresses allow: 16 bytes
// (one pair unit and up to two others a lane), 8 or 4 bytes or single elements,
// several units a lane.  Measured (us, 20000 tokens x 24 heads, bf16): heads of 52,
// single elements in 64 lanes 129, vectors of 4 bytes in 8 lanes 29; heads of 46,
// single elements in 64 lanes 125, in 8 lanes 35.
template <typename T>
hipError_t launch_rotary(const RotaryArgs& a, bool stream, hipStream_t st) {
  constexpr int V16 = 16 / sizeof(T), V8 = 8 / sizeof(T);
  const int rest = a.d - 2 * a.pairs;
  auto fits = [&](int ve) {
    bool ok = a.pairs % ve == 0 && rest % ve == 0;
    for (int i = 0; i < 2; ++i) {
      const RotaryTensor& r = a.t[i];
      if (r.heads == 0) continue;
      const uintptr_t bytes = ve * sizeof(T);
      ok = ok && (uintptr_t)r.x % bytes == 0 && (uintptr_t)r.y % bytes == 0;
      for (int64_t s : {r.xo, r.xi, r.xh, r.yo, r.yi, r.yh}) ok = ok && s % ve == 0;
    }
    return ok;
  };
  // lanes of a row for pu pair units and ru others a lane
  auto lanes = [&](int ve, int pu, int ru) {
    const int up = (a.pairs / ve + pu - 1) / pu, ur = (rest / ve + ru - 1) / ru;
    return pow2_at_least(up > ur ? up : ur);
  };
  if (fits(V16)) {
    const int lg = lanes(V16, 1, 2);
    if (rest == 0)
      return stream ? launch_rotary_v<T, V16, 1, 0, true>(a, lg, st)
                    : launch_rotary_v<T, V16, 1, 0, false>(a, lg, st);
    return stream ? launch_rotary_v<T, V16, 1, 2, true>(a, lg, st)
                  : launch_rotary_v<T, V16, 1, 2, false>(a, lg, st);
  }
  if (fits(V8)) return launch_rotary_v<T, V8, 2, 4, false>(a, lanes(V8, 2, 4), st);
  if (sizeof(T) == 2 && fits(2)) return launch_rotary_v<T, 2, 2, 4, false>(a, lanes(2, 2, 4), st);
  return launch_rotary_v<T, 1, 4, 8, false>(a, lanes(1, 4, 8), st);
}
// (16 bytes: 64 x 4 pairs and 2 x 64 x 4 channels of fp32; 4 bytes: 2 x 64 x 2 and
// 4 x 64 x 2; single ones: 4 x 64 and 8 x 64)
static_assert(CF_ROTARY_MAX_DIM <= 512, "a row takes at most 64 lanes");

}  // namespace

CF_API int cf_rotary(const CfRotaryArgs* p) {
  if (!p) return (int)hipErrorInvalidValue;
  const CfRotaryArgs& x = *p;
  if (x.outer < 0 || x.inner < 0 || x.x_heads < 1 || x.x_heads > CF_SEQ_MAX_HEADS ||
      x.k_heads < 0 || x.k_heads > CF_SEQ_MAX_HEADS || x.d < 1 || x.d > CF_ROTARY_MAX_DIM ||
      x.pairs < 0 || 2 * x.pairs > x.d || x.axes < 1 || x.axes > CF_ROTARY_MAX_AXES ||
      x.dtype < 0 || x.dtype > 2 || x.pos_kind < 0 || x.pos_kind > 2 || !(x.eps >= 0.0))
    return (int)hipErrorInvalidValue;
  RotaryArgs a;
  const int64_t sec[4] = {0, x.section1, x.section2, x.pairs};
  for (int i = 0; i <= x.axes; ++i) {
    a.sec[i] = (int)(i == x.axes ? x.pairs : sec[i]);
    if (i > 0 && (sec[i] < 0 || a.sec[i] < a.sec[i - 1] || a.sec[i] > x.pairs))
      return (int)hipErrorInvalidValue;
  }
  if (x.inner > 0 && x.outer > INT64_MAX / x.inner) return (int)hipErrorInvalidValue;
  if (x.outer == 0 || x.inner == 0) return 0;
  if (!x.x || !x.x_out || (x.k_heads > 0 && (!x.k || !x.k_out)) ||
      (x.pairs > 0 && (!x.positions || !x.freqs)))
    return (int)hipErrorInvalidValue;
  a.t[0] = {x.x, x.x_out, x.x_weight, x.x_weight_f32 != 0, x.x_weight_head,
            x.x_outer, x.x_inner, x.x_head, x.x_out_outer, x.x_out_inner, x.x_out_head,
            (int)x.x_heads};
  a.t[1] = {x.k, x.k_out, x.k_weight, x.k_weight_f32 != 0, x.k_weight_head,
            x.k_outer, x.k_inner, x.k_head, x.k_out_outer, x.k_out_inner, x.k_out_head,
            (int)x.k_heads};
  a.pos = x.positions; a.pos_kind = (int)x.pos_kind;
  a.pa = x.pos_axis; a.po = x.pos_outer; a.pi = x.pos_inner;
  a.freqs = x.freqs;
  a.axes = (int)x.axes;
  a.outer = x.outer; a.inner = x.inner;
  a.d = (int)x.d; a.pairs = (int)x.pairs;
  a.interleaved = x.interleaved != 0; a.norm = x.norm != 0;
  a.eps = (float)x.eps; a.sign = x.inverse ? -1.0f : 1.0f;
  const int64_t rows = x.outer * x.inner, row = (x.x_heads + x.k_heads) * x.d * (x.dtype == SEQ_F32 ? 4 : 2);
  const bool stream = rows > STREAM_BYTES / row;
  hipStream_t st = (hipStream_t)x.stream;
  hipError_t e;
  if (x.dtype == SEQ_F32) e = launch_rotary<float>(a, stream, st);
  else if (x.dtype == SEQ_F16) e = launch_rotary<_Float16>(a, stream, st);
  else e = launch_rotary<bf16_t>(a, stream, st);
  return (int)e;
}
