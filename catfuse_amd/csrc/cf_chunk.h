// Device helpers of the attentions that run by chunks of tokens on the matrix
// cores (decay_attention.hip, delta_attention.hip): numbers as parts of eight
// bits, a chunk's images in LDS, their loads and the operands read from them.
#pragma once
#include "cf_seq.h"

namespace {

typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef short s4 __attribute__((ext_vector_type(4)));

constexpr uint32_t OOB = 0x80000000u;      // an offset beyond every range used here

// Parts of eight bits that an input's number has.
template <typename T> constexpr int parts_of() { return sizeof(T) == 4 ? 3 : 2; }
template <> constexpr int parts_of<bf16_t>() { return 1; }

__device__ __forceinline__ float high_part(float x) {
  return __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, x) & 0xffff0000u);
}
__device__ __forceinline__ uint32_t pack_high(float lo, float hi) {
  return __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, hi), __builtin_bit_cast(uint32_t, lo),
                               0x07060302u);
}

// Two numbers as N parts of eight bits cut off, most significant first, in word
// p of the N operands (what is left each time is exact).
template <int N>
__device__ __forceinline__ void split2(float a, float b, u32x4* out, int p) {
#pragma unroll
  for (int n = 0; n < N; ++n) {
    out[n][p] = pack_high(a, b);
    a -= high_part(a);
    b -= high_part(b);
  }
}
template <int N>
__device__ __forceinline__ void split8(const float* x, u32x4* out) {
#pragma unroll
  for (int p = 0; p < 4; ++p) split2<N>(x[2 * p], x[2 * p + 1], out, p);
}

__device__ __forceinline__ f16v mfma(u32x4 a, u32x4 b, f16v c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf8, a),
                                                 __builtin_bit_cast(bf8, b), c, 0, 0, 0);
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_rsrc(const void* base, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), (short)0, (int)bytes,
                                           0x00020000);
}

// LDS images of a chunk: [part][C rows][D channels] bf16, unpadded, the
// 16-byte pieces of a row exchanged by row so that both kinds of reads spread
// over all banks: 16 bytes of 16 rows on end (operands whose product runs over
// the channels), and 8 bytes of 4 rows on end, 32 channels wide (the
// transposing reads of operands whose product runs over the tokens).
template <int D>
__device__ __forceinline__ int swizzle(int row) {
  constexpr int SH = D >= 128 ? 0 : (D == 64 ? 1 : 2);
  return ((row >> 2) & 3) | (((row & 3) >> SH) << 2);
}
template <int C, int D>
__device__ __forceinline__ int image_at(int part, int row, int piece) {   // in bytes
  return ((part * C + row) * (D / 8) + (piece ^ swizzle<D>(row))) * 16;
}

// One unit of a chunk: 8 channels of a row, as loaded.
template <typename T>
struct Unit { u32x4 w[sizeof(T) / 2]; };

// This thread's units of a chunk's image: piece tid % (D / 8) of the rows
// tid / (D / 8) + i NT / (D / 8).  Rows from n on and channels from d on are
// zeros: out of the buffer's range (VEC: 16-byte loads, from aligned rows of
// whole 16-byte pieces that do not overlap) or masked.
template <typename T, int U, int D, int NT, bool VEC>
__device__ __forceinline__ void load_units(Unit<T>* u, const T* base, int n, int64_t stride, int d) {
  constexpr int PER = 16 / sizeof(T), ROWS = NT / (D / 8);
  const int row = threadIdx.x / (D / 8), c0 = threadIdx.x % (D / 8) * 8;
  if constexpr (VEC) {
    const int st = (int)stride * (int)sizeof(T);   // at least d's: rows from n on are beyond the range
    const __amdgpu_buffer_rsrc_t rsrc =
        rows_rsrc(base, (uint32_t)((n - 1) * st + d * (int)sizeof(T)));
#pragma unroll
    for (int p = 0; p < (int)(sizeof(T) / 2); ++p) {
      const uint32_t at = c0 + p * PER < d ? (uint32_t)(row * st + (c0 + p * PER) * (int)sizeof(T)) : OOB;
#pragma unroll
      for (int i = 0; i < U; ++i)
        u[i].w[p] = __builtin_amdgcn_raw_buffer_load_b128(rsrc, at + (uint32_t)(i * ROWS * st), 0, 0);
    }
  } else {
    // By words from a base brought to one, whatever a row's alignment: a row of 16
    // bits that begins inside a word is put together from five of them.  (The last
    // word may hold two bytes more than the rows do; each word of a load has its own
    // range check.)  Walks over 16 bits took 216 and 100 us so, and 272 and 128 with a load
    // for each element.
    const uintptr_t p = (uintptr_t)base, skip = p & 3;
    const int st = (int)stride * (int)sizeof(T);
    const __amdgpu_buffer_rsrc_t rsrc = rows_rsrc(
        (const void*)(p - skip), (uint32_t)((n - 1) * st + d * (int)sizeof(T) + (int)skip + 3) & ~3u);
    constexpr int WORDS = 2 * sizeof(T);
    uint32_t keep[WORDS];                          // channels from d on are none
#pragma unroll
    for (int j = 0; j < WORDS; ++j) {
      if constexpr (sizeof(T) == 4) keep[j] = c0 + j < d ? ~0u : 0u;
      else keep[j] = c0 + 2 * j + 1 < d ? ~0u : c0 + 2 * j < d ? 0xffffu : 0u;
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int r = row + i * ROWS;
      const uint32_t at = r < n && c0 < d ? (uint32_t)(r * st + c0 * (int)sizeof(T) + (int)skip) : OOB;
      if constexpr (sizeof(T) == 2) {
        const u32x4 w = __builtin_amdgcn_raw_buffer_load_b128(rsrc, at & ~3u, 0, 0);
        const uint32_t last = __builtin_amdgcn_raw_buffer_load_b32(rsrc, (at & ~3u) + 16, 0, 0);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          u[i].w[0][j] = __builtin_amdgcn_alignbyte(j < 3 ? w[j + 1] : last, w[j], at & 2) & keep[j];
      } else {
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const u32x4 w = __builtin_amdgcn_raw_buffer_load_b128(rsrc, at + 16 * q, 0, 0);
#pragma unroll
          for (int j = 0; j < 4; ++j) u[i].w[q][j] = w[j] & keep[4 * q + j];
        }
      }
    }
  }
}

template <typename T, int C, int D>
__device__ __forceinline__ void store_unit(char* image, const Unit<T>& u, int row, int piece) {
  if constexpr (parts_of<T>() == 1) {
    *reinterpret_cast<u32x4*>(image + image_at<C, D>(0, row, piece)) = u.w[0];
  } else {
    typedef Vec<T, 8> V8;
    const V8 x = __builtin_bit_cast(V8, u);
    float f[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = to_f(x.v[i]);
    u32x4 parts[parts_of<T>()];
    split8<parts_of<T>()>(f, parts);
#pragma unroll
    for (int n = 0; n < parts_of<T>(); ++n)
      *reinterpret_cast<u32x4*>(image + image_at<C, D>(n, row, piece)) = parts[n];
  }
}

// An operand of a product over the channels: lane l holds row 32 tile + l % 32,
// channels 16 s + 8 (l / 32) .. + 7.  `at`: row_base plus the image's offset (a
// multiple of a row's bytes, so that the pieces' bits can be exchanged in it).
template <int D>
__device__ __forceinline__ uint32_t row_base(int lane) {
  const int row = lane & 31;
  return (uint32_t)(row * D * 2 + (((lane >> 5) ^ swizzle<D>(row)) << 4));
}
template <int C, int D>
__device__ __forceinline__ u32x4 row_operand(const char* lds, uint32_t at, int part, int tile, int s) {
  return *reinterpret_cast<const u32x4*>(lds + (at ^ (uint32_t)(s << 5)) +
                                         (part * C + 32 * tile) * D * 2);
}

// An operand of a product over the tokens: lane l holds a channel, and of the
// tokens 16 s .. 16 s + 15 those that a 32 x 32 accumulator's registers 8 s' ..
// 8 s' + 7 are rows of: 16 s + 4 (l / 32) + 0 .. 3 and the same plus 8.  Each of
// the two reads turns a block of 4 tokens x 16 channels: lane l % 16 passes the
// address of token (l % 16) / 4, channels 4 (l % 4) .. + 3 and gets channel
// l % 16 of the four tokens.  `turned`: the channels in the order in which the
// rows of an accumulator are contiguous for the lanes (below at S).
template <int D>
__device__ __forceinline__ uint32_t token_base(int lane, bool turned) {
  const int four = lane & 3, block = turned ? ((four & 1) << 1) | (four >> 1) : four;
  const int row = 4 * (lane >> 5) + ((lane & 15) >> 2), piece = 2 * ((lane >> 4) & 1) + (block >> 1);
  return (uint32_t)(row * D * 2 + ((piece ^ swizzle<D>(row)) << 4) + (block & 1) * 8);
}
template <int C, int D>
__device__ __forceinline__ u32x4 token_operand(const char* lds, uint32_t at, int part, int tile, int s) {
  u32x4 r;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    // swizzle(row + 8) = swizzle(row) ^ 2; of 16 rows on it is the same
    const char* p = lds + (at ^ (uint32_t)((tile << 6) | (e << 5))) + (part * C + 16 * s + 8 * e) * D * 2;
    const u32x2 t = __builtin_bit_cast(
        u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)p));
    r[2 * e] = t[0];
    r[2 * e + 1] = t[1];
  }
  return r;
}

// The compiler moves nothing across.
__device__ __forceinline__ void step() { __builtin_amdgcn_sched_barrier(0); }

// The same value in every lane, kept in scalar registers.
__device__ __forceinline__ int64_t uniform(int64_t x) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane((int)(uint32_t)x);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((int)(uint32_t)((uint64_t)x >> 32));
  return (int64_t)(((uint64_t)hi << 32) | lo);
}

// The outputs of one wave: acc[qt] holds 32 columns of the values (rows of the
// accumulator) of 32 queries (its columns, 32 qt + lane % 32).  `op`: the
// workgroup's first column of the chunk's first row, rows `stride` apart; rows
// from n on and columns from dvs on are left alone.
template <typename T, int CT, bool VEC>
__device__ __forceinline__ void store_columns(const f16v* acc, T* op, int n, int dvs, int64_t stride,
                                              int wave) {
  const int lane = threadIdx.x & 63, hi = lane >> 5, col = lane & 31;
  if constexpr (VEC) {
    // rows from n on and columns from dvs on: out of the buffer's range
    const int st = (int)stride * (int)sizeof(T);
    const __amdgpu_buffer_rsrc_t ro =
        rows_rsrc(op, (uint32_t)((n - 1) * st + dvs * (int)sizeof(T)));
    auto at = [&](int i, int c) {
      return c < dvs ? (uint32_t)(i * st + c * (int)sizeof(T)) : OOB;
    };
#pragma unroll
    for (int qt = 0; qt < CT; ++qt) {
      const int i = 32 * qt + col;
      if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          Vec<T, 4> y;
#pragma unroll
          for (int j = 0; j < 4; ++j) y.v[j] = acc[qt][4 * g + j];
          __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, y), ro,
                                                 at(i, 32 * wave + 8 * g + 4 * hi), 0, 0);
        }
      } else {
        // both halves of the wave exchange quads: eight columns a lane
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          uint32_t x[2], y[2];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            Vec<T, 2> lo, up;
            lo.v[0] = from_f<T>(acc[qt][8 * g + 2 * j]);
            lo.v[1] = from_f<T>(acc[qt][8 * g + 2 * j + 1]);
            up.v[0] = from_f<T>(acc[qt][8 * g + 4 + 2 * j]);
            up.v[1] = from_f<T>(acc[qt][8 * g + 4 + 2 * j + 1]);
            const auto sw = __builtin_amdgcn_permlane32_swap(
                __builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, up), false, false);
            x[j] = sw[0];
            y[j] = sw[1];
          }
          const u32x4 out = {x[0], x[1], y[0], y[1]};
          __builtin_amdgcn_raw_buffer_store_b128(out, ro, at(i, 32 * wave + 16 * g + 8 * hi), 0,
                                                 0);
        }
      }
    }
  } else {
#pragma unroll
    for (int qt = 0; qt < CT; ++qt) {
      const int i = 32 * qt + col;
      T* const orow = op + i * stride + 32 * wave;
      if (i < n) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int c = 8 * (r >> 2) + 4 * hi + (r & 3);
          if (32 * wave + c < dvs) orow[c] = from_f<T>(acc[qt][r]);
        }
      }
    }
  }
}

}  // namespace
