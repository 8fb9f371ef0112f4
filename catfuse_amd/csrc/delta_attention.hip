// Softmax-free causal attention whose state fades and corrects itself, over
// whole sequences:
//   S_t = w_t S_{t-1} + k_t u_t^T,  u_t = beta_t (v_t - w_t S_{t-1}^T k_t),
//   o_t = scale q_t S_t,            w_t = exp(log_decay_t)
// per sequence and head, S a dk x dv matrix in fp32; beta and log_decay are each
// token's and head's own.
//
// By chunks of C tokens (t, s the places in a chunk, S the state before it, g_t
// the sum of the chunk's log decays up to t):
//   u_t + sum_{s < t} L_ts u_s = r_t,   L_ts = beta_t e^(g_t - g_s) (k_t . k_s)
//   r_t = beta_t (v_t - e^(g_t) S^T k_t)
//   o_t = scale (e^(g_t) q_t S + sum_{s <= t} e^(g_t - g_s) (q_t . k_s) u_s)
//   S  <- e^(g_end) S + sum_s e^(g_end - g_s) k_s u_s^T
// T = (I + L)^-1 does not depend on the state: delta_solve_kernel makes it for
// all chunks side by side.  What is left for the walk over the chunks are
// products for the matrix cores.  Every power has an exponent of at most zero
// where the log decays have.
//
// Long sequences of few heads are walked in segments side by side.  A segment
// takes the state before it to  M S + N,  N what it makes of zeros and M what it
// makes of the unit matrix without values: the same walk on dv and on dk
// columns; delta_join_kernel goes from segment to segment.
//
// Precision as in decay_attention.hip: numbers that are not bf16 ones enter a
// product as parts of eight bits, products of parts below 2^-24 of the whole
// left out; sums of log decays in 64 bits, the powers that numbers enter and leave
// the state with to 2^-22; T by fp32 forward substitution and products of its blocks.
//
// No counterpart in the reference.
#include "cf_chunk.h"

namespace {

struct DeltaArgs {
  const void* q;
  const void* k;
  const void* v;
  const void* beta;
  const void* log_decay;
  const float* state_in;
  float* state_out;
  void* out;
  const void* cu;
  // workspace: rows that the sequences begin at and segments before them [seqs + 1]
  // each (packed ones); of each
  // chunk and head T, the running sums of its log decays and its betas; of each
  // segment and head N, later the state before it, and M
  int64_t* begins;
  int64_t* before;
  char* solved;
  double* falls;
  float* betas;
  float* own;
  float* moves;
  int cu_wide, beta_f32, decay_f32;
  int zero_rest;             // rows before the first sequence (1) and behind the last (2)
  int group;                 // a group of packed sequences: its rows begin at begins[0]
  int64_t seqs, tokens;      // tokens: rows in all (packed) or of each sequence
  int64_t chunks;            // numbers of chunks, some of none
  int64_t segment, segments; // tokens a segment (0: whole sequences); their numbers, some of none
  int heads, q_group, k_group, v_group, dk, dv, slices, value_slices;
  int64_t first;             // of the launch's pairs of a segment and a key head, or a chunk and a head
  int64_t qb, qt, qh, kb, kt, kh, vb, vt, vh, bb, bt, bh, lb, lt, lh, ob, ot, oh;
  int vec;                   // 16-byte accesses are aligned and whole, rows apart
  float scale;
};

// Chunks or segments of `unit` tokens, numbered through: the first one of a
// sequence has the number  seq + begin / unit  (equal rows: seq times those of
// a sequence), which is beyond all of the sequence before it, since
// ceil(len / unit) <= floor(len / unit) + 1, so that no sums over the
// sequences' lengths are needed.  An empty sequence has one.
__host__ __device__ inline int64_t units_of(int64_t tokens, int64_t unit) {
  return tokens > 0 ? (tokens + unit - 1) / unit : 1;
}

struct Place { int64_t seq, part, parts, begin, len, row0; };   // seq < 0: none has the number;
                                                                // row0: begins are counted from it

// The last of n for which first(i), which does not fall, is at most w, or -1: 64
// probes a time.
template <typename F>
__device__ __forceinline__ int64_t last_at_most(int64_t n, int64_t w, F first) {
  const int lane = threadIdx.x & 63;
  int64_t lo = 0;
  for (;;) {
    const int64_t step = (n + 63) / 64, i = lo + lane * step;
    const bool in = lane * step < n && first(lane * step < n ? i : lo) <= w;
    const uint64_t hit = __ballot(in);
    if (hit == 0) return -1;
    const int l = 63 - __clzll((long long)hit);
    lo = uniform(lo + l * step);
    n = uniform(n - l * step < step ? n - l * step : step);
    if (step == 1) return lo;
  }
}

// Packed sequences that a wave's lanes hold need no launch of their own before the
// others (5 to 6 us): each wave sorts out their offsets for itself (a.begins is
// null).  Not where the waves are many: of 3 prompts of 44 tokens in all, 12 heads
// of 32, 13 us instead of 17; chunks of 24 prompts of 24011 tokens and 16 heads
// solved in 70 us instead of 68, of one of 65536 and 32 heads in 315 instead of 305.
constexpr int64_t LANE_SEQS = 63, LANE_CHUNKS = 8192;

// Place w in a numbering of units: with gaps (above), without, or without the
// sequences' last ones; w becomes the number with gaps.
enum Numbers { GAPS, DENSE, INNER };
__device__ __forceinline__ Place place_in_lanes(const DeltaArgs& a, int64_t& w, int unit, Numbers numbers,
                                                int64_t* ends = nullptr) {
  const int lane = threadIdx.x & 63, seqs = (int)a.seqs;
  int begin = lane <= seqs ? (int)seq_offset(a.cu, a.cu_wide, lane, a.tokens) : 0;
  for (int d = 1; d < 64; d *= 2) {          // none below its predecessor
    const int o = __shfl_up(begin, d, 64);
    if (lane >= d && o > begin) begin = o;
  }
  if (ends != nullptr) {
    ends[0] = __builtin_amdgcn_readlane(begin, 0);
    ends[1] = __builtin_amdgcn_readlane(begin, seqs);
  }
  const int len = __shfl_down(begin, 1, 64) - begin;
  const int units = (int)(((unsigned)len + (unsigned)unit - 1u) / (unsigned)unit), own = len > 0 ? units : 1;
  int first = lane + (int)((unsigned)begin / (unsigned)unit);
  const int gaps = first;
  if (numbers != GAPS) {
    first = lane < seqs ? own - (numbers == INNER ? 1 : 0) : 0;
    const int mine = first;
    for (int d = 1; d < 64; d *= 2) {
      const int o = __shfl_up(first, d, 64);
      if (lane >= d) first += o;
    }
    first -= mine;
  }
  Place s;
  s.seq = -1;
  s.part = s.parts = s.begin = s.len = s.row0 = 0;
  const uint64_t hit = __ballot(lane < seqs && first <= w);
  if (hit == 0) return s;
  const int lo = 63 - __clzll((long long)hit);
  const int64_t part = w - __builtin_amdgcn_readlane(first, lo), parts = __builtin_amdgcn_readlane(own, lo);
  if (part >= parts - (numbers == INNER ? 1 : 0)) return s;
  s.seq = lo;
  s.part = part;
  s.parts = parts;
  s.begin = __builtin_amdgcn_readlane(begin, lo);
  s.len = __builtin_amdgcn_readlane(len, lo);
  w = __builtin_amdgcn_readlane(gaps, lo) + part;
  return s;
}

// ends: of packed sequences, the first one's first row and the row behind the last.
__device__ __forceinline__ Place find_place(const DeltaArgs& a, int64_t w, int64_t unit,
                                            int64_t* ends = nullptr) {
  if (a.cu != nullptr && a.begins == nullptr)
    return place_in_lanes(a, w, (int)(unit < INT32_MAX ? unit : INT32_MAX), GAPS, ends);
  Place s;
  s.row0 = 0;
  if (a.cu == nullptr) {
    s.parts = uniform(units_of(a.tokens, unit));
    s.seq = uniform(w / s.parts);
    s.part = uniform(w % s.parts);
    s.begin = 0;
    s.len = a.tokens;
    if (s.seq >= a.seqs) s.seq = -1;
    return s;
  }
  s.seq = -1;
  s.part = s.parts = s.begin = s.len = s.row0 = 0;
  const int64_t row0 = a.group ? a.begins[0] : 0;
  if (ends != nullptr) {
    ends[0] = a.begins[0];
    ends[1] = a.begins[a.seqs];
  }
  const int64_t lo = last_at_most(a.seqs, w, [&](int64_t i) { return i + (a.begins[i] - row0) / unit; });
  if (lo < 0) return s;
  const int64_t begin = uniform(a.begins[lo]), len = uniform(a.begins[lo + 1]) - begin;
  const int64_t part = uniform(w - (lo + (begin - row0) / unit)), parts = uniform(units_of(len, unit));
  if (part >= parts) return s;
  s.seq = lo;
  s.part = part;
  s.parts = parts;
  s.begin = begin;
  s.len = len;
  s.row0 = uniform(row0);
  return s;
}

// The walks' workgroups of packed segments: numbered without gaps (w becomes the
// segment's own number), all of them or, `inner`, those that are no sequence's
// last.  With the numbers' gaps among them, workgroups that end at once, the others
// spread unevenly: 16 packed sequences of 700 tokens, 8 heads of 256 channels, in
// one segment each took 330 us, and take 194.
__device__ __forceinline__ Place find_segment(const DeltaArgs& a, int64_t& w, bool inner) {
  if (a.cu == nullptr || a.segment == 0) return find_place(a, w, a.segment > 0 ? a.segment : INT64_MAX / 2);
  if (a.begins == nullptr) return place_in_lanes(a, w, (int)a.segment, inner ? INNER : DENSE);
  Place s;
  s.seq = -1;
  s.part = s.parts = s.begin = s.len = s.row0 = 0;
  if (w >= uniform(a.before[a.seqs]) - (inner ? a.seqs : 0)) return s;
  s.seq = last_at_most(a.seqs, w, [&](int64_t i) { return a.before[i] - (inner ? i : 0); });
  s.begin = uniform(a.begins[s.seq]);
  s.len = uniform(a.begins[s.seq + 1]) - s.begin;
  s.part = uniform(w - (a.before[s.seq] - (inner ? s.seq : 0)));
  s.parts = uniform(units_of(s.len, a.segment));
  w = uniform(s.seq + s.begin / a.segment + s.part);
  return s;
}

// The rows that packed sequences begin at: the offsets clamped to the tensors'
// rows, each at least its predecessor; and the segments of those before.  One
// workgroup.
__global__ __launch_bounds__(1024) void delta_begins_kernel(DeltaArgs a) {
  __shared__ int64_t top_sh[2][16];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int64_t before = 0;
  int odd = 0;
  for (int64_t i0 = 0; i0 <= a.seqs; i0 += 1024, odd ^= 1) {
    const int64_t i = i0 + tid;
    int64_t m = i <= a.seqs ? seq_offset(a.cu, a.cu_wide, i, a.tokens) : 0;
    for (int d = 1; d < 64; d *= 2) {
      const int64_t o = __shfl_up(m, d, 64);
      if (lane >= d && o > m) m = o;
    }
    if (lane == 63) top_sh[odd][wave] = m;
    __syncthreads();
    if (before > m) m = before;
    for (int w = 0; w < 16; ++w) {
      const int64_t o = top_sh[odd][w];
      if (w < wave && o > m) m = o;
      if (o > before) before = o;
    }
    if (i <= a.seqs) a.begins[i] = m;
  }
  if (a.segment == 0) return;
  __syncthreads();                           // all begins are written, the tops read
  before = 0;
  odd = 0;
  for (int64_t i0 = 0; i0 <= a.seqs; i0 += 1024, odd ^= 1) {
    const int64_t i = i0 + tid;
    const int64_t own = i < a.seqs ? units_of(a.begins[i + 1] - a.begins[i], a.segment) : 0;
    int64_t m = own;
    for (int d = 1; d < 64; d *= 2) {
      const int64_t o = __shfl_up(m, d, 64);
      if (lane >= d) m += o;
    }
    if (lane == 63) top_sh[odd][wave] = m;
    __syncthreads();
    m += before - own;
    for (int w = 0; w < 16; ++w) {
      const int64_t o = top_sh[odd][w];
      if (w < wave) m += o;
      before += o;
    }
    if (i <= a.seqs) a.before[i] = m;
  }
}

// 2^x to about an ulp, whatever x is: rounded to fp32 alone, x of 16 to 24 would be
// 6.6e-7 of the power off, and every number that goes into the state or comes out of
// it has such a factor.  (A power beyond fp32, or below it, is one.)
__device__ __forceinline__ float power_of_two(double x) {
  const float y = (float)x, e = __builtin_amdgcn_exp2f(y);
  return __builtin_fabsf(y) < 126.0f ? __builtin_fmaf(e, (float)(x - (double)y) * 0.693147182f, e) : e;
}

// T of one chunk and head.  In the workspace T lies as the walk's operands: for
// each tile of 32 x 32 that is not above the diagonal ((0,0) (1,0) (1,1)), each half
// of its columns and each of three parts the eight numbers of each lane: row
// lane % 32, columns 4 (lane / 32) + 0 .. 3 and the same plus 8 of the half's sixteen.
//
// The products k_t . k_s on the matrix cores; blocks of 16 inverted column by
// column in registers, then joined in pairs by fp32 matrix instructions:
//   (A 0; B D)^-1 = (A^-1 0; -D^-1 B A^-1 D^-1).
// L's powers, and the scores' in the walk, are of single floats: rounding x moves 2^x
// by up to |x| 2^-24 ln 2 of itself, and as x is below zero by 0.4 x 2^-24 of a weight
// of one at most.
// Rows of L from the first one that is not finite on are left out, and of T NaN; so are
// those of T from the first row of a B A^-1 on that is not: a product with the zeros
// of D^-1 would make NaN of the rows before it.
// Bound by the substitution's chain of dependent steps and by T's bytes (300 a token
// and head of C = 64, 2.0 TB/s): 65536 tokens x 32 heads of 128 bf16 channels 310 us.
template <int C> constexpr int solved_size() { return (C / 32) * (C / 32 + 1) / 2 * 6144; }   // bytes

typedef float f4v __attribute__((ext_vector_type(4)));

//
// Rows of no sequence are set to zeros here, a part by every workgroup: 1000 tokens of
// 16 heads of 128 bf16 channels in 65536 rows take 150 us (118 into a given output), by
// the walks' first and last workgroups alone 1260.
template <typename T, int NT, bool VEC>
__device__ __forceinline__ void clear_rest(const DeltaArgs& a, int64_t w, int h, const int64_t* ends) {
  constexpr int PER = VEC ? 16 / (int)sizeof(T) : 1;
  const int64_t front = a.zero_rest & 1 ? ends[0] : 0, rest = front + (a.zero_rest & 2 ? a.tokens - ends[1] : 0);
  if (w >= rest) return;
  const int units = a.dv / PER;              // of a row
  const int64_t count = ((rest - w + a.chunks - 1) / a.chunks) * units;
  for (int64_t i = threadIdx.x; i < count; i += NT) {
    const int64_t r = w + i / units * a.chunks, t = r < front ? r : ends[1] + (r - front);
    *reinterpret_cast<Vec<T, PER>*>((T*)a.out + t * a.ot + h * a.oh + i % units * PER) = Vec<T, PER>{};
  }
}

template <typename T, int DKP, int C, int NT, bool VEC>
__global__ __launch_bounds__(NT) void delta_solve_kernel(DeltaArgs a) {
  constexpr int NL = parts_of<T>(), NP = 3, KS = DKP / 16, CT = C / 32, TILES = CT * (CT + 1) / 2;
  constexpr int P = C + 4;
  constexpr int IMAGE = NL * C * DKP * 2, INVERSE = C * P * 4;
  // K's image, after the products the inverse
  __shared__ __attribute__((aligned(512))) char lds[IMAGE > INVERSE ? IMAGE : INVERSE];
  __shared__ __attribute__((aligned(16))) float low[C * P];
  __shared__ double fall[C];
  __shared__ float beta[C];
  __shared__ int bad_sh;
  float* const inv = reinterpret_cast<float*>(lds);
  const int tid = threadIdx.x, lane = tid & 63, hi = lane >> 5, col = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

  const int64_t pair = a.first + blockIdx.x;
  const int64_t w = uniform(pair / a.heads);
  const int h = (int)(pair - w * a.heads);
  int64_t ends[2] = {0, a.tokens};
  const Place pl = find_place(a, w, C, ends);
  if (a.cu != nullptr && a.zero_rest) clear_rest<T, NT, VEC>(a, w, h, ends);
  if (pl.seq < 0 || pl.len == 0) return;
  const int64_t row0 = a.cu != nullptr ? 0 : pl.seq, begin = pl.begin + pl.part * C;
  const int n = (int)(pl.len - pl.part * C < C ? pl.len - pl.part * C : C);

  constexpr int UK = C * (DKP / 8) / NT;
  static_assert(UK * NT == C * (DKP / 8), "whole units");
  Unit<T> ku[UK];
  load_units<T, UK, DKP, NT, VEC>(ku, (const T*)a.k + row0 * a.kb + begin * a.kt + (h / a.k_group) * a.kh,
                                  n, a.kt, a.dk);
  if (tid < C) {
    double g = 0.0;
    float b = 0.0f;
    if (tid < n) {
      if (a.log_decay != nullptr)
        g = load_double<T>(a.log_decay, row0 * a.lb + (begin + tid) * a.lt + h * a.lh, a.decay_f32);
      b = (float)load_double<T>(a.beta, row0 * a.bb + (begin + tid) * a.bt + h * a.bh, a.beta_f32);
    }
    // in powers of two; -inf (only the token itself is kept) as one whose sums
    // and differences are numbers and whose power is zero
    g = g < -1e4 ? -1e4 : g;
    g *= 1.44269504088896340736;
    for (int d = 1; d < C; d *= 2) {
      const double o = __shfl_up(g, d, 64);
      if (tid >= d) g += o;
    }
    fall[tid] = g;
    beta[tid] = b;
    a.falls[pair * C + tid] = g;
    a.betas[pair * C + tid] = b;
  }
  if (tid == 0) bad_sh = C;
#pragma unroll
  for (int i = 0; i < UK; ++i) {
    const int u = tid + NT * i;
    store_unit<T, C, DKP>(lds, ku[i], u / (DKP / 8), u % (DKP / 8));
  }
  __syncthreads();

  const uint32_t at_row = row_base<DKP>(lane);
  for (int tile = wave; tile < TILES; tile += NT / 64) {
    const int tt = tile == 0 ? 0 : 1, ts = tile == 2 ? 1 : 0;
    f16v acc = {};
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      u32x4 x[NL], y[NL];
#pragma unroll
      for (int p = 0; p < NL; ++p) {
        x[p] = row_operand<C, DKP>(lds, at_row, p, tt, s);
        y[p] = row_operand<C, DKP>(lds, at_row, p, ts, s);
      }
#pragma unroll
      for (int i = 0; i < NL; ++i)
#pragma unroll
        for (int j = 0; j < NL; ++j)
          if (i + j < (NL == 1 ? 1 : NP)) acc = mfma(x[i], y[j], acc);
    }
    const int s = 32 * ts + col;
    const double gs = fall[s];
    float z = 0.0f;                          // NaN if any is not finite
    int bad = C;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int t = 32 * tt + 8 * (r >> 2) + 4 * hi + (r & 3);
      const float f = beta[t] * __builtin_amdgcn_exp2f((float)(fall[t] - gs));
      const float x = t > s ? f * acc[r] : 0.0f;
      low[t * P + s] = x;
      z = __builtin_fmaf(x, 0.0f, z);
      bad = !(__builtin_fabsf(x) < __builtin_inff()) && t < bad ? t : bad;
    }
    if (__ballot(z != z) != 0) atomicMin(&bad_sh, bad);
  }
  __syncthreads();
  const int bad_from = bad_sh;
  if (bad_from < C) {
    for (int i = tid; i < (C - bad_from) * C; i += NT) low[(bad_from + i / C) * P + i % C] = 0.0f;
    __syncthreads();
  }

  // Blocks of 16: thread = block and column.  x_t takes what the earlier ones
  // leave of it as soon as each is known.
  if (tid < C) {
    const int b0 = tid & ~15, c = tid & 15;
    float x[16];
#pragma unroll
    for (int t = 0; t < 16; ++t) x[t] = t == c ? 1.0f : 0.0f;
    Vec<float, 4> l[16];
#pragma unroll
    for (int s = 0; s < 15; ++s) {
      if (s % 4 == 0) {
#pragma unroll
        for (int t = 1; t < 16; ++t)
          if (t > s) l[t] = *reinterpret_cast<const Vec<float, 4>*>(low + (b0 + t) * P + b0 + s);
      }
#pragma unroll
      for (int t = 1; t < 16; ++t)
        if (t > s) x[t] = __builtin_fmaf(-l[t].v[s % 4], x[s], x[t]);
    }
#pragma unroll
    for (int t = 0; t < 16; ++t) inv[(b0 + t) * P + b0 + c] = x[t];
  } else if (C > 32) {
    // the blocks above them in the pairs' upper left and lower right
    for (int i = tid - C; i < 512; i += NT - C)
      inv[(i / 256 * 32 + i % 256 / 16) * P + i / 256 * 32 + 16 + i % 16] = 0.0f;
  }
  __syncthreads();
  const int c16 = lane & 15, q16 = lane >> 4;
  // a B A^-1, rows row .. + 3: whether all of it is finite; those numbers that are not out
  auto finite = [&](const f4v& m) {
    const float z = __builtin_fmaf(m[0], 0.0f, m[1] * 0.0f) + __builtin_fmaf(m[2], 0.0f, m[3] * 0.0f);
    return __ballot(z != z) == 0;
  };
  auto keep_finite = [&](f4v& m, int row) {
#pragma unroll
    for (int j = 3; j >= 0; --j)
      if (!(__builtin_fabsf(m[j]) < __builtin_inff())) {
        atomicMin(&bad_sh, row + j);
        m[j] = 0.0f;
      }
  };
  // pairs of 16: B A^-1 (its accumulators are the next product's operand as they
  // lie, if that takes its inner indices 4 q16 + j), then -D^-1 times it
  if (wave < C / 32) {
    const int b0 = 32 * wave;
    f4v m = {}, y;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int k = 4 * j + q16;
      m = __builtin_amdgcn_mfma_f32_16x16x4f32(low[(b0 + 16 + c16) * P + b0 + k],
                                               inv[(b0 + k) * P + b0 + c16], m, 0, 0, 0);
    }
    auto times_m = [&]() {
      y = f4v{};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        y = __builtin_amdgcn_mfma_f32_16x16x4f32(inv[(b0 + 16 + c16) * P + b0 + 16 + 4 * q16 + j], m[j], y,
                                                 0, 0, 0);
    };
    times_m();
    if (!finite(m)) {
      keep_finite(m, b0 + 16 + 4 * q16);
      times_m();
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) inv[(b0 + 16 + 4 * q16 + j) * P + b0 + c16] = -y[j];
  }
  __syncthreads();
  if constexpr (C > 32) {
    // the pair of 32: wave = 16 rows (i) and 16 columns (j) of its lower left block
    const int i0 = 32 + 16 * (wave & 1), j0 = 16 * (wave >> 1);
    f4v m[2] = {{}, {}}, y;
#pragma unroll
    for (int k0 = 0; k0 < 32; k0 += 4) {
      const float x = inv[(k0 + q16) * P + j0 + c16];
#pragma unroll
      for (int e = 0; e < 2; ++e)
        m[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(low[(32 + 16 * e + c16) * P + k0 + q16], x, m[e],
                                                    0, 0, 0);
    }
    auto times_m = [&]() {
      y = f4v{};
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          y = __builtin_amdgcn_mfma_f32_16x16x4f32(inv[(i0 + c16) * P + 32 + 16 * e + 4 * q16 + j], m[e][j],
                                                   y, 0, 0, 0);
    };
    times_m();
    if (!finite(m[0]) || !finite(m[1])) {
#pragma unroll
      for (int e = 0; e < 2; ++e) keep_finite(m[e], 32 + 16 * e + 4 * q16);
      times_m();
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) inv[(i0 + 4 * q16 + j) * P + j0 + c16] = -y[j];
    __syncthreads();
  }

  const int nan_from = bad_sh;
  char* const to = a.solved + pair * solved_size<C>();
  for (int u = tid; u < TILES * 128; u += NT) {
    const int tile = u >> 7, half = (u >> 6) & 1, l = u & 63;
    const int t = 32 * (tile == 0 ? 0 : 1) + (l & 31);
    const int s0 = 32 * (tile == 2 ? 1 : 0) + 16 * half + 4 * (l >> 5);
    float x[8];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const Vec<float, 4> y = *reinterpret_cast<const Vec<float, 4>*>(inv + t * P + s0 + 8 * e);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float z = t >= nan_from ? __builtin_nanf("") : y.v[j];
        x[4 * e + j] = s0 + 8 * e + j <= t ? z : 0.0f;
      }
    }
    u32x4 parts[NP];
    split8<NP>(x, parts);
#pragma unroll
    for (int p = 0; p < NP; ++p)
      *reinterpret_cast<u32x4*>(to + (((u >> 6) * NP + p) * 64 + l) * 16) = parts[p];
  }
}

// The walk.  A workgroup takes a segment of a sequence, one head, 32 NW columns
// of the values; wave w the columns 32 w .. + 31 with their part of S (all DKP
// rows, in accumulators) throughout: a column of u, r and S depends on no other
// column, so the waves share only the chunk's images.  OUT: outputs, from the
// state before the segment; else the segment's N (slices of the values) and M
// (further slices: columns of the unit matrix, no values).
//
// S as accumulators: tile t, register r of a lane is row (channel of k)
// 32 t + 16 (r / 8) + 8 (lane / 32) + r % 8, column lane % 32 (the rows of K's
// operand are taken in that order): eight registers on end are an operand of the
// next products as they lie.  So are eight registers of r and u, tokens
// 16 s + 4 (lane / 32) + 0 .. 3 and the same plus 8, the order in which T, the
// scores and K's turned operand have them.
//
// Bound by the issue of matrix and vector operations by turns, and by the card's
// power: 65536 tokens x 32 heads of 128 bf16 channels in 16 segments, outputs 990 us
// and states 1010 (matrix cores 47 and 53 %, vector issue 44 and 54 %, LDS 18 % of the
// cycles, the clock at 1.8 GHz).  Two workgroups of four waves a CU; chunks of 64 halve
// the products with the state's parts against 32, for which only bf16 heads of 65 to
// 128 channels have the registers.
template <typename T, int DKP, int NW, int C, bool OUT, bool VEC>
__global__ __launch_bounds__(64 * NW, DKP <= 128 ? 2 : 1)
void delta_walk_kernel(DeltaArgs a) {
  constexpr int NL = parts_of<T>(), NP = 3, NT = 64 * NW;
  // operands read ahead: one set; none of three parts, whose products take long
  // enough and whose registers would cost the second workgroup of a CU
  constexpr int AHEAD = NL == 3 ? 0 : 1, SETS = AHEAD + 1;
  constexpr int KT = DKP / 32, KS = DKP / 16, CT = C / 32, CS = C / 16, DVW = 32 * NW;
  constexpr int QK_BYTES = NL * C * DKP * 2, V_BYTES = NL * C * DVW * 2;
  constexpr int TILES = CT * (CT + 1) / 2, T_BYTES = TILES * 2 * NP * 1024;
  static_assert(CT == 1 || NW >= TILES, "a score tile a wave");
  constexpr int Q_AT = QK_BYTES, V_AT = Q_AT + (OUT ? QK_BYTES : 0), IMAGE = V_AT + V_BYTES;
  __shared__ __attribute__((aligned(512))) char lds[IMAGE];     // of K, Q and V
  __shared__ __attribute__((aligned(16))) char tsh[T_BYTES];    // T, later the scores
  // S is kept as 2^G times what is stored, G with the decays that went by: most
  // chunks then need not fade its numbers.
  __shared__ Vec<float, 2> fall_sh[C];       // a token's sum of log2 decays, of two floats
  // beta; beta 2^(G + fall); scale 2^(G + fall); 2^(G' - fall), G' after the chunk
  __shared__ __attribute__((aligned(16))) float beta_sh[C], since_sh[C], query_sh[C], end_sh[C];
  // what the numbers fade by (of two floats) if G is set back; whether; 2^G' (of two)
  __shared__ float fade_sh[5];

  const int tid = threadIdx.x, lane = tid & 63, hi = lane >> 5, col = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t t_lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)tsh;

  // Heads of one key head and the slices of their columns read the same rows:
  // consecutive workgroups of one XCD (workgroup number mod 8).
  const unsigned shared = (unsigned)(a.k_group * a.slices), k_heads = (unsigned)(a.heads / a.k_group);
  const unsigned slot = blockIdx.x >> 3;
  const int64_t super = a.first + slot / shared * 8 + (blockIdx.x & 7);
  const unsigned inner = slot % shared;
  int64_t w = uniform(super / k_heads);
  if (w >= a.segments) return;
  const int hk = (int)uniform(super % k_heads), h = hk * a.k_group + (int)(inner / (unsigned)a.slices);
  const int slice = (int)(inner % (unsigned)a.slices);
  const bool move = !OUT && slice >= a.value_slices;            // columns of M
  const int c0 = (move ? slice - a.value_slices : slice) * DVW, cols = move ? a.dk : a.dv;

  const Place pl = find_segment(a, w, !OUT);
  if (pl.seq < 0) return;
  const bool last = pl.part == pl.parts - 1;
  if (!OUT && last) return;                  // no segment reads it
  const int dvs = cols - c0 < DVW ? cols - c0 : DVW;            // columns of this slice
  const T *kp, *vp, *qp;
  T* op;
  int left;                                  // tokens from here to the segment's end
  int64_t pair;                              // of the chunk and the head
  {
    const int64_t tok0 = pl.part * a.segment, row0 = a.cu != nullptr ? 0 : pl.seq;
    const int64_t begin = pl.begin + tok0, rest = pl.len - tok0;
    left = (int)(a.segment > 0 && rest > a.segment ? a.segment : rest);
    qp = (const T*)a.q + row0 * a.qb + begin * a.qt + (h / a.q_group) * a.qh;
    kp = (const T*)a.k + row0 * a.kb + begin * a.kt + hk * a.kh;
    vp = (const T*)a.v + row0 * a.vb + begin * a.vt + (h / a.v_group) * a.vh + (move ? 0 : c0);
    op = (T*)a.out + row0 * a.ob + begin * a.ot + h * a.oh + c0;
    const int64_t chunk = tok0 / C + (a.cu != nullptr ? pl.seq + (pl.begin - pl.row0) / C
                                                      : pl.seq * units_of(a.tokens, C));
    pair = uniform(chunk * a.heads + h);
  }

  f16v S[KT];
#pragma unroll
  for (int t = 0; t < KT; ++t) S[t] = f16v{};
  const int sc = 32 * wave + col;            // this lane's column of the slice
  // this lane's place in a state (or M): of its first row; the others are cols
  // apart, rows from dk on and columns from dvs on out of the buffer's range
  const uint32_t s_at = sc < dvs ? 4u * (uint32_t)(8 * hi * cols + c0 + sc) : OOB;
  auto s_off = [&](int t, int r) {
    return s_at + 4u * (uint32_t)((32 * t + 16 * (r >> 3) + (r & 7)) * cols);
  };
  auto state_of = [&](const float* base, int64_t i) {
    return rows_rsrc(base + (i * a.heads + h) * (int64_t)a.dk * cols, 4u * a.dk * cols);
  };
  if (OUT) {
    const float* const from = pl.part > 0 ? a.own : a.state_in;
    if (from != nullptr) {
      const __amdgpu_buffer_rsrc_t rs = state_of(from, pl.part > 0 ? w : pl.seq);
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          S[t][r] = __builtin_bit_cast(
              float, __builtin_amdgcn_raw_buffer_load_b32(rs, s_off(t, r), 0, 0));
    }
  } else if (move) {
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        S[t][r] = 32 * t + 16 * (r >> 3) + 8 * hi + (r & 7) == c0 + sc ? 1.0f : 0.0f;
  }

  constexpr int UK = C * (DKP / 8) / NT, UV = C * (DVW / 8) / NT;   // units of a thread
  static_assert(UK * NT == C * (DKP / 8) && UV * NT == C * (DVW / 8), "whole units");
  // T: with the keys where registers are free (the products before it is read are
  // few there, too few to hide its way), else straight to LDS
  constexpr bool T_AHEAD = CT == 1;
  constexpr int UT = T_AHEAD ? (T_BYTES / 16 + NT - 1) / NT : 1;
  auto unit = [&](int i) { return (tid + NT * i) % (T_BYTES / 16); };   // (some twice)
  u32x4 tu[UT];
  Unit<T> ku[UK], vu[UV], qu[OUT ? UK : 1];
  double fall = 0.0, gone = 0.0;             // (G: wave 0's)
  float beta = 0.0f;
  // The next chunk's rows; behind the last chunk the segment's first row again, so
  // that no load is conditional: the registers of one that is not made would stay
  // taken from one chunk to the next.
  const T *const k_first = kp, *const v_first = vp, *const q_first = qp;
  const int64_t pair_first = pair;
  auto rows = [&]() { return left >= C ? C : left > 0 ? left : 1; };
  auto load_keys = [&]() {
    load_units<T, UK, DKP, NT, VEC>(ku, left > 0 ? kp : k_first, rows(), a.kt, a.dk);
    const int64_t at = left > 0 ? pair : pair_first;
    if constexpr (T_AHEAD)
#pragma unroll
      for (int i = 0; i < UT; ++i)
        tu[i] = *reinterpret_cast<const u32x4*>(a.solved + at * solved_size<C>() + unit(i) * 16);
    fall = a.falls[at * C + tid % C];
    beta = a.betas[at * C + tid % C];
  };
  auto load_values = [&]() {
    if (OUT || !move) load_units<T, UV, DVW, NT, VEC>(vu, left > 0 ? vp : v_first, rows(), a.vt, dvs);
  };
  auto load_queries = [&]() {
    if constexpr (OUT) load_units<T, UK, DKP, NT, VEC>(qu, left > 0 ? qp : q_first, rows(), a.qt, a.dk);
  };
  if (!OUT && move)
#pragma unroll
    for (int i = 0; i < UV; ++i) vu[i] = Unit<T>{};

  uint32_t at_row = row_base<DKP>(lane), at_key = token_base<DKP>(lane, true);
  uint32_t at_value = token_base<DVW>(lane, false) ^ (uint32_t)(wave << 6);

  if (left > 0) {
    load_keys();
    load_values();
    load_queries();
  }
  while (left > 0) {
    // opaque: the places derived from them, kept over the chunks, cost more
    // registers than there are
    asm volatile("" : "+v"(at_row), "+v"(at_key), "+v"(at_value));
    const int n = left < C ? left : C;
    __syncthreads();                         // the last chunk's images are read
    if constexpr (T_AHEAD) {
#pragma unroll
      for (int i = 0; i < UT; ++i) *reinterpret_cast<u32x4*>(tsh + unit(i) * 16) = tu[i];
    } else {                                 // landed before it is read
      const i32x4 from = buffer_of(a.solved + pair * solved_size<C>(), T_BYTES);
      for (int i = wave; i < T_BYTES / 1024; i += NW)
        copy16(from, (uint32_t)(lane * 16), (uint32_t)(i * 1024), t_lds + i * 1024);
    }
#pragma unroll
    for (int i = 0; i < UK; ++i) {
      const int u = tid + NT * i, row = u / (DKP / 8), piece = u % (DKP / 8);
      store_unit<T, C, DKP>(lds, ku[i], row, piece);
      if constexpr (OUT) store_unit<T, C, DKP>(lds + Q_AT, qu[i], row, piece);
    }
#pragma unroll
    for (int i = 0; i < UV; ++i) {
      const int u = tid + NT * i, row = u / (DVW / 8), piece = u % (DVW / 8);
      store_unit<T, C, DVW>(lds + V_AT, vu[i], row, piece);
    }
    if (wave == 0) {                         // lane: token lane % C; no lane is masked off
      const double x = fall + gone, end = __shfl(x, C - 1, 64);
      const bool fold = __ballot(!(__builtin_fabs(x) <= 24.0)) == 0;
      const float e = power_of_two(x), high = (float)fall;
      fall_sh[lane % C] = {high, (float)(fall - (double)high)};
      beta_sh[lane % C] = beta;
      since_sh[lane % C] = beta * e;
      query_sh[lane % C] = a.scale * e;
      end_sh[lane % C] = power_of_two(fold ? -x : end - x);
      gone = fold ? end : 0.0;
      auto two = [&](float* to, double f) {
        to[0] = (float)f;
        to[1] = f < 1e300 ? (float)(f - (double)to[0]) : 0.0f;
      };
      two(fade_sh, exp2(end));
      fade_sh[2] = fold ? 1.0f : 0.0f;
      two(fade_sh + 3, exp2(gone));
    }
    __syncthreads();
    left -= n;
    kp += C * a.kt;
    vp += C * a.vt;
    qp += C * a.qt;
    pair += a.heads;

    // In what follows the operands of the next products are read, and made, between
    // the products at hand, and the compiler is held to that order (step()).

    // r = beta v - beta e^g (K S), rows tokens;  O^T = S^T Q^T, rows columns of
    // the values: both of S's parts.
    f16v R[CT], O[OUT ? CT : 1];
    {
      u32x4 sp[SETS][NP], ky[SETS][CT][NL], qy[OUT ? SETS : 1][CT][NL];
      auto state_part = [&](int s) {
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = S[s / 2][8 * (s & 1) + j];
        split8<NP>(x, sp[s % SETS]);
      };
      auto read = [&](int s) {
#pragma unroll
        for (int t = 0; t < CT; ++t)
#pragma unroll
          for (int p = 0; p < NL; ++p) {
            ky[s % SETS][t][p] = row_operand<C, DKP>(lds, at_row, p, t, s);
            if constexpr (OUT) qy[s % SETS][t][p] = row_operand<C, DKP>(lds + Q_AT, at_row, p, t, s);
          }
      };
      if (AHEAD) {
        read(0);
        state_part(0);
      }
#pragma unroll
      for (int t = 0; t < CT; ++t) {
        R[t] = f16v{};
        if constexpr (OUT) O[t] = f16v{};
      }
      if (AHEAD) step();
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        if (s + AHEAD < KS) {
          read(s + AHEAD);
          state_part(s + AHEAD);
        }
#pragma unroll
        for (int p = 0; p < NP; ++p)
#pragma unroll
          for (int l = 0; l < NL; ++l)
#pragma unroll
            for (int t = 0; t < CT; ++t)
              if (p + l < NP) {
                R[t] = mfma(ky[s % SETS][t][l], sp[s % SETS][p], R[t]);
                if constexpr (OUT) O[t] = mfma(sp[s % SETS][p], qy[s % SETS][t][l], O[t]);
              }
        if (AHEAD) step();
      }
    }
    if constexpr (OUT) {
#pragma unroll
      for (int t = 0; t < CT; ++t) {
        const float f = query_sh[32 * t + col];
#pragma unroll
        for (int r = 0; r < 16; ++r) O[t][r] *= f;
      }
    }

    // u = T r, sixteen tokens of r at a time, made while those before are multiplied.
    //
    // A value that is not finite would give NaN wherever it meets a zero of T or
    // of the scores: r and u are zeros from its token on, and what depends on them
    // set to NaN below: this lane's column, the queries from the token on and the
    // state.  (A k, beta or decay that is not finite shows in r too.  The segments'
    // own states keep it: there NaN goes its way.)
    int bad_from = C;
    bool any_bad = false;
    u32x4 rop[2][NP];                        // r, then u, as operands
    auto make_r = [&](int s) {
      u32x4 vop[NL];
#pragma unroll
      for (int p = 0; p < NL; ++p) vop[p] = token_operand<C, DVW>(lds + V_AT, at_value, p, 0, s);
      float x[8], z = 0.0f;                  // z: NaN if any is not finite
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const Vec<float, 4> b = *reinterpret_cast<const Vec<float, 4>*>(beta_sh + 16 * s + 8 * e + 4 * hi);
        const Vec<float, 4> f = *reinterpret_cast<const Vec<float, 4>*>(since_sh + 16 * s + 8 * e + 4 * hi);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float y = 0.0f;
#pragma unroll
          for (int p = 0; p < NL; ++p) {
            const uint32_t word = vop[p][2 * e + (j >> 1)];
            const float part = __builtin_bit_cast(float, j & 1 ? word & 0xffff0000u : word << 16);
            y = p == 0 ? part : y + part;
          }
          x[4 * e + j] = __builtin_fmaf(-f.v[j], R[s / 2][8 * (s & 1) + 4 * e + j], b.v[j] * y);
          if constexpr (OUT) z = __builtin_fmaf(x[4 * e + j], 0.0f, z);
        }
      }
      if constexpr (OUT) {
        any_bad = any_bad || __ballot(z != z) != 0;
        if (any_bad) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int tok = 16 * s + 8 * (j >> 2) + 4 * hi + (j & 3);
            bad_from = !(__builtin_fabsf(x[j]) < __builtin_inff()) && tok < bad_from ? tok : bad_from;
          }
          const int other = __shfl_xor(bad_from, 32, 64);
          bad_from = other < bad_from ? other : bad_from;
#pragma unroll
          for (int j = 0; j < 8; ++j)
            x[j] = 16 * s + 8 * (j >> 2) + 4 * hi + (j & 3) >= bad_from ? 0.0f : x[j];
        }
      }
      split8<NP>(x, rop[s & 1]);
    };
    // T's operands in LDS, later the scores' in their place: of the sixteen columns
    // s, the row tiles that are not above the diagonal
    u32x4 tile_op[CT][NP];
    auto rows_of = [&](int s) { return CT == 1 || s >= 2 ? 1 : 2; };
    auto read_tiles = [&](int s) {
#pragma unroll
      for (int t = 0; t < CT; ++t)
        if (t < rows_of(s)) {
          const int tile = s >= 2 ? 2 : t;
#pragma unroll
          for (int p = 0; p < NP; ++p)
            tile_op[t][p] = *reinterpret_cast<const u32x4*>(
                tsh + (((tile * 2 + (s & 1)) * NP + p) * 64 + lane) * 16);
        }
    };
    make_r(0);
    if constexpr (!T_AHEAD) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
    }
    f16v U[CT];
#pragma unroll
    for (int t = 0; t < CT; ++t) U[t] = f16v{};
    step();
#pragma unroll
    for (int s = 0; s < CS; ++s) {
      read_tiles(s);
      if (s + 1 < CS) make_r(s + 1);
#pragma unroll
      for (int p = 0; p < NP; ++p)
#pragma unroll
        for (int y = 0; y < NP; ++y)
#pragma unroll
          for (int t = 0; t < CT; ++t)
            if (p + y < NP && t < rows_of(s))
              U[s >= 2 ? 1 : t] = mfma(tile_op[t][p], rop[s & 1][y], U[s >= 2 ? 1 : t]);
      step();
    }

    if constexpr (OUT) {
      if (CT > 1) __syncthreads();           // T is read
      // Scores K Q^T of 32 keys (rows) x 32 queries (columns): eight registers
      // on end are an operand of U^T P^T as they lie.  One tile: every wave for
      // itself; three: a tile a wave, exchanged in LDS.
      u32x4 pop[2][NP];
      if (CT == 1 || wave < TILES) {
        const int qt = CT == 1 || wave == 0 ? 0 : 1, kt = CT > 1 && wave == 2 ? 1 : 0;
        u32x4 ak[SETS][NL], bq[SETS][NL];
        auto read = [&](int s) {
#pragma unroll
          for (int p = 0; p < NL; ++p) {
            ak[s % SETS][p] = row_operand<C, DKP>(lds, at_row, p, kt, s);
            bq[s % SETS][p] = row_operand<C, DKP>(lds + Q_AT, at_row, p, qt, s);
          }
        };
        if (AHEAD) read(0);
        f16v acc = {};
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          if (s + AHEAD < KS) read(s + AHEAD);
#pragma unroll
          for (int x = 0; x < NL; ++x)
#pragma unroll
            for (int y = 0; y < NL; ++y)
              if (x + y < (NL == 1 ? 1 : NP)) acc = mfma(ak[s % SETS][x], bq[s % SETS][y], acc);
          if (AHEAD) step();
        }
        const int i = 32 * qt + col;
        const Vec<float, 2> gi = fall_sh[i];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          float x[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int key = 32 * kt + 16 * s + 8 * (j >> 2) + 4 * hi + (j & 3);
            const Vec<float, 2> gk = fall_sh[key];
            const float f = __builtin_amdgcn_exp2f((gi.v[0] - gk.v[0]) + (gi.v[1] - gk.v[1]));
            const float y = acc[8 * s + j] * (a.scale * f);
            x[j] = i >= key ? y : 0.0f;
          }
          split8<NP>(x, pop[s]);
          if constexpr (CT > 1)
#pragma unroll
            for (int p = 0; p < NP; ++p)
              *reinterpret_cast<u32x4*>(tsh + (((wave * 2 + s) * NP + p) * 64 + lane) * 16) = pop[s][p];
        }
      }
      // A correction beyond fp32, of values that are not, is one of those.  (Looked for
      // here, behind the scores, where its products have long been done.)
      float z = 0.0f;
#pragma unroll
      for (int r = 0; r < 16; ++r)
#pragma unroll
        for (int t = 0; t < CT; ++t) z = __builtin_fmaf(U[t][r], 0.0f, z);
      any_bad = any_bad || __ballot(z != z) != 0;
      if (any_bad) {
#pragma unroll
        for (int t = 0; t < CT; ++t)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int tok = 32 * t + 8 * (r >> 2) + 4 * hi + (r & 3);
            bad_from = !(__builtin_fabsf(U[t][r]) < __builtin_inff()) && tok < bad_from ? tok : bad_from;
          }
        const int other = __shfl_xor(bad_from, 32, 64);
        bad_from = other < bad_from ? other : bad_from;
#pragma unroll
        for (int t = 0; t < CT; ++t)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            U[t][r] = 32 * t + 8 * (r >> 2) + 4 * hi + (r & 3) >= bad_from ? 0.0f : U[t][r];
      }
      // O^T += U^T P^T
      auto make_u = [&](int s) {
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = U[s / 2][8 * (s & 1) + j];
        split8<NP>(x, rop[s & 1]);
      };
      make_u(0);
      if constexpr (CT > 1) __syncthreads();
      step();
#pragma unroll
      for (int s = 0; s < CS; ++s) {
        if (CT > 1) read_tiles(s);
        if (s + 1 < CS) make_u(s + 1);
#pragma unroll
        for (int x = 0; x < NP; ++x)
#pragma unroll
          for (int p = 0; p < NP; ++p)
#pragma unroll
            for (int t = 0; t < CT; ++t)
              if (p + x < NP && t < rows_of(s))
                O[s >= 2 ? 1 : t] = mfma(rop[s & 1][x], CT == 1 ? pop[s & 1][p] : tile_op[t][p],
                                         O[s >= 2 ? 1 : t]);
        step();
      }
      if (any_bad) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int from = __shfl(bad_from, 8 * (r >> 2) + 4 * hi + (r & 3), 64);
#pragma unroll
          for (int qt = 0; qt < CT; ++qt)
            O[qt][r] = 32 * qt + col >= from ? __builtin_nanf("") : O[qt][r];
        }
      }
      store_columns<T, CT, VEC>(O, op, n, dvs, a.ot, wave);
      op += C * a.ot;
    }

    // The next chunk's rows, now that the outputs' registers are free, the values
    // and queries as u's get free.
    load_keys();

    // S <- S + K^T (2^(G' - fall) u), faded first if G is set back
    if (__builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, fade_sh[2])) == 0) {
      const float fade = fade_sh[0], low = fade_sh[1];
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) S[t][r] = __builtin_fmaf(S[t][r], fade, S[t][r] * low);
    }
    {
      u32x4 bu[SETS][NP], ak[SETS][NL];
      auto key_tile = [&](int i) {
#pragma unroll
        for (int y = 0; y < NL; ++y)
          ak[i % SETS][y] = token_operand<C, DKP>(lds, at_key, y, i % KT, i / KT);
      };
      Vec<float, 4> wt[2];
      auto weights = [&](int s) {
#pragma unroll
        for (int e = 0; e < 2; ++e)
          wt[e] = *reinterpret_cast<const Vec<float, 4>*>(end_sh + 16 * s + 8 * e + 4 * hi);
      };
      auto weigh = [&](int s, int p) {       // two tokens' of a lane's eight
        const int r = 8 * (s & 1) + 2 * p;
        split2<NP>(U[s / 2][r] * wt[p >> 1].v[2 * (p & 1)], U[s / 2][r + 1] * wt[p >> 1].v[2 * (p & 1) + 1],
                   bu[s % SETS], p);
      };
      weights(0);
      if (AHEAD) {
        key_tile(0);
#pragma unroll
        for (int p = 0; p < 4; ++p) weigh(0, p);
        if (CS > 1) weights(1);
      }
      step();
#pragma unroll
      for (int i = 0; i < CS * KT; ++i) {
        const int s = i / KT, t = i % KT;
        if (i + AHEAD < CS * KT) key_tile(i + AHEAD);
        if (!AHEAD && t == 0) {
          if (s > 0) weights(s);
#pragma unroll
          for (int p = 0; p < 4; ++p) weigh(s, p);
        }
#pragma unroll
        for (int y = 0; y < NL; ++y)
#pragma unroll
          for (int p = 0; p < NP; ++p)
            if (p + y < NP) S[t] = mfma(ak[i % SETS][y], bu[s % SETS][p], S[t]);
        if (AHEAD && s + 1 < CS) {
#pragma unroll
          for (int p = t * 4 / KT; p < (t + 1) * 4 / KT; ++p) weigh(s + 1, p);
          if (t == KT - 1 && s + 2 < CS) weights(s + 2);
        }
        if (AHEAD) step();
        if (i == CS * KT / 2 - 1) load_values();
        if (i == CS * KT * 3 / 4 - 1) load_queries();
      }
    }
    if (any_bad) {
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) S[t][r] = bad_from < C ? __builtin_nanf("") : S[t][r];
    }
  }

  float* const to = OUT ? (last ? a.state_out : nullptr) : move ? a.moves : a.own;
  if (to != nullptr) {
    if (pl.len > 0) {
      const float fade = fade_sh[3], low = fade_sh[4];
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) S[t][r] = __builtin_fmaf(S[t][r], fade, S[t][r] * low);
    }
    const __amdgpu_buffer_rsrc_t rs = state_of(to, OUT ? pl.seq : w);
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, (float)S[t][r]), rs,
                                              s_off(t, r), 0, 0);
  }
}

// The segments' N become the states before them, in place:
//   S_0 = state_in,  S_{m+1} = M_m S_m + N_m.
// A workgroup carries 32 columns of a head along a sequence, wave t their rows
// 32 t .. + 31 in an accumulator (in the walk's order of rows).  Each step puts S
// into LDS as operands, all rows for all waves; M's rows and N of the next step are
// loaded meanwhile.  Bound by the way of M and the barrier of each step: 16 segments
// of 32 heads of 128 x 128 take 80 us, 5 a step; with the products of single numbers
// in lanes, M read by every 8 columns, 620.
template <int DKP, bool VEC>
__global__ __launch_bounds__(2 * DKP) void delta_join_kernel(DeltaArgs a) {
  constexpr int KT = DKP / 32, KS = DKP / 16, NP = 3;
  __shared__ __attribute__((aligned(16))) char ssh[2][KS * NP * 1024];
  // a head's workgroups on one XCD (workgroup number mod 8), whose L2 they read M from
  const int h = blockIdx.z * 8 + (blockIdx.x & 7);
  if (h >= a.heads) return;
  const int64_t w = blockIdx.y;
  const Place pl = find_place(a, w, a.segment);
  if (pl.seq < 0 || pl.part != 0 || pl.parts < 2) return;
  const int tid = threadIdx.x, lane = tid & 63, hi = lane >> 5, col = lane & 31;
  const int t = __builtin_amdgcn_readfirstlane(tid >> 6), c0 = (blockIdx.x >> 3) * 32;
  // rows of an operand in the order in which an accumulator's are the state's
  const int row = 32 * t + 16 * (col >> 4) + 8 * ((col >> 2) & 1) + 4 * ((col >> 3) & 1) + (col & 3);
  const uint32_t s_at = c0 + col < a.dv ? 4u * (uint32_t)((32 * t + 8 * hi) * a.dv + c0 + col) : OOB;
  auto place = [&](const float* base, int64_t i, int cols) {
    return rows_rsrc(base + (i * a.heads + h) * (int64_t)a.dk * cols, 4u * a.dk * cols);
  };
  auto load_state = [&](const float* base, int64_t i) {
    const __amdgpu_buffer_rsrc_t rs = place(base, i, a.dv);
    f16v x;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const uint32_t e = __builtin_amdgcn_raw_buffer_load_b32(
          rs, s_at + 4u * (uint32_t)((16 * (r >> 3) + (r & 7)) * a.dv), 0, 0);
      x[r] = __builtin_bit_cast(float, e);
    }
    return x;
  };
  // this lane's numbers of M: its row, columns 16 s + 8 hi .. + 7
  u32x4 m[KS][2];
  const uint32_t m_at = 4u * (uint32_t)(row * a.dk + 8 * hi);     // rows from dk on: out of the range
  auto load_move = [&](const __amdgpu_buffer_rsrc_t& rs, int s) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int c = 16 * s + 8 * hi + 4 * e;
      if constexpr (VEC) {
        m[s][e] = __builtin_amdgcn_raw_buffer_load_b128(rs, c < a.dk ? m_at + 4u * (16 * s + 4 * e) : OOB,
                                                        0, 0);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          m[s][e][j] = __builtin_amdgcn_raw_buffer_load_b32(
              rs, c + j < a.dk ? m_at + 4u * (16 * s + 4 * e + j) : OOB, 0, 0);
      }
    }
  };
  f16v S = {};
  if (a.state_in != nullptr) S = load_state(a.state_in, pl.seq);
  {
    const __amdgpu_buffer_rsrc_t rm = place(a.moves, w, a.dk);
#pragma unroll
    for (int s = 0; s < KS; ++s) load_move(rm, s);
  }
  f16v next = load_state(a.own, w);
  for (int64_t i = 0; i < pl.parts; ++i) {
    const __amdgpu_buffer_rsrc_t rs = place(a.own, w + i, a.dv);
#pragma unroll
    for (int r = 0; r < 16; ++r)
      __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, (float)S[r]), rs,
                                            s_at + 4u * (uint32_t)((16 * (r >> 3) + (r & 7)) * a.dv), 0, 0);
    if (i + 1 == pl.parts) return;           // (the last one has no M and N)
    char* const image = ssh[i & 1];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = S[8 * e + j];
      u32x4 parts[NP];
      split8<NP>(x, parts);
#pragma unroll
      for (int p = 0; p < NP; ++p)
        *reinterpret_cast<u32x4*>(image + (((2 * t + e) * NP + p) * 64 + lane) * 16) = parts[p];
    }
    __syncthreads();
    S = next;
    // (the last segment has none: the first one's again)
    const int64_t ahead = w + (i + 2 < pl.parts ? i + 1 : 0);
    const __amdgpu_buffer_rsrc_t rm = place(a.moves, ahead, a.dk);
    next = load_state(a.own, ahead);
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      float x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t e = m[s][j >> 2][j & 3];
        x[j] = __builtin_bit_cast(float, e);
      }
      u32x4 mp[NP], sp[NP];
      split8<NP>(x, mp);
      load_move(rm, s);                      // the next step's, in the place of this one's
#pragma unroll
      for (int p = 0; p < NP; ++p)
        sp[p] = *reinterpret_cast<const u32x4*>(image + ((s * NP + p) * 64 + lane) * 16);
#pragma unroll
      for (int p = 0; p < NP; ++p)
#pragma unroll
        for (int q = 0; q < NP; ++q)
          if (p + q < NP) S = mfma(mp[p], sp[q], S);
      step();
    }
  }
}

// A launch has fewer than 2^32 threads: more workgroups take several, in
// multiples of `unit`.
template <typename F>
hipError_t in_launches(int64_t count, int64_t most, F launch) {
  for (int64_t first = 0; first < count; first += most) {
    launch(first, count - first < most ? count - first : most);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

template <typename T, int DKP, int NW, int C, bool VEC>
hipError_t launch_chunks(DeltaArgs a, hipStream_t st) {
  constexpr int NT = C == 64 ? 256 : 64;
  if (a.tokens > 0) {
    const hipError_t e = in_launches(a.chunks * a.heads, 0x7fffff00ll / NT, [&](int64_t first, int64_t n) {
      a.first = first;
      hipLaunchKernelGGL((delta_solve_kernel<T, DKP, C, NT, VEC>), dim3((unsigned)n), dim3(NT), 0, st, a);
    });
    if (e != hipSuccess) return e;
  }
  a.value_slices = (a.dv + 32 * NW - 1) / (32 * NW);
  const int64_t pairs = a.segments * (a.heads / a.k_group);    // of a segment and a key head
  auto launch = [&](auto kernel, int slices) {
    a.slices = slices;
    const int64_t shared = (int64_t)a.k_group * slices;
    return in_launches(pairs, 0xffffffffll / (64 * NW) / (8 * shared) * 8, [&](int64_t first, int64_t n) {
      a.first = first;
      hipLaunchKernelGGL(kernel, dim3((unsigned)((n + 7) / 8 * 8 * shared)), dim3(64 * NW), 0, st, a);
    });
  };
  if (a.segment > 0) {
    hipError_t e = launch(delta_walk_kernel<T, DKP, NW, C, false, VEC>,
                          a.value_slices + (a.dk + 32 * NW - 1) / (32 * NW));
    if (e != hipSuccess) return e;
    const dim3 grid((unsigned)(8 * ((a.dv + 31) / 32)), (unsigned)a.segments, (unsigned)((a.heads + 7) / 8));
    if (a.dk % 4 == 0) hipLaunchKernelGGL((delta_join_kernel<DKP, true>), grid, dim3(2 * DKP), 0, st, a);
    else hipLaunchKernelGGL((delta_join_kernel<DKP, false>), grid, dim3(2 * DKP), 0, st, a);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return launch(delta_walk_kernel<T, DKP, NW, C, true, VEC>, a.value_slices);
}

// bf16 heads of 65 to 128 channels have room for chunks of 64 (CF_DELTA_CHUNK)
inline int chunk_of(int64_t dtype, int64_t dk) { return dtype == SEQ_BF16 && dk > 64 && dk <= 128 ? 64 : 32; }

template <typename T, bool VEC>
hipError_t launch_delta_v(const DeltaArgs& a, hipStream_t st) {
  constexpr int C = parts_of<T>() == 1 ? 64 : 32;
  if (a.dk <= 32) return launch_chunks<T, 32, 1, 32, VEC>(a, st);
  if (a.dk <= 64) return launch_chunks<T, 64, 2, 32, VEC>(a, st);
  if (a.dk <= 128) return launch_chunks<T, 128, 4, C, VEC>(a, st);
  return launch_chunks<T, 256, 4, 32, VEC>(a, st);
}

template <typename T>
hipError_t launch_delta(const DeltaArgs& a, hipStream_t st) {
  return a.vec ? launch_delta_v<T, true>(a, st) : launch_delta_v<T, false>(a, st);
}

}  // namespace

// A block's sizes, whatever its addresses and strides.
static bool sizes_make_sense(const CfDeltaAttentionArgs& x) {
  if (x.seqs < 0 || x.seqs > CF_DECAY_MAX_SEQS || x.tokens < 0 || x.tokens > CF_DECAY_MAX_TOKENS ||
      !delta_heads_fit(x.heads, x.q_heads, x.k_heads, x.v_heads) || x.dk < 1 || x.dk > CF_DECAY_MAX_DK ||
      x.dv < 1 || x.dv > CF_DECAY_MAX_DV || x.dtype < 0 || x.dtype > 2 || x.segment < 0 ||
      x.segment % CF_DECAY_CHUNK != 0)
    return false;
  // the join's grid
  return x.segment == 0 || x.segment >= x.tokens ||
         (x.cu_seqlens ? x.tokens / x.segment + x.seqs : x.seqs * units_of(x.tokens, x.segment)) <= 65535;
}

// T, falls and betas of a chunk, all heads.
static int64_t chunk_bytes(const CfDeltaAttentionArgs& x) {
  const int64_t C = chunk_of(x.dtype, x.dk);
  return x.heads * ((C / 32) * (C / 32 + 1) / 2 * 6144 + 12 * C);
}

// Numbers of chunks, some of none, of `seqs` of the block's sequences.
static int64_t chunks_of(const CfDeltaAttentionArgs& x, int64_t seqs) {
  const int64_t C = chunk_of(x.dtype, x.dk);
  return x.cu_seqlens ? x.tokens / C + seqs : seqs * units_of(x.tokens, C);
}

// Sequences at once.  Each has a chunk of its own in the workspace, however few its
// tokens: those of less than half a chunk on average go in groups, one after another,
// as many at once as have twice the tokens' chunks or fill 2^30 bytes.  (65535 prompts
// of one token and 32 heads of 128 bf16 channels: 1.9 GB, all at once 41.  In groups of
// 2^28 bytes 4096 prompts of two tokens and 16 heads take 3020 us, of 2^30 2970, at once
// 2720.)
static int64_t group_of(const CfDeltaAttentionArgs& x) {
  if (x.tokens == 0 || (x.segment > 0 && x.segment < x.tokens)) return x.seqs;
  const int64_t C = chunk_of(x.dtype, x.dk), tokens = x.cu_seqlens ? x.tokens : x.seqs * x.tokens;
  const int64_t least = (1ll << 30) / chunk_bytes(x);
  const int64_t chunks = 2 * tokens / C > least ? 2 * tokens / C : least;
  int64_t most = chunks / (x.cu_seqlens ? 1 : units_of(x.tokens, C));
  if (most < 1) most = 1;
  if (most >= x.seqs) return x.seqs;
  const int64_t groups = (x.seqs + most - 1) / most;       // of a size
  return (x.seqs + groups - 1) / groups;
}

CF_API int64_t cf_delta_workspace(const CfDeltaAttentionArgs* p) {
  if (!p || !sizes_make_sense(*p)) return -1;
  const CfDeltaAttentionArgs& x = *p;
  int64_t bytes = x.cu_seqlens ? (16 * (x.seqs + 1) + 255) / 256 * 256 : 0;
  if (x.tokens > 0) bytes += chunks_of(x, group_of(x)) * chunk_bytes(x);
  if (x.segment > 0 && x.segment < x.tokens) {
    const int64_t segments = x.cu_seqlens ? x.tokens / x.segment + x.seqs
                                          : x.seqs * units_of(x.tokens, x.segment);
    bytes += segments * x.heads * 4 * x.dk * (x.dv + x.dk);
  }
  return bytes;
}

CF_API int cf_delta_attention(const CfDeltaAttentionArgs* p) {
  if (!p) return (int)hipErrorInvalidValue;
  const CfDeltaAttentionArgs& x = *p;
  if (!sizes_make_sense(x) || x.workspace_bytes < 0) return (int)hipErrorInvalidValue;
  for (int64_t s : {x.q_token, x.k_token, x.v_token, x.out_token})
    if (s < 0 || s > CF_DECAY_MAX_TOKEN_STRIDE) return (int)hipErrorInvalidValue;
  if (x.seqs == 0) return 0;
  if (x.tokens > 0 && (!x.q || !x.k || !x.v || !x.beta || !x.out)) return (int)hipErrorInvalidValue;
  const int64_t need = cf_delta_workspace(p);
  if (x.workspace_bytes < need || (need > 0 && (!x.workspace || (uintptr_t)x.workspace % 256 != 0)))
    return (int)hipErrorInvalidValue;
  DeltaArgs a;
  a.q = x.q; a.k = x.k; a.v = x.v;
  a.beta = x.beta; a.log_decay = x.log_decay;
  a.state_in = x.state_in; a.state_out = x.state_out;
  a.out = x.out;
  a.cu = x.cu_seqlens;
  a.cu_wide = x.cu_wide != 0; a.zero_rest = x.zero_rest ? 3 : 0;
  a.beta_f32 = x.beta_f32 != 0; a.decay_f32 = x.decay_f32 != 0;
  a.seqs = x.seqs; a.tokens = x.tokens;
  a.heads = (int)x.heads;
  a.q_group = (int)(x.heads / x.q_heads);
  a.k_group = (int)(x.heads / x.k_heads);
  a.v_group = (int)(x.heads / x.v_heads);
  a.dk = (int)x.dk; a.dv = (int)x.dv;
  a.first = 0;
  a.slices = a.value_slices = 0;
  const int64_t C = chunk_of(x.dtype, x.dk), group = group_of(x);
  a.chunks = chunks_of(x, group);
  a.group = a.cu && group < x.seqs;
  a.segment = x.segment > 0 && x.segment < x.tokens ? x.segment : 0;
  a.segments = a.segment == 0 ? x.seqs
               : a.cu ? x.tokens / a.segment + x.seqs : x.seqs * units_of(x.tokens, a.segment);
  char* at = (char*)x.workspace;
  a.begins = (int64_t*)at;
  a.before = a.begins + x.seqs + 1;
  if (a.cu) at += (16 * (x.seqs + 1) + 255) / 256 * 256;
  a.solved = at;
  if (x.tokens > 0) at += a.chunks * a.heads * ((C / 32) * (C / 32 + 1) / 2 * 6144);
  a.falls = (double*)at;
  if (x.tokens > 0) at += a.chunks * a.heads * 8 * C;
  a.betas = (float*)at;
  if (x.tokens > 0) at += a.chunks * a.heads * 4 * C;
  a.own = (float*)at;
  a.moves = a.own + a.segments * a.heads * (int64_t)a.dk * a.dv;
  a.qb = x.q_batch; a.qt = x.q_token; a.qh = x.q_head;
  a.kb = x.k_batch; a.kt = x.k_token; a.kh = x.k_head;
  a.vb = x.v_batch; a.vt = x.v_token; a.vh = x.v_head;
  a.bb = x.beta_batch; a.bt = x.beta_token; a.bh = x.beta_head;
  a.lb = x.decay_batch; a.lt = x.decay_token; a.lh = x.decay_head;
  a.ob = x.out_batch; a.ot = x.out_token; a.oh = x.out_head;
  const int size = x.dtype == SEQ_F32 ? 4 : 2, per = 16 / size;
  auto vec = [&](const void* base, int64_t b, int64_t t, int64_t h, int64_t d) {
    return (uintptr_t)base % 16 == 0 && b % per == 0 && t % per == 0 && h % per == 0 &&
           d % per == 0 && t >= d;
  };
  a.vec = vec(x.q, a.qb, a.qt, a.qh, x.dk) && vec(x.k, a.kb, a.kt, a.kh, x.dk) &&
          vec(x.v, a.vb, a.vt, a.vh, x.dv) && vec(x.out, a.ob, a.ot, a.oh, x.dv);
  a.scale = (float)x.scale;
  hipStream_t st = (hipStream_t)x.stream;
  if (a.cu && !a.group && a.seqs <= LANE_SEQS && a.chunks * a.heads <= LANE_CHUNKS) a.begins = nullptr;
  if (a.cu && a.begins != nullptr) {
    hipLaunchKernelGGL(delta_begins_kernel, dim3(1), dim3(1024), 0, st, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
  }
  auto launch = [&](const DeltaArgs& b) {
    if (x.dtype == SEQ_F32) return (int)launch_delta<float>(b, st);
    if (x.dtype == SEQ_F16) return (int)launch_delta<_Float16>(b, st);
    return (int)launch_delta<bf16_t>(b, st);
  };
  if (group == x.seqs) return launch(a);
  for (int64_t s = 0; s < x.seqs; s += group) {
    DeltaArgs b = a;
    b.seqs = b.segments = x.seqs - s < group ? x.seqs - s : group;
    b.chunks = chunks_of(x, b.seqs);
    if (s > 0) b.zero_rest &= 2;
    if (s + b.seqs < x.seqs) b.zero_rest &= 1;
    const int64_t states = s * x.heads * x.dk * x.dv;
    if (b.state_in) b.state_in += states;
    if (b.state_out) b.state_out += states;
    if (b.cu) {
      b.begins += s;
    } else {
      auto rows = [&](const void* p, int64_t batch, int bytes) { return (const char*)p + s * batch * bytes; };
      b.q = rows(a.q, a.qb, size);
      b.k = rows(a.k, a.kb, size);
      b.v = rows(a.v, a.vb, size);
      b.out = const_cast<char*>(rows(a.out, a.ob, size));
      b.beta = rows(a.beta, a.bb, a.beta_f32 ? 4 : size);
      if (b.log_decay) b.log_decay = rows(a.log_decay, a.lb, a.decay_f32 ? 4 : size);
    }
    const int e = launch(b);
    if (e != 0) return e;
  }
  return 0;
}
