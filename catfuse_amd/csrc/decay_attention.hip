// Softmax-free causal attention whose past fades by a factor of its own for
// each head, over whole sequences:
//   S_t = w S_{t-1} + k_t v_t^T,   o_t = scale q_t S_t,   w = exp(log_decay[h])
// per sequence and head, S a dk x dv matrix in fp32.  Query head h reads key
// and value head h / (heads / kv_heads).
//
// By chunks of C tokens (i, j the places in a chunk, S the state before it):
//   o_i = scale (w^(i+1) q_i S + sum_{j <= i} w^(i-j) (q_i . k_j) v_j)
//   S  <- w^C S + sum_j w^(C-1-j) k_j v_j^T
// which is four products for the matrix cores.  Every power of w has an
// exponent of at least zero, so none leaves the range of fp32 where w <= 1.
//
// Precision.  The matrix cores multiply bf16 and add fp32.  A number that is
// not a bf16 one enters a product as a sum of two or three of them, its first,
// second and third eight bits: fp16 inputs as two, and fp32 inputs, the state,
// the scores and the weighted values of the state's update as three (all
// exact).  Products of parts below 2^-24 of the whole are left out.  For 16-bit
// outputs too: two parts of the state and the scores hide behind the output's
// rounding only where their terms do not cancel (channels that share a mean: 2^-16
// of it in the output); they took 718 us where three take 777 at 65536 tokens
// x 32 heads x 128 bf16.
//
// A value that is not finite must not reach the tokens before it, where the
// product has a zero for it (0 * inf is NaN): see below at `bad_from`.  What it
// does reach is NaN as a rule, also where the formula gives an infinity: an
// infinity's second part is inf - inf.
//
// No counterpart in the reference; the causal, ordered relative of the
// spiking attention core in attention.hip.
#include "cf_chunk.h"

namespace {

struct DecayArgs {
  const void* q;
  const void* k;
  const void* v;
  const float* log_decay;
  const float* state_in;
  float* state_out;
  void* out;
  const void* cu;
  float* ws;                 // states of segments [segment][heads][dk][dv], or null
  void* spans;               // which sequence's they are: Span [segment]
  int cu_wide, zero_rest;
  int64_t seqs, tokens;      // tokens: rows in all (packed) or of each sequence
  int64_t segment, segments; // tokens a segment; segments in all at most
  int heads, group, dk, dv, slices;
  unsigned first;            // of the launch's pairs of a segment and a key head
  int64_t qb, qt, qh, kb, kt, kh, vb, vt, vh, ob, ot, oh;
  int vec;                   // 16-byte accesses are aligned and whole, rows apart
  float scale;
};

// Which (sequence, segment) a segment number is.  Packed sequences: every
// wave scans the offsets, 64 a time, each offset at least its predecessor.
// `turn`, of the i-th: the segment whose outputs are the i-th to be made.
struct alignas(16) Span { int64_t seq, part, parts, begin, len, turn; };   // seq < 0: none
static_assert(sizeof(Span) == CF_DECAY_SPAN_BYTES, "the workspace has one a segment");

__device__ __forceinline__ Span find_span(const DecayArgs& a, int64_t w) {
  Span s;
  if (a.cu == nullptr) {
    s.parts = a.tokens > 0 ? (a.tokens + a.segment - 1) / a.segment : 1;
    s.seq = w / s.parts;
    s.part = w % s.parts;
    s.begin = 0;
    s.len = a.tokens;
    if (s.seq >= a.seqs) s.seq = -1;
    return s;
  }
  const int lane = threadIdx.x & 63;
  if (a.segments == a.seqs) {
    // whole sequences (a segment holds every token): the largest offset up to
    // the sequence's, all loads in flight
    int64_t m = 0;
    for (int64_t i = lane; i <= w; i += 64) {
      const int64_t x = seq_offset(a.cu, a.cu_wide, i, a.tokens);
      if (x > m) m = x;
    }
    for (int d = 1; d < 64; d *= 2) {
      const int64_t o = __shfl_xor(m, d, 64);
      if (o > m) m = o;
    }
    const int64_t end = seq_offset(a.cu, a.cu_wide, w + 1, a.tokens);
    s.seq = w;
    s.part = 0;
    s.parts = 1;
    s.begin = uniform(m);
    s.len = uniform(end > m ? end - m : 0);
    return s;
  }
  int64_t before = 0, top = 0;               // segments and the largest offset so far
  for (int64_t b0 = 0; b0 < a.seqs; b0 += 64) {
    const int64_t b = b0 + lane;
    const bool in = b < a.seqs;
    int64_t x = in ? seq_offset(a.cu, a.cu_wide, b, a.tokens) : 0;
    int64_t y = in ? seq_offset(a.cu, a.cu_wide, b + 1, a.tokens) : 0;
    if (x < top) x = top;
    if (y < x) y = x;
    int64_t m = y;                           // running maximum over the lanes
    for (int d = 1; d < 64; d *= 2) {
      const int64_t o = __shfl_up(m, d, 64);
      if (lane >= d && o > m) m = o;
    }
    const int64_t prev = __shfl_up(m, 1, 64);
    const int64_t begin = lane > 0 && prev > x ? prev : x, end = m;
    const int64_t len = end > begin ? end - begin : 0;
    const int64_t parts = !in ? 0 : (len > 0 ? (len + a.segment - 1) / a.segment : 1);
    int64_t sum = parts;
    for (int d = 1; d < 64; d *= 2) {
      const int64_t o = __shfl_up(sum, d, 64);
      if (lane >= d) sum += o;
    }
    const int64_t first = before + sum - parts;
    const uint64_t hit = __ballot(in && w >= first && w < first + parts);
    if (hit != 0) {
      const int l = __ffsll((unsigned long long)hit) - 1;
      s.seq = b0 + l;
      s.part = uniform(w - __shfl(first, l, 64));
      s.parts = uniform(__shfl(parts, l, 64));
      s.begin = uniform(__shfl(begin, l, 64));
      s.len = uniform(__shfl(len, l, 64));
      return s;
    }
    before += uniform(__shfl(sum, 63, 64));
    const int64_t t = uniform(__shfl(m, 63, 64));
    if (t > top) top = t;
  }
  s.seq = -1;
  s.part = s.parts = s.begin = s.len = 0;
  return s;
}

// The same, as the launch of the segments' own states noted it.
__device__ __forceinline__ Span read_span(const DecayArgs& a, int64_t w) {
  const Span s = reinterpret_cast<const Span*>(a.spans)[w];
  return {uniform(s.seq), uniform(s.part), uniform(s.parts), uniform(s.begin), uniform(s.len), 0};
}

// A workgroup takes a segment of a sequence, one head, 32 NW columns of the
// values; wave w the columns 32 w .. + 31 with their part of S (all DKP rows,
// in accumulators) throughout.  OUT: the outputs of the segment, from the state
// before it in the workspace; else the segment's own contribution to the
// state, to the workspace (decay_join_kernel makes the one of the other).
//
// S as accumulators: tile t, register r of a lane is row (channel of k)
// 32 t + 16 (r / 8) + 8 (lane / 32) + r % 8, column lane % 32: the rows of K's
// operand are taken in that order, so that eight registers on end are an
// operand of the next chunk's q S as they lie.
//
// Four waves of 32 columns share a chunk's images of q, k and its scores; S for
// 128 channels takes 64 registers of a wave, so that two workgroups fit a CU.
// Chunks of 64 for bf16 (one image a tensor); two or three parts leave LDS for 32.
// Bound by issue, not by memory: 65536 tokens x 32 heads x 128 bf16, outputs
// 544-647 us, segments' own states 202-234 (matrix cores 45 % of the cycles in
// both, vector issue 50 and 43 %, at 1.72-1.94 GHz); one pass over the data
// at the rate of a copy would take 263.  bf16 chunks of 32, three waves a SIMD,
// images copied straight to LDS: the whole call 769 us against 719 (both with
// two parts of the state).
template <typename T, int DKP, int NW, int C, bool OUT, bool VEC>
__global__ __launch_bounds__(64 * NW, DKP <= 128 ? 2 : 1)
void decay_chunk_kernel(DecayArgs a) {
  constexpr int NL = parts_of<T>(), NP = 3, NT = 64 * NW;
  // operands read ahead: one set; none of three parts, whose products take long
  // enough and whose registers would cost the second workgroup of a CU
  constexpr int AHEAD = NL == 3 ? 0 : 1, SETS = AHEAD + 1;
  constexpr int KT = DKP / 32, KS = DKP / 16, CT = C / 32, CS = C / 16, DVW = 32 * NW;
  constexpr int QK_BYTES = NL * C * DKP * 2, V_BYTES = NL * C * DVW * 2;
  constexpr int TILES = CT * (CT + 1) / 2;                     // score tiles that are not masked
  constexpr int P_BYTES = CT > 1 && OUT ? TILES * 2 * NP * 1024 : 16;
  constexpr int Q_AT = QK_BYTES, V_AT = Q_AT + (OUT ? QK_BYTES : 0), IMAGE = V_AT + V_BYTES;
  __shared__ __attribute__((aligned(512))) char lds[IMAGE];     // of K, Q and V
  __shared__ __attribute__((aligned(16))) char psh[P_BYTES];
  __shared__ float pow_all[32 + C + 1];      // 32 zeros, then scale w^n
  float* const pow_sh = pow_all + 32;
  __shared__ float plain_sh[C];              // w^n
  __shared__ __attribute__((aligned(16))) float end_sh[C];   // w^(n - 1 - j) of a chunk of n tokens
  __shared__ double fade_sh[3];              // w^C, its inverse, error carried on
  __shared__ float chunk_fade_sh[2];         // w^C of the chunk at hand and the next one

  const int tid = threadIdx.x, lane = tid & 63, hi = lane >> 5, col = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

  // Query heads of one key head and the slices of their values read the same
  // rows: consecutive workgroups of one XCD (workgroup number mod 8).
  const unsigned shared = (unsigned)(a.group * a.slices), kv_heads = (unsigned)(a.heads / a.group);
  const unsigned slot = blockIdx.x >> 3;
  const unsigned super = a.first + slot / shared * 8 + (blockIdx.x & 7), inner = slot % shared;
  int64_t w = super / kv_heads;
  if (w >= a.segments) return;
  if (OUT && a.ws != nullptr) w = uniform(reinterpret_cast<const Span*>(a.spans)[w].turn);
  const int hk = (int)(super % kv_heads), h = hk * a.group + (int)(inner / (unsigned)a.slices);
  const int dv0 = (int)(inner % (unsigned)a.slices) * DVW;

  const Span sp = OUT && a.ws != nullptr ? read_span(a, w) : find_span(a, w);
  if (!OUT && hk == 0 && inner == 0 && tid == 0) {
    Span* const note = reinterpret_cast<Span*>(a.spans) + w;
    note->seq = sp.seq;
    note->part = sp.part;
    note->parts = sp.parts;
    note->begin = sp.begin;
    note->len = sp.len;
  }
  if (sp.seq < 0) return;
  const bool last = sp.part == sp.parts - 1;
  if (!OUT && last) return;                  // no segment reads it
  const int dvs = a.dv - dv0 < DVW ? a.dv - dv0 : DVW;         // columns of this slice
  const T *kp, *vp, *qp;
  T* op;
  int left;                                  // tokens from here to the segment's end
  {
    const int64_t tok0 = sp.part * a.segment, row0 = a.cu != nullptr ? 0 : sp.seq;
    const int64_t begin = sp.begin + tok0;
    left = (int)(sp.len - tok0 < a.segment ? sp.len - tok0 : a.segment);
    qp = (const T*)a.q + row0 * a.qb + begin * a.qt + h * a.qh;
    kp = (const T*)a.k + row0 * a.kb + begin * a.kt + hk * a.kh;
    vp = (const T*)a.v + row0 * a.vb + begin * a.vt + hk * a.vh + dv0;
    op = (T*)a.out + row0 * a.ob + begin * a.ot + h * a.oh + dv0;
  }

  const double ld = (double)a.log_decay[h];
  if (tid < 32) pow_all[tid] = 0.0f;
  for (int n = tid; n <= C; n += NT) {
    const double p = n == 0 ? 1.0 : exp(n * ld);
    pow_sh[n] = (float)(p * (double)a.scale);
    if (n < C) plain_sh[n] = end_sh[C - 1 - n] = (float)p;
  }
  // The rounding of w^C would add up over the chunks (2^-25 each, all of one
  // sign): what a chunk's power was off by goes into the next one's, so that the
  // powers' product never is off by more than one rounding.
  if (tid == 0) {
    const double wc = exp(C * ld), inverse = wc > 1e-30 && wc < 1e30 ? 1.0 / wc : 0.0;
    chunk_fade_sh[0] = (float)wc;
    fade_sh[0] = wc;
    fade_sh[1] = inverse;
    fade_sh[2] = (wc - (double)(float)wc) * inverse;
  }
  int odd = 0;                               // which of the two is at hand

  f16v S[KT];
#pragma unroll
  for (int t = 0; t < KT; ++t) S[t] = f16v{};
  const int sc = 32 * wave + col;            // this lane's column of the slice
  // this lane's place in a state: of its first row; the others are dv apart,
  // rows from dk on and columns from dvs on out of the buffer's range
  const uint32_t s_at = sc < dvs ? 4u * (uint32_t)(8 * hi * a.dv + dv0 + sc) : OOB;
  auto s_off = [&](int t, int r) {
    return s_at + 4u * (uint32_t)((32 * t + 16 * (r >> 3) + (r & 7)) * a.dv);
  };
  auto state_of = [&](const float* base, int64_t i) {
    return rows_rsrc(base + (i * a.heads + h) * (int64_t)a.dk * a.dv, 4u * a.dk * a.dv);
  };
  if (OUT) {
    const float* const from = sp.part > 0 ? a.ws : a.state_in;
    if (from != nullptr) {
      const __amdgpu_buffer_rsrc_t rs = state_of(from, sp.part > 0 ? w : sp.seq);
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          S[t][r] = __builtin_bit_cast(
              float, __builtin_amdgcn_raw_buffer_load_b32(rs, s_off(t, r), 0, 0));
    }
  }

  constexpr int UK = C * (DKP / 8) / NT, UV = C * (DVW / 8) / NT;   // units of a thread
  static_assert(UK * NT == C * (DKP / 8) && UV * NT == C * (DVW / 8), "whole units");
  Unit<T> ku[UK], vu[UV], qu[OUT ? UK : 1];
  auto load_chunk = [&]() {
    const int n = left < C ? left : C;
    load_units<T, UK, DKP, NT, VEC>(ku, kp, n, a.kt, a.dk);
    load_units<T, UV, DVW, NT, VEC>(vu, vp, n, a.vt, dvs);
    if constexpr (OUT) load_units<T, UK, DKP, NT, VEC>(qu, qp, n, a.qt, a.dk);
  };

  const uint32_t at_row = row_base<DKP>(lane), at_key = token_base<DKP>(lane, true);
  const uint32_t at_value = token_base<DVW>(lane, false) ^ (uint32_t)(wave << 6);

  if (left > 0) load_chunk();
  while (left > 0) {
    const int n = left < C ? left : C;
    __syncthreads();                         // the last chunk's images are read
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
    if (n < C)                               // (the last chunk: its predecessor's powers are read)
      for (int j = tid; j < C; j += NT) end_sh[j] = j < n ? plain_sh[n - 1 - j] : 0.0f;
    __syncthreads();
    left -= n;
    kp += C * a.kt;
    vp += C * a.vt;
    qp += C * a.qt;

    u32x4 vop[CS][NL];                       // lane: column sc, tokens as token_operand
#pragma unroll
    for (int s = 0; s < CS; ++s)
#pragma unroll
      for (int p = 0; p < NL; ++p) vop[s][p] = token_operand<C, DVW>(lds + V_AT, at_value, p, 0, s);

    // A value that is not finite would give NaN wherever it meets a masked
    // score's zero: it is taken out, and what depends on it set to NaN below
    // (this lane's column: the queries from its token on, and the state).
    // (The segments' own states have no masked scores: there NaN goes its way.)
    int bad_from = C;
    if constexpr (OUT) {
      uint32_t any = 0u;                     // exponents of all ones, of the leading parts
#pragma unroll
      for (int s = 0; s < CS; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) any |= (vop[s][0][i] & 0x7f807f80u) + 0x00800080u;
      if (__ballot((any & 0x80008000u) != 0u) != 0) {
#pragma unroll
        for (int s = 0; s < CS; ++s)
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const uint32_t m = (j & 1) ? 0x7f800000u : 0x00007f80u;
            if ((vop[s][0][j >> 1] & m) == m) {
              const int tok = 16 * s + 8 * (j >> 2) + 4 * hi + (j & 3);
              if (tok < bad_from) bad_from = tok;
#pragma unroll
              for (int p = 0; p < NL; ++p) vop[s][p][j >> 1] &= (j & 1) ? 0xffffu : 0xffff0000u;
            }
          }
        const int other = __shfl_xor(bad_from, 32, 64);
        if (other < bad_from) bad_from = other;
      }
    }
    const bool any_bad = OUT && __ballot(bad_from < C) != 0;

    const float fade = n == C ? chunk_fade_sh[odd] : plain_sh[n];
    odd ^= 1;
    if (tid == 0) {                          // the next chunk's, which no one reads before a barrier
      const double p = __builtin_fma(fade_sh[0], fade_sh[2], fade_sh[0]);
      const float w = (float)p;
      chunk_fade_sh[odd] = w;
      fade_sh[2] = (p - (double)w) * fade_sh[1];
    }

    // The operand w^(n-1-j) v_j of S's update, 16 tokens of it: its weights, and
    // two tokens (2 p, 2 p + 1 of a lane's eight) at a time.
    Vec<float, 4> wt[2];
    auto weights = [&](int s) {
#pragma unroll
      for (int e = 0; e < 2; ++e)
        wt[e] = *reinterpret_cast<const Vec<float, 4>*>(end_sh + 16 * s + 8 * e + 4 * hi);
    };
    auto weigh = [&](int s, int p, u32x4* to) {
      float y[2];
#pragma unroll
      for (int l = 0; l < NL; ++l) {
        const uint32_t word = vop[s][l][p];
        const float lo = __builtin_bit_cast(float, word << 16);
        const float up = __builtin_bit_cast(float, word & 0xffff0000u);
        y[0] = l == 0 ? lo : y[0] + lo;
        y[1] = l == 0 ? up : y[1] + up;
      }
      split2<3>(y[0] * wt[p >> 1].v[2 * (p & 1)], y[1] * wt[p >> 1].v[2 * (p & 1) + 1], to, p);
    };
    f16v acc[CT];

    // In what follows the operands of the next products are read, and made,
    // between the products at hand, and the compiler is held to that order
    // (step()): left alone, short of registers, it reads each operand right
    // before its use and waits for LDS some eighty times a chunk.
    if constexpr (OUT) {
      // Scores K Q^T of 32 keys (rows) x 32 queries (columns): eight registers
      // on end are an operand of V^T P^T as they lie.  One tile: every wave
      // for itself; three: a tile a wave, exchanged in LDS.
      u32x4 pop[CT > 1 ? 1 : 2][NP];
      auto score_tile = [&](int kt, int qt, u32x4 (*ops)[NP]) {
        // query minus key, less a constant of the register; opaque: 16 powers and
        // masks kept over the chunks cost more registers than there are
        int gap0 = 32 * (qt - kt) + col - 4 * hi;
        asm volatile("" : "+v"(gap0));
        const float* const powers = pow_sh + gap0;
        u32x4 ak[SETS][NL], bq[SETS][NL];
        auto read = [&](int s) {
#pragma unroll
          for (int p = 0; p < NL; ++p) {
            ak[s % SETS][p] = row_operand<C, DKP>(lds, at_row, p, kt, s);
            bq[s % SETS][p] = row_operand<C, DKP>(lds + Q_AT, at_row, p, qt, s);
          }
        };
        if (AHEAD) read(0);
        float f[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) f[r] = powers[-(8 * (r >> 2) + (r & 3))];
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
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          float x[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int key = 16 * s + 8 * (j >> 2) + (j & 3);
            const float y = acc[8 * s + j] * f[8 * s + j];
            x[j] = gap0 >= key ? y : 0.0f;
          }
          split8<NP>(x, ops[s]);
        }
      };
      if constexpr (CT > 1) {
        for (int tile = wave; tile < TILES; tile += NW) {
          const int qt = tile == 0 ? 0 : 1, kt = tile == 2 ? 1 : 0;    // (0,0) (0,1) (1,1)
          u32x4 ops[2][NP];
          score_tile(kt, qt, ops);
#pragma unroll
          for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int p = 0; p < NP; ++p)
              *reinterpret_cast<u32x4*>(psh + (((tile * 2 + s) * NP + p) * 64 + lane) * 16) =
                  ops[s][p];
        }
      } else {
        score_tile(0, 0, pop);
      }

      // O^T = scale w^(i+1) S^T Q^T + V^T P^T: rows columns of the values,
      // columns queries (P holds the scale).
      {
        u32x4 as[SETS][NP], bq[SETS][CT][NL];
        auto state_part = [&](int s) {       // S's operand, and S faded
          float x[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            x[j] = S[s / 2][8 * (s & 1) + j];
            S[s / 2][8 * (s & 1) + j] = x[j] * fade;
          }
          split8<NP>(x, as[s % SETS]);
        };
        auto read = [&](int s) {
#pragma unroll
          for (int qt = 0; qt < CT; ++qt)
#pragma unroll
            for (int y = 0; y < NL; ++y)
              bq[s % SETS][qt][y] = row_operand<C, DKP>(lds + Q_AT, at_row, y, qt, s);
        };
        if (AHEAD) {
          read(0);
          state_part(0);
        }
#pragma unroll
        for (int qt = 0; qt < CT; ++qt) acc[qt] = f16v{};
        step();
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          if (s + AHEAD < KS) {
            read(s + AHEAD);
            state_part(s + AHEAD);
          }
#pragma unroll
          for (int x = 0; x < NP; ++x)
#pragma unroll
            for (int y = 0; y < NL; ++y)
#pragma unroll
              for (int qt = 0; qt < CT; ++qt)
                if (x + y < NP) acc[qt] = mfma(as[s % SETS][x], bq[s % SETS][qt][y], acc[qt]);
          if (AHEAD) step();
        }
      }
#pragma unroll
      for (int qt = 0; qt < CT; ++qt) {
        const float f = pow_sh[32 * qt + col + 1];
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[qt][r] *= f;
      }
      if constexpr (CT > 1) {
        __syncthreads();
        u32x4 bp[2][NP];
        constexpr int STEPS = TILES * 2;     // (tile, s)
        auto read = [&](int i) {
#pragma unroll
          for (int y = 0; y < NP; ++y)
            bp[i & 1][y] = *reinterpret_cast<const u32x4*>(psh + ((i * NP + y) * 64 + lane) * 16);
        };
        read(0);
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
          if (i + 1 < STEPS) read(i + 1);
          const int qt = i / 2 == 0 ? 0 : 1, kt = i / 2 == 2 ? 1 : 0, s = i & 1;
#pragma unroll
          for (int y = 0; y < NP; ++y)
#pragma unroll
            for (int p = 0; p < NL; ++p)
              if (p + y < NP) acc[qt] = mfma(vop[2 * kt + s][p], bp[i & 1][y], acc[qt]);
          step();
        }
      } else {
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int y = 0; y < NP; ++y)
#pragma unroll
            for (int p = 0; p < NL; ++p)
              if (p + y < NP) acc[0] = mfma(vop[s][p], pop[s][y], acc[0]);
      }
    } else {
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) S[t][r] *= fade;
    }

    if constexpr (OUT) {
      if (any_bad) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int from = __shfl(bad_from, 8 * (r >> 2) + 4 * hi + (r & 3), 64);
#pragma unroll
          for (int qt = 0; qt < CT; ++qt)
            if (32 * qt + col >= from) acc[qt][r] = __builtin_nanf("");
        }
      }
      store_columns<T, CT, VEC>(acc, op, n, dvs, a.ot, wave);
      op += C * a.ot;
    }

    // The next chunk's rows, now that the outputs' registers are free.
    if (left > 0) load_chunk();

    // S <- w^n S (above) + K^T (w^(n-1-j) V)
    {
      u32x4 bv[SETS][3], ak[SETS][NL];
      auto key_tile = [&](int i) {
#pragma unroll
        for (int y = 0; y < NL; ++y)
          ak[i % SETS][y] = token_operand<C, DKP>(lds, at_key, y, i % KT, i / KT);
      };
      weights(0);
      if (AHEAD) {
        key_tile(0);
#pragma unroll
        for (int p = 0; p < 4; ++p) weigh(0, p, bv[0]);
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
          for (int p = 0; p < 4; ++p) weigh(s, p, bv[0]);
        }
#pragma unroll
        for (int y = 0; y < NL; ++y)
#pragma unroll
          for (int p = 0; p < 3; ++p)
            if (p + y < 3) S[t] = mfma(ak[i % SETS][y], bv[s % SETS][p], S[t]);
        if (AHEAD && s + 1 < CS) {
#pragma unroll
          for (int p = t * 4 / KT; p < (t + 1) * 4 / KT; ++p) weigh(s + 1, p, bv[(s + 1) % SETS]);
          if (t == KT - 1 && s + 2 < CS) weights(s + 2);
        }
        if (AHEAD) step();
      }
    }
    if (any_bad && bad_from < C) {
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) S[t][r] = __builtin_nanf("");
    }
  }

  float* const to = OUT ? (last ? a.state_out : nullptr) : a.ws;
  if (to != nullptr) {
    const __amdgpu_buffer_rsrc_t rs = state_of(to, OUT ? sp.seq : w);
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, (float)S[t][r]), rs,
                                              s_off(t, r), 0, 0);
  }
  if (OUT && a.cu != nullptr && a.zero_rest) {   // rows of no sequence
    T* const all = (T*)a.out + h * a.oh + dv0;
    auto clear = [&](int64_t from, int64_t to) {
      for (int64_t t = from + tid / DVW; t < to; t += NT / DVW)
        if (tid % DVW < dvs) all[t * a.ot + tid % DVW] = from_f<T>(0.0f);
    };
    if (sp.seq == 0 && sp.part == 0) clear(0, sp.begin);
    if (sp.seq == a.seqs - 1 && last) clear(sp.begin + sp.len, a.tokens);
  }
}

// Sorts the segments for the outputs (one workgroup), whole ones first and the
// ends of sequences by eighths of a segment: the last workgroups to start are
// then the shortest.
__device__ __forceinline__ void order_segments(const DecayArgs& a) {
  __shared__ int place[10];
  Span* const spans = reinterpret_cast<Span*>(a.spans);
  const int tid = threadIdx.x;
  auto rank = [&](int64_t i) {               // 0: whole, 8: empty, 9: not one
    const Span& s = spans[i];
    if (s.seq < 0) return 9;
    const int64_t left = s.len - s.part * a.segment, len = left < a.segment ? left : a.segment;
    return 8 - (int)((8 * len + a.segment - 1) / a.segment);
  };
  if (tid < 10) place[tid] = 0;
  __syncthreads();
  for (int64_t i = tid; i < a.segments; i += 256) atomicAdd(&place[rank(i)], 1);
  __syncthreads();
  if (tid == 0) {
    int at = 0;
    for (int r = 0; r < 10; ++r) {
      const int n = place[r];
      place[r] = at;
      at += n;
    }
  }
  __syncthreads();
  for (int64_t i = tid; i < a.segments; i += 256) spans[atomicAdd(&place[rank(i)], 1)].turn = i;
}

// The segments' own states become the states before them, in place:
//   S_0 = state_in,  S_{m+1} = w^segment S_m + (own state of m)
// A thread carries N numbers along a sequence, JOIN_AHEAD loads in flight; one
// workgroup more orders the segments.
// Bound by the latency of those loads: 16 segments of 32 heads of 128 x 128 take
// 15-17 us; with the sum in every workgroup of the outputs instead the call was
// slower (65536 tokens: 871 us, this launch with reads ahead there 740).
constexpr int JOIN_AHEAD = 8;
template <int N>
__global__ __launch_bounds__(256) void decay_join_kernel(DecayArgs a) {
  typedef Vec<float, N> V;
  const int64_t w = blockIdx.y;
  if (w == a.segments) {
    if (blockIdx.x == 0 && blockIdx.z == 0) order_segments(a);
    return;
  }
  const Span sp = read_span(a, w);
  if (sp.seq < 0 || sp.part != 0 || sp.parts < 2) return;
  const int h = blockIdx.z;
  const int64_t size = (int64_t)a.dk * a.dv, i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * N;
  if (i >= size) return;
  // In 64 bits: the rounding of w^segment would add up, and where w > 1 it passes
  // the range of fp32 (exp(64 log_decay) is in it) although the state times it
  // may not.  A state of zero stays one even if it passes that of fp64; any other
  // one leaves fp32 then.
  const double f = exp((double)a.segment * (double)a.log_decay[h]);
  float* const p = a.ws + (w * a.heads + h) * size + i;
  const int64_t step = a.heads * size, n = sp.parts - 1;      // the last one has none of its own
  V s{};
  if (a.state_in != nullptr)
    s = *reinterpret_cast<const V*>(a.state_in + (sp.seq * a.heads + h) * size + i);
  for (int64_t m0 = 0; m0 < n; m0 += JOIN_AHEAD) {
    V x[JOIN_AHEAD];
#pragma unroll
    for (int j = 0; j < JOIN_AHEAD; ++j)
      if (m0 + j < n) x[j] = *reinterpret_cast<const V*>(p + (m0 + j) * step);
#pragma unroll
    for (int j = 0; j < JOIN_AHEAD; ++j) {
      if (m0 + j >= n) break;
      *reinterpret_cast<V*>(p + (m0 + j) * step) = s;
#pragma unroll
      for (int c = 0; c < N; ++c)
        s.v[c] = s.v[c] == 0.0f ? x[j].v[c] : (float)__builtin_fma((double)s.v[c], f, (double)x[j].v[c]);
    }
  }
  *reinterpret_cast<V*>(p + n * step) = s;
}

hipError_t launch_join(const DecayArgs& a, hipStream_t st) {
  const int64_t size = (int64_t)a.dk * a.dv;
  const bool wide = size % 4 == 0 && (uintptr_t)a.ws % 16 == 0 && (uintptr_t)a.state_in % 16 == 0;
  const dim3 grid((unsigned)((size / (wide ? 4 : 1) + 255) / 256), (unsigned)a.segments + 1,
                  (unsigned)a.heads);
  if (wide) hipLaunchKernelGGL(decay_join_kernel<4>, grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL(decay_join_kernel<1>, grid, dim3(256), 0, st, a);
  return hipGetLastError();
}

template <typename T, int DKP, int NW, int C, bool VEC>
hipError_t launch_chunks(DecayArgs a, hipStream_t st) {
  a.slices = (a.dv + 32 * NW - 1) / (32 * NW);
  const int64_t shared = (int64_t)a.group * a.slices;
  const int64_t pairs = a.segments * (a.heads / a.group);      // of a segment and a key head
  // a launch has fewer than 2^32 threads: more pairs take several
  const int64_t most = 0xffffffffll / (64 * NW) / (8 * shared) * 8;
  if (a.ws != nullptr && a.segments >= 65535) return hipErrorInvalidValue;   // the join's grid
  auto launch = [&](auto kernel, size_t lds) {
    for (int64_t first = 0; first < pairs; first += most) {
      const int64_t n = pairs - first < most ? pairs - first : most;
      a.first = (unsigned)first;
      hipLaunchKernelGGL(kernel, dim3((unsigned)((n + 7) / 8 * 8 * shared)), dim3(64 * NW), lds, st,
                         a);
      const hipError_t e = hipGetLastError();
      if (e != hipSuccess) return e;
    }
    return hipSuccess;
  };
  if (a.ws != nullptr) {
    // bf16 heads of 65-128: LDS for two workgroups a CU, though the registers would
    // let three in: where all start at once, some CUs would get three and others one
    // (24 packed prompts of 24011 tokens, 16 heads of 128: 55 us, with two 46).
    hipError_t e = launch(decay_chunk_kernel<T, DKP, NW, C, false, VEC>,
                          DKP == 128 && C == 64 ? 24576 : 0);
    if (e != hipSuccess) return e;
    e = launch_join(a, st);
    if (e != hipSuccess) return e;
  }
  return launch(decay_chunk_kernel<T, DKP, NW, C, true, VEC>, 0);
}

template <typename T, bool VEC>
hipError_t launch_decay_v(const DecayArgs& a, hipStream_t st) {
  constexpr int C = sizeof(T) == 2 && parts_of<T>() == 1 ? 64 : 32;
  if (a.dk <= 32) return launch_chunks<T, 32, 1, C, VEC>(a, st);
  if (a.dk <= 64) return launch_chunks<T, 64, 2, C, VEC>(a, st);
  if (a.dk <= 128) return launch_chunks<T, 128, 4, C, VEC>(a, st);
  return launch_chunks<T, 256, 4, 32, VEC>(a, st);
}

template <typename T>
hipError_t launch_decay(const DecayArgs& a, hipStream_t st) {
  return a.vec ? launch_decay_v<T, true>(a, st) : launch_decay_v<T, false>(a, st);
}

}  // namespace

CF_API int cf_decay_attention(const CfDecayAttentionArgs* p) {
  if (!p) return (int)hipErrorInvalidValue;
  const CfDecayAttentionArgs& x = *p;
  if (x.seqs < 0 || x.tokens < 0 || x.heads < 1 || x.kv_heads < 1 || x.heads % x.kv_heads != 0 ||
      x.heads > CF_SEQ_MAX_HEADS || x.dk < 1 || x.dk > CF_DECAY_MAX_DK || x.dv < 1 ||
      x.dv > CF_DECAY_MAX_DV || x.dtype < 0 || x.dtype > 2 || x.seqs > CF_DECAY_MAX_SEQS ||
      x.tokens > CF_DECAY_MAX_TOKENS || x.segment < 0 || x.segment % CF_DECAY_CHUNK != 0 || x.workspace_bytes < 0)
    return (int)hipErrorInvalidValue;
  for (int64_t s : {x.q_token, x.k_token, x.v_token, x.out_token})
    if (s < 0 || s > CF_DECAY_MAX_TOKEN_STRIDE) return (int)hipErrorInvalidValue;
  if (x.seqs == 0) return 0;
  if (!x.log_decay || (x.tokens > 0 && (!x.q || !x.k || !x.v || !x.out)))
    return (int)hipErrorInvalidValue;
  DecayArgs a;
  a.q = x.q; a.k = x.k; a.v = x.v;
  a.log_decay = x.log_decay;
  a.state_in = x.state_in; a.state_out = x.state_out;
  a.out = x.out;
  a.cu = x.cu_seqlens;
  a.cu_wide = x.cu_wide != 0; a.zero_rest = x.zero_rest != 0;
  a.seqs = x.seqs; a.tokens = x.tokens;
  a.heads = (int)x.heads; a.group = (int)(x.heads / x.kv_heads);
  a.dk = (int)x.dk; a.dv = (int)x.dv;
  a.first = 0;
  a.ws = nullptr;
  a.spans = nullptr;
  a.segment = x.tokens > 0 ? x.tokens : 1;
  a.segments = x.seqs;
  if (x.segment > 0 && x.segment < x.tokens) {
    a.segment = x.segment;
    a.segments = x.cu_seqlens ? x.tokens / x.segment + x.seqs
                              : x.seqs * ((x.tokens + x.segment - 1) / x.segment);
    const int64_t state = 4 * x.heads * x.dk * x.dv;
    if (!x.workspace || (uintptr_t)x.workspace % 16 != 0 ||
        x.workspace_bytes / (state + CF_DECAY_SPAN_BYTES) < a.segments)
      return (int)hipErrorInvalidValue;
    a.spans = x.workspace;
    a.ws = (float*)((char*)x.workspace + a.segments * CF_DECAY_SPAN_BYTES);
  }
  a.qb = x.q_batch; a.qt = x.q_token; a.qh = x.q_head;
  a.kb = x.k_batch; a.kt = x.k_token; a.kh = x.k_head;
  a.vb = x.v_batch; a.vt = x.v_token; a.vh = x.v_head;
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
  hipError_t e;
  if (x.dtype == SEQ_F32) e = launch_decay<float>(a, st);
  else if (x.dtype == SEQ_F16) e = launch_decay<_Float16>(a, st);
  else e = launch_decay<bf16_t>(a, st);
  return (int)e;
}
