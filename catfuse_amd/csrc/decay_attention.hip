// Softmax-free causal attention whose past fades by a factor of its own for
// each head, over whole sequences:
//   S_t = w S_{t-1} + k_t v_t^T,   o_t = scale q_t S_t,   w = exp(log_decay[h])
// per sequence and head, S a dk x dv matrix in fp32.  Query head h reads key
// and value head h / (heads / kv_heads).
//
// No counterpart in the reference; the causal, ordered relative of the
// spiking attention core in attention.hip.
#include "cf_seq.h"

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
  int cu_wide, zero_rest;
  int64_t seqs, tokens;      // tokens: rows in all (packed) or of each sequence
  int heads, group, dk, dv;
  int64_t qb, qt, qh, kb, kt, kh, vb, vt, vh, ob, ot, oh;
  float scale;
};

// One token after another: a workgroup holds 64 columns of one sequence and
// head's state in registers, wave g the rows g R .. g R + R - 1.
template <typename T, int R>
__global__ __launch_bounds__(256) void decay_recurrent_kernel(DecayArgs a) {
  constexpr int TOK = 16, DKP = 4 * R;
  __shared__ float qs[TOK][DKP], ks[TOK][DKP];
  __shared__ float part[TOK][4][64];
  const int tid = threadIdx.x, col = tid & 63, g = tid >> 6;
  const int c = blockIdx.x * 64 + col, h = blockIdx.y;
  const int64_t b = blockIdx.z;
  int64_t begin = 0, len = a.tokens;
  if (a.cu != nullptr) {
    begin = seq_offset(a.cu, a.cu_wide, b, a.tokens);
    const int64_t end = seq_offset(a.cu, a.cu_wide, b + 1, a.tokens);
    len = end > begin ? end - begin : 0;
  }
  const int64_t row0 = a.cu != nullptr ? 0 : b;
  const T* q = (const T*)a.q + row0 * a.qb + begin * a.qt + h * a.qh;
  const T* k = (const T*)a.k + row0 * a.kb + begin * a.kt + (h / a.group) * a.kh;
  const T* v = (const T*)a.v + row0 * a.vb + begin * a.vt + (h / a.group) * a.vh;
  T* o = (T*)a.out + row0 * a.ob + begin * a.ot + h * a.oh;
  const bool mine = c < a.dv;
  const float w = (float)exp((double)a.log_decay[h]);
  float s[R];
  const int64_t sbase = ((b * a.heads + h) * a.dk) * (int64_t)a.dv + c;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int d = g * R + r;
    s[r] = a.state_in != nullptr && mine && d < a.dk ? a.state_in[sbase + (int64_t)d * a.dv] : 0.0f;
  }
  for (int64_t t0 = 0; t0 < len; t0 += TOK) {
    const int n = (int)(len - t0 < TOK ? len - t0 : TOK);
    __syncthreads();
    for (int i = tid; i < TOK * DKP; i += 256) {
      const int t = i / DKP, d = i % DKP;
      const bool in = t < n && d < a.dk;
      qs[t][d] = in ? to_f(q[(t0 + t) * a.qt + d]) : 0.0f;
      ks[t][d] = in ? to_f(k[(t0 + t) * a.kt + d]) : 0.0f;
    }
    __syncthreads();
    for (int t = 0; t < n; ++t) {
      const float x = mine ? to_f(v[(t0 + t) * a.vt + c]) : 0.0f;
      float p = 0.0f;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        s[r] = __builtin_fmaf(s[r], w, ks[t][g * R + r] * x);
        p = __builtin_fmaf(qs[t][g * R + r], s[r], p);
      }
      part[t][g][col] = p;
    }
    __syncthreads();
    for (int t = g; t < n; t += 4)
      if (mine)
        o[(t0 + t) * a.ot + c] = from_f<T>(
            ((part[t][0][col] + part[t][1][col]) + (part[t][2][col] + part[t][3][col])) * a.scale);
  }
  if (a.state_out != nullptr) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int d = g * R + r;
      if (mine && d < a.dk) a.state_out[sbase + (int64_t)d * a.dv] = s[r];
    }
  }
  if (a.cu != nullptr && a.zero_rest) {   // rows of no sequence
    T* all = (T*)a.out + h * a.oh;
    if (b == 0)
      for (int64_t t = g; t < begin; t += 4)
        if (mine) all[t * a.ot + c] = from_f<T>(0.0f);
    if (b == a.seqs - 1)
      for (int64_t t = begin + len + g; t < a.tokens; t += 4)
        if (mine) all[t * a.ot + c] = from_f<T>(0.0f);
  }
}

template <typename T>
hipError_t launch_decay(const DecayArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)((a.dv + 63) / 64), (unsigned)a.heads, (unsigned)a.seqs);
  if (a.dk <= 32) hipLaunchKernelGGL((decay_recurrent_kernel<T, 8>), grid, dim3(256), 0, st, a);
  else if (a.dk <= 64) hipLaunchKernelGGL((decay_recurrent_kernel<T, 16>), grid, dim3(256), 0, st, a);
  else if (a.dk <= 128) hipLaunchKernelGGL((decay_recurrent_kernel<T, 32>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((decay_recurrent_kernel<T, 64>), grid, dim3(256), 0, st, a);
  return hipGetLastError();
}

}  // namespace

CF_API int cf_decay_attention(const CfDecayAttentionArgs* p) {
  if (!p) return (int)hipErrorInvalidValue;
  const CfDecayAttentionArgs& x = *p;
  if (x.seqs < 0 || x.tokens < 0 || x.heads < 1 || x.kv_heads < 1 || x.heads % x.kv_heads != 0 ||
      x.heads > CF_SEQ_MAX_HEADS || x.dk < 1 || x.dk > CF_DECAY_MAX_DK || x.dv < 1 ||
      x.dv > CF_DECAY_MAX_DV || x.dtype < 0 || x.dtype > 2 || x.seqs > CF_DECAY_MAX_SEQS)
    return (int)hipErrorInvalidValue;
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
  a.qb = x.q_batch; a.qt = x.q_token; a.qh = x.q_head;
  a.kb = x.k_batch; a.kt = x.k_token; a.kh = x.k_head;
  a.vb = x.v_batch; a.vt = x.v_token; a.vh = x.v_head;
  a.ob = x.out_batch; a.ot = x.out_token; a.oh = x.out_head;
  a.scale = (float)x.scale;
  hipStream_t st = (hipStream_t)x.stream;
  hipError_t e;
  if (x.dtype == SEQ_F32) e = launch_decay<float>(a, st);
  else if (x.dtype == SEQ_F16) e = launch_decay<_Float16>(a, st);
  else e = launch_decay<bf16_t>(a, st);
  return (int)e;
}
