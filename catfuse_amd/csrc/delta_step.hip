// One token of each running sequence through the delta rule's attention,
// against a pool of states:
//   S <- w S + k u^T,   u = beta (v - w S^T k),   o = scale q S,
//   w = exp(log_decay)
// for row b and head h with S = state[slots[b]][h], dk x dv in fp32, updated
// in place; beta and log_decay are the row's and head's own.  Rows whose slot
// is outside the pool (negative ones mark padding) give zeros and touch no
// state.  Rows with the same slot are consecutive tokens of one sequence, in
// the order of the rows: the first one's workgroup takes them all, so no two
// workgroups meet in a state.
//
// No counterpart in the reference; the correcting relative of decay_step.hip.
#include "cf_seq.h"

namespace {

struct DeltaStepArgs {
  const void* q;
  const void* k;
  const void* v;
  const void* beta;
  const void* log_decay;
  float* state;
  void* out;
  const void* slots;
  int slots_wide, beta_f32, decay_f32;
  int rows, heads, q_group, k_group, v_group, dk, dv;
  int64_t pool, state_slot;
  int64_t qr, qh, kr, kh, vr, vh, br, bh, lr, lh, orow, oh;
  float scale;
};

__device__ __forceinline__ int64_t step_slot(const DeltaStepArgs& a, int i) {
  if (a.slots == nullptr) return i;
  return a.slots_wide ? reinterpret_cast<const int64_t*>(a.slots)[i]
                      : (int64_t)reinterpret_cast<const int32_t*>(a.slots)[i];
}

// A workgroup takes CL * VEC columns of one row's and head's state; thread =
// VEC columns of NR rows, held in registers: k S and q S are both sums over
// the old state, and q S_new = w q S + (q . k) u, so that one pass reads it
// and one writes it.  Bound by HBM: 256 rows of 32 heads of 128 x 128 in 218 us, 4.9
// TB/s, the rate of a large copy; one row of 12 heads of 32 x 32 by its latency, 5.
template <typename T, int VEC, int CL, int NR>
__global__ __launch_bounds__(256) void delta_step_kernel(DeltaStepArgs a) {
  constexpr int RG = 256 / CL, COLS = CL * VEC;
  __shared__ float qs[RG * NR], ks[RG * NR];
  __shared__ float part[2][RG][COLS];
  __shared__ float us[COLS];
  __shared__ float dot_sh[4];
  __shared__ int next_sh;
  const int tid = threadIdx.x, cl = tid % CL, rg = tid / CL;
  const int c = (blockIdx.x * CL + cl) * VEC, h = blockIdx.y;
  int row = blockIdx.z;
  const int64_t slot = step_slot(a, row);
  T* const out = (T*)a.out + h * a.oh;
  const bool mine = c < a.dv;
  if (slot < 0 || slot >= a.pool) {
    if (rg == 0 && mine)
#pragma unroll
      for (int i = 0; i < VEC; ++i) out[row * a.orow + c + i] = from_f<T>(0.0f);
    return;
  }
  float* const s = a.state + slot * a.state_slot + (int64_t)h * a.dk * a.dv + c;
  for (;;) {
    // the next row of this slot; nothing to do if an earlier row has it
    int next = a.rows;
    if (a.slots != nullptr) {
      bool prior = false;
      for (int i = tid; i < a.rows; i += 256) {
        const bool same = step_slot(a, i) == slot;
        if (same && i < row && row == (int)blockIdx.z) prior = true;
        if (same && i > row && i < next) next = i;
      }
      if (tid == 0) next_sh = a.rows;
      if (__syncthreads_or(prior ? 1 : 0)) return;
      if (next < a.rows) atomicMin(&next_sh, next);
      __syncthreads();
      next = next_sh;
    }
    Vec<float, VEC> y[NR];
    if (mine) {
#pragma unroll
      for (int n = 0; n < NR; ++n)
        if (rg + n * RG < a.dk)
          y[n] = *reinterpret_cast<const Vec<float, VEC>*>(s + (int64_t)(rg + n * RG) * a.dv);
    }
    const T* const q = (const T*)a.q + row * a.qr + (h / a.q_group) * a.qh;
    const T* const k = (const T*)a.k + row * a.kr + (h / a.k_group) * a.kh;
    const T* const v = (const T*)a.v + row * a.vr + (h / a.v_group) * a.vh;
    // w as a sum of two floats: the rounding of one would shift the horizon of
    // a slow decay by the token
    const double wd = a.log_decay == nullptr ? 1.0
                          : exp(load_double<T>(a.log_decay, row * a.lr + h * a.lh, a.decay_f32));
    const float w = (float)wd, wl = wd < 1e300 ? (float)(wd - (double)w) : 0.0f;
    const float beta = (float)load_double<T>(a.beta, row * a.br + h * a.bh, a.beta_f32);
    float d = 0.0f;                          // a part of q . k
    for (int i = tid; i < RG * NR; i += 256) {
      const float qi = i < a.dk ? to_f(q[i]) : 0.0f, ki = i < a.dk ? to_f(k[i]) : 0.0f;
      qs[i] = qi;
      ks[i] = ki;
      d = __builtin_fmaf(qi, ki, d);
    }
#pragma unroll
    for (int m = 32; m >= 1; m /= 2) d += __shfl_xor(d, m, 64);
    if ((tid & 63) == 0) dot_sh[tid >> 6] = d;
    __syncthreads();
    float pk[VEC], pq[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) pk[i] = pq[i] = 0.0f;
    if (mine) {
#pragma unroll
      for (int n = 0; n < NR; ++n) {
        const int r = rg + n * RG;
        if (r < a.dk)
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            y[n].v[i] = __builtin_fmaf(y[n].v[i], w, y[n].v[i] * wl);
            pk[i] = __builtin_fmaf(ks[r], y[n].v[i], pk[i]);
            pq[i] = __builtin_fmaf(qs[r], y[n].v[i], pq[i]);
          }
      }
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      part[0][rg][cl * VEC + i] = pk[i];
      part[1][rg][cl * VEC + i] = pq[i];
    }
    __syncthreads();
    if (tid < COLS) {
      const int cc = blockIdx.x * COLS + tid;
      float tk = 0.0f, tq = 0.0f;
#pragma unroll
      for (int g = 0; g < RG; ++g) {
        tk += part[0][g][tid];
        tq += part[1][g][tid];
      }
      const float u = cc < a.dv ? beta * (to_f(v[cc]) - tk) : 0.0f;
      us[tid] = u;
      const float dot = (dot_sh[0] + dot_sh[1]) + (dot_sh[2] + dot_sh[3]);
      if (cc < a.dv) out[row * a.orow + cc] = from_f<T>(a.scale * __builtin_fmaf(dot, u, tq));
    }
    __syncthreads();
    if (mine) {
#pragma unroll
      for (int n = 0; n < NR; ++n) {
        const int r = rg + n * RG;
        if (r < a.dk) {
#pragma unroll
          for (int i = 0; i < VEC; ++i) y[n].v[i] = __builtin_fmaf(ks[r], us[cl * VEC + i], y[n].v[i]);
          *reinterpret_cast<Vec<float, VEC>*>(s + (int64_t)r * a.dv) = y[n];
        }
      }
    }
    if (next >= a.rows) return;
    row = next;
    __syncthreads();
  }
}

template <typename T, int VEC, int CL>
hipError_t launch_step_r(const DeltaStepArgs& a, hipStream_t st) {
  const int units = (a.dv + VEC - 1) / VEC, rows = (a.dk + 256 / CL - 1) / (256 / CL);
  const dim3 grid((unsigned)((units + CL - 1) / CL), (unsigned)a.heads, (unsigned)a.rows);
  if (rows <= 4) hipLaunchKernelGGL((delta_step_kernel<T, VEC, CL, 4>), grid, dim3(256), 0, st, a);
  else if (rows <= 8) hipLaunchKernelGGL((delta_step_kernel<T, VEC, CL, 8>), grid, dim3(256), 0, st, a);
  else if constexpr (CL == 32) hipLaunchKernelGGL((delta_step_kernel<T, VEC, CL, 16>), grid, dim3(256), 0, st, a);
  return hipGetLastError();
}

template <typename T, int VEC>
hipError_t launch_step_v(const DeltaStepArgs& a, hipStream_t st) {
  const int units = (a.dv + VEC - 1) / VEC;
  // 8 vectors of columns a workgroup (rows of dk / 32 a thread) where 32 would leave
  // most of the card idle (us; heads of 128: 256 workgroups of 32 11.7, of 8 10.0; 384
  // 13.1 and 14.5; 2048 62 and 63) or hold more than 16 rows a thread in registers
  // (heads of 256 x 256: 4096 282 and 228; 512 42 and 35)
  if (units <= 8 || a.dk > 128 || (int64_t)a.rows * a.heads * ((units + 31) / 32) < 320)
    return launch_step_r<T, VEC, 8>(a, st);
  return launch_step_r<T, VEC, 32>(a, st);
}

template <typename T>
hipError_t launch_step(const DeltaStepArgs& a, hipStream_t st) {
  const bool wide = a.dv % 4 == 0 && (uintptr_t)a.state % 16 == 0 && a.state_slot % 4 == 0;
  return wide ? launch_step_v<T, 4>(a, st) : launch_step_v<T, 1>(a, st);
}

}  // namespace

CF_API int cf_delta_attention_step(const CfDeltaStepArgs* p) {
  if (!p) return (int)hipErrorInvalidValue;
  const CfDeltaStepArgs& x = *p;
  if (x.rows < 0 || x.rows > CF_DECAY_MAX_SEQS || !delta_heads_fit(x.heads, x.q_heads, x.k_heads, x.v_heads) ||
      x.dk < 1 || x.dk > CF_DECAY_MAX_DK || x.dv < 1 || x.dv > CF_DECAY_MAX_DV || x.dtype < 0 ||
      x.dtype > 2 || x.pool < 0)
    return (int)hipErrorInvalidValue;
  if (x.rows == 0) return 0;
  if (!x.q || !x.k || !x.v || !x.beta || !x.out || (x.pool > 0 && !x.state) ||
      (!x.slots && x.pool < x.rows))
    return (int)hipErrorInvalidValue;
  DeltaStepArgs a;
  a.q = x.q; a.k = x.k; a.v = x.v;
  a.beta = x.beta; a.log_decay = x.log_decay;
  a.state = x.state;
  a.out = x.out;
  a.slots = x.slots; a.slots_wide = x.slots_wide != 0;
  a.beta_f32 = x.beta_f32 != 0; a.decay_f32 = x.decay_f32 != 0;
  a.rows = (int)x.rows; a.heads = (int)x.heads;
  a.q_group = (int)(x.heads / x.q_heads);
  a.k_group = (int)(x.heads / x.k_heads);
  a.v_group = (int)(x.heads / x.v_heads);
  a.dk = (int)x.dk; a.dv = (int)x.dv;
  a.pool = x.pool; a.state_slot = x.state_slot;
  a.qr = x.q_row; a.qh = x.q_head; a.kr = x.k_row; a.kh = x.k_head;
  a.vr = x.v_row; a.vh = x.v_head; a.orow = x.out_row; a.oh = x.out_head;
  a.br = x.beta_row; a.bh = x.beta_head; a.lr = x.decay_row; a.lh = x.decay_head;
  a.scale = (float)x.scale;
  hipStream_t st = (hipStream_t)x.stream;
  hipError_t e;
  if (x.dtype == SEQ_F32) e = launch_step<float>(a, st);
  else if (x.dtype == SEQ_F16) e = launch_step<_Float16>(a, st);
  else e = launch_step<bf16_t>(a, st);
  return (int)e;
}
