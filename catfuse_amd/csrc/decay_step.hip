// One token of each running sequence through the decayed attention, against
// a pool of states:
//   S <- w S + k v^T,   o = scale q S,   w = exp(log_decay[h])
// for row b and head h with S = state[slots[b]][h], dk x dv in fp32, updated
// in place.  Rows whose slot is outside the pool (negative ones mark padding)
// give zeros and touch no state.  Rows with the same slot are consecutive
// tokens of one sequence, in the order of the rows: the first one's workgroup
// takes them all, so no two workgroups meet in a state.
//
// No counterpart in the reference.
#include "cf_seq.h"

namespace {

struct StepArgs {
  const void* q;
  const void* k;
  const void* v;
  const float* log_decay;
  float* state;
  void* out;
  const void* slots;
  int slots_wide;
  int rows, heads, group, dk, dv;
  int64_t pool, state_slot;
  int64_t qr, qh, kr, kh, vr, vh, orow, oh;
  float scale;
};

__device__ __forceinline__ int64_t step_slot(const StepArgs& a, int i) {
  if (a.slots == nullptr) return i;
  return a.slots_wide ? reinterpret_cast<const int64_t*>(a.slots)[i]
                      : (int64_t)reinterpret_cast<const int32_t*>(a.slots)[i];
}

constexpr int STEP_MAX_DK = CF_DECAY_MAX_DK;

// Bound by HBM: every state is read and written once.  A workgroup takes a
// slice of CL * VEC columns of one row and head: thread = VEC columns, 256 /
// CL row groups, U rows in flight each.  256 rows x 32 heads of 128 x 128:
// 214 us, 5.0 TB/s read and written, a large copy's rate; loads of the states
// before the scan of the slots, or streaming stores, were no faster.
template <typename T, int VEC, int CL>
__global__ __launch_bounds__(256) void decay_step_kernel(StepArgs a) {
  constexpr int RG = 256 / CL, U = 8;
  __shared__ float qs[STEP_MAX_DK], ks[STEP_MAX_DK];
  __shared__ float part[RG][CL * VEC];
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
  // w as a sum of two floats: the rounding of one would shift the horizon of a
  // slow decay by the token (1e-4 of a state after 4096 tokens)
  const double wd = exp((double)a.log_decay[h]);
  const float w = (float)wd, wl = wd < 1e300 ? (float)(wd - (double)w) : 0.0f;
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
    const T* const q = (const T*)a.q + row * a.qr + h * a.qh;
    const T* const k = (const T*)a.k + row * a.kr + (h / a.group) * a.kh;
    const T* const v = (const T*)a.v + row * a.vr + (h / a.group) * a.vh;
    for (int i = tid; i < a.dk; i += 256) {
      qs[i] = to_f(q[i]);
      ks[i] = to_f(k[i]);
    }
    float x[VEC], p[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      x[i] = mine ? to_f(v[c + i]) : 0.0f;
      p[i] = 0.0f;
    }
    __syncthreads();
    if (mine) {
      for (int d0 = rg; d0 < a.dk; d0 += RG * U) {
        Vec<float, VEC> y[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (d0 + u * RG < a.dk)
            y[u] = *reinterpret_cast<const Vec<float, VEC>*>(s + (int64_t)(d0 + u * RG) * a.dv);
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int d = d0 + u * RG;
          if (d >= a.dk) break;
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            y[u].v[i] = __builtin_fmaf(y[u].v[i], w, __builtin_fmaf(y[u].v[i], wl, ks[d] * x[i]));
            p[i] = __builtin_fmaf(qs[d], y[u].v[i], p[i]);
          }
          *reinterpret_cast<Vec<float, VEC>*>(s + (int64_t)d * a.dv) = y[u];
        }
      }
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) part[rg][cl * VEC + i] = p[i];
    __syncthreads();
    for (int i = tid; i < CL * VEC; i += 256) {
      const int cc = blockIdx.x * CL * VEC + i;
      if (cc < a.dv) {
        float t = 0.0f;
        for (int g = 0; g < RG; ++g) t += part[g][i];
        out[row * a.orow + cc] = from_f<T>(t * a.scale);
      }
    }
    if (next >= a.rows) return;
    row = next;
    __syncthreads();
  }
}

template <typename T, int VEC>
hipError_t launch_step_v(const StepArgs& a, hipStream_t st) {
  const int units = (a.dv + VEC - 1) / VEC;
  auto grid = [&](int cl) {
    return dim3((unsigned)((units + cl - 1) / cl), (unsigned)a.heads, (unsigned)a.rows);
  };
  if (units <= 8)
    hipLaunchKernelGGL((decay_step_kernel<T, VEC, 8>), grid(8), dim3(256), 0, st, a);
  else if (units <= 16)
    hipLaunchKernelGGL((decay_step_kernel<T, VEC, 16>), grid(16), dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((decay_step_kernel<T, VEC, 32>), grid(32), dim3(256), 0, st, a);
  return hipGetLastError();
}

template <typename T>
hipError_t launch_step(const StepArgs& a, hipStream_t st) {
  const bool wide = a.dv % 4 == 0 && (uintptr_t)a.state % 16 == 0 && a.state_slot % 4 == 0;
  return wide ? launch_step_v<T, 4>(a, st) : launch_step_v<T, 1>(a, st);
}

}  // namespace

CF_API int cf_decay_attention_step(const CfDecayStepArgs* p) {
  if (!p) return (int)hipErrorInvalidValue;
  const CfDecayStepArgs& x = *p;
  if (x.rows < 0 || x.rows > CF_DECAY_MAX_SEQS || x.heads < 1 || x.kv_heads < 1 ||
      x.heads % x.kv_heads != 0 || x.heads > CF_SEQ_MAX_HEADS || x.dk < 1 ||
      x.dk > CF_DECAY_MAX_DK || x.dv < 1 || x.dv > CF_DECAY_MAX_DV || x.dtype < 0 || x.dtype > 2 ||
      x.pool < 0)
    return (int)hipErrorInvalidValue;
  if (x.rows == 0) return 0;
  if (!x.q || !x.k || !x.v || !x.log_decay || !x.out || (x.pool > 0 && !x.state) ||
      (!x.slots && x.pool < x.rows))
    return (int)hipErrorInvalidValue;
  StepArgs a;
  a.q = x.q; a.k = x.k; a.v = x.v;
  a.log_decay = x.log_decay;
  a.state = x.state;
  a.out = x.out;
  a.slots = x.slots; a.slots_wide = x.slots_wide != 0;
  a.rows = (int)x.rows; a.heads = (int)x.heads; a.group = (int)(x.heads / x.kv_heads);
  a.dk = (int)x.dk; a.dv = (int)x.dv;
  a.pool = x.pool; a.state_slot = x.state_slot;
  a.qr = x.q_row; a.qh = x.q_head; a.kr = x.k_row; a.kh = x.k_head;
  a.vr = x.v_row; a.vh = x.v_head; a.orow = x.out_row; a.oh = x.out_head;
  a.scale = (float)x.scale;
  hipStream_t st = (hipStream_t)x.stream;
  hipError_t e;
  if (x.dtype == SEQ_F32) e = launch_step<float>(a, st);
  else if (x.dtype == SEQ_F16) e = launch_step<_Float16>(a, st);
  else e = launch_step<bf16_t>(a, st);
  return (int)e;
}
