// Distillation from a teacher's top logits for gfx950: KL(p || softmax(s / T)) per row where the teacher's distribution p is known on k of the K
// classes only, loss and gradient in one pass over the student's row.
//   kept classes j: without t_lse p_j = softmax over the kept t_j / T; with t_lse (the teacher's log-sum-exp over all K at that temperature)
//   p_j = exp(t_j / T - t_lse), and everything else is one bucket, p_rest = max(0, 1 - sum p_j) against q_rest = sum of q over the classes not kept.
//   loss = w (sum_j p_j (log p_j - log q_j) + p_rest (log p_rest - log q_rest)),   w = coef * row_weight
//   dlogits = w / T * { q_j - p_j  kept;  q_i (1 - p_rest / q_rest)  others }
// Bound by memory: the row is read once and its gradient written once.  A row of up to 64 elements (128 of 16 bits) per thread of one workgroup stays
// in registers between the passes over it (maximum, sum of exponentials, gradient); longer rows are read three times, through the caches.
// The classes not kept are summed on their own (a bitmap in LDS says which are) against their own maximum: q_rest as 1 - sum of the kept q would
// cancel, and p_rest is formed in 64 bits for the same reason.  The kept classes' gradients overwrite the row's after a barrier.
#include "lt_common.h"

namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr int MAX_K = 1024;         // kept entries of a row
constexpr int MAX_CLASSES = 1 << 18;   // (their bitmap and the kept entries fit 64 KiB of LDS)

struct TopkArgs {
  const void* s; void* d;
  const void* t_val; const void* t_idx; const float* t_lse; const float* row_weight;
  float* loss_rows;
  int64_t ld, ldd, ldv, ldi;
  int rows, K, k, idx64, val_dt;
  float inv_temp, coef;
};

struct bf_t { uint16_t u; };
struct hf_t { uint16_t u; };
__device__ __forceinline__ float getf(float x) { return x; }
__device__ __forceinline__ float getf(bf_t x) { return bf2f(x.u); }
__device__ __forceinline__ float getf(hf_t x) { return (float)__builtin_bit_cast(_Float16, x.u); }
template <typename T> __device__ __forceinline__ T putf(float x);
template <> __device__ __forceinline__ float putf<float>(float x) { return x; }
template <> __device__ __forceinline__ bf_t putf<bf_t>(float x) { return {f2bf(x)}; }
template <> __device__ __forceinline__ hf_t putf<hf_t>(float x) { return {__builtin_bit_cast(uint16_t, (_Float16)x)}; }
template <typename T, int E> struct alignas(E * sizeof(T)) Pack { T v[E]; };

__device__ __forceinline__ double wave_sum_d(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
__device__ __forceinline__ double block_sum_d(double v, double* red) {
  v = wave_sum_d(v);
  const int w = threadIdx.x >> 6, nw = (blockDim.x + 63) >> 6;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[w] = v;
  __syncthreads();
  double s = 0.0;
  for (int i = 0; i < nw; ++i) s += red[i];
  return s;
}
__device__ __forceinline__ float teacher_value(const TopkArgs& a, int64_t row, int j) {
  const int64_t at = row * a.ldv + j;
  if (a.val_dt == LT_DT_F32) return static_cast<const float*>(a.t_val)[at];
  if (a.val_dt == LT_DT_BF16) return getf(static_cast<const bf_t*>(a.t_val)[at]);
  return getf(static_cast<const hf_t*>(a.t_val)[at]);
}
// class of entry j, -1 for a missing one (any index outside 0 .. K - 1)
__device__ __forceinline__ int teacher_class(const TopkArgs& a, int64_t row, int j) {
  const int64_t at = row * a.ldi + j, c = a.idx64 ? static_cast<const int64_t*>(a.t_idx)[at] : static_cast<const int32_t*>(a.t_idx)[at];
  return c >= 0 && c < a.K ? (int)c : -1;
}

// NV chunks of E elements per thread, chunk i of thread t at element (i * blockDim + t) * E.  KEEP: they stay in registers; otherwise NV is ignored and
// every pass reads the row again.
template <typename TS, typename TD, int E, int NV, bool KEEP>
__global__ __launch_bounds__(1024) void topk_kl_kernel(const TopkArgs a) {
  extern __shared__ uint32_t dyn[];       // [ceil(K / 32)] kept bits | [k] class | [k] probability
  __shared__ float red[32];
  __shared__ double redd[16];
  __shared__ int twice;
  const int nt = blockDim.x, words = (a.K + 31) >> 5;
  uint32_t* bits = dyn;
  int* cls = reinterpret_cast<int*>(dyn + words);
  float* prob = reinterpret_cast<float*>(cls + a.k);
  const int64_t row = blockIdx.x;
  const TS* s = static_cast<const TS*>(a.s) + row * a.ld;
  TD* d = static_cast<TD*>(a.d) + row * a.ldd;
  const float w = a.coef * (a.row_weight ? a.row_weight[row] : 1.f), c = a.inv_temp * LOG2E;
  const int chunks = (a.K + E - 1) / E;
  typedef Pack<TS, E> PS;
  typedef Pack<TD, E> PD;

  PS v[KEEP ? NV : 1];
  if constexpr (KEEP) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int ch = i * nt + threadIdx.x;
      if (ch < chunks) v[i] = *reinterpret_cast<const PS*>(s + (int64_t)ch * E);
    }
  }
  // ---- the kept entries
  for (int i = threadIdx.x; i < words; i += nt) bits[i] = 0;
  if (threadIdx.x == 0) twice = 0;
  __syncthreads();
  for (int j = threadIdx.x; j < a.k; j += nt) {
    const int x = teacher_class(a, row, j);
    cls[j] = x;
    if (x >= 0 && (atomicOr(&bits[x >> 5], 1u << (x & 31)) >> (x & 31)) & 1) twice = 1;
  }
  __syncthreads();
  if (twice) {     // an index again in its row: its first entry counts
    for (int j = threadIdx.x; j < a.k; j += nt) {
      const int x = teacher_class(a, row, j);
      bool again = false;
      for (int i = 0; i < j && !again; ++i) again = x >= 0 && teacher_class(a, row, i) == x;
      if (again) cls[j] = -1;
    }
    __syncthreads();
  }
  float tmax = -INFINITY, zmax = -INFINITY;
  int mine = 0;
  for (int j = threadIdx.x; j < a.k; j += nt)
    if (cls[j] >= 0) {
      ++mine;
      tmax = fmaxf(tmax, teacher_value(a, row, j));
      zmax = fmaxf(zmax, getf(s[cls[j]]));
    }
  const int kept = (int)block_sum((float)mine, red);   // <= 1024: exact
  tmax = block_max(tmax, red);
  zmax = block_max(zmax, red);
  if (kept == 0 || w == 0.f || (!a.t_lse && tmax == -INFINITY)) {   // nothing known of this row, or nothing asked
    if (threadIdx.x == 0) a.loss_rows[row] = 0.f;
    if (a.d)
      for (int ch = threadIdx.x; ch < chunks; ch += nt) {
        PD o;
#pragma unroll
        for (int e = 0; e < E; ++e) o.v[e] = putf<TD>(0.f);
        *reinterpret_cast<PD*>(d + (int64_t)ch * E) = o;
      }
    return;
  }
  // ---- the student's classes that are not kept: maximum, then the sum of exponentials against it
  float mrest = -INFINITY;
  auto bits_of = [&](int ch) -> uint32_t { return E == 1 ? bits[ch >> 5] >> (ch & 31) : bits[(ch * E) >> 5] >> ((ch * E) & 31); };
  auto each = [&](auto&& f) {
    if constexpr (KEEP) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int ch = i * nt + threadIdx.x;
        if (ch < chunks) f(ch, v[i]);
      }
    } else {
      for (int ch = threadIdx.x; ch < chunks; ch += nt) f(ch, *reinterpret_cast<const PS*>(s + (int64_t)ch * E));
    }
  };
  each([&](int ch, const PS& x) {
    const uint32_t m = bits_of(ch);
#pragma unroll
    for (int e = 0; e < E; ++e) mrest = fmaxf(mrest, (m >> e) & 1 ? -INFINITY : getf(x.v[e]));
  });
  mrest = block_max(mrest, red);
  const float mr = mrest == -INFINITY ? 0.f : mrest, nmr = -mr * c;
  float srest = 0.f;
  each([&](int ch, const PS& x) {
    const uint32_t m = bits_of(ch);
#pragma unroll
    for (int e = 0; e < E; ++e) srest += (m >> e) & 1 ? 0.f : __builtin_amdgcn_exp2f(fmaf(getf(x.v[e]), c, nmr));
  });
  srest = block_sum(srest, red);
  // ---- teacher probabilities and the kept classes' share of the student
  const float m = fmaxf(zmax, mrest);
  float stop = 0.f, tsum = 0.f;
  double psum = 0.0;
  for (int j = threadIdx.x; j < a.k; j += nt) {
    float p = 0.f;
    if (cls[j] >= 0) {
      const float t = teacher_value(a, row, j);
      if (a.t_lse) {
        const double pd = exp((double)t * (double)a.inv_temp - (double)a.t_lse[row]);
        psum += pd;
        p = (float)pd;
      } else {
        p = __expf((t - tmax) * a.inv_temp);
        tsum += p;
      }
      stop += __builtin_amdgcn_exp2f((getf(s[cls[j]]) - m) * c);
    }
    prob[j] = p;
  }
  stop = block_sum(stop, red);
  float rest = 0.f, pmul = 1.f;
  if (a.t_lse) {
    psum = block_sum_d(psum, redd);
    rest = kept < a.K && psum < 1.0 ? (float)(1.0 - psum) : 0.f;
  } else {
    pmul = 1.f / block_sum(tsum, red);
  }
  const float frest = mrest == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((mrest - m) * c);
  const float total = stop + srest * frest, lt = __logf(total);
  float part = 0.f;
  for (int j = threadIdx.x; j < a.k; j += nt)
    if (cls[j] >= 0) {
      const float p = prob[j] * pmul;
      if (p > 0.f) {
        const float logp = a.t_lse ? (float)((double)teacher_value(a, row, j) * (double)a.inv_temp - (double)a.t_lse[row])
                                   : (teacher_value(a, row, j) - tmax) * a.inv_temp + __logf(pmul);
        part += p * (logp - ((getf(s[cls[j]]) - m) * a.inv_temp - lt));
      }
    }
  part = block_sum(part, red);
  if (threadIdx.x == 0) {
    if (rest > 0.f) part += rest * (__logf(rest) - ((mr - m) * a.inv_temp + __logf(srest) - lt));   // srest = 0: +inf
    a.loss_rows[row] = w * part;
  }
  if (!a.d) return;
  // ---- gradient
  const float g = w * a.inv_temp, gr = g * (frest / total - (srest > 0.f ? rest / srest : 0.f));
  each([&](int ch, const PS& x) {
    PD o;
#pragma unroll
    for (int e = 0; e < E; ++e) o.v[e] = putf<TD>(gr * __builtin_amdgcn_exp2f(fmaf(getf(x.v[e]), c, nmr)));
    *reinterpret_cast<PD*>(d + (int64_t)ch * E) = o;
  });
  __syncthreads();
  for (int j = threadIdx.x; j < a.k; j += nt)
    if (cls[j] >= 0) d[cls[j]] = putf<TD>(g * (__builtin_amdgcn_exp2f((getf(s[cls[j]]) - m) * c) / total - prob[j] * pmul));
}

// loss[0] += sum of the rows' losses, in a fixed order
__global__ __launch_bounds__(256) void topk_loss_kernel(const float* __restrict__ terms, int rows, float* __restrict__ loss) {
  __shared__ float red[32];
  float s = 0.f;
  for (int r = threadIdx.x; r < rows; r += 256) s += terms[r];
  s = block_sum(s, red);
  if (threadIdx.x == 0) loss[0] += s;
}

template <typename TS, typename TD, int E, int NV, bool KEEP> void go(const TopkArgs& a, int nt, hipStream_t st) {
  const size_t lds = ((size_t)((a.K + 31) / 32) + 2 * (size_t)a.k) * 4;
  hipLaunchKernelGGL((topk_kl_kernel<TS, TD, E, NV, KEEP>), dim3(a.rows), dim3(nt), lds, st, a);
}
// threads of a workgroup: the fewest waves whose registers hold the row
int threads_for(int chunks, int nv) {
  int nt = 64;
  while (nt < 1024 && (int64_t)nt * nv < chunks) nt *= 2;
  return nt;
}
template <typename TS, typename TD> void dispatch(const TopkArgs& a, hipStream_t st) {
  constexpr int E = 16 / sizeof(TS);
  const bool vec = a.K % E == 0 && a.ld % E == 0 && ((uintptr_t)a.s & 15) == 0 && (!a.d || (a.ldd % E == 0 && ((uintptr_t)a.d & (E * sizeof(TD) - 1)) == 0));
  if (vec) {
    const int chunks = a.K / E;
    if (chunks <= 4 * 1024) go<TS, TD, E, 4, true>(a, threads_for(chunks, 4), st);
    else if (chunks <= 16 * 1024) go<TS, TD, E, 16, true>(a, threads_for(chunks, 16), st);
    else go<TS, TD, E, 1, false>(a, 1024, st);
  } else {   // rows that are not whole 16-byte pieces: one element per lane and load
    if (a.K <= 16 * 1024) go<TS, TD, 1, 16, true>(a, threads_for(a.K, 16), st);
    else go<TS, TD, 1, 1, false>(a, 1024, st);
  }
}

}  // namespace

extern "C" int lt_topk_kl_fwd_bwd(const void* s, int s_dtype, int64_t ld, const void* t_val, int val_dtype, int64_t ldv, const void* t_idx, int idx_is_64, int64_t ldi,
                                  const float* t_lse, const float* row_weight, float inv_temp, float coef, float* loss_rows, float* loss, void* dlogits, int d_dtype,
                                  int64_t ldd, int rows, int K, int k, void* stream) {
  LT_CHECK_ARG(rows >= 0 && K >= 1 && K <= MAX_CLASSES && k >= 1 && k <= MAX_K && k <= K, "lt_topk_kl_fwd_bwd: 1 <= k <= min(K, %d), K <= %d (got K %d, k %d, rows %d)", MAX_K,
               MAX_CLASSES, K, k, rows);
  LT_CHECK_ARG(inv_temp > 0.f && inv_temp < INFINITY, "lt_topk_kl_fwd_bwd: inv_temp must be positive and finite");
  LT_CHECK_ARG(s_dtype >= 0 && s_dtype <= 2 && val_dtype >= 0 && val_dtype <= 2 && (d_dtype == s_dtype || (s_dtype == LT_DT_F32 && d_dtype == LT_DT_BF16)),
               "lt_topk_kl_fwd_bwd: dlogits have the type of s, or are bf16 for f32 s");
  if (rows == 0) return LT_OK;
  LT_CHECK_ARG(s && t_val && t_idx && loss_rows && ld >= K && ldv >= k && ldi >= k && (!dlogits || ldd >= K), "lt_topk_kl_fwd_bwd: missing pointers or rows shorter than K / k");
  TopkArgs a;
  a.s = s; a.d = dlogits; a.t_val = t_val; a.t_idx = t_idx; a.t_lse = t_lse; a.row_weight = row_weight; a.loss_rows = loss_rows;
  a.ld = ld; a.ldd = dlogits ? ldd : 0; a.ldv = ldv; a.ldi = ldi;
  a.rows = rows; a.K = K; a.k = k; a.idx64 = idx_is_64; a.val_dt = val_dtype; a.inv_temp = inv_temp; a.coef = coef;
  hipStream_t st = (hipStream_t)stream;
  if (s_dtype == LT_DT_F32) { if (d_dtype == LT_DT_F32) dispatch<float, float>(a, st); else dispatch<float, bf_t>(a, st); }
  else if (s_dtype == LT_DT_BF16) dispatch<bf_t, bf_t>(a, st);
  else dispatch<hf_t, hf_t>(a, st);
  if (loss) hipLaunchKernelGGL(topk_loss_kernel, dim3(1), dim3(256), 0, st, loss_rows, rows, loss);
  LT_CHECK_LAUNCH("lt_topk_kl_fwd_bwd");
}
