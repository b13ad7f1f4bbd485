// Distillation from a teacher's top logits for gfx950: KL(p || softmax(s / T)) per row where the teacher's distribution p is known on k of the K
// classes only, loss and gradient in one pass over the student's row.
//   kept classes j: without t_lse p_j = softmax over the kept t_j / T; with t_lse (the teacher's log-sum-exp over all K at that temperature)
//   p_j = exp(t_j / T - t_lse), and everything else is one bucket, p_rest = max(0, 1 - sum p_j) against q_rest = sum of q over the classes not kept.
//   loss = w (sum_j p_j (log p_j - log q_j) + p_rest (log p_rest - log q_rest)),   w = coef * row_weight
//   dlogits = w / T * { m q_j - p_j  kept;  q_i (m - p_rest / q_rest)  others },   m = sum p_j + p_rest
// m is 1 wherever there is a bucket (p_rest = 1 - sum p_j) and for renormalised values.  Kept probabilities whose sum passes 1 (values stored in 16 bits next to a
// 32-bit t_lse: up to 1.04 for a sure teacher), or rows of which every class is kept, have no bucket: there m = sum p_j, or the gradient were not the loss's.
// Bound by memory: the row is read once and its gradient written once.  The registers of a workgroup of 512 threads hold a row of up to 65 536 fp32 or 16-bit
// values (32 or 16 pieces of 16 bytes a thread) between the three passes over it (maximum, sum of exponentials, gradient); what does not fit is read again,
// through the caches (a sixteenth of the row costs ~10 us at 2048 x 65 536).  Spilled beside them: 10 registers a lane of row-long values and descriptors in the
// fp32 form, 13 - 17 in the 16-bit forms (12 for their short rows), 2 - 8 where rows are not whole pieces; what that costs was not separated.  Rates reached
// elsewhere: 16-bit rows of 65 536 2.9 TB/s, of 131 072 (half of it streamed) 2.6; 1024 x 50 257 (one element a load) fp32 2.3, bf16 1.7.  One workgroup to a CU walks the rows and requests each piece of the next row behind
// the store of this one's: 2048 x 65 536 fp32 -> bf16 with 256 kept, 207 us (3.9 TB/s of the 5.0 that a copy reaches; one row a workgroup: 246 us).
// The classes not kept are summed on their own (a bitmap in LDS says which are) against their own maximum: q_rest as 1 - sum of the kept q would
// cancel, and p_rest is formed in 64 bits for the same reason.  The kept classes' gradients overwrite the row's after a barrier.
#include "lt_common.h"

namespace {

typedef __attribute__((ext_vector_type(4))) uint32_t u32x4_t;
typedef __attribute__((ext_vector_type(2))) uint32_t u32x2_t;
constexpr float LOG2E = 1.4426950408889634f;
constexpr int CUS = 256;
constexpr int MAX_GRID = 1 << 20;   // (a launch has fewer than 2^32 threads; the workgroups walk what is beyond)
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

// A row behind a buffer descriptor: what lies past its end reads as zeros and is not written, and no lane needs a condition or a 64-bit address.
struct Row {
  __amdgpu_buffer_rsrc_t r;
  __device__ __forceinline__ Row(const void* p, uint32_t bytes) {
    const uint64_t u = (uint64_t)p;
    const uint64_t q = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)u) |
                       ((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(u >> 32)) << 32);
    r = __builtin_amdgcn_make_buffer_rsrc((void*)q, 0, (int)bytes, 0x00020000);
  }
  template <typename P> __device__ __forceinline__ P get(int off) const {
    if constexpr (sizeof(P) == 16) return __builtin_bit_cast(P, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0));
    else if constexpr (sizeof(P) == 4) return __builtin_bit_cast(P, __builtin_amdgcn_raw_buffer_load_b32(r, off, 0, 0));
    else return __builtin_bit_cast(P, __builtin_amdgcn_raw_buffer_load_b16(r, off, 0, 0));
  }
  template <typename P> __device__ __forceinline__ void put(int off, const P& x) const {
    if constexpr (sizeof(P) == 16) __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_t, x), r, off, 0, 0);
    else if constexpr (sizeof(P) == 8) __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2_t, x), r, off, 0, 0);
    else if constexpr (sizeof(P) == 4) __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, x), r, off, 0, 0);
    else __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(uint16_t, x), r, off, 0, 0);
  }
};
__device__ __forceinline__ double wave_sum_d(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
// two maxima and a count over the workgroup, one pair of barriers
__device__ __forceinline__ void block_max2_sum(float& x, float& y, int n, float* red, int& total) {
  x = wave_max(x);
  y = wave_max(y);
  float f = wave_sum((float)n);     // <= 1024: exact
  const int w = threadIdx.x >> 6, nw = (blockDim.x + 63) >> 6;
  float4* r = reinterpret_cast<float4*>(red);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) r[w] = make_float4(x, y, f, 0.f);
  __syncthreads();
  float4 a = r[0];
  for (int i = 1; i < nw; ++i) { const float4 b = r[i]; a.x = fmaxf(a.x, b.x); a.y = fmaxf(a.y, b.y); a.z += b.z; }
  x = a.x; y = a.y;
  total = (int)a.z;
}
// two sums, and two in 64 bits
__device__ __forceinline__ void block_sum4(float& x, float& y, double& p, double& q, float* red, double* redd) {
  x = wave_sum(x);
  y = wave_sum(y);
  p = wave_sum_d(p);
  q = wave_sum_d(q);
  const int w = threadIdx.x >> 6, nw = (blockDim.x + 63) >> 6;
  float2* r = reinterpret_cast<float2*>(red);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) { r[w] = make_float2(x, y); redd[2 * w] = p; redd[2 * w + 1] = q; }
  __syncthreads();
  float2 a = r[0];
  double b = redd[0], d = redd[1];
  for (int i = 1; i < nw; ++i) { a.x += r[i].x; a.y += r[i].y; b += redd[2 * i]; d += redd[2 * i + 1]; }
  x = a.x; y = a.y;
  p = b; q = d;
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

// Chunk i of thread t: E elements at (i * blockDim + t) * E.  The first NV chunks of a thread stay in registers, any further ones are read again in
// every pass.  A workgroup walks rows blockIdx.x, + gridDim.x, ...: the next row's chunk is requested right behind the store of the chunk that held its
// registers, its kept entries ahead of that.
constexpr int EPT = 1;   // kept entries per thread that are requested ahead (all of them up to k = 512: workgroups that walk rows have 512 threads)
template <typename TS, typename TD, int E, int NV, int NTMAX>
__global__ __launch_bounds__(NTMAX) void topk_kl_kernel(const TopkArgs a) {
  extern __shared__ double dyn[];       // [k] exp(t) in 64 bits | [ceil(max(K, NV * blockDim * E) / 32)] kept bits (set past K) | [k] class | [k] teacher value | [k] student logit
  __shared__ __attribute__((aligned(16))) float red[64];
  __shared__ double redd[32];
  __shared__ int twice;
  const int nt = blockDim.x, words = (max(a.K, NV * nt * E) + 31) >> 5;
  double* ex = dyn;
  uint32_t* bits = reinterpret_cast<uint32_t*>(dyn + a.k);
  int* cls = reinterpret_cast<int*>(bits + words);
  float* val = reinterpret_cast<float*>(cls + a.k);
  float* zs = val + a.k;
  const int chunks = (a.K + E - 1) / E;
  const float c = a.inv_temp * LOG2E;
  typedef Pack<TS, E> PS;
  typedef Pack<TD, E> PD;

  PS v[NV];
  int at = threadIdx.x;      // (opaque to the compiler in every row: it would otherwise keep one offset per chunk alive through the loop)
  auto load = [&](const Row& s, int i) { v[i] = s.get<PS>((at + i * nt) * (int)sizeof(PS)); };
  // entry j of a row: class and teacher value, then the student's logit there
  int ecls[EPT];
  float eval[EPT], ez[EPT];
  auto entries = [&](int64_t row) {
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
      const int j = i * nt + threadIdx.x;
      ecls[i] = j < a.k ? teacher_class(a, row, j) : -1;
      eval[i] = j < a.k ? teacher_value(a, row, j) : 0.f;
    }
  };
  auto gather = [&](const TS* s) {
#pragma unroll
    for (int i = 0; i < EPT; ++i) ez[i] = ecls[i] >= 0 ? getf(s[ecls[i]]) : 0.f;
  };
  for (int i = threadIdx.x; i < words; i += nt) bits[i] = i * 32 >= a.K ? 0xffffffffu : a.K - i * 32 >= 32 ? 0u : 0xffffffffu << (a.K - i * 32);
  if (threadIdx.x == 0) twice = 0;
  int64_t row = blockIdx.x;
  entries(row);
  gather(static_cast<const TS*>(a.s) + row * a.ld);
  {
    const Row r(static_cast<const TS*>(a.s) + row * a.ld, a.K * sizeof(TS));
#pragma unroll
    for (int i = 0; i < NV; ++i) load(r, i);
  }
  __syncthreads();

  for (; row < a.rows; row += gridDim.x) {
    asm volatile("" : "+v"(at));
    const TS* s = static_cast<const TS*>(a.s) + row * a.ld;
    TD* d = static_cast<TD*>(a.d) + row * a.ldd;
    const bool more = row + gridDim.x < a.rows;
    const TS* sn = s + (more ? (int64_t)gridDim.x * a.ld : 0);
    const Row rn(sn, more ? a.K * sizeof(TS) : 0), rd(d, a.d ? a.K * sizeof(TD) : 0);
    const float w = a.coef * (a.row_weight ? a.row_weight[row] : 1.f);
    // ---- the kept entries into LDS
    auto keep = [&](int j, int x, float t, float z) {
      cls[j] = x;
      val[j] = t;
      zs[j] = z;
      if (x >= 0 && (atomicOr(&bits[x >> 5], 1u << (x & 31)) >> (x & 31)) & 1) twice = 1;
    };
#pragma unroll
    for (int i = 0; i < EPT; ++i)
      if (i * nt + (int)threadIdx.x < a.k) keep(i * nt + threadIdx.x, ecls[i], eval[i], ez[i]);
    for (int j = EPT * nt + threadIdx.x; j < a.k; j += nt) {
      const int x = teacher_class(a, row, j);
      keep(j, x, teacher_value(a, row, j), x >= 0 ? getf(s[x]) : 0.f);
    }
    __syncthreads();
    if (twice) {     // an index again in its row: its first entry counts
#pragma unroll 1
      for (int j = threadIdx.x; j < a.k; j += nt) {
        const int x = teacher_class(a, row, j);
        bool again = false;
        for (int i = 0; i < j && !again; ++i) again = x >= 0 && teacher_class(a, row, i) == x;
        if (again) cls[j] = -1;
      }
      __syncthreads();
    }
    // ---- teacher probabilities, while the row itself is still on its way.  The loss is a difference of logarithms many times its size: its k terms and
    // the logarithms it ends in are formed in 64 bits.
    float tmax = -INFINITY, zmax = -INFINITY;
    int mine = 0;
#pragma unroll 1
    for (int j = threadIdx.x; j < a.k; j += nt)
      if (cls[j] >= 0) {
        ++mine;
        tmax = fmaxf(tmax, val[j] == val[j] ? val[j] : INFINITY);     // (fmaxf drops NaN: a row that knows nothing else would pass for one without entries)
        zmax = fmaxf(zmax, zs[j]);
      }
    if (!a.t_lse) tmax = block_max(tmax, red);
    const double tref = a.t_lse ? (double)a.t_lse[row] : (double)tmax * (double)a.inv_temp;
    double psum = 0.0, cross = 0.0;
#pragma unroll 1
    for (int j = threadIdx.x; j < a.k; j += nt)
      if (cls[j] >= 0) {
        const double t = (double)val[j] * (double)a.inv_temp - tref, p = exp(t);
        psum += p;
        if (p > 0.0) cross += p * (t - (double)zs[j] * (double)a.inv_temp);
        ex[j] = p;
      }
    // ---- the student's classes that are not kept: maximum, then the sum of exponentials against it.  A kept class becomes -inf here.
    auto hide = [&](int ch, PS& x) {
      const uint32_t m = bits[(ch * E) >> 5] >> ((ch * E) & 31);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        if ((m >> e) & 1) x.v[e] = putf<TS>(-INFINITY);
      }
    };
    auto each = [&](auto&& f) {
#pragma unroll
      for (int i = 0; i < NV; ++i) f(v[i]);
#pragma unroll 2
      for (int ch = NV * nt + threadIdx.x; ch < chunks; ch += nt) {
        PS x = *reinterpret_cast<const PS*>(s + (int64_t)ch * E);
        hide(ch, x);
        f(x);
      }
    };
#pragma unroll
    for (int i = 0; i < NV; ++i) hide(i * nt + at, v[i]);
    float mrest = -INFINITY;
    each([&](const PS& x) {
#pragma unroll
      for (int e = 0; e < E; ++e) mrest = fmaxf(mrest, getf(x.v[e]));
    });
    int kept;
    block_max2_sum(zmax, mrest, mine, red, kept);
    const bool live = kept > 0 && w != 0.f && (a.t_lse || tmax > -INFINITY);   // otherwise nothing is known of this row, or nothing asked
    const float mr = mrest == -INFINITY ? 0.f : mrest, m = fmaxf(zmax, mrest);
    float srest = 0.f, stop = 0.f;
    // (differences first, then the scale: x c - m c would carry the rounding of m c into every term alike, and so into the loss)
    each([&](const PS& x) {
#pragma unroll
      for (int e = 0; e < E; ++e) srest += __builtin_amdgcn_exp2f((getf(x.v[e]) - mr) * c);
    });
#pragma unroll 1
    for (int j = threadIdx.x; j < a.k; j += nt)
      if (cls[j] >= 0) stop += __builtin_amdgcn_exp2f((zs[j] - m) * c);
    block_sum4(srest, stop, psum, cross, red, redd);
    const float rest = a.t_lse && kept < a.K && psum < 1.0 ? (float)(1.0 - psum) : 0.f;
    const float frest = mrest == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((mrest - m) * c);
    const float total = stop + srest * frest, pmul = a.t_lse ? 1.f : (float)(1.0 / psum);
    const float g = w * a.inv_temp, mass = a.t_lse && rest == 0.f ? (float)psum : 1.f, gr = g * (frest / total * mass - (srest > 0.f ? rest / srest : 0.f));
    // ---- gradient
    if (more) { entries(row + gridDim.x); gather(sn); }
    const float cl = live ? c : 0.f, gl = live ? gr : 0.f, ml = live ? mr : 0.f;
    auto grad = [&](const PS& x) {
      PD o;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float z = live ? getf(x.v[e]) : 0.f;      // (a row that is not asked for may hold NaN)
        o.v[e] = putf<TD>(gl * __builtin_amdgcn_exp2f((z - ml) * cl));
      }
      return o;
    };
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      rd.put((at + i * nt) * (int)sizeof(PD), grad(v[i]));
      load(rn, i);
    }
    if (a.d) {
#pragma unroll 2
      for (int ch = NV * nt + threadIdx.x; ch < chunks; ch += nt) *reinterpret_cast<PD*>(d + (int64_t)ch * E) = grad(*reinterpret_cast<const PS*>(s + (int64_t)ch * E));
    }
    __syncthreads();     // the row's stores come before the kept classes'
    if (threadIdx.x == 0) {
      const double lt = log((double)total);
      const double lq = (double)m * (double)a.inv_temp + lt;      // log sum exp of the student's row
      double loss = a.t_lse ? cross + lq * psum : cross / psum - log(psum) + lq;
      if (rest > 0.f) loss += (double)rest * (log((double)rest) - (((double)mr - (double)m) * (double)a.inv_temp + log((double)srest) - lt));   // srest = 0: +inf
      a.loss_rows[row] = live ? (float)((double)w * loss) : 0.f;
      twice = 0;
    }
#pragma unroll 1
    for (int j = threadIdx.x; j < a.k; j += nt) {
      const int x = cls[j];
      if (x < 0) continue;
      atomicAnd(&bits[x >> 5], ~(1u << (x & 31)));
      if (a.d && live) d[x] = putf<TD>(g * (__builtin_amdgcn_exp2f((zs[j] - m) * c) / total * mass - (float)ex[j] * pmul));
    }
    __syncthreads();
  }
}

// loss[0] += sum of the rows' losses, in a fixed order
__global__ __launch_bounds__(256) void topk_loss_kernel(const float* __restrict__ terms, int rows, float* __restrict__ loss) {
  __shared__ float red[32];
  float s = 0.f;
  for (int r = threadIdx.x; r < rows; r += 256) s += terms[r];
  s = block_sum(s, red);
  if (threadIdx.x == 0) loss[0] += s;
}

template <typename TS, typename TD, int E, int NV, int NTMAX> void go(const TopkArgs& a, int grid, hipStream_t st) {
  const int chunks = lt_cdiv(a.K, E);
  int nt = 64;                        // the fewest waves whose registers hold the row
  while (nt < NTMAX && (int64_t)nt * NV < chunks) nt *= 2;
  const int bits = a.K > NV * nt * E ? a.K : NV * nt * E;
  const size_t lds = ((size_t)((bits + 31) / 32) + 5 * (size_t)a.k) * 4;
  hipLaunchKernelGGL((topk_kl_kernel<TS, TD, E, NV, NTMAX>), dim3(grid < a.rows ? grid : a.rows), dim3(nt), lds, st, a);
}
template <typename TS, typename TD> void dispatch(const TopkArgs& a, hipStream_t st) {
  constexpr int E = 16 / sizeof(TS);
  const bool vec = a.K % E == 0 && a.ld % E == 0 && ((uintptr_t)a.s & 15) == 0 && (!a.d || (a.ldd % E == 0 && ((uintptr_t)a.d & (E * sizeof(TD) - 1)) == 0));
  if (vec) {
    if (a.K / E <= 4 * 1024) go<TS, TD, E, 4, 1024>(a, MAX_GRID, st);
    else go<TS, TD, E, sizeof(TS) == 4 ? 32 : 16, 512>(a, CUS, st);
  } else {   // rows that are not whole 16-byte pieces: one element per lane and load
    if (a.K <= 16 * 1024) go<TS, TD, 1, 16, 1024>(a, MAX_GRID, st);
    else go<TS, TD, 1, 80, 512>(a, CUS, st);
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
