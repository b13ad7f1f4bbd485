// Rotary positions with several axes (time, height, width, ...) for gfx950: every token carries one position per axis, every rotary pair i of a
// head turns by pos[axis_i] * freq_i:  (a, b) -> (a cos - b sin, b cos + a sin), the inverse (= the gradient) with -sin.  Pairs are (i, i + dh / 2)
// or, interleaved, (2 i, 2 i + 1).
//
// Bound by memory (every element read and written once).  A workgroup takes T tokens; the dh / 2 angles of a token are formed ONCE, in 64 bits
// (position * frequency in fp32 is off by 0.06 rad at position 10^6), reduced to a quarter turn there, and their sines and cosines stay in
// registers while a thread walks the heads of q and k: T = 256 / (dh / 2) tokens, one angle per thread, 8 (4) head lanes.
// 154 MB of bf16 q and k of video tokens: 26 us warm (5.9 TB/s, part of it from the cache; 36 us a call with fresh tensors); 538 MB of fp32: 104 us = 5.2 TB/s,
// the rate of a copy.
#include "lt_common.h"

namespace {

constexpr int NT = 256;
struct Strides { int64_t b, n, h; };
struct RopeArgs {
  const void *x, *x2;
  void *out, *out2;
  const void* pos;
  const float* freqs;
  const int32_t* axis;
  Strides sx, so, sx2, so2;
  int64_t tokens, pos_b;   // B * N | positions between two batch entries (0: shared)
  int N, H, H2, dh, prefix, axes, pos_float, inverse;
};

template <typename T> struct Vec;
template <> struct Vec<float> {
  static __device__ __forceinline__ float get(float x) { return x; }
  static __device__ __forceinline__ float put(float x) { return x; }
};
struct bf_t { uint16_t u; };
struct hf_t { uint16_t u; };
template <> struct Vec<bf_t> {
  static __device__ __forceinline__ float get(bf_t x) { return bf2f(x.u); }
  static __device__ __forceinline__ bf_t put(float x) { return {f2bf(x)}; }
};
template <> struct Vec<hf_t> {
  static __device__ __forceinline__ float get(hf_t x) { return (float)__builtin_bit_cast(_Float16, x.u); }
  static __device__ __forceinline__ hf_t put(float x) { return {__builtin_bit_cast(uint16_t, (_Float16)x)}; }
};
template <typename T, int U> struct alignas(U * sizeof(T) < 16 ? U * sizeof(T) : 16) Pack { T v[U]; };

// U rotary pairs per thread and head (2 U elements: two runs of U, or one of 2 U when interleaved)
template <typename T, int U, bool IL>
__global__ __launch_bounds__(NT) void rope_axes_kernel(const RopeArgs a) {
  __shared__ __attribute__((aligned(16))) float cs[2][NT];
  const int half = a.dh >> 1, C = half / U, TB = NT / half;     // chunks of a head | tokens of a workgroup
  const int64_t tok0 = (int64_t)blockIdx.x * TB;
  {   // one angle per thread
    const int t = threadIdx.x / half, i = threadIdx.x - t * half;
    const int64_t tok = tok0 + t;
    if (t < TB && tok < a.tokens) {
      const int64_t b = tok / a.N;
      const int n = (int)(tok - b * a.N), ax = a.axis[i];
      float c = 1.f, s = 0.f;
      if (n >= a.prefix && ax >= 0 && ax < a.axes) {
        const int64_t at = (b * a.pos_b + (n - a.prefix)) * a.axes + ax;
        const double p = a.pos_float ? (double)static_cast<const float*>(a.pos)[at] : (double)static_cast<const int32_t*>(a.pos)[at];
        const double quarter = p * (double)a.freqs[i] * 0.63661977236758134308;   // 2 / pi: quarter turns
        const double q = rint(quarter);
        float sr, cr;
        sincospif(0.5f * (float)(quarter - q), &sr, &cr);
        const int k = (int)(q - 4.0 * floor(q * 0.25));
        c = k == 0 ? cr : k == 1 ? -sr : k == 2 ? -cr : sr;
        s = k == 0 ? sr : k == 1 ? cr : k == 2 ? -sr : -cr;
        if (!(fabs(quarter) < INFINITY)) c = s = NAN;
        if (a.inverse) s = -s;
      }
      cs[0][threadIdx.x] = c;
      cs[1][threadIdx.x] = s;
    }
  }
  __syncthreads();
  const int c = threadIdx.x % C, r = threadIdx.x / C, hl = r % U, t = r / U;   // U head lanes: C * U * TB <= 256 threads take part
  const int64_t tok = tok0 + t;
  if (t >= TB || tok >= a.tokens) return;
  float co[U], si[U];
#pragma unroll
  for (int j = 0; j < U; ++j) { co[j] = cs[0][t * half + c * U + j]; si[j] = cs[1][t * half + c * U + j]; }
  const int64_t b = tok / a.N;
  const int n = (int)(tok - b * a.N);
  const int o1 = IL ? 2 * U * c : U * c, o2 = IL ? o1 + U : U * c + half;
  for (int h = hl; h < a.H + a.H2; h += U) {
    const bool second = h >= a.H;
    const int hh = second ? h - a.H : h;
    const Strides& sx = second ? a.sx2 : a.sx;
    const Strides& so = second ? a.so2 : a.so;
    const T* p = static_cast<const T*>(second ? a.x2 : a.x) + b * sx.b + n * sx.n + hh * sx.h;
    T* w = static_cast<T*>(second ? a.out2 : a.out) + b * so.b + n * so.n + hh * so.h;
    Pack<T, U> u = *reinterpret_cast<const Pack<T, U>*>(p + o1), v = *reinterpret_cast<const Pack<T, U>*>(p + o2);
#pragma unroll
    for (int j = 0; j < U; ++j) {
      // pair j of the chunk: (u[j], v[j]) or, interleaved, elements 2 j and 2 j + 1 of the run u v
      T& ea = IL ? (2 * j < U ? u.v[(2 * j) % U] : v.v[(2 * j) % U]) : u.v[j];
      T& eb = IL ? (2 * j + 1 < U ? u.v[(2 * j + 1) % U] : v.v[(2 * j + 1) % U]) : v.v[j];
      const float x = Vec<T>::get(ea), y = Vec<T>::get(eb);
      const bool still = si[j] == 0.f;      // (a pair that does not turn passes as it is: 0 * inf would not)
      ea = Vec<T>::put(still ? x * co[j] : fmaf(x, co[j], -(y * si[j])));
      eb = Vec<T>::put(still ? y * co[j] : fmaf(y, co[j], x * si[j]));
    }
    *reinterpret_cast<Pack<T, U>*>(w + o1) = u;
    *reinterpret_cast<Pack<T, U>*>(w + o2) = v;
  }
}

template <typename T, int U> void launch(const RopeArgs& a, bool il, hipStream_t st) {
  const unsigned grid = (unsigned)lt_cdiv(a.tokens, NT / (a.dh >> 1));
  if (il) hipLaunchKernelGGL((rope_axes_kernel<T, U, true>), dim3(grid), dim3(NT), 0, st, a);
  else hipLaunchKernelGGL((rope_axes_kernel<T, U, false>), dim3(grid), dim3(NT), 0, st, a);
}
bool strides_ok(const int64_t* s, int B, int N, int H, int step) {
  return (B == 1 || (s[0] >= 0 && s[0] % step == 0)) && (N == 1 || (s[1] >= 0 && s[1] % step == 0)) && (H == 1 || (s[2] >= 0 && s[2] % step == 0));
}
Strides st3(const int64_t* s) { return {s[0], s[1], s[2]}; }

}  // namespace

extern "C" int lt_rope_axes(const lt_rope_axes_desc* d, void* stream) {
  LT_CHECK_ARG(d, "lt_rope_axes: no descriptor");
  LT_CHECK_ARG(d->B >= 0 && d->N >= 0 && d->H > 0 && d->H2 >= 0 && d->prefix >= 0 && d->prefix <= d->N, "lt_rope_axes: bad sizes (B %d, N %d, H %d, H2 %d, prefix %d)",
               d->B, d->N, d->H, d->H2, d->prefix);
  LT_CHECK_ARG(d->dh >= 8 && d->dh <= 256 && d->dh % 8 == 0, "lt_rope_axes: head_dim must be a multiple of 8 from 8 to 256 (got %d)", d->dh);
  LT_CHECK_ARG(d->axes >= 1 && d->axes <= 4, "lt_rope_axes: 1 to 4 axes (got %d)", d->axes);
  LT_CHECK_ARG(d->dtype == LT_DT_BF16 || d->dtype == LT_DT_F16 || d->dtype == LT_DT_F32, "lt_rope_axes: bad dtype");
  if (d->B == 0 || d->N == 0) return LT_OK;
  const int step = d->dtype == LT_DT_F32 ? 4 : 8;
  auto ok = [&](const void* p, const int64_t* s, int H) { return p && ((uintptr_t)p & 15) == 0 && strides_ok(s, d->B, d->N, H, step); };
  LT_CHECK_ARG(ok(d->x, d->sx, d->H) && ok(d->out, d->so, d->H) && (d->H2 == 0 || (ok(d->x2, d->sx2, d->H2) && ok(d->out2, d->so2, d->H2))),
               "lt_rope_axes: x, out: missing, or pointers or strides not 16-byte aligned");
  LT_CHECK_ARG(d->freqs && d->axis && (d->pos || d->prefix == d->N), "lt_rope_axes: pos, freqs and axis are needed");
  RopeArgs a;
  a.x = d->x; a.x2 = d->x2; a.out = d->out; a.out2 = d->out2;
  a.pos = d->pos; a.freqs = d->freqs; a.axis = d->axis;
  a.sx = st3(d->sx); a.so = st3(d->so); a.sx2 = st3(d->sx2); a.so2 = st3(d->so2);
  a.tokens = (int64_t)d->B * d->N; a.pos_b = d->pos_per_batch ? d->N - d->prefix : 0;
  a.N = d->N; a.H = d->H; a.H2 = d->H2; a.dh = d->dh; a.prefix = d->prefix; a.axes = d->axes; a.pos_float = d->pos_float; a.inverse = d->inverse;
  LT_CHECK_ARG(a.tokens / (NT / (d->dh >> 1)) < (1ll << 24) - 1, "lt_rope_axes: too many tokens");
  hipStream_t st = (hipStream_t)stream;
  if (d->dtype == LT_DT_F32) launch<float, 4>(a, d->interleaved, st);
  else if (d->dtype == LT_DT_BF16) { if (d->dh % 16 == 0) launch<bf_t, 8>(a, d->interleaved, st); else launch<bf_t, 4>(a, d->interleaved, st); }
  else { if (d->dh % 16 == 0) launch<hf_t, 8>(a, d->interleaved, st); else launch<hf_t, 4>(a, d->interleaved, st); }
  LT_CHECK_LAUNCH("lt_rope_axes");
}
