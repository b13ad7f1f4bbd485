// Cross attention for gfx950: queries q [B, Nq, H, dh] against the keys / values k, v [B, Nk, Hkv, dh] of another sequence (an encoder's states),
// forward and backward, bf16 or f16 operands, fp32 scores, statistics and accumulators; the score matrix never reaches memory.
//   S = scale * q k^T (keys that are not visible: -inf), P = softmax(S), O = P V, lse = ln sum exp S;  a row that sees no key: O = 0, lse = -inf
//   D = rowsum(dO * O), dV = P^T dO, dS = P * (dO V^T - D), dQ = scale * dS K, dK = scale * dS^T Q
// H / Hkv = G query heads share a key head: the G * Nq query rows of a (batch entry, key head) are one matrix, row r = (head r / Nq, query r % Nq),
// so the shared heads read their K / V once and their gradients are summed in registers.
//
// All products are v_mfma_f32_32x32x16 (A: lane l holds row l % 32, k-slots 8 (l / 32) .. + 7; C: lane -> column l % 32, register e -> row
// crow(e)).  A C tile whose contraction index lies in the registers is, packed to 16 bits, the next product's B operand without any data movement
// (the k-slot order {4h .. 4h + 3, 8 + 4h .. 8 + 4h + 3} it implies is applied to the other operand too), so the tiles are formed as
//   forward   S^T = K Q^T  (lane -> query)  ->  O^T  = V^T P^T      softmax statistics are per lane + one exchange between the wave's halves
//   dQ        S^T, dP^T = V dO^T            ->  dQ^T = K^T dS^T
//   dK / dV   S = Q K^T, dP = dO V^T (lane -> key)  ->  dV^T = dO^T P, dK^T = Q^T dS
// One LDS image of a token chunk serves both kinds of operand: rows of d, and (ds_read_b64_tr_b16) columns whose contraction index is the token.
// Keys that are not visible are staged as zeros (what the caller's padding holds is never multiplied) and their scores are -inf.
//
// Roundings to 16 bits: the tiled kernels round P and dS once on their way into the second product, which makes a result's error sqrt(2) of its own rounding
// (measured 1.1 - 1.4 for O, 1.4 for dV, 1.4 - 1.5 for dK and 1.4 - 1.57 for dQ, to which D from the rounded O adds); both halves of dS would cost dQ
// a third more matrix work.  The few-row kernels, which memory bounds, multiply both halves (measured 1.00, dQ <= 1.08).  f16 factors are brought into
// the type's range first (P_LOG2, P_UP, DS_UP): the same figures hold there, at every upstream scale.
#include "lt_common.h"

namespace {

typedef __attribute__((ext_vector_type(8))) short s16x8;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr float M_NONE = -1e30f;   // running maximum before the first visible key (finite: -inf - -inf never forms)
constexpr int NT = 256;            // threads per workgroup, four waves
constexpr int KC = 64;             // tokens per LDS chunk of the tiled kernels
constexpr float P_UP = 4096.f;     // f16 probabilities of the backward are kept times 2^12: 1 / Nk of a long cache would be subnormal
// The forward's probabilities are kept <= 2^GROW (soft_step).  f16: times 2^11 and GROW 4, so <= 2^15 and rounded at 2^-36 of a row's largest at worst: below that the long
// tail behind a dominant key was lost from P V (25 % of its weight at e^-18) while its sum of exponentials counted it.  All 2^24 keys that a call may have
// lose 2^-12 of the result there, half of its own rounding.  The sums carry the factor too: it cancels in O and is divided out of the sum in lse.
template <bool F16> constexpr float P_GROW = F16 ? 4.f : 8.f;
template <bool F16> constexpr float P_LOG2 = F16 ? 11.f : 0.f;

struct Strides { int64_t b, n, h; };
struct XArgs {
  const uint16_t *q, *k, *v, *o, *dout;
  uint16_t *out, *dq, *dk, *dv;
  float *lse, *ws, *delta;
  const int32_t* klen;
  const uint8_t* kmask;
  Strides sq, sk, sv, so, sdo, sdq, sdk, sdv;
  int B, Nq, Nk, H, Hkv, G, R, dh;
  float scale;
  int splits, tiles;   // work items along the contracted axis | row (key) tiles per (batch entry, key head)
};

template <bool F16> __device__ __forceinline__ f32x16 mma(s16x8 a, s16x8 b, f32x16 c) {
  if constexpr (F16) return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <bool F16> __device__ __forceinline__ uint32_t pack2(float a, float b) {   // both round to nearest even
  if constexpr (F16) { f16x2 v; v[0] = (_Float16)a; v[1] = (_Float16)b; return __builtin_bit_cast(uint32_t, v); }
  else return pack_bf2(a, b);
}
template <bool F16> __device__ __forceinline__ float to_f(short x) {
  if constexpr (F16) return (float)__builtin_bit_cast(_Float16, x);
  else return bf2f((uint16_t)x);
}
template <bool F16> __device__ __forceinline__ s16x8 pack8(const f32x16& p, int off) {
  const uint4 u = make_uint4(pack2<F16>(p[off], p[off + 1]), pack2<F16>(p[off + 2], p[off + 3]), pack2<F16>(p[off + 4], p[off + 5]),
                             pack2<F16>(p[off + 6], p[off + 7]));
  return __builtin_bit_cast(s16x8, u);
}
// a factor as two 16-bit parts, hi + lo: where memory bounds a kernel, a second product is free and the factor's rounding goes from 2^-9 to 2^-17 (f16: 2^-22, as
// far as lo is a normal number: from 2^-3 on)
template <bool F16> __device__ __forceinline__ void split8(const f32x16& p, int off, s16x8& hi, s16x8& lo) {
  hi = pack8<F16>(p, off);
  f32x16 r;
#pragma unroll
  for (int j = 0; j < 8; ++j) r[j] = p[off + j] - to_f<F16>(hi[j]);
#pragma unroll
  for (int j = 8; j < 16; ++j) r[j] = 0.f;
  lo = pack8<F16>(r, 0);
}
__device__ __forceinline__ f32x16 splat(float x) {
  f32x16 r;
#pragma unroll
  for (int e = 0; e < 16; ++e) r[e] = x;
  return r;
}
__device__ __forceinline__ int lane() { return threadIdx.x & 63; }
__device__ __forceinline__ int crow(int e, int hi) { return (e & 3) + 8 * (e >> 2) + 4 * hi; }
__device__ __forceinline__ float half_max(float x) {   // over the two lanes l, l ^ 32
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float half_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ s16x8 ld8(const uint16_t* p, bool ok) {
  uint4 u = make_uint4(0, 0, 0, 0);
  if (ok) u = *reinterpret_cast<const uint4*>(p);
  return __builtin_bit_cast(s16x8, u);
}
__device__ __forceinline__ void wait_lds() { __builtin_amdgcn_s_waitcnt(0xc07f); __builtin_amdgcn_wave_barrier(); }   // lgkmcnt(0)

// ---- the LDS image -----------------------------------------------------------------------------------------------------------------
// T tokens x 32 HD columns of 16 bits as [4 tokens][16 d] pieces of 128 B, read both ways: rows of 8 consecutive d (ds_read_b128) and, for products
// over the token index, transposed (ds_read_b64_tr_b16 takes one piece per 16 lanes).  Piece (q = token / 4, b = d / 16) lies at
// q * 2 HD + (b ^ (q & 1)); its token rows are rotated by b and their two 16-byte halves swapped where q & 2: the 16 rows that one phase of a
// ds_read_b128 touches land on 16 different bank groups, and so do the 16-byte stores of a staged row.
template <int HD> __device__ __forceinline__ int img_off(int r, int c) {   // 16-byte chunk c of token r
  const int q = r >> 2, b = c >> 1;
  return (q * (2 * HD) + (b ^ (q & 1))) * 128 + ((((r & 3) + b) & 3) << 5) + (((c ^ (q >> 1)) & 1) << 4);
}
template <int HD> __device__ __forceinline__ s16x8 row_frag(const char* img, int tile, int ks) {   // 32 tokens x 16 d
  const int l = lane(), r = l & 31, q = r >> 2;
  const int at = q * (2 * HD * 128) + (((ks & 3) ^ (q & 1)) << 7) + ((((r & 3) + ks) & 3) << 5) + ((((l >> 5) ^ (q >> 1)) & 1) << 4);
  return *reinterpret_cast<const s16x8*>(img + at + tile * (8 * 2 * HD * 128) + (ks >> 2) * 512);
}
// rows = 32 d (block db), k-slots = 16 tokens from tok16 (a multiple of 16) in the C-layout slot order
template <int HD> __device__ __forceinline__ s16x8 tr_frag(const char* img, int db, int tok16) {
  const int l = lane(), i = l & 15, cb = (l >> 4) & 1, hi = l >> 5;
  const int at = hi * (2 * HD * 128) + ((cb ^ hi) << 7) + ((((i >> 2) + cb + 2 * (db & 1)) & 3) << 5);
  const char* p = img + (tok16 >> 2) * (2 * HD * 128) + db * 256;
  const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + at + ((i & 3) << 3)));
  const s16x4 up = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 2 * (2 * HD * 128) + at + (((i & 3) ^ 2) << 3)));
  return __builtin_shufflevector(lo, up, 0, 1, 2, 3, 4, 5, 6, 7);
}
template <int HD> constexpr int img_bytes() { return KC * HD * 64; }
// KC tokens between memory and the images, through registers (the next chunk's loads stay in flight while a chunk is computed).  The loads go through
// a buffer descriptor that begins at the chunk's first token: a thread's offsets are the same for every chunk, no address arithmetic is left to
// the vector units (it was half of their instructions), and tokens past the end, or columns past head_dim, read as zeros.
constexpr int64_t MAX_STEP = 1 << 24;   // elements between two tokens: 64 tokens stay inside 31 bits
struct Window {
  __amdgpu_buffer_rsrc_t r;
  // `tokens` rows from `base`, sn elements apart, of which dh are read
  __device__ __forceinline__ Window(const uint16_t* base, int64_t sn, int tokens, int dh) {
    const uint32_t bytes = tokens > 0 ? (uint32_t)(((int64_t)min(tokens, KC) - 1) * sn + dh) * 2u : 0u;
    const uint64_t p = (uint64_t)base;
    const uint64_t q = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)p) |
                       ((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(p >> 32)) << 32);
    r = __builtin_amdgcn_make_buffer_rsrc((void*)q, 0, __builtin_amdgcn_readfirstlane((int)bytes), 0x00020000);
  }
  __device__ __forceinline__ uint4 load(uint32_t off) const { return __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(r, (int)off, 0, 0)); }
};
template <int HD> struct Chunk {
  static constexpr int CPR = 4 * HD, PER = KC * CPR / NT;
  uint4 u[PER];
  uint32_t off[PER];
  __device__ __forceinline__ void offsets(int64_t sn, int dh) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int idx = threadIdx.x + NT * i, c = idx % CPR;
      off[i] = c * 8 < dh ? (uint32_t)(idx / CPR) * (uint32_t)sn * 2u + c * 16u : 0xfffffff0u;
    }
  }
  __device__ __forceinline__ void load(const uint16_t* base, int64_t sn, int tok0, int end, int dh) {
    const Window w(base + (int64_t)tok0 * sn, sn, end - tok0, dh);
#pragma unroll
    for (int i = 0; i < PER; ++i) u[i] = w.load(off[i]);
  }
  // query rows r0 .. r0 + KC - 1; n0, g0: token and head of row r0
  __device__ __forceinline__ void load_rows(const uint16_t* base, const Strides& s, int r0, int g0, int n0, int R, int Nq, int dh) {
    if (n0 + KC <= Nq || r0 - n0 + Nq >= R) {   // the chunk lies in one head, or in the last
      load(base + (int64_t)g0 * s.h, s.n, n0, Nq, dh);
    } else {
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int idx = threadIdx.x + NT * i, r = r0 + idx / CPR, c = idx % CPR;
        u[i] = make_uint4(0, 0, 0, 0);
        if (r < R && c * 8 < dh) {
          const int g = r / Nq, n = r - g * Nq;
          u[i] = *reinterpret_cast<const uint4*>(base + n * s.n + g * s.h + c * 8);
        }
      }
    }
  }
  __device__ __forceinline__ void hide(const uint8_t (&m)[PER]) {
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (!m[i]) u[i] = make_uint4(0, 0, 0, 0);
  }
  __device__ __forceinline__ void store(char* img) const {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int idx = threadIdx.x + NT * i;
      *reinterpret_cast<uint4*>(img + img_off<HD>(idx / CPR, idx % CPR)) = u[i];
    }
  }
};
// K and V of a chunk with the mask bytes of the rows that this thread carries, and the score start value (0 / -inf) of key threadIdx.x.  Hidden keys
// are loaded like the others -- a load that waited for its mask byte would expose two latencies per chunk -- and become zeros on the way to LDS.
template <int HD> struct KeyChunk {
  Chunk<HD> k, v;
  uint8_t m[Chunk<HD>::PER], mb;
  bool in;
  __device__ __forceinline__ void offsets(const XArgs& a) {
    k.offsets(a.sk.n, a.dh);
    v.offsets(a.sv.n, a.dh);
  }
  __device__ __forceinline__ void load(const XArgs& a, const uint16_t* kb, const uint16_t* vb, const uint8_t* mask, int c, int kend) {
    k.load(kb, a.sk.n, c * KC, kend, a.dh);
    v.load(vb, a.sv.n, c * KC, kend, a.dh);
    in = c * KC + (int)threadIdx.x < kend;
    if (mask) {
#pragma unroll
      for (int i = 0; i < Chunk<HD>::PER; ++i) {
        const int tok = c * KC + (threadIdx.x + NT * i) / Chunk<HD>::CPR;
        m[i] = tok < kend ? mask[tok] : 0;
      }
      mb = threadIdx.x < KC && in ? mask[c * KC + threadIdx.x] : 0;
    }
  }
  __device__ __forceinline__ float hide(const uint8_t* mask) {   // returns the start value
    if (!mask) return in ? 0.f : -INFINITY;
    k.hide(m);
    v.hide(m);
    return mb ? 0.f : -INFINITY;
  }
};

// the workgroups of one (batch entry, key head) land on one XCD (workgroup i runs on XCD i % 8): they share its K / V in that L2
__device__ __forceinline__ bool my_item(const XArgs& a, int per, int& bh, int& item) {
  const int x = blockIdx.x & 7, i = blockIdx.x >> 3;
  bh = (i / per) * 8 + x;
  item = i % per;
  return bh < a.B * a.Hkv;
}
__device__ __forceinline__ int key_end(const XArgs& a, int b) { return __builtin_amdgcn_readfirstlane(a.klen ? min(max(a.klen[b], 0), a.Nk) : a.Nk); }

// Accumulators acc[HD] in C layout (lane -> row, registers -> d) as 16-bit rows: through 32 rows of an LDS image that belongs to the wave, so that
// 4 HD neighbouring lanes write one row in 16-byte pieces (written from the registers, a store instruction would touch 32 rows 16 bytes each).
// at(r): where row r of the tile goes, nullptr = nowhere.
template <bool F16, int HD, typename At> __device__ __forceinline__ void put_tile(char* img, const f32x16 (&acc)[HD], float mul, int dh, At&& at) {
  const int l = lane(), hi = l >> 5;
#pragma unroll
  for (int db = 0; db < HD; ++db)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<uint2*>(img + img_off<HD>(l & 31, db * 4 + g) + 8 * hi) =
          make_uint2(pack2<F16>(acc[db][4 * g] * mul, acc[db][4 * g + 1] * mul), pack2<F16>(acc[db][4 * g + 2] * mul, acc[db][4 * g + 3] * mul));
  wait_lds();
#pragma unroll
  for (int i = 0; i < 2 * HD; ++i) {
    const int idx = l + 64 * i, r = idx / (4 * HD), c = idx % (4 * HD);
    const uint4 u = *reinterpret_cast<const uint4*>(img + img_off<HD>(r, c));
    uint16_t* p = at(r);
    if (p && c * 8 < dh) *reinterpret_cast<uint4*>(p + c * 8) = u;
  }
  wait_lds();
}
// ... and as fp32 partial rows, straight from the registers
template <int HD> __device__ __forceinline__ void put_partial(float* dst, const f32x16 (&acc)[HD], float mul, int dh) {
  const int hi = lane() >> 5;
#pragma unroll
  for (int db = 0; db < HD; ++db)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = db * 32 + 8 * g + 4 * hi;
      if (d < dh) *reinterpret_cast<float4*>(dst + d) = make_float4(acc[db][4 * g] * mul, acc[db][4 * g + 1] * mul, acc[db][4 * g + 2] * mul, acc[db][4 * g + 3] * mul);
    }
}

// ================================================================================================================== forward
// One online-softmax step of one 32-query tile over NK 32-key tiles of raw scores s (base 2, reference m in raw-score units that moves only when a
// row's maximum passes it by more than P_GROW octaves: probabilities stay <= 2^8, exact in fp32 and bf16 safe; f16: <= 2^4, times 2^11).  lsum is per lane (the
// two halves of a row are added once, at the end).
template <bool F16, int HD, int NK> __device__ __forceinline__ void soft_step(f32x16 (&s)[NK], float c, float& m, float& lsum, f32x16 (&o)[HD]) {
  float mx = s[0][0];
#pragma unroll
  for (int t = 0; t < NK; ++t)
#pragma unroll
    for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[t][e]);
  mx = half_max(mx);
  const bool grow = (mx - m) * c > P_GROW<F16>;
  if (__builtin_amdgcn_ballot_w64(grow) != 0) {
    const float mn = grow ? mx : m, alpha = __builtin_amdgcn_exp2f((m - mn) * c);
    lsum *= alpha;
    m = mn;
#pragma unroll
    for (int db = 0; db < HD; ++db)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[db][e] *= alpha;
  }
  const float nmc = fminf(fmaf(-m, c, P_LOG2<F16>), 3e38f);   // (finite, also for M_NONE at a large scale: a hidden key's -inf stays -inf)
  float r0 = 0.f, r1 = 0.f;
#pragma unroll
  for (int t = 0; t < NK; ++t)
#pragma unroll
    for (int e = 0; e < 16; ++e) s[t][e] = fmaf(s[t][e], c, nmc);
#pragma unroll
  for (int t = 0; t < NK; ++t)
#pragma unroll
    for (int e = 0; e < 16; e += 2) {
      s[t][e] = __builtin_amdgcn_exp2f(s[t][e]);
      s[t][e + 1] = __builtin_amdgcn_exp2f(s[t][e + 1]);
      r0 += s[t][e];
      r1 += s[t][e + 1];
    }
  lsum += r0 + r1;
}

// ln of a row's sum of exponentials
template <bool F16> __device__ __forceinline__ float row_lse(float m, float lsum, float scale) {
  return lsum != 0.f ? m * scale + __logf(F16 ? lsum * 0x1p-11f : lsum) : -INFINITY;
}

// Tiled forward: a workgroup owns 4 waves x QT x 32 query rows of one (batch entry, key head) and walks its share of the keys in chunks of 64.
// No unit is saturated: counted, the matrix unit is busy 22 % (head_dim 128: 40 %) of the cycles, the vector unit by estimate 45 - 50 %, 22 - 37 % of
// the waves' time is waiting; wave priorities around the products and the compiler's interleaving options moved nothing.  1569 x 2 rows against 6273 keys x 16 heads of 64, masked, 160 - 168 us
// = 480 - 510 TFLOP/s over the visible and hidden keys; 3136 rows x 25 088 keys x 8 of 128, 380 - 426 us = 760 - 850 TFLOP/s (a large matrix product reaches 1195).
template <bool F16, int HD, int QT>
__global__ __launch_bounds__(NT, HD <= 2 && QT == 1 ? 3 : 2) void xattn_fwd_kernel(const XArgs a) {
  __shared__ __attribute__((aligned(16))) char smem[2 * (2 * img_bytes<HD>() + KC * 4)];
  constexpr int BUF = 2 * img_bytes<HD>() + KC * 4;
  int bh, item;
  if (!my_item(a, a.tiles * a.splits, bh, item)) return;
  const int b = bh / a.Hkv, hk = bh % a.Hkv, tile = item % a.tiles, split = item / a.tiles;
  const int wave = threadIdx.x >> 6, l = lane(), hi = l >> 5;
  const int kend = key_end(a, b), chunks = (kend + KC - 1) / KC, per = (chunks + a.splits - 1) / a.splits;
  const int c_lo = min(split * per, chunks), c_hi = min(c_lo + per, chunks);
  const uint16_t* kb = a.k + b * a.sk.b + hk * a.sk.h;
  const uint16_t* vb = a.v + b * a.sv.b + hk * a.sv.h;
  const uint8_t* mask = a.kmask ? a.kmask + (int64_t)b * a.Nk : nullptr;

  KeyChunk<HD> in;
  in.offsets(a);
  auto load = [&](int c) { in.load(a, kb, vb, mask, c, kend); };
  auto store = [&](int buf) {
    const float bias = in.hide(mask);
    in.k.store(smem + buf * BUF);
    in.v.store(smem + buf * BUF + img_bytes<HD>());
    if (threadIdx.x < KC) *reinterpret_cast<float*>(smem + buf * BUF + 2 * img_bytes<HD>() + threadIdx.x * 4) = bias;
  };
  if (c_lo < c_hi) load(c_lo);
  s16x8 qf[QT][2 * HD];
  f32x16 o[QT][HD];
  float m[QT], lsum[QT];
  const int row0 = (tile * 4 + wave) * 32 * QT;
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const int r = row0 + t * 32 + (l & 31), g = r / a.Nq, n = r - g * a.Nq;
    const uint16_t* p = a.q + b * a.sq.b + n * a.sq.n + (int64_t)(hk * a.G + g) * a.sq.h;
#pragma unroll
    for (int ks = 0; ks < 2 * HD; ++ks) qf[t][ks] = ld8(p + ks * 16 + hi * 8, r < a.R && ks * 16 + hi * 8 < a.dh);
#pragma unroll
    for (int db = 0; db < HD; ++db) o[t][db] = splat(0.f);
    m[t] = M_NONE;
    lsum[t] = 0.f;
  }
  const float c = a.scale * LOG2E;
  if (c_lo < c_hi) store(0);
  __syncthreads();
  for (int ch = c_lo; ch < c_hi; ++ch) {
    const int buf = (ch - c_lo) & 1;
    const bool more = ch + 1 < c_hi;
    if (more) load(ch + 1);
    const char* K = smem + buf * BUF;
    const char* V = K + img_bytes<HD>();
    const float* bs = reinterpret_cast<const float*>(V + img_bytes<HD>());
    if (row0 < a.R) {
      const bool biased = mask || (ch + 1) * KC > kend;
      f32x16 s[QT][2];
      // (independent accumulators in turn: a product that waits for the one before it leaves the matrix unit idle; the first one starts at the
      // inline constant 0 -- start values from LDS would cost every chunk the moves that only a chunk with hidden keys needs)
#pragma unroll
      for (int ks = 0; ks < 2 * HD; ++ks)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const s16x8 kf = row_frag<HD>(K, t, ks);
#pragma unroll
          for (int qt = 0; qt < QT; ++qt) s[qt][t] = mma<F16>(kf, qf[qt][ks], ks ? s[qt][t] : splat(0.f));
        }
      if (biased) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const float4 x = *reinterpret_cast<const float4*>(bs + t * 32 + 8 * g + 4 * hi);
#pragma unroll
            for (int qt = 0; qt < QT; ++qt) {   // (replaced, not added to: a query that holds NaN must not reach a row without keys)
              s[qt][t][4 * g] = x.x < 0.f ? x.x : s[qt][t][4 * g];
              s[qt][t][4 * g + 1] = x.y < 0.f ? x.y : s[qt][t][4 * g + 1];
              s[qt][t][4 * g + 2] = x.z < 0.f ? x.z : s[qt][t][4 * g + 2];
              s[qt][t][4 * g + 3] = x.w < 0.f ? x.w : s[qt][t][4 * g + 3];
            }
          }
      }
      s16x8 p[QT][4];
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) {
        soft_step<F16, HD, 2>(s[qt], c, m[qt], lsum[qt], o[qt]);
#pragma unroll
        for (int t = 0; t < 2; ++t) { p[qt][2 * t] = pack8<F16>(s[qt][t], 0); p[qt][2 * t + 1] = pack8<F16>(s[qt][t], 8); }
      }
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int db = 0; db < HD; ++db) {
          const s16x8 vf = tr_frag<HD>(V, db, k * 16);
#pragma unroll
          for (int qt = 0; qt < QT; ++qt) o[qt][db] = mma<F16>(vf, p[qt][k], o[qt][db]);
        }
    }
    if (more) store(buf ^ 1);
    __syncthreads();
  }
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const int r = row0 + t * 32 + (l & 31);
    const float ls = half_sum(lsum[t]);
    if (a.splits > 1) {
      if (r >= a.R) continue;
      const int64_t rows = (int64_t)a.B * a.Hkv * a.R, row = split * rows + (int64_t)bh * a.R + r;
      put_partial<HD>(a.ws + row * a.dh, o[t], 1.f, a.dh);
      if (hi == 0) *reinterpret_cast<float2*>(a.ws + a.splits * rows * a.dh + row * 2) = make_float2(m[t], ls);
    } else {
      put_tile<F16, HD>(smem + wave * (32 * HD * 64), o[t], ls != 0.f ? 1.f / ls : 0.f, a.dh, [&](int x) -> uint16_t* {
        const int rr = row0 + t * 32 + x, g = rr / a.Nq, n = rr - g * a.Nq;
        return rr < a.R ? a.out + b * a.so.b + n * a.so.n + (int64_t)(hk * a.G + g) * a.so.h : nullptr;
      });
      if (hi == 0 && a.lse && r < a.R) a.lse[((int64_t)b * a.H + hk * a.G) * a.Nq + r] = row_lse<F16>(m[t], ls, a.scale);   // (rows of a group lie one after the other)
    }
  }
}

// Few rows (R <= 32: pooling by one query, one new token): the waves share the one row tile and split the KEYS.  K fragments are rows and come
// straight from memory, V passes through a wave-private image; the next tile's loads are in flight while a tile is computed.  Bound by reading
// K / V: the padded matrix work of a 32-key tile (12 HD MFMAs) hides under its 8 KiB * HD / 2 of loads.
// 768 heads x 1370 keys of 64: 50 - 54 us (270 MB; 54 us at the 5.03 TB/s of a copy; repeated on the same tensors, some of which the cache still holds); 384 x 785: 17 us.
template <int HD> struct KeyTile {
  s16x8 f[2 * HD];
  __device__ __forceinline__ void load(const uint16_t* base, int64_t sn, int key, bool ok, int dh) {
    const int hi = lane() >> 5;
#pragma unroll
    for (int ks = 0; ks < 2 * HD; ++ks) f[ks] = ld8(base + key * sn + ks * 16 + hi * 8, ok && ks * 16 + hi * 8 < dh);
  }
  __device__ __forceinline__ void hide(bool ok) {
#pragma unroll
    for (int ks = 0; ks < 2 * HD; ++ks)
      if (!ok) f[ks] = s16x8{0, 0, 0, 0, 0, 0, 0, 0};
  }
  __device__ __forceinline__ void store(char* img) const {   // token l % 32, chunk 2 ks + hi
    const int l = lane();
#pragma unroll
    for (int ks = 0; ks < 2 * HD; ++ks) *reinterpret_cast<s16x8*>(img + img_off<HD>(l & 31, 2 * ks + (l >> 5))) = f[ks];
  }
};

template <bool F16, int HD>
__global__ __launch_bounds__(NT, HD <= 2 ? 3 : 2) void xattn_fwd_few_kernel(const XArgs a) {
  constexpr int OST = HD * 32 + 4;   // floats between the rows of a wave's partial output
  __shared__ __attribute__((aligned(16))) char smem[4 * 32 * OST * 4 + 4 * 32 * 8];
  int bh, split;
  if (!my_item(a, a.splits, bh, split)) return;
  const int b = bh / a.Hkv, hk = bh % a.Hkv;
  const int wave = threadIdx.x >> 6, l = lane(), hi = l >> 5;
  const int kend = key_end(a, b), tiles = (kend + 31) / 32, per = (tiles + a.splits - 1) / a.splits;
  const int t_lo = min(split * per, tiles), t_hi = min(t_lo + per, tiles);
  const uint16_t* kb = a.k + b * a.sk.b + hk * a.sk.h;
  const uint16_t* vb = a.v + b * a.sv.b + hk * a.sv.h;
  const uint8_t* mask = a.kmask ? a.kmask + (int64_t)b * a.Nk : nullptr;
  char* img = smem + wave * (32 * HD * 64);

  KeyTile<HD> kf, vf;
  bool in = false;
  uint8_t mb = 1;
  auto load = [&](int t) {
    const int key = t * 32 + (l & 31);
    in = t < t_hi && key < kend;
    kf.load(kb, a.sk.n, key, in, a.dh);
    vf.load(vb, a.sv.n, key, in, a.dh);
    if (mask) mb = in ? mask[key] : 0;
  };
  load(t_lo + wave);
  const int r = l & 31, g = r / a.Nq, n = r - g * a.Nq;
  s16x8 qf[2 * HD];
  const uint16_t* qp = a.q + b * a.sq.b + n * a.sq.n + (int64_t)(hk * a.G + g) * a.sq.h;
#pragma unroll
  for (int ks = 0; ks < 2 * HD; ++ks) qf[ks] = ld8(qp + ks * 16 + hi * 8, r < a.R && ks * 16 + hi * 8 < a.dh);
  f32x16 o[HD];
#pragma unroll
  for (int db = 0; db < HD; ++db) o[db] = splat(0.f);
  float m = M_NONE, lsum = 0.f;
  const float c = a.scale * LOG2E;
  for (int t = t_lo + wave; t < t_hi; t += 4) {
    const bool ok = in && mb;
    const uint32_t seen = (uint32_t)__builtin_amdgcn_ballot_w64(ok);
    f32x16 s[1] = {splat(0.f)};
    if (seen != 0xffffffffu) {
      kf.hide(ok);
      vf.hide(ok);
    }
#pragma unroll
    for (int ks = 0; ks < 2 * HD; ++ks) s[0] = mma<F16>(kf.f[ks], qf[ks], s[0]);
    if (seen != 0xffffffffu) {
#pragma unroll
      for (int e = 0; e < 16; ++e) s[0][e] = (seen >> crow(e, hi)) & 1 ? s[0][e] : -INFINITY;
    }
    vf.store(img);
    load(t + 4);
    soft_step<F16, HD, 1>(s, c, m, lsum, o);
    s16x8 p0, p1, q0, q1;
    split8<F16>(s[0], 0, p0, q0);
    split8<F16>(s[0], 8, p1, q1);
    wait_lds();
#pragma unroll
    for (int db = 0; db < HD; ++db) {
      const s16x8 v0 = tr_frag<HD>(img, db, 0), v1 = tr_frag<HD>(img, db, 16);
      o[db] = mma<F16>(v0, p0, o[db]);
      o[db] = mma<F16>(v0, q0, o[db]);
      o[db] = mma<F16>(v1, p1, o[db]);
      o[db] = mma<F16>(v1, q1, o[db]);
    }
    wait_lds();
  }
  lsum = half_sum(lsum);
  __syncthreads();   // the images become the waves' partial outputs
  float* part = reinterpret_cast<float*>(smem) + wave * 32 * OST;
  float2* ml = reinterpret_cast<float2*>(smem + 4 * 32 * OST * 4);
  if (r < a.R) {
    put_partial<HD>(part + r * OST, o, 1.f, HD * 32);
    if (hi == 0) ml[wave * 32 + r] = make_float2(m, lsum);
  }
  __syncthreads();
  const float* all = reinterpret_cast<const float*>(smem);
  const int d4n = a.dh >> 2;
  for (int i = threadIdx.x; i < a.R * d4n; i += NT) {
    const int row = i / d4n, d = (i - row * d4n) * 4;
    float mm = M_NONE, ls = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) mm = fmaxf(mm, ml[w * 32 + row].x);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = __builtin_amdgcn_exp2f((ml[w * 32 + row].x - mm) * c);
      const float4 x = *reinterpret_cast<const float4*>(all + (w * 32 + row) * OST + d);
      ls += ml[w * 32 + row].y * f;
      acc.x += x.x * f; acc.y += x.y * f; acc.z += x.z * f; acc.w += x.w * f;
    }
    if (a.splits > 1) {
      const int64_t rows = (int64_t)a.B * a.Hkv * a.R, at = split * rows + (int64_t)bh * a.R + row;
      *reinterpret_cast<float4*>(a.ws + at * a.dh + d) = acc;
      if (d == 0) *reinterpret_cast<float2*>(a.ws + a.splits * rows * a.dh + at * 2) = make_float2(mm, ls);
    } else {
      const int gg = row / a.Nq, nn = row - gg * a.Nq, h = hk * a.G + gg;
      const float inv = ls != 0.f ? 1.f / ls : 0.f;
      *reinterpret_cast<uint2*>(a.out + b * a.so.b + nn * a.so.n + h * a.so.h + d) =
          make_uint2(pack2<F16>(acc.x * inv, acc.y * inv), pack2<F16>(acc.z * inv, acc.w * inv));
      if (d == 0 && a.lse) a.lse[((int64_t)b * a.H + h) * a.Nq + nn] = row_lse<F16>(mm, ls, a.scale);
    }
  }
}

// joins the key splits of the forward: per row the largest reference, the rescaled sums in split order
template <bool F16>
__global__ __launch_bounds__(NT) void xattn_join_kernel(const XArgs a) {
  const int d4n = a.dh >> 2;
  const int64_t rows = (int64_t)a.B * a.Hkv * a.R, i = (int64_t)blockIdx.x * NT + threadIdx.x;
  if (i >= rows * d4n) return;
  const int64_t row = i / d4n;
  const int d = (int)(i - row * d4n) * 4, r = (int)(row % a.R);
  const int64_t bh = row / a.R;
  const int b = (int)(bh / a.Hkv), hk = (int)(bh % a.Hkv), g = r / a.Nq, n = r - g * a.Nq, h = hk * a.G + g;
  const float2* ml = reinterpret_cast<const float2*>(a.ws + a.splits * rows * a.dh);
  const float c = a.scale * LOG2E;
  float mm = M_NONE, ls = 0.f;
  for (int s = 0; s < a.splits; ++s) mm = fmaxf(mm, ml[s * rows + row].x);
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s = 0; s < a.splits; ++s) {
    const float2 y = ml[s * rows + row];
    const float f = __builtin_amdgcn_exp2f((y.x - mm) * c);
    const float4 x = *reinterpret_cast<const float4*>(a.ws + (s * rows + row) * a.dh + d);
    ls += y.y * f;
    acc.x += x.x * f; acc.y += x.y * f; acc.z += x.z * f; acc.w += x.w * f;
  }
  const float inv = ls != 0.f ? 1.f / ls : 0.f;
  *reinterpret_cast<uint2*>(a.out + b * a.so.b + n * a.so.n + h * a.so.h + d) = make_uint2(pack2<F16>(acc.x * inv, acc.y * inv), pack2<F16>(acc.z * inv, acc.w * inv));
  if (d == 0 && a.lse) a.lse[((int64_t)b * a.H + h) * a.Nq + n] = row_lse<F16>(mm, ls, a.scale);
}

// ================================================================================================================== backward
// The row statistics enter the products as accumulator start values: S' = S / scale - lse / scale, dP' = dP - D, so P = exp2(c S') and dS = P dP'.
// A row without keys has lse = -inf: it starts at -inf like a row past the end, and every P is 0.
__device__ __forceinline__ float row_start(float lse, float scale) { return lse == -INFINITY ? -INFINITY : -lse / scale; }

// f16 dS = P (dP - D) carries P's 1 / Nk and the size of the upstream gradient: unscaled it lost bits from 2^-14 on, long before the gradients are that small (1.6 % of dQ
// at 784 x 25 088 and an upstream scale of 1e-3), and was infinite past 65504 where they are not.  It is rounded times 2^up instead, up its column's (dQ: a query
// row's, dK: a key's) own: from 40, where dS from 2^-54 on is a normal number, up goes down whenever the column's largest passes 2^15 -- to 2^11 .. 2^12, so that it
// seldom does again -- and the accumulators with it, as under a running maximum.  A column's dS is rounded at 2^-36 of its largest at worst.  2^up comes out
// with the store.
constexpr int DS_UP = 40;
__device__ __forceinline__ float pow2(int e) { return __builtin_amdgcn_ldexpf(1.f, e); }
__device__ __forceinline__ int octaves_down(float mx) { return mx > 32768.f ? max(__builtin_amdgcn_frexp_expf(mx) - 12, 0) : 0; }   // (infinities: 0)
__device__ __forceinline__ float column_max(const f32x16& x) {   // |x| over the two lanes that hold a column
  float mx = 0.f;
#pragma unroll
  for (int e = 0; e < 16; ++e) mx = fmaxf(mx, fabsf(x[e]));
  return half_max(mx);
}
// s, dp: S - lse / scale, dP - D -> P times 2^12 = P_UP and dS times 2^up
__device__ __forceinline__ void scaled_factors(f32x16& s, f32x16& dp, float c, int up) {
  const float f = pow2(up - 12);
#pragma unroll
  for (int e = 0; e < 16; ++e) s[e] = fmaf(s[e], c, 12.f);
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    s[e] = __builtin_amdgcn_exp2f(s[e]);
    dp[e] *= s[e] * f;
  }
}
template <int HD> __device__ __forceinline__ void bring_down(f32x16& ds, int& up, f32x16 (&acc)[HD]) {
  const float mx = column_max(ds);
  if (__builtin_amdgcn_ballot_w64(mx > 32768.f) == 0) return;
  const int n = octaves_down(mx);
  const float f = pow2(-n);
  up -= n;
#pragma unroll
  for (int e = 0; e < 16; ++e) ds[e] *= f;
#pragma unroll
  for (int db = 0; db < HD; ++db)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[db][e] *= f;
}

// dQ: a workgroup owns 128 query rows and walks its share of the keys (196 rows x 1370 keys x 384 heads of 64: 67 us = 590 TFLOP/s; 64 columns and one row tile a
// wave leave three waves to a SIMD -- four spill: 76 -> 165 us, and two row tiles a wave leave two: 74 -> 89 us); D = rowsum(dO * O) of its rows is formed here and left for the dK / dV kernel.
// SUMS (at most two chunks of keys): a pass of its own forms D = sum_k P dP from the fp32 products -- rowsum(dO * O) carries the rounding of O, most of
// dS's error when a row's probabilities are spread over a few keys only.
template <bool F16, int HD, bool SUMS>
__global__ __launch_bounds__(NT, HD <= 2 && !SUMS ? 3 : HD <= 3 ? 2 : 1) void xattn_dq_kernel(const XArgs a) {
  constexpr int BUF = 2 * img_bytes<HD>() + KC * 4;
  __shared__ __attribute__((aligned(16))) char smem[2 * BUF];
  int bh, item;
  if (!my_item(a, a.tiles * a.splits, bh, item)) return;
  const int b = bh / a.Hkv, hk = bh % a.Hkv, tile = item % a.tiles, split = item / a.tiles;
  const int wave = threadIdx.x >> 6, l = lane(), hi = l >> 5;
  const int kend = key_end(a, b), chunks = (kend + KC - 1) / KC, per = (chunks + a.splits - 1) / a.splits;
  const int c_lo = min(split * per, chunks), c_hi = min(c_lo + per, chunks);
  const uint16_t* kb = a.k + b * a.sk.b + hk * a.sk.h;
  const uint16_t* vb = a.v + b * a.sv.b + hk * a.sv.h;
  const uint8_t* mask = a.kmask ? a.kmask + (int64_t)b * a.Nk : nullptr;
  KeyChunk<HD> in;
  in.offsets(a);
  auto load = [&](int c) { in.load(a, kb, vb, mask, c, kend); };
  auto store = [&](int buf) {
    char* p = smem + buf * BUF;
    const float bias = in.hide(mask);
    in.k.store(p);
    in.v.store(p + img_bytes<HD>());
    if (threadIdx.x < KC) *reinterpret_cast<float*>(p + 2 * img_bytes<HD>() + threadIdx.x * 4) = bias;
  };
  if (c_lo < c_hi) load(c_lo);
  const int row0 = (tile * 4 + wave) * 32, r = row0 + (l & 31), g = r / a.Nq, n = r - g * a.Nq;
  const int64_t h = hk * a.G + g;
  const float lse = r < a.R ? a.lse[((int64_t)b * a.H + h) * a.Nq + n] : -INFINITY;
  const bool live = lse != -INFINITY;   // a row without keys takes no part: its dO may hold anything
  s16x8 qf[2 * HD], df[2 * HD];
  float D = 0.f;
#pragma unroll
  for (int ks = 0; ks < 2 * HD; ++ks) {
    const int d = ks * 16 + hi * 8;
    const bool ok = live && d < a.dh;
    qf[ks] = ld8(a.q + b * a.sq.b + n * a.sq.n + h * a.sq.h + d, ok);
    df[ks] = ld8(a.dout + b * a.sdo.b + n * a.sdo.n + h * a.sdo.h + d, ok);
    const s16x8 of = ld8(a.o + b * a.so.b + n * a.so.n + h * a.so.h + d, ok);
#pragma unroll
    for (int j = 0; j < 8; ++j) D = fmaf(to_f<F16>(df[ks][j]), to_f<F16>(of[j]), D);
  }
  D = half_sum(D);
  const float c = a.scale * LOG2E, nl = live ? -lse * LOG2E : -INFINITY;   // P = exp2(c S + nl): 0 for a row without keys or past the end
  f32x16 dq[HD];
#pragma unroll
  for (int db = 0; db < HD; ++db) dq[db] = splat(0.f);
  if (c_lo < c_hi) store(0);
  __syncthreads();
  const int first = SUMS ? c_hi - c_lo : 0, all = first + c_hi - c_lo;
  float Dx = 0.f;
  int up = F16 ? DS_UP : 0;
  for (int it = 0; it < all; ++it) {
    const bool more = it + 1 < all, sums = SUMS && it < first;
    const int ch = c_lo + (sums || !SUMS ? it : it - first), buf = it & 1;
    if (more) load(SUMS && it + 1 >= first ? c_lo + it + 1 - first : c_lo + it + 1);
    if (SUMS && it == first) D = half_sum(Dx);
    const char* K = smem + buf * BUF;
    const char* V = K + img_bytes<HD>();
    const float* bs = reinterpret_cast<const float*>(V + img_bytes<HD>());
    if (row0 < a.R) {
      const bool biased = mask || (ch + 1) * KC > kend;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        f32x16 s, dp;
#pragma unroll
        for (int ks = 0; ks < 2 * HD; ++ks) {
          s = mma<F16>(row_frag<HD>(K, t, ks), qf[ks], ks ? s : splat(0.f));
          dp = mma<F16>(row_frag<HD>(V, t, ks), df[ks], ks ? dp : splat(0.f));
        }
        if (biased) {
#pragma unroll
          for (int gq = 0; gq < 4; ++gq) {
            const float4 x = *reinterpret_cast<const float4*>(bs + t * 32 + 8 * gq + 4 * hi);
            s[4 * gq] += x.x; s[4 * gq + 1] += x.y; s[4 * gq + 2] += x.z; s[4 * gq + 3] += x.w;
          }
        }
        const float off = SUMS && sums ? 0.f : D, nu = F16 && !(SUMS && sums) ? nl + (float)up : nl;
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = fmaf(s[e], c, nu);
#pragma unroll
        for (int e = 0; e < 16; ++e) dp[e] = (dp[e] - off) * __builtin_amdgcn_exp2f(s[e]);
        if (SUMS && sums) {
#pragma unroll
          for (int e = 0; e < 16; ++e) Dx += dp[e];
          continue;
        }
        if constexpr (F16) bring_down<HD>(dp, up, dq);
        const s16x8 d0 = pack8<F16>(dp, 0), d1 = pack8<F16>(dp, 8);
#pragma unroll
        for (int db = 0; db < HD; ++db) dq[db] = mma<F16>(tr_frag<HD>(K, db, t * 32), d0, dq[db]);
#pragma unroll
        for (int db = 0; db < HD; ++db) dq[db] = mma<F16>(tr_frag<HD>(K, db, t * 32 + 16), d1, dq[db]);
      }
    }
    if (more) store(buf ^ 1);
    __syncthreads();
  }
  if (split == 0 && hi == 0 && r < a.R) a.delta[(int64_t)bh * a.R + r] = D;
  const float mul = F16 ? __builtin_amdgcn_ldexpf(a.scale, -up) : a.scale;
  if (a.splits > 1) {
    if (r < a.R) put_partial<HD>(a.ws + ((int64_t)split * a.B * a.Hkv * a.R + (int64_t)bh * a.R + r) * a.dh, dq, mul, a.dh);
    return;
  }
  put_tile<F16, HD>(smem + wave * (32 * HD * 64), dq, mul, a.dh, [&](int x) -> uint16_t* {
    const int rr = row0 + x, gg = rr / a.Nq, nn = rr - gg * a.Nq;
    return rr < a.R ? a.dq + b * a.sdq.b + nn * a.sdq.n + (int64_t)(hk * a.G + gg) * a.sdq.h : nullptr;
  });
}

// dK / dV: a wave owns 32 keys (K, V fragments and both accumulators in registers), the query rows pass through LDS in chunks of 64
// (3138 rows x 6273 keys x 16 heads of 64, masked, the matrix unit busy 31 % of it, waves waiting 44 %: 235 - 247 us = 650 - 685 TFLOP/s, hidden keys counted).
template <bool F16, int HD>
__global__ __launch_bounds__(NT, HD <= 2 ? 2 : 1) void xattn_dkdv_kernel(const XArgs a) {
  constexpr int BUF = 2 * img_bytes<HD>() + 2 * KC * 4;
  __shared__ __attribute__((aligned(16))) char smem[2 * BUF];
  int bh, item;
  if (!my_item(a, a.tiles * a.splits, bh, item)) return;
  const int b = bh / a.Hkv, hk = bh % a.Hkv, tile = item % a.tiles, split = item / a.tiles;
  const int wave = threadIdx.x >> 6, l = lane(), hi = l >> 5;
  const int kend = key_end(a, b);
  const int key = (tile * 4 + wave) * 32 + (l & 31);
  const bool seen = key < kend && (!a.kmask || a.kmask[(int64_t)b * a.Nk + key]);
  const int chunks = tile * 128 < kend ? (a.R + KC - 1) / KC : 0, per = (chunks + a.splits - 1) / a.splits;
  const int c_lo = min(split * per, chunks), c_hi = min(c_lo + per, chunks);
  const uint16_t* qb = a.q + b * a.sq.b + (int64_t)hk * a.G * a.sq.h;
  const uint16_t* db_ = a.dout + b * a.sdo.b + (int64_t)hk * a.G * a.sdo.h;
  Chunk<HD> qr, dr;
  qr.offsets(a.sq.n, a.dh);
  dr.offsets(a.sdo.n, a.dh);
  float l_reg = 0.f, d_reg = 0.f;
  int g0 = __builtin_amdgcn_readfirstlane(c_lo * KC / a.Nq), n0 = c_lo * KC - g0 * a.Nq;   // head and token of the next chunk's first row
  auto load = [&](int ch) {
    qr.load_rows(qb, a.sq, ch * KC, g0, n0, a.R, a.Nq, a.dh);
    dr.load_rows(db_, a.sdo, ch * KC, g0, n0, a.R, a.Nq, a.dh);
    for (n0 += KC; n0 >= a.Nq; n0 -= a.Nq) ++g0;
    if (threadIdx.x < KC) {
      const int r = ch * KC + threadIdx.x;
      l_reg = r < a.R ? row_start(a.lse[((int64_t)b * a.H + hk * a.G) * a.Nq + r], a.scale) : -INFINITY;   // rows of a group lie one after the other
      d_reg = r < a.R ? -a.delta[(int64_t)bh * a.R + r] : 0.f;
    }
  };
  auto store = [&](int buf) {
    char* p = smem + buf * BUF;
    qr.store(p);
    dr.store(p + img_bytes<HD>());
    if (threadIdx.x < KC) {
      float* st = reinterpret_cast<float*>(p + 2 * img_bytes<HD>());
      st[threadIdx.x] = l_reg;
      st[KC + threadIdx.x] = d_reg;
    }
  };
  if (c_lo < c_hi) load(c_lo);
  KeyTile<HD> kf, vf;
  kf.load(a.k + b * a.sk.b + hk * a.sk.h, a.sk.n, key, seen, a.dh);
  vf.load(a.v + b * a.sv.b + hk * a.sv.h, a.sv.n, key, seen, a.dh);
  f32x16 dk[HD], dv[HD];
#pragma unroll
  for (int db = 0; db < HD; ++db) { dk[db] = splat(0.f); dv[db] = splat(0.f); }
  const float c = a.scale * LOG2E;
  int up = F16 ? DS_UP : 0;
  const bool any = __builtin_amdgcn_ballot_w64(seen) != 0;
  if (c_lo < c_hi) store(0);
  __syncthreads();
  for (int ch = c_lo; ch < c_hi; ++ch) {
    const int buf = (ch - c_lo) & 1;
    const bool more = ch + 1 < c_hi;
    if (more) load(ch + 1);
    const char* Q = smem + buf * BUF;
    const char* O = Q + img_bytes<HD>();
    const float* st = reinterpret_cast<const float*>(O + img_bytes<HD>());
    if (any) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      if (t && ch * KC + 32 >= a.R) break;   // the last chunk's second tile holds no rows
      f32x16 s, dp;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const float4 x = *reinterpret_cast<const float4*>(st + t * 32 + 8 * g + 4 * hi);
        const float4 y = *reinterpret_cast<const float4*>(st + KC + t * 32 + 8 * g + 4 * hi);
        s[4 * g] = x.x; s[4 * g + 1] = x.y; s[4 * g + 2] = x.z; s[4 * g + 3] = x.w;
        dp[4 * g] = y.x; dp[4 * g + 1] = y.y; dp[4 * g + 2] = y.z; dp[4 * g + 3] = y.w;
      }   // (a hidden key's column is finite or, for rows without statistics, zero; its results are replaced by zeros at the end)
#pragma unroll
      for (int ks = 0; ks < 2 * HD; ++ks) {
        s = mma<F16>(row_frag<HD>(Q, t, ks), kf.f[ks], s);
        dp = mma<F16>(row_frag<HD>(O, t, ks), vf.f[ks], dp);
      }
      if constexpr (F16) {
        scaled_factors(s, dp, c, up);
        bring_down<HD>(dp, up, dk);
      } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          s[e] = __builtin_amdgcn_exp2f(s[e] * c);
          dp[e] *= s[e];
        }
      }
      const s16x8 p0 = pack8<F16>(s, 0), p1 = pack8<F16>(s, 8), d0 = pack8<F16>(dp, 0), d1 = pack8<F16>(dp, 8);
#pragma unroll
      for (int db = 0; db < HD; ++db) {
        dv[db] = mma<F16>(tr_frag<HD>(O, db, t * 32), p0, dv[db]);
        dk[db] = mma<F16>(tr_frag<HD>(Q, db, t * 32), d0, dk[db]);
      }
#pragma unroll
      for (int db = 0; db < HD; ++db) {
        dv[db] = mma<F16>(tr_frag<HD>(O, db, t * 32 + 16), p1, dv[db]);
        dk[db] = mma<F16>(tr_frag<HD>(Q, db, t * 32 + 16), d1, dk[db]);
      }
    }
    }
    if (more) store(buf ^ 1);
    __syncthreads();
  }
  if (!seen) {   // gradients of keys that are not visible are zero whatever dO holds
#pragma unroll
    for (int db = 0; db < HD; ++db) { dk[db] = splat(0.f); dv[db] = splat(0.f); }
  }
  const float vmul = F16 ? 1.f / P_UP : 1.f, kmul = F16 ? __builtin_amdgcn_ldexpf(a.scale, -up) : a.scale;
  if (a.splits > 1) {
    if (key >= a.Nk) return;
    const int64_t keys = (int64_t)a.B * a.Hkv * a.Nk, at = split * keys + (int64_t)bh * a.Nk + key;
    put_partial<HD>(a.ws + at * a.dh, dk, kmul, a.dh);
    put_partial<HD>(a.ws + (a.splits * keys + at) * a.dh, dv, vmul, a.dh);
    return;
  }
  const int key0 = (tile * 4 + wave) * 32;
  char* img = smem + wave * (32 * HD * 64);
  put_tile<F16, HD>(img, dk, kmul, a.dh, [&](int x) -> uint16_t* { return key0 + x < a.Nk ? a.dk + b * a.sdk.b + (int64_t)(key0 + x) * a.sdk.n + hk * a.sdk.h : nullptr; });
  put_tile<F16, HD>(img, dv, vmul, a.dh, [&](int x) -> uint16_t* { return key0 + x < a.Nk ? a.dv + b * a.sdv.b + (int64_t)(key0 + x) * a.sdv.n + hk * a.sdv.h : nullptr; });
}

// dK / dV with the rows resident (all of q and dO of a (batch entry, key head) in LDS: up to 224 rows at head_dim 64): staged once, after that every
// wave walks its own key tiles without a barrier, the next tile's K / V in flight.  The chunked kernel above spends more on its pipeline's
// start and drain than on the products when there are few chunks (196 rows against 1370 keys, batch 32 x 12 heads: 119 us against 98 us, of which 54 are the bytes of K, V, dK and dV).
template <int HD> constexpr int rows_resident() { return ((HD <= 2 ? 80 : 156) * 1024 - 4 * 32 * HD * 64) / (HD * 128 + 8) / 32 * 32; }   // two workgroups (head_dim > 64: one) to a CU
template <bool F16, int HD>
__global__ __launch_bounds__(NT, HD <= 2 ? 2 : 1) void xattn_dkdv_rows_kernel(const XArgs a) {
  constexpr int RM = rows_resident<HD>();
  __shared__ __attribute__((aligned(16))) char smem[RM * (HD * 128 + 8) + 4 * 32 * HD * 64];
  int bh, split;
  if (!my_item(a, a.splits, bh, split)) return;
  const int b = bh / a.Hkv, hk = bh % a.Hkv;
  const int wave = threadIdx.x >> 6, l = lane(), hi = l >> 5;
  const int kend = key_end(a, b), tiles = (a.Nk + 31) / 32, per = (tiles + a.splits - 1) / a.splits;   // tiles behind kend: zeros to write
  const int t_lo = min(split * per, tiles), t_hi = min(t_lo + per, tiles);
  const uint16_t* kb = a.k + b * a.sk.b + hk * a.sk.h;
  const uint16_t* vb = a.v + b * a.sv.b + hk * a.sv.h;
  const uint8_t* mask = a.kmask ? a.kmask + (int64_t)b * a.Nk : nullptr;
  const int rt = (a.R + 31) / 32;
  char* Q = smem;
  char* O = smem + RM * HD * 64;
  float* st = reinterpret_cast<float*>(smem + 2 * RM * HD * 64);   // [RM] score starts, [RM] -D
  char* img = smem + RM * (HD * 128 + 8) + wave * (32 * HD * 64);
  KeyTile<HD> kn, vn;
  bool in = false;
  uint8_t mb = 1;
  auto load = [&](int t) {
    const int key = t * 32 + (l & 31);
    in = t < t_hi && key < kend;
    kn.load(kb, a.sk.n, key, in, a.dh);
    vn.load(vb, a.sv.n, key, in, a.dh);
    if (mask) mb = in ? mask[key] : 0;
  };
  load(t_lo + wave);
  for (int i = threadIdx.x; i < rt * 32 * 4 * HD; i += NT) {
    const int r = i / (4 * HD), c = i % (4 * HD), g = r / a.Nq, n = r - g * a.Nq;
    const bool ok = r < a.R && c * 8 < a.dh;
    *reinterpret_cast<s16x8*>(Q + img_off<HD>(r, c)) = ld8(a.q + b * a.sq.b + n * a.sq.n + (int64_t)(hk * a.G + g) * a.sq.h + c * 8, ok);
    *reinterpret_cast<s16x8*>(O + img_off<HD>(r, c)) = ld8(a.dout + b * a.sdo.b + n * a.sdo.n + (int64_t)(hk * a.G + g) * a.sdo.h + c * 8, ok);
  }
  for (int r = threadIdx.x; r < rt * 32; r += NT) {
    st[r] = r < a.R ? row_start(a.lse[((int64_t)b * a.H + hk * a.G) * a.Nq + r], a.scale) : -INFINITY;
    st[RM + r] = r < a.R ? -a.delta[(int64_t)bh * a.R + r] : 0.f;
  }
  const float c = a.scale * LOG2E;
  __syncthreads();
  for (int t = t_lo + wave; t < t_hi; t += 4) {
    KeyTile<HD> kf = kn, vf = vn;
    const bool seen = in && mb;
    const uint32_t all = (uint32_t)__builtin_amdgcn_ballot_w64(seen);
    if (all != 0xffffffffu) {
      kf.hide(seen);
      vf.hide(seen);
    }
    load(t + 4);
    f32x16 dk[HD], dv[HD];
#pragma unroll
    for (int db = 0; db < HD; ++db) { dk[db] = splat(0.f); dv[db] = splat(0.f); }
    int up = F16 ? DS_UP : 0;
    for (int x = 0; x < (all ? rt : 0); ++x) {
      f32x16 s, dp;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const float4 y = *reinterpret_cast<const float4*>(st + x * 32 + 8 * g + 4 * hi);
        const float4 z = *reinterpret_cast<const float4*>(st + RM + x * 32 + 8 * g + 4 * hi);
        s[4 * g] = y.x; s[4 * g + 1] = y.y; s[4 * g + 2] = y.z; s[4 * g + 3] = y.w;
        dp[4 * g] = z.x; dp[4 * g + 1] = z.y; dp[4 * g + 2] = z.z; dp[4 * g + 3] = z.w;
      }
#pragma unroll
      for (int ks = 0; ks < 2 * HD; ++ks) {
        s = mma<F16>(row_frag<HD>(Q, x, ks), kf.f[ks], s);
        dp = mma<F16>(row_frag<HD>(O, x, ks), vf.f[ks], dp);
      }
      if constexpr (F16) {   // (a hidden key's column is replaced by zeros below)
        scaled_factors(s, dp, c, up);
        bring_down<HD>(dp, up, dk);
      } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] *= c;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          s[e] = __builtin_amdgcn_exp2f(s[e]);
          dp[e] *= s[e];
        }
      }
      const s16x8 p0 = pack8<F16>(s, 0), p1 = pack8<F16>(s, 8), d0 = pack8<F16>(dp, 0), d1 = pack8<F16>(dp, 8);
#pragma unroll
      for (int db = 0; db < HD; ++db) {
        dv[db] = mma<F16>(tr_frag<HD>(O, db, x * 32), p0, dv[db]);
        dk[db] = mma<F16>(tr_frag<HD>(Q, db, x * 32), d0, dk[db]);
      }
#pragma unroll
      for (int db = 0; db < HD; ++db) {
        dv[db] = mma<F16>(tr_frag<HD>(O, db, x * 32 + 16), p1, dv[db]);
        dk[db] = mma<F16>(tr_frag<HD>(Q, db, x * 32 + 16), d1, dk[db]);
      }
    }
    if (!seen) {
#pragma unroll
      for (int db = 0; db < HD; ++db) { dk[db] = splat(0.f); dv[db] = splat(0.f); }
    }
    put_tile<F16, HD>(img, dk, F16 ? __builtin_amdgcn_ldexpf(a.scale, -up) : a.scale, a.dh, [&](int x) -> uint16_t* { return t * 32 + x < a.Nk ? a.dk + b * a.sdk.b + (int64_t)(t * 32 + x) * a.sdk.n + hk * a.sdk.h : nullptr; });
    put_tile<F16, HD>(img, dv, F16 ? 1.f / P_UP : 1.f, a.dh,
                      [&](int x) -> uint16_t* { return t * 32 + x < a.Nk ? a.dv + b * a.sdv.b + (int64_t)(t * 32 + x) * a.sdv.n + hk * a.sdv.h : nullptr; });
  }
}

// Few rows (R <= 32): every key tile meets the one row tile once, so dK / dV of the tile are complete at once and all three gradients take ONE pass
// over K / V.  Each wave owns key tiles; S is formed in both orientations (lane -> key for dK / dV, lane -> query for dQ): the second set of
// products costs less than turning dS through LDS, and the pass is bound by memory (384 heads x 785 keys of 64, 155 MB: 38 us = 4.0 TB/s; without the second halves of the
// rounded factors 34 us).
template <bool F16, int HD>
__global__ __launch_bounds__(NT, HD <= 2 ? 2 : 1) void xattn_bwd_few_kernel(const XArgs a) {
  constexpr int IMG = 32 * HD * 64, OST = HD * 32 + 4;
  constexpr int TAIL = 4 * 32 * OST * 4, HEAD = 6 * IMG + (2 + 4) * 32 * 4;
  __shared__ __attribute__((aligned(16))) char smem[TAIL > HEAD ? TAIL : HEAD];
  int bh, split;
  if (!my_item(a, a.splits, bh, split)) return;
  const int b = bh / a.Hkv, hk = bh % a.Hkv;
  const int wave = threadIdx.x >> 6, l = lane(), hi = l >> 5;
  const int kend = key_end(a, b), tiles = (a.Nk + 31) / 32, per = (tiles + a.splits - 1) / a.splits;   // tiles behind kend: zeros to write
  const int t_lo = min(split * per, tiles), t_hi = min(t_lo + per, tiles);
  const uint16_t* kb = a.k + b * a.sk.b + hk * a.sk.h;
  const uint16_t* vb = a.v + b * a.sv.b + hk * a.sv.h;
  const uint8_t* mask = a.kmask ? a.kmask + (int64_t)b * a.Nk : nullptr;
  char* Q = smem;
  char* O = smem + IMG;
  char* Kt = smem + (2 + wave) * IMG;
  float* st = reinterpret_cast<float*>(smem + 6 * IMG);   // [32] score starts, [32] -D, [4][32] the waves' shares of D
  KeyTile<HD> kn, vn;
  bool in = false;
  uint8_t mb = 1;
  auto load = [&](int t) {
    const int key = t * 32 + (l & 31);
    in = t < t_hi && key < kend;
    kn.load(kb, a.sk.n, key, in, a.dh);
    vn.load(vb, a.sv.n, key, in, a.dh);
    if (mask) mb = in ? mask[key] : 0;
  };
  load(t_lo + wave);
  const int r = l & 31, g = r / a.Nq, n = r - g * a.Nq;
  const int64_t h = hk * a.G + g;
  const float lse = r < a.R ? a.lse[((int64_t)b * a.H + h) * a.Nq + n] : -INFINITY;
  const bool live = lse != -INFINITY;
  const float s0 = row_start(lse, a.scale), c = a.scale * LOG2E;
  float D = 0.f;
  {
    KeyTile<HD> q, d;
#pragma unroll
    for (int ks = 0; ks < 2 * HD; ++ks) {
      const int dd = ks * 16 + hi * 8;
      const bool ok = live && dd < a.dh;
      q.f[ks] = ld8(a.q + b * a.sq.b + n * a.sq.n + h * a.sq.h + dd, ok);
      d.f[ks] = ld8(a.dout + b * a.sdo.b + n * a.sdo.n + h * a.sdo.h + dd, ok);
      const s16x8 of = ld8(a.o + b * a.so.b + n * a.so.n + h * a.so.h + dd, ok);
#pragma unroll
      for (int j = 0; j < 8; ++j) D = fmaf(to_f<F16>(d.f[ks][j]), to_f<F16>(of[j]), D);
    }
    if (wave == 0) {
      q.store(Q);
      d.store(O);
    }
  }
  D = half_sum(D);
  f32x16 dq[HD];
  int up = F16 ? DS_UP : 0;
#pragma unroll
  for (int db = 0; db < HD; ++db) dq[db] = splat(0.f);
  __syncthreads();
  auto columns = [&](const KeyTile<HD>& kf, const KeyTile<HD>& vf, uint32_t all, float start, f32x16& s, f32x16& dp) {   // lane -> query
    s = splat(s0);
    dp = splat(start);
    if (all != 0xffffffffu) {
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e] = (all >> crow(e, hi)) & 1 ? s[e] : -INFINITY;
    }
#pragma unroll
    for (int ks = 0; ks < 2 * HD; ++ks) {
      s = mma<F16>(kf.f[ks], row_frag<HD>(Q, 0, ks), s);
      dp = mma<F16>(vf.f[ks], row_frag<HD>(O, 0, ks), dp);
    }
  };
  if (a.splits == 1 && tiles <= 4) {
    // Few keys as well: D = sum_k P dP from the fp32 products instead of rowsum(dO * O), whose rounded O would be most of dS's error when a row's
    // probabilities are spread over a few keys only.  Every wave holds its one tile.
    const uint32_t all = (uint32_t)__builtin_amdgcn_ballot_w64(in && mb);
    kn.hide(in && mb);
    vn.hide(in && mb);
    f32x16 s, dp;
    columns(kn, vn, all, 0.f, s, dp);
    D = 0.f;
#pragma unroll
    for (int e = 0; e < 16; ++e) D = fmaf(__builtin_amdgcn_exp2f(s[e] * c), dp[e], D);
    D = half_sum(D);
    if (hi == 0) st[(2 + wave) * 32 + r] = wave < tiles ? D : 0.f;
    __syncthreads();
    D = ((st[2 * 32 + r] + st[3 * 32 + r]) + st[4 * 32 + r]) + st[5 * 32 + r];
  }
  if (wave == 0 && hi == 0) { st[r] = s0; st[32 + r] = -D; }
  __syncthreads();
  for (int t = t_lo + wave; t < t_hi; t += 4) {
    KeyTile<HD> kf = kn, vf = vn;
    const bool seen = in && mb;
    const uint32_t all = (uint32_t)__builtin_amdgcn_ballot_w64(seen);
    if (all != 0xffffffffu) {
      kf.hide(seen);
      vf.hide(seen);
    }
    load(t + 4);
    kf.store(Kt);
    f32x16 s, dp;
    columns(kf, vf, all, -D, s, dp);
#pragma unroll
    for (int e = 0; e < 16; ++e) dp[e] *= __builtin_amdgcn_exp2f(F16 ? fmaf(s[e], c, (float)up) : s[e] * c);
    if constexpr (F16) bring_down<HD>(dp, up, dq);
    s16x8 d0, d1, e0, e1;
    split8<F16>(dp, 0, d0, e0);
    split8<F16>(dp, 8, d1, e1);
    wait_lds();
#pragma unroll
    for (int db = 0; db < HD; ++db) {
      const s16x8 k0 = tr_frag<HD>(Kt, db, 0), k1 = tr_frag<HD>(Kt, db, 16);
      dq[db] = mma<F16>(k0, d0, dq[db]);
      dq[db] = mma<F16>(k0, e0, dq[db]);
      dq[db] = mma<F16>(k1, d1, dq[db]);
      dq[db] = mma<F16>(k1, e1, dq[db]);
    }
    wait_lds();
    // lane -> key
#pragma unroll
    for (int gq = 0; gq < 4; ++gq) {
      const float4 x = *reinterpret_cast<const float4*>(st + 8 * gq + 4 * hi);
      const float4 y = *reinterpret_cast<const float4*>(st + 32 + 8 * gq + 4 * hi);
      s[4 * gq] = x.x; s[4 * gq + 1] = x.y; s[4 * gq + 2] = x.z; s[4 * gq + 3] = x.w;
      dp[4 * gq] = y.x; dp[4 * gq + 1] = y.y; dp[4 * gq + 2] = y.z; dp[4 * gq + 3] = y.w;
    }
#pragma unroll
    for (int ks = 0; ks < 2 * HD; ++ks) {
      s = mma<F16>(row_frag<HD>(Q, 0, ks), kf.f[ks], s);
      dp = mma<F16>(row_frag<HD>(O, 0, ks), vf.f[ks], dp);
    }
    float kmul = a.scale;   // (a hidden key's column is replaced by zeros below)
    if constexpr (F16) {   // every product of a key is here: its largest to 2^11 .. 2^12
      scaled_factors(s, dp, c, 12);
      const int n = min(12 - __builtin_amdgcn_frexp_expf(column_max(dp)), 100);   // (2^n stays finite)
      const float f = pow2(n);
#pragma unroll
      for (int e = 0; e < 16; ++e) dp[e] *= f;
      kmul = __builtin_amdgcn_ldexpf(a.scale, -12 - n);
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        s[e] = __builtin_amdgcn_exp2f(s[e] * c);
        dp[e] *= s[e];
      }
    }
    split8<F16>(dp, 0, d0, e0);
    split8<F16>(dp, 8, d1, e1);
    f32x16 acc[HD];
#pragma unroll
    for (int db = 0; db < HD; ++db) {
      const s16x8 q0 = tr_frag<HD>(Q, db, 0), q1 = tr_frag<HD>(Q, db, 16);
      acc[db] = mma<F16>(q0, d0, splat(0.f));
      acc[db] = mma<F16>(q0, e0, acc[db]);
      acc[db] = mma<F16>(q1, d1, acc[db]);
      acc[db] = mma<F16>(q1, e1, acc[db]);
      if (!seen) acc[db] = splat(0.f);   // whatever dO holds
    }
    put_tile<F16, HD>(Kt, acc, kmul, a.dh, [&](int x) -> uint16_t* { return t * 32 + x < a.Nk ? a.dk + b * a.sdk.b + (int64_t)(t * 32 + x) * a.sdk.n + hk * a.sdk.h : nullptr; });
    split8<F16>(s, 0, d0, e0);
    split8<F16>(s, 8, d1, e1);
#pragma unroll
    for (int db = 0; db < HD; ++db) {
      const s16x8 o0 = tr_frag<HD>(O, db, 0), o1 = tr_frag<HD>(O, db, 16);
      acc[db] = mma<F16>(o0, d0, splat(0.f));
      acc[db] = mma<F16>(o0, e0, acc[db]);
      acc[db] = mma<F16>(o1, d1, acc[db]);
      acc[db] = mma<F16>(o1, e1, acc[db]);
      if (!seen) acc[db] = splat(0.f);
    }
    put_tile<F16, HD>(Kt, acc, F16 ? 1.f / P_UP : 1.f, a.dh,
                      [&](int x) -> uint16_t* { return t * 32 + x < a.Nk ? a.dv + b * a.sdv.b + (int64_t)(t * 32 + x) * a.sdv.n + hk * a.sdv.h : nullptr; });
  }
  __syncthreads();   // images -> the waves' partial dQ rows
  if (r < a.R) put_partial<HD>(reinterpret_cast<float*>(smem) + (wave * 32 + r) * OST, dq, F16 ? __builtin_amdgcn_ldexpf(a.scale, -up) : a.scale, HD * 32);
  __syncthreads();
  const float* part = reinterpret_cast<const float*>(smem);
  const int d4n = a.dh >> 2;
  for (int i = threadIdx.x; i < a.R * d4n; i += NT) {
    const int row = i / d4n, dd = (i - row * d4n) * 4;
    float4 acc = *reinterpret_cast<const float4*>(part + row * OST + dd);
#pragma unroll
    for (int w = 1; w < 4; ++w) {
      const float4 x = *reinterpret_cast<const float4*>(part + (w * 32 + row) * OST + dd);
      acc.x += x.x; acc.y += x.y; acc.z += x.z; acc.w += x.w;
    }
    if (a.splits > 1) {
      *reinterpret_cast<float4*>(a.ws + ((int64_t)split * a.B * a.Hkv * a.R + (int64_t)bh * a.R + row) * a.dh + dd) = acc;
    } else {
      const int gg = row / a.Nq, nn = row - gg * a.Nq;
      *reinterpret_cast<uint2*>(a.dq + b * a.sdq.b + nn * a.sdq.n + (int64_t)(hk * a.G + gg) * a.sdq.h + dd) = make_uint2(pack2<F16>(acc.x, acc.y), pack2<F16>(acc.z, acc.w));
    }
  }
}

// adds the splits' partial rows in split order: row (bh, r) of `part` [splits][B * Hkv * R][dh] -> dst rows of head hk * G + r / Nq, token r % Nq
template <bool F16>
__global__ __launch_bounds__(NT) void xattn_add_kernel(const float* __restrict__ part, uint16_t* __restrict__ dst, Strides s, int splits, int64_t rows, int R,
                                                       int Nq, int G, int Hkv, int dh) {
  const int d4n = dh >> 2;
  const int64_t i = (int64_t)blockIdx.x * NT + threadIdx.x;
  if (i >= rows * d4n) return;
  const int64_t row = i / d4n;
  const int d = (int)(i - row * d4n) * 4;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int k = 0; k < splits; ++k) {
    const float4 x = *reinterpret_cast<const float4*>(part + (k * rows + row) * dh + d);
    acc.x += x.x; acc.y += x.y; acc.z += x.z; acc.w += x.w;
  }
  const int64_t bh = row / R;
  const int r = (int)(row - bh * R), g = r / Nq, n = r - g * Nq;
  const int64_t b = bh / Hkv, h = (bh % Hkv) * G + g;
  *reinterpret_cast<uint2*>(dst + b * s.b + n * s.n + h * s.h + d) = make_uint2(pack2<F16>(acc.x, acc.y), pack2<F16>(acc.z, acc.w));
}

// ================================================================================================================== host
constexpr int CUS = 256;
struct Plan { bool few; int tiles, per_wave, splits; };

int round_up8(int64_t x) { return (int)((x + 7) / 8 * 8); }

// Into how many pieces the contracted axis (`chunks` steps) of `blocks` workgroups is cut, `per_cu` of which a CU holds: the smallest estimated time of
// rounds * (steps + 2) * us_step, plus joining the fp32 partials (`mbytes` per piece: 3.3 MB 4.2 us for 2, 5.5 for 4, 7.9 for 8; 13 MB 8.9 for 2, 15 for 5).  A last round that
// puts n workgroups on a CU costs 1/3 + 2/3 n / per_cu of a full one (measured at head_dim 64: 2.05, 2.8, 3.7 us a chunk with 1, 2, 3 of them): 128
// workgroups over 16 chunks take 30 us uncut, 20.5 + 4 (join) in 2, 17 + 5 in 4 and 17.4 + 6.3 in 6 pieces.  Estimates only rank the cuts; every cut
// gives a right result.
int split_for(int64_t blocks, int chunks, int per_cu, double us_step, double mbytes, double& least) {
  int best = 1;
  least = 1e30;
  for (int s = 1; s <= 64 && s <= (chunks > 1 ? chunks / 2 : 1); ++s) {
    const int64_t full = blocks * s / (per_cu * CUS), rest = blocks * s - full * per_cu * CUS;
    const double rounds = (double)full + (rest ? 1. / 3. + 2. / 3. * (double)((rest + CUS - 1) / CUS) / per_cu : 0.), steps = (double)((chunks + s - 1) / s) + 2;
    const double t = rounds * steps * us_step + (s > 1 ? 3. + 0.2 * s * mbytes : 0.);
    if (t < least) { least = t; best = s; }
  }
  return best;
}
bool few_rows(int R) { return R <= 32; }
// Workgroups that a CU holds (registers; head_dim <= 32 one more than is counted here) and the measured us of a 64-token chunk with that many on it, per
// 32 columns of head_dim:
//   forward, one 32-row tile a wave     3 at head_dim <= 64: 1.15, 2 above: 0.63
//   forward, two tiles a wave           2 at head_dim <= 64: 1.38 (they share every K / V fragment read from LDS: 15 % more rows per us when the card is full)
//   dQ                                  3 at head_dim <= 64: 1.4,  2 up to 96: 1.6, 1 above: 1.0;   dK / dV   2 at head_dim <= 64: 1.15, 1 above: 1.6
// The few-row kernels walk 128 keys a step: 1.5 us (forward; 3 workgroups a CU, 2 above head_dim 64), 2.5 us (backward, 2), 5 us (backward above 64, 1).
// Priced with one more workgroup a CU than is there, head_dim 128 took (both swept): dQ of 8 x 196 x 1370 x 12 heads 169 us in two cuts against 154 uncut; the
// one-query forward of 16 x 1370 x 12 heads 33 us in four against 27 uncut; 16 x 100 x 1025 x 8 heads with resident rows 103 in three against 91 in two.  (The
// one that lost by the right count: the one-query forward of 32 x 1370 x 12 heads, 57 -> 64.)
Plan fwd_plan(int B, int R, int Nk, int Hkv, int dh) {
  const int64_t bh = (int64_t)B * Hkv;
  const int HD = lt_cdiv(dh, 32), chunks = lt_cdiv(Nk, KC);
  const double mb = 4e-6 * bh * R * dh;
  double t1, t2;
  if (few_rows(R)) return {true, 1, 1, split_for(bh, lt_cdiv(Nk, 128), HD <= 2 ? 3 : 2, 1.5, mb, t1)};
  const int n1 = lt_cdiv(R, 128), n2 = lt_cdiv(R, 256);
  const int s1 = split_for(bh * n1, chunks, HD <= 2 ? 3 : 2, (HD <= 2 ? 1.15 : 0.63) * HD, mb, t1);
  if (HD > 2) return {false, n1, 1, s1};
  const int s2 = split_for(bh * n2, chunks, 2, 1.38 * HD, mb, t2);
  return t2 < t1 ? Plan{false, n2, 2, s2} : Plan{false, n1, 1, s1};
}
Plan dq_plan(int B, int R, int Nk, int Hkv, int dh) {
  const int64_t bh = (int64_t)B * Hkv;
  const int HD = lt_cdiv(dh, 32), tiles = lt_cdiv(R, 128);
  const double mb = 4e-6 * bh * R * dh;
  double t;
  if (few_rows(R)) return {true, 1, 1, split_for(bh, lt_cdiv(Nk, 128), HD <= 2 ? 2 : 1, HD <= 2 ? 2.5 : 5., mb, t)};
  return {false, tiles, 1, split_for(bh * tiles, lt_cdiv(Nk, KC), HD <= 2 ? 3 : HD == 3 ? 2 : 1, HD <= 2 ? 1.4 * HD : HD == 3 ? 4.8 : 4., mb, t)};
}
int resident_rows(int HD) { return HD == 1 ? rows_resident<1>() : HD == 2 ? rows_resident<2>() : HD == 3 ? rows_resident<3>() : rows_resident<4>(); }
Plan dkdv_plan(int B, int R, int Nk, int Hkv, int dh) {
  const int HD = lt_cdiv(dh, 32), tiles = lt_cdiv(Nk, 128);
  const int64_t bh = (int64_t)B * Hkv;
  double t;
  if (R <= resident_rows(HD)) {   // no partials to join: cut the keys until the rounds are even; ~4 us to stage the rows, 4 tiles a step
    Plan p{true, 1, 1, 1};
    const int held = (HD <= 2 ? 2 : 1) * CUS;
    double least = 1e30;
    for (int s = 1; s <= tiles && (s == 1 || bh * s <= 16 * held); ++s) {   // (16 rounds: more cuts only stage the rows again)
      const double u = (double)((bh * s + held - 1) / held) * (4. + 0.4 * HD * lt_cdiv(R, 32) * (double)((tiles + s - 1) / s));
      if (u < least) { least = u; p.splits = s; }
    }
    return p;
  }
  return {false, tiles, 1, split_for(bh * tiles, lt_cdiv(R, KC), HD <= 2 ? 2 : 1, (HD <= 2 ? 1.15 : 1.6) * HD, 8e-6 * bh * Nk * dh, t)};
}
int64_t fwd_floats(int B, int R, int Nk, int Hkv, int dh) {
  const Plan p = fwd_plan(B, R, Nk, Hkv, dh);
  return p.splits > 1 ? (int64_t)p.splits * B * Hkv * R * (dh + 2) : 0;
}
int64_t dq_floats(int B, int R, int Nk, int Hkv, int dh) {
  const Plan p = dq_plan(B, R, Nk, Hkv, dh);
  return p.splits > 1 ? (int64_t)p.splits * B * Hkv * R * dh : 0;
}
int64_t delta_floats(int B, int R, int Hkv) { return ((int64_t)B * Hkv * R + 3) / 4 * 4; }
int64_t bwd_floats(int B, int R, int Nk, int Hkv, int dh) {
  int64_t n = dq_floats(B, R, Nk, Hkv, dh);
  if (few_rows(R)) return n;
  const Plan p = dkdv_plan(B, R, Nk, Hkv, dh);
  const int64_t kv = !p.few && p.splits > 1 ? 2 * (int64_t)p.splits * B * Hkv * Nk * dh : 0;
  return delta_floats(B, R, Hkv) + (n > kv ? n : kv);
}

bool strides_ok(const int64_t* s, int B, int N, int H) {
  return (B == 1 || (s[0] >= 0 && s[0] % 8 == 0)) && (N == 1 || (s[1] >= 0 && s[1] % 8 == 0 && s[1] < MAX_STEP)) && (H == 1 || (s[2] >= 0 && s[2] % 8 == 0));
}
Strides st3(const int64_t* s, int N) { return {s[0], N == 1 ? 128 : s[1], s[2]}; }   // (a single token has no step: any will do)
constexpr float MIN_SCALE = 0x1p-100f, MAX_SCALE = 0x1p100f;   // lse / scale and scale * log2(e) have to be finite
constexpr int64_t MAX_GROUPS = 1 << 24;   // 256 threads each: a launch has fewer than 2^32
bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// (what the plans may be asked about: their 32-bit row counts hold it)
bool in_range(int B, int Nq, int Nk, int H, int Hkv) { return (int64_t)Nq * (H / Hkv) < (1 << 24) && Nk < (1 << 24) && (int64_t)B * Hkv < (1 << 20); }

int fill(const lt_cross_attention_desc* d, XArgs& a, const char* who) {
  LT_CHECK_ARG(d->B >= 0 && d->Nq >= 0 && d->Nk >= 0 && d->H > 0 && d->Hkv > 0 && d->H % d->Hkv == 0, "%s: bad sizes (B %d, Nq %d, Nk %d, H %d, Hkv %d)", who, d->B,
               d->Nq, d->Nk, d->H, d->Hkv);
  LT_CHECK_ARG(d->dh >= 8 && d->dh <= 128 && d->dh % 8 == 0, "%s: head_dim must be a multiple of 8 from 8 to 128 (got %d)", who, d->dh);
  LT_CHECK_ARG(d->dtype == LT_DT_BF16 || d->dtype == LT_DT_F16, "%s: dtype must be LT_DT_BF16 or LT_DT_F16", who);
  LT_CHECK_ARG(d->scale >= MIN_SCALE && d->scale <= MAX_SCALE, "%s: scale must lie between 2^-100 and 2^100", who);
  LT_CHECK_ARG(in_range(d->B, d->Nq, d->Nk, d->H, d->Hkv), "%s: sizes out of range", who);
  const int G = d->H / d->Hkv;
  if (d->Nq > 0 && d->B > 0) LT_CHECK_ARG(d->q && aligned16(d->q) && strides_ok(d->sq, d->B, d->Nq, d->H), "%s: q: 16-byte alignment of the pointer and of every stride, token stride below 2^24", who);
  if (d->Nk > 0 && d->B > 0)
    LT_CHECK_ARG(d->k && d->v && aligned16(d->k) && aligned16(d->v) && strides_ok(d->sk, d->B, d->Nk, d->Hkv) && strides_ok(d->sv, d->B, d->Nk, d->Hkv),
                 "%s: k, v: 16-byte alignment of the pointers and of every stride, token strides below 2^24", who);
  if (d->Nq > 0 && d->B > 0) LT_CHECK_ARG(d->out && aligned16(d->out) && strides_ok(d->so, d->B, d->Nq, d->H), "%s: out: 16-byte alignment of the pointer and of every stride, token stride below 2^24", who);
  a = XArgs{};
  a.q = (const uint16_t*)d->q; a.k = (const uint16_t*)d->k; a.v = (const uint16_t*)d->v;
  a.o = (const uint16_t*)d->out; a.out = (uint16_t*)d->out; a.lse = d->lse;
  a.klen = d->key_lens; a.kmask = d->key_mask;
  a.sq = st3(d->sq, d->Nq); a.sk = st3(d->sk, d->Nk); a.sv = st3(d->sv, d->Nk); a.so = st3(d->so, d->Nq);
  a.B = d->B; a.Nq = d->Nq; a.Nk = d->Nk; a.H = d->H; a.Hkv = d->Hkv; a.G = G; a.R = G * d->Nq; a.dh = d->dh; a.scale = d->scale;
  return LT_OK;
}

#define XA_HD(KERNEL, GRID, F16, ...)                                                                                    \
  switch (lt_cdiv(a.dh, 32)) {                                                                                           \
    case 1: hipLaunchKernelGGL((KERNEL<F16, 1 __VA_ARGS__>), dim3(GRID), dim3(NT), 0, (hipStream_t)stream, a); break;    \
    case 2: hipLaunchKernelGGL((KERNEL<F16, 2 __VA_ARGS__>), dim3(GRID), dim3(NT), 0, (hipStream_t)stream, a); break;    \
    case 3: hipLaunchKernelGGL((KERNEL<F16, 3 __VA_ARGS__>), dim3(GRID), dim3(NT), 0, (hipStream_t)stream, a); break;    \
    default: hipLaunchKernelGGL((KERNEL<F16, 4 __VA_ARGS__>), dim3(GRID), dim3(NT), 0, (hipStream_t)stream, a); break;   \
  }

template <bool F16> void run_fwd(const XArgs& a, const Plan& p, void* stream) {
  const int64_t items = (int64_t)round_up8((int64_t)a.B * a.Hkv) * a.tiles * a.splits;
  if (p.few) { XA_HD(xattn_fwd_few_kernel, (unsigned)items, F16) }
  else {
    const int HD = lt_cdiv(a.dh, 32), qt = p.per_wave;
    if (HD == 1 && qt == 2) hipLaunchKernelGGL((xattn_fwd_kernel<F16, 1, 2>), dim3((unsigned)items), dim3(NT), 0, (hipStream_t)stream, a);
    else if (HD == 2 && qt == 2) hipLaunchKernelGGL((xattn_fwd_kernel<F16, 2, 2>), dim3((unsigned)items), dim3(NT), 0, (hipStream_t)stream, a);
    else if (HD == 1) hipLaunchKernelGGL((xattn_fwd_kernel<F16, 1, 1>), dim3((unsigned)items), dim3(NT), 0, (hipStream_t)stream, a);
    else if (HD == 2) hipLaunchKernelGGL((xattn_fwd_kernel<F16, 2, 1>), dim3((unsigned)items), dim3(NT), 0, (hipStream_t)stream, a);
    else if (HD == 3) hipLaunchKernelGGL((xattn_fwd_kernel<F16, 3, 1>), dim3((unsigned)items), dim3(NT), 0, (hipStream_t)stream, a);
    else hipLaunchKernelGGL((xattn_fwd_kernel<F16, 4, 1>), dim3((unsigned)items), dim3(NT), 0, (hipStream_t)stream, a);
  }
  if (a.splits > 1) {
    const int64_t n = (int64_t)a.B * a.Hkv * a.R * (a.dh / 4);
    hipLaunchKernelGGL(xattn_join_kernel<F16>, dim3((unsigned)lt_cdiv(n, NT)), dim3(NT), 0, (hipStream_t)stream, a);
  }
}
template <bool F16> void add_splits(const XArgs& a, const float* part, uint16_t* dst, Strides s, int64_t rows, int R, int Nq, int G, void* stream) {
  hipLaunchKernelGGL(xattn_add_kernel<F16>, dim3((unsigned)lt_cdiv(rows * (a.dh / 4), NT)), dim3(NT), 0, (hipStream_t)stream, part, dst, s, a.splits, rows, R, Nq, G,
                     a.Hkv, a.dh);
}
template <bool F16> void run_bwd(XArgs a, float* ws, void* stream) {
  const int64_t bh8 = round_up8((int64_t)a.B * a.Hkv), rows = (int64_t)a.B * a.Hkv * a.R, keys = (int64_t)a.B * a.Hkv * a.Nk;
  Plan p = dq_plan(a.B, a.R, a.Nk, a.Hkv, a.dh);
  a.tiles = p.tiles; a.splits = p.splits;
  a.delta = ws;
  a.ws = p.few ? ws : ws + delta_floats(a.B, a.R, a.Hkv);
  if (p.few) { XA_HD(xattn_bwd_few_kernel, (unsigned)(bh8 * a.splits), F16) }
  else if (a.splits == 1 && a.Nk <= 2 * KC) { XA_HD(xattn_dq_kernel, (unsigned)(bh8 * a.tiles), F16, , true) }
  else { XA_HD(xattn_dq_kernel, (unsigned)(bh8 * a.tiles * a.splits), F16, , false) }
  if (a.splits > 1) add_splits<F16>(a, a.ws, a.dq, a.sdq, rows, a.R, a.Nq, a.G, stream);
  if (p.few || a.Nk == 0) return;
  p = dkdv_plan(a.B, a.R, a.Nk, a.Hkv, a.dh);
  a.tiles = p.tiles; a.splits = p.splits;
  if (p.few) {
    XA_HD(xattn_dkdv_rows_kernel, (unsigned)(bh8 * a.splits), F16)
    return;
  }
  XA_HD(xattn_dkdv_kernel, (unsigned)(bh8 * a.tiles * a.splits), F16)
  if (a.splits > 1) {
    add_splits<F16>(a, a.ws, a.dk, a.sdk, keys, a.Nk, a.Nk, 1, stream);
    add_splits<F16>(a, a.ws + a.splits * keys * a.dh, a.dv, a.sdv, keys, a.Nk, a.Nk, 1, stream);
  }
}

__global__ void xattn_zero_kernel(uint16_t* dst, Strides s, int64_t n, int N, int H, int d8) {
  for (int64_t i = (int64_t)blockIdx.x * NT + threadIdx.x; i < n; i += (int64_t)gridDim.x * NT) {
    const int c = (int)(i % d8), h = (int)(i / d8 % H);
    const int64_t t = i / d8 / H;
    *reinterpret_cast<uint4*>(dst + t / N * s.b + t % N * s.n + h * s.h + c * 8) = make_uint4(0, 0, 0, 0);
  }
}

}  // namespace

extern "C" int64_t lt_cross_attention_fwd_ws_floats(int B, int Nq, int Nk, int H, int Hkv, int dh) {
  if (B <= 0 || Nq <= 0 || Nk <= 0 || H <= 0 || Hkv <= 0 || H % Hkv || dh <= 0 || dh > 128 || !in_range(B, Nq, Nk, H, Hkv)) return 0;
  return fwd_floats(B, Nq * (H / Hkv), Nk, Hkv, dh);
}
extern "C" int64_t lt_cross_attention_bwd_ws_floats(int B, int Nq, int Nk, int H, int Hkv, int dh) {
  if (B <= 0 || Nq <= 0 || Nk < 0 || H <= 0 || Hkv <= 0 || H % Hkv || dh <= 0 || dh > 128 || !in_range(B, Nq, Nk, H, Hkv)) return 0;
  return bwd_floats(B, Nq * (H / Hkv), Nk, Hkv, dh);
}

extern "C" int lt_cross_attention_fwd(const lt_cross_attention_desc* d, void* stream) {
  LT_CHECK_ARG(d, "lt_cross_attention_fwd: no descriptor");
  XArgs a;
  const int rc = fill(d, a, "lt_cross_attention_fwd");
  if (rc != LT_OK) return rc;
  if (d->B == 0 || d->Nq == 0) return LT_OK;
  const Plan p = fwd_plan(a.B, a.R, a.Nk, a.Hkv, a.dh);
  a.tiles = p.tiles; a.splits = p.splits; a.ws = d->ws;
  const int64_t need = fwd_floats(a.B, a.R, a.Nk, a.Hkv, a.dh);
  LT_CHECK_ARG(need == 0 || (d->ws && aligned16(d->ws) && d->ws_floats >= need), "lt_cross_attention_fwd: a workspace of %lld floats is needed (got %lld)", (long long)need,
               (long long)(d->ws ? d->ws_floats : 0));
  LT_CHECK_ARG((int64_t)round_up8((int64_t)a.B * a.Hkv) * a.tiles * a.splits < MAX_GROUPS, "lt_cross_attention_fwd: too many workgroups");
  if (d->dtype == LT_DT_F16) run_fwd<true>(a, p, stream);
  else run_fwd<false>(a, p, stream);
  LT_CHECK_LAUNCH("lt_cross_attention_fwd");
}

extern "C" int lt_cross_attention_bwd(const lt_cross_attention_desc* d, void* stream) {
  LT_CHECK_ARG(d, "lt_cross_attention_bwd: no descriptor");
  XArgs a;
  const int rc = fill(d, a, "lt_cross_attention_bwd");
  if (rc != LT_OK) return rc;
  if (d->B == 0) return LT_OK;
  if (d->Nq > 0)
    LT_CHECK_ARG(d->lse && d->dout && d->dq && aligned16(d->dout) && aligned16(d->dq) && strides_ok(d->sdo, d->B, d->Nq, d->H) && strides_ok(d->sdq, d->B, d->Nq, d->H),
                 "lt_cross_attention_bwd: lse, dout, dq: missing, pointer or strides not 16-byte aligned, or a token stride of 2^24 or more");
  if (d->Nk > 0)
    LT_CHECK_ARG(d->dk && d->dv && aligned16(d->dk) && aligned16(d->dv) && strides_ok(d->sdk, d->B, d->Nk, d->Hkv) && strides_ok(d->sdv, d->B, d->Nk, d->Hkv),
                 "lt_cross_attention_bwd: dk, dv: missing, pointer or strides not 16-byte aligned, or a token stride of 2^24 or more");
  a.dout = (const uint16_t*)d->dout; a.dq = (uint16_t*)d->dq; a.dk = (uint16_t*)d->dk; a.dv = (uint16_t*)d->dv;
  a.sdo = st3(d->sdo, d->Nq); a.sdq = st3(d->sdq, d->Nq); a.sdk = st3(d->sdk, d->Nk); a.sdv = st3(d->sdv, d->Nk);
  if (d->Nq == 0) {   // no queries: the keys' gradients are zero
    if (d->Nk > 0) {
      const int64_t n = (int64_t)a.B * a.Nk * a.Hkv * (a.dh / 8);
      const unsigned grid = (unsigned)(n < 64 * CUS * NT ? lt_cdiv(n, NT) : 64 * CUS);
      hipLaunchKernelGGL(xattn_zero_kernel, dim3(grid), dim3(NT), 0, (hipStream_t)stream, a.dk, a.sdk, n, a.Nk, a.Hkv, a.dh / 8);
      hipLaunchKernelGGL(xattn_zero_kernel, dim3(grid), dim3(NT), 0, (hipStream_t)stream, a.dv, a.sdv, n, a.Nk, a.Hkv, a.dh / 8);
    }
    LT_CHECK_LAUNCH("lt_cross_attention_bwd");
  }
  const int64_t need = bwd_floats(a.B, a.R, a.Nk, a.Hkv, a.dh);
  LT_CHECK_ARG(need == 0 || (d->ws && aligned16(d->ws) && d->ws_floats >= need), "lt_cross_attention_bwd: a workspace of %lld floats is needed (got %lld)", (long long)need,
               (long long)(d->ws ? d->ws_floats : 0));
  const int64_t bh8 = round_up8((int64_t)a.B * a.Hkv);
  const Plan p1 = dq_plan(a.B, a.R, a.Nk, a.Hkv, a.dh), p2 = dkdv_plan(a.B, a.R, a.Nk, a.Hkv, a.dh);
  LT_CHECK_ARG(bh8 * p1.tiles * p1.splits < MAX_GROUPS && bh8 * p2.tiles * p2.splits < MAX_GROUPS, "lt_cross_attention_bwd: too many workgroups");
  if (d->dtype == LT_DT_F16) run_bwd<true>(a, d->ws, stream);
  else run_bwd<false>(a, d->ws, stream);
  LT_CHECK_LAUNCH("lt_cross_attention_bwd");
}
