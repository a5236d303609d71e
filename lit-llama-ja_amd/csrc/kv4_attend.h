// Attention over the paged 4-bit cache (layout: kv4.h): what its kernels share.
//   S_rj = scale (s_j sum_i q_ri c_ji + o_j sum_i q_ri),  y_r = sum_j p_rj (s'_j c'_j + o'_j),  p the softmax over j <= pos_r
// Codes enter the matrix products as exact small integers, made two at a time by one and-or (16 + c) and, where it costs little, one
// subtraction more (c - 8); scales and offsets are applied in fp32, to the scores and to the weights, so nothing of a key or value is rounded:
//   sum_j p s' c' = sum_j (p s') (c' + bias) - bias sum_j p s',  and sum_j p o':  two scalars a row.
// Queries: bf16 rows as they are, fp32 rows as three bf16 terms (all 24 bits).
// p is taken for a reference that is raised, kv4_slack octaves past the maximum, once a score passes it: p <= 1, and the passes over the
// accumulators that raising costs are few. Weights enter as 2^6 p s' / u with a power of two u of each column's own, up to its largest p s' when u
// was set, and raised once a weight would pass 2^15: weights of 2^-20 of the column's largest are still normal numbers. (One u from the largest s' of
// the tile lost a row its own values once a key of the tile that it does not see, or sees with p near 0, had 2^20 times their scale.) Both checks
// are made on each lane's own keys; only where one fires are the lanes of a column put together.
// fp16, whose 11 bits are 8 times finer than the output's; fp32 rows two fp16 terms, 22 bits. Where the bias is 16 its scalar sums the rounded
// weights: the roundings then weigh |c' + bias| - |bias|, not 3 times the values (0.0020 instead of 0.0017 off in the norm). fp32 rows take c - 8
// throughout.
#pragma once
#include "elem.h"
#include "kv4.h"

namespace llj {

struct Kv4Attend {
  const void* q;  // [M][ldq], head h at column h D
  const void* gate;
  int ldq, ldg;
  const int* work;  // (first row, rows, sequence) per item; NULL: item i is row i of sequence i
  int items, rows;  // rows of an item at most
  const int *pos, *slot, *table;
  int B, slots, ldt;
  Kv4Pool pool;
  void* y;
  int ldy, M, H, D, V, sink;
  float scale;
  float* part;
  int* count;
  int nsplit;
  bool quads;  // y takes 4 values at a time
};

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kFold = 8;  // steps after which the bias' share is taken out of the accumulators, so that they stay at the size of what they sum

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
__device__ __forceinline__ f32x4 mfma_f16(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// fp32 pairs as N terms of 8 (bf16) or 11 (fp16) bits
template <int N>
__device__ __forceinline__ void split_bf(float a, float b, uint32_t (&o)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    o[i] = pack2bf(a, b);
    a -= bflo(o[i]);
    b -= bfhi(o[i]);
  }
}
template <int N>
__device__ __forceinline__ void split_h(float a, float b, uint32_t (&o)[N]) {
  // The terms are of a and b as fp32 numbers. Left to see the products that they are, the compiler rounds those to fp16 a second time,
  // unrounded, for the remainder: another first term now and then, and the sum off by its last place
  if constexpr (N > 1) asm volatile("" : "+v"(a), "+v"(b));
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const f16x2 h = {(_Float16)a, (_Float16)b};
    o[i] = __builtin_bit_cast(uint32_t, h);
    if (i + 1 < N) {
      a -= (float)h[0];
      b -= (float)h[1];
    }
  }
}

// The masks and bases of the unpacking below in registers the compiler cannot see through: as literals they cost it an and and an or each,
// masks in scalar and bases in vector registers one and-or
struct Kv4Codes {
  uint32_t mask_bf, base_bf, mask_h, base_h;
};
__device__ __forceinline__ Kv4Codes kv4_codes() {
  Kv4Codes c;
  asm("s_mov_b32 %0, 0x00780078" : "=s"(c.mask_bf));
  asm("v_mov_b32 %0, 0x41804180" : "=v"(c.base_bf));
  asm("s_mov_b32 %0, 0x03C003C0" : "=s"(c.mask_h));
  asm("v_mov_b32 %0, 0x4C004C00" : "=v"(c.base_h));
  return c;
}
// A codes' word as four pairs of values (j, j + 4) in word j: 16 + c as bf16 (bits 3 .. 6 are its units from 16 on) ...
template <bool EXACT>
__device__ __forceinline__ u32x4 codes_bf(uint32_t w, const Kv4Codes& k) {
  u32x4 o = {and_or(w << 3, k.mask_bf, k.base_bf), and_or(w >> 1, k.mask_bf, k.base_bf), and_or(w >> 5, k.mask_bf, k.base_bf),
             and_or(w >> 9, k.mask_bf, k.base_bf)};
  if constexpr (EXACT) {  // c - 8
#pragma unroll
    for (int i = 0; i < 4; ++i)
      o[i] = __builtin_amdgcn_perm(__float_as_uint(bfhi(o[i]) - 24.f), __float_as_uint(bflo(o[i]) - 24.f), 0x07060302u);
  }
  return o;
}
// ... or as fp16 (bits 6 .. 9)
template <bool EXACT>
__device__ __forceinline__ u32x4 codes_h(uint32_t w, const Kv4Codes& k) {
  u32x4 o = {and_or(w << 6, k.mask_h, k.base_h), and_or(w << 2, k.mask_h, k.base_h), and_or(w >> 2, k.mask_h, k.base_h),
             and_or(w >> 6, k.mask_h, k.base_h)};
  if constexpr (EXACT) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t x = o[i];  // (a bit cast of a vector's element takes the first one)
      o[i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, x) - f16x2{24, 24});
    }
  }
  return o;
}

// A sequence's row of the table through scalar loads: page numbers are the same in all lanes, and as vector loads the move to scalar registers
// would wait, at the point of issue, for every load before them
typedef const __attribute__((address_space(4))) int* kv4_row;
__device__ __forceinline__ kv4_row scalar_row(const int* p) { return (kv4_row)(uintptr_t)p; }

// sum of an fp16 pair added to c
__device__ __forceinline__ float add_pair(uint32_t w, float c) {
  return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, w), f16x2{1, 1}, c, false);
}

// max / sum over the four 16-lane groups of the wave, lane by lane
__device__ __forceinline__ float groups_max(float v) {
  float a, b;
  lane_halves<false>(v, a, b);
  v = fmaxf(a, b);
  lane_halves<true>(v, a, b);
  return fmaxf(a, b);
}
__device__ __forceinline__ float groups_sum(float v) {
  float a, b;
  lane_halves<false>(v, a, b);
  v = a + b;
  lane_halves<true>(v, a, b);
  return a + b;
}

constexpr float kv4_slack(bool f32) { return f32 ? 2.f : 8.f; }  // (fp32 rows: differences of 8 octaves would cost a weight its last two bits)

// A column's unit u: a power of two, at least kUnitMin (the largest bf16 scale is below 2^126), and 2^6 over it
constexpr float kUnitMin = 7.5231638e-37f;  // 2^-120
constexpr float kUnitPast = 512.f;          // raised by a weight past so many of it
__device__ __forceinline__ float pow2_floor(float x) { return __uint_as_float(__float_as_uint(x) & 0x7F800000u); }
__device__ __forceinline__ float weight_unit(float x) { return __uint_as_float(0x7F000000u - __float_as_uint(x)) * 64.f; }
constexpr float kUnweight = 1.f / 64.f;
// A new unit for what is held times corr and for weights up to top; corr becomes the factor of what is held
__device__ __forceinline__ void kv4_raise(float top, float& unit, float& up, float& corr) {
  const float kept = unit * corr;
  unit = pow2_floor(fmaxf(fmaxf(kept, top), kUnitMin));
  up = weight_unit(unit);
  corr = kept * (up * kUnweight);
}

// One item's columns, (row, query head) pairs of one K / V head: column c is row c / R, head c % R
struct Kv4Columns {
  int r0, gh, R, c0, n;  // first row; K / V head; heads that share it; first column of this tile; columns
  __device__ __forceinline__ void at(int c, int& row, int& head) const {
    row = r0 + (c0 + c) / R;
    head = gh * R + (c0 + c) % R;
  }
};

// A column's result from its parts: `o` the sum of weights times values, l the sum of weights, both for the maximum m (in log2 units)
template <typename T>
__device__ __forceinline__ float kv4_factor(const Kv4Attend& p, int row, int head, float m, float l) {
  const float mu = m == -INFINITY ? 0.f : m, mt = p.sink ? fmaxf(mu, 0.f) : mu, e = __builtin_amdgcn_exp2f(mu - mt);
  l = e * l + (p.sink ? __builtin_amdgcn_exp2f(-mt) : 0.f);
  if (l == 0.f) return 0.f;  // a row that sees nothing is zero
  if (p.gate) l *= 1.f + __expf(-ldv((const T*)p.gate, (size_t)row * p.ldg + head));
  return e / l;
}
template <typename T>
__device__ __forceinline__ void kv4_store(const Kv4Attend& p, int row, int head, int v, f32x4 o) {
  T* y = (T*)p.y + (size_t)row * p.ldy + (size_t)head * p.V;
  if (p.quads) {
    if (v < p.V) {
      if constexpr (sizeof(T) == 2) *reinterpret_cast<uint2*>(y + v) = make_uint2(pack2bf(o[0], o[1]), pack2bf(o[2], o[3]));
      else *reinterpret_cast<f32x4*>(y + v) = o;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (v + i < p.V) stv(y, v + i, o[i]);
}
// The same into the partials [M][H][nsplit][VW + 4]: o, then m and l
template <int VW>
__device__ __forceinline__ float* kv4_part(const Kv4Attend& p, int row, int head, int sp) {
  return p.part + (((size_t)row * p.H + head) * p.nsplit + sp) * (VW + 4);
}

// The last of the ranges' workgroups merges them, in range order: device-scope stores, a wait for them, one device-scope counter per tile,
// device-scope loads; nobody waits for another workgroup, and the last one resets the counter. lds: 64 floats a column.
template <typename T, int VW>
__device__ void kv4_merge(const Kv4Attend& p, const Kv4Columns& cs, int ranges, int* counter, float* lds) {
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  __shared__ int last;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (tid == 0) {
    const int done = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    last = done == ranges - 1;
    if (done == ranges - 1) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!last) return;
  for (int c = wave; c < cs.n; c += 4) {  // nsplit <= 64
    int row, head;
    cs.at(c, row, head);
    const float* pr = kv4_part<VW>(p, row, head, 0);
    float2 st = make_float2(-INFINITY, 0.f);
    if (lane < ranges) st = get2(pr + (size_t)lane * (VW + 4) + VW);
    const float m = wave_max(st.x), mu = m == -INFINITY ? 0.f : m;
    const float w = __builtin_amdgcn_exp2f(st.x - mu);
    lds[c * 64 + lane] = w * kv4_factor<T>(p, row, head, m, wave_sum(w * st.y));
  }
  __syncthreads();
  for (int i = tid; i < cs.n * (VW / 4); i += 256) {
    const int c = i / (VW / 4), v = 4 * (i % (VW / 4));
    int row, head;
    cs.at(c, row, head);
    const float* pr = kv4_part<VW>(p, row, head, 0) + v;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < ranges; s += 8) {
      float2 a[8], b[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float* q = pr + (size_t)(s + e < ranges ? s + e : ranges - 1) * (VW + 4);
        a[e] = get2(q);
        b[e] = get2(q + 2);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (s + e < ranges) o += f32x4{a[e].x, a[e].y, b[e].x, b[e].y} * lds[c * 64 + s + e];
    }
    kv4_store<T>(p, row, head, v, o);
  }
}

// A column's query in the order of a key's words (lane (., g): words KT g .. KT g + KT - 1), as NQ bf16 terms; returns the sum of its values
template <typename T, int KT, int NQ>
__device__ __forceinline__ float kv4_query(const Kv4Attend& p, int row, int head, int g, u32x4 (&qf)[NQ][KT]) {
  const T* qr = (const T*)p.q + (size_t)row * p.ldq + (size_t)head * p.D;
  const bool whole = p.D % 8 == 0 && (((uintptr_t)p.q | ((size_t)p.ldq * sizeof(T))) & 15) == 0;
  const float sign = p.scale < 0.f ? -1.f : 1.f;  // scores stay in units of q . k until the softmax: a negative scale turns the query round
  float qs = 0.f;
#pragma unroll
  for (int kk = 0; kk < KT; ++kk) {
    const int d = 8 * (KT * g + kk);
    float x[8];
    if (whole) {
      if (d < p.D) ld8(qr + d, x);
      else
        for (int e = 0; e < 8; ++e) x[e] = 0.f;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = d + e < p.D ? ldv(qr, d + e) : 0.f;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[e] *= sign;
      qs += x[e];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      uint32_t t[NQ];
      split_bf<NQ>(x[e], x[e + 4], t);
#pragma unroll
      for (int i = 0; i < NQ; ++i) qf[i][kk][e] = t[i];
    }
  }
  return groups_sum(qs);
}

// scale in units of log2 (the query took its sign; never 0, which an infinite difference would make NaN)
__device__ __forceinline__ float kv4_scale(const Kv4Attend& p) { return fmaxf(fabsf(p.scale) * kLog2e, 1e-30f); }

// Scores of 4 keys in units of q . k from their product `a` (codes c - 8; else 16 + c, begun at -16 qs, so that it is q . c), their scales and
// offsets (codes c - 8: of + 8 sc)
__device__ __forceinline__ f32x4 kv4_scores(f32x4 a, f32x4 sc, f32x4 of, float qs) {
  f32x4 s;
#pragma unroll
  for (int i = 0; i < 4; ++i) s[i] = fmaf(sc[i], a[i], of[i] * qs);
  return s;
}
// exp2(sl2 (s - mu)). fp32 rows: from the difference, which keeps the top's neighbours exact; bf16 rows: one fma from ms = sl2 mu, whose rounding
// is common to a row's weights
template <bool F32>
__device__ __forceinline__ float kv4_weight(float s, float mu, float ms, float sl2) {
  return __builtin_amdgcn_exp2f(F32 ? (s - mu) * sl2 : fmaf(s, sl2, -ms));
}

// prompt rows; and the column tiles it cuts an item of so many columns into
int kv4_flash(const Kv4Attend& p, int dt, hipStream_t s);
int kv4_flash_tiles(int columns, int D, int V, int dt);

}  // namespace llj
