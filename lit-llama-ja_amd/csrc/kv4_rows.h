// A vector's codes, scale and offset into the paged 4-bit cache (layout and rounding: kv4.h).
#pragma once
#include "elem.h"
#include "kv4.h"

namespace llj {

struct Kv4Part {  // keys or values of a block
  int n, codes, pairs, bytes;  // values a vector; in a block: the codes, the pairs; bytes of codes a token
};
__host__ __device__ inline Kv4Part kv4_keys(const Kv4Pool& p, int D) { return Kv4Part{D, 0, p.ks, kv4_width(D) / 2}; }
__host__ __device__ inline Kv4Part kv4_values(const Kv4Pool& p, int V) { return Kv4Part{V, p.vc, p.vs, kv4_width(V) / 2}; }

// Reductions over the LG lanes of a vector; every lane ends with the result
template <int LG, typename F>
__device__ __forceinline__ float group_all(float v, F f) {
  v = f(v, dpp_f32<kDppXor1>(v));
  v = f(v, dpp_f32<kDppXor2>(v));
  v = f(v, dpp_f32<kDppHalfMirror>(v));
  if constexpr (LG >= 16) v = f(v, dpp_f32<kDppRowMirror>(v));
  if constexpr (LG >= 32) {
    float lo, hi;
    lane_halves<false>(v, lo, hi);
    v = f(lo, hi);
  }
  return v;
}

// the largest bf16 up to x (finite), as its bits
__device__ __forceinline__ uint32_t floor_bf(float x) {
  const uint32_t u = __float_as_uint(x);
  return (u >> 31) && (u & 0xFFFF) ? (u >> 16) + 1 : u >> 16;
}

// block and token of a row; null where it has no place in the pool
__device__ __forceinline__ uint8_t* kv4_block_of(const Kv4Pool& p, int place, int g, int& t) {
  const int page = place >> p.k;
  t = place & ((1 << p.k) - 1);
  if (place < 0 || page >= p.pages) return nullptr;
  return p.p + ((size_t)page * p.G + g) * p.blk;
}

// The codes need the quotient's exact rounding (bf16 values on a grid of bf16 steps are on a border between two codes about once in 300). u = (x - o) / s
// by an approximate reciprocal settles all values but those near a border. There, in a branch: t = x - o, n = rint(u), rem = t - n s (exact: a
// multiple of t's last place below s); n moves by one where |rem| is over half a step, and on the border itself by the rest that t was rounded by,
// then by n's parity. (32,768 rows of 8 heads of 128, before rows were taken four at a time: doubles throughout 93 us, this for every value 70.)
// One vector of n values: values 8 l .. 8 l + 7 in lane l of its LG, whose codes take 4 LG bytes a token (VEC: n is a multiple of 8)
template <int LG, bool VEC>
__device__ __forceinline__ void kv4_write_row(const Kv4Pool& pool, const Kv4Part& r, const float (&v)[8], int l, int place, int g) {
  int t;
  uint8_t* blk = kv4_block_of(pool, place, g, t);
  if (!blk) return;  // (whole groups: the moves below stay inside one)
  float lo = INFINITY, hi = -INFINITY, odd = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (VEC ? 8 * l < r.n : 8 * l + e < r.n) {
      lo = fminf(lo, v[e]);
      hi = fmaxf(hi, v[e]);
      odd = fmaf(v[e], 0.f, odd);  // NaN once a value is not finite
    }
  odd = odd == 0.f ? 0.f : 1.f;
  lo = group_all<LG>(lo, [](float a, float b) { return fminf(a, b); });
  hi = group_all<LG>(hi, [](float a, float b) { return fmaxf(a, b); });
  odd = group_all<LG>(odd, [](float a, float b) { return fmaxf(a, b); });
  const uint32_t ob = floor_bf(lo);
  const float o = __uint_as_float(ob << 16);
  // (hi - o) / 15 in double: the product with 1 / 15, corrected by its remainder
  const double span = (double)hi - (double)o, q = span * (1.0 / 15.0);
  const uint32_t sb = f2bf((float)fma(fma(-15.0, q, span), 1.0 / 15.0, q));
  const bool none = odd != 0.f || (ob & 0x7F80) == 0x7F80;
  const float s0 = __uint_as_float(sb << 16);
  uint32_t w = 0;
  if (!none && s0 > 0.f && 8 * l < r.n) {
    // tiny steps as 2^100 of them, so that the reciprocal is a number; exact
    const float up = s0 < 7.8886e-31f ? 1.2676506e30f : 1.f, s = s0 * up, os = o * up, inv = __builtin_amdgcn_rcpf(s), half = 0.5f * s;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float d = fmaf(v[e], up, -os), u = d * inv;
      float n = rintf(u);
      if (fabsf(u - n) > 0.5f - 0x1p-17f) {  // (u, below 16, is off by 2^-18 at most)
        const float rem = fmaf(-n, s, d), over = fabsf(rem) - half;
        const float xs = v[e] * up, bb = d - xs, rest = (xs - (d - bb)) - (os + bb);  // d + rest = x - o
        const bool move = over != 0.f ? over > 0.f : rest != 0.f ? (rest > 0.f) == (rem > 0.f) : ((int)n & 1) != 0;
        n += move ? copysignf(1.f, rem) : 0.f;
      }
      const int c = (int)fminf(fmaxf(n, 0.f), 15.f);
      if (VEC || 8 * l + e < r.n) w |= (uint32_t)c << (4 * e);
    }
  }
  if (4 * l < r.bytes) *reinterpret_cast<uint32_t*>(blk + r.codes + t * r.bytes + 4 * l) = w;
  if (l == 0) *reinterpret_cast<uint32_t*>(blk + r.pairs + 4 * t) = none ? 0x7FC07FC0u : (sb | ob << 16);
}

}  // namespace llj
