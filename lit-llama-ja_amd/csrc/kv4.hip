// Rows into the paged 4-bit cache and out of it (layout and rounding: kv4.h). LG lanes hold a vector, 8 values each: its minimum and maximum
// over the lanes, then a word of codes per lane. Both directions move each byte once and are bound by memory at many rows, by the launch at few:
// 32,768 rows of 8 heads of 128 in bf16 58 us (171 MB, 2.9 TB/s, beside the codes' arithmetic), out of it into fp32 48 us (304 MB, 6.3 TB/s);
// 8 rows 3.3 and 2.6 us.
#include "kv4.h"
#include "elem.h"
#include "lit_llama_amd.h"

namespace llj {

struct Kv4Rows {  // keys or values: rows of stride ld, heads of stride hs
  void* x;
  size_t ld, hs;
  int n, codes, pairs, bytes;  // values a vector; in a block: the codes, the pairs; bytes of codes a token
};

struct Kv4IO {
  Kv4Rows part[2];
  Kv4Pool pool;
  const int* place;
  int M;
};

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

// A workgroup's rows m0 .. and its head: consecutive rows of one head, whose codes lie one after another in its block, heads side by side in the grid
template <int LG, int N>
__device__ __forceinline__ long long first_row(const Kv4IO& io, int& g) {
  g = blockIdx.x % io.pool.G;
  return (long long)(blockIdx.x / io.pool.G) * (256 / LG * N) + threadIdx.x / LG;
}
// block and token of a row; null where it has no place in the pool
__device__ __forceinline__ uint8_t* block_of(const Kv4IO& io, int place, int g, int& t) {
  const int page = place >> io.pool.k;
  t = place & ((1 << io.pool.k) - 1);
  if (place < 0 || page >= io.pool.pages) return nullptr;
  return io.pool.p + ((size_t)page * io.pool.G + g) * io.pool.blk;
}

// The codes need the quotient's exact rounding (bf16 values on a grid of bf16 steps are on a border between two codes about once in 300). u = (x - o) / s
// by an approximate reciprocal settles all values but those near a border. There, in a branch: t = x - o, n = rint(u), rem = t - n s (exact: a
// multiple of t's last place below s); n moves by one where |rem| is over half a step, and on the border itself by the rest that t was rounded by,
// then by n's parity. (32,768 rows of 8 heads of 128, before rows were taken four at a time: doubles throughout 93 us, this for every value 70.)
// N rows a group, all of them on their way before the first is worked on (one at a time, place before row: 70 us for 32,768 rows).
template <typename T, int LG, bool VEC>
__device__ __forceinline__ void kv4_write_row(const Kv4IO& io, const Kv4Rows& r, const float (&v)[8], int l, int place, int g) {
  int t;
  uint8_t* blk = block_of(io, place, g, t);
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

template <typename T, int LG, bool VEC, int N>
__global__ __launch_bounds__(256) void kv4_write_kernel(Kv4IO io, int first) {
  const Kv4Rows& r = io.part[first + blockIdx.y];
  const int l = threadIdx.x & (LG - 1);
  int g;
  const long long m0 = first_row<LG, N>(io, g);
  float v[N][8];
  int place[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const long long m = m0 + i * (256 / LG);
    place[i] = m < io.M ? io.place[m] : -1;
    const T* x = (const T*)r.x + (m < io.M ? m : 0) * r.ld + g * r.hs;
    if constexpr (VEC) {
      ld8(x + (8 * l < r.n ? 8 * l : 0), v[i]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[i][e] = 8 * l + e < r.n ? ldv(x, 8 * l + e) : 0.f;
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) kv4_write_row<T, LG, VEC>(io, r, v[i], l, place[i], g);
}

template <typename T, int LG, bool VEC, int N>
__global__ __launch_bounds__(256) void kv4_read_kernel(Kv4IO io, int first) {
  const Kv4Rows& r = io.part[first + blockIdx.y];
  const int l = threadIdx.x & (LG - 1);
  int g;
  const long long m0 = first_row<LG, N>(io, g);
  if (8 * l >= r.n) return;
  uint32_t w[N], so[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const long long m = m0 + i * (256 / LG);
    int t;
    const uint8_t* blk = block_of(io, m < io.M ? io.place[m] : -1, g, t);
    w[i] = blk ? *reinterpret_cast<const uint32_t*>(blk + r.codes + t * r.bytes + 4 * l) : 0;
    so[i] = blk ? *reinterpret_cast<const uint32_t*>(blk + r.pairs + 4 * t) : 0;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const long long m = m0 + i * (256 / LG);
    if (m >= io.M) return;
    T* x = (T*)r.x + m * r.ld + g * r.hs;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = fmaf((float)((w[i] >> (4 * e)) & 15), bflo(so[i]), bfhi(so[i]));
    if constexpr (VEC) {
      st8(x + 8 * l, v);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (8 * l + e < r.n) stv(x, 8 * l + e, v[e]);
    }
  }
}

template <typename T, int LG, bool VEC, int N, bool WRITE>
static void kv4_io_go(const Kv4IO& io, int first, int parts, hipStream_t s) {
  const long long per = 256 / LG * N;
  const dim3 grid((unsigned)((io.M + per - 1) / per * io.pool.G), parts);
  if constexpr (WRITE) hipLaunchKernelGGL((kv4_write_kernel<T, LG, VEC, N>), grid, dim3(256), 0, s, io, first);
  else hipLaunchKernelGGL((kv4_read_kernel<T, LG, VEC, N>), grid, dim3(256), 0, s, io, first);
}

template <typename T, int LG, bool WRITE>
static void kv4_io_launch(const Kv4IO& io, int first, int parts, bool vec, hipStream_t s) {
  // four rows a group once that leaves 2,048 workgroups, eight on a CU
  const bool many = (long long)io.M * io.pool.G * parts >= 2048LL * 4 * (256 / LG);
  if (vec && many) kv4_io_go<T, LG, true, 4, WRITE>(io, first, parts, s);
  else if (vec) kv4_io_go<T, LG, true, 1, WRITE>(io, first, parts, s);
  else kv4_io_go<T, LG, false, 1, WRITE>(io, first, parts, s);
}

template <bool WRITE>
static int kv4_io(void* pool, int pages, int page, int G, void* k, size_t ldk, size_t hk, void* v, size_t ldv, size_t hv, const int* place,
                  int M, int D, int V, int dt, void* stream) {
  LLJ_REQUIRE(kv4_sizes(pool, pages, page, G, D, V, dt) && k && v && place && M >= 0 && ((ldk | hk | ldv | hv) >> 40) == 0 &&
              (long long)M * G <= 1 << 26);  // (a grid's threads stay below 2^32)
  if (M == 0) return 0;
  Kv4IO io{};
  io.pool = kv4_pool(pool, pages, G, kv4_page_log2(page), D, V);
  io.place = place;
  io.M = M;
  io.part[0] = Kv4Rows{k, ldk, hk, D, 0, io.pool.ks, kv4_width(D) / 2};
  io.part[1] = Kv4Rows{v, ldv, hv, V, io.pool.vc, io.pool.vs, kv4_width(V) / 2};
  // 16-byte pieces: 8 values in bf16, two pieces of 4 in fp32
  const uintptr_t at = (uintptr_t)k | (uintptr_t)v;
  const bool vec = (at & 15) == 0 && ((ldk | hk | ldv | hv) & (dt ? 3 : 7)) == 0 && (D | V) % 8 == 0;
  hipStream_t s = (hipStream_t)stream;
  const int Dp = kv4_width(D), Vp = kv4_width(V);
#define LLJ_KV4(P, FIRST, N)                                                                            \
  do {                                                                                                  \
    if (dt == 0) {                                                                                      \
      if (P == 64) kv4_io_launch<bf16_t, 8, WRITE>(io, FIRST, N, vec, s);                               \
      else if (P == 128) kv4_io_launch<bf16_t, 16, WRITE>(io, FIRST, N, vec, s);                        \
      else kv4_io_launch<bf16_t, 32, WRITE>(io, FIRST, N, vec, s);                                      \
    } else {                                                                                            \
      if (P == 64) kv4_io_launch<float, 8, WRITE>(io, FIRST, N, vec, s);                                \
      else if (P == 128) kv4_io_launch<float, 16, WRITE>(io, FIRST, N, vec, s);                         \
      else kv4_io_launch<float, 32, WRITE>(io, FIRST, N, vec, s);                                       \
    }                                                                                                   \
  } while (0)
  if (Dp == Vp) {
    LLJ_KV4(Dp, 0, 2);
  } else {
    LLJ_KV4(Dp, 0, 1);
    LLJ_KV4(Vp, 1, 1);
  }
#undef LLJ_KV4
  LLJ_CHECK_LAUNCH();
  return 0;
}

}  // namespace llj

using namespace llj;

extern "C" {

size_t llj_kv4_block_bytes(int page, int dim, int vdim) {
  return kv4_page_log2(page) && dim >= 1 && dim <= 256 && vdim >= 1 && vdim <= 256 ? (size_t)kv4_block(page, kv4_width(dim), kv4_width(vdim)) : 0;
}

int llj_kv4_write(const void* k, size_t ldk, size_t hk, const void* v, size_t ldv, size_t hv, const int* place, int M, int kv_heads, int dim,
                  int vdim, int dt, void* pool, int pages, int page, void* stream) {
  return kv4_io<true>(pool, pages, page, kv_heads, (void*)k, ldk, hk, (void*)v, ldv, hv, place, M, dim, vdim, dt, stream);
}

int llj_kv4_read(const void* pool, int pages, int page, const int* place, int M, int kv_heads, int dim, int vdim, int dt, void* k, size_t ldk,
                 size_t hk, void* v, size_t ldv, size_t hv, void* stream) {
  return kv4_io<false>((void*)pool, pages, page, kv_heads, k, ldk, hk, v, ldv, hv, place, M, dim, vdim, dt, stream);
}

}  // extern "C"
