// Rows into the paged 4-bit cache and out of it (layout and rounding: kv4.h). LG lanes hold a vector, 8 values each: its minimum and maximum
// over the lanes, then a word of codes per lane. Both directions move each byte once and are bound by memory at many rows, by the launch at few.
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

// block and token of vector i of part w (i = row * heads + head); null where the row has no place in the pool
__device__ __forceinline__ uint8_t* block_of(const Kv4IO& io, long long i, long long& m, int& g, int& t) {
  m = i / io.pool.G;
  g = (int)(i - m * io.pool.G);
  const int place = io.place[m], page = place >> io.pool.k;
  t = place & ((1 << io.pool.k) - 1);
  if (place < 0 || page >= io.pool.pages) return nullptr;
  return io.pool.p + ((size_t)page * io.pool.G + g) * io.pool.blk;
}

// The codes need the quotient's exact rounding (values on a border are common: bf16 values on a grid of bf16 steps), so the
// difference and the remainder are formed in double: n = rint(t / s) by a reciprocal, then t - n s against half a step.
template <typename T, int LG, bool VEC>
__global__ __launch_bounds__(256) void kv4_write_kernel(Kv4IO io, int first) {
  const Kv4Rows& r = io.part[first + blockIdx.y];
  const int l = threadIdx.x & (LG - 1);
  const long long i = ((long long)blockIdx.x * 256 + threadIdx.x) / LG;
  if (i >= (long long)io.M * io.pool.G) return;  // (whole groups: the moves below stay inside one)
  long long m;
  int g, t;
  uint8_t* blk = block_of(io, i, m, g, t);
  if (!blk) return;
  const T* x = (const T*)r.x + m * r.ld + g * r.hs;
  float v[8];
  if constexpr (VEC) {
    if (8 * l < r.n) ld8(x + 8 * l, v);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 8 * l + e < r.n ? ldv(x, 8 * l + e) : 0.f;
  }
  float lo = INFINITY, hi = -INFINITY, odd = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (8 * l + e < r.n) {
      lo = fminf(lo, v[e]);
      hi = fmaxf(hi, v[e]);
      odd = fabsf(v[e]) < INFINITY ? odd : 1.f;
    }
  lo = group_all<LG>(lo, [](float a, float b) { return fminf(a, b); });
  hi = group_all<LG>(hi, [](float a, float b) { return fmaxf(a, b); });
  odd = group_all<LG>(odd, [](float a, float b) { return fmaxf(a, b); });
  const uint32_t ob = floor_bf(lo);
  const double o = (double)__uint_as_float(ob << 16);
  const uint32_t sb = f2bf((float)(((double)hi - o) / 15.0));
  const bool none = odd != 0.f || (ob & 0x7F80) == 0x7F80;
  const double s = (double)__uint_as_float(sb << 16), inv = 1.0 / s, half = 0.5 * s;
  uint32_t w = 0;
  if (!none && s > 0.0) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const double d = (double)v[e] - o;
      double n = rint(d * inv);
      const double rem = fma(-n, s, d);
      int c = (int)n;
      if (rem > half || (rem == half && (c & 1))) ++c;
      else if (rem < -half || (rem == -half && (c & 1))) --c;
      c = c < 0 ? 0 : c > 15 ? 15 : c;
      if (8 * l + e < r.n) w |= (uint32_t)c << (4 * e);
    }
  }
  if (4 * l < r.bytes) *reinterpret_cast<uint32_t*>(blk + r.codes + t * r.bytes + 4 * l) = w;
  if (l == 0) *reinterpret_cast<uint32_t*>(blk + r.pairs + 4 * t) = none ? 0x7FC07FC0u : (sb | ob << 16);
}

template <typename T, int LG, bool VEC>
__global__ __launch_bounds__(256) void kv4_read_kernel(Kv4IO io, int first) {
  const Kv4Rows& r = io.part[first + blockIdx.y];
  const int l = threadIdx.x & (LG - 1);
  const long long i = ((long long)blockIdx.x * 256 + threadIdx.x) / LG;
  if (i >= (long long)io.M * io.pool.G || 8 * l >= r.n) return;
  long long m;
  int g, t;
  const uint8_t* blk = block_of(io, i, m, g, t);
  T* x = (T*)r.x + m * r.ld + g * r.hs;
  const uint32_t w = blk ? *reinterpret_cast<const uint32_t*>(blk + r.codes + t * r.bytes + 4 * l) : 0;
  const uint32_t so = blk ? *reinterpret_cast<const uint32_t*>(blk + r.pairs + 4 * t) : 0;
  float v[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = fmaf((float)((w >> (4 * e)) & 15), bflo(so), bfhi(so));
  if constexpr (VEC) {
    st8(x + 8 * l, v);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (8 * l + e < r.n) stv(x, 8 * l + e, v[e]);
  }
}

template <typename T, int LG, bool WRITE>
static void kv4_io_launch(const Kv4IO& io, int first, int parts, bool vec, hipStream_t s) {
  const long long n = (long long)io.M * io.pool.G, per = 256 / LG;
  const dim3 grid((unsigned)((n + per - 1) / per), parts);
  if constexpr (WRITE) {
    if (vec) hipLaunchKernelGGL((kv4_write_kernel<T, LG, true>), grid, dim3(256), 0, s, io, first);
    else hipLaunchKernelGGL((kv4_write_kernel<T, LG, false>), grid, dim3(256), 0, s, io, first);
  } else {
    if (vec) hipLaunchKernelGGL((kv4_read_kernel<T, LG, true>), grid, dim3(256), 0, s, io, first);
    else hipLaunchKernelGGL((kv4_read_kernel<T, LG, false>), grid, dim3(256), 0, s, io, first);
  }
}

template <bool WRITE>
static int kv4_io(void* pool, int pages, int page, int G, void* k, size_t ldk, size_t hk, void* v, size_t ldv, size_t hv, const int* place,
                  int M, int D, int V, int dt, void* stream) {
  LLJ_REQUIRE(kv4_sizes(pool, pages, page, G, D, V, dt) && k && v && place && M >= 0 && ((ldk | hk | ldv | hv) >> 40) == 0 &&
              (long long)M * G <= 1LL << 33);
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
