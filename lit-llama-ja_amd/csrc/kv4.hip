// Rows into the paged 4-bit cache and out of it (layout and rounding: kv4.h). LG lanes hold a vector, 8 values each: its minimum and maximum
// over the lanes, then a word of codes per lane. Both directions move each byte once and are bound by memory at many rows, by the launch at few:
// 32,768 rows of 8 heads of 128 in bf16 58 us (171 MB, 2.9 TB/s, beside the codes' arithmetic), out of it into fp32 48 us (304 MB, 6.3 TB/s);
// 8 rows 3.3 and 2.6 us.
#include "kv4_rows.h"
#include "lit_llama_amd.h"

namespace llj {

struct Kv4Rows {  // keys or values: rows of stride ld, heads of stride hs
  void* x;
  size_t ld, hs;
  Kv4Part to;
};

struct Kv4IO {
  Kv4Rows part[2];
  Kv4Pool pool;
  const int* place;
  int M;
};

// A workgroup's rows m0 .. and its head: consecutive rows of one head, whose codes lie one after another in its block, heads side by side in the grid
template <int LG, int N>
__device__ __forceinline__ long long first_row(const Kv4IO& io, int& g) {
  g = blockIdx.x % io.pool.G;
  return (long long)(blockIdx.x / io.pool.G) * (256 / LG * N) + threadIdx.x / LG;
}
// N rows a group, all of them on their way before the first is worked on (one at a time, place before row: 70 us for 32,768 rows).
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
      ld8(x + (8 * l < r.to.n ? 8 * l : 0), v[i]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[i][e] = 8 * l + e < r.to.n ? ldv(x, 8 * l + e) : 0.f;
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) kv4_write_row<LG, VEC>(io.pool, r.to, v[i], l, place[i], g);
}

template <typename T, int LG, bool VEC, int N>
__global__ __launch_bounds__(256) void kv4_read_kernel(Kv4IO io, int first) {
  const Kv4Rows& r = io.part[first + blockIdx.y];
  const int l = threadIdx.x & (LG - 1);
  int g;
  const long long m0 = first_row<LG, N>(io, g);
  if (8 * l >= r.to.n) return;
  uint32_t w[N], so[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const long long m = m0 + i * (256 / LG);
    int t;
    const uint8_t* blk = kv4_block_of(io.pool, m < io.M ? io.place[m] : -1, g, t);
    w[i] = blk ? *reinterpret_cast<const uint32_t*>(blk + r.to.codes + t * r.to.bytes + 4 * l) : 0;
    so[i] = blk ? *reinterpret_cast<const uint32_t*>(blk + r.to.pairs + 4 * t) : 0;
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
        if (8 * l + e < r.to.n) stv(x, 8 * l + e, v[e]);
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
  io.part[0] = Kv4Rows{k, ldk, hk, kv4_keys(io.pool, D)};
  io.part[1] = Kv4Rows{v, ldv, hv, kv4_values(io.pool, V)};
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
