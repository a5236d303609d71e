// Attention of prompt rows over the paged 4-bit cache (mathematics: kv4_attend.h).
//
// One workgroup per (item, K / V head, key range): the item's columns, (row, query head) pairs, 16 QB to a wave, so a tile of keys and values is
// taken out of its codes once for up to 64 QB columns. Tiles of 64 keys: each wave fetches and unpacks 16 of them, into the order in which
// the product's operands are read (16 bytes a lane, no bank conflicts on reading), two buffers, so that the next tile's codes are in flight over
// this one's products and one barrier a tile is enough. Scores, softmax and weights stay in registers: S^T = K q^T leaves a
// column's weights where O^T = V^T P^T wants them. Workgroups of one head are 8 apart and so on one XCD, whose L2 holds its pages; items
// are taken from the last, which see the most keys.
// Measured, 32 heads on 8, 128 wide: 4,096 rows 216 us, 137 GFLOP of products in 64-key tiles at 0.64 PFLOP/s (a library's bf16 product: 1.17).
// Instructions of the vector units keep them busy 72 % of the time (softmax 150 a tile and 16 columns, unpacking 110 a tile and wave, at four cycles
// each), products a quarter; at 32 columns a wave the rest is LDS and barriers. (16 columns a wave and 8 waves, twice the waves on a CU but
// twice the fragments read: 406 us.) Short prompts are bound by their longest item, 1.6 us a tile alone: six of up to 501 rows, 10 heads of 64 in
// fp32, 23 us.
#include <type_traits>

#include "kv4_attend.h"
#include "lit_llama_amd.h"

namespace llj {

template <int KT, int VH>
struct Kv4Tile {
  static constexpr int kKeys = 4 * KT * 1024, kValues = 8 * VH * 1024;  // bytes of unpacked keys, values
  // pairs: key scales, offsets, value scales, offsets as fp32; here: whether the pages of each 16 keys exist
  static constexpr int kPairs = kKeys + kValues, kHere = kPairs + 1024, kBytes = kHere + 16;
};

template <typename T, int KT, int VH, int QB>
__global__ __launch_bounds__(256, KT <= 4 && VH <= 2 ? 2 : 1) void kv4_flash_kernel(Kv4Attend p) {
  constexpr bool F32 = sizeof(T) == 4;
  constexpr int NQ = F32 ? 3 : 1, NP = F32 ? 2 : 1;
  constexpr int KB = 16 * KT, VB = 32 * VH, VW = 64 * VH, VD = VH >= 2 ? VH / 2 : 1;
  typedef Kv4Tile<KT, VH> Tile;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];  // two tiles
  const Kv4Codes codes = kv4_codes();
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), col = lane & 15, g = lane >> 4;
  constexpr int CW = 64 * QB;  // columns
  const int R = p.H / p.pool.G, CB = (p.rows * R + CW - 1) / CW, x = p.items * CB - 1 - blockIdx.x / p.pool.G;
  const int gh = blockIdx.x % p.pool.G, item = x / CB, cb = x % CB, sp = blockIdx.y;
  int r0 = item, n = 1, b = item;
  if (p.work) {
    r0 = p.work[3 * (size_t)item];
    n = p.work[3 * (size_t)item + 1];
    b = p.work[3 * (size_t)item + 2];
  }
  n = n < p.rows ? n : p.rows;
  if (n <= 0 || r0 < 0 || r0 > p.M - n || b < 0 || b >= p.B) return;  // (uniform; no such rows)
  const Kv4Columns cols{r0, gh, R, cb * CW, n * R - cb * CW < CW ? n * R - cb * CW : CW};
  if (cols.n <= 0) return;
  const int sl = p.slot[b];
  const bool held = sl >= 0 && sl < p.slots;
  // (page numbers are loaded into vector registers and moved to scalar ones a tile later: a move at the load would wait for it)
  const int* tab = p.table + (size_t)(held ? sl : 0) * p.ldt + vzero();
  const int k = p.pool.k, pmask = (1 << k) - 1, most = held ? (p.ldt << k) - 1 : -1;
  // the last position any column sees (a lane a column)
  int plast = -1;
  for (int i = lane; i < cols.n; i += 64) {
    const int o = p.pos[r0 + (cols.c0 + i) / R];
    plast = o > plast ? o : plast;
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int o = __shfl_xor(plast, d, 64);
    plast = o > plast ? o : plast;
  }
  plast = uniform(plast < most ? plast : most);
  const int tiles = plast < 0 ? 0 : plast / 64 + 1, per = (tiles + p.nsplit - 1) / p.nsplit;
  const int t0 = sp * per, t1 = t0 + per < tiles ? t0 + per : tiles;

  // ---- this wave's columns
  int row[QB], head[QB], pc[QB], wfirst = 0x7fffffff;
  u32x4 qf[QB][NQ][KT];
  float qs[QB], qi[QB];
  const float sl2 = kv4_scale(p), slack = kv4_slack(F32) / sl2;
#pragma unroll
  for (int q = 0; q < QB; ++q) {
    const int c = (wave * QB + q) * 16 + col;
    cols.at(c < cols.n ? c : cols.n - 1, row[q], head[q]);
    pc[q] = p.pos[row[q]];
    pc[q] = pc[q] < most ? pc[q] : most;
    wfirst = pc[q] < wfirst ? pc[q] : wfirst;
    qs[q] = kv4_query<T, KT, NQ>(p, row[q], head[q], g, qf[q]);
    qi[q] = F32 ? 0.f : -16.f * qs[q];
  }
#pragma unroll
  for (int d = 1; d < 16; d <<= 1) {
    const int f = __shfl_xor(wfirst, d, 64);
    wfirst = f < wfirst ? f : wfirst;
  }
  wfirst = uniform(wfirst);

  // ---- a tile's codes: this wave's 16 keys of it
  uint32_t kw[KT], vw[4][VD], pair;
  bool ok = false, there = false;
  auto page_of = [&](int t) {
    const int at = (64 * t + 16 * wave) >> k;
    return tab[at < p.ldt ? at : p.ldt - 1];
  };
  auto fetch = [&](int t, int id) {
    ok = id >= 0 && id < p.pool.pages;
    const int off = (64 * t + 16 * wave) & pmask;
    const uint8_t* blk = p.pool.p + ((size_t)(ok ? id : 0) * p.pool.G + gh) * p.pool.blk;
    const uint8_t* ka = blk + (off + col) * KB + 4 * KT * g;
    if constexpr (KT == 2) {
      const uint2 x = *reinterpret_cast<const uint2*>(ka);
      kw[0] = x.x;
      kw[1] = x.y;
    } else {
#pragma unroll
      for (int i = 0; i < KT / 4; ++i) {
        const u32x4 x = *reinterpret_cast<const u32x4*>(ka + 16 * i);
#pragma unroll
        for (int e = 0; e < 4; ++e) kw[4 * i + e] = x[e];
      }
    }
    const uint8_t* va = blk + p.pool.vc + (off + 4 * g) * VB + 2 * VH * col;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (VH == 1) {
        vw[i][0] = *reinterpret_cast<const uint16_t*>(va + i * VB);
      } else if constexpr (VH == 2) {
        vw[i][0] = *reinterpret_cast<const uint32_t*>(va + i * VB);
      } else {
        const uint2 x = *reinterpret_cast<const uint2*>(va + i * VB);
        vw[i][0] = x.x;
        vw[i][1] = x.y;
      }
    }
    pair = *reinterpret_cast<const uint32_t*>(blk + (lane & 16 ? p.pool.vs : p.pool.ks) + 4 * (off + col));
    there = ok && 64 * t + 16 * wave + col <= plast;  // (behind the last row's position stands anything; the pair itself is on its way)
  };
  auto unpack = [&](uint8_t* buf) {
#pragma unroll
    for (int kk = 0; kk < KT; ++kk) *reinterpret_cast<u32x4*>(buf + (kk * 4 + wave) * 1024 + lane * 16) = codes_bf<F32>(kw[kk], codes);
    uint8_t* vb = buf + Tile::kKeys + (wave >> 1) * 4 * VH * 1024 + lane * 16 + 8 * (wave & 1);
#pragma unroll
    for (int v = 0; v < VH; ++v) {
      uint32_t x[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        if constexpr (VH == 1) x[e] = vw[2 * e][0] | vw[2 * e + 1][0] << 16;
        else x[e] = __builtin_amdgcn_perm(vw[2 * e + 1][v / 2], vw[2 * e][v / 2], v % 2 ? 0x07060302u : 0x05040100u);
      }
      const u32x4 a = codes_h<true>(x[0], codes), c = codes_h<true>(x[1], codes);
#pragma unroll
      for (int d = 0; d < 4; ++d) *reinterpret_cast<uint2*>(vb + (4 * v + d) * 1024) = make_uint2(a[d], c[d]);
    }
    const uint32_t so = there ? pair : 0;
    const float sc = bflo(so), of = bfhi(so) + (F32 || lane & 16 ? 8.f * sc : 0.f);  // (codes c - 8)
    float* at = reinterpret_cast<float*>(buf + Tile::kPairs + (lane & 16) * 32) + wave * 16 + col;  // (lanes 32 .. 63 write the same)
    at[0] = sc;
    at[64] = of;
    if (lane == 0) *reinterpret_cast<float*>(buf + Tile::kHere + 4 * wave) = ok ? 1.f : -1.f;
  };

  float m_run[QB], l_run[QB], z_run[QB], unit[QB], up[QB];
  f32x4 acc[QB][4 * VH];
#pragma unroll
  for (int q = 0; q < QB; ++q) {
    m_run[q] = -INFINITY;
    l_run[q] = z_run[q] = 0.f;
    unit[q] = kUnitMin;
    up[q] = weight_unit(kUnitMin);
#pragma unroll
    for (int d = 0; d < 4 * VH; ++d) acc[q][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  // Tile t is multiplied while tile t + 1 goes from registers to LDS, between the first products, and tile t + 2 is on its way to registers
  int next = 0;
  auto last = [&](int t) { return t < t1 ? t : t1 - 1; };
  if (t0 < t1) {
    fetch(t0, uniform(page_of(t0)));
    next = page_of(last(t0 + 1));
    unpack(lds);
    fetch(last(t0 + 1), uniform(next));
    next = page_of(last(t0 + 2));
  }
  __syncthreads();
  for (int t = t0; t < t1; ++t) {
    const uint8_t* buf = lds + ((t - t0) & 1) * Tile::kBytes;
    uint8_t* then = lds + ((t + 1 - t0) & 1) * Tile::kBytes;  // (its last readers passed the barrier before this tile)
    f32x4 s[QB][4];
#pragma unroll
    for (int q = 0; q < QB; ++q)
#pragma unroll
      for (int j = 0; j < 4; ++j) s[q][j] = f32x4{qi[q], qi[q], qi[q], qi[q]};
    // Operands are read ahead of their products, fences keep the compiler from reading each right before its use (which left the LDS latency
    // open 30 times a tile)
    u32x4 a[2][8];
    f32x4 sc[4], of[4];
    const f32x4* pairs = reinterpret_cast<const f32x4*>(buf + Tile::kPairs) + g;
    auto keys = [&](int c) {
#pragma unroll
      for (int i = 0; i < 8; ++i) a[c & 1][i] = *reinterpret_cast<const u32x4*>(buf + (8 * c + i) * 1024 + lane * 16);
    };
    auto products = [&](int c) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int q = 0; q < QB; ++q)
#pragma unroll
          for (int e = 0; e < NQ; ++e)
            s[q][i & 3] = mfma_bf16(__builtin_bit_cast(bf16x8, a[c & 1][i]), __builtin_bit_cast(bf16x8, qf[q][e][2 * c + (i >> 2)]), s[q][i & 3]);
    };
    keys(0);
#pragma unroll
    for (int c = 0; c < KT / 2; ++c) {
      if (c + 1 < KT / 2) keys(c + 1);
      __builtin_amdgcn_sched_barrier(0);
      if (c == 0) unpack(then);
      __builtin_amdgcn_s_setprio(1);  // (products before the other wave's vector work, which runs beside them: 4,096 rows 216 us, 221 without)
      products(c);
      __builtin_amdgcn_s_setprio(0);
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      sc[j] = pairs[4 * j];
      of[j] = pairs[16 + 4 * j];
    }
    fetch(last(t + 2), uniform(next));
    next = page_of(last(t + 3));
    const f32x4 here = *reinterpret_cast<const f32x4*>(buf + Tile::kHere);
    const bool gap = uniform(fminf(fminf(here[0], here[1]), fminf(here[2], here[3])) < 0.f);
    const bool masked = gap || 64 * t + 63 > wfirst;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int q = 0; q < QB; ++q) s[q][j] = kv4_scores(s[q][j], sc[j], of[j], qs[q]);
    if (masked) {
      asm volatile("");  // (else the compiler masks every tile, by selections without a branch)
#pragma unroll
      for (int q = 0; q < QB; ++q)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int lim = here[j] < 0.f ? -1 : pc[q];
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (64 * t + 16 * j + 4 * g + i > lim) s[q][j][i] = -INFINITY;
        }
    }
    float mx[QB], corr[QB], top[QB];
    bool raise = false;
#pragma unroll
    for (int q = 0; q < QB; ++q) {
      mx[q] = -INFINITY;
      corr[q] = 1.f;
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) mx[q] = fmaxf(mx[q], s[q][j][i]);
      raise |= mx[q] > m_run[q];
    }
    raise = __any(raise);
    if (raise) {
#pragma unroll
      for (int q = 0; q < QB; ++q) {
        mx[q] = groups_max(mx[q]);
        const float m_new = mx[q] > m_run[q] ? mx[q] + slack : m_run[q];
        corr[q] = m_run[q] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m_run[q] - m_new) * sl2);
        m_run[q] = m_new;
        l_run[q] *= corr[q];
        z_run[q] *= corr[q];
      }
    }
    u32x4 va[2][4 * VH];
    f32x4 sv[4], zv[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      sv[j] = pairs[32 + 4 * j];
      zv[j] = pairs[48 + 4 * j];
    }
    auto weights = [&](int q, auto some) {  // (some: keys that a column does not see, whose values may be NaN)
      const float mu = m_run[q] == -INFINITY ? 0.f : m_run[q], mus = mu * sl2;
      top[q] = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float e = kv4_weight<F32>(s[q][j][i], mu, mus, sl2);
          const bool seen = !some || s[q][j][i] != -INFINITY;
          l_run[q] += e;
          z_run[q] = fmaf(e, seen ? zv[j][i] : 0.f, z_run[q]);
          s[q][j][i] = e * (seen ? sv[j][i] : 0.f);
          top[q] = fmaxf(top[q], s[q][j][i]);
        }
    };
    auto values = [&](int u) {
#pragma unroll
      for (int d = 0; d < 4 * VH; ++d) va[u][d] = *reinterpret_cast<const u32x4*>(buf + Tile::kKeys + (u * 4 * VH + d) * 1024 + lane * 16);
    };
    auto add = [&](int q, int u, const uint32_t (&pt)[4][2][NP]) {
#pragma unroll
      for (int d = 0; d < 4 * VH; ++d)
#pragma unroll
        for (int i = 0; i < NP; ++i)
          acc[q][d] = mfma_f16(va[u][d], u32x4{pt[2 * u][0][i], pt[2 * u][1][i], pt[2 * u + 1][0][i], pt[2 * u + 1][1][i]}, acc[q][d]);
    };
    uint32_t pt[QB][4][2][NP];
#pragma unroll
    for (int q = 0; q < QB; ++q) {
      if (masked) weights(q, std::true_type{});
      else weights(q, std::false_type{});
      if (raise || __any(top[q] > kUnitPast * unit[q])) {
        kv4_raise(groups_max(top[q]), unit[q], up[q], corr[q]);
#pragma unroll
        for (int d = 0; d < 4 * VH; ++d)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[q][d][i] *= corr[q];
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        split_h<NP>(s[q][j][0] * up[q], s[q][j][1] * up[q], pt[q][j][0]);
        split_h<NP>(s[q][j][2] * up[q], s[q][j][3] * up[q], pt[q][j][1]);
      }
    }
    values(0);  // (the scores' registers are free now)
    values(1);
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int q = 0; q < QB; ++q) add(q, u, pt[q]);
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(0);
    __syncthreads();
  }
  // ---- lane (col, g) holds values VW / 4 g + 4 VH i + 4 v + d of its columns
#pragma unroll
  for (int q = 0; q < QB; ++q) {
    const float down = unit[q] * kUnweight, l = groups_sum(l_run[q]), z = groups_sum(z_run[q]), m = m_run[q] * sl2;
    if ((wave * QB + q) * 16 + col < cols.n) {
      const float f = p.nsplit == 1 ? kv4_factor<T>(p, row[q], head[q], m, l) : 1.f;
      float* dst = p.nsplit == 1 ? nullptr : kv4_part<VW>(p, row[q], head[q], sp);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int v = 0; v < VH; ++v) {
          const int at = VW / 4 * g + 4 * VH * i + 4 * v;
          f32x4 o;
#pragma unroll
          for (int d = 0; d < 4; ++d) o[d] = fmaf(acc[q][4 * v + d][i], down, z);
          if (p.nsplit == 1) kv4_store<T>(p, row[q], head[q], at, o * f);
          else *reinterpret_cast<f32x4*>(dst + at) = o;
        }
      if (p.nsplit > 1 && g == 0) {
        dst[VW] = m;
        dst[VW + 1] = l;
      }
    }
  }
}

// The ranges of a prompt's columns put together by a launch of their own, a wave a column (partials of 128 columns by device-scope stores and a last
// workgroup, as for few rows, took longer than the attention: 512 rows in two ranges 67 us, in one 28).
template <typename T, int VW, int CW>
__global__ __launch_bounds__(256) void kv4_join_kernel(Kv4Attend p) {
  constexpr int N = VW / 64;  // values a lane
  const int R = p.H / p.pool.G, CB = (p.rows * R + CW - 1) / CW, x = blockIdx.x / p.pool.G, gh = blockIdx.x % p.pool.G;
  const int item = x / CB, lane = threadIdx.x & 63, c = x % CB * CW + blockIdx.y * 4 + uniform(threadIdx.x >> 6);
  int r0 = item, n = 1, b = item;
  if (p.work) {
    r0 = p.work[3 * (size_t)item];
    n = p.work[3 * (size_t)item + 1];
    b = p.work[3 * (size_t)item + 2];
  }
  n = n < p.rows ? n : p.rows;
  if (n <= 0 || r0 < 0 || r0 > p.M - n || b < 0 || b >= p.B || c >= n * R) return;
  const int row = r0 + c / R, head = gh * R + c % R;
  const float* pr = kv4_part<VW>(p, row, head, 0);
  float m = -INFINITY, l = 0.f;
  if (lane < p.nsplit) {  // nsplit <= 64
    m = pr[(size_t)lane * (VW + 4) + VW];
    l = pr[(size_t)lane * (VW + 4) + VW + 1];
  }
  const float top = wave_max(m), w = __builtin_amdgcn_exp2f(m - (top == -INFINITY ? 0.f : top)), f = w * kv4_factor<T>(p, row, head, top, wave_sum(w * l));
  float o[N] = {};
  for (int s = 0; s < p.nsplit; ++s) {
    const float ws = __shfl(f, s, 64);
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = fmaf(ws, pr[(size_t)s * (VW + 4) + N * lane + i], o[i]);
  }
  T* y = (T*)p.y + (size_t)row * p.ldy + (size_t)head * p.V;
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (N * lane + i < p.V) stv(y, N * lane + i, o[i]);
}

// 16-column blocks a wave: two where their accumulators and queries leave room for two workgroups on a CU
constexpr int kv4_blocks(int D, int V, int dt) { return dt == 0 && D <= 128 && V <= 128 ? 2 : 1; }
int kv4_flash_tiles(int columns, int D, int V, int dt) { return (columns + 64 * kv4_blocks(D, V, dt) - 1) / (64 * kv4_blocks(D, V, dt)); }

template <typename T, int KT, int VH, int QB>
static int kv4_flash_run(const Kv4Attend& p, hipStream_t s) {
  auto kern = kv4_flash_kernel<T, KT, VH, QB>;
  constexpr size_t lds = 2 * Kv4Tile<KT, VH>::kBytes;
  if constexpr (lds > 64 * 1024) {
    const hipError_t e = hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (e != hipSuccess) return (int)e;
  }
  const int CB = (p.rows * (p.H / p.pool.G) + 64 * QB - 1) / (64 * QB);
  hipLaunchKernelGGL(kern, dim3((unsigned)p.items * CB * p.pool.G, p.nsplit), dim3(256), lds, s, p);
  if (p.nsplit > 1) hipLaunchKernelGGL((kv4_join_kernel<T, 64 * VH, 64 * QB>), dim3((unsigned)p.items * CB * p.pool.G, 16 * QB), dim3(256), 0, s, p);
  LLJ_CHECK_LAUNCH();
  return 0;
}

template <typename T, int KT, int VH>
static int kv4_flash_go(const Kv4Attend& p, hipStream_t s) {
  constexpr int QB = kv4_blocks(32 * KT, 64 * VH, sizeof(T) == 4);
  // 128 columns a workgroup share a tile's unpacking; with those of half the CUs or fewer, twice as many of 64 are done sooner (32 heads on 8 of 128, a
  // prompt of 512 rows 19.4 us, 26.8 in workgroups of 128; of 128 rows 9.2, 13.3; heads of 64, 900 rows 22.5, 30.4)
  if constexpr (QB == 2) {
    const long long wgs = (long long)p.items * p.pool.G * ((p.rows * (p.H / p.pool.G) + 127) / 128) * p.nsplit;
    if (2 * wgs <= 256) return kv4_flash_run<T, KT, VH, 1>(p, s);
  }
  return kv4_flash_run<T, KT, VH, QB>(p, s);
}

template <typename T, int KT>
static int kv4_flash_values(const Kv4Attend& p, hipStream_t s) {
  if (p.V <= 64) return kv4_flash_go<T, KT, 1>(p, s);
  if (p.V <= 128) return kv4_flash_go<T, KT, 2>(p, s);
  return kv4_flash_go<T, KT, 4>(p, s);
}

template <typename T>
static int kv4_flash_keys(const Kv4Attend& p, hipStream_t s) {
  if (p.D <= 64) return kv4_flash_values<T, 2>(p, s);
  if (p.D <= 128) return kv4_flash_values<T, 4>(p, s);
  return kv4_flash_values<T, 8>(p, s);
}

int kv4_flash(const Kv4Attend& p, int dt, hipStream_t s) { return dt == 0 ? kv4_flash_keys<bf16_t>(p, s) : kv4_flash_keys<float>(p, s); }

}  // namespace llj
