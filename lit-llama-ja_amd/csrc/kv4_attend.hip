// Attention of few rows per sequence over the paged 4-bit cache, split over the keys (mathematics: kv4_attend.h).
//
// One workgroup per (item, 16 columns of a K / V head, key range); a column is a (row, query head) pair, so heads that share a K / V head
// and the rows of a short item share its bytes. Waves walk 16 NB keys at a time on their own (no barriers). K fragment: lane (r, g) holds
// words KT g .. KT g + KT - 1 of key r, one load of 4 KT bytes, and the queries are loaded in that order. V fragment: lane (r, g) takes 4 VH
// columns of 8 keys; two keys' halves are permuted into one word first, so no transposition is needed. A wave's results, then the
// workgroups', are merged by their references.
// Items of up to 8 or 4 columns leave most of the product's 16 unused, and with them most lanes of the softmax: the columns are then given PACK
// times, and the copies' lanes take the scores of different 16-key blocks, which they have anyhow. Their weights go back to the first copy by
// moves inside a row of lanes.
// Measured, 32 heads on 8, 128 wide, bf16: 64 rows behind 8,192 tokens each 107 us, 5.4 TB/s of codes and pairs (a plain read of memory: 6.1); one row
// of 32 heads behind 131,071 tokens 104 us, 5.5 TB/s. There memory and the vector units, which take a key out of its codes in as many instructions
// as the products of 16 columns take cycles, are about even. Few keys are bound by a chain of dependent loads (row, slot, page, codes, then the
// merge's counter): 300 keys 7.2 us, 8 rows behind 4,000 tokens 12.5.
#include "kv4_attend.h"
#include "lit_llama_amd.h"

namespace llj {

constexpr int kv4_step_blocks(int KT, int VH) { return KT <= 4 && VH <= 2 ? 4 : 2; }

// f over the copies of a column, the result in every copy; and a word of copy b for the first copy
template <int PACK, typename F>
__device__ __forceinline__ float over_banks(float v, F f) {
  if constexpr (PACK >= 2) v = f(v, dpp_f32<0x128>(v));  // the lane 8 further round its row
  if constexpr (PACK >= 4) v = f(v, dpp_f32<0x124>(v));
  return v;
}
template <int PACK>
__device__ __forceinline__ uint32_t from_bank(uint32_t v, int b) {  // (b: a constant once the loops are unrolled)
  if (PACK == 2) return b ? dpp_u32<0x108>(v) : v;
  if (PACK == 4) return b == 1 ? dpp_u32<0x104>(v) : b == 2 ? dpp_u32<0x108>(v) : b == 3 ? dpp_u32<0x10C>(v) : v;
  return v;
}

template <typename T, int KT, int VH, int PACK>
__global__ __launch_bounds__(256, KT <= 4 && VH <= 2 ? 2 : 1) void kv4_attend_kernel(Kv4Attend p) {
  constexpr bool F32 = sizeof(T) == 4;
  constexpr int NQ = F32 ? 3 : 1, NP = F32 ? 2 : 1;
  constexpr int NB = kv4_step_blocks(KT, VH), STEP = 16 * NB;  // keys a step
  constexpr int NJ = NB / PACK, CW = 16 / PACK;                // blocks of 16 keys to a lane; columns
  constexpr int KB = 16 * KT, VB = 32 * VH;                      // bytes of a key's, a value's codes
  constexpr int VW = 64 * VH, RP = VW + 4;
  constexpr int VD = VH >= 2 ? VH / 2 : 1;  // words of a value in a lane (VH 1: half of one)
  constexpr float BIAS = F32 ? -8.f : 16.f;  // of the values' codes
  extern __shared__ __attribute__((aligned(16))) float red[];  // [4][16][RP], the waves' results; maxima, sums
  float* wm = red + 4 * 16 * RP;
  float* wl = wm + 64;
  const Kv4Codes codes = kv4_codes();
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), col = lane & 15, g = lane >> 4;
  const int bank = col / CW;  // the copy of the columns that this lane is in: its blocks are PACK j + bank
  const int R = p.H / p.pool.G, HB = (p.rows * R + 15) / 16;
  const int item = blockIdx.x, gh = blockIdx.y / HB, hb = blockIdx.y % HB, sp = blockIdx.z;
  int r0 = item, n = 1, b = item;
  if (p.work) {
    r0 = p.work[3 * (size_t)item];
    n = p.work[3 * (size_t)item + 1];
    b = p.work[3 * (size_t)item + 2];
  }
  n = n < p.rows ? n : p.rows;
  if (n <= 0 || r0 < 0 || r0 > p.M - n || b < 0 || b >= p.B) return;  // (uniform; no such rows)
  const int nc = n * R - 16 * hb < 16 ? n * R - 16 * hb : 16;         // columns of this tile
  if (nc <= 0) return;
  const Kv4Columns cols{r0, gh, R, 16 * hb, nc};
  const int sl = p.slot[b];
  const bool held = sl >= 0 && sl < p.slots;
  const kv4_row tab = scalar_row(p.table + (size_t)(held ? uniform(sl) : 0) * p.ldt);
  int row, head;
  cols.at(col % CW < nc ? col % CW : nc - 1, row, head);
  const int k = p.pool.k, pmask = (1 << k) - 1;
  // the keys a column sees: positions up to its row's, in the table
  int pc = p.pos[row];
  const int most = held ? (p.ldt << k) - 1 : -1;
  pc = pc < most ? pc : most;
  int plast = pc, pfirst = pc;  // over the columns
#pragma unroll
  for (int d = 1; d < 16; d <<= 1) {
    const int o = __shfl_xor(plast, d, 64), f = __shfl_xor(pfirst, d, 64);
    plast = o > plast ? o : plast;
    pfirst = f < pfirst ? f : pfirst;
  }
  plast = uniform(plast);
  pfirst = uniform(pfirst);
  // at most as many ranges as there are rounds of the four waves, and one for two rounds (300 keys: 7.5 us in one, 8.1 in two; 600: 8.8 in
  // one, 8.1 in three): what the caller sized for the longest sequence costs a short one nothing
  const int steps = plast < 0 ? 0 : plast / STEP + 1, rounds = (steps + 3) / 4, ranges = rounds <= 2 ? 1 : rounds < p.nsplit ? rounds : p.nsplit;
  if (sp >= ranges) return;
  const int per = (steps + ranges - 1) / ranges;
  const int s0 = sp * per, s1 = s0 + per < steps ? s0 + per : steps;

  u32x4 qf[NQ][KT];
  const float qs = kv4_query<T, KT, NQ>(p, row, head, g, qf), sl2 = kv4_scale(p), qi = F32 ? 0.f : -16.f * qs;
  const float slack = kv4_slack(F32) / sl2;
  const f32x4 begin = {qi, qi, qi, qi};

  // ---- a step's codes and pairs. Each is fetched anew right behind its use, for the wave's next step: no copies, and every load has most of a step
  // to arrive. The page numbers are read a step ahead of that.
  uint32_t kw[NB][KT], vw[NB][4][VD];
  u32x4 kp[NJ], vp[NJ];
  size_t blk[NB];  // blocks of the step being fetched: their places in the pool
  int off[NB], idn[NB];
  bool ok[NB], okn[NB];
  auto pages = [&](int t) {
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      const int at = (STEP * t + 16 * j) >> k;
      idn[j] = tab[at < p.ldt ? at : p.ldt - 1];
    }
  };
  auto blocks = [&](int t) {
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      okn[j] = idn[j] >= 0 && idn[j] < p.pool.pages;
      off[j] = (STEP * t + 16 * j) & pmask;
      blk[j] = ((size_t)(okn[j] ? idn[j] : 0) * p.pool.G + gh) * p.pool.blk;
    }
  };
  auto fetch_keys = [&] {
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      const uint8_t* ka = p.pool.p + blk[j] + (off[j] + col) * KB + 4 * KT * g;
      if constexpr (KT == 2) {
        const uint2 x = *reinterpret_cast<const uint2*>(ka);
        kw[j][0] = x.x;
        kw[j][1] = x.y;
      } else {
#pragma unroll
        for (int i = 0; i < KT / 4; ++i) {
          const u32x4 x = *reinterpret_cast<const u32x4*>(ka + 16 * i);
#pragma unroll
          for (int e = 0; e < 4; ++e) kw[j][4 * i + e] = x[e];
        }
      }
    }
  };
  auto pick = [&](auto of, int j) {  // of(PACK j + bank): all of them, then a selection (selected first, they are indexed in memory)
    const auto a = of(PACK * j);
    if constexpr (PACK == 1) {
      return a;
    } else {
      const auto b = of(PACK * j + 1);
      const auto lo = bank & 1 ? b : a;
      if constexpr (PACK == 2) {
        return lo;
      } else {
        const auto c = of(2), d = of(3), hi = bank & 1 ? d : c;
        return bank & 2 ? hi : lo;
      }
    }
  };
  auto fetch_pairs = [&](u32x4 (&o)[NJ], int at) {
#pragma unroll
    for (int j = 0; j < NJ; ++j) o[j] = *reinterpret_cast<const u32x4*>(p.pool.p + pick([&](int b) { return blk[b] + 4 * off[b]; }, j) + (at + 16 * g));
  };
  auto fetch_values = [&] {
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      const uint8_t* va = p.pool.p + blk[j] + p.pool.vc + (off[j] + 4 * g) * VB + 2 * VH * col;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (VH == 1) {
          vw[j][i][0] = *reinterpret_cast<const uint16_t*>(va + i * VB);
        } else if constexpr (VH == 2) {
          vw[j][i][0] = *reinterpret_cast<const uint32_t*>(va + i * VB);
        } else {
          const uint2 x = *reinterpret_cast<const uint2*>(va + i * VB);
          vw[j][i][0] = x.x;
          vw[j][i][1] = x.y;
        }
      }
    }
  };

  float m_run = -INFINITY, l_run = 0.f, z_run = 0.f, b_run = 0.f;  // column col's reference; this lane's share of its sums of p, p o', weights
  float unit = kUnitMin, up = weight_unit(unit);                   // of its weights
  f32x4 acc[4 * VH];
#pragma unroll
  for (int d = 0; d < 4 * VH; ++d) acc[d] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (s0 + wave < s1) {
    pages(s0 + wave);
    blocks(s0 + wave);
    pages(s0 + wave + 4);
    // (in the order of the loop, so that the waits there are for the loads they need)
    fetch_keys();
    __builtin_amdgcn_sched_barrier(0);
    fetch_pairs(kp, p.pool.ks);
    __builtin_amdgcn_sched_barrier(0);
    fetch_pairs(vp, p.pool.vs);
    __builtin_amdgcn_sched_barrier(0);
    fetch_values();
  }
  int fold = kFold;
  for (int t = s0 + wave; t < s1; t += 4) {
    const int tn = t + 4 < s1 ? t + 4 : t;  // (behind the last step: the same one again, so that every step waits for the same number of loads)
    bool gap = false;
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      ok[j] = okn[j];
      gap |= !ok[j];
    }
    if (tn != t) blocks(tn);
    pages(t + 8);
    // ---- scores: keys STEP t + 16 j + 4 g + i of column col
    f32x4 s[NB];
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      s[j] = begin;
#pragma unroll
      for (int kk = 0; kk < KT; ++kk) {
        const bf16x8 a = __builtin_bit_cast(bf16x8, codes_bf<F32>(kw[j][kk], codes));
#pragma unroll
        for (int i = 0; i < NQ; ++i) s[j] = mfma_bf16(a, __builtin_bit_cast(bf16x8, qf[i][kk]), s[j]);
      }
    }
    fetch_keys();
    f32x4 sm[NJ];  // keys STEP t + 16 (PACK j + bank) + 4 g + i
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      f32x4 sc, of, x;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[i] = pick([&](int b) { return (float)s[b][i]; }, j);
        sc[i] = bflo(kp[j][i]);
        of[i] = F32 ? bfhi(kp[j][i]) + 8.f * sc[i] : bfhi(kp[j][i]);
      }
      sm[j] = kv4_scores(x, sc, of, qs);
    }
    fetch_pairs(kp, p.pool.ks);
    const bool masked = gap || STEP * t + STEP - 1 > pfirst;  // (uniform)
    if (masked) {
      asm volatile("");  // (else the compiler masks every step, by selections without a branch)
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int lim = pick([&](int b) { return ok[b] ? pc : -1; }, j);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (STEP * t + 16 * (PACK * j + bank) + 4 * g + i > lim) {
            sm[j][i] = -INFINITY;
            vp[j][i] = 0;  // (what stands behind a sequence's end is never multiplied in)
          }
      }
    }
    float mx = -INFINITY, corr = 1.f;
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) mx = fmaxf(mx, sm[j][i]);
    const bool raise = __any(mx > m_run);
    if (raise) {
      mx = groups_max(over_banks<PACK>(mx, [](float a, float b) { return fmaxf(a, b); }));
      const float m_new = mx > m_run ? mx + slack : m_run;
      corr = m_run == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m_run - m_new) * sl2);
      m_run = m_new;
      l_run *= corr;
      z_run *= corr;
    }
    const float mu = m_run == -INFINITY ? 0.f : m_run, mus = mu * sl2;
    float top = 0.f;
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float e = kv4_weight<F32>(sm[j][i], mu, mus, sl2);
        l_run += e;
        z_run = fmaf(e, bfhi(vp[j][i]), z_run);
        sm[j][i] = e * bflo(vp[j][i]);
        top = fmaxf(top, sm[j][i]);
      }
    if (raise || __any(top > kUnitPast * unit)) {
      kv4_raise(groups_max(over_banks<PACK>(top, [](float a, float b) { return fmaxf(a, b); })), unit, up, corr);
      b_run *= corr;
#pragma unroll
      for (int d = 0; d < 4 * VH; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[d][i] *= corr;
    }
    uint32_t pm[NJ][2][NP], pt[NB][2][NP];
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      float w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        w[i] = sm[j][i] * up;
        if (F32) b_run += w[i];
      }
      split_h<NP>(w[0], w[1], pm[j][0]);
      split_h<NP>(w[2], w[3], pm[j][1]);
      if (!F32) b_run = add_pair(pm[j][1][0], add_pair(pm[j][0][0], b_run));
    }
#pragma unroll
    for (int j = 0; j < NB; ++j)  // block j's weights to the first copy of the columns (the others' columns are never stored)
#pragma unroll
      for (int i = 0; i < 2 * NP; ++i) pt[j][i / NP][i % NP] = from_bank<PACK>(pm[j / PACK][i / NP][i % NP], j % PACK);
    fetch_pairs(vp, p.pool.vs);
#pragma unroll
    for (int u = 0; u < NB / 2; ++u)
#pragma unroll
      for (int v = 0; v < VH; ++v) {
        u32x4 x[4];  // columns 4 v + d of 8 keys
#pragma unroll
        for (int e = 0; e < 4; ++e) {  // two keys' halves in a word
          const uint32_t a = vw[2 * u + (e >> 1)][2 * (e & 1)][v / 2], c = vw[2 * u + (e >> 1)][2 * (e & 1) + 1][v / 2];
          const u32x4 y = codes_h<F32>(VH == 1 ? a | c << 16 : __builtin_amdgcn_perm(c, a, v % 2 ? 0x07060302u : 0x05040100u), codes);
#pragma unroll
          for (int d = 0; d < 4; ++d) x[d][e] = y[d];
        }
#pragma unroll
        for (int d = 0; d < 4; ++d)
#pragma unroll
          for (int i = 0; i < NP; ++i)
            acc[4 * v + d] = mfma_f16(x[d], u32x4{pt[2 * u][0][i], pt[2 * u][1][i], pt[2 * u + 1][0][i], pt[2 * u + 1][1][i]}, acc[4 * v + d]);
      }
    fetch_values();
    if (!F32 && --fold == 0) {
      fold = kFold;
      const float z = -BIAS * groups_sum(over_banks<PACK>(b_run, [](float a, float b) { return a + b; }));
      b_run = 0.f;
#pragma unroll
      for (int d = 0; d < 4 * VH; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[d][i] += z;
    }
  }
  // ---- the four waves' results, in order. Lane (col, g) holds values VW / 4 g + 4 VH i + d of its column, d = 4 v + e
  const auto plus = [](float a, float b) { return a + b; };
  l_run = groups_sum(over_banks<PACK>(l_run, plus));
  const float down = unit * kUnweight;
  z_run = groups_sum(over_banks<PACK>(z_run - BIAS * down * b_run, plus));
  {
    float* o = red + (wave * 16 + col) * RP + VW / 4 * g;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int v = 0; v < VH; ++v)
        *reinterpret_cast<f32x4*>(o + 4 * VH * i + 4 * v) = f32x4{fmaf(acc[4 * v][i], down, z_run), fmaf(acc[4 * v + 1][i], down, z_run),
                                                                  fmaf(acc[4 * v + 2][i], down, z_run), fmaf(acc[4 * v + 3][i], down, z_run)};
  }
  if (g == 0) {
    wm[wave * 16 + col] = m_run * sl2;
    wl[wave * 16 + col] = l_run;
  }
  __syncthreads();
  for (int i = tid; i < nc * (VW / 4); i += 256) {
    const int cc = i / (VW / 4), v = 4 * (i % (VW / 4));
    const float mx = fmaxf(fmaxf(wm[cc], wm[16 + cc]), fmaxf(wm[32 + cc], wm[48 + cc]));
    const float mu = mx == -INFINITY ? 0.f : mx;  // no keys: every weight is exp2(-inf) = 0
    float l = 0.f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float e = __builtin_amdgcn_exp2f(wm[16 * w + cc] - mu);
      l += e * wl[16 * w + cc];
      o += *reinterpret_cast<const f32x4*>(red + (w * 16 + cc) * RP + v) * e;
    }
    int rr, hh;
    cols.at(cc, rr, hh);
    if (ranges == 1) {
      kv4_store<T>(p, rr, hh, v, o * kv4_factor<T>(p, rr, hh, mx, l));
    } else {
      float* dst = kv4_part<VW>(p, rr, hh, sp);
      put2(dst + v, o[0], o[1]);
      put2(dst + v + 2, o[2], o[3]);
      if (v == 0) put2(dst + VW, mx, l);
    }
  }
  if (ranges > 1) kv4_merge<T, VW>(p, cols, ranges, p.count + (size_t)item * gridDim.y + blockIdx.y, red);
}

template <typename T, int KT, int VH, int PACK>
static int kv4_attend_go(const Kv4Attend& p, hipStream_t s) {
  auto kern = kv4_attend_kernel<T, KT, VH, PACK>;
  constexpr size_t lds = (size_t)(4 * 16 * (64 * VH + 4) + 128) * 4;
  if constexpr (lds > 64 * 1024) {
    const hipError_t e = hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (e != hipSuccess) return (int)e;
  }
  const int R = p.H / p.pool.G, HB = (p.rows * R + 15) / 16;
  hipLaunchKernelGGL(kern, dim3(p.items, p.pool.G * HB, p.nsplit), dim3(256), lds, s, p);
  LLJ_CHECK_LAUNCH();
  return 0;
}

template <typename T, int KT, int VH>
static int kv4_attend_pack(const Kv4Attend& p, hipStream_t s) {
  const int c = p.rows * (p.H / p.pool.G);
  if constexpr (kv4_step_blocks(KT, VH) == 4)
    if (c <= 4) return kv4_attend_go<T, KT, VH, 4>(p, s);
  return c <= 8 ? kv4_attend_go<T, KT, VH, 2>(p, s) : kv4_attend_go<T, KT, VH, 1>(p, s);
}

template <typename T, int KT>
static int kv4_attend_values(const Kv4Attend& p, hipStream_t s) {
  if (p.V <= 64) return kv4_attend_pack<T, KT, 1>(p, s);
  if (p.V <= 128) return kv4_attend_pack<T, KT, 2>(p, s);
  return kv4_attend_pack<T, KT, 4>(p, s);
}

template <typename T>
static int kv4_attend_keys(const Kv4Attend& p, hipStream_t s) {
  if (p.D <= 64) return kv4_attend_values<T, 2>(p, s);
  if (p.D <= 128) return kv4_attend_values<T, 4>(p, s);
  return kv4_attend_values<T, 8>(p, s);
}

constexpr int kv4_few_columns = 64;  // items of up to this many columns take the kernel above

}  // namespace llj

using namespace llj;

extern "C" {

int llj_kv4_part_width(int vdim) { return kv4_width(vdim) + 4; }

int llj_kv4_tiles(int heads, int kv_heads, int dim, int vdim, int rows, int dt) {
  if (heads < 1 || heads > 65535 || kv_heads < 1 || heads % kv_heads || rows < 1 || rows > 65535 || dim < 1 || dim > 256 || vdim < 1 || vdim > 256) return 0;
  const long long c = (long long)rows * (heads / kv_heads);
  if (c > 1 << 24) return 0;
  return kv_heads * (c > kv4_few_columns ? kv4_flash_tiles((int)c, dim, vdim, dt) : (int)(c + 15) / 16);
}

int llj_kv4_attend(const void* q, int ldq, const void* gate, int ldg, const int* work, int items, int rows, const int* pos, const int* slot, int B,
                   const int* table, int slots, int ldt, const void* pool, int pages, int page, float* part, int* count, int nsplit, void* y,
                   int ldy, int M, int heads, int kv_heads, int dim, int vdim, float scale, int sink, int dt, void* stream) {
  LLJ_REQUIRE(kv4_sizes(pool, pages, page, kv_heads, dim, vdim, dt) && q && pos && slot && table && y && items >= 0 && rows >= 1 && rows <= 65535 &&
              B >= 1 && slots >= 1 && ldt >= 1 && ldt <= (1 << 30) / page && M >= 0 && heads >= 1 && heads % kv_heads == 0 && heads <= 65535 &&
              ldq >= heads * dim && ldy >= heads * vdim && (!gate || ldg >= heads) && nsplit >= 1 && nsplit <= 64 && (nsplit == 1 || part) &&
              ((uintptr_t)part & 15) == 0 && ((uintptr_t)count & 3) == 0 && (work || (rows == 1 && items <= M && items <= B)));
  const int tiles = llj_kv4_tiles(heads, kv_heads, dim, vdim, rows, dt);
  const bool few = rows * (heads / kv_heads) <= kv4_few_columns;
  LLJ_REQUIRE(tiles > 0 && (long long)items * tiles < 1 << 24 && (nsplit == 1 || !few || count));
  if (items == 0 || M == 0) return 0;
  Kv4Attend p{};
  p.q = q; p.gate = gate; p.ldq = ldq; p.ldg = ldg; p.work = work; p.items = items; p.rows = rows;
  p.pos = pos; p.slot = slot; p.table = table; p.B = B; p.slots = slots; p.ldt = ldt;
  p.pool = kv4_pool((void*)pool, pages, kv_heads, kv4_page_log2(page), dim, vdim);
  p.y = y; p.ldy = ldy; p.M = M; p.H = heads; p.D = dim; p.V = vdim; p.sink = sink;
  p.scale = scale;
  p.part = part; p.count = count; p.nsplit = nsplit;
  p.quads = vdim % 4 == 0 && ldy % 4 == 0 && ((uintptr_t)y & (dt ? 15 : 7)) == 0;
  hipStream_t s = (hipStream_t)stream;
  if (!few) return kv4_flash(p, dt, s);
  return dt == 0 ? kv4_attend_keys<bf16_t>(p, s) : kv4_attend_keys<float>(p, s);
}

}  // extern "C"
