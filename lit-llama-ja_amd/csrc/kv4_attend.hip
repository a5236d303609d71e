// Attention of few rows per sequence over the paged 4-bit cache (layout: kv4.h), split over the keys.
//   S_rj = scale (s_j sum_i q_ri c_ji + o_j sum_i q_ri),  y_r = sum_j p_rj (s'_j c'_j + o'_j),  p the softmax over j <= pos_r
// The codes go into the MFMA product as exact bf16 integers 16 + c (one and-or per pair); scales and offsets are applied to the scores in fp32, and
// to the weights before the second product, so nothing of a key or value is rounded: sum_j p s' c' = sum_j (p s') (16 + c') + sum_j p (o' - 16 s').
// The weights enter as two bf16 terms (bf16 rows: 16 bits) or three (fp32 rows: all 24), fp32 queries as three.
//
// One workgroup per (item, 16 columns of a K / V head, key range); a column is a (row, query head) pair, so heads that share a K / V head
// and the rows of a short item share its bytes. Waves walk 16 NB keys at a time on their own (no barriers), the next step's codes in registers
// on their way; the page numbers two steps ahead. K fragment: lane (r, g) holds words KT g .. KT g + KT - 1 of key r, one load of 4 KT bytes, and the
// queries are loaded in that order. V fragment: lane (r, g) takes 4 VH columns of 8 keys; two keys' halves are permuted into one word first,
// so no transposition is needed. A wave's results, then the workgroups', are merged by their maxima.
#include "kv4_attend.h"
#include "lit_llama_amd.h"

namespace llj {

template <typename T, int KT, int VH>
__global__ __launch_bounds__(256) void kv4_attend_kernel(Kv4Attend p) {
  constexpr bool F32 = sizeof(T) == 4;
  constexpr int NQ = F32 ? 3 : 1, NP = F32 ? 3 : 2;
  constexpr int NB = KT <= 4 && VH <= 2 ? 4 : 2, STEP = 16 * NB;  // keys a step
  constexpr int KB = 16 * KT, VB = 32 * VH;                      // bytes of a key's, a value's codes
  constexpr int VW = 64 * VH, RP = VW + 4;
  constexpr int VD = VH >= 2 ? VH / 2 : 1;  // words of a value in a lane (VH 1: half of one)
  extern __shared__ __attribute__((aligned(16))) float red[];  // [4][16][RP], the waves' results; maxima, sums
  float* wm = red + 4 * 16 * RP;
  float* wl = wm + 64;
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), col = lane & 15, g = lane >> 4;
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
  const int sl = p.slot[b];
  const int* tab = p.table + (size_t)(sl >= 0 && sl < p.slots ? sl : 0) * p.ldt;
  const int c = 16 * hb + (col < nc ? col : nc - 1), row = r0 + c / R, h = gh * R + c % R;
  const int k = p.pool.k, pmask = (1 << k) - 1;
  // the keys a column sees: positions up to its row's, in the table
  int pc = p.pos[row];
  const int most = sl >= 0 && sl < p.slots ? (p.ldt << k) - 1 : -1;
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
  const int steps = plast < 0 ? 0 : plast / STEP + 1, per = (steps + p.nsplit - 1) / p.nsplit;
  const int s0 = sp * per, s1 = s0 + per < steps ? s0 + per : steps;

  // ---- the queries, in the order of a key's words; their sum
  u32x4 qf[NQ][KT];
  float qs = 0.f;
  {
    const T* qr = (const T*)p.q + (size_t)row * p.ldq + (size_t)h * p.D;
    const bool whole = p.D % 8 == 0 && (((uintptr_t)p.q | ((size_t)p.ldq * sizeof(T))) & 15) == 0;
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
      for (int e = 0; e < 8; ++e) qs += x[e];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        uint32_t t[NQ];
        split_pair<NQ>(x[e], x[e + 4], t);
#pragma unroll
        for (int i = 0; i < NQ; ++i) qf[i][kk][e] = t[i];
      }
    }
    qs = groups_sum(qs);
  }
  const float qs2 = qs * p.sl2, qi = -16.f * qs;
  const uint32_t mask = kCodeMask, base = kCodeBase;

  // ---- a step's codes and pairs
  uint32_t kw[NB][KT], vw[NB][4][VD];
  u32x4 kp[NB], vp[NB];
  int id[NB], idn[NB];  // pages of the step being fetched and of the one after
  bool okf[NB];
  auto pages = [&](int t, int (&o)[NB]) {
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      const int at = (STEP * t + 16 * j) >> k;
      o[j] = tab[at < p.ldt ? at : p.ldt - 1];
    }
  };
  auto fetch = [&](int t) {  // from the pages in id
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      okf[j] = id[j] >= 0 && id[j] < p.pool.pages;
      const int off = (STEP * t + 16 * j) & pmask;
      const uint8_t* blk = p.pool.p + ((size_t)(okf[j] ? id[j] : 0) * p.pool.G + gh) * p.pool.blk;
      const uint8_t* ka = blk + (off + col) * KB + 4 * KT * g;
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
      kp[j] = *reinterpret_cast<const u32x4*>(blk + p.pool.ks + 4 * (off + 4 * g));
      vp[j] = *reinterpret_cast<const u32x4*>(blk + p.pool.vs + 4 * (off + 4 * g));
      const uint8_t* va = blk + p.pool.vc + (off + 4 * g) * VB + 2 * VH * col;
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

  float m_run = -INFINITY, l_run = 0.f, z_run = 0.f;  // maximum of column col; this lane's share of its sums
  f32x4 acc[4 * VH];
#pragma unroll
  for (int d = 0; d < 4 * VH; ++d) acc[d] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (s0 + wave < s1) {
    pages(s0 + wave, id);
    pages(s0 + wave + 4, idn);
    fetch(s0 + wave);
  }
  for (int t = s0 + wave; t < s1; t += 4) {
    // ---- scores: keys STEP t + 16 j + 4 g + i of column col
    f32x4 s[NB];
    bool gap = false, ok[NB];
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      s[j] = f32x4{qi, qi, qi, qi};
      ok[j] = okf[j];
      gap |= !ok[j];
#pragma unroll
      for (int kk = 0; kk < KT; ++kk) {
        const bf16x8 a = __builtin_bit_cast(bf16x8, codes8(kw[j][kk], mask, base));
#pragma unroll
        for (int i = 0; i < NQ; ++i) s[j] = mfma_bf16(a, __builtin_bit_cast(bf16x8, qf[i][kk]), s[j]);
      }
    }
    // the values' bf16 pairs of keys, before their registers are loaded again
    u32x4 pw[NB];
    uint32_t vx[NB / 2][4][VH];  // [32 keys][pair][4 columns]: two keys' halves
#pragma unroll
    for (int u = 0; u < NB / 2; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t(&a)[VD] = vw[2 * u + (e >> 1)][2 * (e & 1)], (&c2)[VD] = vw[2 * u + (e >> 1)][2 * (e & 1) + 1];
        if constexpr (VH == 1) {
          vx[u][e][0] = a[0] | c2[0] << 16;
        } else {
#pragma unroll
          for (int i = 0; i < VD; ++i) {
            vx[u][e][2 * i] = __builtin_amdgcn_perm(c2[i], a[i], 0x05040100u);
            vx[u][e][2 * i + 1] = __builtin_amdgcn_perm(c2[i], a[i], 0x07060302u);
          }
        }
      }
    float mx = -INFINITY;
    const bool masked = gap || STEP * t + STEP - 1 > pfirst;  // (uniform)
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      pw[j] = vp[j];
#pragma unroll
      for (int i = 0; i < 4; ++i) s[j][i] = bflo(kp[j][i]) * p.sl2 * s[j][i] + bfhi(kp[j][i]) * qs2;
      if (masked) {
        const int lim = ok[j] ? pc : -1;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (STEP * t + 16 * j + 4 * g + i > lim) {
            s[j][i] = -INFINITY;
            pw[j][i] = 0;  // (what stands behind a sequence's end is never multiplied in)
          }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) mx = fmaxf(mx, s[j][i]);
    }
    if (t + 4 < s1) {  // in flight over this step's softmax and second product
#pragma unroll
      for (int j = 0; j < NB; ++j) id[j] = idn[j];
      fetch(t + 4);
      pages(t + 8, idn);
    }
    mx = groups_max(mx);
    const float m_new = fmaxf(m_run, mx), mu = m_new == -INFINITY ? 0.f : m_new;
    const float corr = __builtin_amdgcn_exp2f(m_run - mu);
    m_run = m_new;
    l_run *= corr;
    z_run *= corr;
    uint32_t pt[NB][2][NP];
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      float w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float e = __builtin_amdgcn_exp2f(s[j][i] - mu), sv = bflo(pw[j][i]);
        l_run += e;
        z_run += e * (bfhi(pw[j][i]) - 16.f * sv);
        w[i] = e * sv;
      }
      split_pair<NP>(w[0], w[1], pt[j][0]);
      split_pair<NP>(w[2], w[3], pt[j][1]);
    }
    if (__any(corr != 1.f)) {
#pragma unroll
      for (int d = 0; d < 4 * VH; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[d][i] *= corr;
    }
#pragma unroll
    for (int u = 0; u < NB / 2; ++u)
#pragma unroll
      for (int v = 0; v < VH; ++v) {
        u32x4 x[4];  // columns 4 v + d
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const u32x4 y = codes8(vx[u][e][v], mask, base);
#pragma unroll
          for (int d = 0; d < 4; ++d) x[d][e] = y[d];
        }
#pragma unroll
        for (int d = 0; d < 4; ++d)
#pragma unroll
          for (int i = 0; i < NP; ++i) {
            const u32x4 w = {pt[2 * u][0][i], pt[2 * u][1][i], pt[2 * u + 1][0][i], pt[2 * u + 1][1][i]};
            acc[4 * v + d] = mfma_bf16(__builtin_bit_cast(bf16x8, x[d]), __builtin_bit_cast(bf16x8, w), acc[4 * v + d]);
          }
      }
  }
  // ---- the four waves' results, in order. Lane (col, g) holds values VW / 4 g + 4 VH i + d of its column, d = 4 v + e
  l_run = groups_sum(l_run);
  z_run = groups_sum(z_run);
  {
    float* o = red + (wave * 16 + col) * RP + VW / 4 * g;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int v = 0; v < VH; ++v)
        *reinterpret_cast<f32x4*>(o + 4 * VH * i + 4 * v) =
            f32x4{acc[4 * v][i] + z_run, acc[4 * v + 1][i] + z_run, acc[4 * v + 2][i] + z_run, acc[4 * v + 3][i] + z_run};
  }
  if (g == 0) {
    wm[wave * 16 + col] = m_run;
    wl[wave * 16 + col] = l_run;
  }
  __syncthreads();
  auto place = [&](int cc, int& rr, int& hh) {
    rr = r0 + (16 * hb + cc) / R;
    hh = gh * R + (16 * hb + cc) % R;
  };
  auto store = [&](int cc, int v, f32x4 o) {
    int rr, hh;
    place(cc, rr, hh);
    T* y = (T*)p.y + (size_t)rr * p.ldy + (size_t)hh * p.V;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (v + i < p.V) stv(y, v + i, o[i]);
  };
  auto gated = [&](int cc, float l) {  // l (1 + exp(-gate)): what a column's sum is divided by
    if (!p.gate) return l;
    int rr, hh;
    place(cc, rr, hh);
    return l * (1.f + __expf(-ldv((const T*)p.gate, (size_t)rr * p.ldg + hh)));
  };
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
    if (p.nsplit == 1) {
      const float mt = p.sink ? fmaxf(mu, 0.f) : mu, e = __builtin_amdgcn_exp2f(mu - mt);
      l = e * l + (p.sink ? __builtin_amdgcn_exp2f(-mt) : 0.f);
      const float f = l == 0.f ? 0.f : e / gated(cc, l);  // a row that sees nothing is zero
      store(cc, v, o * f);
    } else {
      int rr, hh;
      place(cc, rr, hh);
      float* dst = p.part + (((size_t)rr * p.H + hh) * p.nsplit + sp) * RP;
      put2(dst + v, o[0], o[1]);
      put2(dst + v + 2, o[2], o[3]);
      if (v == 0) put2(dst + VW, mx, l);
    }
  }
  if (p.nsplit == 1) return;
  // ---- the last of the ranges' workgroups merges them: device-scope stores, a wait for them, one device-scope counter per
  // tile, device-scope loads; nobody waits for another workgroup, and the last one resets the counter
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  int* last = reinterpret_cast<int*>(wm);
  if (tid == 0) {
    int* ct = p.count + (size_t)item * gridDim.y + blockIdx.y;
    const int done = __hip_atomic_fetch_add(ct, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    *last = done == p.nsplit - 1;
    if (done == p.nsplit - 1) __hip_atomic_store(ct, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!*last) return;
  float* sw = red;  // [16][64] the ranges' weights
  for (int cc = wave; cc < nc; cc += 4) {  // nsplit <= 64
    int rr, hh;
    place(cc, rr, hh);
    const float* pr = p.part + ((size_t)rr * p.H + hh) * p.nsplit * RP;
    float2 st = make_float2(-INFINITY, 0.f);
    if (lane < p.nsplit) st = get2(pr + (size_t)lane * RP + VW);
    float mt = wave_max(st.x);
    mt = p.sink ? fmaxf(mt, 0.f) : mt == -INFINITY ? 0.f : mt;
    const float w = __builtin_amdgcn_exp2f(st.x - mt);
    const float L = wave_sum(w * st.y) + (p.sink ? __builtin_amdgcn_exp2f(-mt) : 0.f);
    sw[cc * 64 + lane] = L == 0.f ? 0.f : w / gated(cc, L);
  }
  __syncthreads();
  for (int i = tid; i < nc * (VW / 4); i += 256) {
    const int cc = i / (VW / 4), v = 4 * (i % (VW / 4));
    int rr, hh;
    place(cc, rr, hh);
    const float* pr = p.part + ((size_t)rr * p.H + hh) * p.nsplit * RP + v;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    for (int s2 = 0; s2 < p.nsplit; s2 += 8) {
      float2 a[8], c2[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float* q = pr + (size_t)(s2 + e < p.nsplit ? s2 + e : p.nsplit - 1) * RP;
        a[e] = get2(q);
        c2[e] = get2(q + 2);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (s2 + e < p.nsplit) o += f32x4{a[e].x, a[e].y, c2[e].x, c2[e].y} * sw[cc * 64 + s2 + e];
    }
    store(cc, v, o);
  }
}

template <typename T, int KT, int VH>
static int kv4_attend_go(const Kv4Attend& p, hipStream_t s) {
  auto kern = kv4_attend_kernel<T, KT, VH>;
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

template <typename T, int KT>
static int kv4_attend_values(const Kv4Attend& p, hipStream_t s) {
  if (p.V <= 64) return kv4_attend_go<T, KT, 1>(p, s);
  if (p.V <= 128) return kv4_attend_go<T, KT, 2>(p, s);
  return kv4_attend_go<T, KT, 4>(p, s);
}

template <typename T>
static int kv4_attend_keys(const Kv4Attend& p, hipStream_t s) {
  if (p.D <= 64) return kv4_attend_values<T, 2>(p, s);
  if (p.D <= 128) return kv4_attend_values<T, 4>(p, s);
  return kv4_attend_values<T, 8>(p, s);
}

}  // namespace llj

using namespace llj;

extern "C" {

int llj_kv4_part_width(int vdim) { return kv4_width(vdim) + 4; }

int llj_kv4_tiles(int heads, int kv_heads, int rows) {
  if (heads < 1 || kv_heads < 1 || heads % kv_heads || rows < 1 || rows > 65535) return 0;
  const long long n = (long long)kv_heads * (((long long)rows * (heads / kv_heads) + 15) / 16);
  return n <= 65535 ? (int)n : 0;
}

int llj_kv4_attend(const void* q, int ldq, const void* gate, int ldg, const int* work, int items, int rows, const int* pos, const int* slot, int B,
                   const int* table, int slots, int ldt, const void* pool, int pages, int page, float* part, int* count, int nsplit, void* y,
                   int ldy, int M, int heads, int kv_heads, int dim, int vdim, float scale, int sink, int dt, void* stream) {
  LLJ_REQUIRE(kv4_sizes(pool, pages, page, kv_heads, dim, vdim, dt) && q && pos && slot && table && y && items >= 0 && rows >= 1 && rows <= 65535 &&
              B >= 1 && slots >= 1 && ldt >= 1 && ldt <= (1 << 30) / page && M >= 0 && heads >= 1 && heads % kv_heads == 0 && heads <= 65535 &&
              ldq >= heads * dim && ldy >= heads * vdim && (!gate || ldg >= heads) && nsplit >= 1 && nsplit <= 64 && (nsplit == 1 || (part && count)) &&
              (((uintptr_t)part | (uintptr_t)count) & 7) == 0 && (work || (rows == 1 && items <= M && items <= B)));
  LLJ_REQUIRE(llj_kv4_tiles(heads, kv_heads, rows) > 0);
  if (items == 0 || M == 0) return 0;
  Kv4Attend p{};
  p.q = q; p.gate = gate; p.ldq = ldq; p.ldg = ldg; p.work = work; p.items = items; p.rows = rows;
  p.pos = pos; p.slot = slot; p.table = table; p.B = B; p.slots = slots; p.ldt = ldt;
  p.pool = kv4_pool((void*)pool, pages, kv_heads, kv4_page_log2(page), dim, vdim);
  p.y = y; p.ldy = ldy; p.M = M; p.H = heads; p.D = dim; p.V = vdim; p.sink = sink;
  p.sl2 = scale * 1.4426950408889634f;
  p.part = part; p.count = count; p.nsplit = nsplit;
  hipStream_t s = (hipStream_t)stream;
  return dt == 0 ? kv4_attend_keys<bf16_t>(p, s) : kv4_attend_keys<float>(p, s);
}

}  // extern "C"
