// Block tables of paged caches. A page holds 2^k tokens of one sequence; table[slot][i] is the page of the slot's tokens
// i 2^k .. (i + 1) 2^k - 1, seen[slot] the tokens it holds, free_ids[0 .. nfree) a stack of the pages nobody holds.
//   extend   sequence b of a call gets add[b] more tokens: with L = seen[slot[b]], have = ceil(L / page) and
//            new = ceil((L + add) / page) - have, its new page j is free_ids[nfree - 1 - (base[b] + j)], base the exclusive sum of
//            `new` over the call. Row m of the call belongs to the sequence b with row0[b] <= m < row0[b + 1], at position
//            L + m - row0[b], whose place in the cache is table[slot][position / page] * page + position % page.
//   release  the pages of ended sequences back onto the stack.
// Both take or leave everything: a call that cannot be served has no rows and changes no table; *status says so (1: too few free pages, 2: a
// slot outside the tables or named twice, a length or table width passed, more rows than room), and *fault, which keeps every such bit.
//
// The sums run in one workgroup (a call has at most kMaxSeqs sequences, whose sums stay in LDS), so nothing of the tables is handed from one
// workgroup to another inside a launch. Everything else is a flat loop over pages, rows or work items, each of which finds
// its sequence by bisection. Bound by the chain of dependent loads (slot, length, page, place), not by bytes: a step of 8 sequences 3.8 us, 48
// sequences with 9 prompts of 6,400 rows 9.4, 2,048 sequences with 130,000 rows 8.9 and 5.5 (rows).
#include "common.h"
#include "lit_llama_amd.h"

namespace llj {

constexpr int kMaxSeqs = 4096;    // three sums of 16 KiB in LDS
constexpr int kMaxSlots = 65536;  // a bit each in LDS
constexpr int kPlanThreads = 1024;
constexpr int kSat = 0x3fffffff;  // sums saturate here: past every size that is taken
constexpr int kMaxTokens = 1 << 30;  // of a sequence
constexpr int kFewRows = 8192;    // calls up to this many rows and items are one launch (6,400 rows: 9.4 us, in two launches 6.7 + 4.1)

struct ExtendParams {
  const int *slot, *add;
  int B;
  int *seen, *table;
  int slots, ldt;
  const int* free_ids;
  int* nfree;
  int cap, k, commit;
  int *row0, *item0, *row_seq, *pos, *place, *work, *after, *left, *status, *fault;
  int M, nwork, chunk;
};

__device__ __forceinline__ int sat_add(int a, int b) {
  const int s = a + b;  // both at most kSat: no overflow
  return s < kSat ? s : kSat;
}

// the last i in [0, n) with at[i] <= x (at[0] = 0 <= x); of equal entries the last, so empty sequences are passed over
__device__ __forceinline__ int find_seq(const int* at, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (at[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

// v plus the values that the lanes before hold (saturating), through the lanes' neighbours: 6 steps of one move and one sum
template <int CTRL, int ROWS>
__device__ __forceinline__ int scan_step(int v) {
  return sat_add(v, __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, false));
}
__device__ __forceinline__ int wave_scan(int v) {
  v = scan_step<0x111, 0xF>(v);  // row_shr 1, 2, 4, 8
  v = scan_step<0x112, 0xF>(v);
  v = scan_step<0x114, 0xF>(v);
  v = scan_step<0x118, 0xF>(v);
  v = scan_step<0x142, 0xA>(v);         // the end of rows 0 and 2 to 1 and 3
  return scan_step<0x143, 0xC>(v);      // of row 1 to 2 and 3
}

// exclusive sums of three values over the workgroup (right unless they saturate, and then nothing is taken); total in `sum`. part: zero
// behind the workgroup's waves.
__device__ __forceinline__ void scan3(int (&v)[3], int (&sum)[3], int4 (*part)) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int in[3];
#pragma unroll
  for (int i = 0; i < 3; ++i) in[i] = wave_scan(v[i]);
  __syncthreads();  // the last call's readers of part are done
  if (lane == 63) part[wave] = make_int4(in[0], in[1], in[2], 0);
  __syncthreads();
  int before[3] = {0, 0, 0}, all[3] = {0, 0, 0};
#pragma unroll
  for (int w = 0; w < kPlanThreads / 64; ++w) {
    const int4 x = part[w];
    const int a[3] = {x.x, x.y, x.z};
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      before[i] = w == wave ? all[i] : before[i];
      all[i] = sat_add(all[i], a[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    v[i] = sat_add(before[i], in[i] - v[i]);
    sum[i] = all[i];
  }
}

__device__ __forceinline__ void row_out(const ExtendParams& p, const int* row0, const int* item0, int m) {
  if (m >= row0[p.B]) {
    p.row_seq[m] = p.pos[m] = p.place[m] = -1;
    return;
  }
  const int b = find_seq(row0, p.B, m), s = p.slot[b], i = m - row0[b];
  // after = L + add, left behind by the sums (in this launch: by a thread of this workgroup, before a barrier)
  const int ps = p.after[b] - (row0[b + 1] - row0[b]) + i;
  p.row_seq[m] = b;
  p.pos[m] = ps;
  p.place[m] = (p.table[(size_t)s * p.ldt + (ps >> p.k)] << p.k) + (ps & ((1 << p.k) - 1));
  if (p.chunk && i % p.chunk == 0) {
    int* w = p.work + 3 * (size_t)(item0[b] + i / p.chunk);
    const int left = row0[b + 1] - m;
    w[0] = m;
    w[1] = left < p.chunk ? left : p.chunk;
    w[2] = b;
  }
}

__device__ __forceinline__ void item_pad(const ExtendParams& p, int t) {
  p.work[3 * (size_t)t] = p.work[3 * (size_t)t + 1] = p.work[3 * (size_t)t + 2] = 0;
}

__global__ __launch_bounds__(kPlanThreads) void pages_extend_kernel(ExtendParams p, int rows_here) {
  extern __shared__ int lds[];
  int* s_row = lds;                      // [B + 1]
  int* s_new = s_row + p.B + 1;          // [B + 1]
  int* s_item = s_new + p.B + 1;         // [B + 1]
  unsigned* s_used = reinterpret_cast<unsigned*>(s_item + p.B + 1);  // [slots / 32]
  __shared__ int s_bad;
  __shared__ int4 part[kPlanThreads / 64];
  const int tid = threadIdx.x, nt = blockDim.x, page = 1 << p.k;
  for (int i = tid; i < (p.slots + 31) / 32; i += nt) s_used[i] = 0;
  if (tid < kPlanThreads / 64) part[tid] = make_int4(0, 0, 0, 0);
  if (tid == 0) s_bad = 0;
  int nfree = *p.nfree;
  __syncthreads();
  if (nfree < 0 || nfree > p.cap) {
    nfree = 0;
    s_bad = 2;
  }
  int carry[3] = {0, 0, 0};
  for (int b0 = 0; b0 < p.B; b0 += nt) {
    const int b = b0 + tid;
    int v[3] = {0, 0, 0}, sum[3];
    if (b < p.B) {
      const int s = p.slot[b], n = p.add ? p.add[b] : 1;
      bool ok = s >= 0 && s < p.slots && n >= 0 && n <= p.M;
      if (ok) {
        const unsigned bit = 1u << (s & 31);
        if (atomicOr(&s_used[s >> 5], bit) & bit) ok = false;  // a slot twice
        const int L = p.seen[s];
        // (L + n at most 2^31 - 1 in unsigned arithmetic, then against the table's width)
        const unsigned need = (((unsigned)L + (unsigned)n) + page - 1) >> p.k;
        if (L < 0 || L > kMaxTokens || need > (unsigned)p.ldt) ok = false;
        if (ok) {
          v[0] = n;
          v[1] = (int)need - ((L + page - 1) >> p.k);
          v[2] = p.chunk ? (n + p.chunk - 1) / p.chunk : 0;
        }
      }
      if (!ok) atomicOr(&s_bad, 2);
    }
    scan3(v, sum, part);
    if (b < p.B) {
      s_row[b] = sat_add(carry[0], v[0]);
      s_new[b] = sat_add(carry[1], v[1]);
      s_item[b] = sat_add(carry[2], v[2]);
    }
    for (int i = 0; i < 3; ++i) carry[i] = sat_add(carry[i], sum[i]);
  }
  __syncthreads();
  int bad = s_bad;
  if (carry[0] > p.M || (p.chunk && carry[2] > p.nwork)) bad |= 2;
  if (!bad && carry[1] > nfree) bad = 1;
  if (bad) {  // (uniform) nothing is taken: a call without rows
    for (int b = tid; b < p.B; b += nt) s_row[b] = s_new[b] = s_item[b] = 0;
    carry[0] = carry[1] = carry[2] = 0;
    if (tid == 0 && p.fault) atomicOr(p.fault, bad);
  }
  if (tid == 0) {
    s_row[p.B] = carry[0];
    s_new[p.B] = carry[1];
    s_item[p.B] = carry[2];
  }
  __syncthreads();
  for (int b = tid; b <= p.B; b += nt) {
    p.row0[b] = s_row[b];
    p.item0[b] = s_item[b];
    if (b < p.B) {
      const int s = p.slot[b];
      p.after[b] = s >= 0 && s < p.slots ? p.seen[s] + s_row[b + 1] - s_row[b] : 0;
    }
  }
  if (tid == 0) {
    *p.left = nfree - carry[1];
    *p.status = bad;
  }
  for (int t = tid; t < carry[1]; t += nt) {  // the new pages
    const int b = find_seq(s_new, p.B, t), s = p.slot[b];
    p.table[(size_t)s * p.ldt + ((p.seen[s] + page - 1) >> p.k) + t - s_new[b]] = p.free_ids[nfree - 1 - t];
  }
  __syncthreads();  // the table, `after` and everybody's reading of the lengths
  if (p.commit && !bad) {
    for (int b = tid; b < p.B; b += nt) p.seen[p.slot[b]] = p.after[b];
    if (tid == 0) *p.nfree = nfree - carry[1];
  }
  if (!rows_here) return;
  for (int m = tid; m < p.M; m += nt) row_out(p, s_row, s_item, m);
  if (p.chunk)
    for (int t = carry[2] + tid; t < p.nwork; t += nt) item_pad(p, t);
}

// the rows and work items of a call, one per thread, from what the sums left behind
__global__ __launch_bounds__(256) void pages_rows_kernel(ExtendParams p) {
  const int t = blockIdx.x * 256 + threadIdx.x;
  if (t < p.M) row_out(p, p.row0, p.item0, t);
  if (p.chunk && t < p.nwork && t >= p.item0[p.B]) item_pad(p, t);
}

struct ReleaseParams {
  const int* slot;
  int B;
  int *seen, *table;
  int slots, ldt;
  int *free_ids, *nfree;
  int cap, k;
  int *status, *fault;
};

__global__ __launch_bounds__(kPlanThreads) void pages_release_kernel(ReleaseParams p) {
  extern __shared__ int lds[];
  int* s_new = lds;  // [B + 1]
  unsigned* s_used = reinterpret_cast<unsigned*>(s_new + p.B + 1);
  __shared__ int s_bad;
  __shared__ int4 part[kPlanThreads / 64];
  const int tid = threadIdx.x, nt = blockDim.x, page = 1 << p.k;
  for (int i = tid; i < (p.slots + 31) / 32; i += nt) s_used[i] = 0;
  if (tid < kPlanThreads / 64) part[tid] = make_int4(0, 0, 0, 0);
  if (tid == 0) s_bad = 0;
  const int nfree = *p.nfree;
  __syncthreads();
  int carry = 0;
  for (int b0 = 0; b0 < p.B; b0 += nt) {
    const int b = b0 + tid;
    int v[3] = {0, 0, 0}, sum[3];
    if (b < p.B) {
      const int s = p.slot[b];
      bool ok = s >= 0 && s < p.slots;
      if (ok) {
        const unsigned bit = 1u << (s & 31);
        if (atomicOr(&s_used[s >> 5], bit) & bit) ok = false;
        const int L = p.seen[s];
        if (L < 0 || L > kMaxTokens || ((L + page - 1) >> p.k) > p.ldt) ok = false;
        else v[0] = (L + page - 1) >> p.k;
      }
      if (!ok) atomicOr(&s_bad, 2);
    }
    scan3(v, sum, part);
    if (b < p.B) s_new[b] = sat_add(carry, v[0]);
    carry = sat_add(carry, sum[0]);
  }
  if (tid == 0) s_new[p.B] = carry;
  __syncthreads();
  const bool bad = s_bad || nfree < 0 || nfree > p.cap || carry > p.cap - nfree;  // (uniform)
  if (tid == 0) {
    *p.status = bad ? 2 : 0;
    if (bad && p.fault) atomicOr(p.fault, 2);
  }
  if (bad) return;
  for (int t = tid; t < carry; t += nt) {
    const int b = find_seq(s_new, p.B, t), s = p.slot[b];
    int* at = p.table + (size_t)s * p.ldt + t - s_new[b];
    p.free_ids[nfree + t] = *at;
    *at = -1;
  }
  for (int b = tid; b < p.B; b += nt) p.seen[p.slot[b]] = 0;
  if (tid == 0) *p.nfree = nfree + carry;
}

static int page_log2(int page) {
  for (int k = 4; k <= 8; ++k)
    if (page == 1 << k) return k;
  return 0;
}

}  // namespace llj

using namespace llj;

extern "C" {

int llj_pages_extend(const int* slot, const int* add, int B, int* seen, int slots, int* table, int ldt, const int* free_ids, int* nfree,
                     int cap, int page, int commit, int* row0, int* item0, int* row_seq, int* pos, int* place, int M, int* work, int nwork,
                     int chunk, int* after, int* left, int* status, int* fault, void* stream) {
  const int k = page_log2(page);
  LLJ_REQUIRE(slot && seen && table && free_ids && nfree && row0 && item0 && after && left && status && k && B >= 1 && B <= kMaxSeqs &&
              slots >= 1 && slots <= kMaxSlots && ldt >= 1 && ldt <= (1 << 30 >> k) && cap >= 1 && cap <= (1 << 30 >> k) && M >= 0 &&
              M <= 1 << 28 && (M == 0 || (row_seq && pos && place)) && chunk >= 0 && (chunk == 0 || (work && nwork >= 0 && nwork <= 1 << 28)));
  ExtendParams p{slot, add, B, seen, table, slots, ldt, free_ids, nfree, cap, k, commit, row0, item0, row_seq, pos, place, work, after, left,
                 status, fault, M, chunk ? nwork : 0, chunk};
  const int most = M > p.nwork ? M : p.nwork, here = most <= kFewRows;
  const size_t lds = ((size_t)3 * (B + 1) + (slots + 31) / 32) * 4;
  hipStream_t s = (hipStream_t)stream;
  // few sequences, pages and rows: fewer waves to start and to wait for at the barriers
  const int work_here = here ? most : M >> k, want = B > work_here ? B : work_here, nt = want <= 64 ? 64 : want <= 256 ? 256 : kPlanThreads;
  hipLaunchKernelGGL(pages_extend_kernel, dim3(1), dim3(nt), lds, s, p, here);
  if (!here) hipLaunchKernelGGL(pages_rows_kernel, dim3((most + 255) / 256), dim3(256), 0, s, p);
  LLJ_CHECK_LAUNCH();
  return 0;
}

int llj_pages_release(const int* slot, int B, int* seen, int slots, int* table, int ldt, int* free_ids, int* nfree, int cap, int page, int* status,
                      int* fault, void* stream) {
  const int k = page_log2(page);
  LLJ_REQUIRE(slot && seen && table && free_ids && nfree && status && k && B >= 1 && B <= kMaxSeqs && slots >= 1 && slots <= kMaxSlots &&
              ldt >= 1 && ldt <= (1 << 30 >> k) && cap >= 1 && cap <= (1 << 30 >> k));
  ReleaseParams p{slot, B, seen, table, slots, ldt, free_ids, nfree, cap, k, status, fault};
  const size_t lds = ((size_t)(B + 1) + (slots + 31) / 32) * 4;
  hipLaunchKernelGGL(pages_release_kernel, dim3(1), dim3(kPlanThreads), lds, (hipStream_t)stream, p);
  LLJ_CHECK_LAUNCH();
  return 0;
}

}  // extern "C"
