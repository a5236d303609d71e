// Attention over the paged 4-bit cache: what its kernels share.
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
  float sl2;  // scale in units of log2
  float* part;
  int* count;
  int nsplit;
};

// fp32 pairs as NP bf16 terms (1: rounded; 2: hi + lo, 16 bits; 3: all 24)
template <int NP>
__device__ __forceinline__ void split_pair(float a, float b, uint32_t (&o)[NP]) {
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    o[i] = pack2bf(a, b);
    a -= bflo(o[i]);
    b -= bfhi(o[i]);
  }
}

// A codes' word as four bf16 pairs 16 + c, values (j, j + 4) in word j: bits 3 .. 6 of 0x4180 are the units of bf16s from 16 on
__device__ __forceinline__ u32x4 codes8(uint32_t w, uint32_t mask, uint32_t base) {
  return u32x4{and_or(w << 3, mask, base), and_or(w >> 1, mask, base), and_or(w >> 5, mask, base), and_or(w >> 9, mask, base)};
}
constexpr uint32_t kCodeMask = 0x00780078u, kCodeBase = 0x41804180u;

// max over the four 16-lane groups of the wave, lane by lane
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

int kv4_flash(const Kv4Attend& p, int dt, hipStream_t s);

}  // namespace llj
