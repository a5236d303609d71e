// Paged K / V cache in 4 bits. A head's key or value x of n values is held as codes c in 0 .. 15, a bf16 scale s and a bf16 offset o,
// and stands for c s + o:
//   o = the largest bf16 up to min x,  s = bf16(fp32((max x - o) / 15)),  c = clamp(rne((x - o) / s), 0, 15), 0 where s is 0.
// (o and s in bf16: 4 bytes beside n / 2. Rounding o down keeps every value at or above it, so it costs no range; s rounded to 8 bits is off by at
// most 2^-9, 15 steps of it 0.03 of a step.) A vector that is not finite, or begins below bf16's range, is s = o = NaN.
// A block, one head's part of a page of P tokens:
//   [key codes P x Dp / 2 | value codes P x Vp / 2 | key (s, o) P x 4 | value (s, o) P x 4] bytes,
// Dp, Vp = 64, 128 or 256 (codes of zero behind D, V); value i of a vector in bits 4 (i % 8) of its word i / 8. Pool: [pages][heads] blocks.
#pragma once
#include "common.h"

namespace llj {

__host__ __device__ constexpr int kv4_width(int n) { return n <= 64 ? 64 : n <= 128 ? 128 : 256; }
__host__ __device__ constexpr int kv4_block(int page, int Dp, int Vp) { return page * ((Dp + Vp) / 2 + 8); }

struct Kv4Pool {
  uint8_t* p;
  int pages, G, k;       // 2^k tokens a page
  int vc, ks, vs, blk;   // offsets of the value codes, the key pairs and the value pairs in a block; its bytes
};

static inline Kv4Pool kv4_pool(void* p, int pages, int G, int k, int D, int V) {
  const int page = 1 << k, Dp = kv4_width(D), Vp = kv4_width(V);
  const int vc = page * Dp / 2, ks = vc + page * Vp / 2;
  return Kv4Pool{(uint8_t*)p, pages, G, k, vc, ks, ks + 4 * page, kv4_block(page, Dp, Vp)};
}

static inline int kv4_page_log2(int page) {
  for (int k = 4; k <= 8; ++k)
    if (page == 1 << k) return k;
  return 0;
}

// sizes every entry point takes; places stay below 2^31
static inline bool kv4_sizes(const void* pool, int pages, int page, int G, int D, int V, int dt) {
  const int k = kv4_page_log2(page);
  return pool && ((uintptr_t)pool & 15) == 0 && k && pages >= 1 && pages <= (1 << 30 >> k) && G >= 1 && G <= 4096 && D >= 1 && D <= 256 && V >= 1 &&
         V <= 256 && (dt == 0 || dt == 1);
}

}  // namespace llj
