// Paged key/value cache: what the append and the attention kernels share.
//
// The cache of one layer is a pool of pages of `page` tokens (a power of two,
// 16 .. 1024); a sequence's pages lie anywhere in it, page_table[b][i] naming
// the one of its positions [i page, (i + 1) page).  A KV head's part of a page
// is made of 16-token blocks:
//   k (pages, Hk, page, D)             a token's D values side by side
//   v (pages, Hk, page / 16, D, 16)    a block's 16 values of a column side by side
// so that both are read in the order in which the matrix instructions take
// them: a score sums over D, the weighted sum of V over the positions, and
// neither operand is transposed on its way.  Values are fp16, or 8 bits: e4m3
// codes with one scale 2^(byte - 127) (e8m0) for each block of 16 tokens and
// KV head, of its own for k and v.
#pragma once

#include <hip/hip_fp16.h>

#include "glq_gemv_core.h"
#include "glq_internal.h"

namespace glq {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

constexpr int kBlkTokens = 16;  // tokens of a block: one scale each for k and v

struct PagedView {
  void *k, *v;
  uint8_t *ks, *vs;  // null: fp16 pages
  const int* table;
  int64_t table_stride;
  const int* lengths;
  const int* starts;  // null: `each` tokens a sequence
  int B, pages, max_pages, Hk, page_shift, T, each;

  __device__ int start(int b) const {
    return starts ? min(max(starts[b], 0), T) : b * each;
  }
  __device__ int length(int b) const { return max(lengths[b], 0); }
  // Page of a sequence's page index, -1 for an index or an id out of range.
  __device__ int page_of(int b, int i) const {
    if (i < 0 || i >= max_pages) return -1;
    const int p = table[b * table_stride + i];
    return p >= 0 && p < pages ? p : -1;
  }
};

// A ragged batch's work units, numbered on the host without its starts:
// sequence b's units are the slots from floor(start(b) mul / div) + add b on,
// which leaves it floor(new mul / div) + add at least.  Returns the sequence
// of a slot and makes the slot its unit's number.
__device__ __forceinline__ int slot_sequence(const PagedView& c, int mul, int div, int add,
                                             int& slot) {
  int lo = 0, hi = c.B - 1;
  auto base = [&](int b) { return (int)((int64_t)c.start(b) * mul / div) + add * b; };
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (base(mid) <= slot)
      lo = mid;
    else
      hi = mid - 1;
  }
  slot -= base(lo);
  return lo;
}

// e8m0 scale: its value (0xFF: NaN) and its exponent as a float.
__device__ __forceinline__ float e8m0_value(int byte) {
  return __int_as_float(byte == 255 ? 0x7FC00000 : byte == 0 ? 0x00400000 : byte << 23);
}
__device__ __forceinline__ float e8m0_exponent(int byte) {
  return byte == 255 ? __builtin_nanf("") : (float)(byte - 127);
}

// 4 e4m3 codes -> 4 fp16 values (exact).
__device__ __forceinline__ void fp8_to_f16(uint32_t w, f16x2& a, f16x2& b) {
  a = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, 1.0f, false));
  b = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, 1.0f, true));
}
__device__ __forceinline__ f16x8 fp8x8_to_f16(uint32_t w0, uint32_t w1) {
  f16x2 a, b, c, d;
  fp8_to_f16(w0, a, b);
  fp8_to_f16(w1, c, d);
  return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Orders LDS accesses of one wave's lanes among themselves.
__device__ __forceinline__ void paged_lds_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Whether two ranges of bytes have none in common.
inline bool apart(const void* a, int64_t an, const void* b, int64_t bn) {
  return (uintptr_t)a + an <= (uintptr_t)b || (uintptr_t)b + bn <= (uintptr_t)a;
}

// Whether n rows of `row` bytes, `stride` >= row apart, and a range of bytes
// have none in common.
inline bool rows_apart(const void* rows, int64_t row, int64_t stride, int64_t n, const void* b,
                       int64_t bn) {
  const int64_t lo = (int64_t)((uintptr_t)b - (uintptr_t)rows), hi = lo + bn;
  const int64_t i = lo < row ? 0 : (lo - row) / stride + 1;  // the first row that ends past lo
  return i >= n || i * stride >= hi;
}

// Checks a cache and its batch and fills the kernels' view of them (the pages
// themselves may be null in a batch of no tokens).
int paged_view(const glq_paged_cache* c, const int32_t* starts, int64_t tokens, PagedView& view);

}  // namespace glq
