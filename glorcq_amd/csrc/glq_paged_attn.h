// What the two forms of paged attention share: a few query rows
// (glq_paged_attn.hip) and many (glq_paged_prompt.hip).
#pragma once

#include "glq_handoff.h"
#include "glq_paged.h"

namespace glq {

constexpr int kPaRows = 16;      // query rows (tokens x the KV head's q heads) of the first form's unit
constexpr int kPpRows = 128;     // of the second form's
// A sequence with more rows a KV head takes the second form.  The first one
// reads a sequence's pages once for each 16 rows; the second once for 128, but
// computes as if it had them all.  us of the first | second form, 8-bit pages,
// with 32, 64 and 128 rows: 8 sequences of 4000 positions and 4 KV heads 25 |
// 24, 30 | 27, 41 | 32; 64 of 1000 29 | 32, 49 | 34, 73 | 37; 8 of 3000 and 16
// KV heads 28 | 42, 44 | 45, 134 | 53.
constexpr int kPaMostRows = 32;

struct PagedAttnArgs {
  PagedView c;
  const __half* q;  // (T, Hq, D)
  __half* out;      // (T, Hq D)
  float* part;      // parts of units: o, m, l of a row in D + 4
  unsigned* count;  // [unit], zero between calls (first form)
  int rep, window, sinks, slots_each, rows;
  int slots, splits, split_steps, fold;  // second form
  float scale2;                    // scale log2(e)
};

// The query rows of a unit, one a lane, and the positions they see.
struct RowSet {
  int first;         // position of the sequence's first new token
  int s0, n;         // its rows of q
  int row;           // this lane's row: token row / rep, head row % rep
  bool live;
  int lo, hi;        // positions this lane's row sees: [lo, hi)
  int lo_all, hi_all, lo_any, hi_any;  // seen by all rows, by any
  int cap;           // positions of the page table
};

// Sets r for the R rows from r0 on of sequence b's n new tokens, row r0 + li.
template <int R>
__device__ __forceinline__ void set_rows(RowSet& r, const PagedView& c, int b, int r0, int rep,
                                         int window, int li) {
  r.s0 = c.start(b);
  r.n = max((c.starts ? c.start(b + 1) : r.s0 + c.each) - r.s0, 0);
  r.first = c.length(b) - r.n;
  r.cap = c.max_pages << c.page_shift;
  const int rows = r.n * rep, r1 = min(r0 + R, rows) - 1;
  r.live = r0 + li < rows;
  r.row = min(r0 + li, rows - 1);
  auto lo = [&](int pos) { return window > 0 ? max(pos - window + 1, 0) : 0; };
  auto hi = [&](int pos) { return min(max(pos + 1, 0), r.cap); };
  const int pos = r.first + r.row / rep;
  r.lo = lo(pos);
  r.hi = hi(pos);
  r.lo_any = lo(r.first + r0 / rep);
  r.hi_all = hi(r.first + r0 / rep);
  r.lo_all = lo(r.first + r1 / rep);
  r.hi_any = hi(r.first + r1 / rep);
}

// The n tiles of TP positions of which some row sees one, numbered from `begin`
// on: those of positions [lo, hi), a window's or all; with SINKS those of the
// sinks before them, as far as they lie before lo's.  (Without sinks a number is
// the tile's place: as one kernel for both, calls without took 1.5 to 3.5 % more.)
template <int TP, bool SINKS>
struct Span {
  int begin, n, sink = 0, skip = 0;
  __device__ Span(int lo, int hi, int sinks) {
    const int first = lo / TP;
    begin = first;
    n = max((hi + TP - 1) / TP - first, 0);
    if constexpr (SINKS) {
      begin = 0;
      sink = min((sinks + TP - 1) / TP, first);
      skip = first - sink;
      n += sink;
    }
  }
  __device__ int place(int t) const {
    if constexpr (SINKS)
      return t < sink ? t : t + skip;
    else
      return t;
  }
};

// 4 columns of a row's result to memory.
__device__ __forceinline__ void store_row(__half* dst, f32x4 v, float den, int pos, int cap) {
  const float inv = 1.f / den;
  f16x2 y[2];
#pragma unroll
  for (int e = 0; e < 4; ++e)
    y[e >> 1][e & 1] = (_Float16)(pos < 0 ? 0.f : pos >= cap ? __builtin_nanf("") : v[e] * inv);
  *(uint2*)dst = uint2{__builtin_bit_cast(uint32_t, y[0]), __builtin_bit_cast(uint32_t, y[1])};
}

// Merges pieces (m, l, o) of a row's attention, 4 columns a thread.
struct Merge {
  float M = -__builtin_inff(), den = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  __device__ void add(float m, float l, f32x4 v) {
    const float Mn = fmaxf(M, m), Mf = Mn == -__builtin_inff() ? 0.f : Mn;
    const float fo = __builtin_amdgcn_exp2f(M - Mf), fn = __builtin_amdgcn_exp2f(m - Mf);
    den = den * fo + l * fn;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = o[e] * fo + v[e] * fn;
    M = Mn;
  }
};

// Launches the second form over the batch's sequences of more than kPaMostRows
// rows (with starts; of all sequences otherwise).
int paged_prompt_launch(PagedAttnArgs a, int head_dim, hipStream_t stream);
int64_t paged_prompt_scratch_bytes(int64_t seqs, int64_t tokens, int64_t q_heads, int64_t kv_heads);

}  // namespace glq
