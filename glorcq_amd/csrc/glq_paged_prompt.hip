// Causal attention of prompts and chunks of prompts over a paged key/value
// cache (layout and formats: glq_paged.h).

#include <algorithm>
#include <type_traits>

#include "glq_paged_attn.h"

namespace glq {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));

__device__ __forceinline__ f32x16 mfma_32x32x16(f16x8 a, f16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// The larger of a lane's value and that of the lane 32 away.
__device__ __forceinline__ float halves_max(float x) {
  const auto r =
      __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

constexpr int kPpThreads = 256;
constexpr int kPpStep = 32;    // positions of a step: two blocks
constexpr int64_t kPpParts = 2048;  // of units in several, at most: 138 MB
constexpr float kPpLag = 8.f;  // log2 by which a score may pass the running maximum

// One workgroup takes 128 query rows (tokens x the KV head's q heads) of one KV
// head, 32 a wave, over the positions they see (or a split of them), 32 a step:
//   S^T = K Q^T   v_mfma_f32_32x32x16_f16, A = 32 positions of K, B = the rows
//   O^T += V^T P^T                         A = 32 columns of V,   B = the weights
// so that a row of the softmax is a column of both products: its 32 scores of
// a step lie on two lanes, and the weights are the second product's operand as
// they stand.  K and V go through LDS as fp16, decoded once for the four waves,
// in the order of the operands (16-byte pieces, conflict-free both ways).
//
// Three steps are worked on at once, so that matrix and vector instructions of
// a wave have nothing to wait for from each other: step u's exponentials beside
// the scores of u + 2 and the weighted V of u - 1, a vector instruction or four
// between two matrix ones; and the maximum of u + 1 and the way of K of u + 3
// and V of u to LDS with them.  The bytes of two steps more are in flight.
//
// Bound by the waves' instruction streams: of a CU's 2400 to 2700 cycles for two
// workgroups' steps the matrix pipe is busy for 43 % and the vector unit, with
// the issue of matrix instructions, for 63 % of each SIMD's, LDS for 38 %, and
// two waves a SIMD leave gaps between them (a step of a workgroup alone on its
// CU takes 1800, one wave's time to issue it).  4096 tokens of 32 and 4 heads:
// 158 to 189 us, 730 to 870 TF/s of what the mask leaves; 512 behind 30000: 271
// to 301 us, 840 to 940 TF/s (on several cards; on one of them a prompt takes 163
// us between other work, 177 in a row with its like).  A library product of
// 8192^3 reaches 1143 TF/s, these matrix instructions alone 1190.
//
// Softmax: the running maximum m of t + e (e the exponent of V's block, as in
// the first form) follows the scores only when one passes it by more than
// 2^kPpLag: weights up to 2^8 lose nothing, in fp16 or in the fp32 sums, and
// the 64 sums of O a lane are rarely scaled.  Weights are rounded to fp16 for
// the product with V (exact ones would take a second product; V's codes are exact in
// it), not in the denominator; no weight is 1 here as the largest of the first
// form is, so this shows: outputs are 2.9e-4 off the exact ones (root mean
// square, relative), 2.1e-4 of it their own rounding to fp16.
template <int D, bool FP8>
struct PromptStage {
  static constexpr int S = FP8 ? 1 : 2;             // bytes of a value
  static constexpr int PB = FP8 && D == 64 ? 8 : 16;  // bytes of a piece
  static constexpr int KC = D * S / PB;             // pieces of a K row
  static constexpr int VC = 16 * D * S / PB;        // pieces of a V block
  static constexpr int KP = kPpStep * KC / kPpThreads;  // pieces of K, and of V, a thread
  static constexpr int kParts = FP8 && D == 128 ? 2 : KP;  // in which they go to LDS

  using Piece = std::conditional_t<PB == 8, u32x2, u32x4>;
  // Steps whose bytes are in flight, each in registers of its own (pieces of
  // fp16 heads of 128 have none left for two).
  static constexpr int kSets = KP * PB / 4 > 4 ? 1 : 2;
  Piece k[kSets][KP], v[kSets][KP];
  int wave;  // uniform

  // A wave's pieces of a pass lie in one block, K's and V's in the same, so
  // that addresses are scalars but for a lane's constant part.
  static constexpr int NB = KP;  // blocks of a step that a wave fetches of
  __device__ int block(int j) const { return KP == 2 ? j : wave >> 1; }

  // What a step needs to know of its two blocks, of 64 steps, a step a lane: a
  // step finds its own in registers and waits for none.  at: places of the
  // wave's blocks in the pools, in bytes; ks: scale of the scores; ev: exponent
  // of V's scale.
  int base;
  uint32_t at_lo[NB], at_hi[NB];
  float ks[2], ev[2];
  __device__ void look_up(const PagedView& c, int b, int g, float scale2, int step) {
    const int s = c.page_shift - 4;
    base = step;
    int page[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int blk = 2 * (step + (int)(threadIdx.x & 63)) + k;
      const int p = c.table[b * c.table_stride + min(blk >> s, c.max_pages - 1)];
      const bool bad = (unsigned)p >= (unsigned)c.pages;  // page 0 is read, its scores are NaN
      page[k] = bad ? 0 : p;
      ks[k] = scale2;
      ev[k] = 0.f;
      if constexpr (FP8) {
        const int64_t at = place(c, g, page[k], blk);
        ks[k] = e8m0_value(c.ks[at]) * scale2;
        ev[k] = e8m0_exponent(c.vs[at]);
      }
      // not 0, which times the -inf of a score that a row does not see is NaN; to
      // scores, of up to 2^39, 2^-126 is one
      if (ks[k] < 0x1p-126f) ks[k] = 0x1p-126f;
      if (bad) ks[k] = __builtin_nanf("");
    }
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      const int blk = 2 * (step + (int)(threadIdx.x & 63)) + block(j);
      const int64_t at = place(c, g, block(j) ? page[1] : page[0], blk) * (16 * D * S);
      at_lo[j] = (uint32_t)at;
      at_hi[j] = (uint32_t)(at >> 32);
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) asm volatile("" : "+v"(ks[k]), "+v"(ev[k]));  // (waits for them)
  }
  __device__ static int64_t place(const PagedView& c, int g, int p, int blk) {
    const int s = c.page_shift - 4;
    return ((int64_t)p * c.Hk + g << s) + (blk & ((1 << s) - 1));
  }
  __device__ static float lane_value(float x, int lane) {
    return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x), lane));
  }
  __device__ const char* block_of(const void* pool, int step, int j) const {
    const uint32_t lo = __builtin_amdgcn_readlane(at_lo[j], step - base);
    const uint32_t hi = __builtin_amdgcn_readlane(at_hi[j], step - base);
    return (const char*)pool + ((uint64_t)hi << 32 | lo);
  }
  template <int SET>
  __device__ void load_k(const PagedView& c, int step) {
    // (a pass's rows are a block's, or start at a block)
    const unsigned lane = (threadIdx.x / KC & 15) * (D * S) + PB * (threadIdx.x % KC);
#pragma unroll
    for (int j = 0; j < KP; ++j) k[SET][j] = *(const Piece*)(block_of(c.k, step, j) + lane);
  }
  template <int SET>
  __device__ void load_v(const PagedView& c, int step) {
    const unsigned lane = threadIdx.x % VC * PB;
#pragma unroll
    for (int j = 0; j < KP; ++j) v[SET][j] = *(const Piece*)(block_of(c.v, step, j) + lane);
  }

  // LDS places in halves.  K: values 8 d8 .. + 8 of a position at (d8,
  // position), 32 bytes between pairs of d8 so that a row's pieces go to
  // different banks as they are stored (between single d8, the two lane halves
  // of a read collide: half of the LDS cycles); V: 8 values at (block, half,
  // column), half 0 the block's positions 0-3 and 8-11, as lane halves hold them.
  static constexpr int kKPair = 2 * kPpStep * 8 + 16;
  __device__ static int k_at(int d8, int pos) {
    return (d8 >> 1) * kKPair + (d8 & 1) * (kPpStep * 8) + pos * 8;
  }
  static constexpr int kV = D / 16 * kKPair;  // where V begins
  __device__ static int v_at(int blk, int half, int d) { return kV + ((blk * 2 + half) * D + d) * 8; }
  static constexpr int kBytes = 2 * (kV + kPpStep * D);  // of a step

  __device__ static void store_k(_Float16* buf, const Piece (&k)[KP], int part) {
    const int j = KP == 2 ? part : 0, p = kPpThreads * j + threadIdx.x, row = p / KC, n = p % KC;
    if constexpr (!FP8)
      *(Piece*)(buf + k_at(n, row)) = k[j];
    else if constexpr (PB == 8)
      *(f16x8*)(buf + k_at(n, row)) = fp8x8_to_f16(k[0][0], k[0][1]);
    else
      *(f16x8*)(buf + k_at(2 * n + part, row)) = fp8x8_to_f16(k[0][2 * part], k[0][2 * part + 1]);
  }
  __device__ static void store_v(_Float16* buf, const Piece (&v)[KP], int part) {
    const int j = KP == 2 ? part : 0, p = kPpThreads * j + threadIdx.x, blk = p / VC, n = p % VC;
    if constexpr (FP8 && PB == 16) {  // a column of the block
      *(f16x8*)(buf + v_at(blk, part, n)) = fp8x8_to_f16(v[0][part], v[0][part + 2]);
    } else {  // positions 8 (n & 1) .. + 8 of column n / 2
      u32x4 x;
      if constexpr (FP8)
        x = __builtin_bit_cast(u32x4, fp8x8_to_f16(v[0][0], v[0][1]));
      else
        x = v[j];
      *(u32x2*)(buf + v_at(blk, 0, n >> 1) + 4 * (n & 1)) = u32x2{x[0], x[1]};
      *(u32x2*)(buf + v_at(blk, 1, n >> 1) + 4 * (n & 1)) = u32x2{x[2], x[3]};
    }
  }
  // Of a word of values, the top bit of each infinity or NaN (with kOdd).
  static constexpr uint32_t kOdd = FP8 ? 0x80808080u : 0x80008000u;
  __device__ static uint32_t odd_values(uint32_t w) {
    // (the largest exponent field carries into the sign's place)
    return FP8 ? (w & 0x7F7F7F7Fu) + 0x01010101u : (w & 0x7FFF7FFFu) + 0x04000400u;
  }
  __device__ static uint32_t odd_in(const Piece& v) {
    uint32_t any = 0;
#pragma unroll
    for (int e = 0; e < PB / 4; ++e) any |= odd_values(v[e]);
    return any;
  }
  // Infinities and NaN go into LDS as zeros (weight 0 times one that a row does
  // not see is not 0; they are added afterwards): V again, where it has any.
  __device__ static void store_v_finite(_Float16* buf, const Piece (&v)[KP]) {
    Piece u[KP];
#pragma unroll
    for (int j = 0; j < KP; ++j)
#pragma unroll
      for (int e = 0; e < PB / 4; ++e) {
        const uint32_t x = (odd_values(v[j][e]) & kOdd) >> (FP8 ? 7 : 15);
        u[j][e] = v[j][e] & ~(x * (FP8 ? 0xFFu : 0xFFFFu));
      }
#pragma unroll
    for (int i = 0; i < kParts; ++i) store_v(buf, u, i);
  }
};

// Adds the infinities and NaN of V that the row of a lane sees, at positions of
// steps [u0, u1), to its sums: rare, and so a plain walk over the blocks.
template <int D, bool FP8>
__device__ void add_odd_values(f32x16 (&o)[D / 32], const PagedView& c, int b, int g, int u0,
                               int u1, const RowSet& r) {
  using Stage = PromptStage<D, FP8>;
  constexpr int S = FP8 ? 1 : 2, NG = D / 32;
  const int lane = threadIdx.x & 63, half = lane >> 5;
  for (int blk = 2 * u0; blk < 2 * u1; ++blk) {
    const int p = c.page_of(b, blk >> (c.page_shift - 4));
    if (p < 0) continue;  // (the scores are NaN there)
    const char* base = (const char*)c.v + Stage::place(c, g, p, blk) * (16 * D * S);
    uint32_t here = 0;  // positions of the block with one
    for (int d = lane; d < D; d += 64)
#pragma unroll
      for (int i = 0; i < 4 * S; ++i) {
        const uint32_t x = Stage::odd_values(((const uint32_t*)(base + d * 16 * S))[i]) & Stage::kOdd;
        if constexpr (FP8)
          here |= (x >> 7 & 1 | x >> 14 & 2 | x >> 21 & 4 | x >> 28 & 8) << (4 * i);
        else
          here |= (x >> 15 & 1 | x >> 30 & 2) << (2 * i);
      }
#pragma unroll
    for (int k = 32; k >= 1; k >>= 1) here |= __shfl_xor((int)here, k);
    here = __builtin_amdgcn_readfirstlane(here);
    bool all_nan = true;
    while (here) {
      const int j = __builtin_ctz(here), pos = 16 * blk + j;
      here &= here - 1;
      const bool sees = pos >= r.lo && pos < r.hi;
#pragma unroll
      for (int n = 0; n < NG; ++n)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int d = 32 * n + 8 * (e >> 2) + 4 * half + (e & 3);
          float x;
          if constexpr (FP8)
            x = (((const uint8_t*)base)[d * 16 + j] & 0x7F) == 0x7F ? __builtin_nanf("") : 0.f;
          else
            x = (float)((const _Float16*)base)[d * 16 + j];
          if (sees && !(fabsf(x) < __builtin_inff())) o[n][e] += x;
        }
    }
#pragma unroll
    for (int n = 0; n < NG; ++n)
#pragma unroll
      for (int e = 0; e < 16; ++e) all_nan &= o[n][e] != o[n][e];
    if (__builtin_amdgcn_ballot_w64(!all_nan && r.live) == 0) return;
  }
}

// Parts of a unit of so many steps.
__device__ __forceinline__ int split_parts(const PagedAttnArgs& a, int steps) {
  return min(max(steps / a.split_steps, 1), a.splits);
}

template <int D, bool FP8>
__global__ __launch_bounds__(kPpThreads) __attribute__((amdgpu_waves_per_eu(2, 2)))
void paged_prompt_kernel(PagedAttnArgs a) {
  using Stage = PromptStage<D, FP8>;
  constexpr int NG = D / 32, KS = D / 16, PS = D + 4, kOps = KS + 2 * NG;
  extern __shared__ __align__(16) unsigned char smem[];
  _Float16* bufs = (_Float16*)smem;  // 2 x Stage::kBytes
  __shared__ int odds[2][kPpThreads / 64];
  const PagedView& c = a.c;
  // KV head fastest, then the unit, the last rows of a sequence, which see most,
  // first (from `fold` on the first rows first); the split last, so that those
  // that a unit does not have are the grid's end (between others, they leave
  // whole dies without work).
  int id = blockIdx.x;
  const int g = id % c.Hk;
  id /= c.Hk;
  const int split = id / a.slots;
  int slot = a.slots - 1 - id % a.slots, b;
  if (slot < a.slots - a.fold) slot = a.slots - a.fold - 1 - slot;
  const int slot0 = slot;
  if (c.starts) {
    b = slot_sequence(c, a.rep, kPpRows, 1, slot);
  } else {
    b = slot / a.slots_each;
    slot -= b * a.slots_each;
  }
  const int tid = threadIdx.x, lane = tid & 63, col = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  b = __builtin_amdgcn_readfirstlane(b);
  slot = __builtin_amdgcn_readfirstlane(slot);
  RowSet r;
  set_rows<kPpRows>(r, c, b, slot * kPpRows, a.rep, a.window, 0);
  const int rows = r.n * a.rep;
  if (slot < 0 || slot * kPpRows >= rows || (c.starts && rows <= kPaMostRows)) return;  // uniform
  // the unit's steps, and this split's of them
  int u0 = r.lo_any / kPpStep, u1 = (r.hi_any + kPpStep - 1) / kPpStep;
  const int parts = split_parts(a, u1 - u0);
  if (split >= parts) return;  // uniform
  if (parts > 1) {
    const int per = (u1 - u0 + parts - 1) / parts;
    u0 += split * per;
    u1 = min(u1, u0 + per);
  }
  const int r0 = slot * kPpRows + 32 * wave;
  set_rows<32>(r, c, b, min(r0, rows - 1), a.rep, a.window, col);
  r.live = r0 + col < rows;
  const int Hq = c.Hk * a.rep, tok = r.row / a.rep;

  f16x8 q[KS];
  {
    const f16x8* src =
        (const f16x8*)(a.q + ((int64_t)(r.s0 + tok) * Hq + g * a.rep + r.row % a.rep) * D);
    // the sign of the scale goes to q, so that a block's largest product has
    // its largest score; a scale of 0 too
    const _Float16 sign = (_Float16)(a.scale2 < 0.f ? -1.f : a.scale2 == 0.f ? 0.f : 1.f);
#pragma unroll
    for (int s = 0; s < KS; ++s) q[s] = src[2 * s + half];  // (a row that is none: the last one's)
#pragma unroll
    for (int s = 0; s < KS; ++s) q[s] *= r.live ? sign : (_Float16)0.f;
  }
  const float scale2 = a.scale2 == 0.f ? 1.f : fabsf(a.scale2);
  float m = -__builtin_inff(), l = 0.f;
  f32x16 o[NG], sa, sb, sc;
  f16x8 w[2] = {f16x8{}, f16x8{}};
  float ks[2], ev[2];  // the scales of the step whose exponentials are next
#pragma unroll
  for (int i = 0; i < NG; ++i) o[i] = f32x16{};

  Stage st;
  st.wave = wave;
  auto buf = [&](int j) { return bufs + (j & 1) * (Stage::kBytes / 2); };
  // the scores of a step, 16 of a row on a lane: positions 8 (e / 4) + 4 half + e % 4
  auto scores = [&](f32x16& s, int j) {
    s = f32x16{};
#pragma unroll
    for (int k = 0; k < KS; ++k)
      s = mfma_32x32x16(*(const f16x8*)(buf(j) + Stage::k_at(2 * k + half, col)), q[k], s);
  };
  // A step's scales, and its scores' masks where some row does not see all of
  // it: a position that a row does not see has no weight, whatever its block's
  // scale is, so a NaN goes from the scale to the scores.
  auto mask = [&](int j, f32x16& s, float (&ks)[2], float (&ev)[2]) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      ks[k] = Stage::lane_value(st.ks[k], u0 + j - st.base);
      ev[k] = Stage::lane_value(st.ev[k], u0 + j - st.base);
    }
    const int p0 = (u0 + j) * kPpStep;
    if (p0 < r.lo_all || p0 + kPpStep > r.hi_all) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const bool bad = ks[k] != ks[k] || ev[k] != ev[k];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int p = p0 + 16 * k + 8 * (e >> 2) + 4 * half + (e & 3);
          if (bad) s[8 * k + e] = __builtin_nanf("");
          if (p < r.lo || p >= r.hi) s[8 * k + e] = -__builtin_inff();
        }
        if (bad) {
          ks[k] = 1.f;
          ev[k] = 0.f;
        }
      }
    }
  };
  // m follows where a score has passed it by 2^kPpLag, in whole powers of two.
  // The weights in w, of up to 2^8, then keep what fp16 has of them: their
  // factor is applied in two, since as one fp16 value it is 0 from 2^-25 on
  // (down to 2^-16 it is the first alone; below 2^-40 nothing is left of w).
  auto follow = [&](float mx) {
    if (__builtin_amdgcn_ballot_w64(mx > m + kPpLag)) {  // (-inf + lag: any score passes)
      const float mn = fmaxf(m, ceilf(mx)), mf = mn == -__builtin_inff() ? 0.f : mn;
      const float d = m - mf, d0 = fmaxf(d, -16.f), d1 = fmaxf(d - d0, -24.f);
      const float f = __builtin_amdgcn_exp2f(d);
      const _Float16 f0 = (_Float16)__builtin_amdgcn_exp2f(d0);
      const _Float16 f1 = (_Float16)__builtin_amdgcn_exp2f(d1);
      m = mn;
      l *= f;
#pragma unroll
      for (int k = 0; k < 2; ++k) w[k] = w[k] * f0 * f1;
#pragma unroll
      for (int n = 0; n < NG; ++n)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[n][e] *= f;
    }
  };
  const int n = u1 - u0;
  // Step j: s0 its scores, s1 those of j + 1, s2 gets those of j + 2.  other(i):
  // what else the wave has to do, in kOps parts.
  auto step = [&](int j, f32x16& s0, f32x16& s1, f32x16& s2, auto other) {
    // the operands of the matrix instructions below, kAhead of them in flight:
    // in turn K's of the scores and V's
    constexpr int kAhead = 4, kEach = 16 / kOps;
    static_assert(KS == 2 * NG && kOps * kEach == 16, "as many of each");
    const _Float16 *kbuf = buf(j), *vbuf = buf(j - 1);
    auto operand = [&](int n) {
      return n & 1
                 ? *(const f16x8*)(vbuf + Stage::v_at(n / 2 / NG, half, 32 * (n / 2 % NG) + col))
                 : *(const f16x8*)(kbuf + Stage::k_at(n + half, col));
    };
    f16x8 op[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) op[i] = operand(i);
    __builtin_amdgcn_sched_barrier(0);
    float ks1[2], ev1[2];
    mask(j + 1, s1, ks1, ev1);
    const float mf = m == -__builtin_inff() ? 0.f : m;
    const float off[2] = {ev[0] - mf, ev[1] - mf};
    f16x8 wn[2];
    float sum[2] = {0.f, 0.f}, big[2] = {s1[0], s1[8]};
    s2 = f32x16{};
    // (the CU's other workgroup gets its turn between steps, not within: 5 %)
    __builtin_amdgcn_s_setprio(1);
    float last = 0.f;
    int late = 0;
#pragma unroll
    for (int i = 0; i < kOps; ++i) {
      if (i & 1)
        o[i / 2 % NG] = mfma_32x32x16(op[i % kAhead], w[i / 2 / NG], o[i / 2 % NG]);
      else
        s2 = mfma_32x32x16(op[i % kAhead], q[i / 2], s2);
      if (i + kAhead < kOps) op[i % kAhead] = operand(i + kAhead);
      other(i);
#pragma unroll
      for (int e = kEach * i; e < kEach * (i + 1); ++e) {
        const int k = e >> 3;
        float x = __builtin_amdgcn_exp2f(fmaf(s0[e], ks[k], off[k]));
        asm volatile("" : "+v"(x));  // (in this place)
        sum[late >> 3] += last;      // (of the one before: x takes a while)
        last = x;
        late = e;
        wn[k][e & 7] = (_Float16)x;
        if (e & 1) {
          big[k] = fmaxf(fmaxf(big[k], s1[e - 1]), s1[e]);
          asm volatile("" : "+v"(big[k]));
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_s_setprio(0);
    sum[1] += last;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      l = FP8 ? fmaf(sum[k], __builtin_amdgcn_exp2f(-ev[k]), l) : l + sum[k];
      w[k] = wn[k];
      ks[k] = ks1[k];
      ev[k] = ev1[k];
    }
    // (of the step past the last, its scores are of anything)
    if (j + 1 < n)
      follow(halves_max(fmaxf(fmaf(big[0], ks[0], ev[0]), fmaf(big[1], ks[1], ev[1]))));
  };

  // Before the loop: the scores of the first two steps, K of the third in LDS,
  // K of the fourth and V of the first in registers; zeros where the first step
  // looks for the V of the one before it.  Steps past the last are not fetched:
  // their scores, of what LDS held before, are not used.
  constexpr int kSets = Stage::kSets, kOther = kSets - 1;
  st.look_up(c, b, g, scale2, u0);
  {
    Stage s2 = st;
    st.template load_k<0>(c, u0);
    s2.template load_k<0>(c, u0 + 1);
#pragma unroll
    for (int i = 0; i < Stage::kParts; ++i) {
      Stage::store_k(buf(0), st.k[0], i);
      Stage::store_k(buf(1), s2.k[0], i);
    }
  }
  for (int i = tid; i < 4 * D; i += kPpThreads)
    *(u32x4*)(buf(1) + Stage::kV + 8 * i) = u32x4{0u, 0u, 0u, 0u};
  st.template load_k<0>(c, u0 + 2);
  if constexpr (kSets == 2) st.template load_k<kOther>(c, u0 + 3);
  st.template load_v<0>(c, u0);
  __syncthreads();
  scores(sa, 0);
  scores(sb, 1);
  mask(0, sa, ks, ev);
  {
    float big[2] = {sa[0], sa[8]};
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int e = 1; e < 8; ++e) big[k] = fmaxf(big[k], sa[8 * k + e]);
    follow(halves_max(fmaxf(fmaf(big[0], ks[0], ev[0]), fmaf(big[1], ks[1], ev[1]))));
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < Stage::kParts; ++i) Stage::store_k(buf(0), st.k[0], i);
  st.template load_k<0>(c, u0 + 2 + kSets);
  if constexpr (kSets == 2) st.template load_v<kOther>(c, u0 + 1);
  // steps whose V holds infinities or NaN: the wave's first, one past its last
  int odd0 = 0x7FFFFFFF, odd1 = 0;
  // A step of the workgroup.  One barrier parts the writers and the readers of
  // K (read of j + 2, written of j + 3) and V (read of j - 1, written of j).
  auto round = [&](auto parity, int j, f32x16& s0, f32x16& s1, f32x16& s2) {
    // the registers of V of j, and of K of j + 3
    constexpr int VS = decltype(parity)::value % kSets, KS3 = (decltype(parity)::value + 1) % kSets;
    // (of steps j + 1 to j + 5 below)
    if (u0 + j + 6 > st.base + 64) st.look_up(c, b, g, scale2, u0 + j);
    __syncthreads();
    uint32_t found = 0;
    // K of j + 3 and V of j to LDS, K of j + 4 and V of j + 1 on their way
    // (steps past the last: what lies there of the last pages, not used)
    auto other = [&](int i) {
      constexpr int U = kOps / 8;
      // (the compiler would decode before the barrier, and wait there)
      auto here = [](typename Stage::Piece (&x)[Stage::KP]) {
#pragma unroll
        for (int p = 0; p < Stage::KP; ++p) asm volatile("" : "+v"(x[p]));
      };
#pragma unroll
      for (int part = 0; part < Stage::kParts; ++part) {
        if (i == U * part) here(st.k[KS3]);
        if (i == U * (2 + part)) here(st.v[VS]);
        if (i == U * part) Stage::store_k(buf(j + 1), st.k[KS3], part);
        if (i == U * (2 + part)) Stage::store_v(buf(j), st.v[VS], part);
      }
      if (i == U * (Stage::kParts - 1)) st.template load_k<KS3>(c, u0 + j + 3 + kSets);
      if (i == 4 * U) {
#pragma unroll
        for (int p = 0; p < Stage::KP; ++p) found |= Stage::odd_in(st.v[VS][p]);
        st.template load_v<VS>(c, u0 + j + kSets);
      }
    };
    step(j, s0, s1, s2, other);
    if (__builtin_amdgcn_ballot_w64((found & Stage::kOdd) != 0)) {
      st.template load_v<VS>(c, u0 + j);
      Stage::store_v_finite(buf(j), st.v[VS]);
      st.template load_v<VS>(c, u0 + j + kSets);
      odd0 = min(odd0, u0 + j);
      odd1 = u0 + j + 1;
    }
  };
  const std::integral_constant<int, 0> even;
  const std::integral_constant<int, 1> uneven;
  for (int j = 0; j < n; j += 6) {
    round(even, j, sa, sb, sc);
    if (j + 1 < n) round(uneven, j + 1, sb, sc, sa);
    if (j + 2 < n) round(even, j + 2, sc, sa, sb);
    if (j + 3 < n) round(uneven, j + 3, sa, sb, sc);
    if (j + 4 < n) round(even, j + 4, sb, sc, sa);
    if (j + 5 < n) round(uneven, j + 5, sc, sa, sb);
  }
  __syncthreads();
  if (n > 0) {
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int i = 0; i < NG; ++i)
        o[i] = mfma_32x32x16(*(const f16x8*)(buf(n - 1) + Stage::v_at(k, half, 32 * i + col)),
                             w[k], o[i]);
  }
  if (lane == 0) {
    odds[0][wave] = odd0;
    odds[1][wave] = odd1;
  }
  __syncthreads();
  odd0 = min(min(odds[0][0], odds[0][1]), min(odds[0][2], odds[0][3]));
  odd1 = max(max(odds[1][0], odds[1][1]), max(odds[1][2], odds[1][3]));
  if (odd0 < odd1)
    add_odd_values<D, FP8>(o, c, b, g, __builtin_amdgcn_readfirstlane(odd0),
                           __builtin_amdgcn_readfirstlane(odd1), r);
  l += __shfl_xor(l, 32);
  if (!r.live) return;
  if (parts == 1) {
    __half* dst = a.out + ((int64_t)(r.s0 + tok) * Hq + g * a.rep + r.row % a.rep) * D;
#pragma unroll
    for (int i = 0; i < NG; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        store_row(dst + 32 * i + 8 * e + 4 * half,
                  f32x4{o[i][4 * e], o[i][4 * e + 1], o[i][4 * e + 2], o[i][4 * e + 3]}, l,
                  r.first + tok, r.cap);
  } else {
    float* dst = a.part + ((((int64_t)slot0 * c.Hk + g) * a.splits + split) * kPpRows + 32 * wave +
                           col) * PS;
#pragma unroll
    for (int i = 0; i < NG; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        *(f32x4*)(dst + 32 * i + 8 * e + 4 * half) =
            f32x4{o[i][4 * e], o[i][4 * e + 1], o[i][4 * e + 2], o[i][4 * e + 3]};
    if (half == 0) {
      dst[D] = m;
      dst[D + 1] = l;
    }
  }
}

// Merges the splits of units that have several, in order: thread (row, 4
// columns).
template <int D>
__global__ __launch_bounds__(256) void paged_combine_kernel(PagedAttnArgs a) {
  constexpr int PS = D + 4, RW = 256 / (D / 4);
  const PagedView& c = a.c;
  const int g = blockIdx.y;
  int slot = blockIdx.x / (kPpRows / RW), b;
  const int slot0 = slot, rw = blockIdx.x % (kPpRows / RW) * RW + threadIdx.x / (D / 4);
  if (c.starts) {
    b = slot_sequence(c, a.rep, kPpRows, 1, slot);
  } else {
    b = slot / a.slots_each;
    slot -= b * a.slots_each;
  }
  RowSet r;
  set_rows<kPpRows>(r, c, b, slot * kPpRows, a.rep, a.window, rw);
  const int rows = r.n * a.rep;
  if (slot < 0 || slot * kPpRows >= rows || (c.starts && rows <= kPaMostRows) || !r.live) return;
  const int parts = split_parts(
      a, (r.hi_any + kPpStep - 1) / kPpStep - r.lo_any / kPpStep);
  if (parts == 1) return;
  const int d4 = 4 * (threadIdx.x % (D / 4));
  const float* p = a.part + (((int64_t)slot0 * c.Hk + g) * a.splits * kPpRows + rw) * PS;
  Merge acc;
  constexpr int F = 8;  // in flight
  for (int s0 = 0; s0 < parts; s0 += F) {
    float2 ml[F];
    f32x4 o[F];
#pragma unroll
    for (int s = 0; s < F; ++s) {
      const float* ps = p + (int64_t)min(s0 + s, parts - 1) * (kPpRows * PS);
      ml[s] = *(const float2*)(ps + D);
      o[s] = *(const f32x4*)(ps + d4);
    }
#pragma unroll
    for (int s = 0; s < F; ++s)
      if (s0 + s < parts) acc.add(ml[s].x, ml[s].y, o[s]);
  }
  const int tok = r.row / a.rep;
  store_row(a.out + ((int64_t)(r.s0 + tok) * c.Hk * a.rep + g * a.rep + r.row % a.rep) * D + d4,
            acc.o, acc.den, r.first + tok, r.cap);
}

struct PromptShape {
  int64_t slots;
  int splits, split_steps;
};

// Units of 128 rows, and the parts that a long context's steps are cut into.
// The card holds 512 workgroups (two a CU), so up to 256 units take as many
// parts as fill them, of 8 steps and an eighth of the units at least: below
// that, the parts' way through memory and the second launch cost more.  Of
// more units only contexts of 256 steps are split, to even out the last
// workgroups.  Measured with 4 KV heads of 128 and 8 q heads each, us:
//   128 units of 141 steps   67 (4 parts), 76 (2), 113 (one)
//   128 units of 954         302 (4), 376 (2), 672 (one)
//    32 units of 36          24 (4), 27 (2), 35 (one)
//    32 units of 129         39 (16), 36 (8), 99 (one)
//   252 units of up to 32    34 (one), 40 (two of the longest)
//   288 units of up to 32    37 (one), 45 (two of the longest)
//   1024 units of up to 128  188 (one), 235 (two of the longest)
PromptShape prompt_shape(bool ragged, int64_t seqs, int64_t tokens, int64_t rep, int64_t kv_heads) {
  PromptShape s;
  s.slots = ragged ? tokens * rep / kPpRows + seqs
                   : seqs * ((tokens / std::max<int64_t>(seqs, 1) * rep + kPpRows - 1) / kPpRows);
  // (of a ragged batch's slots, about half of those for last rows are there)
  const int64_t n = std::max<int64_t>(s.slots * kv_heads, 1);
  const int64_t units = std::max<int64_t>((s.slots - (ragged ? seqs / 2 : 0)) * kv_heads, 1);
  const int64_t parts = std::min((units <= 256 ? 512 : kPpParts) / units, kPpParts / n);
  s.splits = (int)std::min<int64_t>(16, std::max<int64_t>(1, parts));
  s.split_steps = units <= 256 ? (int)std::max<int64_t>(8, units / 8) : 128;
  return s;
}

}  // namespace

// At least what prompt_shape's parts take, for these sizes and smaller ones.
int64_t paged_prompt_scratch_bytes(int64_t seqs, int64_t tokens, int64_t q_heads,
                                   int64_t kv_heads) {
  const int64_t rep = (q_heads + kv_heads - 1) / kv_heads;
  const int64_t n = (tokens * rep / kPpRows + seqs) * kv_heads;  // (more than without starts)
  const int64_t most = n <= 256 ? std::min<int64_t>(16 * n, 1024) : kPpParts;
  return most * kPpRows * (128 + 4) * 4;
}

int paged_prompt_launch(PagedAttnArgs a, int head_dim, hipStream_t stream) {
  const PromptShape s = prompt_shape(a.c.starts != nullptr, a.c.B, a.c.T, a.rep, a.c.Hk);
  a.slots = (int)s.slots;
  a.slots_each = a.c.starts ? 0 : (int)(s.slots / a.c.B);
  a.splits = s.splits;
  a.split_steps = s.split_steps;
  // no context that needs splitting
  const int64_t steps = (((int64_t)a.c.max_pages << a.c.page_shift) + kPpStep - 1) / kPpStep;
  if (steps < 2 * s.split_steps) a.splits = 1;
  const int64_t grid = s.slots * a.c.Hk * a.splits;
  // A CU holds workgroups i and i + 256: where nothing comes after them, the
  // one that sees least goes to the one that sees most: 2048 fresh tokens of 4
  // KV heads (512 workgroups) 66 us, 70.5 in order; 4096 of 16 KV heads and one
  // q head each 119 and 128.
  a.fold = (int)(grid <= 512 && a.splits == 1 ? std::min<int64_t>(s.slots, 256 / a.c.Hk) : s.slots);
  GLQ_CHECK(a.splits == 1 || grid * kPpRows * (head_dim + 4) * 4 <=
                                 paged_prompt_scratch_bytes(a.c.B, a.c.T, a.rep * a.c.Hk, a.c.Hk),
            "paged prompt parts do not fit their scratch");
  GLQ_CHECK(s.slots * 16 < (1ll << 24) && grid < (1ll << 24), "batch of too many query rows");
  const bool fp8 = a.c.ks != nullptr, wide = head_dim == 128;
  auto kern = wide ? (fp8 ? paged_prompt_kernel<128, true> : paged_prompt_kernel<128, false>)
                   : (fp8 ? paged_prompt_kernel<64, true> : paged_prompt_kernel<64, false>);
  const size_t lds = 2 * (wide ? PromptStage<128, true>::kBytes : PromptStage<64, true>::kBytes);
  static size_t attr[2] = {0, 0};
  if (wide)
    if (int rc = set_lds_limit(kern, lds, attr[fp8])) return rc;
  kern<<<dim3((unsigned)grid), dim3(kPpThreads), lds, stream>>>(a);
  GLQ_LAUNCH_CHECK("paged_prompt_kernel");
  if (a.splits > 1) {
    const dim3 cg((unsigned)(s.slots * (kPpRows / (256 / (head_dim / 4)))), (unsigned)a.c.Hk);
    if (wide)
      paged_combine_kernel<128><<<cg, dim3(256), 0, stream>>>(a);
    else
      paged_combine_kernel<64><<<cg, dim3(256), 0, stream>>>(a);
    GLQ_LAUNCH_CHECK("paged_combine_kernel");
  }
  return GLQ_OK;
}

}  // namespace glq
