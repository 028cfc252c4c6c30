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

constexpr int kPpThreads = 256;
constexpr int kPpTile = 64;    // positions of a step
constexpr float kPpLag = 8.f;  // log2 by which a score may pass the running maximum

// One workgroup takes 128 query rows (tokens x the KV head's q heads) of one KV
// head, 32 a wave, over the positions they see (or a split of them), 64 a step:
//   S^T = K Q^T   v_mfma_f32_32x32x16_f16, A = 32 positions of K, B = the rows
//   O^T += V^T P^T                         A = 32 columns of V,   B = the weights
// so that a row of the softmax is a column of both products: its 64 scores of
// a step lie on two lanes, and the weights are the second product's operand as
// they stand.  The step's K and V go through LDS as fp16, decoded once for the
// four waves, in the order of the operands (16-byte pieces, conflict-free both
// ways), double buffered, one barrier a step.  The next step's bytes are in
// flight meanwhile, page ids one step before them.
//
// Softmax: the running maximum m of t + e (e the exponent of V's block, as in
// the first form) follows the scores only when one passes it by more than
// 2^kPpLag: weights up to 2^8 lose nothing, in fp16 or in the fp32 sums, and
// the 64 sums of O a lane are rarely scaled.
template <int D, bool FP8>
struct PromptStage {
  static constexpr int S = FP8 ? 1 : 2;                       // bytes of a value
  static constexpr int KP = kPpTile * D * S / 16 / kPpThreads;  // 16-byte pieces of K a thread
  static constexpr int KC = D * S / 16;                       // pieces of a K row
  static constexpr int KR = kPpThreads / KC;                  // rows a pass
  static constexpr int VC = 4 * D / kPpThreads;               // V columns (of a block) a thread

  u32x4 k[KP], v[VC][S];
  int ks, vs;  // scale bytes of the wave's block
  bool bad;
  int wave;    // uniform

  // A wave's pieces of a pass lie in one block, so that addresses are scalars
  // but for a lane's constant part.
  __device__ int k_block(int j) const { return KR * j / 16 + wave * 64 / KC / 16; }
  __device__ int v_block(int j) const { return (kPpThreads * j + 64 * wave) / D; }
  static_assert(KR % 16 == 0, "a pass's rows");

  // Page ids of the blocks that the wave fetches, and of the one whose scales
  // it does (block `wave`).
  struct Ids {
    int k[KP], v[VC], own;
  };
  __device__ Ids ids(const PagedView& c, int b, int tile) const {
    const int* row = c.table + b * c.table_stride;
    auto id = [&](int blk) {
      return __builtin_amdgcn_readfirstlane(
          row[min((4 * tile + blk) >> (c.page_shift - 4), c.max_pages - 1)]);
    };
    Ids r;
#pragma unroll
    for (int j = 0; j < KP; ++j) r.k[j] = id(k_block(j));
#pragma unroll
    for (int j = 0; j < VC; ++j) r.v[j] = id(v_block(j));
    r.own = id(wave);
    return r;
  }

  // (ids out of range read page 0)
  __device__ static int64_t place(const PagedView& c, int g, int p, int tile, int blk) {
    const int bpp = 1 << (c.page_shift - 4);
    return ((int64_t)((unsigned)p < (unsigned)c.pages ? p : 0) * c.Hk + g) * bpp +
           ((4 * tile + blk) & (bpp - 1));
  }
  __device__ void load_k(const PagedView& c, int g, int tile, const Ids& r) {
    const int t = threadIdx.x;
    bad = (unsigned)r.own >= (unsigned)c.pages;
    if constexpr (FP8) {
      const int64_t at = place(c, g, r.own, tile, wave);
      ks = c.ks[at];
      vs = c.vs[at];
    }
    const unsigned lane = (t / KC & 15) * (D * S) + 16 * (t % KC);
#pragma unroll
    for (int j = 0; j < KP; ++j)
      k[j] = *(const u32x4*)((const char*)c.k +
                             place(c, g, r.k[j], tile, k_block(j)) * (16 * D * S) + lane);
  }
  __device__ void load_v(const PagedView& c, int g, int tile, const Ids& r) {
    const unsigned lane = threadIdx.x % D * (16 * S);
#pragma unroll
    for (int j = 0; j < VC; ++j)
#pragma unroll
      for (int i = 0; i < S; ++i)
        v[j][i] = *(const u32x4*)((const char*)c.v +
                                  place(c, g, r.v[j], tile, v_block(j)) * (16 * D * S) + lane +
                                  16 * i);
  }

  // LDS places in halves.  K: piece (8 d8 .. + 8 of a position) at (d8,
  // position), 32 bytes between pairs of d8 so that a row's pieces go to
  // different banks as they are stored (between single d8, the two lane halves
  // of a read collide: half of the LDS cycles); V: piece (block, half, column),
  // half 0 the block's positions 0-3 and 8-11, as the lane halves hold them.
  static constexpr int kKPair = 2 * kPpTile * 8 + 16;
  __device__ static int k_at(int d8, int pos) {
    return (d8 >> 1) * kKPair + (d8 & 1) * (kPpTile * 8) + pos * 8;
  }
  __device__ static int v_at(int blk, int half, int d) {
    return D / 16 * kKPair + ((blk * 2 + half) * D + d) * 8;
  }
  static constexpr int kBytes = 2 * (D / 16 * kKPair + kPpTile * D);  // of a step

  __device__ void store_k(_Float16* buf, float* scales, float scale2) const {
    const int t = threadIdx.x;
#pragma unroll
    for (int j = 0; j < KP; ++j) {
      const int row = KR * j + t / KC, piece = t % KC;
      if constexpr (FP8) {
        *(f16x8*)(buf + k_at(2 * piece, row)) = fp8x8_to_f16(k[j][0], k[j][1]);
        *(f16x8*)(buf + k_at(2 * piece + 1, row)) = fp8x8_to_f16(k[j][2], k[j][3]);
      } else {
        *(u32x4*)(buf + k_at(piece, row)) = k[j];
      }
    }
    if ((t & 63) == 0) {
      scales[wave] = bad ? __builtin_nanf("") : FP8 ? e8m0_value(ks) * scale2 : scale2;
      scales[4 + wave] = FP8 ? e8m0_exponent(vs) : 0.f;
    }
  }
  // Infinities and NaN go into LDS as zeros (weight 0 times one that a row does
  // not see is not 0); returns whether the wave's part of V holds any, for
  // them to be added afterwards.
  __device__ bool store_v(_Float16* buf) const {
    const int t = threadIdx.x;
    uint32_t any = 0;
#pragma unroll
    for (int j = 0; j < VC; ++j)
#pragma unroll
      for (int i = 0; i < S; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) any |= odd_values(v[j][i][e]);
    const bool found = __builtin_amdgcn_ballot_w64((any & kOdd) != 0) != 0;
    u32x4 u[VC][S];
#pragma unroll
    for (int j = 0; j < VC; ++j)
#pragma unroll
      for (int i = 0; i < S; ++i) u[j][i] = v[j][i];
    if (found) {
#pragma unroll
      for (int j = 0; j < VC; ++j)
#pragma unroll
        for (int i = 0; i < S; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t x = (odd_values(v[j][i][e]) & kOdd) >> (FP8 ? 7 : 15);
            u[j][i][e] &= ~(x * (FP8 ? 0xFFu : 0xFFFFu));
          }
    }
#pragma unroll
    for (int j = 0; j < VC; ++j) {
      const int blk = v_block(j), d = (kPpThreads * j + t) % D;
      if constexpr (FP8) {
        *(f16x8*)(buf + v_at(blk, 0, d)) = fp8x8_to_f16(u[j][0][0], u[j][0][2]);
        *(f16x8*)(buf + v_at(blk, 1, d)) = fp8x8_to_f16(u[j][0][1], u[j][0][3]);
      } else {
        *(u32x4*)(buf + v_at(blk, 0, d)) = u32x4{u[j][0][0], u[j][0][1], u[j][1][0], u[j][1][1]};
        *(u32x4*)(buf + v_at(blk, 1, d)) = u32x4{u[j][0][2], u[j][0][3], u[j][1][2], u[j][1][3]};
      }
    }
    return found;
  }
  // Of a word of values, the top bit of each infinity or NaN (with kOdd).
  static constexpr uint32_t kOdd = FP8 ? 0x80808080u : 0x80008000u;
  __device__ static uint32_t odd_values(uint32_t w) {
    // (the largest exponent field carries into the sign's place)
    return FP8 ? (w & 0x7F7F7F7Fu) + 0x01010101u : (w & 0x7FFF7FFFu) + 0x04000400u;
  }
};

// Adds the infinities and NaN of V that the row of a lane sees, at positions of
// steps [t0, t1), to its sums: rare, and so a plain walk over the blocks.
template <int D, bool FP8>
__device__ void add_odd_values(f32x16 (&o)[D / 32], const PagedView& c, int b, int g, int t0,
                               int t1, const RowSet& r) {
  using Stage = PromptStage<D, FP8>;
  constexpr int S = FP8 ? 1 : 2, NG = D / 32;
  const int lane = threadIdx.x & 63, half = lane >> 5;
  for (int blk = 4 * t0; blk < 4 * t1; ++blk) {
    const int p = c.page_of(b, blk >> (c.page_shift - 4));
    if (p < 0) continue;  // (the scores are NaN there)
    const char* base = (const char*)c.v + Stage::place(c, g, p, 0, blk) * (16 * D * S);
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

template <int D, bool FP8>
__global__ __launch_bounds__(kPpThreads) __attribute__((amdgpu_waves_per_eu(2, 2)))
void paged_prompt_kernel(PagedAttnArgs a) {
  using Stage = PromptStage<D, FP8>;
  constexpr int NG = D / 32, KS = D / 16, PS = D + 4;
  extern __shared__ __align__(16) unsigned char smem[];
  _Float16* bufs = (_Float16*)smem;  // 2 x Stage::kBytes
  __shared__ float scales[4][8];  // (a step's are read into the next one's first half)
  __shared__ int odds[2][kPpThreads / 64];
  const PagedView& c = a.c;
  // the last rows of a sequence, which see most, first
  int id = blockIdx.x;
  const int split = id % a.splits;
  id /= a.splits;
  const int g = id % c.Hk;
  int slot = a.slots - 1 - id / c.Hk, b;
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
  // the unit's tiles, and this split's of them
  int t0 = r.lo_any / kPpTile, t1 = (r.hi_any + kPpTile - 1) / kPpTile;
  int per = max(t1 - t0, 1), parts = 1;
  if (a.splits > 1) {
    per = max((per + a.splits - 1) / a.splits, a.split_tiles);
    parts = (max(t1 - t0, 1) + per - 1) / per;
    if (split >= parts) return;  // uniform
    t0 += split * per;
    t1 = min(t1, t0 + per);
  }
  const int r0 = slot * kPpRows + 32 * wave;
  const bool any = r0 < rows;  // the wave has rows
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
    for (int s = 0; s < KS; ++s) q[s] = r.live ? src[2 * s + half] * sign : f16x8{};
  }
  const float scale2 = a.scale2 == 0.f ? 1.f : fabsf(a.scale2);
  float m = -__builtin_inff(), l = 0.f;
  f32x16 o[NG], sa = {}, sb = {};
  f16x8 w[2] = {f16x8{}, f16x8{}};
#pragma unroll
  for (int i = 0; i < NG; ++i) o[i] = f32x16{};

  Stage st;
  st.wave = wave;
  auto buf = [&](int t) { return bufs + ((t - t0) & 1) * (Stage::kBytes / 2); };
  // 32 scores a row: positions 32 i .. + 32 of step t
  auto scores = [&](f32x16& s, int t, int i) {
    const _Float16* kb = buf(t);
    s = f32x16{};
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      const f16x8 ka = *(const f16x8*)(kb + Stage::k_at(2 * k + half, 32 * i + col));
      s = mfma_32x32x16(ka, q[k], s);
    }
  };
  // O += the weights of positions 32 i .. of step t times their V
  auto weigh_v = [&](int t, int i) {
    const _Float16* kb = buf(t);
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int n = 0; n < NG; ++n) {
        const f16x8 va = *(const f16x8*)(kb + Stage::v_at(2 * i + k, half, 32 * n + col));
        o[n] = mfma_32x32x16(va, w[k], o[n]);
      }
  };
  // Half a step, on positions 32 i .. of step t, whose scores are in s: the
  // matrix instructions of the half before (its weighted V) and of the half
  // after (its scores, to `next`) run beside this one's exponentials.
  auto half_step = [&](int t, auto i_, f32x16& s, f32x16& next) {
    constexpr int i = i_.value;
    const int p0 = t * kPpTile + 32 * i;
    // the operands of the matrix instructions below, kAhead of them in flight:
    // in turn K's of the scores and V's
    constexpr int kOps = KS + 2 * NG, kAhead = 4;
    static_assert(KS == 2 * NG, "as many of each");
    const _Float16 *kbuf = buf(t + i), *vbuf = buf(t + i - 1);
    auto operand = [&](int n) {
      return n & 1 ? *(const f16x8*)(vbuf + Stage::v_at(2 * (1 - i) + n / 2 / NG, half,
                                                        32 * (n / 2 % NG) + col))
                   : *(const f16x8*)(kbuf + Stage::k_at(n + half, 32 * (1 - i) + col));
    };
    f16x8 op[kAhead];
#pragma unroll
    for (int n = 0; n < kAhead; ++n) op[n] = operand(n);
    __builtin_amdgcn_sched_barrier(0);
    // block 2 i + k of the step: its scales
    const float* sc = scales[(t - t0) & 3] + 2 * i;
    float ks[2] = {sc[0], sc[1]}, ev[2] = {sc[4], sc[5]};
    if (p0 < r.lo_all || p0 + 32 > r.hi_all) {
      // a position that a row does not see has no weight, whatever its block's
      // scale is: a NaN goes from the scale to the scores
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
    float mx = -__builtin_inff();
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      float bm = s[8 * k];
#pragma unroll
      for (int e = 1; e < 8; ++e) bm = fmaxf(bm, s[8 * k + e]);
      mx = fmaxf(mx, fmaf(bm, ks[k], ev[k]));
    }
    mx = fmaxf(mx, __shfl_xor(mx, 32));
    if (__builtin_amdgcn_ballot_w64(mx > m + kPpLag)) {  // (-inf + lag: any score passes)
      // a whole number, so that the factor of the weights in w is a power of two
      const float mn = fmaxf(m, ceilf(mx)), mf = mn == -__builtin_inff() ? 0.f : mn;
      const float f = __builtin_amdgcn_exp2f(m - mf);
      const _Float16 fh = (_Float16)f;
      m = mn;
      l *= f;
#pragma unroll
      for (int k = 0; k < 2; ++k) w[k] *= fh;
#pragma unroll
      for (int n = 0; n < NG; ++n)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[n][e] *= f;
    }
    const float mf = m == -__builtin_inff() ? 0.f : m;
    const float off[2] = {ev[0] - mf, ev[1] - mf};
    f16x8 wn[2];
    float sum[2] = {0.f, 0.f};
    next = f32x16{};
#pragma unroll
    for (int n = 0; n < kOps; ++n) {
      if (n & 1)
        o[n / 2 % NG] = mfma_32x32x16(op[n % kAhead], w[n / 2 / NG], o[n / 2 % NG]);
      else
        next = mfma_32x32x16(op[n % kAhead], q[n / 2], next);
      if (n + kAhead < kOps) op[n % kAhead] = operand(n + kAhead);
#pragma unroll
      for (int e = 16 / kOps * n; e < 16 / kOps * (n + 1); ++e) {
        const int k = e >> 3;
        float x = __builtin_amdgcn_exp2f(fmaf(s[e], ks[k], off[k]));
        asm volatile("" : "+v"(x));  // (in this place)
        sum[k] += x;
        wn[k][e & 7] = (_Float16)x;
      }
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int k = 0; k < 2; ++k)
      l = FP8 ? fmaf(sum[k], __builtin_amdgcn_exp2f(-ev[k]), l) : l + sum[k];
    w[0] = wn[0];
    w[1] = wn[1];
  };

  // Before the loop: K and V of step t0 in LDS, the next step's in registers,
  // zeros where the first half step looks for the V of the one before it.
  typename Stage::Ids ids = st.ids(c, b, t0);
  st.load_k(c, g, t0, ids);
  st.load_v(c, g, t0, ids);
  ids = st.ids(c, b, t0 + 1);
  for (int i = tid; i < 4 * D; i += kPpThreads)
    *(u32x4*)(buf(t0 - 1) + Stage::v_at(2, 0, 0) + 8 * i) = u32x4{0u, 0u, 0u, 0u};
  st.store_k(buf(t0), scales[0], scale2);
  // steps whose V holds infinities or NaN: the wave's first, one past its last
  int odd0 = st.store_v(buf(t0)) ? t0 : 0x7FFFFFFF, odd1 = t0 + 1;
  if (t0 + 1 < t1) {
    st.load_k(c, g, t0 + 1, ids);
    st.load_v(c, g, t0 + 1, ids);
  }
  ids = st.ids(c, b, t0 + 2);
  __syncthreads();
  if (any) scores(sa, t0, 0);
  // A step.  K of the next one is stored in its first half and V in its second,
  // so that the one barrier between the halves parts writers and readers: K of
  // t + 1 is first read after it and K of t - 1 last before the barrier of
  // t - 1; V of t is first read after it, V of t - 2 last before t - 1's.
  using H0 = std::integral_constant<int, 0>;
  using H1 = std::integral_constant<int, 1>;
  for (int t = t0; t < t1; ++t) {
    if (any) half_step(t, H0(), sa, sb);
    if (t + 1 < t1) {
      st.store_k(buf(t + 1), scales[(t + 1 - t0) & 3], scale2);
      if (t + 2 < t1) st.load_k(c, g, t + 2, ids);
    }
    __syncthreads();
    if (any) half_step(t, H1(), sb, sa);
    if (t + 1 < t1) {
      if (st.store_v(buf(t + 1))) {
        odd0 = min(odd0, t + 1);
        odd1 = t + 2;
      }
      if (t + 2 < t1) {
        st.load_v(c, g, t + 2, ids);
        ids = st.ids(c, b, t + 3);
      }
    }
  }
  if (any && t1 > t0) weigh_v(t1 - 1, 1);
  if (lane == 0) {
    odds[0][wave] = odd0;
    odds[1][wave] = odd1;
  }
  __syncthreads();
  odd0 = min(min(odds[0][0], odds[0][1]), min(odds[0][2], odds[0][3]));
  odd1 = max(max(odds[1][0], odds[1][1]), max(odds[1][2], odds[1][3]));
  if (any && odd0 < odd1 && t1 > t0)
    add_odd_values<D, FP8>(o, c, b, g, __builtin_amdgcn_readfirstlane(odd0),
                           __builtin_amdgcn_readfirstlane(min(odd1, t1)), r);
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
  const int tiles =
      max((r.hi_any + kPpTile - 1) / kPpTile - r.lo_any / kPpTile, 1);
  const int per = max((tiles + a.splits - 1) / a.splits, a.split_tiles);
  const int parts = (tiles + per - 1) / per;
  if (parts == 1) return;
  const int d4 = 4 * (threadIdx.x % (D / 4));
  const float* p = a.part + (((int64_t)slot0 * c.Hk + g) * a.splits * kPpRows + rw) * PS;
  Merge acc;
  for (int s = 0; s < parts; ++s, p += kPpRows * PS) acc.add(p[D], p[D + 1], *(const f32x4*)(p + d4));
  const int tok = r.row / a.rep;
  store_row(a.out + ((int64_t)(r.s0 + tok) * c.Hk * a.rep + g * a.rep + r.row % a.rep) * D + d4,
            acc.o, acc.den, r.first + tok, r.cap);
}

struct PromptShape {
  int64_t slots;
  int splits, split_tiles;
};

// Units of 128 rows, and the splits of the positions that fill the 512
// workgroups the card holds of them: with few units, down to 8 steps a split;
// with more, only to even out contexts of very different lengths.
PromptShape prompt_shape(bool ragged, int64_t seqs, int64_t tokens, int64_t rep, int64_t kv_heads) {
  PromptShape s;
  s.slots = ragged ? tokens * rep / kPpRows + seqs
                   : seqs * ((tokens / std::max<int64_t>(seqs, 1) * rep + kPpRows - 1) / kPpRows);
  const int64_t units = std::max<int64_t>(s.slots * kv_heads, 1);
  s.splits = (int)std::min<int64_t>(16, std::max<int64_t>(1, (units < 512 ? 1024 : 2048) / units));
  s.split_tiles = units < 512 ? 8 : 64;
  return s;
}

}  // namespace

int64_t paged_prompt_scratch_bytes(int64_t seqs, int64_t tokens, int64_t q_heads,
                                   int64_t kv_heads) {
  // (either form of the batch; the wider head)
  const int64_t rep = (q_heads + kv_heads - 1) / kv_heads;
  int64_t most = 0;
  for (int ragged = 0; ragged < 2; ++ragged) {
    if (!ragged && seqs > 0 && tokens % seqs) continue;
    const PromptShape s = prompt_shape(ragged, seqs, tokens, rep, kv_heads);
    if (s.splits > 1) most = std::max(most, s.slots * kv_heads * s.splits);
  }
  return most * kPpRows * (128 + 4) * 4;
}

int paged_prompt_launch(PagedAttnArgs a, int head_dim, hipStream_t stream) {
  const PromptShape s = prompt_shape(a.c.starts != nullptr, a.c.B, a.c.T, a.rep, a.c.Hk);
  a.slots = (int)s.slots;
  a.slots_each = a.c.starts ? 0 : (int)(s.slots / a.c.B);
  a.splits = s.splits;
  a.split_tiles = s.split_tiles;
  // no context that needs splitting
  const int64_t tiles = (((int64_t)a.c.max_pages << a.c.page_shift) + kPpTile - 1) / kPpTile;
  if (tiles <= s.split_tiles) a.splits = 1;
  const int64_t grid = s.slots * a.c.Hk * a.splits;
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
