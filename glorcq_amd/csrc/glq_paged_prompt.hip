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
  static constexpr int kBytes = 2 * kPpTile * D * 2;          // K and V of a step in LDS

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

  __device__ void load(const PagedView& c, int g, int tile, const Ids& r) {
    const int t = threadIdx.x, bpp = 1 << (c.page_shift - 4);
    auto place = [&](int p, int blk) {  // ids out of range read page 0
      return ((int64_t)((unsigned)p < (unsigned)c.pages ? p : 0) * c.Hk + g) * bpp +
             ((4 * tile + blk) & (bpp - 1));
    };
    bad = (unsigned)r.own >= (unsigned)c.pages;
    if constexpr (FP8) {
      const int64_t at = place(r.own, wave);
      ks = c.ks[at];
      vs = c.vs[at];
    }
    const unsigned k_lane = (t / KC & 15) * (D * S) + 16 * (t % KC), v_lane = t % D * (16 * S);
#pragma unroll
    for (int j = 0; j < KP; ++j)
      k[j] = *(const u32x4*)((const char*)c.k + place(r.k[j], k_block(j)) * (16 * D * S) + k_lane);
#pragma unroll
    for (int j = 0; j < VC; ++j)
#pragma unroll
      for (int i = 0; i < S; ++i)
        v[j][i] = *(const u32x4*)((const char*)c.v + place(r.v[j], v_block(j)) * (16 * D * S) +
                                  v_lane + 16 * i);
  }

  // K: piece (8 d8 .. + 8 of a position) at (d8, position, its low bits mixed
  // with d8's so that a row's pieces go to different banks); V: piece (block,
  // half, column), half 0 the block's positions 0-3 and 8-11, as lane halves
  // hold them.
  __device__ static int k_at(int d8, int pos) { return (d8 * kPpTile + (pos ^ (d8 & 14))) * 8; }
  __device__ static int v_at(int blk, int half, int d) {
    return kPpTile * D + ((blk * 2 + half) * D + d) * 8;
  }

  // Returns whether the thread's part of V holds an infinity or a NaN.
  __device__ bool store(_Float16* buf, float* scales, float scale2) const {
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
    uint32_t any = 0;
#pragma unroll
    for (int j = 0; j < VC; ++j) {
      const int blk = v_block(j), d = (kPpThreads * j + t) % D;
      if constexpr (FP8) {
        *(f16x8*)(buf + v_at(blk, 0, d)) = fp8x8_to_f16(v[j][0][0], v[j][0][2]);
        *(f16x8*)(buf + v_at(blk, 1, d)) = fp8x8_to_f16(v[j][0][1], v[j][0][3]);
      } else {
        *(u32x4*)(buf + v_at(blk, 0, d)) = u32x4{v[j][0][0], v[j][0][1], v[j][1][0], v[j][1][1]};
        *(u32x4*)(buf + v_at(blk, 1, d)) = u32x4{v[j][0][2], v[j][0][3], v[j][1][2], v[j][1][3]};
      }
      // (the largest exponent field carries into the sign's place)
#pragma unroll
      for (int i = 0; i < S; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          any |= FP8 ? (v[j][i][e] & 0x7F7F7F7Fu) + 0x01010101u
                     : (v[j][i][e] & 0x7FFF7FFFu) + 0x04000400u;
    }
    if ((t & 63) == 0) {
      scales[wave] = bad ? __builtin_nanf("") : FP8 ? e8m0_value(ks) * scale2 : scale2;
      scales[4 + wave] = FP8 ? e8m0_exponent(vs) : 0.f;
    }
    return (any & (FP8 ? 0x80808080u : 0x80008000u)) != 0;
  }
};

template <int D, bool FP8>
__global__ __launch_bounds__(kPpThreads, 2) void paged_prompt_kernel(PagedAttnArgs a) {
  using Stage = PromptStage<D, FP8>;
  constexpr int NG = D / 32, KS = D / 16, PS = D + 4;
  extern __shared__ __align__(16) unsigned char smem[];
  _Float16* bufs = (_Float16*)smem;  // 2 x Stage::kBytes
  __shared__ float scales[2][8];
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
  const int unit_lo = r.lo_all, unit_hi = r.hi_all;  // what all of its rows see
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
  f32x16 o[NG];
#pragma unroll
  for (int i = 0; i < NG; ++i) o[i] = f32x16{};

  Stage st;
  st.wave = wave;
  typename Stage::Ids ids = st.ids(c, b, t0);
  st.load(c, g, t0, ids);
  ids = st.ids(c, b, t0 + 1);
  auto stage = [&](int buf) {
    const bool odd = st.store(bufs + buf * (Stage::kBytes / 2), scales[buf], scale2);
    if (lane == 0) odds[buf][wave] = 0;
    if (__builtin_amdgcn_ballot_w64(odd) && lane == 0) odds[buf][wave] = 1;
  };
  stage(0);
  if (t0 + 1 < t1) {
    const typename Stage::Ids now = ids;
    ids = st.ids(c, b, t0 + 2);
    st.load(c, g, t0 + 1, now);
  }
  __syncthreads();
  // A step.  OddV: V holds an infinity or a NaN in a step that some row does not
  // see all of (rare; a loop of its own, which keeps the other free of copies).
  auto step = [&](int t, auto odd_v) {
    const int cur = (t - t0) & 1;
    const _Float16* kb = bufs + cur * (Stage::kBytes / 2);
    if (t + 1 < t1) {
      stage(cur ^ 1);
      if (t + 2 < t1) {
        const typename Stage::Ids now = ids;
        ids = st.ids(c, b, t + 3);
        st.load(c, g, t + 2, now);
      }
    }
    const int p0 = t * kPpTile;
    if (any && p0 < r.hi_any && p0 + kPpTile > r.lo_any) {  // (uniform in the wave)
      const bool edge = p0 < r.lo_all || p0 + kPpTile > r.hi_all;
      f32x16 s[2];
      s[0] = s[1] = f32x16{};
#pragma unroll
      for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const f16x8 ka = *(const f16x8*)(kb + Stage::k_at(2 * k + half, 32 * i + col));
          s[i] = mfma_32x32x16(ka, q[k], s[i]);
        }
      if (edge) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int p = p0 + 32 * i + 8 * (e >> 2) + 4 * half + (e & 3);
            if (p < r.lo || p >= r.hi) s[i][e] = -__builtin_inff();
          }
      }
      // block 2 i + (e >> 3) of the step: its scales
      const float* sc = scales[cur];
      float mx = -__builtin_inff();
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float bm = s[k >> 1][8 * (k & 1)];
#pragma unroll
        for (int e = 1; e < 8; ++e) bm = fmaxf(bm, s[k >> 1][8 * (k & 1) + e]);
        mx = fmaxf(mx, fmaf(bm, sc[k], sc[4 + k]));
      }
      mx = fmaxf(mx, __shfl_xor(mx, 32));
      if (__builtin_amdgcn_ballot_w64(mx > m + kPpLag)) {  // (-inf + lag: any score passes)
        const float mn = fmaxf(m, mx), mf = mn == -__builtin_inff() ? 0.f : mn;
        const float f = __builtin_amdgcn_exp2f(m - mf);
        m = mn;
        l *= f;
#pragma unroll
        for (int i = 0; i < NG; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e) o[i][e] *= f;
      }
      const float mf = m == -__builtin_inff() ? 0.f : m;
      f16x8 w[4];
      // (a position that a row does not see has no weight, whatever its block's
      // scale is)
      auto weights = [&](auto masked) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float ks = sc[k], ev = sc[4 + k], off = ev - mf;
          float sum = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float v = s[k >> 1][8 * (k & 1) + e];
            float x = __builtin_amdgcn_exp2f(fmaf(v, ks, off));
            if (masked.value) x = v == -__builtin_inff() ? 0.f : x;
            sum += x;
            w[k][e] = (_Float16)x;
          }
          if constexpr (!FP8)
            l += sum;
          else if (masked.value)
            l = sum == 0.f ? l : fmaf(sum, __builtin_amdgcn_exp2f(-ev), l);
          else
            l = fmaf(sum, __builtin_amdgcn_exp2f(-ev), l);
        }
      };
      if (edge)
        weights(std::true_type());
      else
        weights(std::false_type());
      if constexpr (!odd_v.value) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int i = 0; i < NG; ++i) {
            const f16x8 va = *(const f16x8*)(kb + Stage::v_at(k, half, 32 * i + col));
            o[i] = mfma_32x32x16(va, w[k], o[i]);
          }
      } else {
        // weight 0 times an inf or a NaN that a row does not see is not 0: a
        // token's rows at a time, with zeros for the positions behind its own
        const int last = __builtin_amdgcn_readlane(tok, 31);
#pragma nounroll
        for (int n = __builtin_amdgcn_readfirstlane(tok); n <= last; ++n) {
          const int pos = r.first + n, hi = pos + 1, lo = a.window > 0 ? pos - a.window + 1 : 0;
#pragma nounroll
          for (int k = 0; k < 4; ++k) {
            uint32_t keep[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {  // values 2 e, 2 e + 1 of a piece
              const int p = p0 + 16 * k + 8 * (e >> 1) + 4 * half + 2 * (e & 1);
              keep[e] = (p >= lo && p < hi ? 0xFFFFu : 0u) |
                        (p + 1 >= lo && p + 1 < hi ? 0xFFFF0000u : 0u);
            }
            const f16x8 wk = k & 2 ? (k & 1 ? w[3] : w[2]) : (k & 1 ? w[1] : w[0]);
#pragma unroll
            for (int i = 0; i < NG; ++i) {
              u32x4 va = *(const u32x4*)(kb + Stage::v_at(k, half, 32 * i + col));
#pragma unroll
              for (int e = 0; e < 4; ++e) va[e] &= keep[e];
              const f32x16 on = mfma_32x32x16(__builtin_bit_cast(f16x8, va), wk, o[i]);
#pragma unroll
              for (int e = 0; e < 16; ++e) o[i][e] = tok == n ? on[e] : o[i][e];
            }
          }
        }
      }
    }
    __syncthreads();
  };
  int t = t0;
  for (; t < t1; ++t) {
    const int* od = odds[(t - t0) & 1];
    if (__builtin_amdgcn_readfirstlane(od[0] | od[1] | od[2] | od[3]) &&
        (t * kPpTile < unit_lo || (t + 1) * kPpTile > unit_hi))
      break;  // uniform in the workgroup
    step(t, std::false_type());
  }
  for (; t < t1; ++t) step(t, std::true_type());
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
