// Causal attention of a batch's new tokens over a paged key/value cache
// (layout and formats: glq_paged.h), a few query rows a KV head at a time.

#include <algorithm>

#include "glq_paged.h"

namespace glq {
namespace {

constexpr int kPaThreads = 256;
constexpr int kPaRows = 16;  // query rows (tokens x the KV head's q heads) of a unit

struct PagedAttnArgs {
  PagedView c;
  const __half* q;  // (T, Hq, D)
  __half* out;      // (T, Hq D)
  int rep, window, tiles_each;
  float scale2;     // scale log2(e)
};

// The 16 query rows of a unit, column li of the matrix products on the lanes
// (li, kb), and the positions they see.
struct RowSet {
  int first;         // position of the sequence's first new token
  int s0, n;         // its rows of q
  int row;           // this lane's row: token row / rep, head row % rep
  bool live;
  int lo, hi;        // positions this lane's row sees: [lo, hi)
  int lo_all, hi_all, lo_any, hi_any;  // seen by all rows, by any
  int cap;           // positions of the page table
};

template <int D, bool FP8>
struct RowAttention {
  // A tile is TP positions; lane group kb has P consecutive ones of them, as
  // rows 4 kb + j of the NT products of 16 positions and as the P values of a
  // V column, so the weights go from one product to the next in registers.
  static constexpr int TP = FP8 ? 64 : 32, P = TP / 4, NT = TP / 16, NM = P / 8;
  static constexpr int KL = FP8 ? D / 64 : D / 32;  // 16-byte pieces of a K row and lane
  static constexpr int NC = D / 16;

  struct Tile {
    u32x4 k[NT][KL], v[NC];
    int ks, vs;
    bool bad;
  };

  const PagedView& c;
  int b, g, li, kb;
  float scale2;
  RowSet r;
  f16x8 q[D / 32];
  float m, l;
  f32x4 o[NC];

  __device__ RowAttention(const PagedView& c_) : c(c_) {
    li = threadIdx.x & 15;
    kb = (threadIdx.x >> 4) & 3;
  }

  __device__ void begin(const __half* qp, int rep, int Hq) {
    const int t = r.s0 + r.row / rep, h = g * rep + r.row % rep;
    const f16x8* src = (const f16x8*)(qp + ((int64_t)t * Hq + h) * D);
#pragma unroll
    for (int s = 0; s < D / 32; ++s)  // (e4m3: the two halves of a 16-code piece)
      q[s] = r.live ? src[FP8 ? 8 * (s >> 1) + 2 * kb + (s & 1) : 4 * s + kb] : f16x8{};
    m = -__builtin_inff();
    l = 0.f;
#pragma unroll
    for (int i = 0; i < NC; ++i) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  // Block of 16 tokens -> its place in the pool; pages out of range read page 0.
  __device__ int64_t place(int blk, bool& bad) const {
    const int bps = c.page_shift - 4;
    const int i = blk >> bps;
    const int p = c.table[b * c.table_stride + min(i, c.max_pages - 1)];
    bad = p < 0 || p >= c.pages;
    return ((int64_t)(bad ? 0 : p) * c.Hk + g) * (1 << bps) + (blk & ((1 << bps) - 1));
  }

  __device__ void load(Tile& x, int tile) const {
    constexpr int S = FP8 ? 1 : 2;
    bool ignore;
    const int b0 = tile * (TP / 16);
    const int64_t kblk = place(b0 + (FP8 ? li >> 2 : li >> 3), ignore);
    const int64_t vblk = place(b0 + (FP8 ? kb : kb >> 1), x.bad);
    const char* kp = (const char*)c.k + kblk * (16 * D * S);
    const char* vp = (const char*)c.v + vblk * (16 * D * S);
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const int row = (FP8 ? 0 : 8 * ((li >> 2) & 1)) + 4 * i + (li & 3);
#pragma unroll
      for (int t = 0; t < KL; ++t) x.k[i][t] = *(const u32x4*)(kp + row * D * S + 64 * t + 16 * kb);
    }
#pragma unroll
    for (int i = 0; i < NC; ++i)
      x.v[i] = *(const u32x4*)(vp + (16 * i + li) * 16 * S + (FP8 ? 0 : 16 * (kb & 1)));
    if constexpr (FP8) {
      x.ks = c.ks[vblk];
      x.vs = c.vs[vblk];
    }
  }

  __device__ static f16x8 k_frag(const Tile& x, int i, int s) {
    if constexpr (FP8) {
      const u32x4 w = x.k[i][s >> 1];
      return fp8x8_to_f16(w[2 * (s & 1)], w[2 * (s & 1) + 1]);
    } else {
      return __builtin_bit_cast(f16x8, x.k[i][s]);
    }
  }
  __device__ static f16x8 v_frag(const Tile& x, int i, int mm) {
    if constexpr (FP8)
      return fp8x8_to_f16(x.v[i][2 * mm], x.v[i][2 * mm + 1]);
    else
      return __builtin_bit_cast(f16x8, x.v[i]);
  }

  // Online softmax over the tile's positions.  The scale 2^e of a V block goes
  // into the exponent: w = 2^(t + e - m) with m the largest t + e so far, so
  // that w (fp16 for the product) keeps its bits where the block's share of
  // the result is largest; the denominator sums w 2^-e in fp32.
  __device__ void step(const Tile& x, int tile) {
    const int p0 = tile * TP + P * kb;
    const bool edge = tile * TP < r.lo_all || (tile + 1) * TP > r.hi_all;
    float t[NT][4];
    const float ks = FP8 ? e8m0_value(x.ks) * scale2 : scale2;
    const float ev = FP8 ? e8m0_exponent(x.vs) : 0.f;
    float mx = m;
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < D / 32; ++s) acc = mfma_16x16x32(k_frag(x, i, s), q[s], acc);
#pragma unroll
      for (int j = 0; j < 4; ++j) t[i][j] = x.bad ? __builtin_nanf("") : fmaf(acc[j], ks, ev);
      if (edge) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int p = p0 + 4 * i + j;
          if (p < r.lo || p >= r.hi) t[i][j] = -__builtin_inff();
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) mx = fmaxf(mx, t[i][j]);
    }
    mx = fmaxf(mx, __shfl_xor(mx, 16));
    mx = fmaxf(mx, __shfl_xor(mx, 32));
    const float mf = mx == -__builtin_inff() ? 0.f : mx;
    const float f = __builtin_amdgcn_exp2f(m - mf);  // (0 for m = -inf)
    m = mx;
    l *= f;
#pragma unroll
    for (int i = 0; i < NC; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[i][j] *= f;
    f16x8 w[NM];
    float ls = 0.f;
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float e = __builtin_amdgcn_exp2f(t[i][j] - mf);
        ls += e;
        w[i >> 1][4 * (i & 1) + j] = (_Float16)e;
      }
    // (a block that the row does not see may hold any scale)
    l = ls == 0.f ? l : fmaf(ls, __builtin_amdgcn_exp2f(-ev), l);
    // weight 0 times an inf or a NaN behind a row's positions is not 0
    bool odd = false;
    if (edge) {
#pragma unroll
      for (int i = 0; i < NC; ++i)
#pragma unroll
        for (int mm = 0; mm < NM; ++mm) {
          const u32x4 u = __builtin_bit_cast(u32x4, v_frag(x, i, mm));
#pragma unroll
          for (int e = 0; e < 4; ++e)
            odd |= (u[e] & 0x7C00u) == 0x7C00u || (u[e] & 0x7C000000u) == 0x7C000000u;
        }
      odd = __builtin_amdgcn_ballot_w64(odd) != 0;
    }
    if (!odd) {
#pragma unroll
      for (int i = 0; i < NC; ++i)
#pragma unroll
        for (int mm = 0; mm < NM; ++mm) o[i] = mfma_16x16x32(v_frag(x, i, mm), w[mm], o[i]);
    } else {
      // a position at a time, and only into the rows that see it
#pragma unroll
      for (int e = 0; e < P; ++e)
#pragma nounroll
        for (int k4 = 0; k4 < 4; ++k4) {
          const bool mine = kb == k4;
          const int p = tile * TP + P * k4 + e;
          const bool sees = p >= r.lo && p < r.hi;
          f16x8 wp{};
          wp[e & 7] = mine ? w[e >> 3][e & 7] : (_Float16)0.f;
#pragma unroll
          for (int i = 0; i < NC; ++i) {
            const f16x8 vf = v_frag(x, i, e >> 3);
            f16x8 vp{};
            vp[e & 7] = mine ? vf[e & 7] : (_Float16)0.f;
            const f32x4 on = mfma_16x16x32(vp, wp, o[i]);
#pragma unroll
            for (int j = 0; j < 4; ++j) o[i][j] = sees ? on[j] : o[i][j];
          }
        }
    }
  }
};

// Sets r for rows [16 qt, 16 qt + 16) of sequence b's n new tokens.
__device__ __forceinline__ void set_rows(RowSet& r, const PagedView& c, int b, int qt, int rep,
                                         int window, int li) {
  r.s0 = c.start(b);
  r.n = max((c.starts ? c.start(b + 1) : r.s0 + c.each) - r.s0, 0);
  r.first = c.length(b) - r.n;
  r.cap = c.max_pages << c.page_shift;
  const int rows = r.n * rep, r0 = qt * kPaRows, r1 = min(r0 + kPaRows, rows) - 1;
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

template <int D, bool FP8>
__global__ __launch_bounds__(kPaThreads) void paged_rows_kernel(PagedAttnArgs a) {
  using RA = RowAttention<D, FP8>;
  constexpr int W = kPaThreads / 64;
  __shared__ float sm[W][kPaRows], sl[W][kPaRows];
  __shared__ __align__(16) float so[W][kPaRows][D + 4];
  const PagedView& c = a.c;
  int slot = blockIdx.x, b;
  if (c.starts) {
    b = slot_sequence(c, a.rep, kPaRows, 1, slot);
    if (slot < 0) return;
  } else {
    b = slot / a.tiles_each;
    slot -= b * a.tiles_each;
  }
  const int wave = threadIdx.x >> 6;
  RA x(c);
  x.b = b;
  x.g = blockIdx.y;
  x.scale2 = a.scale2;
  set_rows(x.r, c, b, slot, a.rep, a.window, x.li);
  if (slot * kPaRows >= x.r.n * a.rep) return;  // uniform
  const int Hq = c.Hk * a.rep;
  x.begin(a.q, a.rep, Hq);
  for (int t = x.r.lo_any / RA::TP + wave; t * RA::TP < x.r.hi_any; t += W) {
    typename RA::Tile tile;
    x.load(tile, t);
    x.step(tile, t);
  }
  x.l += __shfl_xor(x.l, 16);
  x.l += __shfl_xor(x.l, 32);
  if (x.kb == 0) {
    sm[wave][x.li] = x.m;
    sl[wave][x.li] = x.l;
  }
#pragma unroll
  for (int i = 0; i < RA::NC; ++i) *(f32x4*)&so[wave][x.li][16 * i + 4 * x.kb] = x.o[i];
  __syncthreads();
  // thread (row, 4 columns a step)
  const int row = threadIdx.x >> 4, r = slot * kPaRows + row;
  if (r >= x.r.n * a.rep) return;
  float M = -__builtin_inff();
#pragma unroll
  for (int w = 0; w < W; ++w) M = fmaxf(M, sm[w][row]);
  const float Mf = M == -__builtin_inff() ? 0.f : M;
  float f[W], den = 0.f;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    f[w] = __builtin_amdgcn_exp2f(sm[w][row] - Mf);
    den = fmaf(sl[w][row], f[w], den);
  }
  const int tok = r / a.rep, pos = x.r.first + tok;
  const bool none = pos < 0, beyond = pos >= x.r.cap;
  const float inv = 1.f / den;
  __half* dst = a.out + ((int64_t)(x.r.s0 + tok) * Hq + x.g * a.rep + r % a.rep) * D;
  for (int d = 4 * (threadIdx.x & 15); d < D; d += 64) {
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const f32x4 ow = *(const f32x4*)&so[w][row][d];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = fmaf(ow[e], f[w], v[e]);
    }
    f16x2 y[2];
#pragma unroll
    for (int e = 0; e < 4; ++e)
      y[e >> 1][e & 1] = (_Float16)(none ? 0.f : beyond ? __builtin_nanf("") : v[e] * inv);
    *(uint2*)(dst + d) = uint2{__builtin_bit_cast(uint32_t, y[0]), __builtin_bit_cast(uint32_t, y[1])};
  }
}

}  // namespace
}  // namespace glq

extern "C" int64_t glq_paged_attention_workspace_bytes(int64_t seqs, int64_t tokens,
                                                       int64_t q_heads, int64_t kv_heads,
                                                       int64_t head_dim) {
  if (seqs < 0 || tokens < 0 || q_heads <= 0 || kv_heads <= 0 || head_dim <= 0) return -1;
  return 256;
}

extern "C" int glq_paged_attention(const glq_paged_cache* cache, const int32_t* starts,
                                   int64_t tokens, const void* q, int64_t q_heads, float scale,
                                   int64_t window, void* out, void* workspace,
                                   int64_t workspace_bytes, void* stream) {
  using namespace glq;
  clear_error();
  PagedAttnArgs a{};
  if (int rc = paged_view(cache, starts, tokens, a.c)) return rc;
  const int64_t D = cache->head_dim, Hk = cache->kv_heads;
  GLQ_CHECK(q_heads > 0 && q_heads % Hk == 0 && q_heads <= 8192,
            "q_heads must be a positive multiple of kv_heads (<= 8192)");
  GLQ_CHECK(window >= 0, "window must be >= 0 (0: none)");
  if (tokens == 0 || cache->seqs == 0) return GLQ_OK;
  GLQ_CHECK(q && out && ((uintptr_t)q & 15) == 0 && ((uintptr_t)out & 15) == 0,
            "q and out must be non-null and 16-byte aligned");
  const int64_t need =
      glq_paged_attention_workspace_bytes(cache->seqs, tokens, q_heads, Hk, D);
  GLQ_CHECK(workspace && workspace_bytes >= need && ((uintptr_t)workspace & 255) == 0,
            "a 256-byte aligned workspace of %lld bytes needed (got %lld)", (long long)need,
            (long long)workspace_bytes);
  a.q = (const __half*)q;
  a.out = (__half*)out;
  a.rep = (int)(q_heads / Hk);
  a.window = window >= cache->max_pages * cache->page_size ? 0 : (int)window;
  a.scale2 = scale * 1.44269504088896f;
  GLQ_CHECK(tokens * a.rep < (1ll << 30), "batch of too many (token, head) rows");
  a.tiles_each = (int)(((int64_t)a.c.each * a.rep + kPaRows - 1) / kPaRows);
  const int64_t slots = starts ? tokens * a.rep / kPaRows + cache->seqs : cache->seqs * a.tiles_each;
  GLQ_CHECK(slots < (1ll << 24) && Hk <= 65535, "batch of too many query rows");
  auto kern = D == 128 ? (a.c.ks ? paged_rows_kernel<128, true> : paged_rows_kernel<128, false>)
                       : (a.c.ks ? paged_rows_kernel<64, true> : paged_rows_kernel<64, false>);
  kern<<<dim3((unsigned)slots, (unsigned)Hk), dim3(kPaThreads), 0, (hipStream_t)stream>>>(a);
  GLQ_LAUNCH_CHECK("paged_rows_kernel");
  return GLQ_OK;
}
