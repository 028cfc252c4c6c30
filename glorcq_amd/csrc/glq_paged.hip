// Appending to a paged key/value cache: head RMSNorm and rotary embedding of
// the new tokens' q and k, k and v into their positions' pages (layout and
// formats: glq_paged.h), in one launch for decode steps and prompts alike.

#include "glq_paged.h"

namespace glq {
namespace {

constexpr int kAppThreads = 256;
constexpr int kMinScale = 127 - 32;  // the smallest scale byte written: 2^-32
constexpr int kQPasses = 4;          // of a wave over q

struct AppendArgs {
  PagedView c;
  const __half *q, *k, *v;  // rows of q_stride / k_stride / v_stride values per token; q may be null
  int64_t q_stride, k_stride, v_stride;
  int q_item;  // > 0: q item-major, [Hq D / q_item][T][q_item]
  const __half *qw, *kw;    // null: no norm
  const __half *cos, *sin;  // rows of D, null: no rotation
  int64_t cs_stride;        // 0 when one row serves every token
  __half* q_out;            // (T, Hq, D)
  int Hq;
  int units, slots, kv_waves;
  float eps;
};

__device__ __forceinline__ float rsqrt_of(float x) { return rsqrtf(x); }
__device__ __forceinline__ double rsqrt_of(double x) { return rsqrt(x); }

// A head's D values on D / 8 lanes, 8 each (lane `c` of them: 8 c .. + 8).
//   x -> x rsqrt(mean(x^2) + eps) w   (w != null)
//     -> x cos + rotate_half(x) sin   (cos != null)
// The caller rounds once.  q: in fp32.  k: in fp64, since a value that fp32
// leaves on the wrong side of a border between two e4m3 codes is off by a
// whole step of 2^-3 for as long as the cache lives; the vector fp64 rate is
// half of fp32's, and k has a share Hk / Hq of the work.
template <int D, class F>
__device__ __forceinline__ void head_norm_rope(F (&x)[8], const f16x8* w, const f16x8* cos,
                                               const f16x8* sin, int c, float eps) {
  constexpr int L = D / 8;
  if (w) {
    F ss = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) ss += x[e] * x[e];
#pragma unroll
    for (int o = 1; o < L; o <<= 1) ss += __shfl_xor(ss, o);
    const F r = rsqrt_of(ss / (F)D + (F)eps);
    const f16x8 wv = *w;
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = x[e] * r * (F)wv[e];
  }
  if (cos) {
    const f16x8 cv = *cos, sv = *sin;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const F other = __shfl_xor(x[e], L / 2);  // the value D / 2 away
      x[e] = x[e] * (F)cv[e] + (c < L / 2 ? -other : other) * (F)sv[e];
    }
  }
}

__device__ __forceinline__ bool finite(float x) {
  return (__float_as_uint(x) & 0x7F800000u) != 0x7F800000u;
}

// 8 values -> 8 e4m3 codes of x inv; values without a code (inf, NaN) -> NaN.
__device__ __forceinline__ u32x2 quantize8(const float (&x)[8], float inv) {
  float y[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) y[e] = finite(x[e]) ? x[e] * inv : __builtin_nanf("");
  int a = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
  a = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], a, true);
  int b = __builtin_amdgcn_cvt_pk_fp8_f32(y[4], y[5], 0, false);
  b = __builtin_amdgcn_cvt_pk_fp8_f32(y[6], y[7], b, true);
  return u32x2{(uint32_t)a, (uint32_t)b};
}

// 4 codes scaled by f = 2^-n: exact, but where the result is a subnormal.
__device__ __forceinline__ uint32_t rescale4(uint32_t w, float f) {
  f16x2 a, b;
  fp8_to_f16(w, a, b);
  int r = __builtin_amdgcn_cvt_pk_fp8_f32((float)a[0] * f, (float)a[1] * f, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32((float)b[0] * f, (float)b[1] * f, r, true);
}

// Scale byte of a block whose largest finite value is amax: the smallest
// 2^e >= amax / 448 = amax / (1.75 2^8), at least 2^-32.
__device__ __forceinline__ int scale_byte(float amax) {
  const int b = (int)((__float_as_uint(amax) + 0x1FFFFFu) >> 23) - 8;
  return max(b, kMinScale);
}

// One wave a (16-token block, KV head, k or v): the block's scale is one
// number, so one wave sees all of the block's new values, and nobody else
// writes any of it.  A block that had tokens before keeps its scale unless the
// new ones need a larger one; then its codes are scaled down by the power of
// two.  What lies behind the last token of an 8-bit block is zero.
//
// V goes through LDS, from rows of a token to columns of 16 tokens, so that
// pages are written in 16-byte pieces of whole 16-token columns.
//
// The other waves rotate q, 64 / (D / 8) heads a pass, 4 passes each: 16000
// tokens of 32 heads take 82 us with 4 and 86 with one; up to 4000 tokens
// (19 us) it makes no difference.
//
// Bound by memory: each token's q, k and v are read once, q and the pages
// written once.  8000 tokens of 32 and 4 heads of 128 into 8-bit pages: 34 us;
// 7 ragged prompts of 7200 tokens with norms 30.5 us, 4.8 TB/s, what a copy
// reaches (a first form that gave a workgroup a token: 43).  One token: 6.6 us,
// the launch.
template <int D, bool FP8>
__global__ __launch_bounds__(kAppThreads) void paged_append_kernel(AppendArgs a) {
  constexpr int L = D / 8;         // lanes of a head
  constexpr int TP = 64 / L;       // tokens (heads) a pass
  constexpr int NP = kBlkTokens / TP;
  __shared__ __align__(16) unsigned char smem[4][kBlkTokens * D * (FP8 ? 1 : 2)];
  const PagedView& c = a.c;
  const int lane = threadIdx.x & 63;
  const int wib = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wave = blockIdx.x * (kAppThreads / 64) + wib;
  const int li = lane % L, tk = lane / L;
  if (wave >= a.kv_waves) {
    // rows (token, q head)
    const int Tn = c.starts ? c.start(c.B) : c.T;
    const int64_t rows = (int64_t)Tn * a.Hq;
    int64_t r0 = (int64_t)(wave - a.kv_waves) * kQPasses * TP;
    for (int p = 0; p < kQPasses; ++p, r0 += TP) {
      if (r0 >= rows) return;  // uniform
      const bool in = r0 + tk < rows;
      const int64_t r = in ? r0 + tk : rows - 1;
      const int t = (int)(r / a.Hq), h = (int)(r - (int64_t)t * a.Hq), hc = h * D;
      const __half* src =
          a.q_item > 0 ? a.q + ((int64_t)(hc / a.q_item) * c.T + t) * a.q_item + hc % a.q_item
                       : a.q + t * a.q_stride + hc;
      const f16x8 v = ((const f16x8*)src)[li];
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = (float)v[e];
      head_norm_rope<D>(x, a.qw ? (const f16x8*)a.qw + li : nullptr,
                        a.cos ? (const f16x8*)(a.cos + t * a.cs_stride) + li : nullptr,
                        a.cos ? (const f16x8*)(a.sin + t * a.cs_stride) + li : nullptr, li, a.eps);
      f16x8 o;
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = (_Float16)x[e];
      if (in) ((f16x8*)(a.q_out + r * D))[li] = o;
    }
    return;
  }
  int slot = wave / (2 * c.Hk);
  const int rest = wave - slot * 2 * c.Hk, h = rest >> 1;
  const bool isv = rest & 1;
  if (slot >= a.slots) return;
  int b;
  if (c.starts) {
    b = slot_sequence(c, 1, kBlkTokens, 2, slot);
  } else {
    b = slot / a.units;
    slot -= b * a.units;
  }
  if (slot < 0) return;  // (starts that begin past 0)
  const int s0 = c.start(b), n = max((c.starts ? c.start(b + 1) : s0 + c.each) - s0, 0);
  const int hi = c.length(b), first = hi - n;  // position of the first new token
  const int lo = max(first, 0);
  const int nb = lo / kBlkTokens + slot;       // the sequence's block
  const int64_t p0 = (int64_t)nb * kBlkTokens;
  if (n == 0 || p0 >= hi) return;
  const int pg = c.page_of(b, (int)(p0 >> c.page_shift));
  if (pg < 0) return;
  const int bpp = 1 << (c.page_shift - 4);     // blocks of a page
  const int64_t blk = ((int64_t)pg * c.Hk + h) * bpp + (nb & (bpp - 1));
  // the block's new tokens: 8 values of token TP p + tk a pass
  float x[NP][8];
  bool fresh[NP];
  const __half* src = isv ? a.v : a.k;
  const int64_t stride = isv ? a.v_stride : a.k_stride;
#pragma unroll
  for (int p = 0; p < NP; ++p) {
    const int64_t pos = p0 + TP * p + tk;
    fresh[p] = pos >= lo && pos < hi;
    const int64_t t = fresh[p] ? s0 + (pos - first) : s0;
    const f16x8 v = fresh[p] ? ((const f16x8*)(src + t * stride + h * D))[li] : f16x8{};
    if (isv) {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[p][e] = (float)v[e];
    } else {
      double y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = (double)v[e];
      head_norm_rope<D>(y, a.kw ? (const f16x8*)a.kw + li : nullptr,
                        a.cos ? (const f16x8*)(a.cos + t * a.cs_stride) + li : nullptr,
                        a.cos ? (const f16x8*)(a.sin + t * a.cs_stride) + li : nullptr, li, a.eps);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        // to fp32, and from there to the pages' type, as torch converts fp64
        // (the asm keeps the compiler from making one conversion of the two)
        x[p][e] = (float)y[e];
        asm("" : "+v"(x[p][e]));
      }
    }
  }
  if constexpr (FP8) {
    float amax = 0.f;
#pragma unroll
    for (int p = 0; p < NP; ++p)
      if (fresh[p]) {
#pragma unroll
        for (int e = 0; e < 8; ++e) amax = fmaxf(amax, finite(x[p][e]) ? fabsf(x[p][e]) : 0.f);
      }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) amax = fmaxf(amax, __shfl_xor(amax, o));
    uint8_t* sc = (isv ? c.vs : c.ks) + blk;
    const bool had = p0 < lo;
    const int need = scale_byte(amax), old = had ? *sc : need;
    const int byte = max(need, old);
    const float inv = e8m0_value(max(254 - byte, 0));         // 2^-(byte - 127)
    const float down = e8m0_value(max(127 + old - byte, 0));  // the kept codes' factor
    if (lane == 0) *sc = (uint8_t)byte;
    if (!isv) {
      uint8_t* dst = (uint8_t*)c.k + blk * kBlkTokens * D;
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        const int64_t pos = p0 + TP * p + tk;
        u32x2* at = (u32x2*)(dst + (TP * p + tk) * D) + li;
        u32x2 w = fresh[p] ? quantize8(x[p], inv) : u32x2{0u, 0u};
        if (pos < lo) {
          if (byte == old) continue;
          w = *at;
          w = u32x2{rescale4(w[0], down), rescale4(w[1], down)};
        }
        *at = w;
      }
    } else {
      // to columns through LDS
      uint8_t* ld = smem[wib];
#pragma unroll
      for (int p = 0; p < NP; ++p)
        *((u32x2*)(ld + (TP * p + tk) * D) + li) = fresh[p] ? quantize8(x[p], inv) : u32x2{0u, 0u};
      paged_lds_sync();
      const int kept = (int)min((int64_t)kBlkTokens, max(lo - p0, (int64_t)0));
      u32x4* dst = (u32x4*)((uint8_t*)c.v + blk * kBlkTokens * D);
#pragma unroll
      for (int d = 0; d < D; d += 64) {
        u32x4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint8_t* col = ld + 4 * i * D + d + lane;
          w[i] = (uint32_t)col[0] | (uint32_t)col[D] << 8 | (uint32_t)col[2 * D] << 16 |
                 (uint32_t)col[3 * D] << 24;
        }
        if (kept > 0) {
          u32x4 o = dst[d + lane];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int k4 = min(max(kept - 4 * i, 0), 4);  // kept tokens of the word
            const uint32_t mask = k4 == 4 ? ~0u : (1u << (8 * k4)) - 1u;
            uint32_t ow = o[i];
            if (byte != old) ow = rescale4(ow, down);
            w[i] = (w[i] & ~mask) | (ow & mask);
          }
        }
        dst[d + lane] = w;
      }
    }
  } else {
    __half* base = (__half*)(isv ? c.v : c.k) + blk * kBlkTokens * D;
    f16x8 o[NP];
#pragma unroll
    for (int p = 0; p < NP; ++p)
#pragma unroll
      for (int e = 0; e < 8; ++e) o[p][e] = (_Float16)x[p][e];
    if (!isv) {
#pragma unroll
      for (int p = 0; p < NP; ++p)
        if (fresh[p]) ((f16x8*)(base + (TP * p + tk) * D))[li] = o[p];
    } else {
      _Float16* ld = (_Float16*)smem[wib];
#pragma unroll
      for (int p = 0; p < NP; ++p) *((f16x8*)(ld + (TP * p + tk) * D) + li) = o[p];
      paged_lds_sync();
      const int t0 = (int)max(lo - p0, (int64_t)0), t1 = (int)min((int64_t)kBlkTokens, hi - p0);
#pragma unroll
      for (int d = 0; d < D; d += 64) {
        _Float16* dst = (_Float16*)base + (d + lane) * kBlkTokens;
        f16x8 w[2];
#pragma unroll
        for (int i = 0; i < kBlkTokens; ++i) w[i >> 3][i & 7] = ld[i * D + d + lane];
        if (t0 == 0 && t1 == kBlkTokens) {
          ((f16x8*)dst)[0] = w[0];
          ((f16x8*)dst)[1] = w[1];
        } else {
#pragma unroll
          for (int i = 0; i < kBlkTokens; ++i)
            if (i >= t0 && i < t1) dst[i] = w[i >> 3][i & 7];
        }
      }
    }
  }
}

bool al(const void* p, int n) { return ((uintptr_t)p & (n - 1)) == 0; }

}  // namespace

int paged_view(const glq_paged_cache* c, const int32_t* starts, int64_t tokens, PagedView& w) {
  GLQ_CHECK(c != nullptr, "null cache");
  GLQ_CHECK(c->head_dim == 64 || c->head_dim == 128, "head_dim must be 64 or 128 (got %lld)",
            (long long)c->head_dim);
  GLQ_CHECK(c->page_size >= 16 && c->page_size <= 1024 &&
                (c->page_size & (c->page_size - 1)) == 0,
            "page_size must be a power of two in [16, 1024] (got %lld)", (long long)c->page_size);
  GLQ_CHECK(c->kv_heads > 0 && c->kv_heads <= 1024, "kv_heads must be in [1, 1024]");
  GLQ_CHECK(c->seqs >= 0 && c->seqs <= (1 << 20), "seqs must be in [0, 2^20]");
  GLQ_CHECK(tokens >= 0 && tokens <= (1 << 24), "tokens must be in [0, 2^24]");
  GLQ_CHECK(c->pages >= 0 && c->pages < (1ll << 31) && c->max_pages >= 0 &&
                c->max_pages <= (1ll << 30) / c->page_size && c->table_stride >= c->max_pages,
            "pages < 2^31, max_pages * page_size <= 2^30 and table_stride >= max_pages required");
  if (!starts)
    GLQ_CHECK(c->seqs == 0 ? tokens == 0 : tokens % c->seqs == 0,
              "without starts every sequence has the same number of new tokens (%lld tokens, "
              "%lld sequences)", (long long)tokens, (long long)c->seqs);
  w.B = (int)c->seqs;
  w.T = (int)tokens;
  w.each = starts || c->seqs == 0 ? 0 : (int)(tokens / c->seqs);
  if (tokens == 0 || c->seqs == 0) return GLQ_OK;
  GLQ_CHECK(c->pages > 0 && c->max_pages > 0, "a cache of no pages");
  GLQ_CHECK(c->k_pages && c->v_pages && c->page_table && c->lengths, "null pointer argument");
  GLQ_CHECK(!c->k_scales == !c->v_scales, "k and v scales come together (8-bit pages) or not at all");
  GLQ_CHECK(al(c->k_pages, 16) && al(c->v_pages, 16) && al(c->page_table, 4) &&
                al(c->lengths, 4) && al(starts, 4),
            "pages must be 16-byte aligned, page_table, lengths and starts 4-byte");
  w.k = c->k_pages; w.v = c->v_pages;
  w.ks = (uint8_t*)c->k_scales; w.vs = (uint8_t*)c->v_scales;
  w.table = c->page_table; w.table_stride = c->table_stride;
  w.lengths = c->lengths; w.starts = starts;
  w.pages = (int)c->pages; w.max_pages = (int)c->max_pages; w.Hk = (int)c->kv_heads;
  w.page_shift = __builtin_ctzll(c->page_size);
  return GLQ_OK;
}

}  // namespace glq

extern "C" int glq_paged_append(const glq_paged_append_params* p, void* stream) {
  using namespace glq;
  clear_error();
  GLQ_CHECK(p != nullptr, "null params");
  const glq_paged_cache* cache = &p->cache;
  const int32_t* starts = p->starts;
  const int64_t tokens = p->tokens, k_stride = p->k_stride, v_stride = p->v_stride;
  const int64_t q_heads = p->q_heads, q_stride = p->q_stride, q_item_rows = p->q_item_rows;
  const int64_t cs_stride = p->cs_stride;
  const void *k = p->k, *v = p->v, *q = p->q, *cos = p->cos, *sin = p->sin;
  const void *q_norm_w = p->q_norm_w, *k_norm_w = p->k_norm_w;
  void* q_out = p->q_out;
  AppendArgs a{};
  if (int rc = paged_view(cache, starts, tokens, a.c)) return rc;
  const int64_t D = cache->head_dim, Hk = cache->kv_heads;
  if (tokens == 0 || cache->seqs == 0) return GLQ_OK;
  GLQ_CHECK(k && v, "null pointer argument");
  GLQ_CHECK(k_stride >= Hk * D && v_stride >= Hk * D && k_stride % 8 == 0 && v_stride % 8 == 0,
            "k and v row strides must cover the heads and be multiples of 8");
  GLQ_CHECK(al(k, 16) && al(v, 16), "k and v must be 16-byte aligned");
  GLQ_CHECK(!cos == !sin && cs_stride >= 0 && cs_stride % 8 == 0 &&
                (cs_stride == 0 || cs_stride >= D),
            "cos and sin come together, cs_stride 0 or a multiple of 8 that covers head_dim");
  GLQ_CHECK(al(cos, 16) && al(sin, 16) && al(q_norm_w, 16) && al(k_norm_w, 16),
            "cos, sin and norm weights must be 16-byte aligned");
  if (q) {
    GLQ_CHECK(q_heads > 0 && q_heads % Hk == 0 && q_heads <= 8192,
              "q_heads must be a positive multiple of kv_heads (<= 8192)");
    GLQ_CHECK(q_out && al(q, 16) && al(q_out, 16), "q and q_out must be 16-byte aligned");
    GLQ_CHECK(q_item_rows >= 0 && q_item_rows % D == 0 &&
                  (q_item_rows == 0 || (q_heads * D) % q_item_rows == 0),
              "q_item_rows must be 0 or a multiple of head_dim dividing q_heads * head_dim");
    GLQ_CHECK(q_item_rows > 0 || (q_stride >= q_heads * D && q_stride % 8 == 0),
              "q's row stride must cover the heads and be a multiple of 8");
    const int64_t row = q_heads * D;
    const bool own = q_item_rows == 0 && (q_stride == row || tokens == 1);
    GLQ_CHECK((q == q_out && own) ||
                  apart(q, ((tokens - 1) * (q_item_rows > 0 ? row : q_stride) + row) * 2, q_out,
                        tokens * row * 2),
              "q_out must not overlap q (but for rows side by side, rotated in place)");
    // (other waves read these while q_out is written)
    const int64_t head = D * 2, out_bytes = tokens * row * 2;
    const int64_t cs_step = cs_stride > 0 ? cs_stride * 2 : head;
    const int64_t cs_rows = cs_stride > 0 ? tokens : 1;
    GLQ_CHECK(rows_apart(k, Hk * head, k_stride * 2, tokens, q_out, out_bytes) &&
                  rows_apart(v, Hk * head, v_stride * 2, tokens, q_out, out_bytes) &&
                  (!cos || (rows_apart(cos, head, cs_step, cs_rows, q_out, out_bytes) &&
                            rows_apart(sin, head, cs_step, cs_rows, q_out, out_bytes))) &&
                  (!q_norm_w || apart(q_norm_w, head, q_out, out_bytes)) &&
                  (!k_norm_w || apart(k_norm_w, head, q_out, out_bytes)),
              "q_out must not overlap k, v, cos, sin or the norm weights");
  }
  a.q = (const __half*)q; a.k = (const __half*)k; a.v = (const __half*)v;
  a.q_stride = q_stride; a.k_stride = k_stride; a.v_stride = v_stride;
  a.q_item = (int)q_item_rows;
  a.qw = (const __half*)q_norm_w; a.kw = (const __half*)k_norm_w;
  a.cos = (const __half*)cos; a.sin = (const __half*)sin; a.cs_stride = cs_stride;
  a.q_out = (__half*)q_out; a.Hq = q ? (int)q_heads : 0; a.eps = p->eps;
  // blocks: a sequence's n new tokens touch at most (n + 14) / 16 + 1 of them
  a.units = (int)((a.c.each + kBlkTokens - 2) / kBlkTokens + 1);
  const int64_t slots = starts ? tokens / kBlkTokens + 2 * cache->seqs : cache->seqs * a.units;
  const int64_t kvw = align_up(slots * 2 * Hk, kAppThreads / 64);
  const int64_t rows = q ? tokens * q_heads : 0;
  const int64_t per = 64 / (D / 8) * kQPasses;
  const int64_t qw = (rows + per - 1) / per;
  const int64_t blocks = (kvw + qw + kAppThreads / 64 - 1) / (kAppThreads / 64);
  GLQ_CHECK(blocks < (1ll << 24), "batch of too many (token, head) rows");
  a.kv_waves = (int)kvw;
  a.slots = (int)slots;
  auto kern = D == 128 ? (a.c.ks ? paged_append_kernel<128, true> : paged_append_kernel<128, false>)
                       : (a.c.ks ? paged_append_kernel<64, true> : paged_append_kernel<64, false>);
  kern<<<dim3((unsigned)blocks), dim3(kAppThreads), 0, (hipStream_t)stream>>>(a);
  GLQ_LAUNCH_CHECK("paged_append_kernel");
  return GLQ_OK;
}
