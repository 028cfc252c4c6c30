// Causal attention of a batch's new tokens over a paged key/value cache
// (layout and formats: glq_paged.h), a few query rows a KV head at a time.

#include <algorithm>
#include <type_traits>

#include "glq_paged_attn.h"

namespace glq {
namespace {

constexpr int kPaThreads = 512;
constexpr int kPaWaves = kPaThreads / 64;
constexpr int kPaGrid = 256;

// A wave takes 16 query rows (tokens x the KV head's q heads) of one KV head
// over some of their positions, a tile of 16 KB at a time:
//   S^T = K Q^T   v_mfma_f32_16x16x32_f16, A = 16 positions of K, B = the rows
//   O^T += V^T P^T                         A = 16 columns of V,   B = the weights
// so that a row's scores of a tile lie on the four lanes of its column, and
// need two exchanges for their maximum and none for the second product.
//
// Bound by the pages' bytes, which go from memory to registers, 16 bytes a lane
// and load, without LDS: each is used once.  8 waves of 200 registers a CU keep
// 128 KB in flight there.  64 sequences of 3 to 8000 positions, 8-bit pages:
// 61 us, 4.8 TB/s, what a copy reaches (a read alone 6.1); one sequence of
// 130000: 36 us, 3.7 TB/s; of 517, 10 us, of which 5 are an empty launch's.
template <int D, bool FP8, bool SINKS>
struct RowAttention {
  // A tile is TP positions, in NS parts of TS; of each part, lane group kb has P
  // consecutive ones, as rows 4 kb + j of the NT products of 16 positions and as
  // the P values of a V column, so the weights go from one product to the next
  // in registers.  64 positions of 128 columns or 128 of 64: 16 KB of codes.
  static constexpr int TS = FP8 ? 64 : 32, NS = 128 / D, TP = NS * TS;
  static constexpr int P = TS / 4, NT = TS / 16, NM = P / 8;
  static constexpr int KL = FP8 ? D / 64 : D / 32;  // 16-byte pieces of a K row and lane
  static constexpr int NC = D / 16;
  static constexpr int S = FP8 ? 1 : 2;             // bytes of a value

  struct Tile {
    u32x4 k[NS][NT][KL], v[NS][NC];
    int ks[NS], vs[NS];
    bool bad[NS];
  };

  const PagedView& c;
  int b, g, li, kb, rep, window, sinks;
  float scale2;
  RowSet r;
  f16x8 q[D / 32];
  float m, l;
  f32x4 o[NC];

  __device__ RowAttention(const PagedView& c_) : c(c_) {
    li = threadIdx.x & 15;
    kb = (threadIdx.x >> 4) & 3;
  }

  __device__ void begin(const __half* qp, int Hq) {
    const int t = r.s0 + r.row / rep, h = g * rep + r.row % rep;
    const f16x8* src = (const f16x8*)(qp + ((int64_t)t * Hq + h) * D);
#pragma unroll
    for (int s = 0; s < D / 32; ++s)  // (e4m3: the two halves of a 16-code piece)
      q[s] = src[FP8 ? 8 * (s >> 1) + 2 * kb + (s & 1) : 4 * s + kb];
    m = -__builtin_inff();
    l = 0.f;
#pragma unroll
    for (int i = 0; i < NC; ++i) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  // Page ids of a tile's blocks as a lane needs them, for k's rows and for v
  // (and the scales, which are the blocks' of v's lanes).
  struct Ids {
    int k[NS], v[NS];
  };
  __device__ static int k_block(int tile, int u, int li) {
    return (tile * NS + u) * (TS / 16) + (FP8 ? li >> 2 : li >> 3);
  }
  __device__ static int v_block(int tile, int u, int kb) {
    return (tile * NS + u) * (TS / 16) + (FP8 ? kb : kb >> 1);
  }
  __device__ Ids ids(int tile) const {
    const int bps = c.page_shift - 4;
    const int* row = c.table + b * c.table_stride;
    Ids r;
#pragma unroll
    for (int u = 0; u < NS; ++u) {
      r.k[u] = row[min(k_block(tile, u, li) >> bps, c.max_pages - 1)];
      r.v[u] = row[min(v_block(tile, u, kb) >> bps, c.max_pages - 1)];
    }
    return r;
  }

  // A block's place in the pool; ids out of range read page 0.
  __device__ int64_t place(int p, int blk) const {
    const int bps = c.page_shift - 4;
    return ((int64_t)((unsigned)p < (unsigned)c.pages ? p : 0) * c.Hk + g << bps) +
           (blk & ((1 << bps) - 1));
  }
  __device__ void load_k(Tile& x, int tile, Ids id) const {
#pragma unroll
    for (int u = 0; u < NS; ++u) {
      if constexpr (FP8) {
        const int64_t vblk = place(id.v[u], v_block(tile, u, kb));
        x.ks[u] = c.ks[vblk];
        x.vs[u] = c.vs[vblk];
      }
      x.bad[u] = (unsigned)id.v[u] >= (unsigned)c.pages;
      const char* p = (const char*)c.k + place(id.k[u], k_block(tile, u, li)) * (16 * D * S) +
                      ((FP8 ? 0 : 8 * ((li >> 2) & 1)) + (li & 3)) * D * S + 16 * kb;
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int t = 0; t < KL; ++t) x.k[u][i][t] = *(const u32x4*)(p + 4 * i * D * S + 64 * t);
    }
  }
  __device__ void load_v(Tile& x, int tile, Ids id) const {
#pragma unroll
    for (int u = 0; u < NS; ++u) {
      const char* p = (const char*)c.v + place(id.v[u], v_block(tile, u, kb)) * (16 * D * S) +
                      li * 16 * S + (FP8 ? 0 : 16 * (kb & 1));
#pragma unroll
      for (int i = 0; i < NC; ++i) x.v[u][i] = *(const u32x4*)(p + 16 * i * 16 * S);
    }
  }

  __device__ static f16x8 k_frag(const u32x4 (&k)[KL], int s) {
    if constexpr (FP8)
      return fp8x8_to_f16(k[s >> 1][2 * (s & 1)], k[s >> 1][2 * (s & 1) + 1]);
    else
      return __builtin_bit_cast(f16x8, k[s]);
  }
  __device__ static f16x8 v_frag(u32x4 v, int mm) {
    if constexpr (FP8)
      return fp8x8_to_f16(v[2 * mm], v[2 * mm + 1]);
    else
      return __builtin_bit_cast(f16x8, v);
  }

  // Online softmax over the tile's positions.  The scale 2^e of a V block goes
  // into the exponent: w = 2^(t + e - m) with m the largest t + e so far, so
  // that w keeps its bits where the block's share of the result is largest.  It
  // is rounded to fp16 for the product alone, in which V's codes are exact; the
  // denominator sums w 2^-e in fp32.  The largest weight is 1 and loses nothing:
  // outputs are 2.1e-4 to 2.2e-4 off the exact ones (root mean square, relative),
  // 2.1e-4 of it their own rounding to fp16.
  // `next_k`: fetches the next tile's k into x, whose k has been used by then.
  template <class Next>
  __device__ void step(Tile& x, int tile, Next next_k) {
    const int p0 = tile * TP + P * kb;
    const bool edge =
        (tile * TP < r.lo_all && !(SINKS && (tile + 1) * TP <= sinks)) || (tile + 1) * TP > r.hi_all;
    float t[NS][NT][4], ev[NS];
    float mx = m;
#pragma unroll
    for (int u = 0; u < NS; ++u) {
      const float ks = FP8 ? e8m0_value(x.ks[u]) * scale2 : scale2;
      ev[u] = FP8 ? e8m0_exponent(x.vs[u]) : 0.f;
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < D / 32; ++s) acc = mfma_16x16x32(k_frag(x.k[u][i], s), q[s], acc);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          t[u][i][j] = x.bad[u] ? __builtin_nanf("") : fmaf(acc[j], ks, ev[u]);
        if (edge) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int p = p0 + u * TS + 4 * i + j;
            if ((p < r.lo && !(SINKS && p < sinks)) || p >= r.hi)
              t[u][i][j] = -__builtin_inff();
          }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) mx = fmaxf(mx, t[u][i][j]);
      }
    }
    next_k();
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
    f16x8 w[NS][NM];
#pragma unroll
    for (int u = 0; u < NS; ++u) {
      float ls = 0.f;
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float e = __builtin_amdgcn_exp2f(t[u][i][j] - mf);
          ls += e;
          w[u][i >> 1][4 * (i & 1) + j] = (_Float16)e;
        }
      // (a block that the row does not see may hold any scale)
      l = ls == 0.f ? l : fmaf(ls, __builtin_amdgcn_exp2f(-ev[u]), l);
    }
    // weight 0 times an inf or a NaN behind a row's positions is not 0
    if (!edge || __builtin_amdgcn_ballot_w64(odd(x)) == 0) {
#pragma unroll
      for (int u = 0; u < NS; ++u)
#pragma unroll
        for (int i = 0; i < NC; ++i)
#pragma unroll
          for (int mm = 0; mm < NM; ++mm)
            o[i] = mfma_16x16x32(v_frag(x.v[u][i], mm), w[u][mm], o[i]);
    } else {
      // a token's rows at a time, with zeros for the positions that it does
      // not see
      const int tok = r.row / rep, last = __builtin_amdgcn_readlane(tok, 15);
#pragma nounroll
      for (int k = __builtin_amdgcn_readfirstlane(tok); k <= last; ++k) {
        const int pos = r.first + k, hi = pos + 1, lo = window > 0 ? pos - window + 1 : 0;
#pragma unroll
        for (int u = 0; u < NS; ++u) {
          const int pu = p0 + u * TS;
          const int n0 = min(max(lo - pu, 0), P), n1 = min(max(hi - pu, 0), P);
          const int ns = SINKS ? min(max(sinks - pu, 0), n1) : 0;
          constexpr int E = FP8 ? 4 : 2;  // values of a word
          auto below = [](int n) {        // the bits of its first n values
            return n <= 0 ? 0u : n >= E ? ~0u : (1u << (32 / E * n)) - 1u;
          };
          u32x4 keep;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            keep[e] = (below(n1 - E * e) & ~below(n0 - E * e)) | below(ns - E * e);
#pragma unroll
          for (int i = 0; i < NC; ++i) {
            const u32x4 v = x.v[u][i] & keep;
            f32x4 on = o[i];
#pragma unroll
            for (int mm = 0; mm < NM; ++mm) on = mfma_16x16x32(v_frag(v, mm), w[u][mm], on);
#pragma unroll
            for (int j = 0; j < 4; ++j) o[i][j] = tok == k ? on[j] : o[i][j];
          }
        }
      }
    }
  }

  // Whether this lane's part of V holds an infinity or a NaN.
  __device__ static bool odd(const Tile& x) {
    uint32_t any = 0;
#pragma unroll
    for (int u = 0; u < NS; ++u)
#pragma unroll
      for (int i = 0; i < NC; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          // the largest exponent field carries into the sign's place
          if constexpr (FP8)
            any |= (x.v[u][i][e] & 0x7F7F7F7Fu) + 0x01010101u;
          else
            any |= (x.v[u][i][e] & 0x7FFF7FFFu) + 0x04000400u;
        }
    return (any & (FP8 ? 0x80808080u : 0x80008000u)) != 0;
  }
};

// The tiles of each of a sequence's units.
template <int TP, bool SINKS>
__device__ __forceinline__ Span<TP, SINKS> sequence_span(const RowSet& r, int window, int sinks) {
  return Span<TP, SINKS>(window > 0 ? max(r.first - window + 1, 0) : 0,
                         min(max(r.first + r.n, 0), r.cap), sinks);
}

// The batch's work is a line of tiles: sequence by sequence, unit by unit (KV
// head fastest), the unit's positions.  It is cut into equal pieces, one a
// wave, whatever the lengths: 256 workgroups of 8 waves, a wave's piece running
// over as many units as it does.  A unit inside a piece is written by its wave;
// one that crosses waves is merged by their workgroup through LDS; one that
// crosses workgroups goes through memory, and the last one to arrive (an
// arrival counter, data handed over coherently) merges its parts in order.  So
// a result's sums depend on the lengths alone, and the workspace holds two
// parts a workgroup, not a cache's length of them.
//
// Where every unit fits a workgroup with at most kPaShort tiles a wave, a unit
// gets a workgroup of its own, and nothing goes through memory: one sequence of
// 517 positions 10.2 us, 15.8 without the rule; with 16 tiles a wave, 4
// sequences of 4000 fp16 positions 44 us instead of 33.
constexpr int kPaShort = 4;

// The line, as every wave works it out for itself: 64 sequences a step.
template <int TP, bool SINKS>
struct Line {
  int total, quota, align;

  __device__ static void weigh(const PagedAttnArgs& a, int b, int& tiles, int& units) {
    const PagedView& c = a.c;
    RowSet r;
    r.s0 = c.start(b);
    r.n = max((c.starts ? c.start(b + 1) : r.s0 + c.each) - r.s0, 0);
    r.first = c.length(b) - r.n;
    r.cap = c.max_pages << c.page_shift;
    // 0 for a sequence without new tokens (the rows of others are written even
    // where they see nothing: at least 1)
    tiles = r.n == 0 ? 0 : max(sequence_span<TP, SINKS>(r, a.window, a.sinks).n, 1);
    // (a sequence of more rows is the second form's)
    units = c.starts && r.n * a.rep > kPaMostRows ? 0 : (r.n * a.rep + kPaRows - 1) / kPaRows * c.Hk;
  }
  __device__ int rounded(int tiles) const { return (tiles + align - 1) / align * align; }

  __device__ Line(const PagedAttnArgs& a) : align(1) {
    const int lane = threadIdx.x & 63;
    int sum = 0, widest = 0, units = 0;
    for (int b = lane; b < a.c.B; b += 64) {
      int t, u;
      weigh(a, b, t, u);
      sum += t * u;
      units += u;
      if (u) widest = max(widest, t);
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
      sum += __shfl_xor(sum, o);
      units += __shfl_xor(units, o);
      widest = max(widest, __shfl_xor(widest, o));
    }
    sum = __builtin_amdgcn_readfirstlane(sum);
    units = __builtin_amdgcn_readfirstlane(units);
    widest = __builtin_amdgcn_readfirstlane(widest);
    const int waves = (int)gridDim.x * kPaWaves;
    if (units <= (int)gridDim.x && widest <= kPaShort * kPaWaves) {
      quota = max((widest + kPaWaves - 1) / kPaWaves, 1);
      align = quota * kPaWaves;
      total = units * align;
    } else {
      quota = (sum + waves - 1) / waves;
      total = sum;
    }
  }

  // Sequence of the line's tile p, and p's place from its first one, and what
  // weigh says of the sequence; -1 past the end.
  __device__ int find(const PagedAttnArgs& a, int p, int& off, int& tiles, int& units) const {
    const int lane = threadIdx.x & 63;
    for (int base = 0, before = 0; base < a.c.B; base += 64) {
      int t = 0, u = 0;
      if (base + lane < a.c.B) weigh(a, base + lane, t, u);
      const int w = rounded(t) * u;
      int upto = w;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int v = __shfl_up(upto, o);
        if (lane >= o) upto += v;
      }
      const int at = p - (before + upto - w);
      const uint64_t hit = __builtin_amdgcn_ballot_w64(at >= 0 && at < w);
      if (hit) {
        const int l = __builtin_ctzll(hit);
        off = __builtin_amdgcn_readlane(at, l);
        tiles = __builtin_amdgcn_readlane(t, l);
        units = __builtin_amdgcn_readlane(u, l);
        return base + l;
      }
      before += __builtin_amdgcn_readlane(upto, 63);
    }
    return -1;
  }
};

template <int D, bool FP8, bool SINKS>
__global__ __launch_bounds__(kPaThreads) void paged_rows_kernel(PagedAttnArgs a) {
  using RA = RowAttention<D, FP8, SINKS>;
  constexpr int TP = RA::TP, PS = D + 4;
  struct Seg {  // a unit's piece that did not stay within its wave
    int b, unit, tiles, ended, line;  // line: of the unit's first tile
  };
  extern __shared__ __align__(16) float parts[];  // [wave][2][rows][PS]
  __shared__ Seg seg[kPaWaves][2];
  __shared__ int flag;
  const PagedView& c = a.c;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int Hq = c.Hk * a.rep;
  const Line<TP, SINKS> line(a);
  const int wg_quota = line.quota * kPaWaves, wg0 = blockIdx.x * wg_quota;
  if (wg0 >= line.total) return;  // uniform
  if (lane < 2) seg[wave][lane].unit = -1;

  RA x(c);
  x.scale2 = a.scale2;
  x.rep = a.rep;
  x.window = a.window;
  x.sinks = a.sinks;
  {
    int off = 0, left = line.quota, pos = wg0 + wave * line.quota;
    int tiles = 0, units = 0, b = line.find(a, pos, off, tiles, units);
    while (b >= 0 && left > 0) {  // (b grows, or off to its end)
      const int size = line.rounded(tiles);
      if (off >= size * units) {
        if (++b >= c.B) break;
        off = 0;
        line.weigh(a, b, tiles, units);
        continue;
      }
      const int unit = off / size, t0 = off - unit * size;
      const int run = min(size - t0, left), t1 = min(t0 + run, tiles);
      const int at = pos - t0;
      off += run;
      pos += run;
      left -= run;
      if (t0 >= t1) continue;
      const int qt = unit / c.Hk;
      x.b = b;
      x.g = unit - qt * c.Hk;
      set_rows<kPaRows>(x.r, c, b, qt * kPaRows, a.rep, a.window, x.li);
      const Span<TP, SINKS> span = sequence_span<TP, SINKS>(x.r, a.window, a.sinks);
      // k and v of the next tile are fetched as soon as the present one's have
      // been used, page ids a tile before them
      {
        const int e = span.begin + t1;
        int t = span.begin + t0;
        typename RA::Tile tile;
        typename RA::Ids id = x.ids(span.place(t)), ahead = x.ids(span.place(t + 1));
        x.begin(a.q, Hq);
        x.load_k(tile, span.place(t), id);
        x.load_v(tile, span.place(t), id);
        for (; t < e; ++t) {
          x.step(tile, span.place(t), [&] {
            if (t + 1 < e) {
              id = ahead;
              ahead = x.ids(span.place(t + 2));
              x.load_k(tile, span.place(t + 1), id);
            }
          });
          if (t + 1 < e) x.load_v(tile, span.place(t + 1), id);
        }
      }
      x.l += __shfl_xor(x.l, 16);
      x.l += __shfl_xor(x.l, 32);
      if (t0 == 0 && t1 == tiles) {
        if (x.r.live) {
          const int tok = x.r.row / a.rep;
          __half* dst = a.out + ((int64_t)(x.r.s0 + tok) * Hq + x.g * a.rep + x.r.row % a.rep) * D;
#pragma unroll
          for (int i = 0; i < RA::NC; ++i)
            store_row(dst + 16 * i + 4 * x.kb, x.o[i], x.l, x.r.first + tok, x.r.cap);
        }
      } else {
        const int s = t0 == 0;
        if (x.li < a.rows) {
          float* mine = parts + ((wave * 2 + s) * a.rows + x.li) * PS;
#pragma unroll
          for (int i = 0; i < RA::NC; ++i) *(f32x4*)(mine + 16 * i + 4 * x.kb) = x.o[i];
          if (x.kb == 0) {
            mine[D] = x.m;
            mine[D + 1] = x.l;
          }
        }
        if (lane == 0) seg[wave][s] = Seg{b, unit, tiles, t1 == tiles, at};
      }
    }
  }
  __syncthreads();
  // Chains of pieces of one unit: the one that the workgroup begins in (slot 0 of
  // its first wave), and those that begin in a wave (slot 1 of it).  Thread (row,
  // 4 columns).
  const int row = tid / (D / 4), d4 = 4 * (tid % (D / 4));
  auto store = [&](const RowSet& r, int g, const Merge& acc) {
    const int tok = r.row / a.rep;
    store_row(a.out + ((int64_t)(r.s0 + tok) * Hq + g * a.rep + r.row % a.rep) * D + d4, acc.o,
              acc.den, r.first + tok, r.cap);
  };
  Seg out[2];  // chains that another workgroup has parts of: not begun, not ended here
  out[0].unit = out[1].unit = -1;
  // a bit a (wave, slot)
  const Seg* all = &seg[0][0];
  const uint64_t there =
      __builtin_amdgcn_ballot_w64(lane < 2 * kPaWaves && all[lane % (2 * kPaWaves)].unit >= 0);
  const uint64_t last =
      __builtin_amdgcn_ballot_w64(lane < 2 * kPaWaves && all[lane % (2 * kPaWaves)].ended);
  for (uint64_t heads = there & (0xAAAAAAAAAAAAAAAAull | 1); heads; heads &= heads - 1) {  // uniform
    const int h = __builtin_ctzll(heads), v0 = h >> 1, s0 = h & 1;
    const Seg head = all[h];
    bool ended = last >> h & 1;
    int v1 = v0 + 1;
    while (!ended && v1 < kPaWaves && (there >> 2 * v1 & 1)) ended = last >> 2 * v1++ & 1;
    RowSet r;
    const int qt = head.unit / c.Hk, g = head.unit - qt * c.Hk;
    set_rows<kPaRows>(r, c, head.b, qt * kPaRows, a.rep, a.window, row & 15);
    if (row >= a.rows) r.live = false;
    Merge acc;
    if (r.live) {
      for (int w = v0; w < v1; ++w) {
        const float* p = parts + ((w * 2 + (w == v0 ? s0 : 0)) * a.rows + row) * PS;
        acc.add(p[D], p[D + 1], *(const f32x4*)(p + d4));
      }
    }
    if (s0 && ended) {
      if (r.live) store(r, g, acc);
      continue;
    }
    out[s0] = head;
    if (r.live) {
      float* my = a.part + ((int64_t)(blockIdx.x * 2 + s0) * kPaRows + row) * PS;
      handoff_put((uint64_t*)(my + d4), __builtin_bit_cast(uint64_t, float2{acc.o[0], acc.o[1]}));
      handoff_put((uint64_t*)(my + d4) + 1,
                  __builtin_bit_cast(uint64_t, float2{acc.o[2], acc.o[3]}));
      if (d4 == 0)
        handoff_put((uint64_t*)(my + D), __builtin_bit_cast(uint64_t, float2{acc.M, acc.den}));
    }
  }
  // The last workgroup of a unit to arrive merges its parts: thread (group,
  // row, 4 columns), the groups taking the parts in turn, 8 in flight.
#pragma unroll
  for (int s0 = 0; s0 < 2; ++s0) {
    const Seg head = out[s0];
    if (head.unit < 0) continue;  // uniform
    const int w0 = head.line / wg_quota, w1 = (head.line + head.tiles - 1) / wg_quota;
    const int qt = head.unit / c.Hk, g = head.unit - qt * c.Hk;
    const int slot = c.starts ? (int)((int64_t)c.start(head.b) * a.rep / kPaRows) + head.b
                              : head.b * a.slots_each;
    unsigned* cnt = a.count + (int64_t)(slot + qt) * c.Hk + g;
    if (!handoff_arrive(cnt, (unsigned)(w1 - w0 + 1), &flag)) continue;
    const int groups = kPaThreads / (a.rows * (D / 4)), grp = row / a.rows, rw = row - grp * a.rows;
    Merge acc;
    const float* p0 = a.part + (int64_t)rw * PS;
    for (int w = w0 + grp; w <= w1; w += 8 * groups) {
      float2 ml[8], o[8][2];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int ww = min(w + j * groups, w1);
        const float* p = p0 + (int64_t)(ww * 2 + (ww == w0)) * (kPaRows * PS);
        ml[j] = __builtin_bit_cast(float2, handoff_get((const uint64_t*)(p + D)));
        o[j][0] = __builtin_bit_cast(float2, handoff_get((const uint64_t*)(p + d4)));
        o[j][1] = __builtin_bit_cast(float2, handoff_get((const uint64_t*)(p + d4) + 1));
      }
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (w + j * groups <= w1)
          acc.add(ml[j].x, ml[j].y, f32x4{o[j][0].x, o[j][0].y, o[j][1].x, o[j][1].y});
    }
    if (groups > 1) {  // through LDS, whose pieces have been merged
      float* mine = parts + (grp * a.rows + rw) * PS;
      *(f32x4*)(mine + d4) = acc.o;
      if (d4 == 0) {
        mine[D] = acc.M;
        mine[D + 1] = acc.den;
      }
      __syncthreads();
      if (grp == 0) {
        for (int k = 1; k < groups; ++k) {
          const float* p = parts + (k * a.rows + rw) * PS;
          acc.add(p[D], p[D + 1], *(const f32x4*)(p + d4));
        }
      }
      __syncthreads();
    }
    RowSet r;
    set_rows<kPaRows>(r, c, head.b, qt * kPaRows, a.rep, a.window, rw);
    if (grp == 0 && r.live) store(r, g, acc);
    if (tid == 0) handoff_reset(cnt);
  }
}

}  // namespace
}  // namespace glq

extern "C" int64_t glq_paged_attention_counter_bytes(int64_t seqs, int64_t tokens,
                                                     int64_t q_heads, int64_t kv_heads) {
  using namespace glq;
  if (seqs < 0 || tokens < 0 || q_heads <= 0 || kv_heads <= 0) return -1;
  // a counter a unit of the first form: at most rows / 16 + 1 a sequence and KV head
  const int64_t rep = (q_heads + kv_heads - 1) / kv_heads;
  return align_up(4 * (tokens * rep / kPaRows + seqs) * kv_heads, 256);
}

extern "C" int64_t glq_paged_attention_scratch_bytes(int64_t seqs, int64_t tokens, int64_t q_heads,
                                                     int64_t kv_heads) {
  using namespace glq;
  if (seqs < 0 || tokens < 0 || q_heads <= 0 || kv_heads <= 0) return -1;
  return align_up(std::max((int64_t)kPaGrid * 2 * kPaRows * (128 + 4) * 4,
                           paged_prompt_scratch_bytes(seqs, tokens, q_heads, kv_heads)),
                  256);
}

extern "C" int glq_paged_attention(const glq_paged_attention_params* p, void* stream) {
  using namespace glq;
  clear_error();
  GLQ_CHECK(p != nullptr, "null params");
  const glq_paged_cache* cache = &p->cache;
  const int32_t* starts = p->starts;
  const int64_t tokens = p->tokens, q_heads = p->q_heads, window = p->window, sinks = p->sinks;
  const void* q = p->q;
  void* out = p->out;
  PagedAttnArgs a{};
  if (int rc = paged_view(cache, starts, tokens, a.c)) return rc;
  const int64_t D = cache->head_dim, Hk = cache->kv_heads;
  GLQ_CHECK(q_heads > 0 && q_heads % Hk == 0 && q_heads <= 8192,
            "q_heads must be a positive multiple of kv_heads (<= 8192)");
  GLQ_CHECK(window >= 0 && sinks >= 0, "window and sinks must be >= 0 (0: none)");
  if (tokens == 0 || cache->seqs == 0) return GLQ_OK;
  GLQ_CHECK(q && out && ((uintptr_t)q & 15) == 0 && ((uintptr_t)out & 15) == 0,
            "q and out must be non-null and 16-byte aligned");
  const int64_t cnt = glq_paged_attention_counter_bytes(cache->seqs, tokens, q_heads, Hk);
  const int64_t scr = glq_paged_attention_scratch_bytes(cache->seqs, tokens, q_heads, Hk);
  GLQ_CHECK(p->counters && p->counter_bytes >= cnt && p->scratch && p->scratch_bytes >= scr &&
                ((uintptr_t)p->counters & 3) == 0 && ((uintptr_t)p->scratch & 255) == 0,
            "workspace of %lld (counters) and %lld bytes (scratch, 256-byte aligned) needed "
            "(got %lld, %lld)", (long long)cnt, (long long)scr, (long long)p->counter_bytes,
            (long long)p->scratch_bytes);
  GLQ_CHECK(apart(q, tokens * q_heads * D * 2, out, tokens * q_heads * D * 2),
            "out must not overlap q");
  a.q = (const __half*)q;
  a.out = (__half*)out;
  a.rep = (int)(q_heads / Hk);
  const int64_t cap = cache->max_pages * cache->page_size;
  a.window = window >= cap ? 0 : (int)window;
  a.sinks = a.window > 0 ? (int)std::min(sinks, cap) : 0;
  a.scale2 = p->scale * 1.44269504088896f;
  a.part = (float*)p->scratch;
  a.count = (unsigned*)p->counters;
  const int64_t rows_each = (int64_t)a.c.each * a.rep;
  GLQ_CHECK(tokens * a.rep < (1ll << 30), "batch of too many (token, head) rows");
  // (the first form counts its tiles in 32 bits)
  const int64_t most = (cache->max_pages * cache->page_size + 31) / 32 + 1;
  GLQ_CHECK((!starts && rows_each > kPaMostRows) ||
                std::min(tokens * a.rep / kPaRows + cache->seqs,
                         cache->seqs * ((kPaMostRows + kPaRows - 1) / kPaRows)) * Hk <=
                    (1ll << 31) / most - 1,
            "a batch of too many rows for its page table's length");
  // Many rows take the second form, a sequence at a time; where lengths are the
  // device's, both are launched, each passing over the other's sequences.
  if (starts ? tokens * a.rep > kPaMostRows : rows_each > kPaMostRows) {
    if (int rc = paged_prompt_launch(a, (int)D, (hipStream_t)stream)) return rc;
    if (!starts) return GLQ_OK;
  }
  a.slots_each = (int)((rows_each + kPaRows - 1) / kPaRows);
  // (rows of the pieces' places in LDS: of 8, two threads merge a value's parts;
  // a sequence of 60000 positions 30 us, 37 with 16; 64 of 3000 46 and 45)
  a.rows = !starts && rows_each <= 8 ? 8 : kPaRows;
  const size_t lds = (size_t)kPaWaves * 2 * a.rows * (D + 4) * 4;
  const auto pick = [&](auto sinks_) {
    constexpr bool S = decltype(sinks_)::value;
    return D == 128 ? (a.c.ks ? paged_rows_kernel<128, true, S> : paged_rows_kernel<128, false, S>)
                    : (a.c.ks ? paged_rows_kernel<64, true, S> : paged_rows_kernel<64, false, S>);
  };
  auto kern = a.sinks > 0 ? pick(std::true_type()) : pick(std::false_type());
  static size_t attr[8] = {64 * 1024, 64 * 1024, 64 * 1024, 64 * 1024,
                           64 * 1024, 64 * 1024, 64 * 1024, 64 * 1024};
  if (int rc = set_lds_limit(kern, lds, attr[(a.sinks > 0) * 4 + (D == 64) * 2 + !a.c.ks])) return rc;
  kern<<<dim3(kPaGrid), dim3(kPaThreads), lds, (hipStream_t)stream>>>(a);
  GLQ_LAUNCH_CHECK("paged_rows_kernel");
  return GLQ_OK;
}
