// The best continuations of each prompt over its beams and the vocabulary:
//   c[k][v] = score[k] + logits[k][v] - log sum_u exp(logits[k][u])
// the `num` largest, the lowest (k, v) first among equal ones.

#include <hip/hip_bf16.h>

#include <algorithm>

#include "glq_handoff.h"
#include "glq_paged.h"

namespace glq {
namespace {

constexpr int kBmThreads = 256;
constexpr int kBmWaves = kBmThreads / 64;
constexpr int kBmEach = 8;     // values a thread takes at once
constexpr int kBmMost = 128;   // continuations of a prompt
constexpr int kBmBeams = 64;
constexpr int kBmVocab = 24;   // bits of a token
// Counters have 256 bytes each: arrivals at one line follow each other (2432 of
// them took 6 us less than side by side).  For the same reason many parts of a
// prompt arrive by rows: 152 parts 13.7 us, 14.2 at one counter; 80 parts 12.5 at
// one, 12.9 by rows, 13 parts of one row 13.2 and 13.9.
constexpr int kBmCounter = 64;
constexpr int kBmAtOnce = 100;  // parts of a prompt at one counter
constexpr float kNone = -__builtin_inff();

// e^d for |d| < 700, in fp64 and to 6e-11: 2^(n + f), n from the low bits
// of d log2(e) + 1.5 2^52, 2^f by its Chebyshev series of degree 7 on [-1/2, 1/2].
// Two continuations of different beams compare by sums over the vocabulary, so
// fp32 (1e-7) would put some in the wrong order; fp64 fma runs at fp32's rate
// (5.2 and 4.7 cycles a wave's).  N side by side, so that none waits for itself.
template <int N>
__device__ __forceinline__ void exp_of(double (&d)[N]) {
  constexpr double kLog2e = 1.4426950408889634, kBig = 6755399441055744.0;
  constexpr double kC[] = {0.00015469731972928003, 0.0013333450559898097, 0.009618025602961655,
                           0.05550410941217088, 0.240226512135953, 0.6931471805459295,
                           0.9999999999595484};
  double f[N];
  uint32_t n[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const double big = fma(d[i], kLog2e, kBig);
    f[i] = fma(d[i], kLog2e, kBig - big);
    n[i] = __builtin_bit_cast(u32x2, big)[0];
    d[i] = 1.531008115307486e-05;
  }
#pragma unroll
  for (int k = 0; k < 7; ++k)
#pragma unroll
    for (int i = 0; i < N; ++i) d[i] = fma(d[i], f[i], kC[k]);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    u32x2 b = __builtin_bit_cast(u32x2, d[i]);
    b[1] += n[i] << 20;
    d[i] = __builtin_bit_cast(double, b);
  }
}
// a - b for a <= b, as exp_of takes it (e^-690 counts for nothing; -inf as it).
__device__ __forceinline__ double below(float a, float b) {
  return a == kNone ? -690.0 : fmax((double)a - (double)b, -690.0);
}

// An element: its value and its place k 2^24 + v; the better one has the larger
// value, or the lower place.
struct Element {
  float v;
  uint32_t at;
};

// x of the lane o away (o = 1, 2, 16, 32) or of one of the other half of 2 o
// lanes (o = 4, 8), for values that all lanes of a half share.
template <int O>
__device__ __forceinline__ uint32_t other_half(uint32_t x) {
  if constexpr (O == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    return (threadIdx.x & 16) ? r[0] : r[1];
  } else if constexpr (O == 32) {
    const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return (threadIdx.x & 32) ? r[0] : r[1];
  } else {
    // quad_perm [1, 0, 3, 2], [2, 3, 0, 1], row_half_mirror, row_mirror
    constexpr int kCtrl = O == 1 ? 0xB1 : O == 2 ? 0x4E : O == 4 ? 0x141 : 0x140;
    return (uint32_t)__builtin_amdgcn_update_dpp((int)x, (int)x, kCtrl, 0xF, 0xF, false);
  }
}
template <int O>
__device__ __forceinline__ float other_half(float x) {
  return __uint_as_float(other_half<O>(__float_as_uint(x)));
}
template <int O>
__device__ __forceinline__ double other_half(double x) {
  const uint64_t b = __builtin_bit_cast(uint64_t, x);
  return __builtin_bit_cast(double, (uint64_t)other_half<O>((uint32_t)(b >> 32)) << 32 |
                                        other_half<O>((uint32_t)b));
}
template <class V, class Op>
__device__ __forceinline__ V wave_all(V x, Op op) {
  x = op(x, other_half<1>(x));
  x = op(x, other_half<2>(x));
  x = op(x, other_half<4>(x));
  x = op(x, other_half<8>(x));
  x = op(x, other_half<16>(x));
  return op(x, other_half<32>(x));
}
struct Max {
  __device__ float operator()(float a, float b) const { return fmaxf(a, b); }
};
struct Sum {
  __device__ double operator()(double a, double b) const { return a + b; }
};

// Numbers whose order is that of the values (0 and -0 the same).
__device__ __forceinline__ uint32_t ordered(float v) {
  const uint32_t b = __float_as_uint(v + 0.f);
  return b ^ ((uint32_t)((int)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ uint64_t ordered(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v + 0.0);
  return b ^ ((uint64_t)((int64_t)b >> 63) | 0x8000000000000000ull);
}
__device__ __forceinline__ float value_of(uint32_t k) {
  return __uint_as_float(k ^ (k >> 31 ? 0x80000000u : ~0u));
}
__device__ __forceinline__ double value_of(uint64_t k) {
  return __builtin_bit_cast(double, k ^ (k >> 63 ? 0x8000000000000000ull : ~0ull));
}

// Of a wave: a number that q lanes' x are not below, the largest but for its last 16
// bits, and -inf where there are no such lanes; the same of r lanes' y.  (A bit a
// step, by counting lanes.)
__device__ __forceinline__ float2 wave_nth(float x, int q, float y, int r) {
  const uint32_t k = ordered(x), l = ordered(y);
  uint32_t t = 0, u = 0;
#pragma unroll
  for (uint32_t bit = 1u << 31; bit >= 1u << 16; bit >>= 1) {
    if (__builtin_popcountll(__builtin_amdgcn_ballot_w64(k >= (t | bit))) >= q) t |= bit;
    if (__builtin_popcountll(__builtin_amdgcn_ballot_w64(l >= (u | bit))) >= r) u |= bit;
  }
  return float2{t > ordered(kNone) ? value_of(t) : kNone, u > ordered(kNone) ? value_of(u) : kNone};
}
// At most the key of a wave's num-th best, by its lanes' two largest keys; and a key
// of which the waves of a workgroup have num together, at most the smallest of it.
__device__ __forceinline__ float2 waves_least(int num, float mx, float second) {
  const bool one = num <= 64;  // an element a lane will do
  return wave_nth(one ? mx : second, one ? num : (num + 1) / 2, mx,
                  (num + kBmWaves - 1) / kBmWaves);
}
// At most the key of the workgroup's num-th best, and above -inf.
__device__ __forceinline__ float workgroup_least(const float2 (&of)[kBmWaves]) {
  float a = of[0].x, b = of[0].y;
#pragma unroll
  for (int w = 1; w < kBmWaves; ++w) {
    a = fmaxf(a, of[w].x);
    b = fminf(b, of[w].y);
  }
  return fmaxf(fmaxf(a, b), -__FLT_MAX__);
}

// The lane's place among those of a mask.
__device__ __forceinline__ int place_in(uint64_t mask) {
  return (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32),
                                        __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
}

// Keeps the num best of a wave's list of n > num keys (PLACES: of the same ones the
// lowest in `at`), at its front, and returns what the others' keys were below, or the
// num-th key: a bit a step, by counting lanes.  (Values that rise along the row or
// are mostly the same, beams far apart, num above 64.  By comparing all pairs 128
// rows of 151936 values, most of them -65504, took 1970 us, now 50.)
template <int MOST, bool PLACES>
__device__ __forceinline__ uint64_t keep_best(uint64_t* list, uint32_t* at, int n, int num) {
  constexpr int kEach = MOST / 64;
  const int lane = threadIdx.x & 63;
  paged_lds_sync();
  uint64_t key[kEach];
  uint32_t place[kEach];  // (its complement)
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    key[i] = i * 64 + lane < n ? list[i * 64 + lane] : 0;
    if constexpr (PLACES) place[i] = i * 64 + lane < n ? ~at[i * 64 + lane] : 0;
  }
  uint64_t t = 0;
  int count = n;  // not below t
#pragma unroll 1
  for (uint64_t bit = 1ull << 63; bit && count > num; bit >>= 1) {
    int above = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i)
      above += __builtin_popcountll(__builtin_amdgcn_ballot_w64(key[i] >= (t | bit)));
    if (above >= num) {
      t |= bit;
      count = above;
    }
  }
  uint32_t u = 0;  // of the keys that are t
  if constexpr (PLACES) {
#pragma unroll 1
    for (uint32_t bit = 1u << 31; bit && count > num; bit >>= 1) {
      int above = 0;
#pragma unroll
      for (int i = 0; i < kEach; ++i)
        above += __builtin_popcountll(__builtin_amdgcn_ballot_w64(
            (key[i] > t) | ((key[i] == t) & (place[i] >= (u | bit)))));
      if (above >= num) {
        u |= bit;
        count = above;
      }
    }
  }
  int kept = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    bool in = key[i] >= t;
    if constexpr (PLACES) in = (key[i] > t) | ((key[i] == t) & (place[i] >= u));
    const uint64_t mask = __builtin_amdgcn_ballot_w64(in);
    if (in) {
      list[kept + place_in(mask)] = key[i];
      if constexpr (PLACES) at[kept + place_in(mask)] = ~place[i];
    }
    kept += __builtin_popcountll(mask);
  }
  paged_lds_sync();
  return t;
}

// Ranks the waves' lists (n[w] keys, behind them four zeros) as one: put(rank, w,
// i) for each element, by one thread.  Four lanes have an element, and each looks
// at one list.  ties(w, i, list, length): what else is better, of keys that are
// the same.
template <int MOST, class Ties, class Put>
__device__ __forceinline__ void rank_lists(const uint64_t (&key)[kBmWaves][MOST],
                                           const int (&n)[kBmWaves], int all, Ties ties, Put put) {
  const int tid = threadIdx.x, of = tid & 3;
  const int len = of == 0 ? n[0] : of == 1 ? n[1] : of == 2 ? n[2] : n[3];
  const uint64_t* list = key[of];
  for (int i0 = 0; i0 < all; i0 += kBmThreads / 4) {  // uniform
    const int i = min(i0 + tid / 4, all - 1);
    int at = i, w = 0;
#pragma unroll
    for (int u = 0, before = 0; u < kBmWaves - 1; ++u) {
      before += n[u];
      if (i >= before) {
        at = i - before;
        w = u + 1;
      }
    }
    const uint64_t mine = key[w][at];
    int rank = 0, same = 0;
    for (int j = 0; j < len; j += 4) {
      uint64_t o[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) o[k] = list[j + k];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        rank += o[k] > mine;
        same += o[k] == mine;
      }
    }
    rank += ties(w, at, of, len, same);
    rank += (int)other_half<1>((uint32_t)rank);
    rank += (int)other_half<2>((uint32_t)rank);
    if (of == 0 && i == i0 + tid / 4) put(rank, w, at);
  }
}

// The last stage's elements in LDS: numbers in the order of their values, and
// their places.
struct LastLds {
  static constexpr int kMost = 320;
  uint64_t key[kBmWaves][kMost + 4];
  uint32_t at[kBmWaves][kMost + 4];
  float2 least[kBmWaves];
  int count[kBmWaves];
};

// The num best of the workgroup's elements above -inf, each passed with its rank
// to `put` by one thread; returns how many there are (num at most).  each(add)
// calls add(value, place, whether the list may be full) for all elements that matter,
// a wave at a time; it returns whether the wave has taken any, and where it has not
// there is no need to call it with lower ones.  `mx`: the largest key of some of a
// thread's elements, key(v) a float that never falls where v grows, and above -inf
// where v is.
//
// What is not below the num-th of the lanes' best (of a wave, or a quarter of them
// in each), not many more elements than num of random ones, is collected in LDS, a
// list a wave, and ranked by counting.  A list that is full keeps its num best.
template <class Each, class Key, class Put>
__device__ __forceinline__ int top_n(int num, LastLds& s, float mx, Each each, Key key, Put put) {
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const float2 least_of = waves_least(num, mx, kNone);
  if (lane == 0) s.least[wave] = least_of;
  __syncthreads();
  const float least = workgroup_least(s.least);
  uint64_t low = 0;
  int mine = 0;  // uniform
  auto add = [&](double v, uint32_t at, bool may_fill) {
    const bool in = (key(v) >= least) & (ordered(v) >= low);
    const uint64_t mask = __builtin_amdgcn_ballot_w64(in);
    if (!mask) return false;
    if (may_fill && __builtin_expect(mine > s.kMost - 64, 0)) {
      low = keep_best<LastLds::kMost, true>(s.key[wave], s.at[wave], mine, num);
      mine = num;
    }
    if (in) {
      const int i = mine + place_in(mask);
      s.key[wave][i] = ordered(v);
      s.at[wave][i] = at;
    }
    mine += __builtin_popcountll(mask);
    return true;
  };
  each(add);
  if (__builtin_expect(mine > max(num, 64), 0)) {
    keep_best<LastLds::kMost, true>(s.key[wave], s.at[wave], mine, num);
    mine = num;
  }
  if (lane < 4) s.key[wave][mine + lane] = 0;
  if (lane == 0) s.count[wave] = mine;
  __syncthreads();
  int n[kBmWaves], all = 0;
#pragma unroll
  for (int w = 0; w < kBmWaves; ++w) {
    n[w] = __builtin_amdgcn_readfirstlane(s.count[w]);
    all += n[w];
  }
  rank_lists(
      s.key, n, all,
      [&](int w, int i, int of, int len, int same) {
        int better = 0;
        same += (int)other_half<1>((uint32_t)same);
        same += (int)other_half<2>((uint32_t)same);
        if (__builtin_amdgcn_ballot_w64(same > 1))  // equal values: by place
          for (int j = 0; j < len; j += 4)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              better += (s.key[of][j + k] == s.key[w][i]) & (s.at[of][j + k] < s.at[w][i]);
        return better;
      },
      [&](int rank, int w, int i) {
        if (rank < num) put(rank, value_of(s.key[w][i]), s.at[w][i]);
      });
  return min(all, num);
}

__device__ __forceinline__ float to_float(__half x) { return (float)(_Float16)x; }
__device__ __forceinline__ float to_float(__hip_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(float x) { return x; }

struct BeamArgs {
  const void* logits;  // rows of `stride` values
  int64_t stride;
  const float* scores;
  int K, V, num, parts, part;  // parts of a row, their length
  double* sums;            // [row][part]: of e^(x - shift)
  uint64_t* best;          // [prompt][num][beam][part]; behind them [row][part]: the sums' shifts
  unsigned* count;         // [row] and [prompt], kBmCounter apart, zero between calls
  float* out_scores;
  int64_t *out_parents, *out_tokens;
};

__device__ __forceinline__ uint64_t pack(float v, uint32_t at) {
  return (uint64_t)at << 32 | __float_as_uint(v);
}
__device__ __forceinline__ Element unpack(uint64_t x) {
  return Element{__uint_as_float((uint32_t)x), (uint32_t)(x >> 32)};
}

// The last workgroup of a prompt to arrive: its beams' normalizers, then the best
// of its parts' best.
template <int R>
__device__ void beam_last(const BeamArgs& a, int b, LastLds& top) {
  __shared__ double lse[kBmBeams];  // NaN: so are all of the beam's
  __shared__ float score[kBmBeams];
  __shared__ uint32_t taken[kBmMost];
  __shared__ int rows[kBmBeams], free_of[kBmWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t row0 = (int64_t)b * a.K;
  const uint64_t* best = a.best + row0 * a.parts * a.num;
  const int total = a.K * a.parts * a.num;
  uint64_t mine[R];  // the first of the elements, the others are read when they are needed
#pragma unroll
  for (int i = 0; i < R; ++i)
    mine[i] = handoff_get(best + min(tid + i * kBmThreads, total - 1));
  // two beams a wave at once, two parts a lane (the first 128 parts; others are
  // read twice)
  const uint64_t* max_of = a.best + (int64_t)gridDim.y * a.parts * a.num + row0 * a.parts;
  const double* sum_of = a.sums + row0 * a.parts;
  for (int k0 = wave; k0 < a.K; k0 += 2 * kBmWaves) {
    const int k[2] = {k0, min(k0 + kBmWaves, a.K - 1)};
    float was[2], m[2], pm[2][2];
    double ps[2][2], s[2] = {0.0, 0.0};
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      was[r] = a.scores[row0 + k[r]];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int i = lane + 64 * e, at = k[r] * a.parts + min(i, a.parts - 1);
        pm[r][e] = unpack(handoff_get(max_of + at)).v;
        ps[r][e] = handoff_get(sum_of + at);
        if (i >= a.parts) {
          pm[r][e] = kNone;
          ps[r][e] = 0.0;
        }
      }
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      m[r] = fmaxf(pm[r][0], pm[r][1]);
      for (int i = lane + 128; i < a.parts; i += 64)
        m[r] = fmaxf(m[r], unpack(handoff_get(max_of + k[r] * a.parts + i)).v);
      m[r] = wave_all(m[r], Max());
    }
    // (a sum that is NaN stays: 0 times it is)
    double d[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) d[i] = below(pm[i >> 1][i & 1], m[i >> 1]);
    exp_of(d);
#pragma unroll
    for (int r = 0; r < 2; ++r) {
#pragma unroll
      for (int e = 0; e < 2; ++e) s[r] += ps[r][e] * d[2 * r + e];
      for (int i = lane + 128; i < a.parts; i += 64) {
        const int at = k[r] * a.parts + i;
        double f[1] = {below(unpack(handoff_get(max_of + at)).v, m[r])};
        exp_of(f);
        s[r] += handoff_get(sum_of + at) * f[0];
      }
      s[r] = wave_all(s[r], Sum());
    }
    // (a beam of nothing but -inf has no element that is passed to top_n)
    const double sum = lane == 0 ? s[0] : s[1];
    const float all = lane == 0 ? m[0] : m[1], w = lane == 0 ? was[0] : was[1];
    const bool nan = sum != sum || all == __builtin_inff() || w != w || w == __builtin_inff();
    if (lane < 2) {
      lse[lane ? k[1] : k[0]] = nan ? __builtin_nan("") : all == kNone ? 0.0 : (double)all + log(sum);
      score[lane ? k[1] : k[0]] = w;
    }
  }
  __syncthreads();
  const double lk = lse[min(lane, a.K - 1)];
  const uint64_t of_nan = __builtin_amdgcn_ballot_w64(lane < a.K && lk != lk);
  double c[R];
  float mx = kNone;
  auto value = [&](Element e) {
    const int k = e.at >> kBmVocab;
    return (double)score[k] + ((double)e.v - lse[k]);
  };
  auto key = [](double v) {  // (-inf and NaN: none)
    return v > (double)kNone ? fmaxf((float)v, -__FLT_MAX__) : kNone;
  };
#pragma unroll
  for (int i = 0; i < R; ++i) {
    c[i] = tid + i * kBmThreads < total ? value(unpack(mine[i])) : (double)kNone;
    mx = fmaxf(mx, key(c[i]));
  }
  const int64_t out = (int64_t)b * a.num;
  auto put = [&](int r, double v, int k, int token) {
    a.out_scores[out + r] = (float)v;
    a.out_parents[out + r] = k;
    a.out_tokens[out + r] = token;
  };
  // the beams of NaN, then the others
  const int n_nan = __builtin_popcountll(of_nan);
  if (tid < a.K) {
    const uint64_t before = of_nan & ((1ull << tid) - 1);
    const int nans = __builtin_popcountll(before);
    rows[of_nan >> tid & 1 ? nans : n_nan + tid - nans] = tid;
  }
  // NaN counts as the largest, as where values are sorted
  const int first = (int)min((int64_t)a.num, (int64_t)n_nan * a.V);
  if (first > 0) {  // uniform
    __syncthreads();
    if (tid < first) put(tid, __builtin_nan(""), rows[tid / a.V], tid % a.V);
  }
  const int num = a.num - first;
  if (num == 0) return;  // uniform
  const int found = top_n(
      num, top, mx,
      [&](auto add) {
#pragma unroll
        for (int i = 0; i < R; ++i) add(c[i], (uint32_t)(mine[i] >> 32), R * 64 > LastLds::kMost);
        // the others: 64 parts a wave (all lanes, for its ballots), their first ones,
        // their second ones, until none is taken: a part's are in order
        const int of_all = a.K * a.parts, r0 = R * kBmThreads / of_all;
        if (r0 < a.num)
          for (int p0 = wave * 64; p0 < of_all; p0 += kBmThreads) {
            const int p = min(p0 + lane, of_all - 1);
            uint64_t next = handoff_get(best + r0 * of_all + p);
            for (int r = r0; r < a.num; ++r) {
              const Element e = unpack(next);
              next = handoff_get(best + min(r + 1, a.num - 1) * of_all + p);
              const bool other = p0 + lane < of_all && r * of_all + p >= R * kBmThreads;
              if (!add(other ? value(e) : (double)kNone, e.at, true) && r > r0) break;  // uniform
            }
          }
      },
      key,
      [&](int rank, double v, uint32_t at) {
        put(first + rank, v, at >> kBmVocab, at & ((1 << kBmVocab) - 1));
        taken[rank] = at;
      });
  if (found == num) return;  // uniform
  // The rest are -inf: the lowest places of the other beams that are not among
  // the found ones, which are all there are above -inf.
  __syncthreads();
  const int k = n_nan + tid / a.V;
  const bool there = tid < 2 * kBmMost && k < a.K;
  const uint32_t at = there ? (uint32_t)rows[k] << kBmVocab | tid % a.V : 0u;
  bool is_free = there;
  for (int i = 0; i < found; ++i) is_free = is_free && taken[i] != at;
  const uint64_t mask = __builtin_amdgcn_ballot_w64(is_free);
  if (lane == 0) free_of[wave] = __builtin_popcountll(mask);
  __syncthreads();
  int r = found + __builtin_popcountll(mask & ((1ull << lane) - 1));
  for (int w = 0; w < wave; ++w) r += free_of[w];
  if (is_free && r < num) put(first + r, (double)kNone, at >> kBmVocab, tid % a.V);
}

static_assert(2 * kBmMost <= kBmThreads, "as many places as may be taken and needed");

// A part's elements in LDS: 64-bit numbers that are larger for the better one,
// the value's order above its place's.
struct PartLds {
  static constexpr int kChunk = 64 * kBmEach, kMost = 768;  // of a wave: a chunk's, all
  uint64_t key[kBmWaves][kMost + 4];
  float2 least[kBmWaves];
  int count[kBmWaves];
};

// The smallest number above x.
__device__ __forceinline__ float next_up(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return __uint_as_float((int)b < 0 ? b - 1 : b + 1);
}

// One workgroup a part of a row, in chunks of 2048 values that pass through
// registers, so that memory is read once: the sum of its exponentials, and its
// best.  The last workgroup of a prompt to arrive goes on with all of its parts'.
//
// Many rows are bound by instructions: 30 vector ones a value, 15 of them fp64,
// and the cut's scalar ones: 128 rows of 151936 fp16 values 31 us (1.2 TB/s; a
// copy's rate would be 8).  Few rows are bound by the way of one part (5 us) and
// of a prompt's last workgroup (5 us): 4 rows 12.3 us with the launch.
//
// A thread sums its exponentials over the first value that it saw (or a later one
// 600 above it: fp64 has the room).  A wave collects what is not below the num-th
// of its lanes' best so far; once there are num of them, equal values of later
// chunks, whose places are higher, are none of the best.
// (TINY: rows shorter than a load.)
template <class T, bool TINY>
__global__ __launch_bounds__(kBmThreads) void beam_kernel(BeamArgs a) {
  constexpr int W = 16 / sizeof(T), NV = kBmEach / W;  // values of a load, loads of a chunk
  constexpr int kChunk = kBmThreads * kBmEach;
  __shared__ union Lds {
    PartLds part;
    LastLds last;
    __device__ Lds() {}
  } top;
  __shared__ double sums[kBmWaves];
  __shared__ float maxs[kBmWaves];
  __shared__ int flag;
  PartLds& s = top.part;
  const int tid = threadIdx.x, lane = tid & 63, row = blockIdx.y;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int b = row / a.K, k = row - b * a.K, num = a.num;
  const T* p = (const T*)a.logits + row * a.stride;
  const int lo = blockIdx.x * a.part, hi = min(lo + a.part, a.V);
  const int chunks = max((hi - lo + kChunk - 1) / kChunk, 1);

  // Value i of a chunk's load j: (first, or the last W of the row where those end
  // before: every load is a whole one, and what another thread has is left out).
  // Rows of odd widths begin anywhere: unaligned loads.
  auto first = [&](int c, int j) { return lo + ((c * NV + j) * kBmThreads + tid) * W; };
  auto from = [&](int c, int j) { return min(first(c, j), max(hi - W, 0)); };
  auto load = [&](T (&v)[kBmEach], int c) {
    if constexpr (TINY) {
#pragma unroll
      for (int e = 0; e < kBmEach; ++e) v[e] = p[min(e, a.V - 1)];
    } else {
#pragma unroll
      for (int j = 0; j < NV; ++j) __builtin_memcpy(v + j * W, p + from(c, j), 16);
    }
  };
  float x[kBmEach], mx, top1 = kNone, top2 = kNone, ref = kNone;
  double sum = 0;
  bool nan = false;
  auto take = [&](const T (&v)[kBmEach], int c) {
    if (lo + (c + 1) * kChunk <= hi) {  // uniform
#pragma unroll
      for (int e = 0; e < kBmEach; ++e) x[e] = to_float(v[e]);
    } else {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int skip = first(c, j) - from(c, j), end = hi - from(c, j);
#pragma unroll
        for (int e = 0; e < W; ++e)
          x[j * W + e] = e >= skip && e < end ? to_float(v[j * W + e]) : kNone;
      }
    }
    mx = x[0];
#pragma unroll
    for (int e = 1; e < kBmEach; ++e) mx = fmaxf(mx, x[e]);
#pragma unroll
    for (int e = 0; e < kBmEach; ++e) nan |= x[e] != x[e];
    if (num > 64) {  // uniform
#pragma unroll
      for (int e = 0; e < kBmEach; ++e) {
        top2 = fmaxf(top2, fminf(top1, x[e]));
        top1 = fmaxf(top1, x[e]);
      }
    } else {
      top1 = fmaxf(top1, mx);
    }
    // (by the difference, which fp32 has exactly where the two are near: ref + 600
    // may round to ref + 1024; over -inf any value is, and inf - inf, NaN, is not)
    const bool shift = mx - ref > 600.f;
    if (__builtin_amdgcn_ballot_w64(shift)) {
      const float to = shift ? mx : ref;
      double d[1] = {below(ref, to)};
      exp_of(d);
      sum = shift ? sum * d[0] : sum;
      ref = to;
    }
    const double m = ref;
#pragma unroll
    for (int e = 0; e < kBmEach; e += 4) {
      double d[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) d[i] = fmax((double)x[e + i] - m, -690.0);
      exp_of(d);
      sum += (d[0] + d[1]) + (d[2] + d[3]);
    }
  };
  float cut = -__FLT_MAX__;  // what is below is none of the best
  int mine = 0;              // keys of the wave's list
  auto collect = [&](int c) {
    if (__builtin_expect(mine > s.kMost - s.kChunk, 0)) {
      const uint64_t least = keep_best<PartLds::kMost, false>(s.key[wave], nullptr, mine, num);
      cut = fmaxf(cut, next_up(value_of((uint32_t)(least >> 32))));
      mine = num;
    }
#pragma unroll
    for (int e = 0; e < kBmEach; ++e) {
      const bool in = x[e] >= cut;
      const uint64_t mask = __builtin_amdgcn_ballot_w64(in);
      if (mask) {
        if (in)
          s.key[wave][mine + place_in(mask)] =
              (uint64_t)ordered(x[e]) << 32 |
              ~((uint32_t)k << kBmVocab | (from(c, e / W) + e % W));
        mine += __builtin_popcountll(mask);
      }
    }
  };
  auto middle = [&](const T (&v)[kBmEach], int c) {
    take(v, c);
    const int hits = __builtin_popcountll(__builtin_amdgcn_ballot_w64(mx >= cut));
    if (hits == 0) return;  // uniform
    float least = kNone;
    if (2 * hits > num) {
      least = waves_least(num, top1, top2).x;
      cut = fmaxf(cut, least);
    }
    collect(c);
    if (least > kNone) cut = fmaxf(cut, next_up(least));
  };
  T v0[kBmEach], v1[kBmEach];
  load(v0, 0);
  int c = 0;
  for (; c + 2 < chunks; c += 2) {
    load(v1, c + 1);
    middle(v0, c);
    load(v0, c + 2);
    middle(v1, c + 1);
  }
  if (c + 1 < chunks) {
    load(v1, c + 1);
    middle(v0, c);
    take(v1, ++c);
  } else {
    take(v0, c);
  }
  // the last chunk's best by those of all waves
  {
    const float2 least = waves_least(num, top1, top2);
    const float all = wave_all(ref, Max());
    double d[1] = {below(ref, all)};
    exp_of(d);
    sum = ref == kNone ? 0.0 : sum * d[0];
    if (nan) sum = __builtin_nan("");
    sum = wave_all(sum, Sum());
    if (lane == 0) {
      s.least[wave] = least;
      sums[wave] = sum;
      maxs[wave] = all;
    }
  }
  __syncthreads();
  {
    const float least = workgroup_least(s.least);
    const uint64_t low = (uint64_t)ordered(least) << 32;
    if (mine) {  // what is left of the others'
      paged_lds_sync();
      int kept = 0;
      for (int i = 0; i < mine; i += 64) {
        const uint64_t key = i + lane < mine ? s.key[wave][i + lane] : 0;
        const uint64_t mask = __builtin_amdgcn_ballot_w64(key >= low);
        paged_lds_sync();
        if (key >= low) s.key[wave][kept + place_in(mask)] = key;
        kept += __builtin_popcountll(mask);
      }
      mine = kept;
    }
    cut = fmaxf(cut, least);
    collect(c);
    if (__builtin_expect(mine > max(num, 64), 0)) {
      keep_best<PartLds::kMost, false>(s.key[wave], nullptr, mine, num);
      mine = num;
    }
    if (lane < 4) s.key[wave][mine + lane] = 0;
    if (lane == 0) s.count[wave] = mine;
  }
  __syncthreads();
  int n[kBmWaves], all = 0;
#pragma unroll
  for (int w = 0; w < kBmWaves; ++w) {
    n[w] = __builtin_amdgcn_readfirstlane(s.count[w]);
    all += n[w];
  }
  // (the parts' first ones side by side, then their second ones: the last stage's
  // first lanes have what it looks for)
  const int64_t part = (int64_t)row * a.parts + blockIdx.x;
  const int of_all = a.K * a.parts;
  uint64_t* best = a.best + (int64_t)b * of_all * num + (k * a.parts + blockIdx.x);
  rank_lists(
      s.key, n, all, [](int, int, int, int, int) { return 0; },  // (no two are the same)
      [&](int rank, int w, int i) {
        const uint64_t key = s.key[w][i];
        if (rank < num)
          handoff_put(best + rank * of_all, pack(value_of((uint32_t)(key >> 32)), ~(uint32_t)key));
      });
  if (tid >= all && tid < num)
    handoff_put(best + tid * of_all, pack(kNone, (uint32_t)k << kBmVocab));
  if (wave == 0) {  // the waves' sums, one a lane of four
    const float mine = maxs[lane % kBmWaves];
    float m = fmaxf(mine, other_half<1>(mine));
    m = fmaxf(m, other_half<2>(m));
    double d[1] = {below(mine, m)};
    exp_of(d);
    sum = sums[lane % kBmWaves] * d[0];  // (NaN stays)
    sum += other_half<1>(sum);
    sum += other_half<2>(sum);
    if (lane == 0) {
      handoff_put(a.sums + part, sum);
      handoff_put(a.best + (int64_t)gridDim.y * a.parts * num + part, pack(m, 0));
    }
  }
  // the last of a prompt; of many parts the last of a row, then the last row
  unsigned* of_row = a.count + (int64_t)row * kBmCounter;
  unsigned* of_prompt = a.count + ((int64_t)gridDim.y + b) * kBmCounter;
  const bool by_row = of_all > kBmAtOnce;
  if (by_row) {
    if (!handoff_arrive(of_row, (unsigned)a.parts, &flag)) return;
    if (tid == 0) handoff_reset(of_row);
  }
  if (!handoff_arrive(of_prompt, (unsigned)(by_row ? a.K : of_all), &flag)) return;
  beam_last<4>(a, b, top.last);
  if (tid == 0) handoff_reset(of_prompt);
}

constexpr int64_t kBmFew = 256, kBmMany = 1024;

// Parts of a row and their length, in chunks: so many workgroups as the card holds
// at once, but two chunks each where a CU would get a second workgroup.  4 rows of
// 151936 values: 11.6 us in parts of two chunks, 13.3 of one; 128 rows 34 us in 8
// parts each, 36 in 7, 10 or 15 (both of one build, before the last ones).
void beam_parts(int64_t rows, int64_t vocab, int64_t& parts, int64_t& part) {
  const int64_t chunk = kBmThreads * kBmEach, chunks = (vocab + chunk - 1) / chunk;
  const int64_t all = std::max<int64_t>(rows, 1) * chunks;
  const int64_t each = std::max<int64_t>((all + kBmMany - 1) / kBmMany, all > kBmFew ? 2 : 1);
  parts = (chunks + each - 1) / each;
  part = align_up((vocab + parts - 1) / parts, 8);
}

}  // namespace
}  // namespace glq

extern "C" int64_t glq_beam_select_counter_bytes(int64_t prompts, int64_t beams) {
  return prompts < 0 || prompts > (1 << 20) || beams <= 0 || beams > glq::kBmBeams
             ? -1
             : prompts * (beams + 1) * glq::kBmCounter * 4;
}

extern "C" int64_t glq_beam_select_scratch_bytes(int64_t prompts, int64_t beams, int64_t vocab,
                                                 int64_t num) {
  using namespace glq;
  if (prompts < 0 || beams <= 0 || vocab <= 0 || num <= 0 || prompts > (1 << 20) ||
      beams > kBmBeams || vocab > (1 << kBmVocab) || num > kBmMost)
    return -1;
  int64_t parts, part;
  beam_parts(prompts * beams, vocab, parts, part);
  return align_up(prompts * beams * parts * (num + 2) * 8, 256);
}

extern "C" int glq_beam_select(const glq_beam_select_params* p, void* stream) {
  using namespace glq;
  clear_error();
  GLQ_CHECK(p != nullptr, "null params");
  const int64_t B = p->prompts, K = p->beams, V = p->vocab, N = p->num;
  GLQ_CHECK(B >= 0 && B <= (1 << 20), "prompts must be in [0, 2^20]");
  GLQ_CHECK(B * K <= 65535, "prompts * beams must be at most 65535");
  GLQ_CHECK(K > 0 && K <= kBmBeams, "beams must be in [1, %d] (got %lld)", kBmBeams, (long long)K);
  GLQ_CHECK(V > 0 && V <= (1 << kBmVocab), "vocab must be in [1, 2^24] (got %lld)", (long long)V);
  GLQ_CHECK(N > 0 && N <= kBmMost && N <= K * V, "num must be in [1, %d] and at most beams * vocab "
            "(got %lld)", kBmMost, (long long)N);
  GLQ_CHECK(p->dtype >= 0 && p->dtype <= 2, "dtype must be 0 (fp16), 1 (bf16) or 2 (fp32)");
  GLQ_CHECK(p->row_stride >= V, "row_stride must be >= vocab");
  if (B == 0) return GLQ_OK;
  GLQ_CHECK(p->logits && p->scores && p->out_scores && p->out_parents && p->out_tokens,
            "null pointer argument");
  const int size = p->dtype == 2 ? 4 : 2;
  GLQ_CHECK(((uintptr_t)p->logits & (size - 1)) == 0 && ((uintptr_t)p->scores & 3) == 0 &&
                ((uintptr_t)p->out_scores & 3) == 0 && ((uintptr_t)p->out_parents & 7) == 0 &&
                ((uintptr_t)p->out_tokens & 7) == 0,
            "pointers must be aligned to their type");
  // (a prompt's results are written while others are still read)
  const int64_t in_bytes = ((B * K - 1) * p->row_stride + V) * size;
  const void* const out[3] = {p->out_scores, p->out_parents, p->out_tokens};
  for (int i = 0; i < 3; ++i)
    GLQ_CHECK(apart(p->scores, B * K * 4, out[i], B * N * (i ? 8 : 4)) &&
                  apart(p->logits, in_bytes, out[i], B * N * (i ? 8 : 4)),
              "outputs must not overlap scores or logits");
  const int64_t cnt = glq_beam_select_counter_bytes(B, K);
  const int64_t scr = glq_beam_select_scratch_bytes(B, K, V, N);
  GLQ_CHECK(p->counters && p->counter_bytes >= cnt && p->scratch && p->scratch_bytes >= scr &&
                ((uintptr_t)p->counters & 3) == 0 && ((uintptr_t)p->scratch & 15) == 0,
            "workspace of %lld (counters) and %lld bytes (scratch, 16-byte aligned) needed "
            "(got %lld, %lld)", (long long)cnt, (long long)scr, (long long)p->counter_bytes,
            (long long)p->scratch_bytes);
  BeamArgs a{};
  a.logits = p->logits;
  a.stride = p->row_stride;
  a.scores = p->scores;
  a.K = (int)K; a.V = (int)V; a.num = (int)N;
  int64_t parts, part;
  beam_parts(B * K, V, parts, part);
  a.parts = (int)parts; a.part = (int)part;
  a.sums = (double*)p->scratch;
  a.best = (uint64_t*)(a.sums + B * K * parts);
  a.count = (unsigned*)p->counters;
  a.out_scores = p->out_scores;
  a.out_parents = p->out_parents;
  a.out_tokens = p->out_tokens;
  auto kern = V * size < 16 ? (p->dtype == 0   ? beam_kernel<__half, true>
                               : p->dtype == 1 ? beam_kernel<__hip_bfloat16, true>
                                               : beam_kernel<float, true>)
                            : (p->dtype == 0   ? beam_kernel<__half, false>
                               : p->dtype == 1 ? beam_kernel<__hip_bfloat16, false>
                                               : beam_kernel<float, false>);
  kern<<<dim3((unsigned)parts, (unsigned)(B * K)), dim3(kBmThreads), 0, (hipStream_t)stream>>>(a);
  GLQ_LAUNCH_CHECK("beam_kernel");
  return GLQ_OK;
}
