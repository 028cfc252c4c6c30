// The best continuations of each prompt over its beams and the vocabulary:
//   c[k][v] = score[k] + logits[k][v] - log sum_u exp(logits[k][u])
// the `num` largest, the lowest k vocab + v first among equal ones.

#include <hip/hip_bf16.h>

#include "glq_paged.h"

namespace glq {
namespace {

constexpr int kBmThreads = 256;
constexpr int kBmLastThreads = 512;
constexpr int kBmMost = 128;   // continuations of a prompt
constexpr int kBmBeams = 64;
constexpr int kBmList = 1024;  // elements that top_n ranks at once

// e^d for d <= 0, in fp64 and to 6e-11: 2^(n + f) with 2^f by its Chebyshev
// series of degree 7 on [-1/2, 1/2].  Two continuations of different beams
// compare by sums over the vocabulary, so fp32 (1e-7) would put some in the
// wrong order; the vector fp64 rate is that of unpacked fp32.
__device__ __forceinline__ double exp_neg(double d) {
  const double t = fmax(d, -700.0) * 1.4426950408889634;
  const double n = __builtin_rint(t), f = t - n;
  double y = 1.531008115307486e-05;
  y = fma(y, f, 0.00015469731972928003);
  y = fma(y, f, 0.0013333450559898097);
  y = fma(y, f, 0.009618025602961655);
  y = fma(y, f, 0.05550410941217088);
  y = fma(y, f, 0.240226512135953);
  y = fma(y, f, 0.6931471805459295);
  y = fma(y, f, 0.9999999999595484);
  return __builtin_ldexp(y, (int)n);
}

constexpr float kNone = -__builtin_inff();

// An element: its value and its place; the better one has the larger value, or
// the lower place.
template <class V>
struct Element {
  V v;
  uint32_t at;
  __device__ bool over(const Element& b) const { return v > b.v || (v == b.v && at < b.at); }
};

template <class V>
__device__ __forceinline__ Element<V> shfl_xor(Element<V> e, int o) {
  return Element<V>{__shfl_xor(e.v, o), (uint32_t)__shfl_xor((int)e.at, o)};
}

template <class V, int THREADS>
struct TopLds {
  Element<V> best[kBmMost > THREADS ? kBmMost : THREADS];
  Element<V> list[kBmList];
  int count;
};

// The num best of the workgroup's elements above -inf, each passed with its rank
// to `put` by one thread; returns how many there are (num at most).  each(f)
// calls f(value, place) for every element of a thread, the same ones each time.
//
// The threads are cut into num groups (of lanes side by side in their residues,
// so that no group is without elements before most threads are), and the least
// of the groups' best is at most the num-th best: what is not below it, about
// num log(num) elements of random ones, is collected in LDS and ranked by
// counting.  Where that does not fit (groups that have next to nothing), the
// best are taken one after another.
template <class V, int THREADS, class Each, class Put>
__device__ int top_n(int num, TopLds<V, THREADS>& s, Each each, Put put) {
  using E = Element<V>;
  const int tid = threadIdx.x;
  const E none{(V)kNone, 0xFFFFFFFFu};
  int groups = 1;
  while (groups < num) groups <<= 1;
  E b = none;
  each([&](V v, uint32_t at) {
    const E e{v, at};
    if (v > (V)kNone && e.over(b)) b = e;
  });
  for (int o = 32; o >= groups; o >>= 1) {
    const E e = shfl_xor(b, o);
    if (e.over(b)) b = e;
  }
  __syncthreads();
  if (tid == 0) s.count = 0;
  s.best[tid] = b;
  __syncthreads();
  // (group g: threads g mod groups; of a wave one is enough for each group)
  E least{(V)__builtin_inff(), 0u};
  for (int g = tid & 63; g < groups; g += 64) {
    E m = none;
    for (int t = g; t < THREADS; t += groups < 64 ? 64 : groups)
      if (s.best[t].over(m)) m = s.best[t];
    if (least.over(m)) least = m;
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    const E e = shfl_xor(least, o);
    if (least.over(e)) least = e;
  }
  each([&](V v, uint32_t at) {
    const E e{v, at};
    if (v > (V)kNone && !least.over(e)) {
      const int i = atomicAdd(&s.count, 1);
      if (i < kBmList) s.list[i] = e;
    }
  });
  __syncthreads();
  const int n = s.count;
  if (n <= kBmList) {
    for (int i = tid; i < n; i += THREADS) {
      const E e = s.list[i];
      int rank = 0;
      for (int j = 0; j < n; ++j) rank += s.list[j].over(e);
      if (rank < num) put(rank, e);
    }
    return min(n, num);
  }
  E last{(V)__builtin_inff(), 0u};
  for (int r = 0; r < num; ++r) {  // (more than num of them are there)
    b = none;
    each([&](V v, uint32_t at) {
      const E e{v, at};
      if (v > (V)kNone && e.over(b) && (r == 0 || last.over(e))) b = e;
    });
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
      const E e = shfl_xor(b, o);
      if (e.over(b)) b = e;
    }
    __syncthreads();
    if ((tid & 63) == 0) s.best[tid >> 6] = b;
    __syncthreads();
    last = s.best[0];
    for (int w = 1; w < THREADS / 64; ++w)
      if (s.best[w].over(last)) last = s.best[w];
    if (tid == 0) put(r, last);
  }
  return num;
}

__device__ __forceinline__ float to_float(__half x) { return (float)(_Float16)x; }
__device__ __forceinline__ float to_float(__hip_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(float x) { return x; }

// Of a part of a row: its largest value, the sum of e^(x - it), and its best.
struct Part {
  double sum;
  float max;
  int count;
};

struct BeamArgs {
  const void* logits;  // rows of `stride` values
  int64_t stride;
  const float* scores;
  int K, V, num, parts, part;  // parts of a row, their length
  Part* sums;              // [row][part]
  Element<float>* best;    // [row][part][num], places k V + v
  float* out_scores;
  int64_t *out_parents, *out_tokens;
};

// One workgroup a part of a row, held in registers: a pass over memory.
template <class T, int E>
__global__ __launch_bounds__(kBmThreads) void beam_part_kernel(BeamArgs a) {
  constexpr int W = 16 / sizeof(T), NV = E / W;  // values of a load, loads
  __shared__ TopLds<float, kBmThreads> top;
  __shared__ double sums[kBmThreads / 64];
  const int tid = threadIdx.x, row = blockIdx.y;
  const T* p = (const T*)a.logits + row * a.stride;
  const int lo = blockIdx.x * a.part, hi = min(lo + a.part, a.V);
  // (rows of odd widths begin anywhere: unaligned loads)
  float x[E];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int at = lo + (i * kBmThreads + tid) * W;
    T v[W];
    if (at + W <= hi) {
      __builtin_memcpy(v, p + at, 16);
#pragma unroll
      for (int e = 0; e < W; ++e) x[i * W + e] = to_float(v[e]);
    } else {
#pragma unroll
      for (int e = 0; e < W; ++e) x[i * W + e] = at + e < hi ? to_float(p[at + e]) : kNone;
    }
  }
  float m = kNone;
#pragma unroll
  for (int e = 0; e < E; ++e) m = fmaxf(m, x[e]);
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
  if ((tid & 63) == 0) top.best[tid >> 6].v = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kBmThreads / 64; ++w) m = fmaxf(m, top.best[w].v);
  // (of nothing but -inf: 0; a NaN stays one)
  double sum = 0;
  const double md = m == kNone ? 0.0 : (double)m;
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (x[e] != kNone) sum += x[e] != x[e] ? (double)x[e] : exp_neg((double)x[e] - md);
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) sum += __shfl_xor(sum, o);
  if ((tid & 63) == 0) sums[tid >> 6] = sum;
  const uint32_t at0 = (uint32_t)(row % a.K) * a.V + lo;
  Element<float>* best = a.best + ((int64_t)row * a.parts + blockIdx.x) * a.num;
  const int n = top_n<float, kBmThreads>(
      a.num, top,
      [&](auto f) {
#pragma unroll
        for (int i = 0; i < E; ++i)
          f(x[i], at0 + (uint32_t)((i / W * kBmThreads + tid) * W + i % W));
      },
      [&](int rank, Element<float> e) { best[rank] = e; });
  if (tid == 0) {
    sum = 0;
    for (int w = 0; w < kBmThreads / 64; ++w) sum += sums[w];
    a.sums[(int64_t)row * a.parts + blockIdx.x] = Part{sum, m, n};
  }
}

// One workgroup a prompt: its beams' normalizers, then the best of its parts'.
__global__ __launch_bounds__(kBmLastThreads) void beam_last_kernel(BeamArgs a) {
  __shared__ TopLds<double, kBmLastThreads> top;
  __shared__ double lse[kBmBeams];  // NaN: so are all of the beam's
  __shared__ float score[kBmBeams];
  __shared__ uint32_t taken[kBmMost];
  __shared__ int rows[kBmBeams], n_nan, free_of[kBmLastThreads / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, b = blockIdx.x;
  const Part* sums = a.sums + (int64_t)b * a.K * a.parts;
  for (int k = wave; k < a.K; k += kBmLastThreads / 64) {
    float m = kNone;
    for (int i = lane; i < a.parts; i += 64) m = fmaxf(m, sums[k * a.parts + i].max);
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    double s = 0;
    for (int i = lane; i < a.parts; i += 64) {
      const Part p = sums[k * a.parts + i];
      s += p.sum != p.sum || m == kNone || p.max == kNone
               ? p.sum
               : p.sum * exp_neg((double)p.max - (double)m);
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) s += __shfl_xor(s, o);
    if (lane == 0) {
      const float was = a.scores[b * a.K + k];
      // (a beam of nothing but -inf has no element that is passed to top_n)
      const bool nan = s != s || m == __builtin_inff() || was != was || was == __builtin_inff();
      lse[k] = nan ? __builtin_nan("") : m == kNone ? 0.0 : (double)m + log(s);
      score[k] = was;
    }
  }
  __syncthreads();
  if (tid == 0) {  // the beams of NaN, then the others
    int n = 0;
    for (int k = 0; k < a.K; ++k)
      if (lse[k] != lse[k]) rows[n++] = k;
    n_nan = n;
    for (int k = 0; k < a.K; ++k)
      if (lse[k] == lse[k]) rows[n++] = k;
  }
  __syncthreads();
  const int64_t out = (int64_t)b * a.num;
  auto put = [&](int r, double c, uint32_t at) {
    a.out_scores[out + r] = (float)c;
    a.out_parents[out + r] = at / a.V;
    a.out_tokens[out + r] = at % a.V;
  };
  // NaN counts as the largest, as where values are sorted
  const int first = (int)min((int64_t)a.num, (int64_t)n_nan * a.V);
  if (tid < first)
    put(tid, __builtin_nan(""), (uint32_t)rows[tid / a.V] * a.V + tid % a.V);
  const int num = a.num - first;
  if (num == 0) return;  // uniform
  const Element<float>* best = a.best + (int64_t)b * a.K * a.parts * a.num;
  const int found = top_n<double, kBmLastThreads>(
      num, top,
      [&](auto f) {
        for (int i = tid; i < a.K * a.parts * a.num; i += kBmLastThreads) {
          const int part = i / a.num;
          if (i - part * a.num >= sums[part].count) continue;
          const Element<float> e = best[i];
          const int k = part / a.parts;
          f((double)score[k] + ((double)e.v - lse[k]), e.at);
        }
      },
      [&](int rank, Element<double> e) {
        put(first + rank, e.v, e.at);
        taken[rank] = e.at;
      });
  if (found == num) return;  // uniform
  // The rest are -inf: the lowest places of the other beams that are not among
  // the found ones, which are all there are above -inf.
  __syncthreads();
  uint32_t at = 0xFFFFFFFFu;
  if (tid < 2 * kBmMost && n_nan + tid / a.V < a.K)
    at = (uint32_t)rows[n_nan + tid / a.V] * a.V + tid % a.V;
  bool is_free = at != 0xFFFFFFFFu;
  for (int i = 0; i < found; ++i) is_free = is_free && taken[i] != at;
  const uint64_t mask = __builtin_amdgcn_ballot_w64(is_free);
  if (lane == 0) free_of[wave] = __builtin_popcountll(mask);
  __syncthreads();
  int r = found + __builtin_popcountll(mask & ((1ull << lane) - 1));
  for (int w = 0; w < wave; ++w) r += free_of[w];
  if (is_free && r < num) put(first + r, (double)kNone, at);
}

constexpr int kBmFew = 8, kBmMany = 32;  // values a thread

// Parts of a row and their length.  A row's parts are of up to 8192 values, or
// 2048 where that leaves the card without work.
void beam_parts(int64_t rows, int64_t vocab, int64_t& parts, int64_t& part) {
  const int64_t wide = kBmThreads * kBmMany, narrow = kBmThreads * kBmFew;
  const int64_t most = rows * ((vocab + wide - 1) / wide) < 256 ? narrow : wide;
  parts = (vocab + most - 1) / most;
  part = align_up((vocab + parts - 1) / parts, 8);
}

}  // namespace
}  // namespace glq

extern "C" int64_t glq_beam_select_workspace_bytes(int64_t prompts, int64_t beams, int64_t vocab,
                                                   int64_t num) {
  using namespace glq;
  if (prompts < 0 || beams <= 0 || vocab <= 0 || num <= 0 || prompts > (1 << 20) ||
      beams > kBmBeams || vocab > (1 << 24) || num > kBmMost)
    return -1;
  int64_t parts, part;
  beam_parts(prompts * beams, vocab, parts, part);
  return align_up(prompts * beams * parts * (int64_t)(sizeof(Part) + num * sizeof(Element<float>)),
                  256);
}

extern "C" int glq_beam_select(const glq_beam_select_params* p, void* stream) {
  using namespace glq;
  clear_error();
  GLQ_CHECK(p != nullptr, "null params");
  const int64_t B = p->prompts, K = p->beams, V = p->vocab, N = p->num;
  GLQ_CHECK(B >= 0 && B <= (1 << 20), "prompts must be in [0, 2^20]");
  GLQ_CHECK(B * K <= 65535, "prompts * beams must be at most 65535");
  GLQ_CHECK(K > 0 && K <= kBmBeams, "beams must be in [1, %d] (got %lld)", kBmBeams, (long long)K);
  GLQ_CHECK(V > 0 && V <= (1 << 24), "vocab must be in [1, 2^24] (got %lld)", (long long)V);
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
  GLQ_CHECK(apart(p->scores, B * K * 4, p->out_scores, B * N * 4) &&
                apart(p->scores, B * K * 4, p->out_parents, B * N * 8) &&
                apart(p->scores, B * K * 4, p->out_tokens, B * N * 8),
            "outputs must not overlap scores");
  const int64_t need = glq_beam_select_workspace_bytes(B, K, V, N);
  GLQ_CHECK(p->workspace && p->workspace_bytes >= need && ((uintptr_t)p->workspace & 15) == 0,
            "workspace of %lld bytes, 16-byte aligned, needed (got %lld)", (long long)need,
            (long long)p->workspace_bytes);
  BeamArgs a{};
  a.logits = p->logits;
  a.stride = p->row_stride;
  a.scores = p->scores;
  a.K = (int)K; a.V = (int)V; a.num = (int)N;
  int64_t parts, part;
  beam_parts(B * K, V, parts, part);
  a.parts = (int)parts; a.part = (int)part;
  a.sums = (Part*)p->workspace;
  a.best = (Element<float>*)(a.sums + B * K * parts);
  a.out_scores = p->out_scores;
  a.out_parents = p->out_parents;
  a.out_tokens = p->out_tokens;
  const bool few = part <= kBmThreads * kBmFew;
  auto kern = p->dtype == 0   ? (few ? beam_part_kernel<__half, kBmFew> : beam_part_kernel<__half, kBmMany>)
              : p->dtype == 1 ? (few ? beam_part_kernel<__hip_bfloat16, kBmFew>
                                     : beam_part_kernel<__hip_bfloat16, kBmMany>)
                              : (few ? beam_part_kernel<float, kBmFew> : beam_part_kernel<float, kBmMany>);
  kern<<<dim3((unsigned)parts, (unsigned)(B * K)), dim3(kBmThreads), 0, (hipStream_t)stream>>>(a);
  GLQ_LAUNCH_CHECK("beam_part_kernel");
  beam_last_kernel<<<dim3((unsigned)B), dim3(kBmLastThreads), 0, (hipStream_t)stream>>>(a);
  GLQ_LAUNCH_CHECK("beam_last_kernel");
  return GLQ_OK;
}
