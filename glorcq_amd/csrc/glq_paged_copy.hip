// Copies of pages of a paged key/value cache (layout and formats: glq_paged.h),
// in all layers at once: to pages of the same pools, or to other pools.

#include <cstdlib>

#include "glq_paged.h"

namespace glq {
namespace {

constexpr int kCpThreads = 256;
constexpr int kCpWaves = kCpThreads / 64;
constexpr int kCpPiece = 8192;  // bytes a wave copies
constexpr int kCpPairs = 256;   // of a launch: they travel as its arguments

struct CopyPair {
  int src, dst, blocks;
};

struct CopyArgs {
  const char* from[4];  // k, v, their scales
  char* to[4];
  int64_t from_layer, to_layer;  // pages of a layer's pool
  int page_bytes, head_bytes;    // of k, and of v
  int page_blocks, block_bytes;  // blocks of a head's run, their bytes (whole pages: of all heads)
  int heads, shift;              // runs of a page, log2 of a run's pieces
  CopyPair pair[kCpPairs];
};

// A page's k, and its v, are runs of blocks that lie side by side: one a KV
// head, or, where all pairs copy whole pages, one of all heads.  A wave copies
// 8 KB of a run, 8 loads of 16 bytes a lane in flight, and the first piece's
// wave the run's scales.  Everything but a lane's constant offset is uniform:
// the grid is (pieces of k and v, layers, pairs), and the pairs are arguments.
//
// Bound by memory: 97 pages of 24 layers to another pool (1.2 GB read and written)
// 240 us, 5.1 TB/s, what a large copy reaches; 56 part pages of 48 layers 39 us.
// Three part pages of 48 layers: 4.2 us, a launch.
__global__ __launch_bounds__(kCpThreads) void paged_copy_kernel(CopyArgs a) {
  constexpr int N = kCpPiece / 1024;
  const int lane = threadIdx.x & 63;
  const int id = blockIdx.x * kCpWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int v = id & 1, head = (id >> 1) >> a.shift, piece = (id >> 1) & ((1 << a.shift) - 1);
  if (head >= a.heads) return;
  const CopyPair p = a.pair[blockIdx.z];
  const int64_t fp = blockIdx.y * a.from_layer + p.src, tp = blockIdx.y * a.to_layer + p.dst;
  const int bytes = p.blocks * a.block_bytes, at = piece * kCpPiece;
  if (piece == 0 && a.from[2]) {
    const char* s = a.from[2 + v] + (fp * a.heads + head) * a.page_blocks;
    char* d = a.to[2 + v] + (tp * a.heads + head) * a.page_blocks;
    for (int i = lane; i < p.blocks; i += 64) d[i] = s[i];
  }
  const int64_t off = (int64_t)head * a.head_bytes + at + 16 * lane;
  const u32x4* s = (const u32x4*)(a.from[v] + fp * a.page_bytes + off);
  u32x4* d = (u32x4*)(a.to[v] + tp * a.page_bytes + off);
  const int n = min((bytes - at) / 1024, N);  // (blocks are of 1 KB at least)
  if (n <= 0) return;
  u32x4 x[N];
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = s[64 * min(i, n - 1)];
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (i < n) d[64 * i] = x[i];
}

bool al16(const void* p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace
}  // namespace glq

extern "C" int glq_paged_copy(const glq_paged_copy_params* p, void* stream) {
  using namespace glq;
  clear_error();
  GLQ_CHECK(p != nullptr, "null params");
  const int64_t D = p->head_dim, page = p->page_size, Hk = p->kv_heads, L = p->layers;
  GLQ_CHECK(D == 64 || D == 128, "head_dim must be 64 or 128 (got %lld)", (long long)D);
  GLQ_CHECK(page >= 16 && page <= 1024 && (page & (page - 1)) == 0,
            "page_size must be a power of two in [16, 1024] (got %lld)", (long long)page);
  GLQ_CHECK(Hk > 0 && Hk <= 1024, "kv_heads must be in [1, 1024]");
  GLQ_CHECK(L >= 0 && L <= 65535, "layers must be in [0, 65535]");
  GLQ_CHECK(p->pairs >= 0 && p->pairs <= (1 << 24), "pairs must be in [0, 2^24]");
  const glq_paged_pools &f = p->from, &t = p->to;
  GLQ_CHECK(f.pages >= 0 && f.pages < (1ll << 31) && t.pages >= 0 && t.pages < (1ll << 31),
            "pages must be in [0, 2^31)");
  if (p->pairs == 0 || L == 0) return GLQ_OK;
  GLQ_CHECK(p->src && p->dst, "null pointer argument");
  GLQ_CHECK(f.k_pages && f.v_pages && t.k_pages && t.v_pages, "null pointer argument");
  const bool fp8 = f.k_scales != nullptr;
  GLQ_CHECK(!f.v_scales == !fp8 && !t.k_scales == !fp8 && !t.v_scales == !fp8,
            "k and v scales of both caches come together (8-bit pages) or not at all");
  GLQ_CHECK(al16(f.k_pages) && al16(f.v_pages) && al16(t.k_pages) && al16(t.v_pages),
            "pages must be 16-byte aligned");
  const int64_t bpp = page / kBlkTokens, block = kBlkTokens * D * (fp8 ? 1 : 2);
  const int64_t page_bytes = Hk * bpp * block, page_scales = Hk * bpp;
  const void* const from[4] = {f.k_pages, f.v_pages, f.k_scales, f.v_scales};
  void* const to[4] = {t.k_pages, t.v_pages, t.k_scales, t.v_scales};
  const bool same = from[0] == to[0];
  if (same) {
    GLQ_CHECK(from[1] == to[1] && from[2] == to[2] && from[3] == to[3] && f.pages == t.pages,
              "caches that share some of their memory must be one");
  } else {
    for (int i = 0; i < (fp8 ? 4 : 2); ++i)
      for (int j = 0; j < (fp8 ? 4 : 2); ++j)
        GLQ_CHECK(apart(from[i], L * f.pages * (i < 2 ? page_bytes : page_scales), to[j],
                        L * t.pages * (j < 2 ? page_bytes : page_scales)),
                  "caches that share some of their memory must be one");
  }
  // every page is written once, and none that is read (by pairs that copy anything)
  bool whole = true;
  {
    unsigned char* seen = (unsigned char*)calloc((size_t)(t.pages / 8 + 1), 1);
    GLQ_CHECK(seen != nullptr, "out of host memory");
    const char* what = nullptr;
    int64_t i = 0;
    for (; i < p->pairs && !what; ++i) {
      const int64_t s = p->src[i], d = p->dst[i], n = p->tokens ? p->tokens[i] : page;
      if (s < 0 || s >= f.pages || d < 0 || d >= t.pages)
        what = "page out of range";
      else if (n < 0 || n > page)
        what = "tokens must be in [0, page_size]";
      else if (n == 0)
        continue;
      else if (seen[d / 8] >> (d % 8) & 1)
        what = "a page is written twice";
      else
        seen[d / 8] |= (unsigned char)(1 << (d % 8));
      whole = whole && n > page - kBlkTokens;
    }
    if (same && !what)
      for (i = 0; i < p->pairs && !what; ++i)
        if ((!p->tokens || p->tokens[i]) && (seen[p->src[i] / 8] >> (p->src[i] % 8) & 1))
          what = "a page that is read is written";
    free(seen);
    GLQ_CHECK(!what, "pair %lld: %s", (long long)i - 1, what);
  }
  CopyArgs a{};
  for (int i = 0; i < 4; ++i) {
    a.from[i] = (const char*)from[i];
    a.to[i] = (char*)to[i];
  }
  a.from_layer = f.pages;
  a.to_layer = t.pages;
  a.page_bytes = (int)page_bytes;
  a.block_bytes = (int)block;
  a.heads = whole ? 1 : (int)Hk;
  a.page_blocks = (int)(whole ? Hk * bpp : bpp);
  a.head_bytes = a.page_blocks * a.block_bytes;
  const int64_t pieces = (a.head_bytes + kCpPiece - 1) / kCpPiece;
  while ((1ll << a.shift) < pieces) ++a.shift;
  const int64_t runs = whole ? pieces : Hk << a.shift;
  const dim3 grid((unsigned)((2 * runs + kCpWaves - 1) / kCpWaves), (unsigned)L);
  for (int64_t i = 0; i < p->pairs;) {
    int n = 0;
    for (; i < p->pairs && n < kCpPairs; ++i) {
      const int64_t tokens = p->tokens ? p->tokens[i] : page;
      const int blocks = (int)((tokens + kBlkTokens - 1) / kBlkTokens);
      if (blocks)
        a.pair[n++] = CopyPair{p->src[i], p->dst[i], whole ? a.page_blocks : blocks};
    }
    if (n == 0) break;
    paged_copy_kernel<<<dim3(grid.x, grid.y, (unsigned)n), dim3(kCpThreads), 0,
                        (hipStream_t)stream>>>(a);
    GLQ_LAUNCH_CHECK("paged_copy_kernel");
  }
  return GLQ_OK;
}
