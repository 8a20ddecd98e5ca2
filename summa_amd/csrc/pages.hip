// The pages of a paged KV cache: who holds them, and their contents moved.
//
// AttnCache (summa-llm/src/model/attention.rs:20-40) grows with its one sequence; here sequences
// take pages from a pool as they grow, rollouts of a group share their prompt's full pages
// (GrpoGenerationBatchRequest: one example per group, summa-train/src/posttrain.rs:1206-1216),
// and a page goes back when its last holder leaves it. refs[p] is the number of table entries that hold page p,
// zero for a free one; there is no list of free pages, so nothing can fall out of step with
// it: a page is given out as the lowest free one, found by a scan of refs, which makes every
// result a function of refs and tables alone.
//
// The bookkeeping is whole numbers: a scan of 65536 counts by one workgroup is 16 passes over 4096, 1.8 us
// each. Counts of shared pages are raised and lowered by atomics, whose order does not change
// them. The contents are copies at the memory's rate.
#include <algorithm>

#include "common.hpp"
#include "paged_map.hpp"

namespace sm {

int check_paged_cache(const char* who, const sm_paged_cache* c);
int check_paged_caches(const char* who, const sm_paged_cache* caches, int64_t n);

namespace {

constexpr int kScan = 1024;        // threads of the workgroup that scans
constexpr int kWaves = kScan / kWave;

// Exclusive prefix sum of one value a thread over the workgroup, and the sum of all.
template <typename T>
struct Scan {
  T part[kWaves];
  __device__ inline T exclusive(T v, T& total) {
    const int lane = threadIdx.x % kWave, w = threadIdx.x / kWave;
    T inc = v;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
      const T t = __shfl_up(inc, o, kWave);
      if (lane >= o) inc += t;
    }
    if (lane == kWave - 1) part[w] = inc;
    __syncthreads();
    T base = 0;
    total = 0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
      if (i < w) base += part[i];
      total += part[i];
    }
    __syncthreads();
    return base + inc - v;
  }
};

// Four counts from p on; what is behind the last page counts as held.
__device__ inline void load_refs(const int32_t* refs, int pages, int64_t p, int (&r)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = p + i < pages ? refs[p + i] : 1;
}

// Gives pages to 1024 askers at a time, askers in order and pages from the lowest free one up.
struct Giver {
  Scan<int> scan;
  Scan<int64_t> sums;  // (1024 rows may ask for more than 2^31 pages together)
  int before[kScan];  // pages that the askers before this one get
  int first[kScan];   // column of the asker's first new page
  int row[kScan];     // its table row; -1: none
  int64_t next;       // pages below it are held
};

// Each thread asks for `want` pages from column `col` of table row `r` on. give(row, col, page,
// asker) is called once for each page given. Returns how many were not there (uniform). N holds
// what 1024 askers want together (fork_kernel's one each: 256 children 8.3 us
// with sums in 64 bits, 6.8 in 32).
template <typename N, typename Give>
__device__ inline N give_pages(Scan<N>& sums, Giver& sh, int32_t* refs, int pages, int want, int r,
                               int col, Give give) {
  N asked;
  const N before = sums.exclusive(want, asked);
  const int total = (int)min(asked, (N)pages);  // no more can be given
  sh.before[threadIdx.x] = (int)min(before, (N)pages);
  sh.first[threadIdx.x] = col;
  sh.row[threadIdx.x] = r;
  __syncthreads();
  int given = 0;
  while (given < total && sh.next < pages) {  // (uniform: next is read between barriers)
    const int64_t from = sh.next, p = from + 4 * (int64_t)threadIdx.x;
    int c[4];
    load_refs(refs, pages, p, c);
    int have = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) have += c[i] <= 0;
    int found;
    int rank = given + sh.scan.exclusive(have, found);
    if (threadIdx.x == 0) sh.next = from + 4 * kScan;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (c[i] > 0) continue;
      if (rank < total) {
        // the last asker with before <= rank (those that want none end where they start)
        int lo = 0, hi = kScan - 1;
        while (lo < hi) {
          const int mid = (lo + hi + 1) / 2;
          if (sh.before[mid] <= rank) lo = mid;
          else hi = mid - 1;
        }
        refs[p + i] = 1;
        give(sh.row[lo], sh.first[lo] + rank - sh.before[lo], (int)(p + i), lo);
        if (rank == total - 1) sh.next = p + i + 1;  // (after the barrier: the only writer)
      }
      ++rank;
    }
    given = min(total, given + found);
    __syncthreads();
  }
  return asked - given;
}

__device__ inline int pages_of(int tokens, const Divide& page) {
  return tokens <= 0 ? 0 : page.div(tokens - 1) + 1;
}

// Pages for tokens[s] tokens of every sequence: columns from the first that names none on.
// Bound by latency of one workgroup: a wave looks through its rows' entries 64 at a time, and the pool is
// scanned from its first page to the last one given. 32 sequences of 1000 tokens in pages of 16 6 us;
// 64 of 32 k tokens in pages of 64 13 us, in pages of 16 36 us, 2 more for four pages that are found in
// front, and 0.2 ms (1.7 ms) where the first free one lies behind 450 k (3.6 M) held ones.
__global__ __launch_bounds__(kScan) void reserve_kernel(int32_t* refs, int pages, int32_t* table,
                                                        int S, int cols, const int32_t* tokens,
                                                        Divide page, int32_t* missing) {
  __shared__ Giver sh;
  __shared__ int held[kScan];
  if (threadIdx.x == 0) sh.next = 0;
  __syncthreads();
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  int64_t lacking = 0;
  for (int64_t s0 = 0; s0 < S; s0 += kScan) {
    // columns in use: a wave a row, 64 columns at a time
    for (int i = wave; i < kScan && s0 + i < S; i += kWaves) {
      const int32_t* t = table + (s0 + i) * cols;
      const int need = min(cols, pages_of(tokens[s0 + i], page));
      int n = 0;
      while (n < need) {
        const bool none = n + (int64_t)lane >= need || t[n + lane] < 0;
        const uint64_t m = __ballot(none);
        if (m) {
          n = min(need, n + (int)__builtin_ctzll(m));
          break;
        }
        n += kWave;
      }
      if (lane == 0) held[i] = min(n, need);
    }
    __syncthreads();
    const int64_t s = s0 + threadIdx.x;
    const int asked = s < S ? pages_of(tokens[s], page) : 0;
    const int col = s < S ? held[threadIdx.x] : 0;
    const int want = max(0, min(cols, asked) - col);
    lacking += max(0, asked - cols);  // columns that the table does not have
    const int64_t none = give_pages(sh.sums, sh, refs, pages, want, threadIdx.x, col,
                                    [&](int r, int c, int p, int) {
                                      table[(s0 + r) * cols + c] = p;
                                    });
    if (threadIdx.x == 0) lacking += none;
    __syncthreads();
  }
  if (!missing) return;
  int64_t total;
  sh.sums.exclusive(lacking, total);
  if (threadIdx.x == 0) *missing = (int32_t)min(total, (int64_t)0x7fffffff);
}

struct ForkArgs {
  int32_t *refs, *out, *src, *dst, *missing;
  const int32_t *table, *tokens, *source;
  Divide page;
  int pages, P, C, cols;
};

__global__ void clear_missing_kernel(int32_t* missing) { *missing = 0; }

// *to += n, 2^31 - 1 at most.
__device__ inline void add_missing(int32_t* to, int64_t n) {
  if (n <= 0) return;
  int32_t old = *reinterpret_cast<volatile int32_t*>(to), seen;
  while ((seen = atomicCAS(to, old, (int32_t)min((int64_t)old + n, (int64_t)0x7fffffff))) != old)
    old = seen;
}

// Workgroup 0 gives each child a page of its own for its prompt's unfinished one; the others
// share the full pages, a wave a child. A page that the prompt's row does not hold is not the
// child's either: nothing could be copied to one of its own, which would then show the tokens
// of whoever had it last.
__global__ __launch_bounds__(kScan) void fork_kernel(ForkArgs a) {
  if (blockIdx.x > 0) {
    const int64_t c = (int64_t)(blockIdx.x - 1) * kWaves + threadIdx.x / kWave;
    if (c >= a.C) return;
    const int p = a.source[c], lane = threadIdx.x % kWave;
    const bool ok = p >= 0 && p < a.P;
    const int n = ok ? max(0, a.tokens[p]) : 0, full = a.page.div(n);
    const bool part = n - full * (int)a.page.d > 0;
    int lacking = 0;  // of this lane's columns
    for (int j = lane; j < a.cols; j += kWave) {
      if (j == full && part) continue;  // workgroup 0's
      int page = -1;
      if (j < full) {
        page = a.table[(int64_t)p * a.cols + j];
        if (page < 0 || page >= a.pages) {
          page = -1;
          ++lacking;
        } else {
          atomicAdd(a.refs + page, 1);
        }
      }
      a.out[c * a.cols + j] = page;
    }
    if (!a.missing) return;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) lacking += __shfl_xor(lacking, o, kWave);
    // and the columns that the table does not have
    if (lane == 0)
      add_missing(a.missing, !ok ? 1 : (int64_t)lacking + max(0, full + (part ? 1 : 0) - a.cols));
    return;
  }
  __shared__ Giver sh;
  if (threadIdx.x == 0) sh.next = 0;
  __syncthreads();
  int64_t lacking = 0;
  for (int64_t c0 = 0; c0 < a.C; c0 += kScan) {
    const int64_t c = c0 + threadIdx.x;
    int full = 0, want = 0;
    int32_t from = -1;
    if (c < a.C) {
      const int p = a.source[c];
      if (p >= 0 && p < a.P) {
        const int n = max(0, a.tokens[p]);
        full = a.page.div(n);
        if (full < a.cols && n - full * (int)a.page.d > 0) {
          from = a.table[(int64_t)p * a.cols + full];
          if (from >= a.pages) from = -1;
          want = from >= 0;
          lacking += from < 0;
          a.out[c * a.cols + full] = -1;
        }
      }
      a.src[c] = -1;
      a.dst[c] = -1;
    }
    __syncthreads();
    const int none = give_pages(sh.scan, sh, a.refs, a.pages, want, threadIdx.x, full,
                                [&](int r, int col, int page, int) {
                                  a.out[(c0 + r) * a.cols + col] = page;
                                  a.dst[c0 + r] = page;
                                });
    if (threadIdx.x == 0) lacking += none;
    __syncthreads();
    if (c < a.C && from >= 0 && a.dst[c] >= 0) a.src[c] = from;
    __syncthreads();
  }
  if (!a.missing) return;
  int64_t total;
  sh.sums.exclusive(lacking, total);
  if (threadIdx.x == 0) add_missing(a.missing, total);
}

// A wave a row: entries behind the first tokens[s] tokens' leave their pages.
__global__ __launch_bounds__(256) void free_kernel(int32_t* refs, int pages, int32_t* table, int S,
                                                   int cols, const int32_t* tokens, Divide page) {
  const int64_t s = (int64_t)blockIdx.x * 4 + threadIdx.x / kWave;
  if (s >= S) return;
  const int keep = tokens ? pages_of(tokens[s], page) : 0;
  for (int64_t j = (int64_t)keep + threadIdx.x % kWave; j < cols; j += kWave) {
    int32_t* e = table + s * cols + j;
    const int p = *e;
    if (p >= 0 && p < pages) {
      // an entry too many does not take the count below zero for good
      if (atomicSub(refs + p, 1) <= 0) atomicAdd(refs + p, 1);
    }
    if (p != -1) *e = -1;
  }
}

// Live pages to the front: the i-th live page from L on moves to the i-th free page below L,
// L the number of live pages. No page is read and written.
__global__ __launch_bounds__(kScan) void compact_kernel(const int32_t* refs, int pages,
                                                        int32_t* refs_out, int32_t* where,
                                                        int32_t* src, int32_t* dst) {
  __shared__ Scan<int> scan;
  const int t = threadIdx.x;
  int live = 0;
  for (int64_t p = 4 * t; p < pages; p += 4 * kScan) {
    int c[4];
    load_refs(refs, pages, p, c);
#pragma unroll
    for (int i = 0; i < 4; ++i) live += p + i < pages && c[i] > 0;
  }
  int L;
  scan.exclusive(live, L);
  int holes = 0;
  for (int64_t p0 = 0; p0 < L; p0 += 4 * kScan) {
    const int64_t p = p0 + 4 * t;
    int c[4], n = 0, found;
    load_refs(refs, pages, p, c);
#pragma unroll
    for (int i = 0; i < 4; ++i) n += p + i < L && c[i] <= 0;
    int rank = holes + scan.exclusive(n, found);
    holes += found;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (p + i < L) {
        if (c[i] <= 0) dst[rank++] = (int)(p + i);
        where[p + i] = c[i] > 0 ? (int)(p + i) : -1;
        if (c[i] > 0) refs_out[p + i] = c[i];
      }
  }
  __syncthreads();
  int moved = 0;
  for (int64_t p0 = L; p0 < pages; p0 += 4 * kScan) {
    const int64_t p = p0 + 4 * t;
    int c[4], n = 0, found;
    load_refs(refs, pages, p, c);
#pragma unroll
    for (int i = 0; i < 4; ++i) n += p + i < pages && c[i] > 0;
    int rank = moved + scan.exclusive(n, found);
    moved += found;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (p + i < pages) {
        int to = -1;
        if (c[i] > 0) {
          to = dst[rank];
          src[rank++] = (int)(p + i);
          refs_out[to] = c[i];
        }
        where[p + i] = to;
        refs_out[p + i] = 0;
      }
  }
  for (int i = holes + t; i < pages / 2; i += kScan) src[i] = dst[i] = -1;
}

__global__ __launch_bounds__(256) void remap_kernel(const int32_t* table, int64_t n,
                                                    const int32_t* where, int pages,
                                                    int32_t* out) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  const int p = table[i];
  out[i] = p >= 0 && p < pages ? where[p] : -1;
}

constexpr int kLayers = 32;  // caches of a launch
struct CopyArgs {
  struct {
    uint8_t *k, *v, *ks, *vs;
  } c[kLayers];
  const int32_t *src, *dst;
  Divide parts, layers;
  int64_t page_bytes;  // of k, and of v
  int pages, scale_bytes;
};
constexpr int kPart = 16384;  // bytes of k or v that a workgroup copies

// A workgroup copies up to 16 KB of a page's k or v, four 16-byte loads in flight a lane; the
// page's first also its scales.
__global__ __launch_bounds__(256) void copy_kernel(CopyArgs a) {
  int x = (int)blockIdx.x;
  const int part = a.parts.mod(x), layer = a.layers.mod(x);
  const int s = a.src[x], d = a.dst[x];
  if (s < 0 || d < 0 || s >= a.pages || d >= a.pages || s == d) return;
  const auto& c = a.c[layer];
  const int half = (int)a.parts.d / 2;
  const bool values = part >= half;
  const int64_t at = (int64_t)(values ? part - half : part) * kPart;
  const uint8_t* from = (values ? c.v : c.k) + s * a.page_bytes + at;
  uint8_t* to = (values ? c.v : c.k) + d * a.page_bytes + at;
  const int n = (int)min((int64_t)kPart, a.page_bytes - at);
  u32x4 w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int b = (i * 256 + (int)threadIdx.x) * 16;
    if (b < n) w[i] = *reinterpret_cast<const u32x4*>(from + b);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int b = (i * 256 + (int)threadIdx.x) * 16;
    if (b < n) *reinterpret_cast<u32x4*>(to + b) = w[i];
  }
  if (c.ks && at == 0) {
    uint8_t* sc = values ? c.vs : c.ks;
    for (int i = threadIdx.x; i < a.scale_bytes; i += 256)
      sc[(int64_t)d * a.scale_bytes + i] = sc[(int64_t)s * a.scale_bytes + i];
  }
}

int check_pool(const char* who, const int32_t* refs, int64_t pages, int64_t page_tokens) {
  SM_REQUIRE(refs, "%s: null refs", who);
  SM_REQUIRE(pages > 0 && pages <= 0x7fffffff - 4 * kScan, "%s: pages must be positive, below 2^31 - 4096",
             who);
  SM_REQUIRE(page_tokens > 0 && page_tokens <= 0x7fffffff, "%s: page_tokens must be positive", who);
  return SM_OK;
}
int check_table(const char* who, int64_t S, int64_t cols) {
  SM_REQUIRE(S >= 0 && cols > 0 && cols <= 0x7fffffff && S <= (1 << 24),
             "%s: need 0 to 2^24 sequences and table_cols > 0", who);
  return SM_OK;
}

}  // namespace
}  // namespace sm

using namespace sm;

extern "C" int sm_page_reserve(int32_t* refs, int64_t pages, int32_t* block_table, int64_t S,
                               int64_t table_cols, const int32_t* tokens, int64_t page_tokens,
                               int32_t* missing, void* stream) {
  const char* me = "sm_page_reserve";
  SM_TRY(check_pool(me, refs, pages, page_tokens));
  SM_TRY(check_table(me, S, table_cols));
  SM_REQUIRE(S == 0 || (block_table && tokens), "%s: null buffer", me);
  reserve_kernel<<<1, kScan, 0, as_stream(stream)>>>(refs, (int)pages, block_table, (int)S,
                                                     (int)table_cols, tokens,
                                                     Divide((int)page_tokens), missing);
  SM_LAUNCH_CHECK();
  return SM_OK;
}

extern "C" int sm_page_fork(int32_t* refs, int64_t pages, const int32_t* block_table, int64_t P,
                            int64_t table_cols, const int32_t* tokens, const int32_t* source,
                            int64_t C, int64_t page_tokens, int32_t* out, int32_t* src,
                            int32_t* dst, int32_t* missing, void* stream) {
  const char* me = "sm_page_fork";
  SM_TRY(check_pool(me, refs, pages, page_tokens));
  SM_TRY(check_table(me, P, table_cols));
  SM_TRY(check_table(me, C, table_cols));
  SM_REQUIRE(C == 0 || (source && out && src && dst), "%s: null buffer", me);
  SM_REQUIRE(C == 0 || P == 0 || (block_table && tokens), "%s: null buffer", me);
  const uintptr_t t = reinterpret_cast<uintptr_t>(block_table), o = reinterpret_cast<uintptr_t>(out);
  SM_REQUIRE(C == 0 || P == 0 || t + (size_t)(P * table_cols) * 4 <= o ||
                 o + (size_t)(C * table_cols) * 4 <= t,
             "%s: out must not overlap block_table", me);
  ForkArgs a;
  a.refs = refs;
  a.out = out;
  a.src = src;
  a.dst = dst;
  a.missing = missing;
  a.table = block_table;
  a.tokens = tokens;
  a.source = source;
  a.page = Divide((int)page_tokens);
  a.pages = (int)pages;
  a.P = (int)P;
  a.C = (int)C;
  a.cols = (int)table_cols;
  if (missing) {  // (which all workgroups add to)
    clear_missing_kernel<<<1, 1, 0, as_stream(stream)>>>(missing);
    SM_LAUNCH_CHECK();
  }
  fork_kernel<<<(unsigned)(1 + ceil_div(C, kWaves)), kScan, 0, as_stream(stream)>>>(a);
  SM_LAUNCH_CHECK();
  return SM_OK;
}

extern "C" int sm_page_free(int32_t* refs, int64_t pages, int32_t* block_table, int64_t S,
                            int64_t table_cols, const int32_t* tokens, int64_t page_tokens,
                            void* stream) {
  const char* me = "sm_page_free";
  SM_TRY(check_pool(me, refs, pages, page_tokens));
  SM_TRY(check_table(me, S, table_cols));
  if (S == 0) return SM_OK;
  SM_REQUIRE(block_table, "%s: null buffer", me);
  free_kernel<<<(unsigned)ceil_div(S, 4), 256, 0, as_stream(stream)>>>(
      refs, (int)pages, block_table, (int)S, (int)table_cols, tokens, Divide((int)page_tokens));
  SM_LAUNCH_CHECK();
  return SM_OK;
}

extern "C" int sm_page_compact(const int32_t* refs, int64_t pages, int32_t* refs_out,
                               int32_t* page_map, int32_t* src, int32_t* dst, void* stream) {
  const char* me = "sm_page_compact";
  SM_TRY(check_pool(me, refs, pages, 1));
  SM_REQUIRE(refs_out && page_map && (pages < 2 || (src && dst)), "%s: null buffer", me);
  compact_kernel<<<1, kScan, 0, as_stream(stream)>>>(refs, (int)pages, refs_out, page_map, src,
                                                     dst);
  SM_LAUNCH_CHECK();
  return SM_OK;
}

extern "C" int sm_page_remap(const int32_t* block_table, int64_t n, const int32_t* page_map,
                             int64_t pages, int32_t* out, void* stream) {
  const char* me = "sm_page_remap";
  SM_REQUIRE(n >= 0 && n <= (int64_t)1 << 31 && pages > 0 && pages <= 0x7fffffff,
             "%s: need 0 to 2^31 entries and pages > 0", me);
  if (n == 0) return SM_OK;
  SM_REQUIRE(block_table && page_map && out, "%s: null buffer", me);
  remap_kernel<<<(unsigned)ceil_div(n, 256), 256, 0, as_stream(stream)>>>(
      block_table, n, page_map, (int)pages, out);
  SM_LAUNCH_CHECK();
  return SM_OK;
}

// Shared with the other calls over several layers' caches: all of one geometry.
int sm::check_paged_caches(const char* who, const sm_paged_cache* caches, int64_t n) {
  SM_REQUIRE(n >= 0 && n <= 65535 && (n == 0 || caches), "%s: need 0 to 65535 caches", who);
  for (int64_t i = 0; i < n; ++i) {
    SM_TRY(check_paged_cache(who, caches + i));
    const sm_paged_cache &a = caches[0], &b = caches[i];
    SM_REQUIRE(a.pages == b.pages && a.kv_heads == b.kv_heads && a.page_tokens == b.page_tokens &&
                   a.head_dim == b.head_dim && a.dtype == b.dtype,
               "%s: the caches must have one geometry and dtype", who);
  }
  return SM_OK;
}

extern "C" int sm_paged_copy(const sm_paged_cache* caches, int64_t ncaches, const int32_t* src,
                             const int32_t* dst, int64_t n, void* stream) {
  const char* me = "sm_paged_copy";
  SM_TRY(check_paged_caches(me, caches, ncaches));
  SM_REQUIRE(n >= 0 && n <= 0x7fffffff, "%s: need 0 to 2^31 - 1 pairs", me);
  if (ncaches == 0 || n == 0) return SM_OK;
  SM_REQUIRE(src && dst, "%s: null buffer", me);
  const bool c8 = caches->dtype == SM_F8E4M3;
  CopyArgs a;
  a.pages = (int)caches->pages;
  a.page_bytes = caches->kv_heads * caches->page_tokens * caches->head_dim * (c8 ? 1 : 2);
  a.scale_bytes = (int)(caches->kv_heads * (caches->page_tokens / kBlock));
  const int64_t parts = 2 * ceil_div(a.page_bytes, kPart);
  // (a grid holds less than 2^32 threads: a launch takes the layers and pairs that fit)
  constexpr int64_t most = (1 << 24) - 1;
  if (parts > most || parts * ncaches > 0x7fffffff / n) {
    set_error("%s: problem too large", me);
    return SM_ERR_UNSUPPORTED;
  }
  a.parts = Divide((int)parts);
  const int64_t of_launch = std::min<int64_t>(kLayers, most / parts);
  for (int64_t l0 = 0; l0 < ncaches; l0 += of_launch) {
    const int64_t layers = std::min(of_launch, ncaches - l0);
    a.layers = Divide((int)layers);
    for (int64_t i = 0; i < layers; ++i) {
      const sm_paged_cache& c = caches[l0 + i];
      a.c[i] = {static_cast<uint8_t*>(c.k), static_cast<uint8_t*>(c.v),
                c8 ? c.k_scales : nullptr, c8 ? c.v_scales : nullptr};
    }
    const int64_t each = most / (parts * layers);
    for (int64_t i = 0; i < n; i += each) {
      a.src = src + i;
      a.dst = dst + i;
      copy_kernel<<<(unsigned)(parts * layers * std::min(each, n - i)), 256, 0,
                    as_stream(stream)>>>(a);
      SM_LAUNCH_CHECK();
    }
  }
  return SM_OK;
}
