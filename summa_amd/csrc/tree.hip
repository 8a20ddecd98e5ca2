// Trees of drafted tokens: who sees whom, which path the sampled tokens confirm, and that
// path's keys and values moved together in the paged caches.
//
// TextGenerator::generate (summa-llm/src/generate.rs:68-124) forwards one token a step. With
// drafted continuations it forwards a tree of them: token i of a sequence's n hangs on token
// parents[i] < i (-1: on the context; token 0 is the last token chosen, not yet in the cache).
// Their keys and values go behind the context (sm_paged_append at pos0 .. pos0 + n - 1), each
// sees the context and its ancestors (sm_paged_tree_attention), and where the token sampled
// behind token i is one of i's drafted children, that child is what the step would have
// forwarded next.
#include <algorithm>

#include "common.hpp"
#include "paged_map.hpp"

namespace sm {

int check_paged_caches(const char* who, const sm_paged_cache* caches, int64_t n);

namespace {

constexpr int kTreeRows = 1024;  // rows of a sequence's tree at most

// A token goes up its ancestors, whose numbers fall, so its mask's words are written once each,
// the last first. One workgroup a sequence, parents in LDS.
__global__ __launch_bounds__(256) void tree_masks_kernel(const int32_t* parents, const int32_t* pos0,
                                                         const int32_t* row_start, int rows,
                                                         int max_rows, uint32_t* mask, int words,
                                                         int32_t* positions) {
  __shared__ int32_t up[kTreeRows];
  const int s = (int)blockIdx.x;
  const PagedRows pr(row_start, s, rows, max_rows);
  for (int i = threadIdx.x; i < pr.n; i += 256) up[i] = parents[pr.first + i];
  const int base = pos0 ? pos0[s] : 0;
  __syncthreads();
  for (int i = threadIdx.x; i < pr.n; i += 256) {
    uint32_t* m = mask + (int64_t)(pr.first + i) * words;
    int w = words - 1, depth = -1;
    uint32_t bits = 0;
    for (int at = i; at >= 0;) {
      for (; w > at / 32; --w) {
        m[w] = bits;
        bits = 0;
      }
      bits |= 1u << (at % 32);
      ++depth;
      const int p = up[at];
      at = p < at ? p : -1;  // (a parent comes before its child)
    }
    for (; w >= 0; --w) {
      m[w] = bits;
      bits = 0;
    }
    if (positions) positions[pr.first + i] = base + depth;
  }
}

// One wave a sequence: of the current token's children the first whose drafted token is the one
// sampled behind it, until there is none.
__global__ __launch_bounds__(64) void tree_accept_kernel(const int32_t* parents,
                                                         const int32_t* tokens,
                                                         const int32_t* sampled,
                                                         const int32_t* row_start, int rows,
                                                         int max_rows, int32_t* path,
                                                         int32_t* count, int32_t* emitted) {
  __shared__ int32_t up[kTreeRows], drafted[kTreeRows], chosen[kTreeRows];
  const int s = (int)blockIdx.x, lane = threadIdx.x;
  const PagedRows pr(row_start, s, rows, max_rows);
  for (int i = lane; i < pr.n; i += kWave) {
    up[i] = parents[pr.first + i];
    drafted[i] = tokens[pr.first + i];
    chosen[i] = sampled[pr.first + i];
  }
  __syncthreads();
  int n = 0;
  for (int cur = pr.n > 0 ? 0 : -1; cur >= 0; ++n) {
    const int want = chosen[cur];
    if (lane == 0) {
      path[(int64_t)s * max_rows + n] = cur;
      if (emitted) emitted[(int64_t)s * max_rows + n] = want;
    }
    int next = -1;
    for (int i = cur + 1 + lane; i - lane < pr.n; i += kWave) {
      const uint64_t m = __ballot(i < pr.n && up[i] == cur && drafted[i] == want);
      if (m) {
        next = i - lane + (int)__builtin_ctzll(m);
        break;
      }
    }
    cur = next;
  }
  for (int i = n + lane; i < max_rows; i += kWave) {
    path[(int64_t)s * max_rows + i] = -1;
    if (emitted) emitted[(int64_t)s * max_rows + i] = -1;
  }
  if (lane == 0) count[s] = n;
}

constexpr int kLayers = 32;  // caches of a launch
struct KeepArgs {
  struct {
    uint8_t *k, *v, *ks, *vs;
  } c[kLayers];
  const int32_t *path, *count, *table, *pos0;
  Divide KVH, layers, bpp;
  int units, max_rows, pages, cols;
};

// Codes of a word times f, rounded again; NaN codes stay.
__device__ inline uint32_t rescale4(uint32_t w, float f) {
  const f32x2_t lo = __builtin_amdgcn_cvt_pk_f32_fp8(w, false),
                hi = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
  int y = __builtin_amdgcn_cvt_pk_fp8_f32(lo[0] * f, lo[1] * f, 0, false);
  y = __builtin_amdgcn_cvt_pk_fp8_f32(hi[0] * f, hi[1] * f, y, true);
  // bytes 0x7f and 0xff: 1 in the high bit of x
  const uint32_t x = ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
  const uint32_t nan = (x >> 7) * 0xffu;
  return ((uint32_t)y & ~nan) | (w & nan);
}
__device__ inline float pow2_down(int e) {  // 2^e, e <= 0; zero below f32's normal range
  return __uint_as_float((uint32_t)max(e + 127, 0) << 23);
}

// One wave a head of a sequence in one cache, 16 tokens (a block of the cache) at a time: what
// a block takes is read before it is written, and a block's tokens come from it or from behind
// it, so what later blocks take is still there.
//
// 8-bit: the block's scale becomes the largest of its own and those of the blocks that its
// tokens come from, as a scale never falls while tokens of its block stay; its other codes are
// scaled down with it. No values are looked through.
//
// Bound by latency: lengths, table, scales and tokens one behind the other, then the stores.
template <int HD, bool C8>
__global__ __launch_bounds__(256) void keep_kernel(KeepArgs a) {
  constexpr int ES = C8 ? 1 : 2, BB = kBlock * HD * ES;
  constexpr int NC = BB / 1024;            // 16-byte pieces a lane has of a block of k, and of v
  constexpr int LT = HD * ES / 16;         // lanes of a token's key
  const int unit = (int)(blockIdx.x * 4 + threadIdx.x / kWave), lane = threadIdx.x % kWave;
  if (unit >= a.units) return;
  int s = unit;
  const int kvh = a.KVH.mod(s), layer = a.layers.mod(s);
  const auto& c = a.c[layer];
  const int32_t* trow = a.table + (int64_t)s * a.cols;
  const int32_t* path = a.path + (int64_t)s * a.max_rows;
  const int pos0 = a.pos0[s];
  const int n = pos0 < 0 ? 0 : min(a.count[s], a.max_rows);
  auto block = [&](int blk) {
    return paged_block(trow, a.cols, a.pages, (int)a.KVH.d, kvh, a.bpp, blk);
  };
  int last = -1;  // the path's last entry so far
  for (int j0 = 0; j0 < n;) {
    // tokens j0 .. of the path, up to the end of the block: lane t has the block's token t
    const int64_t to0 = (int64_t)pos0 + j0;
    const int blk = (int)(to0 / kBlock), t0 = (int)(to0 % kBlock);
    const int m = min(kBlock - t0, n - j0);
    const int t = lane % kBlock, j = j0 + t - t0;
    const bool mine = t >= t0 && t < t0 + m;
    const int idx = mine ? path[j] : -1;
    const int before = t == t0 ? last : mine ? path[j - 1] : 0;
    const int64_t from = (int64_t)pos0 + idx;
    int src = -1;
    const int dst = to0 + m - 1 <= 0x7fffffff ? block(blk) : -1;
    if (mine && idx > before && from <= 0x7fffffff && dst >= 0) src = block((int)(from / kBlock));
    const uint64_t bad = __ballot(mine && src < 0 && lane < kBlock);
    const int good = bad ? (int)__builtin_ctzll(bad) : t0 + m;  // first token that is not moved
    if (good <= t0) return;  // (uniform)
    const bool moves = mine && t < good && from != (int64_t)pos0 + j;
    if (__ballot(moves) != 0) {
      const int off = (int)(from % kBlock);
      int own_k = 0, own_v = 0, ek = 0, ev = 0, new_k = 0, new_v = 0;
      if constexpr (C8) {
        own_k = c.ks[dst];
        own_v = c.vs[dst];
        ek = moves ? (int)c.ks[src] : 0;
        ev = moves ? (int)c.vs[src] : 0;
        new_k = max(own_k, (int)wave_max((float)ek));
        new_v = max(own_v, (int)wave_max((float)ev));
      }
      // keys: pieces lane + 64 i of the block, of token piece / LT
      u32x4 w[NC];
      uint32_t put = 0;  // pieces to be written
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        const int piece = i * kWave + lane, tok = piece / LT;
        const bool mv = __shfl((int)moves, tok, kWave);
        const int b = __shfl(src, tok, kWave), o = __shfl(off, tok, kWave);
        const int from_e = __shfl(ek, tok, kWave), e = mv ? from_e : own_k;
        if (mv || (C8 && new_k != own_k)) {
          put |= 1u << i;
          w[i] = *reinterpret_cast<const u32x4*>(
              c.k + (size_t)(mv ? b : dst) * BB + (mv ? o * LT + piece % LT : piece) * 16);
          if constexpr (C8)
            if (e != new_k) {
              const float f = pow2_down(e - new_k);
#pragma unroll
              for (int x = 0; x < 4; ++x) w[i][x] = rescale4(w[i][x], f);
            }
        }
      }
      // values: pieces lane + 64 i of the block hold tokens 4 g .. 4 g + 3 of T dims
      constexpr int T = 4 / ES;
      u32x4 v[NC];
      const int g = lane / 16;
      uint32_t any = 0;  // of this lane's four tokens, those that move
#pragma unroll
      for (int y = 0; y < 4; ++y) any |= (uint32_t)(__shfl((int)moves, 4 * g + y, kWave)) << y;
      const bool store_v = any || (C8 && new_v != own_v);
      if (store_v) {
#pragma unroll
        for (int i = 0; i < NC; ++i)
          v[i] = *reinterpret_cast<const u32x4*>(c.v + (size_t)dst * BB + i * 1024 + lane * 16);
        if constexpr (C8)
          if (new_v != own_v) {
            const float f = pow2_down(own_v - new_v);
#pragma unroll
            for (int i = 0; i < NC; ++i)
#pragma unroll
              for (int x = 0; x < 4; ++x) v[i][x] = rescale4(v[i][x], f);
          }
      }
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const int b = __shfl(src, 4 * g + y, kWave), o = __shfl(off, 4 * g + y, kWave);
        const int e = __shfl(ev, 4 * g + y, kWave);
        if (!(any >> y & 1)) continue;
#pragma unroll
        for (int i = 0; i < NC; ++i) {
          const u32x4 x = *reinterpret_cast<const u32x4*>(
              c.v + (size_t)b * BB + i * 1024 + (o / 4 * 16 + lane % 16) * 16);
          if constexpr (C8) {  // word t: dim t's four tokens
            const float f = pow2_down(e - new_v);
#pragma unroll
            for (int z = 0; z < 4; ++z) {
              const uint32_t q = e != new_v ? rescale4(x[z], f) : x[z];
              const uint32_t byte = q >> (8 * (o % 4)) & 0xffu;
              v[i][z] = (v[i][z] & ~(0xffu << (8 * y))) | byte << (8 * y);
            }
          } else {  // words 2 t, 2 t + 1: dim t's four tokens
#pragma unroll
            for (int z = 0; z < T; ++z) {
              const uint32_t half = (o % 4 < 2 ? x[2 * z] : x[2 * z + 1]) >> (16 * (o % 2)) & 0xffffu;
              const uint32_t old = v[i][2 * z + y / 2];
              v[i][2 * z + y / 2] = (old & ~(0xffffu << (16 * (y % 2)))) | half << (16 * (y % 2));
            }
          }
        }
      }
      // (every load of this block is done before its first store)
#pragma unroll
      for (int i = 0; i < NC; ++i) asm volatile("" : "+v"(w[i]), "+v"(v[i]) : : "memory");
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        if (put >> i & 1)
          *reinterpret_cast<u32x4*>(c.k + (size_t)dst * BB + (i * kWave + lane) * 16) = w[i];
        if (store_v)
          *reinterpret_cast<u32x4*>(c.v + (size_t)dst * BB + i * 1024 + lane * 16) = v[i];
      }
      if (C8 && lane == 0) {
        c.ks[dst] = (uint8_t)new_k;
        c.vs[dst] = (uint8_t)new_v;
      }
    }
    if (good < t0 + m) return;  // (uniform) the path ends there
    last = __shfl(idx, t0 + m - 1, kWave);
    j0 += m;
  }
}

int check_rows(const char* who, int64_t S, int64_t rows, int64_t max_rows,
               const int32_t* row_start) {
  const int64_t most = 0x7fffffff;
  SM_REQUIRE(S >= 0 && rows >= 0 && max_rows >= 0 && S < (1 << 24) && rows < most && max_rows <= rows,
             "%s: need 0 to 2^24 - 1 sequences and 0 <= max_rows <= rows", who);
  SM_REQUIRE(max_rows <= kTreeRows, "%s: a sequence's tree has at most 1024 rows", who);
  SM_REQUIRE(row_start || S == 0 || rows == S * max_rows,
             "%s: without row_start, rows must be S * max_rows", who);
  return SM_OK;
}

}  // namespace
}  // namespace sm

using namespace sm;

extern "C" int sm_tree_masks(const int32_t* parents, const int32_t* pos0, const int32_t* row_start,
                             int64_t S, int64_t rows, int64_t max_rows, int32_t* mask,
                             int64_t words, int32_t* positions, void* stream) {
  const char* me = "sm_tree_masks";
  SM_TRY(check_rows(me, S, rows, max_rows, row_start));
  if (S == 0 || max_rows == 0) return SM_OK;
  SM_REQUIRE(parents && mask && (pos0 || !positions), "%s: null buffer", me);
  SM_REQUIRE(words >= ceil_div(max_rows, 32) && words <= 1 << 20,
             "%s: words must be at least max_rows / 32", me);
  tree_masks_kernel<<<(unsigned)S, 256, 0, as_stream(stream)>>>(
      parents, pos0, row_start, (int)rows, (int)max_rows, reinterpret_cast<uint32_t*>(mask),
      (int)words, positions);
  SM_LAUNCH_CHECK();
  return SM_OK;
}

extern "C" int sm_tree_accept(const int32_t* parents, const int32_t* tokens,
                              const int32_t* sampled, const int32_t* row_start, int64_t S,
                              int64_t rows, int64_t max_rows, int32_t* path, int32_t* count,
                              int32_t* emitted, void* stream) {
  const char* me = "sm_tree_accept";
  SM_TRY(check_rows(me, S, rows, max_rows, row_start));
  if (S == 0) return SM_OK;
  SM_REQUIRE(count && (max_rows == 0 || (parents && tokens && sampled && path)), "%s: null buffer",
             me);
  tree_accept_kernel<<<(unsigned)S, 64, 0, as_stream(stream)>>>(
      parents, tokens, sampled, row_start, (int)rows, (int)max_rows, path, count, emitted);
  SM_LAUNCH_CHECK();
  return SM_OK;
}

extern "C" int sm_paged_keep(const sm_paged_cache* caches, int64_t ncaches, const int32_t* path,
                             const int32_t* count, int64_t S, int64_t max_rows,
                             const int32_t* block_table, int64_t table_cols, const int32_t* pos0,
                             void* stream) {
  const char* me = "sm_paged_keep";
  SM_TRY(check_paged_caches(me, caches, ncaches));
  SM_REQUIRE(S >= 0 && max_rows >= 0 && S < (1 << 24) && max_rows <= 0x7fffffff,
             "%s: need 0 to 2^24 - 1 sequences and max_rows >= 0", me);
  if (ncaches == 0 || S == 0 || max_rows == 0) return SM_OK;
  SM_REQUIRE(path && count && block_table && pos0, "%s: null buffer", me);
  SM_REQUIRE(table_cols > 0 && table_cols <= 0x7fffffff, "%s: table_cols must be positive", me);
  const bool c8 = caches->dtype == SM_F8E4M3;
  const int64_t KVH = caches->kv_heads, most = std::min<int64_t>(ncaches, kLayers);
  if (S * KVH > ((1 << 26) - 4) / most) {  // (a grid holds less than 2^32 threads)
    set_error("%s: problem too large", me);
    return SM_ERR_UNSUPPORTED;
  }
  KeepArgs a;
  a.path = path;
  a.count = count;
  a.table = block_table;
  a.pos0 = pos0;
  a.KVH = Divide((int)KVH);
  a.bpp = Divide((int)(caches->page_tokens / kBlock));
  a.max_rows = (int)max_rows;
  a.pages = (int)caches->pages;
  a.cols = (int)table_cols;
  for (int64_t l0 = 0; l0 < ncaches; l0 += kLayers) {
    const int64_t layers = std::min<int64_t>(kLayers, ncaches - l0);
    a.layers = Divide((int)layers);
    a.units = (int)(S * KVH * layers);
    for (int64_t i = 0; i < layers; ++i) {
      const sm_paged_cache& c = caches[l0 + i];
      a.c[i] = {static_cast<uint8_t*>(c.k), static_cast<uint8_t*>(c.v), c.k_scales, c.v_scales};
    }
    const unsigned wgs = (unsigned)ceil_div(a.units, 4);
    hipStream_t st = as_stream(stream);
    if (caches->head_dim == 64) {
      if (c8) keep_kernel<64, true><<<wgs, 256, 0, st>>>(a);
      else keep_kernel<64, false><<<wgs, 256, 0, st>>>(a);
    } else {
      if (c8) keep_kernel<128, true><<<wgs, 256, 0, st>>>(a);
      else keep_kernel<128, false><<<wgs, 256, 0, st>>>(a);
    }
    SM_LAUNCH_CHECK();
  }
  return SM_OK;
}
