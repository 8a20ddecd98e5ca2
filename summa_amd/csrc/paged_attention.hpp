// Attention over a paged KV cache, 16-bit or 8-bit (e4m3 codes with a power-of-two
// scale per 16 tokens of a head); sm_paged_attention states the layouts.
//
//   MultiHeadAttention::forward_cached / sdpa (summa-llm/src/model/attention.rs:216-265,
//   318-371): softmax(q . K^T / sqrt(hd)) . V over the keys up to the query's position.
//
// A row here is a (token, query head of a KV head's group) pair: the rows of a KV head see
// the same keys, so its K and V are read once for G tokens' heads as for G heads of a token.
//
// Both kernels work on transposed scores, S^T = K Q^T, so that a lane owns one row and its
// scores are, as they come out of the matrix cores, the B operand of O^T += V^T P^T: the sum
// over keys may run in any order, and V is stored in that order. P never leaves the
// registers, and nothing is transposed on the way.
// - The softmax is one pass with a running maximum and sum in f32, in units of log2. The
//   reference that weights are taken from is raised only when a score passes it by more than
//   kWeightMost, so most steps neither reduce over lanes nor rescale O.
// - An 8-bit block's K scale is a factor on its scores. Its V scale 2^e goes into the weights:
//   t = score + e is what the running maximum is taken of, P' = 2^(t - max) multiplies the bare
//   codes, and P' stays in its type's range whatever the scales are. A value's error is that of
//   its weight, relative to the largest |weight x scale| that the row has.
// - The sum of the weights, without their scales, is 2^-e P' block by block while every scale
//   so far is at most 2^kScaleSmall: a P' that f32 rounds to zero then has a weight of less
//   than 2^-50 of the largest. Behind a larger scale it is taken of the scores themselves, with
//   exponentials of its own. It is held kSumShift binary orders up, where the 183 orders between
//   the least and the largest scale lie inside f32 (where a scale of 2^120 sets the reference,
//   weights 33 orders below the largest are still left out), and moved in two factors that f32
//   holds where the product of both is less than it does.
// - P' is rounded to f16 for 8-bit and f16 values (codes are exact in f16), to bf16 for bf16
//   ones, whose range f16 does not hold: at most half a step (2^-11, 2^-8) of each weight,
//   like the one rounding of the output. In f16 weights fill the type's range: the largest is
//   2^11 to 2^15 (f16 ends at 65504), so that only those 25 binary orders below it lose bits
//   and those 36 below it all. (131 k keys 26 orders below one dominant key have 0.2 % of the
//   sum; with the largest weight at 1 all of that would be lost.) The 16-row kernel multiplies the rest of each weight
//   too, in 16 bits again, which costs it 1-2 % (its matrix cores wait for memory) and leaves
//   the output's rounding: error of a rollout step in f16 2.1e-4 with it, 2.6e-4 without. The
//   tile kernel, bound by its products, does not: 2 x 1024 rows on 28 k bf16 keys 494 us and
//   2.3e-3 of error, 661 us and 1.65e-3 (the output's rounding) with the rest; 2 x 1024 on 24-32 k
//   e4m3 keys, f16 queries, 531 us and 2.5e-4, 717 us and 2.1e-4 with it.
//   Scores, maxima, sums and O stay in f32.
#pragma once

#include <algorithm>
#include <cmath>

#include "attn_common.hpp"
#include "common.hpp"
#include "paged_map.hpp"

namespace sm {
namespace {

struct PagedArgs {
  const uint8_t *k, *v;          // cache pages
  const uint8_t *ks, *vs;        // block scales (8-bit cache)
  const uint16_t* q;
  const int32_t *table, *pos0, *row_start;
  void* out;
  float* lse;
  float *part_o, *part_ml;       // per (row, head, split): unnormalised O; (max, sum)
  int64_t ldq;
  PagedMap map;                  // of paged_tile_kernel
  Divide H, KVH, G, bpp, nsplit, tiles, rows_each, tile, seqs;
  int S, rows, max_rows, pages, cols, cb;
  int most;                      // blocks that a table row holds, and one
  const uint32_t* mask;          // tree form: [rows, words], who sees which of its sequence's rows
  int words;
  int share;                     // splits of all sequences together; 0: nsplit each
  int32_t* counts;               // [S], the splits that each sequence was given
  float c2;                      // log2(e) / sqrt(hd)
};

// The keys that a row sees: those up to its own position, or, in the tree form, those before the
// sequence's rows (its context) and of the rows' own keys pos0 .. those with their bit set. The
// words are read in the last blocks or tiles of the keys alone, which are the only ones that have such keys;
// held in registers from the start they make the tile kernel spill (47 -> 640 us). The form costs what
// the causal one does: 32 x 24 rows on 1-4 k e4m3 keys 49-51 us both, 2 x 48-64 rows on 90-131 k 134-147 beside
// 130-142; ragged trees of up to 63 rows, 16 heads of their own, bf16, 54 beside 50.
template <bool TREE>
struct Sees {
  int last;
  __device__ inline Sees() {}
  __device__ inline Sees(const PagedArgs&, const PagedRows&, int pos0, int row)
      : last(pos0 + row) {}
  __device__ inline bool operator()(int key) const { return key <= last; }
  __device__ inline bool none() const { return last < 0; }
};
template <>
struct Sees<true> {
  const uint32_t* m;  // the row's words
  int n, pos0;        // bits that count
  __device__ inline Sees() {}
  __device__ inline Sees(const PagedArgs& a, const PagedRows& pr, int pos0_, int row)
      : m(a.mask + (int64_t)(pr.first + row) * a.words), n(min(pr.n, 32 * a.words)), pos0(pos0_) {}
  __device__ inline uint32_t at(int w) const {
    if (w < 0) return ~0u;
    if (32 * w >= n) return 0u;
    return n - 32 * w >= 32 ? m[w] : m[w] & ((1u << (n - 32 * w)) - 1);
  }
  // keys key .. key + 31, a bit each
  __device__ inline uint32_t bits(int key) const {
    const int rel = key - pos0;
    return (uint32_t)((((uint64_t)at((rel >> 5) + 1) << 32) | at(rel >> 5)) >> (rel & 31));
  }
  __device__ inline bool operator()(int key) const { return bits(key) & 1; }
  __device__ inline bool none() const {
    if (pos0 > 0) return false;
    for (int key = 0; key < pos0 + n; key += 32)
      if (bits(key)) return false;
    return true;
  }
};

// Whether row `row` < pr.n sees no key at all.
template <bool TREE>
__device__ inline bool no_keys(const PagedArgs& a, const PagedRows& pr, int pos0, int row) {
  if (pos0 > 0) return false;
  return Sees<TREE>(a, pr, pos0, row).none();
}

// Split j of all the sequences' together, in the tree form: its calls are few rows on contexts that
// differ, and the splits are as long as gives `share` of them, so that all units end together.
// Every wave finds the length for itself, a sequence a lane (the bounds are close: one to three steps),
// and then the sequence of j. 16 trees of 16 rows on 0.5-30 k e4m3 keys 93 us, 122 with the longest
// sequence's splits for all; 32 x 4 rows on 1-4 k bf16 37 and 44; 17 ragged trees, 16 heads of their own,
// 54 and 60; 2 x 48-64 rows on 90-131 k 139 and 142. Where all are alike, the lengths that the first loads
// wait for cost 2-3 us: 32 x 24 rows on 4000 keys 53.5 and 51.
constexpr int kShared = 256;  // sequences at most
struct TreeSplit {
  int s, split, splits, cb;  // s < 0: there is no such split
  __device__ inline TreeSplit(const PagedArgs& a, int j) : s(-1), split(0), splits(1), cb(kUnit) {
    const int lane = threadIdx.x % kWave;
    constexpr int N = kShared / kWave;
    uint32_t units[N];
    float all = 0.f;
#pragma unroll
    for (int c = 0; c < N; ++c) {
      units[c] = 0;
      const int q = c * kWave + lane;
      if (c * kWave < a.S && q < a.S) {
        const PagedRows pr(a.row_start, q, a.rows, a.max_rows);
        // (PagedKeys' of all of the sequence's rows)
        const int64_t keys = pr.n > 0 ? (int64_t)a.pos0[q] + pr.n : 0;
        const int64_t held = min((int64_t)a.most * kBlock, (int64_t)0x7fffffff);
        units[c] = keys <= 0 ? 0 : ((uint32_t)min(keys, held) - 1) / (kBlock * kUnit) + 1;
      }
      all += (float)units[c];
    }
    all = wave_sum(all);
    int lo, hi;
    PagedShare::bounds(all, a.S, a.share, lo, hi);
    while (lo < hi) {  // (uniform)
      const int mid = lo + (hi - lo) / 2;
      float n = 0.f;
#pragma unroll
      for (int c = 0; c < N; ++c)
        if (c * kWave < a.S && c * kWave + lane < a.S)
          n += (float)PagedShare::most(units[c], mid, a.nsplit.d);
      if (wave_sum(n) <= (float)a.share) hi = mid;
      else lo = mid + 1;
    }
    int before = 0;
#pragma unroll
    for (int c = 0; c < N; ++c) {
      if (s >= 0 || c * kWave >= a.S) continue;  // (uniform)
      const PagedShare ps(units[c], lo, a.nsplit.d);
      const int n = c * kWave + lane < a.S ? ps.splits : 0;
      int end = n;  // sums up to and with this lane's: in rows of 16 lanes, then of the rows
      end += __builtin_amdgcn_update_dpp(0, end, 0x111, 0xF, 0xF, false);  // row_shr 1, 2, 4, 8
      end += __builtin_amdgcn_update_dpp(0, end, 0x112, 0xF, 0xF, false);
      end += __builtin_amdgcn_update_dpp(0, end, 0x114, 0xF, 0xF, false);
      end += __builtin_amdgcn_update_dpp(0, end, 0x118, 0xF, 0xF, false);
      const int r0 = __builtin_amdgcn_readlane(end, 15), r1 = __builtin_amdgcn_readlane(end, 31),
                r2 = __builtin_amdgcn_readlane(end, 47);
      end += lane >= 48 ? r0 + r1 + r2 : lane >= 32 ? r0 + r1 : lane >= 16 ? r0 : 0;
      const uint64_t at = __ballot(j - before < end);
      if (at) {
        const int l = (int)__builtin_ctzll(at);
        s = c * kWave + l;
        splits = __builtin_amdgcn_readlane(n, l);
        split = j - before - (__builtin_amdgcn_readlane(end, l) - splits);
        cb = __builtin_amdgcn_readlane(ps.cb, l);
      }
      before += __builtin_amdgcn_readlane(end, kWave - 1);
    }
  }
};

// Four / eight cache codes of one packed word -> the MFMA operand's 16-bit values.
typedef __bf16 b2 __attribute__((ext_vector_type(2)));
template <bool F16>
__device__ inline uint32_t cvt2(uint32_t w, bool hi) {
  if constexpr (F16)
    return hi ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, true))
              : __builtin_bit_cast(uint32_t,
                                   __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, false));
  else
    return hi ? __builtin_bit_cast(uint32_t,
                                   __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, true))
              : __builtin_bit_cast(uint32_t,
                                   __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, false));
}
template <bool F16>
__device__ inline u32x4 cvt8(uint32_t a, uint32_t b) {
  return u32x4{cvt2<F16>(a, false), cvt2<F16>(a, true), cvt2<F16>(b, false), cvt2<F16>(b, true)};
}

template <bool F16>
__device__ inline f4 mfma16(u32x4 a, u32x4 b, f4 c) {
  return Op8<F16>::mfma(__builtin_bit_cast(typename Op8<F16>::T, a),
                        __builtin_bit_cast(typename Op8<F16>::T, b), c);
}
// log2 of what the largest weight is where the reference is raised, and of what it may reach
// before the next time. (2 x 1024 rows on 24-32 k keys 536 us, prefill of 32 prompts 50.7; with
// 0 and 8 532 and 49.3, with 7 and 15 533 and 49.5, with 13 and 15 539 and 50.9, each with its
// share of weights lost.) bf16 weights have f32's range and stay at 1, for sums of large values.
__device__ constexpr float kWeight(bool f16) { return f16 ? 11.f : 0.f; }
__device__ constexpr float kWeightMost(bool f16) { return f16 ? 15.f : 8.f; }

constexpr int kScaleSmall = 17;  // (8-bit) values up to 5.9e7 need no care in the sum
__device__ constexpr float kSumShift(bool c8) { return c8 ? 20.f : 0.f; }
// Factor of a block's sum of P' in the sum of weights; zero: taken of the scores. (A block behind
// the last key may have any scale byte: its P' are zero, the factor has to be finite.)
template <bool C8>
__device__ inline float sum_factor(float vexp, bool large) {
  return !C8 ? 1.f : large ? 0.f : __builtin_amdgcn_exp2f(fminf(kSumShift(true) - vexp, 100.f));
}
// log2 and reciprocal of a sum that is held up
template <bool C8>
__device__ inline float sum_log2(float m, float l) {
  return m + ((float)__builtin_amdgcn_frexp_expf(l) - kSumShift(C8)) +
         __log2f(__builtin_amdgcn_frexp_mantf(l));
}
template <bool C8>
__device__ inline float sum_inverse(float l) {
  return (C8 ? 1048576.f : 1.f) / l;
}
static_assert(kSumShift(true) == 20.f, "2^20 is sum_inverse's");

template <bool F16>
__device__ inline uint32_t pack2(float a, float b) {
  if constexpr (F16) {
    const f32x2_t v = {a, b};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, h2));
  } else {
    return pack_bf16x2(a, b);
  }
}

// A word of cache values with its infinities and NaN set to zero.
template <bool C8, bool F16>
__device__ inline uint32_t finite_only(uint32_t w) {
  if constexpr (C8) {  // e4m3 has no infinity; NaN is 0x7f or 0xff
    const uint32_t x = ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
    return w & ~((x >> 7) * 0xffu);
  } else {
    constexpr uint32_t m = F16 ? 0x7c00u : 0x7f80u;
    if ((w & m) == m) w &= 0xffff0000u;
    if ((w >> 16 & m) == m) w &= 0x0000ffffu;
    return w;
  }
}

// Values that are not finite. Those that some of a tile's rows see and some do not are kept
// out of the products (a weight of zero would turn an infinity into a NaN for the rows that
// do not see it); those that all see go in, and in 16 bits leave a NaN where a weight, or
// what its rounding leaves, is zero. So where there are any, each row's sums are put right
// after the sweep: a weight is positive, however small, and one infinity or NaN decides a sum.
//
// Blocks first, first + 1, .. below end, 64 at most, that have such values and are the
// caller's: mine(block).
template <int HD, bool C8, bool F16, typename Mine>
__device__ inline uint64_t odd_blocks(const PagedArgs& a, const int32_t* trow, int kvh, int first,
                                      int end, int lane, Mine mine) {
  constexpr int BB = kBlock * HD * (C8 ? 1 : 2);
  uint64_t mask = 0;
  for (int i = 0; i < min(kWave, end - first); ++i) {
    if (!mine(first + i)) continue;
    const int bi = paged_block(trow, a.cols, a.pages, (int)a.KVH.d, kvh, a.bpp, first + i);
    if (bi < 0) continue;
    bool odd = false;
#pragma unroll
    for (int c = 0; c < BB / 1024; ++c) {
      const u32x4 w = *reinterpret_cast<const u32x4*>(a.v + (size_t)bi * BB + c * 1024 + lane * 16);
#pragma unroll
      for (int k = 0; k < 4; ++k) odd |= finite_only<C8, F16>(w[k]) != w[k];
    }
    if (__ballot(odd)) mask |= (uint64_t)1 << i;
  }
  return mask;
}
// sum[i], of dim(i): what the blocks of `mask` have that is not finite and this lane's row
// sees, in place of the sum at first (its bit of `done` is clear), with it from then on.
template <int HD, bool C8, bool F16, bool TREE, int N, typename Dim>
__device__ inline void fix_odd(const PagedArgs& a, const int32_t* trow, int kvh, int first,
                               uint64_t mask, int keys, Sees<TREE> sees, Dim dim, uint32_t& done,
                               int bit, float (&sum)[N]) {
  constexpr int T = C8 ? 4 : 2;
  float x[N];
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = 0.f;
  for (; mask; mask &= mask - 1) {
    const int blk = first + __builtin_ctzll(mask);
    const int bi = paged_block(trow, a.cols, a.pages, (int)a.KVH.d, kvh, a.bpp, blk);
    const size_t base = (size_t)bi * (kBlock * HD);
    for (int t = 0; t < kBlock; ++t) {
      const int key = blk * kBlock + t;
      if (key >= keys) break;
      const bool see = sees(key);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int d = dim(i), n = d / 16;
        const size_t at = base + ((n / T * 4 + t / 4) * 16 + d % 16) * (4 * T) + n % T * 4 + t % 4;
        float v;
        if constexpr (C8) {
          v = (a.v[at] & 0x7f) == 0x7f ? NAN : 0.f;
        } else {
          const uint16_t w = reinterpret_cast<const uint16_t*>(a.v)[at];
          v = F16 ? (float)__builtin_bit_cast(_Float16, w) : bf16_to_f32(w);
          if (fabsf(v) < INFINITY) v = 0.f;
        }
        if (see) x[i] += v;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (!(x[i] == 0.f)) {
      sum[i] = done >> (bit + i) & 1 ? sum[i] + x[i] : x[i];
      done |= 1u << (bit + i);
    }
}

// Partial sums (m, l, o) of one row join as sum l f and sum o f, f = 2^(m - mm) with the largest
// m of them: half of f's exponent is kept, so that l, which scales may hold far up or down, is
// multiplied by two factors that f32 holds. Without keys (m -inf, l 0) it is zero.
struct Join {
  float half;
  __device__ inline Join(float m, float l, float mm)
      : half(m == -INFINITY ? (l == 0.f ? 0.f : NAN) : __builtin_amdgcn_exp2f(0.5f * (m - mm))) {}
  __device__ inline float sum(float l) const { return l * half * half; }
  __device__ inline float weight() const { return half * half; }
};
// A part of O times its weight; one that is not finite stays what it is, as a weight is positive.
__device__ inline float join_o(float o, float weight, float acc) {
  return fabsf(o) < INFINITY ? fmaf(o, weight, acc) : acc + o;
}

// Where 64 blocks of a sequence lie, one to a lane, and their scales.
struct Blocks {
  int at;       // cache block; 0 where there is none
  bool none;
  int ke, ve;   // scale bytes (8-bit cache)
  __device__ inline void find(const PagedArgs& a, const int32_t* trow, int kvh, int blk) {
    const int b = paged_block(trow, a.cols, a.pages, (int)a.KVH.d, kvh, a.bpp, blk);
    none = b < 0;
    at = none ? 0 : b;
    if (a.ks) {  // (uniform)
      ke = a.ks[at];
      ve = a.vs[at];
    }
  }
  // factor of a score in units of log2, NaN without a block; exponent of V's scale
  template <bool C8>
  __device__ inline float kscale(float c2) const {
    return none ? NAN : C8 ? __builtin_amdgcn_ldexpf(c2, ke - 127) : c2;
  }
  template <bool C8>
  __device__ inline float vexp() const {
    return C8 ? (float)(ve - 127) : 0.f;
  }
  // Whether any of the first n of these blocks has a scale above 2^kScaleSmall (uniform).
  template <bool C8>
  __device__ inline bool large(int n) const {
    return C8 && __ballot((int)(threadIdx.x % kWave) < n && !none && ve > 127 + kScaleSmall) != 0;
  }
};

// ---- up to 16 query rows a KV head: bound by reading K and V ----
//
// One workgroup per (split of the keys, KV head, sequence). Its four waves take steps of two
// 16-key blocks in turn and meet in LDS at the end. K and V go from memory into the registers
// as the matrix cores take them, 16 bytes a lane and load; 8-bit codes are converted there
// (one instruction for two). v_mfma_f32_16x16x32: a score tile is 16 keys x 16 rows.
// 256 sequences of 512-1023 tokens, 16 / 4 heads of 128, e4m3 (202 MB): 42 us, 4.8 TB/s; 4 of
// 100-131 k (483 MB): 96-98 us, 5.0; 48 x 4 rows of 1-4 k, 16 heads, bf16 (1.08 GB): 206-216 us,
// 5.0-5.3, where a copy on this card moves 4.8. Two blocks a step beside four: the same time with 40
// registers fewer; four workgroups a unit (128 registers): no faster.
constexpr int kRows16 = 16;  // query rows of a workgroup

template <int HD, bool QF16, bool C8, bool TREE>
__global__ __launch_bounds__(256, 2) void paged_split_kernel(PagedArgs a) {
  constexpr int ES = C8 ? 1 : 2;
  constexpr bool PF16 = C8 || QF16;   // type of P and V in P.V
  constexpr int NB = 2;               // blocks a wave takes at a time
  constexpr int NC = HD * ES / 64;    // 16-byte loads a lane makes of a block of K, and of V
  constexpr int NT = HD / 16;         // 16-dim tiles of O
  constexpr int BB = kBlock * HD * ES;  // bytes of a block
  __shared__ float sm_m[4][kRows16], sm_l[4][kRows16];
  __shared__ __attribute__((aligned(16))) float sm_o[4][kRows16][HD + 4];

  int s = (int)blockIdx.x, split, kvh, tile, cb = a.cb, most_splits = (int)a.nsplit.d;
  if (TREE && a.share) {  // (uniform)
    kvh = a.KVH.mod(s);
    tile = a.tiles.mod(s);
    const TreeSplit ts(a, s);
    if (ts.s < 0) return;
    s = ts.s;
    split = ts.split;
    cb = ts.cb;
    most_splits = ts.splits;
    if (split + kvh + tile == 0 && threadIdx.x == 0) a.counts[s] = most_splits;
  } else {
    split = a.nsplit.mod(s);
    kvh = a.KVH.mod(s);
    tile = a.tiles.mod(s);
  }
  // What the first loads need does not wait for the sequence's lengths: a workgroup without
  // work goes through them too (its rows and table row are there) and leaves after the loop.
  const int32_t* trow = a.table + (int64_t)s * a.cols;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x % kWave;
  const int r = lane % 16, g = lane / 16;
  Blocks cur, next;
  cur.find(a, trow, kvh, split * cb + lane);
  const PagedRows pr(a.row_start, s, a.rows, a.max_rows);
  const int pos0 = a.pos0[s];
  const int row0 = tile * kRows16, all = pr.n * (int)a.G.d;
  const PagedKeys pk(pos0, pr.n, a.G, TREE ? 0 : row0, TREE ? all : kRows16, cb, most_splits,
                     a.most);
  const bool idle = row0 >= all || split >= max(pk.splits, 1);
  const int b0 = split * cb, b1 = idle || pk.keys <= 0 ? b0 : pk.end(split, cb);

  // this lane's query: row row0 + r
  const int qr = max(0, min(row0 + r, all - 1));
  const int qt = a.G.div(qr);
  const Sees<TREE> sees(a, pr, pos0, qt);
  const int pos_first = TREE ? pos0 - 1 : pos0 + a.G.div(row0);  // the tile's rows all see up to it
  u32x4 qf[HD / 32];
  {
    const uint16_t* qp = a.q + (idle ? 0 : (int64_t)(pr.first + qt) * a.ldq) +
                         (int64_t)(kvh * (int)a.G.d + qr - qt * (int)a.G.d) * HD;
#pragma unroll
    for (int c = 0; c < HD / 32; ++c) {
      const int d = C8 ? (c / 2) * 64 + g * 16 + (c % 2) * 8 : c * 32 + g * 8;
      qf[c] = *reinterpret_cast<const u32x4*>(qp + d);
    }
  }
  f4 o[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) o[n] = f4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;
  bool odd = false;    // values that are not finite, among keys that not all rows see
  bool large = false;  // scales of V above 2^kScaleSmall, up to here

  for (int seg = b0; seg < b1; seg += kWave, cur = next) {
    const int nb = min(kWave, b1 - seg);
    if (seg + kWave < b1) next.find(a, trow, kvh, seg + kWave + lane);
    large |= cur.template large<C8>(nb);
    for (int st = wave * NB; st < nb; st += 4 * NB) {
      u32x4 kr[NB][NC], vr[NB][NC];
      float ksc[NB], vex[NB], lf[NB];
#pragma unroll
      for (int u = 0; u < NB; ++u) {
        const size_t at = (size_t)__builtin_amdgcn_readlane(cur.at, min(st + u, nb - 1)) * BB;
#pragma unroll
        for (int c = 0; c < NC; ++c)
          kr[u][c] = *reinterpret_cast<const u32x4*>(a.k + at + r * HD * ES + c * 64 + g * 16);
#pragma unroll
        for (int c = 0; c < NC; ++c)
          vr[u][c] = *reinterpret_cast<const u32x4*>(a.v + at + c * 1024 + lane * 16);
      }
      __builtin_amdgcn_sched_barrier(0);  // (the scales are waited for behind these loads)
      const float kscale = cur.template kscale<C8>(a.c2), vexp = cur.template vexp<C8>();
      const float factor = sum_factor<C8>(vexp, large);
#pragma unroll
      for (int u = 0; u < NB; ++u) {
        ksc[u] = lane_f32(kscale, min(st + u, nb - 1));
        vex[u] = lane_f32(vexp, min(st + u, nb - 1));
        lf[u] = lane_f32(factor, min(st + u, nb - 1));
      }
      // scores, in units of log2 and raised by the exponent of V's scale
      float t[NB][4];
      float mx = -INFINITY;
#pragma unroll
      for (int u = 0; u < NB; ++u) {
        f4 sc = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          if constexpr (C8) {
            sc = mfma16<QF16>(cvt8<QF16>(kr[u][c].x, kr[u][c].y), qf[2 * c], sc);
            sc = mfma16<QF16>(cvt8<QF16>(kr[u][c].z, kr[u][c].w), qf[2 * c + 1], sc);
          } else {
            sc = mfma16<QF16>(kr[u][c], qf[c], sc);
          }
        }
        const int key0 = (seg + st + u) * kBlock;
        uint32_t see = ~0u;  // tree form: this lane's four keys
        if constexpr (TREE) {
          if (key0 + kBlock > pos0) see = sees.bits(key0 + 4 * g);  // (uniform)
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          t[u][i] = C8 ? fmaf(sc[i], ksc[u], vex[u]) : sc[i] * ksc[u];
          if constexpr (TREE) {
            if (!(see >> i & 1) || st + u >= nb) t[u][i] = -INFINITY;
          } else {
            if (key0 + 4 * g + i > sees.last || st + u >= nb) t[u][i] = -INFINITY;
          }
          mx = fmaxf(mx, t[u][i]);
        }
        // values past the tile's last key are not the cache's: no product sees them
        if (key0 + kBlock > pk.keys || st + u >= nb || ksc[u] != ksc[u]) {
          const int have = st + u >= nb || ksc[u] != ksc[u]
                               ? 0 : max(0, min(4, pk.keys - key0 - 4 * g));
          if constexpr (C8) {
            const uint32_t keep = have >= 4 ? ~0u : (1u << (8 * have)) - 1;
#pragma unroll
            for (int c = 0; c < NC; ++c) vr[u][c] &= keep;
          } else {
            const uint32_t k01 = have >= 2 ? ~0u : have == 1 ? 0xffffu : 0u;
            const uint32_t k23 = have >= 4 ? ~0u : have == 3 ? 0xffffu : 0u;
#pragma unroll
            for (int c = 0; c < NC; ++c) vr[u][c] &= u32x4{k01, k23, k01, k23};
          }
        }
        if (key0 + kBlock - 1 > pos_first && pos_first + 1 < pk.keys) {
          bool x = false;
#pragma unroll
          for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t y = finite_only<C8, QF16>(vr[u][c][i]);
              x |= y != vr[u][c][i];
              vr[u][c][i] = y;
            }
          odd |= __ballot(x) != 0;
        }
      }
      if (__ballot(mx > m + kWeightMost(PF16))) {
        mx = fmaxf(mx, __shfl_xor(mx, 16, kWave));
        mx = fmaxf(mx, __shfl_xor(mx, 32, kWave));
        const float mn = fmaxf(m, mx - kWeight(PF16));
        const Join j(m, l, mn);
        m = mn;
        l = j.sum(l);
#pragma unroll
        for (int n = 0; n < NT; ++n) o[n] *= j.weight();
      }
      const float ms = m == -INFINITY ? 0.f : m;
      if (C8 && large) {  // (uniform)
#pragma unroll
        for (int u = 0; u < NB; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            l += __builtin_amdgcn_exp2f(t[u][i] - vex[u] - (ms - kSumShift(C8)));
      }
      u32x4 p[NB / 2], rest[NB / 2];  // rest: what 16 bits leave of the weights
#pragma unroll
      for (int u = 0; u < NB; ++u) {
        float e[4], sum;
#pragma unroll
        for (int i = 0; i < 4; ++i) e[i] = __builtin_amdgcn_exp2f(t[u][i] - ms);
        sum = (e[0] + e[1]) + (e[2] + e[3]);
        l = C8 ? fmaf(sum, lf[u], l) : l + sum;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t w = pack2<PF16>(e[2 * i], e[2 * i + 1]);
          p[u / 2][2 * (u % 2) + i] = w;
          const float lo = PF16 ? (float)as_h2(w)[0] : bf16lo(w),
                      hi = PF16 ? (float)as_h2(w)[1] : bf16hi(w);
          rest[u / 2][2 * (u % 2) + i] = pack2<PF16>(e[2 * i] - lo, e[2 * i + 1] - hi);
        }
      }
#pragma unroll
      for (int w = 0; w < NB / 2; ++w) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          u32x4 va;
          if constexpr (C8) {
            va = cvt8<true>(vr[2 * w][n / 4][n % 4], vr[2 * w + 1][n / 4][n % 4]);
          } else {
            va = u32x4{vr[2 * w][n / 2][2 * (n % 2)], vr[2 * w][n / 2][2 * (n % 2) + 1],
                       vr[2 * w + 1][n / 2][2 * (n % 2)], vr[2 * w + 1][n / 2][2 * (n % 2) + 1]};
          }
          o[n] = mfma16<PF16>(va, p[w], o[n]);
          o[n] = mfma16<PF16>(va, rest[w], o[n]);
        }
      }
    }
  }
  l += __shfl_xor(l, 16, kWave);
  l += __shfl_xor(l, 32, kWave);
  bool all_see = false;  // values that are not finite among the others
  if constexpr (!C8) {   // (a code is finite or NaN, which any weight leaves a NaN)
    float zero = 0.f;
#pragma unroll
    for (int i = 0; i < 4 * NT; ++i) zero = fmaf(o[i / 4][i % 4], 0.f, zero);
    all_see = __ballot(zero != zero && l == l) != 0;
  }
  if (odd || all_see) {  // (uniform per wave)
    uint32_t done = 0;
    for (int seg = all_see ? b0 : max(b0, (pos_first + 1) / kBlock); seg < b1; seg += kWave) {
      const uint64_t mask = odd_blocks<HD, C8, QF16>(
          a, trow, kvh, seg, b1, lane, [&](int blk) { return (blk - b0) % (4 * NB) / NB == wave; });
      if (!mask) continue;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float x[4] = {o[n][0], o[n][1], o[n][2], o[n][3]};
        fix_odd<HD, C8, QF16>(a, trow, kvh, seg, mask, pk.keys, sees,
                              [&](int i) { return 16 * n + 4 * g + i; }, done, 4 * n, x);
#pragma unroll
        for (int i = 0; i < 4; ++i) o[n][i] = x[i];
      }
    }
  }
  if (idle) return;  // (uniform)
  if (g == 0) {
    sm_m[wave][r] = m;
    sm_l[wave][r] = l;
  }
#pragma unroll
  for (int n = 0; n < NT; ++n) *reinterpret_cast<f4*>(&sm_o[wave][r][16 * n + 4 * g]) = o[n];
  __syncthreads();

  // row threadIdx.x / 16, HD / 16 of its dims
  const int y = threadIdx.x / 16, d0 = (threadIdx.x % 16) * (HD / 16);
  if (row0 + y >= all) return;
  int tok = row0 + y;
  const int head = kvh * (int)a.G.d + a.G.mod(tok);
  float mm = sm_m[0][y];
#pragma unroll
  for (int w = 1; w < 4; ++w) mm = fmaxf(mm, sm_m[w][y]);
  float ll = 0.f, f[4];
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const Join j(sm_m[w][y], sm_l[w][y], mm);
    f[w] = j.weight();
    ll += j.sum(sm_l[w][y]);
  }
  float acc[HD / 16];
#pragma unroll
  for (int i = 0; i < HD / 16; ++i) {
    acc[i] = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) acc[i] = join_o(sm_o[w][y][d0 + i], f[w], acc[i]);
  }
  const size_t at = (size_t)(pr.first + tok) * a.H.d + head;
  if (pk.splits > 1) {
    float* po = a.part_o + (at * a.nsplit.d + split) * HD + d0;
#pragma unroll
    for (int i = 0; i < HD / 16; i += 4)
      *reinterpret_cast<f4*>(po + i) = f4{acc[i], acc[i + 1], acc[i + 2], acc[i + 3]};
    if (d0 == 0)
      *reinterpret_cast<float2*>(a.part_ml + (at * a.nsplit.d + split) * 2) = float2{mm, ll};
    return;
  }
  const bool none = no_keys<TREE>(a, pr, pos0, tok);
  const float inv = sum_inverse<C8>(ll);
  uint32_t w2[HD / 32];
#pragma unroll
  for (int i = 0; i < HD / 32; ++i)
    w2[i] = none ? 0u : pack2<QF16>(acc[2 * i] * inv, acc[2 * i + 1] * inv);
  uint32_t* op = reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.out) + at * HD + d0);
#pragma unroll
  for (int i = 0; i < HD / 32; ++i) op[i] = w2[i];
  if (a.lse && d0 == 0)
    a.lse[at] = none ? -INFINITY : sum_log2<C8>(mm, ll) * 0.69314718055994530942f;
}

// ---- more query rows: 128 of them a workgroup, keys staged through LDS ----
//
// Four or eight waves x 32 rows (v_mfma_f32_32x32x16), two waves a SIMD. A tile of 64 keys, in
// 16 bits, sits in one of two LDS buffers; the next tiles' loads are on their way during this
// one's products and are converted and stored before the barrier that ends it.
// 2 x 1024 tokens on 24-32 k keys, 16 / 4 heads of 128, f16 queries, e4m3 (eight waves): 0.51-0.53
// ms from card to card, 0.98-1.02 PF/s, 84 % of what a large f16 product reaches; the clock is
// down to 1.88 GHz, the matrix cores work 46 % and the vector units 48 % of the cycles. With V
// scales above 2^kScaleSmall, whose sum has exponentials of its own, 491 us where it is 434
// (1024 rows on 28 k keys).
// Of four waves' 563 us, staging took 91, the barriers 10, the exponentials 44, the sums 16.
// Prefill of 32 prompts of 257-512 (four waves): 50 us: 1.75 us a tile and 5.6 us a workgroup
// for two round trips to memory and its output.
// bf16 cache: 2 x 1024 tokens on 28 k keys 484-497 us (0.97 PF/s), 16 x 512 on 2 k 192 (0.81); f16
// cache: 8 x 512 on 4 k 163 (0.90), e4m3 there 154. Heads of 64, where a product has half the
// work beside the same softmax: 8 x 1024 on 1 k, 12 heads, bf16 71 us (0.55), e4m3 66.
// Tried and slower: scores of the next tile beside this one's softmax on 32-key tiles (670
// beside 637 us at the time), three workgroups a unit (618 beside 583), two and four times the
// splits (the join's bytes), workgroups that go on to further row tiles with their first loads
// in flight (prefill 65 beside 50 us), half a last tile left out (spills), output and query
// rows kept out of the L2 (60 beside 53; the output alone: the same).

typedef float f32x16 __attribute__((ext_vector_type(16)));
template <bool F16>
__device__ inline f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, a),
                                                  __builtin_bit_cast(h8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf8, a),
                                                   __builtin_bit_cast(bf8, b), c, 0, 0, 0);
}

// (fmaxf of values behind a branch costs the compiler's quieting of each)
__device__ inline float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

constexpr int kTile = 64;  // keys of a tile

template <int HD, bool QF16, bool C8, bool TREE, int W>  // W waves, 32 query rows each
struct TileSweep {
  static constexpr int ES = C8 ? 1 : 2;
  static constexpr bool PF16 = C8 || QF16;
  static constexpr int KS = HD / 16, DB = HD / 32;  // MFMA steps of a score, 32-dim blocks of O
  static constexpr int KP = HD + 8, VP = kTile + 8; // padded LDS rows (elements)
  static constexpr int NB = kTile / kBlock;         // blocks of a tile
  static constexpr int NC = HD * ES / 64;           // kilobytes of a block, each one wave's load
  static constexpr int PER = (NB * NC + W - 1) / W; // of a tile's K, and of its V, for each wave
  static constexpr int BB = kBlock * HD * ES;
  struct Lds {
    __attribute__((aligned(16))) uint16_t ks[2][kTile * KP];
    __attribute__((aligned(16))) uint16_t vts[2][HD * VP];
    // a block's score factor, V exponent and factor of its weights' sum
    __attribute__((aligned(16))) float info[2][NB][4];
    int odd;
  };

  const PagedArgs& a;
  Lds& s;
  const int32_t* trow;
  const uint16_t* qp;  // this lane's query row
  int kvh, b0, b1, keys, pos_first, wave_first, wave_last, wave, lane, j, hf;
  Sees<TREE> sees;
  u32x4 qa[KS];
  f32x16 o[DB];  // o[d][e]: row j, dim 32 d + 8 (e / 4) + 4 hf + e % 4
  float m, l;

  Blocks cur, next;  // of the 64 blocks at hand, and of the next
  bool missing;      // any of those at hand has keys and no page
  bool large;        // scales of V above 2^kScaleSmall, up to those at hand
  u32x4 kr[PER], vr[PER];

  __device__ TileSweep(const PagedArgs& a_, Lds& s_) : a(a_), s(s_) {}

  // The n-th kilobyte that this wave stages of a tile's K and V: whose block, and which of it.
  __device__ inline bool part(int n, int& block, int& c) const {
    const int x = wave * PER + n;
    block = x / NC;
    c = x % NC;
    return W * PER == NB * NC || x < NB * NC;
  }
  __device__ inline void load_tile(int blk) {  // first block of the tile
#pragma unroll
    for (int n = 0; n < PER; ++n) {
      int block, c;
      if (!part(n, block, c)) continue;
      const size_t at =
          (size_t)__builtin_amdgcn_readlane(cur.at, (blk - b0 + block) % kWave) * BB + c * 1024;
      kr[n] = *reinterpret_cast<const u32x4*>(a.k + at + lane * 16);
      vr[n] = *reinterpret_cast<const u32x4*>(a.v + at + lane * 16);
    }
  }
  // Whether blocks with keys have no page, of the 64 from `first` on (uniform).
  __device__ inline bool any_missing(const Blocks& of, int first) const {
    return __ballot(of.none && (first + lane) * kBlock < keys) != 0;
  }
  // `cur` is the 64 blocks from `first` on.
  __device__ inline void at_hand(int first) {
    missing = any_missing(cur, first);
    large |= cur.template large<C8>(b1 - first);
  }
  // Values that are not the cache's, or that only some rows see, out of what is staged.
  __device__ inline void mask_tile(int blk, const Blocks& of) {
    const int g = lane / 16;
    const float kscale = of.template kscale<C8>(a.c2);
#pragma unroll
    for (int n = 0; n < PER; ++n) {
      int block, c;
      if (!part(n, block, c)) continue;
      const int key0 = (blk + block) * kBlock;
      const float kf = lane_f32(kscale, (blk - b0 + block) % kWave);
      if (key0 + kBlock > keys || kf != kf) {  // not the cache's: no product sees them
        const int have = kf != kf ? 0 : max(0, min(4, keys - key0 - 4 * g));
        if constexpr (C8) {
          vr[n] &= have >= 4 ? ~0u : (1u << (8 * have)) - 1;
        } else {
          const uint32_t k01 = have >= 2 ? ~0u : have == 1 ? 0xffffu : 0u;
          const uint32_t k23 = have >= 4 ? ~0u : have == 3 ? 0xffffu : 0u;
          vr[n] &= u32x4{k01, k23, k01, k23};
        }
      }
      if (key0 + kBlock - 1 > pos_first) {  // some rows see these keys and some do not
        bool x = false;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t y = finite_only<C8, QF16>(vr[n][i]);
          x |= y != vr[n][i];
          vr[n][i] = y;
        }
        if (x) s.odd = 1;
      }
    }
  }
  __device__ inline void store_tile(int blk, int buf, const Blocks& of) {
    const int g = lane / 16, r = lane % 16;
    if (missing || (blk + NB) * kBlock > min(keys, pos_first + 1)) mask_tile(blk, of);
    const float kscale = of.template kscale<C8>(a.c2), vexp = of.template vexp<C8>();
#pragma unroll
    for (int n = 0; n < PER; ++n) {
      int block, c;
      if (!part(n, block, c)) continue;
      const int at = (c * 64 + lane) * (16 / ES);  // element of the block
      uint16_t* kp = &s.ks[buf][(block * kBlock + at / HD) * KP + at % HD];
      if constexpr (C8) {
        *reinterpret_cast<u32x4*>(kp) = cvt8<QF16>(kr[n].x, kr[n].y);
        *reinterpret_cast<u32x4*>(kp + 8) = cvt8<QF16>(kr[n].z, kr[n].w);
      } else {
        *reinterpret_cast<u32x4*>(kp) = kr[n];
      }
      // quads of a block in the order 0, 2, 1, 3: the order in which a lane of the
      // transposed score tile holds its keys
      uint16_t* vp = &s.vts[buf][r * VP + block * kBlock + (g % 2 * 2 + g / 2) * 4];
#pragma unroll
      for (int t = 0; t < 4 / ES; ++t) {
        u32x2 w;
        if constexpr (C8) w = u32x2{cvt2<true>(vr[n][t], false), cvt2<true>(vr[n][t], true)};
        else w = u32x2{vr[n][2 * t], vr[n][2 * t + 1]};
        *reinterpret_cast<u32x2*>(vp + (c * (4 / ES) + t) * 16 * VP) = w;
      }
    }
    // (wave 0's lanes that hold the tile's blocks)
    const unsigned i = (unsigned)(threadIdx.x - (blk - b0) % kWave);
    if (i < NB)
      *reinterpret_cast<f4*>(s.info[buf][i]) = f4{kscale, vexp, sum_factor<C8>(vexp, large), 0.f};
  }

  // The next tile, on its way, to LDS, and the one after it on its way.
  __device__ inline void stage(int blk, int buf) {
    store_tile(blk + NB, buf, cur);  // last read before the previous barrier
    const int to = blk + 2 * NB;
    if (to >= b1) return;
    if ((to - b0) % kWave == 0) {
      cur = next;
      at_hand(to);
      if (to + kWave < b1) next.find(a, trow, kvh, to + kWave + lane);
    }
    load_tile(to);
  }
  // One pass over the keys.
  __device__ inline void sweep() {
#pragma unroll
    for (int st = 0; st < KS; ++st)
      qa[st] = *reinterpret_cast<const u32x4*>(qp + st * 16 + hf * 8);
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[d][e] = 0.f;
    m = -INFINITY;
    l = 0.f;
    if (b1 <= b0) return;
    if (threadIdx.x == 0) s.odd = 0;
    __syncthreads();
    load_tile(b0);
    large = false;
    at_hand(b0);
    store_tile(b0, 0, cur);
    __syncthreads();
    int buf = 0;
    if constexpr (W > 4) {
      // Half of the waves stage the next tile before this one's products and half after them,
      // so that the two waves of a SIMD are not in the same part of their work.
      const bool early = wave >= W / 2;
      if (b0 + kWave < b1) next.find(a, trow, kvh, b0 + kWave + lane);
      if (b0 + NB < b1) load_tile(b0 + NB);
      for (int blk = b0; blk < b1; blk += NB, buf ^= 1) {
        const bool more = blk + NB < b1;
        const int key0 = blk * kBlock;
        if (early && more) stage(blk, buf ^ 1);
        if (key0 <= wave_last) tile(buf, key0);  // (uniform per wave) later keys: no row sees them
        if (!early && more) stage(blk, buf ^ 1);
        __syncthreads();
      }
    } else {
      for (int blk = b0; blk < b1; blk += NB, buf ^= 1) {
        const bool more = blk + NB < b1;
        if ((blk - b0) % kWave == 0 && blk + kWave < b1)
          next.find(a, trow, kvh, blk + kWave + lane);
        if (more) {
          if ((blk + NB - b0) % kWave == 0) {
            cur = next;
            at_hand(blk + NB);
          }
          load_tile(blk + NB);
        }
        const int key0 = blk * kBlock;
        if (key0 <= wave_last) tile(buf, key0);
        if (more) store_tile(blk + NB, buf ^ 1, cur);  // last read before the previous barrier
        __syncthreads();
      }
    }
    // (the sums end here for the compiler: it copies them in every tile otherwise)
#pragma unroll
    for (int d = 0; d < DB; ++d) asm volatile("" : "+v"(o[d]));
    l += __shfl_xor(l, 32, kWave);
    bool all_see = false;  // (as in paged_split_kernel)
    if constexpr (!C8) {
      float zero = 0.f;
#pragma unroll
      for (int i = 0; i < 16 * DB; ++i) zero = fmaf(o[i / 16][i % 16], 0.f, zero);
      all_see = __ballot(zero != zero && l == l) != 0;
    }
    if (s.odd || all_see) {  // (uniform per wave)
      uint32_t done[(DB + 1) / 2] = {};
      for (int seg = all_see ? b0 : max(b0, (pos_first + 1) / kBlock); seg < b1; seg += kWave) {
        const uint64_t mask =
            odd_blocks<HD, C8, QF16>(a, trow, kvh, seg, b1, lane, [](int) { return true; });
        if (!mask) continue;
#pragma unroll
        for (int d = 0; d < DB; ++d) {
          float x[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) x[e] = o[d][e];
          fix_odd<HD, C8, QF16>(
              a, trow, kvh, seg, mask, keys, sees,
              [&](int e) { return 32 * d + 8 * (e / 4) + 4 * hf + e % 4; }, done[d / 2],
              d % 2 * 16, x);
#pragma unroll
          for (int e = 0; e < 16; ++e) o[d][e] = x[e];
        }
      }
    }
  }

  __device__ inline void tile(int buf, int key0) {
    f32x16 sc[kTile / 32];
    float kf[NB], vf[NB], lf[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const f4 x = *reinterpret_cast<const f4*>(s.info[buf][b]);
      kf[b] = x[0];
      vf[b] = x[1];
      lf[b] = x[2];
    }
    constexpr int KG = KS / 2;  // steps of a group of key fragments; two groups in flight
    u32x4 kfr[2][KG];
    auto read_k = [&](int g) {
#pragma unroll
      for (int i = 0; i < KG; ++i)
        kfr[g % 2][i] = *reinterpret_cast<const u32x4*>(
            &s.ks[buf][(g / 2 * 32 + j) * KP + (g % 2 * KG + i) * 16 + hf * 8]);
    };
    u32x4 vfr[2][DB];
    auto read_v = [&](int b) {
#pragma unroll
      for (int d = 0; d < DB; ++d)
        vfr[b % 2][d] = *reinterpret_cast<const u32x4*>(
            &s.vts[buf][(d * 32 + j) * VP + b * kBlock + hf * 8]);
    };
    // Two groups of fragments are on their way from LDS while one is multiplied: left to
    // itself the compiler reads each just before its use. The wave in its scores goes before
    // the one of the other workgroup that is in its softmax.
    read_k(0);
    read_k(1);
    __builtin_amdgcn_s_setprio(2);
#pragma unroll
    for (int g = 0; g < NB; ++g) {
      __builtin_amdgcn_sched_barrier(0);
      if (g % 2 == 0)
#pragma unroll
        for (int e = 0; e < 16; ++e) sc[g / 2][e] = 0.f;
#pragma unroll
      for (int i = 0; i < KG; ++i)
        sc[g / 2] = mfma32<QF16>(kfr[g % 2][i], qa[g % 2 * KG + i], sc[g / 2]);
      __builtin_amdgcn_sched_barrier(0);
      if (g + 2 < NB) read_k(g + 2);
      else read_v(g + 2 - NB);
    }
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(0);
    if (key0 + kTile - 1 > wave_first) {  // the diagonal, or past the last key
      // (a block without a page has the factor NaN: only for the rows that see it)
      if constexpr (TREE) {
#pragma unroll
        for (int kb = 0; kb < kTile / 32; ++kb) {
          const uint32_t w = sees.bits(key0 + kb * 32), mine = w >> (4 * hf);
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (!(mine >> (8 * (e / 4) + e % 4) & 1)) sc[kb][e] = -INFINITY;
          if (!(w & 0xffffu)) kf[2 * kb] = a.c2;
          if (!(w >> 16)) kf[2 * kb + 1] = a.c2;
        }
      } else {
        const int lim = sees.last - key0 - 4 * hf;
#pragma unroll
        for (int kb = 0; kb < kTile / 32; ++kb)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (kb * 32 + 8 * (e / 4) + e % 4 > lim) sc[kb][e] = -INFINITY;
#pragma unroll
        for (int b = 0; b < NB; ++b)
          if (b * kBlock > sees.last - key0) kf[b] = a.c2;
      }
    }
    // scores in units of log2, raised by the exponent of V's scale
    float mx = -INFINITY;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const f32x16& z = sc[b / 2];
      const int e = 8 * (b % 2);
      const float x = max3(max3(max3(z[e], z[e + 1], z[e + 2]), z[e + 3], z[e + 4]), z[e + 5],
                           fmaxf(z[e + 6], z[e + 7]));
      mx = fmaxf(mx, C8 ? fmaf(x, kf[b], vf[b]) : x * kf[b]);
    }
    if (__ballot(mx > m + kWeightMost(PF16))) {
      mx = fmaxf(mx, __shfl_xor(mx, 32, kWave));
      const float mn = fmaxf(m, mx - kWeight(PF16));
      const Join j(m, l, mn);
      m = mn;
      l = j.sum(l);
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[d][e] *= j.weight();
    }
    const float ms = m == -INFINITY ? 0.f : m;
    if (C8 && __builtin_amdgcn_readfirstlane(__float_as_int(lf[0])) == 0) {  // (of all blocks)
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int e = 0; e < 8; ++e)
          l += __builtin_amdgcn_exp2f(fmaf(sc[b / 2][8 * (b % 2) + e], kf[b], kSumShift(C8) - ms));
    }
    u32x4 p[NB];  // P^T of a block's 16 keys
#pragma unroll
    for (int b = 0; b < NB + 1; ++b) {
      __builtin_amdgcn_sched_barrier(0);
      if (b < NB) {
        const float off = vf[b] - ms;
        float sum = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = __builtin_amdgcn_exp2f(fmaf(sc[b / 2][8 * (b % 2) + 2 * e], kf[b], off));
          const float y =
              __builtin_amdgcn_exp2f(fmaf(sc[b / 2][8 * (b % 2) + 2 * e + 1], kf[b], off));
          sum += x;
          sum += y;
          p[b][e] = pack2<PF16>(x, y);
        }
        l = C8 ? fmaf(sum, lf[b], l) : l + sum;
      }
      if (b > 0) {
#pragma unroll
        for (int d = 0; d < DB; ++d) o[d] = mfma32<PF16>(vfr[(b - 1) % 2][d], p[b - 1], o[d]);
        if (b + 1 < NB) read_v(b + 1);
      }
      if (b > 0 && b < NB) {  // P V of a block among the exponentials of the next
#pragma unroll
        for (int i = 0; i < DB; ++i) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // MFMA
          __builtin_amdgcn_sched_group_barrier(0x002, 5, 0);  // VALU
          __builtin_amdgcn_sched_group_barrier(0x400, 2, 0);  // transcendental
        }
      }
    }
  }
};

template <int HD, bool QF16, bool C8, bool TREE, int W>
__global__ __launch_bounds__(64 * W, 2) void paged_tile_kernel(PagedArgs a) {
  typedef TileSweep<HD, QF16, C8, TREE, W> T;
  constexpr int kRowsTile = 32 * W;  // query rows of a workgroup
  __shared__ typename T::Lds lds;
  uint32_t grp, place;
  if (!a.map.at(blockIdx.x, grp, place)) return;  // (uniform)
  int s = (int)grp, split, kvh, cb = a.cb, most_splits = (int)a.nsplit.d;
  if constexpr (TREE) {
    kvh = a.KVH.mod(s);
    if (a.share) {  // (uniform)
      const TreeSplit ts(a, s);
      if (ts.s < 0) return;
      s = ts.s;
      split = ts.split;
      cb = ts.cb;
      most_splits = ts.splits;
      if (split + kvh + (int)place == 0 && threadIdx.x == 0) a.counts[s] = most_splits;
    } else {
      // More sequences than share their splits: the first splits of all of them first, so that those
      // which the shorter ones do not have come last, and the units share what there is. One KV
      // head: 300 x 20 rows, 2 heads, on 0.5-4 k e4m3 keys 67 us, 98 with a sequence's splits side by side;
      // 257 x 16 rows, 8 heads, on 1-20 k bf16 keys 1.09 ms and 1.12; 400 x 10 rows on 2 k each 213 both.
      const int seq = a.seqs.mod(s);
      split = s;
      s = seq;
    }
  } else {
    split = a.nsplit.mod(s);
    kvh = a.KVH.mod(s);
  }
  const int tile = (int)a.tiles.d - 1 - (int)place;  // the rows with the most keys first
  T t(a, lds);
  // (as in paged_split_kernel: the first loads do not wait for the lengths)
  t.trow = a.table + (int64_t)s * a.cols;
  t.kvh = kvh;
  t.wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  t.lane = threadIdx.x % kWave;
  t.cur.find(a, t.trow, kvh, split * cb + t.lane);
  const PagedRows pr(a.row_start, s, a.rows, a.max_rows);
  const int pos0 = a.pos0[s];
  const int row0 = tile * kRowsTile, all = pr.n * (int)a.G.d;
  const PagedKeys pk(pos0, pr.n, a.G, TREE ? 0 : row0, TREE ? all : kRowsTile, cb, most_splits,
                     a.most);
  const bool idle = row0 >= all || split >= max(pk.splits, 1);
  const int j = t.j = t.lane % 32, hf = t.hf = t.lane / 32;
  t.b0 = split * cb;
  t.b1 = idle || pk.keys <= 0 ? t.b0 : pk.end(split, cb);
  t.keys = pk.keys;
  const int r0 = row0 + t.wave * 32;  // first row of this wave
  const int qr = max(0, min(r0 + j, all - 1));
  const int qt = a.G.div(qr);
  t.sees = Sees<TREE>(a, pr, pos0, qt);
  if constexpr (TREE) {  // all rows see the context, and any may see the last key
    t.pos_first = t.wave_first = pos0 - 1;
    t.wave_last = r0 < all ? pk.keys - 1 : -1;
  } else {
    t.pos_first = pos0 + a.G.div(row0);
    // positions of the wave's first and last row
    t.wave_first = pos0 + a.G.div(max(0, min(r0, all - 1)));
    t.wave_last = r0 < all ? pos0 + a.G.div(min(r0 + 31, all - 1)) : -1;
  }
  t.qp = a.q + (idle ? 0 : (int64_t)(pr.first + qt) * a.ldq) +
         (int64_t)(kvh * (int)a.G.d + qr - qt * (int)a.G.d) * HD;
  t.sweep();
  if (idle) return;  // (uniform)
  f32x16(&o)[T::DB] = t.o;
  constexpr int DB = T::DB;
  const float l = t.l, m = t.m;
  const int row = r0 + j;
  int tok = row;
  const int head = kvh * (int)a.G.d + a.G.mod(tok);
  const size_t at = (size_t)(pr.first + tok) * a.H.d + head;
  if (pk.splits > 1) {
    if (row >= all) return;
    float* po = a.part_o + (at * a.nsplit.d + split) * HD;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<f4*>(po + d * 32 + 8 * i + 4 * hf) =
            f4{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
    if (hf == 0)
      *reinterpret_cast<float2*>(a.part_ml + (at * a.nsplit.d + split) * 2) = float2{m, l};
    return;
  }
  // Through LDS, so that a store instruction writes whole rows: a lane holds 8 bytes of its
  // row at a time, and 16-byte pieces of 32 rows reach the L2 as as many requests.
  const float inv = sum_inverse<C8>(l);
  const bool none = no_keys<TREE>(a, pr, pos0, min(tok, pr.n - 1));
  constexpr int OP = HD + 8;
  uint16_t* lo = &lds.ks[0][0] + t.wave * 32 * OP;  // (the buffers are free)
  static_assert(2 * W * 32 * OP <= sizeof(lds.ks) + sizeof(lds.vts), "the rows of O fit K and V");
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const u32x2 w = {pack2<QF16>(o[d][4 * i] * inv, o[d][4 * i + 1] * inv),
                       pack2<QF16>(o[d][4 * i + 2] * inv, o[d][4 * i + 3] * inv)};
      *reinterpret_cast<u32x2*>(lo + j * OP + d * 32 + 8 * i + 4 * hf) = none ? u32x2{0u, 0u} : w;
    }
  if (a.lse && hf == 0 && row < all)
    a.lse[at] = none ? -INFINITY : sum_log2<C8>(m, l) * 0.69314718055994530942f;
  __builtin_amdgcn_wave_barrier();  // (one wave's rows: its LDS accesses are in order)
  constexpr int LR = HD / 8;        // lanes of a row
#pragma unroll
  for (int i = 0; i < 32 / (kWave / LR); ++i) {
    const int x = i * (kWave / LR) + t.lane / LR;
    const u32x4 w = *reinterpret_cast<const u32x4*>(lo + x * OP + t.lane % LR * 8);
    if (r0 + x < all) {
      int tk = r0 + x;
      const int hd = kvh * (int)a.G.d + a.G.mod(tk);
      *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(a.out) +
                                ((size_t)(pr.first + tk) * a.H.d + hd) * HD + t.lane % LR * 8) = w;
    }
  }
}

// acc += the sums of N splits, all on their way at once, each times its weight: lane x + k
// holds that of split k.
template <int HD, int N>
__device__ inline void add_splits(const float* po, float weight, int x, int lane,
                                  float (&acc)[HD / kWave]) {
  constexpr int D = HD / kWave;
  float y[N][D];
#pragma unroll
  for (int k = 0; k < N; ++k)
#pragma unroll
    for (int d = 0; d < D; ++d) y[k][d] = po[(size_t)k * HD + lane * D + d];
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const float w = lane_f32(weight, x + k);
#pragma unroll
    for (int d = 0; d < D; ++d) acc[d] = join_o(y[k][d], w, acc[d]);
  }
}

// Joins the splits of a (row, head): one wave each.
template <int HD, bool QF16, bool C8, bool TREE>
__global__ __launch_bounds__(256, 8) void paged_join_kernel(PagedArgs a) {
  int s = (int)(blockIdx.x * 4 + threadIdx.x / kWave);
  const int lane = threadIdx.x % kWave;
  const int head = a.H.mod(s), i = a.rows_each.mod(s);
  if (s >= a.S) return;
  const int given = TREE && a.share ? min(a.counts[s], (int)a.nsplit.d) : 0;
  const PagedRows pr(a.row_start, s, a.rows, a.max_rows);
  if (i >= pr.n) return;
  int x = head;
  const int pos0 = a.pos0[s], row = i * (int)a.G.d + a.G.mod(x);
  const PagedKeys pk(pos0, pr.n, a.G, TREE ? 0 : a.tile.div(row) * (int)a.tile.d,
                     TREE ? pr.n * (int)a.G.d : (int)a.tile.d, a.cb, (int)a.nsplit.d, a.most);
  const int splits = TREE && a.share ? given : pk.splits;
  if (splits <= 1) return;  // written already
  const size_t at = (size_t)(pr.first + i) * a.H.d + head;
  const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + at * a.nsplit.d;
  const float* po = a.part_o + at * a.nsplit.d * HD;
  constexpr int D = HD / kWave;
  float mm = -INFINITY;
  for (int x = lane; x < splits; x += kWave) mm = fmaxf(mm, ml[x].x);
  mm = wave_max(mm);
  float ll = 0.f, acc[D];
#pragma unroll
  for (int d = 0; d < D; ++d) acc[d] = 0.f;
  for (int x0 = 0; x0 < splits; x0 += kWave) {
    const int n = min(kWave, splits - x0);
    const float2 v = lane < n ? ml[x0 + lane] : float2{-INFINITY, 0.f};
    const Join j(v.x, v.y, mm);
    const float f = j.weight();
    ll += wave_sum(j.sum(v.y));
    int x = 0;
    for (; x + 16 <= n; x += 16) add_splits<HD, 16>(po + (size_t)(x0 + x) * HD, f, x, lane, acc);
    for (; x + 8 <= n; x += 8) add_splits<HD, 8>(po + (size_t)(x0 + x) * HD, f, x, lane, acc);
    for (; x + 2 <= n; x += 2) add_splits<HD, 2>(po + (size_t)(x0 + x) * HD, f, x, lane, acc);
    if (x < n) add_splits<HD, 1>(po + (size_t)(x0 + x) * HD, f, x, lane, acc);
  }
  const bool none = no_keys<TREE>(a, pr, pos0, i);
  const float inv = sum_inverse<C8>(ll);
#pragma unroll
  for (int d = 0; d < D; ++d) {
    const float v = none ? 0.f : acc[d] * inv;
    if constexpr (QF16)
      static_cast<_Float16*>(a.out)[at * HD + lane * D + d] = (_Float16)v;
    else
      static_cast<uint16_t*>(a.out)[at * HD + lane * D + d] = f32_to_bf16(v);
  }
  if (a.lse && lane == 0)
    a.lse[at] = none ? -INFINITY : sum_log2<C8>(mm, ll) * 0.69314718055994530942f;
}

// How a call is split: rows of a workgroup, key blocks of a split and splits.
// - 16 rows or fewer a KV head take the 16-row kernel: 32 sequences of 2000 keys, 4 heads to
//   each of 4 KV heads, e4m3, one token 17.3 us beside 20.9 on the 128-row kernel, 4 tokens 18.0
//   beside 22.0. With 5 and 8 tokens two 16-row workgroups are no faster there (21.9, 22.5 beside
//   21.8, 22.7) and slower on 60000 keys: 8 tokens of one sequence 29.5 beside 26.6, of two 46.1
//   beside 35.1, of eight 117 beside 103. (17 to 64 rows leave waves of the 128-row kernel without
//   rows: they stage keys only, and these calls take 1.4 times their bytes' time or more.)
// - Keys are split where there are too few workgroups otherwise, to 1024 (four a unit), 512
//   (two) or 256 (one of 256 rows): 256 sequences x 4 KV heads, already 1024, take 41 us whole
//   and 50 in halves; 32 x 128 rows on 1024 keys, 512 workgroups, 52 whole and 95 in halves.
// - A split has 512 keys at least, for its share of the join: 64 sequences of 300 keys, 256
//   workgroups, take 8.4 us whole and 13.4 in two (16 rows), 13 and 27 (64 rows). (Measured where
//   workgroups fill the chip. Calls with few, as 1 x 64 rows on 4000 keys with 64 of them,
//   21 us, would gain from shorter splits, which this rule does not give them.)
// - 256 rows a workgroup, which stage a tile's keys once for twice the rows (16 % of the time of
//   128), take heads of 128 where sequences are long and workgroups enough: 2 x 1024 rows on
//   24-32 k keys 511 beside 566 us, 8 x 2048 without a context 143 beside 146; but 32 x 512 65
//   beside 56 (one workgroup a unit, whose first loads nothing covers), 1 x 4096 (256
//   workgroups of unequal length) 109 beside 98, 1 x 64 on 4000 (32 of them) 27 beside 21.
//   Heads of 64 have the registers for more than two workgroups of 128: 16 x 512 on 2048 110
//   beside 115, 8 x 2048 117 beside 160.
struct PagedPlan {
  int tile, cb, nsplit;
  int64_t tiles, wgs;
  PagedPlan(int64_t S, int64_t max_rows, int64_t G, int64_t KVH, int64_t hd, int64_t max_tokens) {
    const int64_t all = max_rows * G, units = S * KVH;
    split(all <= kRows16 ? kRows16 : 128, all, units, max_tokens);
    if (tile == 128 && hd == 128 && tiles > 1 && max_tokens > 1024) {
      const PagedPlan narrow = *this;
      split(256, all, units, max_tokens);
      const int64_t least = max_tokens < 2 * max_rows ? 512 : 192;
      if (units * tiles * nsplit < least || 20 * tiles > 11 * narrow.tiles) *this = narrow;
    }
    wgs = tile == kRows16 ? units * tiles * nsplit
                          : PrefillMap((uint32_t)(units * nsplit), (uint32_t)tiles).workgroups();
  }
  void split(int tile_, int64_t all, int64_t units, int64_t max_tokens) {
    tile = tile_;
    tiles = ceil_div(all, tile);
    const int64_t blocks = std::max<int64_t>(1, ceil_div(max_tokens, kBlock));
    const int64_t fill = tile == kRows16 ? 1024 : tile == 128 ? 512 : 256;  // workgroups
    const int64_t want =
        std::max<int64_t>(1, ceil_div(fill, std::max<int64_t>(1, units * tiles)));
    cb = (int)(ceil_div(std::max<int64_t>(32, ceil_div(blocks, want)), 16) * 16);
    nsplit = (int)ceil_div(blocks, cb);
  }
  int64_t threads() const { return wgs * (tile == 256 ? 512 : 256); }
  int64_t bytes(int64_t rows, int64_t H, int64_t hd) const {
    return nsplit > 1 ? rows * H * nsplit * (hd + 2) * 4 : 0;
  }
  // The tree form: where the longest sequence's keys are split, all sequences share `share` splits,
  // as many as fill the units, of which one has four times its even share at most.
  int share = 0;
  void by_length(int64_t S, int64_t KVH, int64_t max_tokens) {
    if (nsplit <= 1 || S > kShared) return;
    const int64_t fill = tile == kRows16 ? 1024 : tile == 128 ? 512 : 256;
    share = (int)ceil_div(fill, KVH * tiles);  // (more than S)
    const int64_t blocks = ceil_div(max_tokens, kBlock);
    nsplit = (int)std::min({ceil_div(blocks, kShare * kUnit), 4 * ceil_div(share, S),
                            (int64_t)share - S + 1});
    nsplit = std::max(nsplit, 2);
    wgs = tile == kRows16 ? KVH * tiles * share
                          : PrefillMap((uint32_t)(KVH * share), (uint32_t)tiles).workgroups();
  }
  int64_t counts(int64_t S) const { return share ? ceil_div(S, 4) * 16 : 0; }  // bytes
};

int check_shape(const char* who, int64_t S, int64_t rows, int64_t max_rows, int64_t H,
                int64_t KVH, int64_t hd, int64_t max_tokens) {
  const int64_t most = 0x7fffffff;
  SM_REQUIRE(S >= 0 && rows >= 0 && max_rows >= 0 && S < most && rows < most && max_rows <= rows,
             "%s: need S >= 0 sequences and 0 <= max_rows <= rows", who);
  SM_REQUIRE(H > 0 && KVH > 0 && H % KVH == 0 && H <= 65535,
             "%s: H must be a multiple of KVH, at most 65535", who);
  SM_REQUIRE(hd == 64 || hd == 128, "%s: head_dim must be 64 or 128", who);
  SM_REQUIRE(max_tokens >= 0 && max_tokens <= most, "%s: max_tokens must be in 0..2^31 - 1", who);
  if (S == 0 || max_rows == 0) return SM_OK;
  const int64_t all = max_rows * (H / KVH);
  // 32 bits index a row of a KV head; the workspace's bytes stay below 2^60; and a grid holds less
  // than 2^32 threads. (The plan's counts fit 64 bits behind the test before it: a workgroup
  // takes 256 rows at most. Keys are split where there are at most 2^16 rows, a wave of the join
  // each.)
  if (all >= most || (double)rows * (double)H >= (double)((int64_t)1 << 40) ||
      (double)S * (double)KVH * (double)ceil_div(all, 256) >= (double)(1 << 24) ||
      PagedPlan(S, max_rows, H / KVH, KVH, hd, max_tokens).threads() >= (int64_t)1 << 32) {
    set_error("%s: problem too large", who);
    return SM_ERR_UNSUPPORTED;
  }
  return SM_OK;
}

}  // namespace

int check_paged_cache(const char* who, const sm_paged_cache* c);

namespace {

// Both forms of the call; mask and words are the tree form's.
template <bool TREE>
int paged_attention(const char* me, const sm_paged_cache* cache, const int32_t* block_table,
                    int64_t table_cols, const int32_t* pos0, const int32_t* row_start, int64_t S,
                    int64_t rows, int64_t max_rows, int64_t max_tokens, const int32_t* mask,
                    int64_t words, const void* q, int dtype, int64_t ldq, int64_t H, void* out,
                    float* lse, void* workspace, int64_t workspace_bytes, void* stream) {
  SM_TRY(check_paged_cache(me, cache));
  const int64_t KVH = cache->kv_heads, hd = cache->head_dim;
  SM_TRY(check_shape(me, S, rows, max_rows, H, KVH, hd, max_tokens));
  SM_REQUIRE(dtype == SM_BF16 || dtype == SM_F16, "%s: dtype must be SM_BF16 or SM_F16", me);
  SM_REQUIRE(cache->dtype == SM_F8E4M3 || cache->dtype == dtype,
             "%s: a 16-bit cache must have the query's dtype", me);
  if (S == 0 || max_rows == 0) return SM_OK;
  SM_REQUIRE(block_table && pos0 && q && out && (!TREE || mask), "%s: null buffer", me);
  SM_REQUIRE(!TREE || (words >= ceil_div(max_rows, 32) && words <= 1 << 20),
             "%s: words must be at least max_rows / 32", me);
  SM_REQUIRE(table_cols > 0 && table_cols <= 0x7fffffff, "%s: table_cols must be positive", me);
  SM_REQUIRE(row_start || rows == S * max_rows,
             "%s: without row_start, rows must be S * max_rows", me);
  const uintptr_t qa = reinterpret_cast<uintptr_t>(q), oa = reinterpret_cast<uintptr_t>(out);
  SM_REQUIRE(ldq >= H * hd && ldq < ((int64_t)1 << 31) && ldq % 8 == 0 && qa % 16 == 0 &&
                 oa % 16 == 0,
             "%s: q rows and out must be 16-byte aligned, ldq >= H * head_dim and ldq < 2^31", me);
  PagedPlan plan(S, max_rows, H / KVH, KVH, hd, max_tokens);
  if (TREE) plan.by_length(S, KVH, max_tokens);
  const int64_t need = plan.bytes(rows, H, hd) + plan.counts(S);
  SM_REQUIRE(need == 0 || (workspace && workspace_bytes >= need &&
                           reinterpret_cast<uintptr_t>(workspace) % 16 == 0),
             "%s: workspace of %lld bytes, %lld needed, 16-byte aligned", me,
             (long long)workspace_bytes, (long long)need);
  SM_REQUIRE(qa + (size_t)((rows - 1) * ldq + H * hd) * 2 <= oa ||
                 oa + (size_t)(rows * H * hd) * 2 <= qa,
             "%s: out must not overlap q", me);
  const int64_t joins = ceil_div(S * max_rows * H, 4);
  hipStream_t st = as_stream(stream);
  PagedArgs a;
  a.k = static_cast<const uint8_t*>(cache->k);
  a.v = static_cast<const uint8_t*>(cache->v);
  a.ks = cache->dtype == SM_F8E4M3 ? cache->k_scales : nullptr;
  a.vs = cache->v_scales;
  a.q = static_cast<const uint16_t*>(q);
  a.table = block_table;
  a.pos0 = pos0;
  a.row_start = row_start;
  a.out = out;
  a.lse = lse;
  a.share = plan.share;
  a.counts = static_cast<int32_t*>(workspace);
  a.part_o = need ? static_cast<float*>(workspace) + plan.counts(S) / 4 : nullptr;
  a.part_ml = need ? a.part_o + rows * H * plan.nsplit * hd : nullptr;
  a.ldq = ldq;
  a.S = (int)S;
  a.rows = (int)rows;
  a.max_rows = (int)max_rows;
  a.H = Divide((int)H);
  a.KVH = Divide((int)KVH);
  a.G = Divide((int)(H / KVH));
  a.rows_each = Divide((int)max_rows);
  a.pages = (int)cache->pages;
  a.bpp = Divide((int)(cache->page_tokens / kBlock));
  a.cols = (int)table_cols;
  a.cb = plan.cb;
  a.mask = reinterpret_cast<const uint32_t*>(mask);
  a.words = (int)words;
  a.most = (int)std::min<int64_t>(table_cols * a.bpp.d + 1, 1 << 27);
  a.nsplit = Divide(plan.nsplit);
  a.seqs = Divide((int)S);
  a.tile = Divide(plan.tile);
  a.tiles = Divide((int)plan.tiles);
  // the keys of a group, and whether an XCD's groups leave a quarter of its 4 MiB L2
  // (shared splits: as long as they are where all sequences have max_tokens)
  const int64_t span = plan.share ? std::max<int64_t>(kShare * kUnit * kBlock,
                                                      ceil_div(S * max_tokens, plan.share))
                       : plan.nsplit > 1 ? (int64_t)plan.cb * kBlock : max_tokens;
  const int64_t kv = span * hd * (cache->dtype == SM_F8E4M3 ? 2 : 4);
  const int64_t groups = KVH * (plan.share ? plan.share : S * plan.nsplit);
  a.map = PagedMap((uint32_t)groups, (uint32_t)plan.tiles, groups / 8 * kv <= 3 << 20);
  a.c2 = 1.44269504088896340736f / sqrtf((float)hd);
  const bool f16 = dtype == SM_F16, c8 = cache->dtype == SM_F8E4M3;
#define SM_PAGED2(HD, F, C)                                                      \
  do {                                                                           \
    if (plan.tile == kRows16)                                                    \
      paged_split_kernel<HD, F, C, TREE><<<(unsigned)plan.wgs, 256, 0, st>>>(a);       \
    else if (HD < 128 || plan.tile == 128)                                       \
      paged_tile_kernel<HD, F, C, TREE, 4><<<(unsigned)plan.wgs, 256, 0, st>>>(a);     \
    else if constexpr (HD == 128)                                                \
      paged_tile_kernel<HD, F, C, TREE, 8><<<(unsigned)plan.wgs, 512, 0, st>>>(a);     \
    if (plan.nsplit > 1)                                                         \
      paged_join_kernel<HD, F, C, TREE><<<(unsigned)joins, 256, 0, st>>>(a);              \
  } while (0)
#define SM_PAGED(HD)                             \
  do {                                           \
    if (f16 && c8) SM_PAGED2(HD, true, true);    \
    else if (f16) SM_PAGED2(HD, true, false);    \
    else if (c8) SM_PAGED2(HD, false, true);     \
    else SM_PAGED2(HD, false, false);            \
  } while (0)
  if (hd == 64) SM_PAGED(64);
  else SM_PAGED(128);
#undef SM_PAGED
#undef SM_PAGED2
  SM_LAUNCH_CHECK();
  return SM_OK;
}

}  // namespace
}  // namespace sm
