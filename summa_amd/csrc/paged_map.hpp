// What a paged batch's sequences, rows and key splits are. Host and device, so that
// the map can be walked on the CPU.
#pragma once

#include <cstdint>

#include <hip/hip_runtime.h>

#include "prefill_map.hpp"

namespace sm {

constexpr int kBlock = 16;  // tokens of a cache block (and of a scale)

// Division of 0 <= n < 2^31 by a divisor that the host knows: a multiply and a shift (round-up
// method: with 2^shift >= d and mul = ceil(2^32 (2^shift - d) / d), or one more where that is
// whole, the quotient is ((n mul >> 32) + n) >> shift). The compiler's own division takes
// about 20 instructions, and a workgroup of few keys makes eight.
struct Divide {
  uint32_t d = 1, mul = 1, shift = 0;
  Divide() = default;
  __host__ __device__ Divide(int by) : d((uint32_t)by), shift(0) {
    while (((uint64_t)1 << shift) < d) ++shift;
    mul = (uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << shift) - d)) / d + 1);
  }
  __host__ __device__ int div(int n) const {
    return (int)(((uint32_t)((uint64_t)(uint32_t)n * mul >> 32) + (uint32_t)n) >> shift);
  }
  // n becomes the quotient, the remainder is returned
  __host__ __device__ int mod(int& n) const {
    const int q = div(n), r = n - q * (int)d;
    n = q;
    return r;
  }
};

// Rows [first, first + n) of sequence s: the ragged form's row_start [S + 1], or
// max_rows each without one. Whatever row_start holds, they lie inside [0, rows).
struct PagedRows {
  int first, n;
  __host__ __device__ PagedRows(const int32_t* row_start, int s, int rows, int max_rows) {
    int a, b;
    if (row_start) {
      a = row_start[s];
      b = row_start[s + 1];
      a = a < 0 ? 0 : a > rows ? rows : a;
      b = b < a ? a : b > rows ? rows : b;
    } else {
      a = s * max_rows;
      b = a + max_rows;
    }
    first = a;
    n = b - a < max_rows ? b - a : max_rows;
  }
};

// The cache block of block `blk` of a sequence, as an index over [pages, KVH, page / 16];
// -1 where the table has no such entry or the entry names no page.
__host__ __device__ inline int paged_block(const int32_t* table_row, int cols, int pages, int KVH,
                                           int kvh, const Divide& bpp, int blk) {
  if (blk < 0) return -1;
  const int col = bpp.div(blk);
  if (col >= cols) return -1;
  const int page = table_row[col];
  if (page < 0 || page >= pages) return -1;
  return (page * KVH + kvh) * (int)bpp.d + (blk - col * (int)bpp.d);
}

// Blocks that n tokens touch at most, wherever the first of them falls.
__host__ __device__ inline int64_t paged_touched(int64_t n) { return (n + kBlock - 2) / kBlock + 1; }

// Keys of one tile of `tile` query rows and their split. A row is a (token, head of
// the KV head's group) pair, G heads to a token, so the tile's last row sees the most
// keys. Split i of `nsplit` takes blocks [i cb, (i + 1) cb); the last one takes what is
// left, so that no key is dropped however long the sequence is. `most`: blocks that a table
// row holds, and one: the first without a page, for all the keys behind it that have none,
// so that a wrong length costs no more than a full table.
struct PagedKeys {
  int keys;    // keys that the tile's last row sees (<= 0: none)
  int blocks;  // blocks that hold them
  int splits;  // splits that have work (0 without keys)
  __host__ __device__ PagedKeys(int pos0, int n, const Divide& G, int first_row, int tile,
                                int cb, int nsplit, int most = 1 << 27) {
    const int all = n * (int)G.d;
    int last = first_row + tile - 1;
    if (last > all - 1) last = all - 1;
    const int64_t k = last < 0 ? 0 : (int64_t)pos0 + G.div(last) + 1;
    const int64_t held = (int64_t)most * kBlock, in = k > held ? held : k;
    keys = in < 0 ? 0 : in > 0x7fffffff ? 0x7fffffff : (int)in;
    blocks = (int)(((int64_t)keys + kBlock - 1) / kBlock);
    const int64_t want = ((int64_t)blocks + cb - 1) / cb;
    splits = want < nsplit ? (int)want : nsplit;
  }
  __host__ __device__ int begin(int split, int cb) const { return split * cb; }
  __host__ __device__ int end(int split, int cb) const {
    return split + 1 >= splits ? blocks : (split + 1) * cb;
  }
};

// Which workgroup takes which (KV head of a sequence's split) and row tile: PrefillMap's
// share of groups for every XCD, whose L2 then reads a group's K and V once, but
// - the eight groups of a set go to the XCDs in another turn in each set, so that a long
//   sequence's KV heads and a short one's do not meet the same XCDs every time, and
// - with by_place, where the K and V of all an XCD's groups stay in its L2, every group's
//   tile with the most keys comes before any group's next, and what runs last is short.
// Prefill of 32 prompts of 257-512 tokens, 4 KV heads: 58.6 -> 57.2 us with the turns,
// 52.4 with both.
struct PagedMap {
  PrefillMap map;
  Divide per, sets;
  bool by_place;
  PagedMap() : map(1, 1), by_place(false) {}
  __host__ __device__ PagedMap(uint32_t groups, uint32_t per_, bool by_place_)
      : map(groups, per_), per((int)per_), sets((int)(groups / 8 ? groups / 8 : 1)),
        by_place(by_place_) {}
  __host__ __device__ bool at(uint32_t wg, uint32_t& group, uint32_t& place) const {
    int set = (int)(wg / 8);
    if (set >= (int)(map.whole / 8 * map.per)) return map.at(wg, group, place);
    if (by_place) {
      const int s = sets.mod(set);
      place = (uint32_t)set;
      set = s;
    } else {
      place = (uint32_t)per.mod(set);
    }
    group = (uint32_t)set * 8 + (wg + 3 * (uint32_t)set) % 8;
    return true;
  }
};

}  // namespace sm
