// New keys and values into a paged KV cache, keys and queries rotated on the way.
//
//   project_qkv's split, RoPE and the AttnCache slice_assign
//   (summa-llm/src/model/attention.rs:142-177, 331-356) over the paged cache of
//   sm_paged_cache.
//
// One wave takes one head of one 16-token cache block at a time: a block's scale is the
// maximum over its tokens, so the wave needs no other wave's values, no two waves write one
// scale, and there is no barrier. A wave goes through several heads of its block where
// there are blocks enough, with the angles of its tokens in registers.
// Queries and keys: lane (i, c) of 64 / (head_dim / 8) x head_dim / 8 holds two times four
// dims of tokens i, i + 64 / (head_dim / 8), ..: in the half layout 4 c .. and 4 c + rot_dim / 2 ..,
// so that both of a pair are in one lane.
// Values: lane (g, c) holds head_dim / 16 dims of tokens 4 g .. 4 g + 3, which is a word (8-bit)
// or two of the stored block a dim; the block goes through LDS to be stored as it lies.
// Bound by memory: 12.6 k bf16 rows of 16 + 2 x 4 heads of 128 into an e4m3 cache (146 MB read
// and written) 33 us, 4.5 TB/s; 4.6 k f16 rows of 36 heads of 64 into an f16 cache (48 MB)
// 11.3 us. A step of 256 sequences, one token each, is 8 us of round trips to memory, one behind
// the other - a key's wave waits for the lengths, its rows and angles, the page and the block's
// scale, a value's for the lengths, the page, its rows, the scale and the block as it was - in
// 9.7 us of the host's call.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "common.hpp"
#include "paged_map.hpp"
#include "rotary.hpp"

namespace sm {

int check_paged_cache(const char* who, const sm_paged_cache* c);

namespace {

struct AppendArgs {
  uint8_t *kc, *vc, *ks, *vs;
  const void *q, *k, *v;
  int64_t ldq, ldk, ldv;
  const float* rope;
  int64_t rope_rows;
  const int32_t *table, *pos0, *row_start;
  void* q_out;
  Divide bpp, touched, groups;
  int S, rows, max_rows, H, KVH, pages, cols, rot, half_layout, q_f16, each;
};

// D consecutive values of a row as f32 (8: 16-byte loads; 4: 8- or 16-byte ones).
template <typename T, int D>
__device__ inline void load_dims(const T* p, float (&f)[D]) {
  if constexpr (D == 8) {
    load8<T>(p, f);
  } else if constexpr (sizeof(T) == 4) {
    const float4 a = *reinterpret_cast<const float4*>(p);
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
  } else {
    const u32x2 v = *reinterpret_cast<const u32x2*>(p);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if constexpr (__is_same(T, _Float16)) {
        const h2 x = as_h2(v[i]);
        f[2 * i] = (float)x[0];
        f[2 * i + 1] = (float)x[1];
      } else {
        f[2 * i] = bf16lo(v[i]);
        f[2 * i + 1] = bf16hi(v[i]);
      }
    }
  }
}

// Four f32 -> e4m3 codes (nearest even), the first in the low byte.
__device__ inline uint32_t pack_e4m3(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}
// The codes of a word times f, rounded again.
__device__ inline uint32_t rescale_e4m3(uint32_t w, float f) {
  const f32x2_t lo = __builtin_amdgcn_cvt_pk_f32_fp8(w, false),
                hi = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
  return pack_e4m3(lo[0] * f, lo[1] * f, hi[0] * f, hi[1] * f);
}
__device__ inline float pow2f(int e) { return __uint_as_float((uint32_t)max(e + 127, 0) << 23); }

// The least e >= -63 with amax <= 448 * 2^e (448 = 1.75 * 2^8, the largest e4m3 value).
__device__ inline int scale_exponent(float amax) {
  const uint32_t b = __float_as_uint(amax);
  return max(-63, (int)(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0));
}

// Four consecutive values of a row as they lie, and as f32.
template <typename T>
struct Four {
  u32x2 w;
  __device__ inline void get(float (&f)[4]) const {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if constexpr (__is_same(T, _Float16)) {
        const h2 x = as_h2(w[i]);
        f[2 * i] = (float)x[0];
        f[2 * i + 1] = (float)x[1];
      } else {
        f[2 * i] = bf16lo(w[i]);
        f[2 * i + 1] = bf16hi(w[i]);
      }
    }
  }
};
template <>
struct Four<float> {
  u32x4 w;
  __device__ inline void get(float (&f)[4]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(w[i]);
  }
};

template <typename T, int HD, int CT>  // CT: cache type, 0 bf16, 1 f16, 2 e4m3
struct Append {
  static constexpr int LPT = HD / 8, TPL = HD / 32, STEP = kWave / LPT;
  static constexpr int D = HD / 16;
  static constexpr int ES = CT == 2 ? 1 : 2;
  static constexpr int NC = HD * ES / 64;  // kilobytes of a block
  typedef typename std::conditional<CT == 1, _Float16, uint16_t>::type TC;

  const AppendArgs& a;
  int lane, t0, t1;
  int64_t base, row0;  // position and row of the block's token 0
  const int32_t* trow;
  u32x4* lds;          // this wave's NC kilobytes
  float cs[TPL][4], sn[TPL][4];
  Four<T> x[TPL][2];   // the slot at hand, as loaded
  bool turn;           // this lane's dims are rotated

  // The lane number anew: what a head's addresses are made of, so that those of all heads
  // (30 registers) are not kept through the loop over heads.
  __device__ inline int lane_again() const {
    int l = lane;
    asm volatile("" : "+v"(l));
    return l;
  }
  __device__ inline bool mine(int t) const { return t >= t0 && t < t1; }
  static __device__ inline int token(int l, int j) { return l / LPT + j * STEP; }
  // first dims of a lane's two fours
  __device__ inline int dim_a(int l) const {
    return a.half_layout && turn ? 4 * (l % LPT) : 8 * (l % LPT);
  }
  __device__ inline int dim_b(int l) const {
    return dim_a(l) + (a.half_layout && turn ? a.rot / 2 : 4);
  }

  __device__ inline void angles() {
    turn = 8 * (lane % LPT) < a.rot;
#pragma unroll
    for (int j = 0; j < TPL; ++j)  // (dims and tokens that are not to be rotated read some too)
      load_angles<4>(a.rope, a.rope_rows, a.rot / 2, base + token(lane, j),
                     turn ? 4 * (lane % LPT) : 0, cs[j], sn[j]);
  }
  // a query's or key's head
  __device__ inline void load_row(const void* p, int64_t ld, int head) {
    const T* src = static_cast<const T*>(p) + (int64_t)head * HD;
    const int l = lane_again();
#pragma unroll
    for (int j = 0; j < TPL; ++j) {
      const int t = token(l, j);
      x[j][0] = x[j][1] = Four<T>{};
      if (mine(t)) {
        x[j][0] = *reinterpret_cast<const Four<T>*>(src + (row0 + t) * ld + dim_a(l));
        x[j][1] = *reinterpret_cast<const Four<T>*>(src + (row0 + t) * ld + dim_b(l));
      }
    }
  }
  __device__ inline void rotate(float (&y)[TPL * 8]) const {
    const bool half = a.half_layout;  // (values are chosen, not places: those would go to memory)
#pragma unroll
    for (int j = 0; j < TPL; ++j) {
      const bool on = turn && mine(token(lane, j));
      float u[4], w[4], p[4], q[4];
      x[j][0].get(u);
      x[j][1].get(w);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        p[i] = half ? u[i] : i < 2 ? u[2 * i] : w[2 * i - 4];
        q[i] = half ? w[i] : i < 2 ? u[2 * i + 1] : w[2 * i - 3];
        if (on) rotate_pair(p[i], q[i], cs[j][i], sn[j][i]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        y[8 * j + i] = half ? p[i] : i % 2 ? q[i / 2] : p[i / 2];
        y[8 * j + 4 + i] = half ? q[i] : i % 2 ? q[2 + i / 2] : p[2 + i / 2];
      }
    }
  }
  template <typename TQ>
  __device__ inline void store_q(const float (&y)[TPL * 8], int head) const {
    const int l = lane_again();
#pragma unroll
    for (int j = 0; j < TPL; ++j) {
      const int t = token(l, j);
      if (!mine(t)) continue;
      TQ* p = static_cast<TQ*>(a.q_out) + ((row0 + t) * a.H + head) * HD;
      *reinterpret_cast<u32x2*>(p + dim_a(l)) =
          u32x2{round2<TQ>(y[8 * j + 0], y[8 * j + 1]), round2<TQ>(y[8 * j + 2], y[8 * j + 3])};
      *reinterpret_cast<u32x2*>(p + dim_b(l)) =
          u32x2{round2<TQ>(y[8 * j + 4], y[8 * j + 5]), round2<TQ>(y[8 * j + 6], y[8 * j + 7])};
    }
  }

  // The block's exponent for the values y of this call, with the earlier tokens' where some
  // stay; `again` scales those down.
  template <int N>
  __device__ inline void scale(const float (&y)[N], uint8_t* sp, float& inv, float& again,
                               bool& grown, bool& odd) const {
    // (as bits, infinities and NaN are above every finite value)
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) most = max(most, __float_as_uint(y[i]) & 0x7fffffffu);
    odd = __ballot(most >= 0x7f800000u) != 0;
    if (odd) {
      most = 0;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const uint32_t v = __float_as_uint(y[i]) & 0x7fffffffu;
        most = max(most, v < 0x7f800000u ? v : 0u);
      }
    }
    const float amax = __uint_as_float(most);
    int e = scale_exponent(wave_max(amax)), old = e;
    if (t0 > 0) {
      old = (int)*sp - 127;
      e = max(e, old);
    }
    grown = e > old;  // (uniform)
    again = pow2f(old - e);
    inv = pow2f(-e);
    if (lane == 0) *sp = (uint8_t)(e + 127);
  }
  // Four values -> codes; infinities and NaN are the NaN code.
  static __device__ inline uint32_t encode(const float (&y)[4], bool odd) {
    uint32_t w = pack_e4m3(y[0], y[1], y[2], y[3]);
    if (odd) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (!(fabsf(y[i]) < INFINITY)) w = (w & ~(0xffu << (8 * i))) | (0x7fu << (8 * i));
    }
    return w;
  }

  __device__ inline int block(int head) const {
    return paged_block(trow, a.cols, a.pages, a.KVH, head, a.bpp, (int)(base / kBlock));
  }
  __device__ inline void store_k(float (&y)[TPL * 8], int head) const {
    const int bi = block(head);
    if (bi < 0) return;  // (uniform) no page for these tokens
    const int l = lane_again();
    if constexpr (CT == 2) {
      float inv, again;
      bool grown, odd;
      scale(y, a.ks + bi, inv, again, grown, odd);
      uint8_t* page = a.kc + (size_t)bi * (kBlock * HD);
#pragma unroll
      for (int j = 0; j < TPL; ++j) {
        const int t = token(l, j);
        uint32_t* pa = reinterpret_cast<uint32_t*>(page + t * HD + dim_a(l));
        uint32_t* pb = reinterpret_cast<uint32_t*>(page + t * HD + dim_b(l));
        if (mine(t)) {
          const float u[4] = {y[8 * j + 0] * inv, y[8 * j + 1] * inv, y[8 * j + 2] * inv, y[8 * j + 3] * inv};
          const float w[4] = {y[8 * j + 4] * inv, y[8 * j + 5] * inv, y[8 * j + 6] * inv, y[8 * j + 7] * inv};
          *pa = encode(u, odd);
          *pb = encode(w, odd);
        } else if (t < t0 && grown) {
          *pa = rescale_e4m3(*pa, again);
          *pb = rescale_e4m3(*pb, again);
        }
      }
    } else {
      TC* page = reinterpret_cast<TC*>(a.kc) + (size_t)bi * (kBlock * HD);
#pragma unroll
      for (int j = 0; j < TPL; ++j) {
        const int t = token(l, j);
        if (!mine(t)) continue;
        *reinterpret_cast<u32x2*>(page + t * HD + dim_a(l)) =
            u32x2{round2<TC>(y[8 * j + 0], y[8 * j + 1]), round2<TC>(y[8 * j + 2], y[8 * j + 3])};
        *reinterpret_cast<u32x2*>(page + t * HD + dim_b(l)) =
            u32x2{round2<TC>(y[8 * j + 4], y[8 * j + 5]), round2<TC>(y[8 * j + 6], y[8 * j + 7])};
      }
    }
  }

  __device__ inline void append_v(int head) const {
    const int bi = block(head);
    if (bi < 0) return;  // (uniform)
    const int g = lane / 16, c = lane % 16;
    const T* src = static_cast<const T*>(a.v) + (int64_t)head * HD + D * c;
    float v[4 * D];  // [token 4 g + j][dim D c + i]
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float f[D];
      const int t = 4 * g + j;
#pragma unroll
      for (int i = 0; i < D; ++i) f[i] = 0.f;
      if (mine(t)) load_dims<T, D>(src + (row0 + t) * a.ldv, f);
#pragma unroll
      for (int i = 0; i < D; ++i) v[j * D + i] = f[i];
    }
    float inv = 1.f, again = 1.f;
    bool grown = false, odd = false;
    if constexpr (CT == 2) scale(v, a.vs + bi, inv, again, grown, odd);
    // To LDS: 16-byte pieces in the block's order (piece ((d / 16 T) 4 + g) 16 + d % 16), each
    // eight times 16 pieces in an order of their own, which spreads the words over the banks.
    constexpr int TT = 4 / ES;
#pragma unroll
    for (int i = 0; i < D; ++i) {
      const int d = D * c + i, n = d / 16;
      const int piece = (n / TT * 4 + g) * 16 + d % 16, at = piece ^ (piece / 16 % 8);
      const float y[4] = {v[i] * inv, v[D + i] * inv, v[2 * D + i] * inv, v[3 * D + i] * inv};
      if constexpr (CT == 2)
        reinterpret_cast<uint32_t*>(lds + at)[n % TT] = encode(y, odd);
      else
        reinterpret_cast<u32x2*>(lds + at)[n % TT] = u32x2{round2<TC>(y[0], y[1]), round2<TC>(y[2], y[3])};
    }
    __builtin_amdgcn_wave_barrier();  // (one wave's LDS accesses are in order)
    // masks of the call's tokens and of earlier ones in the quad of this lane's pieces
    uint32_t m[2] = {0, 0}, older = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int t = 4 * g + j;
      if constexpr (CT == 2) {
        if (mine(t)) m[0] |= 0xffu << (8 * j);
        if (t < t0) older |= 0xffu << (8 * j);
      } else if (mine(t)) {
        m[j / 2] |= 0xffffu << (16 * (j % 2));
      }
    }
    if constexpr (CT == 2) m[1] = m[0];
    u32x4* page = reinterpret_cast<u32x4*>(a.vc + (size_t)bi * (kBlock * HD * ES)) + lane;
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const int piece = k * kWave + lane;
      u32x4 w = lds[piece ^ (piece / 16 % 8)];
      if (!(m[0] | m[1]) && !(grown && older)) continue;
      const u32x4 keep = {m[0], m[1], m[0], m[1]};
      if (~(m[0] & m[1])) {
        u32x4 was = page[k * kWave];
        if constexpr (CT == 2) {
          if (grown) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              was[i] = (was[i] & ~older) | (rescale_e4m3(was[i], again) & older);
          }
        }
        w = (w & keep) | (was & ~keep);
      }
      page[k * kWave] = w;
    }
    __builtin_amdgcn_wave_barrier();
  }
};

template <typename T, int HD, int CT>
__global__ __launch_bounds__(256, 4) void paged_append_kernel(AppendArgs a) {
  typedef Append<T, HD, CT> A;
  __shared__ u32x4 lds[4][A::NC * kWave];
  int s = (int)blockIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int group = a.groups.mod(s), nth = a.touched.mod(s);
  const PagedRows pr(a.row_start, s, a.rows, a.max_rows);
  const int pos0 = a.pos0[s];
  const int64_t end = (int64_t)pos0 + pr.n;  // one past the last position
  A x{a};
  x.lane = threadIdx.x % kWave;
  x.base = (int64_t)(max(pos0, 0) / kBlock + nth) * kBlock;
  x.t0 = (int)max((int64_t)max(pos0, 0) - x.base, (int64_t)0);
  x.t1 = (int)min(end - x.base, (int64_t)kBlock);
  if (x.t0 >= x.t1) return;  // (uniform) the block holds none of the rows
  x.row0 = pr.first + (x.base - pos0);
  x.trow = a.table + (int64_t)s * a.cols;
  x.lds = lds[wave];
  x.turn = false;
  // slots: query heads, key heads, value heads
  const int slots = a.H + 2 * a.KVH, turned = a.H + a.KVH;
  int slot = group * 4 * a.each + wave;
  const int stop = min(slots, (group + 1) * 4 * a.each);
  if (slot < turned && a.rot > 0) x.angles();
  for (; slot < min(stop, turned); slot += 4) {
    float y[A::TPL * 8];
    if (slot < a.H) x.load_row(a.q, a.ldq, slot);
    else x.load_row(a.k, a.ldk, slot - a.H);
    x.rotate(y);
    if (slot >= a.H) x.store_k(y, slot - a.H);
    else if (a.q_f16) x.template store_q<_Float16>(y, slot);
    else x.template store_q<uint16_t>(y, slot);
  }
  for (; slot < stop; slot += 4) x.append_v(slot - turned);
}

}  // namespace
}  // namespace sm

extern "C" int sm_paged_append(const sm_paged_cache* cache, const int32_t* block_table,
                               int64_t table_cols, const int32_t* pos0, const int32_t* row_start,
                               int64_t S, int64_t rows, int64_t max_rows, const void* q,
                               int64_t ldq, const void* k, int64_t ldk, const void* v, int64_t ldv,
                               int dtype, int64_t H, const float* rope_table, int64_t rope_rows,
                               int64_t rot_dim, int layout, void* q_out, int q_dtype,
                               void* stream) {
  using namespace sm;
  const char* me = "sm_paged_append";
  SM_TRY(check_paged_cache(me, cache));
  const int64_t KVH = cache->kv_heads, hd = cache->head_dim, most = 0x7fffffff;
  SM_REQUIRE(S >= 0 && rows >= 0 && max_rows >= 0 && S < most && rows < most && max_rows <= rows,
             "%s: need S >= 0 sequences and 0 <= max_rows <= rows", me);
  SM_REQUIRE(dtype == SM_F32 || dtype == SM_BF16 || dtype == SM_F16,
             "%s: dtype must be SM_F32, SM_BF16 or SM_F16", me);
  SM_REQUIRE(!q || (H > 0 && H <= 65535), "%s: need 0 < H <= 65535 query heads", me);
  SM_REQUIRE(!q || q_dtype == SM_BF16 || q_dtype == SM_F16, "%s: q_dtype must be SM_BF16 or SM_F16",
             me);
  if (rope_table) {
    SM_REQUIRE(layout == SM_ROPE_INTERLEAVED || layout == SM_ROPE_HALF,
               "%s: layout must be SM_ROPE_INTERLEAVED or SM_ROPE_HALF", me);
    SM_REQUIRE(rot_dim >= 16 && rot_dim % 16 == 0 && rot_dim <= hd,
               "%s: rot_dim must be a multiple of 16 up to head_dim", me);
    SM_REQUIRE(rope_rows > 0 && reinterpret_cast<uintptr_t>(rope_table) % 16 == 0,
               "%s: rope_table must be 16-byte aligned and have rows", me);
  } else {
    SM_REQUIRE(rot_dim == 0, "%s: rot_dim without a rope_table", me);
  }
  if (S == 0 || max_rows == 0) return SM_OK;
  SM_REQUIRE(block_table && pos0 && k && v && (!q || q_out), "%s: null buffer", me);
  SM_REQUIRE(table_cols > 0 && table_cols <= most, "%s: table_cols must be positive", me);
  SM_REQUIRE(row_start || rows == S * max_rows,
             "%s: without row_start, rows must be S * max_rows", me);
  const int64_t each = dtype == SM_F32 ? 4 : 8;  // values of 16 bytes
  const int64_t wide = (int64_t)1 << 31;
  SM_REQUIRE(ldk >= KVH * hd && ldv >= KVH * hd && ldk % each == 0 && ldv % each == 0 &&
                 ldk < wide && ldv < wide &&
                 (!q || (ldq >= H * hd && ldq % each == 0 && ldq < wide)),
             "%s: rows must be 16-byte aligned and hold their heads", me);
  if (q) {
    const size_t size = 16 / each;
    const uintptr_t o0 = reinterpret_cast<uintptr_t>(q_out), o1 = o0 + (size_t)(rows * H * hd * 2);
    auto apart = [&](const void* p, int64_t ld, int64_t width) {
      const uintptr_t a0 = reinterpret_cast<uintptr_t>(p);
      return a0 + (size_t)((rows - 1) * ld + width) * size <= o0 || o1 <= a0;
    };
    SM_REQUIRE(apart(q, ldq, H * hd) && apart(k, ldk, KVH * hd) && apart(v, ldv, KVH * hd),
               "%s: q_out must not overlap q, k or v", me);
  }
  for (const void* p : {k, v, q, (const void*)q_out})
    SM_REQUIRE(reinterpret_cast<uintptr_t>(p) % 16 == 0, "%s: buffers must be 16-byte aligned", me);
  AppendArgs a;
  a.kc = static_cast<uint8_t*>(cache->k);
  a.vc = static_cast<uint8_t*>(cache->v);
  a.ks = cache->k_scales;
  a.vs = cache->v_scales;
  a.q = q;
  a.k = k;
  a.v = v;
  a.ldq = ldq;
  a.ldk = ldk;
  a.ldv = ldv;
  a.rope = rope_table;
  a.rope_rows = rope_rows;
  a.table = block_table;
  a.pos0 = pos0;
  a.row_start = row_start;
  a.q_out = q_out;
  a.S = (int)S;
  a.rows = (int)rows;
  a.max_rows = (int)max_rows;
  a.H = q ? (int)H : 0;
  a.KVH = (int)KVH;
  a.pages = (int)cache->pages;
  a.bpp = Divide((int)(cache->page_tokens / kBlock));
  a.cols = (int)table_cols;
  a.rot = rope_table ? (int)rot_dim : 0;
  a.half_layout = layout == SM_ROPE_HALF;
  a.q_f16 = q_dtype == SM_F16;
  a.touched = Divide((int)paged_touched(max_rows));
  // Heads that a wave goes through, for the angles that it then reads once: as many as leave
  // 2048 workgroups, two for every place on the chip. (12.6 k bf16 rows of 16 + 2 x 4 heads of
  // 128, 3.3 times that many blocks of work: one head a wave 40 us, three 33.)
  const int64_t slots = a.H + 2 * KVH;
  a.each = (int)std::max<int64_t>(
      1, std::min<int64_t>(ceil_div(slots, 4), S * a.touched.d * ceil_div(slots, 4) / 2048));
  a.groups = Divide((int)ceil_div(slots, 4 * a.each));
  if ((double)S * a.touched.d * a.groups.d >= (double)(1 << 24)) {
    set_error("%s: problem too large", me);
    return SM_ERR_UNSUPPORTED;
  }
  const unsigned wgs = (unsigned)(S * a.touched.d * a.groups.d);
  hipStream_t st = as_stream(stream);
#define SM_APP3(T, HD, CT) paged_append_kernel<T, HD, CT><<<wgs, 256, 0, st>>>(a)
#define SM_APP2(T, HD)                                  \
  do {                                                  \
    if (cache->dtype == SM_F8E4M3) SM_APP3(T, HD, 2);   \
    else if (cache->dtype == SM_F16) SM_APP3(T, HD, 1); \
    else SM_APP3(T, HD, 0);                             \
  } while (0)
#define SM_APP(T)                \
  do {                           \
    if (hd == 64) SM_APP2(T, 64); \
    else SM_APP2(T, 128);        \
  } while (0)
  if (dtype == SM_F32) SM_APP(float);
  else if (dtype == SM_BF16) SM_APP(uint16_t);
  else SM_APP(_Float16);
#undef SM_APP
#undef SM_APP2
#undef SM_APP3
  SM_LAUNCH_CHECK();
  return SM_OK;
}
