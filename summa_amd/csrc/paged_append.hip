// New keys and values into a paged KV cache, keys and queries rotated on the way.
//
//   project_qkv's split, RoPE and the AttnCache slice_assign
//   (summa-llm/src/model/attention.rs:142-177, 331-356) over the paged cache of
//   sm_paged_cache.
//
// One wave takes one head of one 16-token cache block: a block's scale is the maximum
// over its tokens, so the wave needs no other wave's values and no two waves write one
// scale. Lane (g, c) holds dims D c .. D c + D - 1 (D = head_dim / 16) of tokens 4 g .. 4 g + 3.
#include <cmath>

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
  int S, rows, max_rows, H, KVH, pages, cols, rot, half_layout, q_f16;
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
template <typename T, int D>
__device__ inline void store_dims(T* p, const float (&f)[D]) {
  if constexpr (D == 8) {
    store8<T>(p, f);
  } else {
    *reinterpret_cast<u32x2*>(p) = u32x2{round2<T>(f[0], f[1]), round2<T>(f[2], f[3])};
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

template <typename T, int HD, int CT>  // CT: cache type, 0 bf16, 1 f16, 2 e4m3
__global__ __launch_bounds__(256) void paged_append_kernel(AppendArgs a) {
  constexpr int D = HD / 16;
  int s = (int)blockIdx.x;
  const int slot = a.groups.mod(s) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int nth = a.touched.mod(s);  // of the blocks that the sequence's rows touch
  const PagedRows pr(a.row_start, s, a.rows, a.max_rows);
  const int first_slot = a.q ? 0 : a.H;
  if (slot + first_slot >= a.H + 2 * a.KVH || pr.n == 0) return;
  const int head = slot + first_slot;
  const int pos0 = a.pos0[s];
  const int64_t end = (int64_t)pos0 + pr.n;            // one past the last position
  const int64_t base = (int64_t)(max(pos0, 0) / kBlock + nth) * kBlock;
  const int t0 = (int)max((int64_t)max(pos0, 0) - base, (int64_t)0);
  const int t1 = (int)min(end - base, (int64_t)kBlock);
  if (t0 >= t1) return;  // (uniform: the wave's block holds none of the rows)
  const int lane = threadIdx.x % kWave, g = lane / 16, c = lane % 16, d0 = D * c;

  const bool is_q = head < a.H, is_k = !is_q && head < a.H + a.KVH;
  const int hd_at = (is_q ? head : is_k ? head - a.H : head - a.H - a.KVH);
  const T* src = static_cast<const T*>(is_q ? a.q : is_k ? a.k : a.v) + (int64_t)hd_at * HD;
  const int64_t ld = is_q ? a.ldq : is_k ? a.ldk : a.ldv;
  const int64_t row0 = pr.first + (base - pos0);  // the row of token 0 of the block
  float x[4][D];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int t = 4 * g + j;
    if (t >= t0 && t < t1) {
      load_dims<T, D>(src + (row0 + t) * ld + d0, x[j]);
    } else {
#pragma unroll
      for (int i = 0; i < D; ++i) x[j][i] = 0.f;
    }
  }
  if ((is_q || is_k) && d0 < a.rot) {
    const int half = a.rot / 2;
    const bool low = d0 < half;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int t = 4 * g + j;
      if (t < t0 || t >= t1) continue;
      if (a.half_layout) {
        float p[D], cs[D], sn[D];
        load_dims<T, D>(src + (row0 + t) * ld + (low ? d0 + half : d0 - half), p);
        load_angles<D>(a.rope, a.rope_rows, half, base + t, low ? d0 : d0 - half, cs, sn);
#pragma unroll
        for (int i = 0; i < D; ++i) {
          float u = low ? x[j][i] : p[i], w = low ? p[i] : x[j][i];
          rotate_pair(u, w, cs[i], sn[i]);
          x[j][i] = low ? u : w;
        }
      } else {
        float cs[D / 2], sn[D / 2];
        load_angles<D / 2>(a.rope, a.rope_rows, half, base + t, d0 / 2, cs, sn);
#pragma unroll
        for (int i = 0; i < D / 2; ++i) rotate_pair(x[j][2 * i], x[j][2 * i + 1], cs[i], sn[i]);
      }
    }
  }
  if (is_q) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int t = 4 * g + j;
      if (t < t0 || t >= t1) continue;
      const int64_t at = ((row0 + t) * a.H + head) * HD + d0;
      if (a.q_f16) store_dims<_Float16, D>(static_cast<_Float16*>(a.q_out) + at, x[j]);
      else store_dims<uint16_t, D>(static_cast<uint16_t*>(a.q_out) + at, x[j]);
    }
    return;
  }
  const int bi = paged_block(a.table + (int64_t)s * a.cols, a.cols, a.pages, a.KVH, hd_at, a.bpp,
                             (int)(base / kBlock));
  if (bi < 0) return;  // (uniform) no page for these tokens
  if constexpr (CT == 2) {
    float amax = 0.f;
    bool odd = false;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < D; ++i) {
        const float v = fabsf(x[j][i]);
        if (v < INFINITY) amax = fmaxf(amax, v);
        else odd = true;
      }
    int e = scale_exponent(wave_max(amax));
    uint8_t* sp = (is_k ? a.ks : a.vs) + bi;
    int old = e;
    if (t0 > 0) {
      old = (int)*sp - 127;
      e = max(e, old);
    }
    const bool grown = e > old;  // (uniform)
    const float again = pow2f(old - e), inv = pow2f(-e);
    if (lane == 0) *sp = (uint8_t)(e + 127);
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < D; ++i) x[j][i] *= inv;
    uint8_t* page = (is_k ? a.kc : a.vc) + (size_t)bi * (kBlock * HD);
    // infinities and NaN are the NaN code: the scale is that of the finite values
    auto nan4 = [&](uint32_t w, float p, float q, float r, float z) {
      const float y[4] = {p, q, r, z};
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (!(fabsf(y[i]) < INFINITY)) w = (w & ~(0xffu << (8 * i))) | (0x7fu << (8 * i));
      return w;
    };
    const bool any_odd = __ballot(odd) != 0;
    if (is_k) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int t = 4 * g + j;
        uint32_t* p = reinterpret_cast<uint32_t*>(page + t * HD + d0);
        if (t >= t0 && t < t1) {
          uint32_t w[D / 4];
#pragma unroll
          for (int i = 0; i < D / 4; ++i) {
            w[i] = pack_e4m3(x[j][4 * i], x[j][4 * i + 1], x[j][4 * i + 2], x[j][4 * i + 3]);
            if (any_odd)
              w[i] = nan4(w[i], x[j][4 * i], x[j][4 * i + 1], x[j][4 * i + 2], x[j][4 * i + 3]);
          }
          if constexpr (D == 8) *reinterpret_cast<u32x2*>(p) = u32x2{w[0], w[1]};
          else *p = w[0];
        } else if (t < t0 && grown) {
#pragma unroll
          for (int i = 0; i < D / 4; ++i) p[i] = rescale_e4m3(p[i], again);
        }
      }
    } else {
      uint32_t mine = 0, older = 0;  // bytes of the quad: the call's tokens, earlier ones
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int t = 4 * g + j;
        if (t >= t0 && t < t1) mine |= 0xffu << (8 * j);
        if (t < t0) older |= 0xffu << (8 * j);
      }
      if (mine || (grown && older)) {
#pragma unroll
        for (int i = 0; i < D; ++i) {
          const int d = d0 + i, n = d / 16;
          uint32_t* p =
              reinterpret_cast<uint32_t*>(page + ((n / 4 * 4 + g) * 16 + d % 16) * 16 + n % 4 * 4);
          uint32_t w = pack_e4m3(x[0][i], x[1][i], x[2][i], x[3][i]);
          if (any_odd) w = nan4(w, x[0][i], x[1][i], x[2][i], x[3][i]);
          if (~mine) {
            uint32_t was = *p;
            if (grown) was = (was & ~older) | (rescale_e4m3(was, again) & older);
            w = (w & mine) | (was & ~mine);
          }
          *p = w;
        }
      }
    }
  } else {
    typedef typename std::conditional<CT == 1, _Float16, uint16_t>::type TC;
    TC* page = reinterpret_cast<TC*>(is_k ? a.kc : a.vc) + (size_t)bi * (kBlock * HD);
    if (is_k) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int t = 4 * g + j;
        if (t >= t0 && t < t1) store_dims<TC, D>(page + t * HD + d0, x[j]);
      }
    } else {
      uint32_t m01 = 0, m23 = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int t = 4 * g + j;
        if (t >= t0 && t < t1) (j < 2 ? m01 : m23) |= 0xffffu << (16 * (j % 2));
      }
      if (m01 | m23) {
#pragma unroll
        for (int i = 0; i < D; ++i) {
          const int d = d0 + i, n = d / 16;
          u32x2* p = reinterpret_cast<u32x2*>(page + ((n / 2 * 4 + g) * 16 + d % 16) * 8 + n % 2 * 4);
          u32x2 w = {round2<TC>(x[0][i], x[1][i]), round2<TC>(x[2][i], x[3][i])};
          if (~(m01 & m23)) {
            const u32x2 was = *p;
            w = (w & u32x2{m01, m23}) | (was & u32x2{~m01, ~m23});
          }
          *p = w;
        }
      }
    }
  }
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
    SM_REQUIRE(rope_rows >= 0 && reinterpret_cast<uintptr_t>(rope_table) % 16 == 0,
               "%s: rope_table must be 16-byte aligned", me);
  }
  if (S == 0 || max_rows == 0) return SM_OK;
  SM_REQUIRE(block_table && pos0 && k && v && (!q || q_out), "%s: null buffer", me);
  SM_REQUIRE(table_cols > 0 && table_cols <= most, "%s: table_cols must be positive", me);
  SM_REQUIRE(row_start || rows == S * max_rows,
             "%s: without row_start, rows must be S * max_rows", me);
  const int64_t each = dtype == SM_F32 ? 4 : 8;  // values of 16 bytes
  SM_REQUIRE(ldk >= KVH * hd && ldv >= KVH * hd && ldk % each == 0 && ldv % each == 0 &&
                 (!q || (ldq >= H * hd && ldq % each == 0)),
             "%s: rows must be 16-byte aligned and hold their heads", me);
  if (q) {
    const uintptr_t qa = reinterpret_cast<uintptr_t>(q), oa = reinterpret_cast<uintptr_t>(q_out);
    SM_REQUIRE(qa + (size_t)(((rows - 1) * ldq + H * hd) * (16 / each)) <= oa ||
                   oa + (size_t)(rows * H * hd * 2) <= qa,
               "%s: q_out must not overlap q", me);
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
  a.groups = Divide((int)ceil_div(a.H + 2 * KVH, 4));
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
