// Rotary positions: the angle table (with the scalings for long contexts) and the
// rotation of query and key heads, forward and gradient.
//
//   MultiHeadAttention's RoPE (summa-llm/src/model/attention.rs:142-177), in adjacent
//   pairs and in the half-split layout, over the whole head or its first rot_dim dims.
#include <cmath>

#include "common.hpp"
#include "rotary.hpp"

namespace sm {
namespace {

// One thread per (position, pair). Angles in f64: position * frequency passes 2^20 turns'
// worth of radians at long contexts, where f32 would leave 4 of its 24 bits after the
// point. Written once per context length; not a hot kernel: 2^20 positions of 64 pairs (537 MB)
// 0.54 ms, 1.0 TB/s, 0.62 by parts, bound by the f64 power and sine of every element.
__global__ __launch_bounds__(256) void rope_table_kernel(double theta, int half, int kind,
                                                         double factor, double original,
                                                         double lo, double hi, double magnitude,
                                                         int64_t n, float2* __restrict__ table) {
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (id >= n) return;
  const int p = (int)(id % half);
  const double pos = (double)(id / half);
  double f = pow(theta, -(double)p / (double)half);
  if (kind == SM_ROPE_SCALE_LINEAR) {
    f /= factor;
  } else if (kind == SM_ROPE_SCALE_PARTS) {
    const double turns = original * f / 6.283185307179586476925286766559;
    const double keep = fmin(1.0, fmax(0.0, (turns - lo) / (hi - lo)));
    f = (1.0 - keep) * (f / factor) + keep * f;
  }
  double s, c;
  sincos(pos * f, &s, &c);
  table[id] = float2{(float)(c * magnitude), (float)(s * magnitude)};
}

// One wave per row at a time; a lane takes the same two 8-dim chunks of every head it
// visits (chunk u and its partner: the other half of its pairs in the half layout, the
// chunk units later otherwise), so a row's cosines and sines are read once for all heads.
template <typename T, bool HALF>
__global__ __launch_bounds__(256) void rope_kernel(const T* x, int64_t ldx,
                                                   T* y, int64_t ldy,
                                                   const float* __restrict__ table,
                                                   int64_t table_rows,
                                                   const int32_t* __restrict__ positions,
                                                   int64_t rows, int heads, int hd, int rot,
                                                   float sign) {
  const int64_t row = (int64_t)blockIdx.x * 4 + threadIdx.x / kWave;
  if (row >= rows) return;
  const int lane = threadIdx.x % kWave;
  const int units = hd / 16, hpp = kWave / units;  // lanes of a head, heads of a pass
  const int u = lane % units, h0 = lane / units;
  if (h0 >= hpp) return;
  const int half = rot / 2, ru = rot / 16;  // units of the rotated part
  // chunks at dims d0 and d1
  const bool turn0 = HALF ? u < ru : 8 * u < rot;
  const int d0 = HALF ? (u < ru ? 8 * u : rot + 8 * (u - ru)) : 8 * u;
  const int d1 = HALF ? (u < ru ? d0 + half : d0 + (hd - rot) / 2) : d0 + hd / 2;
  const bool turn1 = HALF ? turn0 : d1 < rot;
  constexpr int N = HALF ? 8 : 4;
  float c0[N], s0[N], c1[4], s1[4];
  const int64_t pos = positions[row];
  // (dims that are not rotated read the first pairs' angles and do not use them)
  load_angles<N>(table, table_rows, half, pos, !turn0 ? 0 : HALF ? d0 : d0 / 2, c0, s0);
  if (!HALF) load_angles<4>(table, table_rows, half, pos, turn1 ? d1 / 2 : 0, c1, s1);
  const T* xr = x + row * ldx;
  T* yr = y + row * ldy;
  for (int h = h0; h < heads; h += 2 * hpp) {  // two heads' loads in flight
    float a[2][8], b[2][8];
    const bool second = h + hpp < heads;
    load8<T>(xr + (int64_t)h * hd + d0, a[0]);
    load8<T>(xr + (int64_t)h * hd + d1, b[0]);
    if (second) {
      load8<T>(xr + (int64_t)(h + hpp) * hd + d0, a[1]);
      load8<T>(xr + (int64_t)(h + hpp) * hd + d1, b[1]);
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (k && !second) break;
      if constexpr (HALF) {
        if (turn0)
#pragma unroll
          for (int i = 0; i < 8; ++i) rotate_pair(a[k][i], b[k][i], c0[i], s0[i] * sign);
      } else {
        if (turn0)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            rotate_pair(a[k][2 * i], a[k][2 * i + 1], c0[i], s0[i] * sign);
        if (turn1)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            rotate_pair(b[k][2 * i], b[k][2 * i + 1], c1[i], s1[i] * sign);
      }
      store8<T>(yr + (int64_t)(h + k * hpp) * hd + d0, a[k]);
      store8<T>(yr + (int64_t)(h + k * hpp) * hd + d1, b[k]);
    }
  }
}

}  // namespace
}  // namespace sm

extern "C" int sm_rope_table(double theta, int64_t rot_dim, int64_t positions, int scaling,
                             double factor, double original_positions, double low_turns,
                             double high_turns, double magnitude, float* table, void* stream) {
  using namespace sm;
  SM_REQUIRE(std::isfinite(theta) && theta > 0, "sm_rope_table: theta must be finite and positive");
  SM_REQUIRE(rot_dim > 0 && rot_dim % 2 == 0 && rot_dim <= 65536,
             "sm_rope_table: rot_dim must be even, 2 to 65536");
  SM_REQUIRE(positions >= 0 && positions <= 0x7fffffff,
             "sm_rope_table: positions must be in 0..2^31 - 1");
  SM_REQUIRE(scaling == SM_ROPE_SCALE_NONE || scaling == SM_ROPE_SCALE_LINEAR ||
                 scaling == SM_ROPE_SCALE_THETA || scaling == SM_ROPE_SCALE_PARTS,
             "sm_rope_table: unknown scaling %d", scaling);
  SM_REQUIRE(std::isfinite(magnitude) && magnitude > 0,
             "sm_rope_table: magnitude must be finite and positive");
  if (scaling != SM_ROPE_SCALE_NONE)
    SM_REQUIRE(std::isfinite(factor) && factor > 0, "sm_rope_table: factor must be finite and positive");
  if (scaling == SM_ROPE_SCALE_THETA)
    SM_REQUIRE(rot_dim > 2, "sm_rope_table: a scaled theta needs rot_dim > 2");
  if (scaling == SM_ROPE_SCALE_PARTS)
    SM_REQUIRE(std::isfinite(original_positions) && original_positions > 0 &&
                   std::isfinite(low_turns) && std::isfinite(high_turns) && low_turns < high_turns,
               "sm_rope_table: scaling by parts needs original_positions > 0 and low_turns < "
               "high_turns");
  if (positions == 0) return SM_OK;
  SM_REQUIRE(table, "sm_rope_table: null buffer");
  const int64_t half = rot_dim / 2, n = positions * half;
  if (ceil_div(n, 256) >= (1 << 24)) {
    set_error("sm_rope_table: problem too large");
    return SM_ERR_UNSUPPORTED;
  }
  if (scaling == SM_ROPE_SCALE_THETA)
    theta *= std::pow(factor, (double)rot_dim / (double)(rot_dim - 2));
  rope_table_kernel<<<(unsigned)ceil_div(n, 256), 256, 0, as_stream(stream)>>>(
      theta, (int)half, scaling, factor, original_positions, low_turns, high_turns, magnitude, n,
      reinterpret_cast<float2*>(table));
  SM_LAUNCH_CHECK();
  return SM_OK;
}

extern "C" int sm_rope(const void* x, int64_t ldx, void* y, int64_t ldy, int dtype,
                       const float* table, int64_t table_rows, const int32_t* positions,
                       int64_t rows, int64_t heads, int64_t head_dim, int64_t rot_dim, int layout,
                       int backward, void* stream) {
  using namespace sm;
  SM_REQUIRE(dtype == SM_F32 || dtype == SM_BF16 || dtype == SM_F16,
             "sm_rope: dtype must be SM_F32, SM_BF16 or SM_F16");
  SM_REQUIRE(layout == SM_ROPE_INTERLEAVED || layout == SM_ROPE_HALF,
             "sm_rope: layout must be SM_ROPE_INTERLEAVED or SM_ROPE_HALF");
  // (four rows a workgroup, and a grid holds less than 2^24 workgroups of 256 threads)
  SM_REQUIRE(rows >= 0 && rows < ((int64_t)1 << 26) - 4 && heads > 0 && heads <= 65535,
             "sm_rope: need 0 <= rows < 2^26 - 4 and 0 < heads <= 65535");
  SM_REQUIRE(head_dim >= 16 && head_dim % 16 == 0 && head_dim <= 1024,
             "sm_rope: head_dim must be a multiple of 16 up to 1024");
  SM_REQUIRE(rot_dim >= 16 && rot_dim % 16 == 0 && rot_dim <= head_dim,
             "sm_rope: rot_dim must be a multiple of 16 up to head_dim");
  SM_REQUIRE(table_rows > 0, "sm_rope: the table has no rows");
  const int64_t size = dtype == SM_F32 ? 4 : 2, each = 16 / size, width = heads * head_dim;
  SM_REQUIRE(ldx >= width && ldy >= width && ldx % each == 0 && ldy % each == 0 &&
                 ldx < ((int64_t)1 << 31) && ldy < ((int64_t)1 << 31),
             "sm_rope: rows must be 16-byte aligned and hold heads * head_dim values");
  if (rows == 0) return SM_OK;
  SM_REQUIRE(x && y && table && positions, "sm_rope: null buffer");
  const uintptr_t xa = reinterpret_cast<uintptr_t>(x), ya = reinterpret_cast<uintptr_t>(y);
  SM_REQUIRE(xa % 16 == 0 && ya % 16 == 0 && reinterpret_cast<uintptr_t>(table) % 16 == 0,
             "sm_rope: x, y and table must be 16-byte aligned");
  const uintptr_t xe = xa + ((rows - 1) * ldx + width) * size,
                  ye = ya + ((rows - 1) * ldy + width) * size;
  SM_REQUIRE((xa == ya && ldx == ldy) || xe <= ya || ye <= xa,
             "sm_rope: y is x, row for row, or does not overlap it");
  const unsigned blocks = (unsigned)ceil_div(rows, 4);
  const float sign = backward ? -1.f : 1.f;
  hipStream_t st = as_stream(stream);
#define SM_ROPE2(T, HALF)                                                                     \
  rope_kernel<T, HALF><<<blocks, 256, 0, st>>>((const T*)x, ldx, (T*)y, ldy, table,           \
                                               table_rows, positions, rows, (int)heads,       \
                                               (int)head_dim, (int)rot_dim, sign)
#define SM_ROPE1(T)                                     \
  do {                                                  \
    if (layout == SM_ROPE_HALF) SM_ROPE2(T, true);      \
    else SM_ROPE2(T, false);                            \
  } while (0)
  if (dtype == SM_F32) SM_ROPE1(float);
  else if (dtype == SM_BF16) SM_ROPE1(uint16_t);
  else SM_ROPE1(_Float16);
#undef SM_ROPE1
#undef SM_ROPE2
  SM_LAUNCH_CHECK();
  return SM_OK;
}
