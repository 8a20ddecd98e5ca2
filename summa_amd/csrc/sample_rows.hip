// Next tokens from given random numbers, each row with its own temperature, top-k, top-p and
// min-p (sm_sample_rows; select_next_token / sample_from_values, summa-llm/src/generate.rs:127-250).
//
// w_i = exp((x_i - max) / T) in 64 bits, rounded to a whole number of 2^-46 (fewer for
// vocabularies past 2^17, so that a row's sum fits 63 bits). Sums of whole numbers do not
// depend on their order, so neither does which token the sum passes u at; in f32 one sum in a
// few hundred rows would fall on the other side of its border.
#include <cmath>
#include <type_traits>

#include "common.hpp"

namespace sm {
namespace {

constexpr int kThreads = 1024, kWaves = kThreads / kWave;

struct RowsArgs {
  const void* logits;
  int64_t ld;
  const float* uniforms;
  sm_row_sampling o;
  int32_t* tokens;
  float* logprobs;
  int vocab, bits;
};

__device__ inline uint32_t key_of(float f) {
  const uint32_t u = __float_as_uint(f + 0.f);  // (-0 is 0)
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

struct Cut {  // keys above T are kept, and those at T up to index `last`
  uint32_t T = 0;
  int last = 0x7fffffff;
  __device__ inline bool keeps(uint32_t key, int v) const {
    return key > T || (key == T && v <= last);
  }
};

struct Shared {
  unsigned long long hist[256], total;
  unsigned long long part[kWaves];
  float f[kWaves];
  int i[kWaves];
  int bin, last;
  unsigned long long left;
};

__device__ inline unsigned long long block_sum(unsigned long long x, Shared& sh) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o, kWave);
  if (threadIdx.x % kWave == 0) sh.part[threadIdx.x / kWave] = x;
  __syncthreads();
  unsigned long long s = 0;
  for (int i = 0; i < kWaves; ++i) s += sh.part[i];
  __syncthreads();
  return s;
}
__device__ inline unsigned long long block_before(unsigned long long x, Shared& sh,
                                                  unsigned long long& total) {
  const int lane = threadIdx.x % kWave, w = threadIdx.x / kWave;
  unsigned long long inc = x;
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const unsigned long long t = __shfl_up(inc, o, kWave);
    if (lane >= o) inc += t;
  }
  if (lane == kWave - 1) sh.part[w] = inc;
  __syncthreads();
  unsigned long long base = 0;
  total = 0;
  for (int i = 0; i < kWaves; ++i) {
    if (i < w) base += sh.part[i];
    total += sh.part[i];
  }
  __syncthreads();
  return base + inc - x;
}

template <typename T>
struct Row {
  const T* p;
  int vocab, bits;
  float m;
  double inv;
  __device__ inline float at(int v) const {
    float x;
    if constexpr (std::is_same<T, uint16_t>::value) x = bf16_to_f32(p[v]);
    else x = (float)p[v];
    return x == x ? x : -INFINITY;
  }
  __device__ inline double weight(float x) const {
    if (x == m) return 1.0;
    if (x == -INFINITY || m == INFINITY) return 0.0;
    return exp(((double)x - (double)m) * inv);
  }
  __device__ inline unsigned long long whole(float x) const {
    return (unsigned long long)rint(ldexp(weight(x), bits));
  }
};

// The place in (value, index) order up to which the elements kept by `outer` amount to
// `target`, counted or weighed.
template <bool MASS, typename T>
__device__ Cut select(const Row<T>& row, const Cut& outer, unsigned long long target, Shared& sh) {
  uint32_t prefix = 0, mask = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = threadIdx.x; i < 256; i += kThreads) sh.hist[i] = 0;
    __syncthreads();
    for (int v = threadIdx.x; v < row.vocab; v += kThreads) {
      const float x = row.at(v);
      const uint32_t key = key_of(x);
      if ((key & mask) != prefix || !outer.keeps(key, v)) continue;
      const unsigned long long w = MASS ? row.whole(x) : 1ull;
      if (w) atomicAdd(&sh.hist[key >> shift & 255u], w);
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      unsigned long long left = target;
      int b = 255;
      for (; b > 0 && sh.hist[b] < left; --b) left -= sh.hist[b];
      sh.bin = b;
      sh.left = left;
    }
    __syncthreads();
    prefix |= (uint32_t)sh.bin << shift;
    mask |= 255u << shift;
    target = sh.left;
    __syncthreads();
  }
  Cut c;
  c.T = prefix;
  if (threadIdx.x == 0) sh.last = 0x7fffffff;
  __syncthreads();
  unsigned long long before = 0;  // of the elements at the value, by index
  for (int v0 = 0; v0 < row.vocab; v0 += kThreads) {
    const int v = v0 + threadIdx.x;
    unsigned long long w = 0;
    if (v < row.vocab) {
      const float x = row.at(v);
      const uint32_t key = key_of(x);
      if (key == prefix && outer.keeps(key, v)) w = MASS ? row.whole(x) : 1ull;
    }
    unsigned long long total;
    const unsigned long long at = before + block_before(w, sh, total);
    if (w && at < target && at + w >= target) sh.last = v;
    before += total;
  }
  __syncthreads();
  c.last = sh.last;
  __syncthreads();
  return c;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_rows_kernel(RowsArgs a) {
  __shared__ Shared sh;
  const int r = (int)blockIdx.x, tid = threadIdx.x;
  Row<T> row;
  row.p = static_cast<const T*>(a.logits) + r * a.ld;
  row.vocab = a.vocab;
  row.bits = a.bits;
  const float temperature = a.o.temperatures ? a.o.temperatures[r] : a.o.temperature;
  const int top_k = a.o.top_ks ? a.o.top_ks[r] : a.o.top_k;
  const float top_p = a.o.top_ps ? a.o.top_ps[r] : a.o.top_p;
  const float min_p = a.o.min_ps ? a.o.min_ps[r] : a.o.min_p;
  // the largest, and the first place of it
  float m = -INFINITY;
  for (int v = tid; v < a.vocab; v += kThreads) m = fmaxf(m, row.at(v));
  m = wave_max(m);
  if (tid % kWave == 0) sh.f[tid / kWave] = m;
  __syncthreads();
  for (int i = 0; i < kWaves; ++i) m = fmaxf(m, sh.f[i]);
  __syncthreads();
  row.m = m;
  if (m == -INFINITY) {
    if (tid == 0) {
      a.tokens[r] = -1;
      if (a.logprobs) a.logprobs[r] = -INFINITY;
    }
    return;
  }
  float s = 0.f;
  int first = 0x7fffffff;
  for (int v = tid; v < a.vocab; v += kThreads) {
    const float x = row.at(v);
    s += x == m ? 1.f : m == INFINITY ? 0.f : __expf(x - m);
    if (x == m) first = min(first, v);
  }
  s = wave_sum(s);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) first = min(first, __shfl_xor(first, o, kWave));
  if (tid % kWave == 0) {
    sh.f[tid / kWave] = s;
    sh.i[tid / kWave] = first;
  }
  __syncthreads();
  s = 0.f;
  for (int i = 0; i < kWaves; ++i) {
    s += sh.f[i];
    first = min(first, sh.i[i]);
  }
  __syncthreads();
  int token = first;
  if (temperature > 0.f) {
    row.inv = 1.0 / (double)temperature;
    Cut ck, cp;
    if (top_k >= 1 && top_k < a.vocab) ck = select<false>(row, Cut{}, (unsigned long long)top_k, sh);
    if (top_p < 1.f) {
      unsigned long long w = 0;
      for (int v = tid; v < a.vocab; v += kThreads) {
        const float x = row.at(v);
        if (ck.keeps(key_of(x), v)) w += row.whole(x);
      }
      w = block_sum(w, sh);
      const double t = ceil((double)w * (double)top_p);
      cp = select<true>(row, ck, t < 1.0 ? 1ull : (unsigned long long)t, sh);
    }
    const double least = min_p > 0.f ? fmin((double)min_p, 1.0) : 0.0;
    auto kept = [&](int v, float x) {
      const uint32_t key = key_of(x);
      if (!ck.keeps(key, v) || !cp.keeps(key, v)) return 0ull;
      return least > 0.0 && row.weight(x) < least ? 0ull : row.whole(x);
    };
    unsigned long long w = 0;
    for (int v = tid; v < a.vocab; v += kThreads) w += kept(v, row.at(v));
    w = block_sum(w, sh);
    // whole numbers: the sum passes u w where it passes floor(u w)
    const double u = fmin(fmax((double)a.uniforms[r], 0.0), 1.0 - 0x1p-53);
    const unsigned long long u64 = (unsigned long long)(u * 0x1p64);
    const unsigned long long aim = __umul64hi(w, u64);
    if (tid == 0) sh.last = a.uniforms[r] > 0.f ? first : 0x7fffffff;
    unsigned long long before = 0;
    if (!(a.uniforms[r] > 0.f)) {
      // u = 0: the first of any weight, also of one that rounds to no 2^-46 (the least u above
      // it, 2^-24, is past the sum of all of those)
      __syncthreads();
      for (int v = tid; v < a.vocab; v += kThreads) {
        const float x = row.at(v);
        const uint32_t key = key_of(x);
        if (!ck.keeps(key, v) || !cp.keeps(key, v)) continue;
        const double y = row.weight(x);
        if (y > 0.0 && y >= least) atomicMin(&sh.last, v);
      }
      before = ~0ull;
    }
    for (int v0 = 0; v0 < a.vocab && before <= aim; v0 += kThreads) {
      const int v = v0 + tid;
      const unsigned long long x = v < a.vocab ? kept(v, row.at(v)) : 0ull;
      unsigned long long total;
      const unsigned long long at = before + block_before(x, sh, total);
      if (at <= aim && at + x > aim) sh.last = v;
      before += total;
    }
    __syncthreads();
    token = sh.last;
  }
  if (tid == 0) {
    a.tokens[r] = token;
    if (a.logprobs) a.logprobs[r] = (m == INFINITY ? 0.f : row.at(token) - m) - __logf(s);
  }
}

int check_rows(const char* who, int64_t rows, int64_t vocab, int dtype) {
  SM_REQUIRE(rows >= 0 && rows < (1 << 22) && vocab > 0 && vocab < (1 << 30),
             "%s: need 0 to 2^22 - 1 rows and 1 to 2^30 - 1 logits", who);
  SM_REQUIRE(dtype == SM_F32 || dtype == SM_BF16 || dtype == SM_F16,
             "%s: dtype must be SM_F32, SM_BF16 or SM_F16", who);
  return SM_OK;
}

}  // namespace
}  // namespace sm

using namespace sm;

extern "C" int64_t sm_sample_rows_workspace_bytes(int64_t rows, int64_t vocab, int dtype) {
  if (check_rows("sm_sample_rows_workspace_bytes", rows, vocab, dtype) != SM_OK) return -1;
  return 0;
}

extern "C" int sm_sample_rows(const void* logits, int dtype, int64_t rows, int64_t ld,
                              int64_t vocab, const float* uniforms, const sm_row_sampling* options,
                              int32_t* tokens, float* logprobs, void* workspace,
                              int64_t workspace_bytes, void* stream) {
  const char* me = "sm_sample_rows";
  SM_TRY(check_rows(me, rows, vocab, dtype));
  SM_REQUIRE(options, "%s: null options", me);
  SM_REQUIRE(ld >= vocab, "%s: ld must be at least vocab", me);
  SM_REQUIRE(options->temperatures || !std::isnan(options->temperature),
             "%s: temperature must not be NaN", me);
  SM_REQUIRE(options->top_ps || (options->top_p > 0.f && options->top_p <= 1.f),
             "%s: top_p must be in (0, 1]", me);
  SM_REQUIRE(options->min_ps || (options->min_p >= 0.f && options->min_p <= 1.f),
             "%s: min_p must be in [0, 1]", me);
  if (rows == 0) return SM_OK;
  SM_REQUIRE(logits && uniforms && tokens, "%s: null buffer", me);
  RowsArgs a;
  a.logits = logits;
  a.ld = ld;
  a.uniforms = uniforms;
  a.o = *options;
  a.tokens = tokens;
  a.logprobs = logprobs;
  a.vocab = (int)vocab;
  a.bits = 46;
  while (((int64_t)1 << (63 - a.bits)) < vocab) --a.bits;
  hipStream_t st = as_stream(stream);
  if (dtype == SM_F32) sample_rows_kernel<float><<<(unsigned)rows, kThreads, 0, st>>>(a);
  else if (dtype == SM_BF16) sample_rows_kernel<uint16_t><<<(unsigned)rows, kThreads, 0, st>>>(a);
  else sample_rows_kernel<_Float16><<<(unsigned)rows, kThreads, 0, st>>>(a);
  SM_LAUNCH_CHECK();
  return SM_OK;
}
