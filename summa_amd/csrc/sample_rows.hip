// Next tokens from given random numbers, each row with its own temperature, top-k, top-p and
// min-p (sm_sample_rows; select_next_token / sample_from_values, summa-llm/src/generate.rs:127-250).
//
// The token is decided by where u falls among running sums of w_i = exp((x_i - max) / T): with
// sums in f32 (2^-20 of the whole off) one row in a few hundred of a flat distribution over 65536
// logits would take a neighbour. Weights and sums are held in 64 bits where they decide, in a fixed order,
// and in f32 where they only say where to look.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "common.hpp"

namespace sm {
namespace {

struct RowsArgs {
  const void* logits;
  int64_t ld;
  const float* uniforms;
  sm_row_sampling o;
  int32_t* tokens;
  float* logprobs;
  int vocab;
  int steps;  // slots of a wave
  int parts;  // workgroups of a row
  uint8_t* ws;
};

__device__ inline uint32_t key_of(float f) {
  const uint32_t u = __float_as_uint(f + 0.f);  // (-0 is 0)
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__device__ inline float key_value(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k ^ 0x80000000u) : ~k);
}

struct Cut {  // keys above T are kept, and those at T up to index `last`
  uint32_t T = 0;
  int last = 0x7fffffff;
  __device__ inline bool keeps(uint32_t key, int v) const {
    return key > T || (key == T && v <= last);
  }
};

// What is called for every step, and what takes the rows' state by reference, is not left to the
// compiler's measure of size: a call puts that in scratch (256 rows of 65536 with top-p 52 -> 72 us).
#define SM_INLINE __attribute__((always_inline)) inline

// Sums of weights by atomics, in any order: whole numbers of 128 bits, in units of 2^-96 of the
// largest weight, so that the sums of 2^30 logits hold and are off by less than 2^-66 of it.
struct Wide {
  unsigned long long hi, lo;
  __device__ inline bool less(const Wide& o) const { return hi < o.hi || (hi == o.hi && lo < o.lo); }
  __device__ inline void add(const Wide& o) {
    lo += o.lo;
    hi += o.hi + (lo < o.lo);
  }
  __device__ inline void take(const Wide& o) {
    hi -= o.hi + (lo < o.lo);
    lo -= o.lo;
  }
  __device__ inline Wide times(unsigned long long c) const { return {hi * c + __umul64hi(lo, c), lo * c}; }
  __device__ inline double value() const { return (double)hi * 0x1p64 + (double)lo; }
  __device__ static inline Wide of(double x) {  // its whole part, x < 2^127
    const unsigned long long hi = (unsigned long long)(x * 0x1p-64);
    return {hi, (unsigned long long)(x - (double)hi * 0x1p64)};
  }
};

// Sums of weights in a fixed order, in f64 with what each addition rounds off beside them: a row of
// 2^30 logits is 2^20 additions a thread.
struct Sum {
  double s = 0.0, rest = 0.0;
  __device__ inline void add(double x) {
    const double t = s + x, y = t - s;
    rest += (s - (t - y)) + (x - y);
    s = t;
  }
  __device__ inline double value() const { return s + rest; }
};

template <int THREADS>
struct Shared {
  unsigned long long hist[256], high[256];
  unsigned long long part[THREADS / kWave];
  double f[THREADS / kWave], rest[THREADS / kWave];
  int i[THREADS / kWave];
  int bin, last;
  Wide left;
};

template <int THREADS>
__device__ inline Wide block_sum(Wide x, Shared<THREADS>& sh) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x.add({__shfl_xor(x.hi, o, kWave), __shfl_xor(x.lo, o, kWave)});
  if (threadIdx.x % kWave == 0) {
    sh.hist[threadIdx.x / kWave] = x.lo;
    sh.high[threadIdx.x / kWave] = x.hi;
  }
  __syncthreads();
  Wide s{0, 0};
  for (int i = 0; i < THREADS / kWave; ++i) s.add({sh.high[i], sh.hist[i]});
  __syncthreads();
  return s;
}
template <int THREADS>
__device__ inline double block_sum(Sum x, Shared<THREADS>& sh) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const double rest = __shfl_xor(x.rest, o, kWave);
    x.add(__shfl_xor(x.s, o, kWave));
    x.rest += rest;
  }
  if (threadIdx.x % kWave == 0) {
    sh.f[threadIdx.x / kWave] = x.s;
    sh.rest[threadIdx.x / kWave] = x.rest;
  }
  __syncthreads();
  Sum s;
  for (int i = 0; i < THREADS / kWave; ++i) {
    s.add(sh.f[i]);
    s.rest += sh.rest[i];
  }
  __syncthreads();
  return s.value();
}
template <int THREADS>
__device__ inline unsigned long long block_before(unsigned long long x, Shared<THREADS>& sh,
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
  for (int i = 0; i < THREADS / kWave; ++i) {
    if (i < w) base += sh.part[i];
    total += sh.part[i];
  }
  __syncthreads();
  return base + inc - x;
}
// Up to and with this thread's.
template <int THREADS>
__device__ inline double block_inclusive(double x, Shared<THREADS>& sh, double& total) {
  const int lane = threadIdx.x % kWave, w = threadIdx.x / kWave;
  double inc = x;
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const double t = __shfl_up(inc, o, kWave);
    if (lane >= o) inc += t;
  }
  if (lane == kWave - 1) sh.f[w] = inc;
  __syncthreads();
  double base = 0.0;
  total = 0.0;
  for (int i = 0; i < THREADS / kWave; ++i) {
    if (i < w) base += sh.f[i];
    total += sh.f[i];
  }
  __syncthreads();
  return base + inc;
}

template <typename T>
struct Row {
  const T* p;
  int vocab;
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
  __device__ inline Wide whole(float x) const { return Wide::of(weight(x) * 0x1p96); }
};

// The place in (value, index) order up to which the elements kept by `outer` amount to
// `target`, counted or weighed.
template <bool MASS, int THREADS, typename T>
__device__ Cut select(const Row<T>& row, const Cut& outer, Wide target, Shared<THREADS>& sh) {
  uint32_t prefix = 0, mask = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = threadIdx.x; i < 256; i += THREADS) sh.hist[i] = sh.high[i] = 0;
    __syncthreads();
    for (int v = threadIdx.x; v < row.vocab; v += THREADS) {
      const float x = row.at(v);
      const uint32_t key = key_of(x);
      if ((key & mask) != prefix || !outer.keeps(key, v)) continue;
      const uint32_t bin = key >> shift & 255u;
      Wide w{0, 1};
      if constexpr (MASS) w = row.whole(x);
      if (w.lo) {
        const unsigned long long old = atomicAdd(&sh.hist[bin], w.lo);
        w.hi += old + w.lo < old;
      }
      if (w.hi) atomicAdd(&sh.high[bin], w.hi);
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      Wide left = target;
      int b = 255;
      for (; b > 0 && Wide{sh.high[b], sh.hist[b]}.less(left); --b) left.take({sh.high[b], sh.hist[b]});
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
  // of the elements at the value, which all weigh the same, the least count that amounts to it
  unsigned long long need = target.lo;
  if constexpr (MASS) {
    const Wide w = row.whole(key_value(prefix));
    unsigned long long lo = 1, hi = 1ull << 30;
    while (lo < hi) {
      const unsigned long long mid = (lo + hi) / 2;
      if (w.times(mid).less(target)) lo = mid + 1;
      else hi = mid;
    }
    need = lo;
  }
  if (threadIdx.x == 0) sh.last = 0x7fffffff;
  __syncthreads();
  unsigned long long before = 0;  // of the elements at the value, by index
  for (int v0 = 0; v0 < row.vocab && before < need; v0 += THREADS) {
    const int v = v0 + threadIdx.x;
    unsigned long long w = 0;
    if (v < row.vocab) {
      const uint32_t key = key_of(row.at(v));
      w = key == prefix && outer.keeps(key, v);
    }
    unsigned long long total;
    const unsigned long long at = before + block_before(w, sh, total);
    if (w && at + 1 == need) sh.last = v;
    before += total;
  }
  __syncthreads();
  c.last = sh.last;
  __syncthreads();
  return c;
}

// One row by passes over memory: takes every row, and is what rows that the kernel below does not
// hold in its lists come to. Bound by its passes, each with an exponential in f64 for every logit.
template <int THREADS, typename T>
__device__ SM_INLINE void by_passes(const RowsArgs& a, int r, const Row<T>& row, int top_k, float top_p,
                          float min_p, Shared<THREADS>& sh) {
  const int tid = threadIdx.x;
  int first = 0x7fffffff;
  Sum s;
  for (int v = tid; v < a.vocab; v += THREADS) {
    const float x = row.at(v);
    s.s += (double)(x == row.m ? 1.f : row.m == INFINITY ? 0.f : __expf(x - row.m));
    if (x == row.m) first = min(first, v);
  }
  const float exps = (float)block_sum(s, sh);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) first = min(first, __shfl_xor(first, o, kWave));
  if (tid % kWave == 0) sh.i[tid / kWave] = first;
  __syncthreads();
  for (int i = 0; i < THREADS / kWave; ++i) first = min(first, sh.i[i]);
  __syncthreads();
  int token = first;
  if (row.inv > 0.0 || row.inv == 0.0) {  // (not greedy: NaN)
    Cut ck, cp;
    if (top_k >= 1 && top_k < a.vocab)
      ck = select<false, THREADS>(row, Cut{}, Wide{0, (unsigned long long)top_k}, sh);
    if (top_p < 1.f) {
      Wide w{0, 0};
      for (int v = tid; v < a.vocab; v += THREADS) {
        const float x = row.at(v);
        if (ck.keeps(key_of(x), v)) w.add(row.whole(x));
      }
      w = block_sum(w, sh);
      const double t = ceil(w.value() * (double)top_p);
      cp = select<true, THREADS>(row, ck, t < 1.0 ? Wide{0, 1} : Wide::of(t), sh);
    }
    const double least = min_p > 0.f ? fmin((double)min_p, 1.0) : 0.0;
    auto kept = [&](int v) {
      const float x = row.at(v);
      const uint32_t key = key_of(x);
      if (!ck.keeps(key, v) || !cp.keeps(key, v)) return 0.0;
      const double w = row.weight(x);
      return w < least ? 0.0 : w;
    };
    Sum w;
    int last = -1;  // (where the sums below come to less than u = 1 - 2^-53 of this one)
    for (int v = tid; v < a.vocab; v += THREADS) {
      const double x = kept(v);
      w.add(x);
      if (x > 0.0) last = v;
    }
    const double u = fmin(fmax((double)a.uniforms[r], 0.0), 1.0 - 0x1p-53);
    const double aim = fmax(u * block_sum(w, sh), 0x1p-900);
    if (tid == 0) {
      sh.last = 0x7fffffff;
      sh.bin = -1;
    }
    __syncthreads();
    if (last >= 0) atomicMax(&sh.bin, last);
    // four logits a thread and step: what passes is looked for in the first thread's that does
    constexpr int PER = 4;
    Sum before;
    token = 0x7fffffff;
    for (int v0 = 0; v0 < a.vocab && token == 0x7fffffff; v0 += PER * THREADS) {
      double x[PER], part = 0.0, total;
#pragma unroll
      for (int e = 0; e < PER; ++e) {
        const int v = v0 + tid * PER + e;
        x[e] = v < a.vocab ? kept(v) : 0.0;
        part += x[e];
      }
      const double inc = block_inclusive(part, sh, total);
      const double left = (aim - before.s) - before.rest;
      if (part > 0.0 && inc > left) {
        double at = inc - part;
        int got = -1;
        bool passed = false;
#pragma unroll
        for (int e = 0; e < PER; ++e) {
          at += x[e];
          if (x[e] > 0.0 && !passed) got = e;
          passed |= x[e] > 0.0 && at > left;
        }
        atomicMin(&sh.last, v0 + tid * PER + got);
      }
      __syncthreads();
      token = sh.last;
      before.add(total);
    }
    if (token == 0x7fffffff) token = sh.bin;
  }
  if (tid == 0) {
    a.tokens[r] = token;
    if (a.logprobs)
      a.logprobs[r] = (row.m == INFINITY ? 0.f : row.at(token) - row.m) - __logf(exps);
  }
}

// Four at a time, step by step: left to itself the compiler makes one after the other, and each
// operation waits for the one before it.
__device__ SM_INLINE void side_by_side(double (&x)[4]) {
  asm volatile("" : "+v"(x[0]), "+v"(x[1]), "+v"(x[2]), "+v"(x[3]));
}
// 2^(d c), d <= 0, d c >= -1022: a polynomial of degree 9 on the half octave to either side of a whole
// one (interpolated at the Chebyshev nodes; 2^-44.59 off at its ends). Beside it c, a quotient and a
// product that are rounded, is off by 2^-51.7 of itself, which every octave adds to: 2^-44 of the weight down
// to 2^-80 of the largest, 2^-42 at the least.
__device__ SM_INLINE void exp2_f64(const double (&d)[4], double c, double (&p)[4]) {
  constexpr double magic = 0x1.8p52;
  constexpr double co[] = {0x1.63ef9699120e2p-20, 0x1.ffcb767842e11p-17, 0x1.43088e2580989p-13,
                           0x1.5d87fe908fb19p-10, 0x1.3b2ab72b175e1p-7,  0x1.c6b08d7044117p-5,
                           0x1.ebfbdff8149f2p-3,  0x1.62e42fefa39f7p-1,  1.0};
  double t[4], r[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) t[i] = fma(d[i], c, magic);
  side_by_side(t);
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = t[i] - magic;
  side_by_side(r);
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = fma(d[i], c, -r[i]);
  side_by_side(r);
#pragma unroll
  for (int i = 0; i < 4; ++i) p[i] = fma(r[i], 0x1.b6571e229927fp-24, co[0]);
#pragma unroll
  for (int k = 1; k < 9; ++k) {
    side_by_side(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = fma(p[i], r[i], co[k]);
  }
  side_by_side(p);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    p[i] = __builtin_amdgcn_ldexp(p[i], (int)(uint32_t)__builtin_bit_cast(uint64_t, t[i]));
}
__device__ inline double exp2_f64(double d, double c) {
  const double x[4] = {d, d, d, d};
  double p[4];
  exp2_f64(x, c, p);
  return p[0];
}

__device__ inline uint64_t ballot(bool x) { return __builtin_amdgcn_ballot_w64(x); }

template <int CTRL>
__device__ inline double dpp_f64(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, 0xF, 0xF, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, 0xF, 0xF, false);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ inline double lane_f64(double v, int l) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)u, l);
  const uint32_t hi = __builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), l);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ inline double wave_add(double v) {  // (as wave_sum)
  v += dpp_f64<kDppXor1>(v);
  v += dpp_f64<kDppXor2>(v);
  v += dpp_f64<kDppHalfMirror>(v);
  v += dpp_f64<kDppMirror>(v);
  return (lane_f64(v, 0) + lane_f64(v, 16)) + (lane_f64(v, 32) + lane_f64(v, 48));
}
__device__ inline double wave_inclusive(double v) {
  const int lane = threadIdx.x % kWave;
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const double t = __shfl_up(v, o, kWave);
    if (lane >= o) v += t;
  }
  return v;
}

constexpr float kLog2e = 1.44269504088896340736f;
constexpr int kSlot = 512;   // consecutive logits, a wave's share of a step: a sum of its own
constexpr int kSlots = 512;  // sums held: rows of up to 262144 logits
constexpr float kOctaves = 40.f;  // that the bins cover

template <int THREADS>
struct RowLds {
  static constexpr int BINS = THREADS >= 512 ? 4096 : 1024;
  static constexpr int CAP = THREADS >= 512 ? 1024 : 512;  // candidates held
  uint32_t bin[BINS + kWave];
  unsigned long long own[THREADS / kWave][CAP / (THREADS / kWave)];
  union {
    struct {
      unsigned long long key[CAP];  // order key, ~index
      double w[CAP];
      int rank[CAP];                // how many come before: by value, and by index (high half)
      uint16_t order[CAP], place[CAP];  // the list by value, by index
    } c;
    Shared<THREADS> passes;
  };
  double slot[THREADS >= 512 ? kSlots : 64];
  double all[THREADS / kWave], above[THREADS / kWave];
  float m[THREADS / kWave], s[THREADS / kWave], w[THREADS / kWave], low[THREADS / kWave];
  int n[THREADS / kWave];
  uint32_t part[THREADS / kWave];
  int lo, hi, listed;
};

// A row in the registers of a workgroup: wave w has the slots w steps .., a slot a step; of each
// quarter (f32) or all (16 bits) of 1 KB of it lane l has 16 bytes. Steps past STEPS are read again at each use.
template <typename T, int THREADS, int STEPS>
struct Held {
  static constexpr int G = 16 / sizeof(T);   // logits of a lane's 16 bytes
  static constexpr int W = 8 / G;            // 16-byte pieces of a step
  const T* p;
  int vocab, steps, first;  // first: of this wave
  // The row as vectors of registers that a uniform index reaches: a loop over the steps is a loop
  // in the code too. (Unrolled, a pass over 64-bit weights is 12 KB of it, and fetching the code
  // took most of the kernel's time.)
  static constexpr int R = STEPS * W * 4 < 32 ? 16 : 32, V = (STEPS * W * 4 + R - 1) / R;
  typedef uint32_t Vec __attribute__((ext_vector_type(R)));
  Vec reg[V];

  struct __attribute__((packed, aligned(2))) Piece {
    u32x4 w;
  };
  // Where a piece lies: at the row's end, where it would pass that, and the first `skip` of it are
  // then others'.
  __device__ inline int place(int step, int i, int& skip) const {
    const int base = first + step * kSlot + (i * kWave + (int)(threadIdx.x % kWave)) * G;
    const int at = min(base, vocab - G);
    skip = base - at;
    return at;
  }
  __device__ inline void read(int step, u32x4 (&w)[W]) const {
#pragma unroll
    for (int i = 0; i < W; ++i) {
      int skip;
      w[i] = reinterpret_cast<const Piece*>(p + place(step, i, skip))->w;
    }
  }
  __device__ inline void load() {
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      u32x4 w[W] = {};
      if (i < steps) read(i, w);
#pragma unroll
      for (int j = 0; j < 4 * W; ++j) reg[(i * 4 * W + j) / R][(i * 4 * W + j) % R] = w[j / 4][j % 4];
    }
  }
  // The values of a step, eight a lane, piece after piece; what is less than `floor`, not the lane's, or NaN
  // is `floor`. CLEAN: without NaN.
  template <bool CLEAN>
  __device__ SM_INLINE void values(const u32x4 (&w)[W], int step, float floor, float (&x)[8]) const {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if constexpr (W == 2)
        x[e] = __uint_as_float(w[e / 4][e % 4]);
      else if constexpr (std::is_same<T, uint16_t>::value)
        x[e] = e % 2 ? bf16hi(w[0][e / 2]) : bf16lo(w[0][e / 2]);
      else
        x[e] = (float)as_h2(w[0][e / 2])[e % 2];
      // (fmaxf is two instructions: the first for signalling NaN)
      if constexpr (CLEAN) asm("v_max_f32 %0, %1, %0" : "+v"(x[e]) : "s"(floor));
      else x[e] = fmaxf(x[e], floor);
    }
    if (first + (step + 1) * kSlot > vocab) {  // (uniform per wave)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        int skip;
        place(step, e / G, skip);
        if (e % G < skip) x[e] = floor;
      }
    }
  }
  __device__ SM_INLINE void clean(const float (&x)[8], u32x4 (&w)[W]) const {
#pragma unroll
    for (int j = 0; j < 4 * W; ++j) {
      if constexpr (W == 2)
        w[j / 4][j % 4] = __float_as_uint(x[j]);
      else if constexpr (std::is_same<T, uint16_t>::value)
        w[0][j] = __float_as_uint(x[2 * j]) >> 16 | (__float_as_uint(x[2 * j + 1]) & 0xffff0000u);
      else
        w[0][j] = __builtin_bit_cast(uint32_t, h2{(_Float16)x[2 * j], (_Float16)x[2 * j + 1]});
    }
  }
  template <typename F>
  __device__ SM_INLINE void step_again(int i, float floor, F f) const {
    u32x4 w[W];
    read(i, w);
    float x[8];
    values<false>(w, i, floor, x);
    f(i, x);
  }
  // f(step, values) of every step; the first time through, as the loads arrive
  template <typename F>
  __device__ SM_INLINE void each_arriving(F f) {
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      if (i >= steps) continue;  // (uniform)
      u32x4 w[W];
#pragma unroll
      for (int j = 0; j < 4 * W; ++j) w[j / 4][j % 4] = reg[(i * 4 * W + j) / R][(i * 4 * W + j) % R];
      float x[8];
      values<false>(w, i, -INFINITY, x);
      f(i, x);
      clean(x, w);
#pragma unroll
      for (int j = 0; j < 4 * W; ++j) reg[(i * 4 * W + j) / R][(i * 4 * W + j) % R] = w[j / 4][j % 4];
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll 1
    for (int i = STEPS; i < steps; ++i) step_again(i, -INFINITY, f);
  }
  // Steps of which this wave has a value above `bar` (those past STEPS without a look), a bit each.
  __device__ SM_INLINE uint64_t above(float bar) const {
    uint64_t m = 0;
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      if (i >= steps) continue;
      u32x4 w[W];
#pragma unroll
      for (int j = 0; j < 4 * W; ++j) w[j / 4][j % 4] = reg[(i * 4 * W + j) / R][(i * 4 * W + j) % R];
      float g = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4 * W; ++j) {
        if constexpr (W == 2) g = fmaxf(g, __uint_as_float(w[j / 4][j % 4]));
        else if constexpr (std::is_same<T, uint16_t>::value) g = fmaxf(fmaxf(g, bf16lo(w[0][j])), bf16hi(w[0][j]));
        else g = fmaxf(fmaxf(g, (float)as_h2(w[0][j])[0]), (float)as_h2(w[0][j])[1]);
      }
      if (__builtin_amdgcn_ballot_w64(g > bar)) m |= (uint64_t)1 << i;
    }
    if (steps > STEPS) m |= ~(uint64_t)0 << STEPS;
    return m;
  }
  template <typename F>
  __device__ SM_INLINE void each(float floor, F f, uint64_t which = ~(uint64_t)0) {
#pragma unroll 1
    for (int i = 0; i < steps; ++i) {
      if (!(which >> i & 1)) continue;
      u32x4 w[W];
      if (i < STEPS) {
        const int at = i * 4 * W % R;
#pragma unroll
        for (int v = 0; v < V; ++v)
          if (i * 4 * W / R == v) {
#pragma unroll
            for (int j = 0; j < 4 * W; ++j) w[j / 4][j % 4] = reg[v][at + j];
          }
        float x[8];
        values<true>(w, i, floor, x);
        f(i, x);
      } else {
        step_again(i, floor, f);
      }
    }
  }
};

// What the kernels of a row in parts leave each other.
struct RowShare {
  static constexpr int PARTS = 64, WAVES = 512, KEYS = 1024;
  int listed, first;       // the list's entries; the largest logit's first place
  float list_lo, list_hi;
  float m[PARTS], s[PARTS], w[PARTS], low[PARTS];
  double all[WAVES], above[WAVES];
  double slot[kSlots];
  unsigned long long key[KEYS];
  uint32_t bin[4096];
};

// ---- the kernel ----
//
// A workgroup holds a row in registers (up to 65536 f32 or 131072 16-bit logits of 1024 threads), so
// that memory is read once, and what follows works on registers and LDS:
// - the largest logit, and in f32 the sums of the exponentials (for the log-prob) and of the
//   weights, as the loads arrive;
// - top-k up to half of the list: the k-th largest of the threads' own maxima, four each, has at least k
//   logits at or above it and seldom twice as many. These go to a list in LDS, are put in order by
//   counting, and everything else is done on them;
// - top-p without that: the weights in f32 are added up in bins of a hundredth of an octave (LDS
//   atomics on whole numbers: any order gives the same). The logits of the bins around p times the
//   sum, within what f32 may be off, go to the list; one pass with 64-bit weights gives the sums of all
//   and of those above the list, and the exact border is found in the list;
// - the draw: sums of 512 consecutive logits are kept by the 64-bit pass; those that u falls in are
//   read again. One wave does it.
// Rows that the list does not hold (more logits at a border than it has room for, a larger top-k), and those
// with +inf, go by passes: 256 rows of 65536 f32 640 us with top-p where all logits are nearly equal, 420 with
// top-k 3000. What a wave's part of the list has no room for takes places of the others' through one LDS counter:
// rows in falling order with top-p 90 us (493 by passes), flat ones (spread 0.1) with top-p 0.9 109 (643).
//
// Bound by instructions, not by memory. 256 rows of 65536 f32 with top-p 49 us (1.36 TB/s; the logits are 14
// us of HBM): 20 us until the row is there and in bins, 2 for the border's, 19 for the 64-bit pass (an f64
// operation takes 4.9 clocks of a SIMD with four waves, of which a weight needs 16 and its sums 3
// and a logit's share of the rest 14 of 3.3), 7 for list and draw. Without a filter 25 us for 128 rows, with top-k 22.
// 768 rows of 50001 bf16 with options of all kinds 98 us: 17 us a row with top-k, most of it eight
// barriers' waits with one workgroup a unit, 38 with top-p.
// Tried, where 256 rows took 54 us: 512 threads with twice the registers (66: two waves a SIMD issue 5.7 clocks apart), two
// workgroups of 64 registers a thread a unit (16 bits: spills, 98 -> 466) or of 512 threads (117: a row
// takes twice as long), the rows in the order of their length (94, for a scan before the first load), loops unrolled over the
// row's registers (code of 120 KB, fetched anew by every phase: 87), 64-bit bins (8 -> 12).
//
// PHASE 0: all of it, a workgroup a row. 1 to 4: a few large rows in `parts` workgroups each, whose parts
// meet in memory between four kernels: 1 maxima and f32 sums, 2 bins, 3 the list and the 64-bit
// sums, 4 the draw, a workgroup a row again. 6 rows of 131072 f32 with top-p and min-p 83 -> 31 us (3.5,
// 4.6, 8.2 and 13 in the kernels).
template <typename T, int THREADS, int STEPS, int PHASE>
__global__ __launch_bounds__(THREADS, sizeof(T) * STEPS <= 32 ? 4 : 2) void sample_rows_kernel(RowsArgs a) {
  typedef RowLds<THREADS> L;
  constexpr int NW = THREADS / kWave;
  constexpr bool PARTS = PHASE > 0;
  __shared__ L sh;
  const int tid = threadIdx.x, lane = tid % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  int r = (int)blockIdx.x, nth = 0;
  if constexpr (PHASE >= 1 && PHASE <= 3) {
    nth = r % a.parts;
    r /= a.parts;
  }
  RowShare* const rs = PARTS ? reinterpret_cast<RowShare*>(a.ws) + r : nullptr;
  Row<T> row;
  row.p = static_cast<const T*>(a.logits) + r * a.ld;
  row.vocab = a.vocab;
  const float temperature = a.o.temperatures ? a.o.temperatures[r] : a.o.temperature;
  const int top_k = a.o.top_ks ? a.o.top_ks[r] : a.o.top_k;
  const float top_p = a.o.top_ps ? a.o.top_ps[r] : a.o.top_p;
  const float min_p = a.o.min_ps ? a.o.min_ps[r] : a.o.min_p;
  const bool small = a.vocab < 8;
  typedef Held<T, THREADS, STEPS> H;
  H held;
  held.p = row.p;
  held.vocab = a.vocab;
  held.steps = small || PHASE == 4 ? 0 : a.steps;
  held.first = (nth * NW + wave) * a.steps * kSlot;
  if (!small && PHASE != 4) held.load();

  // maximum; sums of exp(x - maximum) for the log-prob and of the weights, in f32
  const bool greedy = !(temperature > 0.f);
  const bool by_k = top_k >= 1 && top_k < a.vocab, by_p = top_p < 1.f;
  const bool weigh = by_p && !by_k && !greedy;
  const float ct = weigh ? lane_f32(kLog2e / temperature, 0) : 0.f;
  // (four maxima a thread, for top-k)
  float four[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY}, tm = -INFINITY, ts = 0.f, tw = 0.f;
  held.each_arriving([&](int, const float(&x)[8]) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < 4; ++e) four[e] = fmaxf(four[e], fmaxf(x[2 * e], x[2 * e + 1]));
    const float n = fmaxf(fmaxf(four[0], four[1]), fmaxf(four[2], four[3]));
    const float ref = n == -INFINITY ? 0.f : n;
    if (PHASE < 2 && a.logprobs) {  // (uniform)
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) s += __builtin_amdgcn_exp2f((x[e] - ref) * kLog2e);
      ts = fmaf(ts, __builtin_amdgcn_exp2f((tm - ref) * kLog2e), s);
    }
    if (PHASE < 2 && weigh) {  // (uniform)
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) s += __builtin_amdgcn_exp2f((x[e] - ref) * ct);
      tw = fmaf(tw, __builtin_amdgcn_exp2f((tm - ref) * ct), s);
    }
    tm = n;
  });
  if (small)
    for (int v = tid; v < a.vocab; v += THREADS) tm = fmaxf(tm, row.at(v));
  float m, sum, whole, low_of_parts = INFINITY;
  {
    // of this wave, of the workgroup, of the parts; uniform values are read to scalar registers
    auto merge = [&](float wm, float ws, float ww) __attribute__((always_inline)) {
      m = lane_f32(wave_max(wm), 0);
      const bool none = wm == -INFINITY;
      const float d = none ? 0.f : wm - m;
      sum = lane_f32(wave_sum(none ? 0.f : ws * __builtin_amdgcn_exp2f(d * kLog2e)), 0);
      whole = lane_f32(wave_sum(none ? 0.f : ww * __builtin_amdgcn_exp2f(d * ct)), 0);
    };
    if constexpr (PHASE < 2) {
      merge(tm, ts, tw);
      float low = INFINITY;
      if constexpr (PHASE == 1) {
#pragma unroll
        for (int e = 0; e < 4; ++e) low = four[e] > -INFINITY ? fminf(low, four[e]) : low;
        low = -wave_max(-low);
      }
      if (lane == 0) {
        sh.m[wave] = m;
        sh.s[wave] = sum;
        sh.w[wave] = whole;
        sh.low[wave] = low;
      }
      __syncthreads();
      const int of = lane < NW ? lane : 0;
      merge(lane < NW ? sh.m[of] : -INFINITY, sh.s[of], sh.w[of]);
      if constexpr (PHASE == 1) {
        low = -wave_max(-sh.low[of]);
        if (tid == 0) {
          rs->m[nth] = m;
          rs->s[nth] = sum;
          rs->w[nth] = whole;
          rs->low[nth] = low;
          if (nth == 0) {
            rs->listed = 0;
            rs->first = 0x7fffffff;
          }
        }
        for (int i = nth * THREADS + tid; i < L::BINS; i += a.parts * THREADS) rs->bin[i] = 0;
        return;
      }
    } else {
      const int of = lane < a.parts ? lane : 0;
      merge(lane < a.parts ? rs->m[of] : -INFINITY, rs->s[of], rs->w[of]);
      low_of_parts = lane_f32(-wave_max(-rs->low[of]), 0);
    }
  }
  row.m = m;
  if (m == -INFINITY) {
    if (tid == 0 && (PHASE == 0 || PHASE == 4)) {
      a.tokens[r] = -1;
      if (a.logprobs) a.logprobs[r] = -INFINITY;
    }
    return;
  }
  row.inv = greedy ? NAN : 1.0 / (double)temperature;
  const double c2 = lane_f64(row.inv * 1.4426950408889634074, 0), m64 = lane_f64((double)m, 0);
  const float c = lane_f32((float)c2, 0);
  // Weights of 2^-1000 of the largest and less are none: logits below `live` are raised to it, and the
  // draw does not take them.
  const float live = lane_f32(m - 1000.f / c, 0);
  const bool plain = !small && m < INFINITY && a.vocab <= kSlots * kSlot &&
                     (greedy || (temperature <= 1e30f && temperature >= 1e-30f &&
                                 (m - live) * c > 980.f && (m - live) * c < 1020.f));
  auto log_prob = [&](float x) { return (x - m) - __logf(sum); };
  if (plain && greedy) {
    if constexpr (PHASE == 2) return;
    int first = PHASE == 4 ? rs->first : 0x7fffffff;
    held.each(-INFINITY, [&](int i, const float(&x)[8]) __attribute__((always_inline)) {
#pragma unroll
      for (int e = 7; e >= 0; --e) {
        int skip;
        const int at = held.place(i, e / H::G, skip);
        if (x[e] == m) first = min(first, at + e % H::G);
      }
    });
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) first = min(first, __shfl_xor(first, o, kWave));
    if (lane == 0) sh.n[wave] = first;
    __syncthreads();
    if (tid == 0) {
#pragma unroll
      for (int i = 0; i < NW; ++i) first = min(first, sh.n[i]);
      if constexpr (PHASE == 3) {
        atomicMin(&rs->first, first);
      } else {
        a.tokens[r] = first;
        if (a.logprobs) a.logprobs[r] = log_prob(m);
      }
    }
    return;
  }
  auto weights = [&](const float* x, double(&w)[4]) __attribute__((always_inline)) {
    double d[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) d[i] = (double)x[i] - m64;
    side_by_side(d);
    exp2_f64(d, c2, w);
  };
  auto weight = [&](float x) __attribute__((always_inline)) { return exp2_f64((double)x - m64, c2); };  // (1 for the largest)
  const double least = lane_f64(min_p > 0.f ? fmin((double)min_p, 1.0) : 0.0, 0);
  bool fits = plain && !(by_k && top_k > L::CAP / 2);  // (uniform from here on)
  float list_lo = m, list_hi = m;  // the list: logits from list_lo to list_hi
  int n = 0;
  // Adds what piece j of a step has of it, in no order: with top-k, where few pieces have any, to the
  // list; else to the wave's part of it, which needs no answer from LDS, until that is full (a border
  // that lies in one stretch of the vocabulary).
  int mine = 0;
  auto to_list = [&](int i, int j, const float* x) __attribute__((always_inline)) {
    bool hit[H::G];
    int put = 0, hits = 0;  // hits of the lanes before this one; of all
#pragma unroll
    for (int e = 0; e < H::G; ++e) {
      hit[e] = x[e] >= list_lo && x[e] <= list_hi;
      const uint64_t b = ballot(hit[e]);
      hits += (int)__builtin_popcountll(b);
      put = (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(b >> 32),
                                           __builtin_amdgcn_mbcnt_lo((uint32_t)b, put));
    }
    if (hits == 0) return;  // (uniform)
    int end = L::CAP;
    unsigned long long* to = PARTS ? rs->key : sh.c.key;
    if (PARTS || by_k) {
      int base = 0;
      if (lane == 0) base = atomicAdd(PARTS ? &rs->listed : &sh.listed, hits);
      put += __builtin_amdgcn_readfirstlane(base);
    } else {
      to = sh.own[wave];
      end = L::CAP / NW;
      put += mine;
      mine += hits;
    }
    int skip;
    const int place = held.place(i, j, skip);
    int before = 0;  // of this lane's hits
#pragma unroll
    for (int e = 0; e < H::G; ++e)
      if (hit[e]) {
        if (put < end) to[put] = (unsigned long long)key_of(x[e]) << 32 | (uint32_t)~(place + e);
        ++put;
        ++before;
      }
    if (!PARTS && !by_k && mine > end) {  // (uniform; seldom)
      const int from = max(mine - hits, end);  // the first that the part does not hold
      int base = 0;
      if (lane == 0) base = atomicAdd(&sh.listed, mine - from);
      base = __builtin_amdgcn_readfirstlane(base) - from;
      put -= before;
#pragma unroll
      for (int e = 0; e < H::G; ++e)
        if (hit[e]) {
          if (put >= end && base + put < L::CAP)
            sh.c.key[base + put] = (unsigned long long)key_of(x[e]) << 32 | (uint32_t)~(place + e);
          ++put;
        }
    }
  };
  if constexpr (PHASE == 4) {
    list_lo = lane_f32(rs->list_lo, 0);
    list_hi = lane_f32(rs->list_hi, 0);
  }
  if (PHASE != 4 && fits && (by_k || by_p)) {
    float scale;  // bins to a unit of logit
    for (int i = tid; i < L::BINS; i += THREADS) sh.bin[i] = PHASE == 3 ? rs->bin[i] : 0;
    if (tid == 0) {
      sh.lo = 0;
      sh.hi = L::BINS - 1;
      sh.listed = 0;
    }
    if (by_k) {
      // bins between the least and the largest of the threads' maxima
      float low = m;
      if constexpr (PARTS) {
        low = fmaxf(low_of_parts, live);
        __syncthreads();
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) low = four[e] > live ? fminf(low, four[e]) : low;
        low = -wave_max(-low);
        if (lane == 0) sh.low[wave] = low;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NW; ++i) low = fminf(low, sh.low[i]);
      }
      scale = m > low ? (float)L::BINS * 0.999f / (m - low) : 0.f;
      scale = lane_f32(scale < 1e30f ? scale : 1e30f, 0);
      if constexpr (PHASE != 3)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (four[e] > live) atomicAdd(&sh.bin[(int)fminf((m - four[e]) * scale, (float)(L::BINS - 1))], 1u);
    } else {
      // the weights in f32, in units of 2^-31 of their sum, so that a bin's sum fits 32 bits
      scale = lane_f32(c * ((float)L::BINS / kOctaves), 0);
      const float unit = lane_f32(31.f - __log2f(whole), 0);
      const float top = lane_f32(m * scale, 0), rest = (float)(L::BINS + lane);
      __syncthreads();
      if constexpr (PHASE != 3)
      held.each(live, [&](int, const float(&x)[8]) __attribute__((always_inline)) {
#pragma unroll
        for (int h = 0; h < 8; h += 4) {
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int e = h; e < h + 4; ++e) {
            const float d = fmaf(-scale, x[e], top);
            const float w = __builtin_amdgcn_exp2f(fmaf(d, -kOctaves / (float)L::BINS, unit));
            // (what lies behind the bins goes to one of the lane's own, where it meets nobody)
            atomicAdd(&sh.bin[(int)__builtin_amdgcn_fmed3f(d, 0.f, rest)], (uint32_t)(w + 0.5f));
          }
        }
      });
    }
    if constexpr (PHASE == 2) {
      __syncthreads();
      for (int i = tid; i < L::BINS; i += THREADS)
        if (sh.bin[i]) atomicAdd(&rs->bin[i], sh.bin[i]);
      return;
    }
    __syncthreads();
    // the bins where the running sum reaches the border, and what f32 may be off
    constexpr int PER = L::BINS / THREADS;
    uint32_t v[PER], sum_v = 0;  // (all are 2^31 and a bit, or four a thread)
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      v[i] = sh.bin[tid * PER + i];
      sum_v += v[i];
    }
    uint32_t inc = sum_v;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
      const uint32_t t = __shfl_up(inc, o, kWave);
      if (lane >= o) inc += t;
    }
    if (lane == kWave - 1) sh.part[wave] = inc;
    __syncthreads();
    uint32_t before = 0, total = 0;
#pragma unroll
    for (int i = 0; i < NW; ++i) {
      if (i < wave) before += sh.part[i];
      total += sh.part[i];
    }
    before += inc - sum_v;
    uint32_t first = 0, last = (uint32_t)top_k;
    if (!by_k) {
      // half a unit a logit, f32's exponentials (of up to kOctaves octaves: 2^-18) and this product
      const double t = (double)total * (double)fmaxf(top_p, 0.f),
                   off = (double)total * 0x1p-17 + 0.5 * (double)a.vocab;
      first = (uint32_t)fmax(t - off, 0.0);
      last = (uint32_t)(t + off) + 1;
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const uint32_t after = before + v[i];
      if (before < first && after >= first) sh.lo = tid * PER + i;
      if (before < last && after >= last) sh.hi = tid * PER + i;
      before = after;
    }
    __syncthreads();
    // The logits of these bins, and what rounding may take for them: d is off by three roundings of
    // up to |m| scale + BINS.
    const float guard = (fabsf(m) + (float)L::BINS / fmaxf(scale, 1e-30f)) * 0x1p-21f;
    list_hi = lane_f32(sh.lo > 0 ? m - (float)sh.lo / scale + guard : m, 0);
    list_lo = lane_f32(sh.hi < L::BINS - 1 && scale > 0.f ? m - (float)(sh.hi + 1) / scale - guard
                                                         : -INFINITY, 0);
    // (above `live`: the next f32)
    const float next = key_value(key_of(live) + 1);
    list_lo = fmaxf(list_lo, next);
    if constexpr (PHASE == 3)
      if (tid == 0 && nth == 0) {
        rs->list_lo = list_lo;
        rs->list_hi = list_hi;
      }
    if (by_k)  // few reach it: none in most steps
      held.each(live, [&](int i, const float(&x)[8]) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < H::W; ++j) to_list(i, j, x + j * H::G);
      }, held.above(key_value(key_of(list_lo) - 1)));
  }
  if constexpr (PHASE == 2) return;
  double* const slots_of_row = PARTS ? rs->slot : sh.slot;
  if (PHASE != 4 && fits && !by_k) {
    // sums in 64 bits: of all (top-p), of those above the list, and of those that are kept, by slots
    if (by_p) {
      double all = 0.0, above = 0.0;
      auto sums = [&](auto MIN_P) __attribute__((always_inline)) {
        held.each(live, [&](int i, const float(&x)[8]) __attribute__((always_inline)) {
          double k = 0.0, z = 0.0;
          uint64_t some = 0;  // lanes with a part of the list
#pragma unroll
          for (int h = 0; h < 8; h += 4) {
            __builtin_amdgcn_sched_barrier(0);
            double w[4];
            weights(x + h, w);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const bool over = x[h + e] > list_hi;
              all += w[e];
              k = fma(w[e], over ? 1.0 : 0.0, k);
              if constexpr (MIN_P.value) z = fma(w[e], over && w[e] >= least ? 1.0 : 0.0, z);
              some |= ballot(x[h + e] >= list_lo) & ~ballot(over);
            }
            if ((h + 4) % H::G == 0) {  // a piece
              if (some) to_list(i, h / H::G, x + h / H::G * H::G);
              some = 0;
            }
          }
          above += k;
          k = wave_add(MIN_P.value ? z : k);
          if (lane == 0 && held.first + i * kSlot < a.vocab) slots_of_row[held.first / kSlot + i] = k;
        });
      };
      if (least > 0.0) sums(std::true_type{});
      else sums(std::false_type{});
      all = wave_add(all);
      above = wave_add(above);
      if (lane == 0) {
        (PARTS ? rs->all : sh.all)[nth * NW + wave] = all;
        (PARTS ? rs->above : sh.above)[nth * NW + wave] = above;
        sh.n[wave] = min(mine, L::CAP / NW);
      }
    } else {
      for (int i = lane; i < a.steps; i += kWave)
        if (held.first + i * kSlot < a.vocab) slots_of_row[held.first / kSlot + i] = 0.0;
      // in f32, what may pass min-p
      const float bar = min_p > 0.f ? fmaxf(live, m + (__log2f(fminf(min_p, 1.f)) - 0.01f) / c) : live;
      held.each(live, [&](int i, const float(&x)[8]) __attribute__((always_inline)) {
        double k = 0.0;
#pragma unroll
        for (int h = 0; h < 8; h += 4) {
          __builtin_amdgcn_sched_barrier(0);
          double w[4];
          weights(x + h, w);
#pragma unroll
          for (int e = 0; e < 4; ++e) k = fma(w[e], w[e] >= least ? 1.0 : 0.0, k);
        }
        k = wave_add(k);
        if (lane == 0 && held.first + i * kSlot < a.vocab) slots_of_row[held.first / kSlot + i] = k;
      }, min_p > 0.f ? held.above(key_value(key_of(lane_f32(bar, 0)) - 1)) : ~(uint64_t)0);
    }
  }
  if constexpr (PHASE == 3) return;
  __syncthreads();
  if constexpr (PHASE == 4) {
    if (fits && !by_k) {  // (loads that do not wait for the list's length)
      for (int i = tid; i < (a.vocab + kSlot - 1) / kSlot; i += THREADS) sh.slot[i] = rs->slot[i];
      double all = 0.0, above = 0.0;
      if (by_p)
        for (int i = tid; i < a.parts * (512 / kWave); i += THREADS) {
          all += rs->all[i];
          above += rs->above[i];
        }
      all = wave_add(all);
      above = wave_add(above);
      if (lane == 0) {
        sh.all[wave] = all;
        sh.above[wave] = above;
      }
    }
    if (fits && (by_k || by_p)) {
      n = rs->listed;
      fits = n <= L::CAP;
      if (fits)
        for (int i = tid; i < n; i += THREADS) sh.c.key[i] = rs->key[i];
      __syncthreads();
    }
  } else if (fits && by_k) {
    n = sh.listed;
    fits = n <= L::CAP;
  } else if (fits && by_p) {  // the waves' parts, behind what they did not hold
    n = sh.listed;
    int at = n;
#pragma unroll
    for (int i = 0; i < NW; ++i) {
      if (i < wave) at += sh.n[i];
      n += sh.n[i];
    }
    fits = n <= L::CAP;
    if (fits)
      for (int i = lane; i < sh.n[wave]; i += kWave) sh.c.key[at + i] = sh.own[wave][i];
    __syncthreads();
  }
  if (!fits) {
    __syncthreads();
    by_passes<THREADS, T>(a, r, row, top_k, top_p, min_p, sh.passes);
    return;
  }
  // the list's orders, by value and by place: how many come before
  if (n > 0) {
    for (int i = tid; i < n; i += THREADS) {
      sh.c.rank[i] = 0;
      sh.c.w[i] = weight(key_value((uint32_t)(sh.c.key[i] >> 32)));
    }
    __syncthreads();
    int wide = 64;
    while (wide < n) wide *= 2;
    const int parts = max(1, THREADS / wide);
    for (int i = tid % wide; i < n; i += THREADS) {
      const unsigned long long key = sh.c.key[i];
      int before = 0;
#pragma unroll 4
      for (int j = tid / wide; j < n; j += parts) {
        const unsigned long long other = sh.c.key[j];
        before += (other > key) + ((uint32_t)other > (uint32_t)key ? 1 << 16 : 0);
      }
      if (before) atomicAdd(&sh.c.rank[i], before);
    }
    __syncthreads();
    for (int i = tid; i < n; i += THREADS) {
      sh.c.order[sh.c.rank[i] & 0xffff] = (uint16_t)i;
      sh.c.place[sh.c.rank[i] >> 16] = (uint16_t)i;
    }
  }
  __syncthreads();
  if (wave > 0) return;

  // one wave from here on
  const double u = fmin(fmax((double)a.uniforms[r], 0.0), 1.0 - 0x1p-53);
  unsigned long long cut = ~0ull;  // the last key of the list that is kept
  double all = 0.0, above = 0.0;
  if (n > 0) {
    if (!by_k) {
      all = lane < NW ? sh.all[lane] : 0.0;
      above = lane < NW ? sh.above[lane] : 0.0;
      all = wave_add(all);
      above = wave_add(above);
    }
    const int per = (n + kWave - 1) / kWave, q0 = lane * per;
    const int most = by_k ? min(n, top_k) : n;
    double part = 0.0;
    for (int q = q0; q < min(q0 + per, most); ++q) part += sh.c.w[sh.c.order[q]];
    const double inc = wave_inclusive(part);
    if (by_k) all = lane_f64(inc, kWave - 1);
    double before = above + (inc - part);
    const double border = by_p ? (double)fmaxf(top_p, 0.f) * all : INFINITY;
    int kept = 0;
    for (int q = q0; q < min(q0 + per, most); ++q) {
      const double w = sh.c.w[sh.c.order[q]];
      if ((before < border || (q == 0 && list_hi == m)) && w >= least) kept = q + 1;
      before += w;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) kept = max(kept, __shfl_xor(kept, o, kWave));
    if (kept > 0) cut = sh.c.key[sh.c.order[kept - 1]];
  }
  if (by_k) {
    // the draw among the list, in the vocabulary's order
    const int per = (n + kWave - 1) / kWave, i0 = lane * per;
    double part = 0.0;
    for (int q = i0; q < min(i0 + per, n); ++q) {
      const int i = sh.c.place[q];
      if (sh.c.key[i] >= cut) part += sh.c.w[i];
    }
    const double inc = wave_inclusive(part);
    const double aim = fmax(u * lane_f64(inc, kWave - 1), 0x1p-900);
    const uint64_t pass = ballot(inc > aim);
    const int who = pass ? (int)__builtin_ctzll(pass) : kWave - 1;
    if (lane != who) return;
    double at = inc - part;
    int got = -1;
    for (int q = i0; q < min(i0 + per, n); ++q) {
      const int i = sh.c.place[q];
      if (sh.c.key[i] >= cut) {
        at += sh.c.w[i];
        got = i;
        if (at > aim) break;
      }
    }
    if (got < 0) got = sh.c.order[0];
    const unsigned long long key = sh.c.key[got];
    a.tokens[r] = (int)~(uint32_t)key;
    if (a.logprobs) a.logprobs[r] = log_prob(key_value((uint32_t)(key >> 32)));
    return;
  }
  // the draw among the slots, the kept of the list in theirs
  const int slots = (a.vocab + kSlot - 1) / kSlot, per = (slots + kWave - 1) / kWave, s0 = lane * per;
  double part = 0.0;
  int i = 0;
  if (n > 0) {  // the list's first entry of this lane's slots
    int top = n;
    while (i < top) {
      const int mid = (i + top) / 2;
      if ((int)~(uint32_t)sh.c.key[sh.c.place[mid]] < s0 * kSlot) i = mid + 1;
      else top = mid;
    }
  }
  for (int s = s0; s < min(s0 + per, slots); ++s) {
    double k = sh.slot[s];
    for (; i < n; ++i) {
      const int at = sh.c.place[i];
      if ((int)~(uint32_t)sh.c.key[at] >= (s + 1) * kSlot) break;
      if (sh.c.key[at] >= cut) k += sh.c.w[at];
    }
    sh.slot[s] = k;
    part += k;
  }
  const double inc = wave_inclusive(part);
  const double aim = fmax(u * lane_f64(inc, kWave - 1), 0x1p-900);
  const uint64_t pass = ballot(inc > aim);
  int who = pass ? (int)__builtin_ctzll(pass) : kWave - 1;
  double left = 0.0;  // of the slot that u falls in
  int slot = 0;
  if (lane == who) {
    double at = inc - part;
    for (int s = s0; s < min(s0 + per, slots); ++s) {
      const double k = sh.slot[s];
      if (k > 0.0) {
        slot = s;
        left = aim - at;
      }
      at += k;
      if (at > aim) break;
    }
  }
  slot = __builtin_amdgcn_readlane(slot, who);
  left = lane_f64(left, who);
  const int base = slot * kSlot + lane * 8;
  double w[8];
  float x[8];
  part = 0.0;
#pragma unroll
  for (int e = 0; e < 8; ++e)
    x[e] = fmaxf(base + e < a.vocab ? row.at(base + e) : -INFINITY, live);
  {
    double lo[4], hi[4];
    weights(x, lo);
    weights(x + 4, hi);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      w[e] = lo[e];
      w[4 + e] = hi[e];
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    bool keep = w[e] >= least && x[e] > live;
    if (by_p) {
      const unsigned long long key = (unsigned long long)key_of(x[e]) << 32 | (uint32_t)~(base + e);
      keep &= x[e] > list_hi || (x[e] >= list_lo && key >= cut);
    }
    if (!keep) w[e] = 0.0;
    part += w[e];
  }
  const double in = wave_inclusive(part);
  uint64_t hit = ballot(in > left && part > 0.0);
  if (!hit) {
    hit = ballot(part > 0.0);
    hit = hit ? (uint64_t)1 << (63 - __builtin_clzll(hit)) : 1;
  }
  who = (int)__builtin_ctzll(hit);
  if (lane != who) return;
  double at = in - part;
  int got = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if (w[e] > 0.0 && at <= left) got = e;
    at += w[e];
  }
  float chosen = x[0];
#pragma unroll
  for (int e = 1; e < 8; ++e)
    if (e == got) chosen = x[e];
  a.tokens[r] = base + got;
  if (a.logprobs) a.logprobs[r] = log_prob(chosen);
}

int check_rows(const char* who, int64_t rows, int64_t vocab, int dtype) {
  SM_REQUIRE(rows >= 0 && rows < (1 << 22) && vocab > 0 && vocab < (1 << 30),
             "%s: need 0 to 2^22 - 1 rows and 1 to 2^30 - 1 logits", who);
  SM_REQUIRE(dtype == SM_F32 || dtype == SM_BF16 || dtype == SM_F16,
             "%s: dtype must be SM_F32, SM_BF16 or SM_F16", who);
  return SM_OK;
}

// Workgroups of a row: as many as a call's rows leave units for, where that is faster than one. The
// four launches take 18 us of the host. f32, us in parts / whole: 32 rows of 65536 with top-p 33 / 49,
// no filter 19 / 23, top-k 23 / 20; 64 rows 44 / 49, 22 / 24, 28 / 20. 64 rows of 131072 69 / 95, 28 / 44, 33 / 34; 128
// rows 110 / 100. 16 rows of 32768 25 / 31, 19 / 16, 20 / 16.
int row_parts(int64_t rows, int64_t vocab) {
  const int64_t parts = std::min<int64_t>({256 / std::max<int64_t>(1, rows), ceil_div(vocab, 4096),
                                           RowShare::PARTS});
  return vocab <= kSlots * kSlot && ((vocab > 49152 && parts >= 8) || (vocab > 98304 && parts >= 4))
             ? (int)parts : 1;
}

}  // namespace
}  // namespace sm

using namespace sm;

extern "C" int64_t sm_sample_rows_workspace_bytes(int64_t rows, int64_t vocab, int dtype) {
  if (check_rows("sm_sample_rows_workspace_bytes", rows, vocab, dtype) != SM_OK) return -1;
  return row_parts(rows, vocab) > 1 ? rows * (int64_t)sizeof(RowShare) : 0;
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
  hipStream_t st = as_stream(stream);
  a.parts = row_parts(rows, vocab);
  a.ws = static_cast<uint8_t*>(workspace);
#define SM_ROWS(T, THREADS, STEPS, PHASE, GRID) \
  sample_rows_kernel<T, THREADS, STEPS, PHASE><<<(unsigned)(GRID), THREADS, 0, st>>>(a)
  if (a.parts > 1) {
    const int64_t need = rows * (int64_t)sizeof(RowShare);
    SM_REQUIRE(workspace && workspace_bytes >= need && reinterpret_cast<uintptr_t>(workspace) % 16 == 0,
               "%s: workspace of %lld bytes, %lld needed, 16-byte aligned", me,
               (long long)workspace_bytes, (long long)need);
    a.steps = (int)ceil_div(vocab, (int64_t)a.parts * 8 * kSlot);
#define SM_ROWS_PARTS(T, STEPS)                 \
  do {                                          \
    SM_ROWS(T, 512, STEPS, 1, rows * a.parts);  \
    SM_ROWS(T, 512, STEPS, 2, rows * a.parts);  \
    SM_ROWS(T, 512, STEPS, 3, rows * a.parts);  \
  } while (0)
#define SM_ROWS_OF(T)                           \
  do {                                          \
    if (a.steps <= 2) SM_ROWS_PARTS(T, 2);      \
    else SM_ROWS_PARTS(T, 8);                   \
    SM_ROWS(T, 512, 2, 4, rows);                \
  } while (0)
    if (dtype == SM_F32) SM_ROWS_OF(float);
    else if (dtype == SM_BF16) SM_ROWS_OF(uint16_t);
    else SM_ROWS_OF(_Float16);
#undef SM_ROWS_OF
#undef SM_ROWS_PARTS
    SM_LAUNCH_CHECK();
    return SM_OK;
  }
  // 256 threads hold rows of up to 16384 logits, so that several are in flight on a unit
  const int threads = vocab <= 16384 ? 256 : vocab > 32768 ? 1024 : 512;
  a.steps = (int)ceil_div(vocab, kSlot * (threads / kWave));
#define SM_ROWS_OF(T, MOST)                                            \
  do {                                                                 \
    if (threads == 256 && a.steps <= 2) SM_ROWS(T, 256, 2, 0, rows);   \
    else if (threads == 256) SM_ROWS(T, 256, 8, 0, rows);              \
    else if (threads == 512) SM_ROWS(T, 512, 8, 0, rows);              \
    else if (a.steps <= 8) SM_ROWS(T, 1024, 8, 0, rows);               \
    else SM_ROWS(T, 1024, MOST, 0, rows);                              \
  } while (0)
  if (dtype == SM_F32) SM_ROWS_OF(float, 8);
  else if (dtype == SM_BF16) SM_ROWS_OF(uint16_t, 16);
  else SM_ROWS_OF(_Float16, 16);
#undef SM_ROWS_OF
#undef SM_ROWS
  SM_LAUNCH_CHECK();
  return SM_OK;
}
