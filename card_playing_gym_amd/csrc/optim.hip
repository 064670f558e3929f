// The optimiser step of an update on the device (gfx950): AdamW over many tensors at once, with
// moments in 32 bits or in 8-bit blocks, and the global norm of a set of gradients.
//
// Per element (t counts from 1, g the gradient times the clipping factor):
//   m = beta1 m + (1 - beta1) g,   v = beta2 v + (1 - beta2) g^2
//   p = p - lr wd p - lr / (1 - beta1^t) * m / (sqrt(v / (1 - beta2^t)) + eps)
// A step is: partial sums of the squares (only when it clips by its own norm), one block that joins
// them and forms every tensor's scalars, and the update.  Tensors' addresses travel in the kernel
// arguments, so a launch covers as many tensors as 4 KB of arguments hold and a captured graph keeps
// them; the step counts are read and advanced on the device, so its replays count on.
//
// The update is bound by HBM: 28 bytes an element with fp32 parameters and moments, 16 with moments
// in 8 bits, 22 and 10 with 16-bit parameters.
#include <cmath>

#include "common.h"

namespace cg {
namespace {

constexpr int THREADS = 256;
// Elements of one tensor that a block updates.  With moments in 32 bits 1024 (against 4096 us: 11.4 M elements
// 63 -> 58, 174 M 889 -> 868); in 8 bits, where a block's start weighs against more arithmetic, 1024 below
// STREAM_BYTES (11.4 M 52 -> 43) and 4096 above (174 M bf16 376, 404 with 1024).
constexpr int CHUNK = 1024, LONG_CHUNK = 4096;
constexpr int NORM_CHUNK = 8192;  // elements whose squares a block sums at a time
constexpr int NORM_BLOCKS = 2048; // most blocks (and partial sums) of a step's norm, over all its launches
constexpr int MOMENT_BLOCK = 256; // elements that share a scale: four a lane

// ---- what a launch carries in its arguments (at most 4 KB) ---------------------------------

constexpr int NORM_TENSORS = 192, PREPARE_TENSORS = 320, UPDATE_TENSORS = 88, UPDATE_TENSORS_8 = 64;

struct NormArgs {
  const void *g[NORM_TENSORS];
  int64_t n[NORM_TENSORS];
  int32_t first_chunk[NORM_TENSORS];  // chunks of the tensors before
  int32_t tensors, chunks;
  double *partials;
};

// The scalars of a step, at the start of its workspace: a header, then one entry a tensor.
struct StepHeader {
  double clip;  // the gradients' factor
  float decay;  // lr * weight_decay
  float pad[5];
};
struct TensorScalars {
  float rate;    // lr / (1 - beta1^t)
  float second;  // 1 / sqrt(1 - beta2^t)
  uint32_t key;  // of the rounding's random words
  uint32_t pad;
};

struct PrepareArgs {
  float *step[PREPARE_TENSORS];
  int32_t index[PREPARE_TENSORS];  // of the tensor's random words
  int32_t tensors;
  int32_t entry;            // of the first tensor's scalars
  int32_t partials;         // partial sums to join; 0: none
  const double *sums;
  double *norm;             // written when there are partial sums, else read; NULL: no clipping
  const float *lr_device;   // NULL: lr
  double lr, log_beta1, log_beta2, weight_decay, max_norm;  // logarithms to base 2
  uint32_t seed;
  StepHeader *header;
};

struct Tensor32 {
  void *p;
  const void *g;
  float *m, *v;
  int64_t n;
};
struct Tensor8 {
  void *p;
  const void *g;
  uint8_t *m, *v;
  float *m_scale, *v_scale;
  int64_t n;
};
template <typename T, int N>
struct UpdateArgs {
  T t[N];
  int32_t first_chunk[N];
  int32_t tensors;
  int32_t entry;  // of the first tensor's scalars
  const StepHeader *header;
  double beta1, beta2;
  float eps;
};
static_assert(sizeof(NormArgs) <= 4096 && sizeof(PrepareArgs) <= 4096, "kernel arguments");
static_assert(sizeof(UpdateArgs<Tensor32, UPDATE_TENSORS>) <= 4096, "kernel arguments");
static_assert(sizeof(UpdateArgs<Tensor8, UPDATE_TENSORS_8>) <= 4096, "kernel arguments");

// The tensor that holds chunk `c`: the last whose first chunk is not past it.  The wave's lanes look
// at the starts side by side (empty tensors share a start with the next one and are never the last).
template <int N>
__device__ __forceinline__ int tensor_of(const int32_t (&first)[N], int tensors, int c) {
  const int lane = threadIdx.x & 63;
  int count = 0;
#pragma unroll
  for (int base = 0; base < N; base += 64) {
    const int i = base + lane;
    count += __popcll(__ballot(i < tensors && first[i < N ? i : 0] <= c));
  }
  return __builtin_amdgcn_readfirstlane(count - 1);
}

// ---- four consecutive elements -----------------------------------------------------------

// STREAM: past the caches' lines that are kept (non-temporal), for data that will not be met there again.
template <bool STREAM, typename V>
__device__ __forceinline__ V load_as(const void *at) {
  if constexpr (STREAM)
    return __builtin_nontemporal_load(static_cast<const V *>(at));
  else
    return *static_cast<const V *>(at);
}
template <bool STREAM, typename V>
__device__ __forceinline__ void store_as(void *at, V x) {
  if constexpr (STREAM)
    __builtin_nontemporal_store(x, static_cast<V *>(at));
  else
    *static_cast<V *>(at) = x;
}
template <bool STREAM, typename T>
__device__ __forceinline__ f32x4 load4(const T *at) {
  if constexpr (sizeof(T) == 4) {
    return load_as<STREAM, f32x4>(at);
  } else {
    struct V {
      T e[4];
    };
    const V q = __builtin_bit_cast(V, load_as<STREAM, u32x2>(at));
    return f32x4{to_f32(q.e[0]), to_f32(q.e[1]), to_f32(q.e[2]), to_f32(q.e[3])};
  }
}
template <bool STREAM, typename T>
__device__ __forceinline__ void store4(T *at, f32x4 x) {
  if constexpr (sizeof(T) == 4)
    store_as<STREAM>(at, x);
  else
    store_as<STREAM>(at, cvt4<T>(x));
}
// The first `count` of four elements; the others are zero, or left alone.
template <typename T>
__device__ __forceinline__ f32x4 load_some(const T *at, int count) {
  f32x4 x{};
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (k < count) x[k] = to_f32(at[k]);
  return x;
}
template <typename T>
__device__ __forceinline__ void store_some(T *at, f32x4 x, int count) {
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (k < count) at[k] = from_f32<T>(x[k]);
}

template <typename T>
__device__ __forceinline__ bool aligned4(const T *at) {
  return reinterpret_cast<uintptr_t>(at) % (4 * sizeof(T)) == 0;
}

// ---- the norm -----------------------------------------------------------------------------

// The block's sum in a fixed order; the result is thread 0's.
__device__ __forceinline__ double block_sum(double x) {
  __shared__ double wave_sums[THREADS / 64];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o, 64);
  if ((threadIdx.x & 63) == 0) wave_sums[threadIdx.x >> 6] = x;
  __syncthreads();
  double s = 0;
  if (threadIdx.x == 0)
    for (int w = 0; w < THREADS / 64; ++w) s += wave_sums[w];
  return s;
}

// Squares of fp32 numbers are exact in fp64 and neither overflow nor vanish there, so the sum needs
// no scaling and the norm is the same whatever the launch shape up to fp64's rounding.
template <typename T, bool STREAM>
__global__ __launch_bounds__(THREADS) void square_sums_kernel(const NormArgs a) {
  double sum = 0;
  for (int c = blockIdx.x; c < a.chunks; c += gridDim.x) {
    const int i = tensor_of(a.first_chunk, a.tensors, c);
    const int64_t begin = int64_t(c - a.first_chunk[i]) * NORM_CHUNK;
    const int64_t left = a.n[i] - begin;
    const T *g = static_cast<const T *>(a.g[i]) + begin;
    const int n = left < NORM_CHUNK ? int(left) : NORM_CHUNK;
    if (n == NORM_CHUNK && aligned4(g)) {
      f32x4 x[NORM_CHUNK / (4 * THREADS)];
#pragma unroll
      for (int k = 0; k < NORM_CHUNK / (4 * THREADS); ++k) x[k] = load4<STREAM>(g + 4 * (k * THREADS + int(threadIdx.x)));
#pragma unroll
      for (int k = 0; k < NORM_CHUNK / (4 * THREADS); ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) sum = fma(double(x[k][e]), double(x[k][e]), sum);
    } else {
      for (int k = threadIdx.x; k < n; k += THREADS) sum = fma(double(to_f32(g[k])), double(to_f32(g[k])), sum);
    }
  }
  sum = block_sum(sum);
  if (threadIdx.x == 0) a.partials[blockIdx.x] = sum;
}

__device__ __forceinline__ double joined_norm(const double *sums, int count) {
  double s = 0;
  for (int k = threadIdx.x; k < count; k += THREADS) s += sums[k];
  return sqrt(block_sum(s));
}

__global__ __launch_bounds__(THREADS) void norm_kernel(const double *sums, int count, double *norm) {
  const double s = joined_norm(sums, count);
  if (threadIdx.x == 0) *norm = s;
}

// ---- the scalars ------------------------------------------------------------------------------

// Two multiplications by odd constants between folds of the upper bits into the lower (the
// multipliers are those of the Philox generators: Salmon et al., SC 2011): a bijection of 32-bit words.
__device__ __forceinline__ uint32_t mix(uint32_t x) {
  x ^= x >> 16;
  x *= 0xD2511F53u;
  x ^= x >> 15;
  x *= 0xCD9E8D57u;
  return x ^ x >> 16;
}

__global__ __launch_bounds__(THREADS) void prepare_kernel(const PrepareArgs a) {
  const double lr = a.lr_device ? double(*a.lr_device) : a.lr;
  const double sum = a.partials ? joined_norm(a.sums, a.partials) : 0;
  if (threadIdx.x == 0 && a.entry == 0) {
    double clip = 1;
    if (a.norm) {
      if (a.partials) *a.norm = sum;
      const double scale = a.max_norm / ((a.partials ? sum : *a.norm) + 1e-6);
      clip = scale > 1 ? 1 : scale;  // (a NaN norm stays NaN)
    }
    a.header->clip = clip;
    a.header->decay = float(lr * a.weight_decay);
  }
  TensorScalars *out = reinterpret_cast<TensorScalars *>(a.header + 1) + a.entry;
  for (int i = threadIdx.x; i < a.tensors; i += THREADS) {
    const float t = *a.step[i] + 1;
    *a.step[i] = t;
    TensorScalars s;
    s.rate = float(lr / (1 - exp2(a.log_beta1 * t)));
    s.second = float(1 / sqrt(1 - exp2(a.log_beta2 * t)));
    s.key = mix(mix(mix(a.seed) + uint32_t(t)) + uint32_t(a.index[i]));
    s.pad = 0;
    out[i] = s;
  }
}

// ---- the update, moments in 32 bits -----------------------------------------------------------

struct Rates {
  float clip, beta1, one1, beta2, one2, eps, decay, rate, second;
};

__device__ __forceinline__ void adamw4(f32x4 &p, const f32x4 g, f32x4 &m, f32x4 &v, const Rates &r) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float x = g[k] * r.clip;
    m[k] = fmaf(r.beta1, m[k], r.one1 * x);
    v[k] = fmaf(r.beta2, v[k], r.one2 * x * x);
    const float step = r.rate * m[k] / fmaf(sqrtf(v[k]), r.second, r.eps);
    p[k] -= fmaf(r.decay, p[k], step);
  }
}

template <typename T, bool STREAM>
__global__ __launch_bounds__(THREADS) void adamw_kernel(const UpdateArgs<Tensor32, UPDATE_TENSORS> a) {
  const int i = tensor_of(a.first_chunk, a.tensors, blockIdx.x);
  const Tensor32 t = a.t[i];
  const int64_t begin = int64_t(int(blockIdx.x) - a.first_chunk[i]) * CHUNK;
  const int64_t left = t.n - begin;
  const int n = left < CHUNK ? int(left) : CHUNK;
  T *p = static_cast<T *>(t.p) + begin;
  const T *g = static_cast<const T *>(t.g) + begin;
  float *m = t.m + begin, *v = t.v + begin;
  const TensorScalars s = reinterpret_cast<const TensorScalars *>(a.header + 1)[a.entry + i];
  const Rates r{float(a.header->clip), float(a.beta1), float(1 - a.beta1), float(a.beta2), float(1 - a.beta2),
                a.eps, a.header->decay, s.rate, s.second};
  const bool vec = aligned4(p) && aligned4(g) && aligned4(m) && aligned4(v);
#pragma unroll
  for (int c = 0; c < CHUNK / (4 * THREADS); ++c) {
    const int e = 4 * (c * THREADS + int(threadIdx.x));
    if (e >= n) break;
    if (vec && e + 4 <= n) {
      f32x4 x = load4<STREAM>(p + e), mm = load4<STREAM>(m + e), vv = load4<STREAM>(v + e);
      const f32x4 gg = load4<STREAM>(g + e);
      adamw4(x, gg, mm, vv, r);
      store4<STREAM>(p + e, x), store4<STREAM>(m + e, mm), store4<STREAM>(v + e, vv);
    } else {
      const int some = n - e < 4 ? n - e : 4;
      f32x4 x = load_some(p + e, some), mm = load_some(m + e, some), vv = load_some(v + e, some);
      const f32x4 gg = load_some(g + e, some);
      adamw4(x, gg, mm, vv, r);
      store_some(p + e, x, some), store_some(m + e, mm, some), store_some(v + e, vv, some);
    }
  }
}

// ---- the update, moments in 8 bits -------------------------------------------------------------
//
// A block of 256 elements has one fp32 scale, its largest |m| or v, and a code an element.  A code q
// above 0 is the exponent and the top three mantissa bits of value / scale, counted down from 1.0 =
// the largest code: 16 octaves below the scale for m (sign and 7 bits), 32 for v (8 bits), eight codes
// each.  v needs no root: 32 octaves of v are 16 of sqrt(v), whose codes are then 3 to 6 % apart.
//
// The scale moves with the block in full precision, but an element moves within its block by
// (1 - beta2) (g^2 / v - 1), about 0.1 % of v a step, far less than the 6 to 12 % between codes: rounded
// to nearest, v would stay where the first steps left it, a fraction of the mean of g^2.  So codes are
// rounded up with the probability of the fraction cut off (16 random bits hashed from seed, step, tensor
// and element), which keeps the running means unbiased.  A v above 0 never becomes 0, or a kept m would
// be divided by eps alone, except where a whole block's v is below fp32's normal numbers (gradients below
// 3e-18): its codes are 0, and sqrt(v) was far below any eps of 1e-16 or more.
//
// New moments are formed in fp64 and their codes cut from its bits: a code is a border for the
// rounding, so equal inputs give equal codes whatever forms the same products elsewhere.  (fp64 adds
// and products have fp32's rate here.)  Each product is rounded: beta1 = 0.9 leaves (9 m + g) / 10 of
// fp32 numbers often within fp64's last bit of the middle of two, where a fused product would round
// the scale another way.

constexpr uint32_t ONE = 8184;  // 1.0: a double's exponent and top three mantissa bits

template <int MOST>
__device__ __forceinline__ double code_value(uint32_t q, uint32_t sign = 0) {
  return __hiloint2double(int(q ? (q + (ONE - MOST)) << 17 | sign : 0u), 0);
}

__device__ __forceinline__ double moment(double beta, double held, double one, double x) {
#pragma clang fp contract(off)
  const double kept = beta * held, added = one * x;
  return kept + added;
}

// The code above ONE - MOST: a quotient's upper word and 17 random bits (16, and the middle of their
// step), cut off behind the third mantissa bit.  least: the lowest to return.
__device__ __forceinline__ uint32_t code_of(uint32_t hi, uint32_t noise, int least) {
  const int q = int((hi + noise) >> 17);
  return uint32_t(min(max(q, least), int(ONE)));
}

// The largest over the wave; patterns of non-negative floats, of which NaN's is above infinity's.
// Lanes take in their neighbours 1, 2, 4 and 8 below inside rows of 16, then rows the one before and
// the two before (out of range: 0); lane 63 has seen all.
template <int CONTROL, int ROWS>
__device__ __forceinline__ uint32_t larger_of(uint32_t x) {
  const uint32_t other = uint32_t(__builtin_amdgcn_update_dpp(0, int(x), CONTROL, ROWS, 0xf, ROWS == 0xf));
  return other > x ? other : x;
}
__device__ __forceinline__ float wave_largest(uint32_t x) {
  x = larger_of<0x111, 0xf>(x);  // row_shr:1, 2, 4, 8
  x = larger_of<0x112, 0xf>(x);
  x = larger_of<0x114, 0xf>(x);
  x = larger_of<0x118, 0xf>(x);
  x = larger_of<0x142, 0xa>(x);  // row_bcast:15, 31
  x = larger_of<0x143, 0xc>(x);
  return __uint_as_float(uint32_t(__builtin_amdgcn_readlane(int(x), 63)));
}

__device__ __forceinline__ double inverse_of(float scale) {
  return scale < 1.17549435e-38f ? 0.0 : double(1.0f / scale);
}

// Roots within an ulp.  The instruction alone takes subnormal numbers for 0, which beside an eps of
// 2^-40 or more is far below the sum's last bit.
__device__ __forceinline__ void roots_of(const float (&v)[4], float (&root)[4], float eps) {
  if (eps >= 0x1p-40f) {
#pragma unroll
    for (int k = 0; k < 4; ++k) root[k] = __builtin_amdgcn_sqrtf(v[k]);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const bool small = v[k] < 0x1p-96f;
      const float r = __builtin_amdgcn_sqrtf(small ? v[k] * 0x1p64f : v[k]);
      root[k] = small ? r * 0x1p-32f : r;
    }
  }
}

struct Rates8 {
  double clip, beta1, one1, beta2, one2;
  float eps, decay, rate, second;
};

// Four elements of a lane, the block's across the wave: parameters and codes in place, new scales.
// index, high: the lower and (times an odd constant) the upper 32 bits of the first element's index.
__device__ __forceinline__ void adamw8(f32x4 &x, const f32x4 g, uint32_t &mq, uint32_t &vq, float &m_scale,
                                       float &v_scale, uint32_t index, uint32_t key, uint32_t high, const Rates8 &r) {
  double m[4], v[4];
  float m32[4], v32[4], root[4];
  uint32_t m_top = 0, v_top = 0;
  const double ms = m_scale, vs = v_scale;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const double d = double(g[k]) * r.clip;
    const uint32_t q = mq >> 8 * k;
    m[k] = moment(r.beta1, code_value<127>(q & 127, q << 24 & 0x80000000u) * ms, r.one1, d);
    v[k] = moment(r.beta2, code_value<255>(vq >> 8 * k & 255) * vs, r.one2, d * d);
    m32[k] = float(m[k]), v32[k] = float(v[k]);
    m_top = max(m_top, __float_as_uint(m32[k]) & 0x7fffffffu);
    v_top = max(v_top, __float_as_uint(v32[k]));  // (a sign, of a NaN, puts it on top too)
  }
  roots_of(v32, root, r.eps);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float step = r.rate * m32[k] * __builtin_amdgcn_rcpf(fmaf(root[k], r.second, r.eps));
    x[k] -= fmaf(r.decay, x[k], step);
  }
  m_scale = wave_largest(m_top), v_scale = wave_largest(v_top);
  const double m_inv = inverse_of(m_scale), v_inv = inverse_of(v_scale);
  // Each code is formed above 0's, ONE - 127 and ONE - 255; the four offsets come off at once.
  constexpr uint32_t M0 = ONE - 127, V0 = ONE - 255;
  mq = -(M0 * 0x01010101u), vq = -(V0 * 0x01010101u);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint32_t word = mix(((index + k) ^ key) + high);
    const uint32_t m_hi = uint32_t(__double2hiint(m[k] * m_inv)), v_hi = uint32_t(__double2hiint(v[k] * v_inv));
    const uint32_t q = code_of(m_hi & 0x7fffffffu, (word << 1 & 0x1fffeu) | 1, M0);
    mq += (q + (q != M0 ? m_hi >> 24 & 128 : 0u)) << 8 * k;
    vq += code_of(v_hi, (word >> 15 & 0x1fffeu) | 1, v_hi ? V0 + 1 : V0) << 8 * k;  // (no quotient is subnormal)
  }
}

template <typename T, bool STREAM>
__global__ __launch_bounds__(THREADS) void adamw8_kernel(const UpdateArgs<Tensor8, UPDATE_TENSORS_8> a) {
  const int i = tensor_of(a.first_chunk, a.tensors, blockIdx.x);
  const Tensor8 t = a.t[i];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const TensorScalars s = reinterpret_cast<const TensorScalars *>(a.header + 1)[a.entry + i];
  const Rates8 r{a.header->clip, a.beta1, 1 - a.beta1, a.beta2, 1 - a.beta2, a.eps, a.header->decay, s.rate, s.second};
  const bool vec = aligned4(static_cast<T *>(t.p)) && aligned4(static_cast<const T *>(t.g)) && aligned4(t.m) && aligned4(t.v);
  constexpr int BLOCKS = (STREAM ? LONG_CHUNK : CHUNK) / MOMENT_BLOCK;
  const int64_t blocks = (t.n + MOMENT_BLOCK - 1) / MOMENT_BLOCK;
  const int64_t first = int64_t(int(blockIdx.x) - a.first_chunk[i]) * BLOCKS;
#pragma unroll
  for (int c = 0; c < BLOCKS / (THREADS / 64); ++c) {
    const int64_t b = first + c * (THREADS / 64) + wave;
    if (b >= blocks) break;  // whole wave
    const int64_t at = b * MOMENT_BLOCK;
    T *p = static_cast<T *>(t.p) + at;
    const T *g = static_cast<const T *>(t.g) + at;
    uint8_t *m = t.m + at, *v = t.v + at;
    const int e = 4 * lane;
    const uint32_t index = uint32_t(at) + e, high = uint32_t(uint64_t(at) >> 32) * 0x9E3779B9u;
    float m_scale = t.m_scale[b], v_scale = t.v_scale[b];
    f32x4 x, grad;
    uint32_t mq = 0, vq = 0;
    if (vec && t.n - at >= MOMENT_BLOCK) {  // whole wave
      x = load4<STREAM>(p + e), grad = load4<STREAM>(g + e);
      mq = load_as<STREAM, uint32_t>(m + e), vq = load_as<STREAM, uint32_t>(v + e);
      adamw8(x, grad, mq, vq, m_scale, v_scale, index, s.key, high, r);
      store4<STREAM>(p + e, x);
      store_as<STREAM>(m + e, mq), store_as<STREAM>(v + e, vq);
    } else {
      const int left = int(t.n - at < MOMENT_BLOCK ? t.n - at : MOMENT_BLOCK) - e;
      const int some = left > 4 ? 4 : left > 0 ? left : 0;
      x = load_some(p + e, some), grad = load_some(g + e, some);
      for (int k = 0; k < some; ++k) mq |= uint32_t(m[e + k]) << 8 * k, vq |= uint32_t(v[e + k]) << 8 * k;
      adamw8(x, grad, mq, vq, m_scale, v_scale, index, s.key, high, r);
      store_some(p + e, x, some);
      for (int k = 0; k < some; ++k) m[e + k] = uint8_t(mq >> 8 * k), v[e + k] = uint8_t(vq >> 8 * k);
    }
    if (lane == 0) t.m_scale[b] = m_scale, t.v_scale[b] = v_scale;
  }
}

// What the codes of n elements stand for, in fp32.
template <int MOST>
__global__ __launch_bounds__(THREADS) void moment_values_kernel(const uint8_t *__restrict__ codes,
                                                                const float *__restrict__ scales,
                                                                float *__restrict__ values, int64_t n) {
  const int64_t e = 4 * (int64_t(blockIdx.x) * THREADS + threadIdx.x);
  if (e >= n) return;
  const int some = n - e >= 4 ? 4 : int(n - e);
  const bool vec = some == 4 && aligned4(codes) && aligned4(values);
  uint32_t q = 0;
  if (vec)
    q = *reinterpret_cast<const uint32_t *>(codes + e);
  else
    for (int k = 0; k < some; ++k) q |= uint32_t(codes[e + k]) << 8 * k;
  const double scale = scales[e / MOMENT_BLOCK];
  f32x4 x;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint32_t c = q >> 8 * k & 255;
    x[k] = float(code_value<MOST>(c & MOST, MOST == 127 ? c << 24 & 0x80000000u : 0u) * scale);
  }
  if (vec)
    store4<true>(values + e, x);
  else
    store_some(values + e, x, some);
}

// ---- host side ----------------------------------------------------------------------------------

// A launch counts its threads in 32 bits.
constexpr int64_t MOST_ELEMENTS = int64_t(1) << 33, MOST_BLOCKS = (int64_t(1) << 24) - 1;
static_assert(MOST_ELEMENTS / CHUNK <= MOST_BLOCKS && MOST_BLOCKS * THREADS < (int64_t(1) << 32), "grid");

int64_t chunks_of(int64_t n, int chunk) { return (n + chunk - 1) / chunk; }

struct GradList {
  const void *const *g;
  const int64_t *n;  // stride in 8-byte words: the sizes may sit inside larger records
  int64_t stride;
  int count;
  int64_t size(int i) const { return n[i * stride]; }
};

// Launches the partial sums of the tensors of type `dtype`; returns how many sums were written.
template <typename T>
int launch_square_sums(const GradList &list, const int32_t *dtypes, int32_t dtype, int budget, bool streams,
                       double *partials, hipStream_t stream) {
  int written = 0, at = 0;
  while (at < list.count) {
    NormArgs a{};
    int64_t chunks = 0;
    for (; at < list.count && a.tensors < NORM_TENSORS; ++at) {
      if (list.g[at] == nullptr || list.size(at) == 0 || (dtypes && dtypes[at] != dtype)) continue;
      const int64_t more = chunks_of(list.size(at), NORM_CHUNK);
      if (chunks + more > INT32_MAX) break;
      a.g[a.tensors] = list.g[at];
      a.n[a.tensors] = list.size(at);
      a.first_chunk[a.tensors++] = int32_t(chunks);
      chunks += more;
    }
    if (a.tensors == 0) continue;
    a.chunks = int32_t(chunks);
    a.partials = partials + written;
    const int grid = int(chunks < budget ? chunks : budget);
    (streams ? square_sums_kernel<T, true> : square_sums_kernel<T, false>)<<<grid, THREADS, 0, stream>>>(a);
    CG_LAUNCHED();
    written += grid;
  }
  return written;
}

// Blocks a launch of the norm may have: its share of NORM_BLOCKS.
int norm_budget(int tensors, int dtypes) {
  const int launches = (tensors + NORM_TENSORS - 1) / NORM_TENSORS * dtypes;
  const int share = NORM_BLOCKS / (launches > 0 ? launches : 1);
  return share > 256 ? share : 256;
}

size_t partial_bytes(int tensors, int dtypes) {
  const int launches = (tensors + NORM_TENSORS - 1) / NORM_TENSORS * dtypes;
  return size_t(launches) * norm_budget(tensors, dtypes) * sizeof(double);
}

size_t scalars_bytes(int n) { return sizeof(StepHeader) + size_t(n) * sizeof(TensorScalars); }

int dtype_index(int32_t dtype) {
  CG_REQUIRE(dtype == CG_F32 || dtype == CG_BF16 || dtype == CG_F16, CG_ERR_INVALID, "unknown dtype");
  return dtype;
}

// Above this many bytes of parameters, gradients and state together a step goes past the caches
// (the Infinity Cache has 256 MB): what one launch leaves there is gone before it is met again.
// fp32 parameters and moments, in blocks of 4096, us: 174 M elements (2.8 GB) norm 167 -> 105, update 912 -> 884;
// but 11.4 M (182 MB) norm 16 -> 10.5 and the update, which meets gradients that the norm has read, 53 -> 67.
constexpr int64_t STREAM_BYTES = 512 << 20;

int launch_norm(const GradList &list, const int32_t *dtypes, int32_t dtype, bool streams, double *partials,
                hipStream_t stream) {
  bool seen[3] = {};
  for (int i = 0; i < list.count; ++i) seen[dtype_index(dtypes ? dtypes[i] : dtype)] = true;
  const int budget = norm_budget(list.count, dtypes ? 3 : 1);
  int sums = 0;
  if (seen[CG_F32]) sums += launch_square_sums<float>(list, dtypes, CG_F32, budget, streams, partials + sums, stream);
  if (seen[CG_BF16]) sums += launch_square_sums<bf16>(list, dtypes, CG_BF16, budget, streams, partials + sums, stream);
  if (seen[CG_F16]) sums += launch_square_sums<f16>(list, dtypes, CG_F16, budget, streams, partials + sums, stream);
  return sums;
}

template <typename T, int N, typename Fill>
void launch_updates(void (*kernel)(UpdateArgs<T, N>), int chunk, const cg_adamw_tensor *tensors, const void *const *grads, int n,
                    const cg_adamw_config &c, StepHeader *header, hipStream_t stream, const Fill &fill) {
  int at = 0, entry = 0;  // entries count the tensors that take part
  while (at < n) {
    UpdateArgs<T, N> a{};
    a.entry = entry;
    int64_t chunks = 0;
    for (; at < n && a.tensors < N; ++at) {
      if (grads[at] == nullptr || tensors[at].n == 0) continue;
      const int64_t more = chunks_of(tensors[at].n, chunk);
      if (chunks + more > MOST_BLOCKS) break;
      a.t[a.tensors] = fill(tensors[at], grads[at]);
      a.first_chunk[a.tensors++] = int32_t(chunks);
      chunks += more;
    }
    if (a.tensors == 0) continue;
    entry += a.tensors;
    a.header = header;
    a.beta1 = c.beta1;
    a.beta2 = c.beta2;
    a.eps = float(c.eps);
    kernel<<<unsigned(chunks), THREADS, 0, stream>>>(a);
    CG_LAUNCHED();
  }
}

}  // namespace
}  // namespace cg

using namespace cg;

extern "C" {

size_t cg_grad_norm_workspace_size(int32_t n) { return n > 0 ? partial_bytes(n, 3) : 0; }

int cg_grad_norm(const void *const *grads, const int64_t *sizes, const int32_t *dtypes, int32_t n, double *norm,
                 void *workspace, size_t workspace_size, void *stream) {
  return guarded([&] {
    CG_REQUIRE(n >= 0, CG_ERR_INVALID, "the number of gradients must be non-negative");
    CG_REQUIRE(norm != nullptr, CG_ERR_INVALID, "norm is NULL");
    CG_REQUIRE(n == 0 || (grads && sizes && dtypes), CG_ERR_INVALID, "grads, sizes and dtypes are required");
    CG_REQUIRE(n == 0 || workspace, CG_ERR_INVALID, "workspace is NULL");
    CG_REQUIRE(workspace_size >= cg_grad_norm_workspace_size(n), CG_ERR_INVALID, "workspace too small");
    for (int i = 0; i < n; ++i)
      CG_REQUIRE(sizes[i] >= 0 && sizes[i] <= MOST_ELEMENTS, CG_ERR_RANGE, "a gradient's size is out of range");
    double *partials = static_cast<double *>(workspace);
    int64_t bytes = 0;
    for (int i = 0; i < n; ++i) bytes += grads[i] ? sizes[i] * dtype_size(dtypes[i]) : 0;
    const int sums = launch_norm(GradList{grads, sizes, 1, n}, dtypes, 0, bytes > STREAM_BYTES, partials, as_stream(stream));
    norm_kernel<<<1, THREADS, 0, as_stream(stream)>>>(partials, sums, norm);
    CG_LAUNCHED();
  });
}

size_t cg_adamw_workspace_size(int32_t n) { return n > 0 ? (scalars_bytes(n) + 15) / 16 * 16 + partial_bytes(n, 1) : 0; }

int cg_adamw_step(const cg_adamw_tensor *tensors, const void *const *grads, int32_t n, const cg_adamw_config *config,
                  double *norm, void *workspace, size_t workspace_size, void *stream) {
  return guarded([&] {
    CG_REQUIRE(config != nullptr, CG_ERR_INVALID, "config is NULL");
    CG_REQUIRE(n >= 0, CG_ERR_INVALID, "the number of tensors must be non-negative");
    const cg_adamw_config &c = *config;
    dtype_index(c.dtype);
    CG_REQUIRE(c.state_bits == 32 || c.state_bits == 8, CG_ERR_INVALID, "state_bits must be 32 or 8");
    CG_REQUIRE(c.beta1 >= 0 && c.beta1 < 1 && c.beta2 >= 0 && c.beta2 < 1, CG_ERR_INVALID, "betas must lie in [0, 1)");
    CG_REQUIRE(c.clip == CG_CLIP_NONE || c.clip == CG_CLIP_OWN_NORM || c.clip == CG_CLIP_GIVEN_NORM, CG_ERR_INVALID,
               "unknown clip mode");
    CG_REQUIRE(c.clip == CG_CLIP_NONE || norm, CG_ERR_INVALID, "clipping needs norm");
    const hipStream_t s = as_stream(stream);
    const auto zero_norm = [&] {  // no gradient at all
      if (c.clip != CG_CLIP_OWN_NORM) return;
      norm_kernel<<<1, THREADS, 0, s>>>(nullptr, 0, norm);
      CG_LAUNCHED();
    };
    if (n == 0) return zero_norm();
    CG_REQUIRE(tensors && grads && workspace, CG_ERR_INVALID, "tensors, grads and workspace are required");
    CG_REQUIRE(workspace_size >= cg_adamw_workspace_size(n), CG_ERR_INVALID, "workspace too small");
    CG_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, CG_ERR_INVALID, "workspace must be 16-byte aligned");
    for (int i = 0; i < n; ++i) {
      const cg_adamw_tensor &t = tensors[i];
      CG_REQUIRE(t.n >= 0 && t.n <= MOST_ELEMENTS, CG_ERR_RANGE, "a tensor's size is out of range");
      if (t.n == 0 || grads[i] == nullptr) continue;
      CG_REQUIRE(t.param && t.exp_avg && t.exp_avg_sq && t.step, CG_ERR_INVALID, "a tensor's state is NULL");
      CG_REQUIRE(c.state_bits == 32 || (t.exp_avg_scale && t.exp_avg_sq_scale), CG_ERR_INVALID,
                 "moments in 8 bits need their scales");
    }
    int64_t elements = 0;
    for (int i = 0; i < n; ++i) elements += grads[i] ? tensors[i].n : 0;
    const bool streams = elements > STREAM_BYTES / (2 * dtype_size(c.dtype) + c.state_bits / 4);
    StepHeader *header = static_cast<StepHeader *>(workspace);
    double *partials = reinterpret_cast<double *>(static_cast<char *>(workspace) + (scalars_bytes(n) + 15) / 16 * 16);
    int sums = 0;
    if (c.clip == CG_CLIP_OWN_NORM)
      sums = launch_norm(GradList{grads, &tensors[0].n, int64_t(sizeof(cg_adamw_tensor) / 8), n}, nullptr, c.dtype, streams, partials, s);
    if (sums == 0) zero_norm();
    int entry = 0;
    for (int at = 0; at < n;) {
      PrepareArgs a{};
      a.entry = entry;
      a.partials = entry == 0 ? sums : 0;
      a.sums = partials;
      a.norm = c.clip == CG_CLIP_NONE ? nullptr : norm;
      a.lr_device = c.lr_device;
      a.lr = c.lr, a.log_beta1 = std::log2(c.beta1), a.log_beta2 = std::log2(c.beta2), a.weight_decay = c.weight_decay, a.max_norm = c.max_norm;
      a.seed = c.seed;
      a.header = header;
      for (; at < n && a.tensors < PREPARE_TENSORS; ++at) {
        if (grads[at] == nullptr || tensors[at].n == 0) continue;
        a.index[a.tensors] = c.first + at;
        a.step[a.tensors++] = tensors[at].step;
      }
      if (a.tensors == 0) continue;
      entry += a.tensors;
      prepare_kernel<<<1, THREADS, 0, s>>>(a);
      CG_LAUNCHED();
    }
    const auto wide = [](const cg_adamw_tensor &t, const void *g) {
      return Tensor32{t.param, g, static_cast<float *>(t.exp_avg), static_cast<float *>(t.exp_avg_sq), t.n};
    };
    const auto narrow = [](const cg_adamw_tensor &t, const void *g) {
      return Tensor8{t.param, g, static_cast<uint8_t *>(t.exp_avg), static_cast<uint8_t *>(t.exp_avg_sq),
                     t.exp_avg_scale, t.exp_avg_sq_scale, t.n};
    };
    const auto run = [&](auto type) {
      using T = decltype(type);
      if (c.state_bits == 32)
        launch_updates<Tensor32, UPDATE_TENSORS>(streams ? adamw_kernel<T, true> : adamw_kernel<T, false>, CHUNK,
                                                 tensors, grads, n, c, header, s, wide);
      else
        launch_updates<Tensor8, UPDATE_TENSORS_8>(streams ? adamw8_kernel<T, true> : adamw8_kernel<T, false>,
                                                  streams ? LONG_CHUNK : CHUNK, tensors, grads, n, c, header, s, narrow);
    };
    if (c.dtype == CG_F32)
      run(float{});
    else if (c.dtype == CG_BF16)
      run(bf16{});
    else
      run(f16{});
  });
}

int cg_moment_values(const uint8_t *codes, const float *scales, int32_t is_signed, float *values, int64_t n,
                     void *stream) {
  return guarded([&] {
    CG_REQUIRE(n >= 0 && n <= MOST_ELEMENTS, CG_ERR_RANGE, "n is out of range");
    if (n == 0) return;
    CG_REQUIRE(codes && scales && values, CG_ERR_INVALID, "codes, scales and values are required");
    const unsigned grid = unsigned(chunks_of(n, 4 * THREADS));
    const auto kernel = is_signed ? moment_values_kernel<127> : moment_values_kernel<255>;
    kernel<<<grid, THREADS, 0, as_stream(stream)>>>(codes, scales, values, n);
    CG_LAUNCHED();
  });
}

}  // extern "C"
