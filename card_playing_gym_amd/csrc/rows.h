// Rows of logits shared by groups of lanes: loads in stored form, reductions, exponentials (gfx950).
#pragma once

#include <cmath>

#include "common.h"

namespace cg {
namespace {

constexpr float LOG2E = 1.44269504088896340736f, LOG2E_REST = float(1.44269504088896340736 - double(LOG2E));

// ---- a group of G lanes that share a row: reductions that leave the result in every lane ---------------

template <int CONTROL>
__device__ __forceinline__ float dpp(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CONTROL, 0xf, 0xf, false));
}
template <int CONTROL>
__device__ __forceinline__ double dpp(double x) {
  return __hiloint2double(__builtin_amdgcn_update_dpp(0, __double2hiint(x), CONTROL, 0xf, 0xf, false),
                          __builtin_amdgcn_update_dpp(0, __double2loint(x), CONTROL, 0xf, 0xf, false));
}
template <int CONTROL>
__device__ __forceinline__ uint64_t dpp(uint64_t x) {
  return __builtin_bit_cast(uint64_t, dpp<CONTROL>(__builtin_bit_cast(double, x)));
}
template <int CONTROL>
__device__ __forceinline__ int dpp(int x) {
  return __builtin_amdgcn_update_dpp(0, x, CONTROL, 0xf, 0xf, false);
}
struct Plus {
  template <typename X>
  __device__ __forceinline__ X operator()(X a, X b) const {
    return a + b;
  }
};
struct Add {
  __device__ __forceinline__ double operator()(double a, double b) const { return a + b; }
};
struct Most {
  __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); }
};

// A wave's LDS writes, visible to its own reads.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}
// The same over a group.
template <int G>
__device__ __forceinline__ void group_sync() {
  if constexpr (G > 64)
    __syncthreads();
  else
    wave_sync();
}

// Within a wave: the lane's neighbour, the pair's, the quad's (mirrored halves of eight), the other eight
// of the row of 16, the other rows.
template <int G, typename X, typename Op>
__device__ __forceinline__ X lanes_join(X x, Op op) {
  x = op(x, dpp<0xB1>(x));   // quad_perm [1, 0, 3, 2]
  x = op(x, dpp<0x4E>(x));   // quad_perm [2, 3, 0, 1]
  if constexpr (G > 4) x = op(x, dpp<0x141>(x));  // row_half_mirror
  if constexpr (G > 8) x = op(x, dpp<0x128>(x));  // row_ror:8
  if constexpr (G > 16) x = op(x, __shfl_xor(x, 16, 64));
  if constexpr (G > 32) x = op(x, __shfl_xor(x, 32, 64));
  return x;
}

// Over several waves through LDS.  Each reduction of a row has a slot of its own, so a slot is written
// again only behind another's barrier, which every wave reaches after its reads.
template <int G, int N, typename X, typename Op>
__device__ __forceinline__ void join(X (&x)[N], X *slot, Op op) {
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = lanes_join<(G < 64 ? G : 64)>(x[i], op);
  if constexpr (G > 64) {
    constexpr int W = G / 64;
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int i = 0; i < N; ++i) slot[i * W + (threadIdx.x >> 6)] = x[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = lanes_join<W>(slot[i * W + threadIdx.x % W], op);
  }
}

// ---- exponentials and logarithms -------------------------------------------------------------------------

// e^x for x <= 0 (-inf: 0), about an ulp and the rounding of the product.  FINE: what that rounding cuts off
// comes back as a factor, for sums whose logarithms are then subtracted.
template <bool FINE = false>
__device__ __forceinline__ float exp_of(float x) {
  const float t = x * LOG2E, e = __builtin_amdgcn_exp2f(t);
  if constexpr (!FINE) return e;
  const float cut = fmaf(x, LOG2E_REST, fmaf(x, LOG2E, -t));
  return x > -126.f ? fmaf(e, cut * 0.69314718f, e) : e;  // (below it: inf - inf)
}

// Reciprocal of a normal number within an ulp or two: the instruction's 2^-26, squared twice.
__device__ __forceinline__ double reciprocal(double x) {
  double r = __builtin_amdgcn_rcp(x);
  r = fma(fma(-x, r, 1.0), r, r);
  return fma(fma(-x, r, 1.0), r, r);
}

// A constant formed where it is used, in scalar registers: the compiler keeps those of a loop's body in
// vector registers around it, 60 of them here, and puts the row into scratch memory for that.
__device__ __forceinline__ double here(double c) {
  int lo = __double2loint(c), hi = __double2hiint(c);
  asm volatile("" : "+s"(lo), "+s"(hi));
  return __hiloint2double(hi, lo);
}

// log x = k log 2 + 2 atanh t for x = 2^k f, f in [1/sqrt 2, sqrt 2), t = (f - 1) / (f + 1): t^2 is below 0.0295,
// so the series to t^15 is off by less than 1e-13.  x: positive and normal, or NaN.
__device__ __forceinline__ double log_of(double x) {
  int k = __builtin_amdgcn_frexp_exp(x);
  double f = __builtin_amdgcn_frexp_mant(x);  // [1/2, 1)
  const bool low = f < here(0.70710678118654752440);
  f = low ? 2 * f : f;
  k -= low;
  const double t = (f - 1) * reciprocal(f + 1), u = t * t;
  double p = here(2.0 / 15);
  p = fma(p, u, here(2.0 / 13));
  p = fma(p, u, here(2.0 / 11));
  p = fma(p, u, here(2.0 / 9));
  p = fma(p, u, here(2.0 / 7));
  p = fma(p, u, here(2.0 / 5));
  p = fma(p, u, here(2.0 / 3));
  p = fma(p, u, 2.0);
  return fma(double(k), here(0.69314718055994530942), t * p);
}

// e^x = 2^k e^r, |r| <= log(2) / 2: the series to r^11 is off by less than 1e-14 of it.
__device__ __forceinline__ double exp_of(double x) {
  x = x > 800 ? 800 : x < -800 ? -800 : x;  // infinity and 0 from here on; NaN stays
  const double k = __builtin_rint(x * here(1.44269504088896340736));
  const double r = fma(k, here(-2.3190468138462996e-17), fma(k, here(-0.69314718055994530942), x));
  double p = here(1.0 / 39916800);
  p = fma(p, r, here(1.0 / 3628800));
  p = fma(p, r, here(1.0 / 362880));
  p = fma(p, r, here(1.0 / 40320));
  p = fma(p, r, here(1.0 / 5040));
  p = fma(p, r, here(1.0 / 720));
  p = fma(p, r, here(1.0 / 120));
  p = fma(p, r, here(1.0 / 24));
  p = fma(p, r, here(1.0 / 6));
  p = fma(p, r, 0.5);
  p = fma(p, r, 1.0);
  p = fma(p, r, 1.0);
  return __builtin_amdgcn_ldexp(p, int(k));
}

// ---- entries --------------------------------------------------------------------------------------------

template <typename T>
constexpr int VEC = 16 / sizeof(T);

template <typename T>
constexpr uint32_t NEGATIVE_INFINITY = __is_same(T, float) ? 0xff800000u : __is_same(T, bf16) ? 0xff80ff80u : 0xfc00fc00u;

// E entries as they are stored, four bytes a word.
template <typename T, int E>
struct Entries {
  static constexpr int PER = 4 / sizeof(T), WORDS = E / PER;
  uint32_t w[WORDS];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int j = 0; j < WORDS; ++j) w[j] = NEGATIVE_INFINITY<T>;
  }
  // From here on what was formed of the entries is formed again: a row's exponentials, kept for the next
  // pass over it, would take twice the registers of its entries.
  __device__ __forceinline__ void forget() {
    if constexpr (E > 1) {
#pragma unroll
      for (int j = 0; j < WORDS; ++j) asm volatile("" : "+v"(w[j]));
    }
  }
  __device__ __forceinline__ float operator[](int k) const {
    if constexpr (PER == 1) {
      return __uint_as_float(w[k]);
    } else {
      const uint32_t q = w[k / 2];
      if constexpr (sizeof(T) == 2 && __is_same(T, bf16)) return __uint_as_float(k % 2 ? q & 0xffff0000u : q << 16);
      return to_f32(T{uint16_t(k % 2 ? q >> 16 : q)});
    }
  }
};

typedef uint32_t Word4 __attribute__((ext_vector_type(4), aligned(2)));  // wherever a row begins

// Four mask bytes: bit 7 of each byte set where the byte is not 0.
__device__ __forceinline__ uint32_t nonzero_bytes(uint32_t b) { return ((b & 0x7f7f7f7fu) + 0x7f7f7f7fu) | b; }

// Four entries, -inf for those whose byte of `legal` is 0.
template <typename T>
__device__ __forceinline__ void bar(uint32_t *w, uint32_t legal) {
  constexpr uint32_t NONE = NEGATIVE_INFINITY<T>;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = legal >> 8 * k & 255 ? w[k] : NONE;
  } else {
    // Sign bits of bytes 0 and 1, then 2 and 3, spread over a half each (v_perm_b32's selectors 8 to 11
    // repeat the signs of bytes 1, 3, 5 and 7).
    const uint32_t t = nonzero_bytes(legal);
    const uint32_t lo = __builtin_amdgcn_perm(t << 8, t, 0x08080a0au), hi = __builtin_amdgcn_perm(t << 8, t, 0x09090b0bu);
    w[0] = (w[0] & lo) | (NONE & ~lo);
    w[1] = (w[1] & hi) | (NONE & ~hi);
  }
}

// A lane's entries of a row: vectors of V from entry (c G + lane) V on for c < C, -inf for those past the row's
// end or not legal.  Rows may start anywhere: 16 bytes are loaded wherever they begin.  A vector over the
// row's end is loaded as its last V entries, of which the first, that a vector before has, count as
// -inf.  Rows shorter than 16 bytes are loaded entry by entry (V = 1) and kept as fp32.
template <int G, int C, int V, typename T>
__device__ __forceinline__ void load_entries(uint32_t *w, const T *row, const uint8_t *legal, int first, int width,
                                             bool streams = false) {
  constexpr int PER = 4 / sizeof(T);
  constexpr uint32_t NONE = NEGATIVE_INFINITY<T>;
  if constexpr (V == 1) {
    w[0] = first < width && (!legal || legal[first]) ? __float_as_uint(to_f32(row[first])) : NEGATIVE_INFINITY<float>;
  } else {
    // inside(c): every lane's vector is (the same for the whole launch)
    const auto inside = [&](int c) { return G > 1 && (c + 1) * G * V <= width; };
    const auto at = [&](int c) { return inside(c) ? first + c * G * V : min(first + c * G * V, width - V); };
#pragma unroll
    for (int c = 0; c < C; ++c) {
      if (streams) {
        const Word4 q = __builtin_nontemporal_load(reinterpret_cast<const Word4 *>(row + at(c)));
        __builtin_memcpy(w + 4 * c, &q, 16);
      } else {
        __builtin_memcpy(w + 4 * c, row + at(c), 16);
      }
    }
    if (legal) {
      uint32_t b[C * (V / 4)];
#pragma unroll
      for (int c = 0; c < C; ++c) __builtin_memcpy(b + c * (V / 4), legal + at(c), V);
#pragma unroll
      for (int j = 0; j < C * (V / 4); ++j) bar<T>(w + 4 / PER * j, b[j]);
    }
#pragma unroll
    for (int c = 0; c < C; ++c) {
      if (inside(c)) continue;
      const int seen = first + c * G * V - at(c);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const uint32_t part = PER == 1 ? ~0u : k % 2 ? 0xffff0000u : 0xffffu;
        uint32_t &x = w[4 * c + k / PER];
        x = k < seen ? (x & ~part) | (NONE & part) : x;
      }
    }
  }
}

// Four gradients rounded to nearest even; a NaN stays one, whichever.
template <typename T>
__device__ __forceinline__ u32x2 packed(f32x4 g) {
  if constexpr (__is_same(T, bf16))
    return __builtin_bit_cast(u32x2, __builtin_convertvector(g, bf16x4));
  else
    return cvt4<T>(g);
}

// The gradients of a vector from entry i on.
template <int V, typename T>
__device__ __forceinline__ void store_entries(T *row, const float *g, int i, int width, bool inside, bool streams = false) {
  if constexpr (V == 1) {
    if (i < width) row[i] = from_f32<T>(g[0]);
  } else if (inside || i + V <= width) {
    Word4 q;
    if constexpr (sizeof(T) == 4) {
      __builtin_memcpy(&q, g, 16);
    } else {
      const u32x2 lo = packed<T>(f32x4{g[0], g[1], g[2], g[3]}), hi = packed<T>(f32x4{g[4], g[5], g[6], g[7]});
      q = Word4{lo[0], lo[1], hi[0], hi[1]};
    }
    if (streams)
      __builtin_nontemporal_store(q, reinterpret_cast<Word4 *>(row + i));
    else
      __builtin_memcpy(row + i, &q, 16);
  } else if (i < width) {
#pragma unroll
    for (int k = 1; k < V; ++k)
      if (width - V + k >= i) row[width - V + k] = from_f32<T>(g[k]);
  }
}

// ---- a loss over rows: its scalars, its partial sums ------------------------------------------------------

struct Scalar {
  float value;
  const float *at;  // NULL: value
};
__device__ __forceinline__ double read(const Scalar &s) { return double(s.at ? *s.at : s.value); }
Scalar scalar(const cg_scalar &s) { return Scalar{s.value, s.device}; }

// The block's sum of `value` over its threads, to its partial sum, or the loss where it is the only one.
template <typename Args>
__device__ __forceinline__ void block_loss(const Args &a, double value) {
  __shared__ double sums[16];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) value += __shfl_xor(value, o, 64);
  if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = value;
  __syncthreads();
  if (threadIdx.x != 0) return;
  double s = 0;
  for (int w = 0; w < int(blockDim.x >> 6); ++w) s += sums[w];
  if (gridDim.x == 1)
    *a.loss = float(s / read(a.normalizer));
  else
    a.partials[blockIdx.x] = s;
}

// The loss of all blocks, in a fixed order: one block, whose threads each add up every THREADS-th partial sum.
template <typename Args, int THREADS = 256>
__global__ __launch_bounds__(THREADS) void loss_kernel(const Args a, int count) {
  double s = 0;
#pragma unroll 8
  for (int k = threadIdx.x; k < count; k += THREADS) s += a.partials[k];
  block_loss(a, s);  // (of one block)
}

// Whether this call has nothing to do: a backward whose gradient is in place already.
template <typename Args>
__device__ __forceinline__ bool done(const Args &a) { return a.upstream && a.written && *a.upstream == 1.0f; }

}  // namespace
}  // namespace cg
