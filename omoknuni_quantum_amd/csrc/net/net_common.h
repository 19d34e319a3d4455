// Helpers shared by the policy-network operators (gfx950, wave64): element types, loads and
// stores of eight elements, reductions over the lanes that share a row, the dropout mask.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "omq_net_ops.h"

namespace omq_net {

constexpr int kWave = 64;

using bf16 = __bf16;
using f16 = _Float16;

// Eight elements are the unit of work of a lane: 16 bytes of a 16-bit type.  The types carry the
// alignment of one element: gfx950 loads and stores 16 bytes at any address that an element may
// have, so odd row lengths and sliced tensors take the same instructions as aligned ones.
template <class T>
using Vec8 __attribute__((aligned(sizeof(T)))) = T __attribute__((ext_vector_type(8)));
using F8 = float __attribute__((ext_vector_type(8)));

template <class T>
__device__ inline F8 to_f8(Vec8<T> v) {
  return __builtin_convertvector(v, F8);
}

// Eight elements from p, of which n are there (n >= 8: all); the others are `fill`.
template <class T>
__device__ inline Vec8<T> load_raw(const T* p, int n, T fill = T(0)) {
  if (n >= 8) return *reinterpret_cast<const Vec8<T>*>(p);
  Vec8<T> v;
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = j < n ? p[j] : fill;
  return v;
}

template <class T>
__device__ inline F8 load8(const T* p, int n) {
  return to_f8<T>(load_raw<T>(p, n));
}

// Rounds to T (to nearest even) and stores the first n of eight.
template <class T>
__device__ inline void store8(T* p, F8 v, int n) {
  using V = T __attribute__((ext_vector_type(8)));
  const V t = __builtin_convertvector(v, V);
  if (n >= 8) {
    *reinterpret_cast<Vec8<T>*>(p) = t;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n) p[j] = t[j];
  }
}

// A weight of the rows' type or of float32.
template <class T>
__device__ inline F8 load_weight(const void* w, bool w_f32, int64_t at, int n) {
  return w_f32 ? load8<float>(static_cast<const float*>(w) + at, n)
               : load8<T>(static_cast<const T*>(w) + at, n);
}

// ---- reductions ---------------------------------------------------------------------------
// Butterflies in registers: within 16 lanes by DPP, then across by the row swaps of gfx950.
// Every lane gets the same value, formed in the same order.
template <int kCtrl>
__device__ inline float dpp(float x) {
  return __int_as_float(
      __builtin_amdgcn_update_dpp(0, __float_as_int(x), kCtrl, 0xF, 0xF, false));
}

struct Sum {
  __device__ static float of(float a, float b) { return a + b; }
  static constexpr float kNone = 0.0f;
};
struct Max {
  __device__ static float of(float a, float b) { return fmaxf(a, b); }
  static constexpr float kNone = -__builtin_inff();
};

// Over each aligned group of `kLanes` lanes (16, 32 or 64), or of 8 or fewer where asked.
template <class Op, int kLanes>
__device__ inline float lanes_reduce(float v) {
  static_assert(kLanes == 8 || kLanes == 16 || kLanes == 32 || kLanes == 64);
  v = Op::of(v, dpp<0xB1>(v));   // quad_perm 1,0,3,2: lane ^ 1
  v = Op::of(v, dpp<0x4E>(v));   // quad_perm 2,3,0,1: lane ^ 2
  v = Op::of(v, dpp<0x141>(v));  // row_half_mirror: the other quad of 8 lanes
  if constexpr (kLanes >= 16) v = Op::of(v, dpp<0x140>(v));  // row_mirror: the other 8 of 16
  if constexpr (kLanes >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                    false);
    v = Op::of(__uint_as_float(r[0]), __uint_as_float(r[1]));
  }
  if constexpr (kLanes >= 64) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                    false);
    v = Op::of(__uint_as_float(r[0]), __uint_as_float(r[1]));
  }
  return v;
}

// Over the kThreads threads of a row: lanes of a wave (16..64), or whole waves of a workgroup
// that holds one row (then every thread of it must come here; `smem` has a float per wave and is
// free again when the next barrier has passed).
template <class Op, int kThreads>
__device__ inline float row_reduce(float v, float* smem) {
  if constexpr (kThreads <= kWave) {
    return lanes_reduce<Op, kThreads>(v);
  } else {
    constexpr int kWaves = kThreads / kWave;
    v = lanes_reduce<Op, kWave>(v);
    if ((threadIdx.x & (kWave - 1)) == 0) smem[threadIdx.x / kWave] = v;
    __syncthreads();
    float s = smem[0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) s = Op::of(s, smem[w]);
    return s;
  }
}

// ---- dropout ------------------------------------------------------------------------------
// SplitMix64's output function (Steele, Lea, Flood, OOPSLA 2014) of a counter: 64 bits serve
// four elements, 16 bits each.
constexpr uint64_t kGolden = 0x9E3779B97F4A7C15ull;

__host__ __device__ inline uint64_t mix64(uint64_t z) {
  z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
  z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
  return z ^ (z >> 31);
}

struct Dropout {
  uint64_t base;       // key + golden: the word of quad q is mix64(base + golden * q)
  uint32_t threshold;  // an element is kept when its 16 bits are at least this
  float scale;
};

inline Dropout make_dropout(double p, uint64_t seed, uint64_t offset) {
  Dropout d;
  const uint64_t key = mix64((mix64(seed + kGolden) ^ offset) + kGolden);
  d.base = key + kGolden;
  d.threshold = (uint32_t)(p * 65536.0 + 0.5);
  d.scale = d.threshold < 65536u ? (float)(65536.0 / (double)(65536u - d.threshold)) : 0.0f;
  return d;
}

// Eight elements from column 8*block of a row whose quads begin at `quad0`.
__device__ inline F8 drop8(F8 v, const Dropout& d, uint64_t quad0, uint32_t block) {
  const uint64_t at = d.base + kGolden * (quad0 + 2ull * block);
  const uint64_t w0 = mix64(at), w1 = mix64(at + kGolden);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t b0 = (uint32_t)(w0 >> (16 * j)) & 0xFFFFu;
    const uint32_t b1 = (uint32_t)(w1 >> (16 * j)) & 0xFFFFu;
    v[j] = b0 >= d.threshold ? v[j] * d.scale : 0.0f;
    v[4 + j] = b1 >= d.threshold ? v[4 + j] * d.scale : 0.0f;
  }
  return v;
}

// ---- host side ----------------------------------------------------------------------------
int net_fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
int net_status(const char* what);  // of the launches made since the last call

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline bool dtype_known(int d) { return d == OMQ_NET_F32 || d == OMQ_NET_BF16 || d == OMQ_NET_F16; }
inline int dtype_size(int d) { return d == OMQ_NET_F32 ? 4 : 2; }

}  // namespace omq_net
