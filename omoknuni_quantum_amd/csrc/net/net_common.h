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

// Eight elements (a block) are the unit of work of a lane: 16 bytes of a 16-bit type.  The types
// carry the alignment of one element: gfx950 loads and stores 16 bytes at any address that an
// element may have, so odd row lengths and sliced tensors take the same instructions as aligned
// ones.
//
// Loading is in two steps, so that a lane has all its loads in flight before it waits for one:
// load_raw is free of branches (a block that is not whole, or beyond the row, is read from the
// row's last eight elements), and to_front and block_of_raw, where the values are used, move a
// part block's elements to the front (and fill up with zeros).  A branch at the load would make the compiler
// wait for each load before the next: the sums of the embedding's gradient ran at 2.5 TB/s so.
//
// kWhole: rows are whole blocks (the columns a multiple of 8), and all this is left out.
template <class T>
using Vec8 __attribute__((aligned(sizeof(T)))) = T __attribute__((ext_vector_type(8)));
template <class T>
using Reg8 = T __attribute__((ext_vector_type(8)));
using F8 = float __attribute__((ext_vector_type(8)));

// The block at column col (a multiple of 8) of a row of `dim` elements, as described above.
template <class T, bool kWhole>
__device__ inline Reg8<T> load_raw(const T* row, int col, int dim) {
  const int last = dim - 8;
  if (kWhole || dim >= 8) return *reinterpret_cast<const Vec8<T>*>(row + (col < last ? col : last));
  Reg8<T> v = {};  // (a row shorter than a block: uniform over the launch)
#pragma unroll
  for (int j = 0; j < 7; ++j)
    if (j < dim) v[j] = row[j];
  return v;
}

// The block moved to the front; what follows the row's end is whatever was there.
template <class T, bool kWhole>
__device__ inline Reg8<T> to_front(Reg8<T> v, int col, int dim) {
  if (!kWhole && dim >= 8) {
    const int s = dim - col < 8 ? (col - dim) & 7 : 0;  // the places to move by
    if constexpr (sizeof(T) == 2) {
      using U4 = uint32_t __attribute__((ext_vector_type(4)));
      U4 d = __builtin_bit_cast(U4, v);
      const bool four = s & 4, two = s & 2;
      const uint32_t one = (s & 1) * 16;
      d[0] = four ? d[2] : d[0], d[1] = four ? d[3] : d[1];
      d[0] = two ? d[1] : d[0], d[1] = two ? d[2] : d[1], d[2] = two ? d[3] : d[2];
      d[0] = __builtin_amdgcn_alignbit(d[1], d[0], one);
      d[1] = __builtin_amdgcn_alignbit(d[2], d[1], one);
      d[2] = __builtin_amdgcn_alignbit(d[3], d[2], one);
      d[3] >>= one;
      v = __builtin_bit_cast(Reg8<T>, d);
    } else {
      const bool four = s & 4, two = s & 2, one = s & 1;
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = four ? v[j + 4] : v[j];
#pragma unroll
      for (int j = 0; j < 6; ++j) v[j] = two ? v[j + 2] : v[j];
#pragma unroll
      for (int j = 0; j < 7; ++j) v[j] = one ? v[j + 1] : v[j];
    }
  }
  return v;
}

// The same with zeros from column dim on.
template <class T, bool kWhole>
__device__ inline Reg8<T> block_of_raw(Reg8<T> v, int col, int dim) {
  v = to_front<T, kWhole>(v, col, dim);
  const int n = dim - col;
  if constexpr (kWhole) {
    if (n <= 0) v = Reg8<T>{};
  } else if (n < 8) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < n ? v[j] : T(0);
  }
  return v;
}

template <class T, bool kWhole>
__device__ inline F8 widen(Reg8<T> v, int col, int dim) {
  return __builtin_convertvector((block_of_raw<T, kWhole>(v, col, dim)), F8);
}

// Rounds to T (to nearest even) and stores the block at column col of the row.  kStream: past the
// caches, for what this kernel does not read again while it still needs what they hold.
template <class T, bool kWhole, bool kStream = false>
__device__ inline void store8(T* row, int col, int dim, F8 v) {
  Reg8<T> t = __builtin_convertvector(v, Reg8<T>);
  T* p = row + col;
  const int n = dim - col;
  if (kWhole ? n > 0 : n >= 8) {
    if constexpr (kStream)
      __builtin_nontemporal_store(t, reinterpret_cast<Vec8<T>*>(p));
    else
      *reinterpret_cast<Vec8<T>*>(p) = t;
  } else if (!kWhole && n > 0) {
    using V4 __attribute__((aligned(sizeof(T)))) = T __attribute__((ext_vector_type(4)));
    using V2 __attribute__((aligned(sizeof(T)))) = T __attribute__((ext_vector_type(2)));
    if (n & 4) {
      *reinterpret_cast<V4*>(p) = V4{t[0], t[1], t[2], t[3]};
      p += 4;
      t = Reg8<T>{t[4], t[5], t[6], t[7], T(0), T(0), T(0), T(0)};
    }
    if (n & 2) {
      *reinterpret_cast<V2*>(p) = V2{t[0], t[1]};
      p += 2;
      t[0] = t[2];
    }
    if (n & 1) *p = t[0];
  }
}

// A weight of the rows' type or of float32 (uniform over the launch).
template <class T>
struct Weight8 {
  Reg8<T> t;
  F8 f;
};

template <class T, bool kWhole>
__device__ inline Weight8<T> load_weight(const void* w, bool w_f32, int col, int dim) {
  Weight8<T> r = {};
  if (w_f32 || sizeof(T) == 4)
    r.f = load_raw<float, kWhole>(static_cast<const float*>(w), col, dim);
  else
    r.t = load_raw<T, kWhole>(static_cast<const T*>(w), col, dim);
  return r;
}

template <class T, bool kWhole>
__device__ inline F8 widen(const Weight8<T>& w, bool w_f32, int col, int dim) {
  return w_f32 || sizeof(T) == 4 ? widen<float, kWhole>(w.f, col, dim)
                                 : widen<T, kWhole>(w.t, col, dim);
}

// Which of the rows of its workgroup a thread belongs to, kThreads threads a row: a scalar where
// a row has whole waves.
template <int kThreads>
__device__ inline int row_slot() {
  const int slot = threadIdx.x / kThreads;
  return kThreads >= kWave ? __builtin_amdgcn_readfirstlane(slot) : slot;
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

// What the words of a row start from.
__device__ inline uint64_t drop_row(const Dropout& d, int64_t row, int dim) {
  return d.base + kGolden * ((uint64_t)row * (uint32_t)((dim + 3) / 4));
}

// The block at column col of the row.
__device__ inline F8 drop8(F8 v, const Dropout& d, uint64_t row_base, int col) {
  const uint64_t at = row_base + kGolden * (uint32_t)(col / 4);
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

// ---- grids --------------------------------------------------------------------------------
// A launch has fewer than 2^32 threads along x: grids of more workgroups go on along y.
__device__ inline int64_t block_index() {
  return (int64_t)blockIdx.x + (int64_t)blockIdx.y * gridDim.x;
}

inline dim3 grid_of(int64_t blocks, int threads) {
  const int64_t most = 0xFFFFFFFFll / threads;
  if (blocks <= most) return dim3((uint32_t)blocks);
  return dim3((uint32_t)most, (uint32_t)((blocks + most - 1) / most));
}

// ---- host side ----------------------------------------------------------------------------
int net_fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
int net_status(const char* what);  // of the launches made since the last call

// Workspaces and the rows' statistics hold 16-byte records.
inline bool on_16_bytes(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline bool dtype_known(int d) { return d == OMQ_NET_F32 || d == OMQ_NET_BF16 || d == OMQ_NET_F16; }
inline int dtype_size(int d) { return d == OMQ_NET_F32 ? 4 : 2; }

}  // namespace omq_net
