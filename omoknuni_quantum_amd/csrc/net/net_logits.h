// Rows of logits over legal actions: loading them eight at a time with their mask, the largest of
// them, and the exponential and the logarithm of their sum (gfx950).
#pragma once

#include "net_common.h"

namespace omq_net {

constexpr float kInf = __builtin_inff();
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// e^x from one product and the instruction of 2^x: the product's rounding makes a relative error of
// about |x| 2^-24 (4e-6 at -60, in a term of 1e-26 of the largest), and results below 2^-126 are 0.
__device__ inline float exp_fast(float x) { return __builtin_amdgcn_exp2f(x * kLog2e); }

// log s to about 2^-25 absolute, whatever its size: the exponent's part in 64 bits, the rest, below
// 1/2 in magnitude, from the float32 instruction.
__device__ inline double log_of_sum(float s) {
  float f = __builtin_amdgcn_frexp_mantf(s);
  int k = __builtin_amdgcn_frexp_expf(s);
  const bool low = f < 0.70710678f;
  f = low ? 2.0f * f : f;
  k = low ? k - 1 : k;
  return (double)k * 0.6931471805599453 + (double)(__builtin_amdgcn_logf(f) * kLn2);
}

// A row's arrays.
template <class T>
struct RowIn {
  const T* logits;
  const uint8_t* legal;
  const float* target;
  int cols;
};

// Eight actions of a row as they are loaded (every load is in flight before the first use).
template <class T, bool kTarget>
struct Block {
  Reg8<T> z;
  uint64_t legal;
  F8 pi;
};

template <class T, bool kTarget, bool kWhole>
__device__ inline Block<T, kTarget> load_block(const RowIn<T>& in, int col) {
  Block<T, kTarget> b;
  b.z = load_raw<T, kWhole>(in.logits, col, in.cols);
  b.legal = 0;
  if (in.legal) {
    const int last = in.cols - 8;
    if (kWhole || in.cols >= 8)
      __builtin_memcpy(&b.legal, in.legal + (col < last ? col : last), 8);
    else
      for (int j = 0; j < in.cols; ++j) b.legal |= (uint64_t)in.legal[j] << (8 * j);
  }
  if constexpr (kTarget) b.pi = load_raw<float, kWhole>(in.target, col, in.cols);
  return b;
}

// Which of a block's actions are there and legal: the highest bit of byte j of eight.
template <class T, bool kTarget, bool kWhole>
__device__ inline uint64_t ok_bytes(const Block<T, kTarget>& b, const RowIn<T>& in, int col) {
  constexpr uint64_t kHigh = 0x8080808080808080ull;
  const int left = in.cols - col;
  uint64_t ok = kHigh;
  if (in.legal) {
    uint64_t f = b.legal;
    if (!kWhole && in.cols >= 8 && left < 8) f >>= 8 * ((col - in.cols) & 7);
    ok = (((f & ~kHigh) + ~kHigh) | f) & kHigh;  // (a byte that is not 0)
  }
  if (kWhole ? left <= 0 : left < 8) ok &= left > 0 ? kHigh >> (8 * (8 - left)) : 0;
  return ok;
}

// All ones where action j of the block is there and legal, else 0.
__device__ inline uint32_t ok_mask(uint64_t ok, int j) {
  const int32_t half = (int32_t)(j < 4 ? ok : ok >> 32);
  return (uint32_t)((half << (8 * (3 - (j & 3)))) >> 31);
}

__device__ inline float masked(float x, uint32_t mask, float other) {
  return __uint_as_float((__float_as_uint(x) & mask) | (__float_as_uint(other) & ~mask));
}

// The logits, -inf where there is no legal action.
template <class T, bool kTarget, bool kWhole>
__device__ inline F8 legal_logits(const Block<T, kTarget>& b, const RowIn<T>& in, int col,
                                  uint64_t ok) {
  F8 z = __builtin_convertvector((to_front<T, kWhole>(b.z, col, in.cols)), F8);
  if (kWhole && !in.legal) {
    if (!ok) z = F8{-kInf, -kInf, -kInf, -kInf, -kInf, -kInf, -kInf, -kInf};
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) z[j] = masked(z[j], ok_mask(ok, j), -kInf);
  }
  return z;
}

// The larger of two and of three; the other ones where one is NaN.  (The instruction itself:
// fmaxf costs a second one, which quiets signalling NaN first.)
__device__ inline float larger(float a, float b) {
  float r;
  asm("v_max_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
  return r;
}

__device__ inline float larger(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

__device__ inline float largest(F8 z) {
  return larger(larger(larger(larger(z[0], z[1]), z[2], z[3]), z[4], z[5]), z[6], z[7]);
}

}  // namespace omq_net
