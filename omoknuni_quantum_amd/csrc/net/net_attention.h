// What the attention's forward and backward kernels share (gfx950): the tiles of a launch, tiles
// in LDS, and products of 32 x 32 blocks on the matrix cores.
//
// The query heads of one key head are rows side by side: row r of a sequence is the query r / group
// of the head r % group, so that grouped heads share the keys and values that a workgroup loads.
//
// A product's result has a lane per column and its rows spread over the lane's registers: register
// r of lane l is row 8 * (r / 4) + 4 * (l / 32) + r % 4 of column l % 32.  Scores are formed with
// the rows of the stationary side (queries, or keys in the gradient by keys) as columns, so that a
// softmax's statistics are a lane's own, and probabilities go straight from the registers into the
// next product as its second operand: its sum runs over the rows in the order in which the
// registers hold them, and the first operand is read from LDS in the same order (16-bit types
// with the transposing load).
#pragma once

#include <type_traits>

#include "net_common.h"

namespace omq_net {

using F16 = float __attribute__((ext_vector_type(16)));
using F4 = float __attribute__((ext_vector_type(4)));

constexpr float kInf32 = __builtin_inff();
constexpr float kLog2E = 1.4426950408889634f;

constexpr int kWaves = 4;               // waves of a workgroup
constexpr int kWaveRows = 32;           // rows of the stationary side that a wave has
constexpr int kTileRows = kWaves * kWaveRows;
constexpr int kTileKeys = 64;           // rows of the moving side in LDS

struct AttentionArgs {
  omq_attention_args a;
  int group;        // query heads of a key head
  int64_t slots;    // tiles a key head, some of them empty
  int64_t batch_tiles;  // tiles of a sequence of a batch
  float score_scale;    // scale * log2 e
  void* out;
  float* lse;
  const void* grad_out;
  const void* out_in;
  const float* lse_in;
  float* delta;     // [rows of q, q_heads]: sum of grad_out * out
  void *grad_q, *grad_k, *grad_v;
};

// ---- sequences ------------------------------------------------------------------------------
// A sequence's rows in the arrays; lk: its keys in use, of `room`.
struct Sequence {
  int64_t q_first, k_first;  // row in out, lse, grad_q; in grad_k, grad_v
  int64_t q_at, k_at, v_at;  // element of row 0
  int lq, lk, room;
};

__device__ inline int cut(int x, int64_t lo, int64_t hi) {
  return x < lo ? (int)lo : x > hi ? (int)hi : x;
}

// Start s of the n + 2 pieces of [0, total]: before the first sequence, the n sequences, behind
// the last.
__device__ inline int piece_start(const int32_t* starts, int64_t n, int64_t total, int64_t s) {
  if (s == 0) return 0;
  if (s == n + 2) return (int)total;
  return cut(starts[s - 1], 0, total);
}

// The piece that tile `slot` belongs to and the tile's number in it, tiles of `tile` rows of
// `group` to a start's unit: piece s has the tiles from start * group / tile + s, more than it
// needs.  A search of 64 places at a time.
__device__ inline int64_t find_piece(const int32_t* starts, int64_t n, int64_t total, int group,
                                     int tile, int64_t slot, int64_t* index) {
  const int lane = threadIdx.x & (kWave - 1);
  int64_t lo = 0, count = n + 2;
  const auto first = [&](int64_t s) {
    return (int64_t)piece_start(starts, n, total, s) * group / tile + s;
  };
  while (count > 1) {
    const int64_t step = (count + kWave - 1) / kWave, mine = lane * step;
    const bool reached = mine < count && first(lo + mine) <= slot;
    const uint64_t b = __ballot(reached);
    const int64_t at = b ? (int64_t)(63 - __builtin_clzll(b)) * step : 0;
    lo += at;
    count = count - at < step ? count - at : step;
  }
  const int64_t s = ((int64_t)__builtin_amdgcn_readfirstlane((int)(lo >> 32)) << 32) |
                    (uint32_t)__builtin_amdgcn_readfirstlane((int)lo);
  *index = slot - first(s);
  return s;
}

__device__ inline int64_t uniform64(int64_t x) {
  return ((int64_t)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32) |
         (uint32_t)__builtin_amdgcn_readfirstlane((int)x);
}

// The sequence of piece s (packed), or s itself (batch).
__device__ inline Sequence sequence_of(const AttentionArgs& args, int64_t s) {
  const omq_attention_args& a = args.a;
  Sequence q{};
  if (!a.q_starts) {
    q.q_first = s * a.q_len, q.k_first = s * a.k_len;
    q.q_at = s * a.q_seq_stride, q.k_at = s * a.k_seq_stride, q.v_at = s * a.v_seq_stride;
    q.lq = (int)a.q_len, q.room = (int)a.k_len;
    q.lk = a.k_lengths ? cut(a.k_lengths[s], 0, q.room) : q.room;
    return q;
  }
  const int qb = piece_start(a.q_starts, a.sequences, a.q_len, s);
  const int qe = piece_start(a.q_starts, a.sequences, a.q_len, s + 1);
  const int kb = piece_start(a.k_starts, a.sequences, a.k_len, s);
  const int ke = piece_start(a.k_starts, a.sequences, a.k_len, s + 1);
  q.q_first = qb, q.k_first = kb;
  q.q_at = qb * a.q_row_stride, q.k_at = kb * a.k_row_stride, q.v_at = kb * a.v_row_stride;
  q.lq = qe > qb ? qe - qb : 0, q.room = ke > kb ? ke - kb : 0;
  const bool real = s > 0 && s <= a.sequences;  // (else rows of no sequence)
  q.lk = !real ? 0 : a.k_lengths ? cut(a.k_lengths[s - 1], 0, q.room) : q.room;
  return q;
}

// ---- products -------------------------------------------------------------------------------
// 16 bytes a lane are an operand: kChunk columns of the sum, half of them in each half of the wave.
template <class T>
struct Operand {
  using Frag = Reg8<T>;
  static constexpr int kChunk = 16;
};
template <>
struct Operand<float> {
  using Frag = F4;
  static constexpr int kChunk = 8;
};

__device__ inline F16 mma(Reg8<bf16> a, Reg8<bf16> b, F16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ inline F16 mma(Reg8<f16> a, Reg8<f16> b, F16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ inline F16 mma(F4 a, F4 b, F16 c) {
#pragma unroll
  for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b[i], c, 0, 0, 0);
  return c;
}

// A tile in LDS: rows of kDim columns, 16 bytes between them, so that 16 rows' 16 bytes of one
// column lie in different banks.
template <class T, int kDim>
struct Tile {
  using Frag = typename Operand<T>::Frag;
  static constexpr int kChunk = Operand<T>::kChunk;
  static constexpr int kPitch = kDim * (int)sizeof(T) + 16;
  static constexpr int kChunks = kDim / kChunk;   // operands of a row
  static constexpr int kParts = kWaveRows / kChunk;  // operands of 32 rows down a column
  static constexpr int kBytes = kTileKeys * kPitch;

  // Chunk c of the row row0 + lane % 32.
  __device__ static Frag row(const char* tile, int row0, int c) {
    const int lane = threadIdx.x & 63;
    const char* p = tile + (row0 + (lane & 31)) * kPitch + (c * kChunk + (lane >> 5) * (kChunk / 2)) *
                                                               (int)sizeof(T);
    return *reinterpret_cast<const Frag*>(p);
  }

  // Column col0 + lane % 32 of part t of the rows from row0, in the order of a product's registers.
  __device__ static Frag column(const char* tile, int row0, int col0, int t) {
    const int lane = threadIdx.x & 63, half = lane >> 5;
    if constexpr (sizeof(T) == 2) {
      // 16 lanes address four rows of 16 columns, and get a column of four rows each
      const int r = row0 + 16 * t + 4 * half + ((lane & 15) >> 2);
      const int c = col0 + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
      const char* p = tile + r * kPitch + c * 2;
      using S4 = short __attribute__((ext_vector_type(4)));
      using Lds = __attribute__((address_space(3))) S4;
      struct Both {
        S4 lo, hi;
      } v;
      v.lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds*)p);
      v.hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds*)(p + 8 * kPitch));
      return __builtin_bit_cast(Frag, v);
    } else {
      Frag f;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        f[i] = *reinterpret_cast<const float*>(tile + (row0 + 8 * t + 4 * half + i) * kPitch +
                                               (col0 + (lane & 31)) * 4);
      return f;
    }
  }

  // Part t of 32 rows of a result, as the second operand of a product.
  __device__ static Frag part(const F16& x, int t) {
    Frag f;
#pragma unroll
    for (int i = 0; i < kChunk / 2; ++i) f[i] = (T)x[t * (kChunk / 2) + i];
    return f;
  }
};

// The row of register r of a result.
__device__ inline int result_row(int r) {
  return 8 * (r / 4) + 4 * ((threadIdx.x & 63) >> 5) + r % 4;
}

__device__ inline float other_half(float x) {
  const auto r =
      __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float((threadIdx.x & 63) < 32 ? r[1] : r[0]);
}

// ---- values that are not finite -------------------------------------------------------------
// A hidden key's probability is 0, and 0 times an infinity or a NaN is NaN.  Tiles that a mask cuts
// are looked over while they are loaded, and where one holds such a value the product takes 0 in
// its place and adds what visible ones make of the result from a second product: of a code of the
// value (NaN 1, infinities 64 and 4096: sums of 32 of them, exact in every type) and of 1 where the
// key is seen.
template <class T>
__device__ inline bool not_finite(T x) {
  const float f = (float)x;
  return !(__builtin_fabsf(f) < kInf32);
}

template <class T>
__device__ inline bool any_not_finite(const Reg8<T>& v) {
  bool any = false;
#pragma unroll
  for (int j = 0; j < 8; ++j) any = any || not_finite(v[j]);
  return any;
}

// acc += (columns of the tile's 32 rows from row0) x w; careful: as above, w being 0 where `seen`
// is.
template <class T, int kDim>
__device__ inline void add_columns(F16 (&acc)[kDim / 32], const char* tile, int row0,
                                   const F16& w, const F16& seen, bool careful) {
  using L = Tile<T, kDim>;
  typename L::Frag part[L::kParts];
#pragma unroll
  for (int t = 0; t < L::kParts; ++t) part[t] = L::part(w, t);
  if (!careful) {
#pragma unroll
    for (int d = 0; d < kDim / 32; ++d)
#pragma unroll
      for (int t = 0; t < L::kParts; ++t)
        acc[d] = mma(L::column(tile, row0, 32 * d, t), part[t], acc[d]);
    return;
  }
#pragma unroll
  for (int d = 0; d < kDim / 32; ++d) {
    F16 codes = {};
#pragma unroll
    for (int t = 0; t < L::kParts; ++t) {
      typename L::Frag v = L::column(tile, row0, 32 * d, t), code;
#pragma unroll
      for (int i = 0; i < L::kChunk / 2; ++i) {
        const float f = (float)v[i];
        const bool bad = not_finite(v[i]);
        code[i] = (T)(!bad ? 0.0f : f != f ? 1.0f : f > 0.0f ? 64.0f : 4096.0f);
        v[i] = bad ? (T)0.0f : v[i];
      }
      acc[d] = mma(v, part[t], acc[d]);
      codes = mma(code, L::part(seen, t), codes);
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int n = (int)codes[r];
      if (n & 63) acc[d][r] = __builtin_nanf("");
      if (n & (63 << 6)) acc[d][r] += kInf32;
      if (n >> 12) acc[d][r] -= kInf32;
    }
  }
}

// ---- loading and storing --------------------------------------------------------------------
// Eight columns of a row that is there, 0 from column dim on.
template <class T>
__device__ inline Reg8<T> load_piece(const T* row, int col, int dim) {
  if (dim % 8 == 0) return block_of_raw<T, true>(load_raw<T, true>(row, col, dim), col, dim);
  return block_of_raw<T, false>(load_raw<T, false>(row, col, dim), col, dim);
}

// The operands of a row: its chunks, 0 from column dim on.
template <class T, int kDim>
__device__ inline void load_row(typename Operand<T>::Frag (&f)[kDim / Operand<T>::kChunk],
                                const T* row, int dim) {
  const int half = (threadIdx.x & 63) >> 5;
#pragma unroll
  for (int c = 0; c < kDim / Operand<T>::kChunk; ++c) {
    if constexpr (sizeof(T) == 2) {
      f[c] = load_piece(row, 16 * c + 8 * half, dim);
    } else {
      const Reg8<T> v = load_piece(row, 8 * c, dim);
#pragma unroll
      for (int i = 0; i < 4; ++i) f[c][i] = half ? v[4 + i] : v[i];
    }
  }
}

// Loads kTileKeys rows into LDS, zeros for rows from `rows` on (of which there is at least one);
// row_at(i): row i < rows.  True where a value is not finite.
template <class T, int kDim, class RowAt>
__device__ inline bool load_tile(char* tile, int rows, int dim, RowAt&& row_at) {
  constexpr int kPieces = kDim / 8;
  bool bad = false;
#pragma unroll
  for (int i = threadIdx.x; i < kTileKeys * kPieces; i += kWaves * kWave) {
    const int r = i / kPieces, col = i % kPieces * 8;
    Reg8<T> v = load_piece<T>(row_at(r < rows ? r : rows - 1), col, dim);
    if (r >= rows) v = Reg8<T>{};
    bad = bad || any_not_finite<T>(v);
    using Out __attribute__((aligned(16))) = Reg8<T>;
    *reinterpret_cast<Out*>(tile + r * Tile<T, kDim>::kPitch + col * (int)sizeof(T)) = v;
  }
  return bad;
}

// Stores a lane's column of a result [kDim columns of a row, 32 rows] as a row, times `scale`.
template <class T, int kDim>
__device__ inline void store_column(T* row, const F16 (&x)[kDim / 32], float scale, int dim) {
#pragma unroll
  for (int d = 0; d < kDim / 32; ++d)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const int col = 32 * d + result_row(r);
      using V4 __attribute__((aligned(sizeof(T)))) = T __attribute__((ext_vector_type(4)));
      if (col + 4 <= dim) {
        *reinterpret_cast<V4*>(row + col) =
            V4{(T)(x[d][r] * scale), (T)(x[d][r + 1] * scale), (T)(x[d][r + 2] * scale),
               (T)(x[d][r + 3] * scale)};
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (col + i < dim) row[col + i] = (T)(x[d][r + i] * scale);
      }
    }
}

// ---- host side ------------------------------------------------------------------------------
int check_attention(const char* name, const omq_attention_args* a);

inline AttentionArgs attention_layout(const omq_attention_args& a) {
  AttentionArgs r{};
  r.a = a;
  r.group = a.q_heads / a.k_heads;
  r.score_scale = a.scale * kLog2E;
  return r;
}

// The tiles a key head of a launch over `rows` units of `group` rows each (of a sequence, or of
// all packed ones).
inline void tiles_of(AttentionArgs* r, int64_t rows, int64_t group, int64_t tile) {
  r->batch_tiles = ceil_div(rows * group, tile);
  r->slots = r->a.q_starts ? rows * group / tile + r->a.sequences + 2
                           : r->batch_tiles * r->a.sequences;
}

template <class F>
void with_head(int dtype, int dim, F&& f) {
  const auto sized = [&](auto t) {
    using T = decltype(t);
    if (dim <= 32) return f(T{}, std::integral_constant<int, 32>{});
    if (dim <= 64) return f(T{}, std::integral_constant<int, 64>{});
    return f(T{}, std::integral_constant<int, 128>{});
  };
  if (dtype == OMQ_NET_F32) return sized(float{});
  if (dtype == OMQ_NET_BF16) return sized(bf16{});
  return sized(f16{});
}

}  // namespace omq_net
