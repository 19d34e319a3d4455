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

// Waves a SIMD that a kernel's registers have to leave room for: two, so that one's products run
// while the other forms its probabilities (float32 heads of 128 columns: their operands alone take
// the registers of one).
template <class T, int kDim>
constexpr int waves_per_simd() {
  return sizeof(T) == 4 && kDim > 64 ? 1 : 2;
}

struct AttentionArgs {
  omq_attention_args a;
  int group;        // query heads of a key head
  int64_t slots;    // tiles a key head, some of them empty
  int64_t batch_tiles;  // tiles of a sequence of a batch
  float score_scale;    // scale * log2 e
  int even;             // the moving side's rows are EvenRows
  int paired;           // (place_of_keys)
  int splits;           // parts of a sequence's keys, each a workgroup's
  float* parts;         // [splits, rows of out, dim] sums, and behind them
  float2* part_stats;   // [splits, rows of out] maximum and sum of the exponentials
  int64_t out_rows;
  uint32_t group_mul;   // a row's query is umulhi(row, group_mul) >> group_shift; 0: the row
  int group_shift;
  void* out;
  float* lse;
  const void* grad_out;
  const void* out_in;
  const float* lse_in;
  float* delta;     // [rows of q, q_heads]: sum of grad_out * out
  void *grad_q, *grad_k, *grad_v;
};

// The query of a row and its head in the group.
__device__ inline int query_of(const AttentionArgs& args, int row) {
  return args.group_mul ? (int)(__umulhi((uint32_t)row, args.group_mul) >> args.group_shift) : row;
}

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

// The tile of a launch by rows of queries: its sequence and number, or false.  Those of the last rows
// come first: in a causal sequence they see the most keys.
struct Place {
  Sequence q;
  int kv;
  int64_t tile;
};

__device__ inline bool place_of_queries(const AttentionArgs& args, int tile_rows, int64_t block,
                                        Place* p) {
  const omq_attention_args& a = args.a;
  int64_t slot = block / a.k_heads;
  if (slot >= args.slots) return false;
  slot = args.slots - 1 - slot;
  p->kv = (int)(block % a.k_heads);
  if (a.q_starts) {
    p->q = sequence_of(args, find_piece(a.q_starts, a.sequences, a.q_len, args.group, tile_rows,
                                        slot, &p->tile));
  } else {
    p->q = sequence_of(args, slot % a.sequences);
    p->tile = slot / a.sequences;
  }
  return p->tile >= 0 && p->tile * tile_rows < (int64_t)p->q.lq * args.group;
}

// The same by keys, the first ones first: in a causal sequence the most queries see them.  Where all
// workgroups run at once, two on a compute unit (`paired`), the second half comes in the other
// order, so that a long one shares its unit with a short one.
__device__ inline bool place_of_keys(const AttentionArgs& args, int tile_rows, int64_t block,
                                     Place* p) {
  const omq_attention_args& a = args.a;
  int64_t slot = block / a.k_heads;
  if (slot >= args.slots) return false;
  const int64_t half = (args.slots + 1) / 2;
  if (args.paired && slot >= half) slot = args.slots - 1 - (slot - half);
  p->kv = (int)(block % a.k_heads);
  if (a.q_starts) {
    p->q = sequence_of(args,
                       find_piece(a.k_starts, a.sequences, a.k_len, 1, tile_rows, slot, &p->tile));
  } else {
    p->q = sequence_of(args, slot % a.sequences);
    p->tile = slot / a.sequences;
  }
  return p->tile >= 0 && p->tile * tile_rows < p->q.room;
}

// What a lane's row sees of its sequence, and which keys the rows of its wave see.
struct Rows {
  int query, head;   // of the row, or of the last one
  bool there;
  int limit;         // keys that the row sees
  int least, most;   // that all of the wave's rows see, and that some do
  int block_most;    // that some row of the workgroup sees
};

template <int kTileRows_ = kTileRows>
__device__ inline Rows rows_of(const AttentionArgs& args, const Sequence& q, int kv, int r0,
                               int rows) {
  const int shift = q.lk - q.lq, lane = threadIdx.x & 63;
  const int first = r0 + kWaveRows * __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const auto sees = [&](int row) {
    return args.a.causal ? cut(query_of(args, row < rows ? row : rows - 1) + shift + 1, 0, q.lk)
                         : q.lk;
  };
  Rows x;
  const int mine = first + (lane & 31);
  x.there = mine < rows;
  const int row = x.there ? mine : rows - 1;
  x.query = query_of(args, row);
  x.head = kv * args.group + row - x.query * args.group;
  x.limit = sees(row);
  x.least = sees(first);
  x.most = first < rows ? sees(first + kWaveRows - 1) : 0;
  x.block_most = sees(r0 + kTileRows_ - 1);
  return x;
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

// A tile in LDS: kTileKeys rows of kDim columns, their 16-byte chunks exchanged within a row (chunk
// c of row r at place c ^ swap(r)) so that neither the chunks of one column from 16 rows nor a
// column's elements from four rows and 32 columns share banks.  Rows follow each other without
// gaps, as loads from memory straight into LDS need it.
template <class T, int kDim>
struct Tile {
  using Frag = typename Operand<T>::Frag;
  static constexpr int kChunk = Operand<T>::kChunk;
  static constexpr int kPitch = kDim * (int)sizeof(T);
  static constexpr int kPer = kPitch / 16;           // chunks of a row
  static constexpr int kChunks = kDim / kChunk;      // operands of a row
  static constexpr int kParts = kWaveRows / kChunk;  // operands of 32 rows down a column
  static constexpr int kBytes = kTileKeys * kPitch;

  __device__ static int swap(int r) {
    if constexpr (kPer == 4) return (r >> 2) & 3;
    if constexpr (sizeof(T) == 2)
      return kPer == 8 ? (((r >> 1) & 1) << 2) | ((r >> 2) & 3) : ((r & 3) << 2) | ((r >> 2) & 3);
    else
      return kPer == 8 ? (r >> 1) & 7
                       : (((r >> 2) & 1) << 3) | (((r >> 3) & 1) << 2) | (r & 3);
  }
  __device__ static int place(int r, int chunk) { return r * kPitch + ((chunk ^ swap(r)) << 4); }

  // Where a lane's operands are: of row lane % 32, and of its columns.  An operand's own address is
  // one exclusive or away (swap is a permutation of a row's bits); `renew` keeps the compiler from
  // forming all of them before a loop, for which there are no registers.
  struct Lane {
    int row, column;
    __device__ Lane() {
      const int lane = threadIdx.x & 63, half = lane >> 5;
      row = place(lane & 31, half);
      if constexpr (sizeof(T) == 2) {
        // 16 lanes address four rows of 16 columns, and get a column of four rows each
        const int c = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
        column = place(4 * half + ((lane & 15) >> 2), c >> 3) + (c & 4) * 2;
      } else {
        column = place(4 * half, (lane & 31) >> 2) + (lane & 3) * 4;
      }
    }
    __device__ void renew() { asm volatile("" : "+v"(row), "+v"(column)); }
  };

  // Chunk c of the row row0 + lane % 32 (row0 a multiple of 32).
  __device__ static Frag row(const char* tile, int row0, int c, const Lane& lane) {
    return *reinterpret_cast<const Frag*>(tile + row0 * kPitch + (lane.row ^ (c << 5)));
  }

  // Column col0 + lane % 32 of part t of the rows from row0, in the order of a product's registers
  // (row0 and col0 multiples of 32).
  __device__ static Frag column(const char* tile, int row0, int col0, int t, const Lane& lane) {
    if constexpr (sizeof(T) == 2) {
      const char* p = tile + (row0 + 16 * t) * kPitch;
      const int lo = lane.column ^ (col0 << 1), hi = lo ^ (swap(8) << 4);
      using S4 = short __attribute__((ext_vector_type(4)));
      using Lds = __attribute__((address_space(3))) S4;
      struct Both {
        S4 lo, hi;
      } v;
      v.lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds*)(p + lo));
      v.hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds*)(p + 8 * kPitch + hi));
      return __builtin_bit_cast(Frag, v);
    } else {
      Frag f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = 8 * t + i;
        f[i] = *reinterpret_cast<const float*>(
            tile + (row0 + r) * kPitch + (lane.column ^ (swap(r) << 4) ^ (col0 << 2)));
      }
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
// A hidden key's probability is 0, and 0 times an infinity or a NaN is NaN.  In tiles that a mask
// cuts, products take 0 in place of such values, and note it; what those among them that are seen
// make of a result is added when it has been stored (add_hidden).
//
// Puts 0 in place of an operand's values that are not finite (all bits of the exponent set: one
// more carries out of them) and says in `found` where there was one.
template <class T, class Frag>
__device__ inline Frag finite_only(const Frag& v, uint32_t& found) {
  constexpr uint32_t kExp = sizeof(T) == 4            ? 0x7F800000u
                            : std::is_same_v<T, bf16> ? 0x7F807F80u
                                                      : 0x7C007C00u;
  constexpr uint32_t kOne = sizeof(T) == 4            ? 0x00800000u
                            : std::is_same_v<T, bf16> ? 0x00800080u
                                                      : 0x04000400u;
  using U4 = uint32_t __attribute__((ext_vector_type(4)));
  U4 x = __builtin_bit_cast(U4, v);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t bad = ((x[i] & kExp) + kOne) & (sizeof(T) == 4 ? 0x80000000u : 0x80008000u);
    found |= bad;
    // (the sign's bit and those below it)
    x[i] &= sizeof(T) == 4 ? ~(uint32_t)((int32_t)bad >> 31) : ~((bad << 1) - (bad >> 15));
  }
  return __builtin_bit_cast(Frag, x);
}

// Keeps the compiler from moving instructions across: reads of LDS are under way this far ahead of
// the products that use them, and no further, for which there are no registers.
__device__ __attribute__((always_inline)) inline void here() {
  __builtin_amdgcn_sched_barrier(0);
}

// Products of two blocks of 32 rows with 32 rows in registers, each of its own tile, the second
// one's reads under way with the first one's products.
template <class T, int kDim>
__device__ __attribute__((always_inline)) inline void two_products(
    F16& s, const char* tile, int row0,
    const typename Operand<T>::Frag (&f)[kDim / Operand<T>::kChunk],
    F16& s2, const char* tile2, int row2,
    const typename Operand<T>::Frag (&f2)[kDim / Operand<T>::kChunk],
    const typename Tile<T, kDim>::Lane& lane) {
  using L = Tile<T, kDim>;
  typename L::Frag a[L::kChunks], b[L::kChunks];
#pragma unroll
  for (int c = 0; c < L::kChunks; ++c) a[c] = L::row(tile, row0, c, lane);
  here();
  s = F16{}, s2 = F16{};
#pragma unroll
  for (int c = 0; c < L::kChunks; ++c) {
    b[c] = L::row(tile2, row2, c, lane);
    s = mma(a[c], f[c], s);
  }
  here();
#pragma unroll
  for (int c = 0; c < L::kChunks; ++c) s2 = mma(b[c], f2[c], s2);
}

template <class T, int kDim>
__device__ __attribute__((always_inline)) inline void one_product(
    F16& s, const char* tile, int row0,
    const typename Operand<T>::Frag (&f)[kDim / Operand<T>::kChunk],
    const typename Tile<T, kDim>::Lane& lane) {
  using L = Tile<T, kDim>;
  typename L::Frag a[L::kChunks];
#pragma unroll
  for (int c = 0; c < L::kChunks; ++c) a[c] = L::row(tile, row0, c, lane);
  here();
  s = F16{};
#pragma unroll
  for (int c = 0; c < L::kChunks; ++c) s = mma(a[c], f[c], s);
}

// acc += (columns of the tile's 32 rows from row0) x w, a group of the columns' operands at a time;
// the first group is read (Columns::read) before w is formed.
template <class T, int kDim>
struct Columns {
  using L = Tile<T, kDim>;
  static constexpr int kAll = kDim / 32 * L::kParts, kGroup = kAll < 4 ? kAll : 4;
  typename L::Frag v[kGroup];

  __device__ __attribute__((always_inline)) void read(const char* tile, int row0, int group,
                                                      const typename L::Lane& lane) {
#pragma unroll
    for (int i = 0; i < kGroup; ++i) {
      const int at = group * kGroup + i;
      v[i] = L::column(tile, row0, at / L::kParts * 32, at % L::kParts, lane);
    }
  }
};

// cuts: a mask cuts the tile.  kTwice: w to twice the type's bits, what its rounding leaves in a
// second product.  beside(i): what runs beside product i of kAll.
struct Nothing {
  __device__ void operator()(int) const {}
};

template <class T, int kDim, bool kTwice, class Beside = Nothing>
__device__ __attribute__((always_inline)) inline void add_columns(
    F16 (&acc)[kDim / 32], Columns<T, kDim>& first, const char* tile, int row0, const F16& w,
    bool cuts, uint32_t& found, const typename Tile<T, kDim>::Lane& lane,
    Beside&& beside = Beside()) {
  using L = Tile<T, kDim>;
  using C = Columns<T, kDim>;
  constexpr bool kRest = kTwice && sizeof(T) == 2;
  typename L::Frag part[L::kParts], rest[kRest ? L::kParts : 1];
#pragma unroll
  for (int t = 0; t < L::kParts; ++t) {
    part[t] = L::part(w, t);
    if constexpr (kRest) {
      F16 left = w;
#pragma unroll
      for (int i = 0; i < L::kChunk / 2; ++i) left[t * (L::kChunk / 2) + i] -= (float)part[t][i];
      rest[t] = L::part(left, t);
    }
  }
  C now = first;
#pragma unroll
  for (int g = 0; g < C::kAll / C::kGroup; ++g) {
    C next;
    here();
    if (g + 1 < C::kAll / C::kGroup) next.read(tile, row0, g + 1, lane);
    if (cuts) {
#pragma unroll
      for (int i = 0; i < C::kGroup; ++i) now.v[i] = finite_only<T>(now.v[i], found);
    }
    here();
#pragma unroll
    for (int i = 0; i < C::kGroup; ++i) {
      const int d = (g * C::kGroup + i) / L::kParts, t = (g * C::kGroup + i) % L::kParts;
      acc[d] = mma(now.v[i], part[t], acc[d]);
      if constexpr (kRest) acc[d] = mma(now.v[i], rest[t], acc[d]);
      beside(g * C::kGroup + i);
    }
    now = next;
  }
  here();
}

// Adds to a stored row what the values that are not finite make of it, of the rows from `from` to
// `to` of a factor that it sees: themselves (a factor of probabilities), or NaN.  (Rows of tiles
// that no mask cut may be among them: an infinity twice is one.)
template <class T, bool kNan, class O, class RowAt>
__device__ inline void add_hidden(O* row, int dim, int from, int to, RowAt&& row_at) {
#pragma unroll 1
  for (int j = from; j < to; ++j) {
    const T* p = row_at(j);
#pragma unroll 1
    for (int d = 0; d < dim; ++d) {
      const float x = (float)p[d];
      if (!(__builtin_fabsf(x) < kInf32))
        row[d] = (O)((float)row[d] + (kNan ? __builtin_nanf("") : x));
    }
  }
}

// ---- loading and storing --------------------------------------------------------------------
// Eight columns of a row that is there, 0 from column dim on; kWhole: dim is a multiple of 8.
template <class T, bool kWhole>
__device__ inline Reg8<T> load_piece(const T* row, int col, int dim) {
  return block_of_raw<T, kWhole>(load_raw<T, kWhole>(row, col, dim), col, dim);
}

// The operands of a row: its chunks, 0 from column dim on.
template <class T, int kDim, bool kWhole>
__device__ inline void load_row(typename Operand<T>::Frag (&f)[kDim / Operand<T>::kChunk],
                                const T* row, int dim) {
  const int half = (threadIdx.x & 63) >> 5;
#pragma unroll
  for (int c = 0; c < kDim / Operand<T>::kChunk; ++c) {
    if constexpr (sizeof(T) == 2) {
      f[c] = load_piece<T, kWhole>(row, 16 * c + 8 * half, dim);
    } else {
      const Reg8<T> v = load_piece<T, kWhole>(row, 8 * c, dim);
#pragma unroll
      for (int i = 0; i < 4; ++i) f[c][i] = half ? v[4 + i] : v[i];
    }
  }
}

// Whether rows are whole chunks of 16 bytes on such a boundary, which can be loaded straight into
// LDS.
inline bool chunks_aligned(int dtype, int64_t dim, std::initializer_list<const void*> pointers,
                           std::initializer_list<int64_t> strides) {
  const int64_t size = dtype_size(dtype);
  bool ok = dim % 8 == 0;
  for (const void* p : pointers) ok = ok && on_16_bytes(p);
  for (const int64_t s : strides) ok = ok && s * size % 16 == 0;
  return ok;
}

// Keys and values for the loads straight into LDS; others pass through registers.  8 x 8 heads of
// 1024 keys of 64 columns, bf16: 28 us straight, 52 with rows 2 bytes off (of 128: 45 and 92).
inline bool direct_tiles(const omq_attention_args& a) {
  return chunks_aligned(a.dtype, a.dim, {a.k, a.v},
                        {a.k_seq_stride, a.k_row_stride, a.k_head_stride, a.v_seq_stride,
                         a.v_row_stride, a.v_head_stride});
}

// Zeros where a tile's rows have no column (from dim on): before the first load_tile, and a
// barrier between the two.
template <class T, int kDim, int kThreads = kWaves * kWave, int kRows = kTileKeys>
__device__ inline void clear_tile(char* tile, int dim) {
  if (dim == kDim) return;
  for (int i = threadIdx.x; i < kRows * Tile<T, kDim>::kPitch / 16; i += kThreads)
    *reinterpret_cast<uint4*>(tile + 16 * i) = make_uint4(0, 0, 0, 0);
}

// Loads kRows rows into LDS, the last of `rows` (at least one) again in place of those behind it;
// row_at(i): row i < rows.  kDirect: chunks_aligned; the loads are under way when this returns,
// tile_loads of them for every wave.
template <class T, int kDim, int kThreads, int kRows>
constexpr int tile_loads() {
  return kRows * Tile<T, kDim>::kPitch / (kThreads * 16);
}

template <class T, int kDim, bool kDirect, int kThreads = kWaves * kWave, int kRows = kTileKeys,
          class RowAt>
__device__ inline void load_tile(char* tile, int rows, int dim, RowAt&& row_at) {
  using L = Tile<T, kDim>;
  if constexpr (kDirect) {
    constexpr int kEach = 16 / (int)sizeof(T), kStep = kThreads * 16;  // bytes at a time
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r0 = (int)threadIdx.x / L::kPer, place = threadIdx.x % L::kPer;
    // (the places of a row repeat with the steps where those are 16 rows or more)
    constexpr bool kSame = kStep / L::kPitch >= 16;
    if (!kSame || (place ^ L::swap(r0)) * kEach < dim) {
#pragma unroll
      for (int i = 0; i < tile_loads<T, kDim, kThreads, kRows>(); ++i) {
        const int r = r0 + i * (kStep / L::kPitch), chunk = place ^ L::swap(kSame ? r0 : r);
        if (kSame || chunk * kEach < dim)
          __builtin_amdgcn_global_load_lds(
              (const __attribute__((address_space(1))) void*)(row_at(r < rows ? r : rows - 1) +
                                                              chunk * kEach),
              (__attribute__((address_space(3))) void*)(tile + i * kStep + wave * kWave * 16), 16,
              0, 0);
      }
    }
  } else {
    constexpr int kPieces = kDim / 8;
#pragma unroll 1
    for (int i = threadIdx.x; i < kRows * kPieces; i += kThreads) {
      const int r = i / kPieces, col = i % kPieces * 8;
      const Reg8<T> v = load_piece<T, false>(row_at(r < rows ? r : rows - 1), col, dim);
      using Frag = typename L::Frag;
      Frag f[sizeof(T) / 2];
      __builtin_memcpy(f, &v, sizeof(v));
#pragma unroll
      for (int h = 0; h < (int)sizeof(T) / 2; ++h)
        *reinterpret_cast<Frag*>(tile + L::place(r, col * (int)sizeof(T) / 16 + h)) = f[h];
    }
  }
}

// A lane's place in the rows of a tile that are all there and lie as far apart at every step of its
// loads: bytes from the tile's first row, the same for every tile.  A load then has a scalar
// address and a 32-bit one, where a lane's rows otherwise take some ten instructions a load.
template <class T, int kDim>
struct EvenRows {
  using L = Tile<T, kDim>;
  static constexpr int kStep = kWaves * kWave * 16;
  static constexpr int kRowsAStep = kStep / L::kPitch;
  static constexpr int kPeriod = kRowsAStep >= 16 ? 1 : 16 / kRowsAStep;  // of a row's places
  static constexpr int kEach = 16 / (int)sizeof(T);
  uint32_t own[kPeriod];
  bool on;  // the lane has columns (kPeriod 1; all lanes have where the columns are kDim)

  // Whether rows can be taken so: at most 2^31 bytes apart.
  static bool possible(int dim, int64_t farthest) {
    return (kPeriod == 1 || dim == kDim) && farthest * (int64_t)sizeof(T) < (1ll << 31);
  }

  // at(r): elements from the first row to row r.
  template <class At>
  __device__ EvenRows(int dim, At&& at) {
    const int r = (int)threadIdx.x / L::kPer, place = threadIdx.x % L::kPer;
#pragma unroll
    for (int i = 0; i < kPeriod; ++i) {
      const int chunk = place ^ L::swap(r + i * kRowsAStep);
      own[i] = (uint32_t)((at(r) + chunk * kEach) * (int64_t)sizeof(T));
      on = kPeriod > 1 || chunk * kEach < dim;
    }
  }

  // first: the tile's first row; step: elements from a load's rows to the next one's.
  __device__ __attribute__((always_inline)) void load(char* tile, const T* first,
                                                      int64_t step) const {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (!on) return;
#pragma unroll
    for (int i = 0; i < L::kBytes / kStep; ++i)
      __builtin_amdgcn_global_load_lds(
          (const __attribute__((address_space(1))) void*)(reinterpret_cast<const char*>(
                                                              first + i * step) +
                                                          own[i % kPeriod]),
          (__attribute__((address_space(3))) void*)(tile + i * kStep + wave * kWave * 16), 16, 0,
          0);
  }
};

template <class T, int kDim>
bool even_keys(const omq_attention_args& a) {
  const int64_t far = a.k_row_stride > a.v_row_stride ? a.k_row_stride : a.v_row_stride;
  return EvenRows<T, kDim>::possible(a.dim, far < (1ll << 31) ? kTileKeys * far + kDim : far);
}

// The loads into LDS of this wave have arrived, and all waves come here.
__device__ inline void tiles_ready() {
  __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
  __syncthreads();
}

// Stores a lane's column of a result [kDim columns of a row, 32 rows] as a row, times `scale`.
// kWhole: dim is a multiple of 8.
template <class T, int kDim, bool kWhole>
__device__ inline void store_column(T* row, const F16 (&x)[kDim / 32], float scale, int dim) {
#pragma unroll
  for (int d = 0; d < kDim / 32; ++d)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const int col = 32 * d + result_row(r);
      using V4 __attribute__((aligned(sizeof(T)))) = T __attribute__((ext_vector_type(4)));
      if (kWhole ? col < dim : col + 4 <= dim) {
        *reinterpret_cast<V4*>(row + col) =
            V4{(T)(x[d][r] * scale), (T)(x[d][r + 1] * scale), (T)(x[d][r + 2] * scale),
               (T)(x[d][r + 3] * scale)};
      } else if (!kWhole) {
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
  if (r.group > 1) {  // exact for rows below 2^31
    int log = 0;
    while ((1ll << log) < r.group) ++log;
    r.group_mul = (uint32_t)((1ull << (31 + log)) / r.group + 1);
    r.group_shift = log - 1;
  }
  return r;
}

// The tiles a key head of a launch over `rows` units of `group` rows each (of a sequence, or of
// all packed ones).
inline void tiles_of(AttentionArgs* r, int64_t rows, int64_t group, int64_t tile) {
  r->batch_tiles = ceil_div(rows * group, tile);
  r->slots = r->a.q_starts ? rows * group / tile + r->a.sequences + 2
                           : r->batch_tiles * r->a.sequences;
}

// f(element, columns that are held, whether tiles go straight into LDS) for a launch.
template <class F>
void with_head(int dtype, int dim, bool direct, F&& f) {
  const auto loaded = [&](auto t, auto held) {
    if (direct) return f(t, held, std::true_type{});
    return f(t, held, std::false_type{});
  };
  const auto sized = [&](auto t) {
    if (dim <= 32) return loaded(t, std::integral_constant<int, 32>{});
    if (dim <= 64) return loaded(t, std::integral_constant<int, 64>{});
    return loaded(t, std::integral_constant<int, 128>{});
  };
  if (dtype == OMQ_NET_F32) return sized(float{});
  if (dtype == OMQ_NET_BF16) return sized(bf16{});
  return sized(f16{});
}

}  // namespace omq_net
