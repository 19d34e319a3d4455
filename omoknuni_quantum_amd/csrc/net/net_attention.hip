// Attention with grouped heads over batches, packed sequences and caches (gfx950).
//
// One pass over the keys with the running maximum m and sum l of a row's softmax:
//   s_ij = scale q_i.k_j;  m' = max(m, s);  l' = e^(m - m') l + sum e^(s - m');
//   o' = e^(m - m') o + sum e^(s - m') v;   out = o / l,  lse = m + log l
// A workgroup has 128 rows (queries x heads of a group), a wave 32 of them, in registers: queries,
// the sums of the output and the softmax's m and l.  64 keys and values at a time pass through
// LDS.  A probability is rounded to the elements' type for the second product, half a step of the
// type at most, as the output's own rounding; m and l are float32.
//
// Bound by a wave's products, its exponentials and its reads of LDS, which overlap only in part:
// eight causal texts of up to 8192 with 32 heads over 8 of 128, bf16: 1090 to 1216 us over several
// cards, 860 to 960 TFLOP/s (a large product of matrices: 1336), matrix cores 45 % busy.  256 boards
// of 49 to 361 cells with 8 heads of 64, float16: 75 us, of 128-row tiles that are half full; 32
// boards of 225 cells: 12.7 us; 64 of 225 cells with 4 heads of 32, float32: 28.
#include "net_attention.h"

namespace omq_net {
namespace {

// Probabilities are formed about a maximum that follows the running one only where that has grown
// by more than a factor of 2^8: the sums' rescaling, a product for each of a row's columns, is
// left out for most tiles, and a probability is at most 2^8.  Float16 holds 2^15 and loses bits below
// 2^-14: its probabilities are taken times 2^7, and so are their sums l and o.
constexpr float kLag = 8.0f;
template <class T>
constexpr float kUp = std::is_same_v<T, f16> ? 7.0f : 0.0f;  // log2

// A row's output so far: sums about the maximum m; l over this half's keys.
template <int kDim>
struct Softmax {
  F16 o[kDim / 32] = {};
  float m = -kInf32, l = 0.0f;
  uint32_t found = 0;
};

template <class T>
__device__ inline float lse_of(float m, float l, float scale) {
  constexpr float kDown = std::is_same_v<T, f16> ? 0x1p-7f : 1.0f;  // 2^-kUp
  return l == 0.0f ? -kInf32 : fmaf(m, scale, __builtin_amdgcn_logf(l * kDown) * 0.6931471805599453f);
}

// Attends to one or two blocks of 32 keys from k0, of which the row sees those below `limit`; cuts:
// some row of the wave does not see all of them.
template <class T, int kDim, int kBlocks>
__device__ __attribute__((always_inline)) inline void attend(
    Softmax<kDim>& x, const char* keys, const char* values,
    const typename Operand<T>::Frag (&qf)[kDim / Operand<T>::kChunk], int k0, bool cuts, int limit,
    float scale, const typename Tile<T, kDim>::Lane& lane) {
  F16 s[kBlocks];
  if constexpr (kBlocks == 2)
    two_products<T, kDim>(s[0], keys, 0, qf, s[1], keys, 32, qf, lane);
  else
    one_product<T, kDim>(s[0], keys, 0, qf, lane);
  Columns<T, kDim> columns;
  columns.read(values, 0, 0, lane);
  here();
  if (cuts) {
#pragma unroll
    for (int b = 0; b < kBlocks; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (k0 + 32 * b + result_row(r) >= limit) s[b][r] = -kInf32;
  }
  float top = -kInf32;
#pragma unroll
  for (int b = 0; b < kBlocks; ++b)
#pragma unroll
    for (int r = 0; r < 16; ++r) top = fmaxf(top, s[b][r]);
  top = fmaxf(top, other_half(top));
  if (__any((top - x.m) * scale > kLag)) {  // (m is -inf at first)
    const float next = fmaxf(x.m, top);
    const float keep = next == -kInf32 ? 1.0f : __builtin_amdgcn_exp2f((x.m - next) * scale);
    x.m = next;
    x.l *= keep;
#pragma unroll
    for (int d = 0; d < kDim / 32; ++d) x.o[d] *= keep;
  }
  const float base = (x.m == -kInf32 ? 0.0f : x.m * scale) - kUp<T>;
  float l = 0.0f;  // (a sum of its own: each step of a long one would round at its size)
  const auto form = [&](int b, int r) __attribute__((always_inline)) {
    s[b][r] = __builtin_amdgcn_exp2f(fmaf(s[b][r], scale, -base));
    l += s[b][r];
  };
  here();
#pragma unroll
  for (int r = 0; r < 16; ++r) form(0, r);
  if constexpr (kBlocks == 1) {
    add_columns<T, kDim, false>(x.o, columns, values, 0, s[0], cuts, x.found, lane);
  } else {
    // (a wave's products run while it forms the other block's probabilities)
    constexpr int kAll = Columns<T, kDim>::kAll, kEach = 16 / kAll > 0 ? 16 / kAll : 1;
    add_columns<T, kDim, false>(x.o, columns, values, 0, s[0], cuts, x.found, lane, [&](int i) {
#pragma unroll
      for (int r = 0; r < kEach; ++r)
        if (i * kEach + r < 16) form(1, i * kEach + r);
      here();
    });
    columns.read(values, 32, 0, lane);
    here();
    add_columns<T, kDim, false>(x.o, columns, values, 32, s[1], cuts, x.found, lane);
  }
  x.l += l;
}

template <class T, int kDim, bool kDirect>
__global__ __launch_bounds__(kWaves* kWave, (waves_per_simd<T, kDim>())) void
attention_kernel(AttentionArgs args) {
  using L = Tile<T, kDim>;
  __shared__ __attribute__((aligned(1024))) char keys0[L::kBytes], keys1[L::kBytes];
  __shared__ __attribute__((aligned(1024))) char values0[L::kBytes], values1[L::kBytes];
  const omq_attention_args& a = args.a;
  Place at;
  if (!place_of_queries(args, kTileRows, block_index(), &at)) return;
  const Sequence& q = at.q;
  const int rows = (int)((int64_t)q.lq * args.group), lane = threadIdx.x & 63;
  const Rows x = rows_of(args, q, at.kv, (int)(at.tile * kTileRows), rows);

  const T* k_rows = static_cast<const T*>(a.k) + q.k_at + at.kv * a.k_head_stride;
  const T* v_rows = static_cast<const T*>(a.v) + q.v_at + at.kv * a.v_head_stride;
  const EvenRows<T, kDim> k_own(a.dim, [&](int r) { return r * a.k_row_stride; });
  const EvenRows<T, kDim> v_own(a.dim, [&](int r) { return r * a.v_row_stride; });
  const auto load = [&](int k0, char* keys, char* values) {
    if (kDirect && args.even && q.lk - k0 >= kTileKeys) {
      constexpr int kRowsAStep = EvenRows<T, kDim>::kRowsAStep;
      k_own.load(keys, k_rows + k0 * a.k_row_stride, kRowsAStep * a.k_row_stride);
      v_own.load(values, v_rows + k0 * a.v_row_stride, kRowsAStep * a.v_row_stride);
      return;
    }
    load_tile<T, kDim, kDirect>(keys, q.lk - k0, a.dim, [&](int i) {
      return k_rows + (int64_t)(k0 + i) * a.k_row_stride;
    });
    load_tile<T, kDim, kDirect>(values, q.lk - k0, a.dim, [&](int i) {
      return v_rows + (int64_t)(k0 + i) * a.v_row_stride;
    });
  };
  if (kDirect && a.dim < kDim) {
    clear_tile<T, kDim>(keys0, a.dim), clear_tile<T, kDim>(keys1, a.dim);
    clear_tile<T, kDim>(values0, a.dim), clear_tile<T, kDim>(values1, a.dim);
    __syncthreads();
  }
  if (x.block_most > 0) load(0, keys0, values0);
  typename L::Frag qf[L::kChunks];
  load_row<T, kDim, kDirect>(qf, static_cast<const T*>(a.q) + q.q_at + x.query * a.q_row_stride +
                            x.head * a.q_head_stride, a.dim);

  Softmax<kDim> sum;
  typename L::Lane own;
  const auto step = [&](int k0, const char* keys, const char* values, char* next_keys,
                        char* next_values) __attribute__((always_inline)) {
    tiles_ready();
    own.renew();
    if (k0 + kTileKeys < x.block_most) load(k0 + kTileKeys, next_keys, next_values);
    if (k0 < x.most)
      attend<T, kDim, 2>(sum, keys, values, qf, k0, k0 + kTileKeys > x.least, x.limit,
                         args.score_scale, own);
  };
  // (two steps a turn, so that the tiles' arrays are told apart: the compiler would wait for all
  // loads under way before it reads an array that they may write)
  for (int k0 = 0; k0 < x.block_most; k0 += 2 * kTileKeys) {
    step(k0, keys0, values0, keys1, values1);
    if (k0 + kTileKeys < x.block_most) step(k0 + kTileKeys, keys1, values1, keys0, values0);
  }
  const float l = sum.l + other_half(sum.l);
  const bool hidden = __any(sum.found != 0) && lane < 32;  // (a lane finds for other lanes' rows)
  if (!x.there) return;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  const int64_t out_row = (q.q_first + x.query) * a.q_heads + x.head;
  T* out = static_cast<T*>(args.out) + out_row * a.dim;
  store_column<T, kDim, kDirect>(out, sum.o, inv, a.dim);
  if (__builtin_expect(hidden, 0))
    add_hidden<T, false>(out, a.dim, x.least / kTileKeys * kTileKeys, x.limit,
                         [=](int j) { return v_rows + j * a.v_row_stride; });
  if (args.lse && lane < 32) args.lse[out_row] = lse_of<T>(sum.m, l, a.scale);
}

// ---- few rows ---------------------------------------------------------------------------------
// Where a sequence has few rows (single tokens over a cache), bound by reading its keys and values:
// a workgroup is one wave, with 32 rows and a part of the keys, 32 of them at a time, loaded while
// the 32 before are attended to.  The parts' sums are joined in their order by a second launch.  64
// caches of up to 8192 keys with 32 heads over 8 of 128, bf16: 213 us, 5.2 TB/s, and 4 for the join.
constexpr int kPartKeys = 32;

template <class T, int kDim, bool kDirect>
__global__ __launch_bounds__(kWave) void attention_few_kernel(AttentionArgs args) {
  using L = Tile<T, kDim>;
  constexpr int kLoads = 2 * tile_loads<T, kDim, kWave, kPartKeys>();
  static_assert(kLoads < 64);
  constexpr int kBytes = kPartKeys * L::kPitch;
  __shared__ __attribute__((aligned(1024))) char keys0[kBytes], keys1[kBytes];
  __shared__ __attribute__((aligned(1024))) char values0[kBytes], values1[kBytes];
  const omq_attention_args& a = args.a;
  const int64_t block = block_index();
  const int split = (int)(block % args.splits);
  Place at;
  if (!place_of_queries(args, kWaveRows, block / args.splits, &at)) return;
  const Sequence& q = at.q;
  const int rows = (int)((int64_t)q.lq * args.group), lane = threadIdx.x;
  const Rows x = rows_of<kWaveRows>(args, q, at.kv, (int)(at.tile * kWaveRows), rows);
  // this part's keys
  const int tiles_in_all = (x.most + kPartKeys - 1) / kPartKeys;
  const int each = (tiles_in_all + args.splits - 1) / args.splits;
  const int64_t begin64 = (int64_t)split * each * kPartKeys;
  const int begin = begin64 < x.most ? (int)begin64 : x.most;
  const int end = begin + each * kPartKeys < x.most ? begin + each * kPartKeys : x.most;

  const T* k_rows = static_cast<const T*>(a.k) + q.k_at + at.kv * a.k_head_stride;
  const T* v_rows = static_cast<const T*>(a.v) + q.v_at + at.kv * a.v_head_stride;
  const auto load = [&](int k0, char* keys, char* values) {
    load_tile<T, kDim, kDirect, kWave, kPartKeys>(keys, q.lk - k0, a.dim, [&](int i) {
      return k_rows + (int64_t)(k0 + i) * a.k_row_stride;
    });
    load_tile<T, kDim, kDirect, kWave, kPartKeys>(values, q.lk - k0, a.dim, [&](int i) {
      return v_rows + (int64_t)(k0 + i) * a.v_row_stride;
    });
  };
  if (kDirect && a.dim < kDim) {
    for (char* t : {keys0, keys1, values0, values1})
      clear_tile<T, kDim, kWave, kPartKeys>(t, a.dim);
    __syncthreads();
  }
  typename L::Frag qf[L::kChunks];
  load_row<T, kDim, kDirect>(qf, static_cast<const T*>(a.q) + q.q_at + x.query * a.q_row_stride +
                                     x.head * a.q_head_stride, a.dim);
  if (begin < end) load(begin, keys0, values0);
  Softmax<kDim> sum;
  typename L::Lane own;
  const auto step = [&](int k0, const char* keys, const char* values, char* next_keys,
                        char* next_values) __attribute__((always_inline)) {
    if (k0 + kPartKeys < end) {
      load(k0 + kPartKeys, next_keys, next_values);
      // this tile's loads have arrived when no more are under way than the next one's
      __builtin_amdgcn_s_waitcnt((kLoads & 15) | 0x0F70 | ((kLoads >> 4) << 14));
    } else {
      __builtin_amdgcn_s_waitcnt(0x0F70);
    }
    // (a barrier would wait for the next tile; LDS accesses of one wave are in order)
    asm volatile("" ::: "memory");
    __builtin_amdgcn_wave_barrier();
    own.renew();
    attend<T, kDim, 1>(sum, keys, values, qf, k0, k0 + kPartKeys > x.least, x.limit,
                       args.score_scale, own);
  };
  for (int k0 = begin; k0 < end; k0 += 2 * kPartKeys) {  // (as above)
    step(k0, keys0, values0, keys1, values1);
    if (k0 + kPartKeys < end) step(k0 + kPartKeys, keys1, values1, keys0, values0);
  }
  const float l = sum.l + other_half(sum.l);
  const bool hidden = __any(sum.found != 0) && lane < 32;  // (as above)
  if (!x.there) return;
  const int64_t out_row = (q.q_first + x.query) * a.q_heads + x.head;
  const int least = x.least / kPartKeys * kPartKeys;
  const int from = begin > least ? begin : least, to = end < x.limit ? end : x.limit;
  const auto value = [=](int j) { return v_rows + j * a.v_row_stride; };
  if (args.splits == 1) {
    T* out = static_cast<T*>(args.out) + out_row * a.dim;
    store_column<T, kDim, kDirect>(out, sum.o, l == 0.0f ? 0.0f : 1.0f / l, a.dim);
    if (hidden) add_hidden<T, false>(out, a.dim, from, to, value);
    if (args.lse && lane < 32) args.lse[out_row] = lse_of<T>(sum.m, l, a.scale);
    return;
  }
  const int64_t part = split * args.out_rows + out_row;
  store_column<float, kDim, kDirect>(args.parts + part * a.dim, sum.o, 1.0f, a.dim);
  if (hidden) add_hidden<T, false>(args.parts + part * a.dim, a.dim, from, to, value);
  if (lane < 32) args.part_stats[part] = make_float2(sum.m, l);
}

// A row of the output from its parts (at most 64), a wave a row.
template <class T>
__global__ __launch_bounds__(256) void attention_join_kernel(AttentionArgs args) {
  const int64_t row = block_index() * 4 + row_slot<kWave>();
  if (row >= args.out_rows) return;
  const int lane = threadIdx.x & 63, dim = args.a.dim;
  float2 mine = make_float2(-kInf32, 0.0f);
  if (lane < args.splits) mine = args.part_stats[lane * args.out_rows + row];
  const float m = lanes_reduce<Max, kWave>(mine.x);
  // (a part without keys has a sum of 0; NaN is a sum)
  const float w = mine.x == -kInf32 ? (mine.y == 0.0f ? 0.0f : 1.0f)
                                    : __builtin_amdgcn_exp2f((mine.x - m) * args.score_scale);
  const float l = lanes_reduce<Sum, kWave>(mine.y == 0.0f ? 0.0f : w * mine.y);
  const float scale = l == 0.0f ? 0.0f : w / l;
  float x[2] = {};
  constexpr int kAhead = 8;  // (loads under way)
  for (int s0 = 0; s0 < args.splits; s0 += kAhead) {
    float part[kAhead][2];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int s = s0 + i < args.splits ? s0 + i : args.splits - 1;
      const float* from = args.parts + (s * args.out_rows + row) * dim;
      part[i][0] = from[lane < dim ? lane : 0];
      part[i][1] = from[lane + 64 < dim ? lane + 64 : 0];
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const float f = s0 + i < args.splits ? __shfl(scale, s0 + i) : 0.0f;
      // (a part without keys is zeros; of weight 0, nothing beside the others)
#pragma unroll
      for (int d = 0; d < 2; ++d) x[d] = f != 0.0f ? fmaf(f, part[i][d], x[d]) : x[d];
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
    if (lane + 64 * i < dim)
      static_cast<T*>(args.out)[row * dim + lane + 64 * i] = (T)x[i];
  if (args.lse && lane == 0) args.lse[row] = lse_of<T>(m, l, args.a.scale);
}

// Whether a call takes the kernel for few rows, and with how many parts (all us, bf16 unless said).
//  * Parts fill the chip where the pairs of heads and 32 rows do not, with 1024 waves: 64 tokens x 2
//    heads over 2048 keys of 128: 27 (parts), 41 (wide); 16 x 8 heads x 64 rows over 2048 of 64: 24,
//    31; twice and four times the waves cost 10 % and more there, of parts written and read.
//  * 4096 waves where lengths differ and there are few rows to write (64 x 8 heads x 1 row over up
//    to 4096: 60, with 1024 waves 93, wide 67), and for float32, whose products take 8 times as long
//    (64 x 8 x 1 over 4096: 273, 350, 286).  Half the keys a part with elements of twice the size
//    (512 keys of 64, float32: 13 for 18).
//  * At least 4 parts and 2 KB of a column's keys: 128 rows x 8 heads over 512 of 64 take 10 either
//    way, over 256 7 (wide) and 9.
//  * Without parts it serves float32 with rows enough for the chip: 512 x 8 heads over 128 of 64: 81,
//    wide 145, whose second wave on a SIMD has no registers (bf16: 23.6 and 24.8, but 64 x 8 heads x
//    32 rows over 512: 15.8 and 13.9).
bool few_rows(const omq_attention_args& a, int* splits, int64_t* out_rows) {
  const int64_t group = a.q_heads / a.k_heads, n = a.q_starts ? a.sequences : 1;
  const int64_t all = a.q_starts ? 1 : a.sequences;
  *out_rows = all * a.q_len * a.q_heads;
  const int64_t rows = n > 0 ? ceil_div(a.q_len * group, n) : 0;  // (of a sequence, in the mean)
  const int64_t keys = n > 0 ? ceil_div(a.k_len, n) : 0;
  const int64_t sequences = a.sequences > 0 ? a.sequences : 1;
  const int64_t units = ceil_div(rows > 0 ? rows : 1, kWaveRows) * sequences * a.k_heads;
  const int64_t size = dtype_size(a.dtype);
  const bool uneven = a.q_starts || a.k_lengths;
  const int64_t waves = rows <= kWaveRows && (size == 4 || (uneven && rows <= 8)) ? 4096 : 1024;
  int64_t parts = waves / units;
  const int64_t most = keys * size / (8 * kPartKeys);
  parts = parts < most ? parts : most;
  parts = parts < 64 ? parts : 64;
  const bool split = parts >= 4 && keys * size >= 2048;
  *splits = split ? (int)parts : 1;
  return split || (size == 4 && rows <= kWaveRows && units >= 512);
}

int64_t parts_bytes(const omq_attention_args& a, int splits, int64_t out_rows) {
  return splits > 1 ? splits * out_rows * (a.dim + 2) * (int64_t)sizeof(float) : 0;
}

}  // namespace

int check_attention(const char* name, const omq_attention_args* a) {
  if (!a) return net_fail(OMQ_NET_E_ARG, "%s: a null array", name);
  if (!dtype_known(a->dtype)) return net_fail(OMQ_NET_E_ARG, "%s: heads of type %d", name, a->dtype);
  if (a->sequences < 0 || a->q_len < 0 || a->k_len < 0 || a->q_heads < 1 || a->k_heads < 1 ||
      a->dim < 1 || a->q_heads % a->k_heads)
    return net_fail(OMQ_NET_E_ARG,
                    "%s: sequences %lld, queries %lld, keys %lld, heads %d over %d, dim %d", name,
                    (long long)a->sequences, (long long)a->q_len, (long long)a->k_len, a->q_heads,
                    a->k_heads, a->dim);
  const int64_t n = a->q_starts ? 1 : a->sequences;
  const int64_t most = OMQ_NET_MAX_COUNT - 4095;  // (a tile past the last is counted in 32 bits)
  if (a->dim > OMQ_NET_MAX_HEAD_DIM || a->sequences > most || a->q_len > most || a->k_len > most ||
      a->q_len * a->q_heads > most || (n > 0 && a->q_len * a->q_heads > most / n))
    return net_fail(OMQ_NET_E_LIMIT,
                    "%s: sequences %lld of %lld queries and %lld keys (at most %d), %d heads (rows "
                    "of heads of queries at most %d), dim %d (at most %d)",
                    name, (long long)a->sequences, (long long)a->q_len, (long long)a->k_len,
                    (int)most, a->q_heads, (int)most, a->dim, OMQ_NET_MAX_HEAD_DIM);
  if (!(a->scale > 0.0f && a->scale <= 0x1p127f))  // (its product with log2 e is finite)
    return net_fail(OMQ_NET_E_ARG, "%s: scale %g must be above 0 and at most 2^127", name, a->scale);
  if (!a->q_starts != !a->k_starts)
    return net_fail(OMQ_NET_E_ARG, "%s: starts of queries and keys, or of neither", name);
  if (a->q_seq_stride < 0 || a->q_row_stride < 0 || a->q_head_stride < 0 || a->k_seq_stride < 0 ||
      a->k_row_stride < 0 || a->k_head_stride < 0 || a->v_seq_stride < 0 || a->v_row_stride < 0 ||
      a->v_head_stride < 0)
    return net_fail(OMQ_NET_E_ARG, "%s: negative stride", name);
  const bool queries = a->q_len > 0 && n > 0, keys = a->k_len > 0 && n > 0;
  if ((queries && !a->q) || (keys && (!a->k || !a->v)))
    return net_fail(OMQ_NET_E_ARG, "%s: a null array", name);
  return OMQ_NET_OK;
}

}  // namespace omq_net

using namespace omq_net;

extern "C" {

int64_t omq_attention_forward_workspace(const omq_attention_args* a) {
  if (const int rc = check_attention("omq_attention_forward_workspace", a)) return rc;
  int splits;
  int64_t out_rows;
  return few_rows(*a, &splits, &out_rows) ? parts_bytes(*a, splits, out_rows) : 0;
}

int omq_attention_forward(const omq_attention_args* a, void* out, float* lse, void* workspace,
                          int64_t workspace_bytes, void* stream) {
  const char* name = "omq_attention_forward";
  if (int rc = check_attention(name, a)) return rc;
  if (a->q_len == 0 || (a->sequences == 0 && !a->q_starts)) return OMQ_NET_OK;
  if (!out) return net_fail(OMQ_NET_E_ARG, "%s: a null array", name);
  AttentionArgs args = attention_layout(*a);
  args.out = out, args.lse = lse;
  const bool few = few_rows(*a, &args.splits, &args.out_rows);
  const int64_t need = few ? parts_bytes(*a, args.splits, args.out_rows) : 0;
  if (need > 0 && (!workspace || workspace_bytes < need || !on_16_bytes(workspace)))
    return net_fail(OMQ_NET_E_ARG, "%s: workspace of %lld bytes at %p, %lld on a 16-byte boundary "
                    "needed", name, (long long)workspace_bytes, workspace, (long long)need);
  hipStream_t st = (hipStream_t)stream;
  if (!few) {
    tiles_of(&args, a->q_len, args.group, kTileRows);
    const dim3 grid = grid_of(args.slots * a->k_heads, kWaves * kWave);
    with_head(a->dtype, a->dim, direct_tiles(*a), [&](auto t, auto dim, auto direct) {
      args.even = even_keys<decltype(t), dim.value>(*a);
      attention_kernel<decltype(t), dim.value, direct.value><<<grid, kWaves * kWave, 0, st>>>(args);
    });
    return net_status(name);
  }
  tiles_of(&args, a->q_len, args.group, kWaveRows);
  if (need > 0) {
    args.part_stats = static_cast<float2*>(workspace);
    args.parts = static_cast<float*>(workspace) + 2 * args.splits * args.out_rows;
  }
  const dim3 grid = grid_of(args.slots * a->k_heads * args.splits, kWave);
  with_head(a->dtype, a->dim, direct_tiles(*a), [&](auto t, auto dim, auto direct) {
    attention_few_kernel<decltype(t), dim.value, direct.value><<<grid, kWave, 0, st>>>(args);
  });
  if (args.splits > 1) {
    const dim3 rows = grid_of(ceil_div(args.out_rows, 4), 256);
    if (a->dtype == OMQ_NET_F32)
      attention_join_kernel<float><<<rows, 256, 0, st>>>(args);
    else if (a->dtype == OMQ_NET_BF16)
      attention_join_kernel<bf16><<<rows, 256, 0, st>>>(args);
    else
      attention_join_kernel<f16><<<rows, 256, 0, st>>>(args);
  }
  return net_status(name);
}

}  // extern "C"
