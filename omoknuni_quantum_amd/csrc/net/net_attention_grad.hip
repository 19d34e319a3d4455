// Gradients of the attention (gfx950).  With the forward pass's p_ij = e^(s_ij - lse_i) formed
// again from its lse, and g the gradient of out:
//   delta_i = g_i . out_i;   ds_ij = p_ij (g_i . v_j - delta_i) scale
//   dq_i = sum_j ds_ij k_j;  dk_j = sum_i ds_ij q_i;  dv_j = sum_i p_ij g_i
// Two launches, each with its sums in registers: by queries (dq, and delta for the other) and by
// keys (dk and dv).  Scores are formed in both, and no sum is split over workgroups, which would
// take atomics or float32 copies of dq; every result is the same bits at every call.  For five
// products of the formulas that is seven; in 16 bits dq takes one more (below), and where the sums
// by keys are apart (sums_apart) the scores one more: eight up to 64 columns, nine above.  Rows of
// queries that share a key head are rows of one sum.
//
// Two causal sequences of 4096 with 16 heads over 4 of 128, bf16: 285 us by queries, 515 by keys
// (960 and 670 TFLOP/s of what they multiply); 256 boards of 49 to 361 cells with 8 heads over 4 of
// 64, float16: 116 and 143 us; 64 of 225 cells with 4 heads of 32, float32: 40 and 52.  Matrix cores
// are busy for a fifth of the time (boards) to a half (by queries), in float32 for three fifths: a
// wave's products, its exponentials and its reads of LDS follow one another, and two waves a SIMD,
// for which the registers are just enough, cover a part of that.  By keys the workgroups of a causal
// sequence are few and of all lengths; the rows that they read do not bound them (half the traffic,
// by an order of the workgroups in which the memory's parts share them, took as long).
//
// ds is rounded to the elements' type for its products, times scale, without which float16 would
// overflow earlier.  Its sum over a row is 0 but for what the rounding of out took from delta, which
// the first launch so finds and the second has again; dq, for which that comes too late, has ds to
// twice the type's bits instead, and rows that see few keys (of whose outs the roundings weigh
// most) form their ds twice: where a workgroup's keys are two tiles, both stay in LDS and the first
// time over them only corrects delta.  (With none of it, the gradients are off by 1.6 times their own
// rounding and more, those of few keys by 2 and more; with all of it by 1.1 to 1.4 times.)
#include "net_attention.h"

namespace omq_net {
namespace {

// How far from 1 the sum of a whole row's probabilities may be: lse's rounding takes it 2^-25 |lse|
// away and its sum's less; the share of hidden keys that passes for rounding is below out's own
// (2^-9, 2^-12).
constexpr float kWhole = 0x1p-12f;

// float16 holds 2^-14 to 2^16 in full.  A slope is a probability, 1 / keys or so, times a gradient
// of out, which a mean over a batch makes small: its float16 products take it times a power of two,
// a column's own (a query's of dq, a key's of dk), that puts the column's largest slope so far at 2^9
// to 2^15; the sums so far are brought along where it changes.  (Without, dq and dk of 225 keys are
// off by 1e-2 of their size where grad_out is of 1e-4; it takes 3 % of packed boards' training, 323
// -> 334 us.)
template <class T>
struct Lift {
  static constexpr bool kOn = std::is_same_v<T, f16>;
  float up, down;  // the power of two (over that of the probabilities), and what undoes both
  float most = 0.0f;  // that a slope may be, times the power of two; 0 before the first one

  // What the slopes s and the sums so far have to be multiplied by, 1 mostly (then `changed` is false
  // throughout the wave).
  __device__ __attribute__((always_inline)) float next(const F16& s, bool& changed) {
    float top = 0.0f;
#pragma unroll
    for (int r = 0; r < 16; ++r) top = fmaxf(top, __builtin_fabsf(s[r]));
    changed = __any(top > most);
    if (__builtin_expect(!changed, 1)) return 1.0f;
    top = fmaxf(top, other_half(top));  // (a column is two lanes)
    if (!(top > most && top < kInf32)) return 1.0f;
    most = 0x1p15f;
    const int e = 10 - __builtin_amdgcn_frexp_expf(top), by = e < 60 ? e : 60;
    up = ldexpf(up, by), down = ldexpf(down, -by);
    return ldexpf(1.0f, by);
  }
};
// That of probabilities that multiply gradients, which are 1 at most: log2.
template <class T>
constexpr float kProbabilityUp = std::is_same_v<T, f16> ? 12.0f : 0.0f;

template <class T, int kDim, bool kDirect>
__global__ __launch_bounds__(kWaves* kWave, (waves_per_simd<T, kDim>())) void
attention_grad_q_kernel(AttentionArgs args) {
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
  typename L::Frag qf[L::kChunks], gf[L::kChunks];
  load_row<T, kDim, kDirect>(qf, static_cast<const T*>(a.q) + q.q_at + x.query * a.q_row_stride +
                                     x.head * a.q_head_stride, a.dim);
  const int64_t out_row = (q.q_first + x.query) * a.q_heads + x.head;
  load_row<T, kDim, kDirect>(gf, static_cast<const T*>(args.grad_out) + out_row * a.dim, a.dim);
  float delta = 0.0f;
  {
    typename L::Frag of[L::kChunks];
    load_row<T, kDim, kDirect>(of, static_cast<const T*>(args.out_in) + out_row * a.dim, a.dim);
#pragma unroll
    for (int c = 0; c < L::kChunks; ++c)
#pragma unroll
      for (int i = 0; i < L::kChunk / 2; ++i) delta = fmaf((float)gf[c][i], (float)of[c][i], delta);
  }
  delta += other_half(delta);
  const float lse = args.lse_in[out_row];
  const float base = lse == -kInf32 ? 0.0f : lse * kLog2E;

  F16 dq[kDim / 32] = {};
  uint32_t found = 0;
  // sums of ds and p: scale times what out's rounding took from delta, where the probabilities are a
  // whole row's
  float rest = 0.0f, mass = 0.0f;
  Lift<T> lift{1.0f, 1.0f};
  float scale = a.scale;  // times lift.up, as are all slopes
  const auto lost = [&] {
    const float r = rest + other_half(rest), m = mass + other_half(mass);
    return __builtin_fabsf(m - 1.0f) <= kWhole ? r / scale : 0.0f;
  };
  typename L::Lane own;
  // the two products of 32 keys, and ds in place of s
  const auto slopes = [&](int k0, int b, F16& s, const F16& dp, float shift, bool cuts)
      __attribute__((always_inline)) {
    if (cuts) {
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (k0 + 32 * b + result_row(r) >= x.limit) s[r] = -kInf32;
    }
    float here_mass = 0.0f;  // (each step of a long sum would round at its size)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const float p = __builtin_amdgcn_exp2f(fmaf(s[r], args.score_scale, -base));
      here_mass += p;
      s[r] = p * fmaf(dp[r], scale, -shift);
      // (or all of p would wait in registers for its sum)
      if (r % 4 == 3) asm volatile("" : "+v"(here_mass));
    }
    mass += here_mass;
    if (cuts) {
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (k0 + 32 * b + result_row(r) >= x.limit) s[r] = 0.0f;
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) rest += s[r];
  };
  const bool twice = sizeof(T) == 2 && x.block_most <= 2 * kTileKeys;
  if (twice) {
    if (x.block_most > kTileKeys) load(kTileKeys, keys1, values1);
    tiles_ready();
#pragma unroll 1
    for (int i = 0; i < 4 && 32 * i < x.most; ++i) {
      F16 s, dp;
      const char *keys = i < 2 ? keys0 : keys1, *values = i < 2 ? values0 : values1;
      two_products<T, kDim>(s, keys, 32 * (i % 2), qf, dp, values, 32 * (i % 2), gf, own);
      slopes(0, i, s, dp, delta * scale, 32 * i + 32 > x.least);
    }
    delta += lost();
    rest = mass = 0.0f;
  }
  float shift = delta * scale;
  const auto step = [&](int k0, const char* keys, const char* values, char* next_keys,
                        char* next_values) __attribute__((always_inline)) {
    tiles_ready();
    own.renew();
    if (k0 + kTileKeys < x.block_most && !twice) load(k0 + kTileKeys, next_keys, next_values);
    if (k0 >= x.most) return;
    const bool cuts = k0 + kTileKeys > x.least;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      F16 s, dp;
      two_products<T, kDim>(s, keys, 32 * b, qf, dp, values, 32 * b, gf, own);
      Columns<T, kDim> columns;
      columns.read(keys, 32 * b, 0, own);
      here();
      slopes(k0, b, s, dp, shift, cuts);
      if constexpr (lift.kOn) {
        bool changed;
        const float by = lift.next(s, changed);
        if (changed) {
          s *= by, scale *= by, shift *= by, rest *= by;
#pragma unroll
          for (int d = 0; d < kDim / 32; ++d) dq[d] *= by;
        }
      }
      add_columns<T, kDim, true>(dq, columns, keys, 32 * b, s, cuts, found, own);
    }
  };
  // (two steps a turn: as in the forward kernel)
  for (int k0 = 0; k0 < x.block_most; k0 += 2 * kTileKeys) {
    step(k0, keys0, values0, keys1, values1);
    if (k0 + kTileKeys < x.block_most) step(k0 + kTileKeys, keys1, values1, keys0, values0);
  }
  delta += lost();
  const bool hidden = __any(found != 0) && lane < 32;  // (a lane finds for other lanes' rows)
  if (!x.there) return;
  if (lane < 32) args.delta[out_row] = delta;
  T* grad = static_cast<T*>(args.grad_q) + out_row * a.dim;
  store_column<T, kDim, kDirect>(grad, dq, lift.down, a.dim);
  if (__builtin_expect(hidden, 0))
    add_hidden<T, true>(grad, a.dim, x.least / kTileKeys * kTileKeys, x.limit,
                        [=](int j) { return k_rows + j * a.k_row_stride; });
}

// What a row of queries brings to the gradients by keys: the base of its probabilities, its delta
// times scale, and the keys that it sees.
struct RowStats {
  float base[kTileKeys], delta[kTileKeys];
  int limit[kTileKeys];
};

// A workgroup has 128 keys, a wave 32 of them; 64 rows of queries at a time pass through LDS.
// kKeys, kValues: the sums that it forms.
template <class T, int kDim, bool kDirect, bool kKeys, bool kValues>
__device__ __attribute__((always_inline)) inline void grad_kv(const AttentionArgs& args,
                                                              int64_t block, char* queries0,
                                                              char* queries1, char* grads0,
                                                              char* grads1, RowStats& stats0,
                                                              RowStats& stats1) {
  using L = Tile<T, kDim>;
  const omq_attention_args& a = args.a;
  Place at;
  if (!place_of_keys(args, kTileRows, block, &at)) return;
  const Sequence& q = at.q;
  const int j0 = (int)(at.tile * kTileRows), group = args.group, kv = at.kv;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int from = j0 + kWaveRows * wave, mine = from + (lane & 31);
  const bool there = mine < q.room;
  const int key = there ? mine : q.room - 1;
  const int shift = q.lk - q.lq;
  const int rows = (int)((int64_t)q.lq * group);
  // the rows that see a key of the workgroup: from `first` (on a tile's boundary) to `end`
  int64_t first = 0;
  if (a.causal && j0 > shift)
    first = (int64_t)(j0 - shift) * group / kTileKeys * kTileKeys;
  const int end = j0 < q.lk ? rows : 0;

  const T* q_rows = static_cast<const T*>(a.q) + q.q_at + kv * group * a.q_head_stride;
  const int64_t out_first = q.q_first * a.q_heads + kv * group;
  const T* g_rows = static_cast<const T*>(args.grad_out) + out_first * a.dim;
  // row r's place in q, and in arrays of rows of heads
  const auto q_place = [&](int r) {
    const int query = query_of(args, r);
    return query * a.q_row_stride + (r - query * group) * a.q_head_stride;
  };
  const auto out_place = [&](int r) {
    const int query = query_of(args, r);
    return (int64_t)query * a.q_heads + (r - query * group);
  };
  const EvenRows<T, kDim> q_own(a.dim, q_place);
  const EvenRows<T, kDim> g_own(a.dim, [&](int r) { return out_place(r) * a.dim; });
  const auto load = [&](int r0, char* queries, char* grads) {
    if (kDirect && args.even && rows - r0 >= kTileKeys) {
      const int queries_a_step = EvenRows<T, kDim>::kRowsAStep / group, query = query_of(args, r0);
      q_own.load(queries, q_rows + query * a.q_row_stride, queries_a_step * a.q_row_stride);
      const int64_t heads = (int64_t)a.q_heads * a.dim;
      g_own.load(grads, g_rows + query * heads, queries_a_step * heads);
      return;
    }
    load_tile<T, kDim, kDirect>(queries, rows - r0, a.dim,
                                [&](int i) { return q_rows + q_place(r0 + i); });
    load_tile<T, kDim, kDirect>(grads, rows - r0, a.dim,
                                [&](int i) { return g_rows + out_place(r0 + i) * a.dim; });
  };
  // the first wave brings what belongs to a tile's rows
  float lse = 0.0f, delta = 0.0f;
  const auto fetch = [&](int r0) {
    if (threadIdx.x < kTileKeys) {
      const int64_t i = out_first + out_place(r0 + lane < rows ? r0 + lane : rows - 1);
      lse = args.lse_in[i], delta = args.delta[i];
    }
  };
  const auto put = [&](int r0, RowStats& stats) {
    if (threadIdx.x < kTileKeys) {
      const int r = r0 + lane;
      stats.base[lane] = (lse == -kInf32 ? 0.0f : lse * kLog2E) - kProbabilityUp<T>;
      stats.delta[lane] = delta * a.scale;
      stats.limit[lane] = r >= rows ? 0
                          : a.causal ? cut(query_of(args, r) + shift + 1, 0, q.lk)
                                     : q.lk;
    }
  };
  if (kDirect && a.dim < kDim) {
    clear_tile<T, kDim>(queries0, a.dim), clear_tile<T, kDim>(queries1, a.dim);
    clear_tile<T, kDim>(grads0, a.dim), clear_tile<T, kDim>(grads1, a.dim);
    __syncthreads();
  }
  if (first < end) {
    load((int)first, queries0, grads0);
    fetch((int)first);
    put((int)first, stats0);
  }
  typename L::Frag kf[L::kChunks], vf[kKeys ? L::kChunks : 1];
  load_row<T, kDim, kDirect>(kf, static_cast<const T*>(a.k) + q.k_at + key * a.k_row_stride +
                                     kv * a.k_head_stride, a.dim);
  if constexpr (kKeys)
    load_row<T, kDim, kDirect>(vf, static_cast<const T*>(a.v) + q.v_at + key * a.v_row_stride +
                                       kv * a.v_head_stride, a.dim);
  F16 dk[kDim / 32] = {}, dv[kDim / 32] = {};
  constexpr float kUp = Lift<T>::kOn ? 0x1p12f : 1.0f;  // 2^kProbabilityUp, of p here
  Lift<T> lift{1.0f / kUp, 1.0f};
  uint32_t found_q = 0, found_g = 0;
  typename L::Lane own;
  const auto step = [&](int64_t next, const char* queries, const char* grads,
                        const RowStats& stats, char* next_queries, char* next_grads,
                        RowStats& next_stats) __attribute__((always_inline)) {
    const int r0 = (int)next;
    const bool more = next + kTileKeys < end;
    tiles_ready();
    own.renew();
    if (more) load(r0 + kTileKeys, next_queries, next_grads), fetch(r0 + kTileKeys);
    // some row does not see all of the wave's keys; or none does
    const int low = a.causal ? query_of(args, r0) + shift + 1 : q.lk;
    const int high = a.causal ? query_of(args, r0 + kTileKeys - 1) + shift + 1 : q.lk;
    const bool cuts = r0 + kTileKeys > rows || from + kWaveRows > q.lk || from + kWaveRows > low;
    if (from < high && from < q.lk) {
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        F16 s, dp;
        if constexpr (kKeys)
          two_products<T, kDim>(s, queries, 32 * b, kf, dp, grads, 32 * b, vf, own);
        else
          one_product<T, kDim>(s, queries, 32 * b, kf, own);
        Columns<T, kDim> columns;
        columns.read(kValues ? grads : queries, 32 * b, 0, own);
        here();
        F16 p;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int i = 32 * b + result_row(r);
          p[r] = __builtin_amdgcn_exp2f(fmaf(s[r], args.score_scale, -stats.base[i]));
          if constexpr (kKeys) {
            s[r] = p[r] * fmaf(dp[r], a.scale, -stats.delta[i]);
            if constexpr (lift.kOn) s[r] *= lift.up;
          }
        }
        if (cuts) {
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const bool sees = mine < stats.limit[32 * b + result_row(r)];
            p[r] = sees ? p[r] : 0.0f;
            s[r] = sees ? s[r] : 0.0f;
          }
        }
        if constexpr (kValues)
          add_columns<T, kDim, false>(dv, columns, grads, 32 * b, p, cuts, found_g, own);
        if constexpr (kKeys) {
          if constexpr (kValues) columns.read(queries, 32 * b, 0, own);
          if constexpr (lift.kOn) {
            bool changed;
            const float by = lift.next(s, changed);
            if (changed) {
              s *= by;
#pragma unroll
              for (int d = 0; d < kDim / 32; ++d) dk[d] *= by;
            }
          }
          add_columns<T, kDim, false>(dk, columns, queries, 32 * b, s, cuts, found_q, own);
        }
      }
    }
    if (more) put(r0 + kTileKeys, next_stats);
  };
  for (int64_t r0 = first; r0 < end; r0 += 2 * kTileKeys) {  // (as in the forward kernel)
    step(r0, queries0, grads0, stats0, queries1, grads1, stats1);
    if (r0 + kTileKeys < end)
      step(r0 + kTileKeys, queries1, grads1, stats1, queries0, grads0, stats0);
  }
  const bool hidden = __any((found_q | found_g) != 0) && lane < 32;  // (as above)
  if (!there) return;
  if (mine >= q.lk) {  // (whatever the queries hold)
#pragma unroll
    for (int d = 0; d < kDim / 32; ++d) dk[d] = F16{}, dv[d] = F16{};
  }
  const int64_t out = ((q.k_first + key) * a.k_heads + kv) * a.dim;
  T *grad_k = static_cast<T*>(args.grad_k) + out, *grad_v = static_cast<T*>(args.grad_v) + out;
  if constexpr (kKeys) store_column<T, kDim, kDirect>(grad_k, dk, lift.down, a.dim);
  if constexpr (kValues) store_column<T, kDim, kDirect>(grad_v, dv, 1.0f / kUp, a.dim);
  if (__builtin_expect(hidden, 0) && mine < q.lk) {
    const int64_t least = a.causal && mine > shift ? (int64_t)(mine - shift) * group : 0;
    const int sees = least < rows ? (int)least : rows;  // the first row that sees this key
    if constexpr (kKeys)
      add_hidden<T, true>(grad_k, a.dim, sees, rows, [=](int r) { return q_rows + q_place(r); });
    if constexpr (kValues)
      add_hidden<T, false>(grad_v, a.dim, sees, rows,
                           [=](int r) { return g_rows + out_place(r) * a.dim; });
  }
}

constexpr int kComputeUnits = 256;

// Sums of 128 columns are a workgroup's each, of the keys or of the values (scores are formed in
// both: five products in place of four): with both a wave has no room for a second one on its SIMD,
// whose products run while the first forms its probabilities.  (All three gradients of 8 x 8 heads
// of 1024 keys, bf16: 182 us, 268 together; of 64 columns 118 apart, 91 together.)  In float32 a
// wave is alone on its SIMD in either case, and they are apart only where the workgroups are fewer
// than the compute units: 8 x 8 heads 1460 us, 1116 together; 8 x 2 key heads 1402 and 1683.
template <class T, int kDim>
bool sums_apart(int64_t blocks) {
  return kDim > 64 && (sizeof(T) == 2 || blocks < kComputeUnits);
}

template <class T, int kDim, bool kDirect, bool kApart>
__global__ __launch_bounds__(kWaves* kWave, (waves_per_simd<T, kDim>())) void
attention_grad_kv_kernel(AttentionArgs args) {
  using L = Tile<T, kDim>;
  __shared__ __attribute__((aligned(1024))) char queries0[L::kBytes], queries1[L::kBytes];
  __shared__ __attribute__((aligned(1024))) char grads0[L::kBytes], grads1[L::kBytes];
  __shared__ __attribute__((aligned(16))) RowStats stats0, stats1;
  const int64_t block = block_index();
  if constexpr (!kApart)
    grad_kv<T, kDim, kDirect, true, true>(args, block, queries0, queries1, grads0, grads1, stats0,
                                          stats1);
  else if (block % 2 == 0)
    grad_kv<T, kDim, kDirect, true, false>(args, block / 2, queries0, queries1, grads0, grads1,
                                           stats0, stats1);
  else
    grad_kv<T, kDim, kDirect, false, true>(args, block / 2, queries0, queries1, grads0, grads1,
                                           stats0, stats1);
}

int64_t delta_bytes(const omq_attention_args& a) {
  const int64_t n = a.q_starts ? 1 : a.sequences;
  return n * a.q_len * a.q_heads * (int64_t)sizeof(float);
}

}  // namespace
}  // namespace omq_net

using namespace omq_net;

extern "C" {

int64_t omq_attention_grad_workspace(const omq_attention_args* a) {
  const int rc = check_attention("omq_attention_grad_workspace", a);
  return rc ? rc : delta_bytes(*a);
}

int omq_attention_grad(const omq_attention_args* a, const void* grad_out, const void* out,
                       const float* lse, void* grad_q, void* grad_k, void* grad_v,
                       void* workspace, int64_t workspace_bytes, void* stream) {
  const char* name = "omq_attention_grad";
  if (int rc = check_attention(name, a)) return rc;
  const int64_t n = a->q_starts ? 1 : a->sequences;
  const bool queries = n > 0 && a->q_len > 0, keys = n > 0 && a->k_len > 0;
  if ((queries && (!grad_out || !out || !lse || !grad_q)) || (keys && (!grad_k || !grad_v)))
    return net_fail(OMQ_NET_E_ARG, "%s: a null array", name);
  const int64_t need = delta_bytes(*a);
  if (need > 0 && (!workspace || workspace_bytes < need || !on_16_bytes(workspace)))
    return net_fail(OMQ_NET_E_ARG, "%s: workspace of %lld bytes at %p, %lld on a 16-byte boundary "
                    "needed", name, (long long)workspace_bytes, workspace, (long long)need);
  AttentionArgs args = attention_layout(*a);
  args.grad_out = grad_out, args.out_in = out, args.lse_in = lse;
  args.delta = static_cast<float*>(workspace);
  args.grad_q = grad_q, args.grad_k = grad_k, args.grad_v = grad_v;
  hipStream_t st = (hipStream_t)stream;
  if (queries) {
    tiles_of(&args, a->q_len, args.group, kTileRows);
    const dim3 grid = grid_of(args.slots * a->k_heads, kWaves * kWave);
    with_head(a->dtype, a->dim, direct_tiles(*a), [&](auto t, auto dim, auto direct) {
      args.even = even_keys<decltype(t), dim.value>(*a);
      attention_grad_q_kernel<decltype(t), dim.value, direct.value>
          <<<grid, kWaves * kWave, 0, st>>>(args);
    });
  }
  if (keys) {
    tiles_of(&args, a->k_len, 1, kTileRows);
    const bool rows_direct = chunks_aligned(a->dtype, a->dim, {a->q, grad_out},
                                            {a->q_seq_stride, a->q_row_stride, a->q_head_stride});
    with_head(a->dtype, a->dim, rows_direct, [&](auto t, auto dim, auto direct) {
      // (rows of a group lie as far apart at every step that has whole groups)
      using Even = EvenRows<decltype(t), dim.value>;
      const int64_t far = a->q_row_stride < (1ll << 31) && a->q_head_stride < (1ll << 31)
                              ? (kTileKeys + 1) * a->q_row_stride + args.group * a->q_head_stride
                              : 1ll << 31;
      const int64_t far_out = (kTileKeys + 1) * (int64_t)a->q_heads * a->dim;
      args.even = Even::kRowsAStep % args.group == 0 &&
                  Even::possible(a->dim, far > far_out ? far : far_out);
      using T = decltype(t);
      int64_t blocks = args.slots * a->k_heads;
      const bool apart = sums_apart<T, dim.value>(blocks);
      blocks *= apart ? 2 : 1;
      // (all gradients of causal sequences of 4096, bf16: two with 16 heads over 4 of 128 784 us, in
      // one order 829; one with 16 over 8 of 128 428 and 450; neighbours paired 817 and 444)
      args.paired = a->causal && blocks > kComputeUnits && blocks <= 2 * kComputeUnits;
      const dim3 grid = grid_of(blocks, kWaves * kWave);
      const auto go = [&](auto split) {
        attention_grad_kv_kernel<T, dim.value, direct.value, split.value>
            <<<grid, kWaves * kWave, 0, st>>>(args);
      };
      if constexpr (dim.value <= 64) {
        go(std::false_type{});
      } else if constexpr (sizeof(T) == 2) {
        go(std::true_type{});
      } else if (apart) {
        go(std::true_type{});
      } else {
        go(std::false_type{});
      }
    });
  }
  return net_status(name);
}

}  // extern "C"
