// Gradients of the attention (gfx950).  With the forward pass's p_ij = e^(s_ij - lse_i) formed
// again from its lse, and g the gradient of out:
//   delta_i = g_i . out_i;   ds_ij = p_ij (g_i . v_j - delta_i) scale
//   dq_i = sum_j ds_ij k_j;  dk_j = sum_i ds_ij q_i;  dv_j = sum_i p_ij g_i
// Two launches, each with its sums in registers: by queries (dq, and delta for the other) and by
// keys (dk and dv).  Scores are formed in both, seven products in place of five, and no sum is
// split over workgroups, which would take atomics or float32 copies of dq; every result is the
// same bits at every call.  Rows of queries that share a key head are rows of one sum.
// ds is rounded to the elements' type for its products, times scale, without which float16 would
// overflow earlier.
#include "net_attention.h"

namespace omq_net {
namespace {

template <class T, int kDim>
__global__ __launch_bounds__(kWaves* kWave) void attention_grad_q_kernel(AttentionArgs args) {
  using L = Tile<T, kDim>;
  __shared__ __attribute__((aligned(16))) char keys[L::kBytes];
  __shared__ __attribute__((aligned(16))) char values[L::kBytes];
  __shared__ int bad[2];
  const omq_attention_args& a = args.a;
  const int64_t block = block_index();
  const int64_t slot = block / a.k_heads;
  if (slot >= args.slots) return;
  const int kv = (int)(block % a.k_heads), group = args.group;
  int64_t tile;
  Sequence q;
  if (a.q_starts) {
    q = sequence_of(args, find_piece(a.q_starts, a.sequences, a.q_len, group, kTileRows, slot,
                                     &tile));
  } else {
    q = sequence_of(args, slot / args.batch_tiles);
    tile = slot % args.batch_tiles;
  }
  const int64_t rows = (int64_t)q.lq * group, r0 = tile * kTileRows;
  if (tile < 0 || r0 >= rows) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (threadIdx.x < 2) bad[threadIdx.x] = 0;
  const int64_t mine = r0 + kWaveRows * wave + (lane & 31);
  const bool there = mine < rows;
  const int64_t row = there ? mine : rows - 1;
  const int query = (int)(row / group), head = kv * group + (int)(row % group);
  const int shift = q.lk - q.lq;
  const int limit = a.causal ? cut(query + shift + 1, 0, q.lk) : q.lk;
  const int64_t last_row = r0 + kTileRows < rows ? r0 + kTileRows - 1 : rows - 1;
  const int most = a.causal ? cut((int)(last_row / group) + shift + 1, 0, q.lk) : q.lk;
  const int least = a.causal ? cut((int)(r0 / group) + shift + 1, 0, q.lk) : q.lk;

  typename L::Frag qf[L::kChunks], gf[L::kChunks];
  load_row<T, kDim>(qf, static_cast<const T*>(a.q) + q.q_at + query * a.q_row_stride +
                            head * a.q_head_stride, a.dim);
  const int64_t out_row = (q.q_first + query) * a.q_heads + head;
  load_row<T, kDim>(gf, static_cast<const T*>(args.grad_out) + out_row * a.dim, a.dim);
  float delta = 0.0f;
  {
    typename L::Frag of[L::kChunks];
    load_row<T, kDim>(of, static_cast<const T*>(args.out_in) + out_row * a.dim, a.dim);
#pragma unroll
    for (int c = 0; c < L::kChunks; ++c)
#pragma unroll
      for (int i = 0; i < L::kChunk / 2; ++i) delta = fmaf((float)gf[c][i], (float)of[c][i], delta);
  }
  delta += other_half(delta);
  if (there && lane < 32) args.delta[out_row] = delta;
  const float lse = args.lse_in[out_row];
  const float base = lse == -kInf32 ? 0.0f : lse * kLog2E;

  const T* k_rows = static_cast<const T*>(a.k) + q.k_at + kv * a.k_head_stride;
  const T* v_rows = static_cast<const T*>(a.v) + q.v_at + kv * a.v_head_stride;
  F16 dq[kDim / 32] = {};
  for (int k0 = 0, turn = 0; k0 < most; k0 += kTileKeys, turn ^= 1) {
    const int left = q.lk - k0;
    __syncthreads();
    if (threadIdx.x == 0) bad[turn ^ 1] = 0;
    const bool found = load_tile<T, kDim>(
        keys, left, a.dim, [&](int i) { return k_rows + (int64_t)(k0 + i) * a.k_row_stride; });
    load_tile<T, kDim>(values, left, a.dim,
                       [&](int i) { return v_rows + (int64_t)(k0 + i) * a.v_row_stride; });
    if (found) bad[turn] = 1;
    __syncthreads();
    const bool cuts = k0 + kTileKeys > least, careful = cuts && bad[turn];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      F16 s = {}, dp = {};
#pragma unroll
      for (int c = 0; c < L::kChunks; ++c) s = mma(L::row(keys, 32 * b, c), qf[c], s);
#pragma unroll
      for (int c = 0; c < L::kChunks; ++c) dp = mma(L::row(values, 32 * b, c), gf[c], dp);
      F16 seen = {};
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float p = __builtin_amdgcn_exp2f(fmaf(s[r], args.score_scale, -base));
        s[r] = p * (dp[r] - delta) * a.scale;
        if (cuts) {
          const bool sees = k0 + 32 * b + result_row(r) < limit;
          s[r] = sees ? s[r] : 0.0f;
          seen[r] = sees ? 1.0f : 0.0f;
        }
      }
      add_columns<T, kDim>(dq, keys, 32 * b, s, seen, careful);
    }
  }
  if (there)
    store_column<T, kDim>(static_cast<T*>(args.grad_q) + out_row * a.dim, dq, 1.0f, a.dim);
}

// A workgroup has 128 keys, a wave 32 of them; 64 rows of queries at a time pass through LDS.
template <class T, int kDim>
__global__ __launch_bounds__(kWaves* kWave) void attention_grad_kv_kernel(AttentionArgs args) {
  using L = Tile<T, kDim>;
  __shared__ __attribute__((aligned(16))) char queries[L::kBytes];
  __shared__ __attribute__((aligned(16))) char grads[L::kBytes];
  __shared__ __attribute__((aligned(16))) float bases[kTileKeys], deltas[kTileKeys];
  __shared__ __attribute__((aligned(16))) int limits[kTileKeys];
  __shared__ int bad[2];
  const omq_attention_args& a = args.a;
  const int64_t block = block_index();
  const int64_t slot = block / a.k_heads;
  if (slot >= args.slots) return;
  const int kv = (int)(block % a.k_heads), group = args.group;
  int64_t tile;
  Sequence q;
  if (a.q_starts) {
    q = sequence_of(args, find_piece(a.k_starts, a.sequences, a.k_len, 1, kTileRows, slot, &tile));
  } else {
    q = sequence_of(args, slot / args.batch_tiles);
    tile = slot % args.batch_tiles;
  }
  const int64_t j0 = tile * kTileRows;
  if (tile < 0 || j0 >= q.room) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (threadIdx.x < 2) bad[threadIdx.x] = 0;
  const int mine = (int)j0 + kWaveRows * wave + (lane & 31);
  const bool there = mine < q.room, used = mine < q.lk;
  const int key = there ? mine : q.room - 1;
  const int shift = q.lk - q.lq;
  const int64_t rows = (int64_t)q.lq * group;

  typename L::Frag kf[L::kChunks], vf[L::kChunks];
  load_row<T, kDim>(kf, static_cast<const T*>(a.k) + q.k_at + key * a.k_row_stride +
                            kv * a.k_head_stride, a.dim);
  load_row<T, kDim>(vf, static_cast<const T*>(a.v) + q.v_at + key * a.v_row_stride +
                            kv * a.v_head_stride, a.dim);
  F16 dk[kDim / 32] = {}, dv[kDim / 32] = {};
  // the first row that sees a key of this tile; the last key of it that is in use
  int64_t first = 0;
  if (a.causal && j0 > shift) first = (j0 - shift) * group / kTileKeys * kTileKeys;
  const int last_key = (int)(j0 + kTileRows < q.lk ? j0 + kTileRows : q.lk) - 1;
  const int64_t end = j0 < q.lk ? rows : 0;
  int turn = 0;
  for (int64_t r0 = first; r0 < end; r0 += kTileKeys, turn ^= 1) {
    const int left = rows - r0 < kTileKeys ? (int)(rows - r0) : kTileKeys;
    const auto query_of = [&](int i) { return (int)((r0 + i) / group); };
    const auto head_of = [&](int i) { return kv * group + (int)((r0 + i) % group); };
    __syncthreads();
    if (threadIdx.x == 0) bad[turn ^ 1] = 0;
    bool found = load_tile<T, kDim>(queries, left, a.dim, [&](int i) {
      return static_cast<const T*>(a.q) + q.q_at + query_of(i) * a.q_row_stride +
             head_of(i) * a.q_head_stride;
    });
    found |= load_tile<T, kDim>(grads, left, a.dim, [&](int i) {
      return static_cast<const T*>(args.grad_out) +
             ((q.q_first + query_of(i)) * a.q_heads + head_of(i)) * a.dim;
    });
    if (found) bad[turn] = 1;
    if (threadIdx.x < kTileKeys) {
      const int i = threadIdx.x < left ? threadIdx.x : left - 1;
      const int64_t at = (q.q_first + query_of(i)) * a.q_heads + head_of(i);
      const float lse = args.lse_in[at];
      bases[threadIdx.x] = lse == -kInf32 ? 0.0f : lse * kLog2E;
      deltas[threadIdx.x] = args.delta[at];
      limits[threadIdx.x] = (int)threadIdx.x >= left ? 0
                            : a.causal ? cut(query_of(i) + shift + 1, 0, q.lk) : q.lk;
    }
    __syncthreads();
    const bool cuts = left < kTileKeys || j0 + kTileRows > q.lk ||
                      (a.causal && last_key >= query_of(0) + shift + 1);
    const bool careful = cuts && bad[turn];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      F16 s = {}, dp = {};
#pragma unroll
      for (int c = 0; c < L::kChunks; ++c) s = mma(L::row(queries, 32 * b, c), kf[c], s);
#pragma unroll
      for (int c = 0; c < L::kChunks; ++c) dp = mma(L::row(grads, 32 * b, c), vf[c], dp);
      F16 p, seen = {};
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int i = 32 * b + result_row(r);
        p[r] = __builtin_amdgcn_exp2f(fmaf(s[r], args.score_scale, -bases[i]));
        s[r] = p[r] * (dp[r] - deltas[i]) * a.scale;
        if (cuts) {
          const bool sees = mine < limits[i];
          p[r] = sees ? p[r] : 0.0f;
          s[r] = sees ? s[r] : 0.0f;
          seen[r] = sees ? 1.0f : 0.0f;
        }
      }
      add_columns<T, kDim>(dv, grads, 32 * b, p, seen, careful);
      add_columns<T, kDim>(dk, queries, 32 * b, s, seen, careful);
    }
  }
  if (!there) return;
  if (!used) {  // (whatever the queries hold)
#pragma unroll
    for (int d = 0; d < kDim / 32; ++d) dk[d] = F16{}, dv[d] = F16{};
  }
  const int64_t at = ((q.k_first + key) * a.k_heads + kv) * a.dim;
  store_column<T, kDim>(static_cast<T*>(args.grad_k) + at, dk, 1.0f, a.dim);
  store_column<T, kDim>(static_cast<T*>(args.grad_v) + at, dv, 1.0f, a.dim);
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
    with_head(a->dtype, a->dim, [&](auto t, auto dim) {
      attention_grad_q_kernel<decltype(t), dim.value><<<grid, kWaves * kWave, 0, st>>>(args);
    });
  }
  if (keys) {
    tiles_of(&args, a->k_len, 1, kTileRows);
    const dim3 grid = grid_of(args.slots * a->k_heads, kWaves * kWave);
    with_head(a->dtype, a->dim, [&](auto t, auto dim) {
      attention_grad_kv_kernel<decltype(t), dim.value><<<grid, kWaves * kWave, 0, st>>>(args);
    });
  }
  return net_status(name);
}

}  // extern "C"
