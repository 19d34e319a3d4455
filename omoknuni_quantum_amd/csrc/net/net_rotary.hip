// The norm of each head of queries and keys with the rotation by the token's positions, and its
// gradients (gfx950).
//
//   n = x r w,  r = 1 / sqrt(mean(x^2) + eps);   out = R(t) n,  t_j = position[axis of j] f_j
//   gradient: d = R(-t) g,  dx = r (d w - x r^2 mean(d w x)),  dw = sum over tokens and heads d x r
//
// Bound by memory: each element is read and written once.  A lane has eight pairs of columns (two
// blocks of eight elements, which lie a half of the rotated columns apart, or side by side where
// pairs are), or sixteen columns that do not rotate, and 1 to 32 lanes share a head, so that the
// rotation needs no exchange between lanes.  A workgroup takes all heads of queries or of keys of
// some tokens: it forms the sines and cosines of the tokens' pairs once, in LDS, for all of them (an
// angle costs about as many instructions as a lane's norm).  The next heads' loads are under way
// while one's are formed.  With inputs out of the caches 115200 tokens with 4 + 4 heads of 32,
// float32, take 62 us (3.8 TB/s; 56 where they repeat), the gradient of 16384 tokens with 32 + 8
// heads of 128, bf16, 106 us (4.8 TB/s): memory, and its latency where rows are short.
#include <type_traits>

#include "net_common.h"

namespace omq_net {
namespace {

constexpr int kThreads = 256;
constexpr int kGradGroups = 1024;  // of queries and of keys, at most
constexpr int kMostTiles = 256;    // that few tokens are cut into

// One of queries and keys: each has workgroups of its own, so that a thread has one weight and one
// of the weights' sums.
struct Side {
  const void *x, *weight;
  const void* g;       // gradient of the output
  void* out;           // the gradient: of x
  int64_t token_stride, head_stride;
  int heads;
  int tile;            // tokens of a workgroup
  uint32_t magic;      // 2^32 / heads, rounded up; 0 for one head
  int64_t tiles, groups;  // workgroups: of all tiles, or fewer that take turns
};

struct RotaryArgs {
  omq_rotary r;
  Side side[2];
  float* partial;                 // [workgroups, dim] sums of a weight's gradient, or NULL
  int turning, slots, lanes_log;  // lanes of a head that rotate, that work, and all (a power of 2)
  float inv_dim;
};

// A lane's two blocks: at column a and b of segments of a head.
struct Place {
  int seg_a, col_a, len_a, seg_b, col_b, len_b;
};

__device__ inline Place place_of(const RotaryArgs& a, int slot) {
  const int n = a.r.pairs, rest = a.r.dim - 2 * n, at = 16 * (slot - a.turning);
  if (slot >= a.turning) return {2 * n, at, rest, 2 * n, at + 8, rest};
  if (a.r.interleaved) return {0, 16 * slot, 2 * n, 0, 16 * slot + 8, 2 * n};
  return {0, 8 * slot, n, n, 8 * slot, n};
}

// Over the 2^lanes_log lanes of a head (uniform over the launch).
__device__ inline float head_sum(float v, int lanes_log) {
  if (lanes_log > 0) v += dpp<0xB1>(v);
  if (lanes_log > 1) v += dpp<0x4E>(v);
  if (lanes_log > 2) v += dpp<0x141>(v);
  if (lanes_log > 3) v += dpp<0x140>(v);
  if (lanes_log > 4) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                    false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  return v;
}

// The tile's cosines and sines: [token][pair], pairs up to whole blocks of eight.
__device__ inline void form_angles(const RotaryArgs& a, int64_t first, int tokens, float2* turn) {
  const int padded = 8 * ((a.r.pairs + 7) / 8);
  const int64_t first_row = a.r.pairs ? first % a.r.position_rows : 0;
  for (int i = threadIdx.x; i < tokens * padded; i += kThreads) {
    const int token = i / padded, pair = i - token * padded;
    float2 cs = make_float2(1.0f, 0.0f);
    if (pair < a.r.pairs) {
      int axis = 0;
#pragma unroll
      for (int s = 0; s < OMQ_NET_MAX_AXES - 1; ++s)
        axis += s < a.r.axes - 1 && pair >= a.r.section_end[s];
      int64_t row = first_row + token;
      if (row >= a.r.position_rows) row %= a.r.position_rows;
      const int64_t at = row * a.r.axes + axis;
      const double p = a.r.positions_are_64
                           ? (double)static_cast<const int64_t*>(a.r.positions)[at]
                           : (double)static_cast<const int32_t*>(a.r.positions)[at];
      const double turns = p * a.r.frequencies[pair] * 0.15915494309189535;  // 1 / (2 pi)
      sincospif((float)(2.0 * (turns - rint(turns))), &cs.y, &cs.x);
    }
    turn[i] = cs;
  }
}

// The pairs of a lane's two blocks turned by cs (back: the other way).
template <bool kBack>
__device__ inline void rotate(F8& x, F8& y, const float2* cs, bool interleaved) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float c = cs[j].x, s = kBack ? -cs[j].y : cs[j].y;
    if (interleaved) {
      F8& v = j < 4 ? x : y;
      const int at = 2 * (j & 3);
      const float u = v[at], w = v[at + 1];
      v[at] = u * c - w * s;
      v[at + 1] = w * c + u * s;
    } else {
      const float u = x[j], w = y[j];
      x[j] = u * c - w * s;
      y[j] = w * c + u * s;
    }
  }
}

template <class T, bool kWhole, bool kGrad>
__global__ __launch_bounds__(kThreads, (kWhole ? 4 : 3)) void rotary_kernel(RotaryArgs a) {
  extern __shared__ float4 shared[];
  float2* turn = reinterpret_cast<float2*>(shared);
  const int64_t block = block_index();
  const bool is_key = block >= a.side[0].groups;
  const Side& side = a.side[is_key];
  const int64_t group = is_key ? block - a.side[0].groups : block;
  if (group >= side.groups) return;
  const int lanes = 1 << a.lanes_log, heads = side.heads, dim = a.r.dim;
  const int own = threadIdx.x & (lanes - 1);
  const bool works = own < a.slots;
  const int slot = works ? own : 0;  // (lanes beyond a head load its first blocks, to no use)
  const Place at = place_of(a, slot);
  const int padded = 8 * ((a.r.pairs + 7) / 8);
  const bool turns = slot < a.turning, weighted = side.weight != nullptr;
  F8 w_u = {}, w_v = {};
  if (weighted) {
    const bool w_f32 = a.r.weight_dtype == OMQ_NET_F32;
    const int w_size = w_f32 ? 4 : (int)sizeof(T);
    const char* w = static_cast<const char*>(side.weight);
    w_u = widen<T, kWhole>(load_weight<T, kWhole>(w + at.seg_a * w_size, w_f32, at.col_a, at.len_a),
                           w_f32, at.col_a, at.len_a);
    w_v = widen<T, kWhole>(load_weight<T, kWhole>(w + at.seg_b * w_size, w_f32, at.col_b, at.len_b),
                           w_f32, at.col_b, at.len_b);
  }
  F8 dw_u = {}, dw_v = {};
  for (int64_t tile = group; tile < side.tiles; tile += side.groups) {
    const int64_t first = tile * side.tile, left = a.r.tokens - first;
    const int tokens = left < side.tile ? (int)left : side.tile;
    if (tile != group) __syncthreads();  // (the tile before has used its angles)
    const int step = kThreads >> a.lanes_log, rows = tokens * heads;
    const auto token_of = [&](int i) {
      return side.magic ? (int)__umulhi((uint32_t)i, side.magic) : i;
    };
    Reg8<T> next_a, next_b;
    const auto load = [&](int i) {
      const int t = token_of(i);
      const T* x = static_cast<const T*>(side.x) + (first + t) * side.token_stride +
                   (i - t * heads) * side.head_stride;
      next_a = load_raw<T, kWhole>(x + at.seg_a, at.col_a, at.len_a);
      next_b = load_raw<T, kWhole>(x + at.seg_b, at.col_b, at.len_b);
    };
    // (the first heads are under way while the angles are formed, and the next ones later)
    const int start = threadIdx.x >> a.lanes_log;
    if (!kGrad && start < rows) load(start);
    form_angles(a, first, tokens, turn);
    __syncthreads();
    for (int i = start; i < rows; i += step) {
      const int t = token_of(i), head = i - t * heads;
      const int64_t token = first + t;
      const int64_t flat = (token * heads + head) * dim;
      if (kGrad) load(i);
      const Reg8<T> raw_a = next_a, raw_b = next_b;
      if (!kGrad && i + step < rows) load(i + step);
      Reg8<T> g_a = {}, g_b = {};
      if constexpr (kGrad) {
        const T* g = static_cast<const T*>(side.g) + flat;
        g_a = load_raw<T, kWhole>(g + at.seg_a, at.col_a, at.len_a);
        g_b = load_raw<T, kWhole>(g + at.seg_b, at.col_b, at.len_b);
      }
      F8 u = widen<T, kWhole>(raw_a, at.col_a, at.len_a);
      F8 v = widen<T, kWhole>(raw_b, at.col_b, at.len_b);
      float r = 1.0f;
      if (weighted) {
        float sq = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) sq = fmaf(u[j], u[j], sq);
#pragma unroll
        for (int j = 0; j < 8; ++j) sq = fmaf(v[j], v[j], sq);
        sq = head_sum(works ? sq : 0.0f, a.lanes_log);
        r = 1.0f / sqrtf(fmaf(sq, a.inv_dim, a.r.eps));
      }
      float2 cs[8];
      if (turns) {
#pragma unroll
        for (int j = 0; j < 8; j += 2)
          *reinterpret_cast<float4*>(&cs[j]) =
              *reinterpret_cast<const float4*>(&turn[t * padded + 8 * slot + j]);
      }
      T* out = static_cast<T*>(side.out) + flat;
      if constexpr (!kGrad) {
        if (weighted) u = u * r * w_u, v = v * r * w_v;
        if (turns) rotate<false>(u, v, cs, a.r.interleaved);
        if (works) {
          store8<T, kWhole>(out + at.seg_a, at.col_a, at.len_a, u);
          store8<T, kWhole>(out + at.seg_b, at.col_b, at.len_b, v);
        }
      } else {
        F8 du = widen<T, kWhole>(g_a, at.col_a, at.len_a);
        F8 dv = widen<T, kWhole>(g_b, at.col_b, at.len_b);
        if (turns) rotate<true>(du, dv, cs, a.r.interleaved);
        if (weighted) {
          dw_u += du * u * r, dw_v += dv * v * r;
          du *= w_u, dv *= w_v;
          float dot = 0.0f;
#pragma unroll
          for (int j = 0; j < 8; ++j) dot = fmaf(du[j], u[j], dot);
#pragma unroll
          for (int j = 0; j < 8; ++j) dot = fmaf(dv[j], v[j], dot);
          dot = head_sum(works ? dot : 0.0f, a.lanes_log);
          const float k = dot * a.inv_dim * r * r;
          du = (du - u * k) * r, dv = (dv - v * k) * r;
        }
        if (works) {
          store8<T, kWhole>(out + at.seg_a, at.col_a, at.len_a, du);
          store8<T, kWhole>(out + at.seg_b, at.col_b, at.len_b, dv);
        }
      }
    }
  }
  if constexpr (kGrad) {
    if (!a.partial) return;
    // the lane groups' sums, in their order
    float* sum = reinterpret_cast<float*>(shared);
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      sum[j * kThreads + threadIdx.x] = dw_u[j];
      sum[(8 + j) * kThreads + threadIdx.x] = dw_v[j];
    }
    __syncthreads();
    if ((int)threadIdx.x < dim) {
      const int c = threadIdx.x, n = a.r.pairs;
      int lane, e;  // the column's lane and its place among its sixteen
      if (c >= 2 * n)
        lane = a.turning + (c - 2 * n) / 16, e = (c - 2 * n) % 16;
      else if (a.r.interleaved)
        lane = c / 16, e = c % 16;
      else
        lane = (c < n ? c : c - n) / 8, e = (c < n ? c : c - n) % 8 + (c < n ? 0 : 8);
      float s = 0.0f;
      for (int g = 0; g < kThreads >> a.lanes_log; ++g)
        s += sum[e * kThreads + (g << a.lanes_log) + lane];
      a.partial[block * dim + c] = s;
    }
  }
}

// The weights' gradients from the workgroups' sums (of queries, then of keys): 32 columns, 32 slices
// side by side, the slices added in order.
template <class O>
__global__ __launch_bounds__(1024) void join_weights_kernel(const float* __restrict__ partial,
                                                            int q_groups, int k_groups, int dim,
                                                            O* __restrict__ q, O* __restrict__ k) {
  __shared__ float part[32][33];
  const int blocks = (dim + 31) / 32;
  const bool is_key = (int)blockIdx.x >= blocks;
  const int groups = is_key ? k_groups : q_groups;
  if (is_key) partial += (int64_t)q_groups * dim;
  const int c = threadIdx.x % 32, slice = threadIdx.x / 32;
  const int col = ((int)blockIdx.x - (is_key ? blocks : 0)) * 32 + c;
  float s = 0.0f;
  if (col < dim)
    for (int g = slice; g < groups; g += 32 * 8) {  // eight loads in flight, the last ones too
      float v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u)
        v[u] = partial[(int64_t)(g + 32 * u < groups ? g + 32 * u : g) * dim + col];
#pragma unroll
      for (int u = 0; u < 8; ++u) s += g + 32 * u < groups ? v[u] : 0.0f;
    }
  part[slice][c] = s;
  __syncthreads();
  if (threadIdx.x < 32 && col < dim) {
    s = part[0][c];
    for (int i = 1; i < 32; ++i) s += part[i][c];
    (is_key ? k : q)[col] = (O)s;
  }
}

// ---- launches -------------------------------------------------------------------------------
template <class F>
void with_type(int dtype, F&& f) {
  if (dtype == OMQ_NET_F32) return f(float{});
  if (dtype == OMQ_NET_BF16) return f(bf16{});
  return f(f16{});
}

int check_rotary(const char* name, const omq_rotary* r) {
  if (!r) return net_fail(OMQ_NET_E_ARG, "%s: a null array", name);
  if (!dtype_known(r->dtype) || (r->q_weight && r->weight_dtype != r->dtype &&
                                 r->weight_dtype != OMQ_NET_F32))
    return net_fail(OMQ_NET_E_ARG, "%s: heads of type %d with weights of type %d", name, r->dtype,
                    r->weight_dtype);
  if (r->tokens < 0 || r->q_heads < 1 || r->k_heads < 1 || r->dim < 1 || r->pairs < 0 ||
      2 * (int64_t)r->pairs > r->dim || r->axes < 1)
    return net_fail(OMQ_NET_E_ARG, "%s: tokens %lld, heads %d and %d, dim %d, pairs %d, axes %d",
                    name, (long long)r->tokens, r->q_heads, r->k_heads, r->dim, r->pairs, r->axes);
  if (r->tokens > OMQ_NET_MAX_COUNT || r->dim > OMQ_NET_MAX_ROTARY_DIM ||
      r->axes > OMQ_NET_MAX_AXES || r->q_heads > 32768 || r->k_heads > 32768)
    return net_fail(OMQ_NET_E_LIMIT,
                    "%s: tokens %lld (at most %d), heads %d and %d (at most 32768), dim %d (at most "
                    "%d), axes %d (at most %d)",
                    name, (long long)r->tokens, OMQ_NET_MAX_COUNT, r->q_heads, r->k_heads, r->dim,
                    OMQ_NET_MAX_ROTARY_DIM, r->axes, OMQ_NET_MAX_AXES);
  int before = 0;
  for (int i = 0; i < r->axes; before = r->section_end[i++])
    if (r->section_end[i] < before || r->section_end[i] > r->pairs)
      return net_fail(OMQ_NET_E_ARG, "%s: sections that do not cut %d pairs", name, r->pairs);
  if (before != r->pairs)
    return net_fail(OMQ_NET_E_ARG, "%s: sections that do not cut %d pairs", name, r->pairs);
  if (!r->q_weight != !r->k_weight)
    return net_fail(OMQ_NET_E_ARG, "%s: both weights or neither", name);
  if (r->q_token_stride < 0 || r->q_head_stride < 0 || r->k_token_stride < 0 ||
      r->k_head_stride < 0)
    return net_fail(OMQ_NET_E_ARG, "%s: negative stride", name);
  if (r->tokens > 0 &&
      (!r->q || !r->k || (r->pairs && (!r->positions || !r->frequencies || r->position_rows < 1))))
    return net_fail(OMQ_NET_E_ARG, "%s: a null array", name);
  return OMQ_NET_OK;
}

// How the heads are cut, but for the outputs of a call.
RotaryArgs layout_of(const omq_rotary& r, bool grad) {
  RotaryArgs a{};
  a.r = r;
  a.turning = (r.pairs + 7) / 8;
  a.slots = a.turning + (r.dim - 2 * r.pairs + 15) / 16;
  while ((1 << a.lanes_log) < a.slots) ++a.lanes_log;
  a.inv_dim = 1.0f / (float)r.dim;
  a.side[0] = {r.q, r.q_weight, nullptr, nullptr, r.q_token_stride, r.q_head_stride, r.q_heads};
  a.side[1] = {r.k, r.k_weight, nullptr, nullptr, r.k_token_stride, r.k_head_stride, r.k_heads};
  for (Side& s : a.side) {
    // four rounds of a workgroup's threads or one token (16384 tokens, 32 + 8 heads of 128, bf16:
    // 67 us, one round 98, two 71, eight 66), and fewer where the tokens are few (1024 tokens, 8 + 8
    // heads of 64, gradient: 11 us in 256 tiles, 16 in 1024; 2048 tokens, 32 + 8 of 128: 17 and 21)
    int64_t tile = 4 * kThreads / ((int64_t)s.heads << a.lanes_log);
    tile = tile < r.tokens / kMostTiles ? tile : r.tokens / kMostTiles;
    s.tile = (int)(tile < 1 ? 1 : tile);
    s.tiles = ceil_div(r.tokens, s.tile);
    s.magic = s.heads > 1 ? (uint32_t)((0x100000000ull + s.heads - 1) / s.heads) : 0;
    // (of the gradient: enough for the chip, few enough for their sums: 16384 tokens as above 106 us,
    // of 512 groups 109, of 2048 111, of as many as tiles 117)
    s.groups = grad && r.q_weight && s.tiles > kGradGroups ? kGradGroups : s.tiles;
  }
  return a;
}

int64_t grad_groups(const RotaryArgs& a) { return a.side[0].groups + a.side[1].groups; }

template <bool kGrad>
void launch_rotary(const RotaryArgs& a, hipStream_t st) {
  const int n = a.r.pairs, rest = a.r.dim - 2 * n;
  const int tile = a.side[0].tile > a.side[1].tile ? a.side[0].tile : a.side[1].tile;
  size_t bytes = (size_t)tile * 8 * ((n + 7) / 8) * sizeof(float2);
  if (kGrad && a.partial && bytes < 16 * kThreads * sizeof(float))
    bytes = 16 * kThreads * sizeof(float);
  const dim3 grid = grid_of(grad_groups(a), kThreads);
  const bool whole = (a.r.interleaved ? 2 * n : n) % 8 == 0 && rest % 8 == 0;
  with_type(a.r.dtype, [&](auto t) {
    using T = decltype(t);
    const auto kernel = whole ? rotary_kernel<T, true, kGrad> : rotary_kernel<T, false, kGrad>;
    kernel<<<grid, kThreads, bytes, st>>>(a);
  });
}

}  // namespace
}  // namespace omq_net

using namespace omq_net;

extern "C" {

int omq_head_norm_rotary(const omq_rotary* r, void* q_out, void* k_out, void* stream) {
  const char* name = "omq_head_norm_rotary";
  if (int rc = check_rotary(name, r)) return rc;
  if (r->tokens == 0) return OMQ_NET_OK;
  if (!q_out || !k_out) return net_fail(OMQ_NET_E_ARG, "%s: a null array", name);
  RotaryArgs a = layout_of(*r, false);
  a.side[0].out = q_out, a.side[1].out = k_out;
  launch_rotary<false>(a, (hipStream_t)stream);
  return net_status(name);
}

int64_t omq_head_norm_rotary_grad_workspace(const omq_rotary* r) {
  const int rc = check_rotary("omq_head_norm_rotary_grad_workspace", r);
  if (rc) return rc;
  if (!r->q_weight) return 0;
  return grad_groups(layout_of(*r, true)) * r->dim * (int64_t)sizeof(float);
}

int omq_head_norm_rotary_grad(const omq_rotary* r, const void* grad_q_out, const void* grad_k_out,
                              void* grad_q, void* grad_k, void* grad_q_weight,
                              void* grad_k_weight, void* workspace, int64_t workspace_bytes,
                              void* stream) {
  const char* name = "omq_head_norm_rotary_grad";
  if (int rc = check_rotary(name, r)) return rc;
  const bool weighted = r->q_weight != nullptr;
  if (weighted && (!grad_q_weight || !grad_k_weight))
    return net_fail(OMQ_NET_E_ARG, "%s: a null array", name);
  if (r->tokens > 0 && (!grad_q_out || !grad_k_out || !grad_q || !grad_k))
    return net_fail(OMQ_NET_E_ARG, "%s: a null array", name);
  RotaryArgs a = layout_of(*r, true);
  const int64_t need = weighted ? grad_groups(a) * r->dim * (int64_t)sizeof(float) : 0;
  if (need > 0 && (!workspace || workspace_bytes < need || !on_16_bytes(workspace)))
    return net_fail(OMQ_NET_E_ARG, "%s: workspace of %lld bytes at %p, %lld on a 16-byte boundary "
                    "needed", name, (long long)workspace_bytes, workspace, (long long)need);
  a.side[0].g = grad_q_out, a.side[1].g = grad_k_out;
  a.side[0].out = grad_q, a.side[1].out = grad_k;
  a.partial = weighted ? static_cast<float*>(workspace) : nullptr;
  if (r->tokens > 0) launch_rotary<true>(a, (hipStream_t)stream);
  if (weighted)
    with_type(r->weight_dtype, [&](auto t) {
      using O = decltype(t);
      const uint32_t grid = 2 * (uint32_t)ceil_div(r->dim, 32);
      join_weights_kernel<O><<<grid, 1024, 0, (hipStream_t)stream>>>(
          static_cast<const float*>(workspace), (int)a.side[0].groups, (int)a.side[1].groups,
          r->dim, static_cast<O*>(grad_q_weight), static_cast<O*>(grad_k_weight));
    });
  return net_status(name);
}

}  // extern "C"
