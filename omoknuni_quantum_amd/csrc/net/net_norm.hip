// Root-mean-square norm of a residual sum, with dropout on the branch, an 8-bit output and the
// gradients (gfx950).
//
//   h = residual + dropout(x),  y = h * r * weight,  r = 1 / sqrt(mean(h^2) + eps)
//
// All three kernels move each element once and are bound by memory: a row's elements stay in
// registers between the reduction and their use.  A row belongs to as many threads as it has
// blocks of eight columns: 16 to 64 lanes of a wave (no barrier), then a workgroup of 128 to 1024.
// With one block a thread a workgroup is short-lived and small, and the chip stays full to the
// end: 11552 rows of 2048 bfloat16 to 8 bits take 32 us (5.2 TB/s, as a large copy) so, 39 us
// with a wave of four blocks a lane.  Measured besides: 115200 x 256 float16 with dropout 42 us
// (5.6 TB/s); one row of 4096 to 8 bits 2.4 us on the chip; the gradient of 16384 x 4096 bfloat16
// with dropout 128 us (5.2 TB/s), of which 5 us add the workgroups' sums for the weight.
#include <type_traits>

#include "net_common.h"

namespace omq_net {
namespace {

struct NormArgs {
  const void *x, *residual, *weight;
  int64_t x_stride, residual_stride;
  int64_t rows;
  int dim;
  int w_f32;
  float eps, inv_dim;
  void *y, *h;
  uint8_t* q;
  float* scales;
  Dropout drop;
};

enum Mode { kPlain, kDrop, kFp8Row, kFp8Group };

template <int kThreads>
constexpr int block_of() {
  return kThreads <= kWave ? 256 : kThreads;
}

// v times the rounded inverse of the scale, not the quotient: a value on a tie of two 8-bit numbers
// may go to either (1e-5 of the values of bfloat16 rows; the last bit of the norm's root moves
// twice as many).
__device__ inline uint2 to_fp8(F8 v, float inv) {
  v *= inv;
  uint2 r;
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
  r.x = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], w, true);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(v[4], v[5], 0, false);
  r.y = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[6], v[7], w, true);
  return r;
}

__device__ inline void store_bytes(uint8_t* p, uint2 v, int n) {
  if (n >= 8) {
    __builtin_memcpy(p, &v, 8);
  } else {
    for (int j = 0; j < n; ++j) p[j] = (uint8_t)((j < 4 ? v.x : v.y) >> (8 * (j & 3)));
  }
}

__device__ inline float largest(F8 v) {
  float m = 0.0f;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = fmaxf(m, fabsf(v[j]));
  return m;
}

constexpr float kFp8Max = 448.0f;
constexpr float kLeastScale = 0x1p-126f;

template <class T, int kThreads, int kVecs, int kMode, bool kWhole>
__global__ __launch_bounds__(block_of<kThreads>()) void norm_kernel(NormArgs a) {
  constexpr int kRows = block_of<kThreads>() / kThreads;
  __shared__ float smem[2][16];
  const int lane = threadIdx.x % kThreads;
  const int64_t row = block_index() * kRows + row_slot<kThreads>();
  if (row >= a.rows) return;  // (whole rows leave: no barrier or reduction spans two rows)
  const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
  const T* res = static_cast<const T*>(a.residual) + row * a.residual_stride;
  T* hout = static_cast<T*>(a.h) + row * a.dim;
  const uint64_t drop = drop_row(a.drop, row, a.dim);
  Reg8<T> x_raw[kVecs], res_raw[kVecs];
  Weight8<T> w_raw[kVecs];
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    const int col = 8 * (lane + i * kThreads);
    x_raw[i] = load_raw<T, kWhole>(x, col, a.dim);
    res_raw[i] = a.residual ? load_raw<T, kWhole>(res, col, a.dim) : Reg8<T>{};
    w_raw[i] = load_weight<T, kWhole>(a.weight, a.w_f32, col, a.dim);
  }
  F8 h[kVecs];
  float sq = 0.0f;
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    const int col = 8 * (lane + i * kThreads);
    h[i] = widen<T, kWhole>(x_raw[i], col, a.dim);
    if constexpr (kMode == kDrop) h[i] = drop8(h[i], a.drop, drop, col);
    if (a.residual) h[i] += widen<T, kWhole>(res_raw[i], col, a.dim);
    if (a.h) store8<T, kWhole>(hout, col, a.dim, h[i]);
#pragma unroll
    for (int j = 0; j < 8; ++j) sq = fmaf(h[i][j], h[i][j], sq);
  }
  sq = row_reduce<Sum, kThreads>(sq, smem[0]);
  const float r = 1.0f / sqrtf(fmaf(sq, a.inv_dim, a.eps));
  float top = 0.0f;
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    const int col = 8 * (lane + i * kThreads), n = a.dim - col;
    h[i] = h[i] * r * widen<T, kWhole>(w_raw[i], a.w_f32, col, a.dim);
    if constexpr (kMode == kPlain || kMode == kDrop) {
      store8<T, kWhole>(static_cast<T*>(a.y) + row * a.dim, col, a.dim, h[i]);
    } else if constexpr (kMode == kFp8Row) {
      top = fmaxf(top, largest(h[i]));
    } else {
      // 16 lanes hold the 128 columns of a group (lane and i*kThreads are multiples of 16 apart)
      const float m = lanes_reduce<Max, 16>(largest(h[i]));
      const float s = fmaxf(m / kFp8Max, kLeastScale);
      if (n > 0) {
        store_bytes(a.q + row * a.dim + col, to_fp8(h[i], 1.0f / s), n);
        if (lane % 16 == 0) a.scales[row * ((a.dim + 127) / 128) + col / 128] = s;
      }
    }
  }
  if constexpr (kMode == kFp8Row) {
    top = row_reduce<Max, kThreads>(top, smem[1]);
    const float s = fmaxf(top / kFp8Max, kLeastScale);
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      const int col = 8 * (lane + i * kThreads), n = a.dim - col;
      if (n > 0) store_bytes(a.q + row * a.dim + col, to_fp8(h[i], 1.0f / s), n);
    }
    if (lane == 0) a.scales[row] = s;
  }
}

// ---- gradients ------------------------------------------------------------------------------
struct NormGradArgs {
  const void *gy, *gh, *h, *weight;
  int64_t gy_stride, gh_stride, h_stride;
  int64_t rows;
  int dim;
  int w_f32;
  float eps, inv_dim;
  void *gx, *gr, *gw;
  float* partial;  // [groups, dim] sums of grad_weight, or NULL
  Dropout drop;
};

// A workgroup takes the rows blockIdx.x*kRows + slot, and every gridDim.x*kRows-th after them,
// and keeps the sum of grad_y * n over them in registers.
template <class T, int kThreads, int kVecs, bool kDropped, bool kWhole>
__global__ __launch_bounds__(block_of<kThreads>()) void norm_grad_kernel(NormGradArgs a) {
  constexpr int kBlock = block_of<kThreads>(), kRows = kBlock / kThreads;
  __shared__ float smem[2][2][16];
  __shared__ float joined[kRows > 1 ? 8 * kThreads * kVecs : 1];
  const int lane = threadIdx.x % kThreads, slot = row_slot<kThreads>();
  F8 dw[kVecs] = {}, w[kVecs];
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    const int col = 8 * (lane + i * kThreads);
    w[i] = widen<T, kWhole>(load_weight<T, kWhole>(a.weight, a.w_f32, col, a.dim), a.w_f32, col,
                            a.dim);
  }
  int turn = 0;
  for (int64_t row = (int64_t)blockIdx.x * kRows + slot; row < a.rows;
       row += (int64_t)gridDim.x * kRows, turn ^= 1) {
    const T* gy = static_cast<const T*>(a.gy) + row * a.gy_stride;
    const T* hp = static_cast<const T*>(a.h) + row * a.h_stride;
    const T* gh = static_cast<const T*>(a.gh) + row * a.gh_stride;
    Reg8<T> h_raw[kVecs], g_raw[kVecs], gh_raw[kVecs];
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      const int col = 8 * (lane + i * kThreads);
      h_raw[i] = load_raw<T, kWhole>(hp, col, a.dim);
      g_raw[i] = load_raw<T, kWhole>(gy, col, a.dim);
      gh_raw[i] = a.gh ? load_raw<T, kWhole>(gh, col, a.dim) : Reg8<T>{};
    }
    float sq = 0.0f, dot = 0.0f;
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      const int col = 8 * (lane + i * kThreads);
      const F8 h = widen<T, kWhole>(h_raw[i], col, a.dim);
      const F8 gw = widen<T, kWhole>(g_raw[i], col, a.dim) * w[i];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        sq = fmaf(h[j], h[j], sq);
        dot = fmaf(gw[j], h[j], dot);
      }
    }
    sq = row_reduce<Sum, kThreads>(sq, smem[turn][0]);
    dot = row_reduce<Sum, kThreads>(dot, smem[turn][1]);
    const float r = 1.0f / sqrtf(fmaf(sq, a.inv_dim, a.eps));
    const float k = dot * a.inv_dim * r * r;  // grad = r * (g*w - h*k) + grad_h
    const uint64_t drop = drop_row(a.drop, row, a.dim);
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      const int col = 8 * (lane + i * kThreads);
      const F8 h = widen<T, kWhole>(h_raw[i], col, a.dim), g = widen<T, kWhole>(g_raw[i], col, a.dim);
      dw[i] += g * h * r;
      F8 d = (g * w[i] - h * k) * r;
      if (a.gh) d += widen<T, kWhole>(gh_raw[i], col, a.dim);
      if (a.gr) store8<T, kWhole>(static_cast<T*>(a.gr) + row * a.dim, col, a.dim, d);
      if constexpr (kDropped)
        store8<T, kWhole>(static_cast<T*>(a.gx) + row * a.dim, col, a.dim,
                  drop8(d, a.drop, drop, col));
    }
  }
  if (!a.partial) return;
  if constexpr (kRows > 1) {  // the slots' sums in order
    for (int s = 0; s < kRows; ++s) {
      if (slot == s) {
#pragma unroll
        for (int i = 0; i < kVecs; ++i)
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int at = 8 * (lane + i * kThreads) + j;
            if (s > 0) dw[i][j] += joined[at];
            if (s < kRows - 1) joined[at] = dw[i][j];
          }
      }
      __syncthreads();
    }
  }
  if (slot == kRows - 1) {
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      const int col = 8 * (lane + i * kThreads);
      store8<float, kWhole>(a.partial + (int64_t)blockIdx.x * a.dim, col, a.dim, dw[i]);
    }
  }
}

// grad_weight from the workgroups' sums: a workgroup takes 32 columns (a line of memory), 32
// slices of the sums side by side, the slices added in order.
template <class O>
__global__ __launch_bounds__(1024) void join_weight_kernel(const float* __restrict__ partial,
                                                           int groups, int dim,
                                                           O* __restrict__ out) {
  __shared__ float part[32][33];
  const int c = threadIdx.x % 32, slice = threadIdx.x / 32;
  const int col = blockIdx.x * 32 + c;
  float s = 0.0f;
  if (col < dim) {
    for (int g = slice; g < groups; g += 32 * 8) {  // eight loads in flight, the last ones too
      float v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u)
        v[u] = partial[(int64_t)(g + 32 * u < groups ? g + 32 * u : g) * dim + col];
#pragma unroll
      for (int u = 0; u < 8; ++u) s += g + 32 * u < groups ? v[u] : 0.0f;
    }
  }
  part[slice][c] = s;
  __syncthreads();
  if (threadIdx.x < 32 && col < dim) {
    s = part[0][c];
    for (int k = 1; k < 32; ++k) s += part[k][c];
    out[col] = (O)s;
  }
}

// ---- launches -------------------------------------------------------------------------------
// f is called with the row's layout for `dim` columns.
template <int kThreads_, int kVecs_>
struct Layout {
  static constexpr int kThreads = kThreads_, kVecs = kVecs_;
};

template <bool kGrad, class F>
void with_layout(int64_t dim, F&& f) {
  if (dim <= 128) return f(Layout<16, 1>{});
  if (dim <= 256) return f(Layout<32, 1>{});
  if (dim <= 512) return f(Layout<64, 1>{});
  if (dim <= 1024) return f(Layout<128, 1>{});
  if (dim <= 2048) return f(Layout<256, 1>{});
  if (dim <= 4096) return f(Layout<512, 1>{});
  if (dim <= 8192) return f(Layout<1024, 1>{});
  // (the gradient holds five arrays of a row: 1024 threads have too few registers for 16 columns)
  if constexpr (kGrad) return f(Layout<512, 4>{});
  else return f(Layout<1024, 2>{});
}

template <class F>
void with_type(int dtype, F&& f) {
  if (dtype == OMQ_NET_F32) return f(float{});
  if (dtype == OMQ_NET_BF16) return f(bf16{});
  return f(f16{});
}

template <int kMode>
void launch_norm(const NormArgs& a, int dtype, hipStream_t st) {
  with_type(dtype, [&](auto t) {
    using T = decltype(t);
    with_layout<false>(a.dim, [&](auto l) {
      using L = decltype(l);
      constexpr int kBlock = block_of<L::kThreads>();
      const dim3 grid = grid_of(ceil_div(a.rows, kBlock / L::kThreads), kBlock);
      const auto kernel = a.dim % 8 == 0 ? norm_kernel<T, L::kThreads, L::kVecs, kMode, true>
                                         : norm_kernel<T, L::kThreads, L::kVecs, kMode, false>;
      kernel<<<grid, kBlock, 0, st>>>(a);
    });
  });
}

// Workgroups of the gradient: 16 waves a compute unit (with 32, 16384 rows of 4096 take 135 us
// instead of 128: more partial sums of the weight's gradient), and where the rows are few, four
// rows or more each for the same reason, as long as the compute units have one.
constexpr int64_t kGradWaves = 256 * 16;

int64_t grad_groups(int64_t rows, int64_t dim) {
  int64_t groups = 0;
  with_layout<true>(dim, [&](auto l) {
    using L = decltype(l);
    constexpr int kBlock = block_of<L::kThreads>();
    const int64_t all = ceil_div(rows, kBlock / L::kThreads);
    const int64_t few = ceil_div(all, 4) < 256 ? 256 : ceil_div(all, 4);
    const int64_t most = kGradWaves * kWave / kBlock < few ? kGradWaves * kWave / kBlock : few;
    groups = all < most ? all : most;
  });
  return groups;
}

int check_norm(const char* name, int64_t rows, int64_t dim, int dtype, int weight_dtype) {
  if (!dtype_known(dtype) || (weight_dtype != dtype && weight_dtype != OMQ_NET_F32))
    return net_fail(OMQ_NET_E_ARG, "%s: rows of type %d with a weight of type %d", name, dtype,
                    weight_dtype);
  if (rows < 0 || dim < 1)
    return net_fail(OMQ_NET_E_ARG, "%s: rows %lld, dim %lld", name, (long long)rows,
                    (long long)dim);
  if (rows > OMQ_NET_MAX_COUNT || dim > OMQ_NET_MAX_NORM_DIM)
    return net_fail(OMQ_NET_E_LIMIT, "%s: rows %lld (at most %d), dim %lld (at most %d)", name,
                    (long long)rows, OMQ_NET_MAX_COUNT, (long long)dim, OMQ_NET_MAX_NORM_DIM);
  return OMQ_NET_OK;
}

int check_p(const char* name, double p) {
  if (!(p >= 0.0 && p <= 1.0))
    return net_fail(OMQ_NET_E_ARG, "%s: p %g outside [0, 1]", name, p);
  return OMQ_NET_OK;
}

}  // namespace

int check_dropout(const char* name, double p) { return check_p(name, p); }

}  // namespace omq_net

using namespace omq_net;

extern "C" {

int omq_add_rms_norm(const void* x, int64_t x_stride, const void* residual,
                     int64_t residual_stride, const void* weight, int weight_dtype, int64_t rows,
                     int64_t dim, int dtype, float eps, double p, uint64_t seed, uint64_t offset,
                     void* y, void* h, void* stream) {
  const char* name = "omq_add_rms_norm";
  if (int rc = check_norm(name, rows, dim, dtype, weight_dtype)) return rc;
  if (int rc = check_p(name, p)) return rc;
  if (x_stride < 0 || residual_stride < 0)
    return net_fail(OMQ_NET_E_ARG, "%s: negative stride", name);
  if (rows == 0) return OMQ_NET_OK;
  if (!x || !weight || !y) return net_fail(OMQ_NET_E_ARG, "%s: a null array", name);
  NormArgs a{};
  a.x = x, a.residual = residual, a.weight = weight, a.x_stride = x_stride;
  a.residual_stride = residual_stride, a.rows = rows, a.dim = (int)dim;
  a.w_f32 = weight_dtype == OMQ_NET_F32, a.eps = eps, a.inv_dim = 1.0f / (float)dim;
  a.y = y, a.h = h, a.drop = make_dropout(p, seed, offset);
  if (a.drop.threshold)
    launch_norm<kDrop>(a, dtype, (hipStream_t)stream);
  else
    launch_norm<kPlain>(a, dtype, (hipStream_t)stream);
  return net_status(name);
}

int omq_add_rms_norm_fp8(const void* x, int64_t x_stride, const void* residual,
                         int64_t residual_stride, const void* weight, int weight_dtype,
                         int64_t rows, int64_t dim, int dtype, float eps, int group, uint8_t* q,
                         float* scales, void* h, void* stream) {
  const char* name = "omq_add_rms_norm_fp8";
  if (int rc = check_norm(name, rows, dim, dtype, weight_dtype)) return rc;
  if (group != 0 && group != 128)
    return net_fail(OMQ_NET_E_ARG, "%s: group %d is neither 0 (a row) nor 128", name, group);
  if (x_stride < 0 || residual_stride < 0)
    return net_fail(OMQ_NET_E_ARG, "%s: negative stride", name);
  if (rows == 0) return OMQ_NET_OK;
  if (!x || !weight || !q || !scales) return net_fail(OMQ_NET_E_ARG, "%s: a null array", name);
  NormArgs a{};
  a.x = x, a.residual = residual, a.weight = weight, a.x_stride = x_stride;
  a.residual_stride = residual_stride, a.rows = rows, a.dim = (int)dim;
  a.w_f32 = weight_dtype == OMQ_NET_F32, a.eps = eps, a.inv_dim = 1.0f / (float)dim;
  a.q = q, a.scales = scales, a.h = h;
  if (group)
    launch_norm<kFp8Group>(a, dtype, (hipStream_t)stream);
  else
    launch_norm<kFp8Row>(a, dtype, (hipStream_t)stream);
  return net_status(name);
}

int64_t omq_add_rms_norm_grad_workspace(int64_t rows, int64_t dim) {
  if (rows < 0 || dim < 1 || rows > OMQ_NET_MAX_COUNT || dim > OMQ_NET_MAX_NORM_DIM)
    return OMQ_NET_E_ARG;
  return 4 * dim * grad_groups(rows, dim);
}

int omq_add_rms_norm_grad(const void* grad_y, int64_t grad_y_stride, const void* grad_h,
                          int64_t grad_h_stride, const void* h, int64_t h_stride,
                          const void* weight, int weight_dtype, int64_t rows, int64_t dim,
                          int dtype, float eps, double p, uint64_t seed, uint64_t offset,
                          void* grad_x, void* grad_residual, void* grad_weight, void* workspace,
                          int64_t workspace_bytes, void* stream) {
  const char* name = "omq_add_rms_norm_grad";
  if (int rc = check_norm(name, rows, dim, dtype, weight_dtype)) return rc;
  if (int rc = check_p(name, p)) return rc;
  if (grad_y_stride < 0 || grad_h_stride < 0 || h_stride < 0)
    return net_fail(OMQ_NET_E_ARG, "%s: negative stride", name);
  NormGradArgs a{};
  a.drop = make_dropout(p, seed, offset);
  if ((a.drop.threshold != 0) != (grad_x != nullptr) && rows > 0)
    return net_fail(OMQ_NET_E_ARG, "%s: grad_x is written when p (%g) is not 0, and only then",
                    name, p);
  const int64_t need = grad_weight ? 4 * dim * grad_groups(rows, dim) : 0;
  if (need > 0 && (!workspace || workspace_bytes < need))
    return net_fail(OMQ_NET_E_ARG, "%s: workspace of %lld bytes, %lld needed", name,
                    (long long)workspace_bytes, (long long)need);
  if (rows > 0 && (!grad_y || !h || !weight))
    return net_fail(OMQ_NET_E_ARG, "%s: a null array", name);
  hipStream_t st = (hipStream_t)stream;
  a.gy = grad_y, a.gh = grad_h, a.h = h, a.weight = weight, a.gy_stride = grad_y_stride;
  a.gh_stride = grad_h_stride, a.h_stride = h_stride, a.rows = rows, a.dim = (int)dim;
  a.w_f32 = weight_dtype == OMQ_NET_F32, a.eps = eps, a.inv_dim = 1.0f / (float)dim;
  a.gx = grad_x, a.gr = grad_residual;
  a.partial = grad_weight ? static_cast<float*>(workspace) : nullptr;
  const int64_t groups = grad_groups(rows, dim);
  if (rows > 0)
    with_type(dtype, [&](auto t) {
      using T = decltype(t);
      with_layout<true>(dim, [&](auto l) {
        using L = decltype(l);
        constexpr int kBlock = block_of<L::kThreads>();
        const auto go = [&](auto dropped, auto whole) {
          norm_grad_kernel<T, L::kThreads, L::kVecs, dropped.value, whole.value>
              <<<(uint32_t)groups, kBlock, 0, st>>>(a);
        };
        using Yes = std::true_type;
        using No = std::false_type;
        if (a.drop.threshold)
          dim % 8 == 0 ? go(Yes{}, Yes{}) : go(Yes{}, No{});
        else
          dim % 8 == 0 ? go(No{}, Yes{}) : go(No{}, No{});
      });
    });
  if (grad_weight) {
    const uint32_t grid = (uint32_t)ceil_div(dim, 32);
    with_type(weight_dtype, [&](auto t) {
      using O = decltype(t);
      join_weight_kernel<O><<<grid, 1024, 0, st>>>(static_cast<const float*>(workspace),
                                                  (int)groups, (int)dim,
                                                  static_cast<O*>(grad_weight));
    });
  }
  return net_status(name);
}

}  // extern "C"
