// The clipped policy loss over legal actions with a KL term, and its gradient (gfx950).
//
// Per row, with m the largest legal logit, s = sum e^(z-m), tp = sum pi, tz = sum pi (z - m) and
// tl = sum pi log pi over the legal actions (pi the target):
//   logq_a = z_a - m - log s
//   kl     = tl - tz + tp log s
//   dz_a   = push p_a + slope [a taken] - kl_coef pi_a,   p_a = e^(z_a - m) / s,
// where slope is the loss's derivative by logp and push = kl_coef tp - slope.
//
// One pass over the logits where the row fits the registers of the threads that share it (the
// maximum, the sums and the gradient all come from the same loads); longer rows, and rows so
// few that they would leave most of the chip idle, are cut into spans whose running (m, s, tp,
// tz, tl) are joined, and the gradient is a second, element-wise pass.  Bound by memory.
#include "net_common.h"

namespace omq_net {
namespace {

constexpr float kInf = __builtin_inff();
constexpr float kLog2e = 1.4426950408889634f;

// Running statistics of a part of a row.
struct Stats {
  float m, s, tp, tz, tl;
};

__device__ inline Stats no_stats() { return Stats{-kInf, 0.0f, 0.0f, 0.0f, 0.0f}; }

__device__ inline float exp_fast(float x) { return __builtin_amdgcn_exp2f(x * kLog2e); }

// m for exponents: -inf (nothing legal yet) and +-inf logits must not give inf - inf where the
// true weight is 0.
__device__ inline float base_of(float m) { return m == -kInf ? 0.0f : m; }

__device__ inline Stats join(const Stats& a, const Stats& b) {
  Stats r;
  r.m = fmaxf(a.m, b.m);
  const float base = base_of(r.m);
  const float ea = a.m == r.m ? 1.0f : exp_fast(a.m - base);
  const float eb = b.m == r.m ? 1.0f : exp_fast(b.m - base);
  r.s = a.s * ea + b.s * eb;
  r.tp = a.tp + b.tp;
  r.tl = a.tl + b.tl;
  // sum pi (z - m) about another m; a part whose m is -inf was formed about 0
  r.tz = a.tz + b.tz;
  if (a.tp != 0.0f) r.tz += a.tp * (base_of(a.m) - base);
  if (b.tp != 0.0f) r.tz += b.tp * (base_of(b.m) - base);
  return r;
}

// What the gradient of a row needs.
struct RowGrad {
  float m, inv_s;  // p = e^(z - m) * inv_s; inv_s = 0: the row has no gradient
  float push, slope;
};

struct RowOut {
  float loss, logp, kl;
  RowGrad g;
};

// z_taken: the logit of the taken action, `taken`: it is legal and in range.
__device__ inline RowOut finish_row(const omq_policy_rows& r, int64_t row, const Stats& t,
                                    float z_taken, bool taken) {
  RowOut o{};
  const bool live = !(t.m == -kInf && t.s == 0.0f);
  if (!live) return o;
  const float base = base_of(t.m);
  const float log_s = logf(t.s);
  float slope = 0.0f;
  if (taken) {
    o.logp = z_taken - base - log_s;
    const float adv = r.advantages[row];
    const float ratio = expf(o.logp - r.old_logp[row]);
    const float one = ratio * adv;
    const float two = fminf(fmaxf(ratio, 1.0f - r.clip_low), 1.0f + r.clip_high) * adv;
    o.loss = -(one <= two || one != one ? one : two);
    if (one <= two || one != one) slope = -one;
    if (r.ref_logp) {
      const float d = r.ref_logp[row] - o.logp, e = expm1f(d);
      o.kl = e - d;
      slope -= r.kl_coef * e;
    }
  }
  if (r.target) o.kl = t.tl - t.tz + (t.tp != 0.0f ? t.tp * log_s : 0.0f);
  o.loss += r.kl_coef != 0.0f ? r.kl_coef * o.kl : 0.0f;
  o.g.m = base;
  o.g.inv_s = 1.0f / t.s;
  o.g.slope = slope;
  o.g.push = (r.kl_coef != 0.0f ? r.kl_coef * t.tp : 0.0f) - slope;
  // a row that adds nothing to the loss has no gradient, whatever its logits hold (padding)
  if (slope == 0.0f && o.g.push == 0.0f && (!r.target || r.kl_coef == 0.0f)) o.g.inv_s = 0.0f;
  return o;
}

// The taken action of a row, -1 when it is out of range.
__device__ inline int64_t taken_of(const omq_policy_rows& r, int64_t row) {
  const int64_t a = r.taken_are_64 ? static_cast<const int64_t*>(r.taken)[row]
                                   : (int64_t) static_cast<const int32_t*>(r.taken)[row];
  return a >= 0 && a < r.actions ? a : -1;
}

// Bit j: action 8*block + j of the row is there and legal.
__device__ inline uint32_t legal_bits(const uint8_t* legal, int64_t col, int64_t n) {
  uint32_t bits = n >= 8 ? 0xFFu : (1u << n) - 1u;
  if (!legal) return bits;
  uint64_t b = 0;
  if (n >= 8) {
    __builtin_memcpy(&b, legal + col, 8);
  } else {
    for (int j = 0; j < (int)n; ++j) b |= (uint64_t)legal[col + j] << (8 * j);
  }
  uint32_t some = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) some |= ((b >> (8 * j)) & 0xFFu) ? 1u << j : 0u;
  return bits & some;
}

__device__ inline float gradient(const RowGrad& g, float z, bool is_taken, float pi, float coef) {
  const float p = exp_fast(z - g.m) * g.inv_s;
  float d = g.push * p;
  if (is_taken) d += g.slope;
  if (pi > 0.0f) d -= coef * pi;
  return d;
}

// ---- rows in registers ----------------------------------------------------------------------
template <int kThreads>
constexpr int block_of() {
  return kThreads < 256 ? 256 : kThreads;
}

template <class T, int kThreads, int kVecs, bool kGrad>
__global__ __launch_bounds__(block_of<kThreads>()) void loss_rows_kernel(
    omq_policy_rows r, const float* __restrict__ row_weight, float* __restrict__ loss,
    float* __restrict__ logp, float* __restrict__ kl, float4* __restrict__ stats,
    T* __restrict__ grad) {
  constexpr int kRows = block_of<kThreads>() / kThreads;
  __shared__ float smem[5][16];
  const int lane = threadIdx.x % kThreads;
  const int64_t row = (int64_t)blockIdx.x * kRows + threadIdx.x / kThreads;
  if (row >= r.rows) return;
  const int cols = (int)r.actions;
  const T* logits = static_cast<const T*>(r.logits) + row * r.logits_stride;
  const uint8_t* legal = r.legal ? r.legal + row * r.legal_stride : nullptr;
  const float* target = r.target ? r.target + row * r.target_stride : nullptr;
  const int64_t act = taken_of(r, row);
  const bool taken = act >= 0 && (!legal || legal[act]);
  const float z_taken = taken ? (float)logits[act] : 0.0f;
  Vec8<T> z[kVecs];
  uint32_t ok[kVecs];
  Stats t = no_stats();
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    const int col = 8 * (lane + i * kThreads), n = cols - col;
    ok[i] = 0;
    if (n > 0) {
      z[i] = load_raw<T>(logits + col, n);
      ok[i] = legal_bits(legal, col, n);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (ok[i] >> j & 1) t.m = fmaxf(t.m, (float)z[i][j]);
    }
  }
  t.m = row_reduce<Max, kThreads>(t.m, smem[0]);
  const float base = base_of(t.m);
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    const int col = 8 * (lane + i * kThreads), n = cols - col;
    if (n > 0) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (ok[i] >> j & 1) t.s += exp_fast((float)z[i][j] - base);
      if (target) {
        const F8 pi = load8<float>(target + col, n);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if ((ok[i] >> j & 1) && pi[j] > 0.0f) {
            t.tp += pi[j];
            t.tz += pi[j] * ((float)z[i][j] - base);
            t.tl += pi[j] * logf(pi[j]);
          }
      }
    }
  }
  t.s = row_reduce<Sum, kThreads>(t.s, smem[1]);
  if (target) {
    t.tp = row_reduce<Sum, kThreads>(t.tp, smem[2]);
    t.tz = row_reduce<Sum, kThreads>(t.tz, smem[3]);
    t.tl = row_reduce<Sum, kThreads>(t.tl, smem[4]);
  }
  const RowOut o = finish_row(r, row, t, z_taken, taken);
  if (lane == 0) {
    loss[row] = o.loss;
    logp[row] = o.logp;
    kl[row] = o.kl;
    if (stats) stats[row] = make_float4(o.g.m, o.g.inv_s, o.g.push, o.g.slope);
  }
  if constexpr (kGrad) {
    const float w = row_weight ? row_weight[row] : 1.0f;
    T* g = grad + row * cols;
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      const int col = 8 * (lane + i * kThreads), n = cols - col;
      if (n > 0) {
        F8 pi = {}, d = {};
        if (target) pi = load8<float>(target + col, n);
        if (o.g.inv_s != 0.0f) {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (ok[i] >> j & 1)
              d[j] = w * gradient(o.g, (float)z[i][j], taken && col + j == act, pi[j], r.kl_coef);
        }
        store8<T>(g + col, d, n);
      }
    }
  }
}

// ---- spans of rows --------------------------------------------------------------------------
// Statistics of span blockIdx.x of row blockIdx.y.
template <class T>
__global__ __launch_bounds__(256) void loss_span_kernel(omq_policy_rows r, int64_t row0,
                                                        int64_t span, Stats* __restrict__ parts) {
  __shared__ Stats waves[4];
  const int64_t row = row0 + blockIdx.y;
  const T* logits = static_cast<const T*>(r.logits) + row * r.logits_stride;
  const uint8_t* legal = r.legal ? r.legal + row * r.legal_stride : nullptr;
  const float* target = r.target ? r.target + row * r.target_stride : nullptr;
  const int64_t from = blockIdx.x * span;
  const int64_t to = from + span < r.actions ? from + span : r.actions;
  Stats t = no_stats();
  for (int64_t col = from + 8 * threadIdx.x; col < to; col += 8 * 256) {
    const int64_t n = to - col;
    const F8 z = load8<T>(logits + col, n < 8 ? (int)n : 8);
    const uint32_t ok = legal_bits(legal, col, n);
    Stats u = no_stats();
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (ok >> j & 1) u.m = fmaxf(u.m, z[j]);
    const float base = base_of(u.m);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (ok >> j & 1) u.s += exp_fast(z[j] - base);
    if (target) {
      const F8 pi = load8<float>(target + col, n < 8 ? (int)n : 8);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if ((ok >> j & 1) && pi[j] > 0.0f) {
          u.tp += pi[j];
          u.tz += pi[j] * (z[j] - base);
          u.tl += pi[j] * logf(pi[j]);
        }
    }
    t = join(t, u);
  }
  for (int d = 1; d < kWave; d <<= 1) {
    Stats u;
    u.m = __shfl_xor(t.m, d);
    u.s = __shfl_xor(t.s, d);
    u.tp = __shfl_xor(t.tp, d);
    u.tz = __shfl_xor(t.tz, d);
    u.tl = __shfl_xor(t.tl, d);
    t = join(t, u);
  }
  if ((threadIdx.x & (kWave - 1)) == 0) waves[threadIdx.x / kWave] = t;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 4; ++w) t = join(t, waves[w]);
    parts[row * gridDim.x + blockIdx.x] = t;
  }
}

// A thread a row: its spans joined in order.
template <class T>
__global__ __launch_bounds__(64) void loss_join_kernel(omq_policy_rows r,
                                                       const Stats* __restrict__ parts, int spans,
                                                       float* __restrict__ loss,
                                                       float* __restrict__ logp,
                                                       float* __restrict__ kl,
                                                       float4* __restrict__ stats) {
  const int64_t row = (int64_t)blockIdx.x * 64 + threadIdx.x;
  if (row >= r.rows) return;
  Stats t = no_stats();
  for (int k = 0; k < spans; ++k) t = join(t, parts[row * spans + k]);
  const int64_t act = taken_of(r, row);
  const bool taken = act >= 0 && (!r.legal || r.legal[row * r.legal_stride + act]);
  const float z =
      taken ? (float)static_cast<const T*>(r.logits)[row * r.logits_stride + act] : 0.0f;
  const RowOut o = finish_row(r, row, t, z, taken);
  loss[row] = o.loss;
  logp[row] = o.logp;
  kl[row] = o.kl;
  if (stats) stats[row] = make_float4(o.g.m, o.g.inv_s, o.g.push, o.g.slope);
}

// The gradient from a row's statistics: 2048 columns of a row a workgroup.
template <class T>
__global__ __launch_bounds__(256) void loss_grad_kernel(omq_policy_rows r, int blocks,
                                                        const float4* __restrict__ stats,
                                                        const float* __restrict__ row_weight,
                                                        T* __restrict__ grad) {
  const int64_t first = (int64_t)blockIdx.x * 256;
  const int64_t row0 = first / blocks;
  const uint32_t in = (uint32_t)(first - row0 * blocks) + threadIdx.x;
  const int64_t row = row0 + in / (uint32_t)blocks;
  const int64_t col = 8ll * (in % (uint32_t)blocks);
  if (row >= r.rows) return;
  const int64_t left = r.actions - col;
  const int n = left < 8 ? (int)left : 8;
  const float4 st = stats[row];
  const RowGrad g{st.x, st.y, st.z, st.w};
  const float w = row_weight ? row_weight[row] : 1.0f;
  const int64_t act = taken_of(r, row);
  F8 d = {};
  if (g.inv_s != 0.0f) {
    const F8 z = load8<T>(static_cast<const T*>(r.logits) + row * r.logits_stride + col, n);
    const uint32_t ok = legal_bits(r.legal ? r.legal + row * r.legal_stride : nullptr, col, n);
    F8 pi = {};
    if (r.target) pi = load8<float>(r.target + row * r.target_stride + col, n);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (ok >> j & 1) d[j] = w * gradient(g, z[j], col + j == act, pi[j], r.kl_coef);
  }
  store8<T>(grad + row * r.actions + col, d, n);
}

// ---- launches -------------------------------------------------------------------------------
template <int kThreads_, int kVecs_>
struct Layout {
  static constexpr int kThreads = kThreads_, kVecs = kVecs_;
};

constexpr int64_t kRowActions = 16384;  // the longest row that is held in registers

template <class F>
void with_layout(int64_t cols, F&& f) {
  if (cols <= 128) return f(Layout<16, 1>{});
  if (cols <= 256) return f(Layout<32, 1>{});
  if (cols <= 512) return f(Layout<64, 1>{});
  if (cols <= 1024) return f(Layout<64, 2>{});
  if (cols <= 2048) return f(Layout<64, 4>{});
  if (cols <= 4096) return f(Layout<256, 2>{});
  if (cols <= 8192) return f(Layout<256, 4>{});
  return f(Layout<256, 8>{});
}

template <class F>
void with_type(int dtype, F&& f) {
  if (dtype == OMQ_NET_F32) return f(float{});
  if (dtype == OMQ_NET_BF16) return f(bf16{});
  return f(f16{});
}

struct LossPlan {
  bool in_rows;
  int64_t span, spans, at_parts, at_stats, bytes;
};

LossPlan loss_plan(int64_t rows, int64_t actions) {
  LossPlan p{};
  p.in_rows = actions <= kRowActions;
  if (p.in_rows) return p;
  // spans for about 2048 workgroups, of at least 8192 columns
  int64_t spans = ceil_div(2048, rows > 0 ? rows : 1);
  const int64_t most = ceil_div(actions, 8192);
  spans = spans < 1 ? 1 : spans > most ? most : spans;
  p.span = ceil_div(ceil_div(actions, spans), 8) * 8;
  p.spans = ceil_div(actions, p.span);
  p.at_stats = 0;
  p.at_parts = 16 * rows;
  p.bytes = p.at_parts + (int64_t)sizeof(Stats) * rows * p.spans;
  return p;
}

bool loss_sizes_ok(int64_t rows, int64_t actions) {
  return rows >= 0 && actions >= 1 && rows <= OMQ_NET_MAX_COUNT && actions <= OMQ_NET_MAX_COUNT &&
         ceil_div(rows * ceil_div(actions, 8), 256) <= OMQ_NET_MAX_COUNT;
}

int check_rows(const char* name, const omq_policy_rows* r) {
  if (!r) return net_fail(OMQ_NET_E_ARG, "%s: rows is null", name);
  if (!dtype_known(r->dtype))
    return net_fail(OMQ_NET_E_ARG, "%s: unknown type %d", name, r->dtype);
  if (!loss_sizes_ok(r->rows, r->actions))
    return net_fail(r->rows < 0 || r->actions < 1 ? OMQ_NET_E_ARG : OMQ_NET_E_LIMIT,
                    "%s: rows %lld, actions %lld", name, (long long)r->rows,
                    (long long)r->actions);
  if (r->logits_stride < 0 || r->legal_stride < 0 || r->target_stride < 0)
    return net_fail(OMQ_NET_E_ARG, "%s: negative stride", name);
  if (r->target && r->ref_logp)
    return net_fail(OMQ_NET_E_ARG, "%s: target and ref_logp exclude each other", name);
  if (r->rows > 0 && (!r->logits || !r->taken || !r->advantages || !r->old_logp))
    return net_fail(OMQ_NET_E_ARG, "%s: a null array", name);
  return OMQ_NET_OK;
}

template <bool kGrad>
void launch_rows(const omq_policy_rows& r, const float* row_weight, float* loss, float* logp,
                 float* kl, float* stats, void* grad, hipStream_t st) {
  with_type(r.dtype, [&](auto t) {
    using T = decltype(t);
    with_layout(r.actions, [&](auto l) {
      using L = decltype(l);
      constexpr int kBlock = block_of<L::kThreads>();
      const uint32_t grid = (uint32_t)ceil_div(r.rows, kBlock / L::kThreads);
      loss_rows_kernel<T, L::kThreads, L::kVecs, kGrad><<<grid, kBlock, 0, st>>>(
          r, row_weight, loss, logp, kl, reinterpret_cast<float4*>(stats),
          static_cast<T*>(grad));
    });
  });
}

void launch_spans(const omq_policy_rows& r, const LossPlan& p, float* loss, float* logp, float* kl,
                  float* stats, char* ws, hipStream_t st) {
  Stats* parts = reinterpret_cast<Stats*>(ws + p.at_parts);
  with_type(r.dtype, [&](auto t) {
    using T = decltype(t);
    for (int64_t row0 = 0; row0 < r.rows; row0 += 65535) {
      const int64_t n = r.rows - row0 < 65535 ? r.rows - row0 : 65535;
      loss_span_kernel<T><<<dim3((uint32_t)p.spans, (uint32_t)n), 256, 0, st>>>(r, row0, p.span,
                                                                               parts);
    }
    loss_join_kernel<T><<<(uint32_t)ceil_div(r.rows, 64), 64, 0, st>>>(
        r, parts, (int)p.spans, loss, logp, kl, reinterpret_cast<float4*>(stats));
  });
}

void launch_grad(const omq_policy_rows& r, const float* stats, const float* row_weight, void* grad,
                 hipStream_t st) {
  with_type(r.dtype, [&](auto t) {
    using T = decltype(t);
    const int blocks = (int)ceil_div(r.actions, 8);
    const uint32_t grid = (uint32_t)ceil_div(r.rows * blocks, 256);
    loss_grad_kernel<T><<<grid, 256, 0, st>>>(r, blocks, reinterpret_cast<const float4*>(stats),
                                              row_weight, static_cast<T*>(grad));
  });
}

int check_workspace(const char* name, const LossPlan& p, const void* ws, int64_t bytes) {
  if (p.bytes > 0 && (!ws || bytes < p.bytes))
    return net_fail(OMQ_NET_E_ARG, "%s: workspace of %lld bytes, %lld needed", name,
                    (long long)bytes, (long long)p.bytes);
  return OMQ_NET_OK;
}

}  // namespace
}  // namespace omq_net

using namespace omq_net;

extern "C" {

int64_t omq_clipped_policy_loss_workspace(int64_t rows, int64_t actions) {
  if (!loss_sizes_ok(rows, actions)) return OMQ_NET_E_ARG;
  return loss_plan(rows, actions).bytes;
}

int omq_clipped_policy_loss(const omq_policy_rows* r, float* loss, float* logp, float* kl,
                            float* stats, void* workspace, int64_t workspace_bytes,
                            void* stream) {
  const char* name = "omq_clipped_policy_loss";
  if (int rc = check_rows(name, r)) return rc;
  if (r->rows == 0) return OMQ_NET_OK;
  const LossPlan p = loss_plan(r->rows, r->actions);
  if (int rc = check_workspace(name, p, workspace, workspace_bytes)) return rc;
  if (!loss || !logp || !kl) return net_fail(OMQ_NET_E_ARG, "%s: a null array", name);
  hipStream_t st = (hipStream_t)stream;
  if (p.in_rows)
    launch_rows<false>(*r, nullptr, loss, logp, kl, stats, nullptr, st);
  else
    launch_spans(*r, p, loss, logp, kl, stats, static_cast<char*>(workspace), st);
  return net_status(name);
}

int omq_clipped_policy_loss_grad(const omq_policy_rows* r, const float* stats,
                                 const float* row_weight, void* grad, void* stream) {
  const char* name = "omq_clipped_policy_loss_grad";
  if (int rc = check_rows(name, r)) return rc;
  if (r->rows == 0) return OMQ_NET_OK;
  if (!stats || !grad) return net_fail(OMQ_NET_E_ARG, "%s: a null array", name);
  launch_grad(*r, stats, row_weight, grad, (hipStream_t)stream);
  return net_status(name);
}

int omq_clipped_policy_loss_with_grad(const omq_policy_rows* r, const float* row_weight,
                                      float* loss, float* logp, float* kl, void* grad,
                                      void* workspace, int64_t workspace_bytes, void* stream) {
  const char* name = "omq_clipped_policy_loss_with_grad";
  if (int rc = check_rows(name, r)) return rc;
  if (r->rows == 0) return OMQ_NET_OK;
  const LossPlan p = loss_plan(r->rows, r->actions);
  if (int rc = check_workspace(name, p, workspace, workspace_bytes)) return rc;
  if (!loss || !logp || !kl || !grad) return net_fail(OMQ_NET_E_ARG, "%s: a null array", name);
  hipStream_t st = (hipStream_t)stream;
  if (p.in_rows) {
    launch_rows<true>(*r, row_weight, loss, logp, kl, nullptr, grad, st);
  } else {
    float* stats = reinterpret_cast<float*>(static_cast<char*>(workspace) + p.at_stats);
    launch_spans(*r, p, loss, logp, kl, stats, static_cast<char*>(workspace), st);
    launch_grad(*r, stats, row_weight, grad, st);
  }
  return net_status(name);
}

}  // extern "C"
