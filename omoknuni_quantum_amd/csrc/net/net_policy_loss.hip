// The clipped policy loss over legal actions with a KL term, and its gradient (gfx950).
//
// Per row, about a base m near the largest legal logit, with s = sum e^(z-m), tp = sum pi and
// tk = sum pi (log pi - (z - m)) over the legal actions (pi the target):
//   logq_a = z_a - m - log s
//   kl     = tk + tp log s
//   dz_a   = push p_a + slope [a taken] - kl_coef pi_a,   p_a = e^(z_a - m) / s,
// where slope is the loss's derivative by logp and push = kl_coef tp - slope.  The taken action is
// left out of s while it is formed (`rest`): 1 - p of the taken action, by which its slope is
// multiplied, is rest / s, and keeps its bits where p is near 1.
//
// Bound by memory, and for rows of a few hundred actions by the instructions of a row as well
// (32768 rows of 362 bfloat16 with target and mask 31 us, 3.4 TB/s).  Measured with gradient: 4096
// rows of 4672 36 us (4.7 TB/s), 4096 of 131072 without target 437 us (4.9 TB/s); without: 4096 of
// 4672 27 us (4.9 TB/s).  Three ways through a row:
//   - short rows are held in registers: the base, the sums and the gradient come from one load;
//   - a long row is read twice by its workgroup, for the sums and for the gradient, the second
//     time from the last-level cache (256 MB; the rows under way are 64 KB to 1 MB each);
//   - where the long rows are too few to occupy the chip they are cut into spans, a workgroup
//     each; their statistics are joined, and the gradient is an element-wise launch.
#include "net_logits.h"

namespace omq_net {
namespace {

// Statistics of a part of a row; m is -inf while nothing in it has weight; rest is s without the
// taken action.
struct Stats {
  float m, rest, tp, tk;
};

__device__ inline Stats no_stats() { return Stats{-kInf, 0.0f, 0.0f, 0.0f}; }

// The base that the sums of a part with base m were formed about.
__device__ inline float base_of(float m) { return m == -kInf ? 0.0f : m; }

// The statistics about another base, which is finite or that of a part without weight.
__device__ inline void rebase(Stats& t, float m) {
  if (t.m != m) {
    t.rest *= exp_fast(t.m - base_of(m));
    if (t.tp != 0.0f) t.tk -= t.tp * (base_of(t.m) - base_of(m));
    t.m = m;
  }
}

// Over the kLanes lanes of a group, of one base or of any: all get the joined statistics.
template <int kLanes, bool kTarget>
__device__ inline void lanes_sum(Stats& t) {
  t.rest = lanes_reduce<Sum, kLanes>(t.rest);
  if constexpr (kTarget) {
    t.tp = lanes_reduce<Sum, kLanes>(t.tp);
    t.tk = lanes_reduce<Sum, kLanes>(t.tk);
  }
}

template <int kLanes, bool kTarget>
__device__ inline void lanes_join(Stats& t) {
  rebase(t, lanes_reduce<Max, kLanes>(t.m));
  lanes_sum<kLanes, kTarget>(t);
}

// Over the kThreads threads of a row (as row_reduce), with one barrier.  kSame: the lanes of a
// wave have one base.
template <int kThreads, bool kTarget, bool kSame>
__device__ inline void row_join(Stats& t, Stats* smem) {
  if constexpr (!kSame)
    lanes_join<(kThreads < kWave ? kThreads : kWave), kTarget>(t);
  else
    lanes_sum<(kThreads < kWave ? kThreads : kWave), kTarget>(t);
  if constexpr (kThreads > kWave) {
    static_assert(kThreads <= 16 * kWave);
    const int lane = threadIdx.x & (kWave - 1);
    if (lane == 0) smem[threadIdx.x / kWave] = t;
    __syncthreads();
    const int w = lane & 15;
    t = w < kThreads / kWave ? smem[w] : no_stats();
    lanes_join<16, kTarget>(t);
  }
}

// What the gradient of a row needs.
struct RowGrad {
  float m, inv_s;  // p = e^(z - m) * inv_s; inv_s = 0: the row has no gradient
  float push, slope;
  float others;  // 1 - p of the taken action
  float mass;    // kl_coef tp
};

// Its place in the statistics that the loss leaves for its gradient: eight floats a row.
__device__ inline void write_stats(float4* stats, int64_t row, const RowGrad& g) {
  stats[2 * row] = make_float4(g.m, g.inv_s, g.push, g.slope);
  stats[2 * row + 1] = make_float4(g.others, g.mass, 0.0f, 0.0f);
}

__device__ inline RowGrad read_stats(const float4* stats, int64_t row) {
  const float4 a = stats[2 * row], b = stats[2 * row + 1];
  return RowGrad{a.x, a.y, a.z, a.w, b.x, b.y};
}

struct RowOut {
  float loss, logp, kl;
  RowGrad g;
};

// e^d - 1 and e^d - 1 - d, the latter without its cancellation about 0.
__device__ inline float exp_above_line(float d, float* above_one) {
  if (fabsf(d) > 0.5f) {
    *above_one = expm1f(d);
    return d == kInf ? kInf : *above_one - d;  // (not inf - inf)
  }
  float p = 1.0f / 40320.0f;  // Taylor; the next term is below 2^-24 of the sum
  p = fmaf(p, d, 1.0f / 5040.0f);
  p = fmaf(p, d, 1.0f / 720.0f);
  p = fmaf(p, d, 1.0f / 120.0f);
  p = fmaf(p, d, 1.0f / 24.0f);
  p = fmaf(p, d, 1.0f / 6.0f);
  p = d * d * fmaf(p, d, 0.5f);
  *above_one = p + d;
  return p;
}

// z_taken: the logit of the taken action, `taken`: it is legal and in range.  The differences of
// log-probabilities are formed in 64 bits: a few operations a row, and the ratio and the kl do not
// lose the bits that a log-probability of about -10 rounds away in float32.
__device__ inline RowOut finish_row(const omq_policy_rows& r, int64_t row, const Stats& t,
                                    float z_taken, bool taken) {
  RowOut o{};
  const float base = base_of(t.m);
  const float s = taken ? t.rest + exp_fast(z_taken - base) : t.rest;
  const bool live = !(t.m == -kInf && s == 0.0f);
  if (!live) return o;
  const double log_s = log_of_sum(s);
  float slope = 0.0f;
  if (taken) {
    const double logp = (double)z_taken - (double)base - log_s;
    o.logp = (float)logp;
    const float adv = r.advantages[row];
    const float ratio =
        __builtin_amdgcn_exp2f((float)((logp - (double)r.old_logp[row]) * 1.4426950408889634));
    const float one = ratio * adv;
    const float two = fminf(fmaxf(ratio, 1.0f - r.clip_low), 1.0f + r.clip_high) * adv;
    o.loss = -(one <= two || one != one ? one : two);
    if (one <= two || one != one) slope = -one;
    if (r.ref_logp) {
      const float d = (float)((double)r.ref_logp[row] - logp);
      float above_one;  // (not kl + d, which loses the bits of -1 where d is far below 0)
      o.kl = exp_above_line(d, &above_one);
      // (without a coefficient the kl is only watched: it may overflow)
      if (r.kl_coef != 0.0f) slope -= r.kl_coef * above_one;
    }
  }
  if (r.target) o.kl = (float)((double)t.tk + (t.tp != 0.0f ? (double)t.tp * log_s : 0.0));
  o.loss += r.kl_coef != 0.0f ? r.kl_coef * o.kl : 0.0f;
  o.g.m = base;
  o.g.inv_s = 1.0f / s;
  o.g.others = t.rest * o.g.inv_s;
  o.g.slope = slope;
  o.g.mass = r.kl_coef != 0.0f ? r.kl_coef * t.tp : 0.0f;
  o.g.push = o.g.mass - slope;
  // a row that adds nothing to the loss has no gradient, whatever its logits hold (padding; tp is
  // 0 without a target, and where nothing in it is positive)
  if (slope == 0.0f && o.g.push == 0.0f && (r.kl_coef == 0.0f || t.tp == 0.0f)) o.g.inv_s = 0.0f;
  return o;
}

__device__ inline void write_row(const RowOut& o, int64_t row, float* loss, float* logp, float* kl,
                                 float4* stats) {
  loss[row] = o.loss;
  logp[row] = o.logp;
  kl[row] = o.kl;
  if (stats) write_stats(stats, row, o.g);
}

// A row's action as it is given.  (Loaded before the row's blocks: loads are waited for in their
// order.)
__device__ inline int64_t action_of(const omq_policy_rows& r, int64_t row) {
  return r.taken_are_64 ? static_cast<const int64_t*>(r.taken)[row]
                        : (int64_t) static_cast<const int32_t*>(r.taken)[row];
}

// The taken action of a row, -1 when it is out of range or not legal, and its logit.
template <class T>
__device__ inline int taken_of(const omq_policy_rows& r, int64_t row, int64_t a, float* z) {
  *z = 0.0f;
  if (a < 0 || a >= r.actions || (r.legal && !r.legal[row * r.legal_stride + a])) return -1;
  *z = (float)static_cast<const T*>(r.logits)[row * r.logits_stride + a];
  return (int)a;
}

template <class T>
__device__ inline RowIn<T> row_in(const omq_policy_rows& r, int64_t row) {
  return {static_cast<const T*>(r.logits) + row * r.logits_stride,
          r.legal + (r.legal ? row * r.legal_stride : 0),
          r.target + (r.target ? row * r.target_stride : 0), (int)r.actions};
}

// The target, 0 where it is not legal.
template <class T, bool kWhole>
__device__ inline F8 legal_target(const Block<T, true>& b, const RowIn<T>& in, int col,
                                  uint64_t ok) {
  F8 pi = to_front<float, kWhole>(b.pi, col, in.cols);
#pragma unroll
  for (int j = 0; j < 8; ++j) pi[j] = masked(pi[j], ok_mask(ok, j), 0.0f);
  return pi;
}

// Takes the taken action, where it is in the block (at its place `at`), out of the block's sum.
__device__ inline void leave_out(F8& z, int at) {
  if ((uint32_t)at < 8u) {
#pragma unroll
    for (int j = 0; j < 8; ++j) z[j] = j == at ? -kInf : z[j];
  }
}

// Adds a block's exponentials, which take the place of its logits.
__device__ inline void add_logits(Stats& t, F8& z, float base) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    z[j] = exp_fast(z[j] - base);
    t.rest += z[j];
  }
}

// Adds a block's targets, about the same base, and leaves 0 in place of those that are not
// positive.  (The logarithm takes subnormals for 0: what they add is nothing beside the rest.  The
// legacy product is 0 where a factor is 0: the logit of a target of 0 may be -inf.)
__device__ inline void add_target(Stats& t, F8& pi, F8 z, float base) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    pi[j] = larger(pi[j], 0.0f);
    const float log_pi = __builtin_amdgcn_logf(larger(pi[j], 0x1p-126f));  // (base 2)
    float term;
    asm("v_mul_legacy_f32 %0, %1, %2"
        : "=v"(term)
        : "v"(pi[j]), "v"(fmaf(log_pi, kLn2, base - z[j])));
    t.tk += term;
    t.tp += pi[j];
  }
}

// The gradient of eight actions but for the slope of the taken one, times the row's weight w: e
// holds e^(z - m), scale is w * push / s (or that about the base of e).
template <bool kTarget, bool kAll>
__device__ inline F8 gradient(F8 e, F8 pi, uint64_t ok, float scale, float w_coef) {
  F8 d = e * scale;
  if constexpr (kTarget) {
    // (fmaf where a product and a sum could be contracted one way here and another there: the
    // gradient has the same bits whichever kernel forms it from the same statistics, but for rows
    // in the registers of several waves, whose exponentials are about each wave's own base)
#pragma unroll
    for (int j = 0; j < 8; ++j) d[j] = fmaf(-pi[j], w_coef, d[j]);
  }
  if constexpr (!kAll) {
#pragma unroll
    for (int j = 0; j < 8; ++j) d[j] = masked(d[j], ok_mask(ok, j), 0.0f);
  }
  return d;
}

// The element of the taken action, in full; written by the thread that wrote its block, after it.
// kl_coef tp p + slope (1 - p), not push p + slope, which cancels where p is near 1 and is NaN where
// the slope overflows.
template <class T>
__device__ inline void put_taken(T* grad, const RowIn<T>& in, const RowGrad& g, float z_taken,
                                 int taken, float coef, float w) {
  float d = fmaf(g.mass, exp_fast(z_taken - g.m) * g.inv_s, g.slope * g.others);
  if (in.target) d = fmaf(-larger(in.target[taken], 0.0f), coef, d);
  grad[taken] = (T)(w * d);
}

// ---- rows in registers ----------------------------------------------------------------------
template <int kThreads>
constexpr int block_of() {
  return kThreads <= kWave ? 256 : kThreads;
}

template <class T, int kThreads, int kVecs, bool kTarget, bool kWhole>
__global__ __launch_bounds__(block_of<kThreads>()) void loss_rows_kernel(
    omq_policy_rows r, const float* __restrict__ row_weight, float* __restrict__ loss,
    float* __restrict__ logp, float* __restrict__ kl, float4* __restrict__ stats,
    T* __restrict__ grad) {
  constexpr int kRows = block_of<kThreads>() / kThreads;
  __shared__ Stats smem[16];
  const int lane = threadIdx.x % kThreads;
  const int64_t row = block_index() * kRows + row_slot<kThreads>();
  if (row >= r.rows) return;
  const RowIn<T> in = row_in<T>(r, row);
  const int64_t action = action_of(r, row);
  Block<T, kTarget> b[kVecs];
#pragma unroll
  for (int i = 0; i < kVecs; ++i)
    b[i] = load_block<T, kTarget, kWhole>(in, 8 * (lane + i * kThreads));
  float z_taken;
  const int taken = taken_of<T>(r, row, action, &z_taken);
  F8 z[kVecs], pi[kTarget ? kVecs : 1];
  uint64_t ok[kVecs];
  Stats t = no_stats();
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    const int col = 8 * (lane + i * kThreads);
    ok[i] = ok_bytes<T, kTarget, kWhole>(b[i], in, col);
    z[i] = legal_logits<T, kTarget, kWhole>(b[i], in, col, ok[i]);
    t.m = larger(t.m, largest(z[i]));
  }
  t.m = lanes_reduce<Max, (kThreads < kWave ? kThreads : kWave)>(t.m);
  const float m = t.m, base = base_of(m);  // (of this wave)
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    if constexpr (kTarget) {
      pi[i] = legal_target<T, kWhole>(b[i], in, 8 * (lane + i * kThreads), ok[i]);
      add_target(t, pi[i], z[i], base);
    }
    leave_out(z[i], taken - 8 * (lane + i * kThreads));
    add_logits(t, z[i], base);
  }
  row_join<kThreads, kTarget, true>(t, smem);
  const RowOut o = finish_row(r, row, t, z_taken, taken >= 0);
  if (lane == 0) write_row(o, row, loss, logp, kl, stats);
  if (!grad) return;
  const float w = row_weight ? row_weight[row] : 1.0f;
  // From the wave's base to the row's: 0 where the wave has no weight.  (Its base is 0 then, which
  // may lie any distance above the row's.)
  const float scale = w * o.g.push * o.g.inv_s * exp_fast(m - o.g.m);
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    const int col = 8 * (lane + i * kThreads);
    F8 d = {};
    if (o.g.inv_s != 0.0f)
      d = gradient<kTarget, false>(z[i], pi[kTarget ? i : 0], ok[i], scale, w * r.kl_coef);
    store8<T, kWhole>(grad + row * in.cols, col, in.cols, d);
  }
  if (taken >= 0 && o.g.inv_s != 0.0f && lane == (taken / 8) % kThreads)
    put_taken(grad + row * in.cols, in, o.g, z_taken, taken, r.kl_coef, w);
}

// ---- long rows ------------------------------------------------------------------------------
// Blocks that a thread has in flight: four of rows that are whole blocks (4096 rows of 131072
// bfloat16 with gradient: 437 us, 453 with one; 2000 of 65536 float32: 231 and 267 us; but 1024 of
// 20000 bfloat16: 24 and 17 us), else one (4096 of 100003: 402 us, 482 with four; 2018 of 87390
// float32: 308 and 351 us: blocks at odd addresses take two lines each).
template <bool kTarget, bool kWhole>
constexpr int kInFlight = kWhole && !kTarget ? 4 : 1;

// kAll: the blocks are whole and every action is legal, so that nothing is masked.  Long rows
// without a mask are made of such blocks but for their end.  (4096 rows of 131072 bfloat16 with
// gradient: the masks are a third of the instructions and 7 of 444 us.)
template <class T, bool kTarget, bool kWhole, bool kAll>
__device__ inline F8 logits_of(const Block<T, kTarget>& b, const RowIn<T>& in, int col,
                               uint64_t ok) {
  if constexpr (kAll) return __builtin_convertvector(b.z, F8);
  return legal_logits<T, kTarget, kWhole>(b, in, col, ok);
}

template <class T, bool kWhole, bool kAll>
__device__ inline F8 target_of(const Block<T, true>& b, const RowIn<T>& in, int col, uint64_t ok) {
  if constexpr (kAll) return b.pi;
  return legal_target<T, kWhole>(b, in, col, ok);
}

// Adds a thread's kCount blocks, kStep columns apart, of the columns from `at` on to its
// statistics.  The base follows the logits only when one passes it by more than kSlack: e^kSlack
// is far from any limit, and after a few blocks no thread changes its base again.
template <class T, bool kTarget, bool kWhole, bool kAll, int kCount, int kStep>
__device__ inline void add_blocks(Stats& t, const RowIn<T>& in, int at, int to, int taken) {
  constexpr float kSlack = 8.0f;
  const int col = at + 8 * (int)threadIdx.x;
  Block<T, kTarget> b[kCount];
#pragma unroll
  for (int u = 0; u < kCount; ++u)
    b[u] = load_block<T, kTarget, kWhole || kAll>(in, col + kStep * u);
  F8 z[kCount];
  uint64_t ok[kCount];
  float m = -kInf;
#pragma unroll
  for (int u = 0; u < kCount; ++u) {
    const int c = col + kStep * u;
    ok[u] = kAll ? 0 : c < to ? ok_bytes<T, kTarget, kWhole>(b[u], in, c) : 0;
    z[u] = logits_of<T, kTarget, kWhole, kAll>(b[u], in, c, ok[u]);
    m = larger(m, largest(z[u]));
  }
  if (m > t.m + kSlack) rebase(t, m);  // (from -inf: at the first weight)
  const float base = base_of(t.m);
  const bool takes = taken >= at && taken < at + kStep * kCount;  // (uniform)
#pragma unroll
  for (int u = 0; u < kCount; ++u) {
    if constexpr (kTarget) {
      F8 pi = target_of<T, kWhole, kAll>(b[u], in, col + kStep * u, ok[u]);
      add_target(t, pi, z[u], base);
    }
    if (takes) leave_out(z[u], taken - (col + kStep * u));
    add_logits(t, z[u], base);
  }
}

// Statistics of the columns from `from` on, up to `to`, that fall to this thread.
template <class T, bool kTarget, bool kWhole, int kThreads>
__device__ inline void stream(Stats& t, const RowIn<T>& in, int from, int to, int taken) {
  constexpr int kCount = kInFlight<kTarget, kWhole>, kStep = 8 * kThreads;
  constexpr int kChunk = kStep * kCount;
  int at = from;
  if (!in.legal)
    for (; at + kChunk <= to; at += kChunk)
      add_blocks<T, kTarget, kWhole, true, kCount, kStep>(t, in, at, to, taken);
  for (; at < to; at += kChunk)
    add_blocks<T, kTarget, kWhole, false, kCount, kStep>(t, in, at, to, taken);
}

// The gradient of the block at column col.
template <class T, bool kTarget, bool kWhole, bool kAll, bool kStream>
__device__ inline void put_gradient(T* grad, const Block<T, kTarget>& b, const RowIn<T>& in,
                                    int col, const RowGrad& g, float coef, float w) {
  F8 d = {}, pi = {};
  if (g.inv_s != 0.0f) {
    const uint64_t ok = kAll ? 0 : ok_bytes<T, kTarget, kWhole>(b, in, col);
    F8 z = logits_of<T, kTarget, kWhole, kAll>(b, in, col, ok);
    if constexpr (kTarget) {
      pi = target_of<T, kWhole, kAll>(b, in, col, ok);
#pragma unroll
      for (int j = 0; j < 8; ++j) pi[j] = larger(pi[j], 0.0f);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) z[j] = exp_fast(z[j] - g.m);
    d = gradient<kTarget, kAll>(z, pi, ok, w * g.push * g.inv_s, w * coef);
  }
  store8<T, kWhole || kAll, kStream>(grad, col, in.cols, d);
}

// The gradients of a thread's kCount blocks of the columns from `at` on.
template <class T, bool kTarget, bool kWhole, bool kAll, int kCount, int kStep>
__device__ inline void put_blocks(T* grad, const RowIn<T>& in, int at, const RowGrad& g, float coef,
                                  float w) {
  const int col = at + 8 * (int)threadIdx.x;
  Block<T, kTarget> b[kCount];
#pragma unroll
  for (int u = 0; u < kCount; ++u)
    b[u] = load_block<T, kTarget, kWhole || kAll>(in, col + kStep * u);
#pragma unroll
  for (int u = 0; u < kCount; ++u)
    put_gradient<T, kTarget, kWhole, kAll, true>(grad, b[u], in, col + kStep * u, g, coef, w);
}

// A workgroup a row: the sums, then the gradient, for which the blocks are read again, the last
// read first.
template <class T, int kThreads, bool kTarget, bool kWhole>
__global__ __launch_bounds__(kThreads) void loss_long_kernel(
    omq_policy_rows r, const float* __restrict__ row_weight, float* __restrict__ loss,
    float* __restrict__ logp, float* __restrict__ kl, float4* __restrict__ stats,
    T* __restrict__ grad) {
  constexpr int kCount = kInFlight<kTarget, kWhole>, kStep = 8 * kThreads;
  constexpr int kChunk = kStep * kCount;
  __shared__ Stats smem[16];
  const int64_t row = block_index();
  if (row >= r.rows) return;
  const RowIn<T> in = row_in<T>(r, row);
  float z_taken;
  const int taken = taken_of<T>(r, row, action_of(r, row), &z_taken);
  Stats t = no_stats();
  stream<T, kTarget, kWhole, kThreads>(t, in, 0, in.cols, taken);
  row_join<kThreads, kTarget, false>(t, smem);
  const RowOut o = finish_row(r, row, t, z_taken, taken >= 0);
  if (threadIdx.x == 0) write_row(o, row, loss, logp, kl, stats);
  if (!grad) return;
  const float w = row_weight ? row_weight[row] : 1.0f;
  T* g = grad + row * in.cols;
  const int whole = in.legal ? 0 : in.cols / kChunk * kChunk;  // (of blocks that kAll is true of)
  int at = (in.cols - 1) / kChunk * kChunk;
  for (; at >= whole; at -= kChunk)
    put_blocks<T, kTarget, kWhole, false, kCount, kStep>(g, in, at, o.g, r.kl_coef, w);
  for (; at >= 0; at -= kChunk)
    put_blocks<T, kTarget, kWhole, true, kCount, kStep>(g, in, at, o.g, r.kl_coef, w);
  if (taken >= 0 && o.g.inv_s != 0.0f && (int)threadIdx.x == (taken / 8) % kThreads)
    put_taken(g, in, o.g, z_taken, taken, r.kl_coef, w);
}

// Statistics of span blockIdx.x of row blockIdx.y.
template <class T, bool kTarget, bool kWhole>
__global__ __launch_bounds__(256) void loss_span_kernel(omq_policy_rows r, int span,
                                                        Stats* __restrict__ parts) {
  __shared__ Stats smem[16];
  const int64_t row = blockIdx.y;
  const RowIn<T> in = row_in<T>(r, row);
  const int64_t from = (int64_t)blockIdx.x * span;
  const int to = from + span < in.cols ? (int)(from + span) : in.cols;
  float z_taken;
  const int taken = taken_of<T>(r, row, action_of(r, row), &z_taken);
  Stats t = no_stats();
  stream<T, kTarget, kWhole, 256>(t, in, (int)from, to, taken);
  row_join<256, kTarget, false>(t, smem);
  if (threadIdx.x == 0) parts[row * gridDim.x + blockIdx.x] = t;
}

// A wave a row: its spans joined.
template <class T>
__global__ __launch_bounds__(64) void loss_join_kernel(omq_policy_rows r,
                                                       const Stats* __restrict__ parts, int spans,
                                                       float* __restrict__ loss,
                                                       float* __restrict__ logp,
                                                       float* __restrict__ kl,
                                                       float4* __restrict__ stats) {
  const int64_t row = blockIdx.x;
  float z;
  const int taken = taken_of<T>(r, row, action_of(r, row), &z);
  Stats t = no_stats();
  for (int k = threadIdx.x; k < spans; k += kWave) {
    Stats u = parts[row * spans + k];
    const float m = fmaxf(t.m, u.m);
    rebase(t, m);
    rebase(u, m);
    t = Stats{m, t.rest + u.rest, t.tp + u.tp, t.tk + u.tk};
  }
  lanes_join<kWave, true>(t);
  if (threadIdx.x == 0) write_row(finish_row(r, row, t, z, taken >= 0), row, loss, logp, kl, stats);
}

// The gradient from the rows' statistics, a block of eight actions a thread.
template <class T, bool kTarget, bool kWhole>
__global__ __launch_bounds__(256) void loss_grad_kernel(omq_policy_rows r, int blocks,
                                                        const float4* __restrict__ stats,
                                                        const float* __restrict__ row_weight,
                                                        T* __restrict__ grad) {
  const int64_t first = block_index() * 256;
  const int64_t row0 = first / blocks;
  const uint32_t at = (uint32_t)(first - row0 * blocks) + threadIdx.x;
  const int64_t row = row0 + at / (uint32_t)blocks;
  const int col = 8 * (int)(at % (uint32_t)blocks);
  if (row >= r.rows) return;
  const RowIn<T> in = row_in<T>(r, row);
  const Block<T, kTarget> b = load_block<T, kTarget, kWhole>(in, col);
  const RowGrad g = read_stats(stats, row);
  const float w = row_weight ? row_weight[row] : 1.0f;
  float z_taken;
  const int taken = taken_of<T>(r, row, action_of(r, row), &z_taken);
  T* to = grad + row * in.cols;
  put_gradient<T, kTarget, kWhole, false, false>(to, b, in, col, g, r.kl_coef, w);
  if (taken >= 0 && g.inv_s != 0.0f && taken / 8 == col / 8)
    put_taken(to, in, g, z_taken, taken, r.kl_coef, w);
}

// ---- launches -------------------------------------------------------------------------------
template <int kThreads_, int kVecs_>
struct Layout {
  static constexpr int kThreads = kThreads_, kVecs = kVecs_;
};

// The longest rows that are held in registers, without and with a target.
constexpr int64_t kRowActions = 16384, kRowActionsTarget = 8192;
// Longer rows are a workgroup each, unless they are fewer than kLongRows and longer than
// kWideActions: those are cut into spans (with their gradients, in bfloat16: 8 rows of 131072 take
// 12 us so and 21 us with a workgroup each; 16 rows of 20000 take 7 us with a workgroup each and
// 13 us cut; 128 rows of 131072 the same).
constexpr int64_t kLongRows = 128, kWideActions = 65536;
// A workgroup of 1024 threads for rows over kWideActions, so that the rows under way stay in the
// last-level cache (4096 rows of 131072 bfloat16: 437 us, 447 with 512 threads), and where there
// are fewer rows than compute units (128 rows of 65536: 12 us, 13 with 512); else 512 (4096 rows of
// 32768: 103 us, 128 with 1024).
bool wide_row(int64_t rows, int64_t actions) { return actions > kWideActions || rows < 256; }

template <bool kTarget, class F>
void with_layout(int64_t cols, F&& f) {
  if (cols <= 128) return f(Layout<16, 1>{});
  if (cols <= 256) return f(Layout<32, 1>{});
  if (cols <= 512) return f(Layout<64, 1>{});
  if (cols <= 1024) return f(Layout<128, 1>{});
  if (cols <= 2048) return f(Layout<256, 1>{});
  if (cols <= 4096) return f(Layout<256, 2>{});
  if (cols <= 6144) return f(Layout<256, 3>{});
  if constexpr (kTarget) {
    return f(Layout<256, 4>{});
  } else {
    if (cols <= 8192) return f(Layout<256, 4>{});
    return f(Layout<256, 8>{});
  }
}

template <class F>
void with_type(int dtype, F&& f) {
  if (dtype == OMQ_NET_F32) return f(float{});
  if (dtype == OMQ_NET_BF16) return f(bf16{});
  return f(f16{});
}

template <bool kTarget, bool kWhole>
struct Kind {
  static constexpr bool target = kTarget, whole = kWhole;
};

template <class F>
void with_kind(const omq_policy_rows& r, F&& f) {
  if (r.target)
    r.actions % 8 == 0 ? f(Kind<true, true>{}) : f(Kind<true, false>{});
  else
    r.actions % 8 == 0 ? f(Kind<false, true>{}) : f(Kind<false, false>{});
}

// How rows are cut into spans, where they are.
struct SpanPlan {
  int64_t span, spans, at_parts, bytes;
};

SpanPlan span_plan(int64_t rows, int64_t actions) {
  SpanPlan p{};
  if (rows >= kLongRows || actions <= kWideActions) return p;
  // spans for about 1024 workgroups, of at least 4096 columns
  int64_t spans = ceil_div(1024, rows > 0 ? rows : 1);
  const int64_t most = ceil_div(actions, 4096);
  spans = spans > most ? most : spans;
  p.span = ceil_div(ceil_div(actions, spans), 8) * 8;
  p.spans = ceil_div(actions, p.span);
  p.at_parts = 32 * rows;  // (the rows' statistics for the gradient come first)
  p.bytes = p.at_parts + (int64_t)sizeof(Stats) * rows * p.spans;
  return p;
}

enum Way { kInRows, kLong, kSpans };

Way way_of(const omq_policy_rows& r) {
  if (r.actions <= (r.target ? kRowActionsTarget : kRowActions)) return kInRows;
  return r.rows >= kLongRows || r.actions <= kWideActions ? kLong : kSpans;
}

bool loss_sizes_ok(int64_t rows, int64_t actions) {
  return rows >= 0 && actions >= 1 && rows <= OMQ_NET_MAX_COUNT &&
         actions <= OMQ_NET_MAX_ACTIONS &&
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

struct LossOut {
  float *loss, *logp, *kl, *stats;
};

void launch_rows(const omq_policy_rows& r, const float* row_weight, const LossOut& o, void* grad,
                 hipStream_t st) {
  with_type(r.dtype, [&](auto t) {
    using T = decltype(t);
    with_kind(r, [&](auto kind) {
      using K = decltype(kind);
      with_layout<K::target>(r.actions, [&](auto l) {
        using L = decltype(l);
        constexpr int kBlock = block_of<L::kThreads>();
        const dim3 grid = grid_of(ceil_div(r.rows, kBlock / L::kThreads), kBlock);
        loss_rows_kernel<T, L::kThreads, L::kVecs, K::target, K::whole><<<grid, kBlock, 0, st>>>(
            r, row_weight, o.loss, o.logp, o.kl, reinterpret_cast<float4*>(o.stats),
            static_cast<T*>(grad));
      });
    });
  });
}

void launch_long(const omq_policy_rows& r, const float* row_weight, const LossOut& o, void* grad,
                 hipStream_t st) {
  with_type(r.dtype, [&](auto t) {
    using T = decltype(t);
    with_kind(r, [&](auto kind) {
      using K = decltype(kind);
      const bool wide = wide_row(r.rows, r.actions);
      const auto kernel = wide ? loss_long_kernel<T, 1024, K::target, K::whole>
                               : loss_long_kernel<T, 512, K::target, K::whole>;
      const int threads = wide ? 1024 : 512;
      kernel<<<grid_of(r.rows, threads), threads, 0, st>>>(
          r, row_weight, o.loss, o.logp, o.kl, reinterpret_cast<float4*>(o.stats),
          static_cast<T*>(grad));
    });
  });
}

void launch_spans(const omq_policy_rows& r, const SpanPlan& p, const LossOut& o, char* ws,
                  hipStream_t st) {
  Stats* parts = reinterpret_cast<Stats*>(ws + p.at_parts);
  with_type(r.dtype, [&](auto t) {
    using T = decltype(t);
    with_kind(r, [&](auto kind) {
      using K = decltype(kind);
      loss_span_kernel<T, K::target, K::whole>
          <<<dim3((uint32_t)p.spans, (uint32_t)r.rows), 256, 0, st>>>(r, (int)p.span, parts);
    });
    loss_join_kernel<T><<<(uint32_t)r.rows, kWave, 0, st>>>(
        r, parts, (int)p.spans, o.loss, o.logp, o.kl, reinterpret_cast<float4*>(o.stats));
  });
}

void launch_grad(const omq_policy_rows& r, const float* stats, const float* row_weight, void* grad,
                 hipStream_t st) {
  with_type(r.dtype, [&](auto t) {
    using T = decltype(t);
    with_kind(r, [&](auto kind) {
      using K = decltype(kind);
      const int blocks = (int)ceil_div(r.actions, 8);
      const dim3 grid = grid_of(ceil_div(r.rows * blocks, 256), 256);
      loss_grad_kernel<T, K::target, K::whole><<<grid, 256, 0, st>>>(
          r, blocks, reinterpret_cast<const float4*>(stats), row_weight, static_cast<T*>(grad));
    });
  });
}

int check_workspace(const char* name, const SpanPlan& p, const void* ws, int64_t bytes) {
  if (p.bytes > 0 && (!ws || bytes < p.bytes))
    return net_fail(OMQ_NET_E_ARG, "%s: workspace of %lld bytes, %lld needed", name,
                    (long long)bytes, (long long)p.bytes);
  if (p.bytes > 0 && !on_16_bytes(ws))
    return net_fail(OMQ_NET_E_ARG, "%s: workspace is not on a 16-byte boundary", name);
  return OMQ_NET_OK;
}

}  // namespace
}  // namespace omq_net

using namespace omq_net;

extern "C" {

int64_t omq_clipped_policy_loss_workspace(int64_t rows, int64_t actions) {
  if (!loss_sizes_ok(rows, actions)) return OMQ_NET_E_ARG;
  return span_plan(rows, actions).bytes;
}

int omq_clipped_policy_loss(const omq_policy_rows* r, float* loss, float* logp, float* kl,
                            float* stats, void* workspace, int64_t workspace_bytes,
                            void* stream) {
  const char* name = "omq_clipped_policy_loss";
  if (int rc = check_rows(name, r)) return rc;
  if (r->rows == 0) return OMQ_NET_OK;
  const SpanPlan p = span_plan(r->rows, r->actions);
  if (int rc = check_workspace(name, p, workspace, workspace_bytes)) return rc;
  if (!loss || !logp || !kl) return net_fail(OMQ_NET_E_ARG, "%s: a null array", name);
  if (!on_16_bytes(stats))
    return net_fail(OMQ_NET_E_ARG, "%s: stats is not on a 16-byte boundary", name);
  hipStream_t st = (hipStream_t)stream;
  const LossOut o{loss, logp, kl, stats};
  switch (way_of(*r)) {
    case kInRows: launch_rows(*r, nullptr, o, nullptr, st); break;
    case kLong: launch_long(*r, nullptr, o, nullptr, st); break;
    case kSpans: launch_spans(*r, p, o, static_cast<char*>(workspace), st); break;
  }
  return net_status(name);
}

int omq_clipped_policy_loss_grad(const omq_policy_rows* r, const float* stats,
                                 const float* row_weight, void* grad, void* stream) {
  const char* name = "omq_clipped_policy_loss_grad";
  if (int rc = check_rows(name, r)) return rc;
  if (r->rows == 0) return OMQ_NET_OK;
  if (!stats || !grad) return net_fail(OMQ_NET_E_ARG, "%s: a null array", name);
  if (!on_16_bytes(stats))
    return net_fail(OMQ_NET_E_ARG, "%s: stats is not on a 16-byte boundary", name);
  launch_grad(*r, stats, row_weight, grad, (hipStream_t)stream);
  return net_status(name);
}

int omq_clipped_policy_loss_with_grad(const omq_policy_rows* r, const float* row_weight,
                                      float* loss, float* logp, float* kl, void* grad,
                                      void* workspace, int64_t workspace_bytes, void* stream) {
  const char* name = "omq_clipped_policy_loss_with_grad";
  if (int rc = check_rows(name, r)) return rc;
  if (r->rows == 0) return OMQ_NET_OK;
  const SpanPlan p = span_plan(r->rows, r->actions);
  if (int rc = check_workspace(name, p, workspace, workspace_bytes)) return rc;
  if (!loss || !logp || !kl || !grad) return net_fail(OMQ_NET_E_ARG, "%s: a null array", name);
  hipStream_t st = (hipStream_t)stream;
  LossOut o{loss, logp, kl, nullptr};
  switch (way_of(*r)) {
    case kInRows: launch_rows(*r, row_weight, o, grad, st); break;
    case kLong: launch_long(*r, row_weight, o, grad, st); break;
    case kSpans:
      o.stats = static_cast<float*>(workspace);
      launch_spans(*r, p, o, static_cast<char*>(workspace), st);
      launch_grad(*r, o.stats, row_weight, grad, st);
      break;
  }
  return net_status(name);
}

}  // extern "C"
