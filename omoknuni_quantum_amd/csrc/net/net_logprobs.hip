// The log-probabilities of given tokens over the legal ones, with the entropy and the best
// alternatives, and their gradient (gfx950).
//
// Per row, about a base m at the largest legal logit, with x = z - m, rest = sum e^x and
// xe = sum e^x x over the legal tokens but the given one, t, and s = rest + e^(x_t):
//   logp    = x_t - log s
//   entropy = log s - (xe + e^(x_t) x_t) / s
//   dz_j    = a ([j = t] - p_j) - b p_j (log p_j + entropy),   p_j = e^(x_j) / s,
// for weights a of logp and b of the entropy.  The given token is left out of `rest`, so that its
// 1 - p, which is rest / s, keeps its bits where p is near 1.
//
// The best alternatives come without a sort of the row.  Every thread knows its largest logit; the
// threads form 64 groups, and the top-th largest of the groups' largest is a bound that at least
// `top` logits reach and few others do.  Only threads whose largest reaches it look at their
// logits again; the candidates (a logit and an index in 64 bits, no two alike) are ranked by
// counting.  Where more candidates tie than the list holds, they are found one after another.
//
// Bound by memory and, with a gradient, as much by instructions: a row of up to 16384 tokens is held
// in registers (8192 rows of 4672, bf16, mask and gradient: 43 us, 4.4 TB/s, 40 where the inputs
// repeat); a longer one is read by a workgroup, its alternatives from the few threads that hold them,
// and a second time for the gradient (2048 rows of 131072, bf16: 102 us, 5.3 TB/s, and 13 for 8
// alternatives; 301 with the gradient).  Under autograd the forward pass leaves a row's statistics,
// and the gradient is a launch that reads the logits again: 29 + 39 us of the former rows, 102 + 191
// of the latter.
#include <type_traits>

#include "net_logits.h"

namespace omq_net {
namespace {

struct LogprobArgs {
  omq_logprob_rows r;
  const float *logp_weight, *entropy_weight;
  float *logp, *entropy, *top_logp;
  int64_t* top_tokens;
  float4* stats;
  void* grad;
  int top;
};

// Sums of a part of a row about its largest logit m; m is -inf while nothing in it has weight.  An
// exponential is 2^y, y = z log2 e - exponent_of(m), a product and a difference rounded once: what
// the exponent of m was rounded by cancels however large the logits are.  xe is the sum of 2^y y.
struct Sums {
  float m, rest, xe;
};

__device__ inline Sums no_sums() { return Sums{-kInf, 0.0f, 0.0f}; }

__device__ inline float base_of(float m) { return m == -kInf ? 0.0f : m; }

// m log2 e, rounded to float32 as long as that holds it.
__device__ inline double exponent_of(float m) {
  return fabsf(m) < 0x1p126f ? (double)(m * kLog2e) : (double)m * (double)kLog2e;
}

// y of a logit, and of a part's m about another one's.
__device__ inline float y_of(float z, float m) {
  return fabsf(m) < 0x1p126f ? fmaf(z, kLog2e, -(m * kLog2e)) : (z - m) * kLog2e;
}

__device__ inline float y_between(float from, float to) {
  return from == -kInf ? -kInf : (float)(exponent_of(from) - exponent_of(to));
}

// About another base, which is finite or that of a part without weight.
__device__ inline void rebase(Sums& t, float m) {
  if (t.m != m) {
    const float d = y_between(t.m, base_of(m)), scale = __builtin_amdgcn_exp2f(d);
    t.rest *= scale;
    t.xe = scale != 0.0f ? fmaf(d, t.rest, scale * t.xe) : t.rest;  // (0, or NaN; d may be -inf)
    t.m = m;
  }
}

template <int kLanes>
__device__ inline void lanes_join(Sums& t) {
  rebase(t, lanes_reduce<Max, kLanes>(t.m));
  t.rest = lanes_reduce<Sum, kLanes>(t.rest);
  t.xe = lanes_reduce<Sum, kLanes>(t.xe);
}

// Over the kThreads threads of a row; every thread gets the row's sums.
template <int kThreads>
__device__ inline void row_join(Sums& t, Sums* smem) {
  lanes_join<kWave>(t);
  if constexpr (kThreads > kWave) {
    const int lane = threadIdx.x & (kWave - 1);
    if (lane == 0) smem[threadIdx.x / kWave] = t;
    __syncthreads();
    const int w = lane & 15;
    t = w < kThreads / kWave ? smem[w] : no_sums();
    lanes_join<16>(t);
  }
}

// The largest number of a block, or -inf.
__device__ inline float largest_number(const F8& z) {
  float m = larger(-kInf, largest(z));
  if (m != m) {  // (a signalling NaN)
    m = -kInf;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = z[j] > m ? z[j] : m;
  }
  return m;
}

// Adds a block of logits about a base; `at`: the given token's place in it, if it is there.  y and
// e: a logit's y, no less than -2^100, for which the products with e = 0 are 0, and 2^y.
__device__ inline void exponentials(const F8& z, float base, F8& y, F8& e) {
  if (fabsf(base) < 0x1p126f) {
    const float exponent = base * kLog2e;
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = fmaf(z[j], kLog2e, -exponent);
  } else {
    y = (z - base) * kLog2e;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    e[j] = __builtin_amdgcn_exp2f(y[j]);  // (a NaN is kept here)
    y[j] = larger(y[j], -0x1p100f);
  }
}

__device__ inline void add_block(Sums& t, const F8& z, float base, int at, F8& y, F8& e) {
  exponentials(z, base, y, e);
  F8 added = e;
  if ((uint32_t)at < 8u) {
#pragma unroll
    for (int j = 0; j < 8; ++j) added[j] = j == at ? 0.0f : e[j];
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    t.rest += added[j];
    t.xe = fmaf(added[j], y[j], t.xe);
  }
}

// What a row's gradient and its alternatives need.
struct RowEnd {
  float base, inv_s, log_s, entropy, others;
  double log_s64;
  float logp;
  bool live;
};

// log p of a legal logit.
__device__ inline double logp_of(const RowEnd& o, float z) {
  return ((double)z * (double)kLog2e - exponent_of(o.base)) * 0.6931471805599453 - o.log_s64;
}

__device__ inline RowEnd finish_row(const Sums& t, float z_token, bool given) {
  RowEnd o{};
  o.base = base_of(t.m);
  const float y = given ? y_of(z_token, o.base) : 0.0f;
  const float e = given ? __builtin_amdgcn_exp2f(y) : 0.0f;
  const float s = t.rest + e;
  o.live = !(t.m == -kInf && s == 0.0f);
  if (!o.live) return o;
  o.log_s64 = log_of_sum(s);
  o.log_s = (float)o.log_s64;
  o.inv_s = 1.0f / s;
  o.others = t.rest * o.inv_s;
  const float xe = e != 0.0f ? fmaf(e, y, t.xe) : t.xe;
  o.entropy = (float)(o.log_s64 - (double)xe * (double)o.inv_s * 0.6931471805599453);
  if (given) o.logp = (float)logp_of(o, z_token);
  return o;
}

template <class T>
__device__ inline RowIn<T> row_in(const omq_logprob_rows& r, int64_t row) {
  return {static_cast<const T*>(r.logits) + row * r.logits_stride,
          r.legal + (r.legal ? row * r.legal_stride : 0), nullptr, (int)r.vocab};
}

// The given token of a row, -1 when it is out of range or not legal, and its logit.
template <class T>
__device__ inline int token_of(const omq_logprob_rows& r, int64_t row, float* z) {
  const int64_t a = r.tokens_are_64 ? static_cast<const int64_t*>(r.tokens)[row]
                                    : (int64_t) static_cast<const int32_t*>(r.tokens)[row];
  *z = 0.0f;
  if (a < 0 || a >= r.vocab || (r.legal && !r.legal[row * r.legal_stride + a])) return -1;
  *z = (float)static_cast<const T*>(r.logits)[row * r.logits_stride + a];
  return (int)a;
}

// A row's gradient from its y and e about another base: but for the given token's it is
// -p (a + b (log p + entropy)), p = e inv.
struct RowSlope {
  float inv, shift, slope;  // the bracket is slope * y + shift
};

__device__ inline RowSlope slope_of(const RowEnd& o, float base, float a, float b) {
  // (a part without weight has only e = 0 and NaN; 2^d of it may be infinite, and 0 times that NaN)
  if (base == -kInf) return {o.inv_s, 0.0f, 0.0f};
  const float d = y_between(base, o.base);
  const float scale = __builtin_amdgcn_exp2f(d);
  if (scale == 0.0f) return {scale * o.inv_s, 0.0f, 0.0f};  // (d may be -inf)
  return {scale * o.inv_s, fmaf(b, d * kLn2 - o.log_s + o.entropy, a), b * kLn2};
}

__device__ inline F8 gradient(const F8& y, const F8& e, const RowSlope& r) {
  F8 g;
#pragma unroll
  for (int j = 0; j < 8; ++j) g[j] = -(e[j] * r.inv) * fmaf(y[j], r.slope, r.shift);
  return g;
}

__device__ inline float gradient_of_token(const RowEnd& o, float z, float a, float b) {
  const float y = y_of(z, o.base), p = __builtin_amdgcn_exp2f(y) * o.inv_s;
  const float h =
      b != 0.0f ? b * p * (larger(y, -0x1p100f) * kLn2 - o.log_s + o.entropy) : 0.0f;
  return fmaf(a, o.others, -h);
}

// ---- the best alternatives ------------------------------------------------------------------
constexpr int kListed = 512;  // candidates that a row's list holds

// Rises with the logit and, among equal ones (-0 is 0), falls with the index.
__device__ inline uint64_t key_of(float z, int index) {
  const uint32_t b = __float_as_uint(z + 0.0f);
  const uint32_t v = b >> 31 ? ~b : b | 0x80000000u;
  return ((uint64_t)v << 32) | (0xFFFFFFFFu - (uint32_t)index);
}

__device__ inline float logit_of(uint64_t key) {
  const uint32_t v = (uint32_t)(key >> 32);
  return __uint_as_float(v >> 31 ? v & 0x7FFFFFFFu : ~v);
}

template <int kThreads>
struct TopSpace {
  static constexpr int kWaves = kThreads / kWave;
  float largest[kWaves > 1 ? kWaves : 1][kWave];
  uint64_t list[kListed];
  uint64_t best[2];
  uint32_t count, reaching;
  uint16_t thread[kThreads];  // that reach the bound, in a long row
};

// All threads of a row: a workgroup, or one wave, whose LDS accesses are in order.
template <int kThreads>
__device__ inline void row_sync() {
  if constexpr (kThreads > kWave) {
    __syncthreads();
  } else {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}

// The top-th largest of the 64 lanes' values.
__device__ inline float largest_but(float v, int top) {
  int above = 0;  // the values before this one in falling order
  const int lane = threadIdx.x & (kWave - 1);
#pragma unroll
  for (int j = 0; j < kWave; ++j) {
    const float w = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), j));
    above += w > v || (w == v && j < lane);
  }
  const uint64_t at = __ballot(above == top - 1);
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), __builtin_ctzll(at)));
}

// mine: the thread's largest logit.  each(f): f(logit, index) for the thread's logits;
// some(reaches, f): the same for those of the threads for which `reaches` is true, by whichever
// threads.
template <int kThreads, class Each, class Some>
__device__ inline void best_of_row(const LogprobArgs& a, int64_t row, const RowEnd& o, float mine,
                                   TopSpace<kThreads>& sp, Each&& each, Some&& some) {
  const int lane = threadIdx.x & (kWave - 1), thread = threadIdx.x % kThreads;
  if (thread == 0) sp.count = sp.reaching = 0;
  float v = mine;
  if constexpr (kThreads > kWave) {
    sp.largest[threadIdx.x / kWave][lane] = mine;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kThreads / kWave; ++w) v = larger(v, sp.largest[w][lane]);
  } else {
    row_sync<kThreads>();
  }
  const float bound = largest_but(v, a.top);
  const auto reaches = [&](float z) { return z >= bound && z > -kInf; };
  some(reaches(mine), [&](float z, int index) {
    if (!reaches(z)) return;
    const uint32_t at = atomicAdd(&sp.count, 1u);
    if (at < (uint32_t)kListed) sp.list[at] = key_of(z, index);
  });
  row_sync<kThreads>();
  const int n = (int)sp.count;
  float* logp = a.top_logp + row * a.top;
  int64_t* tokens = a.top_tokens + row * a.top;
  const auto put = [&](int rank, uint64_t key) {
    logp[rank] = (float)logp_of(o, logit_of(key));
    tokens[rank] = (int64_t)(0xFFFFFFFFu - (uint32_t)key);
  };
  const auto none = [&](int rank) { logp[rank] = -kInf, tokens[rank] = -1; };
  if (n <= kListed) {
    if (thread < kWave) {
      for (int i = lane; i < n; i += kWave) {
        const uint64_t key = sp.list[i];
        int rank = 0;
        for (int j = 0; j < n; ++j) rank += sp.list[j] > key;
        if (rank < a.top) put(rank, key);
      }
      if (lane >= n && lane < a.top) none(lane);
    }
    return;
  }
  // ties beyond the list: one after another (there are more than `top` of them)
  uint64_t before = ~0ull;
  for (int rank = 0; rank < a.top; ++rank) {
    if (thread == 0) sp.best[rank & 1] = 0;
    row_sync<kThreads>();
    uint64_t best = 0;
    each([&](float z, int index) {
      const uint64_t key = key_of(z, index);
      if (z > -kInf && key < before && key > best) best = key;
    });
    if (best) atomicMax((unsigned long long*)&sp.best[rank & 1], (unsigned long long)best);
    row_sync<kThreads>();
    before = sp.best[rank & 1];
    if (thread == 0) put(rank, before);
  }
}

// ---- a row's results ------------------------------------------------------------------------
__device__ inline void write_row(const LogprobArgs& a, int64_t row, const RowEnd& o) {
  a.logp[row] = o.logp;
  a.entropy[row] = o.entropy;
  if (a.stats) {
    a.stats[2 * row] = make_float4(o.base, o.inv_s, o.log_s, o.entropy);
    a.stats[2 * row + 1] = make_float4(o.others, o.live ? 1.0f : 0.0f, 0.0f, 0.0f);
  }
}

// The weights of a row; false: it has no gradient.
__device__ inline bool weights_of(const LogprobArgs& a, int64_t row, bool live, bool given,
                                  float* wl, float* we) {
  *wl = given && a.logp_weight ? a.logp_weight[row] : 0.0f;
  *we = a.entropy_weight ? a.entropy_weight[row] : 0.0f;
  return live && (*wl != 0.0f || *we != 0.0f);
}

// Stores the gradient of the block at column col from its y and e.
template <class T, bool kWhole, bool kStream>
__device__ inline void put_gradient(T* grad, const F8& y, const F8& e, const RowSlope& r,
                                    const RowEnd& o, bool some, float wl, float we, int col,
                                    int cols, int token, float z_token) {
  F8 g = {};
  if (some) {
    g = gradient(y, e, r);
    // (a slope above 2^26 may be infinite times y, and 0 times that is NaN; NaN of a row reaches the
    // legal logits alone)
    const bool number = r.inv == r.inv;
    if (!(number && fabsf(r.slope) <= 0x1p26f && fabsf(r.shift) <= 0x1p126f)) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        g[j] = e[j] == 0.0f && (number || y[j] == -0x1p100f) ? 0.0f : g[j];
    }
    if ((uint32_t)(token - col) < 8u) {
      const float gt = gradient_of_token(o, z_token, wl, we);
#pragma unroll
      for (int j = 0; j < 8; ++j) g[j] = col + j == token ? gt : g[j];
    }
  }
  store8<T, kWhole, kStream>(grad, col, cols, g);
}

template <int kThreads>
constexpr int block_of() {
  return kThreads <= kWave ? 256 : kThreads;
}

// Rows in registers: kThreads threads of kVecs blocks each.
template <class T, int kThreads, int kVecs, bool kWhole, bool kGrad>
__global__ __launch_bounds__(block_of<kThreads>()) void logprob_rows_kernel(LogprobArgs a) {
  constexpr int kRows = block_of<kThreads>() / kThreads;
  __shared__ Sums smem[16];
  __shared__ TopSpace<kThreads> space[kGrad ? 1 : kRows];
  const int lane = threadIdx.x % kThreads, slot = row_slot<kThreads>();
  const int64_t row = block_index() * kRows + slot;
  if (row >= a.r.rows) return;  // (whole waves or workgroups)
  const RowIn<T> in = row_in<T>(a.r, row);
  Block<T, false> raw[kVecs];
#pragma unroll
  for (int i = 0; i < kVecs; ++i)
    raw[i] = load_block<T, false, kWhole>(in, 8 * (lane + i * kThreads));
  float z_token;
  const int token = token_of<T>(a.r, row, &z_token);
  F8 z[kVecs];
  Sums t = no_sums();
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    const int col = 8 * (lane + i * kThreads);
    z[i] = legal_logits<T, false, kWhole>(raw[i], in, col,
                                          ok_bytes<T, false, kWhole>(raw[i], in, col));
    t.m = larger(t.m, largest_number(z[i]));
  }
  const float mine = t.m;
  t.m = lanes_reduce<Max, kWave>(t.m);
  const float base = t.m;  // (of this wave)
  F8 y[kVecs], e[kVecs];
#pragma unroll
  for (int i = 0; i < kVecs; ++i)
    add_block(t, z[i], base_of(base), token - 8 * (lane + i * kThreads), y[i], e[i]);
  row_join<kThreads>(t, smem);
  const RowEnd o = finish_row(t, z_token, token >= 0);
  if (lane == 0) write_row(a, row, o);
  if constexpr (kGrad) {
    float wl, we;
    const bool some = weights_of(a, row, o.live, token >= 0, &wl, &we);
    const RowSlope r = slope_of(o, base, wl, we);
    T* grad = static_cast<T*>(a.grad) + row * a.r.vocab;
#pragma unroll
    for (int i = 0; i < kVecs; ++i)
      put_gradient<T, kWhole, false>(grad, y[i], e[i], r, o, some, wl, we,
                                     8 * (lane + i * kThreads), in.cols, token, z_token);
  } else if (a.top) {
    const auto each = [&](auto&& f) {
#pragma unroll
      for (int i = 0; i < kVecs; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) f(z[i][j], 8 * (lane + i * kThreads) + j);
    };
    best_of_row<kThreads>(a, row, o, mine, space[slot], each, [&](bool reaches, auto&& f) {
      if (reaches) each(f);
    });
  }
}

// Rows that are longer: a workgroup reads kAhead blocks a thread at a time.
constexpr int kAhead = 4;

template <class T, bool kWhole>
__device__ inline F8 logits_at(const RowIn<T>& in, int col) {
  const Block<T, false> b = load_block<T, false, kWhole>(in, col);
  return legal_logits<T, false, kWhole>(b, in, col, ok_bytes<T, false, kWhole>(b, in, col));
}

template <class T, int kLongThreads, bool kWhole, bool kGrad>
__global__ __launch_bounds__(kLongThreads) void logprob_long_kernel(LogprobArgs a) {
  __shared__ Sums smem[16];
  __shared__ TopSpace<kLongThreads> space[1];
  constexpr int kStep = 8 * kLongThreads;
  const int64_t row = block_index();
  if (row >= a.r.rows) return;
  const RowIn<T> in = row_in<T>(a.r, row);
  float z_token;
  const int token = token_of<T>(a.r, row, &z_token);
  const int first = 8 * threadIdx.x;
  Sums t = no_sums();
  float mine = -kInf;
  for (int64_t at = first; at < in.cols; at += kAhead * kStep) {
    Block<T, false> raw[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int64_t col = at + (int64_t)u * kStep;
      raw[u] = load_block<T, false, kWhole>(in, (int)(col < in.cols ? col : first));
    }
    F8 z[kAhead];
    float m = -kInf;
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int64_t col = at + (int64_t)u * kStep;
      const uint64_t ok = col < in.cols ? ok_bytes<T, false, kWhole>(raw[u], in, (int)col) : 0;
      z[u] = legal_logits<T, false, kWhole>(raw[u], in, (int)(col < in.cols ? col : first), ok);
      m = larger(m, largest_number(z[u]));
    }
    mine = larger(mine, m);
    if (m > t.m) rebase(t, m);
    const float base = base_of(t.m);
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      F8 y, e;
      add_block(t, z[u], base, (int)(token - at - (int64_t)u * kStep), y, e);
    }
  }
  row_join<kLongThreads>(t, smem);
  const RowEnd o = finish_row(t, z_token, token >= 0);
  if (threadIdx.x == 0) write_row(a, row, o);
  if constexpr (kGrad) {
    float wl, we;
    const bool some = weights_of(a, row, o.live, token >= 0, &wl, &we);
    T* grad = static_cast<T*>(a.grad) + row * a.r.vocab;
    const RowSlope r = slope_of(o, o.base, wl, we);
    for (int64_t col = first; col < in.cols; col += kStep) {
      F8 y, e;
      exponentials(logits_at<T, kWhole>(in, (int)col), o.base, y, e);
      put_gradient<T, kWhole, true>(grad, y, e, r, o, some, wl, we, (int)col, in.cols, token,
                                    z_token);
    }
  } else if (a.top) {
    const auto at = [&](int64_t col, auto&& f) {
      const F8 z = logits_at<T, kWhole>(in, (int)col);
#pragma unroll
      for (int j = 0; j < 8; ++j) f(z[j], (int)col + j);
    };
    // (the blocks of the threads that reach the bound are shared out: one after another they would
    // take such a thread longer than the row's first reading took all)
    TopSpace<kLongThreads>& sp = space[0];
    best_of_row<kLongThreads>(
        a, row, o, mine, sp,
        [&](auto&& f) {
          for (int64_t col = first; col < in.cols; col += kStep) at(col, f);
        },
        [&](bool reaches, auto&& f) {
          if (reaches) sp.thread[atomicAdd(&sp.reaching, 1u)] = (uint16_t)threadIdx.x;
          __syncthreads();
          // (fewer than 2^27 + 1024 blocks: rows have at most 2^30 tokens)
          const uint32_t blocks = (uint32_t)((in.cols - 1) / kStep + 1), all = sp.reaching * blocks;
          for (uint32_t i = threadIdx.x; i < all; i += kLongThreads) {
            const uint32_t who = i / blocks;
            const int64_t col = 8 * (int64_t)sp.thread[who] + (int64_t)(i - who * blocks) * kStep;
            if (col < in.cols) at(col, f);
          }
        });
  }
}

// The gradient from a row's statistics: a wave a piece of 512 tokens.
template <class T, bool kWhole>
__global__ __launch_bounds__(256) void logprob_grad_kernel(LogprobArgs a, int64_t pieces) {
  const int64_t unit = block_index() * 4 + row_slot<kWave>();
  const int64_t row = unit / pieces;
  if (row >= a.r.rows) return;
  const int64_t at = unit % pieces * 512 + 8 * (threadIdx.x % kWave);
  if (at >= a.r.vocab) return;
  const int col = (int)at;
  const RowIn<T> in = row_in<T>(a.r, row);
  const Block<T, false> raw = load_block<T, false, kWhole>(in, col);
  float z_token;
  const int token = token_of<T>(a.r, row, &z_token);
  const float4 s = a.stats[2 * row], more = a.stats[2 * row + 1];
  RowEnd o{};
  o.base = s.x, o.inv_s = s.y, o.log_s = s.z, o.entropy = s.w, o.others = more.x;
  float wl, we;
  const bool some = weights_of(a, row, more.y != 0.0f, token >= 0, &wl, &we);
  const F8 z = legal_logits<T, false, kWhole>(raw, in, col,
                                              ok_bytes<T, false, kWhole>(raw, in, col));
  F8 y, e;
  exponentials(z, o.base, y, e);
  put_gradient<T, kWhole, false>(static_cast<T*>(a.grad) + row * a.r.vocab, y, e,
                                 slope_of(o, o.base, wl, we), o, some, wl, we, col, in.cols, token,
                                 z_token);
}

// ---- launches -------------------------------------------------------------------------------
template <class F>
void with_type(int dtype, F&& f) {
  if (dtype == OMQ_NET_F32) return f(float{});
  if (dtype == OMQ_NET_BF16) return f(bf16{});
  return f(f16{});
}

template <class T, int kThreads, int kVecs, bool kGrad>
void launch_rows(const LogprobArgs& a, hipStream_t st) {
  constexpr int kBlock = block_of<kThreads>();
  const dim3 grid = grid_of(ceil_div(a.r.rows, kBlock / kThreads), kBlock);
  const auto kernel = a.r.vocab % 8 == 0
                          ? logprob_rows_kernel<T, kThreads, kVecs, true, kGrad>
                          : logprob_rows_kernel<T, kThreads, kVecs, false, kGrad>;
  kernel<<<grid, kBlock, 0, st>>>(a);
}

template <bool kGrad>
void launch_logprobs(const LogprobArgs& a, hipStream_t st) {
  with_type(a.r.dtype, [&](auto t) {
    using T = decltype(t);
    const int64_t v = a.r.vocab;
    // as few threads a row as hold it in two or three blocks each: what a row costs beside its loads
    // goes by its waves (8192 rows of 4672, bf16, with gradient: 44 us by 256 threads, 56 by 512;
    // 65536 of 362: 42 by 64, 76 by 128; 4096 of 10000: 46 by 512, 52 by 1024)
    if (v <= 512) return launch_rows<T, 64, 1, kGrad>(a, st);
    if (v <= 1024) return launch_rows<T, 64, 2, kGrad>(a, st);
    if (v <= 2048) return launch_rows<T, 128, 2, kGrad>(a, st);
    if (v <= 4096) return launch_rows<T, 256, 2, kGrad>(a, st);
    if (v <= 6144) return launch_rows<T, 256, 3, kGrad>(a, st);
    if (v <= 8192) return launch_rows<T, 512, 2, kGrad>(a, st);
    if (v <= 12288) return launch_rows<T, 512, 3, kGrad>(a, st);
    if (v <= 16384) return launch_rows<T, 1024, 2, kGrad>(a, st);
    // workgroups of 256 threads where there is one for each compute unit twice: a row's end (its
    // sums' join, its alternatives) takes as long in all, and the other rows' loads go on (131072
    // tokens, bf16, 8 alternatives: 2048 rows 117 us, 157 with 1024 threads; 512 rows 41 and 41; 256
    // rows 33 and 21)
    const auto go = [&](auto threads) {
      constexpr int kThreads = threads.value;
      const dim3 grid = grid_of(a.r.rows, kThreads);
      const auto kernel = v % 8 == 0 ? logprob_long_kernel<T, kThreads, true, kGrad>
                                     : logprob_long_kernel<T, kThreads, false, kGrad>;
      kernel<<<grid, kThreads, 0, st>>>(a);
    };
    if (a.r.rows >= 512)
      go(std::integral_constant<int, 256>{});
    else
      go(std::integral_constant<int, 1024>{});
  });
}

int check_rows(const char* name, const omq_logprob_rows* r) {
  if (!r) return net_fail(OMQ_NET_E_ARG, "%s: a null array", name);
  if (!dtype_known(r->dtype))
    return net_fail(OMQ_NET_E_ARG, "%s: logits of type %d", name, r->dtype);
  if (r->rows < 0 || r->vocab < 1 || r->logits_stride < 0 || (r->legal && r->legal_stride < 0))
    return net_fail(OMQ_NET_E_ARG, "%s: rows %lld, vocab %lld, strides %lld and %lld", name,
                    (long long)r->rows, (long long)r->vocab, (long long)r->logits_stride,
                    (long long)r->legal_stride);
  if (r->rows > OMQ_NET_MAX_COUNT || r->vocab > OMQ_NET_MAX_ACTIONS)
    return net_fail(OMQ_NET_E_LIMIT, "%s: rows %lld (at most %d), vocab %lld (at most %d)", name,
                    (long long)r->rows, OMQ_NET_MAX_COUNT, (long long)r->vocab,
                    OMQ_NET_MAX_ACTIONS);
  if (r->rows > 0 && (!r->logits || !r->tokens))
    return net_fail(OMQ_NET_E_ARG, "%s: a null array", name);
  return OMQ_NET_OK;
}

}  // namespace
}  // namespace omq_net

using namespace omq_net;

extern "C" {

int omq_token_logprobs(const omq_logprob_rows* r, int32_t top, float* logp, float* entropy,
                       float* top_logp, int64_t* top_tokens, float* stats, void* stream) {
  const char* name = "omq_token_logprobs";
  if (int rc = check_rows(name, r)) return rc;
  if (top < 0) return net_fail(OMQ_NET_E_ARG, "%s: top %d", name, top);
  if (top > OMQ_NET_MAX_TOP)
    return net_fail(OMQ_NET_E_LIMIT, "%s: top %d (at most %d)", name, top, OMQ_NET_MAX_TOP);
  if (r->rows == 0) return OMQ_NET_OK;
  if (!logp || !entropy || (top && (!top_logp || !top_tokens)))
    return net_fail(OMQ_NET_E_ARG, "%s: a null array", name);
  if (stats && !on_16_bytes(stats))
    return net_fail(OMQ_NET_E_ARG, "%s: stats must begin on a 16-byte boundary", name);
  LogprobArgs a{};
  a.r = *r, a.logp = logp, a.entropy = entropy, a.top = top, a.top_logp = top_logp;
  a.top_tokens = top_tokens, a.stats = reinterpret_cast<float4*>(stats);
  launch_logprobs<false>(a, (hipStream_t)stream);
  return net_status(name);
}

int omq_token_logprobs_grad(const omq_logprob_rows* r, const float* stats,
                            const float* logp_weight, const float* entropy_weight, void* grad,
                            void* stream) {
  const char* name = "omq_token_logprobs_grad";
  if (int rc = check_rows(name, r)) return rc;
  if (r->rows == 0) return OMQ_NET_OK;
  if (!stats || !grad) return net_fail(OMQ_NET_E_ARG, "%s: a null array", name);
  if (!on_16_bytes(stats))
    return net_fail(OMQ_NET_E_ARG, "%s: stats must begin on a 16-byte boundary", name);
  LogprobArgs a{};
  a.r = *r, a.logp_weight = logp_weight, a.entropy_weight = entropy_weight, a.grad = grad;
  a.stats = reinterpret_cast<float4*>(const_cast<float*>(stats));
  const int64_t pieces = ceil_div(r->vocab, 512);
  const dim3 grid = grid_of(ceil_div(r->rows * pieces, 4), 256);
  with_type(r->dtype, [&](auto t) {
    using T = decltype(t);
    const auto kernel =
        r->vocab % 8 == 0 ? logprob_grad_kernel<T, true> : logprob_grad_kernel<T, false>;
    kernel<<<grid, 256, 0, (hipStream_t)stream>>>(a, pieces);
  });
  return net_status(name);
}

int omq_token_logprobs_with_grad(const omq_logprob_rows* r, const float* logp_weight,
                                 const float* entropy_weight, float* logp, float* entropy,
                                 void* grad, void* stream) {
  const char* name = "omq_token_logprobs_with_grad";
  if (int rc = check_rows(name, r)) return rc;
  if (r->rows == 0) return OMQ_NET_OK;
  if (!logp || !entropy || !grad) return net_fail(OMQ_NET_E_ARG, "%s: a null array", name);
  LogprobArgs a{};
  a.r = *r, a.logp_weight = logp_weight, a.entropy_weight = entropy_weight, a.logp = logp;
  a.entropy = entropy, a.grad = grad;
  launch_logprobs<true>(a, (hipStream_t)stream);
  return net_status(name);
}

}  // extern "C"
