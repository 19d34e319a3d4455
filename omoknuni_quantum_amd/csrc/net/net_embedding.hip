// The token embedding with a scale, and its gradient over the sorted tokens (gfx950).
//
// Forward: a gather of rows; bound by the bytes of the output.
//
// Gradient: out[v] = scale * sum of grad[t] over the tokens t of v.  The tokens are sorted by id
// (stable, so that every sum runs in ascending t), then the sorted tokens and the vocabulary's
// rows are walked as one merged list: token i comes before the end of row v when key[i] <= v.
// The list is cut into pieces of equal length, so a piece has the same work whether it holds the
// many tokens of one row or many rows without tokens.  A row that lies in one piece is written
// by it; a row that crosses pieces leaves partial sums in float32, which a second launch adds in
// the order of the pieces.  No atomics on floating-point values: the result is the same at every
// call.
#include "net_common.h"

namespace omq_net {
namespace {

// ---- forward --------------------------------------------------------------------------------
template <class T, class Id>
__global__ __launch_bounds__(256) void embed_kernel(const Id* __restrict__ ids, int64_t tokens,
                                                    const T* __restrict__ weight,
                                                    int64_t weight_stride, int64_t vocab,
                                                    int dim, int blocks, float scale,
                                                    T* __restrict__ out) {
  const int64_t first = (int64_t)blockIdx.x * 256;
  const int64_t row0 = first / blocks;
  const uint32_t in = (uint32_t)(first - row0 * blocks) + threadIdx.x;
  const int64_t t = row0 + in / (uint32_t)blocks;
  const int col = 8 * (int)(in % (uint32_t)blocks);
  if (t >= tokens) return;
  const int64_t id = (int64_t)ids[t];
  F8 v = {};
  if (id >= 0 && id < vocab) v = load8<T>(weight + id * weight_stride + col, dim - col) * scale;
  store8<T>(out + t * dim + col, v, dim - col);
}

// ---- sort -----------------------------------------------------------------------------------
// A pair is (key, token).  Keys lie in [0, vocab]; `vocab` stands for an id outside the
// vocabulary, so those tokens sort behind all others.
constexpr int kMaxDigitBits = 11;
constexpr int kTile = 2048;       // tokens of a workgroup of the radix passes
constexpr int kSmallSort = 4096;  // tokens that one workgroup sorts in LDS

template <class Id>
__device__ inline uint32_t key_of(const Id* ids, int64_t t, int64_t vocab) {
  const int64_t id = (int64_t)ids[t];
  return id >= 0 && id < vocab ? (uint32_t)id : (uint32_t)vocab;
}

// The lanes of the wave whose digit equals this lane's, among the lanes of `active`.
__device__ inline uint64_t match_digit(uint32_t digit, int bits, uint64_t active) {
  uint64_t m = active;
  for (int b = 0; b < bits; ++b) {
    const uint64_t set = __ballot((digit >> b) & 1u);
    m &= (digit >> b) & 1u ? set : ~set;
  }
  return m;
}

__device__ inline int lanes_below(uint64_t m) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32),
                                   __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0u));
}

// Exclusive prefix sums of n counters in LDS by the whole workgroup of kThreads threads.
template <int kThreads>
__device__ inline void block_scan(uint32_t* counts, int n, uint32_t* wave_sums) {
  const int per = (n + kThreads - 1) / kThreads;
  const int from = threadIdx.x * per;
  uint32_t mine = 0;
  for (int j = 0; j < per; ++j)
    if (from + j < n) mine += counts[from + j];
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  uint32_t incl = mine;
  for (int d = 1; d < kWave; d <<= 1) {
    const uint32_t up = __shfl_up(incl, d);
    if (lane >= d) incl += up;
  }
  if (lane == kWave - 1) wave_sums[wave] = incl;
  __syncthreads();
  uint32_t base = incl - mine;
  for (int w = 0; w < wave; ++w) base += wave_sums[w];
  for (int j = 0; j < per; ++j)
    if (from + j < n) {
      const uint32_t c = counts[from + j];
      counts[from + j] = base;
      base += c;
    }
  __syncthreads();
}

// One wave takes 64 digits in order: the place of each among all that the wave has seen of its
// digit, from next[digit], which advances.
__device__ inline uint32_t take_places(uint32_t digit, int bits, bool here, uint32_t* next) {
  const uint64_t active = __ballot(here);
  const uint64_t same = match_digit(digit, bits, active);
  uint32_t place = 0;
  const int below = lanes_below(same);
  if (here) place = next[digit] + below;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  if (here && below == 0) next[digit] += __popcll(same);
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  return place;
}

// All passes of up to kSmallSort tokens in one workgroup.  8-bit digits.
template <class Id>
__global__ __launch_bounds__(1024) void sort_small_kernel(const Id* __restrict__ ids, int tokens,
                                                          int64_t vocab, int bits,
                                                          uint2* __restrict__ pairs) {
  constexpr int kWaves = 16, kRounds = kSmallSort / 1024;
  __shared__ uint2 kept[kSmallSort];
  __shared__ uint32_t next[kWaves][256];
  __shared__ uint32_t base[256];
  __shared__ uint32_t wave_sums[kWaves];
  const int wave = threadIdx.x / kWave, lane = threadIdx.x & (kWave - 1);
  uint2 mine[kRounds];
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const int i = (wave * kRounds + r) * kWave + lane;
    if (i < tokens) mine[r] = make_uint2(key_of(ids, i, vocab), (uint32_t)i);
  }
  for (int shift = 0; shift < bits; shift += 8) {
    for (int j = threadIdx.x; j < kWaves * 256; j += 1024) (&next[0][0])[j] = 0;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
      const int i = (wave * kRounds + r) * kWave + lane;
      if (i < tokens) atomicAdd(&next[wave][(mine[r].x >> shift) & 255u], 1u);
    }
    __syncthreads();
    if (threadIdx.x < 256) {
      uint32_t sum = 0;
      for (int w = 0; w < kWaves; ++w) {
        const uint32_t c = next[w][threadIdx.x];
        next[w][threadIdx.x] = sum;
        sum += c;
      }
      base[threadIdx.x] = sum;
    }
    __syncthreads();
    block_scan<1024>(base, 256, wave_sums);
    for (int j = threadIdx.x; j < kWaves * 256; j += 1024) (&next[0][0])[j] += base[j & 255];
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
      const int i = (wave * kRounds + r) * kWave + lane;
      const bool here = i < tokens;
      const uint32_t digit = here ? (mine[r].x >> shift) & 255u : 0u;
      const uint32_t at = take_places(digit, 8, here, next[wave]);
      if (here) kept[at] = mine[r];
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
      const int i = (wave * kRounds + r) * kWave + lane;
      if (i < tokens) mine[r] = kept[i];
    }
    __syncthreads();
  }
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const int i = (wave * kRounds + r) * kWave + lane;
    if (i < tokens) pairs[i] = mine[r];
  }
}

// Radix pass, step 1: counts[digit * tiles + tile].
template <class Id>
__global__ __launch_bounds__(256) void digit_counts_kernel(const Id* __restrict__ ids,
                                                           const uint2* __restrict__ in,
                                                           int64_t tokens, int64_t vocab,
                                                           int shift, int bits,
                                                           uint32_t* __restrict__ counts) {
  __shared__ uint32_t hist[1 << kMaxDigitBits];
  const int bins = 1 << bits;
  for (int j = threadIdx.x; j < bins; j += 256) hist[j] = 0;
  __syncthreads();
  const int64_t first = (int64_t)blockIdx.x * kTile;
#pragma unroll
  for (int r = 0; r < kTile / 256; ++r) {
    const int64_t t = first + r * 256 + threadIdx.x;
    if (t < tokens) {
      const uint32_t key = in ? in[t].x : key_of(ids, t, vocab);
      atomicAdd(&hist[(key >> shift) & (bins - 1)], 1u);
    }
  }
  __syncthreads();
  for (int j = threadIdx.x; j < bins; j += 256)
    counts[(int64_t)j * gridDim.x + blockIdx.x] = hist[j];
}

// Step 2: per digit (one wave), the exclusive prefix sums over the tiles, and the total.
__global__ __launch_bounds__(256) void digit_scan_kernel(uint32_t* __restrict__ counts, int tiles,
                                                         int bins, uint32_t* __restrict__ totals) {
  const int digit = blockIdx.x * 4 + threadIdx.x / kWave;
  const int lane = threadIdx.x & (kWave - 1);
  if (digit >= bins) return;
  uint32_t* row = counts + (int64_t)digit * tiles;
  uint32_t carry = 0;
  for (int t0 = 0; t0 < tiles; t0 += kWave) {
    const int t = t0 + lane;
    const uint32_t mine = t < tiles ? row[t] : 0u;
    uint32_t incl = mine;
    for (int d = 1; d < kWave; d <<= 1) {
      const uint32_t up = __shfl_up(incl, d);
      if (lane >= d) incl += up;
    }
    if (t < tiles) row[t] = carry + incl - mine;
    carry += __shfl(incl, kWave - 1);
  }
  if (lane == 0) totals[digit] = carry;
}

// Step 3: every pair to its place.
template <class Id>
__global__ __launch_bounds__(256) void digit_scatter_kernel(
    const Id* __restrict__ ids, const uint2* __restrict__ in, int64_t tokens, int64_t vocab,
    int shift, int bits, const uint32_t* __restrict__ counts, const uint32_t* __restrict__ totals,
    uint2* __restrict__ out) {
  constexpr int kWaves = 4, kRounds = kTile / 256;
  __shared__ uint32_t next[kWaves][1 << kMaxDigitBits];
  __shared__ uint32_t base[1 << kMaxDigitBits];
  __shared__ uint32_t wave_sums[kWaves];
  const int bins = 1 << bits;
  const int wave = threadIdx.x / kWave, lane = threadIdx.x & (kWave - 1);
  const int64_t first = (int64_t)blockIdx.x * kTile + wave * (kTile / kWaves);
  uint2 mine[kRounds];
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const int64_t t = first + r * kWave + lane;
    if (t < tokens) mine[r] = in ? in[t] : make_uint2(key_of(ids, t, vocab), (uint32_t)t);
  }
  for (int j = threadIdx.x; j < bins; j += 256) {
    base[j] = totals[j];
    for (int w = 0; w < kWaves; ++w) next[w][j] = 0;
  }
  __syncthreads();
  block_scan<256>(base, bins, wave_sums);
#pragma unroll
  for (int r = 0; r < kRounds; ++r)
    if (first + r * kWave + lane < tokens)
      atomicAdd(&next[wave][(mine[r].x >> shift) & (bins - 1)], 1u);
  __syncthreads();
  for (int j = threadIdx.x; j < bins; j += 256) {
    uint32_t at = base[j] + counts[(int64_t)j * gridDim.x + blockIdx.x];
    for (int w = 0; w < kWaves; ++w) {
      const uint32_t c = next[w][j];
      next[w][j] = at;
      at += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const bool here = first + r * kWave + lane < tokens;
    const uint32_t digit = here ? (mine[r].x >> shift) & (bins - 1) : 0u;
    const uint32_t at = take_places(digit, bits, here, next[wave]);
    if (here) out[at] = mine[r];
  }
}

// ---- sums -----------------------------------------------------------------------------------
// What a piece of the merged list leaves for the join.
struct Piece {
  int32_t first_row;  // the row its first partial sum belongs to, -1: it has none in `heads`
  int32_t last_row;   // the row that is open at its end
  int32_t open;       // it left a sum of last_row in `tails`
  int32_t unused;
};

// The number of tokens among the first `at` items of the merged list, by a search in which the
// kLanes lanes of a piece probe together: each step leaves 1/(kLanes+1) of the range.
template <int kLanes>
__device__ inline int64_t tokens_before(const uint2* pairs, int64_t tokens, int64_t vocab,
                                        int64_t at) {
  int64_t lo = at > vocab ? at - vocab : 0, hi = at < tokens ? at : tokens;
  const int lane = threadIdx.x & (kLanes - 1);
  const int shift = (threadIdx.x & (kWave - 1)) & ~(kLanes - 1);
  while (__any(lo < hi)) {  // (the pieces of a wave go on until the last is done)
    const int64_t n = hi - lo;
    // probes lo + n*(lane+1)/(kLanes+1), in [lo, hi)
    const int64_t i = lo + n * (lane + 1) / (kLanes + 1);
    const bool before = n > 0 && (int64_t)pairs[i < hi ? i : hi - 1].x <= at - i - 1;
    // token i is among the first `at` items; true for a prefix of the probes
    const uint64_t all = __ballot(before) >> shift;
    const int count = __popcll(kLanes == 64 ? all : all & ((1ull << (kLanes & 63)) - 1));
    if (n > 0) {
      const int64_t new_lo = count > 0 ? lo + n * count / (kLanes + 1) + 1 : lo;
      const int64_t new_hi = count < kLanes ? lo + n * (count + 1) / (kLanes + 1) : hi;
      lo = new_lo;
      hi = new_hi;
    }
  }
  return lo;
}

template <class T, class O, int kLanes>
__global__ __launch_bounds__(256) void sum_pieces_kernel(
    const T* __restrict__ grad, int64_t grad_stride, const uint2* __restrict__ pairs,
    int64_t tokens, int64_t vocab, int dim, float scale, int64_t piece, int64_t pieces,
    O* __restrict__ out, Piece* __restrict__ info, float* __restrict__ heads,
    float* __restrict__ tails) {
  constexpr int kBatch = 4;  // rows of `grad` in flight
  const int64_t c = (int64_t)blockIdx.x * (256 / kLanes) + threadIdx.x / kLanes;
  const int col = 8 * (int)(blockIdx.y * kLanes + (threadIdx.x & (kLanes - 1)));
  const int n = dim - col;
  const int64_t items = tokens + vocab;
  const int64_t d0 = c * piece < items ? c * piece : items;
  const int64_t d1 = d0 + piece < items ? d0 + piece : items;
  int64_t i = tokens_before<kLanes>(pairs, tokens, vocab, d0);
  const int64_t i1 = tokens_before<kLanes>(pairs, tokens, vocab, d1);
  if (c >= pieces) return;
  int64_t row = d0 - i;
  const int64_t row0 = row, row1 = d1 - i1;
  const bool shared = row0 < vocab && i > 0 && (int64_t)pairs[i - 1].x == row0;
  F8 acc = {};
  bool open = false;
  const auto end_row = [&]() {
    if (n > 0) {
      if (shared && row == row0)
        store8<float>(heads + c * dim + col, acc, n);
      else
        store8<O>(out + row * dim + col, acc * scale, n);
    }
    acc = F8{};
    open = false;
    ++row;
  };
  while (i < i1) {
    uint2 p[kBatch];
    F8 v[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      p[u] = i + u < i1 ? pairs[i + u] : make_uint2(0xFFFFFFFFu, 0u);
      if ((int64_t)p[u].x >= vocab) p[u].x = 0xFFFFFFFFu;
    }
#pragma unroll
    for (int u = 0; u < kBatch; ++u)
      if (p[u].x != 0xFFFFFFFFu && n > 0)
        v[u] = load8<T>(grad + (int64_t)p[u].y * grad_stride + col, n);
#pragma unroll
    for (int u = 0; u < kBatch; ++u)
      if (p[u].x != 0xFFFFFFFFu) {
        while (row < (int64_t)p[u].x) end_row();
        if (n > 0) acc += v[u];
        open = true;
      }
    i += kBatch;
  }
  while (row < row1) end_row();
  if (open && n > 0) store8<float>(tails + c * dim + col, acc, n);
  if (blockIdx.y == 0 && (threadIdx.x & (kLanes - 1)) == 0)
    info[c] = Piece{shared && row1 > row0 ? (int32_t)row0 : -1, (int32_t)row1, open ? 1 : 0, 0};
}

// The row that piece c ends and did not begin: the sums that the pieces before it left open, in
// their order, then its own.  64 columns a workgroup: 16 lanes of four columns, 16 slots of
// pieces, the slots' sums added in order.
template <class O>
__global__ __launch_bounds__(256) void join_pieces_kernel(const Piece* __restrict__ info, int dim,
                                                          float scale,
                                                          const float* __restrict__ heads,
                                                          const float* __restrict__ tails,
                                                          O* __restrict__ out) {
  __shared__ float part[16][64];
  const int64_t c = blockIdx.x;
  const int32_t row = info[c].first_row;
  if (row < 0) return;
  int64_t lo = 0, hi = c;  // the first piece at whose end `row` is open (or a later row)
  while (lo < hi) {
    const int64_t mid = (lo + hi) / 2;
    if (info[mid].last_row >= row)
      hi = mid;
    else
      lo = mid + 1;
  }
  const int slot = threadIdx.x / 16, col = blockIdx.y * 64 + 4 * (threadIdx.x & 15);
  float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int64_t k = lo + slot; k < c; k += 16)
    if (info[k].open) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (col + j < dim) acc[j] += tails[k * dim + col + j];
    }
#pragma unroll
  for (int j = 0; j < 4; ++j) part[slot][4 * (threadIdx.x & 15) + j] = acc[j];
  __syncthreads();
  const int at = blockIdx.y * 64 + threadIdx.x;
  if (threadIdx.x < 64 && at < dim) {
    float s = part[0][threadIdx.x];
    for (int k = 1; k < 16; ++k) s += part[k][threadIdx.x];
    s += heads[c * dim + at];
    out[(int64_t)row * dim + at] = (O)(s * scale);
  }
}

// ---- plan -----------------------------------------------------------------------------------
struct GradPlan {
  int bits, passes, digit_bits;
  int64_t tiles, piece, pieces;
  int lanes, col_tiles;
  int64_t at_pairs[2], at_counts, at_totals, at_info, at_heads, at_tails, bytes;
};

int64_t take(int64_t* at, int64_t bytes) {
  const int64_t here = *at;
  *at += ceil_div(bytes, 256) * 256;
  return here;
}

bool grad_sizes_ok(int64_t tokens, int64_t vocab, int64_t dim) {
  return tokens >= 0 && tokens <= OMQ_NET_MAX_COUNT && vocab >= 1 && vocab < OMQ_NET_MAX_COUNT &&
         dim >= 1 && dim <= OMQ_NET_MAX_DIM;
}

GradPlan grad_plan(int64_t tokens, int64_t vocab, int64_t dim) {
  GradPlan p{};
  while (p.bits < 32 && (vocab >> p.bits) != 0) ++p.bits;
  p.passes = (int)ceil_div(p.bits, kMaxDigitBits);
  p.digit_bits = (int)ceil_div(p.bits, p.passes);
  p.tiles = ceil_div(tokens, kTile);
  p.lanes = dim <= 64 ? 8 : dim <= 128 ? 16 : dim <= 256 ? 32 : 64;
  p.col_tiles = (int)ceil_div(dim, 8 * p.lanes);
  // pieces for about 4096 waves, of 16 to 1024 items
  const int64_t items = tokens + vocab;
  const int64_t wanted = ceil_div(4096ll * (kWave / p.lanes), p.col_tiles);
  p.piece = ceil_div(items, wanted);
  p.piece = p.piece < 16 ? 16 : p.piece > 1024 ? 1024 : p.piece;
  p.pieces = ceil_div(items, p.piece);
  int64_t at = 0;
  p.at_pairs[0] = take(&at, 8 * tokens);
  const bool radix = tokens > kSmallSort;
  p.at_pairs[1] = take(&at, radix && p.passes > 1 ? 8 * tokens : 0);
  p.at_counts = take(&at, radix ? 4 * (p.tiles << p.digit_bits) : 0);
  p.at_totals = take(&at, radix ? 4ll << p.digit_bits : 0);
  p.at_info = take(&at, (int64_t)sizeof(Piece) * p.pieces);
  p.at_heads = take(&at, 4 * p.pieces * dim);
  p.at_tails = take(&at, 4 * p.pieces * dim);
  p.bytes = at;
  return p;
}

// The sorted pairs; returns where they are.
template <class Id>
const uint2* sort_tokens(const GradPlan& p, const Id* ids, int64_t tokens, int64_t vocab, char* ws,
                         hipStream_t st) {
  uint2* buf[2] = {reinterpret_cast<uint2*>(ws + p.at_pairs[0]),
                   reinterpret_cast<uint2*>(ws + p.at_pairs[1])};
  if (tokens == 0) return buf[0];
  if (tokens <= kSmallSort) {
    sort_small_kernel<Id><<<1, 1024, 0, st>>>(ids, (int)tokens, vocab, p.bits, buf[0]);
    return buf[0];
  }
  uint32_t* counts = reinterpret_cast<uint32_t*>(ws + p.at_counts);
  uint32_t* totals = reinterpret_cast<uint32_t*>(ws + p.at_totals);
  const uint2* in = nullptr;
  for (int pass = 0; pass < p.passes; ++pass) {
    uint2* to = buf[pass & 1];
    const int shift = pass * p.digit_bits, bins = 1 << p.digit_bits;
    digit_counts_kernel<Id><<<(uint32_t)p.tiles, 256, 0, st>>>(ids, in, tokens, vocab, shift,
                                                              p.digit_bits, counts);
    digit_scan_kernel<<<(uint32_t)ceil_div(bins, 4), 256, 0, st>>>(counts, (int)p.tiles, bins,
                                                                 totals);
    digit_scatter_kernel<Id><<<(uint32_t)p.tiles, 256, 0, st>>>(
        ids, in, tokens, vocab, shift, p.digit_bits, counts, totals, to);
    in = to;
  }
  return in;
}

template <class T, class O, int kLanes>
void launch_sums(const GradPlan& p, const void* grad, int64_t grad_stride, const uint2* pairs,
                 int64_t tokens, int64_t vocab, int dim, float scale, void* out, char* ws,
                 hipStream_t st) {
  Piece* info = reinterpret_cast<Piece*>(ws + p.at_info);
  float* heads = reinterpret_cast<float*>(ws + p.at_heads);
  float* tails = reinterpret_cast<float*>(ws + p.at_tails);
  const dim3 grid((uint32_t)ceil_div(p.pieces, 256 / kLanes), (uint32_t)p.col_tiles);
  sum_pieces_kernel<T, O, kLanes><<<grid, 256, 0, st>>>(
      static_cast<const T*>(grad), grad_stride, pairs, tokens, vocab, dim, scale, p.piece,
      p.pieces, static_cast<O*>(out), info, heads, tails);
  if (p.pieces > 1)
    join_pieces_kernel<O><<<dim3((uint32_t)p.pieces, (uint32_t)ceil_div(dim, 64)), 256, 0, st>>>(
        info, dim, scale, heads, tails, static_cast<O*>(out));
}

template <class T, class O, class... A>
void launch_sums_lanes(const GradPlan& p, A... a) {
  switch (p.lanes) {
    case 8: return launch_sums<T, O, 8>(p, a...);
    case 16: return launch_sums<T, O, 16>(p, a...);
    case 32: return launch_sums<T, O, 32>(p, a...);
    default: return launch_sums<T, O, 64>(p, a...);
  }
}

template <class T, class Id>
void launch_embed(const void* ids, int64_t tokens, const void* weight, int64_t weight_stride,
                  int64_t vocab, int dim, float scale, void* out, hipStream_t st) {
  const int blocks = (int)ceil_div(dim, 8);
  const int64_t groups = ceil_div(tokens * blocks, 256);
  embed_kernel<T, Id><<<(uint32_t)groups, 256, 0, st>>>(
      static_cast<const Id*>(ids), tokens, static_cast<const T*>(weight), weight_stride, vocab,
      dim, blocks, scale, static_cast<T*>(out));
}

}  // namespace
}  // namespace omq_net

using namespace omq_net;

extern "C" {

int omq_token_embedding(const void* ids, int ids_are_64, int64_t tokens, const void* weight,
                        int64_t weight_stride, int64_t vocab, int64_t dim, int dtype, float scale,
                        void* out, void* stream) {
  if (!dtype_known(dtype))
    return net_fail(OMQ_NET_E_ARG, "omq_token_embedding: unknown type %d", dtype);
  if (tokens < 0 || vocab < 1 || dim < 1 || weight_stride < 0)
    return net_fail(OMQ_NET_E_ARG, "omq_token_embedding: tokens %lld, vocab %lld, dim %lld, "
                    "weight_stride %lld", (long long)tokens, (long long)vocab, (long long)dim,
                    (long long)weight_stride);
  if (tokens > OMQ_NET_MAX_COUNT || vocab > OMQ_NET_MAX_COUNT || dim > OMQ_NET_MAX_DIM ||
      ceil_div(tokens * ceil_div(dim, 8), 256) > OMQ_NET_MAX_COUNT)
    return net_fail(OMQ_NET_E_LIMIT, "omq_token_embedding: tokens %lld, vocab %lld or dim %lld "
                    "too large", (long long)tokens, (long long)vocab, (long long)dim);
  if (tokens == 0) return OMQ_NET_OK;
  if (!ids || !weight || !out)
    return net_fail(OMQ_NET_E_ARG, "omq_token_embedding: a null array");
  hipStream_t st = (hipStream_t)stream;
  const auto go = [&](auto t) {
    using T = decltype(t);
    if (ids_are_64)
      launch_embed<T, int64_t>(ids, tokens, weight, weight_stride, vocab, (int)dim, scale, out, st);
    else
      launch_embed<T, int32_t>(ids, tokens, weight, weight_stride, vocab, (int)dim, scale, out, st);
  };
  if (dtype == OMQ_NET_F32) go(float{});
  else if (dtype == OMQ_NET_BF16) go(bf16{});
  else go(f16{});
  return net_status("omq_token_embedding");
}

int64_t omq_token_embedding_grad_workspace(int64_t tokens, int64_t vocab, int64_t dim) {
  if (!grad_sizes_ok(tokens, vocab, dim)) return OMQ_NET_E_ARG;
  return grad_plan(tokens, vocab, dim).bytes;
}

int omq_token_embedding_grad(const void* grad, int64_t grad_stride, int dtype, const void* ids,
                             int ids_are_64, int64_t tokens, int64_t vocab, int64_t dim,
                             float scale, void* out, int out_dtype, void* workspace,
                             int64_t workspace_bytes, void* stream) {
  const char* name = "omq_token_embedding_grad";
  if (!dtype_known(dtype) || (out_dtype != dtype && out_dtype != OMQ_NET_F32))
    return net_fail(OMQ_NET_E_ARG, "%s: types %d -> %d", name, dtype, out_dtype);
  if (!grad_sizes_ok(tokens, vocab, dim) || grad_stride < 0)
    return net_fail(OMQ_NET_E_ARG, "%s: tokens %lld, vocab %lld, dim %lld, grad_stride %lld", name,
                    (long long)tokens, (long long)vocab, (long long)dim, (long long)grad_stride);
  const GradPlan p = grad_plan(tokens, vocab, dim);
  if (workspace_bytes < p.bytes || !workspace)
    return net_fail(OMQ_NET_E_ARG, "%s: workspace of %lld bytes, %lld needed", name,
                    (long long)workspace_bytes, (long long)p.bytes);
  if (!out || (tokens > 0 && (!grad || !ids)))
    return net_fail(OMQ_NET_E_ARG, "%s: a null array", name);
  hipStream_t st = (hipStream_t)stream;
  char* ws = static_cast<char*>(workspace);
  const uint2* pairs =
      ids_are_64 ? sort_tokens(p, static_cast<const int64_t*>(ids), tokens, vocab, ws, st)
                 : sort_tokens(p, static_cast<const int32_t*>(ids), tokens, vocab, ws, st);
  const auto go = [&](auto t) {
    using T = decltype(t);
    if (out_dtype == OMQ_NET_F32)
      launch_sums_lanes<T, float>(p, grad, grad_stride, pairs, tokens, vocab, (int)dim, scale, out,
                                  ws, st);
    else
      launch_sums_lanes<T, T>(p, grad, grad_stride, pairs, tokens, vocab, (int)dim, scale, out, ws,
                              st);
  };
  if (dtype == OMQ_NET_F32) go(float{});
  else if (dtype == OMQ_NET_BF16) go(bf16{});
  else go(f16{});
  return net_status(name);
}

}  // extern "C"
