// The token embedding with a scale, and its gradient over the sorted tokens (gfx950).
//
// Forward: a gather of rows; bound by the bytes of the output (184832 x 512 bfloat16 in 41 us,
// 4.7 TB/s).
//
// Gradient: out[v] = scale * sum of grad[t] over the tokens t of v.  The tokens are sorted by id
// (stable, so that every sum runs in ascending t), then the sorted tokens and the vocabulary's
// rows are walked as one merged list: token i comes before the end of row v when key[i] <= v.
// The list is cut into pieces of equal length, so a piece has the same work whether it holds the
// many tokens of one row or many rows without tokens.  A row that lies in one piece is written
// by it; a row that crosses pieces leaves partial sums in float32, which a second launch adds in
// the order of the pieces.  No atomics on floating-point values: the result is the same at every
// call.
//
// Measured, bfloat16: 115200 tokens of 675 rows, 256 columns 31 us (13 us sort, 14 us sums at 4.2
// TB/s, 5 us join); 131071 tokens of 65536 rows, 1024 columns 120 us (29 us sort in two passes,
// 90 us sums at 4.5 TB/s, 5 us join).  The sums are bound by memory, the sort by the latency of its
// two or three short launches a pass.
#include <type_traits>

#include "net_common.h"

namespace omq_net {
namespace {

// ---- forward --------------------------------------------------------------------------------
// A thread takes kBlocks blocks of eight columns, 256 blocks apart: their ids, then their rows are
// in flight together.
template <class T, class Id, bool kWhole, int kBlocks>
__global__ __launch_bounds__(256) void embed_kernel(const Id* __restrict__ ids, int64_t tokens,
                                                    const T* __restrict__ weight,
                                                    int64_t weight_stride, int64_t vocab,
                                                    int dim, int blocks, float scale,
                                                    T* __restrict__ out) {
  const int64_t first = block_index() * (256 * kBlocks);
  const int64_t row0 = first / blocks;
  const uint32_t in = (uint32_t)(first - row0 * blocks) + threadIdx.x;
  int64_t t[kBlocks], id[kBlocks];
  int col[kBlocks];
#pragma unroll
  for (int k = 0; k < kBlocks; ++k) {
    const uint32_t down = (in + 256 * k) / (uint32_t)blocks;
    t[k] = row0 + down;
    col[k] = 8 * (int)(in + 256 * k - down * (uint32_t)blocks);
    id[k] = (int64_t)ids[t[k] < tokens ? t[k] : tokens - 1];
  }
  Reg8<T> raw[kBlocks];
#pragma unroll
  for (int k = 0; k < kBlocks; ++k) {
    const bool in_table = id[k] >= 0 && id[k] < vocab;
    raw[k] = load_raw<T, kWhole>(weight + (in_table ? id[k] : 0) * weight_stride, col[k], dim);
  }
#pragma unroll
  for (int k = 0; k < kBlocks; ++k) {
    const bool in_table = id[k] >= 0 && id[k] < vocab;
    if (t[k] < tokens)
      store8<T, kWhole>(out + t[k] * dim, col[k], dim,
                        in_table ? widen<T, kWhole>(raw[k], col[k], dim) * scale : F8{});
  }
}

// ---- sort -----------------------------------------------------------------------------------
// A pair is (key, token).  Keys lie in [0, vocab]; `vocab` stands for an id outside the
// vocabulary, so those tokens sort behind all others.
constexpr int kMaxDigitBits = 11;
constexpr int kTile = 1024;       // tokens of a workgroup of the radix passes
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

// All passes of up to kTokens tokens in one workgroup.  8-bit digits.
template <class Id, int kTokens>
__global__ __launch_bounds__(1024) void sort_small_kernel(const Id* __restrict__ ids, int tokens,
                                                          int64_t vocab, int bits,
                                                          uint2* __restrict__ pairs) {
  constexpr int kThreads = 1024, kRounds = kTokens / kThreads, kWaves = kThreads / kWave;
  __shared__ uint2 kept[kThreads * kRounds];
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
    for (int j = threadIdx.x; j < kWaves * 256; j += kThreads) (&next[0][0])[j] = 0;
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
    block_scan<kThreads>(base, 256, wave_sums);
    for (int j = threadIdx.x; j < kWaves * 256; j += kThreads) (&next[0][0])[j] += base[j & 255];
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

// Radix pass, step 1: counts[tile * bins + digit].
template <class Id>
__global__ __launch_bounds__(256) void digit_counts_kernel(const Id* __restrict__ ids,
                                                           const uint2* __restrict__ in,
                                                           int64_t tokens, int64_t vocab,
                                                           int shift, int bits, int bins,
                                                           uint32_t* __restrict__ counts) {
  __shared__ uint32_t hist[1 << kMaxDigitBits];
  const uint32_t mask = (1u << bits) - 1;
  const int64_t first = (int64_t)blockIdx.x * kTile;
  uint32_t key[kTile / 256];
#pragma unroll
  for (int r = 0; r < kTile / 256; ++r) {
    const int64_t t = first + r * 256 + threadIdx.x;
    if (t < tokens) key[r] = in ? in[t].x : key_of(ids, t, vocab);
  }
  for (int j = threadIdx.x; j < bins; j += 256) hist[j] = 0;
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kTile / 256; ++r)
    if (first + r * 256 + threadIdx.x < tokens)
      atomicAdd(&hist[(key[r] >> shift) & mask], 1u);
  __syncthreads();
  for (int j = threadIdx.x; j < bins; j += 256) counts[(int64_t)blockIdx.x * bins + j] = hist[j];
}

// Step 2: per digit, the exclusive prefix sums over the tiles, and the total.  A workgroup takes
// 64 digits; its 16 waves take a sixteenth of the tiles each.
__global__ __launch_bounds__(1024) void digit_scan_kernel(uint32_t* __restrict__ counts, int tiles,
                                                          int bins, uint32_t* __restrict__ totals) {
  __shared__ uint32_t sums[16][kWave];
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const int digit = blockIdx.x * kWave + lane;
  const int per = (tiles + 15) / 16;
  const int from = wave * per < tiles ? wave * per : tiles;
  const int to = from + per < tiles ? from + per : tiles;
  // (eight loads in flight, the last ones too)
  const uint32_t* column = counts + (digit < bins ? digit : bins - 1);
  const auto eight = [&](int t, uint32_t (&c)[8]) {
#pragma unroll
    for (int u = 0; u < 8; ++u) c[u] = column[(int64_t)(t + u < to ? t + u : to - 1) * bins];
  };
  uint32_t held[8], sum = 0;  // the first eight, for the second time too
  eight(from, held);
  const auto add = [&](int t, const uint32_t (&c)[8]) {
#pragma unroll
    for (int u = 0; u < 8; ++u) sum += t + u < to ? c[u] : 0u;
  };
  add(from, held);
  for (int t = from + 8; t < to; t += 8) {
    uint32_t c[8];
    eight(t, c);
    add(t, c);
  }
  sums[wave][lane] = sum;
  __syncthreads();
  uint32_t base = 0;
  for (int w = 0; w < wave; ++w) base += sums[w][lane];
  if (digit >= bins) return;
  if (wave == 15) totals[digit] = base + sum;
  const auto put = [&](int t, const uint32_t (&c)[8]) {
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (t + u < to) {
        counts[(int64_t)(t + u) * bins + digit] = base;
        base += c[u];
      }
  };
  put(from, held);
  for (int t = from + 8; t < to; t += 8) {
    uint32_t c[8];
    eight(t, c);
    put(t, c);
  }
}

// Step 3: every pair to its place.  Eight waves of two rounds; the waves' counters of a tile have
// 16 bits, two to a word.  (5.4 to 6.2 us for 115200 tokens, 6.9 to 8 with four waves of four
// rounds and counters of 32 bits.)
//
// kScan: there was no step 2; the tiles are few (kScanTiles), and every workgroup adds the counts
// of its digits over all of them itself.  16 tiles and two passes: 32 us for the whole gradient, 36
// with step 2; 32 tiles: one pass 26.4 and 25.8, two passes 40 and 42; 113 tiles: 41 and 32.
constexpr int kScanTiles = 32;

template <class Id, bool kScan>
__global__ __launch_bounds__(512) void digit_scatter_kernel(
    const Id* __restrict__ ids, const uint2* __restrict__ in, int64_t tokens, int64_t vocab,
    int shift, int bits, int bins, const uint32_t* __restrict__ counts,
    const uint32_t* __restrict__ totals, uint2* __restrict__ out) {
  constexpr int kThreads = 512, kWaves = kThreads / kWave, kRounds = kTile / kThreads;
  constexpr int kBins = 1 << kMaxDigitBits;
  __shared__ uint32_t next[kWaves][kBins / 2];
  __shared__ uint32_t base[kBins];
  __shared__ uint32_t wave_sums[kWaves];
  const uint32_t mask = (1u << bits) - 1;
  const int wave = threadIdx.x / kWave, lane = threadIdx.x & (kWave - 1);
  const int64_t first = (int64_t)blockIdx.x * kTile + wave * (kTile / kWaves);
  const int words = (bins + 1) / 2;
  uint2 mine[kRounds];
  uint32_t before[kBins / kThreads];  // of this thread's digits, in the tiles before
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const int64_t t = first + r * kWave + lane;
    if (t < tokens) mine[r] = in ? in[t] : make_uint2(key_of(ids, t, vocab), (uint32_t)t);
  }
#pragma unroll
  for (int k = 0; k < kBins / kThreads; ++k) {
    const int j = k * kThreads + threadIdx.x;
    if (j < bins && kScan) {
      uint32_t sum = 0, ahead = 0;
      for (int t = 0; t < (int)gridDim.x; t += 8) {  // eight loads in flight, the last ones too
        uint32_t c[8];
#pragma unroll
        for (int u = 0; u < 8; ++u)
          c[u] = counts[(int64_t)(t + u < (int)gridDim.x ? t + u : t) * bins + j];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          sum += t + u < (int)gridDim.x ? c[u] : 0u;
          ahead += t + u < (int)blockIdx.x ? c[u] : 0u;
        }
      }
      before[k] = ahead;
      base[j] = sum;
    } else if (j < bins) {
      before[k] = counts[(int64_t)blockIdx.x * bins + j];
      base[j] = totals[j];
    }
  }
  for (int j = threadIdx.x; j < words; j += kThreads)
#pragma unroll
    for (int w = 0; w < kWaves; ++w) next[w][j] = 0;
  __syncthreads();
  block_scan<kThreads>(base, bins, wave_sums);
#pragma unroll
  for (int r = 0; r < kRounds; ++r)
    if (first + r * kWave + lane < tokens) {
      const uint32_t d = (mine[r].x >> shift) & mask;
      atomicAdd(&next[wave][d >> 1], 1u << (16 * (d & 1)));
    }
#pragma unroll
  for (int k = 0; k < kBins / kThreads; ++k) {
    const int j = k * kThreads + threadIdx.x;
    if (j < bins) base[j] += before[k];
  }
  __syncthreads();
  for (int j = threadIdx.x; j < words; j += kThreads) {
    uint32_t at = 0, c[kWaves];
#pragma unroll
    for (int w = 0; w < kWaves; ++w) c[w] = next[w][j];
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      next[w][j] = at;
      at += c[w];  // (both halves: a tile has fewer than 2^16 pairs)
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const bool here = first + r * kWave + lane < tokens;
    const uint32_t d = here ? (mine[r].x >> shift) & mask : 0u;
    const uint64_t same = match_digit(d, bits, __ballot(here));
    const int below = lanes_below(same);
    uint32_t* word = &next[wave][d >> 1];
    uint32_t at = 0;
    if (here) at = base[d] + ((*word >> (16 * (d & 1))) & 0xFFFFu) + below;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (here && below == 0) atomicAdd(word, (uint32_t)__popcll(same) << (16 * (d & 1)));
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
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

// The numbers of tokens among the first at[0] and at[1] items of the merged list: two searches
// side by side, in each of which the kLanes lanes of a piece probe together, so that a step
// leaves 1/(kLanes+1) of the range.
template <int kLanes>
__device__ inline void tokens_before(const uint2* pairs, int64_t tokens, int64_t vocab,
                                     const int64_t (&at)[2], int64_t (&found)[2]) {
  int64_t lo[2], hi[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    lo[k] = at[k] > vocab ? at[k] - vocab : 0;
    hi[k] = at[k] < tokens ? at[k] : tokens;
  }
  const int lane = threadIdx.x & (kLanes - 1);
  const int shift = (threadIdx.x & (kWave - 1)) & ~(kLanes - 1);
  while (__any(lo[0] < hi[0] || lo[1] < hi[1])) {  // (until the last piece of the wave is done)
    bool before[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      // probe lo + n*(lane+1)/(kLanes+1), in [lo, hi): is that token among the first `at` items?
      const int64_t n = hi[k] - lo[k], i = lo[k] + n * (lane + 1) / (kLanes + 1);
      before[k] = n > 0 && (int64_t)pairs[i].x <= at[k] - i - 1;
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {  // true for a prefix of the probes
      const int64_t n = hi[k] - lo[k];
      const uint64_t all = __ballot(before[k]) >> shift;
      const int count = __popcll(kLanes == 64 ? all : all & ((1ull << (kLanes & 63)) - 1));
      if (n > 0) {
        const int64_t from = lo[k];
        if (count > 0) lo[k] = from + n * count / (kLanes + 1) + 1;
        if (count < kLanes) hi[k] = from + n * (count + 1) / (kLanes + 1);
      }
    }
  }
  found[0] = lo[0];
  found[1] = lo[1];
}

// The value that lane `from` of this lane's group of kLanes holds; uniform over a whole wave
// where the group is one (the loops over it are scalar then).
template <int kLanes>
__device__ inline uint32_t group_read(uint32_t v, int from) {
  if constexpr (kLanes == kWave) return (uint32_t)__builtin_amdgcn_readlane((int)v, from);
  return (uint32_t)__shfl((int)v, from, kLanes);
}

template <int kLanes>
__device__ inline int64_t group_uniform(int64_t v) {
  if constexpr (kLanes == kWave) {
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)v);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(v >> 32));
    return (int64_t)((uint64_t)hi << 32 | lo);
  }
  return v;
}

template <class T, class O, int kLanes, bool kWhole>
__global__ __launch_bounds__(256) void sum_pieces_kernel(
    const T* __restrict__ grad, int64_t grad_stride, const uint2* __restrict__ pairs,
    int64_t tokens, int64_t vocab, int dim, float scale, int64_t piece, int64_t pieces,
    O* __restrict__ out, Piece* __restrict__ info, float* __restrict__ heads,
    float* __restrict__ tails) {
  constexpr int kBatch = 8;  // rows of `grad` in flight
  int64_t c = (int64_t)blockIdx.x * (256 / kLanes) + threadIdx.x / kLanes;
  if constexpr (kLanes == kWave)
    c = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int lane = threadIdx.x & (kLanes - 1);
  const int col = 8 * (int)(blockIdx.y * kLanes + lane);
  const int64_t items = tokens + vocab;
  const int64_t d0 = c * piece < items ? c * piece : items;
  const int64_t d1 = d0 + piece < items ? d0 + piece : items;
  const int64_t ends[2] = {d0, d1};
  int64_t at[2];
  tokens_before<kLanes>(pairs, tokens, vocab, ends, at);
  const int64_t i0 = group_uniform<kLanes>(at[0]), i1 = group_uniform<kLanes>(at[1]);
  if (c >= pieces) return;
  const int64_t row0 = d0 - i0, row1 = d1 - i1;
  const bool shared = row0 < vocab && i0 > 0 && (int64_t)pairs[i0 - 1].x == row0;
  int64_t row = row0;
  F8 acc = {};
  bool open = false;
  const auto end_row = [&]() {
    if (shared && row == row0)
      store8<float, kWhole>(heads + c * dim, col, dim, acc);
    else
      store8<O, kWhole>(out + row * dim, col, dim, acc * scale);
    acc = F8{};
    open = false;
    ++row;
  };
  for (int64_t i = i0; i < i1; i += kLanes) {
    const uint2 mine = i + lane < i1 ? pairs[i + lane] : make_uint2(0u, 0u);
    const int here = i1 - i < kLanes ? (int)(i1 - i) : kLanes;
    for (int k = 0; k < here; k += kBatch) {
      Reg8<T> v[kBatch];
      uint32_t key[kBatch];
#pragma unroll
      for (int e = 0; e < kBatch; ++e) {
        const int at = k + e < here ? k + e : here - 1;
        key[e] = group_read<kLanes>(mine.x, at);
        const uint32_t token = group_read<kLanes>(mine.y, at);
        v[e] = load_raw<T, kWhole>(grad + (int64_t)token * grad_stride, col, dim);
      }
#pragma unroll
      for (int e = 0; e < kBatch; ++e)
        if (k + e < here && (int64_t)key[e] < vocab) {
          while (row < (int64_t)key[e]) end_row();
          acc += widen<T, kWhole>(v[e], col, dim);
          open = true;
        }
    }
  }
  while (row < row1) end_row();
  if (open) store8<float, kWhole>(tails + c * dim, col, dim, acc);
  if (blockIdx.y == 0 && lane == 0)
    info[c] = Piece{shared && row1 > row0 ? (int32_t)row0 : -1, (int32_t)row1, open ? 1 : 0, 0};
}

// The rows that a piece ends and did not begin: the sums that the pieces before it left open (its
// run), in their order, then its own.  A wave takes a piece and 256 columns, four a lane; a run of
// more than kOwnRun pieces is taken by all 16 waves of the workgroup, every 16th piece each, and
// their sums are added in order.
constexpr int kJoinWaves = 16, kOwnRun = 32;

template <class O>
__global__ __launch_bounds__(1024) void join_pieces_kernel(const Piece* __restrict__ info,
                                                           int64_t pieces, int dim, float scale,
                                                           const float* __restrict__ heads,
                                                           const float* __restrict__ tails,
                                                           O* __restrict__ out) {
  using F4 = float __attribute__((ext_vector_type(4)));
  __shared__ F4 part[kJoinWaves][kWave];
  __shared__ int64_t run_from[kJoinWaves];  // of the long runs, else -1
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int64_t c0 = (int64_t)blockIdx.x * kJoinWaves;
  const int col = 4 * ((int)blockIdx.y * kWave + lane);
  const auto four = [&](const float* p) {
    F4 v = {};
    if (col + 3 < dim) {
      using F4u __attribute__((aligned(4))) = F4;
      v = *reinterpret_cast<const F4u*>(p + col);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (col + j < dim) v[j] = p[col + j];
    }
    return v;
  };
  const auto sum = [&](F4 acc, int64_t from, int64_t to, int step) {
    for (int64_t k = from; k < to; k += 8 * step) {  // eight loads in flight, the last ones too
      F4 v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = four(tails + (k + u * step < to ? k + u * step : k) * dim);
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (k + u * step < to) acc += v[u];
    }
    return acc;
  };
  const auto write = [&](int64_t row, F4 acc) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (col + j < dim) out[row * dim + col + j] = (O)(acc[j] * scale);
  };
  const int64_t c = c0 + wave;
  // lane 0: piece c - 1, lane 1: the one before, ...
  const Piece own = c < pieces ? info[c] : Piece{-1, 0, 0, 0};
  const Piece near = c < pieces && c - 1 - lane >= 0 ? info[c - 1 - lane] : Piece{-1, -1, 0, 0};
  const int32_t row = own.first_row;
  int64_t long_from = -1;
  if (row >= 0) {
    // the run: the pieces just before c at whose end `row` is open
    const uint64_t all = __ballot(near.last_row == row);
    int64_t from;
    bool open;  // the first may end with the end of the row before; the others left something
    if (~all != 0) {
      const int n = __builtin_ctzll(~all);
      from = c - n;
      open = (__ballot(near.open != 0) >> (n - 1)) & 1;
    } else {  // the first of all pieces whose last row is `row` or a later one
      int64_t lo = 0, hi = c - kWave;
      while (lo < hi) {
        const int64_t n = hi - lo, i = lo + n * (lane + 1) / (kWave + 1);
        const int below = __popcll(__ballot(info[i].last_row < row));
        const int64_t was = lo;
        if (below > 0) lo = was + n * below / (kWave + 1) + 1;
        if (below < kWave) hi = was + n * (below + 1) / (kWave + 1);
      }
      from = lo;
      open = info[from].open;
    }
    if (!open) ++from;
    const F4 head = four(heads + c * dim);
    if (c - from <= kOwnRun)
      write(row, sum(F4{}, from, c, 1) + head);
    else
      long_from = from;
  }
  if (lane == 0) run_from[wave] = long_from;
  __syncthreads();
  for (int w = 0; w < kJoinWaves; ++w) {
    const int64_t from = run_from[w];
    if (from < 0) continue;
    F4 acc = sum(F4{}, from + wave, c0 + w, kJoinWaves);
    part[wave][lane] = acc;
    __syncthreads();
    if (wave == 0) {
      for (int k = 1; k < kJoinWaves; ++k) acc += part[k][lane];
      write(info[c0 + w].first_row, acc + four(heads + (c0 + w) * dim));
    }
    __syncthreads();
  }
}

// ---- few tokens -----------------------------------------------------------------------------
// Few tokens take one launch: a workgroup has some rows of the vocabulary (and 512 columns), lists
// the tokens of those rows out of all in their order, and its waves take a row each in turn; a row
// of more than kHotRow tokens is taken by all waves, a stretch of the list each, whose sums are
// added in order.
//
// Up to 1024 tokens, and up to kListedTokens where the vocabulary's rows have four or fewer on
// average.  The work of a row of many tokens is not spread over workgroups here, so that more
// tokens are sorted: 225 tokens of 675 rows and 128 columns take 5 us a call (15 sorted), 1000 of
// 1083 rows 5 us (18), 1734 of 867 rows 5.5 us (24); but 2048 of two rows 43 us (17), 8000 of 1000
// rows unevenly 91 us (24).  A workgroup has a wave's row at least, so that few rows are few
// workgroups.  With 1024 columns, listed and sorted, us:
//                  2 rows      16 rows     64 rows     675 rows
//   256 tokens     13   14.5   6    15     5.3  14.5   5.3  17
//   512 tokens     17   15.5   15   15     7    16     5.4  18
//   1024 tokens    23   17     47   15.5   10   16     5.3  19
// (The smallest board's table has 147 rows.)
constexpr int kListedTokens = 2048, kHotRow = 64;

bool use_list(int64_t tokens, int64_t vocab) {
  return tokens <= 1024 || (tokens <= kListedTokens && tokens <= 4 * vocab);
}

template <class T, class O, class Id, bool kWhole, int kThreads>
__global__ __launch_bounds__(kThreads) void sum_listed_kernel(
    const T* __restrict__ grad, int64_t grad_stride, const Id* __restrict__ ids, int tokens,
    int64_t vocab, int dim, float scale, int rows, O* __restrict__ out) {
  constexpr int kBatch = 8;  // rows of `grad` in flight
  constexpr int kWaves = kThreads / kWave;
  extern __shared__ uint32_t listed[];  // [tokens] rows, then [tokens] tokens of 16 bits
  __shared__ int counts[2][kWaves];
  __shared__ F8 joined[kWave];
  __shared__ int hot[kListedTokens / kHotRow], hot_rows;
  uint32_t* row_of = listed;
  uint16_t* token_of = reinterpret_cast<uint16_t*>(listed + tokens);
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int64_t row0 = (int64_t)blockIdx.x * rows;
  const int64_t end = row0 + rows < vocab ? row0 + rows : vocab;
  if (threadIdx.x == 0) hot_rows = 0;
  int total = 0;
  int64_t next = (int)threadIdx.x < tokens ? (int64_t)ids[threadIdx.x] : -1;
  for (int base = 0, turn = 0; base < tokens; base += kThreads, turn ^= 1) {
    const int64_t id = next;
    const int ahead = base + kThreads + (int)threadIdx.x;
    next = ahead < tokens ? (int64_t)ids[ahead] : -1;
    const bool mine = id >= row0 && id < end;
    const uint64_t here = __ballot(mine);
    if (lane == 0) counts[turn][wave] = __popcll(here);
    __syncthreads();
    int place = total + lanes_below(here);
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const int c = counts[turn][w];
      place += w < wave ? c : 0;
      total += c;
    }
    if (mine) {
      token_of[place] = (uint16_t)(base + threadIdx.x);
      row_of[place] = (uint32_t)(id - row0);
    }
  }
  __syncthreads();
  total = __builtin_amdgcn_readfirstlane(total);
  const int col = 8 * ((int)blockIdx.y * kWave + lane);
  const auto matches = [&](int r, int base, int to, uint32_t* token) {
    const bool there = base + lane < to;
    *token = there ? token_of[base + lane] : 0u;
    return __ballot(there && row_of[base + lane] == (uint32_t)r);
  };
  const auto add = [&](F8 acc, int r, int from, int to) {  // the list's stretch [from, to)
    for (int base = from; base < to; base += kWave) {
      uint32_t token;
      uint64_t mine = matches(r, base, to, &token);
      while (mine) {
        Reg8<T> v[kBatch];
        const int n = __popcll(mine);
#pragma unroll
        for (int e = 0; e < kBatch; ++e) {  // (the last one again where there are no more)
          const uint32_t t =
              (uint32_t)__builtin_amdgcn_readlane((int)token, __builtin_ctzll(mine));
          v[e] = load_raw<T, kWhole>(grad + (int64_t)t * grad_stride, col, dim);
          if (mine & (mine - 1)) mine &= mine - 1;
        }
#pragma unroll
        for (int e = 0; e < kBatch; ++e)
          if (e < n) acc += widen<T, kWhole>(v[e], col, dim);
        if (n <= kBatch) mine = 0;
      }
    }
    return acc;
  };
  const auto put = [&](int r, F8 acc) {
    store8<O, kWhole>(out + (row0 + r) * dim, col, dim, acc * scale);
  };
  for (int r = wave; row0 + r < end; r += kWaves) {
    int n = total;
    if (total > kHotRow) {
      n = 0;
      uint32_t token;
      for (int base = 0; base < total; base += kWave)
        n += __popcll(matches(r, base, total, &token));
    }
    if (n <= kHotRow)
      put(r, n ? add(F8{}, r, 0, total) : F8{});
    else if (lane == 0)
      hot[atomicAdd(&hot_rows, 1)] = r;
  }
  __syncthreads();
  const int stretch = (total + kThreads - 1) / kThreads * kWave;  // of whole waves
  for (int h = 0; h < hot_rows; ++h) {
    const int r = __builtin_amdgcn_readfirstlane(hot[h]);
    const int from = wave * stretch < total ? wave * stretch : total;
    const F8 acc = add(F8{}, r, from, from + stretch < total ? from + stretch : total);
    for (int w = 0; w < kWaves; ++w) {
      if (w == wave) joined[lane] = w ? joined[lane] + acc : acc;
      __syncthreads();
    }
    if (wave == 0) put(r, joined[lane]);
    __syncthreads();
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

// One workgroup's sort is one launch, a pass of the radix sort two.  1100 tokens of 200 rows and
// 1024 columns take 15.8 us a call with it (19 without; 16.8 with the larger one's registers); 3000
// of 50000 rows and 256 columns, whose radix sort has two passes, 24.7 us (30.3); but 4096 of 1000
// rows, which it has to pass twice and the radix sort once, 25.5 us (22.5), and 2048 of 400 rows,
// the same, 21 us (20.2).
bool use_small_sort(int64_t tokens, int passes) {
  return tokens <= (passes > 1 ? kSmallSort : kSmallSort / 2);
}

GradPlan grad_plan(int64_t tokens, int64_t vocab, int64_t dim) {
  GradPlan p{};
  if (use_list(tokens, vocab)) return p;  // (no workspace)
  while (p.bits < 32 && (vocab >> p.bits) != 0) ++p.bits;
  p.passes = (int)ceil_div(p.bits, kMaxDigitBits);
  p.digit_bits = (int)ceil_div(p.bits, p.passes);
  p.tiles = ceil_div(tokens, kTile);
  p.lanes = dim <= 64 ? 8 : dim <= 128 ? 16 : dim <= 256 ? 32 : 64;
  p.col_tiles = (int)ceil_div(dim, 8 * p.lanes);
  // Pieces for 2048 waves, of 16 to 1024 items.  Fewer leave memory idle, more are more partial
  // sums: 115200 tokens of 675 rows and 256 columns take 32 us, 36 with 1024 waves and 38 with
  // 4096; 131071 of 65536 rows and 1024 columns 116, 129 and 122.
  const int64_t items = tokens + vocab;
  const int64_t wanted = ceil_div(2048ll * (kWave / p.lanes), p.col_tiles);
  p.piece = ceil_div(items, wanted);
  p.piece = p.piece < 16 ? 16 : p.piece > 1024 ? 1024 : p.piece;
  p.pieces = ceil_div(items, p.piece);
  int64_t at = 0;
  p.at_pairs[0] = take(&at, 8 * tokens);
  const bool radix = !use_small_sort(tokens, p.passes);
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
  if (use_small_sort(tokens, p.passes)) {
    const auto sort = tokens <= kSmallSort / 2 ? sort_small_kernel<Id, kSmallSort / 2>
                                               : sort_small_kernel<Id, kSmallSort>;
    sort<<<1, 1024, 0, st>>>(ids, (int)tokens, vocab, p.bits, buf[0]);
    return buf[0];
  }
  uint32_t* counts = reinterpret_cast<uint32_t*>(ws + p.at_counts);
  uint32_t* totals = reinterpret_cast<uint32_t*>(ws + p.at_totals);
  const uint2* in = nullptr;
  for (int pass = 0; pass < p.passes; ++pass) {
    uint2* to = buf[pass & 1];
    // the digits that occur: the largest key is `vocab`
    const int shift = pass * p.digit_bits;
    const int64_t top = (vocab >> shift) + 1, all = 1 << p.digit_bits;
    const int bins = (int)(top < all ? top : all);
    digit_counts_kernel<Id><<<(uint32_t)p.tiles, 256, 0, st>>>(ids, in, tokens, vocab, shift,
                                                              p.digit_bits, bins, counts);
    const bool scan = p.tiles <= kScanTiles;
    if (!scan)
      digit_scan_kernel<<<(uint32_t)ceil_div(bins, kWave), 1024, 0, st>>>(counts, (int)p.tiles,
                                                                        bins, totals);
    const auto scatter = scan ? digit_scatter_kernel<Id, true> : digit_scatter_kernel<Id, false>;
    scatter<<<(uint32_t)p.tiles, 512, 0, st>>>(
        ids, in, tokens, vocab, shift, p.digit_bits, bins, counts, totals, to);
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
  const auto kernel = dim % 8 == 0 ? sum_pieces_kernel<T, O, kLanes, true>
                                   : sum_pieces_kernel<T, O, kLanes, false>;
  kernel<<<grid, 256, 0, st>>>(
      static_cast<const T*>(grad), grad_stride, pairs, tokens, vocab, dim, scale, p.piece,
      p.pieces, static_cast<O*>(out), info, heads, tails);
  if (p.pieces > 1)
    join_pieces_kernel<O><<<dim3((uint32_t)ceil_div(p.pieces, kJoinWaves),
                                 (uint32_t)ceil_div(dim, 4 * kWave)),
                            1024, 0, st>>>(info, p.pieces, dim, scale, heads, tails,
                                           static_cast<O*>(out));
}

template <class T, class O, class Id, bool kWhole>
void launch_listed(const void* grad, int64_t grad_stride, const void* ids, int tokens,
                   int64_t vocab, int dim, float scale, void* out, hipStream_t st) {
  const auto go = [&](auto kernel, int threads, int64_t groups) {
    const int64_t col_tiles = ceil_div(dim, 8 * kWave), waves = threads / kWave;
    const int64_t rows = ceil_div(ceil_div(vocab * col_tiles, groups), waves) * waves;
    const dim3 grid((uint32_t)ceil_div(vocab, rows), (uint32_t)col_tiles);
    kernel<<<grid, threads, 6 * tokens, st>>>(
        static_cast<const T*>(grad), grad_stride, static_cast<const Id*>(ids), tokens, vocab, dim,
        scale, (int)rows, static_cast<O*>(out));
  };
  if (tokens <= 256)
    go(sum_listed_kernel<T, O, Id, kWhole, 256>, 256, 2048);
  else
    go(sum_listed_kernel<T, O, Id, kWhole, 1024>, 1024, 1024);
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
  // Four blocks a thread once there are enough for four workgroups a compute unit all the same:
  // 184832 rows of 512 bfloat16 take 41 us so and 56 us with one each.
  const bool many = tokens * blocks >= 256 * 4 * 1024;
  const int64_t groups = ceil_div(tokens * blocks, many ? 1024 : 256);
  const auto kernel = dim % 8 == 0 ? (many ? embed_kernel<T, Id, true, 4> : embed_kernel<T, Id, true, 1>)
                                   : (many ? embed_kernel<T, Id, false, 4> : embed_kernel<T, Id, false, 1>);
  kernel<<<grid_of(groups, 256), 256, 0, st>>>(
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
  if (p.bytes > 0 && (workspace_bytes < p.bytes || !workspace))
    return net_fail(OMQ_NET_E_ARG, "%s: workspace of %lld bytes, %lld needed", name,
                    (long long)workspace_bytes, (long long)p.bytes);
  if (p.bytes > 0 && !on_16_bytes(workspace))
    return net_fail(OMQ_NET_E_ARG, "%s: workspace is not on a 16-byte boundary", name);
  if (!out || (tokens > 0 && (!grad || !ids)))
    return net_fail(OMQ_NET_E_ARG, "%s: a null array", name);
  hipStream_t st = (hipStream_t)stream;
  char* ws = static_cast<char*>(workspace);
  const bool listed = use_list(tokens, vocab);
  const uint2* pairs = nullptr;
  if (!listed)
    pairs = ids_are_64 ? sort_tokens(p, static_cast<const int64_t*>(ids), tokens, vocab, ws, st)
                       : sort_tokens(p, static_cast<const int32_t*>(ids), tokens, vocab, ws, st);
  const auto sums = [&](auto t, auto o) {
    using T = decltype(t);
    using O = decltype(o);
    const auto go = [&](auto id, auto whole) {
      launch_listed<T, O, decltype(id), whole.value>(grad, grad_stride, ids, (int)tokens, vocab,
                                                     (int)dim, scale, out, st);
    };
    using Yes = std::true_type;
    using No = std::false_type;
    if (listed && ids_are_64)
      dim % 8 == 0 ? go(int64_t{}, Yes{}) : go(int64_t{}, No{});
    else if (listed)
      dim % 8 == 0 ? go(int32_t{}, Yes{}) : go(int32_t{}, No{});
    else
      launch_sums_lanes<T, O>(p, grad, grad_stride, pairs, tokens, vocab, (int)dim, scale, out, ws,
                              st);
  };
  const auto go = [&](auto t) { out_dtype == OMQ_NET_F32 ? sums(t, float{}) : sums(t, t); };
  if (dtype == OMQ_NET_F32) go(float{});
  else if (dtype == OMQ_NET_BF16) go(bf16{});
  else go(f16{});
  return net_status(name);
}

}  // extern "C"
