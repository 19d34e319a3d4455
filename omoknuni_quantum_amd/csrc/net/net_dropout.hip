// Dropout from a counter-based generator (gfx950): the mask is a function of the element's
// position, formed where it is needed and never stored.  Bound by memory: each element is read
// and written once, 65536 x 4096 bfloat16 in 173 us (6.2 TB/s).  A lane takes eight elements of a
// row, two words of the generator: four 64-bit products, which fit under the memory's time because
// a word serves four elements.
#include "net_common.h"

namespace omq_net {

int check_dropout(const char* name, double p);

namespace {

template <class T, bool kWhole>
__global__ __launch_bounds__(256) void dropout_kernel(const T* x, int64_t rows, int dim,
                                                      int blocks, Dropout d, T* out) {
  const int64_t first = block_index() * 256;
  const int64_t row0 = first / blocks;
  const uint32_t in = (uint32_t)(first - row0 * blocks) + threadIdx.x;
  const int64_t row = row0 + in / (uint32_t)blocks;
  const int col = 8 * (int)(in % (uint32_t)blocks);
  if (row >= rows) return;
  const F8 v = widen<T, kWhole>(load_raw<T, kWhole>(x + row * dim, col, dim), col, dim);
  store8<T, kWhole>(out + row * dim, col, dim, drop8(v, d, drop_row(d, row, dim), col));
}

}  // namespace
}  // namespace omq_net

using namespace omq_net;

extern "C" int omq_dropout(const void* x, int64_t rows, int64_t dim, int dtype, double p,
                           uint64_t seed, uint64_t offset, void* out, void* stream) {
  const char* name = "omq_dropout";
  if (!dtype_known(dtype)) return net_fail(OMQ_NET_E_ARG, "%s: unknown type %d", name, dtype);
  if (int rc = check_dropout(name, p)) return rc;
  if (rows < 0 || dim < 1)
    return net_fail(OMQ_NET_E_ARG, "%s: rows %lld, dim %lld", name, (long long)rows,
                    (long long)dim);
  if (rows > OMQ_NET_MAX_COUNT || dim > OMQ_NET_MAX_DIM ||
      ceil_div(rows * ceil_div(dim, 8), 256) > OMQ_NET_MAX_COUNT)
    return net_fail(OMQ_NET_E_LIMIT, "%s: rows %lld, dim %lld too large", name, (long long)rows,
                    (long long)dim);
  if (rows == 0) return OMQ_NET_OK;
  if (!x || !out) return net_fail(OMQ_NET_E_ARG, "%s: a null array", name);
  const Dropout d = make_dropout(p, seed, offset);
  const int blocks = (int)ceil_div(dim, 8);
  const dim3 grid = grid_of(ceil_div(rows * blocks, 256), 256);
  hipStream_t st = (hipStream_t)stream;
  const auto go = [&](auto t) {
    using T = decltype(t);
    const auto kernel = dim % 8 == 0 ? dropout_kernel<T, true> : dropout_kernel<T, false>;
    kernel<<<grid, 256, 0, st>>>(static_cast<const T*>(x), rows, (int)dim, blocks, d,
                                 static_cast<T*>(out));
  };
  if (dtype == OMQ_NET_F32) go(float{});
  else if (dtype == OMQ_NET_BF16) go(bf16{});
  else go(f16{});
  return net_status(name);
}
