// The torch operators of the policy network (libomq_net_torch.so, loaded with
// torch.ops.load_library): each checks its tensors, allocates its outputs and its workspace from
// torch's allocator and calls the C ABI (omq_net_ops.h) on the caller's current HIP stream.
//
//   omq_net::token_embedding, omq_net::token_embedding_grad
//   omq_net::add_rms_norm, omq_net::add_rms_norm_fp8, omq_net::add_rms_norm_grad
//   omq_net::dropout
//   omq_net::clipped_policy_loss, omq_net::clipped_policy_loss_grad, omq_net::clipped_policy_loss_with_grad
//
// Tensors must be on one HIP device; host tensors are refused (there is no CPU implementation).
// On meta tensors the operators give the shapes only.
#include <torch/library.h>

#include <ATen/EmptyTensor.h>
#include <ATen/core/Tensor.h>
#include <ATen/hip/impl/HIPCachingAllocatorMasqueradingAsCUDA.h>
#include <ATen/ops/empty.h>
#include <c10/hip/HIPGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>

#include <array>
#include <optional>
#include <string>
#include <tuple>

#include "omq_net_ops.h"

namespace {

using OptTensor = std::optional<at::Tensor>;

const at::Tensor* get(const OptTensor& t) {
  return t.has_value() && t->defined() ? &*t : nullptr;
}

void check_rc(int rc, const char* what) {
  TORCH_CHECK(rc == OMQ_NET_OK, what, ": ", omq_net_last_error());
}

// The tensors' common device: a HIP device, or meta.
c10::Device common_device(const char* name, std::initializer_list<const at::Tensor*> ts) {
  const c10::Device dev = (*ts.begin())->device();
  TORCH_CHECK(dev.is_cuda() || dev.is_meta(), "omq_net::", name,
              ": tensors must be on a HIP device (got ", dev, ")");
  for (const at::Tensor* t : ts)
    if (t) TORCH_CHECK(t->device() == dev, "omq_net::", name, ": all tensors must be on ", dev);
  return dev;
}

int type_of(const char* name, const char* arg, const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return OMQ_NET_F32;
    case at::kBFloat16: return OMQ_NET_BF16;
    case at::kHalf: return OMQ_NET_F16;
    default: break;
  }
  TORCH_CHECK(false, "omq_net::", name, ": ", arg, " must be float32, bfloat16 or float16, not ",
              t.scalar_type());
}

bool ids_are_64(const char* name, const char* arg, const at::Tensor& t) {
  TORCH_CHECK(t.scalar_type() == at::kInt || t.scalar_type() == at::kLong, "omq_net::", name, ": ",
              arg, " must be int32 or int64, not ", t.scalar_type());
  TORCH_CHECK(t.is_contiguous(), "omq_net::", name, ": ", arg, " must be contiguous");
  return t.scalar_type() == at::kLong;
}

// The distance between the rows of a tensor of rows along its last dimension: its elements must
// be adjacent and its leading dimensions one run of equally spaced rows.
int64_t row_stride(const char* name, const char* arg, const at::Tensor& t) {
  if (t.is_contiguous()) return t.size(-1);
  int64_t stride = -1, expected = 0;
  bool ok = t.size(-1) == 1 || t.stride(-1) == 1;
  for (int64_t i = t.dim() - 2; i >= 0; --i) {
    if (t.size(i) == 1) continue;
    if (stride < 0)
      stride = t.stride(i);
    else
      ok = ok && t.stride(i) == expected;
    expected = t.stride(i) * t.size(i);
  }
  TORCH_CHECK(ok, "omq_net::", name, ": the rows of ", arg,
              " must have adjacent elements and equal distances (use .contiguous())");
  return stride < 0 ? t.size(-1) : stride;
}

void* stream_of(c10::Device dev) { return c10::hip::getCurrentHIPStream(dev.index()).stream(); }

// Makes a HIP device current for a call; nothing for meta tensors.
struct Guard {
  explicit Guard(c10::Device dev) {
    if (!dev.is_meta()) hip.set_index(dev.index());
  }
  c10::hip::OptionalHIPGuard hip;
};

// A new contiguous tensor on `dev`, which is current.  (From torch's allocator without a pass
// through the dispatcher: 0.7 us less of a call that has few to spare.)
at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, c10::Device dev) {
  if (dev.is_meta()) return at::empty(sizes, at::TensorOptions().dtype(type).device(dev));
  return at::Tensor(at::detail::empty_generic(
      sizes, c10::hip::HIPCachingAllocatorMasqueradingAsCUDA::get(),
      c10::DispatchKeySet(c10::DispatchKey::CUDA), type, std::nullopt));
}

// Three float32 rows of one allocation.
std::array<at::Tensor, 3> fresh_rows(int64_t n, c10::Device dev) {
  if (dev.is_meta())
    return {fresh({n}, at::kFloat, dev), fresh({n}, at::kFloat, dev), fresh({n}, at::kFloat, dev)};
  const at::Tensor all = fresh({3, n}, at::kFloat, dev);
  std::array<at::Tensor, 3> rows;
  for (int k = 0; k < 3; ++k) {
    rows[k] = at::Tensor(at::detail::make_tensor_base<c10::TensorImpl>(
        c10::Storage(all.storage()), c10::DispatchKeySet(c10::DispatchKey::CUDA), all.dtype()));
    rows[k].unsafeGetTensorImpl()->set_sizes_contiguous({n});
    rows[k].unsafeGetTensorImpl()->set_storage_offset(k * n);
  }
  return rows;
}

struct Workspace {
  Workspace(const char* name, int64_t bytes, c10::Device dev) : bytes(bytes) {
    TORCH_CHECK(bytes >= 0, "omq_net::", name, ": sizes beyond the library's limits");
    if (bytes > 0) tensor = fresh({bytes}, at::kByte, dev);
  }
  void* data() const { return bytes > 0 ? tensor.data_ptr() : nullptr; }
  int64_t bytes;
  at::Tensor tensor;
};

bool drops(const char* name, double p) {
  TORCH_CHECK(p >= 0.0 && p <= 1.0, "omq_net::", name, ": p ", p, " outside [0, 1]");
  return (uint32_t)(p * 65536.0 + 0.5) != 0;
}

void check_same(const char* name, const char* arg, const at::Tensor& t, const at::Tensor& x) {
  TORCH_CHECK(t.sizes() == x.sizes() && t.scalar_type() == x.scalar_type(), "omq_net::", name, ": ",
              arg, " must have the rows' shape and type (", x.sizes(), ", ", x.scalar_type(),
              "), not ", t.sizes(), ", ", t.scalar_type());
}

int check_weight(const char* name, const at::Tensor& w, const at::Tensor& x) {
  TORCH_CHECK(w.dim() == 1 && w.size(0) == x.size(-1) && w.is_contiguous(), "omq_net::", name,
              ": weight must be contiguous [", x.size(-1), "]");
  TORCH_CHECK(w.scalar_type() == x.scalar_type() || w.scalar_type() == at::kFloat, "omq_net::", name,
              ": weight must be ", x.scalar_type(), " or float32, not ", w.scalar_type());
  return type_of(name, "weight", w);
}

void check_rows_of(const char* name, const char* arg, const at::Tensor& x) {
  TORCH_CHECK(x.dim() >= 1 && x.size(-1) >= 1, "omq_net::", name, ": ", arg,
              " must have a last dimension of at least 1");
}

// ---- embedding ------------------------------------------------------------------------------
at::Tensor token_embedding(const at::Tensor& ids, const at::Tensor& weight, double scale) {
  const char* name = "token_embedding";
  const c10::Device dev = common_device(name, {&weight, &ids});
  const Guard guard(dev);
  const bool wide = ids_are_64(name, "ids", ids);
  const int type = type_of(name, "weight", weight);
  TORCH_CHECK(weight.dim() == 2 && weight.size(0) >= 1 && weight.size(1) >= 1, "omq_net::", name,
              ": weight must be [vocabulary, dim]");
  const int64_t stride = row_stride(name, "weight", weight);
  auto shape = ids.sizes().vec();
  shape.push_back(weight.size(1));
  at::Tensor out = fresh(shape, weight.scalar_type(), dev);
  if (dev.is_meta()) return out;
  check_rc(omq_token_embedding(ids.data_ptr(), wide, ids.numel(), weight.data_ptr(), stride,
                               weight.size(0), weight.size(1), type, (float)scale, out.data_ptr(),
                               stream_of(dev)),
           "omq_token_embedding");
  return out;
}

at::Tensor token_embedding_grad(const at::Tensor& grad, const at::Tensor& ids,
                                int64_t num_embeddings, double scale,
                                std::optional<at::ScalarType> dtype) {
  const char* name = "token_embedding_grad";
  const c10::Device dev = common_device(name, {&grad, &ids});
  const Guard guard(dev);
  const bool wide = ids_are_64(name, "ids", ids);
  const int type = type_of(name, "grad", grad);
  check_rows_of(name, "grad", grad);
  TORCH_CHECK(grad.sizes().slice(0, grad.dim() - 1) == ids.sizes(), "omq_net::", name,
              ": grad must be ids' shape and a last dimension");
  TORCH_CHECK(num_embeddings >= 1, "omq_net::", name, ": num_embeddings ", num_embeddings, " < 1");
  const at::ScalarType to = dtype.value_or(grad.scalar_type());
  TORCH_CHECK(to == grad.scalar_type() || to == at::kFloat, "omq_net::", name, ": dtype must be ",
              grad.scalar_type(), " or float32, not ", to);
  const int64_t dim = grad.size(-1), stride = row_stride(name, "grad", grad);
  at::Tensor out = fresh({num_embeddings, dim}, to, dev);
  if (dev.is_meta()) return out;
  const Workspace ws(
      name, omq_token_embedding_grad_workspace(ids.numel(), num_embeddings, dim), dev);
  check_rc(omq_token_embedding_grad(grad.data_ptr(), stride, type, ids.data_ptr(), wide,
                                    ids.numel(), num_embeddings, dim, (float)scale,
                                    out.data_ptr(), type_of(name, "dtype", out), ws.data(),
                                    ws.bytes, stream_of(dev)),
           "omq_token_embedding_grad");
  return out;
}

// ---- dropout --------------------------------------------------------------------------------
at::Tensor dropout(const at::Tensor& x, double p, int64_t seed, int64_t offset) {
  const char* name = "dropout";
  const c10::Device dev = common_device(name, {&x});
  const Guard guard(dev);
  const int type = type_of(name, "x", x);
  check_rows_of(name, "x", x);
  drops(name, p);
  TORCH_CHECK(x.is_contiguous(), "omq_net::", name, ": tensors must be contiguous");
  at::Tensor out = fresh(x.sizes(), x.scalar_type(), dev);
  if (dev.is_meta()) return out;
  const int64_t dim = x.size(-1);
  check_rc(omq_dropout(x.data_ptr(), x.numel() / dim, dim, type, p, (uint64_t)seed,
                       (uint64_t)offset, out.data_ptr(), stream_of(dev)),
           "omq_dropout");
  return out;
}

// ---- norm -----------------------------------------------------------------------------------
// (y, h); h is empty where there is neither a residual nor a dropped element: it is x then
std::tuple<at::Tensor, at::Tensor> add_rms_norm(const at::Tensor& x, const OptTensor& residual,
                                                const at::Tensor& weight, double eps, double p,
                                                int64_t seed, int64_t offset) {
  const char* name = "add_rms_norm";
  const at::Tensor* res = get(residual);
  const c10::Device dev = common_device(name, {&x, res, &weight});
  const Guard guard(dev);
  check_rows_of(name, "x", x);
  const int type = type_of(name, "x", x), w_type = check_weight(name, weight, x);
  if (res) check_same(name, "residual", *res, x);
  const bool want_h = drops(name, p) || res;
  const int64_t dim = x.size(-1), stride = row_stride(name, "x", x);
  const int64_t r_stride = res ? row_stride(name, "residual", *res) : 0;
  at::Tensor y = fresh(x.sizes(), x.scalar_type(), dev);
  at::Tensor h = want_h ? fresh(x.sizes(), x.scalar_type(), dev) : fresh({0}, x.scalar_type(), dev);
  if (dev.is_meta()) return {y, h};
  check_rc(omq_add_rms_norm(x.data_ptr(), stride, res ? res->data_ptr() : nullptr, r_stride,
                            weight.data_ptr(), w_type, x.numel() / dim, dim, type, (float)eps, p,
                            (uint64_t)seed, (uint64_t)offset, y.data_ptr(),
                            want_h ? h.data_ptr() : nullptr, stream_of(dev)),
           "omq_add_rms_norm");
  return {y, h};
}

// (q, scales, h); h as above
std::tuple<at::Tensor, at::Tensor, at::Tensor> add_rms_norm_fp8(const at::Tensor& x,
                                                                const OptTensor& residual,
                                                                const at::Tensor& weight,
                                                                double eps, int64_t group) {
  const char* name = "add_rms_norm_fp8";
  const at::Tensor* res = get(residual);
  const c10::Device dev = common_device(name, {&x, res, &weight});
  const Guard guard(dev);
  check_rows_of(name, "x", x);
  const int type = type_of(name, "x", x), w_type = check_weight(name, weight, x);
  if (res) check_same(name, "residual", *res, x);
  TORCH_CHECK(group == 0 || group == 128, "omq_net::", name, ": group must be 0 (a row) or 128, not ",
              group);
  const int64_t dim = x.size(-1), stride = row_stride(name, "x", x);
  const int64_t r_stride = res ? row_stride(name, "residual", *res) : 0;
  auto scale_shape = x.sizes().vec();
  scale_shape.back() = group ? (dim + group - 1) / group : 1;
  at::Tensor q = fresh(x.sizes(), at::kFloat8_e4m3fn, dev);
  at::Tensor scales = fresh(scale_shape, at::kFloat, dev);
  at::Tensor h = res ? fresh(x.sizes(), x.scalar_type(), dev) : fresh({0}, x.scalar_type(), dev);
  if (dev.is_meta()) return {q, scales, h};
  check_rc(omq_add_rms_norm_fp8(x.data_ptr(), stride, res ? res->data_ptr() : nullptr, r_stride,
                                weight.data_ptr(), w_type, x.numel() / dim, dim, type, (float)eps,
                                (int)group, static_cast<uint8_t*>(q.data_ptr()),
                                scales.data_ptr<float>(), res ? h.data_ptr() : nullptr,
                                stream_of(dev)),
           "omq_add_rms_norm_fp8");
  return {q, scales, h};
}

// (grad_x, grad_residual, grad_weight); grad_x is empty where no element is dropped: it is
// grad_residual then
std::tuple<at::Tensor, at::Tensor, at::Tensor> add_rms_norm_grad(
    const at::Tensor& grad_y, const OptTensor& grad_h, const at::Tensor& h,
    const at::Tensor& weight, double eps, double p, int64_t seed, int64_t offset) {
  const char* name = "add_rms_norm_grad";
  const at::Tensor* gh = get(grad_h);
  const c10::Device dev = common_device(name, {&h, &grad_y, gh, &weight});
  const Guard guard(dev);
  check_rows_of(name, "h", h);
  const int type = type_of(name, "h", h), w_type = check_weight(name, weight, h);
  check_same(name, "grad_y", grad_y, h);
  if (gh) check_same(name, "grad_h", *gh, h);
  const bool dropped = drops(name, p);
  const int64_t dim = h.size(-1), rows = h.numel() / dim;
  const int64_t h_stride = row_stride(name, "h", h), gy_stride = row_stride(name, "grad_y", grad_y);
  const int64_t gh_stride = gh ? row_stride(name, "grad_h", *gh) : 0;
  at::Tensor gr = fresh(h.sizes(), h.scalar_type(), dev);
  at::Tensor gx = dropped ? fresh(h.sizes(), h.scalar_type(), dev) : fresh({0}, h.scalar_type(), dev);
  at::Tensor gw = fresh(weight.sizes(), weight.scalar_type(), dev);
  if (dev.is_meta()) return {gx, gr, gw};
  const Workspace ws(name, omq_add_rms_norm_grad_workspace(rows, dim), dev);
  check_rc(omq_add_rms_norm_grad(grad_y.data_ptr(), gy_stride, gh ? gh->data_ptr() : nullptr,
                                 gh_stride, h.data_ptr(), h_stride, weight.data_ptr(), w_type,
                                 rows, dim, type, (float)eps, p, (uint64_t)seed, (uint64_t)offset,
                                 dropped ? gx.data_ptr() : nullptr, gr.data_ptr(), gw.data_ptr(),
                                 ws.data(), ws.bytes, stream_of(dev)),
           "omq_add_rms_norm_grad");
  return {gx, gr, gw};
}

// ---- policy loss ----------------------------------------------------------------------------
const float* row_floats(const char* name, const char* arg, const at::Tensor& t, int64_t rows) {
  TORCH_CHECK(t.dim() == 1 && t.size(0) == rows && t.scalar_type() == at::kFloat &&
                  t.is_contiguous(),
              "omq_net::", name, ": ", arg, " must be contiguous float32 [", rows, "]");
  return t.is_meta() ? nullptr : t.data_ptr<float>();
}

omq_policy_rows policy_rows(const char* name, const at::Tensor& logits, const at::Tensor& actions,
                            const at::Tensor& advantages, const at::Tensor& old_logp,
                            double clip_low, double clip_high, double kl_coef,
                            const OptTensor& ref_logp, const OptTensor& target,
                            const OptTensor& legal) {
  const at::Tensor *ref = get(ref_logp), *pi = get(target), *ok = get(legal);
  const c10::Device dev =
      common_device(name, {&logits, &actions, &advantages, &old_logp, ref, pi, ok});
  TORCH_CHECK(logits.dim() == 2 && logits.size(1) >= 1, "omq_net::", name,
              ": logits must be [rows, actions]");
  TORCH_CHECK(!(ref && pi), "omq_net::", name, ": ref_logp and target exclude each other");
  omq_policy_rows r{};
  r.rows = logits.size(0);
  r.actions = logits.size(1);
  r.dtype = type_of(name, "logits", logits);
  r.logits_stride = row_stride(name, "logits", logits);
  r.taken_are_64 = ids_are_64(name, "actions", actions);
  TORCH_CHECK(actions.dim() == 1 && actions.size(0) == r.rows, "omq_net::", name,
              ": actions must be [", r.rows, "]");
  r.advantages = row_floats(name, "advantages", advantages, r.rows);
  r.old_logp = row_floats(name, "old_logp", old_logp, r.rows);
  if (ref) r.ref_logp = row_floats(name, "ref_logp", *ref, r.rows);
  if (pi) {
    TORCH_CHECK(pi->sizes() == logits.sizes() && pi->scalar_type() == at::kFloat, "omq_net::", name,
                ": target must be float32 ", logits.sizes());
    r.target_stride = row_stride(name, "target", *pi);
  }
  if (ok) {
    TORCH_CHECK(ok->sizes() == logits.sizes() && ok->scalar_type() == at::kBool, "omq_net::", name,
                ": legal must be bool ", logits.sizes());
    r.legal_stride = row_stride(name, "legal", *ok);
  }
  TORCH_CHECK(clip_low >= 0.0 && clip_high >= 0.0, "omq_net::", name, ": clip_low ", clip_low,
              " and clip_high ", clip_high, " must not be negative");
  r.clip_low = (float)clip_low;
  r.clip_high = (float)clip_high;
  r.kl_coef = (float)kl_coef;
  if (!dev.is_meta()) {
    r.logits = logits.data_ptr();
    r.taken = actions.data_ptr();
    if (pi) r.target = pi->data_ptr<float>();
    if (ok) r.legal = reinterpret_cast<const uint8_t*>(ok->data_ptr<bool>());
  }
  return r;
}

// (loss, logp, kl, stats)
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> clipped_policy_loss(
    const at::Tensor& logits, const at::Tensor& actions, const at::Tensor& advantages,
    const at::Tensor& old_logp, double clip_low, double clip_high, double kl_coef,
    const OptTensor& ref_logp, const OptTensor& target, const OptTensor& legal, bool want_stats) {
  const char* name = "clipped_policy_loss";
  const omq_policy_rows r = policy_rows(name, logits, actions, advantages, old_logp, clip_low,
                                        clip_high, kl_coef, ref_logp, target, legal);
  const c10::Device dev = logits.device();
  const Guard guard(dev);
  auto [loss, logp, kl] = fresh_rows(r.rows, dev);
  at::Tensor stats = fresh({want_stats ? r.rows : 0, OMQ_NET_STATS}, at::kFloat, dev);
  if (dev.is_meta()) return {loss, logp, kl, stats};
  const Workspace ws(name, omq_clipped_policy_loss_workspace(r.rows, r.actions), dev);
  check_rc(omq_clipped_policy_loss(&r, loss.data_ptr<float>(), logp.data_ptr<float>(),
                                   kl.data_ptr<float>(),
                                   want_stats ? stats.data_ptr<float>() : nullptr, ws.data(),
                                   ws.bytes, stream_of(dev)),
           "omq_clipped_policy_loss");
  return {loss, logp, kl, stats};
}

at::Tensor clipped_policy_loss_grad(const at::Tensor& logits, const at::Tensor& actions,
                                    const at::Tensor& advantages, const at::Tensor& old_logp,
                                    double clip_low, double clip_high, double kl_coef,
                                    const OptTensor& ref_logp, const OptTensor& target,
                                    const OptTensor& legal, const at::Tensor& stats,
                                    const OptTensor& row_weight) {
  const char* name = "clipped_policy_loss_grad";
  const omq_policy_rows r = policy_rows(name, logits, actions, advantages, old_logp, clip_low,
                                        clip_high, kl_coef, ref_logp, target, legal);
  const at::Tensor* w = get(row_weight);
  common_device(name, {&logits, &stats, w});
  TORCH_CHECK(stats.dim() == 2 && stats.size(0) == r.rows && stats.size(1) == OMQ_NET_STATS &&
                  stats.scalar_type() == at::kFloat && stats.is_contiguous(),
              "omq_net::", name, ": stats must be those of clipped_policy_loss");
  const float* wp = w ? row_floats(name, "row_weight", *w, r.rows) : nullptr;
  const c10::Device dev = logits.device();
  const Guard guard(dev);
  at::Tensor grad = fresh({r.rows, r.actions}, logits.scalar_type(), dev);
  if (dev.is_meta()) return grad;
  check_rc(omq_clipped_policy_loss_grad(&r, stats.data_ptr<float>(), wp, grad.data_ptr(),
                                        stream_of(dev)),
           "omq_clipped_policy_loss_grad");
  return grad;
}

// (loss, logp, kl, grad)
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> clipped_policy_loss_with_grad(
    const at::Tensor& logits, const at::Tensor& actions, const at::Tensor& advantages,
    const at::Tensor& old_logp, double clip_low, double clip_high, double kl_coef,
    const OptTensor& ref_logp, const OptTensor& target, const OptTensor& legal,
    const OptTensor& row_weight) {
  const char* name = "clipped_policy_loss_with_grad";
  const omq_policy_rows r = policy_rows(name, logits, actions, advantages, old_logp, clip_low,
                                        clip_high, kl_coef, ref_logp, target, legal);
  const at::Tensor* w = get(row_weight);
  common_device(name, {&logits, w});
  const float* wp = w ? row_floats(name, "row_weight", *w, r.rows) : nullptr;
  const c10::Device dev = logits.device();
  const Guard guard(dev);
  auto [loss, logp, kl] = fresh_rows(r.rows, dev);
  at::Tensor grad = fresh({r.rows, r.actions}, logits.scalar_type(), dev);
  if (dev.is_meta()) return {loss, logp, kl, grad};
  const Workspace ws(name, omq_clipped_policy_loss_workspace(r.rows, r.actions), dev);
  check_rc(omq_clipped_policy_loss_with_grad(&r, wp, loss.data_ptr<float>(),
                                             logp.data_ptr<float>(), kl.data_ptr<float>(),
                                             grad.data_ptr(), ws.data(), ws.bytes,
                                             stream_of(dev)),
           "omq_clipped_policy_loss_with_grad");
  return {loss, logp, kl, grad};
}

// ---- registration ---------------------------------------------------------------------------
// The operators have no derivatives of their own (net_ops.py's autograd functions call them): a
// tangent is refused, and a backward pass through one raises.  Without this kernel torch drops
// tangents without a word and leaves gradients out with a warning.  (torch's fallback for operators
// without a derivative does the same and takes 0.1 to 0.4 us more of a call.)
template <auto Fn>
struct NoDerivative;

template <class R, class... A, R (*Fn)(A...)>
struct NoDerivative<Fn> {
  static std::string& name() {
    static std::string given;
    return given;
  }

  template <class T>
  static const at::Tensor* tensor(const T& t) {
    if constexpr (std::is_same_v<T, at::Tensor>) return &t;
    else if constexpr (std::is_same_v<T, OptTensor>) return get(t);
    else return nullptr;
  }

  static void record(const std::shared_ptr<torch::autograd::Node>& node, at::Tensor& out) {
    torch::autograd::set_history(out, node);
  }

  template <class... T>
  static void record(const std::shared_ptr<torch::autograd::Node>& node, std::tuple<T...>& out) {
    std::apply([&](auto&... t) { (record(node, t), ...); }, out);
  }

  static R call(c10::DispatchKeySet keys, A... args) {
    static const auto op =
        c10::Dispatcher::singleton().findSchemaOrThrow(name().c_str(), "").template typed<R(A...)>();
    const at::Tensor* tensors[] = {tensor(args)...};
    bool needed = false;
    for (const at::Tensor* t : tensors) {
      if (!t) continue;
      TORCH_CHECK_NOT_IMPLEMENTED(!t->_fw_grad(/*level=*/0).defined(), name(),
                                  " has no forward-mode derivative");
      needed = needed || t->requires_grad();
    }
    R out = op.redispatch(keys & c10::after_autograd_keyset, args...);
    if (needed && at::GradMode::is_enabled()) {
      const std::shared_ptr<torch::autograd::Node> node(new torch::autograd::NotImplemented(name()),
                                                        torch::autograd::deleteNode);
      torch::autograd::edge_list edges;
      for (const at::Tensor* t : tensors)
        if (t) edges.push_back(torch::autograd::impl::gradient_edge(*t));
      node->set_next_edges(std::move(edges));
      record(node, out);
    }
    return out;
  }
};

// Defines `name` with one function for HIP, host (which it refuses) and meta tensors.
template <auto Fn>
void define(torch::Library& m, const std::string& name, const std::string& schema) {
  m.def((name + schema).c_str());
  for (const auto key : {c10::DispatchKey::CUDA, c10::DispatchKey::CPU, c10::DispatchKey::Meta})
    m.impl(name.c_str(), torch::dispatch(key, Fn));
  NoDerivative<Fn>::name() = "omq_net::" + name;
  m.impl(name.c_str(), torch::dispatch(c10::DispatchKey::Autograd, &NoDerivative<Fn>::call));
}

const std::string kLossArgs =
    "Tensor logits, Tensor actions, Tensor advantages, Tensor old_logp, float clip_low, "
    "float clip_high, float kl_coef, Tensor? ref_logp, Tensor? target, Tensor? legal";

}  // namespace

TORCH_LIBRARY(omq_net, m) {
  define<token_embedding>(m, "token_embedding",
                          "(Tensor ids, Tensor weight, float scale) -> Tensor");
  define<token_embedding_grad>(m, "token_embedding_grad",
         "(Tensor grad, Tensor ids, int num_embeddings, float scale, ScalarType? dtype) -> Tensor");
  define<dropout>(m, "dropout", "(Tensor x, float p, int seed, int offset) -> Tensor");
  define<add_rms_norm>(m, "add_rms_norm",
         "(Tensor x, Tensor? residual, Tensor weight, float eps, float p, int seed, int offset) "
         "-> (Tensor, Tensor)");
  define<add_rms_norm_fp8>(m, "add_rms_norm_fp8",
         "(Tensor x, Tensor? residual, Tensor weight, float eps, int group) "
         "-> (Tensor, Tensor, Tensor)");
  define<add_rms_norm_grad>(m, "add_rms_norm_grad",
         "(Tensor grad_y, Tensor? grad_h, Tensor h, Tensor weight, float eps, float p, int seed, "
         "int offset) -> (Tensor, Tensor, Tensor)");
  define<clipped_policy_loss>(m, "clipped_policy_loss",
         "(" + kLossArgs + ", bool want_stats) -> (Tensor, Tensor, Tensor, Tensor)");
  define<clipped_policy_loss_grad>(m, "clipped_policy_loss_grad",
         "(" + kLossArgs + ", Tensor stats, Tensor? row_weight) -> Tensor");
  define<clipped_policy_loss_with_grad>(m, "clipped_policy_loss_with_grad",
         "(" + kLossArgs + ", Tensor? row_weight) -> (Tensor, Tensor, Tensor, Tensor)");
}
