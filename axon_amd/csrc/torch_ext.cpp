// Host side of the small per-token operators: operand checks, output tensors, the launch through the C ABI and the
// autograd node of a loss, in one native call each.
//
// A call of such an operator takes the GPU 5 to 20 us and took the host 18 to 30 us in Python, and a Python backward
// some 40 us more than a native one: the engine's device thread has to get the interpreter lock from the thread that
// waits for it.  Per call: policy_loss 18 -> 9 us, group_advantage 28 -> 13, reverse_scan 24 -> 7; whole passes
// (advantage, loss, backward), with the sums that the launch sends to the host itself: GRPO + PPO on 128 x 1024 165 -> 94 us,
// sampler correction + GSPO on 65536 tokens 254 -> 166, correction + PPO on 8.4 M 402 -> 352, GAE + value loss on 2.1 M 176 -> 115.
//
// Nothing here computes: the arithmetic is behind axon_amd.h.  The functions take what the Python wrappers of the same
// names (axon_amd/_ops.py) have normalised, and run without the interpreter lock, as a call through ctypes does.
#include <ATen/ATen.h>
#include <hip/hip_runtime_api.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <ATen/EmptyTensor.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/VirtualGuardImpl.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/grad_mode.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <array>
#include <atomic>
#include <chrono>
#include <cmath>
#include <cstring>
#include <memory>
#include <mutex>
#include <utility>
#include <vector>

#include "../../include/axon_amd.h"

namespace py = pybind11;
using at::Tensor;
using OptTensor = std::optional<Tensor>;

namespace {

PyObject* g_error = nullptr;  // axon_amd._lib.AxonAmdError
struct AxonError : torch::PyTorchError {  // the autograd engine hands it on as what it is
  using PyTorchError::PyTorchError;
  PyObject* python_type() override { return g_error; }
};

void check(int rc, const char* what) {
  if (rc != 0) throw AxonError(std::string(what) + ": " + axon_amd_error_string(rc) + " (code " + std::to_string(rc) + ")");
}

// The HIP path only.  (The Python wrappers look at the first operand of every other function.)
void require_device(const Tensor& t, const char* what) {
  if (!t.is_cuda())
    throw AxonError(std::string(what) + ": tensor is on " + t.device().str() +
                    "; the axon_amd path runs on MI355X only and has no CPU fallback");
}

void* stream() { return c10::hip::getCurrentHIPStream().stream(); }
bool capturing() { return c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None; }

const void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
const void* ptr(const OptTensor& t) { return t ? t->data_ptr() : nullptr; }

// The kernels move four values per access: a view that starts off a 16-byte boundary is copied.
Tensor on_16_bytes(Tensor t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 ? t : t.clone(); }

// fp32, contiguous, aligned, outside the graph; the usual operand passes through untouched.
Tensor f32(const Tensor& x) {
  Tensor t = x.requires_grad() ? x.detach() : x;
  if (t.scalar_type() != at::kFloat || !t.is_contiguous()) t = t.to(at::kFloat).contiguous();
  return on_16_bytes(std::move(t));
}
Tensor f32(const OptTensor& x) { return x ? f32(*x) : Tensor(); }

// A response mask: fp32 and int64 are read natively.
std::pair<Tensor, int> mask_arg(const Tensor& x) {
  Tensor t = x.requires_grad() ? x.detach() : x;
  if (!t.is_contiguous()) t = t.contiguous();
  if (t.scalar_type() == at::kLong) return {on_16_bytes(std::move(t)), 1};
  if (t.scalar_type() != at::kFloat) t = t.to(at::kFloat);
  return {on_16_bytes(std::move(t)), 0};
}

// The kernels index every operand with the same token (or row) index.
void same_len(const char* what, const char* name, int64_t n, const Tensor& t) {
  if (t.numel() != n)
    throw py::value_error(std::string(what) + ": " + name + " has " + std::to_string(t.numel()) + " elements, expected " +
                          std::to_string(n));
}
void same_len(const char* what, const char* name, int64_t n, const OptTensor& t) {
  if (t) same_len(what, name, n, *t);
}

at::TensorOptions opts(const Tensor& like, at::ScalarType dtype = at::kFloat) {
  return at::TensorOptions().dtype(dtype).device(like.device());
}

// See _ops._acc8.
Tensor acc8(int64_t n_slots, const Tensor& like, const OptTensor& acc) {
  Tensor a = acc ? *acc : at::empty({8}, opts(like));
  if (n_slots == 0) return a.zero_();
  return capturing() ? a.fill_(std::numeric_limits<float>::quiet_NaN()) : a;
}

struct Rows {  // _ops.Rows, its offsets checked to be on the device
  int64_t n_rows, n_slots, uniform_len;
  OptTensor cu;
  std::vector<int64_t> shape;
  const int32_t* offsets() const { return cu ? cu->data_ptr<int32_t>() : nullptr; }
};
typedef std::tuple<int64_t, int64_t, int64_t, OptTensor, std::vector<int64_t>> RowsTuple;
Rows rows_of(const RowsTuple& t) {
  Rows r{std::get<0>(t), std::get<1>(t), std::get<2>(t), std::get<3>(t), std::get<4>(t)};
  if (r.cu && !r.cu->is_cuda())
    throw AxonError("cu_seqlens is on " + r.cu->device().str() +
                    ": the row offsets must live on the GPU (rows_of puts them on the device of the tensor it is given)");
  return r;
}

// The sums of a loss on their way to the host (axon_policy_loss_post): `also`, a tensor that earlier work of the stream has
// written, and the loss's eight sums behind it.
// One launch writes to a slot of pinned memory at a time; a slot goes back once its words have arrived.  One that nobody
// waits for any more (its loss raised behind the launch) is set aside until they have, which the next taker finds out: to wait
// in a destructor would hold the interpreter lock for the rest of the queue.  The slots, one kilobyte each, are as many as
// posts were ever under way together and live until the process ends.
struct Slot {
  uint32_t* host;
  uint32_t* device;
  uint32_t seq;
  bool arrived() const { return __atomic_load_n(host, __ATOMIC_ACQUIRE) == seq; }
};
class Slots {
 public:
  static constexpr int kWords = 16 + AXON_MAIL_MAX_WORDS + 8, kBytes = 1024, kPerBlock = 64;
  static_assert(kWords * 4 <= kBytes, "");
  static Slots& get() {
    static auto* const slots = new Slots;
    return *slots;
  }
  Slot take() {
    const std::lock_guard<std::mutex> lock(mutex_);
    const auto back = std::partition(aside_.begin(), aside_.end(), [](const Slot& s) { return !s.arrived(); });
    free_.insert(free_.end(), back, aside_.end());
    aside_.erase(back, aside_.end());
    if (free_.empty()) {
      void *host = nullptr, *device = nullptr;
      if (hipHostMalloc(&host, kBytes * kPerBlock, hipHostMallocPortable | hipHostMallocMapped | hipHostMallocCoherent) !=
              hipSuccess ||
          hipHostGetDevicePointer(&device, host, 0) != hipSuccess)
        throw AxonError("no pinned host memory for the sums of a loss");
      std::memset(host, 0, kBytes * kPerBlock);
      for (int i = 0; i < kPerBlock; ++i)
        free_.push_back(Slot{static_cast<uint32_t*>(host) + i * (kBytes / 4), static_cast<uint32_t*>(device) + i * (kBytes / 4), 0});
      made_ += kPerBlock;
    }
    Slot s = free_.back();
    free_.pop_back();
    ++s.seq;
    return s;
  }
  void give(const Slot& s) {
    const std::lock_guard<std::mutex> lock(mutex_);
    free_.push_back(s);
  }
  void set_aside(const Slot& s) {
    const std::lock_guard<std::mutex> lock(mutex_);
    aside_.push_back(s);
  }
  int made() {
    const std::lock_guard<std::mutex> lock(mutex_);
    return made_;
  }

 private:
  std::mutex mutex_;
  std::vector<Slot> free_, aside_;
  int made_ = 0;
};

class Post {
 public:
  explicit Post(OptTensor also) : also_(std::move(also)) {
    if (!also_) return;  // the launch reads nbytes() / 4 words from data_ptr() on
    require_device(*also_, "the words in front of a loss's sums");
    if (!also_->is_contiguous() || also_->nbytes() % 4 != 0 || also_->nbytes() > 4 * AXON_MAIL_MAX_WORDS)
      throw AxonError("the words in front of a loss's sums must be a contiguous tensor of whole words, at most " +
                      std::to_string(AXON_MAIL_MAX_WORDS) + "; got " + std::to_string(also_->nbytes()) + " bytes");
  }
  ~Post() {  // never waited for
    if (!sent_) return;
    try {
      Slots::get().set_aside(slot_);
    } catch (...) {  // no memory for the list: the slot is not used again
    }
  }
  const void* also() const { return also_ ? also_->data_ptr() : nullptr; }
  int64_t n_also() const { return also_ ? (int64_t)also_->nbytes() / 4 : 0; }
  const Slot& send(void* stream) {
    if (sent_) throw AxonError("these sums are on their way already");
    slot_ = Slots::get().take();
    stream_ = (hipStream_t)stream;
    return slot_;
  }
  void sent(int rc) {  // a refused launch writes nothing
    if (rc == 0) sent_ = true;
    else Slots::get().give(slot_);
  }
  bool is_sent() const { return sent_; }
  // The loss's eight sums.
  std::vector<double> sums() {
    arrive();
    float v[8];
    std::memcpy(v, slot_.host + 16 + n_also(), sizeof v);
    Slots::get().give(slot_);
    return {v, v + 8};
  }
  // All words as an fp32 tensor on the host.
  Tensor wait() {
    arrive();
    const int64_t words = n_also() + 8;
    Tensor out = at::empty({words}, at::TensorOptions().dtype(at::kFloat));
    std::memcpy(out.data_ptr(), slot_.host + 16, words * 4);
    Slots::get().give(slot_);
    return out;
  }

 private:
  // Spins while the words can be expected at once, then leaves the waiting to the runtime; the stream's end or its error
  // ends it in any case.
  void arrive() {
    if (!sent_) throw AxonError("no sums are on their way");
    sent_ = false;
    const auto start = std::chrono::steady_clock::now();
    for (int n = 1; !slot_.arrived(); ++n) {
      if (n % 1024) {
        __builtin_ia32_pause();
        continue;
      }
      if (std::chrono::steady_clock::now() - start < std::chrono::milliseconds(2)) continue;
      const hipError_t err = hipStreamSynchronize(stream_);
      if (err == hipSuccess && slot_.arrived()) break;
      // the slot is not used again: the device may be in any state
      throw AxonError(std::string("the sums of a loss did not arrive: ") + hipGetErrorString(err));
    }
  }

  OptTensor also_;
  Slot slot_{};
  hipStream_t stream_ = nullptr;
  bool sent_ = false;
};

std::tuple<Tensor, Tensor> policy_loss(int kind, const Tensor& log_probs, const Tensor& old_log_probs,
                                       const Tensor& advantages, const Tensor& mask, const OptTensor& is_weights,
                                       const RowsTuple& rows_tuple, int token_reduce, int batch_reduce,
                                       const OptTensor& per_row_count, const OptTensor& program_tokens,
                                       const OptTensor& program_steps, const OptTensor& valid, double ratio_lo,
                                       double ratio_hi, double clip_c, const OptTensor& acc_place, double loss_scale,
                                       bool one_pass, const Tensor& ws, Post* post) {
  const Rows rows = rows_of(rows_tuple);
  const int64_t n = rows.n_slots;
  same_len("policy_loss", "log_probs", n, log_probs);
  same_len("policy_loss", "old_log_probs", n, old_log_probs);
  same_len("policy_loss", "advantages", n, advantages);
  same_len("policy_loss", "mask", n, mask);
  same_len("policy_loss", "is_weights", n, is_weights);
  const Tensor lp = f32(log_probs), old = f32(old_log_probs), adv = f32(advantages), isw = f32(is_weights);
  const auto mk = mask_arg(mask);
  Tensor grad = at::empty(rows.shape, opts(lp)), acc = acc8(n, lp, acc_place);
  const float *lp_p = (const float*)ptr(lp), *old_p = (const float*)ptr(old), *adv_p = (const float*)ptr(adv),
              *isw_p = (const float*)ptr(isw);
  float *grad_p = grad.data_ptr<float>(), *acc_p = acc.data_ptr<float>(), *ws_p = ws.data_ptr<float>();
  const double *prtc_p = (const double*)ptr(per_row_count), *npt_p = (const double*)ptr(program_tokens),
               *nps_p = (const double*)ptr(program_steps), *valid_p = (const double*)ptr(valid);
  const float lo = (float)ratio_lo, hi = (float)ratio_hi, clip = (float)clip_c, scale = (float)loss_scale;
  void* const st = stream();
  // (nobody can wait inside a capture, and nothing is launched without tokens: the sums stay on the device then)
  if (post != nullptr && n > 0 && !capturing()) {
    const Slot& slot = post->send(st);
    const int rc =
        one_pass ? axon_policy_loss_post(kind, lp_p, old_p, adv_p, ptr(mk.first), mk.second, isw_p, rows.offsets(), rows.n_rows,
                                         n, rows.uniform_len, scale, valid_p, lo, hi, clip, grad_p, acc_p, ws_p,
                                         post->also(), post->n_also(), slot.device, slot.seq, st)
                 : axon_policy_loss_rows_post(kind, lp_p, old_p, adv_p, ptr(mk.first), mk.second, isw_p, rows.offsets(),
                                              rows.n_rows, n, rows.uniform_len, token_reduce, batch_reduce, prtc_p, npt_p,
                                              nps_p, valid_p, lo, hi, clip, grad_p, acc_p, ws_p, post->also(),
                                              post->n_also(), slot.device, slot.seq, st);
    post->sent(rc);
    check(rc, one_pass ? "axon_policy_loss" : "axon_policy_loss_rows");
  } else if (one_pass) {
    check(axon_policy_loss(kind, lp_p, old_p, adv_p, ptr(mk.first), mk.second, isw_p, rows.offsets(), rows.n_rows, n,
                           rows.uniform_len, nullptr, nullptr, scale, 1, valid_p, lo, hi, clip, grad_p, acc_p, ws_p, st),
          "axon_policy_loss");
  } else {
    check(axon_policy_loss_rows(kind, lp_p, old_p, adv_p, ptr(mk.first), mk.second, isw_p, rows.offsets(), rows.n_rows, n,
                                rows.uniform_len, token_reduce, batch_reduce, prtc_p, npt_p, nps_p, valid_p, lo, hi, clip,
                                grad_p, acc_p, ws_p, st),
          "axon_policy_loss_rows");
  }
  return {acc, grad};
}

Tensor group_advantage(const Tensor& rewards, const Tensor& mask, const Tensor& gidx, int64_t n_groups,
                       const RowsTuple& rows_tuple, double eps, int mode, double clamp_abs, const Tensor& ws) {
  const Rows rows = rows_of(rows_tuple);
  const int64_t n = rows.n_slots;
  same_len("group_advantage", "rewards", n, rewards);
  same_len("group_advantage", "mask", n, mask);
  same_len("group_advantage", "gidx", rows.n_rows, gidx);
  const Tensor rw = f32(rewards);
  const auto mk = mask_arg(mask);
  Tensor scratch = at::empty({2 * rows.n_rows}, opts(rw)), out = at::empty(rows.shape, opts(rw));
  check(axon_group_advantage((const float*)ptr(rw), ptr(mk.first), mk.second, rows.offsets(), rows.n_rows, n,
                             rows.uniform_len, gidx.data_ptr<int64_t>(), n_groups, (float)eps, mode, (float)clamp_abs,
                             scratch.data_ptr<float>(), out.data_ptr<float>(), ws.data_ptr<float>(), stream()),
        "axon_group_advantage");
  return out;
}

// (weights or none, new mask)
std::tuple<OptTensor, Tensor> sampler_correction_diag(
    const Tensor& old_log_probs, const Tensor& sampler_log_probs, const Tensor& mask, const RowsTuple& rows_tuple,
    int is_mode, double is_threshold, int rs_mode, double rs_lr_lo, double rs_lr_hi, std::optional<double> log_veto,
    double is_lo, double is_hi, double rs_lo, double rs_hi, double log_is_lo, double log_is_hi, double log_rs_lo,
    double log_rs_hi, const Tensor& acc, const Tensor& diag, const Tensor& part) {
  const Rows rows = rows_of(rows_tuple);
  const int64_t n = rows.n_slots;
  same_len("sampler_correction", "old_log_probs", n, old_log_probs);
  same_len("sampler_correction", "sampler_log_probs", n, sampler_log_probs);
  same_len("sampler_correction", "mask", n, mask);
  const Tensor old = f32(old_log_probs), samp = f32(sampler_log_probs);
  const auto mk = mask_arg(mask);
  OptTensor isw;
  if (is_mode) isw = at::empty(rows.shape, opts(old));
  Tensor new_mask = at::empty(rows.shape, opts(old));
  Tensor ws = at::empty({axon_sampler_correction_diag_workspace_bytes(rows.n_rows, n) / 4}, opts(old));
  check(axon_sampler_correction_diag(
        (const float*)ptr(old), (const float*)ptr(samp), ptr(mk.first), mk.second, rows.offsets(), rows.n_rows, n,
        rows.uniform_len, is_mode, (float)is_threshold, rs_mode, (float)rs_lr_lo, (float)rs_lr_hi, log_veto ? 1 : 0,
        (float)log_veto.value_or(0.0), (float)is_lo, (float)is_hi, (float)rs_lo, (float)rs_hi, (float)log_is_lo,
        (float)log_is_hi, (float)log_rs_lo, (float)log_rs_hi, isw ? isw->data_ptr<float>() : nullptr,
        new_mask.data_ptr<float>(), (float*)acc.data_ptr(), part.data_ptr<float>(), ws.data_ptr<float>(),
        diag.data_ptr<double>(), stream()),
        "axon_sampler_correction_diag");
  return {isw, new_mask};
}

// (adv or none, ret)
std::tuple<OptTensor, Tensor> reverse_scan(int mode, const Tensor& rewards, const OptTensor& values, const Tensor& mask,
                                           const RowsTuple& rows_tuple, double gamma, double lam,
                                           const OptTensor& row_baseline, bool want_adv) {
  const Rows rows = rows_of(rows_tuple);
  const int64_t n = rows.n_slots;
  same_len("reverse_scan", "rewards", n, rewards);
  same_len("reverse_scan", "values", n, values);
  same_len("reverse_scan", "mask", n, mask);
  const Tensor rw = f32(rewards), val = f32(values), base = f32(row_baseline);
  if (base.defined() && base.numel() != rows.n_rows)
    throw py::value_error("row_baseline has " + std::to_string(base.numel()) + " entries, batch has " +
                          std::to_string(rows.n_rows) + " rows");
  const auto mk = mask_arg(mask);
  OptTensor adv;
  if (want_adv) adv = at::empty(rows.shape, opts(rw));
  Tensor ret = at::empty(rows.shape, opts(rw));
  check(axon_reverse_scan(mode, (const float*)ptr(rw), (const float*)ptr(val), ptr(mk.first), mk.second, rows.offsets(),
                          rows.n_rows, n, rows.uniform_len, (float)gamma, (float)lam, (const float*)ptr(base),
                          adv ? adv->data_ptr<float>() : nullptr, ret.data_ptr<float>(), stream()),
        "axon_reverse_scan");
  return {adv, ret};
}

// x * s1 * s2 (device scalars, s2 may be missing) as a new fp32 tensor shaped like x
Tensor scale_f32(const Tensor& x, const Tensor& s1, const OptTensor& s2) {
  require_device(x, "scale_f32");  // a backward comes here without Python, with what a saved-tensor hook has handed back
  const Tensor xf = f32(x);
  const auto scalar = [&](const Tensor& s) {
    Tensor t = s.detach();
    return t.scalar_type() == at::kFloat && t.device() == xf.device() ? t : t.to(xf.device(), at::kFloat);
  };
  const Tensor a = scalar(s1), b = s2 ? scalar(*s2) : Tensor();
  Tensor out = at::empty_like(xf);
  check(axon_scale_f32((const float*)ptr(xf), (const float*)ptr(a), (const float*)ptr(b), out.data_ptr<float>(), xf.numel(),
                       stream()),
        "axon_scale_f32");
  return out.view(x.sizes());
}

// The node of a loss whose kernel has left the gradient beside it: loss = factor * acc[0], and in the backward
// grad * (factor * upstream) * acc[slot] (slot < 0: no such factor).
struct FinishedLoss : torch::autograd::Function<FinishedLoss> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& acc, const Tensor& grad,
                        double factor, int64_t slot) {
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({grad, acc});
    ctx->saved_data["factor"] = factor;
    ctx->saved_data["slot"] = slot;
    ctx->saved_data["dtype"] = (int64_t)x.scalar_type();
    if (factor != 1.0) return acc.select(0, 0) * factor;
    // acc[0] as a tensor of its own: no view (the caller may change it in place, and nothing reads it again)
    return at::empty({0}, acc.options()).set_(acc.storage(), acc.storage_offset(), {}, {});
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list upstream) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &grad = saved[0], &acc = saved[1];
    const double factor = ctx->saved_data["factor"].toDouble();
    const int64_t slot = ctx->saved_data["slot"].toInt();
    Tensor g = upstream[0].defined() ? upstream[0] : at::zeros({}, grad.options());
    if (factor != 1.0) g = g * factor;
    const Tensor out = scale_f32(grad, g, slot < 0 ? OptTensor() : OptTensor(acc.select(0, slot)));
    return {out.to((at::ScalarType)ctx->saved_data["dtype"].toInt()), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

// ---------------------------------------------------------------------------------------------------------------------
// Alternatives of materialised logits and the router's balance loss: operators with an autograd node of their own.
// ---------------------------------------------------------------------------------------------------------------------

using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

[[noreturn]] void refuse(const char* what, const std::string& why) { throw py::value_error(std::string(what) + ": " + why); }

std::string shape_text(const Tensor& t) {
  std::string s = "(";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + (t.dim() == 1 ? ",)" : ")");
}

int logits_dtype(const char* what, const Tensor& t) {
  if (t.scalar_type() == at::kFloat) return AXON_LOGITS_F32;
  if (t.scalar_type() == at::kBFloat16) return AXON_LOGITS_BF16;
  refuse(what, std::string("logits must be fp32 or bf16, got ") + c10::toString(t.scalar_type()));
}
bool is_index(const Tensor& t) { return t.scalar_type() == at::kInt || t.scalar_type() == at::kLong; }
int is_i64(const Tensor& t) { return t.scalar_type() == at::kLong; }

// Rows of logits as the kernels read them: [rows, vocab], unit stride over the vocabulary, rows that do not share storage.
Tensor rows_of_logits(const Tensor& logits) {
  if (logits.dim() < 1) throw py::value_error("logits must be [..., vocab]");
  const int64_t v = logits.size(-1);
  Tensor flat = logits.detach().reshape({v > 0 ? logits.numel() / v : 0, v});
  if (flat.stride(1) != 1 || (flat.size(0) > 1 && flat.stride(0) < v)) flat = flat.contiguous();
  return flat;
}
int64_t row_stride(const Tensor& rows) { return rows.size(0) > 1 ? rows.stride(0) : rows.size(1); }

// What a saved-tensor hook has handed back is looked at again: a pointer into host memory would fault the GPU.
void same_place(const char* what, const Tensor& like, std::initializer_list<const Tensor*> others) {
  require_device(like, what);
  for (const Tensor* t : others) {
    if (!t->defined()) continue;
    if (t->device() != like.device()) refuse(what, "operands live on different devices");
    if (!t->is_contiguous()) refuse(what, "operands must be contiguous");
  }
}

void same_type(const char* what, at::ScalarType type, std::initializer_list<const Tensor*> tensors) {
  for (const Tensor* t : tensors)
    if (t->defined() && t->scalar_type() != type) refuse(what, "a saved tensor has come back in another type");
}

// A gradient that cannot be differentiated again says so, instead of being a constant.
Tensor once(Tensor grad, const char* what) {
  if (!at::GradMode::is_enabled()) return grad;
  auto error = std::make_shared<torch::autograd::DelayedError>(std::string(what) + ": the gradient cannot be differentiated again", 1);
  return (*error)({grad.detach().requires_grad_(true)})[0];
}

// Forward-mode gradients are not offered: a tangent would be dropped without a word.
void no_tangent(const char* what, const Tensor& t) {
  if (t._fw_grad(0).defined()) throw AxonError(std::string(what) + ": forward-mode differentiation is not supported");
}

struct AlternativesNode : torch::autograd::Node {
  SavedVariable rows, ids, labels, lse, entropy;
  std::vector<int64_t> shape;
  bool inplace = false, spent = false;
  static constexpr const char* kWhat = "logits_tokens_backward";
  std::string name() const override { return "AlternativesBackward"; }
  void release_variables() override {
    for (SavedVariable* s : {&rows, &ids, &labels, &lse, &entropy}) s->reset_data();
  }
  // gradients of entropy, log-probabilities of the tokens, log-probability of the label (with labels)
  variable_list apply(variable_list&& g) override {
    const bool with_label = g.size() > 2 && g[2].defined();
    if (!g[0].defined() && !g[1].defined() && !with_label) return {Tensor()};
    if (spent) throw AxonError("the logits' storage holds the gradient of an earlier backward (inplace_backward)");
    const Tensor x = rows.unpack(), at = ids.unpack(), lab = labels.unpack(), l = lse.unpack(),
                 ent = entropy.unpack(shared_from_this());
    std::optional<at::NoGradGuard> no_grad(std::in_place);
    const Tensor g_en = g[0].defined() ? f32(g[0]) : Tensor(), g_ids = g[1].defined() ? f32(g[1]) : Tensor(),
                 g_lab = with_label ? f32(g[2]) : Tensor();
    same_place(kWhat, x, {&at, &lab, &l, &ent, &g_en, &g_ids, &g_lab});
    const int dtype = logits_dtype(kWhat, x);
    const int64_t n = x.size(0), v = x.size(1), k = at.size(1);
    if ((v > 1 && x.stride(1) != 1) || (n > 1 && x.stride(0) < v)) refuse(kWhat, "logits must be [tokens, vocab] with unit stride over the vocabulary");
    same_type(kWhat, at::kFloat, {&l, &ent});
    if (!is_index(at) || (lab.defined() && !is_index(lab))) refuse(kWhat, "a saved tensor has come back in another type");
    same_len(kWhat, "lse", 2 * n, l);
    same_len(kWhat, "entropy", n, ent);
    same_len(kWhat, "ids", n * k, at);
    if (g_en.defined()) same_len(kWhat, "g_entropy", n, g_en);
    if (g_ids.defined()) same_len(kWhat, "g_logprobs", n * k, g_ids);
    if (g_lab.defined()) { same_len(kWhat, "g_label", n, g_lab); same_len(kWhat, "labels", n, lab); }
    const c10::DeviceGuard device(x.device());
    Tensor out = inplace ? x : at::empty({n, v}, x.options());
    check(axon_logits_tokens_bwd(x.data_ptr(), dtype, row_stride(x), n, v, at.data_ptr(), is_i64(at), k, ptr(lab),
                                 lab.defined() && is_i64(lab), (const float*)l.data_ptr(), (const float*)ent.data_ptr(),
                                 (const float*)ptr(g_ids), (const float*)ptr(g_lab), (const float*)ptr(g_en), out.data_ptr(),
                                 row_stride(out), ::stream()),
          "axon_logits_tokens_bwd");
    spent = inplace;
    // what has been saved of these logits by others is no longer there: they refuse, as after any write in place
    if (inplace && !x.is_inference()) x.unsafeGetTensorImpl()->bump_version();
    out = out.view(shape);
    no_grad.reset();
    return {once(std::move(out), kWhat)};
  }
};

// The k best tokens of every position (ids_in none) or given ones: (label's log-probability or none, entropy, log-probabilities
// [..., k], ids).
std::tuple<OptTensor, Tensor, Tensor, Tensor> alternatives(const char* what, const Tensor& logits, int64_t k, const OptTensor& ids_in,
                                                           const OptTensor& labels, bool inplace) {
  const bool wants_grad = at::GradMode::is_enabled() && logits.requires_grad();
  no_tangent(what, logits);
  Tensor entropy, lp, label_lp, lse, ids, lab, rows;
  std::vector<int64_t> batch(logits.sizes().begin(), logits.dim() ? logits.sizes().end() - 1 : logits.sizes().end());
  {
    const at::NoGradGuard no_grad;
    rows = rows_of_logits(logits);
    const int64_t n = rows.size(0), v = rows.size(1);
    const int dtype = logits_dtype(what, rows);
    if (labels) {
      if (!is_index(*labels)) refuse(what, "labels must be int32 or int64");
      if (labels->device() != logits.device()) refuse(what, "operands live on different devices");
      if (labels->sizes() != at::IntArrayRef(batch))
        refuse(what, "labels " + shape_text(*labels) + " do not lie beside logits " + shape_text(logits));
      lab = labels->reshape({n}).contiguous();
    }
    if (ids_in) {
      const Tensor& t = *ids_in;
      if (!is_index(t)) refuse(what, std::string("token_ids must be int32 or int64, got ") + c10::toString(t.scalar_type()));
      if (t.device() != logits.device()) refuse(what, "operands live on different devices");
      if (t.dim() != logits.dim() || t.sizes().slice(0, t.dim() - 1) != logits.sizes().slice(0, logits.dim() - 1))
        refuse(what, "token_ids " + shape_text(t) + " do not lie beside logits " + shape_text(logits));
      k = t.size(-1);
      if (k < 1 || k > AXON_MAX_TOKEN_IDS)
        refuse(what, "between 1 and " + std::to_string(AXON_MAX_TOKEN_IDS) + " token ids per position, got " + std::to_string(k));
      ids = t.reshape({n, k}).contiguous();
    } else if (const int64_t most = std::min<int64_t>(AXON_MAX_TOP, v); k < 1 || k > most) {
      refuse(what, "k must be between 1 and " + std::to_string(most) + " (at most " + std::to_string(AXON_MAX_TOP) +
                       ", at most the vocabulary), got " + std::to_string(k));
    }
    require_device(rows, what);
    const c10::DeviceGuard device(rows.device());
    std::vector<int64_t> wide = batch;
    wide.push_back(k);
    entropy = at::empty(batch, opts(rows));
    lp = at::empty(wide, opts(rows));
    lse = at::empty({2, n}, opts(rows));
    if (lab.defined()) label_lp = at::empty(batch, opts(rows));
    const int64_t need = ids_in ? axon_logits_tokens_workspace_bytes(dtype, n, v) : axon_logits_top_workspace_bytes(dtype, n, v);
    const Tensor ws = need > 0 ? at::empty({need / 4}, opts(rows)) : Tensor();
    float *const ent_p = entropy.data_ptr<float>(), *const lse_p = lse.data_ptr<float>(), *const lp_p = lp.data_ptr<float>();
    if (ids_in) {
      check(axon_logits_tokens_fwd(rows.data_ptr(), dtype, row_stride(rows), n, v, ids.data_ptr(), is_i64(ids), k, lp_p, ent_p,
                                   lse_p, (float*)ptr(ws), std::max<int64_t>(need, 0), wants_grad, stream()),
            "axon_logits_tokens_fwd");
    } else {
      ids = at::empty(wide, opts(rows, at::kLong));
      check(axon_logits_top_fwd(rows.data_ptr(), dtype, row_stride(rows), n, v, k, ptr(lab), lab.defined() && is_i64(lab),
                                (float*)ptr(label_lp), ent_p, lse_p, lp_p, ids.data_ptr<int64_t>(), (float*)ptr(ws),
                                std::max<int64_t>(need, 0), wants_grad, stream()),
            "axon_logits_top_fwd");
    }
  }
  if (wants_grad) {
    std::shared_ptr<AlternativesNode> node(new AlternativesNode, torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(logits));
    node->shape = logits.sizes().vec();
    // writing the gradient over the logits is only possible in the caller's own storage
    node->inplace = inplace && rows.data_ptr() == logits.data_ptr();
    torch::autograd::set_history(entropy, node);
    torch::autograd::set_history(lp, node);
    if (label_lp.defined()) torch::autograd::set_history(label_lp, node);
    node->rows = SavedVariable(rows, false);
    node->ids = SavedVariable(ids.reshape({rows.size(0), k}), false);
    node->labels = SavedVariable(lab, false);
    node->lse = SavedVariable(lse, false);
    node->entropy = SavedVariable(entropy, true);
  }
  return {label_lp.defined() ? OptTensor(label_lp) : OptTensor(), entropy, lp, ids};
}

// The layers' router logits as the entry points take them.
struct RouterRows {
  std::vector<const void*> ptrs;
  int64_t ld = 0, n = 0, experts = 0;
  int dtype = 0;
};
// Rows of all layers with one row stride; a layer that lies otherwise is copied.
RouterRows router_rows(const char* what, variable_list& rows) {
  RouterRows r;
  const Tensor& first = rows[0];
  r.n = first.size(0);
  r.experts = first.size(1);
  r.dtype = logits_dtype(what, first);
  r.ld = r.n > 1 ? first.stride(0) : r.experts;
  bool same = r.ld >= r.experts;
  for (const Tensor& t : rows) {
    if (t.dim() != 2 || t.size(0) != r.n || t.size(1) != r.experts || t.scalar_type() != first.scalar_type() || t.device() != first.device())
      refuse(what, "the layers' logits must agree in shape, type and device");
    same = same && t.stride(1) == 1 && (r.n <= 1 || t.stride(0) == r.ld);
  }
  if (!same) {
    for (Tensor& t : rows) t = t.contiguous();
    r.ld = r.experts;
  }
  r.ptrs.reserve(rows.size());
  for (const Tensor& t : rows) r.ptrs.push_back(t.data_ptr());
  return r;
}

struct RouterBalanceNode : torch::autograd::Node {
  std::vector<SavedVariable> rows;
  SavedVariable mask, cu, coef, scale;
  std::vector<std::vector<int64_t>> shapes;  // of the inputs
  bool stacked = false;
  int mask_kind = 0, score = 0;
  static constexpr const char* kWhat = "router_balance_loss";
  std::string name() const override { return "RouterBalanceBackward"; }
  void release_variables() override {
    for (SavedVariable& s : rows) s.reset_data();
    for (SavedVariable* s : {&mask, &cu, &coef, &scale}) s->reset_data();
  }
  variable_list apply(variable_list&& g) override {
    variable_list grads(shapes.size());
    variable_list x;
    x.reserve(rows.size());
    for (SavedVariable& s : rows) x.push_back(s.unpack());
    const Tensor m = mask.unpack(), offsets = cu.unpack(), c = coef.unpack(), sc = scale.unpack();
    if (!g[0].defined()) return grads;
    {
      const at::NoGradGuard no_grad;
      const Tensor up = f32(g[0]);
      same_place(kWhat, x[0], {&m, &offsets, &c, &sc, &up});
      const RouterRows r = router_rows(kWhat, x);
      const int64_t layers = (int64_t)x.size(), seqs = offsets.defined() ? offsets.numel() - 1 : 1;
      same_type(kWhat, at::kFloat, {&c, &sc});
      same_type(kWhat, at::kInt, {&offsets});
      same_type(kWhat, mask_kind == AXON_MASK_I64 ? at::kLong : at::kFloat, {&m});
      same_len(kWhat, "coefficients", seqs * layers * r.experts, c);
      same_len(kWhat, "upstream gradient", 1, up);
      same_len(kWhat, "scale", 1, sc);
      for (const std::vector<int64_t>& shape : shapes)
        if (c10::multiply_integers(shape) != r.n * r.experts * (stacked ? layers : 1)) refuse(kWhat, "the saved logits have another size");
      if (m.defined()) same_len(kWhat, "token_mask", r.n, m);
      const c10::DeviceGuard device(x[0].device());
      // Every layer's gradient is a tensor with a storage of its own, which is kept, saved, resized or freed alone (48 of them,
      // without the dispatcher: 80 us of host time more than one allocation that they share).
      const int64_t eb = (int64_t)x[0].element_size(), cells = r.n * r.experts;
      c10::Allocator* const allocator = at::empty({0}, x[0].options()).storage().allocator();  // the one of tensors on this device
      std::vector<void*> out(layers, nullptr);
      for (size_t i = 0; i < shapes.size(); ++i) {
        if (!task_should_compute_output(i)) continue;
        grads[i] = at::detail::empty_generic(shapes[i], allocator, c10::DispatchKeySet(c10::DispatchKey::CUDA), x[0].scalar_type(),
                                             std::nullopt);
        char* const base = static_cast<char*>(grads[i].data_ptr());
        if (!stacked) out[i] = base;
        else
          for (int64_t l = 0; l < layers; ++l) out[l] = base + l * cells * eb;
      }
      check(axon_router_balance_bwd(r.ptrs.data(), r.dtype, r.ld, layers, r.n, r.experts, ptr(m), mask_kind,
                                    (const int32_t*)ptr(offsets), seqs, score, (const float*)ptr(c), (const float*)ptr(sc),
                                    (const float*)ptr(up), out.data(), ::stream()),
            "axon_router_balance_bwd");
    }
    if (at::GradMode::is_enabled())
      for (Tensor& t : grads)
        if (t.defined()) t = once(t, kWhat);
    return grads;
  }
};

// (loss, counts [layers, experts]); `logits`: the layers' [..., experts] or, stacked, one [layers, tokens, experts]; ids: one
// [..., k] per layer, or none.
std::tuple<Tensor, Tensor> router_balance(const variable_list& logits, bool stacked, int64_t k, const OptTensor& token_mask,
                                          const OptTensor& cu_seqlens, const std::optional<variable_list>& expert_ids, int score) {
  const char* const what = RouterBalanceNode::kWhat;
  bool wants_grad = false;
  for (const Tensor& t : logits) {
    wants_grad = wants_grad || t.requires_grad();
    no_tangent(what, t);
  }
  wants_grad = wants_grad && at::GradMode::is_enabled();
  variable_list rows, ids;
  Tensor mask, cu, loss, scale, coef, counts;
  int kind = 0;
  {
    const at::NoGradGuard no_grad;
    if (stacked) {
      rows = logits[0].detach().unbind(0);
    } else {
      rows.reserve(logits.size());
      for (const Tensor& t : logits) rows.push_back(t.dim() == 2 ? t : t.reshape({t.numel() / t.size(-1), t.size(-1)}));
    }
    const Tensor first = rows[0];
    const int64_t n = first.size(0), e = first.size(1), layers = (int64_t)rows.size();
    if (e > AXON_MAX_EXPERTS) refuse(what, "between 1 and " + std::to_string(AXON_MAX_EXPERTS) + " experts, got " + std::to_string(e));
    const RouterRows r = router_rows(what, rows);
    if (token_mask) {
      same_len(what, "token_mask", n, *token_mask);
      if (token_mask->device() != first.device()) refuse(what, "operands live on different devices");
      std::tie(mask, kind) = mask_arg(*token_mask);
    }
    if (cu_seqlens) {
      if (cu_seqlens->dim() != 1 || cu_seqlens->numel() < 1) refuse(what, "cu_seqlens must be [sequences + 1]");
      cu = cu_seqlens->detach().to(first.device(), at::kInt).contiguous();
    }
    std::vector<const void*> id_ptrs;
    if (expert_ids) {
      if ((int64_t)expert_ids->size() != layers)
        refuse(what, "expert_ids for " + std::to_string(expert_ids->size()) + " layers, logits of " + std::to_string(layers));
      for (const Tensor& t : *expert_ids) {
        if (!is_index(t) || t.scalar_type() != expert_ids->front().scalar_type())
          refuse(what, "expert_ids must be int32 or int64, the same in all layers");
        if (t.device() != first.device()) refuse(what, "operands live on different devices");
        if (t.dim() < 2 || t.size(-1) != k || t.numel() != n * k)
          refuse(what, "expert_ids " + shape_text(t) + " are not " + std::to_string(k) + " per token of " + std::to_string(n));
        ids.push_back(t.contiguous());
        id_ptrs.push_back(ids.back().data_ptr());
      }
    }
    require_device(first, what);
    const c10::DeviceGuard device(first.device());
    const int64_t seqs = cu.defined() ? cu.numel() - 1 : 1;
    loss = at::empty({}, opts(first));
    scale = at::empty({1}, opts(first));
    coef = at::empty({seqs, layers, e}, opts(first));
    counts = at::empty({layers, e}, opts(first, at::kLong));
    const int64_t bytes = axon_router_balance_workspace_bytes(n, seqs, layers, e);
    const Tensor ws = at::empty({bytes}, opts(first, at::kByte));
    check(axon_router_balance_fwd(r.ptrs.data(), r.dtype, r.ld, layers, n, e, k, expert_ids ? id_ptrs.data() : nullptr,
                                  expert_ids ? is_i64(ids[0]) : 0, ptr(mask), kind, (const int32_t*)ptr(cu), seqs, score,
                                  loss.data_ptr<float>(), coef.data_ptr<float>(), scale.data_ptr<float>(),
                                  counts.data_ptr<int64_t>(), ws.data_ptr(), bytes, stream()),
          "axon_router_balance_fwd");
  }
  if (wants_grad) {
    std::shared_ptr<RouterBalanceNode> node(new RouterBalanceNode, torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(logits));
    torch::autograd::set_history(loss, node);
    node->rows.reserve(rows.size());
    for (const Tensor& t : rows) node->rows.emplace_back(t, false);
    node->mask = SavedVariable(mask, false);
    node->cu = SavedVariable(cu, false);
    node->coef = SavedVariable(coef, false);
    node->scale = SavedVariable(scale, false);
    for (const Tensor& t : logits) node->shapes.push_back(t.sizes().vec());
    node->stacked = stacked;
    node->mask_kind = kind;
    node->score = score;
  }
  return {loss, counts};
}

// ---------------------------------------------------------------------------------------------------------------------
// Controls of logits: what a sampler does to them before it draws.
// ---------------------------------------------------------------------------------------------------------------------

// The operands of axon_controls, checked and held.  Nothing is computed here: the tensors are read by every launch.
class Controls {
 public:
  enum Which { kTokens, kOffsets, kOwnMask, kRepetition, kFrequency, kPresence, kTemperature, kBiasIds, kBias, kAllowed, kIndex, kCount };
  typedef std::pair<double, OptTensor> Value;  // for all sequences, or one for each

  Controls(const OptTensor& token_ids, const OptTensor& cu_seqlens, bool every_position, const OptTensor& own_mask, const Value& repetition,
           const Value& frequency, const Value& presence, const OptTensor& bias_ids, const OptTensor& bias, const OptTensor& allowed,
           const OptTensor& allowed_index, const Value& temperature) {
    const at::NoGradGuard no_grad;
    c_.every_position = every_position;
    c_.n_seqs = -1;  // not known yet
    if (cu_seqlens) {
      if (cu_seqlens->dim() != 1 || cu_seqlens->numel() < 1) refuse(kWhat, "cu_seqlens must be [sequences + 1]");
      hold(kOffsets, cu_seqlens->detach().to(at::kInt).contiguous());
      c_.cu_seqlens = (const int32_t*)ptr(held_[kOffsets]);
      c_.n_seqs = cu_seqlens->numel() - 1;
    }
    if (token_ids) {
      if (!is_index(*token_ids)) refuse(kWhat, std::string("token_ids must be int32 or int64, got ") + c10::toString(token_ids->scalar_type()));
      if (!cu_seqlens) {
        if (token_ids->dim() != 1 && token_ids->dim() != 2) refuse(kWhat, "token_ids must be [sequences, length], or packed with cu_seqlens");
        c_.uniform_len = token_ids->size(-1);
        c_.n_seqs = token_ids->dim() == 2 ? token_ids->size(0) : 1;
      }
      if (token_ids->numel() >= INT32_MAX) refuse(kWhat, "more tokens than 32 bits count");
      c_.n_tokens = token_ids->numel();
      hold(kTokens, token_ids->detach().contiguous());
      c_.token_ids = c_.n_tokens > 0 ? held_[kTokens].data_ptr() : nullptr;  // no tokens, no history
      c_.token_ids_i64 = is_i64(*token_ids);
    }
    if (own_mask) {
      if (!token_ids || own_mask->numel() != token_ids->numel()) refuse(kWhat, "response_mask does not lie beside token_ids");
      auto m = mask_arg(*own_mask);
      c_.mask_kind = m.second;
      hold(kOwnMask, std::move(m.first));
      c_.own_mask = ptr(held_[kOwnMask]);
    }
    c_.repetition_all = (float)repetition.first;
    c_.frequency_all = (float)frequency.first;
    c_.presence_all = (float)presence.first;
    c_.temperature_all = (float)temperature.first;
    c_.repetition = value(kRepetition, repetition, "repetition_penalty");
    c_.frequency = value(kFrequency, frequency, "frequency_penalty");
    c_.presence = value(kPresence, presence, "presence_penalty");
    c_.temperature = value(kTemperature, temperature, "temperature");
    const auto usable = [](float x, bool positive) { return std::isfinite(x) && (!positive || x >= 0x1p-126f); };
    if (!usable(c_.repetition_all, true)) refuse(kWhat, "repetition_penalty must be positive (2^-126 or more)");
    if (!usable(c_.temperature_all, true)) refuse(kWhat, "temperature must be positive (2^-126 or more)");
    if (!usable(c_.frequency_all, false) || !usable(c_.presence_all, false)) refuse(kWhat, "frequency_penalty and presence_penalty must be finite");
    if (!token_ids && (c_.repetition || c_.frequency || c_.presence || c_.repetition_all != 1.f || c_.frequency_all != 0.f || c_.presence_all != 0.f))
      refuse(kWhat, "penalties need token_ids");
    if (bias_ids.has_value() != bias.has_value()) refuse(kWhat, "bias_ids and bias come together");
    if (bias) {
      if (!is_index(*bias_ids)) refuse(kWhat, "bias_ids must be int32 or int64");
      if (bias_ids->sizes() != bias->sizes() || bias->dim() < 1 || bias->dim() > 2)
        refuse(kWhat, "bias_ids " + shape_text(*bias_ids) + " and bias " + shape_text(*bias) + " must both be [k] or [sequences, k]");
      constant(*bias, "bias");
      if (bias->dim() == 2) sequences(bias->size(0), "bias");
      c_.bias_per_seq = bias->dim() == 2;
      c_.n_bias = bias->size(-1);
      c_.bias_ids_i64 = is_i64(*bias_ids);
      hold(kBiasIds, bias_ids->detach().contiguous());
      hold(kBias, f32(*bias));
      c_.bias_ids = held_[kBiasIds].data_ptr();
      c_.bias = (const float*)held_[kBias].data_ptr();
    }
    if (allowed_index && !allowed) refuse(kWhat, "allowed_index without allowed");
    if (allowed) {
      if (allowed->scalar_type() != at::kInt || allowed->dim() < 1 || allowed->dim() > 2 || allowed->size(-1) < 1 || allowed->size(0) < 1)
        refuse(kWhat, "allowed must be int32 [words] or [masks, words], 32 tokens a word");
      Tensor a = allowed->dim() == 1 ? allowed->detach().unsqueeze(0) : allowed->detach();
      if (a.stride(1) != 1 || (a.size(0) > 1 && a.stride(0) < a.size(1))) a = a.contiguous();
      c_.allowed = (const int32_t*)a.data_ptr();
      c_.allowed_rows = a.size(0);
      c_.allowed_stride = a.size(0) > 1 ? a.stride(0) : a.size(1);
      words_ = a.size(1);
      hold(kAllowed, std::move(a));
      if (allowed_index) {
        if (!is_index(*allowed_index)) refuse(kWhat, "allowed_index must be int32 or int64");
        hold(kIndex, allowed_index->detach().contiguous());
        c_.allowed_index = held_[kIndex].data_ptr();
        c_.allowed_index_i64 = is_i64(*allowed_index);
      }
    }
    for (const Tensor& t : held_)
      if (t.defined() && t.is_cuda()) made_on_ = c10::impl::VirtualGuardImpl(t.device().type()).getStream(t.device());
  }

  // For n rows of v logits that lie where `like` does.
  axon_controls of(const char* what, const Tensor& like, int64_t n, int64_t v) const {
    axon_controls c = c_;
    for (const Tensor& t : held_)
      if (t.defined() && t.device() != like.device()) refuse(what, "logits and controls live on different devices");
    if (made_on_) {  // what is held may be a copy that nobody else knows of: its memory waits for other streams' launches too
      const c10::Stream now = c10::impl::VirtualGuardImpl(like.device().type()).getStream(like.device());
      if (now != *made_on_)
        for (const Tensor& t : held_)
          if (t.defined()) t.record_stream(now);
    }
    if (c.every_position ? (held_[kTokens].defined() && n != c.n_tokens) : (c.n_seqs >= 0 && n != c.n_seqs))
      refuse(what, std::to_string(n) + " rows of logits for controls of " +
                       (c.every_position ? std::to_string(c.n_tokens) + " positions" : std::to_string(c.n_seqs) + " sequences"));
    if (n > 0 && c.every_position && !c.cu_seqlens && c.uniform_len == 0 && c.n_seqs >= 0)
      refuse(what, "values for each sequence need token_ids or cu_seqlens");
    if (c.n_seqs < 0) c.n_seqs = 0;
    if (c.allowed) {
      if (words_ < (v + 31) / 32) refuse(what, "allowed has " + std::to_string(words_) + " words for a vocabulary of " + std::to_string(v));
      const Tensor& index = held_[kIndex];
      if (index.defined() ? index.numel() != n : (c.allowed_rows != 1 && c.allowed_rows != n))
        refuse(what, "allowed needs one mask, one for each of the " + std::to_string(n) + " rows, or an allowed_index of as many entries");
    }
    return c;
  }
  const Tensor& held(int i) const { return held_[i]; }

 private:
  static constexpr const char* kWhat = "LogitControls";
  void hold(Which i, Tensor t) { held_[i] = std::move(t); }
  void constant(const Tensor& t, const char* name) {
    if (t.requires_grad()) refuse(kWhat, std::string(name) + " has no gradient: pass it detached");
  }
  void sequences(int64_t n, const char* name) {
    if (c_.n_seqs >= 0 && n != c_.n_seqs)
      refuse(kWhat, std::string(name) + " for " + std::to_string(n) + " sequences of " + std::to_string(c_.n_seqs));
    c_.n_seqs = n;
  }
  const float* value(Which i, const Value& v, const char* name) {
    if (!v.second) return nullptr;
    if (v.second->dim() != 1 || !v.second->is_floating_point()) refuse(kWhat, std::string(name) + " must be a number or a float tensor [sequences]");
    constant(*v.second, name);
    sequences(v.second->numel(), name);
    hold(i, f32(*v.second));
    return (const float*)ptr(held_[i]);
  }

  axon_controls c_{};
  std::array<Tensor, kCount> held_;
  c10::optional<c10::Stream> made_on_;
  int64_t words_ = 0;
};

// The controls' tensors as a node saves them: one that is written to before the backward is noticed.
struct SavedControls {
  std::shared_ptr<Controls> controls;
  std::vector<SavedVariable> held;
  void save(std::shared_ptr<Controls> c) {
    for (int i = 0; i < Controls::kCount; ++i)
      if (c->held(i).defined()) held.emplace_back(c->held(i), false);
    controls = std::move(c);
  }
  void release() {
    for (SavedVariable& s : held) s.reset_data();
  }
  const Controls& unpack() {
    for (SavedVariable& s : held) (void)s.unpack();  // raises where one has changed
    return *controls;
  }
};

// The saved rows of logits, as a hook may have handed them back.
void check_saved_rows(const char* what, const Tensor& x) {
  require_device(x, what);
  if (x.dim() != 2 || (x.size(1) > 1 && x.stride(1) != 1) || (x.size(0) > 1 && x.stride(0) < x.size(1)))
    refuse(what, "logits must be [tokens, vocab] with unit stride over the vocabulary");
}

struct ControlledLogitsNode : torch::autograd::Node {
  SavedVariable rows;
  SavedControls controls;
  std::vector<int64_t> shape;
  static constexpr const char* kWhat = "controlled_logits_backward";
  std::string name() const override { return "ControlledLogitsBackward"; }
  void release_variables() override {
    rows.reset_data();
    controls.release();
  }
  variable_list apply(variable_list&& g) override {
    if (!g[0].defined()) return {Tensor()};
    const Tensor x = rows.unpack();
    const Controls& ctl = controls.unpack();
    Tensor out;
    {
      const at::NoGradGuard no_grad;
      check_saved_rows(kWhat, x);
      const int64_t n = x.size(0), v = x.size(1);
      const int dtype = logits_dtype(kWhat, x);
      if (g[0].numel() != n * v || g[0].device() != x.device()) refuse(kWhat, "the gradient does not lie beside the logits");
      const Tensor up = rows_of_logits(g[0].to(x.scalar_type()));
      const axon_controls c = ctl.of(kWhat, x, n, v);
      const c10::DeviceGuard device(x.device());
      out = at::empty({n, v}, x.options());
      check(axon_controls_apply_bwd(x.data_ptr(), dtype, row_stride(x), n, v, &c, up.data_ptr(), row_stride(up), out.data_ptr(), v,
                                    ::stream()),
            "axon_controls_apply_bwd");
      out = out.view(shape);
    }
    return {once(std::move(out), kWhat)};
  }
};

Tensor controlled_logits(const Tensor& logits, std::shared_ptr<Controls> controls, bool inplace) {
  const char* const what = "controlled_logits";
  const bool wants_grad = at::GradMode::is_enabled() && logits.requires_grad();
  no_tangent(what, logits);
  if (inplace && wants_grad) refuse(what, "logits that require a gradient cannot be written over");
  Tensor rows, out;
  {
    const at::NoGradGuard no_grad;
    rows = rows_of_logits(logits);
    const int64_t n = rows.size(0), v = rows.size(1);
    const int dtype = logits_dtype(what, rows);
    if (inplace && rows.data_ptr() != logits.data_ptr()) refuse(what, "logits can be written over only where their rows lie as they are read");
    const axon_controls c = controls->of(what, rows, n, v);
    require_device(rows, what);
    const c10::DeviceGuard device(rows.device());
    out = inplace ? rows : at::empty({n, v}, rows.options());
    check(axon_controls_apply(rows.data_ptr(), dtype, row_stride(rows), n, v, &c, out.data_ptr(), row_stride(out), stream()),
          "axon_controls_apply");
    if (inplace && !logits.is_inference()) logits.unsafeGetTensorImpl()->bump_version();
    out = inplace ? logits : out.view(logits.sizes());
  }
  if (wants_grad) {
    std::shared_ptr<ControlledLogitsNode> node(new ControlledLogitsNode, torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(logits));
    node->shape = logits.sizes().vec();
    torch::autograd::set_history(out, node);
    node->rows = SavedVariable(rows, false);
    node->controls.save(std::move(controls));
  }
  return out;
}

struct ControlledLogprobsNode : torch::autograd::Node {
  SavedVariable rows, labels, stats;
  SavedControls controls;
  std::vector<int64_t> shape;
  bool inplace = false, spent = false;
  static constexpr const char* kWhat = "controlled_logprobs_backward";
  std::string name() const override { return "ControlledLogprobsBackward"; }
  void release_variables() override {
    for (SavedVariable* s : {&rows, &labels, &stats}) s->reset_data();
    controls.release();
  }
  // gradients of the log-probability and the entropy
  variable_list apply(variable_list&& g) override {
    if (!g[0].defined() && !g[1].defined()) return {Tensor()};
    if (spent) throw AxonError("the logits' storage holds the gradient of an earlier backward (inplace_backward)");
    const Tensor x = rows.unpack(), lab = labels.unpack(), st = stats.unpack();
    const Controls& ctl = controls.unpack();
    Tensor out;
    {
      const at::NoGradGuard no_grad;
      check_saved_rows(kWhat, x);
      const int64_t n = x.size(0), v = x.size(1);
      const Tensor g_lp = g[0].defined() ? f32(g[0]) : Tensor(), g_en = g[1].defined() ? f32(g[1]) : Tensor();
      same_place(kWhat, x, {&lab, &st, &g_lp, &g_en});
      const int dtype = logits_dtype(kWhat, x);
      same_type(kWhat, at::kFloat, {&st});
      if (!is_index(lab)) refuse(kWhat, "a saved tensor has come back in another type");
      same_len(kWhat, "labels", n, lab);
      same_len(kWhat, "statistics", 3 * n, st);
      if (g_lp.defined()) same_len(kWhat, "g_logprobs", n, g_lp);
      if (g_en.defined()) same_len(kWhat, "g_entropy", n, g_en);
      const axon_controls c = ctl.of(kWhat, x, n, v);
      const c10::DeviceGuard device(x.device());
      out = inplace ? x : at::empty({n, v}, x.options());
      check(axon_controls_logprob_bwd(x.data_ptr(), dtype, row_stride(x), n, v, &c, lab.data_ptr(), is_i64(lab), (const float*)st.data_ptr(),
                                      (const float*)ptr(g_lp), (const float*)ptr(g_en), out.data_ptr(), row_stride(out), ::stream()),
            "axon_controls_logprob_bwd");
      spent = inplace;
      if (inplace && !x.is_inference()) x.unsafeGetTensorImpl()->bump_version();
      out = out.view(shape);
    }
    return {once(std::move(out), kWhat)};
  }
};

// (log-probability of the label, entropy)
std::tuple<Tensor, Tensor> controlled_logprobs(const Tensor& logits, const Tensor& labels, std::shared_ptr<Controls> controls, bool inplace) {
  const char* const what = "controlled_logprobs_from_logits";
  const bool wants_grad = at::GradMode::is_enabled() && logits.requires_grad();
  no_tangent(what, logits);
  Tensor rows, lab, lp, entropy, stats;
  {
    const at::NoGradGuard no_grad;
    rows = rows_of_logits(logits);
    const int64_t n = rows.size(0), v = rows.size(1);
    const int dtype = logits_dtype(what, rows);
    const std::vector<int64_t> batch(logits.sizes().begin(), logits.sizes().end() - 1);
    if (!is_index(labels)) refuse(what, "labels must be int32 or int64");
    if (labels.device() != logits.device()) refuse(what, "operands live on different devices");
    if (labels.sizes() != at::IntArrayRef(batch))
      refuse(what, "labels " + shape_text(labels) + " do not lie beside logits " + shape_text(logits));
    lab = labels.detach().reshape({n}).contiguous();
    const axon_controls c = controls->of(what, rows, n, v);
    require_device(rows, what);
    const c10::DeviceGuard device(rows.device());
    lp = at::empty(batch, opts(rows));
    entropy = at::empty(batch, opts(rows));
    stats = at::empty({3, n}, opts(rows));
    const int64_t need = axon_controls_logprob_workspace_bytes(n, v);
    const Tensor ws = at::empty({std::max<int64_t>(need, 0)}, opts(rows, at::kByte));
    check(axon_controls_logprob_fwd(rows.data_ptr(), dtype, row_stride(rows), n, v, &c, lab.data_ptr(), is_i64(lab), lp.data_ptr<float>(),
                                    entropy.data_ptr<float>(), stats.data_ptr<float>(), ws.data_ptr(), need, wants_grad, stream()),
          "axon_controls_logprob_fwd");
  }
  if (wants_grad) {
    std::shared_ptr<ControlledLogprobsNode> node(new ControlledLogprobsNode, torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(logits));
    node->shape = logits.sizes().vec();
    node->inplace = inplace && rows.data_ptr() == logits.data_ptr();
    torch::autograd::set_history(lp, node);
    torch::autograd::set_history(entropy, node);
    node->rows = SavedVariable(rows, false);
    node->labels = SavedVariable(lab, false);
    node->stats = SavedVariable(stats, false);
    node->controls.save(std::move(controls));
  }
  return {lp, entropy};
}

// ---------------------------------------------------------------------------------------------------------------------
// Distillation from a teacher's top logits.
// ---------------------------------------------------------------------------------------------------------------------

// The graph that the current stream is being captured into, 0 outside of a capture.
unsigned long long capture_id() {
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  unsigned long long id = 0;
  if (hipStreamGetCaptureInfo((hipStream_t)::stream(), &status, &id) != hipSuccess) throw AxonError("the state of the stream cannot be asked for");
  return status == hipStreamCaptureStatusActive ? id : 0;
}

struct DistillNode : torch::autograd::Node {
  SavedVariable rows, ids, state, weights;  // state: coefficients [4][n], then the gradients of the tokens' log-probabilities [n][k]
  Tensor ready;  // with weights: the gradient of an upstream gradient of 1, which the forward has left
  unsigned long long captured = 0;  // ... into this graph
  std::vector<int64_t> shape;
  float temperature = 1.f;
  bool weighted = false, inplace = false, spent = false;
  static constexpr const char* kWhat = "distillation_backward";
  std::string name() const override { return "DistillationBackward"; }
  void release_variables() override {
    for (SavedVariable* s : {&rows, &ids, &state, &weights}) s->reset_data();
    ready.reset();
  }
  variable_list apply(variable_list&& g) override {
    if (!g[0].defined()) return {Tensor()};
    if (spent) throw AxonError("the logits' storage holds the gradient of an earlier backward (inplace_backward)");
    const Tensor x = rows.unpack(), at = ids.unpack(), st = state.unpack(), w = weights.unpack();
    Tensor out;
    {
      const at::NoGradGuard no_grad;
      check_saved_rows(kWhat, x);
      const int64_t n = x.size(0), v = x.size(1);
      const Tensor up = f32(g[0]);
      same_place(kWhat, x, {&at, &st, &w, &up});
      const int dtype = logits_dtype(kWhat, x);
      same_type(kWhat, at::kFloat, {&st, &w});
      if (!is_index(at) || at.dim() != 2) refuse(kWhat, "a saved tensor has come back in another type");
      const int64_t k = at.size(1);
      same_len(kWhat, "ids", n * k, at);
      same_len(kWhat, "coefficients", n * (4 + k), st);
      same_len(kWhat, "upstream gradient", weighted ? 1 : n, up);
      if (weighted) same_len(kWhat, "token_weights", n, w);
      const c10::DeviceGuard device(x.device());
      // The gradient that the forward has left is handed on once, and only where a replay of this launch comes behind one of the
      // forward's: what a caller does to it must not come back.
      const bool there = ready.defined() && captured == capture_id();
      out = there ? ready : inplace ? x : at::empty({n, v}, x.options());
      ready.reset();
      check(axon_distill_bwd(x.data_ptr(), dtype, row_stride(x), n, v, at.data_ptr(), is_i64(at), k, (const float*)ptr(w), temperature,
                             (const float*)st.data_ptr() + 4 * n, (const float*)st.data_ptr(), (const float*)up.data_ptr(), there, out.data_ptr(),
                             row_stride(out), ::stream()),
            "axon_distill_bwd");
      spent = inplace;
      if (inplace && !x.is_inference()) x.unsafeGetTensorImpl()->bump_version();
      out = out.view(shape);
    }
    return {once(std::move(out), kWhat)};
  }
};

// (weighted sum of the losses or none, losses, covered)
std::tuple<OptTensor, Tensor, Tensor> distill(const char* what, const Tensor& logits, const Tensor& teacher_ids, const Tensor& teacher_logprobs,
                                              const OptTensor& token_weights, int divergence, int tail, double beta, double temperature,
                                              bool inplace) {
  const bool wants_grad = at::GradMode::is_enabled() && logits.requires_grad();
  no_tangent(what, logits);
  Tensor rows, ids, w, loss, losses, covered, state, ready;
  {
    const at::NoGradGuard no_grad;
    rows = rows_of_logits(logits);
    const int64_t n = rows.size(0), v = rows.size(1);
    const int dtype = logits_dtype(what, rows);
    const std::vector<int64_t> batch(logits.sizes().begin(), logits.sizes().end() - 1);
    if (!is_index(teacher_ids)) refuse(what, std::string("teacher_ids must be int32 or int64, got ") + c10::toString(teacher_ids.scalar_type()));
    if (!teacher_logprobs.is_floating_point()) refuse(what, "teacher_logprobs must be floating point");
    if (teacher_ids.dim() != logits.dim() || teacher_ids.sizes().slice(0, teacher_ids.dim() - 1) != at::IntArrayRef(batch))
      refuse(what, "teacher_ids " + shape_text(teacher_ids) + " do not lie beside logits " + shape_text(logits));
    if (teacher_logprobs.sizes() != teacher_ids.sizes())
      refuse(what, "teacher_logprobs " + shape_text(teacher_logprobs) + " do not lie beside teacher_ids " + shape_text(teacher_ids));
    if (teacher_logprobs.requires_grad()) refuse(what, "teacher_logprobs have no gradient: pass them detached");
    const int64_t k = teacher_ids.size(-1);
    if (k < 1 || k > AXON_MAX_TOKEN_IDS)
      refuse(what, "between 1 and " + std::to_string(AXON_MAX_TOKEN_IDS) + " teacher_ids per position, got " + std::to_string(k));
    for (const Tensor* t : {&teacher_ids, &teacher_logprobs})
      if (t->device() != logits.device()) refuse(what, "operands live on different devices");
    if (token_weights) {
      if (token_weights->sizes() != at::IntArrayRef(batch))
        refuse(what, "token_weights " + shape_text(*token_weights) + " do not lie beside logits " + shape_text(logits));
      if (token_weights->requires_grad()) refuse(what, "token_weights have no gradient: pass them detached");
      if (token_weights->device() != logits.device()) refuse(what, "operands live on different devices");
    }
    require_device(rows, what);
    const c10::DeviceGuard device(rows.device());
    ids = teacher_ids.reshape({n, k}).contiguous();
    const Tensor lq = f32(teacher_logprobs);
    if (teacher_logprobs.scalar_type() == at::kBFloat16) tail |= AXON_DISTILL_FROM_BF16;
    else if (teacher_logprobs.scalar_type() == at::kHalf) tail |= AXON_DISTILL_FROM_F16;
    if (token_weights) w = f32(*token_weights);
    losses = at::empty(batch, opts(rows));
    covered = at::empty(batch, opts(rows));
    state = at::empty({n * (4 + k)}, opts(rows));
    const int64_t need = axon_distill_workspace_bytes(dtype, n, v);
    const Tensor ws = at::empty({std::max<int64_t>(need, 0)}, opts(rows, at::kByte));
    float *const losses_p = losses.data_ptr<float>(), *const covered_p = covered.data_ptr<float>(), *const coef_p = state.data_ptr<float>(),
                *const grads_p = coef_p + 4 * n;
    if (token_weights) {
      loss = at::empty({}, opts(rows));
      if (wants_grad) ready = at::empty({n, v}, rows.options());
      check(axon_distill_loss(rows.data_ptr(), dtype, row_stride(rows), n, v, ids.data_ptr(), is_i64(ids), (const float*)lq.data_ptr(), k,
                              (const float*)w.data_ptr(), divergence, tail, (float)beta, (float)temperature, loss.data_ptr<float>(), losses_p,
                              covered_p, grads_p, coef_p, wants_grad ? ready.data_ptr() : nullptr, v, ws.data_ptr(), need, stream()),
            "axon_distill_loss");
    } else {
      check(axon_distill_fwd(rows.data_ptr(), dtype, row_stride(rows), n, v, ids.data_ptr(), is_i64(ids), (const float*)lq.data_ptr(), k, nullptr,
                             divergence, tail, (float)beta, (float)temperature, losses_p, covered_p, grads_p, coef_p, ws.data_ptr(), need,
                             wants_grad, stream()),
            "axon_distill_fwd");
    }
  }
  if (wants_grad) {
    std::shared_ptr<DistillNode> node(new DistillNode, torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(logits));
    node->shape = logits.sizes().vec();
    node->weighted = token_weights.has_value();
    node->inplace = !node->weighted && inplace && rows.data_ptr() == logits.data_ptr();
    node->temperature = (float)temperature;
    torch::autograd::set_history(node->weighted ? loss : losses, node);
    node->rows = SavedVariable(rows, false);
    node->ids = SavedVariable(ids, false);
    node->state = SavedVariable(state, false);
    node->weights = SavedVariable(w, false);
    if (node->weighted) {
      const c10::DeviceGuard device(rows.device());
      node->captured = capture_id();
      node->ready = std::move(ready);
    }
  }
  return {loss.defined() ? OptTensor(loss) : OptTensor(), losses, covered};
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  g_error = py::object(py::module_::import("axon_amd._lib").attr("AxonAmdError")).release().ptr();
  py::register_exception_translator([](std::exception_ptr e) {
    try {
      if (e) std::rethrow_exception(e);
    } catch (const AxonError& err) {
      PyErr_SetString(g_error, err.what());
    }
  });
  // what this file was compiled against: axon_amd/_lib.py refuses another
  m.attr("abi_version") = AXON_AMD_ABI_VERSION;
  m.attr("torch_version") = AXON_TORCH_VERSION;
  const py::call_guard<py::gil_scoped_release> unlocked;
  py::class_<Post>(m, "Post")
      .def(py::init<OptTensor>())
      .def_property_readonly("sent", &Post::is_sent)
      .def("sums", &Post::sums, unlocked)
      .def("wait", &Post::wait, unlocked);
  m.def("post_slots", [] { return Slots::get().made(); });
  m.def("policy_loss", &policy_loss, unlocked);
  m.def("group_advantage", &group_advantage, unlocked);
  m.def("sampler_correction_diag", &sampler_correction_diag, unlocked);
  m.def("reverse_scan", &reverse_scan, unlocked);
  m.def("scale_f32", &scale_f32, unlocked);
  m.def("finished_loss", [](const Tensor& x, const Tensor& acc, const Tensor& grad, double factor,
                            int64_t slot) { return FinishedLoss::apply(x, acc, grad, factor, slot); }, unlocked);
  m.def("top_logprobs", [](const Tensor& logits, int64_t k, const OptTensor& labels, bool inplace) {
    return alternatives("top_logprobs_from_logits", logits, k, OptTensor(), labels, inplace);
  }, unlocked);
  m.def("token_logprobs", [](const Tensor& logits, const Tensor& token_ids, bool inplace) {
    return alternatives("token_logprobs_from_logits", logits, 0, token_ids, OptTensor(), inplace);
  }, unlocked);
  m.def("router_balance", &router_balance, unlocked);
  py::class_<Controls, std::shared_ptr<Controls>>(m, "Controls")
      .def(py::init<const OptTensor&, const OptTensor&, bool, const OptTensor&, const Controls::Value&, const Controls::Value&,
                    const Controls::Value&, const OptTensor&, const OptTensor&, const OptTensor&, const OptTensor&, const Controls::Value&>(),
           unlocked);
  m.def("distill", [](const Tensor& logits, const Tensor& ids, const Tensor& logprobs, const OptTensor& weights, int divergence, int tail,
                      double beta, double temperature, bool inplace) {
    return distill(weights ? "distillation_loss_from_logits" : "distillation_from_logits", logits, ids, logprobs, weights, divergence, tail,
                   beta, temperature, inplace);
  }, unlocked);
  m.def("controlled_logits", &controlled_logits, unlocked);
  m.def("controlled_logprobs", &controlled_logprobs, unlocked);
}
