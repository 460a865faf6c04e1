// Eager calls of the distribution operators as torch autograd nodes (host code only).
//
// The kernels are reached through the C ABI (depthwarp.h) like everywhere else; this file holds what an eager call
// does around them -- outputs, workspace, stream, and the node of the backward pass.  It is C++ because small
// training steps are bound by it: a node written in Python runs in the autograd engine's own thread, where the
// interpreter's lock and cold caches took about half of such a step (80 to 90 us, 4 x 64 x 4 x 4).
//
// The library's functions come from Python as addresses, what a call has to know as a list of words: which build of
// the library is in use, and what the shapes and types decide, is settled there (distribution.py).  These calls launch
// by pointer, so nothing that records or replaces tensor operations sees more of them than their outputs being made:
// distribution.py calls the registered operators wherever something of the kind watches.
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/library.h>

#include <cstring>
#include <optional>
#include <string>
#include <vector>

#include "depthwarp.h"

namespace {
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Library {
  decltype(&dw_strerror) strerror;
  decltype(&dw_log_probs_fwd) log_probs_fwd;
  decltype(&dw_log_probs_bwd) log_probs_bwd;
  decltype(&dw_distill_fwd) distill_fwd;
  decltype(&dw_distill_bwd) distill_bwd;
} lib{};

void bind(int64_t strerror, int64_t lp_fwd, int64_t lp_bwd, int64_t ds_fwd, int64_t ds_bwd) {
  lib.strerror = reinterpret_cast<decltype(lib.strerror)>(strerror);
  lib.log_probs_fwd = reinterpret_cast<decltype(lib.log_probs_fwd)>(lp_fwd);
  lib.log_probs_bwd = reinterpret_cast<decltype(lib.log_probs_bwd)>(lp_bwd);
  lib.distill_fwd = reinterpret_cast<decltype(lib.distill_fwd)>(ds_fwd);
  lib.distill_bwd = reinterpret_cast<decltype(lib.distill_bwd)>(ds_bwd);
}
void check(int code, const char* what) {
  TORCH_CHECK(code == DW_OK, what, " failed: ", lib.strerror(code), " (code ", code, ")");
}
void* stream_of(const Tensor& t) {
  return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}
template <class T>
T* data(const Tensor& t) { return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr; }
void* data(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
// (a tensor may stand for its memory's values with the other sign: at::_neg_view)
Tensor contiguous(const Tensor& t) { return t.defined() ? t.resolve_neg().contiguous() : t; }
// How the kernels read a tensor: in memory order, with the classes (or entries) last in memory, or neither: a copy of it
enum Layout : int64_t { kInOrder = 0, kLast = 1, kCopy = 2 };
Tensor in_place(const Tensor& t, int64_t layout) { return layout == kCopy ? contiguous(t) : t.resolve_neg(); }
bool has_last(const Tensor& t, int64_t dim) {
  int64_t step = t.size(dim);
  bool ok = step == 1 || t.stride(dim) == 1;
  for (int64_t i = t.dim() - 1; i >= 0; --i) {
    if (i == dim || t.size(i) == 1) continue;
    ok = ok && t.stride(i) == step;
    step *= t.size(i);
  }
  return ok;
}
// The same in the backward pass, where hooks for saved tensors may have brought them back in another order
Tensor saved_in_place(const Tensor& saved, int64_t layout, int64_t dim) {
  if (layout != kLast) return contiguous(saved);
  const Tensor t = saved.resolve_neg();
  return has_last(t, dim) ? t : t.movedim(dim, -1).contiguous().movedim(-1, dim);
}
Tensor workspace(const Tensor& x, int64_t bytes) {
  // allocated for each call: calls on other streams, or captured into other graphs, have their own
  return bytes ? at::empty({bytes}, x.options().dtype(at::kByte)) : Tensor();
}
std::vector<int64_t> with(at::IntArrayRef rows, int64_t at, int64_t n) {
  std::vector<int64_t> s(rows.begin(), rows.end());
  s.insert(s.begin() + at, n);
  return s;
}

// What a call has to know, by value (a call that is kept for later holds no address of this process): the words of this
// struct.  They travel with the node to the backward pass.
struct Call {
  dw_dist_desc desc;
  int64_t nbytes, dim, top, layout, list_layout;
};
Call call_of(at::IntArrayRef words) {
  Call c;
  static_assert(sizeof c % sizeof(int64_t) == 0);
  TORCH_CHECK(words.size() * sizeof(int64_t) == sizeof c, "expected ", sizeof c / sizeof(int64_t), " words, got ", words.size());
  std::memcpy(&c, words.data(), sizeof c);
  return c;
}
void keep(AutogradContext* ctx, const Call& c) {
  ctx->saved_data["call"] = std::string(reinterpret_cast<const char*>(&c), sizeof c);
}
Call kept(AutogradContext* ctx) {
  Call c;
  std::memcpy(&c, ctx->saved_data["call"].toStringRef().data(), sizeof c);
  return c;
}
// The gradients are differentiable once.  Where a pass builds a graph of itself, using that graph is an error.
Tensor once(Tensor grad) {
  if (!at::GradMode::is_enabled()) return grad;
  grad = grad.detach();
  grad.requires_grad_(true);
  auto node = std::make_shared<torch::autograd::DelayedError>(
      "trying to differentiate twice a function that was marked with @once_differentiable", 1);
  return (*node)({grad})[0];
}

struct LogProbs : torch::autograd::Function<LogProbs> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const std::optional<Tensor>& given,
                               at::IntArrayRef words, at::IntArrayRef rows, bool train) {
    const Call c = call_of(words);
    const int64_t top = c.top;
    const Tensor x = in_place(logits, c.layout), index_in = given ? *given : Tensor(), index = contiguous(index_in);
    const c10::OptionalDeviceGuard guard(x.device());
    const auto f32 = x.options().dtype(at::kFloat).memory_format(std::nullopt);
    Tensor ent = at::empty(rows, f32), lp, stats, top_lp, top_idx;
    if (index.defined()) lp = at::empty(rows, f32);
    if (train) stats = at::empty(with(rows, rows.size(), 3), f32);
    if (top && c.layout == kLast) {  // the kernels write the list of a row together, too
      top_lp = at::empty(with(rows, rows.size(), top), f32).movedim(-1, c.dim);
      top_idx = at::empty(with(rows, rows.size(), top), f32.dtype(at::kInt)).movedim(-1, c.dim);
    } else if (top) {
      top_lp = at::empty(with(rows, c.dim, top), f32);
      top_idx = at::empty(with(rows, c.dim, top), f32.dtype(at::kInt));
    }
    const Tensor ws = workspace(x, c.nbytes);
    check(lib.log_probs_fwd(&c.desc, data(x), data(index), data<float>(lp),
                            data<float>(ent), data<float>(top_lp), data<int32_t>(top_idx), data<float>(stats), data(ws),
                            c.nbytes, stream_of(x)),
          "dw_log_probs_fwd");
    variable_list out;
    if (index.defined()) out.push_back(lp);
    out.push_back(ent);
    if (top) {
      out.push_back(top_lp);
      out.push_back(top_idx);
    }
    if (train) {
      ctx->set_materialize_grads(false);
      if (top) ctx->mark_non_differentiable({top_lp, top_idx});
      ctx->save_for_backward({logits, index_in, stats});
      keep(ctx, c);
    }
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto saved = ctx->get_saved_variables();
    const Tensor index = contiguous(saved[1]), stats = contiguous(saved[2]);
    Tensor g_lp, g_ent;
    if (index.defined()) g_lp = contiguous(g[0]);
    g_ent = contiguous(g[index.defined() ? 1 : 0]);
    variable_list out(5);
    if (!g_lp.defined() && !g_ent.defined()) return out;
    const c10::OptionalDeviceGuard guard(saved[0].device());
    const Call c = kept(ctx);
    const Tensor x = saved_in_place(saved[0], c.layout, c.dim);
    Tensor grad = at::empty_like(x);
    check(lib.log_probs_bwd(&c.desc, data(x), data(index), data<float>(stats), data<float>(g_lp), data<float>(g_ent),
                            data(grad), stream_of(x)),
          "dw_log_probs_bwd");
    out[0] = once(grad);
    return out;
  }
};

struct Distill : torch::autograd::Function<Distill> {
  static Tensor forward(AutogradContext* ctx, const Tensor& logits, const Tensor& teacher_in, const Tensor& index_in,
                        at::IntArrayRef words, at::IntArrayRef rows, bool train) {
    const Call c = call_of(words);
    const Tensor x = in_place(logits, c.layout), teacher = in_place(teacher_in, c.list_layout),
                 index = in_place(index_in, c.list_layout);
    const c10::OptionalDeviceGuard guard(x.device());
    const auto f32 = x.options().dtype(at::kFloat).memory_format(std::nullopt);
    Tensor loss = at::empty(rows, f32), stats;
    if (train) stats = at::empty(with(rows, rows.size(), 4), f32);
    const Tensor ws = workspace(x, c.nbytes);
    check(lib.distill_fwd(&c.desc, data(x), data(teacher), data(index),
                          data<float>(loss), data<float>(stats), data(ws), c.nbytes, stream_of(x)),
          "dw_distill_fwd");
    if (train) {
      ctx->set_materialize_grads(false);
      ctx->save_for_backward({logits, teacher_in, index_in, stats});
      keep(ctx, c);
    }
    return loss;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    variable_list out(6);
    if (!g[0].defined()) return out;
    const auto saved = ctx->get_saved_variables();
    const c10::OptionalDeviceGuard guard(saved[0].device());
    const Call c = kept(ctx);
    const Tensor x = saved_in_place(saved[0], c.layout, c.dim), teacher = saved_in_place(saved[1], c.list_layout, c.dim),
                 index = saved_in_place(saved[2], c.list_layout, c.dim), stats = contiguous(saved[3]), up = contiguous(g[0]);
    Tensor grad = at::empty_like(x);
    check(lib.distill_bwd(&c.desc, data(x), data(teacher), data(index), data<float>(stats), data<float>(up), data(grad),
                          stream_of(x)),
          "dw_distill_bwd");
    out[0] = once(grad);
    return out;
  }
};

// [log_prob if there is an index, entropy, and the two top lists if top > 0]
std::vector<Tensor> log_probs(const Tensor& logits, const std::optional<Tensor>& index, at::IntArrayRef call,
                              at::IntArrayRef rows) {
  const bool train = logits.requires_grad() && at::GradMode::is_enabled();
  return LogProbs::apply(logits, index, call, rows, train);
}
Tensor distill(const Tensor& logits, const Tensor& teacher, const Tensor& index, at::IntArrayRef call, at::IntArrayRef rows) {
  const bool train = logits.requires_grad() && at::GradMode::is_enabled();
  return Distill::apply(logits, teacher, index, call, rows, train);
}
}  // namespace

TORCH_LIBRARY_FRAGMENT(depthwarp, m) {
  m.def("_bind_distribution(int strerror, int lp_fwd, int lp_bwd, int ds_fwd, int ds_bwd) -> ()", &bind);
  m.def("_log_probs_eager(Tensor logits, Tensor? index, int[] call, int[] rows) -> Tensor[]", &log_probs);
  m.def("_distill_eager(Tensor logits, Tensor teacher, Tensor index, int[] call, int[] rows) -> Tensor", &distill);
}
