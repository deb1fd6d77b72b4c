// Eager-mode call path of the operators around attention (chill_attention/rotary.py, beams.py, cache.py): argument checks, outputs and
// workspace from torch's allocator, C-ABI calls of include/chill_decode.h, and the rotation's autograd node.  Part of the native module that torch_ext.cpp
// defines.  A check that fails returns None; the caller repeats the checks in Python for the message.
#include <ATen/core/dispatch/Dispatcher.h>
#include <ATen/ops/empty_like.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/utils/pybind.h>

#include <memory>
#include <optional>
#include <string>
#include <utility>
#include <vector>

#include "chill_decode.h"
#include "torch_call.h"
#include "torch_ext.h"

namespace py = pybind11;
using at::Tensor;
using namespace chill_torch;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

namespace {

struct DecodeLibrary {
  decltype(&chill_rotate) rotate;
  decltype(&chill_rotate_append) rotate_append;
  decltype(&chill_beam_select) select;
  decltype(&chill_select_workspace_bytes) select_bytes;
  decltype(&chill_pages_fork) fork;
  decltype(&chill_pages_trim_shared) trim;
  decltype(&chill_pages_compact) compact;
  decltype(&chill_share_workspace_bytes) workspace_bytes;
  decltype(&chill_cache_copy) copy;
  decltype(&chill_status_string) status_string;
  decltype(&chill_decode_last_cuda_error) cuda_error;
};

void check(const DecodeLibrary& lib, int status, const char* what) {
  if (status == CHILL_OK) return;
  std::string msg = std::string(what) + " failed: " + lib.status_string(status) + " (status " + std::to_string(status) + ")";
  if (status == CHILL_E_CUDA) msg += std::string(" ") + lib.cuda_error();
  throw_chill_error(msg);
}

// ------------------------------------------------------------------------------------------------------------ rotation
// What turns: kept by an autograd node too.
struct Turn : torch::CustomClassHolder {
  std::shared_ptr<const DecodeLibrary> lib;
  bool interleaved, inverse;
};
struct Where {
  Tensor positions, inv_freq, axes;  // axes may be undefined
};

Tensor empty_as(const Tensor& t) {
  if (t.is_non_overlapping_and_dense()) return at::detail::empty_strided_cuda(t.sizes(), t.strides(), t.scalar_type(), t.device());
  return at::empty_like(t, at::MemoryFormat::Preserve);  // the strides that the dispatcher op's fake implementation says
}

void where_args(chill_rotate_args& a, const Where& w, bool interleaved) {
  a.pairs = (int32_t)w.inv_freq.size(0);
  a.inv_freq = w.inv_freq.const_data_ptr<float>();
  a.axes = w.axes.defined() ? w.axes.const_data_ptr<int32_t>() : nullptr;
  a.positions = w.positions.const_data_ptr<int32_t>();
  const bool several = w.positions.dim() == 3;
  a.n_axes = several ? (int32_t)w.positions.size(0) : 1;
  a.position_strides[0] = several ? w.positions.stride(0) : 0;
  a.position_strides[1] = w.positions.stride(several ? 1 : 0);
  a.position_strides[2] = w.positions.stride(several ? 2 : 1);
  a.interleaved = interleaved;
}

// One or two tensors (b may be undefined).
std::pair<Tensor, Tensor> launch_rotate(const DecodeLibrary& lib, const Tensor& x, const Tensor& y, const Where& w, bool interleaved, bool inverse) {
  c10::cuda::CUDAGuard guard(x.device());
  chill_rotate_args a{};
  a.B = (int32_t)x.size(0); a.H = (int32_t)x.size(1); a.L = (int32_t)x.size(2); a.D = (int32_t)x.size(3);
  a.dtype = dtype_of(x);
  a.inverse = inverse;
  where_args(a, w, interleaved);
  Tensor x_out = empty_as(x), y_out;
  a.q = x.const_data_ptr(); a.q_out = x_out.mutable_data_ptr();
  set_strides(a.q_strides, x); set_strides(a.q_out_strides, x_out);
  if (y.defined()) {
    y_out = empty_as(y);
    a.H_kv = (int32_t)y.size(1);
    a.k = y.const_data_ptr(); a.k_out = y_out.mutable_data_ptr();
    set_strides(a.k_strides, y); set_strides(a.k_out_strides, y_out);
  }
  check(lib, lib.rotate(&a, current_stream(x)), "chill_rotate");
  return {x_out, y_out};
}

std::pair<Tensor, Tensor> rotate_any(const Tensor& x, const Tensor& y, const Where& w, c10::intrusive_ptr<Turn> turn);

// The dispatcher op (rotary.py), for gradients that are more than their memory: subclasses, several at a time, signs still to be applied.
std::pair<Tensor, Tensor> rotate_by_dispatcher(const Tensor& x, const Tensor& y, const Where& w, const Turn& turn) {
  static const auto op = c10::Dispatcher::singleton()
                             .findSchemaOrThrow("chill_attention::rotate", "")
                             .typed<std::tuple<Tensor, Tensor>(const Tensor&, const std::optional<Tensor>&, const Tensor&, const Tensor&, const std::optional<Tensor>&, bool, bool)>();
  auto optional = [](const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; };
  auto [x_out, y_out] = op.call(x, optional(y), w.positions, w.inv_freq, optional(w.axes), turn.interleaved, turn.inverse);
  return {x_out, y.defined() ? y_out : Tensor()};
}

// Linear in its input: the gradient is turned by the opposite angle, and nothing but the positions is kept.  The backward is this function again, so it can
// be differentiated in its turn.
struct RotateFn : torch::autograd::Function<RotateFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const std::optional<Tensor>& y, const Tensor& positions, const Tensor& inv_freq,
                               const std::optional<Tensor>& axes, c10::intrusive_ptr<Turn> turn) {
    const Where w{positions, inv_freq, axes.has_value() ? *axes : Tensor()};
    auto [x_out, y_out] = launch_rotate(*turn->lib, x, y.has_value() ? *y : Tensor(), w, turn->interleaved, turn->inverse);
    ctx->save_for_backward({positions, inv_freq, w.axes});
    ctx->saved_data["turn"] = c10::IValue::make_capsule(std::move(turn));
    ctx->set_materialize_grads(false);
    if (!y.has_value()) return {x_out};
    if (!x.requires_grad()) ctx->mark_non_differentiable({x_out});  // a constant turned is a constant
    if (!y->requires_grad()) ctx->mark_non_differentiable({y_out});
    return {x_out, y_out};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const auto holder = ctx->saved_data["turn"].toCapsule();
    const Turn& turn = *static_cast<const Turn*>(holder.get());
    auto back = c10::make_intrusive<Turn>();
    back->lib = turn.lib;
    back->interleaved = turn.interleaved;
    back->inverse = !turn.inverse;
    const Where w{saved[0], saved[1], saved[2]};
    const Tensor gx = grads[0], gy = grads.size() > 1 ? grads[1] : Tensor();
    Tensor dx, dy;
    if (gx.defined()) std::tie(dx, dy) = rotate_any(gx, gy, w, std::move(back));
    else if (gy.defined()) dy = rotate_any(gy, Tensor(), w, std::move(back)).first;
    return {dx, dy, Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

std::pair<Tensor, Tensor> rotate_any(const Tensor& x, const Tensor& y, const Where& w, c10::intrusive_ptr<Turn> turn) {
  if (watched({&x}, y.defined() ? std::optional<Tensor>(y) : std::nullopt)) return rotate_by_dispatcher(x, y, w, *turn);
  if (at::GradMode::is_enabled() && (x.requires_grad() || (y.defined() && y.requires_grad()))) {
    auto optional = [](const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; };
    variable_list out = RotateFn::apply(x, optional(y), w.positions, w.inv_freq, optional(w.axes), std::move(turn));
    return {out[0], out.size() > 1 ? out[1] : Tensor()};
  }
  return launch_rotate(*turn->lib, x, y, w, turn->interleaved, turn->inverse);
}

bool floats4(const Tensor& t) { return t.dim() == 4 && t.numel() > 0 && fit(t) && dtype_of(t) >= 0 && t.is_cuda(); }

// Positions, frequencies and axes that go with a tensor [batch, heads, tokens, channels].
bool where_ok(const Tensor& x, const Tensor& positions, const Tensor& inv_freq, const std::optional<Tensor>& axes) {
  const int64_t B = x.size(0), L = x.size(2), D = x.size(3);
  if (B * L > INT32_MAX / D) return false;
  if (inv_freq.scalar_type() != at::kFloat || inv_freq.dim() != 1 || !inv_freq.is_contiguous() || inv_freq.device() != x.device()) return false;
  const int64_t pairs = inv_freq.size(0);
  if (pairs < 1 || 2 * pairs > D) return false;
  if (axes.has_value() && !ints(*axes, {pairs}, x)) return false;
  if (positions.scalar_type() != at::kInt || positions.device() != x.device()) return false;
  const int64_t d = positions.dim();
  if (d == 3 && positions.size(0) > 1 && !axes.has_value()) return false;
  return (d == 2 || (d == 3 && positions.size(0) >= 1 && positions.size(0) <= INT32_MAX)) && positions.size(d - 2) == B && positions.size(d - 1) == L;
}

py::object rotate(std::shared_ptr<DecodeLibrary> lib, const Tensor& q, const std::optional<Tensor>& k, const Tensor& positions, const Tensor& inv_freq,
                  const std::optional<Tensor>& axes, bool interleaved, bool inverse) {
  if (watched({&q, &positions, &inv_freq}, k, axes) || !floats4(q) || !where_ok(q, positions, inv_freq, axes) || wants_grad({&inv_freq})) return py::none();
  if (k.has_value() && (!floats4(*k) || k->scalar_type() != q.scalar_type() || k->device() != q.device() || k->size(0) != q.size(0) ||
                        k->size(2) != q.size(2) || k->size(3) != q.size(3)))
    return py::none();
  if (c10::AutogradState::get_tls_state().get_fw_grad_mode() && (q._fw_grad(0).defined() || (k.has_value() && k->_fw_grad(0).defined()))) return py::none();
  auto turn = c10::make_intrusive<Turn>();
  turn->lib = std::move(lib);
  turn->interleaved = interleaved;
  turn->inverse = inverse;
  std::pair<Tensor, Tensor> out;
  {
    py::gil_scoped_release no_gil;
    out = rotate_any(q, k.has_value() ? *k : Tensor(), {positions, inv_freq, axes.has_value() ? *axes : Tensor()}, std::move(turn));
  }
  return py::make_tuple(out.first, k.has_value() ? py::cast(out.second) : py::none());
}

py::object rotate_append(const DecodeLibrary& lib, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& kc, const Tensor& vc, const Tensor& slots,
                         const Tensor& positions, const Tensor& inv_freq, const std::optional<Tensor>& axes, bool interleaved) {
  if (watched({&q, &k, &v, &kc, &vc, &slots, &positions, &inv_freq}, axes) || !floats4(q) || !floats4(k) || !floats4(kc) || !where_ok(q, positions, inv_freq, axes)) return py::none();
  if (kc.sizes() != vc.sizes() || vc.scalar_type() != kc.scalar_type() || vc.device() != kc.device() || k.sizes() != v.sizes()) return py::none();
  if (k.size(0) != q.size(0) || k.size(2) != q.size(2) || k.size(3) != q.size(3) || k.size(1) != kc.size(1) || k.size(3) != kc.size(3)) return py::none();
  for (const Tensor* t : {&q, &k, &v})
    if (t->scalar_type() != kc.scalar_type() || t->device() != kc.device()) return py::none();
  if (!ints(slots, {q.size(0), q.size(2)}, q) || wants_grad({&q, &k, &v, &kc, &vc, &inv_freq})) return py::none();
  c10::cuda::CUDAGuard guard(q.device());
  chill_rotate_args a{};
  a.B = (int32_t)q.size(0); a.H = (int32_t)q.size(1); a.L = (int32_t)q.size(2); a.D = (int32_t)q.size(3); a.H_kv = (int32_t)k.size(1);
  a.dtype = dtype_of(q);
  where_args(a, {positions, inv_freq, axes.has_value() ? *axes : Tensor()}, interleaved);
  Tensor out = empty_as(q);
  a.q = q.const_data_ptr(); a.q_out = out.mutable_data_ptr(); a.k = k.const_data_ptr(); a.v = v.const_data_ptr();
  a.k_cache = kc.mutable_data_ptr(); a.v_cache = vc.mutable_data_ptr();
  set_strides(a.q_strides, q); set_strides(a.q_out_strides, out); set_strides(a.k_strides, k); set_strides(a.v_strides, v);
  set_strides(a.k_cache_strides, kc); set_strides(a.v_cache_strides, vc);
  a.slots = slots.const_data_ptr<int32_t>();
  a.num_pages = (int32_t)kc.size(0); a.page_size = (int32_t)kc.size(2);
  check(lib, lib.rotate_append(&a, current_stream(q)), "chill_rotate_append");
  changed({&kc, &vc});
  return py::cast(out);
}

// ------------------------------------------------------------------------------------------------------------ selection
py::object beam_select(const DecodeLibrary& lib, const Tensor& logits, const Tensor& scores, int64_t count, const std::optional<Tensor>& finished, int64_t end_token) {
  if (watched({&logits, &scores}, finished) || logits.dim() != 2 || logits.numel() == 0 || !fit(logits) || dtype_of(logits) < 0 || !logits.is_cuda()) return py::none();
  const int64_t rows = logits.size(0), V = logits.size(1);
  if ((logits.stride(1) != 1 && V > 1) || V > (1 << 26)) return py::none();
  if (scores.dim() != 2 || scores.scalar_type() != at::kFloat || !scores.is_contiguous() || scores.device() != logits.device() || scores.numel() != rows) return py::none();
  const int64_t G = scores.size(0), K = scores.size(1);
  if (K > CHILL_SELECT_MAX || rows > 65535 || count < 1 || count > CHILL_SELECT_MAX || count > K * V) return py::none();
  if (finished.has_value() && (finished->scalar_type() != at::kBool || finished->sizes() != scores.sizes() || !finished->is_contiguous() ||
                               finished->device() != logits.device() || end_token < 0 || end_token >= V))
    return py::none();
  if (wants_grad({&logits, &scores})) return py::none();
  c10::cuda::CUDAGuard guard(logits.device());
  Tensor out = empty({G, count}, at::kFloat, logits), parents = empty({G, count}, at::kInt, logits), tokens = empty({G, count}, at::kInt, logits);
  chill_select_args a{};
  a.G = (int32_t)G; a.K = (int32_t)K; a.M = (int32_t)count; a.V = V;
  a.dtype = dtype_of(logits);
  a.logits = logits.const_data_ptr();
  a.row_stride = logits.stride(0);
  a.scores = scores.const_data_ptr<float>();
  a.finished = finished.has_value() ? reinterpret_cast<const uint8_t*>(finished->const_data_ptr<bool>()) : nullptr;
  a.end_token = end_token;
  a.out_scores = out.mutable_data_ptr<float>(); a.out_rows = parents.mutable_data_ptr<int32_t>(); a.out_tokens = tokens.mutable_data_ptr<int32_t>();
  a.workspace_bytes = lib.select_bytes(&a);
  Tensor work = empty({(int64_t)a.workspace_bytes}, at::kByte, logits);
  a.workspace = work.mutable_data_ptr();
  check(lib, lib.select(&a, current_stream(logits)), "chill_beam_select");
  return py::make_tuple(out, parents, tokens);
}

// ------------------------------------------------------------------------------------------------------------ pages
bool pages_ok(const Tensor& table, const Tensor& held, const Tensor& free, const Tensor& n_free, int64_t page) {
  if (!table_ok(table) || page < 1 || page > INT32_MAX || free.dim() != 1 || free.size(0) < 1 || !fit(free)) return false;
  return ints(held, {table.size(0)}, table) && ints(free, {free.size(0)}, table) && ints(n_free, {1}, table);
}

// The arguments that all three calls have, and a workspace of the call's own.
chill_share_args share_args(const DecodeLibrary& lib, const Tensor& table, const Tensor& held, const Tensor& free, const Tensor& n_free, int64_t page, Tensor& work) {
  chill_share_args a{};
  a.B = (int32_t)table.size(0); a.page_size = (int32_t)page; a.num_pages = (int32_t)free.size(0); a.table_width = (int32_t)table.size(1);
  a.table = table.mutable_data_ptr<int32_t>(); a.table_stride = table.stride(0);
  a.held = held.mutable_data_ptr<int32_t>(); a.free_pages = free.mutable_data_ptr<int32_t>(); a.n_free = n_free.mutable_data_ptr<int32_t>();
  a.workspace_bytes = lib.workspace_bytes(&a);
  work = empty({(int64_t)a.workspace_bytes}, at::kByte, table);
  a.workspace = work.mutable_data_ptr();
  return a;
}

struct Copies {
  Tensor source, target, rows, count;
  Copies(chill_share_args& a, int64_t n, const Tensor& like)
      : source(empty({n}, at::kInt, like)), target(empty({n}, at::kInt, like)), rows(empty({n}, at::kInt, like)), count(empty({1}, at::kInt, like)) {
    a.source = source.mutable_data_ptr<int32_t>(); a.target = target.mutable_data_ptr<int32_t>();
    a.rows = rows.mutable_data_ptr<int32_t>(); a.count = count.mutable_data_ptr<int32_t>();
  }
};

py::object pages_fork(const DecodeLibrary& lib, const Tensor& table, const Tensor& held, const Tensor& free, const Tensor& n_free, const Tensor& missing,
                const Tensor& shared, const Tensor& lens, const Tensor& parents, int64_t page) {
  if (watched({&table, &held, &free, &n_free, &missing, &shared, &lens, &parents}) || !pages_ok(table, held, free, n_free, page)) return py::none();
  const int64_t B = table.size(0);
  if (!ints(missing, {1}, table) || !ints(shared, {free.size(0)}, table) || !ints(lens, {B}, table) || !ints(parents, {B}, table)) return py::none();
  c10::cuda::CUDAGuard guard(table.device());
  Tensor work, out_lens = empty({B}, at::kInt, table);
  chill_share_args a = share_args(lib, table, held, free, n_free, page, work);
  Copies c(a, B, table);
  a.shared = shared.mutable_data_ptr<int32_t>(); a.missing = missing.mutable_data_ptr<int32_t>();
  a.lens = lens.const_data_ptr<int32_t>(); a.parents = parents.const_data_ptr<int32_t>(); a.out_lens = out_lens.mutable_data_ptr<int32_t>();
  check(lib, lib.fork(&a, current_stream(table)), "chill_pages_fork");
  changed({&table, &held, &free, &n_free, &missing, &shared});
  return py::make_tuple(out_lens, c.source, c.target, c.rows, c.count);
}

bool pages_trim(const DecodeLibrary& lib, const Tensor& table, const Tensor& held, const Tensor& free, const Tensor& n_free, const Tensor& shared, const Tensor& lens,
          int64_t page) {
  if (watched({&table, &held, &free, &n_free, &shared, &lens}) || !pages_ok(table, held, free, n_free, page)) return false;
  if (!ints(shared, {free.size(0)}, table) || !ints(lens, {table.size(0)}, table)) return false;
  c10::cuda::CUDAGuard guard(table.device());
  Tensor work;
  chill_share_args a = share_args(lib, table, held, free, n_free, page, work);
  a.shared = shared.mutable_data_ptr<int32_t>(); a.lens = lens.const_data_ptr<int32_t>();
  check(lib, lib.trim(&a, current_stream(table)), "chill_pages_trim_shared");
  changed({&table, &held, &free, &n_free, &shared});
  return true;
}

py::object pages_compact(const DecodeLibrary& lib, const Tensor& table, const Tensor& held, const Tensor& free, const Tensor& n_free, const std::optional<Tensor>& shared,
                   int64_t page) {
  if (watched({&table, &held, &free, &n_free}, shared) || !pages_ok(table, held, free, n_free, page)) return py::none();
  if (shared.has_value() && !ints(*shared, {free.size(0)}, table)) return py::none();
  c10::cuda::CUDAGuard guard(table.device());
  Tensor work;
  chill_share_args a = share_args(lib, table, held, free, n_free, page, work);
  Copies c(a, std::max<int64_t>(free.size(0) / 2, 1), table);
  a.shared = shared.has_value() ? shared->mutable_data_ptr<int32_t>() : nullptr;
  check(lib, lib.compact(&a, current_stream(table)), "chill_pages_compact");
  changed({&table, &free, &n_free});
  if (shared.has_value()) changed({&*shared});
  return py::make_tuple(c.source, c.target, c.rows, c.count);
}

bool cache_copy(const DecodeLibrary& lib, const Tensor& kc, const Tensor& vc, const Tensor& source, const Tensor& target, const Tensor& rows, const Tensor& count) {
  if (watched({&kc, &vc, &source, &target, &rows, &count}) || (kc.dim() != 4 && kc.dim() != 5) || !fit(kc) || kc.numel() == 0 || kc.sizes() != vc.sizes() ||
      dtype_of(kc) < 0 || vc.scalar_type() != kc.scalar_type() || !kc.is_cuda() || vc.device() != kc.device())
    return false;
  if (source.dim() != 1 || source.size(0) < 1 || !fit(source) || !ints(source, {source.size(0)}, kc) || !ints(target, {source.size(0)}, kc) ||
      !ints(rows, {source.size(0)}, kc) || !ints(count, {1}, kc) || wants_grad({&kc, &vc}))
    return false;
  c10::cuda::CUDAGuard guard(kc.device());
  chill_copy_args a{};
  const int64_t first = kc.dim() - 4;
  a.layers = first ? (int32_t)kc.size(0) : 1;
  a.num_pages = (int32_t)kc.size(first); a.H_kv = (int32_t)kc.size(first + 1); a.page_size = (int32_t)kc.size(first + 2); a.D = (int32_t)kc.size(first + 3);
  a.dtype = dtype_of(kc);
  a.k_cache = kc.mutable_data_ptr(); a.v_cache = vc.mutable_data_ptr();
  set_strides(a.k_cache_strides + 1 - first, kc); set_strides(a.v_cache_strides + 1 - first, vc);
  a.source = source.const_data_ptr<int32_t>(); a.target = target.const_data_ptr<int32_t>();
  a.rows = rows.const_data_ptr<int32_t>(); a.count = count.const_data_ptr<int32_t>();
  a.orders = (int32_t)source.size(0);
  check(lib, lib.copy(&a, current_stream(kc)), "chill_cache_copy");
  changed({&kc, &vc});
  return true;
}

}  // namespace

void bind_decode(py::module_& m) {
  py::class_<DecodeLibrary, std::shared_ptr<DecodeLibrary>>(m, "DecodeLibrary").def(py::init([](const std::vector<uint64_t>& fn) {
    if (fn.size() != 11) throw py::value_error("eleven entry points");
    return std::make_shared<DecodeLibrary>(DecodeLibrary{pointer<decltype(&chill_rotate)>(fn[0]), pointer<decltype(&chill_rotate_append)>(fn[1]),
                           pointer<decltype(&chill_beam_select)>(fn[2]), pointer<decltype(&chill_select_workspace_bytes)>(fn[3]),
                           pointer<decltype(&chill_pages_fork)>(fn[4]), pointer<decltype(&chill_pages_trim_shared)>(fn[5]),
                           pointer<decltype(&chill_pages_compact)>(fn[6]), pointer<decltype(&chill_share_workspace_bytes)>(fn[7]),
                           pointer<decltype(&chill_cache_copy)>(fn[8]), pointer<decltype(&chill_status_string)>(fn[9]),
                           pointer<decltype(&chill_decode_last_cuda_error)>(fn[10])});
  }));
  m.def("rotate", &rotate);
  m.def("rotate_append", &rotate_append);
  m.def("beam_select", &beam_select);
  m.def("pages_fork", &pages_fork);
  m.def("pages_trim_shared", &pages_trim);
  m.def("pages_compact", &pages_compact);
  m.def("cache_copy", &cache_copy);
}
