// Eager-mode call path of the paged-cache operators (chill_attention/cache.py): argument checks, outputs and workspace from torch's
// allocator, C-ABI calls.  Part of the native module that torch_ext.cpp defines.  A check that fails returns None; the caller
// repeats the checks in Python for the message.
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/utils/pybind.h>

#include <memory>
#include <optional>
#include <string>
#include <vector>

#include "chill_cache.h"
#include "torch_call.h"
#include "torch_ext.h"

namespace py = pybind11;
using at::Tensor;
using namespace chill_torch;

namespace {

struct CacheLibrary {
  decltype(&chill_cached_fwd) fwd;
  decltype(&chill_cached_workspace_bytes) workspace_bytes;
  decltype(&chill_pages_reserve_stored) reserve;
  decltype(&chill_pages_trim) trim;
  decltype(&chill_cache_append) append;
  decltype(&chill_cache_commit) commit;
  decltype(&chill_status_string) status_string;
  decltype(&chill_cache_last_cuda_error) cuda_error;
};

void check(const CacheLibrary& lib, int status, const char* what) {
  if (status == CHILL_OK) return;
  std::string msg = std::string(what) + " failed: " + lib.status_string(status) + " (status " + std::to_string(status) + ")";
  if (status == CHILL_E_CUDA) msg += std::string(" ") + lib.cuda_error();
  throw_chill_error(msg);
}

bool pools_ok(const Tensor& k, const Tensor& v) {
  return k.dim() == 4 && fit(k) && k.sizes() == v.sizes() && k.numel() > 0 && k.scalar_type() == v.scalar_type() && dtype_of(k) >= 0 && k.is_cuda() && v.device() == k.device();
}

py::object reserve(const CacheLibrary& lib, const Tensor& table, const Tensor& held, const Tensor& free, const Tensor& n_free, const Tensor& missing,
                   const Tensor& lens, const Tensor& new_lens, int64_t N, int64_t page, const std::optional<Tensor>& parents, const std::optional<Tensor>& stored) {
  if (watched({&table, &held, &free, &n_free, &missing, &lens, &new_lens}, parents, stored) || !table_ok(table) || N < 1 || N > INT32_MAX || page < 1 || page > INT32_MAX) return py::none();
  const int64_t B = table.size(0);
  if (!ints(held, {B}, table) || free.dim() != 1 || free.size(0) < 1 || !fit(free) || !ints(free, {free.size(0)}, table) || !ints(n_free, {1}, table) ||
      !ints(missing, {1}, table) || !ints(lens, {B}, table) || !ints(new_lens, {B}, table) || (parents.has_value() && !ints(*parents, {B, N}, table)) || (stored.has_value() && !ints(*stored, {B}, table)))
    return py::none();
  c10::cuda::CUDAGuard guard(table.device());
  Tensor slots = empty({B, N}, at::kInt, table), positions = empty({B, N}, at::kInt, table), ancestors;
  if (parents.has_value()) ancestors = empty({B, N, (N + 31) / 32}, at::kInt, table);
  chill_pages_args a{};
  a.B = (int32_t)B; a.N = (int32_t)N; a.page_size = (int32_t)page; a.num_pages = (int32_t)free.size(0); a.table_width = (int32_t)table.size(1);
  a.table = table.mutable_data_ptr<int32_t>(); a.table_stride = table.stride(0);
  a.held = held.mutable_data_ptr<int32_t>(); a.free_pages = free.mutable_data_ptr<int32_t>(); a.n_free = n_free.mutable_data_ptr<int32_t>();
  a.missing = missing.mutable_data_ptr<int32_t>();
  a.lens = lens.const_data_ptr<int32_t>(); a.new_lens = new_lens.const_data_ptr<int32_t>(); a.parents = optional_ints(parents);
  a.slots = slots.mutable_data_ptr<int32_t>(); a.positions = positions.mutable_data_ptr<int32_t>();
  a.ancestors = parents.has_value() ? ancestors.mutable_data_ptr<int32_t>() : nullptr;
  check(lib, lib.reserve(&a, stored.has_value() ? stored->mutable_data_ptr<int32_t>() : nullptr, current_stream(table)), "chill_pages_reserve");
  changed({&table, &held, &free, &n_free, &missing});
  if (stored.has_value()) changed({&*stored});
  return py::make_tuple(slots, positions, parents.has_value() ? py::cast(ancestors) : py::none());
}

bool trim(const CacheLibrary& lib, const Tensor& table, const Tensor& held, const Tensor& free, const Tensor& n_free, const Tensor& lens, int64_t page) {
  if (watched({&table, &held, &free, &n_free, &lens}) || !table_ok(table) || page < 1 || page > INT32_MAX) return false;
  const int64_t B = table.size(0);
  if (!ints(held, {B}, table) || free.dim() != 1 || free.size(0) < 1 || !fit(free) || !ints(free, {free.size(0)}, table) || !ints(n_free, {1}, table) || !ints(lens, {B}, table))
    return false;
  c10::cuda::CUDAGuard guard(table.device());
  chill_pages_args a{};
  a.B = (int32_t)B; a.page_size = (int32_t)page; a.num_pages = (int32_t)free.size(0); a.table_width = (int32_t)table.size(1);
  a.table = table.mutable_data_ptr<int32_t>(); a.table_stride = table.stride(0);
  a.held = held.mutable_data_ptr<int32_t>(); a.free_pages = free.mutable_data_ptr<int32_t>(); a.n_free = n_free.mutable_data_ptr<int32_t>();
  a.lens = lens.const_data_ptr<int32_t>();
  check(lib, lib.trim(&a, current_stream(table)), "chill_pages_trim");
  changed({&table, &held, &free, &n_free});
  return true;
}

// What both row operators take of the caches.
chill_cache_rows_args rows_args(const Tensor& kc, const Tensor& vc) {
  chill_cache_rows_args a{};
  a.num_pages = (int32_t)kc.size(0); a.H_kv = (int32_t)kc.size(1); a.page_size = (int32_t)kc.size(2); a.D = (int32_t)kc.size(3);
  a.dtype = dtype_of(kc);
  a.k_cache = kc.mutable_data_ptr(); a.v_cache = vc.mutable_data_ptr();
  set_strides(a.k_cache_strides, kc); set_strides(a.v_cache_strides, vc);
  return a;
}

bool append(const CacheLibrary& lib, const Tensor& kc, const Tensor& vc, const Tensor& k, const Tensor& v, const Tensor& slots) {
  if (watched({&kc, &vc, &k, &v, &slots}) || !pools_ok(kc, vc) || k.dim() != 4 || k.numel() == 0 || !fit(k) || k.sizes() != v.sizes() || k.size(1) != kc.size(1) || k.size(3) != kc.size(3)) return false;
  if (k.scalar_type() != kc.scalar_type() || v.scalar_type() != kc.scalar_type() || k.device() != kc.device() || v.device() != kc.device()) return false;
  if (!ints(slots, {k.size(0), k.size(2)}, kc) || wants_grad({&kc, &vc, &k, &v})) return false;
  c10::cuda::CUDAGuard guard(kc.device());
  chill_cache_rows_args a = rows_args(kc, vc);
  a.B = (int32_t)k.size(0); a.N = (int32_t)k.size(2);
  a.k = k.const_data_ptr(); a.v = v.const_data_ptr();
  set_strides(a.k_strides, k); set_strides(a.v_strides, v);
  a.slots = slots.const_data_ptr<int32_t>();
  check(lib, lib.append(&a, current_stream(kc)), "chill_cache_append");
  changed({&kc, &vc});
  return true;
}

py::object commit(const CacheLibrary& lib, const Tensor& kc, const Tensor& vc, const Tensor& table, const Tensor& lens, const Tensor& new_lens,
                  int64_t N, const Tensor& path, const Tensor& accepted) {
  if (watched({&kc, &vc, &table, &lens, &new_lens, &path, &accepted}) || !pools_ok(kc, vc) || !table_ok(table) || table.device() != kc.device() || path.dim() != 2 || path.size(1) < 1 || !fit(path) || N < 1 || N > INT32_MAX) return py::none();
  const int64_t B = table.size(0);
  if (!ints(lens, {B}, kc) || !ints(new_lens, {B}, kc) || !ints(path, {B, path.size(1)}, kc) || !ints(accepted, {B}, kc) || wants_grad({&kc, &vc})) return py::none();
  c10::cuda::CUDAGuard guard(kc.device());
  Tensor out = empty({B}, at::kInt, table);
  chill_cache_rows_args a = rows_args(kc, vc);
  a.B = (int32_t)B; a.N = (int32_t)N; a.A = (int32_t)path.size(1); a.table_width = (int32_t)table.size(1);
  a.table = table.const_data_ptr<int32_t>(); a.table_stride = table.stride(0);
  a.lens = lens.const_data_ptr<int32_t>(); a.new_lens = new_lens.const_data_ptr<int32_t>();
  a.path = path.const_data_ptr<int32_t>(); a.accepted = accepted.const_data_ptr<int32_t>(); a.out_lens = out.mutable_data_ptr<int32_t>();
  check(lib, lib.commit(&a, current_stream(kc)), "chill_cache_commit");
  changed({&kc, &vc});
  return py::cast(out);
}

// O, (O, LSE) when return_lse.  The workspace goes back to the allocator when the call returns: the allocator hands it out again for
// work behind this call on the same stream only (and a captured graph keeps it in its own pool).
py::object attention(const CacheLibrary& lib, int32_t functor_id, const Tensor& q, const Tensor& kc, const Tensor& vc, const Tensor& table,
                     const Tensor& lens, const Tensor& new_lens, const Tensor& positions, const std::optional<Tensor>& ancestors,
                     const py::tuple& mask_args, double sm_scale, bool return_lse, uint32_t flags) {
  if (watched({&q, &kc, &vc, &table, &lens, &new_lens, &positions}, ancestors) || !pools_ok(kc, vc) || !table_ok(table) || table.device() != kc.device() || q.dim() != 4 || q.numel() == 0 || !fit(q)) return py::none();
  const int64_t B = q.size(0), H = q.size(1), N = q.size(2), D = q.size(3);
  if (table.size(0) != B || kc.size(3) != D || H % kc.size(1) != 0 || q.scalar_type() != kc.scalar_type() || q.device() != kc.device()) return py::none();
  if (D != 16 && D != 32 && D != 64 && D != 128 && D != 256) return py::none();
  if (!ints(lens, {B}, q) || !ints(new_lens, {B}, q) || !ints(positions, {B, N}, q)) return py::none();
  if (ancestors.has_value() && !ints(*ancestors, {B, N, (N + 31) / 32}, q)) return py::none();
  if (wants_grad({&q, &kc, &vc})) return py::none();
  c10::cuda::CUDAGuard guard(q.device());
  chill_cached_args a{};
  a.mask.id = functor_id;
  set_mask_constants(a.mask, mask_args);
  a.B = (int32_t)B; a.H = (int32_t)H; a.N = (int32_t)N; a.D = (int32_t)D;
  a.num_pages = (int32_t)kc.size(0); a.H_kv = (int32_t)kc.size(1); a.page_size = (int32_t)kc.size(2); a.table_width = (int32_t)table.size(1);
  a.dtype = dtype_of(q);
  a.sm_scale = (float)sm_scale;
  a.flags = flags;
  Tensor o = empty(q.sizes(), q.scalar_type(), q), lse;
  a.q = q.const_data_ptr(); a.k_cache = kc.const_data_ptr(); a.v_cache = vc.const_data_ptr(); a.o = o.mutable_data_ptr();
  set_strides(a.q_strides, q); set_strides(a.k_cache_strides, kc); set_strides(a.v_cache_strides, vc); set_strides(a.o_strides, o);
  if (return_lse) {
    lse = empty(q.sizes().slice(0, 3), at::kFloat, q);
    a.lse = lse.mutable_data_ptr<float>();
    set_strides(a.lse_strides, lse);
  }
  a.table = table.const_data_ptr<int32_t>(); a.table_stride = table.stride(0);
  a.lens = lens.const_data_ptr<int32_t>(); a.new_lens = new_lens.const_data_ptr<int32_t>();
  a.positions = positions.const_data_ptr<int32_t>(); a.ancestors = optional_ints(ancestors);
  const size_t bytes = lib.workspace_bytes(&a);
  Tensor work = empty({(int64_t)bytes}, at::kByte, q);
  a.workspace = work.mutable_data_ptr();
  a.workspace_bytes = bytes;
  check(lib, lib.fwd(&a, current_stream(q)), "chill_cached_fwd");
  if (!return_lse) return py::cast(o);
  return py::make_tuple(o, lse);
}

}  // namespace

void bind_cache(py::module_& m) {
  py::class_<CacheLibrary, std::shared_ptr<CacheLibrary>>(m, "CacheLibrary").def(py::init([](const std::vector<uint64_t>& fn) {
    if (fn.size() != 8) throw py::value_error("eight entry points");
    return std::make_shared<CacheLibrary>(CacheLibrary{pointer<decltype(&chill_cached_fwd)>(fn[0]), pointer<decltype(&chill_cached_workspace_bytes)>(fn[1]),
                          pointer<decltype(&chill_pages_reserve_stored)>(fn[2]), pointer<decltype(&chill_pages_trim)>(fn[3]),
                          pointer<decltype(&chill_cache_append)>(fn[4]), pointer<decltype(&chill_cache_commit)>(fn[5]),
                          pointer<decltype(&chill_status_string)>(fn[6]), pointer<decltype(&chill_cache_last_cuda_error)>(fn[7])});
  }));
  m.def("pages_reserve", &reserve);
  m.def("pages_trim", &trim);
  m.def("cache_append", &append);
  m.def("cache_commit", &commit);
  m.def("cached_attention", &attention);
}
