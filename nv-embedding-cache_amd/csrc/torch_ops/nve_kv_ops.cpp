// nve_kv_ops.cpp -- the nve_ops torch library's operators of the paged key-value
// cache (HIP tensors), calling libnve_amd.so's C ABI (nve_amd_kv_*) directly:
//
//   kv_append, kv_append_norm, kv_attend, kv_attend_lse, kv_evict   (schemas below)
//
// Shapes, types and devices are checked here, the rest by the C ABI; work runs
// on the current stream, workspaces come from torch's allocator.  The operators
// serve: none has a gradient, and inputs that ask for one are refused, the cache
// and the rotary table among them.
#include <ATen/DeviceGuard.h>
#include <ATen/core/Tensor.h>
#include <ATen/core/grad_mode.h>
#include <ATen/ops/empty.h>
#include <c10/hip/HIPStream.h>
#include <torch/library.h>

#include <cstdint>
#include <optional>
#include <string>
#include <tuple>
#include <vector>

#include "nve_amd_ext.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

void check_status(nve_status_t st) {
  if (st == NVE_SUCCESS) return;
  const char* m = nullptr;
  nve_get_last_error(&m);
  const std::string what = m ? m : "no message";
  TORCH_CHECK_VALUE(st != NVE_ERROR_INVALID_ARGUMENT, "nve_ops: invalid argument: ", what);
  TORCH_CHECK(false, "nve_ops: status ", (int)st, ": ", what);
}

nve_data_type_t dtype_of(const Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case at::kFloat: return NVE_DTYPE_FLOAT32;
    case at::kHalf: return NVE_DTYPE_FLOAT16;
    case at::kBFloat16: return NVE_DTYPE_BFLOAT16;
    case at::kFloat8_e4m3fn: return NVE_DTYPE_E4M3;
    case at::kFloat4_e2m1fn_x2: return NVE_DTYPE_X_MXFP4;
    default: break;
  }
  TORCH_CHECK_TYPE(false, "nve_ops: ", name, " cannot be ", t.scalar_type());
  return NVE_DTYPE_UNKNOWN;
}

void check_type(const Tensor& t, at::ScalarType want, const char* name) {
  TORCH_CHECK_TYPE(t.scalar_type() == want, "nve_ops: ", name, " must be ", want, ", got ", t.scalar_type());
}

void check_device(const Tensor& t, const Tensor& like, const char* name) {
  TORCH_CHECK_VALUE(t.device() == like.device(), "nve_ops: ", name, " is on ", t.device(), ", the pages on ",
                    like.device());
}

void check_dense(const Tensor& t, const char* name) {
  TORCH_CHECK_VALUE(t.is_contiguous(), "nve_ops: ", name, " must be contiguous");
}

void check_grad(const Tensor& t, const char* name) {
  TORCH_CHECK(!(t.requires_grad() && at::GradMode::is_enabled()), "nve_ops: ", name,
              " asks for a gradient, and the key-value cache's operators have none (use torch.no_grad())");
}

// Values of a head's row: 4-bit pages hold two in an element.
int64_t dim_of(const Tensor& pages) {
  return pages.size(3) * (pages.scalar_type() == at::kFloat4_e2m1fn_x2 ? 2 : 1);
}

// [rows, heads, dim] with a contiguous last dimension, any strides of the others.
void check_rows(const Tensor& t, const Tensor& pages, const char* name) {
  check_device(t, pages, name);
  TORCH_CHECK_VALUE(t.dim() == 3 && t.size(2) == dim_of(pages), "nve_ops: ", name, " must be [rows, heads, ",
                    dim_of(pages), "], got ", t.sizes());
  TORCH_CHECK_VALUE(t.stride(2) == 1 || t.numel() == 0, "nve_ops: the last dimension of ", name,
                    " must be contiguous");
  check_grad(t, name);
}

const void* optional_row(const OptTensor& t, const Tensor& pages, at::ScalarType type, int64_t n, const char* name) {
  if (!t.has_value() || !t->defined()) return nullptr;
  check_device(*t, pages, name);
  check_type(*t, type, name);
  check_dense(*t, name);
  TORCH_CHECK_VALUE(t->dim() == 1 && t->size(0) == n, "nve_ops: ", name, " must be [", n, "], got ", t->sizes());
  return t->data_ptr();
}

// A [pages, heads, page] companion of the pages.
template <typename T>
T* slot_values(const OptTensor& t, const Tensor& pages, at::ScalarType type, const char* name) {
  if (!t.has_value() || !t->defined()) return nullptr;
  check_device(*t, pages, name);
  check_type(*t, type, name);
  check_dense(*t, name);
  check_grad(*t, name);
  TORCH_CHECK_VALUE(t->sizes() == pages.sizes().slice(0, 3), "nve_ops: ", name, " must be ",
                    pages.sizes().slice(0, 3), ", got ", t->sizes());
  return static_cast<T*>(t->data_ptr());
}

// The scales of e4m3 pages (one float32 a row) or of 4-bit pages (one e8m0 for every 32 values).
float* scales_of(const OptTensor& t, const Tensor& pages, const char* name) {
  if (pages.scalar_type() != at::kFloat4_e2m1fn_x2) return slot_values<float>(t, pages, at::kFloat, name);
  if (!t.has_value() || !t->defined()) return nullptr;
  check_device(*t, pages, name);
  check_type(*t, at::kFloat8_e8m0fnu, name);
  check_dense(*t, name);
  check_grad(*t, name);
  TORCH_CHECK_VALUE(t->dim() == 4 && t->sizes().slice(0, 3) == pages.sizes().slice(0, 3) &&
                        t->size(3) * 32 == dim_of(pages),
                    "nve_ops: ", name, " must be ", pages.sizes().slice(0, 3), " rows of ", dim_of(pages) / 32, ", got ",
                    t->sizes());
  return static_cast<float*>(t->data_ptr());
}

nve_amd_kv_pages_t pages_of(const Tensor& k, const Tensor& v, const OptTensor& k_scale, const OptTensor& v_scale,
                            const OptTensor& weights, const OptTensor& index) {
  TORCH_CHECK_VALUE(k.dim() == 4, "nve_ops: the pages must be [pages, heads, page, dim], got ", k.sizes());
  TORCH_CHECK_VALUE(v.sizes() == k.sizes(), "nve_ops: the k pages are ", k.sizes(), ", the v pages ", v.sizes());
  TORCH_CHECK_TYPE(v.scalar_type() == k.scalar_type(), "nve_ops: the k pages are ", k.scalar_type(),
                   ", the v pages ", v.scalar_type());
  TORCH_CHECK_VALUE(k.size(1) <= INT32_MAX && k.size(2) <= INT32_MAX && dim_of(k) <= INT32_MAX,
                    "nve_ops: pages too large");
  check_device(v, k, "v_pages");
  check_dense(k, "k_pages");
  check_dense(v, "v_pages");
  check_grad(k, "k_pages");
  check_grad(v, "v_pages");
  nve_amd_kv_pages_t p{};
  p.k = k.data_ptr();
  p.v = v.data_ptr();
  p.k_scale = scales_of(k_scale, k, "k_scale");
  p.v_scale = scales_of(v_scale, k, "v_scale");
  p.weights = slot_values<float>(weights, k, at::kFloat, "weights");
  p.index = slot_values<int32_t>(index, k, at::kInt, "index_pages");
  p.num_pages = k.size(0);
  p.num_heads = (int32_t)k.size(1);
  p.page_size = (int32_t)k.size(2);
  p.head_dim = (int32_t)dim_of(k);
  p.dtype = dtype_of(k, "k_pages");
  return p;
}

void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

Tensor bytes(uint64_t n, const Tensor& like) {
  return at::empty({(int64_t)n}, like.options().dtype(at::kByte));
}

// The weight of a norm: [dim] of the rows' type.
const void* norm_weight(const OptTensor& t, const Tensor& k, const Tensor& pages, const char* name) {
  if (!t.has_value() || !t->defined()) return nullptr;
  check_grad(*t, name);
  return optional_row(t, pages, k.scalar_type(), dim_of(pages), name);
}

Tensor append(const Tensor& k, const Tensor& v, const Tensor& k_pages, const Tensor& v_pages, const Tensor& slots,
              const OptTensor& q, const OptTensor& positions, const OptTensor& cos_sin,
              const std::optional<std::vector<int64_t>>& sections, bool interleaved, const OptTensor& index,
              const OptTensor& k_scale, const OptTensor& v_scale, const OptTensor& weights,
              const OptTensor& index_pages, const OptTensor& q_norm, const OptTensor& k_norm,
              std::optional<double> eps) {
  const at::DeviceGuard guard(k_pages.device());
  const nve_amd_kv_pages_t pages = pages_of(k_pages, v_pages, k_scale, v_scale, weights, index_pages);
  check_rows(k, k_pages, "k");
  check_rows(v, k_pages, "v");
  TORCH_CHECK_VALUE(k.sizes() == v.sizes() && k.size(1) == k_pages.size(1), "nve_ops: k and v must be [tokens, ",
                    k_pages.size(1), ", ", dim_of(k_pages), "], got ", k.sizes(), " and ", v.sizes());
  TORCH_CHECK_TYPE(k.scalar_type() == v.scalar_type(), "nve_ops: k is ", k.scalar_type(), ", v ", v.scalar_type());
  const int64_t n = k.size(0);
  nve_amd_kv_append_t c{};
  c.num_tokens = n;
  c.slots = static_cast<const int64_t*>(optional_row(slots, k_pages, at::kLong, n, "slots"));
  c.dtype = dtype_of(k, "k");
  c.k = k.data_ptr();
  c.k_token_stride = k.stride(0);
  c.k_head_stride = k.stride(1);
  c.v = v.data_ptr();
  c.v_token_stride = v.stride(0);
  c.v_head_stride = v.stride(1);
  c.index = static_cast<const int32_t*>(optional_row(index, k_pages, at::kInt, n, "index"));
  Tensor q_out;
  if (q.has_value() && q->defined()) {
    check_rows(*q, k_pages, "q");
    TORCH_CHECK_VALUE(q->size(0) == n, "nve_ops: q has ", q->size(0), " tokens, k ", n);
    TORCH_CHECK_TYPE(q->scalar_type() == k.scalar_type(), "nve_ops: q is ", q->scalar_type(), ", k ",
                     k.scalar_type());
    q_out = at::empty(q->sizes(), k.options());
    c.q = q->data_ptr();
    c.q_token_stride = q->stride(0);
    c.q_head_stride = q->stride(1);
    c.q_out = q_out.data_ptr();
    c.q_out_token_stride = q_out.stride(0);
    c.q_out_head_stride = q_out.stride(1);
    c.num_q_heads = (int32_t)q->size(1);
  } else {
    q_out = at::empty({0}, k.options());
  }
  TORCH_CHECK_VALUE(positions.has_value() || !cos_sin.has_value(), "nve_ops: cos_sin needs positions");
  if (positions.has_value() && positions->defined()) {
    const Tensor& p = *positions;
    check_device(p, k_pages, "positions");
    check_type(p, at::kInt, "positions");
    TORCH_CHECK_VALUE((p.dim() == 1 || p.dim() == 2) && p.size(-1) == n && (p.stride(-1) == 1 || n <= 1),
                      "nve_ops: positions must be [", n, "] or [axes, ", n, "] with a contiguous last dimension, got ",
                      p.sizes());
    c.positions = static_cast<const int32_t*>(p.data_ptr());
    c.num_axes = p.dim() == 2 ? (int32_t)p.size(0) : 1;
    c.axis_stride = p.dim() == 2 ? p.stride(0) : 0;
    TORCH_CHECK_VALUE(c.num_axes >= 1 && c.num_axes <= 4, "nve_ops: positions have ", c.num_axes,
                      " axes: 1 to 4 are supported");
    if (cos_sin.has_value() && cos_sin->defined()) {
      const Tensor& t = *cos_sin;
      check_device(t, k_pages, "cos_sin");
      check_type(t, at::kFloat, "cos_sin");
      check_dense(t, "cos_sin");
      check_grad(t, "cos_sin");
      TORCH_CHECK_VALUE(t.dim() == 2 && t.size(1) <= dim_of(k_pages), "nve_ops: cos_sin must be [positions, rot_dim <= ",
                        dim_of(k_pages), "], got ", t.sizes());
      c.cos_sin = static_cast<const float*>(t.data_ptr());
      c.max_position = t.size(0);
      c.rot_dim = (int32_t)t.size(1);
      if (sections.has_value()) {
        TORCH_CHECK_VALUE((int64_t)sections->size() == c.num_axes, "nve_ops: ", sections->size(), " sections for ",
                          c.num_axes, " axes of positions");
        for (size_t i = 0; i < sections->size(); ++i) {
          TORCH_CHECK_VALUE((*sections)[i] >= 0 && (*sections)[i] <= c.rot_dim, "nve_ops: invalid section ",
                            (*sections)[i]);
          c.sections[i] = (int32_t)(*sections)[i];
        }
      } else {
        TORCH_CHECK_VALUE(c.num_axes == 1, "nve_ops: positions of ", c.num_axes, " axes need sections");
        c.sections[0] = c.rot_dim / 2;
      }
    }
  }
  c.interleaved = interleaved;
  if (eps.has_value()) {
    nve_amd_kv_norm_t norm{};
    norm.q_weight = norm_weight(q_norm, k, k_pages, "q_norm");
    norm.k_weight = norm_weight(k_norm, k, k_pages, "k_norm");
    TORCH_CHECK_VALUE(!norm.q_weight || (q.has_value() && q->defined()), "nve_ops: q_norm needs q");
    norm.eps = *eps;
    check_status(nve_amd_kv_append_norm(&pages, &c, &norm, stream_of(k_pages)));
  } else {
    check_status(nve_amd_kv_append(&pages, &c, stream_of(k_pages)));
  }
  return q_out;
}

Tensor kv_append(const Tensor& k, const Tensor& v, const Tensor& k_pages, const Tensor& v_pages, const Tensor& slots,
                 const OptTensor& q, const OptTensor& positions, const OptTensor& cos_sin,
                 const std::optional<std::vector<int64_t>>& sections, bool interleaved, const OptTensor& index,
                 const OptTensor& k_scale, const OptTensor& v_scale, const OptTensor& weights,
                 const OptTensor& index_pages) {
  return append(k, v, k_pages, v_pages, slots, q, positions, cos_sin, sections, interleaved, index, k_scale, v_scale,
                weights, index_pages, std::nullopt, std::nullopt, std::nullopt);
}

Tensor kv_append_norm(const Tensor& k, const Tensor& v, const Tensor& k_pages, const Tensor& v_pages,
                      const Tensor& slots, const OptTensor& q, const OptTensor& positions, const OptTensor& cos_sin,
                      const std::optional<std::vector<int64_t>>& sections, bool interleaved, const OptTensor& index,
                      const OptTensor& k_scale, const OptTensor& v_scale, const OptTensor& weights,
                      const OptTensor& index_pages, const OptTensor& q_norm, const OptTensor& k_norm, double eps) {
  return append(k, v, k_pages, v_pages, slots, q, positions, cos_sin, sections, interleaved, index, k_scale, v_scale,
                weights, index_pages, q_norm, k_norm, eps);
}

std::tuple<Tensor, Tensor> attend(const Tensor& q, const Tensor& k_pages, const Tensor& v_pages,
                                  const Tensor& block_tables, const Tensor& lengths, double scale,
                                  const OptTensor& k_scale, const OptTensor& v_scale, const OptTensor& weights,
                                  int64_t max_length, bool want_lse) {
  const at::DeviceGuard guard(k_pages.device());
  const nve_amd_kv_pages_t pages = pages_of(k_pages, v_pages, k_scale, v_scale, weights, std::nullopt);
  check_rows(q, k_pages, "q");
  const int64_t n = q.size(0);
  check_device(block_tables, k_pages, "block_tables");
  check_type(block_tables, at::kInt, "block_tables");
  TORCH_CHECK_VALUE(block_tables.dim() == 2 && block_tables.size(0) == n &&
                        (block_tables.stride(1) == 1 || block_tables.size(1) <= 1 || n == 0),
                    "nve_ops: block_tables must be [", n, ", pages] with a contiguous last dimension, got ",
                    block_tables.sizes());
  TORCH_CHECK_VALUE(q.size(1) <= INT32_MAX, "nve_ops: too many query heads");
  Tensor out = at::empty(q.sizes(), q.options());
  Tensor lse;
  nve_amd_kv_attend_t c{};
  c.num_seqs = n;
  c.num_q_heads = (int32_t)q.size(1);
  c.dtype = dtype_of(q, "q");
  c.q = q.data_ptr();
  c.q_seq_stride = q.stride(0);
  c.q_head_stride = q.stride(1);
  c.out = out.data_ptr();
  c.out_seq_stride = out.stride(0);
  c.out_head_stride = out.stride(1);
  if (want_lse) {
    lse = at::empty({n, q.size(1)}, q.options().dtype(at::kFloat));
    c.lse = static_cast<float*>(lse.data_ptr());
  }
  c.block_tables = static_cast<const int32_t*>(block_tables.data_ptr());
  c.table_stride = block_tables.stride(0);
  c.max_pages = block_tables.size(1);
  c.lengths = static_cast<const int32_t*>(optional_row(lengths, k_pages, at::kInt, n, "lengths"));
  c.max_length = max_length;
  c.scale = (float)scale;
  c.accumulate = pages.weights != nullptr;
  uint64_t need = 0;
  check_status(nve_amd_kv_attend_workspace_size(&pages, &c, &need));
  Tensor ws;
  if (need > 0) ws = bytes(need, k_pages);
  check_status(nve_amd_kv_attend(&pages, &c, need > 0 ? ws.data_ptr() : nullptr, need, stream_of(k_pages)));
  return {out, lse};
}

Tensor kv_attend(const Tensor& q, const Tensor& k_pages, const Tensor& v_pages, const Tensor& block_tables,
                 const Tensor& lengths, double scale, const OptTensor& k_scale, const OptTensor& v_scale,
                 const OptTensor& weights, int64_t max_length) {
  return std::get<0>(
      attend(q, k_pages, v_pages, block_tables, lengths, scale, k_scale, v_scale, weights, max_length, false));
}

std::tuple<Tensor, Tensor> kv_attend_lse(const Tensor& q, const Tensor& k_pages, const Tensor& v_pages,
                                         const Tensor& block_tables, const Tensor& lengths, double scale,
                                         const OptTensor& k_scale, const OptTensor& v_scale, const OptTensor& weights,
                                         int64_t max_length) {
  return attend(q, k_pages, v_pages, block_tables, lengths, scale, k_scale, v_scale, weights, max_length, true);
}

Tensor kv_evict(const Tensor& k_pages, const Tensor& v_pages, const Tensor& weights, const Tensor& index_pages,
                const Tensor& block_tables, const Tensor& lengths, int64_t budget, int64_t sinks, int64_t recent,
                const OptTensor& k_scale, const OptTensor& v_scale) {
  const at::DeviceGuard guard(k_pages.device());
  const nve_amd_kv_pages_t pages = pages_of(k_pages, v_pages, k_scale, v_scale, weights, index_pages);
  check_device(block_tables, k_pages, "block_tables");
  check_type(block_tables, at::kInt, "block_tables");
  TORCH_CHECK_VALUE(block_tables.dim() == 2 && (block_tables.stride(1) == 1 || block_tables.size(1) <= 1 ||
                                                 block_tables.size(0) == 0),
                    "nve_ops: block_tables must be [sequences, pages] with a contiguous last dimension, got ",
                    block_tables.sizes());
  const int64_t n = block_tables.size(0);
  nve_amd_kv_evict_t c{};
  c.num_seqs = n;
  c.block_tables = static_cast<const int32_t*>(block_tables.data_ptr());
  c.table_stride = block_tables.stride(0);
  c.max_pages = block_tables.size(1);
  c.lengths = static_cast<const int32_t*>(optional_row(lengths, k_pages, at::kInt, n, "lengths"));
  Tensor out = at::empty({n}, lengths.options());
  c.new_lengths = static_cast<int32_t*>(out.data_ptr());
  c.budget = budget;
  c.sinks = sinks;
  c.recent = recent;
  uint64_t need = 0;
  check_status(nve_amd_kv_evict_workspace_size(&pages, &c, &need));
  Tensor ws;
  if (need > 0) ws = bytes(need, k_pages);
  check_status(nve_amd_kv_evict(&pages, &c, need > 0 ? ws.data_ptr() : nullptr, need, stream_of(k_pages)));
  return out;
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(nve_ops, m) {
  m.def(
      "kv_append(Tensor k, Tensor v, Tensor(a!) k_pages, Tensor(b!) v_pages, Tensor slots, Tensor? q, "
      "Tensor? positions, Tensor? cos_sin, int[]? sections, bool interleaved, Tensor? index, Tensor(c!)? k_scale, "
      "Tensor(d!)? v_scale, Tensor(e!)? weights, Tensor(f!)? index_pages) -> Tensor");
  m.def(
      "kv_append_norm(Tensor k, Tensor v, Tensor(a!) k_pages, Tensor(b!) v_pages, Tensor slots, Tensor? q, "
      "Tensor? positions, Tensor? cos_sin, int[]? sections, bool interleaved, Tensor? index, Tensor(c!)? k_scale, "
      "Tensor(d!)? v_scale, Tensor(e!)? weights, Tensor(f!)? index_pages, Tensor? q_norm, Tensor? k_norm, "
      "float eps) -> Tensor");
  m.def(
      "kv_attend(Tensor q, Tensor k_pages, Tensor v_pages, Tensor block_tables, Tensor lengths, float scale, "
      "Tensor? k_scale, Tensor? v_scale, Tensor(a!)? weights, int max_length) -> Tensor");
  m.def(
      "kv_attend_lse(Tensor q, Tensor k_pages, Tensor v_pages, Tensor block_tables, Tensor lengths, float scale, "
      "Tensor? k_scale, Tensor? v_scale, Tensor(a!)? weights, int max_length) -> (Tensor, Tensor)");
  m.def(
      "kv_evict(Tensor(a!) k_pages, Tensor(b!) v_pages, Tensor(c!) weights, Tensor(d!) index_pages, "
      "Tensor block_tables, Tensor lengths, int budget, int sinks, int recent, Tensor(e!)? k_scale, "
      "Tensor(f!)? v_scale) -> Tensor");
}

TORCH_LIBRARY_IMPL(nve_ops, CUDA, m) {
  m.impl("kv_append", &kv_append);
  m.impl("kv_append_norm", &kv_append_norm);
  m.impl("kv_attend", &kv_attend);
  m.impl("kv_attend_lse", &kv_attend_lse);
  m.impl("kv_evict", &kv_evict);
}
