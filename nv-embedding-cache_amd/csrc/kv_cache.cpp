// kv_cache.cpp -- the paged key-value cache of an attention layer: argument
// checks and launches of append, attend and evict (kernels/kv_*.hip).
//
// Everything the host can see is checked here; slots, positions, page ids and
// lengths lie in device memory and are checked by the kernels.
#include "kv_cache.hpp"

#include <algorithm>
#include <cmath>
#include <limits>

#include "dtypes.hpp"
#include "kernels/kv_launch.hpp"
#include "runtime.hpp"

namespace nve_amd {

namespace {

constexpr int64_t kMaxGrid = std::numeric_limits<int32_t>::max();

bool aligned(const void* p, uintptr_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

KvPages pages_of(const nve_amd_kv_pages_t* p) {
  NVE_CHECK_ARG(p != nullptr, "pages must not be NULL");
  NVE_CHECK_ARG(p->num_pages >= 0 && p->num_pages <= kMaxGrid, "Invalid num_pages ", p->num_pages);
  NVE_CHECK_ARG(p->num_heads >= 1 && p->num_heads <= 65535, "Invalid num_heads ", p->num_heads);
  NVE_CHECK_ARG(p->page_size >= 8 && p->page_size <= 1024 && (p->page_size & (p->page_size - 1)) == 0,
                "page_size must be a power of two from 8 to 1024 (got ", p->page_size, ")");
  NVE_CHECK_ARG(p->head_dim >= 8 && p->head_dim <= 256 && p->head_dim % 8 == 0,
                "head_dim must be a multiple of 8 from 8 to 256 (got ", p->head_dim, ")");
  const int dt = (int)p->dtype;
  NVE_CHECK_ARG(dt == kF32 || dt == kF16 || dt == kBF16 || dt == kE4M3,
                "pages must be float32, float16, bfloat16 or e4m3 (got type ", dt, ")");
  if (p->num_pages > 0) NVE_CHECK_ARG(p->k && p->v, "k and v pages must not be NULL");
  NVE_CHECK_ARG(aligned(p->k, 16) && aligned(p->v, 16), "k and v pages must be 16-byte aligned");
  if (dt == kE4M3) {
    if (p->num_pages > 0) NVE_CHECK_ARG(p->k_scale && p->v_scale, "e4m3 pages need k_scale and v_scale");
  } else {
    NVE_CHECK_ARG(!p->k_scale && !p->v_scale, "only e4m3 pages have scales");
  }
  NVE_CHECK_ARG((int64_t)p->num_heads * p->page_size * p->head_dim * value_elem_bytes(dt) <= kMaxGrid,
                "a page of all heads must be smaller than 2 GiB");
  KvPages c{};
  c.k = static_cast<uint8_t*>(p->k);
  c.v = static_cast<uint8_t*>(p->v);
  c.k_scale = p->k_scale;
  c.v_scale = p->v_scale;
  c.weights = p->weights;
  c.index = p->index;
  c.num_pages = p->num_pages;
  c.heads = p->num_heads;
  c.page = p->page_size;
  c.page_bits = __builtin_ctz((unsigned)p->page_size);
  c.dim = p->head_dim;
  c.dtype = dt;
  return c;
}

void check_dtype(const KvPages& c, nve_data_type_t dtype) {
  if (c.dtype == kE4M3)
    NVE_CHECK_ARG(dtype == NVE_DTYPE_FLOAT16 || dtype == NVE_DTYPE_BFLOAT16,
                  "e4m3 pages take float16 or bfloat16 rows (got type ", (int)dtype, ")");
  else
    NVE_CHECK_ARG((int)dtype == c.dtype, "the rows' type ", (int)dtype, " is not the pages' type ", c.dtype);
}

// The slots a table row of max_pages entries can name, at most max_length (0: no bound).
int64_t extent(const KvPages& c, int64_t max_pages, int64_t max_length) {
  NVE_CHECK_ARG(max_pages >= 0 && max_pages <= kMaxGrid / c.page, "Invalid max_pages ", max_pages);
  NVE_CHECK_ARG(max_length >= 0, "Invalid max_length ", max_length);
  const int64_t all = max_pages * c.page;
  return max_length > 0 && max_length < all ? max_length : all;
}

KvAppend append_of(const nve_amd_kv_pages_t* pages, const nve_amd_kv_append_t* p) {
  KvAppend a{};
  a.pages = pages_of(pages);
  NVE_CHECK_ARG(p != nullptr, "call must not be NULL");
  check_dtype(a.pages, p->dtype);
  NVE_CHECK_ARG(p->num_tokens >= 0, "Invalid num_tokens ", p->num_tokens);
  a.q_heads = p->q ? p->num_q_heads : 0;
  // the launches go by whole tokens, of fewer than 2^26 rows
  NVE_CHECK_ARG(a.q_heads >= 0 && a.q_heads < (1 << 25), "Invalid num_q_heads ", p->num_q_heads);
  NVE_CHECK_ARG(p->num_tokens <= kMaxGrid / (a.q_heads + 2 * (int64_t)a.pages.heads), "Too many tokens");
  if (p->num_tokens > 0) {
    NVE_CHECK_ARG(p->slots && p->k && p->v, "slots, k and v must not be NULL");
    if (a.q_heads > 0) NVE_CHECK_ARG(p->q_out != nullptr, "q_out must not be NULL");
  }
  NVE_CHECK_ARG(p->rot_dim >= 0 && p->rot_dim % 2 == 0 && p->rot_dim <= a.pages.dim,
                "rot_dim must be even and at most head_dim (got ", p->rot_dim, ")");
  a.tokens = p->num_tokens;
  a.slots = p->slots;
  a.dtype = (int)p->dtype;
  a.k = {static_cast<const uint8_t*>(p->k), p->k_token_stride, p->k_head_stride};
  a.v = {static_cast<const uint8_t*>(p->v), p->v_token_stride, p->v_head_stride};
  a.q = {static_cast<const uint8_t*>(p->q), p->q_token_stride, p->q_head_stride};
  a.q_out = static_cast<uint8_t*>(p->q_out);
  a.q_out_token_stride = p->q_out_token_stride;
  a.q_out_head_stride = p->q_out_head_stride;
  a.index = p->index;
  a.positions = p->positions;
  a.axis_stride = p->axis_stride;
  a.rot = p->rot_dim;
  a.interleaved = p->interleaved != 0;
  a.axes = 1;
  if (a.rot > 0) {
    NVE_CHECK_ARG(p->num_axes >= 1 && p->num_axes <= 4, "num_axes must be 1 to 4 (got ", p->num_axes, ")");
    NVE_CHECK_ARG(p->max_position >= 0, "Invalid max_position ", p->max_position);
    if (p->num_tokens > 0) NVE_CHECK_ARG(p->positions != nullptr, "rotary rows need positions");
    if (p->num_tokens > 0 && p->max_position > 0) NVE_CHECK_ARG(p->cos_sin != nullptr, "cos_sin must not be NULL");
    a.cos_sin = p->cos_sin;
    a.max_position = p->max_position;
    a.axes = p->num_axes;
    int64_t end = 0;
    for (int i = 0; i < a.axes; ++i) {
      NVE_CHECK_ARG(p->sections[i] >= 0, "Invalid section ", p->sections[i]);
      end += p->sections[i];
      NVE_CHECK_ARG(end <= a.rot / 2, "the sections hold more than rot_dim / 2 pairs");
      a.ends[i] = (int)end;
    }
    NVE_CHECK_ARG(end == a.rot / 2, "the sections hold ", end, " pairs, not rot_dim / 2 = ", a.rot / 2);
  }
  return a;
}

KvAttend attend_of(const nve_amd_kv_pages_t* pages, const nve_amd_kv_attend_t* p) {
  KvAttend a{};
  a.pages = pages_of(pages);
  NVE_CHECK_ARG(p != nullptr, "call must not be NULL");
  check_dtype(a.pages, p->dtype);
  NVE_CHECK_ARG(p->num_seqs >= 0 && p->num_seqs <= 65535, "num_seqs must be in [0, 65535] (got ", p->num_seqs, ")");
  NVE_CHECK_ARG(p->num_q_heads >= 1 && p->num_q_heads <= 65535 && p->num_q_heads % a.pages.heads == 0,
                "num_q_heads (", p->num_q_heads, ") must be a multiple of the pages' num_heads (", a.pages.heads, ")");
  // a workgroup of 256 threads for each, and a launch has fewer than 2^32 threads
  NVE_CHECK_ARG(p->num_seqs * a.pages.heads < (1 << 24), "Too many heads: ", p->num_seqs, " sequences of ",
                a.pages.heads);
  NVE_CHECK_ARG(!std::isnan(p->scale), "scale must not be NaN");
  a.max_length = extent(a.pages, p->max_pages, p->max_length);
  // the kernels count tiles of at least 64 slots in 32 bits
  NVE_CHECK_ARG((a.max_length / 64 + 1) * p->num_seqs <= kMaxGrid / p->num_q_heads, "Too many slots: ", p->num_seqs,
                " sequences of up to ", a.max_length);
  if (p->num_seqs > 0) {
    NVE_CHECK_ARG(p->q && p->out && p->lengths, "q, out and lengths must not be NULL");
    if (a.max_length > 0) NVE_CHECK_ARG(p->block_tables != nullptr, "block_tables must not be NULL");
    if (p->accumulate && a.pages.num_pages > 0)
      NVE_CHECK_ARG(a.pages.weights != nullptr, "accumulate needs the pages' weights");
  }
  a.seqs = p->num_seqs;
  a.q_heads = p->num_q_heads;
  a.dtype = (int)p->dtype;
  a.q = {static_cast<const uint8_t*>(p->q), p->q_seq_stride, p->q_head_stride};
  a.out = static_cast<uint8_t*>(p->out);
  a.out_seq_stride = p->out_seq_stride;
  a.out_head_stride = p->out_head_stride;
  a.lse = p->lse;
  a.tables = p->block_tables;
  a.table_stride = p->table_stride;
  a.lengths = p->lengths;
  a.scale = p->scale;
  a.accumulate = p->accumulate != 0;
  return a;
}

KvEvict evict_of(const nve_amd_kv_pages_t* pages, const nve_amd_kv_evict_t* p) {
  KvEvict a{};
  a.pages = pages_of(pages);
  NVE_CHECK_ARG(p != nullptr, "call must not be NULL");
  NVE_CHECK_ARG(p->num_seqs >= 0 && p->num_seqs * a.pages.heads <= kMaxGrid && p->num_seqs <= 65535,
                "num_seqs must be in [0, 65535] (got ", p->num_seqs, ")");
  NVE_CHECK_ARG(p->budget >= 0 && p->sinks >= 0 && p->recent >= 0, "budget, sinks and recent must not be negative");
  a.max_length = extent(a.pages, p->max_pages, 0);
  if (p->num_seqs > 0) {
    NVE_CHECK_ARG(p->lengths && p->new_lengths, "lengths and new_lengths must not be NULL");
    if (a.max_length > 0) NVE_CHECK_ARG(p->block_tables != nullptr, "block_tables must not be NULL");
    if (a.pages.num_pages > 0)
      NVE_CHECK_ARG(a.pages.weights && a.pages.index, "eviction needs the pages' weights and index");
  }
  a.seqs = p->num_seqs;
  a.tables = p->block_tables;
  a.table_stride = p->table_stride;
  a.lengths = p->lengths;
  a.new_lengths = p->new_lengths;
  const int64_t cap = (int64_t)1 << 40;  // past every slot and index
  a.budget = std::min(p->budget, cap);
  a.sinks = std::min(p->sinks, cap);
  a.recent = std::min(p->recent, cap);
  return a;
}

void check_workspace(const void* ws, size_t have, size_t need) {
  if (need == 0) return;
  NVE_CHECK_ARG(ws != nullptr && have >= need, "Workspace too small: ", have, " bytes, ", need, " needed");
  NVE_CHECK_ARG(aligned(ws, 16), "The workspace must be 16-byte aligned");
}

}  // namespace

void kv_append_run(const nve_amd_kv_pages_t* pages, const nve_amd_kv_append_t* call, hipStream_t s) {
  NVE_HIP(launch_kv_append(append_of(pages, call), s));
}

size_t kv_attend_workspace_bytes(const nve_amd_kv_pages_t* pages, const nve_amd_kv_attend_t* call) {
  return kv_attend_workspace(attend_of(pages, call));
}

void kv_attend_run(const nve_amd_kv_pages_t* pages, const nve_amd_kv_attend_t* call, void* ws, size_t ws_bytes,
                   hipStream_t s) {
  const KvAttend a = attend_of(pages, call);
  check_workspace(ws, ws_bytes, kv_attend_workspace(a));
  NVE_HIP(launch_kv_attend(a, ws, s));
}

size_t kv_evict_workspace_bytes(const nve_amd_kv_pages_t* pages, const nve_amd_kv_evict_t* call) {
  return kv_evict_workspace(evict_of(pages, call));
}

void kv_evict_run(const nve_amd_kv_pages_t* pages, const nve_amd_kv_evict_t* call, void* ws, size_t ws_bytes,
                  hipStream_t s) {
  const KvEvict a = evict_of(pages, call);
  check_workspace(ws, ws_bytes, kv_evict_workspace(a));
  // every head of a sequence reads its length, the first one writes the new one
  NVE_CHECK_ARG(a.new_lengths + a.seqs <= a.lengths || a.lengths + a.seqs <= a.new_lengths,
                "new_lengths must not overlap lengths");
  NVE_HIP(launch_kv_evict(a, ws, s));
}

}  // namespace nve_amd
