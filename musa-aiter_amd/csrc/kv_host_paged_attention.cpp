// Host-side argument handling of the operators on paged caches of plain values (third part of the _kv_host module), as
// in kv_host_serving.cpp: the common arguments are checked, packed and passed on here, everything else is left to the
// Python layer's checks with nothing launched.  One of these calls costs 6 us of host time, 20 less than in Python.
#include <torch/extension.h>

#include <cstdint>

#include "kv_host_checks.h"
#include "musa_aiter_kv_paged_attention.h"

namespace py = pybind11;

namespace {

using namespace kv_host;
using Call = musa_aiter_hip_paged_attention_call;

constexpr int64_t kMaxRoom = int64_t{1} << 29;

// Query rows, one or two caches and the tables of a call; false where they are not taken as they are.
bool pack_rows(Call& c, int64_t device, const at::Tensor* q, const at::Tensor* kc, const at::Tensor* vc,
               const at::Tensor* tables, const at::Tensor* lens, const py::handle& starts_h, int64_t longest,
               double softmax_scale, int64_t window, int64_t sinks) {
  if (!q || !kc || !vc || !tables || !lens) return false;
  const at::Tensor* starts = nullptr;
  if (!starts_h.is_none() && (starts = plain(starts_h, device)) == nullptr) return false;
  if (q->dim() != 3 || kc->dim() != 4 || vc->sizes() != kc->sizes() || tables->dim() != 2 || lens->dim() != 1) return false;
  const int64_t rows = q->size(0), heads = q->size(1), hd = q->size(2), batch = tables->size(0);
  const int64_t nb = kc->size(0), nh = kc->size(1), bs = kc->size(3), width = tables->size(1);
  const auto type = q->scalar_type();
  if (rows < 1 || rows > kMaxRoom || heads < 1 || heads > 65535 || nh < 1 || heads % nh != 0 || hd < 1 || hd > 512 ||
      kc->size(2) != hd || lens->size(0) != batch || !float_kind(type) || kc->scalar_type() != type ||
      vc->scalar_type() != type || !packed_blocks(*kc) || !packed_blocks(*vc) || (hd > 1 && q->stride(2) != 1) ||
      !index_kind(tables->scalar_type()) || !index_kind(lens->scalar_type()) || !rows_packed(*tables) ||
      !rows_packed(*lens) || rows * heads >= int64_t{1} << 31 || width * bs > kMaxRoom)
    return false;
  if (starts ? starts->dim() != 1 || starts->size(0) != batch + 1 || !index_kind(starts->scalar_type()) ||
                   !rows_packed(*starts)
             : rows != batch)
    return false;
  c.query = q->data_ptr();
  const at::Tensor* caches[2] = {kc, vc};
  for (int i = 0; i < 2; ++i) {
    c.cache[i] = caches[i]->data_ptr();
    c.cache_block_stride[i] = caches[i]->stride(0) * caches[i]->element_size();
  }
  c.tables = tables->data_ptr();
  c.lens = lens->data_ptr();
  c.starts = starts ? starts->data_ptr() : nullptr;
  c.rows = rows;
  c.batch = batch;
  c.heads = heads;
  c.kv_heads = nh;
  c.head_dim = hd;
  c.block_size = bs;
  c.num_blocks = nb;
  c.max_blocks = width;
  c.query_row_stride = q->stride(0);
  c.query_head_stride = q->stride(1);
  c.table_stride = tables->stride(0);
  c.window = window;
  c.sinks = window > 0 ? sinks : 0;
  c.longest = longest < 0 ? width * bs : longest;
  c.softmax_scale = softmax_scale;
  c.dtype = float_id(type);
  c.wide_tables = tables->scalar_type() == at::kLong;
  c.wide_lens = lens->scalar_type() == at::kLong;
  c.wide_starts = starts && starts->scalar_type() == at::kLong;
  return true;
}

// kv_paged_attention (masks None) and kv_paged_attention_tree.  `longest` < 0: what the tables have room for.  Returns
// (status, out, lse or None).
py::tuple paged_attention_call(const py::handle& query_h, const py::handle& key_h, const py::handle& value_h,
                               const py::handle& tables_h, const py::handle& lens_h, const py::handle& masks_h,
                               const py::handle& starts_h, const py::handle& out_h, int64_t longest,
                               double softmax_scale, int64_t window, int64_t sinks, bool with_lse, uint64_t entry,
                               uint64_t workspace_entry, uint64_t stream, int64_t device) {
  const at::Tensor* q = plain(query_h, device);
  Call c{};
  if (!pack_rows(c, device, q, plain(key_h, device), plain(value_h, device), plain(tables_h, device),
                 plain(lens_h, device), starts_h, longest, softmax_scale, window, sinks))
    return not_taken();
  if (!masks_h.is_none()) {
    const at::Tensor* masks = plain(masks_h, device);
    if (!masks || masks->dim() != 2 || masks->size(0) != c.rows || masks->size(1) < 1 ||
        masks->scalar_type() != at::kLong || !rows_packed(*masks))
      return not_taken();
    c.masks = static_cast<const int64_t*>(masks->data_ptr());
    c.mask_words = masks->size(1);
    c.mask_stride = masks->stride(0);
  }
  at::Tensor out, lse;
  if (out_h.is_none()) {
    out = at::empty(q->sizes(), q->options().memory_format(at::MemoryFormat::Contiguous));
  } else {
    const at::Tensor* o = plain(out_h, device);
    if (!o || o->sizes() != q->sizes() || o->scalar_type() != q->scalar_type() || !o->is_contiguous()) return not_taken();
    for (const py::handle& h : {query_h, key_h, value_h, tables_h, lens_h, starts_h, masks_h}) {
      const at::Tensor* read = plain(h, device);
      if (read && spans_meet(*o, *read)) return not_taken();
    }
    out = *o;
  }
  if (with_lse) lse = at::empty({c.rows, c.heads}, q->options().dtype(at::kFloat));
  c.out = out.data_ptr();
  c.lse = with_lse ? static_cast<float*>(lse.data_ptr()) : nullptr;
  c.fill_rows = out_h.is_none();
  at::Tensor workspace;
  c.workspace_bytes = reinterpret_cast<decltype(&musa_aiter_hip_paged_attention_workspace)>(workspace_entry)(&c);
  if (c.workspace_bytes > 0) {
    workspace = at::empty({c.workspace_bytes}, q->options().dtype(at::kByte));
    c.workspace = workspace.data_ptr();
  }
  const int64_t status = reinterpret_cast<decltype(&musa_aiter_hip_paged_attention)>(entry)(&c, reinterpret_cast<void*>(stream));
  if (with_lse) return py::make_tuple(status, out, lse);
  return py::make_tuple(status, out, py::none());
}

// kv_accumulate_attention_weights.  Returns the status.
int64_t attention_weights_call(const py::handle& weights_h, const py::handle& query_h, const py::handle& key_h,
                               const py::handle& tables_h, const py::handle& lens_h, const py::handle& lse_h,
                               const py::handle& starts_h, int64_t longest, double softmax_scale, int64_t window,
                               int64_t sinks, uint64_t entry, uint64_t stream, int64_t device) {
  const at::Tensor *key = plain(key_h, device), *weights = plain(weights_h, device), *lse = plain(lse_h, device);
  Call c{};
  if (!weights || !lse ||
      !pack_rows(c, device, plain(query_h, device), key, key, plain(tables_h, device), plain(lens_h, device), starts_h,
                 longest, softmax_scale, window, sinks))
    return kNotTaken;
  if (weights->dim() != 3 || weights->size(0) != c.batch || weights->size(1) != c.kv_heads || weights->size(2) < 1 ||
      !rows_packed(*weights) || weights->scalar_type() != at::kFloat || lse->dim() != 2 || lse->size(0) != c.rows ||
      lse->size(1) != c.heads || lse->scalar_type() != at::kFloat || !lse->is_contiguous() || c.batch > 65535 ||
      c.kv_heads > 65535)
    return kNotTaken;
  for (int64_t i = 0; i < 2; ++i)
    if (weights->size(i) > 1 && weights->stride(i) == 0) return kNotTaken;
  c.weights = static_cast<float*>(weights->data_ptr());
  c.lse = static_cast<float*>(lse->data_ptr());
  c.weight_tokens = weights->size(2);
  c.weight_row_stride = weights->stride(0);
  c.weight_head_stride = weights->stride(1);
  return reinterpret_cast<decltype(&musa_aiter_hip_attention_weights)>(entry)(&c, reinterpret_cast<void*>(stream));
}

// kv_evict_paged_tokens; refs may be None.  Returns (status, kept, None).
py::tuple evict_call(const py::handle& key_h, const py::handle& value_h, const py::handle& weights_h,
                     const py::handle& tables_h, const py::handle& lens_h, const py::handle& keep_h,
                     const py::handle& refs_h, int64_t sinks, int64_t recent, uint64_t entry, uint64_t workspace_entry,
                     uint64_t stream, int64_t device) {
  const at::Tensor *kc = plain(key_h, device), *vc = plain(value_h, device), *weights = plain(weights_h, device),
                   *tables = plain(tables_h, device), *lens = plain(lens_h, device), *keep = plain(keep_h, device);
  if (!kc || !vc || !weights || !tables || !lens || !keep) return not_taken();
  const at::Tensor* refs = nullptr;
  if (!refs_h.is_none() && (refs = plain(refs_h, device)) == nullptr) return not_taken();
  const int64_t lead = kc->dim() - 4;
  if ((lead != 0 && lead != 1) || vc->sizes() != kc->sizes() || vc->scalar_type() != kc->scalar_type() ||
      tables->dim() != 2 || lens->dim() != 1 || keep->dim() != 1 || weights->dim() != 3 + lead)
    return not_taken();
  const int64_t layers = lead ? kc->size(0) : 1, nb = kc->size(lead), nh = kc->size(lead + 1), hd = kc->size(lead + 2),
                bs = kc->size(lead + 3), batch = tables->size(0), width = tables->size(1), elt = kc->element_size();
  if ((elt != 1 && elt != 2 && elt != 4) || batch < 1 || kc->data_ptr() == vc->data_ptr() || lens->size(0) != batch || keep->size(0) != batch ||
      !packed_blocks(*kc) || !packed_blocks(*vc) || blocks_meet(*kc, *vc) || !index_kind(tables->scalar_type()) ||
      !index_kind(lens->scalar_type()) || !index_kind(keep->scalar_type()) || !rows_packed(*tables) ||
      !rows_packed(*lens) || !rows_packed(*keep) || weights->scalar_type() != at::kFloat ||
      (lead && weights->size(0) != layers) || weights->size(lead) != batch || weights->size(lead + 1) != nh ||
      weights->size(lead + 2) < 1 || !rows_packed(*weights) || width * bs > kMaxRoom || hd > 65535 ||
      layers * batch * nh >= int64_t{1} << 31)
    return not_taken();
  for (int64_t i = 0; i < 2 + lead; ++i)
    if (weights->size(i) > 1 && weights->stride(i) == 0) return not_taken();
  if (refs && (refs->dim() != 1 || refs->size(0) != nb || !index_kind(refs->scalar_type()) || !rows_packed(*refs)))
    return not_taken();
  musa_aiter_hip_evict_call c{};
  const at::Tensor* caches[2] = {kc, vc};
  for (int i = 0; i < 2; ++i) {
    c.cache[i] = caches[i]->data_ptr();
    c.cache_layer_stride[i] = lead ? caches[i]->stride(0) * elt : 0;
    c.cache_block_stride[i] = caches[i]->stride(lead) * elt;
  }
  c.weights = static_cast<float*>(weights->data_ptr());
  c.tables = tables->data_ptr();
  c.lens = lens->data_ptr();
  c.keep = keep->data_ptr();
  c.refs = refs ? refs->data_ptr() : nullptr;
  c.layers = layers;
  c.batch = batch;
  c.kv_heads = nh;
  c.head_dim = hd;
  c.block_size = bs;
  c.num_blocks = nb;
  c.max_blocks = width;
  c.element_bytes = elt;
  c.weight_tokens = weights->size(lead + 2);
  c.weight_layer_stride = lead ? weights->stride(0) : 0;
  c.weight_row_stride = weights->stride(lead);
  c.weight_head_stride = weights->stride(lead + 1);
  c.table_stride = tables->stride(0);
  c.sinks = sinks;
  c.recent = recent;
  c.wide_tables = tables->scalar_type() == at::kLong;
  c.wide_lens = lens->scalar_type() == at::kLong;
  c.wide_keep = keep->scalar_type() == at::kLong;
  c.wide_refs = refs && refs->scalar_type() == at::kLong;
  at::Tensor kept = at::empty({batch}, tables->options().dtype(at::kLong));
  c.kept = static_cast<int64_t*>(kept.data_ptr());
  c.workspace_bytes = reinterpret_cast<decltype(&musa_aiter_hip_evict_workspace)>(workspace_entry)(&c);
  at::Tensor workspace = at::empty({c.workspace_bytes}, tables->options().dtype(at::kByte));
  c.workspace = workspace.data_ptr();
  const int64_t status = reinterpret_cast<decltype(&musa_aiter_hip_evict)>(entry)(&c, reinterpret_cast<void*>(stream));
  return py::make_tuple(status, kept, py::none());
}

}  // namespace

void add_paged_attention_calls(py::module_& m) {
  m.def("paged_attention_call", taken_or_left(&paged_attention_call));
  m.def("attention_weights_call", &attention_weights_call);
  m.def("evict_call", taken_or_left(&evict_call));
}
