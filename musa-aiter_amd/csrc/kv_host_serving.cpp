// Host-side argument handling of the operators on block-scaled FP8 caches and pages (second part of the _kv_host
// module).  As paged_call in kv_host.cpp: each function takes the common arguments as they are, packs the C call and
// makes it, and returns kNotTaken, with nothing launched, for everything else; the Python layer then makes its own
// checks, which convert or raise.  In Python the checks cost 25 us a call, more than a decode step's kernels.
#include <c10/util/Exception.h>
#include <torch/extension.h>

#include <cstdint>

#include "kv_host_calls.h"
#include "kv_host_checks.h"
#include "musa_aiter_kv_serving.h"

namespace py = pybind11;

namespace {

using namespace kv_host;

// kv_paged_attention_fp8.  `longest` < 0: what the tables have room for.  Returns (status, out, lse or None).
py::tuple attention_call(const py::handle& query_h, const py::handle& key_h, const py::handle& value_h,
                         const py::handle& tables_h, const py::handle& lens_h, const py::handle& ks_h,
                         const py::handle& vs_h, const py::handle& starts_h, const py::handle& out_h, int64_t longest,
                         double softmax_scale, int64_t window, int codec, bool with_lse, uint64_t entry,
                         uint64_t splits_entry, uint64_t workspace_entry, uint64_t stream, int64_t device) {
  const at::Tensor *q = plain(query_h, device), *kc = plain(key_h, device), *vc = plain(value_h, device),
                   *tables = plain(tables_h, device), *lens = plain(lens_h, device), *ks = plain(ks_h, device),
                   *vs = plain(vs_h, device);
  if (!q || !kc || !vc || !tables || !lens || !ks || !vs) return not_taken();
  const at::Tensor* starts = nullptr;
  if (!starts_h.is_none() && (starts = plain(starts_h, device)) == nullptr) return not_taken();
  if (q->dim() != 3 || kc->dim() != 4 || vc->sizes() != kc->sizes() || tables->dim() != 2 || lens->dim() != 1 ||
      ks->dim() != 2 || vs->dim() != 2)
    return not_taken();
  const int64_t rows = q->size(0), heads = q->size(1), hd = q->size(2), batch = tables->size(0);
  const int64_t nb = kc->size(0), nh = kc->size(1), bs = kc->size(3), width = tables->size(1);
  if (rows < 1 || heads < 1 || nh < 1 || heads % nh != 0 || kc->size(2) != hd || hd < 1 || hd > 512 ||
      lens->size(0) != batch || ks->size(0) != nb || ks->size(1) != nh || vs->sizes() != ks->sizes() ||
      ks->scalar_type() != at::kFloat || vs->scalar_type() != at::kFloat || !float_kind(q->scalar_type()) ||
      !fp8_kind(kc->scalar_type()) || !fp8_kind(vc->scalar_type()) || !packed_blocks(*kc) || !packed_blocks(*vc) ||
      (hd > 1 && q->stride(2) != 1) || !index_kind(tables->scalar_type()) || !index_kind(lens->scalar_type()) ||
      !rows_packed(*tables) || !rows_packed(*lens) || rows * heads >= int64_t{1} << 31 ||
      width * bs > int64_t{1} << 29)
    return not_taken();
  if (starts ? starts->dim() != 1 || starts->size(0) != batch + 1 || !index_kind(starts->scalar_type()) ||
                   !rows_packed(*starts)
             : rows != batch)
    return not_taken();
  at::Tensor out;
  if (out_h.is_none()) {
    out = at::empty(q->sizes(), q->options().memory_format(at::MemoryFormat::Contiguous));
  } else {
    const at::Tensor* o = plain(out_h, device);
    if (!o || o->sizes() != q->sizes() || o->scalar_type() != q->scalar_type() || !o->is_contiguous()) return not_taken();
    out = *o;
  }
  at::Tensor lse;
  if (with_lse) lse = at::empty({rows, heads}, q->options().dtype(at::kFloat));
  musa_aiter_hip_attention_call c{};
  c.query = q->data_ptr();
  c.out = out.data_ptr();
  c.lse = with_lse ? static_cast<float*>(lse.data_ptr()) : nullptr;
  const at::Tensor* caches[2] = {kc, vc};
  const at::Tensor* scales[2] = {ks, vs};
  for (int i = 0; i < 2; ++i) {
    c.cache[i] = caches[i]->data_ptr();
    c.cache_block_stride[i] = caches[i]->stride(0);
    c.scale[i] = static_cast<const float*>(scales[i]->data_ptr());
    c.scale_block_stride[i] = scales[i]->stride(0);
    c.scale_head_stride[i] = scales[i]->stride(1);
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
  c.splits = 1;
  c.softmax_scale = softmax_scale;
  c.dtype = float_id(q->scalar_type());
  c.codec = codec;
  c.wide_tables = tables->scalar_type() == at::kLong;
  c.wide_lens = lens->scalar_type() == at::kLong;
  c.wide_starts = starts && starts->scalar_type() == at::kLong;
  c.fill_rows = out_h.is_none();
  at::Tensor workspace;
  c.splits = reinterpret_cast<decltype(&musa_aiter_hip_attention_splits)>(splits_entry)(&c, longest < 0 ? width * bs : longest);
  if (c.splits != 1) {
    c.workspace_bytes = reinterpret_cast<decltype(&musa_aiter_hip_attention_workspace)>(workspace_entry)(&c);
    workspace = at::empty({c.workspace_bytes}, q->options().dtype(at::kByte));
    c.workspace = workspace.data_ptr();
  }
  const int64_t status = reinterpret_cast<decltype(&musa_aiter_hip_attention)>(entry)(&c, reinterpret_cast<void*>(stream));
  if (with_lse) return py::make_tuple(status, out, lse);
  return py::make_tuple(status, out, py::none());
}

// kv_linear_to_paged_fp8_block outside of captures; the caller holds the stream's lock.  Returns the status.
int64_t block_store_call(const py::handle& lk_h, const py::handle& lv_h, const py::handle& key_h,
                         const py::handle& value_h, const py::handle& slots_h, const py::handle& ks_h,
                         const py::handle& vs_h, int codec, uint64_t entry, uint64_t claims, uint64_t report,
                         uint64_t guard, int64_t report_words, int64_t stamp, uint64_t stream, int64_t device) {
  const at::Tensor *lk = plain(lk_h, device), *lv = plain(lv_h, device), *kc = plain(key_h, device),
                   *vc = plain(value_h, device), *slots = plain(slots_h, device), *ks = plain(ks_h, device),
                   *vs = plain(vs_h, device);
  if (!lk || !lv || !kc || !vc || !slots || !ks || !vs) return kNotTaken;
  const int64_t lead = kc->dim() - 4;
  if ((lead != 0 && lead != 1) || vc->sizes() != kc->sizes() || lk->dim() != 3 + lead || lv->sizes() != lk->sizes() ||
      slots->dim() != 1 || slots->scalar_type() != at::kLong || !slots->is_contiguous() || ks->dim() != 2 + lead ||
      vs->sizes() != ks->sizes())
    return kNotTaken;
  const int64_t layers = lead ? kc->size(0) : 1, nb = kc->size(lead), nh = kc->size(lead + 1), hd = kc->size(lead + 2),
                bs = kc->size(lead + 3), tokens = slots->size(0);
  if (tokens < 1 || lk->size(lead) != tokens || lk->size(lead + 1) != nh || lk->size(lead + 2) != hd ||
      (lead && lk->size(0) != layers) || ks->size(lead) != nb || ks->size(lead + 1) != nh ||
      (lead && ks->size(0) != layers) || !fp8_kind(kc->scalar_type()) || !fp8_kind(vc->scalar_type()) ||
      !packed_blocks(*kc) || !packed_blocks(*vc) || !float_kind(lk->scalar_type()) ||
      lv->scalar_type() != lk->scalar_type() || !lk->is_contiguous() || !lv->is_contiguous() ||
      ks->scalar_type() != at::kFloat || vs->scalar_type() != at::kFloat || !ks->is_contiguous() ||
      !vs->is_contiguous())
    return kNotTaken;
  musa_aiter_hip_block_store_call c{};
  const at::Tensor* lin[2] = {lk, lv};
  const at::Tensor* caches[2] = {kc, vc};
  const at::Tensor* scales[2] = {ks, vs};
  for (int i = 0; i < 2; ++i) {
    c.linear[i] = lin[i]->data_ptr();
    c.cache[i] = caches[i]->data_ptr();
    c.scale[i] = static_cast<float*>(scales[i]->data_ptr());
    c.cache_block_stride[i] = caches[i]->stride(lead);
    c.cache_layer_stride[i] = lead ? caches[i]->stride(0) : 0;
  }
  c.slots = static_cast<const int64_t*>(slots->data_ptr());
  c.claims = reinterpret_cast<const musa_aiter_hip_claims*>(claims);
  c.report = reinterpret_cast<int64_t*>(report);
  c.guard = reinterpret_cast<int64_t*>(guard);
  c.stamp = stamp;
  c.report_words = report_words;
  c.num_layers = layers;
  c.num_tokens = tokens;
  c.num_blocks = nb;
  c.num_heads = nh;
  c.head_dim = hd;
  c.block_size = bs;
  c.lin_token_stride = nh * hd;
  c.lin_layer_stride = tokens * nh * hd;
  c.codec = codec;
  c.lin_dtype = float_id(lk->scalar_type());
  if (claims != 0 && c.claims->capacity < nb * bs) return kNotTaken;
  const auto fn = reinterpret_cast<decltype(&musa_aiter_hip_block_store)>(entry);
  py::gil_scoped_release unlocked;  // the entry waits for the device's verdict
  return fn(&c, reinterpret_cast<void*>(stream));
}

// The page operations: `lens`, `rows`, caches and scales None where the operation has none.  Returns (status, slots
// [batch, max_new] or None, result or None).
py::tuple pages_call(const py::handle& key_h, const py::handle& value_h, const py::handle& tables_h,
                     const py::handle& lens_h, const py::handle& refs_h, const py::handle& rows_h,
                     const py::handle& ks_h, const py::handle& vs_h, int64_t block_size, int64_t max_new, int kind,
                     uint64_t entry, uint64_t workspace_entry, uint64_t stream, int64_t device) {
  constexpr int kExtend = 1, kCompact = 2, kFree = 3;  // the numbers of musa_aiter_hip_pages_workspace, and free
  const at::Tensor *tables = plain(tables_h, device), *refs = plain(refs_h, device);
  if (!tables || !refs || tables->dim() != 2 || refs->dim() != 1 || tables->size(0) < 1 || tables->size(1) < 1 ||
      refs->size(0) < 1 || !index_kind(tables->scalar_type()) || refs->scalar_type() != tables->scalar_type() ||
      !refs->is_contiguous() || !rows_packed(*tables) ||
      (tables->size(0) > 1 && tables->stride(0) < tables->size(1)))
    return not_taken();
  const int64_t batch = tables->size(0);
  musa_aiter_hip_pages_call c{};
  c.tables = tables->data_ptr();
  c.refs = refs->data_ptr();
  if (kind != kCompact) {
    const at::Tensor *lens = plain(lens_h, device), *rows = plain(rows_h, device);
    if (!lens || !rows || lens->dim() != 1 || rows->dim() != 1 || lens->size(0) != batch || rows->size(0) != batch ||
        lens->scalar_type() != tables->scalar_type() || !index_kind(rows->scalar_type()) || !lens->is_contiguous() ||
        !rows->is_contiguous())
      return not_taken();
    c.lens = lens->data_ptr();
    c.rows = rows->data_ptr();
    c.wide_rows = rows->scalar_type() == at::kLong;
  }
  c.batch = batch;
  c.max_blocks = tables->size(1);
  c.table_stride = tables->stride(0);
  c.num_blocks = refs->size(0);
  c.block_size = block_size;
  c.wide = tables->scalar_type() == at::kLong;
  at::Tensor slots, result;
  if (kind == kExtend || kind == kCompact) {
    const at::Tensor *kc = plain(key_h, device), *vc = plain(value_h, device);
    if (!kc || !vc) return not_taken();
    const int64_t lead = kc->dim() - 4;
    if ((lead != 0 && lead != 1) || vc->sizes() != kc->sizes() || vc->scalar_type() != kc->scalar_type() ||
        kc->size(lead) != refs->size(0) || !packed_blocks(*kc) || !packed_blocks(*vc) || max_new < 0)
      return not_taken();
    const at::Tensor* caches[2] = {kc, vc};
    const py::handle given[2] = {ks_h, vs_h};
    if (ks_h.is_none() != vs_h.is_none()) return not_taken();
    c.layers = lead ? kc->size(0) : 1;
    c.block_bytes = kc->element_size() * kc->size(lead + 1) * kc->size(lead + 2) * kc->size(lead + 3);
    c.scale_values = kc->size(lead + 1);
    c.block_size = kc->size(lead + 3);
    for (int i = 0; i < 2; ++i) {
      c.cache[i] = caches[i]->data_ptr();
      c.block_stride[i] = caches[i]->stride(lead) * kc->element_size();
      c.layer_stride[i] = lead ? caches[i]->stride(0) * kc->element_size() : 0;
      if (given[i].is_none()) continue;
      const at::Tensor* s = plain(given[i], device);
      if (!s || s->dim() != 2 + lead || s->scalar_type() != at::kFloat || !s->is_contiguous() ||
          s->size(lead) != refs->size(0) || s->size(lead + 1) != c.scale_values || (lead && s->size(0) != c.layers))
        return not_taken();
      c.scale[i] = static_cast<float*>(s->data_ptr());
    }
    const auto options = tables->options().dtype(at::kLong);
    if (kind == kExtend) {
      slots = at::empty({batch, max_new}, options);
      c.slots = static_cast<int64_t*>(slots.data_ptr());
      c.max_new = max_new;
    }
    result = at::empty({}, options);
    c.result = static_cast<int64_t*>(result.data_ptr());
  } else if (block_size < 1) {
    return not_taken();
  }
  at::Tensor workspace;
  if (kind != kFree) {
    c.workspace_bytes = reinterpret_cast<decltype(&musa_aiter_hip_pages_workspace)>(workspace_entry)(&c, kind);
    workspace = at::empty({c.workspace_bytes}, tables->options().dtype(at::kByte));
    c.workspace = workspace.data_ptr();
  }
  const int64_t status = reinterpret_cast<decltype(&musa_aiter_hip_pages_free)>(entry)(&c, reinterpret_cast<void*>(stream));
  return py::make_tuple(status, slots.defined() ? py::cast(slots) : py::none(),
                        result.defined() ? py::cast(result) : py::none());
}

}  // namespace

void add_serving_calls(py::module_& m) {
  m.def("attention_call", taken_or_left(&attention_call));
  m.def("block_store_call", &block_store_call);
  m.def("pages_call", taken_or_left(&pages_call));
}
