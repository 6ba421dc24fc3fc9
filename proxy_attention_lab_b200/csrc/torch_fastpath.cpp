// Host-side fast path of the Python operators: the common case of paged_attention_decode, paged_attention_prefill and
// fill_kv_pages - CUDA tensors that are already contiguous and already carry 32-bit (64-bit for slot ids) indices,
// torch's current stream, a workspace that exists - checked and handed to the C ABI (include/pal_b200.h) from C++.
//
// The Python wrappers in ops.py mirror the reference's operator layer (src/proxy_attention_lab/ops.py:33-171,
// src/pal_core/src/ops.cpp:36-239) and do the same through ctypes; a small call spends most of its ~16 us there, in
// attribute reads and argument marshalling.  Every function here returns None when a call is not the common case
// (another dtype, a non-contiguous tensor, an index tensor to convert, no workspace yet, a shape it does not like), and
// the wrapper then takes its usual path, which converts what has to be converted and raises the reference's errors.
// Nothing is computed here, and there is no other route to the GPU than the C ABI.
#include <torch/extension.h>

#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <stdexcept>
#include <vector>

#include "pal_b200.h"

namespace {

inline int dtype_code(const at::Tensor& t) {
  if (t.scalar_type() == at::kHalf) return PAL_DTYPE_F16;
  if (t.scalar_type() == at::kBFloat16) return PAL_DTYPE_BF16;
  return -1;
}
inline bool dense_cuda(const at::Tensor& t, const c10::Device& dev) { return t.is_cuda() && t.device() == dev && t.is_contiguous(); }
inline bool int32_like(const at::Tensor& t) { return t.scalar_type() == at::kInt || t.scalar_type() == at::kUInt32; }

void raise_for(int rc) {
  if (rc == PAL_OK) return;
  const char* msg = pal_last_error();
  std::string text = (msg && *msg) ? msg : ("pal_b200 error " + std::to_string(rc));
  if (rc == PAL_ERR_BAD_ARG) throw py::value_error(text);
  throw std::runtime_error(text);
}

// The newest workspace the Python layer holds for (device, stream), if it has `need` bytes; nullptr otherwise.
// `registry` is ops._WORKSPACES: {(device index, cudaStream_t as int): [tensor, ...]}.
void* held_workspace(const py::dict& registry, int device_index, cudaStream_t stream, size_t need, size_t* bytes) {
  py::tuple key = py::make_tuple(device_index, reinterpret_cast<uintptr_t>(stream));
  PyObject* held = PyDict_GetItem(registry.ptr(), key.ptr());  // borrowed
  if (!held || !PyList_Check(held) || PyList_GET_SIZE(held) == 0) return nullptr;
  PyObject* last = PyList_GET_ITEM(held, PyList_GET_SIZE(held) - 1);
  if (!THPVariable_Check(last)) return nullptr;
  const at::Tensor& ws = THPVariable_Unpack(last);
  if ((size_t)ws.numel() < need) return nullptr;
  *bytes = (size_t)ws.numel();
  return ws.data_ptr();
}

// paged_attention_decode / paged_attention_decode_append (new_k, new_v given)
py::object decode(const at::Tensor& q, const at::Tensor& k_pool, const at::Tensor& v_pool, const at::Tensor& page_table,
                  const at::Tensor& seq_lens, int partition_pages, double scale, bool out_f32, const py::dict& registry,
                  const c10::optional<at::Tensor>& new_k, const c10::optional<at::Tensor>& new_v) {
  if (!q.is_cuda()) return py::none();
  const c10::Device dev = q.device();
  const int code = dtype_code(q);
  if (code < 0 || v_pool.dim() != 4 || k_pool.dim() != 5 || page_table.dim() != 2 || q.dim() != 3) return py::none();
  if (!dense_cuda(q, dev) || !dense_cuda(k_pool, dev) || !dense_cuda(v_pool, dev) || !dense_cuda(page_table, dev) ||
      !dense_cuda(seq_lens, dev) || !int32_like(page_table) || !int32_like(seq_lens) || k_pool.scalar_type() != q.scalar_type() ||
      v_pool.scalar_type() != q.scalar_type())
    return py::none();
  const int64_t num_pages = v_pool.size(0), hkv = v_pool.size(1), d = v_pool.size(2), tpp = v_pool.size(3);
  const int64_t S = page_table.size(0), mp = page_table.size(1), hq = q.size(1);
  if (S == 0 || mp == 0 || num_pages == 0 || hkv == 0 || q.size(0) < S || q.size(2) != d || seq_lens.numel() < S || hq % hkv != 0 ||
      k_pool.size(0) != num_pages || k_pool.size(1) != hkv || k_pool.size(2) * 8 != d || k_pool.size(3) != tpp || k_pool.size(4) != 8)
    return py::none();
  const bool append = new_k.has_value();
  if (append) {
    if (!new_v.has_value()) return py::none();
    for (const at::Tensor* t : {&*new_k, &*new_v})
      if (!dense_cuda(*t, dev) || t->scalar_type() != q.scalar_type() || t->dim() != 3 || t->size(0) != S || t->size(1) != hkv || t->size(2) != d)
        return py::none();
  }
  c10::cuda::CUDAGuard guard(dev);
  const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
  const size_t need = pal_decode_workspace_bytes((int)S, (int)hq, (int)hkv, (int)d, (int)tpp, (int)mp, partition_pages);
  size_t ws_bytes = 0;
  void* ws = held_workspace(registry, dev.index(), stream, need > 256 ? need : 256, &ws_bytes);
  if (!ws) return py::none();
  at::Tensor out = at::empty({S, hq, d}, q.options().dtype(out_f32 ? at::kFloat : q.scalar_type()));
  const int dt = code | (out_f32 ? PAL_OUT_F32 : 0);
  int rc;
  if (append)
    rc = pal_paged_attention_decode_append(new_k->data_ptr(), new_v->data_ptr(), q.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(),
                                           page_table.data_ptr(), static_cast<const int32_t*>(seq_lens.data_ptr()), out.data_ptr(), (int)S,
                                           (int)hq, (int)hkv, (int)d, (int)tpp, num_pages, (int)mp, (float)scale, dt, partition_pages, ws,
                                           ws_bytes, stream);
  else
    rc = pal_paged_attention_decode(q.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), page_table.data_ptr(),
                                    static_cast<const int32_t*>(seq_lens.data_ptr()), out.data_ptr(), (int)S, (int)hq, (int)hkv, (int)d,
                                    (int)tpp, num_pages, (int)mp, (float)scale, dt, partition_pages, ws, ws_bytes, stream);
  raise_for(rc);
  return py::cast(out);
}

// paged_attention_prefill (uniform batches) / paged_attention_prefill_ragged (cu_seqlens and the longest count given)
py::object prefill(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& k_pool, const at::Tensor& v_pool,
                   const at::Tensor& page_table, const at::Tensor& hist, int impl, double scale, bool out_f32, const py::dict& registry,
                   const c10::optional<at::Tensor>& cu_seqlens, int max_new_tokens) {
  if (!q.is_cuda()) return py::none();
  const c10::Device dev = q.device();
  const int code = dtype_code(q);
  if (code < 0 || v_pool.dim() != 4 || k_pool.dim() != 5 || page_table.dim() != 2 || q.dim() != 3 || k.dim() != 3 || v.dim() != 3)
    return py::none();
  for (const at::Tensor* t : {&q, &k, &v, &k_pool, &v_pool})
    if (!dense_cuda(*t, dev) || t->scalar_type() != q.scalar_type()) return py::none();
  if (!dense_cuda(page_table, dev) || !dense_cuda(hist, dev) || !int32_like(page_table) || !int32_like(hist)) return py::none();
  const int64_t num_pages = v_pool.size(0), hkv = v_pool.size(1), d = v_pool.size(2), tpp = v_pool.size(3);
  const int64_t S = page_table.size(0), mp = page_table.size(1), total = q.size(0), hq = q.size(1);
  const bool ragged = cu_seqlens.has_value();
  if (ragged && (!dense_cuda(*cu_seqlens, dev) || !int32_like(*cu_seqlens) || cu_seqlens->dim() != 1 || cu_seqlens->numel() != S + 1 ||
                 max_new_tokens <= 0))
    return py::none();
  if (S == 0 || total == 0 || (!ragged && total % S != 0) || num_pages == 0 || mp == 0 || hkv == 0 || hq % hkv != 0 || q.size(2) != d ||
      k.size(0) != total || v.size(0) != total || k.size(1) != hkv || v.size(1) != hkv || k.size(2) != d || v.size(2) != d ||
      hist.numel() < S || k_pool.size(0) != num_pages || k_pool.size(1) != hkv || k_pool.size(2) * 8 != d || k_pool.size(3) != tpp ||
      k_pool.size(4) != 8)
    return py::none();
  c10::cuda::CUDAGuard guard(dev);
  const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
  size_t ws_bytes = 0;
  const int per_seq = ragged ? max_new_tokens : (int)(total / S);
  const size_t need = pal_prefill_workspace_bytes((int)S, per_seq, (int)hq, (int)hkv, (int)d);
  void* ws = held_workspace(registry, dev.index(), stream, need > 256 ? need : 256, &ws_bytes);
  if (!ws) return py::none();
  at::Tensor out = at::empty({total * hq, d}, q.options().dtype(out_f32 ? at::kFloat : q.scalar_type()));
  const int dt = code | (out_f32 ? PAL_OUT_F32 : 0);
  int rc;
  if (ragged)
    rc = pal_paged_attention_prefill_ragged(q.data_ptr(), k.data_ptr(), v.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), page_table.data_ptr(),
                                            static_cast<const int32_t*>(hist.data_ptr()), static_cast<const int32_t*>(cu_seqlens->data_ptr()),
                                            out.data_ptr(), (int)S, total, max_new_tokens, (int)hq, (int)hkv, (int)d, (int)tpp, num_pages,
                                            (int)mp, (float)scale, dt, impl, ws, ws_bytes, stream);
  else
    rc = pal_paged_attention_prefill(q.data_ptr(), k.data_ptr(), v.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), page_table.data_ptr(),
                                     static_cast<const int32_t*>(hist.data_ptr()), out.data_ptr(), (int)S, per_seq, (int)hq, (int)hkv, (int)d,
                                     (int)tpp, num_pages, (int)mp, (float)scale, dt, impl, ws, ws_bytes, stream);
  raise_for(rc);
  return py::cast(out);
}

// fill_kv_pages, in place; `a` is the slot mapping (int64) when `pos` and `seq_map` are None, else the page table.
// Returns True when the call was made.
bool fill(const at::Tensor& new_k, const at::Tensor& new_v, const at::Tensor& k_pool, const at::Tensor& v_pool, const at::Tensor& a,
          const c10::optional<at::Tensor>& pos, const c10::optional<at::Tensor>& seq_map) {
  if (!v_pool.is_cuda()) return false;
  const c10::Device dev = v_pool.device();
  const int code = dtype_code(v_pool);
  if (code < 0 || v_pool.dim() != 4 || k_pool.dim() != 5 || new_k.dim() != 3 || new_v.dim() != 3) return false;
  for (const at::Tensor* t : {&new_k, &new_v, &k_pool, &v_pool})
    if (!dense_cuda(*t, dev) || t->scalar_type() != v_pool.scalar_type()) return false;
  const int64_t num_pages = v_pool.size(0), hkv = v_pool.size(1), d = v_pool.size(2), tpp = v_pool.size(3), T = new_k.size(0);
  if (T == 0 || num_pages == 0 || new_k.size(1) != hkv || new_k.size(2) != d || new_v.size(0) != T || new_v.size(1) != hkv ||
      new_v.size(2) != d || k_pool.size(0) != num_pages || k_pool.size(1) != hkv || k_pool.size(2) * 8 != d || k_pool.size(3) != tpp ||
      k_pool.size(4) != 8 || !dense_cuda(a, dev))
    return false;
  c10::cuda::CUDAGuard guard(dev);
  const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
  int rc;
  if (!pos.has_value()) {
    if (seq_map.has_value() || a.scalar_type() != at::kLong || a.numel() != T) return false;
    rc = pal_fill_kv_pages_slots(new_k.data_ptr(), new_v.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(),
                                 static_cast<const int64_t*>(a.data_ptr()), T, (int)hkv, (int)d, (int)tpp, num_pages, code, stream);
  } else {
    if (!seq_map.has_value() || a.dim() != 2 || !int32_like(a) || !dense_cuda(*pos, dev) || !dense_cuda(*seq_map, dev) || !int32_like(*pos) ||
        !int32_like(*seq_map) || pos->numel() != T || seq_map->numel() != T)
      return false;
    rc = pal_fill_kv_pages(new_k.data_ptr(), new_v.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), a.data_ptr(),
                           static_cast<const int32_t*>(pos->data_ptr()), seq_map->data_ptr(), T, (int)a.size(0), (int)hkv, (int)d, (int)tpp,
                           num_pages, (int)a.size(1), code, stream);
  }
  raise_for(rc);
  return true;
}

// ---- rotary positions ----------------------------------------------------------------------
// The rotation of a call, if it is the common case: contiguous int32 / int64 positions [T] or [axes, T] and float32
// frequencies on `dev`.  Sections, their order and the pairing are checked by the C ABI.
bool rotation_of(pal_rotation* r, const at::Tensor& positions, const at::Tensor& inv_freq, const c10::optional<std::vector<int64_t>>& sections,
                 int order, int pairing, double magnitude, int64_t tokens, const c10::Device& dev) {
  if (!dense_cuda(positions, dev) || !dense_cuda(inv_freq, dev) || inv_freq.scalar_type() != at::kFloat || inv_freq.dim() != 1) return false;
  const bool wide = positions.scalar_type() == at::kLong;
  if (!wide && positions.scalar_type() != at::kInt) return false;
  const int64_t axes = sections ? (int64_t)sections->size() : 1;
  if (axes < 1 || axes > PAL_MAX_ROTARY_AXES) return false;
  if (!(positions.dim() == 2 && positions.size(0) == axes && positions.size(1) == tokens) &&
      !(axes == 1 && positions.dim() == 1 && positions.size(0) == tokens))
    return false;
  r->positions = positions.data_ptr();
  r->positions_axis_stride = tokens;
  r->inv_freq = static_cast<const float*>(inv_freq.data_ptr());
  r->magnitude = (float)magnitude;
  r->num_freqs = (int32_t)inv_freq.size(0);
  r->num_axes = (int32_t)axes;
  for (int64_t a = 0; a < PAL_MAX_ROTARY_AXES; ++a) {
    const int64_t n = sections ? (a < axes ? (*sections)[a] : 0) : (a == 0 ? inv_freq.size(0) : 0);
    if (n < 0 || n > 0x7fffffff) return false;
    r->sections[a] = (int32_t)n;
  }
  // (a single section has to hold all frequencies too; the C ABI looks at sections from two axes on)
  if (axes == 1 && r->sections[0] != r->num_freqs) return false;
  r->section_order = order;
  r->pairing = pairing;
  r->positions_64bit = wide ? 1 : 0;
  return true;
}
// [T, H, D] rows on `dev` with neighbouring elements
bool rows_of(pal_rows* r, const at::Tensor& t, int64_t T, int64_t H, int64_t D, at::ScalarType type, const c10::Device& dev) {
  if (!t.is_cuda() || t.device() != dev || t.scalar_type() != type || t.dim() != 3 || t.size(0) != T || t.size(1) != H || t.size(2) != D ||
      (D > 1 && t.stride(2) != 1))
    return false;
  r->data = t.data_ptr();
  r->token_stride = t.stride(0);
  r->head_stride = t.stride(1);
  return true;
}

py::object rotary(const at::Tensor& x, const at::Tensor& positions, const at::Tensor& inv_freq, const c10::optional<std::vector<int64_t>>& sections,
                  int order, int pairing, double magnitude) {
  if (!x.is_cuda() || x.dim() != 3 || x.numel() == 0) return py::none();
  const c10::Device dev = x.device();
  const int code = dtype_code(x);
  const int64_t T = x.size(0), H = x.size(1), D = x.size(2);
  pal_rows src, dst;
  pal_rotation rot;
  if (code < 0 || !rows_of(&src, x, T, H, D, x.scalar_type(), dev) ||
      !rotation_of(&rot, positions, inv_freq, sections, order, pairing, magnitude, T, dev))
    return py::none();
  c10::cuda::CUDAGuard guard(dev);
  at::Tensor out = at::empty({T, H, D}, x.options());
  rows_of(&dst, out, T, H, D, x.scalar_type(), dev);
  raise_for(pal_rotary_embedding(&src, &dst, &rot, T, (int)H, (int)D, code, c10::cuda::getCurrentCUDAStream(dev.index()).stream()));
  return py::cast(out);
}

// Returns the rotated queries (True when there are none), or None when the call was not made.
py::object fill_rotary(const at::Tensor& new_k, const at::Tensor& new_v, const at::Tensor& k_pool, const at::Tensor& v_pool, const at::Tensor& a,
                       const c10::optional<at::Tensor>& pos, const c10::optional<at::Tensor>& seq_map, const c10::optional<at::Tensor>& positions,
                       const at::Tensor& inv_freq, const c10::optional<std::vector<int64_t>>& sections, int order, int pairing, double magnitude,
                       const c10::optional<at::Tensor>& queries) {
  if (!v_pool.is_cuda() || v_pool.dim() != 4 || k_pool.dim() != 5 || new_k.dim() != 3) return py::none();
  const c10::Device dev = v_pool.device();
  const int code = dtype_code(v_pool);
  const at::ScalarType type = v_pool.scalar_type();
  if (code < 0 || !dense_cuda(k_pool, dev) || !dense_cuda(v_pool, dev) || k_pool.scalar_type() != type) return py::none();
  const int64_t num_pages = v_pool.size(0), hkv = v_pool.size(1), d = v_pool.size(2), tpp = v_pool.size(3), T = new_k.size(0);
  if (T == 0 || num_pages == 0 || hkv == 0 || k_pool.size(0) != num_pages || k_pool.size(1) != hkv || k_pool.size(2) * 8 != d ||
      k_pool.size(3) != tpp || k_pool.size(4) != 8 || !dense_cuda(a, dev))
    return py::none();
  const bool slots = !pos.has_value();
  if (slots ? (seq_map.has_value() || a.scalar_type() != at::kLong || a.numel() != T || !positions.has_value())
            : (!seq_map.has_value() || a.dim() != 2 || !int32_like(a) || !dense_cuda(*pos, dev) || !dense_cuda(*seq_map, dev) || !int32_like(*pos) ||
               !int32_like(*seq_map) || pos->numel() != T || seq_map->numel() != T || (!positions.has_value() && (pos->dim() != 1 || pos->scalar_type() != at::kInt))))
    return py::none();
  pal_rows k, v, q, qo;
  pal_rotation rot;
  if (!rows_of(&k, new_k, T, hkv, d, type, dev) || !rows_of(&v, new_v, T, hkv, d, type, dev) ||
      !rotation_of(&rot, positions ? *positions : *pos, inv_freq, sections, order, pairing, magnitude, T, dev))
    return py::none();
  int64_t hq = 0;
  if (queries) {
    if (queries->dim() != 3) return py::none();
    hq = queries->size(1);
    if (!rows_of(&q, *queries, T, hq, d, type, dev)) return py::none();
  }
  c10::cuda::CUDAGuard guard(dev);
  at::Tensor out;
  if (queries) {
    out = at::empty({T, hq, d}, queries->options());
    rows_of(&qo, out, T, hq, d, type, dev);
  }
  raise_for(pal_fill_kv_pages_rotary(&k, &v, queries ? &q : nullptr, queries ? &qo : nullptr, k_pool.data_ptr(), v_pool.data_ptr(),
                                     slots ? static_cast<const int64_t*>(a.data_ptr()) : nullptr, slots || a.numel() == 0 ? nullptr : a.data_ptr(),
                                     slots ? nullptr : static_cast<const int32_t*>(pos->data_ptr()), slots ? nullptr : seq_map->data_ptr(), &rot, T,
                                     slots ? 0 : (int)a.size(0), (int)hq, (int)hkv, (int)d, (int)tpp, num_pages, slots ? 0 : (int)a.size(1), code,
                                     c10::cuda::getCurrentCUDAStream(dev.index()).stream()));
  return queries ? py::cast(out) : py::cast(true);
}

// ---- paged_attention_chunk -----------------------------------------------------------------
// `status_pages` is ops._STATUS_PAGES: {device index: tensor}.
py::object chunk(const at::Tensor& q, const at::Tensor& k_pool, const at::Tensor& v_pool, const at::Tensor& page_table, const at::Tensor& seq_lens,
                 const c10::optional<at::Tensor>& cu_seqlens, bool causal, int64_t window, double scale, bool out_f32,
                 const c10::optional<at::Tensor>& out_given, const py::dict& status_pages) {
  if (!q.is_cuda() || q.dim() != 3 || k_pool.dim() != 5 || v_pool.dim() != 4 || page_table.dim() != 2) return py::none();
  const c10::Device dev = q.device();
  const int code = dtype_code(q);
  if (code < 0 || !dense_cuda(k_pool, dev) || !dense_cuda(v_pool, dev) || !dense_cuda(page_table, dev) || !dense_cuda(seq_lens, dev) ||
      !int32_like(page_table) || !int32_like(seq_lens) || k_pool.scalar_type() != q.scalar_type() || v_pool.scalar_type() != q.scalar_type())
    return py::none();
  const int64_t num_pages = v_pool.size(0), hkv = v_pool.size(1), d = v_pool.size(2), tpp = v_pool.size(3);
  const int64_t S = page_table.size(0), mp = page_table.size(1), total = q.size(0), hq = q.size(1);
  if (S == 0 || mp == 0 || total == 0 || num_pages == 0 || hkv == 0 || hq == 0 || hq % hkv != 0 || q.size(2) != d || seq_lens.numel() != S ||
      k_pool.size(0) != num_pages || k_pool.size(1) != hkv || k_pool.size(2) * 8 != d || k_pool.size(3) != tpp || k_pool.size(4) != 8 || window < 0 ||
      window > 0x7fffffff)
    return py::none();
  if (cu_seqlens ? (!dense_cuda(*cu_seqlens, dev) || !int32_like(*cu_seqlens) || cu_seqlens->dim() != 1 || cu_seqlens->numel() != S + 1) : total % S != 0)
    return py::none();
  const int64_t st = q.stride(0), sh = q.stride(1);
  if (q.stride(2) != 1 || st % 8 != 0 || sh % 8 != 0 || st <= 0 || sh <= 0 || reinterpret_cast<uintptr_t>(q.data_ptr()) % 16 != 0) return py::none();
  const at::ScalarType otype = out_f32 ? at::kFloat : q.scalar_type();
  if (out_given && (!dense_cuda(*out_given, dev) || out_given->scalar_type() != otype || out_given->sizes() != q.sizes())) return py::none();
  PyObject* page = PyDict_GetItem(status_pages.ptr(), py::int_((int)dev.index()).ptr());  // borrowed
  if (!page || !THPVariable_Check(page)) return py::none();
  c10::cuda::CUDAGuard guard(dev);
  at::Tensor out = out_given ? *out_given : at::empty({total, hq, d}, q.options().dtype(otype));
  const size_t need = pal_chunk_scratch_bytes(total, (int)hq, (int)hkv, (int)d);
  at::Tensor scratch = at::empty({(int64_t)need}, q.options().dtype(at::kByte));
  raise_for(pal_paged_attention_chunk(q.data_ptr(), st, sh, k_pool.data_ptr(), v_pool.data_ptr(), page_table.data_ptr(),
                                      static_cast<const int32_t*>(seq_lens.data_ptr()),
                                      cu_seqlens ? static_cast<const int32_t*>(cu_seqlens->data_ptr()) : nullptr, out.data_ptr(), (int)S, total,
                                      (int)hq, (int)hkv, (int)d, (int)tpp, num_pages, (int)mp, (float)scale, causal ? 1 : 0, (int)window,
                                      code | (out_f32 ? PAL_OUT_F32 : 0), scratch.data_ptr(), need,
                                      static_cast<char*>(THPVariable_Unpack(page).data_ptr()) + 4,
                                      c10::cuda::getCurrentCUDAStream(dev.index()).stream()));
  return py::cast(out);
}

}  // namespace

PYBIND11_MODULE(_pal_fast, m) {
  m.doc() = "C++ fast path of the pal_b200 Python operators (argument checks and the C-ABI call without ctypes)";
  m.def("decode", &decode);
  m.def("prefill", &prefill);
  m.def("fill", &fill);
  m.def("rotary", &rotary);
  m.def("fill_rotary", &fill_rotary);
  m.def("chunk", &chunk);
}
