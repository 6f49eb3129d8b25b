// Tensor front end of the paged operators (hc_extend_pages, hc_release_pages,
// hc_append_paged, hc_prefix_attn; include/hotcold_hip.h) for the Python
// package: checks the tensors against each other, reads pointers and strides,
// allocates outputs and the call's workspace, and launches.  A serving step
// makes these calls once per layer and token, and marshalling their forty-odd
// fields from Python takes longer than the kernels of a short step.
//
// The workspace is allocated per call from torch's caching allocator on the
// current stream, so calls on two streams, and two captured graphs, never
// share one.
//
// Shapes and types are checked before devices, so that a refusal is the same
// on a machine without a GPU.
#include <torch/extension.h>

#include <initializer_list>
#include <tuple>

#include "hotcold_hip.h"

namespace {

using Opt = c10::optional<at::Tensor>;

void need_device(const char* what, std::initializer_list<const at::Tensor*> ts) {
  const at::Tensor* first = nullptr;
  for (const at::Tensor* t : ts) {
    if (!t) continue;
    TORCH_CHECK(t->is_cuda(), "hotcold_kv: the hot-tier kernels run on ROCm device tensors only (got a tensor on ",
                t->device(), ")");
    if (!first) first = t;
    TORCH_CHECK(t->device() == first->device(), what, ": tensors on ", first->device(), " and ", t->device());
  }
}

// A 1-D int32 tensor of n (or, n < 0, any number of) elements side by side.
int32_t* ints(const char* what, const char* name, const at::Tensor& t, int64_t n) {
  TORCH_CHECK(t.dim() == 1 && t.scalar_type() == at::kInt && (n < 0 ? t.size(0) >= 1 : t.size(0) == n) &&
                  t.is_contiguous(),
              what, ": ", name, " must be a contiguous int32 vector", n < 0 ? "" : " of ", n < 0 ? "" : std::to_string(n),
              "; got ", t.sizes(), " ", c10::toString(t.scalar_type()));
  return static_cast<int32_t*>(t.data_ptr());
}

void table(const char* what, const at::Tensor& t, int64_t B) {
  TORCH_CHECK(t.dim() == 2 && t.scalar_type() == at::kInt && t.size(0) == B && t.size(1) >= 1 && t.stride(1) == 1,
              what, ": tables must be (", B, ", pages) int32 with a unit last stride; got ", t.sizes(), " ",
              c10::toString(t.scalar_type()));
}

// A stride that is used only where its dimension has more than one entry.
int64_t step(const at::Tensor& t, int d) { return t.size(d) > 1 ? t.stride(d) : 0; }

int64_t row_stride(const at::Tensor& t, int64_t B) { return B > 1 ? t.stride(0) : t.size(1); }

int dtype_code(const char* what, at::ScalarType t) {
  switch (t) {
    case at::kFloat: return HC_DTYPE_F32;
    case at::kHalf: return HC_DTYPE_F16;
    case at::kBFloat16: return HC_DTYPE_BF16;
    default: break;
  }
  TORCH_CHECK_TYPE(false, what, ": unsupported dtype ", c10::toString(t));
  return -1;
}

// (rows, heads, D) of a (N,H,D) or (N,H,1,D) tensor, copied if its last
// dimension is strided.
at::Tensor rows3(const char* what, const char* name, const at::Tensor& t) {
  at::Tensor x = t;
  if (x.dim() == 4 && x.size(2) == 1) x = x.select(2, 0);
  TORCH_CHECK(x.dim() == 3, what, ": ", name, " must be (rows, heads, head_dim); got ", t.sizes());
  if (x.size(2) > 1 && x.stride(2) != 1) x = x.contiguous();
  return x;
}

// The pools [pages][H][P][D]; returns P.
int64_t pools(const char* what, const at::Tensor& k, const at::Tensor& v, int64_t H, int64_t D, at::ScalarType st) {
  TORCH_CHECK(k.dim() == 4 && k.sizes() == v.sizes() && k.size(0) >= 1 && k.size(1) == H && k.size(2) >= 1 &&
                  k.size(3) == D && k.scalar_type() == st && v.scalar_type() == st && k.stride(3) == 1 &&
                  v.stride(3) == 1,
              what, ": k_pages, v_pages must be (pages, ", H, ", page_size, ", D, ") ", c10::toString(st),
              " with a unit last stride; got ", k.sizes(), " ", c10::toString(k.scalar_type()), " and ", v.sizes(), " ",
              c10::toString(v.scalar_type()));
  return k.size(2);
}

// n contiguous elements of type t from byte `from` of base's storage: an
// output of a call that makes several, from one allocation (each at::empty and
// each view through the dispatcher takes about a microsecond of the host: a
// step's extend_pages took 8.8 us there, of a GPU time of 3, and takes 7.0).
at::Tensor part(const at::Tensor& base, at::ScalarType t, int64_t from, int64_t n) {
  at::Tensor x = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(base.storage()), base.key_set(),
                                                          c10::scalarTypeToTypeMeta(t));
  c10::TensorImpl* impl = x.unsafeGetTensorImpl();
  impl->set_storage_offset(from / (int64_t)c10::elementSize(t));
  impl->set_sizes_contiguous({n});
  return x;
}

at::Tensor room(const at::Tensor& like, int64_t bytes) {
  return at::empty({bytes}, like.options().dtype(at::kByte));
}
int64_t up16(int64_t n) { return (n + 15) & ~(int64_t)15; }

}  // namespace

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, int64_t> extend_pages(
    const at::Tensor& lens, const at::Tensor& new_lens, const at::Tensor& tables, const at::Tensor& free_pages,
    const at::Tensor& free_count, int64_t page_size, int64_t num_tokens, const Opt& lens_out, const Opt& count_out,
    int64_t stream) {
  const char* what = "extend_pages";
  ints(what, "lens", lens, -1);
  const int64_t B = lens.size(0);
  ints(what, "new_lens", new_lens, B);
  table(what, tables, B);
  ints(what, "free_pages", free_pages, -1);
  ints(what, "free_count", free_count, 1);
  TORCH_CHECK(num_tokens >= 0, what, ": num_tokens ", num_tokens);
  if (lens_out.has_value()) ints(what, "lens_out", *lens_out, B);
  if (count_out.has_value()) ints(what, "count_out", *count_out, 1);
  need_device(what, {&lens, &new_lens, &tables, &free_pages, &free_count, lens_out.has_value() ? &*lens_out : nullptr,
                     count_out.has_value() ? &*count_out : nullptr});
  const c10::DeviceGuard guard(lens.device());
  const int64_t at_pos = up16(8 * num_tokens), at_cu = 2 * at_pos, at_lens = at_cu + up16(4 * (B + 1)),
                at_count = at_lens + up16(4 * B);
  const at::Tensor base = room(lens, at_count + 4);
  at::Tensor slots = part(base, at::kLong, 0, num_tokens), pos = part(base, at::kLong, at_pos, num_tokens),
             cu = part(base, at::kInt, at_cu, B + 1);
  at::Tensor lo = lens_out.has_value() ? *lens_out : part(base, at::kInt, at_lens, B),
             co = count_out.has_value() ? *count_out : part(base, at::kInt, at_count, 1);
  const int rc = hc_extend_pages(B, lens.data_ptr<int32_t>(), new_lens.data_ptr<int32_t>(), tables.data_ptr<int32_t>(),
                                 row_stride(tables, B), tables.size(1), free_pages.data_ptr<int32_t>(),
                                 free_pages.size(0), free_count.data_ptr<int32_t>(), page_size, num_tokens,
                                 lo.data_ptr<int32_t>(), co.data_ptr<int32_t>(), cu.data_ptr<int32_t>(),
                                 slots.data_ptr<int64_t>(), pos.data_ptr<int64_t>(), reinterpret_cast<void*>(stream));
  return {lo, co, cu, slots, pos, rc};
}

std::tuple<at::Tensor, at::Tensor, int64_t> release_pages(const at::Tensor& lens, const at::Tensor& keep_lens,
                                                          const at::Tensor& tables, const at::Tensor& free_pages,
                                                          const at::Tensor& free_count, int64_t page_size,
                                                          const Opt& lens_out, const Opt& count_out, int64_t stream) {
  const char* what = "release_pages";
  ints(what, "lens", lens, -1);
  const int64_t B = lens.size(0);
  ints(what, "keep_lens", keep_lens, B);
  table(what, tables, B);
  ints(what, "free_pages", free_pages, -1);
  ints(what, "free_count", free_count, 1);
  if (lens_out.has_value()) ints(what, "lens_out", *lens_out, B);
  if (count_out.has_value()) ints(what, "count_out", *count_out, 1);
  need_device(what, {&lens, &keep_lens, &tables, &free_pages, &free_count, lens_out.has_value() ? &*lens_out : nullptr,
                     count_out.has_value() ? &*count_out : nullptr});
  const c10::DeviceGuard guard(lens.device());
  at::Tensor base, lo, co;
  const int64_t at_count = up16(4 * B);
  if (!lens_out.has_value() || !count_out.has_value()) base = room(lens, at_count + 4);
  lo = lens_out.has_value() ? *lens_out : part(base, at::kInt, 0, B);
  co = count_out.has_value() ? *count_out : part(base, at::kInt, at_count, 1);
  const int rc = hc_release_pages(B, lens.data_ptr<int32_t>(), keep_lens.data_ptr<int32_t>(), tables.data_ptr<int32_t>(),
                                  row_stride(tables, B), tables.size(1), free_pages.data_ptr<int32_t>(),
                                  free_pages.size(0), free_count.data_ptr<int32_t>(), page_size, lo.data_ptr<int32_t>(),
                                  co.data_ptr<int32_t>(), reinterpret_cast<void*>(stream));
  return {lo, co, rc};
}

int64_t append_paged(const at::Tensor& slots, const at::Tensor& k_new, const at::Tensor& v_new,
                     const at::Tensor& k_pages, const at::Tensor& v_pages, int64_t stream) {
  const char* what = "append_paged";
  const at::Tensor k = rows3(what, "k_new", k_new), v = rows3(what, "v_new", v_new);
  const int64_t N = k.size(0), H = k.size(1), D = k.size(2);
  const int code = dtype_code(what, k.scalar_type());
  TORCH_CHECK(v.sizes() == k.sizes() && v.scalar_type() == k.scalar_type(), what, ": k_new ", k_new.sizes(), " ",
              c10::toString(k.scalar_type()), " and v_new ", v_new.sizes(), " ", c10::toString(v.scalar_type()),
              " must match");
  TORCH_CHECK(slots.dim() == 1 && slots.size(0) == N && slots.scalar_type() == at::kLong && slots.is_contiguous(), what,
              ": slots must be a contiguous int64 vector of ", N, "; got ", slots.sizes(), " ",
              c10::toString(slots.scalar_type()));
  const int64_t P = pools(what, k_pages, v_pages, H, D, k.scalar_type());
  need_device(what, {&k, &v, &slots, &k_pages, &v_pages});
  const c10::DeviceGuard guard(k.device());
  return hc_append_paged(code, N, H, D, slots.data_ptr<int64_t>(), k.data_ptr(), step(k, 0), step(k, 1), v.data_ptr(),
                         step(v, 0), step(v, 1), k_pages.data_ptr(), step(k_pages, 0), step(k_pages, 1),
                         step(k_pages, 2), v_pages.data_ptr(), step(v_pages, 0), step(v_pages, 1), step(v_pages, 2),
                         k_pages.size(0), P, reinterpret_cast<void*>(stream));
}

std::tuple<at::Tensor, Opt, int64_t> prefix_attention(const at::Tensor& q_in, const Opt& k_prefix, const Opt& v_prefix,
                                                      const at::Tensor& k_pages, const at::Tensor& v_pages,
                                                      const at::Tensor& tables, const at::Tensor& lens, double scaling,
                                                      const Opt& cu_new, const c10::optional<int64_t>& max_new,
                                                      const Opt& prefix_lens, const Opt& out_in, bool with_lse,
                                                      int64_t stream) {
  const char* what = "prefix_attention";
  const at::Tensor q = rows3(what, "q", q_in);
  const at::ScalarType st = q.scalar_type();
  hc_prefix_attn_args a{};
  a.dtype = dtype_code(what, st);
  a.N = q.size(0);
  a.Hq = q.size(1);
  a.D = q.size(2);
  ints(what, "lens", lens, -1);
  a.B = lens.size(0);
  TORCH_CHECK(k_pages.dim() == 4, what, ": k_pages must be (pages, Hk, page_size, D); got ", k_pages.sizes());
  a.Hk = k_pages.size(1);
  a.page_size = pools(what, k_pages, v_pages, a.Hk, a.D, st);
  a.num_pages = k_pages.size(0);
  table(what, tables, a.B);
  TORCH_CHECK(k_prefix.has_value() == v_prefix.has_value(), what, ": k_prefix and v_prefix go together");
  at::Tensor kp, vp;
  if (k_prefix.has_value()) {
    kp = k_prefix->dim() == 4 && k_prefix->size(0) == 1 ? k_prefix->select(0, 0) : *k_prefix;
    vp = v_prefix->dim() == 4 && v_prefix->size(0) == 1 ? v_prefix->select(0, 0) : *v_prefix;
    TORCH_CHECK(kp.dim() == 3 && kp.sizes() == vp.sizes() && kp.size(0) == a.Hk && kp.size(2) == a.D &&
                    kp.scalar_type() == st && vp.scalar_type() == st &&
                    (kp.size(1) == 0 || (kp.stride(2) == 1 && vp.stride(2) == 1)),
                what, ": k_prefix, v_prefix must be (1, ", a.Hk, ", rows, ", a.D, ") or (", a.Hk, ", rows, ", a.D, ") ",
                c10::toString(st), " with a unit last stride; got ", k_prefix->sizes(), " ",
                c10::toString(kp.scalar_type()), " and ", v_prefix->sizes(), " ", c10::toString(vp.scalar_type()));
    a.prefix_rows = kp.size(1);
  }
  if (prefix_lens.has_value()) a.prefix_lens = ints(what, "prefix_lens", *prefix_lens, a.B);
  if (cu_new.has_value()) {
    a.cu_new = ints(what, "cu_new", *cu_new, a.B + 1);
    TORCH_CHECK(max_new.has_value(), what, ": cu_new needs max_new, an upper bound on a request's tokens");
    a.max_new = *max_new;
  } else {
    TORCH_CHECK(a.N == a.B && max_new.value_or(1) == 1, what, ": without cu_new every request has one token; got ", a.N,
                " tokens, ", a.B, " requests, max_new ", max_new.value_or(1));
    a.max_new = 1;
  }
  if (out_in.has_value())
    TORCH_CHECK(out_in->dim() == 3 && out_in->sizes() == q.sizes() && out_in->scalar_type() == st &&
                    out_in->stride(2) == 1,
                what, ": out must be ", q.sizes(), " ", c10::toString(st), " with a unit last stride; got ",
                out_in->sizes(), " ", c10::toString(out_in->scalar_type()));
  need_device(what, {&q, &k_pages, &v_pages, &tables, &lens, kp.defined() ? &kp : nullptr, vp.defined() ? &vp : nullptr,
                     cu_new.has_value() ? &*cu_new : nullptr, prefix_lens.has_value() ? &*prefix_lens : nullptr,
                     out_in.has_value() ? &*out_in : nullptr});
  const c10::DeviceGuard guard(q.device());
  at::Tensor out = out_in.has_value() ? *out_in : at::empty({a.N, a.Hq, a.D}, q.options());
  Opt lse;
  if (with_lse) {
    lse = at::empty({a.N, a.Hq}, q.options().dtype(at::kFloat));
    a.lse = lse->data_ptr<float>();
    a.l_sn = a.Hq;
    a.l_sh = 1;
  }
  a.q = q.data_ptr(); a.q_sn = step(q, 0); a.q_sh = step(q, 1);
  if (kp.defined() && a.prefix_rows > 0) {
    a.k_prefix = kp.data_ptr(); a.kp_sh = step(kp, 0); a.kp_ss = step(kp, 1);
    a.v_prefix = vp.data_ptr(); a.vp_sh = step(vp, 0); a.vp_ss = step(vp, 1);
  }
  a.k_pages = k_pages.data_ptr(); a.kg_sp = step(k_pages, 0); a.kg_sh = step(k_pages, 1); a.kg_ss = step(k_pages, 2);
  a.v_pages = v_pages.data_ptr(); a.vg_sp = step(v_pages, 0); a.vg_sh = step(v_pages, 1); a.vg_ss = step(v_pages, 2);
  a.tables = tables.data_ptr<int32_t>(); a.t_sb = row_stride(tables, a.B); a.table_width = tables.size(1);
  a.lens = lens.data_ptr<int32_t>();
  a.scaling = scaling;
  a.out = out.data_ptr(); a.o_sn = step(out, 0); a.o_sh = step(out, 1);
  const int64_t bytes = hc_prefix_attn_workspace_size(&a);
  at::Tensor ws;
  if (bytes > 0) {
    ws = at::empty({bytes}, q.options().dtype(at::kByte));
    a.workspace = ws.data_ptr();
    a.workspace_bytes = bytes;
  }
  const int rc = hc_prefix_attn(&a, reinterpret_cast<void*>(stream));
  return {out, lse, rc};
}
