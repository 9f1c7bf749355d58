// The torch ops for one new token a row (basal::paged_attention, kv_append, kv_copy_pages, gdn_step, constrain_logits):
// their schemas, the checks of their tensors, and the calls of libbasal200's C ABI. Their kernels run for a few
// microseconds at the sizes of a decoding step, where a call through torch.library and ctypes takes 25 to 32 us of host
// time and one from here 5 to 10, so these ops are registered in C++ (libbasal200_torch-<torch version>.so, loaded by ops.py;
// their documentation is there).
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/autograd_not_implemented_fallback.h>
#include <torch/library.h>

#include <vector>

#include "../../include/basal200.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

const Tensor* get(const OptTensor& t) { return t.has_value() && t->defined() ? &*t : nullptr; }

void need_cuda(const Tensor& t) {
  TORCH_CHECK_VALUE(t.is_cuda(), "basal_b200 computes on CUDA tensors only (sm_100a); the CPU maths of the reference is "
                                 "not part of this package");
}

void on(const Tensor& t, c10::Device dev) {
  need_cuda(t);
  TORCH_CHECK_VALUE(t.device() == dev, "basal_b200: a tensor is on ", t.device(), ", another on ", dev);
}
void on(const OptTensor& t, c10::Device dev) {
  if (get(t)) on(*t, dev);
}

int code(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return BASAL200_BF16;
    case at::kHalf: return BASAL200_F16;
    case at::kFloat: return BASAL200_F32;
    default: TORCH_CHECK_VALUE(false, "basal_b200: dtype ", t.scalar_type(), " is not supported (bfloat16, float16, float32)");
  }
}

// t is int32 of these sizes (-1: any)
void need_int32(const char* what, const Tensor& t, at::IntArrayRef shape) {
  bool ok = t.scalar_type() == at::kInt && t.dim() == (int64_t)shape.size();
  for (size_t i = 0; ok && i < shape.size(); ++i) ok = shape[i] < 0 || t.size(i) == shape[i];
  TORCH_CHECK_VALUE(ok, what, " must be int32 ", shape, " (-1: any), not ", t.scalar_type(), " ", t.sizes());
}

int to_int(const char* what, int64_t v) {
  TORCH_CHECK_VALUE(v >= INT32_MIN && v <= INT32_MAX, what, ": ", v, " is out of range");
  return (int)v;
}

void done(const char* name, int rc) {
  if (rc == BASAL200_OK) return;
  const bool value = rc == BASAL200_ERR_ARG || rc == BASAL200_ERR_SHAPE || rc == BASAL200_ERR_ALIGN ||
                     rc == BASAL200_ERR_DTYPE || rc == BASAL200_ERR_LIMIT;
  TORCH_CHECK_VALUE(!value, name, ": ", basal200_status_string(rc), " (status ", rc, ")");
  TORCH_CHECK(false, name, ": ", basal200_status_string(rc), " (status ", rc, ")");
}

void* ptr(const Tensor& t) { return t.data_ptr(); }

// A tensor that the call writes: its version counter says so, as after any torch op that writes its argument.
void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
void written(const OptTensor& t) {
  if (get(t)) written(*t);
}
template <typename T>
T* ptr_or_null(const OptTensor& t) {
  return get(t) ? static_cast<T*>(t->data_ptr()) : nullptr;
}

// t contiguous, of type s (a to() that changes nothing still costs a trip through the dispatcher)
Tensor as(const Tensor& t, at::ScalarType s) { return t.scalar_type() == s ? t.contiguous() : t.to(s).contiguous(); }

bool aligned(const Tensor& t, uintptr_t bytes) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % bytes == 0; }

// A copy of t in memory of its own, contiguous and aligned (contiguous() hands back a view that is contiguous where it
// lies: at an odd offset, or one row with any row stride).
Tensor copied(const Tensor& t) { return t.clone(at::MemoryFormat::Contiguous); }

// A cache's pages, scales and table, checked.
struct Cache {
  int64_t pages, page, head, token, s_page = 0, s_head = 0, table_row;
  int Hk, page_size, D, dtype, width;
  float *ks = nullptr, *vs = nullptr;
  const int32_t* table;
};

Cache cache_of(const char* what, const Tensor& k, const Tensor& v, const OptTensor& ks, const OptTensor& vs,
               const Tensor& table, int64_t rows, at::ScalarType dtype) {
  TORCH_CHECK_VALUE(k.dim() == 4 && k.sizes() == v.sizes() && k.strides() == v.strides() &&
                        k.scalar_type() == v.scalar_type(),
                    what, ": the key and value pages must be [pages, kv heads, page size, D] alike, not ", k.sizes(), " ",
                    k.scalar_type(), " and ", v.sizes(), " ", v.scalar_type());
  TORCH_CHECK_VALUE(k.stride(3) == 1 || k.numel() == 0, what, ": the pages' last dimension must be contiguous");
  const bool fp8 = k.scalar_type() == at::kFloat8_e4m3fn;
  TORCH_CHECK_VALUE(fp8 || k.scalar_type() == dtype, what, ": pages of ", k.scalar_type(), " with tokens of ", dtype);
  Cache c;
  c.pages = k.size(0);
  c.Hk = to_int(what, k.size(1));
  c.page_size = to_int(what, k.size(2));
  c.D = to_int(what, k.size(3));
  c.page = k.stride(0);
  c.head = k.stride(1);
  c.token = k.stride(2);
  c.dtype = fp8 ? BASAL200_E4M3 : code(k);
  if (fp8) {
    const Tensor *a = get(ks), *b = get(vs);
    TORCH_CHECK_VALUE(a && b && a->sizes() == k.sizes().slice(0, 3) && b->sizes() == a->sizes() &&
                          a->strides() == b->strides() && a->scalar_type() == at::kFloat &&
                          b->scalar_type() == at::kFloat && (c.page_size < 2 || a->stride(2) == 1),
                      what, ": 8-bit pages need fp32 scales k_scale, v_scale [", c.pages, ", ", c.Hk, ", ", c.page_size, "]");
    c.s_page = a->stride(0);
    c.s_head = a->stride(1);
    c.ks = static_cast<float*>(a->data_ptr());
    c.vs = static_cast<float*>(b->data_ptr());
  } else {
    TORCH_CHECK_VALUE(!get(ks) && !get(vs), what, ": scales are for 8-bit pages");
  }
  need_int32("the table", table, {rows, -1});
  TORCH_CHECK_VALUE(table.size(1) < 2 || table.stride(1) == 1, what, ": a table's rows must be contiguous");
  c.table = static_cast<const int32_t*>(table.data_ptr());
  c.table_row = table.stride(0);
  c.width = to_int(what, table.size(1));
  return c;
}

Tensor paged_attention(const Tensor& q_in, const Tensor& k, const Tensor& v, const Tensor& table, const Tensor& lengths_in,
                       double scale, int64_t window, const OptTensor& ks, const OptTensor& vs) {
  const char* what = "paged_attention";
  need_cuda(q_in);
  const c10::Device dev = q_in.device();
  on(k, dev), on(v, dev), on(table, dev), on(lengths_in, dev), on(ks, dev), on(vs, dev);
  TORCH_CHECK_VALUE(q_in.dim() == 3, what, ": q must be [rows, heads, D], not ", q_in.sizes());
  const int64_t rows = q_in.size(0), H = q_in.size(1), D = q_in.size(2);
  const Cache c = cache_of(what, k, v, ks, vs, table, rows, q_in.scalar_type());
  TORCH_CHECK_VALUE(D == c.D && H > 0 && c.Hk > 0 && H % c.Hk == 0, what, ": ", H, " heads of ", D, " over pages of ", c.Hk,
                    " heads of ", c.D);
  need_int32("lengths", lengths_in, {rows});
  const bool fits = q_in.stride(2) == 1 && q_in.stride(0) % 8 == 0 && q_in.stride(1) % 8 == 0 && aligned(q_in, 16);
  const Tensor q = fits ? q_in : copied(q_in), lengths = lengths_in.contiguous();
  const c10::cuda::CUDAGuard guard(dev);
  Tensor out = at::empty({rows, H, D}, q.options());
  const int r = to_int(what, rows), h = to_int(what, H), w = to_int(what, window);
  const int64_t n = basal200_paged_attention_workspace_bytes(r, h, c.Hk, c.D, c.dtype, c.width, c.page_size, w);
  Tensor work;
  if (n > 0) work = at::empty({n}, q.options().dtype(at::kByte));
  done(what, basal200_paged_attention(ptr(q), code(q), q.stride(0), q.stride(1), ptr(k), ptr(v), c.dtype, c.page, c.head,
                                      c.token, c.ks, c.vs, c.s_page, c.s_head, c.pages, c.page_size, c.table, c.table_row,
                                      c.width, static_cast<const int32_t*>(ptr(lengths)), r, h, c.Hk, c.D, (float)scale, w,
                                      ptr(out), n > 0 ? ptr(work) : nullptr, n,
                                      c10::cuda::getCurrentCUDAStream(dev.index()).stream()));
  return out;
}

void kv_append(const Tensor& k_in, const Tensor& v_in, const Tensor& k_pages, const Tensor& v_pages, const Tensor& table,
               const Tensor& start_in, const OptTensor& count_in, const OptTensor& ks, const OptTensor& vs) {
  const char* what = "kv_append";
  need_cuda(k_in);
  const c10::Device dev = k_in.device();
  on(v_in, dev), on(k_pages, dev), on(v_pages, dev), on(table, dev), on(start_in, dev), on(count_in, dev), on(ks, dev),
      on(vs, dev);
  TORCH_CHECK_VALUE(k_in.dim() == 4 && k_in.sizes() == v_in.sizes() && k_in.scalar_type() == v_in.scalar_type(), what,
                    ": k and v must be [rows, tokens, kv heads, D] alike, not ", k_in.sizes(), " and ", v_in.sizes());
  const int64_t rows = k_in.size(0), T = k_in.size(1);
  const Cache c = cache_of(what, k_pages, v_pages, ks, vs, table, rows, k_in.scalar_type());
  TORCH_CHECK_VALUE(k_in.size(2) == c.Hk && k_in.size(3) == c.D, what, ": tokens of ", k_in.size(2), " heads of ",
                    k_in.size(3), " into pages of ", c.Hk, " heads of ", c.D);
  need_int32("start", start_in, {rows});
  Tensor count;
  if (get(count_in)) {
    need_int32("count", *count_in, {rows});
    count = count_in->contiguous();
  }
  auto fit = [](const Tensor& x) {
    return x.stride(3) == 1 && (x.stride(0) | x.stride(1) | x.stride(2)) % 8 == 0 && aligned(x, 16) ? x : copied(x);
  };
  const Tensor k = fit(k_in), v = fit(v_in), start = start_in.contiguous();
  const c10::cuda::CUDAGuard guard(dev);
  done(what, basal200_kv_append(ptr(k), ptr(v), code(k), k.stride(0), k.stride(1), k.stride(2), v.stride(0), v.stride(1),
                                v.stride(2), ptr(k_pages), ptr(v_pages), c.dtype, c.page, c.head, c.token, c.ks, c.vs,
                                c.s_page, c.s_head, c.pages, c.page_size, c.table, c.table_row, c.width,
                                static_cast<const int32_t*>(ptr(start)),
                                count.defined() ? static_cast<const int32_t*>(ptr(count)) : nullptr, to_int(what, rows),
                                to_int(what, T), c.Hk, c.D, c10::cuda::getCurrentCUDAStream(dev.index()).stream()));
  written(k_pages), written(v_pages), written(ks), written(vs);
}

void kv_copy_pages(at::TensorList pools, at::IntArrayRef src, at::IntArrayRef dst) {
  const char* what = "kv_copy_pages";
  TORCH_CHECK_VALUE(src.size() == dst.size(), what, ": ", src.size(), " pages to read, ", dst.size(), " to write");
  for (const Tensor& p : pools) need_cuda(p);
  const c10::Device dev = pools[0].device();
  const int64_t N = pools[0].dim() > 1 ? pools[0].size(1) : -1;
  TORCH_CHECK_VALUE(pools.size() <= 8, what, ": at most 8 pools, not ", pools.size());
  void* base[8];
  int layers[8];
  int64_t bytes[8];
  int held = 0;  // pools that hold anything
  for (const Tensor& p : pools) {
    on(p, dev);
    TORCH_CHECK_VALUE(p.dim() >= 3 && p.size(1) == N && p.is_contiguous(), what,
                      ": the pools must be contiguous [layers, pages, ...] of equally many pages");
    if (p.numel() == 0) continue;
    base[held] = ptr(p);
    layers[held] = to_int(what, p.size(0));
    bytes[held++] = p.stride(1) * p.element_size();
  }
  std::vector<int32_t> moves(src.size() * 2);
  for (size_t i = 0; i < src.size(); ++i) {
    TORCH_CHECK_VALUE(src[i] >= 0 && src[i] < N && dst[i] >= 0 && dst[i] < N && N <= INT32_MAX, what,
                      ": a page is outside [0, ", N, ")");
    moves[i] = (int32_t)src[i];
    moves[src.size() + i] = (int32_t)dst[i];
  }
  if (!held || src.empty()) return;
  const c10::cuda::CUDAGuard guard(dev);
  done(what, basal200_kv_copy_pages(base, layers, bytes, held, N, moves.data(), moves.data() + src.size(),
                                    to_int(what, (int64_t)src.size()),
                                    c10::cuda::getCurrentCUDAStream(dev.index()).stream()));
  for (const Tensor& p : pools) written(p);
}

Tensor gdn_step(const Tensor& proj_in, const Tensor& tail, const Tensor& conv_in, const Tensor& A_log_in,
                const Tensor& dt_bias_in, const Tensor& state, int64_t Hk, int64_t Hv, int64_t b_off, int64_t a_off,
                const OptTensor& slots_in) {
  const char* what = "gdn_step";
  need_cuda(proj_in);
  const c10::Device dev = proj_in.device();
  on(tail, dev), on(conv_in, dev), on(A_log_in, dev), on(dt_bias_in, dev), on(state, dev), on(slots_in, dev);
  const at::ScalarType dt = proj_in.scalar_type();
  TORCH_CHECK_VALUE(proj_in.dim() == 2 && Hk > 0 && Hv > 0 && Hv < (1 << 20) && Hv % Hk == 0, what,
                    ": proj must be [rows, width], Hv a multiple of Hk, not ", proj_in.sizes(), ", ", Hv, ", ", Hk);
  const int64_t rows = proj_in.size(0), width = proj_in.size(1), C = (2 * Hk + Hv) * 128;
  TORCH_CHECK_VALUE(state.dim() == 4 && state.size(1) == Hv && state.size(2) == 128 && state.size(3) == 128 &&
                        state.scalar_type() == at::kFloat && state.is_contiguous(),
                    what, ": the state must be contiguous fp32 [slots, ", Hv, ", 128, 128]");
  const int64_t slots = state.size(0);
  TORCH_CHECK_VALUE(tail.dim() == 3 && tail.size(0) == slots && tail.size(1) == 3 && tail.size(2) == C &&
                        tail.scalar_type() == dt && tail.is_contiguous(),
                    what, ": the tail must be contiguous ", dt, " [", slots, ", 3, ", C, "]");
  TORCH_CHECK_VALUE(conv_in.sizes() == at::IntArrayRef({C, 4}) && A_log_in.sizes() == at::IntArrayRef({Hv}) &&
                        dt_bias_in.sizes() == at::IntArrayRef({Hv}),
                    what, ": conv must be [", C, ", 4], A_log and dt_bias [", Hv, "]");
  TORCH_CHECK_VALUE(b_off >= 0 && a_off >= 0 && C <= width && b_off + Hv <= width && a_off + Hv <= width, what,
                    ": the projection has ", width, " columns");
  Tensor at_slot;
  if (get(slots_in)) {
    need_int32("slots", *slots_in, {rows});
    at_slot = slots_in->contiguous();
  } else {
    TORCH_CHECK_VALUE(rows <= slots, what, ": ", rows, " rows, ", slots, " states");
  }
  const c10::cuda::CUDAGuard guard(dev);
  Tensor proj = proj_in;
  const bool fits = proj.stride(1) == 1 && proj.stride(0) % 4 == 0 && (rows < 2 || proj.stride(0) >= width) && aligned(proj, 8);
  if (rows > 0 && !fits) {  // rows at multiples of 16 bytes, one after another
    proj = at::empty({rows, (width + 7) / 8 * 8}, proj_in.options()).narrow(1, 0, width);
    proj.copy_(proj_in);
  }
  Tensor conv = as(conv_in, dt);
  if (!aligned(conv, 16)) conv = copied(conv);
  const Tensor A_log = as(A_log_in, at::kFloat), dt_bias = as(dt_bias_in, dt);
  Tensor o = at::empty({rows, Hv, 1, 128}, proj_in.options());
  done(what, basal200_gdn_step(ptr(proj), code(proj), rows > 1 ? proj.stride(0) : (width + 3) / 4 * 4, ptr(tail), ptr(conv),
                               static_cast<const float*>(ptr(A_log)), ptr(dt_bias), (int)b_off, (int)a_off,
                               static_cast<float*>(ptr(state)),
                               at_slot.defined() ? static_cast<const int32_t*>(ptr(at_slot)) : nullptr, slots,
                               to_int(what, rows), (int)Hk, (int)Hv, ptr(o),
                               c10::cuda::getCurrentCUDAStream(dev.index()).stream()));
  written(tail), written(state);
  return o;
}

Tensor constrain_logits(const Tensor& logits_in, const OptTensor& mask_in, const OptTensor& past_in,
                        const OptTensor& repetition, const OptTensor& presence, const OptTensor& frequency,
                        const OptTensor& ids_in, const OptTensor& values_in) {
  const char* what = "constrain_logits";
  need_cuda(logits_in);
  const c10::Device dev = logits_in.device();
  on(mask_in, dev), on(past_in, dev), on(repetition, dev), on(presence, dev), on(frequency, dev), on(ids_in, dev),
      on(values_in, dev);
  TORCH_CHECK_VALUE(logits_in.dim() == 2, what, ": logits must be [rows, vocabulary], not ", logits_in.sizes());
  const int64_t rows = logits_in.size(0), V = logits_in.size(1);
  const Tensor logits = logits_in.stride(1) == 1 || V < 2 ? logits_in : logits_in.contiguous();
  Tensor per_row[3];
  const float* rowwise[3] = {nullptr, nullptr, nullptr};
  const OptTensor* given[3] = {&repetition, &presence, &frequency};
  for (int i = 0; i < 3; ++i) {
    if (!get(*given[i])) continue;
    const Tensor& t = **given[i];
    TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == rows && t.scalar_type() == at::kFloat, what,
                      ": repetition, presence and frequency must be fp32 [", rows, "], not ", t.scalar_type(), " ", t.sizes());
    TORCH_CHECK_VALUE(get(past_in), what, ": penalties need the rows' history (past)");
    per_row[i] = t.contiguous();
    rowwise[i] = static_cast<const float*>(ptr(per_row[i]));
  }
  TORCH_CHECK_VALUE(!get(ids_in) == !get(values_in), what, ": bias_ids and bias_values come together");
  Tensor mask, past, ids, values;
  int64_t mrow = 0, T = 0, N = 0;
  if (get(mask_in)) {
    need_int32("the mask", *mask_in, {-1, (V + 31) / 32});
    TORCH_CHECK_VALUE(mask_in->size(0) == 1 || mask_in->size(0) == rows, what, ": a mask of ", mask_in->size(0), " rows for ",
                      rows);
    mask = mask_in->contiguous();
    mrow = mask.size(0) == rows ? mask.size(1) : 0;
  }
  if (get(past_in)) {
    need_int32("past", *past_in, {rows, -1});
    past = past_in->contiguous();
    T = past.size(1);
  }
  if (get(ids_in)) {
    need_int32("bias_ids", *ids_in, {rows, -1});
    TORCH_CHECK_VALUE(values_in->sizes() == ids_in->sizes() && values_in->scalar_type() == at::kFloat, what,
                      ": bias_values must be fp32 ", ids_in->sizes());
    ids = ids_in->contiguous();
    values = values_in->contiguous();
    N = ids.size(1);
  }
  const c10::cuda::CUDAGuard guard(dev);
  Tensor out = at::empty({rows, V}, logits.options().dtype(at::kFloat));
  done(what, basal200_constrain_logits(
                 ptr(logits), code(logits), rows > 1 ? logits.stride(0) : V, to_int(what, rows), to_int(what, V),
                 mask.defined() ? static_cast<const uint32_t*>(ptr(mask)) : nullptr, mrow,
                 past.defined() ? static_cast<const int32_t*>(ptr(past)) : nullptr, T, to_int(what, T), rowwise[0],
                 rowwise[1], rowwise[2], ids.defined() ? static_cast<const int32_t*>(ptr(ids)) : nullptr,
                 values.defined() ? static_cast<const float*>(ptr(values)) : nullptr, N, to_int(what, N),
                 static_cast<float*>(ptr(out)), c10::cuda::getCurrentCUDAStream(dev.index()).stream()));
  return out;
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(basal, m) {
  m.def("paged_attention(Tensor q, Tensor k_pages, Tensor v_pages, Tensor table, Tensor lengths, float scale, int window=0, "
        "Tensor? k_scale=None, Tensor? v_scale=None) -> Tensor");
  m.def("kv_append(Tensor k, Tensor v, Tensor(a!) k_pages, Tensor(b!) v_pages, Tensor table, Tensor start, Tensor? "
        "count=None, Tensor(c!)? k_scale=None, Tensor(d!)? v_scale=None) -> ()");
  m.def("kv_copy_pages(Tensor(a!)[] pools, int[] src, int[] dst) -> ()");
  m.def("gdn_step(Tensor proj, Tensor(a!) tail, Tensor conv, Tensor A_log, Tensor dt_bias, Tensor(b!) state, int Hk, int Hv, "
        "int b_off, int a_off, Tensor? slots=None) -> Tensor");
  m.def("constrain_logits(Tensor logits, Tensor? mask=None, Tensor? past=None, Tensor? repetition=None, Tensor? "
        "presence=None, Tensor? frequency=None, Tensor? bias_ids=None, Tensor? bias_values=None) -> Tensor");
}

#define BASAL_STEP_OPS(m)                    \
  m.impl("paged_attention", paged_attention); \
  m.impl("kv_append", kv_append);             \
  m.impl("kv_copy_pages", kv_copy_pages);     \
  m.impl("gdn_step", gdn_step);               \
  m.impl("constrain_logits", constrain_logits)

TORCH_LIBRARY_IMPL(basal, CUDA, m) { BASAL_STEP_OPS(m); }
TORCH_LIBRARY_IMPL(basal, CPU, m) { BASAL_STEP_OPS(m); }  // for the refusal: there is no CPU implementation

// No gradients, as the package's other ops: a backward pass through an output raises (torch's default for an op from C++ is a
// warning, and no gradient).
#define BASAL_NO_GRADIENT(m, op) m.impl(op, torch::autograd::autogradNotImplementedFallback())
TORCH_LIBRARY_IMPL(basal, Autograd, m) {
  BASAL_NO_GRADIENT(m, "paged_attention");
  BASAL_NO_GRADIENT(m, "kv_append");
  BASAL_NO_GRADIENT(m, "kv_copy_pages");
  BASAL_NO_GRADIENT(m, "gdn_step");
  BASAL_NO_GRADIENT(m, "constrain_logits");
}
