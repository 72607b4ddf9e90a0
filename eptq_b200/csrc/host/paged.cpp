// Host path of the paged-cache operators: tensor checks, output and scratch allocation and the C-ABI call in one native
// function per call.  Over ctypes a call took 20 to 28 us, beside kernels of 3 to 10 us.
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/utils/object_ptr.h>
#include <ATen/core/grad_mode.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGuard.h>

#include "../../../include/eptq_b200.h"
#include "scratch.hpp"

namespace {

#define REFUSE_UNLESS(cond, ...) TORCH_CHECK(cond, "eptq_b200: ", __VA_ARGS__)

const at::Tensor& tensor(PyObject* o, const char* name) {
    REFUSE_UNLESS(THPVariable_Check(o), "`", name, "` must be a tensor");
    return THPVariable_Unpack(o);
}

// On the GPU, on `device` where one is given, and without a gradient to form, backward or forward.
const at::Tensor& on_gpu(PyObject* o, const char* name, const c10::Device* device = nullptr) {
    const at::Tensor& t = tensor(o, name);
    REFUSE_UNLESS(t.is_cuda(), "`", name, "` must be a CUDA tensor (there is no CPU path)");
    REFUSE_UNLESS(device == nullptr || t.device() == *device, "`", name, "` is on ", t.device(), ", not on ", *device);
    REFUSE_UNLESS(!t.requires_grad() || !at::GradMode::is_enabled(), "`", name, "` wants a gradient, and the paged operators form none");
    REFUSE_UNLESS(!t._fw_grad(0).defined() || !c10::AutogradState::get_tls_state().get_fw_grad_mode(), "`", name,
                  "` carries a forward-mode tangent, and the paged operators form none");
    return t;
}

void whole(const at::Tensor& t, const char* name, at::ScalarType type, int64_t numel = -1) {
    REFUSE_UNLESS(t.scalar_type() == type && t.is_contiguous() && (numel < 0 || t.numel() == numel), "`", name, "` must be a contiguous ", type,
                  " tensor", numel < 0 ? std::string() : " of " + std::to_string(numel) + " values");
}

int dtype_of(const at::Tensor& q, const char* what) {
    REFUSE_UNLESS(q.scalar_type() == at::kHalf || q.scalar_type() == at::kBFloat16, what, " takes fp16 or bf16 tensors");
    return q.scalar_type() == at::kHalf ? EPTQ_FP16 : EPTQ_BF16;
}

bool aligned(const at::Tensor& t) { return (reinterpret_cast<uintptr_t>(t.const_data_ptr()) & 15u) == 0; }
const uint16_t* data(const at::Tensor& t) { return static_cast<const uint16_t*>(t.const_data_ptr()); }
// For what a call writes: copy-on-write storage gets memory of its own, and autograd and whoever else watches the version
// learns of the change.
uint16_t* mutable_data(const at::Tensor& t) { return static_cast<uint16_t*>(t.mutable_data_ptr()); }
void written(const at::Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
int narrow(int64_t v, const char* name) {
    REFUSE_UNLESS(v >= INT32_MIN && v <= INT32_MAX, name, " is out of range");
    return static_cast<int>(v);
}

// Rows of whole heads, possibly column ranges of a wider tensor; returns the elements from row to row.
int64_t packed(const at::Tensor& t, const char* name, at::ScalarType type, int64_t rows) {
    REFUSE_UNLESS(t.dim() == 2 && t.scalar_type() == type && t.size(0) == rows, "`", name, "` must be a (", rows, ", heads * head_dim) ", type, " tensor");
    if (t.numel() == 0 || rows == 1) {
        REFUSE_UNLESS(t.numel() == 0 || ((t.size(1) == 1 || t.stride(1) == 1) && aligned(t)), "`", name, "` needs unit stride in a row and 16-byte alignment");
        return t.size(1);
    }
    REFUSE_UNLESS(t.stride(1) == 1 && t.stride(0) % 8 == 0 && t.stride(0) >= t.size(1) && aligned(t), "`", name,
                  "` needs unit stride in a row, a row stride that is a multiple of 8 and 16-byte alignment");
    return t.stride(0);
}

struct Cache { int n_pages, heads, page_size, head_dim; int64_t stride; };

Cache cache_of(const at::Tensor& k, const at::Tensor& v, at::ScalarType type) {
    Cache c;
    const at::Tensor* both[2] = {&k, &v};
    for (int i = 0; i < 2; ++i) {
        const at::Tensor& t = *both[i];
        const char* name = i == 0 ? "k_cache" : "v_cache";
        REFUSE_UNLESS(t.dim() == 4 && t.scalar_type() == type && t.sizes() == k.sizes(), "`", name, "` must be a (n_pages, n_kv_heads, page_size, head_dim) ",
                      type, " tensor, k_cache and v_cache alike");
        const int64_t n = t.size(0), g = t.size(1), ps = t.size(2), hd = t.size(3);
        REFUSE_UNLESS(ps == 16 || ps == 32 || ps == 64 || ps == 128, "page_size must be 16, 32, 64 or 128");
        REFUSE_UNLESS(g > 0 && hd > 0, "`", name, "` holds no heads");
        if (t.numel() == 0) continue;
        REFUSE_UNLESS((hd == 1 || t.stride(3) == 1) && t.stride(2) == hd && (g == 1 || t.stride(1) == ps * hd) && (n == 1 || (t.stride(0) >= g * ps * hd && t.stride(0) % 8 == 0)) && aligned(t),
                      "`", name, "`: a page must be contiguous and 16-byte aligned, pages a multiple of 8 values apart");
        REFUSE_UNLESS(n == 1 || t.stride(0) == k.stride(0), "k_cache and v_cache must have their pages equally far apart");
    }
    c.n_pages = narrow(k.size(0), "the number of pages");
    c.heads = narrow(k.size(1), "the number of key/value heads");
    c.page_size = static_cast<int>(k.size(2));
    c.head_dim = narrow(k.size(3), "head_dim");
    c.stride = k.size(0) > 1 ? k.stride(0) : k.size(1) * k.size(2) * k.size(3);
    return c;
}

int64_t table_of(const at::Tensor& t, int64_t B) {
    REFUSE_UNLESS(t.dim() == 2 && t.scalar_type() == at::kInt && t.size(0) == B && (t.numel() == 0 || ((t.size(1) == 1 || t.stride(1) == 1) && (B == 1 || t.stride(0) >= t.size(1)))),
                  "`tables` must be an int32 (", B, ", width) tensor with unit stride in a row");
    return t.numel() != 0 && B > 1 ? t.stride(0) : t.size(1);
}

struct Input { const at::Tensor& t; const char* name; };

bool overlap(const at::Tensor& a, const at::Tensor& b) {
    uintptr_t from[2], to[2];
    const at::Tensor* const both[2] = {&a, &b};
    for (int i = 0; i < 2; ++i) {
        const at::Tensor& t = *both[i];
        if (t.numel() == 0) return false;
        int64_t last = 0;
        for (int64_t d = 0; d < t.dim(); ++d) last += (t.size(d) - 1) * t.stride(d);
        from[i] = reinterpret_cast<uintptr_t>(t.const_data_ptr());
        to[i] = from[i] + (last + 1) * t.element_size();
    }
    return from[0] < to[1] && from[1] < to[0];
}

// The output, in memory apart from what the call reads meanwhile; q itself will do, each of its rows is read before it is written.
at::Tensor output(PyObject* o, const at::Tensor& q, std::initializer_list<Input> others) {
    if (o == Py_None) return at::empty(q.sizes(), q.options());
    const c10::Device device = q.device();
    const at::Tensor& out = on_gpu(o, "out", &device);
    REFUSE_UNLESS(out.sizes() == q.sizes() && out.scalar_type() == q.scalar_type() && out.is_contiguous() && aligned(out),
                  "`out` must be contiguous, of q's shape and type");
    out.mutable_data_ptr();                       // a lazy copy gets memory of its own here, apart from its original's
    REFUSE_UNLESS((q.is_contiguous() && q.const_data_ptr() == out.const_data_ptr()) || !overlap(out, q), "`out` overlaps `q` and is not q itself");
    for (const Input& i : others) REFUSE_UNLESS(!overlap(out, i.t), "`out` overlaps `", i.name, "`");
    return out;
}

// `n` values of `type` from the `at`-th on in the storage of `all`, as a tensor of its own.
at::Tensor part(const at::Tensor& all, at::ScalarType type, int64_t at, int64_t n) {
    auto t = c10::make_intrusive<at::TensorImpl>(c10::Storage(all.storage()), all.key_set(), c10::scalarTypeToTypeMeta(type));
    t->set_storage_offset(at);
    t->set_sizes_contiguous({n});
    return at::Tensor(std::move(t));
}

void done(int status, const char* what) { TORCH_CHECK(status == EPTQ_OK, "eptq ", what, ": ", eptq_strerror(status), " (eptq status ", status, ")"); }

void arguments(Py_ssize_t n, Py_ssize_t want, const char* usage) { TORCH_CHECK_TYPE(n == want, usage); }

int64_t integer(PyObject* o) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw python_error();
    return v;
}
double number(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw python_error();
    return v;
}

// plan_pages(cached, new, tables, free_pages, n_free, page_size, rows) -> (cu_rows, kv_lens, positions, slots, n_free)
PyObject* plan_pages(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    arguments(n, 7, "plan_pages(cached, new, tables, free_pages, n_free, page_size, rows)");
    const at::Tensor& cached = on_gpu(a[0], "cached");
    const c10::Device device = cached.device();
    const at::Tensor& fresh = on_gpu(a[1], "new", &device);
    const at::Tensor& tables = on_gpu(a[2], "tables", &device);
    const at::Tensor& free_pages = on_gpu(a[3], "free_pages", &device);
    const at::Tensor& n_free = on_gpu(a[4], "n_free", &device);
    const int64_t B = cached.numel();
    whole(cached, "cached", at::kInt);
    whole(fresh, "new", at::kInt, B);
    whole(free_pages, "free_pages", at::kInt);
    whole(n_free, "n_free", at::kInt, 1);
    const int64_t stride = table_of(tables, B);
    const int64_t rows = integer(a[6]);
    const int page_size = narrow(integer(a[5]), "page_size"), n_rows = narrow(rows, "rows");
    const int batch = narrow(B, "the number of requests"), width = narrow(tables.size(1), "the table's width"), cap = narrow(free_pages.numel(), "the free list");
    REFUSE_UNLESS(page_size == 16 || page_size == 32 || page_size == 64 || page_size == 128, "page_size must be 16, 32, 64 or 128");
    REFUSE_UNLESS(rows >= 0, "rows must not be negative");
    const c10::cuda::OptionalCUDAGuard guard(device);
    // One allocation for the five outputs, each a part of it: five cost more than the kernel.
    const at::Tensor all = at::empty({2 * rows + B + 1}, cached.options().dtype(at::kLong));
    at::Tensor out[5] = {part(all, at::kInt, 4 * rows, B + 1), part(all, at::kInt, 4 * rows + B + 1, B), part(all, at::kLong, 0, rows),
                         part(all, at::kLong, rows, rows), part(all, at::kInt, 4 * rows + 2 * B + 1, 1)};
    const auto stream = c10::cuda::getCurrentCUDAStream(device.index());
    int32_t* const table = tables.mutable_data_ptr<int32_t>();
    done(eptq_plan_pages(cached.const_data_ptr<int32_t>(), fresh.const_data_ptr<int32_t>(), batch, table, stride, width,
                         free_pages.const_data_ptr<int32_t>(), cap, n_free.const_data_ptr<int32_t>(), page_size, n_rows, out[0].data_ptr<int32_t>(),
                         out[1].data_ptr<int32_t>(), out[2].data_ptr<int64_t>(), out[3].data_ptr<int64_t>(), out[4].data_ptr<int32_t>(), stream.stream()), "plan_pages");
    written(tables);
    THPObjectPtr r(PyTuple_New(5));
    if (!r) return nullptr;
    for (int i = 0; i < 5; ++i) PyTuple_SET_ITEM(r.get(), i, THPVariable_Wrap(std::move(out[i])));
    return r.release();
    END_HANDLE_TH_ERRORS
}

// rope_append_paged(q, k, v, k_cache, v_cache, positions, slots, inv_freq, scaling, out or None) -> out
PyObject* rope_append_paged(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    arguments(n, 10, "rope_append_paged(q, k, v, k_cache, v_cache, positions, slots, inv_freq, scaling, out)");
    const at::Tensor& q = on_gpu(a[0], "q");
    const c10::Device device = q.device();
    const at::Tensor& k = on_gpu(a[1], "k", &device);
    const at::Tensor& v = on_gpu(a[2], "v", &device);
    const at::Tensor& k_cache = on_gpu(a[3], "k_cache", &device);
    const at::Tensor& v_cache = on_gpu(a[4], "v_cache", &device);
    const at::Tensor& positions = on_gpu(a[5], "positions", &device);
    const at::Tensor& slots = on_gpu(a[6], "slots", &device);
    const at::Tensor& inv_freq = on_gpu(a[7], "inv_freq", &device);
    const int dtype = dtype_of(q, "rope_append_paged");
    REFUSE_UNLESS(q.dim() == 2, "`q` must be a (rows, heads * head_dim) tensor");
    const int64_t rows = q.size(0);
    const int64_t qs = packed(q, "q", q.scalar_type(), rows), ks = packed(k, "k", q.scalar_type(), rows), vs = packed(v, "v", q.scalar_type(), rows);
    const Cache c = cache_of(k_cache, v_cache, q.scalar_type());
    const int64_t kv_width = static_cast<int64_t>(c.heads) * c.head_dim;
    REFUSE_UNLESS(q.size(1) > 0 && q.size(1) % c.head_dim == 0 && k.size(1) == kv_width && v.size(1) == kv_width,
                  "q, k and v must hold whole heads of the caches' head_dim, k and v as many as the caches");
    whole(positions, "positions", at::kLong, rows);
    whole(slots, "slots", at::kLong, rows);
    whole(inv_freq, "inv_freq", at::kFloat, c.head_dim / 2);
    const float scaling = static_cast<float>(number(a[8]));
    const c10::cuda::OptionalCUDAGuard guard(device);
    uint16_t *const kc = mutable_data(k_cache), *const vc = mutable_data(v_cache);
    REFUSE_UNLESS(rows == 0 || k_cache.numel() == 0 || kc != vc, "k_cache and v_cache are the same memory");
    at::Tensor out = output(a[9], q, {{k, "k"}, {v, "v"}, {k_cache, "k_cache"}, {v_cache, "v_cache"}, {positions, "positions"}, {slots, "slots"}, {inv_freq, "inv_freq"}});
    const auto stream = c10::cuda::getCurrentCUDAStream(device.index());
    uint16_t* const out_at = mutable_data(out);
    done(eptq_rope_append_paged(dtype, data(q), qs, data(k), ks, data(v), vs, out_at, kc, vc, c.stride, positions.const_data_ptr<int64_t>(),
                                slots.const_data_ptr<int64_t>(), inv_freq.const_data_ptr<float>(), narrow(rows, "the number of rows"), narrow(q.size(1) / c.head_dim, "the number of heads"),
                                c.heads, c.head_dim, c.n_pages, c.page_size, scaling, stream.stream()), "rope_append_paged");
    written(k_cache);
    written(v_cache);
    if (a[9] != Py_None) written(out);
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

PyObject* attend(EptqAttention& a, const at::Tensor& q, int64_t q_stride, const at::Tensor& cu_rows, std::initializer_list<Input> others, PyObject* scale,
                 PyObject* out_or_none, const char* what) {
    const c10::Device device = q.device();
    const c10::cuda::OptionalCUDAGuard guard(device);
    at::Tensor out = output(out_or_none, q, others);
    a.clear_rest = out_or_none == Py_None;          // memory of the allocator's: rows of no request would show what it held
    a.rows = narrow(q.size(0), "the number of rows");
    a.batch = narrow(cu_rows.numel() - 1, "the number of requests");
    a.scale = static_cast<float>(scale == Py_None ? 1.0 / std::sqrt(static_cast<double>(a.head_dim)) : number(scale));
    a.q_stride = q_stride;
    a.out = mutable_data(out);
    a.q = data(q);
    a.cu_rows = cu_rows.const_data_ptr<int32_t>();
    const auto stream = c10::cuda::getCurrentCUDAStream(device.index());
    // Scratch of its own for every call, from torch's allocator: calls on different streams, and graphs captured on one
    // stream and replayed on others, share none.  The status word is that of the stream's scratch.
    a.status = reinterpret_cast<int32_t*>(static_cast<char*>(scratch_for(device.index(), stream, 1u << 20).data_ptr()) + EPTQ_STATUS_BYTE);
    const size_t need = eptq_ragged_attention_workspace_bytes(&a);
    const at::Tensor ws = need == 0 ? at::Tensor() : at::empty({static_cast<int64_t>(need)}, q.options().dtype(at::kByte));
    done(eptq_ragged_attention(&a, need == 0 ? nullptr : ws.data_ptr(), need, stream.stream()), what);
    if (out_or_none != Py_None) written(out);
    return THPVariable_Wrap(std::move(out));
}

void rows_of(const at::Tensor& cu_rows) {
    whole(cu_rows, "cu_rows", at::kInt);
    REFUSE_UNLESS(cu_rows.numel() >= 1, "`cu_rows` must hold one value more than there are requests");
}

// paged_attention(q, k_cache, v_cache, tables, kv_lens, cu_rows, max_rows, scale or None, out or None) -> out
PyObject* paged_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    arguments(n, 9, "paged_attention(q, k_cache, v_cache, tables, kv_lens, cu_rows, max_rows, scale, out)");
    const at::Tensor& q = on_gpu(a[0], "q");
    const c10::Device device = q.device();
    const at::Tensor& k_cache = on_gpu(a[1], "k_cache", &device);
    const at::Tensor& v_cache = on_gpu(a[2], "v_cache", &device);
    const at::Tensor& tables = on_gpu(a[3], "tables", &device);
    const at::Tensor& kv_lens = on_gpu(a[4], "kv_lens", &device);
    const at::Tensor& cu_rows = on_gpu(a[5], "cu_rows", &device);
    EptqAttention p = {};
    p.dtype = dtype_of(q, "paged_attention");
    REFUSE_UNLESS(q.dim() == 2, "`q` must be a (rows, heads * head_dim) tensor");
    const int64_t q_stride = packed(q, "q", q.scalar_type(), q.size(0));
    const Cache c = cache_of(k_cache, v_cache, q.scalar_type());
    REFUSE_UNLESS(q.size(1) > 0 && q.size(1) % c.head_dim == 0, "q must hold whole heads of the caches' head_dim");
    rows_of(cu_rows);
    const int64_t B = cu_rows.numel() - 1;
    whole(kv_lens, "kv_lens", at::kInt, B);
    p.table_stride = table_of(tables, B);
    p.n_heads = narrow(q.size(1) / c.head_dim, "the number of heads");
    p.n_kv_heads = c.heads;
    p.head_dim = c.head_dim;
    const int64_t max_rows = integer(a[6]);
    p.max_rows = static_cast<int>(max_rows < 0 ? 0 : max_rows > INT32_MAX ? INT32_MAX : max_rows);
    p.page_size = c.page_size;
    p.n_pages = c.n_pages;
    p.table_width = narrow(tables.size(1), "the table's width");
    p.k_stride = p.v_stride = c.stride;
    p.k = data(k_cache);
    p.v = data(v_cache);
    p.tables = tables.const_data_ptr<int32_t>();
    p.kv_lens = kv_lens.const_data_ptr<int32_t>();
    return attend(p, q, q_stride, cu_rows, {{k_cache, "k_cache"}, {v_cache, "v_cache"}, {tables, "tables"}, {kv_lens, "kv_lens"}, {cu_rows, "cu_rows"}}, a[7], a[8],
                  "paged_attention");
    END_HANDLE_TH_ERRORS
}

// prompt_attention(q, k, v, cu_rows, head_dim, scale or None, out or None) -> out
PyObject* prompt_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    arguments(n, 7, "prompt_attention(q, k, v, cu_rows, head_dim, scale, out)");
    const at::Tensor& q = on_gpu(a[0], "q");
    const c10::Device device = q.device();
    const at::Tensor& k = on_gpu(a[1], "k", &device);
    const at::Tensor& v = on_gpu(a[2], "v", &device);
    const at::Tensor& cu_rows = on_gpu(a[3], "cu_rows", &device);
    EptqAttention p = {};
    p.dtype = dtype_of(q, "prompt_attention");
    REFUSE_UNLESS(q.dim() == 2, "`q` must be a (rows, heads * head_dim) tensor");
    const int64_t q_stride = packed(q, "q", q.scalar_type(), q.size(0));
    p.k_stride = packed(k, "k", q.scalar_type(), q.size(0));
    p.v_stride = packed(v, "v", q.scalar_type(), q.size(0));
    const int64_t hd = integer(a[4]);
    REFUSE_UNLESS(hd > 0 && q.size(1) > 0 && k.size(1) > 0 && q.size(1) % hd == 0 && k.size(1) % hd == 0 && v.size(1) == k.size(1),
                  "q, k and v must hold whole heads of head_dim, k and v as many");
    rows_of(cu_rows);
    p.n_heads = narrow(q.size(1) / hd, "the number of heads");
    p.n_kv_heads = narrow(k.size(1) / hd, "the number of key/value heads");
    p.head_dim = narrow(hd, "head_dim");
    p.max_rows = narrow(q.size(0), "the number of rows");
    p.k = data(k);
    p.v = data(v);
    return attend(p, q, q_stride, cu_rows, {{k, "k"}, {v, "v"}, {cu_rows, "cu_rows"}}, a[5], a[6], "prompt_attention");
    END_HANDLE_TH_ERRORS
}

}  // namespace

#define METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef paged_methods[] = {METHOD(plan_pages), METHOD(rope_append_paged), METHOD(paged_attention), METHOD(prompt_attention),
                               {nullptr, nullptr, 0, nullptr}};
