// Python face of the decoder-layer operators: argument checks on torch tensors, the stream, and the call of the library's
// C entry point, natively, because a decode step makes a few of these calls per layer and each takes the GPU only
// microseconds (in Python the checks and the ctypes call took 13 to 16 us per call).
//
// The module has no state but the entry points' addresses, which `decoder.py` takes from the loaded library (setup()),
// and its exception class.  No C++ exception leaves a function: each becomes a Python one.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <stdexcept>
#include <string>

#include "../../include/draco_moe_b200.h"

namespace {

PyObject* g_error = nullptr;    // DracoError
decltype(&draco_b200_last_error) f_last_error = nullptr;
decltype(&draco_b200_plan_blocks) f_plan_blocks = nullptr;
decltype(&draco_b200_kv4_append) f_append = nullptr;
decltype(&draco_b200_kv4_read) f_read = nullptr;
decltype(&draco_b200_kv4_attention_workspace) f_workspace = nullptr;
decltype(&draco_b200_kv4_attention_checked) f_attention = nullptr;
decltype(&draco_b200_rmsnorm_q8) f_norm = nullptr;
void (*f_checked)(int) = nullptr;
unsigned long long (*f_capture_id)(void*) = nullptr;

struct Refused : std::runtime_error {
    using std::runtime_error::runtime_error;
};
struct PythonError {};    // already set

void need(bool ok, const char* what) {
    if (!ok) throw Refused(what);
}

const at::Tensor& tensor(PyObject* o, const char* what) {
    if (!THPVariable_Check(o)) throw Refused(std::string(what) + " must be a tensor");
    return THPVariable_Unpack(o);
}
const at::Tensor* maybe(PyObject* o, const char* what) { return o == Py_None ? nullptr : &tensor(o, what); }

const at::Tensor& vector_of(PyObject* o, at::ScalarType type, const char* what) {
    const at::Tensor& t = tensor(o, what);
    if (t.scalar_type() != type || !t.is_cuda() || t.dim() != 1 || !t.is_contiguous())
        throw Refused(std::string(what) + (type == at::kInt ? " must be a contiguous int32 vector on the GPU"
                                                             : " must be a contiguous fp32 vector on the GPU"));
    return t;
}

long number(PyObject* o) {
    const long v = PyLong_AsLong(o);
    if (v == -1 && PyErr_Occurred()) throw PythonError{};
    return v;
}
int small(PyObject* o, const char* what) {
    const long v = number(o);
    if (v < -2147483647l || v > 2147483647l) throw Refused(std::string(what) + " does not fit 32 bits");
    return (int)v;
}
double real(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw PythonError{};
    return v;
}
int fits(int64_t v, const char* what) {
    if (v > 2147483647l) throw Refused(std::string(what) + " does not fit 32 bits");
    return (int)v;
}

int dtype_of(const at::Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return 0;
        case at::kHalf: return 1;
        case at::kBFloat16: return 2;
        default: return -1;
    }
}

// the tensors' device made current for the call, as a launch needs it; made when every tensor was seen to be on it
struct OnDevice {
    c10::DeviceIndex old, now;
    explicit OnDevice(const at::Device& d) : old(c10::cuda::current_device()), now(d.index()) {
        if (now != old) c10::cuda::set_device(now);
        f_checked(1);
    }
    ~OnDevice() {
        f_checked(0);
        if (now != old) c10::cuda::set_device(old);
    }
};
// None: torch's current stream of the device, else a cudaStream_t as a number
void* stream_of(PyObject* o, const at::Device& d) {
    if (o == Py_None) return (void*)c10::cuda::getCurrentCUDAStream(d.index()).stream();
    void* p = PyLong_AsVoidPtr(o);
    if (!p && PyErr_Occurred()) throw PythonError{};
    return p;
}

PyObject* done(int rc, const char* who) {
    if (rc) throw Refused(std::string(who) + " failed (" + std::to_string(rc) + "): " + f_last_error());
    Py_RETURN_NONE;
}

template <class F>
PyObject* guarded(Py_ssize_t given, Py_ssize_t wanted, F&& body) {
    try {
        if (given != wanted) throw Refused("wrong number of arguments");
        need(f_norm != nullptr, "the library is not loaded");
        return body();
    } catch (const PythonError&) {
    } catch (const Refused& e) {
        PyErr_SetString(g_error ? g_error : PyExc_RuntimeError, e.what());
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}

// setup(DracoError, {name: address})
PyObject* setup(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 2 || !PyDict_Check(a[1])) {
        PyErr_SetString(PyExc_TypeError, "setup(error, {name: address})");
        return nullptr;
    }
    auto take = [&](const char* name, auto& f) {
        PyObject* v = PyDict_GetItemString(a[1], name);
        void* p = v ? PyLong_AsVoidPtr(v) : nullptr;
        f = reinterpret_cast<std::decay_t<decltype(f)>>(p);
        if (!p && !PyErr_Occurred()) PyErr_Format(PyExc_KeyError, "%s", name);
        return p != nullptr;
    };
    if (!take("draco_b200_last_error", f_last_error) || !take("draco_b200_plan_blocks", f_plan_blocks) ||
        !take("draco_b200_kv4_append", f_append) || !take("draco_b200_kv4_read", f_read) ||
        !take("draco_b200_kv4_attention_workspace", f_workspace) || !take("draco_b200_kv4_attention_checked", f_attention) ||
        !take("draco_b200_pointers_checked", f_checked) || !take("draco_b200_capture_id", f_capture_id) || !take("draco_b200_rmsnorm_q8", f_norm))
        return nullptr;
    Py_INCREF(a[0]);
    Py_XSETREF(g_error, a[0]);
    Py_RETURN_NONE;
}

// (ctx_len, new_len, block_table, free_pages, n_free, page_size, cu_new, seq_len, slots, positions, n_free_out, refused, stream)
PyObject* plan_blocks(PyObject*, PyObject* const* a, Py_ssize_t given) {
    return guarded(given, 13, [&] {
        const at::Tensor &ctx = vector_of(a[0], at::kInt, "ctx_len"), &add = vector_of(a[1], at::kInt, "new_len"),
                         &free = vector_of(a[3], at::kInt, "free_pages"), &n_free = vector_of(a[4], at::kInt, "n_free"),
                         &cu = vector_of(a[6], at::kInt, "cu_new"), &seq = vector_of(a[7], at::kInt, "seq_len"),
                         &slots = vector_of(a[8], at::kInt, "slots"), &pos = vector_of(a[9], at::kInt, "positions"),
                         &left = vector_of(a[10], at::kInt, "n_free"), &refused = vector_of(a[11], at::kInt, "refused");
        const at::Tensor& table = tensor(a[2], "block_table");
        const int64_t n = ctx.numel();
        need(add.numel() == n && seq.numel() == n && cu.numel() == n + 1 && n_free.numel() == 1 && left.numel() == 1 &&
                 refused.numel() == 1 && slots.numel() == pos.numel(),
             "plan_blocks: ctx_len, new_len and the plan must have the same number of requests, n_free one value");
        need(table.scalar_type() == at::kInt && table.is_cuda() && table.dim() == 2 && table.size(0) == n &&
                 (table.stride(1) == 1 || table.size(1) <= 1) && (n <= 1 || table.stride(0) >= table.size(1)),
             "block_table must be an int32 matrix on the GPU with a contiguous row for each request");
        const at::Device dev = ctx.device();
        for (const at::Tensor* t : {&add, &free, &n_free, &cu, &seq, &slots, &pos, &left, &refused, &table})
            need(t->device() == dev, "plan_blocks: all tensors must be on one device");
        const OnDevice on(dev);
        const int width = fits(table.size(1), "the table's width");
        return done(f_plan_blocks(ctx.data_ptr<int>(), add.data_ptr<int>(), fits(n, "the number of requests"),
                                  small(a[5], "page_size"), table.data_ptr<int>(), std::max<long>(table.stride(0), width),
                                  width, free.data_ptr<int>(), fits(free.numel(), "the free list"),
                                  n_free.data_ptr<int>(), fits(slots.numel(), "the number of slots"), cu.data_ptr<int>(),
                                  seq.data_ptr<int>(), slots.data_ptr<int>(), pos.data_ptr<int>(), left.data_ptr<int>(),
                                  refused.data_ptr<int>(), stream_of(a[12], dev)),
                    "draco_b200_plan_blocks");
    });
}

DracoKV4Cache cache_of(const at::Tensor& pages, PyObject* page_size, PyObject* head_dim) {
    return DracoKV4Cache{pages.data_ptr(), fits(pages.size(0), "the number of pages"), small(page_size, "page_size"),
                         fits(pages.size(1), "the number of heads"), small(head_dim, "head_dim")};
}

// (pages, page_size, head_dim, k, v, slots, stream)
PyObject* rows(PyObject* const* a, Py_ssize_t given, bool append) {
    return guarded(given, 7, [&] {
        const at::Tensor &pages = tensor(a[0], "pages"), &k = tensor(a[3], "k"), &v = tensor(a[4], "v"),
                         &slots = vector_of(a[5], at::kInt, "slots");
        const DracoKV4Cache c = cache_of(pages, a[1], a[2]);
        const int64_t n = slots.numel();
        const int dtype = dtype_of(k);
        for (const at::Tensor* t : {&k, &v})
            need(dtype >= 0 && t->scalar_type() == k.scalar_type() && t->dim() == 3 && t->size(0) == n &&
                     t->size(1) == c.n_kv_heads && t->size(2) == c.head_dim && t->stride(2) == 1,
                 "keys and values must be [slots, n_kv_heads, head_dim] tensors of one floating type with contiguous "
                 "channels");
        const at::Device dev = pages.device();
        need(k.device() == dev && v.device() == dev && slots.device() == dev, "tensors must be on the cache's device");
        const OnDevice on(dev);
        void* s = stream_of(a[6], dev);
        const int count = fits(n, "the number of tokens");
        return append ? done(f_append(&c, dtype, k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0),
                                      v.stride(1), slots.data_ptr<int>(), count, s), "draco_b200_kv4_append")
                      : done(f_read(&c, dtype, k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0),
                                    v.stride(1), slots.data_ptr<int>(), count, s), "draco_b200_kv4_read");
    });
}
PyObject* kv4_append(PyObject*, PyObject* const* a, Py_ssize_t n) { return rows(a, n, true); }
PyObject* kv4_read(PyObject*, PyObject* const* a, Py_ssize_t n) { return rows(a, n, false); }

// (pages, page_size, head_dim, scratch, grow, q, out, cu_q, seq_len, block_table, max_q_len, max_seq_len, scale, window,
//  sinks, lse, stream, workspace, status); where workspace is None: scratch: {stream: tensor}, for calls that no graph captures,
//  grow(stream, bytes, capture): another buffer, of the stream or of the capture
PyObject* kv4_attend(PyObject*, PyObject* const* a, Py_ssize_t given) {
    return guarded(given, 19, [&] {
        const at::Tensor &pages = tensor(a[0], "pages"), &q = tensor(a[5], "q"), &out = tensor(a[6], "out"),
                         &cu = vector_of(a[7], at::kInt, "cu_q"), &seq = vector_of(a[8], at::kInt, "seq_len"),
                         &table = tensor(a[9], "block_table");
        const at::Tensor* lse = maybe(a[15], "lse");
        const DracoKV4Cache c = cache_of(pages, a[1], a[2]);
        const int64_t n_req = seq.numel();
        const int dtype = dtype_of(q);
        need(dtype >= 0 && out.scalar_type() == q.scalar_type() && q.dim() == 3 && q.size(2) == c.head_dim &&
                 out.sizes() == q.sizes() && q.stride(2) == 1 && out.stride(2) == 1,
             "q and out must be [tokens, heads, head_dim] tensors of one floating type with contiguous channels");
        need(cu.numel() == n_req + 1 && table.scalar_type() == at::kInt && table.dim() == 2 && table.size(0) == n_req &&
                 (table.stride(1) == 1 || table.size(1) <= 1),
             "cu_q must have one value more than seq_len, block_table (int32) a contiguous row for each request");
        const at::Device dev = pages.device();
        need(q.device() == dev && out.device() == dev && cu.device() == dev && seq.device() == dev && table.device() == dev,
             "tensors must be on the cache's device");
        need(!lse || (lse->scalar_type() == at::kFloat && lse->dim() == 2 && lse->size(0) == q.size(0) &&
                      lse->size(1) == q.size(1) && lse->is_contiguous() && lse->device() == dev),
             "lse must be a contiguous fp32 tensor [tokens, heads]");
        const OnDevice on(dev);
        void* s = stream_of(a[16], dev);
        DracoKV4Attention p{};
        p.q = q.data_ptr(), p.out = out.data_ptr(), p.lse = lse ? lse->data_ptr<float>() : nullptr;
        p.q_token_stride = q.stride(0), p.q_head_stride = q.stride(1);
        p.out_token_stride = out.stride(0), p.out_head_stride = out.stride(1);
        p.dtype = dtype, p.n_heads = fits(q.size(1), "the number of heads");
        p.n_req = fits(n_req, "the number of requests"), p.n_tokens = fits(q.size(0), "the number of tokens");
        p.cu_q = cu.data_ptr<int>(), p.seq_len = seq.data_ptr<int>(), p.block_table = table.data_ptr<int>();
        p.table_stride = table.stride(0), p.table_width = fits(table.size(1), "the table's width");
        p.max_q_len = small(a[10], "max_q_len"), p.max_seq_len = small(a[11], "max_seq_len");
        p.scale = (float)real(a[12]), p.window = small(a[13], "window"), p.sinks = small(a[14], "sinks");
        const size_t bytes = f_workspace(&c, &p);
        if (const at::Tensor* ws = maybe(a[17], "workspace")) {
            need(ws->device() == dev && ws->is_contiguous(), "workspace must be a contiguous tensor on the cache's device");
            p.workspace = ws->data_ptr(), p.workspace_bytes = ws->nbytes();
        } else if (bytes) {
            // a captured call keeps its buffer's address, and its graph may run on any stream: captures have their own
            const unsigned long long capture = f_capture_id(s);
            // the per-thread default stream is another one in each thread
            PyObject* key = s == (void*)cudaStreamPerThread ? PyLong_FromLongLong(-(long long)PyThread_get_thread_ident())
                                                            : PyLong_FromVoidPtr(s);
            if (!key) throw PythonError{};
            PyObject* buf = capture ? nullptr : PyDict_GetItemWithError(a[3], key);    // borrowed
            if (buf && THPVariable_Check(buf) && THPVariable_Unpack(buf).nbytes() >= bytes) {
                Py_INCREF(buf);
            } else {
                buf = PyErr_Occurred() ? nullptr : PyObject_CallFunction(a[4], "OnK", key, (Py_ssize_t)bytes, capture);
            }
            Py_DECREF(key);
            if (!buf) throw PythonError{};
            if (THPVariable_Check(buf)) {     // what grow() keeps alive
                p.workspace = THPVariable_Unpack(buf).data_ptr();
                p.workspace_bytes = THPVariable_Unpack(buf).nbytes();
            }
            Py_DECREF(buf);
        }
        const at::Tensor& status = vector_of(a[18], at::kInt, "status");
        need(status.device() == dev && status.numel() > 0, "status must be on the cache's device");
        return done(f_attention(&c, &p, status.data_ptr<int>(), 0, s), "draco_b200_kv4_attention");
    });
}

// (x, weight, eps, codes, scales, residual, h, y, group, stream)
PyObject* rmsnorm_q8(PyObject*, PyObject* const* a, Py_ssize_t given) {
    return guarded(given, 10, [&] {
        const at::Tensor &x = tensor(a[0], "x"), &w = vector_of(a[1], at::kFloat, "weight"), &codes = tensor(a[3], "codes"),
                         &scales = tensor(a[4], "scales");
        const at::Tensor *r = maybe(a[5], "residual"), *h = maybe(a[6], "h"), *y = maybe(a[7], "y");
        const int dtype = dtype_of(x);
        const int fmt = codes.scalar_type() == at::kChar ? 0 : codes.scalar_type() == at::kFloat8_e4m3fn ? 1 : -1;
        const int group = small(a[8], "group");
        need(x.dim() == 2, "rmsnorm_q8: x must be [rows, hidden]");
        const int64_t n = x.size(0), hidden = x.size(1), width = group > 0 ? group : hidden;
        need(dtype >= 0 && x.is_cuda() && fmt >= 0 && scales.scalar_type() == at::kFloat && width > 0 &&
                 w.numel() == hidden && codes.sizes() == x.sizes() && scales.dim() == 2 && scales.size(0) == n &&
                 scales.size(1) == hidden / width,
             "rmsnorm_q8: x [rows, hidden] floating, codes alike in int8 or e4m3, scales fp32 [rows, hidden // group]");
        need(!r == !h, "rmsnorm_q8: residual and h go together");
        const at::Device dev = x.device();
        for (const at::Tensor* t : {&x, r, h, y, &codes, &scales})
            need(!t || (t->device() == dev && (t->dim() == 2 && (t->stride(1) == 1 || t->size(1) <= 1 || n == 0))),
                 "rmsnorm_q8: tensors must be on one device with contiguous rows");
        for (const at::Tensor* t : {r, h, y})
            need(!t || (t->scalar_type() == x.scalar_type() && t->sizes() == x.sizes()),
                 "rmsnorm_q8: residual, h and y must have x's shape and type");
        need(w.device() == dev, "rmsnorm_q8: tensors must be on one device with contiguous rows");
        if (n == 0) Py_RETURN_NONE;
        const OnDevice on(dev);
        DracoNormQ8 p{};
        p.x = x.data_ptr(), p.weight = w.data_ptr<float>(), p.codes = codes.data_ptr(), p.scales = scales.data_ptr<float>();
        p.residual = r ? r->data_ptr() : nullptr, p.h = h ? h->data_ptr() : nullptr, p.y = y ? y->data_ptr() : nullptr;
        p.x_stride = x.stride(0), p.codes_stride = codes.stride(0), p.scales_stride = scales.stride(0);
        p.residual_stride = r ? r->stride(0) : 0, p.h_stride = h ? h->stride(0) : 0, p.y_stride = y ? y->stride(0) : 0;
        p.dtype = dtype, p.fmt = fmt, p.n_rows = fits(n, "the number of rows"), p.hidden = fits(hidden, "hidden");
        p.group = group, p.eps = (float)real(a[2]);
        return done(f_norm(&p, stream_of(a[9], dev)), "draco_b200_rmsnorm_q8");
    });
}

using Fast = PyObject* (*)(PyObject*, PyObject* const*, Py_ssize_t);
PyCFunction as_method(Fast f) { return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)); }
PyMethodDef g_methods[] = {{"setup", as_method(setup), METH_FASTCALL, nullptr},
                           {"plan_blocks", as_method(plan_blocks), METH_FASTCALL, nullptr},
                           {"kv4_append", as_method(kv4_append), METH_FASTCALL, nullptr},
                           {"kv4_read", as_method(kv4_read), METH_FASTCALL, nullptr},
                           {"kv4_attend", as_method(kv4_attend), METH_FASTCALL, nullptr},
                           {"rmsnorm_q8", as_method(rmsnorm_q8), METH_FASTCALL, nullptr},
                           {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_decoder", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// torch_version: the torch whose headers this was built with
PyMODINIT_FUNC PyInit__decoder(void) {
    PyObject* m = PyModule_Create(&g_module);
    if (m && PyModule_AddStringConstant(m, "torch_version", DRACO_TORCH_VERSION)) Py_CLEAR(m);
    return m;
}
