// py_serve.cpp -- saccade_core._serve: the checks, allocations and calls of the serving operators
// (saccade_core/paged.py, saccade_core/logits.py) as one CPython call each.
//
// A decode step's operators run for 4 to 10 us on the device, less than their argument checks took in
// Python (24 us a call at first, 15 us when trimmed); here a call's host side is 4 us (append) to 8 us (logits with
// the best token: two kernels), most of it the launches.  The library's entry points come as addresses from the ctypes binding (bind), so
// there is one library, whatever SACCADE_CTARQ_LIB says.
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <optional>
#include <stdexcept>
#include <string>

#include "saccade_qwen2.h"

namespace {

decltype(&sc_qwen2_paged_append) f_append;
decltype(&sc_qwen2_paged_attention) f_attention;
decltype(&sc_qwen2_paged_attention_scratch) f_attention_scratch;
decltype(&sc_qwen2_process_logits) f_logits;
decltype(&sc_qwen2_process_logits_scratch) f_logits_scratch;
PyObject* f_check;  // raises a status other than SC_OK

using at::Tensor;

void require(bool ok, const std::string& what) {
    if (!ok) throw std::invalid_argument(what);
}
void require(bool ok, const char* what) {
    if (!ok) throw std::invalid_argument(what);
}

const Tensor& tensor(PyObject* o, const char* what) {
    if (!THPVariable_Check(o)) throw std::invalid_argument(std::string(what) + " must be a tensor");
    return THPVariable_Unpack(o);
}
bool none(PyObject* o) { return o == Py_None; }

// SC_F32 / SC_F16 / SC_BF16, or -1.
int code(at::ScalarType t) {
    return t == at::kFloat ? SC_F32 : t == at::kHalf ? SC_F16 : t == at::kBFloat16 ? SC_BF16 : -1;
}
at::ScalarType scalar(int c) { return c == SC_F32 ? at::kFloat : c == SC_F16 ? at::kHalf : at::kBFloat16; }

int gpu_of(const Tensor& t) { return t.is_cuda() ? t.device().index() : -1; }

// Row stride of a [tokens, heads, dim] tensor whose heads are contiguous.
int64_t rows(const Tensor& t, const char* what) {
    const bool ok = t.dim() == 3 && t.stride(2) == 1 && (t.stride(1) == t.size(2) || t.size(1) == 1);
    if (!ok)
        throw std::invalid_argument(std::string(what) +
                                    " must be [tokens, heads, head_dim] with each token's heads contiguous");
    return t.stride(0);
}

uint32_t* status_ptr(PyObject* o, int dev) {
    if (none(o)) return nullptr;
    const Tensor& t = tensor(o, "status");
    require(t.scalar_type() == at::kInt && gpu_of(t) == dev && t.numel() >= 1,
            "status must be an int32 tensor on the other tensors' device");
    return static_cast<uint32_t*>(t.data_ptr());
}

struct Cache {
    void *k, *v;
    int dtype;
    int64_t pages, nkv, page, hd, stride, seqs, max_pages;
    const int32_t *table, *cu_q, *kv_len;
    int dev;
};

Cache cache_of(PyObject* const* a) {  // k_pages, v_pages, block_table, cu_q, kv_len
    const Tensor &k = tensor(a[0], "k_pages"), &v = tensor(a[1], "v_pages"), &table = tensor(a[2], "block_table"),
                 &cu = tensor(a[3], "cu_q"), &kv = tensor(a[4], "kv_len");
    require(k.dim() == 4 && v.sizes() == k.sizes() && v.scalar_type() == k.scalar_type(),
            "k_pages and v_pages must both be [pages, kv heads, page size, head dim] of one type");
    Cache c;
    c.dtype = code(k.scalar_type());
    require(c.dtype >= 0, "the cache must be float32, float16 or bfloat16");
    c.pages = k.size(0), c.nkv = k.size(1), c.page = k.size(2), c.hd = k.size(3), c.stride = k.stride(0);
    require(k.stride(1) == c.page * c.hd && k.stride(2) == c.hd && k.stride(3) == 1 && v.strides() == k.strides(),
            "each page must be contiguous, and k_pages and v_pages equally far apart");
    c.seqs = kv.dim() == 1 ? kv.size(0) : -1;
    require(table.scalar_type() == at::kInt && cu.scalar_type() == at::kInt && kv.scalar_type() == at::kInt &&
                table.dim() == 2 && table.size(0) == c.seqs && cu.dim() == 1 && cu.size(0) == c.seqs + 1,
            "block_table [seqs, max pages], cu_q [seqs + 1] and kv_len [seqs] must be int32");
    require(table.is_contiguous() && cu.is_contiguous() && kv.is_contiguous(),
            "block_table, cu_q and kv_len must be contiguous");
    c.dev = gpu_of(k);
    require(c.dev >= 0 && gpu_of(v) == c.dev && gpu_of(table) == c.dev && gpu_of(cu) == c.dev &&
                gpu_of(kv) == c.dev,
            "the pages, the block table and the lengths must be on one CUDA device");
    c.k = k.data_ptr(), c.v = v.data_ptr(), c.max_pages = table.size(1);
    c.table = static_cast<const int32_t*>(table.data_ptr());
    c.cu_q = static_cast<const int32_t*>(cu.data_ptr());
    c.kv_len = static_cast<const int32_t*>(kv.data_ptr());
    return c;
}

// Device `dev` current while this lives, and its current stream.
struct On {
    c10::cuda::OptionalCUDAGuard guard;
    void* stream;
    explicit On(int dev) {
        if (c10::cuda::current_device() != dev) guard.set_index(static_cast<c10::DeviceIndex>(dev));
        stream = c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(dev)).stream();
    }
};

// A call's scratch, from torch's allocator and back to it for the stream's next call.
c10::DataPtr scratch(size_t bytes) { return c10::cuda::CUDACachingAllocator::get()->allocate(bytes); }

// A status other than SC_OK becomes the library's exception.
bool passed(sc_status st) {
    if (st == SC_OK) return true;
    PyObject* r = PyObject_CallFunction(f_check, "i", static_cast<int>(st));
    Py_XDECREF(r);
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "a call of the library failed");
    return false;
}

template <typename F>
PyObject* guarded(F&& body) {
    try {
        return body();
    } catch (const std::invalid_argument& e) {
        PyErr_SetString(PyExc_ValueError, e.what());
    } catch (const std::exception& e) {
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, e.what());
    } catch (...) {
        PyErr_SetString(PyExc_RuntimeError, "an unknown C++ exception");
    }
    return nullptr;
}

bool takes(Py_ssize_t n, Py_ssize_t want) {
    if (n == want) return true;
    PyErr_Format(PyExc_TypeError, "%zd arguments, %zd wanted", n, want);
    return false;
}

int64_t integer(PyObject* o, const char* what) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) {
        PyErr_Clear();
        throw std::invalid_argument(std::string(what) + " must be an integer");
    }
    return v;
}

bool truth(PyObject* o, const char* what) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) {
        PyErr_Clear();
        throw std::invalid_argument(std::string(what) + " must be true or false");
    }
    return v != 0;
}

// paged_append(q, k, v, cos, sin, k_pages, v_pages, block_table, cu_q, kv_len, out, status)
PyObject* paged_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (!takes(n, 12)) return nullptr;
    return guarded([&]() -> PyObject* {
        const Cache c = cache_of(a + 5);
        const Tensor &q = tensor(a[0], "q"), &k = tensor(a[1], "k"), &v = tensor(a[2], "v"), &cos = tensor(a[3], "cos"),
                     &sin = tensor(a[4], "sin");
        const int64_t qs = rows(q, "q"), ks = rows(k, "k"), vs = rows(v, "v"), tokens = q.size(0), nh = q.size(1);
        require(q.size(2) == c.hd && k.size(0) == tokens && k.size(1) == c.nkv && k.size(2) == c.hd && v.sizes() == k.sizes(),
                "q must be [tokens, heads, head_dim], k and v [tokens, kv heads, head_dim] of the cache's heads");
        const int dt = code(q.scalar_type());
        require((dt == SC_F32 || dt == c.dtype) && k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(),
                "q, k and v must all be float32 or all of the cache's type");
        require(cos.scalar_type() == at::kFloat && sin.scalar_type() == at::kFloat && cos.dim() == 2 &&
                    cos.size(1) == c.hd && sin.sizes() == cos.sizes() && cos.is_contiguous() && sin.is_contiguous(),
                "cos and sin must be contiguous float32 [positions, head_dim]");
        require(gpu_of(q) == c.dev && gpu_of(k) == c.dev && gpu_of(v) == c.dev && gpu_of(cos) == c.dev &&
                    gpu_of(sin) == c.dev,
                "every tensor must be on the cache's device");
        Tensor out;
        if (!none(a[10])) {
            out = tensor(a[10], "out");
            require(out.sizes() == q.sizes() && code(out.scalar_type()) == c.dtype && gpu_of(out) == c.dev &&
                        out.is_contiguous(),
                    "out must be a contiguous tensor of q's shape and the cache's type on its device");
        }
        uint32_t* st = status_ptr(a[11], c.dev);
        const On on(c.dev);
        if (!out.defined()) out = at::empty({tokens, nh, c.hd}, q.options().dtype(scalar(c.dtype)).requires_grad(false));
        if (tokens > 0 && c.seqs > 0 &&
            !passed(f_append(q.data_ptr(), k.data_ptr(), v.data_ptr(), dt, qs, ks, vs, tokens,
                             static_cast<const float*>(cos.data_ptr()), static_cast<const float*>(sin.data_ptr()), cos.size(0),
                             static_cast<int>(nh), static_cast<int>(c.nkv), static_cast<int>(c.hd), c.k, c.v, c.dtype, c.pages,
                             c.stride, static_cast<int>(c.page), c.table, c.max_pages, c.cu_q, c.kv_len, c.seqs,
                             out.data_ptr(), st, on.stream)))
            return nullptr;
        return THPVariable_Wrap(out);
    });
}

// paged_attention(q, k_pages, v_pages, block_table, cu_q, kv_len, max_q_len, max_kv_len, scale, out, out_dtype, return_lse,
//                 status); out_dtype: an SC_ code, or -1 for the cache's
PyObject* paged_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (!takes(n, 13)) return nullptr;
    return guarded([&]() -> PyObject* {
        const Cache c = cache_of(a + 1);
        const Tensor& q = tensor(a[0], "q");
        const int64_t qs = rows(q, "q"), tokens = q.size(0), nh = q.size(1);
        require(q.size(2) == c.hd && code(q.scalar_type()) == c.dtype && gpu_of(q) == c.dev,
                "q must be [tokens, heads, head_dim] of the cache's type, head_dim and device");
        int64_t max_q = integer(a[6], "max_q_len");
        const int64_t max_kv = integer(a[7], "max_kv_len");
        const double scale = none(a[8]) ? 1.0 / std::sqrt(static_cast<double>(c.hd)) : PyFloat_AsDouble(a[8]);
        if (PyErr_Occurred()) {
            PyErr_Clear();
            throw std::invalid_argument("scale must be a number");
        }
        int odt = static_cast<int>(integer(a[10], "out_dtype"));
        Tensor out;
        if (!none(a[9])) {
            out = tensor(a[9], "out");
            if (odt < 0) odt = code(out.scalar_type());
            require(out.sizes() == q.sizes() && code(out.scalar_type()) == odt && gpu_of(out) == c.dev && out.is_contiguous(),
                    "out must be a contiguous tensor of q's shape and out_dtype on the cache's device");
        }
        if (odt < 0) odt = c.dtype;
        require(odt == c.dtype || (c.dtype == SC_F32 && odt == SC_F16),
                "out must be of the cache's type, or float16 from a float32 cache");
        const bool want_lse = truth(a[11], "return_lse");
        uint32_t* st = status_ptr(a[12], c.dev);
        const On on(c.dev);
        const at::TensorOptions opt = q.options().requires_grad(false);
        if (!out.defined()) out = at::empty({tokens, nh, c.hd}, opt.dtype(scalar(odt)));
        Tensor lse;
        if (want_lse) lse = at::empty({tokens, nh}, opt.dtype(at::kFloat));
        if (tokens > 0 && c.seqs > 0) {
            if (max_q > tokens) max_q = tokens;
            const size_t bytes = f_attention_scratch(c.seqs, static_cast<int>(nh), static_cast<int>(c.nkv),
                                                     static_cast<int>(c.hd), max_q, max_kv, c.dtype);
            const c10::DataPtr ws = scratch(bytes);
            if (!passed(f_attention(q.data_ptr(), qs, c.k, c.v, c.dtype, c.pages, c.stride, static_cast<int>(c.page), c.table,
                                    c.max_pages, c.cu_q, c.kv_len, c.seqs, tokens, static_cast<int>(nh),
                                    static_cast<int>(c.nkv), static_cast<int>(c.hd), max_q, max_kv, static_cast<float>(scale),
                                    out.data_ptr(), odt, want_lse ? static_cast<float*>(lse.data_ptr()) : nullptr, ws.get(),
                                    bytes, st, on.stream)))
                return nullptr;
        }
        if (!want_lse) return THPVariable_Wrap(out);
        PyObject *x = THPVariable_Wrap(out), *y = x ? THPVariable_Wrap(lse) : nullptr;
        PyObject* r = x && y ? PyTuple_Pack(2, x, y) : nullptr;
        Py_XDECREF(x);
        Py_XDECREF(y);
        return r;
    });
}

// A contiguous vector's data, or null for None.
template <typename T>
const T* vector_of(PyObject* o, const char* what, int64_t n, at::ScalarType type, int dev) {
    if (none(o)) return nullptr;
    const Tensor& t = tensor(o, what);
    const bool ok = t.dim() == 1 && t.size(0) == n && t.scalar_type() == type && gpu_of(t) == dev && t.is_contiguous();
    if (!ok)
        throw std::invalid_argument(std::string(what) + " must be a contiguous " + c10::toString(type) + " tensor [" +
                                    std::to_string(n) + "] on the logits' device");
    return static_cast<const T*>(t.data_ptr());
}

// process_logits(logits, history, prompt_len, hist_len, repetition, presence, frequency, bias_ptr, bias_ids, bias_vals, mask,
//                mask_row, vocab_begin, out, return_best, status)
PyObject* process_logits(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (!takes(n, 16)) return nullptr;
    return guarded([&]() -> PyObject* {
        const Tensor& x = tensor(a[0], "logits");
        const int dt = code(x.scalar_type()), dev = gpu_of(x);
        require(x.dim() == 2 && dt >= 0 && dev >= 0, "logits must be a float32, float16 or bfloat16 CUDA tensor [rows, vocab]");
        const int64_t r = x.size(0), vocab = x.size(1), begin = integer(a[12], "vocab_begin");
        require(x.stride(1) == 1 || vocab <= 1, "each row of the logits must be contiguous");
        require(vocab >= 1 && begin >= 0, "the logits must have a token, and vocab_begin must not be negative");
        Tensor out;
        if (!none(a[13])) {
            out = tensor(a[13], "out");
            require(out.sizes() == x.sizes() && out.scalar_type() == x.scalar_type() && gpu_of(out) == dev &&
                        (out.stride(1) == 1 || vocab <= 1),
                    "out must be of the logits' shape, type and device, each row contiguous");
        }
        const int32_t *hist = nullptr, *plen = nullptr, *hlen = nullptr;
        int64_t width = 0;
        if (!none(a[1])) {
            const Tensor& h = tensor(a[1], "history");
            require(h.dim() == 2 && h.size(0) == r && h.scalar_type() == at::kInt && gpu_of(h) == dev && h.is_contiguous(),
                    "history must be a contiguous int32 tensor [rows, width] on the logits' device");
            require(!none(a[3]), "a history needs hist_len");
            width = h.size(1);
            hist = static_cast<const int32_t*>(h.data_ptr());
            plen = vector_of<int32_t>(a[2], "prompt_len", r, at::kInt, dev);
            hlen = vector_of<int32_t>(a[3], "hist_len", r, at::kInt, dev);
        } else {
            require(none(a[2]) && none(a[3]), "hist_len and prompt_len are a history's");
        }
        const float* rep = vector_of<float>(a[4], "repetition", r, at::kFloat, dev);
        const float* pres = vector_of<float>(a[5], "presence", r, at::kFloat, dev);
        const float* freq = vector_of<float>(a[6], "frequency", r, at::kFloat, dev);
        const int32_t *bptr = nullptr, *bids = nullptr;
        const float* bvals = nullptr;
        int64_t nbias = 0;
        if (!none(a[7])) {
            require(!none(a[8]) && !none(a[9]) && tensor(a[8], "bias_ids").dim() == 1, "bias_ptr needs bias_ids and bias_vals [entries]");
            nbias = tensor(a[8], "bias_ids").size(0);
            bptr = vector_of<int32_t>(a[7], "bias_ptr", r + 1, at::kInt, dev);
            bids = vector_of<int32_t>(a[8], "bias_ids", nbias, at::kInt, dev);
            bvals = vector_of<float>(a[9], "bias_vals", nbias, at::kFloat, dev);
        } else {
            require(none(a[8]) && none(a[9]), "bias entries need bias_ptr");
        }
        const int32_t *mask = nullptr, *mrow = nullptr;
        int64_t masks = 0, words = 0;
        if (!none(a[10])) {
            const Tensor& m = tensor(a[10], "mask");
            require(m.dim() == 2 && m.scalar_type() == at::kInt && gpu_of(m) == dev && m.is_contiguous(),
                    "mask must be a contiguous int32 tensor [masks, words] on the logits' device");
            masks = m.size(0), words = m.size(1);
            require(words * 32 >= begin + vocab, "the mask's words do not cover the logits' tokens");
            mrow = vector_of<int32_t>(a[11], "mask_row", r, at::kInt, dev);
            require(mrow != nullptr || !none(a[11]) || masks >= r, "fewer masks than rows (mask_row names each row's)");
            mask = static_cast<const int32_t*>(m.data_ptr());
        } else {
            require(none(a[11]), "mask_row needs a mask");
        }
        const bool want = truth(a[14], "return_best");
        uint32_t* st = status_ptr(a[15], dev);
        const On on(dev);
        const at::TensorOptions opt = x.options().requires_grad(false);
        if (!out.defined()) out = at::empty({r, vocab}, opt);
        Tensor best, value;
        if (want) {
            best = at::empty({r}, opt.dtype(at::kLong));
            value = at::empty({r}, opt);
        }
        if (r > 0) {
            const size_t bytes = want ? f_logits_scratch(r, vocab) : 0;
            const c10::DataPtr ws = scratch(bytes);
            if (!passed(f_logits(x.data_ptr(), dt, r, vocab, x.stride(0), begin, hist, width, plen, hlen, rep, pres, freq, bptr,
                                 bids, bvals, nbias, mask, words, masks, mrow, out.data_ptr(), out.stride(0),
                                 want ? static_cast<int64_t*>(best.data_ptr()) : nullptr, want ? value.data_ptr() : nullptr,
                                 ws.get(), bytes, st, on.stream)))
                return nullptr;
        }
        if (!want) return THPVariable_Wrap(out);
        PyObject *p = THPVariable_Wrap(out), *b = p ? THPVariable_Wrap(best) : nullptr, *v = b ? THPVariable_Wrap(value) : nullptr;
        PyObject* t = v ? PyTuple_Pack(3, p, b, v) : nullptr;
        Py_XDECREF(p);
        Py_XDECREF(b);
        Py_XDECREF(v);
        return t;
    });
}

// bind(check, {name: address}): the library's entry points
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (!takes(n, 2)) return nullptr;
    return guarded([&]() -> PyObject* {
        auto address = [&](const char* name) {
            PyObject* o = PyDict_GetItemString(a[1], name);
            if (!o) throw std::invalid_argument(std::string("no address of ") + name);
            void* p = PyLong_AsVoidPtr(o);
            if (!p) throw std::invalid_argument(std::string("no address of ") + name);
            return p;
        };
        f_append = reinterpret_cast<decltype(f_append)>(address("sc_qwen2_paged_append"));
        f_attention = reinterpret_cast<decltype(f_attention)>(address("sc_qwen2_paged_attention"));
        f_attention_scratch = reinterpret_cast<decltype(f_attention_scratch)>(address("sc_qwen2_paged_attention_scratch"));
        f_logits = reinterpret_cast<decltype(f_logits)>(address("sc_qwen2_process_logits"));
        f_logits_scratch = reinterpret_cast<decltype(f_logits_scratch)>(address("sc_qwen2_process_logits_scratch"));
        Py_INCREF(a[0]);
        Py_XDECREF(f_check);
        f_check = a[0];
        Py_RETURN_NONE;
    });
}

PyMethodDef methods[] = {
    {"bind", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(bind)), METH_FASTCALL, nullptr},
    {"paged_append", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(paged_append)), METH_FASTCALL, nullptr},
    {"paged_attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(paged_attention)), METH_FASTCALL, nullptr},
    {"process_logits", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(process_logits)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_serve", "The serving operators' host side.", -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__serve() { return PyModule_Create(&module); }
