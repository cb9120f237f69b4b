// The short way from Python to the entry points of the small, often made calls: reading a dozen
// tensors' layouts, checking them and converting thirty arguments costs 8 to 18 us in Python, more
// than the kernels take. Each function here launches if everything is as the kernel needs it
// and returns the result; otherwise it touches nothing and returns None, and the Python caller goes
// its own way, which checks step by step and says what is wrong. The kernels are those of the C ABI,
// whose addresses `bind` is given; nothing is kept between calls.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <vector>

#include "../../include/latentserve_b200.h"

namespace {

decltype(&ls_paged_decode_int4) f_decode;
decltype(&ls_int4_write) f_write;
decltype(&ls_int4_read) f_read;
decltype(&ls_copy_pages) f_copy;
decltype(&ls_rotary) f_rotary;

using at::Tensor;

constexpr int kPage = 16, kDim = 128;

const Tensor* tensor(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }

bool aligned(const Tensor& t, uintptr_t bytes) { return reinterpret_cast<uintptr_t>(t.const_data_ptr()) % bytes == 0; }

// A stride; 0 for an axis of one, whose stride says nothing.
int64_t step(const Tensor& t, int axis) { return t.size(axis) > 1 ? t.stride(axis) : 0; }

bool on(const Tensor& t, c10::Device device, at::ScalarType type) {
    return t.is_cuda() && t.device() == device && t.scalar_type() == type && t.layout() == at::kStrided;
}

// The current stream of `device` if that is the current device (the library launches there).
bool stream_of(c10::Device device, void** out) {
    if (c10::cuda::current_device() != device.index()) return false;
    *out = c10::cuda::getCurrentCUDAStream(device.index()).stream();
    return true;
}

int groups_of(const Tensor& pool) {
    const int64_t extra = pool.size(2) - 2048;
    return extra == 512 ? 4 : extra == 256 ? 2 : extra == 128 ? 1 : 0;
}

bool pool_ok(const Tensor& pool, c10::Device device, int64_t heads) {
    return on(pool, device, at::kByte) && pool.dim() == 3 && groups_of(pool) && pool.size(0) > 0 &&
           pool.size(0) <= INT32_MAX && pool.size(1) == heads && pool.stride(2) == 1 && aligned(pool, 16) &&
           pool.stride(0) % 16 == 0 && pool.stride(1) % 16 == 0 && pool.stride(0) >= pool.size(2) &&
           pool.stride(1) >= pool.size(2);
}

bool vector_ok(const Tensor& t, c10::Device device, int64_t batch) {
    return on(t, device, at::kInt) && t.dim() == 1 && t.size(0) >= batch && (t.size(0) == 1 || t.stride(0) == 1);
}

bool tables_ok(const Tensor& tables, const Tensor& lens, c10::Device device, int64_t batch) {
    return on(tables, device, at::kInt) && tables.dim() == 2 && tables.is_contiguous() && tables.size(0) >= batch &&
           tables.size(1) >= 1 && tables.size(1) <= INT32_MAX && vector_ok(lens, device, batch);
}

bool rows_ok(const Tensor& t, c10::Device device) {
    return on(t, device, at::kHalf) && t.dim() == 4 && t.size(3) == kDim && t.stride(3) == 1 && aligned(t, 16) &&
           step(t, 0) % 8 == 0 && step(t, 1) % 8 == 0 && step(t, 2) % 8 == 0;
}

PyObject* status(int rc, const char* what) {
    if (rc > 0) PyErr_Format(PyExc_RuntimeError, "%s: CUDA error %d at launch", what, rc);
    if (rc != 0) return rc > 0 ? nullptr : Py_NewRef(Py_None);      // a refusal: the caller says which
    return Py_NewRef(Py_True);
}

const int32_t* ints(const Tensor* t) { return t ? static_cast<const int32_t*>(t->const_data_ptr()) : nullptr; }

// decode(q, pool, tables, lens, out | None, scale, part address, seg address, chunks, min_chunk, flags)
PyObject* decode(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    const Tensor *q = n == 11 ? tensor(a[0]) : nullptr, *pool = q ? tensor(a[1]) : nullptr;
    const Tensor *tables = q ? tensor(a[2]) : nullptr, *lens = q ? tensor(a[3]) : nullptr;
    if (!q || !pool || !tables || !lens || !q->is_cuda() || q->dim() != 4) Py_RETURN_NONE;
    const c10::Device device = q->device();
    const int64_t b = q->size(0), h = q->size(1), r = q->size(2);
    if (!on(*q, device, at::kHalf) || q->size(3) != kDim || q->stride(3) != 1 || r < 1 || r > 8 || b < 1 || b > 1024 ||
        h < 1 || !aligned(*q, 16) || q->stride(0) % 8 || q->stride(1) % 8 || q->stride(2) % 8 ||
        !pool_ok(*pool, device, h) || !tables_ok(*tables, *lens, device, b))
        Py_RETURN_NONE;
    Tensor out;
    if (a[4] == Py_None) {
        out = at::empty_like(*q, at::MemoryFormat::Contiguous);
    } else {
        const Tensor* given = tensor(a[4]);
        if (!given || !on(*given, device, at::kHalf) || given->sizes() != q->sizes() || given->stride(3) != 1 ||
            !aligned(*given, 8) || given->stride(0) % 4 || given->stride(1) % 4 || given->stride(2) % 4)
            Py_RETURN_NONE;
        out = *given;
    }
    void* stream;
    if (!stream_of(device, &stream)) Py_RETURN_NONE;
    const double scale = PyFloat_AsDouble(a[5]);
    void *part = PyLong_AsVoidPtr(a[6]), *seg = PyLong_AsVoidPtr(a[7]);
    const long chunks = PyLong_AsLong(a[8]), min_chunk = PyLong_AsLong(a[9]), flags = PyLong_AsLong(a[10]);
    if (PyErr_Occurred()) return nullptr;
    const int rc = f_decode(q->const_data_ptr(), pool->const_data_ptr(), ints(tables), ints(lens), static_cast<float*>(part),
                            static_cast<int32_t*>(seg), out.data_ptr(), b, h, r, groups_of(*pool), kDim, kPage,
                            tables->size(1), pool->size(0), chunks, min_chunk, flags, q->stride(0), q->stride(1),
                            q->stride(2), pool->stride(0), pool->stride(1), out.stride(0), out.stride(1), out.stride(2),
                            static_cast<float>(scale), stream);
    PyObject* ok = status(rc, "paged_decode_int4");
    if (ok != Py_True) return ok;
    Py_DECREF(ok);
    return a[4] == Py_None ? THPVariable_Wrap(std::move(out)) : Py_NewRef(a[4]);
    END_HANDLE_TH_ERRORS
}

// write(k, v, pool, tables, lens, new_lens | None)
PyObject* write(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    const Tensor* t[6] = {};
    if (n != 6) Py_RETURN_NONE;
    for (int i = 0; i < 6; ++i)
        if (!(t[i] = tensor(a[i])) && !(i == 5 && a[i] == Py_None)) Py_RETURN_NONE;
    const Tensor &k = *t[0], &v = *t[1], &pool = *t[2], &tables = *t[3], &lens = *t[4];
    if (!k.is_cuda() || k.dim() != 4) Py_RETURN_NONE;
    const c10::Device device = k.device();
    const int64_t b = k.size(0);
    if (!rows_ok(k, device) || !rows_ok(v, device) || v.sizes() != k.sizes() || k.numel() == 0 || b > 65535 ||
        k.size(2) > (1 << 30) || !pool_ok(pool, device, k.size(1)) || !tables_ok(tables, lens, device, b) ||
        (t[5] && !vector_ok(*t[5], device, b)))
        Py_RETURN_NONE;
    void* stream;
    if (!stream_of(device, &stream)) Py_RETURN_NONE;
    return status(f_write(k.const_data_ptr(), v.const_data_ptr(), pool.data_ptr(), ints(&tables), ints(&lens), ints(t[5]), b,
                          k.size(1), k.size(2), groups_of(pool), kDim, kPage, tables.size(1), pool.size(0), step(k, 0),
                          step(k, 1), step(k, 2), step(v, 0), step(v, 1), step(v, 2), pool.stride(0), pool.stride(1), stream),
                  "int4 write");
    END_HANDLE_TH_ERRORS
}

// read(pool, tables, lens, length, start | None) -> (k, v)
PyObject* read(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    const Tensor *pool = n == 5 ? tensor(a[0]) : nullptr, *tables = pool ? tensor(a[1]) : nullptr;
    const Tensor *lens = pool ? tensor(a[2]) : nullptr, *start = pool ? tensor(a[4]) : nullptr;
    if (!pool || !tables || !lens || (!start && a[4] != Py_None) || !PyLong_CheckExact(a[3])) Py_RETURN_NONE;
    if (!pool->is_cuda() || pool->dim() != 3 || lens->dim() != 1) Py_RETURN_NONE;
    const c10::Device device = pool->device();
    const int64_t b = lens->size(0), h = pool->size(1);
    int overflow = 0;
    const long long length = PyLong_AsLongLongAndOverflow(a[3], &overflow);
    if (overflow || length < 1 || length > (1 << 30) || b < 1 || b > 65535 || !pool_ok(*pool, device, h) ||
        !tables_ok(*tables, *lens, device, b) || (start && !vector_ok(*start, device, b)))
        Py_RETURN_NONE;
    void* stream;
    if (!stream_of(device, &stream)) Py_RETURN_NONE;
    const auto options = pool->options().dtype(at::kHalf);
    Tensor k = at::empty({b, h, length, kDim}, options), v = at::empty({b, h, length, kDim}, options);
    const int64_t sb = h * length * kDim, sh = length * kDim;
    PyObject* ok = status(f_read(pool->const_data_ptr(), k.data_ptr(), v.data_ptr(), ints(tables), ints(lens), ints(start), b, h,
                                 length, groups_of(*pool), kDim, kPage, tables->size(1), pool->size(0), sb, sh, kDim, sb, sh,
                                 kDim, pool->stride(0), pool->stride(1), stream),
                          "int4 read");
    if (ok != Py_True) return ok;
    Py_DECREF(ok);
    PyObject* pair = PyTuple_New(2);
    if (!pair) return nullptr;
    PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(std::move(k)));
    PyTuple_SET_ITEM(pair, 1, THPVariable_Wrap(std::move(v)));
    return pair;
    END_HANDLE_TH_ERRORS
}

bool page_ids(PyObject* o, std::vector<int32_t>& out) {
    if (!PyList_CheckExact(o)) return false;
    const Py_ssize_t n = PyList_GET_SIZE(o);
    out.resize(n);
    for (Py_ssize_t i = 0; i < n; ++i) {
        PyObject* x = PyList_GET_ITEM(o, i);
        int overflow = 0;
        const long v = PyLong_CheckExact(x) ? PyLong_AsLongAndOverflow(x, &overflow) : -1;
        if (overflow || v < 0 || v > INT32_MAX) return false;
        out[i] = static_cast<int32_t>(v);
    }
    return true;
}

// copy_pages(list of pools, list of ids, list of ids, block_dim)
PyObject* copy_pages(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 4 || !PyList_CheckExact(a[0]) || !PyLong_CheckExact(a[3])) Py_RETURN_NONE;
    const long axis = PyLong_AsLong(a[3]);
    const Py_ssize_t count = PyList_GET_SIZE(a[0]);
    if (axis < 0 || axis > 1 || count < 1 || count > 4096) Py_RETURN_NONE;
    std::vector<ls_page_pool> pools(count);
    const Tensor* first = tensor(PyList_GET_ITEM(a[0], 0));
    if (!first || !first->is_cuda() || first->dim() <= axis) Py_RETURN_NONE;
    const int64_t blocks = first->size(axis);
    for (Py_ssize_t i = 0; i < count; ++i) {
        const Tensor* t = tensor(PyList_GET_ITEM(a[0], i));
        if (!t || !t->is_cuda() || t->device() != first->device() || t->layout() != at::kStrided || t->dim() <= axis ||
            t->size(axis) != blocks)
            Py_RETURN_NONE;
        int64_t run = 1;
        for (int64_t d = t->dim() - 1; d > axis; --d) {
            if (t->size(d) != 1 && t->stride(d) != run) Py_RETURN_NONE;
            run *= t->size(d);
        }
        const int64_t size = t->element_size(), layers = axis ? t->size(0) : 1;
        if (run * size < 1 || run * size > INT32_MAX || layers < 1 || layers > INT32_MAX) Py_RETURN_NONE;
        pools[i] = {t->data_ptr(), axis ? t->stride(0) * size : 0, t->stride(axis) * size, static_cast<int32_t>(run * size),
                    static_cast<int32_t>(layers)};
    }
    std::vector<int32_t> src, dst;
    if (blocks < 1 || blocks > INT32_MAX || !page_ids(a[1], src) || !page_ids(a[2], dst) || src.size() != dst.size())
        Py_RETURN_NONE;
    void* stream;
    if (!stream_of(first->device(), &stream)) Py_RETURN_NONE;
    return status(f_copy(pools.data(), count, src.data(), dst.data(), src.size(), blocks, stream), "copy_pages");
    END_HANDLE_TH_ERRORS
}

// rotary(q, k, cos, sin, positions, interleaved, inverse, q_out | None, k_out | None) -> (q_out, k_out)
PyObject* rotary(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 9) Py_RETURN_NONE;
    const Tensor* t[5];
    for (int i = 0; i < 5; ++i)
        if (!(t[i] = tensor(a[i]))) Py_RETURN_NONE;
    const Tensor &q = *t[0], &k = *t[1], &cos = *t[2], &sin = *t[3], &pos = *t[4];
    if (!q.is_cuda() || q.dim() != 3 || k.dim() != 3 || cos.dim() != 2 || sin.dim() != 2 || pos.dim() != 1) Py_RETURN_NONE;
    const c10::Device device = q.device();
    const at::ScalarType type = q.scalar_type();
    const int kind = type == at::kHalf ? 0 : type == at::kBFloat16 ? 1 : type == at::kFloat ? 2 : -1;
    const int64_t tokens = q.size(0), dim = q.size(2), rot = 2 * cos.size(1);
    auto rows = [&](const Tensor& x) {
        return on(x, device, type) && x.dim() == 3 && x.size(0) == tokens && x.size(2) == dim &&
               (dim == 1 || x.stride(2) == 1) && x.size(1) <= 65536;
    };
    if (kind < 0 || !rows(q) || !rows(k) || tokens < 1 || tokens > INT32_MAX || q.size(1) + k.size(1) < 1 || dim > 65536 ||
        !on(cos, device, at::kFloat) || !on(sin, device, at::kFloat) || cos.sizes() != sin.sizes() ||
        cos.strides() != sin.strides() || rot < 2 || rot > dim || cos.size(0) < 1 || (rot > 2 && cos.stride(1) != 1) ||
        (cos.size(0) > 1 && cos.stride(0) < cos.size(1)) || !on(pos, device, at::kLong) || pos.size(0) != tokens ||
        (tokens > 1 && pos.stride(0) != 1))
        Py_RETURN_NONE;
    Tensor out[2];
    for (int i = 0; i < 2; ++i) {
        const Tensor& x = *t[i];
        if (a[7 + i] == Py_None) {
            out[i] = at::empty_like(x, at::MemoryFormat::Contiguous);
            continue;
        }
        const Tensor* given = tensor(a[7 + i]);
        if (!given || !rows(*given) || given->size(1) != x.size(1)) Py_RETURN_NONE;
        for (int d = 0; d < 3; ++d)
            if (given->size(d) > 1 && given->stride(d) == 0) Py_RETURN_NONE;
        if (x.numel() && given->const_data_ptr() == x.const_data_ptr() && (step(*given, 0) != step(x, 0) || step(*given, 1) != step(x, 1)))
            Py_RETURN_NONE;
        out[i] = *given;
    }
    void* stream;
    if (!stream_of(device, &stream)) Py_RETURN_NONE;
    PyObject* ok = status(
        f_rotary(q.const_data_ptr(), k.const_data_ptr(), out[0].data_ptr(), out[1].data_ptr(),
                 static_cast<const float*>(cos.const_data_ptr()), static_cast<const float*>(sin.const_data_ptr()),
                 static_cast<const int64_t*>(pos.const_data_ptr()), tokens, q.size(1), k.size(1), dim, rot, kind,
                 PyObject_IsTrue(a[5]) == 1, PyObject_IsTrue(a[6]) == 1, cos.size(0),
                 cos.size(0) > 1 ? cos.stride(0) : cos.size(1), step(q, 0), step(q, 1), step(k, 0), step(k, 1),
                 step(out[0], 0), step(out[0], 1), step(out[1], 0), step(out[1], 1), stream),
        "apply_rotary");
    if (ok != Py_True) return ok;
    Py_DECREF(ok);
    PyObject* pair = PyTuple_New(2);
    if (!pair) return nullptr;
    for (int i = 0; i < 2; ++i)
        PyTuple_SET_ITEM(pair, i, a[7 + i] == Py_None ? THPVariable_Wrap(std::move(out[i])) : Py_NewRef(a[7 + i]));
    return pair;
    END_HANDLE_TH_ERRORS
}

// bind(addresses of ls_paged_decode_int4, ls_int4_write, ls_int4_read, ls_copy_pages, ls_rotary)
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
    void* f[5];
    if (n != 5) {
        PyErr_SetString(PyExc_TypeError, "bind takes five addresses");
        return nullptr;
    }
    for (int i = 0; i < 5; ++i) {
        f[i] = PyLong_AsVoidPtr(a[i]);
        if (!f[i]) {
            if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "bind was given a null address");
            return nullptr;
        }
    }
    f_decode = reinterpret_cast<decltype(f_decode)>(f[0]);
    f_write = reinterpret_cast<decltype(f_write)>(f[1]);
    f_read = reinterpret_cast<decltype(f_read)>(f[2]);
    f_copy = reinterpret_cast<decltype(f_copy)>(f[3]);
    f_rotary = reinterpret_cast<decltype(f_rotary)>(f[4]);
    Py_RETURN_NONE;
}

#define LS_METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {LS_METHOD(bind), LS_METHOD(decode), LS_METHOD(write), LS_METHOD(read),
                         LS_METHOD(copy_pages), LS_METHOD(rotary), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "ls_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_ls_binding() { return PyModule_Create(&module); }
