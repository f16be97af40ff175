// paged_python.cpp -- the calls of secure_infer_b200/paged.py that run for every
// layer and step, as a CPython extension: it looks the tensors over, makes the
// outputs and calls the C ABI (include/secure_infer_paged.h).  The same through
// ctypes took 11 us of host time for an append whose kernel takes 3.
//
// Handles come as the addresses of the structures that the Python objects hold,
// the stream as its handle.  Refused arguments raise ValueError, refused
// launches RuntimeError.
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/Exceptions.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>

#include <string>

#include "../../include/secure_infer_paged.h"

namespace {

constexpr int64_t kDim = SECURE_INFER_HEAD_DIM;

struct Refused {
    std::string why;
};

void need(bool ok, const char* why)
{
    if (!ok) throw Refused{why};
}

const at::Tensor& tensor(PyObject* o, const char* what)
{
    if (!THPVariable_Check(o)) throw Refused{std::string(what) + " must be a tensor"};
    return THPVariable_Unpack(o);
}

template <typename P>
P* address(PyObject* o)
{
    return static_cast<P*>(PyLong_AsVoidPtr(o));
}

bool aligned(const at::Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0; }

at::ScalarType type_of(const secure_infer_pages* p) { return p->dtype == SECURE_INFER_FP16 ? at::kHalf : at::kBFloat16; }

struct Rows {
    void* data;
    int64_t heads, token, head;   // and strides
};

// [tokens, heads, 128] of a type on a device.
Rows rows(const at::Tensor& t, const char* what, int64_t tokens, at::ScalarType type, int64_t device)
{
    const auto bad = [&](const char* why) { throw Refused{std::string(what) + why}; };
    if (t.dim() != 3 || t.size(0) != tokens || t.size(2) != kDim) bad(" must be [tokens, heads, 128]");
    if (t.scalar_type() != type || !t.is_cuda() || t.get_device() != device) bad(" must have the cache's type and device");
    Rows r{t.data_ptr(), t.size(1), tokens > 1 ? t.stride(0) : kDim, t.size(1) > 1 ? t.stride(1) : kDim};
    if (t.stride(2) != 1 || r.token <= 0 || r.head <= 0 || ((r.token | r.head) & 7) || !aligned(t))
        bad(": a head's values must be adjacent, the address and strides multiples of 16 bytes");
    return r;
}

at::Tensor output(PyObject* given, const at::Tensor& like)
{
    if (given == Py_None) return at::empty_like(like, at::MemoryFormat::Contiguous);
    const at::Tensor& t = tensor(given, "out");
    need(t.sizes() == like.sizes() && t.scalar_type() == like.scalar_type() && t.device() == like.device() &&
             t.is_contiguous() && aligned(t),
         "out must be dense, with q's shape, type and device");
    return t;
}

const int32_t* ints(const at::Tensor& t, int64_t dims, int64_t device, const char* why)
{
    need(t.scalar_type() == at::kInt && t.dim() == dims && t.is_cuda() && t.get_device() == device &&
             (t.numel() == 0 || t.stride(-1) == 1),
         why);
    return static_cast<const int32_t*>(t.data_ptr());
}

PyObject* failed(const char* name)
{
    PyErr_Format(PyExc_RuntimeError, "%s refused its arguments or failed to launch", name);
    return nullptr;
}

// Exceptions of the body become Python's.
template <class Body>
PyObject* guarded(Body body)
{
    try {
        return body();
    } catch (const Refused& r) {
        PyErr_SetString(PyExc_ValueError, r.why.c_str());
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}

bool counted(Py_ssize_t n, Py_ssize_t want)
{
    if (n == want) return true;
    PyErr_Format(PyExc_TypeError, "%zd arguments, not %zd", want, n);
    return false;
}

// attend(pages, chunk, device, q, out, return_lse, scale, causal, window, workspace, stream)
PyObject* attend(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    if (!counted(n, 11)) return nullptr;
    return guarded([&]() -> PyObject* {
        const auto* pages = address<const secure_infer_pages>(a[0]);
        secure_infer_chunk chunk = *address<const secure_infer_chunk>(a[1]);
        const int64_t device = PyLong_AsLongLong(a[2]);
        const at::Tensor& q = tensor(a[3], "q");
        const int64_t tokens = q.dim() > 0 ? q.size(0) : 0;
        const Rows r = rows(q, "q", tokens, type_of(pages), device);
        need(r.heads > 0 && r.heads % pages->heads == 0, "q's heads must be a multiple of the cache's");
        const double scale = PyFloat_AsDouble(a[6]);
        const int causal = PyObject_IsTrue(a[7]);
        const int64_t window = PyLong_AsLongLong(a[8]);
        if (PyErr_Occurred()) return nullptr;
        need(window >= 0 && window < int64_t(1) << 31 && (window == 0 || causal),
             "window must be zero or positive, and goes with causal");
        at::Tensor out = output(a[4], q), lse;
        const bool want_lse = PyObject_IsTrue(a[5]);
        if (want_lse) lse = at::empty({tokens, r.heads}, q.options().dtype(at::kFloat));
        if (tokens > 0) {
            const at::Tensor& workspace = tensor(a[9], "workspace");
            need(workspace.is_cuda() && workspace.get_device() == device && workspace.is_contiguous() &&
                     (reinterpret_cast<uintptr_t>(workspace.data_ptr()) & 255) == 0 &&
                     static_cast<uint64_t>(workspace.nbytes()) >= secure_infer_paged_attend_workspace(),
                 "workspace must come from attend_workspace of the cache's device");
            need(tokens <= UINT32_MAX, "too many tokens");
            chunk.tokens = static_cast<uint32_t>(tokens);
            if (secure_infer_paged_attend(pages, &chunk, r.data, r.token, r.head, static_cast<uint32_t>(r.heads),
                                          out.data_ptr(), want_lse ? static_cast<float*>(lse.data_ptr()) : nullptr,
                                          static_cast<float>(scale), causal, static_cast<uint32_t>(window),
                                          workspace.data_ptr(), address<void>(a[10])) != 0)
                return failed("secure_infer_paged_attend");
        }
        if (!want_lse) return THPVariable_Wrap(std::move(out));
        PyObject* first = THPVariable_Wrap(std::move(out));
        PyObject* second = THPVariable_Wrap(std::move(lse));
        PyObject* both = first != nullptr && second != nullptr ? PyTuple_Pack(2, first, second) : nullptr;
        Py_XDECREF(first);
        Py_XDECREF(second);
        return both;
    });
}

// append(pages, chunk, device, q, k, v, phase, axis, axes, interleaved, positions, out, stream)
PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    if (!counted(n, 13)) return nullptr;
    return guarded([&]() -> PyObject* {
        const auto* pages = address<const secure_infer_pages>(a[0]);
        secure_infer_chunk chunk = *address<const secure_infer_chunk>(a[1]);
        const int64_t device = PyLong_AsLongLong(a[2]);
        const at::Tensor &kt = tensor(a[4], "k"), &vt = tensor(a[5], "v");
        const int64_t tokens = kt.dim() > 0 ? kt.size(0) : 0;
        const at::ScalarType type = type_of(pages);
        const Rows k = rows(kt, "k", tokens, type, device), v = rows(vt, "v", tokens, type, device);
        need(k.heads == pages->heads && v.heads == k.heads, "k and v must have the cache's heads");
        Rows q{};
        at::Tensor out;
        if (a[3] != Py_None) {
            const at::Tensor& qt = tensor(a[3], "q");
            q = rows(qt, "q", tokens, type, device);
            out = output(a[11], qt);
        } else {
            need(a[11] == Py_None, "out goes with q");
        }
        const auto* phase = address<const uint64_t>(a[6]);
        const auto* axis = address<const uint32_t>(a[7]);
        const int64_t axes = PyLong_AsLongLong(a[8]);
        const int interleaved = PyObject_IsTrue(a[9]);
        if (PyErr_Occurred()) return nullptr;
        const int32_t* positions = nullptr;
        int64_t position_stride = 0;
        if (a[10] != Py_None) {
            need(phase != nullptr, "positions go with rotary");
            const at::Tensor& t = tensor(a[10], "positions");
            const bool flat = t.dim() == 1;
            need((flat && axes == 1 && t.size(0) == tokens) || (t.dim() == 2 && t.size(0) == axes && t.size(1) == tokens),
                 "positions must be [axes, tokens]");
            positions = ints(t, t.dim(), device, "positions must be int32 of the cache's device, dense along the tokens");
            position_stride = axes > 1 ? t.stride(0) : tokens;
            need(position_stride >= 0, "positions has a negative stride");
        }
        if (tokens > 0) {
            need(tokens <= UINT32_MAX, "too many tokens");
            chunk.tokens = static_cast<uint32_t>(tokens);
            if (secure_infer_paged_append(pages, &chunk, q.data, q.token, q.head, static_cast<uint32_t>(q.heads),
                                          out.defined() ? out.data_ptr() : nullptr, k.data, k.token, k.head, v.data, v.token,
                                          v.head, phase, axis, positions, position_stride, static_cast<uint32_t>(axes),
                                          interleaved, address<void>(a[12])) != 0)
                return failed("secure_infer_paged_append");
        }
        if (!out.defined()) Py_RETURN_NONE;
        return THPVariable_Wrap(std::move(out));
    });
}

// free(block_table, lens, refs, pages, device, seqs, stream): new tables of the same shapes.
PyObject* free_sequences(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    if (!counted(n, 7)) return nullptr;
    return guarded([&]() -> PyObject* {
        const at::Tensor &table = tensor(a[0], "block_table"), &lens = tensor(a[1], "lens"), &refs = tensor(a[2], "refs");
        const int64_t pages = PyLong_AsLongLong(a[3]), device = PyLong_AsLongLong(a[4]);
        if (PyErr_Occurred()) return nullptr;
        secure_infer_tables in{}, out{};
        in.block_table = const_cast<int32_t*>(ints(table, 2, device, "block_table must be int32 [seqs, width] of the cache's device"));
        in.lens = const_cast<int32_t*>(ints(lens, 1, device, "lens must be int32 [seqs] of the cache's device"));
        in.refs = const_cast<int32_t*>(ints(refs, 1, device, "refs must be int32 [pages] of the cache's device"));
        need(table.is_contiguous() && lens.is_contiguous() && refs.is_contiguous(), "tables must be dense");
        need(table.size(0) > 0 && table.size(1) > 0 && table.size(0) <= UINT32_MAX && table.size(1) <= UINT32_MAX,
             "block_table is empty");
        need(lens.size(0) == table.size(0) && refs.size(0) == pages,
             "lens needs an entry for each row of the block table, refs one for each page");
        const at::Tensor& seqs = tensor(a[5], "seqs");
        const int32_t* ended = ints(seqs, 1, device, "seqs must be an int32 tensor of the cache's device");
        need(seqs.size(0) <= INT32_MAX, "too many requests");
        in.seqs = static_cast<uint32_t>(table.size(0));
        in.width = static_cast<uint32_t>(table.size(1));
        in.pages = static_cast<uint32_t>(pages);
        out = in;
        at::Tensor t = at::empty_like(table), l = at::empty_like(lens), r = at::empty_like(refs);
        out.block_table = static_cast<int32_t*>(t.data_ptr());
        out.lens = static_cast<int32_t*>(l.data_ptr());
        out.refs = static_cast<int32_t*>(r.data_ptr());
        const uint32_t count = static_cast<uint32_t>(seqs.size(0));
        at::Tensor scratch = at::empty({static_cast<int64_t>(secure_infer_paged_scratch(&in, count) / 4)}, table.options());
        if (secure_infer_paged_free(&in, &out, ended, count, scratch.data_ptr(), address<void>(a[6])) != 0)
            return failed("secure_infer_paged_free");
        PyObject* parts[3] = {THPVariable_Wrap(std::move(t)), THPVariable_Wrap(std::move(l)), THPVariable_Wrap(std::move(r))};
        PyObject* all = parts[0] && parts[1] && parts[2] ? PyTuple_Pack(3, parts[0], parts[1], parts[2]) : nullptr;
        for (PyObject* o : parts) Py_XDECREF(o);
        return all;
    });
}

PyMethodDef methods[] = {
    {"attend", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(attend)), METH_FASTCALL, nullptr},
    {"append", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(append)), METH_FASTCALL, nullptr},
    {"free", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(free_sequences)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "paged_python", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_paged_python(void) { return PyModule_Create(&module); }
