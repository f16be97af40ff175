// paged_python.cpp -- the calls of secure_infer_b200/paged.py as a CPython
// extension: it looks the tensors over, makes the outputs and calls the C ABI
// (include/secure_infer_paged.h).  The same through ctypes took 11 us of host
// time for an append whose kernel takes 3.
//
// Handles come as the addresses of the structures that the Python objects hold,
// the stream as its handle.  Refused arguments raise ValueError, refused
// launches RuntimeError.
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/Exceptions.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>

#include <algorithm>
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

// Exceptions of the body become Python's, torch's own as they do elsewhere in torch.
template <class Body>
PyObject* guarded(Body body)
{
    HANDLE_TH_ERRORS
    try {
        return body();
    } catch (const Refused& r) {
        PyErr_SetString(PyExc_ValueError, r.why.c_str());
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

bool counted(Py_ssize_t n, Py_ssize_t want)
{
    if (n == want) return true;
    PyErr_Format(PyExc_TypeError, "%zd arguments, not %zd", want, n);
    return false;
}

PyObject* pair(at::Tensor a, at::Tensor b)
{
    PyObject* first = THPVariable_Wrap(std::move(a));
    PyObject* second = THPVariable_Wrap(std::move(b));
    PyObject* both = first != nullptr && second != nullptr ? PyTuple_Pack(2, first, second) : nullptr;
    Py_XDECREF(first);
    Py_XDECREF(second);
    return both;
}

// attend(pages, chunk, device, q, out, return_lse, scale, causal, window, workspace, stream), and perhaps (sinks, plan
// of a shared prefix or None, its groups, most tokens in common)
PyObject* attend(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    if (n != 11 && !counted(n, 15)) return nullptr;
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
        secure_infer_attend_options options{};
        at::Tensor parts;
        if (n > 11) {
            const int64_t sinks = PyLong_AsLongLong(a[11]), groups = PyLong_AsLongLong(a[13]), most = PyLong_AsLongLong(a[14]);
            if (PyErr_Occurred()) return nullptr;
            need(sinks >= 0 && sinks < int64_t(1) << 31 && (sinks == 0 || window > 0),
                 "sinks must be zero or positive, and go with a window");
            options.sinks = static_cast<uint32_t>(sinks);
            if (a[12] != Py_None) {
                need(window == 0, "a shared prefix does not go with a window");
                need(groups > 0 && groups <= chunk.seqs, "a shared prefix has one group for each sequence at most");
                const at::Tensor& plan = tensor(a[12], "the shared prefix's plan");
                options.groups = static_cast<uint32_t>(groups);
                options.max_common = static_cast<uint32_t>(std::min<int64_t>(std::max<int64_t>(most, 0), UINT32_MAX));
                options.plan = ints(plan, 1, device, "the shared prefix must be on the cache's device");
                need(static_cast<uint64_t>(plan.numel()) >= secure_infer_shared_prefix_ints(chunk.seqs, options.groups) &&
                         aligned(plan), "the shared prefix is another chunk's");
            }
        }
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
            if (const uint64_t bytes = options.groups > 0 ? secure_infer_attend_parts(pages, &chunk, r.heads, &options) : 0; bytes > 0) {
                parts = at::empty({static_cast<int64_t>(bytes / sizeof(float))}, q.options().dtype(at::kFloat));
                options.parts = static_cast<float*>(parts.data_ptr());
            }
            if (secure_infer_attend(pages, &chunk, r.data, r.token, r.head, static_cast<uint32_t>(r.heads), out.data_ptr(),
                                    want_lse ? static_cast<float*>(lse.data_ptr()) : nullptr, static_cast<float>(scale),
                                    causal, static_cast<uint32_t>(window), &options, workspace.data_ptr(),
                                    address<void>(a[10])) != 0) {
                need(secure_infer_attend_fits_window(pages, &chunk, static_cast<uint32_t>(r.heads), static_cast<uint32_t>(window),
                                                     options.sinks),
                     "more work than one call takes: fewer tokens, or a narrower block table");
                return failed("secure_infer_attend");
            }
        }
        return want_lse ? pair(std::move(out), std::move(lse)) : THPVariable_Wrap(std::move(out));
    });
}

// join(outs, lses, device, out, stream)
PyObject* join(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    if (!counted(n, 5)) return nullptr;
    return guarded([&]() -> PyObject* {
        need(PyTuple_Check(a[0]) && PyTuple_Check(a[1]), "outs and lses must be tuples of tensors");
        const Py_ssize_t count = PyTuple_GET_SIZE(a[0]);
        need(count > 0 && count <= static_cast<Py_ssize_t>(SECURE_INFER_JOIN_PARTS) && PyTuple_GET_SIZE(a[1]) == count,
             "outs and lses must be one to eight tensors each, as many of both");
        const int64_t device = PyLong_AsLongLong(a[2]);
        if (PyErr_Occurred()) return nullptr;
        const at::Tensor& like = tensor(PyTuple_GET_ITEM(a[0], 0), "an output");
        const at::ScalarType type = like.scalar_type();
        need(type == at::kHalf || type == at::kBFloat16, "outputs are bf16 or fp16");
        const int64_t tokens = like.dim() > 0 ? like.size(0) : 0;
        secure_infer_attend_part parts[SECURE_INFER_JOIN_PARTS];
        int64_t heads = 0;
        for (Py_ssize_t i = 0; i < count; ++i) {
            const at::Tensor& o = tensor(PyTuple_GET_ITEM(a[0], i), "an output");
            need(o.dim() == 3 && o.sizes() == like.sizes() && o.scalar_type() == type && o.is_cuda() && o.get_device() == device,
                 "the outputs differ in shape, type or device");
            const Rows r = rows(o, "an output", tokens, type, device);
            const at::Tensor& l = tensor(PyTuple_GET_ITEM(a[1], i), "a logarithm of sums");
            need(l.dim() == 2 && l.size(0) == tokens && l.size(1) == r.heads && l.scalar_type() == at::kFloat && l.is_cuda() &&
                     l.get_device() == device && l.stride(0) >= 0 && l.stride(1) >= 0,
                 "lses must be float32 [tokens, heads] of the outputs' device");
            heads = r.heads;
            parts[i] = {r.data, static_cast<const float*>(l.data_ptr()), {r.token, r.head}, {l.stride(0), l.stride(1)}};
        }
        need(heads > 0 && heads <= 1 << 16 && tokens <= 1 << 28 && tokens * heads <= int64_t(1) << 34, "more rows than one call takes");
        at::Tensor out = output(a[3], like);
        // Rows are read before they are written, so a part may be written over, but not by its neighbours.
        const char* begin = static_cast<const char*>(out.data_ptr());
        for (Py_ssize_t i = 0; i < count && a[3] != Py_None && tokens > 0; ++i) {
            const char* from = static_cast<const char*>(parts[i].out);
            const int64_t span = ((tokens - 1) * parts[i].out_stride[0] + (heads - 1) * parts[i].out_stride[1] + kDim) * 2;
            const bool same = from == begin && (heads == 1 || parts[i].out_stride[1] == kDim) &&
                              (tokens == 1 || parts[i].out_stride[0] == heads * kDim);
            need(same || from + span <= begin || begin + out.nbytes() <= from, "out overlaps a part");
            const char* sums = reinterpret_cast<const char*>(parts[i].lse);
            const int64_t end = ((tokens - 1) * parts[i].lse_stride[0] + (heads - 1) * parts[i].lse_stride[1] + 1) * 4;
            need(sums + end <= begin || begin + out.nbytes() <= sums, "out overlaps a part");
        }
        at::Tensor lse = at::empty({tokens, heads}, like.options().dtype(at::kFloat));
        if (secure_infer_attend_join(parts, static_cast<uint32_t>(count), static_cast<uint32_t>(tokens),
                                     static_cast<uint32_t>(heads),
                                     type == at::kHalf ? SECURE_INFER_FP16 : SECURE_INFER_BF16, out.data_ptr(),
                                     static_cast<float*>(lse.data_ptr()), address<void>(a[4])) != 0)
            return failed("secure_infer_attend_join");
        return pair(std::move(out), std::move(lse));
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

struct Tables {
    at::Tensor table, lens, refs;
    secure_infer_tables c;
};

// block_table, lens and refs of a cache of `pages`.
Tables tables(PyObject* const* a, int64_t pages, int64_t device)
{
    Tables t{tensor(a[0], "block_table"), tensor(a[1], "lens"), tensor(a[2], "refs"), {}};
    t.c.block_table = const_cast<int32_t*>(ints(t.table, 2, device, "block_table must be int32 [seqs, width] of the cache's device"));
    t.c.lens = const_cast<int32_t*>(ints(t.lens, 1, device, "lens must be int32 [seqs] of the cache's device"));
    t.c.refs = const_cast<int32_t*>(ints(t.refs, 1, device, "refs must be int32 [pages] of the cache's device"));
    need(t.table.is_contiguous() && t.lens.is_contiguous() && t.refs.is_contiguous(), "tables must be dense");
    need(t.table.size(0) > 0 && t.table.size(1) > 0 && t.table.size(0) <= INT32_MAX && t.table.size(1) <= INT32_MAX,
         "block_table is empty");
    need(t.lens.size(0) == t.table.size(0) && t.refs.size(0) == pages,
         "lens needs an entry for each row of the block table, refs one for each page");
    t.c.seqs = static_cast<uint32_t>(t.table.size(0));
    t.c.width = static_cast<uint32_t>(t.table.size(1));
    t.c.pages = static_cast<uint32_t>(pages);
    return t;
}

// Part of a dense tensor from element `first` on, in a shape.
at::Tensor part_of(const at::Tensor& t, int64_t first, at::IntArrayRef sizes)
{
    at::Tensor part = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(t.storage()), t.key_set(), t.dtype());
    part.unsafeGetTensorImpl()->set_storage_offset(t.storage_offset() + first);
    part.unsafeGetTensorImpl()->set_sizes_contiguous(sizes);
    return part;
}

// New tables of the same shapes, or the given ones.
Tables outputs(PyObject* given, const Tables& in, int64_t pages, int64_t device)
{
    if (given == Py_None) {
        // In one piece of memory, each from a whole 256 bytes on: an allocation takes the host 1.0 us.
        const auto end = [](int64_t ints) { return (ints + 63) / 64 * 64; };
        const int64_t lens = end(in.table.numel()), refs = lens + end(in.lens.numel());
        const at::Tensor all = at::empty({refs + end(in.refs.numel())}, in.table.options());
        Tables t{part_of(all, 0, in.table.sizes()), part_of(all, lens, in.lens.sizes()), part_of(all, refs, in.refs.sizes()), in.c};
        t.c.block_table = static_cast<int32_t*>(t.table.data_ptr());
        t.c.lens = static_cast<int32_t*>(t.lens.data_ptr());
        t.c.refs = static_cast<int32_t*>(t.refs.data_ptr());
        return t;
    }
    need(PyTuple_Check(given) && PyTuple_GET_SIZE(given) == 3, "out must be PageTables");
    PyObject* parts[3] = {PyTuple_GET_ITEM(given, 0), PyTuple_GET_ITEM(given, 1), PyTuple_GET_ITEM(given, 2)};
    const Tables t = tables(parts, pages, device);
    need(t.table.sizes() == in.table.sizes(), "out differs in shape from the tables");
    const at::Tensor* outs[3] = {&t.table, &t.lens, &t.refs};
    for (const at::Tensor* a : {&in.table, &in.lens, &in.refs})
        for (const at::Tensor* b : outs) {
            const char *x = static_cast<const char*>(a->data_ptr()), *y = static_cast<const char*>(b->data_ptr());
            need(x + a->nbytes() <= y || y + b->nbytes() <= x, "out overlaps the tables");
        }
    for (int i = 0; i < 3; i++)
        for (int j = 0; j < i; j++) {
            const char *x = static_cast<const char*>(outs[i]->data_ptr()), *y = static_cast<const char*>(outs[j]->data_ptr());
            need(x + outs[i]->nbytes() <= y || y + outs[j]->nbytes() <= x, "out overlaps itself");
        }
    return t;
}

// Entries of a list of requests, as many in both.
uint32_t requests(const at::Tensor& a, const at::Tensor& b)
{
    need(a.size(0) == b.size(0), "the lists of requests differ in length");
    need(a.size(0) <= INT32_MAX, "too many requests");
    return static_cast<uint32_t>(a.size(0));
}

at::Tensor scratch_of(const Tables& t, uint32_t n)
{
    return at::empty({static_cast<int64_t>(secure_infer_paged_scratch(&t.c, n) / 4)}, t.table.options());
}

int32_t* data(const at::Tensor& t) { return static_cast<int32_t*>(t.data_ptr()); }

// (block_table, lens, refs, further tensors...)
PyObject* results(std::initializer_list<at::Tensor> tensors)
{
    PyObject* all = PyTuple_New(static_cast<Py_ssize_t>(tensors.size()));
    Py_ssize_t i = 0;
    for (const at::Tensor& t : tensors) {
        PyObject* o = all != nullptr ? THPVariable_Wrap(t) : nullptr;
        if (o == nullptr) {
            Py_XDECREF(all);
            return nullptr;
        }
        PyTuple_SET_ITEM(all, i++, o);
    }
    return all;
}

constexpr const char* kRequests = "requests must be int32 [n] of the cache's device";

// The operations on tables: (block_table, lens, refs, pages, device, their own arguments, stream, out), where `out` is
// None for new tables.

// fork(..., tensors, count, page bytes, parents, children, ...)
PyObject* fork_sequences(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    if (!counted(n, 12)) return nullptr;
    return guarded([&]() -> PyObject* {
        const int64_t pages = PyLong_AsLongLong(a[3]), device = PyLong_AsLongLong(a[4]);
        const auto* copied = address<const secure_infer_page_tensor>(a[5]);
        const int64_t count = PyLong_AsLongLong(a[6]), bytes = PyLong_AsLongLong(a[7]);
        if (PyErr_Occurred()) return nullptr;
        const Tables in = tables(a, pages, device), out = outputs(a[11], in, pages, device);
        const at::Tensor &parents = tensor(a[8], "parents"), &children = tensor(a[9], "children");
        const int32_t *p = ints(parents, 1, device, kRequests), *c = ints(children, 1, device, kRequests);
        const uint32_t asked = requests(parents, children);
        at::Tensor granted = at::empty({asked}, in.table.options()), scratch = scratch_of(in, asked);
        if (secure_infer_paged_fork(copied, static_cast<uint32_t>(count), static_cast<uint64_t>(bytes), &in.c, &out.c, p, c,
                                    asked, data(granted), scratch.data_ptr(), address<void>(a[10])) != 0)
            return failed("secure_infer_paged_fork");
        return results({out.table, out.lens, out.refs, granted});
    });
}

// reserve(..., seqs, lens, ...)
PyObject* reserve(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    if (!counted(n, 9)) return nullptr;
    return guarded([&]() -> PyObject* {
        const int64_t pages = PyLong_AsLongLong(a[3]), device = PyLong_AsLongLong(a[4]);
        if (PyErr_Occurred()) return nullptr;
        const Tables in = tables(a, pages, device), out = outputs(a[8], in, pages, device);
        const at::Tensor &seqs = tensor(a[5], "seqs"), &lens = tensor(a[6], "lens");
        const int32_t *s = ints(seqs, 1, device, kRequests), *l = ints(lens, 1, device, kRequests);
        const uint32_t asked = requests(seqs, lens);
        at::Tensor granted = at::empty({asked}, in.table.options()), scratch = scratch_of(in, asked);
        if (secure_infer_paged_reserve(&in.c, &out.c, s, l, asked, data(granted), scratch.data_ptr(), address<void>(a[7])) != 0)
            return failed("secure_infer_paged_reserve");
        return results({out.table, out.lens, out.refs, granted});
    });
}

// free(..., seqs, ...), `out` may be left out
PyObject* free_sequences(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    if (n != 7 && !counted(n, 8)) return nullptr;
    return guarded([&]() -> PyObject* {
        const int64_t pages = PyLong_AsLongLong(a[3]), device = PyLong_AsLongLong(a[4]);
        if (PyErr_Occurred()) return nullptr;
        const Tables in = tables(a, pages, device), out = outputs(n > 7 ? a[7] : Py_None, in, pages, device);
        const at::Tensor& seqs = tensor(a[5], "seqs");
        const int32_t* ended = ints(seqs, 1, device, kRequests);
        const uint32_t asked = requests(seqs, seqs);
        at::Tensor scratch = scratch_of(in, asked);
        if (secure_infer_paged_free(&in.c, &out.c, ended, asked, scratch.data_ptr(), address<void>(a[6])) != 0)
            return failed("secure_infer_paged_free");
        return results({out.table, out.lens, out.refs});
    });
}

// trim(..., seqs, window, sinks, ...)
PyObject* trim(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    if (!counted(n, 10)) return nullptr;
    return guarded([&]() -> PyObject* {
        const int64_t pages = PyLong_AsLongLong(a[3]), device = PyLong_AsLongLong(a[4]);
        const int64_t window = PyLong_AsLongLong(a[6]), sinks = PyLong_AsLongLong(a[7]);
        if (PyErr_Occurred()) return nullptr;
        need(window > 0 && window < int64_t(1) << 31, "window must be positive");
        need(sinks >= 0 && sinks < int64_t(1) << 31, "sinks must be zero or positive, and below 2^31");
        // As many as a table can hold keep every page.
        constexpr int64_t most = int64_t(1) << 30;
        const Tables in = tables(a, pages, device), out = outputs(a[9], in, pages, device);
        const at::Tensor& seqs = tensor(a[5], "seqs");
        const int32_t* named = ints(seqs, 1, device, kRequests);
        const uint32_t asked = requests(seqs, seqs);
        at::Tensor scratch = scratch_of(in, asked);
        if (secure_infer_trim(&in.c, &out.c, named, asked, static_cast<uint32_t>(window),
                              static_cast<uint32_t>(std::min(sinks, most)), scratch.data_ptr(), address<void>(a[8])) != 0)
            return failed("secure_infer_trim");
        return results({out.table, out.lens, out.refs});
    });
}

// compact(..., tensors, count, page bytes, ...)
PyObject* compact(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    if (!counted(n, 10)) return nullptr;
    return guarded([&]() -> PyObject* {
        const int64_t pages = PyLong_AsLongLong(a[3]), device = PyLong_AsLongLong(a[4]);
        const auto* copied = address<const secure_infer_page_tensor>(a[5]);
        const int64_t count = PyLong_AsLongLong(a[6]), bytes = PyLong_AsLongLong(a[7]);
        if (PyErr_Occurred()) return nullptr;
        const Tables in = tables(a, pages, device), out = outputs(a[9], in, pages, device);
        at::Tensor moved = at::empty({pages}, in.table.options()), live = at::empty({1}, in.table.options());
        at::Tensor scratch = scratch_of(in, 0);
        if (secure_infer_paged_compact(copied, static_cast<uint32_t>(count), static_cast<uint64_t>(bytes), &in.c, &out.c,
                                       data(moved), data(live), scratch.data_ptr(), address<void>(a[8])) != 0)
            return failed("secure_infer_paged_compact");
        return results({out.table, out.lens, out.refs, moved, live});
    });
}

// capture_id(stream)
PyObject* capture_id(PyObject*, PyObject* stream) { return PyLong_FromUnsignedLongLong(secure_infer_capture_id(address<void>(stream))); }

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyCFunction fast() { return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(F)); }

PyMethodDef methods[] = {
    {"attend", fast<attend>(), METH_FASTCALL, nullptr},
    {"append", fast<append>(), METH_FASTCALL, nullptr},
    {"join", fast<join>(), METH_FASTCALL, nullptr},
    {"trim", fast<trim>(), METH_FASTCALL, nullptr},
    {"fork", fast<fork_sequences>(), METH_FASTCALL, nullptr},
    {"reserve", fast<reserve>(), METH_FASTCALL, nullptr},
    {"free", fast<free_sequences>(), METH_FASTCALL, nullptr},
    {"compact", fast<compact>(), METH_FASTCALL, nullptr},
    {"capture_id", capture_id, METH_O, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "paged_python", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_paged_python(void) { return PyModule_Create(&module); }
