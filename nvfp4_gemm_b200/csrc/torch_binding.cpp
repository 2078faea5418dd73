// CPython module between torch tensors and the C ABI (include/nvfp4_b200.h): turns the operator's
// 7-tuple (template.py:9-18 in the reference project) into struct nvfp4_problem and makes the call on
// torch's current stream.
//
// What bounds a small matmul is the time to issue it: the kernel launch itself takes the CPU
// 2.3-2.5 us.  The translation reads about forty sizes and strides; through Python attributes and
// ctypes a call took 11-12 us (128 x 256 x 256: 10.3 us a pass although the kernel runs for 3.3 us),
// and a table of translated tuples by address does not help a caller whose tensors are new.  From C++
// the same reads take well under a microsecond, so nothing is remembered between calls (128 x 256 x 256:
// 3.75 us a pass; a first call on new tensors 28.5 -> 17.6 us, waited for).
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstring>
#include <exception>
#include <initializer_list>

#include "../../include/nvfp4_b200.h"

namespace {

struct PythonError {};   // a Python exception is set

[[noreturn]] void raise(PyObject* type, const char* text) {
    PyErr_SetString(type, text);
    throw PythonError{};
}

// A tensor of the tuple, or null for None.
const at::Tensor* tensor_or_none(PyObject* o) {
    if (o == Py_None) return nullptr;
    if (!THPVariable_Check(o)) {
        PyErr_Format(PyExc_TypeError, "expected a tensor, got %s", Py_TYPE(o)->tp_name);
        throw PythonError{};
    }
    return &THPVariable_Unpack(o);
}

int64_t batch_stride(const at::Tensor& t, int64_t dim) {
    if (t.dim() <= dim) raise(PyExc_IndexError, "tensor has no batch dimension");
    return t.size(dim) > 1 ? t.stride(dim) : 0;
}

struct Operands {
    PyObject* seq;            // keeps the tensors alive
    const at::Tensor* t[7];   // a, b, sfa, sfb, sfa_permuted, sfb_permuted, c; the last five may be null
    explicit Operands(PyObject* data) : seq(PySequence_Fast(data, "expected (a, b, sfa, sfb, sfa_permuted, sfb_permuted, c)")) {
        if (!seq) throw PythonError{};
        try {
            if (PySequence_Fast_GET_SIZE(seq) != 7) raise(PyExc_ValueError, "expected seven values: (a, b, sfa, sfb, sfa_permuted, sfb_permuted, c)");
            for (int i = 0; i < 7; ++i) t[i] = tensor_or_none(PySequence_Fast_GET_ITEM(seq, i));
            if (!t[0] || !t[1]) raise(PyExc_TypeError, "a and b must be tensors");
        } catch (const PythonError&) {
            Py_DECREF(seq);
            throw;
        }
    }
    ~Operands() { Py_DECREF(seq); }
    Operands(const Operands&) = delete;
    Operands& operator=(const Operands&) = delete;
    void require_cuda() const {
        for (const at::Tensor* x : t)
            if (x && !x->is_cuda()) raise(PyExc_ValueError, "custom_kernel needs CUDA tensors (there is no CPU fallback)");
    }
};

nvfp4_problem make_problem(const Operands& o) {
    const at::Tensor &a = *o.t[0], &b = *o.t[1];
    const at::Tensor* c = o.t[6];
    if (a.dim() != 3 || b.dim() != 3 || (c && c->dim() != 3)) raise(PyExc_ValueError, "a, b and c must have three dimensions (rows, columns, batch)");
    const int64_t m = a.size(0), k_bytes = a.size(1), l = a.size(2), n = b.size(0);
    if (b.size(1) != k_bytes || b.size(2) != l) {
        PyErr_Format(PyExc_ValueError, "a (%lld, %lld, %lld) and b (%lld, %lld, %lld) disagree on k or l", (long long)m, (long long)k_bytes,
                     (long long)l, (long long)n, (long long)b.size(1), (long long)b.size(2));
        throw PythonError{};
    }
    if (c && (c->size(0) != m || c->size(1) != n || c->size(2) != l)) {
        PyErr_Format(PyExc_ValueError, "c has shape (%lld, %lld, %lld), expected (%lld, %lld, %lld)", (long long)c->size(0), (long long)c->size(1),
                     (long long)c->size(2), (long long)m, (long long)n, (long long)l);
        throw PythonError{};
    }
    if (m > INT32_MAX || n > INT32_MAX || k_bytes > INT32_MAX / 2 || l > INT32_MAX) raise(PyExc_ValueError, "sizes must fit 32 bits");
    if (a.stride(1) != 1 || b.stride(1) != 1 || (c && c->stride(1) != 1 && n > 1))
        raise(PyExc_ValueError, "a, b must be K-major (stride 1 along k) and c row-major");
    bool types = a.element_size() == 1 && b.element_size() == 1 && (!c || c->scalar_type() == at::kHalf);
    for (int i = 2; i < 6; ++i) types = types && (!o.t[i] || o.t[i]->element_size() == 1);
    if (!types) raise(PyExc_ValueError, "expected packed fp4 (1 byte per 2 values), 1-byte scales and fp16 output");

    nvfp4_problem p;
    std::memset(&p, 0, sizeof(p));
    p.a = a.data_ptr();
    p.b = b.data_ptr();
    p.c = c ? c->data_ptr() : nullptr;
    p.m = static_cast<int32_t>(m);
    p.n = static_cast<int32_t>(n);
    p.k = static_cast<int32_t>(2 * k_bytes);
    p.l = static_cast<int32_t>(l);
    p.a_row_stride = a.stride(0);
    p.a_batch_stride = batch_stride(a, 2);
    p.b_row_stride = n > 1 ? b.stride(0) : k_bytes;
    p.b_batch_stride = batch_stride(b, 2);
    if (const at::Tensor* s = o.t[2]) {
        p.sfa = s->data_ptr();
        p.sfa_batch_stride = batch_stride(*s, 2);
        p.sfa_row_stride = s->stride(0);
    }
    if (const at::Tensor* s = o.t[3]) {
        p.sfb = s->data_ptr();
        p.sfb_batch_stride = batch_stride(*s, 2);
        p.sfb_row_stride = n > 1 ? s->stride(0) : k_bytes / 8;
    }
    // permuted scales: [32, 4, rest_rows, 4, rest_k, L]; the batch is the last dimension
    if (const at::Tensor* s = o.t[4]) {
        p.sfa_perm = s->data_ptr();
        p.sfa_perm_batch_stride = batch_stride(*s, 5);
    }
    if (const at::Tensor* s = o.t[5]) {
        p.sfb_perm = s->data_ptr();
        p.sfb_perm_batch_stride = batch_stride(*s, 5);
    }
    if (c) {
        p.c_row_stride = c->stride(0);
        p.c_batch_stride = batch_stride(*c, 2);
    }
    return p;
}

// Calls f(stream) with the tensors' device current, on torch's current stream of that device and
// without the interpreter lock (a launch waits when the queue of the device is full).  Only f, which
// answers with a status and throws nothing, runs unlocked: the guard and the stream throw where CUDA reports an error, and
// an exception that left with the lock released would be turned into a Python one without a thread state.
template <class F>
int on_current_stream(const at::Tensor& a, F f) {
    const c10::DeviceIndex dev = a.device().index();
    const c10::cuda::CUDAGuard guard(dev);
    void* stream = c10::cuda::getCurrentCUDAStream(dev).stream();
    int rc = 0;
    Py_BEGIN_ALLOW_THREADS
    rc = f(stream);
    Py_END_ALLOW_THREADS
    return rc;
}

template <class F>
PyObject* guarded(F f) {
    try {
        return f();
    } catch (const PythonError&) {
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}

// matmul(data) -> status of nvfp4_matmul
PyObject* py_matmul(PyObject*, PyObject* data) {
    return guarded([&] {
        const Operands o(data);
        o.require_cuda();
        const nvfp4_problem p = make_problem(o);
        return PyLong_FromLong(on_current_stream(*o.t[0], [&](void* stream) { return nvfp4_matmul(&p, stream); }));
    });
}

// fill_problem(data, address): writes struct nvfp4_problem at `address`
PyObject* py_fill_problem(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        if (n != 2) raise(PyExc_TypeError, "fill_problem(data, address)");
        void* dst = PyLong_AsVoidPtr(args[1]);
        if (!dst) {
            if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "address is NULL");
            throw PythonError{};
        }
        const nvfp4_problem p = make_problem(Operands(args[0]));
        std::memcpy(dst, &p, sizeof(p));
        Py_RETURN_NONE;
    });
}

int int_arg(PyObject* o) {
    const long v = PyLong_AsLong(o);
    if (v == -1 && PyErr_Occurred()) throw PythonError{};
    if (v < INT32_MIN || v > INT32_MAX) raise(PyExc_OverflowError, "argument does not fit 32 bits");
    return static_cast<int>(v);
}

// gemm_epilogue(data, bias, activation, out, tile_n, grid, cta_group, split_k[, residual]) -> status of
// nvfp4_gemm_epilogue, or of nvfp4_gemm_residual.  out: None for fp16 into data[6], else (packed, sf, sf_permuted) with dense rows.
PyObject* py_gemm_epilogue(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    return guarded([&] {
        if (nargs != 8 && nargs != 9) raise(PyExc_TypeError, "gemm_epilogue(data, bias, activation, out, tile_n, grid, cta_group, split_k[, residual])");
        const Operands o(args[0]);
        o.require_cuda();
        if (args[3] == Py_None && !o.t[6]) raise(PyExc_ValueError, "an fp16 output needs data[6]");
        const nvfp4_problem p = make_problem(o);
        nvfp4_epilogue e;
        std::memset(&e, 0, sizeof(e));
        if (const at::Tensor* bias = tensor_or_none(args[1])) {
            if (bias->device() != o.t[0]->device()) raise(PyExc_ValueError, "bias must be on the device of a");
            if (bias->scalar_type() != at::kHalf || bias->numel() != p.n || !bias->is_contiguous())
                raise(PyExc_ValueError, "bias must be a contiguous fp16 vector of length n");
            e.bias = bias->data_ptr();
        }
        e.activation = int_arg(args[2]);
        if (args[3] != Py_None) {
            struct Sequence {          // any sequence will do
                PyObject* seq;
                ~Sequence() { Py_XDECREF(seq); }
            } const out{PySequence_Fast(args[3], "out must be (packed, sf, sf_permuted)")};
            if (!out.seq) throw PythonError{};
            if (PySequence_Fast_GET_SIZE(out.seq) < 3) raise(PyExc_IndexError, "out must be (packed, sf, sf_permuted)");
            const int64_t m = p.m, n = p.n;
            const int64_t needed[3] = {p.l * m * (n / 2), p.l * m * (n / 16), p.l * ((m + 127) / 128) * (n / 64) * 512};
            void* ptr[3];
            for (int i = 0; i < 3; ++i) {
                const at::Tensor* t = tensor_or_none(PySequence_Fast_GET_ITEM(out.seq, i));
                if (!t) raise(PyExc_TypeError, "out must be (packed, sf, sf_permuted)");
                if (t->device() != o.t[0]->device()) raise(PyExc_ValueError, "out must be on the device of a");
                if (t->element_size() != 1 || t->numel() < needed[i] || !t->is_non_overlapping_and_dense())
                    raise(PyExc_ValueError, "out must be dense 1-byte tensors that hold the packed result, its scales and their permuted form");
                ptr[i] = t->data_ptr();
            }
            e.output = NVFP4_OUT_NVFP4;
            e.out_packed = ptr[0];
            e.out_sf = ptr[1];
            e.out_sf_perm = ptr[2];
            e.out_packed_row_stride = n / 2;
            e.out_packed_batch_stride = m * (n / 2);
            e.out_sf_row_stride = n / 16;
            e.out_sf_batch_stride = m * (n / 16);
            e.out_sf_perm_batch_stride = ((m + 127) / 128) * (n / 64) * 512;
        }
        nvfp4_gemm_config cfg = {int_arg(args[4]), 0, int_arg(args[5]), int_arg(args[6]), int_arg(args[7]), 0};
        if (const at::Tensor* r = nargs == 9 ? tensor_or_none(args[8]) : nullptr) {
            if (!r->is_cuda() || r->device() != o.t[0]->device()) raise(PyExc_ValueError, "residual must be on the device of a");
            if (r->scalar_type() != at::kHalf || r->dim() != 3 || r->size(0) != p.m || r->size(1) != p.n || r->size(2) != p.l || r->stride(1) != 1)
                raise(PyExc_ValueError, "residual must be fp16 (m, n, l), row-major");
            const void* const add = r->data_ptr();
            const int64_t row = p.m > 1 ? r->stride(0) : p.n, batch = batch_stride(*r, 2);
            return PyLong_FromLong(on_current_stream(*o.t[0], [&](void* stream) { return nvfp4_gemm_residual(&p, &cfg, &e, add, row, batch, stream); }));
        }
        return PyLong_FromLong(on_current_stream(*o.t[0], [&](void* stream) { return nvfp4_gemm_epilogue(&p, &cfg, &e, stream); }));
    });
}

// ------------------------------------------------------------------------------------- mixture of experts
// Each call checks its tensors, allocates its results and answers with them, or with the status (an int) where the C ABI refused.

const at::Tensor& tensor_arg(PyObject* o, const char* name) {
    if (!THPVariable_Check(o)) {
        PyErr_Format(PyExc_TypeError, "%s must be a tensor, got %s", name, Py_TYPE(o)->tp_name);
        throw PythonError{};
    }
    return THPVariable_Unpack(o);
}

[[noreturn]] void raise_value(const char* fmt, const char* name) {
    PyErr_Format(PyExc_ValueError, fmt, name);
    throw PythonError{};
}

// `t` lives on the device of `on` (a CUDA device).
void same_device(const at::Tensor& t, const at::Tensor& on, const char* name) {
    if (!on.is_cuda() || !t.is_cuda()) raise(PyExc_ValueError, "the experts' operators need CUDA tensors (there is no CPU fallback)");
    if (t.device() != on.device()) raise_value("%s is on another device than the first tensor", name);
}

int32_t size_arg(int64_t v, const char* name) {
    if (v > INT32_MAX) raise_value("%s does not fit 32 bits", name);
    return static_cast<int32_t>(v);
}

// A [rows, columns] tensor whose rows are contiguous.
void rows_of(const at::Tensor& t, const char* name) {
    if (t.dim() != 2 || (t.size(1) > 1 && t.stride(1) != 1)) raise_value("%s must have two dimensions, the second contiguous", name);
}
int64_t row_stride(const at::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

// Results of a call: tensors of their own on one allocation from torch's allocator (current device and stream), which lives as long
// as any of them.  Straight from the allocator: an at::empty() for each took longer than a small kernel runs.
class Slab {
public:
    explicit Slab(int64_t bytes)
        : storage_(c10::Storage::use_byte_size_t(), static_cast<size_t>(bytes), c10::cuda::CUDACachingAllocator::get()->allocate(static_cast<size_t>(bytes)),
                   c10::cuda::CUDACachingAllocator::get(), false) {}
    static int64_t room(int64_t bytes) { return (bytes + 255) & ~int64_t{255}; }
    at::Tensor take(at::IntArrayRef sizes, at::ScalarType type) {
        auto impl = c10::make_intrusive<c10::TensorImpl>(c10::Storage(storage_), c10::DispatchKeySet(c10::DispatchKey::CUDA), c10::scalarTypeToTypeMeta(type));
        const int64_t item = static_cast<int64_t>(c10::elementSize(type));
        impl->set_storage_offset(used_ / item);
        impl->set_sizes_contiguous(sizes);
        used_ += room(c10::multiply_integers(sizes) * item);
        return at::Tensor(std::move(impl));
    }

private:
    c10::Storage storage_;
    int64_t used_ = 0;
};
// (with the tensors' device current)
at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType type) {
    return Slab(c10::multiply_integers(sizes) * static_cast<int64_t>(c10::elementSize(type))).take(sizes, type);
}

PyObject* status_object(int rc) { return PyLong_FromLong(rc); }

// (a number, if given, behind the tensors)
PyObject* pack(std::initializer_list<at::Tensor> tensors, int64_t number = -1) {
    PyObject* out = PyTuple_New(static_cast<Py_ssize_t>(tensors.size()) + (number >= 0));
    if (!out) throw PythonError{};
    Py_ssize_t i = 0;
    for (const at::Tensor& t : tensors) {
        PyObject* o = THPVariable_Wrap(t);
        if (!o) {
            Py_DECREF(out);
            throw PythonError{};
        }
        PyTuple_SET_ITEM(out, i++, o);
    }
    if (number >= 0) {
        PyObject* o = PyLong_FromLongLong(number);
        if (!o) {
            Py_DECREF(out);
            throw PythonError{};
        }
        PyTuple_SET_ITEM(out, i, o);
    }
    return out;
}

// The routing that belongs to choices of this shape, with new memory for what is not given.
struct Routing {
    nvfp4_routing r;
    int64_t sf_rows = 0;
    at::Tensor row, offset, plan;
    int status;
    at::Tensor expert, weight;
    // new rows, offsets and plan for [tokens, top_k] choices, and the choices and their weights too (choose)
    Routing(int64_t tokens, int64_t top_k, int64_t experts, bool choose) {
        int64_t plan_bytes = 0;
        status = size(tokens, top_k, experts, &plan_bytes);
        if (status) return;
        const int64_t per_pair = Slab::room(tokens * top_k * 4);
        Slab slab(per_pair * (choose ? 3 : 1) + Slab::room((experts + 1) * 4) + Slab::room(plan_bytes));
        row = slab.take({tokens, top_k}, at::kInt);
        offset = slab.take({experts + 1}, at::kInt);
        plan = slab.take({plan_bytes / 4}, at::kInt);
        if (choose) {
            expert = slab.take({tokens, top_k}, at::kInt);
            weight = slab.take({tokens, top_k}, at::kFloat);
            r.expert = expert.data_ptr<int32_t>();
        }
        r.row = row.data_ptr<int32_t>();
        r.offset = offset.data_ptr<int32_t>();
        r.plan = plan.data_ptr();
    }
    // the rows and plan of an earlier call
    Routing(const at::Tensor& on, PyObject* rows, PyObject* plan_o, PyObject* experts) {
        row = tensor_arg(rows, "rows");
        plan = tensor_arg(plan_o, "plan");
        same_device(row, on, "rows");
        same_device(plan, on, "plan");
        if (row.dim() != 2 || row.scalar_type() != at::kInt || !row.is_contiguous() || plan.scalar_type() != at::kInt || !plan.is_contiguous())
            raise(PyExc_ValueError, "rows and plan must be what route() or plan() returned (contiguous int32)");
        int64_t plan_bytes = 0;
        const long long e = PyLong_AsLongLong(experts);
        if (e == -1 && PyErr_Occurred()) throw PythonError{};
        status = size(row.size(0), row.size(1), e, &plan_bytes);
        if (status) return;
        if (plan.numel() * 4 != plan_bytes) raise(PyExc_ValueError, "plan does not belong to rows of this shape and to this number of experts");
        r.row = row.data_ptr<int32_t>();
        r.plan = plan.data_ptr();
    }

private:
    int size(int64_t tokens, int64_t top_k, int64_t experts, int64_t* plan_bytes) {
        std::memset(&r, 0, sizeof(r));
        r.tokens = size_arg(tokens, "the number of tokens");
        r.top_k = size_arg(top_k, "top_k");
        r.experts = size_arg(experts, "the number of experts");
        return nvfp4_routing_plan(r.tokens, r.top_k, r.experts, nullptr, plan_bytes, &sf_rows);
    }
};

double float_arg(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw PythonError{};
    return v;
}

// route(logits, top_k, scoring, bias, groups, top_groups, group_top, renormalize, scale) -> (experts, weights, rows, offsets, plan, number of experts)
PyObject* py_route(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    return guarded([&]() -> PyObject* {
        if (nargs != 9) raise(PyExc_TypeError, "route(logits, top_k, scoring, bias, groups, top_groups, group_top, renormalize, scale)");
        const at::Tensor& logits = tensor_arg(args[0], "logits");
        same_device(logits, logits, "logits");
        rows_of(logits, "logits");
        nvfp4_router o;
        std::memset(&o, 0, sizeof(o));
        if (logits.scalar_type() == at::kFloat) o.logits_type = NVFP4_LOGITS_FP32;
        else if (logits.scalar_type() == at::kBFloat16) o.logits_type = NVFP4_LOGITS_BF16;
        else if (logits.scalar_type() == at::kHalf) o.logits_type = NVFP4_LOGITS_FP16;
        else raise(PyExc_ValueError, "logits must be fp16, bf16 or fp32");
        const int top_k = int_arg(args[1]);
        o.scoring = int_arg(args[2]);
        if (const at::Tensor* bias = tensor_or_none(args[3])) {
            same_device(*bias, logits, "bias");
            if (bias->scalar_type() != at::kFloat || bias->dim() != 1 || bias->size(0) != logits.size(1) || !bias->is_contiguous())
                raise(PyExc_ValueError, "bias must be a contiguous fp32 vector with an entry per expert");
            o.bias = bias->data_ptr<float>();
        }
        o.groups = int_arg(args[4]);
        o.top_groups = int_arg(args[5]);
        o.group_top = int_arg(args[6]);
        o.renormalize = int_arg(args[7]);
        o.scale = static_cast<float>(float_arg(args[8]));
        const c10::cuda::CUDAGuard guard(logits.device());
        Routing routing(logits.size(0), top_k, logits.size(1), true);
        if (routing.status) return status_object(routing.status);
        o.logits = logits.data_ptr();
        o.logits_row_stride = row_stride(logits);
        o.weights = routing.weight.data_ptr<float>();
        const int rc = on_current_stream(logits, [&](void* stream) { return nvfp4_route(&o, &routing.r, stream); });
        return rc ? status_object(rc) : pack({routing.expert, routing.weight, routing.row, routing.offset, routing.plan}, logits.size(1));
    });
}

// plan(experts, number of experts) -> (rows, offsets, plan)
PyObject* py_plan(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    return guarded([&]() -> PyObject* {
        if (nargs != 2) raise(PyExc_TypeError, "plan(experts, number of experts)");
        const at::Tensor& experts = tensor_arg(args[0], "experts");
        same_device(experts, experts, "experts");
        if (experts.dim() != 2 || experts.scalar_type() != at::kInt || !experts.is_contiguous())
            raise(PyExc_ValueError, "experts must be a contiguous int32 tensor [tokens, top_k]");
        const c10::cuda::CUDAGuard guard(experts.device());
        Routing routing(experts.size(0), experts.size(1), int_arg(args[1]), false);
        if (routing.status) return status_object(routing.status);
        routing.r.expert = experts.data_ptr<int32_t>();
        const int rc = on_current_stream(experts, [&](void* stream) { return nvfp4_plan_experts(&routing.r, stream); });
        return rc ? status_object(rc) : pack({routing.row, routing.offset, routing.plan});
    });
}

// quantize_routed(x, rows, plan, number of experts) -> (packed, sf)
PyObject* py_quantize_routed(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    return guarded([&]() -> PyObject* {
        if (nargs != 4) raise(PyExc_TypeError, "quantize_routed(x, rows, plan, number of experts)");
        const at::Tensor& x = tensor_arg(args[0], "x");
        same_device(x, x, "x");
        rows_of(x, "x");
        if (x.scalar_type() != at::kHalf && x.scalar_type() != at::kBFloat16) raise(PyExc_ValueError, "x must be fp16 or bf16");
        const c10::cuda::CUDAGuard guard(x.device());
        Routing routing(x, args[1], args[2], args[3]);
        if (routing.status) return status_object(routing.status);
        if (routing.r.tokens != x.size(0)) raise(PyExc_ValueError, "x must have a row per token of the routing");
        const int64_t k = size_arg(x.size(1), "the width of x");
        const int64_t rows = routing.row.numel();
        Slab slab(Slab::room(rows * (k / 2)) + Slab::room(routing.sf_rows * (k / 16)));
        const at::Tensor packed = slab.take({rows, k / 2}, at::kFloat4_e2m1fn_x2), sf = slab.take({routing.sf_rows * (k / 16)}, at::kFloat8_e4m3fn);
        const void* const src = x.data_ptr();
        void *const codes = packed.data_ptr(), *const scales = sf.data_ptr();
        const bool bf16 = x.scalar_type() == at::kBFloat16;
        const int64_t stride = row_stride(x);
        const int rc = on_current_stream(
            x, [&](void* stream) { return nvfp4_quantize_routed(src, bf16, stride, static_cast<int32_t>(k), &routing.r, codes, k / 2, scales, stream); });
        return rc ? status_object(rc) : pack({packed, sf});
    });
}

// expert_gemm(packed, sf, rows, plan, number of experts, w, w_sf_permuted, alpha, bias, activation, out_scale, nvfp4_out, out)
//   -> (y,) or (packed, sf)
PyObject* py_expert_gemm(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    return guarded([&]() -> PyObject* {
        if (nargs != 13)
            raise(PyExc_TypeError, "expert_gemm(packed, sf, rows, plan, number of experts, w, w_sf_permuted, alpha, bias, activation, out_scale, nvfp4_out, out)");
        const at::Tensor &a = tensor_arg(args[0], "packed"), &sfa = tensor_arg(args[1], "sf");
        const at::Tensor &w = tensor_arg(args[5], "w"), &sfw = tensor_arg(args[6], "w_sf_permuted");
        same_device(a, a, "packed");
        same_device(sfa, a, "sf");
        same_device(w, a, "w");
        same_device(sfw, a, "w_sf_permuted");
        const c10::cuda::CUDAGuard guard(a.device());
        Routing routing(a, args[2], args[3], args[4]);
        if (routing.status) return status_object(routing.status);
        const int64_t experts = routing.r.experts, rows = routing.row.numel();
        rows_of(a, "packed");
        if (w.dim() != 3 || w.stride(1) != 1) raise(PyExc_ValueError, "w must be [n, k / 2, experts] with the second dimension contiguous");
        const int64_t n = w.size(0), kb = w.size(1), rest_n = (n + 127) / 128, rest_k = kb / 32;
        if (a.element_size() != 1 || w.element_size() != 1 || sfa.element_size() != 1 || sfw.element_size() != 1)
            raise(PyExc_ValueError, "expected packed fp4 (1 byte per 2 values) and 1-byte scales");
        if (a.size(0) != rows || a.size(1) != kb || w.size(2) != experts) raise(PyExc_ValueError, "packed, w and the routing disagree on rows, k or experts");
        if (!sfa.is_contiguous() || sfa.numel() != routing.sf_rows * (kb / 8)) raise(PyExc_ValueError, "sf is not the scales of a routed operand of this routing and k");
        const int64_t sizes[6] = {32, 4, rest_n, 4, rest_k, experts}, strides[5] = {16, 4, rest_k * 512, 1, 512};
        bool fits = sfw.dim() == 6;
        for (int i = 0; fits && i < 6; ++i) fits = sfw.size(i) == sizes[i] && (i == 5 || sizes[i] == 1 || sfw.stride(i) == strides[i]);
        if (!fits) raise(PyExc_ValueError, "w_sf_permuted must be [32, 4, n / 128, 4, k / 64, experts] in 512-byte atoms");
        nvfp4_expert_problem p;
        std::memset(&p, 0, sizeof(p));
        if (const at::Tensor* t = tensor_or_none(args[7])) {
            same_device(*t, a, "alpha");
            if (t->scalar_type() != at::kFloat || t->dim() != 1 || t->size(0) != experts || !t->is_contiguous())
                raise(PyExc_ValueError, "alpha must be a contiguous fp32 vector with an entry per expert");
            p.alpha = t->data_ptr<float>();
        }
        if (const at::Tensor* t = tensor_or_none(args[8])) {
            same_device(*t, a, "bias");
            if (t->scalar_type() != at::kHalf || t->dim() != 2 || t->size(0) != experts || t->size(1) != n || (n > 1 && t->stride(1) != 1))
                raise(PyExc_ValueError, "bias must be fp16 [experts, n] with contiguous rows");
            p.bias = t->data_ptr();
            p.bias_expert_stride = t->size(0) > 1 ? t->stride(0) : n;
        }
        p.activation = int_arg(args[9]);
        p.out_scale = static_cast<float>(float_arg(args[10]));
        const bool to_nvfp4 = int_arg(args[11]) != 0;
        const int64_t n_out = p.activation == NVFP4_ACT_SWIGLU ? n / 2 : n;
        p.a = a.data_ptr();
        p.sfa = sfa.data_ptr();
        p.w = w.data_ptr();
        p.sfw_perm = sfw.data_ptr();
        p.n = size_arg(n, "n");
        p.k = size_arg(2 * kb, "k");
        p.a_row_stride = rows > 1 ? a.stride(0) : kb;
        p.w_row_stride = w.stride(0);
        p.w_expert_stride = w.stride(2);
        p.sfw_perm_expert_stride = sfw.stride(5);
        at::Tensor out, out_sf;
        if (to_nvfp4) {
            if (args[12] != Py_None) raise(PyExc_ValueError, "out is for the fp16 result");
            Slab slab(Slab::room(rows * (n_out / 2)) + Slab::room(routing.sf_rows * (n_out / 16)));
            out = slab.take({rows, n_out / 2}, at::kFloat4_e2m1fn_x2);
            out_sf = slab.take({routing.sf_rows * (n_out / 16)}, at::kFloat8_e4m3fn);
            p.output = NVFP4_OUT_NVFP4;
            p.out_row_stride = n_out / 2;
            p.out_sf = out_sf.data_ptr();
        } else if (const at::Tensor* t = tensor_or_none(args[12])) {
            same_device(*t, a, "out");
            rows_of(*t, "out");
            if (t->scalar_type() != at::kHalf || t->size(0) != rows || t->size(1) != n_out) raise(PyExc_ValueError, "out must be fp16 [tokens * top_k, columns]");
            out = *t;
            p.out_row_stride = row_stride(out);
        } else {
            out = fresh({rows, n_out}, at::kHalf);
            p.out_row_stride = n_out;
        }
        p.out = out.data_ptr();
        const int rc = on_current_stream(a, [&](void* stream) { return nvfp4_expert_gemm(&p, &routing.r, stream); });
        if (rc) return status_object(rc);
        return to_nvfp4 ? pack({out, out_sf}) : pack({out});
    });
}

// combine(y, rows, weights, residual, out, bf16) -> (out,)
PyObject* py_combine(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    return guarded([&]() -> PyObject* {
        if (nargs != 6) raise(PyExc_TypeError, "combine(y, rows, weights, residual, out, bf16)");
        const at::Tensor &y = tensor_arg(args[0], "y"), &rows = tensor_arg(args[1], "rows"), &weights = tensor_arg(args[2], "weights");
        same_device(y, y, "y");
        same_device(rows, y, "rows");
        same_device(weights, y, "weights");
        rows_of(y, "y");
        if (y.scalar_type() != at::kHalf) raise(PyExc_ValueError, "y must be fp16");
        if (rows.dim() != 2 || rows.scalar_type() != at::kInt || !rows.is_contiguous()) raise(PyExc_ValueError, "rows must be contiguous int32 [tokens, top_k]");
        if (weights.sizes() != rows.sizes() || weights.scalar_type() != at::kFloat || !weights.is_contiguous())
            raise(PyExc_ValueError, "weights must be contiguous fp32 of the shape of rows");
        const int64_t tokens = rows.size(0), n = y.size(1);
        const at::ScalarType type = int_arg(args[5]) ? at::kBFloat16 : at::kHalf;
        const at::Tensor* residual = tensor_or_none(args[3]);
        const at::Tensor* given = tensor_or_none(args[4]);
        const char* const names[2] = {"residual", "out"};
        for (int i = 0; i < 2; ++i)
            if (const at::Tensor* t = i ? given : residual) {
                same_device(*t, y, names[i]);
                rows_of(*t, names[i]);
                if (t->size(0) != tokens || t->size(1) != n || t->scalar_type() != type) raise_value("%s must be [tokens, n] of the output's type", names[i]);
            }
        const c10::cuda::CUDAGuard guard(y.device());
        const at::Tensor out = given ? *given : fresh({tokens, n}, type);
        const int32_t y_rows = size_arg(y.size(0), "y"), t = size_arg(tokens, "the number of tokens"), top_k = size_arg(rows.size(1), "top_k"), cols = size_arg(n, "n");
        const void *const src = y.data_ptr(), *const add = residual ? residual->data_ptr() : nullptr;
        const int32_t* const row = rows.data_ptr<int32_t>();
        const float* const weight = weights.data_ptr<float>();
        void* const dst = out.data_ptr();
        const int64_t y_stride = row_stride(y), add_stride = residual ? row_stride(*residual) : 0, out_stride = row_stride(out);
        const int rc = on_current_stream(y, [&](void* stream) {
            return nvfp4_combine_experts(src, y_stride, y_rows, row, weight, t, top_k, cols, add, add_stride, dst, out_stride, type == at::kBFloat16, stream);
        });
        return rc ? status_object(rc) : pack({out});
    });
}

// Read from the file by nvfp4_gemm_b200/build.py: the types of torch and Python that this code has the layouts of.
[[gnu::used]] const char built_for[] = "nvfp4_native built for: " NVFP4_BUILT_FOR;

PyMethodDef methods[] = {
    {"matmul", py_matmul, METH_O, "matmul(data) -> status"},
    {"fill_problem", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_fill_problem)), METH_FASTCALL, "fill_problem(data, address)"},
    {"gemm_epilogue", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_gemm_epilogue)), METH_FASTCALL,
     "gemm_epilogue(data, bias, activation, out, tile_n, grid, cta_group, split_k[, residual]) -> status"},
    {"route", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_route)), METH_FASTCALL,
     "route(logits, top_k, scoring, bias, groups, top_groups, group_top, renormalize, scale) -> (experts, weights, rows, offsets, plan, number of experts) or status"},
    {"plan", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_plan)), METH_FASTCALL, "plan(experts, number of experts) -> (rows, offsets, plan) or status"},
    {"quantize_routed", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_quantize_routed)), METH_FASTCALL,
     "quantize_routed(x, rows, plan, number of experts) -> (packed, sf) or status"},
    {"expert_gemm", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_expert_gemm)), METH_FASTCALL,
     "expert_gemm(packed, sf, rows, plan, number of experts, w, w_sf_permuted, alpha, bias, activation, out_scale, nvfp4_out, out) -> (y,), (packed, sf) or status"},
    {"combine", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_combine)), METH_FASTCALL, "combine(y, rows, weights, residual, out, bf16) -> (out,) or status"},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_native", "torch tensors to the C ABI of libnvfp4_b200", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__native() { return PyModule_Create(&module); }
