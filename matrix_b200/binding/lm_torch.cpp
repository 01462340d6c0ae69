// The torch side of matrix_b200.lm: checks a call's tensors, makes its outputs and hands both to the C ABI
// (include/mtxc.h).  Written against torch's C++ API and not ctypes because these operators serve single tokens:
// there the host's work is the call's whole cost (a block norm with its saved deviations took 21 us per call
// through ctypes).
//
// Every function takes its arguments by position (matrix_b200/lm.py names them) and returns a tuple of tensors
// and None, or the C ABI's status where that is not zero.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/cuda/EmptyTensor.h>
#include <ATen/ops/empty_like.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <optional>
#include <stdexcept>
#include <string>
#include <utility>

#include "mtxc.h"

namespace {

using Tensor = at::Tensor;
using invalid = std::invalid_argument;  // ValueError in Python

// ------------------------------------------------------------------------------------------
// Arguments
// ------------------------------------------------------------------------------------------
struct PythonError {};  // a Python exception is already set
struct Refused {        // by the C ABI
    int status;
};

const Tensor* maybe(PyObject* o, const char* what) {
    if (o == Py_None) return nullptr;
    if (!THPVariable_Check(o)) {
        PyErr_Format(PyExc_TypeError, "%s: expected a tensor", what);
        throw PythonError();
    }
    return &THPVariable_Unpack(o);
}

const Tensor& tensor(PyObject* o, const char* what) {
    const Tensor* t = maybe(o, what);
    if (!t) {
        PyErr_Format(PyExc_TypeError, "%s: expected a tensor", what);
        throw PythonError();
    }
    return *t;
}

double number(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw PythonError();
    return v;
}

bool flag(PyObject* o) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw PythonError();
    return v != 0;
}

uint64_t word(PyObject* o) {  // modulo 2^64
    const uint64_t v = PyLong_AsUnsignedLongLongMask(o);
    if (v == (uint64_t)-1 && PyErr_Occurred()) throw PythonError();
    return v;
}

std::string quoted(const char* what, const char* message) { return std::string(what) + ": " + message; }

// The C ABI's code, or -1, which it refuses.
int code_of(const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return MTXC_FLOAT;
        case at::kHalf: return MTXC_FLOAT16;
        case at::kBFloat16: return MTXC_BFLOAT16;
        case at::kInt: return MTXC_INT32;
        case at::kLong: return MTXC_INT64;
        case at::kShort: return MTXC_INT16;
        case at::kChar: return MTXC_INT8;
        case at::kByte: return MTXC_UINT8;
        case at::kBool: return MTXC_BOOL;
        default: return -1;
    }
}

// The CUDA device that all the tensors (NULL: absent) are on: the one that the thread is bound to, whose stream the
// kernels run on.
c10::DeviceIndex device_of(const Tensor& x, std::initializer_list<const Tensor*> others) {
    if (!x.is_cuda()) throw invalid("expected tensors on a CUDA device");
    for (const Tensor* t : others)
        if (t && (!t->is_cuda() || t->get_device() != x.get_device()))
            throw invalid("expected all tensors on the same CUDA device");
    int bound;
    if (const int status = mtxc_get_device(&bound)) throw Refused{status};
    if (x.get_device() != bound)
        throw invalid("expected tensors on cuda:" + std::to_string(bound) + ", the device that the thread is bound to");
    return (c10::DeviceIndex)bound;
}

// New tensors come from the memory of the stream that the kernels run on.
struct Memory {
    std::optional<c10::cuda::CUDAStreamGuard> guard;
    c10::Device device;
    explicit Memory(c10::DeviceIndex dev) : device(c10::kCUDA, dev) {
        cudaStream_t s = static_cast<cudaStream_t>(mtxc_get_stream());
        if (s != c10::cuda::getCurrentCUDAStream(dev).stream()) guard.emplace(c10::cuda::getStreamFromExternal(s, dev));
    }
    Tensor empty(c10::IntArrayRef shape, at::ScalarType type) const {
        return Tensor(at::detail::empty_cuda(shape, type, device, std::nullopt));
    }
    Tensor like(const Tensor& x) const { return empty(x.sizes(), x.scalar_type()); }
};

// The stride from row to row of a tensor whose leading axes fold into one.
uint64_t row_stride(const Tensor& t, const char* what, bool written = false) {
    const auto shape = t.sizes();
    const int64_t width = shape.back();
    if (t.is_contiguous()) return (uint64_t)width;
    const auto strides = t.strides();
    if (width > 1 && strides.back() != 1) throw invalid(quoted(what, "the last axis needs unit stride"));
    int64_t stride = width, span = -1;  // span: what the next axis out must have as its stride
    for (int64_t i = (int64_t)shape.size() - 2; i >= 0; --i) {
        if (shape[i] == 1) continue;
        if (span < 0) stride = strides[i], span = stride * shape[i];
        else if (strides[i] == span) span *= shape[i];
        else throw invalid(quoted(what, "its leading axes do not fold into rows at a constant stride"));
        if (written && stride < width) throw invalid(quoted(what, "its rows overlap"));
    }
    return (uint64_t)stride;
}

// A tensor that a call writes in place: raises its version, by which autograd notices that a saved tensor has changed.
const Tensor& written(const Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
    return t;
}

Tensor output(const Memory& memory, const Tensor& x, const Tensor* out, const char* what) {
    if (!out) return memory.like(x);
    if (out->sizes() != x.sizes() || out->scalar_type() != x.scalar_type() || !out->is_cuda() ||
        out->get_device() != x.get_device())
        throw invalid(quoted(what, "expected a tensor of the input's shape, dtype and device"));
    return written(*out);
}

void same(const Tensor* t, const Tensor& x, const char* what) {
    if (t && (t->sizes() != x.sizes() || t->scalar_type() != x.scalar_type()))
        throw invalid(quoted(what, "expected the residual's shape and dtype"));
}

struct Rows {
    int64_t rows, width;
    explicit Rows(const Tensor& x, const char* what) {
        if (x.dim() == 0) throw invalid(quoted(what, "expected rows"));
        width = x.size(-1);
        rows = width ? x.numel() / width : 0;
        if (!width) {
            rows = 1;
            for (int64_t i = 0; i + 1 < x.dim(); ++i) rows *= x.size(i);
        }
    }
};

mtxc_dropout_state drop_state(PyObject* p, PyObject* seed, PyObject* offset, PyObject* device_offset, c10::DeviceIndex dev) {
    mtxc_dropout_state s;
    s.p = number(p);
    s.seed = word(seed);
    s.offset = word(offset);
    s.device_offset = nullptr;
    if (const Tensor* t = maybe(device_offset, "device_offset")) {
        if ((t->scalar_type() != at::kLong && t->scalar_type() != at::kUInt64) || t->numel() != 1 || !t->is_cuda() ||
            t->get_device() != dev)
            throw invalid("device_offset: expected one 64-bit integer on the tensors' device");
        s.device_offset = static_cast<const uint64_t*>(t->const_data_ptr());
    }
    return s;
}

const void* at_or_null(const Tensor* t) { return t ? t->const_data_ptr() : nullptr; }
void* at_or_null(Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }

// A tuple of tensors, None for undefined ones; or the status.
template <typename... Ts>
PyObject* result(int status, const Ts&... tensors) {
    if (status) return PyLong_FromLong(status);
    PyObject* tuple = PyTuple_New(sizeof...(tensors));
    Py_ssize_t i = 0;
    (PyTuple_SET_ITEM(tuple, i++, tensors.defined() ? THPVariable_Wrap(tensors) : (Py_INCREF(Py_None), Py_None)), ...);
    return tuple;
}

template <PyObject* (*F)(PyObject* const*), Py_ssize_t N>
PyObject* call(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != N) return PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", N, n);
    try {
        return F(args);
    } catch (const PythonError&) {
        return nullptr;
    } catch (const Refused& e) {
        return PyLong_FromLong(e.status);
    } catch (const std::invalid_argument& e) {
        PyErr_SetString(PyExc_ValueError, e.what());
    } catch (const c10::OutOfMemoryError& e) {
        PyErr_SetString(PyExc_MemoryError, e.what_without_backtrace());
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}

// ------------------------------------------------------------------------------------------
// Dropout: x, p, seed, offset, device_offset, out
// ------------------------------------------------------------------------------------------
PyObject* dropout(PyObject* const* a) {
    const Tensor& x = tensor(a[0], "x");
    const auto dev = device_of(x, {});
    const mtxc_dropout_state state = drop_state(a[1], a[2], a[3], a[4], dev);
    Tensor out = output(Memory(dev), x, maybe(a[5], "out"), "out");
    uint64_t rows = 1, width = 1, xs = 1, os = 1;
    if (x.dim()) {
        const Rows r(x, "x");
        rows = (uint64_t)r.rows, width = (uint64_t)r.width;
        xs = row_stride(x, "x"), os = row_stride(out, "out", true);
    }
    return result(mtxc_dropout(code_of(x), out.mutable_data_ptr(), x.const_data_ptr(), rows, width, os, xs, &state), out);
}

// ------------------------------------------------------------------------------------------
// Block norm
// ------------------------------------------------------------------------------------------
const void* weight(const Tensor* w, int64_t width, const char* what) {
    if (!w) return nullptr;
    if (w->dim() != 1 || w->size(0) != width || (width > 1 && w->stride(0) != 1))
        throw invalid(quoted(what, ("expected " + std::to_string(width) + " contiguous values").c_str()));
    return w->const_data_ptr();
}

int weight_dtype(const Tensor* a, const Tensor* b) {
    if (a && b && a->scalar_type() != b->scalar_type()) throw invalid("post_weight and next_weight: expected one dtype");
    return a ? code_of(*a) : b ? code_of(*b) : MTXC_FLOAT;
}

// How many consecutive rows of x share a row of the gate: its leading axes are x's up to one, then ones.
uint64_t gate_rows(const Tensor& gate, const Tensor& x, int64_t rows) {
    if (gate.dim() == 0 || gate.size(-1) != x.size(-1) || gate.dim() > x.dim())
        throw invalid("gate: expected the rows' width and at most their axes");
    int64_t i = gate.dim() - 1, share = 1;
    while (i > 0 && gate.size(i - 1) == 1) --i;
    if (i == 0) return (uint64_t)std::max<int64_t>(1, rows);
    bool fits = gate.dim() == x.dim();
    for (int64_t k = 0; fits && k < i; ++k) fits = gate.size(k) == x.size(k);
    if (!fits) throw invalid("gate: expected one row, or the leading axes with the last ones of extent 1");
    for (int64_t k = i; k + 1 < x.dim(); ++k) share *= x.size(k);
    return (uint64_t)std::max<int64_t>(1, share);
}

// residual, branch, post_weight, gate, next_weight, residual_scale, branch_scale, weight_offset, eps, dropout, seed,
// offset, device_offset, save_rstd, out, normed_out -> residual, normed, post_rstd, next_rstd
PyObject* block_norm(PyObject* const* a) {
    const Tensor& x = tensor(a[0], "residual");
    const Tensor *b = maybe(a[1], "branch"), *post = maybe(a[2], "post_weight"), *gate = maybe(a[3], "gate"),
                 *next = maybe(a[4], "next_weight"), *out = maybe(a[14], "out"), *normed_out = maybe(a[15], "normed_out");
    const auto dev = device_of(x, {b, post, gate, next});
    same(b, x, "branch");
    const Rows r(x, "residual");
    if (!b && (post || gate)) throw invalid("post_weight and gate need a branch");
    if (normed_out && !next) throw invalid("normed_out needs next_weight");
    mtxc_block_norm_args m{};
    m.rows = (uint64_t)r.rows;
    m.width = (uint64_t)r.width;
    m.residual = x.const_data_ptr();
    m.residual_stride = row_stride(x, "residual");
    if (b) m.branch = b->const_data_ptr(), m.branch_stride = row_stride(*b, "branch");
    m.post_weight = weight(post, r.width, "post_weight");
    m.next_weight = weight(next, r.width, "next_weight");
    m.weight_dtype = weight_dtype(post, next);
    if (gate) {
        m.gate_rows = gate_rows(*gate, x, r.rows);
        m.gate = gate->const_data_ptr();
        m.gate_stride = row_stride(*gate, "gate");
        m.gate_dtype = code_of(*gate);
    }
    m.residual_scale = (float)number(a[5]);
    m.branch_scale = (float)number(a[6]);
    m.weight_offset = (float)number(a[7]);
    m.eps = (float)number(a[8]);
    m.drop = drop_state(a[9], a[10], a[11], a[12], dev);
    const Memory memory(dev);
    Tensor h = x, normed, post_rstd, next_rstd;
    if (b || m.residual_scale != 1.0f || out) {
        h = output(memory, x, out, "out");
        m.residual_out = h.mutable_data_ptr();
        m.residual_out_stride = row_stride(h, "out", true);
    }
    if (next) {
        normed = output(memory, x, normed_out, "normed_out");
        m.normed = normed.mutable_data_ptr();
        m.normed_stride = row_stride(normed, "normed_out", true);
    }
    if (flag(a[13])) {
        if (post) post_rstd = memory.empty({r.rows}, at::kFloat), m.post_rstd = static_cast<float*>(at_or_null(post_rstd));
        if (next) next_rstd = memory.empty({r.rows}, at::kFloat), m.next_rstd = static_cast<float*>(at_or_null(next_rstd));
    }
    return result(mtxc_block_norm(code_of(x), &m), h, normed, post_rstd, next_rstd);
}

const float* rstd(const Tensor* t, int64_t rows, const Tensor* of, const char* what) {
    if (!of) return nullptr;
    if (!t || t->scalar_type() != at::kFloat || t->numel() != rows || !t->is_contiguous())
        throw invalid(quoted(what, ("expected " + std::to_string(rows) + " contiguous float32 values, as block_norm saves them").c_str()));
    return static_cast<const float*>(t->const_data_ptr());
}

// d_residual, d_normed, residual, branch, post_rstd, next_rstd, post_weight, gate, next_weight, residual_scale,
// branch_scale, weight_offset, dropout, seed, offset, device_offset, parameters
// -> the gradients of residual, branch, post_weight, gate, next_weight
PyObject* block_norm_backward(PyObject* const* a) {
    const Tensor *dh = maybe(a[0], "d_residual"), *da = maybe(a[1], "d_normed"), *b = maybe(a[3], "branch"),
                 *r_post = maybe(a[4], "post_rstd"), *r_next = maybe(a[5], "next_rstd"), *post = maybe(a[6], "post_weight"),
                 *gate = maybe(a[7], "gate"), *next = maybe(a[8], "next_weight");
    const Tensor& h = tensor(a[2], "residual");
    const auto dev = device_of(h, {dh, da, b, r_post, r_next, post, gate, next});
    same(dh, h, "d_residual");
    same(da, h, "d_normed");
    same(b, h, "branch");
    const Rows r(h, "residual");
    if (!da != !next) throw invalid("d_normed and next_weight go together");
    if (!b && (post || gate)) throw invalid("post_weight and gate need a branch");
    mtxc_block_norm_backward_args m{};
    m.rows = (uint64_t)r.rows;
    m.width = (uint64_t)r.width;
    m.d_residual_out = at_or_null(dh);
    if (dh) m.d_residual_out_stride = row_stride(*dh, "d_residual");
    m.d_normed = at_or_null(da);
    if (da) m.d_normed_stride = row_stride(*da, "d_normed");
    m.residual_out = h.const_data_ptr();
    m.residual_out_stride = row_stride(h, "residual");
    m.branch = at_or_null(b);
    if (b) m.branch_stride = row_stride(*b, "branch");
    m.post_rstd = rstd(r_post, r.rows, post, "post_rstd");
    m.next_rstd = rstd(r_next, r.rows, next, "next_rstd");
    m.post_weight = weight(post, r.width, "post_weight");
    m.next_weight = weight(next, r.width, "next_weight");
    m.weight_dtype = weight_dtype(post, next);
    if (gate) {
        m.gate_rows = gate_rows(*gate, h, r.rows);
        m.gate = gate->const_data_ptr();
        m.gate_stride = row_stride(*gate, "gate");
        m.gate_dtype = code_of(*gate);
    }
    m.residual_scale = (float)number(a[9]);
    m.branch_scale = (float)number(a[10]);
    m.weight_offset = (float)number(a[11]);
    m.drop = drop_state(a[12], a[13], a[14], a[15], dev);
    const Memory memory(dev);
    Tensor dx = memory.like(h), db, dp, dg, dn;
    if (b) db = memory.like(h);
    if (flag(a[16])) {
        if (post) dp = memory.empty({r.width}, at::kFloat);
        if (next) dn = memory.empty({r.width}, at::kFloat);
        if (gate) dg = memory.like(*gate);
    }
    m.d_residual = dx.mutable_data_ptr();
    m.d_branch = at_or_null(db);
    m.d_post_weight = static_cast<float*>(at_or_null(dp));
    m.d_next_weight = static_cast<float*>(at_or_null(dn));
    m.d_gate = at_or_null(dg);
    m.d_residual_stride = m.d_branch_stride = m.d_gate_stride = (uint64_t)r.width;
    if (r.rows == 0 && dg.defined())  // a sum over no rows (the call itself knows of no gate row then)
        if (const int status = mtxc_memset(dg.mutable_data_ptr(), 0, dg.nbytes())) return result(status);
    return result(mtxc_block_norm_backward(code_of(h), &m), dx, db, dp, dg, dn);
}

// ------------------------------------------------------------------------------------------
// Rotary: q, k, positions, frequencies, scale, interleaved, inverse, q_out, k_out -> q, k
// ------------------------------------------------------------------------------------------
void put_strides(const Tensor& t, uint64_t (&to)[3]) {
    const int64_t lead = t.dim() - 1;  // 2 or 3
    for (int64_t i = 0; i < 3; ++i) to[i] = i + lead >= 3 ? (uint64_t)t.stride(i + lead - 3) : 0;
}

// Refuses an output of heads with two elements at one address: from the innermost axis out, each stride has to pass
// what lies inside it.  (The last axis has unit stride.)
void no_overlap(const Tensor& t, const char* what) {
    std::pair<int64_t, int64_t> axes[3];  // stride, size
    int n = 0;
    for (int64_t i = 0; i + 1 < t.dim(); ++i)
        if (t.size(i) > 1) axes[n++] = {t.stride(i), t.size(i)};
    if (t.numel() == 0) return;
    std::sort(axes, axes + n);
    int64_t span = t.size(-1);
    for (int i = 0; i < n; ++i) {
        if (axes[i].first < span) throw invalid(quoted(what, "its elements overlap"));
        span += axes[i].first * (axes[i].second - 1);
    }
}

PyObject* rotary(PyObject* const* a) {
    const Tensor& q = tensor(a[0], "q");
    const Tensor* k = maybe(a[1], "k");
    const Tensor &positions = tensor(a[2], "positions"), &frequencies = tensor(a[3], "frequencies");
    const auto dev = device_of(q, {k, &positions, &frequencies});
    if (q.dim() != 3 && q.dim() != 4)
        throw invalid("q: expected [batch, length, heads, head_dim] or [length, heads, head_dim]");
    if (k) {
        bool fits = k->dim() == q.dim() && k->scalar_type() == q.scalar_type() && k->size(-1) == q.size(-1);
        for (int64_t i = 0; fits && i + 2 < q.dim(); ++i) fits = k->size(i) == q.size(i);
        if (!fits) throw invalid("k: expected q's batch, length, head_dim and dtype");
    }
    if (frequencies.dim() != 1 || frequencies.scalar_type() != at::kDouble || !frequencies.is_contiguous())
        throw invalid("frequencies: expected contiguous float64 values");
    mtxc_rotary_args m{};
    const int64_t batch = q.dim() == 4 ? q.size(0) : 1, length = q.size(-3);
    m.batch = (uint64_t)batch;
    m.length = (uint64_t)length;
    m.head_dim = (uint32_t)q.size(-1);
    m.rotary_dim = (uint32_t)(2 * frequencies.size(0));
    if (positions.scalar_type() != at::kInt && positions.scalar_type() != at::kLong)
        throw invalid("positions: expected int32 or int64");
    if (positions.dim() == 1 && positions.size(0) == length) m.position_strides[1] = (uint64_t)positions.stride(0);
    else if (q.dim() == 4 && positions.dim() == 2 && positions.size(1) == length &&
             (positions.size(0) == 1 || positions.size(0) == batch)) {
        m.position_strides[0] = positions.size(0) == batch ? (uint64_t)positions.stride(0) : 0;
        m.position_strides[1] = (uint64_t)positions.stride(1);
    } else throw invalid("positions: expected [batch, length] or [length]");
    m.positions = positions.const_data_ptr();
    m.position_dtype = code_of(positions);
    m.frequencies = static_cast<const double*>(frequencies.const_data_ptr());
    m.scale = (float)number(a[4]);
    m.interleaved = flag(a[5]);
    m.inverse = flag(a[6]);
    const Memory memory(dev);
    Tensor out[2];
    const char* names[2] = {"q", "k"};
    for (int i = 0; i < 2; ++i) {
        const Tensor* x = i ? k : &q;
        const Tensor* given = maybe(a[7 + i], names[i]);
        if (!x) continue;
        if (x->size(-1) > 1 && x->stride(-1) != 1) throw invalid(quoted(names[i], "the last axis needs unit stride"));
        if (!given) {
            // heads stored as x stores them; x's axes may overlap, and then their order does not say which is the innermost
            out[i] = x->is_contiguous() ? memory.like(*x) : at::empty_like(*x);
            if (x->size(-1) > 1 && out[i].stride(-1) != 1) out[i] = memory.like(*x);
        } else {
            if (given->sizes() != x->sizes() || given->scalar_type() != x->scalar_type() || !given->is_cuda() ||
                given->get_device() != dev || (x->size(-1) > 1 && given->stride(-1) != 1))
                throw invalid(quoted(names[i], "expected an output of its shape, dtype and device, with unit stride in its last axis"));
            no_overlap(*given, names[i]);
            out[i] = written(*given);
        }
        m.heads[i] = (uint32_t)x->size(-2);
        m.src[i] = x->const_data_ptr();
        m.dst[i] = out[i].mutable_data_ptr();
        put_strides(*x, m.src_strides[i]);
        put_strides(out[i], m.dst_strides[i]);
    }
    return result(mtxc_rotary(code_of(q), &m), out[0], out[1]);
}

// ------------------------------------------------------------------------------------------
// Logits: logits, tokens, lengths, prompt_lengths, repetition, frequency, presence, bias_tokens, bias_values, mask, out
// ------------------------------------------------------------------------------------------
const void* per_row(const Tensor* t, int64_t rows, at::ScalarType type, const char* what) {
    if (!t) return nullptr;
    if (t->scalar_type() != type || t->dim() != 1 || t->size(0) != rows || (rows > 1 && t->stride(0) != 1))
        throw invalid(quoted(what, ("expected " + std::to_string(rows) + " contiguous values, int32 lengths or float32 penalties").c_str()));
    return t->const_data_ptr();
}

// Lists [rows, n], or [n] or [1, n] for all rows: the row stride; n in `count`.
uint64_t lists(const Tensor* t, int64_t rows, bool fits, const char* what, int64_t& count) {
    count = 0;
    if (!t) return 0;
    if (!fits || (t->dim() != 1 && t->dim() != 2) || (t->dim() == 2 && t->size(0) != 1 && t->size(0) != rows) ||
        (t->size(-1) > 1 && t->stride(-1) != 1))
        throw invalid(quoted(what, "expected [rows, n] or [n] with unit stride along n: tokens and masks int32, values float32"));
    count = t->size(-1);
    return t->dim() == 2 && t->size(0) == rows ? (uint64_t)t->stride(0) : 0;
}

PyObject* logits_rules(PyObject* const* a) {
    const Tensor& x = tensor(a[0], "logits");
    const Tensor *tokens = maybe(a[1], "tokens"), *lengths = maybe(a[2], "lengths"), *prompts = maybe(a[3], "prompt_lengths"),
                 *repetition = maybe(a[4], "repetition"), *frequency = maybe(a[5], "frequency"),
                 *presence = maybe(a[6], "presence"), *bias_tokens = maybe(a[7], "bias_tokens"),
                 *bias_values = maybe(a[8], "bias_values"), *mask = maybe(a[9], "mask"), *given = maybe(a[10], "out");
    const auto dev = device_of(x, {tokens, lengths, prompts, repetition, frequency, presence, bias_tokens, bias_values, mask});
    if (x.dim() != 2) throw invalid("logits: expected [rows, vocab]");
    if (!tokens && (lengths || prompts || repetition || frequency || presence))
        throw invalid("penalties need the rows' tokens");
    if (!bias_tokens != !bias_values) throw invalid("bias_tokens and bias_values go together");
    const int64_t rows = x.size(0), vocab = x.size(1);
    mtxc_logits_args m{};
    int64_t history, biases, values, words;
    m.tokens_stride = lists(tokens, rows, tokens && tokens->scalar_type() == at::kInt, "tokens", history);
    m.bias_tokens_stride = lists(bias_tokens, rows, bias_tokens && bias_tokens->scalar_type() == at::kInt, "bias_tokens", biases);
    m.bias_values_stride = lists(bias_values, rows, bias_values && bias_values->scalar_type() == at::kFloat, "bias_values", values);
    m.mask_stride = lists(mask, rows, mask && (mask->scalar_type() == at::kInt || mask->scalar_type() == at::kUInt32), "mask", words);
    if (values != biases) throw invalid("bias_values: expected one for each of bias_tokens");
    if (mask && words != (vocab + 31) / 32) throw invalid("mask: expected one bit for each token, in words of 32");
    m.rows = (uint64_t)rows;
    m.vocab = (uint64_t)vocab;
    m.src = x.const_data_ptr();
    m.src_stride = row_stride(x, "logits");
    m.tokens = static_cast<const int32_t*>(at_or_null(tokens));
    m.history = (uint64_t)history;
    m.lengths = static_cast<const int32_t*>(per_row(lengths, rows, at::kInt, "lengths"));
    m.prompt_lengths = static_cast<const int32_t*>(per_row(prompts, rows, at::kInt, "prompt_lengths"));
    m.repetition = static_cast<const float*>(per_row(repetition, rows, at::kFloat, "repetition"));
    m.frequency = static_cast<const float*>(per_row(frequency, rows, at::kFloat, "frequency"));
    m.presence = static_cast<const float*>(per_row(presence, rows, at::kFloat, "presence"));
    m.bias_tokens = static_cast<const int32_t*>(at_or_null(bias_tokens));
    m.bias_values = static_cast<const float*>(at_or_null(bias_values));
    m.biases = (uint64_t)biases;
    m.mask = static_cast<const uint32_t*>(at_or_null(mask));
    Tensor out = output(Memory(dev), x, given, "out");
    m.dst = out.mutable_data_ptr();
    m.dst_stride = row_stride(out, "out", true);
    return result(mtxc_logits_rules(code_of(x), &m), out);
}

PyMethodDef methods[] = {
    {"dropout", (PyCFunction)(void (*)())call<dropout, 6>, METH_FASTCALL, nullptr},
    {"block_norm", (PyCFunction)(void (*)())call<block_norm, 16>, METH_FASTCALL, nullptr},
    {"block_norm_backward", (PyCFunction)(void (*)())call<block_norm_backward, 17>, METH_FASTCALL, nullptr},
    {"rotary", (PyCFunction)(void (*)())call<rotary, 9>, METH_FASTCALL, nullptr},
    {"logits_rules", (PyCFunction)(void (*)())call<logits_rules, 11>, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_lm", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__lm(void) {
    PyObject* m = PyModule_Create(&module);
    if (m && PyModule_AddStringConstant(m, "torch_version", MTX_TORCH_VERSION)) Py_CLEAR(m);
    return m;
}
