// torch_ops.cpp -- torch tensors to the argument blocks of the plaintext
// operators (include/tsgpu.h): the checks, the allocations and the current
// stream of provenloop_b200.adapters, .logits and .losses.
//
// A decode step makes these calls at every projection, and a call on one
// token is shorter on the GPU than its checks were in Python: this module is
// those checks, compiled.  It does not link against the library: the entry
// points' addresses come from the binding that loaded it (bind).
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/core/grad_mode.h>
#include <c10/core/AutogradState.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAStream.h>

#include <climits>
#include <memory>
#include <sstream>
#include <stdexcept>
#include <string>
#include <vector>

#include "../../include/tsgpu.h"

namespace {

struct {
    decltype(&ts_adapter_workspace) workspace = nullptr;
    decltype(&ts_adapter_project) project = nullptr;
    decltype(&ts_adapter_project_backward) backward = nullptr;
    decltype(&ts_logit_rules) rules = nullptr;
    decltype(&ts_loss_workspace) loss_workspace = nullptr;
    decltype(&ts_token_logprobs) losses[4] = {};  // by TS_LOSS_*
    decltype(&ts_clip_workspace) clip_workspace = nullptr;
    decltype(&ts_clip_gradients) clip = nullptr;
    PyObject* check = nullptr;  // _lib.check: raises for a status
} g;

// Becomes a ValueError.
[[noreturn]] void bad(const std::string& msg) { throw std::invalid_argument(msg); }

// A Python error is set.
struct PyFailed {};

bool truth(PyObject* o) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw PyFailed{};
    return v;
}

const at::Tensor* tensor(PyObject* o, const char* name, bool optional = false) {
    if (optional && o == Py_None) return nullptr;
    if (!THPVariable_Check(o)) bad(std::string(name) + " must be a tensor");
    return &THPVariable_Unpack(o);
}

std::string shape_of(at::IntArrayRef s) {
    std::ostringstream o;
    o << "(";
    for (size_t i = 0; i < s.size(); i++) o << (i ? ", " : "") << s[i];
    o << (s.size() == 1 ? ",)" : ")");
    return o.str();
}

std::string type_of(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return "torch.float32";
        case at::kBFloat16: return "torch.bfloat16";
        case at::kHalf: return "torch.float16";
        case at::kInt: return "torch.int32";
        case at::kLong: return "torch.int64";
        default: return std::string("torch.") + at::toString(t);
    }
}

int dtype_code(at::ScalarType t) {
    if (t == at::kFloat) return TS_DTYPE_F32;
    if (t == at::kBFloat16) return TS_DTYPE_BF16;
    if (t == at::kHalf) return TS_DTYPE_F16;
    bad("dtype must be float32, bfloat16 or float16, not " + type_of(t));
}

// Stride between the rows of t [..., d] seen as [n, d].
int64_t row_stride(const at::Tensor& t, const char* name) {
    const auto size = t.sizes(), stride = t.strides();
    const int64_t dim = t.dim();
    if (dim < 2) bad(std::string(name) + " must be [..., d] with at least two dimensions, not " + shape_of(size));
    if (size[dim - 1] > 1 && stride[dim - 1] != 1) bad(std::string("the last dimension of ") + name + " must be contiguous");
    if (dim == 2) return stride[0];
    int64_t row = -1, next = 0;
    for (int64_t i = dim - 2; i >= 0; i--) {
        if (size[i] == 1) continue;
        if (row < 0) row = stride[i];
        else if (t.numel() && stride[i] != next) bad(std::string("the leading dimensions of ") + name + " do not form rows of one stride");
        next = stride[i] * size[i];
    }
    return row < 0 ? size[dim - 1] : row;
}

void same(const at::Tensor& t, const char* name, at::ScalarType dtype, const at::Tensor& like, at::IntArrayRef shape) {
    if (t.scalar_type() != dtype) bad(std::string(name) + " must be " + type_of(dtype) + ", not " + type_of(t.scalar_type()));
    if (t.sizes() != shape) bad(std::string(name) + " must be " + shape_of(shape) + ", not " + shape_of(t.sizes()));
    if (t.device() != like.device()) bad(std::string(name) + " is on " + t.device().str() + ", not on " + like.device().str());
}

void whole(const at::Tensor& t, const char* name, at::ScalarType dtype, const at::Tensor& like, at::IntArrayRef shape) {
    same(t, name, dtype, like, shape);
    if (!t.is_contiguous()) bad(std::string(name) + " must be contiguous");
}

void no_history(const at::Tensor* t) {
    if (t && t->requires_grad() && at::GradMode::is_enabled())
        bad("an input requires a gradient, which this call does not record: call it under torch.no_grad() (adapter_project_backward "
            "gives the adapters' gradients, the losses their logits')");
    if (t && c10::AutogradState::get_tls_state().get_fw_grad_mode() && t->_fw_grad(0).defined())
        bad("an input has a forward-mode tangent, which this call would lose: call it on the primal (torch.autograd.forward_ad.unpack_dual)");
}

// `t` has been written: autograd finds out if it had saved it.
void written(const at::Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

void finish(int rc, const char* what) {
    if (rc == TS_OK) return;
    PyObject* r = PyObject_CallFunction(g.check, "is", rc, what);
    Py_XDECREF(r);
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, what);
    throw PyFailed{};
}

PyObject* none_or(const at::Tensor& t) {
    if (t.defined()) return THPVariable_Wrap(t);
    Py_RETURN_NONE;
}

void arity(Py_ssize_t n, Py_ssize_t want) {
    if (n != want) bad("wrong number of arguments");
    if (!g.check) bad("the library is not bound");
}

// Runs `body`, which returns a new reference; C++ errors become Python's.
template <class F>
PyObject* guarded(F body) {
    try {
        return body();
    } catch (const PyFailed&) {
        return nullptr;
    } catch (const std::invalid_argument& e) {
        PyErr_SetString(PyExc_ValueError, e.what());
    } catch (const std::exception& e) {
        // out of memory keeps torch's type and message
        torch::translate_exception_to_python(std::current_exception());
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}

// Fields that both directions share, checked.
void common(ts_adapter_args& q, const at::Tensor& x, const at::Tensor& a, const at::Tensor& b, const at::Tensor& ids, const at::Tensor* w,
            const at::Tensor* scale) {
    const at::ScalarType dtype = x.scalar_type();
    q.dtype = dtype_code(dtype);
    q.x_stride = row_stride(x, "x");
    const auto size = x.sizes();
    const int64_t lead = x.dim() - 1, d_in = size[lead];
    if (a.dim() != 3 || b.dim() != 3) bad("lora_a must be [adapters, r, d_in] and lora_b [adapters, d_out, r]");
    const int64_t adapters = a.size(0), r = a.size(1), d_out = b.size(1);
    whole(a, "lora_a", dtype, x, {adapters, r, d_in});
    whole(b, "lora_b", dtype, x, {adapters, d_out, r});
    const auto isize = ids.sizes();
    if (isize.empty() || (int64_t)isize.size() > lead || size.slice(0, isize.size()) != isize)
        bad("adapter must hold one index per leading entry of x " + shape_of(size.slice(0, lead)) + ", not " + shape_of(isize));
    whole(ids, "adapter", at::kInt, x, isize);
    int64_t per = 1, n = 1;
    for (int64_t i = 0; i < lead; i++) {
        n *= size[i];
        if (i >= (int64_t)isize.size()) per *= size[i];
    }
    if (w) {
        same(*w, "weight", dtype, x, {d_out, d_in});
        if (d_in > 1 && w->stride(1) != 1) bad("the last dimension of weight must be contiguous");
        q.weight = w->const_data_ptr();
        q.weight_stride = w->stride(0);
    }
    if (scale) {
        whole(*scale, "scale", at::kFloat, x, {adapters});
        q.scale = static_cast<const float*>(scale->const_data_ptr());
    }
    for (const at::Tensor* t : {&x, &a, &b, w, scale}) no_history(t);
    const int64_t most = 0xffffffffll;
    if (d_in > most || d_out > most || r > most || adapters > most) bad("a dimension is too large");
    q.n = (uint64_t)n, q.tokens_per_id = (uint64_t)(per ? per : 1);
    q.d_in = (uint32_t)d_in, q.d_out = (uint32_t)d_out, q.r = (uint32_t)r, q.adapters = (uint32_t)adapters;
    q.x = x.const_data_ptr(), q.lora_a = a.const_data_ptr(), q.lora_b = b.const_data_ptr();
    q.adapter = static_cast<const int32_t*>(ids.const_data_ptr());
}

int on_device(const at::Tensor& like, const char* what) {
    if (!like.is_cuda()) bad(std::string(what) + " must be on a CUDA device: there is no CPU form");
    return like.get_device();
}

// Queues the call on the current stream, with a workspace from the allocator
// that is free again for what is queued on that stream afterwards.
void run(ts_adapter_args& q, bool backward, const at::Tensor& x) {
    q.device = on_device(x, "the tensors");
    const cudaStream_t s = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)q.device).stream();
    q.stream = s;
    uint64_t bytes = 0;
    finish(g.workspace(&q, backward, &bytes), "ts_adapter_workspace");
    at::Tensor ws;
    if (bytes) {
        ws = at::empty({(int64_t)bytes}, x.options().dtype(at::kByte));
        q.workspace = ws.mutable_data_ptr();
        q.workspace_bytes = bytes;
    }
    finish(backward ? g.backward(&q) : g.project(&q), backward ? "ts_adapter_project_backward" : "ts_adapter_project");
}

// (x, lora_a, lora_b, adapter, weight, bias, base, scale, out) -> out
PyObject* project(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&] {
        arity(n, 9);
        const at::Tensor &x = *tensor(args[0], "x"), &a = *tensor(args[1], "lora_a"), &b = *tensor(args[2], "lora_b"), &ids = *tensor(args[3], "adapter");
        const at::Tensor *w = tensor(args[4], "weight", true), *bias = tensor(args[5], "bias", true), *base = tensor(args[6], "base", true),
                         *scale = tensor(args[7], "scale", true), *given = tensor(args[8], "out", true);
        ts_adapter_args q{};
        common(q, x, a, b, ids, w, scale);
        c10::SmallVector<int64_t, 5> shape(x.sizes().begin(), x.sizes().end());
        shape.back() = q.d_out;
        if (bias) {
            whole(*bias, "bias", x.scalar_type(), x, {(int64_t)q.d_out});
            no_history(bias);
            q.bias = bias->const_data_ptr();
        }
        if (base) {
            same(*base, "base", x.scalar_type(), x, shape);
            q.base_stride = row_stride(*base, "base");
            no_history(base);
            q.base = base->const_data_ptr();
        }
        at::Tensor out;
        if (given) {
            same(*given, "out", x.scalar_type(), x, shape);
            q.out_stride = row_stride(*given, "out");
            no_history(given);
            out = *given;
        } else {
            on_device(x, "the tensors");
            out = at::empty(shape, x.options());
            q.out_stride = q.d_out;
        }
        q.out = out.mutable_data_ptr();
        run(q, false, x);
        if (given) {
            written(*given);
            Py_INCREF(args[8]);
            return args[8];
        }
        return THPVariable_Wrap(out);
    });
}

// (grad, x, lora_a, lora_b, adapter, weight, scale, need_x, need_adapters) -> (dx, da, db)
PyObject* backward(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        arity(n, 9);
        const at::Tensor &dy = *tensor(args[0], "grad"), &x = *tensor(args[1], "x"), &a = *tensor(args[2], "lora_a"), &b = *tensor(args[3], "lora_b"),
                         &ids = *tensor(args[4], "adapter");
        const at::Tensor *w = tensor(args[5], "weight", true), *scale = tensor(args[6], "scale", true);
        const bool need_x = truth(args[7]), need_adapters = truth(args[8]);
        ts_adapter_args q{};
        common(q, x, a, b, ids, w, scale);
        c10::SmallVector<int64_t, 5> shape(x.sizes().begin(), x.sizes().end());
        shape.back() = q.d_out;
        same(dy, "grad", x.scalar_type(), x, shape);
        q.grad_stride = row_stride(dy, "grad");
        no_history(&dy);
        q.grad = dy.const_data_ptr();
        if (!need_x && !need_adapters) bad("no gradient is asked for");
        on_device(x, "the tensors");
        at::Tensor dx, da, db;
        if (need_x) {
            dx = at::empty(x.sizes(), x.options());
            q.out = dx.mutable_data_ptr();
            q.out_stride = q.d_in;
        }
        if (need_adapters) {
            da = at::empty(a.sizes(), a.options()), db = at::empty(b.sizes(), b.options());
            q.grad_a = da.mutable_data_ptr(), q.grad_b = db.mutable_data_ptr();
        }
        run(q, true, x);
        PyObject* r = PyTuple_New(3);
        if (!r) throw PyFailed{};
        PyTuple_SET_ITEM(r, 0, none_or(dx));
        PyTuple_SET_ITEM(r, 1, none_or(da));
        PyTuple_SET_ITEM(r, 2, none_or(db));
        return r;
    });
}

const void* per_row(const at::Tensor* t, const char* name, at::ScalarType dtype, int64_t n, const at::Tensor& like) {
    if (!t) return nullptr;
    if (t->scalar_type() != dtype || t->dim() != 1 || t->size(0) != n || !t->is_contiguous())
        bad(std::string(name) + " must be a contiguous " + type_of(dtype) + " tensor of shape (" + std::to_string(n) + ",)");
    if (t->device() != like.device()) bad(std::string(name) + " is on " + t->device().str() + ", logits on " + like.device().str());
    return t->const_data_ptr();
}

// Stride between rows of t [n, cols] (cols < 0: any), or 0 for one row [cols] for all.
int64_t table(const at::Tensor& t, const char* name, bool type_ok, const char* types, int64_t n, int64_t cols, const at::Tensor& like) {
    if (!type_ok) bad(std::string(name) + " must be " + types + ", not " + type_of(t.scalar_type()));
    const int64_t dim = t.dim();
    if (dim < 1 || dim > 2 || (dim == 2 && t.size(0) != n) || (cols >= 0 && t.size(dim - 1) != cols))
        bad(std::string(name) + " must be [" + std::to_string(n) + ", " + (cols < 0 ? "k" : std::to_string(cols)) + "] or one such row, not " +
            shape_of(t.sizes()));
    if (t.size(dim - 1) > 1 && t.stride(dim - 1) != 1) bad(std::string("the last dimension of ") + name + " must be contiguous");
    if (t.device() != like.device()) bad(std::string(name) + " is on " + t.device().str() + ", logits on " + like.device().str());
    return dim == 2 ? t.stride(0) : 0;
}

// (logits, tokens, lengths, prompt_lengths, repetition, frequency, presence, bias_ids, bias_values, mask, out, write, pick)
// -> (logits or None, picks or None)
PyObject* rules(PyObject*, PyObject* const* args, Py_ssize_t count) {
    return guarded([&]() -> PyObject* {
        arity(count, 13);
        const at::Tensor& x = *tensor(args[0], "logits");
        static const char* const names[] = {"logits", "tokens", "lengths", "prompt_lengths", "repetition", "frequency", "presence",
                                            "bias_ids", "bias_values", "mask", "out"};
        const at::Tensor* t[11];
        for (int i = 1; i < 11; i++) t[i] = tensor(args[i], names[i], true);
        const bool write = truth(args[11]), pick = truth(args[12]);
        ts_rules_args q{};
        q.dtype = q.out_dtype = dtype_code(x.scalar_type());
        if (x.dim() != 2 || (x.size(1) > 1 && x.stride(1) != 1)) bad("logits must be [n, vocab] with contiguous rows");
        const int64_t n = x.size(0), vocab = x.size(1);
        if (vocab == 0) bad("the vocabulary is empty");
        if (vocab > 0x7fffffffll) bad("the vocabulary is too large");
        const auto ints = [](const at::Tensor& v) { return v.scalar_type() == at::kLong || v.scalar_type() == at::kInt; };
        if (const at::Tensor* v = t[1]) {
            if (v->dim() != 2) bad("tokens must be [n, k]");
            q.tokens_stride = table(*v, "tokens", ints(*v), "int32 or int64", n, -1, x);
            if (v->size(1) > TS_RULES_MAX_HISTORY) bad("the history is longer than " + std::to_string(TS_RULES_MAX_HISTORY));
            q.token_cols = (uint32_t)v->size(1);
            q.ids64 |= v->scalar_type() == at::kLong;
            q.tokens = v->const_data_ptr();
        }
        for (int i = 2; i < 7; i++)
            if (t[i] && !t[1]) bad(std::string(names[i]) + " needs tokens");
        q.lengths = static_cast<const int32_t*>(per_row(t[2], names[2], at::kInt, n, x));
        q.prompt_lengths = static_cast<const int32_t*>(per_row(t[3], names[3], at::kInt, n, x));
        q.repetition = static_cast<const float*>(per_row(t[4], names[4], at::kFloat, n, x));
        q.frequency = static_cast<const float*>(per_row(t[5], names[5], at::kFloat, n, x));
        q.presence = static_cast<const float*>(per_row(t[6], names[6], at::kFloat, n, x));
        if (!t[7] != !t[8]) bad("bias_ids and bias_values come together");
        if (const at::Tensor* v = t[7]) {
            q.bias_ids_stride = table(*v, "bias_ids", ints(*v), "int32 or int64", n, -1, x);
            const int64_t cols = v->size(-1);
            q.bias_values_stride = table(*t[8], "bias_values", t[8]->scalar_type() == at::kFloat, "float32", n, cols, x);
            if (cols > TS_RULES_MAX_BIASES) bad("more than " + std::to_string(TS_RULES_MAX_BIASES) + " biases in a row");
            q.bias_cols = (uint32_t)cols;
            q.ids64 |= (v->scalar_type() == at::kLong) << 1;
            q.bias_ids = v->const_data_ptr();
            q.bias_values = static_cast<const float*>(t[8]->const_data_ptr());
        }
        if (const at::Tensor* v = t[9]) {
            q.mask_stride = table(*v, "mask", v->scalar_type() == at::kInt, "int32", n, (vocab + 31) / 32, x);
            q.mask = static_cast<const int32_t*>(v->const_data_ptr());
        }
        for (const at::Tensor* v : {&x, t[4], t[5], t[6], t[8]}) no_history(v);
        at::Tensor out;
        if (const at::Tensor* v = t[10]) {
            if (!write) bad("out is given, but write is false");
            if ((v->scalar_type() != x.scalar_type() && v->scalar_type() != at::kFloat) || v->sizes() != x.sizes() || v->device() != x.device())
                bad("out must be " + shape_of(x.sizes()) + " on " + x.device().str() + ", " + type_of(x.scalar_type()) + " or torch.float32");
            if (vocab > 1 && v->stride(1) != 1) bad("the rows of out must be contiguous");
            no_history(v);
            q.out_dtype = dtype_code(v->scalar_type());
            out = *v;
        }
        if (!write && !pick) bad("neither logits nor picks are asked for");
        q.device = on_device(x, "logits");
        if (write && !out.defined()) out = at::empty({n, vocab}, x.options());
        at::Tensor picks;
        if (pick) picks = at::empty({n}, x.options().dtype(at::kLong));
        q.n = (uint64_t)n, q.vocab = (uint32_t)vocab;
        q.logits = x.const_data_ptr(), q.logits_stride = x.stride(0);
        if (out.defined()) q.out = out.mutable_data_ptr(), q.out_stride = out.stride(0);
        if (picks.defined()) q.pick = static_cast<int64_t*>(picks.mutable_data_ptr());
        q.stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)q.device).stream();
        finish(g.rules(&q), "ts_logit_rules");
        if (t[10]) written(*t[10]);
        PyObject* r = PyTuple_New(2);
        if (!r) throw PyFailed{};
        if (t[10]) {
            Py_INCREF(args[10]);
            PyTuple_SET_ITEM(r, 0, args[10]);
        } else {
            PyTuple_SET_ITEM(r, 0, none_or(out));
        }
        PyTuple_SET_ITEM(r, 1, none_or(picks));
        return r;
    });
}

double number(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw PyFailed{};
    return v;
}

int whole_number(PyObject* o) {
    const long v = PyLong_AsLong(o);
    if (v == -1 && PyErr_Occurred()) throw PyFailed{};
    if (v < INT_MIN || v > INT_MAX) bad("a number is too large");
    return (int)v;
}

// f32 per row, of the targets' shape.
const float* like_targets(const at::Tensor* t, const char* name, const at::Tensor& targets, const at::Tensor& x) {
    if (!t) return nullptr;
    whole(*t, name, at::kFloat, x, targets.sizes());
    no_history(t);
    return static_cast<const float*>(t->const_data_ptr());
}

const float* one_value(const at::Tensor* t, const char* name, const at::Tensor& x) {
    if (!t) return nullptr;
    if (t->scalar_type() != at::kFloat || t->numel() != 1) bad(std::string(name) + " must be one float32 value, not " + type_of(t->scalar_type()) + " " + shape_of(t->sizes()));
    if (t->device() != x.device()) bad(std::string(name) + " is on " + t->device().str() + ", not on " + x.device().str());
    no_history(t);
    return static_cast<const float*>(t->const_data_ptr());
}

// Logits and targets of the losses and of the log-probabilities.
void loss_rows(ts_loss_args& q, const at::Tensor& x, const at::Tensor& targets) {
    q.dtype = dtype_code(x.scalar_type());
    q.logits_stride = row_stride(x, "logits");
    const auto size = x.sizes();
    const int64_t vocab = size.back();
    if (vocab == 0) bad("the vocabulary is empty");
    if (vocab > 0x7fffffffll) bad("the vocabulary is too large");
    if (targets.scalar_type() != at::kLong && targets.scalar_type() != at::kInt) bad("targets must be int32 or int64, not " + type_of(targets.scalar_type()));
    whole(targets, "targets", targets.scalar_type(), x, size.slice(0, size.size() - 1));
    no_history(&x);
    q.targets64 = targets.scalar_type() == at::kLong;
    q.n = (uint64_t)targets.numel(), q.vocab = (uint32_t)vocab;
    q.logits = x.const_data_ptr(), q.targets = targets.const_data_ptr();
}

// The sequences that the rows of a loss form.
void loss_sequences(ts_loss_args& q, const at::Tensor& x, const at::Tensor& targets, const at::Tensor* starts) {
    if (starts) {
        if (targets.dim() != 1) bad("with starts, logits must be [rows, vocab] and targets [rows]");
        if (starts->dim() != 1 || starts->size(0) < 2) bad("starts must hold the sequences' first rows and the end of the last, not " + shape_of(starts->sizes()));
        whole(*starts, "starts", at::kInt, x, {starts->size(0)});
        if (starts->size(0) > 0x40000000ll) bad("too many sequences");
        q.starts = static_cast<const int32_t*>(starts->const_data_ptr());
        q.sequences = (uint32_t)(starts->size(0) - 1);
    } else {
        if (targets.dim() > 1 && targets.size(0) > 0x40000000ll) bad("too many sequences");
        q.sequences = targets.dim() > 1 ? (uint32_t)targets.size(0) : 1;
    }
}

// The gradient's tensor: `given`, or a new one, or none.  Everything else has
// been checked; sets the device.
at::Tensor loss_grad(ts_loss_args& q, const at::Tensor& x, const at::Tensor* given, bool need) {
    at::Tensor grad;
    if (given) {
        if (!need) bad("out is given, but no gradient is asked for");
        same(*given, "out", x.scalar_type(), x, x.sizes());
        q.grad_stride = row_stride(*given, "out");
        no_history(given);
        grad = *given;
    }
    q.device = on_device(x, "the tensors");
    if (!given && need) {
        grad = at::empty(x.sizes(), x.options());
        q.grad_stride = x.sizes().back();
    }
    if (grad.defined()) q.grad = grad.mutable_data_ptr();
    return grad;
}

void run_loss(ts_loss_args& q, int op, const at::Tensor& x) {
    static const char* const names[] = {"ts_token_logprobs", "ts_token_logprobs_backward", "ts_policy_loss", "ts_preference_loss"};
    q.stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)q.device).stream();
    uint64_t bytes = 0;
    finish(g.loss_workspace(&q, op, &bytes), "ts_loss_workspace");
    at::Tensor ws;
    if (bytes) {
        ws = at::empty({(int64_t)bytes}, x.options().dtype(at::kByte));
        q.workspace = ws.mutable_data_ptr();
        q.workspace_bytes = bytes;
    }
    finish(g.losses[op](&q), names[op]);
}

PyObject* given_or(const at::Tensor* given, PyObject* object, const at::Tensor& t) {
    if (!given) return none_or(t);
    written(*given);
    Py_INCREF(object);
    return object;
}

// (logits, targets) -> logprobs
PyObject* logprobs(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&] {
        arity(n, 2);
        const at::Tensor &x = *tensor(args[0], "logits"), &targets = *tensor(args[1], "targets");
        ts_loss_args q{};
        loss_rows(q, x, targets);
        q.device = on_device(x, "the tensors");
        at::Tensor out = at::empty(targets.sizes(), x.options().dtype(at::kFloat));
        q.logprobs = static_cast<float*>(out.mutable_data_ptr());
        run_loss(q, TS_LOSS_LOGPROBS, x);
        return THPVariable_Wrap(out);
    });
}

// (grad, logits, targets, out) -> gradient of logits
PyObject* logprobs_backward(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&] {
        arity(n, 4);
        const at::Tensor &dy = *tensor(args[0], "grad"), &x = *tensor(args[1], "logits"), &targets = *tensor(args[2], "targets");
        const at::Tensor* given = tensor(args[3], "out", true);
        ts_loss_args q{};
        loss_rows(q, x, targets);
        q.grad_logprobs = like_targets(&dy, "grad", targets, x);
        const at::Tensor grad = loss_grad(q, x, given, true);
        run_loss(q, TS_LOSS_LOGPROBS_BACKWARD, x);
        return given_or(given, args[3], grad);
    });
}

// (logits, targets, old, advantages, ref, starts, clip_low, clip_high, kl, kind, grad_scale, need_grad, out) -> (loss, logprobs, grad or None)
PyObject* policy(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        arity(n, 13);
        const at::Tensor &x = *tensor(args[0], "logits"), &targets = *tensor(args[1], "targets"), &adv = *tensor(args[3], "advantages");
        const at::Tensor *old = tensor(args[2], "old_logprobs", true), *ref = tensor(args[4], "ref_logprobs", true),
                         *starts = tensor(args[5], "starts", true), *scale = tensor(args[10], "grad_scale", true), *given = tensor(args[12], "out", true);
        ts_loss_args q{};
        loss_rows(q, x, targets);
        loss_sequences(q, x, targets, starts);
        q.old_logprobs = like_targets(old, "old_logprobs", targets, x);
        q.ref_logprobs = like_targets(ref, "ref_logprobs", targets, x);
        if (adv.sizes() == targets.sizes()) {
            q.advantages = like_targets(&adv, "advantages", targets, x);
            q.advantage_rows = 1;
        } else {
            whole(adv, "advantages", at::kFloat, x, {(int64_t)q.sequences});
            no_history(&adv);
            q.advantages = static_cast<const float*>(adv.const_data_ptr());
        }
        q.clip_low = (float)number(args[6]), q.clip_high = (float)number(args[7]), q.kl = (float)number(args[8]);
        q.kind = whole_number(args[9]);
        q.grad_scale = one_value(scale, "grad_scale", x);
        const bool need = truth(args[11]);
        const at::Tensor grad = loss_grad(q, x, given, need);
        at::Tensor loss = at::empty({}, x.options().dtype(at::kFloat)), lp = at::empty(targets.sizes(), x.options().dtype(at::kFloat));
        q.loss = static_cast<float*>(loss.mutable_data_ptr()), q.logprobs = static_cast<float*>(lp.mutable_data_ptr());
        run_loss(q, TS_LOSS_POLICY, x);
        PyObject* r = PyTuple_New(3);
        if (!r) throw PyFailed{};
        PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(loss));
        PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(lp));
        PyTuple_SET_ITEM(r, 2, given_or(given, args[12], grad));
        return r;
    });
}

// (logits, targets, ref, starts, beta, kind, smoothing, average, grad_scale, need_grad, out) -> (loss, margins, logprobs, grad or None)
PyObject* preference(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        arity(n, 11);
        const at::Tensor &x = *tensor(args[0], "logits"), &targets = *tensor(args[1], "targets");
        const at::Tensor *ref = tensor(args[2], "ref_logprobs", true), *starts = tensor(args[3], "starts", true),
                         *scale = tensor(args[8], "grad_scale", true), *given = tensor(args[10], "out", true);
        ts_loss_args q{};
        loss_rows(q, x, targets);
        loss_sequences(q, x, targets, starts);
        if (q.sequences % 2) bad("the sequences must be the chosen ones and as many rejected ones, not " + std::to_string(q.sequences));
        q.ref_logprobs = like_targets(ref, "ref_logprobs", targets, x);
        q.beta = (float)number(args[4]), q.kind = whole_number(args[5]), q.smoothing = (float)number(args[6]);
        q.average = truth(args[7]);
        q.grad_scale = one_value(scale, "grad_scale", x);
        const bool need = truth(args[9]);
        const at::Tensor grad = loss_grad(q, x, given, need);
        const auto f32 = x.options().dtype(at::kFloat);
        at::Tensor loss = at::empty({}, f32), margins = at::empty({(int64_t)(q.sequences / 2)}, f32), lp = at::empty(targets.sizes(), f32);
        q.loss = static_cast<float*>(loss.mutable_data_ptr()), q.margins = static_cast<float*>(margins.mutable_data_ptr());
        q.logprobs = static_cast<float*>(lp.mutable_data_ptr());
        run_loss(q, TS_LOSS_PREFERENCE, x);
        PyObject* r = PyTuple_New(4);
        if (!r) throw PyFailed{};
        PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(loss));
        PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(margins));
        PyTuple_SET_ITEM(r, 2, THPVariable_Wrap(lp));
        PyTuple_SET_ITEM(r, 3, given_or(given, args[10], grad));
        return r;
    });
}

// A list or tuple for a scope.
struct Items {
    PyObject* o;
    Items(PyObject* list, const char* name) : o(PySequence_Check(list) && !THPVariable_Check(list) ? PySequence_Fast(list, "") : nullptr) {
        if (!o) {
            PyErr_Clear();
            bad(std::string(name) + " must be a list of tensors");
        }
    }
    ~Items() { Py_DECREF(o); }
    Items(const Items&) = delete;
    Items& operator=(const Items&) = delete;
    Py_ssize_t size() const { return PySequence_Fast_GET_SIZE(o); }
    PyObject* operator[](Py_ssize_t i) const { return PySequence_Fast_GET_ITEM(o, i); }
    // Entries some places on, whose parts lie far apart in memory.
    void ahead(Py_ssize_t i) const {
        if (i + 12 < size()) __builtin_prefetch((*this)[i + 12]);
        if (i + 6 < size() && THPVariable_CheckExact((*this)[i + 6])) __builtin_prefetch(THPVariable_Unpack((*this)[i + 6]).unsafeGetTensorImpl());
    }
};

// (grads, max_norm, adapters or None, out or None) -> norms
PyObject* clip(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        arity(n, 4);
        const Items grads(args[0], "grads");
        const bool apart = args[3] != Py_None;
        std::unique_ptr<Items> outs(apart ? new Items(args[3], "out") : nullptr);
        if (apart && outs->size() != grads.size()) bad("out must have as many tensors as grads");
        const bool each = args[2] != Py_None;
        const int groups = each ? whole_number(args[2]) : 1;
        if (groups < 1 || groups > TS_CLIP_MAX_GROUPS) bad("the number of adapters must be in 1 .. " + std::to_string(TS_CLIP_MAX_GROUPS));
        // whether a tensor may have a forward-mode tangent at all: to ask each of hundreds takes as long as the call
        const bool tangents = c10::AutogradState::get_tls_state().get_fw_grad_mode() && torch::autograd::ForwardADLevel::try_get_by_idx(0);
        const auto history = [&](const at::Tensor& t) {
            if (tangents || t.requires_grad()) no_history(&t);
        };
        std::vector<ts_clip_tensor> list;
        list.reserve(grads.size());
        const at::Tensor* like = nullptr;
        for (Py_ssize_t i = 0; i < grads.size(); i++) {
            grads.ahead(i);
            if (apart) outs->ahead(i);
            if (grads[i] == Py_None) continue;
            const at::Tensor& t = *tensor(grads[i], "every entry of grads");
            if (!like) like = &t;
            ts_clip_tensor c{};
            c.dtype = c.out_dtype = dtype_code(t.scalar_type());
            if (t.device() != like->device()) bad("a gradient is on " + t.device().str() + ", not on " + like->device().str());
            if (each ? !t.is_contiguous() : !t.is_non_overlapping_and_dense())
                bad(each ? "the gradients of stacked adapters must be contiguous" : "the gradients must be dense in memory");
            if (each && (t.dim() < 1 || t.size(0) != groups))
                bad("the gradients of " + std::to_string(groups) + " stacked adapters must have that leading dimension, not " + shape_of(t.sizes()));
            history(t);
            c.elements = (uint64_t)t.numel();
            if (apart) {
                const at::Tensor& o = *tensor((*outs)[i], "every entry of out");
                if (o.sizes() != t.sizes() || o.device() != t.device() || (o.scalar_type() != t.scalar_type() && o.scalar_type() != at::kFloat))
                    bad("an entry of out must be " + shape_of(t.sizes()) + " on " + t.device().str() + ", " + type_of(t.scalar_type()) + " or torch.float32");
                if (o.strides() != t.strides() && !(o.is_contiguous() && t.is_contiguous())) bad("an entry of out must have its gradient's layout in memory");
                history(o);
                c.out_dtype = dtype_code(o.scalar_type());
                c.out = o.mutable_data_ptr();
                c.grad = t.const_data_ptr();
            } else {
                c.grad = c.out = t.mutable_data_ptr();
            }
            list.push_back(c);
        }
        if (!like) bad("grads has no tensors");
        ts_clip_args q{};
        q.groups = (uint32_t)groups, q.count = list.size(), q.tensors = list.data();
        if (THPVariable_Check(args[1])) {
            const at::Tensor& m = THPVariable_Unpack(args[1]);
            q.one_max = m.numel() == 1;
            if (m.scalar_type() != at::kFloat || !m.is_contiguous() || (!q.one_max && (!each || m.dim() != 1 || m.size(0) != groups)))
                bad("max_norm must be a number, one float32 value or one for each adapter, not " + type_of(m.scalar_type()) + " " + shape_of(m.sizes()));
            if (m.device() != like->device()) bad("max_norm is on " + m.device().str() + ", not on " + like->device().str());
            no_history(&m);
            q.max_norms = static_cast<const float*>(m.const_data_ptr());
        } else {
            q.max_norm = (float)number(args[1]);
            if (!(q.max_norm >= 0.f)) bad("max_norm must not be negative");
        }
        q.device = on_device(*like, "the tensors");
        at::Tensor norms = each ? at::empty({groups}, like->options().dtype(at::kFloat)) : at::empty({}, like->options().dtype(at::kFloat));
        q.norms = static_cast<float*>(norms.mutable_data_ptr());
        q.stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)q.device).stream();
        uint64_t bytes = 0;
        finish(g.clip_workspace(&q, &bytes), "ts_clip_workspace");
        at::Tensor ws = at::empty({(int64_t)bytes}, like->options().dtype(at::kByte));
        q.workspace = ws.mutable_data_ptr();
        q.workspace_bytes = bytes;
        finish(g.clip(&q), "ts_clip_gradients");
        const Items& changed = apart ? *outs : grads;
        for (Py_ssize_t i = 0; i < grads.size(); i++)
            if (grads[i] != Py_None) written(THPVariable_Unpack(changed[i]));
        return THPVariable_Wrap(norms);
    });
}

// (addresses of ts_adapter_workspace, ts_adapter_project, ts_adapter_project_backward, ts_logit_rules, ts_loss_workspace,
// ts_token_logprobs, ts_token_logprobs_backward, ts_policy_loss, ts_preference_loss, ts_clip_workspace, ts_clip_gradients, _lib.check)
PyObject* bind(PyObject*, PyObject* args) {
    unsigned long long a[11];
    PyObject* check;
    if (!PyArg_ParseTuple(args, "KKKKKKKKKKKO", &a[0], &a[1], &a[2], &a[3], &a[4], &a[5], &a[6], &a[7], &a[8], &a[9], &a[10], &check)) return nullptr;
    g.workspace = reinterpret_cast<decltype(g.workspace)>(a[0]);
    g.project = reinterpret_cast<decltype(g.project)>(a[1]);
    g.backward = reinterpret_cast<decltype(g.backward)>(a[2]);
    g.rules = reinterpret_cast<decltype(g.rules)>(a[3]);
    g.loss_workspace = reinterpret_cast<decltype(g.loss_workspace)>(a[4]);
    for (int i = 0; i < 4; i++) g.losses[i] = reinterpret_cast<decltype(g.losses[i])>(a[5 + i]);
    g.clip_workspace = reinterpret_cast<decltype(g.clip_workspace)>(a[9]);
    g.clip = reinterpret_cast<decltype(g.clip)>(a[10]);
    Py_INCREF(check);
    Py_XSETREF(g.check, check);
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {{"bind", bind, METH_VARARGS, nullptr},
                         {"project", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(project)), METH_FASTCALL, nullptr},
                         {"backward", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(backward)), METH_FASTCALL, nullptr},
                         {"rules", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(rules)), METH_FASTCALL, nullptr},
                         {"logprobs", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(logprobs)), METH_FASTCALL, nullptr},
                         {"logprobs_backward", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(logprobs_backward)), METH_FASTCALL, nullptr},
                         {"policy", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(policy)), METH_FASTCALL, nullptr},
                         {"preference", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(preference)), METH_FASTCALL, nullptr},
                         {"clip", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(clip)), METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_torch_ops", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__torch_ops() {
    PyObject* m = PyModule_Create(&module);
    if (m && PyModule_AddStringConstant(m, "built_for", TSGPU_BUILT_FOR) < 0) Py_CLEAR(m);
    return m;
}
