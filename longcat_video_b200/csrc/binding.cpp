// The dense attention and the 1-D rotary embedding as Python functions and autograd nodes.
//
// The C ABI of liblcbsa.so does the work, as everywhere in this package; what is here is the way to it.  Through ctypes a call of one
// token costs the host 17 us, three times what the GPU needs for it, and a training step of 511 tokens 190 us for 45 on the GPU, most of it
// for a backward that has to wait for the interpreter.  Arguments are checked in Python (modules/dense_attention.py, modules/rotary.py).
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/variable.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include "../../include/lcbsa.h"

namespace {

struct LibraryError {  // a call into liblcbsa.so failed: LcbsaError of _lib.py
    int code;
    std::string message;
};
void check(int rc) {
    if (rc != LCBSA_OK) throw LibraryError{rc, lcbsa_last_error()};
}

// A [B, H, S, D] operand and its description; copied where the 16-byte rules or a missing stride along S ask for it.  The stride of an axis
// of one is nobody's: it may be anything and counts for nothing.
struct Rows {
    at::Tensor t;
    LcbsaTensor d;
};
Rows rows(at::Tensor t) {
    auto stride = [&t](int i) { return t.size(i) > 1 ? t.stride(i) : i < 3 ? t.size(3) : 1; };
    if (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) t = t.clone(at::MemoryFormat::Contiguous);
    else if (stride(3) != 1 || ((stride(0) | stride(1) | stride(2)) & 7) || (stride(2) == 0)) t = t.contiguous();
    LcbsaTensor d{};
    d.data = t.data_ptr();
    d.dtype = t.scalar_type() == at::kBFloat16 ? LCBSA_BF16 : t.scalar_type() == at::kHalf ? LCBSA_FP16 : LCBSA_FP32;
    for (int i = 0; i < 4; ++i) {
        d.size[i] = t.size(i);
        d.stride[i] = stride(i);
    }
    return Rows{std::move(t), d};
}
at::Tensor dense_like(const at::Tensor& t) { return at::empty(t.sizes(), t.options()); }
void* stream_of(const at::Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

// The scores as LcbsaScores has them, with the tensors that it points into.
struct Scores {
    double scale, cap;
    bool causal;
    int64_t impl;
    at::Tensor slopes, cu_q, cu_k, k_lens, prefix;  // undefined: none

    LcbsaScores desc() const {
        auto ints = [](const at::Tensor& t) { return t.defined() ? static_cast<const int32_t*>(t.data_ptr()) : nullptr; };
        LcbsaScores s{};
        s.scale = (float)scale;
        s.cap = (float)cap;
        s.causal = causal;
        s.impl = (int32_t)impl;
        s.slopes = slopes.defined() ? static_cast<const float*>(slopes.data_ptr()) : nullptr;
        s.cu_q = ints(cu_q);
        s.cu_k = ints(cu_k);
        s.k_len = ints(k_lens);
        s.prefix = ints(prefix);
        if (cu_q.defined()) {
            s.docs = (int32_t)cu_q.size(-1) - 1;
            s.cu_stride = cu_q.dim() == 2 ? cu_q.size(-1) : 0;
        }
        if (prefix.defined() && prefix.dim() == 2) s.prefix_stride = prefix.size(-1);
        return s;
    }
};

struct Result {
    at::Tensor out, lse, rest;
};
Result dense_forward(const at::Tensor& q_in, const at::Tensor& k_in, const at::Tensor& v_in, const Scores& scores, bool need_lse, bool need_rest) {
    const c10::cuda::CUDAGuard guard(q_in.device());
    Result r;
    r.out = dense_like(q_in);
    if (need_lse) r.lse = at::empty(q_in.sizes().slice(0, 3), q_in.options().dtype(at::kFloat));
    if (need_rest) r.rest = at::empty(q_in.sizes(), q_in.options());
    const Rows q = rows(q_in), k = rows(k_in), v = rows(v_in), o = rows(r.out);
    const LcbsaScores s = scores.desc();
    const size_t need = lcbsa_dense_attn_workspace_bytes(&q.d, &k.d, s.impl, 0);
    const at::Tensor ws = need ? at::empty({(int64_t)need}, q_in.options().dtype(at::kByte)) : at::Tensor();
    check(lcbsa_dense_attn_fwd(&q.d, &k.d, &v.d, &s, &o.d, need_lse ? static_cast<float*>(r.lse.data_ptr()) : nullptr,
                               need_rest ? r.rest.data_ptr() : nullptr, need ? ws.data_ptr() : nullptr, need, stream_of(q_in)));
    return r;
}

// What a gradient is differentiated with: an error, when it is asked for (there is no second derivative here).
torch::autograd::variable_list once(torch::autograd::variable_list grads, const char* what) {
    if (!at::GradMode::is_enabled()) return grads;
    for (at::Tensor& g : grads) g = g.detach().set_requires_grad(true);  // else the node is not attached
    auto node = std::make_shared<torch::autograd::DelayedError>(std::string("trying to differentiate twice through ") + what, (int64_t)grads.size());
    return (*node)(std::move(grads));
}
// Errors of a backward leave through the engine, which knows no LcbsaError.
template <typename F>
void in_backward(F&& f) {
    try {
        f();
    } catch (const LibraryError& e) {
        TORCH_CHECK(false, "lcbsa error ", e.code, ": ", e.message);
    }
}

struct DenseAttention : torch::autograd::Function<DenseAttention> {
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k,
                                                  const at::Tensor& v, const Scores& scores) {
        const Result r = dense_forward(q, k, v, scores, true, true);
        ctx->save_for_backward({q, k, v, r.out, r.lse, r.rest, scores.slopes, scores.cu_q, scores.cu_k, scores.k_lens, scores.prefix});
        ctx->saved_data["scale"] = scores.scale;
        ctx->saved_data["cap"] = scores.cap;
        ctx->saved_data["causal"] = scores.causal;
        ctx->mark_non_differentiable({r.lse});
        ctx->set_materialize_grads(false);
        return {r.out, r.lse};
    }

    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        torch::autograd::variable_list out(4);
        if (!grads[0].defined()) return out;
        torch::autograd::variable_list d;
        {
            const at::NoGradGuard no_grad;
            const c10::cuda::CUDAGuard guard(saved[0].device());
            const Scores scores{ctx->saved_data["scale"].toDouble(), ctx->saved_data["cap"].toDouble(), ctx->saved_data["causal"].toBool(),
                                LCBSA_ATTN_AUTO, saved[6], saved[7], saved[8], saved[9], saved[10]};
            const Rows q = rows(saved[0]), k = rows(saved[1]), v = rows(saved[2]), o = rows(saved[3]), g = rows(grads[0]);
            const Rows dq = rows(dense_like(q.t)), dk = rows(dense_like(k.t)), dv = rows(dense_like(v.t));
            const LcbsaScores s = scores.desc();
            const size_t need = lcbsa_dense_attn_workspace_bytes(&q.d, &k.d, s.impl, 1);
            const at::Tensor ws = at::empty({(int64_t)need}, q.t.options().dtype(at::kByte));
            in_backward([&] {
                check(lcbsa_dense_attn_bwd(&q.d, &k.d, &v.d, &o.d, &g.d, &s, static_cast<const float*>(saved[4].data_ptr()), saved[5].data_ptr(),
                                           &dq.d, &dk.d, &dv.d, ws.data_ptr(), need, stream_of(q.t)));
            });
            d = {dq.t, dk.t, dv.t};
        }
        d = once(std::move(d), "dense_attention");
        out[0] = d[0];
        out[1] = d[1];
        out[2] = d[2];
        return out;
    }
};

struct RotaryCall {
    const uint64_t* turns;
    int pairs;
    double factor;
    at::Tensor positions;  // undefined: none
    int64_t offset;
    bool interleaved;
};
torch::autograd::variable_list rotary_launch(const torch::autograd::variable_list& xs, const RotaryCall& c, bool inverse) {
    const c10::cuda::CUDAGuard guard(xs[0].device());
    torch::autograd::variable_list outs, keep;
    LcbsaTensor xd[2], od[2];
    for (size_t i = 0; i < xs.size(); ++i) {
        outs.push_back(dense_like(xs[i]));
        const Rows x = rows(xs[i]), o = rows(outs[i]);
        xd[i] = x.d;
        od[i] = o.d;
        keep.push_back(x.t);
    }
    const void* pos = nullptr;
    int bits = 32;
    int64_t sb = 0, ss = 0;
    if (c.positions.defined()) {
        pos = c.positions.data_ptr();
        bits = c.positions.scalar_type() == at::kLong ? 64 : 32;
        ss = c.positions.stride(-1);
        sb = c.positions.dim() == 2 && c.positions.size(0) > 1 ? c.positions.stride(0) : 0;
    }
    check(lcbsa_rotary(xd, od, (int)xs.size(), c.turns, c.pairs, c.interleaved, inverse, (float)c.factor, pos, bits, sb, ss, c.offset,
                       stream_of(xs[0])));
    return outs;
}

// The embedding is linear: the gradient is the rotation back, times the same factor.
struct Rotary : torch::autograd::Function<Rotary> {
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const RotaryCall& c, const at::Tensor& x0, const std::optional<at::Tensor>& x1) {
        ctx->saved_data["turns"] = std::vector<int64_t>(reinterpret_cast<const int64_t*>(c.turns), reinterpret_cast<const int64_t*>(c.turns) + c.pairs);
        ctx->saved_data["factor"] = c.factor;
        ctx->saved_data["offset"] = c.offset;
        ctx->saved_data["interleaved"] = c.interleaved;
        ctx->save_for_backward({c.positions});
        ctx->set_materialize_grads(false);
        return rotary_launch(x1 ? torch::autograd::variable_list{x0, *x1} : torch::autograd::variable_list{x0}, c, false);
    }

    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
        const auto turns = ctx->saved_data["turns"].toIntVector();
        const RotaryCall c{reinterpret_cast<const uint64_t*>(turns.data()), (int)turns.size(), ctx->saved_data["factor"].toDouble(),
                           ctx->get_saved_variables()[0], ctx->saved_data["offset"].toInt(), ctx->saved_data["interleaved"].toBool()};
        torch::autograd::variable_list there, out(3);
        std::vector<size_t> where;
        for (size_t i = 0; i < grads.size(); ++i)
            if (grads[i].defined()) {
                there.push_back(grads[i]);
                where.push_back(i);
            }
        if (there.empty()) return out;
        torch::autograd::variable_list d;
        {
            const at::NoGradGuard no_grad;
            in_backward([&] { d = rotary_launch(there, c, true); });
        }
        d = once(std::move(d), "the rotary embedding");
        for (size_t i = 0; i < where.size(); ++i) out[1 + where[i]] = d[i];
        return out;
    }
};

// ------------------------------------------------------------------------------------------ Python

at::Tensor maybe(PyObject* o) { return o == Py_None ? at::Tensor() : THPVariable_Unpack(o); }

PyObject* raise(const LibraryError& e) {
    PyObject* lib = PyImport_ImportModule("longcat_video_b200._lib");
    if (lib == nullptr) return nullptr;
    PyObject* type = PyObject_GetAttrString(lib, "LcbsaError");
    Py_DECREF(lib);
    if (type == nullptr) return nullptr;
    PyObject* err = PyObject_CallFunction(type, "is", e.code, e.message.c_str());
    if (err != nullptr) PyErr_SetObject(type, err);
    Py_XDECREF(err);
    Py_DECREF(type);
    return nullptr;
}

PyObject* tuple_of(const torch::autograd::variable_list& ts) {
    PyObject* r = PyTuple_New((Py_ssize_t)ts.size());
    for (size_t i = 0; r != nullptr && i < ts.size(); ++i) PyTuple_SET_ITEM(r, (Py_ssize_t)i, THPVariable_Wrap(ts[i]));
    return r;
}

// Whether the call is recorded for a backward.  Under stream capture a leaf that also belongs to a live graph made on another stream is
// refused: the backward would wait for that stream, which no capture can, and the error would come up in the engine.
bool wants_grad(std::initializer_list<const at::Tensor*> ts) {
    if (!at::GradMode::is_enabled()) return false;
    bool wants = false;
    for (const at::Tensor* t : ts) wants |= t->requires_grad();
    if (wants && c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None) {
        for (const at::Tensor* t : ts) {
            if (!t->requires_grad() || t->grad_fn() != nullptr) continue;
            const auto node = torch::autograd::impl::try_get_grad_accumulator(*t);
            if (node == nullptr) continue;
            const auto stream = node->stream();
            TORCH_CHECK(!stream || *stream == c10::cuda::getCurrentCUDAStream(t->get_device()).unwrap(),
                        "a leaf of this captured call also belongs to a live graph made on another stream: release that graph before the capture");
        }
    }
    return wants;
}

// There is no rule that carries a tangent on: an input that has one is an error, not a result without it.
void no_tangents(std::initializer_list<const at::Tensor*> ts) {
    for (const at::Tensor* t : ts)
        TORCH_CHECK_NOT_IMPLEMENTED(!t->_fw_grad(0).defined(), "no forward-mode derivative: an input carries a tangent");
}

// dense_attention(q, k, v, scale, cap, causal, slopes, cu_q, cu_k, k_lens, prefix, return_lse, impl) -> out or (out, lse)
PyObject* py_dense_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    try {
        if (n != 13) return PyErr_Format(PyExc_TypeError, "13 arguments");
        const at::Tensor q = THPVariable_Unpack(a[0]), k = THPVariable_Unpack(a[1]), v = THPVariable_Unpack(a[2]);
        const Scores s{PyFloat_AsDouble(a[3]), PyFloat_AsDouble(a[4]), PyObject_IsTrue(a[5]) == 1, PyLong_AsLongLong(a[12]), maybe(a[6]), maybe(a[7]), maybe(a[8]), maybe(a[9]), maybe(a[10])};
        if (PyErr_Occurred()) return nullptr;
        const bool return_lse = PyObject_IsTrue(a[11]) == 1;
        no_tangents({&q, &k, &v});
        at::Tensor out, lse;
        if (wants_grad({&q, &k, &v})) {
            const auto r = DenseAttention::apply(q, k, v, s);
            out = r[0];
            lse = r[1];
        } else {
            Result r = dense_forward(q, k, v, s, return_lse, false);
            out = std::move(r.out);
            lse = std::move(r.lse);
        }
        return return_lse ? tuple_of({out, lse}) : THPVariable_Wrap(out);
    } catch (const LibraryError& e) {
        return raise(e);
    }
    END_HANDLE_TH_ERRORS
}

// rotary(xs, address of the turns, pairs, factor, positions, offset, interleaved) -> tuple; xs: one or two tensors
PyObject* py_rotary(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    try {
        if (n != 7 || !PyTuple_Check(a[0]) || PyTuple_GET_SIZE(a[0]) < 1 || PyTuple_GET_SIZE(a[0]) > 2) return PyErr_Format(PyExc_TypeError, "7 arguments, the first one or two tensors");
        torch::autograd::variable_list xs;
        for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(a[0]); ++i) xs.push_back(THPVariable_Unpack(PyTuple_GET_ITEM(a[0], i)));
        const RotaryCall c{static_cast<const uint64_t*>(PyLong_AsVoidPtr(a[1])), (int)PyLong_AsLong(a[2]), PyFloat_AsDouble(a[3]), maybe(a[4]),
                           PyLong_AsLongLong(a[5]), PyObject_IsTrue(a[6]) == 1};
        if (PyErr_Occurred()) return nullptr;
        for (const at::Tensor& x : xs) no_tangents({&x});
        const bool grad = xs.size() == 2 ? wants_grad({&xs[0], &xs[1]}) : wants_grad({&xs[0]});
        return tuple_of(grad ? Rotary::apply(c, xs[0], xs.size() == 2 ? std::optional<at::Tensor>(xs[1]) : std::nullopt) : rotary_launch(xs, c, false));
    } catch (const LibraryError& e) {
        return raise(e);
    }
    END_HANDLE_TH_ERRORS
}

PyMethodDef kMethods[] = {
    {"dense_attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_dense_attention)), METH_FASTCALL, nullptr},
    {"rotary", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_rotary)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_binding", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__binding(void) { return PyModule_Create(&kModule); }
