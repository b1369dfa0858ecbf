// answers_bind.cpp — the Python entry points of ytm_b200.answers: argument
// checks, output tensors and the calls of libytm's C ABI.  They stand here and
// not in Python because one sample's answer takes the GPU 2 us and an
// interpreter's share of a call 10.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cfloat>
#include <string>

#include "../../include/ytm.h"

namespace {

using at::ScalarType;
using at::Tensor;

// Raised as the Python exception `type` with the message.
struct Error {
    PyObject *type;
    std::string text;
};

// An exception class of a module (never released: it lives as long as that).
PyObject *exception(const char *module, const char *name) {
    PyObject *m = PyImport_ImportModule(module);
    PyObject *type = m ? PyObject_GetAttrString(m, name) : nullptr;
    Py_XDECREF(m);
    if (type) return type;
    PyErr_Clear();
    return PyExc_RuntimeError;
}

[[noreturn]] void type_error(const std::string &s) { throw Error{PyExc_TypeError, s}; }
[[noreturn]] void value_error(const std::string &s) { throw Error{PyExc_ValueError, s}; }

std::string num(int64_t v) { return std::to_string(v); }

enum : unsigned { I32 = 1, F32 = 2, F16 = 4, BF16 = 8, I64 = 16, U8 = 32, FLOATS = F32 | F16 | BF16, SUMS = I32 | FLOATS };

unsigned bit_of(ScalarType t) {
    switch (t) {
        case ScalarType::Int: return I32;
        case ScalarType::Float: return F32;
        case ScalarType::Half: return F16;
        case ScalarType::BFloat16: return BF16;
        case ScalarType::Long: return I64;
        case ScalarType::Byte: return U8;
        default: return 0;
    }
}

std::string names(unsigned types) {
    static const char *const of[] = {"int32", "float32", "float16", "bfloat16", "int64", "uint8"};
    std::string s;
    for (int i = 0; i < 6; ++i)
        if (types >> i & 1) s += (s.empty() ? "" : " or ") + std::string(of[i]);
    return s;
}

int ytm_type(ScalarType t) {
    return t == ScalarType::Int ? YTM_I32 : t == ScalarType::Float ? YTM_F32 : t == ScalarType::Half ? YTM_F16 : YTM_BF16;
}

// One tensor argument, checked, with contiguous rows.
Tensor need(PyObject *o, const char *name, int dim, unsigned types, const Tensor *with = nullptr) {
    if (!THPVariable_Check(o)) type_error(std::string(name) + " must be a torch tensor, got " + Py_TYPE(o)->tp_name);
    const Tensor &t = THPVariable_Unpack(o);
    if (t.layout() != at::kStrided) type_error(std::string(name) + " must be strided, got " + c10::str(t.layout()));
    if (!(bit_of(t.scalar_type()) & types)) type_error(std::string(name) + " must be " + names(types) + ", got " + c10::toString(t.scalar_type()));
    if (t.dim() != dim) value_error(std::string(name) + " must have " + num(dim) + " dimension" + (dim != 1 ? "s" : "") + ", got " + num(t.dim()));
    if (!t.is_cuda()) value_error(std::string(name) + " must be on a CUDA device, got " + t.device().str());
    if (with && t.device() != with->device())
        value_error(std::string(name) + " is on " + t.device().str() + ", the other tensors on " + with->device().str());
    if (t.requires_grad() && c10::GradMode::is_enabled())
        value_error(std::string(name) + " requires grad: these operators do not record into autograd (detach it)");
    if (t._fw_grad(0).defined() && c10::AutogradState::get_tls_state().get_fw_grad_mode())
        value_error(std::string(name) + " carries a forward-mode tangent: these operators do not compute one (detach it)");
    if (t.numel() && !t.const_data_ptr()) value_error(std::string(name) + " has no memory of its own");
    if (t.is_neg()) return t.resolve_neg().contiguous();
    return dim && t.stride(-1) != 1 && t.size(-1) > 1 ? t.contiguous() : t;
}

Tensor vector(PyObject *o, const char *name, int64_t n, unsigned types, const Tensor &with) {
    Tensor t = need(o, name, 1, types, &with);
    if (t.size(0) != n) value_error(std::string(name) + " must have " + num(n) + " values, got " + num(t.size(0)));
    return t;
}

Tensor allowed_words(PyObject *o, int64_t n, int64_t k, const Tensor &with) {
    Tensor t = need(o, "allowed", 2, I32, &with);
    if (t.size(1) != (k + 31) / 32 || (t.size(0) != 1 && t.size(0) != n))
        value_error("allowed must be int32 [" + num(n) + " or 1, " + num((k + 31) / 32) + "], got [" + num(t.size(0)) + ", " + num(t.size(1)) + "]");
    return t;
}

int64_t row_stride(const Tensor &t) { return t.size(0) > 1 ? t.stride(0) : 0; }

// A number for all rows (a tensor without dimensions on the CPU is one), or float32
// [n], or [] for all rows.
struct Knob {
    Tensor rows;
    float all = 0.f;
    const float *ptr() const { return rows.defined() ? rows.const_data_ptr<float>() : nullptr; }
};

Knob knob(PyObject *o, const char *name, int64_t n, const Tensor &with, bool positive) {
    Knob k;
    if (THPVariable_Check(o)) {
        const Tensor &t = THPVariable_Unpack(o);
        if (t.dim() || t.is_cuda()) {
            k.rows = t.dim() ? vector(o, name, n, F32, with) : need(o, name, 0, F32, &with).expand({n}).contiguous();
            return k;
        }
    }
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw Error{nullptr, ""};
    k.all = (float)v;
    // below the smallest normal number the reciprocal leaves the type
    if (positive && !(k.all >= FLT_MIN)) {
        char text[32];
        PyOS_snprintf(text, sizeof text, "%g", v);
        value_error(std::string(name) + " must be positive (at least 2^-126), got " + text);
    }
    return k;
}

int64_t integer(PyObject *o) {
    const int64_t v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw Error{nullptr, ""};
    return v;
}

Tensor empty(at::IntArrayRef size, ScalarType type, const Tensor &with) {
    return at::empty(size, at::TensorOptions().dtype(type).device(with.device()));
}

// A library call on the current stream of the tensors' device, which is the
// current one, without the interpreter's lock; f does nothing but the call.
template <typename F>
void call(const char *what, const Tensor &with, F f) {
    void *stream = c10::cuda::getCurrentCUDAStream(with.device().index()).stream();
    ytm_status rc;
    std::string text;
    Py_BEGIN_ALLOW_THREADS
    rc = f(stream);
    if (rc) text = ytm_last_error();  // of this thread
    Py_END_ALLOW_THREADS
    if (!rc) return;
    throw Error{exception("ytm_b200._lib", "YTMError"), std::string(what) + ": status " + num(rc) + ": " + text};
}

PyObject *wrap(const Tensor &t) {
    if (t.defined()) return THPVariable_Wrap(t);
    Py_RETURN_NONE;
}

PyObject *tuple(std::initializer_list<Tensor> ts) {
    PyObject *r = PyTuple_New((Py_ssize_t)ts.size());
    Py_ssize_t i = 0;
    for (const Tensor &t : ts) PyTuple_SET_ITEM(r, i++, wrap(t));
    return r;
}

// Runs f with exceptions turned into Python's.
template <typename F>
PyObject *guarded(Py_ssize_t got, Py_ssize_t want, F f) {
    if (got != want) {
        PyErr_Format(PyExc_TypeError, "%zd arguments expected, got %zd", want, got);
        return nullptr;
    }
    try {
        return f();
    } catch (const Error &e) {
        if (e.type) PyErr_SetString(e.type, e.text.c_str());
    } catch (const c10::OutOfMemoryError &e) {
        PyErr_SetString(exception("torch", "OutOfMemoryError"), e.what_without_backtrace());
    } catch (const c10::Error &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
    } catch (const std::exception &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}

void check_group(int64_t group) {
    if (group != 32 && group != 64 && group != 128) value_error("group must be 32, 64 or 128");
}

ScalarType float_type(PyObject *o, const char *name) {
    if (!THPDtype_Check(o)) type_error(std::string(name) + " must be float32, float16 or bfloat16");
    const ScalarType t = reinterpret_cast<THPDtype *>(o)->scalar_type;
    if (!(bit_of(t) & FLOATS)) type_error(std::string(name) + " must be float32, float16 or bfloat16");
    return t;
}

// (weights, group, scale_dtype)
PyObject *q4_pack(PyObject *, PyObject *const *a, Py_ssize_t argc) {
    return guarded(argc, 3, [&]() -> PyObject * {
        Tensor w = need(a[0], "weights", 2, I32 | F32);
        const int64_t C = w.size(0), K = w.size(1), group = integer(a[1]);
        if (!C || !K) value_error("weights must have at least one clause and one class");
        if (C > INT32_MAX || K > INT32_MAX) value_error("weights are too large");
        check_group(group);
        const ScalarType st = float_type(a[2], "scale_dtype");
        const c10::cuda::CUDAGuard guard(w.device());
        if (C > 1 && w.stride(0) < K) w = w.contiguous();
        Tensor packed = empty({K, (C + 31) / 32 * 16}, ScalarType::Byte, w), scales = empty({K, (C + group - 1) / group}, st, w);
        const void *const from = w.const_data_ptr();
        uint8_t *const to = packed.mutable_data_ptr<uint8_t>();
        void *const to_scales = scales.mutable_data_ptr();
        call("ytm_q4_pack", w, [&](void *s) {
            return ytm_q4_pack(from, ytm_type(w.scalar_type()), C > 1 ? w.stride(0) : K, (int32_t)C, (int32_t)K, (int32_t)group, to,
                               to_scales, ytm_type(st), s);
        });
        return tuple({packed, scales});
    });
}

// (x, packed, scales, group, bias, clauses, out_dtype)
PyObject *q4_votes(PyObject *, PyObject *const *a, Py_ssize_t argc) {
    return guarded(argc, 7, [&]() -> PyObject * {
        const Tensor x = need(a[0], "x", 2, SUMS), packed = need(a[1], "packed", 2, U8, &x), scales = need(a[2], "scales", 2, FLOATS, &x);
        const int64_t n = x.size(0), K = packed.size(0), group = integer(a[3]);
        const bool bits = x.scalar_type() == ScalarType::Int;
        if (a[5] == Py_None && bits) value_error("clauses must be given with clause bits");
        const int64_t C = a[5] == Py_None ? x.size(1) : integer(a[5]);
        if (C < 1 || K < 1) value_error("needs at least one clause and one class");
        if (C > INT32_MAX || K > INT32_MAX) value_error("too many clauses or classes");
        check_group(group);
        const int64_t words = (C + 31) / 32, G = (C + group - 1) / group, width = bits ? words : C;
        if (x.size(1) != width) value_error("x has " + num(x.size(1)) + " columns, " + num(C) + " clauses need " + num(width));
        if (packed.size(1) != words * 16 || !packed.is_contiguous())
            value_error("packed must be contiguous [classes, " + num(words * 16) + "] for " + num(C) + " clauses");
        if (scales.size(0) != K || scales.size(1) != G || !scales.is_contiguous())
            value_error("scales must be contiguous [" + num(K) + ", " + num(G) + "]");
        const ScalarType yt = float_type(a[6], "out_dtype");
        Tensor bias;
        if (a[4] != Py_None) bias = vector(a[4], "bias", K, F32, x);
        Tensor y = empty({n, K}, yt, x);
        if (!n) return wrap(y);
        const int xt = bits ? YTM_BITS : ytm_type(x.scalar_type());
        const c10::cuda::CUDAGuard guard(x.device());
        Tensor ws = empty({(int64_t)ytm_q4_votes_workspace_bytes(xt, n, (int32_t)C, (int32_t)K, (int32_t)group)}, ScalarType::Byte, x);
        const void *const px = x.const_data_ptr(), *const ps = scales.const_data_ptr();
        const uint8_t *const pw = packed.const_data_ptr<uint8_t>();
        const float *const pb = bias.defined() ? bias.const_data_ptr<float>() : nullptr;
        void *const py = y.mutable_data_ptr(), *const scratch = ws.mutable_data_ptr();
        call("ytm_q4_votes", x, [&](void *s) {
            return ytm_q4_votes(px, xt, row_stride(x), n, (int32_t)C, pw, ps, ytm_type(scales.scalar_type()), (int32_t)group, (int32_t)K,
                                pb, py, ytm_type(yt), scratch, s);
        });
        return wrap(y);
    });
}

// (cs, bias, allowed, history, lengths, repetition, frequency, presence, temperature, adjusted)
PyObject *answer(PyObject *, PyObject *const *a, Py_ssize_t argc) {
    return guarded(argc, 10, [&]() -> PyObject * {
        const Tensor cs = need(a[0], "cs", 2, SUMS);
        const int64_t n = cs.size(0), k = cs.size(1);
        if (k < 1) value_error("cs must have at least one class");
        if (k > INT32_MAX) value_error("cs has too many classes");
        ytm_answer_args g = {};
        g.cs = cs.const_data_ptr();
        g.cs_stride = row_stride(cs);
        g.n = n;
        g.k = (int32_t)k;
        g.cs_type = ytm_type(cs.scalar_type());
        Tensor bias, allowed, history, lengths;
        if (a[1] != Py_None) {
            if (THPVariable_Check(a[1]) && THPVariable_Unpack(a[1]).dim() == 2) {
                bias = need(a[1], "bias", 2, F32, &cs);
                if (bias.size(0) != n || bias.size(1) != k)
                    value_error("bias must be [" + num(k) + "] or [" + num(n) + ", " + num(k) + "], got [" + num(bias.size(0)) + ", " + num(bias.size(1)) + "]");
                g.bias_stride = row_stride(bias);
            } else {
                bias = vector(a[1], "bias", k, F32, cs);
            }
            g.bias = bias.const_data_ptr<float>();
        }
        if (a[2] != Py_None) {
            allowed = allowed_words(a[2], n, k, cs);
            g.allowed = (const uint32_t *)allowed.const_data_ptr();
            g.allowed_stride = row_stride(allowed);
        }
        if (a[3] != Py_None) {
            history = need(a[3], "history", 2, I32 | I64, &cs);
            if (history.size(0) != n) value_error("history must have " + num(n) + " rows, got " + num(history.size(0)));
            if (a[4] != Py_None) lengths = vector(a[4], "lengths", n, I32, cs);
            if (history.size(1) > INT32_MAX) value_error("history must have fewer than 2^31 entries a row");
            if (history.size(1)) {
                g.history = history.const_data_ptr();
                g.history_stride = row_stride(history);
                g.history_len = (int32_t)history.size(1);
                g.history_64 = history.scalar_type() == ScalarType::Long;
                g.lengths = lengths.defined() ? lengths.const_data_ptr<int32_t>() : nullptr;
            }
        } else if (a[4] != Py_None) {
            value_error("lengths needs history");
        }
        const Knob rep = knob(a[5], "repetition", n, cs, true), fre = knob(a[6], "frequency", n, cs, false),
                   pre = knob(a[7], "presence", n, cs, false), tem = knob(a[8], "temperature", n, cs, true);
        g.repetition = rep.ptr();
        g.frequency = fre.ptr();
        g.presence = pre.ptr();
        g.temperature = tem.ptr();
        g.repetition_all = rep.all;
        g.frequency_all = fre.all;
        g.presence_all = pre.all;
        g.temperature_all = tem.all;
        const int adjusted = PyObject_IsTrue(a[9]);
        if (adjusted < 0) throw Error{nullptr, ""};
        Tensor choice = empty({n}, ScalarType::Long, cs), logprob = empty({n}, ScalarType::Float, cs), z;
        if (adjusted) z = empty({n, k}, ScalarType::Float, cs);
        g.choice = choice.mutable_data_ptr<int64_t>();
        g.logprob = logprob.mutable_data_ptr<float>();
        g.adjusted = adjusted ? z.mutable_data_ptr<float>() : nullptr;
        const c10::cuda::CUDAGuard guard(cs.device());
        call("ytm_answer", cs, [&](void *s) { return ytm_answer(&g, s); });
        return tuple({choice, logprob, z});
    });
}

// (cs, target, bias, allowed, temperature, weight)
PyObject *class_loss(PyObject *, PyObject *const *a, Py_ssize_t argc) {
    return guarded(argc, 6, [&]() -> PyObject * {
        const Tensor cs = need(a[0], "cs", 2, SUMS);
        const int64_t n = cs.size(0), k = cs.size(1);
        if (k < 1) value_error("cs must have at least one class");
        if (k > INT32_MAX) value_error("cs has too many classes");
        ytm_loss_args g = {};
        g.cs = cs.const_data_ptr();
        g.cs_stride = row_stride(cs);
        g.n = n;
        g.k = (int32_t)k;
        g.cs_type = ytm_type(cs.scalar_type());
        const Tensor target = vector(a[1], "target", n, I32 | I64, cs);
        g.target = target.const_data_ptr();
        g.target_64 = target.scalar_type() == ScalarType::Long;
        Tensor bias, allowed, weight, dcs, dbias, ws;
        if (a[2] != Py_None) {
            bias = vector(a[2], "bias", k, F32, cs);
            g.bias = bias.const_data_ptr<float>();
        }
        if (a[3] != Py_None) {
            allowed = allowed_words(a[3], n, k, cs);
            g.allowed = (const uint32_t *)allowed.const_data_ptr();
            g.allowed_stride = row_stride(allowed);
        }
        const Knob tem = knob(a[4], "temperature", 1, cs, true);
        g.temperature = tem.ptr();
        g.temperature_all = tem.all;
        if (a[5] != Py_None) {
            weight = vector(a[5], "weight", n, F32, cs);
            g.weight = weight.const_data_ptr<float>();
        }
        Tensor loss = empty({n}, ScalarType::Float, cs), dtem = empty({1}, ScalarType::Float, cs);
        g.loss = loss.mutable_data_ptr<float>();
        g.dtemperature = dtem.mutable_data_ptr<float>();
        if (g.cs_type != YTM_I32) {
            dcs = empty({n, k}, cs.scalar_type(), cs);
            g.dcs = dcs.mutable_data_ptr();
        }
        if (bias.defined()) {
            dbias = empty({k}, ScalarType::Float, cs);
            g.dbias = dbias.mutable_data_ptr<float>();
        }
        const c10::cuda::CUDAGuard guard(cs.device());
        const uint64_t bytes = ytm_class_loss_workspace_bytes(n, g.k, g.cs_type, g.cs_stride);
        if (bytes) ws = empty({(int64_t)bytes}, ScalarType::Byte, cs);
        void *const scratch = bytes ? ws.mutable_data_ptr() : nullptr;
        call("ytm_class_loss", cs, [&](void *s) { return ytm_class_loss(&g, scratch, s); });
        return tuple({loss, dcs, dbias, dtem});
    });
}

#define YTM_METHOD(f) {#f, (PyCFunction)(void (*)(void))f, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {YTM_METHOD(q4_pack), YTM_METHOD(q4_votes), YTM_METHOD(answer), YTM_METHOD(class_loss), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_answers", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__answers() { return PyModule_Create(&module); }
