// The host side of the training operators: checks of arguments, output tensors and the call of libisingdiff's entry points, as the
// Python module isingdiff._host.  No kernels here and no link with the library: bind() is given the addresses of its entry points.
//
// Why not in Python: an operator of a small map takes the device 6 us and a step over 66 tensors 9 us, while asking each of 66
// parameters and gradients for its type, device, shape, strides and address through Python alone takes 40 us.  Here group_norm_forward
// costs the host 6.5 us (few groups; the plan weighs every tile, 4 096 groups of 4 take it 30 us more each time), a step over 66 tensors 8.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/full.h>
#include <ATen/ops/zeros.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/VirtualGuardImpl.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/variable.h>

#include <algorithm>
#include <cmath>
#include <string>
#include <vector>

#include "../../include/isingdiff.h"

namespace {

struct Refused { std::string why; };   // becomes a ValueError
struct Raised {};                      // a Python error is set

[[noreturn]] void refuse(const std::string &why) { throw Refused{why}; }

struct {
    decltype(&idm_group_norm_workspace) norm_workspace;
    decltype(&idm_group_norm_forward) norm_forward;
    decltype(&idm_group_norm_backward) norm_backward;
    decltype(&idm_adamw_step) adamw_step;
    decltype(&idm_adamw_moments) adamw_moments;
    PyObject *check, *stream;          // check(rc) raises the library's error; stream(index) is the current hipStream_t
    PyObject *keys[5];                 // of a state, interned
} lib;
enum { STEP, M, V, M_BASE, V_BASE };
const char *const kKeys[5] = {"step", "m", "v", "m_base", "v_base"};

void check(int rc)
{
    if (!rc) return;
    PyObject *none = PyObject_CallFunction(lib.check, "i", rc);
    Py_XDECREF(none);
    if (none) PyErr_SetString(PyExc_RuntimeError, "a call failed without an error");
    throw Raised{};
}

void *stream_of(const at::Tensor &t)
{
    PyObject *index = PyLong_FromLong(t.get_device()), *got = index ? PyObject_CallFunctionObjArgs(lib.stream, index, nullptr) : nullptr;
    Py_XDECREF(index);
    if (!got) throw Raised{};
    void *s = PyLong_AsVoidPtr(got);
    Py_DECREF(got);
    if (!s && PyErr_Occurred()) throw Raised{};
    return s;
}

// fn(args) with the errors of both kinds as Python's
template <typename F> PyObject *guarded(F &&fn)
{
    HANDLE_TH_ERRORS
    try {
        return fn();
    } catch (const Refused &r) {
        PyErr_SetString(PyExc_ValueError, r.why.c_str());
    } catch (const Raised &) {
    }
    return nullptr;
    END_HANDLE_TH_ERRORS
}

int dtype_of(const at::Tensor &t)
{
    switch (t.scalar_type()) {
    case at::kFloat: return IDM_DT_F32;
    case at::kBFloat16: return IDM_DT_BF16;
    case at::kHalf: return IDM_DT_F16;
    default: return -1;
    }
}

// A tensor in memory whose values are what its memory holds (a view that negates is written out)
at::Tensor plain(const at::Tensor &t) { return t.is_neg() ? t.resolve_neg() : t; }

double number(PyObject *o)
{
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw Raised{};
    return v;
}

// ---- group normalisation ----------------------------------------------------------------------------------------------------

struct Norm {
    at::Tensor x, gamma, beta, shift;
    idm_group_norm_desc d = {};
    int64_t batch, channels, groups;
};

// Stride of a sample and of a pixel of t (B, ..., C) where its middle axes are evenly strided; else t becomes a dense copy
void layout(at::Tensor &t, int64_t &sample, int64_t &pixel)
{
    t = plain(t);
    const auto shape = t.sizes(), stride = t.strides();
    const int64_t axes = t.dim(), c = shape[axes - 1], b = shape[0];
    if (!t.is_contiguous()) {
        bool even = t.numel() && (stride[axes - 1] == 1 || c == 1);
        int64_t want = 0;
        pixel = c;
        bool first = true;
        for (int64_t i = axes - 2; even && i >= 1; --i) {
            if (shape[i] == 1) continue;
            if (first) {
                pixel = want = stride[i];
                even = pixel >= c;
                first = false;
            }
            even = even && stride[i] == want;
            want = stride[i] * shape[i];
        }
        if (even) {
            sample = b > 1 ? stride[0] : 0;
            return;
        }
        t = t.contiguous();
    }
    sample = t.numel() / std::max<int64_t>(1, b);
    pixel = c;
}

at::Tensor optional_tensor(PyObject *o, const char *name)
{
    if (o == Py_None) return {};
    if (!THPVariable_Check(o)) refuse(std::string(name) + " must be a tensor or None");
    return THPVariable_Unpack(o);
}

// x, gamma, beta, shift, groups, activation: the checks that forward and backward share
Norm norm_args(PyObject *x, PyObject *gamma, PyObject *beta, PyObject *shift, PyObject *groups, PyObject *activation)
{
    Norm a;
    PyObject *whole = PyNumber_Index(groups);   // (first: it may run anybody's code)
    a.groups = whole ? PyLong_AsLongLong(whole) : 0;
    Py_XDECREF(whole);
    if (PyErr_Occurred()) PyErr_Clear();
    if (!THPVariable_Check(x) || THPVariable_Unpack(x).dim() < 2) refuse("x must be a tensor (B, ..., C)");
    a.x = THPVariable_Unpack(x);
    a.d.dtype = dtype_of(a.x);
    if (a.d.dtype < 0 || a.x.layout() != at::kStrided) refuse("x must be dense float32, bfloat16 or float16");
    const char *act = PyUnicode_Check(activation) ? PyUnicode_AsUTF8(activation) : nullptr;
    if (act && !strcmp(act, "swish")) a.d.activation = IDM_ACT_SWISH;
    else if (act && !strcmp(act, "none")) a.d.activation = IDM_ACT_NONE;
    else { PyErr_Clear(); refuse("activation must be 'none' or 'swish'"); }
    a.batch = a.x.size(0);
    a.channels = a.x.size(-1);
    if (a.groups <= 0 || !a.channels || a.channels % a.groups || a.channels > (1 << 30))
        refuse("groups must divide the " + std::to_string(a.channels) + " channels");
    const int64_t b = a.batch, c = a.channels;
    for (auto [name, from, to] : {std::make_tuple("gamma", gamma, &a.gamma), std::make_tuple("beta", beta, &a.beta)}) {
        *to = optional_tensor(from, name);
        if (to->defined() && (to->scalar_type() != at::kFloat || to->dim() != 1 || to->size(0) != c || to->device() != a.x.device()))
            refuse(std::string(name) + " must be (" + std::to_string(c) + ",) float32 on the device of x");
    }
    a.shift = optional_tensor(shift, "shift");
    if (a.shift.defined()) {
        const at::Tensor &s = a.shift;
        const bool fits = s.dim() == 1 ? s.size(0) == c : s.dim() == 2 && s.size(1) == c && (s.size(0) == 1 || s.size(0) == b);
        if (s.scalar_type() != at::kFloat || s.device() != a.x.device() || !fits)
            refuse("shift must be (" + std::to_string(b) + ", " + std::to_string(c) + "), (1, " + std::to_string(c) + ") or (" +
                   std::to_string(c) + ",) float32 on the device of x");
        if (s.dim() == 2 && b > 1 && s.size(0) == b) a.d.shift_sample = c;
    }
    if (!a.x.is_cuda()) refuse("x must be a CUDA tensor");
    return a;
}

void dense(at::Tensor &t)
{
    if (t.defined()) t = plain(t).contiguous();
}

const void *read(const at::Tensor &t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void *write(const at::Tensor &t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }

bool aligned(std::initializer_list<const void *> ptrs)
{
    uintptr_t all = 0;
    for (const void *p : ptrs) all |= (uintptr_t)p;
    return !(all & 15);
}

// The rest of the descriptor, and the workspace that the call needs
at::Tensor workspace(Norm &a, bool backward, size_t &bytes)
{
    a.d.batch = a.batch;
    a.d.pixels = a.x.numel() / (a.batch * a.channels);
    a.d.channels = (int32_t)a.channels;
    a.d.groups = (int32_t)a.groups;
    check(lib.norm_workspace(&a.d, backward, &bytes));
    return bytes ? at::empty({(int64_t)bytes}, a.x.options().dtype(at::kByte)) : at::Tensor();
}

PyObject *group_norm_forward(PyObject *, PyObject *const *arg, Py_ssize_t)
{
    return guarded([&]() -> PyObject * {
        const double eps = number(arg[5]);
        if (!(eps >= 0) || !std::isfinite((float)eps) || (eps > 0 && (float)eps == 0))
            refuse("eps must be finite, not negative, and above zero in float32 if it is above zero");
        Norm a = norm_args(arg[0], arg[1], arg[2], arg[3], arg[4], arg[6]);
        a.d.eps = (float)eps;
        layout(a.x, a.d.x_sample, a.d.x_pixel);
        const auto opt = a.x.options(), f32 = opt.dtype(at::kFloat);
        at::Tensor y = at::empty(a.x.sizes(), opt), mean, rstd;
        if (!a.x.numel()) {
            mean = at::zeros({a.batch, a.groups}, f32);
            rstd = at::full({a.batch, a.groups}, 1.0 / std::sqrt(eps), f32);
        } else {
            const c10::DeviceGuard guard(a.x.device());
            mean = at::empty({a.batch, a.groups}, f32);
            rstd = at::empty({a.batch, a.groups}, f32);
            dense(a.gamma), dense(a.beta), dense(a.shift);
            const void *x = read(a.x), *gamma = read(a.gamma), *beta = read(a.beta), *shift = read(a.shift);
            a.d.aligned = aligned({x, gamma, beta, shift, write(y)});
            size_t bytes;
            const at::Tensor ws = workspace(a, false, bytes);
            check(lib.norm_forward(a.x.get_device(), &a.d, x, (const float *)gamma, (const float *)beta, (const float *)shift, write(y),
                                   (float *)write(mean), (float *)write(rstd), write(ws), bytes, stream_of(a.x)));
        }
        PyObject *out = PyTuple_New(3);
        if (!out) throw Raised{};
        PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(y));
        PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(mean));
        PyTuple_SET_ITEM(out, 2, THPVariable_Wrap(rstd));
        return out;
    });
}

PyObject *wrap_or_none(const at::Tensor &t)
{
    if (t.defined()) return THPVariable_Wrap(t);
    Py_RETURN_NONE;
}

PyObject *group_norm_backward(PyObject *, PyObject *const *arg, Py_ssize_t)
{
    return guarded([&]() -> PyObject * {
        Norm a = norm_args(arg[1], arg[4], arg[5], arg[6], arg[7], arg[8]);
        at::Tensor dy = optional_tensor(arg[0], "dy"), mean = optional_tensor(arg[2], "mean"), rstd = optional_tensor(arg[3], "rstd");
        if (!dy.defined() || dy.sizes() != a.x.sizes() || dy.scalar_type() != a.x.scalar_type() || dy.device() != a.x.device() ||
            dy.layout() != at::kStrided)
            refuse("dy must have the shape, type and device of x");
        for (const at::Tensor *t : {&mean, &rstd})
            if (!t->defined() || t->dim() != 2 || t->size(0) != a.batch || t->size(1) != a.groups || t->scalar_type() != at::kFloat ||
                t->device() != a.x.device())
                refuse("mean and rstd must be (" + std::to_string(a.batch) + ", " + std::to_string(a.groups) + ") float32 on the device of x");
        const c10::DeviceGuard guard(a.x.device());
        layout(a.x, a.d.x_sample, a.d.x_pixel);
        layout(dy, a.d.dy_sample, a.d.dy_pixel);
        const auto make = [&](const at::Tensor &like) {
            return !like.defined() ? at::Tensor() : a.x.numel() ? at::empty(like.sizes(), like.options()) : at::zeros(like.sizes(), like.options());
        };
        at::Tensor dx = at::empty(a.x.sizes(), a.x.options()), dgamma = make(a.gamma), dbeta = make(a.beta), dshift = make(a.shift);
        if (a.x.numel()) {
            dense(a.gamma), dense(a.beta), dense(a.shift), dense(mean), dense(rstd);
            const void *g = read(dy), *x = read(a.x), *gamma = read(a.gamma), *beta = read(a.beta), *shift = read(a.shift);
            a.d.aligned = aligned({g, x, gamma, beta, shift, write(dx)});
            size_t bytes;
            const at::Tensor ws = workspace(a, true, bytes);
            check(lib.norm_backward(a.x.get_device(), &a.d, g, x, (const float *)read(mean), (const float *)read(rstd), (const float *)gamma,
                                    (const float *)beta, (const float *)shift, write(dx), (float *)write(dgamma), (float *)write(dbeta),
                                    (float *)write(dshift), write(ws), bytes, stream_of(a.x)));
        }
        PyObject *out = PyTuple_New(4);
        if (!out) throw Raised{};
        PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(dx));
        PyTuple_SET_ITEM(out, 1, wrap_or_none(dgamma));
        PyTuple_SET_ITEM(out, 2, wrap_or_none(dbeta));
        PyTuple_SET_ITEM(out, 3, wrap_or_none(dshift));
        return out;
    });
}

PyObject *layout_py(PyObject *, PyObject *t)
{
    return guarded([&]() -> PyObject * {
        if (!THPVariable_Check(t)) refuse("not a tensor");
        at::Tensor x = THPVariable_Unpack(t);
        int64_t sample, pixel;
        layout(x, sample, pixel);
        return Py_BuildValue("(NLL)", THPVariable_Wrap(x), (long long)sample, (long long)pixel);
    });
}

// Whether a backward pass that is captured on the current stream would add into the gradient of one of these on another stream: a leaf
// adds on the stream of the first graph that it was part of, as long as one of those is alive.  (Such a capture ends the process.)
PyObject *adds_elsewhere(PyObject *, PyObject *const *arg, Py_ssize_t n)
{
    return guarded([&]() -> PyObject * {
        for (Py_ssize_t i = 0; i < n; ++i) {
            if (!THPVariable_Check(arg[i])) continue;
            const at::Tensor &t = THPVariable_Unpack(arg[i]);
            if (!t.is_cuda() || !t.requires_grad() || !t.is_leaf()) continue;
            const auto node = torch::autograd::impl::try_get_grad_accumulator(t);
            const auto at = node ? node->stream() : std::nullopt;
            if (at && *at != c10::impl::VirtualGuardImpl(t.device().type()).getStream(t.device())) Py_RETURN_TRUE;
        }
        Py_RETURN_FALSE;
    });
}

// ---- AdamW ---------------------------------------------------------------------------------------------------------------------

constexpr int64_t BLOCK = IDM_ADAMW_BLOCK;

struct State {
    at::Tensor t[5];
    bool eight;
    void *at(int k) const { return t[k].defined() ? t[k].mutable_data_ptr() : nullptr; }
};

// The tensors of a state, as they are
State state_of(PyObject *dict)
{
    State s;
    const auto take = [&](int k) {
        PyObject *o = PyObject_GetItem(dict, lib.keys[k]);
        if (!o) throw Raised{};
        const bool is = THPVariable_Check(o);
        if (is) s.t[k] = THPVariable_Unpack(o);
        Py_DECREF(o);
        if (!is) refuse(std::string("state['") + kKeys[k] + "'] must be a tensor");
    };
    take(M);
    s.eight = s.t[M].scalar_type() == at::kByte;
    for (int k : {STEP, V}) take(k);
    if (s.eight)
        for (int k : {M_BASE, V_BASE}) take(k);
    return s;
}

// Refuses a state that does not fit `total` entries (-1: any whole number of blocks) on `dev` (null: where it is)
void check_state(const State &s, int64_t total, const c10::Device *dev)
{
    const c10::Device on = dev ? *dev : s.t[M].device();
    if (total < 0) total = s.t[M].numel() / BLOCK * BLOCK;
    for (int k = 0; k < (s.eight ? 5 : 3); ++k) {
        const auto want = k == STEP ? at::kLong : k >= M_BASE ? at::kShort : s.eight ? at::kByte : at::kFloat;
        const int64_t n = k == STEP ? 1 : k >= M_BASE ? total / BLOCK : total;
        const at::Tensor &t = s.t[k];
        if (t.scalar_type() != want || t.numel() != n || t.device() != on || t.layout() != at::kStrided || !t.is_contiguous() || t.is_neg())
            refuse(std::string("state['") + kKeys[k] + "'] must be " + std::to_string(n) + " dense " + c10::toString(want) + " values on " +
                   on.str() + ": make it with adamw_state for these parameters");
    }
    if (total && s.at(M) == s.at(V)) refuse("state['m'] and state['v'] are the same memory");
}

struct Items {   // of any iterable: references of its own, so that nothing that runs meanwhile can drop them
    PyObject *all;
    explicit Items(PyObject *o) : all(PySequence_Tuple(o))
    {
        if (!all) throw Raised{};
    }
    ~Items() { Py_DECREF(all); }
    Items(const Items &) = delete;
    int64_t size() const { return PyTuple_GET_SIZE(all); }
    PyObject *operator[](int64_t i) const { return PyTuple_GET_ITEM(all, i); }
};

PyObject *adamw_step(PyObject *, PyObject *const *arg, Py_ssize_t)
{
    return guarded([&]() -> PyObject * {
        const Items params(arg[0]), grads(arg[1]), betas(arg[4]);
        const int64_t n = params.size();
        if (!n || n != grads.size()) refuse("params and grads must be lists of the same length, not empty");
        if (betas.size() != 2) refuse("betas must be two numbers");
        // numbers and state first: asking for them may run anybody's code, and no tensor changes any more once it has been looked at
        std::vector<float> decay(n);
        idm_adamw_cfg cfg = {};
        if (PyFloat_Check(arg[6]) || PyLong_Check(arg[6]) || (PyNumber_Check(arg[6]) && !PySequence_Check(arg[6]))) {
            std::fill(decay.begin(), decay.end(), (float)number(arg[6]));
        } else {
            const Items each(arg[6]);
            if (each.size() != n) refuse("weight_decay must be a number or one per tensor");
            for (int64_t i = 0; i < n; ++i) decay[i] = (float)number(each[i]);
        }
        cfg.lr = number(arg[3]);
        cfg.beta1 = number(betas[0]);
        cfg.beta2 = number(betas[1]);
        cfg.eps = number(arg[5]);
        bool fine = std::isfinite(cfg.lr) && cfg.lr >= 0 && std::isfinite(cfg.eps) && cfg.eps >= 0 && cfg.beta1 >= 0 && cfg.beta1 < 1 &&
                    cfg.beta2 >= 0 && cfg.beta2 < 1;
        for (const float d : decay) fine = fine && d >= 0 && std::isfinite(d);
        if (!fine) refuse("lr, eps and weight_decay must be finite and not negative, betas in [0, 1)");
        const State s = state_of(arg[2]);
        std::vector<at::Tensor> keep;              // dense copies of gradients, until the launch
        std::vector<const at::Tensor *> changed;
        std::vector<void *> param_at(n);
        std::vector<const void *> grad_at(n);
        std::vector<int64_t> sizes(n);
        changed.reserve(n);
        int64_t total = 0;
        const at::Tensor *first = nullptr, *first_grad = nullptr;
        for (int64_t i = 0; i < n; ++i) {
            if (!THPVariable_Check(params[i])) refuse("params must be a list of tensors");
            const at::Tensor &p = THPVariable_Unpack(params[i]);
            if (!first) {
                first = &p;
                cfg.param_dtype = dtype_of(p);
                if (cfg.param_dtype < 0) refuse("parameters and gradients must be float32, bfloat16 or float16");
            }
            if (p.scalar_type() != first->scalar_type() || p.device() != first->device() || p.layout() != at::kStrided || !p.is_contiguous() ||
                p.is_neg())
                refuse("parameters must be dense, of one type and on one device");
            sizes[i] = p.numel();
            total += (sizes[i] + BLOCK - 1) / BLOCK * BLOCK;
            if (grads[i] == Py_None) continue;
            if (!THPVariable_Check(grads[i])) refuse("grads must be a list of tensors, None where there is no gradient");
            const at::Tensor &g = THPVariable_Unpack(grads[i]);
            if (!first_grad) {
                first_grad = &g;
                cfg.grad_dtype = dtype_of(g);
                if (cfg.grad_dtype < 0) refuse("parameters and gradients must be float32, bfloat16 or float16");
            }
            if (g.scalar_type() != first_grad->scalar_type()) refuse("all gradients must be of one type");
            if (g.sizes() != p.sizes() || g.device() != p.device() || g.layout() != at::kStrided)
                refuse("a gradient must have its parameter's shape and device, and be dense");
            changed.push_back(&p);
        }
        if (!first_grad) cfg.grad_dtype = cfg.param_dtype;
        const c10::Device dev = first->device();
        check_state(s, total, &dev);
        cfg.moment_bits = s.eight ? 8 : 32;
        if (!dev.is_cuda()) refuse("parameters must be CUDA tensors");
        const c10::DeviceGuard guard(dev);
        for (int64_t i = 0; i < n; ++i) {
            const bool has = grads[i] != Py_None;
            param_at[i] = has ? THPVariable_Unpack(params[i]).mutable_data_ptr() : nullptr;
            if (!has) continue;
            const at::Tensor &g = THPVariable_Unpack(grads[i]);
            if (g.is_contiguous() && !g.is_neg()) {
                grad_at[i] = g.const_data_ptr();
            } else {
                keep.push_back(plain(g).contiguous());
                grad_at[i] = keep.back().const_data_ptr();
            }
        }
        const at::Tensor scratch = at::empty({2}, first->options().dtype(at::kLong));
        check(lib.adamw_step(dev.index(), &cfg, n, param_at.data(), grad_at.data(), sizes.data(), decay.data(), s.at(M), s.at(V),
                             (int16_t *)s.at(M_BASE), (int16_t *)s.at(V_BASE), s.t[M].numel(), (int64_t *)s.at(STEP), scratch.mutable_data_ptr(),
                             stream_of(*first)));
        // the kernel writes behind autograd's back: a backward pass that saved a parameter has to see that it changed
        for (const at::Tensor *p : changed)
            if (!p->is_inference()) p->unsafeGetTensorImpl()->bump_version();
        Py_RETURN_NONE;
    });
}

PyObject *adamw_moments(PyObject *, PyObject *dict)
{
    return guarded([&]() -> PyObject * {
        const State s = state_of(dict);
        check_state(s, -1, nullptr);
        if (!s.eight) return Py_BuildValue("(NN)", THPVariable_Wrap(s.t[M]), THPVariable_Wrap(s.t[V]));
        if (!s.t[M].is_cuda()) refuse("the state must be on a CUDA device");
        const c10::DeviceGuard guard(s.t[M].device());
        const int64_t n = s.t[M].numel();
        const at::Tensor m = at::empty({n}, s.t[M].options().dtype(at::kFloat)), v = at::empty({n}, m.options());
        check(lib.adamw_moments(s.t[M].get_device(), (const uint8_t *)read(s.t[M]), (const uint8_t *)read(s.t[V]), (const int16_t *)read(s.t[M_BASE]),
                                (const int16_t *)read(s.t[V_BASE]), (float *)write(m), (float *)write(v), n, stream_of(m)));
        return Py_BuildValue("(NN)", THPVariable_Wrap(m), THPVariable_Wrap(v));
    });
}

// bind(addresses of the five entry points, check, stream)
PyObject *bind(PyObject *, PyObject *args)
{
    unsigned long long at[5];
    PyObject *check_, *stream_;
    if (!PyArg_ParseTuple(args, "(KKKKK)OO", &at[0], &at[1], &at[2], &at[3], &at[4], &check_, &stream_)) return nullptr;
    lib.norm_workspace = (decltype(lib.norm_workspace))at[0];
    lib.norm_forward = (decltype(lib.norm_forward))at[1];
    lib.norm_backward = (decltype(lib.norm_backward))at[2];
    lib.adamw_step = (decltype(lib.adamw_step))at[3];
    lib.adamw_moments = (decltype(lib.adamw_moments))at[4];
    Py_INCREF(check_);
    Py_INCREF(stream_);
    Py_XSETREF(lib.check, check_);
    Py_XSETREF(lib.stream, stream_);
    for (int k = 0; k < 5; ++k)
        if (!lib.keys[k] && !(lib.keys[k] = PyUnicode_InternFromString(kKeys[k]))) return nullptr;
    Py_RETURN_NONE;
}

// A fixed number of positional arguments: the callers in norm.py and optim.py give the defaults
template <PyObject *(*F)(PyObject *, PyObject *const *, Py_ssize_t), Py_ssize_t N> PyObject *with(PyObject *self, PyObject *const *arg, Py_ssize_t n)
{
    if (n == N) return F(self, arg, n);
    PyErr_Format(PyExc_TypeError, "%zd arguments expected", N);
    return nullptr;
}

PyMethodDef methods[] = {
    {"bind", bind, METH_VARARGS, nullptr},
    {"group_norm_forward", (PyCFunction)(void *)with<group_norm_forward, 7>, METH_FASTCALL, nullptr},
    {"group_norm_backward", (PyCFunction)(void *)with<group_norm_backward, 9>, METH_FASTCALL, nullptr},
    {"adds_elsewhere", (PyCFunction)(void *)adds_elsewhere, METH_FASTCALL, nullptr},
    {"layout", layout_py, METH_O, nullptr},
    {"adamw_step", (PyCFunction)(void *)with<adamw_step, 7>, METH_FASTCALL, nullptr},
    {"adamw_moments", adamw_moments, METH_O, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module_ = {PyModuleDef_HEAD_INIT, "isingdiff._host", "Host side of the training operators", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host() { return PyModule_Create(&module_); }
