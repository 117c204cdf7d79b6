// Host side of the residual-stream operators in native code: the checks, allocations, launches and autograd nodes of ordinary calls of
// residual.py.  A call that is not ordinary - a tensor subclass, a functorch transform, tracing, whatever a check refuses - returns
// None and takes the Python route there, which is the definition and says what is wrong.  The launches are the C-ABI library's.
//
// Nothing is kept from one call for the next.  Nodes save their tensors as torch's own do (versions checked, hooks called) and need no Python.
#include <torch/extension.h>
#include <torch/version.h>

#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>

#include "../../include/spiky_b200.h"
#include "call_checks.h"

namespace {

using at::Tensor;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

struct Library {
    decltype(&lutb_dropout) dropout;
    decltype(&lutb_dropout_advance) dropout_advance;
    decltype(&lutb_join_forward) join_forward;
    decltype(&lutb_join_backward) join_backward;
    decltype(&lutb_join_backward_workspace) join_backward_workspace;
};
Library lib;
PyObject *tensor_class, *parameter_class, *check_status;

void check(int status) {
    if (status == 0) return;
    pybind11::gil_scoped_acquire gil;
    Ref r(PyObject_CallFunction(check_status, "i", status));   // raises what the Python route raises
    raise_current();
}

// ------------------------------------------------------------------------------------------------ arguments
int type_of(at::ScalarType t) {
    return t == at::kFloat ? LUTB_F32 : t == at::kBFloat16 ? LUTB_BF16 : t == at::kHalf ? LUTB_F16 : -1;
}
// An ordinary tensor of a type the kernels know on the device, or none where that is allowed; false for all else.
bool take_tensor(PyObject *o, c10::DeviceIndex device, bool optional, Tensor &out) {
    if (o == Py_None) return optional;
    if ((PyObject *)Py_TYPE(o) != tensor_class && (PyObject *)Py_TYPE(o) != parameter_class) return false;
    out = THPVariable_Unpack(o);
    if (type_of(out.scalar_type()) < 0) return false;
    if (device < 0) {
        if (!out.is_cuda()) return false;
        device = out.device().index();
    }
    return plain_cuda(out, out.scalar_type(), device) && !out._fw_grad(0).defined();
}
bool take_float(PyObject *o, double &v) {
    if (!PyFloat_Check(o) && !(PyLong_Check(o) && !PyBool_Check(o))) return false;
    v = PyFloat_AsDouble(o);
    return !(v == -1.0 && PyErr_Occurred()) && std::isfinite(v);
}
bool take_int(PyObject *o, int64_t &v) {
    if (!PyLong_Check(o) || PyBool_Check(o)) return false;
    v = PyLong_AsLongLong(o);
    return !(v == -1 && PyErr_Occurred());
}
bool take_norm(PyObject *o, int32_t &v) {
    if (o == Py_None) {
        v = LUTB_NORM_NONE;
    } else if (PyUnicode_Check(o)) {
        v = PyUnicode_CompareWithASCIIString(o, "rms") == 0 ? LUTB_NORM_RMS : PyUnicode_CompareWithASCIIString(o, "layer") == 0 ? LUTB_NORM_LAYER : -1;
    } else {
        v = -1;
    }
    return v >= 0;
}
bool take_state(PyObject *o, c10::DeviceIndex device, Tensor &out) {
    if ((PyObject *)Py_TYPE(o) != tensor_class) return false;
    out = THPVariable_Unpack(o);
    if (!out.is_cuda()) return false;
    return plain_cuda(out, at::kLong, device < 0 ? out.device().index() : device) && out.dim() == 1 && out.size(0) == 2 && out.is_contiguous();
}

void *pointer(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
const int64_t *random_of(const Tensor &t) { return t.defined() ? static_cast<const int64_t *>(t.data_ptr()) : nullptr; }
Tensor whole(const Tensor &t) { return t.defined() ? t.contiguous() : t; }
void *stream_on(c10::DeviceIndex device) { return c10::cuda::getCurrentCUDAStream(device).stream(); }
Tensor new_like(const Tensor &t, at::ScalarType type) { return at::empty(t.sizes(), at::TensorOptions().dtype(type).device(t.device())); }
bool needs_graph(std::initializer_list<const Tensor *> list) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor *t : list)
        if (t->defined() && t->requires_grad()) return true;
    return false;
}

struct ResidualNode : public torch::autograd::Node {
    std::vector<SavedVariable> saved;
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        for (auto &s : saved) s.reset_data();
    }
    std::vector<Tensor> unpack() {
        std::vector<Tensor> s;
        std::lock_guard<std::mutex> lock(mutex_);
        s.reserve(saved.size());
        for (auto &v : saved) s.push_back(v.unpack());
        return s;
    }
};

// What a backward pass is handed can come from hooks: the kernels get nothing that is not what the forward pass had.
void expect(const Tensor &t, at::ScalarType type, int64_t numel, c10::DeviceIndex device, const char *name) {
    TORCH_CHECK(plain_cuda(t, type, device) && t.numel() == numel, name, " is not what the forward pass saved: ", numel, " elements of ", type, " on cuda:", (int)device);
    TORCH_CHECK(!t._fw_grad(0).defined(), name, " has a tangent: residual operators have no forward-mode derivatives");
}
// As residual.py's _refuse_recording.
void refuse_recording() {
    TORCH_CHECK(!torch::jit::tracer::isTracing() && !c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value(),
                "residual operators cannot be traced: their kernels would be missing from what is recorded");
}
// A gradient as the kernels read it: no lazy negation, no stand-in for zeros.
Tensor settled(const Tensor &t) {
    if (!t.defined()) return t;
    if (t._is_zerotensor()) return at::zeros(t.sizes(), at::TensorOptions().dtype(t.scalar_type()).device(t.device()));
    return t.is_neg() ? t.resolve_neg() : t;
}
at::ScalarType scalar_type_of(int type) { return type == LUTB_F32 ? at::kFloat : type == LUTB_BF16 ? at::kBFloat16 : at::kHalf; }

// ------------------------------------------------------------------------------------------------ dropout
Tensor dropout(const Tensor &x, double p, const Tensor &state, int64_t site);

struct DropoutNode : public ResidualNode {
    double p = 0.0;
    int64_t site = 0;
    std::string name() const override { return "_CounterDropoutBackward"; }
    variable_list apply(variable_list &&grads) override {
        const std::vector<Tensor> s = unpack();
        if (!grads[0].defined() || !task_should_compute_output(0)) return variable_list(1);
        refuse_recording();
        const Tensor dy = settled(grads[0]);
        expect(dy, dy.scalar_type(), dy.numel(), dy.device().index(), "the gradient");
        expect(s[0], at::kLong, 2, dy.device().index(), "state");
        TORCH_CHECK(type_of(dy.scalar_type()) >= 0 && s[0].is_contiguous(), "the gradient or state is not what the forward pass had");
        return {dropout(dy, p, s[0], site)};   // (with a graph of its own where one is asked for)
    }
};

Tensor dropout(const Tensor &x, double p, const Tensor &state, int64_t site) {
    const bool graph = needs_graph({&x});
    Tensor y;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        c10::cuda::CUDAGuard guard(x.device());
        const Tensor xc = x.contiguous();
        y = new_like(x, x.scalar_type());
        check(lib.dropout(type_of(x.scalar_type()), x.numel(), p, random_of(state), site, pointer(xc), pointer(y), stream_on(x.device().index())));
    }
    if (graph) {
        auto node = std::shared_ptr<DropoutNode>(new DropoutNode(), torch::autograd::deleteNode);
        node->p = p;
        node->site = site;
        node->set_next_edges(torch::autograd::collect_next_edges(x));
        node->saved.emplace_back(state, false);
        torch::autograd::set_history(y, node);
    }
    return y;
}

// dropout(x, p, state, site)
PyObject *dropout_entry(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK_TYPE(n == 4, "dropout(x, p, state, site)");
    Tensor x, state;
    double p;
    int64_t site;
    if (!take_tensor(args[0], -1, false, x) || !take_float(args[1], p) || !take_int(args[3], site) || !(p > 0.0 && p <= 1.0) || site < 0 ||
        !take_state(args[2], x.device().index(), state) || !ordinary_context() || (needs_graph({&x}) && (x.is_inference() || state.is_inference()))) {
        PyErr_Clear();
        Py_RETURN_NONE;
    }
    return THPVariable_Wrap(dropout(x, p, state, site));
    END_HANDLE_TH_ERRORS
}

// take(state, count)
PyObject *take_entry(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK_TYPE(n == 2, "take(state, count)");
    Tensor state;
    int64_t count;
    if (!take_state(args[0], -1, state) || !take_int(args[1], count) || count < 0 || !ordinary_context() || state.is_inference() ||
        (at::GradMode::is_enabled() && state.requires_grad())) {
        PyErr_Clear();
        Py_RETURN_NONE;
    }
    Tensor used;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        c10::cuda::CUDAGuard guard(state.device());
        used = new_like(state, at::kLong);
        check(lib.dropout_advance(static_cast<int64_t *>(state.data_ptr()), count, static_cast<int64_t *>(used.data_ptr()), stream_on(state.device().index())));
    }
    state.unsafeGetTensorImpl()->bump_version();
    return THPVariable_Wrap(used);
    END_HANDLE_TH_ERRORS
}

// ------------------------------------------------------------------------------------------------ joins
enum { X, F, GATE, AW, AB, BW, BB, TENSORS };

struct JoinNode : public ResidualNode {
    lutb_join_cfg cfg;
    bool has_h = false, had[TENSORS] = {}, kept[TENSORS] = {};   // what the call had, what of it the backward pass reads
    c10::DeviceIndex device = 0;
    std::vector<int64_t> shape, gate_shape;
    std::string name() const override { return "_ResidualJoinBackward"; }
    // Which tensors gradient k depends on, as residual.py's _sources; a bit each.
    uint32_t sources(int k, bool next) const {
        if (next) return k == BB ? 0 : (1u << BB) - 1;
        const bool normed = cfg.after != LUTB_NORM_NONE;
        switch (k) {
            case F: return 1u << GATE | (normed ? 1u << F | 1u << AW : 0);
            case GATE: return 1u << F | (normed ? 1u << AW | 1u << AB : 0);
            case AW: return 1u << F | 1u << GATE;
            case AB: return 1u << GATE;
            default: return 0;
        }
    }
    variable_list apply(variable_list &&grads) override {
        std::vector<Tensor> s = unpack();   // the seven tensors, state, stats
        const Tensor dh = has_h ? settled(grads[0]) : Tensor(), dy = cfg.before != LUTB_NORM_NONE ? settled(grads[has_h ? 1 : 0]) : Tensor();
        variable_list out(TENSORS);
        if (!dh.defined() && !dy.defined()) return out;
        refuse_recording();
        const std::vector<Tensor> given = at::GradMode::is_enabled() ? s : std::vector<Tensor>();   // (with the graph behind them)
        const int64_t all = cfg.rows * cfg.width;
        const int types[TENSORS] = {cfg.stream_type, cfg.branch_type, cfg.gate_type, cfg.param_type, cfg.param_type, cfg.param_type, cfg.param_type};
        static const char *const what[TENSORS] = {"x", "branch", "gate", "branch_weight", "branch_bias", "next_weight", "next_bias"};
        for (int k = 0; k < TENSORS; k++)
            if (kept[k]) expect(s[k], scalar_type_of(types[k]), k <= F ? all : k == GATE ? all / cfg.gate_rows : cfg.width, device, what[k]);
        if (cfg.dropout > 0.0) {
            expect(s[TENSORS], at::kLong, 2, device, "state");
            s[TENSORS] = s[TENSORS].contiguous();
        }
        if (cfg.after != LUTB_NORM_NONE || cfg.before != LUTB_NORM_NONE) {
            expect(s[TENSORS + 1], at::kFloat, 4 * cfg.rows, device, "stats");
            s[TENSORS + 1] = s[TENSORS + 1].contiguous();
        }
        if (dh.defined()) expect(dh, scalar_type_of(cfg.stream_type), all, device, "the gradient");
        if (dy.defined()) expect(dy, scalar_type_of(cfg.branch_type), all, device, "the gradient");
        {
            at::AutoDispatchBelowADInplaceOrView below;
            c10::cuda::CUDAGuard guard(device);
            for (int k = 0; k < TENSORS; k++)
                if (had[k] && task_should_compute_output(k) && (k < BW || dy.defined()))
                    out[k] = at::empty(k <= F ? at::IntArrayRef(shape) : k == GATE ? at::IntArrayRef(gate_shape) : at::IntArrayRef(cfg.width),
                                       at::TensorOptions().dtype(scalar_type_of(types[k])).device(at::kCUDA, device));
            for (int k = 0; k < BB; k++) s[k] = whole(s[k]);
            const Tensor dhc = whole(dh), dyc = whole(dy);
            Tensor ws;
            size_t need = 0;
            if (out[AW].defined() || out[AB].defined() || out[BW].defined() || out[BB].defined() || (out[GATE].defined() && cfg.gate_rows > 1)) {
                need = lib.join_backward_workspace(&cfg);
                ws = at::empty({(int64_t)need}, at::TensorOptions().dtype(at::kByte).device(at::kCUDA, device));
            }
            check(lib.join_backward(&cfg, pointer(s[X]), pointer(s[F]), pointer(s[GATE]), pointer(s[AW]), pointer(s[AB]), pointer(s[BW]),
                                    random_of(s[TENSORS]), static_cast<const float *>(pointer(s[TENSORS + 1])), pointer(dhc), pointer(dyc), pointer(out[X]),
                                    pointer(out[F]), pointer(out[GATE]), pointer(out[AW]), pointer(out[AB]), pointer(out[BW]), pointer(out[BB]),
                                    pointer(ws), need, stream_on(device)));
        }
        for (int k = 0; k < TENSORS && !given.empty(); k++) {   // a graph is asked for: one that says so when it is used
            if (!out[k].defined()) continue;
            std::vector<Tensor> of;
            for (const Tensor *t : {&dh, &dy})
                if (t->defined() && t->requires_grad()) of.push_back(*t);
            for (int i = 0; i < BB; i++)
                if ((sources(k, dy.defined()) >> i & 1) && given[i].defined() && given[i].requires_grad()) of.push_back(given[i]);
            if (of.empty()) continue;
            auto error = std::shared_ptr<torch::autograd::Error>(
                new torch::autograd::Error("a residual join is differentiable once", torch::autograd::collect_next_edges(at::ArrayRef<Tensor>(of))), torch::autograd::deleteNode);
            torch::autograd::set_history(out[k], error);
        }
        return out;
    }
};

// gate_rows of a gate for x, as residual.py's _gate_rows; 0: not one of those shapes
int64_t gate_rows_of(const Tensor &gate, const Tensor &x) {
    const int64_t d = x.dim(), lead = d - gate.dim();
    if (gate.dim() == 0 || lead < 0 || gate.size(-1) != x.size(-1)) return 0;
    auto mine = [&](int64_t k) { return k < lead ? 1 : gate.size(k - lead); };
    int64_t k = d - 1, rows = 1;
    while (k > 0 && mine(k - 1) == 1) rows *= x.size(--k);
    for (int64_t j = 0; j < k; j++)
        if (mine(j) != x.size(j)) return 0;
    return rows;
}

// join(x, branch, dtype of the branch's type or None, after, aw, ab, gate, skip_scale, branch_scale, p, state, site, before, bw, bb, eps) -> (h, y)
PyObject *join_entry(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK_TYPE(n == 16, "join takes 16 arguments");
    Tensor t[TENSORS], state;
    lutb_join_cfg cfg{};
    double skip, branch, p, eps;
    auto arguments = [&]() {
        if (!ordinary_context() || !take_tensor(args[0], -1, false, t[X])) return false;
        const Tensor &x = t[X];
        const c10::DeviceIndex device = x.device().index();
        if (x.dim() == 0 || x.numel() == 0) return false;
        if (!take_tensor(args[1], device, true, t[F]) || (t[F].defined() && t[F].sizes() != x.sizes())) return false;
        at::ScalarType type = t[F].defined() ? t[F].scalar_type() : x.scalar_type();
        if (args[2] != Py_None) {
            if (!THPDtype_Check(args[2]) || t[F].defined()) return false;
            type = reinterpret_cast<THPDtype *>(args[2])->scalar_type;
        }
        const int own = type_of(x.scalar_type()), of_branch = type_of(type);
        if (of_branch < 0 || (own != of_branch && own != LUTB_F32)) return false;
        cfg.stream_type = own;
        cfg.branch_type = of_branch;
        cfg.width = x.size(-1);
        cfg.rows = x.numel() / cfg.width;
        if (!take_norm(args[3], cfg.after) || !take_norm(args[12], cfg.before)) return false;
        const int at[4] = {4, 5, 13, 14}, which[4] = {AW, AB, BW, BB};
        cfg.param_type = -1;
        for (int k = 0; k < 4; k++) {
            Tensor &v = t[which[k]];
            if (!take_tensor(args[at[k]], device, true, v)) return false;
            if (!v.defined()) continue;
            const int type_v = type_of(v.scalar_type());
            if (v.dim() != 1 || v.size(0) != cfg.width || (type_v != LUTB_F32 && type_v != of_branch)) return false;
            if ((k < 2 ? cfg.after : cfg.before) == LUTB_NORM_NONE || (cfg.param_type >= 0 && cfg.param_type != type_v)) return false;
            cfg.param_type = type_v;
        }
        if (cfg.param_type < 0) cfg.param_type = LUTB_F32;
        if (!take_tensor(args[6], device, true, t[GATE])) return false;
        cfg.gate_type = LUTB_F32;
        if (t[GATE].defined()) {
            cfg.gate_type = type_of(t[GATE].scalar_type());
            if (!t[F].defined() || (cfg.gate_type != LUTB_F32 && cfg.gate_type != of_branch)) return false;
            cfg.gate_rows = gate_rows_of(t[GATE], x);
            if (cfg.gate_rows == 0) return false;   // (or one element, which the Python route spreads)
        }
        if (!take_float(args[7], skip) || !take_float(args[8], branch) || !take_float(args[9], p) || !take_int(args[11], cfg.site) || !take_float(args[15], eps))
            return false;
        cfg.skip_scale = (float)skip;
        cfg.branch_scale = (float)branch;
        cfg.eps = (float)eps;
        cfg.dropout = p;
        if (!std::isfinite(cfg.skip_scale) || !std::isfinite(cfg.branch_scale) || !std::isfinite(cfg.eps) || !(cfg.eps > 0.0f)) return false;
        if (!(p >= 0.0 && p <= 1.0) || cfg.site < 0 || (p > 0.0 && !take_state(args[10], device, state))) return false;
        return t[F].defined() || (cfg.before != LUTB_NORM_NONE && cfg.after == LUTB_NORM_NONE && p == 0.0);
    };
    if (!arguments()) {
        PyErr_Clear();
        Py_RETURN_NONE;
    }
    const bool graph = needs_graph({&t[X], &t[F], &t[GATE], &t[AW], &t[AB], &t[BW], &t[BB]});
    if (graph) {
        for (const Tensor &v : t)
            if (v.defined() && v.is_inference()) Py_RETURN_NONE;
        if (state.defined() && state.is_inference()) Py_RETURN_NONE;
    }
    Tensor h, y, stats;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        const Tensor &x = t[X];
        c10::cuda::CUDAGuard guard(x.device());
        Tensor c[TENSORS];
        for (int k = 0; k < TENSORS; k++) c[k] = whole(t[k]);
        if (t[F].defined()) h = new_like(x, x.scalar_type());
        if (cfg.before != LUTB_NORM_NONE)
            y = new_like(x, scalar_type_of(cfg.branch_type));
        if (graph && (cfg.after != LUTB_NORM_NONE || cfg.before != LUTB_NORM_NONE))
            stats = at::empty({cfg.rows, 4}, at::TensorOptions().dtype(at::kFloat).device(x.device()));
        check(lib.join_forward(&cfg, pointer(c[X]), pointer(c[F]), pointer(c[GATE]), pointer(c[AW]), pointer(c[AB]), pointer(c[BW]), pointer(c[BB]),
                               random_of(state), pointer(h), pointer(y), static_cast<float *>(pointer(stats)), stream_on(x.device().index())));
    }
    if (graph) {
        auto node = std::shared_ptr<JoinNode>(new JoinNode(), torch::autograd::deleteNode);
        node->cfg = cfg;
        node->has_h = h.defined();
        node->device = t[X].device().index();
        node->shape = t[X].sizes().vec();
        if (t[GATE].defined()) node->gate_shape = t[GATE].sizes().vec();
        const bool norms = cfg.after != LUTB_NORM_NONE || cfg.before != LUTB_NORM_NONE;
        for (int k = 0; k < TENSORS; k++) {
            node->had[k] = t[k].defined();
            node->kept[k] = t[k].defined() && (k == X ? cfg.before != LUTB_NORM_NONE : k == F ? norms || (t[GATE].defined() && t[GATE].requires_grad()) : k != BB);
        }
        node->set_next_edges(torch::autograd::collect_next_edges(t[X], t[F], t[GATE], t[AW], t[AB], t[BW], t[BB]));
        for (int k = 0; k < TENSORS; k++) node->saved.emplace_back(node->kept[k] ? t[k] : Tensor(), false);
        node->saved.emplace_back(state, false);
        node->saved.emplace_back(stats, false);
        variable_list outputs;
        if (h.defined()) outputs.push_back(h);
        if (y.defined()) outputs.push_back(y);
        torch::autograd::set_history(outputs, node);
    }
    Ref result(PyTuple_New(2));
    if (!result) return nullptr;
    PyTuple_SET_ITEM(result.get(), 0, h.defined() ? THPVariable_Wrap(h) : Py_NewRef(Py_None));
    PyTuple_SET_ITEM(result.get(), 1, y.defined() ? THPVariable_Wrap(y) : Py_NewRef(Py_None));
    return Py_NewRef(result.get());
    END_HANDLE_TH_ERRORS
}

void setup(pybind11::dict addresses, pybind11::object check_fn) {
    auto take = [&](const char *name, auto &fn) { fn = reinterpret_cast<std::decay_t<decltype(fn)>>(addresses[name].cast<uintptr_t>()); };
    take("lutb_dropout", lib.dropout);
    take("lutb_dropout_advance", lib.dropout_advance);
    take("lutb_join_forward", lib.join_forward);
    take("lutb_join_backward", lib.join_backward);
    take("lutb_join_backward_workspace", lib.join_backward_workspace);
    auto keep = [](pybind11::object o) { return o.release().ptr(); };   // for the life of the process
    check_status = keep(check_fn);
    tensor_class = keep(pybind11::module_::import("torch").attr("Tensor"));
    parameter_class = keep(pybind11::module_::import("torch.nn").attr("Parameter"));
}

PyMethodDef methods[] = {{"join", (PyCFunction)(void (*)(void))join_entry, METH_FASTCALL, "(h, y) of a join, or None"},
                         {"dropout", (PyCFunction)(void (*)(void))dropout_entry, METH_FASTCALL, "dropout of x, or None"},
                         {"take", (PyCFunction)(void (*)(void))take_entry, METH_FASTCALL, "a copy of a dropout state that moves on, or None"},
                         {nullptr, nullptr, 0, nullptr}};

}  // namespace

PYBIND11_MODULE(_residual_calls, m) {
    m.def("setup", &setup);
    m.attr("torch_version") = TORCH_VERSION;
    PyModule_AddFunctions(m.ptr(), methods);
}
