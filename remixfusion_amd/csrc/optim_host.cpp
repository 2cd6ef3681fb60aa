// optim_host.cpp -- the host's share of an optimizer step as a CPython module (no device code; librfx's entry points come in as
// addresses).  A step over a dozen small tensors runs 4 us on the GPU; gathering a dozen gradients, checking that everything is
// where it was and writing the descriptors costs 1 us per tensor in Python and some 30 ns here.
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>
#include <ATen/ATen.h>
#include <optional>
#include <vector>
#include "../../include/rfx.h"

namespace py = pybind11;

namespace {

struct {
    decltype(&rfx_adamw_step) adamw_step;
    decltype(&rfx_adamw_workspace_bytes) adamw_workspace_bytes;
    decltype(&rfx_adamw_moments) adamw_moments;
    decltype(&rfx_grad_norm_workspace_bytes) grad_norm_workspace_bytes;
    decltype(&rfx_grad_clip) grad_clip;
} rfx;

void bind(const py::dict& at) {
    const auto get = [&](const char* name, auto& fn) { fn = reinterpret_cast<std::decay_t<decltype(fn)>>(at[name].cast<uintptr_t>()); };
    get("rfx_adamw_step", rfx.adamw_step);
    get("rfx_adamw_workspace_bytes", rfx.adamw_workspace_bytes);
    get("rfx_adamw_moments", rfx.adamw_moments);
    get("rfx_grad_norm_workspace_bytes", rfx.grad_norm_workspace_bytes);
    get("rfx_grad_clip", rfx.grad_clip);
}

int type_of(at::ScalarType t) {
    return t == at::kFloat ? RFX_F32 : t == at::kBFloat16 ? RFX_BF16 : t == at::kHalf ? RFX_F16 : -1;
}

const at::Tensor& tensor(PyObject* o) {
    if (!THPVariable_Check(o)) throw py::type_error("a tensor is expected");
    return THPVariable_Unpack(o);
}

// borrowed; an error if the key is missing
PyObject* item(PyObject* dict, PyObject* key) {
    PyObject* v = PyDict_GetItemWithError(dict, key);
    if (!v) {
        if (PyErr_Occurred()) throw py::error_already_set();
        throw py::key_error(PyUnicode_AsUTF8(key));
    }
    return v;
}

double number(PyObject* o) {
    const double x = PyFloat_AsDouble(o);
    if (x == -1.0 && PyErr_Occurred()) throw py::error_already_set();
    return x;
}

struct Keys {
    PyObject *params, *lr, *betas, *eps, *weight_decay, *seed, *state_bits, *maximize, *master_weights, *capturable, *step, *exp_avg,
        *exp_avg_sq, *exponents, *master, *amsgrad, *differentiable, *decoupled;
    Keys() {
        const auto make = [](const char* s) { return PyUnicode_InternFromString(s); };
        params = make("params"); lr = make("lr"); betas = make("betas"); eps = make("eps"); weight_decay = make("weight_decay");
        seed = make("seed"); state_bits = make("state_bits"); maximize = make("maximize"); master_weights = make("master_weights");
        capturable = make("capturable"); step = make("step"); exp_avg = make("exp_avg"); exp_avg_sq = make("exp_avg_sq");
        exponents = make("exponents"); master = make("master"); amsgrad = make("amsgrad"); differentiable = make("differentiable");
        decoupled = make("decoupled_weight_decay");
    }
};
const Keys& keys() { static const Keys* k = new Keys; return *k; }

// autograd notices a tensor that is written behind its back only by its version
void written(const at::Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// fp32 tensor of these sizes and strides in `flat`'s memory, without the dispatcher's round that as_strided() makes
py::object part_of(const at::Tensor& flat, int64_t at, at::IntArrayRef sizes, at::IntArrayRef strides) {
    auto impl = c10::make_intrusive<c10::TensorImpl>(c10::Storage(flat.storage()), flat.key_set(), flat.dtype());
    impl->set_storage_offset(at);
    impl->set_sizes_and_strides(sizes, strides);
    return py::reinterpret_steal<py::object>(THPVariable_Wrap(at::Tensor(std::move(impl))));
}

// a call's workspace behind the 16 bytes whose first hold the norm that it returns
struct Workspace {
    at::Tensor memory;
    size_t bytes;
    Workspace(size_t n, at::Device device)
        : memory(at::empty({4 + (int64_t)(n + 3) / 4}, at::TensorOptions().dtype(at::kFloat).device(device))), bytes(n) {}
    float* norm() const { return static_cast<float*>(memory.data_ptr()); }
    void* rest() const { return norm() + 4; }
    py::object norm_tensor() const { return part_of(memory, 0, {}, {}); }
};

// what a step's outcome is to the caller: a negative status of librfx, or one of these
enum Outcome { DONE = 0, STALE = 1, OTHER_ORDER = 2 };

struct Memory {                         // where a tensor was
    void* ptr;
    at::ScalarType dtype;
    std::vector<int64_t> sizes, strides;
    explicit Memory(const at::Tensor& t) : ptr(t.data_ptr()), dtype(t.scalar_type()), sizes(t.sizes().vec()), strides(t.strides().vec()) {}
    bool like(const at::Tensor& t) const {
        return t.layout() == at::kStrided && t.scalar_type() == dtype && t.sizes() == at::IntArrayRef(sizes) && t.strides() == at::IntArrayRef(strides);
    }
};

// What the descriptors of a step hold that stays the same from step to step: the parameters that have a gradient, on one device, and
// their state.  Every step checks it against the optimizer's own lists; where anything moved, the caller builds another.
class Plan {
    // A tensor of a state as it was, without keeping it alive: its impl's address is taken by no other while this weak reference lasts
    struct Part {
        c10::weak_intrusive_ptr<c10::TensorImpl> impl;
        void* ptr;
        int64_t n;
        at::ScalarType dtype;
        static void* at(const at::Tensor& t) { return t.has_storage() ? t.data_ptr() : nullptr; }
        explicit Part(const at::Tensor& t) : impl(t.getIntrusivePtr()), ptr(at(t)), n(t.numel()), dtype(t.scalar_type()) {}
        bool is(const at::Tensor& t) const {
            return t.unsafeGetTensorImpl() == impl._unsafe_get_target() && at(t) == ptr && t.numel() == n && t.scalar_type() == dtype;
        }
    };

    std::vector<py::object> params_;
    std::vector<std::pair<PyObject*, PyObject*>> entries_;      // the optimizer's states: addresses only, that keep nothing alive
    std::vector<PyObject*> states_;                             // the planned parameters' among them: looked into once all are found where they were
    std::vector<Part> parts_;                           // (a user may keep something of their own in a state: only tensors count)
    std::vector<Memory> where_;
    std::vector<int> group_of_;
    std::vector<float*> counts_;        // host step counts; null: on the device
    std::vector<rfx_adamw_tensor> rows_;
    std::vector<rfx_grad_tensor> grads_;
    std::vector<rfx_adamw_group> groups_;
    struct Settings { long state_bits; bool master, capturable; double seed; bool refused; };      // refused: the caller's check says why
    std::vector<Settings> settings_;    // per parameter group
    at::Device device_;
    bool ordered_ = true, counted_ = false, host_counted_ = false;

    static bool set(PyObject* g, PyObject* key, bool otherwise) {
        PyObject* v = PyDict_GetItemWithError(g, key);
        const int on = v ? PyObject_IsTrue(v) : otherwise;
        if (on < 0 || (!v && PyErr_Occurred())) throw py::error_already_set();
        return on == 1;
    }

    static Settings settings_of(PyObject* g) {
        const Keys& k = keys();
        return {(long)number(item(g, k.state_bits)), PyObject_IsTrue(item(g, k.master_weights)) == 1, PyObject_IsTrue(item(g, k.capturable)) == 1,
                number(item(g, k.seed)), set(g, k.amsgrad, false) || set(g, k.differentiable, false) || !set(g, k.decoupled, true)};
    }

public:
    // entries: (parameter, place in the optimizer, parameter group), states as the step needs them (types, memory order, devices)
    Plan(const py::list& entries, const py::list& param_groups, const py::dict& state) : device_(at::kCPU) {
        const Keys& k = keys();
        for (const auto& g : param_groups) settings_.push_back(settings_of(g.ptr()));
        for (const auto& e : entries) {
            const py::tuple t = py::cast<py::tuple>(e);
            const at::Tensor& p = tensor(t[0].ptr());
            const int index = t[1].cast<int>(), group = t[2].cast<int>();
            const Settings& s = settings_.at(group);
            PyObject* st = item(state.ptr(), t[0].ptr());
            const at::Tensor &m = tensor(item(st, k.exp_avg)), &v = tensor(item(st, k.exp_avg_sq)), &step = tensor(item(st, k.step));
            device_ = p.device();
            params_.push_back(py::reinterpret_borrow<py::object>(t[0]));
            states_.push_back(st);
            where_.emplace_back(p);
            group_of_.push_back(group);
            ordered_ &= p.strides() == m.strides();
            PyObject *key, *value;
            for (Py_ssize_t at = 0; PyDict_Next(st, &at, &key, &value);)
                if (THPVariable_Check(value)) parts_.emplace_back(THPVariable_Unpack(value));
            rfx_adamw_tensor r{};
            r.param = p.data_ptr();
            r.exp_avg = m.data_ptr();
            r.exp_avg_sq = v.data_ptr();
            if (s.state_bits == 8) r.exponents = static_cast<int8_t*>(tensor(item(st, k.exponents)).data_ptr());
            if (s.master && p.scalar_type() != at::kFloat) r.master = static_cast<float*>(tensor(item(st, k.master)).data_ptr());
            TORCH_CHECK(step.scalar_type() == at::kFloat && step.numel() == 1 && step.device() == (s.capturable ? device_ : at::Device(at::kCPU)),
                        "a step count of another type or place");
            if (s.capturable) r.step_dev = static_cast<float*>(step.data_ptr());
            counts_.push_back(s.capturable ? nullptr : static_cast<float*>(step.data_ptr()));
            (s.capturable ? counted_ : host_counted_) = true;
            r.n = p.numel();
            r.index = (uint32_t)index;
            r.dtype = type_of(p.scalar_type());
            rows_.push_back(r);
            rfx_grad_tensor gr{};
            gr.n = r.n;
            gr.dtype = r.dtype;
            grads_.push_back(gr);
        }
        PyObject *key, *value;
        for (Py_ssize_t at = 0; PyDict_Next(state.ptr(), &at, &key, &value);) entries_.emplace_back(key, value);
    }

    bool host_counted() const { return host_counted_; }

    // the whole step where everything is as planned; else nothing has happened yet
    py::object step(const py::list& param_groups, const py::dict& state, double limit, uintptr_t stream) {
        const Keys& k = keys();
        if (param_groups.size() != settings_.size() || (size_t)PyDict_Size(state.ptr()) != entries_.size())
            return py::int_((int)STALE);
        size_t n = 0, at_value = 0, at_part = 0;
        bool other = !ordered_;
        for (size_t gi = 0; gi < settings_.size(); ++gi) {
            PyObject* g = PyList_GET_ITEM(param_groups.ptr(), (Py_ssize_t)gi);
            const Settings s = settings_of(g);
            if (s.state_bits != settings_[gi].state_bits || s.master != settings_[gi].master || s.capturable != settings_[gi].capturable
                || s.seed != settings_[gi].seed || s.refused)
                return py::int_((int)STALE);
            PyObject* list = item(g, k.params);
            if (!PyList_Check(list)) return py::int_((int)STALE);
            for (Py_ssize_t i = 0; i < PyList_GET_SIZE(list); ++i) {
                PyObject* o = PyList_GET_ITEM(list, i);
                const at::Tensor& p = tensor(o);
                const at::Tensor& grad = p.grad();
                if (!grad.defined()) continue;
                if (n == params_.size() || params_[n].ptr() != o || group_of_[n] != (int)gi) return py::int_((int)STALE);
                if (!where_[n].like(p) || p.data_ptr() != where_[n].ptr) return py::int_((int)STALE);
                other |= !where_[n].like(grad) || grad.device() != device_;
                if (!other) rows_[n].grad = grad.data_ptr();
                ++n;
            }
        }
        if (n != params_.size()) return py::int_((int)STALE);
        PyObject *key, *value;
        for (Py_ssize_t at = 0; PyDict_Next(state.ptr(), &at, &key, &value); ++at_value)
            if (entries_[at_value].first != key || entries_[at_value].second != value) return py::int_((int)STALE);
        for (PyObject* st : states_) {
            if (!PyDict_Check(st)) return py::int_((int)STALE);
            for (Py_ssize_t at = 0; PyDict_Next(st, &at, &key, &value);)
                if (THPVariable_Check(value) && (at_part == parts_.size() || !parts_[at_part++].is(THPVariable_Unpack(value))))
                    return py::int_((int)STALE);
        }
        if (at_part != parts_.size()) return py::int_((int)STALE);
        if (other) return py::int_((int)OTHER_ORDER);
        return run(rows_, param_groups, limit, stream);
    }

    // the step with gradients (and parameters) that the caller brought to the memory order of the moments
    py::object launch(const py::list& params, const py::list& grads, const py::list& param_groups, double limit, uintptr_t stream) {
        std::vector<rfx_adamw_tensor> rows = rows_;
        if (params.size() != rows.size() || grads.size() != rows.size()) throw py::value_error("a parameter and a gradient for each of the plan's");
        for (size_t i = 0; i < rows.size(); ++i) {
            const at::Tensor &p = tensor(params[i].ptr()), &g = tensor(grads[i].ptr());
            if (p.numel() != rows[i].n || g.numel() != rows[i].n || type_of(p.scalar_type()) != rows[i].dtype || type_of(g.scalar_type()) != rows[i].dtype
                || p.device() != device_ || g.device() != device_)
                throw py::value_error("a parameter or gradient of another size, type or device than planned");
            rows[i].param = p.data_ptr();
            rows[i].grad = g.data_ptr();
        }
        return run(rows, param_groups, limit, stream);
    }

private:
    py::object run(std::vector<rfx_adamw_tensor>& rows, const py::list& param_groups, double limit, uintptr_t stream) {
        const Keys& k = keys();
        groups_.clear();
        const size_t n = rows.size();
        size_t first = 0;                                                  // of this parameter group's entries
        for (size_t i = 0; i < n; ++i) {
            const int gi = group_of_[i];
            const int64_t step = counts_[i] ? (int64_t)*counts_[i] + 1 : 1;
            if (i == 0 || group_of_[i - 1] != gi) {
                PyObject* g = PyList_GET_ITEM(param_groups.ptr(), gi);
                rfx_adamw_group e{};
                PyObject *lr = item(g, k.lr), *betas = item(g, k.betas);
                if (THPVariable_Check(lr)) {
                    const at::Tensor& t = THPVariable_Unpack(lr);
                    if (!settings_[gi].capturable || t.device() != device_ || t.scalar_type() != at::kFloat || t.numel() != 1)
                        throw py::value_error("a tensor lr needs capturable=True and has to be one float32 on the parameters' device");
                    e.lr_dev = static_cast<const float*>(t.data_ptr());
                } else {
                    e.lr = number(lr);
                }
                e.beta1 = number(py::object(py::reinterpret_borrow<py::object>(betas)[py::int_(0)]).ptr());
                e.beta2 = number(py::object(py::reinterpret_borrow<py::object>(betas)[py::int_(1)]).ptr());
                e.eps = number(item(g, k.eps));
                e.weight_decay = number(item(g, k.weight_decay));
                e.seed = (uint32_t)(int64_t)number(item(g, k.seed));
                e.state_bits = (int32_t)settings_[gi].state_bits;
                e.maximize = PyObject_IsTrue(item(g, k.maximize)) == 1;
                e.step = step;
                first = groups_.size();
                groups_.push_back(e);
            }
            size_t at = first;                                             // parameters that joined at different steps: an entry for each count
            while (at < groups_.size() && groups_[at].step != step) ++at;
            if (at == groups_.size()) {
                groups_.push_back(groups_[first]);
                groups_.back().step = step;
            }
            rows[i].group = (int32_t)at;
        }
        const bool clipped = limit >= 0.0;
        std::optional<Workspace> ws;
        if (clipped || counted_) ws.emplace(rfx.adamw_workspace_bytes((int)n), device_);
        if (clipped)
            for (size_t i = 0; i < n; ++i) grads_[i].grad = const_cast<void*>(rows[i].grad);
        const int rc = rfx.adamw_step(rows.data(), (int)n, groups_.data(), (int)groups_.size(), clipped ? grads_.data() : nullptr, limit,
                                      clipped ? ws->norm() : nullptr, ws ? ws->rest() : nullptr, ws ? ws->bytes : 0, (rfx_stream)stream);
        if (rc != RFX_OK) return py::int_(rc);
        for (size_t i = 0; i < n; ++i) {
            if (counts_[i]) *counts_[i] += 1.f;
            written(tensor(params_[i].ptr()));
        }
        return clipped ? ws->norm_tensor() : py::none();
    }
};

// norm and scaling of the gradients of `parameters`; OTHER_ORDER: something about them needs the caller's care
py::object clip(const py::list& parameters, int kind, double limit, int device, uintptr_t stream) {
    std::vector<rfx_grad_tensor> rows;
    rows.reserve(parameters.size());
    at::Device dev(at::kCPU);
    for (const auto& o : parameters) {
        const at::Tensor& g = tensor(o.ptr()).grad();
        if (!g.defined()) continue;
        rfx_grad_tensor r{};
        if (!g.is_cuda() || g.device().index() != device || g.layout() != at::kStrided || (r.dtype = type_of(g.scalar_type())) < 0
            || !g.is_non_overlapping_and_dense())
            return py::int_((int)OTHER_ORDER);
        dev = g.device();
        r.grad = g.data_ptr();
        r.n = g.numel();
        rows.push_back(r);
    }
    if (rows.empty()) return py::int_((int)OTHER_ORDER);
    const Workspace ws(rfx.grad_norm_workspace_bytes((int)rows.size()), dev);
    const int rc = rfx.grad_clip(rows.data(), (int)rows.size(), kind, limit, ws.norm(), ws.rest(), ws.bytes, (rfx_stream)stream);
    if (rc != RFX_OK) return py::int_(rc);
    for (const auto& o : parameters) {
        const at::Tensor& g = tensor(o.ptr()).grad();
        if (g.defined()) written(g);
    }
    return ws.norm_tensor();
}

// the moments of all parameters in fp32: the state's own tensors where they are held in 32 bits, the codes' values where in 8
// (of one device; OTHER_ORDER: of several), zeros where there is no state yet
py::object moments(const py::list& param_groups, const py::dict& state, int device, uintptr_t stream) {
    const Keys& k = keys();
    std::vector<rfx_moment_tensor> rows;
    std::vector<std::pair<size_t, at::Tensor>> codes;
    py::list avg, avg_sq;
    int64_t total = 0;
    for (const auto& g : param_groups) {
        for (const auto& p : py::reinterpret_borrow<py::list>(item(g.ptr(), k.params))) {
            PyObject* st = PyDict_GetItemWithError(state.ptr(), p.ptr());
            if (!st && PyErr_Occurred()) throw py::error_already_set();
            if (!st || PyDict_Size(st) == 0) {
                const at::Tensor like = tensor(p.ptr()).detach();
                for (py::list* to : {&avg, &avg_sq})
                    to->append(py::reinterpret_steal<py::object>(THPVariable_Wrap(at::zeros_like(like, like.options().dtype(at::kFloat)))));
                continue;
            }
            PyObject *om = item(st, k.exp_avg), *ov = item(st, k.exp_avg_sq);
            const at::Tensor &m = tensor(om), &v = tensor(ov);
            if (m.scalar_type() != at::kByte) {                            // (torch's own step on the CPU holds them in the parameter's type)
                const bool as_is = m.scalar_type() == at::kFloat && v.scalar_type() == at::kFloat;
                avg.append(as_is ? py::reinterpret_borrow<py::object>(om) : py::reinterpret_steal<py::object>(THPVariable_Wrap(m.to(at::kFloat))));
                avg_sq.append(as_is ? py::reinterpret_borrow<py::object>(ov) : py::reinterpret_steal<py::object>(THPVariable_Wrap(v.to(at::kFloat))));
                continue;
            }
            const at::Tensor& e = tensor(item(st, k.exponents));
            if (v.scalar_type() != at::kByte || e.scalar_type() != at::kChar || !m.is_cuda() || v.device() != m.device() || e.device() != m.device()
                || m.sizes() != v.sizes() || m.strides() != v.strides() || !m.is_non_overlapping_and_dense() || !e.is_contiguous()
                || e.numel() != 2 * ((m.numel() + RFX_ADAMW_BLOCK - 1) / RFX_ADAMW_BLOCK))
                throw py::value_error("this is not the state of 8-bit moments");
            if (m.device().index() != device) return py::int_((int)OTHER_ORDER);
            rfx_moment_tensor r{};
            r.exp_avg = static_cast<const uint8_t*>(m.data_ptr());
            r.exp_avg_sq = static_cast<const uint8_t*>(v.data_ptr());
            r.exponents = static_cast<const int8_t*>(e.data_ptr());
            r.n = m.numel();
            total += (r.n + 3) & ~(int64_t)3;                              // every output at a multiple of 16 bytes
            rows.push_back(r);
            codes.emplace_back(avg.size(), m);
            avg.append(py::none());
            avg_sq.append(py::none());
        }
    }
    if (!rows.empty()) {
        const at::Tensor flat = at::empty({2 * total}, at::TensorOptions().dtype(at::kFloat).device(codes[0].second.device()));
        float* base = static_cast<float*>(flat.data_ptr());
        int64_t at = 0;
        for (size_t i = 0; i < rows.size(); ++i) {
            rows[i].out_avg = base + at;
            rows[i].out_avg_sq = base + total + at;
            avg[codes[i].first] = part_of(flat, at, codes[i].second.sizes(), codes[i].second.strides());
            avg_sq[codes[i].first] = part_of(flat, total + at, codes[i].second.sizes(), codes[i].second.strides());
            at += (rows[i].n + 3) & ~(int64_t)3;
        }
        const int rc = rfx.adamw_moments(rows.data(), (int)rows.size(), (rfx_stream)stream);
        if (rc != RFX_OK) return py::int_(rc);
    }
    return py::make_tuple(avg, avg_sq);
}

}  // namespace

PYBIND11_MODULE(_optim_host, m) {
    m.def("bind", &bind);
    m.def("clip", &clip);
    m.def("moments", &moments);
    m.attr("STALE") = (int)STALE;
    m.attr("OTHER_ORDER") = (int)OTHER_ORDER;
    py::class_<Plan>(m, "Plan")
        .def(py::init<const py::list&, const py::list&, const py::dict&>())
        .def("step", &Plan::step)
        .def("launch", &Plan::launch)
        .def_property_readonly("host_counted", &Plan::host_counted);
}
