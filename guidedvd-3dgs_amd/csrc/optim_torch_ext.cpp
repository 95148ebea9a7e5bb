// optim_torch_ext.cpp -- the host half of FusedAdamW.step() over the C-ABI (include/gvd_optim.h): the walk over parameter groups, the checks of every tensor,
// the count of steps and the table of a launch, in one call.  No kernel lives here.  A step of four small tensors takes 6 to 7 us on the host this way, by the machine
// (0.4 of them for arrays that overlap), against 36 with all of it in Python and 8.2 with the walk alone there.
//
// Plain C++ (g++); the entry points are resolved from the library path that Python hands to init(), so A/B builds share one instance.
#include <torch/extension.h>
#include <torch/csrc/autograd/python_variable.h>

#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <dlfcn.h>

#include <algorithm>
#include <cmath>

#include "../../include/gvd_optim.h"

namespace {

struct Api {
    decltype(&gvd_adamw_step) step = nullptr;
    decltype(&gvd_adamw_scalars) scalars = nullptr;
    decltype(&gvd_adamw_key) key = nullptr;
    decltype(&gvd_optim_last_error) last_error = nullptr;
} g_api;

void init(const std::string& path)
{
    void* h = dlopen(path.c_str(), RTLD_NOW | RTLD_LOCAL);
    TORCH_CHECK(h != nullptr, "cannot load ", path, ": ", dlerror());
    auto sym = [&](const char* name) {
        void* p = dlsym(h, name);
        TORCH_CHECK(p != nullptr, path, " does not export ", name);
        return p;
    };
    g_api.step = reinterpret_cast<decltype(g_api.step)>(sym("gvd_adamw_step"));
    g_api.scalars = reinterpret_cast<decltype(g_api.scalars)>(sym("gvd_adamw_scalars"));
    g_api.key = reinterpret_cast<decltype(g_api.key)>(sym("gvd_adamw_key"));
    g_api.last_error = reinterpret_cast<decltype(g_api.last_error)>(sym("gvd_optim_last_error"));
}

void check(int rc) { TORCH_CHECK(rc == 0, "gvd_optim error ", rc, ": ", g_api.last_error()); }

// Whether two tensors of one shape lie in the same memory order.  The stride of a dimension of size 1 moves nothing, and there are several spellings of it.
bool same_order(const at::Tensor& a, const at::Tensor& b)
{
    if (a.numel() <= 1) return true;
    for (int64_t d = 0; d < a.dim(); d++)
        if (a.size(d) != 1 && a.stride(d) != b.stride(d)) return false;
    return true;
}

// A state tensor of parameter p: its type, shape, device and memory order.
void check_state(const at::Tensor& p, const at::Tensor& t, at::ScalarType type, const char* name, int64_t bits)
{
    TORCH_CHECK(t.scalar_type() == type && t.sizes() == p.sizes() && t.device() == p.device() && t.layout() == at::kStrided && same_order(p, t),
                "FusedAdamW: the state '", name, "' does not fit its parameter ", p.sizes(), " (state_bits=", bits, "): it takes ", type,
                " in the parameter's shape, device and memory order; got ", t.scalar_type(), " ", t.sizes(), " with strides ", t.strides(), " on ", t.device());
}

void check_scale(const at::Tensor& p, const at::Tensor& t, const char* name)
{
    TORCH_CHECK(t.scalar_type() == at::kFloat && t.dim() == 1 && t.size(0) == (p.numel() + GVD_ADAMW_BLOCK - 1) / GVD_ADAMW_BLOCK && t.device() == p.device() &&
                    t.is_contiguous(),
                "FusedAdamW: the state '", name, "' does not fit its parameter ", p.sizes());
}

typedef std::pair<const char*, const char*> Span;   // bytes that a dense tensor fills, the end excluded
Span span(const at::Tensor& t) { return {(const char*)t.data_ptr(), (const char*)t.data_ptr() + t.nbytes()}; }

// The tensors that go into one launch: all of one type and device, under one rule.
struct Launch {
    at::Device device = at::kCPU;
    at::ScalarType type = at::kFloat;
    double beta1 = 0, beta2 = 0, eps = 0;
    int64_t bits = 32, seed = 0;
    bool capturable = false;
    std::vector<at::Tensor> flat;   // for every tensor param, grad, step, first moment, second moment, and with 8 bits their scales
    std::vector<double> lr, weight_decay;
    std::vector<at::Tensor> lr_at;  // the device tensor that holds lr; undefined: the number in lr
    std::vector<int64_t> place;     // among all parameters of the optimizer
    // made by check():
    std::vector<gvd_adamw_tensor> table;
    std::vector<at::Tensor> grads;  // (keeps copies made here alive)

    size_t per() const { return bits == 8 ? 7 : 5; }
    bool takes(const Launch& x) const
    {
        return device == x.device && type == x.type && beta1 == x.beta1 && beta2 == x.beta2 && eps == x.eps && bits == x.bits && seed == x.seed && capturable == x.capturable;
    }
    int param_type() const { return type == at::kFloat ? 0 : type == at::kHalf ? 1 : type == at::kBFloat16 ? 2 : -1; }
    void* stream() const { return (void*)c10::hip::getCurrentHIPStream(device.index()).stream(); }

    void check_all()
    {
        const size_t n = place.size(), k = per();
        TORCH_CHECK_TYPE(param_type() >= 0, "FusedAdamW: parameters are float32, float16 or bfloat16, not ", type);
        // (groups are dicts that a program may change between steps)
        TORCH_CHECK_VALUE(bits == 8 || bits == 32, "FusedAdamW: state_bits must be 8 or 32, not ", bits);
        TORCH_CHECK_VALUE(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0, "FusedAdamW: invalid betas (", beta1, ", ", beta2, ")");
        TORCH_CHECK_VALUE(eps >= 0.0 && std::isfinite(eps), "FusedAdamW: invalid eps ", eps);
        const at::ScalarType moment = bits == 8 ? at::kFloat8_e4m3fn : at::kFloat;
        if (!capturable) {
            hipStreamCaptureStatus capture = hipStreamCaptureStatusNone;
            TORCH_CHECK(hipStreamIsCapturing((hipStream_t)stream(), &capture) == hipSuccess, "FusedAdamW: the stream cannot be asked whether it is capturing");
            TORCH_CHECK(capture == hipStreamCaptureStatusNone, "FusedAdamW: step() in a graph capture needs capturable=True (the count of steps would be frozen)");
        }
        table.resize(n);
        grads.resize(n);
        std::vector<Span> written;
        written.reserve(n * (k - 2));
        for (size_t i = 0; i < n; i++) {
            const at::Tensor &p = flat[i * k], &g = flat[i * k + 1], &step = flat[i * k + 2], &m = flat[i * k + 3], &v = flat[i * k + 4];
            TORCH_CHECK(g.layout() == at::kStrided, "FusedAdamW: sparse gradients are not supported");
            TORCH_CHECK(g.scalar_type() == type && g.device() == device && g.sizes() == p.sizes(), "FusedAdamW: a gradient of ", g.scalar_type(), " ", g.sizes(), " on ",
                        g.device(), " for a parameter of ", type, " ", p.sizes(), " on ", device);
            TORCH_CHECK(p.is_non_overlapping_and_dense(), "FusedAdamW: parameters must be dense (no gaps, no element twice)");
            check_state(p, m, moment, "exp_avg", bits);
            check_state(p, v, moment, bits == 8 ? "exp_avg_rms" : "exp_avg_sq", bits);
            TORCH_CHECK(step.scalar_type() == at::kFloat && step.numel() == 1 && (capturable ? step.device() == device : step.is_cpu()),
                        "FusedAdamW: the state 'step' is one float32 on ", capturable ? "the parameter's device (capturable=True)" : "the CPU");
            gvd_adamw_tensor& t = table[i];
            t = {};
            if (bits == 8) {
                check_scale(p, flat[i * k + 5], "exp_avg_scale");
                check_scale(p, flat[i * k + 6], "exp_avg_rms_scale");
                t.exp_avg_scale = flat[i * k + 5].data_ptr<float>();
                t.exp_avg_sq_scale = flat[i * k + 6].data_ptr<float>();
            }
            written.push_back(span(p));
            for (size_t j = 3; j < k; j++) written.push_back(span(flat[i * k + j]));
            grads[i] = same_order(p, g) ? g : at::empty_like(p).copy_(g);
            t.param = p.data_ptr();
            t.grad = grads[i].data_ptr();
            t.exp_avg = m.data_ptr();
            t.exp_avg_sq = v.data_ptr();
            t.n = p.numel();
            TORCH_CHECK_VALUE(t.n <= GVD_ADAMW_MOST, "FusedAdamW: a parameter of ", t.n, " elements (at most ", GVD_ADAMW_MOST, ")");
            if (lr_at[i].defined()) {
                TORCH_CHECK(lr_at[i].device() == device, "FusedAdamW: lr is on another device than its parameters");
                TORCH_CHECK_VALUE(lr_at[i].scalar_type() == at::kFloat && lr_at[i].numel() == 1, "FusedAdamW: a tensor lr is one float32 on the parameters' device, not ",
                                  lr_at[i].scalar_type(), " ", lr_at[i].sizes());
            }
        }
        // What the launch writes is read by no other tensor's workgroups, which run in any order.
        written.erase(std::remove_if(written.begin(), written.end(), [](const Span& x) { return x.first == x.second; }), written.end());
        std::sort(written.begin(), written.end());
        for (size_t i = 1; i < written.size(); i++)
            TORCH_CHECK(written[i].first >= written[i - 1].second, "FusedAdamW: two parameters share memory, or their states do");
        for (size_t i = 0; i < n; i++) {
            const Span g = span(grads[i]);
            if (g.first == g.second || g == span(flat[i * k])) continue;   // (a gradient that is the parameter itself: each element is read before it is written)
            const auto next = std::lower_bound(written.begin(), written.end(), Span(g.second, nullptr));   // the first that begins at or behind the gradient's end
            TORCH_CHECK(next == written.begin() || std::prev(next)->second <= g.first, "FusedAdamW: a gradient shares memory with a parameter or a state that the step writes");
        }
    }

    void run()
    {
        const size_t n = place.size(), k = per();
        at::Tensor scalars;
        if (capturable) {
            scalars = at::empty({(int64_t)(4 * n)}, flat[0].options().dtype(at::kFloat));
            std::vector<float*> steps(n);
            std::vector<const float*> lrs(n, nullptr);
            std::vector<unsigned> ids(n);
            for (size_t i = 0; i < n; i++) {
                steps[i] = flat[i * k + 2].data_ptr<float>();
                if (lr_at[i].defined()) lrs[i] = lr_at[i].data_ptr<float>();
                ids[i] = (unsigned)place[i];
            }
            check(g_api.scalars(steps.data(), lrs.data(), lr.data(), weight_decay.data(), ids.data(), (int)n, beta1, beta2, (unsigned)seed, scalars.data_ptr(), stream()));
        } else {
            for (size_t i = 0; i < n; i++) {
                const float t = *flat[i * k + 2].data_ptr<float>() + 1.f;
                table[i].step_size = (float)(lr[i] / (1.0 - std::pow(beta1, (double)t)));
                table[i].root_factor = (float)(1.0 / std::sqrt(1.0 - std::pow(beta2, (double)t)));
                table[i].keep = (float)(1.0 - lr[i] * weight_decay[i]);
                if (bits == 8) table[i].key = g_api.key((unsigned)seed, (unsigned)place[i], (unsigned)t);
            }
        }
        check(g_api.step(table.data(), (int)n, param_type(), (int)bits, beta1, beta2, eps, capturable ? scalars.data_ptr() : nullptr, stream()));
        if (!capturable)
            for (size_t i = 0; i < n; i++) ++*flat[i * k + 2].data_ptr<float>();   // (counted once the launch stands)
        // all were written behind autograd's back: graphs that saved them, and images that were packed from them, go by their version
        for (size_t i = 0; i < flat.size(); i++)
            if (i % k != 1 && !flat[i].is_inference()) flat[i].unsafeGetTensorImpl()->bump_version();
    }
};

struct Names {   // interned once
    PyObject *params, *betas, *eps, *lr, *weight_decay, *state_bits, *capturable, *seed, *step, *moments32[2], *moments8[4];
    Names()
    {
        auto s = [](const char* x) { return PyUnicode_InternFromString(x); };
        params = s("params"); betas = s("betas"); eps = s("eps"); lr = s("lr"); weight_decay = s("weight_decay"); state_bits = s("state_bits");
        capturable = s("capturable"); seed = s("seed"); step = s("step");
        moments32[0] = s("exp_avg"); moments32[1] = s("exp_avg_sq");
        moments8[0] = s("exp_avg"); moments8[1] = s("exp_avg_rms"); moments8[2] = s("exp_avg_scale"); moments8[3] = s("exp_avg_rms_scale");
    }
};

PyObject* item(PyObject* dict, PyObject* key)   // borrowed; null where it is missing
{
    PyObject* x = PyDict_GetItemWithError(dict, key);
    if (!x && PyErr_Occurred()) throw py::error_already_set();
    return x;
}

PyObject* entry(PyObject* group, PyObject* key)
{
    PyObject* x = item(group, key);
    if (!x) throw py::key_error(PyUnicode_AsUTF8(key));
    return x;
}

double number(PyObject* x)
{
    const double v = PyFloat_AsDouble(x);
    if (v == -1.0 && PyErr_Occurred()) throw py::error_already_set();
    return v;
}

// One step of every parameter that has a gradient.  Everything of every launch is checked before anything is counted or launched.
void step(const py::object& optimizer, const py::list& groups, const py::dict& state)
{
    static const Names N;
    at::NoGradGuard no_grad;
    std::vector<Launch> launches;
    int64_t place = -1;
    for (py::handle group_ : groups) {
        PyObject* g = group_.ptr();
        TORCH_CHECK(PyDict_Check(g), "FusedAdamW: a parameter group is a dict");
        Launch rule;
        const py::object betas = py::reinterpret_steal<py::object>(PySequence_Tuple(entry(g, N.betas)));
        if (!betas) throw py::error_already_set();
        TORCH_CHECK(PyTuple_GET_SIZE(betas.ptr()) == 2, "FusedAdamW: betas are two numbers");
        rule.beta1 = number(PyTuple_GET_ITEM(betas.ptr(), 0));
        rule.beta2 = number(PyTuple_GET_ITEM(betas.ptr(), 1));
        rule.eps = number(entry(g, N.eps));
        rule.bits = (int64_t)number(entry(g, N.state_bits));
        rule.capturable = PyObject_IsTrue(entry(g, N.capturable)) == 1;
        if (rule.bits == 8) rule.seed = (int64_t)number(entry(g, N.seed));
        const double decay = number(entry(g, N.weight_decay));
        PyObject* lr_ = entry(g, N.lr);
        const at::Tensor lr_at = THPVariable_Check(lr_) ? THPVariable_Unpack(lr_) : at::Tensor();
        TORCH_CHECK(!lr_at.defined() || rule.capturable, "FusedAdamW: lr may be a tensor with capturable=True only (reading it would wait for the device)");
        const double lr = lr_at.defined() ? 0.0 : number(lr_);
        PyObject* params = entry(g, N.params);
        TORCH_CHECK(PyList_Check(params), "FusedAdamW: a group's parameters are a list");
        Launch* at = nullptr;
        for (Py_ssize_t i = 0; i < PyList_GET_SIZE(params); i++) {
            place++;
            PyObject* p_ = PyList_GET_ITEM(params, i);
            TORCH_CHECK_TYPE(THPVariable_Check(p_), "FusedAdamW: a parameter is a tensor");
            const at::Tensor& p = THPVariable_Unpack(p_);
            const at::Tensor& grad = p.grad();
            if (!grad.defined()) continue;
            TORCH_CHECK(p.is_cuda(), "FusedAdamW: parameter on ", p.device(), "; there is no CPU path");
            py::object st = py::reinterpret_borrow<py::object>(item(state.ptr(), p_));
            if (!st || PyObject_Size(st.ptr()) == 0) {
                st = optimizer.attr("_new_state")(py::handle(p_), group_);
                state[py::handle(p_)] = st;
            }
            TORCH_CHECK(PyDict_Check(st.ptr()), "FusedAdamW: the state of a parameter is a dict");
            if (!at || at->device != p.device() || at->type != p.scalar_type()) {
                rule.device = p.device();
                rule.type = p.scalar_type();
                at = nullptr;
                for (Launch& x : launches)
                    if (x.takes(rule)) at = &x;
                if (!at) { launches.push_back(rule); at = &launches.back(); }
            }
            at->flat.push_back(p);
            at->flat.push_back(grad);
            auto held = [&](PyObject* name) {
                PyObject* t = item(st.ptr(), name);
                TORCH_CHECK(t != nullptr, "FusedAdamW: the state '", PyUnicode_AsUTF8(name), "' of a parameter is missing: it does not fit state_bits=", rule.bits);
                TORCH_CHECK(THPVariable_Check(t), "FusedAdamW: the state '", PyUnicode_AsUTF8(name), "' of a parameter is no tensor");
                at->flat.push_back(THPVariable_Unpack(t));
            };
            held(N.step);
            if (rule.bits == 8) for (PyObject* name : N.moments8) held(name);
            else for (PyObject* name : N.moments32) held(name);
            at->lr.push_back(lr);
            at->lr_at.push_back(lr_at);
            at->weight_decay.push_back(decay);
            at->place.push_back(place);
        }
    }
    for (Launch& x : launches) {
        c10::DeviceGuard guard(x.device);
        x.check_all();
    }
    for (Launch& x : launches) {
        c10::DeviceGuard guard(x.device);
        x.run();
    }
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m)
{
    m.doc() = "FusedAdamW's step over libgvd_optim.so (see csrc/optim_torch_ext.cpp)";
    m.def("init", &init, "resolve the C-ABI entry points from the given library path");
    m.def("step", &step, "one step of every parameter that has a gradient");
}
