// optim_torch_ext.cpp -- the host half of FusedAdamW.step() over the C-ABI (include/gvd_optim.h): the checks of every tensor, the count of steps and the
// table of a launch, in one call for all tensors of a type.  No kernel lives here.  With Python doing this the step of a few small tensors took 9 us a
// tensor on the host (88 us for ten tensors whose kernel runs 26 us); here it is below 1 us a tensor.
//
// Plain C++ (g++); the entry points are resolved from the library path that Python hands to init(), so A/B builds share one instance.
#include <torch/extension.h>

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

bool same_order(const at::Tensor& a, const at::Tensor& b) { return a.numel() <= 1 || a.strides() == b.strides(); }

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

// `flat`: for every tensor param, grad, step, first moment, second moment, and with 8 bits their scales.  All parameters have one type and device.
// lr_at: empty, or the device tensors that hold lr (none: the number in lr).
void adamw_step(const std::vector<at::Tensor>& flat, const std::vector<double>& lr, const std::vector<c10::optional<at::Tensor>>& lr_at, const std::vector<double>& weight_decay,
                const std::vector<int64_t>& place, double beta1, double beta2, double eps, int64_t bits, bool capturable, int64_t seed)
{
    const size_t n = place.size(), per = bits == 8 ? 7 : 5;
    TORCH_CHECK(n > 0 && flat.size() == n * per && lr.size() == n && weight_decay.size() == n, "adamw_step: lists of different lengths");
    const at::Device device = flat[0].device();
    TORCH_CHECK(device.is_cuda(), "FusedAdamW: parameter on ", device, "; this build has no CPU path");
    const at::ScalarType type = flat[0].scalar_type();
    const int param_type = type == at::kFloat ? 0 : type == at::kHalf ? 1 : type == at::kBFloat16 ? 2 : -1;
    TORCH_CHECK_TYPE(param_type >= 0, "FusedAdamW: parameters are float32, float16 or bfloat16, not ", type);
    const at::ScalarType moment = bits == 8 ? at::kFloat8_e4m3fn : at::kFloat;
    c10::DeviceGuard guard(device);

    std::vector<gvd_adamw_tensor> table(n);
    std::vector<at::Tensor> grads(n);   // (keeps copies made here alive)
    std::vector<std::pair<const char*, const char*>> spans(n);
    for (size_t i = 0; i < n; i++) {    // everything is checked before anything is counted or launched
        const at::Tensor &p = flat[i * per], &g = flat[i * per + 1], &step = flat[i * per + 2], &m = flat[i * per + 3], &v = flat[i * per + 4];
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
            check_scale(p, flat[i * per + 5], "exp_avg_scale");
            check_scale(p, flat[i * per + 6], "exp_avg_rms_scale");
            t.exp_avg_scale = flat[i * per + 5].data_ptr<float>();
            t.exp_avg_sq_scale = flat[i * per + 6].data_ptr<float>();
        }
        spans[i] = {(const char*)p.data_ptr(), (const char*)p.data_ptr() + p.nbytes()};
        grads[i] = same_order(p, g) ? g : at::empty_like(p).copy_(g);
        t.param = p.data_ptr();
        t.grad = grads[i].data_ptr();
        t.exp_avg = m.data_ptr();
        t.exp_avg_sq = v.data_ptr();
        t.n = p.numel();
        if (!lr_at.empty() && lr_at[i]) TORCH_CHECK(lr_at[i]->device() == device, "FusedAdamW: lr is on another device than its parameters");
    }
    std::sort(spans.begin(), spans.end());
    for (size_t i = 1; i < n; i++)
        TORCH_CHECK(spans[i].first >= spans[i - 1].second || spans[i - 1].first == spans[i - 1].second, "FusedAdamW: two parameters share memory");
    void* stream = (void*)c10::hip::getCurrentHIPStream(device.index()).stream();
    at::Tensor scalars;
    if (capturable) {
        scalars = at::empty({(int64_t)(4 * n)}, flat[0].options().dtype(at::kFloat));
        std::vector<float*> steps(n);
        std::vector<const float*> lrs(n, nullptr);
        std::vector<unsigned> ids(n);
        for (size_t i = 0; i < n; i++) {
            steps[i] = flat[i * per + 2].data_ptr<float>();
            if (!lr_at.empty() && lr_at[i]) lrs[i] = lr_at[i]->data_ptr<float>();
            ids[i] = (unsigned)place[i];
        }
        check(g_api.scalars(steps.data(), lrs.data(), lr.data(), weight_decay.data(), ids.data(), (int)n, beta1, beta2, (unsigned)seed, scalars.data_ptr(), stream));
    } else {
        for (size_t i = 0; i < n; i++) {
            const float t = ++*flat[i * per + 2].data_ptr<float>();
            table[i].step_size = (float)(lr[i] / (1.0 - std::pow(beta1, (double)t)));
            table[i].root_factor = (float)(1.0 / std::sqrt(1.0 - std::pow(beta2, (double)t)));
            table[i].keep = (float)(1.0 - lr[i] * weight_decay[i]);
            if (bits == 8) table[i].key = g_api.key((unsigned)seed, (unsigned)place[i], (unsigned)t);
        }
    }
    check(g_api.step(table.data(), (int)n, param_type, (int)bits, beta1, beta2, eps, capturable ? scalars.data_ptr() : nullptr, stream));
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m)
{
    m.doc() = "FusedAdamW's step over libgvd_optim.so (see csrc/optim_torch_ext.cpp)";
    m.def("init", &init, "resolve the C-ABI entry points from the given library path");
    m.def("adamw_step", &adamw_step, "one step of all tensors of a type on a device");
}
