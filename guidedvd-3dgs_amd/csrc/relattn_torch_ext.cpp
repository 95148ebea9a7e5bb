// relattn_torch_ext.cpp -- relative_bias_attention as one node of the autograd graph over the C-ABI (include/gvd_relattn.h): checks of arguments, strides, outputs,
// workspaces, and the backward without Python.  No kernel lives here.  With a Python autograd function a training pass took 180 us of host time, as much
// as its kernels at the sizes of a temporal layer; here it takes 42 to 80 by the machine, of which autograd's engine takes 17 to 33 for any graph.
//
// Plain C++ (g++); the entry points are resolved from the library path that Python hands to init(), so A/B builds share one instance.
#include <torch/extension.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>

#include <ATen/hip/EmptyTensor.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/VirtualGuardImpl.h>
#include <c10/hip/HIPStream.h>
#include <dlfcn.h>

#include <algorithm>
#include <climits>
#include <unordered_set>

#include "../../include/gvd_relattn.h"

namespace {

struct Api {
    decltype(&gvd_relattn_fwd) fwd = nullptr;
    decltype(&gvd_relattn_bwd) bwd = nullptr;
    decltype(&gvd_relattn_fwd_workspace) fwd_workspace = nullptr;
    decltype(&gvd_relattn_bwd_workspace) bwd_workspace = nullptr;
    decltype(&gvd_relattn_last_error) last_error = nullptr;
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
    g_api.fwd = reinterpret_cast<decltype(g_api.fwd)>(sym("gvd_relattn_fwd"));
    g_api.bwd = reinterpret_cast<decltype(g_api.bwd)>(sym("gvd_relattn_bwd"));
    g_api.fwd_workspace = reinterpret_cast<decltype(g_api.fwd_workspace)>(sym("gvd_relattn_fwd_workspace"));
    g_api.bwd_workspace = reinterpret_cast<decltype(g_api.bwd_workspace)>(sym("gvd_relattn_bwd_workspace"));
    g_api.last_error = reinterpret_cast<decltype(g_api.last_error)>(sym("gvd_relattn_last_error"));
}

long long check(long long rc)
{
    TORCH_CHECK(rc >= 0, "gvd_relattn error ", rc, ": ", g_api.last_error());
    return rc;
}

struct Config {
    at::Tensor first, kv_lens;   // CPU int32: the least distance of each bucket of one side; device int32 or undefined
    int64_t heads, q_start;
    bool both, causal, frame_major;
    double scale;
    int batch_dim() const { return frame_major ? 1 : 0; }
    int row_dim() const { return frame_major ? 0 : 1; }
};

bool aligned(const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }

at::Tensor packed(const at::Tensor& t)   // contiguous and 16-byte aligned (a contiguous view may begin anywhere)
{
    at::Tensor c = t.contiguous();
    return aligned(c) ? c : c.clone();
}

bool in_place(const at::Tensor& t) { return t.stride(2) == 1 && t.stride(0) % 8 == 0 && t.stride(1) % 8 == 0 && aligned(t); }

// (batch, row) strides; a batch of one serves any batch, and the stride of a dimension of one row is never used
std::pair<long long, long long> strides(const at::Tensor& t, const Config& c)
{
    const int bd = c.batch_dim(), rd = c.row_dim();
    return {t.size(bd) == 1 ? 0 : t.stride(bd), t.size(rd) == 1 ? t.size(2) : t.stride(rd)};
}

gvd_relattn_problem problem(const at::Tensor& q, const at::Tensor& k, const at::Tensor& out, const at::Tensor& table, const at::Tensor& q_starts, const Config& c)
{
    gvd_relattn_problem p = {};
    auto whole = [](int64_t n) { return (int)std::min<int64_t>(n, INT_MAX); };   // (an expanded tensor may have any size: what an int does not hold is refused as too large)
    p.B = whole(q.size(c.batch_dim()));
    p.H = whole(c.heads);
    p.Nq = whole(q.size(c.row_dim()));
    p.Nk = whole(k.size(c.row_dim()));
    p.D = (int)(q.size(2) / c.heads);
    p.is_bf16 = q.scalar_type() == at::kBFloat16;
    p.table_type = table.scalar_type() == at::kFloat ? 0 : table.scalar_type() == at::kHalf ? 1 : 2;
    p.buckets = (int)table.size(0);
    p.both = c.both;
    p.causal = c.causal;
    p.first = c.first.data_ptr<int>();
    p.scale = (float)c.scale;
    p.q_start = (int)c.q_start;
    p.q_starts = q_starts.defined() ? q_starts.data_ptr<int>() : nullptr;
    p.kv_lens = c.kv_lens.defined() ? c.kv_lens.data_ptr<int>() : nullptr;
    std::tie(p.q_bs, p.q_rs) = strides(q, c);
    std::tie(p.kv_bs, p.kv_rs) = strides(k, c);
    std::tie(p.o_bs, p.o_rs) = strides(out, c);
    return p;
}

// Straight from the allocator: through the dispatcher each took some 2 us in the engine's thread (a training pass makes seven).
at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const at::Tensor& like) { return at::detail::empty_cuda(sizes, type, like.device(), c10::nullopt); }
at::Tensor fresh_like(const at::Tensor& t) { return fresh(t.sizes(), t.scalar_type(), t); }   // (contiguous)
at::Tensor bytes(long long n, const at::Tensor& like) { return n ? fresh({n}, at::kByte, like) : at::Tensor(); }
void* ptr(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
void* stream_of(const at::Tensor& t) { return (void*)c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

at::Tensor forward_(at::Tensor q, at::Tensor k, at::Tensor v, const at::Tensor& table, const at::Tensor& q_starts, const Config& c, at::Tensor* lse)
{
    const c10::DeviceGuard guard(q.device());
    const int bd = c.batch_dim(), rd = c.row_dim();
    at::Tensor out = fresh_like(q);
    if (lse) *lse = fresh({q.size(bd), c.heads, q.size(rd)}, at::kFloat, q);
    if (q.numel() == 0 || k.size(rd) == 0) return out.zero_();
    if (!in_place(q)) q = packed(q);
    if (!in_place(k)) k = packed(k);
    if (!in_place(v)) v = packed(v);
    if (strides(k, c) != strides(v, c)) {
        k = packed(k);
        v = packed(v);
    }
    const gvd_relattn_problem p = problem(q, k, out, table, q_starts, c);
    const at::Tensor ws = bytes(check(g_api.fwd_workspace(&p)), q);
    check(g_api.fwd(&p, q.data_ptr(), k.data_ptr(), v.data_ptr(), table.data_ptr(), out.data_ptr(), lse ? lse->data_ptr<float>() : nullptr, ptr(ws), stream_of(q)));
    return out;
}

struct RelativeBiasAttentionBackward : torch::autograd::Node {
    torch::autograd::SavedVariable q, k, v, table, out, kv_lens;
    at::Tensor lse;
    Config c;   // (kv_lens aside)

    std::string name() const override { return "RelativeBiasAttentionBackward"; }
    void release_variables() override
    {
        for (torch::autograd::SavedVariable* x : {&q, &k, &v, &table, &out, &kv_lens}) x->reset_data();
        lse.reset();
    }
    torch::autograd::variable_list apply(torch::autograd::variable_list&& grads) override
    {
        TORCH_CHECK(!at::GradMode::is_enabled(), "relative_bias_attention: its gradients have no gradients (create_graph=True)");
        if (!grads[0].defined()) return torch::autograd::variable_list(4);
        Config c_ = c;
        const at::Tensor q_ = q.unpack(), k_ = k.unpack(), v_ = v.unpack(), table_ = table.unpack(), out_ = out.unpack(shared_from_this());
        c_.kv_lens = kv_lens.unpack();
        const c10::DeviceGuard guard(q_.device());
        at::AutoDispatchBelowAutograd below;
        at::Tensor dq = fresh_like(q_), dk = fresh_like(k_), dv = fresh_like(v_), dtable = fresh_like(table_);
        if (q_.numel() == 0 || k_.numel() == 0) {
            for (at::Tensor* t : {&dq, &dk, &dv, &dtable}) t->zero_();
        } else {
            const at::Tensor g = packed(grads[0]);
            const gvd_relattn_problem p = problem(q_, k_, out_, table_, at::Tensor(), c_);
            const at::Tensor ws = bytes(check(g_api.bwd_workspace(&p)), q_);
            check(g_api.bwd(&p, q_.data_ptr(), k_.data_ptr(), v_.data_ptr(), table_.data_ptr(), out_.data_ptr(), g.data_ptr(), lse.data_ptr<float>(), dq.data_ptr(), dk.data_ptr(),
                            dv.data_ptr(), dtable.data_ptr(), ptr(ws), stream_of(q_)));
        }
        return {dq, dk, dv, dtable};
    }
};

// Whether a stream other than the current one takes part in a capture (it was joined to it before).  The default stream never does.
bool captured(const c10::Stream& s)
{
    if (s.id() == 0) return false;
    const c10::hip::HIPStream stream(c10::hip::HIPStream::UNCHECKED, c10::Stream(c10::Stream::UNSAFE, c10::Device(c10::DeviceType::HIP, s.device_index()), s.id()));
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    return hipStreamIsCapturing(stream.stream(), &status) == hipSuccess && status == hipStreamCaptureStatusActive;
}

// A node of the graph belongs to the stream that it was made on, and a leaf's accumulating node lives as long as some graph of the leaf does.  A backward pass that is
// captured while an eager graph of the same leaf lives would make that stream wait for a captured one, in the engine's thread, where the error ends the process: refused
// here, before.  The leaf may lie behind other nodes (a projection, a cast, a view, or the copies and views that this file makes of its arguments), so all that the
// inputs come from are looked at: in a capture only, where a call is made once.
void refuse_foreign_nodes(std::initializer_list<const at::Tensor*> inputs, const at::Device& device)
{
    hipStreamCaptureStatus capture = hipStreamCaptureStatusNone;
    TORCH_CHECK(hipStreamIsCapturing(c10::hip::getCurrentHIPStream(device.index()).stream(), &capture) == hipSuccess, "relative_bias_attention: the stream cannot be asked whether it is capturing");
    if (capture == hipStreamCaptureStatusNone) return;
    const c10::Stream now = c10::impl::VirtualGuardImpl(device.type()).getStream(device);
    auto look_at = [&](torch::autograd::Node* node) {
        const auto stream = node->stream();
        TORCH_CHECK(!stream || *stream == now || captured(*stream),
                    "relative_bias_attention: a training pass cannot be captured while an eager graph of the same leaf lives (drop its outputs first), nor on from an eager graph");
    };
    std::vector<torch::autograd::Node*> open;
    std::unordered_set<torch::autograd::Node*> met;
    for (const at::Tensor* t : inputs) {
        if (!t->requires_grad()) continue;
        if (!t->is_leaf()) open.push_back(t->grad_fn().get());
        else if (const auto accumulate = torch::autograd::impl::try_get_grad_accumulator(*t)) look_at(accumulate.get());
    }
    while (!open.empty()) {
        torch::autograd::Node* node = open.back();
        open.pop_back();
        if (!met.insert(node).second) continue;
        look_at(node);
        for (const torch::autograd::Edge& e : node->next_edges())
            if (e.function) open.push_back(e.function.get());
    }
}

at::Tensor differentiable(const at::Tensor& q_, const at::Tensor& k_, const at::Tensor& v_, const at::Tensor& table, const Config& c)
{
    const std::shared_ptr<RelativeBiasAttentionBackward> node(new RelativeBiasAttentionBackward(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(q_, k_, v_, table));
    at::Tensor out;
    {
        at::AutoDispatchBelowAutograd below;
        const at::Tensor q = packed(q_), k = packed(k_), v = packed(v_);
        out = forward_(q, k, v, table, at::Tensor(), c, &node->lse);
        node->q = torch::autograd::SavedVariable(q, false);
        node->k = torch::autograd::SavedVariable(k, false);
        node->v = torch::autograd::SavedVariable(v, false);
    }
    node->table = torch::autograd::SavedVariable(table, false);
    node->kv_lens = torch::autograd::SavedVariable(c.kv_lens, false);
    node->c = c;
    node->c.kv_lens.reset();
    torch::autograd::set_history(out, node);
    node->out = torch::autograd::SavedVariable(out, true);
    return out;
}

#define GVD_WANT(cond, ...) TORCH_CHECK_VALUE(cond, "relative_bias_attention: ", __VA_ARGS__)

// Nothing where the kernels do not cover the call (types, head dim) or a number is out of range: the caller looks closer.
c10::optional<at::Tensor> attend(const at::Tensor& q, at::Tensor k, at::Tensor v, const at::Tensor& table_, int64_t heads, const at::Tensor& first, bool both, bool causal,
                                 const py::object& start, const c10::optional<at::Tensor>& kv_lens_, const c10::optional<double>& scale_, bool frame_major)
{
    TORCH_CHECK(first.is_cpu() && first.scalar_type() == at::kInt && first.dim() == 1 && first.numel() > 0 && first.is_contiguous(),
                "relative_bias_attention: the buckets' first distances are read by the host, as a contiguous int32 row; got ", first.scalar_type(), " ", first.sizes(), " on ", first.device());
    at::Tensor q_starts;
    int64_t q_start = 0;
    if (THPVariable_Check(start.ptr())) q_starts = THPVariable_Unpack(start.ptr());
    else q_start = start.cast<int64_t>();
    const at::Tensor kv_lens = kv_lens_.value_or(at::Tensor());
    const double scale = scale_.value_or(0.125);
    if (!q.is_cuda() || (q.scalar_type() != at::kHalf && q.scalar_type() != at::kBFloat16) || k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type() ||
        heads <= 0 || q.dim() != 3 || q.size(2) != heads * 64 || !(scale > 1e-30 && scale < 1e30) || q_start < -(1 << 29) || q_start > 1 << 29)
        return c10::nullopt;
    // a tangent needs no requires_grad and outlives no_grad(): looked for in every call, also in those that keep nothing for a backward
    if (c10::AutogradState::get_tls_state().get_fw_grad_mode())
        for (const at::Tensor* t : std::initializer_list<const at::Tensor*>{&q, &k, &v, &table_})
            TORCH_CHECK_NOT_IMPLEMENTED(!t->_fw_grad(0).defined(), "relative_bias_attention: no forward-mode derivatives");
    const Config c = {first, kv_lens, heads, q_start, both, causal, frame_major, scale};
    const int bd = c.batch_dim();
    GVD_WANT(q.dim() == 3 && k.dim() == 3 && k.sizes() == v.sizes(), "q ", q.sizes(), ", k ", k.sizes(), ", v ", v.sizes(), ": three dimensions each, k and v of one shape");
    const int64_t B = q.size(bd), C = q.size(2);
    GVD_WANT(heads > 0 && C % heads == 0 && k.size(2) == C && (k.size(bd) == 1 || k.size(bd) == B), "q ", q.sizes(), ", k ", k.sizes(), " with ", heads,
             " heads: channels heads * d on either side, and one batch size (or one K / V for the whole batch)");
    GVD_WANT(table_.dim() == 2 && table_.size(1) == heads && table_.size(0) == (both ? 2 : 1) * first.numel() &&
                 (table_.scalar_type() == at::kFloat || table_.scalar_type() == at::kHalf || table_.scalar_type() == at::kBFloat16),
             "table ", table_.scalar_type(), " ", table_.sizes(), ": [buckets, heads] of float32, float16 or bfloat16, an even number of buckets where both directions have "
             "their own");
    for (const at::Tensor* t : std::initializer_list<const at::Tensor*>{&k, &v, &table_}) GVD_WANT(t->device() == q.device(), t == &k ? "k" : t == &v ? "v" : "table", " is on ", t->device(), ", q on ", q.device());
    for (const at::Tensor* t : std::initializer_list<const at::Tensor*>{&q_starts, &kv_lens})
        GVD_WANT(!t->defined() || (t->scalar_type() == at::kInt && t->dim() == 1 && t->size(0) == B && t->device() == q.device() && t->is_contiguous()),
                 t == &kv_lens ? "kv_lens" : "q_start", ": ", t->scalar_type(), " ", t->sizes(), " on ", t->device(), "; a contiguous int32 [", B, "] on ", q.device(), " is wanted");
    const at::Tensor table = table_.contiguous();
    if (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad() || table.requires_grad())) {
        TORCH_CHECK_NOT_IMPLEMENTED(!q_starts.defined(), "relative_bias_attention: gradients with one q_start for the whole batch only (a tensor of them is for inference)");
        if (k.size(bd) != B) {   // one K / V for the whole batch: the backward addresses one per entry, autograd sums their gradients
            std::vector<int64_t> shape = k.sizes().vec();
            shape[bd] = B;
            k = k.expand(shape);
            v = v.expand(shape);
        }
        refuse_foreign_nodes({&q, &k, &v, &table}, q.device());
        return differentiable(q, k, v, table, c);
    }
    return forward_(q, k, v, table, q_starts, c, nullptr);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m)
{
    m.doc() = "relative_bias_attention over libgvd_relattn.so (see csrc/relattn_torch_ext.cpp)";
    m.def("init", &init, "resolve the C-ABI entry points from the given library path");
    m.def("attend", &attend, "attention with a learned relative position bias, differentiable");
}
