// Host path of the Python package, in native code: argument checks, output allocation, workspaces, autograd nodes and the
// calls into the C ABI (include/inferno_b200_attn.h), on torch tensors.
//
// The kernels know nothing of torch; this module is the one place where the two meet.  It finds the ABI's entry points in
// the shared object it is given (bind), so that another build of the library (the range-checked one) can stand in.
//
// Why native: a forward + backward of a small problem keeps the GPU busy for 25-50 us, and the same path written in Python
// (autograd.Function, ctypes marshalling of 30 arguments, views for the slices of a packed projection) took the host 200 us
// (4 x 4 heads, T = 128, fp32) -- small calls were bound by it.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/version.h>

#include <ATen/ATen.h>
#include <ATen/core/LegacyTypeDispatch.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <dlfcn.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <deque>
#include <map>
#include <memory>
#include <mutex>
#include <optional>
#include <string>
#include <utility>
#include <vector>

#include "../../include/inferno_b200_attn.h"

namespace {

using at::Tensor;
using torch::autograd::SavedVariable;
using torch::autograd::Variable;
using torch::autograd::variable_list;

// ---- the C ABI, resolved once ----------------------------------------------------
struct Abi {
    decltype(&ib200_attn_workspace_bytes) workspace_bytes = nullptr;
    decltype(&ib200_attn_fwd_strided) attn_fwd = nullptr;
    decltype(&ib200_attn_fwd_chunk) attn_fwd_chunk = nullptr;
    decltype(&ib200_attn_bwd_strided) attn_bwd = nullptr;
    decltype(&ib200_linear_workspace_bytes) linear_workspace_bytes = nullptr;
    decltype(&ib200_linear_fwd_ws) linear_fwd = nullptr;
    decltype(&ib200_linear_bwd_ws) linear_bwd = nullptr;
    decltype(&ib200_fused_linear_workspace_bytes) fused_linear_workspace_bytes = nullptr;
    decltype(&ib200_fused_linear_fwd) fused_linear_fwd = nullptr;
    decltype(&ib200_fused_linear_bwd) fused_linear_bwd = nullptr;
    decltype(&ib200_feed_forward_workspace_bytes) feed_forward_workspace_bytes = nullptr;
    decltype(&ib200_feed_forward_bwd) feed_forward_bwd = nullptr;
    decltype(&ib200_layer_norm_workspace_bytes) layer_norm_workspace_bytes = nullptr;
    decltype(&ib200_layer_norm_fwd) layer_norm_fwd = nullptr;
    decltype(&ib200_layer_norm_bwd) layer_norm_bwd = nullptr;
    decltype(&ib200_attn_set_timing_events) set_timing_events = nullptr;
    decltype(&ib200_status_string) status_string = nullptr;
    PyObject* error_class = nullptr;      // the package's exception type, constructed from (status, where)
};
Abi g_abi;

// A status other than IB200_OK from the library.  It reaches Python as the package's own exception type, from the caller's thread
// (guarded) and from autograd's worker threads (in_node) alike.
struct StatusError : std::runtime_error {
    int status;
    const char* where;
    StatusError(int s, const char* w)
        : std::runtime_error(std::string(w) + ": " + g_abi.status_string(s) + " (status " + std::to_string(s) + ")"), status(s), where(w) {}
};
inline void check_status(int rc, const char* where) {
    if (rc != IB200_OK) throw StatusError(rc, where);
}

// ---- workspaces: caller-owned scratch of the C ABI, one per (device, stream), grown on demand ----------------------
// The number of entries is bounded by the number of streams a process uses (torch hands out a fixed pool of them).  A call
// holds its entry's lock while it issues its launches, so two host threads that share a stream cannot interleave the
// launches of two passes over one scratch buffer.  The table is never destroyed: at process exit the CUDA context may
// already be gone.  Attention and projections have a buffer each: a graph captured with the one must not lose it because an
// eager call of the other needs more.
struct Workspace {
    std::mutex launching;
    Tensor buf;            // attention; begins with the status header
    Tensor linear;
};
std::mutex g_ws_mutex;
std::map<std::pair<int, int64_t>, std::unique_ptr<Workspace>>& workspace_table() {
    static auto* t = new std::map<std::pair<int, int64_t>, std::unique_ptr<Workspace>>();
    return *t;
}
Workspace& workspace_of(int device, cudaStream_t stream) {
    const std::pair<int, int64_t> key{device, reinterpret_cast<int64_t>(stream)};
    std::lock_guard<std::mutex> lock(g_ws_mutex);
    auto& slot = workspace_table()[key];
    if (!slot) slot = std::make_unique<Workspace>();
    return *slot;
}
// under ws.launching
Tensor empty_bytes(size_t bytes, c10::Device device) { return at::empty({static_cast<int64_t>(bytes)}, at::TensorOptions().dtype(at::kByte).device(device)); }
void reserve(Tensor& buf, size_t bytes, c10::Device device) {
    if (!buf.defined() || static_cast<size_t>(buf.numel()) < bytes) buf = empty_bytes(bytes, device);
}
// The scratch of a projection or a layer norm.  While the stream is being captured it comes from the graph's own memory, and goes back there after the
// call: the graph then depends on nothing that a later call could replace.
Tensor linear_scratch(Workspace& ws, size_t bytes, c10::Device device) {
    if (c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None) return empty_bytes(bytes, device);
    reserve(ws.linear, bytes, device);
    return ws.linear;
}

// ---- timing events queued by a harness: one {start, stop} pair per attention call, forward and backward ----------------
struct TimingQueue {
    std::mutex m;
    std::deque<std::pair<cudaEvent_t, cudaEvent_t>> fwd, bwd;
    std::atomic<bool> any{false};
};
TimingQueue g_timing;
struct TimingScope {
    bool on = false;
    explicit TimingScope(bool backward) {
        if (!g_timing.any) return;
        std::lock_guard<std::mutex> lock(g_timing.m);
        auto& q = backward ? g_timing.bwd : g_timing.fwd;
        if (q.empty()) return;
        const auto ev = q.front();
        q.pop_front();
        g_timing.any = !g_timing.fwd.empty() || !g_timing.bwd.empty();
        auto e = [](cudaEvent_t x) { return reinterpret_cast<ib200_event_t>(x); };
        on = backward ? g_abi.set_timing_events(nullptr, nullptr, e(ev.first), e(ev.second)) == IB200_OK
                      : g_abi.set_timing_events(e(ev.first), e(ev.second), nullptr, nullptr) == IB200_OK;
    }
    ~TimingScope() {
        if (on) g_abi.set_timing_events(nullptr, nullptr, nullptr, nullptr);
    }
};

// ---- attention: checks and layouts -----------------------------------------------
int dtype_code(const Tensor& t) { return t.scalar_type() == at::kFloat ? IB200_DTYPE_F32 : IB200_DTYPE_BF16; }

void check_inputs(std::initializer_list<const Tensor*> ts) {
    const Tensor& q = **ts.begin();
    TORCH_CHECK_VALUE(q.dim() == 4, "causal_attention expects [B, H, T, D] tensors");
    for (const Tensor* t : ts) {
        TORCH_CHECK(t->is_cuda(), "causal_attention: tensor is not on a CUDA device (there is no CPU path)");
        TORCH_CHECK(t->device() == q.device(), "causal_attention: tensors are on different devices");
        TORCH_CHECK_TYPE(t->scalar_type() == q.scalar_type() && (t->scalar_type() == at::kFloat || t->scalar_type() == at::kBFloat16),
                         "causal_attention: dtype must be float32 or bfloat16, the same for all tensors");
        TORCH_CHECK_VALUE(t->sizes() == q.sizes(), "causal_attention: q, k, v (and dO) must have the same shape");
    }
}
// Caller-supplied outputs: any strides the kernels can address.
void check_like(const Tensor& t, const Tensor& q, const char* name) {
    TORCH_CHECK_VALUE(t.sizes() == q.sizes() && t.scalar_type() == q.scalar_type() && t.device() == q.device(), "causal_attention: `", name,
                      "` must match q in shape, dtype and device");
}
// The log-sum-exp vector is addressed densely by the kernels.
void check_lse_of(const Tensor& lse, c10::Device device, int64_t B, int64_t H, int64_t T) {
    TORCH_CHECK_VALUE(lse.scalar_type() == at::kFloat && lse.device() == device && lse.dim() == 3 && lse.size(0) == B && lse.size(1) == H &&
                          lse.size(2) == T && lse.is_contiguous(),
                      "causal_attention: `lse` must be a contiguous float32 [B, H, T] tensor on q's device");
}
void check_lse(const Tensor& lse, const Tensor& q) { check_lse_of(lse, q.device(), q.size(0), q.size(1), q.size(2)); }
// A packed [B, T, 3*H*D] operand.
void check_packed(const Tensor& qkv, int64_t H) {
    TORCH_CHECK_VALUE(qkv.dim() == 3 && H > 0, "causal_attention_packed expects a [B, T, 3*C] tensor and a positive number of heads");
    TORCH_CHECK(qkv.size(2) / 3 / H * H * 3 == qkv.size(2), "causal_attention_packed: the last axis (", qkv.size(2), ") is not 3 * num_heads * head_dim");
    TORCH_CHECK(qkv.is_cuda(), "causal_attention: tensor is not on a CUDA device (there is no CPU path)");
    TORCH_CHECK_TYPE(qkv.scalar_type() == at::kFloat || qkv.scalar_type() == at::kBFloat16,
                     "causal_attention: dtype must be float32 or bfloat16, the same for all tensors");
}

// A [B, H, T, D] operand as the C ABI takes it.
struct Operand {
    void* ptr;
    ib200_layout lay;
};
Operand operand(const Tensor& t) {
    TORCH_CHECK_VALUE(t.stride(3) == 1, "causal_attention: the head-dim axis must be contiguous");
    return {t.data_ptr(), {t.stride(0), t.stride(1), t.stride(2)}};
}
// In place when the kernels can address the tensor (contiguous rows, 16-byte aligned strides); otherwise the dense copy the
// reference makes with .contiguous().
Tensor dense_or_view(const Tensor& t) {
    const int64_t unit = 16 / t.element_size();
    bool ok = t.stride(3) == 1 && (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) == 0;
    for (int a = 0; a < 3; ++a) ok = ok && t.stride(a) > 0 && t.stride(a) % unit == 0;
    return ok ? t : t.contiguous();
}
// The same for a packed [B, T, n*H*D] tensor.
Tensor dense_or_packed(const Tensor& t) {
    const int64_t unit = 16 / t.element_size();
    const bool ok = t.stride(2) == 1 && t.stride(0) > 0 && t.stride(1) > 0 && t.stride(0) % unit == 0 && t.stride(1) % unit == 0 &&
                    (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) == 0;
    return ok ? t : t.contiguous();
}
// One third of a packed [B, T, 3, H, D] buffer, as a [B, H, T, D] operand.
Operand packed_operand(const Tensor& p, int which, int64_t C, int64_t D) {
    return {static_cast<char*>(p.data_ptr()) + static_cast<int64_t>(which) * C * p.element_size(), {p.stride(0), D, p.stride(1)}};
}

struct Shape {
    int B, H, T, D, dtype;
};
Shape shape_of(const Tensor& q) {
    return {static_cast<int>(q.size(0)), static_cast<int>(q.size(1)), static_cast<int>(q.size(2)), static_cast<int>(q.size(3)), dtype_code(q)};
}
float scale_of(const std::optional<double>& s, int64_t D) { return static_cast<float>(s ? *s : 1.0 / std::sqrt(static_cast<double>(D))); }

// ---- launches (the caller has made the tensors' device current) ------------------------------------------
void launch_fwd(const Shape& s, const Operand& q, const Operand& k, const Operand& v, const Operand& o, float* lse, float scale, bool causal,
                int math_mode, c10::Device device, int total_heads = 0) {
    size_t bytes = 0;
    check_status(g_abi.workspace_bytes(s.B, s.H, s.T, s.D, s.dtype, IB200_PASS_FWD, &bytes), "ib200_attn_workspace_bytes");
    cudaStream_t stream = c10::cuda::getCurrentCUDAStream(device.index()).stream();
    Workspace& ws = workspace_of(device.index(), stream);
    std::lock_guard<std::mutex> lock(ws.launching);
    reserve(ws.buf, bytes, device);
    TimingScope timing(false);
    if (total_heads > 0) {
        check_status(g_abi.attn_fwd_chunk(q.ptr, k.ptr, v.ptr, o.ptr, lse, &q.lay, &k.lay, &v.lay, &o.lay, total_heads, s.B, s.H, s.T, s.D, scale, causal,
                                          s.dtype, math_mode, ws.buf.data_ptr(), ws.buf.numel(), reinterpret_cast<ib200_stream_t>(stream)),
                     "ib200_attn_fwd_chunk");
        return;
    }
    check_status(g_abi.attn_fwd(q.ptr, k.ptr, v.ptr, o.ptr, lse, &q.lay, &k.lay, &v.lay, &o.lay, s.B, s.H, s.T, s.D, scale, causal, s.dtype, math_mode,
                                ws.buf.data_ptr(), ws.buf.numel(), reinterpret_cast<ib200_stream_t>(stream)),
                 "ib200_attn_fwd_strided");
}

void launch_bwd(const Shape& s, const Operand& q, const Operand& k, const Operand& v, const Operand& o, const Operand& dO, const float* lse,
                const Operand& dq, const Operand& dk, const Operand& dv, float scale, bool causal, int math_mode, c10::Device device) {
    size_t bytes = 0;
    check_status(g_abi.workspace_bytes(s.B, s.H, s.T, s.D, s.dtype, IB200_PASS_BWD, &bytes), "ib200_attn_workspace_bytes");
    cudaStream_t stream = c10::cuda::getCurrentCUDAStream(device.index()).stream();
    Workspace& ws = workspace_of(device.index(), stream);
    std::lock_guard<std::mutex> lock(ws.launching);
    reserve(ws.buf, bytes, device);
    TimingScope timing(true);
    check_status(g_abi.attn_bwd(q.ptr, k.ptr, v.ptr, o.ptr, dO.ptr, lse, dq.ptr, dk.ptr, dv.ptr, &q.lay, &k.lay, &v.lay, &o.lay, &dO.lay, &dq.lay, &dk.lay,
                                &dv.lay, s.B, s.H, s.T, s.D, scale, causal, s.dtype, math_mode, ws.buf.data_ptr(), ws.buf.numel(),
                                reinterpret_cast<ib200_stream_t>(stream)),
                 "ib200_attn_bwd_strided");
}

Tensor empty_lse(const Tensor& q, const Shape& s) { return at::empty({s.B, s.H, s.T}, q.options().dtype(at::kFloat)); }
// A [B, H, T, D] view over [B, T, H, D] memory: `y.transpose(1, 2).reshape(B, T, C)` is then free.
Tensor empty_bthd(const Tensor& q, const Shape& s) {
    const int64_t D = s.D, HD = static_cast<int64_t>(s.H) * D;
    return at::empty_strided({s.B, s.H, s.T, s.D}, {s.T * HD, D, HD, 1}, q.options());
}

// Forward on [B, H, T, D] tensors or views.
std::pair<Tensor, Tensor> attention_forward(const Tensor& q_, const Tensor& k_, const Tensor& v_, const std::optional<double>& scale, bool causal,
                                            int math_mode, const Tensor& out, const Tensor& lse_, bool bthd, int total_heads = 0) {
    check_inputs({&q_, &k_, &v_});
    const c10::cuda::CUDAGuard guard(q_.device());
    const Tensor q = dense_or_view(q_), k = dense_or_view(k_), v = dense_or_view(v_);
    const Shape s = shape_of(q);
    if (out.defined()) check_like(out, q, "out");
    if (lse_.defined()) check_lse(lse_, q);
    Tensor o = out.defined() ? out : bthd ? empty_bthd(q, s) : at::empty(q.sizes(), q.options());
    Tensor lse = lse_.defined() ? lse_ : empty_lse(q, s);
    launch_fwd(s, operand(q), operand(k), operand(v), operand(o), lse.data_ptr<float>(), scale_of(scale, s.D), causal, math_mode, q.device(), total_heads);
    return {o, lse};
}

struct Grads {
    Tensor dq, dk, dv;
};
Grads attention_backward(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& o_, const Tensor& dO_, const Tensor& lse,
                         const std::optional<double>& scale, bool causal, int math_mode, Tensor dq, Tensor dk, Tensor dv) {
    check_inputs({&q_, &k_, &v_, &o_, &dO_});
    const c10::cuda::CUDAGuard guard(q_.device());
    const Tensor q = dense_or_view(q_), k = dense_or_view(k_), v = dense_or_view(v_), o = dense_or_view(o_), dO = dense_or_view(dO_);
    const Shape s = shape_of(q);
    check_lse(lse, q);
    auto output = [&](Tensor& t, const char* name) {
        if (t.defined()) check_like(t, q, name); else t = at::empty(q.sizes(), q.options());
    };
    output(dq, "dq");
    output(dk, "dk");
    output(dv, "dv");
    launch_bwd(s, operand(q), operand(k), operand(v), operand(o), operand(dO), lse.data_ptr<float>(), operand(dq), operand(dk), operand(dv),
               scale_of(scale, s.D), causal, math_mode, q.device());
    return {dq, dk, dv};
}

// ---- autograd nodes ----------------------------------------------------------------
void set_python_error(const StatusError& e) {      // with the GIL
    PyObject* err = PyObject_CallFunction(g_abi.error_class, "is", e.status, e.where);
    if (!err) return;
    PyErr_SetObject(g_abi.error_class, err);
    Py_DECREF(err);
}
// Body of a node: a status becomes a Python exception that the engine carries over to the thread that called backward.
template <class F>
variable_list in_node(F&& f) {
    try {
        return f();
    } catch (const StatusError& e) {
        python_error err;
        {
            pybind11::gil_scoped_acquire gil;
            set_python_error(e);
            err.persist();
        }
        throw err;
    }
}
// The ops have no forward-mode derivative: a dual input must not lose its tangent silently.
void refuse_tangents(std::initializer_list<const Tensor*> ts, const char* op) {
    for (const Tensor* t : ts)
        TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(0).defined(), op, ": forward-mode differentiation is not implemented");
}

// The backward node of the fused op: saves q, k, v, out and lse; produces dq, dk, dv.  Plays the role a
// `class AttentionBackward : public Node` has in the reference (src/inferno/gradfn/node.h:23-45).
// The gradients of the operators below are not differentiable themselves.  Made with create_graph they get this node, so that a second derivative
// raises; without one it would come out short by their part of it.
struct NoSecondDerivative : torch::autograd::Node {
    const char* op;
    explicit NoSecondDerivative(const char* op_) : op(op_) {}
    variable_list apply(variable_list&&) override {
        TORCH_CHECK_NOT_IMPLEMENTED(false, op, ": second derivatives are not implemented");
    }
    std::string name() const override { return "NoSecondDerivative"; }
};
// `from`: which of the backward node's inputs the gradients depend on, saved there or not; all of them depend on dy.
void refuse_second_derivative(std::initializer_list<Tensor*> grads, const torch::autograd::Node& backward, std::initializer_list<uint32_t> from, const Tensor& dy,
                              const char* op) {
    if (!at::GradMode::is_enabled()) return;
    torch::autograd::edge_list edges = torch::autograd::collect_next_edges(dy);
    for (uint32_t i : from) edges.push_back(backward.next_edge(i));
    if (std::none_of(edges.begin(), edges.end(), [](const torch::autograd::Edge& e) { return e.is_valid(); })) return;
    auto node = std::shared_ptr<NoSecondDerivative>(new NoSecondDerivative(op), torch::autograd::deleteNode);
    node->set_next_edges(std::move(edges));
    for (Tensor* g : grads)
        if (g->defined()) torch::autograd::set_history(*g, node);
}

struct AttentionBackward : torch::autograd::Node {
    SavedVariable q, k, v, o, lse;
    double scale = 0;
    bool causal = true;
    int math_mode = 0;

    variable_list apply(variable_list&& grads) override {
        return in_node([&] { return backward(grads); });
    }
    variable_list backward(const variable_list& grads) {
        if (!grads[0].defined()) return variable_list(3);
        const Tensor tq = q.unpack(), tk = k.unpack(), tv = v.unpack(), to = o.unpack(shared_from_this()), tl = lse.unpack();
        at::AutoDispatchBelowADInplaceOrView below;
        const int64_t B = tq.size(0), H = tq.size(1), T = tq.size(2), D = tq.size(3), step = H * D * tq.element_size();
        auto at_byte = [](const Tensor& t) { return static_cast<const char*>(t.data_ptr()); };
        Tensor dq, dk, dv;
        // slices of one packed [B, T, 3, H, D] buffer get their gradients in one buffer of the same layout
        if (tq.strides() == tk.strides() && tk.strides() == tv.strides() && tq.stride(2) == 3 * H * D && tq.stride(1) == D &&
            at_byte(tk) - at_byte(tq) == step && at_byte(tv) - at_byte(tk) == step) {
            const Tensor g = at::empty({B, T, 3, H, D}, tq.options());
            dq = g.select(2, 0).transpose(1, 2);
            dk = g.select(2, 1).transpose(1, 2);
            dv = g.select(2, 2).transpose(1, 2);
        }
        Grads r = attention_backward(tq, tk, tv, to, grads[0], tl, scale, causal, math_mode, dq, dk, dv);
        refuse_second_derivative({&r.dq, &r.dk, &r.dv}, *this, {0, 1, 2}, grads[0], "causal_attention");
        return {r.dq, r.dk, r.dv};
    }
    void release_variables() override {
        q.reset_data(); k.reset_data(); v.reset_data(); o.reset_data(); lse.reset_data();
    }
    std::string name() const override { return "AttentionBackward"; }
};

Tensor causal_attention(const Tensor& q, const Tensor& k, const Tensor& v, const std::optional<double>& scale, bool causal, int math_mode, bool bthd,
                        int total_heads) {
    refuse_tangents({&q, &k, &v}, "causal_attention");
    const bool differentiable = torch::autograd::compute_requires_grad(q, k, v);
    Tensor o, lse;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        std::tie(o, lse) = attention_forward(q, k, v, scale, causal, math_mode, Tensor(), Tensor(), bthd, total_heads);
    }
    if (differentiable) {
        auto node = std::shared_ptr<AttentionBackward>(new AttentionBackward(), torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(q, k, v));
        node->q = SavedVariable(q, false);
        node->k = SavedVariable(k, false);
        node->v = SavedVariable(v, false);
        node->lse = SavedVariable(lse, false);
        node->scale = scale ? *scale : 1.0 / std::sqrt(static_cast<double>(q.size(3)));
        node->causal = causal;
        node->math_mode = math_mode;
        torch::autograd::set_history(o, node);
        node->o = SavedVariable(o, true);
    }
    return o;
}

// The same op on a fused projection output [B, T, 3*C]: one input, one gradient.  Written for three views of the packed
// buffer, autograd would fill a zeroed buffer per view, copy each slice's gradient into it and add the three up (240 of the
// 490 us of a 12-head T = 1024 B = 16 layer); here dq, dk, dv land in their places in the gradient itself.
struct PackedAttentionBackward : torch::autograd::Node {
    SavedVariable qkv, o, lse;      // o: [B, T, C]
    int64_t H = 0;
    float scale = 0;
    int math_mode = 0;

    variable_list apply(variable_list&& grads) override {
        return in_node([&] { return backward(grads); });
    }
    variable_list backward(const variable_list& grads) {
        if (!grads[0].defined()) return variable_list(1);
        const Tensor p_ = qkv.unpack(), o_ = o.unpack(shared_from_this()), tl = lse.unpack();
        at::AutoDispatchBelowADInplaceOrView below;
        // what was saved has passed through the user's saved-tensor hooks, and may come back with other strides, or as something else
        check_packed(p_, H);
        const c10::cuda::CUDAGuard guard(p_.device());
        const int64_t B = p_.size(0), T = p_.size(1), C = p_.size(2) / 3, D = C / H;
        for (const Tensor& t : {o_, grads[0]}) {
            TORCH_CHECK(t.device() == p_.device(), "causal_attention: tensors are on different devices");
            TORCH_CHECK_TYPE(t.scalar_type() == p_.scalar_type(), "causal_attention: dtype must be float32 or bfloat16, the same for all tensors");
            TORCH_CHECK_VALUE(t.dim() == 3 && t.size(0) == B && t.size(1) == T && t.size(2) == C, "causal_attention: the output and its gradient must be [B, T, C]");
        }
        check_lse_of(tl, p_.device(), B, H, T);
        const Tensor p = dense_or_packed(p_), to = dense_or_packed(o_), dy = dense_or_packed(grads[0]);
        const Shape s{static_cast<int>(B), static_cast<int>(H), static_cast<int>(T), static_cast<int>(D), dtype_code(p)};
        Tensor g = at::empty({B, T, 3 * C}, p.options());
        launch_bwd(s, packed_operand(p, 0, C, D), packed_operand(p, 1, C, D), packed_operand(p, 2, C, D), packed_operand(to, 0, C, D),
                   packed_operand(dy, 0, C, D), tl.data_ptr<float>(), packed_operand(g, 0, C, D), packed_operand(g, 1, C, D), packed_operand(g, 2, C, D), scale,
                   true, math_mode, p.device());
        refuse_second_derivative({&g}, *this, {0}, grads[0], "causal_attention");
        return {g};
    }
    void release_variables() override {
        qkv.reset_data(); o.reset_data(); lse.reset_data();
    }
    std::string name() const override { return "PackedAttentionBackward"; }
};

Tensor causal_attention_packed(const Tensor& qkv, int64_t H, const std::optional<double>& scale, int math_mode, int total_heads) {
    check_packed(qkv, H);
    const int64_t B = qkv.size(0), T = qkv.size(1), C = qkv.size(2) / 3, D = C / H;
    refuse_tangents({&qkv}, "causal_attention");
    const bool differentiable = torch::autograd::compute_requires_grad(qkv);
    Tensor o, lse, p;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        const c10::cuda::CUDAGuard guard(qkv.device());
        p = dense_or_packed(qkv);
        const Shape s{static_cast<int>(B), static_cast<int>(H), static_cast<int>(T), static_cast<int>(D), dtype_code(p)};
        o = at::empty({B, T, C}, p.options());
        lse = at::empty({B, H, T}, p.options().dtype(at::kFloat));
        launch_fwd(s, packed_operand(p, 0, C, D), packed_operand(p, 1, C, D), packed_operand(p, 2, C, D), packed_operand(o, 0, C, D), lse.data_ptr<float>(),
                   scale_of(scale, D), true, math_mode, p.device(), total_heads);
    }
    if (differentiable) {
        auto node = std::shared_ptr<PackedAttentionBackward>(new PackedAttentionBackward(), torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(qkv));
        node->qkv = SavedVariable(p, false);
        node->lse = SavedVariable(lse, false);
        node->H = H;
        node->scale = scale_of(scale, D);
        node->math_mode = math_mode;
        torch::autograd::set_history(o, node);
        node->o = SavedVariable(o, true);
    }
    return o;
}

// ---- projections -------------------------------------------------------------------
// Shapes first, ahead of any allocation: the kernels get no more than the pointers and M, K, N.
void check_linear_shapes(const Tensor& x, const Tensor& w) {
    TORCH_CHECK_VALUE(w.dim() == 2, "linear: w must be [in, out]");
    TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) == w.size(0), "linear: the last axis of x must be w's first (", w.size(0), "), x is ", x.sizes());
}
void check_same_device(const Tensor& t, const Tensor& x, const char* name) {
    TORCH_CHECK_VALUE(t.device() == x.device(), "linear: ", name, " is on ", t.device(), ", x on ", x.device());
}
void check_bf16_cuda(const Tensor& t, const char* name) {
    TORCH_CHECK(t.is_cuda(), "linear: ", name, " is not on a CUDA device (there is no CPU path)");
    TORCH_CHECK_TYPE(t.scalar_type() == at::kBFloat16, "linear: ", name, " must be bfloat16");
}

// The sizes that the kernels number (ib200_fused_linear_fwd).
constexpr int64_t kMaxLinearSize = 0x7fffff00 - 1;
int rows_of(const Tensor& x, int64_t K) {
    const int64_t M = x.numel() / K;
    TORCH_CHECK_VALUE(M <= kMaxLinearSize, "linear: too many rows, x is ", x.sizes());
    return static_cast<int>(M);
}
void check_weight_size(const Tensor& w) {
    const int64_t K = w.size(0), N = w.size(1);
    TORCH_CHECK_VALUE(K > 0 && N > 0 && K <= kMaxLinearSize && N <= kMaxLinearSize, "linear: w must have rows and columns, up to 2^31 - 257 of each, w is ", w.sizes());
}

Tensor linear_forward(const Tensor& x, const Tensor& w, const Tensor& bias) {
    check_linear_shapes(x, w);
    check_weight_size(w);
    const int64_t K = w.size(0), N = w.size(1);
    const int M = rows_of(x, K);
    TORCH_CHECK_VALUE(!bias.defined() || bias.numel() == N, "linear: the bias must have ", N, " elements");
    check_bf16_cuda(x, "x");
    check_bf16_cuda(w, "w");
    check_same_device(w, x, "w");
    if (bias.defined()) check_same_device(bias, x, "the bias");
    const c10::cuda::CUDAGuard guard(x.device());
    const Tensor x2 = x.reshape({-1, K}).contiguous(), wc = w.contiguous();
    Tensor b = bias;
    if (b.defined() && b.scalar_type() != at::kBFloat16) b = b.to(at::kFloat);
    if (b.defined()) b = b.contiguous();
    // the kernel reads a bias in place: a bf16 slice that does not begin on 16 bytes is copied, as it was when every bias became fp32
    if (b.defined() && b.scalar_type() == at::kBFloat16 && (reinterpret_cast<uintptr_t>(b.data_ptr()) & 15u)) b = b.clone();
    auto shape = x.sizes().vec();
    shape.back() = N;
    Tensor y = at::empty(shape, x.options());
    if (M == 0) return y;
    const size_t bytes = g_abi.linear_workspace_bytes(M, static_cast<int>(K), static_cast<int>(N), IB200_PASS_FWD);
    cudaStream_t stream = c10::cuda::getCurrentCUDAStream(x.device().index()).stream();
    std::unique_lock<std::mutex> lock;
    Tensor scratch;
    if (bytes) {
        Workspace& ws = workspace_of(x.device().index(), stream);
        lock = std::unique_lock<std::mutex>(ws.launching);
        scratch = linear_scratch(ws, bytes, x.device());
    }
    check_status(g_abi.linear_fwd(x2.data_ptr(), wc.data_ptr(), b.defined() ? b.data_ptr() : nullptr, b.defined() ? dtype_code(b) : IB200_DTYPE_F32,
                                  y.data_ptr(), M, static_cast<int>(K), static_cast<int>(N), bytes ? scratch.data_ptr() : nullptr, bytes,
                                  reinterpret_cast<ib200_stream_t>(stream)),
                 "ib200_linear_fwd_ws");
    return y;
}

struct LinearGrads {
    Tensor dx, dw, db;
};
LinearGrads linear_backward(const Tensor& x, const Tensor& w, const Tensor& dy, bool need_dx, bool need_dw, bool need_db, bool db_bf16) {
    check_linear_shapes(x, w);
    check_weight_size(w);
    const int64_t K = w.size(0), N = w.size(1);
    const int M = rows_of(x, K);
    TORCH_CHECK_VALUE(dy.dim() >= 1 && dy.size(-1) == N && dy.numel() / N == M,
                      "linear: dy must have the rows of x and ", N, " columns, dy is ", dy.sizes(), ", x is ", x.sizes());
    check_bf16_cuda(x, "x");
    check_bf16_cuda(w, "w");
    check_bf16_cuda(dy, "dy");
    check_same_device(w, x, "w");
    check_same_device(dy, x, "dy");
    const c10::cuda::CUDAGuard guard(x.device());
    const Tensor x2 = x.reshape({-1, K}).contiguous(), dy2 = dy.reshape({-1, N}).contiguous(), wc = w.contiguous();
    LinearGrads g;
    const auto db_type = x.options().dtype(db_bf16 ? at::kBFloat16 : at::kFloat);
    if (need_dx) g.dx = at::empty(x.sizes(), x.options());
    if (need_dw) g.dw = M ? at::empty({K, N}, x.options()) : at::zeros({K, N}, x.options());
    if (need_db) g.db = M ? at::empty({N}, db_type) : at::zeros({N}, db_type);
    if (M == 0) return g;
    const size_t bytes = g_abi.linear_workspace_bytes(M, static_cast<int>(K), static_cast<int>(N), IB200_PASS_BWD);
    cudaStream_t stream = c10::cuda::getCurrentCUDAStream(x.device().index()).stream();
    Workspace& ws = workspace_of(x.device().index(), stream);
    std::lock_guard<std::mutex> lock(ws.launching);
    const Tensor scratch = linear_scratch(ws, bytes, x.device());
    auto ptr = [](const Tensor& t) -> void* { return t.defined() ? t.data_ptr() : nullptr; };
    check_status(g_abi.linear_bwd(x2.data_ptr(), wc.data_ptr(), dy2.data_ptr(), ptr(g.dx), ptr(g.dw), ptr(g.db), db_bf16 ? IB200_DTYPE_BF16 : IB200_DTYPE_F32, M,
                                  static_cast<int>(K), static_cast<int>(N), scratch.data_ptr(), bytes,
                                  reinterpret_cast<ib200_stream_t>(stream)),
                 "ib200_linear_bwd_ws");
    return g;
}

struct LinearBackward : torch::autograd::Node {
    SavedVariable x, w;
    bool has_bias = false;
    at::ScalarType bias_type = at::kFloat;

    variable_list apply(variable_list&& grads) override {
        return in_node([&] { return backward(grads); });
    }
    variable_list backward(const variable_list& grads) {
        variable_list out(3);
        if (!grads[0].defined()) return out;
        const Tensor tx = x.unpack(), tw = w.unpack();
        at::AutoDispatchBelowADInplaceOrView below;
        LinearGrads g = linear_backward(tx, tw, grads[0], task_should_compute_output(0), task_should_compute_output(1),
                                        has_bias && task_should_compute_output(2), bias_type == at::kBFloat16);
        if (g.db.defined()) g.db = g.db.to(bias_type);      // fp32 and bf16 come in the right type
        refuse_second_derivative({&g.dx, &g.dw, &g.db}, *this, {0, 1}, grads[0], "linear");
        out = {g.dx, g.dw, g.db};
        return out;
    }
    void release_variables() override { x.reset_data(); w.reset_data(); }
    std::string name() const override { return "LinearBackward"; }
};

Tensor linear(const Tensor& x, const Tensor& w, const Tensor& bias) {
    refuse_tangents({&x, &w, &bias}, "linear");
    const bool differentiable = torch::autograd::compute_requires_grad(x, w, bias);
    Tensor y;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        y = linear_forward(x, w, bias);
    }
    if (differentiable) {
        auto node = std::shared_ptr<LinearBackward>(new LinearBackward(), torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(x, w, bias));
        node->x = SavedVariable(x, false);
        node->w = SavedVariable(w, false);
        node->has_bias = bias.defined();
        if (bias.defined()) node->bias_type = bias.scalar_type();
        torch::autograd::set_history(y, node);
    }
    return y;
}

// ---- projections with an activation and a residual, and the feed-forward block of two of them ----------------------------
void* ptr_or_null(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
// What the kernels address: dense, on 16 bytes.
Tensor dense16(const Tensor& t) {
    if (!t.defined()) return t;
    const Tensor d = t.contiguous();
    return reinterpret_cast<uintptr_t>(d.data_ptr()) & 15u ? d.clone() : d;
}
// A projection's weight and bias, the shapes ahead of devices and types; `like`: a tensor on the device they must be on.
void check_weight_shapes(const Tensor& w, const Tensor& bias) {
    check_weight_size(w);
    const int64_t N = w.size(1);
    TORCH_CHECK_VALUE(!bias.defined() || (bias.dim() == 1 && bias.size(0) == N), "linear: the bias must be [", N, "]");
}
void check_weight_types(const Tensor& w, const Tensor& bias, const Tensor& like) {
    check_bf16_cuda(w, "w");
    check_same_device(w, like, "w");
    if (!bias.defined()) return;
    check_same_device(bias, like, "the bias");
    TORCH_CHECK_TYPE(bias.scalar_type() == at::kFloat || bias.scalar_type() == at::kBFloat16, "linear: the bias must be float32 or bfloat16");
}
// A tensor of the output's shape: x's, with N columns.
void check_output_like(const Tensor& t, const Tensor& x, int64_t N, const char* name) {
    const bool ok = t.dim() == x.dim() && t.size(-1) == N && t.sizes().slice(0, t.dim() - 1) == x.sizes().slice(0, x.dim() - 1);
    TORCH_CHECK_VALUE(ok, "linear: ", name, " must have the output's shape, x's with a last axis of ", N, "; it is ", t.sizes(), ", x is ", x.sizes());
}
void check_output_type(const Tensor& t, const Tensor& x, const char* name) {
    check_same_device(t, x, name);
    check_bf16_cuda(t, name);
}
void check_fused(const Tensor& x, const Tensor& w, const Tensor& bias, const Tensor& residual) {
    check_linear_shapes(x, w);
    check_weight_shapes(w, bias);
    if (residual.defined()) check_output_like(residual, x, w.size(1), "the residual");
    rows_of(x, w.size(0));
    check_bf16_cuda(x, "x");
    check_weight_types(w, bias, x);
    if (residual.defined()) check_output_type(residual, x, "the residual");
}
// Scratch of one call, held with the stream's lock until its launches are issued.
struct Scratch {
    std::unique_lock<std::mutex> lock;
    Tensor buf;
    Scratch(size_t bytes, c10::Device device, cudaStream_t stream) {
        if (!bytes) return;
        Workspace& ws = workspace_of(device.index(), stream);
        lock = std::unique_lock<std::mutex>(ws.launching);
        buf = linear_scratch(ws, bytes, device);
    }
    void* ptr() const { return ptr_or_null(buf); }
};

struct Fused {
    Tensor y, slope;
};
// y = act(x w + bias) + residual; with `keep` (and an activation) act'(x w + bias) as fp16, for the backward.
Fused fused_linear_forward(const Tensor& x_, const Tensor& w_, const Tensor& bias_, int act, const Tensor& residual_, bool keep) {
    check_fused(x_, w_, bias_, residual_);
    const c10::cuda::CUDAGuard guard(x_.device());
    const int64_t K = w_.size(0), N = w_.size(1);
    const int M = rows_of(x_, K);
    auto shape = x_.sizes().vec();
    shape.back() = N;
    Fused r;
    r.y = at::empty(shape, x_.options());
    if (keep && act != IB200_ACT_NONE) r.slope = at::empty(shape, x_.options().dtype(at::kHalf));
    if (M == 0) return r;
    const Tensor x = dense16(x_), w = dense16(w_), b = dense16(bias_), res = dense16(residual_);
    const int k = static_cast<int>(K), n = static_cast<int>(N);
    cudaStream_t stream = c10::cuda::getCurrentCUDAStream(x.device().index()).stream();
    const size_t bytes = g_abi.fused_linear_workspace_bytes(M, k, n, act, IB200_PASS_FWD);
    const Scratch scratch(bytes, x.device(), stream);
    check_status(g_abi.fused_linear_fwd(x.data_ptr(), w.data_ptr(), ptr_or_null(b), b.defined() ? dtype_code(b) : IB200_DTYPE_F32, ptr_or_null(res), act,
                                        r.y.data_ptr(), ptr_or_null(r.slope), M, k, n, scratch.ptr(), bytes, reinterpret_cast<ib200_stream_t>(stream)),
                 "ib200_fused_linear_fwd");
    return r;
}
void check_slope(const Tensor& slope, const Tensor& x, int64_t N) {
    TORCH_CHECK_VALUE(slope.defined() && slope.numel() == x.numel() / x.size(-1) * N && slope.device() == x.device() && slope.scalar_type() == at::kHalf,
                      "linear: slope must be the float16 tensor that the forward kept");
}
LinearGrads fused_linear_backward(const Tensor& x_, const Tensor& w_, const Tensor& dy_, const Tensor& slope_, int act, bool need_dx, bool need_dw, bool need_db,
                                  bool db_bf16) {
    check_linear_shapes(x_, w_);
    const int64_t K = w_.size(0), N = w_.size(1);
    check_output_like(dy_, x_, N, "dy");
    check_fused(x_, w_, Tensor(), Tensor());
    check_output_type(dy_, x_, "dy");
    if (act != IB200_ACT_NONE) check_slope(slope_, x_, N);
    const c10::cuda::CUDAGuard guard(x_.device());
    const int M = rows_of(x_, K);
    LinearGrads g;
    const auto db_type = x_.options().dtype(db_bf16 ? at::kBFloat16 : at::kFloat);
    if (need_dx) g.dx = at::empty(x_.sizes(), x_.options());
    if (need_dw) g.dw = M ? at::empty({K, N}, x_.options()) : at::zeros({K, N}, x_.options());
    if (need_db) g.db = M ? at::empty({N}, db_type) : at::zeros({N}, db_type);
    if (M == 0 || (!need_dx && !need_dw && !need_db)) return g;
    const Tensor x = dense16(x_), w = dense16(w_), dy = dense16(dy_), slope = act != IB200_ACT_NONE ? dense16(slope_) : Tensor();
    const int k = static_cast<int>(K), n = static_cast<int>(N);
    cudaStream_t stream = c10::cuda::getCurrentCUDAStream(x.device().index()).stream();
    const size_t bytes = g_abi.fused_linear_workspace_bytes(M, k, n, act, IB200_PASS_BWD);
    const Scratch scratch(bytes, x.device(), stream);
    check_status(g_abi.fused_linear_bwd(x.data_ptr(), w.data_ptr(), dy.data_ptr(), ptr_or_null(slope), act, ptr_or_null(g.dx), ptr_or_null(g.dw), ptr_or_null(g.db),
                                        db_bf16 ? IB200_DTYPE_BF16 : IB200_DTYPE_F32, M, k, n, scratch.ptr(), bytes, reinterpret_cast<ib200_stream_t>(stream)),
                 "ib200_fused_linear_bwd");
    return g;
}

struct FusedLinearBackward : torch::autograd::Node {
    SavedVariable x, w, slope;
    int act = IB200_ACT_NONE;
    at::ScalarType bias_type = at::kFloat;

    variable_list apply(variable_list&& grads) override {
        return in_node([&] { return backward(grads); });
    }
    variable_list backward(const variable_list& grads) {
        variable_list out(4);
        if (!grads[0].defined()) return out;
        const Tensor tx = x.unpack(), tw = w.unpack(), tp = act != IB200_ACT_NONE ? slope.unpack() : Tensor();
        at::AutoDispatchBelowADInplaceOrView below;
        LinearGrads g = fused_linear_backward(tx, tw, grads[0], tp, act, task_should_compute_output(0), task_should_compute_output(1),
                                              task_should_compute_output(2), bias_type == at::kBFloat16);
        // the slope of an activation was taken at x w + bias
        if (act != IB200_ACT_NONE) refuse_second_derivative({&g.dx, &g.dw, &g.db}, *this, {0, 1, 2}, grads[0], "fused_linear");
        else refuse_second_derivative({&g.dx, &g.dw, &g.db}, *this, {0, 1}, grads[0], "fused_linear");
        out = {g.dx, g.dw, g.db, task_should_compute_output(3) ? grads[0] : Tensor()};      // the residual's gradient is dy itself
        return out;
    }
    void release_variables() override { x.reset_data(); w.reset_data(); slope.reset_data(); }
    std::string name() const override { return "FusedLinearBackward"; }
};

Tensor fused_linear(const Tensor& x, const Tensor& w, const Tensor& bias, int act, const Tensor& residual) {
    refuse_tangents({&x, &w, &bias, &residual}, "fused_linear");
    const bool differentiable = torch::autograd::compute_requires_grad(x, w, bias, residual);
    Fused r;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        r = fused_linear_forward(x, w, bias, act, residual, differentiable);
    }
    if (differentiable) {
        auto node = std::shared_ptr<FusedLinearBackward>(new FusedLinearBackward(), torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(x, w, bias, residual));
        node->x = SavedVariable(x, false);
        node->w = SavedVariable(w, false);
        node->act = act;
        if (r.slope.defined()) node->slope = SavedVariable(r.slope, false);
        if (bias.defined()) node->bias_type = bias.scalar_type();
        torch::autograd::set_history(r.y, node);
    }
    return r.y;
}

// y = gelu(x w1 + b1) w2 + b2 (+ residual)
void check_feed_forward(const Tensor& x, const Tensor& w1, const Tensor& b1, const Tensor& w2, const Tensor& b2, const Tensor& residual) {
    check_linear_shapes(x, w1);
    TORCH_CHECK_VALUE(w2.dim() == 2 && w2.size(0) == w1.size(1) && w2.size(1) == w1.size(0), "feed_forward: w2 must be w1's shape turned round, w1 is ", w1.sizes(),
                      ", w2 is ", w2.sizes());
    check_weight_shapes(w1, b1);
    check_weight_shapes(w2, b2);
    if (residual.defined()) check_output_like(residual, x, x.size(-1), "the residual");
    rows_of(x, w1.size(0));
    check_bf16_cuda(x, "x");
    check_weight_types(w1, b1, x);
    check_weight_types(w2, b2, x);
    if (residual.defined()) check_output_type(residual, x, "the residual");
}
struct FeedForwardGrads {
    Tensor dx, dw1, db1, dw2, db2;
};
FeedForwardGrads feed_forward_backward(const Tensor& x_, const Tensor& w1_, const Tensor& slope_, const Tensor& h_, const Tensor& w2_, const Tensor& dy_,
                                       const bool (&need)[5], at::ScalarType b1_type, at::ScalarType b2_type) {
    check_feed_forward(x_, w1_, Tensor(), w2_, Tensor(), Tensor());
    const int64_t C = w1_.size(0), H = w1_.size(1);
    check_output_like(dy_, x_, C, "dy");
    check_output_type(dy_, x_, "dy");
    check_slope(slope_, x_, H);
    TORCH_CHECK_VALUE(h_.numel() == slope_.numel() && h_.device() == x_.device() && h_.scalar_type() == at::kBFloat16, "feed_forward: h must be the forward's hidden layer");
    const c10::cuda::CUDAGuard guard(x_.device());
    const int M = rows_of(x_, C);
    auto output = [&](bool wanted, at::IntArrayRef shape, at::ScalarType type) {
        if (!wanted) return Tensor();
        return M ? at::empty(shape, x_.options().dtype(type)) : at::zeros(shape, x_.options().dtype(type));
    };
    FeedForwardGrads g{output(need[0], x_.sizes(), at::kBFloat16), output(need[1], {C, H}, at::kBFloat16), output(need[2], {H}, b1_type),
                       output(need[3], {H, C}, at::kBFloat16), output(need[4], {C}, b2_type)};
    if (M == 0) return g;
    const Tensor x = dense16(x_), w1 = dense16(w1_), slope = dense16(slope_), h = dense16(h_), w2 = dense16(w2_), dy = dense16(dy_);
    const int c = static_cast<int>(C), hh = static_cast<int>(H);
    auto code = [](at::ScalarType t) { return t == at::kBFloat16 ? IB200_DTYPE_BF16 : IB200_DTYPE_F32; };
    cudaStream_t stream = c10::cuda::getCurrentCUDAStream(x.device().index()).stream();
    const size_t bytes = g_abi.feed_forward_workspace_bytes(M, c, hh);
    const Scratch scratch(bytes, x.device(), stream);
    check_status(g_abi.feed_forward_bwd(x.data_ptr(), w1.data_ptr(), slope.data_ptr(), h.data_ptr(), w2.data_ptr(), dy.data_ptr(), ptr_or_null(g.dx), ptr_or_null(g.dw1),
                                        ptr_or_null(g.db1), code(b1_type), ptr_or_null(g.dw2), ptr_or_null(g.db2), code(b2_type), M, c, hh, scratch.ptr(), bytes,
                                        reinterpret_cast<ib200_stream_t>(stream)),
                 "ib200_feed_forward_bwd");
    return g;
}

struct FeedForwardBackward : torch::autograd::Node {
    SavedVariable x, w1, slope, h, w2;
    at::ScalarType b1_type = at::kFloat, b2_type = at::kFloat;

    variable_list apply(variable_list&& grads) override {
        return in_node([&] { return backward(grads); });
    }
    variable_list backward(const variable_list& grads) {
        if (!grads[0].defined()) return variable_list(6);
        const Tensor tx = x.unpack(), t1 = w1.unpack(), tp = slope.unpack(), th = h.unpack(), t2 = w2.unpack();
        at::AutoDispatchBelowADInplaceOrView below;
        bool need[5];
        for (int i = 0; i < 5; ++i) need[i] = task_should_compute_output(i);
        FeedForwardGrads g = feed_forward_backward(tx, t1, tp, th, t2, grads[0], need, b1_type, b2_type);
        refuse_second_derivative({&g.dx, &g.dw1, &g.db1, &g.dw2, &g.db2}, *this, {0, 1, 2, 3}, grads[0], "feed_forward");      // x, w1, b1, w2
        return {g.dx, g.dw1, g.db1, g.dw2, g.db2, task_should_compute_output(5) ? grads[0] : Tensor()};
    }
    void release_variables() override {
        x.reset_data(); w1.reset_data(); slope.reset_data(); h.reset_data(); w2.reset_data();
    }
    std::string name() const override { return "FeedForwardBackward"; }
};

Tensor feed_forward(const Tensor& x, const Tensor& w1, const Tensor& b1, const Tensor& w2, const Tensor& b2, const Tensor& residual) {
    refuse_tangents({&x, &w1, &b1, &w2, &b2, &residual}, "feed_forward");
    check_feed_forward(x, w1, b1, w2, b2, residual);
    const bool differentiable = torch::autograd::compute_requires_grad(x, w1, b1, w2, b2, residual);
    Fused hidden, r;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        hidden = fused_linear_forward(x, w1, b1, IB200_ACT_GELU, Tensor(), differentiable);
        r = fused_linear_forward(hidden.y, w2, b2, IB200_ACT_NONE, residual, false);
    }
    if (differentiable) {
        auto node = std::shared_ptr<FeedForwardBackward>(new FeedForwardBackward(), torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(x, w1, b1, w2, b2, residual));
        node->x = SavedVariable(x, false);
        node->w1 = SavedVariable(w1, false);
        node->slope = SavedVariable(hidden.slope, false);
        node->h = SavedVariable(hidden.y, false);
        node->w2 = SavedVariable(w2, false);
        if (b1.defined()) node->b1_type = b1.scalar_type();
        if (b2.defined()) node->b2_type = b2.scalar_type();
        torch::autograd::set_history(r.y, node);
    }
    return r.y;
}

// ---- layer norm ----------------------------------------------------------------------
int type_code(const Tensor& t, const char* op, const char* name) {
    TORCH_CHECK_TYPE(t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16, op, ": ", name, " must be float32 or bfloat16");
    return dtype_code(t);
}
// Shapes first, as for the projections.
void check_layer_norm(const Tensor& x, const Tensor& weight, const Tensor& bias) {
    TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) > 0, "layer_norm: x needs a last axis to normalise, x is ", x.sizes());
    const int64_t C = x.size(-1);
    TORCH_CHECK_VALUE(x.numel() / C <= 0x7fffffff && C <= 0x7fffffff, "layer_norm: too many rows or columns, x is ", x.sizes());
    for (const Tensor* p : {&weight, &bias})
        TORCH_CHECK_VALUE(!p->defined() || (p->dim() == 1 && p->size(0) == C), "layer_norm: weight and bias must be [", C, "] like the last axis of x");
    TORCH_CHECK(x.is_cuda(), "layer_norm: x is not on a CUDA device (there is no CPU path)");
    type_code(x, "layer_norm", "x");
    for (const Tensor* p : {&weight, &bias}) {
        if (!p->defined()) continue;
        type_code(*p, "layer_norm", "weight and bias");
        TORCH_CHECK_VALUE(p->device() == x.device(), "layer_norm: weight and bias must be on x's device");
    }
    TORCH_CHECK_TYPE(!weight.defined() || !bias.defined() || weight.scalar_type() == bias.scalar_type(), "layer_norm: weight and bias must have the same dtype");
}
// The rows of a [..., C] tensor one pitch apart: in place where its axes allow it, otherwise a dense copy.
struct RowView {
    Tensor t;
    int64_t pitch;
};
RowView row_view(const Tensor& t) {
    const int64_t C = t.size(-1);
    if (t.numel() == 0) return {t, C};
    bool ok = C == 1 || t.stride(-1) == 1;
    int64_t pitch = C, span = 0;      // span: elements from one index of the axis above to the next, if the rows go on evenly
    for (int64_t a = t.dim() - 2; ok && a >= 0; --a) {
        if (t.size(a) == 1) continue;
        if (span == 0) pitch = t.stride(a);
        else ok = t.stride(a) == span;
        span = t.stride(a) * t.size(a);
        if (span == 0) ok = false;    // a broadcast axis: copied
    }
    if (ok) return {t, pitch};
    return {t.contiguous(), C};
}

struct Norm {
    Tensor y, mean, rstd;
};
Norm layer_norm_forward(const Tensor& x_, const Tensor& weight_, const Tensor& bias_, double eps, bool stats) {
    check_layer_norm(x_, weight_, bias_);
    TORCH_CHECK_VALUE(eps >= 0 && std::isfinite(eps), "layer_norm: eps must be finite and not negative, got ", eps);
    const c10::cuda::CUDAGuard guard(x_.device());
    const int64_t C = x_.size(-1);
    const RowView x = row_view(x_);
    const Tensor w = weight_.defined() ? weight_.contiguous() : weight_, b = bias_.defined() ? bias_.contiguous() : bias_;
    const int param = w.defined() ? dtype_code(w) : b.defined() ? dtype_code(b) : IB200_DTYPE_F32;
    Norm r;
    r.y = at::empty(x_.sizes(), x_.options());
    if (stats) {
        auto shape = x_.sizes().vec();
        shape.pop_back();
        r.mean = at::empty(shape, x_.options().dtype(at::kFloat));
        r.rstd = at::empty(shape, x_.options().dtype(at::kFloat));
    }
    if (x_.numel() == 0) return r;
    cudaStream_t stream = c10::cuda::getCurrentCUDAStream(x_.device().index()).stream();
    check_status(g_abi.layer_norm_fwd(x.t.data_ptr(), x.pitch, ptr_or_null(w), ptr_or_null(b), param, r.y.data_ptr(), static_cast<float*>(ptr_or_null(r.mean)),
                                      static_cast<float*>(ptr_or_null(r.rstd)), static_cast<int>(x_.numel() / C), static_cast<int>(C), static_cast<float>(eps), dtype_code(x_),
                                      reinterpret_cast<ib200_stream_t>(stream)),
                 "ib200_layer_norm_fwd");
    return r;
}

struct NormGrads {
    Tensor dx, dw, db;
};
// dw and db have the type of `weight` (without one: `param_type`).
NormGrads layer_norm_backward(const Tensor& x_, const Tensor& dy_, const Tensor& mean_, const Tensor& rstd_, const Tensor& weight_, bool need_dx, bool need_dw,
                              bool need_db, at::ScalarType param_type) {
    check_layer_norm(x_, weight_, Tensor());
    const int64_t C = x_.size(-1), M = x_.numel() / C;
    TORCH_CHECK_VALUE(dy_.sizes() == x_.sizes() && dy_.device() == x_.device(), "layer_norm: dy must have x's shape and device, dy is ", dy_.sizes(), ", x is ",
                      x_.sizes());
    TORCH_CHECK_TYPE(dy_.scalar_type() == x_.scalar_type(), "layer_norm: dy must have x's dtype");
    for (const Tensor* t : {&mean_, &rstd_})
        TORCH_CHECK_VALUE(t->numel() == M && t->scalar_type() == at::kFloat && t->device() == x_.device(),
                          "layer_norm: mean and rstd must be float32, one value per row of x, on its device");
    const c10::cuda::CUDAGuard guard(x_.device());
    const RowView x = row_view(x_), dy = row_view(dy_);
    const Tensor mean = mean_.contiguous(), rstd = rstd_.contiguous(), w = weight_.defined() ? weight_.contiguous() : weight_;
    if (w.defined()) param_type = w.scalar_type();
    NormGrads g;
    if (need_dx) g.dx = at::empty(x_.sizes(), x_.options());
    const auto param = x_.options().dtype(param_type);
    if (need_dw) g.dw = M ? at::empty({C}, param) : at::zeros({C}, param);
    if (need_db) g.db = M ? at::empty({C}, param) : at::zeros({C}, param);
    if (M == 0 || (!need_dx && !need_dw && !need_db)) return g;
    const int m = static_cast<int>(M), c = static_cast<int>(C), dtype = dtype_code(x_);
    const size_t bytes = need_dw || need_db ? g_abi.layer_norm_workspace_bytes(m, c, dtype) : 0;
    cudaStream_t stream = c10::cuda::getCurrentCUDAStream(x_.device().index()).stream();
    const Scratch scratch(bytes, x_.device(), stream);
    check_status(g_abi.layer_norm_bwd(x.t.data_ptr(), x.pitch, ptr_or_null(w), dy.t.data_ptr(), dy.pitch, mean.data_ptr<float>(), rstd.data_ptr<float>(), ptr_or_null(g.dx), ptr_or_null(g.dw),
                                      ptr_or_null(g.db), param_type == at::kBFloat16 ? IB200_DTYPE_BF16 : IB200_DTYPE_F32, m, c, dtype, scratch.ptr(), bytes,
                                      reinterpret_cast<ib200_stream_t>(stream)),
                 "ib200_layer_norm_bwd");
    return g;
}

struct LayerNormBackward : torch::autograd::Node {
    SavedVariable x, weight, mean, rstd;
    bool has_weight = false;
    at::ScalarType param_type = at::kFloat;

    variable_list apply(variable_list&& grads) override {
        return in_node([&] { return backward(grads); });
    }
    variable_list backward(const variable_list& grads) {
        if (!grads[0].defined()) return variable_list(3);
        const Tensor tx = x.unpack(), tw = has_weight ? weight.unpack() : Tensor(), tm = mean.unpack(), tr = rstd.unpack();
        at::AutoDispatchBelowADInplaceOrView below;
        NormGrads g = layer_norm_backward(tx, grads[0], tm, tr, tw, task_should_compute_output(0), task_should_compute_output(1),
                                          task_should_compute_output(2), param_type);
        refuse_second_derivative({&g.dx, &g.dw, &g.db}, *this, {0, 1}, grads[0], "layer_norm");      // x, weight
        return {g.dx, g.dw, g.db};
    }
    void release_variables() override {
        x.reset_data(); weight.reset_data(); mean.reset_data(); rstd.reset_data();
    }
    std::string name() const override { return "LayerNormBackward"; }
};

Tensor layer_norm(const Tensor& x, const Tensor& weight, const Tensor& bias, double eps) {
    refuse_tangents({&x, &weight, &bias}, "layer_norm");
    const bool differentiable = torch::autograd::compute_requires_grad(x, weight, bias);
    Norm r;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        r = layer_norm_forward(x, weight, bias, eps, differentiable);
    }
    if (differentiable) {
        auto node = std::shared_ptr<LayerNormBackward>(new LayerNormBackward(), torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(x, weight, bias));
        node->x = SavedVariable(x, false);
        node->mean = SavedVariable(r.mean, false);
        node->rstd = SavedVariable(r.rstd, false);
        node->has_weight = weight.defined();
        if (weight.defined()) node->weight = SavedVariable(weight, false);
        if (bias.defined()) node->param_type = bias.scalar_type();
        torch::autograd::set_history(r.y, node);
    }
    return r.y;
}

// ---- Python boundary ---------------------------------------------------------------
// Plain METH_FASTCALL functions: positional arguments, None for an absent tensor or the default scale.
const Tensor& arg_tensor(PyObject* o) {
    TORCH_CHECK_TYPE(THPVariable_Check(o), "expected a torch.Tensor, got ", Py_TYPE(o)->tp_name);
    return THPVariable_Unpack(o);
}
Tensor arg_opt_tensor(PyObject* o) { return o == Py_None ? Tensor() : arg_tensor(o); }
double arg_double(PyObject* o) {
    const double d = PyFloat_AsDouble(o);
    if (d == -1.0 && PyErr_Occurred()) throw python_error();
    return d;
}
std::optional<double> arg_scale(PyObject* o) {
    if (o == Py_None) return std::nullopt;
    return arg_double(o);
}
int64_t arg_int(PyObject* o) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw python_error();
    return v;
}
// None (0): the call is the whole problem; otherwise the heads of the problem that it is a part of.
int arg_total_heads(PyObject* o) {
    if (o == Py_None) return 0;
    const int64_t n = arg_int(o);
    TORCH_CHECK_VALUE(n > 0 && n <= 0x7fffffff, "causal_attention: total_heads must be a positive number of heads, got ", n);
    return static_cast<int>(n);
}
int arg_activation(PyObject* o) {
    if (o == Py_None) return IB200_ACT_NONE;
    const char* name = PyUnicode_Check(o) ? PyUnicode_AsUTF8(o) : nullptr;
    if (!name && PyErr_Occurred()) throw python_error();
    TORCH_CHECK_VALUE(name && std::string(name) == "gelu", "linear: activation must be None or \"gelu\"");
    return IB200_ACT_GELU;
}
bool arg_bool(PyObject* o) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw python_error();
    return v != 0;
}
void want(Py_ssize_t got, Py_ssize_t n) {
    TORCH_CHECK_TYPE(got == n, "expected ", n, " arguments, got ", got);
}
PyObject* wrap(const Tensor& t) {
    if (!t.defined()) Py_RETURN_NONE;
    return THPVariable_Wrap(t);
}
PyObject* wrap_tuple(std::initializer_list<const Tensor*> ts) {
    PyObject* out = PyTuple_New(static_cast<Py_ssize_t>(ts.size()));
    if (!out) throw python_error();
    Py_ssize_t i = 0;
    for (const Tensor* t : ts) PyTuple_SET_ITEM(out, i++, wrap(*t));
    return out;
}

template <class F>
PyObject* guarded(F&& f) {
    HANDLE_TH_ERRORS
    try {
        return f();
    } catch (const StatusError& e) {
        set_python_error(e);
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

PyObject* py_bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        want(n, 2);
        const char* path = PyUnicode_AsUTF8(a[0]);
        if (!path) throw python_error();
        void* so = dlopen(path, RTLD_NOW | RTLD_LOCAL);
        TORCH_CHECK(so, "cannot load ", path, ": ", dlerror());
        auto get = [&](auto& fn, const char* name) {
            fn = reinterpret_cast<std::decay_t<decltype(fn)>>(dlsym(so, name));
            TORCH_CHECK(fn, path, " does not export ", name);
        };
        get(g_abi.workspace_bytes, "ib200_attn_workspace_bytes");
        get(g_abi.attn_fwd, "ib200_attn_fwd_strided");
        get(g_abi.attn_fwd_chunk, "ib200_attn_fwd_chunk");
        get(g_abi.attn_bwd, "ib200_attn_bwd_strided");
        get(g_abi.linear_workspace_bytes, "ib200_linear_workspace_bytes");
        get(g_abi.linear_fwd, "ib200_linear_fwd_ws");
        get(g_abi.linear_bwd, "ib200_linear_bwd_ws");
        get(g_abi.fused_linear_workspace_bytes, "ib200_fused_linear_workspace_bytes");
        get(g_abi.fused_linear_fwd, "ib200_fused_linear_fwd");
        get(g_abi.fused_linear_bwd, "ib200_fused_linear_bwd");
        get(g_abi.feed_forward_workspace_bytes, "ib200_feed_forward_workspace_bytes");
        get(g_abi.feed_forward_bwd, "ib200_feed_forward_bwd");
        get(g_abi.layer_norm_workspace_bytes, "ib200_layer_norm_workspace_bytes");
        get(g_abi.layer_norm_fwd, "ib200_layer_norm_fwd");
        get(g_abi.layer_norm_bwd, "ib200_layer_norm_bwd");
        get(g_abi.set_timing_events, "ib200_attn_set_timing_events");
        get(g_abi.status_string, "ib200_status_string");
        Py_INCREF(a[1]);
        Py_XDECREF(g_abi.error_class);
        g_abi.error_class = a[1];
        Py_RETURN_NONE;
    });
}

// (q, k, v, scale, causal, math_mode, out, lse, total_heads) -> (o, lse)
PyObject* py_attention_forward(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        want(n, 9);
        const Tensor &q = arg_tensor(a[0]), &k = arg_tensor(a[1]), &v = arg_tensor(a[2]);
        const auto scale = arg_scale(a[3]);
        const bool causal = arg_bool(a[4]);
        const int math_mode = static_cast<int>(arg_int(a[5]));
        const Tensor out = arg_opt_tensor(a[6]), lse = arg_opt_tensor(a[7]);
        const int total_heads = arg_total_heads(a[8]);
        std::pair<Tensor, Tensor> r;
        {
            pybind11::gil_scoped_release nogil;
            at::AutoDispatchBelowADInplaceOrView below;
            r = attention_forward(q, k, v, scale, causal, math_mode, out, lse, false, total_heads);
        }
        return wrap_tuple({&r.first, &r.second});
    });
}

// (q, k, v, o, dO, lse, scale, causal, math_mode, dq, dk, dv) -> (dq, dk, dv)
PyObject* py_attention_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        want(n, 12);
        const Tensor &q = arg_tensor(a[0]), &k = arg_tensor(a[1]), &v = arg_tensor(a[2]), &o = arg_tensor(a[3]), &dO = arg_tensor(a[4]), &lse = arg_tensor(a[5]);
        const auto scale = arg_scale(a[6]);
        const bool causal = arg_bool(a[7]);
        const int math_mode = static_cast<int>(arg_int(a[8]));
        const Tensor dq = arg_opt_tensor(a[9]), dk = arg_opt_tensor(a[10]), dv = arg_opt_tensor(a[11]);
        Grads g;
        {
            pybind11::gil_scoped_release nogil;
            at::AutoDispatchBelowADInplaceOrView below;
            g = attention_backward(q, k, v, o, dO, lse, scale, causal, math_mode, dq, dk, dv);
        }
        return wrap_tuple({&g.dq, &g.dk, &g.dv});
    });
}

// (q, k, v, scale, causal, math_mode, bthd_out, total_heads) -> y, differentiable
PyObject* py_causal_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        want(n, 8);
        const Tensor &q = arg_tensor(a[0]), &k = arg_tensor(a[1]), &v = arg_tensor(a[2]);
        const auto scale = arg_scale(a[3]);
        const bool causal = arg_bool(a[4]);
        const int math_mode = static_cast<int>(arg_int(a[5]));
        const bool bthd = arg_bool(a[6]);
        const int total_heads = arg_total_heads(a[7]);
        Tensor y;
        {
            pybind11::gil_scoped_release nogil;
            y = causal_attention(q, k, v, scale, causal, math_mode, bthd, total_heads);
        }
        return wrap(y);
    });
}

// (qkv, num_heads, scale, math_mode, total_heads) -> y, differentiable
PyObject* py_causal_attention_packed(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        want(n, 5);
        const Tensor& qkv = arg_tensor(a[0]);
        const int64_t H = arg_int(a[1]);
        const auto scale = arg_scale(a[2]);
        const int math_mode = static_cast<int>(arg_int(a[3]));
        const int total_heads = arg_total_heads(a[4]);
        Tensor y;
        {
            pybind11::gil_scoped_release nogil;
            y = causal_attention_packed(qkv, H, scale, math_mode, total_heads);
        }
        return wrap(y);
    });
}

// (x, w, bias) -> y; the differentiable form and the plain one
PyObject* py_linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        want(n, 3);
        const Tensor &x = arg_tensor(a[0]), &w = arg_tensor(a[1]);
        const Tensor bias = arg_opt_tensor(a[2]);
        Tensor y;
        {
            pybind11::gil_scoped_release nogil;
            y = linear(x, w, bias);
        }
        return wrap(y);
    });
}
PyObject* py_linear_forward(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        want(n, 3);
        const Tensor &x = arg_tensor(a[0]), &w = arg_tensor(a[1]);
        const Tensor bias = arg_opt_tensor(a[2]);
        Tensor y;
        {
            pybind11::gil_scoped_release nogil;
            at::AutoDispatchBelowADInplaceOrView below;
            y = linear_forward(x, w, bias);
        }
        return wrap(y);
    });
}
// (x, w, dy, need_dx, need_dw, need_db) -> (dx, dw, db)
PyObject* py_linear_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        want(n, 6);
        const Tensor &x = arg_tensor(a[0]), &w = arg_tensor(a[1]), &dy = arg_tensor(a[2]);
        const bool need_dx = arg_bool(a[3]), need_dw = arg_bool(a[4]), need_db = arg_bool(a[5]);
        LinearGrads g;
        {
            pybind11::gil_scoped_release nogil;
            at::AutoDispatchBelowADInplaceOrView below;
            g = linear_backward(x, w, dy, need_dx, need_dw, need_db, false);
        }
        return wrap_tuple({&g.dx, &g.dw, &g.db});
    });
}

// (x, w, bias, activation, residual) -> y, differentiable
PyObject* py_fused_linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        want(n, 5);
        const Tensor &x = arg_tensor(a[0]), &w = arg_tensor(a[1]);
        const Tensor bias = arg_opt_tensor(a[2]), residual = arg_opt_tensor(a[4]);
        const int act = arg_activation(a[3]);
        Tensor y;
        {
            pybind11::gil_scoped_release nogil;
            y = fused_linear(x, w, bias, act, residual);
        }
        return wrap(y);
    });
}
// (x, w, bias, activation, residual, keep_slope) -> (y, slope)
PyObject* py_fused_linear_forward(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        want(n, 6);
        const Tensor &x = arg_tensor(a[0]), &w = arg_tensor(a[1]);
        const Tensor bias = arg_opt_tensor(a[2]), residual = arg_opt_tensor(a[4]);
        const int act = arg_activation(a[3]);
        const bool keep = arg_bool(a[5]);
        Fused r;
        {
            pybind11::gil_scoped_release nogil;
            at::AutoDispatchBelowADInplaceOrView below;
            r = fused_linear_forward(x, w, bias, act, residual, keep);
        }
        return wrap_tuple({&r.y, &r.slope});
    });
}
// (x, w, dy, slope, activation, need_dx, need_dw, need_db) -> (dx, dw, db)
PyObject* py_fused_linear_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        want(n, 8);
        const Tensor &x = arg_tensor(a[0]), &w = arg_tensor(a[1]), &dy = arg_tensor(a[2]);
        const Tensor slope = arg_opt_tensor(a[3]);
        const int act = arg_activation(a[4]);
        const bool need_dx = arg_bool(a[5]), need_dw = arg_bool(a[6]), need_db = arg_bool(a[7]);
        LinearGrads g;
        {
            pybind11::gil_scoped_release nogil;
            at::AutoDispatchBelowADInplaceOrView below;
            g = fused_linear_backward(x, w, dy, slope, act, need_dx, need_dw, need_db, false);
        }
        return wrap_tuple({&g.dx, &g.dw, &g.db});
    });
}
// (x, w1, b1, w2, b2, residual) -> y, differentiable
PyObject* py_feed_forward(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        want(n, 6);
        const Tensor &x = arg_tensor(a[0]), &w1 = arg_tensor(a[1]), &w2 = arg_tensor(a[3]);
        const Tensor b1 = arg_opt_tensor(a[2]), b2 = arg_opt_tensor(a[4]), residual = arg_opt_tensor(a[5]);
        Tensor y;
        {
            pybind11::gil_scoped_release nogil;
            y = feed_forward(x, w1, b1, w2, b2, residual);
        }
        return wrap(y);
    });
}

// (x, weight, bias, eps) -> y, differentiable
PyObject* py_layer_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        want(n, 4);
        const Tensor& x = arg_tensor(a[0]);
        const Tensor weight = arg_opt_tensor(a[1]), bias = arg_opt_tensor(a[2]);
        const double eps = arg_double(a[3]);
        Tensor y;
        {
            pybind11::gil_scoped_release nogil;
            y = layer_norm(x, weight, bias, eps);
        }
        return wrap(y);
    });
}
// (x, weight, bias, eps) -> (y, mean, rstd)
PyObject* py_layer_norm_forward(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        want(n, 4);
        const Tensor& x = arg_tensor(a[0]);
        const Tensor weight = arg_opt_tensor(a[1]), bias = arg_opt_tensor(a[2]);
        const double eps = arg_double(a[3]);
        Norm r;
        {
            pybind11::gil_scoped_release nogil;
            at::AutoDispatchBelowADInplaceOrView below;
            r = layer_norm_forward(x, weight, bias, eps, true);
        }
        return wrap_tuple({&r.y, &r.mean, &r.rstd});
    });
}
// (x, dy, mean, rstd, weight, need_dx, need_dw, need_db) -> (dx, dw, db)
PyObject* py_layer_norm_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        want(n, 8);
        const Tensor &x = arg_tensor(a[0]), &dy = arg_tensor(a[1]), &mean = arg_tensor(a[2]), &rstd = arg_tensor(a[3]);
        const Tensor weight = arg_opt_tensor(a[4]);
        const bool need_dx = arg_bool(a[5]), need_dw = arg_bool(a[6]), need_db = arg_bool(a[7]);
        NormGrads g;
        {
            pybind11::gil_scoped_release nogil;
            at::AutoDispatchBelowADInplaceOrView below;
            g = layer_norm_backward(x, dy, mean, rstd, weight, need_dx, need_dw, need_db, at::kFloat);
        }
        return wrap_tuple({&g.dx, &g.dw, &g.db});
    });
}

// () -> {(device index, stream handle): workspace tensor}
PyObject* py_workspaces(PyObject*, PyObject* const*, Py_ssize_t) {
    return guarded([&]() -> PyObject* {
        std::vector<std::pair<std::pair<int, int64_t>, Tensor>> list;
        {
            // A launch holds its entry's lock without the GIL and may come to need it there (to free a buffer that Python has seen, or
            // to allocate under a Python dispatch mode), so nobody waits for that lock with the GIL in hand.
            pybind11::gil_scoped_release nogil;
            std::lock_guard<std::mutex> lock(g_ws_mutex);
            for (const auto& [key, ws] : workspace_table()) {
                std::lock_guard<std::mutex> launching(ws->launching);
                if (ws->buf.defined()) list.emplace_back(key, ws->buf);
            }
        }
        PyObject* out = PyDict_New();
        if (!out) throw python_error();
        for (const auto& [key, buf] : list) {
            PyObject* k = Py_BuildValue("(iL)", key.first, static_cast<long long>(key.second));
            PyObject* v = wrap(buf);
            if (k && v) PyDict_SetItem(out, k, v);
            Py_XDECREF(k);
            Py_XDECREF(v);
        }
        return out;
    });
}

// ([(start, stop), ...] forward, the same for backward): CUDA event handles, consumed one pair per attention call in call order
PyObject* py_queue_timing_events(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        want(n, 2);
        std::deque<std::pair<cudaEvent_t, cudaEvent_t>> queues[2];      // filled first: reading a sequence may run Python code, which must not happen under the lock
        for (int i = 0; i < 2; ++i) {
            auto& q = queues[i];
            PyObject* seq = PySequence_Fast(a[i], "expected a sequence of event pairs");
            if (!seq) throw python_error();
            for (Py_ssize_t j = 0; j < PySequence_Fast_GET_SIZE(seq); ++j) {
                unsigned long long e0 = 0, e1 = 0;
                if (!PyArg_ParseTuple(PySequence_Fast_GET_ITEM(seq, j), "KK", &e0, &e1)) {
                    Py_DECREF(seq);
                    throw python_error();
                }
                q.emplace_back(reinterpret_cast<cudaEvent_t>(e0), reinterpret_cast<cudaEvent_t>(e1));
            }
            Py_DECREF(seq);
        }
        std::lock_guard<std::mutex> lock(g_timing.m);
        g_timing.fwd.swap(queues[0]);
        g_timing.bwd.swap(queues[1]);
        g_timing.any = !g_timing.fwd.empty() || !g_timing.bwd.empty();
        Py_RETURN_NONE;
    });
}

#define IB200_PY(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_##name)), METH_FASTCALL, nullptr}
PyMethodDef g_methods[] = {IB200_PY(bind),
                           IB200_PY(attention_forward),
                           IB200_PY(attention_backward),
                           IB200_PY(causal_attention),
                           IB200_PY(causal_attention_packed),
                           IB200_PY(linear),
                           IB200_PY(linear_forward),
                           IB200_PY(linear_backward),
                           IB200_PY(fused_linear),
                           IB200_PY(fused_linear_forward),
                           IB200_PY(fused_linear_backward),
                           IB200_PY(feed_forward),
                           IB200_PY(layer_norm),
                           IB200_PY(layer_norm_forward),
                           IB200_PY(layer_norm_backward),
                           IB200_PY(workspaces),
                           IB200_PY(queue_timing_events),
                           {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_host_ops", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host_ops() {
    PyObject* m = PyModule_Create(&g_module);
    // the torch whose classes this module was compiled against
    if (m && PyModule_AddStringConstant(m, "torch_version", TORCH_VERSION) < 0) {
        Py_DECREF(m);
        return nullptr;
    }
    return m;
}
