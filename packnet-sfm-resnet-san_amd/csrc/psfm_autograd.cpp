// psfm_autograd.cpp — linear_act and dropout as autograd nodes in C++ (module _psfm_autograd; networks/layers/linear.py and
// dropout.py check the arguments and call it).
//
// A training step of a small layer is host time: the forward and backward of these operators as Python functions
// took 45 and 36 us of a 137 us step on a 16 x 64 x 64 layer whose kernels take 15, and the two hand-overs
// to autograd's device thread, which sleeps longer the longer it waits, most of the rest.  The nodes call the
// C-ABI (include/psfm_linear.h, psfm_dropout.h) through the function pointers that the loaded library gave.
//
// HIP graphs: a node whose forward ran outside any capture, and whose graph lives, is counted by its stream, and the
// Python hooks on CUDAGraph.capture_begin ask for the counts (_hip.py says why such a capture is refused).
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/utils/pybind.h>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>

#include <atomic>
#include <mutex>
#include <unordered_map>

#include "psfm_linear.h"

namespace {

using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

const char* const VERSION = "psfm-autograd src=" PSFM_SRC_HASH;

struct Abi {
    decltype(&psfm_linear_fwd_ws_bytes) fwd_ws = nullptr;
    decltype(&psfm_linear_fwd) fwd = nullptr;
    decltype(&psfm_linear_bwd_ws_bytes) bwd_ws = nullptr;
    decltype(&psfm_linear_bwd) bwd = nullptr;
    decltype(&psfm_linear_last_error) linear_error = nullptr;
    decltype(&psfm_dropout) drop = nullptr;
    decltype(&psfm_dropout_last_error) drop_error = nullptr;
} entry;

// ---- live eager nodes --------------------------------------------------------------------------
struct Registry {
    std::mutex m;
    std::unordered_map<uintptr_t, int64_t> pending;   // by stream: forward ran, backward has not
    int64_t held = 0;                                 // backward ran on the default stream, graph still held
};
Registry& registry() {
    static Registry* r = new Registry;   // outlives every node
    return *r;
}
std::atomic<int> captures{0};
PyObject* refusal = nullptr;             // Python: joins the streams, returns the message

bool capturing() {
    return captures.load() > 0 && c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None;
}

class Live {
   public:
    void ran_forward(uintptr_t stream) {
        std::lock_guard<std::mutex> l(registry().m);
        stream_ = stream, state_ = PENDING;
        ++registry().pending[stream];
    }
    void ran_backward() {
        std::lock_guard<std::mutex> l(registry().m);
        leave();
        if (state_ == PENDING) state_ = stream_ == 0 ? HELD : NONE;
        if (state_ == HELD) ++registry().held;
    }
    ~Live() {
        std::lock_guard<std::mutex> l(registry().m);
        leave();
    }

   private:
    enum State { NONE, PENDING, HELD };
    void leave() {
        if (state_ == PENDING && --registry().pending[stream_] == 0) registry().pending.erase(stream_);
        if (state_ == HELD) --registry().held;
    }
    uintptr_t stream_ = 0;
    State state_ = NONE;
};

// (pending on other streams than this one, held)
std::pair<int64_t, int64_t> alive(uintptr_t stream) {
    std::lock_guard<std::mutex> l(registry().m);
    int64_t n = 0;
    for (const auto& e : registry().pending)
        if (e.first != stream) n += e.second;
    return {n, registry().held};
}

void refuse_foreign_capture() {
    if (captures.load() == 0 || capturing()) return;
    std::string msg;
    {
        py::gil_scoped_acquire gil;
        msg = py::reinterpret_borrow<py::object>(refusal)().cast<std::string>();
    }
    TORCH_CHECK(false, msg);
}

// A captured backward accumulates into a leaf on the stream that the leaf's accumulator is bound to, and an accumulator
// lives as long as any graph of its leaf does.  One left from eager work on the default stream cannot take part in a
// capture (the process ends in capture_end), so the forward is refused; and so where the leaf is reached through views and
// casts (conv1x1_act's weight, autocast's copies), one of which may itself be such a node.
void refuse_bound(const std::optional<c10::Stream>& s) {
    TORCH_CHECK(!s || s->id() != 0,
                "psfm: a HIP-graph capture is in progress and a graph from eager work on the default stream still holds one "
                "of this call's leaves, whose gradient a captured backward would accumulate on that stream.  Free the "
                "outputs of that work first (or run it on a side stream)");
}
void refuse_bound_leaf(const at::Tensor& t) {
    if (!t.defined() || !t.requires_grad()) return;
    if (t.is_leaf()) {
        if (const auto accumulator = torch::autograd::impl::try_get_grad_accumulator(t)) refuse_bound(accumulator->stream());
        return;
    }
    for (auto f = t.grad_fn(); f; f = f->num_outputs() == 1 ? f->next_edge(0).function : nullptr) refuse_bound(f->stream());
}

// ---- tensors -------------------------------------------------------------------------------------
void* at_of(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

void* stream_of(const at::Tensor& t) { return (void*)c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

int32_t dtype_of(const at::Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return PSFM_DTYPE_F32;
        case at::kHalf: return PSFM_DTYPE_F16;
        case at::kBFloat16: return PSFM_DTYPE_BF16;
        default: TORCH_CHECK(false, "float32, float16 or bfloat16 expected, got ", t.scalar_type());
    }
}

// t as a [rows, last dimension] matrix of one row stride (ld), copied where it is none
at::Tensor as_rows(const at::Tensor& t, int64_t& ld) {
    const int64_t cols = t.size(-1);
    ld = cols;
    if (t.is_contiguous()) return t;
    bool ok = t.stride(-1) == 1 || cols == 1, first = true;
    int64_t reach = 0;
    for (int64_t d = t.dim() - 2; ok && d >= 0; --d) {
        if (t.size(d) == 1) continue;
        if (first)
            ld = t.stride(d), first = false;
        else
            ok = t.stride(d) == reach;
        reach = t.stride(d) * t.size(d);
    }
    if (ok && ld >= cols) return t;
    ld = cols;
    return t.contiguous();
}

int64_t mask_rows(at::IntArrayRef shape, bool channels) {
    int64_t n = 1;
    if (channels)
        for (size_t d = 1; d + 1 < shape.size(); ++d) n *= shape[d];
    return std::max<int64_t>(n, 1);
}

int64_t lead_of(at::IntArrayRef shape) {
    int64_t n = 1;
    for (size_t d = 0; d + 1 < shape.size(); ++d) n *= shape[d];
    return n;
}

at::Tensor workspace(int64_t bytes, const at::Tensor& like) {
    return bytes > 0 ? at::empty({bytes}, like.options().dtype(at::kByte)) : at::Tensor();
}

bool wants(const at::Tensor& t) { return t.defined() && t.requires_grad(); }

// Forward-mode derivatives are refused: the result would silently carry none.
void refuse_tangents(const at::Tensor& t, const char* what) {
    TORCH_CHECK(!torch::autograd::isFwGradDefined(t), what, " has no forward-mode derivative");
}

// A gradient asked for with a graph of its own (create_graph) raises when that is differentiated.
at::Tensor once(const at::Tensor& g, const char* what) {
    if (!g.defined() || !at::GradMode::is_enabled()) return g;
    variable_list v{g.detach().set_requires_grad(true)};
    return torch::autograd::DelayedError(std::string(what) + " cannot be differentiated twice", 1).apply(std::move(v))[0];
}

// A saved tensor as it was kept, if it was.  Saved-tensor hooks may give back another one: it need not have the strides
// of the one that they took (a slice of a wider buffer comes back dense from the host), but its shape, type and
// device.
at::Tensor unpacked(const SavedVariable& v, const std::shared_ptr<torch::autograd::Node>& node, at::IntArrayRef shape,
                    at::ScalarType type, c10::Device device, const char* what) {
    const at::Tensor t = v.unpack(node);
    TORCH_CHECK(!t.defined() || (t.sizes() == shape && t.scalar_type() == type && t.device() == device), what,
                ": saved as ", shape, " ", type, " on ", device, ", given back as ", t.sizes(), " ", t.scalar_type(), " on ",
                t.device());
    return t;
}

at::Tensor dense(const at::Tensor& t) { return t.defined() ? t.contiguous() : t; }

// ---- linear_act ------------------------------------------------------------------------------------
struct LinearMeta {
    at::DimVector xshape, rshape;
    int64_t N, K, share;
    int32_t act;
    double p;
};

// what z is kept in: psfm_linear_fwd
at::ScalarType kept_type(at::ScalarType x, int act) {
    if (act == PSFM_ACT_RELU) return x;
    return x == at::kBFloat16 ? at::kHalf : at::kFloat;
}

struct LinearActBackward : public torch::autograd::Node {
    SavedVariable x, weight, z, rng;
    LinearMeta m;
    Live live;

    std::string name() const override { return "LinearActBackward"; }
    void release_variables() override {
        x.reset_data();
        weight.reset_data();
        z.reset_data();
        rng.reset_data();
    }

    variable_list apply(variable_list&& grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        refuse_foreign_capture();
        live.ran_backward();
        variable_list out(4);
        const at::Tensor& dy = grads[0];
        if (!dy.defined()) return out;
        const bool dx = task_should_compute_output(0), dw = task_should_compute_output(1),
                   db = task_should_compute_output(2);
        if (dx || dw || db) {
            const at::ScalarType type = dy.scalar_type();
            const c10::Device device = dy.device();
            c10::DeviceGuard guard(device);
            const auto self = shared_from_this();
            at::DimVector zshape = m.xshape;
            zshape.back() = m.N;
            // above autograd: a hook may run a checkpointed forward again, whose operators record their graphs
            const at::Tensor xu = unpacked(x, self, m.xshape, type, device, "linear_act: x"),
                             wu = unpacked(weight, self, {m.N, m.K}, type, device, "linear_act: weight"),
                             zu = unpacked(z, self, zshape, kept_type(type, m.act), device, "linear_act: z"),
                             ru = unpacked(rng, self, m.rshape, at::kLong, device, "linear_act: rng");
            at::AutoDispatchBelowADInplaceOrView below;
            int64_t ldx = m.K;
            const at::Tensor g = dy.contiguous(), xs = xu.defined() ? as_rows(xu, ldx) : xu, ws = dense(wu), zs = dense(zu),
                             rs = dense(ru);
            if (dx) out[0] = at::empty(m.xshape, g.options());
            if (dw) out[1] = at::empty({m.N, m.K}, g.options());
            if (db) out[2] = at::empty({m.N}, g.options());
            const psfm_linear d{lead_of(m.xshape), m.N, m.K, ldx, 0, dtype_of(g), m.act, m.p, m.share,
                                (const int64_t*)at_of(rs)};
            const int64_t n = entry.bwd_ws(&d, dx, dw, db);
            TORCH_CHECK(n >= 0, "psfm_linear_bwd_ws_bytes failed: ", entry.linear_error());
            const at::Tensor work = workspace(n, g);
            const int rc = entry.bwd(&d, at_of(g), at_of(xs), at_of(ws), at_of(zs), at_of(out[0]), at_of(out[1]), at_of(out[2]),
                                   at_of(work), stream_of(g));
            TORCH_CHECK(rc == 0, "psfm_linear_bwd failed (", rc, "): ", entry.linear_error());
        }
        for (int k = 0; k < 3; ++k) out[k] = once(out[k], "linear_act");
        if (task_should_compute_output(3)) out[3] = dy;
        return out;
    }
};

at::Tensor linear_act(const at::Tensor& x_, const at::Tensor& weight_, const std::optional<at::Tensor>& bias_, int64_t act,
                      const std::optional<at::Tensor>& residual_, double p, const std::optional<at::Tensor>& rng_,
                      bool channels) {
    refuse_foreign_capture();
    const at::Tensor bias_in = bias_.value_or(at::Tensor()), res_in = residual_.value_or(at::Tensor()),
                     rng = rng_.value_or(at::Tensor());
    for (const at::Tensor* t : {&x_, &weight_, &bias_in, &res_in}) refuse_tangents(*t, "linear_act");
    const bool grad_x = wants(x_), grad_w = wants(weight_), grad_b = wants(bias_in);
    std::shared_ptr<LinearActBackward> node;
    const bool in_capture = capturing();
    if (at::GradMode::is_enabled() && (grad_x || grad_w || grad_b || wants(res_in))) {
        if (in_capture)
            for (const at::Tensor& t : {x_, weight_, bias_in, res_in}) refuse_bound_leaf(t);
        node = std::shared_ptr<LinearActBackward>(new LinearActBackward(), torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(x_, weight_, bias_in, res_in));
    }
    at::Tensor y, z, x, weight;
    LinearMeta m;
    // ReLU's slope is the sign of its output where nothing follows it
    const bool from_y = act == PSFM_ACT_RELU && !res_in.defined() && !rng.defined();
    {
        at::AutoDispatchBelowADInplaceOrView below;
        c10::DeviceGuard guard(x_.device());
        int64_t ldx = 0, ldr = 0;
        x = as_rows(x_, ldx);
        weight = weight_.contiguous();
        const at::Tensor bias = bias_in.defined() ? bias_in.contiguous() : bias_in,
                         res = res_in.defined() ? as_rows(res_in, ldr) : res_in;
        m.xshape = at::DimVector(x.sizes());
        m.N = weight.size(0), m.K = weight.size(1), m.act = (int32_t)act, m.p = p;
        m.share = mask_rows(m.xshape, channels);
        if (rng.defined()) m.rshape = at::DimVector(rng.sizes());
        at::DimVector shape = m.xshape;
        shape.back() = m.N;
        y = at::empty(shape, x.options());
        if (node && act != PSFM_ACT_NONE && !from_y && (grad_x || grad_w || grad_b))
            z = at::empty(shape, x.options().dtype(kept_type(x.scalar_type(), (int)act)));
        const psfm_linear d{lead_of(m.xshape), m.N, m.K, ldx, ldr, dtype_of(x), m.act, p, m.share,
                            (const int64_t*)at_of(rng)};
        const int64_t n = entry.fwd_ws(&d);
        TORCH_CHECK(n >= 0, "psfm_linear_fwd_ws_bytes failed: ", entry.linear_error());
        const at::Tensor work = workspace(n, x);
        void* stream = stream_of(x);
        if (node && !in_capture) node->live.ran_forward((uintptr_t)stream);
        const int rc = entry.fwd(&d, at_of(x), at_of(weight), at_of(bias), at_of(res), at_of(y), at_of(z), at_of(work), stream);
        TORCH_CHECK(rc == 0, "psfm_linear_fwd failed (", rc, "): ", entry.linear_error());
    }
    if (node) {
        node->m = m;
        if (grad_w) node->x = SavedVariable(x, false);
        if (grad_x) node->weight = SavedVariable(weight, false);
        if (rng.defined()) node->rng = SavedVariable(rng, false);
        torch::autograd::set_history(y, node);
        if (from_y)
            node->z = SavedVariable(y, true);
        else if (z.defined())
            node->z = SavedVariable(z, false);
    }
    return y;
}

// ---- dropout ---------------------------------------------------------------------------------------
at::Tensor drop_launch(const at::Tensor& x_, const at::Tensor& res_, double p, const at::Tensor& rng, int64_t share) {
    at::AutoDispatchBelowADInplaceOrView below;
    c10::DeviceGuard guard(x_.device());
    int64_t ldx = 0, ldr = 0;
    const at::Tensor x = as_rows(x_, ldx), res = res_.defined() ? as_rows(res_, ldr) : res_;
    at::Tensor y = at::empty(x.sizes(), x.options());
    if (y.numel() == 0) return y;
    const int rc = entry.drop(at_of(x), ldx, at_of(res), ldr, dtype_of(x), lead_of(x.sizes()), x.size(-1), share, p,
                            (const int64_t*)at_of(rng), at_of(y), stream_of(x));
    TORCH_CHECK(rc == 0, "psfm_dropout failed (", rc, "): ", entry.drop_error());
    return y;
}

struct DropoutBackward : public torch::autograd::Node {
    SavedVariable rng;
    at::DimVector rshape;
    double p = 0;
    int64_t share = 1;
    Live live;

    std::string name() const override { return "DropoutBackward"; }
    void release_variables() override { rng.reset_data(); }

    variable_list apply(variable_list&& grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        refuse_foreign_capture();
        live.ran_backward();
        variable_list out(2);
        const at::Tensor& dy = grads[0];
        if (!dy.defined()) return out;
        const at::Tensor r = dense(unpacked(rng, shared_from_this(), rshape, at::kLong, dy.device(), "dropout: rng"));
        if (task_should_compute_output(0)) out[0] = once(drop_launch(dy, at::Tensor(), p, r, share), "dropout");
        if (task_should_compute_output(1)) out[1] = dy;
        return out;
    }
};

at::Tensor dropout(const at::Tensor& x, const std::optional<at::Tensor>& residual, double p, const at::Tensor& rng,
                   bool channels) {
    refuse_foreign_capture();
    const at::Tensor res = residual.value_or(at::Tensor());
    for (const at::Tensor* t : {&x, &res}) refuse_tangents(*t, "dropout");
    const int64_t share = mask_rows(x.sizes(), channels);
    std::shared_ptr<DropoutBackward> node;
    if (at::GradMode::is_enabled() && (wants(x) || wants(res))) {
        const bool in_capture = capturing();
        if (in_capture)
            for (const at::Tensor& t : {x, res}) refuse_bound_leaf(t);
        node = std::shared_ptr<DropoutBackward>(new DropoutBackward(), torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(x, res));
        c10::DeviceGuard guard(x.device());
        if (!in_capture) node->live.ran_forward((uintptr_t)stream_of(x));
    }
    at::Tensor y = drop_launch(x, res, p, rng, share);
    if (node) {
        node->p = p, node->share = share;
        node->rshape = at::DimVector(rng.sizes());
        node->rng = SavedVariable(rng, false);
        torch::autograd::set_history(y, node);
    }
    return y;
}

template <typename F>
void take(F& f, const py::dict& addresses, const char* name) {
    f = (F)addresses[name].cast<uintptr_t>();
}

}  // namespace

PYBIND11_MODULE(_psfm_autograd, m) {
    m.def("version", []() { return VERSION; });
    m.def("init", [](const py::dict& a, const py::object& refuse, int active) {
        take(entry.fwd_ws, a, "psfm_linear_fwd_ws_bytes");
        take(entry.fwd, a, "psfm_linear_fwd");
        take(entry.bwd_ws, a, "psfm_linear_bwd_ws_bytes");
        take(entry.bwd, a, "psfm_linear_bwd");
        take(entry.linear_error, a, "psfm_linear_last_error");
        take(entry.drop, a, "psfm_dropout");
        take(entry.drop_error, a, "psfm_dropout_last_error");
        refusal = py::object(refuse).release().ptr();
        captures = active;
    });
    m.def("set_captures", [](int n) { captures = n; });
    m.def("alive", &alive);
    m.def("linear_act", &linear_act);
    m.def("dropout", &dropout);
}
