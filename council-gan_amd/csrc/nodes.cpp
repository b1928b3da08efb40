// Autograd nodes of the channel-MLP operators: what a call does on the host, in C++.
//
// A training call of a few rows is over on the GPU in 10 to 40 us, while a Python autograd function spends 50 to 130 us on the host: its
// backward pass runs on the engine's own thread, often on another core complex, where every Python object it touches is a cache miss.
// These nodes check the arguments, allocate, and call the library; ops.py explains what was wrong when one of them declines.
// The library's entry points come in by address (`bind`), so that whichever build of it the process loaded is the one that runs.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/utils/pybind.h>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>

#include <array>
#include <memory>
#include <string>
#include <vector>

#include "../../include/council_gan_hip.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

namespace {

struct Api {
    decltype(&cg_last_error) last_error = nullptr;
    decltype(&cg_channel_norm_fwd) norm_fwd = nullptr;
    decltype(&cg_channel_norm_bwd_workspace) norm_bwd_ws = nullptr;
    decltype(&cg_channel_norm_bwd) norm_bwd = nullptr;
    decltype(&cg_dropout) dropout = nullptr;
    decltype(&cg_gated_ff_pack_bytes) gated_pack = nullptr;
    decltype(&cg_gated_ff_fwd_workspace) gated_fwd_ws = nullptr;
    decltype(&cg_gated_ff_fwd) gated_fwd = nullptr;
    decltype(&cg_gated_ff_bwd_workspace) gated_bwd_ws = nullptr;
    decltype(&cg_gated_ff_bwd) gated_bwd = nullptr;
} api;

void check(int rc, const char* what) { TORCH_CHECK(rc == 0, what, " failed (", rc, "): ", api.last_error()); }
cg_stream_t stream_of(const Tensor& t) { return (cg_stream_t)c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

int dt_of(at::ScalarType t) {
    return t == at::kFloat ? CG_DT_F32 : t == at::kHalf ? CG_DT_F16 : t == at::kBFloat16 ? CG_DT_BF16 : -1;
}
int64_t channels(const Tensor& x) { return x.dim() == 4 ? x.size(1) : x.dim() ? x.size(-1) : 0; }
// what a kernel reads: no gaps, and no sign kept as a bit beside the values (a view of a conjugate's imaginary part)
Tensor dense(const Tensor& v) {
    const Tensor t = v.is_neg() ? v.resolve_neg() : v;
    return t.dim() == 4 ? t.contiguous(at::MemoryFormat::ChannelsLast) : t.contiguous();
}
// the device memory of a tensor that may be undefined (no data_ptr of a tensor without storage is taken)
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
bool grad_on(const Tensor& t) { return t.defined() && t.requires_grad(); }
void once(const char* what) {
    TORCH_CHECK(!c10::GradMode::is_enabled(), what, ": the backward pass cannot be differentiated again");
}
// the operators have no forward-mode formulas: a tangent would be lost without a word
void refuse_tangents(const char* what, std::initializer_list<const Tensor*> inputs) {
    for (const Tensor* t : inputs)
        TORCH_CHECK(!t->defined() || !t->_fw_grad(0).defined(), what, ": forward-mode differentiation is not supported");
}
Tensor scratch(size_t bytes, const Tensor& like) {
    return bytes ? at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)) : Tensor();
}

// What a node saved, dense.  Saved-tensor hooks (activation checkpointing, offloading) may bring it back elsewhere and in another layout,
// but as the same values.
Tensor saved(const SavedVariable& s, const char* what, int64_t numel, at::ScalarType type, const at::Device& device) {
    const Tensor t = dense(s.unpack());
    TORCH_CHECK(t.numel() == numel && t.scalar_type() == type && t.device() == device, what, s.has_hooks() ?
                ": a saved tensor came back with another size, type or device" : ": an input changed its size since the forward pass");
    return t;
}
// t itself, or a copy, so far off 16 bytes as `was`: a product's operands have a copy in `pack` or not by that
Tensor placed(const Tensor& t, const void* was) {
    if (!t.numel() || (((uintptr_t)t.data_ptr() ^ (uintptr_t)was) & 15) == 0) return t;
    const int64_t off = ((uintptr_t)was & 15) / t.element_size();
    const Tensor c = at::empty({t.numel() + off}, t.options()).narrow(0, off, t.numel()).as_strided(t.sizes(), t.strides());
    return Tensor(c).copy_(t);
}

// the gradient buffer that a parameter's optimizer keeps (the parameter's _cg_grad), or nothing
struct Buffer {
    Tensor t;
    PyObject* obj = nullptr;
    Buffer() = default;
    explicit Buffer(const py::handle& h) {      // with the interpreter's lock held
        if (h.is_none()) return;
        obj = h.inc_ref().ptr();
        t = THPVariable_Unpack(obj);
    }
    Buffer(Buffer&& o) noexcept : t(std::move(o.t)), obj(o.obj) { o.obj = nullptr; }
    Buffer& operator=(Buffer&& o) noexcept {
        std::swap(t, o.t);
        std::swap(obj, o.obj);
        return *this;
    }
    Buffer(const Buffer&) = delete;
    ~Buffer() {
        if (!obj || !Py_IsInitialized()) return;
        py::gil_scoped_acquire lock;
        Py_DECREF(obj);
    }
    void touch() const {
        py::gil_scoped_acquire lock;
        if (PyObject_SetAttrString(obj, "_cg_touched", Py_True) != 0) PyErr_Clear();
    }
};

struct Target { Tensor out, ret, shared; bool add = false; };       // what the kernel writes, what the node returns
Target target(const Tensor& p, const Buffer& buf, bool wanted, int members) {
    Target r;
    if (!p.defined() || !wanted) return r;
    TORCH_CHECK(!buf.t.defined() || (buf.t.device() == p.device() && buf.t.sizes() == p.sizes()),
                "a parameter's gradient buffer is on another device, or has another shape: its optimizer was materialized before the parameter moved");
    if (buf.t.defined() && buf.t.scalar_type() == p.scalar_type() && buf.t.is_contiguous()) {
        buf.touch();
        r.out = buf.t;
        r.add = true;
        return r;
    }
    TORCH_CHECK(members == 1, "member-batched backward needs the pool's gradient buffers");
    r.out = r.ret = at::empty(p.sizes(), p.options());
    return r;
}

// Targets that share a buffer (a tensor that serves as two parameters): all but the first get memory of their own, since one launch may
// write them side by side; `settle` adds it to the buffer.
template <size_t N> void separate(std::array<Target, N>& t, int members) {
    for (size_t i = 1; i < N; ++i)
        for (size_t j = 0; j < i; ++j)
            if (t[i].add && t[j].out.defined() && t[i].out.data_ptr() == t[j].out.data_ptr()) {
                TORCH_CHECK(members == 1, "member-batched backward: one parameter is used twice in a call");
                t[i].shared = t[i].out;
                t[i].out = at::empty_like(t[i].shared);
                t[i].add = false;
                break;
            }
}
template <size_t N> void settle(const std::array<Target, N>& t) {
    for (const Target& x : t)
        if (x.shared.defined()) Tensor(x.shared).add_(x.out);
}

// A backward pass captured into a graph must not meet a gradient accumulator that an eager graph holds: it belongs to that graph's
// stream, which the engine would make wait for the capture, and the capture (or the process) ends with that.
void refuse_eager_graph(const char* what, std::initializer_list<std::pair<const Tensor*, const Buffer*>> leaves) {
    if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
    for (const auto& [t, buf] : leaves) {
        if (!grad_on(*t) || !t->is_leaf() || (buf && buf->t.defined())) continue;
        const auto acc = torch::autograd::impl::try_get_grad_accumulator(*t);
        if (!acc) continue;
        const auto st = acc->stream();
        TORCH_CHECK(!st || st->id() == c10::hip::getCurrentHIPStream(t->device().index()).id(), what,
                    ": captured while an eager graph of the same leaves lives: drop what it computed first");
    }
}

struct Members {
    cg_group g{1, 0, 0};
    const cg_group* get() const { return g.n > 1 ? &g : nullptr; }
};

template <typename N> std::shared_ptr<N> make_node() { return std::shared_ptr<N>(new N(), torch::autograd::deleteNode); }

// -- channel_norm ----------------------------------------------------------------------------------
constexpr int64_t MAX_CHANNELS = 1 << 29;       // as the library has it

struct ChannelNorm : public torch::autograd::Node {
    SavedVariable x_, w_, stats_;
    Tensor b_;
    size_t rows = 0, C = 0;
    at::ScalarType type{}, wtype{};
    c10::Device device{c10::kCUDA, 0};
    Members members;
    Buffer wbuf, bbuf;

    std::string name() const override { return "ChannelNorm"; }
    void release_variables() override {
        x_.reset_data();
        w_.reset_data();
        stats_.reset_data();
    }
    variable_list apply(variable_list&& grads) override {
        once("channel_norm");
        variable_list out(3);
        if (!grads[0].defined()) return out;
        const char* what = "channel_norm";
        const Tensor x = saved(x_, what, rows * C, type, device), w = saved(w_, what, C, wtype, device),
                     stats = saved(stats_, what, 2 * rows, at::kFloat, device), dy = dense(grads[0]);
        const bool need_w = task_should_compute_output(1), need_b = b_.defined() && task_should_compute_output(2);
        Tensor dx;
        if (task_should_compute_output(0)) out[0] = dx = at::empty_like(x);
        std::array<Target, 2> t{target(w, wbuf, need_w, members.g.n), target(b_, bbuf, need_b, members.g.n)};
        separate(t, members.g.n);
        const int dt = dt_of(x.scalar_type()), wdt = dt_of(w.scalar_type());
        const size_t nws = need_w || need_b ? api.norm_bwd_ws(members.get(), rows, (int)C, dt) : 0;
        const Tensor ws = scratch(nws, x);
        float* st = (float*)stats.data_ptr();
        check(api.norm_bwd(members.get(), ptr(dy), ptr(x), ptr(w), st, st + rows, ptr(dx), ptr(t[0].out), ptr(t[1].out), t[0].add | t[1].add << 1,
                           rows, (int)C, dt, wdt, ptr(ws), nws, stream_of(x)),
              "cg_channel_norm_bwd");
        settle(t);
        out[1] = t[0].ret;
        out[2] = t[1].ret;
        return out;
    }
};

py::object channel_norm(const Tensor& x, const Tensor& w, const std::optional<Tensor>& bias, double eps, int n, int64_t stride,
                        const py::object& wbuf, const py::object& bbuf) {
    const Tensor b = bias.value_or(Tensor());
    refuse_tangents("channel_norm", {&x, &w, &b});
    const int64_t C = channels(x);
    const int dt = dt_of(x.scalar_type()), wdt = dt_of(w.scalar_type());
    if (!x.is_cuda() || C < 1 || C > MAX_CHANNELS || dt < 0 || !(eps >= 0) || w.dim() != 1 || w.size(0) != C || w.device() != x.device() ||
        (wdt != dt && wdt != CG_DT_F32) ||
        (b.defined() && (b.dim() != 1 || b.size(0) != C || b.scalar_type() != w.scalar_type() || b.device() != x.device())))
        return py::none();
    const bool record = c10::GradMode::is_enabled() && (grad_on(x) || grad_on(w) || grad_on(b));
    std::shared_ptr<ChannelNorm> node;
    if (record) {
        node = make_node<ChannelNorm>();
        node->wbuf = Buffer(wbuf);
        node->bbuf = Buffer(bbuf);
    }
    Tensor y;
    {
        py::gil_scoped_release unlock;
        const c10::DeviceGuard device(x.device());
        Members members{{n, 0, stride}};
        Tensor xd, wd, bd, stats;
        const size_t rows = x.numel() / C;
        {
            const at::NoGradGuard plain;
            if (record) refuse_eager_graph("channel_norm", {{&x, nullptr}, {&w, &node->wbuf}, {&b, &node->bbuf}});
            xd = dense(x);
            wd = dense(w);
            if (b.defined()) bd = dense(b);
            y = at::empty_like(xd);
            if (record) stats = at::empty({2, (int64_t)rows}, x.options().dtype(at::kFloat));
            float* st = record ? (float*)stats.data_ptr() : nullptr;
            check(api.norm_fwd(members.get(), ptr(xd), ptr(wd), ptr(bd), ptr(y), st, record ? st + rows : nullptr, rows, (int)C, dt, wdt,
                               (float)eps, stream_of(x)),
                  "cg_channel_norm_fwd");
        }
        if (record) {
            node->set_next_edges(torch::autograd::collect_next_edges(x, w, b));
            node->x_ = SavedVariable(xd, false);
            node->w_ = SavedVariable(wd, false);
            node->b_ = bd.defined() ? bd.detach() : bd;
            node->stats_ = SavedVariable(stats, false);
            node->rows = rows, node->C = C, node->type = x.scalar_type(), node->wtype = w.scalar_type(), node->device = x.device();
            node->members = members;
            torch::autograd::set_history(y, node);
        }
    }
    return py::cast(y);
}

// -- dropout -----------------------------------------------------------------------------------------
struct Dropout : public torch::autograd::Node {
    SavedVariable key_;
    int threshold = 0;

    std::string name() const override { return "Dropout"; }
    void release_variables() override { key_.reset_data(); }
    variable_list apply(variable_list&& grads) override {
        once("dropout");
        variable_list out(2);
        if (!grads[0].defined()) return out;
        const Tensor key = saved(key_, "dropout", 2, at::kLong, grads[0].device());
        if (task_should_compute_output(0)) {
            const Tensor dy = dense(grads[0]);
            out[0] = at::empty_like(dy);
            check(api.dropout(ptr(dy), nullptr, ptr(out[0]), dy.numel(), threshold, ptr(key), dt_of(dy.scalar_type()), stream_of(dy)),
                  "cg_dropout");
        }
        if (task_should_compute_output(1)) out[1] = grads[0];
        return out;
    }
};

py::object dropout(const Tensor& x, const std::optional<Tensor>& residual, int threshold, const Tensor& key) {
    const Tensor res = residual.value_or(Tensor());
    refuse_tangents("dropout", {&x, &res});
    const int dt = dt_of(x.scalar_type());
    if (!x.is_cuda() || x.dim() < 1 || dt < 0 || key.scalar_type() != at::kLong || key.numel() != 2 || !key.is_contiguous() ||
        key.device() != x.device() ||
        (res.defined() && (res.sizes() != x.sizes() || res.scalar_type() != x.scalar_type() || res.device() != x.device())))
        return py::none();
    Tensor y;
    {
        py::gil_scoped_release unlock;
        const c10::DeviceGuard device(x.device());
        {
            const bool record = c10::GradMode::is_enabled();
            const at::NoGradGuard plain;
            if (record) refuse_eager_graph("dropout", {{&x, nullptr}, {&res, nullptr}});
            const Tensor xd = dense(x), rd = res.defined() ? dense(res) : res;
            y = at::empty_like(xd);
            check(api.dropout(ptr(xd), ptr(rd), ptr(y), xd.numel(), threshold, ptr(key), dt, stream_of(x)), "cg_dropout");
        }
        if (c10::GradMode::is_enabled() && (grad_on(x) || grad_on(res))) {
            auto node = make_node<Dropout>();
            node->set_next_edges(torch::autograd::collect_next_edges(x, res));
            node->key_ = SavedVariable(key, false);
            node->threshold = threshold;
            torch::autograd::set_history(y, node);
        }
    }
    return py::cast(y);
}

constexpr int64_t MAX_WIDTH = 1 << 21;       // as the library has it

// -- gated_feed_forward --------------------------------------------------------------------------------
struct Gated : public torch::autograd::Node {
    SavedVariable x_, wg_, wv_, wo_;
    SavedVariable h_, kept_, pack_;      // kept_: u and p; pack_: the forward pass's copies of operands that are not on 16 bytes
    int64_t kept_n = 0, pack_n = 0;
    std::array<Tensor, 3> biases;
    at::ScalarType type{};
    c10::Device device{c10::kCUDA, 0};
    cg_gated_dims dims{};
    Members members;
    std::array<Buffer, 6> bufs;
    std::array<void*, 4> read{};      // x, wg, wv, wo as the forward pass read them

    std::string name() const override { return "GatedFeedForward"; }
    void release_variables() override {
        x_.reset_data();
        wg_.reset_data();
        wv_.reset_data();
        wo_.reset_data();
        h_.reset_data();
        kept_.reset_data();
        pack_.reset_data();
    }
    variable_list apply(variable_list&& grads) override {
        once("gated_feed_forward");
        variable_list out(7);
        if (!grads[0].defined()) return out;
        const char* what = "gated_feed_forward";
        const int64_t D = dims.D, F = dims.F, O = dims.O;
        auto operand = [&](const SavedVariable& s, int i, int64_t numel) {
            const Tensor t = saved(s, what, numel, type, device);
            TORCH_CHECK(s.has_hooks() || ptr(t) == read[i], what, ": an operand moved since the forward pass");
            return placed(t, read[i]);
        };
        auto own = [&](const SavedVariable& s, int64_t numel, at::ScalarType as) {
            return numel ? placed(saved(s, what, numel, as, device), nullptr) : Tensor();
        };
        const Tensor x = operand(x_, 0, dims.rows * D), dy = dense(grads[0]);
        const std::array<Tensor, 6> p{operand(wg_, 1, F * D), operand(wv_, 2, F * D), O ? operand(wo_, 3, O * F) : Tensor(),
                                      biases[0], biases[1], biases[2]};
        const int64_t pitch = (F + 7) & ~(int64_t)7;
        const Tensor h = own(h_, O ? dims.rows * pitch : 0, type), kept = own(kept_, kept_n, type), pack = own(pack_, pack_n, at::kByte);
        Tensor dx;
        if (task_should_compute_output(0)) out[0] = dx = at::empty_like(x);
        std::array<void*, 6> to;
        int add = 0;
        std::array<Target, 6> t;
        for (int i = 0; i < 6; ++i) {
            t[i] = target(p[i], bufs[i], task_should_compute_output(1 + i), members.g.n);
            out[1 + i] = t[i].ret;
        }
        separate(t, members.g.n);
        for (int i = 0; i < 6; ++i) {
            to[i] = ptr(t[i].out);
            add |= t[i].add << i;
        }
        const size_t nws = api.gated_bwd_ws(&dims, members.get());
        const Tensor ws = scratch(nws, x);
        check(api.gated_bwd(&dims, members.get(), ptr(dy), ptr(x), ptr(p[0]), ptr(p[1]), ptr(p[2]), ptr(h), ptr(kept), ptr(dx), to[0], to[1], to[2],
                            to[3], to[4], to[5], add, ptr(pack), ptr(ws), nws, stream_of(x)),
              "cg_gated_ff_bwd");
        settle(t);
        return out;
    }
};

py::object gated(const Tensor& x, const Tensor& wg, const Tensor& wv, const std::optional<Tensor>& w_out, const std::optional<Tensor>& b_gate,
                 const std::optional<Tensor>& b_value, const std::optional<Tensor>& b_out, int gate, int n, int64_t stride,
                 const py::object& bufs) {
    const Tensor none;
    const Tensor wo = w_out.value_or(none);
    const std::array<Tensor, 3> b{b_gate.value_or(none), b_value.value_or(none), b_out.value_or(none)};
    refuse_tangents("gated_feed_forward", {&x, &wg, &wv, &wo, &b[0], &b[1], &b[2]});
    const int dt = dt_of(x.scalar_type());
    auto like = [&](const Tensor& t) { return t.scalar_type() == x.scalar_type() && t.device() == x.device(); };
    if (!x.is_cuda() || dt < 0 || gate < 0 || wg.dim() != 2 || wv.dim() != 2 || wg.sizes() != wv.sizes() || !like(wg) || !like(wv) ||
        channels(x) != wg.size(1) || wg.size(0) < 1 || wg.size(1) < 1 || wg.size(0) > MAX_WIDTH || wg.size(1) > MAX_WIDTH ||
        x.numel() / wg.size(1) > 1 << 30)
        return py::none();
    const int64_t F = wg.size(0), D = wg.size(1);
    if (wo.defined() && (wo.dim() != 2 || wo.size(1) != F || wo.size(0) < 1 || wo.size(0) > MAX_WIDTH || !like(wo))) return py::none();
    const int64_t O = wo.defined() ? wo.size(0) : 0;
    for (int i = 0; i < 3; ++i)
        if (b[i].defined() && (b[i].dim() != 1 || b[i].size(0) != (i < 2 ? F : O) || !like(b[i]) || (i == 2 && !O))) return py::none();
    const bool record = c10::GradMode::is_enabled() && (grad_on(x) || grad_on(wg) || grad_on(wv) || grad_on(wo) || grad_on(b[0]) ||
                                                        grad_on(b[1]) || grad_on(b[2]));
    std::shared_ptr<Gated> node;
    if (record) {
        node = make_node<Gated>();
        if (!bufs.is_none()) {
            int i = 0;
            for (const py::handle& o : py::cast<py::tuple>(bufs)) node->bufs[i++] = Buffer(o);
        }
    }
    Tensor y;
    {
        py::gil_scoped_release unlock;
        const c10::DeviceGuard device(x.device());
        Members members{{n, 0, stride}};
        Tensor xd, h, kept, pack;
        std::array<Tensor, 6> p{wg, wv, wo, b[0], b[1], b[2]};
        const int64_t rows = x.numel() / D;
        cg_gated_dims dims{rows, (int32_t)D, (int32_t)F, (int32_t)O, dt, gate, 0};
        {
            const at::NoGradGuard plain;
            if (record)
                refuse_eager_graph("gated_feed_forward", {{&x, nullptr}, {&wg, &node->bufs[0]}, {&wv, &node->bufs[1]}, {&wo, &node->bufs[2]},
                                                          {&b[0], &node->bufs[3]}, {&b[1], &node->bufs[4]}, {&b[2], &node->bufs[5]}});
            xd = dense(x);
            for (Tensor& t : p)
                if (t.defined()) t = dense(t);
            auto rows_like = [&](int64_t c) {
                std::vector<int64_t> s = x.sizes().vec();
                s[x.dim() == 4 ? 1 : x.dim() - 1] = c;
                return x.dim() == 4 ? at::empty(s, x.options(), at::MemoryFormat::ChannelsLast) : at::empty(s, x.options());
            };
            const int64_t pitch = (F + 7) & ~(int64_t)7;
            h = O ? at::empty({rows, pitch}, x.options()) : rows_like(F);
            if (O) y = rows_like(O);
            if (record) kept = at::empty({dt == CG_DT_F32 ? 2 : 3, rows, pitch}, x.options());
            pack = scratch(api.gated_pack(&dims, members.get(), ptr(xd), ptr(p[0]), ptr(p[1]), ptr(p[2])), x);
            const size_t nws = api.gated_fwd_ws(&dims, members.get());
            const Tensor ws = scratch(nws, x);
            check(api.gated_fwd(&dims, members.get(), ptr(xd), ptr(p[0]), ptr(p[1]), ptr(p[2]), ptr(p[3]), ptr(p[4]), ptr(p[5]), ptr(h), ptr(kept),
                                ptr(y), ptr(pack), ptr(ws), nws, stream_of(x)),
                  "cg_gated_ff_fwd");
        }
        if (record) {
            node->set_next_edges(torch::autograd::collect_next_edges(x, wg, wv, wo, b[0], b[1], b[2]));
            node->x_ = SavedVariable(xd, false);
            node->wg_ = SavedVariable(p[0], false);
            node->wv_ = SavedVariable(p[1], false);
            if (O) {
                node->wo_ = SavedVariable(p[2], false);
                node->h_ = SavedVariable(h, false);
            }
            for (int i = 0; i < 3; ++i)
                if (p[3 + i].defined()) node->biases[i] = p[3 + i].detach();
            node->kept_ = SavedVariable(kept, false);
            node->kept_n = kept.numel();
            if (pack.defined()) node->pack_ = SavedVariable(pack, false), node->pack_n = pack.numel();
            node->type = x.scalar_type(), node->device = x.device();
            node->dims = dims;
            node->members = members;
            node->read = {ptr(xd), ptr(p[0]), ptr(p[1]), ptr(p[2])};
            if (!O) y = h;
            torch::autograd::set_history(y, node);
        } else if (!O) {
            y = h;
        }
    }
    return py::cast(y);
}

void bind(const py::dict& d) {
    auto at = [&](const char* name) { return (void*)d[name].cast<size_t>(); };
#define CG_BIND(member, fn) api.member = (decltype(api.member))at(#fn)
    CG_BIND(last_error, cg_last_error);
    CG_BIND(norm_fwd, cg_channel_norm_fwd);
    CG_BIND(norm_bwd_ws, cg_channel_norm_bwd_workspace);
    CG_BIND(norm_bwd, cg_channel_norm_bwd);
    CG_BIND(dropout, cg_dropout);
    CG_BIND(gated_pack, cg_gated_ff_pack_bytes);
    CG_BIND(gated_fwd_ws, cg_gated_ff_fwd_workspace);
    CG_BIND(gated_fwd, cg_gated_ff_fwd);
    CG_BIND(gated_bwd_ws, cg_gated_ff_bwd_workspace);
    CG_BIND(gated_bwd, cg_gated_ff_bwd);
#undef CG_BIND
}

}  // namespace

PYBIND11_MODULE(cg_nodes, m) {
    m.def("bind", &bind);
    // None: the arguments do not fit (ops.py says which).  Wrapped: exceptions of saved-tensor hooks pass through as they are.
    m.def("channel_norm", torch::wrap_pybind_function(channel_norm));
    m.def("dropout", torch::wrap_pybind_function(dropout));
    m.def("gated", torch::wrap_pybind_function(gated));
}
