// The feature operators as torch functions: checks have been made in Python, here tensors are laid out,
// results allocated, the C entry points of libta_b200.so called on the current stream, and autograd's
// nodes built - in C++, because a training step's backward pass runs in autograd's own thread, where Python code
// costs tens of microseconds per operator.  The library itself stays free of torch; this file is its client.
#include <dlfcn.h>

#include <mutex>

#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/extension.h>

#include "../../include/ta_b200.h"

namespace {

using at::Tensor;
using std::optional;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

// ----------------------------------------------------------------------------- the library
struct Api {
    decltype(&ta_b200_group_norm) group_norm, group_norm_backward;
    decltype(&ta_b200_group_norm_scratch_bytes) group_norm_scratch_bytes;
    decltype(&ta_b200_dropout) dropout;
    decltype(&ta_b200_rotary) rotary;
    decltype(&ta_b200_last_error) last_error;
} api;

PyObject *library_error = nullptr;      // _lib.LibraryError

struct LibraryError : std::runtime_error {
    using std::runtime_error::runtime_error;
};

void check(int rc, const char *what)
{
    if (rc != 0) throw LibraryError(std::string(what) + " failed with status " + std::to_string(rc) + ": " + api.last_error());
}

void bind(const std::string &path, const py::object &error)
{
    void *lib = dlopen(path.c_str(), RTLD_NOW);
    if (!lib) throw std::runtime_error(std::string("cannot load ") + path + ": " + dlerror());
    const auto find = [&](const char *name) {
        void *f = dlsym(lib, name);
        if (!f) throw std::runtime_error(path + " has no " + name);
        return f;
    };
    api.group_norm = (decltype(api.group_norm))find("ta_b200_group_norm");
    api.group_norm_backward = (decltype(api.group_norm_backward))find("ta_b200_group_norm_backward");
    api.group_norm_scratch_bytes = (decltype(api.group_norm_scratch_bytes))find("ta_b200_group_norm_scratch_bytes");
    api.dropout = (decltype(api.dropout))find("ta_b200_dropout");
    api.rotary = (decltype(api.rotary))find("ta_b200_rotary");
    api.last_error = (decltype(api.last_error))find("ta_b200_last_error");
    library_error = error.inc_ref().ptr();
}

void *stream_of(const Tensor &t) { return at::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

// ----------------------------------------------------------------------------- common
int code_of(at::ScalarType t) { return t == at::kFloat ? TA_B200_F32 : t == at::kHalf ? TA_B200_F16 : TA_B200_BF16; }

void *address(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }

Tensor given(const optional<Tensor> &t) { return t.has_value() ? *t : Tensor(); }

// `t` with its values in memory: a view of a conjugate's imaginary part holds them negated
Tensor stored(const Tensor &t) { return t.defined() && t.is_neg() ? t.resolve_neg() : t; }

// `t` with its channels (dimension -3) last in memory and no gaps; `t` itself if it is already
Tensor channels_last(const Tensor &given)
{
    const Tensor t = stored(given);
    if (t.dim() == 4) return t.contiguous(at::MemoryFormat::ChannelsLast);
    const Tensor last = t.movedim(-3, -1);
    return last.is_contiguous() ? t : last.contiguous().movedim(-1, -3);
}

bool wants_grad(std::initializer_list<const Tensor *> ts)
{
    for (const Tensor *t : ts)
        if (t->defined() && t->_fw_grad(0).defined()) throw py::value_error("forward-mode derivatives are not supported");
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor *t : ts)
        if (t->defined() && t->requires_grad()) return true;
    return false;
}

// Gradients that were asked for as part of a graph (create_graph) raise when they are differentiated: these
// operators have no second derivative.
variable_list once_differentiable(variable_list grads, const char *name)
{
    if (!at::GradMode::is_enabled()) return grads;
    auto error = std::make_shared<torch::autograd::DelayedError>(std::string(name) + " can be differentiated once only", (int64_t)grads.size());
    variable_list inputs;
    for (const Tensor &g : grads) inputs.push_back(g.defined() ? g.detach().requires_grad_() : g);
    return (*error)(std::move(inputs));
}

// ----------------------------------------------------------------------------- group norm
struct GroupNormCall {
    int64_t groups, samples;
    double eps;
    int act;
};

ta_b200_group_norm_params group_norm_params(const GroupNormCall &c, const Tensor &x, const Tensor &weight, const Tensor &bias, const Tensor &stats)
{
    ta_b200_group_norm_params p = {};
    p.struct_size = sizeof(p);
    p.dtype = code_of(x.scalar_type());
    const Tensor &param = weight.defined() ? weight : bias;
    p.param_dtype = param.defined() ? code_of(param.scalar_type()) : TA_B200_F32;
    p.activation = c.act;
    p.channels = (int32_t)x.size(-3);
    p.n = c.samples;
    p.rows = c.samples ? x.numel() / (c.samples * p.channels) : 0;
    p.groups = (int32_t)c.groups;
    p.eps = (float)c.eps;
    p.x = address(x);
    p.weight = address(weight);
    p.bias = address(bias);
    p.mean = (float *)address(stats);
    p.rstd = p.mean + c.samples * c.groups;
    return p;
}

void group_norm_call(ta_b200_group_norm_params &p, const Tensor &x, bool backward)
{
    const size_t need = api.group_norm_scratch_bytes(&p, backward);
    Tensor scratch;                     // stream-ordered: may be released after the launch
    if (need) {
        scratch = at::empty({(int64_t)need}, x.options().dtype(at::kByte));
        p.scratch = scratch.data_ptr();
        p.scratch_bytes = need;
    }
    if (backward) check(api.group_norm_backward(&p, stream_of(x)), "ta_b200_group_norm_backward");
    else check(api.group_norm(&p, stream_of(x)), "ta_b200_group_norm");
}

struct GroupNormBackward : Node {
    SavedVariable x, weight, bias, stats;
    GroupNormCall call;

    variable_list apply(variable_list &&grads) override
    {
        const std::lock_guard<std::mutex> lock(mutex_);        // two threads may go backward through one graph
        const Tensor &dy0 = grads[0];
        variable_list out(3);
        if (!dy0.defined()) return out;
        {
            at::AutoGradMode off(false);
            const Tensor xs = x.unpack(), w = weight.unpack(), b = bias.unpack(), st = stats.unpack(), dy = channels_last(dy0);
            const c10::cuda::OptionalCUDAGuard guard(xs.device());
            if (task_should_compute_output(0)) out[0] = at::empty_like(xs);
            if (w.defined() && task_should_compute_output(1)) out[1] = at::empty_like(w);
            if (b.defined() && task_should_compute_output(2)) out[2] = at::empty_like(b);
            ta_b200_group_norm_params p = group_norm_params(call, xs, w, b, st);
            p.dy = address(dy);
            p.dx = address(out[0]);
            p.dweight = address(out[1]);
            p.dbias = address(out[2]);
            group_norm_call(p, xs, true);
        }
        return once_differentiable(std::move(out), "group_norm");
    }
    void release_variables() override
    {
        const std::lock_guard<std::mutex> lock(mutex_);
        x.reset_data();
        weight.reset_data();
        bias.reset_data();
        stats.reset_data();
    }
    std::string name() const override { return "TaGroupNormBackward"; }
};

Tensor group_norm(const Tensor &x0, const optional<Tensor> &weight0, const optional<Tensor> &bias0, int64_t groups, double eps, int act, int64_t samples)
{
    const Tensor weight = given(weight0), bias = given(bias0);
    const c10::cuda::OptionalCUDAGuard guard(x0.device());
    const bool grad = wants_grad({&x0, &weight, &bias});
    const GroupNormCall call = {groups, samples, eps, act};
    Tensor x, w, b, y, stats;
    {
        at::AutoGradMode off(false);
        x = channels_last(x0);
        w = weight.defined() ? stored(weight).contiguous() : weight;
        b = bias.defined() ? stored(bias).contiguous() : bias;
        y = at::empty_like(x);
        stats = at::empty({2 * samples * groups}, x.options().dtype(at::kFloat));
        ta_b200_group_norm_params p = group_norm_params(call, x, w, b, stats);
        p.y = address(y);
        group_norm_call(p, x, false);
    }
    if (grad) {
        std::shared_ptr<GroupNormBackward> node(new GroupNormBackward(), torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(x0, weight, bias));
        node->x = SavedVariable(x, false);
        node->weight = SavedVariable(w, false);
        node->bias = SavedVariable(b, false);
        node->stats = SavedVariable(stats, false);
        node->call = call;
        torch::autograd::set_history(y, node);
    }
    return y;
}

// ----------------------------------------------------------------------------- dropout
struct DropoutCall {
    double p;
    uint64_t seed;
    uint32_t offset, shared;
    int64_t sizes[4];
    bool last;                          // channels last in memory
};

Tensor in_order(const Tensor &t, bool last) { return last ? channels_last(t) : stored(t).contiguous(); }

Tensor dropout_call(const DropoutCall &c, const Tensor &x, const Tensor &residual, const Tensor &seed)
{
    Tensor y = at::empty_like(x);
    ta_b200_dropout_params a = {};
    a.struct_size = sizeof(a);
    a.dtype = code_of(x.scalar_type());
    for (int d = 0; d < 4; ++d) a.sizes[d] = c.sizes[d];
    a.shared = c.shared;
    a.offset = c.offset;
    a.p = c.p;
    a.seed = c.seed;
    a.seed_ptr = (const uint64_t *)address(seed);
    a.x = address(x);
    a.residual = address(residual);
    a.y = address(y);
    check(api.dropout(&a, stream_of(x)), "ta_b200_dropout");
    return y;
}

struct DropoutBackward : Node {
    SavedVariable seed;
    DropoutCall call;

    variable_list apply(variable_list &&grads) override
    {
        const std::lock_guard<std::mutex> lock(mutex_);        // two threads may go backward through one graph
        variable_list out(2);
        if (!grads[0].defined()) return out;
        if (task_should_compute_output(1)) out[1] = grads[0];
        if (task_should_compute_output(0)) {
            at::AutoGradMode off(false);
            const c10::cuda::OptionalCUDAGuard guard(grads[0].device());
            out[0] = dropout_call(call, in_order(grads[0], call.last), Tensor(), seed.unpack());
        }
        return once_differentiable(std::move(out), "dropout");
    }
    void release_variables() override
    {
        const std::lock_guard<std::mutex> lock(mutex_);
        seed.reset_data();
    }
    std::string name() const override { return "TaDropoutBackward"; }
};

// layout: the four sizes of x in memory order, the bits of those the mask is shared along, channels last
Tensor dropout(const Tensor &x0, const optional<Tensor> &residual0, double p, uint64_t seed, const optional<Tensor> &seed_tensor0, uint32_t offset,
               int mode, bool same_on_batch, bool same_on_frame, const py::function &layout)
{
    const Tensor residual = given(residual0), seed_tensor = given(seed_tensor0);
    const c10::cuda::OptionalCUDAGuard guard(x0.device());
    const bool grad = wants_grad({&x0, &residual});
    DropoutCall call = {p, seed, offset, 0, {1, 1, 1, x0.numel()}, false};
    Tensor y;
    {
        at::AutoGradMode off(false);
        Tensor x = stored(x0);
        if (!x.is_contiguous()) {
            call.last = x.dim() >= 3 && x.dim() <= 5 && x.movedim(-3, -1).is_contiguous();
            if (!call.last) x = x.contiguous();
        }
        if (mode != 0 || same_on_batch || same_on_frame) {
            const py::tuple l = layout(py::cast(x.sizes().vec()), call.last, mode, same_on_batch, same_on_frame);
            const py::tuple sizes = l[0];
            for (int d = 0; d < 4; ++d) call.sizes[d] = sizes[d].cast<int64_t>();
            call.shared = l[1].cast<uint32_t>();
        }
        y = dropout_call(call, x, residual.defined() ? in_order(residual, call.last) : residual, seed_tensor);
    }
    if (grad) {
        std::shared_ptr<DropoutBackward> node(new DropoutBackward(), torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(x0, residual));
        node->seed = SavedVariable(seed_tensor, false);
        node->call = call;
        torch::autograd::set_history(y, node);
    }
    return y;
}

// ----------------------------------------------------------------------------- rotary positions
struct RotaryCall {
    ta_b200_rotary_params base;         // what does not depend on the tensors
};

// One launch on q and k, either of which may be undefined; the results have their layouts
variable_list rotary_call(const RotaryCall &c, const Tensor &q, const Tensor &k, const Tensor &positions, const Tensor &top, const Tensor &left,
                          const Tensor &flip, bool inverse)
{
    const Tensor &first = q.defined() ? q : k;
    ta_b200_rotary_params a = c.base;
    a.dtype = code_of(first.scalar_type());
    a.n = first.size(0);
    a.tokens = first.size(1);
    a.dim = (int32_t)first.size(3);
    a.inverse = inverse;
    if (positions.defined()) {
        a.position_kind = positions.scalar_type() == at::kLong ? TA_B200_POS_I64 : positions.scalar_type() == at::kFloat ? TA_B200_POS_F32 : TA_B200_POS_I32;
        a.positions = address(positions);
        const int64_t d = positions.dim();
        for (int i = 0; i < 3; ++i) a.position_strides[i] = i == 0 && d == 2 ? 0 : positions.stride(i - 3);
    }
    a.top = (const float *)address(top);
    a.left = (const float *)address(left);
    a.flip = (const uint8_t *)address(flip);
    variable_list out(2);
    Tensor dense[2];
    for (int which = 0; which < 2; ++which) {
        const Tensor &t = which ? k : q;
        if (!t.defined()) continue;
        dense[which] = t.stride(-1) == 1 || t.size(-1) == 1 ? stored(t) : stored(t).contiguous();
        out[which] = at::empty_like(dense[which]);
        if (out[which].stride(-1) != 1 && t.size(-1) != 1)      // an expanded input: its copy is laid out by size
            out[which] = at::empty(t.sizes(), t.options());
        (which ? a.k_heads : a.q_heads) = (int32_t)t.size(2);
        (which ? a.k : a.q) = address(dense[which]);
        (which ? a.k_out : a.q_out) = address(out[which]);
        for (int i = 0; i < 3; ++i) {
            (which ? a.k_strides : a.q_strides)[i] = dense[which].stride(i);
            (which ? a.k_out_strides : a.q_out_strides)[i] = out[which].stride(i);
        }
    }
    check(api.rotary(&a, stream_of(first)), "ta_b200_rotary");
    return out;
}

struct RotaryBackward : Node {
    SavedVariable positions, top, left, flip;
    RotaryCall call;

    variable_list apply(variable_list &&grads) override
    {
        const std::lock_guard<std::mutex> lock(mutex_);        // two threads may go backward through one graph
        variable_list out(2);
        const Tensor dq = task_should_compute_output(0) ? grads[0] : Tensor();
        const Tensor dk = grads.size() > 1 && task_should_compute_output(1) ? grads[1] : Tensor();
        if (dq.defined() || dk.defined()) {
            at::AutoGradMode off(false);
            const c10::cuda::OptionalCUDAGuard guard((dq.defined() ? dq : dk).device());
            out = rotary_call(call, dq, dk, positions.unpack(), top.unpack(), left.unpack(), flip.unpack(), true);
        }
        return once_differentiable(std::move(out), "rotary_embedding");
    }
    void release_variables() override
    {
        const std::lock_guard<std::mutex> lock(mutex_);
        positions.reset_data();
        top.reset_data();
        left.reset_data();
        flip.reset_data();
    }
    std::string name() const override { return "TaRotaryBackward"; }
};

py::capsule rotary_spec(std::vector<int> sections, int pairing, int spectrum, int prefix, double base, const optional<std::vector<int>> &grid, double patch)
{
    auto *c = new RotaryCall();
    ta_b200_rotary_params &a = c->base;
    a.struct_size = sizeof(a);
    a.prefix = prefix;
    a.axes = (int32_t)sections.size();
    for (size_t i = 0; i < sections.size() && i < 3; ++i) a.sections[i] = sections[i];
    a.pairing = pairing;
    a.spectrum = spectrum;
    a.base = base;
    a.position_kind = TA_B200_POS_GRID;
    if (grid.has_value())
        for (size_t i = 0; i < grid->size() && i < 3; ++i) a.grid[i] = (*grid)[i];
    a.patch = (float)patch;
    return py::capsule(c, [](void *p) { delete (RotaryCall *)p; });
}

py::object rotary(const Tensor &q, const optional<Tensor> &k0, const optional<Tensor> &positions0, const optional<Tensor> &top0, const optional<Tensor> &left0,
                  const optional<Tensor> &flip0, const py::capsule &spec)
{
    const Tensor k = given(k0), positions = stored(given(positions0)), top = given(top0), left = given(left0), flip = given(flip0);
    const c10::cuda::OptionalCUDAGuard guard(q.device());
    const RotaryCall &call = *spec.get_pointer<RotaryCall>();
    const bool grad = wants_grad({&q, &k});
    variable_list out;
    {
        at::AutoGradMode off(false);
        out = rotary_call(call, q, k, positions, top, left, flip, false);
    }
    if (grad) {
        std::shared_ptr<RotaryBackward> node(new RotaryBackward(), torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(q, k));
        node->positions = SavedVariable(positions, false);
        node->top = SavedVariable(top, false);
        node->left = SavedVariable(left, false);
        node->flip = SavedVariable(flip, false);
        node->call = call;
        if (k.defined()) torch::autograd::set_history(out, node);
        else torch::autograd::set_history(out[0], node);
    }
    if (!k.defined()) return py::cast(out[0]);
    return py::make_tuple(out[0], out[1]);
}

}  // namespace

PYBIND11_MODULE(_ta_torch, m)
{
    py::register_exception_translator([](std::exception_ptr p) {
        try {
            if (p) std::rethrow_exception(p);
        } catch (const LibraryError &e) {
            PyErr_SetString(library_error ? library_error : PyExc_RuntimeError, e.what());
        }
    });
    m.def("bind", &bind);
    m.def("group_norm", &group_norm);
    m.def("dropout", &dropout);
    m.def("rotary_spec", &rotary_spec);
    m.def("rotary", &rotary);
}
