// Host side of the autograd front-end: argument checks, output allocation, graph nodes and the calls into the C ABI
// (include/sortdist.h), one C++ function per op of sortnet_amd/functional.py.
//
// Why native: a small layer (128 x 3072 x 1024) keeps the device busy for 50 us per forward and backward, and the same
// calls made from Python (autograd.Function, a device context, a dozen checked ctypes arguments per entry point, the
// backward once more through the interpreter) took 120 us of host time, so the host set the pace.  Here a call
// is a few tensor headers, one graph node and the launches; the backward runs on autograd's own thread without the
// interpreter.  Tensors stay torch's: outputs come from its caching allocator and work is queued on its current
// stream.
#include <array>
#include <cmath>
#include <mutex>
#include <stdexcept>
#include <string>

#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/utils/pybind.h>

#include "../../include/sortdist.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::collect_next_edges;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::set_history;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

namespace {

// ---- arguments --------------------------------------------------------------------------------------------------
template <class T>
T* data(const Tensor& t, const char* name, at::ScalarType type) {
    if (!t.is_cuda()) throw std::runtime_error(std::string(name) + " must be a CUDA tensor");
    if (!t.is_contiguous()) throw std::runtime_error(std::string(name) + " must be contiguous");
    if (t.scalar_type() != type)
        throw std::runtime_error(std::string(name) + " must have dtype " + (type == at::kFloat ? "torch.float32" : "torch.int32"));
    return static_cast<T*>(t.data_ptr());
}
float* floats(const Tensor& t, const char* name) { return data<float>(t, name, at::kFloat); }
int* ints(const Tensor& t, const char* name) { return data<int>(t, name, at::kInt); }
int* ints(const OptTensor& t, const char* name) { return t && t->defined() ? ints(*t, name) : nullptr; }

void require(int rc, const char* who) {
    if (rc == 0) return;
    const char* msg = sd_last_error();
    throw std::runtime_error(std::string(who) + " failed (status " + std::to_string(rc) + "): " + (msg ? msg : "?"));
}

// torch's current stream on t's GPU (queried while the arguments of an entry point are formed, perhaps before t is checked)
sd_stream_t stream_of(const Tensor& t) {
    if (!t.is_cuda()) throw std::runtime_error("input must be a CUDA tensor");
    return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

// the graph capture that work on this stream goes into: its number, 0 for none, -1 where the runtime does not say
int64_t capture_of(sd_stream_t stream) {
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    unsigned long long id = 0;
    if (hipStreamGetCaptureInfo(static_cast<hipStream_t>(stream), &status, &id) != hipSuccess) { (void)hipGetLastError(); return -1; }
    return status == hipStreamCaptureStatusNone ? 0 : status == hipStreamCaptureStatusActive ? (int64_t)id : -1;
}

// sizes of a layer call on x (B, C, HW)
struct Dims {
    int B, CI, HW, CO, G;
    Dims(const Tensor& x, int64_t groups, int64_t channels)
        : B((int)x.size(0)), CI((int)x.size(1)), HW((int)x.size(2)), CO((int)channels), G((int)groups) {}
};

Tensor new_floats(const Tensor& like, at::IntArrayRef size) { return at::empty(size, like.options().dtype(at::kFloat)); }
Tensor new_ints(const Tensor& like, at::IntArrayRef size) { return at::empty(size, like.options().dtype(at::kInt)); }
Tensor new_out(const Tensor& x, int64_t channels) { return new_floats(x, {x.size(0), channels, x.size(2)}); }

// The nodes below hold backward formulas and nothing else.  An input with a forward-mode tangent would come out without
// one, which a caller reads as a zero derivative, and the kernels know nothing of the wrapped tensors of torch.func: both
// are refused, as an autograd function without `jvp` and `setup_context` refuses them.
template <class... T>
void reverse_mode_only(const char* who, const T&... t) {
    if (c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchDynamicLayerFrontMode))   // inside a transform
        throw std::runtime_error(std::string("sortnet_amd.") + who + " does not support the transforms of torch.func (vmap, grad, jvp, ...)");
    TORCH_CHECK_NOT_IMPLEMENTED(!(... || (t.defined() && t._fw_grad(0).defined())),
                                "sortnet_amd.", who, " does not support forward mode AD: an input carries a tangent");
}

template <class... T>
bool want_grad(const T&... t) { return at::GradMode::is_enabled() && (t.requires_grad() || ...); }

// Every node takes its mutex_ while it reads or frees what it saved: two threads may run backward through a graph that they
// share.  Saved tensors are unpacked before autograd is switched off, since the caller's unpack hooks run inside.
using Locked = std::lock_guard<std::mutex>;

// The gradient that flows into output `i` of a node, zeros where none does (an op behind it that has no gradient to give):
// the inputs then get zeros and not nothing.
Tensor incoming(const Node& node, const variable_list& grads, int i) {
    return grads[i].defined() ? grads[i].contiguous() : node.input_metadata(i).zeros_like();
}

template <class N>
std::shared_ptr<N> new_node() { return std::shared_ptr<N>(new N(), torch::autograd::deleteNode); }

// ---- l-inf, masked and l-p layers: x, weight -> y -----------------------------------------------------------------
// A node has two edges, x and weight; `kind` names the backward entry points.
struct DistNode : Node {
    enum Kind { MAX, SORT, POWER } kind;
    SavedVariable x, weight, state;            // state: positions (MAX, SORT) or the output (POWER)
    SavedVariable ci, co;
    int groups, truncate = 0;
    double p = 0, q = 0;

    variable_list apply(variable_list&& grads) override {
        const Locked lock(mutex_);
        variable_list out(2);
        const bool want_w = task_should_compute_output(1), want_x = task_should_compute_output(0);
        if (!want_w && !want_x) return out;
        const Tensor xs = x.unpack(), ws = weight.unpack(), st = state.unpack(shared_from_this());
        const Tensor cis = ci.unpack(), cos = co.unpack();
        at::AutoDispatchBelowADInplaceOrView below;
        const Tensor g = incoming(*this, grads, 0);
        const c10::DeviceGuard guard(g.device());
        const int B = (int)g.size(0), CO = (int)g.size(1), HW = (int)g.size(2), CI = (int)xs.size(1), G = groups;
        const int W_CO = (int)ws.size(0), W_CI = (int)ws.size(1) * G;
        Tensor gx = at::empty(xs.sizes(), xs.options()), gw;
        const float* gp = floats(g, "grad_output");
        const int *cip = cis.defined() ? ints(cis, "w_index_ci") : nullptr, *cop = cos.defined() ? ints(cos, "w_index_co") : nullptr;
        const sd_stream_t s = stream_of(g);
        if (want_w) gw = at::empty(ws.sizes(), ws.options());
        float *gxp = floats(gx, "grad_input"), *gwp = want_w ? floats(gw, "grad_weight") : nullptr;
        if (kind == MAX) {
            const int* pos = ints(st, "pos");
            if (want_w) require(sd_inf_dist_backward_input_weight(gp, pos, B, CO, CI, G, HW, gxp, gwp, cip, cop, W_CO, W_CI, s),
                                "sd_inf_dist_backward_input_weight");
            else require(sd_inf_dist_backward_input(gp, pos, B, CO, CI, G, HW, gxp, s), "sd_inf_dist_backward_input");
        } else if (kind == SORT) {
            const int* pos = ints(st, "pos");
            if (want_w) require(sd_sort_neuron_backward_input_weight(gp, pos, B, CO, CI, G, HW, gxp, gwp, (float)q, truncate, s),
                                "sd_sort_neuron_backward_input_weight");
            else require(sd_sort_neuron_backward_input(gp, pos, B, CO, CI, G, HW, gxp, (float)q, truncate, s),
                         "sd_sort_neuron_backward_input");
        } else {
            const float *xp = floats(xs, "input"), *wp = floats(ws, "weight"), *yp = floats(st, "output");
            if (want_w) require(sd_norm_dist_backward_input_weight(gp, xp, wp, yp, B, CO, CI, G, HW, gxp, gwp, (float)p, cip, cop,
                                                                   W_CO, W_CI, s), "sd_norm_dist_backward_input_weight");
            else require(sd_norm_dist_backward_input(gp, xp, wp, yp, B, CO, CI, G, HW, gxp, (float)p, cip, cop, W_CO, W_CI, s),
                         "sd_norm_dist_backward_input");
        }
        if (want_x) out[0] = gx;
        if (want_w) out[1] = gw;
        return out;
    }
    void release_variables() override {
        const Locked lock(mutex_);
        x.reset_data(); weight.reset_data(); state.reset_data(); ci.reset_data(); co.reset_data();
    }
    std::string name() const override { return "DistNode"; }
};

// makes y the output of a node over (x, weight); the caller adds what its kind needs
std::shared_ptr<DistNode> attach(const Tensor& x, const Tensor& w, int64_t groups, DistNode::Kind kind) {
    auto node = new_node<DistNode>();
    node->set_next_edges(collect_next_edges(x, w));
    node->kind = kind;
    node->groups = (int)groups;
    node->x = SavedVariable(x, false);
    node->weight = SavedVariable(w, false);
    return node;
}

Tensor norm_dist_lists(const Tensor& x, const Tensor& w, const OptTensor& ci, const OptTensor& co, int64_t groups, double p,
                       bool lists) {
    reverse_mode_only("norm_dist", x, w);
    const bool grad = want_grad(x, w);
    const int64_t channels = co && co->defined() ? co->size(-1) * groups : w.size(0);
    Tensor y, pos;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        const c10::DeviceGuard guard(x.device());
        y = new_out(x, channels);
        const Dims d(x, groups, channels);
        const float *xp = floats(x, "input"), *wp = floats(w, "weight");
        const int *cip = ints(ci, "w_index_ci"), *cop = ints(co, "w_index_co");
        const int W_CO = (int)w.size(0), W_CI = (int)(w.size(1) * groups);
        if (std::isinf(p)) {
            if (grad || lists) {
                pos = new_ints(x, y.sizes());
                require(sd_inf_dist_forward(xp, wp, d.B, d.CO, d.CI, d.G, d.HW, floats(y, "output"), ints(pos, "pos"), cip, cop,
                                            W_CO, W_CI, stream_of(x)), "sd_inf_dist_forward");
            } else
                require(sd_inf_dist_forward_nograd(xp, wp, d.B, d.CO, d.CI, d.G, d.HW, floats(y, "output"), stream_of(x)),
                        "sd_inf_dist_forward_nograd");
        } else
            require(sd_norm_dist_forward(xp, wp, d.B, d.CO, d.CI, d.G, d.HW, floats(y, "output"), (float)p, cip, cop, W_CO, W_CI,
                                         stream_of(x)), "sd_norm_dist_forward");
    }
    if (grad) {
        const bool power = !std::isinf(p);
        auto node = attach(x, w, groups, power ? DistNode::POWER : DistNode::MAX);
        node->p = p;
        if (ci && ci->defined()) node->ci = SavedVariable(*ci, false);
        if (co && co->defined()) node->co = SavedVariable(*co, false);
        set_history(y, node);
        node->state = power ? SavedVariable(y, true) : SavedVariable(pos, false);
    }
    return y;
}

Tensor norm_dist(const Tensor& x, const Tensor& w, int64_t groups, double p) {
    return norm_dist_lists(x, w, {}, {}, groups, p, false);
}
Tensor norm_dist_dropout(const Tensor& x, const Tensor& w, const OptTensor& ci, const OptTensor& co, int64_t groups, double p) {
    return norm_dist_lists(x, w, ci, co, groups, p, true);
}

Tensor masked_inf_dist(const Tensor& x, const Tensor& w, int64_t groups, double q, uint32_t seed, int mode) {
    reverse_mode_only("masked_inf_dist", x, w);
    const bool grad = want_grad(x, w);
    Tensor y, pos;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        const c10::DeviceGuard guard(x.device());
        y = new_out(x, w.size(0));
        if (grad) pos = new_ints(x, y.sizes());
        const Dims d(x, groups, w.size(0));
        require(sd_masked_inf_dist_forward(floats(x, "input"), floats(w, "weight"), d.B, d.CO, d.CI, d.G, d.HW, floats(y, "output"),
                                           grad ? ints(pos, "pos") : nullptr, (float)q, seed, mode, stream_of(x)),
                "sd_masked_inf_dist_forward");
    }
    if (grad) {
        auto node = attach(x, w, groups, DistNode::MAX);
        set_history(y, node);
        node->state = SavedVariable(pos, false);
    }
    return y;
}

Tensor sort_neuron(const Tensor& x, const Tensor& w, int64_t groups, double q, int truncate) {
    reverse_mode_only("sort_neuron", x, w);
    const bool grad = want_grad(x, w);
    Tensor y, pos;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        const c10::DeviceGuard guard(x.device());
        y = new_out(x, w.size(0));
        const Dims d(x, groups, w.size(0));
        const float *xp = floats(x, "input"), *wp = floats(w, "weight");
        if (grad) {
            pos = new_ints(x, {(int64_t)truncate, x.size(0), w.size(0), x.size(2)});
            require(sd_sort_neuron_forward(xp, wp, d.B, d.CO, d.CI, d.G, d.HW, floats(y, "output"), ints(pos, "pos"), (float)q,
                                           truncate, stream_of(x)), "sd_sort_neuron_forward");
        } else
            require(sd_sort_neuron_forward_nograd(xp, wp, d.B, d.CO, d.CI, d.G, d.HW, floats(y, "output"), (float)q, truncate,
                                                  stream_of(x)), "sd_sort_neuron_forward_nograd");
    }
    if (grad) {
        auto node = attach(x, w, groups, DistNode::SORT);
        node->q = q; node->truncate = truncate;
        set_history(y, node);
        node->state = SavedVariable(pos, false);
    }
    return y;
}

// ---- interval bounds: lower, upper, weight -> lower, upper -----------------------------------------------------------
struct BoundNode : Node {
    SavedVariable xl, xu, weight, pl, pu;
    int groups = 1;

    variable_list apply(variable_list&& grads) override {
        const Locked lock(mutex_);
        variable_list out(3);
        const bool want_l = task_should_compute_output(0), want_u = task_should_compute_output(1), want_w = task_should_compute_output(2);
        if (!want_l && !want_u && !want_w) return out;
        const Tensor l = xl.unpack(), u = xu.unpack(), w = weight.unpack(), posl = pl.unpack(), posu = pu.unpack();
        at::AutoDispatchBelowADInplaceOrView below;
        const Tensor gl = incoming(*this, grads, 0), gu = incoming(*this, grads, 1);
        const c10::DeviceGuard guard(l.device());
        const int B = (int)gl.size(0), CO = (int)gl.size(1), HW = (int)gl.size(2), CI = (int)l.size(1);
        // One bound alone, with a frozen weight, gets no gradient from this op (core/norm_dist.py:157-173: zeros).  What
        // counts is which inputs require a gradient (should_compute_output: the graph's edges), not which of them this
        // backward pass asks for (task_should_compute_output).
        if (!should_compute_output(2) && !(should_compute_output(0) && should_compute_output(1))) {
            if (want_l) out[0] = at::zeros_like(l);
            if (want_u) out[1] = at::zeros_like(u);
            return out;
        }
        // the entry points write every element of the three gradients
        Tensor gxl = at::empty(l.sizes(), l.options()), gxu = at::empty(u.sizes(), u.options());
        const float *glp = floats(gl, "grad_outputL"), *gup = floats(gu, "grad_outputU");
        const int *plp = ints(posl, "posL"), *pup = ints(posu, "posU");
        if (want_w) {
            out[2] = at::empty(w.sizes(), w.options());
            require(sd_bound_inf_dist_backward_input_weight(glp, gup, plp, pup, B, CO, CI, groups, HW, floats(gxl, "grad_inputL"),
                                                            floats(gxu, "grad_inputU"), floats(out[2], "grad_weight"), stream_of(l)),
                    "sd_bound_inf_dist_backward_input_weight");
        } else
            require(sd_bound_inf_dist_backward_input(glp, gup, plp, pup, B, CO, CI, groups, HW, floats(gxl, "grad_inputL"),
                                                     floats(gxu, "grad_inputU"), stream_of(l)), "sd_bound_inf_dist_backward_input");
        if (want_l) out[0] = gxl;
        if (want_u) out[1] = gxu;
        return out;
    }
    void release_variables() override {
        const Locked lock(mutex_);
        xl.reset_data(); xu.reset_data(); weight.reset_data(); pl.reset_data(); pu.reset_data();
    }
    std::string name() const override { return "BoundNode"; }
};

std::pair<Tensor, Tensor> bound_inf_dist(const Tensor& xl, const Tensor& xu, const Tensor& w, int64_t groups) {
    reverse_mode_only("bound_inf_dist", xl, xu, w);
    const bool grad = want_grad(xl, xu, w);
    Tensor lo, up, pl, pu;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        const c10::DeviceGuard guard(xl.device());
        lo = new_out(xl, w.size(0));
        up = new_out(xl, w.size(0));
        const Dims d(xl, groups, w.size(0));
        const float *lp = floats(xl, "inputL"), *upp = floats(xu, "inputU"), *wp = floats(w, "weight");
        if (grad) {
            pl = new_ints(xl, lo.sizes());
            pu = new_ints(xl, lo.sizes());
            require(sd_bound_inf_dist_forward(lp, upp, wp, d.B, d.CO, d.CI, d.G, d.HW, floats(lo, "outputL"), floats(up, "outputU"),
                                              ints(pl, "posL"), ints(pu, "posU"), stream_of(xl)), "sd_bound_inf_dist_forward");
        } else
            require(sd_bound_inf_dist_forward_nograd(lp, upp, wp, d.B, d.CO, d.CI, d.G, d.HW, floats(lo, "outputL"),
                                                     floats(up, "outputU"), stream_of(xl)), "sd_bound_inf_dist_forward_nograd");
    }
    if (grad) {
        auto node = new_node<BoundNode>();
        node->set_next_edges(collect_next_edges(xl, xu, w));
        node->groups = (int)groups;
        node->xl = SavedVariable(xl, false); node->xu = SavedVariable(xu, false); node->weight = SavedVariable(w, false);
        node->pl = SavedVariable(pl, false); node->pu = SavedVariable(pu, false);
        set_history(variable_list{lo, up}, node);
    }
    return {lo, up};
}

std::pair<Tensor, Tensor> bound_sort_neuron(const Tensor& xl, const Tensor& xu, const Tensor& w, int64_t groups, double q,
                                            int truncate) {
    reverse_mode_only("bound_sort_neuron", xl, xu, w);
    at::AutoDispatchBelowADInplaceOrView below;
    const c10::DeviceGuard guard(xl.device());
    Tensor lo = new_out(xl, w.size(0)), up = new_out(xl, w.size(0));
    const Dims d(xl, groups, w.size(0));
    require(sd_bound_sort_neuron_forward(floats(xl, "inputL"), floats(xu, "inputU"), floats(w, "weight"), d.B, d.CO, d.CI, d.G, d.HW,
                                         floats(lo, "outputL"), floats(up, "outputU"), (float)q, truncate, stream_of(xl)),
            "sd_bound_sort_neuron_forward");
    return {lo, up};
}

// ---- mean shift: the gradient of the centring is the centring of the gradient ----------------------------------------
void shift_kernels(const Tensor& x, const Tensor& index, int64_t channels, const Tensor& mean, const OptTensor& running,
                   double momentum, const Tensor& y) {
    float* rp = running && running->defined() ? floats(*running, "running_mean") : nullptr;
    if (index.defined()) {
        const int G = (int)index.size(-2), cnt = (int)index.size(-1);
        if (G == 0) throw std::runtime_error("index names no groups: its size must be (sub-batches, groups, channels)");
        require(sd_mean_shift_index_forward(floats(x, "input"), ints(index, "index"), (int)x.size(0), G, cnt, (int)(channels / G),
                                            (int)x.size(2), floats(mean, "mean"), rp, (float)momentum, floats(y, "output"),
                                            stream_of(x)), "sd_mean_shift_index_forward");
    } else
        require(sd_mean_shift_forward(floats(x, "input"), (int)x.size(0), (int)x.size(1), (int)x.size(2), floats(mean, "mean"), rp,
                                      (float)momentum, floats(y, "output"), stream_of(x)), "sd_mean_shift_forward");
}

struct ShiftNode : Node {
    SavedVariable index;
    int64_t channels = 0;

    variable_list apply(variable_list&& grads) override {
        const Locked lock(mutex_);
        variable_list out(1);
        if (!task_should_compute_output(0)) return out;
        const Tensor idx = index.unpack();
        at::AutoDispatchBelowADInplaceOrView below;
        const Tensor g = incoming(*this, grads, 0);
        const c10::DeviceGuard guard(g.device());
        out[0] = at::empty(g.sizes(), g.options());
        shift_kernels(g, idx, channels, new_floats(g, {channels}), {}, 0.0, out[0]);
        return out;
    }
    void release_variables() override {
        const Locked lock(mutex_);
        index.reset_data();
    }
    std::string name() const override { return "ShiftNode"; }
};

std::pair<Tensor, Tensor> mean_shift_index(const Tensor& x_in, const OptTensor& index, int64_t channels, const OptTensor& running,
                                           double momentum) {
    reverse_mode_only("mean_shift", x_in);
    const bool grad = want_grad(x_in);
    Tensor y, mean, idx = index ? *index : Tensor();
    {
        at::AutoDispatchBelowADInplaceOrView below;
        const c10::DeviceGuard guard(x_in.device());
        const Tensor x = x_in.contiguous();
        y = at::empty(x.sizes(), x.options());
        mean = new_floats(x, {channels});
        shift_kernels(x, idx, channels, mean, running, momentum, y);
    }
    if (grad) {
        auto node = new_node<ShiftNode>();
        node->set_next_edges(collect_next_edges(x_in));
        node->channels = channels;
        if (idx.defined()) node->index = SavedVariable(idx, false);
        set_history(y, node);
    }
    return {y, mean};
}

std::pair<Tensor, Tensor> mean_shift(const Tensor& x, const OptTensor& running, double momentum) {
    return mean_shift_index(x, {}, x.size(1), running, momentum);
}

// (sub_batches, groups, count) ascending kept channels, drawn on the current stream of `device`
Tensor sample_index_lists(int64_t seed, int64_t sub_batches, int64_t groups, int64_t channels, int64_t count, at::Device device) {
    const c10::DeviceGuard guard(device);
    const Tensor out = at::empty({sub_batches, groups, count}, at::TensorOptions().dtype(at::kInt).device(device));
    if (count > 0)
        require(sd_sample_index_lists((uint32_t)seed, (int)sub_batches, (int)groups, (int)channels, (int)count, ints(out, "index"),
                                      stream_of(out)), "sd_sample_index_lists");
    return out;
}

// z + sign * vec[channel], outside any graph
Tensor channel_shift(const Tensor& z_in, const Tensor& vec_in, double sign) {
    reverse_mode_only("channel_shift", z_in, vec_in);
    at::AutoDispatchBelowADInplaceOrView below;
    const c10::DeviceGuard guard(z_in.device());
    const Tensor z = z_in.contiguous(), vec = vec_in.contiguous();
    Tensor out = at::empty(z.sizes(), z.options());
    require(sd_channel_shift(floats(z, "input"), floats(vec, "shift"), (int)z.size(0), (int)z.size(1), (int)z.size(2), (float)sign,
                             floats(out, "output"), stream_of(z)), "sd_channel_shift");
    return out;
}

// ---- evaluation pass: a layer's values or bounds with sign * shift[channel] added, outside any graph ------------------
Tensor norm_dist_shifted(const Tensor& x, const Tensor& w, int64_t groups, const Tensor& shift_in, double sign) {
    reverse_mode_only("norm_dist", x, w, shift_in);
    at::AutoDispatchBelowADInplaceOrView below;
    const c10::DeviceGuard guard(x.device());
    Tensor y = new_out(x, w.size(0));
    const Tensor shift = shift_in.contiguous();
    const Dims d(x, groups, w.size(0));
    require(sd_inf_dist_forward_shifted(floats(x, "input"), floats(w, "weight"), d.B, d.CO, d.CI, d.G, d.HW, floats(y, "output"),
                                        floats(shift, "shift"), (float)sign, stream_of(x)), "sd_inf_dist_forward_shifted");
    return y;
}

Tensor sort_neuron_shifted(const Tensor& x, const Tensor& w, int64_t groups, double q, int truncate, const Tensor& shift_in, double sign) {
    reverse_mode_only("sort_neuron", x, w, shift_in);
    at::AutoDispatchBelowADInplaceOrView below;
    const c10::DeviceGuard guard(x.device());
    Tensor y = new_out(x, w.size(0));
    const Tensor shift = shift_in.contiguous();
    const Dims d(x, groups, w.size(0));
    require(sd_sort_neuron_forward_shifted(floats(x, "input"), floats(w, "weight"), d.B, d.CO, d.CI, d.G, d.HW, floats(y, "output"), (float)q,
                                           truncate, floats(shift, "shift"), (float)sign, stream_of(x)), "sd_sort_neuron_forward_shifted");
    return y;
}

std::pair<Tensor, Tensor> bound_inf_dist_shifted(const Tensor& xl, const Tensor& xu, const Tensor& w, int64_t groups, const Tensor& shift_in,
                                                 double sign) {
    reverse_mode_only("bound_inf_dist", xl, xu, w, shift_in);
    at::AutoDispatchBelowADInplaceOrView below;
    const c10::DeviceGuard guard(xl.device());
    Tensor lo = new_out(xl, w.size(0)), up = new_out(xl, w.size(0));
    const Tensor shift = shift_in.contiguous();
    const Dims d(xl, groups, w.size(0));
    require(sd_bound_inf_dist_forward_shifted(floats(xl, "inputL"), floats(xu, "inputU"), floats(w, "weight"), d.B, d.CO, d.CI, d.G, d.HW,
                                              floats(lo, "outputL"), floats(up, "outputU"), floats(shift, "shift"), (float)sign, stream_of(xl)),
            "sd_bound_inf_dist_forward_shifted");
    return {lo, up};
}

std::pair<Tensor, Tensor> bound_sort_neuron_shifted(const Tensor& xl, const Tensor& xu, const Tensor& w, int64_t groups, double q, int truncate,
                                                    const Tensor& shift_in, double sign) {
    reverse_mode_only("bound_sort_neuron", xl, xu, w, shift_in);
    at::AutoDispatchBelowADInplaceOrView below;
    const c10::DeviceGuard guard(xl.device());
    Tensor lo = new_out(xl, w.size(0)), up = new_out(xl, w.size(0));
    const Tensor shift = shift_in.contiguous();
    const Dims d(xl, groups, w.size(0));
    require(sd_bound_sort_neuron_forward_shifted(floats(xl, "inputL"), floats(xu, "inputU"), floats(w, "weight"), d.B, d.CO, d.CI, d.G, d.HW,
                                                 floats(lo, "outputL"), floats(up, "outputU"), (float)q, truncate, floats(shift, "shift"),
                                                 (float)sign, stream_of(xl)), "sd_bound_sort_neuron_forward_shifted");
    return {lo, up};
}

// values and bounds of a layer together
std::tuple<Tensor, Tensor, Tensor> sort_neuron_box_shifted(const Tensor& x, const Tensor& xl, const Tensor& xu, const Tensor& w, int64_t groups,
                                                           double q, int truncate, const Tensor& shift_in, double sign) {
    reverse_mode_only("sort_neuron", x, xl, xu, w, shift_in);
    at::AutoDispatchBelowADInplaceOrView below;
    const c10::DeviceGuard guard(x.device());
    Tensor y = new_out(x, w.size(0)), lo = new_out(xl, w.size(0)), up = new_out(xl, w.size(0));
    const Tensor shift = shift_in.contiguous();
    const Dims d(x, groups, w.size(0));
    require(sd_sort_neuron_box_forward(floats(x, "input"), floats(xl, "inputL"), floats(xu, "inputU"), floats(w, "weight"), d.B, d.CO, d.CI, d.G,
                                       d.HW, floats(y, "output"), floats(lo, "outputL"), floats(up, "outputU"), (float)q, truncate,
                                       floats(shift, "shift"), (float)sign, stream_of(x)), "sd_sort_neuron_box_forward");
    return {y, lo, up};
}

// ---- windows of a convolutional layer as columns; the gradient is the sum back into the image --------------------------
struct UnfoldNode : Node {   // saves sizes only, which nothing changes or frees
    int B, C, H, W, KH, KW, stride, pad, dil;

    variable_list apply(variable_list&& grads) override {
        at::AutoDispatchBelowADInplaceOrView below;
        variable_list out(1);
        if (!grads[0].defined() || !task_should_compute_output(0)) return out;
        const Tensor g = grads[0].contiguous();
        const c10::DeviceGuard guard(g.device());
        out[0] = new_floats(g, {B, C, H, W});
        require(sd_fold(floats(g, "grad_output"), B, C, H, W, KH, KW, stride, pad, dil, floats(out[0], "grad_input"), stream_of(g)),
                "sd_fold");
        return out;
    }
    std::string name() const override { return "UnfoldNode"; }
};

Tensor unfold(const Tensor& x_in, int kh, int kw, int dil, int pad, int stride) {
    reverse_mode_only("unfold", x_in);
    const bool grad = want_grad(x_in);
    const int B = (int)x_in.size(0), C = (int)x_in.size(1), H = (int)x_in.size(2), W = (int)x_in.size(3);
    Tensor y;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        const c10::DeviceGuard guard(x_in.device());
        const Tensor x = x_in.contiguous();
        if (stride < 1) throw std::runtime_error("unfold: stride=" + std::to_string(stride) + " must be positive");
        const int64_t oh = (H + 2 * pad - dil * (kh - 1) - 1) / stride + 1, ow = (W + 2 * pad - dil * (kw - 1) - 1) / stride + 1;
        y = new_floats(x, {B, (int64_t)C * kh * kw, oh > 0 && ow > 0 ? oh * ow : 1});   // a window that does not fit is refused below
        require(sd_unfold(floats(x, "input"), B, C, H, W, kh, kw, stride, pad, dil, floats(y, "output"), stream_of(x)), "sd_unfold");
    }
    if (grad) {
        auto node = new_node<UnfoldNode>();
        node->set_next_edges(collect_next_edges(x_in));
        node->B = B; node->C = C; node->H = H; node->W = W; node->KH = kh; node->KW = kw;
        node->stride = stride; node->pad = pad; node->dil = dil;
        set_history(y, node);
    }
    return y;
}

// ---- losses on the log probability of a label, from logits in fp32, bf16 or fp16 --------------------------------------
int element_type(const Tensor& t, const char* name) {
    if (!t.is_cuda()) throw std::runtime_error(std::string(name) + " must be a CUDA tensor");
    switch (t.scalar_type()) {
        case at::kFloat: return SD_FLOAT32;
        case at::kBFloat16: return SD_BFLOAT16;
        case at::kHalf: return SD_FLOAT16;
        default: throw std::runtime_error(std::string(name) + " must have dtype torch.float32, torch.bfloat16 or torch.float16");
    }
}

void same_device(const Tensor& t, const char* name, const Tensor& like) {
    if (!t.is_cuda()) throw std::runtime_error(std::string(name) + " must be a CUDA tensor");
    if (t.device() != like.device()) throw std::runtime_error(std::string(name) + " is on another device than the outputs");
}

// The logits as the kernels read them: classes next to each other, at most two further dimensions with strides of their own
// (padded vocabularies, rows of a larger batch); anything else is copied.
Tensor readable_logits(const Tensor& z) {
    const bool rows = z.dim() <= 3 && (z.size(-1) == 1 || z.stride(-1) == 1);
    return rows ? z : z.contiguous();
}

// A saved tensor of a few entries for each row: the caller's hooks may hand it back with other strides than it had, and so may they the logits.
Tensor handed_back(const Tensor& t, const Tensor& grad) {
    if (!t.defined()) return t;
    same_device(t, "what a saved tensor's hook gives", grad);
    return t.contiguous();
}

sd_label_rows label_rows(const Tensor& z, const Tensor& labels, int64_t ignore) {
    sd_label_rows a{};
    a.dtype = element_type(z, "outputs");
    a.logits = z.data_ptr();
    a.labels = labels.data_ptr<int64_t>();
    a.classes = z.size(-1);
    a.rows = labels.numel();
    if (z.dim() == 3) {
        a.inner = z.size(1);
        a.outer_stride = z.stride(0); a.inner_stride = z.stride(1);
    } else {
        a.inner = a.rows;
        a.inner_stride = z.dim() == 2 ? z.stride(0) : z.size(-1);
    }
    a.ignore_index = ignore;
    return a;
}

Tensor label_indices(const Tensor& targets, const Tensor& outputs) {
    same_device(targets, "targets", outputs);
    if (targets.scalar_type() != at::kLong && targets.scalar_type() != at::kInt) throw std::runtime_error("targets must have dtype torch.int64 or torch.int32");
    if (outputs.dim() < 2 || targets.sizes() != outputs.sizes().slice(0, outputs.dim() - 1))
        throw std::runtime_error("targets must have the sizes of outputs without their last dimension, the classes");
    return targets.to(at::kLong).contiguous();
}

// a constant per row: no gradient flows into it
void check_constants(const Tensor& t, const char* name, const Tensor& targets) {
    same_device(t, name, targets);
    if (t.scalar_type() != at::kFloat) throw std::runtime_error(std::string(name) + " must have dtype torch.float32");
    if (t.sizes() != targets.sizes()) throw std::runtime_error(std::string(name) + " must have the sizes of targets");
    if (at::GradMode::is_enabled() && t.requires_grad())
        throw std::runtime_error(std::string(name) + " must not require a gradient: the loss is differentiated with respect to outputs alone");
}

// What a call works in, as one tensor (an allocation is a microsecond of the host): where the gradient is wanted what it needs of the
// rows - (top, 1 / sum), and for the losses the rows' weights and their scale - and behind it the scratch.
struct Work {
    Tensor whole;
    float *stats = nullptr, *weight = nullptr, *scale = nullptr, *scratch = nullptr;
    Work() = default;
    Work(const Tensor& like, const sd_label_rows& a, bool loss, bool grad) {
        const int64_t n = sd_label_scratch(&a, loss);
        if (n < 0) require(SD_ERR_ARG, "sd_label_scratch");
        if (n + floats_of(a.rows, loss, grad) == 0) return;
        whole = new_floats(like, {n + floats_of(a.rows, loss, grad)});
        places(whole, a.rows, loss, grad);
    }
    // the places in the tensor of a call whose gradient is wanted
    Work(const Tensor& saved, int64_t rows, bool loss) : whole(saved) { places(whole, rows, loss, true); }

private:
    static int64_t round4(int64_t n) { return (n + 3) / 4 * 4; }
    static int64_t floats_of(int64_t rows, bool loss, bool grad) { return (grad ? round4(2 * rows) + (loss ? round4(rows) : 0) : 0) + (loss ? 4 : 0); }
    void places(const Tensor& t, int64_t rows, bool loss, bool grad) {
        float* p = floats(t, "work");
        if (loss) { scale = p; p += 4; }
        if (grad) { stats = p; p += round4(2 * rows); }
        if (grad && loss) { weight = p; p += round4(rows); }
        scratch = p;
    }
};

// Stands behind a gradient that create_graph asked for: the first derivative is right, a second one would be more than these
// kernels know.
struct OnceNode : Node {
    variable_list apply(variable_list&&) override {
        throw std::runtime_error("sortnet_amd: label_log_probs, preference_loss, policy_loss and distill_loss can be differentiated once: their gradients have no derivatives");
    }
    std::string name() const override { return "OnceNode"; }
};

struct LabelNode : Node {
    enum Kind { VALUES, PREFERENCE, POLICY } kind;
    SavedVariable logits, labels, work;
    Tensor made;            // the gradient for an upstream gradient of 1, where the forward made it
    int64_t capture = 0;    // the graph capture that made it
    int64_t ignore = 0;
    bool last = false;      // this backward is the graph's last: `made` may be given away

    variable_list apply(variable_list&& grads) override {
        const Locked lock(mutex_);
        variable_list out(1);
        if (!task_should_compute_output(0)) return out;
        const Tensor saved = logits.unpack(), saved_labels = labels.unpack(), wk = work.unpack();
        std::shared_ptr<OnceNode> once;
        if (at::GradMode::is_enabled()) {
            once = new_node<OnceNode>();
            once->set_next_edges({next_edge(0), grads[0].defined() ? torch::autograd::impl::gradient_edge(grads[0]) : torch::autograd::Edge()});
        }
        at::AutoDispatchBelowADInplaceOrView below;
        const Tensor g = incoming(*this, grads, 0), z = readable_logits(saved), l = handed_back(saved_labels, g);
        const c10::DeviceGuard guard(z.device());
        // A gradient that is there already is only written again for another upstream gradient than 1, which the device knows; one that a
        // later backward may want, too, stays as it is, and so does one of another capture: that graph may run again without the forward that
        // writes it, after the caller has changed it or with another upstream gradient.
        const int64_t now = made.defined() && last ? capture_of(stream_of(z)) : -1;
        const bool there = now >= 0 && now == capture, loss = kind != VALUES;
        out[0] = there ? std::move(made) : at::empty(z.sizes(), z.options());
        if (out[0].numel() > 0) {
            const sd_label_rows a = label_rows(z, l, ignore);
            const Work w(wk, a.rows, loss);
            const float* gp = floats(g, "grad_output");     // of log probabilities: the rows' weights
            require(sd_label_gradient(&a, w.stats, loss ? w.weight : gp, kind == POLICY ? w.scale : nullptr, loss ? gp : nullptr, there, out[0].data_ptr(), stream_of(z)),
                    "sd_label_gradient");
        }
        if (once) set_history(out[0], once);
        return out;
    }
    void will_release_variables() override {
        const Locked lock(mutex_);
        last = true;
    }
    void release_variables() override {
        const Locked lock(mutex_);
        logits.reset_data(); labels.reset_data(); work.reset_data();
        made.reset();
    }
    std::string name() const override { return "LabelNode"; }
};

// makes y the output of a node over the logits
void attach_labels(const Tensor& y, LabelNode::Kind kind, const Tensor& outputs, const Tensor& z, const Tensor& labels, int64_t ignore, const Tensor& work, const Tensor& made) {
    auto node = new_node<LabelNode>();
    node->set_next_edges(collect_next_edges(outputs));
    node->kind = kind;
    node->ignore = ignore;
    node->logits = SavedVariable(z, false);
    node->labels = SavedVariable(labels, false);
    node->work = SavedVariable(work, false);
    node->made = made;
    if (made.defined()) node->capture = capture_of(stream_of(z));
    set_history(y, node);
}

Tensor label_log_probs(const Tensor& outputs, const Tensor& targets, int64_t ignore) {
    reverse_mode_only("label_log_probs", outputs);
    const bool grad = want_grad(outputs);
    Tensor y, z, labels;
    Work work;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        element_type(outputs, "outputs");
        const c10::DeviceGuard guard(outputs.device());
        labels = label_indices(targets, outputs);
        z = readable_logits(outputs);
        y = new_floats(z, targets.sizes());
        if (y.numel() > 0) {
            const sd_label_rows a = label_rows(z, labels, ignore);
            work = Work(z, a, false, grad);
            require(sd_label_log_probs(&a, floats(y, "log_probs"), work.stats, work.scratch, stream_of(z)), "sd_label_log_probs");
        } else work.whole = new_floats(z, {0});
    }
    if (grad) attach_labels(y, LabelNode::VALUES, outputs, z, labels, ignore, work.whole, {});
    return y;
}

std::pair<Tensor, Tensor> preference_loss(const Tensor& outputs, const Tensor& targets, const Tensor& ref_in, const OptTensor& offsets_in, double beta,
                                          double smoothing, int64_t ignore) {
    reverse_mode_only("preference_loss", outputs, ref_in);
    const bool grad = want_grad(outputs);
    Tensor loss, rewards, z, labels;
    Work work;
    {
        const bool packed = offsets_in && offsets_in->defined();
        element_type(outputs, "outputs");
        check_constants(ref_in, "ref_log_probs", targets);
        at::AutoDispatchBelowADInplaceOrView below;
        const c10::DeviceGuard guard(outputs.device());
        labels = label_indices(targets, outputs);
        z = readable_logits(outputs);
        const Tensor ref = ref_in.contiguous();
        Tensor offsets;
        int64_t answers = 0, tokens = 0;
        if (packed) {
            same_device(*offsets_in, "offsets", outputs);
            if (offsets_in->scalar_type() != at::kLong && offsets_in->scalar_type() != at::kInt) throw std::runtime_error("offsets must have dtype torch.int64 or torch.int32");
            if (offsets_in->dim() != 1 || outputs.dim() != 2) throw std::runtime_error("packed answers need outputs (rows, classes) and offsets (answers + 1)");
            offsets = offsets_in->contiguous();
            answers = offsets.size(0) - 1;
        } else {
            answers = outputs.size(0);
            tokens = answers > 0 ? labels.numel() / answers : 0;
        }
        if (answers < 2 || answers % 2 != 0 || answers / 2 > INT32_MAX)
            throw std::runtime_error("preference_loss needs an even number of answers, the chosen ones before the rejected: got " + std::to_string(answers));
        const sd_label_rows a = label_rows(z, labels, ignore);
        work = Work(z, a, true, grad);
        loss = new_floats(z, {});
        rewards = new_floats(z, {answers});
        require(sd_preference_loss(&a, floats(ref, "ref_log_probs"), packed ? offsets.data_ptr() : nullptr, packed ? (int)offsets.element_size() : 0, tokens,
                                   (int)(answers / 2), beta, smoothing, work.stats, work.weight, floats(rewards, "rewards"), floats(loss, "loss"), work.scratch,
                                   stream_of(z)), "sd_preference_loss");
    }
    if (grad) attach_labels(loss, LabelNode::PREFERENCE, outputs, z, labels, ignore, work.whole, {});
    return {loss, rewards};
}

std::pair<Tensor, Tensor> policy_loss(const Tensor& outputs, const Tensor& targets, const Tensor& old_in, const Tensor& advantages, const OptTensor& ref_in,
                                      double clip_low, double clip_high, double kl, int64_t ignore) {
    reverse_mode_only("policy_loss", outputs, old_in, advantages);
    if (ref_in && ref_in->defined()) reverse_mode_only("policy_loss", *ref_in);
    const bool grad = want_grad(outputs);
    Tensor loss, means, z, labels, made;
    Work work;
    {
        const bool has_ref = ref_in && ref_in->defined();
        element_type(outputs, "outputs");
        check_constants(old_in, "old_log_probs", targets);
        if (has_ref) check_constants(*ref_in, "ref_log_probs", targets);
        check_constants(advantages, "advantages", targets);
        at::AutoDispatchBelowADInplaceOrView below;
        const c10::DeviceGuard guard(outputs.device());
        labels = label_indices(targets, outputs);
        z = readable_logits(outputs);
        const sd_label_rows a = label_rows(z, labels, ignore);
        const Tensor old = old_in.contiguous(), ref = has_ref ? ref_in->contiguous() : Tensor(), adv = advantages.dim() > 2 ? advantages.contiguous() : advantages;
        // one advantage for all rows of an answer comes as an expanded tensor, which is read where it is
        const bool two = z.dim() == 3;
        const int64_t outer = two ? adv.stride(0) : 0, inner = two ? adv.stride(1) : adv.dim() == 1 ? adv.stride(0) : 1;
        work = Work(z, a, true, grad);
        loss = new_floats(z, {});
        means = new_floats(z, {3});
        if (grad && sd_policy_fuses(&a)) made = at::empty(z.sizes(), z.options());
        require(sd_policy_loss(&a, floats(old, "old_log_probs"), static_cast<const float*>(adv.data_ptr()), outer, inner, has_ref ? floats(ref, "ref_log_probs") : nullptr,
                               clip_low, clip_high, kl, work.stats, work.weight, work.scale, made.defined() ? made.data_ptr() : nullptr, floats(loss, "loss"),
                               floats(means, "means"), work.scratch, stream_of(z)), "sd_policy_loss");
    }
    if (grad) attach_labels(loss, LabelNode::POLICY, outputs, z, labels, ignore, work.whole, made);
    return {loss, means};
}

// ---- dropout under a mask that is made again in the backward; up to three tensors share one --------------------------------
void drop(const std::array<Tensor, 3>& x, const std::array<Tensor, 3>& y, double q, uint32_t seed, const Tensor& seeds) {
    const Tensor* first = nullptr;
    const void* in[3] = {nullptr, nullptr, nullptr};
    void* out[3] = {nullptr, nullptr, nullptr};
    for (int k = 0; k < 3; k++)
        if (x[k].defined()) {
            if (!first) first = &x[k];
            in[k] = x[k].data_ptr(); out[k] = y[k].data_ptr();
        }
    if (!first || first->numel() == 0) return;
    require(sd_dropout(in[0], in[1], in[2], element_type(*first, "input"), first->numel(), q, seed, seeds.defined() ? seeds.data_ptr<int64_t>() : nullptr,
                       out[0], out[1], out[2], stream_of(*first)), "sd_dropout");
}

struct DropNode : Node {
    SavedVariable seeds;
    double q = 1.0;
    uint32_t seed = 0;

    // Under create_graph the results depend on the incoming gradients as the outputs do on the inputs: their node, or none.
    std::shared_ptr<DropNode> of_gradients(const variable_list& grads, const Tensor& sd) {
        torch::autograd::edge_list edges(grads.size());
        bool any = false;
        for (size_t k = 0; k < grads.size(); k++)
            if (at::GradMode::is_enabled() && task_should_compute_output(k) && grads[k].defined() && grads[k].requires_grad()) {
                edges[k] = torch::autograd::impl::gradient_edge(grads[k]);
                any = true;
            }
        if (!any) return nullptr;
        auto node = new_node<DropNode>();
        node->set_next_edges(std::move(edges));
        node->q = q;
        node->seed = seed;
        if (sd.defined()) node->seeds = SavedVariable(sd, false);
        return node;
    }

    variable_list apply(variable_list&& grads) override {
        const Locked lock(mutex_);
        const int count = (int)grads.size();
        variable_list out(count);
        const Tensor sd = seeds.unpack();
        const std::shared_ptr<DropNode> again = of_gradients(grads, sd);
        at::AutoDispatchBelowADInplaceOrView below;
        std::array<Tensor, 3> g, gx;
        c10::OptionalDeviceGuard guard;
        for (int k = 0; k < count; k++) {
            if (!task_should_compute_output(k)) continue;
            g[k] = incoming(*this, grads, k);
            guard.reset_device(g[k].device());
            out[k] = gx[k] = at::empty(g[k].sizes(), g[k].options());
        }
        drop(g, gx, q, seed, sd);
        if (again) set_history(out, again);
        return out;
    }
    void release_variables() override {
        const Locked lock(mutex_);
        seeds.reset_data();
    }
    std::string name() const override { return "DropNode"; }
};

// One output per tensor that is there, in order.
std::vector<Tensor> dropout(const std::vector<Tensor>& inputs, double q, int64_t seed, const OptTensor& seeds) {
    if (inputs.empty() || inputs.size() > 3) throw std::runtime_error("dropout takes one to three tensors");
    bool grad = false;
    for (const Tensor& t : inputs) {
        reverse_mode_only("dropout", t);
        element_type(t, "input");
        if (t.sizes() != inputs[0].sizes() || t.scalar_type() != inputs[0].scalar_type() || t.device() != inputs[0].device())
            throw std::runtime_error("tensors under one mask must have one size, dtype and device");
        grad = grad || want_grad(t);
    }
    if (!(q >= 0.0 && q <= 1.0)) throw std::runtime_error("dropout: keep probability q=" + std::to_string(q) + " outside 0..1");
    Tensor sd;
    if (seeds && seeds->defined()) {
        same_device(*seeds, "seed", inputs[0]);
        if (seeds->scalar_type() != at::kLong || seeds->numel() != 1) throw std::runtime_error("a seed on the device must be one torch.int64");
        sd = *seeds;
    }
    std::array<Tensor, 3> x, y;
    std::vector<Tensor> out;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        const c10::DeviceGuard guard(inputs[0].device());
        for (size_t k = 0; k < inputs.size(); k++) {
            x[k] = inputs[k].contiguous();
            y[k] = at::empty(x[k].sizes(), x[k].options());
            out.push_back(y[k]);
        }
        drop(x, y, q, (uint32_t)seed, sd);
    }
    if (grad) {
        auto node = new_node<DropNode>();
        node->set_next_edges(collect_next_edges(inputs));
        node->q = q;
        node->seed = (uint32_t)seed;
        if (sd.defined()) node->seeds = SavedVariable(sd, false);
        set_history(out, node);
    }
    return out;
}

// ---- logits as they stand when a class is chosen -------------------------------------------------------------------------
// rows of logits that readable_logits has made readable
sd_logit_rows logit_rows(const Tensor& z) {
    sd_logit_rows a{};
    a.dtype = element_type(z, "outputs");
    a.logits = z.data_ptr();
    a.classes = z.size(-1);
    a.rows = a.classes > 0 ? z.numel() / a.classes : 0;
    if (z.dim() == 3) {
        a.inner = z.size(1);
        a.outer_stride = z.stride(0); a.inner_stride = z.stride(1);
    } else {
        a.inner = a.rows;
        a.inner_stride = z.dim() == 2 ? z.stride(0) : a.classes;
    }
    return a;
}

void check_outputs(const Tensor& outputs) {
    element_type(outputs, "outputs");
    if (outputs.dim() < 2 || outputs.size(-1) < 1) throw std::runtime_error("outputs must have the sizes (..., classes), with one class at least");
}

// What stands beside the rows of logits: entries of a row next to each other, rows with the strides of the logits' dimensions, or one row for all
// (its only dimension).
struct Beside {
    Tensor t;
    int64_t outer = 0, inner = 0;
    Beside() = default;
    explicit Beside(const Tensor& given) : t(given) {
        if (!t.defined()) return;
        if ((t.size(-1) > 1 && t.stride(-1) != 1) || t.dim() > 3) t = t.contiguous();
        if (t.dim() == 1) return;
        if (t.dim() == 3) outer = t.stride(0);
        inner = t.dim() <= 3 ? t.stride(-2) : t.size(-1);
    }
};

Beside beside(const Tensor& t, const char* name, const Tensor& z, bool may_be_shared, int64_t entries) {
    same_device(t, name, z);
    const bool shared = may_be_shared && t.dim() == 1;
    if (!shared && (t.dim() != z.dim() || t.sizes().slice(0, t.dim() - 1) != z.sizes().slice(0, z.dim() - 1)))
        throw std::runtime_error(std::string(name) + " must have the sizes of outputs before the classes");
    if (entries >= 0 && t.size(-1) != entries) throw std::runtime_error(std::string(name) + " must have " + std::to_string(entries) + " entries for each row, not " + std::to_string(t.size(-1)));
    return Beside(t);
}

void no_gradient(const Tensor& t, const char* name) {
    if (at::GradMode::is_enabled() && t.requires_grad()) throw std::runtime_error(std::string(name) + " must not require a gradient: the result is differentiated with respect to outputs alone");
}

struct Constraints {
    Tensor z;       // the logits
    Beside history, bias, allowed;
    Tensor lengths, rows[3];
    double numbers[3] = {1.0, 0.0, 0.0};    // repetition, presence, frequency, where there is no tensor of them

    bool narrow() const { return history.t.defined() || allowed.t.defined(); }   // (else the gradient passes as it is)
    void call(const Tensor* grad, const Tensor& out) const {
        if (out.numel() == 0) return;
        const sd_logit_rows a = logit_rows(z);
        sd_constraints c{};
        if (history.t.defined() && history.t.size(-1) > 0) {     // (a history of no places, which has no address, penalises nothing)
            c.history = history.t.data_ptr();
            c.history_bytes = (int)history.t.element_size();
            c.history_length = history.t.size(-1);
            c.history_outer = history.outer; c.history_inner = history.inner;
            if (lengths.defined()) { c.lengths = lengths.data_ptr(); c.length_bytes = (int)lengths.element_size(); }
            if (rows[0].defined()) c.repetition_rows = floats(rows[0], "repetition");
            if (rows[1].defined()) c.presence_rows = floats(rows[1], "presence");
            if (rows[2].defined()) c.frequency_rows = floats(rows[2], "frequency");
        }
        c.repetition = numbers[0]; c.presence = numbers[1]; c.frequency = numbers[2];
        if (bias.t.defined()) { c.bias = static_cast<const float*>(bias.t.data_ptr()); c.bias_outer = bias.outer; c.bias_inner = bias.inner; }
        if (allowed.t.defined()) {
            c.allowed = allowed.t.data_ptr();
            c.allowed_kind = allowed.t.scalar_type() == at::kBool ? SD_ALLOWED_FLAGS : SD_ALLOWED_BITS;
            c.allowed_outer = allowed.outer; c.allowed_inner = allowed.inner;
        }
        if (grad) require(sd_constrain_gradient(&a, &c, grad->data_ptr(), out.data_ptr(), stream_of(z)), "sd_constrain_gradient");
        else require(sd_constrain_logits(&a, &c, out.data_ptr(), stream_of(z)), "sd_constrain_logits");
    }
};

// The results are linear in the gradients, with one factor each: the derivative of this node's is the node again.
struct ConstrainNode : Node {
    SavedVariable logits, history, allowed, lengths, rows[3];
    Constraints given;      // all but the tensors

    void save(const Constraints& c) {
        given = c;
        given.z = given.history.t = given.bias.t = given.allowed.t = given.lengths = Tensor();
        for (Tensor& t : given.rows) t = Tensor();
        const auto keep = [](SavedVariable& v, const Tensor& t) { if (t.defined()) v = SavedVariable(t, false); };
        if (c.history.t.defined()) keep(logits, c.z);      // (else the gradient does not depend on them)
        keep(history, c.history.t); keep(allowed, c.allowed.t); keep(lengths, c.lengths);
        for (int k = 0; k < 3; k++) keep(rows[k], c.rows[k]);
    }
    variable_list apply(variable_list&& grads) override {
        const Locked lock(mutex_);
        variable_list out(1);
        if (!task_should_compute_output(0)) return out;
        Constraints c = given;
        c.z = logits.unpack(); c.history.t = history.unpack(); c.allowed.t = allowed.unpack(); c.lengths = lengths.unpack();
        for (int k = 0; k < 3; k++) c.rows[k] = rows[k].unpack();
        const bool again = at::GradMode::is_enabled() && grads[0].defined() && grads[0].requires_grad();
        std::shared_ptr<ConstrainNode> next;
        if (again) {
            next = new_node<ConstrainNode>();
            next->set_next_edges({torch::autograd::impl::gradient_edge(grads[0])});
            next->save(c);
        }
        at::AutoDispatchBelowADInplaceOrView below;
        const Tensor g = incoming(*this, grads, 0);
        const c10::DeviceGuard guard(g.device());
        c.z = c.z.defined() ? readable_logits(c.z) : g;
        for (Beside* b : {&c.history, &c.allowed}) {        // (see handed_back; strides of their own are read as they are)
            if (!b->t.defined()) continue;
            same_device(b->t, "what a saved tensor's hook gives", g);
            *b = Beside(b->t);
        }
        c.lengths = handed_back(c.lengths, g);
        for (Tensor& t : c.rows) t = handed_back(t, g);
        out[0] = at::empty(c.z.sizes(), c.z.options());
        c.call(&g, out[0]);
        if (again) set_history(out[0], next);
        return out;
    }
    void release_variables() override {
        const Locked lock(mutex_);
        for (SavedVariable* v : {&logits, &history, &allowed, &lengths, &rows[0], &rows[1], &rows[2]}) v->reset_data();
    }
    std::string name() const override { return "ConstrainNode"; }
};

struct PassNode : Node {       // a bias alone: the gradient as it is
    variable_list apply(variable_list&& grads) override { return {task_should_compute_output(0) ? grads[0] : Tensor()}; }
    std::string name() const override { return "PassNode"; }
};

Tensor constrain_logits(const Tensor& outputs, const OptTensor& history, const OptTensor& lengths, double repetition, double presence, double frequency,
                        const OptTensor& repetitions, const OptTensor& presences, const OptTensor& frequencies, const OptTensor& bias, const OptTensor& allowed) {
    reverse_mode_only("constrain_logits", outputs);
    const auto there = [](const OptTensor& t) { return t && t->defined(); };
    check_outputs(outputs);
    const bool grad = want_grad(outputs);
    const OptTensor* of_rows[3] = {&repetitions, &presences, &frequencies};
    const char* names[3] = {"repetition", "presence", "frequency"};
    for (int k = 0; k < 3; k++)
        if (there(*of_rows[k])) { reverse_mode_only("constrain_logits", **of_rows[k]); no_gradient(**of_rows[k], names[k]); }
    if (there(bias)) { reverse_mode_only("constrain_logits", *bias); no_gradient(*bias, "bias"); }
    Constraints c;
    Tensor out;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        const c10::DeviceGuard guard(outputs.device());
        const auto whole = [](const Tensor& t) { return t.scalar_type() == at::kLong || t.scalar_type() == at::kInt; };
        c.numbers[0] = repetition; c.numbers[1] = presence; c.numbers[2] = frequency;
        for (int k = 0; k < 3; k++) {
            if (!there(*of_rows[k])) continue;
            const Tensor& t = **of_rows[k];
            same_device(t, names[k], outputs);
            if (t.scalar_type() != at::kFloat) throw std::runtime_error(std::string(names[k]) + " must have dtype torch.float32");
            if (t.sizes() != outputs.sizes().slice(0, outputs.dim() - 1)) throw std::runtime_error(std::string(names[k]) + " must be a number or have the sizes of outputs before the classes");
            c.rows[k] = t.contiguous();
        }
        if (there(history)) {
            if (!whole(*history)) throw std::runtime_error("history must have dtype torch.int64 or torch.int32");
            c.history = beside(*history, "history", outputs, false, -1);
        }
        if (there(lengths)) {
            if (!there(history)) throw std::runtime_error("lengths are those of a history: none was given");
            same_device(*lengths, "lengths", outputs);
            if (!whole(*lengths)) throw std::runtime_error("lengths must have dtype torch.int64 or torch.int32");
            if (lengths->sizes() != outputs.sizes().slice(0, outputs.dim() - 1)) throw std::runtime_error("lengths must have the sizes of outputs before the classes");
            c.lengths = lengths->contiguous();
        }
        if (there(bias)) {
            if (bias->scalar_type() != at::kFloat) throw std::runtime_error("bias must have dtype torch.float32");
            c.bias = beside(*bias, "bias", outputs, true, outputs.size(-1));
        }
        if (there(allowed)) {
            if (allowed->scalar_type() != at::kBool && allowed->scalar_type() != at::kInt) throw std::runtime_error("allowed must have dtype torch.bool, or torch.int32 with a bit for each class");
            c.allowed = beside(*allowed, "allowed", outputs, true, allowed->scalar_type() == at::kBool ? outputs.size(-1) : (outputs.size(-1) + 31) / 32);
        }
        c.z = readable_logits(outputs);
        out = at::empty(c.z.sizes(), c.z.options());
        c.call(nullptr, out);
    }
    if (grad) {
        std::shared_ptr<Node> node;
        if (c.narrow()) {
            auto full = new_node<ConstrainNode>();
            full->save(c);
            node = full;
        } else node = new_node<PassNode>();
        node->set_next_edges(collect_next_edges(outputs));
        set_history(out, node);
    }
    return out;
}

// ---- the largest logits ----------------------------------------------------------------------------------------------------
std::tuple<Tensor, Tensor, Tensor> top_logits(const Tensor& outputs, int64_t k, double temperature) {
    reverse_mode_only("top_logits", outputs);
    check_outputs(outputs);
    at::AutoDispatchBelowADInplaceOrView below;
    const c10::DeviceGuard guard(outputs.device());
    if (k < 1 || k > SD_MOST_TOP || k > outputs.size(-1))
        throw std::runtime_error("top_logits: k=" + std::to_string(k) + " of " + std::to_string(outputs.size(-1)) + " classes: 1.." + std::to_string(SD_MOST_TOP) + " are possible");
    const Tensor z = readable_logits(outputs);
    std::vector<int64_t> sizes(outputs.sizes().begin(), outputs.sizes().end() - 1);
    const Tensor rest = new_floats(z, sizes);
    sizes.push_back(k);
    const Tensor values = at::empty(sizes, z.options()), classes = new_ints(z, sizes);
    if (rest.numel() > 0) {
        const sd_logit_rows a = logit_rows(z);
        const int64_t n = sd_top_scratch(&a, k);
        if (n < 0) require(SD_ERR_ARG, "sd_top_logits");
        const Tensor scratch = n > 0 ? new_floats(z, {n}) : Tensor();
        require(sd_top_logits(&a, k, temperature, values.data_ptr(), ints(classes, "classes"), floats(rest, "rest"), n > 0 ? floats(scratch, "scratch") : nullptr, stream_of(z)),
                "sd_top_logits");
    }
    return {values, classes, rest};
}

// ---- distillation from a teacher's top logits ----------------------------------------------------------------------------
// k entries for each row, one behind the other
struct Lists {
    Tensor values, classes, rest;
    sd_top_lists call() const {
        sd_top_lists l{};
        l.values = values.data_ptr();
        l.classes = classes.data_ptr();
        l.rest = rest.defined() ? floats(rest, "top_rest") : nullptr;
        l.k = values.size(-1);
        l.dtype = element_type(values, "top_values");
        l.class_bytes = (int)classes.element_size();
        return l;
    }
};

// What a call works in, as one tensor: where the gradient is wanted what it needs, behind it the scratch (of nothing else the start).
struct DistillWork {
    float *scale = nullptr, *stats = nullptr, *entries = nullptr, *scratch = nullptr;
    static int64_t floats_of(int64_t rows, int64_t k) { return 4 + (2 * rows + 3) / 4 * 4 + (rows * k + 3) / 4 * 4; }
    DistillWork(const Tensor& whole, int64_t rows, int64_t k, bool grad) {
        float* p = floats(whole, "work");
        scratch = p;
        if (!grad) return;
        scale = p; stats = p + 4; entries = stats + (2 * rows + 3) / 4 * 4;
        scratch = p + floats_of(rows, k);
    }
};

struct DistillNode : Node {
    SavedVariable logits, values, classes, rest, work;
    Tensor made;            // as LabelNode's
    int64_t capture = 0;
    bool last = false;
    double temperature = 1.0;

    variable_list apply(variable_list&& grads) override {
        const Locked lock(mutex_);
        variable_list out(1);
        if (!task_should_compute_output(0)) return out;
        const Tensor saved = logits.unpack(), wk = work.unpack();
        Lists l;
        l.values = values.unpack(); l.classes = classes.unpack(); l.rest = rest.unpack();
        std::shared_ptr<OnceNode> once;
        if (at::GradMode::is_enabled()) {
            once = new_node<OnceNode>();
            once->set_next_edges({next_edge(0), grads[0].defined() ? torch::autograd::impl::gradient_edge(grads[0]) : torch::autograd::Edge()});
        }
        at::AutoDispatchBelowADInplaceOrView below;
        const Tensor g = incoming(*this, grads, 0), z = readable_logits(saved);
        for (Tensor* t : {&l.values, &l.classes, &l.rest}) *t = handed_back(*t, g);
        const c10::DeviceGuard guard(z.device());
        // (as in LabelNode: a gradient that is there is written again for another upstream gradient than 1)
        const int64_t now = made.defined() && last ? capture_of(stream_of(z)) : -1;
        const bool there = now >= 0 && now == capture;
        out[0] = there ? std::move(made) : at::empty(z.sizes(), z.options());
        const sd_logit_rows a = logit_rows(z);
        const sd_top_lists lists = l.call();
        const DistillWork w(wk, a.rows, lists.k, true);
        require(sd_distill_gradient(&a, &lists, temperature, w.stats, w.entries, w.scale, floats(g, "grad_output"), there, out[0].data_ptr(), stream_of(z)), "sd_distill_gradient");
        if (once) set_history(out[0], once);
        return out;
    }
    void will_release_variables() override {
        const Locked lock(mutex_);
        last = true;
    }
    void release_variables() override {
        const Locked lock(mutex_);
        for (SavedVariable* v : {&logits, &values, &classes, &rest, &work}) v->reset_data();
        made.reset();
    }
    std::string name() const override { return "DistillNode"; }
};

std::pair<Tensor, Tensor> distill_loss(const Tensor& outputs, const Tensor& values, const Tensor& classes, const OptTensor& rest, double temperature, double weight) {
    reverse_mode_only("distill_loss", outputs, values);
    const bool has_rest = rest && rest->defined();
    if (has_rest) reverse_mode_only("distill_loss", *rest);
    const bool grad = want_grad(outputs);
    check_outputs(outputs);
    const auto rows_of = [&](const Tensor& t, const char* name, bool entries) {
        same_device(t, name, outputs);
        if (t.dim() != outputs.dim() - !entries || t.sizes().slice(0, outputs.dim() - 1) != outputs.sizes().slice(0, outputs.dim() - 1))
            throw std::runtime_error(std::string(name) + (entries ? " must have the sizes of outputs before the classes, and entries" : " must have the sizes of outputs before the classes"));
        if (at::GradMode::is_enabled() && t.requires_grad())
            throw std::runtime_error(std::string(name) + " must not require a gradient: the loss is differentiated with respect to outputs alone");
    };
    rows_of(values, "top_values", true);
    rows_of(classes, "top_classes", true);
    if (has_rest) rows_of(*rest, "top_rest", false);
    element_type(values, "top_values");
    if (classes.scalar_type() != at::kLong && classes.scalar_type() != at::kInt) throw std::runtime_error("top_classes must have dtype torch.int64 or torch.int32");
    if (classes.sizes() != values.sizes()) throw std::runtime_error("top_classes must have the sizes of top_values");
    if (has_rest && rest->scalar_type() != at::kFloat) throw std::runtime_error("top_rest must have dtype torch.float32");
    Tensor loss, divergences, z, work, made;
    Lists l;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        const c10::DeviceGuard guard(outputs.device());
        z = readable_logits(outputs);
        const sd_logit_rows a = logit_rows(z);
        l.values = values.contiguous(); l.classes = classes.contiguous();
        if (has_rest) l.rest = rest->contiguous();
        const sd_top_lists lists = l.call();
        const int64_t n = sd_distill_scratch(&a, lists.k);
        if (n < 0) require(SD_ERR_ARG, "sd_distill_loss");
        work = new_floats(z, {n + (grad ? DistillWork::floats_of(a.rows, lists.k) : 0)});
        const DistillWork w(work, a.rows, lists.k, grad);
        loss = new_floats(z, {});
        divergences = new_floats(z, outputs.sizes().slice(0, outputs.dim() - 1));
        if (grad && sd_distill_fuses(&a)) made = at::empty(z.sizes(), z.options());
        require(sd_distill_loss(&a, &lists, temperature, weight, w.stats, w.entries, w.scale, made.defined() ? made.data_ptr() : nullptr, floats(loss, "loss"),
                                floats(divergences, "divergences"), w.scratch, stream_of(z)), "sd_distill_loss");
    }
    if (grad) {
        auto node = new_node<DistillNode>();
        node->set_next_edges(collect_next_edges(outputs));
        node->logits = SavedVariable(z, false);
        node->values = SavedVariable(l.values, false);
        node->classes = SavedVariable(l.classes, false);
        if (has_rest) node->rest = SavedVariable(l.rest, false);
        node->work = SavedVariable(work, false);
        node->made = made;
        if (made.defined()) node->capture = capture_of(stream_of(z));
        node->temperature = temperature;
        set_history(loss, node);
    }
    return {loss, divergences};
}

}  // namespace

PYBIND11_MODULE(_host, m) {
    m.doc() = "Autograd front-end of libsortdist.so";
    using released = py::call_guard<py::gil_scoped_release>;
    m.def("norm_dist", &norm_dist, released());
    m.def("norm_dist_dropout", &norm_dist_dropout, released());
    m.def("masked_inf_dist", &masked_inf_dist, released());
    m.def("sort_neuron", &sort_neuron, released());
    m.def("bound_sort_neuron", &bound_sort_neuron, released());
    m.def("bound_inf_dist", &bound_inf_dist, released());
    m.def("mean_shift", &mean_shift, released());
    m.def("mean_shift_index", &mean_shift_index, released());
    m.def("channel_shift", &channel_shift, released());
    m.def("sample_index_lists", &sample_index_lists, released());
    m.def("norm_dist_shifted", &norm_dist_shifted, released());
    m.def("sort_neuron_shifted", &sort_neuron_shifted, released());
    m.def("bound_inf_dist_shifted", &bound_inf_dist_shifted, released());
    m.def("bound_sort_neuron_shifted", &bound_sort_neuron_shifted, released());
    m.def("sort_neuron_box_shifted", &sort_neuron_box_shifted, released());
    m.def("unfold", &unfold, released());
    m.def("label_log_probs", &label_log_probs, released());
    m.def("preference_loss", &preference_loss, released());
    m.def("policy_loss", &policy_loss, released());
    m.def("dropout", &dropout, released());
    m.def("constrain_logits", &constrain_logits, released());
    m.def("top_logits", &top_logits, released());
    m.def("distill_loss", &distill_loss, released());
}
