// The differentiable forms of the sequence operators (isaacgym_amd.sequence): checks, allocation, autograd nodes and the
// launches through libigx's C ABI.  They are C++ because a small call is bound by its host time, and a node written in Python
// costs more than the kernels of a rollout of 4 096 environments (forward and backward of the recurrence: 125 us in Python).
//
// The library is not linked: isaacgym_amd._lib, its only loader, hands over the addresses of its entry points.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <map>
#include <numeric>
#include <unordered_set>

#include "../../include/igx.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

// ---- libigx ---------------------------------------------------------------------------------------------------------

struct Library {
    decltype(&igx_last_error_string) last_error;
    decltype(&igx_linear_recurrence_workspace) recurrence_workspace;
    decltype(&igx_linear_recurrence_with_rest) recurrence;
    decltype(&igx_linear_recurrence_backward_with_rest) recurrence_backward;
    decltype(&igx_block_norm_workspace) norm_workspace;
    decltype(&igx_block_norm_forward) norm;
    decltype(&igx_block_norm_backward) norm_backward;
    decltype(&igx_pack8) pack8;
    decltype(&igx_unpack8) unpack8;
} lib;

struct IgxFailure : std::runtime_error {
    int code;
    IgxFailure(int code, const std::string &text) : std::runtime_error(text), code(code) {}
};

void check(int64_t rc)
{
    if (rc) throw IgxFailure((int)rc, lib.last_error());
}

igx_stream_t stream_of(const Tensor &t)
{
    return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.get_device()).stream();
}

// ---- checks of arguments -------------------------------------------------------------------------------------------

int element(const Tensor &t, const char *name)
{
    const auto type = t.scalar_type();
    const int e = type == at::kFloat ? IGX_F32 : type == at::kHalf ? IGX_F16 : type == at::kBFloat16 ? IGX_BF16 : -1;
    TORCH_CHECK_TYPE(e >= 0, name, ": expected float32, float16 or bfloat16, got ", type);
    TORCH_CHECK_VALUE(t.is_cuda(), "libigx works on device tensors only (", name, " is a ", t.device(), " tensor)");
    return e;
}

void same(const Tensor &t, const char *name, at::IntArrayRef shape, at::ScalarType type, const Tensor &like)
{
    TORCH_CHECK_VALUE(t.is_cuda(), "libigx works on device tensors only (", name, " is a ", t.device(), " tensor)");
    TORCH_CHECK_TYPE(t.scalar_type() == type, name, ": expected dtype ", type, ", got ", t.scalar_type());
    TORCH_CHECK_VALUE(t.get_device() == like.get_device(), name, " is on ", t.device(), ", others on ", like.device());
    TORCH_CHECK_VALUE(t.sizes() == shape, name, ": expected shape ", shape, ", got ", t.sizes());
}

// the address of a contiguous tensor (undefined: NULL)
template <typename T> T *packed(const Tensor &t, const char *name, at::IntArrayRef shape, at::ScalarType type, const Tensor &like)
{
    if (!t.defined()) return nullptr;
    same(t, name, shape, type, like);
    TORCH_CHECK_VALUE(t.is_contiguous(), name, " must be contiguous");
    return static_cast<T *>(t.data_ptr());
}

bool adjacent(const Tensor &t) { return t.size(-1) <= 1 || t.stride(-1) == 1; }

int64_t address(const Tensor &t) { return reinterpret_cast<int64_t>(t.data_ptr()); }

// from a tensor's first byte to behind its last
int64_t reach(const Tensor &t)
{
    const auto sizes = t.sizes(), strides = t.strides();
    int64_t elements = 1;
    for (size_t i = 0; i < sizes.size(); i++) elements += (sizes[i] - 1) * strides[i];
    return elements * (int64_t)t.element_size();
}

// A tensor's bytes: runs of `run` bytes, one for every index into the dimensions that are left (their sizes and strides).
struct Bytes {
    int64_t run;
    std::vector<std::pair<int64_t, int64_t>> outer;  // (stride in bytes, size)
    explicit Bytes(const Tensor &t) : run(t.element_size())
    {
        for (int64_t i = 0; i < t.dim(); i++)
            if (t.size(i) > 1 && t.stride(i) != 0) outer.emplace_back(t.stride(i) * t.element_size(), t.size(i));
        std::sort(outer.begin(), outer.end());
        size_t kept = 0;
        for (const auto &d : outer) {
            if (d.first <= run) run += d.first * (d.second - 1);
            else outer[kept++] = d;
        }
        outer.resize(kept);
    }
};

// Is there a solution with d + sum of c[k].stride * x[k] inside (low, high), low[k] <= x[k] <= high[k]?  Strides in falling
// order, so that what the smaller ones reach leaves few candidates for each; should a call need more than `budget` steps
// after all, the answer is yes.
struct Term {
    int64_t stride, low, high;
};

bool solvable(const std::vector<Term> &c, size_t k, int64_t d, int64_t low, int64_t high, int64_t &budget)
{
    if (--budget < 0) return true;
    if (k == c.size()) return low < d && d < high;
    int64_t least = 0, most = 0;  // of the terms behind this one
    for (size_t j = k + 1; j < c.size(); j++) {
        least += c[j].stride * c[j].low;
        most += c[j].stride * c[j].high;
    }
    auto below = [](int64_t a, int64_t b) { return a >= 0 ? a / b : -((-a + b - 1) / b); };
    // low - d - most < stride x < high - d - least
    const int64_t s = c[k].stride, from = std::max(c[k].low, below(low - d - most, s) + 1), to = std::min(c[k].high, below(high - d - least - 1, s));
    for (int64_t x = from; x <= to; x++)
        if (solvable(c, k + 1, d + s * x, low, high, budget)) return true;
    return false;
}

// do two tensors share a byte?  Exact, also for views that lie between each other's rows or steps.
bool overlap(const Tensor &a, const Tensor &b)
{
    if (!a.defined() || !b.defined() || !a.numel() || !b.numel()) return false;
    const int64_t at = address(a), to = address(b);
    if (at + reach(a) <= to || to + reach(b) <= at) return false;
    const Bytes p(a), q(b);
    if (p.outer.empty() && q.outer.empty()) return true;
    std::map<int64_t, Term, std::greater<int64_t>> terms;  // of q's run less p's
    for (const auto &d : p.outer) terms.emplace(d.first, Term{d.first, 0, 0}).first->second.low -= d.second - 1;
    for (const auto &d : q.outer) terms.emplace(d.first, Term{d.first, 0, 0}).first->second.high += d.second - 1;
    std::vector<Term> c;
    for (const auto &t : terms) c.push_back(t.second);
    int64_t budget = 1 << 18;
    return solvable(c, 0, to - at, -q.run, p.run, budget);
}

// no tensor that a call writes shares memory with one that it reads, or with another one that it writes
template <typename List> void apart(const List &written, const List &read)
{
    for (auto w = std::begin(written); w != std::end(written); ++w) {
        for (const auto &r : read)
            TORCH_CHECK_VALUE(!overlap(*w, r), "a written tensor must not overlap another one of the call");
        for (auto v = std::begin(written); v != w; ++v)
            TORCH_CHECK_VALUE(!overlap(*w, *v), "a written tensor must not overlap another one of the call");
    }
}

Tensor given(const OptTensor &t) { return t ? *t : Tensor(); }
OptTensor maybe(const Tensor &t) { return t.defined() ? OptTensor(t) : OptTensor(); }

// What would give a value with nothing to show that its derivative or its computation is missing: the tangent of a
// forward-mode dual tensor, which does not require grad, and the kernels' part of a traced function, of which only the
// allocations would be recorded.
void refuse_traces()
{
    TORCH_CHECK_NOT_IMPLEMENTED(!torch::jit::tracer::isTracing(), "the sequence operators cannot be recorded by torch.jit.trace");
}

void refuse_tangents(std::initializer_list<const Tensor *> tensors)
{
    refuse_traces();
    for (const Tensor *t : tensors)
        TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(0).defined(),
                                    "the sequence operators have no forward-mode derivatives (a dual tensor was given)");
}

bool differentiated(std::initializer_list<const Tensor *> tensors)
{
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor *t : tensors)
        if (t->defined() && t->requires_grad()) return true;
    return false;
}

// The nodes of a captured backward pass run on the streams their forward ran on; one that belongs to another stream - a
// leaf's accumulator that an eager graph still holds, or an eager node further up - would drag that stream into the capture,
// which ends the process.  Such a capture is refused.
void refuse_foreign_nodes(std::initializer_list<const Tensor *> tensors, const Tensor &like)
{
    c10::DeviceGuard guard(like.device());
    if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
    const c10::Stream now = c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(like.get_device()).unwrap();
    std::vector<std::shared_ptr<torch::autograd::Node>> open;
    std::unordered_set<const torch::autograd::Node *> seen;
    auto reach = [&](std::shared_ptr<torch::autograd::Node> node) {
        if (node && seen.insert(node.get()).second) open.push_back(std::move(node));
    };
    for (const Tensor *t : tensors) {
        if (!t->defined() || !t->requires_grad()) continue;
        reach(t->is_leaf() ? torch::autograd::impl::try_get_grad_accumulator(*t) : t->grad_fn());
    }
    while (!open.empty()) {
        const auto node = open.back();
        open.pop_back();
        const auto made = node->stream();
        TORCH_CHECK(!made || made->device_index() != now.device_index() || *made == now,
                    "a tensor that requires grad is still part of an eager autograd graph: release that graph's outputs before "
                    "capturing one with the same tensor");
        for (const auto &edge : node->next_edges()) reach(edge.function);
    }
}

void once(const AutogradContext *)
{
    TORCH_CHECK(!at::GradMode::is_enabled(), "the sequence operators' gradients cannot be differentiated again (create_graph=True)");
}

// ---- linear recurrence ---------------------------------------------------------------------------------------------

// (stride over steps, over environments) of a [T, N, D] tensor with adjacent channels; its address
template <typename P> void rollout(const Tensor &t, const char *name, const Tensor &like, P &address, int64_t (&stride)[2])
{
    if (!t.defined()) return;
    same(t, name, like.sizes(), like.scalar_type(), like);
    TORCH_CHECK_VALUE(adjacent(t), name, ": the channels (last dimension) must be adjacent, their stride is ", t.stride(2));
    address = t.data_ptr();
    stride[0] = t.stride(0);
    stride[1] = t.stride(1);
}

// what forward and backward share; `like` gives shape, type and device
igx_recurrence recurrence_args(const Tensor &gate, const Tensor &like, const Tensor &state, const Tensor &reset, bool reverse)
{
    igx_recurrence r = {};
    TORCH_CHECK_VALUE(like.dim() == 3, "linear_recurrence: rollouts are [steps, environments, channels] tensors");
    r.dtype = element(like, "inp");
    r.reverse = reverse;
    r.steps = like.size(0);
    r.envs = like.size(1);
    r.width = like.size(2);
    same(gate, "gate", like.sizes(), like.scalar_type(), like);
    const int64_t sd = like.size(2) > 1 ? gate.stride(2) : 1;
    TORCH_CHECK_VALUE(sd == 0 || sd == 1, "gate: the channels (last dimension) must be adjacent or share one gate, their stride is ", sd);
    r.gate = gate.data_ptr();
    r.gate_stride[0] = gate.stride(0);
    r.gate_stride[1] = gate.stride(1);
    r.gate_stride[2] = sd;
    r.state = packed<float>(state, "state", like.sizes().slice(1), at::kFloat, like);
    if (reset.defined()) {
        same(reset, "reset", like.sizes().slice(0, 2), at::kLong, like);
        r.reset = static_cast<const int64_t *>(reset.data_ptr());
        r.reset_stride[0] = reset.stride(0);
        r.reset_stride[1] = reset.stride(1);
    }
    return r;
}

// a call's workspace; back to the stream's pool when it goes out of scope, behind the launch
Tensor recurrence_workspace(igx_recurrence &r, const Tensor &like)
{
    const int64_t size = lib.recurrence_workspace(&r);
    if (size < 0) check(size);
    Tensor ws;
    if (size) {
        ws = at::empty({size}, like.options().dtype(at::kByte));
        r.workspace = ws.data_ptr();
        r.workspace_bytes = size;
    }
    return ws;
}

igx_recurrence_rest rest_args(const Tensor &rest, const Tensor &like)
{
    same(rest, "rest", like.sizes(), at::kChar, like);
    TORCH_CHECK_VALUE(adjacent(rest), "rest: the channels (last dimension) must be adjacent, their stride is ", rest.stride(2));
    return {static_cast<int8_t *>(rest.data_ptr()), {rest.stride(0), rest.stride(1)}};
}

// (out, last); rest (16-bit types): filled in, in out's layout
std::pair<Tensor, Tensor> run_recurrence(const Tensor &gate, const Tensor &inp, const Tensor &state, const Tensor &reset, bool reverse,
                                         Tensor *rest = nullptr)
{
    igx_recurrence r = recurrence_args(gate, inp, state, reset, reverse);
    rollout(inp, "inp", inp, r.inp, r.inp_stride);
    c10::DeviceGuard guard(inp.device());
    Tensor out = at::empty_like(inp);  // in inp's layout, so that neighbouring operators see the one they were given
    if (!adjacent(out) || (!out.is_contiguous() && !out.is_non_overlapping_and_dense())) out = at::empty(inp.sizes(), inp.options());
    Tensor last = at::empty(inp.sizes().slice(1), inp.options().dtype(at::kFloat));
    rollout(out, "out", inp, r.out, r.out_stride);
    r.last = static_cast<float *>(last.data_ptr());
    const Tensor ws = recurrence_workspace(r, inp);
    igx_recurrence_rest kept = {};
    if (rest) kept = rest_args(*rest = at::empty_like(out, out.options().dtype(at::kChar)), out);
    check(lib.recurrence(&r, rest ? &kept : nullptr, stream_of(inp)));
    return {out, last};
}

struct LinearRecurrence : torch::autograd::Function<LinearRecurrence> {
    static variable_list forward(AutogradContext *ctx, const Tensor &gate, const Tensor &inp, const OptTensor &state_,
                                 const OptTensor &reset_, bool reverse, bool unrounded)
    {
        const Tensor state = given(state_), reset = given(reset_);
        Tensor rest;
        const bool keep = unrounded && gate.requires_grad() && inp.scalar_type() != at::kFloat;
        ctx->set_materialize_grads(false);
        auto [out, last] = run_recurrence(gate, inp, state, reset, reverse, keep ? &rest : nullptr);
        ctx->save_for_backward({gate, out, state, reset, rest});
        ctx->saved_data["reverse"] = reverse;
        return {out, last};
    }

    static variable_list backward(AutogradContext *ctx, const variable_list &grads)
    {
        once(ctx);
        Tensor d_out = grads[0], d_last = grads[1];
        variable_list result(6);
        if (!d_out.defined() && !d_last.defined()) return result;
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &gate = saved[0], &out = saved[1], &state = saved[2], &reset = saved[3], &rest = saved[4];
        c10::DeviceGuard guard(out.device());
        if (d_out.defined() && !adjacent(d_out)) d_out = d_out.contiguous();
        if (d_last.defined()) d_last = d_last.contiguous();
        igx_recurrence r = recurrence_args(gate, out, state, reset, ctx->saved_data["reverse"].toBool());
        igx_recurrence_grad g = {};
        rollout(out, "out", out, r.out, r.out_stride);
        rollout(d_out, "d_out", out, g.d_out, g.d_out_stride);
        g.d_last = packed<float>(d_last, "d_last", out.sizes().slice(1), at::kFloat, out);
        if (ctx->needs_input_grad(0)) rollout(result[0] = at::empty_like(out), "d_gate", out, g.d_gate, g.d_gate_stride);
        if (ctx->needs_input_grad(1)) rollout(result[1] = at::empty_like(out), "d_inp", out, g.d_inp, g.d_inp_stride);
        if (state.defined() && ctx->needs_input_grad(2)) {
            result[2] = at::empty_like(state);
            g.d_state = static_cast<float *>(result[2].data_ptr());
        }
        const Tensor ws = recurrence_workspace(r, out);
        igx_recurrence_rest kept = {};
        if (rest.defined()) kept = rest_args(rest, out);
        check(lib.recurrence_backward(&r, &g, rest.defined() ? &kept : nullptr, stream_of(out)));
        return result;
    }
};

std::pair<Tensor, Tensor> linear_recurrence(const Tensor &gate_, const Tensor &inp, const OptTensor &state_, const OptTensor &reset_,
                                            bool reverse, bool unrounded)
{
    const Tensor gate = gate_.sizes() == inp.sizes() ? gate_ : gate_.expand(inp.sizes());
    const Tensor state = given(state_), reset = given(reset_);
    refuse_tangents({&gate, &inp, &state});
    if (!differentiated({&gate, &inp, &state})) return run_recurrence(gate, inp, state, reset, reverse);
    if (inp.is_cuda()) refuse_foreign_nodes({&gate, &inp, &state}, inp);
    const variable_list v = LinearRecurrence::apply(gate, inp, maybe(state), maybe(reset), reverse, unrounded);
    return {v[0], v[1]};
}

Tensor linear_recurrence_step(const Tensor &gate_, const Tensor &inp, const Tensor &state, const OptTensor &reset_,
                              const OptTensor &state_out, const OptTensor &out_)
{
    refuse_traces();
    TORCH_CHECK_VALUE(inp.dim() == 2, "linear_recurrence_step: gate and inp are [environments, channels] tensors");
    const at::NoGradGuard no_grad;
    const Tensor gate = gate_.sizes() == inp.sizes() ? gate_ : gate_.expand(inp.sizes()), reset = given(reset_);
    igx_recurrence r = {};
    r.dtype = element(inp, "inp");
    r.steps = 1;
    r.envs = inp.size(0);
    r.width = inp.size(1);
    same(gate, "gate", inp.sizes(), inp.scalar_type(), inp);
    const int64_t sd = r.width > 1 ? gate.stride(1) : 1;
    TORCH_CHECK_VALUE(sd == 0 || sd == 1, "gate: the channels (last dimension) must be adjacent or share one gate, their stride is ", sd);
    TORCH_CHECK_VALUE(adjacent(inp), "inp: the channels (last dimension) must be adjacent, their stride is ", inp.stride(1));
    r.gate = gate.data_ptr();
    r.gate_stride[1] = gate.stride(0);
    r.gate_stride[2] = sd;
    r.inp = inp.data_ptr();
    r.inp_stride[1] = inp.stride(0);
    r.state = packed<float>(state, "state", inp.sizes(), at::kFloat, inp);
    const Tensor to = state_out ? *state_out : state;
    r.last = packed<float>(to, "state_out", inp.sizes(), at::kFloat, inp);
    if (reset.defined()) {
        same(reset, "reset", inp.sizes().slice(0, 1), at::kLong, inp);
        r.reset = static_cast<const int64_t *>(reset.data_ptr());
        r.reset_stride[1] = reset.stride(0);
    }
    c10::DeviceGuard guard(inp.device());
    const Tensor out = out_ ? *out_ : at::empty(inp.sizes(), inp.options());
    packed<char>(out, "out", inp.sizes(), inp.scalar_type(), inp);
    // state_out may be state: a lane has read its channels before it writes them
    const bool in_place = r.last == r.state;
    if (out_ || !in_place) {
        const std::initializer_list<Tensor> written = {to, out}, read = {gate, inp, reset, in_place ? Tensor() : state};
        apart(written, read);
    } else {
        const std::initializer_list<Tensor> written = {to}, read = {gate, inp, reset};
        apart(written, read);
    }
    r.out = out.data_ptr();
    r.out_stride[1] = r.width;
    // A graph that saved what is overwritten has to notice.  Before the launch, for outside inference mode a tensor that was
    // made in it is refused here: the step must not have been taken then.
    if (out_) torch::autograd::impl::bump_version(out);
    torch::autograd::impl::bump_version(to);
    check(lib.recurrence(&r, nullptr, stream_of(inp)));
    return out;
}

// ---- block norms ---------------------------------------------------------------------------------------------------

// Are the rows (all but the last dimension) of a [..., width] tensor evenly spaced in the order of its dimensions?  Then
// `stride` is the distance from row to row.
bool even_rows(const Tensor &t, int64_t &stride)
{
    stride = t.size(-1);
    if (t.is_contiguous()) return true;
    int64_t reach = 0;  // rows between two entries of the dimension in front; 0 as long as there is one row
    for (int64_t i = t.dim() - 2; i >= 0; i--) {
        if (t.size(i) == 1) continue;
        if (reach == 0) {
            stride = t.stride(i);
            reach = t.size(i);
        } else {
            if (t.stride(i) != stride * reach) return false;
            reach *= t.size(i);
        }
    }
    return true;
}

// the address of a [..., width] tensor with adjacent columns and evenly spaced rows, and the stride from row to row
template <typename P> void row_array(const Tensor &t, const char *name, const Tensor &like, P &address, int64_t &stride)
{
    if (!t.defined()) return;
    same(t, name, like.sizes(), like.scalar_type(), like);
    address = t.data_ptr();
    TORCH_CHECK_VALUE(t.is_contiguous() || adjacent(t), name, ": the columns (last dimension) must be adjacent, their stride is ", t.stride(-1));
    TORCH_CHECK_VALUE(even_rows(t, stride), name, ": its rows (all but the last dimension) must be evenly spaced, in one order for the whole call");
}

// Rows do not know of each other, so any order will do that suits x, y and gate alike.  The order of their dimensions in
// which all of them have evenly spaced rows; empty where that is the one they have, or where there is none.
std::vector<int64_t> row_order(const Tensor &x, const Tensor &y, const Tensor &gate)
{
    int64_t stride;
    const Tensor *odd = nullptr;
    for (const Tensor *t : {&gate, &y, &x})
        if (t->defined() && t->dim() > 0 && !even_rows(*t, stride)) odd = t;
    if (!odd) return {};
    if (y.defined()) same(y, "y", x.sizes(), x.scalar_type(), x);
    if (gate.defined()) same(gate, "gate", x.sizes(), x.scalar_type(), x);
    std::vector<int64_t> order(x.dim());
    std::iota(order.begin(), order.end(), 0);
    std::stable_sort(order.begin(), order.end() - 1, [&](int64_t i, int64_t j) { return odd->stride(i) > odd->stride(j); });
    const at::NoGradGuard no_grad;
    for (const Tensor *t : {&x, &y, &gate})
        if (t->defined() && !even_rows(t->permute(order), stride)) return {};
    return order;
}

int64_t rows_of(const Tensor &t) { return t.size(-1) ? t.numel() / t.size(-1) : 0; }

std::vector<int64_t> scales_shape(const Tensor &t)
{
    std::vector<int64_t> s = t.sizes().vec();
    s.back() = (s.back() + IGX_PACK8_GROUP - 1) / IGX_PACK8_GROUP;
    return s;
}

// 8-bit codes of y (and gate) as a call writes or reads them
void code_args(igx_block_norm &b, const Tensor *codes, size_t count, const Tensor &like)
{
    if (count < 2) return;
    const std::vector<int64_t> groups = scales_shape(like);
    b.y8 = packed<int8_t>(codes[0], "y codes", like.sizes(), at::kChar, like);
    b.y8_scale = packed<float>(codes[1], "y scales", groups, at::kFloat, like);
    if (count < 4) return;
    b.gate8 = packed<int8_t>(codes[2], "gate codes", like.sizes(), at::kChar, like);
    b.gate8_scale = packed<float>(codes[3], "gate scales", groups, at::kFloat, like);
}

struct Parameters {
    Tensor weight, scale, next_weight;
};

igx_block_norm norm_args(const Tensor &like, const Parameters &p, const Tensor &inv_rms, int64_t activation, double eps)
{
    igx_block_norm b = {};
    b.dtype = element(like, "x");
    b.activation = (int32_t)activation;
    b.rows = rows_of(like);
    b.width = like.size(-1);
    b.eps = (float)eps;
    const auto vector = like.sizes().slice(like.dim() - 1);
    b.weight = packed<float>(p.weight, "weight", vector, at::kFloat, like);
    b.scale = packed<float>(p.scale, "scale", vector, at::kFloat, like);
    b.next_weight = packed<float>(p.next_weight, "next_weight", vector, at::kFloat, like);
    if (inv_rms.defined() && b.rows) {
        b.y_inv_rms = packed<float>(inv_rms, "inv_rms", {2, b.rows}, at::kFloat, like);
        b.out_inv_rms = b.y_inv_rms + b.rows;
    }
    return b;
}

// (out, next); undefined where the call has none.  inv_rms and the codes are filled in where defined.
std::pair<Tensor, Tensor> run_norm(const Tensor &x, const Tensor &y, const Tensor &gate, const Parameters &p, int64_t activation,
                                   double eps, const Tensor &inv_rms, const variable_list &codes)
{
    igx_block_norm b = norm_args(x, p, inv_rms, activation, eps);
    row_array(x, "x", x, b.x, b.x_stride);
    row_array(y, "y", x, b.y, b.y_stride);
    row_array(gate, "gate", x, b.gate, b.gate_stride);
    c10::DeviceGuard guard(x.device());
    Tensor out, next;
    if (y.defined()) out = at::empty(x.sizes(), x.options());
    if (p.next_weight.defined()) next = at::empty(x.sizes(), x.options());
    if (out.defined()) b.out = out.data_ptr();
    if (next.defined()) b.next = next.data_ptr();
    code_args(b, codes.data(), codes.size(), x);
    check(lib.norm(&b, stream_of(x)));
    return {out, next};
}

// a gradient as the kernels can read it: copied only where its rows are not evenly spaced or its columns not adjacent
Tensor readable_rows(const Tensor &t)
{
    int64_t stride;
    return !t.defined() || (adjacent(t) && even_rows(t, stride)) ? t : t.contiguous();
}

struct BlockNorm : torch::autograd::Function<BlockNorm> {
    static variable_list forward(AutogradContext *ctx, const Tensor &x, const OptTensor &y_, const OptTensor &weight_,
                                 const OptTensor &gate_, const OptTensor &scale_, const OptTensor &next_weight_, int64_t activation,
                                 double eps, bool checkpoint)
    {
        const Tensor y = given(y_), weight = given(weight_), gate = given(gate_), scale = given(scale_), next_weight = given(next_weight_);
        ctx->set_materialize_grads(false);
        element(x, "x");
        c10::DeviceGuard guard(x.device());
        const Tensor inv_rms = at::empty({2, rows_of(x)}, x.options().dtype(at::kFloat));
        variable_list codes;
        if (checkpoint) {
            for (int i = 0; i < (gate.defined() ? 2 : 1); i++) {
                codes.push_back(at::empty(x.sizes(), x.options().dtype(at::kChar)));
                codes.push_back(at::empty(scales_shape(x), x.options().dtype(at::kFloat)));
            }
        }
        auto [out, next] = run_norm(x, y, gate, {weight, scale, next_weight}, activation, eps, inv_rms, codes);
        const bool keep_x = next_weight.defined() && (y.defined() || !checkpoint);
        variable_list saved = {keep_x ? x : Tensor(), checkpoint ? Tensor() : y, checkpoint ? Tensor() : gate, weight, scale,
                               next_weight, inv_rms};
        saved.insert(saved.end(), codes.begin(), codes.end());
        ctx->save_for_backward(saved);
        ctx->saved_data["activation"] = activation;
        ctx->saved_data["eps"] = eps;
        variable_list outs;
        if (out.defined()) outs.push_back(out);
        if (next.defined()) outs.push_back(next);
        return outs;
    }

    static variable_list backward(AutogradContext *ctx, const variable_list &grads)
    {
        once(ctx);
        variable_list result(9);
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &y = saved[1], &gate = saved[2];
        const Parameters p = {saved[3], saved[4], saved[5]};
        const bool block = p.weight.defined(), behind = p.next_weight.defined(), codes = saved.size() > 7;
        const Tensor given_out = block ? grads[0] : Tensor();
        const Tensor d_out = readable_rows(given_out), d_next = readable_rows(behind ? grads.back() : Tensor());
        if (!d_out.defined() && !d_next.defined()) return result;
        const Tensor &like = d_out.defined() ? d_out : d_next;
        c10::DeviceGuard guard(like.device());
        igx_block_norm b = norm_args(like, p, saved[6], ctx->saved_data["activation"].toInt(), ctx->saved_data["eps"].toDouble());
        row_array(x, "x", like, b.x, b.x_stride);
        row_array(y, "y", like, b.y, b.y_stride);
        row_array(gate, "gate", like, b.gate, b.gate_stride);
        if (codes) {
            code_args(b, &saved[7], saved.size() - 7, like);
            if (block) b.y = b.y8;  // they say which parts there are; not read
            b.gate = b.gate8;
        }
        igx_block_norm_grad g = {};
        row_array(d_out, "d_out", like, g.d_out, g.d_out_stride);
        row_array(d_next, "d_next", like, g.d_next, g.d_next_stride);
        // autograd numbers the edges of the inputs that there are
        const bool there[6] = {true, block, block, codes ? saved.size() > 9 : gate.defined(), p.scale.defined(), behind};
        auto wanted = [&](int i) {
            int edge = 0;
            for (int j = 0; j < i; j++) edge += there[j];
            return there[i] && ctx->needs_input_grad(edge);
        };
        auto rows = [&](int i, void *&to) {
            if (!wanted(i)) return;
            result[i] = at::empty(like.sizes(), like.options());
            to = result[i].data_ptr();
        };
        // without a norm behind, the gradient of x is that of out
        if (d_next.defined()) rows(0, g.d_x);
        else if (wanted(0)) result[0] = given_out;
        rows(1, g.d_y);
        rows(3, g.d_gate);
        auto vector = [&](int i, float *&to) {
            if (!wanted(i)) return;
            result[i] = at::empty({like.size(-1)}, like.options().dtype(at::kFloat));
            to = static_cast<float *>(result[i].data_ptr());
        };
        vector(2, g.d_weight);
        vector(4, g.d_scale);
        vector(5, g.d_next_weight);
        Tensor ws;
        if (g.d_weight || g.d_scale || g.d_next_weight) {
            g.workspace_bytes = lib.norm_workspace(&b);
            if (g.workspace_bytes < 0) check(g.workspace_bytes);
            ws = at::empty({g.workspace_bytes}, like.options().dtype(at::kByte));
            g.workspace = ws.data_ptr();
        }
        check(lib.norm_backward(&b, &g, stream_of(like)));
        return result;
    }
};

std::pair<Tensor, Tensor> block_norm_of(const Tensor &x, const Tensor &y, const Tensor &gate, const Parameters &p, int64_t act, double eps,
                                        bool checkpoint)
{
    const std::initializer_list<const Tensor *> inputs = {&x, &y, &p.weight, &gate, &p.scale, &p.next_weight};
    if (!differentiated(inputs)) return run_norm(x, y, gate, p, act, eps, {}, {});
    if (x.is_cuda()) refuse_foreign_nodes(inputs, x);
    const variable_list v = BlockNorm::apply(x, maybe(y), maybe(p.weight), maybe(gate), maybe(p.scale), maybe(p.next_weight), act, eps, checkpoint);
    return {y.defined() ? v[0] : Tensor(), p.next_weight.defined() ? v.back() : Tensor()};
}

std::pair<Tensor, Tensor> block_norm(const Tensor &x, const OptTensor &y_, const OptTensor &weight_, const OptTensor &gate_,
                                     const OptTensor &scale_, const OptTensor &next_weight_, const std::string &activation, double eps,
                                     bool checkpoint)
{
    const int64_t act = activation == "silu" ? IGX_GATE_SILU : activation == "sigmoid" ? IGX_GATE_SIGMOID : activation == "none" ? IGX_GATE_NONE : -1;
    TORCH_CHECK_VALUE(act >= 0, "activation must be one of 'none', 'sigmoid', 'silu', got '", activation, "'");
    TORCH_CHECK_VALUE(x.dim() >= 1, "x must be a tensor of at least one dimension");
    const Tensor y = given(y_), gate = given(gate_);
    const Parameters p = {given(weight_), given(scale_), given(next_weight_)};
    refuse_tangents({&x, &y, &p.weight, &gate, &p.scale, &p.next_weight});
    const std::vector<int64_t> order = row_order(x, y, gate);
    if (order.empty()) return block_norm_of(x, y, gate, p, act, eps, checkpoint);
    // a rollout kept environment by environment, for one: its rows in the order they are stored, the results laid out like it
    auto turned = [&](const Tensor &t) { return t.defined() ? t.permute(order) : t; };
    std::vector<int64_t> back(order.size());
    for (size_t i = 0; i < order.size(); i++) back[order[i]] = i;
    const auto [out, next] = block_norm_of(turned(x), turned(y), turned(gate), p, act, eps, checkpoint);
    return {out.defined() ? out.permute(back) : out, next.defined() ? next.permute(back) : next};
}

// ---- 8-bit checkpoints ----------------------------------------------------------------------------------------------

std::pair<Tensor, Tensor> pack8(const Tensor &x)
{
    refuse_traces();
    TORCH_CHECK_VALUE(x.dim() >= 1, "x must be a tensor of at least one dimension");
    const at::NoGradGuard no_grad;
    const int e = element(x, "x");
    const void *p = nullptr;
    int64_t stride = 0;
    row_array(x, "x", x, p, stride);
    c10::DeviceGuard guard(x.device());
    const Tensor codes = at::empty(x.sizes(), x.options().dtype(at::kChar));
    const Tensor scales = at::empty(scales_shape(x), x.options().dtype(at::kFloat));
    check(lib.pack8(p, e, rows_of(x), x.size(-1), stride, static_cast<int8_t *>(codes.data_ptr()),
                    static_cast<float *>(scales.data_ptr()), stream_of(x)));
    return {codes, scales};
}

Tensor unpack8(const Tensor &codes, const Tensor &scales, const py::object &dtype)
{
    refuse_traces();
    TORCH_CHECK_VALUE(codes.dim() >= 1, "codes must be a tensor of at least one dimension");
    TORCH_CHECK_VALUE(codes.is_cuda(), "libigx works on device tensors only (codes is a ", codes.device(), " tensor)");
    TORCH_CHECK_TYPE(THPDtype_Check(dtype.ptr()), "dtype must be a torch.dtype");
    c10::DeviceGuard guard(codes.device());
    const Tensor out = at::empty(codes.sizes(), codes.options().dtype(reinterpret_cast<THPDtype *>(dtype.ptr())->scalar_type));
    const int e = element(out, "dtype");
    const auto *q = packed<int8_t>(codes, "codes", codes.sizes(), at::kChar, codes);
    const auto *s = packed<float>(scales, "scales", scales_shape(codes), at::kFloat, codes);
    check(lib.unpack8(q, s, e, rows_of(codes), codes.size(-1), out.data_ptr(), stream_of(codes)));
    return out;
}

}  // namespace

PYBIND11_MODULE(_sequence, m)
{
    m.doc() = "Differentiable forms of the sequence operators; isaacgym_amd.sequence is their documented interface.";
    m.def("bind", [](const py::dict &addresses, const py::object &error) {
        auto take = [&](const char *name, auto &fn) {
            fn = reinterpret_cast<std::decay_t<decltype(fn)>>(addresses[name].cast<uintptr_t>());
        };
        take("igx_last_error_string", lib.last_error);
        take("igx_linear_recurrence_workspace", lib.recurrence_workspace);
        take("igx_linear_recurrence_with_rest", lib.recurrence);
        take("igx_linear_recurrence_backward_with_rest", lib.recurrence_backward);
        take("igx_block_norm_workspace", lib.norm_workspace);
        take("igx_block_norm_forward", lib.norm);
        take("igx_block_norm_backward", lib.norm_backward);
        take("igx_pack8", lib.pack8);
        take("igx_unpack8", lib.unpack8);
        // isaacgym_amd._lib.IgxError(code, text); never released, so that no order of teardown matters
        static py::object *error_class = nullptr;
        if (error_class) return;
        error_class = new py::object(error);
        py::register_exception_translator([](std::exception_ptr p) {
            try {
                if (p) std::rethrow_exception(p);
            } catch (const IgxFailure &e) {
                const py::object value = (*error_class)(e.code, std::string(e.what()));
                PyErr_SetObject(error_class->ptr(), value.ptr());
            }
        });
    });
    m.def("overlap", &overlap);
    m.def("apart", [](const std::vector<OptTensor> &written, const std::vector<OptTensor> &read) {
        std::vector<Tensor> w, r;
        for (const auto &t : written) w.push_back(given(t));
        for (const auto &t : read) r.push_back(given(t));
        apart(w, r);
    });
    m.def("linear_recurrence", &linear_recurrence);
    m.def("linear_recurrence_step", &linear_recurrence_step);
    m.def("block_norm", &block_norm);
    m.def("pack8", &pack8);
    m.def("unpack8", &unpack8);
}
