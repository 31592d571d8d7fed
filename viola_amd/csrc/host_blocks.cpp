// The operators around a block on the native host path: norms with gate and residual sum, and the routing of a mixture of experts, as
// autograd nodes over the library's entry points. They take tensors as a program has them (any leading dimensions, strided rows, vectors
// of another type) and make what a kernel cannot read contiguous first.
#include "host.hpp"

#include <torch/csrc/autograd/functions/utils.h>

using namespace viola_host;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

namespace {

// ---------------------------------------------------------------------------------------------------- norms
enum { X, Y, AFTER_WEIGHT, AFTER_BIAS, WEIGHT, BIAS, GATE, SCALE, SHIFT, INPUTS };
const char* const INPUT_NAMES[INPUTS] = {"x", "y", "after_weight", "after_bias", "weight", "bias", "gate", "scale", "shift"};

// Leading dimensions of a vector that are not one, which have to be the first ones of x: a vector for each index of those.
std::vector<int64_t> prefix_of(const char* name, const Tensor& v, const Tensor& x, int what) {
    TORCH_CHECK(v.dim() >= 1 && v.size(-1) == x.size(-1), name, ": ", INPUT_NAMES[what], " has to end in ", x.size(-1), " features, got ", v.sizes());
    std::vector<int64_t> prefix(v.sizes().begin(), v.sizes().end() - 1);
    while (!prefix.empty() && prefix.back() == 1) prefix.pop_back();
    bool fits = prefix.size() < (size_t)x.dim();
    for (size_t i = 0; fits && i < prefix.size(); ++i) fits = prefix[i] == x.size(i);
    TORCH_CHECK(fits, name, ": ", INPUT_NAMES[what], " of ", v.sizes(), " is neither one vector nor one for each of the first dimensions of ", x.sizes());
    return prefix;
}

struct NormPlan {
    int after = VIOLA_NORM_NONE, before = VIOLA_NORM_NONE;
    double residual_scale = 1.0, branch_scale = 1.0, eps = 0.0;
    at::ScalarType branch = at::kFloat, weight_type = at::kFloat, vector_type = at::kFloat;
    int64_t groups = 1;
    bool by_group[3] = {false, false, false};                    // gate, scale, shift: one vector for each group

    at::ScalarType type_of(int i) const { return i < GATE ? weight_type : vector_type; }
    // A vector as the kernels read it: [cols], or [groups, cols] with whole rows.
    Tensor readable(int i, const Tensor& t, int64_t cols) const {
        const bool grouped = i >= GATE && by_group[i - GATE];
        Tensor v = t.to(type_of(i));
        v = grouped ? v.reshape({groups, cols}) : v.reshape({cols}).contiguous();
        if (grouped && ((cols > 1 && v.stride(1) != 1) || v.stride(0) < cols)) v = v.contiguous();
        // whole pieces of 16 bytes, as the rows have them: a copy of a vector is little beside what it spares the rows
        const bool whole = reinterpret_cast<uintptr_t>(ptr(v)) % 16 == 0 && (!grouped || v.stride(0) % 8 == 0);
        return whole || cols % 8 ? v : v.clone(at::MemoryFormat::Contiguous);
    }
};

struct NormBackward : public Node {
    NormPlan plan;
    SavedVariable saved[INPUTS], stats;
    bool has[INPUTS] = {}, kept[INPUTS] = {};                    // given; its values are read by a gradient
    std::vector<int64_t> shape[INPUTS];
    at::ScalarType type[INPUTS];
    int64_t rows = 0;
    bool has_out = false, has_h = false;

    variable_list apply(variable_list&& grads) override;
    std::string name() const override { return "ViolaNormBackward"; }
    void release_variables() override {
        for (SavedVariable& v : saved) v.reset_data();
        stats.reset_data();
    }
};

// The pointers and distances of the vectors along the row as an entry point takes them.
struct Vectors {
    const void* data[INPUTS] = {};
    int64_t pitch[3] = {};
    void set(const NormPlan& plan, const Tensor (&t)[INPUTS], int64_t cols) {
        for (int i = AFTER_WEIGHT; i < INPUTS; ++i) data[i] = ptr(t[i]);
        // of one whose values are not kept (a shift's in backward): as its gradient has it
        for (int i = 0; i < 3; ++i) pitch[i] = !plan.by_group[i] ? 0 : t[GATE + i].defined() ? t[GATE + i].stride(0) : cols;
    }
};

std::vector<Tensor> norm(const char* name, const Tensor (&input)[INPUTS], NormPlan plan, bool want_out, bool want_h) {
    Tensor t[INPUTS];
    for (int i = 0; i < INPUTS; ++i) t[i] = input[i];
    const Tensor& x = t[X];
    check_seen(name, input);
    TORCH_CHECK(x.dim() >= 1 && x.size(-1) > 0, name, ": x needs a last dimension of features, got ", x.sizes());
    const at::Device device = x.device();
    for (int i = 0; i < INPUTS; ++i)
        if (t[i].defined()) check_float(name, INPUT_NAMES[i], t[i], device);
    const int64_t cols = x.size(-1);
    if (t[Y].defined()) {
        TORCH_CHECK(t[Y].sizes() == x.sizes(), name, ": x and y have to be of one shape, got ", x.sizes(), " and ", t[Y].sizes());
        plan.branch = t[Y].scalar_type();
    }
    for (int i = AFTER_WEIGHT; i <= BIAS; ++i)
        TORCH_CHECK(!t[i].defined() || t[i].sizes() == at::IntArrayRef({cols}), name, ": ", INPUT_NAMES[i], " has to be of shape [", cols, "], got ", t[i].sizes());
    TORCH_CHECK(plan.branch == at::kFloat || plan.branch == at::kBFloat16 || plan.branch == at::kHalf, name, ": dtype has to be float32, bfloat16 or float16, not ", plan.branch);
    TORCH_CHECK(plan.eps >= 0, name, ": eps is negative");
    const c10::DeviceGuard guard(device);
    const Rows xr(x);
    // vectors for different groups: all as finely as the finest
    std::vector<int64_t> finest;
    std::vector<int64_t> prefix[3];
    for (int i = 0; i < 3; ++i)
        if (t[GATE + i].defined()) {
            prefix[i] = prefix_of(name, t[GATE + i], x, GATE + i);
            if (prefix[i].size() > finest.size()) finest = prefix[i];
        }
    for (int64_t n : finest) plan.groups *= n;
    for (int i = 0; i < 3; ++i) {
        Tensor& v = t[GATE + i];
        if (!v.defined()) continue;
        if (prefix[i].size() < finest.size() && !prefix[i].empty()) {
            std::vector<int64_t> aligned = prefix[i], wide = finest;
            aligned.resize(finest.size(), 1);
            aligned.push_back(cols);
            wide.push_back(cols);
            v = v.reshape(aligned).expand(wide);
        }
        plan.by_group[i] = !prefix[i].empty() && plan.groups != 1;
    }
    bool need = false;
    if (at::GradMode::is_enabled())
        for (const Tensor& v : t) need = need || wants(v);
    auto node = need ? std::shared_ptr<NormBackward>(new NormBackward(), torch::autograd::deleteNode) : nullptr;
    Tensor out, h, stats, value[INPUTS];
    {
        at::AutoDispatchBelowADInplaceOrView below;
        const viola_stream_t stream = stream_of(x);
        // one type for the weights and one for the vectors of groups; 32 bits where they differ
        auto common = [&](int first, int last) {
            at::ScalarType type = at::kFloat;
            bool any = false;
            for (int i = first; i <= last; ++i)
                if (t[i].defined()) {
                    if (any && t[i].scalar_type() != type) return at::kFloat;
                    type = t[i].scalar_type();
                    any = true;
                }
            return type;
        };
        plan.weight_type = common(AFTER_WEIGHT, BIAS);
        plan.vector_type = common(GATE, SHIFT);
        for (int i = AFTER_WEIGHT; i < INPUTS; ++i)
            if (t[i].defined()) value[i] = plan.readable(i, t[i], cols);
        const std::optional<Rows> yr = t[Y].defined() ? std::optional<Rows>(t[Y]) : std::nullopt;
        if (want_out) out = room(x.sizes(), x.scalar_type(), device);
        if (want_h) h = room(x.sizes(), plan.branch, device);
        if (need) stats = room({xr.count, 4}, at::kFloat, device);
        if (xr.count) {
            Vectors v;
            v.set(plan, value, cols);
            VIOLA_CALL(viola_norm_forward, xr.data(), xr.pitch, code_of(x.scalar_type()), yr ? yr->data() : nullptr, yr ? yr->pitch : cols, code_of(plan.branch), xr.count,
                       cols, plan.after, v.data[AFTER_WEIGHT], v.data[AFTER_BIAS], plan.before, v.data[WEIGHT], v.data[BIAS], code_of(plan.weight_type), v.data[GATE],
                       v.pitch[0], v.data[SCALE], v.pitch[1], v.data[SHIFT], v.pitch[2], code_of(plan.vector_type), xr.count / plan.groups, (float)plan.residual_scale,
                       (float)plan.branch_scale, (float)plan.eps, want_out ? out.mutable_data_ptr() : nullptr, want_h ? h.mutable_data_ptr() : nullptr,
                       need ? static_cast<float*>(stats.mutable_data_ptr()) : nullptr, stream);
        }
    }
    if (need) {
        node->plan = plan;
        node->rows = xr.count;
        node->has_out = want_out;
        node->has_h = want_h;
        for (int i = 0; i < INPUTS; ++i) {
            if (!t[i].defined()) continue;
            node->has[i] = true;
            node->shape[i] = t[i].sizes().vec();
            node->type[i] = t[i].scalar_type();
            // The rest may change and go: x where it is only added to, a shift always, biases where only a gate's or a scale's gradient would read them.
            node->kept[i] = i == X ? want_h : i == AFTER_BIAS ? want_h || wants(t[GATE]) : i == BIAS ? wants(t[SCALE]) : i != SHIFT;
            if (node->kept[i]) node->saved[i] = SavedVariable(t[i], false);
        }
        node->stats = SavedVariable(stats, false);
        node->set_next_edges(torch::autograd::collect_next_edges(t[X], t[Y], t[AFTER_WEIGHT], t[AFTER_BIAS], t[WEIGHT], t[BIAS], t[GATE], t[SCALE], t[SHIFT]));
        if (want_out) torch::autograd::set_history(out, node);
        if (want_h) torch::autograd::set_history(h, node);
    }
    std::vector<Tensor> outputs;
    if (want_out) outputs.push_back(out);
    if (want_h) outputs.push_back(h);
    return outputs;
}

variable_list NormBackward::apply(variable_list&& grads) {
    check_once("the norm around a block");
    variable_list result(INPUTS);
    const Tensor d_out = has_out ? grads[0] : Tensor(), d_h = has_h ? grads[has_out ? 1 : 0] : Tensor();
    if (!d_out.defined() && !d_h.defined()) return result;
    at::AutoDispatchBelowADInplaceOrView below;
    const at::Device device = (d_out.defined() ? d_out : d_h).device();
    const c10::DeviceGuard guard(device);
    check_eager("a norm around a block", d_out.defined() ? d_out : d_h);
    Tensor t[INPUTS];
    for (int i = 0; i < INPUTS; ++i) {
        if (!kept[i] || (i == X && !d_h.defined())) continue;
        t[i] = saved[i].unpack();
        TORCH_CHECK(t[i].device() == device && t[i].scalar_type() == type[i] && t[i].sizes() == at::IntArrayRef(shape[i]),
                    "a tensor saved by a norm around a block came back changed");
    }
    const int64_t cols = shape[X].back();
    // without dh the part before the next block has no gradient at all
    const bool wanted[INPUTS] = {task_should_compute_output(X), has[Y] && task_should_compute_output(Y),
                                 has[AFTER_WEIGHT] && task_should_compute_output(AFTER_WEIGHT), has[AFTER_BIAS] && task_should_compute_output(AFTER_BIAS),
                                 has[WEIGHT] && d_h.defined() && task_should_compute_output(WEIGHT), has[BIAS] && d_h.defined() && task_should_compute_output(BIAS),
                                 has[GATE] && task_should_compute_output(GATE), has[SCALE] && d_h.defined() && task_should_compute_output(SCALE),
                                 has[SHIFT] && d_h.defined() && task_should_compute_output(SHIFT)};
    Tensor grad[INPUTS];
    for (int i = 0; i < INPUTS; ++i) {
        if (!wanted[i]) continue;
        const at::ScalarType to = i < AFTER_WEIGHT ? type[i] : plan.type_of(i);
        grad[i] = rows ? room(shape[i], to, device) : at::zeros(shape[i], at::TensorOptions().device(device).dtype(to));
    }
    if (rows) {
        const Tensor dout = d_out.defined() ? d_out.contiguous() : Tensor(), dh = d_h.defined() ? d_h.contiguous() : Tensor();
        const Tensor state = restored(stats, device, at::kFloat, {rows, 4});
        const std::optional<Rows> xr = t[X].defined() ? std::optional<Rows>(t[X]) : std::nullopt;
        const std::optional<Rows> yr = has[Y] ? std::optional<Rows>(t[Y]) : std::nullopt;
        // the sums over rows that the wanted gradients are made of
        const int sums = (wanted[AFTER_WEIGHT] || wanted[GATE]) + (wanted[AFTER_BIAS] || (wanted[GATE] && has[AFTER_BIAS])) + (wanted[WEIGHT] || wanted[SCALE]) +
                         (wanted[BIAS] || wanted[SHIFT] || (wanted[SCALE] && has[BIAS]));
        const int64_t floats = viola_norm_portions(rows, cols, rows / plan.groups) * sums * cols;
        const Tensor parts = sums ? room({floats}, at::kFloat, device) : Tensor();
        for (int i = AFTER_WEIGHT; i < INPUTS; ++i)
            if (t[i].defined()) t[i] = plan.readable(i, t[i], cols);
        Vectors v;
        v.set(plan, t, cols);
        auto to = [&](int i) { return grad[i].defined() ? grad[i].mutable_data_ptr() : nullptr; };
        VIOLA_CALL(viola_norm_backward, xr ? xr->data() : nullptr, xr ? xr->pitch : cols, code_of(type[X]), yr ? yr->data() : nullptr, yr ? yr->pitch : cols, code_of(plan.branch), rows, cols,
                   plan.after, v.data[AFTER_WEIGHT], v.data[AFTER_BIAS], dh.defined() ? plan.before : VIOLA_NORM_NONE, v.data[WEIGHT], v.data[BIAS],
                   code_of(plan.weight_type), v.data[GATE], v.pitch[0], v.data[SCALE], v.pitch[1], v.data[SHIFT], v.pitch[2], code_of(plan.vector_type), rows / plan.groups,
                   (float)plan.residual_scale, (float)plan.branch_scale, static_cast<const float*>(state.const_data_ptr()), ptr(dout), ptr(dh), to(X), to(Y),
                   parts.defined() ? static_cast<float*>(parts.mutable_data_ptr()) : nullptr, floats, to(AFTER_WEIGHT), to(AFTER_BIAS), to(WEIGHT), to(BIAS), to(GATE),
                   to(SCALE), to(SHIFT), stream_of(state));
    }
    for (int i = 0; i < INPUTS; ++i)
        if (grad[i].defined()) result[i] = grad[i].scalar_type() == type[i] ? grad[i] : grad[i].to(type[i]);
    return result;
}

// ---------------------------------------------------------------------------------------------------- router
struct RouterPlan {
    int64_t tokens = 0, experts = 0, top_k = 0, sequence = 1;
    int score = VIOLA_SOFTMAX;
    bool normalize = true, given = false, biased = false;
    double scale = 1.0;
    int64_t groups = 0, top_groups = 1, group_top = 1;           // groups 0: the choice is by the logits alone
};

struct RouterBackward : public Node {
    RouterPlan plan;
    SavedVariable logits, chosen, kept;
    std::vector<int64_t> shape;
    at::ScalarType type = at::kFloat;
    int64_t kept_bytes = 0, stats_at = 0;

    variable_list apply(variable_list&& grads) override;
    std::string name() const override { return plan.given ? "ViolaBalanceBackward" : "ViolaRouteBackward"; }
    void release_variables() override {
        for (SavedVariable* v : {&logits, &chosen, &kept}) v->reset_data();
    }
};

struct Routed {
    Tensor chosen, gates, positions, counts, offsets, balance;
};

// given: choices made elsewhere; only counts and balance come back then
Routed router(const char* name, const Tensor& logits, const Tensor& given, const Tensor& mask, RouterPlan plan, bool per_sequence, const Tensor& bias = Tensor()) {
    check_seen(name, {logits, given, mask, bias});
    TORCH_CHECK(logits.dim() >= 2 && logits.size(-1) > 0, name, ": logits have to be [..., tokens, experts], got ", logits.sizes());
    const at::Device device = logits.device();
    check_float(name, "logits", logits, device);
    plan.experts = logits.size(-1);
    plan.given = given.defined();
    const auto lead = logits.sizes().slice(0, logits.dim() - 1);
    if (plan.given) {
        TORCH_CHECK(given.dim() == logits.dim() && given.sizes().slice(0, given.dim() - 1) == lead && given.size(-1) > 0, name, ": experts have to be [",
                    "..., tokens, chosen] beside logits of ", logits.sizes(), ", got ", given.sizes());
        TORCH_CHECK(given.device() == device && (given.scalar_type() == at::kInt || given.scalar_type() == at::kLong), name, ": experts have to be int32 or int64 on ", device);
        plan.top_k = given.size(-1);
    }
    TORCH_CHECK(plan.experts <= 1024, name, " takes up to 1024 experts, got ", plan.experts);
    TORCH_CHECK(plan.top_k >= 1 && plan.top_k <= 32 && (plan.given || plan.top_k <= plan.experts), name, ": ", plan.top_k, " choices of ", plan.experts,
                " experts (1 to 32, and no more than there are)");
    TORCH_CHECK(!mask.defined() || (mask.device() == device && mask.scalar_type() == at::kBool && mask.sizes() == lead), name, ": mask has to be bool of shape ", lead, " on ",
                device);
    if (bias.defined()) {
        check_float(name, "bias", bias, device);
        TORCH_CHECK(bias.sizes() == at::IntArrayRef({plan.experts}), name, ": bias has to be of shape [", plan.experts, "], got ", bias.sizes());
        plan.biased = true;
        TORCH_CHECK(!bias.requires_grad(), name, ": bias steers a choice, which has no gradient: it cannot require one");
    }
    if (plan.groups) {
        TORCH_CHECK(plan.groups > 0 && plan.groups <= 64 && plan.experts % plan.groups == 0, name, ": ", plan.groups, " groups of ", plan.experts, " experts (1 to 64, of one size)");
        const int64_t size = plan.experts / plan.groups;
        TORCH_CHECK(plan.top_groups >= 1 && plan.top_groups <= plan.groups && (plan.group_top == 1 || plan.group_top == 2) && plan.group_top <= size, name, ": top_groups has to be 1 to ",
                    plan.groups, " and group_top 1 or 2 and no more than the ", size, " experts of a group, got ", plan.top_groups, " and ", plan.group_top);
        TORCH_CHECK(plan.top_k <= plan.top_groups * size, name, ": ", plan.top_k, " choices of ", plan.top_groups, " groups of ", size, " experts");
        if (plan.top_groups == plan.groups) plan.groups = plan.top_groups = plan.group_top = 1;      // all are open
        if (plan.groups == 1 && !bias.defined()) plan.groups = 0;
    }
    const c10::DeviceGuard guard(device);
    const bool need = at::GradMode::is_enabled() && logits.requires_grad();
    auto node = need ? std::shared_ptr<RouterBackward>(new RouterBackward(), torch::autograd::deleteNode) : nullptr;
    Routed r;
    Arena kept;
    int64_t stats_at = 0;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        const Rows rows(logits);
        plan.tokens = rows.count;
        TORCH_CHECK(plan.tokens < (int64_t{1} << 26), name, " takes fewer than 2^26 tokens");
        plan.sequence = plan.tokens ? per_sequence ? logits.size(-2) : plan.tokens : 1;
        const auto ints = logits.options().dtype(at::kInt), floats = logits.options().dtype(at::kFloat);
        std::vector<int64_t> choices = lead.vec();
        choices.push_back(plan.top_k);
        const int64_t sequences = plan.tokens / plan.sequence;
        if (!plan.tokens) {
            r.counts = at::zeros({plan.experts}, ints);
            r.balance = at::zeros({}, floats);
        } else {
            r.counts = room({plan.experts}, at::kInt, device);
            r.balance = room({}, at::kFloat, device);
        }
        if (!plan.given) {
            r.chosen = room(choices, at::kInt, device);
            r.gates = room(choices, at::kFloat, device);
            r.positions = room(choices, at::kInt, device);
            r.offsets = plan.tokens ? room({plan.experts + 1}, at::kInt, device) : at::zeros({plan.experts + 1}, ints);
        }
        if (plan.tokens) {
            const Tensor counted = mask.defined() ? mask.contiguous() : Tensor();
            const uint8_t* mask_p = counted.defined() ? static_cast<const uint8_t*>(counted.const_data_ptr()) : nullptr;
            const int64_t cost_at = kept.take(sequences * plan.experts * 4);
            stats_at = need ? kept.take(plan.tokens * 8) : 0;
            const int64_t words = (plan.groups ? viola_route_steered_workspace : viola_route_workspace)(plan.tokens, plan.experts, plan.sequence);
            Arena freed, &temp = need ? freed : kept;                        // nothing is kept without a gradient
            const int64_t temp_at = temp.take(words * 4);
            kept.make(device);
            if (need) freed.make(device);
            float* stats = need ? kept.as<float>(stats_at) : nullptr;
            const viola_stream_t stream = stream_of(logits);
            const int type = code_of(logits.scalar_type());
            int* counts = static_cast<int*>(r.counts.mutable_data_ptr());
            float* loss = static_cast<float*>(r.balance.mutable_data_ptr());
            if (plan.given) {
                const Tensor choice = given.contiguous();
                VIOLA_CALL(viola_balance_forward, rows.data(), rows.pitch, type, plan.tokens, plan.experts, (int)plan.top_k, plan.score, mask_p, plan.sequence,
                           choice.const_data_ptr(), choice.scalar_type() == at::kLong, counts, loss, kept.as<float>(cost_at), stats, temp.as<int32_t>(temp_at), words, stream);
            } else if (plan.groups) {
                const Tensor steer = bias.defined() ? bias.to(at::kFloat).contiguous() : Tensor();
                VIOLA_CALL(viola_route_steered_forward, rows.data(), rows.pitch, type, plan.tokens, plan.experts, (int)plan.top_k, plan.score, plan.normalize, (float)plan.scale,
                           static_cast<const float*>(ptr(steer)), (int)plan.groups, (int)plan.top_groups, (int)plan.group_top, mask_p, plan.sequence,
                           static_cast<int*>(r.chosen.mutable_data_ptr()), static_cast<float*>(r.gates.mutable_data_ptr()), static_cast<int*>(r.positions.mutable_data_ptr()),
                           counts, static_cast<int*>(r.offsets.mutable_data_ptr()), loss, kept.as<float>(cost_at), stats, temp.as<int32_t>(temp_at), words, stream);
            } else {
                VIOLA_CALL(viola_route_forward, rows.data(), rows.pitch, type, plan.tokens, plan.experts, (int)plan.top_k, plan.score, plan.normalize, (float)plan.scale, mask_p,
                           plan.sequence, static_cast<int*>(r.chosen.mutable_data_ptr()), static_cast<float*>(r.gates.mutable_data_ptr()),
                           static_cast<int*>(r.positions.mutable_data_ptr()), counts, static_cast<int*>(r.offsets.mutable_data_ptr()), loss, kept.as<float>(cost_at), stats,
                           temp.as<int32_t>(temp_at), words, stream);
            }
        }
    }
    if (need) {
        node->plan = plan;
        node->shape = logits.sizes().vec();
        node->type = logits.scalar_type();
        node->stats_at = stats_at;
        node->kept_bytes = kept.size();
        node->logits = SavedVariable(logits, false);
        if (!plan.given) node->chosen = SavedVariable(r.chosen, false);
        if (kept.size()) node->kept = SavedVariable(kept.tensor(), false);
        node->set_next_edges(torch::autograd::collect_next_edges(logits));
        if (!plan.given) torch::autograd::set_history(r.gates, node);
        torch::autograd::set_history(r.balance, node);
    }
    return r;
}

variable_list RouterBackward::apply(variable_list&& grads) {
    check_once("the router");
    variable_list result(1);
    const Tensor d_gates = plan.given ? Tensor() : grads[0], d_loss = grads[plan.given ? 0 : 1];
    if ((!d_gates.defined() && !d_loss.defined()) || !task_should_compute_output(0)) return result;
    at::AutoDispatchBelowADInplaceOrView below;
    const at::Device device = (d_gates.defined() ? d_gates : d_loss).device();
    const c10::DeviceGuard guard(device);
    check_eager("the router", d_gates.defined() ? d_gates : d_loss);
    const Tensor l = logits.unpack();
    TORCH_CHECK(l.device() == device && l.scalar_type() == type && l.sizes() == at::IntArrayRef(shape), "the logits of a router were moved or replaced between forward and backward");
    result[0] = room(shape, type, device);
    if (!plan.tokens) return result;
    const Tensor arena = restored(kept, device, at::kByte, {kept_bytes});
    const float* base = static_cast<const float*>(arena.const_data_ptr());
    std::vector<int64_t> choices(shape.begin(), shape.end() - 1);
    choices.push_back(plan.top_k);
    const Tensor choice = plan.given ? Tensor() : restored(chosen, device, at::kInt, choices);
    const Tensor dg = d_gates.defined() ? d_gates.contiguous() : Tensor(), dl = d_loss.defined() ? d_loss.contiguous() : Tensor();
    const Rows rows(l);
    const char* const call = plan.biased ? "viola_route_steered_backward" : "viola_route_backward";
    check(call, timed(call, [&] {
        return (plan.biased ? viola_route_steered_backward : viola_route_backward)(
            rows.data(), rows.pitch, code_of(type), plan.tokens, plan.experts, (int)plan.top_k, plan.score, plan.normalize, (float)plan.scale, plan.sequence,
            static_cast<const int*>(ptr(choice)), base, base + stats_at / 4, static_cast<const float*>(ptr(dg)), static_cast<const float*>(ptr(dl)),
            result[0].mutable_data_ptr(), stream_of(l));
    }));
    return result;
}

// ---------------------------------------------------------------------------------------------------- rows
// [..., top_k] places and where the experts' places begin, as the router gives them
void check_places(const char* name, const Tensor& positions, const Tensor& offsets, const at::Device& device) {
    TORCH_CHECK(positions.dim() >= 1 && positions.size(-1) > 0 && positions.device() == device && positions.scalar_type() == at::kInt, name,
                ": positions have to be int32 [..., chosen] on ", device);
    TORCH_CHECK(offsets.dim() == 1 && offsets.numel() >= 1 && offsets.device() == device && offsets.scalar_type() == at::kInt, name, ": offsets have to be int32 [experts + 1] on ",
                device);
    TORCH_CHECK(positions.numel() < (int64_t{1} << 31), name, " takes fewer than 2^31 choices");
}

const int* total_of(const Tensor& offsets) { return static_cast<const int*>(offsets.const_data_ptr()) + offsets.numel() - 1; }

void gather(const Tensor& rows, const Tensor& positions, const Tensor& gates, const Tensor& out) {
    const Rows r(rows);
    VIOLA_CALL(viola_rows_gather, r.data(), r.pitch, r.count, code_of(rows.scalar_type()), r.cols, static_cast<const int*>(ptr(positions)), static_cast<const float*>(ptr(gates)),
               positions.numel() / positions.size(-1), (int)positions.size(-1), out.mutable_data_ptr(), stream_of(rows));
}

// rows and dots may be undefined
void scatter(const Tensor& x, const Tensor& positions, const Tensor& offsets, const Tensor& gates, const Tensor& rows, int64_t row_count, const Tensor& values,
             const Tensor& dots) {
    const Rows r(x);
    const std::optional<Rows> v = values.defined() ? std::optional<Rows>(values) : std::nullopt;
    VIOLA_CALL(viola_rows_scatter, r.data(), r.pitch, code_of(x.scalar_type()), r.cols, static_cast<const int*>(ptr(positions)), static_cast<const float*>(ptr(gates)),
               positions.numel() / positions.size(-1), (int)positions.size(-1), total_of(offsets), rows.defined() ? rows.mutable_data_ptr() : nullptr, row_count,
               v ? v->data() : nullptr, v ? v->pitch : r.cols, dots.defined() ? static_cast<float*>(dots.mutable_data_ptr()) : nullptr, stream_of(x));
}

struct DispatchBackward : public Node {
    SavedVariable positions;
    std::vector<int64_t> shape, places;
    at::ScalarType type = at::kFloat;

    variable_list apply(variable_list&& grads) override {
        check_once("dispatch");
        variable_list result(1);
        if (!grads[0].defined() || !task_should_compute_output(0)) return result;
        at::AutoDispatchBelowADInplaceOrView below;
        const c10::DeviceGuard guard(grads[0].device());
        check_eager("dispatch", grads[0]);
        const Tensor p = restored(positions, grads[0].device(), at::kInt, places);
        result[0] = room(shape, type, grads[0].device());
        if (result[0].numel()) gather(grads[0], p, Tensor(), result[0]);
        return result;
    }
    std::string name() const override { return "ViolaDispatchBackward"; }
    void release_variables() override { positions.reset_data(); }
};

Tensor dispatch(const Tensor& x, const Tensor& positions_, const Tensor& offsets_, std::optional<int64_t> wanted) {
    check_seen("dispatch", {x, positions_, offsets_});
    TORCH_CHECK(!wanted || *wanted >= 0, "dispatch: rows is negative");
    const at::Device device = x.device();
    check_float("dispatch", "x", x, device);
    check_places("dispatch", positions_, offsets_, device);
    TORCH_CHECK(x.dim() >= 1 && x.size(-1) > 0, "dispatch: x needs a last dimension of features, got ", x.sizes());
    const int64_t cols = x.size(-1), tokens = x.numel() / cols, top_k = positions_.size(-1);
    TORCH_CHECK(positions_.numel() == tokens * top_k, "dispatch: positions of ", positions_.sizes(), " do not belong to x of ", x.sizes());
    const int64_t rows = wanted.value_or(tokens * top_k);
    TORCH_CHECK(rows < (int64_t{1} << 31), "dispatch lays out fewer than 2^31 rows");
    const c10::DeviceGuard guard(device);
    const bool need = at::GradMode::is_enabled() && x.requires_grad();
    auto node = need ? std::shared_ptr<DispatchBackward>(new DispatchBackward(), torch::autograd::deleteNode) : nullptr;
    Tensor out, positions;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        positions = positions_.contiguous();
        out = tokens ? room({rows, cols}, x.scalar_type(), device) : at::zeros({rows, cols}, x.options());
        if (tokens && rows) scatter(x, positions, offsets_.contiguous(), Tensor(), out, rows, Tensor(), Tensor());
    }
    if (need) {
        node->shape = x.sizes().vec();
        node->places = positions.sizes().vec();
        node->type = x.scalar_type();
        node->positions = SavedVariable(positions, false);
        node->set_next_edges(torch::autograd::collect_next_edges(x));
        torch::autograd::set_history(out, node);
    }
    return out;
}

struct CombineBackward : public Node {
    SavedVariable y, gates, positions, offsets;
    std::vector<int64_t> shape, places;
    int64_t experts = 0;
    at::ScalarType type = at::kFloat, gates_type = at::kFloat;
    bool has_gates = false;

    variable_list apply(variable_list&& grads) override {
        check_once("combine");
        variable_list result(2);
        if (!grads[0].defined()) return result;
        at::AutoDispatchBelowADInplaceOrView below;
        const at::Device device = grads[0].device();
        const c10::DeviceGuard guard(device);
        check_eager("combine", grads[0]);
        const bool needs_y = task_should_compute_output(0), needs_gates = has_gates && task_should_compute_output(1);
        const Tensor p = restored(positions, device, at::kInt, places), o = restored(offsets, device, at::kInt, {experts});
        const Tensor g = has_gates && needs_y ? restored(gates, device, at::kFloat, places) : Tensor();
        Tensor rows;
        if (needs_gates) {
            rows = y.unpack();
            TORCH_CHECK(rows.device() == device && rows.scalar_type() == type && rows.sizes() == at::IntArrayRef(shape), "a tensor saved by combine came back changed");
        }
        const auto options = at::TensorOptions().device(device);
        const bool any = p.numel() && shape[0];
        if (needs_y) result[0] = any ? room(shape, type, device) : at::zeros(shape, options.dtype(type));
        Tensor dots = needs_gates ? any ? room(places, at::kFloat, device) : at::zeros(places, options.dtype(at::kFloat)) : Tensor();
        if (any && (needs_y || needs_gates)) scatter(grads[0], p, o, g, result[0], shape[0], rows, dots);
        if (needs_gates) result[1] = gates_type == at::kFloat ? dots : dots.to(gates_type);
        return result;
    }
    std::string name() const override { return "ViolaCombineBackward"; }
    void release_variables() override {
        for (SavedVariable* v : {&y, &gates, &positions, &offsets}) v->reset_data();
    }
};

Tensor combine(const Tensor& y, const Tensor& positions_, const Tensor& offsets_, const Tensor& gates_) {
    check_seen("combine", {y, positions_, offsets_, gates_});
    const at::Device device = y.device();
    check_float("combine", "y", y, device);
    check_places("combine", positions_, offsets_, device);
    TORCH_CHECK(y.dim() == 2 && y.size(1) > 0 && y.size(0) < (int64_t{1} << 31), "combine: y has to be [rows, features] with fewer than 2^31 rows, got ", y.sizes());
    if (gates_.defined()) {
        check_float("combine", "gates", gates_, device);
        TORCH_CHECK(gates_.sizes() == positions_.sizes(), "combine: gates of ", gates_.sizes(), " do not belong to positions of ", positions_.sizes());
    }
    const c10::DeviceGuard guard(device);
    const bool need = at::GradMode::is_enabled() && (y.requires_grad() || wants(gates_));
    auto node = need ? std::shared_ptr<CombineBackward>(new CombineBackward(), torch::autograd::deleteNode) : nullptr;
    Tensor out, positions, offsets, gates;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        positions = positions_.contiguous();
        offsets = offsets_.contiguous();
        if (gates_.defined()) gates = gates_.to(at::kFloat).contiguous();
        std::vector<int64_t> shape(positions.sizes().begin(), positions.sizes().end() - 1);
        shape.push_back(y.size(1));
        out = room(shape, y.scalar_type(), device);
        if (out.numel()) gather(y, positions, gates, out);
    }
    if (need) {
        node->shape = y.sizes().vec();
        node->places = positions.sizes().vec();
        node->experts = offsets.numel();
        node->type = y.scalar_type();
        node->has_gates = gates.defined();
        if (gates.defined()) {
            node->gates_type = gates_.scalar_type();
            if (y.requires_grad()) node->gates = SavedVariable(gates, false);            // their own gradient is made of the rows
        }
        if (wants(gates_)) node->y = SavedVariable(y, false);
        node->positions = SavedVariable(positions, false);
        node->offsets = SavedVariable(offsets, false);
        node->set_next_edges(torch::autograd::collect_next_edges(y, gates_));
        torch::autograd::set_history(out, node);
    }
    return out;
}

}  // namespace

void viola_host::register_blocks(py::module_& m) {
    // How the operators below read a tensor: (rows, distance between them in elements, whether they are a copy's). Stride arithmetic only, for tests on the host.
    m.def("row_layout", torch::wrap_pybind_function([](const Tensor& t) {
        const Rows r(t);
        return std::make_tuple(r.count, r.pitch, !r.holder.is_same(t));
    }));
    // (name, x, y, after_weight, after_bias, weight, bias, gate, scale, shift, kind after, kind before, residual scale, branch scale, eps, type of h, with out,
    // with h) -> [out], [h] or [out, h]
    m.def("norm", torch::wrap_pybind_function([](const std::string& name, const Tensor& x, const std::optional<Tensor>& y, const std::optional<Tensor>& after_weight,
                                                 const std::optional<Tensor>& after_bias, const std::optional<Tensor>& weight, const std::optional<Tensor>& bias,
                                                 const std::optional<Tensor>& gate, const std::optional<Tensor>& scale, const std::optional<Tensor>& shift, int after,
                                                 int before, double residual_scale, double branch_scale, double eps, const py::object& type, bool want_out, bool want_h) {
        NormPlan plan;
        plan.after = after;
        plan.before = before;
        plan.residual_scale = residual_scale;
        plan.branch_scale = branch_scale;
        plan.eps = eps;
        plan.branch = type.is_none() ? x.scalar_type() : torch::python::detail::py_object_to_dtype(type);
        const Tensor input[INPUTS] = {x, or_none(y), or_none(after_weight), or_none(after_bias), or_none(weight), or_none(bias), or_none(gate), or_none(scale), or_none(shift)};
        py::gil_scoped_release release;
        return norm(name.c_str(), input, plan, want_out, want_h);
    }));
    m.def("route", torch::wrap_pybind_function([](const Tensor& logits, int64_t top_k, int score, bool normalize, double scale, const std::optional<Tensor>& mask,
                                                  bool per_sequence, const std::optional<Tensor>& bias, int64_t groups, int64_t top_groups, int64_t group_top) {
        RouterPlan plan;
        plan.top_k = top_k;
        plan.score = score;
        plan.normalize = normalize;
        plan.scale = scale;
        plan.groups = groups;
        plan.top_groups = top_groups;
        plan.group_top = group_top;
        Routed r;
        {
            py::gil_scoped_release release;
            r = router("route", logits, Tensor(), or_none(mask), plan, per_sequence, or_none(bias));
        }
        return std::make_tuple(r.chosen, r.gates, r.positions, r.counts, r.offsets, r.balance);
    }));
    m.def("balance_loss", torch::wrap_pybind_function([](const Tensor& logits, const Tensor& experts, int score, const std::optional<Tensor>& mask, bool per_sequence) {
        RouterPlan plan;
        plan.score = score;
        Routed r;
        {
            py::gil_scoped_release release;
            r = router("balance_loss", logits, experts, or_none(mask), plan, per_sequence);
        }
        return std::make_tuple(r.balance, r.counts);
    }));
    m.def("dispatch", torch::wrap_pybind_function([](const Tensor& x, const Tensor& positions, const Tensor& offsets, std::optional<int64_t> rows) {
        py::gil_scoped_release release;
        return dispatch(x, positions, offsets, rows);
    }));
    m.def("combine", torch::wrap_pybind_function([](const Tensor& y, const Tensor& positions, const Tensor& offsets, const std::optional<Tensor>& gates) {
        py::gil_scoped_release release;
        return combine(y, positions, offsets, or_none(gates));
    }));
}
