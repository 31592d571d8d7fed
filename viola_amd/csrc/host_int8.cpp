// Products of 8-bit integers on the native host path: rows are quantized with a scale each, multiplied by fixed codes with a scale for each channel, whole or by
// groups of rows whose places are on the GPU, and the gradient goes back the same way, as an autograd node over the library's entry points.
#include "host.hpp"

#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/utils/pybind.h>

using namespace viola_host;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

namespace {

constexpr int64_t MOST_K = 1 << 17;                                          // products of 127 by 128 that 32 bits hold the sum of

// Fixed weights [n, k] or [groups, n, k] as a product reads them: rows whole 16-byte pieces apart. Others are laid out anew.
struct Codes {
    Tensor holder;
    int64_t n, k, pitch, stride;
    Codes(const Tensor& t, viola_stream_t stream) : holder(t), n(t.size(-2)), k(t.size(-1)), pitch(t.stride(-2)), stride(t.dim() == 3 ? t.stride(0) : 0) {
        if (n == 1 && pitch < k) pitch = ceil_to(k, 16);                     // one row has no distance of its own
        if (t.dim() == 3 && t.size(0) == 1) stride = 0;
        const bool fits = (k == 1 || t.stride(-1) == 1) && pitch >= k && pitch % 16 == 0 && stride >= 0 && stride % 16 == 0 &&
                          reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0 && pitch <= (int64_t{1} << 22) && (n > 1 || k % 16 == 0);
        if (fits || !t.numel()) return;
        const Tensor whole = t.contiguous();
        pitch = ceil_to(k, 16);
        stride = n * pitch;
        std::vector<int64_t> shape = t.sizes().vec();
        shape.back() = pitch;
        holder = room(shape, at::kChar, t.device());
        VIOLA_CALL(viola_codes_repack, whole.const_data_ptr(), holder.mutable_data_ptr(), t.dim() == 3 ? t.size(0) : 1, n, k, pitch, nullptr, nullptr, 1, 1, 0, stream);
    }
    // The transposed codes [.., k, n] of weights without a copy of them
    static Codes turned(const Tensor& t, viola_stream_t stream) {
        const Tensor whole = t.contiguous();
        const int64_t n = t.size(-2), k = t.size(-1), batch = t.dim() == 3 ? t.size(0) : 1, pitch = ceil_to(n, 16);
        std::vector<int64_t> shape = t.sizes().vec();
        shape[shape.size() - 2] = k;
        shape.back() = pitch;
        const Tensor out = room(shape, at::kChar, t.device());
        VIOLA_CALL(viola_codes_transpose_pitched, whole.const_data_ptr(), out.mutable_data_ptr(), batch, n, k, pitch, nullptr, nullptr, 1, 1, 0, nullptr, 0, 0, nullptr, 0, stream);
        return Codes(out.narrow(-1, 0, n), stream);
    }
    const int8_t* data() const { return static_cast<const int8_t*>(holder.const_data_ptr()); }
};

struct Plan {
    int activation = -1;                                                     // of a row [g | u]; negative: none
    int64_t rows = 0, n = 0, k = 0, groups = 0;                              // groups 0: one weight for all rows
    at::ScalarType x_type = at::kFloat, out_type = at::kFloat, bias_type = at::kFloat;
};

// sum over k of codes by codes, times the scales, plus bias
void product(const Plan& p, const int8_t* codes, int64_t pitch, const float* scales, const Codes& w, const float* channels, const Tensor& offsets, const Tensor& bias,
             int64_t n, int64_t k, void* out, at::ScalarType type, viola_stream_t stream) {
    VIOLA_CALL(viola_int8_gemm, codes, pitch, scales, w.data(), w.pitch, w.stride, channels, static_cast<const int32_t*>(ptr(offsets)), p.groups, p.rows, n, k, ptr(bias),
               bias.defined() ? code_of(bias.scalar_type()) : VIOLA_F32, out, code_of(type), stream);
}

struct ProductBackward : public Node {
    Plan plan;
    SavedVariable weight, weight_t, scale, x, offsets;
    std::vector<int64_t> shape;
    std::string label;
    bool has_bias = false, has_turned = false;

    variable_list apply(variable_list&& grads) override;
    std::string name() const override { return "ViolaInt8ProductBackward"; }
    void release_variables() override {
        for (SavedVariable* v : {&weight, &weight_t, &scale, &x, &offsets}) v->reset_data();
    }
};

Tensor aligned(const Tensor& t) {
    const Tensor whole = t.contiguous();
    return reinterpret_cast<uintptr_t>(whole.const_data_ptr()) % 16 == 0 ? whole : whole.clone();
}

Tensor run(const char* name, const Tensor& x, const Tensor& weight, const Tensor& scale, const Tensor& bias, const Tensor& offsets, int activation,
           std::optional<at::ScalarType> type, const Tensor& weight_t) {
    check_seen(name, {x, weight, scale, bias, offsets, weight_t});
    const at::Device device = x.device();
    check_float(name, "x", x, device);
    const bool grouped = offsets.defined();
    TORCH_CHECK(weight.dim() == (grouped ? 3 : 2) && weight.scalar_type() == at::kChar && weight.device() == device, name, ": weight has to be int8 codes [",
                grouped ? "groups, " : "", "out, in] on ", device);
    Plan plan;
    plan.activation = activation;
    plan.groups = grouped ? weight.size(0) : 0;
    plan.n = weight.size(-2);
    plan.k = weight.size(-1);
    plan.x_type = x.scalar_type();
    plan.out_type = type.value_or(plan.x_type);
    TORCH_CHECK(plan.n > 0 && plan.k > 0 && (!grouped || plan.groups > 0), name, ": weight of ", weight.sizes(), " is empty");
    TORCH_CHECK(plan.k <= MOST_K, name, " adds up at most ", MOST_K, " products, got ", plan.k);
    TORCH_CHECK(plan.groups <= 1024, name, " takes up to 1024 groups, got ", plan.groups);
    TORCH_CHECK(x.dim() >= 1 && x.size(-1) == plan.k * (activation >= 0 ? 2 : 1), name, ": x has to end in ", plan.k * (activation >= 0 ? 2 : 1), " features, got ", x.sizes());
    TORCH_CHECK(!grouped || x.dim() == 2, name, ": x has to be [rows, features], got ", x.sizes());
    TORCH_CHECK(scale.device() == device && scale.scalar_type() == at::kFloat && scale.sizes() == weight.sizes().slice(0, weight.dim() - 1), name,
                ": weight_scale has to be float32 of shape ", weight.sizes().slice(0, weight.dim() - 1), " on ", device);
    TORCH_CHECK(!scale.requires_grad(), name, ": weights are fixed codes: weight_scale cannot require a gradient");
    TORCH_CHECK(plan.out_type == at::kFloat || plan.out_type == at::kBFloat16 || plan.out_type == at::kHalf, name, ": dtype has to be float32, bfloat16 or float16, not ", plan.out_type);
    if (bias.defined()) {
        check_float(name, "bias", bias, device);
        TORCH_CHECK(bias.sizes() == at::IntArrayRef({plan.n}), name, ": bias has to be of shape [", plan.n, "], got ", bias.sizes());
        plan.bias_type = bias.scalar_type();
    }
    if (grouped)
        TORCH_CHECK(offsets.device() == device && offsets.scalar_type() == at::kInt && offsets.sizes() == at::IntArrayRef({plan.groups + 1}), name,
                    ": offsets have to be int32 of shape [", plan.groups + 1, "] on ", device);
    if (weight_t.defined()) {
        std::vector<int64_t> turned = weight.sizes().vec();
        std::swap(turned[turned.size() - 1], turned[turned.size() - 2]);
        TORCH_CHECK(weight_t.scalar_type() == at::kChar && weight_t.device() == device && weight_t.sizes() == at::IntArrayRef(turned), name, ": weight_t has to be int8 of shape ",
                    at::IntArrayRef(turned), " on ", device);
    }
    const c10::DeviceGuard guard(device);
    const bool need = at::GradMode::is_enabled() && (x.requires_grad() || wants(bias));
    TORCH_CHECK(!need || plan.n <= MOST_K, name, "'s gradient adds up at most ", MOST_K, " products, got ", plan.n);
    auto node = need ? std::shared_ptr<ProductBackward>(new ProductBackward(), torch::autograd::deleteNode) : nullptr;
    Tensor out, places;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        const viola_stream_t stream = stream_of(x);
        const Rows rows(x);
        plan.rows = rows.count;
        TORCH_CHECK(plan.rows < (int64_t{1} << 31), name, " takes fewer than 2^31 rows");
        std::vector<int64_t> result(x.sizes().begin(), x.sizes().end() - 1);
        result.push_back(plan.n);
        out = room(result, plan.out_type, device);
        if (grouped) places = offsets.contiguous();
        if (plan.rows) {
            const Codes w(weight, stream);
            const Tensor channels = scale.contiguous(), b = bias.defined() ? bias.contiguous() : Tensor();
            const float* channel_data = static_cast<const float*>(channels.const_data_ptr());
            int status = VIOLA_EUNSUPPORTED;
            if (!grouped && plan.rows <= 4) {                                // few rows: quantized on the way into the product
                status = VIOLA_TRY(viola_int8_rows_linear, rows.data(), rows.pitch, code_of(plan.x_type), plan.rows, plan.k, activation, w.data(), w.pitch, channel_data, plan.n,
                                   ptr(b), b.defined() ? code_of(b.scalar_type()) : VIOLA_F32, out.mutable_data_ptr(), code_of(plan.out_type), stream);
                if (status != VIOLA_EUNSUPPORTED) check("viola_int8_rows_linear", status);
            }
            if (status == VIOLA_EUNSUPPORTED) {
                const int64_t pitch = ceil_to(plan.k, 16);
                Arena temp;
                const int64_t scales_at = temp.take(plan.rows * 4), codes_at = temp.take(plan.rows * pitch);
                temp.make(device);
                VIOLA_CALL(viola_int8_quantize, rows.data(), rows.pitch, code_of(plan.x_type), plan.rows, plan.k, activation, nullptr, nullptr, 0, temp.as<int8_t>(codes_at), pitch,
                           temp.as<float>(scales_at), nullptr, stream);
                product(plan, temp.as<int8_t>(codes_at), pitch, temp.as<float>(scales_at), w, channel_data, places, b, plan.n, plan.k, out.mutable_data_ptr(), plan.out_type, stream);
            }
        }
    }
    if (need) {
        node->plan = plan;
        node->label = name;
        node->shape = x.sizes().vec();
        node->has_bias = bias.defined();
        node->has_turned = weight_t.defined() && x.requires_grad();
        if (x.requires_grad()) {
            if (node->has_turned) node->weight_t = SavedVariable(weight_t, false);
            else node->weight = SavedVariable(weight, false);
            if (activation >= 0) node->x = SavedVariable(x, false);
            node->scale = SavedVariable(scale, false);
            if (grouped) node->offsets = SavedVariable(places, false);
        }
        node->set_next_edges(torch::autograd::collect_next_edges(x, bias));
        torch::autograd::set_history(out, node);
    }
    return out;
}

variable_list ProductBackward::apply(variable_list&& grads) {
    check_once(label.c_str());
    variable_list result(2);
    const bool needs_x = task_should_compute_output(0), needs_bias = has_bias && task_should_compute_output(1);
    if (!grads[0].defined() || (!needs_x && !needs_bias)) return result;
    at::AutoDispatchBelowADInplaceOrView below;
    const Tensor& dy = grads[0];
    const at::Device device = dy.device();
    const c10::DeviceGuard guard(device);
    check_eager(label.c_str(), dy);
    const auto options = at::TensorOptions().device(device);
    if (!plan.rows) {
        if (needs_x) result[0] = at::empty(shape, options.dtype(plan.x_type));
        if (needs_bias) result[1] = at::zeros({plan.n}, options.dtype(plan.bias_type));
        return result;
    }
    const viola_stream_t stream = stream_of(dy);
    const Rows rows(dy);
    const int64_t pitch = ceil_to(plan.n, 16), parts = needs_bias ? viola_int8_sum_parts(plan.rows, plan.n) : 0;
    Arena temp;
    const int64_t scales_at = temp.take(plan.rows * 4), codes_at = temp.take(plan.rows * pitch), sums_at = temp.take(parts * plan.n * 4);
    temp.make(device);
    std::vector<int64_t> channel_shape;
    if (plan.groups) channel_shape.push_back(plan.groups);
    channel_shape.push_back(plan.n);
    // for a bias alone the channels' scales are not there, and any factors serve
    const Tensor channels = needs_x ? aligned(restored(scale, device, at::kFloat, channel_shape)) : at::ones({plan.n}, options.dtype(at::kFloat));
    const Tensor places = plan.groups ? restored(offsets, device, at::kInt, {plan.groups + 1}) : Tensor();
    VIOLA_CALL(viola_int8_quantize, rows.data(), rows.pitch, code_of(dy.scalar_type()), plan.rows, plan.n, -1, static_cast<const float*>(channels.const_data_ptr()),
               static_cast<const int32_t*>(ptr(places)), plan.groups, temp.as<int8_t>(codes_at), pitch, temp.as<float>(scales_at), needs_bias ? temp.as<float>(sums_at) : nullptr, stream);
    if (needs_bias) {
        result[1] = room({plan.n}, plan.bias_type, device);
        VIOLA_CALL(viola_column_reduce, temp.as<float>(sums_at), parts, plan.n, result[1].mutable_data_ptr(), code_of(plan.bias_type), stream);
    }
    if (!needs_x) return result;
    const Tensor w = has_turned ? weight_t.unpack() : weight.unpack();
    const int64_t turned[2] = {has_turned ? plan.k : plan.n, has_turned ? plan.n : plan.k};
    TORCH_CHECK(w.defined() && w.device() == device && w.scalar_type() == at::kChar && w.size(-2) == turned[0] && w.size(-1) == turned[1] &&
                    (plan.groups ? w.dim() == 3 && w.size(0) == plan.groups : w.dim() == 2), "a tensor saved by ", label, " came back changed");
    const Codes back = has_turned ? Codes(w, stream) : Codes::turned(w, stream);
    result[0] = room(shape, plan.x_type, device);
    const int8_t* codes = temp.as<int8_t>(codes_at);
    const float* scales = temp.as<float>(scales_at);
    if (plan.activation < 0) {
        product(plan, codes, pitch, scales, back, nullptr, places, Tensor(), plan.k, plan.n, result[0].mutable_data_ptr(), plan.x_type, stream);
        return result;
    }
    const Tensor z = x.unpack();
    TORCH_CHECK(z.defined() && z.device() == device && z.scalar_type() == plan.x_type && z.sizes() == at::IntArrayRef(shape), "a tensor saved by ", label, " came back changed");
    const Rows zr(z);
    const int status = VIOLA_TRY(viola_int8_gemm_gated_backward, codes, pitch, scales, back.data(), back.pitch, back.stride, static_cast<const int32_t*>(ptr(places)), plan.groups,
                                 plan.rows, plan.k, plan.n, zr.data(), zr.pitch, code_of(plan.x_type), plan.activation, result[0].mutable_data_ptr(), stream);
    if (status != VIOLA_EUNSUPPORTED) {
        check("viola_int8_gemm_gated_backward", status);
        return result;
    }
    const Tensor dh = room({plan.rows, plan.k}, at::kFloat, device);         // few rows, long sums
    product(plan, codes, pitch, scales, back, nullptr, places, Tensor(), plan.k, plan.n, dh.mutable_data_ptr(), at::kFloat, stream);
    VIOLA_CALL(viola_int8_gated_backward, zr.data(), zr.pitch, code_of(plan.x_type), plan.rows, plan.k, plan.activation, static_cast<const float*>(dh.const_data_ptr()),
               plan.groups ? static_cast<const int32_t*>(places.const_data_ptr()) + plan.groups : nullptr, result[0].mutable_data_ptr(), stream);
    return result;
}

std::tuple<Tensor, Tensor> quantize(const Tensor& x, int activation) {
    check_seen("quantize_int8", {x});
    const at::Device device = x.device();
    check_float("quantize_int8", "x", x, device);
    TORCH_CHECK(x.dim() >= 1 && x.size(-1) > 0 && (activation < 0 || x.size(-1) % 2 == 0), "quantize_int8: x needs a last dimension of features", activation < 0 ? "" : ", [g | u]",
                ", got ", x.sizes());
    const c10::DeviceGuard guard(device);
    at::AutoDispatchBelowADInplaceOrView below;
    const Rows rows(x);
    const int64_t cols = x.size(-1) / (activation < 0 ? 1 : 2), pitch = ceil_to(cols, 16);
    std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end() - 1);
    const Tensor scales = room(shape, at::kFloat, device);
    shape.push_back(pitch);
    Tensor codes = room(shape, at::kChar, device);
    if (rows.count)
        VIOLA_CALL(viola_int8_quantize, rows.data(), rows.pitch, code_of(x.scalar_type()), rows.count, cols, activation, nullptr, nullptr, 0,
                   static_cast<int8_t*>(codes.mutable_data_ptr()), pitch, static_cast<float*>(scales.mutable_data_ptr()), nullptr, stream_of(x));
    if (pitch != cols) codes = codes.narrow(-1, 0, cols);
    return {codes, scales};
}

}  // namespace

void viola_host::register_int8(py::module_& m) {
    m.def("quantize_int8", torch::wrap_pybind_function([](const Tensor& x, int activation) {
        py::gil_scoped_release release;
        return quantize(x, activation);
    }));
    // (name, x, weight, weight_scale, bias, offsets, activation, dtype, weight_t) -> y
    m.def("int8_product", torch::wrap_pybind_function([](const std::string& name, const Tensor& x, const Tensor& weight, const Tensor& scale, const std::optional<Tensor>& bias,
                                                         const std::optional<Tensor>& offsets, int activation, const py::object& dtype, const std::optional<Tensor>& weight_t) {
        std::optional<at::ScalarType> type;
        if (!dtype.is_none()) type = torch::python::detail::py_object_to_dtype(dtype);
        py::gil_scoped_release release;
        return run(name.c_str(), x, weight, scale, or_none(bias), or_none(offsets), activation, type, or_none(weight_t));
    }));
}
