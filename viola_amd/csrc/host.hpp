// Shared by the native host files (host.cpp: modules, host_blocks.cpp: norms around a block and routing, host_int8.cpp: products of 8-bit
// integers, host_optim.cpp: optimizer and wire codec): calling the library's entry points, tensor helpers, arenas.
#pragma once
#include <torch/extension.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/saved_variable.h>

#include <ATen/hip/EmptyTensor.h>

#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>

#include <atomic>
#include <memory>
#include <optional>
#include <string>
#include <vector>

#include "../../include/viola_hip.h"

namespace viola_host {

namespace py = pybind11;
using at::Tensor;

// ---------------------------------------------------------------------------------------------------- calls
// Instrumented mode (the `timeline` of viola_amd._lib): every call is bracketed by two timing events on the current stream.
inline std::atomic<bool> recording{false};
// the list and torch.cuda.Event; process-wide and never released (the interpreter may be gone before static destructors run)
inline py::object* timeline_sink = nullptr;
inline py::object* event_class = nullptr;

inline void check(const char* name, int status) {
    TORCH_CHECK(status == 0, name, " failed: ", viola_error_string(status), " (status ", status, ")");
}

template <typename F>
int timed(const char* name, F&& f) {
    if (__builtin_expect(!recording.load(std::memory_order_relaxed), 1)) return f();
    py::gil_scoped_acquire gil;
    if (!timeline_sink || timeline_sink->is_none()) return f();
    py::object start = (*event_class)(py::arg("enable_timing") = true), end = (*event_class)(py::arg("enable_timing") = true);
    start.attr("record")();
    const int status = f();
    end.attr("record")();
    timeline_sink->attr("append")(py::make_tuple(name, start, end));
    return status;
}
// VIOLA_CALL raises on a non-zero status, VIOLA_TRY hands VIOLA_EUNSUPPORTED back to a caller that has another route
#define VIOLA_CALL(fn, ...) check(#fn, timed(#fn, [&] { return fn(__VA_ARGS__); }))
#define VIOLA_TRY(fn, ...) timed(#fn, [&] { return fn(__VA_ARGS__); })

inline int code_of(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return VIOLA_F32;
        case at::kBFloat16: return VIOLA_BF16;
        case at::kHalf: return VIOLA_F16;
        case at::kFloat8_e4m3fn: return VIOLA_E4M3;
        case at::kFloat8_e5m2: return VIOLA_E5M2;
        default: TORCH_CHECK(false, "viola_amd kernels do not take tensors of type ", t);
    }
}

inline viola_stream_t stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
inline const void* ptr(const Tensor& t) { return t.defined() && t.numel() ? t.const_data_ptr() : nullptr; }
inline int64_t ceil_to(int64_t n, int64_t unit) { return (n + unit - 1) / unit * unit; }
inline int64_t ceil_div(int64_t n, int64_t unit) { return (n + unit - 1) / unit; }

// Several buffers of one lifetime as one allocation: take() reserves, make() allocates, at() hands out addresses.
class Arena {
public:
    int64_t take(int64_t bytes) {
        const int64_t begin = size_;
        size_ += ceil_to(bytes, 256);
        return begin;
    }
    void make(const at::Device& device) {
        if (size_) buffer_ = at::empty({size_}, at::TensorOptions().dtype(at::kByte).device(device));
    }
    void* at(int64_t offset) const { return static_cast<char*>(buffer_.mutable_data_ptr()) + offset; }
    template <typename T> T* as(int64_t offset) const { return static_cast<T*>(at(offset)); }
    void release() { buffer_ = Tensor(); }
    const Tensor& tensor() const { return buffer_; }
    int64_t size() const { return size_; }

private:
    int64_t size_ = 0;
    Tensor buffer_;
};

inline bool holds(const Tensor& t, const at::Device& device, at::ScalarType type, at::IntArrayRef sizes) {
    return t.defined() && t.device() == device && t.scalar_type() == type && t.sizes() == sizes && t.is_contiguous();
}

// A tensor subclass with its own dispatch, or a dual number of forward-mode differentiation, whose tangent would be lost here.
inline bool plain(const Tensor& t) { return !t.defined() || (!t.unsafeGetTensorImpl()->is_python_dispatch() && !t._fw_grad(0).defined()); }

// Raises where what runs here would not be seen by who has to see it: derivatives and transforms that have no rule for it, and whatever records a graph of
// operators (torch.jit.trace, make_fx, fake tensors), in which this call's result would stand as a constant for every input. Modes of a program's own that only
// watch (a counter of operations, selective checkpointing) are no obstacle: to them these kernels are as any code below the dispatcher.
inline void check_seen(const char* name, at::ArrayRef<Tensor> tensors) {
    using c10::DispatchKey;
    using c10::impl::TorchDispatchModeKey;
    bool transformed = c10::impl::tls_is_dispatch_key_included(DispatchKey::FuncTorchDynamicLayerFrontMode);
    for (const Tensor& t : tensors) transformed = transformed || !plain(t);
    TORCH_CHECK_NOT_IMPLEMENTED(!transformed, name, " has neither forward-mode derivatives nor rules for functorch transforms");
    bool recorded = c10::impl::tls_is_dispatch_key_included(DispatchKey::Tracer) || c10::impl::tls_is_dispatch_key_included(DispatchKey::PreDispatch);
    if (c10::impl::dispatch_mode_enabled())
        for (const auto mode : {TorchDispatchModeKey::FAKE, TorchDispatchModeKey::PROXY, TorchDispatchModeKey::FUNCTIONAL})
            recorded = recorded || c10::impl::TorchDispatchModeTLS::get_mode(mode).has_value();
    TORCH_CHECK_NOT_IMPLEMENTED(!recorded, name, " cannot be recorded into a graph of operators: its result would be a constant there");
}

// A tensor that was saved for backward, as it comes back: a saved-tensor hook may have moved it or made another of it.
inline Tensor restored(const torch::autograd::SavedVariable& saved, const at::Device& device, at::ScalarType type, at::IntArrayRef sizes) {
    const Tensor t = saved.unpack();
    TORCH_CHECK(t.defined() && t.device() == device && t.scalar_type() == type && t.sizes() == sizes, "a tensor saved by a viola module came back changed");
    return t.contiguous();
}

inline void check_float(const char* name, const char* what, const Tensor& t, const at::Device& device) {
    TORCH_CHECK(t.is_cuda(), "viola_amd kernels run on the GPU only");
    TORCH_CHECK(t.device() == device, name, ": ", what, " is on ", t.device(), ", not on ", device);
    const at::ScalarType type = t.scalar_type();
    TORCH_CHECK(type == at::kFloat || type == at::kBFloat16 || type == at::kHalf, name, ": ", what, " has to be float32, bfloat16 or float16, not ", type);
}

// The gradients of these nodes are computed by kernels that autograd does not see.
inline void check_once(const char* name) { TORCH_CHECK_NOT_IMPLEMENTED(!at::GradMode::is_enabled(), name, " can be differentiated once only (create_graph is not supported)"); }
// A backward pass under capture ends the process where an eager graph of the same leaves lives (its accumulators stand on another stream), which a node cannot see: refused, by
// every node around a block and of 8-bit integers. (Gradients that autograd hands to leaves before it reaches the first of these nodes are out of their sight.)
inline void check_eager(const char* name, const Tensor& t) {
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    TORCH_CHECK(hipStreamIsCapturing(static_cast<hipStream_t>(stream_of(t)), &status) == hipSuccess, name, " could not ask for the state of its stream");
    TORCH_CHECK(status == hipStreamCaptureStatusNone, name, ": a backward pass cannot be captured into a graph (a forward pass can)");
}

// Memory for a result: the allocator at once, without the dispatcher's two rounds (a router has up to eight results and workspaces, and a
// decoding step's call of it takes as long on the host as on the GPU).
inline Tensor room(at::IntArrayRef sizes, at::ScalarType type, const at::Device& device) { return Tensor(at::detail::empty_cuda(sizes, type, device, std::nullopt)); }

inline bool wants(const Tensor& t) { return t.defined() && t.requires_grad(); }

// A tensor as rows of its last dimension with one distance between them; copied where it has none, and where rows overlap: those of a
// broadcast dimension, whose distance is 0, too (autograd hands out such gradients: that of a sum over tokens repeats every row).
struct Rows {
    Tensor holder;
    int64_t count, cols, pitch;
    explicit Rows(const Tensor& t) : holder(t), count(1), cols(t.size(-1)), pitch(cols) {
        for (int64_t i = 0; i + 1 < t.dim(); ++i) count *= t.size(i);
        bool whole = cols <= 1 || t.stride(-1) == 1, first = true;
        int64_t expected = 0;                                    // distance of a dimension's rows where all inside of it lie `pitch` apart
        for (int64_t i = t.dim() - 2; i >= 0 && whole; --i) {
            if (t.size(i) == 1) continue;
            if (first) pitch = t.stride(i);
            whole = pitch >= cols && (first || t.stride(i) == expected);
            expected = t.stride(i) * t.size(i);
            first = false;
        }
        if (!whole) {
            holder = t.contiguous();
            pitch = cols;
        }
    }
    const void* data() const { return ptr(holder); }
};

inline Tensor or_none(const std::optional<Tensor>& t) { return t ? *t : Tensor(); }

void register_optimizer(py::module_& m);                         // host_optim.cpp
void register_blocks(py::module_& m);                            // host_blocks.cpp
void register_int8(py::module_& m);                              // host_int8.cpp

}  // namespace viola_host
