// Shared by the native host files (host.cpp: modules, host_blocks.cpp: norms around a block and routing, host_optim.cpp: optimizer and
// wire codec): calling the library's entry points, tensor helpers, arenas.
#pragma once
#include <torch/extension.h>
#include <torch/csrc/autograd/saved_variable.h>

#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>

#include <atomic>
#include <memory>
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

void register_optimizer(py::module_& m);                         // host_optim.cpp
void register_blocks(py::module_& m);                            // host_blocks.cpp

}  // namespace viola_host
