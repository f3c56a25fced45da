// ops.embedding as an operator of torch with a native gradient node, and what only torch's own side can tell about a graph.
//
// A gradient node written in Python runs its Python on autograd's own thread, whose core holds none of the interpreter's objects: a
// small lookup's step took 92 us of which the GPU needs 15 - 35 (a node that does nothing: 40 us).  This file only moves tensors
// to the C entry points of libphc_hip.so, which the Python layer hands over once (phc_torch_bind): it is linked to torch, not to the engine.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/VirtualGuardImpl.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/library.h>

#include "phc_hip.h"

namespace {

struct Engine {
    decltype(&phc_embedding_fwd) fwd = nullptr;
    decltype(&phc_embedding_bwd) bwd = nullptr;
    decltype(&phc_embedding_bwd_ws_bytes) ws_bytes = nullptr;
    decltype(&phc_last_error) last_error = nullptr;
} engine;

// a 2-D tensor the kernels can read in place: unit column stride, rows that do not overlap; anything else is copied
at::Tensor rows(const at::Tensor &t) {
    return t.stride(1) == 1 && (t.stride(0) >= t.size(1) || t.size(0) == 1) ? t : t.contiguous();
}
int64_t row_stride(const at::Tensor &t) { return std::max(t.stride(0), t.size(1)); }
const int64_t *words(const at::Tensor &t) { return t.numel() ? t.const_data_ptr<int64_t>() : nullptr; }
int dtype_id(at::ScalarType t) { return t == at::kFloat ? PHC_DTYPE_F32 : t == at::kBFloat16 ? PHC_DTYPE_BF16 : PHC_DTYPE_F16; }

void check(int rc, const char *who) { TORCH_CHECK(rc == 0, who, " failed (", rc, "): ", engine.last_error()); }

struct Embedding : torch::autograd::Function<Embedding> {
    static at::Tensor forward(torch::autograd::AutogradContext *ctx, const at::Tensor &tokens, const at::Tensor &weight, double scale, int64_t pad) {
        const at::Tensor w = rows(weight);
        const int64_t N = tokens.numel(), V = w.size(0), D = w.size(1);
        const c10::DeviceGuard guard(w.device());
        std::vector<int64_t> sizes = tokens.sizes().vec();
        sizes.push_back(D);
        at::Tensor out = at::empty(sizes, w.options());
        check(engine.fwd(words(tokens), w.const_data_ptr(), N, V, D, row_stride(w), dtype_id(w.scalar_type()), (float)scale, out.data_ptr(),
                         c10::hip::getCurrentHIPStream(w.get_device()).stream()),
              "phc_embedding_fwd");
        ctx->save_for_backward({tokens});
        ctx->saved_data["call"] = std::vector<int64_t>{V, D, (int64_t)w.scalar_type(), pad};
        ctx->saved_data["scale"] = scale;
        return out;
    }

    static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx, torch::autograd::variable_list grads) {
        const bool again = at::GradMode::is_enabled() && grads[0].requires_grad();
        at::Tensor dw;
        {
            const at::NoGradGuard no_grad;
            const at::Tensor tokens = ctx->get_saved_variables()[0];
            const auto call = ctx->saved_data["call"].toIntVector();
            const int64_t N = tokens.numel(), V = call[0], D = call[1], pad = call[3];
            const auto type = (at::ScalarType)call[2];
            const c10::DeviceGuard guard(tokens.device());
            const at::Tensor dy = rows(grads[0].to(type).reshape({N, D}));
            dw = at::empty({V, D}, dy.options());
            const size_t bytes = engine.ws_bytes(N, V, D);
            const at::Tensor ws = at::empty({(int64_t)bytes}, dy.options().dtype(at::kByte));
            check(engine.bwd(words(tokens), N ? dy.const_data_ptr() : nullptr, N, V, D, row_stride(dy), dtype_id(type), (float)ctx->saved_data["scale"].toDouble(), pad,
                             dw.data_ptr(), ws.data_ptr(), bytes, c10::hip::getCurrentHIPStream(tokens.get_device()).stream()),
                  "phc_embedding_bwd");
        }
        if (again) {
            const auto refusal = std::make_shared<torch::autograd::DelayedError>(
                "embedding: its gradient is once_differentiable, second derivatives are not offered", 1);
            dw = (*refusal)({dw.set_requires_grad(true)})[0];
        }
        return {at::Tensor(), dw, at::Tensor(), at::Tensor()};
    }
};

at::Tensor embedding(const at::Tensor &tokens, const at::Tensor &weight, double scale, int64_t pad) {
    TORCH_CHECK(engine.fwd, "embedding: the engine is not bound");
    return Embedding::apply(tokens, weight, scale, pad);
}

// whether a live graph ends in this leaf whose gradient node belongs to another stream than the current one
bool gradient_on_another_stream(const at::Tensor &leaf) {
    const auto node = torch::autograd::impl::try_get_grad_accumulator(leaf);
    if (!node) return false;
    const auto stream = node->stream();
    return stream && *stream != c10::impl::VirtualGuardImpl(leaf.device().type()).getStream(leaf.device());
}

}  // namespace

// the engine's entry points, from the library that the Python layer has loaded
extern "C" void phc_torch_bind(void *fwd, void *bwd, void *ws_bytes, void *last_error) {
    engine.fwd = reinterpret_cast<decltype(engine.fwd)>(fwd);
    engine.bwd = reinterpret_cast<decltype(engine.bwd)>(bwd);
    engine.ws_bytes = reinterpret_cast<decltype(engine.ws_bytes)>(ws_bytes);
    engine.last_error = reinterpret_cast<decltype(engine.last_error)>(last_error);
}

TORCH_LIBRARY(phc_gnn_amd, m) {
    m.def("embedding(Tensor tokens, Tensor weight, float scale, int pad) -> Tensor", &embedding);
    m.def("gradient_on_another_stream(Tensor leaf) -> bool", &gradient_on_another_stream);
}
