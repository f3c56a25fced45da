// ops.embedding and ops.linear_cross_entropy as operators of torch with native gradient nodes, the lists of tensors that clipping takes, and
// what only torch's own side can tell about a graph.
//
// A gradient node written in Python runs its Python on autograd's own thread, whose core holds none of the interpreter's objects: a
// small lookup's step took 92 us of which the GPU needs 15 - 35, and takes 53 as written here (a node that does nothing: 41).  This file only
// moves tensors to the C entry points of libphc_hip.so, which the Python layer hands over once (phc_torch_bind): it is linked to torch, not to
// the engine.
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
    decltype(&phc_linear_xent_fwd) xent_fwd = nullptr;
    decltype(&phc_linear_xent_bwd) xent_bwd = nullptr;
    decltype(&phc_linear_xent_state_bytes) xent_state_bytes = nullptr;
    decltype(&phc_linear_xent_ws_bytes) xent_ws_bytes = nullptr;
    decltype(&phc_grad_norm_ws_bytes) norm_ws_bytes = nullptr;
    decltype(&phc_grad_norm_clip) norm_clip = nullptr;
    decltype(&phc_last_error) last_error = nullptr;
} engine;

// a 2-D tensor the kernels can read in place: unit column stride, rows that do not overlap; anything else is copied
at::Tensor rows(const at::Tensor &t) {
    return t.stride(1) == 1 && (t.stride(0) >= t.size(1) || t.size(0) == 1) ? t : t.contiguous();
}
int64_t row_stride(const at::Tensor &t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }
const int64_t *words(const at::Tensor &t) { return t.numel() ? t.const_data_ptr<int64_t>() : nullptr; }
int dtype_id(at::ScalarType t) { return t == at::kFloat ? PHC_DTYPE_F32 : t == at::kBFloat16 ? PHC_DTYPE_BF16 : PHC_DTYPE_F16; }

void check(int rc, const char *who) { TORCH_CHECK(rc == 0, who, " failed (", rc, "): ", engine.last_error()); }
void *stream_of(const at::Tensor &t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

// gradients that were asked for with a graph of their own: the refusal comes when that graph is used
void refuse_twice(const char *who, torch::autograd::variable_list &grads) {
    torch::autograd::variable_list known;
    for (const at::Tensor &g : grads)
        if (g.defined()) known.push_back(g.set_requires_grad(true));
    const auto refusal = std::make_shared<torch::autograd::DelayedError>(
        std::string(who) + ": its gradient is once_differentiable, second derivatives are not offered (detach it where what follows does not require gradients)",
        (int64_t)known.size());
    known = (*refusal)(std::move(known));
    size_t k = 0;
    for (at::Tensor &g : grads)
        if (g.defined()) g = known[k++];
}

struct Embedding : torch::autograd::Function<Embedding> {
    static at::Tensor forward(torch::autograd::AutogradContext *ctx, const at::Tensor &tokens, const at::Tensor &weight, double scale, int64_t pad) {
        const at::Tensor w = rows(weight);
        const int64_t N = tokens.numel(), V = w.size(0), D = w.size(1);
        const c10::DeviceGuard guard(w.device());
        std::vector<int64_t> sizes = tokens.sizes().vec();
        sizes.push_back(D);
        at::Tensor out = at::empty(sizes, w.options());
        check(engine.fwd(words(tokens), w.const_data_ptr(), N, V, D, row_stride(w), dtype_id(w.scalar_type()), (float)scale, out.data_ptr(),
                         stream_of(w)),
              "phc_embedding_fwd");
        ctx->save_for_backward({tokens});
        ctx->saved_data["call"] = std::vector<int64_t>{V, D, (int64_t)w.scalar_type(), pad};
        ctx->saved_data["scale"] = scale;
        return out;
    }

    static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx, torch::autograd::variable_list grads) {
        const bool again = at::GradMode::is_enabled() && grads[0].requires_grad();       // (linear in grads[0], and does not depend on the table)
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
                             dw.data_ptr(), ws.data_ptr(), bytes, stream_of(tokens)),
                  "phc_embedding_bwd");
        }
        torch::autograd::variable_list out{at::Tensor(), dw, at::Tensor(), at::Tensor()};
        if (again) refuse_twice("embedding", out);
        return out;
    }
};

struct LinearCrossEntropy : torch::autograd::Function<LinearCrossEntropy> {
    static phc_linear_xent_desc describe(const at::Tensor &x, const at::Tensor &w, const at::Tensor &bias, const at::Tensor &target, const at::Tensor &state,
                                         int64_t ignore, int64_t reduction, int64_t piece) {
        phc_linear_xent_desc d{};
        d.N = x.size(0), d.D = x.size(1), d.V = w.size(0);
        d.ldx = row_stride(x), d.ldw = row_stride(w);
        d.ignore_index = ignore, d.piece = piece;
        d.dtype = dtype_id(x.scalar_type()), d.reduction = (int32_t)reduction;
        d.x = x.const_data_ptr(), d.W = w.const_data_ptr(), d.bias = bias.defined() ? bias.const_data_ptr() : nullptr;
        d.target = target.const_data_ptr<int64_t>();
        d.state = state.data_ptr();
        return d;
    }
    static at::Tensor workspace(phc_linear_xent_desc &d, int backward, const at::TensorOptions &bytes) {
        const size_t n = engine.xent_ws_bytes(&d, backward);
        TORCH_CHECK(n, "phc_linear_xent: ", engine.last_error());
        at::Tensor ws = at::empty({(int64_t)n}, bytes);
        d.ws = ws.data_ptr(), d.ws_bytes = n;
        return ws;
    }

    static at::Tensor forward(torch::autograd::AutogradContext *ctx, const at::Tensor &x, const at::Tensor &weight, const std::optional<at::Tensor> &bias,
                              const at::Tensor &target, int64_t ignore, int64_t reduction, int64_t piece) {
        const int64_t N = target.numel(), D = weight.size(1);
        const c10::DeviceGuard guard(x.device());
        const at::TensorOptions f32 = x.options().dtype(at::kFloat), bytes = x.options().dtype(at::kByte);
        at::Tensor w = rows(weight);
        if (row_stride(w) > (1 << 22)) w = w.contiguous();           // (32-bit offsets inside a tile of rows)
        const at::Tensor x2 = rows(x.reshape({N, D})), b = bias && bias->defined() ? bias->contiguous() : at::Tensor();
        ctx->saved_data["call"] = std::vector<int64_t>{ignore, reduction, piece, b.defined()};
        ctx->saved_data["shape"] = x.sizes().vec();
        if (N == 0) {
            ctx->save_for_backward({x2, w, b, at::Tensor(), at::Tensor()});
            return reduction == PHC_REDUCE_NONE ? at::zeros(target.sizes(), f32)
                                                : at::full({}, reduction == PHC_REDUCE_MEAN ? std::numeric_limits<double>::quiet_NaN() : 0.0, f32);
        }
        const at::Tensor t = target.reshape({N}).contiguous();
        at::Tensor loss = reduction == PHC_REDUCE_NONE ? at::empty(target.sizes(), f32) : at::empty({}, f32);
        const at::Tensor state = at::empty({(int64_t)engine.xent_state_bytes(N)}, bytes);
        phc_linear_xent_desc d = describe(x2, w, b, t, state, ignore, reduction, piece);
        d.loss = loss.data_ptr<float>();
        const at::Tensor ws = workspace(d, 0, bytes);
        check(engine.xent_fwd(&d, stream_of(x)), "phc_linear_xent_fwd");
        ctx->save_for_backward({x2, w, b, t, state});
        return loss;
    }

    static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx, torch::autograd::variable_list grads) {
        const bool again = at::GradMode::is_enabled();               // (they depend on x, W and b, one of which asks for gradients, whatever grads[0] does)
        const auto call = ctx->saved_data["call"].toIntVector(), shape = ctx->saved_data["shape"].toIntVector();
        at::Tensor dx, dw, db;
        {
            const at::NoGradGuard no_grad;
            const auto saved = ctx->get_saved_variables();
            const at::Tensor &x = saved[0], &w = saved[1], &b = saved[2], &t = saved[3], &state = saved[4];
            const c10::DeviceGuard guard(w.device());
            const bool none = !state.defined();                  // no rows
            if (ctx->needs_input_grad(0)) dx = none ? at::zeros(shape, w.options()) : at::empty(shape, w.options());
            if (ctx->needs_input_grad(1)) dw = none ? at::zeros(w.sizes(), w.options()) : at::empty(w.sizes(), w.options());
            if (call[3] && ctx->needs_input_grad(2)) db = none ? at::zeros(b.sizes(), w.options()) : at::empty(b.sizes(), w.options());
            if (!none) {
                const at::Tensor g = grads[0].to(at::kFloat).contiguous();
                phc_linear_xent_desc d = describe(x, w, b, t, state, call[0], call[1], call[2]);
                d.dloss = g.const_data_ptr<float>();
                d.dx = dx.defined() ? dx.data_ptr() : nullptr, d.dW = dw.defined() ? dw.data_ptr() : nullptr, d.db = db.defined() ? db.data_ptr() : nullptr;
                const at::Tensor ws = workspace(d, 1, w.options().dtype(at::kByte));
                check(engine.xent_bwd(&d, stream_of(w)), "phc_linear_xent_bwd");
            }
        }
        torch::autograd::variable_list out{dx, dw, db, at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
        if (again) refuse_twice("linear_cross_entropy", out);
        return out;
    }
};

at::Tensor embedding(const at::Tensor &tokens, const at::Tensor &weight, double scale, int64_t pad) {
    TORCH_CHECK(engine.fwd, "embedding: the engine is not bound");
    return Embedding::apply(tokens, weight, scale, pad);
}

at::Tensor linear_cross_entropy(const at::Tensor &x, const at::Tensor &weight, const std::optional<at::Tensor> &bias, const at::Tensor &target, int64_t ignore,
                                int64_t reduction, int64_t piece) {
    TORCH_CHECK(engine.xent_fwd, "linear_cross_entropy: the engine is not bound");
    return LinearCrossEntropy::apply(x, weight, bias, target, ignore, reduction, piece);
}

bool known_type(const at::Tensor &t) {
    const at::ScalarType s = t.scalar_type();
    return s == at::kFloat || s == at::kBFloat16 || s == at::kHalf;
}

// {norm, coefficient, scratch}.  mode 0: the norm, 1: grads scaled in place, 2: into out.  Layouts that the kernels do not take ("phc_layout")
// are the Python layer's to name or to copy.
at::Tensor norm_clip(at::TensorList grads, at::TensorList out, int64_t mode, double max_norm, int64_t kind) {
    TORCH_CHECK(engine.norm_clip && !grads.empty() && (mode != 2 || out.size() == grads.size()), "norm_clip: bad call");
    const size_t n = grads.size();
    const at::TensorList &results = mode == 2 ? out : grads;
    std::vector<const void *> src(n);
    std::vector<void *> dst(n);
    std::vector<int64_t> numel(n);
    std::vector<int32_t> types(n), out_types(n);
    const c10::Device device = grads[0].device();
    for (size_t i = 0; i < n; ++i) {
        const at::Tensor &g = grads[i], &o = results[i];
        TORCH_CHECK(g.layout() == at::kStrided && o.layout() == at::kStrided && g.is_cuda() && g.device() == device && o.device() == device && known_type(g) &&
                        known_type(o) && (mode == 2 ? g.is_contiguous() && o.is_contiguous() && g.sizes() == o.sizes() : g.is_non_overlapping_and_dense()),
                    "phc_layout");
        src[i] = g.const_data_ptr();
        dst[i] = mode ? o.data_ptr() : nullptr;
        numel[i] = g.numel();
        types[i] = dtype_id(g.scalar_type());
        out_types[i] = dtype_id(o.scalar_type());
    }
    const c10::DeviceGuard guard(device);
    const size_t bytes = engine.norm_ws_bytes((int)n, numel.data());
    at::Tensor res = at::empty({(int64_t)(2 + bytes / 4)}, grads[0].options().dtype(at::kFloat));
    float *at = res.data_ptr<float>();
    check(engine.norm_clip((int)n, src.data(), numel.data(), types.data(), (int)kind, max_norm, mode ? dst.data() : nullptr, mode ? out_types.data() : nullptr, at,
                           at + 2, bytes, stream_of(res)),
          "phc_grad_norm_clip");
    if (mode)
        for (const at::Tensor &o : results)
            if (!o.is_inference()) o.unsafeGetTensorImpl()->bump_version();
    return res;
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
extern "C" void phc_torch_bind(void *const *entry) {
    engine.fwd = reinterpret_cast<decltype(engine.fwd)>(entry[0]);
    engine.bwd = reinterpret_cast<decltype(engine.bwd)>(entry[1]);
    engine.ws_bytes = reinterpret_cast<decltype(engine.ws_bytes)>(entry[2]);
    engine.xent_fwd = reinterpret_cast<decltype(engine.xent_fwd)>(entry[3]);
    engine.xent_bwd = reinterpret_cast<decltype(engine.xent_bwd)>(entry[4]);
    engine.xent_state_bytes = reinterpret_cast<decltype(engine.xent_state_bytes)>(entry[5]);
    engine.xent_ws_bytes = reinterpret_cast<decltype(engine.xent_ws_bytes)>(entry[6]);
    engine.norm_ws_bytes = reinterpret_cast<decltype(engine.norm_ws_bytes)>(entry[7]);
    engine.norm_clip = reinterpret_cast<decltype(engine.norm_clip)>(entry[8]);
    engine.last_error = reinterpret_cast<decltype(engine.last_error)>(entry[9]);
}

TORCH_LIBRARY(phc_gnn_amd, m) {
    m.def("embedding(Tensor tokens, Tensor weight, float scale, int pad) -> Tensor", &embedding);
    m.def("linear_cross_entropy(Tensor x, Tensor weight, Tensor? bias, Tensor target, int ignore_index, int reduction, int piece) -> Tensor",
          &linear_cross_entropy);
    m.def("norm_clip(Tensor[] grads, Tensor[] out, int mode, float max_norm, int kind) -> Tensor", &norm_clip);
    m.def("gradient_on_another_stream(Tensor leaf) -> bool", &gradient_on_another_stream);
}
