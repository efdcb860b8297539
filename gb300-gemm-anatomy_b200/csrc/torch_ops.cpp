// torch operators over the C ABI, for calls whose cost is the host's: argument
// checks, allocation and differentiation without the interpreter. The entry
// points of libb200gemm.so are handed over by the Python loader (bind), so both
// bindings always use the same library.
//
// b200gemm::vocab_loss is the losses at the vocabulary projection
// (b200_vocab_loss_forward / _backward) as one differentiable operator. A small
// training step is bound by the host: 230 us as a Python autograd.Function,
// of which 60 us on the GPU; see b200gemm/vocab_loss.py for its public form.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <cstring>
#include <optional>

#include "b200gemm.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct EntryPoints {
    decltype(&b200_vocab_loss_info) info = nullptr;
    decltype(&b200_vocab_loss_forward) forward = nullptr;
    decltype(&b200_vocab_loss_backward) backward = nullptr;
    decltype(&b200_last_error) last_error = nullptr;
};
EntryPoints g_api;

void bind(int64_t info, int64_t forward, int64_t backward, int64_t last_error) {
    g_api.info = reinterpret_cast<decltype(g_api.info)>(info);
    g_api.forward = reinterpret_cast<decltype(g_api.forward)>(forward);
    g_api.backward = reinterpret_cast<decltype(g_api.backward)>(backward);
    g_api.last_error = reinterpret_cast<decltype(g_api.last_error)>(last_error);
}

void check_rc(int rc, const char* what) {
    TORCH_CHECK(rc == B200_OK, what, " failed (code ", rc, "): ", g_api.last_error());
}

// Rows of the operand: contiguous inside, a multiple of 16 bytes apart.
int64_t row_pitch(const Tensor& t, const char* name) {
    const int64_t rows = t.size(0), d = t.size(1);
    if (rows <= 1) return d;
    TORCH_CHECK_VALUE(t.stride(0) >= d && t.stride(0) % 8 == 0, name,
                      " rows must be a multiple of 8 elements apart and not overlap, strides ", t.strides());
    return t.stride(0);
}

int64_t operand_code(at::ScalarType t) { return t == at::kHalf ? B200_VL_F16 : B200_VL_BF16; }

struct Problem {
    B200VocabLossDesc desc;
    B200VocabLossInfo info;
};

// The description travels from the forward to the backward pass in saved_data,
// as bytes: the sizes and pitches are those that the forward pass checked.
c10::IValue pack(const Problem& p) { return std::string(reinterpret_cast<const char*>(&p), sizeof(p)); }
Problem unpack(const c10::IValue& v) {
    Problem p;
    std::memcpy(&p, v.toStringRef().data(), sizeof(p));
    return p;
}

Tensor workspace(int64_t bytes, const Tensor& like) { return at::empty({bytes}, like.options().dtype(at::kByte)); }

struct VocabLoss : public torch::autograd::Function<VocabLoss> {
    static Tensor forward(AutogradContext* ctx, const Tensor& hidden, const Tensor& weight, const Tensor& index,
                          const std::optional<Tensor>& teacher, int64_t ignore_index, int64_t reduction,
                          double temperature) {
        const int64_t rows = hidden.size(0);
        const bool per_row = reduction == B200_VL_NONE;
        const auto f32 = hidden.options().dtype(at::kFloat);
        ctx->saved_data["empty"] = rows == 0;
        if (rows == 0) {
            ctx->save_for_backward({hidden, weight});
            return per_row ? at::empty({0}, f32) : at::zeros({}, f32);
        }
        Problem p{};
        B200VocabLossDesc& d = p.desc;
        d.rows = rows;
        d.vocab = weight.size(0);
        d.hidden = weight.size(1);
        d.ld_hidden = row_pitch(hidden, "hidden");
        d.ld_weight = row_pitch(weight, "weight");
        d.dtype = operand_code(hidden.scalar_type());
        d.index_bytes = index.element_size();
        d.ignore_index = ignore_index;
        d.reduction = reduction;
        d.temperature = temperature;
        if (teacher) {
            d.top = d.ld_index = d.ld_teacher = teacher->size(1);
            d.teacher_dtype = teacher->scalar_type() == at::kFloat ? static_cast<int64_t>(B200_VL_F32)
                                                                   : operand_code(teacher->scalar_type());
        }
        const c10::cuda::CUDAGuard guard(hidden.device());
        check_rc(g_api.info(&d, at::cuda::getCurrentDeviceProperties()->multiProcessorCount, &p.info),
                 "b200_vocab_loss_info");
        Tensor loss = per_row ? at::empty({rows}, f32) : at::empty({}, f32);
        Tensor lse = at::empty({rows}, f32), target_logp = at::empty({rows, teacher ? d.top : 1}, f32);
        Tensor ws = workspace(p.info.workspace_forward, hidden);
        check_rc(g_api.forward(&d, hidden.const_data_ptr(), weight.const_data_ptr(), index.const_data_ptr(),
                               teacher ? teacher->const_data_ptr() : nullptr, loss.mutable_data_ptr<float>(),
                               lse.mutable_data_ptr<float>(), target_logp.mutable_data_ptr<float>(), ws.mutable_data_ptr(), p.info.workspace_forward,
                               c10::cuda::getCurrentCUDAStream().stream()),
                 "b200_vocab_loss_forward");
        ctx->save_for_backward({hidden, weight, index, teacher.value_or(Tensor()), lse, target_logp});
        ctx->saved_data["problem"] = pack(p);
        return loss;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        TORCH_CHECK(!at::GradMode::is_enabled(),
                    "the losses at the vocabulary projection are differentiable once (create_graph=True)");
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &hidden = saved[0], &weight = saved[1];
        const bool want_h = ctx->needs_input_grad(0), want_w = ctx->needs_input_grad(1);
        Tensor dh, dw;
        if (ctx->saved_data["empty"].toBool()) {
            if (want_h) dh = at::zeros(hidden.sizes(), hidden.options());
            if (want_w) dw = at::zeros(weight.sizes(), weight.options());
            return {dh, dw, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
        }
        const Problem p = unpack(ctx->saved_data["problem"]);
        const Tensor &index = saved[2], &teacher = saved[3], &lse = saved[4], &target_logp = saved[5];
        const c10::cuda::CUDAGuard guard(hidden.device());
        const Tensor grad = grads[0].to(at::kFloat).contiguous();
        if (want_h) dh = at::empty(hidden.sizes(), hidden.options());
        if (want_w) dw = at::empty(weight.sizes(), weight.options());
        if (want_h || want_w) {
            Tensor ws = workspace(p.info.workspace_backward, hidden);
            check_rc(g_api.backward(&p.desc, hidden.const_data_ptr(), weight.const_data_ptr(), index.const_data_ptr(),
                                    teacher.defined() ? teacher.const_data_ptr() : nullptr,
                                    lse.const_data_ptr<float>(), target_logp.const_data_ptr<float>(),
                                    grad.const_data_ptr<float>(),
                                    want_h ? dh.mutable_data_ptr() : nullptr, want_w ? dw.mutable_data_ptr() : nullptr,
                                    ws.mutable_data_ptr(), p.info.workspace_backward,
                                    c10::cuda::getCurrentCUDAStream().stream()),
                     "b200_vocab_loss_backward");
        }
        return {dh, dw, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

bool is_operand(at::ScalarType t) { return t == at::kBFloat16 || t == at::kHalf; }
bool is_index(at::ScalarType t) { return t == at::kInt || t == at::kLong; }

Tensor vocab_loss(const Tensor& hidden, const Tensor& weight, const Tensor& index, const std::optional<Tensor>& teacher,
                  int64_t ignore_index, int64_t reduction, double temperature) {
    TORCH_CHECK(g_api.forward != nullptr, "the entry points of libb200gemm.so are not bound");
    TORCH_CHECK_VALUE(is_operand(hidden.scalar_type()), "hidden must be bfloat16 or float16, got ", hidden.scalar_type());
    TORCH_CHECK_VALUE(weight.scalar_type() == hidden.scalar_type(), "weight must be ", hidden.scalar_type(),
                      " like hidden, got ", weight.scalar_type());
    TORCH_CHECK_VALUE(hidden.dim() >= 1 && weight.dim() == 2 && hidden.size(-1) == weight.size(1),
                      "hidden (... x D) and weight (V x D) do not match: shapes ", hidden.sizes(), " and ", weight.sizes());
    const int64_t d = weight.size(1);
    TORCH_CHECK_VALUE(weight.size(0) >= 1 && d >= 1 && d % 8 == 0, "weight has shape ", weight.sizes(),
                      ": V and D must be positive and D a multiple of 8 (rows of whole 16-byte units)");
    TORCH_CHECK_VALUE(hidden.numel() == 0 || hidden.stride(-1) == 1,
                      "hidden must have contiguous rows (D innermost), strides ", hidden.strides());
    TORCH_CHECK_VALUE(weight.stride(1) == 1, "weight must have contiguous rows (D innermost), strides ", weight.strides());
    const auto lead = hidden.sizes().slice(0, hidden.dim() - 1);
    if (teacher) {
        TORCH_CHECK_VALUE(teacher->scalar_type() == at::kFloat || is_operand(teacher->scalar_type()),
                          "teacher_logits must be float32, bfloat16 or float16, got ", teacher->scalar_type());
        TORCH_CHECK_VALUE(is_index(index.scalar_type()), "teacher_index must be int32 or int64, got ", index.scalar_type());
        TORCH_CHECK_VALUE(teacher->sizes() == index.sizes() && teacher->dim() == hidden.dim() &&
                              teacher->sizes().slice(0, teacher->dim() - 1) == lead,
                          "teacher_logits and teacher_index must both be ", lead, " x K, got ", teacher->sizes(), " and ",
                          index.sizes());
        TORCH_CHECK_VALUE(teacher->size(-1) >= 1 && teacher->size(-1) <= 256,
                          "a teacher's row holds 1 to 256 logits, got ", teacher->size(-1));
        TORCH_CHECK_VALUE(!teacher->requires_grad(), "teacher_logits gets no gradient: detach it");
        TORCH_CHECK_VALUE(temperature >= 0x1p-20 && temperature <= 0x1p20,
                          "temperature must be between 2^-20 and 2^20, got ", temperature);
    } else {
        TORCH_CHECK_VALUE(is_index(index.scalar_type()), "target must be int32 or int64, got ", index.scalar_type());
        TORCH_CHECK_VALUE(index.sizes() == lead, "target has shape ", index.sizes(), ", expected ", lead);
    }
    TORCH_CHECK_VALUE(hidden.is_cuda(), "hidden must live on a CUDA device, got ", hidden.device());
    TORCH_CHECK_VALUE(weight.device() == hidden.device(), "weight must be on ", hidden.device(), " like hidden, got ",
                      weight.device());
    TORCH_CHECK_VALUE(index.device() == hidden.device(), teacher ? "teacher_index" : "target", " must be on ",
                      hidden.device(), " like hidden, got ", index.device());
    TORCH_CHECK_VALUE(!teacher || teacher->device() == hidden.device(), "teacher_logits must be on ", hidden.device(),
                      " like hidden, got ", teacher ? teacher->device() : hidden.device());
    const Tensor h = hidden.dim() == 2 ? hidden : hidden.reshape({-1, d});
    for (const Tensor* t : {&h, &weight})
        TORCH_CHECK_VALUE(reinterpret_cast<uintptr_t>(t->const_data_ptr()) % 16 == 0, t == &h ? "hidden" : "weight",
                          " must start on a 16-byte boundary");
    Tensor loss;
    if (teacher) {
        const int64_t k = teacher->size(-1);
        loss = VocabLoss::apply(h, weight, index.reshape({-1, k}).contiguous(),
                                std::optional<Tensor>(teacher->reshape({-1, k}).contiguous()), ignore_index, reduction,
                                temperature);
    } else {
        loss = VocabLoss::apply(h, weight, index.dim() == 1 ? index.contiguous() : index.reshape({-1}).contiguous(),
                                std::optional<Tensor>(), ignore_index, reduction, temperature);
    }
    return reduction == B200_VL_NONE && hidden.dim() != 2 ? loss.reshape(lead) : loss;
}

}  // namespace

TORCH_LIBRARY(b200gemm, m) {
    m.def("bind(int info, int forward, int backward, int last_error) -> ()", &bind);
    m.def("vocab_loss(Tensor hidden, Tensor weight, Tensor index, Tensor? teacher, int ignore_index, int reduction, "
          "float temperature) -> Tensor",
          torch::dispatch(c10::DispatchKey::CompositeImplicitAutograd, &vocab_loss));
}
