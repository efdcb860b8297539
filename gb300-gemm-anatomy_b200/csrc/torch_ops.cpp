// torch operators over the C ABI, for calls whose cost is the host's: argument
// checks, allocation and differentiation without the interpreter. The entry
// points of libb200gemm.so are handed over by the Python loader (bind), so both
// bindings always use the same library.
//
// b200gemm::vocab_loss is the losses at the vocabulary projection
// (b200_vocab_loss_forward / _backward) as one differentiable operator. A small
// call is bound by the host: a training step took 230 us as a Python
// autograd.Function and takes 87 as this one, 38 on the GPU; a loss alone takes 12, on
// the GPU 12 to 14. Its public form is b200gemm/vocab_loss.py.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <algorithm>
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
bool rows_fit(const Tensor& t) { return t.size(0) <= 1 || (t.stride(0) >= t.size(1) && t.stride(0) % 8 == 0); }
bool starts_on_unit(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0; }
int64_t row_pitch(const Tensor& t, const char* name) {
    TORCH_CHECK_VALUE(rows_fit(t), name, " rows must be a multiple of 8 elements apart and not overlap, strides ",
                      t.strides());
    return t.size(0) <= 1 ? t.size(1) : t.stride(0);
}

// Tensors without storage of their own (FakeTensor, under torch.compile and
// torch.export, and other subclasses that take every call themselves) have nothing that
// a kernel could read.
void check_ordinary(const Tensor& t, const char* name) {
    TORCH_CHECK_TYPE(!t.key_set().has(c10::DispatchKey::Python), name,
                     " must be an ordinary tensor, got a subclass without storage of its own; the losses at the vocabulary "
                     "projection cannot be traced: call them through torch.compiler.disable");
}

// A tensor that the backward pass reads again. Saved-tensor hooks
// (torch.autograd.graph.save_on_cpu, a checkpoint) may give back the same values in
// another layout: the kernels go by the layout that is there now.
void check_saved(const Tensor& t, const char* name, at::IntArrayRef sizes, at::ScalarType type, at::Device device) {
    TORCH_CHECK(t.defined() && t.sizes() == sizes && t.scalar_type() == type && t.device() == device, name,
                " came back to the backward pass as another tensor than was saved: expected ", sizes, " ", type, " on ",
                device);
    check_ordinary(t, name);
}
Tensor as_saved(const Tensor& t, const char* name, at::IntArrayRef sizes, at::ScalarType type, at::Device device) {
    check_saved(t, name, sizes, type, device);
    return t.contiguous();
}
// The same for an operand, which may keep a pitch that the kernels can take.
Tensor as_saved_operand(const Tensor& t, const char* name, at::IntArrayRef sizes, at::ScalarType type, at::Device device) {
    check_saved(t, name, sizes, type, device);
    return t.stride(1) == 1 && rows_fit(t) && starts_on_unit(t) ? t : t.clone(at::MemoryFormat::Contiguous);
}

int64_t operand_code(at::ScalarType t) { return t == at::kHalf ? B200_VL_F16 : B200_VL_BF16; }

struct Problem {
    B200VocabLossDesc desc;
    B200VocabLossInfo info;
};

// The description travels from the forward to the backward pass in saved_data, as
// bytes. Its sizes hold there; its pitches are those of the tensors that the forward
// pass was given, and the backward pass takes its own from what comes back (see
// as_saved).
c10::IValue pack(const Problem& p) { return std::string(reinterpret_cast<const char*>(&p), sizeof(p)); }
Problem unpack(const c10::IValue& v) {
    Problem p;
    std::memcpy(&p, v.toStringRef().data(), sizeof(p));
    return p;
}

Tensor workspace(int64_t bytes, const Tensor& like) {
    Tensor ws = at::empty({bytes}, like.options().dtype(at::kByte));
    check_ordinary(ws, "the workspace");
    return ws;
}

int64_t align_up(int64_t a, int64_t b) { return (a + b - 1) / b * b; }

// The loss, and in `saved` what the backward pass reads again: per row the
// logarithm of the sum of exponentials, then the log-probabilities at the targets.
// Without a backward pass (null) they lie behind the workspace: an allocation is
// 0.8 us of a small call's 16.
Tensor forward_pass(Problem& p, const Tensor& hidden, const Tensor& weight, const Tensor& index,
                    const std::optional<Tensor>& teacher, int64_t ignore_index, int64_t reduction, double temperature,
                    Tensor* saved) {
    const int64_t rows = hidden.size(0);
    const bool per_row = reduction == B200_VL_NONE;
    const auto f32 = hidden.options().dtype(at::kFloat);
    if (rows == 0) return per_row ? at::empty({0}, f32) : at::zeros({}, f32);
    const c10::cuda::CUDAGuard guard(hidden.device());
    Tensor loss = per_row ? at::empty({rows}, f32) : at::empty({}, f32);
    check_ordinary(loss, "the result");
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
    check_rc(g_api.info(&d, at::cuda::getCurrentDeviceProperties()->multiProcessorCount, &p.info),
             "b200_vocab_loss_info");
    const int64_t kept = rows * (1 + (teacher ? d.top : 1)), behind = align_up(p.info.workspace_forward, 256);
    if (saved != nullptr) *saved = at::empty({kept}, f32);
    Tensor ws = workspace(saved != nullptr ? p.info.workspace_forward : behind + kept * 4, hidden);
    uint8_t* base = ws.mutable_data_ptr<uint8_t>();
    float* lse = saved != nullptr ? saved->mutable_data_ptr<float>() : reinterpret_cast<float*>(base + behind);
    check_rc(g_api.forward(&d, hidden.const_data_ptr(), weight.const_data_ptr(), index.const_data_ptr(),
                           teacher ? teacher->const_data_ptr() : nullptr, loss.mutable_data_ptr<float>(), lse, lse + rows,
                           base, p.info.workspace_forward, c10::cuda::getCurrentCUDAStream().stream()),
             "b200_vocab_loss_forward");
    return loss;
}

struct VocabLoss : public torch::autograd::Function<VocabLoss> {
    static Tensor forward(AutogradContext* ctx, const Tensor& hidden, const Tensor& weight, const Tensor& index,
                          const std::optional<Tensor>& teacher, int64_t ignore_index, int64_t reduction,
                          double temperature) {
        Problem p{};
        Tensor saved;
        const Tensor loss =
            forward_pass(p, hidden, weight, index, teacher, ignore_index, reduction, temperature, &saved);
        ctx->save_for_backward({hidden, weight, index, teacher.value_or(Tensor()), saved});
        ctx->saved_data["problem"] = pack(p);
        return loss;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        TORCH_CHECK(!at::GradMode::is_enabled(),
                    "the losses at the vocabulary projection are differentiable once (create_graph=True)");
        const variable_list saved = ctx->get_saved_variables();
        const bool want_h = ctx->needs_input_grad(0), want_w = ctx->needs_input_grad(1);
        Tensor dh, dw;
        Problem p = unpack(ctx->saved_data["problem"]);
        if (p.desc.rows == 0) {
            const Tensor &hidden = saved[0], &weight = saved[1];
            if (want_h) dh = at::zeros(hidden.sizes(), hidden.options());
            if (want_w) dw = at::zeros(weight.sizes(), weight.options());
            return {dh, dw, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
        }
        B200VocabLossDesc& d = p.desc;
        const at::Device device = grads[0].device();
        const c10::cuda::CUDAGuard guard(device);
        const at::ScalarType type = d.dtype == B200_VL_F16 ? at::kHalf : at::kBFloat16;
        const Tensor hidden = as_saved_operand(saved[0], "hidden", {d.rows, d.hidden}, type, device);
        const Tensor weight = as_saved_operand(saved[1], "weight", {d.vocab, d.hidden}, type, device);
        d.ld_hidden = row_pitch(hidden, "hidden");
        d.ld_weight = row_pitch(weight, "weight");
        const at::ScalarType index_type = d.index_bytes == 8 ? at::kLong : at::kInt;
        Tensor index, teacher;
        if (d.top > 0) {
            const at::ScalarType teacher_type = d.teacher_dtype == B200_VL_F32   ? at::kFloat
                                                : d.teacher_dtype == B200_VL_F16 ? at::kHalf
                                                                                 : at::kBFloat16;
            index = as_saved(saved[2], "teacher_index", {d.rows, d.top}, index_type, device);
            teacher = as_saved(saved[3], "teacher_logits", {d.rows, d.top}, teacher_type, device);
        } else {
            index = as_saved(saved[2], "target", {d.rows}, index_type, device);
        }
        const Tensor kept = as_saved(saved[4], "a result of the forward pass", {d.rows * (1 + std::max<int64_t>(d.top, 1))},
                                     at::kFloat, device);
        const float* lse = kept.const_data_ptr<float>();
        check_ordinary(grads[0], "the gradient of the loss");
        const Tensor grad = grads[0].to(at::kFloat).contiguous();
        if (want_h) dh = at::empty(hidden.sizes(), hidden.options());
        if (want_w) dw = at::empty(weight.sizes(), weight.options());
        if (want_h || want_w) {
            Tensor ws = workspace(p.info.workspace_backward, hidden);
            check_rc(g_api.backward(&p.desc, hidden.const_data_ptr(), weight.const_data_ptr(), index.const_data_ptr(),
                                    teacher.defined() ? teacher.const_data_ptr() : nullptr,
                                    lse, lse + p.desc.rows, grad.const_data_ptr<float>(),
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
    check_ordinary(hidden, "hidden");
    check_ordinary(weight, "weight");
    check_ordinary(index, teacher ? "teacher_index" : "target");
    if (teacher) check_ordinary(*teacher, "teacher_logits");
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
        TORCH_CHECK_VALUE(starts_on_unit(*t), t == &h ? "hidden" : "weight",
                          " must start on a 16-byte boundary");
    Tensor rows_index;
    std::optional<Tensor> rows_teacher;
    if (teacher) {
        const int64_t k = teacher->size(-1);
        rows_index = index.reshape({-1, k}).contiguous();
        rows_teacher = teacher->reshape({-1, k}).contiguous();
    } else {
        rows_index = (index.dim() == 1 ? index : index.reshape({-1})).contiguous();
    }
    Tensor loss;
    // Forward mode has to go through autograd too, which refuses it.
    const bool tangents = h._fw_grad(0).defined() || weight._fw_grad(0).defined();
    if (tangents || (at::GradMode::is_enabled() && (hidden.requires_grad() || weight.requires_grad()))) {
        loss = VocabLoss::apply(h, weight, rows_index, rows_teacher, ignore_index, reduction, temperature);
    } else {
        Problem p{};
        loss = forward_pass(p, h, weight, rows_index, rows_teacher, ignore_index, reduction, temperature, nullptr);
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
