// Argument checks, autograd and launches of the training operators.
#include "training.h"

#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <cmath>
#include <cstring>
#include <limits>

#include "hgemm_sm100_train.h"

namespace {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

int64_t round8(int64_t n) { return (n + 7) / 8 * 8; }

void check_matrix(const Tensor& t, const char* name, const Tensor& x) {
    TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
    TORCH_CHECK(t.device() == x.device(), name, " must be on the same CUDA device as x");
    TORCH_CHECK(t.scalar_type() == x.scalar_type(), name, " must have the dtype of x");
    TORCH_CHECK(t.dim() == 2, name, " must be two-dimensional, got ", t.dim(), " dimensions");
}

void check_input(const Tensor& x) {
    TORCH_CHECK(x.is_cuda(), "x must be a CUDA tensor");
    TORCH_CHECK(x.scalar_type() == torch::kFloat16 || x.scalar_type() == torch::kBFloat16,
                "x must have dtype torch.float16 or torch.bfloat16");
    TORCH_CHECK(x.dim() >= 1, "x must have at least one dimension");
}

// The values in memory: torch may hold a tensor negated by a bit alone (the
// imaginary part of a conjugate).
Tensor as_stored(const Tensor& t) { return t.is_neg() ? t.resolve_neg() : t; }

// A [rows, cols] operand as the kernels take it: unit column stride, 16-byte
// aligned rows, both sides padded with zeros to what is asked for. The tensor
// itself where it already is that, else a copy. `dense`: no gap between rows.
Tensor operand(const Tensor& t, int64_t rows, int64_t cols, bool dense) {
    Tensor r = as_stored(t);
    if (t.size(0) != rows || t.size(1) != cols)
        r = torch::constant_pad_nd(r, {0, cols - t.size(1), 0, rows - t.size(0)});
    const int64_t ld = r.stride(0);
    const bool as_is = r.stride(1) == 1 && (ld == cols || (!dense && ld > cols && ld % 8 == 0)) &&
                       reinterpret_cast<uintptr_t>(r.data_ptr()) % 16 == 0;
    // A dense view at an odd offset is contiguous already: clone, not contiguous().
    return as_is ? r : r.clone(torch::MemoryFormat::Contiguous);
}

Tensor cut(const Tensor& t, int64_t rows, int64_t cols) {
    if (t.size(0) == rows && t.size(1) == cols) return t;
    return t.narrow(0, 0, rows).narrow(1, 0, cols).contiguous();
}

// Where kernels of this process record a wait that ran out: a word in host memory
// that every device can write, so that the next call finds it without waiting for
// the device. Never freed: captured graphs hold its address.
volatile int32_t* status_word() {
    static int32_t* const word = [] {
        // Allowed while another stream is captured; the allocation is no part of it.
        cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
        C10_CUDA_CHECK(cudaThreadExchangeStreamCaptureMode(&mode));
        void* p = nullptr;
        const cudaError_t rc = cudaHostAlloc(&p, 64, cudaHostAllocPortable | cudaHostAllocMapped);
        C10_CUDA_CHECK(cudaThreadExchangeStreamCaptureMode(&mode));
        C10_CUDA_CHECK(rc);
        std::memset(p, 0, 64);
        return static_cast<int32_t*>(p);
    }();
    return word;
}

HgemmSm100TrainCommon common_of(const Tensor& x) {
    const int32_t failed = training_status(true);
    TORCH_CHECK(failed == HGEMM_SM100_OK, "a kernel of an earlier call of the training operators failed (",
                hgemm_sm100_status_string(failed), "); what it returned, and what came of it, is not valid");
    HgemmSm100TrainCommon c{};
    c.status = const_cast<int32_t*>(status_word());
    c.dtype = x.scalar_type() == torch::kBFloat16 ? HGEMM_SM100_TRAIN_BF16 : HGEMM_SM100_TRAIN_F16;
    return c;
}

void check_status(int rc, const char* what) {
    TORCH_CHECK(rc == HGEMM_SM100_OK, what, " failed: ", hgemm_sm100_status_string(rc));
}

void no_double_backward(const char* what) {
    // Gradient mode is on inside a backward pass only under create_graph=True.
    TORCH_CHECK(!torch::GradMode::is_enabled(), what, " has no second derivative (create_graph=True)");
}

// A dual tensor needs no requires_grad: without this its tangent would be dropped,
// which reads as zero.
void no_forward_mode(const char* what, std::initializer_list<const Tensor*> tensors) {
    for (const Tensor* t : tensors)
        TORCH_CHECK(!t->_fw_grad(/*level=*/0).defined(), what, " has no forward-mode derivative");
}

// A gradient goes on to the node of its leaf, which lives on as long as any graph
// of that leaf does, on the stream where the first of them was recorded. In a
// capture the engine makes that stream wait for the captured one and joins it
// again at the end, which any other stream can do (torch.cuda.make_graphed_callables
// leaves its warm-up's there). The legacy default stream can be no part of a
// capture: there the engine's wait ends the process, so it is refused here.
void check_capture(const char* what) {
    using c10::cuda::CaptureStatus;
    if (c10::cuda::currentStreamCaptureStatusMayInitCtx() == CaptureStatus::None) return;
    const auto node = torch::autograd::get_current_node();
    if (node == nullptr) return;
    for (uint32_t i = 0; i < node->num_outputs(); ++i) {
        if (!node->task_should_compute_output(i)) continue;
        const std::optional<c10::Stream> next = node->next_edge(i).function->stream();
        if (!next.has_value()) continue;
        const cudaStream_t stream = c10::cuda::CUDAStream(*next).stream();
        TORCH_CHECK(stream != nullptr && stream != cudaStreamLegacy, what,
                    " backward cannot be captured into a CUDA graph while a graph of the same tensors from the default "
                    "stream is alive: delete its outputs first");
    }
}

// An uninitialised tensor on the device of `like`, without the dispatcher's way.
Tensor fresh(at::IntArrayRef shape, torch::ScalarType dtype, const Tensor& like) {
    return at::detail::empty_cuda(shape, dtype, like.device(), std::nullopt);
}

Tensor bytes(size_t n, const Tensor& like) { return fresh({static_cast<int64_t>(n)}, torch::kUInt8, like); }

// [tokens, n] view of an activation.
Tensor rows_of(const Tensor& t, int64_t tokens, int64_t n) { return t.dim() == 2 ? t : t.reshape({tokens, n}); }

// ------------------------------------------------------------ feed-forward --

struct FfnSizes {
    int64_t tokens, hidden, inter, out;      // as the caller has them
    int64_t hidden8, inter8, out8;           // as the kernels take them
};

FfnSizes ffn_sizes(const Tensor& x, const Tensor& gate, const Tensor& down) {
    FfnSizes s{};
    s.hidden = gate.size(1);
    s.inter = gate.size(0);
    s.out = down.size(0);
    s.tokens = x.numel() / s.hidden;
    s.hidden8 = round8(s.hidden);
    s.inter8 = round8(s.inter);
    s.out8 = round8(s.out);
    return s;
}

struct FfnForward {
    Tensor y;
    Tensor kept;   // [tokens, inter] (h), or [3, tokens, inter]: h, silu(g), u silu'(g); padded sizes
};

FfnForward ffn_forward(const Tensor& x, const Tensor& gate, const Tensor& up, const Tensor& down, const FfnSizes& s,
                       bool keep) {
    const c10::cuda::CUDAGuard device_guard(x.device());
    const Tensor xp = operand(rows_of(x, s.tokens, s.hidden), s.tokens, s.hidden8, false);
    const Tensor gp = operand(gate, s.inter8, s.hidden8, true), up_ = operand(up, s.inter8, s.hidden8, true);
    const Tensor dp = operand(down, s.out8, s.inter8, true);
    FfnForward r;
    const torch::ScalarType dtype = x.scalar_type();
    const int64_t plane = s.tokens * s.inter8 * 2;   // a multiple of 16 bytes
    r.y = fresh({s.tokens, s.out8}, dtype, x);
    r.kept = keep ? fresh({3, s.tokens, s.inter8}, dtype, x) : fresh({s.tokens, s.inter8}, dtype, x);
    uint8_t* kept = static_cast<uint8_t*>(r.kept.data_ptr());
    HgemmSm100FfnForward a{};
    a.common = common_of(x);
    a.x = xp.data_ptr();
    a.gate = gp.data_ptr();
    a.up = up_.data_ptr();
    a.down = dp.data_ptr();
    a.y = r.y.data_ptr();
    a.h = kept;
    a.silu = keep ? kept + plane : nullptr;
    a.slope = keep ? kept + 2 * plane : nullptr;
    a.tokens = s.tokens;
    a.hidden = s.hidden8;
    a.inter = s.inter8;
    a.out = s.out8;
    a.ldx = xp.stride(0);
    Tensor ws;
    if ((a.workspace_bytes = hgemm_sm100_ffn_forward_workspace(&a)) > 0) {
        ws = bytes(a.workspace_bytes, x);
        a.workspace = ws.data_ptr();
    }
    check_status(hgemm_sm100_ffn_forward(&a, c10::cuda::getCurrentCUDAStream(x.get_device()).stream()), "gated_ffn");
    return r;
}

std::vector<int64_t> with_last(const Tensor& x, int64_t n) {
    std::vector<int64_t> shape = x.sizes().vec();
    shape.back() = n;
    return shape;
}

class GatedFfn : public torch::autograd::Function<GatedFfn> {
  public:
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& gate, const Tensor& up,
                          const Tensor& down) {
        const FfnSizes s = ffn_sizes(x, gate, down);
        FfnForward r = ffn_forward(x, gate, up, down, s, true);
        ctx->save_for_backward({x, gate, up, down, r.kept});
        const Tensor y = cut(r.y, s.tokens, s.out);
        return x.dim() == 2 ? y : y.view(with_last(x, s.out));
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        no_double_backward("gated_ffn");
        const variable_list v = ctx->get_saved_variables();
        const Tensor &x = v[0], &gate = v[1], &up = v[2], &down = v[3];
        const FfnSizes s = ffn_sizes(x, gate, down);
        if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
        const c10::cuda::CUDAGuard device_guard(x.device());
        check_capture("gated_ffn");
        const Tensor dy = operand(rows_of(grads[0], s.tokens, s.out), s.tokens, s.out8, false);
        const Tensor xp = operand(rows_of(x, s.tokens, s.hidden), s.tokens, s.hidden8, false);
        const Tensor gp = operand(gate, s.inter8, s.hidden8, true), up_ = operand(up, s.inter8, s.hidden8, true);
        const Tensor dp = operand(down, s.out8, s.inter8, true);
        const bool need_x = ctx->needs_input_grad(0), need_g = ctx->needs_input_grad(1);
        const bool need_u = ctx->needs_input_grad(2), need_d = ctx->needs_input_grad(3);
        const torch::ScalarType dtype = x.scalar_type();
        const int64_t plane = s.tokens * s.inter8 * 2;
        const uint8_t* kept = static_cast<const uint8_t*>(v[4].const_data_ptr());
        const Tensor pre = fresh({2, s.tokens, s.inter8}, dtype, x);
        Tensor dx, dgate, dup, ddown;
        if (need_x) dx = fresh({s.tokens, s.hidden8}, dtype, x);
        if (need_g) dgate = fresh({s.inter8, s.hidden8}, dtype, x);
        if (need_u) dup = fresh({s.inter8, s.hidden8}, dtype, x);
        if (need_d) ddown = fresh({s.out8, s.inter8}, dtype, x);
        HgemmSm100FfnBackward a{};
        a.common = common_of(x);
        a.dy = dy.data_ptr();
        a.x = xp.data_ptr();
        a.gate = gp.data_ptr();
        a.up = up_.data_ptr();
        a.down = dp.data_ptr();
        a.h = kept;
        a.silu = kept + plane;
        a.slope = kept + 2 * plane;
        a.dgate_pre = pre.data_ptr();
        a.dup_pre = static_cast<uint8_t*>(pre.data_ptr()) + plane;
        a.dx = need_x ? dx.data_ptr() : nullptr;
        a.dgate = need_g ? dgate.data_ptr() : nullptr;
        a.dup = need_u ? dup.data_ptr() : nullptr;
        a.ddown = need_d ? ddown.data_ptr() : nullptr;
        a.tokens = s.tokens;
        a.hidden = s.hidden8;
        a.inter = s.inter8;
        a.out = s.out8;
        a.ldx = xp.stride(0);
        a.lddy = dy.stride(0);
        Tensor ws;
        if ((a.workspace_bytes = hgemm_sm100_ffn_backward_workspace(&a)) > 0) {
            ws = bytes(a.workspace_bytes, x);
            a.workspace = ws.data_ptr();
        }
        check_status(hgemm_sm100_ffn_backward(&a, c10::cuda::getCurrentCUDAStream(x.get_device()).stream()),
                     "gated_ffn backward");
        if (need_x) dx = cut(dx, s.tokens, s.hidden);
        if (need_x && x.dim() != 2) dx = dx.view(x.sizes());
        if (need_g) dgate = cut(dgate, s.inter, s.hidden);
        if (need_u) dup = cut(dup, s.inter, s.hidden);
        if (need_d) ddown = cut(ddown, s.out, s.inter);
        return {dx, dgate, dup, ddown};
    }
};

// ------------------------------------------------------------ cross entropy --

struct LossForward {
    Tensor loss, lse;
};

LossForward loss_forward(const Tensor& x, const Tensor& weight, const Tensor& target, int64_t tokens,
                         int32_t reduction, int64_t ignore_index) {
    const c10::cuda::CUDAGuard device_guard(x.device());
    const int64_t hidden = weight.size(1), hidden8 = round8(hidden);
    const Tensor xp = operand(rows_of(x, tokens, hidden), tokens, hidden8, false);
    const Tensor wp = operand(weight, weight.size(0), hidden8, true);
    LossForward r;
    r.lse = fresh({tokens}, torch::kFloat32, x);
    r.loss = reduction == HGEMM_SM100_LOSS_NONE ? fresh({tokens}, torch::kFloat32, x) : fresh({}, torch::kFloat32, x);
    HgemmSm100LossForward a{};
    a.common = common_of(x);
    a.x = xp.data_ptr();
    a.weight = wp.data_ptr();
    a.target = target.data_ptr<int64_t>();
    a.loss = r.loss.data_ptr<float>();
    a.lse = r.lse.data_ptr<float>();
    a.tokens = tokens;
    a.hidden = hidden8;
    a.vocab = weight.size(0);
    a.ldx = xp.stride(0);
    a.ignore_index = ignore_index;
    a.reduction = reduction;
    a.workspace_bytes = hgemm_sm100_loss_forward_workspace(&a);
    const Tensor ws = bytes(a.workspace_bytes, x);
    a.workspace = ws.data_ptr();
    check_status(hgemm_sm100_loss_forward(&a, c10::cuda::getCurrentCUDAStream(x.get_device()).stream()),
                 "linear_cross_entropy");
    return r;
}

class LinearCrossEntropy : public torch::autograd::Function<LinearCrossEntropy> {
  public:
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const Tensor& target,
                          int64_t tokens, int64_t reduction, int64_t ignore_index) {
        LossForward r = loss_forward(x, weight, target, tokens, static_cast<int32_t>(reduction), ignore_index);
        ctx->save_for_backward({x, weight, target, r.lse});
        ctx->saved_data["reduction"] = reduction;
        ctx->saved_data["ignore_index"] = ignore_index;
        return r.loss;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        no_double_backward("linear_cross_entropy");
        variable_list out(6);
        if (!grads[0].defined()) return out;
        const variable_list v = ctx->get_saved_variables();
        const Tensor &x = v[0], &weight = v[1], &target = v[2], &lse = v[3];
        const c10::cuda::CUDAGuard device_guard(x.device());
        check_capture("linear_cross_entropy");
        const int64_t tokens = target.numel(), hidden = weight.size(1), hidden8 = round8(hidden);
        const Tensor xp = operand(rows_of(x, tokens, hidden), tokens, hidden8, false);
        const Tensor wp = operand(weight, weight.size(0), hidden8, true);
        const Tensor dloss = as_stored(grads[0]).contiguous();
        const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1);
        Tensor dx, dw;
        if (need_x) dx = fresh({tokens, hidden8}, x.scalar_type(), x);
        if (need_w) dw = fresh({weight.size(0), hidden8}, x.scalar_type(), x);
        HgemmSm100LossBackward a{};
        a.common = common_of(x);
        a.x = xp.data_ptr();
        a.weight = wp.data_ptr();
        a.target = target.data_ptr<int64_t>();
        a.lse = lse.data_ptr<float>();
        a.dloss = dloss.data_ptr<float>();
        a.dx = need_x ? dx.data_ptr() : nullptr;
        a.dweight = need_w ? dw.data_ptr() : nullptr;
        a.tokens = tokens;
        a.hidden = hidden8;
        a.vocab = weight.size(0);
        a.ldx = xp.stride(0);
        a.ignore_index = ctx->saved_data["ignore_index"].toInt();
        a.reduction = static_cast<int32_t>(ctx->saved_data["reduction"].toInt());
        a.workspace_bytes = hgemm_sm100_loss_backward_workspace(&a);
        const Tensor ws = bytes(a.workspace_bytes, x);
        a.workspace = ws.data_ptr();
        check_status(hgemm_sm100_loss_backward(&a, c10::cuda::getCurrentCUDAStream(x.get_device()).stream()),
                     "linear_cross_entropy backward");
        if (need_x) out[0] = cut(dx, tokens, hidden);
        if (need_x && x.dim() != 2) out[0] = out[0].view(x.sizes());
        if (need_w) out[1] = cut(dw, weight.size(0), hidden);
        return out;
    }
};

}  // namespace

int64_t training_status_address() { return static_cast<int64_t>(reinterpret_cast<uintptr_t>(status_word())); }

int32_t training_status(bool clear) {
    volatile int32_t* const word = status_word();
    const int32_t value = *word;
    if (clear && value != 0) *word = 0;
    return value;
}

Tensor gated_ffn(const Tensor& x, const Tensor& gate, const Tensor& up, const Tensor& down) {
    no_forward_mode("gated_ffn", {&x, &gate, &up, &down});
    check_input(x);
    check_matrix(gate, "gate", x);
    check_matrix(up, "up", x);
    check_matrix(down, "down", x);
    TORCH_CHECK(gate.sizes() == up.sizes(), "gate and up must have the same shape");
    TORCH_CHECK(x.size(-1) == gate.size(1), "x.shape[-1]=", x.size(-1), " must match gate.shape[1]=", gate.size(1));
    TORCH_CHECK(down.size(1) == gate.size(0), "down.shape[1]=", down.size(1), " must match gate.shape[0]=",
                gate.size(0));
    TORCH_CHECK(gate.numel() > 0 && down.numel() > 0, "the weights must not be empty");
    if (x.numel() == 0) {
        // No tokens: nothing to launch; zero gradients through plain products.
        const Tensor x2 = x.reshape({0, x.size(-1)});
        const Tensor h = torch::silu(torch::matmul(x2, gate.t())) * torch::matmul(x2, up.t());
        return torch::matmul(h, down.t()).view(with_last(x, down.size(0)));
    }
    const bool keep = torch::GradMode::is_enabled() && (x.requires_grad() || gate.requires_grad() ||
                                                        up.requires_grad() || down.requires_grad());
    if (keep) return GatedFfn::apply(x, gate, up, down);
    const FfnSizes s = ffn_sizes(x, gate, down);
    return cut(ffn_forward(x, gate, up, down, s, false).y, s.tokens, s.out).view(with_last(x, s.out));
}

Tensor linear_cross_entropy(const Tensor& x, const Tensor& weight, const Tensor& target, const std::string& reduction,
                            int64_t ignore_index) {
    no_forward_mode("linear_cross_entropy", {&x, &weight});
    check_input(x);
    check_matrix(weight, "weight", x);
    TORCH_CHECK(weight.numel() > 0, "weight must not be empty");
    TORCH_CHECK(x.size(-1) == weight.size(1), "x.shape[-1]=", x.size(-1), " must match weight.shape[1]=",
                weight.size(1));
    TORCH_CHECK(target.is_cuda() && target.device() == x.device(), "target must be on the same CUDA device as x");
    TORCH_CHECK(target.scalar_type() == torch::kInt64 || target.scalar_type() == torch::kInt32,
                "target must have dtype torch.int64 or torch.int32");
    TORCH_CHECK(target.sizes() == x.sizes().slice(0, x.dim() - 1), "target must have the shape of x without its last "
                "dimension");
    const int32_t kind = reduction == "none"   ? HGEMM_SM100_LOSS_NONE
                         : reduction == "mean" ? HGEMM_SM100_LOSS_MEAN
                         : reduction == "sum"  ? HGEMM_SM100_LOSS_SUM
                                               : -1;
    TORCH_CHECK(kind >= 0, "unknown reduction '", reduction, "' (none, mean, sum)");
    const int64_t tokens = target.numel();
    if (tokens == 0) {
        const Tensor each = (x.reshape({0, x.size(-1)}).to(torch::kFloat32).sum(-1) +
                             weight.to(torch::kFloat32).sum() * 0).view(target.sizes());
        return kind == HGEMM_SM100_LOSS_NONE ? each : kind == HGEMM_SM100_LOSS_MEAN ? each.mean() : each.sum();
    }
    const c10::cuda::CUDAGuard device_guard(x.device());
    Tensor flat = target.dim() == 1 ? target : target.reshape({tokens});
    if (flat.scalar_type() != torch::kInt64) flat = flat.to(torch::kInt64);
    flat = as_stored(flat).contiguous();
    const bool keep = torch::GradMode::is_enabled() && (x.requires_grad() || weight.requires_grad());
    const Tensor loss = keep ? LinearCrossEntropy::apply(x, weight, flat, tokens, static_cast<int64_t>(kind),
                                                         ignore_index)
                             : loss_forward(x, weight, flat, tokens, kind, ignore_index).loss;
    return kind == HGEMM_SM100_LOSS_NONE && target.dim() != 1 ? loss.view(target.sizes()) : loss;
}

Tensor orthogonalize(const Tensor& g, int64_t steps, double a, double b, double c, double eps) {
    TORCH_CHECK(g.is_cuda(), "g must be a CUDA tensor");
    TORCH_CHECK(g.scalar_type() == torch::kFloat16 || g.scalar_type() == torch::kBFloat16,
                "g must have dtype torch.float16 or torch.bfloat16");
    TORCH_CHECK(g.dim() >= 2, "g must have at least two dimensions, got ", g.dim());
    TORCH_CHECK(steps >= 0 && steps <= 1000, "steps must be between 0 and 1000, got ", steps);
    TORCH_CHECK(std::isfinite(a) && std::isfinite(b) && std::isfinite(c), "coefficients must be finite");
    TORCH_CHECK(eps >= 0 && std::isfinite(eps), "eps must be finite and not negative");
    const torch::NoGradGuard no_grad;
    const c10::cuda::CUDAGuard device_guard(g.device());
    const Tensor out = fresh(g.sizes(), g.scalar_type(), g);
    if (g.numel() == 0) return out;
    const int64_t rows = g.size(-2), cols = g.size(-1), batch = g.numel() / (rows * cols);
    TORCH_CHECK(batch <= 65535, "at most 65535 matrices in one call, got ", batch);
    Tensor m = as_stored(g.detach()).reshape({batch, rows, cols});
    if (m.stride(2) != 1 || m.stride(1) < cols || m.stride(0) < 0) m = m.contiguous();
    HgemmSm100Orthogonalize args{};
    args.common = common_of(g);
    args.g = m.data_ptr();
    args.out = out.data_ptr();
    args.batch = batch;
    args.rows = rows;
    args.cols = cols;
    args.ldg = rows > 1 ? m.stride(1) : cols;
    args.batch_stride = batch > 1 ? m.stride(0) : 0;
    args.steps = static_cast<int32_t>(steps);
    args.a = static_cast<float>(a);
    args.b = static_cast<float>(b);
    args.c = static_cast<float>(c);
    args.eps = eps;
    Tensor ws;
    if ((args.workspace_bytes = hgemm_sm100_orthogonalize_workspace(&args)) > 0) {
        ws = bytes(args.workspace_bytes, g);
        args.workspace = ws.data_ptr();
    }
    check_status(hgemm_sm100_orthogonalize(&args, c10::cuda::getCurrentCUDAStream(g.get_device()).stream()),
                 "orthogonalize");
    return out;
}
