// extern "C" entry points of the operators around the experts: norm, scored routing, dense
// products and gradient clipping. Argument checks, then the launches on the caller's stream;
// nothing here allocates, synchronises or throws.
#include <algorithm>

#include "linear.h"
#include "row_ops.h"

using namespace moe;

namespace {

template <typename Args>
int check_struct(const Args* args) {
    MOE_REQUIRE(args && args->struct_bytes == static_cast<int64_t>(sizeof(Args)), MOE_ERR_INVALID_ARGUMENT,
                "argument struct of another size");
    return MOE_OK;
}

int check_rows(int64_t tokens, int64_t hidden, int64_t dtype, int64_t most = kMaxNormWidth) {
    MOE_REQUIRE(valid_dtype(dtype), MOE_ERR_INVALID_ARGUMENT, "only FP32, FP16 and BF16 are supported");
    MOE_REQUIRE(tokens >= 0, MOE_ERR_INVALID_ARGUMENT, "tokens must be >= 0");
    MOE_REQUIRE(tokens <= kMaxLayerTokens, MOE_ERR_CAPACITY, "takes up to %lld tokens", (long long)kMaxLayerTokens);
    MOE_REQUIRE(hidden >= 1 && hidden <= most, MOE_ERR_UNSUPPORTED, "rows have 1..%lld elements", (long long)most);
    return MOE_OK;
}

int check_scored(int64_t tokens, int64_t experts, int64_t topk) {
    MOE_REQUIRE(tokens >= 0, MOE_ERR_INVALID_ARGUMENT, "tokens must be >= 0");
    MOE_REQUIRE(tokens <= kMaxLayerTokens, MOE_ERR_CAPACITY, "takes up to %lld tokens", (long long)kMaxLayerTokens);
    MOE_REQUIRE(experts >= 1 && experts <= kMaxScoredExperts, MOE_ERR_UNSUPPORTED, "scored routing supports 1..%d experts",
                kMaxScoredExperts);
    MOE_REQUIRE(topk >= 1 && topk <= kMaxTopk, MOE_ERR_UNSUPPORTED, "topk must be in 1..8");
    return MOE_OK;
}

bool valid_linear(int64_t tokens, int64_t hidden, int64_t width, int64_t activation, bool e4m3) {
    const int64_t unit = e4m3 ? 16 : 8;
    return tokens >= 0 && tokens <= kMaxLinearTokens && hidden >= unit && hidden % unit == 0 &&
           hidden <= kMaxLinearWidth && width >= 8 && width % 8 == 0 && width <= kMaxLinearWidth &&
           activation >= MOE_ACT_NONE && activation <= MOE_ACT_SWIGLU;
}

LinearArgs linear_shape(int64_t tokens, int64_t hidden, int64_t width, int64_t activation, bool e4m3) {
    LinearArgs a{};
    a.tokens = tokens;
    a.k_bytes = hidden * (e4m3 ? 1 : 2);
    a.n = width;
    a.rows = activation == MOE_ACT_SWIGLU ? 2 * width : width;
    a.fp8 = e4m3;
    a.activation = static_cast<int>(activation);
    return a;
}

}  // namespace

extern "C" {

int moe_rms_norm(const moe_rms_norm_args* p, void* stream) {
    int rc = check_struct(p);
    if (rc == MOE_OK) rc = check_rows(p->tokens, p->hidden, p->dtype);
    if (rc != MOE_OK) return rc;
    MOE_REQUIRE(p->weight_dtype == p->dtype || p->weight_dtype == MOE_DTYPE_F32, MOE_ERR_INVALID_ARGUMENT,
                "weight has the rows' type or FP32");
    MOE_REQUIRE(p->eps >= 0.0 && p->eps < 1e30, MOE_ERR_INVALID_ARGUMENT, "eps must be finite and >= 0");
    if (p->tokens == 0) return MOE_OK;
    MOE_REQUIRE(p->x && p->output && (!p->residual || p->total), MOE_ERR_INVALID_ARGUMENT, "null pointer");
    const uintptr_t elem = dtype_size(static_cast<int>(p->dtype));
    MOE_REQUIRE(aligned_to(p->x, elem) && aligned_to(p->residual, elem) && aligned_to(p->total, elem) &&
                    aligned_to(p->weight, dtype_size(static_cast<int>(p->weight_dtype))) &&
                    (p->scales || aligned_to(p->output, elem)) && aligned_to(p->scales, 4) && aligned_to(p->rstd, 4),
                MOE_ERR_INVALID_ARGUMENT, "pointers must be aligned to their element size");
    const NormArgs a{p->x, p->residual, p->weight, p->total, p->output, p->scales, p->rstd, p->tokens,
                     static_cast<int>(p->hidden), static_cast<int>(p->dtype), static_cast<int>(p->weight_dtype),
                     static_cast<float>(p->eps)};
    return launch_rms_norm(a, static_cast<hipStream_t>(stream));
}

int moe_quantize_rows(const void* x, int dtype, void* values, float* scales, int64_t tokens, int64_t hidden,
                      void* stream) {
    const int rc = check_rows(tokens, hidden, dtype, kMaxQuantizeWidth);
    if (rc != MOE_OK || tokens == 0) return rc;
    MOE_REQUIRE(x && values && scales, MOE_ERR_INVALID_ARGUMENT, "null pointer");
    MOE_REQUIRE(aligned_to(x, dtype_size(dtype)) && aligned_to(scales, 4), MOE_ERR_INVALID_ARGUMENT,
                "pointers must be aligned to their element size");
    const NormArgs a{x, nullptr, nullptr, nullptr, values, scales, nullptr, tokens, static_cast<int>(hidden), dtype,
                     dtype, 0.0f};
    return launch_quantize_rows(a, static_cast<hipStream_t>(stream));
}

int64_t moe_rms_norm_backward_scratch_bytes(int64_t tokens, int64_t hidden, int dtype) {
    if (tokens < 0 || tokens > kMaxLayerTokens || hidden < 1 || hidden > kMaxNormWidth || !valid_dtype(dtype)) return -1;
    return rms_norm_backward_scratch_bytes(tokens, hidden, dtype);
}

int moe_rms_norm_backward(const void* grad_output, const void* x, int dtype, const void* weight, int weight_dtype,
                          const float* rstd, const void* grad_x_base, void* grad_x, float* grad_weight, void* scratch,
                          int64_t scratch_bytes, int64_t tokens, int64_t hidden, void* stream) {
    const int rc = check_rows(tokens, hidden, dtype);
    if (rc != MOE_OK) return rc;
    MOE_REQUIRE(weight_dtype == dtype || weight_dtype == MOE_DTYPE_F32, MOE_ERR_INVALID_ARGUMENT,
                "weight has the rows' type or FP32");
    MOE_REQUIRE(tokens >= 1, MOE_ERR_INVALID_ARGUMENT, "norm gradients need at least one token");
    if (!grad_x && !grad_weight) return MOE_OK;
    MOE_REQUIRE(grad_output && x && rstd, MOE_ERR_INVALID_ARGUMENT, "null pointer");
    const int64_t need = grad_weight ? rms_norm_backward_scratch_bytes(tokens, hidden, dtype) : 0;
    MOE_REQUIRE(need == 0 || (scratch && scratch_bytes >= need), MOE_ERR_WORKSPACE,
                "norm gradient scratch needs %lld bytes, got %lld", (long long)need, (long long)scratch_bytes);
    const uintptr_t elem = dtype_size(dtype);
    MOE_REQUIRE(aligned_to(grad_output, elem) && aligned_to(x, elem) && aligned_to(weight, dtype_size(weight_dtype)) &&
                    aligned_to(grad_x_base, elem) && aligned_to(grad_x, elem) && aligned_to(rstd, 4) &&
                    aligned_to(grad_weight, 4) && aligned_to(scratch, 4),
                MOE_ERR_INVALID_ARGUMENT, "pointers must be aligned to their element size");
    const NormGradArgs a{grad_output, x, weight, rstd, grad_x_base, grad_x, grad_weight, static_cast<float*>(scratch),
                         tokens, static_cast<int>(hidden), dtype, weight_dtype};
    return launch_rms_norm_backward(a, static_cast<hipStream_t>(stream));
}

int moe_route_scored(const moe_route_scored_args* p, void* stream) {
    int rc = check_struct(p);
    if (rc == MOE_OK) rc = check_scored(p->tokens, p->experts, p->topk);
    if (rc != MOE_OK) return rc;
    MOE_REQUIRE(p->groups >= 1 && p->groups <= 64 && p->experts % p->groups == 0, MOE_ERR_UNSUPPORTED,
                "groups must be in 1..64 and divide the experts");
    MOE_REQUIRE(p->top_groups >= 1 && p->top_groups <= p->groups &&
                    p->topk <= p->top_groups * (p->experts / p->groups),
                MOE_ERR_INVALID_ARGUMENT, "top_groups must be in 1..groups and hold topk experts");
    MOE_REQUIRE(p->group_best == 1 || p->group_best == 2, MOE_ERR_INVALID_ARGUMENT, "group_best must be 1 or 2");
    if (p->tokens == 0) return MOE_OK;
    MOE_REQUIRE(p->logits && p->ids && p->weights, MOE_ERR_INVALID_ARGUMENT, "null pointer");
    MOE_REQUIRE(aligned_to(p->logits, 4) && aligned_to(p->bias, 4) && aligned_to(p->ids, 4) && aligned_to(p->weights, 4),
                MOE_ERR_INVALID_ARGUMENT, "pointers must be aligned to their element size");
    const ScoreArgs a{p->logits, p->bias, p->ids, p->weights, p->tokens, static_cast<int>(p->experts),
                      static_cast<int>(p->topk), static_cast<int>(p->groups), static_cast<int>(p->top_groups),
                      static_cast<int>(p->group_best), p->sigmoid != 0, p->renormalize != 0,
                      static_cast<float>(p->scale)};
    return launch_route_scored(a, static_cast<hipStream_t>(stream));
}

int moe_route_scored_backward(const moe_route_scored_backward_args* p, void* stream) {
    int rc = check_struct(p);
    if (rc == MOE_OK) rc = check_scored(p->tokens, p->experts, p->topk);
    if (rc != MOE_OK || p->tokens == 0) return rc;
    MOE_REQUIRE(p->grad_weights && p->logits && p->ids && p->grad_logits, MOE_ERR_INVALID_ARGUMENT, "null pointer");
    MOE_REQUIRE(aligned_to(p->grad_weights, 4) && aligned_to(p->logits, 4) && aligned_to(p->ids, 4) &&
                    aligned_to(p->grad_logits, 4),
                MOE_ERR_INVALID_ARGUMENT, "pointers must be aligned to their element size");
    const ScoreGradArgs a{p->grad_weights, p->logits, p->ids, p->grad_logits, p->tokens, static_cast<int>(p->experts),
                          static_cast<int>(p->topk), p->sigmoid != 0, p->renormalize != 0, static_cast<float>(p->scale)};
    return launch_route_scored_backward(a, static_cast<hipStream_t>(stream));
}

int64_t moe_linear_scratch_bytes(int64_t tokens, int64_t hidden, int64_t width, int64_t activation, int e4m3) {
    if (!valid_linear(tokens, hidden, width, activation, e4m3 != 0)) return -1;
    return linear_scratch_bytes(linear_shape(tokens, hidden, width, activation, e4m3 != 0));
}

int moe_linear(const moe_linear_args* p, void* stream) {
    const int rc = check_struct(p);
    if (rc != MOE_OK) return rc;
    const bool e4m3 = p->x_scales != nullptr || p->weight_scales != nullptr;
    MOE_REQUIRE(valid_linear(p->tokens, p->hidden, p->width, p->activation, e4m3), MOE_ERR_UNSUPPORTED,
                "rows must be multiples of 16 bytes, width a multiple of 8, both up to 2^20, tokens up to 2^21, "
                "activation a MOE_ACT_*");
    LinearArgs a = linear_shape(p->tokens, p->hidden, p->width, p->activation, e4m3);
    const int64_t size = e4m3 ? 1 : 2;
    a.w_stride = p->row_stride * size;
    MOE_REQUIRE(p->row_stride >= p->hidden && a.w_stride % 16 == 0 && p->row_stride <= 2 * kMaxLinearWidth,
                MOE_ERR_UNSUPPORTED, "weight row stride must be at least the row length and a multiple of 16 bytes");
    MOE_REQUIRE(a.w_stride * a.rows < (int64_t{1} << 32), MOE_ERR_CAPACITY, "weight must be below 4 GiB");
    if (p->tokens == 0) return MOE_OK;
    MOE_REQUIRE(p->x && p->weight && p->output && (!e4m3 || (p->x_scales && p->weight_scales)), MOE_ERR_INVALID_ARGUMENT,
                "null pointer");
    MOE_REQUIRE(p->bias_dtype == MOE_DTYPE_F32 || p->bias_dtype == MOE_DTYPE_BF16, MOE_ERR_INVALID_ARGUMENT,
                "bias is FP32 or BF16");
    MOE_REQUIRE(aligned_to(p->x, 16) && aligned_to(p->weight, 16) && aligned_to(p->residual, 16) &&
                    aligned_to(p->output, 16) && aligned_to(p->scratch, 16) && aligned_to(p->x_scales, 4) &&
                    aligned_to(p->weight_scales, 4) &&
                    aligned_to(p->bias, p->bias_dtype == MOE_DTYPE_F32 ? 4 : 2),
                MOE_ERR_INVALID_ARGUMENT, "rows must be 16-byte aligned, scales and bias to their element");
    const int64_t need = linear_scratch_bytes(a);
    MOE_REQUIRE(need == 0 || (p->scratch && p->scratch_bytes >= need), MOE_ERR_WORKSPACE,
                "linear scratch needs %lld bytes, got %lld", (long long)need, (long long)p->scratch_bytes);
    a.x = static_cast<const uint8_t*>(p->x);
    a.weight = static_cast<const uint8_t*>(p->weight);
    a.x_scales = p->x_scales;
    a.w_scales = p->weight_scales;
    a.bias = p->bias;
    a.bias_bf16 = p->bias_dtype == MOE_DTYPE_BF16;
    a.residual = static_cast<const uint16_t*>(p->residual);
    a.output = static_cast<uint16_t*>(p->output);
    return launch_linear(a, p->scratch, static_cast<hipStream_t>(stream));
}

int64_t moe_clip_scratch_bytes(void) { return kClipPartials * 8; }

int moe_clip_gradients(const moe_clip_args* p, void* stream) {
    const int rc = check_struct(p);
    if (rc != MOE_OK) return rc;
    MOE_REQUIRE(p->tensors >= 0 && p->tensors <= kMaxClipTensors, MOE_ERR_CAPACITY, "takes up to %lld tensors",
                (long long)kMaxClipTensors);
    MOE_REQUIRE(p->max_norm > 0.0, MOE_ERR_INVALID_ARGUMENT, "max_norm must be positive");
    MOE_REQUIRE(p->norm && aligned_to(p->norm, 4), MOE_ERR_INVALID_ARGUMENT, "norm must be a 4-byte aligned address");
    MOE_REQUIRE(p->scratch && aligned_to(p->scratch, 8) && p->scratch_bytes >= kClipPartials * 8, MOE_ERR_WORKSPACE,
                "clip scratch needs %lld bytes, got %lld", (long long)(kClipPartials * 8), (long long)p->scratch_bytes);
    MOE_REQUIRE(p->tensors == 0 || (p->grads && p->outputs && p->elements && p->dtypes), MOE_ERR_INVALID_ARGUMENT,
                "null pointer");
    int64_t total = 0;
    for (int64_t i = 0; i < p->tensors; ++i) {
        MOE_REQUIRE(valid_dtype(p->dtypes[i]), MOE_ERR_INVALID_ARGUMENT, "only FP32, FP16 and BF16 are supported");
        MOE_REQUIRE(p->elements[i] >= 0 && p->elements[i] <= (int64_t{1} << 40), MOE_ERR_CAPACITY, "invalid element count");
        total += p->elements[i];
        MOE_REQUIRE(total <= (int64_t{1} << 40), MOE_ERR_CAPACITY, "takes up to 2^40 elements");
        const uintptr_t elem = dtype_size(static_cast<int>(p->dtypes[i]));
        MOE_REQUIRE(p->elements[i] == 0 || (p->grads[i] && p->outputs[i]), MOE_ERR_INVALID_ARGUMENT, "null pointer");
        MOE_REQUIRE(aligned_to(p->grads[i], elem) && aligned_to(p->outputs[i], elem), MOE_ERR_INVALID_ARGUMENT,
                    "pointers must be aligned to their element size");
    }
    return launch_clip_gradients(p->grads, p->outputs, p->elements, p->dtypes, p->tensors, p->max_norm, p->norm,
                                 static_cast<double*>(p->scratch), static_cast<hipStream_t>(stream));
}

int moe_clip_overlap(const void* const* grads, const void* const* outputs, const int64_t* elements,
                     const int64_t* dtypes, uint64_t* room, int64_t tensors) {
    if (tensors <= 0) return 0;
    MOE_REQUIRE(grads && outputs && elements && dtypes && room, MOE_ERR_INVALID_ARGUMENT, "null pointer");
    struct Range {
        uint64_t from, to;
    };
    Range* ranges = reinterpret_cast<Range*>(room);
    int64_t count = 0;
    for (int64_t i = 0; i < tensors; ++i) {
        const uint64_t bytes = static_cast<uint64_t>(elements[i]) * dtype_size(static_cast<int>(dtypes[i]));
        if (bytes == 0) continue;
        const uint64_t g = reinterpret_cast<uint64_t>(grads[i]), o = reinterpret_cast<uint64_t>(outputs[i]);
        ranges[count++] = Range{g, g + bytes};
        if (o != g) ranges[count++] = Range{o, o + bytes};
    }
    std::sort(ranges, ranges + count, [](const Range& a, const Range& b) { return a.from < b.from; });
    for (int64_t i = 1; i < count; ++i)
        if (ranges[i - 1].to > ranges[i].from) return 1;
    return 0;
}

}  // extern "C"
