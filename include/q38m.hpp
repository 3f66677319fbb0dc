// C++ wrapper over the q38m C ABI with the reference's function names,
// argument order and error behaviour (include/q38/cuda_moe_prefill.h:98-133,
// include/q38/cuda_moe.h:17-39, include/q38/cuda_kernels.h:83-91): invalid
// arguments throw std::invalid_argument, device failures throw
// std::runtime_error (cuda/q38_moe_prefill.cu:33-68).
//
// A caller of the reference switches by including this header and
// qualifying calls with q38m:: instead of q38::, with these differences
// (the activation format of this data plane is int8 per token, not bf16):
//  - cuda_moe_grouped_gate_up_v1 takes the int8 token rows xq[T][2048] and
//    their scales xs[T] (from q38m_moe_route_quantize_v1 or
//    quantize_rows_i8) instead of the packed bf16 rows of
//    cuda_moe_pack_hidden_v1; it gathers the rows through
//    packed_assignment itself, so the pack step is not needed;
//  - cuda_moe_grouped_down_v1 takes weighted_mid quantised to int8 rows
//    (one quantize_rows_i8 call between gate/up and down);
//  - expert tensors are q38m_expert_weights_v1 descriptors in the MFMA16
//    device layouts instead of CudaTensorViewV1;
//  - cuda_moe_routed_bf16 serves tokens == 1 only (the legacy route-wise
//    atomic path for tokens > 1 is not built);
//  - both grouped modes are accepted and the legacy atomic mode is
//    rejected, as validate_grouped_mode does.
#ifndef Q38M_HPP
#define Q38M_HPP

#include <cstddef>
#include <cstdint>
#include <stdexcept>
#include <string>

#include "q38m.h"

namespace q38m {

using Q38ExpertMmqTaskV1 = q38m_task_v1;
using Q38RoutePlanHeaderV1 = q38m_route_plan_header_v1;
using Q38RoutePlanStorageV1 = q38m_route_plan_v1;
using ExpertWeightsV1 = q38m_expert_weights_v1;
using PrefillWorkspaceV1 = q38m_prefill_workspace_v1;

// Q38PrefillMoeModeV1, include/q38/cuda_moe_prefill.h:67-71
enum class Q38PrefillMoeModeV1 : std::uint32_t {
    kGroupedMmq = Q38M_MOE_MODE_GROUPED_MMQ,
    kGroupedMmqSafe = Q38M_MOE_MODE_GROUPED_MMQ_SAFE,
    kLegacyAtomicDiagnostic = Q38M_MOE_MODE_LEGACY_ATOMIC_DIAGNOSTIC,
};

static_assert(sizeof(Q38ExpertMmqTaskV1) == 8, "Q38ExpertMmqTaskV1 ABI changed");
static_assert(sizeof(Q38RoutePlanHeaderV1) == 64, "Q38RoutePlanHeaderV1 ABI changed");

inline void check(int status) {
    if (status == Q38M_OK) return;
    const std::string message = q38m_last_error();
    if (status == Q38M_ERR_INVALID_ARGUMENT || status == Q38M_ERR_UNSUPPORTED)
        throw std::invalid_argument(message);
    throw std::runtime_error(message);
}

constexpr std::uint32_t q38_moe_prefill_routes_v1(std::uint32_t tokens) {
    return tokens * Q38M_ROUTE_TOPK;
}

constexpr std::uint32_t q38_moe_prefill_max_tasks_v1(std::uint32_t tokens) {
    return (tokens * Q38M_ROUTE_TOPK < Q38M_ROUTE_EXPERTS ? tokens * Q38M_ROUTE_TOPK
                                                           : Q38M_ROUTE_EXPERTS) +
           (tokens * Q38M_ROUTE_TOPK -
            (tokens * Q38M_ROUTE_TOPK < Q38M_ROUTE_EXPERTS ? tokens * Q38M_ROUTE_TOPK
                                                            : Q38M_ROUTE_EXPERTS)) /
               Q38M_MMQ_M;
}

constexpr std::size_t q38_moe_route_plan_bytes_v1(std::uint32_t tokens) {
    return sizeof(Q38RoutePlanHeaderV1) + Q38M_ROUTE_EXPERTS * sizeof(std::uint16_t) +
           2 * (Q38M_ROUTE_EXPERTS + 1) * sizeof(std::uint32_t) +
           2 * static_cast<std::size_t>(q38_moe_prefill_routes_v1(tokens)) *
               sizeof(std::uint32_t) +
           q38_moe_prefill_max_tasks_v1(tokens) * sizeof(Q38ExpertMmqTaskV1);
}

inline Q38RoutePlanStorageV1 cuda_moe_route_plan_storage_v1(void* allocation,
                                                            std::size_t allocation_bytes,
                                                            std::uint32_t tokens) {
    Q38RoutePlanStorageV1 plan{};
    check(q38m_moe_route_plan_storage_v1(allocation, allocation_bytes, tokens, &plan));
    return plan;
}

// The reference always computes the FNV hashes; so does this wrapper.  The
// fast path (q38m_moe_prefill_v1) skips them.
inline void cuda_moe_build_route_plan_v1(const std::int32_t* expert_ids, std::uint32_t tokens,
                                         Q38RoutePlanStorageV1 plan, void* stream, int device) {
    check(q38m_moe_build_route_plan_v1(expert_ids, tokens, &plan, Q38M_PLAN_FLAG_HASHES, stream,
                                       device));
}

inline void cuda_moe_pack_hidden_v1(const std::uint16_t* hidden,
                                    const std::uint32_t* packed_assignment,
                                    std::uint32_t routes, std::uint16_t* packed_hidden,
                                    void* stream, int device) {
    check(q38m_moe_pack_hidden_v1(hidden, packed_assignment, routes, Q38M_HIDDEN, packed_hidden,
                                  stream, device));
}

inline void quantize_rows_i8(const std::uint16_t* x, std::uint32_t rows, std::uint32_t width,
                             std::int8_t* q, float* scales, void* stream, int device) {
    check(q38m_quantize_rows_i8(x, rows, width, q, scales, stream, device));
}

inline void cuda_moe_grouped_gate_up_v1(const ExpertWeightsV1& gate_up_experts,
                                        const std::int8_t* xq, const float* xs,
                                        const std::uint32_t* packed_assignment,
                                        const float* token_rank_weights,
                                        const Q38ExpertMmqTaskV1* tasks,
                                        std::uint32_t task_count, std::uint16_t* weighted_mid,
                                        Q38PrefillMoeModeV1 mode, void* stream, int device) {
    check(q38m_moe_grouped_gate_up_v1(&gate_up_experts, xq, xs, packed_assignment,
                                      token_rank_weights, tasks, task_count, weighted_mid,
                                      static_cast<std::uint32_t>(mode), stream, device));
}

inline void cuda_moe_grouped_down_v1(const ExpertWeightsV1& down_experts,
                                     const std::int8_t* mid_q, const float* mid_scales,
                                     const Q38ExpertMmqTaskV1* tasks, std::uint32_t task_count,
                                     float* route_output, Q38PrefillMoeModeV1 mode, void* stream,
                                     int device) {
    check(q38m_moe_grouped_down_v1(&down_experts, mid_q, mid_scales, tasks, task_count,
                                   route_output, static_cast<std::uint32_t>(mode), stream,
                                   device));
}

// No reference counterpart: the gate/up, mid quantisation and down calls
// above as one (one launch for W4 gate/up with per-channel W8 down), same
// results; task_flags (9 * task_count words) zero on entry, see q38m.h.
inline void moe_clear_task_flags_v1(std::uint32_t* task_flags, std::uint32_t task_count,
                                    void* stream, int device) {
    check(q38m_moe_clear_task_flags_v1(task_flags, task_count, stream, device));
}

inline void moe_grouped_gate_up_down_v1(const ExpertWeightsV1& gate_up_experts,
                                        const ExpertWeightsV1& down_experts,
                                        const std::int8_t* xq, const float* xs,
                                        const std::uint32_t* packed_assignment,
                                        const float* token_rank_weights,
                                        const Q38ExpertMmqTaskV1* tasks,
                                        std::uint32_t task_count, std::uint16_t* weighted_mid,
                                        std::int8_t* mid_q, float* mid_scales,
                                        std::uint32_t* task_flags, std::uint32_t* plan_status,
                                        float* route_output, Q38PrefillMoeModeV1 mode,
                                        void* stream, int device) {
    check(q38m_moe_grouped_gate_up_down_v1(&gate_up_experts, &down_experts, xq, xs,
                                           packed_assignment, token_rank_weights, tasks,
                                           task_count, weighted_mid, mid_q, mid_scales,
                                           task_flags, plan_status, route_output,
                                           static_cast<std::uint32_t>(mode), stream, device));
}

inline void cuda_moe_reduce_top10_and_combine_shared_v1(
    const float* route_output, const std::uint32_t* assignment_to_packed,
    const std::uint16_t* shared_output, const std::uint16_t* shared_gate, std::uint32_t tokens,
    std::uint16_t* output, void* stream, int device) {
    check(q38m_moe_reduce_top10_and_combine_shared_v1(route_output, assignment_to_packed,
                                                      shared_output, shared_gate, tokens,
                                                      output, stream, device));
}

// tokens == 1 branch of cuda_moe_routed_bf16; the scratch replaces the
// reference's gate_up/activated/accumulation scratch buffers.
inline void cuda_moe_routed_bf16(const ExpertWeightsV1& gate_up_experts,
                                 const ExpertWeightsV1& down_experts,
                                 const std::uint16_t* hidden, const std::int32_t* expert_ids,
                                 const float* expert_weights, std::uint32_t tokens,
                                 std::uint32_t top_k, void* scratch,
                                 std::uint16_t* routed_output, void* stream, int device) {
    if (tokens != 1)
        throw std::invalid_argument(
            "q38m routed MoE handles tokens == 1; use the grouped prefill path");
    check(q38m_moe_routed_decode_v1(&gate_up_experts, &down_experts, hidden, expert_ids,
                                    expert_weights, top_k, scratch, routed_output, stream,
                                    device));
}

// Fused tokens == 1 MoE step from fp32 router logits: top-k, routed experts
// and the optional gated shared term (and residual), in two launches.
inline void moe_decode(const q38m_expert_weights_v1& gate_up_experts,
                       const q38m_expert_weights_v1& down_experts, const std::uint16_t* hidden,
                       const float* logits, std::uint32_t top_k,
                       const std::uint16_t* shared_output, const std::uint16_t* shared_gate,
                       const std::uint16_t* residual, void* scratch, std::uint16_t* output,
                       void* stream, int device) {
    check(q38m_moe_decode_v1(&gate_up_experts, &down_experts, hidden, logits, top_k,
                             shared_output, shared_gate, residual, scratch, output, stream,
                             device));
}

inline void cuda_moe_combine_shared_bf16(const std::uint16_t* routed_output,
                                         const std::uint16_t* shared_output,
                                         const std::uint16_t* shared_gate,
                                         std::uint16_t* output, std::uint32_t tokens,
                                         void* stream, int device) {
    check(q38m_moe_combine_shared_bf16(routed_output, shared_output, shared_gate, output, tokens,
                                       stream, device));
}

// cuda_topk_router_bf16 (include/q38/cuda_kernels.h:83-91): same name and
// arguments as the reference.
inline void cuda_topk_router_bf16(const std::uint16_t* logits, std::int32_t* expert_ids,
                                  float* expert_weights, std::uint32_t tokens,
                                  std::uint32_t experts, std::uint32_t top_k,
                                  bool normalize_top_k, void* stream, int device) {
    check(q38m_topk_router_bf16(logits, expert_ids, expert_weights, tokens, experts, top_k,
                                normalize_top_k ? 1 : 0, stream, device));
}

// Router top-k over fp32 logits (the BASELINE router output).
inline void cuda_topk_router_f32(const float* logits, std::int32_t* expert_ids,
                                 float* expert_weights, std::uint32_t tokens,
                                 std::uint32_t experts, std::uint32_t top_k,
                                 bool normalize_top_k, void* stream, int device) {
    check(q38m_topk_router_f32(logits, expert_ids, expert_weights, tokens, experts, top_k,
                               normalize_top_k ? 1 : 0, stream, device));
}

// The whole run_moe step for one slab (cuda/cuda_backend.cu:1523-1601).
inline void run_moe_prefill(const ExpertWeightsV1& gate_up, const ExpertWeightsV1& down,
                            const std::uint16_t* hidden, const float* logits,
                            std::uint32_t tokens, const PrefillWorkspaceV1& workspace,
                            const std::uint16_t* shared_output,
                            const std::uint16_t* shared_gate, std::uint16_t* output,
                            void* stream, int device) {
    check(q38m_moe_prefill_v1(&gate_up, &down, hidden, logits, tokens, &workspace,
                              shared_output, shared_gate, output, stream, device));
}

// Router logits (cuda_backend.cu:1518-1519): fp32 [tokens][512] from
// hidden rows of hidden_width (must be 2048) values.
// The whole MoE block of one decode step (run_moe's tokens == 1 branch,
// cuda_backend.cu:1516-1605): router GEMV, routed experts, bf16 shared
// expert, gated combine and optional residual in three launches; equal to
// moe_router + moe_shared_expert + moe_decode bit for bit.
inline void moe_decode_block(const q38m_expert_weights_v1& gate_up_experts,
                             const q38m_expert_weights_v1& down_experts,
                             const std::uint16_t* hidden, const std::uint16_t* router,
                             const std::uint16_t* w_gate, const std::uint16_t* w_up,
                             const std::uint16_t* w_down, const std::uint16_t* w_out_gate,
                             std::uint32_t shared_inter, std::uint32_t top_k,
                             const std::uint16_t* residual, void* scratch,
                             std::uint16_t* output, void* stream, int device) {
    check(q38m_moe_decode_block_v1(&gate_up_experts, &down_experts, hidden, router, w_gate,
                                   w_up, w_down, w_out_gate, shared_inter, top_k, residual,
                                   scratch, output, stream, device));
}

inline void moe_router(const std::uint16_t* hidden, const std::uint16_t* router,
                       std::uint32_t tokens, std::uint32_t hidden_width, float* logits,
                       void* stream, int device) {
    check(q38m_moe_router_v1(hidden, router, tokens, hidden_width, logits, stream, device));
}

// Shared expert (cuda_backend.cu:1573-1590): shared_output bf16 [tokens][2048]
// and shared_gate bf16 [tokens] for the gated combine.
inline void moe_shared_expert(const std::uint16_t* hidden, const std::uint16_t* w_gate,
                              const std::uint16_t* w_up, const std::uint16_t* w_down,
                              const std::uint16_t* w_out_gate, std::uint32_t tokens,
                              std::uint32_t hidden_width, std::uint32_t inter, void* scratch,
                              std::uint16_t* shared_output, std::uint16_t* shared_gate,
                              void* stream, int device) {
    check(q38m_moe_shared_expert_v1(hidden, w_gate, w_up, w_down, w_out_gate, tokens,
                                    hidden_width, inter, scratch, shared_output, shared_gate,
                                    stream, device));
}

// ---- microscaled 4-bit rows and sorted tokens: no reference counterpart; the
// entry points of the same names in q38m.h, whose comments say what they do.
using MxMatrixV1 = q38m_mx_matrix_v1;

enum class DtypeV1 : std::uint32_t { kF32 = Q38M_DTYPE_F32, kBf16 = Q38M_DTYPE_BF16 };
enum class MxEpilogueV1 : std::uint32_t {
    kNone = Q38M_MX_EPILOGUE_NONE,
    kSwiglu = Q38M_MX_EPILOGUE_SWIGLU,
};

inline void mx_quantize(const void* x, DtypeV1 dtype, std::uint64_t x_stride,
                        const MxMatrixV1& dst, void* rounded, void* stream, int device) {
    check(q38m_mx_quantize_v1(x, static_cast<std::uint32_t>(dtype), x_stride, &dst, rounded,
                              stream, device));
}

inline void mx_gemm(const MxMatrixV1& a, const MxMatrixV1& b, float* c_f32,
                    std::uint16_t* c_bf16, std::uint64_t c_stride, void* stream, int device) {
    check(q38m_mx_gemm_v1(&a, &b, c_f32, c_bf16, c_stride, stream, device));
}

inline void mx_grouped_gemm(const MxMatrixV1& weights, const MxMatrixV1& rows,
                            const std::uint32_t* expert_offsets,
                            const std::uint32_t* packed_assignment, std::uint32_t top_k,
                            std::uint32_t routes, MxEpilogueV1 epilogue, float* c_f32,
                            std::uint16_t* c_bf16, void* stream, int device) {
    check(q38m_mx_grouped_gemm_v1(&weights, &rows, expert_offsets, packed_assignment, top_k,
                                  routes, static_cast<std::uint32_t>(epilogue), c_f32, c_bf16,
                                  stream, device));
}

inline void moe_sort_routes(const std::int32_t* expert_ids, std::uint32_t tokens,
                            std::uint32_t top_k, std::uint32_t experts,
                            std::uint32_t* expert_offsets, std::uint32_t* packed_assignment,
                            std::uint32_t* assignment_to_packed, void* scratch,
                            std::size_t scratch_bytes, void* stream, int device) {
    check(q38m_moe_sort_routes_v1(expert_ids, tokens, top_k, experts, expert_offsets,
                                  packed_assignment, assignment_to_packed, scratch,
                                  scratch_bytes, stream, device));
}

inline void moe_permute_rows(const void* x, DtypeV1 dtype,
                             const std::uint32_t* assignment_to_packed, std::uint32_t tokens,
                             std::uint32_t top_k, std::uint32_t width, void* rows, void* stream,
                             int device) {
    check(q38m_moe_permute_rows_v1(x, static_cast<std::uint32_t>(dtype), assignment_to_packed,
                                   tokens, top_k, width, rows, stream, device));
}

inline void moe_unpermute_rows(const void* rows, DtypeV1 dtype,
                               const std::uint32_t* assignment_to_packed,
                               const float* route_weights, std::uint32_t tokens,
                               std::uint32_t top_k, std::uint32_t width, void* y, void* stream,
                               int device) {
    check(q38m_moe_unpermute_rows_v1(rows, static_cast<std::uint32_t>(dtype),
                                     assignment_to_packed, route_weights, tokens, top_k, width,
                                     y, stream, device));
}

inline void moe_unpermute_backward(const void* dy, const void* rows, DtypeV1 dtype,
                                   const std::uint32_t* assignment_to_packed,
                                   const float* route_weights, std::uint32_t tokens,
                                   std::uint32_t top_k, std::uint32_t width, void* d_rows,
                                   float* d_weights, void* stream, int device) {
    check(q38m_moe_unpermute_backward_v1(dy, rows, static_cast<std::uint32_t>(dtype),
                                         assignment_to_packed, route_weights, tokens, top_k,
                                         width, d_rows, d_weights, stream, device));
}

// ---- bf16 products with epilogues and gradients: no reference counterpart; the
// entry points of the same names in q38m.h.  A null pointer is nothing.
using TensorV1 = q38m_tensor_v1;

enum class ActivationV1 : std::uint32_t {
    kNone = Q38M_ACT_NONE,
    kRelu = Q38M_ACT_RELU,
    kSilu = Q38M_ACT_SILU,
    kSigmoid = Q38M_ACT_SIGMOID,
    kGelu = Q38M_ACT_GELU,
    kGeluTanh = Q38M_ACT_GELU_TANH,
};
enum class EpilogueV1 : std::uint32_t {
    kNone = Q38M_EPILOGUE_NONE,
    kSwiglu = Q38M_EPILOGUE_SWIGLU,
};

inline void linear(const TensorV1& x, const TensorV1& weight, const TensorV1* bias,
                   ActivationV1 activation, const TensorV1* residual, const TensorV1& y,
                   const TensorV1* pre, void* scratch, std::size_t scratch_bytes, void* stream,
                   int device) {
    check(q38m_linear_v1(&x, &weight, bias, static_cast<std::uint32_t>(activation), residual, &y,
                         pre, scratch, scratch_bytes, stream, device));
}

inline void linear_backward_input(const TensorV1& dz, const TensorV1& weight,
                                  const TensorV1* pre, ActivationV1 activation,
                                  const TensorV1* residual, const TensorV1& dx, void* scratch,
                                  std::size_t scratch_bytes, void* stream, int device) {
    check(q38m_linear_backward_input_v1(&dz, &weight, pre, static_cast<std::uint32_t>(activation),
                                        residual, &dx, scratch, scratch_bytes, stream, device));
}

inline void linear_backward_weight(const TensorV1& dz, const TensorV1* x,
                                   const TensorV1* residual, const TensorV1* d_weight,
                                   const TensorV1* d_bias, void* scratch,
                                   std::size_t scratch_bytes, void* stream, int device) {
    check(q38m_linear_backward_weight_v1(&dz, x, residual, d_weight, d_bias, scratch,
                                         scratch_bytes, stream, device));
}

inline void linear_backward_activation(const TensorV1& dy, const TensorV1& pre,
                                       ActivationV1 activation, const TensorV1& dz, void* stream,
                                       int device) {
    check(q38m_linear_backward_activation_v1(&dy, &pre, static_cast<std::uint32_t>(activation),
                                             &dz, stream, device));
}

inline void moe_expert_gemm(const TensorV1& weights, const TensorV1& rows,
                            const std::uint32_t* expert_offsets,
                            const std::uint32_t* packed_assignment, std::uint32_t top_k,
                            EpilogueV1 epilogue, const TensorV1& c, const TensorV1* pre,
                            void* stream, int device) {
    check(q38m_moe_expert_gemm_v1(&weights, &rows, expert_offsets, packed_assignment, top_k,
                                  static_cast<std::uint32_t>(epilogue), &c, pre, stream, device));
}

inline void moe_expert_backward_rows(const TensorV1& weights, const TensorV1& d_c,
                                     const std::uint32_t* expert_offsets, const TensorV1* pre,
                                     const TensorV1& d_rows, void* stream, int device) {
    check(q38m_moe_expert_backward_rows_v1(&weights, &d_c, expert_offsets, pre, &d_rows, stream,
                                           device));
}

inline void moe_expert_backward_weights(const TensorV1& d_c, const TensorV1& rows,
                                        const std::uint32_t* expert_offsets,
                                        const std::uint32_t* packed_assignment,
                                        std::uint32_t top_k, const TensorV1* residual,
                                        const TensorV1& d_weights, void* stream, int device) {
    check(q38m_moe_expert_backward_weights_v1(&d_c, &rows, expert_offsets, packed_assignment,
                                              top_k, residual, &d_weights, stream, device));
}

inline bool cuda_q38_moe_prefill_compiled() { return q38m_moe_compiled() == 1; }
inline bool cuda_q38_moe_compiled() { return q38m_moe_compiled() == 1; }

}  // namespace q38m

#endif
