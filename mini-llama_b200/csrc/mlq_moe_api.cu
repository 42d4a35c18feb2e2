// mlq_moe_api.cu -- C entry points of the mixture-of-experts layer and of
// the linear with an epilogue (include/mlq.h).  Arguments are checked on the
// host before any CUDA call; nothing throws across the ABI.
#include <cuda_runtime.h>

#include <string>

#include "mlq.h"
#include "mlq_device.cuh"
#include "mlq_kernels.h"

namespace {

mlq_status fail(mlq_status st, const std::string& msg) {
    mlq::set_last_error(msg);
    return st;
}

mlq_status fail_cuda(const std::string& what, cudaError_t e) {
    cudaGetLastError();
    return fail(MLQ_ERR_CUDA, "CUDA error in " + what + ": " + cudaGetErrorString(e));
}

bool known_format(int f) { return f == MLQ_Q8_0 || f == MLQ_Q4_0 || f == MLQ_Q4_1; }

constexpr int kMaxFeatures = 1 << 20;   // of x, an expert's hidden vector, a linear's input
constexpr int kMaxOut = 1 << 24;

mlq_status check_workspace(const std::string& who, const void* ws, size_t have, size_t need) {
    if (ws == nullptr) return fail(MLQ_ERR_NULL, who + ": null workspace");
    if (reinterpret_cast<uintptr_t>(ws) % 256 != 0)
        return fail(MLQ_ERR_RANGE, who + ": the workspace must be 256-byte aligned");
    if (have < need)
        return fail(MLQ_ERR_RANGE, who + ": workspace of " + std::to_string(have) + " bytes, " + std::to_string(need) +
                                       " needed");
    return MLQ_OK;
}

mlq_status check_router(const std::string& who, const mlq_router* r) {
    if (r == nullptr) return fail(MLQ_ERR_NULL, who + ": null router");
    if (r->w == nullptr) return fail(MLQ_ERR_NULL, who + ": null router weights");
    if (r->n_experts <= 0 || r->in_features <= 0 || r->top_k <= 0)
        return fail(MLQ_ERR_EMPTY, who + ": empty tensors are not supported");
    if (r->n_experts > MLQ_MOE_MAX_EXPERTS)
        return fail(MLQ_ERR_RANGE, who + ": at most " + std::to_string(MLQ_MOE_MAX_EXPERTS) + " experts");
    if (r->top_k > r->n_experts || r->top_k > MLQ_MOE_MAX_TOP_K)
        return fail(MLQ_ERR_RANGE, who + ": top_k must be at most n_experts and " + std::to_string(MLQ_MOE_MAX_TOP_K));
    if (r->in_features > kMaxFeatures) return fail(MLQ_ERR_RANGE, who + ": in_features too large");
    if (r->scoring != MLQ_SCORE_SOFTMAX && r->scoring != MLQ_SCORE_SIGMOID)
        return fail(MLQ_ERR_RANGE, who + ": unknown scoring");
    if (r->renormalize != 0 && r->renormalize != 1) return fail(MLQ_ERR_RANGE, who + ": renormalize must be 0 or 1");
    return MLQ_OK;
}

mlq_status check_experts(const std::string& who, const mlq_experts* m) {
    if (m == nullptr) return fail(MLQ_ERR_NULL, who + ": null experts");
    if (!known_format(m->fmt) || !known_format(m->fmt_down)) return fail(MLQ_ERR_FORMAT, who + ": unknown block format");
    if (m->w_gate == nullptr || m->w_up == nullptr || m->w_down == nullptr)
        return fail(MLQ_ERR_NULL, who + ": null weight pointer");
    if (m->n_experts <= 0 || m->in_features <= 0 || m->hidden <= 0 || m->out_features <= 0)
        return fail(MLQ_ERR_EMPTY, who + ": empty tensors are not supported");
    if (m->n_experts > MLQ_MOE_MAX_EXPERTS)
        return fail(MLQ_ERR_RANGE, who + ": at most " + std::to_string(MLQ_MOE_MAX_EXPERTS) + " experts");
    if (m->in_features > kMaxFeatures || m->hidden > kMaxFeatures || m->out_features > kMaxOut ||
        (long long)m->n_experts * m->hidden > 0x7fffff00LL || (long long)m->n_experts * m->out_features > 0x7fffff00LL)
        return fail(MLQ_ERR_RANGE, who + ": a dimension is too large");
    const size_t up = (size_t)m->n_experts * mlq_block_count(m->hidden, m->in_features);
    const size_t down = (size_t)m->n_experts * mlq_block_count(m->out_features, m->hidden);
    if (m->block_count != up)
        return fail(MLQ_ERR_BLOCK_COUNT, who + ": gate/up block count mismatch: expected " + std::to_string(up) +
                                             ", got " + std::to_string(m->block_count));
    if (m->block_count_down != down)
        return fail(MLQ_ERR_BLOCK_COUNT, who + ": down block count mismatch: expected " + std::to_string(down) +
                                             ", got " + std::to_string(m->block_count_down));
    return MLQ_OK;
}

mlq_status check_top_k(const std::string& who, int top_k) {
    if (top_k <= 0) return fail(MLQ_ERR_EMPTY, who + ": empty tensors are not supported");
    if (top_k > MLQ_MOE_MAX_TOP_K)
        return fail(MLQ_ERR_RANGE, who + ": top_k must be at most " + std::to_string(MLQ_MOE_MAX_TOP_K));
    return MLQ_OK;
}

// Everything but the block count and the pointers.
mlq_status check_linear(const std::string& who, int fmt, int out, int in, int rows) {
    if (!known_format(fmt)) return fail(MLQ_ERR_FORMAT, who + ": unknown block format");
    if (in <= 0 || out <= 0 || rows <= 0) return fail(MLQ_ERR_EMPTY, who + ": empty tensors are not supported");
    if (in > kMaxFeatures || out > kMaxOut) return fail(MLQ_ERR_RANGE, who + ": a dimension is too large");
    return MLQ_OK;
}

mlq_status check_rows(const std::string& who, int rows, long long per_row) {
    if (rows <= 0) return fail(MLQ_ERR_EMPTY, who + ": empty tensors are not supported");
    if ((long long)rows * per_row > 0x7fffffffLL) return fail(MLQ_ERR_RANGE, who + ": too many rows");
    return MLQ_OK;
}

mlq::MoeShape shape_of(const mlq_experts& m) {
    return mlq::MoeShape{m.fmt, m.fmt_down, m.n_experts, m.in_features, m.hidden, m.out_features};
}

mlq_status run_route(const char* who, const mlq_router& r, const float* x, int rows, int32_t* ids, float* weights,
                     float* logits, void* ws, size_t ws_bytes, mlq_stream stream) {
    mlq::DeviceFacts f{};
    mlq_status st = mlq::current_device_facts(&f);
    if (st != MLQ_OK) return st;
    cudaError_t e = mlq::launch_route(r, x, rows, ids, weights, logits, ws, ws_bytes, f.err, stream);
    return e == cudaSuccess ? MLQ_OK : fail_cuda(std::string(who) + " launch", e);
}

mlq_status run_experts(const char* who, const mlq_experts& m, const float* x, int rows, int top_k, const int32_t* ids,
                       const float* weights, const float* residual, float* y, void* ws, size_t ws_bytes,
                       mlq_stream stream) {
    mlq::DeviceFacts f{};
    mlq_status st = mlq::current_device_facts(&f);
    if (st != MLQ_OK) return st;
    cudaError_t e = mlq::launch_experts(shape_of(m), static_cast<const uint8_t*>(m.w_gate),
                                        static_cast<const uint8_t*>(m.w_up), static_cast<const uint8_t*>(m.w_down), x,
                                        rows, top_k, ids, weights, residual, y, ws, ws_bytes, f.sm_count,
                                        f.smem_per_sm, f.err, stream);
    return e == cudaSuccess ? MLQ_OK : fail_cuda(std::string(who) + " launch", e);
}

}  // namespace

extern "C" {

MLQ_API size_t mlq_moe_route_workspace_bytes(const mlq_router* router, int rows) {
    try {
        const char* who = "mlq_moe_route_workspace_bytes";
        if (check_router(who, router) != MLQ_OK || check_rows(who, rows, router->top_k) != MLQ_OK) return 0;
        return mlq::route_workspace_bytes(router->n_experts, router->in_features, rows);
    } catch (...) {
        return 0;
    }
}

MLQ_API mlq_status mlq_moe_route(const mlq_router* router, const float* x, int rows, int32_t* ids, float* weights,
                                 float* logits, void* workspace, size_t workspace_bytes, mlq_stream stream) {
    try {
        const char* who = "mlq_moe_route";
        mlq_status st = check_router(who, router);
        if (st == MLQ_OK) st = check_rows(who, rows, router->top_k);
        if (st != MLQ_OK) return st;
        if (!x || !ids || !weights) return fail(MLQ_ERR_NULL, std::string(who) + ": null input/output pointer");
        st = check_workspace(who, workspace, workspace_bytes, mlq::route_workspace_bytes(router->n_experts, router->in_features, rows));
        if (st != MLQ_OK) return st;
        return run_route(who, *router, x, rows, ids, weights, logits, workspace, workspace_bytes, stream);
    } catch (...) {
        return fail(MLQ_ERR_CUDA, "mlq_moe_route: host exception");
    }
}

MLQ_API size_t mlq_moe_experts_workspace_bytes(const mlq_experts* experts, int rows, int top_k) {
    try {
        const char* who = "mlq_moe_experts_workspace_bytes";
        if (check_experts(who, experts) != MLQ_OK || check_top_k(who, top_k) != MLQ_OK ||
            check_rows(who, rows, top_k) != MLQ_OK)
            return 0;
        return mlq::experts_workspace_bytes(shape_of(*experts), rows, top_k);
    } catch (...) {
        return 0;
    }
}

MLQ_API mlq_status mlq_moe_experts(const mlq_experts* experts, const float* x, int rows, int top_k, const int32_t* ids,
                                   const float* weights, const float* residual, float* y, void* workspace,
                                   size_t workspace_bytes, mlq_stream stream) {
    try {
        const char* who = "mlq_moe_experts";
        mlq_status st = check_experts(who, experts);
        if (st != MLQ_OK) return st;
        st = check_top_k(who, top_k);
        if (st == MLQ_OK) st = check_rows(who, rows, top_k);
        if (st != MLQ_OK) return st;
        if (!x || !ids || !weights || !y) return fail(MLQ_ERR_NULL, std::string(who) + ": null input/output pointer");
        st = check_workspace(who, workspace, workspace_bytes,
                             mlq::experts_workspace_bytes(shape_of(*experts), rows, top_k));
        if (st != MLQ_OK) return st;
        return run_experts(who, *experts, x, rows, top_k, ids, weights, residual, y, workspace, workspace_bytes, stream);
    } catch (...) {
        return fail(MLQ_ERR_CUDA, "mlq_moe_experts: host exception");
    }
}

MLQ_API size_t mlq_moe_layer_workspace_bytes(const mlq_router* router, const mlq_experts* experts, int rows) {
    try {
        const char* who = "mlq_moe_layer_workspace_bytes";
        if (check_router(who, router) != MLQ_OK || check_experts(who, experts) != MLQ_OK ||
            check_rows(who, rows, router->top_k) != MLQ_OK)
            return 0;
        return mlq::route_workspace_bytes(router->n_experts, router->in_features, rows) +
               mlq::experts_workspace_bytes(shape_of(*experts), rows, router->top_k);
    } catch (...) {
        return 0;
    }
}

MLQ_API mlq_status mlq_moe_layer(const mlq_router* router, const mlq_experts* experts, const float* x, int rows,
                                 const float* residual, float* y, int32_t* ids, float* weights, void* workspace,
                                 size_t workspace_bytes, mlq_stream stream) {
    try {
        const char* who = "mlq_moe_layer";
        mlq_status st = check_router(who, router);
        if (st == MLQ_OK) st = check_experts(who, experts);
        if (st == MLQ_OK) st = check_rows(who, rows, router->top_k);
        if (st != MLQ_OK) return st;
        if (router->n_experts != experts->n_experts || router->in_features != experts->in_features)
            return fail(MLQ_ERR_SHAPE, std::string(who) + ": router and experts differ in n_experts or in_features");
        if (!x || !ids || !weights || !y) return fail(MLQ_ERR_NULL, std::string(who) + ": null input/output pointer");
        const size_t rb = mlq::route_workspace_bytes(router->n_experts, router->in_features, rows);
        st = check_workspace(who, workspace, workspace_bytes,
                             rb + mlq::experts_workspace_bytes(shape_of(*experts), rows, router->top_k));
        if (st != MLQ_OK) return st;
        st = run_route(who, *router, x, rows, ids, weights, nullptr, workspace, rb, stream);
        if (st != MLQ_OK) return st;
        return run_experts(who, *experts, x, rows, router->top_k, ids, weights, residual, y,
                           static_cast<char*>(workspace) + rb, workspace_bytes - rb, stream);
    } catch (...) {
        return fail(MLQ_ERR_CUDA, "mlq_moe_layer: host exception");
    }
}

MLQ_API size_t mlq_linear_epilogue_workspace_bytes(mlq_format fmt, int out_features, int in_features, int rows) {
    try {
        if (check_linear("mlq_linear_epilogue_workspace_bytes", fmt, out_features, in_features, rows) != MLQ_OK) return 0;
        return mlq::epilogue_workspace_bytes(fmt, in_features, rows);
    } catch (...) {
        return 0;
    }
}

MLQ_API mlq_status mlq_linear_epilogue(mlq_format fmt, const void* w, size_t block_count, int out_features,
                                       int in_features, const float* x, int rows, const mlq_epilogue* epilogue,
                                       float* y, void* workspace, size_t workspace_bytes, mlq_stream stream) {
    try {
        const std::string who = "mlq_linear_epilogue";
        mlq_status st = check_linear(who, fmt, out_features, in_features, rows);
        if (st != MLQ_OK) return st;
        if (w == nullptr) return fail(MLQ_ERR_NULL, who + ": null weight pointer");
        if (!x || !y || !epilogue) return fail(MLQ_ERR_NULL, who + ": null input/output pointer");
        const size_t expected = mlq_block_count(out_features, in_features);
        if (block_count != expected)
            return fail(MLQ_ERR_BLOCK_COUNT, who + ": block count mismatch: expected " + std::to_string(expected) +
                                                 ", got " + std::to_string(block_count));
        if (epilogue->activation < MLQ_ACT_NONE || epilogue->activation > MLQ_ACT_SIGMOID)
            return fail(MLQ_ERR_RANGE, who + ": unknown activation");
        st = check_workspace(who, workspace, workspace_bytes, mlq::epilogue_workspace_bytes(fmt, in_features, rows));
        if (st != MLQ_OK) return st;
        mlq::DeviceFacts f{};
        st = mlq::current_device_facts(&f);
        if (st != MLQ_OK) return st;
        cudaError_t e = mlq::launch_linear_epilogue(fmt, static_cast<const uint8_t*>(w), out_features, in_features, x,
                                                    rows, *epilogue, y, workspace, workspace_bytes, f.sm_count,
                                                    f.smem_per_sm, f.err, stream);
        return e == cudaSuccess ? MLQ_OK : fail_cuda(who + " launch", e);
    } catch (...) {
        return fail(MLQ_ERR_CUDA, "mlq_linear_epilogue: host exception");
    }
}

}  // extern "C"
