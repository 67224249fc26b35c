// The operator object behind the C entry points: how one is made, checked, enqueued and given back.
#pragma once
#include <memory>
#include <vector>

#include "ops_common.h"

namespace chip {

struct DiscardOperator {
    void operator()(cldnn_hip_operator op) const
    {
        if (op->workspace) {
            (void)hipFree(op->workspace);
            op->engine->used.fetch_sub(op->info.workspace_bytes);
        }
        cldnn_hip_engine e = op->engine;
        delete op;
        (void)cldnn_hip_engine_release(e);
    }
};

// plan(op, init): fills in what the operator's kind keeps, its info, and what its workspace starts with
template <typename F>
cldnn_hip_status create_operator(cldnn_hip_engine e, const void* desc, cldnn_hip_operator* out, OperatorKind kind, F&& plan)
{
    return guarded([&] {
        CHIP_REQUIRE(e && desc && out, CLDNN_HIP_INVALID_ARG, "null argument");
        *out = nullptr;
        std::unique_ptr<cldnn_hip_operator_s, DiscardOperator> op(new cldnn_hip_operator_s());
        op->engine = e;
        op->kind = kind;
        e->refs.fetch_add(1);
        std::vector<char> init;
        plan(*op, init);
        if (const size_t bytes = (size_t)op->info.workspace_bytes) {
            e->make_current();
            const hipError_t r = hipMalloc(&op->workspace, bytes);
            if (r != hipSuccess) {
                op->workspace = nullptr;
                (void)hipGetLastError();
                throw error(CLDNN_HIP_OUT_OF_RESOURCES, std::string("hipMalloc: ") + hipGetErrorString(r));
            }
            const int64_t used = e->used.fetch_add((int64_t)bytes) + (int64_t)bytes;
            int64_t most = e->max_used.load();
            while (used > most && !e->max_used.compare_exchange_weak(most, used)) {}
            if (!init.empty()) CHIP_CHECK(hipMemcpy(op->workspace, init.data(), init.size(), hipMemcpyHostToDevice));
        }
        *out = op.release();
    });
}

inline void check_operator(cldnn_hip_operator op, OperatorKind kind)
{
    CHIP_REQUIRE(op, CLDNN_HIP_INVALID_ARG, "null operator");
    CHIP_REQUIRE(op->kind == kind, CLDNN_HIP_INVALID_ARG, "an operator of another kind");
}

// launch(): the call's kernels, in one piece where they hand each other the object's scratch memory
template <typename F>
void enqueue_operator(cldnn_hip_operator op, F&& launch)
{
    op->engine->make_current();
    std::unique_lock<std::mutex> alone(op->engine->together, std::defer_lock);
    if (op->info.launches > 1) alone.lock();
    // a recording's kernels go on using the object's memory: it holds the object
    if (op->workspace && op->engine->launch_stream() != op->engine->stream) {
        op->engine->hold([op] { (void)cldnn_hip_operator_release(op); });
        op->refs.fetch_add(1);
    }
    launch(op->engine->launch_stream());
}

}  // namespace chip
