// What the kernels of the attention over shared pages have in common.
#pragma once
#include "t2sx_pool.cuh"

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <utility>

namespace t2sx {
namespace attn {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kWeightExp = 7.0f;   // c above: weights are at most 2^7

// A tile of rows against a range of a node's pages.
struct Item {
    int32_t tokens_at;   // the node's tokens start here in `tokens`
    int32_t row0, rows;  // rows of the node: token row / group, head row % group
    int32_t pages_at;    // page ids
    int32_t n_pages;
    int32_t pos0;        // position of the first page's first key
    int32_t split;       // which range of the node's pages this is
    int32_t end;         // the node's filled positions end here
    int32_t new_pos;     // from this position on the keys are the step's own (of one sequence) ...
    int32_t new_row;     // ... and that one is this row of the step
    int32_t launch;      // 0: tcgen05, 1: pages of several sequences, 2: the others
    int32_t keys;        // of its pages that a row sees
};

// A token as one of a node's: what it is, and where its parts are.  A token's parts are numbers
// part_at .. part_at + n_parts - 1, those of the node's splits from part0 on.
struct alignas(16) Token {
    int32_t row;         // of the step
    int32_t limit;       // positions that it sees; its own is the last of them
    int32_t page;        // page of its own position
    int32_t part0, part_at;
    int32_t n_parts;     // one: the item writes the result itself
    int32_t ends_here;   // the node's item completes the token: its own part is the last one, and the others are
                         // those of the launch before
    int32_t pad;
};

struct PlanView {
    const Token* tokens;     // nodes' tokens
    const int32_t* pages;
    const Item* items;
    const Token* joins;      // tokens of several parts
    float* part_o;           // [part][query head of the group][K/V head][dim]
    float2* part_ml;         // [part][query head of the group][K/V head]
    const Token* rows_of;    // the step's rows (for a launch that writes their keys and values)
    // items: n_tc of up to kTcRows rows, then n_shared of pages of several sequences, then n_own others
    int rows, n_tc, n_shared, n_own, n_joins, group, n_kv;
};

// Strided tensors of one call.
template <typename T>
struct Tensors {
    const T* q;
    T *k, *v;                // the layer's first page
    const T *k_new, *v_new;  // the rows' own keys and values, or null: they are in the cache
    long long kv_stride;
    T* out;
    float* lse;
    long long q_stride, out_stride;
    float scale2;            // scale * log2(e)
};

__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ uint32_t pack2(__half, float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(__nv_bfloat16, float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void dependents_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void dependents_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// With `early` the kernel may start while the one before it runs (it waits for it itself).
template <typename... P, typename... A>
cudaError_t launch(void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t st, bool early, A&&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = threads;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &at;
    cfg.numAttrs = early ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, std::forward<A>(args)...);
}

// Items of up to kTcRows rows on the tcgen05 tensor cores (t2sx_prefix_tc.cu).
constexpr int kTcRows = 256;
bool tc_maps(const t2sx_pool* p, CUtensorMap* k, CUtensorMap* v);
template <typename T>
cudaError_t launch_tc(const PlanView& w, const Tensors<T>& x, const t2sx_pool* p, const CUtensorMap& k, const CUtensorMap& v, int layer_page,
                      int32_t* err, bool early, cudaStream_t st);

}  // namespace attn
}  // namespace t2sx
