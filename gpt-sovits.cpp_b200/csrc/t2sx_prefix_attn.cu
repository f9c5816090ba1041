// Attention of one step's tokens over a pool of shared cache pages.
#include "t2sx_pool.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <memory>

using namespace t2sx;

namespace {

__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// The rows of a plan on the device.
struct RowView {
    const int32_t* limit;       // [rows] positions that the row sees; its own is the last of them
    const int32_t* table_at;    // [rows] where its sequence's page ids start in `table`
    const int32_t* table;
    int rows;
};

// One 16-byte word per thread: the rows' keys and values go to their positions.
__global__ void __launch_bounds__(256)
k_write_rows(RowView r, const uint4* __restrict__ kn, const uint4* __restrict__ vn, long long stride_vec, uint4* __restrict__ k,
             uint4* __restrict__ v, size_t layer_page0, int n_kv, int row_vec) {
    const int per_row = n_kv * row_vec;
    const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= (long long)r.rows * per_row) return;
    const int row = (int)(i / per_row), j = (int)(i - (long long)row * per_row), h = j / row_vec, c = j - h * row_vec;
    const int pos = r.limit[row] - 1;
    const size_t page = layer_page0 + r.table[r.table_at[row] + pos / kPoolPage];
    const size_t dst = ((page * n_kv + h) * kPoolPage + pos % kPoolPage) * row_vec + c;
    k[dst] = kn[row * stride_vec + j];
    v[dst] = vn[row * stride_vec + j];
}

// One warp per (row, query head): 32 positions at a time, one per lane for the scores, the lanes'
// shares of the head for the output.
template <typename T, int D>
__global__ void __launch_bounds__(128)
k_attend_rows(RowView r, const T* __restrict__ q, long long q_stride, const T* __restrict__ k, const T* __restrict__ v,
              size_t layer_page0, int n_heads, int n_kv, float scale, T* __restrict__ out, long long out_stride,
              float* __restrict__ lse) {
    const int lane = threadIdx.x & 31, head = blockIdx.y * 4 + (threadIdx.x >> 5), row = blockIdx.x;
    if (head >= n_heads) return;
    const int kvh = head / (n_heads / n_kv), limit = r.limit[row];
    const int32_t* table = r.table + r.table_at[row];
    const T* qr = q + row * q_stride + head * D;
    float m = -INFINITY, l = 0.0f, o[D / 32] = {};
    for (int p0 = 0; p0 < limit; p0 += 32) {
        const size_t at = (((layer_page0 + table[p0 / kPoolPage]) * n_kv + kvh) * kPoolPage + p0 % kPoolPage) * D;
        float s = 0.0f;
        for (int d = 0; d < D; ++d) s = fmaf(to_f32(qr[d]), to_f32(k[at + lane * D + d]), s);
        s = p0 + lane < limit ? s * scale : -INFINITY;
        float mx = s;
        for (int x = 16; x; x >>= 1) mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, x));
        mx = fmaxf(mx, m);
        const float base = mx == -INFINITY ? 0.0f : mx;
        const float p = expf(s - base), f = expf(m - base);
        m = mx;
        l = fmaf(l, f, p);
        for (int j = 0; j < D / 32; ++j) o[j] *= f;
        for (int t = 0; t < 32 && p0 + t < limit; ++t) {
            const float pt = __shfl_sync(~0u, p, t);
            for (int j = 0; j < D / 32; ++j) o[j] = fmaf(pt, to_f32(v[at + t * D + j * 32 + lane]), o[j]);
        }
    }
    for (int x = 16; x; x >>= 1) l += __shfl_xor_sync(~0u, l, x);
    for (int j = 0; j < D / 32; ++j)
        out[row * out_stride + head * D + j * 32 + lane] = from_f32<T>(l > 0.0f ? o[j] / l : 0.0f);
    if (lse && lane == 0) lse[(size_t)row * n_heads + head] = l > 0.0f ? m + logf(l) : -INFINITY;
}

int bad(const char* m) { return t2sx_set_error(T2SX_ERR_INVALID, m); }

}  // namespace

struct t2sx_plan {
    t2sx_pool* pool = nullptr;
    int n_heads = 0;
    bool ready = false;
    uint64_t version = 0;          // of the pool at the update
    int rows = 0;
    // host copy of what the device gets, in pinned memory: two buffers, so that an update need not
    // wait for the previous one's upload
    uint8_t* host[2] = {};
    size_t host_bytes[2] = {};
    cudaEvent_t sent[2] = {};
    int turn = 0;
    uint8_t* dev = nullptr;
    size_t dev_bytes = 0;
    RowView view = {};
};

static void plan_release(t2sx_plan* a) {
    t2sx_pool* p = a->pool;
    DeviceGuard dg;
    dg.set(p->device);
    cudaEventSynchronize(p->done);
    for (int i = 0; i < 2; ++i) {
        if (a->sent[i]) cudaEventDestroy(a->sent[i]);
        if (a->host[i]) cudaFreeHost(a->host[i]);
    }
    if (a->dev) cudaFree(a->dev);
    delete a;
    if (--p->n_plans == 0 && p->closed) t2sx_pool_release_object(p);
}

extern "C" int t2sx_plan_create(t2sx_pool* p, int32_t n_heads, t2sx_plan** out) {
    if (!out) return bad("t2sx_plan_create: null out");
    *out = nullptr;
    if (!p || p->closed) return bad("t2sx_plan_create: null or closed pool");
    if (n_heads <= 0 || n_heads % p->n_kv || n_heads > 65535) return bad("t2sx_plan_create: n_heads must be a positive multiple of n_kv_heads");
    return t2sx_guarded("t2sx_plan_create", [&]() -> int {
        DeviceGuard dg;
        POOL_CK(dg.set(p->device));
        std::unique_ptr<t2sx_plan, void (*)(t2sx_plan*)> a(new t2sx_plan(), plan_release);
        a->pool = p;
        a->n_heads = n_heads;
        ++p->n_plans;
        for (int i = 0; i < 2; ++i) POOL_CK(cudaEventCreateWithFlags(&a->sent[i], cudaEventDisableTiming));
        *out = a.release();
        return T2SX_OK;
    });
}

extern "C" void t2sx_plan_free(t2sx_plan* a) {
    if (a) plan_release(a);
}

extern "C" int t2sx_plan_update(t2sx_plan* a, int32_t n, const int32_t* seqs, const int32_t* n_new, void* stream) {
    if (!a || n < 0 || (n > 0 && (!seqs || !n_new))) return bad("t2sx_plan_update: bad arguments");
    t2sx_pool* p = a->pool;
    if (p->closed) return bad("t2sx_plan_update: the pool is closed");
    cudaStream_t st = (cudaStream_t)stream;
    return t2sx_guarded("t2sx_plan_update", [&]() -> int {
        int64_t rows = 0, entries = 0;
        for (int32_t i = 0; i < n; ++i) {
            if (seqs[i] < 0 || seqs[i] >= p->max_seqs || n_new[i] < 0 || n_new[i] > p->len[seqs[i]])
                return bad("t2sx_plan_update: sequence id or number of rows out of range");
            rows += n_new[i];
            entries += (int64_t)p->table[seqs[i]].size();
        }
        if (rows > (1 << 24) || entries > (1 << 28)) return bad("t2sx_plan_update: too many rows");
        for (int32_t i = 0; i < n; ++i) {
            if (p->mark[seqs[i]]) {
                for (int32_t j = 0; j < i; ++j) p->mark[seqs[j]] = 0;
                return bad("t2sx_plan_update: a sequence is given twice");
            }
            p->mark[seqs[i]] = 1;
        }
        for (int32_t i = 0; i < n; ++i) p->mark[seqs[i]] = 0;
        a->ready = false;
        DeviceGuard dg;
        POOL_CK(dg.set(p->device));
        const size_t bytes = (size_t)(2 * rows + entries) * 4;
        const int b = a->turn ^= 1;
        POOL_CK(cudaEventSynchronize(a->sent[b]));
        if (a->host_bytes[b] < bytes) {
            if (a->host[b]) POOL_CK(cudaFreeHost(a->host[b]));
            a->host[b] = nullptr;
            a->host_bytes[b] = 0;
            POOL_CK(cudaMallocHost(&a->host[b], bytes * 2));
            a->host_bytes[b] = bytes * 2;
        }
        POOL_CK(p->begin(st));
        if (a->dev_bytes < bytes) {
            POOL_CK(cudaEventSynchronize(p->done));
            if (a->dev) POOL_CK(cudaFree(a->dev));
            a->dev = nullptr;
            a->dev_bytes = 0;
            POOL_CK(cudaMalloc(&a->dev, bytes * 2));
            a->dev_bytes = bytes * 2;
        }
        int32_t *limit = (int32_t*)a->host[b], *table_at = limit + rows, *table = table_at + rows;
        int64_t r = 0, e = 0;
        for (int32_t i = 0; i < n; ++i) {
            const std::vector<int32_t>& t = p->table[seqs[i]];
            for (int32_t j = 0; j < n_new[i]; ++j, ++r) {
                limit[r] = (int32_t)(p->len[seqs[i]] - n_new[i] + j + 1);
                table_at[r] = (int32_t)e;
            }
            std::copy(t.begin(), t.end(), table + e);
            e += (int64_t)t.size();
        }
        if (bytes) POOL_CK(cudaMemcpyAsync(a->dev, a->host[b], bytes, cudaMemcpyHostToDevice, st));
        POOL_CK(cudaEventRecord(a->sent[b], st));
        POOL_CK(p->end(st));
        const int32_t* d = (const int32_t*)a->dev;
        a->view = RowView{d, d + rows, d + 2 * rows, (int)rows};
        a->rows = (int)rows;
        a->version = p->version;
        a->ready = true;
        return T2SX_OK;
    });
}

template <typename T>
static void launch_attend(t2sx_plan* a, size_t page0, const void* q, int64_t q_stride, float scale, void* out, int64_t out_stride,
                          float* lse, cudaStream_t st) {
    t2sx_pool* p = a->pool;
    const dim3 grid(a->rows, (a->n_heads + 3) / 4);
    auto go = [&](auto kernel) {
        kernel<<<grid, 128, 0, st>>>(a->view, (const T*)q, q_stride, (const T*)p->k, (const T*)p->v, page0, a->n_heads, p->n_kv,
                                     scale, (T*)out, out_stride, lse);
    };
    if (p->dim == 32) go(k_attend_rows<T, 32>);
    else if (p->dim == 64) go(k_attend_rows<T, 64>);
    else go(k_attend_rows<T, 128>);
}

extern "C" int t2sx_plan_attend(t2sx_plan* a, int32_t layer, const void* q_dev, int64_t q_stride, const void* k_new_dev,
                                const void* v_new_dev, int64_t kv_stride, float scale, void* out_dev, int64_t out_stride,
                                float* lse_dev, void* stream) {
    if (!a) return bad("t2sx_plan_attend: null plan");
    t2sx_pool* p = a->pool;
    if (p->closed) return bad("t2sx_plan_attend: the pool is closed");
    if (!a->ready || a->version != p->version)
        return t2sx_set_error(T2SX_ERR_STATE, "t2sx_plan_attend: the plan has no update since pages were released or moved");
    if (layer < 0 || layer >= p->n_layers) return bad("t2sx_plan_attend: layer out of range");
    if (a->rows == 0) return T2SX_OK;
    if (!q_dev || !out_dev || !k_new_dev != !v_new_dev) return bad("t2sx_plan_attend: null q or out, or only one of k_new and v_new");
    if (!std::isfinite(scale)) return bad("t2sx_plan_attend: scale must be finite");
    const int64_t row = (int64_t)a->n_heads * p->dim, kv_row = (int64_t)p->n_kv * p->dim;
    if (q_stride < row || out_stride < row || q_stride % 8 || out_stride % 8 || (k_new_dev && (kv_stride < kv_row || kv_stride % 8)))
        return bad("t2sx_plan_attend: strides must be multiples of 8 and no less than a row");
    if (((uintptr_t)q_dev | (uintptr_t)out_dev | (uintptr_t)k_new_dev | (uintptr_t)v_new_dev) & 15 || ((uintptr_t)lse_dev & 3))
        return bad("t2sx_plan_attend: tensors must be 16-byte aligned");
    cudaStream_t st = (cudaStream_t)stream;
    DeviceGuard dg;
    POOL_CK(dg.set(p->device));
    POOL_CK(p->begin(st));
    const size_t page0 = (size_t)layer * p->n_pages;
    if (k_new_dev) {
        const int row_vec = p->dim * 2 / 16;
        const int64_t vecs = (int64_t)a->rows * p->n_kv * row_vec;
        k_write_rows<<<(unsigned)((vecs + 255) / 256), 256, 0, st>>>(a->view, (const uint4*)k_new_dev, (const uint4*)v_new_dev,
                                                                    kv_stride / 8, (uint4*)p->k, (uint4*)p->v, page0, p->n_kv, row_vec);
        POOL_CK(cudaGetLastError());
    }
    if (p->type == T2SX_TYPE_F16) launch_attend<__half>(a, page0, q_dev, q_stride, scale, out_dev, out_stride, lse_dev, st);
    else launch_attend<__nv_bfloat16>(a, page0, q_dev, q_stride, scale, out_dev, out_stride, lse_dev, st);
    POOL_CK(cudaGetLastError());
    POOL_CK(p->end(st));
    return T2SX_OK;
}
