// Attention over shared pages for many rows: tiles of 128 rows on the tcgen05 tensor cores.
//
// A CTA takes 128 rows (tokens x query heads of one K/V head's group) against a range of pages, one page
// (64 keys) at a time:
//   warps 0-3  the softmax, one row per thread: scores from TMEM, running maximum and sum, weights back to
//              TMEM in 16 bits.  The accumulated output is rescaled only when the maximum grows by more than
//              2^8 (the weights then stay below 2^15, in the range of f16);
//   warp 4     TMA: the K and V tiles of a page, in two rings;
//   warp 5     the MMAs: S = Q K^T (M 128, N 64) into one of two score buffers, then O += P V with P from TMEM
//              (M 128, N head dim).  S of the next page is issued before O of this one, so that the tensor
//              cores work while the softmax does.
// Two CTAs share an SM (96 KB of shared memory and 256 TMEM columns each), one's softmax over the other's MMAs.
// TMEM columns: scores and weights 2 x 64, output from column 128 on.
//
// Every wait is bounded; a CTA whose wait runs out raises its abort flag, lets its copies and MMAs land, writes
// NaN and sets the plan's error word.
#include "t2sx_prefix_attn.cuh"
#include "t2sx_tcgen.cuh"

#include <mutex>

namespace t2sx {
namespace attn {
namespace {

using namespace tc;

constexpr int kKeys = kPoolPage;      // keys of a tile
constexpr int kSoftWarps = 4, kTmaWarp = 4, kMmaWarp = 5, kThreads = 192;
constexpr int kTmemCols = 256, kOutCol = 2 * kKeys;
constexpr float kHeadroom = 8.0f;     // log2 of how far weights may pass those of the reference maximum

template <int D>
struct TcShape {
    static constexpr int STAGES = D == 128 ? 2 : 4;
    static constexpr int PITCH = D == 32 ? 64 : 128;               // bytes of a row of a swizzled block
    static constexpr int HALVES = D == 128 ? 2 : 1;                // blocks of 64 dims
    static constexpr int TILE = kKeys * D * 2, Q = kTcRows * D * 2;
    static constexpr int BARS = 4 * STAGES + 2 + 2 + 3;            // K, V full and empty; scores; weights; output, end, stall
    static constexpr int SMEM = 1024 + Q + 2 * STAGES * TILE + BARS * 8 + 16;
};

// Shared-memory descriptor of an operand whose rows are PITCH bytes, swizzled within them; groups of eight rows
// follow one another.  K-major (Q, K): rows are the M or N index.  MN-major (V): rows are the K index, `lead`
// the distance of the blocks of 64 dims.
template <int PITCH>
__device__ __forceinline__ uint64_t operand(uint32_t saddr, uint32_t lead) {
    return (uint64_t)((saddr >> 4) & 0x3FFF) | (uint64_t)((lead >> 4) & 0x3FFF) << 16 | (uint64_t)((8 * PITCH) >> 4) << 32 |
           (uint64_t)1 << 46 | (uint64_t)(PITCH == 128 ? 2 : 4) << 61;
}

// kind::f16, f32 accumulators: M = 128, N, both operands f16 or bf16, B (the second) MN-major or not
template <typename T>
constexpr uint32_t instr(int n, bool b_mn) {
    const uint32_t type = std::is_same<T, __half>::value ? 0u : 1u;
    return (1u << 4) | (type << 7) | (type << 10) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kTcRows >> 4) << 24);
}

// D[tmem] (=|+=) A[smem] . B[smem]
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d), "l"(a),
                 "l"(b), "r"(idesc), "r"(acc)
                 : "memory");
}
// D[tmem] (=|+=) A[tmem] . B[smem]
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d), "r"(a),
                 "l"(b), "r"(idesc), "r"(acc)
                 : "memory");
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n" ::"r"(dst),
                 "l"((uint64_t)map), "r"(x), "r"(y), "r"(z), "r"(bar)
                 : "memory");
}

#define REGS8(v, i) "=r"(v[i]), "=r"(v[i + 1]), "=r"(v[i + 2]), "=r"(v[i + 3]), "=r"(v[i + 4]), "=r"(v[i + 5]), "=r"(v[i + 6]), "=r"(v[i + 7])
#define SRCS8(v, i) "r"(v[i]), "r"(v[i + 1]), "r"(v[i + 2]), "r"(v[i + 3]), "r"(v[i + 4]), "r"(v[i + 5]), "r"(v[i + 6]), "r"(v[i + 7])
// 32 columns of this thread's lane (tmem_wait_ld makes them readable)
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t* v) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,"
        "%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
        : REGS8(v, 0), REGS8(v, 8), REGS8(v, 16), REGS8(v, 24)
        : "r"(addr));
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t* v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,"
        "%24,%25,%26,%27,%28,%29,%30,%31};\n" ::SRCS8(v, 0),
        SRCS8(v, 8), SRCS8(v, 16), SRCS8(v, 24), "r"(addr)
        : "memory");
}
#undef REGS8
#undef SRCS8
template <int N>
__device__ __forceinline__ void tmem_wait_ld(uint32_t (&v)[N]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+r"(v[i]));   // not read before
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory"); }

__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(*reinterpret_cast<uint64_t*>(&a)), "l"(*reinterpret_cast<uint64_t*>(&b)));
    return *reinterpret_cast<float2*>(&r);
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(r)
        : "l"(*reinterpret_cast<uint64_t*>(&a)), "l"(*reinterpret_cast<uint64_t*>(&b)), "l"(*reinterpret_cast<uint64_t*>(&c)));
    return *reinterpret_cast<float2*>(&r);
}

// bar_wait of a whole warp: one answer for all of its lanes
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, long long limit) {
    return __all_sync(~0u, bar_wait(bar, parity, abort_flag, limit));
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 2)
k_attend_tc(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, PlanView pv, Tensors<T> x, int layer_page,
            int32_t* err, long long spin, int stall) {
    using S = TcShape<D>;
    constexpr int NS = S::STAGES;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    const uint32_t sq = smem_u32(smem), sk = sq + S::Q, sv = sk + NS * S::TILE, bars = sv + NS * S::TILE;
    uint8_t* tail = smem + S::Q + 2 * NS * S::TILE + S::BARS * 8;
    uint32_t* tmem_holder = (uint32_t*)tail;
    volatile int* abort_flag = (volatile int*)(tail + 4);
    auto k_full = [&](int s) { return bars + 8 * s; };
    auto k_empty = [&](int s) { return bars + 8 * (NS + s); };
    auto v_full = [&](int s) { return bars + 8 * (2 * NS + s); };
    auto v_empty = [&](int s) { return bars + 8 * (3 * NS + s); };
    auto s_full = [&](int b) { return bars + 8 * (4 * NS + b); };
    auto p_full = [&](int b) { return bars + 8 * (4 * NS + 2 + b); };
    const uint32_t o_done = bars + 8 * (4 * NS + 4), end_bar = o_done + 8, stall_bar = o_done + 16;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int kvh = blockIdx.x % pv.n_kv, group = pv.group;
    const Item it = pv.items[blockIdx.x / pv.n_kv];
    const int n = it.n_pages, soft_warps = (it.rows + 31) / 32;
    if (tid == 0) {
        for (int s = 0; s < NS; ++s) { bar_init(k_full(s), 1); bar_init(k_empty(s), 1); bar_init(v_full(s), 1); bar_init(v_empty(s), 1); }
        for (int b = 0; b < 2; ++b) { bar_init(s_full(b), 1); bar_init(p_full(b), soft_warps); }
        bar_init(o_done, 1);
        bar_init(end_bar, 1);
        bar_init(stall_bar, 1);   // no thread ever arrives on it
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(tmem_holder)), "r"(kTmemCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }
    // Q, row by row: a negative scale goes into its signs, a zero one makes it zero
    const int mr = it.row0 + tid, g = mr % group;
    const bool live = warp < kSoftWarps && tid < it.rows;
    Token tok = {};
    if (live) tok = pv.tokens[it.tokens_at + mr / group];
    const int head = kvh * group + g;
    dependents_wait();     // the step's own keys and values
    dependents_launch();   // not before: the launch after this one reads them, too
    if (warp < kSoftWarps) {
        const uint4* src = reinterpret_cast<const uint4*>(x.q + tok.row * x.q_stride + head * D);
        const uint32_t flip = x.scale2 < 0.0f ? 0x80008000u : 0u, keep = x.scale2 != 0.0f ? 0xFFFFFFFFu : 0u;
#pragma unroll
        for (int c = 0; c < D / 8; ++c) {
            uint4 w = live ? src[c] : make_uint4(0, 0, 0, 0);
            w.x = (w.x ^ flip) & keep; w.y = (w.y ^ flip) & keep; w.z = (w.z ^ flip) & keep; w.w = (w.w ^ flip) & keep;
            const int at = D == 32 ? tid * 64 + ((c ^ (tid >> 1)) & 3) * 16 : (c >> 3) * (kTcRows * 128) + tid * 128 + ((c ^ tid) & 7) * 16;
            *reinterpret_cast<uint4*>(smem + at) = w;
        }
        fence_proxy_async_smem();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_holder;
    const float scale = x.scale2 == 0.0f ? 1.0f : fabsf(x.scale2);

    float m = -INFINITY, l = 0.0f;
    bool gone = false;
    if (warp == kTmaWarp) {
        // ---- copies ----
        int page = 0, j = 0;
        for (; j < n; ++j) {
            if ((j & 31) == 0) page = j + lane < n ? pv.pages[it.pages_at + j + lane] : 0;
            const int z = layer_page + __shfl_sync(~0u, page, j & 31), s = j % NS;
            int ok = 1;
            if (lane == 0) {
                const uint32_t phase = ((j / NS) & 1) ^ 1;
                ok = bar_wait(k_empty(s), phase, abort_flag, spin);
                if (ok) {
                    bar_expect_tx(k_full(s), S::TILE);
                    for (int h = 0; h < S::HALVES; ++h) tma_load_3d(sk + s * S::TILE + h * (kKeys * 128), &map_k, h * 64, kvh * kKeys, z, k_full(s));
                    ok = bar_wait(v_empty(s), phase, abort_flag, spin);
                    if (ok) {
                        bar_expect_tx(v_full(s), S::TILE);
                        for (int h = 0; h < S::HALVES; ++h) tma_load_3d(sv + s * S::TILE + h * (kKeys * 128), &map_v, h * 64, kvh * kKeys, z, v_full(s));
                    } else {
                        ok = 2;   // K of this page is under way
                    }
                }
            }
            ok = __shfl_sync(~0u, ok, 0);
            if (ok != 1) {
                gone = true;
                if (lane == 0) {   // let what was requested land before the CTA ends
                    const int k_end = ok == 2 ? j + 1 : j;
                    for (int i = max(0, k_end - NS); i < k_end; ++i) {
                        const long long t0 = clock64();
                        while (!bar_try(k_full(i % NS), (i / NS) & 1) && clock64() - t0 < kSpinCycles) {}
                    }
                    for (int i = max(0, j - NS); i < j; ++i) {
                        const long long t0 = clock64();
                        while (!bar_try(v_full(i % NS), (i / NS) & 1) && clock64() - t0 < kSpinCycles) {}
                    }
                }
                break;
            }
        }
        if (!gone && lane == 0) {   // the end of a CTA that is given up elsewhere: the last copies have landed
            for (int i = max(0, n - NS); i < n; ++i) {
                const long long t0 = clock64();
                while (!(bar_try(k_full(i % NS), (i / NS) & 1) && bar_try(v_full(i % NS), (i / NS) & 1)) && clock64() - t0 < kSpinCycles) {}
            }
        }
        __syncwarp();
    } else if (warp == kMmaWarp) {
        // ---- MMAs ----
        constexpr uint32_t idesc_s = instr<T>(kKeys, false), idesc_o = instr<T>(D, true);
        auto scores = [&](int j) {   // S(j) = Q K(j)^T
            const int s = j % NS;
            if (!warp_wait(k_full(s), (j / NS) & 1, abort_flag, spin)) return false;
            tc_fence_after();
            if (lane == 0) {
#pragma unroll
                for (int k = 0; k < D / 16; ++k) {
                    const uint32_t qa = sq + (k / 4) * (D == 32 ? 0 : kTcRows * 128) + (k % 4) * 32;
                    const uint32_t ka = sk + s * S::TILE + (k / 4) * (D == 32 ? 0 : kKeys * 128) + (k % 4) * 32;
                    mma_ss(tmem + (j & 1) * kKeys, operand<S::PITCH>(qa, 16), operand<S::PITCH>(ka, 16), idesc_s, k > 0);
                }
                tc_commit(k_empty(s));
                tc_commit(s_full(j & 1));
            }
            __syncwarp();
            return true;
        };
        gone = !scores(0);
        for (int j = 0; j < n && !gone; ++j) {
            if (j + 1 < n && !scores(j + 1)) { gone = true; break; }
            const int s = j % NS;
            if (!warp_wait(v_full(s), (j / NS) & 1, abort_flag, spin)) { gone = true; break; }
            const int filled = it.end - (it.pos0 + j * kKeys);
            if (filled < kKeys) {
                // what stands beyond the filled positions may be NaN: as values (times the weight 0) it counts 0
                uint8_t* vt = smem + S::Q + NS * S::TILE + s * S::TILE;
                for (int h = 0; h < S::HALVES; ++h)
                    for (int b = filled * S::PITCH + lane * 16; b < kKeys * S::PITCH; b += 512)
                        *reinterpret_cast<uint4*>(vt + h * (kKeys * 128) + b) = make_uint4(0, 0, 0, 0);
                fence_proxy_async_smem();
                __syncwarp();
            }
            if (!warp_wait(p_full(j & 1), (j >> 1) & 1, abort_flag, spin)) { gone = true; break; }
            tc_fence_after();
            if (lane == 0) {
#pragma unroll
                for (int k = 0; k < kKeys / 16; ++k)
                    mma_ts(tmem + kOutCol, tmem + (j & 1) * kKeys + k * 8, operand<S::PITCH>(sv + s * S::TILE + k * 16 * S::PITCH, kKeys * 128),
                           idesc_o, j > 0 || k > 0);
                tc_commit(v_empty(s));
                tc_commit(o_done);
            }
            __syncwarp();
        }
        if (lane == 0) {   // all MMAs: the output is whole, and nothing reads shared memory any more
            tc_commit(end_bar);
            const long long t0 = clock64();
            while (!bar_try(end_bar, 0) && clock64() - t0 < kSpinCycles) {}
        }
        __syncwarp();
    } else if (warp < soft_warps) {
        // ---- softmax: one row per thread ----
        const uint32_t lanes = tmem + ((uint32_t)(warp * 32) << 16);
        const int limit = live ? tok.limit : INT32_MAX;
        int free_to = limit;
        for (int y = 16; y; y >>= 1) free_to = min(free_to, __shfl_xor_sync(~0u, free_to, y));
        for (int j = 0; j < n; ++j) {
            const int b = j & 1, pos = it.pos0 + j * kKeys;
            if ((stall && j == 0 && !warp_wait(stall_bar, 0, abort_flag, spin)) || !warp_wait(s_full(b), (j >> 1) & 1, abort_flag, spin)) {
                gone = true;
                break;
            }
            tc_fence_after();
            uint32_t sc[kKeys];
            tmem_ld32(lanes + b * kKeys, sc);
            tmem_ld32(lanes + b * kKeys + 32, sc + 32);
            tmem_wait_ld(sc);
            if (pos + kKeys > free_to) {
                const int seen = limit - pos;
#pragma unroll
                for (int c = 0; c < kKeys; ++c)
                    if (c >= seen) sc[c] = 0xFF800000u;
            }
            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int c = 0; c < kKeys; c += 8)
#pragma unroll
                for (int e = 0; e < 4; ++e) mx[e] = fmaxf(mx[e], fmaxf(__uint_as_float(sc[c + 2 * e]), __uint_as_float(sc[c + 2 * e + 1])));
            const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * scale;
            const bool grew = top > m + kHeadroom;   // also when there was none before
            if (__any_sync(~0u, grew)) {
                const float f = grew ? (m == -INFINITY ? 0.0f : ex2(m - top)) : 1.0f;
                if (grew) m = top;
                l *= f;
                if (j > 0) {   // (the scores of j came after the output of page j - 2)
                    if (!warp_wait(o_done, (j - 1) & 1, abort_flag, spin)) { gone = true; break; }
                    tc_fence_after();
#pragma unroll
                    for (int c = 0; c < D; c += 32) {
                        uint32_t o[32];
                        tmem_ld32(lanes + kOutCol + c, o);
                        tmem_wait_ld(o);
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                        tmem_st32(lanes + kOutCol + c, o);
                    }
                }
            }
            const float base = m == -INFINITY ? 0.0f : kWeightExp - m;
            float2 sum[2] = {{0.0f, 0.0f}, {0.0f, 0.0f}};
            uint32_t p[kKeys / 2];
#pragma unroll
            for (int c = 0; c < kKeys / 2; ++c) {
                const float2 y = fma2(make_float2(__uint_as_float(sc[2 * c]), __uint_as_float(sc[2 * c + 1])), make_float2(scale, scale), make_float2(base, base));
                const float2 e = make_float2(ex2(y.x), ex2(y.y));
                sum[c & 1] = add2(sum[c & 1], e);
                p[c] = pack2(T(), e.x, e.y);
            }
            l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
            tmem_st32(lanes + b * kKeys, p);
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) bar_arrive(p_full(b));
            __syncwarp();
        }
        // (not o_done: two of its phases may be outstanding here, which a wait by parity does not tell apart)
        if (!gone && !warp_wait(end_bar, 0, abort_flag, spin)) gone = true;
        tc_fence_after();
        gone = __any_sync(~0u, gone);
        const bool counts = live && tok.limit > it.pos0, whole = tok.n_parts == 1;
        const size_t part = ((size_t)(tok.part0 + it.split) * group + g) * pv.n_kv + kvh;
        const float inv = gone ? NAN : l > 0.0f ? 1.0f / l : 0.0f;
#pragma unroll
        for (int c = 0; c < D; c += 32) {
            uint32_t o[32];
            if (!gone) {
                tmem_ld32(lanes + kOutCol + c, o);
                tmem_wait_ld(o);
            } else {
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] = 0x7FC00000u;
            }
            if (!counts) continue;
            if (whole) {
                uint4* dst = reinterpret_cast<uint4*>(x.out + tok.row * x.out_stride + head * D + c);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t w[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        w[e] = pack2(T(), __uint_as_float(o[8 * i + 2 * e]) * inv, __uint_as_float(o[8 * i + 2 * e + 1]) * inv);
                    dst[i] = make_uint4(w[0], w[1], w[2], w[3]);
                }
            } else {
                uint4* dst = reinterpret_cast<uint4*>(pv.part_o + part * D + c);
#pragma unroll
                for (int i = 0; i < 8; ++i) dst[i] = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
            }
        }
        if (counts) {
            if (gone) l = NAN;
            if (!whole) pv.part_ml[part] = make_float2(gone ? 0.0f : m, l);
            else if (x.lse)
                x.lse[(size_t)tok.row * (pv.n_kv * group) + head] = gone ? NAN : l > 0.0f ? (m - kWeightExp + log2f(l)) * kLn2 : -INFINITY;
        }
    }
    tc_fence_before();
    __syncthreads();
    if (*abort_flag && tid == 0) {
        *(volatile int32_t*)err = kErrTimeout;
        __threadfence_system();
    }
    if (warp == kMmaWarp) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(kTmemCols) : "memory");
    }
}

template <typename T, int D>
cudaError_t run(const PlanView& w, const Tensors<T>& x, const CUtensorMap& k, const CUtensorMap& v, int layer_page, int32_t* err, bool early,
                int device, cudaStream_t st) {
    static std::once_flag once[64];
    std::call_once(once[device & 63],
                   [] { cudaFuncSetAttribute(k_attend_tc<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, TcShape<D>::SMEM); });
    const long long test = tc_test_wait_cycles();
    return launch(k_attend_tc<T, D>, dim3((unsigned)w.n_tc * w.n_kv), kThreads, TcShape<D>::SMEM, st, early, k, v, w, x, layer_page, err,
                  test > 0 ? test : kSpinCycles, test > 0 ? 1 : 0);
}

}  // namespace

// The storage as [layer and page][K/V head x position][dim]; a tile is one head's 64 positions of up to 64 dims.
bool tc_maps(const t2sx_pool* p, CUtensorMap* k, CUtensorMap* v) {
    auto fn = encode_fn();
    if (!fn) return false;
    const cuuint64_t dims[3] = {(cuuint64_t)p->dim, (cuuint64_t)p->n_kv * kPoolPage, (cuuint64_t)p->n_layers * p->n_pages};
    const cuuint64_t strides[2] = {(cuuint64_t)p->dim * 2, (cuuint64_t)p->dim * 2 * p->n_kv * kPoolPage};
    const cuuint32_t box[3] = {(cuuint32_t)(p->dim < 64 ? p->dim : 64), (cuuint32_t)kPoolPage, 1}, steps[3] = {1, 1, 1};
    for (int i = 0; i < 2; ++i)
        if (fn(i ? v : k, CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, i ? p->v : p->k, dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
               p->dim == 32 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
            return false;
    return true;
}

template <typename T>
cudaError_t launch_tc(const PlanView& w, const Tensors<T>& x, const t2sx_pool* p, const CUtensorMap& k, const CUtensorMap& v, int layer_page,
                      int32_t* err, bool early, cudaStream_t st) {
    if (p->dim == 32) return run<T, 32>(w, x, k, v, layer_page, err, early, p->device, st);
    if (p->dim == 64) return run<T, 64>(w, x, k, v, layer_page, err, early, p->device, st);
    return run<T, 128>(w, x, k, v, layer_page, err, early, p->device, st);
}
template cudaError_t launch_tc<__half>(const PlanView&, const Tensors<__half>&, const t2sx_pool*, const CUtensorMap&, const CUtensorMap&, int,
                                       int32_t*, bool, cudaStream_t);
template cudaError_t launch_tc<__nv_bfloat16>(const PlanView&, const Tensors<__nv_bfloat16>&, const t2sx_pool*, const CUtensorMap&,
                                              const CUtensorMap&, int, int32_t*, bool, cudaStream_t);

}  // namespace attn
}  // namespace t2sx
