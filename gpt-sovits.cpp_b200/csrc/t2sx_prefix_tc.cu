// Attention over shared pages for many rows: tiles of 128 rows on the tcgen05 tensor cores.
//
// A CTA, one per SM, has two tiles of 128 rows (tokens x query heads of one K/V head's group) and a range of
// pages, and takes one page (64 keys) at a time.  An item of more than 128 rows fills both tiles, and each
// page's K and V serve both; a smaller one is in both, with every second page, and the two results are joined
// at the end.
//   warps 0-7  the softmax, one row per thread: scores from TMEM, weights back to TMEM in 16 bits, their sum.
//              (the sum is of the weights before that rounding, in f32).  The maximum that the weights refer to
//              is looked for, and the output rescaled, only when a tile's weights add up to 2^15 (f16 ends at 2^16);
//   warp 8     TMA: the K and V tiles of the pages, in two rings;
//   warps 9-10 the MMAs, one thread for each tile: S = Q K^T (M 128, N 64) into one of two score buffers of a
//              tile, then O += P V with P from TMEM (M 128, N head dim).  S is issued two pages ahead, so that the
//              tensor cores work while the softmax does.
// TMEM columns of a tile: scores and weights 2 x 64, output from column 128 on.
//
// What bounds it: the tensor cores.  An MMA of M 128 and N 64 takes as long as one of N 128 (64 cycles for 16 of
// the K index), so a page costs the two tiles 2 x (8 x 64 + 4 x 64) = 1536 cycles at head dim 128, and the loop takes
// 1526.  At head dim 64 the MMAs take 1024 and the exponentials (8 cycles to a warp's instruction) 1066, but the loop
// 1555: a third of it is one waiting for the other.  A step of 256 sequences over one prompt of 16384 positions (32 heads, 8 K/V heads
// of 128 dims, bf16; up to 256 positions each of their own) takes 103 us a call, calls one after another.  By itself, from cold caches,
// this kernel takes 79 of it: 64 pages are 58 at the 1.67 GHz that it runs at, a CTA's start and end most of the rest.
// When the call took 116, it took with
//   scores of 128 keys in one buffer (N 128): 135, and 128 with 16 softmax warps, since the MMAs then wait for the
//              softmax; there is no TMEM for a second buffer of that size beside two outputs;
//   one tile per CTA, two CTAs per SM: 153;    16 softmax warps on these buffers: 117;
//   the tiles' softmax taking turns: 146;      a polynomial for 4 of 32 pairs of exponentials: 113, for 8: 117.
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
constexpr int kTileM = kTcRows / 2;   // rows of a tile
constexpr int kSoftWarps = 8, kTmaWarp = 8, kMmaWarp = 9, kThreads = 352;   // one MMA warp per tile
constexpr int kTileCols = 256, kTmemCols = 2 * kTileCols, kOutCol = 2 * kKeys;
constexpr int kAhead = 4;   // pages that a CTA asks for at its start, no more than the rings hold
// A tile's weights against the reference maximum add up to less than this, or the reference is moved: f16 ends at
// 2^16, and 64 weights at the reference itself make 2^13.
constexpr float kSumLimit = 32768.0f;

template <int D>
struct TcShape {
    // even: where the tiles take every second page, a stage is always the same tile's, whose thread then sees all phases
    // of its barriers (a wait by parity does not tell a phase from the one before the last)
    static constexpr int STAGES = D == 128 ? 4 : 8;
    static_assert(STAGES % 2 == 0, "see above");
    static_assert(STAGES >= kAhead, "the first pages wait for no stage");
    static constexpr int PITCH = D == 32 ? 64 : 128;               // bytes of a row of a swizzled block
    static constexpr int HALVES = D == 128 ? 2 : 1;                // blocks of 64 dims
    static constexpr int TILE = kKeys * D * 2, Q = kTileM * D * 2;
    static constexpr int BARS = 4 * STAGES + 2 * (2 + 2 + 1) + 4;  // K, V full and empty; a tile's scores, weights, output; end, stall, tail, zero
    static constexpr int SMEM = 1024 + 2 * Q + 2 * STAGES * TILE + BARS * 8 + kTileM * 8 + 16;
    static_assert(2 * Q + 2 * STAGES * TILE >= 2 * kTileM * (D + 4) * 4, "the tiles' outputs take the place of Q and the rings");
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
    return (1u << 4) | (type << 7) | (type << 10) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kTileM >> 4) << 24);
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

// A wait of all threads of a warp, whose next instruction may be one that takes the warp as a whole (.sync.aligned: the loads
// and stores of TMEM, a named barrier).  Each thread leaves the wait's loop by itself; the warp is brought together again here.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, long long limit) {
    const bool ok = bar_wait(bar, parity, abort_flag, limit);
    __syncwarp();
    return ok;
}
// True in one lane of the warp, the leader.  The compiler knows that only one thread passes, and needs no loop around
// the instructions that take their operands from uniform registers.
__device__ __forceinline__ bool elect_one(uint32_t& leader) {
    uint32_t r;
    asm volatile("{\n.reg .pred p;\nelect.sync %1|p, 0xFFFFFFFF;\nselp.u32 %0, 1, 0, p;\n}\n" : "=r"(r), "=r"(leader));
    return r != 0;
}
// The steps of weights(), volatile so that they stay in its order.
__device__ __forceinline__ void v_fma2(float2& d, float2 a, float2 b, float2 c) {
    uint64_t r;
    asm volatile("fma.rn.f32x2 %0, %1, %2, %3;"
                 : "=l"(r)
                 : "l"(*reinterpret_cast<uint64_t*>(&a)), "l"(*reinterpret_cast<uint64_t*>(&b)), "l"(*reinterpret_cast<uint64_t*>(&c)));
    d = *reinterpret_cast<float2*>(&r);
}
__device__ __forceinline__ void v_add2(float2& d, float2 a) {
    uint64_t r;
    asm volatile("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(*reinterpret_cast<uint64_t*>(&d)), "l"(*reinterpret_cast<uint64_t*>(&a)));
    d = *reinterpret_cast<float2*>(&r);
}
__device__ __forceinline__ void v_ex2(float& x) { asm volatile("ex2.approx.ftz.f32 %0, %0;" : "+f"(x)); }
__device__ __forceinline__ void v_pack2(__half, uint32_t& d, float2 a) { asm volatile("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(a.y), "f"(a.x)); }
__device__ __forceinline__ void v_pack2(__nv_bfloat16, uint32_t& d, float2 a) {
    asm volatile("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(a.y), "f"(a.x));
}

// The softmax weights of a row's scores in 16 bits, two to a word, and their sum: 2^(scale s - m + kWeightExp).
// The exponential unit takes a warp's instruction every 8 cycles, and a warp issues in order: the multiplications of
// later scores and the additions and conversions of earlier ones stand between the exponentials, which then follow
// one another without a pause (left to the compiler the 64 of them took 1000 cycles instead of 610).
template <typename T>
__device__ __forceinline__ float weights(const uint32_t (&sc)[kKeys], uint32_t (&p)[kKeys / 2], float scale, float m) {
    constexpr int N = kKeys / 2, AHEAD = 4, LAG = 3;
    const float base = m == -INFINITY ? 0.0f : kWeightExp - m;
    const float2 scale2 = make_float2(scale, scale), base2 = make_float2(base, base);
    float2 y[N], sum[2] = {{0.0f, 0.0f}, {0.0f, 0.0f}};
    auto multiply = [&](int c) { v_fma2(y[c], make_float2(__uint_as_float(sc[2 * c]), __uint_as_float(sc[2 * c + 1])), scale2, base2); };
#pragma unroll
    for (int c = 0; c < AHEAD; ++c) multiply(c);
#pragma unroll
    for (int c = 0; c < N + LAG; ++c) {
        if (c < N) v_ex2(y[c].x);
        if (c + AHEAD < N) multiply(c + AHEAD);
        if (c >= LAG) v_add2(sum[c & 1], y[c - LAG]);
        if (c < N) v_ex2(y[c].y);
        if (c >= LAG) v_pack2(T(), p[c - LAG], y[c - LAG]);
    }
    return (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1)
k_attend_tc(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, PlanView pv, Tensors<T> x, int layer_page,
            int32_t* err, long long spin, int stall) {
    using S = TcShape<D>;
    constexpr int NS = S::STAGES;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint8_t* rings = smem + 2 * S::Q;
    const uint32_t sq = smem_u32(smem), sk = smem_u32(rings), sv = sk + NS * S::TILE, bars = sv + NS * S::TILE;
    float2* tile1_ml = (float2*)(rings + 2 * NS * S::TILE + S::BARS * 8);
    uint32_t* tmem_holder = (uint32_t*)(tile1_ml + kTileM);
    volatile int* abort_flag = (volatile int*)(tmem_holder + 1);
    auto k_full = [&](int s) { return bars + 8 * s; };
    auto k_empty = [&](int s) { return bars + 8 * (NS + s); };
    auto v_full = [&](int s) { return bars + 8 * (2 * NS + s); };
    auto v_empty = [&](int s) { return bars + 8 * (3 * NS + s); };
    auto s_full = [&](int tile, int b) { return bars + 8 * (4 * NS + tile * 5 + b); };
    auto p_full = [&](int tile, int b) { return bars + 8 * (4 * NS + tile * 5 + 2 + b); };
    auto o_done = [&](int tile) { return bars + 8 * (4 * NS + tile * 5 + 4); };
    const uint32_t end_bar = bars + 8 * (4 * NS + 10), stall_bar = end_bar + 8, tail_bar = end_bar + 16, zero_bar = end_bar + 24;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int kvh = blockIdx.x % pv.n_kv, group = pv.group;
    const Item it = pv.items[blockIdx.x / pv.n_kv];
    const bool alternate = it.rows <= kTileM;   // both tiles have the item's rows, and every second page
    const int n = it.n_pages;
    // a tile's pages are numbers 0 .. pages_of_tile - 1: which one of the item's
    auto tile_pages = [&](int tile) { return alternate ? (n - tile + 1) / 2 : n; };
    auto tile_rows = [&](int tile) { return alternate ? it.rows : min(kTileM, it.rows - tile * kTileM); };
    auto nth = [&](int tile, int k) { return alternate ? 2 * k + tile : k; };
    if (warp == kTmaWarp && lane == 0) {
        const int users = alternate ? 1 : 2;   // tiles that read a page
        for (int s = 0; s < NS; ++s) { bar_init(k_full(s), 1); bar_init(k_empty(s), users); bar_init(v_full(s), 1); bar_init(v_empty(s), users); }
        for (int tile = 0; tile < 2; ++tile) {
            for (int b = 0; b < 2; ++b) { bar_init(s_full(tile, b), 1); bar_init(p_full(tile, b), (tile_rows(tile) + 31) / 32); }
            bar_init(o_done(tile), 1);
        }
        bar_init(end_bar, 2);
        bar_init(stall_bar, 1);   // no thread ever arrives on it
        bar_init(tail_bar, 1);
        bar_init(zero_bar, 31);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
        fence_proxy_async_smem();
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(tmem_holder)), "r"(kTmemCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }
    // Q, row by row: a negative scale goes into its signs, a zero one makes it zero
    const int tile = (warp >> 2) & 1, r = tid & (kTileM - 1);   // of a softmax thread
    const int mr = it.row0 + r + (alternate ? 0 : tile * kTileM), g = mr % group;
    const bool live = warp < kSoftWarps && r < tile_rows(tile);
    Token tok = {};
    if (live) tok = pv.tokens[it.tokens_at + mr / group];
    const int head = kvh * group + g;
    dependents_wait();     // the step's own keys and values
    dependents_launch();   // not before: the launch after this one reads them, too
    auto load_k = [&](int j, int z) {
        const int s = j % NS;
        bar_expect_tx(k_full(s), S::TILE);
        for (int h = 0; h < S::HALVES; ++h) tma_load_3d(sk + s * S::TILE + h * (kKeys * 128), &map_k, h * 64, kvh * kKeys, z, k_full(s));
    };
    auto load_v = [&](int j, int z) {
        const int s = j % NS;
        bar_expect_tx(v_full(s), S::TILE);
        for (int h = 0; h < S::HALVES; ++h) tma_load_3d(sv + s * S::TILE + h * (kKeys * 128), &map_v, h * 64, kvh * kKeys, z, v_full(s));
    };
    const int ahead = min(n, kAhead);
    int page = 0;
    if (warp == kTmaWarp) {   // the first pages come while the others fetch Q
        page = lane < n ? pv.pages[it.pages_at + lane] : 0;
        for (int j = 0; j < ahead; ++j) {
            const int z = layer_page + __shfl_sync(~0u, page, j);
            if (lane == 0) { load_k(j, z); load_v(j, z); }
        }
        __syncwarp();
    }
    if (warp < kSoftWarps && !(alternate && tile == 1)) {
        // a warp's 32 rows, neighbouring lanes on neighbouring 16-byte words of a row
        constexpr int W = D / 8, R = 32 / W;
        const uint32_t flip = x.scale2 < 0.0f ? 0x80008000u : 0u, keep = x.scale2 != 0.0f ? 0xFFFFFFFFu : 0u;
        const int c = lane % W;
        const T* mine = x.q + tok.row * x.q_stride + head * D;
        uint4 w[32 / R];   // all loads before the stores, which they are not known to differ from
#pragma unroll
        for (int i = 0; i < 32 / R; ++i) {
            const int from = i * R + lane / W, rr = (warp & 3) * 32 + from;
            const uint4* src = reinterpret_cast<const uint4*>(__shfl_sync(~0u, (unsigned long long)mine, from));
            w[i] = rr < tile_rows(tile) ? src[c] : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < 32 / R; ++i) {
            const int rr = (warp & 3) * 32 + i * R + lane / W;
            uint4 u = w[i];
            u.x = (u.x ^ flip) & keep; u.y = (u.y ^ flip) & keep; u.z = (u.z ^ flip) & keep; u.w = (u.w ^ flip) & keep;
            const int at = D == 32 ? rr * 64 + ((c ^ (rr >> 1)) & 3) * 16 : (c >> 3) * (kTileM * 128) + rr * 128 + ((c ^ rr) & 7) * 16;
            *reinterpret_cast<uint4*>(smem + tile * S::Q + at) = u;
        }
        fence_proxy_async_smem();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_holder;
    const float scale = x.scale2 == 0.0f ? 1.0f : fabsf(x.scale2);

    bool gone = false;
    if (warp == kTmaWarp) {
        // ---- copies ----
        int j = ahead;
        for (; j < n; ++j) {
            if ((j & 31) == 0) page = j + lane < n ? pv.pages[it.pages_at + j + lane] : 0;
            const int z = layer_page + __shfl_sync(~0u, page, j & 31), s = j % NS;
            int ok = 1;
            if (lane == 0) {
                const uint32_t phase = ((j / NS) & 1) ^ 1;
                ok = bar_wait(k_empty(s), phase, abort_flag, spin);
                if (ok) {
                    load_k(j, z);
                    ok = bar_wait(v_empty(s), phase, abort_flag, spin);
                    if (ok) load_v(j, z);
                    else ok = 2;   // K of this page is under way
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
    } else if (warp >= kMmaWarp) {
        // ---- MMAs: one thread for each tile ----
        constexpr uint32_t idesc_s = instr<T>(kKeys, false), idesc_o = instr<T>(D, true);
        const int tile = warp - kMmaWarp, nt = tile_pages(tile);
        const int filled = it.end - (it.pos0 + (n - 1) * kKeys), last = (n - 1) % NS;
        const bool clears = filled < kKeys && (alternate ? tile == ((n - 1) & 1) : tile == 0);   // this warp's lanes see to the rest
        uint32_t leader;
        if (elect_one(leader)) {
            const uint64_t q_desc = operand<S::PITCH>(sq + (alternate ? 0 : tile * S::Q), 16), k_desc = operand<S::PITCH>(sk, 16),
                           v_desc = operand<S::PITCH>(sv, kKeys * 128);
            const uint32_t cols = tmem + tile * kTileCols;
            auto scores = [&](int k) {   // S = Q K^T of the tile's k-th page
                const int j = nth(tile, k), s = j % NS;
                if (!bar_wait(k_full(s), (j / NS) & 1, abort_flag, spin)) return false;
                const uint64_t kd = k_desc + s * (S::TILE >> 4);
                const uint32_t d = cols + (k & 1) * kKeys;
#pragma unroll
                for (int i = 0; i < D / 16; ++i)
                    mma_ss(d, q_desc + (((i / 4) * (kTileM * 128) + (i % 4) * 32) >> 4), kd + (((i / 4) * (kKeys * 128) + (i % 4) * 32) >> 4), idesc_s,
                           i > 0);
                tc_commit(s_full(tile, k & 1));
                tc_commit(k_empty(s));
                return true;
            };
            auto outputs = [&](int k) {   // O += P V
                const int j = nth(tile, k), s = j % NS;
                if (!bar_wait(v_full(s), (j / NS) & 1, abort_flag, spin)) return false;
                if (filled < kKeys && j == n - 1) {
                    if (clears) bar_arrive(tail_bar);
                    if (!bar_wait(zero_bar, 0, abort_flag, spin)) return false;
                }
                if (!bar_wait(p_full(tile, k & 1), (k >> 1) & 1, abort_flag, spin)) return false;
                tc_fence_after();
                const uint64_t vd = v_desc + s * (S::TILE >> 4);
                const uint32_t d = cols + kOutCol, pa = cols + (k & 1) * kKeys;
#pragma unroll
                for (int i = 0; i < kKeys / 16; ++i) mma_ts(d, pa + i * 8, vd + ((i * 16 * S::PITCH) >> 4), idesc_o, i > 0 ? 1u : (uint32_t)(k > 0));
                tc_commit(o_done(tile));
                tc_commit(v_empty(s));
                return true;
            };
            // Two pages' scores ahead: S(k + 2) follows O(k), whose weights were in the same score buffer (MMAs of
            // a thread run in order).
            gone = (nt > 0 && !scores(0)) || (nt > 1 && !scores(1));
            for (int k = 0; k < nt && !gone; ++k) gone = !outputs(k) || (k + 2 < nt && !scores(k + 2));
            // all MMAs: the output is whole, and nothing reads shared memory any more
            tc_commit(end_bar);
            const long long t0 = clock64();
            while (!bar_try(end_bar, 0) && clock64() - t0 < kSpinCycles) {}
        } else if (clears) {
            // The other lanes: what stands beyond the filled positions of the last page may be NaN; as values (times
            // the weight 0) it counts 0.
            if (bar_wait(tail_bar, 0, abort_flag, spin)) {
                uint8_t* vt = rings + NS * S::TILE + last * S::TILE;
                const int words = (kKeys - filled) * (S::PITCH / 16);
                const int rank = (lane - (int)leader - 1) & 31;   // 0 .. 30
                for (int h = 0; h < S::HALVES; ++h)
                    for (int i = rank; i < words; i += 31)
                        *reinterpret_cast<uint4*>(vt + h * (kKeys * 128) + filled * S::PITCH + i * 16) = make_uint4(0, 0, 0, 0);
                fence_proxy_async_smem();
                bar_arrive(zero_bar);
            }
        }
        __syncwarp();
    } else if (warp < kSoftWarps && (warp & 3) < (tile_rows(tile) + 31) / 32 && tile_pages(tile) > 0) {
        // ---- softmax: one row per thread ----
        const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16) + tile * kTileCols;
        const int limit = live ? tok.limit : INT32_MAX, nt = tile_pages(tile);
        float m = -INFINITY, l = 0.0f;
        int free_to = limit;
        for (int y = 16; y; y >>= 1) free_to = min(free_to, __shfl_xor_sync(~0u, free_to, y));
        // In this loop a wait that is given up changes nothing in what the warp does: it goes on with whatever it finds,
        // and its results are replaced at the end.
        if (stall) gone = !bar_wait(stall_bar, 0, abort_flag, spin);
        for (int k = 0; k < nt; ++k) {
            const int b = k & 1, pos = it.pos0 + nth(tile, k) * kKeys;
            gone |= !warp_wait(s_full(tile, b), (k >> 1) & 1, abort_flag, spin);
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
            // Weights against the reference maximum so far; they are right unless one passes 2^15, and then the sum does.
            uint32_t p[kKeys / 2];
            float sum = weights<T>(sc, p, scale, m);
            const bool grew = !(sum < kSumLimit) || m == -INFINITY;
            if (__any_sync(~0u, grew)) {
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int c = 0; c < kKeys; c += 8)
#pragma unroll
                    for (int e = 0; e < 4; ++e) mx[e] = fmaxf(mx[e], fmaxf(__uint_as_float(sc[c + 2 * e]), __uint_as_float(sc[c + 2 * e + 1])));
                const float top = fmaxf(m, fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * scale);
                const float f = !grew ? 1.0f : m == -INFINITY ? 0.0f : ex2(m - top);
                if (grew) m = top;
                l *= f;
                if (k > 0) {   // (the scores of k came after the output of page k - 2)
                    gone |= !warp_wait(o_done(tile), (k - 1) & 1, abort_flag, spin);
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
                sum = weights<T>(sc, p, scale, m);
            }
            l += sum;
            tmem_st32(lanes + b * kKeys, p);
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) bar_arrive(p_full(tile, b));
            __syncwarp();
        }
        // (not o_done: two of its phases may be outstanding here, which a wait by parity does not tell apart)
        gone |= !warp_wait(end_bar, 0, abort_flag, spin);
        gone = __any_sync(~0u, gone);
        tc_fence_after();
        // The output goes through shared memory (the place of Q and the rings), row by row, so that neighbouring lanes write
        // neighbouring words of a row; rows are four words apart in the banks.
        constexpr int ROW = D + 4;
        float* stage = reinterpret_cast<float*>(smem) + (size_t)(tile * kTileM + r) * ROW;
        const bool two = alternate && n > 1;   // this row's other half is in the other tile
        const bool writes = !two || tile == 0;
        float f0 = 1.0f, f1 = 0.0f;
        if (two) {
            if (tile == 1) {
                tile1_ml[r] = make_float2(m, gone ? NAN : l);
#pragma unroll
                for (int c = 0; c < D; c += 32) {
                    uint32_t o[32];
                    tmem_ld32(lanes + kOutCol + c, o);
                    tmem_wait_ld(o);
#pragma unroll
                    for (int i = 0; i < 32; i += 4) *reinterpret_cast<uint4*>(stage + c + i) = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
                }
            }
            asm volatile("bar.sync 1, %0;" ::"r"(64 * ((it.rows + 31) / 32)) : "memory");
            if (tile == 0) {
                const float2 o = tile1_ml[r];
                const float M = fmaxf(m, o.x);
                f0 = m == -INFINITY ? 0.0f : ex2(m - M);
                f1 = o.x == -INFINITY ? 0.0f : ex2(o.x - M);
                m = M;
                l = fmaf(l, f0, o.y * f1);
                gone |= !(o.y == o.y);
            }
        }
        if (writes) {
            const bool counts = live && tok.limit > it.pos0, whole = tok.n_parts == 1;
            const size_t part = ((size_t)(tok.part0 + it.split) * group + g) * pv.n_kv + kvh;
            const float inv = gone ? NAN : !whole ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
            for (int c = 0; c < D; c += 32) {
                uint32_t o[32];
                tmem_ld32(lanes + kOutCol + c, o);
                tmem_wait_ld(o);
#pragma unroll
                for (int i = 0; i < 32; i += 4) {
                    float4 y = make_float4(__uint_as_float(o[i]), __uint_as_float(o[i + 1]), __uint_as_float(o[i + 2]), __uint_as_float(o[i + 3]));
                    if (two) {
                        const float4 z = *reinterpret_cast<const float4*>(stage + kTileM * ROW + c + i);
                        y = make_float4(fmaf(y.x, f0, z.x * f1), fmaf(y.y, f0, z.y * f1), fmaf(y.z, f0, z.z * f1), fmaf(y.w, f0, z.w * f1));
                    }
                    *reinterpret_cast<float4*>(stage + c + i) = make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv);
                }
            }
            __syncwarp();
            constexpr int W = D / 4, R = 32 / W;   // lanes of a row, rows of the warp at a time
            const char* to = reinterpret_cast<const char*>(whole ? (const void*)(x.out + tok.row * x.out_stride + head * D) : (const void*)(pv.part_o + part * D));
            const int kind = !counts ? 0 : whole ? 1 : 2;
#pragma unroll 4
            for (int i = 0; i < 32; i += R) {
                const int from = i + lane / W, c = lane % W;
                const int what = __shfl_sync(~0u, kind, from);
                char* dst = reinterpret_cast<char*>(__shfl_sync(~0u, (unsigned long long)to, from));
                const float4 y = *reinterpret_cast<const float4*>(reinterpret_cast<float*>(smem) + (size_t)(tile * kTileM + (warp & 3) * 32 + from) * ROW + 4 * c);
                if (what == 1) reinterpret_cast<uint2*>(dst)[c] = make_uint2(pack2(T(), y.x, y.y), pack2(T(), y.z, y.w));
                else if (what == 2) reinterpret_cast<float4*>(dst)[c] = y;
            }
            if (counts) {
                if (!whole) pv.part_ml[part] = gone ? make_float2(0.0f, NAN) : make_float2(m, l);
                else if (x.lse) x.lse[(size_t)tok.row * (pv.n_kv * group) + head] = gone ? NAN : (m - kWeightExp + log2f(l)) * kLn2;
            }
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
