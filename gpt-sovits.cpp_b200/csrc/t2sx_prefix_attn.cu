// Attention of one step's tokens over a pool of shared cache pages.
//
// A plan arranges the sequences' page lists as a trie: a node is a run of pages that a set of sequences has
// in common, and the tokens of that set are its rows.  Each node's pages are read once for all of
// its rows.  Per node, K/V head and range of pages (a split), rows x keys is a small attention of its own:
//     m = max_j s_j,  l = sum_j 2^(s_j - m + c),  O = sum_j 2^(s_j - m + c) v_j,   s_j = scale log2(e) q . k_j
// and a token's result follows from its parts: M = max m_i, out = sum 2^(m_i - M) O_i / sum 2^(m_i - M) l_i.
// The constant c keeps small weights above the subnormal numbers of f16 (and is harmless for bf16).
// Scores, m, l, O and the joins are f32.  The weights alone are rounded to the cache's 16-bit type, in which the tensor cores take
// them to the product with v, so an output carries two such roundings, theirs and its own: 2.3e-4 to 2.9e-4 of its
// length from the 64-bit result in f16 and 1.9e-3 to 2.3e-3 in bf16, where its own rounding alone makes 2.1e-4 and
// 1.7e-3.  Weights as the sum of two 16-bit parts would take the first one away and double the products with v, a
// third more tensor work at head dim 128.
// A row is a (token, query head of the K/V head's group); `group` heads of a token are neighbours.
//
// Times in this file's comments are the device's, of calls one after another with the same tensors (what fits stays in L2), where they
// do not say otherwise; the two sides of a rule were measured alike.
#include "t2sx_prefix_attn.cuh"

#include <algorithm>
#include <cmath>
#include <cstring>
#include <memory>
#include <mutex>
#include <type_traits>

using namespace t2sx;
using namespace t2sx::attn;

namespace {

constexpr int kTileRows = 16;        // rows of a warp's tile (the m of mma.m16n8k16)
constexpr int kWarpsPerPlace = 3;    // warps of a launch for each one that the device holds at a time, where items are many
constexpr int kLongItem = 256;       // keys: shorter items of several K/V heads share a warp; 2048 sequences with 20 positions each of
                                     // their own take 87 us so and 93 without, with 100 each 116 and 123
constexpr int kShortItem = 8;        // keys per head dim: up to which, on average, items that are more than the warps that the device
                                     // holds take the tiles for short ones (see TileShape).  256 sequences over one prompt, 8 heads of
                                     // 128, 500 positions each of their own: 126 us with them, 134 without; 64 sequences of 9000, 8
                                     // heads of 64: 162, 134; 2048 sequences of 500, 16 heads of 32, from cold caches: 374, 365
constexpr int kMinChunk = 2;         // pages of a split at least
constexpr int kSplitCost = 4, kTcSplitCost = 8, kJoinCost = 4;   // in pages: what a split costs beside its pages, and joining parts
constexpr double kClear = 1.5;       // a node's costs with one kernel and the other differ clearly (see choose_kernels)
constexpr int kTcMinChunk = 4;       // pages of a split of such a node at least
constexpr int kFoldParts = 4;        // parts of a token up to which the item of its own pages folds them in, one after the other:
                                     // 2048 sequences, 32 to a prompt, take 340 us so and 351 with a launch that joins them; with up
                                     // to eight parts 256 sequences of one long prompt took 117 when they took 107 so
constexpr int64_t kMaxNodeTokens = 1 << 28;   // of all nodes together: 8 GB of tokens, whose places are 32-bit numbers
constexpr int kSmallWork = 2048;     // pages x head dim of a CTA of a small step at most, an eighth of it with two CTAs to an SM

__device__ __forceinline__ void mma16816(__half, float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16816(__nv_bfloat16, float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// 16 bytes, or as many zeros
__device__ __forceinline__ void cp16(uint32_t smem, const void* gmem, bool real = true) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem), "l"(gmem), "r"(real ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// One 16-byte word per thread: the rows' keys and values go to their positions (for the tcgen05 kernel on pages of one
// sequence, which reads them from the cache by tensor copies).
__global__ void __launch_bounds__(256)
k_write_rows(const Token* __restrict__ rows_of, int rows, const uint4* __restrict__ kn, const uint4* __restrict__ vn,
             long long stride_vec, uint4* __restrict__ k, uint4* __restrict__ v, int n_kv, int row_vec) {
    dependents_launch();
    const int per_row = n_kv * row_vec;
    const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= (long long)rows * per_row) return;
    const int row = (int)(i / per_row), j = (int)(i - (long long)row * per_row), h = j / row_vec, c = j - h * row_vec;
    const Token t = rows_of[row];
    const size_t dst = (((size_t)t.page * n_kv + h) * kPoolPage + (t.limit - 1) % kPoolPage) * row_vec + c;
    k[dst] = kn[row * stride_vec + j];
    v[dst] = vn[row * stride_vec + j];
}

// Tiles of a head dimension: keys per stage of a warp's ring, its stages, the warps of an SM that this leaves
// room for, and the warps of a CTA that shares out one item.  Measured as (keys, stages, warps), in us:
//   dim 32   2048 sequences, 32 to a prompt, 500 positions each of their own: (32, 3, 16) 342, (32, 4, 13) 352, (64, 3, 9) 363,
//            (64, 2, 13) 386, (16, 4, 20) 340;  100 positions: (32, 3, 16) 115, (16, 4, 20) 116, (16, 6, 16) 123;
//            20 positions: 87, 80, 92
//   dim 64   64 sequences of 8000, 8 heads:  (32, 3, 9) 134, (16, 3, 13) 140, (16, 4, 13) 140, (16, 5, 10) 136
//            512 sequences, 32 to a prompt, 20 positions each of their own: 40, 36, 38, 40;  100: 51, 48, 48, 50
//   dim 128  64 sequences of 4000, 8 heads:  (32, 3, 4) 138, (16, 3, 8) 148, (16, 4, 7) 151, (16, 5, 5) 137
//            1024 sequences, 128 to a prompt, 50 positions each of their own: 138, 109, 116, 123
// Long items want their copies far ahead, short ones many warps: an item's start is a chain of waits (item, token, page, keys).
template <int D>
constexpr int kTeam = D == 128 ? 4 : 8;
template <int D, bool SHORT>
struct TileShape {
    static constexpr int KEYS = SHORT ? 16 : 32, STAGES = SHORT && D == 32 ? 4 : 3;
    static constexpr int RESIDENT = SHORT ? (D == 32 ? 20 : D == 64 ? 13 : 8) : D == 32 ? 16 : D == 64 ? 9 : 4;
    static constexpr int HALF = KEYS * D * 2;   // bytes of a stage's K (or V)
    static constexpr int RING = STAGES * 2 * HALF;
    static_assert(RING >= kTileRows * D * 4, "a warp's results take the place of its ring");
};

// 16-byte chunk `c` of key `row` in a tile: chunks are exchanged within 128 bytes so that the eight rows
// of an ldmatrix matrix lie in different banks.
template <int D>
__device__ __forceinline__ uint32_t tile_at(int row, int c) {
    if constexpr (D == 32) return row * 64 + ((c ^ (row >> 1)) & 3) * 16;
    else return row * (D * 2) + ((c & ~7) | ((c ^ row) & 7)) * 16;
}

// At most 16 rows per item.  W = 1: a warp takes `heads_per` K/V heads of an item one after the other, its ring
// running on from one to the next, so that a short item's start is paid once.  W > 1: a
// CTA per (item, K/V head), whose warps share out the item's tiles, each with a ring of its own, and join their
// results in shared memory.
//
// Bound by the cache's bytes where a page has few rows: 2048 sequences, 32 to a prompt, 16 heads of 32 dims, some
// 500 positions each of their own, take 340 us for 2.2 GB (6.4 TB/s); one sequence of 65536 positions, 8 heads of 128, 43 us
// and 10 for the join, which run into one another (53 a call).
// Warps alone (no CTA-wide barrier in the loop) because items differ in length; mma.sync because a page of a few
// rows is a memory-bound product, whatever the tensor cores' rate.  A small step runs the W > 1 form as its only
// launch: 6.9 us for four candidates of one prompt.
template <typename T, int D, int W, bool SHORT>
__global__ void __launch_bounds__(32 * W, W == 1 ? TileShape<D, SHORT>::RESIDENT : 1)
k_attend_tiles(PlanView pv, Tensors<T> x, int item0, int heads_per, int folds) {
    using S = TileShape<D, SHORT>;
    constexpr int NT = S::KEYS / 8, DT = D / 8, KS = D / 16;   // key tiles, dim tiles, steps along the dims
    extern __shared__ __align__(1024) unsigned char ring[];
    const int lane = threadIdx.x & 31, warp = W == 1 ? 0 : threadIdx.x >> 5;
    const int ways = (pv.n_kv + heads_per - 1) / heads_per;
    const int kv0 = (int)(blockIdx.x % ways) * heads_per, kv1 = min(pv.n_kv, kv0 + heads_per);   // neighbours read one page
    const uint32_t ring0 = (uint32_t)__cvta_generic_to_shared(ring) + warp * S::RING;
    const Item it = pv.items[item0 + blockIdx.x / ways];
    const int group = pv.group;
    dependents_launch();   // the next launch fills what this one leaves free

    // rows lane / 4 and lane / 4 + 8
    int row_of[2], g_of[2], limit[2], n_parts[2], part[2];
    long long q_at[2];
    bool live[2], ends[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int r = lane / 4 + 8 * i, mr = it.row0 + r, g = mr % group;
        live[i] = r < it.rows;
        const Token t = pv.tokens[it.tokens_at + (live[i] ? mr / group : 0)];
        row_of[i] = t.row;
        g_of[i] = g;
        q_at[i] = t.row * x.q_stride + g * D;
        limit[i] = live[i] ? t.limit : 0;
        n_parts[i] = t.n_parts;
        ends[i] = t.ends_here;
        part[i] = t.part0 + it.split;
    }
    const int all = (it.keys + S::KEYS - 1) / S::KEYS, first = all * warp / W, tiles = all * (warp + 1) / W;
    int page_base = 0;                                // pages [page_base, page_base + 32) are in the lanes
    int page_id = lane < it.n_pages ? pv.pages[it.pages_at + lane] : 0;
    // tiles of one K/V head after those of another
    int next_t = first, next_kv = first < tiles ? kv0 : kv1, stage_in = 0;
    auto request = [&]() {
        if (next_kv < kv1) {
            const int t = next_t, kvh = next_kv;
            const int pg = t / (kPoolPage / S::KEYS), sub = t % (kPoolPage / S::KEYS);
            if (pg < page_base || pg >= page_base + 32) {
                page_base = pg;
                page_id = page_base + lane < it.n_pages ? pv.pages[it.pages_at + page_base + lane] : 0;
            }
            const int page = __shfl_sync(~0u, page_id, pg - page_base);
            const size_t at = (((size_t)page * pv.n_kv + kvh) * kPoolPage + sub * S::KEYS) * D;
            const uint32_t dst = ring0 + stage_in * 2 * S::HALF;
            const char *ks = reinterpret_cast<const char*>(x.k + at), *vs = reinterpret_cast<const char*>(x.v + at);
            const int pos = it.pos0 + t * S::KEYS;
            const bool plain = pos + S::KEYS <= min(it.end, x.k_new ? it.new_pos : INT32_MAX);
#pragma unroll
            for (int i = 0; i < S::HALF / 512; ++i) {
                const int c = i * 32 + lane;
                const uint32_t d = dst + tile_at<D>(c / (D / 8), c % (D / 8));
                if (plain) {
                    cp16(d, ks + c * 16);
                    cp16(d + S::HALF, vs + c * 16);
                } else {
                    // the step's own keys come from the call's tensors; what stands beyond the filled positions may
                    // be anything, and counts as zeros
                    const int at_pos = pos + c / (D / 8);
                    const bool real = at_pos < it.end, own = x.k_new && real && at_pos >= it.new_pos;
                    const long long off = (it.new_row + at_pos - it.new_pos) * x.kv_stride + kvh * D + (c % (D / 8)) * 8;
                    cp16(d, own ? reinterpret_cast<const char*>(x.k_new + off) : ks + c * 16, real);
                    cp16(d + S::HALF, own ? reinterpret_cast<const char*>(x.v_new + off) : vs + c * 16, real);
                }
            }
            if (++next_t == tiles) { next_t = first; ++next_kv; }
            stage_in = stage_in + 1 == S::STAGES ? 0 : stage_in + 1;
        }
        cp_commit();
    };
    for (int i = 0; i < S::STAGES - 1; ++i) request();
    // The item with a token's own position writes its key and value to the cache: read here, written after
    // the tiles for the first token (a decode step's only one).
    auto own = [&](int r) -> const Token* {
        const Token* t = pv.tokens + it.tokens_at + (it.row0 + r) / group;
        return x.k_new && r < it.rows && (it.row0 + r) % group == 0 && t->limit > it.pos0 &&
               t->limit <= it.pos0 + it.n_pages * kPoolPage && lane < D / 4 && warp == 0 ? t : nullptr;
    };
    auto own_src = [&](const Token* t, int kvh) {
        return reinterpret_cast<const uint4*>((lane >= D / 8 ? x.v_new : x.k_new) + t->row * x.kv_stride + kvh * D) + lane % (D / 8);
    };
    auto own_dst = [&](const Token* t, int kvh) {
        return reinterpret_cast<uint4*>((lane >= D / 8 ? x.v : x.k) +
                                        (((size_t)t->page * pv.n_kv + kvh) * kPoolPage + (t->limit - 1) % kPoolPage) * D) + lane % (D / 8);
    };
    const Token* own0 = own(0);
    // the smallest limit of the rows: keys below it need no mask
    int free_to = min(live[0] ? limit[0] : INT32_MAX, live[1] ? limit[1] : INT32_MAX);
    for (int y = 16; y; y >>= 1) free_to = min(free_to, __shfl_xor_sync(~0u, free_to, y));

    const bool upper = it.rows > 8;
    int stage = 0;
    for (int kvh = kv0; kvh < kv1; ++kvh) {
        int head_of[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) head_of[i] = kvh * group + g_of[i];
        auto part_index = [&](int i, int part) { return ((size_t)part * group + g_of[i]) * pv.n_kv + kvh; };
        uint4 own_word = make_uint4(0, 0, 0, 0);
        if (own0) own_word = *own_src(own0, kvh);
        uint32_t qf[KS][4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t* src = reinterpret_cast<const uint32_t*>(x.q + q_at[i] + (long long)kvh * group * D);
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                qf[k][i] = live[i] ? src[k * 8 + lane % 4] : 0;
                qf[k][i + 2] = live[i] ? src[k * 8 + 4 + lane % 4] : 0;
            }
        }
        float o[DT][4] = {}, m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
        // The parts of the launch before: the first head's are folded in at its end (they may not be there yet), those
        // of the others are what the head starts from.
        const bool start_from = W == 1 && kvh > kv0;
        int folded[2] = {0, 0};
        if (start_from) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (!live[i] || !ends[i] || n_parts[i] < 2 || limit[i] <= it.pos0) continue;
                const size_t at = part_index(i, part[i] - 1);
                const float2 ml = __ldcg(&pv.part_ml[at]);
                m[i] = ml.x;
                l[i] = lane % 4 == 0 ? ml.y : 0.0f;
                const float2* src = reinterpret_cast<const float2*>(pv.part_o + at * D);
#pragma unroll
                for (int d = 0; d < DT; ++d) {
                    const float2 y = __ldcg(&src[d * 4 + lane % 4]);
                    o[d][2 * i] = y.x;
                    o[d][2 * i + 1] = y.y;
                }
                folded[i] = 1;
            }
        }
        for (int t = first; t < tiles; ++t) {
            cp_wait<S::STAGES - 2>();
            __syncwarp();
            const uint32_t kt = ring0 + stage * 2 * S::HALF, vt = kt + S::HALF;
            stage = stage + 1 == S::STAGES ? 0 : stage + 1;
            const int pos = it.pos0 + t * S::KEYS;
            float s[NT][4] = {};
#pragma unroll
            for (int n = 0; n < NT; n += 2)
#pragma unroll
                for (int k = 0; k < KS; ++k) {
                    uint32_t b[4];
                    ldsm4(b, kt + tile_at<D>(n * 8 + (lane & 7) + ((lane >> 4) << 3), 2 * k + ((lane >> 3) & 1)));
                    mma16816(T(), s[n], qf[k], b[0], b[1]);
                    mma16816(T(), s[n + 1], qf[k], b[2], b[3]);
                }
            const bool masked = pos + S::KEYS > free_to;
            uint32_t p[NT][2];
            bool grew = false;
            float alpha[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (i == 1 && !upper) {
                    alpha[1] = 1.0f;
#pragma unroll
                    for (int n = 0; n < NT; ++n) p[n][1] = 0;
                    break;
                }
                float mx = -INFINITY;
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float y = s[n][2 * i + e] * x.scale2;
                        if (masked && pos + n * 8 + 2 * (lane % 4) + e >= limit[i]) y = -INFINITY;
                        s[n][2 * i + e] = y;
                        mx = fmaxf(mx, y);
                    }
                mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, 2));
                mx = fmaxf(mx, m[i]);
                const float base = mx == -INFINITY ? 0.0f : mx - kWeightExp;
                alpha[i] = m[i] == -INFINITY ? 0.0f : ex2(m[i] - mx);
                grew |= mx > m[i];
                m[i] = mx;
                float sum = 0.0f;
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const float a = ex2(s[n][2 * i] - base), b = ex2(s[n][2 * i + 1] - base);
                    sum += a + b;
                    p[n][i] = pack2(T(), a, b);
                }
                l[i] = fmaf(l[i], alpha[i], sum);
            }
            if (__any_sync(~0u, grew)) {
#pragma unroll
                for (int d = 0; d < DT; ++d) {
                    o[d][0] *= alpha[0]; o[d][1] *= alpha[0];
                    o[d][2] *= alpha[1]; o[d][3] *= alpha[1];
                }
            }
#pragma unroll
            for (int n = 0; n < NT; n += 2) {
                const uint32_t a[4] = {p[n][0], p[n][1], p[n + 1][0], p[n + 1][1]};
#pragma unroll
                for (int d = 0; d < DT; d += 2) {
                    uint32_t b[4];
                    ldsm4_t(b, vt + tile_at<D>(n * 8 + (lane & 15), d + (lane >> 4)));
                    mma16816(T(), o[d], a, b[0], b[1]);
                    mma16816(T(), o[d + 1], a, b[2], b[3]);
                }
            }
            __syncwarp();
            request();
        }
        if (own0) *own_dst(own0, kvh) = own_word;
        for (int r = 1; r < it.rows; ++r)
            if (const Token* t = own(r)) *own_dst(t, kvh) = *own_src(t, kvh);
        float sum[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            sum[i] = l[i];
            sum[i] += __shfl_xor_sync(~0u, sum[i], 1);
            sum[i] += __shfl_xor_sync(~0u, sum[i], 2);
        }
        if constexpr (W > 1) {
            // the warps' results in the place of their rings; then each warp joins the dim tiles warp, warp + W, ...
            __shared__ float2 ml[W][16];
            cp_wait<0>();
            __syncthreads();
            float2* all_o = reinterpret_cast<float2*>(ring);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (lane % 4 == 0) ml[warp][lane / 4 + 8 * i] = make_float2(m[i], sum[i]);
#pragma unroll
                for (int d = 0; d < DT; ++d) all_o[((warp * 2 + i) * DT + d) * 32 + lane] = make_float2(o[d][2 * i], o[d][2 * i + 1]);
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float M = -INFINITY;
                for (int j = 0; j < W; ++j) M = fmaxf(M, ml[j][lane / 4 + 8 * i].x);
                m[i] = M;
                sum[i] = 0.0f;
#pragma unroll
                for (int d = 0; d < DT; ++d) o[d][2 * i] = o[d][2 * i + 1] = 0.0f;
                for (int j = 0; j < W; ++j) {
                    const float2 part = ml[j][lane / 4 + 8 * i];
                    const float f = part.x == -INFINITY ? 0.0f : ex2(part.x - M);
                    sum[i] = fmaf(part.y, f, sum[i]);
#pragma unroll
                    for (int d = 0; d < DT; ++d) {
                        if (d % W != warp) continue;
                        const float2 y = all_o[((j * 2 + i) * DT + d) * 32 + lane];
                        o[d][2 * i] = fmaf(y.x, f, o[d][2 * i]);
                        o[d][2 * i + 1] = fmaf(y.y, f, o[d][2 * i + 1]);
                    }
                }
            }
        }
        auto mine = [&](int d) { return W == 1 || d % W == warp; };
        // The parts of the launch before.  Where none are folded in, one CTA waits, so that this launch does not end before that
        // one, and the others go on beside it.
        if (folds || blockIdx.x == gridDim.x - 1) dependents_wait();
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (!live[i] || limit[i] <= it.pos0) continue;   // such a row has no part here
            if (n_parts[i] > 1 && !ends[i]) {
                const size_t at = part_index(i, part[i]);
                float2* dst = reinterpret_cast<float2*>(pv.part_o + at * D);
#pragma unroll
                for (int d = 0; d < DT; ++d)
                    if (mine(d)) dst[d * 4 + lane % 4] = make_float2(o[d][2 * i], o[d][2 * i + 1]);
                if (lane % 4 == 0 && warp == 0) pv.part_ml[at] = make_float2(m[i], sum[i]);
                continue;
            }
            if constexpr (W == 1) {
                for (int j = n_parts[i] - 1 - folded[i]; j-- > 0;) {   // the other parts, if any
                    const size_t at = part_index(i, part[i] - n_parts[i] + 1 + j);
                    const float2 ml = __ldcg(&pv.part_ml[at]);
                    const float2* src = reinterpret_cast<const float2*>(pv.part_o + at * D);
                    float2 y[DT];
#pragma unroll
                    for (int d = 0; d < DT; ++d) y[d] = __ldcg(&src[d * 4 + lane % 4]);
                    const float M = fmaxf(m[i], ml.x), f = m[i] == -INFINITY ? 0.0f : ex2(m[i] - M), g = ml.x == -INFINITY ? 0.0f : ex2(ml.x - M);
                    m[i] = M;
                    sum[i] = fmaf(sum[i], f, ml.y * g);
#pragma unroll
                    for (int d = 0; d < DT; ++d) {
                        o[d][2 * i] = fmaf(o[d][2 * i], f, y[d].x * g);
                        o[d][2 * i + 1] = fmaf(o[d][2 * i + 1], f, y[d].y * g);
                    }
                }
            }
            const float inv = sum[i] == 0.0f ? 0.0f : 1.0f / sum[i];
            uint32_t* dst = reinterpret_cast<uint32_t*>(x.out + row_of[i] * x.out_stride + head_of[i] * D);
#pragma unroll
            for (int d = 0; d < DT; ++d)
                if (mine(d)) dst[d * 4 + lane % 4] = pack2(T(), o[d][2 * i] * inv, o[d][2 * i + 1] * inv);
            if (x.lse && lane % 4 == 0 && warp == 0)
                x.lse[(size_t)row_of[i] * (pv.n_kv * group) + head_of[i]] = (m[i] - kWeightExp + log2f(sum[i])) * kLn2;
        }
    }
}

// Joining the parts: out = sum 2^(m_i - M) O_i / sum 2^(m_i - M) l_i.  Bound by the parts' bytes, which the launch before
// has just left in the L2 cache, and by latency.
//
// Four warps, each with a (token, query head) of few parts (at most 32; 256 sequences of one long prompt took 107 us so and
// 113 with a CTA for each of their rows): the lanes are D / 4 columns of four dims x 32 / (D / 4) parts.
template <typename T, int D>
__global__ void __launch_bounds__(128)
k_join_few(PlanView pv, Tensors<T> x) {
    constexpr int COLS = D / 4, LANES = 32 / COLS;
    const int lane = threadIdx.x & 31, heads = pv.n_kv * pv.group;
    const long long at = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    dependents_wait();
    if (at >= (long long)pv.n_joins * heads) return;
    const int head = (int)(at % heads), kvh = head / pv.group, g = head % pv.group;
    const Token t = pv.joins[at / heads];
    auto part = [&](int i) { return ((size_t)(t.part_at + i) * pv.group + g) * pv.n_kv + kvh; };
    const float2 mine = lane < t.n_parts ? __ldcg(&pv.part_ml[part(lane)]) : make_float2(-INFINITY, 0.0f);
    float M = mine.x;
    for (int y = 16; y; y >>= 1) M = fmaxf(M, __shfl_xor_sync(~0u, M, y));
    const float weight = mine.x == -INFINITY ? 0.0f : ex2(mine.x - M);
    float l = weight * mine.y;
    for (int y = 16; y; y >>= 1) l += __shfl_xor_sync(~0u, l, y);
    float4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (int i0 = 0; i0 < t.n_parts; i0 += LANES) {
        const int i = i0 + lane / COLS;
        const float f = __shfl_sync(~0u, weight, i & 31);
        if (i >= t.n_parts) continue;
        const float4 o = __ldcg(reinterpret_cast<const float4*>(pv.part_o + part(i) * D) + lane % COLS);
        acc.x = fmaf(f, o.x, acc.x);
        acc.y = fmaf(f, o.y, acc.y);
        acc.z = fmaf(f, o.z, acc.z);
        acc.w = fmaf(f, o.w, acc.w);
    }
#pragma unroll
    for (int y = COLS; y < 32; y <<= 1) {
        acc.x += __shfl_xor_sync(~0u, acc.x, y);
        acc.y += __shfl_xor_sync(~0u, acc.y, y);
        acc.z += __shfl_xor_sync(~0u, acc.z, y);
        acc.w += __shfl_xor_sync(~0u, acc.w, y);
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    if (lane < COLS)
        reinterpret_cast<uint2*>(x.out + t.row * x.out_stride + head * D)[lane] =
            make_uint2(pack2(T(), acc.x * inv, acc.y * inv), pack2(T(), acc.z * inv, acc.w * inv));
    if (x.lse && lane == 0) x.lse[(size_t)t.row * heads + head] = (M - kWeightExp + log2f(l)) * kLn2;
}

// One CTA of four warps per (token of several parts, query head), for tokens of many parts: each warp joins every
// fourth part, then the first one the four results.
template <typename T, int D>
__global__ void __launch_bounds__(128)
k_join_parts(PlanView pv, Tensors<T> x) {
    constexpr int COLS = D / 4, LANES = 128 / COLS;
    __shared__ float4 so[128];
    __shared__ float sl[LANES], sm[4];
    dependents_wait();
    const int tid = threadIdx.x, lane = tid & 31, heads = pv.n_kv * pv.group;
    const int head = (int)(blockIdx.x % heads), kvh = head / pv.group, g = head % pv.group;
    const Token t = pv.joins[blockIdx.x / heads];
    const int row = t.row;
    auto part = [&](int i) { return ((size_t)(t.part_at + i) * pv.group + g) * pv.n_kv + kvh; };
    float M = -INFINITY;
    for (int i = tid; i < t.n_parts; i += 128)
        M = fmaxf(M, __ldcg(&pv.part_ml[part(i)]).x);
    for (int y = 16; y; y >>= 1) M = fmaxf(M, __shfl_xor_sync(~0u, M, y));
    if (lane == 0) sm[tid >> 5] = M;
    __syncthreads();
    M = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
    float4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    float l = 0.0f;
#pragma unroll 4
    for (int i = tid / COLS; i < t.n_parts; i += LANES) {
        const size_t at = part(i);
        const float2 ml = __ldcg(&pv.part_ml[at]);
        const float4 o = __ldcg(reinterpret_cast<const float4*>(pv.part_o + at * D) + tid % COLS);
        const float f = ml.x == -INFINITY ? 0.0f : ex2(ml.x - M);
        l = fmaf(f, ml.y, l);
        acc.x = fmaf(f, o.x, acc.x);
        acc.y = fmaf(f, o.y, acc.y);
        acc.z = fmaf(f, o.z, acc.z);
        acc.w = fmaf(f, o.w, acc.w);
    }
    so[tid] = acc;
    if (tid % COLS == 0) sl[tid / COLS] = l;
    __syncthreads();
    if (tid >= COLS) return;
    acc = so[tid];
    l = sl[0];
    for (int j = 1; j < LANES; ++j) {
        const float4 o = so[j * COLS + tid];
        acc.x += o.x; acc.y += o.y; acc.z += o.z; acc.w += o.w;
        l += sl[j];
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    reinterpret_cast<uint2*>(x.out + row * x.out_stride + head * D)[tid] =
        make_uint2(pack2(T(), acc.x * inv, acc.y * inv), pack2(T(), acc.z * inv, acc.w * inv));
    if (x.lse && tid == 0) x.lse[(size_t)row * heads + head] = (M - kWeightExp + log2f(l)) * kLn2;
}

int bad(const char* m) { return t2sx_set_error(T2SX_ERR_INVALID, m); }

// A run of pages that a set of sequences shares (or that one has for itself).
struct Node {
    int32_t tokens_at, n_tokens;
    int32_t pages_at, n_pages;
    int32_t pos0, end;
    int32_t new_pos, new_row;
    bool tc;             // for the tcgen05 kernel
};

int resident_warps(int dim) {
    return dim == 32 ? TileShape<32, false>::RESIDENT : dim == 64 ? TileShape<64, false>::RESIDENT : TileShape<128, false>::RESIDENT;
}

int sm_count(int device) {
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) != cudaSuccess || n <= 0) return 148;
    return n;
}

}  // namespace

struct t2sx_plan {
    t2sx_pool* pool = nullptr;
    int n_heads = 0, n_sm = 148;
    bool ready = false, shared_rows = false, small = false, tc_writes = false, folds = false;
    int32_t most_parts = 0;            // of a token in `joins`
    int64_t launch_keys[2] = {0, 0};   // of the items of the launches of k_attend_tiles
    CUtensorMap map_k, map_v;
    int32_t *err = nullptr, *err_dev = nullptr;   // pinned: what a kernel that gave up a wait reports
    uint64_t version = 0;          // of the pool at the update
    uint64_t shares = 0;           // of the pool when shared_rows was found
    std::vector<int32_t> row_pages;   // that the rows' own positions are in
    // host copy of what the device gets, in pinned memory: two buffers, so that an update need not
    // wait for the previous one's upload
    uint8_t* host[2] = {};
    size_t host_bytes[2] = {};
    cudaEvent_t sent[2] = {};
    int turn = 0;
    uint8_t *dev = nullptr, *work = nullptr;
    size_t dev_bytes = 0, work_bytes = 0;
    PlanView view = {};
    // scratch of an update
    std::vector<int32_t> order, next_order, group_of, count, group_page, node_rows, pages;
    std::vector<int32_t> stamp, stamp_group, row0;
    int32_t round = 0;             // splits of all updates
    std::vector<Token> info, tokens, joins;   // the step's rows; nodes' tokens; those of several parts
    std::vector<Node> nodes;
    std::vector<Item> items;
};

static void plan_release(t2sx_plan* a) {
    t2sx_pool* p = a->pool;
    DeviceGuard dg;
    dg.set(p->device);
    p->settle();
    for (int i = 0; i < 2; ++i) {
        if (a->sent[i]) cudaEventDestroy(a->sent[i]);
        if (a->host[i]) cudaFreeHost(a->host[i]);
    }
    if (a->dev) cudaFree(a->dev);
    if (a->work) cudaFree(a->work);
    if (a->err) cudaFreeHost(a->err);
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
        a->n_sm = sm_count(p->device);
        if (!tc_maps(p, &a->map_k, &a->map_v)) return t2sx_set_error(T2SX_ERR_CUDA, "t2sx_plan_create: the driver gives no tensor maps");
        POOL_CK(cudaHostAlloc(&a->err, 4, cudaHostAllocMapped));
        *a->err = 0;
        POOL_CK(cudaHostGetDevicePointer(&a->err_dev, a->err, 0));
        for (int i = 0; i < 2; ++i) POOL_CK(cudaEventCreateWithFlags(&a->sent[i], cudaEventDisableTiming));
        *out = a.release();
        return T2SX_OK;
    });
}

extern "C" void t2sx_plan_free(t2sx_plan* a) {
    if (a) plan_release(a);
}

// The trie of the sequences' page lists: every entry of a list is looked at once or twice.  Sequences are
// split by the page that follows their common run, keeping their order.  False: the nodes have too many tokens.
static bool build_nodes(t2sx_plan* a, int32_t n, const int32_t* seqs, const int32_t* n_new) {
    t2sx_pool* p = a->pool;
    a->nodes.clear(); a->node_rows.clear(); a->pages.clear();
    a->order.clear();
    for (int32_t i = 0; i < n; ++i)
        if (n_new[i] > 0) a->order.push_back(i);
    struct Set { int32_t lo, hi, depth; };   // a range of `order`, and the pages above it
    auto emit = [&](const Set& s, int32_t to) {
        Node nd;
        nd.tokens_at = (int32_t)a->node_rows.size();
        int64_t tokens = nd.tokens_at;
        for (int32_t j = s.lo; j < s.hi; ++j) tokens += n_new[a->order[j]];
        if (tokens > kMaxNodeTokens) return false;
        for (int32_t j = s.lo; j < s.hi; ++j) {
            const int32_t i = a->order[j];
            for (int32_t k = 0; k < n_new[i]; ++k) a->node_rows.push_back(a->row0[i] + k);
        }
        nd.n_tokens = (int32_t)a->node_rows.size() - nd.tokens_at;
        const std::vector<int32_t>& t = p->table[seqs[a->order[s.lo]]];
        nd.pages_at = (int32_t)a->pages.size();
        a->pages.insert(a->pages.end(), t.begin() + s.depth, t.begin() + to);
        nd.n_pages = to - s.depth;
        nd.pos0 = s.depth * kPoolPage;
        // pages of several sequences are full; a sequence's own ones end with it
        nd.end = s.hi - s.lo > 1 ? to * kPoolPage : (int32_t)std::min<int64_t>((int64_t)to * kPoolPage, p->len[seqs[a->order[s.lo]]]);
        // rows of several sequences have no position in the node's pages (or the step writes nothing)
        const int32_t i0 = a->order[s.lo];
        nd.new_pos = s.hi - s.lo > 1 ? INT32_MAX : (int32_t)(p->len[seqs[i0]] - n_new[i0]);
        nd.new_row = a->row0[i0];
        a->nodes.push_back(nd);
        return true;
    };
    if (a->small) {   // nothing is shared: one node for each sequence
        for (int32_t j = 0; j < (int32_t)a->order.size(); ++j)
            if (!emit({j, j + 1, 0}, (int32_t)p->table[seqs[a->order[j]]].size())) return false;
        return true;
    }
    // A page's stamp says in which split it was seen last.  Splits (no more of them than sequences) are numbered on from
    // update to update, so that an update costs what its sequences have, not what the pool has.
    if (a->stamp.empty() || a->round > INT32_MAX / 2) {
        a->stamp_group.resize(p->n_pages);
        a->stamp.assign(p->n_pages, -1);
        a->round = 0;
    }
    std::vector<Set> todo;
    if (!a->order.empty()) todo.push_back({0, (int32_t)a->order.size(), 0});
    while (!todo.empty()) {
        const Set s = todo.back();
        todo.pop_back();
        const std::vector<int32_t>& t = p->table[seqs[a->order[s.lo]]];
        if (s.hi - s.lo == 1) {
            if ((size_t)s.depth < t.size() && !emit(s, (int32_t)t.size())) return false;
            continue;
        }
        int32_t common = (int32_t)t.size();
        for (int32_t j = s.lo + 1; j < s.hi; ++j) {
            const std::vector<int32_t>& o = p->table[seqs[a->order[j]]];
            const int32_t most = std::min<int32_t>(common, (int32_t)o.size());
            int32_t k = s.depth;
            while (k < most && o[k] == t[k]) ++k;
            common = k;
        }
        if (common > s.depth && !emit(s, common)) return false;
        // split by the next page
        const int32_t here = a->round++;
        a->count.clear();
        a->group_of.assign(s.hi - s.lo, -1);
        for (int32_t j = s.lo; j < s.hi; ++j) {
            const std::vector<int32_t>& o = p->table[seqs[a->order[j]]];
            if (o.size() <= (size_t)common) continue;   // ends here
            const int32_t page = o[common];
            if (a->stamp[page] != here) {
                a->stamp[page] = here;
                a->stamp_group[page] = (int32_t)a->count.size();
                a->count.push_back(0);
            }
            a->group_of[j - s.lo] = a->stamp_group[page];
            ++a->count[a->stamp_group[page]];
        }
        a->next_order.resize(s.hi - s.lo);
        int32_t at = 0;
        for (int32_t& c : a->count) { const int32_t size = c; c = at; at += size; }
        a->group_page.assign(a->count.begin(), a->count.end());   // where each one starts
        for (int32_t j = s.lo; j < s.hi; ++j)
            if (a->group_of[j - s.lo] >= 0) a->next_order[a->count[a->group_of[j - s.lo]]++] = a->order[j];
        std::copy(a->next_order.begin(), a->next_order.begin() + at, a->order.begin() + s.lo);
        for (size_t g = a->count.size(); g-- > 0;)
            todo.push_back({s.lo + a->group_page[g], s.lo + a->count[g], common});
    }
    return true;
}

// The kernels of the nodes, by cost.  In pages of the tcgen05 kernel's two tiles, an SM's time: such a CTA costs its start and end and
// its pages (half as much each where its two tiles share them out); a warp tile of 16 rows costs a share of that for each of its pages
// and for kSplitCost more.  In us, with the tcgen05 kernel and without:
//   heads of 128: 16 prompts of 4032 with 16 rows 63, 56; with 24 61, 77;   32 prompts of 500 with 32 rows 45, 46;
//   heads of 64:  16 of 4032 with 24 rows 38, 44;   32 of 1000 with 32 rows and 250 positions each of their own 56, 49;
//                 32 of 500 with 64 rows 37, 40;    32 of 3000 with 64 rows 64, 105
//   heads of 32:  16 of 4032 with 48 rows 23, 25, with 64 23, 30;   40 of 350 with 48 rows, 16 K/V heads, 105, 88
// Nodes that are near the balance (up to kClear of it) go all one way, by their sum: launches of both kinds cost more than
// the better choice gains (8 prompts of 1500 with 24 rows, heads of 64: 17 with, 19 without, 26 with some of each).
static void choose_kernels(t2sx_plan* a) {
    const int group = a->n_heads / a->pool->n_kv, dim = a->pool->dim;
    const double share = dim == 128 ? 0.7 : dim == 64 ? 0.4 : 0.28;
    auto costs = [&](const Node& nd) {   // warp tiles, tcgen05
        const int64_t rows = (int64_t)nd.n_tokens * group, items = (rows + kTcRows - 1) / kTcRows, tiles = (rows + kTileRows - 1) / kTileRows;
        return std::make_pair(tiles * share * (nd.n_pages + kSplitCost), items * kTcSplitCost + nd.n_pages * (rows <= kTcRows / 2 ? 0.5 : items));
    };
    double warp = 0, tc = 0;
    for (Node& nd : a->nodes) {
        nd.tc = !a->small && (int64_t)nd.n_tokens * group > kTileRows;
        if (!nd.tc) continue;
        const auto c = costs(nd);
        warp += c.first;
        tc += c.second;
    }
    for (Node& nd : a->nodes) {
        if (!nd.tc) continue;
        const auto c = costs(nd);
        nd.tc = c.first > kClear * c.second || (c.first * kClear > c.second && warp > tc);
    }
}

// Pages of a split, for the nodes of one kind: of the even divisions of the longest node, the one that ends first,
// where a split costs its pages and as much again as kSplitCost of them, `slots` of them run at a time, and
// they start the longest first.
static int64_t best_chunk(const t2sx_plan* a, bool tc, int64_t slots) {
    const int group = a->n_heads / a->pool->n_kv, tile = tc ? kTcRows : kTileRows;
    const int64_t least = tc ? kTcMinChunk : kMinChunk;
    int64_t longest = 0, tc_nodes = 0;
    for (const Node& nd : a->nodes) {
        if (nd.tc == tc) longest = std::max<int64_t>(longest, nd.n_pages);
        tc_nodes += nd.tc;
    }
    int64_t best = std::max<int64_t>(longest, 1);
    double best_cost = 1e300;
    for (int64_t parts = 1; parts <= 512 && (parts == 1 || (longest + parts - 1) / parts >= least); parts += parts < 32 ? 1 : parts / 16) {
        int64_t chunk = (longest + parts - 1) / parts;
        if (tc) chunk += chunk & 1;   // it takes two pages at a time
        int64_t items = 0, few = 0;
        double pages = 0;
        for (const Node& nd : a->nodes) {
            if (nd.tc != tc) continue;
            const int64_t rows = nd.n_tokens * (int64_t)group, tiles = (rows + tile - 1) / tile * a->pool->n_kv;
            items += tiles * ((nd.n_pages + chunk - 1) / chunk);
            pages += tiles * nd.n_pages * (tc && rows <= kTcRows / 2 ? 0.5 : 1.0);   // its tiles share the pages out
            few += rows <= kTcRows / 2;
        }
        const double split = tc ? kTcSplitCost : kSplitCost, longest_item = tc && few == tc_nodes ? chunk * 0.5 : chunk;
        const double waves = (double)((items + slots - 1) / slots) * (longest_item + split);
        const double even = (pages + items * split) / slots + (items > slots ? longest_item : 0);
        const double cost = std::min(waves, std::max(even, longest_item + split)) + (parts > 1 ? kJoinCost : 0);
        if (cost < best_cost) { best_cost = cost; best = chunk; }
    }
    return best;
}

// Items and parts from the nodes; returns the number of parts.  A node's pages are split so that there are
// several items for each warp that the device holds, and each part's result is small against the keys that
// it stands for.
static int64_t build_items(t2sx_plan* a) {
    const int group = a->n_heads / a->pool->n_kv, n_kv = a->pool->n_kv;
    a->items.clear(); a->joins.clear();
    choose_kernels(a);
    const int64_t warp_chunk = a->small ? INT32_MAX : best_chunk(a, false, (int64_t)a->n_sm * resident_warps(a->pool->dim));
    const int64_t tc_chunk = best_chunk(a, true, a->n_sm);
    a->tokens.resize(a->node_rows.size());
    for (const Node& nd : a->nodes) {
        const int64_t chunk = nd.tc ? tc_chunk : warp_chunk;
        const int tile = nd.tc ? kTcRows : kTileRows;
        const int32_t n_splits = (int32_t)((nd.n_pages + chunk - 1) / chunk);
        int32_t per = (nd.n_pages + n_splits - 1) / n_splits;
        if (nd.tc) per += per & 1;
        const int32_t* rows_of = a->node_rows.data() + nd.tokens_at;
        // a token has parts for the splits that begin below its limit, the first ones
        for (int32_t j = 0; j < nd.n_tokens; ++j) {
            Token& t = a->info[rows_of[j]];
            a->tokens[nd.tokens_at + j].part0 = t.n_parts;   // among the token's; its own number is added below
            const int32_t seen = pages_of(t.limit) - nd.pos0 / kPoolPage;
            if (seen > 0) t.n_parts += std::min((nd.n_pages + per - 1) / per, (seen + per - 1) / per);
            if (nd.new_pos != INT32_MAX) t.ends_here = seen > 0 && n_splits == 1 && !nd.tc;
        }
        const int64_t rows = (int64_t)nd.n_tokens * group;
        for (int32_t split = 0, pg = 0; pg < nd.n_pages; ++split, pg += per) {
            const int32_t start = nd.pos0 + pg * kPoolPage;
            for (int64_t r = 0; r < rows; r += tile) {
                const int32_t n = (int32_t)std::min<int64_t>(tile, rows - r);
                int32_t sees = 0;
                for (int64_t j = r / group; j <= (r + n - 1) / group; ++j) sees = std::max(sees, a->info[rows_of[j]].limit);
                const int32_t pages = std::min(std::min(per, nd.n_pages - pg), pages_of(sees) - start / kPoolPage);
                if (pages <= 0) continue;
                a->items.push_back({nd.tokens_at, (int32_t)r, n, nd.pages_at + pg, pages, start, split, nd.end, nd.new_pos, nd.new_row,
                                    nd.tc ? 0 : nd.new_pos == INT32_MAX ? 1 : 2,
                                    std::min(pages * kPoolPage, std::min(sees, nd.end) - start)});
            }
        }
    }
    // by launch, the longest items first
    std::stable_sort(a->items.begin(), a->items.end(), [](const Item& x, const Item& y) {
        return x.launch != y.launch ? x.launch < y.launch : x.n_pages > y.n_pages;
    });
    int32_t n_launch[3] = {0, 0, 0};
    a->launch_keys[0] = a->launch_keys[1] = 0;
    a->tc_writes = false;
    for (const Item& it : a->items) {
        ++n_launch[it.launch];
        if (it.launch > 0) a->launch_keys[it.launch - 1] += it.keys;
        a->tc_writes |= it.launch == 0 && it.new_pos != INT32_MAX;
    }
    int64_t parts = 0;
    a->most_parts = 0;
    a->folds = false;
    for (Token& t : a->info) {
        t.part_at = (int32_t)std::min<int64_t>(parts, INT32_MAX);
        if (t.n_parts > 1) parts += t.n_parts;
        t.ends_here &= t.n_parts <= kFoldParts;
        a->folds |= t.ends_here && t.n_parts > 1;
        if (t.n_parts > 1 && !t.ends_here) {
            a->joins.push_back(t);
            a->most_parts = std::max(a->most_parts, t.n_parts);
        }
    }
    for (size_t i = 0; i < a->tokens.size(); ++i) {
        const int32_t ordinal = a->tokens[i].part0;
        a->tokens[i] = a->info[a->node_rows[i]];
        a->tokens[i].part0 = a->tokens[i].part_at + ordinal;
        a->tokens[i].ends_here &= ordinal == a->tokens[i].n_parts - 1;
    }
    a->view.n_tc = n_launch[0];
    a->view.n_shared = n_launch[1];
    a->view.n_own = n_launch[2];
    a->view.n_joins = (int)a->joins.size();
    a->view.group = group;
    a->view.n_kv = n_kv;
    a->view.rows = (int)a->info.size();
    return parts;
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
        bool twice = false;
        for (int32_t i = 0; i < n; ++i) { twice |= p->mark[seqs[i]]; p->mark[seqs[i]] = 1; }
        for (int32_t i = 0; i < n; ++i) p->mark[seqs[i]] = 0;
        if (twice) return bad("t2sx_plan_update: a sequence is given twice");
        a->ready = false;
        a->shared_rows = false;
        a->info.resize(rows);
        a->row0.resize(n);
        a->row_pages.clear();
        int32_t r = 0;
        for (int32_t i = 0; i < n; ++i) {
            a->row0[i] = r;
            for (int32_t j = 0; j < n_new[i]; ++j, ++r) {
                const int32_t limit = (int32_t)(p->len[seqs[i]] - n_new[i] + j + 1);
                const int32_t page = p->table[seqs[i]][(limit - 1) / kPoolPage];
                a->shared_rows |= p->users[page] > 1;
                if (j == 0 || page != a->row_pages.back()) a->row_pages.push_back(page);
                a->info[r] = Token{r, limit, page, 0, 0, 0, 0, 0};
            }
        }
        // A small step: a CTA for each (tile of rows, K/V head), all at one time, with no parts to join; its shared pages
        // come from L2 however often they are read.  By CTAs, pages and head dim, us with it and without:
        //   64, 6, 32: 6.9, 12.6     128, 24, 32: 10.5, 12.5    128, 6, 64: 8.4, 14.6    128, 24, 64: 12.7, 16.6
        //   288, 6, 32: 12.0, 12.7   192, 24, 32: 15.0, 12.6    256, 6, 64: 14.6, 12.6   32, 24, 128: 24.7, 16.7
        int64_t row_tiles = 0, longest = 0;
        for (int32_t i = 0; i < n; ++i) {
            row_tiles += ((int64_t)n_new[i] * (a->n_heads / p->n_kv) + kTileRows - 1) / kTileRows;
            if (n_new[i]) longest = std::max(longest, (int64_t)p->table[seqs[i]].size());
        }
        const int64_t ctas = row_tiles * p->n_kv;
        a->small = ctas <= 2 * a->n_sm && longest * p->dim <= (ctas <= a->n_sm ? kSmallWork : kSmallWork / 8);
        if (!build_nodes(a, n, seqs, n_new)) return bad("t2sx_plan_update: too many rows over shared pages");
        const int64_t n_parts = build_items(a);
        if (n_parts >= INT32_MAX || a->items.size() * p->n_kv > (size_t)INT32_MAX ||
            a->joins.size() * (size_t)a->n_heads > (size_t)INT32_MAX)
            return bad("t2sx_plan_update: too many rows");

        DeviceGuard dg;
        POOL_CK(dg.set(p->device));
        size_t bytes = 0;
        auto place = [&](auto const& v) { const size_t at = bytes; bytes = (bytes + v.size() * sizeof(v[0]) + 15) & ~(size_t)15; return at; };
        if (!a->tc_writes) a->info.clear();   // the rows by themselves are needed on the device where a launch writes them
        const size_t o_info = place(a->info), o_items = place(a->items), o_tokens = place(a->tokens), o_pages = place(a->pages), o_joins = place(a->joins);
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
        auto grow = [&](uint8_t*& mem, size_t& have, size_t want) -> cudaError_t {
            if (have >= want) return cudaSuccess;
            cudaError_t e = p->settle();   // nothing of the plan runs any more
            if (e == cudaSuccess && mem) e = cudaFree(mem);
            mem = nullptr;
            have = 0;
            if (e == cudaSuccess) e = cudaMalloc(&mem, want + want / 2);
            if (e == cudaSuccess) have = want + want / 2;
            else cudaGetLastError();
            return e;
        };
        POOL_CK(grow(a->dev, a->dev_bytes, bytes));
        // results of parts, where tokens have several
        const size_t part_rows = (size_t)n_parts * a->n_heads, o_bytes = part_rows * p->dim * 4;
        POOL_CK(grow(a->work, a->work_bytes, o_bytes + part_rows * 8));
        auto put = [&](size_t at, auto const& v) { if (!v.empty()) memcpy(a->host[b] + at, v.data(), v.size() * sizeof(v[0])); };
        put(o_info, a->info); put(o_items, a->items); put(o_tokens, a->tokens); put(o_pages, a->pages); put(o_joins, a->joins);
        if (bytes) {
            POOL_CK(cudaMemcpyAsync(a->dev, a->host[b], bytes, cudaMemcpyHostToDevice, st));
            p->end(st);
        }
        POOL_CK(cudaEventRecord(a->sent[b], st));
        PlanView& w = a->view;
        w.rows_of = (const Token*)(a->dev + o_info);
        w.items = (const Item*)(a->dev + o_items);
        w.tokens = (const Token*)(a->dev + o_tokens);
        w.pages = (const int32_t*)(a->dev + o_pages);
        w.joins = (const Token*)(a->dev + o_joins);
        w.part_o = (float*)a->work;
        w.part_ml = (float2*)(a->work + o_bytes);
        a->version = p->version;
        a->shares = p->shares;
        a->ready = true;
        return T2SX_OK;
    });
}

template <typename T, int D>
static cudaError_t launch_attend(t2sx_plan* a, Tensors<T> x, int layer, cudaStream_t st) {
    const PlanView& w = a->view;
    using S = TileShape<D, false>;
    using Short = TileShape<D, true>;
    static std::once_flag once[64];
    std::call_once(once[a->pool->device & 63], [] {
        cudaFuncSetAttribute(k_attend_tiles<T, D, 1, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::RING);
        cudaFuncSetAttribute(k_attend_tiles<T, D, 1, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, Short::RING);
        cudaFuncSetAttribute(k_attend_tiles<T, D, kTeam<D>, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, kTeam<D> * S::RING);
    });
    auto queued = [&](cudaError_t e) {   // a launch's status; what was queued before a failure is the pool's work, too
        if (e == cudaSuccess) a->pool->end(st);
        return e;
    };
    if (a->small)
        return queued(launch(k_attend_tiles<T, D, kTeam<D>, false>, dim3((unsigned)w.n_own * w.n_kv), 32 * kTeam<D>, kTeam<D> * S::RING, st, false, w, x, 0,
                             1, 1));
    // One choice for both launches: between kernels of different shares of shared memory an SM has to run empty (2048
    // sequences of 500 positions take 350 us with one launch of each kind, 340 with two of either).
    const int64_t n_items = w.n_shared + w.n_own;
    const bool is_short = n_items * w.n_kv > (int64_t)a->n_sm * S::RESIDENT && a->launch_keys[0] + a->launch_keys[1] <= n_items * kShortItem * D;
    auto tiles = [&](int which, bool early) {   // 0: pages of several sequences, 1: the others
        const int n = which ? w.n_own : w.n_shared;
        if (!n) return cudaSuccess;
        // Short items (below kLongItem keys, on average) share a warp, as many heads as leave several warps for each place:
        // a long one hides its own start.
        const int64_t keys = a->launch_keys[which] / n;
        const int64_t places = (int64_t)a->n_sm * (is_short ? Short::RESIDENT : S::RESIDENT);
        const int64_t heads = std::min<int64_t>({(int64_t)w.n_kv, (int64_t)n * w.n_kv / (places * kWarpsPerPlace) + 1, kLongItem / (keys + 1) + 1});
        return queued(launch(is_short ? k_attend_tiles<T, D, 1, true> : k_attend_tiles<T, D, 1, false>, dim3((unsigned)(n * ((w.n_kv + heads - 1) / heads))),
                             32, is_short ? Short::RING : S::RING, st, early, w, x, w.n_tc + (which ? w.n_shared : 0), (int)heads,
                             which ? (int)a->folds : 0));
    };
    cudaError_t e = cudaSuccess;
    bool early = false;   // a launch of this call comes before
    if (w.n_tc) {
        if (x.k_new && a->tc_writes) {
            const int row_vec = D * 2 / 16;
            const int64_t vecs = (int64_t)w.rows * w.n_kv * row_vec;
            k_write_rows<<<(unsigned)((vecs + 255) / 256), 256, 0, st>>>(w.rows_of, w.rows, (const uint4*)x.k_new, (const uint4*)x.v_new,
                                                                        x.kv_stride / 8, (uint4*)x.k, (uint4*)x.v, w.n_kv, row_vec);
            e = queued(cudaGetLastError());
            x.k_new = x.v_new = nullptr;
            early = true;
        }
        if (e == cudaSuccess) e = queued(launch_tc(w, x, a->pool, a->map_k, a->map_v, layer * a->pool->n_pages, a->err_dev, early, st));
        early = true;
    }
    if (e == cudaSuccess) e = tiles(0, early);
    early |= w.n_shared > 0;
    if (e == cudaSuccess) e = tiles(1, early);
    if (e == cudaSuccess && w.n_joins) {
        const int64_t rows = (int64_t)w.n_joins * a->n_heads;
        e = queued(a->most_parts <= 32 ? launch(k_join_few<T, D>, dim3((unsigned)((rows + 3) / 4)), 128, 0, st, true, w, x)
                                       : launch(k_join_parts<T, D>, dim3((unsigned)rows), 128, 0, st, true, w, x));
    }
    return e;
}

template <typename T>
static cudaError_t attend(t2sx_plan* a, int32_t layer, const void* q, int64_t q_stride, const void* k_new, const void* v_new,
                          int64_t kv_stride, float scale, void* out, int64_t out_stride, float* lse, cudaStream_t st) {
    t2sx_pool* p = a->pool;
    const size_t first = (size_t)layer * p->n_pages * p->n_kv * kPoolPage * p->dim;
    const Tensors<T> x = {(const T*)q, (T*)p->k + first, (T*)p->v + first, (const T*)k_new, (const T*)v_new, kv_stride,
                          (T*)out, lse, q_stride, out_stride, scale * kLog2e};
    if (p->dim == 32) return launch_attend<T, 32>(a, x, layer, st);
    if (p->dim == 64) return launch_attend<T, 64>(a, x, layer, st);
    return launch_attend<T, 128>(a, x, layer, st);
}

static int plan_error(t2sx_plan* a) {
    volatile int32_t* e = a->err;
    if (!*e) return T2SX_OK;
    *e = 0;
    return t2sx_set_error(T2SX_ERR_TIMEOUT, "a tensor-core attention of this plan gave up waiting; its outputs are NaN");
}

extern "C" int t2sx_plan_sync(t2sx_plan* a) {
    if (!a) return bad("t2sx_plan_sync: null plan");
    DeviceGuard dg;
    POOL_CK(dg.set(a->pool->device));
    POOL_CK(a->pool->settle());
    return plan_error(a);
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
    if (a->view.rows == 0) return T2SX_OK;
    if (!q_dev || !out_dev || !k_new_dev != !v_new_dev) return bad("t2sx_plan_attend: null q or out, or only one of k_new and v_new");
    if (!std::isfinite(scale)) return bad("t2sx_plan_attend: scale must be finite");
    const int64_t row = (int64_t)a->n_heads * p->dim, kv_row = (int64_t)p->n_kv * p->dim;
    if (q_stride < row || out_stride < row || q_stride % 8 || out_stride % 8 || (k_new_dev && (kv_stride < kv_row || kv_stride % 8)))
        return bad("t2sx_plan_attend: strides must be multiples of 8 and no less than a row");
    if (((uintptr_t)q_dev | (uintptr_t)out_dev | (uintptr_t)k_new_dev | (uintptr_t)v_new_dev) & 15 || ((uintptr_t)lse_dev & 3))
        return bad("t2sx_plan_attend: tensors must be 16-byte aligned");
    if (a->shares != p->shares) {   // forks since: full pages of the rows may be shared by now
        for (int32_t page : a->row_pages) a->shared_rows |= p->users[page] > 1;
        a->shares = p->shares;
    }
    if (k_new_dev && a->shared_rows)
        return t2sx_set_error(T2SX_ERR_STATE, "t2sx_plan_attend: a row's position is in a page of several sequences, which is not written");
    if (int rc = plan_error(a)) return rc;
    cudaStream_t st = (cudaStream_t)stream;
    DeviceGuard dg;
    POOL_CK(dg.set(p->device));
    POOL_CK(p->begin(st));
    auto go = p->type == T2SX_TYPE_F16 ? attend<__half> : attend<__nv_bfloat16>;
    POOL_CK(go(a, layer, q_dev, q_stride, k_new_dev, v_new_dev, kv_stride, scale, out_dev, out_stride, lse_dev, st));
    return T2SX_OK;
}
