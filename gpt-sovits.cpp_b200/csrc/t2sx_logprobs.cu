// Log probabilities of given tokens, with the rows' entropy, the tokens' ranks and the best tokens.
//
//   m = max x,  s = sum e^(x - m),  w = sum e^(x - m) (x - m)     (over x > -inf)
//   logprob = x_t - m - log s,   entropy = log s - w / s
//   rank = #{x > x_t} + #{j < t: x_j = x_t}
//
// One pass over the logits: each thread holds a running (m, s, w), rescaled when its maximum grows
// (s' = s e^(m - m'), w' = e^(m - m') (w + (m - m') s)), and leaves the maximum of each slot of
// kGroup x slot_groups vectors in shared memory.  A value T that at least top_k elements reach follows
// from the threads' maxima alone (T0 below); the slots that reach T, a few, are read again
// and their elements >= T are the candidates, whose places in the list are counted.
#include "../../include/t2sx.h"
#include "t2sx_kernels.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdio>
#include <mutex>

using namespace t2sx;

int t2sx_set_error(int code, const char* msg);

namespace {

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }

constexpr int kGroup = 4;            // 16-byte vectors that a thread has in flight
constexpr int kCandidates = 1024;    // of one CTA of eight warps, a quarter of it for rows of fewer
constexpr int kHits = 512;           // slots of one CTA that candidates come from (a quarter likewise)
constexpr int kMaxTop = 32;
constexpr int kMaxSplit = 8;         // CTAs per row (a portable cluster)
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kExtreme = 5e37f;    // maxima from here on (also below -5e37) leave the range of x log2(e)

// What a thread subtracts from x log2(e): 0 while it has seen nothing.
__device__ __forceinline__ float reference(float m) { return m > -INFINITY ? fminf(fmaxf(m, -kExtreme), kExtreme) * kLog2e : 0.0f; }

// Value and id of a candidate as one key: greater keys come first (values descending, ids
// ascending).  -inf and NaN have no place in a list.
__device__ __forceinline__ unsigned long long order_key(float x, unsigned id) {
    unsigned b = __float_as_uint(x + 0.0f);   // one zero
    b = (b & 0x80000000u) ? ~b : b | 0x80000000u;
    return (unsigned long long)b << 32 | (0xFFFFFFFFu - id);
}
__device__ __forceinline__ float key_value(unsigned long long key) {
    unsigned b = (unsigned)(key >> 32);
    return __uint_as_float((b & 0x80000000u) ? b & 0x7FFFFFFFu : ~b);
}

// 2^x; the instruction's error is two units in the last place
__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {   // NaN if one of them is
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    unsigned long long r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(*reinterpret_cast<unsigned long long*>(&a)), "l"(*reinterpret_cast<unsigned long long*>(&b)));
    return *reinterpret_cast<float2*>(&r);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    unsigned long long r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(*reinterpret_cast<unsigned long long*>(&a)), "l"(*reinterpret_cast<unsigned long long*>(&b)));
    return *reinterpret_cast<float2*>(&r);
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    unsigned long long r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(*reinterpret_cast<unsigned long long*>(&a)), "l"(*reinterpret_cast<unsigned long long*>(&b)),
        "l"(*reinterpret_cast<unsigned long long*>(&c)));
    return *reinterpret_cast<float2*>(&r);
}

// Masks of two comparisons, 0xFFFF for each half, added up modulo 2^32: with l ones in the low halves and h in the high
// ones that is 65536 (l - h) - l (less than 65536 of either).
struct CountMasks {
    unsigned acc = 0;
    __device__ __forceinline__ int sum() const {
        const unsigned l = -acc & 0xFFFFu;
        return (int)(l + (l - ((acc + l) >> 16) & 0xFFFFu));
    }
};

// A 16-byte vector of logits: its elements in f32, its maximum (NaN left out), -inf in every place.
template <typename T>
struct Vec;
template <>
struct Vec<float> {
    static constexpr int E = 4;
    static __device__ __forceinline__ uint4 none() { return make_uint4(0xFF800000u, 0xFF800000u, 0xFF800000u, 0xFF800000u); }
    static __device__ __forceinline__ float2 pair(unsigned const (&w)[4], int i) {
        return make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
    }
    static __device__ __forceinline__ void raise(uint4&) {}   // done to y instead
    static constexpr float kLow = -kExtreme;
    static __device__ __forceinline__ float max(const uint4 (&u)[kGroup]) {
        float m = -INFINITY;
#pragma unroll
        for (int g = 0; g < kGroup; ++g)
            m = fmaxf(m, fmaxf(fmaxf(__uint_as_float(u[g].x), __uint_as_float(u[g].y)), fmaxf(__uint_as_float(u[g].z), __uint_as_float(u[g].w))));
        return m;
    }
    // elements greater than a threshold, counted in the halves of acc
    struct Count {
        int n = 0;
        __device__ __forceinline__ void add(const uint4& u, float above) {
            n += (__uint_as_float(u.x) > above) + (__uint_as_float(u.y) > above) + (__uint_as_float(u.z) > above) + (__uint_as_float(u.w) > above);
        }
        __device__ __forceinline__ int sum() const { return n; }
    };
    // the greatest value of the type below x (not for -inf)
    static __device__ __forceinline__ float below(float x) {
        const unsigned b = __float_as_uint(x);
        return __uint_as_float((b & 0x7FFFFFFFu) == 0 ? 0x80000001u : (b & 0x80000000u) ? b + 1 : b - 1);
    }
};
template <>
struct Vec<__half> {
    static constexpr int E = 8;
    static __device__ __forceinline__ uint4 none() { return make_uint4(0xFC00FC00u, 0xFC00FC00u, 0xFC00FC00u, 0xFC00FC00u); }
    static __device__ __forceinline__ float2 pair(unsigned const (&w)[4], int i) { return __half22float2(*reinterpret_cast<const __half2*>(&w[i])); }
    // the lowest finite value instead of -inf: as good as -inf unless the row's maximum is near it
    static __device__ __forceinline__ void raise(uint4& u) {
        __half2* h = reinterpret_cast<__half2*>(&u);
        const __half2 low = __half2half2(__ushort_as_half(0xFBFFu));
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = __hmax2_nan(h[i], low);
    }
    static constexpr float kLow = -65000.0f;   // rows whose maximum is below have sums of their own
    static __device__ __forceinline__ float max(const uint4 (&u)[kGroup]) {
        __half2 m;
#pragma unroll
        for (int g = 0; g < kGroup; ++g) {
            const __half2* h = reinterpret_cast<const __half2*>(&u[g]);
            const __half2 y = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
            m = g ? __hmax2(m, y) : y;
        }
        return fmaxf(__low2float(m), __high2float(m));
    }
    struct Count : CountMasks {
        __device__ __forceinline__ void add(const uint4& u, float above) {
            const __half2 *h = reinterpret_cast<const __half2*>(&u), a = __float2half2_rn(above);
            acc += __hgt2_mask(h[0], a) + __hgt2_mask(h[1], a);
            acc += __hgt2_mask(h[2], a) + __hgt2_mask(h[3], a);
        }
    };
    static __device__ __forceinline__ float below(float x) {
        const unsigned b = __half_as_ushort(__float2half_rn(x));
        const unsigned short r = (unsigned short)((b & 0x7FFFu) == 0 ? 0x8001u : (b & 0x8000u) ? b + 1 : b - 1);
        return __half2float(__ushort_as_half(r));
    }
};
template <>
struct Vec<__nv_bfloat16> {
    static constexpr int E = 8;
    static __device__ __forceinline__ uint4 none() { return make_uint4(0xFF80FF80u, 0xFF80FF80u, 0xFF80FF80u, 0xFF80FF80u); }
    static __device__ __forceinline__ float2 pair(unsigned const (&w)[4], int i) {
        return make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xFFFF0000u));
    }
    static __device__ __forceinline__ void raise(uint4& u) {   // to -2^127, whose product with log2(e) is finite
        __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&u);
        const __nv_bfloat162 low = __bfloat162bfloat162(__ushort_as_bfloat16(0xFF00u));
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = __hmax2_nan(h[i], low);
    }
    static constexpr float kLow = -kExtreme;
    static __device__ __forceinline__ float max(const uint4 (&u)[kGroup]) {
        __nv_bfloat162 m;
#pragma unroll
        for (int g = 0; g < kGroup; ++g) {
            const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&u[g]);
            const __nv_bfloat162 y = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
            m = g ? __hmax2(m, y) : y;
        }
        return fmaxf(__low2float(m), __high2float(m));
    }
    struct Count : CountMasks {
        __device__ __forceinline__ void add(const uint4& u, float above) {
            const __nv_bfloat162 *h = reinterpret_cast<const __nv_bfloat162*>(&u), a = __float2bfloat162_rn(above);
            acc += __hgt2_mask(h[0], a) + __hgt2_mask(h[1], a);
            acc += __hgt2_mask(h[2], a) + __hgt2_mask(h[3], a);
        }
    };
    static __device__ __forceinline__ float below(float x) {
        const unsigned b = __bfloat16_as_ushort(__float2bfloat16_rn(x));
        const unsigned short r = (unsigned short)((b & 0x7FFFu) == 0 ? 0x8001u : (b & 0x8000u) ? b + 1 : b - 1);
        return __bfloat162float(__ushort_as_bfloat16(r));
    }
};

// A slot's maximum in 16 bits, never below it (the upper half of an f32, rounded up).
__device__ __forceinline__ unsigned short slot_up(float x) {
    const unsigned b = __float_as_uint(x);
    return (unsigned short)((b & 0x80000000u) ? b >> 16 : (b + 0xFFFFu) >> 16);
}
__device__ __forceinline__ float slot_value(unsigned short b) { return __uint_as_float((unsigned)b << 16); }

struct Stat {   // of part of a row
    float m, s, w;      // s, w relative to m; all of them 0 but m where every element is -inf
    int before;
};
__device__ __forceinline__ Stat join(const Stat& a, const Stat& b) {
    Stat r;
    r.m = fmaxf(a.m, b.m);
    // a part without an element above -inf has s = w = 0 (or NaN, which stays)
    const float da = a.m == r.m ? 0.0f : fmaxf(a.m - r.m, -1e30f), db = b.m == r.m ? 0.0f : fmaxf(b.m - r.m, -1e30f);
    const float fa = ex2(da * kLog2e), fb = ex2(db * kLog2e);
    r.s = fmaf(a.s, fa, b.s * fb);
    r.w = fmaf(fa, fmaf(da, a.s, a.w), fb * fmaf(db, b.s, b.w));
    r.before = a.before + b.before;
    return r;
}
__device__ __forceinline__ Stat warp_join(Stat a) {
    for (int x = 16; x; x >>= 1) {
        Stat b;
        b.m = __shfl_xor_sync(~0u, a.m, x);
        b.s = __shfl_xor_sync(~0u, a.s, x);
        b.w = __shfl_xor_sync(~0u, a.w, x);
        b.before = __shfl_xor_sync(~0u, a.before, x);
        // both lanes take the same operands in the same order
        a = (threadIdx.x & x) ? join(b, a) : join(a, b);
    }
    return a;
}

// The lanes' values in descending order.
__device__ __forceinline__ float warp_sort(float v) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
        for (int x = size >> 1; x; x >>= 1) {
            const float o = __shfl_xor_sync(~0u, v, x);
            const bool keep_max = ((lane & x) == 0) == ((lane & size) == 0);
            v = keep_max ? fmaxf(v, o) : fminf(v, o);
        }
    return v;
}

struct Args {
    long long stride;
    int rows, vocab, top_k, slot_groups;
    const int32_t* tokens;
    float *logprob, *entropy;
    int32_t *rank, *top_ids;
    float* top_logprobs;
};

template <int WARPS>
struct Shared {   // of one row's threads in a CTA
    Stat stat[WARPS];
    float best_max[WARPS][32];
    int count, n_hits;
    unsigned short hits[WARPS < 8 ? kHits / 4 : kHits];   // slots that reach T0: number x threads + thread
    unsigned long long best[WARPS];
    static constexpr int PARTS = WARPS < 8 ? 1 : kMaxSplit;
    Stat joined[PARTS];                                  // in the first CTA of a row: all of its CTAs'
    unsigned long long lists[PARTS][kMaxTop];
    unsigned long long cand[WARPS < 8 ? kCandidates / 4 : kCandidates];
};

// WARPS == 1: a warp per row, four rows in a CTA.  Else a row per CTA, or (WARPS == 8) per cluster of `split` CTAs:
// each takes a range of the row's vectors, and the first one joins what they found.
//
// While 16-bit rows are read, issue and the exponential unit bound it: an element is an exponential (16 a cycle and SM) and some eight
// other instructions, packed ones counted once.  Over the whole of 2048 rows of 100003 in bf16 with the 20 best neither is full, nor
// is DRAM (63, 61 and 61%): the rows of a wave come to their lists, where nothing is loaded, together.  That takes 85 us, 4.8 TB/s (77
// without list and rank).  4 rows of 131072 in f16 take 10.3 us, of which most is the way from launch to the joined lists.
// 2048 rows of 1025 in f32 take 9 us where 8 rows take 6: a row's phases after its loads (the maxima sorted, the slots, their vectors
// again, places) follow one another.  Times are the device's, of calls one after another with the same logits.
template <typename T, int WARPS>
__global__ void __launch_bounds__(WARPS == 1 ? 128 : 32 * WARPS, WARPS == 1 ? 6 : 32 / WARPS)
k_logprobs(const T* __restrict__ logits, Args a) {
    constexpr int E = Vec<T>::E, N = 32 * WARPS, ROWS = WARPS == 1 ? 4 : 1;
    constexpr int CAND = WARPS < 8 ? kCandidates / 4 : kCandidates, HITS = WARPS < 8 ? kHits / 4 : kHits;
    extern __shared__ __align__(16) unsigned char raw[];
    const int sub = WARPS == 1 ? threadIdx.x >> 5 : 0, tid = WARPS == 1 ? threadIdx.x & 31 : threadIdx.x;
    const int lane = threadIdx.x & 31, warp = WARPS == 1 ? 0 : threadIdx.x >> 5;
    Shared<WARPS>& sh = reinterpret_cast<Shared<WARPS>*>(raw)[sub];
    const int split = WARPS < 8 ? 1 : (int)gridDim.y, part = WARPS < 8 ? 0 : (int)blockIdx.y;
    const long long row = (long long)blockIdx.x * ROWS + sub;
    if (WARPS == 1 && row >= a.rows) return;   // warps of such a CTA wait for none of the others
    auto sync = [] {
        if constexpr (WARPS == 1) __syncwarp();
        else __syncthreads();
    };
    if (split > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");   // this CTA runs: its memory may be written
    const T* x = logits + row * a.stride;
    const int t = a.tokens[row];
    const bool given = t >= 0 && t < a.vocab;

    // The row on the grid of aligned vectors, and the elements before and after its whole ones: those are
    // fewer than E each, and one thread takes one.
    const int off = (int)(((uintptr_t)x & 15) / sizeof(T));
    const uint4* xv = reinterpret_cast<const uint4*>(x - off);
    const int full0 = off ? 1 : 0, full1 = max(full0, (int)(((long long)off + a.vocab) / E));
    const int per = (full1 - full0 + split - 1) / split, v0 = full0 + part * per, v1 = min(full1, v0 + per);
    int edge = tid < E ? tid : full1 * E - off + tid - E;   // its id
    if (tid < E ? part != 0 || edge >= min(a.vocab, full0 * E - off) : part != split - 1 || tid >= 2 * E || edge < 0) edge = a.vocab;
    auto load = [&](int v) -> uint4 { return v < v1 ? __ldg(xv + v) : Vec<T>::none(); };

    uint4 u[kGroup];
#pragma unroll
    for (int g = 0; g < kGroup; ++g) u[g] = load(v0 + g * N + tid);
    const float edge_x = edge < a.vocab ? to_f32(x[edge]) : -INFINITY;
    const float xt = given ? to_f32(x[t]) : INFINITY, xt_below = Vec<T>::below(xt);
    unsigned short* slots = reinterpret_cast<unsigned short*>(raw + ROWS * sizeof(Shared<WARPS>));
    int n_slots = 0;
    // The edge's element is the first one of the thread, its weight against the rounded reference like all others' (below): the
    // reference's rounding, up to half a unit of it, is taken out of their sum at the end.
    float m = fmaxf(edge_x, -INFINITY), ref = reference(m), slot = -INFINITY;
    const float edge_y = max_nan(fmaf(edge_x, kLog2e, -ref), -1e30f), edge_e = ex2(edge_y);
    float2 s = {edge_e, 0.0f}, w = {edge_e * edge_y, 0.0f};
    int before = edge < a.vocab && (edge_x > xt || (edge_x == xt && edge < t));
    for (int base = v0, group = 0; base < v1; base += kGroup * N) {
        uint4 c[kGroup];
#pragma unroll
        for (int g = 0; g < kGroup; ++g) {
            c[g] = u[g];
            u[g] = Vec<T>::none();
        }
        if (base + 2 * kGroup * N <= v1) {
#pragma unroll
            for (int g = 0; g < kGroup; ++g) u[g] = __ldg(xv + (base + tid) + (kGroup + g) * N);
        } else if (base + kGroup * N < v1) {
#pragma unroll
            for (int g = 0; g < kGroup; ++g) u[g] = load(base + (kGroup + g) * N + tid);
        }
        const float g_max = Vec<T>::max(c);
        slot = fmaxf(slot, g_max);
        if (++group == a.slot_groups) {
            slots[(n_slots++ * ROWS + sub) * N + tid] = slot_up(slot);
            slot = -INFINITY;
            group = 0;
        }
        if (g_max > m) {
            const float up = reference(g_max);
            if (m > -INFINITY) {
                const float d = fmaxf(ref - up, -1e30f), f = ex2(d);
                w = mul2(make_float2(f, f), fma2(make_float2(d, d), s, w));
                s = mul2(make_float2(f, f), s);
            }
            m = g_max;
            ref = up;
        }
        if (g_max >= xt) {
            typename Vec<T>::Count more;
            // up to the token equal values come before it, too
            const bool after = base * E - off > t;
            if ((after || (base + kGroup * N) * E - off <= t) && xt > -INFINITY) {
#pragma unroll
                for (int g = 0; g < kGroup; ++g) more.add(c[g], after ? xt : xt_below);
            } else
#pragma unroll
            for (int g = 0; g < kGroup; ++g) {
                const int vec = base + g * N + tid, j = vec * E - off;
                if ((j + E <= t || j > t) && xt > -INFINITY) {
                    more.add(c[g], j > t ? xt : xt_below);
                } else if (vec < v1) {
                    const unsigned b[4] = {c[g].x, c[g].y, c[g].z, c[g].w};
#pragma unroll
                    for (int i = 0; i < E; ++i) {
                        const float2 p = Vec<T>::pair(b, i / 2);
                        const float v = (i & 1) ? p.y : p.x;
                        before += v > xt || (v == xt && j + i < t);
                    }
                }
            }
            before += more.sum();
        }
        // y = x log2(e) - ref, rounded once; what lies below the floor has the weight 0 in finite numbers, and NaN
        // stays in the sums
#pragma unroll
        for (int g = 0; g < kGroup; ++g) {
            Vec<T>::raise(c[g]);
            const unsigned b[4] = {c[g].x, c[g].y, c[g].z, c[g].w};
#pragma unroll
            for (int i = 0; i < E / 2; ++i) {
                float2 y = fma2(Vec<T>::pair(b, i), make_float2(kLog2e, kLog2e), make_float2(-ref, -ref));
                if (E == 4) { y.x = max_nan(y.x, -1e30f); y.y = max_nan(y.y, -1e30f); }
                const float2 e = make_float2(ex2(y.x), ex2(y.y));
                s = add2(s, e);
                w = fma2(e, y, w);
            }
        }
        if (base + kGroup * N >= v1 && group) slots[(n_slots++ * ROWS + sub) * N + tid] = slot_up(slot);
    }

    // this thread's part relative to m itself (ref is a rounded number), then the warp's, then the CTA's
    const float rest = fabsf(m) < kExtreme ? fmaf(m, kLog2e, -ref) : 0.0f, back = ex2(-rest);
    const float s1 = s.x + s.y;
    Stat st = warp_join(Stat{m, s1 * back, kLn2 * back * fmaf(-rest, s1, w.x + w.y), before});
    // T0: the top_k-th greatest of the threads' maxima, so at least top_k elements reach it (-inf: fewer than
    // top_k threads have an element above -inf)
    float T0 = a.top_k ? warp_sort(m) : -INFINITY;
    if constexpr (WARPS > 1) {
        if (lane == 0) sh.stat[warp] = st;
        if (tid == 0) sh.count = sh.n_hits = 0;
        if (a.top_k) {
            sh.best_max[warp][lane] = T0;
            for (int h = WARPS / 2; h; h /= 2) {   // the 32 greatest of two lists, again in order
                __syncthreads();
                if (warp < h) {
                    T0 = fmaxf(T0, sh.best_max[warp + h][31 - lane]);
#pragma unroll
                    for (int y = 16; y; y >>= 1) {
                        const float o = __shfl_xor_sync(~0u, T0, y);
                        T0 = (lane & y) ? fminf(T0, o) : fmaxf(T0, o);
                    }
                    sh.best_max[warp][lane] = T0;
                }
            }
        }
        __syncthreads();
        st = sh.stat[0];
        for (int i = 1; i < WARPS; ++i) st = join(st, sh.stat[i]);
        if (a.top_k) T0 = sh.best_max[0][a.top_k - 1];
    } else {
        if (a.top_k) T0 = __shfl_sync(~0u, T0, a.top_k - 1);
        if (lane == 0) sh.count = sh.n_hits = 0;
        __syncwarp();
    }

    if (st.m > -INFINITY && (st.m < Vec<T>::kLow || st.m > kExtreme)) {
        // a maximum near the ends of the type's range: the sums anew, from x - m
        float ss = 0.0f, sw = 0.0f;
        auto add = [&](float v) {
            const float d = max_nan(v - st.m, -1e30f), e = ex2(d * kLog2e);
            ss += e;
            sw = fmaf(e, d, sw);
        };
        add(edge_x);
        for (int v = v0 + tid; v < v1; v += N) {
            const uint4 q = load(v);
            const unsigned b[4] = {q.x, q.y, q.z, q.w};
            for (int i = 0; i < E / 2; ++i) {
                const float2 p = Vec<T>::pair(b, i);
                add(p.x);
                add(p.y);
            }
        }
        for (int y = 16; y; y >>= 1) { ss += __shfl_xor_sync(~0u, ss, y); sw += __shfl_xor_sync(~0u, sw, y); }
        if constexpr (WARPS > 1) {
            __syncthreads();   // everyone has read the warps' parts
            if (lane == 0) { sh.stat[warp].s = ss; sh.stat[warp].w = sw; }
            __syncthreads();
            ss = sw = 0.0f;
            for (int i = 0; i < WARPS; ++i) { ss += sh.stat[i].s; sw += sh.stat[i].w; }
        }
        st.s = ss;
        st.w = sw;
    }
    if (split > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (a.top_k) {
        // the elements that reach T0, from the slots that do (each thread reads its own)
        if (edge_x >= T0 && edge_x > -INFINITY) {
            const int at = atomicAdd(&sh.count, 1);
            if (at < CAND) sh.cand[at] = order_key(edge_x, edge);
        }
        for (int k = 0; k < n_slots; ++k) {
            if (!(slot_value(slots[(k * ROWS + sub) * N + tid]) >= T0)) continue;
            const int at = atomicAdd(&sh.n_hits, 1);
            if (at < HITS) sh.hits[at] = (unsigned short)(k * N + tid);
        }
        sync();
        // their vectors, shared out anew: one round trip to L2 for all of them
        const int n_hits = min(sh.n_hits, HITS) * kGroup;
        for (int sg = 0; sg < a.slot_groups; ++sg)
            for (int i = tid; i < n_hits; i += N) {
                const int hit = sh.hits[i / kGroup];
                const int v = v0 + ((hit / N * a.slot_groups + sg) * kGroup + i % kGroup) * N + hit % N;
                const uint4 q = load(v);
                const unsigned b[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const float2 p = Vec<T>::pair(b, e / 2);
                    const float y = (e & 1) ? p.y : p.x;
                    if (y >= T0 && y > -INFINITY) {
                        const int at = atomicAdd(&sh.count, 1);
                        if (at < CAND) sh.cand[at] = order_key(y, v * E - off + e);
                    }
                }
            }
        sync();
        const int n = sh.n_hits > HITS ? CAND + 1 : sh.count;
        unsigned long long* list = sh.lists[0];
        if (split > 1) {   // in the first CTA of the row
            unsigned long long* mine = sh.lists[part];
            asm("mapa.u64 %0, %1, 0;" : "=l"(list) : "l"(mine));
        }
        for (int i = tid; i < a.top_k; i += N) list[i] = 0;
        sync();
        if (n <= CAND) {
            // a candidate's place is the number of greater ones: keys differ, whatever order they came in
            for (int i = tid; i < n; i += N) {
                const unsigned long long key = sh.cand[i];
                int place = 0;
#pragma unroll 4
                for (int j = 0; j < n; ++j) place += sh.cand[j] > key;
                if (place < a.top_k) list[place] = key;
            }
        } else {
            // more ties than the list of candidates holds: place by place, the greatest key below the last one
            unsigned long long last = ~0ull;
            for (int i = 0; i < a.top_k && last; ++i) {
                unsigned long long best = edge_x > -INFINITY ? order_key(edge_x, edge) : 0;
                if (best >= last) best = 0;
                for (int v = v0 + tid; v < v1; v += N) {
                    const uint4 q = load(v);
                    const unsigned b[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        const float2 p = Vec<T>::pair(b, e / 2);
                        const float y = (e & 1) ? p.y : p.x;
                        if (!(y > -INFINITY)) continue;
                        const unsigned long long key = order_key(y, v * E - off + e);
                        if (key < last && key > best) best = key;
                    }
                }
                for (int y = 16; y; y >>= 1) {
                    const unsigned long long o = __shfl_xor_sync(~0u, best, y);
                    best = o > best ? o : best;
                }
                if constexpr (WARPS > 1) {
                    __syncthreads();
                    if (lane == 0) sh.best[warp] = best;
                    __syncthreads();
                    for (int k = 0; k < WARPS; ++k) best = sh.best[k] > best ? sh.best[k] : best;
                }
                if (tid == 0) list[i] = best;
                last = best;
            }
        }
    }
    if (split > 1) {
        if (tid == 0) {
            Stat *mine = &sh.joined[part], *first;
            asm("mapa.u64 %0, %1, 0;" : "=l"(first) : "l"(mine));
            *first = st;
        }
        asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
        if (part != 0) return;
        st = sh.joined[0];
        for (int i = 1; i < split; ++i) st = join(st, sh.joined[i]);
    } else {
        sync();
    }
    const bool bad = !(st.s < INFINITY);   // NaN or +inf in the row
    const float log_s = st.s > 0.0f ? logf(st.s) : 0.0f;
    if (tid == 0) {
        a.logprob[row] = t == -1 ? 0.0f : !given || bad ? NAN : st.s > 0.0f ? xt - st.m - log_s : -INFINITY;
        if (a.entropy) a.entropy[row] = bad ? NAN : st.s > 0.0f ? log_s - st.w / st.s : 0.0f;
        if (a.rank) a.rank[row] = given ? st.before : -1;
    }
    // the parts' lists, each in order: an entry's place is the number of greater ones (empty ones: of earlier ones)
    for (int i = tid; i < split * kMaxTop; i += N) {
        const int mine = i / kMaxTop, at = i % kMaxTop;
        if (at >= a.top_k) continue;
        const unsigned long long key = sh.lists[mine][at];
        int place = at;
        for (int q = 0; q < split; ++q) {
            if (q == mine) continue;
#pragma unroll 4
            for (int j = 0; j < a.top_k; ++j) place += sh.lists[q][j] > key || (key == 0 && q < mine);
        }
        if (place < a.top_k) {
            const unsigned id = 0xFFFFFFFFu - (unsigned)key;
            a.top_ids[row * a.top_k + place] = key ? (int)id : -1;
            a.top_logprobs[row * a.top_k + place] = bad ? NAN : key ? key_value(key) - st.m - log_s : -INFINITY;
        }
    }
}

template <typename T, int WARPS>
cudaError_t launch(const T* x, Args a, int split, cudaStream_t st) {
    constexpr int N = 32 * WARPS, ROWS = WARPS == 1 ? 4 : 1;
    // slots of 16 bits: at most 32 KB of them, so that a CTA's share of shared memory stays small
    const long long vecs = ((long long)a.vocab / Vec<T>::E + 1 + split - 1) / split;
    const long long groups = (vecs + (long long)kGroup * N - 1) / ((long long)kGroup * N);
    const int most = (32 << 10) / (2 * N * ROWS);
    a.slot_groups = (int)((groups + most - 1) / most);
    const size_t smem = ROWS * sizeof(Shared<WARPS>) + (size_t)((groups + a.slot_groups - 1) / a.slot_groups) * ROWS * N * 2;
    static std::once_flag once[64];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    std::call_once(once[dev & 63], [&] {
        cudaFuncSetAttribute(k_logprobs<T, WARPS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (32 << 10) + ROWS * (int)sizeof(Shared<WARPS>));
    });
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(((long long)a.rows + ROWS - 1) / ROWS), split);
    cfg.blockDim = WARPS == 1 ? 128 : N;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = 1;
    at.val.clusterDim.y = split;
    at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = split > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, k_logprobs<T, WARPS>, x, a);
}

template <typename T>
cudaError_t dispatch(const T* x, const Args& a, int sms, cudaStream_t st) {
    // Warps of a row: those that let all rows run at one time, since what follows a row's pass (the merges of the
    // warps' maxima, the candidates) costs each of its warps as much.  With 1, 2, 4, 8 warps, 20 best, in us:
    //   2048 x 1025 f32   10.4  10.4  14.6  27.2        2048 x 200 f32      8.3  10.3  14.4  26.8
    //   2048 x 4096 f32   16.6  14.5  18.6  28.8        2048 x 100003 bf16  105   84.6  86.1  92.6
    //   1184 x 50000 bf16 46.8  33.4  32.9  39.2        512 x 32000 f16    25.0  18.2  15.5  16.6
    //   256 x 1025 f32     8.4   7.0   6.3   8.3        8 x 1025 f32        8.3   6.5   6.2   7.4
    //   256 x 32000 bf16  26.9  15.8  12.5  12.4        4 x 131072 f16     82.6   -     -    18.8
    if (a.rows > 8 * sms) return a.vocab <= 2048 ? launch<T, 1>(x, a, 1, st) : launch<T, 2>(x, a, 1, st);
    if (a.rows > 2 * sms || a.vocab <= 4096) return launch<T, 4>(x, a, 1, st);
    // CTAs of a row: 4 x 131072 takes 18.8, 14.6, 12.4, 11.6 us with 1, 2, 4, 8 of them; 64 x 8192 8.3 with one, 10.4
    // with four
    int split = 1;
    while (split < kMaxSplit && a.rows * split <= sms && a.vocab / (2 * split) >= 4096) split *= 2;
    return launch<T, 8>(x, a, split, st);
}

int bad(const char* m) { return t2sx_set_error(T2SX_ERR_INVALID, m); }

}  // namespace

extern "C" int t2sx_token_logprobs(int32_t device, int32_t type, int64_t rows, int64_t vocab, const void* logits_dev,
                                   int64_t stride, const int32_t* tokens_dev, int32_t top_k, float* logprob_dev,
                                   float* entropy_dev, int32_t* rank_dev, int32_t* top_ids_dev, float* top_logprobs_dev,
                                   void* stream) {
    if (type != T2SX_TYPE_F32 && type != T2SX_TYPE_F16 && type != T2SX_TYPE_BF16)
        return bad("t2sx_token_logprobs: the type must be f32, f16 or bf16");
    if (rows < 0 || rows > INT32_MAX || vocab <= 0 || vocab > (1 << 30) || stride < vocab || stride > (int64_t)1 << 40)
        return bad("t2sx_token_logprobs: rows, vocab or stride out of range");
    if (top_k < 0 || top_k > 32) return bad("t2sx_token_logprobs: top_k must be 0 to 32");
    if (rows == 0) return T2SX_OK;
    if (!logits_dev || !tokens_dev || !logprob_dev || (top_k > 0 && (!top_ids_dev || !top_logprobs_dev)))
        return bad("t2sx_token_logprobs: null logits, tokens or output");
    if (((uintptr_t)logits_dev % (type == T2SX_TYPE_F32 ? 4 : 2)) ||
        (((uintptr_t)tokens_dev | (uintptr_t)logprob_dev | (uintptr_t)entropy_dev | (uintptr_t)rank_dev | (uintptr_t)top_ids_dev |
          (uintptr_t)top_logprobs_dev) & 3))
        return bad("t2sx_token_logprobs: misaligned pointer");
    DeviceGuard dg;
    cudaError_t e = dg.set(device);
    if (e != cudaSuccess) return t2sx_set_error(T2SX_ERR_CUDA, cudaGetErrorString(e));
    int sms = 0;
    e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
    if (e != cudaSuccess) return t2sx_set_error(T2SX_ERR_CUDA, cudaGetErrorString(e));
    cudaStream_t st = (cudaStream_t)stream;
    const Args a = {(long long)stride, (int)rows, (int)vocab, top_k, 1, tokens_dev, logprob_dev, entropy_dev, rank_dev, top_ids_dev,
                    top_logprobs_dev};
    if (type == T2SX_TYPE_F32) e = dispatch((const float*)logits_dev, a, sms, st);
    else if (type == T2SX_TYPE_F16) e = dispatch((const __half*)logits_dev, a, sms, st);
    else e = dispatch((const __nv_bfloat16*)logits_dev, a, sms, st);
    if (e != cudaSuccess) return t2sx_set_error(T2SX_ERR_CUDA, cudaGetErrorString(e));
    return T2SX_OK;
}
