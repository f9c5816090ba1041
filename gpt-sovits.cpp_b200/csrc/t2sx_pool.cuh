// A pool of cache pages that sequences share: host bookkeeping and the order of its device work.
#pragma once
#include "../../include/t2sx.h"
#include "t2sx_kernels.cuh"

#include <cuda_runtime.h>

#include <cstdint>
#include <cstdio>
#include <vector>

int t2sx_set_error(int code, const char* msg);

namespace t2sx {

constexpr int kPoolPage = 64;                   // positions per page
constexpr int kPoolMaxPages = 1 << 26;
constexpr int64_t kPoolMaxLen = (int64_t)1 << 30;

inline int32_t pages_of(int64_t len) { return (int32_t)((len + kPoolPage - 1) / kPoolPage); }

// One page copy: the first `fill` positions of every layer and head.
struct PageMove {
    int32_t src, dst, fill;
};

}  // namespace t2sx

struct t2sx_pool {
    int device = 0, type = 0, n_layers = 0, n_pages = 0, n_kv = 0, dim = 0, max_seqs = 0;
    uint16_t *k = nullptr, *v = nullptr;
    std::vector<std::vector<int32_t>> table;   // [max_seqs] page ids
    std::vector<int64_t> len;                  // [max_seqs]
    std::vector<int32_t> users;                // [n_pages] sequences that hold the page
    std::vector<uint64_t> free_bits;           // bit p % 64 of word p / 64: page p is free
    size_t first_free_word = 0;                // no word before it has a free page
    int64_t n_free = 0;
    uint64_t version = 0;                      // changes when a page may have passed to another owner
    uint64_t shares = 0;                       // changes when a page may have got another user
    std::vector<uint8_t> mark;                 // [max_seqs] scratch of the argument checks
    std::vector<t2sx::PageMove> moves;         // scratch of a call
    int n_plans = 0;
    bool closed = false;
    cudaEvent_t done = nullptr;
    cudaStream_t last = nullptr;               // the last device work's
    bool worked = false;

    int32_t take() {   // the lowest free page; the caller has checked n_free
        while (!free_bits[first_free_word]) ++first_free_word;
        const int b = __builtin_ctzll(free_bits[first_free_word]);
        free_bits[first_free_word] &= free_bits[first_free_word] - 1;
        --n_free;
        const int32_t p = (int32_t)(first_free_word * 64 + b);
        users[p] = 1;
        return p;
    }
    void drop(int32_t p) {
        if (--users[p]) return;
        free_bits[p >> 6] |= (uint64_t)1 << (p & 63);
        if ((size_t)(p >> 6) < first_free_word) first_free_word = p >> 6;
        ++n_free;
    }
    // Device work of a call comes after begin, which waits for work on another stream; end follows each piece that was queued,
    // so that a call which fails halfway leaves a right `last`.  The event is recorded when the stream changes, not after
    // every call (which took a fifth of a small call's time on the host).
    cudaError_t begin(cudaStream_t st) {
        if (!worked || st == last) return cudaSuccess;
        cudaError_t e = cudaEventRecord(done, last);
        return e == cudaSuccess ? cudaStreamWaitEvent(st, done, 0) : e;
    }
    void end(cudaStream_t st) {
        last = st;
        worked = true;
    }
    // All device work is done.
    cudaError_t settle() {
        if (!worked) return cudaSuccess;
        cudaError_t e = cudaEventRecord(done, last);
        if (e == cudaSuccess) e = cudaEventSynchronize(done);
        if (e == cudaSuccess) worked = false;   // nothing to wait for: `last` is not looked at any more
        return e;
    }
};

void t2sx_pool_release_object(t2sx_pool* p);

#define POOL_CK(x)                                                                                      \
    do {                                                                                                \
        cudaError_t e_ = (x);                                                                           \
        if (e_ != cudaSuccess) {                                                                        \
            char m_[256];                                                                               \
            snprintf(m_, sizeof(m_), "%s: %s", #x, cudaGetErrorString(e_));                             \
            return t2sx_set_error(e_ == cudaErrorMemoryAllocation ? T2SX_ERR_OOM : T2SX_ERR_CUDA, m_);  \
        }                                                                                               \
    } while (0)

// The body of a C entry point: host allocation failures come back as a status.
template <typename F>
int t2sx_guarded(const char* who, F&& body) {
    try {
        return body();
    } catch (const std::exception& e) {
        char m[256];
        snprintf(m, sizeof(m), "%s: %s", who, e.what());
        return t2sx_set_error(T2SX_ERR_OOM, m);
    }
}
