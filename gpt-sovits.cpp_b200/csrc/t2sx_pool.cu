// Pages of a K/V cache that sequences share: fork, copy, release and compact.
//
// A sequence is a list of page ids kept on the host; a page counts its users.  Forking shares full
// pages by counting and copies the filled positions of the last, partial one, so pages with several
// users are never written.  Data moves only in k_move_pages: a fork's partial pages, a copy's pages,
// a compaction's pages; the sources of one launch are never among its destinations (a fork or copy
// whose source is also one of its destinations is refused, a compaction moves pages across a line).
#include "t2sx_pool.cuh"

#include <algorithm>
#include <cstring>
#include <memory>

using namespace t2sx;

namespace {

// Moves per launch: the list travels as a kernel parameter (no staging buffer, nothing to order).
// Two sizes of it: the host's time of a launch grows with its parameters.
constexpr int kFewMoves = 32, kMovesPerLaunch = 512;
constexpr int kFan = 8;            // destinations that one read of a page serves
constexpr int kHeadsPerCta = 8;    // one per warp
struct Fan {                       // moves of one source and fill
    int32_t src;
    uint16_t first, n, fill, pad;
};
template <int N>
struct MoveList {
    int32_t dst[N];
    Fan fan[N];
};

// One CTA per (fan, layer, K or V, 8 heads); a head's filled positions are contiguous in its page.  Bound by
// the bytes written: a fork's partial page is read once for up to eight copies.  Calls one after another, 512 copies of 32 pages of 24 layers
// (16 heads of 32 dims) take 138 us, 5.5 TB/s; with a read through the L2 cache for each copy they took 306.  Rewriting
// 32 of 64 sequences and compacting, 3.65 GB in and out, takes 557 us (6.5 TB/s).
template <int N>
__global__ void __launch_bounds__(32 * kHeadsPerCta)
k_move_pages(const __grid_constant__ MoveList<N> list, uint4* __restrict__ k, uint4* __restrict__ v, int n_pages, int n_kv,
             int row_vec) {
    const Fan f = list.fan[blockIdx.x];
    const int lane = threadIdx.x & 31, h = (blockIdx.z >> 1) * kHeadsPerCta + (threadIdx.x >> 5);
    if (h >= n_kv) return;
    uint4* base = (blockIdx.z & 1) ? v : k;
    const size_t head_vec = (size_t)kPoolPage * row_vec, page_vec = head_vec * n_kv;
    base += (size_t)blockIdx.y * n_pages * page_vec + h * head_vec;
    const uint4* s = base + f.src * page_vec;
    const int run = f.fill * row_vec;   // 16-byte words of a head
    for (int j = lane; j < run; j += 128) {
        uint4 w[4];
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (j + 32 * u < run) w[u] = s[j + 32 * u];
        for (int i = 0; i < f.n; ++i) {
            uint4* d = base + list.dst[f.first + i] * page_vec;
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (j + 32 * u < run) d[j + 32 * u] = w[u];
        }
    }
}

template <int N>
void launch_list(t2sx_pool* p, const PageMove* moves, int n, cudaStream_t st) {
    MoveList<N> list;
    int fans = 0;
    for (int i = 0; i < n; ++i) {
        const PageMove& m = moves[i];
        list.dst[i] = m.dst;
        if (fans && list.fan[fans - 1].src == m.src && list.fan[fans - 1].n < kFan) ++list.fan[fans - 1].n;
        else list.fan[fans++] = Fan{m.src, (uint16_t)i, 1, (uint16_t)m.fill, 0};
    }
    k_move_pages<N><<<dim3(fans, p->n_layers, 2 * ((p->n_kv + kHeadsPerCta - 1) / kHeadsPerCta)), 32 * kHeadsPerCta, 0, st>>>(
        list, reinterpret_cast<uint4*>(p->k), reinterpret_cast<uint4*>(p->v), p->n_pages, p->n_kv, p->dim * 2 / 16);
}

int launch_moves(t2sx_pool* p, const std::vector<PageMove>& moves, cudaStream_t st) {
    if (moves.empty()) return T2SX_OK;
    DeviceGuard dg;
    POOL_CK(dg.set(p->device));
    POOL_CK(p->begin(st));
    for (size_t at = 0; at < moves.size(); at += kMovesPerLaunch) {
        const int n = (int)std::min<size_t>(kMovesPerLaunch, moves.size() - at);
        if (n <= kFewMoves) launch_list<kFewMoves>(p, moves.data() + at, n, st);
        else launch_list<kMovesPerLaunch>(p, moves.data() + at, n, st);
        POOL_CK(cudaGetLastError());
        p->end(st);
    }
    return T2SX_OK;
}

int bad(const char* m) { return t2sx_set_error(T2SX_ERR_INVALID, m); }

// Ids in range and distinct.  Leaves `mark` clear.
bool distinct(t2sx_pool* p, int32_t n, const int32_t* seqs) {
    bool ok = true;
    int32_t i = 0;
    for (; i < n && ok; ++i) {
        if (seqs[i] < 0 || seqs[i] >= p->max_seqs || p->mark[seqs[i]]) { ok = false; break; }
        p->mark[seqs[i]] = 1;
    }
    for (int32_t j = 0; j < i; ++j) p->mark[seqs[j]] = 0;
    return ok;
}

void clear(t2sx_pool* p, int32_t seq) {
    for (int32_t page : p->table[seq]) p->drop(page);
    p->table[seq].clear();
    p->len[seq] = 0;
}

// fork (share: full pages are shared) and copy
int derive(t2sx_pool* p, int32_t n, const int32_t* srcs, const int32_t* dsts, cudaStream_t st, bool share, const char* who) {
    if (!p || p->closed || n < 0 || (n > 0 && (!srcs || !dsts))) return bad("pool fork/copy: bad arguments");
    return t2sx_guarded(who, [&]() -> int {
        for (int32_t i = 0; i < n; ++i)
            if (srcs[i] < 0 || srcs[i] >= p->max_seqs) return bad("pool fork/copy: source id out of range");
        if (!distinct(p, n, dsts)) return bad("pool fork/copy: destination ids out of range or given twice");
        int64_t need = 0;
        for (int32_t i = 0; i < n; ++i) {
            if (p->len[dsts[i]]) return t2sx_set_error(T2SX_ERR_STATE, "pool fork/copy: a destination is not empty");
            const int64_t len = p->len[srcs[i]];
            need += share ? (len % kPoolPage != 0) : pages_of(len);
        }
        // a source that this call fills would be copied while it is written, and its pages are not in `need`
        bool both = false;
        for (int32_t i = 0; i < n; ++i) p->mark[dsts[i]] = 1;
        for (int32_t i = 0; i < n; ++i) both |= p->mark[srcs[i]] != 0;
        for (int32_t i = 0; i < n; ++i) p->mark[dsts[i]] = 0;
        if (both) return bad("pool fork/copy: a source is also a destination of the call");
        if (need > p->n_free) return t2sx_set_error(T2SX_ERR_OOM, "pool fork/copy: not enough free pages");
        // everything that can fail on the host is allocated before the state changes
        p->moves.clear();
        p->moves.reserve((size_t)need);
        for (int32_t i = 0; i < n; ++i) p->table[dsts[i]].reserve(p->table[srcs[i]].size());
        p->shares += share;
        for (int32_t i = 0; i < n; ++i) {
            const int64_t len = p->len[srcs[i]];
            const std::vector<int32_t>& from = p->table[srcs[i]];
            std::vector<int32_t>& to = p->table[dsts[i]];
            const int32_t full = share ? (int32_t)(len / kPoolPage) : 0;
            for (int32_t j = 0; j < full; ++j) ++p->users[from[j]];
            to.assign(from.begin(), from.begin() + full);
            for (int32_t j = full; j < pages_of(len); ++j) {
                const int32_t page = p->take();
                to.push_back(page);
                p->moves.push_back(PageMove{from[j], page, (int)std::min<int64_t>(kPoolPage, len - (int64_t)j * kPoolPage)});
            }
            p->len[dsts[i]] = len;
        }
        const int rc = launch_moves(p, p->moves, st);
        if (rc != T2SX_OK)   // what was copied by then stands in pages that are free again
            for (int32_t i = 0; i < n; ++i) clear(p, dsts[i]);
        return rc;
    });
}

}  // namespace

void t2sx_pool_release_object(t2sx_pool* p) {
    DeviceGuard dg;
    dg.set(p->device);
    p->settle();
    if (p->done) cudaEventDestroy(p->done);
    delete p;
}

extern "C" int t2sx_pool_create(int32_t device, int32_t type, int32_t n_layers, int32_t n_pages, int32_t n_kv_heads,
                                int32_t head_dim, int32_t max_seqs, void* k_dev, void* v_dev, t2sx_pool** out) {
    if (!out) return bad("t2sx_pool_create: null out");
    *out = nullptr;
    if (!k_dev || !v_dev || n_layers <= 0 || n_pages <= 0 || n_kv_heads <= 0 || max_seqs <= 0)
        return bad("t2sx_pool_create: null storage or a size that is not positive");
    if (type != T2SX_TYPE_F16 && type != T2SX_TYPE_BF16) return bad("t2sx_pool_create: the type must be f16 or bf16");
    if (head_dim != 32 && head_dim != 64 && head_dim != 128) return bad("t2sx_pool_create: head_dim must be 32, 64 or 128");
    if (n_pages > kPoolMaxPages || n_layers > 65535 || n_kv_heads > 65535 || (int64_t)n_layers * n_pages > INT32_MAX)
        return bad("t2sx_pool_create: too many pages, layers or heads");
    if (((uintptr_t)k_dev | (uintptr_t)v_dev) & 15) return bad("t2sx_pool_create: storage must be 16-byte aligned");
    return t2sx_guarded("t2sx_pool_create", [&]() -> int {
        DeviceGuard dg;
        POOL_CK(dg.set(device));
        auto drop = [](t2sx_pool* q) { t2sx_pool_release_object(q); };
        std::unique_ptr<t2sx_pool, decltype(drop)> p(new t2sx_pool(), drop);
        p->device = device; p->type = type; p->n_layers = n_layers; p->n_pages = n_pages; p->n_kv = n_kv_heads;
        p->dim = head_dim; p->max_seqs = max_seqs;
        p->k = (uint16_t*)k_dev; p->v = (uint16_t*)v_dev;
        p->table.resize(max_seqs);
        p->len.assign(max_seqs, 0);
        p->mark.assign(max_seqs, 0);
        p->users.assign(n_pages, 0);
        p->free_bits.assign(((size_t)n_pages + 63) / 64, ~(uint64_t)0);
        if (n_pages % 64) p->free_bits.back() = ((uint64_t)1 << (n_pages % 64)) - 1;
        p->n_free = n_pages;
        POOL_CK(cudaEventCreateWithFlags(&p->done, cudaEventDisableTiming));
        *out = p.release();
        return T2SX_OK;
    });
}

extern "C" void t2sx_pool_free(t2sx_pool* p) {
    if (!p || p->closed) return;
    p->closed = true;
    if (p->n_plans == 0) return t2sx_pool_release_object(p);
    DeviceGuard dg;   // the object stays for its plans, the caller's storage need not
    if (dg.set(p->device) == cudaSuccess) p->settle();
}

extern "C" int t2sx_pool_available(t2sx_pool* p, int32_t* n_pages) {
    if (!p || p->closed || !n_pages) return bad("t2sx_pool_available: bad arguments");
    *n_pages = (int32_t)p->n_free;
    return T2SX_OK;
}

extern "C" int64_t t2sx_pool_length(t2sx_pool* p, int32_t seq) {
    if (!p || p->closed || seq < 0 || seq >= p->max_seqs) {
        bad("t2sx_pool_length: sequence id out of range");
        return -1;
    }
    return p->len[seq];
}

extern "C" int t2sx_pool_table(t2sx_pool* p, int32_t n, const int32_t* seqs, int32_t width, int32_t* out, int32_t* longest) {
    if (!p || p->closed || n < 0 || (n > 0 && !seqs) || (out && width < 0) || (!out && !longest))
        return bad("t2sx_pool_table: bad arguments");
    size_t most = 0;
    for (int32_t i = 0; i < n; ++i) {
        if (seqs[i] < 0 || seqs[i] >= p->max_seqs) return bad("t2sx_pool_table: sequence id out of range");
        most = std::max(most, p->table[seqs[i]].size());
    }
    if (longest) *longest = (int32_t)most;
    if (!out) return T2SX_OK;
    if (most > (size_t)width) return bad("t2sx_pool_table: a sequence has more pages than the width");
    for (int32_t i = 0; i < n; ++i) {
        const std::vector<int32_t>& t = p->table[seqs[i]];
        int32_t* row = out + (size_t)i * width;
        std::copy(t.begin(), t.end(), row);
        std::fill(row + t.size(), row + width, -1);
    }
    return T2SX_OK;
}

extern "C" int t2sx_pool_extend(t2sx_pool* p, int32_t n, const int32_t* seqs, const int64_t* counts) {
    if (!p || p->closed || n < 0 || (n > 0 && (!seqs || !counts))) return bad("t2sx_pool_extend: bad arguments");
    return t2sx_guarded("t2sx_pool_extend", [&]() -> int {
        if (!distinct(p, n, seqs)) return bad("t2sx_pool_extend: sequence ids out of range or given twice");
        int64_t need = 0;
        for (int32_t i = 0; i < n; ++i) {
            if (counts[i] < 0 || counts[i] > kPoolMaxLen || p->len[seqs[i]] + counts[i] > kPoolMaxLen)
                return bad("t2sx_pool_extend: count out of range");
            need += pages_of(p->len[seqs[i]] + counts[i]) - (int64_t)p->table[seqs[i]].size();
        }
        if (need > p->n_free) return t2sx_set_error(T2SX_ERR_OOM, "t2sx_pool_extend: not enough free pages");
        for (int32_t i = 0; i < n; ++i) {
            std::vector<int32_t>& t = p->table[seqs[i]];
            const size_t want = pages_of(p->len[seqs[i]] + counts[i]);
            if (want > t.capacity()) t.reserve(std::max(want, t.capacity() * 2));
        }
        for (int32_t i = 0; i < n; ++i) {
            std::vector<int32_t>& t = p->table[seqs[i]];
            p->len[seqs[i]] += counts[i];
            while ((int32_t)t.size() < pages_of(p->len[seqs[i]])) t.push_back(p->take());
        }
        return T2SX_OK;
    });
}

extern "C" int t2sx_pool_fork(t2sx_pool* p, int32_t n, const int32_t* srcs, const int32_t* dsts, void* stream) {
    return derive(p, n, srcs, dsts, (cudaStream_t)stream, true, "t2sx_pool_fork");
}

extern "C" int t2sx_pool_copy(t2sx_pool* p, int32_t n, const int32_t* srcs, const int32_t* dsts, void* stream) {
    return derive(p, n, srcs, dsts, (cudaStream_t)stream, false, "t2sx_pool_copy");
}

extern "C" int t2sx_pool_release(t2sx_pool* p, int32_t n, const int32_t* seqs) {
    if (!p || p->closed || n < 0 || (n > 0 && !seqs)) return bad("t2sx_pool_release: bad arguments");
    if (!distinct(p, n, seqs)) return bad("t2sx_pool_release: sequence ids out of range or given twice");
    for (int32_t i = 0; i < n; ++i) {
        if (p->len[seqs[i]]) ++p->version;
        clear(p, seqs[i]);
    }
    return T2SX_OK;
}

extern "C" int t2sx_pool_compact(t2sx_pool* p, int32_t* moved, void* stream) {
    if (!p || p->closed) return bad("t2sx_pool_compact: bad arguments");
    if (moved) *moved = 0;
    return t2sx_guarded("t2sx_pool_compact", [&]() -> int {
        const int32_t n_live = (int32_t)(p->n_pages - p->n_free);
        // the i-th used page at n_live or above -> the i-th free page below it
        std::vector<int32_t> to(p->n_pages - n_live, -1);
        size_t hole = 0;
        int32_t n_moves = 0;
        auto next_hole = [&]() {
            while (!(p->free_bits[hole >> 6] >> (hole & 63) & 1)) ++hole;
            return (int32_t)hole++;
        };
        for (int32_t page = n_live; page < p->n_pages; ++page)
            if (p->users[page]) { to[page - n_live] = next_hole(); ++n_moves; }
        if (!n_moves) return T2SX_OK;
        p->moves.clear();
        p->moves.reserve(n_moves);
        for (int32_t s = 0; s < p->max_seqs; ++s)
            for (size_t j = 0; j < p->table[s].size(); ++j) {
                const int32_t page = p->table[s][j];
                if (page < n_live) continue;
                const int32_t dst = to[page - n_live];
                if (p->users[dst]) continue;
                p->users[dst] = p->users[page];   // the first sequence that holds the page moves it
                p->moves.push_back(PageMove{page, dst, (int)std::min<int64_t>(kPoolPage, p->len[s] - (int64_t)j * kPoolPage)});
            }
        const int rc = launch_moves(p, p->moves, (cudaStream_t)stream);
        if (rc != T2SX_OK) {
            for (const PageMove& m : p->moves) p->users[m.dst] = 0;
            return rc;
        }
        for (std::vector<int32_t>& t : p->table)
            for (int32_t& page : t)
                if (page >= n_live) page = to[page - n_live];
        for (const PageMove& m : p->moves) p->users[m.src] = 0;
        std::fill(p->free_bits.begin(), p->free_bits.end(), 0);
        for (int32_t page = n_live; page < p->n_pages; ++page) p->free_bits[page >> 6] |= (uint64_t)1 << (page & 63);
        p->first_free_word = std::min<size_t>(n_live / 64, p->free_bits.size() - 1);
        ++p->version;
        if (moved) *moved = n_moves;
        return T2SX_OK;
    });
}
