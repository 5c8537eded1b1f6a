// A paged cache's pages: taken, shared, copied and given back, and the accepted path of a tree of drafts moved to where the text goes on.
//
// What the allocator knows - tables, counts, the free pages - is worked on by one workgroup: a call has at most kCacheMost sequences, and pages are dealt out and taken back
// in the order of the sequences, so that the same calls leave the same pages in the same places. A sequence a thread, the pages' entries over all threads (an entry finds its
// sequence in the prefix sums). What bounds these is the chain of trips to memory, four or five a call (4 slots of 28 layers: reserve 3.8 us, fork 5.2, release 5.6; 48 slots 7 to 9). Tokens are moved by kernels of their own,
// a workgroup a sequence, layer and side (K or V), and memory bounds them: each byte is read once and written once (64 sequences, 48 layers, 100 MB in 21.4 us: 4.7 TB/s).
#pragma once

#include "ws_common.h"
#include "ws_cycle.h"

namespace ws {

__device__ __forceinline__ uint32_t pages_for(uint32_t tokens, uint32_t shift) { return (tokens >> shift) + ((tokens & ((1u << shift) - 1u)) != 0u ? 1u : 0u); }
// the memory that every compute unit sees: counts that atomics of this launch have changed
__device__ __forceinline__ int32_t fresh(const int32_t* at) { return __hip_atomic_load(at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// The slots of a call in LDS, and whether slot i was named before. (Every thread looks at the ones before its own: 1024 of them take some 4 us, 64 a quarter of one.)
__device__ __forceinline__ bool named_before(const int32_t* names, uint32_t i) {
    bool found = false;
    for (uint32_t j = 0; j < i; ++j) found = found || names[j] == names[i];
    return found;
}
// the sequence whose entries [first[i], first[i + 1]) hold e
__device__ __forceinline__ uint32_t sequence_of(const uint64_t* first, uint32_t n, uint64_t e) {
    uint32_t lo = 0, hi = n;
    while (hi - lo > 1u) {
        const uint32_t mid = (lo + hi) >> 1;
        if (first[mid] <= e) lo = mid;
        else hi = mid;
    }
    return lo;
}

struct PagesLds {
    int32_t name[kCacheMost];
    uint32_t at[kCacheMost];        // the first page of the sequence's entries
    uint64_t first[kCacheMost + 1];  // prefix sums of entries
    uint64_t red[WS_WAVES];
};

// Takes `wanted` pages for each thread's sequence, in order, where they suffice: whether this one got them, the place of its first in the order; `total`: all that were taken.
__device__ __forceinline__ bool take_pages(uint32_t wanted, int32_t n_free, uint64_t* red, uint64_t& before, uint64_t& total) {
    uint64_t all = 0;
    before = block_excl_scan(static_cast<uint64_t>(wanted), red, &all);
    const bool served = before + wanted <= static_cast<uint64_t>(n_free);
    __syncthreads();
    total = 0;
    block_excl_scan(static_cast<uint64_t>(served ? wanted : 0u), red, &total);
    return served;
}

__device__ __forceinline__ int32_t free_count(const CacheRef& C) {
    const int32_t n = C.n_free[0];
    return n < 0 ? 0 : (static_cast<uint32_t>(n) > C.pages ? static_cast<int32_t>(C.pages) : n);
}

__global__ void __launch_bounds__(WS_BLOCK) cache_reserve_kernel(PagesArgs A) {
    __shared__ PagesLds L;
    const uint32_t t = threadIdx.x;
    const CacheRef& C = A.C;
    const int32_t n_free = free_count(C);
    const int32_t name = t < A.n ? A.slot[t] : -1, tokens = t < A.n ? A.tokens[t] : 0;
    L.name[t] = name;
    __syncthreads();
    int32_t status = kCacheOk;
    uint32_t held = 0, wanted = 0;
    if (t < A.n) {
        if (static_cast<uint32_t>(name) >= C.slots || tokens < 0 || named_before(L.name, t)) {
            status = kCacheBad;
        } else {
            held = min(static_cast<uint32_t>(max(C.held[name], 0)), C.slot_pages);
            const uint32_t need = pages_for(static_cast<uint32_t>(tokens), C.page_shift);
            if (need > C.slot_pages) status = kCacheFull;
            else wanted = need > held ? need - held : 0u;
        }
    }
    uint64_t before, total;
    const bool served = take_pages(wanted, n_free, L.red, before, total);
    if (!served && wanted) {
        status = kCacheFull;
        wanted = 0;
        before = total;
    }
    // (those not served come behind all that are: their places are the end)
    L.first[t] = min(before, total);
    L.at[t] = held;
    if (t == 0u) L.first[kCacheMost] = total;
    __syncthreads();
    for (uint64_t e = t; e < total; e += WS_BLOCK) {
        const uint32_t i = sequence_of(L.first, A.n, e);
        const int32_t page = C.free[static_cast<uint64_t>(n_free) - 1u - e];
        C.table[static_cast<uint64_t>(L.name[i]) * C.table_stride + L.at[i] + (e - L.first[i])] = page;
        if (static_cast<uint32_t>(page) < C.pages) C.refs[page] = 1;
    }
    if (t < A.n) {
        if (wanted) C.held[name] = static_cast<int32_t>(held + wanted);
        A.status[t] = status;
    }
    if (t == 0u) C.n_free[0] = n_free - static_cast<int32_t>(total);
}

__global__ void __launch_bounds__(WS_BLOCK) cache_fork_kernel(PagesArgs A) {
    __shared__ PagesLds L;
    __shared__ int32_t from[kCacheMost];
    const uint32_t t = threadIdx.x;
    const CacheRef& C = A.C;
    const int32_t n_free = free_count(C);
    const int32_t name = t < A.n ? A.slot[t] : -1, src = t < A.n ? A.src[t] : -1, tokens = t < A.n ? A.tokens[t] : 0;
    L.name[t] = name;
    from[t] = src;
    __syncthreads();
    int32_t status = kCacheOk;
    uint32_t whole = 0, part = 0;
    if (t < A.n) {
        if (static_cast<uint32_t>(name) >= C.slots || static_cast<uint32_t>(src) >= C.slots || name == src || tokens < 0 || named_before(L.name, t)) {
            status = kCacheBad;
        } else {
            whole = static_cast<uint32_t>(tokens) >> C.page_shift;
            part = (static_cast<uint32_t>(tokens) & ((1u << C.page_shift) - 1u)) != 0u ? 1u : 0u;
            if (C.held[name] != 0 || whole + part > C.slot_pages || C.held[src] < static_cast<int32_t>(whole + part)) status = kCacheBad;
        }
        if (status != kCacheOk) whole = part = 0u;
    }
    uint64_t before, total;
    if (!take_pages(part, n_free, L.red, before, total) && part) {
        status = kCacheFull;
        whole = part = 0u;
    }
    __syncthreads();
    uint64_t shared = 0;
    L.first[t] = block_excl_scan(static_cast<uint64_t>(whole), L.red, &shared);
    __syncthreads();  // (every count has been read)
    for (uint64_t e = t; e < shared; e += WS_BLOCK) {
        const uint32_t i = sequence_of(L.first, A.n, e), k = static_cast<uint32_t>(e - L.first[i]);
        const int32_t page = C.table[static_cast<uint64_t>(from[i]) * C.table_stride + k];
        C.table[static_cast<uint64_t>(L.name[i]) * C.table_stride + k] = page;
        if (static_cast<uint32_t>(page) < C.pages) atomicAdd(&C.refs[page], 1);
    }
    if (t < A.n) {
        if (part) {
            const int32_t page = C.free[static_cast<uint64_t>(n_free) - 1u - before];
            C.table[static_cast<uint64_t>(name) * C.table_stride + whole] = page;
            if (static_cast<uint32_t>(page) < C.pages) C.refs[page] = 1;
        }
        if (whole + part) C.held[name] = static_cast<int32_t>(whole + part);
        A.status[t] = status;
    }
    if (t == 0u) C.n_free[0] = n_free - static_cast<int32_t>(total);
}

// What the workgroup's atomics have done is in the memory that all of them see (one compute unit's: no cache is written back or emptied for it, which takes microseconds)
__device__ __forceinline__ void arrived() {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
}

// A page that several of the call's sequences give back goes where the first of them has it. Who is that does not depend on the order of the atomics: all take theirs off the count; where
// it is 0, it becomes the smallest number of an entry (kMark below 0), whose thread then gives the page back and makes the count 0 again.
constexpr int32_t kMark = -2147483647 - 1;
__device__ __forceinline__ bool is_mark(int32_t refs) { return refs < -1073741824; }
__global__ void __launch_bounds__(WS_BLOCK) cache_release_kernel(PagesArgs A) {
    __shared__ PagesLds L;
    const uint32_t t = threadIdx.x;
    const CacheRef& C = A.C;
    const int32_t n_free = free_count(C);
    const int32_t name = t < A.n ? A.slot[t] : -1, tokens = t < A.n ? A.tokens[t] : 0;
    L.name[t] = name;
    __syncthreads();
    int32_t status = kCacheOk;
    uint32_t kept = 0, gone = 0;
    if (t < A.n) {
        if (static_cast<uint32_t>(name) >= C.slots || tokens < 0 || named_before(L.name, t)) {
            status = kCacheBad;
        } else {
            const uint32_t held = min(static_cast<uint32_t>(max(C.held[name], 0)), C.slot_pages);
            kept = min(pages_for(static_cast<uint32_t>(tokens), C.page_shift), held);
            gone = held - kept;
        }
    }
    uint64_t total = 0;
    L.first[t] = block_excl_scan(static_cast<uint64_t>(gone), L.red, &total);
    L.at[t] = kept;
    __syncthreads();
    // From the last entry to the first, so that the first comes to lie uppermost. A thread keeps what it finds of the first round of entries, the only one but of calls that give much back.
    auto entry = [&](uint64_t e) {
        const uint32_t i = sequence_of(L.first, A.n, e);
        return C.table + static_cast<uint64_t>(L.name[i]) * C.table_stride + L.at[i] + (e - L.first[i]);
    };
    int32_t* const place0 = t < total ? entry(total - 1u - t) : nullptr;
    const int32_t page0 = place0 ? *place0 : -1;
    auto page_of = [&](uint64_t at) { return at == 0u ? page0 : (at + t < total ? *entry(total - 1u - at - t) : -1); };
    for (uint64_t at = 0; at < total; at += WS_BLOCK) {
        const int32_t page = page_of(at);
        if (static_cast<uint32_t>(page) < C.pages) atomicSub(&C.refs[page], 1);
    }
    arrived();
    for (uint64_t at = 0; at < total; at += WS_BLOCK) {
        const int32_t page = page_of(at);
        if (static_cast<uint32_t>(page) >= C.pages) continue;
        const int32_t left = fresh(&C.refs[page]);
        if (left == 0 || is_mark(left)) atomicMin(&C.refs[page], kMark + static_cast<int32_t>(total - 1u - at - t));
    }
    arrived();
    uint64_t put = 0;
    for (uint64_t at = 0; at < total; at += WS_BLOCK) {
        const int32_t page = page_of(at);
        const bool mine = static_cast<uint32_t>(page) < C.pages && fresh(&C.refs[page]) == kMark + static_cast<int32_t>(total - 1u - at - t);
        uint64_t all = 0;
        const uint64_t rank = block_excl_scan(static_cast<uint64_t>(mine ? 1u : 0u), L.red, &all);
        if (mine) {
            const uint64_t to = static_cast<uint64_t>(n_free) + put + rank;
            if (to < C.pages) C.free[to] = page;
            C.refs[page] = 0;
        }
        if (at + t < total) *(at == 0u ? place0 : entry(total - 1u - at - t)) = -1;
        put += all;
        __syncthreads();
    }
    if (t < A.n) {
        if (gone) C.held[name] = static_cast<int32_t>(kept);
        if (A.status) A.status[t] = status;
    }
    if (t == 0u) C.n_free[0] = static_cast<int32_t>(min(static_cast<uint64_t>(n_free) + put, static_cast<uint64_t>(C.pages)));
}

// ---- tokens: a workgroup a sequence (x), layer (y) and side (z)
constexpr uint32_t kMoveThreads = 256u;
__device__ __forceinline__ uint4 load16(const unsigned char* at) { return *reinterpret_cast<const uint4*>(at); }
__device__ __forceinline__ void store16(unsigned char* at, const uint4& v) { *reinterpret_cast<uint4*>(at) = v; }

// the filled part of the last page of a fork's source, which cache_fork_kernel has put the page for into the destination's table
__global__ void __launch_bounds__(kMoveThreads) cache_copy_kernel(PagesArgs A) {
    const CacheRef& C = A.C;
    const uint32_t i = blockIdx.x;
    const uint32_t tokens = static_cast<uint32_t>(A.tokens[i]), part = tokens & ((1u << C.page_shift) - 1u);
    if (A.status[i] != kCacheOk || part == 0u) return;
    const uint64_t last = tokens >> C.page_shift;
    const int32_t from = C.table[static_cast<uint64_t>(A.src[i]) * C.table_stride + last], to = C.table[static_cast<uint64_t>(A.slot[i]) * C.table_stride + last];
    if (static_cast<uint32_t>(from) >= C.pages || static_cast<uint32_t>(to) >= C.pages) return;
    const CacheSide& S = C.side[blockIdx.z];
    unsigned char* at = S.at + blockIdx.y * S.layer;
    const unsigned char* a = at + static_cast<uint64_t>(from) * S.page;
    unsigned char* b = at + static_cast<uint64_t>(to) * S.page;
    const uint32_t per_head = C.head_bytes / 16u, per_token = per_head * C.kv_heads, all = per_token * part;
    auto offset = [&](uint32_t v) {
        const uint32_t token = v / per_token, rest = v - token * per_token, head = rest / per_head;
        return token * S.token + head * S.head + (rest - head * per_head) * 16u;
    };
    constexpr uint32_t kU = 4u;
    for (uint32_t v = threadIdx.x; v < all; v += kU * kMoveThreads) {
        uint4 x[kU];
        uint64_t o[kU];
#pragma unroll
        for (uint32_t u = 0; u < kU; ++u) {
            o[u] = offset(min(v + u * kMoveThreads, all - 1u));
            x[u] = load16(a + o[u]);
        }
#pragma unroll
        for (uint32_t u = 0; u < kU; ++u)
            if (v + u * kMoveThreads < all) store16(b + o[u], x[u]);
    }
}

// Position length + 1 + i from length + path[i]. path[i] > i, and no later copy reads what an earlier one has written (it would have to lie at or before it), so a thread loads several tokens
// before it stores the first.
__global__ void __launch_bounds__(kMoveThreads) cache_keep_kernel(KeepArgs A) {
    __shared__ uint64_t from[kTreeNodes], to[kTreeNodes];
    __shared__ uint32_t n_moves;
    const CacheRef& C = A.C;
    const uint32_t s = blockIdx.x, t = threadIdx.x;
    const CacheSide& S = C.side[blockIdx.z];
    if (t < 64u) {
        const int32_t n = A.n_accepted[s];
        const uint32_t slot = A.slot ? A.slot[s] : s, length = A.length[s];
        const uint32_t accepted = min(min(static_cast<uint32_t>(max(n, 0)), A.depth), kTreeNodes - 1u);
        const int32_t node = t < accepted ? A.path[static_cast<uint64_t>(s) * A.depth + t] : -1;
        const int32_t before = __shfl_up(node, 1);  // (by all lanes: one that is not there gives nothing)
        const bool fine = t < accepted && node > (t == 0u ? 0 : before) && node < static_cast<int32_t>(kTreeNodes);
        const uint64_t stop = __ballot(!fine);
        const uint32_t good = stop ? static_cast<uint32_t>(__ffsll(static_cast<long long>(stop)) - 1) : 64u;
        // (moves of a token to its own place are left out)
        bool moves = t < good && slot < C.slots && node != static_cast<int32_t>(t + 1u);
        uint64_t a = 0, b = 0;
        if (moves) {
            const uint64_t p = static_cast<uint64_t>(length) + static_cast<uint32_t>(node), q = static_cast<uint64_t>(length) + 1u + t;
            moves = (p >> C.page_shift) < C.slot_pages;  // (q is not behind p)
            if (moves) {
                const int32_t* row = C.table + static_cast<uint64_t>(slot) * C.table_stride;
                const int32_t pa = row[p >> C.page_shift], pb = row[q >> C.page_shift];
                moves = static_cast<uint32_t>(pa) < C.pages && static_cast<uint32_t>(pb) < C.pages;
                const uint64_t in = (uint64_t{1} << C.page_shift) - 1u;
                a = static_cast<uint64_t>(static_cast<uint32_t>(pa)) * S.page + (p & in) * S.token;
                b = static_cast<uint64_t>(static_cast<uint32_t>(pb)) * S.page + (q & in) * S.token;
            }
        }
        const uint64_t all = __ballot(moves);
        if (moves) {
            const uint32_t at = static_cast<uint32_t>(__popcll(all & ((uint64_t{1} << t) - 1u)));
            from[at] = a;
            to[at] = b;
        }
        if (t == 0u) n_moves = static_cast<uint32_t>(__popcll(all));
    }
    __syncthreads();
    const uint32_t n = n_moves;
    if (n == 0u) return;
    const uint32_t per_head = C.head_bytes / 16u, per_token = per_head * C.kv_heads;
    unsigned char* at = S.at + blockIdx.y * S.layer;
    constexpr uint32_t kU = 8u;
    for (uint32_t v = t; v < per_token; v += kMoveThreads) {
        const uint32_t head = v / per_head;
        unsigned char* mine = at + head * S.head + (v - head * per_head) * 16u;
        for (uint32_t i = 0; i < n; i += kU) {
            uint4 x[kU];
#pragma unroll
            for (uint32_t u = 0; u < kU; ++u) x[u] = load16(mine + from[min(i + u, n - 1u)]);
#pragma unroll
            for (uint32_t u = 0; u < kU; ++u)
                if (i + u < n) store16(mine + to[i + u], x[u]);
        }
    }
}

}  // namespace ws
