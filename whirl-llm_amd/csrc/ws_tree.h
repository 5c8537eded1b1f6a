// A cycle's drafts as trees: what a row sees and where it stands (tree_stage_kernel), and the drafts' verification against the target's logits (tree_rows_kernel, tree_draw_kernel).
//
// Verification. With w_v = exp((x_v - m) t) over the allowed tokens of a node's row, S = sum w_v and P = w / S, a child with token y is accepted if u Q(y) < P(y); after
// a rejection P becomes max(P - Q, 0) divided by its sum Z. Q is 0 but at 32 ids at most (or at one, where the child is a guess), so that outside of them P stays w times one number c:
// what is carried along is c and the P and Q of those ids, a lane each, and the mass outside of them, 1 - sum P at first. No pass over the row is made for a rejection.
//
// Which child a node passes the walk on to, if any, does not depend on how the walk came to it. So tree_rows_kernel decides all nodes with children at once, one pass over a row, its workgroups meeting
// without waiting for each other; nodes are numbered level by level as far as the grid can, and one whose parent has decided against it by then is not read. (A kernel that walked, row after row, waited for memory
// and for its parts at each: 64 trees of 16 nodes 83 us, 256 of 25 237 us, five rows 40 us.) tree_draw_kernel then goes down the tree along what was decided and draws from the row where
// that ends, which its workgroups hold in registers.
// What bounds them is latency (the same three: 30 + 26, 96 + 40, 8 + 13 us): trips to memory one after the other - offsets, decisions, the row, the q entry and its ids' logits, the parts' words -, and workgroups that
// only find that their node is not needed, 2 ns each; vector units are 40 to 65 % busy, memory is read at 2 to 3 TB/s. (Every workgroup of a sequence going where the walk may come to next, reading
// as it goes, instead of one a node: 37 and 131 us for then 35 and 101.)
//
// Accuracy. The comparisons u Q < P are made in 64 bits, S is added up from powers of 32 bits (1e-8 of S where many tokens count): of ten million drafts one may be judged otherwise than by an
// exact sum. The token behind the walk is looked for among some 100 000 steps of a cumulative sum, whose places would move by 1e-8 of the sum, a hundredth of a step where tokens are
// unlikely: there the powers are taken in 64 bits (to 1e-11), and S, Z and the P of the listed ids once more from them.
#pragma once

#include "ws_cycle.h"
#include "ws_loss.h"

namespace ws {

// the nodes of sequence s: the first row, how many
__device__ __forceinline__ uint32_t tree_rows(const uint32_t* seq_off, uint32_t s, uint32_t rows, uint32_t& n) {
    const uint32_t a = min(seq_off[s], rows), b = min(seq_off[s + 1u], rows);
    n = b > a ? min(b - a, kTreeNodes) : 0u;
    return a;
}

// A wave a sequence, a lane a node: ancestors by doubling (after k steps a node knows 2^k of them), six steps for 64 nodes.
__global__ void __launch_bounds__(64) tree_stage_kernel(TreeStageArgs A) {
    const uint32_t s = blockIdx.x, lane = threadIdx.x;
    uint32_t n;
    const uint32_t first = tree_rows(A.seq_off, s, A.rows, n);
    const uint32_t len = A.len ? A.len[A.slot ? A.slot[s] : s] : 0u;
    if (lane == 0u && A.length) A.length[s] = len;
    int32_t up = -1;
    if (lane > 0u && lane < n) up = A.parent ? A.parent[first + lane] : static_cast<int32_t>(lane) - 1;
    if (up >= static_cast<int32_t>(lane)) up = -1;
    if (up < 0) up = -1;
    uint32_t lo = lane < 32u ? 1u << lane : 0u, hi = lane < 32u ? 0u : 1u << (lane - 32u);
#pragma unroll
    for (int k = 0; k < 6; ++k) {
        const int from = max(up, 0);
        const uint32_t plo = __shfl(lo, from), phi = __shfl(hi, from);
        const int32_t next = __shfl(up, from);
        if (up >= 0) {
            lo |= plo;
            hi |= phi;
            up = next;
        }
    }
    // (a node whose ancestors do not end at the root is never reached)
    if (!(lo & 1u)) {
        lo = lane < 32u ? 1u << lane : 0u;
        hi = lane < 32u ? 0u : 1u << (lane - 32u);
    }
    if (lane >= n) return;
    if (A.mask) A.mask[first + lane] = (static_cast<uint64_t>(hi) << 32) | lo;
    if (A.position) A.position[first + lane] = static_cast<int32_t>(len + __popc(lo) + __popc(hi) - 1u);
}

// 2^z for z <= 0 to 1e-11: z = k + f, |f| <= 1/2, and of 2^f = e^(f ln 2) the first ten terms of its series (the next is 0.35^10 / 10! = 7e-12). What lies below 2^-1075, -inf too, is 0 (ldexp; k stays in what it takes as z is cut at -2885). Not
// for NaN, which is told apart where it is looked for. (k by a sum whose last bit is worth one: of rounding and conversion an instruction takes several times as long.)
__device__ __forceinline__ double power64(double z) {
    z = fmax(z, -2885.0);
    const double k = z + 0x1.8p52, f = z - (k - 0x1.8p52);
    double p = 0x1.b5253d395e7c4p-24;
    p = fma(p, f, 0x1.62c0223a5c824p-20);
    p = fma(p, f, 0x1.ffcbfc588b0c7p-17);
    p = fma(p, f, 0x1.430912f86c787p-13);
    p = fma(p, f, 0x1.5d87fe78a6731p-10);
    p = fma(p, f, 0x1.3b2ab6fba4e77p-7);
    p = fma(p, f, 0x1.c6b08d704a0c0p-5);
    p = fma(p, f, 0x1.ebfbdff82c58fp-3);
    p = fma(p, f, 0x1.62e42fefa39efp-1);
    p = fma(p, f, 0x1.0000000000000p+0);
    return ldexp(p, __double2loint(k));
}
// exponents of base two: a row's factor
__device__ __forceinline__ double tree_factor(float inv_t) { return static_cast<double>(inv_t) * 1.4426950408889634074; }

// part `part` of a row: vectors [j0, j1) of 16 bytes, numbered from the row's first token, wherever that lies; a wave's are neighbours, so that sums go in id order
template <int DT, bool MASK, int T, int NV>
struct TreeShare {
    static constexpr uint32_t kPer = Elem<DT>::kPer;
    uint32_t j0, j1, rounds;
    uint4 q[NV];
    __device__ __forceinline__ void place(uint32_t V, uint32_t part, uint32_t per) {
        const uint32_t all = (V + kPer - 1u) / kPer;
        j0 = min(part * per, all);
        j1 = min(j0 + per, all);
        rounds = (per + T - 1u) / T;
    }
    __device__ __forceinline__ uint32_t vector(uint32_t u) const { return j0 + wave_id() * 64u * rounds + u * 64u + lane_id(); }
    // its logits, -inf where there are none or they are not allowed
    __device__ __forceinline__ void load(const unsigned char* base, const uint32_t* allow, uint32_t V) {
        constexpr uint32_t none = Elem<DT>::kNone;
        uint32_t bits[NV];
        const uint32_t whole = V / kPer;  // vectors that lie inside the row
        if (whole != 0u) {
#pragma unroll
            for (int u = 0; u < NV; ++u) {
                if (static_cast<uint32_t>(u) < rounds) {  // (uniform)
                    const uint32_t j = min(vector(u), whole - 1u);
                    if constexpr (MASK) bits[u] = static_cast<uint32_t>(reinterpret_cast<const unsigned char*>(allow)[j * kPer / 8u]) >> (j * kPer % 8u);
                    q[u] = load_loose(base + static_cast<size_t>(j) * 16u);
                }
            }
        }
#pragma unroll
        for (int u = 0; u < NV; ++u) {
            const uint32_t j = vector(u);
            const bool mine = static_cast<uint32_t>(u) < rounds && j < j1;
            if (mine && j < whole) {
                if constexpr (MASK) q[u] = only_allowed<DT>(q[u], bits[u]);
            } else {
                q[u] = make_uint4(none, none, none, none);
                if (mine) {  // the row's last, partly filled vector
                    uint32_t w[4] = {none, none, none, none};
                    for (uint32_t e = 0; e < V - whole * kPer; ++e) {
                        const uint32_t i = whole * kPer + e;
                        if (MASK && !allowed(allow, i)) continue;
                        const uint32_t b = DT == 0 ? reinterpret_cast<const uint32_t*>(base)[i] : reinterpret_cast<const uint16_t*>(base)[i];
#pragma unroll
                        for (uint32_t k = 0; k < 4u; ++k) {
                            if (DT == 0) {
                                if (k == e) w[k] = b;
                            } else if (k == e / 2u) {
                                w[k] = e % 2u ? (w[k] & 0xffffu) | (b << 16) : (w[k] & 0xffff0000u) | b;
                            }
                        }
                    }
                    q[u] = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
        }
    }
    // the largest of its logits; whether one is NaN or they have no largest
    __device__ __forceinline__ float largest(bool& odd) const {
        float m = -FLT_MAX;
#pragma unroll
        for (int u = 0; u < NV; ++u) {
            if (static_cast<uint32_t>(u) < rounds) {
                float x[kPer];
                unpack<DT>(q[u], x);
#pragma unroll
                for (uint32_t e = 0; e < kPer; e += 2u) {
                    m = max3(m, x[e], x[e + 1u]);
                    odd = odd || __builtin_isunordered(x[e], x[e + 1u]);
                }
            }
        }
        odd = odd || m == INFINITY;
        return m;
    }
};

// What a walk holds at a node, by the lanes of a wave: lane l an id that Q or the guesses name.
struct TreeNode {
    bool listed, guess;
    uint32_t id;
    float x;        // its logit, -inf where not allowed
    double drawn, Q, P;  // what Q gives it at first, and now; its probability
    double out, c;       // that of all that is not listed as the node begins, and what it has been multiplied by
};
// the node's probabilities, S and what of it lies outside the listed ids known (out_known < 0: not)
__device__ __forceinline__ void tree_begin(TreeNode& N, float m, double factor, double S, double out_known) {
    N.P = N.listed ? power64((static_cast<double>(N.x) - static_cast<double>(m)) * factor) / S : 0.0;
    N.Q = N.drawn;
    N.c = 1.0;
    N.out = out_known >= 0.0 ? out_known / S : fmax(1.0 - wave_sum(N.P), 0.0);
}
// the token y of a child: its place among the listed (64: none)
__device__ __forceinline__ uint32_t tree_find(const TreeNode& N, uint32_t y) {
    const uint64_t at = __ballot(N.listed && N.id == y);
    return at ? static_cast<uint32_t>(__ffsll(static_cast<long long>(at)) - 1) : 64u;
}
__device__ __forceinline__ void tree_reject(TreeNode& N, uint32_t place) {
    const bool here = lane_id() == static_cast<int>(place);
    const double rest = N.guess ? (here ? 0.0 : N.P) : fmax(N.P - N.Q, 0.0);  // (NaN: 0, and the sum of the others says it)
    const double Z = N.c * N.out + wave_sum(rest);
    if (Z > 0.0) {
        N.P = rest / Z;
        N.c /= Z;
    }
    if (!N.guess) {
        if (here) N.Q = 0.0;
        const double left = wave_sum(N.Q);
        if (left > 0.0) N.Q /= left;
    }
}

// The trees' nodes, a lane each.
struct TreeLane {
    int32_t above;   // its parent, -1: none
    uint32_t token;
    double u;
};
__device__ __forceinline__ TreeLane tree_lane(const TreeVerifyArgs& A, uint32_t first, uint32_t n) {
    TreeLane L{-1, 0xffffffffu, 0.0};
    const uint32_t t = lane_id();
    if (t < n) {
        L.above = A.parent ? A.parent[first + t] : static_cast<int32_t>(t) - 1;
        if (t == 0u || L.above >= static_cast<int32_t>(t)) L.above = -1;
        L.token = static_cast<uint32_t>(A.R.ids[first + t]);
        L.u = A.u_accept[first + t];
    }
    return L;
}
// The children of a node and what the distribution they were drawn from names (its entry at word off of q), for a wave; false where the entry lies outside q.
template <int DT, bool MASK>
__device__ __forceinline__ bool tree_drafts(const TreeVerifyArgs& A, int32_t off, const unsigned char* base, const uint32_t* allow, const TreeLane& L, uint64_t kids, uint32_t* seen, TreeNode& N, float& x_child) {
    const uint32_t t = lane_id(), V = A.R.vocab;
    auto logit = [&](uint32_t id) { return id < V && (!MASK || allowed(allow, id)) ? load_logit<DT>(base, id) : -INFINITY; };
    N.guess = off < 0;
    N.drawn = 0.0;
    x_child = kids >> t & 1u ? logit(L.token) : -INFINITY;
    if (N.guess) {
        N.listed = kids >> t & 1u;
        N.id = L.token;
        N.x = x_child;
    } else if (kids == 0ull) {
        N.listed = false;
    } else {
        if (static_cast<uint64_t>(off) + kTreeEntryWords > A.q_words) return false;
        const int32_t* entry = A.q + off;
        const int32_t count = entry[0], id = entry[1u + min(t, kTreeListed - 1u)];  // (all at once: one trip to memory)
        const float q = __int_as_float(entry[33u + min(t, kTreeListed - 1u)]);
        N.listed = t < kTreeListed && static_cast<int32_t>(t) < count;
        N.id = static_cast<uint32_t>(id);
        N.drawn = N.listed ? static_cast<double>(q) : 0.0;
        N.x = N.listed ? logit(N.id) : -INFINITY;
    }
    // An id that is named before counts there. Whether there is one: a bit an id, in a table of 8192, is there when it comes (of 32 ids that differ once in 16 times: then they are gone through)
    const uint4 none = make_uint4(0u, 0u, 0u, 0u);
    reinterpret_cast<uint4*>(seen)[t] = none;
    __builtin_amdgcn_wave_barrier();  // (one wave: its LDS stores are done before its atomics)
    const uint32_t hash = N.id * 2654435761u >> 19;
    const bool again = N.listed && (atomicOr(&seen[hash >> 5], 1u << (hash & 31u)) >> (hash & 31u) & 1u);
    if (__ballot(again) == 0ull) return true;
    for (uint64_t left = __ballot(N.listed); left; left &= left - 1ull) {
        const uint32_t l = static_cast<uint32_t>(__ffsll(static_cast<long long>(left)) - 1), id = lane_value(N.id, l);
        const uint64_t same = __ballot(N.listed && N.id == id) & (~0ull << l);
        if ((same & (same - 1ull)) == 0ull) continue;
        const double sum = wave_sum((same >> t & 1u) ? N.drawn : 0.0);
        if (t == l) N.drawn = sum;
        else if (same >> t & 1u) N.listed = false;
        left &= ~same | (1ull << l);
    }
    return true;
}

// The words of a launch (ws_loss.h) have a tag that no other launch has, but the replays of a captured one: so no launch leaves its words behind where its next replay looks for them. The draw's
// are taken apart by the next rows' kernel, when no draw runs; the rows' and the decisions by the draw's workgroups, when all of a sequence's have read them. All of them, a part's maximum and its
// sum: who looks between the two may find the one from now and the other, were it still whole, from the replay before.

// ---- what each node decides: the child that it passes the walk on to (with the log-probability of that one's token), or none; or that the walk does not come to it, or that its q entry is none
constexpr uint32_t kDecNone = 64u, kDecNever = 65u, kDecBad = 66u;
constexpr uint32_t kRowThreads = 256u, kParentLooks = 64u;  // (a look: a microsecond)
__device__ __forceinline__ unsigned long long* tree_decision(const TreeVerifyArgs& A, uint32_t row) { return A.decided + 2u * static_cast<size_t>(row); }

// (Three workgroups a unit with a mask, whose loads take registers: four spill, 101 us for 125. Without, four: 35 us for 32.)
template <int DT, bool MASK>
__global__ void __launch_bounds__(kRowThreads, MASK ? 3 : 4) tree_rows_kernel(TreeVerifyArgs A) {
    constexpr uint32_t T = kRowThreads, kPer = Elem<DT>::kPer, kU = 4u;  // vectors of a thread on their way together
    __shared__ float red_m[T / 64];
    __shared__ double red_s[T / 64], red_t[T / 64];
    __shared__ uint32_t s_never;
    __shared__ __attribute__((aligned(16))) uint32_t s_seen[256];
    const uint32_t y = grid_row(), level = y / A.n_seq, s = y - level * A.n_seq, part = blockIdx.x, t = threadIdx.x, V = A.R.vocab;
    const unsigned long long tag = A.tag;
    if (level >= A.levels) return;
    if (level == 0u && part == 0u && A.parts > 1u && t < 2u * A.parts) {  // (128 at most) a part's maximum, a part's sum
        const uint32_t word = t < A.parts ? 0u : 1u;
        break_word(A.meet + (static_cast<size_t>(s) * kTreeWords + 2u * word) * A.parts + (t - word * A.parts), A.parts);
    }
    uint32_t n;
    const uint32_t first = tree_rows(A.seq_off, s, A.R.rows, n);
    if (level >= n) return;
    const TreeLane L = tree_lane(A, first, n);
    for (uint32_t node = level; node < n; node += A.levels) {  // (uniform; one, but of sequences with more nodes than the others)
        const uint32_t row = first + node;
        const unsigned char* base = A.R.logits + row * A.R.row_bytes;
        const uint32_t* allow = MASK ? A.R.allow + row * A.R.allow_stride : nullptr;
        const RowSpan<DT> span(base, V);
        const Share<DT, MASK, T> share(base, allow, span, V, part, A.row_per);
        const uint32_t j0 = share.j0, j1 = share.any() ? share.j1 : share.j0;
        // whether anybody needs the node's decision: it has children, a parent, and that one has not decided against it
        uint64_t kids = 0;
        auto needed = [&]() {
            kids = __ballot(L.above == static_cast<int32_t>(node));
            return kids != 0ull && (node == 0u || static_cast<int32_t>(lane_value(static_cast<uint32_t>(L.above), node)) >= 0);
        };
        if (A.look) {
            if (!needed()) continue;
            if (node > 0u) {
                // A parent's first child is read before that one has decided, as it will mostly be needed; another waits, bounded. (All waiting 41 and 123 us instead of 32 and 95, none 35 and 101.)
                const uint32_t up = lane_value(static_cast<uint32_t>(L.above), node);
                const uint64_t siblings = __ballot(L.above == static_cast<int32_t>(up)) & ((uint64_t{1} << node) - 1ull);
                const uint32_t looks = siblings == 0ull || up % A.levels > level ? 1u : min(A.looks, kParentLooks);  // (a parent of workgroups that come later may not even have begun)
                if (t == 0u) {
                    unsigned long long v = 0;
                    bool known = false;
                    for (uint32_t look = 0; look < looks && !known; ++look) {
                        if (look != 0u) __builtin_amdgcn_s_sleep(8);
                        known = find_word(tree_decision(A, first + up), 1u, tag, v);
                    }
                    s_never = known && static_cast<uint32_t>(v & 0xffu) != node ? 1u : 0u;
                    if (s_never) leave_word(tree_decision(A, row), 1u, kDecNever, tag);
                }
                __syncthreads();
                const bool never = s_never != 0u;
                __syncthreads();
                if (never) continue;
            }
        }
        uint4 q[kU];
        uint32_t bits[kU];
        if (j0 < j1) {
#pragma unroll
            for (uint32_t u = 0; u < kU; ++u) q[u] = share.load(j0 + u * T + t, bits[u]);
        }
        const float inv_t32 = A.R.inv_t ? A.R.inv_t[row] : 1.f;
        const int32_t off = A.q ? A.q_off[row] : -1;
        if (!A.look && !needed()) continue;  // (few rows: it is read while that is found out)
        TreeNode N{};
        float x_child = -INFINITY;
        bool fine = true;
        if (t < 64u) fine = tree_drafts<DT, MASK>(A, off, base, allow, L, kids, s_seen, N, x_child);  // (while the row travels)
        const Scale c(inv_t32);
        Running<false> a;
        for (uint32_t jb = j0; jb < j1; jb += kU * T) {
            uint4 next[kU];
            uint32_t next_bits[kU];
            const bool more = jb + kU * T < j1;
            if (more) {
#pragma unroll
                for (uint32_t u = 0; u < kU; ++u) next[u] = share.load(jb + (kU + u) * T + t, next_bits[u]);
            }
#pragma unroll
            for (uint32_t u = 0; u < kU; ++u) {
                if (jb + u * T < j1) {  // (uniform)
                    float x[kPer];
                    unpack<DT>(share.own(q[u], bits[u], jb + u * T), x);
                    a.take(x, c);
                }
            }
            if (more) {
#pragma unroll
                for (uint32_t u = 0; u < kU; ++u) {
                    q[u] = next[u];
                    bits[u] = next_bits[u];
                }
            }
        }
        if (part == 0u && t < span.rest) {
            const uint32_t i = span.rest_index(t);
            if (!MASK || allowed(allow, i)) a.take1(load_logit<DT>(base, i), c);
        }
        RowSums r = block_sums<false, T>(a, c, red_m, red_s, red_t);
        bool mine = t < 64u;
        if (mine && A.row_parts > 1u) {  // (at most 64) who finds everybody's words decides; several may, and write the same
            unsigned long long* at = A.row_meet + static_cast<size_t>(row) * A.row_parts * 4u;
            if (t == 0u) {
                leave_word(at + part, A.row_parts, __float_as_uint(r.m), tag);
                leave_word(at + 2u * A.row_parts + part, A.row_parts, static_cast<unsigned long long>(__double_as_longlong(r.s)), tag);
            }
            words_arrived();
            const bool in = t < A.row_parts;
            unsigned long long wm = 0, ws = 0;
            bool here = !in;
            if (in) {
                here = find_word(at + t, A.row_parts, tag, wm);
                here = find_word(at + 2u * A.row_parts + t, A.row_parts, tag, ws) && here;
            }
            mine = __ballot(!here) == 0ull;
            r = join_parts<false>(in, PartSums{__uint_as_float(static_cast<uint32_t>(wm)), 0.f, __longlong_as_double(static_cast<long long>(ws)), 0.0}, c);
        }
        if (mine) {  // (a wave)
            const double inv_t = static_cast<double>(inv_t32), factor = tree_factor(inv_t32);
            uint32_t next = fine ? kDecNone : kDecBad;
            tree_begin(N, r.m, factor, r.s, -1.0);
            const double w_child = power64((static_cast<double>(x_child) - static_cast<double>(r.m)) * factor) / r.s;
            for (uint64_t left = fine ? kids : 0ull; left; left &= left - 1ull) {
                const uint32_t k = static_cast<uint32_t>(__ffsll(static_cast<long long>(left)) - 1), place = tree_find(N, lane_value(L.token, k));
                const double P = place < 64u ? lane_value(N.P, place) : N.c * lane_value(w_child, k);
                const double Q = N.guess ? 1.0 : (place < 64u ? lane_value(N.Q, place) : 0.0);
                if (lane_value(L.u, k) * Q < P) {
                    next = k;
                    break;
                }
                tree_reject(N, place);
            }
            const float lp = static_cast<float>((static_cast<double>(x_child) - static_cast<double>(r.m)) * inv_t - log(r.s));
            if (t == (next < 64u ? next : 0u)) leave_word(tree_decision(A, row), 1u, (static_cast<unsigned long long>(__float_as_uint(lp)) << 32) | next, tag);
        }
        __syncthreads();
    }
}

// ---- the walk, and the token behind it
constexpr uint32_t kDrawThreads = 256u;
template <int DT, bool MASK, int NV, int WAVES>
__global__ void __launch_bounds__(kDrawThreads, WAVES) tree_draw_kernel(TreeVerifyArgs A) {
    constexpr uint32_t T = kDrawThreads, kPer = Elem<DT>::kPer, kW = T / 64u;
    __shared__ float red_m[kW];
    __shared__ double red_t[kW];
    __shared__ float part_m[64];
    __shared__ double part_s[64];
    __shared__ unsigned long long missing;
    __shared__ uint32_t taken_out[T * NV / 4];  // a byte a vector of the share: which of its tokens are listed
    __shared__ uint32_t special_id[64];
    __shared__ double special_w[64];
    __shared__ uint32_t s_part, s_wave, s_token, s_last;
    __shared__ double s_target, s_wave_before;
    __shared__ float s_x;
    __shared__ double round_sum[NV][T];
    __shared__ __attribute__((aligned(16))) uint32_t s_seen[256];
    const uint32_t s = grid_row();
    if (s >= A.n_seq) return;
    const uint32_t part = blockIdx.x, t = threadIdx.x, lane = lane_id(), V = A.R.vocab, per = A.per, parts = A.parts;
    uint32_t n;
    const uint32_t first = tree_rows(A.seq_off, s, A.R.rows, n);
    unsigned long long* meet = A.meet + static_cast<size_t>(s) * parts * kTreeWords;

    const unsigned long long tag = A.tag;
    const double u_draw = A.u_draw[s];
    // down the tree, every wave by itself: a lane a node, and a lane a level for what was accepted
    const TreeLane L = tree_lane(A, first, n);
    unsigned long long decided = 0ull;
    const bool known = lane < n && find_word(tree_decision(A, first + lane), 1u, tag, decided);
    const uint32_t next_of = known ? static_cast<uint32_t>(decided & 0xffu) : kDecBad;
    int32_t path = -1;
    float path_lp = 0.f;
    uint32_t levels = 0, cur = 0;
    uint64_t kids = 0;
    bool bad = n == 0u;
    while (!bad) {
        kids = __ballot(L.above == static_cast<int32_t>(cur));
        if (kids == 0ull) break;
        const uint32_t next = lane_value(next_of, cur);
        if (next == kDecNone) break;
        if (next >= n || next <= cur) {
            bad = true;
            break;
        }
        const uint32_t lp = lane_value(static_cast<uint32_t>(decided >> 32), cur);
        if (lane == levels) {
            path = static_cast<int32_t>(next);
            path_lp = __uint_as_float(lp);
        }
        ++levels;
        cur = next;
    }

    // whether all of the sequence's workgroups have read the decisions: the last of them to leave its words finds everybody's at its first look, others may
    bool all_read = parts == 1u;
    if (bad) {
        __syncthreads();
        if (t < 64u && parts > 1u) {  // (the words of the draw, that say only that they are there)
            if (t == 0u) leave_word(meet + part, parts, 0ull, tag);
            words_arrived();
            unsigned long long w;
            const unsigned long long none = __ballot(t < parts && !find_word(meet + t, parts, tag, w));
            if (t == 0u) s_last = none == 0ull ? 1u : 0u;
        }
        __syncthreads();
        all_read = all_read || s_last != 0u;
    }

    uint32_t chosen = 0xffffffffu, target_part = 0;
    float chosen_x = 0.f, m = 0.f;
    double S = 0.0, inv_t = 1.0;
    if (!bad) {
        const uint32_t row = first + cur;
        const unsigned char* base = A.R.logits + row * A.R.row_bytes;
        const uint32_t* allow = MASK ? A.R.allow + row * A.R.allow_stride : nullptr;
        TreeShare<DT, MASK, T, NV> share;
        TreeNode N{};
        const float inv_t32 = A.R.inv_t ? A.R.inv_t[row] : 1.f;
        inv_t = static_cast<double>(inv_t32);
        const double factor = tree_factor(inv_t32);
        const int32_t off = A.q ? A.q_off[row] : -1;
        const bool no_t = !(inv_t > 0.0 && inv_t < static_cast<double>(INFINITY));
        float share_m = 0.f;
        // weights of a share's tokens that are not listed, against the share's own maximum: the sum of each round of a thread, and of the workgroup
        auto weights = [&](uint32_t u_, double (&w)[kPer]) {
            float x[kPer];
            unpack<DT>(share.q[u_], x);
            const double share_at = static_cast<double>(share_m) * factor;
            const uint32_t out = reinterpret_cast<const unsigned char*>(taken_out)[wave_id() * 64u * share.rounds + u_ * 64u + lane];
#pragma unroll
            for (uint32_t e = 0; e < kPer; ++e) {  // (those as if they were not there: a branch around each power would have one wait for the other)
                const float mine = out >> e & 1u ? -INFINITY : x[e];
                w[e] = power64(fma(static_cast<double>(mine), factor, -share_at));
                if (e % 4u == 3u) __builtin_amdgcn_sched_barrier(0);  // (more of them together take the registers that the row is in)
            }
        };
        auto outside_sum = [&]() {
            for (uint32_t i = t; i < T * NV / 4u; i += T) taken_out[i] = 0u;
            bool odd = no_t;
            const float mine = wave_max(share.largest(odd));
            const uint64_t odds = __ballot(odd);
            if (lane == 0u) red_m[wave_id()] = odds ? __builtin_nanf("") : mine;
            __syncthreads();
            if (t < 64u && N.listed && N.id < V) {
                const uint32_t j = N.id / kPer;
                if (j >= share.j0 && j < share.j1) atomicOr(&taken_out[(j - share.j0) / 4u], 1u << ((j - share.j0) % 4u * 8u + N.id % kPer));
            }
            share_m = -FLT_MAX;
            bool any_odd = false;
#pragma unroll
            for (uint32_t w = 0; w < kW; ++w) {
                any_odd = any_odd || red_m[w] != red_m[w];
                share_m = fmaxf(share_m, red_m[w]);
            }
            __syncthreads();
            double sum = 0.0;
#pragma unroll
            for (uint32_t v = 0; v < NV; ++v) {
                if (v < share.rounds) {  // (uniform)
                    double w[kPer], of_round = 0.0;
                    weights(v, w);
#pragma unroll
                    for (uint32_t e = 0; e < kPer; ++e) of_round += w[e];
                    round_sum[v][t] = of_round;  // (read again by the wave that the target lies in)
                    sum += of_round;
                }
            }
            sum = wave_sum(sum);
            if (lane == 0u) red_t[wave_id()] = sum;
            __syncthreads();
            double all = 0.0;
            for (uint32_t w = 0; w < kW; ++w) all += red_t[w];
            return any_odd ? __builtin_nan("") : all;  // (no sum: nothing can be drawn)
        };
        unsigned long long late = 0;
        uint32_t p = part;
        for (bool first_turn = true;; first_turn = false) {  // the own share, those of workgroups that have not come, then the own again where it is no longer there
            share.place(V, p, per);
            share.load(base, allow, V);
            if (first_turn && t < 64u) {  // (while the row travels)
                float x_child;
                tree_drafts<DT, MASK>(A, off, base, allow, L, kids, s_seen, N, x_child);
            }
            const double sum = outside_sum();
            if (first_turn && parts > 1u) {
                if (t < 64u) {  // everybody's maximum and sum
                    if (t == 0u) {
                        leave_word(meet + part, parts, __float_as_uint(share_m), tag);
                        leave_word(meet + 2u * parts + part, parts, static_cast<unsigned long long>(__double_as_longlong(sum)), tag);
                    }
                    words_arrived();
                    bool here = t >= parts;
                    unsigned long long wm = 0, ws = 0;
                    uint32_t look = 0;
                    for (; look < A.looks; ++look) {
                        if (!here) {
                            here = find_word(meet + t, parts, tag, wm);
                            here = find_word(meet + 2u * parts + t, parts, tag, ws) && here;
                        }
                        if (__ballot(!here) == 0ull) break;
                        __builtin_amdgcn_s_sleep(2);
                    }
                    const unsigned long long none = __ballot(!here);
                    part_m[t] = __uint_as_float(static_cast<uint32_t>(wm));
                    part_s[t] = __longlong_as_double(static_cast<long long>(ws));
                    if (t == 0u) {
                        missing = none;
                        s_last = look == 0u ? 1u : 0u;
                    }
                }
            } else if (t == 0u && (first_turn || p != part)) {
                part_m[p] = share_m;
                part_s[p] = sum;
            }
            __syncthreads();
            if (parts == 1u) break;
            if (first_turn) {
                late = missing;
                all_read = s_last != 0u;
            }
            else if (p == part) break;
            else late &= late - 1ull;
            if (first_turn && late == 0ull) break;
            p = late ? static_cast<uint32_t>(__ffsll(late) - 1) : part;
        }
        if (t < 64u) {
            const float mine_m = t < parts ? part_m[t] : -FLT_MAX;
            m = wave_max(mine_m);
            const double scale = power64((static_cast<double>(mine_m) - static_cast<double>(m)) * factor);
            const double outside = t < parts ? part_s[t] * scale : 0.0, out_all = wave_sum(outside);
            const double w = N.listed ? power64((static_cast<double>(N.x) - static_cast<double>(m)) * factor) : 0.0;
            S = out_all + wave_sum(w);
            tree_begin(N, m, factor, S, out_all);
            for (uint64_t left = kids; left; left &= left - 1ull)
                tree_reject(N, tree_find(N, lane_value(L.token, static_cast<uint32_t>(__ffsll(static_cast<long long>(left)) - 1))));
            // in units of the weights outside
            const double special = N.listed && N.id < V ? N.P / N.c * S : 0.0;
            double in_part = outside;
            for (uint64_t left = __ballot(special > 0.0); left; left &= left - 1ull) {
                const uint32_t l = static_cast<uint32_t>(__ffsll(static_cast<long long>(left)) - 1);
                if (lane_value(N.id, l) / kPer / per == t) in_part += lane_value(special, l);
            }
            const double upto = wave_incl_scan(in_part), all = last_lane(upto), target = u_draw * all;
            // the first part up to which there is more than the target; else the last with any
            const uint64_t over = __ballot(upto > target && in_part > 0.0), any = __ballot(in_part > 0.0);
            const uint32_t at = over ? static_cast<uint32_t>(__ffsll(static_cast<long long>(over)) - 1) : (any ? 63u - static_cast<uint32_t>(__clzll(static_cast<long long>(any))) : 0u);
            const bool none = !(all > 0.0 && all < static_cast<double>(INFINITY));
            const double before = at ? lane_value(upto, at - 1u) : 0.0, unit = lane_value(scale, at);
            // what the part's workgroup goes on with is in its own units
            special_id[t] = special > 0.0 ? N.id : 0xffffffffu;
            special_w[t] = special / unit;
            if (t == 0u) {
                s_part = none ? 0xffffffffu : at;
                s_target = (target - before) / unit;
            }
        }
        __syncthreads();
        bad = s_part == 0xffffffffu;
        target_part = bad ? 0u : s_part;
        if (!bad && target_part == part) {  // (uniform)
            const double target = s_target;
            const uint32_t wave_vectors = 64u * share.rounds;
            // what the listed ids of [lo, hi) weigh; the same for the whole wave
            auto special_sum = [&](uint32_t lo, uint32_t hi) {
                const uint32_t id = special_id[lane];
                return wave_sum(id >= lo && id < hi ? special_w[lane] : 0.0);
            };
            if (t < 64u) {
                double before = 0.0;
                uint32_t at = 0xffffffffu, last = 0;
                double at_before = before, last_before = before;
                for (uint32_t w = 0; w < kW; ++w) {
                    const uint32_t lo = (share.j0 + w * wave_vectors) * kPer, hi = min(share.j0 + (w + 1u) * wave_vectors, share.j1) * kPer;
                    const double sum = red_t[w] + (lo < hi ? special_sum(lo, hi) : 0.0), upto = before + sum;
                    if (sum > 0.0) {
                        last = w;
                        last_before = before;
                    }
                    if (at == 0xffffffffu && upto > target && sum > 0.0) {
                        at = w;
                        at_before = before;
                    }
                    before = upto;
                }
                if (t == 0u) {
                    s_wave = at == 0xffffffffu ? last : at;
                    s_wave_before = at == 0xffffffffu ? last_before : at_before;
                }
            }
            __syncthreads();
            if (s_wave == static_cast<uint32_t>(wave_id())) {
                double before = s_wave_before, at_before = before, last_before = before;
                uint32_t at = 0xffffffffu, last = 0;
                const uint32_t j_wave = share.j0 + wave_id() * wave_vectors;
                for (uint32_t v = 0; v < share.rounds; ++v) {
                    const uint32_t lo = j_wave + v * 64u, hi = min(lo + 64u, share.j1);
                    const double sum = wave_sum(round_sum[v][t]) + (lo < hi ? special_sum(lo * kPer, hi * kPer) : 0.0), upto = before + sum;
                    if (sum > 0.0) {
                        last = v;
                        last_before = before;
                    }
                    if (at == 0xffffffffu && upto > target && sum > 0.0) {
                        at = v;
                        at_before = before;
                    }
                    before = upto;
                }
                if (at == 0xffffffffu) {
                    at = last;
                    at_before = last_before;
                }
                double w[kPer];
                float x[kPer];
#pragma unroll
                for (uint32_t v = 0; v < NV; ++v) {
                    if (v == at) {  // (uniform)
                        weights(v, w);
                        unpack<DT>(share.q[v], x);
                    }
                }
                const uint32_t id0 = (j_wave + at * 64u + lane) * kPer;
                const uint32_t listed = special_id[lane], of_round = (j_wave + at * 64u) * kPer;
                for (uint64_t left = __ballot(listed - of_round < 64u * kPer); left; left &= left - 1ull) {  // those of this round
                    const uint32_t l = static_cast<uint32_t>(__ffsll(static_cast<long long>(left)) - 1), id = lane_value(listed, l);
#pragma unroll
                    for (uint32_t e = 0; e < kPer; ++e)
                        if (id == id0 + e) w[e] = special_w[l];
                }
                double sum = 0.0;
#pragma unroll
                for (uint32_t e = 0; e < kPer; ++e) sum += w[e];
                const double upto = wave_incl_scan(sum);
                const uint64_t any = __ballot(sum > 0.0);
                uint64_t over = __ballot(at_before + upto > target && sum > 0.0);
                if (!over) over = any ? 1ull << (63u - static_cast<uint32_t>(__clzll(static_cast<long long>(any)))) : 1ull;
                const uint32_t l = static_cast<uint32_t>(__ffsll(static_cast<long long>(over)) - 1);
                if (lane == l) {
                    double run = at_before + (upto - sum);
                    uint32_t pick = 0xffffffffu, end = 0;
                    float pick_x = 0.f, end_x = x[0];
#pragma unroll
                    for (uint32_t e = 0; e < kPer; ++e) {
                        run += w[e];
                        if (w[e] > 0.0) {
                            end = e;
                            end_x = x[e];
                            if (pick == 0xffffffffu && run > target) {
                                pick = e;
                                pick_x = x[e];
                            }
                        }
                    }
                    s_token = id0 + (pick == 0xffffffffu ? end : pick);
                    s_x = pick == 0xffffffffu ? end_x : pick_x;
                }
            }
            __syncthreads();
            chosen = s_token;
            chosen_x = s_x;
        }
    }

    if (target_part == part && t < 64u) {
        uint32_t status = bad ? kAcceptHost : 0u;
        uint32_t accepted = levels;
        if (!bad && A.hist.tokens) {
            const uint32_t slot = A.hist.slot ? A.hist.slot[s] : s;
            int32_t* text = A.hist.tokens + static_cast<size_t>(slot) * A.hist.cap;
            const uint32_t len = A.hist.len[slot];
            // (a path without room: the cache could not be brought to what the history would say)
            const uint32_t full = (static_cast<uint64_t>(len) + accepted + 2u > A.hist.cap ? kAcceptHistoryFull : 0u) | (accepted > A.depth ? kAcceptPathFull : 0u);
            if (full) {
                status = full | kAcceptHost;
                accepted = 0u;
                chosen = 0xffffffffu;
            } else {
                const int32_t kept = __shfl(static_cast<int32_t>(L.token), max(path, 0));
                if (t < accepted) text[len + 1u + t] = kept;
                if (t == 0u) {
                    text[len + 1u + accepted] = static_cast<int32_t>(chosen);
                    A.hist.len[slot] = len + 1u + accepted;
                    if (A.hist.n_gen) A.hist.n_gen[slot] += accepted + 1ull;
                }
            }
        }
        const bool drawn = chosen != 0xffffffffu;
        if (t == 0u) {
            A.n_accepted[s] = static_cast<int32_t>(accepted);
            A.chosen[s] = static_cast<int32_t>(chosen);
            A.status[s] = status;
        }
        if (t < A.depth) A.path[static_cast<size_t>(s) * A.depth + t] = t < accepted ? path : -1;
        if (A.logprob) {
            float lp = t < accepted ? path_lp : 0.f;
            if (t == accepted && drawn) lp = static_cast<float>((static_cast<double>(chosen_x) - static_cast<double>(m)) * inv_t - log(S));
            float* to = A.logprob + static_cast<size_t>(s) * (A.depth + 1u);
            if (t <= A.depth) to[t] = lp;
            if (t == 0u && A.depth == 64u) to[64] = 0.f;  // (63 drafts at most are accepted: the chosen one's is in the 64th place)
        }
    }
    if (all_read) {  // the rows' words are taken apart (by all of a sequence's workgroups: five rows 11 -> 14.5 us)
        for (uint32_t i = t; i < n; i += T) break_word(tree_decision(A, first + i), 1u);
        if (A.row_parts > 1u) {
            for (uint32_t i = t; i < 2u * n * A.row_parts; i += T) {  // a row's maxima, its sums, the next row's
                const uint32_t w = i / A.row_parts;
                break_word(A.row_meet + (static_cast<size_t>(first) * 2u + w) * A.row_parts * 2u + (i - w * A.row_parts), A.row_parts);
            }
        }
    }
}

}  // namespace ws
