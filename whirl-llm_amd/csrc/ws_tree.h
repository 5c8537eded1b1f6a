// A cycle's drafts as trees: what a row sees and where it stands (tree_stage_kernel), and the drafts' verification against the target's logits (tree_verify_kernel).
//
// Verification. With w_v = exp((x_v - m) t) over the allowed tokens of a node's row, S = sum w_v and P = w / S, a child with token y is accepted if u Q(y) < P(y); after
// a rejection P becomes max(P - Q, 0) divided by its sum Z. Q is 0 but at 32 ids at most (or at one, where the child is a guess), so that outside of them P stays w times one number c:
// what a walk carries along is c and the P and Q of those ids, a lane each, and the mass outside of them, 1 - sum P at first. No pass over the row is made for a rejection. What is read:
// the rows that the walk meets, once, for m and S; the one that it ends at a second time, out of the registers that hold it.
//
// Accuracy. The comparisons u Q < P are made in 64 bits, S is added up from powers of 32 bits (1e-8 of S where many tokens count): of ten million drafts one may be judged otherwise than by an
// exact sum. The token behind the walk is looked for among some 100 000 steps of a cumulative sum, whose places would move by 1e-8 of the sum, a hundredth of a step where tokens are
// unlikely: there the powers are taken in 64 bits (to 1e-12), and S, Z and the P of the listed ids once more from them.
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

// e^y for y <= 0 to 1e-12: y = k ln 2 + r, |r| <= 0.35, the Taylor polynomial of e^r to its tenth power (the next is 0.35^11 / 11! = 2e-13)
__device__ __forceinline__ double exp64(double y) {
    const double k = rint(y * 1.4426950408889634074);
    double r = fma(k, -0x1.62e42f0000000p-1, y);  // (ln 2 in two parts, the first of 25 bits: k times it is exact)
    r = fma(k, -0x1.df473de6af279p-26, r);
    double p = 1.0 / 3628800.0;
    p = fma(p, r, 1.0 / 362880.0);
    p = fma(p, r, 1.0 / 40320.0);
    p = fma(p, r, 1.0 / 5040.0);
    p = fma(p, r, 1.0 / 720.0);
    p = fma(p, r, 1.0 / 120.0);
    p = fma(p, r, 1.0 / 24.0);
    p = fma(p, r, 1.0 / 6.0);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    const double e = ldexp(p, static_cast<int>(k));
    return y < -700.0 ? 0.0 : e;  // (-inf too; NaN stays)
}

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
    __device__ __forceinline__ void sums(const Scale& c, Running<false>& a) const {
#pragma unroll
        for (int u = 0; u < NV; ++u) {
            if (static_cast<uint32_t>(u) < rounds) {
                float x[kPer];
                unpack<DT>(q[u], x);
                a.take(x, c);
            }
        }
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
__device__ __forceinline__ void tree_begin(TreeNode& N, float m, double inv_t, double S, double out_known) {
    N.P = N.listed ? exp64((static_cast<double>(N.x) - static_cast<double>(m)) * inv_t) / S : 0.0;
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

template <int DT, bool MASK, int T, int NV, int WAVES>
__global__ void __launch_bounds__(T, WAVES) tree_verify_kernel(TreeVerifyArgs A) {
    constexpr uint32_t kPer = Elem<DT>::kPer, kW = T / 64u;
    __shared__ float red_m[kW];
    __shared__ double red_s[kW], red_t[kW];
    __shared__ float part_m[64];
    __shared__ double part_s[64];
    __shared__ unsigned long long missing;
    __shared__ uint32_t s_next;
    __shared__ float s_m;
    __shared__ uint32_t taken_out[T * NV / 4];  // a byte a vector of the share: which of its tokens are listed
    __shared__ uint32_t special_id[64];
    __shared__ double special_w[64];
    __shared__ uint32_t s_part, s_wave, s_token;
    __shared__ double s_before, s_target, s_wave_before;
    __shared__ float s_x;
    __shared__ double round_sum[NV][T];
    const uint32_t s = grid_row();
    if (s >= A.n_seq) return;
    const uint32_t part = blockIdx.x, t = threadIdx.x, lane = lane_id(), V = A.R.vocab, per = A.per, parts = A.parts;
    uint32_t n;
    const uint32_t first = tree_rows(A.seq_off, s, A.R.rows, n);
    unsigned long long* meet = A.meet + static_cast<size_t>(s) * parts * kTreeWords;

    // what the first wave knows of the nodes, a lane a node, and of the walk, a lane a level
    int32_t above = -1;
    uint32_t token = 0xffffffffu;
    double u = 0.0;
    int32_t path = -1;
    float path_lp = 0.f;
    uint32_t levels = 0;
    if (t < n) {
        above = A.parent ? A.parent[first + t] : static_cast<int32_t>(t) - 1;
        if (t == 0u || above >= static_cast<int32_t>(t)) above = -1;
        token = static_cast<uint32_t>(A.R.ids[first + t]);
        u = A.u_accept[first + t];
    }
    TreeShare<DT, MASK, T, NV> share;
    TreeNode N{};
    uint64_t kids = 0;
    bool bad = n == 0u, own = false;
    uint32_t cur = 0, step = 0;
    float m = 0.f;
    double S = 0.0, inv_t = 1.0;
    const unsigned char* base = nullptr;
    const uint32_t* allow = nullptr;

    // everybody's words of this step, two a part, by the first wave: in part_m, part_s, and a bit in `missing` for each that has not come
    auto meet_parts = [&](float mine_m, double mine_s) {
        if (t >= 64u) return;
        unsigned long long* at = meet + (step & 1u) * 4u * parts;
        const unsigned long long tag = A.tag + (step + 1ull) * 0x9E3779B97F4A7C15ull;
        if (t == 0u) {
            leave_word(at + part, parts, __float_as_uint(mine_m), tag);
            leave_word(at + 2u * parts + part, parts, static_cast<unsigned long long>(__double_as_longlong(mine_s)), tag);
        }
        words_arrived();
        bool here = t >= parts;
        unsigned long long wm = 0, ws = 0;
        for (uint32_t look = 0; look < A.looks; ++look) {
            if (!here) {
                here = find_word(at + t, parts, tag, wm);
                here = find_word(at + 2u * parts + t, parts, tag, ws) && here;
            }
            if (__ballot(!here) == 0ull) break;
            __builtin_amdgcn_s_sleep(2);
        }
        const unsigned long long late = __ballot(!here);
        part_m[t] = __uint_as_float(static_cast<uint32_t>(wm));
        part_s[t] = __longlong_as_double(static_cast<long long>(ws));
        if (t == 0u) missing = late;
    };
    // the sums of the share in `share`, in the first wave
    auto row_sums = [&](const Scale& c) {
        Running<false> a;
        share.sums(c, a);
        return block_sums<false, T>(a, c, red_m, red_s, red_t);
    };

    while (!bad) {  // a node a turn
        const uint32_t row = first + cur;
        base = A.R.logits + row * A.R.row_bytes;
        allow = MASK ? A.R.allow + row * A.R.allow_stride : nullptr;
        const float inv_t32 = A.R.inv_t ? A.R.inv_t[row] : 1.f;
        inv_t = static_cast<double>(inv_t32);
        float x_child = -INFINITY;
        bool entry_bad = false;
        auto drafts = [&]() {  // the first wave's: the node's children and what their distribution names
            kids = __ballot(above == static_cast<int32_t>(cur));
            auto logit = [&](uint32_t id) { return id < V && (!MASK || allowed(allow, id)) ? load_logit<DT>(base, id) : -INFINITY; };
            const int32_t off = A.q ? A.q_off[row] : -1;
            N.guess = off < 0;
            N.drawn = 0.0;
            if (kids >> t & 1u) x_child = logit(token);
            if (N.guess) {
                N.listed = kids >> t & 1u;
                N.id = token;
                N.x = x_child;
            } else if (kids == 0ull) {
                N.listed = false;
            } else {
                entry_bad = static_cast<uint64_t>(off) + kTreeEntryWords > A.q_words;
                const int32_t* entry = A.q + (entry_bad ? 0 : off);
                const int32_t count = entry_bad ? 0 : entry[0];
                N.listed = t < kTreeListed && static_cast<int32_t>(t) < count;
                if (N.listed) {
                    N.id = static_cast<uint32_t>(entry[1u + t]);
                    N.drawn = static_cast<double>(__int_as_float(entry[33u + t]));
                }
                N.x = N.listed ? logit(N.id) : -INFINITY;
                if (entry_bad) kids = 0ull;  // (none is looked at)
            }
            // an id that is named before counts there
            const uint64_t names = __ballot(N.listed);
            for (uint64_t left = names; left; left &= left - 1ull) {
                const uint32_t l = static_cast<uint32_t>(__ffsll(static_cast<long long>(left)) - 1), id = lane_value(N.id, l);
                const uint64_t same = __ballot(N.listed && N.id == id) & (~0ull << l);
                if ((same & (same - 1ull)) == 0ull) continue;
                const double sum = wave_sum((same >> t & 1u) ? N.drawn : 0.0);
                if (t == l) N.drawn = sum;
                else if (same >> t & 1u) N.listed = false;
                left &= ~same | (1ull << l);
            }
        };
        const Scale c(inv_t32);
        RowSums r;
        unsigned long long late = 0;
        uint32_t p = part;
        for (bool first_turn = true;; first_turn = false) {  // the own share, then those of workgroups that have not come (in one loop: the code is there once)
            share.place(V, p, per);
            share.load(base, allow, V);
            if (first_turn && t < 64u) drafts();  // (while the row travels)
            r = row_sums(c);
            if (parts == 1u) break;
            if (first_turn) {
                meet_parts(r.m, r.s);
            } else if (t == 0u) {
                part_m[p] = r.m;
                part_s[p] = r.s;
            }
            __syncthreads();
            late = first_turn ? missing : late & (late - 1ull);
            if (late == 0ull) break;
            p = static_cast<uint32_t>(__ffsll(late) - 1);
        }
        own = p == part;
        if (parts > 1u && t < 64u) {
            __builtin_amdgcn_wave_barrier();
            r = join_parts<false>(t < parts, PartSums{part_m[t], 0.f, part_s[t], 0.0}, c);
        }
        ++step;
        if (t < 64u) {
            const double lnS = log(r.s);
            uint32_t next = 0xffffffffu;
            tree_begin(N, r.m, inv_t, r.s, -1.0);
            const double w_child = exp64((static_cast<double>(x_child) - static_cast<double>(r.m)) * inv_t) / r.s;
            for (uint64_t left = kids; left; left &= left - 1ull) {
                const uint32_t k = static_cast<uint32_t>(__ffsll(static_cast<long long>(left)) - 1), place = tree_find(N, lane_value(token, k));
                const double P = place < 64u ? lane_value(N.P, place) : N.c * lane_value(w_child, k);
                const double Q = N.guess ? 1.0 : (place < 64u ? lane_value(N.Q, place) : 0.0);
                if (lane_value(u, k) * Q < P) {
                    next = k;
                    break;
                }
                tree_reject(N, place);
            }
            if (next != 0xffffffffu) {
                const float lp = static_cast<float>((static_cast<double>(__uint_as_float(lane_value(__float_as_uint(x_child), next))) - static_cast<double>(r.m)) * inv_t - lnS);
                if (t == levels) {
                    path = static_cast<int32_t>(next);
                    path_lp = lp;
                }
                ++levels;
            }
            if (t == 0u) {
                s_next = entry_bad ? 0xfffffffeu : next;
                s_m = r.m;
            }
        }
        __syncthreads();
        const uint32_t next = s_next;
        m = s_m;
        __syncthreads();
        if (next == 0xfffffffeu) bad = true;
        if (next >= 0xfffffffeu) break;
        cur = next;
    }

    // the token behind the walk
    uint32_t chosen = 0xffffffffu;
    float chosen_x = 0.f;
    uint32_t target_part = 0;
    if (!bad) {
        // weights of a share's tokens that are not listed: the sum of each round of a thread, and of the workgroup
        auto weights = [&](uint32_t u_, double (&w)[kPer]) {
            float x[kPer];
            unpack<DT>(share.q[u_], x);
            const uint32_t out = reinterpret_cast<const unsigned char*>(taken_out)[wave_id() * 64u * share.rounds + u_ * 64u + lane];
#pragma unroll
            for (uint32_t e = 0; e < kPer; ++e) w[e] = out >> e & 1u ? 0.0 : exp64((static_cast<double>(x[e]) - static_cast<double>(m)) * inv_t);
        };
        auto outside_sum = [&]() {
            for (uint32_t i = t; i < T * NV / 4u; i += T) taken_out[i] = 0u;
            __syncthreads();
            if (t < 64u && N.listed && N.id < V) {
                const uint32_t j = N.id / kPer;
                if (j >= share.j0 && j < share.j1) atomicOr(&taken_out[(j - share.j0) / 4u], 1u << ((j - share.j0) % 4u * 8u + N.id % kPer));
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
                    round_sum[v][t] = of_round;  // (LDS: read again by the wave that the target lies in)
                    sum += of_round;
                }
            }
            sum = wave_sum(sum);
            if (lane == 0u) red_t[wave_id()] = sum;
            __syncthreads();
            double all = 0.0;
            for (uint32_t w = 0; w < kW; ++w) all += red_t[w];
            return all;
        };
        unsigned long long late = 0;
        uint32_t p = part;
        for (bool first_turn = true;; first_turn = false) {  // the own share, those of workgroups that have not come, then the own again where it is no longer there
            if (!own || !first_turn) {
                share.place(V, p, per);
                share.load(base, allow, V);
                __syncthreads();  // (taken_out and red_t are free)
            }
            const double sum = outside_sum();
            if (first_turn) {
                if (parts > 1u) meet_parts(0.f, sum);
                else if (t == 0u) part_s[0] = sum;
            } else if (t == 0u && p != part) {
                part_s[p] = sum;
            }
            __syncthreads();
            if (parts == 1u) break;
            if (first_turn) late = missing;
            else if (p == part) break;
            else late &= late - 1ull;
            if (first_turn && late == 0ull) break;
            p = late ? static_cast<uint32_t>(__ffsll(late) - 1) : part;
        }
        if (t < 64u) {
            const double outside = t < parts ? part_s[t] : 0.0, out_all = wave_sum(outside);
            const double w = N.listed ? exp64((static_cast<double>(N.x) - static_cast<double>(m)) * inv_t) : 0.0;
            S = out_all + wave_sum(w);
            tree_begin(N, m, inv_t, S, out_all);
            for (uint64_t left = kids; left; left &= left - 1ull)
                tree_reject(N, tree_find(N, lane_value(token, static_cast<uint32_t>(__ffsll(static_cast<long long>(left)) - 1))));
            // in units of the weights outside
            const double special = N.listed && N.id < V ? N.P / N.c * S : 0.0;
            special_id[t] = special > 0.0 ? N.id : 0xffffffffu;
            special_w[t] = special;
            double in_part = outside;
            for (uint64_t left = __ballot(special > 0.0); left; left &= left - 1ull) {
                const uint32_t l = static_cast<uint32_t>(__ffsll(static_cast<long long>(left)) - 1);
                if (lane_value(N.id, l) / kPer / per == t) in_part += lane_value(special, l);
            }
            const double upto = wave_incl_scan(in_part), all = last_lane(upto), target = A.u_draw[s] * all;
            // the first part up to which there is more than the target; else the last with any
            const uint64_t over = __ballot(upto > target && in_part > 0.0), any = __ballot(in_part > 0.0);
            const uint32_t p = over ? static_cast<uint32_t>(__ffsll(static_cast<long long>(over)) - 1) : (any ? 63u - static_cast<uint32_t>(__clzll(static_cast<long long>(any))) : 0u);
            const bool none = !(all > 0.0 && all < static_cast<double>(INFINITY));
            const double before = p ? lane_value(upto, p - 1u) : 0.0;  // (upto of the lane before, not upto - in_part: no rounding of the difference)
            if (t == 0u) {
                s_part = none ? 0xffffffffu : p;
                s_before = before;
                s_target = target;
            }
        }
        __syncthreads();
        bad = s_part == 0xffffffffu;
        target_part = bad ? 0u : s_part;
        if (!bad && target_part == part) {  // (uniform)
            const double target = s_target;
            const uint32_t wave_vectors = 64u * share.rounds;
            // what the listed ids of [lo, hi) weigh, a lane each; the same for the whole wave
            auto special_sum = [&](uint32_t lo, uint32_t hi) {
                const uint32_t id = special_id[lane];
                return wave_sum(id >= lo && id < hi ? special_w[lane] : 0.0);
            };
            if (t < 64u) {
                double before = s_before;
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
#pragma unroll
                for (uint32_t v = 0; v < NV; ++v) {
                    if (v < share.rounds) {
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
                for (uint32_t l = 0; l < 64u; ++l) {
                    const uint32_t id = special_id[l];
                    if (id == 0xffffffffu) continue;  // (uniform)
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
            if (static_cast<uint64_t>(len) + accepted + 2u > A.hist.cap) {
                status = kAcceptHistoryFull | kAcceptHost;
                accepted = 0u;
                chosen = 0xffffffffu;
            } else {
                const int32_t kept = __shfl(static_cast<int32_t>(token), max(path, 0));
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
    if (parts > 1u && n != 0u && t < 64u) {
        // all words of this part have arrived; who finds everybody's mark breaks the sequence's words, for a captured launch has its tag again at every replay
        unsigned long long* marks = meet + 8u * parts;
        words_arrived();
        if (t == 0u) leave_word(marks + part, parts, 0ull, A.tag);
        words_arrived();
        unsigned long long v;
        const bool here = t >= parts || find_word(marks + t, parts, A.tag, v);
        if (__ballot(!here) == 0ull && t < parts) {
#pragma unroll
            for (uint32_t k = 0; k < 5u; ++k) break_word(meet + 2u * k * parts + t, parts);
        }
    }
}

}  // namespace ws
