// Log-probabilities of given tokens, the losses over them and the gradients with respect to the logits.
//
// A row of logits x with inverse temperature t and allowed set L (all tokens without a mask): m = max x_v, S = sum over L of
// exp((x_v - m) t), p_v = exp((x_v - m) t) / S. The token y of the row has log p_y = (x_y - m) t - ln S, the row the entropy
// H = ln S - (1 / S) sum exp(d_v) d_v with d_v = (x_v - m) t. With g = dF/d(log p_y) and h = dF/dH of any loss F
//     dF/dx_v = t [ g (1[v = y] - p_v) - h p_v (ln p_v + H) ].
// Both directions are one pass over the row: forwards every thread keeps a maximum, a sum and (for H) a sum of products that are
// scaled down when its maximum grows, backwards every logit gives its own derivative. Exponentials go to base two with the factor
// t log2(e) split in two floats (a rounded one alone would move every exponent the same way, 1e-6 of a sum); sums are held
// in 32 bits by a thread, over some 120 terms at most where a row's workgroups share it (scores without a workspace: over the 4096 that a thread has of the longest row),
// and in 64 bits from the wave on; ln S, log p and the loss of a token in 64 bits.
#pragma once

#include "ws_common.h"

#include <float.h>

namespace ws {

struct LossRows {
    const unsigned char* logits;
    uint64_t row_bytes;
    uint32_t rows, vocab;
    const int32_t* ids;
    const float* inv_t;
    const uint32_t* allow;
    uint64_t allow_stride;
};

// the clipped policy loss of a token (ws_policy)
struct PolicyIn {
    const float* old_logprob;
    const float* ref_logprob;
    const float* advantage;
    const float* weight;
    double weight_all;  // without `weight`
    double clip_low, clip_high, dual_clip, kl_coef, entropy_coef;
};
constexpr uint32_t kPolicySums = 5u;  // loss, surrogate, KL, entropy, clipped share
struct PolicyToken {
    double g, h;  // derivatives by the log-probability and the entropy
    double sum[kPolicySums];
};

struct PolicyRow {  // a token's entries
    float old_logprob, ref_logprob, advantage;
    double weight;
};
__device__ __forceinline__ double policy_weight(const PolicyIn& P, uint32_t row) { return P.weight ? static_cast<double>(P.weight[row]) : P.weight_all; }
__device__ __forceinline__ PolicyRow policy_row(const PolicyIn& P, uint32_t row) {
    return PolicyRow{P.old_logprob[row], P.ref_logprob ? P.ref_logprob[row] : 0.f, P.advantage[row], policy_weight(P, row)};
}

// gain = min(r A, clip(r) A) with r = exp(lp - old); for A < 0 not below dual_clip * A. Where the clip holds it there is no
// derivative, so the comparison is made in 64 bits: rounded to 32, one token in some million would fall on the other side.
__device__ __forceinline__ PolicyToken policy_token(const PolicyIn& P, const PolicyRow& T, double lp, double H) {
    PolicyToken o{};
    if (static_cast<float>(lp) == -INFINITY) {
        lp = -static_cast<double>(INFINITY);  // (as the caller sees it, and compares it with the others')
        if (T.old_logprob == -INFINITY) return o;  // neither model can give it, and the ratio has no value: it counts for nothing
    }
    const double w = T.weight, A = static_cast<double>(T.advantage), e = exp(lp - static_cast<double>(T.old_logprob)), r = e > DBL_MAX ? DBL_MAX : e;  // (+inf times an advantage of 0: NaN)
    const double free = r * A, held = fmin(fmax(r, 1.0 - P.clip_low), 1.0 + P.clip_high) * A;
    double gain = held < free ? held : free;
    bool clipped = held < free;
    if (P.dual_clip > 0.0 && A < 0.0 && gain < P.dual_clip * A) {
        gain = P.dual_clip * A;
        clipped = true;
    }
    double kl = 0.0, back = 0.0;
    if (P.ref_logprob) {  // exp(b) - b - 1 with b = ref - lp, never negative; +inf where b is (not inf - inf); 0 where both are -inf: no token of either's
        const double ref = static_cast<double>(T.ref_logprob), b = ref == lp ? 0.0 : ref - lp;
        back = expm1(b);
        kl = b == static_cast<double>(INFINITY) ? b : back - b;
    }
    o.g = w * ((clipped ? 0.0 : -free) - (P.kl_coef != 0.0 ? P.kl_coef * back : 0.0));
    o.h = -P.entropy_coef * w;
    o.sum[0] = w * (-gain + (P.kl_coef != 0.0 ? P.kl_coef * kl : 0.0) - (P.entropy_coef != 0.0 ? P.entropy_coef * H : 0.0));
    o.sum[1] = -w * gain;
    o.sum[2] = w * kl;
    o.sum[3] = w * H;
    o.sum[4] = clipped ? w : 0.0;
    return o;
}

// ---- workgroups that meet in memory of any contents, as argmax_shared does (ws_top.h): every word is left twice, once mixed with a
// tag that no other launch has; whoever finds all pairs together goes on, the one whose words come last does, others may and
// write the same. The pairs are then broken, for a captured launch has its tag again at every replay. `apart`: words between the two of
// a pair, with the same word of the other workgroups between them: everybody looks at everybody's, past the caches, and a look at words
// side by side is an eighth of the requests (64 parts of a row of 151936, their words 32 bytes apart: 8.3 us, the launch without them 5.8).
__device__ __forceinline__ void leave_word(unsigned long long* at, uint32_t apart, unsigned long long v, unsigned long long tag) {
    __hip_atomic_store(at, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __hip_atomic_store(at + apart, v ^ tag, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ bool find_word(const unsigned long long* at, uint32_t apart, unsigned long long tag, unsigned long long& v) {
    v = __hip_atomic_load(at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return (v ^ __hip_atomic_load(at + apart, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)) == tag;
}
__device__ __forceinline__ void break_word(unsigned long long* at, uint32_t apart) {
    __hip_atomic_store(at, 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __hip_atomic_store(at + apart, 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void words_arrived() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// `slots` workgroups (kMostSlots at most) that add up K sums each, by their first waves: each leaves its own (lane 0's), and when they have arrived gathers everybody's, added up in
// the same order whoever does it; false where somebody is still to come. meet: [K][2][slots], and behind them for more than 64 slots [K][2][64]: then 16 or 64
// neighbours meet first, one of them - who takes the first pair apart - leaves their sum for the next meeting. (With everybody looking at everybody's words
// 256 slots take 14 us, their requests go to the same few places.)
constexpr uint32_t kMostSlots = 4096u;
__device__ __host__ constexpr uint32_t slot_group(uint32_t slots) { return slots <= 1024u ? 16u : 64u; }
template <int K>
__device__ __forceinline__ void leave_sums(unsigned long long* meet, uint32_t slots, uint32_t slot, const double (&sum)[K], unsigned long long tag) {
#pragma unroll
    for (uint32_t k = 0; k < K; ++k) leave_word(meet + static_cast<size_t>(2u * k) * slots + slot, slots, static_cast<unsigned long long>(__double_as_longlong(sum[k])), tag);
}
template <int K, bool ALONE>  // n slots (64 at most) from `first`; ALONE: one wave at most gets true
__device__ __forceinline__ bool take_sums(unsigned long long* meet, uint32_t slots, uint32_t first, uint32_t n, double (&sum)[K], unsigned long long tag) {
    const uint32_t lane = lane_id();
    auto word = [&](uint32_t k) { return meet + static_cast<size_t>(2u * k) * slots + first + lane; };
    bool here = true;
    unsigned long long v[K] = {};
    if (lane < n) {
#pragma unroll
        for (uint32_t k = 0; k < K; ++k) here = find_word(word(k), slots, tag, v[k]) && here;
    }
    if (__ballot(!here) != 0ull) return false;
    if (ALONE) {
        bool won = false;
        if (lane == 0u) {
            unsigned long long was = v[0] ^ tag;
            won = __hip_atomic_compare_exchange_strong(word(0u) + slots, &was, 0ull, __ATOMIC_RELAXED, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        if (__ballot(won) == 0ull) return false;
    }
    if (lane < n) {
#pragma unroll
        for (uint32_t k = 0; k < K; ++k) break_word(word(k), slots);
    }
#pragma unroll
    for (uint32_t k = 0; k < K; ++k) sum[k] = wave_sum(__longlong_as_double(static_cast<long long>(v[k])));
    return true;
}
template <int K>
__device__ __forceinline__ bool gather_sums(unsigned long long* meet, uint32_t slots, uint32_t slot, double (&sum)[K], unsigned long long tag) {
    if (slots <= 64u) return take_sums<K, false>(meet, slots, 0u, slots, sum, tag);
    const uint32_t group = slot_group(slots), g = slot / group, first = g * group;
    if (!take_sums<K, true>(meet, slots, first, min(group, slots - first), sum, tag)) return false;
    unsigned long long* next = meet + static_cast<size_t>(2 * K) * slots;
    if (lane_id() == 0u) leave_sums(next, 64u, g, sum, tag);
    words_arrived();
    return take_sums<K, false>(next, 64u, 0u, (slots + group - 1u) / group, sum, tag);
}

// a launch of `parts` workgroups a row: the parts in x, the rows in y and z (dispatched in this order, a row's parts one after the other)
constexpr uint32_t kGridRows = 32768u;
__device__ __forceinline__ uint32_t grid_row() { return blockIdx.z * kGridRows + blockIdx.y; }
// bytes of the words of `slots` workgroups that add up K sums
inline uint64_t sums_bytes(uint32_t slots, uint32_t K) { return slots < 2u ? 0u : (uint64_t{slots} + (slots > 64u ? 64u : 0u)) * K * 16u; }
inline dim3 grid_of(uint32_t parts, uint32_t rows) {
    return rows <= kGridRows ? dim3(parts, rows) : dim3(parts, kGridRows, (rows + kGridRows - 1u) / kGridRows);
}

// ---- a row's logits
template <int DT>
struct Elem {
    static constexpr uint32_t kBytes = DT == 0 ? 4u : 2u, kPer = 16u / kBytes;  // of a vector
    static constexpr uint32_t kNone = DT == 0 ? 0xff800000u : 0xff80ff80u;      // -inf
};

// a row as whole vectors between the 16-byte boundaries of `at`, numbered from the last boundary of 128 bytes before them ([first, end), so that 8 vectors of
// a round are one line, and the up to 2 (kPer - 1) logits before and behind them
template <int DT>
struct RowSpan {
    uint32_t head, first, end, rest;
    __device__ __forceinline__ RowSpan(const void* at, uint32_t V) {
        const uint32_t addr = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(at)), off = (16u - (addr & 15u)) & 15u;
        head = min(off / Elem<DT>::kBytes, V);
        first = ((addr + off) >> 4) & 7u;
        const uint32_t vectors = (V - head) / Elem<DT>::kPer;
        end = first + vectors;
        rest = V - vectors * Elem<DT>::kPer;
    }
    __device__ __forceinline__ uint32_t rest_index(uint32_t i) const { return i < head ? i : (end - first) * Elem<DT>::kPer + i; }
    __device__ __forceinline__ uint32_t index(uint32_t j) const { return head + (j - first) * Elem<DT>::kPer; }
    __device__ __forceinline__ bool has(uint32_t j) const { return j - first < end - first; }
};

__device__ __forceinline__ uint4 load_loose(const unsigned char* at) {
    const LooseVec v = *reinterpret_cast<const LooseVec*>(at);
    return make_uint4(v.x, v.y, v.z, v.w);
}
// a gradient's vector, `past` the caches or through them. (The first written out: the compiler makes one store of the two, the second. The pause is what the store's data registers
// need before they are written again, which the compiler sees to for its own stores.)
__device__ __forceinline__ void store_vector(unsigned char* at, const uint4& q, bool past) {
    typedef uint32_t four __attribute__((ext_vector_type(4)));
    const four v{q.x, q.y, q.z, q.w};
    if (past) asm volatile("global_store_dwordx4 %0, %1, off nt\n\ts_nop 1" ::"v"(at), "v"(v) : "memory");
    else *reinterpret_cast<four*>(at) = v;
}
template <int DT>
__device__ __forceinline__ float load_logit(const unsigned char* row, uint32_t i) {
    if constexpr (DT == 0) return reinterpret_cast<const float*>(row)[i];
    else return bf16_to_f32(reinterpret_cast<const uint16_t*>(row)[i]);
}
template <int DT>
__device__ __forceinline__ void unpack(const uint4& q, float (&x)[Elem<DT>::kPer]) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if constexpr (DT == 0) {
            x[k] = __uint_as_float(w[k]);
        } else {
            x[2 * k] = __uint_as_float(w[k] << 16);
            x[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
        }
    }
}
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {  // round to nearest even
    typedef __bf16 two_bf16 __attribute__((ext_vector_type(2)));
    typedef float two_f32 __attribute__((ext_vector_type(2)));
    const two_f32 f = {a, b};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f, two_bf16));
}
template <int DT>
__device__ __forceinline__ uint4 pack(const float (&x)[Elem<DT>::kPer]) {
    if constexpr (DT == 0) return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
    else return make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
}
template <int DT>
__device__ __forceinline__ void store_logit(unsigned char* row, uint32_t i, float v) {
    if constexpr (DT == 0) reinterpret_cast<float*>(row)[i] = v;
    else reinterpret_cast<uint16_t*>(row)[i] = static_cast<uint16_t>(pack_bf16(v, v));
}

// the row's bitmap: bit i, and the bits of a vector that begins at token i, from the two bytes that they lie in (or the row's last two). One load instead of two
// words': 200 masked rows of 50257 fp32 13.8 us, and 13.2.
struct __attribute__((packed, aligned(1))) LooseBits {
    uint16_t v;
};
__device__ __forceinline__ bool allowed(const uint32_t* allow, uint32_t i) { return (allow[i >> 5] >> (i & 31u)) & 1u; }
__device__ __forceinline__ uint32_t allowed_from(const uint32_t* allow, uint32_t i, uint32_t last_byte) {
    const uint32_t at = min(i >> 3, last_byte - 1u);
    return static_cast<uint32_t>(reinterpret_cast<const LooseBits*>(reinterpret_cast<const unsigned char*>(allow) + at)->v) >> (i - 8u * at);
}
// what is not allowed becomes -inf, whatever it was
template <int DT>
__device__ __forceinline__ uint4 only_allowed(const uint4& q, uint32_t bits) {
    uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        uint32_t keep;
        if constexpr (DT == 0) {
            keep = static_cast<uint32_t>(__builtin_amdgcn_sbfe(static_cast<int>(bits), static_cast<uint32_t>(k), 1u));
        } else {
            const uint32_t lo = static_cast<uint32_t>(__builtin_amdgcn_sbfe(static_cast<int>(bits), static_cast<uint32_t>(2 * k), 1u));
            const uint32_t hi = static_cast<uint32_t>(__builtin_amdgcn_sbfe(static_cast<int>(bits), static_cast<uint32_t>(2 * k + 1), 1u));
            keep = (lo & 0xffffu) | (hi & 0xffff0000u);
        }
        w[k] = (w[k] & keep) | (Elem<DT>::kNone & ~keep);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// the vectors [j0, j1) of a row that a workgroup works on, `base` where the row begins. Loads go to the nearest of them where a thread has none
// (a load behind a branch would be waited for there); what it read then counts as -inf.
template <int DT, bool MASK, int T>
struct Share {
    const unsigned char* base;
    const uint32_t* allow;
    RowSpan<DT> span;
    uint32_t last_byte, j0, j1;
    // part `part` of shares of `per` vectors
    __device__ __forceinline__ Share(const unsigned char* row, const uint32_t* mask, const RowSpan<DT>& s, uint32_t V, uint32_t part, uint32_t per)
        : base(row), allow(mask), span(s), last_byte(((V + 31u) >> 5) * 4u - 1u), j0(min(part * per, s.end)), j1(min(j0 + per, s.end)) {}
    __device__ __forceinline__ bool any() const { return j1 > max(j0, span.first); }
    // the vector as it is, and its bits of the mask: what is done with them waits for them
    __device__ __forceinline__ uint4 load(uint32_t j, uint32_t& bits) const {
        const uint32_t i = span.index(max(min(j, j1 - 1u), span.first));
        bits = 0u;
        if constexpr (MASK) bits = allowed_from(allow, i, last_byte);
        return load_loose(base + static_cast<size_t>(i) * Elem<DT>::kBytes);
    }
    __device__ __forceinline__ bool mine(uint32_t j) const { return j < j1 && j >= span.first; }
    // the vector of round jb .. jb + T, for a thread that may have none in it
    __device__ __forceinline__ uint4 own(uint4 q, uint32_t bits, uint32_t jb) const {
        constexpr uint32_t none = Elem<DT>::kNone;
        if constexpr (MASK) q = only_allowed<DT>(q, bits);
        if (jb + T <= j1 && jb >= span.first) return q;  // (uniform)
        return mine(jb + threadIdx.x) ? q : make_uint4(none, none, none, none);
    }
};

// ---- exponentials: (x - m) t log2(e), the factor as hi + lo with lo > 0 (so that a difference of -inf stays -inf)
struct Scale {
    float hi, lo;
    __device__ __forceinline__ explicit Scale(float inv_t) {
        const double c = static_cast<double>(inv_t) * 1.4426950408889634074;
        float h = static_cast<float>(c);
        if (static_cast<double>(h) >= c) h = __uint_as_float(__float_as_uint(h) - 1u);
        hi = inv_t > 0.f && inv_t < INFINITY ? h : __builtin_nanf("");  // (a temperature that is none makes the row NaN)
        lo = fmaxf(static_cast<float>(c - static_cast<double>(h)), 0x1p-149f);  // (the smallest there is: factors below 2^-102 have a second float as small)
    }
    __device__ __forceinline__ float of(float d) const { return fmaf(d, hi, __fmul_rn(d, lo)); }
};
__device__ __forceinline__ float exp2_fast(float a) { return __builtin_amdgcn_exp2f(a); }  // (below 2^-126: 0)
// two more values into a maximum. (Written out: of fmaxf the compiler makes another instruction a value, to quiet NaN.)
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}
constexpr float kFarBelow = -1000.f;  // an exponent whose power is 0: stands for -inf in products

// running maximum, sum of powers, sum of powers times exponents (base two, against the maximum). The maximum begins at the lowest
// number, not at -inf: a row of nothing but -inf has the sum 0, a row of nothing but the lowest number is a uniform one.
template <bool ENT>
struct Running {
    float m = -FLT_MAX, s = 0.f, t = 0.f;
    template <int N>
    __device__ __forceinline__ void take(const float (&x)[N], const Scale& c) {
        float M = m;
#pragma unroll
        for (int k = 0; k < N; k += 2) M = max3(M, x[k], x[k + 1]);
        move(M, c);
        float s0 = 0.f, s1 = 0.f, t0 = 0.f, t1 = 0.f;
#pragma unroll
        for (int k = 0; k < N; k += 2) {
            const float a = c.of(x[k] - M), b = c.of(x[k + 1] - M), ea = exp2_fast(a), eb = exp2_fast(b);
            s0 = __fadd_rn(s0, ea);
            s1 = __fadd_rn(s1, eb);
            if constexpr (ENT) {
                t0 = fmaf(ea, fmaxf(a, kFarBelow), t0);
                t1 = fmaf(eb, fmaxf(b, kFarBelow), t1);
            }
        }
        s = __fadd_rn(s, __fadd_rn(s0, s1));
        if constexpr (ENT) t = __fadd_rn(t, __fadd_rn(t0, t1));
    }
    __device__ __forceinline__ void take1(float x, const Scale& c) {
        const float two[2] = {x, -INFINITY};
        take(two, c);
    }
    // against the maximum M >= m
    __device__ __forceinline__ void move(float M, const Scale& c) {
        const float a = c.of(m - M), e = exp2_fast(a);
        if constexpr (ENT) t = __fmul_rn(e, fmaf(s, fmaxf(a, kFarBelow), t));
        s = __fmul_rn(s, e);
        m = M;
    }
};

// a row's sums, known: 64 bits from here on
struct RowSums {
    float m;
    double s, t;
};
struct RowValue {
    double lp, H;
    double rise;  // H - ln S
    bool any;     // some token is allowed
};
__device__ __forceinline__ RowValue row_value(const RowSums& r, float inv_t, bool has_id, float x_id) {
    RowValue v;
    v.any = !(r.s == 0.0);
    if (!v.any) {  // nothing is allowed: no token has a probability
        v.lp = has_id ? -static_cast<double>(INFINITY) : 0.0;
        v.H = v.rise = 0.0;
        return v;
    }
    const double lnS = log(r.s);
    v.lp = has_id ? (static_cast<double>(x_id) - static_cast<double>(r.m)) * static_cast<double>(inv_t) - lnS : 0.0;
    v.rise = -0.69314718055994530942 * (r.t / r.s);
    v.H = lnS + v.rise;
    return v;
}

// the block's sums from its threads', for the first wave (every lane)
template <bool ENT, int T>
__device__ __forceinline__ RowSums block_sums(Running<ENT>& a, const Scale& c, float* red_m, double* red_s, double* red_t) {
    a.move(wave_max(a.m), c);
    const double s = wave_sum(static_cast<double>(a.s));
    const double t = ENT ? wave_sum(static_cast<double>(a.t)) : 0.0;
    if (lane_id() == 0) {
        red_m[wave_id()] = a.m;
        red_s[wave_id()] = s;
        if (ENT) red_t[wave_id()] = t;
    }
    __syncthreads();
    RowSums r{-FLT_MAX, 0.0, 0.0};
    if (wave_id() != 0) return r;
    const uint32_t l = lane_id();
    const bool in = l < T / 64u;
    const float m = in ? red_m[l] : -FLT_MAX;
    r.m = wave_max(m);
    const float d = c.of(m - r.m);
    const double e = static_cast<double>(exp2_fast(d)), sw = in ? red_s[l] : 0.0;
    r.s = wave_sum(sw * e);
    if constexpr (ENT) r.t = wave_sum(e * ((in ? red_t[l] : 0.0) + sw * static_cast<double>(fmaxf(d, kFarBelow))));
    return r;
}

// ---- the parts of a row: what each leaves for the others, and what they make of it (in the order of the parts, whoever does). The sums in 64 bits:
// rounded to 32, a log-probability near the middle of two floats comes out as the other one in twenty, which adds up in the ratio of a long answer.
struct PartSums {
    float m, x;  // x: the logit of the row's token, from the part that has it
    double s, t;
};
constexpr uint32_t kPartWords = 6u;  // 64-bit words a part: three, each twice
// part p's words among those of `parts`: m and x, s, t (ENT)
template <bool ENT>
__device__ __forceinline__ void leave_part(unsigned long long* meet, uint32_t parts, uint32_t p, const PartSums& w, unsigned long long tag) {
    leave_word(meet + p, parts, (static_cast<unsigned long long>(__float_as_uint(w.x)) << 32) | __float_as_uint(w.m), tag);
    leave_word(meet + 2u * parts + p, parts, static_cast<unsigned long long>(__double_as_longlong(w.s)), tag);
    if (ENT) leave_word(meet + 4u * parts + p, parts, static_cast<unsigned long long>(__double_as_longlong(w.t)), tag);
}
template <bool ENT>
__device__ __forceinline__ bool find_part(const unsigned long long* meet, uint32_t parts, uint32_t p, unsigned long long tag, PartSums& w) {
    unsigned long long mx, s, t = 0ull;
    bool here = find_word(meet + p, parts, tag, mx);
    here = find_word(meet + 2u * parts + p, parts, tag, s) && here;
    if (ENT) here = find_word(meet + 4u * parts + p, parts, tag, t) && here;
    w = PartSums{__uint_as_float(static_cast<uint32_t>(mx)), __uint_as_float(static_cast<uint32_t>(mx >> 32)), __longlong_as_double(static_cast<long long>(s)),
                 __longlong_as_double(static_cast<long long>(t))};
    return here;
}
template <bool ENT>
__device__ __forceinline__ void break_part(unsigned long long* meet, uint32_t parts, uint32_t p) {
    break_word(meet + p, parts);
    break_word(meet + 2u * parts + p, parts);
    if (ENT) break_word(meet + 4u * parts + p, parts);
}
// a wave, a lane a part
template <bool ENT>
__device__ __forceinline__ RowSums join_parts(bool in, const PartSums& w, const Scale& c) {
    RowSums r{};
    const float m = in ? w.m : -FLT_MAX;
    const double s = in ? w.s : 0.0;
    r.m = wave_max(m);
    const float d = c.of(m - r.m);
    const double e = static_cast<double>(exp2_fast(d));
    r.s = wave_sum(s * e);
    if (ENT) r.t = wave_sum(e * ((in ? w.t : 0.0) + s * static_cast<double>(fmaxf(d, kFarBelow))));
    return r;
}

// ---- log-probabilities: a workgroup a row, or `parts` of them. The next four vectors of a thread are on their way while it works on four. What bounds it: memory, and of bf16 rows the vector units as
// much (7.8 instructions a logit, and some 200 a wave for its sums): 2048 x 151936 bf16 111 us = 5.6 TB/s, fp32 209 us = 5.95 TB/s.
struct ScoreArgs {
    LossRows R;
    float* logprob;
    float* stats;
    float* entropy;
    uint32_t parts, per;       // workgroups a row, vectors each
    unsigned long long* meet;  // parts > 1: [rows][kPartWords][parts], broken again by whoever joins them
    unsigned long long tag;
};

template <int DT, bool ENT, bool MASK, int T>
__global__ void __launch_bounds__(T) score_rows_kernel(ScoreArgs A) {
    constexpr uint32_t kPer = Elem<DT>::kPer, kU = 4u;  // vectors of a thread on their way together
    __shared__ float red_m[T / 64];
    __shared__ double red_s[T / 64], red_t[T / 64];
    uint32_t row = grid_row();
    if (row >= A.R.rows) return;
    row = A.R.rows - 1u - row;
    const uint32_t part = blockIdx.x, t = threadIdx.x, V = A.R.vocab;
    const unsigned char* base = A.R.logits + row * A.R.row_bytes;
    const RowSpan<DT> span(base, V);
    const Share<DT, MASK, T> share(base, MASK ? A.R.allow + row * A.R.allow_stride : nullptr, span, V, part, A.per);
    const uint32_t j0 = share.j0, j1 = share.any() ? share.j1 : share.j0;
    uint4 q[kU];
    uint32_t bits[kU];
    if (j0 < j1) {
#pragma unroll
        for (uint32_t u = 0; u < kU; ++u) q[u] = share.load(j0 + u * T + t, bits[u]);
    }
    // (the row's own entries come while its logits do)
    const int32_t id = A.R.ids ? A.R.ids[row] : -1;
    const bool has_id = static_cast<uint32_t>(id) < V;
    const float inv_t = A.R.inv_t ? A.R.inv_t[row] : 1.f;
    float x_id = -INFINITY;
    if (t < 64u && has_id && (!MASK || allowed(share.allow, static_cast<uint32_t>(id)))) x_id = load_logit<DT>(base, static_cast<uint32_t>(id));
    const Scale c(inv_t);
    Running<ENT> a;
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
        if (!MASK || allowed(share.allow, i)) a.take1(load_logit<DT>(base, i), c);
    }
    RowSums r = block_sums<ENT, T>(a, c, red_m, red_s, red_t);
    if (t >= 64u) return;
    if (A.parts > 1u) {  // (at most 64)
        unsigned long long* meet = A.meet + static_cast<size_t>(row) * A.parts * kPartWords;
        if (t == 0u) leave_part<ENT>(meet, A.parts, part, PartSums{r.m, 0.f, r.s, r.t}, A.tag);
        words_arrived();
        const bool in = t < A.parts;
        PartSums w{};
        const bool here = !in || find_part<ENT>(meet, A.parts, t, A.tag, w);
        if (__ballot(!here) != 0ull) return;  // somebody is still to come
        if (in) break_part<ENT>(meet, A.parts, t);
        r = join_parts<ENT>(in, w, c);
    }
    if (t != 0u) return;
    const RowValue v = row_value(r, inv_t, has_id, x_id);
    A.stats[2 * static_cast<size_t>(row)] = !v.any ? -INFINITY : (r.s == r.s ? r.m : static_cast<float>(r.s));  // (NaN is not the largest of anything)
    A.stats[2 * static_cast<size_t>(row) + 1] = static_cast<float>(r.s);
    A.logprob[row] = static_cast<float>(v.lp);
    if (ENT) A.entropy[row] = static_cast<float>(v.H);
}

// ---- the gradient: two vectors a thread and no more, so that many workgroups are at different stages (four: 1024 x 151936 bf16, a quarter of the rows without derivatives, 101 us, two: 90; one: 106, three: 93;
// all past the caches). Memory bounds it: 5.8 TB/s there.
struct GradArgs {
    LossRows R;
    const float* stats;
    const float* entropy;
    const float* d_logprob;
    const float* d_entropy;
    unsigned char* out;
    uint64_t out_bytes;  // between rows
    uint32_t past_row;   // from this row on the gradient goes past the caches
};

// what a row's derivatives need: dx = e (a + b d) with e = 2^d, d = (x - m) t log2(e), and g t more at the row's token
struct RowSlope {
    float m, a, b, at_id;
    bool none;
};
template <bool ENT>
__device__ __forceinline__ RowSlope row_slope(float m, float S, float inv_t, float g, float h, float rise) {  // rise: H - ln S
    RowSlope r;
    r.m = m;
    r.none = (g == 0.f && (!ENT || h == 0.f)) || S == 0.f;
    // v t / S, the factor below 1 last: one that leaves the floats' range on the way would lose bits there
    const float share = -1.f / S;
    auto factor = [&](float v) { return inv_t < 1.f ? v * share * inv_t : inv_t * share * v; };
    // held so that a + b d, |d| <= 1000 where it counts, is finite: an infinity times a power of 0 would be NaN, in every masked place
    auto held = [](float v, float most) { return fabsf(v) > most ? copysignf(most, v) : v; };
    const float h_held = held(h, 0x1p100f);
    r.a = held(factor(ENT ? fmaf(h_held, rise, held(g, FLT_MAX)) : g), 0x1p126f);
    r.b = ENT ? held(factor(h_held) * 0.69314718f, 0x1p112f) : 0.f;
    r.at_id = g * inv_t;
    return r;
}
// bf16 results take the exponent with the factor's first float alone, which is rounded down: a power is up to 2^-23 ln 2 |d| of itself too large - a thousandth of the results' half step of
// 2^-8 where the power is 2^-48 and more, a four hundredth at the smallest - for an instruction a logit less (4096 x 262144 747 us, and 740). A factor rounded to nearest takes another register, and the masked
// build with entropy spills it.
template <int DT, bool ENT>
__device__ __forceinline__ float slope_at(float x, const RowSlope& r, const Scale& c) {
    const float d = DT == 0 ? c.of(x - r.m) : __fmul_rn(x - r.m, c.hi), e = exp2_fast(d);
    return e * (ENT ? fmaf(r.b, fmaxf(d, kFarBelow), r.a) : r.a);
}
template <int DT, bool ENT>
__device__ __forceinline__ uint4 slope_vector(const uint4& q, uint32_t first, const RowSlope& r, const Scale& c, uint32_t id) {
    constexpr uint32_t kPer = Elem<DT>::kPer;
    float x[kPer], y[kPer];
    unpack<DT>(q, x);
#pragma unroll
    for (uint32_t k = 0; k < kPer; ++k) y[k] = slope_at<DT, ENT>(x[k], r, c);
    if (id - first < kPer) {
#pragma unroll
        for (uint32_t k = 0; k < kPer; ++k)
            if (id - first == k && x[k] != -INFINITY) y[k] += r.at_id;
    }
    return pack<DT>(y);
}

template <int DT, bool ENT, bool MASK, int T, int U>
__global__ void __launch_bounds__(T) grad_rows_kernel(GradArgs A) {
    uint32_t row = grid_row();
    if (row >= A.R.rows) return;
    row = A.R.rows - 1u - row;
    const bool past = row >= A.past_row;
    const uint32_t chunk = blockIdx.x, t = threadIdx.x, V = A.R.vocab;
    const unsigned char* base = A.R.logits + row * A.R.row_bytes;
    unsigned char* out = A.out + row * A.out_bytes;
    const RowSpan<DT> span(out, V);
    const uint32_t* allow = MASK ? A.R.allow + row * A.R.allow_stride : nullptr;
    const Share<DT, MASK, T> share(base, allow, span, V, 0u, span.end);
    const float inv_t = A.R.inv_t ? A.R.inv_t[row] : 1.f;
    const int32_t id = A.R.ids ? A.R.ids[row] : -1;
    const bool has_id = static_cast<uint32_t>(id) < V;
    const Scale c(inv_t);
    const float S = A.stats[2 * static_cast<size_t>(row) + 1];
    const RowSlope r = row_slope<ENT>(A.stats[2 * static_cast<size_t>(row)], S, inv_t, has_id && A.d_logprob ? A.d_logprob[row] : 0.f, ENT ? A.d_entropy[row] : 0.f,
                                      ENT ? A.entropy[row] - __logf(S) : 0.f);
    const uint32_t j0 = chunk * (T * U) + t;
    auto store = [&](uint32_t j, const uint4& q) { store_vector(out + static_cast<size_t>(span.index(j)) * Elem<DT>::kBytes, q, past); };
    if (r.none) {  // (uniform) not read
#pragma unroll
        for (uint32_t u = 0; u < U; ++u)
            if (span.has(j0 + u * T)) store(j0 + u * T, make_uint4(0u, 0u, 0u, 0u));
        if (chunk == 0u && t < span.rest) store_logit<DT>(out, span.rest_index(t), 0.f);
        return;
    }
    uint4 q[U];
    uint32_t bits[U];
    if (share.any()) {
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) q[u] = share.load(j0 + u * T, bits[u]);
    }
    if (chunk == 0u && t < span.rest) {
        const uint32_t i = span.rest_index(t);
        const float x = !MASK || allowed(allow, i) ? load_logit<DT>(base, i) : -INFINITY;
        float y = slope_at<DT, ENT>(x, r, c);
        if (i == static_cast<uint32_t>(id) && x != -INFINITY) y += r.at_id;
        store_logit<DT>(out, i, y);
    }
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {
        const uint32_t j = j0 + u * T;
        if (span.has(j)) {
            if constexpr (MASK) q[u] = only_allowed<DT>(q[u], bits[u]);
            store(j, slope_vector<DT, ENT>(q[u], span.index(j), r, c, static_cast<uint32_t>(id)));
        }
    }
}

// ---- the policy loss from logits to its gradient in one pass: the parts of a row (one, or up to 64 workgroups) keep their share in registers, NV vectors
// a thread, leave their sums for each other, wait for the others' and write the share's gradient. The wait is bounded, since nothing says
// that all parts run at once: a part that does not find another's words in time works that part's sums out itself, in the
// same order and so to the same bits. (Where the gradient goes over the logits: a part writes only after its words have arrived. So logits
// read before a look that still finds no words are the logits, and the token's logit goes with the words, not to be read
// by a part that comes late.) The words stay until every part has seen them: where the rows' terms meet in this launch too (`terms` is NULL), the parts leave a mark each when they are
// through, and whoever sees all marks of a row breaks its words; else a second launch adds up the terms and breaks the words.
// What bounds it: memory, and the vector units at 80 to 85 % (16.7 instructions a logit, 23.6 with entropy and its gradient). 2048 x 151936 bf16 with entropy, a fifth of the rows not counting, 215 to
// 220 us = 5.3 TB/s; 4096 x 262144 750 to 780 us = 5.7 TB/s; a row in one workgroup of 1024 threads, what its registers do not hold read twice, 282 and 988. Shares of 11, 14, 16 or 19 vectors a thread are up to 8 % slower, workgroups of 512
// threads 10 to 20 %: a unit then holds fewer of them, and fewer are at another stage than their neighbours.
struct RowsArgs {
    LossRows R;
    PolicyIn P;
    float* logprob;
    float* entropy;
    unsigned char* out;
    uint64_t out_bytes;
    uint32_t past_row;  // as GradArgs
    double* terms;             // [kPolicySums][rows], or:
    unsigned long long* sums_meet;  // [kPolicySums][2][rows] and, of more than 64, [kPolicySums][2][64]: for rows that meet in this launch
    float* sums;
    uint32_t parts, per;       // workgroups a row, vectors each
    unsigned long long* meet;  // parts > 1: [rows][kPartWords][parts]; of rows that meet in this launch [rows][kPartWords + 2][parts], the last two the parts' marks
    unsigned long long tag;
    uint32_t looks;  // for the other parts' words, a microsecond each
};

template <int DT, bool ENT, bool SLOPE, bool MASK, int T, int NV, int WAVES>  // WAVES: a SIMD's at least
__global__ void __launch_bounds__(T, WAVES) policy_rows_kernel(RowsArgs A) {
    constexpr uint32_t kPer = Elem<DT>::kPer;
    __shared__ float red_m[T / 64];
    __shared__ double red_s[T / 64], red_t[T / 64];
    __shared__ RowSlope shared_slope;
    __shared__ unsigned long long missing;
    __shared__ PartSums found[64];
    uint32_t row = grid_row();
    if (row >= A.R.rows) return;
    row = A.R.rows - 1u - row;
    const bool past = row >= A.past_row;
    const uint32_t part = blockIdx.x, t = threadIdx.x, V = A.R.vocab, per = A.per;
    const unsigned char* base = A.R.logits + row * A.R.row_bytes;
    unsigned char* out = A.out + row * A.out_bytes;
    const RowSpan<DT> span(out, V);
    const uint32_t* allow = MASK ? A.R.allow + row * A.R.allow_stride : nullptr;
    const Share<DT, MASK, T> share(base, allow, span, V, part, per);
    const uint32_t j0 = share.j0, j1 = share.any() ? share.j1 : share.j0;
    const int32_t id = A.R.ids[row];
    const bool has_id = static_cast<uint32_t>(id) < V;
    const double weight = policy_weight(A.P, row);
    const bool rest = part == 0u && t < span.rest;
    const uint32_t rest_i = rest ? span.rest_index(t) : 0u;
    auto store = [&](uint32_t j, const uint4& q) { store_vector(out + static_cast<size_t>(span.index(j)) * Elem<DT>::kBytes, q, past); };
    auto nothing = [&]() {
        for (uint32_t j = j0 + t; j < j1; j += T)
            if (j >= span.first) store(j, make_uint4(0u, 0u, 0u, 0u));
        if (rest) store_logit<DT>(out, rest_i, 0.f);
    };
    unsigned long long* meet = A.meet + static_cast<size_t>(row) * A.parts * (A.terms ? kPartWords : kPartWords + 2u);
    double terms[kPolicySums] = {};
    auto leave_terms = [&]() {  // the row's, by the first thread of its first part
        if (!A.terms) {
            if (A.R.rows > 1u) leave_sums(A.sums_meet, A.R.rows, row, terms, A.tag);
            return;
        }
#pragma unroll
        for (uint32_t k = 0; k < kPolicySums; ++k) A.terms[static_cast<size_t>(k) * A.R.rows + row] = terms[k];
    };
    auto finish = [&]() {  // by its first wave, when everything else is done
        if (A.terms || (A.R.rows > 1u && !gather_sums(A.sums_meet, A.R.rows, row, terms, A.tag))) return;
#pragma unroll
        for (uint32_t k = 0; k < kPolicySums; ++k)
            if (t == 0u) A.sums[k] = static_cast<float>(terms[k]);
    };
    if (!has_id || weight == 0.0) {  // (uniform) counts for nothing: not read
        if (part == 0u && t == 0u) {
            A.logprob[row] = 0.f;
            if (A.entropy) A.entropy[row] = 0.f;
            leave_terms();
        }
        nothing();
        if (part == 0u && t < 64u) {
            words_arrived();
            finish();
        }
        return;
    }
    uint4 q[NV];
    uint32_t bits[NV];
    if (j0 < j1) {
#pragma unroll
        for (int k = 0; k < NV; ++k)
            if (k == 0 || j0 + k * T < j1) q[k] = share.load(j0 + k * T + t, bits[k]);  // (uniform)
    }
    float x_rest = -INFINITY;
    if (rest && (!MASK || allowed(allow, rest_i))) x_rest = load_logit<DT>(base, rest_i);
    const float inv_t = A.R.inv_t ? A.R.inv_t[row] : 1.f;
    // the part that has the row's token, and its logit
    const uint32_t id_at = (static_cast<uint32_t>(id) - span.head) / kPer + span.first;
    const uint32_t id_part = static_cast<uint32_t>(id) >= span.head && id_at < span.end ? id_at / per : 0u;
    auto token_logit = [&]() { return !MASK || allowed(allow, static_cast<uint32_t>(id)) ? load_logit<DT>(base, static_cast<uint32_t>(id)) : -INFINITY; };
    PolicyRow token{};
    float x_id = 0.f;
    if (t < 64u) {  // (uniform for the wave)
        token = policy_row(A.P, row);
        if (part == id_part) x_id = token_logit();
    }
    const Scale c(inv_t);
    Running<ENT> a;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        if (j0 + k * T < j1) {  // (uniform)
            float x[kPer];
            q[k] = share.own(q[k], bits[k], j0 + k * T);
            unpack<DT>(q[k], x);
            a.take(x, c);
        }
    }
    if (rest) a.take1(x_rest, c);
    RowSums r = block_sums<ENT, T>(a, c, red_m, red_s, red_t);
    if (A.parts > 1u) {
        if (t < 64u) {
            if (t == 0u) leave_part<ENT>(meet, A.parts, part, PartSums{r.m, x_id, r.s, r.t}, A.tag);
            words_arrived();
            const bool in = t < A.parts;
            PartSums w{};
            bool here = !in;
            for (uint32_t look = 0; look < A.looks; ++look) {
                if (!here) here = find_part<ENT>(meet, A.parts, t, A.tag, w);
                if (__ballot(!here) == 0ull) break;
                __builtin_amdgcn_s_sleep(4);
            }
            const unsigned long long late = __ballot(!here);
            found[t] = w;
            if (t == 0u) missing = late;
        }
        __syncthreads();
        for (unsigned long long late = missing; late; late &= late - 1ull) {  // (uniform)
            const uint32_t p = static_cast<uint32_t>(__ffsll(late) - 1);
            const Share<DT, MASK, T> theirs(base, allow, span, V, p, per);
            Running<ENT> b;
            for (uint32_t jb = theirs.j0; theirs.any() && jb < theirs.j1; jb += T) {
                float x[kPer];
                uint32_t bits_late;
                const uint4 late_q = theirs.load(jb + t, bits_late);
                unpack<DT>(theirs.own(late_q, bits_late, jb), x);
                b.take(x, c);
            }
            if (p == 0u && t < span.rest) {
                const uint32_t i = span.rest_index(t);
                b.take1(!MASK || allowed(allow, i) ? load_logit<DT>(base, i) : -INFINITY, c);
            }
            const float x_late = t == 0u && p == id_part ? token_logit() : 0.f;
            __syncthreads();
            const RowSums o = block_sums<ENT, T>(b, c, red_m, red_s, red_t);
            if (t == 0u) {  // (everybody's logits have come: the barrier in block_sums)
                PartSums w{o.m, x_late, o.s, o.t}, came{};
                words_arrived();
                if (find_part<ENT>(meet, A.parts, p, A.tag, came)) w = came;
                found[p] = w;
            }
        }
        if (t < 64u) {
            __builtin_amdgcn_wave_barrier();  // (one wave: its LDS stores are done before its loads)
            r = join_parts<ENT>(t < A.parts, found[t], c);
            x_id = found[id_part].x;
            if (t == 0u && !A.terms) leave_word(meet + kPartWords * A.parts + part, A.parts, 0ull, A.tag);  // (the mark)
        }
    }
    if (t == 0u) {
        const RowValue v = row_value(r, inv_t, true, x_id);
        const PolicyToken o = policy_token(A.P, token, v.lp, ENT ? v.H : 0.0);
        shared_slope = row_slope<SLOPE>(r.m, static_cast<float>(r.s), inv_t, static_cast<float>(o.g), static_cast<float>(o.h),
                                        static_cast<float>(v.rise));  // (the difference of H and ln S as floats: 1e-6 off where an even row has 0)
        if (part == 0u) {
            A.logprob[row] = static_cast<float>(v.lp);
            if (ENT) A.entropy[row] = static_cast<float>(v.H);
#pragma unroll
            for (uint32_t k = 0; k < kPolicySums; ++k) terms[k] = o.sum[k];
            leave_terms();
        }
    }
    __syncthreads();
    const RowSlope s = shared_slope;
    if (s.none) {  // (uniform)
        nothing();
    } else {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const uint32_t j = j0 + k * T + t;
            if (share.mine(j)) store(j, slope_vector<DT, SLOPE>(q[k], span.index(j), s, c, static_cast<uint32_t>(id)));
        }
        if (rest) {
            float y = slope_at<DT, SLOPE>(x_rest, s, c);
            if (rest_i == static_cast<uint32_t>(id) && x_rest != -INFINITY) y += s.at_id;
            store_logit<DT>(out, rest_i, y);
        }
    }
    if (t >= 64u || A.terms) return;
    words_arrived();
    if (A.parts > 1u) {
        unsigned long long* marks = meet + kPartWords * A.parts;
        unsigned long long mark;
        const bool in = t < A.parts, here = !in || find_word(marks + t, A.parts, A.tag, mark);
        if (__ballot(!here) == 0ull && in) {  // everybody is through
            break_part<ENT>(meet, A.parts, t);
            break_word(marks + t, A.parts);
        }
    }
    if (part == 0u) finish();
}

// ---- the loss over log-probabilities, or the sum of rows' terms: the workgroups' sums meet
struct PolicyArgs {
    PolicyIn P;
    uint32_t rows;
    const float* logprob;
    const float* entropy;
    const double* terms;  // [kPolicySums][rows]: worked out already (then only they are read, and only the sums written)
    float* d_logprob;
    float* d_entropy;
    float* sums;
    unsigned long long* meet;  // [kPolicySums][2][workgroups] and, of more than 64, [kPolicySums][2][64]
    unsigned long long tag;
    unsigned long long* words;  // the rows' parts' words, to be broken
    uint64_t n_words;
};

template <int T>
__global__ void __launch_bounds__(T) policy_kernel(PolicyArgs A) {
    __shared__ double red[kPolicySums][T / 64];
    const uint32_t t = threadIdx.x, groups = gridDim.x;
    for (uint64_t i = static_cast<uint64_t>(blockIdx.x) * T + t; i < A.n_words; i += static_cast<uint64_t>(groups) * T) A.words[i] = 0ull;
    double sum[kPolicySums] = {};
    for (uint32_t row = blockIdx.x * T + t; row < A.rows; row += groups * T) {
        if (A.terms) {
#pragma unroll
            for (uint32_t k = 0; k < kPolicySums; ++k) sum[k] += A.terms[static_cast<size_t>(k) * A.rows + row];
            continue;
        }
        const PolicyRow token = policy_row(A.P, row);
        const double lp = static_cast<double>(A.logprob[row]), H = A.entropy ? static_cast<double>(A.entropy[row]) : 0.0;
        PolicyToken o{};
        if (token.weight != 0.0) o = policy_token(A.P, token, lp, H);
        A.d_logprob[row] = static_cast<float>(o.g);
        if (A.d_entropy) A.d_entropy[row] = static_cast<float>(o.h);
#pragma unroll
        for (uint32_t k = 0; k < kPolicySums; ++k) sum[k] += o.sum[k];
    }
#pragma unroll
    for (uint32_t k = 0; k < kPolicySums; ++k) {
        const double s = wave_sum(sum[k]);
        if (lane_id() == 0) red[k][wave_id()] = s;
    }
    __syncthreads();
    if (t >= 64u) return;
#pragma unroll
    for (uint32_t k = 0; k < kPolicySums; ++k) sum[k] = wave_sum(t < T / 64u ? red[k][t] : 0.0);
    if (groups > 1u) {
        if (t == 0u) leave_sums(A.meet, groups, blockIdx.x, sum, A.tag);
        words_arrived();
        if (!gather_sums(A.meet, groups, blockIdx.x, sum, A.tag)) return;
    }
    if (t == 0u) {
#pragma unroll
        for (uint32_t k = 0; k < kPolicySums; ++k) A.sums[k] = static_cast<float>(sum[k]);
    }
}

// ---- paired log ratios: a workgroup a pair (or several, one after the other), the pairs' losses meet
struct PreferenceArgs {
    uint32_t rows, pairs;
    const uint32_t* seq_off;
    const float* logprob;
    const float* ref_logprob;
    const float* weight;
    double weight_all, beta, smoothing;
    float* loss;
    float* pair_loss;
    float* reward;
    float* d_logprob;
    unsigned long long* meet;  // [2][workgroups]
    unsigned long long tag;
};

template <int T>
__global__ void __launch_bounds__(T) preference_kernel(PreferenceArgs A) {
    __shared__ double red[2][T / 64];
    __shared__ float slope;
    __shared__ bool again;
    const uint32_t t = threadIdx.x, groups = gridDim.x;
    double mine = 0.0;
    for (uint32_t p = blockIdx.x; p < A.pairs; p += groups) {
        uint32_t at[3];  // the chosen answer is [at0, at1), the other [at1, at2); offsets past the rows end there
#pragma unroll
        for (uint32_t k = 0; k < 3u; ++k) at[k] = min(A.seq_off[2u * p + k], A.rows);
        // A token that neither model can give counts for nothing. It makes its answer's sum NaN (-inf - -inf), and only where one is
        // are such tokens looked for, in a second pass. (Looked for in the first: 64 pairs of answers of up to 2048 tokens 7.3 us, and 7.1.)
        auto neither = [&](uint32_t row) { return A.logprob[row] == -INFINITY && A.ref_logprob && A.ref_logprob[row] == -INFINITY; };
        bool skip = false;
        while (true) {  // (twice at most)
            double s[2] = {0.0, 0.0};
            if (!skip) {
#pragma unroll
                for (uint32_t k = 0; k < 2u; ++k)
                    for (uint32_t row = at[k] + t; row < at[k + 1u]; row += T) s[k] += static_cast<double>(A.logprob[row]) - (A.ref_logprob ? static_cast<double>(A.ref_logprob[row]) : 0.0);
            } else {
#pragma unroll
                for (uint32_t k = 0; k < 2u; ++k)
                    for (uint32_t row = at[k] + t; row < at[k + 1u]; row += T) s[k] += neither(row) ? 0.0 : static_cast<double>(A.logprob[row]) - static_cast<double>(A.ref_logprob[row]);
            }
#pragma unroll
            for (uint32_t k = 0; k < 2u; ++k) {
                s[k] = wave_sum(s[k]);
                if (lane_id() == 0) red[k][wave_id()] = s[k];
            }
            __syncthreads();
            if (t < 64u) {
#pragma unroll
                for (uint32_t k = 0; k < 2u; ++k) s[k] = wave_sum(t < T / 64u ? red[k][t] : 0.0);
                const bool look = !skip && A.ref_logprob && (s[0] != s[0] || s[1] != s[1]);
                const double w = A.weight ? static_cast<double>(A.weight[p]) : A.weight_all, h = A.beta * (s[0] - s[1]);
                const double tail = log1p(exp(-fabs(h)));  // of both ln(1 + exp(+-h)) what the larger of +-h and 0 leaves
                // a term of factor 0 is left out: the other answer's sum may be -inf, and 0 times the term's infinity NaN
                const double loss = (A.smoothing != 1.0 ? (1.0 - A.smoothing) * (fmax(-h, 0.0) + tail) : 0.0) + (A.smoothing != 0.0 ? A.smoothing * (fmax(h, 0.0) + tail) : 0.0);
                if (w != 0.0 && !look) mine += w * loss;
                if (t == 0u) {
                    A.pair_loss[p] = static_cast<float>(loss);
                    A.reward[2u * static_cast<size_t>(p)] = static_cast<float>(A.beta * s[0]);
                    A.reward[2u * static_cast<size_t>(p) + 1u] = static_cast<float>(A.beta * s[1]);
                    slope = w != 0.0 ? static_cast<float>(w * A.beta * (A.smoothing - 1.0 / (1.0 + exp(h)))) : 0.f;
                    again = look;
                }
            }
            __syncthreads();
            if (!again) break;
            skip = true;
        }
        const float c = slope;
        for (uint32_t row = at[0] + t; row < at[2]; row += T) A.d_logprob[row] = skip && neither(row) ? 0.f : (row < at[1] ? c : -c);
    }
    // rows of no answer: before the first, behind the last
    const uint32_t first = min(A.seq_off[0], A.rows), behind = min(A.seq_off[2u * A.pairs], A.rows);
    for (uint32_t row = blockIdx.x * T + t; row < first; row += groups * T) A.d_logprob[row] = 0.f;
    for (uint32_t row = behind + blockIdx.x * T + t; row < A.rows; row += groups * T) A.d_logprob[row] = 0.f;
    if (t >= 64u) return;
    double sum[1] = {mine};
    if (groups > 1u) {
        if (t == 0u) leave_sums(A.meet, groups, blockIdx.x, sum, A.tag);
        words_arrived();
        if (!gather_sums(A.meet, groups, blockIdx.x, sum, A.tag)) return;
    }
    if (t == 0u) A.loss[0] = static_cast<float>(sum[0]);
}

}  // namespace ws
