// Log-probabilities of given tokens, the losses over them and the gradients with respect to the logits.
//
// A row of logits x with inverse temperature t and allowed set L (all tokens without a mask): m = max x_v, S = sum over L of
// exp((x_v - m) t), p_v = exp((x_v - m) t) / S. The token y of the row has log p_y = (x_y - m) t - ln S, the row the entropy
// H = ln S - (1 / S) sum exp(d_v) d_v with d_v = (x_v - m) t. With g = dF/d(log p_y) and h = dF/dH of any loss F
//     dF/dx_v = t [ g (1[v = y] - p_v) - h p_v (ln p_v + H) ].
// Both directions are one pass over the row: forwards every thread keeps a maximum, a sum and (for H) a sum of products that are
// scaled down when its maximum grows, backwards every logit gives its own derivative. Exponentials go to base two with the factor
// t log2(e) split in two floats (a rounded one alone would move every exponent the same way, 1e-6 of a sum); sums are held
// in 32 bits by a thread, over some hundred terms, and in 64 bits from the wave on; ln S, log p and the loss of a token in 64 bits.
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

__device__ __forceinline__ double policy_weight(const PolicyIn& P, uint32_t row) { return P.weight ? static_cast<double>(P.weight[row]) : P.weight_all; }

// gain = min(r A, clip(r) A) with r = exp(lp - old); for A < 0 not below dual_clip * A. Where the clip holds it there is no
// derivative, so the comparison is made in 64 bits: rounded to 32, one token in some million would fall on the other side.
__device__ __forceinline__ PolicyToken policy_token(const PolicyIn& P, uint32_t row, double w, double lp, double H) {
    PolicyToken o;
    const double A = static_cast<double>(P.advantage[row]), r = exp(lp - static_cast<double>(P.old_logprob[row]));
    const double free = r * A, held = fmin(fmax(r, 1.0 - P.clip_low), 1.0 + P.clip_high) * A;
    double gain = held < free ? held : free;
    bool clipped = held < free;
    if (P.dual_clip > 0.0 && A < 0.0 && gain < P.dual_clip * A) {
        gain = P.dual_clip * A;
        clipped = true;
    }
    double kl = 0.0, back = 0.0;
    if (P.ref_logprob) {  // exp(b) - b - 1 with b = ref - lp, never negative
        const double b = static_cast<double>(P.ref_logprob[row]) - lp;
        back = expm1(b);
        kl = back - b;
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
// write the same. The pairs are then broken, for a captured launch has its tag again at every replay.
__device__ __forceinline__ void leave_word(unsigned long long* at, unsigned long long v, unsigned long long tag) {
    __hip_atomic_store(at, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __hip_atomic_store(at + 1, v ^ tag, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ bool find_word(const unsigned long long* at, unsigned long long tag, unsigned long long& v) {
    v = __hip_atomic_load(at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return (v ^ __hip_atomic_load(at + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)) == tag;
}
__device__ __forceinline__ void break_word(unsigned long long* at) {
    __hip_atomic_store(at, 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __hip_atomic_store(at + 1, 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void words_arrived() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// ---- a row's logits
template <int DT>
struct Elem {
    static constexpr uint32_t kBytes = DT == 0 ? 4u : 2u, kPer = 16u / kBytes;  // of a vector
    static constexpr uint32_t kNone = DT == 0 ? 0xff800000u : 0xff80ff80u;      // -inf
};

// a row as whole vectors between the 16-byte boundaries of `at`, and the up to 2 (kPer - 1) logits before and behind them
template <int DT>
struct RowSpan {
    uint32_t head, vectors, rest;
    __device__ __forceinline__ RowSpan(const void* at, uint32_t V) {
        const uint32_t off = (16u - (static_cast<uint32_t>(reinterpret_cast<uintptr_t>(at)) & 15u)) & 15u;
        head = min(off / Elem<DT>::kBytes, V);
        vectors = (V - head) / Elem<DT>::kPer;
        rest = V - vectors * Elem<DT>::kPer;
    }
    __device__ __forceinline__ uint32_t rest_index(uint32_t i) const { return i < head ? i : vectors * Elem<DT>::kPer + i; }
    __device__ __forceinline__ uint32_t index(uint32_t j) const { return head + j * Elem<DT>::kPer; }
};

__device__ __forceinline__ uint4 load_loose(const unsigned char* at) {
    const LooseVec v = *reinterpret_cast<const LooseVec*>(at);
    return make_uint4(v.x, v.y, v.z, v.w);
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

// the row's bitmap: bit i, and the bits of a vector that begins at token i (it may lie across two words)
__device__ __forceinline__ bool allowed(const uint32_t* allow, uint32_t i) { return (allow[i >> 5] >> (i & 31u)) & 1u; }
__device__ __forceinline__ uint32_t allowed_from(const uint32_t* allow, uint32_t i, uint32_t last_word) {
    const uint32_t w = i >> 5;
    return __builtin_amdgcn_alignbit(allow[min(w + 1u, last_word)], allow[w], i & 31u);
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

// ---- exponentials: (x - m) t log2(e), the factor as hi + lo with lo > 0 (so that a difference of -inf stays -inf)
struct Scale {
    float hi, lo;
    __device__ __forceinline__ explicit Scale(float inv_t) {
        const double c = static_cast<double>(inv_t) * 1.4426950408889634074;
        float h = static_cast<float>(c);
        if (static_cast<double>(h) >= c) h = __uint_as_float(__float_as_uint(h) - 1u);
        hi = inv_t > 0.f && inv_t < INFINITY ? h : __builtin_nanf("");  // (a temperature that is none makes the row NaN)
        lo = fmaxf(static_cast<float>(c - static_cast<double>(h)), FLT_MIN);
    }
    __device__ __forceinline__ float of(float d) const { return fmaf(d, hi, d * lo); }
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
            s0 += ea;
            s1 += eb;
            if constexpr (ENT) {
                t0 = fmaf(ea, fmaxf(a, kFarBelow), t0);
                t1 = fmaf(eb, fmaxf(b, kFarBelow), t1);
            }
        }
        s += s0 + s1;
        if constexpr (ENT) t += t0 + t1;
    }
    __device__ __forceinline__ void take1(float x, const Scale& c) {
        const float two[2] = {x, -INFINITY};
        take(two, c);
    }
    // against the maximum M >= m
    __device__ __forceinline__ void move(float M, const Scale& c) {
        const float a = c.of(m - M), e = exp2_fast(a);
        if constexpr (ENT) t = e * fmaf(s, fmaxf(a, kFarBelow), t);
        s *= e;
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
    bool any;  // some token is allowed
};
__device__ __forceinline__ RowValue row_value(const RowSums& r, float inv_t, bool has_id, float x_id) {
    RowValue v;
    v.any = !(r.s == 0.0);
    if (!v.any) {  // nothing is allowed: no token has a probability
        v.lp = has_id ? -static_cast<double>(INFINITY) : 0.0;
        v.H = 0.0;
        return v;
    }
    const double lnS = log(r.s);
    v.lp = has_id ? (static_cast<double>(x_id) - static_cast<double>(r.m)) * static_cast<double>(inv_t) - lnS : 0.0;
    v.H = lnS - 0.69314718055994530942 * (r.t / r.s);
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

// ---- log-probabilities: a workgroup a row, or `parts` of them
struct ScoreArgs {
    LossRows R;
    float* logprob;
    float* stats;
    float* entropy;
    uint32_t parts;
    unsigned long long* meet;  // parts > 1: [rows][parts][4 or 2] words
    unsigned long long tag;
    // with a policy loss
    PolicyIn P;
    float* d_logprob;
    float* d_entropy;
    double* terms;  // [rows][kPolicySums]
};

template <bool POLICY>
__device__ __forceinline__ void write_row(const ScoreArgs& A, uint32_t row, const RowSums& r, float inv_t, bool has_id, float x_id) {
    const RowValue v = row_value(r, inv_t, has_id, x_id);
    A.stats[2 * static_cast<size_t>(row)] = v.any ? r.m : -INFINITY;
    A.stats[2 * static_cast<size_t>(row) + 1] = static_cast<float>(r.s);
    A.logprob[row] = static_cast<float>(v.lp);
    if (A.entropy) A.entropy[row] = static_cast<float>(v.H);
    if constexpr (POLICY) {
        const PolicyToken o = policy_token(A.P, row, policy_weight(A.P, row), v.lp, A.entropy ? v.H : 0.0);
        A.d_logprob[row] = static_cast<float>(o.g);
        if (A.d_entropy) A.d_entropy[row] = static_cast<float>(o.h);
#pragma unroll
        for (uint32_t k = 0; k < kPolicySums; ++k) A.terms[static_cast<size_t>(row) * kPolicySums + k] = o.sum[k];
    }
}
// a row that counts for nothing
__device__ __forceinline__ void write_no_row(const ScoreArgs& A, uint32_t row) {
    A.logprob[row] = 0.f;
    if (A.entropy) A.entropy[row] = 0.f;
    if (A.d_logprob) A.d_logprob[row] = 0.f;
    if (A.d_entropy) A.d_entropy[row] = 0.f;
#pragma unroll
    for (uint32_t k = 0; k < kPolicySums; ++k) A.terms[static_cast<size_t>(row) * kPolicySums + k] = 0.0;
}

template <int DT, bool ENT, bool MASK, bool POLICY, int T>
__global__ void __launch_bounds__(T) score_rows_kernel(ScoreArgs A) {
    constexpr uint32_t kPer = Elem<DT>::kPer, kU = 4u;  // vectors of a thread on their way together
    __shared__ float red_m[T / 64];
    __shared__ double red_s[T / 64], red_t[T / 64];
    const uint32_t row = blockIdx.x / A.parts, part = blockIdx.x % A.parts, t = threadIdx.x, V = A.R.vocab;
    const int32_t id = A.R.ids ? A.R.ids[row] : -1;
    const bool has_id = static_cast<uint32_t>(id) < V;
    if constexpr (POLICY) {
        if (!has_id || policy_weight(A.P, row) == 0.0) {  // (uniform)
            if (part == 0u && t == 0u) write_no_row(A, row);
            return;
        }
    }
    const unsigned char* base = A.R.logits + row * A.R.row_bytes;
    const uint32_t* allow = MASK ? A.R.allow + row * A.R.allow_stride : nullptr;
    const uint32_t last_word = (V - 1u) >> 5;
    const float inv_t = A.R.inv_t ? A.R.inv_t[row] : 1.f;
    float x_id = -INFINITY;
    if (has_id && (!MASK || allowed(allow, static_cast<uint32_t>(id)))) x_id = load_logit<DT>(base, static_cast<uint32_t>(id));
    const Scale c(inv_t);
    const RowSpan<DT> span(base, V);
    const uint32_t per = (span.vectors + A.parts - 1u) / A.parts, j0 = min(part * per, span.vectors), j1 = min(j0 + per, span.vectors);
    Running<ENT> a;
    auto get = [&](uint32_t j) {
        uint4 q = *reinterpret_cast<const uint4*>(base + static_cast<size_t>(span.index(j)) * Elem<DT>::kBytes);
        if constexpr (MASK) q = only_allowed<DT>(q, allowed_from(allow, span.index(j), last_word));
        return q;
    };
    uint32_t j = j0 + t;
    for (; j + (kU - 1u) * T < j1; j += kU * T) {
        uint4 q[kU];
#pragma unroll
        for (uint32_t u = 0; u < kU; ++u) q[u] = get(j + u * T);
#pragma unroll
        for (uint32_t u = 0; u < kU; ++u) {
            float x[kPer];
            unpack<DT>(q[u], x);
            a.take(x, c);
        }
    }
    for (; j < j1; j += T) {
        float x[kPer];
        unpack<DT>(get(j), x);
        a.take(x, c);
    }
    if (part == 0u && t < span.rest) {
        const uint32_t i = span.rest_index(t);
        if (!MASK || allowed(allow, i)) a.take1(load_logit<DT>(base, i), c);
    }
    RowSums r = block_sums<ENT, T>(a, c, red_m, red_s, red_t);
    if (t >= 64u) return;
    if (A.parts > 1u) {  // (at most 64)
        constexpr uint32_t kWords = ENT ? 2u : 1u;
        unsigned long long* meet = A.meet + static_cast<size_t>(row) * A.parts * (2u * kWords);
        auto word = [&](uint32_t p, uint32_t k) { return meet + (p * kWords + k) * 2u; };
        if (t == 0u) {
            const float s = static_cast<float>(r.s);
            leave_word(word(part, 0u), (static_cast<unsigned long long>(__float_as_uint(s)) << 32) | __float_as_uint(r.m), A.tag);
            if (ENT) leave_word(word(part, kWords - 1u), static_cast<unsigned long long>(__double_as_longlong(r.t)), A.tag);
        }
        words_arrived();
        const bool in = t < A.parts;
        unsigned long long ms = 0ull, tt = 0ull;
        bool here = true;
        if (in) {
            here = find_word(word(t, 0u), A.tag, ms);
            if (ENT) here = find_word(word(t, kWords - 1u), A.tag, tt) && here;
        }
        if (__ballot(!here) != 0ull) return;  // somebody is still to come
        if (in) {
            break_word(word(t, 0u));
            if (ENT) break_word(word(t, kWords - 1u));
        }
        const float m = in ? __uint_as_float(static_cast<uint32_t>(ms)) : -FLT_MAX;
        const double s = in ? static_cast<double>(__uint_as_float(static_cast<uint32_t>(ms >> 32))) : 0.0;
        r.m = wave_max(m);
        const float d = c.of(m - r.m);
        const double e = static_cast<double>(exp2_fast(d));
        r.s = wave_sum(s * e);
        if (ENT) r.t = wave_sum(e * ((in ? __longlong_as_double(static_cast<long long>(tt)) : 0.0) + s * static_cast<double>(fmaxf(d, kFarBelow))));
    }
    if (t == 0u) write_row<POLICY>(A, row, r, inv_t, has_id, x_id);
}

// ---- the gradient
struct GradArgs {
    LossRows R;
    const float* stats;
    const float* entropy;
    const float* d_logprob;
    const float* d_entropy;
    unsigned char* out;
    uint64_t out_bytes;  // between rows
    uint32_t chunks;     // workgroups a row
};

// what a row's derivatives need: dx = e (a + b d) with e = 2^d, d = (x - m) t log2(e), and g t more at the row's token
struct RowSlope {
    float m, a, b, at_id;
    bool none;
};
template <bool ENT>
__device__ __forceinline__ RowSlope row_slope(float m, float S, float inv_t, float g, float h, float H) {
    RowSlope r;
    r.m = m;
    r.none = (g == 0.f && (!ENT || h == 0.f)) || S == 0.f;
    const float f = -inv_t / S;
    r.a = f * (ENT ? fmaf(h, H - __logf(S), g) : g);
    r.b = ENT ? f * h * 0.69314718f : 0.f;
    r.at_id = g * inv_t;
    return r;
}
template <bool ENT>
__device__ __forceinline__ float slope_at(float x, const RowSlope& r, const Scale& c) {
    const float d = c.of(x - r.m), e = exp2_fast(d);
    return e * (ENT ? fmaf(r.b, fmaxf(d, kFarBelow), r.a) : r.a);
}
template <int DT, bool ENT>
__device__ __forceinline__ uint4 slope_vector(const uint4& q, uint32_t first, const RowSlope& r, const Scale& c, uint32_t id) {
    constexpr uint32_t kPer = Elem<DT>::kPer;
    float x[kPer], y[kPer];
    unpack<DT>(q, x);
#pragma unroll
    for (uint32_t k = 0; k < kPer; ++k) y[k] = slope_at<ENT>(x[k], r, c);
    if (id - first < kPer) {
#pragma unroll
        for (uint32_t k = 0; k < kPer; ++k)
            if (id - first == k && x[k] != -INFINITY) y[k] += r.at_id;
    }
    return pack<DT>(y);
}

template <int DT, bool ENT, bool MASK, int T, int U>
__global__ void __launch_bounds__(T) grad_rows_kernel(GradArgs A) {
    const uint32_t row = blockIdx.x / A.chunks, chunk = blockIdx.x % A.chunks, t = threadIdx.x, V = A.R.vocab;
    const unsigned char* base = A.R.logits + row * A.R.row_bytes;
    unsigned char* out = A.out + row * A.out_bytes;
    const RowSpan<DT> span(out, V);
    const uint32_t* allow = MASK ? A.R.allow + row * A.R.allow_stride : nullptr;
    const uint32_t last_word = (V - 1u) >> 5;
    const float inv_t = A.R.inv_t ? A.R.inv_t[row] : 1.f;
    const int32_t id = A.R.ids ? A.R.ids[row] : -1;
    const bool has_id = static_cast<uint32_t>(id) < V;
    const Scale c(inv_t);
    const RowSlope r = row_slope<ENT>(A.stats[2 * static_cast<size_t>(row)], A.stats[2 * static_cast<size_t>(row) + 1], inv_t,
                                      has_id && A.d_logprob ? A.d_logprob[row] : 0.f, ENT ? A.d_entropy[row] : 0.f, ENT ? A.entropy[row] : 0.f);
    const uint32_t j0 = chunk * (T * U) + t;
    auto store = [&](uint32_t j, const uint4& q) { *reinterpret_cast<uint4*>(out + static_cast<size_t>(span.index(j)) * Elem<DT>::kBytes) = q; };
    if (r.none) {  // (uniform) not read
#pragma unroll
        for (uint32_t u = 0; u < U; ++u)
            if (j0 + u * T < span.vectors) store(j0 + u * T, make_uint4(0u, 0u, 0u, 0u));
        if (chunk == 0u && t < span.rest) store_logit<DT>(out, span.rest_index(t), 0.f);
        return;
    }
    uint4 q[U];
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {
        const uint32_t j = j0 + u * T;
        if (j < span.vectors) {
            q[u] = load_loose(base + static_cast<size_t>(span.index(j)) * Elem<DT>::kBytes);
            if constexpr (MASK) q[u] = only_allowed<DT>(q[u], allowed_from(allow, span.index(j), last_word));
        }
    }
    if (chunk == 0u && t < span.rest) {
        const uint32_t i = span.rest_index(t);
        const float x = !MASK || allowed(allow, i) ? load_logit<DT>(base, i) : -INFINITY;
        float y = slope_at<ENT>(x, r, c);
        if (i == static_cast<uint32_t>(id) && x != -INFINITY) y += r.at_id;
        store_logit<DT>(out, i, y);
    }
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {
        const uint32_t j = j0 + u * T;
        if (j < span.vectors) store(j, slope_vector<DT, ENT>(q[u], span.index(j), r, c, static_cast<uint32_t>(id)));
    }
}

// ---- the policy loss from logits to its gradient, a workgroup a row: what of the row the registers hold (NV vectors a thread) is read
// once, the rest of a longer row a second time.
struct RowsArgs {
    ScoreArgs S;
    unsigned char* out;
    uint64_t out_bytes;
};
template <int DT, bool ENT, bool SLOPE, bool MASK, int T, int NV>
__global__ void __launch_bounds__(T) policy_rows_kernel(RowsArgs B) {
    constexpr uint32_t kPer = Elem<DT>::kPer;
    __shared__ float red_m[T / 64];
    __shared__ double red_s[T / 64], red_t[T / 64];
    __shared__ RowSlope shared_slope;
    const ScoreArgs& A = B.S;
    const uint32_t row = blockIdx.x, t = threadIdx.x, V = A.R.vocab;
    const unsigned char* base = A.R.logits + row * A.R.row_bytes;
    unsigned char* out = B.out + row * B.out_bytes;
    const RowSpan<DT> span(out, V);
    const int32_t id = A.R.ids[row];
    const bool has_id = static_cast<uint32_t>(id) < V;
    auto store = [&](uint32_t j, const uint4& q) { *reinterpret_cast<uint4*>(out + static_cast<size_t>(span.index(j)) * Elem<DT>::kBytes) = q; };
    auto nothing = [&]() {
        for (uint32_t j = t; j < span.vectors; j += T) store(j, make_uint4(0u, 0u, 0u, 0u));
        if (t < span.rest) store_logit<DT>(out, span.rest_index(t), 0.f);
    };
    if (!has_id || policy_weight(A.P, row) == 0.0) {  // (uniform) not read
        nothing();
        if (t == 0u) write_no_row(A, row);
        return;
    }
    const uint32_t* allow = MASK ? A.R.allow + row * A.R.allow_stride : nullptr;
    const uint32_t last_word = (V - 1u) >> 5;
    const float inv_t = A.R.inv_t ? A.R.inv_t[row] : 1.f;
    auto get = [&](uint32_t j) {
        uint4 q = load_loose(base + static_cast<size_t>(span.index(j)) * Elem<DT>::kBytes);
        if constexpr (MASK) q = only_allowed<DT>(q, allowed_from(allow, span.index(j), last_word));
        return q;
    };
    uint4 q[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const uint32_t j = k * T + t;
        q[k] = make_uint4(Elem<DT>::kNone, Elem<DT>::kNone, Elem<DT>::kNone, Elem<DT>::kNone);
        if (j < span.vectors) q[k] = get(j);
    }
    float x_id = -INFINITY;
    if (t == 0u && (!MASK || allowed(allow, static_cast<uint32_t>(id)))) x_id = load_logit<DT>(base, static_cast<uint32_t>(id));
    float x_rest = -INFINITY;
    if (t < span.rest) {
        const uint32_t i = span.rest_index(t);
        if (!MASK || allowed(allow, i)) x_rest = load_logit<DT>(base, i);
    }
    const Scale c(inv_t);
    Running<ENT> a;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        if (k * T < span.vectors) {  // (uniform)
            float x[kPer];
            unpack<DT>(q[k], x);
            a.take(x, c);
        }
    }
    for (uint32_t j = NV * T + t; j < span.vectors; j += T) {
        float x[kPer];
        unpack<DT>(get(j), x);
        a.take(x, c);
    }
    if (t < span.rest) a.take1(x_rest, c);
    const RowSums r = block_sums<ENT, T>(a, c, red_m, red_s, red_t);
    if (t == 0u) {
        const RowValue v = row_value(r, inv_t, true, x_id);
        A.logprob[row] = static_cast<float>(v.lp);
        if (A.entropy) A.entropy[row] = static_cast<float>(v.H);
        const PolicyToken o = policy_token(A.P, row, policy_weight(A.P, row), v.lp, ENT ? v.H : 0.0);
#pragma unroll
        for (uint32_t k = 0; k < kPolicySums; ++k) A.terms[static_cast<size_t>(row) * kPolicySums + k] = o.sum[k];
        shared_slope = row_slope<SLOPE>(r.m, static_cast<float>(r.s), inv_t, static_cast<float>(o.g), static_cast<float>(o.h), static_cast<float>(v.H));
    }
    __syncthreads();
    const RowSlope s = shared_slope;
    if (s.none) {
        nothing();
        return;
    }
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const uint32_t j = k * T + t;
        if (j < span.vectors) store(j, slope_vector<DT, SLOPE>(q[k], span.index(j), s, c, static_cast<uint32_t>(id)));
    }
    for (uint32_t j = NV * T + t; j < span.vectors; j += T) store(j, slope_vector<DT, SLOPE>(get(j), span.index(j), s, c, static_cast<uint32_t>(id)));
    if (t < span.rest) {
        const uint32_t i = span.rest_index(t);
        float y = slope_at<SLOPE>(x_rest, s, c);
        if (i == static_cast<uint32_t>(id) && x_rest != -INFINITY) y += s.at_id;
        store_logit<DT>(out, i, y);
    }
}

// ---- sums of a batch's tokens: at most 64 workgroups, whose partial sums meet
struct PolicyArgs {
    PolicyIn P;
    uint32_t rows;
    const float* logprob;
    const float* entropy;
    const double* terms;  // the rows' terms, already worked out (then nothing else is read or written but the sums)
    float* d_logprob;
    float* d_entropy;
    float* sums;
    unsigned long long* meet;  // [workgroups][kPolicySums][2]
    unsigned long long tag;
};

template <int T>
__global__ void __launch_bounds__(T) policy_kernel(PolicyArgs A) {
    __shared__ double red[kPolicySums][T / 64];
    const uint32_t t = threadIdx.x, groups = gridDim.x;
    double sum[kPolicySums] = {};
    for (uint32_t row = blockIdx.x * T + t; row < A.rows; row += groups * T) {
        if (A.terms) {
#pragma unroll
            for (uint32_t k = 0; k < kPolicySums; ++k) sum[k] += A.terms[static_cast<size_t>(row) * kPolicySums + k];
            continue;
        }
        const double w = policy_weight(A.P, row);
        PolicyToken o{};
        if (w != 0.0) o = policy_token(A.P, row, w, static_cast<double>(A.logprob[row]), A.entropy ? static_cast<double>(A.entropy[row]) : 0.0);
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
        auto word = [&](uint32_t p, uint32_t k) { return A.meet + (static_cast<size_t>(p) * kPolicySums + k) * 2u; };
        if (t == 0u) {
#pragma unroll
            for (uint32_t k = 0; k < kPolicySums; ++k) leave_word(word(blockIdx.x, k), static_cast<unsigned long long>(__double_as_longlong(sum[k])), A.tag);
        }
        words_arrived();
        bool here = true;
        unsigned long long v[kPolicySums] = {};
        if (t < groups) {
#pragma unroll
            for (uint32_t k = 0; k < kPolicySums; ++k) here = find_word(word(t, k), A.tag, v[k]) && here;
        }
        if (__ballot(!here) != 0ull) return;
        if (t < groups) {
#pragma unroll
            for (uint32_t k = 0; k < kPolicySums; ++k) break_word(word(t, k));
        }
#pragma unroll
        for (uint32_t k = 0; k < kPolicySums; ++k) sum[k] = wave_sum(t < groups ? __longlong_as_double(static_cast<long long>(v[k])) : 0.0);
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
    unsigned long long* meet;  // [workgroups][2]
    unsigned long long tag;
};
__device__ __forceinline__ double softplus(double v) { return fmax(v, 0.0) + log1p(exp(-fabs(v))); }

template <int T>
__global__ void __launch_bounds__(T) preference_kernel(PreferenceArgs A) {
    __shared__ double red[2][T / 64];
    __shared__ float slope;
    const uint32_t t = threadIdx.x, groups = gridDim.x;
    double mine = 0.0;
    for (uint32_t p = blockIdx.x; p < A.pairs; p += groups) {
        uint32_t at[3];  // the chosen answer is [at0, at1), the other [at1, at2); offsets past the rows end there
#pragma unroll
        for (uint32_t k = 0; k < 3u; ++k) at[k] = min(A.seq_off[2u * p + k], A.rows);
        double s[2] = {0.0, 0.0};
#pragma unroll
        for (uint32_t k = 0; k < 2u; ++k)
            for (uint32_t row = at[k] + t; row < at[k + 1u]; row += T) s[k] += static_cast<double>(A.logprob[row]) - (A.ref_logprob ? static_cast<double>(A.ref_logprob[row]) : 0.0);
#pragma unroll
        for (uint32_t k = 0; k < 2u; ++k) {
            s[k] = wave_sum(s[k]);
            if (lane_id() == 0) red[k][wave_id()] = s[k];
        }
        __syncthreads();
        if (t < 64u) {
#pragma unroll
            for (uint32_t k = 0; k < 2u; ++k) s[k] = wave_sum(t < T / 64u ? red[k][t] : 0.0);
            const double w = A.weight ? static_cast<double>(A.weight[p]) : A.weight_all, h = A.beta * (s[0] - s[1]);
            const double loss = (1.0 - A.smoothing) * softplus(-h) + A.smoothing * softplus(h);
            if (w != 0.0) mine += w * loss;
            if (t == 0u) {
                A.pair_loss[p] = static_cast<float>(loss);
                A.reward[2u * static_cast<size_t>(p)] = static_cast<float>(A.beta * s[0]);
                A.reward[2u * static_cast<size_t>(p) + 1u] = static_cast<float>(A.beta * s[1]);
                slope = w != 0.0 ? static_cast<float>(w * A.beta * (A.smoothing - 1.0 / (1.0 + exp(h)))) : 0.f;
            }
        }
        __syncthreads();
        const float c = slope;
        for (uint32_t row = at[0] + t; row < at[2]; row += T) A.d_logprob[row] = row < at[1] ? c : -c;
    }
    // rows of no answer: before the first, behind the last
    const uint32_t first = min(A.seq_off[0], A.rows), behind = min(A.seq_off[2u * A.pairs], A.rows);
    for (uint32_t row = blockIdx.x * T + t; row < first; row += groups * T) A.d_logprob[row] = 0.f;
    for (uint32_t row = behind + blockIdx.x * T + t; row < A.rows; row += groups * T) A.d_logprob[row] = 0.f;
    if (t >= 64u) return;
    if (groups > 1u) {
        if (t == 0u) leave_word(A.meet + 2u * blockIdx.x, static_cast<unsigned long long>(__double_as_longlong(mine)), A.tag);
        words_arrived();
        bool here = true;
        double all = 0.0;
        for (uint32_t p = t; p < groups; p += 64u) {
            unsigned long long v;
            here = find_word(A.meet + 2u * p, A.tag, v) && here;
            all += __longlong_as_double(static_cast<long long>(v));
        }
        if (__ballot(!here) != 0ull) return;
        for (uint32_t p = t; p < groups; p += 64u) break_word(A.meet + 2u * p);
        mine = wave_sum(all);
    }
    if (t == 0u) A.loss[0] = static_cast<float>(mine);
}

}  // namespace ws
