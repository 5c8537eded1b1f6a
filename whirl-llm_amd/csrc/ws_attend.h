// Attention of the rows of trees over a paged cache: out_r = sum_t p_rt v_t, p = softmax of scale q_r . k_t over the positions t that row r sees.
//
// The rows of a sequence that read the same kv head - its nodes times the heads of a group - are the columns of S^T = K Q^T and of O^T = V^T P^T, both products on the matrix cores with
// sums in 32 bits. So a column's softmax lies in the lanes that hold it: its maximum and sum never cross to other lanes but where a maximum grows, and P^T is the
// second product's operand where the first one leaves it. Of V a lane takes 8 tokens' neighbouring elements, which two permutes a pair of tokens turn into 8 tokens of an element.
//
// One pass: a column keeps its maximum, sum and O^T; powers are of base two, and a column is scaled down only when a lane's eight powers against the maximum so far make more than kMost (32 bits
// hold what is larger than one as exactly): else no maximum is looked for. A wave works on 32 positions at a time. Few columns (WM = 1): the four waves of a workgroup take different positions, K and V go from memory
// into the registers of their operands. Many (WM = 4): the waves take different columns of the same positions; K and V go from memory straight into LDS, the next ones' while these are worked on, and
// bf16's V is turned by the instruction that reads it from there.
//
// Work: units of kUnit positions of a sequence, a kv head and a tile of columns; the workgroups share them evenly, whatever the sequences' lengths, each a run of neighbours (AttendSpan).
// A run that does not hold all units of a tile leaves maximum, sum and O^T in the workspace, and attend_join_kernel joins them.
//
// What bounds it. Few columns: memory (64 rows over 4096 positions at most, 32 heads, 8 of K and V, 128 bf16: 575 MB in 120 us, 4.8 TB/s). Many (2 x 64 nodes over 131072, 32 heads, 4 of K and V: 206 GFLOP in 270 to 346 us,
// 600 to 760 TFLOP/s; a matrix product of 8192^3 reaches 1207): matrix cores 34 % and vector units 44 % busy, each wave waiting for its own products, LDS and barriers in turn, and the clock, which the card
// lowers from 2.15 to 1.8 GHz in launches one behind the other. Tried there and not faster: 8 waves and 256 columns a workgroup (360 us of then 357); three buffers instead of two (385); K of
// the next 32 positions read while these are added up (356 to 383); 64 columns a wave (680).
#pragma once

#include "ws_common.h"
#include "ws_cycle.h"

#include <float.h>

#include <type_traits>

namespace ws {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr uint32_t kAttendThreads = 256u;
constexpr float kMost = 256.f;

// 16 lanes' 8 bytes each in LDS, 4 by 16 elements of 16 bits, the other way round
__device__ __forceinline__ u32x2 turned(const unsigned char* at) {
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)at));
}

// 16 bytes a lane from memory into LDS, 1024 neighbouring bytes a wave
__device__ __forceinline__ void to_lds(const unsigned char* from, unsigned char* wave_to) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from, (__attribute__((address_space(3))) void*)wave_to, 16, 0, 0);
}

// a type's operands and their products
template <int DT>
struct Mat;
template <>
struct Mat<1> {  // bf16
    static constexpr uint32_t kBytes = 2u, kPer = 8u, kDepth = 32u;  // elements of a 16-byte load, depth of a product
    typedef bf16x8 Frag;
    static __device__ __forceinline__ f32x4 mul(const uint4& a, const uint4& b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
    // eight tokens' element e, in a word each, times their powers
    static __device__ __forceinline__ f32x4 mul_tokens(const uint32_t (&word)[8], uint32_t e, const uint4 (&p)[1], f32x4 c) {
        const uint32_t half = e % 2u ? 0x07060302u : 0x05040100u;
        return mul(make_uint4(__builtin_amdgcn_perm(word[1], word[0], half), __builtin_amdgcn_perm(word[3], word[2], half), __builtin_amdgcn_perm(word[5], word[4], half),
                              __builtin_amdgcn_perm(word[7], word[6], half)), p[0], c);
    }
    // all bits of the elements of a word that are infinities or NaN: an exponent of ones and one more carry into the sign's place
    static __device__ __forceinline__ uint32_t special(uint32_t w) {
        const uint32_t f = ((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
        return (f - (f >> 15)) | f;
    }
    static __device__ __forceinline__ float element(const unsigned char* at, uint32_t i) { return bf16_to_f32(reinterpret_cast<const uint16_t*>(at)[i]); }
};
template <>
struct Mat<0> {  // fp32: four products of depth 4, lane group g's i-th element in the i-th
    static constexpr uint32_t kBytes = 4u, kPer = 4u, kDepth = 16u;
    static __device__ __forceinline__ f32x4 mul(const uint4& a, const uint4& b, f32x4 c) {
        const uint32_t x[4] = {a.x, a.y, a.z, a.w}, y[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(x[i]), __uint_as_float(y[i]), c, 0, 0, 0);
        return c;
    }
    static __device__ __forceinline__ f32x4 mul_tokens(const uint32_t (&word)[8], uint32_t, const uint4 (&p)[2], f32x4 c) {
        c = mul(make_uint4(word[0], word[1], word[2], word[3]), p[0], c);
        return mul(make_uint4(word[4], word[5], word[6], word[7]), p[1], c);
    }
    static __device__ __forceinline__ uint32_t special(uint32_t w) {
        const uint32_t f = ((w & 0x7f800000u) + 0x00800000u) & 0x80000000u;
        return (f - (f >> 31)) | f;
    }
    static __device__ __forceinline__ float element(const unsigned char* at, uint32_t i) { return reinterpret_cast<const float*>(at)[i]; }
};

// The larger of two, as the middle of them and infinity. (Of fmaxf the compiler makes another instruction a value, to quiet NaN; inline assembly may not read what the matrix cores have
// just written: the compiler does not see to the pause that takes.)
__device__ __forceinline__ float larger(float a, float b) { return __builtin_amdgcn_fmed3f(a, b, INFINITY); }

// A build: DT, DP (head_dim rounded up to 64, 128 or 256), MS tiles of 16 columns a wave, WM waves over columns (4 / WM over positions)
template <int DT, int DP, int MS, int WM>
struct AttendShape {
    static constexpr uint32_t kTileCols = 16u * MS * WM;
    static constexpr bool kTurned = DT == 1 && WM > 1;  // V is turned by its reads from LDS: a lane asks for 4 elements of a token and gets 4 tokens' of an element
    static constexpr uint32_t kEach = kTurned ? 1u : 16u / Mat<DT>::kBytes;  // elements of V a lane loads together: a lane holds elements kEach c + e of a block of 16 kEach
    static constexpr uint32_t kBlocks = DP / (16u * kEach);
    static constexpr uint32_t kOuts = kBlocks * kEach;                 // products' results that make up O^T of 16 columns, 4 floats a lane each
    static constexpr uint32_t kChunks = DP / Mat<DT>::kDepth;
    static constexpr uint32_t kSubFloats = 64u * (4u * kOuts + 2u);    // of 16 columns in the workspace: maximum and sum, O^T, as the lanes hold them
    static constexpr uint32_t kPartFloats = MS * WM * kSubFloats;
    // through LDS: bytes of a token, tokens at a time (32 where 64 would take the registers that two tiles of columns need: 128 columns of 128 bf16 151 us instead of 163), a token's 16-byte
    // pieces, those of a thread
    static constexpr uint32_t kRow = DP * Mat<DT>::kBytes, kTokens = kRow * MS <= 256u ? 64u : 32u, kPieces = kRow / 16u, kMine = kTokens * kPieces / 256u;
    static constexpr uint32_t kBuffer = kTokens * kRow;
    // positions that work is counted in: what a workgroup's waves take together
    static constexpr uint32_t kUnit = WM > 1 ? kTokens : 128u;
    // A token's pieces lie in another order for each of 16 neighbours, so that a piece of all of them, which K's operand takes together, lies in different banks, and a pair of pieces of 8 of them,
    // which half a wave takes of V.
    static __device__ __forceinline__ uint32_t order(uint32_t token) {
        return (kPieces == 8u ? token & 6u : (token & 7u) << 1) | (token >> 3 & 1u);
    }
    // the piece of a token that the at-th place holds
    static __device__ __forceinline__ uint32_t piece(uint32_t at) { return (at % kPieces) ^ order(at / kPieces); }
    static __device__ __forceinline__ uint32_t place(uint32_t token, uint32_t piece) { return token * kRow + (piece ^ order(token)) * 16u; }
};

// which of four positions from `pos` on a row sees: those before `length` and the nodes behind, by its bits. (A select a position, position < length ? true : bit, has been compiled
// to the bit alone.)
__device__ __forceinline__ uint32_t sees_four(uint64_t sees, uint32_t pos, uint32_t length) {
    const int32_t behind = static_cast<int32_t>(pos) - static_cast<int32_t>(length);  // (both below 2^31)
    const uint32_t before = static_cast<uint32_t>(min(max(-behind, 0), 4));           // of the four
    const uint32_t nodes = behind >= 0 ? (behind < 64 ? static_cast<uint32_t>(sees >> behind) : 0u) : static_cast<uint32_t>(sees) << before;
    return ((1u << before) - 1u) | (nodes & 15u);
}

struct AttendWork {  // a sequence's
    uint32_t first, nodes, total, length, tiles, units;  // row, nodes, positions, those before the nodes, tiles of columns, units of a tile
    uint64_t all;                                        // units of all heads and tiles
};
__device__ __forceinline__ AttendWork attend_work(const AttendArgs& A, uint32_t s, uint32_t cols, uint32_t unit) {
    AttendWork w;
    const uint32_t a = min(A.seq_off[s], A.rows), b = min(A.seq_off[s + 1u], A.rows);
    w.first = a;
    w.nodes = b > a ? min(b - a, kTreeNodes) : 0u;
    const uint64_t room = static_cast<uint64_t>(A.slot_pages) << A.page_shift;  // (below 2^31)
    w.length = A.length[s];
    w.total = static_cast<uint32_t>(min(static_cast<uint64_t>(w.length) + w.nodes, room));
    w.tiles = (w.nodes * A.group + cols - 1u) / cols;
    w.units = max((w.total + unit - 1u) / unit, 1u);
    w.all = static_cast<uint64_t>(w.tiles) * A.kv_heads * w.units;
    return w;
}

// exclusive prefix over the workgroup's 256 threads
__device__ __forceinline__ uint64_t scan256(uint64_t v, uint64_t* red, uint64_t& total) {
    const uint64_t inc = wave_incl_scan(v);
    __syncthreads();
    if (lane_id() == 63) red[wave_id()] = inc;
    __syncthreads();
    uint64_t base = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const uint64_t x = red[w];
        if (w < wave_id()) base += x;
        total += x;
    }
    return base + inc - v;
}

struct AttendFind {
    uint64_t red[4];
    uint64_t seq_first;  // the first unit of sequence `seq`, which holds the one that is looked for
    uint32_t seq;
    AttendWork work;
};
// What a workgroup works on. All units in a row, sequences behind one another, a head's tiles behind one another, in runs of `per`, that do not end at sequences; or, in gangs: where sequences have
// several tiles, these read the same K and V, so that as many runs as a sequence has tiles, `apart` in number, take the same positions, each of its own tile, at the same time and on one part of
// the chip: what one has read the others find in its cache (2 x 64 nodes, 512 columns, over 131072: without, K and V came from memory 3.5 times). Then runs end at sequences, which leaves
// some a little shorter than others: taken where sequences are few.
struct AttendSpan {
    uint64_t per, begin, end;  // units; from the first of all, or of the sequence's
    uint32_t tile, apart;      // of a gang: the run's tile
    bool gang;
};
// A sequence a thread, 256 at a time. False: there is nothing for this run.
template <bool GANGS>
__device__ __forceinline__ bool attend_find(const AttendArgs& A, uint32_t cols, uint32_t unit, uint32_t run, AttendFind& F, AttendSpan& S) {
    const uint32_t t = threadIdx.x;
    uint64_t mine = 0, tiles = 0, all = 0, all_tiles = 0;
    AttendWork w{};
    for (uint32_t s = t; s < A.n_seq; s += kAttendThreads) {
        w = attend_work(A, s, cols, unit);
        mine += w.all;
        tiles += w.tiles;
    }
    uint64_t before = scan256(mine, F.red, all);
    if (GANGS) scan256(tiles, F.red, all_tiles);
    S.gang = GANGS && all_tiles > A.n_seq && all_tiles <= A.groups / 8u;  // (so that there are fewer sequences than threads)
    const uint64_t runs = A.groups - (S.gang ? all_tiles : 0u);
    S.per = max((all + runs - 1u) / runs, uint64_t{1});  // (two units at least: one row over 4096 positions 15.4 us instead of 11.5, four 20.6; the join 5.4 and 5.0 instead of 6.8)
    uint64_t at = S.per * run;
    if (S.gang) {  // each sequence has as many runs as it needs: all_tiles more than an even split at most
        mine = w.tiles * ((static_cast<uint64_t>(A.kv_heads) * w.units + S.per - 1u) / S.per);
        before = scan256(mine, F.red, all);
        at = run;
    }
    if (at >= all) return false;  // (uniform)
    uint64_t base = 0;
    for (uint32_t s0 = 0; s0 < A.n_seq; s0 += kAttendThreads) {
        if (A.n_seq > kAttendThreads) {  // (the sums above were of several)
            w = AttendWork{};
            if (s0 + t < A.n_seq) w = attend_work(A, s0 + t, cols, unit);
            mine = w.all;
            uint64_t total;
            before = base + scan256(mine, F.red, total);
            base += total;
        }
        if (mine && at >= before && at - before < mine) {
            F.seq = s0 + t;
            F.seq_first = before;
            F.work = w;
        }
        if (at < base) break;  // (uniform)
    }
    __syncthreads();
    S.tile = 0u;
    S.apart = 1u;
    if (S.gang) {
        const uint32_t in_seq = static_cast<uint32_t>(run - F.seq_first);
        S.apart = F.work.tiles;
        S.tile = in_seq % S.apart;
        S.begin = in_seq / S.apart * S.per;
        S.end = min(S.begin + S.per, static_cast<uint64_t>(A.kv_heads) * F.work.units);
    } else {
        S.begin = at;
        S.end = min(at + S.per, all);
    }
    return true;
}

// What the products leave out: infinities and NaN in the V of nodes, which must not reach the rows that do not see them (0 times NaN is NaN). Rare, so it is done where a column is
// written: element d of each such node that the column sees is added to it (an infinity to whatever the others have made: the same sum).
template <int DT>
__device__ __forceinline__ float attend_odd(const AttendArgs& A, const unsigned char* v_token, uint32_t d, bool sees) {
    const float x = d < A.head_dim ? Mat<DT>::element(v_token, d) : 0.f;
    return sees && !(fabsf(x) <= FLT_MAX) ? x : 0.f;
}

// a column's results: a lane's 4 kEach-element pieces of each block
template <int DT, uint32_t EACH, uint32_t BLOCKS>
__device__ __forceinline__ void attend_write(const AttendArgs& A, unsigned char* to, uint32_t g, const f32x4 (&o)[BLOCKS * EACH], float by) {
#pragma unroll
    for (uint32_t b = 0; b < BLOCKS; ++b) {
        if constexpr (EACH == 1u) {
            static_assert(DT == 1);
            const uint32_t d = b * 16u + 4u * g;
            if (d >= A.head_dim) continue;
            __bf16 y[4];
#pragma unroll
            for (uint32_t l = 0; l < 4u; ++l) y[l] = static_cast<__bf16>(o[b][l] * by);
            __builtin_memcpy(__builtin_assume_aligned(to + d * 2u, 8u), y, 8u);
            continue;
        }
#pragma unroll
        for (uint32_t l = 0; l < 4u; ++l) {
            const uint32_t d = b * 16u * EACH + (4u * g + l) * EACH;
            if (d >= A.head_dim) continue;
            if constexpr (DT == 1) {
                __bf16 y[EACH];
#pragma unroll
                for (uint32_t e = 0; e < EACH; ++e) y[e] = static_cast<__bf16>(o[b * EACH + e][l] * by);
                __builtin_memcpy(__builtin_assume_aligned(to + d * 2u, EACH * 2u), y, EACH * 2u);
            } else {
                float y[EACH];
#pragma unroll
                for (uint32_t e = 0; e < EACH; ++e) y[e] = o[b * EACH + e][l] * by;
                __builtin_memcpy(__builtin_assume_aligned(to + d * 4u, EACH * 4u), y, EACH * 4u);
            }
        }
    }
}

// bytes to a token's piece of 16 bytes, from strides in such pieces: two multiplications of 32 bits, added up in 64
__device__ __forceinline__ uint64_t attend_offset(uint32_t page, uint32_t page_stride, uint32_t token, uint32_t token_stride, uint32_t piece) {
    return (static_cast<uint64_t>(page) * page_stride + (static_cast<uint64_t>(token) * token_stride + piece)) << 4;
}

// the page of a position of the slot whose table row this is; `pages` where there is none. (No branch: what is loaded behind one is waited for there, and with it everything loaded before.)
__device__ __forceinline__ uint32_t attend_page(const AttendArgs& A, const int32_t* row, uint32_t pos, uint32_t end) {
    const uint32_t at = pos >> A.page_shift, page = static_cast<uint32_t>(row[min(at, A.slot_pages - 1u)]);
    return pos < end && at < A.slot_pages ? min(page, A.pages) : A.pages;
}

// Zeros for K and V behind head_dim, which no load overwrites: q is 0 there, but what memory holds may be infinite, and that times 0 is NaN.
template <typename H, int DT>
__device__ __forceinline__ void attend_fill(uint32_t head_dim, unsigned char* buffer) {
#pragma unroll
    for (uint32_t l = 0; l < H::kMine; ++l) {
        const uint32_t at = l * 256u + threadIdx.x;
        if (H::piece(at) * Mat<DT>::kPer < head_dim) continue;
        *reinterpret_cast<uint4*>(buffer + at * 16u) = make_uint4(0u, 0u, 0u, 0u);
        *reinterpret_cast<uint4*>(buffer + H::kBuffer + at * 16u) = make_uint4(0u, 0u, 0u, 0u);
    }
}

template <int DT, int DP, int MS, int WM, int OCC>
__global__ void __launch_bounds__(256, OCC) attend_kernel(AttendArgs A) {
    typedef AttendShape<DT, DP, MS, WM> H;
    constexpr uint32_t kWT = 4u / WM, kOuts = H::kOuts, kEach = H::kEach, kBlocks = H::kBlocks, kChunks = H::kChunks, E = Mat<DT>::kBytes;
    constexpr uint32_t kDump = 4u * kOuts * 64u;  // floats of 16 columns' O^T
    constexpr bool kStaged = WM > 1;
    static_assert(WM == 1 || WM == 4);
    __shared__ AttendFind F;
    __shared__ uint32_t s_odd[2];  // a tile's and the next one's, in turn: cleared where a meeting lies between that and who sets it, and between that and who has read it
    __shared__ float s_part[kWT > 1u ? (kWT / 2u) * MS * (kDump + 128u) : 1u];
    // two buffers of K, then V. (Two variables: of one that is indexed the compiler has every read wait for what is on its way to the other half.)
    __shared__ uint4 s_even[kStaged ? 2u * H::kBuffer / 16u : 1u], s_odds[kStaged ? 2u * H::kBuffer / 16u : 1u];
    const uint32_t t = threadIdx.x, lane = lane_id(), c = lane & 15u, g = lane >> 4, wave = wave_id(), wm = wave % WM, wt = wave / WM;

    // (neighbouring runs on the same part of the chip: workgroup b runs on XCD b % 8)
    const uint32_t in_xcd = A.groups / 8u, run_id = blockIdx.x < in_xcd * 8u ? (blockIdx.x & 7u) * in_xcd + (blockIdx.x >> 3) : blockIdx.x;
    AttendSpan S;
    if (t < 2u) s_odd[t] = 0u;  // (attend_find's waves meet)
    const bool any = attend_find<kStaged>(A, H::kTileCols, H::kUnit, run_id, F, S);
    uint32_t run_odd = 0u;  // (the first thread's)
    if (t == 0u) A.run[run_id].more = 0u;
    if (!any) return;
    uint32_t s = F.seq;
    uint64_t seq_first = F.seq_first;
    AttendWork W = F.work;

    if constexpr (kStaged) {
        if (A.head_dim < DP) {  // (uniform; the waves meet before they read)
            attend_fill<H, DT>(A.head_dim, reinterpret_cast<unsigned char*>(s_even));
            attend_fill<H, DT>(A.head_dim, reinterpret_cast<unsigned char*>(s_odds));
        }
    }
    uint32_t turn_odd = 0u;
    for (uint64_t at = S.begin; at < S.end;) {
        while (!S.gang && at - seq_first >= W.all) {
            seq_first += W.all;
            ++s;  // (there is one: at < S.end)
            W = attend_work(A, s, H::kTileCols, H::kUnit);
        }
        const uint64_t in_seq = S.gang ? at : at - seq_first;
        const uint32_t item = static_cast<uint32_t>(in_seq / W.units), u0 = static_cast<uint32_t>(in_seq - static_cast<uint64_t>(item) * W.units);
        const uint32_t u1 = static_cast<uint32_t>(min(static_cast<uint64_t>(W.units), u0 + (S.end - at)));
        const uint32_t head = S.gang ? item : item / W.tiles, tile = S.gang ? S.tile : item - head * W.tiles;
        const uint32_t cols = W.nodes * A.group, col0 = tile * H::kTileCols + wm * (16u * MS);
        const uint32_t slot = A.slot ? A.slot[s] : s;
        const int32_t* table = A.table + static_cast<uint64_t>(slot) * A.table_stride;
        const bool no_slot = slot >= A.slots;
        const uint32_t total = no_slot ? 0u : W.total, length = min(W.length, total);

        // the columns: Q in its operand's places, what a column sees of the nodes
        uint4 q[MS][kChunks];
        uint64_t sees[MS];
        float top[MS], sum[MS];
        f32x4 o[MS][kOuts];
#pragma unroll
        for (int m = 0; m < MS; ++m) {
            const uint32_t col = min(col0 + m * 16u + c, cols - 1u), node = col / A.group, h = head * A.group + (col - node * A.group);
            const unsigned char* at_q = A.q + static_cast<uint64_t>(W.first + node) * A.q_row + static_cast<uint64_t>(h) * A.q_head;
#pragma unroll
            for (uint32_t j = 0; j < kChunks; ++j) {
                const uint32_t d = j * Mat<DT>::kDepth + g * Mat<DT>::kPer;
                q[m][j] = make_uint4(0u, 0u, 0u, 0u);
                if (d < A.head_dim) q[m][j] = *reinterpret_cast<const uint4*>(at_q + d * E);
            }
            sees[m] = A.mask ? A.mask[W.first + node] : (node < 63u ? (uint64_t{2} << node) - 1u : ~uint64_t{0});
            top[m] = -FLT_MAX;
            sum[m] = 0.f;
#pragma unroll
            for (uint32_t r = 0; r < kOuts; ++r) o[m][r] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
        const unsigned char* k_base = A.k + head * A.k_head;
        const unsigned char* v_base = A.v + head * A.v_head;
        const uint32_t in_page = (1u << A.page_shift) - 1u;

        const uint32_t p_end = min(u1 * H::kUnit, total);
        // A lane looks up the page of one position of those that are worked on next, and asks the others for theirs: one load ahead of the ones that need it
        constexpr uint32_t kAhead = kStaged ? H::kTokens : 32u;
        uint32_t pg = 0u, pg_next = 0u, pg_pos = 0u;
        // (What is loaded is not looked at before the next turn: that waits for all loads before it, too.)
        auto page_of = [&](uint32_t p) __attribute__((always_inline)) {
            pg_pos = p + (lane & (kAhead - 1u));
            pg_next = static_cast<uint32_t>(table[min(pg_pos >> A.page_shift, A.slot_pages - 1u)]);
        };
        auto page_from = [&](uint32_t pg, uint32_t token) __attribute__((always_inline)) { return static_cast<uint32_t>(__shfl(static_cast<int>(pg), static_cast<int>(token))); };
        // pg: of the positions that are worked on next; have: a bit for each that is there. (A page that is not: the first one's, not looked at.)
        uint64_t have = 0ull;
        auto turn = [&]() __attribute__((always_inline)) {
            const bool is = pg_pos < p_end && pg_pos >> A.page_shift < A.slot_pages && pg_next < A.pages;
            have = __ballot(is);  // (of 32 positions: the upper lanes say the same)
            pg = is ? pg_next : 0u;
        };
        uint4 kx[2][kChunks];
        uint4 vx[8][kBlocks];
        // token i of a lane's eight: 4 g + i of the first 16 positions, 4 g + i - 4 of the second
        auto v_pos = [&](uint32_t p0, uint32_t i) __attribute__((always_inline)) { return p0 + (i < 4u ? 0u : 12u) + 4u * g + i; };
        auto load_k = [&](uint32_t p0, uint32_t pg) __attribute__((always_inline)) {
#pragma unroll
            for (uint32_t i = 0; i < 2u; ++i) {
                const unsigned char* at_k = k_base + attend_offset(page_from(pg, 16u * i + c), A.k_page, (p0 + 16u * i + c) & in_page, A.k_token, 0u);
#pragma unroll
                for (uint32_t j = 0; j < kChunks; ++j) {
                    const uint32_t d = j * Mat<DT>::kDepth + g * Mat<DT>::kPer;
                    kx[i][j] = *reinterpret_cast<const uint4*>(at_k + (d < A.head_dim ? d : 0u) * E);
                }
            }
        };
        auto load_v = [&](uint32_t p0, uint32_t pg) __attribute__((always_inline)) {
#pragma unroll
            for (uint32_t i = 0; i < 8u; ++i) {
                const unsigned char* at_v = v_base + attend_offset(page_from(pg, v_pos(0u, i)), A.v_page, v_pos(p0, i) & in_page, A.v_token, 0u);
#pragma unroll
                for (uint32_t b = 0; b < kBlocks; ++b) {
                    const uint32_t d = b * 16u * kEach + c * kEach;
                    vx[i][b] = *reinterpret_cast<const uint4*>(at_v + (d < A.head_dim ? d : 0u) * E);
                }
            }
        };
        // a bit for each of a lane's eight tokens, of a bit for each token from `sub` on
        auto mine_of = [&](uint64_t all, uint32_t sub) __attribute__((always_inline)) {
            return (static_cast<uint32_t>(all >> (sub + 4u * g)) & 15u) | (static_cast<uint32_t>(all >> (sub + 4u * g + 16u)) & 15u) << 4;
        };

        // the word that holds element e of a token's
        auto element_word = [](const uint4& v, uint32_t e) __attribute__((always_inline)) {
            const uint32_t w = e * E / 4u;
            return w == 0u ? v.x : (w == 1u ? v.y : (w == 2u ? v.z : v.w));
        };
        constexpr uint32_t kStep = 32u * kWT;
        uint32_t odd = 0u;
        uint4 px[MS][DT == 1 ? 1 : 2];
        // the powers of 32 positions' scores from their K (k_of: piece j of tokens c and 16 + c); here: a bit a token of the lane; `then` is done when K has been read
        auto powers = [&](uint32_t p0, bool plain, uint32_t here, auto&& k_of, auto&& then) __attribute__((always_inline)) {
            f32x4 x[MS][2];
#pragma unroll
            for (uint32_t j = 0; j < kChunks; ++j)
#pragma unroll
                for (uint32_t i = 0; i < 2u; ++i) {
                    const uint4 k = k_of(i, j);
#pragma unroll
                    for (int m = 0; m < MS; ++m) x[m][i] = Mat<DT>::mul(k, q[m][j], j ? x[m][i] : f32x4{0.f, 0.f, 0.f, 0.f});
                }
            then();
            if (!plain) {  // (uniform)
#pragma unroll
                for (int m = 0; m < MS; ++m) {
                    const uint32_t seen = here & (sees_four(sees[m], v_pos(p0, 0u), length) | sees_four(sees[m], v_pos(p0, 4u), length) << 4);
#pragma unroll
                    for (uint32_t i = 0; i < 8u; ++i) x[m][i / 4u][i % 4u] = seen >> i & 1u ? x[m][i / 4u][i % 4u] : -INFINITY;
                }
            }
            float p[MS][8], part[MS];
            auto raise = [&](int m) __attribute__((always_inline)) {
#pragma unroll
                for (uint32_t i = 0; i < 8u; ++i) p[m][i] = __builtin_amdgcn_exp2f(fmaf(x[m][i / 4u][i % 4u], A.scale_log2, -top[m]));
                part[m] = ((p[m][0] + p[m][1]) + (p[m][2] + p[m][3])) + ((p[m][4] + p[m][5]) + (p[m][6] + p[m][7]));
            };
            bool grown = false;
#pragma unroll
            for (int m = 0; m < MS; ++m) {
                raise(m);
                grown |= part[m] > kMost;
            }
            if (__ballot(grown) != 0ull) {  // (uniform) some column's maximum has grown: only then they are looked for
#pragma unroll
                for (int m = 0; m < MS; ++m) {
                    float most = larger(larger(larger(x[m][0][0], x[m][0][1]), larger(x[m][0][2], x[m][0][3])), larger(larger(x[m][1][0], x[m][1][1]), larger(x[m][1][2], x[m][1][3])));
                    most *= A.scale_log2;
                    most = fmaxf(most, __shfl_xor(most, 16));
                    most = fmaxf(most, __shfl_xor(most, 32));
                    const float to = fmaxf(top[m], most), down = __builtin_amdgcn_exp2f(top[m] - to);
                    top[m] = to;
                    sum[m] *= down;
#pragma unroll
                    for (uint32_t r = 0; r < kOuts; ++r) o[m][r] *= down;
                    raise(m);
                }
            }
#pragma unroll
            for (int m = 0; m < MS; ++m) {
                sum[m] += part[m];
                if constexpr (DT == 1) {
                    bf16x8 b;
#pragma unroll
                    for (int i = 0; i < 8; ++i) b[i] = static_cast<__bf16>(p[m][i]);
                    px[m][0] = __builtin_bit_cast(uint4, b);
                } else {
#pragma unroll
                    for (int i = 0; i < 2; ++i)
                        px[m][i] = make_uint4(__float_as_uint(p[m][4 * i]), __float_as_uint(p[m][4 * i + 1]), __float_as_uint(p[m][4 * i + 2]), __float_as_uint(p[m][4 * i + 3]));
                }
            }
        };
        // V that is not there counts as 0, whatever the place holds; of nodes, which some columns see and others do not, what is no number is left for later
        auto clean = [&](uint4 v, bool there_, bool node) __attribute__((always_inline)) {
            const uint32_t keep = there_ ? 0xffffffffu : 0u;
            v = make_uint4(v.x & keep, v.y & keep, v.z & keep, v.w & keep);
            if (node) {
                const uint4 z = make_uint4(Mat<DT>::special(v.x), Mat<DT>::special(v.y), Mat<DT>::special(v.z), Mat<DT>::special(v.w));
                odd |= z.x | z.y | z.z | z.w;
                v = make_uint4(v.x & ~z.x, v.y & ~z.y, v.z & ~z.z, v.w & ~z.w);
            }
            return v;
        };
        auto add_up = [&](auto&& v_of) __attribute__((always_inline)) {  // O^T; v_of: block b of a lane's token i
#pragma unroll
            for (uint32_t b = 0; b < kBlocks; ++b) {
                uint4 v[8];
#pragma unroll
                for (uint32_t i = 0; i < 8u; ++i) v[i] = v_of(i, b);
#pragma unroll
                for (uint32_t e = 0; e < kEach; ++e) {
                    uint32_t word[8];
#pragma unroll
                    for (uint32_t i = 0; i < 8u; ++i) word[i] = element_word(v[i], e);
#pragma unroll
                    for (int m = 0; m < MS; ++m) o[m][b * kEach + e] = Mat<DT>::mul_tokens(word, e, px[m], o[m][b * kEach + e]);
                }
            }
        };
        if constexpr (!kStaged) {
            uint32_t p0 = u0 * H::kUnit + wt * 32u;
            if (p0 < p_end) {
                page_of(p0);
                turn();
                page_of(p0 + kStep);
                load_k(p0, pg);
            }
            for (; p0 < p_end; p0 += kStep) {
                load_v(p0, pg);
                if (A.head_dim < DP) {  // (uniform) what K is filled up with: 0, as q there is (infinity times 0 would be NaN)
#pragma unroll
                    for (uint32_t j = 0; j < kChunks; ++j)
                        if (j * Mat<DT>::kDepth + g * Mat<DT>::kPer >= A.head_dim) kx[0][j] = kx[1][j] = make_uint4(0u, 0u, 0u, 0u);
                }
                // whether all 32 positions are there and every column sees them (uniform)
                const bool plain = p0 + 32u <= length && static_cast<uint32_t>(have) == 0xffffffffu;
                const uint32_t here = mine_of(have, 0u);
                powers(p0, plain, here, [&](uint32_t i, uint32_t j) { return kx[i][j]; }, [&]() {  // the next positions' K while these are worked on
                    if (p0 + kStep < p_end) {
                        turn();
                        load_k(p0 + kStep, pg);
                        page_of(p0 + 2u * kStep);
                    }
                });
                if (!plain) {
#pragma unroll
                    for (uint32_t i = 0; i < 8u; ++i)
#pragma unroll
                        for (uint32_t b = 0; b < kBlocks; ++b) vx[i][b] = clean(vx[i][b], here >> i & 1u, v_pos(p0, i) >= length);
                }
                add_up([&](uint32_t i, uint32_t b) { return vx[i][b]; });
            }
        } else {
            unsigned char* const even = reinterpret_cast<unsigned char*>(s_even);
            unsigned char* const odds = reinterpret_cast<unsigned char*>(s_odds);
            // 16 bytes a thread, K's and V's pieces in the places that they have in LDS: who loads which is turned about as they lie there. Behind head_dim nothing is loaded: 0 stays there (attend_fill).
            const uint32_t wave_at = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(wave))) * 1024u;
            auto fetch_of = [&](uint32_t p, unsigned char* k_lds, auto all) __attribute__((always_inline)) {
#pragma unroll
                for (uint32_t l = 0; l < H::kMine; ++l) {
                    const uint32_t token = (l * 256u + t) / H::kPieces, piece = H::piece(l * 256u + t);
                    const uint32_t page = page_from(pg, token), in = (p + token) & in_page;
                    if (!all() && piece * Mat<DT>::kPer >= A.head_dim) continue;
                    to_lds(k_base + attend_offset(page, A.k_page, in, A.k_token, piece), k_lds + l * 4096u + wave_at);
                    to_lds(v_base + attend_offset(page, A.v_page, in, A.v_token, piece), k_lds + H::kBuffer + l * 4096u + wave_at);
                }
            };
            // (Two copies: lanes switched off and on around each load cost 5 x 9 nodes over 1001 positions of fp32 18.3 instead of 17.9 us, 2 x 64 over 131072 of bf16 286.8 instead of 285.)
            auto fetch = [&](uint32_t p, unsigned char* k_lds) __attribute__((always_inline)) {
                if (A.head_dim == DP) fetch_of(p, k_lds, []() { return true; });  // (uniform)
                else fetch_of(p, k_lds, []() { return false; });
            };
            // where a lane reads: of K piece 4 j + g of tokens c, of V (turned) 4 elements of token 4 g + c / 4; a token's order is the same 16 behind it
            const uint32_t k_row = c * H::kRow, k_piece = (g ^ H::order(c)) * 16u;
            const uint32_t v_row = (4u * g + c / 4u) * H::kRow + (c & 1u) * 8u, v_piece = ((c >> 1 & 1u) ^ H::order(4u * g + c / 4u)) * 16u;
            uint32_t p = u0 * H::kUnit;
            if (p < p_end) {
                page_of(p);
                turn();
                page_of(p + H::kTokens);
                fetch(p, even);
            }
            auto chunk = [&](unsigned char* const k_lds, unsigned char* const next_lds) __attribute__((always_inline)) {
                unsigned char* const v_lds = k_lds + H::kBuffer;
                const uint64_t here = have;
                const bool nodes = p + H::kTokens > length;        // (uniform)
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (what is on its way to LDS)
                __syncthreads();
                if (here != ~0ull || nodes) {
#pragma unroll
                    for (uint32_t l = 0; l < H::kMine; ++l) {
                        const uint32_t token = (l * 256u + t) / H::kPieces;
                        uint4& v = *reinterpret_cast<uint4*>(v_lds + (l * 256u + t) * 16u);
                        v = clean(v, here >> token & 1u, p + token >= length);
                    }
                    __syncthreads();
                }
                if (p + H::kTokens < p_end) {
                    turn();
                    page_of(p + 2u * H::kTokens);
                    fetch(p + H::kTokens, next_lds);
                }
                if (col0 >= cols) return;
#pragma unroll
                for (uint32_t sub = 0; sub < H::kTokens; sub += 32u) {
                    const uint32_t p0 = p + sub;
                    if (p0 >= p_end) break;
                    const bool plain = p0 + 32u <= length && static_cast<uint32_t>(here >> sub) == 0xffffffffu;
                    u32x2 v[H::kTurned ? kOuts : 1u][2];
                    powers(p0, plain, mine_of(here, sub), [&](uint32_t i, uint32_t j) { return *reinterpret_cast<const uint4*>(k_lds + k_row + (k_piece ^ j * 64u) + (sub + 16u * i) * H::kRow); }, [&]() {
                        if constexpr (H::kTurned) {  // of 4 tokens 16 elements: lane c of 16 asks for 4 elements of token c / 4, gets the tokens' c-th
#pragma unroll
                            for (uint32_t r = 0; r < kOuts; ++r)
#pragma unroll
                                for (uint32_t i = 0; i < 2u; ++i) v[r][i] = turned(v_lds + v_row + (v_piece ^ r * 32u) + (sub + 16u * i) * H::kRow);
                        }
                    });
                    if constexpr (H::kTurned) {
#pragma unroll
                        for (uint32_t r = 0; r < kOuts; ++r)
#pragma unroll
                            for (int m = 0; m < MS; ++m) o[m][r] = Mat<1>::mul(make_uint4(v[r][0].x, v[r][0].y, v[r][1].x, v[r][1].y), px[m][0], o[m][r]);
                    } else {
                        add_up([&](uint32_t i, uint32_t b) { return *reinterpret_cast<const uint4*>(v_lds + H::place(v_pos(sub, i), b * 16u + c)); });
                    }
                }
            };
            for (; p < p_end; p += H::kTokens) {  // (the same for the workgroup)
                chunk(even, odds);
                p += H::kTokens;
                if (p >= p_end) break;
                chunk(odds, even);
            }
        }
        if (__ballot(odd != 0u) != 0ull && lane == 0u) s_odd[turn_odd] = 1u;
        // a column's sum over its four lanes
#pragma unroll
        for (int m = 0; m < MS; ++m) {
            sum[m] += __shfl_xor(sum[m], 16);
            sum[m] += __shfl_xor(sum[m], 32);
        }
        // the waves of other positions: the upper half leaves what it has, the lower half joins it, and so on
        auto join = [&](int m, float their_top, float their_sum, auto&& theirs) __attribute__((always_inline)) {
            const float to = fmaxf(top[m], their_top), a = __builtin_amdgcn_exp2f(top[m] - to), z = __builtin_amdgcn_exp2f(their_top - to);
            top[m] = to;
            sum[m] = sum[m] * a + their_sum * z;
#pragma unroll
            for (uint32_t r = 0; r < kOuts; ++r) o[m][r] = o[m][r] * a + theirs(r) * z;
        };
        if constexpr (kWT > 1u) {
#pragma unroll
            for (uint32_t half = kWT / 2u; half >= 1u; half /= 2u) {
                __syncthreads();
                if (wt >= half && wt < 2u * half) {
#pragma unroll
                    for (int m = 0; m < MS; ++m) {
                        float* to = s_part + ((wt - half) * MS + m) * (kDump + 128u);
                        to[lane] = top[m];
                        to[64u + lane] = sum[m];
#pragma unroll
                        for (uint32_t r = 0; r < kOuts; ++r) *reinterpret_cast<f32x4*>(to + 128u + (r * 64u + lane) * 4u) = o[m][r];
                    }
                }
                __syncthreads();
                if (wt < half) {
#pragma unroll
                    for (int m = 0; m < MS; ++m) {
                        const float* from = s_part + (wt * MS + m) * (kDump + 128u);
                        join(m, from[lane], from[64u + lane], [&](uint32_t r) { return *reinterpret_cast<const f32x4*>(from + 128u + (r * 64u + lane) * 4u); });
                    }
                }
            }
        }
        __syncthreads();
        const bool any_odd = s_odd[turn_odd] != 0u;
        turn_odd ^= 1u;
        if (t == 0u) s_odd[turn_odd] = 0u;
        if (wt == 0u) {
            if (u0 == 0u && u1 == W.units) {
                if (any_odd) {  // (uniform)
#pragma unroll 1
                    for (uint32_t j = 0; j < W.nodes; ++j) {
                        const uint32_t pos = W.length + j, pg = W.length < total && pos < total ? attend_page(A, table, pos, total) : A.pages;
                        if (pg >= A.pages) continue;
                        const unsigned char* at_v = v_base + attend_offset(pg, A.v_page, pos & in_page, A.v_token, 0u);
#pragma unroll
                        for (uint32_t r = 0; r < kOuts; ++r) {
#pragma unroll
                            for (uint32_t l = 0; l < 4u; ++l)
#pragma unroll
                                for (int m = 0; m < MS; ++m)
                                    o[m][r][l] += attend_odd<DT>(A, at_v, (r / kEach) * 16u * kEach + (4u * g + l) * kEach + r % kEach, (sees[m] >> j & 1u) != 0u);
                            __builtin_amdgcn_sched_barrier(0);  // (loads of all of them together would take the registers that the products need)
                        }
                    }
                }
#pragma unroll
                for (int m = 0; m < MS; ++m) {
                    const uint32_t col = col0 + m * 16u + c;
                    if (col >= cols) continue;
                    const uint32_t node = col / A.group, h = head * A.group + (col - node * A.group);
                    const float by = sum[m] == 0.f ? 0.f : 1.f / sum[m];
                    if (A.lse && g == 0u)
                        A.lse[static_cast<uint64_t>(W.first + node) * A.heads + h] = sum[m] == 0.f ? -INFINITY : (top[m] + __builtin_amdgcn_logf(sum[m])) * 0.69314718f;
                    unsigned char* to = A.out + static_cast<uint64_t>(W.first + node) * A.out_row + static_cast<uint64_t>(h) * A.out_head;
                    attend_write<DT, kEach, kBlocks>(A, to, g, o[m], by);
                }
            } else {
                float* part = A.part + (static_cast<uint64_t>(run_id) * 2u + (u0 == 0u ? 1u : 0u)) * H::kPartFloats + wm * MS * H::kSubFloats;
#pragma unroll
                for (int m = 0; m < MS; ++m) {
                    if (col0 + m * 16u >= cols) continue;  // (a wave's)
                    float* to = part + m * H::kSubFloats;
                    to[lane] = top[m];
                    to[64u + lane] = sum[m];
#pragma unroll
                    for (uint32_t r = 0; r < kOuts; ++r) *reinterpret_cast<f32x4*>(to + 128u + (r * 64u + lane) * 4u) = o[m][r];
                }
            }
        }
        if (t == 0u && any_odd) run_odd |= u0 != 0u ? 1u : 2u;
        if (t == 0u && u0 == 0u && u1 < W.units) {
            // the workgroups that hold the rest of this tile
            const uint64_t first = at, last = at + W.units - 1u;
            AttendRun r;
            r.seq = s;
            r.head = head;
            r.tile = tile;
            r.more = static_cast<uint32_t>(last / S.per - first / S.per);
            r.apart = S.apart;
            r.odd = 0u;
            r.first = W.first, r.nodes = W.nodes, r.length = length, r.total = total;  // (of a slot that does not exist nothing is there: the join reads no table)
            A.run[run_id] = r;
        }
        at += u1 - u0;
        __syncthreads();
    }
    if (t == 0u) A.run[run_id].odd = run_odd;
}

// A workgroup joins 16 columns of the tile that begins in run x: the tile's first piece is that run's second part, the others are the first parts of the runs behind it. A wave takes every eighth
// (fourth, of the builds with many columns) piece, the next while it adds one, and what the waves have is joined through LDS, in an order that does not depend on who comes first.
// Tiles of many columns lie in few runs, and there are as many workgroups as tiles have 16 columns: 8, 4, 2 waves take 20, 13, 12 us for 16 x 48 over 8192, 14, 12.6, 19 for 2 x 64 over 131072; one row over 4096 7, 8, 12 (16 waves: 7.9).
// (Four pieces of a wave on their way instead of two: registers that leave fewer workgroups to find that they have nothing to do, 13 to 17 and 6.2 to 8.8 us for 64 rows.)
template <int WM>
constexpr uint32_t kJoinWavesOf = WM > 1 ? 4u : 8u;
template <int DT, int DP, int MS, int WM>
__global__ void __launch_bounds__(64 * kJoinWavesOf<WM>) attend_join_kernel(AttendArgs A) {
    typedef AttendShape<DT, DP, MS, WM> H;
    constexpr uint32_t kOuts = H::kOuts, kEach = H::kEach, kJoinWaves = kJoinWavesOf<WM>;
    __shared__ f32x4 s_o[kJoinWaves / 2u][kOuts][64];
    __shared__ float s_top[kJoinWaves / 2u][64], s_sum[kJoinWaves / 2u][64];
    const uint32_t x = blockIdx.x, sub = blockIdx.y, t = threadIdx.x, lane = t & 63u, wave = t >> 6, c = lane & 15u, g = lane >> 4;
    const AttendRun R = A.run[x];
    if (R.more == 0u) return;
    const uint32_t cols = R.nodes * A.group, col = R.tile * H::kTileCols + sub * 16u + c;
    if (col - c >= cols) return;
    auto piece = [&](uint32_t i) { return A.part + ((static_cast<uint64_t>(x) + static_cast<uint64_t>(i) * R.apart) * 2u + (i == 0u ? 1u : 0u)) * H::kPartFloats + sub * H::kSubFloats; };
    float top = -FLT_MAX, sum = 0.f;
    f32x4 o[kOuts];
#pragma unroll
    for (uint32_t r = 0; r < kOuts; ++r) o[r] = f32x4{0.f, 0.f, 0.f, 0.f};
    float their_top = -FLT_MAX, their_sum = 0.f;
    f32x4 theirs[kOuts];
    auto load = [&](uint32_t i) __attribute__((always_inline)) {
        const float* from = piece(i);
        their_top = from[lane];
        their_sum = from[64u + lane];
#pragma unroll
        for (uint32_t r = 0; r < kOuts; ++r) theirs[r] = *reinterpret_cast<const f32x4*>(from + 128u + (r * 64u + lane) * 4u);
    };
    auto join = [&]() __attribute__((always_inline)) {
        const float to = fmaxf(top, their_top), a = __builtin_amdgcn_exp2f(top - to), z = __builtin_amdgcn_exp2f(their_top - to);
        top = to;
        sum = sum * a + their_sum * z;
#pragma unroll
        for (uint32_t r = 0; r < kOuts; ++r) o[r] = o[r] * a + theirs[r] * z;
    };
    if (wave <= R.more) load(wave);
    // whether any of those that have the nodes - three pieces at most, of 32 positions at least - has met such (the same entry again where there are fewer)
    const uint32_t last = x + R.more * R.apart;
    const uint32_t odd = ((A.run[last].odd | A.run[last - (R.more > 1u ? R.apart : 0u)].odd | A.run[last - (R.more > 2u ? 2u * R.apart : 0u)].odd) & 1u) | (R.more < 3u ? R.odd & 2u : 0u);
    for (uint32_t i = wave; i <= R.more; i += kJoinWaves) {
        join();
        if (i + kJoinWaves <= R.more) load(i + kJoinWaves);
    }
#pragma unroll
    for (uint32_t half = kJoinWaves / 2u; half >= 1u; half /= 2u) {
        __syncthreads();
        if (wave >= half && wave < 2u * half) {
            s_top[wave - half][lane] = top;
            s_sum[wave - half][lane] = sum;
#pragma unroll
            for (uint32_t r = 0; r < kOuts; ++r) s_o[wave - half][r][lane] = o[r];
        }
        __syncthreads();
        if (wave < half) {
            their_top = s_top[wave][lane];
            their_sum = s_sum[wave][lane];
#pragma unroll
            for (uint32_t r = 0; r < kOuts; ++r) theirs[r] = s_o[wave][r][lane];
            join();
        }
    }
    if (wave != 0u || col >= cols) return;
    const uint32_t node = col / A.group, h = R.head * A.group + (col - node * A.group);
    if (odd != 0u) {
        const int32_t* table = A.table + static_cast<uint64_t>(A.slot ? A.slot[R.seq] : R.seq) * A.table_stride;
        const uint64_t sees = A.mask ? A.mask[R.first + node] : (node < 63u ? (uint64_t{2} << node) - 1u : ~uint64_t{0});
#pragma unroll 1
        for (uint32_t j = 0; j < R.nodes && R.length + j < R.total; ++j) {
            const uint32_t pos = R.length + j, pg = attend_page(A, table, pos, R.total);
            if (pg >= A.pages) continue;
            const unsigned char* at_v = A.v + R.head * A.v_head + attend_offset(pg, A.v_page, pos & ((1u << A.page_shift) - 1u), A.v_token, 0u);
#pragma unroll
            for (uint32_t r = 0; r < kOuts; ++r) {
#pragma unroll
                for (uint32_t l = 0; l < 4u; ++l) o[r][l] += attend_odd<DT>(A, at_v, (r / kEach) * 16u * kEach + (4u * g + l) * kEach + r % kEach, (sees >> j & 1u) != 0u);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    }
    const float by = sum == 0.f ? 0.f : 1.f / sum;
    if (A.lse && g == 0u) A.lse[static_cast<uint64_t>(R.first + node) * A.heads + h] = sum == 0.f ? -INFINITY : (top + __builtin_amdgcn_logf(sum)) * 0.69314718f;
    attend_write<DT, kEach, H::kBlocks>(A, A.out + static_cast<uint64_t>(R.first + node) * A.out_row + static_cast<uint64_t>(h) * A.out_head, g, o, by);
}

}  // namespace ws
