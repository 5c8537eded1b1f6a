// What the calls over a cycle with a tree of drafts (ws_abi.hip) hand to their kernels (ws_tree.hip, ws_attend.hip, ws_cache.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "ws_history.h"
#include "ws_loss.h"

namespace ws {

constexpr uint32_t kTreeNodes = 64u, kTreeListed = 32u, kTreeEntryWords = 72u;

// ---- ws_tree.hip
struct TreeStageArgs {
    uint32_t n_seq, rows;
    const uint32_t* seq_off;
    const int32_t* parent;
    const uint32_t* len;
    const uint32_t* slot;
    uint64_t* mask;
    int32_t* position;
    uint32_t* length;
};

struct TreeVerifyArgs {
    LossRows R;
    uint32_t n_seq;
    const uint32_t* seq_off;
    const int32_t* parent;
    const int32_t* q;
    uint64_t q_words;
    const int32_t* q_off;
    const double* u_accept;
    const double* u_draw;
    uint32_t depth;
    int32_t* n_accepted;
    int32_t* path;
    int32_t* chosen;
    uint32_t* status;
    float* logprob;
    HistoryRef hist;
    // of the rows' decisions: nodes of a sequence that have workgroups of their own, whether a node asks for its parent's decision first, workgroups a row, vectors each
    uint32_t levels, look, row_parts, row_per;
    unsigned long long* row_meet;  // row_parts > 1: [rows][4][row_parts]
    unsigned long long* decided;   // [rows][2]
    // of the draw: workgroups a sequence, vectors each (at most kDrawThreads * NV), how often one looks for the others
    uint32_t parts, per, looks;
    unsigned long long* meet;  // parts > 1: [n_seq][kTreeWords][parts]
    unsigned long long tag;
};
// 64-bit words a part: maximum and sum, each twice
constexpr uint32_t kTreeWords = 4u;

int launch_tree_stage(hipStream_t stream, const TreeStageArgs& a);
int launch_tree_verify(hipStream_t stream, int dtype, const TreeVerifyArgs& a);
uint32_t tree_most_share(int dtype);
int prepare_tree();

// ---- ws_attend.hip
struct AttendArgs {
    const unsigned char* k;
    const unsigned char* v;
    uint32_t k_page, k_token, v_page, v_token;  // pieces of 16 bytes between
    uint64_t k_head, v_head;                    // bytes
    uint32_t pages, page_shift, kv_heads, head_dim;
    const int32_t* table;
    uint32_t slots, slot_pages;
    uint64_t table_stride;
    uint32_t n_seq, rows, heads, group;
    const unsigned char* q;
    uint64_t q_row, q_head;
    unsigned char* out;
    uint64_t out_row, out_head;
    float* lse;
    const uint32_t* seq_off;
    const uint32_t* length;
    const uint32_t* slot;
    const uint64_t* mask;
    float scale_log2;  // scale times log2(e)
    uint32_t groups;
    float* part;       // [groups][2][kPartFloats of the build]
    struct AttendRun* run;  // [groups]
};
// what the join needs of a workgroup: the tile that begins in its run and does not end there (`more` runs behind it, `apart` in number, hold the rest)
struct AttendRun {
    uint32_t seq, head, tile, more, apart;
    uint32_t first, nodes, length, total;  // of the sequence: row, nodes, positions before the nodes, all positions (0 where its slot does not exist; length no more than that)
    uint32_t odd;  // bits: whether its first part (of a tile that began before), its last (of the one that begins) has met nodes whose V holds infinities or NaN
};

struct AttendPlan {
    uint32_t build, groups;
    uint64_t part_bytes, bytes;
};
AttendPlan attend_plan(int dtype, uint32_t head_dim, uint32_t cols, uint32_t compute_units);
int launch_attend(hipStream_t stream, const AttendPlan& plan, const AttendArgs& a);
int prepare_attend();

// ---- ws_cache.hip
constexpr uint32_t kCacheMost = 1024u;
constexpr int32_t kCacheOk = 0, kCacheFull = 1, kCacheBad = 2;

struct CacheSide {
    unsigned char* at;
    uint64_t layer, page, token, head;  // bytes between
};
struct CacheRef {
    CacheSide side[2];  // K, V
    uint32_t layers, pages, page_shift, kv_heads, head_bytes;
    int32_t* table;
    uint32_t slots, slot_pages;
    uint64_t table_stride;
    int32_t* held;
    int32_t* refs;
    int32_t* free;
    int32_t* n_free;
};

struct PagesArgs {
    CacheRef C;
    const int32_t* slot;    // of a fork: dst
    const int32_t* src;     // of a fork
    const int32_t* tokens;  // wanted, kept or copied
    uint32_t n;
    int32_t* status;
};

struct KeepArgs {
    CacheRef C;
    const int32_t* path;
    uint32_t depth;
    const int32_t* n_accepted;
    const uint32_t* length;
    const uint32_t* slot;
    uint32_t n_seq;
};
int prepare_cache();
int launch_cache_reserve(hipStream_t stream, const PagesArgs& a);
int launch_cache_fork(hipStream_t stream, const PagesArgs& a);
int launch_cache_release(hipStream_t stream, const PagesArgs& a);
int launch_cache_keep(hipStream_t stream, const KeepArgs& a);

}  // namespace ws
