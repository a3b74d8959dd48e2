// Attention of decoder rows to keys and values that several sequences hold:
// a paged cache's (paged.hip) or an encoder's states (cross.hip).
#pragma once

#include "internal.h"

namespace trit {

// Tokens of a block of keys or values, the unit every kernel works on.
constexpr int BLOCK_TOKENS = 64;
// Sequences of one launch (their entries are kernel arguments).
constexpr int CALL_SEQS = 128;

// Where element e of token t of a block lies (HDP: head_dim rounded up to 64
// or 128). The orders are the matrix instructions' operand order, so that a
// wave reads a 1 KB fragment in lane order: 16 bytes a lane, lane 16 q + m.
//  K: m is the token of a 16-token tile, the lane's values consecutive e.
//  V: m is e of a 16-wide tile, the lane's values the tokens 4 q + r of each
//     16-token tile -- the tokens whose scores the same lane holds, so that
//     probabilities go from one product to the next within their lane.
template <int HDP>
__host__ __device__ constexpr int k8_at(int t, int e) {
    return (((t / 16) * (HDP / 64) + e / 64) * 64 + (e % 64) / 16 * 16 + t % 16) * 16 + e % 16;
}
template <int HDP>
__host__ __device__ constexpr int v8_at(int t, int e) {
    return (e / 16 * 64 + (t % 16) / 4 * 16 + e % 16) * 16 + t / 16 * 4 + t % 4;
}
// f16 fragments hold 8 values a lane: 32 e of K, 32 tokens of V.
template <int HDP>
__host__ __device__ constexpr int k16_at(int t, int e) {
    return (((t / 16) * (HDP / 32) + e / 32) * 64 + (e % 32) / 8 * 16 + t % 16) * 8 + e % 8;
}
template <int HDP>
__host__ __device__ constexpr int v16_at(int t, int e) {
    return ((e / 16 * 2 + t / 32) * 64 + (t % 16) / 4 * 16 + e % 16) * 8 + t % 32 / 16 * 4 + t % 4;
}

// One sequence (or audio) of an attention call.
struct AttendSeq {
    int place;  // row of the page table and of the open blocks, or slot of the states
    int len;    // keys
    int rows;   // query rows
    int first;  // its first row in q and out
    // Set by attend(): its first item of the launch; its first group of items
    // that are joined, and its first item among those; the items its keys are
    // split into.
    int start, group, part, chunks;
};

// Device memory of a handle for keys that are split over workgroups: each
// one's sums, and a counter for each group of them (0 between launches).
struct AttendScratch {
    DeviceMemory memory;
    // For heads of hdp (64 or 128) values; clears the counters on `s`.
    void make(int hdp, hipStream_t s);
};

struct AttendArgs {
    const float* q = nullptr;  // rows of stride qs
    long long qs = 0;
    float* out = nullptr;  // rows of heads * hd
    float scale = 0.0f;    // on the scores
    int kv_heads = 0, group = 0, hd = 0;
    // Full blocks (a paged cache): int8 codes, K then V, and their two scales, by
    // page and head; the table's rows.
    const uint8_t* codes = nullptr;
    const float2* scales = nullptr;
    const int* table = nullptr;
    int table_stride = 0;
    // f16 blocks, K then V: one for each place and head (a paged cache's open
    // blocks), or `blocks` of them (states).
    const _Float16* f16 = nullptr;
    int blocks = 1;
    // Set by attend(): the scratch's parts, and the blocks of a chunk.
    float* sums = nullptr;
    uint64_t* tops = nullptr;
    int* counters = nullptr;
    int chunk = 0;
    bool aligned = false, aligned_out = false;  // 16-byte loads of the queries, stores of the outputs
    int n = 0;
    AttendSeq s[CALL_SEQS];
};

// `seqs`: place .. first set. Queued on `s`, where no other call with the same
// scratch may overlap.
void attend(AttendArgs& a, const std::vector<AttendSeq>& seqs, bool paged, AttendScratch& scratch, hipStream_t s);

}  // namespace trit
