// ebx_kv_share.h -- requests that share cache blocks: arguments and launchers shared by the translation
// units that fork, compact and copy blocks, find common prefixes and attend over them.
#pragma once

#include "ebx_kv.h"

namespace ebx {

// `shares` holds for every block the number of rows beyond the first that hold it: 0 for a free block
// and for one that a single row holds.
struct KvForkArgs {
    const int32_t* lengths;
    const int32_t* tables;
    const int32_t* shares;
    int32_t* free_ring;
    const int64_t* ring;
    const int32_t* parents;
    const int32_t* keep;      // may be null: everything
    int32_t* out_lengths;
    int32_t* out_tables;
    int32_t* out_shares;
    int64_t* ring_out;
    int32_t* sources;         // [requests]
    int32_t* targets;
    int requests, width, shift, blocks, free_size;
};

struct KvCompactArgs {
    const int32_t* lengths;
    const int32_t* tables;
    const int32_t* shares;
    int32_t* out_tables;
    int32_t* out_shares;
    int32_t* free_out;        // [blocks]
    int64_t* ring_out;
    int32_t* sources;         // [blocks / 2]
    int32_t* targets;
    int requests, width, shift, blocks;
};
constexpr int kKvMostCompact = 1 << 19;  // blocks whose bits kv_compact keeps in shared memory

constexpr int kKvCopyLayers = 64;  // layers of a launch

struct KvCopyArgs {
    const int32_t* sources;
    const int32_t* targets;
    const int64_t* count;     // may be null: n
    int64_t bytes;            // codes of a block, one side
    int n, layers, blocks, kv_heads;
    struct {
        int8_t* codes[2];
        float* scales[2];
    } layer[kKvCopyLayers];
};

// What kv_prefixes finds.  Requests whose tables begin alike form a group, which has the number of its
// first request; the other numbers are empty groups.
struct KvPrefixes {
    int32_t* group_starts;  // [requests + 1]: first token of each group in `list`
    int32_t* shared;        // [requests]: tokens that the group shares
    int32_t* own_first;     // [requests]: the first token that the request does not share
    int32_t* list;          // [tokens]: the groups' tokens
    int32_t* state;         // [tokens]: 0: of no request, 1: of a request by itself, 2: of one in a group
    int32_t* largest;       // tokens of the largest group
};

// All in one buffer of 3 * requests + 2 + 2 * tokens ints, in the order of the structure.
inline KvPrefixes prefixes_at(int32_t* p, int64_t requests, int64_t tokens) {
    return {p, p + requests + 1, p + 2 * requests + 1, p + 3 * requests + 1, p + 3 * requests + 1 + tokens,
            p + 3 * requests + 1 + 2 * tokens};
}

struct KvPrefixArgs {
    const int32_t* tables;
    const int32_t* lengths;
    const int32_t* starts;
    KvPrefixes out;
    int64_t tokens;
    int requests, width, shift, blocks;
    int size;               // a power of two, requests or more (set by the launch)
};
constexpr int kKvMostPrefixes = 8192;  // requests that kv_prefixes sorts in shared memory

cudaError_t launch_kv_fork(const KvForkArgs& a, cudaStream_t s);
cudaError_t launch_kv_compact(const KvCompactArgs& a, cudaStream_t s);
cudaError_t launch_kv_copy(const KvCopyArgs& a, int sms, int dev, cudaStream_t s);
cudaError_t launch_kv_prefixes(KvPrefixArgs a, cudaStream_t s);

}  // namespace ebx
