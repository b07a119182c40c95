// ebx_kv_share_capi.cu -- the extern "C" entries for requests that share cache blocks (include/ebx.h): every
// check that the host can make, then the launch.
#include <algorithm>
#include <cmath>

#include "ebx_kv_check.h"
#include "ebx_kv_share.h"

namespace {

// Null, or what is wrong with a table of `requests` rows over `blocks` blocks.
const char* table_of(int32_t requests, int32_t width, int32_t block_size, int32_t blocks) {
    if (requests < 0 || requests > ebx::kKvMaxRequests) return "kv tables: need 0 <= requests <= 16384";
    if (log2_of(block_size) < 0) return "kv tables: block_size must be 16, 32, 64 or 128";
    if (width < 1 || int64_t(width) * block_size > INT32_MAX) return "kv tables: need width >= 1 and width * block_size < 2^31";
    if (blocks < 1 || int64_t(blocks) * block_size > INT32_MAX) return "kv tables: need blocks >= 1 and blocks * block_size < 2^31";
    return nullptr;
}

// Can attention over prefixes be asked for with these sizes?
bool shared_sizes(const ebx_kv_pool* pool, int32_t heads, int32_t requests, int64_t tokens, int32_t max_new, int32_t max_length,
                  ebx::KvPool& p) {
    return !pool_of(pool, p) && heads >= 1 && heads % p.kv_heads == 0 && requests >= 0 && requests <= ebx::kKvMostPrefixes &&
           tokens >= 0 && tokens <= INT32_MAX && max_new >= 0 && max_length >= 0;
}

}  // namespace

extern "C" {

ebx_status ebx_kv_fork(const int32_t* lengths, const int32_t* tables, int32_t width, int32_t block_size,
                       const int32_t* shares, int32_t blocks, int32_t* free_ring, int32_t free_size,
                       const int64_t* ring, const int32_t* parents, const int32_t* keep, int32_t requests,
                       int32_t* out_lengths, int32_t* out_tables, int32_t* out_shares, int64_t* ring_out,
                       int32_t* sources, int32_t* targets, int32_t device, void* stream) {
    if (const char* msg = table_of(requests, width, block_size, blocks)) return invalid(msg);
    if (!shares || !free_ring || !ring || !out_shares || !ring_out ||
        (requests > 0 && (!lengths || !tables || !parents || !out_lengths || !out_tables || !sources || !targets)))
        return invalid("null argument");
    if (free_size < 1) return invalid("ebx_kv_fork: need free_size >= 1");
    if (out_shares == shares || ring_out == ring ||
        (requests > 0 && (out_lengths == lengths || out_tables == tables)))
        return invalid("ebx_kv_fork: outputs must not be inputs");
    Device d(device);
    if (d.err != cudaSuccess) return launched(d.err, "cudaSetDevice");
    const ebx::KvForkArgs a{lengths, tables, shares, free_ring, ring, parents, keep, out_lengths, out_tables, out_shares,
                            ring_out, sources, targets, requests, width, log2_of(block_size), blocks, free_size};
    return launched(ebx::launch_kv_fork(a, static_cast<cudaStream_t>(stream)), "ebx_kv_fork");
}

ebx_status ebx_kv_compact(const int32_t* lengths, const int32_t* tables, int32_t width, int32_t block_size,
                          const int32_t* shares, int32_t blocks, int32_t requests, int32_t* out_tables,
                          int32_t* out_shares, int32_t* free_out, int64_t* ring_out, int32_t* sources,
                          int32_t* targets, int32_t device, void* stream) {
    if (const char* msg = table_of(requests, width, block_size, blocks)) return invalid(msg);
    if (blocks > ebx::kKvMostCompact) return invalid("ebx_kv_compact: need blocks <= 524288");
    if (!shares || !out_shares || !free_out || !ring_out || (blocks > 1 && (!sources || !targets)) ||
        (requests > 0 && (!lengths || !tables || !out_tables)))
        return invalid("null argument");
    if (out_shares == shares || (requests > 0 && out_tables == tables))
        return invalid("ebx_kv_compact: outputs must not be inputs");
    Device d(device);
    if (d.err != cudaSuccess) return launched(d.err, "cudaSetDevice");
    const ebx::KvCompactArgs a{lengths, tables, shares, out_tables, out_shares, free_out, ring_out, sources, targets,
                               requests, width, log2_of(block_size), blocks};
    return launched(ebx::launch_kv_compact(a, static_cast<cudaStream_t>(stream)), "ebx_kv_compact");
}

ebx_status ebx_kv_copy(const ebx_kv_pool* pools, int32_t layers, const int32_t* sources, const int32_t* targets,
                       const int64_t* count, int32_t n, void* stream) {
    if (layers < 0 || n < 0) return invalid("ebx_kv_copy: need layers >= 0 and n >= 0");
    if (layers == 0) return EBX_OK;
    if (!pools) return invalid("null argument");
    for (int32_t i = 0; i < layers; ++i) {
        ebx::KvPool p;
        if (const char* msg = pool_of(pools + i, p)) return invalid(msg);
        if (pools[i].blocks != pools->blocks || pools[i].kv_heads != pools->kv_heads ||
            pools[i].block_size != pools->block_size || pools[i].head_dim != pools->head_dim ||
            pools[i].device != pools->device)
            return invalid("ebx_kv_copy: pools must have the same sizes and device");
    }
    if (n == 0) return EBX_OK;
    if (!sources || !targets) return invalid("null argument");
    Device d(pools->device);
    if (d.err != cudaSuccess) return launched(d.err, "cudaSetDevice");
    const int sms = ebx::gemm_sm_count(pools->device);
    ebx::KvCopyArgs a{};
    a.sources = sources;
    a.targets = targets;
    a.count = count;
    a.bytes = int64_t(pools->kv_heads) * pools->block_size * pools->head_dim;
    a.n = n;
    a.blocks = pools->blocks;
    a.kv_heads = pools->kv_heads;
    for (int32_t first = 0; first < layers; first += ebx::kKvCopyLayers) {
        a.layers = std::min(layers - first, int32_t(ebx::kKvCopyLayers));
        for (int i = 0; i < a.layers; ++i) {
            const ebx_kv_pool& p = pools[first + i];
            a.layer[i].codes[0] = static_cast<int8_t*>(p.k_codes);
            a.layer[i].codes[1] = static_cast<int8_t*>(p.v_codes);
            a.layer[i].scales[0] = p.k_scales;
            a.layer[i].scales[1] = p.v_scales;
        }
        const ebx_status st = launched(ebx::launch_kv_copy(a, sms, pools->device, static_cast<cudaStream_t>(stream)), "ebx_kv_copy");
        if (st != EBX_OK) return st;
    }
    return EBX_OK;
}

uint64_t ebx_kv_prefixes_ints(int32_t requests, int64_t tokens) {
    return requests < 0 || tokens < 0 ? 0 : 3 * uint64_t(requests) + 2 + 2 * uint64_t(tokens);
}

ebx_status ebx_kv_prefixes(const int32_t* tables, int32_t width, int32_t block_size, int32_t blocks,
                           const int32_t* lengths, const int32_t* starts, int32_t requests, int64_t tokens,
                           int32_t* prefixes, int32_t device, void* stream) {
    if (const char* msg = table_of(requests, width, block_size, blocks)) return invalid(msg);
    if (requests > ebx::kKvMostPrefixes) return invalid("ebx_kv_prefixes: need requests <= 8192");
    if (tokens < 0 || tokens > INT32_MAX) return invalid("ebx_kv_prefixes: need 0 <= tokens < 2^31");
    if (requests == 0) return EBX_OK;
    if (!tables || !lengths || !starts || !prefixes) return invalid("null argument");
    Device d(device);
    if (d.err != cudaSuccess) return launched(d.err, "cudaSetDevice");
    ebx::KvPrefixArgs a{};
    a.tables = tables;
    a.lengths = lengths;
    a.starts = starts;
    a.out = ebx::prefixes_at(prefixes, requests, tokens);
    a.tokens = tokens;
    a.requests = requests;
    a.width = width;
    a.shift = log2_of(block_size);
    a.blocks = blocks;
    return launched(ebx::launch_kv_prefixes(a, static_cast<cudaStream_t>(stream)), "ebx_kv_prefixes");
}

uint64_t ebx_kv_shared_attention_workspace_bytes(const ebx_kv_pool* pool, int32_t heads, int32_t requests,
                                                 int64_t tokens, int32_t max_new, int32_t max_length) {
    ebx::KvPool p;
    if (!shared_sizes(pool, heads, requests, tokens, max_new, max_length, p)) return 0;
    Device d(pool->device);
    if (d.err != cudaSuccess) return 0;
    return ebx::kv_shared_workspace_bytes(p, heads, requests, tokens, max_new, max_length);
}

int32_t ebx_kv_takes_prefixes(const ebx_kv_pool* pool, int32_t heads, int32_t requests, int64_t tokens,
                              int32_t max_new, int32_t max_length) {
    ebx::KvPool p;
    return shared_sizes(pool, heads, requests, tokens, max_new, max_length, p) &&
           ebx::kv_takes_prefixes(p, heads, requests, tokens, max_new, max_length);
}

ebx_status ebx_kv_shared_attention(const ebx_kv_pool* pool, const void* q, int64_t q_token_stride,
                                   int64_t q_head_stride, int32_t heads, int32_t dtype, const int32_t* tables,
                                   int32_t width, const int32_t* lengths, const int32_t* starts,
                                   const int32_t* prefixes, int32_t requests, int64_t tokens, int32_t causal,
                                   float scale, int32_t max_new, int32_t max_length, void* out, float* lse,
                                   void* workspace, uint64_t workspace_bytes, void* stream) {
    ebx::KvPool p;
    if (const char* msg = pool_of(pool, p)) return invalid(msg);
    if (dtype != ebx::kKvF16 && dtype != ebx::kKvBF16)
        return invalid("ebx_kv_shared_attention: dtype must be fp16 or bf16");
    if (heads < 1 || heads % p.kv_heads != 0 || heads > (1 << 20))
        return invalid("ebx_kv_shared_attention: heads must be a multiple of kv_heads");
    if (requests < 0 || requests > ebx::kKvMostPrefixes || width < 1 || int64_t(width) * p.block_size > INT32_MAX / 2 ||
        tokens < 0 || tokens > INT32_MAX || tokens * (heads / p.kv_heads) > INT32_MAX / 2)
        return invalid("ebx_kv_shared_attention: requests, table width or tokens out of range");
    if (!std::isfinite(scale * 1.4426950408889634f)) return invalid("ebx_kv_shared_attention: scale must be finite");
    if (max_new < 0 || max_length < 0) return invalid("ebx_kv_shared_attention: max_new and max_length are >= 0");
    if (tokens == 0 || requests == 0) return EBX_OK;  // rows of no request are left as they are
    if (!out || !starts || !tables || !lengths || !prefixes) return invalid("null argument");
    ebx::KvRows rows;
    if (const char* msg = rows_of(q, q_token_stride, q_head_stride, rows)) return invalid(msg);
    if (!aligned16(out) || !aligned16(workspace))
        return invalid("ebx_kv_shared_attention: out and workspace must be 16-byte aligned");
    Device d(pool->device);
    if (d.err != cudaSuccess) return launched(d.err, "cudaSetDevice");
    const int group = heads / p.kv_heads;
    const uint64_t need = ebx::kv_shared_workspace_bytes(p, heads, requests, tokens, max_new, max_length);
    if (need > 0 && (!workspace || workspace_bytes < need)) {
        ebx::set_error("ebx_kv_shared_attention: workspace smaller than ebx_kv_shared_attention_workspace_bytes");
        return EBX_ERR_WORKSPACE;
    }
    ebx::KvAttnArgs a{};
    a.pool = p;
    a.q = rows;
    a.tables = tables;
    a.lengths = lengths;
    a.starts = starts;
    a.out = out;
    a.lse = lse;
    a.tokens = tokens;
    a.requests = requests;
    a.width = width;
    a.heads = heads;
    a.set_group(group);
    a.causal = causal != 0;
    a.scale_log2 = scale * 1.4426950408889634f;
    const ebx::KvPrefixes found = ebx::prefixes_at(const_cast<int32_t*>(prefixes), requests, tokens);
    a.group_starts = found.group_starts;
    a.shared = found.shared;
    a.own_first = found.own_first;
    a.list = found.list;
    a.state = found.state;
    a.largest = found.largest;
    return launched(ebx::launch_kv_shared_attention(a, dtype == ebx::kKvBF16, max_new, max_length, workspace,
                                                    static_cast<cudaStream_t>(stream)), "ebx_kv_shared_attention");
}

}  // extern "C"
