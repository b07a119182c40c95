// ebx_kv_capi.cu -- the extern "C" entries of the 8-bit paged key/value cache (include/ebx.h):
// every check that the host can make, then the launch.
#include <cmath>

#include "ebx_kv_check.h"

extern "C" {

ebx_status ebx_kv_plan(const int32_t* past, const int32_t* added, int32_t requests, int32_t* tables,
                       int32_t width, int32_t block_size, int32_t* free_ring, int32_t free_size,
                       const int64_t* ring, int64_t* ring_out, int32_t* lengths, int32_t* starts,
                       int64_t* slots, int32_t* positions, int64_t tokens, int32_t device, void* stream) {
    if (!ring || !ring_out || !starts || !free_ring ||
        (requests > 0 && (!past || !added || !tables || !lengths)) || (tokens > 0 && (!slots || !positions)))
        return invalid("null argument");
    if (requests < 0 || requests > ebx::kKvMaxRequests) return invalid("ebx_kv_plan: need 0 <= requests <= 16384");
    if (width < 1 || free_size < 1) return invalid("ebx_kv_plan: need width >= 1 and free_size >= 1");
    // lengths and positions have 31 bits, so a row that holds more could carry a request past them
    if (int64_t(width) * block_size > INT32_MAX) return invalid("ebx_kv_plan: need width * block_size < 2^31");
    if (tokens < 0 || tokens > INT32_MAX) return invalid("ebx_kv_plan: need 0 <= tokens < 2^31");
    if (log2_of(block_size) < 0) return invalid("ebx_kv_plan: block_size must be 16, 32, 64 or 128");
    if (ring_out == ring || (requests > 0 && lengths == past))
        return invalid("ebx_kv_plan: ring_out and lengths must not be ring and past");
    Device d(device);
    if (d.err != cudaSuccess) return launched(d.err, "cudaSetDevice");
    const ebx::KvPlanArgs a{past, added, tables, free_ring, ring, ring_out, lengths, starts, slots,
                            positions, tokens, requests, width, log2_of(block_size), free_size};
    return launched(ebx::launch_kv_plan(a, static_cast<cudaStream_t>(stream)), "ebx_kv_plan");
}

ebx_status ebx_kv_append(const ebx_kv_pool* pool, const void* k, int64_t k_token_stride,
                         int64_t k_head_stride, const void* v, int64_t v_token_stride,
                         int64_t v_head_stride, const int64_t* slots, int64_t tokens, int32_t dtype,
                         void* stream) {
    ebx::KvPool p;
    if (const char* msg = pool_of(pool, p)) return invalid(msg);
    if (dtype != ebx::kKvF16 && dtype != ebx::kKvBF16) return invalid("ebx_kv_append: dtype must be fp16 or bf16");
    if (tokens < 0 || tokens > INT32_MAX) return invalid("ebx_kv_append: need 0 <= tokens < 2^31");
    if (tokens == 0) return EBX_OK;
    if (!slots) return invalid("null argument");
    ebx::KvRows kr, vr;
    if (const char* msg = rows_of(k, k_token_stride, k_head_stride, kr)) return invalid(msg);
    if (const char* msg = rows_of(v, v_token_stride, v_head_stride, vr)) return invalid(msg);
    Device d(pool->device);
    if (d.err != cudaSuccess) return launched(d.err, "cudaSetDevice");
    return launched(ebx::launch_kv_append(p, kr, vr, slots, tokens, dtype == ebx::kKvBF16,
                                          static_cast<cudaStream_t>(stream)), "ebx_kv_append");
}

ebx_status ebx_kv_materialize(const ebx_kv_pool* pool, const int32_t* tables, int32_t width,
                              const int32_t* starts, const int32_t* first, int32_t requests,
                              int64_t tokens, int32_t dtype, void* k, void* v, void* stream) {
    ebx::KvPool p;
    if (const char* msg = pool_of(pool, p)) return invalid(msg);
    if (dtype < ebx::kKvF32 || dtype > ebx::kKvBF16)
        return invalid("ebx_kv_materialize: dtype must be fp32, fp16 or bf16");
    if (requests < 0 || width < 1 || tokens < 0 || tokens > INT32_MAX)
        return invalid("ebx_kv_materialize: need requests >= 0, width >= 1 and 0 <= tokens < 2^31");
    // a CTA counts the elements of its tokens, kv_heads * head_dim of them, in 31 bits
    if (int64_t(p.kv_heads) * p.head_dim > INT32_MAX / 2)
        return invalid("ebx_kv_materialize: need kv_heads * head_dim < 2^30");
    if (tokens == 0) return EBX_OK;
    if (!starts || !k || !v || (requests > 0 && !tables)) return invalid("null argument");
    if (!aligned16(k) || !aligned16(v)) return invalid("ebx_kv_materialize: outputs must be 16-byte aligned");
    Device d(pool->device);
    if (d.err != cudaSuccess) return launched(d.err, "cudaSetDevice");
    return launched(ebx::launch_kv_materialize(p, tables, width, starts, first, requests, tokens, dtype, k,
                                               v, static_cast<cudaStream_t>(stream)), "ebx_kv_materialize");
}

uint64_t ebx_kv_attention_workspace_bytes(const ebx_kv_pool* pool, int32_t heads, int64_t tokens,
                                          int32_t max_new, int32_t max_length) {
    ebx::KvPool p;
    if (pool_of(pool, p) || heads < 1 || heads % p.kv_heads != 0 || tokens < 0 || tokens > INT32_MAX ||
        max_new < 0 || max_length < 0)
        return 0;
    Device d(pool->device);
    if (d.err != cudaSuccess) return 0;
    return ebx::kv_attention_workspace_bytes(p.head_dim, heads / p.kv_heads, tokens, max_new, max_length);
}

ebx_status ebx_kv_attention(const ebx_kv_pool* pool, const void* q, int64_t q_token_stride,
                            int64_t q_head_stride, int32_t heads, int32_t dtype, const int32_t* tables,
                            int32_t width, const int32_t* lengths, const int32_t* starts,
                            const int32_t* first, int32_t requests, int64_t tokens, int32_t causal,
                            int32_t window, float scale, int32_t max_new, int32_t max_length, void* out,
                            float* lse, void* workspace, uint64_t workspace_bytes, void* stream) {
    ebx::KvPool p;
    if (const char* msg = pool_of(pool, p)) return invalid(msg);
    if (dtype != ebx::kKvF16 && dtype != ebx::kKvBF16)
        return invalid("ebx_kv_attention: dtype must be fp16 or bf16");
    if (heads < 1 || heads % p.kv_heads != 0 || heads > (1 << 20))
        return invalid("ebx_kv_attention: heads must be a multiple of kv_heads");
    if (requests < 0 || requests > (1 << 20) || width < 1 || int64_t(width) * p.block_size > INT32_MAX / 2 ||
        tokens < 0 || tokens > INT32_MAX || tokens * (heads / p.kv_heads) > INT32_MAX / 2)
        return invalid("ebx_kv_attention: requests, table width or tokens out of range");
    if (window < 0 || (window > 0 && !causal)) return invalid("ebx_kv_attention: a window is causal and > 0");
    if (!std::isfinite(scale * 1.4426950408889634f)) return invalid("ebx_kv_attention: scale must be finite");
    if (max_new < 0 || max_length < 0) return invalid("ebx_kv_attention: max_new and max_length are >= 0");
    if (tokens == 0 || requests == 0) return EBX_OK;  // rows of no request are left as they are
    if (!out || !starts || !tables || !lengths) return invalid("null argument");
    ebx::KvRows rows;
    if (const char* msg = rows_of(q, q_token_stride, q_head_stride, rows)) return invalid(msg);
    if (!aligned16(out) || !aligned16(workspace))
        return invalid("ebx_kv_attention: out and workspace must be 16-byte aligned");
    Device d(pool->device);
    if (d.err != cudaSuccess) return launched(d.err, "cudaSetDevice");
    const uint64_t need = ebx::kv_attention_workspace_bytes(p.head_dim, heads / p.kv_heads, tokens, max_new, max_length);
    if (need > 0 && (!workspace || workspace_bytes < need)) {
        ebx::set_error("ebx_kv_attention: workspace smaller than ebx_kv_attention_workspace_bytes");
        return EBX_ERR_WORKSPACE;
    }
    ebx::KvAttnArgs a{};
    a.pool = p;
    a.q = rows;
    a.tables = tables;
    a.lengths = lengths;
    a.starts = starts;
    a.first = first;
    a.out = out;
    a.lse = lse;
    a.tokens = tokens;
    a.requests = requests;
    a.width = width;
    a.heads = heads;
    a.set_group(heads / p.kv_heads);
    a.causal = causal != 0;
    a.window = window < int64_t(width) * p.block_size ? window : 0;  // longer than any request: no window
    a.scale_log2 = scale * 1.4426950408889634f;
    return launched(ebx::launch_kv_attention(a, dtype == ebx::kKvBF16, max_new, max_length, workspace,
                                             static_cast<cudaStream_t>(stream)), "ebx_kv_attention");
}

}  // extern "C"
