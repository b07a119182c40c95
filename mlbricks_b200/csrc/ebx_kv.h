// ebx_kv.h -- the 8-bit paged key/value cache: arguments and launchers shared by the
// ebx_kv_*.cu translation units.
//
// A pool holds, for keys and for values, int8 codes [blocks][kv_heads][block_size][head_dim]
// and one fp32 scale for each (block, head); value = code * scale.  A request's tokens lie in
// the blocks that its row of the block table names, block_size of them in each.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace ebx {

constexpr int kKvMaxRequests = 16384;  // ebx_kv_plan keeps 12 bytes a request in shared memory
constexpr int kKvF32 = 0, kKvF16 = 1, kKvBF16 = 2;  // dtype codes of the C ABI

struct KvPool {
    int8_t* k_codes;
    float* k_scales;
    int8_t* v_codes;
    float* v_scales;
    int blocks, kv_heads, block_size, head_dim;
    int shift;  // log2(block_size)
};

struct KvPlanArgs {
    const int32_t* past;
    const int32_t* added;
    int32_t* tables;
    int32_t* free_ring;
    const int64_t* ring;
    int64_t* ring_out;
    int32_t* lengths;
    int32_t* starts;
    int64_t* slots;
    int32_t* positions;
    int64_t tokens;
    int requests, width, shift, free_size;
};

// A 16-bit tensor [tokens, heads, head_dim] whose last dimension is contiguous; strides in elements.
struct KvRows {
    const uint16_t* p;
    int64_t token_stride, head_stride;
};

struct KvAttnArgs {
    KvPool pool;
    KvRows q;
    const int32_t* tables;
    const int32_t* lengths;
    const int32_t* starts;
    const int32_t* first;  // may be null: every key from 0 on
    void* out;
    float* lse;            // may be null
    int64_t tokens;
    int requests, width, heads, group;
    int causal, window;
    int whole;             // row tiles are not shared among CTAs
    int least_rows, most_rows;  // the launch takes requests with that many rows (tokens * group)
    float scale_log2;      // softmax scale * log2(e)
    uint32_t group_mul, group_shift;  // n / group = n * group_mul >> group_shift
    // partial results of row tiles that several CTAs share
    float* part;           // [grid][2][rows][head_dim + 2]
    int4* desc;            // [grid]

    // With 2^(k-1) < g <= 2^k and mul = ceil(2^(31+k) / g), mul * g exceeds 2^(31+k) by less than
    // g <= 2^k, so n * mul >> (31 + k) is n / g for every n < 2^31.
    void set_group(int g) {
        group = g;
        uint32_t k = 0;
        while ((1u << k) < uint32_t(g)) ++k;
        group_shift = 31 + k;
        group_mul = uint32_t(((uint64_t(1) << group_shift) + uint32_t(g) - 1) / uint32_t(g));
    }
};

cudaError_t launch_kv_plan(const KvPlanArgs& a, cudaStream_t s);
cudaError_t launch_kv_append(const KvPool& pool, const KvRows& k, const KvRows& v, const int64_t* slots,
                             int64_t tokens, bool bf16, cudaStream_t s);
cudaError_t launch_kv_materialize(const KvPool& pool, const int32_t* tables, int width,
                                  const int32_t* starts, const int32_t* first, int requests,
                                  int64_t tokens, int dtype, void* k, void* v, cudaStream_t s);
uint64_t kv_attention_workspace_bytes(int head_dim, int group, int64_t tokens, int max_new, int max_length);
cudaError_t launch_kv_attention(KvAttnArgs a, bool bf16, int max_new, int max_length, void* ws, cudaStream_t s);
cudaError_t read_kv_status(int* status, bool clear, cudaStream_t s);

// ebx_kv_prompt.cu: the same for many rows.
uint64_t kv_prompt_workspace_bytes(int head_dim, int sms);
cudaError_t launch_kv_prompt(const KvAttnArgs& a, bool bf16, void* ws, int dev, cudaStream_t s);
cudaError_t read_kv_prompt_status(int* status, bool clear, cudaStream_t s);

// A launch that may begin while the grid before it ends: the kernel waits (griddepcontrol.wait)
// for that grid's end before it touches memory that calls share.
template <class... P, class... A>
cudaError_t launch_early(void (*kern)(P...), dim3 grid, int threads, size_t smem, cudaStream_t s, const A&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(unsigned(threads));
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, P(args)...);
}

// ebx_gemm.cu: cuTensorMapEncodeTiled of the loaded driver (null without one).
void* tensor_map_encoder();
int gemm_sm_count(int dev);

}  // namespace ebx
