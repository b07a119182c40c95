// ebx_kv_work.cuh -- how attention's work is shared out: row tiles, their key tiles, and the
// joining of row tiles that several CTAs worked on.
//
// The rows of request i and key/value head h are its new tokens times the `group` query heads
// that share h (row r: token r / group, head h * group + r % group), in tiles of RT rows.  A row
// tile reads the key tiles of KT tokens between the first and the last key that one of its rows
// sees.  All (request, head, row tile, key tile) units lie on one line in that order, and every
// CTA takes the same length of it, so that ragged requests, causal masks and single long
// requests all fill the GPU alike.  A row tile that crosses the end of a CTA's length is left as
// partial results {O, m, l}, which kv_join_kernel adds up in order: no atomics, no waiting.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>

#include "ebx_common.cuh"
#include "ebx_kv.h"

#include <cuda_bf16.h>

namespace ebx {

struct KvRequest {
    int length;   // tokens in the cache
    int begin;    // position of its first new token
    int rows;     // new tokens * group
    int token0;   // its first new token in q
    int first;    // keys ahead of it are not seen
};

__device__ __forceinline__ KvRequest kv_request(const KvAttnArgs& a, int i) {
    KvRequest r;
    const int64_t s0 = a.starts[i], s1 = a.starts[i + 1];
    const int64_t lo = s0 < 0 ? 0 : s0, hi = s1 > a.tokens ? a.tokens : s1;
    const int n = hi > lo ? int(hi - lo) : 0;
    const int64_t cap = int64_t(a.width) << a.pool.shift;
    const int len = a.lengths[i];
    r.length = len < 0 ? 0 : int64_t(len) > cap ? int(cap) : len;
    r.begin = r.length - n;
    r.rows = n * a.group;
    r.token0 = int(lo);
    r.first = a.first ? max(a.first[i], 0) : 0;
    return r;
}

// Keys [lo, hi) that some row of the tile sees, as key tiles [t0, t0 + n), n >= 1 (a tile that
// sees nothing still has its zeros to write).
template <int RT, int KT>
__device__ __forceinline__ void kv_key_tiles(const KvAttnArgs& a, const KvRequest& r, int rt, int& t0, int& n) {
    const int last = min((rt + 1) * RT, r.rows) - 1;
    const int p0 = r.begin + rt * RT / a.group, p1 = r.begin + last / a.group;
    const int hi = a.causal ? min(p1 + 1, r.length) : r.length;
    const int lo = max(r.first, a.window > 0 ? p0 - a.window + 1 : 0);
    t0 = max(lo, 0) / KT;
    n = hi > lo ? (hi + KT - 1) / KT - t0 : 1;
    n = max(n, 1);
}

// Units of one head of the request.
template <int RT, int KT>
__device__ __forceinline__ int64_t kv_head_units(const KvAttnArgs& a, const KvRequest& r) {
    int64_t sum = 0;
    for (int rt = 0; rt * RT < r.rows; ++rt) {
        int t0, n;
        kv_key_tiles<RT, KT>(a, r, rt, t0, n);
        sum += n;
    }
    return sum;
}

// A CTA's walk along the line: which (request, head, row tile) it is at, and which of its key
// tiles are the CTA's.  Every warp keeps its own copy.
template <int RT, int KT>
struct KvWalk {
    int64_t left;        // units from here to the CTA's end
    int request, head, rt;
    KvRequest r;
    int64_t head_units;
    int skip;            // key tiles of the current row tile that belong to the CTA before
    // the current segment
    int t0, n;           // its key tiles
    bool begins, ends;   // it holds the row tile's first / last key tile

    // at: the unit of the line at which this CTA begins, counted from the start of `req`
    __device__ __forceinline__ void start(const KvAttnArgs& a, int req, int64_t at, int64_t units) {
        left = units;
        request = req;
        head = rt = skip = 0;
        if (left <= 0) return;
        r = kv_request(a, request);
        head_units = kv_head_units<RT, KT>(a, r);
        head = int(at / head_units);
        int64_t rest = at - head * head_units;
        for (;; ++rt) {
            kv_key_tiles<RT, KT>(a, r, rt, t0, n);
            if (rest < n) break;
            rest -= n;
        }
        skip = int(rest);
        segment(a);
    }
    __device__ __forceinline__ void segment(const KvAttnArgs& a) {
        kv_key_tiles<RT, KT>(a, r, rt, t0, n);
        begins = skip == 0;
        t0 += skip;
        n -= skip;
        ends = n <= left;
        if (!ends) n = int(left);
    }
    __device__ __forceinline__ bool done() const { return left <= 0; }
    __device__ __forceinline__ void next(const KvAttnArgs& a) {
        left -= n;
        if (left <= 0) return;
        skip = 0;
        ++rt;
        if (rt * RT >= r.rows) {
            rt = 0;
            if (++head == a.pool.kv_heads) {
                head = 0;
                do {  // units are left, so a request with rows follows
                    r = kv_request(a, ++request);
                } while (r.rows == 0);
            }
        }
        segment(a);
    }
};

// Where this CTA's share begins: `request`, `at` units into it, `units` long.  Called by all
// NT threads of the block; `scratch` holds NT / 32 + 2 int64.
template <int RT, int KT, int NT>
__device__ __forceinline__ void kv_share(const KvAttnArgs& a, int64_t least, int64_t* scratch, int& request,
                                         int64_t& at, int64_t& units) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    constexpr int W = NT / 32;
    auto request_units = [&](int i) {
        if (i >= a.requests) return int64_t(0);
        const KvRequest r = kv_request(a, i);
        return kv_head_units<RT, KT>(a, r) * a.pool.kv_heads;
    };
    int64_t mine = 0;
    for (int i = tid; i < a.requests; i += NT) mine += request_units(i);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, d);
    if (lane == 0) scratch[warp] = mine;
    __syncthreads();
    int64_t total = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) total += scratch[w];
    int64_t per = (total + gridDim.x - 1) / gridDim.x;
    per = per < least ? least : per;
    const int64_t w0 = per * blockIdx.x;
    units = total - w0 < per ? total - w0 : per;
    request = 0;
    at = 0;
    if (units <= 0) {
        units = 0;
        return;
    }
    // the request that holds unit w0: scan the requests' units NT at a time
    int64_t base = 0;
    for (int i0 = 0;; i0 += NT) {
        const int64_t u = request_units(i0 + tid);
        int64_t v = u;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int64_t o = __shfl_up_sync(0xffffffffu, v, d);
            if (lane >= d) v += o;
        }
        __syncthreads();
        if (lane == 31) scratch[warp] = v;
        __syncthreads();
        int64_t ahead = base;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            if (w < warp) ahead += scratch[w];
            base += scratch[w];
        }
        const int64_t begin = ahead + v - u;
        if (u > 0 && begin <= w0 && w0 < begin + u) {  // exactly one thread
            scratch[W] = i0 + tid;
            scratch[W + 1] = w0 - begin;
        }
        if (base > w0) break;
    }
    __syncthreads();
    request = int(scratch[W]);
    at = scratch[W + 1];
}

// ---- partial results ----------------------------------------------------------------------
// CTA c leaves at most two: part 0, which continues a row tile of the CTA before, and part 1,
// which begins one that the next CTA continues.  desc = {1 + row tile's first row and ends flag
// (0: none), first token row, head, rows}.
constexpr int kKvEnds = 1 << 30;

__device__ __forceinline__ int4 kv_desc(const KvRequest& r, int rt, int rt_rows, int head, bool ends) {
    return make_int4((rt * rt_rows + 1) | (ends ? kKvEnds : 0), r.token0, head,
                     min(rt_rows, r.rows - rt * rt_rows));
}

// Weights are 2^(t - m + kShift), m at most kLag below the maximum so far: the largest is below
// 2^15, and of the fp16 range nothing is left unused below it (a weight 2^-22 of the largest
// still has all its 11 bits).
constexpr float kLag = 8.0f, kShift = 7.0f;
// V scale of 16 tokens that no block holds: their keys are not seen.
constexpr float kKvNone = -1.0f;

template <bool BF16>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
    if constexpr (BF16) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&b);
    } else {
        return pack_half2(lo, hi);
    }
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float lg2(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ void kv_tma_2d(uint32_t dst, const CUtensorMap* map, int c0, int c1, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4}], [%2];\n" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1)
        : "memory");
}

// Two int8 codes (already xor 0x80: code + 128) as fp16: 0x64 above a byte is 1024 + byte.
__device__ __forceinline__ uint32_t codes_to_half2(uint32_t w, uint32_t sel) {
    return hsub2_u(__byte_perm(w, 0x64646464u, sel), 0x64806480u);  // - 1152
}

// Row tiles that several CTAs worked on: CTA (c, y) joins the one that begins in CTA c, its rows
// y, y + gridDim.y, ..., reading c's part 1 and then part 0 of the CTAs after it until one ends it.
template <int D, int RT, bool BF16>
__global__ void __launch_bounds__(128) kv_join_kernel(const __grid_constant__ KvAttnArgs a, int ctas) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    constexpr int LANES = D / 4;            // threads of a row, 4 values each
    constexpr int WAYS = 128 / LANES;       // parts of a row read at once
    __shared__ float s_m[WAYS][LANES], s_l[WAYS][LANES];
    __shared__ float4 s_o[WAYS][LANES];
    __shared__ int s_last;
    const int c = blockIdx.x;
    const int4 d1 = a.desc[2 * c + 1];
    if (d1.x == 0) return;
    if (threadIdx.x == 0) s_last = ctas - 1;
    for (int base = c + 1;; base += 128) {  // the CTA that ends the row tile
        const int k = base + int(threadIdx.x);
        const bool end = k >= ctas - 1 || (a.desc[2 * k].x & kKvEnds) != 0;
        const bool any = __syncthreads_or(end);
        if (end) atomicMin(&s_last, k);
        if (any) break;
    }
    __syncthreads();
    const int last = s_last;
    const int lane = threadIdx.x % LANES, way = threadIdx.x / LANES;
    for (int r = blockIdx.y; r < d1.w; r += gridDim.y) {
        float m = -INFINITY, l = 0.0f;
        float4 o = make_float4(0, 0, 0, 0);
        for (int k = c + way; k <= last; k += WAYS) {
            const float* src = a.part + ((2 * int64_t(k) + (k == c ? 1 : 0)) * RT + r) * (D + 2);
            const float2 v0 = *reinterpret_cast<const float2*>(src + 4 * lane);
            const float2 v1 = *reinterpret_cast<const float2*>(src + 4 * lane + 2);
            const float2 ml = *reinterpret_cast<const float2*>(src + D);
            const float mn = fmaxf(m, ml.x);
            const float f0 = m == mn ? 1.0f : ex2(m - mn), f1 = ml.x == mn ? 1.0f : ex2(ml.x - mn);
            o.x = o.x * f0 + v0.x * f1; o.y = o.y * f0 + v0.y * f1;
            o.z = o.z * f0 + v1.x * f1; o.w = o.w * f0 + v1.y * f1;
            l = l * f0 + ml.y * f1;
            m = mn;
        }
        s_m[way][lane] = m;
        s_l[way][lane] = l;
        s_o[way][lane] = o;
        __syncthreads();
        if (way == 0) {
#pragma unroll
            for (int w = 1; w < WAYS; ++w) {
                const float m1 = s_m[w][lane];
                const float4 v = s_o[w][lane];
                const float mn = fmaxf(m, m1);
                const float f0 = m == mn ? 1.0f : ex2(m - mn), f1 = m1 == mn ? 1.0f : ex2(m1 - mn);
                o.x = o.x * f0 + v.x * f1; o.y = o.y * f0 + v.y * f1;
                o.z = o.z * f0 + v.z * f1; o.w = o.w * f0 + v.w * f1;
                l = l * f0 + s_l[w][lane] * f1;
                m = mn;
            }
            const int row = (d1.x & (kKvEnds - 1)) - 1 + r;
            const int64_t at = int64_t(d1.y + row / a.group) * a.heads + d1.z * a.group + row % a.group;
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            uint2 pk;
            pk.x = pack16<BF16>(o.x * inv, o.y * inv);
            pk.y = pack16<BF16>(o.z * inv, o.w * inv);
            *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + at * D + 4 * lane) = pk;
            if (a.lse && lane == 0) a.lse[at] = l == 0.0f ? -INFINITY : (m + lg2(l)) * 0.6931471805599453f;
        }
        __syncthreads();
    }
}

// Codes as rows of head_dim bytes, in boxes of box_rows swizzled over the row's own width; boxes
// past the pool read as zeros.
inline bool code_map(CUtensorMap* map, const int8_t* codes, const KvPool& p, int box_rows) {
    auto fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(tensor_map_encoder());
    if (!fn) return false;
    const cuuint64_t dims[2] = {cuuint64_t(p.head_dim), cuuint64_t(p.blocks) * p.kv_heads * p.block_size};
    const cuuint64_t strides[1] = {cuuint64_t(p.head_dim)};
    const cuuint32_t box[2] = {cuuint32_t(p.head_dim), cuuint32_t(box_rows)};
    const cuuint32_t estr[2] = {1, 1};
    const CUtensorMapSwizzle sw = p.head_dim == 128 ? CU_TENSOR_MAP_SWIZZLE_128B
                                  : p.head_dim == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_32B;
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<int8_t*>(codes), dims, strides, box, estr,
              CU_TENSOR_MAP_INTERLEAVE_NONE, sw, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// The join of a launch of `ctas` CTAs, started while the last of them still run.
template <int D, int RT, bool BF16>
cudaError_t launch_join(const KvAttnArgs& a, int ctas, int ways, cudaStream_t s) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(ctas), unsigned(ways));
    cfg.blockDim = dim3(128);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kv_join_kernel<D, RT, BF16>, a, ctas);
}

// Reads (and clears) a translation unit's status word; synchronizes `s`.
inline cudaError_t read_status_word(const int& word, int* status, bool clear, cudaStream_t s) {
    void* p = nullptr;
    cudaError_t e = cudaGetSymbolAddress(&p, word);
    if (e == cudaSuccess) e = cudaMemcpyAsync(status, p, sizeof(int), cudaMemcpyDeviceToHost, s);
    if (e == cudaSuccess) e = cudaStreamSynchronize(s);
    if (e == cudaSuccess && clear) e = cudaMemsetAsync(p, 0, sizeof(int), s);
    if (e == cudaSuccess && clear) e = cudaStreamSynchronize(s);
    return e;
}

}  // namespace ebx
