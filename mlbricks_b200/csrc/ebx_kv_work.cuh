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

}  // namespace ebx
