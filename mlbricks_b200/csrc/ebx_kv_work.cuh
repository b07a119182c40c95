// ebx_kv_work.cuh -- how attention's work is shared out: row tiles, their key tiles, and the
// joining of row tiles that several CTAs worked on.
//
// The rows of request i and key/value head h are its new tokens times the `group` query heads
// that share h (row r: token r / group, head h * group + r % group), in tiles of RT rows.  A row
// tile reads the key tiles of KT tokens between the first and the last key that one of its rows
// sees.  All (request, head, row tile, key tile) units lie on one line in that order, EXTRA more
// for the begin and the end of each row tile, and every CTA takes the same length of it, so that
// ragged requests, causal masks and single long requests all fill the GPU alike.  A row tile that
// crosses the end of a CTA's length is left as partial results {O, m, l}, which kv_join_kernel adds
// up in order: no atomics, no waiting.  With `whole`, the line's units are row tiles: nothing is
// left for a join.
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

// Does this launch take request i, with n new tokens?  SHARED: with prefixes, where it chooses among groups only.
template <bool SHARED>
__device__ __forceinline__ bool kv_taken(const KvAttnArgs& a, int i, int64_t n) {
    if (SHARED && i >= a.groups) return true;
    return n * a.group >= a.least_rows && n * a.group <= a.most_rows;
}

template <bool SHARED>
__device__ __forceinline__ KvRequest kv_request(const KvAttnArgs& a, int i) {
    KvRequest r;
    if constexpr (SHARED) {
        const bool whole = i < a.groups;  // a group: every key of it is ahead of every row
        const int own = whole ? i : i - a.groups;
        const int32_t* starts = (whole ? a.group_starts : a.starts) + own;
        const int64_t lo = max(starts[0], 0), hi = min(int64_t(starts[1]), a.tokens);
        const int n = hi > lo ? int(hi - lo) : 0;
        const int64_t cap = int64_t(a.width) << a.pool.shift;
        r.length = int(min(int64_t(max(whole ? a.shared[own] : a.lengths[own], 0)), cap));
        r.begin = whole ? r.length : r.length - n;
        r.rows = kv_taken<true>(a, i, n) ? n * a.group : 0;
        r.token0 = int(lo);
        r.first = whole ? 0 : min(max(a.own_first[own], 0), r.length);
        return r;
    }
    const int64_t s0 = a.starts[i], s1 = a.starts[i + 1];
    const int64_t lo = s0 < 0 ? 0 : s0, hi = s1 > a.tokens ? a.tokens : s1;
    const int n = hi > lo ? int(hi - lo) : 0;
    const int64_t cap = int64_t(a.width) << a.pool.shift;
    const int len = a.lengths[i];
    r.length = len < 0 ? 0 : int64_t(len) > cap ? int(cap) : len;
    r.begin = r.length - n;
    r.rows = kv_taken<false>(a, i, n) ? n * a.group : 0;
    r.token0 = int(lo);
    r.first = a.first ? min(max(a.first[i], 0), r.length) : 0;
    return r;
}

// The token of row tile rows whose number among the request's tokens is n; the table row of a request.
template <bool SHARED>
__device__ __forceinline__ int kv_token(const KvAttnArgs& a, int request, const KvRequest& r, int n) {
    if (SHARED && request < a.groups) return min(max(a.list[r.token0 + n], 0), int(a.tokens) - 1);
    return r.token0 + n;
}
template <bool SHARED>
__device__ __forceinline__ int kv_table_row(const KvAttnArgs& a, int request) {
    return SHARED && request >= a.groups ? request - a.groups : request;
}

// n / group for 0 <= n < 2^31 (KvAttnArgs::set_group).
__device__ __forceinline__ int by_group(const KvAttnArgs& a, int n) {
    return int(uint64_t(uint32_t(n)) * a.group_mul >> a.group_shift);
}

// Keys [lo, hi) that some row of the tile sees, as key tiles [t0, t0 + n), n >= 1 (a tile that
// sees nothing still has its zeros to write).
template <int RT, int KT>
__device__ __forceinline__ void kv_key_tiles(const KvAttnArgs& a, const KvRequest& r, int rt, int& t0, int& n) {
    const int last = min((rt + 1) * RT, r.rows) - 1;
    const int p0 = r.begin + by_group(a, rt * RT), p1 = r.begin + by_group(a, last);
    const int hi = a.causal ? min(p1 + 1, r.length) : r.length;
    const int lo = max(r.first, a.window > 0 ? p0 - a.window + 1 : 0);
    t0 = max(lo, 0) / KT;
    n = hi > lo ? (hi + KT - 1) / KT - t0 : 1;
    n = max(n, 1);
}

// Where a CTA's share of the line begins, and how long it is.
struct KvShare {
    int64_t units;
    int per;     // every CTA's length
    int request, head, rt;
    int skip;    // units of that row tile that belong to the CTA before
};

// A CTA's walk along the line: which (request, head, row tile) it is at, and which of its key
// tiles are the CTA's.  Every warp keeps its own copy.
template <int RT, int KT, int EXTRA, bool SHARED = false>
struct KvWalk {
    int left;            // units from here to the CTA's end
    int per, request, head, rt;
    KvRequest r;
    int skip;
    // the current segment
    int t0, n;           // its key tiles
    int rest;            // key tiles of the row tile behind it, for the next CTAs
    bool begins;         // it holds the row tile's first key tile

    __device__ __forceinline__ void start(const KvAttnArgs& a, const KvShare& s) {
        left = int(s.units);  // at most per
        per = s.per;
        request = s.request;
        head = s.head;
        rt = s.rt;
        skip = s.skip;
        if (left <= 0) return;
        r = kv_request<SHARED>(a, request);
        segment(a);
    }
    __device__ __forceinline__ void segment(const KvAttnArgs& a) {
        kv_key_tiles<RT, KT>(a, r, rt, t0, n);
        rest = 0;
        begins = true;
        if (a.whole) return;
        const int before = max(skip - EXTRA, 0);
        begins = before == 0;
        t0 += before;
        n -= before;
        const int room = left - max(EXTRA - skip, 0);
        if (room < n) {
            rest = n - max(room, 0);
            n -= rest;
            if (n == 0) left = 0;  // the share ends ahead of the first key tile
        }
    }
    __device__ __forceinline__ bool done() const { return left <= 0; }
    __device__ __forceinline__ bool whole() const { return begins && rest == 0; }
    // the last CTA that works on the row tile
    __device__ __forceinline__ int last() const { return int(blockIdx.x) + (rest + per - 1) / per; }
    __device__ __forceinline__ void next(const KvAttnArgs& a) {
        left -= a.whole ? 1 : n + max(EXTRA - skip, 0);
        if (rest > 0) left = 0;
        if (left <= 0) return;
        skip = 0;
        ++rt;
        if (rt * RT >= r.rows) {
            rt = 0;
            if (++head == a.pool.kv_heads) {
                head = 0;
                do {  // units are left, so a request with rows follows
                    r = kv_request<SHARED>(a, ++request);
                } while (r.rows == 0);
            }
        }
        segment(a);
    }
};

// x / y of 64 bits, as 32 where they fit.
__device__ __forceinline__ int64_t kv_divide(int64_t x, int64_t y) {
    return ((x | y) >> 32) == 0 ? int64_t(uint32_t(x) / uint32_t(y)) : x / y;
}

// This CTA's share.  Called by all NT threads of the block.  Where there are no more requests than threads and
// none has more than kShareFew row tiles, as in decode steps, a thread counts a request's key tiles: one pass over the
// requests, one sum.  Else in two steps over windows of requests:
// a thread per request counts its row tiles, then a thread per row tile counts its key tiles, so
// that one long prompt and many short requests cost the same few loads a thread.  `scratch`:
// kShareInts ints of shared memory, free again when the last barrier in here is passed.
constexpr int kShareWindow = 1024;
constexpr int kShareInts = 3 * kShareWindow + 128;
constexpr int kShareFew = 4;

template <int RT, int KT, int EXTRA, int NT, bool SHARED = false>
__device__ __forceinline__ KvShare kv_share(const KvAttnArgs& a, int64_t least, int* scratch) {
    constexpr int W = NT / 32;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int* tiles = scratch;                       // row tiles of the window's requests ahead of i
    // key tiles of one head of request i, low and high words (a long prompt in tiles of 8 rows passes 2^32)
    uint32_t* units = reinterpret_cast<uint32_t*>(scratch + kShareWindow);
    uint32_t* carry = units + kShareWindow;
    auto units_of = [&](int i) { return int64_t(carry[i]) << 32 | units[i]; };
    int64_t* sums = reinterpret_cast<int64_t*>(scratch + 3 * kShareWindow);  // [W] and the answer
    static_assert(W + 3 <= 64, "scratch of kv_share");
    // exclusive scan over the block; total receives the sum
    auto scan = [&](int64_t v, int64_t& total) {
        int64_t x = v;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int64_t o = __shfl_up_sync(0xffffffffu, x, d);
            if (lane >= d) x += o;
        }
        __syncthreads();
        if (lane == 31) sums[warp] = x;
        __syncthreads();
        int64_t y = lane < W ? sums[lane] : 0;
#pragma unroll
        for (int d = 1; d < W; d <<= 1) {
            const int64_t o = __shfl_up_sync(0xffffffffu, y, d);
            if (lane >= d) y += o;
        }
        total = __shfl_sync(0xffffffffu, y, W - 1);
        const int64_t before = __shfl_sync(0xffffffffu, y, warp > 0 ? warp - 1 : 0);
        return x - v + (warp > 0 ? before : 0);
    };
    // fills `units` for the requests [i0, i0 + n)
    auto count = [&](int i0, int n) {
        int64_t all = 0;
        for (int b = 0; b < n; b += NT) {
            const int i = b + tid;
            int64_t rts = 0, total;
            if (i < n) {
                const int32_t* starts = a.starts;
                int at = i0 + i;
                if constexpr (SHARED) {
                    if (at < a.groups) starts = a.group_starts; else at -= a.groups;
                }
                const int64_t s0 = max(starts[at], 0), s1 = min(int64_t(starts[at + 1]), a.tokens);
                rts = s1 > s0 && kv_taken<SHARED>(a, i0 + i, s1 - s0) ? ((s1 - s0) * a.group + RT - 1) / RT : 0;
            }
            const int64_t ahead = all + scan(rts, total);
            if (i < n) {
                tiles[i] = int(ahead);
                units[i] = carry[i] = 0;
            }
            all += total;
        }
        __syncthreads();
        for (int64_t x = tid; x < all; x += NT) {
            int lo = 0, hi = n;  // the last request with tiles[lo] <= x: it has row tiles
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (tiles[mid] <= x) lo = mid; else hi = mid;
            }
            int t0, k;
            kv_key_tiles<RT, KT>(a, kv_request<SHARED>(a, i0 + lo), int(x) - tiles[lo], t0, k);
            const uint32_t more = a.whole ? 1 : k + EXTRA;
            if (atomicAdd(units + lo, more) > ~more) atomicAdd(carry + lo, 1u);
        }
        __syncthreads();
    };
    int64_t total = 0, few_units = 0, few_ahead = 0;
    bool few = a.requests <= NT;
    if (few) {
        bool many = false;
        if (tid < a.requests) {
            const KvRequest r = kv_request<SHARED>(a, tid);
            many = r.rows > kShareFew * RT;
            for (int rt = 0; rt * RT < r.rows && !many; ++rt) {
                int t0, k;
                kv_key_tiles<RT, KT>(a, r, rt, t0, k);
                few_units += a.whole ? 1 : k + EXTRA;
            }
        }
        few = !__syncthreads_or(many);
    }
    if (few) {
        int64_t all;
        few_ahead = scan(few_units, all);
        total = all * a.pool.kv_heads;
    }
    for (int i0 = 0; i0 < a.requests && !few; i0 += kShareWindow) {
        const int n = min(kShareWindow, a.requests - i0);
        count(i0, n);
        int64_t mine = 0, all;
        for (int i = tid; i < n; i += NT) mine += units_of(i);
        scan(mine, all);
        total += all * a.pool.kv_heads;
    }
    int64_t per = kv_divide(total + gridDim.x - 1, gridDim.x);
    per = per < least && !a.whole ? least : per;
    const int64_t w0 = per * blockIdx.x;
    KvShare out;
    out.units = total - w0 < per ? total - w0 : per;
    out.per = int(per < INT32_MAX ? per : INT32_MAX);
    out.request = out.head = out.rt = out.skip = 0;
    if (out.units <= 0) {
        out.units = 0;
        __syncthreads();
        return out;
    }
    if (few) {
        const int64_t u = few_units * a.pool.kv_heads, begin = few_ahead * a.pool.kv_heads;
        if (u > 0 && begin <= w0 && w0 < begin + u) {  // exactly one thread
            const int64_t head = kv_divide(w0 - begin, few_units);
            sums[W] = tid;
            sums[W + 1] = head;
            sums[W + 2] = w0 - begin - head * few_units;
        }
    }
    int64_t base = 0;  // units ahead of the window
    for (int i0 = 0; !few; i0 += kShareWindow) {
        const int n = min(kShareWindow, a.requests - i0);
        if (a.requests > kShareWindow) count(i0, n);  // else they are still there
        bool found = false;
        for (int b = 0; b < n; b += NT) {
            const int i = b + tid;
            const int64_t u = i < n ? units_of(i) * a.pool.kv_heads : 0;
            int64_t all;
            const int64_t begin = base + scan(u, all);
            if (u > 0 && begin <= w0 && w0 < begin + u) {  // exactly one thread
                const int64_t at = w0 - begin;
                sums[W] = i0 + i;
                sums[W + 1] = at / units_of(i);
                sums[W + 2] = at % units_of(i);
            }
            base += all;
            found = base > w0;
            if (found) break;
        }
        if (found) break;
    }
    __syncthreads();
    out.request = int(sums[W]);
    out.head = int(sums[W + 1]);
    // the row tile: each warp for itself, 32 at a time
    int64_t rest = sums[W + 2];
    const KvRequest r = kv_request<SHARED>(a, out.request);
    for (int rt0 = 0;; rt0 += 32) {
        int t0, k = 0;
        if ((rt0 + lane) * RT < r.rows) {
            kv_key_tiles<RT, KT>(a, r, rt0 + lane, t0, k);
            k = a.whole ? 1 : k + EXTRA;
        }
        int x = k;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int o = __shfl_up_sync(0xffffffffu, x, d);
            if (lane >= d) x += o;
        }
        const unsigned past = __ballot_sync(0xffffffffu, x > rest);
        if (past) {
            const int f = __ffs(past) - 1;
            out.rt = rt0 + f;
            out.skip = int(rest) - __shfl_sync(0xffffffffu, x - k, f);
            break;
        }
        rest -= __shfl_sync(0xffffffffu, x, 31);
    }
    __syncthreads();
    return out;
}

// ---- partial results ----------------------------------------------------------------------
// CTA c leaves at most two: part 0, which continues a row tile of a CTA before, and part 1, which
// begins one that later CTAs continue.  desc[c] tells of part 1: {1 + the row tile's first row (0:
// none), first token row, head, rows | CTAs behind c << 16}.
__device__ __forceinline__ int4 kv_desc(const KvRequest& r, int rt, int rt_rows, int head, int behind) {
    return make_int4(rt * rt_rows + 1, r.token0, head, min(rt_rows, r.rows - rt * rt_rows) | behind << 16);
}

// Weights are 2^(t - m + kShift), m at most kLag below the maximum so far: the largest is below
// 2^15 and at least 2^kShift, so that a weight 2^-21 of the largest (2^-14: the smallest normal
// fp16) still has all its 11 bits.
constexpr float kLag = 8.0f, kShift = 7.0f;
// V scale of 16 tokens that no block holds: their keys are not seen.
constexpr float kKvNone = -1.0f;

// A part: O as float4 [head_dim / 4][RT] (neighbouring rows are neighbours, for threads that hold a
// row each), then {m, l} [RT].
template <int D, int RT>
__device__ __forceinline__ float* kv_part(const KvAttnArgs& a, int cta, int slot) {
    return a.part + (2 * int64_t(cta) + slot) * RT * (D + 2);
}
template <int D, int RT>
__device__ __forceinline__ float2* kv_part_ml(const KvAttnArgs& a, int cta, int slot) {
    return reinterpret_cast<float2*>(kv_part<D, RT>(a, cta, slot) + RT * D);
}

// With prefixes a row of q has two results, over the prefix (side 0) and over what is its request's own (side 1), each whole or in
// parts; `where` says which, written by the two functions below: {-1, 0}: whole, in `sums`; else {first CTA, CTAs behind << 8 | row of the tile}, the
// CTA of the kernel for prompts as ~CTA - 1.  kv_shared_join_kernel makes one of all.
__device__ __forceinline__ void kv_whole(const KvAttnArgs& a, int side, int64_t row) {
    a.where[side * a.tokens * a.heads + row] = make_int2(-1, 0);
}
__device__ __forceinline__ void kv_begins(const KvAttnArgs& a, int side, int64_t row, bool prompt, int behind, int tile_row) {
    a.where[side * a.tokens * a.heads + row] =
        make_int2(prompt ? -2 - int(blockIdx.x) : int(blockIdx.x), behind << 8 | tile_row);
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
__device__ __forceinline__ float rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
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

// Row tiles that several CTAs worked on: CTA (c, y) joins rows 4 y .. 4 y + 3 (and so on, gridDim.y
// fours at a time: the grid goes by what the caller says of the rows) of the one that begins in CTA c, c's part 1 and then part 0 of the CTAs behind it.  Threads: 4 rows x 8 column groups x
// WAYS parts at a time.
template <int D, int RT, int WAYS, bool BF16>
__global__ void __launch_bounds__(32 * WAYS) kv_join_kernel(const __grid_constant__ KvAttnArgs a) {
    asm volatile("griddepcontrol.launch_dependents;\n\tgriddepcontrol.wait;" ::: "memory");
    constexpr int COLS = D / 32;  // float4 columns of a thread: groups of 8 apart
    __shared__ float2 s_ml[WAYS][8][4];
    __shared__ float4 s_o[COLS][WAYS][8][4];
    const int c = blockIdx.x;
    const int4 d = a.desc[c];
    const int rows = d.w & 0xffff, last = c + (d.w >> 16);
    if (d.x == 0) return;
    const int ri = threadIdx.x & 3, col = (threadIdx.x >> 2) & 7, way = threadIdx.x >> 5;
    for (int r0 = blockIdx.y * 4; r0 < rows; r0 += gridDim.y * 4) {
        const int r = r0 + ri;
        float m = -INFINITY, l = 0.0f;
        float4 o[COLS];
#pragma unroll
        for (int x = 0; x < COLS; ++x) o[x] = make_float4(0, 0, 0, 0);
        auto join = [&](float m1, float l1, const float4 (&v)[COLS]) {
            const float mn = fmaxf(m, m1);
            const float f0 = m == mn ? 1.0f : ex2(m - mn), f1 = m1 == mn ? 1.0f : ex2(m1 - mn);
#pragma unroll
            for (int x = 0; x < COLS; ++x) {
                o[x].x = o[x].x * f0 + v[x].x * f1;
                o[x].y = o[x].y * f0 + v[x].y * f1;
                o[x].z = o[x].z * f0 + v[x].z * f1;
                o[x].w = o[x].w * f0 + v[x].w * f1;
            }
            l = l * f0 + l1 * f1;
            m = mn;
        };
        if (r < rows) {
            constexpr int AHEAD = 4;  // parts on their way at once
            for (int k0 = c + way; k0 <= last; k0 += AHEAD * WAYS) {
                float4 v[AHEAD][COLS];
                float2 ml[AHEAD];
#pragma unroll
                for (int i = 0; i < AHEAD; ++i) {
                    const int k = k0 + i * WAYS, slot = k == c ? 1 : 0;
                    ml[i] = make_float2(-INFINITY, 0.0f);
                    if (k > last) continue;
                    const float4* src = reinterpret_cast<const float4*>(kv_part<D, RT>(a, k, slot));
#pragma unroll
                    for (int x = 0; x < COLS; ++x) v[i][x] = src[(x * 8 + col) * RT + r];
                    ml[i] = kv_part_ml<D, RT>(a, k, slot)[r];
                }
#pragma unroll
                for (int i = 0; i < AHEAD; ++i)
                    if (k0 + i * WAYS <= last) join(ml[i].x, ml[i].y, v[i]);
            }
        }
        s_ml[way][col][ri] = make_float2(m, l);
#pragma unroll
        for (int x = 0; x < COLS; ++x) s_o[x][way][col][ri] = o[x];
        __syncthreads();
        if (way == 0 && r < rows) {
            for (int w = 1; w < min(WAYS, last - c + 1); ++w) {
                float4 v[COLS];
#pragma unroll
                for (int x = 0; x < COLS; ++x) v[x] = s_o[x][w][col][ri];
                join(s_ml[w][col][ri].x, s_ml[w][col][ri].y, v);
            }
            const int row = d.x - 1 + r;
            const int token = by_group(a, row);
            const int64_t at = int64_t(d.y + token) * a.heads + d.z * a.group + row - token * a.group;
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
            for (int x = 0; x < COLS; ++x) {
                uint2 pk;
                pk.x = pack16<BF16>(o[x].x * inv, o[x].y * inv);
                pk.y = pack16<BF16>(o[x].z * inv, o[x].w * inv);
                *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + at * D + 4 * (x * 8 + col)) = pk;
            }
            if (a.lse && col == 0) a.lse[at] = l == 0.0f ? -INFINITY : (m + lg2(l)) * 0.6931471805599453f;
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

// The join of a launch of `ctas` CTAs whose row tiles have at most `rows` rows.
template <int D, int RT, int WAYS, bool BF16>
cudaError_t launch_join(const KvAttnArgs& a, int ctas, int rows, cudaStream_t s) {
    if (a.whole) return cudaSuccess;
    return launch_early(kv_join_kernel<D, RT, WAYS, BF16>, dim3(unsigned(ctas), unsigned((rows + 3) / 4)), 32 * WAYS, 0, s, a);
}

}  // namespace ebx
