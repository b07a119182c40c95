// ebx_kv_cache.cu -- the 8-bit paged key/value cache: who owns which block (plan), writing
// keys and values (append), and reading them back (materialize).  No reference counterpart:
// the reference's caches (mlbricks/cache.py) hold whole 16-bit tensors.
#include <algorithm>

#include "ebx_common.cuh"
#include "ebx_kv.h"

#include <cuda_bf16.h>

namespace ebx {
namespace {

// ---- plan ---------------------------------------------------------------------------------

constexpr int kPlanThreads = 256;

// Inclusive scan over the block; `total` receives the sum.
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t* warp_sums, int64_t& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int64_t u = __shfl_up_sync(0xffffffffu, v, d);
        if (lane >= d) v += u;
    }
    __syncthreads();  // the previous round's sums have been read
    if (lane == 31) warp_sums[warp] = v;
    __syncthreads();
    total = 0;
#pragma unroll
    for (int w = 0; w < kPlanThreads / 32; ++w) {
        if (w == warp) v += total;
        total += warp_sums[w];
    }
    return v;
}

// Request i holds past[i] tokens and adds added[i]; it needs ceil((past + added) / B) -
// ceil(past / B) more blocks.  With before[i] the sum of the needs of the requests ahead of it,
// it gets entries before[i].. of the free ring if they are there, so requests are served in
// order and the exclusive sums alone say who gets what.  A request that needs more blocks than its
// row holds, or whose tokens end past the room for slots (which counts in 31 bits), gets nothing;
// starts end at the room.  added[i] < 0 releases the request: its blocks go behind the ring's tail.  A new block always begins with a new token, so the
// threads that write the tokens' slots also write the table.
// Every CTA computes the sums for itself (a few loads per thread: cheaper than a second
// launch or a grid barrier) and then writes its share of the tokens.  What bounds it is latency: the
// lengths, the sums, a token's binary search, its block (64 requests of one token 7 us, 1000 requests
// with 120 thousand tokens 12 us, from cold caches; the 1.5 MB alone would take 0.2 us).
__global__ void __launch_bounds__(kPlanThreads) kv_plan_kernel(KvPlanArgs a) {
    asm volatile("griddepcontrol.launch_dependents;\n\tgriddepcontrol.wait;" ::: "memory");
    extern __shared__ int32_t plan_smem[];
    int32_t* s_start = plan_smem;                 // [requests]: first token
    int32_t* s_before = s_start + a.requests;     // blocks taken ahead of it, -1: refused
    int32_t* s_gone = s_before + a.requests;      // blocks released ahead of it
    __shared__ int64_t warp_sums[kPlanThreads / 32];
    __shared__ int s_taken;
    __shared__ unsigned long long s_short;  // whole rows of counts may be out of range, and still add up
    const int tid = threadIdx.x;
    const int bsize = 1 << a.shift;
    // A ring that claims more blocks than its size holds the first of them.  Counters past 2^62 begin
    // anew at their place, so that they never pass 2^63.
    const int64_t begin = max(a.ring[0], int64_t(0));
    const int64_t avail = min(max(a.ring[1], begin) - begin, int64_t(a.free_size));  // blocks to give
    const int64_t room = a.free_size - avail;                                        // places for released ones
    const int64_t head = begin >> 62 ? begin % a.free_size : begin, tail = head + avail;
    const uint32_t size = uint32_t(a.free_size);
    const uint32_t front = uint32_t(head % a.free_size), back = uint32_t(tail % a.free_size);
    auto wrapped = [&](uint32_t place) { return place < size ? place : place - size; };  // place < 2 size < 2^32
    if (tid == 0) {
        s_taken = 0;
        s_short = 0;
    }
    int64_t tokens = 0, blocks = 0, released = 0;
    for (int base = 0; base < a.requests; base += kPlanThreads) {
        const int i = base + tid;
        int64_t add = 0, need = 0, wanted = 0, gone = 0;
        bool refused = false, live = false;
        if (i < a.requests) {
            live = a.added[i] >= 0;
            add = live ? a.added[i] : 0;
        }
        int64_t t_tok, t_need, t_gone;
        const int64_t i_tok = block_scan(add, warp_sums, t_tok);
        if (i < a.requests) {
            const int64_t past = max(a.past[i], 0);
            const int64_t had = (past + bsize - 1) >> a.shift;
            gone = live ? 0 : min(had, int64_t(a.width));
            wanted = ((past + add + bsize - 1) >> a.shift) - had;
            refused = had + wanted > a.width || (add > 0 && tokens + i_tok > a.tokens);
            need = refused ? 0 : wanted;
        }
        const int64_t i_need = block_scan(need, warp_sums, t_need);
        const int64_t i_gone = block_scan(gone, warp_sums, t_gone);
        if (i < a.requests) {
            const int64_t before = blocks + i_need - need;
            const bool fits = live && !refused && (need == 0 || before + need <= avail);
            s_start[i] = int32_t(min(tokens + i_tok - add, a.tokens));
            s_before[i] = !fits ? -1 : need > 0 ? int32_t(before) : 0;
            s_gone[i] = int32_t(min(released + i_gone - gone, room));
            if (fits && need > 0) atomicMax(&s_taken, int(before + need));
            if (!fits && wanted > 0) atomicAdd(&s_short, static_cast<unsigned long long>(wanted));
        }
        tokens += t_tok;
        blocks += t_need;
        released += t_gone;
    }
    __syncthreads();

    const int64_t gtid = int64_t(blockIdx.x) * kPlanThreads + tid;
    const int64_t gthreads = int64_t(gridDim.x) * kPlanThreads;
    if (gtid == 0) {
        a.starts[a.requests] = int32_t(min(tokens, a.tokens));
        a.ring_out[0] = head + s_taken;
        a.ring_out[1] = tail + min(released, room);
        a.ring_out[2] = int64_t(s_short);
        a.ring_out[3] = tokens;
    }
    for (int64_t i = gtid; i < a.requests; i += gthreads) {
        a.starts[i] = s_start[i];
        const int add = a.added[i], past = max(a.past[i], 0);
        a.lengths[i] = add < 0 ? 0 : s_before[i] < 0 ? past : past + add;
    }
    // released blocks, a warp to a request
    for (int64_t i = gtid >> 5; i < a.requests; i += gthreads >> 5) {
        if (a.added[i] >= 0) continue;
        const int64_t had = min((int64_t(max(a.past[i], 0)) + bsize - 1) >> a.shift, int64_t(a.width));
        const int left = int(min(had, room - s_gone[i]));
        for (int j = tid & 31; j < left; j += 32)
            a.free_ring[wrapped(back + s_gone[i] + j)] = a.tables[i * a.width + j];
    }
    for (int64_t t = gtid; t < a.tokens; t += gthreads) {
        int64_t slot = -1;
        int place = 0;
        if (t < tokens) {
            int lo = 0, hi = a.requests;  // the last request that starts at or before t
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (s_start[mid] <= t) lo = mid; else hi = mid;
            }
            const int past = max(a.past[lo], 0);
            place = int(min(past + t - s_start[lo], int64_t(INT32_MAX)));  // past it: a refused request's
            const int before = s_before[lo];
            if (before >= 0) {
                const int column = place >> a.shift;
                const int fresh = column - int((int64_t(past) + bsize - 1) >> a.shift);
                int32_t* entry = a.tables + int64_t(lo) * a.width + column;
                int id;
                if (fresh >= 0) {
                    id = a.free_ring[wrapped(front + before + fresh)];
                    if ((place & (bsize - 1)) == 0) *entry = id;
                } else {
                    id = *entry;
                }
                slot = id < 0 ? -1 : (int64_t(id) << a.shift) + (place & (bsize - 1));
            }
        }
        a.slots[t] = slot;
        a.positions[t] = place;
    }
}

// ---- append -------------------------------------------------------------------------------

constexpr int kAppendWarps = 4;

template <bool BF16>
__device__ __forceinline__ float2 unpack16(uint32_t v) {
    if constexpr (BF16) {
        return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
    } else {
        return __half22float2(*reinterpret_cast<const __half2*>(&v));
    }
}

// rint(x / s) of eight values of one 16-byte load as int8 codes.  r = 1 / s, so y = x * r is within
// 2^-22 |y| < 2^-15 of the correctly rounded x / s (|y| <= 127): unless y is that near to a tie, both
// round to the same integer.  Near one, or where r is infinite (a subnormal s), the division is done.
// Rounding adds 1.5 * 2^23; the low byte of the sum is the code.
template <bool BF16>
__device__ __forceinline__ uint2 quant8(const uint4& x, float s, float r) {
    constexpr float kMagic = 12582912.0f;
    const uint32_t in[4] = {x.x, x.y, x.z, x.w};
    uint32_t c[8];
    float off = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = unpack16<BF16>(in[i]);
        const float y0 = f.x * r, y1 = f.y * r;
        const float n0 = y0 + kMagic, n1 = y1 + kMagic;
        off = fmaxf(off, fmaxf(fabsf(y0 - (n0 - kMagic)), fabsf(y1 - (n1 - kMagic))));
        c[2 * i] = __float_as_uint(n0);
        c[2 * i + 1] = __float_as_uint(n1);
    }
    if (off > 0.5f - 0x1p-15f || isinf(r)) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = unpack16<BF16>(in[i]);
            c[2 * i] = uint32_t(min(max(__float2int_rn(__fdiv_rn(f.x, s)), -127), 127));
            c[2 * i + 1] = uint32_t(min(max(__float2int_rn(__fdiv_rn(f.y, s)), -127), 127));
        }
    }
    uint2 out;
    out.x = __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
    out.y = __byte_perm(__byte_perm(c[4], c[5], 0x0040), __byte_perm(c[6], c[7], 0x0040), 0x5410);
    return out;
}

// A run is a maximal sequence of tokens whose slots follow one another inside one block; a
// warp takes a run for one head, of keys or of values:
//   s = max(s_old, max|x| / 127),  code = rint(x / s),
// s_old = the block's scale if the run does not begin the block (its earlier tokens then keep
// their codes, or are moved to the larger scale: rint(code * s_old / s)), else 0.  A value that
// is not finite makes the scale NaN, so that whatever reads the block shows it.
// Runs, not blocks, are the unit because the slots alone then say everything: no atomics, no second
// pass over other warps' tokens.  A run's values stay in registers between the largest and the codes
// (up to 16 tokens at head_dim 128; longer ones are read again from L2).  What bounds it: 27 424
// tokens of 8 heads of 128 in bf16 take 42 us = 4.0 TB/s of 168 MB.  Nothing is full (DRAM 40 %, the
// integer pipe 51 %, the issue slots 62 %): a warp takes its runs in turn, load, largest, codes, store,
// and waits for memory at each, with a third of an SM's warps there to fill in.  With a division for
// each value it was 78 us.
template <int D, bool BF16>
__global__ void __launch_bounds__(kAppendWarps * 32)
    kv_append_kernel(KvPool pool, KvRows k, KvRows v, const int64_t* slots, int64_t tokens, int span) {
    asm volatile("griddepcontrol.launch_dependents;\n\tgriddepcontrol.wait;" ::: "memory");
    constexpr int kLanes = D / 8;         // lanes that share a token, 8 values each
    constexpr int kPer = 32 / kLanes;     // tokens in a warp's load
    constexpr int kHold = 8;              // loads held in registers
    const int lane = threadIdx.x & 31;
    const int64_t item = int64_t(blockIdx.x) * kAppendWarps + (threadIdx.x >> 5);
    const int h = int(item % pool.kv_heads);
    const int64_t t0 = item / pool.kv_heads * span;
    if (t0 >= tokens) return;
    const bool values = blockIdx.y != 0;
    const KvRows x = values ? v : k;
    int8_t* codes = values ? pool.v_codes : pool.k_codes;
    float* scales = values ? pool.v_scales : pool.k_scales;
    const int bsize = pool.block_size;
    const int64_t most = int64_t(pool.blocks) << pool.shift;
    const int part = lane % kLanes, sub = lane / kLanes;

    // the window's tokens, a lane each: which begin a run, which go on with one
    const int64_t mine = t0 + lane < tokens ? slots[t0 + lane] : -1;
    int64_t prev = __shfl_up_sync(0xffffffffu, mine, 1);
    if (lane == 0) prev = t0 > 0 ? slots[t0 - 1] : -1;
    const bool held = mine >= 0 && mine < most;
    const bool goes_on = held && (mine & (bsize - 1)) != 0 && prev == mine - 1;
    const unsigned going = __ballot_sync(0xffffffffu, goes_on);
    unsigned begin = __ballot_sync(0xffffffffu, held && !goes_on && lane < span);
    for (; begin != 0; begin &= begin - 1) {
        const int first = __ffs(begin) - 1;
        const int64_t t = t0 + first, slot = __shfl_sync(0xffffffffu, mine, first);
        const int off = int(slot & (bsize - 1));
        int n = first == 31 ? 1 : __ffs(~(going >> (first + 1)));  // the run's length in the window
        if (first + n == 32) {
            for (int base = 32;; base += 32) {
                const int j = base - first + lane;
                const bool in = off + j < bsize && t + j < tokens && slots[t + j] == slot + j;
                const unsigned m = __ballot_sync(0xffffffffu, in);
                n = base - first + (m == 0xffffffffu ? 32 : __ffs(~m) - 1);
                if (m != 0xffffffffu) break;
            }
        }
        const uint16_t* src = x.p + t * x.token_stride + h * x.head_stride + part * 8;
        uint4 hold[kHold];
        uint32_t top = 0;
        for (int base = 0; base < n; base += kHold * kPer) {
#pragma unroll
            for (int i = 0; i < kHold; ++i) {
                const int j = base + i * kPer + sub;
                hold[i] = j < n ? __ldg(reinterpret_cast<const uint4*>(src + j * x.token_stride))
                                : make_uint4(0, 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < kHold; ++i) {
                // sizes of 16-bit floats order as their bits do, infinities and NaN above the rest
                const uint32_t m = 0x7fff7fffu;
                top = __vmaxu2(top, __vmaxu2(__vmaxu2(hold[i].x & m, hold[i].y & m),
                                             __vmaxu2(hold[i].z & m, hold[i].w & m)));
            }
        }
        top = max(top & 0xffffu, top >> 16);
        top = __reduce_max_sync(0xffffffffu, top);
        const float most_abs = top >= (BF16 ? 0x7f80u : 0x7c00u) ? __uint_as_float(0x7fc00000u)
                                                                 : unpack16<BF16>(top).x;
        const int64_t cell = (slot >> pool.shift) * pool.kv_heads + h;
        const float fresh = __fdiv_rn(most_abs, 127.0f);
        const float old = off != 0 ? scales[cell] : 0.0f;
        // the larger of the two, or NaN if either is
        const float s = isnan(old) || old > fresh ? old : fresh;
        int8_t* dst = codes + (cell << pool.shift) * D;
        if (off != 0 && s > old) {  // the block's earlier tokens move to the larger scale
            const float ratio = __fdiv_rn(old, s);
            uint4* w = reinterpret_cast<uint4*>(dst);
#pragma unroll 4
            for (int j = lane; j < off * (D / 16); j += 32) {
                const uint4 c = w[j];
                uint32_t in[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    uint32_t r = 0;
#pragma unroll
                    for (int b = 0; b < 4; ++b)
                        r |= (uint32_t(__float2int_rn(float(int8_t(in[q] >> (8 * b))) * ratio)) & 0xffu) << (8 * b);
                    in[q] = r;
                }
                w[j] = make_uint4(in[0], in[1], in[2], in[3]);
            }
        }
        const bool live = s > 0.0f;  // neither an all-zero block nor NaN
        const float r = __frcp_rn(s);
        for (int base = 0; base < n; base += kHold * kPer) {
            if (n > kHold * kPer) {  // the run did not fit the registers: read it again (L2)
#pragma unroll
                for (int i = 0; i < kHold; ++i) {
                    const int j = base + i * kPer + sub;
                    if (j < n) hold[i] = __ldg(reinterpret_cast<const uint4*>(src + j * x.token_stride));
                }
            }
#pragma unroll
            for (int i = 0; i < kHold; ++i) {
                const int j = base + i * kPer + sub;
                if (j >= n) continue;
                const uint2 c = live ? quant8<BF16>(hold[i], s, r) : make_uint2(0, 0);
                *reinterpret_cast<uint2*>(dst + (off + j) * D + part * 8) = c;
            }
        }
        __syncwarp();  // every lane has read the old scale
        if (lane == 0) scales[cell] = s;
    }
}

// ---- materialize --------------------------------------------------------------------------

constexpr int kMatThreads = 256;
constexpr int kMatTokens = 16;  // tokens of a CTA

// Eight codes times their scale, rounded to the type DT, at out[at].
template <int DT>
__device__ __forceinline__ void store8(void* out, int64_t at, uint32_t lo, uint32_t hi, float scale) {
    float f[8];
#pragma unroll
    for (int b = 0; b < 8; ++b) f[b] = float(int8_t((b < 4 ? lo : hi) >> (8 * (b & 3)))) * scale;
    if constexpr (DT == kKvF32) {
        float4* p = reinterpret_cast<float4*>(static_cast<float*>(out) + at);
        p[0] = make_float4(f[0], f[1], f[2], f[3]);
        p[1] = make_float4(f[4], f[5], f[6], f[7]);
    } else {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (DT == kKvF16) {
                w[i] = pack_half2(f[2 * i], f[2 * i + 1]);
            } else {
                const __nv_bfloat162 b = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
                w[i] = *reinterpret_cast<const uint32_t*>(&b);
            }
        }
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(out) + at) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// out[t, h, :] = code * scale, rounded once: token t is place first[i] + t - starts[i] of the
// request i that it falls into.  Tokens that no request has, or whose place has no block, are 0.
// One pass: 499 MB in 86 us = 5.8 TB/s, 0.89 of a copy's rate.  One item a thread at a time: two or
// four unrolled, or smaller and larger CTAs, were 2 to 14 % slower.
template <int DT>
__global__ void __launch_bounds__(kMatThreads)
    kv_materialize_kernel(KvPool pool, const int32_t* tables, int width, const int32_t* starts,
                          const int32_t* first, int requests, int64_t tokens, void* k, void* v) {
    asm volatile("griddepcontrol.launch_dependents;\n\tgriddepcontrol.wait;" ::: "memory");
    __shared__ int64_t s_slot[kMatTokens];
    const int64_t t0 = int64_t(blockIdx.x) * kMatTokens;
    if (threadIdx.x < kMatTokens) {
        const int64_t t = t0 + threadIdx.x;
        int64_t slot = -1;
        if (t < tokens && t >= starts[0] && t < starts[requests]) {
            int lo = 0, hi = requests;
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (starts[mid] <= t) lo = mid; else hi = mid;
            }
            const int64_t place = (first ? int64_t(first[lo]) : 0) + t - starts[lo];
            const int64_t column = place >> pool.shift;
            if (place >= 0 && column < width) {
                const int id = tables[int64_t(lo) * width + column];
                if (id >= 0 && id < pool.blocks)
                    slot = (int64_t(id) << pool.shift) + (place & (pool.block_size - 1));
            }
        }
        s_slot[threadIdx.x] = slot;
    }
    __syncthreads();
    const int per_head = pool.head_dim / 16;  // 16 codes a thread: 16 bytes in, 32 out of each side
    const int per_token = pool.kv_heads * per_head;
    const int64_t left = tokens - t0;
    const int work = int(left < kMatTokens ? left : kMatTokens) * per_token;
#pragma unroll 1
    for (int w = threadIdx.x; w < work; w += kMatThreads) {
        const int j = w / per_token, rest = w - j * per_token;
        const int h = rest / per_head, part = rest - h * per_head;
        const int64_t slot = s_slot[j];
        uint4 ck = make_uint4(0, 0, 0, 0), cv = make_uint4(0, 0, 0, 0);
        float sk = 0.0f, sv = 0.0f;
        if (slot >= 0) {
            const int64_t cell = (slot >> pool.shift) * pool.kv_heads + h;
            const int64_t at = ((cell << pool.shift) + (slot & (pool.block_size - 1))) * pool.head_dim + part * 16;
            ck = __ldg(reinterpret_cast<const uint4*>(pool.k_codes + at));
            cv = __ldg(reinterpret_cast<const uint4*>(pool.v_codes + at));
            sk = __ldg(pool.k_scales + cell);
            sv = __ldg(pool.v_scales + cell);
        }
        const int64_t to = ((t0 + j) * pool.kv_heads + h) * pool.head_dim + part * 16;
        store8<DT>(k, to, ck.x, ck.y, sk);
        store8<DT>(k, to + 8, ck.z, ck.w, sk);
        store8<DT>(v, to, cv.x, cv.y, sv);
        store8<DT>(v, to + 8, cv.z, cv.w, sv);
    }
}

}  // namespace

cudaError_t launch_kv_plan(const KvPlanArgs& a, cudaStream_t s) {
    const size_t smem = size_t(a.requests) * 12;
    if (smem > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(
            kv_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kKvMaxRequests * 12);
        if (e != cudaSuccess) return e;
    }
    const int64_t work = std::max<int64_t>(a.tokens, a.requests);
    // Every CTA repeats the sums, so more of them pay where the tokens are many and the requests few.
    // At most 148 / 592 / 1184 of them, captured: 64 requests of 2048 tokens 5.3 / 4.9 / 4.9 us, 16 of 8000
    // 4.9 / 4.6 / 4.6, but 1000 of 120 9.5 / 12.8 / 12.8.
    const int64_t grid = std::min<int64_t>((work + kPlanThreads - 1) / kPlanThreads, 592);
    return launch_early(kv_plan_kernel, dim3(unsigned(std::max<int64_t>(grid, 1))), kPlanThreads, smem, s, a);
}

cudaError_t launch_kv_append(const KvPool& pool, const KvRows& k, const KvRows& v, const int64_t* slots,
                             int64_t tokens, bool bf16, cudaStream_t s) {
    if (tokens <= 0) return cudaSuccess;
    // A warp looks through `span` tokens for the runs that begin there: 16, or one when there are few.  The
    // host does not know whether the tokens follow one another.  If they do, 16 spares reading slots (8 heads of
    // 128, 16 / one: 512 tokens 9.4 / 10.6 us, 2048 tokens 18.5 / 24.0); if each is in a block of its own, a warp has
    // 16 runs to take in turn (64 tokens 19.8 / 3.2 us, 512 tokens 20.2 / 7.0, 2048 tokens 30.2 / 21.6).  So
    // one for as many tokens as steps bring.
    const int span = tokens * pool.kv_heads <= 4096 ? 1 : 16;
    const int64_t items = (tokens + span - 1) / span * pool.kv_heads;
    const int64_t grid = (items + kAppendWarps - 1) / kAppendWarps;
    if (grid > INT32_MAX) return cudaErrorInvalidValue;
    const dim3 g{unsigned(grid), 2};
#define EBX_KV_APPEND(DD)                                                                            \
    bf16 ? launch_early(kv_append_kernel<DD, true>, g, kAppendWarps * 32, 0, s, pool, k, v, slots, tokens, span) \
         : launch_early(kv_append_kernel<DD, false>, g, kAppendWarps * 32, 0, s, pool, k, v, slots, tokens, span)
    switch (pool.head_dim) {
        case 32: return EBX_KV_APPEND(32);
        case 64: return EBX_KV_APPEND(64);
        default: return EBX_KV_APPEND(128);
    }
#undef EBX_KV_APPEND
}

cudaError_t launch_kv_materialize(const KvPool& pool, const int32_t* tables, int width,
                                  const int32_t* starts, const int32_t* first, int requests,
                                  int64_t tokens, int dtype, void* k, void* v, cudaStream_t s) {
    if (tokens <= 0) return cudaSuccess;
    const int64_t grid = (tokens + kMatTokens - 1) / kMatTokens;
    if (grid > INT32_MAX) return cudaErrorInvalidValue;
    auto kern = dtype == kKvF32 ? kv_materialize_kernel<kKvF32>
                : dtype == kKvF16 ? kv_materialize_kernel<kKvF16> : kv_materialize_kernel<kKvBF16>;
    return launch_early(kern, dim3(unsigned(grid)), kMatThreads, 0, s, pool, tables, width, starts, first, requests, tokens, k, v);
}

}  // namespace ebx
