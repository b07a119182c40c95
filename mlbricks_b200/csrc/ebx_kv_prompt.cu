// ebx_kv_prompt.cu -- attention over the 8-bit paged cache for many rows (prompts, chunks): the
// formulas of ebx_kv_attention.cu on the 5th-generation tensor cores.
//
// A row tile is 256 rows (two of 128: the M of tcgen05.mma), a key tile 128 tokens.  One CTA per
// SM, 24 warps (two idle):
//   * warp 20 loads int8 key and value tiles (TMA, a box per block) and their scales;
//   * warps 16-19 turn codes into fp16 tiles [64 dimensions][128 rows of 128 bytes] with the
//     128-byte swizzle: exact integers, so the scales stay out of the products.  The same layout
//     is K-major for q . k (rows = N) and N-major for w . v (rows = K), so values need no transpose;
//   * warp 21 issues S = q k^T and O += w v.  The accumulators of both row tiles (S 2 x 128 columns,
//     O 2 x 128) fill the tensor memory; the weights overwrite S as the second product's A operand.
//     While it works on one row tile, the other's weights are computed;
//   * warps 0-7 and 8-15: two threads per row of each row tile, 64 keys of the tile each, in two
//     passes over S in tensor memory: the largest t; the weights and their sum.  O is rescaled (in
//     tensor memory) only when t grew by more than the lag.
// What bounds it: the chain S -> weights -> O of a row tile, of which the products of the other row
// tile cover only a part, and the issue slots when both compute weights.  A key tile takes some 5000
// clocks for both row tiles: the products 2500 of them (8 of 128 x 128 x 16 take 670 from shared
// memory, 600 with the weights in tensor memory), the largest and the weights 2700, the way from one
// to the other the rest.  4096 tokens behind 12000, 32 heads over 8 of 128: 1.10 ms, 850 TFLOP/s.
// Measured and not kept, for that case: one thread a row 1274 us; the row in registers (one read of
// S) 1299; S of 64 keys twice over, so that the weights never wait for it, 1277 (a product of 64
// columns takes as long as one of 128).
// Every mbarrier wait is bounded; a timeout sets the device status word, after which the row warps
// wait no more but still meet each other's barriers, and the other roles leave, the loader and the
// issuer once (bounded again) what they had sent for has come to its end.
#include <algorithm>
#include <atomic>
#include <climits>
#include <cmath>

#include "ebx_kv_work.cuh"

namespace ebx {
namespace {

constexpr int kPromptRows = 256;
constexpr int kPromptKeys = 128;
constexpr int kRowWarps = 16, kConvert = 16, kLoad = 20, kIssue = 21;  // first warps of the roles
constexpr int kPromptThreads = 24 * 32;
constexpr int kHalf = 128 * 128;   // bytes of 128 rows x 64 fp16
constexpr int kPromptExtra = 2;    // a row tile's begin and end, in key tiles
constexpr int kRaw = 4;            // int8 tiles in flight
constexpr int kBufs = 3;           // fp16 tiles: a value tile, the next key tile, and one being filled
constexpr int kTabs = 4;           // scale tables of key tiles
constexpr int kSCol = 0, kOCol = 256;  // tensor memory columns: S of both row tiles, O of both

template <int D>
struct PromptCfg {
    static constexpr int HALVES = (D + 63) / 64;
    static constexpr int kTile = HALVES * kHalf;      // an fp16 tile
    static constexpr int kRawTile = kPromptKeys * D;
    static constexpr int kBufOff = 2 * kTile;         // after the two q tiles
    static constexpr int kRawOff = kBufOff + kBufs * kTile;
    static constexpr int kTabOff = kRawOff + kRaw * kRawTile;
    static constexpr int kBytes = kTabOff + kTabs * 8 * 16 + kRaw * 16 * 4 + 256;
    static constexpr int kSmem = kBytes + 2 * 2 * 128 * 4;  // and what the two threads of a row tell each other
    static constexpr uint32_t kIdescS = (1u << 4) | (uint32_t(kPromptKeys >> 3) << 17) | (8u << 24);
    static constexpr uint32_t kIdescO = (1u << 4) | (1u << 16) | (uint32_t(D >> 3) << 17) | (8u << 24);
};

__device__ int g_kv_prompt_status = 0;
__device__ const float kv_prompt_none = kKvNone;

__device__ __forceinline__ bool pwait(const uint64_t* bar, int phase) {
    if (mbar_wait_bounded(smem_u32(bar), uint32_t(phase & 1))) return true;
    atomicExch(&g_kv_prompt_status, 0x7105);
    return false;
}

// 128-byte swizzled tile: rows of 128 bytes, 8-row groups 1024 bytes apart, 64-element blocks of
// the contiguous dimension kHalf apart (used when that dimension is N; K steps inside one block).
// An offset of b bytes is b / 16 more.
__device__ __forceinline__ uint64_t tile_desc(uint32_t saddr) {
    return uint64_t((saddr & 0x3FFFFu) >> 4) | uint64_t(kHalf >> 4) << 16 | uint64_t(1024 >> 4) << 32 |
           uint64_t(1) << 46 | uint64_t(2) << 61;
}
template <bool ACC>
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
                 "l"(a), "l"(b), "r"(idesc), "n"(ACC ? 1 : 0) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
                 "r"(a), "l"(b), "r"(idesc), "r"(acc) : "memory");
}
__device__ __forceinline__ bool elected() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ void commit(const uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n" ::"r"(smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ void after_sync() { asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void before_sync() { asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory"); }

// 16 columns of the thread's lane; valid after tmem_wait on the same registers.
template <int N>
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&v)[N], int at) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
        : "=r"(v[at]), "=r"(v[at + 1]), "=r"(v[at + 2]), "=r"(v[at + 3]), "=r"(v[at + 4]), "=r"(v[at + 5]),
          "=r"(v[at + 6]), "=r"(v[at + 7]), "=r"(v[at + 8]), "=r"(v[at + 9]), "=r"(v[at + 10]), "=r"(v[at + 11]),
          "=r"(v[at + 12]), "=r"(v[at + 13]), "=r"(v[at + 14]), "=r"(v[at + 15])
        : "r"(taddr) : "memory");
}
template <int COUNT, int N>
__device__ __forceinline__ void tmem_wait(uint32_t (&v)[N], int at = 0) {
    asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
#pragma unroll
    for (int i = at; i < at + COUNT; i += 8)  // no use of the registers moves above the wait
        asm volatile("" : "+r"(v[i]), "+r"(v[i + 1]), "+r"(v[i + 2]), "+r"(v[i + 3]), "+r"(v[i + 4]),
                     "+r"(v[i + 5]), "+r"(v[i + 6]), "+r"(v[i + 7]));
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};\n" ::"r"(v[0]),
        "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&v)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};\n" ::"r"(v[0]),
                 "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(taddr) : "memory");
}

// Two fp32 values in one register pair.
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ float lo2(uint64_t v) { return __uint_as_float(uint32_t(v)); }
__device__ __forceinline__ float hi2(uint64_t v) { return __uint_as_float(uint32_t(v >> 32)); }

// What a thread knows of its row.
struct Row {
    float unit;   // what q was divided by
    float mr;     // weights are 2^(t - mr); -infinity: nothing seen yet
    float l;
    int lo, hi;   // it sees keys [lo, hi)
};

// Bit i: the row sees key key0 + i.
__device__ __forceinline__ uint32_t seen32(const Row& row, int key0) {
    const int lo = min(max(row.lo - key0, 0), 32), hi = min(max(row.hi - key0, 0), 32);
    return hi > lo ? (0xffffffffu >> (32 - (hi - lo))) << lo : 0u;
}

// Walks 64 columns of the row's S, a unit of 16 tokens at a time, the next on its way: f(v, e, at,
// seen) with v the columns from `at` on, e = {ks * scale * log2 e, log2 vs, 1 / vs} of the unit, and
// with MASK the columns that the row sees of the tile, which begins at key0.
template <bool MASK, class F>
__device__ __forceinline__ void columns(uint32_t s, const float4* tab, const Row& row, int key0, F f) {
    uint32_t v[32];
    tmem_ld16(s, v, 0);
#pragma unroll 1
    for (int c = 0; c < 64; c += 32) {
        const uint32_t seen = MASK ? seen32(row, key0 + c) : 0u;
        const float4 e0 = tab[c / 16];  // ahead of the wait: both take their time
        tmem_wait<16>(v, 0);
        tmem_ld16(s + c + 16, v, 16);
        f(v, e0, c, seen);
        const float4 e1 = tab[c / 16 + 1];
        tmem_wait<16>(v, 16);
        if (c == 0) tmem_ld16(s + c + 32, v, 0);
        f(v + 16, e1, c + 16, seen >> 16);
    }
}

// t - mr of columns i and i + 1.
template <bool MASK>
__device__ __forceinline__ uint64_t t_pair(const uint32_t* v, int i, uint64_t c2, uint64_t b2, uint32_t seen) {
    const uint64_t t2 = fma2(uint64_t(v[i]) | uint64_t(v[i + 1]) << 32, c2, b2);
    if constexpr (!MASK) return t2;
    return pack2f(seen & (1u << i) ? lo2(t2) : -INFINITY, seen & (2u << i) ? hi2(t2) : -INFINITY);
}

// The largest t of the 64 columns.  t = c S + b grows with S (c >= 0: a negative scale is a negative
// q), and rounding keeps the order, so of a unit only the largest S is scaled.  A NaN c is not seen
// here but in the weights.
template <bool MASK>
__device__ __forceinline__ float largest(uint32_t s, const float4* tab, const Row& row, int key0) {
    float top = -INFINITY;
    columns<MASK>(s, tab, row, key0, [&](const uint32_t* v, const float4& e, int, uint32_t seen) {
        float most[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            float x[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                x[k] = __uint_as_float(v[i + k]);
                if constexpr (MASK) x[k] = seen & (1u << (i + k)) ? x[k] : -INFINITY;
            }
            most[0] = fmaxf(most[0], fmaxf(x[0], x[1]));
            most[1] = fmaxf(most[1], fmaxf(x[2], x[3]));
        }
        top = fmaxf(top, fmaf(fmaxf(most[0], most[1]), e.x * row.unit, e.y));
    });
    return top;
}

// Weights 2^(t - mr) as fp16 pairs over the columns of S that were read, and their sum over vs.
// (A quarter of the exponentials as polynomials on the FMA units made this loop slower, 1103 ->
// 1152 us for a chunk of 4096 tokens behind 12000: it is instructions that it lacks time for.)
template <bool MASK>
__device__ __forceinline__ float weigh(uint32_t s, const float4* tab, const Row& row, float mr, int key0) {
    float l = 0.0f;
    columns<MASK>(s, tab, row, key0, [&](const uint32_t* v, const float4& e, int at, uint32_t seen) {
        uint32_t p[8];
        const float c = e.x * row.unit, b = e.y - mr;
        const uint64_t c2 = pack2f(c, c), b2 = pack2f(b, b);
        uint64_t w2 = 0;
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
            const uint64_t t2 = t_pair<MASK>(v, i, c2, b2, seen);
            const float w0 = ex2(lo2(t2)), w1 = ex2(hi2(t2));
            w2 = add2(w2, pack2f(w0, w1));
            p[i / 2] = pack_half2(w0, w1);  // 11 bits, as the codes' operands need
        }
        l = fmaf(lo2(w2) + hi2(w2), e.z, l);
        tmem_st8(s + at / 2, p);
    });
    return l;
}

// Barriers of the two warps that share 32 rows.
__device__ __forceinline__ void pair_sync(int id) { asm volatile("bar.sync %0, 64;" ::"r"(id) : "memory"); }
__device__ __forceinline__ bool pair_any(int id, bool mine) {
    uint32_t any;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 q, %1, 0;\n\tbar.red.or.pred p, %2, 64, q;\n\t"
                 "selp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(any) : "r"(uint32_t(mine)), "r"(id) : "memory");
    return any != 0;
}

// The segment's key tiles [j0, j1), at least one, counted from its first, that rows of row tile x
// see: the rows of the other tile may begin earlier or end later.
template <bool SHARED>
using PromptWalk = KvWalk<kPromptRows, kPromptKeys, kPromptExtra, SHARED>;
template <bool SHARED>
__device__ __forceinline__ void tiles_seen(const KvAttnArgs& a, const PromptWalk<SHARED>& w, int x, int& j0, int& j1) {
    int t0, n;
    kv_key_tiles<128, kPromptKeys>(a, w.r, 2 * w.rt + x, t0, n);
    j0 = min(max(t0 - w.t0, 0), w.n - 1);
    j1 = max(min(t0 + n - w.t0, w.n), j0 + 1);
}

// A role gives up: what it sent for comes to its end (or a bounded wait does) before the CTA's memory is
// another's: the last copies of a loader that sent `sent`, the products of the issuer (`sent` -1).  One
// function out of line: inside the roles this moves the hot loops' code, and prompts of 64 wide heads took
// 137 us in place of 132, of 128 wide ones 149 in place of 144 (so they take 146).
__device__ __noinline__ void drain(const uint64_t* raw_full, const uint64_t* drained, int sent) {
    if (sent >= 0) {
        for (int i = max(sent - kRaw, 0); i < sent; ++i) pwait(raw_full + i % kRaw, i / kRaw);
    } else {
        if (elected()) commit(drained);
        __syncwarp();
        pwait(drained, 0);
    }
}

template <int D, bool BF16, bool SHARED>
__global__ void __launch_bounds__(kPromptThreads, 1)
    kv_prompt_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                     const __grid_constant__ KvAttnArgs a, int least) {
    using C = PromptCfg<D>;
    extern __shared__ __align__(1024) uint8_t smem[];
    float4* tabs = reinterpret_cast<float4*>(smem + C::kTabOff);             // [kTabs][8]
    float* raw_scales = reinterpret_cast<float*>(tabs + kTabs * 8);          // [kRaw][k, v][8]
    uint64_t* raw_full = reinterpret_cast<uint64_t*>(raw_scales + kRaw * 16);
    uint64_t* raw_empty = raw_full + kRaw;
    uint64_t* buf_full = raw_empty + kRaw;
    uint64_t* buf_empty = buf_full + kBufs;
    uint64_t* tab_full = buf_empty + kBufs;
    uint64_t* q_full = tab_full + kTabs;   // [2]: one for each row tile, as the next three
    uint64_t* s_full = q_full + 2;
    uint64_t* p_full = s_full + 2;
    uint64_t* o_done = p_full + 2;
    uint64_t* drained = o_done + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drained + 1);
    float* told = reinterpret_cast<float*>(smem + C::kBytes);               // [row tile][half][row]

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (warp == kLoad) {
        if (lane == 0) {
            for (int i = 0; i < kRaw; ++i) {
                mbar_init(smem_u32(raw_full + i), 1 + 32);  // the copies' bytes, and each lane's scales
                mbar_init(smem_u32(raw_empty + i), 4);
            }
            for (int i = 0; i < kBufs; ++i) {
                mbar_init(smem_u32(buf_full + i), 4);
                mbar_init(smem_u32(buf_empty + i), 1);
            }
            for (int i = 0; i < kTabs; ++i) mbar_init(smem_u32(tab_full + i), 1);
            for (int i = 0; i < 2; ++i) {
                mbar_init(smem_u32(q_full + i), 8);
                mbar_init(smem_u32(s_full + i), 1);
                mbar_init(smem_u32(p_full + i), 8);
                mbar_init(smem_u32(o_done + i), 1);
            }
            mbar_init(smem_u32(drained), 1);
            fence_proxy_async_smem();
        }
        __syncwarp();
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;\n" ::"r"(smem_u32(tmem_slot))
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");  // nothing of the call's inputs is read before
    if constexpr (SHARED) {
        if (int64_t(*a.largest) * a.group < a.least_rows) {  // the host does not know the groups
            before_sync();
            __syncthreads();
            if (warp == kLoad) {
                after_sync();
                asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;\n" ::"r"(*tmem_slot) : "memory");
            }
            return;
        }
    }
    const KvShare share = kv_share<kPromptRows, kPromptKeys, kPromptExtra, kPromptThreads, SHARED>(a, least, reinterpret_cast<int*>(smem));
    fence_proxy_async_smem();  // copies will overwrite what kv_share kept there
    if (!SHARED && threadIdx.x == 0) a.desc[blockIdx.x] = make_int4(0, 0, 0, 0);
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the join waits for this grid's end
    before_sync();
    __syncthreads();
    after_sync();
    const uint32_t tmem = *tmem_slot;
    PromptWalk<SHARED> walk;
    walk.start(a, share);

    if (warp < kRowWarps) {
        // ---------------- two threads per row ----------------
        const int x = warp >> 3;                               // row tile
        const int half = (warp >> 2) & 1;                      // 64 of the 128 keys, half of O's columns
        const int quarter = warp & 3;                          // the warp's 32 lanes of tensor memory
        const int pair = 1 + x * 4 + quarter;                  // barrier of the two warps that share them
        const uint32_t lane_base = uint32_t(quarter * 32) << 16;
        const uint32_t s_addr = tmem + lane_base + kSCol + x * 128 + half * 64;
        const uint32_t o_addr = tmem + lane_base + kOCol + x * 128 + half * (D / 2);
        float* tell = told + (x * 2 + half) * 128 + quarter * 32 + lane;
        const float* other = told + (x * 2 + (half ^ 1)) * 128 + quarter * 32 + lane;
        // q and the output pass through shared memory, PER lanes to a row of 16-byte chunks
        constexpr int PER = D / 8, ROWS = 32 / PER;
        uint8_t* staged = smem + x * C::kTile + quarter * 32 * 128;
        const int mine = lane / PER, chunk = lane % PER;
        auto stage_at = [&](int i) {  // this lane's 16 bytes of the warps' row i
            return reinterpret_cast<uint4*>(staged + (chunk / 8) * kHalf + i * 128 + (((chunk & 7) ^ (i & 7)) << 4));
        };
        int g = 0;   // key tiles of this row tile so far
        int gj = 0;  // key tiles of the CTA so far
        bool ok = true;
        auto wait = [&](const uint64_t* bar, int phase) {
            if (ok) ok = __all_sync(0xffffffffu, pwait(bar, phase));
            after_sync();
        };
        for (; !walk.done(); walk.next(a)) {
            if (x == 1 && walk.r.rows - walk.rt * kPromptRows <= 128) {
                gj += walk.n;
                continue;
            }
            const int row0 = walk.rt * kPromptRows + x * 128 + quarter * 32;  // the warps' first row
            // this lane's row; past the last one: the last, whose result is not kept
            const bool live = row0 + lane < walk.r.rows;
            const int token = by_group(a, min(row0 + lane, walk.r.rows - 1));
            const int head = walk.head * a.group + min(row0 + lane, walk.r.rows - 1) - token * a.group;
            Row row;
            row.unit = 1.0f;
            row.mr = -INFINITY;
            row.l = 0.0f;
            const int place = walk.r.begin + token;
            auto q_token = [&] { return kv_token<SHARED>(a, walk.request, walk.r, token); };
            row.hi = !live ? INT_MAX : a.causal ? min(place + 1, walk.r.length) : walk.r.length;
            row.lo = !live ? 0 : max(walk.r.first, a.window > 0 ? place - a.window + 1 : 0);
            {
                const int64_t off = q_token() * a.q.token_stride + head * a.q.head_stride;
                uint4 v[PER / 2];  // each of the two warps brings every other load's rows
#pragma unroll
                for (int i = 0; i < PER / 2; ++i)
                    v[i] = __ldg(reinterpret_cast<const uint4*>(
                                     a.q.p + __shfl_sync(0xffffffffu, off, (2 * i + half) * ROWS + mine)) + chunk);
#pragma unroll
                for (int i = 0; i < PER / 2; ++i) {
                    const int ri = (2 * i + half) * ROWS + mine;
                    if constexpr (BF16) {
                        // over the power of two at the row's largest element, as in ebx_kv_attention.cu
                        const uint32_t m = 0x7fff7fffu;
                        uint32_t top = __vmaxu2(__vmaxu2(v[i].x & m, v[i].y & m), __vmaxu2(v[i].z & m, v[i].w & m));
                        top = max(top & 0xffffu, top >> 16);
#pragma unroll
                        for (int d = 1; d < PER; d <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
                        const uint32_t e = min(max(top >> 7, 1u), 253u);
                        const float down = __uint_as_float((254u - e) << 23);
                        if (chunk == 0) told[x * 256 + quarter * 32 + ri] = __uint_as_float(e << 23);
                        auto halves = [&](uint32_t b) {
                            return pack_half2(__uint_as_float(b << 16) * down, __uint_as_float(b & 0xffff0000u) * down);
                        };
                        v[i] = make_uint4(halves(v[i].x), halves(v[i].y), halves(v[i].z), halves(v[i].w));
                    }
                    const uint32_t sign = a.scale_log2 < 0.0f ? 0x80008000u : 0u;
                    *stage_at(ri) = make_uint4(v[i].x ^ sign, v[i].y ^ sign, v[i].z ^ sign, v[i].w ^ sign);
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(q_full + x));
                if constexpr (BF16) {
                    pair_sync(pair);
                    row.unit = told[x * 256 + quarter * 32 + lane];
                    pair_sync(pair);
                }
            }
            // keys that every row of the warp sees
            const int all_lo = __reduce_max_sync(0xffffffffu, row.lo), all_hi = __reduce_min_sync(0xffffffffu, row.hi);
            int j0, j1;
            tiles_seen<SHARED>(a, walk, x, j0, j1);
            for (int j = j0; j < j1; ++j, ++g) {
                const int at = gj + j;
                wait(s_full + x, g);
                wait(tab_full + at % kTabs, at / kTabs);
                const float4* tab = tabs + (at % kTabs) * 8 + half * 4;
                const int key0 = (walk.t0 + j) * kPromptKeys + half * 64;
                const bool mask = key0 < all_lo || key0 + 64 > all_hi;
                float top = mask ? largest<true>(s_addr, tab, row, key0) : largest<false>(s_addr, tab, row, key0);
                if (pair_any(pair, top > row.mr + (kLag + kShift))) {
                    // mr moves in the rows whose t grew, and with it what was summed
                    *tell = top;
                    pair_sync(pair);
                    top = fmaxf(top, *other);
                    const bool up = top > row.mr + (kLag + kShift);
                    const float next = up ? top - kShift : row.mr;
                    const float f = up ? ex2(row.mr - next) : 1.0f;
                    row.mr = next;
                    row.l *= f;
                    if (j > j0) {
                        wait(o_done + x, g - 1);
#pragma unroll 1
                        for (int c = 0; c < D / 2; c += 16) {
                            uint32_t v[16];
                            tmem_ld16(o_addr + c, v, 0);
                            tmem_wait<16>(v);
#pragma unroll
                            for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * f);
                            tmem_st16(o_addr + c, v);
                        }
                    }
                    pair_sync(pair);  // `told` is free again
                }
                const float now = row.mr == -INFINITY ? 0.0f : row.mr;
                row.l += mask ? weigh<true>(s_addr, tab, row, now, key0) : weigh<false>(s_addr, tab, row, now, key0);
                asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory");
                before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(p_full + x));
            }
            gj += walk.n;
            // the sums of both halves, and O
            *tell = row.l;
            pair_sync(pair);
            const float l = half ? *other + row.l : row.l + *other;
            wait(o_done + x, g - 1);
            const bool whole = walk.whole();
            const int64_t at_row = int64_t(q_token()) * a.heads + head;
            const int slot = walk.begins ? 1 : 0;
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            float4* part = whole ? nullptr
                                 : reinterpret_cast<float4*>(kv_part<D, kPromptRows>(a, blockIdx.x, slot)) + x * 128 + quarter * 32 + lane;
#pragma unroll 1
            for (int c = 0; c < D / 2; c += 16) {
                uint32_t v[16];
                tmem_ld16(o_addr + c, v, 0);
                tmem_wait<16>(v);
                const int d0 = half * (D / 2) + c;
                if (SHARED && whole) {
                    if (live) {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            *reinterpret_cast<float4*>(a.sums + at_row * D + d0 + 4 * i) =
                                make_float4(__uint_as_float(v[4 * i]), __uint_as_float(v[4 * i + 1]),
                                            __uint_as_float(v[4 * i + 2]), __uint_as_float(v[4 * i + 3]));
                    }
                } else if (whole) {  // through shared memory, so that rows are written whole
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        uint32_t h[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            h[k] = pack16<BF16>(__uint_as_float(v[8 * i + 2 * k]) * inv, __uint_as_float(v[8 * i + 2 * k + 1]) * inv);
                        const int q = d0 / 8 + i;
                        *reinterpret_cast<uint4*>(staged + (q / 8) * kHalf + lane * 128 + (((q & 7) ^ (lane & 7)) << 4)) =
                            make_uint4(h[0], h[1], h[2], h[3]);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        part[(d0 / 4 + i) * kPromptRows] =
                            make_float4(__uint_as_float(v[4 * i]), __uint_as_float(v[4 * i + 1]),
                                        __uint_as_float(v[4 * i + 2]), __uint_as_float(v[4 * i + 3]));
                }
            }
            before_sync();
            pair_sync(pair);
            if (!SHARED && whole) {
#pragma unroll
                for (int i = 0; i < PER / 2; ++i) {
                    const int ri = (2 * i + half) * ROWS + mine;
                    const int64_t to = __shfl_sync(0xffffffffu, at_row, ri);
                    if (row0 + ri < walk.r.rows) *(reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + to * D) + chunk) = *stage_at(ri);
                }
                pair_sync(pair);  // the staged rows are free again
            }
            if constexpr (SHARED) {  // groups only: side 0
                if (half == 0 && live) {
                    if (whole) {
                        a.sums_ml[at_row] = make_float2(row.mr, l);
                        kv_whole(a, 0, at_row);
                    } else if (walk.begins) {
                        kv_begins(a, 0, at_row, true, walk.last() - int(blockIdx.x), x * 128 + quarter * 32 + lane);
                    }
                }
            }
            if (!SHARED && half == 0 && live && whole && a.lse)
                a.lse[at_row] = l == 0.0f ? -INFINITY : (row.mr + lg2(l)) * 0.6931471805599453f;
            if (half == 0 && !whole)
                kv_part_ml<D, kPromptRows>(a, blockIdx.x, slot)[x * 128 + quarter * 32 + lane] = make_float2(row.mr, l);
            if (!SHARED && walk.begins && !whole && threadIdx.x == 0)
                a.desc[blockIdx.x] = kv_desc(walk.r, walk.rt, kPromptRows, walk.head, walk.last() - int(blockIdx.x));
        }
    } else if (warp >= kLoad) {
        if (warp == kLoad) {
            // ---------------- loader ----------------
            const int bsize = a.pool.block_size, none = a.pool.blocks;
            const int64_t past_pool = int64_t(none) * a.pool.kv_heads * bsize;  // TMA fills with zeros
            const int boxes = kPromptKeys / bsize;  // at most 8
            int it = 0;
            bool ok = true;
            for (; !walk.done() && ok; walk.next(a)) {
                const int32_t* row = a.tables + int64_t(kv_table_row<SHARED>(a, walk.request)) * a.width;
                auto block_of = [&](int token) {
                    const int column = token >> a.pool.shift;
                    if (token >= walk.r.length || column >= a.width) return none;
                    const int id = __ldg(row + column);
                    return id < 0 || id > none ? none : id;
                };
                const int box_row = (lane & 7) * bsize, unit_row = (lane & 7) * 16;
                int id_next = lane < boxes ? block_of(walk.t0 * kPromptKeys + box_row) : none;
                int sid_next = block_of(walk.t0 * kPromptKeys + unit_row);
                for (int j = 0; j < walk.n && ok; ++j) {
                    const int key0 = (walk.t0 + j) * kPromptKeys;
                    const int id = id_next, sid = sid_next;
                    if (j + 1 < walk.n) {
                        if (lane < boxes) id_next = block_of(key0 + kPromptKeys + box_row);
                        sid_next = block_of(key0 + kPromptKeys + unit_row);
                    }
                    for (int side = 0; side < 2; ++side, ++it) {
                        const int st = it % kRaw;
                        const bool free = it < kRaw || pwait(raw_empty + st, it / kRaw - 1);
                        if (!__all_sync(0xffffffffu, free)) {
                            ok = false;
                            break;
                        }
                        const uint32_t bar = smem_u32(raw_full + st);
                        if (lane == 0) mbar_expect_tx(bar, C::kRawTile);
                        __syncwarp();
                        if (lane < boxes)
                            kv_tma_2d(smem_u32(smem + C::kRawOff + st * C::kRawTile + box_row * D), side ? &map_v : &map_k, 0,
                                      int(id == none ? past_pool : (int64_t(id) * a.pool.kv_heads + walk.head) * bsize), bar);
                        if (side == 0 && lane < 16) {  // both sides' scales travel with the keys
                            const int64_t cell = int64_t(sid) * a.pool.kv_heads + walk.head;
                            cp_async4(smem_u32(raw_scales + st * 16 + lane),
                                      sid == none ? &kv_prompt_none : (lane < 8 ? a.pool.k_scales : a.pool.v_scales) + cell);
                        }
                        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];\n" ::"r"(bar) : "memory");
                    }
                }
            }
            asm volatile("cp.async.wait_all;\n" ::: "memory");
            if (!ok) drain(raw_full, drained, it);
        } else if (warp == kIssue) {
            // ---------------- products: the warp together, one elected lane issues ----------------
            const uint64_t q0 = tile_desc(smem_u32(smem)), buf0 = tile_desc(smem_u32(smem + C::kBufOff));
            int it = 0;            // fp16 tiles used: key and value tiles in turn
            int seg = 0, segb = 0; // segments of either row tile
            int g[2] = {0, 0};     // key tiles of either row tile
            bool ok = true;
            auto scores = [&](int x, int buf) {
                const uint64_t q = q0 + uint32_t(x * (C::kTile >> 4)), k = buf0 + uint32_t(buf * (C::kTile >> 4));
                const uint32_t d = tmem + kSCol + x * 128;
                if (elected()) {
                    mma_ss<false>(d, q, k, C::kIdescS);
#pragma unroll
                    for (int i = 1; i < D / 16; ++i) {
                        constexpr uint32_t kBlock = kHalf >> 4;
                        mma_ss<true>(d, q + (i / 4) * kBlock + (i % 4) * 2, k + (i / 4) * kBlock + (i % 4) * 2, C::kIdescS);
                    }
                    commit(s_full + x);
                }
                __syncwarp();
            };
            auto values = [&](int x, int buf, bool first) {
                const uint64_t v = buf0 + uint32_t(buf * (C::kTile >> 4));
                const uint32_t d = tmem + kOCol + x * 128, w = tmem + kSCol + x * 128;
                if (elected()) {
#pragma unroll
                    for (int i = 0; i < kPromptKeys / 16; ++i)
                        mma_ts(d, w + (i / 4) * 64 + (i % 4) * 8, v + i * (2048 >> 4), C::kIdescO, i == 0 ? !first : 1);
                    commit(o_done + x);
                }
                __syncwarp();
            };
            auto release = [&](int buf) {
                if (elected()) commit(buf_empty + buf);
                __syncwarp();
            };
            auto wait = [&](const uint64_t* bar, int phase) {
                const bool got = __all_sync(0xffffffffu, pwait(bar, phase));
                after_sync();
                return got;
            };
            for (; !walk.done() && ok; walk.next(a)) {
                const bool two = walk.r.rows - walk.rt * kPromptRows > 128;
                int from[2], to[2];  // the segment's key tiles that either row tile sees
                tiles_seen<SHARED>(a, walk, 0, from[0], to[0]);
                tiles_seen<SHARED>(a, walk, 1, from[1], to[1]);
                if (!two) from[1] = to[1] = 0;
                // S of every row tile that begins at key tile j (counted from the segment's first)
                auto step = [&](int x, int j, int buf, int phase) {
                    if (j < from[x] || j >= to[x]) return true;
                    if (!wait(buf_full + buf, phase)) return false;
                    if (j == from[x] && !(x == 0 ? wait(q_full, seg++) : wait(q_full + 1, segb++))) return false;
                    scores(x, buf);
                    return true;
                };
                // every buffer is waited for, used or not, so that its phases are never overrun
                ok = wait(buf_full + it % kBufs, it / kBufs) && step(0, 0, it % kBufs, it / kBufs) && step(1, 0, it % kBufs, it / kBufs);
                if (!ok) break;
                release(it % kBufs);
                ++it;
                for (int j = 0; j < walk.n; ++j) {
                    const int vb = it % kBufs, kb = (it + 1) % kBufs;
                    const bool more = j + 1 < walk.n;
                    if (!(ok = wait(buf_full + vb, it / kBufs))) break;
                    for (int x = 0; x < 2 && ok; ++x) {
                        if (j >= from[x] && j < to[x]) {
                            if (!(ok = wait(p_full + x, g[x]))) break;
                            ++g[x];
                            values(x, vb, j == from[x]);
                        }
                        // after the product above, which reads the same columns
                        if (more) ok = step(x, j + 1, kb, (it + 1) / kBufs);
                    }
                    if (!ok) break;
                    release(vb);
                    if (more) {
                        if (!(ok = wait(buf_full + kb, (it + 1) / kBufs))) break;
                        release(kb);
                    }
                    it += more ? 2 : 1;
                }
            }
            if (!ok) drain(raw_full, drained, -1);
        }
    } else {
        // ---------------- codes to fp16 ----------------
        const int w = warp - kConvert;
        int it = 0, gj = 0;
        bool ok = true;
        for (; !walk.done() && ok; walk.next(a)) {
            for (int j = 0; j < walk.n && ok; ++j, ++gj) {
                for (int side = 0; side < 2; ++side, ++it) {
                    const int st = it % kRaw, buf = it % kBufs;
                    ok = pwait(raw_full + st, it / kRaw) && (it < kBufs || pwait(buf_empty + buf, it / kBufs - 1));
                    if (!__all_sync(0xffffffffu, ok)) {
                        ok = false;
                        break;
                    }
                    if (side == 0 && w == 0) {
                        if (lane < 8) {
                            const float ks = raw_scales[st * 16 + lane], vs = raw_scales[st * 16 + 8 + lane];
                            const bool none = vs < 0.0f;                        // kKvNone
                            const float vsc = vs < 0x1p-100f ? 0x1p-100f : vs;  // NaN stays
                            // NaN goes through t, where the mask stops it, and not through 1 / vs
                            tabs[(gj % kTabs) * 8 + lane] =
                                make_float4(none ? 0.0f : ks * fabsf(a.scale_log2), none ? -INFINITY : lg2(vsc),
                                            none ? 0.0f : vs == vs ? 1.0f / vsc : 1.0f, 0.0f);
                        }
                        __syncwarp();
                        if (lane == 0) mbar_arrive(smem_u32(tab_full + gj % kTabs));
                    }
                    const uint8_t* raw = smem + C::kRawOff + st * C::kRawTile;
                    uint8_t* out = smem + C::kBufOff + buf * C::kTile;
                    constexpr int CH = D / 16 < 4 ? D / 16 : 4;  // 16-byte chunks of a row that neighbouring lanes read
                    constexpr int STEP = 32 / CH;                // rows of a warp's load
#pragma unroll 2
                    for (int g = 0; g < 32 / STEP; ++g)
#pragma unroll
                        for (int h = 0; h < C::HALVES; ++h) {
                            // rows in an order that keeps both the swizzled loads and stores free of conflicts
                            const int r8 = CH == 4 ? (lane >> 3) ^ ((lane & 4) ? 5 : 0)
                                                   : ((lane >> 1) & 1) | ((lane >> 2) & 1) << 2 | ((lane >> 3) & 1) << 1 | ((lane >> 4) << 3);
                            const int r = w * 32 + g * STEP + r8;
                            const int c = (lane % CH) + 4 * h;
                            const int x = D == 128 ? (r & 7) : D == 64 ? ((r >> 1) & 3) : ((r >> 2) & 1);
                            const uint4 v = *reinterpret_cast<const uint4*>(raw + r * D + ((c ^ x) << 4));
                            const uint32_t in[4] = {v.x ^ 0x80808080u, v.y ^ 0x80808080u, v.z ^ 0x80808080u, v.w ^ 0x80808080u};
                            uint32_t o[8];
#pragma unroll
                            for (int q = 0; q < 4; ++q) {
                                o[2 * q] = codes_to_half2(in[q], 0x4140);
                                o[2 * q + 1] = codes_to_half2(in[q], 0x4342);
                            }
                            uint8_t* dst = out + h * kHalf + r * 128;
                            const int q0 = 2 * (c & 3);
                            *reinterpret_cast<uint4*>(dst + ((q0 ^ (r & 7)) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
                            *reinterpret_cast<uint4*>(dst + (((q0 + 1) ^ (r & 7)) << 4)) = make_uint4(o[4], o[5], o[6], o[7]);
                        }
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        mbar_arrive(smem_u32(buf_full + buf));
                        mbar_arrive(smem_u32(raw_empty + st));
                    }
                }
            }
        }
    }

    before_sync();
    __syncthreads();
    if (warp == kLoad) {
        after_sync();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;\n" ::"r"(tmem) : "memory");
    }
}

// Units a CTA takes at least.  It decides for short prompts only; there fewer are faster, down to the begin
// and end alone (2 / 4 / 8 / 16 units, 32 heads over 8 of 128, captured: a prompt of 200 tokens 29 / 32 / 42 / 59 us,
// of 700 35 / 35 / 44 / 64, of 1500 60 / 60 / 60 / 66, three of 2048 184 with any).
constexpr int kPromptLeast = 8;
// Groups: 64 requests behind 8192 tokens, with the rest, 58 / 58 / 67 us for 1 / 2 / 8, 16 behind 2000 32 / 33 / 46.
constexpr int kSharedLeast = 2;

// SHARED: `ws` holds the parts, and the caller joins.
template <int D, bool BF16, bool SHARED = false>
cudaError_t launch_prompt(KvAttnArgs a, void* ws, int dev, cudaStream_t s) {
    using C = PromptCfg<D>;
    static_assert(C::kSmem <= 227 * 1024, "shared memory of the prompt kernel");
    auto kern = kv_prompt_kernel<D, BF16, SHARED>;
    static std::atomic<uint64_t> configured{0};
    const uint64_t bit = 1ull << (dev & 63);
    if (!(configured.load(std::memory_order_relaxed) & bit)) {
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
        if (e != cudaSuccess) return e;
        configured.fetch_or(bit);
    }
    CUtensorMap mk, mv;
    if (!code_map(&mk, a.pool.k_codes, a.pool, a.pool.block_size) || !code_map(&mv, a.pool.v_codes, a.pool, a.pool.block_size))
        return cudaErrorInvalidValue;
    const int grid = gemm_sm_count(dev);
    a.desc = static_cast<int4*>(ws);
    a.part = reinterpret_cast<float*>(SHARED ? a.desc : a.desc + grid);
    const cudaError_t e = launch_early(kern, dim3(grid), kPromptThreads, C::kSmem, s, mk, mv, a, SHARED ? kSharedLeast : kPromptLeast);
    if (e != cudaSuccess || SHARED) return e;
    return launch_join<D, kPromptRows, 4, BF16>(a, grid, kPromptRows, s);
}

}  // namespace

uint64_t kv_prompt_workspace_bytes(int head_dim, int sms) {
    return uint64_t(round_up(int64_t(sms) * int64_t(sizeof(int4) + 2 * kPromptRows * (head_dim + 2) * sizeof(float)), 256));
}

cudaError_t launch_kv_prompt(const KvAttnArgs& a, bool bf16, void* ws, int dev, cudaStream_t s) {
    switch (a.pool.head_dim) {
        case 32: return bf16 ? launch_prompt<32, true>(a, ws, dev, s) : launch_prompt<32, false>(a, ws, dev, s);
        case 64: return bf16 ? launch_prompt<64, true>(a, ws, dev, s) : launch_prompt<64, false>(a, ws, dev, s);
        default: return bf16 ? launch_prompt<128, true>(a, ws, dev, s) : launch_prompt<128, false>(a, ws, dev, s);
    }
}

cudaError_t launch_kv_prompt_shared(const KvAttnArgs& a, bool bf16, void* ws, int dev, cudaStream_t s) {
    switch (a.pool.head_dim) {
        case 32: return bf16 ? launch_prompt<32, true, true>(a, ws, dev, s) : launch_prompt<32, false, true>(a, ws, dev, s);
        case 64: return bf16 ? launch_prompt<64, true, true>(a, ws, dev, s) : launch_prompt<64, false, true>(a, ws, dev, s);
        default: return bf16 ? launch_prompt<128, true, true>(a, ws, dev, s) : launch_prompt<128, false, true>(a, ws, dev, s);
    }
}

cudaError_t read_kv_prompt_status(int* status, bool clear, cudaStream_t s) {
    return read_status_word(g_kv_prompt_status, status, clear, s);
}

}  // namespace ebx
