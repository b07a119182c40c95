// ebx_kv_prompt.cu -- attention over the 8-bit paged cache for many rows (prompts, chunks): the
// formulas of ebx_kv_attention.cu on the 5th-generation tensor cores.
//
// A row tile is 256 rows (two of 128: the M of tcgen05.mma), a key tile 128 tokens.  One CTA per
// SM, 14 warps:
//   * warp 12 loads int8 key and value tiles (TMA, a box per block) and their scales;
//   * warps 8-11 turn codes into fp16 tiles [64 dimensions][128 rows of 128 bytes] with the
//     128-byte swizzle: exact integers, so the scales stay out of the products.  The same layout
//     is K-major for q . k (rows = N) and N-major for w . v (rows = K), so values need no transpose;
//   * one thread of warp 13 issues S = q k^T and O += w v.  The accumulators of both row tiles
//     (S 2 x 128 columns, O 2 x 128) fill the tensor memory; the weights overwrite S as the second
//     product's A operand.  While it works on one row tile, the other's weights are computed;
//   * warps 0-3 and 4-7: a thread per row of each row tile.  One pass over S: t, its maximum, the
//     weights and their sum.  Only if t grew by more than the lag is the pass done again and O
//     rescaled, so O stays in tensor memory for nearly all of the row's life.
// Every mbarrier wait is bounded; a timeout sets the device status word and the roles leave.
#include <algorithm>
#include <atomic>
#include <climits>
#include <cmath>

#include "ebx_kv_work.cuh"

namespace ebx {
namespace {

constexpr int kPromptRows = 256;
constexpr int kPromptKeys = 128;
constexpr int kPromptThreads = 14 * 32;
constexpr int kHalf = 128 * 128;   // bytes of 128 rows x 64 fp16
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
    static constexpr int kSmem = kBytes + 1024;
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
__device__ __forceinline__ uint64_t tile_desc(uint32_t saddr) {
    return uint64_t((saddr & 0x3FFFFu) >> 4) | uint64_t(kHalf >> 4) << 16 | uint64_t(1024 >> 4) << 32 |
           uint64_t(1) << 46 | uint64_t(2) << 61;
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool acc) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
                 "l"(a), "l"(b), "r"(idesc), "r"(uint32_t(acc)) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool acc) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
                 "r"(a), "l"(b), "r"(idesc), "r"(uint32_t(acc)) : "memory");
}
__device__ __forceinline__ void commit(const uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n" ::"r"(smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ void after_sync() { asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void before_sync() { asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory"); }

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
        "tcgen05.wait::ld.sync.aligned;\n"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
          "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
          "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]),
          "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(taddr) : "memory");
}
template <int AT, int N>
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&v)[N]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};\n" ::"r"(v[AT + 0]),
        "r"(v[AT + 1]), "r"(v[AT + 2]), "r"(v[AT + 3]), "r"(v[AT + 4]), "r"(v[AT + 5]), "r"(v[AT + 6]),
        "r"(v[AT + 7]), "r"(v[AT + 8]), "r"(v[AT + 9]), "r"(v[AT + 10]), "r"(v[AT + 11]), "r"(v[AT + 12]),
        "r"(v[AT + 13]), "r"(v[AT + 14]), "r"(v[AT + 15]), "r"(v[AT + 16]), "r"(v[AT + 17]), "r"(v[AT + 18]),
        "r"(v[AT + 19]), "r"(v[AT + 20]), "r"(v[AT + 21]), "r"(v[AT + 22]), "r"(v[AT + 23]), "r"(v[AT + 24]),
        "r"(v[AT + 25]), "r"(v[AT + 26]), "r"(v[AT + 27]), "r"(v[AT + 28]), "r"(v[AT + 29]), "r"(v[AT + 30]),
        "r"(v[AT + 31]), "r"(taddr) : "memory");
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

// One pass over a row of S: weights 2^(t - mr) as fp16 pairs, their sum over vs, and the largest
// t - mr.  tab[u] = {ks * scale * log2 e, log2 vs, 1 / vs} of 16 tokens.  MASK: the row may not
// see all of the tile, which begins at key0.
template <bool MASK>
__device__ __forceinline__ void weigh(uint32_t s, const float4* tab, const Row& row, float mr, int key0,
                                      uint32_t (&p)[64], float& sum, float& top) {
    top = -INFINITY;
    sum = 0.0f;
    const uint32_t from = uint32_t(row.lo - key0), width = row.hi > row.lo ? uint32_t(row.hi - row.lo) : 0u;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        uint32_t v[32];
        tmem_ld32(s + c * 32, v);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const float4 e = tab[2 * c + u];
            const float cf = e.x * row.unit, b = e.y - mr;
            const uint64_t cf2 = pack2f(cf, cf), b2 = pack2f(b, b);
            uint64_t w2 = 0;
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
                const uint64_t t2 = fma2(uint64_t(v[16 * u + i]) | uint64_t(v[16 * u + i + 1]) << 32, cf2, b2);
                float t0 = lo2(t2), t1 = hi2(t2);
                if constexpr (MASK) {
                    const uint32_t k = uint32_t(32 * c + 16 * u + i);
                    if (k - from >= width) t0 = -INFINITY;
                    if (k + 1 - from >= width) t1 = -INFINITY;
                }
                top = fmaxf(top, fmaxf(t0, t1));
                const float w0 = ex2(t0), w1 = ex2(t1);
                w2 = add2(w2, pack2f(w0, w1));
                p[16 * c + 8 * u + i / 2] = pack_half2(w0, w1);  // 11 bits, as the codes' operands need
            }
            sum = fmaf(lo2(w2) + hi2(w2), e.z, sum);
        }
    }
}

// The largest t of a row of S.
__device__ __forceinline__ float largest(uint32_t s, const float4* tab, const Row& row, int key0) {
    float top = -INFINITY;
    const uint32_t from = uint32_t(row.lo - key0), width = row.hi > row.lo ? uint32_t(row.hi - row.lo) : 0u;
#pragma unroll 1
    for (int c = 0; c < 4; ++c) {
        uint32_t v[32];
        tmem_ld32(s + c * 32, v);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const float4 e = tab[2 * c + u];
            const float cf = e.x * row.unit;
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (uint32_t(32 * c + 16 * u + i) - from < width)
                    top = fmaxf(top, fmaf(__uint_as_float(v[16 * u + i]), cf, e.y));
        }
    }
    return top;
}

template <int D, bool BF16>
__global__ void __launch_bounds__(kPromptThreads, 1)
    kv_prompt_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                     const __grid_constant__ KvAttnArgs a, int least) {
    using C = PromptCfg<D>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
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
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_done + 2);
    __shared__ int64_t scratch[kPromptThreads / 32 + 2];

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (warp == 12) {
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
                mbar_init(smem_u32(q_full + i), 4);
                mbar_init(smem_u32(s_full + i), 1);
                mbar_init(smem_u32(p_full + i), 4);
                mbar_init(smem_u32(o_done + i), 1);
            }
            fence_proxy_async_smem();
        }
        __syncwarp();
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;\n" ::"r"(smem_u32(tmem_slot))
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }
    int request;
    int64_t at, units;
    kv_share<kPromptRows, kPromptKeys, kPromptThreads>(a, least, scratch, request, at, units);
    if (threadIdx.x < 2) a.desc[2 * blockIdx.x + threadIdx.x] = make_int4(0, 0, 0, 0);
    before_sync();
    __syncthreads();
    after_sync();
    const uint32_t tmem = *tmem_slot;
    KvWalk<kPromptRows, kPromptKeys> walk;
    walk.start(a, request, at, units);

    if (warp == 12) {
        // ---------------- loader ----------------
        const int bsize = a.pool.block_size, none = a.pool.blocks;
        const int64_t past_pool = int64_t(none) * a.pool.kv_heads * bsize;  // TMA fills with zeros
        const int boxes = kPromptKeys / bsize;  // at most 8
        int it = 0;
        bool ok = true;
        for (; !walk.done() && ok; walk.next(a)) {
            const int32_t* row = a.tables + int64_t(walk.request) * a.width;
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
    } else if (warp == 13) {
        // ---------------- products ----------------
        if (lane == 0) {
            const uint32_t q0 = smem_u32(smem), bufs = smem_u32(smem + C::kBufOff);
            int it = 0;            // fp16 tiles used: key and value tiles in turn
            int seg = 0, segb = 0; // segments of either row tile
            int g[2] = {0, 0};     // key tiles of either row tile
            bool ok = true;
            auto scores = [&](int x, int buf) {
                const uint32_t q = q0 + x * C::kTile, k = bufs + buf * C::kTile;
#pragma unroll
                for (int i = 0; i < D / 16; ++i) {
                    const uint32_t off = (i / 4) * kHalf + (i % 4) * 32;
                    mma_ss(tmem + kSCol + x * 128, tile_desc(q + off), tile_desc(k + off), C::kIdescS, i != 0);
                }
                commit(s_full + x);
            };
            auto values = [&](int x, int buf, bool first) {
                const uint32_t v = bufs + buf * C::kTile;
#pragma unroll
                for (int i = 0; i < kPromptKeys / 16; ++i)
                    mma_ts(tmem + kOCol + x * 128, tmem + kSCol + x * 128 + i * 8, tile_desc(v + i * 2048), C::kIdescO,
                           !first || i != 0);
                commit(o_done + x);
            };
            for (; !walk.done() && ok; walk.next(a)) {
                const bool two = walk.r.rows - walk.rt * kPromptRows > 128;
                ok = pwait(buf_full + it % kBufs, it / kBufs) && pwait(q_full, seg);
                ++seg;
                if (!ok) break;
                after_sync();
                scores(0, it % kBufs);
                if (two) {
                    if (!(ok = pwait(q_full + 1, segb))) break;
                    ++segb;
                    after_sync();
                    scores(1, it % kBufs);
                }
                commit(buf_empty + it % kBufs);
                ++it;
                for (int j = 0; j < walk.n; ++j) {
                    const int vb = it % kBufs, kb = (it + 1) % kBufs;
                    const bool more = j + 1 < walk.n;
                    if (!(ok = pwait(buf_full + vb, it / kBufs) && pwait(p_full, g[0]))) break;
                    ++g[0];
                    after_sync();
                    values(0, vb, j == 0);
                    if (more) {
                        if (!(ok = pwait(buf_full + kb, (it + 1) / kBufs))) break;
                        after_sync();
                        scores(0, kb);  // after the product above, which reads the same columns
                    }
                    if (two) {
                        if (!(ok = pwait(p_full + 1, g[1]))) break;
                        ++g[1];
                        after_sync();
                        values(1, vb, j == 0);
                    }
                    commit(buf_empty + vb);
                    if (more) {
                        if (two) scores(1, kb);
                        commit(buf_empty + kb);
                    }
                    it += more ? 2 : 1;
                }
            }
        }
        __syncwarp();
    } else if (warp >= 8) {
        // ---------------- codes to fp16 ----------------
        const int w = warp - 8;
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
                            tabs[(gj % kTabs) * 8 + lane] = make_float4(
                                none ? 0.0f : ks * a.scale_log2, none ? -INFINITY : lg2(vsc), vs == vs ? 1.0f / vsc : 1.0f, 0.0f);
                        }
                        __syncwarp();
                        if (lane == 0) mbar_arrive(smem_u32(tab_full + gj % kTabs));
                    }
                    const uint8_t* raw = smem + C::kRawOff + st * C::kRawTile;
                    uint8_t* out = smem + C::kBufOff + buf * C::kTile;
                    constexpr int CH = D / 16 < 4 ? D / 16 : 4;  // 16-byte chunks of a row that neighbouring lanes read
                    constexpr int STEP = 32 / CH;                // rows of a warp's load
#pragma unroll
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
    } else {
        // ---------------- a thread per row ----------------
        const int x = warp >> 2;                               // row tile
        const int rl = (warp & 3) * 32 + lane;                 // row in it = tensor memory lane
        const uint32_t lane_base = uint32_t((warp & 3) * 32) << 16;
        const uint32_t s_addr = tmem + lane_base + kSCol + x * 128, o_addr = tmem + lane_base + kOCol + x * 128;
        int g = 0;   // key tiles of this row tile so far
        int gj = 0;  // key tiles of the CTA so far
        bool ok = true;
        for (; !walk.done() && ok; walk.next(a)) {
            if (x == 1 && walk.r.rows - walk.rt * kPromptRows <= 128) {
                gj += walk.n;
                continue;
            }
            const int r = walk.rt * kPromptRows + x * 128 + rl;
            const bool live = r < walk.r.rows;
            const int token = live ? r / a.group : 0, head = walk.head * a.group + (live ? r % a.group : 0);
            Row row;
            row.unit = 1.0f;
            row.mr = -INFINITY;
            row.l = 0.0f;
            const int place = walk.r.begin + token;
            row.hi = !live ? INT_MAX : a.causal ? min(place + 1, walk.r.length) : walk.r.length;
            row.lo = !live ? 0 : max(walk.r.first, a.window > 0 ? place - a.window + 1 : 0);
            {
                const uint16_t* src = a.q.p + (walk.r.token0 + token) * a.q.token_stride + head * a.q.head_stride;
                uint4 v[D / 8];
#pragma unroll
                for (int i = 0; i < D / 8; ++i)
                    v[i] = live ? __ldg(reinterpret_cast<const uint4*>(src) + i) : make_uint4(0, 0, 0, 0);
                if constexpr (BF16) {
                    // over the power of two at the row's largest element, as in ebx_kv_attention.cu
                    uint32_t top = 0;
#pragma unroll
                    for (int i = 0; i < D / 8; ++i) {
                        const uint32_t m = 0x7fff7fffu;
                        top = __vmaxu2(top, __vmaxu2(__vmaxu2(v[i].x & m, v[i].y & m), __vmaxu2(v[i].z & m, v[i].w & m)));
                    }
                    top = max(top & 0xffffu, top >> 16);
                    const uint32_t e = min(max(top >> 7, 1u), 253u);
                    const float down = __uint_as_float((254u - e) << 23);
                    row.unit = __uint_as_float(e << 23);
                    auto half = [&](uint32_t b) {
                        return pack_half2(__uint_as_float(b << 16) * down, __uint_as_float(b & 0xffff0000u) * down);
                    };
#pragma unroll
                    for (int i = 0; i < D / 8; ++i) v[i] = make_uint4(half(v[i].x), half(v[i].y), half(v[i].z), half(v[i].w));
                }
                uint8_t* dst = smem + x * C::kTile + rl * 128;
#pragma unroll
                for (int i = 0; i < D / 8; ++i)
                    *reinterpret_cast<uint4*>(dst + (i / 8) * kHalf + (((i & 7) ^ (rl & 7)) << 4)) = v[i];
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(q_full + x));
            }
            // keys that every row of the warp sees
            const int all_lo = __reduce_max_sync(0xffffffffu, row.lo), all_hi = __reduce_min_sync(0xffffffffu, row.hi);
            // moves mr of the rows whose t reached `top`, and what was summed with the old one
            auto raise = [&](float top, int j) {
                const bool up = top > row.mr + (kLag + kShift);
                const float mr = up ? top - kShift : row.mr;
                const float f = up ? ex2(row.mr - mr) : 1.0f;
                row.mr = mr;
                row.l *= f;
                if (j == 0) return true;
                if (!__all_sync(0xffffffffu, pwait(o_done + x, g - 1))) return false;
                after_sync();
#pragma unroll 1
                for (int c = 0; c < D / 32; ++c) {
                    uint32_t v[32];
                    tmem_ld32(o_addr + c * 32, v);
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * f);
                    tmem_st32<0>(o_addr + c * 32, v);
                }
                return true;
            };
            for (int j = 0; j < walk.n; ++j, ++g, ++gj) {
                ok = pwait(s_full + x, g) && pwait(tab_full + gj % kTabs, gj / kTabs);
                if (!__all_sync(0xffffffffu, ok)) {
                    ok = false;
                    break;
                }
                after_sync();
                const float4* tab = tabs + (gj % kTabs) * 8;
                const int key0 = (walk.t0 + j) * kPromptKeys;
                const bool mask = key0 < all_lo || key0 + kPromptKeys > all_hi;
                uint32_t p[64];
                float sum, top;
                if (__any_sync(0xffffffffu, row.mr == -INFINITY)) {
                    ok = raise(largest(s_addr, tab, row, key0), j);
                    if (!__all_sync(0xffffffffu, ok)) {
                        ok = false;
                        break;
                    }
                }
                for (int again = 0; again < 2; ++again) {
                    const float mr = row.mr == -INFINITY ? 0.0f : row.mr;
                    if (mask) weigh<true>(s_addr, tab, row, mr, key0, p, sum, top);
                    else weigh<false>(s_addr, tab, row, mr, key0, p, sum, top);
                    if (!__any_sync(0xffffffffu, top > kLag + kShift)) break;
                    if (again == 0 && !__all_sync(0xffffffffu, raise(top + mr, j))) {
                        ok = false;
                        break;
                    }
                }
                if (!ok) break;
                row.l += sum;
                tmem_st32<0>(s_addr, p);
                tmem_st32<32>(s_addr + 32, p);
                asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory");
                before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(p_full + x));
            }
            if (!ok) break;
            if (!__all_sync(0xffffffffu, pwait(o_done + x, g - 1))) {
                ok = false;
                break;
            }
            after_sync();
            const bool whole = walk.begins && walk.ends;
            const int slot = walk.begins ? 1 : 0;
            const float inv = row.l == 0.0f ? 0.0f : 1.0f / row.l;
            const int64_t at_row = int64_t(walk.r.token0 + token) * a.heads + head;
            float* part = whole ? nullptr
                                : a.part + ((2 * int64_t(blockIdx.x) + slot) * kPromptRows + x * 128 + rl) * (D + 2);
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
                uint32_t v[32];
                tmem_ld32(o_addr + c * 32, v);
                if (live && whole) {
                    uint4* dst = reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + at_row * D + c * 32);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint32_t h[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            h[k] = pack16<BF16>(__uint_as_float(v[8 * i + 2 * k]) * inv, __uint_as_float(v[8 * i + 2 * k + 1]) * inv);
                        dst[i] = make_uint4(h[0], h[1], h[2], h[3]);
                    }
                } else if (live) {
#pragma unroll
                    for (int i = 0; i < 32; i += 2)
                        *reinterpret_cast<uint2*>(part + c * 32 + i) = make_uint2(v[i], v[i + 1]);
                }
                __syncwarp();
            }
            before_sync();
            if (live && whole && a.lse)
                a.lse[at_row] = row.l == 0.0f ? -INFINITY : (row.mr + lg2(row.l)) * 0.6931471805599453f;
            if (live && !whole) *reinterpret_cast<float2*>(part + D) = make_float2(row.mr, row.l);
            if (!whole && threadIdx.x == 0)
                a.desc[2 * blockIdx.x + slot] = kv_desc(walk.r, walk.rt, kPromptRows, walk.head, walk.ends);
        }
    }

    before_sync();
    __syncthreads();
    if (warp == 12) {
        after_sync();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;\n" ::"r"(tmem) : "memory");
    }
}

constexpr int kPromptLeast = 4;  // key tiles a CTA takes at least

template <int D, bool BF16>
cudaError_t launch_prompt(KvAttnArgs a, void* ws, int dev, cudaStream_t s) {
    using C = PromptCfg<D>;
    static_assert(C::kSmem <= 227 * 1024, "shared memory of the prompt kernel");
    auto kern = kv_prompt_kernel<D, BF16>;
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
    a.part = reinterpret_cast<float*>(a.desc + 2 * grid);
    kern<<<grid, kPromptThreads, C::kSmem, s>>>(mk, mv, a, kPromptLeast);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    return launch_join<D, kPromptRows, BF16>(a, grid, 16, s);
}

}  // namespace

uint64_t kv_prompt_workspace_bytes(int head_dim, int sms) {
    return uint64_t(round_up(int64_t(sms) * 2 * int64_t(sizeof(int4) + kPromptRows * (head_dim + 2) * sizeof(float)), 256));
}

cudaError_t launch_kv_prompt(const KvAttnArgs& a, bool bf16, void* ws, int dev, cudaStream_t s) {
    switch (a.pool.head_dim) {
        case 32: return bf16 ? launch_prompt<32, true>(a, ws, dev, s) : launch_prompt<32, false>(a, ws, dev, s);
        case 64: return bf16 ? launch_prompt<64, true>(a, ws, dev, s) : launch_prompt<64, false>(a, ws, dev, s);
        default: return bf16 ? launch_prompt<128, true>(a, ws, dev, s) : launch_prompt<128, false>(a, ws, dev, s);
    }
}

cudaError_t read_kv_prompt_status(int* status, bool clear, cudaStream_t s) {
    return read_status_word(g_kv_prompt_status, status, clear, s);
}

}  // namespace ebx
