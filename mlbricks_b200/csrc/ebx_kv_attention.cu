// ebx_kv_attention.cu -- attention over the 8-bit paged cache.
//
// For a query row q of head h at position p, over the keys j that it sees:
//     s_j = scale * (q . kc_j) * ks_j,   out = sum_j e^(s_j) vs_j vc_j / sum_j e^(s_j),
// kc, vc the int8 codes and ks, vs the scales of the key's block.  The codes are exact fp16
// operands (an integer below 2048 is), so the products run on the tensor cores and the scales
// stay in fp32: with c = scale * log2(e) * ks_j and b = log2(vs_j),
//     t_j = c (q . kc_j) + b,  w_j = 2^(t_j - m),  O = sum_j w_j vc_j,  l = sum_j w_j / vs_j,
// m near the running maximum of t, so that the weight w_j, which carries the value's scale, fits
// fp16 for the second product whatever the scale's size, and one exponential serves both sums.  V scales
// below 2^-100 count as 2^-100.  out = O / l and the log-sum-exp is ln2 * (m + log2 l).
#include <algorithm>
#include <atomic>
#include <climits>
#include <cmath>

#include "ebx_kv_work.cuh"

namespace ebx {
namespace {

__device__ int g_kv_status = 0;
__device__ const float kv_none = kKvNone;  // for the copies of scales

__device__ __forceinline__ bool kv_wait(uint32_t bar, uint32_t parity) {
    if (mbar_wait_bounded(bar, parity)) return true;
    atomicExch(&g_kv_status, 0x7104);
    return false;
}

// ---- few rows: decode ---------------------------------------------------------------------
//
// A CTA streams key tiles of 8 KB a side through a ring of three stages (TMA boxes of one block,
// swizzled over the row's own width so that the fragment loads below are free of bank conflicts);
// four warps take 16 tokens each with a maximum, sums and O of their own, which are merged once per
// row tile.  S^T = K q^T and O^T = V^T w^T: the codes are the 16-row operand of mma.m16n8k16 and the
// 8 queries its columns, so a group of four heads fills half of the product and not a quarter of one
// with 16 rows (166 -> 112 us for 64 requests), and V is never transposed: its fragments are byte
// permutes of four rows.  What bounds it: 64 requests of 1 to 8192 tokens, 8 heads of 128, stream
// 568 MB in 93 to 96 us inside the kernel = 6.0 TB/s, 0.91 of a copy's rate; the call takes 107 us with its
// launch, the shares and the join.  Two CTAs with four stages 114 us, four CTAs with two 120 us.

constexpr int kConsumers = 4;    // warps that compute; one more loads
constexpr int kStepThreads = 32 * (kConsumers + 1);
constexpr int kStages = 3;
constexpr int kStepLeast = 4;   // units a CTA takes at least: a partial result costs about as much
constexpr int kStepExtra = 2;   // a row tile's begin and end, in key tiles (64 requests: 0 / 1 / 2: 112 / 109 / 106 us)

// D: head_dim; NQ: blocks of 8 rows (queries) in a row tile, the N of mma.m16n8k16, whose M is 16
// keys of the first product and 16 dimensions of the second.
template <int D, int NQ>
struct StepCfg {
    static constexpr int ROWS = 8 * NQ;
    static constexpr int PER_SM = NQ == 1 ? 3 : 2;   // CTAs of an SM that the registers allow
    static constexpr int KT = 8192 / D;              // tokens of a key tile: 8 KB of codes a side
    static constexpr int UNITS = KT / 16;            // 16 tokens lie in one block: one scale
    static constexpr int PER_WARP = UNITS / kConsumers;
    static constexpr int kStageBytes = 2 * 8192;
    static constexpr int kMergeBytes = kConsumers * ROWS * (D + 4) * 4;
    static constexpr int kSmem = 1024 + kStages * kStageBytes + kMergeBytes + kStages * 2 * UNITS * 4 + 256;
};

// Byte `b` of row `r` in a tile that TMA wrote with the swizzle of a D-byte row.
template <int D>
__device__ __forceinline__ uint32_t swz(int r, int b) {
    const int x = D == 128 ? (r & 7) : D == 64 ? ((r >> 1) & 3) : ((r >> 2) & 1);
    return uint32_t(r * D + (b ^ (x << 4)));
}

// Row i of an 8-key block of the first product is key {0,5,2,7,1,4,3,6}[i] of its eight: with this
// order the loads of K rows (by i) and of V rows (by i / 2, for i even and odd) are free of bank
// conflicts under each of the three swizzles.
__device__ __forceinline__ int key_even(int c) { return ((c & 1) << 1) | (c >> 1); }        // 0 2 1 3
__device__ __forceinline__ int key_odd(int c) { return 4 + (key_even(c) ^ 1); }             // 5 7 4 6

template <int BYTES>
__device__ __forceinline__ void lds(uint32_t addr, uint32_t (&w)[BYTES / 4]) {
    if constexpr (BYTES == 16)
        asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                     : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(addr));
    else if constexpr (BYTES == 8)
        asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(addr));
    else
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[0]) : "r"(addr));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

template <int D, int NQ, bool BF16>
__global__ void __launch_bounds__(kStepThreads, (StepCfg<D, NQ>::PER_SM))
    kv_step_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                   const __grid_constant__ KvAttnArgs a, int least) {
    using C = StepCfg<D, NQ>;
    constexpr int KT = C::KT, UNITS = C::UNITS, kRows = C::ROWS;
    constexpr int KB = D >= 64 ? 16 : 8;        // bytes of a K row that a lane loads at once
    constexpr int KL = D / (4 * KB);            // such loads for a row
    constexpr int KW = KB / 4;                  // words of it = products of depth 16
    constexpr int VB = D / 8;                   // bytes of a V row that a lane loads
    constexpr int MT = D / 16;                  // 16-dimension tiles of O
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    float* merge = reinterpret_cast<float*>(smem + kStages * C::kStageBytes);
    float* scales = reinterpret_cast<float*>(smem + kStages * C::kStageBytes + C::kMergeBytes);  // [stage][k, v][unit]
    uint64_t* full = reinterpret_cast<uint64_t*>(scales + kStages * 2 * UNITS);
    uint64_t* empty = full + kStages;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < kStages; ++i) {
            mbar_init(smem_u32(&full[i]), 1 + 32);  // the copies' bytes, and each loading lane's scales
            mbar_init(smem_u32(&empty[i]), kConsumers);
        }
        fence_proxy_async_smem();
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");  // nothing of the call's inputs is read before
    const KvShare share = kv_share<kRows, KT, kStepExtra, kStepThreads>(a, least, reinterpret_cast<int*>(smem));
    fence_proxy_async_smem();  // the ring's copies may overwrite what kv_share kept there
    if (threadIdx.x == 0 && !a.whole) a.desc[blockIdx.x] = make_int4(0, 0, 0, 0);
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the join waits for this grid's end
    __syncthreads();
    KvWalk<kRows, KT, kStepExtra> walk;
    walk.start(a, share);
    const int bsize = a.pool.block_size;

    if (warp == kConsumers) {
        // ---- loader: codes by TMA, a box per block, scales by cp.async ----
        const int box = min(bsize, KT);           // tokens of a box
        const int boxes = KT / box;
        const int ops = 2 * boxes;                // <= 32: a lane each
        const bool op = lane < ops, op_v = lane >= boxes;
        const int op_row = (op_v ? lane - boxes : lane) * box;
        const bool sc = lane < 2 * UNITS, sc_v = lane >= UNITS;
        const int sc_row = (sc_v ? lane - UNITS : lane) * 16;
        int it = 0;
        bool ok = true;
        const int none = a.pool.blocks;           // past the pool: TMA fills with zeros
        for (; !walk.done() && ok; walk.next(a)) {
            const int32_t* row = a.tables + int64_t(walk.request) * a.width;
            auto block_of = [&](int tile, int r) {  // the block of a key tile's token r
                const int token = tile * KT + r, column = token >> a.pool.shift;
                if (token >= walk.r.length || column >= a.width) return none;
                const int id = __ldg(row + column);
                return id < 0 || id > none ? none : id;
            };
            int id_next = block_of(walk.t0, op_row), sid_next = block_of(walk.t0, sc_row);
            for (int j = 0; j < walk.n; ++j, ++it) {
                const int tile = walk.t0 + j, st = it % kStages;
                const int id = id_next, sid = sid_next;
                if (j + 1 < walk.n) {
                    id_next = block_of(tile + 1, op_row);
                    sid_next = block_of(tile + 1, sc_row);
                }
                bool free = true;
                if (it >= kStages) free = kv_wait(smem_u32(&empty[st]), uint32_t((it / kStages - 1) & 1));
                if (!__all_sync(0xffffffffu, free)) {
                    ok = false;
                    break;
                }
                const uint32_t bar = smem_u32(&full[st]);
                if (lane == 0) mbar_expect_tx(bar, C::kStageBytes);
                __syncwarp();
                const uint32_t stage = smem_u32(smem + st * C::kStageBytes);
                if (op) {
                    const int token = tile * KT + op_row;
                    const int64_t r = (int64_t(id) * a.pool.kv_heads + walk.head) * bsize + (token & (bsize - 1));
                    const int64_t rows = int64_t(none) * a.pool.kv_heads * bsize;
                    kv_tma_2d(stage + (op_v ? 8192 : 0) + op_row * D, op_v ? &map_v : &map_k, 0,
                              int(id == none ? rows : r), bar);
                }
                if (sc) {
                    const int64_t cell = int64_t(sid) * a.pool.kv_heads + walk.head;
                    const float* src = sid == none ? &kv_none : (sc_v ? a.pool.v_scales : a.pool.k_scales) + cell;
                    cp_async4(smem_u32(scales + (st * 2 + (sc_v ? 1 : 0)) * UNITS + sc_row / 16), src);
                }
                asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];\n" ::"r"(bar) : "memory");
            }
        }
        asm volatile("cp.async.wait_all;\n" ::: "memory");
        if (!ok)  // given up: copies on their way land before this shared memory is another CTA's
            for (int i = max(it - kStages, 0); i < it; ++i) kv_wait(smem_u32(&full[i % kStages]), uint32_t((i / kStages) & 1));
        return;
    }

    // ---- consumers: warp w takes tokens [w KT/4, (w + 1) KT/4) of every key tile ----
    const int c = lane & 3, n8 = lane >> 2;
    const int krow = (n8 & 1) ? key_odd(n8 >> 1) : key_even(n8 >> 1);
    const int vrow0 = key_even(c), vrow1 = key_odd(c);
    // the D / 8 bytes of a V row, and dimensions of O, of this lane
    const int vbyte = D == 128 ? 16 * ((n8 >> 1) | ((n8 & 1) << 2))
                      : D == 64 ? 8 * (2 * ((((n8 >> 1) & 1) << 1) | (n8 >> 2)) + (n8 & 1)) : 4 * n8;
    int it = 0;
    bool ok = true;
    for (; !walk.done(); walk.next(a)) {
        // q: row n8 of each block of 8, this lane's dimensions of the KL KW products of depth 16
        uint32_t qb[NQ][KL * KW][2];
        float unit[NQ][2];               // what the rows 2c and 2c + 1 of q were divided by
        int lo[NQ][2], hi[NQ][2];        // they see keys [lo, hi); a row past the last is not kept
#pragma unroll
        for (int nq = 0; nq < NQ; ++nq) {
            {
                const int r = walk.rt * kRows + 8 * nq + n8;
                const bool in = r < walk.r.rows;
                const int token = in ? by_group(a, r) : 0;
                const uint16_t* src = a.q.p + (walk.r.token0 + token) * a.q.token_stride +
                                      (walk.head * a.group + (in ? r - token * a.group : 0)) * a.q.head_stride + c * KB;
#pragma unroll
                for (int l = 0; l < KL; ++l)
#pragma unroll
                    for (int q = 0; q < KW; q += 2) {
                        uint4 v = make_uint4(0, 0, 0, 0);
                        if (in) v = __ldg(reinterpret_cast<const uint4*>(src + l * 4 * KB + q * 4));
                        qb[nq][l * KW + q][0] = v.x;
                        qb[nq][l * KW + q][1] = v.y;
                        qb[nq][l * KW + q + 1][0] = v.z;
                        qb[nq][l * KW + q + 1][1] = v.w;
                    }
            }
            if constexpr (BF16) {
                // fp16 operands: each row over the power of two at its largest element, so that every
                // element of at least 2^-14 of it is exact and the others are off by 2^-25 of it
                uint32_t top = 0;
#pragma unroll
                for (int i = 0; i < KL * KW; ++i)
                    top = __vmaxu2(top, __vmaxu2(qb[nq][i][0] & 0x7fff7fffu, qb[nq][i][1] & 0x7fff7fffu));
                top = max(top & 0xffffu, top >> 16);
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const uint32_t e = min(max(top >> 7, 1u), 253u);  // 2^(e - 127)
                const float down = __uint_as_float((254u - e) << 23);
#pragma unroll
                for (int i = 0; i < KL * KW; ++i)
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        const uint32_t v = qb[nq][i][q];
                        qb[nq][i][q] = pack_half2(__uint_as_float(v << 16) * down, __uint_as_float(v & 0xffff0000u) * down);
                    }
#pragma unroll
                for (int i = 0; i < 2; ++i) unit[nq][i] = __uint_as_float(__shfl_sync(0xffffffffu, e << 23, (2 * c + i) * 4));
            } else {
                unit[nq][0] = unit[nq][1] = 1.0f;
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int r = walk.rt * kRows + 8 * nq + 2 * c + i;
                const bool in = r < walk.r.rows;
                const int place = walk.r.begin + by_group(a, r);
                hi[nq][i] = !in ? INT_MAX : a.causal ? min(place + 1, walk.r.length) : walk.r.length;
                lo[nq][i] = !in ? 0 : max(walk.r.first, a.window > 0 ? place - a.window + 1 : 0);
            }
        }
        float o[NQ][MT][4];
        float m[NQ][2], l[NQ][2];
        int all_lo = 0, all_hi = INT_MAX;
#pragma unroll
        for (int nq = 0; nq < NQ; ++nq) {
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[nq][t][i] = 0.0f;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                m[nq][i] = -INFINITY;
                l[nq][i] = 0.0f;
                all_lo = max(all_lo, lo[nq][i]);
                all_hi = min(all_hi, hi[nq][i]);
            }
        }
        // the keys that every row of the tile sees
        all_lo = __reduce_max_sync(0xffffffffu, all_lo);
        all_hi = __reduce_min_sync(0xffffffffu, all_hi);

        for (int j = 0; j < walk.n; ++j, ++it) {
            const int st = it % kStages;
            if (ok) ok = __all_sync(0xffffffffu, kv_wait(smem_u32(&full[st]), uint32_t((it / kStages) & 1)));
            if (!ok) continue;  // recorded; the barriers below are still met
            const uint32_t kbase = smem_u32(smem + st * C::kStageBytes), vbase = kbase + 8192;
#pragma unroll 1
            for (int u0 = 0; u0 < C::PER_WARP; ++u0) {
                const int u = warp * C::PER_WARP + u0;
                const int key0 = (walk.t0 + j) * KT + u * 16;
                const float ks = scales[st * 2 * UNITS + u], vs = scales[(st * 2 + 1) * UNITS + u];
                // S^T: 16 keys (rows) by 8 queries; this lane's keys krow, krow + 8, queries 2c, 2c + 1
                float s[NQ][4];
#pragma unroll
                for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[nq][i] = 0.0f;
#pragma unroll
                for (int x = 0; x < KL; ++x) {
                    uint32_t w0[KW], w1[KW];
                    lds<KB>(kbase + swz<D>(u * 16 + krow, x * 4 * KB + c * KB), w0);
                    lds<KB>(kbase + swz<D>(u * 16 + 8 + krow, x * 4 * KB + c * KB), w1);
#pragma unroll
                    for (int q = 0; q < KW; ++q) {
                        const uint32_t v0 = w0[q] ^ 0x80808080u, v1 = w1[q] ^ 0x80808080u;
                        const uint32_t ka[4] = {codes_to_half2(v0, 0x4140), codes_to_half2(v1, 0x4140),
                                                codes_to_half2(v0, 0x4342), codes_to_half2(v1, 0x4342)};
#pragma unroll
                        for (int nq = 0; nq < NQ; ++nq) mma_16816(s[nq], ka, qb[nq][x * KW + q][0], qb[nq][x * KW + q][1]);
                    }
                }
                uint32_t v00[VB / 4], v01[VB / 4], v10[VB / 4], v11[VB / 4];
                lds<VB>(vbase + swz<D>(u * 16 + vrow0, vbyte), v00);
                lds<VB>(vbase + swz<D>(u * 16 + vrow1, vbyte), v01);
                lds<VB>(vbase + swz<D>(u * 16 + 8 + vrow0, vbyte), v10);
                lds<VB>(vbase + swz<D>(u * 16 + 8 + vrow1, vbyte), v11);
                const bool none = vs < 0.0f;  // kKvNone
                const float vsc = vs < 0x1p-100f ? 0x1p-100f : vs;  // NaN stays
                const float b = none ? -INFINITY : lg2(vsc);
                const float inv = vs == vs ? rcp(vsc) : 1.0f;  // NaN goes through t, where the mask stops it
                const float cs = none ? 0.0f : ks * a.scale_log2;
                const bool edge = key0 < all_lo || key0 + 16 > all_hi;
                uint32_t p[NQ][2];  // w^T as the second product's keys-by-queries operand
                float top[NQ][2];
                bool grew = false;
#pragma unroll
                for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const float cf = cs * unit[nq][i];
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            float& t = s[nq][2 * h + i];
                            t = fmaf(t, cf, b);
                            if (edge) {
                                const int key = key0 + 8 * h + krow;
                                if (key < lo[nq][i] || key >= hi[nq][i]) t = -INFINITY;
                            }
                        }
                        top[nq][i] = fmaxf(s[nq][i], s[nq][2 + i]);
                        grew |= top[nq][i] > m[nq][i] + kLag;
                    }
                // the running maximum moves only when it grew by more than 2^kLag, so that most
                // tiles rescale nothing (and need not agree on their largest)
                if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
                    for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            float t = top[nq][i];
                            t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 4));
                            t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 8));
                            t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 16));
                            const float mn = fmaxf(m[nq][i], t);
                            const float f = mn == m[nq][i] ? 1.0f : ex2(m[nq][i] - mn);
                            m[nq][i] = mn;
                            l[nq][i] *= f;
#pragma unroll
                            for (int y = 0; y < MT; ++y) {
                                o[nq][y][i] *= f;
                                o[nq][y][2 + i] *= f;
                            }
                        }
                }
#pragma unroll
                for (int nq = 0; nq < NQ; ++nq) {
                    float w[4];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const float mr = m[nq][i] == -INFINITY ? 0.0f : m[nq][i] - kShift;
                        w[i] = ex2(s[nq][i] - mr);
                        w[2 + i] = ex2(s[nq][2 + i] - mr);
                        l[nq][i] = fmaf(w[i] + w[2 + i], inv, l[nq][i]);
                    }
                    p[nq][0] = transpose8x8(pack_half2(w[0], w[1]));  // 11 bits, as the codes' operands need
                    p[nq][1] = transpose8x8(pack_half2(w[2], w[3]));
                }
#pragma unroll
                for (int q = 0; q < VB / 4; ++q) {
#pragma unroll
                    for (int y = 0; y < 2; ++y) {  // dimensions 4q + 2y and 4q + 2y + 1 of the lane's
                        const uint32_t sel = y ? 0x7362 : 0x5140;  // {even key, odd key} of each
                        const uint32_t x0 = __byte_perm(v00[q], v01[q], sel) ^ 0x80808080u;
                        const uint32_t x1 = __byte_perm(v10[q], v11[q], sel) ^ 0x80808080u;
                        const uint32_t va[4] = {codes_to_half2(x0, 0x4140), codes_to_half2(x0, 0x4342),
                                                codes_to_half2(x1, 0x4140), codes_to_half2(x1, 0x4342)};
#pragma unroll
                        for (int nq = 0; nq < NQ; ++nq) mma_16816(o[nq][2 * q + y], va, p[nq][0], p[nq][1]);
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&empty[st]));
        }

        // ---- the four warps' results become one ----
        const int rows = min(kRows, walk.r.rows - walk.rt * kRows);
        float* mine = merge + warp * kRows * (D + 4);  // row: D values, m, l
#pragma unroll
        for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float sum = l[nq][i];
                sum += __shfl_xor_sync(0xffffffffu, sum, 4);
                sum += __shfl_xor_sync(0xffffffffu, sum, 8);
                sum += __shfl_xor_sync(0xffffffffu, sum, 16);
                const int r = 8 * nq + 2 * c + i;
                if (r < rows) {
                    float* dst = mine + r * (D + 4);
#pragma unroll
                    for (int t = 0; t < MT; t += 2)
                        *reinterpret_cast<float4*>(dst + vbyte + 2 * t) =
                            make_float4(o[nq][t][i], o[nq][t][2 + i], o[nq][t + 1][i], o[nq][t + 1][2 + i]);
                    if (n8 == 0) {
                        dst[D] = m[nq][i] - kShift;
                        dst[D + 1] = sum;
                    }
                }
            }
        asm volatile("bar.sync 1, %0;" ::"n"(32 * kConsumers) : "memory");
        const bool whole = walk.whole();
        const int slot = walk.begins ? 1 : 0;
        for (int w = threadIdx.x; w < rows * (D / 4); w += 32 * kConsumers) {
            const int r = w / (D / 4), d = (w % (D / 4)) * 4;
            const float* src = merge + r * (D + 4);
            float mm = -INFINITY;
#pragma unroll
            for (int x = 0; x < kConsumers; ++x) mm = fmaxf(mm, src[x * kRows * (D + 4) + D]);
            float4 sum = make_float4(0, 0, 0, 0);
            float ll = 0.0f;
#pragma unroll
            for (int x = 0; x < kConsumers; ++x) {
                const float* y = src + x * kRows * (D + 4);
                const float f = y[D] == mm ? 1.0f : ex2(y[D] - mm);
                const float4 v = *reinterpret_cast<const float4*>(y + d);
                sum.x = fmaf(v.x, f, sum.x); sum.y = fmaf(v.y, f, sum.y);
                sum.z = fmaf(v.z, f, sum.z); sum.w = fmaf(v.w, f, sum.w);
                ll = fmaf(y[D + 1], f, ll);
            }
            if (whole) {
                const int row = walk.rt * kRows + r;
                const int token = by_group(a, row);
                const int64_t at_row = int64_t(walk.r.token0 + token) * a.heads + walk.head * a.group + row - token * a.group;
                const float inv = ll == 0.0f ? 0.0f : 1.0f / ll;
                uint2 pk;
                pk.x = pack16<BF16>(sum.x * inv, sum.y * inv);
                pk.y = pack16<BF16>(sum.z * inv, sum.w * inv);
                *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + at_row * D + d) = pk;
                if (a.lse && d == 0) a.lse[at_row] = ll == 0.0f ? -INFINITY : (mm + lg2(ll)) * 0.6931471805599453f;
            } else {
                reinterpret_cast<float4*>(kv_part<D, kRows>(a, blockIdx.x, slot))[d / 4 * kRows + r] = sum;
                if (d == 0) kv_part_ml<D, kRows>(a, blockIdx.x, slot)[r] = make_float2(mm, ll);
            }
        }
        if (walk.begins && !whole && threadIdx.x == 0)
            a.desc[blockIdx.x] = kv_desc(walk.r, walk.rt, kRows, walk.head, walk.last() - int(blockIdx.x));
        asm volatile("bar.sync 1, %0;" ::"n"(32 * kConsumers) : "memory");  // merge is free again
    }
}

template <int D, int NQ, bool BF16>
cudaError_t launch_step(KvAttnArgs a, int rows, void* ws, int dev, cudaStream_t s) {
    using C = StepCfg<D, NQ>;
    auto kern = kv_step_kernel<D, NQ, BF16>;
    static std::atomic<uint64_t> configured{0};
    const uint64_t bit = 1ull << (dev & 63);
    if (!(configured.load(std::memory_order_relaxed) & bit)) {
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
        if (e != cudaSuccess) return e;
        configured.fetch_or(bit);
    }
    CUtensorMap mk, mv;
    const int box = std::min(a.pool.block_size, C::KT);
    if (!code_map(&mk, a.pool.k_codes, a.pool, box) || !code_map(&mv, a.pool.v_codes, a.pool, box))
        return cudaErrorInvalidValue;
    const int grid = gemm_sm_count(dev) * C::PER_SM;
    a.desc = static_cast<int4*>(ws);
    a.part = reinterpret_cast<float*>(a.desc + grid);
    const cudaError_t e = launch_early(kern, dim3(grid), kStepThreads, C::kSmem, s, mk, mv, a, kStepLeast);
    if (e != cudaSuccess) return e;
    return launch_join<D, C::ROWS, 4, BF16>(a, grid, std::min(rows, C::ROWS), s);
}

}  // namespace

namespace {

// From kPromptMin rows of a request and head on, row tiles of 256 rows on tcgen05; below, tiles of 8
// or 16.  Measured with the rule at 17 and at 65 rows (step / prompt kernel): 16 requests of 4000
// tokens, 8 heads of 128, 32 rows 66 / 95 us, 48 rows 94 / 96, 64 rows 119 / 97; 64 requests of 2000
// tokens, 2 heads of 64, 48 rows 39 / 54, 64 rows 47 / 54; one request of 16000, 48 rows 31 / 41.
constexpr int kPromptMin = 49;

// Short requests: a second launch, to join, would cost more than sharing row tiles gains.  With / without
// this, captured: 8 requests of 600 tokens, 12 heads over one of 32, 9.5 / 12.5 us; 8 of 256, 32 heads over 8 of 128,
// 7.7 / 11.4; 64 of 100 11.7 / 12.8, of 256 15.4 / 14.9.  At twice the length it depends on how many there are:
// 8 of 512 9.9 / 12.0, 64 of 512 23.2 / 19.8.
bool takes_whole(int head_dim, int max_length) {
    constexpr int kTiles = 4;
    return max_length > 0 && max_length <= kTiles * (8192 / head_dim);
}

// Rows of one request and key/value head, at most.
int64_t most_rows(int group, int64_t tokens, int max_new) {
    return (max_new > 0 ? std::min<int64_t>(max_new, tokens) : tokens) * group;
}

// A prompt or two among decode steps: if the other requests bring fewer than kPromptMin / 2 rows on
// average, both kernels run, each for its own requests: a decode row streams at a third of its rate
// in the prompt kernel.  Measured, both / the prompt kernel alone, 32 heads over 8 of 128: 63 requests
// of 4000 tokens and a prompt of 2048 188 / 383 us, of 256 141 / 310; 200 of 500 and one of 300 101 / 189.
bool takes_both(int group, int requests, int64_t tokens, int max_new) {
    return requests > 1 && max_new > 0 && tokens > max_new && int64_t(max_new) * group >= kPromptMin &&
           (tokens - max_new) * group * 2 < int64_t(requests - 1) * kPromptMin;
}

}  // namespace

uint64_t kv_attention_workspace_bytes(int head_dim, int group, int64_t tokens, int max_new, int max_length) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return 0;
    const int sms = gemm_sm_count(dev);
    const int64_t most = most_rows(group, tokens, max_new);
    if (most >= kPromptMin) return kv_prompt_workspace_bytes(head_dim, sms);  // more than the step kernel's
    if (takes_whole(head_dim, max_length)) return 0;
    const int nq = most <= 8 ? 1 : 2, ctas = sms * (nq == 1 ? StepCfg<32, 1>::PER_SM : StepCfg<32, 2>::PER_SM);
    return uint64_t(round_up(int64_t(ctas) * int64_t(sizeof(int4) + 2 * 8 * nq * (head_dim + 2) * sizeof(float)), 256));
}

cudaError_t launch_kv_attention(KvAttnArgs a, bool bf16, int max_new, int max_length, void* ws, cudaStream_t s) {
    if (a.tokens <= 0 || a.requests <= 0) return cudaSuccess;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    a.least_rows = 0;
    a.most_rows = INT_MAX;
    int rows = int(most_rows(a.group, a.tokens, max_new));
    if (rows >= kPromptMin) {
        const bool both = takes_both(a.group, a.requests, a.tokens, max_new);
        if (both) a.least_rows = kPromptMin;
        e = launch_kv_prompt(a, bf16, ws, dev, s);
        if (e != cudaSuccess || !both) return e;
        a.least_rows = 0;
        a.most_rows = kPromptMin - 1;
        rows = a.group <= 8 ? a.group : kPromptMin - 1;  // most are single tokens; others take more row tiles
    } else {
        a.whole = takes_whole(a.pool.head_dim, max_length);
    }
    const bool few = rows <= 8;
#define EBX_KV_STEP(DD)                                                                              \
    (few ? (bf16 ? launch_step<DD, 1, true>(a, rows, ws, dev, s) : launch_step<DD, 1, false>(a, rows, ws, dev, s)) \
         : (bf16 ? launch_step<DD, 2, true>(a, rows, ws, dev, s) : launch_step<DD, 2, false>(a, rows, ws, dev, s)))
    switch (a.pool.head_dim) {
        case 32: return EBX_KV_STEP(32);
        case 64: return EBX_KV_STEP(64);
        default: return EBX_KV_STEP(128);
    }
#undef EBX_KV_STEP
}

cudaError_t read_kv_status(int* status, bool clear, cudaStream_t s) {
    int prompt = 0;
    cudaError_t e = read_status_word(g_kv_status, status, clear, s);
    if (e == cudaSuccess) e = read_kv_prompt_status(&prompt, clear, s);
    if (*status == 0) *status = prompt;
    return e;
}

}  // namespace ebx
