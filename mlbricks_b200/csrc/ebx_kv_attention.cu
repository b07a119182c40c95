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

template <int D, int NQ, bool BF16, bool SHARED>
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
    const KvShare share = kv_share<kRows, KT, kStepExtra, kStepThreads, SHARED>(a, least, reinterpret_cast<int*>(smem));
    fence_proxy_async_smem();  // the ring's copies may overwrite what kv_share kept there
    if (!SHARED && threadIdx.x == 0 && !a.whole) a.desc[blockIdx.x] = make_int4(0, 0, 0, 0);
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the join waits for this grid's end
    __syncthreads();
    KvWalk<kRows, KT, kStepExtra, SHARED> walk;
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
            const int32_t* row = a.tables + int64_t(kv_table_row<SHARED>(a, walk.request)) * a.width;
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
    // Where this lane's bytes of rows u * 16 + r and 8 rows on are: the swizzle there is that of row r.  Of 16 rows of a
    // prefix (four requests of 131000 shared tokens) that is 73 us and not 75; decode steps of 8 rows have no
    // registers for it (64 requests of up to 8192 tokens 96 us, not 95).
    constexpr bool KEPT = SHARED && NQ == 2;
    uint32_t k_at[KL];
#pragma unroll
    for (int x = 0; x < KL; ++x) k_at[x] = swz<D>(krow, x * 4 * KB + c * KB);
    const uint32_t v_at[2] = {swz<D>(vrow0, vbyte), swz<D>(vrow1, vbyte)};
    auto k_byte = [&](int u, int x, int on) {
        return KEPT ? uint32_t(u * 16 * D) + k_at[x] + on * D : swz<D>(u * 16 + on + krow, x * 4 * KB + c * KB);
    };
    auto v_byte = [&](int u, int odd, int on) {
        return KEPT ? uint32_t(u * 16 * D) + v_at[odd] + on * D : swz<D>(u * 16 + on + (odd ? vrow1 : vrow0), vbyte);
    };
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
                const uint16_t* src = a.q.p + kv_token<SHARED>(a, walk.request, walk.r, token) * a.q.token_stride +
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
                    lds<KB>(kbase + k_byte(u, x, 0), w0);
                    lds<KB>(kbase + k_byte(u, x, 8), w1);
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
                lds<VB>(vbase + v_byte(u, 0, 0), v00);
                lds<VB>(vbase + v_byte(u, 1, 0), v01);
                lds<VB>(vbase + v_byte(u, 0, 8), v10);
                lds<VB>(vbase + v_byte(u, 1, 8), v11);
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
            if constexpr (SHARED) {
                const int row = walk.rt * kRows + r;
                const int token = by_group(a, row), side = walk.request < a.groups ? 0 : 1;
                const int64_t at_row = int64_t(kv_token<true>(a, walk.request, walk.r, token)) * a.heads + walk.head * a.group +
                                       row - token * a.group;
                if (whole) {
                    const int64_t at = side * a.tokens * a.heads + at_row;
                    *reinterpret_cast<float4*>(a.sums + at * D + d) = sum;
                    if (d == 0) a.sums_ml[at] = make_float2(mm, ll);
                } else {
                    reinterpret_cast<float4*>(kv_part<D, kRows>(a, blockIdx.x, slot))[d / 4 * kRows + r] = sum;
                    if (d == 0) kv_part_ml<D, kRows>(a, blockIdx.x, slot)[r] = make_float2(mm, ll);
                }
                if (d == 0 && whole) kv_whole(a, side, at_row);
                else if (d == 0 && walk.begins) kv_begins(a, side, at_row, false, walk.last() - int(blockIdx.x), r);
            } else if (whole) {
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
        if (!SHARED && walk.begins && !whole && threadIdx.x == 0)
            a.desc[blockIdx.x] = kv_desc(walk.r, walk.rt, kRows, walk.head, walk.last() - int(blockIdx.x));
        asm volatile("bar.sync 1, %0;" ::"n"(32 * kConsumers) : "memory");  // merge is free again
    }
}

// SHARED: `ws` holds the parts, and the caller joins.
template <int D, int NQ, bool BF16, bool SHARED = false>
cudaError_t launch_step(KvAttnArgs a, int rows, void* ws, int dev, cudaStream_t s) {
    using C = StepCfg<D, NQ>;
    auto kern = kv_step_kernel<D, NQ, BF16, SHARED>;
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
    a.part = reinterpret_cast<float*>(SHARED ? a.desc : a.desc + grid);
    const cudaError_t e = launch_early(kern, dim3(grid), kStepThreads, C::kSmem, s, mk, mv, a, kStepLeast);
    if (e != cudaSuccess || SHARED) return e;
    return launch_join<D, C::ROWS, 4, BF16>(a, grid, std::min(rows, C::ROWS), s);
}

// ---- the join of rows over a prefix and their own part -----------------------------------------

struct SharedParts {
    const float* step;     // parts of either kernel, row tiles of step_rows and of kPromptTile
    const float* prompt;
    int step_rows, step_ctas, prompt_ctas;
};
constexpr int kPromptTile = 256;

// CTA y joins rows 4 y .. 4 y + 3 of [tokens * heads]: 4 rows x 8 column groups x WAYS that take the row's
// results in turn, those over the prefix first.  Only what the kernels before it wrote is followed.
template <int D, bool BF16, int WAYS>
__global__ void __launch_bounds__(32 * WAYS) kv_shared_join_kernel(const __grid_constant__ KvAttnArgs a, SharedParts parts) {
    asm volatile("griddepcontrol.launch_dependents;\n\tgriddepcontrol.wait;" ::: "memory");
    constexpr int COLS = D / 32;  // float4 columns of a thread: groups of 8 apart
    __shared__ float2 s_ml[WAYS][8][4];
    __shared__ float4 s_o[COLS][WAYS][8][4];
    const int ri = threadIdx.x & 3, col = (threadIdx.x >> 2) & 7, way = threadIdx.x >> 5;
    const int64_t rows = a.tokens * a.heads, row = int64_t(blockIdx.x) * 4 + ri;
    const int state = row < rows ? a.state[row / a.heads] : 0;
    int first[2], tile_row[2], count[2] = {0, 0};
    int2 both[2];
#pragma unroll
    for (int side = 0; side < 2; ++side) both[side] = row < rows ? a.where[side * rows + row] : make_int2(0, 0);
#pragma unroll
    for (int side = 0; side < 2; ++side) {
        if (state < 2 - side) continue;  // `where` then holds anything
        const int2 w = both[side];
        const int ctas = w.x < -1 ? parts.prompt_ctas : parts.step_ctas, c = w.x < -1 ? -2 - w.x : w.x;
        first[side] = w.x;
        tile_row[side] = w.y & 0xff;
        count[side] = w.x == -1 ? 1 : c < ctas ? min(max(w.y >> 8, 0) + 1, ctas - c) : 0;
        if (w.x != -1 && tile_row[side] >= (w.x < -1 ? kPromptTile : parts.step_rows)) count[side] = 0;
    }
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
    const int total = count[0] + count[1];
    constexpr int AHEAD = 4;  // results on their way at once
    for (int p0 = way; p0 < total; p0 += AHEAD * WAYS) {
        float4 v[AHEAD][COLS];
        float2 ml[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const int p = p0 + i * WAYS;
            if (p >= total) continue;
            const int side = p < count[0] ? 0 : 1, k = side ? p - count[0] : p;
            const int at = side ? first[1] : first[0], r = side ? tile_row[1] : tile_row[0];
            const float4* src;
            int stride;
            if (at == -1) {
                src = reinterpret_cast<const float4*>(a.sums + (side * rows + row) * D);
                stride = 1;
                ml[i] = a.sums_ml[side * rows + row];
            } else {
                const int tile = at < -1 ? kPromptTile : parts.step_rows;
                const float* part = (at < -1 ? parts.prompt : parts.step) +
                                    (2 * int64_t((at < -1 ? -2 - at : at) + k) + (k == 0)) * tile * (D + 2);
                src = reinterpret_cast<const float4*>(part) + r;
                stride = tile;
                ml[i] = reinterpret_cast<const float2*>(part + tile * D)[r];
            }
#pragma unroll
            for (int x = 0; x < COLS; ++x) v[i][x] = src[(x * 8 + col) * stride];
        }
#pragma unroll
        for (int i = 0; i < AHEAD; ++i)
            if (p0 + i * WAYS < total) join(ml[i].x, ml[i].y, v[i]);
    }
    s_ml[way][col][ri] = make_float2(m, l);
#pragma unroll
    for (int x = 0; x < COLS; ++x) s_o[x][way][col][ri] = o[x];
    __syncthreads();
    if (way != 0 || state == 0) return;
    for (int w = 1; w < min(WAYS, total); ++w) {
        float4 v[COLS];
#pragma unroll
        for (int x = 0; x < COLS; ++x) v[x] = s_o[x][w][col][ri];
        join(s_ml[w][col][ri].x, s_ml[w][col][ri].y, v);
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int x = 0; x < COLS; ++x) {
        uint2 pk;
        pk.x = pack16<BF16>(o[x].x * inv, o[x].y * inv);
        pk.y = pack16<BF16>(o[x].z * inv, o[x].w * inv);
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + row * D + 4 * (x * 8 + col)) = pk;
    }
    if (a.lse && col == 0) a.lse[row] = l == 0.0f ? -INFINITY : (m + lg2(l)) * 0.6931471805599453f;
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

// ---- with prefixes ------------------------------------------------------------------------------
//
// A softmax over a prefix and a rest is that of either, joined by their maxima and sums: with {O, m, l} of both,
//     m = max(m_p, m_r),  O = O_p 2^(m_p - m) + O_r 2^(m_r - m),  l likewise,  out = O / l,
// the same join that a row tile's parts need.  So a group of requests that share a prefix is one request more: its rows
// are the queries of all members, its keys the shared ones, none of which is masked, and every request keeps the keys
// behind them.  Groups and requests lie on one line of work; groups of kPromptMin rows and more go to the kernel for
// prompts, whose 256 rows read a key tile once.  A row's results, one or in parts, are then found through `where` and joined
// in one launch.  64 requests of 32 heads over 8 of 128, behind 8192 shared tokens and up to 500 of their own: 55 us (28 over the
// prefix, 15 over the rest, 7 to join, the rest between launches), where each by itself reads 1.1 GB from L2 in 158; four
// requests behind 131000 70 us, not 151, of which the prefix's 268 MB from DRAM take 64.  What bounds the first is latency: at most
// four key tiles of 3.4 us a CTA and the same start for every launch; the second the instructions of 16 rows.

namespace {

// Does reading prefixes once pay?  A request of kPromptMin rows and more is never taken: here the step kernel has every request's
// own part, and a prompt's would take long.  That is simple, and for some steps it is lost: without it, `prefixes` included,
// shared / each by itself, 32 heads over 8 of 128 behind 8192 shared tokens, 64 requests of 13 tokens (52 rows) 253 / 566 us, of 32
// (128 rows) 544 / 570, 63 single tokens and a chunk of 512 202 / 267; 64 of 5 tokens of 32 heads over 2 112 / 159.
// Nor does it pay where everything that the requests read (`most` bytes of codes, from L2) takes less time than the
// launches do that sharing adds.  Captured, shared / each by itself, 32 heads over 8 of 128, and 16 of 64: 4 requests of 2050
// tokens (17 MB) 15.5 / 13.7 and 14.7 / 15.0 us, 12 of 2050 (50 MB) 17.6 / 17.9 and 16.5 / 21.4, 12 of 8050 (198 MB) 26 / 38
// and 20 / 53.  With groups of kPromptMin rows and more, for which the other kernel is launched as well: 64 of 550 (72 MB)
// 38 / 22 and 37 / 28, 64 of 1000 (131 MB) 43 / 27 and 43 / 34, 32 of 2050 (134 MB) 34 / 30 and 22 / 39, 64 of 2050 (269 MB)
// 38 / 49 and 37 / 67, 200 of 8050 of 12 heads over one of 32 (103 MB) 47 / 62.
// `max_length` may be a capacity that the requests do not fill, as SharedKVCache's is; then the rule says yes too early, 32 heads
// over 8 of 128: four requests of 600 tokens in a cache for 131072 11.5 us, and 6.6 for `prefixes` once a step, by themselves 11.0; 64
// of 600 that share nothing, in one for 8192, 24.3 / 22.2, 12 of 4000 31.1 / 24.5.
bool takes_prefixes(const KvPool& pool, int group, int requests, int64_t tokens, int max_new, int max_length) {
    if (most_rows(group, tokens, max_new) >= kPromptMin) return false;
    if (max_length == 0) return true;  // unknown
    const double most = double(requests) * max_length * pool.kv_heads * pool.head_dim * 2;  // passes 64 bits
    return most >= (tokens * group >= kPromptMin ? 128e6 : 48e6);
}

struct SharedPlan {
    bool prompt;           // groups of kPromptMin rows and more may occur
    int sms, nq, step_ctas, prompt_ctas;
    int64_t where, ml, sums, step, prompt_at, bytes;  // places in the workspace
};

SharedPlan shared_plan(int head_dim, int heads, int group, int64_t tokens, int max_new, int sms) {
    SharedPlan p;
    p.sms = sms;
    p.prompt = tokens * group >= kPromptMin;
    // Rows of most row tiles: the requests' own, or, without the other kernel, also those of the groups.  16 in either case:
    // 64 requests behind 8192 tokens, 4 rows each, 63 us, not 58; 200 behind 500 82, not 69.
    p.nq = (p.prompt ? most_rows(group, tokens, max_new) : tokens * group) <= 8 ? 1 : 2;
    p.step_ctas = sms * (p.nq == 1 ? StepCfg<32, 1>::PER_SM : StepCfg<32, 2>::PER_SM);
    p.prompt_ctas = p.prompt ? sms : 0;
    int64_t at = 0;
    auto take = [&](int64_t bytes) {
        const int64_t here = at;
        at += round_up(bytes, 256);
        return here;
    };
    const int64_t rows = 2 * tokens * heads;
    p.where = take(rows * int64_t(sizeof(int2)));
    p.ml = take(rows * int64_t(sizeof(float2)));
    p.sums = take(rows * head_dim * int64_t(sizeof(float)));
    p.step = take(int64_t(p.step_ctas) * 2 * 8 * p.nq * (head_dim + 2) * int64_t(sizeof(float)));
    p.prompt_at = take(int64_t(p.prompt_ctas) * 2 * kPromptTile * (head_dim + 2) * int64_t(sizeof(float)));
    p.bytes = at;
    return p;
}

template <int D, bool BF16>
cudaError_t launch_shared(KvAttnArgs a, const SharedPlan& p, char* ws, int dev, cudaStream_t s) {
    a.where = reinterpret_cast<int2*>(ws + p.where);
    a.sums_ml = reinterpret_cast<float2*>(ws + p.ml);
    a.sums = reinterpret_cast<float*>(ws + p.sums);
    a.least_rows = 0;
    a.most_rows = INT_MAX;
    cudaError_t e = cudaSuccess;
    const int requests = a.requests;
    if (p.prompt) {
        a.least_rows = kPromptMin;
        a.requests = a.groups;  // groups only
        e = launch_kv_prompt_shared(a, BF16, ws + p.prompt_at, dev, s);
        if (e != cudaSuccess) return e;
        a.least_rows = 0;
        a.most_rows = kPromptMin - 1;
    }
    a.requests = a.groups + requests;
    e = p.nq == 1 ? launch_step<D, 1, BF16, true>(a, 0, ws + p.step, dev, s)
                  : launch_step<D, 2, BF16, true>(a, 0, ws + p.step, dev, s);
    if (e != cudaSuccess) return e;
    const int64_t grid = (a.tokens * a.heads + 3) / 4;
    if (grid > INT32_MAX) return cudaErrorInvalidValue;
    const SharedParts parts{reinterpret_cast<const float*>(ws + p.step), reinterpret_cast<const float*>(ws + p.prompt_at),
                            8 * p.nq, p.step_ctas, p.prompt_ctas};
    // Few rows have many parts each.  With 4 / 8 / 16 ways, the whole call: 128 rows of four requests behind 131000 tokens 73.0 /
    // 70.6 / 71.1 us, 256 behind 8192 20.5 / 19.6 / 19.6; 2048 rows of 64 requests 54.7 / 56.2 / 62.3, 6400 66 / 72 / 84.
    if (grid <= p.sms) return launch_early(kv_shared_join_kernel<D, BF16, 8>, dim3(unsigned(grid)), 32 * 8, 0, s, a, parts);
    return launch_early(kv_shared_join_kernel<D, BF16, 4>, dim3(unsigned(grid)), 32 * 4, 0, s, a, parts);
}

}  // namespace

bool kv_takes_prefixes(const KvPool& pool, int heads, int requests, int64_t tokens, int max_new, int max_length) {
    return takes_prefixes(pool, heads / pool.kv_heads, requests, tokens, max_new, max_length);
}

uint64_t kv_shared_workspace_bytes(const KvPool& pool, int heads, int requests, int64_t tokens, int max_new, int max_length) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return 0;
    const int group = heads / pool.kv_heads;
    if (!takes_prefixes(pool, group, requests, tokens, max_new, max_length))
        return kv_attention_workspace_bytes(pool.head_dim, group, tokens, max_new, max_length);
    return uint64_t(shared_plan(pool.head_dim, heads, group, tokens, max_new, gemm_sm_count(dev)).bytes);
}

cudaError_t launch_kv_shared_attention(KvAttnArgs a, bool bf16, int max_new, int max_length, void* ws, cudaStream_t s) {
    if (a.tokens <= 0 || a.requests <= 0) return cudaSuccess;
    if (!takes_prefixes(a.pool, a.group, a.requests, a.tokens, max_new, max_length))
        return launch_kv_attention(a, bf16, max_new, max_length, ws, s);
    int dev = 0;
    const cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const SharedPlan p = shared_plan(a.pool.head_dim, a.heads, a.group, a.tokens, max_new, gemm_sm_count(dev));
    a.groups = a.requests;
    a.whole = 0;
    char* base = static_cast<char*>(ws);
    switch (a.pool.head_dim) {
        case 32: return bf16 ? launch_shared<32, true>(a, p, base, dev, s) : launch_shared<32, false>(a, p, base, dev, s);
        case 64: return bf16 ? launch_shared<64, true>(a, p, base, dev, s) : launch_shared<64, false>(a, p, base, dev, s);
        default: return bf16 ? launch_shared<128, true>(a, p, base, dev, s) : launch_shared<128, false>(a, p, base, dev, s);
    }
}

cudaError_t read_kv_status(int* status, bool clear, cudaStream_t s) {
    int prompt = 0, copy = 0;
    cudaError_t e = read_status_word(g_kv_status, status, clear, s);
    if (e == cudaSuccess) e = read_kv_prompt_status(&prompt, clear, s);
    if (e == cudaSuccess) e = read_kv_copy_status(&copy, clear, s);
    if (*status == 0) *status = prompt != 0 ? prompt : copy;
    return e;
}

}  // namespace ebx
