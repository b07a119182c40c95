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

constexpr int kRows = 16;        // rows of a tile: the M of mma.m16n8k16
constexpr int kConsumers = 4;    // warps that compute; one more loads
constexpr int kStepThreads = 32 * (kConsumers + 1);
constexpr int kStages = 3;
template <int D>
struct StepCfg {
    static constexpr int KT = 8192 / D;              // tokens of a key tile: 8 KB of codes a side
    static constexpr int UNITS = KT / 16;            // 16 tokens lie in one block: one scale
    static constexpr int PER_WARP = UNITS / kConsumers;
    static constexpr int kStageBytes = 2 * 8192;
    static constexpr int kMergeBytes = kConsumers * kRows * (D + 4) * 4;
    static constexpr int kSmem = 1024 + kStages * kStageBytes + kMergeBytes + kStages * 2 * UNITS * 4 + 256;
};

// Byte `b` of row `r` in a tile that TMA wrote with the swizzle of a D-byte row.
template <int D>
__device__ __forceinline__ uint32_t swz(int r, int b) {
    const int x = D == 128 ? (r & 7) : D == 64 ? ((r >> 1) & 3) : ((r >> 2) & 1);
    return uint32_t(r * D + (b ^ (x << 4)));
}

// Column n of an 8-key product is key {0,5,2,7,1,4,3,6}[n] of its eight: with this order the
// loads of K rows (by n) and of V rows (by n / 2, for n even and odd) are free of bank conflicts
// under each of the three swizzles.
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

template <int D, bool BF16>
__global__ void __launch_bounds__(kStepThreads)
    kv_step_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                   const __grid_constant__ KvAttnArgs a, int least) {
    using C = StepCfg<D>;
    constexpr int KT = C::KT, UNITS = C::UNITS;
    constexpr int KB = D >= 64 ? 16 : 8;        // bytes of a K row that a lane loads at once
    constexpr int KL = D / (4 * KB);            // such loads for a row
    constexpr int KW = KB / 4;                  // words of it = products of depth 16
    constexpr int VB = D / 8;                   // bytes of a V row that a lane loads
    constexpr int NT = VB;                      // 8-wide column tiles of O
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
    const KvShare share = kv_share<kRows, KT, kStepThreads>(a, least, reinterpret_cast<int*>(smem));
    fence_proxy_async_smem();  // the ring's copies may overwrite what kv_share kept there
    if (threadIdx.x < 2) a.desc[2 * blockIdx.x + threadIdx.x] = make_int4(0, 0, 0, 0);
    __syncthreads();
    KvWalk<kRows, KT> walk;
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
        return;
    }

    // ---- consumers: warp w takes tokens [w KT/4, (w + 1) KT/4) of every key tile ----
    const int c = lane & 3, n8 = lane >> 2;
    const int krow = (n8 & 1) ? key_odd(n8 >> 1) : key_even(n8 >> 1);
    const int vrow0 = key_even(c), vrow1 = key_odd(c);
    // the D / 8 bytes of a V row that this lane's column n8 of each of the NT column tiles holds
    const int vbyte = D == 128 ? 16 * ((n8 >> 1) | ((n8 & 1) << 2))
                      : D == 64 ? 8 * (2 * ((((n8 >> 1) & 1) << 1) | (n8 >> 2)) + (n8 & 1)) : 4 * n8;
    // O: column tile t of columns 2c and 2c + 1 is dimension odim0 + t and odim1 + t
    const int odim0 = D == 128 ? 16 * c : D == 64 ? 16 * (((c & 1) << 1) | (c >> 1)) : 8 * c;
    const int odim1 = D == 128 ? odim0 + 64 : odim0 + VB;
    int it = 0;
    bool ok = true;
    for (; !walk.done(); walk.next(a)) {
        // q: rows n8 and n8 + 8, this lane's 4 KL KW products of depth 16
        uint32_t qa[KL * KW][4];
        float unit[2] = {1.0f, 1.0f};  // what q was divided by
        int lo[2], hi[2];              // the row sees keys [lo, hi); a row past the last is not kept
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int r = walk.rt * kRows + n8 + 8 * half;
            const bool in = r < walk.r.rows;
            const int token = in ? by_group(a, r) : 0;
            const int place = walk.r.begin + token;
            hi[half] = !in ? INT_MAX : a.causal ? min(place + 1, walk.r.length) : walk.r.length;
            lo[half] = !in ? 0 : max(walk.r.first, a.window > 0 ? place - a.window + 1 : 0);
            const uint16_t* src = a.q.p + (walk.r.token0 + token) * a.q.token_stride +
                                  (walk.head * a.group + (in ? r - token * a.group : 0)) * a.q.head_stride + c * KB;
#pragma unroll
            for (int l = 0; l < KL; ++l)
#pragma unroll
                for (int q = 0; q < KW; q += 2) {
                    uint4 v = make_uint4(0, 0, 0, 0);
                    if (in) v = __ldg(reinterpret_cast<const uint4*>(src + l * 4 * KB + q * 4));
                    qa[l * KW + q][half] = v.x;
                    qa[l * KW + q][half + 2] = v.y;
                    qa[l * KW + q + 1][half] = v.z;
                    qa[l * KW + q + 1][half + 2] = v.w;
                }
        }
        if constexpr (BF16) {
            // fp16 operands: each row over the power of two at its largest element, so that every
            // element of at least 2^-14 of it is exact and the others are off by 2^-25 of it
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                uint32_t top = 0;
#pragma unroll
                for (int i = 0; i < KL * KW; ++i)
                    top = __vmaxu2(top, __vmaxu2(qa[i][half] & 0x7fff7fffu, qa[i][half + 2] & 0x7fff7fffu));
                top = max(top & 0xffffu, top >> 16);
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const uint32_t e = min(max(top >> 7, 1u), 253u);  // 2^(e - 127)
                const float down = __uint_as_float((254u - e) << 23);
                unit[half] = __uint_as_float(e << 23);
#pragma unroll
                for (int i = 0; i < KL * KW; ++i)
#pragma unroll
                    for (int q = half; q < 4; q += 2) {
                        const uint32_t v = qa[i][q];
                        qa[i][q] = pack_half2(__uint_as_float(v << 16) * down,
                                              __uint_as_float(v & 0xffff0000u) * down);
                    }
            }
        }
        float o[NT][4];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[t][i] = 0.0f;
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
        // the keys that every row of the tile sees
        const int all_lo = __reduce_max_sync(0xffffffffu, max(lo[0], lo[1]));
        const int all_hi = __reduce_min_sync(0xffffffffu, min(hi[0], hi[1]));

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
                float s[2][4];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[h][i] = 0.0f;
                    const int r = u * 16 + h * 8 + krow;
#pragma unroll
                    for (int x = 0; x < KL; ++x) {
                        uint32_t w[KW];
                        lds<KB>(kbase + swz<D>(r, x * 4 * KB + c * KB), w);
#pragma unroll
                        for (int q = 0; q < KW; ++q) {
                            const uint32_t v = w[q] ^ 0x80808080u;
                            mma_16816(s[h], qa[x * KW + q], codes_to_half2(v, 0x4140), codes_to_half2(v, 0x4342));
                        }
                    }
                }
                const bool none = vs < 0.0f;  // kKvNone
                const float vsc = vs < 0x1p-100f ? 0x1p-100f : vs;  // NaN stays
                const float b = none ? -INFINITY : lg2(vsc);
                const float inv = vs == vs ? 1.0f / vsc : 1.0f;  // NaN goes through t, where the mask stops it
                const float cs = none ? 0.0f : ks * a.scale_log2;
                const bool edge = key0 < all_lo || key0 + 16 > all_hi;
                float top[2];
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const float cf = cs * unit[half];
                    top[half] = -INFINITY;
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            float& t = s[h][2 * half + i];
                            t = fmaf(t, cf, b);
                            if (edge) {
                                const int key = key0 + h * 8 + (i ? vrow1 : vrow0);
                                if (key < lo[half] || key >= hi[half]) t = -INFINITY;
                            }
                            top[half] = fmaxf(top[half], t);
                        }
                    top[half] = fmaxf(top[half], __shfl_xor_sync(0xffffffffu, top[half], 1));
                    top[half] = fmaxf(top[half], __shfl_xor_sync(0xffffffffu, top[half], 2));
                }
                // the running maximum moves only when it grew by more than 2^kLag, so that most
                // tiles rescale nothing
                if (__any_sync(0xffffffffu, top[0] > m[0] + kLag || top[1] > m[1] + kLag)) {
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const float mn = fmaxf(m[half], top[half]);
                        const float f = mn == m[half] ? 1.0f : ex2(m[half] - mn);
                        m[half] = mn;
                        l[half] *= f;
#pragma unroll
                        for (int t = 0; t < NT; ++t) {
                            o[t][2 * half] *= f;
                            o[t][2 * half + 1] *= f;
                        }
                    }
                }
                uint32_t p[4];
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const float mr = m[half] == -INFINITY ? 0.0f : m[half] - kShift;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float w0 = ex2(s[h][2 * half] - mr), w1 = ex2(s[h][2 * half + 1] - mr);
                        l[half] = fmaf(w0 + w1, inv, l[half]);
                        p[2 * h + half] = pack_half2(w0, w1);  // 11 bits, as the codes' operands need
                    }
                }
                uint32_t v00[VB / 4], v01[VB / 4], v10[VB / 4], v11[VB / 4];
                lds<VB>(vbase + swz<D>(u * 16 + vrow0, vbyte), v00);
                lds<VB>(vbase + swz<D>(u * 16 + vrow1, vbyte), v01);
                lds<VB>(vbase + swz<D>(u * 16 + 8 + vrow0, vbyte), v10);
                lds<VB>(vbase + swz<D>(u * 16 + 8 + vrow1, vbyte), v11);
#pragma unroll
                for (int q = 0; q < VB / 4; ++q) {
#pragma unroll
                    for (int y = 0; y < 2; ++y) {  // dimensions 4q + 2y and 4q + 2y + 1
                        const uint32_t sel = y ? 0x7362 : 0x5140;  // {even key, odd key} of each
                        const uint32_t x0 = __byte_perm(v00[q], v01[q], sel) ^ 0x80808080u;
                        const uint32_t x1 = __byte_perm(v10[q], v11[q], sel) ^ 0x80808080u;
                        mma_16816(o[4 * q + 2 * y], p, codes_to_half2(x0, 0x4140), codes_to_half2(x1, 0x4140));
                        mma_16816(o[4 * q + 2 * y + 1], p, codes_to_half2(x0, 0x4342), codes_to_half2(x1, 0x4342));
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&empty[st]));
        }

        // ---- the four warps' results become one ----
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            l[half] += __shfl_xor_sync(0xffffffffu, l[half], 1);
            l[half] += __shfl_xor_sync(0xffffffffu, l[half], 2);
        }
        const int rows = min(kRows, walk.r.rows - walk.rt * kRows);
        float* mine = merge + warp * kRows * (D + 4);  // row: D values, m, l
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int r = n8 + 8 * half;
            if (r < rows) {
                float* dst = mine + r * (D + 4);
#pragma unroll
                for (int t = 0; t < NT; t += 4) {
                    *reinterpret_cast<float4*>(dst + odim0 + t) =
                        make_float4(o[t][2 * half], o[t + 1][2 * half], o[t + 2][2 * half], o[t + 3][2 * half]);
                    *reinterpret_cast<float4*>(dst + odim1 + t) =
                        make_float4(o[t][2 * half + 1], o[t + 1][2 * half + 1], o[t + 2][2 * half + 1],
                                    o[t + 3][2 * half + 1]);
                }
                if (c == 0) {
                    dst[D] = m[half] - kShift;
                    dst[D + 1] = l[half];
                }
            }
        }
        asm volatile("bar.sync 1, %0;" ::"n"(32 * kConsumers) : "memory");
        const bool whole = walk.begins && walk.ends;
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
        if (!whole && threadIdx.x == 0)
            a.desc[2 * blockIdx.x + slot] = kv_desc(walk.r, walk.rt, kRows, walk.head, walk.ends);
        asm volatile("bar.sync 1, %0;" ::"n"(32 * kConsumers) : "memory");  // merge is free again
    }
}

constexpr int kStepPerSm = 2;   // CTAs of an SM
constexpr int kStepLeast = 4;   // key tiles a CTA takes at least: a partial result costs about as much

template <int D, bool BF16>
cudaError_t launch_step(KvAttnArgs a, void* ws, int dev, cudaStream_t s) {
    using C = StepCfg<D>;
    auto kern = kv_step_kernel<D, BF16>;
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
    const int grid = gemm_sm_count(dev) * kStepPerSm;
    a.desc = static_cast<int4*>(ws);
    a.part = reinterpret_cast<float*>(a.desc + 2 * grid);
    kern<<<grid, kStepThreads, C::kSmem, s>>>(mk, mv, a, kStepLeast);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    return launch_join<D, kRows, BF16>(a, grid, std::min(kRows, a.group), s);
}

}  // namespace

namespace {

// Row tiles of 256 rows on tcgen05 from kPromptMin rows of a request on; below, tiles of 16.
constexpr int kPromptMin = 33;

bool takes_prompt(int group, int64_t tokens, int max_new) {
    const int64_t most = max_new > 0 ? std::min<int64_t>(max_new, tokens) : tokens;
    return most * group >= kPromptMin;
}

}  // namespace

uint64_t kv_attention_workspace_bytes(int head_dim, int group, int64_t tokens, int max_new) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return 0;
    const int sms = gemm_sm_count(dev);
    if (takes_prompt(group, tokens, max_new)) return kv_prompt_workspace_bytes(head_dim, sms);
    return uint64_t(round_up(int64_t(sms) * kStepPerSm * 2 * int64_t(sizeof(int4) + kRows * (head_dim + 2) * sizeof(float)), 256));
}

cudaError_t launch_kv_attention(const KvAttnArgs& a, bool bf16, int max_new, void* ws, cudaStream_t s) {
    if (a.tokens <= 0 || a.requests <= 0) return cudaSuccess;
    int dev = 0;
    const cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (takes_prompt(a.group, a.tokens, max_new)) return launch_kv_prompt(a, bf16, ws, dev, s);
    switch (a.pool.head_dim) {
        case 32: return bf16 ? launch_step<32, true>(a, ws, dev, s) : launch_step<32, false>(a, ws, dev, s);
        case 64: return bf16 ? launch_step<64, true>(a, ws, dev, s) : launch_step<64, false>(a, ws, dev, s);
        default: return bf16 ? launch_step<128, true>(a, ws, dev, s) : launch_step<128, false>(a, ws, dev, s);
    }
}

cudaError_t read_kv_status(int* status, bool clear, cudaStream_t s) {
    int prompt = 0;
    cudaError_t e = read_status_word(g_kv_status, status, clear, s);
    if (e == cudaSuccess) e = read_kv_prompt_status(&prompt, clear, s);
    if (*status == 0) *status = prompt;
    return e;
}

}  // namespace ebx
