// ebx_kv_share.cu -- requests that share cache blocks: fork (and free, and roll back), compact, copying blocks,
// and finding the prefixes that requests share.  No reference counterpart.
//
// The bookkeeping kernels (fork, compact, prefixes) are one cluster of CTAs each: their phases need what all
// rows or all blocks gave in the phase before, and a cluster's barrier costs a fraction of a launch.  That is for tables of
// up to a few hundred kilobytes; a larger one is still read and written by eight SMs (fork, all rows staying: 128 rows of 64
// blocks 8 us, 1024 of 256 16 us, 1024 of 2048, 8 MB, 68 us, 8192 of 1024 444 us).  Counts are changed by atomic additions only, whose order does not change
// them, and whatever is given an order (blocks to the ring, copies) gets it from sums over rows or ids.
//
// Each kernel lets the next one begin only after its own wait: kernels that begin while two others still run hold
// places that the copies lack (690 blocks compacted in 2 layers, one call after the other, 91 us in place of 77).
#include <algorithm>
#include <atomic>
#include <climits>

#include <cooperative_groups.h>

#include "ebx_common.cuh"
#include "ebx_kv_share.h"

namespace ebx {
namespace {

namespace cg = cooperative_groups;

constexpr int kCluster = 8;
constexpr int kShareThreads = 1024;

// Exclusive sum over the block; `total` receives the whole.
__device__ __forceinline__ int block_sum(int v, int* warp_sums, int& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int x = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, x, d);
        if (lane >= d) x += u;
    }
    __syncthreads();  // the previous call's sums have been read
    if (lane == 31) warp_sums[warp] = x;
    __syncthreads();
    const int y = warp_sums[lane];
    int z = y;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, z, d);
        if (lane >= d) z += u;
    }
    total = __shfl_sync(0xffffffffu, z, 31);
    return x - v + __shfl_sync(0xffffffffu, z - y, warp);
}

// Tells every CTA of the cluster this CTA's number; after it each has all of them in `all`.
__device__ __forceinline__ void tell(cg::cluster_group& cluster, int* all, int mine) {
    if (threadIdx.x < kCluster) cluster.map_shared_rank(all, threadIdx.x)[cluster.block_rank()] = mine;
    cluster.sync();
}

// ---- fork ---------------------------------------------------------------------------------

struct ForkRow {
    int parent;   // -1: none
    int had, keep;
    bool changed, begun;
};

__device__ __forceinline__ int fork_length(const KvForkArgs& a, int r) {
    const int64_t cap = int64_t(a.width) << a.shift;
    return int(min(int64_t(max(a.lengths[r], 0)), cap));
}
__device__ __forceinline__ ForkRow fork_row(const KvForkArgs& a, int r) {
    ForkRow f;
    const int p = a.parents[r];
    f.parent = p >= 0 && p < a.requests ? p : -1;
    f.had = fork_length(a, r);
    f.keep = f.parent < 0 ? 0 : f.parent == r ? f.had : fork_length(a, f.parent);
    if (a.keep) f.keep = min(f.keep, max(a.keep[r], 0));
    f.changed = f.parent != r || f.keep != f.had;
    f.begun = f.changed && (f.keep & ((1 << a.shift) - 1)) != 0;
    return f;
}

// Row r goes on from the first keep[r] tokens of what row parents[r] held.  Of every block the holders are
// counted: rows that change give up what they held and take hold of the full blocks that they keep.  A
// block that is begun can be one row's only, which will write to it: where no row holds it whole, the first
// that wants it keeps it, the parent itself ahead of others; every other row gets a copy in a block
// from the ring's front, in row order, or, when there are none left, nothing at all.  Blocks that nobody holds then go
// to the ring's back in the order of their numbers.
// What bounds it is latency: 16 or 128 rows 9.5 us, 11 from cold caches, a launch and four barriers of the cluster
// (and one more where blocks are missing) with two or three dependent reads between each.
__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(kShareThreads, 1) kv_fork_kernel(const __grid_constant__ KvForkArgs a) {
    asm volatile("griddepcontrol.wait;\n\tgriddepcontrol.launch_dependents;" ::: "memory");
    cg::cluster_group cluster = cg::this_cluster();
    __shared__ int warp_sums[32];
    __shared__ int counts[kCluster];
    __shared__ int s_missing;
    const int tid = threadIdx.x, lane = tid & 31, rank = int(cluster.block_rank());
    const int gtid = rank * kShareThreads + tid, gwarp = gtid >> 5;
    constexpr int kAll = kCluster * kShareThreads, kAllWarps = kAll / 32;
    const int64_t begin = max(a.ring[0], int64_t(0));
    const int64_t avail = min(max(a.ring[1], begin) - begin, int64_t(a.free_size));  // blocks to give
    const int64_t room = a.free_size - avail;                                        // places for freed ones
    const int64_t head = begin >> 62 ? begin % a.free_size : begin, tail = head + avail;
    const int front = int(head % a.free_size), back = int(tail % a.free_size);
    auto wrapped = [&](int64_t place) { return place < a.free_size ? place : place - a.free_size; };
    auto block = [&](int id) { return id >= 0 && id < a.blocks; };
    if (tid == 0) s_missing = 0;

    for (int b = gtid; b < a.blocks; b += kAll) a.out_shares[b] = a.shares[b];
    for (int r = gtid; r < a.requests; r += kAll) a.sources[r] = a.targets[r] = -1;
    auto tail_of = [&](const ForkRow& f) { return a.tables[int64_t(f.parent) * a.width + (f.keep >> a.shift)]; };
    ForkRow mine{};  // the row of this thread below
    int my_tail = -1;
    if (rank == 0 && tid < a.requests) {
        mine = fork_row(a, tid);
        if (mine.begun) my_tail = tail_of(mine);
    }
    cluster.sync();

    for (int r = gwarp; r < a.requests; r += kAllWarps) {
        const ForkRow f = fork_row(a, r);
        const int mask = (1 << a.shift) - 1;
        const int had = (f.had >> a.shift) + ((f.had & mask) != 0), full = f.keep >> a.shift, held = full + ((f.keep & mask) != 0);
        const int32_t* old = a.tables + int64_t(r) * a.width;
        const int32_t* from = a.tables + int64_t(max(f.parent, 0)) * a.width;
        int32_t* to = a.out_tables + int64_t(r) * a.width;
        const int same = f.parent == r ? full : 0;  // blocks that the row neither gives up nor takes
        for (int j = lane; j < a.width; j += 32) {
            const int id = j < held ? from[j] : -1;
            to[j] = id;
            if (!f.changed || j < same) continue;
            if (j < had) {
                const int gone = old[j];
                if (block(gone)) atomicSub(a.out_shares + gone, 1);
            }
            if (j < full && block(id)) atomicAdd(a.out_shares + id, 1);
        }
        if (lane == 0) a.out_lengths[r] = f.keep;
    }
    cluster.sync();

    // Begun blocks, by the cluster's first CTA, a thread to a row.  Who keeps one that no row holds whole: its count, -1,
    // becomes the lowest of the rows' claims.
    if (rank == 0) {
        auto claim_of = [&](const ForkRow& f, int r) { return INT_MIN + (f.parent == r ? r : r + a.requests); };
        auto each_row = [&](auto go) {  // the first kShareThreads rows are known already
            for (int base = 0; base < a.requests; base += kShareThreads) {
                const int r = base + tid;
                ForkRow f = mine;
                int id = my_tail;
                if (base > 0) {
                    f.begun = false;
                    id = -1;
                    if (r < a.requests) f = fork_row(a, r);
                    if (f.begun) id = tail_of(f);
                }
                go(r, f, id);
            }
        };
        each_row([&](int r, const ForkRow& f, int id) {
            if (f.begun && block(id) && __ldcg(a.out_shares + id) < 0) atomicMin(a.out_shares + id, claim_of(f, r));
        });
        __syncthreads();
        int64_t taken = 0;
        each_row([&](int r, const ForkRow& f, int id) {
            bool need = f.begun && block(id);
            if (need && __ldcg(a.out_shares + id) == claim_of(f, r)) {  // no other row has that claim
                a.out_shares[id] = 0;
                need = false;
            }
            int total;
            const int64_t before = taken + block_sum(need, warp_sums, total);
            if (need) {
                if (before < avail) {
                    const int fresh = a.free_ring[wrapped(front + before)];
                    a.out_tables[int64_t(r) * a.width + (f.keep >> a.shift)] = fresh;
                    a.sources[before] = id;
                    a.targets[before] = fresh;
                } else {
                    a.out_lengths[r] = 0;
                    atomicAdd(&s_missing, 1);
                }
            }
            taken += total;
        });
        __syncthreads();
        if (tid == 0) {
            taken = min(taken, avail);
            a.ring_out[0] = head + taken;
            a.ring_out[2] = s_missing;
            a.ring_out[3] = taken;
        }
    }
    cluster.sync();

    if (*const_cast<volatile int64_t*>(a.ring_out + 2) != 0) {  // rows that got nothing let go of what they took
        for (int r = gwarp; r < a.requests; r += kAllWarps) {
            const ForkRow f = fork_row(a, r);
            if (!f.begun || a.out_lengths[r] != 0) continue;
            const int full = f.keep >> a.shift;
            int32_t* to = a.out_tables + int64_t(r) * a.width;
            for (int j = lane; j <= full; j += 32) {
                const int id = to[j];
                if (j < full && block(id)) atomicSub(a.out_shares + id, 1);
                to[j] = -1;
            }
        }
        cluster.sync();
    }

    // a part of the blocks each: count those that nobody holds, then write them behind those of the parts before
    const int per = int((int64_t(a.blocks) + kCluster - 1) / kCluster);
    const int b0 = min(rank * int64_t(per), int64_t(a.blocks)), b1 = min(b0 + int64_t(per), int64_t(a.blocks));
    int gone_here = 0, total;
    for (int b = b0 + tid; b < b1; b += kShareThreads) gone_here += a.out_shares[b] < 0;
    block_sum(gone_here, warp_sums, total);
    tell(cluster, counts, total);
    int64_t at = 0, all = 0;
    for (int c = 0; c < kCluster; ++c) {
        if (c < rank) at += counts[c];
        all += counts[c];
    }
    if (total > 0) {
        for (int base = b0; base < b1; base += kShareThreads) {
            const int b = base + tid;
            const bool gone = b < b1 && a.out_shares[b] < 0;
            const int64_t place = at + block_sum(gone, warp_sums, total);
            if (gone) {
                a.out_shares[b] = 0;
                if (place < room) a.free_ring[wrapped(back + place)] = b;
            }
            at += total;
        }
    }
    if (gtid == 0) a.ring_out[1] = tail + min(all, room);
}

// ---- compact ------------------------------------------------------------------------------

// With H blocks held, those whose number is H or more move into the free ones below H, the first into the
// first and so on: the fewest moves there can be, and no block is read and written.  Every CTA marks a part of the
// rows' blocks in a bitmap of its own, puts the cluster's together and counts the bits ahead of each word; the rank of a
// bit and the place of the k-th free number below H then answer everything without a list.  2900 blocks 8.8 us from cold
// caches, and 5.7 us for a small cache's, both latency; with lists in global memory and six barriers 13.3 and 9.7.
__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(kShareThreads, 1) kv_compact_kernel(const __grid_constant__ KvCompactArgs a) {
    asm volatile("griddepcontrol.wait;\n\tgriddepcontrol.launch_dependents;" ::: "memory");
    cg::cluster_group cluster = cg::this_cluster();
    extern __shared__ uint32_t bits[];     // [words]: this CTA's rows
    __shared__ int warp_sums[32];
    const int words = (a.blocks + 31) / 32;
    uint32_t* held_bits = bits + words;                            // [words]: all rows
    int* before = reinterpret_cast<int*>(held_bits + words);       // [words]: bits ahead of a word
    const int tid = threadIdx.x, lane = tid & 31, rank = int(cluster.block_rank());
    const int gtid = rank * kShareThreads + tid, gwarp = gtid >> 5;
    constexpr int kAll = kCluster * kShareThreads, kAllWarps = kAll / 32;
    auto block = [&](int id) { return id >= 0 && id < a.blocks; };
    auto held_by = [&](int r) {
        const int64_t n = (int64_t(max(a.lengths[r], 0)) + (1 << a.shift) - 1) >> a.shift;
        return int(min(n, int64_t(a.width)));
    };
    for (int w = tid; w < words; w += kShareThreads) bits[w] = 0;
    __syncthreads();
    for (int r = gwarp; r < a.requests; r += kAllWarps) {
        const int n = held_by(r);
        for (int j = lane; j < n; j += 32) {
            const int id = a.tables[int64_t(r) * a.width + j];
            if (block(id)) atomicOr(bits + (id >> 5), 1u << (id & 31));
        }
    }
    cluster.sync();
    int held = 0;
    for (int w0 = 0; w0 < words; w0 += kShareThreads) {
        const int w = w0 + tid;
        uint32_t x = 0;
        if (w < words)
            for (int c = 0; c < kCluster; ++c) x |= cluster.map_shared_rank(bits, c)[w];
        int total;
        const int ahead = block_sum(__popc(x), warp_sums, total);
        if (w < words) {
            held_bits[w] = x;
            before[w] = held + ahead;
        }
        held += total;
    }
    cluster.sync();  // also: nobody leaves while its bits are read
    auto is_held = [&](int id) { return (held_bits[id >> 5] >> (id & 31) & 1) != 0; };
    auto rank_of = [&](int id) {  // held blocks ahead of block id <= blocks
        return (id >> 5) < words ? before[id >> 5] + __popc(held_bits[id >> 5] & ((1u << (id & 31)) - 1)) : held;
    };
    const int low = rank_of(held), moves = held - low;  // held ones below H stay
    auto free_below = [&](int k) {  // the k-th number that is not held
        int lo = 0, hi = words;     // the last word with at most k of them ahead
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (32 * mid - before[mid] <= k) lo = mid; else hi = mid;
        }
        uint32_t x = ~held_bits[lo];
        int left = k - (32 * lo - before[lo]), at = 0;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) {
            const int n = __popc(x & ((1u << d) - 1));
            if (left >= n) {
                left -= n;
                at += d;
                x >>= d;
            }
        }
        return 32 * lo + at;
    };
    auto moved = [&](int id) { return id < held ? id : free_below(rank_of(id) - low); };
    for (int at = gwarp; at < a.requests; at += kAllWarps) {
        const int n = held_by(at);
        for (int j = lane; j < a.width; j += 32) {
            const int id = j < n ? a.tables[int64_t(at) * a.width + j] : -1;
            a.out_tables[int64_t(at) * a.width + j] = block(id) ? moved(id) : -1;
        }
    }
    for (int b = gtid; b < a.blocks; b += kAll) {
        if (is_held(b)) {
            const int to = moved(b);
            a.out_shares[to] = a.shares[b];
            if (b >= held) {
                a.sources[rank_of(b) - low] = b;
                a.targets[rank_of(b) - low] = to;
            }
        }
        if (b >= held) a.out_shares[b] = 0;
        a.free_out[b] = b < a.blocks - held ? held + b : -1;
    }
    for (int j = moves + gtid; j < a.blocks / 2; j += kAll) a.sources[j] = a.targets[j] = -1;
    if (gtid == 0) {
        a.ring_out[0] = 0;
        a.ring_out[1] = a.blocks - held;
        a.ring_out[2] = 0;
        a.ring_out[3] = moves;
    }
}

// ---- copy ---------------------------------------------------------------------------------

constexpr int kCopyThreads = 128;     // a warp for the codes, the others for scales
constexpr int kCopySegment = 4096;    // bytes of a unit
// Stages x segment x CTAs of an SM, for the two cases below and 1 KB blocks of 3 layers: 8 x 4 KB x 6 69.9, 93.1, 3.0 us;
// 8 x 8 KB x 3 69.8, 93.1, 3.7; 4 x 16 KB x 3 74.9, 99.1, 3.7; 4 x 4 KB x 8 77.9, 114.7, 2.9; 6 x 32 KB x 1 72.6, 98.9, 7.3.
constexpr int kCopyStages = 8;
constexpr int kCopyCtas = 6;          // of an SM

__device__ int g_kv_copy_status = 0;

__device__ __forceinline__ bool copy_wait(uint32_t bar, uint32_t parity) {
    if (mbar_wait_bounded(bar, parity)) return true;
    atomicExch(&g_kv_copy_status, 0x7106);
    return false;
}

// Unit: a segment of one side of one pair of blocks in one layer.  One thread sends a CTA's units through a ring of
// shared memory by bulk copies, which need no registers on the way.  What bounds it is DRAM: 223 MB read and written in 70 us =
// 6.4 TB/s, 0.98 of a copy's rate; 124 copies of 4 blocks (520 MB written, the sources from L2) 93 us = 5.6 TB/s of
// writes.  Loads and stores of 16 bytes a thread, 64 KB an SM on their way, 86 and 115 us.
__global__ void __launch_bounds__(kCopyThreads) kv_copy_kernel(const __grid_constant__ KvCopyArgs a) {
    extern __shared__ __align__(128) uint8_t copy_smem[];
    __shared__ uint64_t full[kCopyStages];
    __shared__ int8_t* s_to[kCopyStages];
    __shared__ uint32_t s_bytes[kCopyStages];
    if (threadIdx.x == 0) {
        for (int i = 0; i < kCopyStages; ++i) mbar_init(smem_u32(&full[i]), 1);
        fence_proxy_async_smem();
    }
    asm volatile("griddepcontrol.wait;\n\tgriddepcontrol.launch_dependents;" ::: "memory");
    const int64_t pairs = a.count ? min(max(*a.count, int64_t(0)), int64_t(a.n)) : a.n;
    auto block = [&](int id) { return id >= 0 && id < a.blocks; };
    if (threadIdx.x >= 32) {
        const int64_t all = pairs * a.layers * 2 * a.kv_heads, step = int64_t(gridDim.x) * (kCopyThreads - 32);
        for (int64_t x = int64_t(blockIdx.x) * (kCopyThreads - 32) + threadIdx.x - 32; x < all; x += step) {
            const int64_t cell = x / a.kv_heads, h = x - cell * a.kv_heads, unit = cell >> 1, pair = unit / a.layers;
            const int from = a.sources[pair], to = a.targets[pair];
            if (!block(from) || !block(to)) continue;
            float* scales = a.layer[int(unit - pair * a.layers)].scales[cell & 1];
            scales[int64_t(to) * a.kv_heads + h] = scales[int64_t(from) * a.kv_heads + h];
        }
        return;
    }
    if (threadIdx.x != 0) return;
    const int segments = int((a.bytes + kCopySegment - 1) / kCopySegment);
    const int64_t units = pairs * a.layers * 2 * segments;
    int64_t u = blockIdx.x;
    const int8_t* src = nullptr;
    int8_t* dst = nullptr;
    uint32_t bytes = 0;
    auto next = [&]() {  // the CTA's next unit that there is
        for (; u < units; u += gridDim.x) {
            const int64_t cell = u / segments, unit = cell >> 1, pair = unit / a.layers;
            const int from = a.sources[pair], to = a.targets[pair];
            if (!block(from) || !block(to) || from == to) continue;
            const int64_t at = (u - cell * segments) * kCopySegment;
            int8_t* codes = a.layer[int(unit - pair * a.layers)].codes[cell & 1];
            src = codes + from * a.bytes + at;
            dst = codes + to * a.bytes + at;
            bytes = uint32_t(min(a.bytes - at, int64_t(kCopySegment)));
            u += gridDim.x;
            return true;
        }
        return false;
    };
    bool more = next(), ok = true;
    int sent = 0, stored = 0;  // units on their way here, and from here
    for (;;) {
        while (more && sent < stored + kCopyStages - 1) {
            const int st = sent % kCopyStages;
            // the stage's unit before, sent - kCopyStages <= stored - 2, has left: all but the last store have read theirs
            if (sent >= kCopyStages) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
            const uint32_t bar = smem_u32(&full[st]);
            mbar_expect_tx(bar, bytes);
            bulk_g2s(smem_u32(copy_smem + st * kCopySegment), src, bytes, bar);
            s_to[st] = dst;
            s_bytes[st] = bytes;
            ++sent;
            more = next();
        }
        if (stored == sent) break;
        const int st = stored % kCopyStages;
        ok = copy_wait(smem_u32(&full[st]), uint32_t((stored / kCopyStages) & 1));
        if (!ok) break;
        asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;\n\tcp.async.bulk.commit_group;" ::"l"(s_to[st]),
                     "r"(smem_u32(copy_smem + st * kCopySegment)), "r"(s_bytes[st]) : "memory");
        ++stored;
    }
    if (!ok)  // given up: what is on its way lands before this shared memory is another CTA's
        for (; stored < sent; ++stored) copy_wait(smem_u32(&full[stored % kCopyStages]), uint32_t((stored / kCopyStages) & 1));
    asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
}

// ---- prefixes -----------------------------------------------------------------------------

constexpr int kPrefixThreads = 512;
constexpr int kPrefixColumns = 128;   // entries that a warp compares at a time
constexpr int kPrefixFew = 8;         // tokens of a request that a thread writes
// Dynamic shared memory that needs no leave: 48 KB hold the kernel's static shared memory as well.
constexpr size_t kPrefixPlainSmem = 40 * 1024;

// Ascending, in place; `size` a power of two, 64 at least.  Called by all threads of the block.  Exchanges over less than 64
// places are a warp's own, two keys a lane, without barriers: of 64 keys all 21.
__device__ __forceinline__ void sort(uint64_t* keys, int size) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    // the exchanges over 32 and fewer places of the steps k0 .. k1
    auto within = [&](int k0, int k1) {
        for (int base = warp * 64; base < size; base += kPrefixThreads / 32 * 64) {
            uint64_t x = keys[base + lane], y = keys[base + 32 + lane];
            for (int k = k0; k <= k1; k <<= 1) {
                const bool up_x = ((base + lane) & k) == 0, up_y = ((base + 32 + lane) & k) == 0;
                if (k >= 64 && (x > y) == up_x) {
                    const uint64_t z = x;
                    x = y;
                    y = z;
                }
                for (int j = min(k >> 1, 16); j > 0; j >>= 1) {
                    const uint64_t ox = __shfl_xor_sync(0xffffffffu, x, j), oy = __shfl_xor_sync(0xffffffffu, y, j);
                    const bool low = (lane & j) == 0;
                    x = (low == up_x) == (x < ox) ? x : ox;
                    y = (low == up_y) == (y < oy) ? y : oy;
                }
            }
            keys[base + lane] = x;
            keys[base + 32 + lane] = y;
        }
    };
    __syncthreads();
    within(2, 64);
    for (int k = 128; k <= size; k <<= 1) {
        for (int j = k >> 1; j >= 64; j >>= 1) {
            __syncthreads();
            for (int t = threadIdx.x; t < size / 2; t += kPrefixThreads) {
                const int i = 2 * t - (t & (j - 1)), o = i + j;
                const uint64_t x = keys[i], y = keys[o];
                if ((x > y) == ((i & k) == 0)) {
                    keys[i] = y;
                    keys[o] = x;
                }
            }
        }
        __syncthreads();
        within(k, k);
    }
    __syncthreads();
}

// Requests that bring tokens and whose tables begin with the same block are compared with the first of
// them: common[i] full blocks ahead of the new tokens are the same.  Of the lengths that occur, the one that
// saves most reading, (members with at least that much in common - 1) * length, becomes the group's.
//
// Every CTA sorts the requests by their first blocks, so that each knows everyone's leader; the comparisons are shared
// out among the cluster, and minima kept in the first CTA, which then sorts by leader and length: a request's place among
// its leader's is one less than the members that its length would have.  What bounds it is latency: 4 requests 6.3 us, 64
// of 137 blocks 8.5, 4 of 2053 blocks 6.5 (a warp to a row 29), 200 of 13 10.1 (12.1 with a warp to the tokens of each
// request and an addition for each member).
__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(kPrefixThreads, 1)
    kv_prefixes_kernel(const __grid_constant__ KvPrefixArgs a) {
    cg::cluster_group cluster = cg::this_cluster();
    extern __shared__ __align__(16) uint8_t prefix_smem[];
    __shared__ int warp_sums[32];
    const int n = a.requests, size = a.size;
    uint64_t* keys = reinterpret_cast<uint64_t*>(prefix_smem);                            // [size]
    unsigned long long* best = reinterpret_cast<unsigned long long*>(keys + size);  // [n]: saved << 13 | place; before that
    int* full = reinterpret_cast<int*>(best);  // [n]: a request's full blocks ahead of its new tokens
    int* leader = full + n;                    // [n]
    int* common = leader + n;                  // [n], then of a place: its leader's first place, its tokens' in the list
    int* tokens = common + n;                  // [n], of a group
    int* first_token = tokens + n;             // [n]
    __shared__ int past_last, s_largest, s_many;  // first_token[n]; tokens of the largest group; a request with many
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rank = int(cluster.block_rank());
    constexpr int kWarps = kPrefixThreads / 32;
    if (tid < 32) warp_sums[tid] = 0;
    if (tid == 0) s_largest = s_many = 0;
    for (int i = tid; i < n; i += kPrefixThreads) common[i] = INT_MAX;
    asm volatile("barrier.cluster.arrive.release;" ::: "memory");  // waited for ahead of the first minimum
    asm volatile("griddepcontrol.wait;\n\tgriddepcontrol.launch_dependents;" ::: "memory");
    auto start_of = [&](int i) { return int(min(max(int64_t(a.starts[i]), int64_t(0)), a.tokens)); };
    auto brings = [&](int i) { return max((i + 1 < n ? first_token[i + 1] : past_last) - first_token[i], 0); };

    // keys: block << 13 | request; behind them those that share nothing, and none at all
    constexpr uint64_t kAlone = uint64_t(1) << 44, kNone = ~uint64_t(0);
    for (int i = tid; i < size; i += kPrefixThreads) {
        uint64_t key = kNone;
        if (i < n) {
            const int64_t cap = int64_t(a.width) << a.shift;
            const int begin = start_of(i), end = start_of(i + 1), count = max(end - begin, 0);
            first_token[i] = begin;
            if (i + 1 == n) past_last = end;
            const int64_t past = min(int64_t(max(a.lengths[i], 0)), cap) - count;
            full[i] = past > 0 && count > 0 ? int(past >> a.shift) : 0;
            const int id = full[i] > 0 ? a.tables[int64_t(i) * a.width] : -1;
            key = (id >= 0 && id < a.blocks ? uint64_t(id) << 13 : kAlone) | uint64_t(i);
        }
        keys[i] = key;
    }
    sort(keys, size);
    // the first place in [0, p] whose key begins like that of place p
    auto begins = [&](int p, int shift) {
        int lo = -1, hi = p;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (keys[mid] >> shift == keys[p] >> shift) hi = mid; else lo = mid;
        }
        return hi;
    };
    for (int p = tid; p < n; p += kPrefixThreads)
        if (keys[p] < kAlone) leader[keys[p] & 8191] = int(keys[begins(p, 13)] & 8191);
    for (int64_t t = int64_t(rank) * kPrefixThreads + tid; t < a.tokens; t += kCluster * kPrefixThreads) a.out.state[t] = 0;
    __syncthreads();
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
    // a warp to a piece of a row
    int* minima = cluster.map_shared_rank(common, 0);
    const int pieces = (a.width + kPrefixColumns - 1) / kPrefixColumns;
    for (int64_t x = int64_t(rank) * kWarps + warp; x < int64_t(n) * pieces; x += kCluster * kWarps) {
        const int place = int(x / pieces), j0 = int(x - int64_t(place) * pieces) * kPrefixColumns;
        if (keys[place] >= kAlone) break;  // and all behind it
        const int i = int(keys[place] & 8191), first = leader[i];
        const int most = min(full[i], full[first]);
        if (i == first || j0 >= most) continue;
        const int32_t* mine = a.tables + int64_t(i) * a.width;
        const int32_t* its = a.tables + int64_t(first) * a.width;
        bool differ[kPrefixColumns / 32];
#pragma unroll
        for (int q = 0; q < kPrefixColumns / 32; ++q) {
            const int j = j0 + q * 32 + lane;
            differ[q] = j < most && mine[j] != its[j];
        }
        int at = INT_MAX;
#pragma unroll
        for (int q = kPrefixColumns / 32 - 1; q >= 0; --q) {
            const unsigned any = __ballot_sync(0xffffffffu, differ[q]);
            if (any) at = j0 + q * 32 + __ffs(any) - 1;
        }
        if (lane == 0 && at != INT_MAX) atomicMin(minima + i, at);
    }
    cluster.sync();
    if (rank != 0) return;

    // keys: leader << 40 | (kMost - length) << 13 | request; those that share nothing have the leader 8192
    constexpr uint64_t kMost = (1 << 27) - 1;
    for (int p = tid; p < n; p += kPrefixThreads) {
        const int i = int(keys[p] & 8191);
        const bool alone = keys[p] >= kAlone;
        const int first = alone ? 8192 : leader[i];
        const int length = alone ? 0 : min(common[i], min(full[i], full[first]));
        keys[p] = uint64_t(first) << 40 | (kMost - uint64_t(length)) << 13 | uint64_t(i);
    }
    __syncthreads();
    for (int i = tid; i < n; i += kPrefixThreads) best[i] = 0;  // where leaders and full blocks were
    sort(keys, size);
    auto length_of = [&](int p) { return int(kMost - (keys[p] >> 13 & kMost)); };
    int* begin = common;
    for (int p = tid; p < n; p += kPrefixThreads) {
        tokens[p] = 0;
        const int b = begins(p, 40);
        begin[p] = b;
        if (p > b) atomicMax(best + b, static_cast<unsigned long long>(int64_t(p - b) * length_of(p)) << 13 | unsigned(p));
    }
    __syncthreads();
    int64_t listed = 0;
    for (int p0 = 0; p0 < n; p0 += kPrefixThreads) {
        const int p = p0 + tid;
        int depth = 0, count = 0, total;
        if (p < n) {
            const unsigned long long b = best[begin[p]];
            depth = b >> 13 ? length_of(int(b & 8191)) : 0;  // what the group shares
            if (length_of(p) < depth) depth = 0;
            count = brings(int(keys[p] & 8191));
            if (count > kPrefixFew) s_many = 1;
            if (depth == 0) count = 0;
        }
        const int64_t to = listed + block_sum(count, warp_sums, total);
        listed += total;
        // a group's members are neighbours: one addition for those of a warp
        const int group = depth > 0 ? int(keys[p] >> 40) : -1;
        const unsigned same = __match_any_sync(0xffffffffu, group);
        const int64_t end = __shfl_sync(0xffffffffu, to + count, 31 - __clz(same));
        if (group >= 0 && lane == __ffs(same) - 1) atomicAdd(tokens + group, int(min(end - to, int64_t(INT_MAX))));
        if (p >= n) continue;
        const int i = int(keys[p] & 8191), first = int(keys[p] >> 40);
        a.out.shared[i] = first == i ? depth << a.shift : 0;
        a.out.own_first[i] = depth << a.shift;
        begin[p] = depth > 0 ? int(min(to, int64_t(INT_MAX))) : -1;
    }
    __syncthreads();
    int64_t ahead = 0;
    int largest = 0;
    for (int g0 = 0; g0 < n; g0 += kPrefixThreads) {
        const int g = g0 + tid;
        int total;
        largest = max(largest, g < n ? tokens[g] : 0);
        const int64_t start = ahead + block_sum(g < n ? tokens[g] : 0, warp_sums, total);
        if (g < n) a.out.group_starts[g] = int(min(start, a.tokens));
        ahead += total;
    }
    largest = __reduce_max_sync(0xffffffffu, largest);
    if (lane == 0 && largest > 0) atomicMax(&s_largest, largest);
    if (tid == 0) a.out.group_starts[n] = int(min(ahead, a.tokens));
    __syncthreads();
    if (tid == 0) *a.out.largest = s_largest;
    // tokens of a request: a thread, or, where a request has many, a warp
    auto write = [&](int p, int t, int step, int least, int most) {
        const int i = int(keys[p] & 8191), to = begin[p], t0 = first_token[i], count = brings(i);
        if (count < least || count > most) return;
        for (; t < count; t += step) {
            a.out.state[t0 + t] = to >= 0 ? 2 : 1;
            if (to >= 0 && int64_t(to) + t < a.tokens) a.out.list[to + t] = t0 + t;
        }
    };
    for (int p = tid; p < n; p += kPrefixThreads) write(p, 0, 1, 0, kPrefixFew);
    for (int p = warp; p < n && s_many; p += kWarps) write(p, lane, 32, kPrefixFew + 1, INT_MAX);
}

}  // namespace

cudaError_t launch_kv_fork(const KvForkArgs& a, cudaStream_t s) {
    return launch_early(kv_fork_kernel, dim3(kCluster), kShareThreads, 0, s, a);
}

cudaError_t launch_kv_compact(const KvCompactArgs& a, cudaStream_t s) {
    const size_t smem = size_t((a.blocks + 31) / 32) * 3 * sizeof(uint32_t);
    if (smem > 40 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(kv_compact_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   kKvMostCompact / 32 * 3 * int(sizeof(uint32_t)));
        if (e != cudaSuccess) return e;
    }
    return launch_early(kv_compact_kernel, dim3(kCluster), kShareThreads, smem, s, a);
}

cudaError_t launch_kv_copy(const KvCopyArgs& a, int sms, int dev, cudaStream_t s) {
    if (a.n <= 0 || a.layers <= 0) return cudaSuccess;
    constexpr int kSmem = kCopyStages * kCopySegment;
    static std::atomic<uint64_t> configured{0};
    const uint64_t bit = 1ull << (dev & 63);
    if (!(configured.load(std::memory_order_relaxed) & bit)) {
        const cudaError_t e = cudaFuncSetAttribute(kv_copy_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
        if (e != cudaSuccess) return e;
        configured.fetch_or(bit);
    }
    const int64_t segments = (a.bytes + kCopySegment - 1) / kCopySegment;
    const int64_t units = int64_t(a.n) * a.layers * 2 * segments;
    const int64_t grid = std::min<int64_t>(units, int64_t(sms) * kCopyCtas);
    return launch_early(kv_copy_kernel, dim3(unsigned(grid)), kCopyThreads, kSmem, s, a);
}

cudaError_t read_kv_copy_status(int* status, bool clear, cudaStream_t s) {
    return read_status_word(g_kv_copy_status, status, clear, s);
}

cudaError_t launch_kv_prefixes(KvPrefixArgs a, cudaStream_t s) {
    a.size = 64;
    while (a.size < a.requests) a.size *= 2;
    constexpr int kMostSmem = kKvMostPrefixes * (8 + 8 + 3 * 4);
    const size_t smem = size_t(a.size) * 8 + size_t(a.requests) * (8 + 3 * 4);
    if (smem > kPrefixPlainSmem) {
        const cudaError_t e = cudaFuncSetAttribute(kv_prefixes_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostSmem);
        if (e != cudaSuccess) return e;
    }
    return launch_early(kv_prefixes_kernel, dim3(kCluster), kPrefixThreads, smem, s, a);
}

}  // namespace ebx
