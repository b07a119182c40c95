// ebx_kv_share.cu -- requests that share cache blocks: fork (and free, and roll back), compact, copying blocks,
// and finding the prefixes that requests share.  No reference counterpart.
//
// The bookkeeping kernels (fork, compact, prefixes) are one cluster of CTAs each: their phases need what all
// rows or all blocks gave in the phase before, the data are a few hundred kilobytes, and a cluster's barrier costs
// a fraction of a launch.  Counts are changed by atomic additions only, whose order does not change
// them, and whatever is given an order (blocks to the ring, copies) gets it from sums over rows or ids.
#include <algorithm>
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
__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(kShareThreads, 1) kv_fork_kernel(const __grid_constant__ KvForkArgs a) {
    asm volatile("griddepcontrol.launch_dependents;\n\tgriddepcontrol.wait;" ::: "memory");
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

    for (int b = gtid; b < a.blocks; b += kAll) {
        a.out_shares[b] = a.shares[b];
        a.claim[b] = INT_MAX;
    }
    for (int r = gtid; r < a.requests; r += kAll) a.sources[r] = a.targets[r] = -1;
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

    // who keeps a begun block that no row holds whole
    auto key_of = [&](const ForkRow& f, int r) { return f.parent == r ? r : r + a.requests; };
    auto tail_of = [&](const ForkRow& f) { return a.tables[int64_t(f.parent) * a.width + (f.keep >> a.shift)]; };
    for (int r = gtid; r < a.requests; r += kAll) {
        const ForkRow f = fork_row(a, r);
        if (!f.begun) continue;
        const int id = tail_of(f);
        if (block(id) && a.out_shares[id] < 0) atomicMin(a.claim + id, key_of(f, r));
    }
    cluster.sync();

    if (rank == 0) {
        int64_t taken = 0;
        for (int base = 0; base < a.requests; base += kShareThreads) {
            const int r = base + tid;
            bool need = false;
            int id = -1, column = 0;
            if (r < a.requests) {
                const ForkRow f = fork_row(a, r);
                if (f.begun) {
                    id = tail_of(f);
                    column = f.keep >> a.shift;
                    need = block(id);
                    if (need && a.claim[id] == key_of(f, r)) {
                        atomicAdd(a.out_shares + id, 1);
                        need = false;
                    }
                }
            }
            int total;
            const int64_t before = taken + block_sum(need, warp_sums, total);
            if (need) {
                if (before < avail) {
                    const int fresh = a.free_ring[wrapped(front + before)];
                    a.out_tables[int64_t(r) * a.width + column] = fresh;
                    a.sources[before] = id;
                    a.targets[before] = fresh;
                } else {
                    a.out_lengths[r] = 0;
                    atomicAdd(&s_missing, 1);
                }
            }
            taken += total;
        }
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
    int mine = 0;
    for (int b = b0 + tid; b < b1; b += kShareThreads) mine += a.out_shares[b] < 0;
    int total;
    block_sum(mine, warp_sums, total);
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
// first and so on: the fewest moves there can be, and no block is read and written.
__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(kShareThreads, 1) kv_compact_kernel(const __grid_constant__ KvCompactArgs a) {
    asm volatile("griddepcontrol.launch_dependents;\n\tgriddepcontrol.wait;" ::: "memory");
    cg::cluster_group cluster = cg::this_cluster();
    __shared__ int warp_sums[32];
    __shared__ int counts[3][kCluster];
    const int tid = threadIdx.x, lane = tid & 31, rank = int(cluster.block_rank());
    const int gtid = rank * kShareThreads + tid, gwarp = gtid >> 5;
    constexpr int kAll = kCluster * kShareThreads, kAllWarps = kAll / 32;
    const int half = a.blocks / 2;
    auto block = [&](int id) { return id >= 0 && id < a.blocks; };
    auto held_by = [&](int r) {
        const int64_t n = (int64_t(max(a.lengths[r], 0)) + (1 << a.shift) - 1) >> a.shift;
        return int(min(n, int64_t(a.width)));
    };
    for (int b = gtid; b < a.blocks; b += kAll) a.map[b] = -1;
    for (int j = gtid; j < half; j += kAll) a.sources[j] = a.targets[j] = -1;
    cluster.sync();
    for (int r = gwarp; r < a.requests; r += kAllWarps) {
        const int n = held_by(r);
        for (int j = lane; j < n; j += 32) {
            const int id = a.tables[int64_t(r) * a.width + j];
            if (block(id)) a.map[id] = 0;
        }
    }
    cluster.sync();
    const int per = int((int64_t(a.blocks) + kCluster - 1) / kCluster);
    const int b0 = min(rank * int64_t(per), int64_t(a.blocks)), b1 = min(b0 + int64_t(per), int64_t(a.blocks));
    int mine = 0, total;
    for (int b = b0 + tid; b < b1; b += kShareThreads) mine += a.map[b] >= 0;
    block_sum(mine, warp_sums, total);
    tell(cluster, counts[0], total);
    int held = 0;
    for (int c = 0; c < kCluster; ++c) held += counts[0][c];
    int high = 0, low = 0;
    for (int b = b0 + tid; b < b1; b += kShareThreads) {
        const bool is = a.map[b] >= 0;
        high += is && b >= held;
        low += !is && b < held;
    }
    int highs, lows;
    block_sum(high, warp_sums, highs);
    block_sum(low, warp_sums, lows);
    tell(cluster, counts[1], highs);
    tell(cluster, counts[2], lows);
    int at_high = 0, at_low = 0, moves = 0;
    for (int c = 0; c < kCluster; ++c) {
        if (c < rank) {
            at_high += counts[1][c];
            at_low += counts[2][c];
        }
        moves += counts[1][c];
    }
    for (int base = b0; base < b1; base += kShareThreads) {
        const int b = base + tid;
        const bool is = b < b1 && a.map[b] >= 0;
        const bool is_high = is && b >= held, is_low = b < b1 && !is && b < held;
        const int h = at_high + block_sum(is_high, warp_sums, highs);
        const int l = at_low + block_sum(is_low, warp_sums, lows);
        if (is_high) {
            a.sources[h] = b;
            a.map[b] = h;
        }
        if (is_low) a.targets[l] = b;
        at_high += highs;
        at_low += lows;
    }
    cluster.sync();
    auto moved = [&](int id) { return id < held ? id : a.targets[a.map[id]]; };
    for (int64_t at = gwarp; at < a.requests; at += kAllWarps) {
        const int n = held_by(int(at));
        for (int j = lane; j < a.width; j += 32) {
            const int id = j < n ? a.tables[at * a.width + j] : -1;
            a.out_tables[at * a.width + j] = block(id) ? moved(id) : -1;
        }
    }
    for (int b = gtid; b < a.blocks; b += kAll) {
        if (a.map[b] >= 0) a.out_shares[moved(b)] = a.shares[b];
        if (b >= held) a.out_shares[b] = 0;
        a.free_out[b] = b < a.blocks - held ? held + b : -1;
    }
    if (gtid == 0) {
        a.ring_out[0] = 0;
        a.ring_out[1] = a.blocks - held;
        a.ring_out[2] = 0;
        a.ring_out[3] = moves;
    }
}

// ---- copy ---------------------------------------------------------------------------------

constexpr int kCopyThreads = 256;
constexpr int kCopySegment = kCopyThreads * 16 * 4;  // bytes of a unit

// Unit: a segment of one side of one pair of blocks in one layer; the first segment brings the scales along.
__global__ void __launch_bounds__(kCopyThreads) kv_copy_kernel(const __grid_constant__ KvCopyArgs a) {
    asm volatile("griddepcontrol.launch_dependents;\n\tgriddepcontrol.wait;" ::: "memory");
    const int64_t pairs = a.count ? min(max(*a.count, int64_t(0)), int64_t(a.n)) : a.n;
    const int segments = int((a.bytes + kCopySegment - 1) / kCopySegment);
    const int64_t units = pairs * a.layers * 2 * segments;
    for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
        const int64_t side_unit = u / segments;
        const int segment = int(u - side_unit * segments), side = int(side_unit & 1);
        const int64_t layer_unit = side_unit >> 1;
        const int64_t pair = layer_unit / a.layers;
        const int layer = int(layer_unit - pair * a.layers);
        const int from = a.sources[pair], to = a.targets[pair];
        if (from < 0 || from >= a.blocks || to < 0 || to >= a.blocks || from == to) continue;
        const int8_t* src = a.layer[layer].codes[side] + from * a.bytes;
        int8_t* dst = a.layer[layer].codes[side] + to * a.bytes;
        const int64_t first = int64_t(segment) * kCopySegment + threadIdx.x * 16;
        uint4 v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (first + i * kCopyThreads * 16 < a.bytes) v[i] = *reinterpret_cast<const uint4*>(src + first + i * kCopyThreads * 16);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (first + i * kCopyThreads * 16 < a.bytes) *reinterpret_cast<uint4*>(dst + first + i * kCopyThreads * 16) = v[i];
        if (segment == 0) {
            float* scales = a.layer[layer].scales[side];
            for (int h = threadIdx.x; h < a.kv_heads; h += kCopyThreads)
                scales[int64_t(to) * a.kv_heads + h] = scales[int64_t(from) * a.kv_heads + h];
        }
    }
}

// ---- prefixes -----------------------------------------------------------------------------

// Requests that bring tokens and whose tables begin with the same block are compared with the first of
// them: common[i] full blocks ahead of the new tokens are the same.  Of the lengths that occur, the one that
// saves most reading, (members with at least that much in common - 1) * length, becomes the group's.
__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(kShareThreads, 1) kv_prefixes_kernel(const __grid_constant__ KvPrefixArgs a) {
    asm volatile("griddepcontrol.launch_dependents;\n\tgriddepcontrol.wait;" ::: "memory");
    cg::cluster_group cluster = cg::this_cluster();
    extern __shared__ int2 found[];  // [requests]: leader, blocks in common
    __shared__ int warp_sums[32];
    const int tid = threadIdx.x, lane = tid & 31, rank = int(cluster.block_rank());
    const int gtid = rank * kShareThreads + tid, gwarp = gtid >> 5;
    constexpr int kAll = kCluster * kShareThreads, kAllWarps = kAll / 32;
    const int n = a.requests;
    unsigned long long* best = reinterpret_cast<unsigned long long*>(a.scratch);  // [n]: saved << 14 | request
    int2* pairs = reinterpret_cast<int2*>(a.scratch + 2 * n);                     // [n]: `found`
    int* offset = a.scratch + 4 * n;                                              // [n]: tokens of the group ahead
    int* totals = a.scratch + 5 * n;                                              // [n]: tokens of group i
    auto from = [&](int i) { return int(min(max(int64_t(a.starts[i]), int64_t(0)), a.tokens)); };
    auto brings = [&](int i) { return max(from(i + 1) - from(i), 0); };
    auto ahead = [&](int i) {  // full blocks ahead of the new tokens
        const int64_t cap = int64_t(a.width) << a.shift;
        const int64_t past = min(int64_t(max(a.lengths[i], 0)), cap) - brings(i);
        return past > 0 && brings(i) > 0 ? int(past >> a.shift) : 0;
    };
    auto block = [&](int id) { return id >= 0 && id < a.blocks; };
    auto key_of = [&](int i) {
        const int id = ahead(i) > 0 ? a.tables[int64_t(i) * a.width] : -1;
        return block(id) ? id : -1;
    };

    for (int i = gtid; i < n; i += kAll) {
        const int key = key_of(i);
        if (key >= 0) a.first_with[key] = INT_MAX;
        best[i] = 0;
    }
    for (int64_t t = gtid; t < a.tokens; t += kAll) a.out.state[t] = 0;
    cluster.sync();
    for (int i = gtid; i < n; i += kAll) {
        const int key = key_of(i);
        if (key >= 0) atomicMin(a.first_with + key, i);
    }
    cluster.sync();
    for (int i = gwarp; i < n; i += kAllWarps) {
        const int key = key_of(i);
        const int leader = key >= 0 ? a.first_with[key] : -1;
        int common = 0;
        if (leader == i) common = ahead(i);
        if (leader >= 0 && leader != i) {
            const int most = min(ahead(i), ahead(leader));
            const int32_t* x = a.tables + int64_t(i) * a.width;
            const int32_t* y = a.tables + int64_t(leader) * a.width;
            common = most;
            for (int j0 = 0; j0 < most; j0 += 128) {
                unsigned differ[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int j = j0 + q * 32 + lane;
                    differ[q] = __ballot_sync(0xffffffffu, j < most && x[j] != y[j]);
                }
                int at = -1;
#pragma unroll
                for (int q = 3; q >= 0; --q)
                    if (differ[q]) at = j0 + q * 32 + __ffs(differ[q]) - 1;
                if (at >= 0) {
                    common = at;
                    break;
                }
            }
        }
        if (lane == 0) pairs[i] = make_int2(leader, common);
    }
    cluster.sync();
    for (int i = tid; i < n; i += kShareThreads) found[i] = pairs[i];
    __syncthreads();
    for (int i = gtid; i < n; i += kAll) {
        const int2 me = found[i];
        if (me.x < 0) continue;
        int members = 0;
        for (int j = me.x; j < n; ++j) {
            const int2 it = found[j];
            members += it.x == me.x && it.y >= me.y;
        }
        if (members > 1) atomicMax(best + me.x, static_cast<unsigned long long>(int64_t(members - 1) * me.y) << 14 | unsigned(i));
    }
    cluster.sync();
    // blocks that group g shares; 0: no group
    auto depth = [&](int g) { return best[g] == 0 ? 0 : found[int(best[g] & 0x3fff)].y; };
    auto grouped = [&](int i) { return found[i].x >= 0 && depth(found[i].x) > 0 && found[i].y >= depth(found[i].x); };
    for (int i = gtid; i < n; i += kAll) {
        const int2 me = found[i];
        const bool in = grouped(i);
        const int deep = in ? depth(me.x) : 0;
        int ahead_of_me = 0, all = 0;
        if (in) {
            for (int j = me.x; j < (me.x == i ? n : i); ++j) {
                const int2 it = found[j];
                const int m = it.x == me.x && it.y >= deep ? brings(j) : 0;
                if (j < i) ahead_of_me += m;
                all += m;
            }
        }
        offset[i] = ahead_of_me;
        totals[i] = in && me.x == i ? all : 0;
        a.out.shared[i] = in && me.x == i ? deep << a.shift : 0;
        a.out.own_first[i] = deep << a.shift;
    }
    cluster.sync();
    // every CTA sums for itself; `found` then holds the groups' first tokens in place of the leaders
    int base = 0;
    for (int i0 = 0; i0 < n; i0 += kShareThreads) {
        const int i = i0 + tid;
        int total;
        const int start = base + block_sum(i < n ? totals[i] : 0, warp_sums, total);
        if (i < n && rank == 0) a.out.group_starts[i] = int(min(int64_t(start), a.tokens));
        if (i < n) found[i].y = start;
        base += total;
    }
    if (gtid == 0) a.out.group_starts[n] = int(min(int64_t(base), a.tokens));
    __syncthreads();
    for (int i = gwarp; i < n; i += kAllWarps) {
        const bool in = a.out.own_first[i] > 0;
        const int64_t to = in ? int64_t(found[found[i].x].y) + offset[i] : 0;
        const int t0 = from(i), count = brings(i);
        for (int t = lane; t < count; t += 32) {
            a.out.state[t0 + t] = in ? 2 : 1;
            if (in && uint64_t(to + t) < uint64_t(a.tokens)) a.out.list[to + t] = t0 + t;
        }
    }
}

}  // namespace

cudaError_t launch_kv_fork(const KvForkArgs& a, cudaStream_t s) {
    return launch_early(kv_fork_kernel, dim3(kCluster), kShareThreads, 0, s, a);
}

cudaError_t launch_kv_compact(const KvCompactArgs& a, cudaStream_t s) {
    return launch_early(kv_compact_kernel, dim3(kCluster), kShareThreads, 0, s, a);
}

cudaError_t launch_kv_copy(const KvCopyArgs& a, int sms, cudaStream_t s) {
    if (a.n <= 0 || a.layers <= 0) return cudaSuccess;
    const int64_t segments = (a.bytes + kCopySegment - 1) / kCopySegment;
    const int64_t units = int64_t(a.n) * a.layers * 2 * segments;
    const int64_t grid = std::min<int64_t>(units, int64_t(sms) * 8);
    return launch_early(kv_copy_kernel, dim3(unsigned(grid)), kCopyThreads, 0, s, a);
}

cudaError_t launch_kv_prefixes(const KvPrefixArgs& a, cudaStream_t s) {
    const size_t smem = size_t(a.requests) * sizeof(int2);
    if (smem > 40 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(kv_prefixes_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   kKvMaxRequests * int(sizeof(int2)));
        if (e != cudaSuccess) return e;
    }
    return launch_early(kv_prefixes_kernel, dim3(kCluster), kShareThreads, smem, s, a);
}

}  // namespace ebx
