// ebx_rotary.cu -- rotary positions.
//
// A pair (a, b) of a head's elements turns by the angle that its token's position p and the pair's
// frequency f give:
//     a' = s (a cos(p f) - b sin(p f)),   b' = s (b cos(p f) + a sin(p f)).
// Pair i is (i, part / 2 + i) in the half layout and (2 i, 2 i + 1) in the interleaved one; the elements
// behind `part` are copied.  p f is a number of turns p f / (2 pi) in 64 bits, of which whole turns are
// dropped before it becomes 32 bits: at position 131071 a 32-bit p f would be off by 2^-8.
#include <algorithm>
#include <cmath>

#include <cuda_bf16.h>

#include "ebx_common.cuh"
#include "ebx_kv_check.h"

namespace ebx {
namespace {

constexpr int kRotThreads = 256;
constexpr int kRotCtas = 4;        // CTAs of an SM (4 / 5 / 6: 20000 tokens, below, 72 / 76 / 77 us, 6144 24.6 / 23.9 / 32)
constexpr int kRotTable = 2048;    // pairs in a CTA's table: 16 KB
constexpr int kRotMostDim = 2 * kRotTable;

// n / d for n < 2^31: with 2^(k-1) < d <= 2^k and mul = ceil(2^(31+k) / d), mul * d exceeds 2^(31+k) by less than d.
struct ByConstant {
    uint32_t mul, shift;
    void set(uint32_t d) {
        uint32_t k = 0;
        while ((uint64_t(1) << k) < d) ++k;
        shift = 31 + k;
        mul = uint32_t(((uint64_t(1) << shift) + d - 1) / d);
    }
    __device__ __forceinline__ uint32_t of(uint32_t n) const { return uint32_t(uint64_t(n) * mul >> shift); }
};

struct RotSide {
    const char* in;
    char* out;
    int64_t in_token, in_head, out_token, out_head;  // strides in elements
};

struct RotArgs {
    RotSide q, k;
    const void* positions;
    const void* frequencies;
    int64_t tokens;
    int q_heads, heads;    // queries' heads, and all
    int turning, chunks;   // a head's chunks that turn; these and those that are copied
    int dim, part;
    int64_t share, span;   // items of a CTA; tokens of a piece of them
    ByConstant by_chunks, by_heads, by_half;
    int wide_positions, wide_frequencies;
    float scale;
};

template <class T, int V>
struct alignas(sizeof(T) * V) Pack {
    T v[V];
};

__device__ __forceinline__ float up(float x) { return x; }
__device__ __forceinline__ float up(__half x) { return __half2float(x); }
__device__ __forceinline__ float up(__nv_bfloat16 x) { return __bfloat162float(x); }
template <class T>
__device__ __forceinline__ T down(float x) {
    if constexpr (sizeof(T) == 4) return x;
    else if constexpr (std::is_same<T, __half>::value) return __float2half_rn(x);
    else return __float2bfloat16_rn(x);
}

// An item: two vectors of V elements of a head, `second` apart, that have V pairs (in either layout the same vector of
// both halves, but neighbours for interleaved elements one by one), or one vector that is copied.
template <class T, int V>
struct RotItem {
    Pack<T, V> u, v;
    T* to;
    int at;  // its first entry in the table; -1: copied
};

// The items of all tokens, head by head, lie on one line, of which every CTA takes an equal share, in pieces whose tokens'
// sines and cosines fit the table.  The next item of a thread is on its way while it turns one, and the first of
// a piece while the table is filled.
// What bounds it: reading and writing, 20000 tokens of 40 heads of 128 in fp16 72 us = 5.7 TB/s, 0.87 of a copy's rate; 6144
// tokens (126 MB) 24.5 us; the smallest calls take a launch, 2 us.  A thread for each item, which computes its own
// angles, 121 and 42 us: 40 heads use an angle, and a sine costs 40 instructions.  A thread that keeps its angles in registers
// for every n-th head 68 to 95 and 30 to 54, as its number of waves has it; equal CTAs of 256 items that do not go on 88 to
// 105 and 24: with a table each and half the bytes on their way.  Interleaved items of one vector 98: half the bytes again.
template <class T, int V, bool PAIRS>
__global__ void __launch_bounds__(kRotThreads, kRotCtas) rotate_kernel(const __grid_constant__ RotArgs a) {
    asm volatile("griddepcontrol.wait;\n\tgriddepcontrol.launch_dependents;" ::: "memory");
    using P = Pack<T, V>;
    constexpr bool SINGLE = PAIRS && V == 1;
    constexpr int W = V >= 2 ? V / 2 : 1;   // table entries of an item, of two pairs each (one where V = 1)
    using Entry = typename std::conditional<(V >= 2), float4, float2>::type;
    using Item = RotItem<T, V>;
    extern __shared__ __align__(16) uint8_t rot_smem[];
    Entry* table = reinterpret_cast<Entry*>(rot_smem);  // [token][W][chunk]: neighbouring lanes read neighbours
    const int64_t per_token = int64_t(a.heads) * a.chunks, total = a.tokens * per_token;
    int64_t first = blockIdx.x * a.share;
    const int64_t end = min(first + a.share, total);
    const int half = a.part / 2, second = SINGLE ? 1 : half;
    for (; first < end;) {
        const int64_t t0 = first / per_token;
        const uint32_t skip = uint32_t(first - t0 * per_token);  // items of its first token ahead of the piece
        const uint32_t last = uint32_t(min(end - t0 * per_token, a.span * per_token));  // its end, counted from t0
        auto load = [&](uint32_t item, Item& x) {
            const uint32_t row = a.by_chunks.of(item), token = a.by_heads.of(row);
            const int chunk = int(item - row * a.chunks), head = int(row - token * a.heads);
            const bool q = head < a.q_heads, turns = chunk < a.turning;
            const RotSide& side = q ? a.q : a.k;
            const int h = q ? head : head - a.q_heads;
            const int e0 = !turns ? a.part + (chunk - a.turning) * V : SINGLE ? 2 * chunk : chunk * V;
            const T* in = reinterpret_cast<const T*>(side.in) + (t0 + token) * side.in_token + h * side.in_head + e0;
            x.to = reinterpret_cast<T*>(side.out) + (t0 + token) * side.out_token + h * side.out_head + e0;
            x.at = turns ? int(token) * W * a.turning + chunk : -1;
            x.u = *reinterpret_cast<const P*>(in);
            if (turns) x.v = *reinterpret_cast<const P*>(in + second);
        };
        Item x;
        uint32_t item = skip + threadIdx.x;
        if (item < last) load(item, x);
        const uint32_t entries = (a.by_heads.of(a.by_chunks.of(last - 1)) + 1) * half;
        for (uint32_t e = threadIdx.x; e < entries; e += kRotThreads) {
            const uint32_t token = a.by_half.of(e);
            const int pair = int(e - token * half);
            // its item, and its place there: the first half of an item's interleaved pairs are the first vector's
            const int back = PAIRS && V > 1 && pair >= half / 2, of = back ? pair - half / 2 : pair;
            constexpr int N = PAIRS && V > 1 ? V / 2 : V;
            const int chunk = of / N, i = of % N + (back ? N : 0);
            const double p = a.wide_positions ? double(static_cast<const int64_t*>(a.positions)[t0 + token])
                                              : double(static_cast<const int32_t*>(a.positions)[t0 + token]);
            const double f = a.wide_frequencies ? static_cast<const double*>(a.frequencies)[pair]
                                                : double(static_cast<const float*>(a.frequencies)[pair]);
            const double turn = p * f * 0.15915494309189533577;  // 1 / (2 pi)
            // half turns as 32 bits and what they leave: sin(pi (h + r)) = sin(pi h) + pi r cos(pi h) to 2^-48
            const double half_turns = 2.0 * (turn - rint(turn));
            const float h = float(half_turns), r = 3.14159265f * float(half_turns - double(h));
            float sine, cosine;
            sincospif(h, &sine, &cosine);
            const float along = fmaf(-r, sine, cosine);
            sine = fmaf(r, cosine, sine);
            cosine = along;
            float2* entry = reinterpret_cast<float2*>(table + (token * W + i / (V / W)) * a.turning + chunk);
            entry[i % (V / W)] = make_float2(cosine * a.scale, sine * a.scale);
        }
        __syncthreads();
        while (item < last) {
            Item y = x;
            item += kRotThreads;
            if (item < last) load(item, x);
            if (y.at >= 0) {
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    const Entry e = table[y.at + w * a.turning];
                    const float2* turn = reinterpret_cast<const float2*>(&e);
#pragma unroll
                    for (int k = 0; k < V / W; ++k) {
                        const int i = w * (V / W) + k;
                        const float c = turn[k].x, s = turn[k].y;
                        T& one = !PAIRS || SINGLE ? y.u.v[i] : (2 * i < V ? y.u : y.v).v[2 * i % V];
                        T& other = !PAIRS || SINGLE ? y.v.v[i] : (2 * i < V ? y.u : y.v).v[(2 * i + 1) % V];
                        const float fa = up(one), fb = up(other);
                        one = down<T>(fa * c - fb * s);
                        other = down<T>(fb * c + fa * s);
                    }
                }
                *reinterpret_cast<P*>(y.to + second) = y.v;
            }
            *reinterpret_cast<P*>(y.to) = y.u;
        }
        first = t0 * per_token + last;
        if (first < end) __syncthreads();  // the table is free again
    }
}

// Elements of a vector: the widest, of 16 bytes at most, whose chunks the halves, the part that is copied, the
// strides and the bases all allow.
int vector_of(const RotArgs& a, int size) {
    int v = 16 / size;
    auto fits = [&](const RotSide& x) {
        return (x.in_token | x.in_head | x.out_token | x.out_head) % v == 0 &&
               (reinterpret_cast<uintptr_t>(x.in) | reinterpret_cast<uintptr_t>(x.out)) % uintptr_t(v * size) == 0;
    };
    while (v > 1 && (a.part / 2 % v != 0 || (a.dim - a.part) % v != 0 || !fits(a.q) || !fits(a.k))) v /= 2;
    return v;
}

template <class T, int V>
cudaError_t launch(RotArgs a, bool pairs, bool in_place, int sms, cudaStream_t s) {
    a.turning = a.part / 2 / V;
    a.chunks = a.turning + (in_place ? 0 : (a.dim - a.part) / V);  // in place the part behind stays as it is
    const int64_t per_token = int64_t(a.heads) * a.chunks, total = a.tokens * per_token;
    a.by_chunks.set(a.chunks);
    a.by_heads.set(a.heads);
    a.by_half.set(uint32_t(a.part / 2));
    // as many CTAs as run at once, with whole rounds of their threads
    const int64_t most = int64_t(sms) * kRotCtas, rounds = (total + most * kRotThreads - 1) / (most * kRotThreads);
    a.share = rounds * kRotThreads;
    const dim3 grid{unsigned((total + a.share - 1) / a.share)};
    // tokens of a piece: what the table holds and 31 bits count, and no more than a share may touch
    a.span = std::min<int64_t>(std::max(kRotTable / (a.part / 2), 1), std::max<int64_t>(INT32_MAX / per_token - 1, 1));
    a.span = std::min(a.span, a.share / per_token + 2);
    const size_t smem = size_t(a.span) * (a.part / 2) * sizeof(float2);
    return pairs ? launch_early(rotate_kernel<T, V, true>, grid, kRotThreads, smem, s, a)
                 : launch_early(rotate_kernel<T, V, false>, grid, kRotThreads, smem, s, a);
}

template <class T>
cudaError_t launch_type(const RotArgs& a, bool pairs, bool in_place, int sms, cudaStream_t s) {
    switch (vector_of(a, int(sizeof(T)))) {
        case 8:
            if constexpr (sizeof(T) == 2) return launch<T, 8>(a, pairs, in_place, sms, s);
            return cudaErrorInvalidValue;
        case 4: return launch<T, 4>(a, pairs, in_place, sms, s);
        case 2: return launch<T, 2>(a, pairs, in_place, sms, s);
        default: return launch<T, 1>(a, pairs, in_place, sms, s);
    }
}

RotSide side_of(const ebx_rotary_side& x) {
    return RotSide{static_cast<const char*>(x.in), static_cast<char*>(x.out), x.in_token_stride, x.in_head_stride,
                   x.out_token_stride, x.out_head_stride};
}

// Null, or what is wrong with a side of elements of `size` bytes.
const char* wrong(const ebx_rotary_side& x, int size, int64_t tokens) {
    if (x.heads < 0 || x.heads > (1 << 16)) return "ebx_rotate: need 0 <= heads <= 65536";
    if (x.heads == 0 || tokens == 0) return nullptr;
    if (!x.in || !x.out) return "null argument";
    if (reinterpret_cast<uintptr_t>(x.in) % size || reinterpret_cast<uintptr_t>(x.out) % size)
        return "ebx_rotate: bases must be aligned to their elements";
    return nullptr;
}

}  // namespace
}  // namespace ebx

extern "C" ebx_status ebx_rotate(const ebx_rotary_side* q, const ebx_rotary_side* k, int32_t head_dim,
                                 int32_t rotary_dim, int32_t dtype, const void* positions,
                                 int32_t position_bits, const void* frequencies, int32_t frequency_bits,
                                 int64_t tokens, int32_t interleaved, float scale, int32_t device, void* stream) {
    if (!q) return invalid("null argument");
    if (dtype < ebx::kKvF32 || dtype > ebx::kKvBF16) return invalid("ebx_rotate: dtype must be fp32, fp16 or bf16");
    if (head_dim < 2 || head_dim > ebx::kRotMostDim || rotary_dim < 2 || rotary_dim % 2 != 0 || rotary_dim > head_dim)
        return invalid("ebx_rotate: need an even rotary_dim, 2 <= rotary_dim <= head_dim <= 4096");
    if (position_bits != 32 && position_bits != 64) return invalid("ebx_rotate: positions have 32 or 64 bits");
    if (frequency_bits != 32 && frequency_bits != 64) return invalid("ebx_rotate: frequencies have 32 or 64 bits");
    if (!std::isfinite(scale)) return invalid("ebx_rotate: scale must be finite");
    if (tokens < 0 || tokens > INT32_MAX) return invalid("ebx_rotate: need 0 <= tokens < 2^31");
    const int size = dtype == ebx::kKvF32 ? 4 : 2;
    if (const char* msg = ebx::wrong(*q, size, tokens)) return invalid(msg);
    if (k)
        if (const char* msg = ebx::wrong(*k, size, tokens)) return invalid(msg);
    ebx::RotArgs a{};
    a.q_heads = q->heads;
    a.heads = q->heads + (k ? k->heads : 0);  // at most 2^17 heads of 2^12 chunks: below 2^31 items a token
    if (tokens == 0 || a.heads == 0) return EBX_OK;
    if (!positions || !frequencies) return invalid("null argument");
    a.q = q->heads ? ebx::side_of(*q) : ebx::RotSide{};
    a.k = k && k->heads ? ebx::side_of(*k) : ebx::RotSide{};
    auto stays = [](const ebx::RotSide& x) {
        return x.in == x.out && x.in_token == x.out_token && x.in_head == x.out_head;
    };
    a.positions = positions;
    a.frequencies = frequencies;
    a.tokens = tokens;
    a.dim = head_dim;
    a.part = rotary_dim;
    a.wide_positions = position_bits == 64;
    a.wide_frequencies = frequency_bits == 64;
    a.scale = scale;
    Device d(device);
    if (d.err != cudaSuccess) return launched(d.err, "cudaSetDevice");
    const bool in_place = stays(a.q) && stays(a.k), pairs = interleaved != 0;
    const auto s = static_cast<cudaStream_t>(stream);
    const int sms = ebx::gemm_sm_count(device);
    return launched(dtype == ebx::kKvF32 ? ebx::launch_type<float>(a, pairs, in_place, sms, s)
                    : dtype == ebx::kKvF16 ? ebx::launch_type<__half>(a, pairs, in_place, sms, s)
                                           : ebx::launch_type<__nv_bfloat16>(a, pairs, in_place, sms, s), "ebx_rotate");
}
