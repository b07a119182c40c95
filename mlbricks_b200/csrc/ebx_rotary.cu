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
    int turning, chunks;   // chunks of V pairs that turn; these and the chunks of V elements behind them
    int dim, part;
    int slices;            // threads that share a token's chunk, every slices-th head each
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

// A thread has a chunk of V pairs of one token, whose angles it computes once, and every slices-th head.
template <class T, int V, bool PAIRS>
__global__ void __launch_bounds__(kRotThreads) rotate_kernel(const __grid_constant__ RotArgs a) {
    asm volatile("griddepcontrol.launch_dependents;\n\tgriddepcontrol.wait;" ::: "memory");
    using P = Pack<T, V>;
    const int64_t id = int64_t(blockIdx.x) * kRotThreads + threadIdx.x;
    const int64_t rest = id / a.chunks;
    const int chunk = int(id - rest * a.chunks);
    const int64_t token = rest / a.slices;
    const int slice = int(rest - token * a.slices);
    if (token >= a.tokens) return;
    if (chunk >= a.turning) {
        const int e = a.part + (chunk - a.turning) * V;
        for (int h = slice; h < a.heads; h += a.slices) {
            const RotSide& x = h < a.q_heads ? a.q : a.k;
            const int g = h < a.q_heads ? h : h - a.q_heads;
            const T* in = reinterpret_cast<const T*>(x.in) + token * x.in_token + g * x.in_head + e;
            T* out = reinterpret_cast<T*>(x.out) + token * x.out_token + g * x.out_head + e;
            *reinterpret_cast<P*>(out) = *reinterpret_cast<const P*>(in);
        }
        return;
    }
    float c[V], s[V];
    {
        const double p = a.wide_positions ? double(static_cast<const int64_t*>(a.positions)[token])
                                          : double(static_cast<const int32_t*>(a.positions)[token]);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int at = chunk * V + i;
            const double f = a.wide_frequencies ? static_cast<const double*>(a.frequencies)[at]
                                                : double(static_cast<const float*>(a.frequencies)[at]);
            const double turns = p * f * 0.15915494309189533577;  // 1 / (2 pi)
            sincospif(float(2.0 * (turns - rint(turns))), &s[i], &c[i]);
            s[i] *= a.scale;
            c[i] *= a.scale;
        }
    }
    const int e0 = PAIRS ? 2 * chunk * V : chunk * V, e1 = PAIRS ? e0 + V : e0 + a.part / 2;
    for (int h = slice; h < a.heads; h += a.slices) {
        const RotSide& x = h < a.q_heads ? a.q : a.k;
        const int g = h < a.q_heads ? h : h - a.q_heads;
        const T* in = reinterpret_cast<const T*>(x.in) + token * x.in_token + g * x.in_head;
        T* out = reinterpret_cast<T*>(x.out) + token * x.out_token + g * x.out_head;
        P u = *reinterpret_cast<const P*>(in + e0), v = *reinterpret_cast<const P*>(in + e1);
        P y, z;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            // element j of u, v together: a pair is (j, j + 1) or one of each
            T& ta = PAIRS ? (2 * i < V ? u.v[2 * i % V] : v.v[2 * i % V]) : u.v[i];
            T& tb = PAIRS ? (2 * i + 1 < V ? u.v[(2 * i + 1) % V] : v.v[(2 * i + 1) % V]) : v.v[i];
            const float fa = up(ta), fb = up(tb);
            const T na = down<T>(fa * c[i] - fb * s[i]), nb = down<T>(fb * c[i] + fa * s[i]);
            if constexpr (PAIRS) {
                (2 * i < V ? y.v[2 * i % V] : z.v[2 * i % V]) = na;
                (2 * i + 1 < V ? y.v[(2 * i + 1) % V] : z.v[(2 * i + 1) % V]) = nb;
            } else {
                y.v[i] = na;
                z.v[i] = nb;
            }
        }
        *reinterpret_cast<P*>(out + e0) = y;
        *reinterpret_cast<P*>(out + e1) = z;
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
cudaError_t launch(RotArgs a, bool pairs, bool in_place, cudaStream_t s) {
    a.turning = a.part / 2 / V;
    a.chunks = a.turning + (in_place ? 0 : (a.dim - a.part) / V);  // in place the part behind stays as it is
    a.slices = a.heads;
    const int64_t grid = (a.tokens * a.slices * a.chunks + kRotThreads - 1) / kRotThreads;
    if (grid > INT32_MAX) return cudaErrorInvalidValue;
    return pairs ? launch_early(rotate_kernel<T, V, true>, dim3(unsigned(grid)), kRotThreads, 0, s, a)
                 : launch_early(rotate_kernel<T, V, false>, dim3(unsigned(grid)), kRotThreads, 0, s, a);
}

template <class T>
cudaError_t launch_type(const RotArgs& a, bool pairs, bool in_place, cudaStream_t s) {
    switch (vector_of(a, int(sizeof(T)))) {
        case 8:
            if constexpr (sizeof(T) == 2) return launch<T, 8>(a, pairs, in_place, s);
            return cudaErrorInvalidValue;
        case 4: return launch<T, 4>(a, pairs, in_place, s);
        case 2: return launch<T, 2>(a, pairs, in_place, s);
        default: return launch<T, 1>(a, pairs, in_place, s);
    }
}

RotSide side_of(const ebx_rotary_side& x) {
    return RotSide{static_cast<const char*>(x.in), static_cast<char*>(x.out), x.in_token_stride, x.in_head_stride,
                   x.out_token_stride, x.out_head_stride};
}

// Null, or what is wrong with a side of elements of `size` bytes.
const char* wrong(const ebx_rotary_side& x, int size, int64_t tokens) {
    if (x.heads < 0 || x.heads > (1 << 20)) return "ebx_rotate: need 0 <= heads <= 2^20";
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
    if (head_dim < 2 || head_dim > (1 << 20) || rotary_dim < 2 || rotary_dim % 2 != 0 || rotary_dim > head_dim)
        return invalid("ebx_rotate: need an even rotary_dim, 2 <= rotary_dim <= head_dim <= 2^20");
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
    a.heads = q->heads + (k ? k->heads : 0);
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
    return launched(dtype == ebx::kKvF32 ? ebx::launch_type<float>(a, pairs, in_place, s)
                    : dtype == ebx::kKvF16 ? ebx::launch_type<__half>(a, pairs, in_place, s)
                                           : ebx::launch_type<__nv_bfloat16>(a, pairs, in_place, s), "ebx_rotate");
}
