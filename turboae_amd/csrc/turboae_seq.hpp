// What the sequence operators (turboae_seq_*.hip) share: element types, vector loads and stores, reductions over lanes, and the checks of
// their C entry points.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <cmath>
#include <exception>
#include <type_traits>

#include "turboae_seq_plan.hpp"

namespace tae {

int fail_msg(int code, const char* msg);      // sets the calling thread's tae_last_error string, returns `code`

namespace seq {

using bf16 = __bf16;
using f16 = _Float16;

// V adjacent elements; loads and stores of up to 16 bytes are one instruction each
template <class T, int V>
struct alignas(sizeof(T) * V < 16 ? sizeof(T) * V : 16) Pack {
    T v[V];
};

template <class T, int V>
__device__ __forceinline__ Pack<T, V> load(const T* p) { return *reinterpret_cast<const Pack<T, V>*>(p); }
template <class T, int V>
__device__ __forceinline__ void store(T* p, const Pack<T, V>& a) { *reinterpret_cast<Pack<T, V>*>(p) = a; }

// The same from and to an address that is aligned to its elements only
template <class T, int V>
__device__ __forceinline__ Pack<T, V> load_any(const T* p) {
    Pack<T, V> a;
    __builtin_memcpy(&a, p, sizeof(a));
    return a;
}
template <class T, int V>
__device__ __forceinline__ void store_any(T* p, const Pack<T, V>& a) { __builtin_memcpy(p, &a, sizeof(a)); }

// Four elements of T in `w` without the first n of them (0 to 3), those behind them moved up, zeros at the end
template <class T>
__device__ __forceinline__ void drop_first(uint32_t* w, int n) {
    if constexpr (sizeof(T) == 2) {
        const uint64_t u = ((uint64_t)w[1] << 32 | w[0]) >> (16 * n);
        w[0] = (uint32_t)u, w[1] = (uint32_t)(u >> 32);
    } else {
        if (n & 1) w[0] = w[1], w[1] = w[2], w[2] = w[3], w[3] = 0;
        if (n & 2) w[0] = w[2], w[1] = w[3], w[2] = w[3] = 0;
    }
}

// V adjacent elements as they were loaded, in whole registers: an element is taken out when it is used, so that a load stays in flight until
// then and 16-bit elements need no registers of their own.
template <class T, int V>
struct Raw {
    static constexpr int BYTES = sizeof(T) * V, WORDS = (BYTES + 3) / 4;
    uint32_t w[WORDS];
    __device__ __forceinline__ void from(const T* p) {
        if constexpr (BYTES == 2) {
            w[0] = *reinterpret_cast<const uint16_t*>(p);
        } else if constexpr (BYTES == 4) {
            w[0] = *reinterpret_cast<const uint32_t*>(p);
        } else if constexpr (BYTES == 8) {
            const uint2 u = *reinterpret_cast<const uint2*>(p);
            w[0] = u.x, w[1] = u.y;
        } else {
            static_assert(BYTES % 16 == 0, "whole 16-byte loads");
#pragma unroll
            for (int i = 0; i < BYTES / 16; ++i) {
                const uint4 u = reinterpret_cast<const uint4*>(p)[i];
                w[4 * i] = u.x, w[4 * i + 1] = u.y, w[4 * i + 2] = u.z, w[4 * i + 3] = u.w;
            }
        }
    }
    // from an address that is aligned to its elements only
    __device__ __forceinline__ void from_any(const T* p) {
        if constexpr (BYTES < 4) from(p);
        else __builtin_memcpy(w, p, BYTES);
    }
    __device__ __forceinline__ void drop(int n) {
        static_assert(V == 4, "four elements");
        drop_first<T>(w, n);
    }
    __device__ __forceinline__ float operator[](int i) const {
        if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
        else return (float)__builtin_bit_cast(T, (uint16_t)(i & 1 ? w[i / 2] >> 16 : w[i / 2] & 0xFFFFu));
    }
};

constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.693147180559945309f;

__device__ __forceinline__ float exp_fast(float x) { return __builtin_amdgcn_exp2f(x * kLog2e); }       // relative error 2^-22 |x| and up to one ulp
__device__ __forceinline__ float sigmoid(float x) { return __builtin_amdgcn_rcpf(1.0f + exp_fast(-x)); }
__device__ __forceinline__ float silu(float x) { return x * sigmoid(x); }
// log(1 + e^x) = max(x, 0) + log(1 + w), w = e^-|x|.  u = 1 + w loses the last digits of a small w; log(u) plus what was lost, w - (u - 1), has
// the relative accuracy that log(u) alone has not (next to u = 1 the two differ by the loss itself).
__device__ __forceinline__ float softplus(float x) {
    const float w = exp_fast(-fabsf(x)), u = 1.0f + w;
    return fmaxf(x, 0.0f) + __builtin_fmaf(__builtin_amdgcn_logf(u), kLn2, w - (u - 1.0f));
}

// A value from another lane of the same 16: quad_perm [1,0,3,2], [2,3,0,1], row_half_mirror, row_mirror, row_ror:8.  All lanes that take part
// have to be active: never inside a choice that lanes make differently.
constexpr int kXor1 = 0xB1, kXor2 = 0x4E, kHalfMirror = 0x141, kMirror = 0x140, kRor8 = 0x128;
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, true));
}
__device__ __forceinline__ float lane_value(float v, int lane) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane)); }

// `op` over the W adjacent lanes that share a value (W a power of two up to 64); every lane gets the result.  The mirrors pair lanes that
// already hold the same partial result.
template <int W, class Op>
__device__ __forceinline__ float lanes_join(float v, Op&& op) {
    if constexpr (W >= 2) v = op(v, dpp<kXor1>(v));
    if constexpr (W >= 4) v = op(v, dpp<kXor2>(v));
    if constexpr (W >= 8) v = op(v, dpp<kHalfMirror>(v));
    if constexpr (W >= 16) v = op(v, dpp<kMirror>(v));
    if constexpr (W == 32) v = op(v, __shfl_xor(v, 16, 64));
    if constexpr (W == 64) v = op(op(lane_value(v, 0), lane_value(v, 16)), op(lane_value(v, 32), lane_value(v, 48)));
    return v;
}
template <int W>
__device__ __forceinline__ float lanes_sum(float v) {
    return lanes_join<W>(v, [](float a, float b) { return a + b; });
}
template <int W>
__device__ __forceinline__ float lanes_max(float v) {
    return lanes_join<W>(v, [](float a, float b) { return fmaxf(a, b); });
}

inline bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) % n) == 0; }
// every pointer on a multiple of its elements' size (NULL is)
template <class... P>
inline bool elements_aligned(size_t n, const P*... p) { return (aligned(p, n) && ...); }
// How wide loads and stores may be: collects sizes, strides and addresses; fits(n) says whether all of them are multiples of n bytes.
struct Width {
    size_t bytes;
    int64_t all = 0;                             // bits of every size, stride (in elements) and address
    explicit Width(size_t element) : bytes(element) {}
    Width& elements(int64_t n) { all |= n * (int64_t)bytes; return *this; }
    Width& pointer(const void* p) { all |= (int64_t)reinterpret_cast<uintptr_t>(p); return *this; }
    bool fits(size_t n) const { return (all & (int64_t)(n - 1)) == 0; }
};

// A launch of n workgroups, n up to 2^40: one grid dimension holds fewer than 2^32 work items.  Workgroups behind the last have nothing to do.
constexpr int kGridX = 1 << 20;
inline dim3 grid_of(int64_t n) { return n <= kGridX ? dim3((uint32_t)n) : dim3(kGridX, (uint32_t)ceil_div(n, kGridX)); }
__device__ __forceinline__ int64_t block_index() { return (int64_t)blockIdx.y * kGridX + blockIdx.x; }

// Quotients by a number that the host knows, with one product (Granlund and Montgomery 1994): for n < 2^31, n / d = (mulhi(n, m) + n) >> s
// with s = ceil(log2 d), m = floor(2^32 (2^s - d) / d) + 1.  Larger n are divided.
struct Divisor {
    uint32_t d, m, s;
    Divisor() = default;
    explicit Divisor(int64_t by) : d((uint32_t)by), s(0) {
        while ((1ull << s) < d) ++s;
        m = (uint32_t)(((1ull << 32) * ((1ull << s) - d)) / d + 1);
    }
    __device__ __forceinline__ void split(int64_t n, int64_t& quotient, int& rest) const {
        if (n >> 31) {
            quotient = n / d;
            rest = (int)(n % d);
        } else {
            const uint32_t u = (uint32_t)n, q = (uint32_t)(((uint64_t)__umulhi(u, m) + u) >> s);
            quotient = q;
            rest = (int)(u - q * d);
        }
    }
};

// The launches of a C entry point: no exception leaves it, and a failed launch is an error of this call.
template <class F>
int guarded(F&& f) {
    try {
        const int rc = f();
        if (rc != TAE_OK) return rc;
        const hipError_t e = hipGetLastError();
        return e == hipSuccess ? TAE_OK : fail_msg(TAE_EHIP, hipGetErrorString(e));
    } catch (const std::exception& e) {
        return fail_msg(TAE_ENOMEM, e.what());
    } catch (...) {
        return fail_msg(TAE_ENOMEM, "unknown exception");
    }
}

}  // namespace seq
}  // namespace tae
