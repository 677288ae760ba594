// tae_token_logprobs: log probability of a given token, entropy and the most probable tokens of each row of logits.
//
// Bound by memory.  A row, or a part of a long one, is read once into registers; its maximum m, s = sum e^(x - m) and t = sum (x - m) e^(x - m)
// give log p = x - m - log s and the entropy log s - t / s, and parts join by rescaling to the largest m.  Elements are ordered by a 64-bit
// key (value, then the lower index), all different, so that every choice of parts gives the same ids.
//
// Measured, bf16, 2048 x 131072 with 8 alternatives (537 MB): 106 to 124 us, 4.3 to 5.1 TB/s (a large copy: 5.2), 8 of them the join.  14.5
// vector instructions for each element of a lane keep the SIMDs as busy as memory: taking each of bf16's elements apart once and holding it
// costs more (157 us: half the waves), parts of 512 lanes more too.  8 x 50001 in fp32 with 20: 7 us and 5 for the join, mostly waiting.
#include "turboae_seq.hpp"

namespace tae {
namespace seq {

using u64 = unsigned long long;

struct LogprobsArgs {
    const void* logits;
    const void* tokens;
    float *logp, *entropy, *top_logp;
    int64_t* top_ids;
    float* stats;                                // workspace: (rows, parts, 4): m, s, t, -
    u64* keys;                                   // workspace: (rows, parts, top)
    int64_t row;
    int rows, vocab, top, parts, part_len, token_bytes;
};

constexpr float kNegInf = -__builtin_inff();

// larger value first, then lower index; 0 is below every element
__device__ __forceinline__ u64 key_of(float v, uint32_t index) {
    const uint32_t u = __float_as_uint(v + 0.0f);                  // -0 equals +0
    const uint32_t order = u & 0x80000000u ? ~u : u | 0x80000000u;
    return ((u64)order << 32) | (uint32_t)~index;
}
__device__ __forceinline__ float key_value(u64 k) {
    const uint32_t o = (uint32_t)(k >> 32);
    return __uint_as_float(o & 0x80000000u ? o & 0x7FFFFFFFu : ~o);
}
__device__ __forceinline__ uint32_t key_index(u64 k) { return ~(uint32_t)k; }

template <int CTRL>
__device__ __forceinline__ u64 dpp_key(u64 k) {
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)k, CTRL, 0xF, 0xF, true), hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(k >> 32), CTRL, 0xF, 0xF, true);
    return ((u64)hi << 32) | lo;
}
template <int W>
__device__ __forceinline__ u64 lanes_max_key(u64 k) {
    auto op = [](u64 a, u64 b) { return a > b ? a : b; };
    k = op(k, dpp_key<kXor1>(k));
    k = op(k, dpp_key<kXor2>(k));
    k = op(k, dpp_key<kHalfMirror>(k));
    if constexpr (W == 64) {
        k = op(k, dpp_key<kMirror>(k));
        k = op(k, __shfl_xor(k, 16, 64));
        k = op(k, __shfl_xor(k, 32, 64));
    }
    static_assert(W == 8 || W == 64, "lanes of a row");
    return k;
}

struct Stats {
    float m, s, t;
};
// Rescaled to the larger maximum.  A factor of 0 takes its part away whatever its t (a mask of the type's lowest value has an infinite one).
// A row with a NaN has the maximum NaN.
__device__ __forceinline__ Stats join(const Stats& a, const Stats& b) {
    const float m = __builtin_elementwise_maximum(a.m, b.m);
    const float da = a.m == kNegInf ? kNegInf : a.m - m, db = b.m == kNegInf ? kNegInf : b.m - m;
    const float fa = exp_fast(da), fb = exp_fast(db);
    const float ta = fa == 0.0f ? 0.0f : __builtin_fmaf(da, a.s, a.t) * fa, tb = fb == 0.0f ? 0.0f : __builtin_fmaf(db, b.s, b.t) * fb;
    return Stats{m, __builtin_fmaf(a.s, fa, b.s * fb), ta + tb};
}

// The results of one row, by the first lane of its lanes.
__device__ __forceinline__ void finish_row(const LogprobsArgs& a, int64_t row, const Stats& st, float log_s, bool none, float x_token, int64_t token) {
    float lp, h;
    if (none) {
        lp = h = __builtin_nanf("");
    } else if (st.m == kNegInf) {
        lp = kNegInf;
        h = 0.0f;
    } else {
        lp = x_token - st.m - log_s;
        h = fmaxf(log_s - st.t / st.s, 0.0f);
    }
    if (token < 0) lp = none ? __builtin_nanf("") : 0.0f;
    else if (token >= a.vocab) lp = __builtin_nanf("");
    a.logp[row] = lp;
    a.entropy[row] = h;
}

template <class T>
__device__ __forceinline__ int64_t token_of(const LogprobsArgs& a, int64_t row, float& x) {
    const int64_t token = a.token_bytes == 8 ? ((const int64_t*)a.tokens)[row] : ((const int32_t*)a.tokens)[row];
    x = token >= 0 && token < a.vocab ? (float)((const T*)a.logits)[row * a.row + token] : 0.0f;
    return token;
}

__device__ __forceinline__ void write_top(const LogprobsArgs& a, int64_t row, int i, u64 key, const Stats& st, float log_s, bool none) {
    a.top_ids[row * a.top + i] = none ? -1 : (int64_t)key_index(key);
    a.top_logp[row * a.top + i] = none ? __builtin_nanf("") : st.m == kNegInf ? kNegInf : key_value(key) - st.m - log_s;
}

__device__ __forceinline__ uint32_t order_of(u64 k) { return (uint32_t)(k >> 32); }

// W lanes (64 or fewer: a share of a wave; more: the workgroup) read a part of a row into registers, EPT elements each, in granules of V.
//
// Alternatives: `top` lanes have a largest element at or above the top-th largest lane maximum, so no element below it is among the `top`.
// The bound is found by bits, by counting lanes that reach it (16 of them: a lower bound does no harm), first in each wave, then among
// what reaches the largest of these.  Elements at or above it, hardly more than `top` in a usual row, are collected in LDS and sorted by
// counting larger keys.  Rows with more than fit (many equal
// values) take the largest one by one.
template <class T, int W, int EPT, int V, int THREADS>
__global__ __launch_bounds__(THREADS) void logprobs_part_kernel(LogprobsArgs a) {
    constexpr int G = EPT / V, WAVES = W > 64 ? W / 64 : 1, WW = W < 64 ? W : 64, ROOM = W < 64 ? 1 : 128;
    __shared__ float lds_f[WAVES][3];
    __shared__ u64 lds_k[2][WAVES], found[WAVES][ROOM];
    __shared__ uint32_t lds_u[WAVES], lds_n[WAVES], tops[64], tops_n;
    const int lane = threadIdx.x % W;
    const int64_t unit = block_index() * (THREADS / W) + threadIdx.x / W;
    if (unit >= (int64_t)a.rows * a.parts) return;                  // whole workgroups, or lanes of W < 64, which meet no barrier
    const int64_t row = unit / a.parts;
    const int part = (int)(unit % a.parts);
    const int lo = part * a.part_len, hi = min(lo + a.part_len, a.vocab);
    const T* x = (const T*)a.logits + row * a.row;
    // granules in step with 16-byte addresses
    const int skew = V == 1 ? 0 : (int)(reinterpret_cast<uintptr_t>(x + lo) / sizeof(T) % V);
    auto place = [&](int g) { return lo - skew + (g * W + lane) * V; };
    // as whole registers, taken apart anew in each pass over them (`again` keeps the compiler from holding the parts)
    constexpr int D = V == 1 ? 1 : 4;            // registers of a granule
    uint32_t w[G][D];
    auto value = [&](int g, int i) -> float {
        if constexpr (V == 1 || sizeof(T) == 4) return __uint_as_float(w[g][i]);
        // by bits: of a conversion the compiler would make bf16 maxima, back and forth
        else if constexpr (std::is_same_v<T, bf16>) return __uint_as_float(i & 1 ? w[g][i / 2] & 0xFFFF0000u : w[g][i / 2] << 16);
        else return (float)__builtin_bit_cast(T, (uint16_t)(i & 1 ? w[g][i / 2] >> 16 : w[g][i / 2] & 0xFFFFu));
    };
    auto again = [&]() {
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
            for (int i = 0; i < D; ++i) asm volatile("" : "+v"(w[g][i]));
    };
    if constexpr (V == 1) {
#pragma unroll
        for (int g = 0; g < G; ++g) w[g][0] = __float_as_uint(place(g) < hi ? (float)x[place(g)] : kNegInf);
    } else {
        // whole granules first, all loads in flight at once (others repeat one), then the elements of the outermost ones
        const int low = lo + (V - skew) % V, high = lo - skew + (hi - lo + skew) / V * V - V;
        if (high >= low) {
#pragma unroll
            for (int g = 0; g < G; ++g) {
                const uint4 u = *reinterpret_cast<const uint4*>(x + min(max(place(g), low), high));
                w[g][0] = u.x, w[g][1] = u.y, w[g][2] = u.z, w[g][3] = u.w;
            }
        }
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const int at = place(g);
            if (at < low || at > high) {
                Pack<T, V> p;
#pragma unroll
                for (int i = 0; i < V; ++i) p.v[i] = (T)kNegInf;
                if (at + V > lo && at < hi) {
#pragma unroll
                    for (int i = 0; i < V; ++i)
                        if (at + i >= lo && at + i < hi) p.v[i] = x[at + i];
                }
                const uint4 u = __builtin_bit_cast(uint4, p);
                w[g][0] = u.x, w[g][1] = u.y, w[g][2] = u.z, w[g][3] = u.w;
            }
        }
    }
    again();
    const int wave = threadIdx.x >> 6;
    float mine = kNegInf, of[G];                 // largest of the lane and of its granules; NaN if there is one
    // granules behind the row for a whole wave are left out
    auto filled = [&](int g) { return W < 64 || __builtin_amdgcn_readfirstlane(place(g)) < hi; };
#pragma unroll
    for (int g = 0; g < G; ++g) {
        of[g] = kNegInf;
        if (!filled(g)) continue;
        of[g] = value(g, 0);
#pragma unroll
        for (int i = 1; i < V; ++i) of[g] = __builtin_elementwise_maximum(of[g], value(g, i));
        mine = __builtin_elementwise_maximum(mine, of[g]);
    }
    again();
    float m = lanes_join<WW>(mine, [](float a, float b) { return __builtin_elementwise_maximum(a, b); });
    uint32_t bound = 0, own = 0;
    // the largest 16-bit prefix that `top` of the wave's 64 values reach
    auto reached = [&](uint32_t v) {
        uint32_t prefix = 0;
#pragma unroll
        for (int bit = 31; bit >= 16; --bit) {
            const uint32_t with = prefix | 1u << bit;
            if (__popcll(__ballot(v >= with)) >= a.top) prefix = with;
        }
        return prefix;
    };
    if constexpr (W >= 64) {
        if (a.top) {
            own = lo - skew + lane * V < hi ? order_of(key_of(mine, 0)) : 0u;
            bound = reached(own);
        }
    }
    if constexpr (W > 64) {
        if ((threadIdx.x & 63) == 0) { lds_f[wave][0] = m; lds_u[wave] = bound; }
        if (threadIdx.x == 0) tops_n = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < WAVES; ++i) { m = __builtin_elementwise_maximum(m, lds_f[i][0]); bound = max(bound, lds_u[i]); }
    }
    if constexpr (W > 64) {
        // lane maxima at or above that bound, of the whole workgroup: where they fit one wave, they give a closer one below
        const u64 set = __ballot(a.top && own >= bound);
        if (set) {
            uint32_t first = 0;
            if ((threadIdx.x & 63) == 0) first = atomicAdd(&tops_n, (uint32_t)__popcll(set));
            first = __builtin_amdgcn_readfirstlane(first);
            const uint32_t slot = first + __builtin_amdgcn_mbcnt_hi((uint32_t)(set >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)set, 0));
            if (a.top && own >= bound && slot < 64) tops[slot] = own;
        }
    }
    // e^(x - m) = 2^(x log2 e - c), c = m log2 e rounded, with one fused product; by how much c was rounded is known exactly (`off`) and put
    // right in the sums.  Where that could be much (a maximum like the type's lowest value) the difference comes first.  -inf, and what is
    // far below m, is taken at 2^-1000 = 0, so that 0 times its distance is 0.
    const float base = m == kNegInf ? 0.0f : m, c = base * kLog2e;
    const bool near = fabsf(base) < 0x1p20f;
    const float off = near ? __builtin_fmaf(base, kLog2e, -c) : 0.0f;
    float s = 0.0f, t = 0.0f;
    auto sums = [&](auto&& distance) {
#pragma unroll
        for (int g = 0; g < G; ++g) {
            if (!filled(g)) continue;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float d = fmaxf(distance(value(g, i)), -1000.0f), e = __builtin_amdgcn_exp2f(d);
                s += e;
                t = __builtin_fmaf(d, e, t);
            }
        }
    };
    if (near) sums([&](float x) { return __builtin_fmaf(x, kLog2e, -c); });
    else sums([&](float x) { return (x - base) * kLog2e; });
    again();
    s = lanes_sum<WW>(s);
    t = lanes_sum<WW>(t);
    if constexpr (W > 64) {
        if ((threadIdx.x & 63) == 0) { lds_f[wave][1] = s; lds_f[wave][2] = t; }
        __syncthreads();
        s = t = 0.0f;
#pragma unroll
        for (int i = 0; i < WAVES; ++i) { s += lds_f[i][1]; t += lds_f[i][2]; }
    }
    const float back = __builtin_amdgcn_exp2f(-off);
    s *= back;
    t = __builtin_fmaf(t, back, -off * s);
    const Stats st{m, s, t * kLn2};
    const bool none = m != m || m == __builtin_inff();
    const float log_s = __builtin_amdgcn_logf(s) * kLn2;
    if (lane == 0) {
        if (a.parts == 1) {
            float xt;
            const int64_t token = token_of<T>(a, row, xt);
            finish_row(a, row, st, log_s, none, xt, token);
        } else {
            store<float, 4>(a.stats + unit * 4, Pack<float, 4>{m, s, st.t, 0.0f});
        }
    }
    if (!a.top) return;
    auto put = [&](int j, u64 k) {
        if (a.parts == 1) write_top(a, row, j, k, st, log_s, none);
        else a.keys[unit * a.top + j] = k;
    };
    if constexpr (W >= 64) {
        if constexpr (W > 64) {
            if (tops_n <= 64) bound = max(bound, reached((threadIdx.x & 63) < tops_n ? tops[threadIdx.x & 63] : 0u));
        }
        // each wave's own list, filled in the order of granules and lanes; granules without a candidate cost one comparison
        const float least = bound ? key_value((u64)bound << 32) : kNegInf;
        uint32_t n = 0;
#pragma unroll
        for (int g = 0; g < G; ++g) {
            if (!__any(!(of[g] < least))) continue;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float v = value(g, i);
                if (!__any(!(v < least))) continue;
                const int at = place(g) + i;
                const bool yes = !(v < least) && at >= lo && at < hi;
                const u64 set = __ballot(yes);
                const uint32_t slot = n + __builtin_amdgcn_mbcnt_hi((uint32_t)(set >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)set, 0));
                if (yes && slot < ROOM) found[wave][slot] = key_of(v, at);
                n += __popcll(set);
            }
        }
        if ((threadIdx.x & 63) < 8 && n + (threadIdx.x & 63) < ROOM) found[wave][n + (threadIdx.x & 63)] = 0;      // whole groups of eight
        bool fits = n <= ROOM;
        uint32_t total = n;
        if constexpr (W > 64) {
            if ((threadIdx.x & 63) == 0) lds_n[wave] = n;
            __syncthreads();
            total = 0;
            fits = true;
#pragma unroll
            for (int i = 0; i < WAVES; ++i) {
                total += lds_n[i];
                fits = fits && lds_n[i] <= ROOM;
            }
        } else {
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
        if (fits) {
            for (int j = total + lane; j < a.top; j += W) put(j, 0);      // a part with fewer elements
            for (int c = threadIdx.x & 63; c < (int)n; c += 64) {
                const u64 k = found[wave][c];
                int rank = 0;
                for (int u = 0; u < WAVES; ++u) {
                    const int count = W > 64 ? (int)lds_n[u] : (int)n;
                    for (int i = 0; i < count; i += 8) {
#pragma unroll
                        for (int j = 0; j < 8; ++j) rank += found[u][i + j] > k;
                    }
                }
                if (rank < a.top) put(rank, k);
            }
            return;
        }
    }
    // the largest key of this lane's elements that is below `limit`
    auto best_below = [&](u64 limit) {
        u64 best = 0;
        if constexpr (W < 64) {
#pragma unroll
            for (int g = 0; g < G; ++g) {
                const u64 k = place(g) < hi ? key_of(value(g, 0), place(g)) : 0;
                best = k > best && k < limit ? k : best;
            }
        } else {                                 // read again, so that this rare way costs the usual one no registers
#pragma unroll 1
            for (int g = 0; g < G; ++g)
#pragma unroll 1
                for (int i = 0; i < V; ++i) {
                    const int at = place(g) + i;
                    const u64 k = at >= lo && at < hi ? key_of((float)x[at], at) : 0;
                    best = k > best && k < limit ? k : best;
                }
        }
        return best;
    };
    u64 best = best_below(~0ull);
    for (int j = 0; j < a.top; ++j) {
        u64 k = lanes_max_key<WW>(best);
        if constexpr (W > 64) {
            if ((threadIdx.x & 63) == 0) lds_k[j & 1][wave] = k;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < WAVES; ++i) k = lds_k[j & 1][i] > k ? lds_k[j & 1][i] : k;
        }
        if (best == k) best = best_below(k);     // keys differ, so one lane (or, with none left, all of them)
        if (lane == 0) put(j, k);
    }
}

// Joins the parts of a row, one workgroup for each: the statistics by rescaling, the sorted lists of alternatives by counting larger keys.
// What cannot be among them is left out beforehand: with j = ceil(top / parts), r = ceil(top / j), the r-th largest of the lists' j-th keys has
// j r >= top keys at or above it.
template <class T>
__global__ __launch_bounds__(256) void logprobs_join_kernel(LogprobsArgs a) {
    extern __shared__ u64 lists[];               // parts x top
    __shared__ u64 found[1024], bound;
    __shared__ uint32_t count;
    __shared__ Stats lds[4];
    const int64_t row = block_index();
    if (row >= a.rows) return;
    const int tid = threadIdx.x, all = a.parts * a.top;
    for (int i = tid; i < all; i += 256) lists[i] = a.keys[row * all + i];
    if (tid == 0) { bound = 1; count = 0; }
    Stats st{kNegInf, 0.0f, 0.0f};
    for (int p = tid; p < a.parts; p += 256) {
        const Pack<float, 4> q = load<float, 4>(a.stats + (row * a.parts + p) * 4);
        st = join(st, Stats{q.v[0], q.v[1], q.v[2]});
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) st = join(st, Stats{__shfl_xor(st.m, o, 64), __shfl_xor(st.s, o, 64), __shfl_xor(st.t, o, 64)});
    if ((tid & 63) == 0) lds[tid >> 6] = st;
    __syncthreads();
    st = join(join(lds[0], lds[1]), join(lds[2], lds[3]));
    const bool none = st.m != st.m || st.m == __builtin_inff();
    const float log_s = __builtin_amdgcn_logf(st.s) * kLn2;
    if (tid == 0) {
        float xt;
        const int64_t token = token_of<T>(a, row, xt);
        finish_row(a, row, st, log_s, none, xt, token);
    }
    if (!a.top) return;
    const int jth = (a.top + a.parts - 1) / a.parts, rth = (a.top + jth - 1) / jth;
    for (int p = tid; p < a.parts; p += 256) {
        const u64 k = lists[p * a.top + jth - 1];
        int rank = 0;
        for (int i = 0; i < a.parts; ++i) rank += lists[i * a.top + jth - 1] > k;
        if (rank == rth - 1 && k) bound = k;
    }
    __syncthreads();
    // at most rth lists of top keys each and jth - 1 of the others are left: 1024 at the most, with top = 32
    for (int i = tid; i < all; i += 256) {
        const u64 k = lists[i];
        if (k >= bound) found[atomicAdd(&count, 1u)] = k;
    }
    __syncthreads();
    if (tid < 8 && count + tid < 1024) found[count + tid] = 0;      // whole groups of eight
    __syncthreads();
    for (int c = tid; c < (int)count; c += 256) {
        const u64 k = found[c];
        int rank = 0;
        for (int i = 0; i < (int)count; i += 8) {
#pragma unroll
            for (int j = 0; j < 8; ++j) rank += found[i + j] > k;
        }
        if (rank < a.top) write_top(a, row, rank, k, st, log_s, none);
    }
}

template <class T>
static void launch_logprobs(const LogprobsArgs& a, const LogprobsPlan& s, hipStream_t st) {
    constexpr int V = 16 / sizeof(T);
    const int64_t units = (int64_t)a.rows * a.parts;
    if (s.lanes == 8) hipLaunchKernelGGL((logprobs_part_kernel<T, 8, 8, 1, 256>), grid_of(ceil_div(units, 32)), dim3(256), 0, st, a);
    else if (s.lanes == 64 && s.ept == 8 && a.top) hipLaunchKernelGGL((logprobs_part_kernel<T, 64, 8, 1, 64>), grid_of(units), dim3(64), 0, st, a);
    else if (s.lanes == 64 && s.ept == 8) hipLaunchKernelGGL((logprobs_part_kernel<T, 64, 8, V, 64>), grid_of(units), dim3(64), 0, st, a);
    else if (s.lanes == 64) hipLaunchKernelGGL((logprobs_part_kernel<T, 64, 32, V, 64>), grid_of(units), dim3(64), 0, st, a);
    else if (s.ept == 32) hipLaunchKernelGGL((logprobs_part_kernel<T, 256, 32, V, 256>), grid_of(units), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((logprobs_part_kernel<T, 256, 64, V, 256>), grid_of(units), dim3(256), 0, st, a);
    if (a.parts > 1) hipLaunchKernelGGL((logprobs_join_kernel<T>), grid_of(a.rows), dim3(256), (size_t)a.parts * a.top * 8, st, a);
}

}  // namespace seq
}  // namespace tae

extern "C" {

size_t tae_token_logprobs_workspace(const tae_logprobs_args* p) {
    using namespace tae::seq;
    LogprobsPlan s, u;
    if (!p || p->struct_size != (int32_t)sizeof(tae_logprobs_args) || !plan_logprobs(p, true, &s) || !plan_logprobs(p, false, &u)) return 0;
    return std::max(s.bytes, u.bytes);
}

int tae_token_logprobs(const tae_logprobs_args* p, void* stream) {
    using namespace tae;
    using namespace tae::seq;
    if (!p || p->struct_size != (int32_t)sizeof(tae_logprobs_args)) return fail_msg(TAE_EINVAL, "tae_logprobs_args: NULL or struct_size mismatch (ABI)");
    if (!dtype_ok(p->dtype)) return fail_msg(TAE_EINVAL, "token_logprobs: dtype must be a TAE_DTYPE_* code");
    if (p->rows < 1 || p->vocab < 1 || p->vocab > (1 << 21)) return fail_msg(TAE_EINVAL, "token_logprobs: rows must be >= 1, vocab in 1..2^21");
    if (p->top < 0 || p->top > 32 || p->top > p->vocab) return fail_msg(TAE_EINVAL, "token_logprobs: top must be in 0..32 and at most vocab");
    if (p->token_bytes != 4 && p->token_bytes != 8) return fail_msg(TAE_EINVAL, "token_logprobs: token_bytes must be 4 or 8");
    if (!p->logits || !p->tokens || !p->logp || !p->entropy) return fail_msg(TAE_EINVAL, "token_logprobs: logits, tokens, logp and entropy must not be NULL");
    if (p->top && (!p->top_ids || !p->top_logp)) return fail_msg(TAE_EINVAL, "token_logprobs: top needs top_ids and top_logp");
    if (!elements_aligned(dtype_bytes(p->dtype), p->logits) || !elements_aligned(p->token_bytes, p->tokens) || !elements_aligned(4, p->logp, p->entropy, p->top_logp) ||
        !elements_aligned(8, p->top_ids))
        return fail_msg(TAE_EINVAL, "token_logprobs: a pointer is not aligned to its elements");
    LogprobsPlan s;
    const bool rows16 = aligned(p->logits, 16) && p->logits_row * (int64_t)dtype_bytes(p->dtype) % 16 == 0;
    if (!plan_logprobs(p, rows16, &s)) return fail_msg(TAE_EINVAL, "token_logprobs: bad sizes");
    if ((int64_t)p->rows * s.parts > ((int64_t)kGridX << 15)) return fail_msg(TAE_EINVAL, "token_logprobs: too many rows for one call");
    if (s.bytes && (!p->workspace || p->workspace_bytes < s.bytes || !aligned(p->workspace, 16)))
        return fail_msg(TAE_EINVAL, "token_logprobs: the workspace is missing, misaligned or smaller than tae_token_logprobs_workspace");
    LogprobsArgs a{p->logits, p->tokens, p->logp, p->entropy, p->top_logp, p->top_ids, s.bytes ? (float*)p->workspace : nullptr,
                   s.bytes ? (u64*)((char*)p->workspace + s.stats_bytes) : nullptr, p->logits_row, p->rows, p->vocab, p->top, s.parts, s.part_len, p->token_bytes};
    return guarded([&] {
        hipStream_t st = (hipStream_t)stream;
        switch (p->dtype) {
            case TAE_DTYPE_F32: launch_logprobs<float>(a, s, st); break;
            case TAE_DTYPE_F16: launch_logprobs<f16>(a, s, st); break;
            default: launch_logprobs<bf16>(a, s, st); break;
        }
        return (int)TAE_OK;
    });
}

}  // extern "C"
