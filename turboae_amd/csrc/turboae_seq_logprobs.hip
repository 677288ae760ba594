// tae_token_logprobs: log probability of a given token, entropy and the most probable tokens of each row of logits.
//
// Bound by memory.  A row, or a part of a long one, is read once into registers; its maximum m, s = sum e^(x - m) and t = sum (x - m) e^(x - m)
// give log p = x - m - log s and the entropy log s - t / s, and parts join by rescaling to the largest m.  Alternatives are picked one by
// one: elements are ordered by a 64-bit key (value, then the lower index), all different, so that every choice of parts gives the same ids.
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

template <int W>
__device__ __forceinline__ u64 lanes_max_key(u64 k) {
#pragma unroll
    for (int o = 1; o < W; o <<= 1) {
        const u64 other = __shfl_xor(k, o, 64);
        k = other > k ? other : k;
    }
    return k;
}

struct Stats {
    float m, s, t;
};
// Rescaled to the larger maximum.  A factor of 0 takes its part away whatever its t (a mask of the type's lowest value has an infinite one),
// but not a NaN of its s.
__device__ __forceinline__ Stats join(const Stats& a, const Stats& b) {
    const float m = fmaxf(a.m, b.m);
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

// W lanes (64 or fewer: a share of a wave; more: the workgroup) read a part of up to W * EPT - 15 elements.
template <class T, int W, int EPT, int THREADS>
__global__ __launch_bounds__(THREADS) void logprobs_part_kernel(LogprobsArgs a) {
    constexpr int V = 16 / sizeof(T), G = EPT / V, WAVES = W > 64 ? W / 64 : 1;
    __shared__ float lds_f[16][3];
    __shared__ u64 lds_k[2][16];
    const int lane = threadIdx.x % W;
    const int64_t unit = block_index() * (THREADS / W) + threadIdx.x / W;
    if (unit >= (int64_t)a.rows * a.parts) return;                  // whole workgroups, or lanes of W <= 64, which meet no barrier
    const int64_t row = unit / a.parts;
    const int part = (int)(unit % a.parts);
    const int lo = part * a.part_len, hi = min(lo + a.part_len, a.vocab);
    const T* x = (const T*)a.logits + row * a.row;
    // 16-byte granules in step with the addresses; elements in front of lo or behind hi in the outermost ones are not touched
    const int skew = (int)(reinterpret_cast<uintptr_t>(x + lo) / sizeof(T) % V);
    Pack<T, V> r[G];
#pragma unroll
    for (int g = 0; g < G; ++g) {
        const int at = lo - skew + (g * W + lane) * V;
        if (at >= lo && at + V <= hi) {
            r[g] = load<T, V>(x + at);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) r[g].v[i] = at + i >= lo && at + i < hi ? x[at + i] : (T)kNegInf;
        }
    }
    float m = kNegInf;
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
        for (int i = 0; i < V; ++i) m = fmaxf(m, (float)r[g].v[i]);
    m = lanes_max<(W < 64 ? W : 64)>(m);
    const int wave = threadIdx.x >> 6;
    if constexpr (W > 64) {
        if ((threadIdx.x & 63) == 0) lds_f[wave][0] = m;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < WAVES; ++i) m = fmaxf(m, lds_f[i][0]);
    }
    const float base = m == kNegInf ? 0.0f : m;
    float s = 0.0f, t = 0.0f;
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float d = (float)r[g].v[i] - base, e = exp_fast(d);
            s += e;
            t += e == 0.0f ? 0.0f : d * e;
        }
    s = lanes_sum<(W < 64 ? W : 64)>(s);
    t = lanes_sum<(W < 64 ? W : 64)>(t);
    if constexpr (W > 64) {
        if ((threadIdx.x & 63) == 0) { lds_f[wave][1] = s; lds_f[wave][2] = t; }
        __syncthreads();
        s = t = 0.0f;
#pragma unroll
        for (int i = 0; i < WAVES; ++i) { s += lds_f[i][1]; t += lds_f[i][2]; }
    }
    const Stats st{m, s, t};
    const bool none = s != s || m == __builtin_inff();
    const float log_s = __builtin_amdgcn_logf(s) * kLn2;
    if (lane == 0) {
        if (a.parts == 1) {
            float xt;
            const int64_t token = token_of<T>(a, row, xt);
            finish_row(a, row, st, log_s, none, xt, token);
        } else {
            store<float, 4>(a.stats + unit * 4, Pack<float, 4>{m, s, t, 0.0f});
        }
    }
    if (!a.top) return;
    // the largest key of this lane's elements that is below `limit`
    auto best_below = [&](u64 limit) {
        u64 best = 0;
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const int at = lo - skew + (g * W + lane) * V;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const u64 k = at + i >= lo && at + i < hi ? key_of((float)r[g].v[i], at + i) : 0;
                best = k > best && k < limit ? k : best;
            }
        }
        return best;
    };
    u64 best = best_below(~0ull);
    for (int j = 0; j < a.top; ++j) {
        u64 k = lanes_max_key<(W < 64 ? W : 64)>(best);
        if constexpr (W > 64) {
            if ((threadIdx.x & 63) == 0) lds_k[j & 1][wave] = k;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < WAVES; ++i) k = lds_k[j & 1][i] > k ? lds_k[j & 1][i] : k;
        }
        if (best == k) best = best_below(k);     // keys differ, so one lane (or, with none left, all of them)
        if (lane == 0) {
            if (a.parts == 1) write_top(a, row, j, k, st, log_s, none);
            else a.keys[unit * a.top + j] = k;
        }
    }
}

// Joins the parts of a row, one wave for each; lane l takes parts l, l + 64, ...
template <class T>
__global__ __launch_bounds__(64) void logprobs_join_kernel(LogprobsArgs a) {
    const int64_t row = block_index();
    if (row >= a.rows) return;
    const int lane = threadIdx.x;
    Stats st{kNegInf, 0.0f, 0.0f};
    for (int p = lane; p < a.parts; p += 64) {
        const Pack<float, 4> q = load<float, 4>(a.stats + (row * a.parts + p) * 4);
        st = join(st, Stats{q.v[0], q.v[1], q.v[2]});
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) st = join(st, Stats{__shfl_xor(st.m, o, 64), __shfl_xor(st.s, o, 64), __shfl_xor(st.t, o, 64)});
    const bool none = st.s != st.s || st.m == __builtin_inff();
    const float log_s = __builtin_amdgcn_logf(st.s) * kLn2;
    if (lane == 0) {
        float xt;
        const int64_t token = token_of<T>(a, row, xt);
        finish_row(a, row, st, log_s, none, xt, token);
    }
    u64 limit = ~0ull;
    for (int j = 0; j < a.top; ++j) {
        u64 best = 0;
        for (int p = lane; p < a.parts; p += 64) {
            const u64* k = a.keys + (row * a.parts + p) * a.top;
            for (int i = 0; i < a.top; ++i) {                       // sorted: the first below the limit is the part's largest
                if (k[i] < limit) {
                    best = k[i] > best ? k[i] : best;
                    break;
                }
            }
        }
        limit = lanes_max_key<64>(best);
        if (lane == 0) write_top(a, row, j, limit, st, log_s, none);
    }
}

struct LogprobsPlan {
    int lanes = 64, parts = 1, part_len = 0;
    size_t stats_bytes = 0, bytes = 0;
};

static bool plan_logprobs(const tae_logprobs_args* p, LogprobsPlan* s) {
    if (p->rows < 1 || p->vocab < 1 || p->vocab > (1 << 21) || p->top < 0 || p->top > 32 || p->top > p->vocab || !dtype_ok(p->dtype)) return false;
    const int V = 16 / (int)dtype_bytes(p->dtype);
    auto parts_of = [&](int lanes, int ept) {
        s->lanes = lanes;
        const int most = lanes * ept - V;
        s->parts = (int)ceil_div(p->vocab, most);
        s->part_len = (int)ceil_div(ceil_div(p->vocab, s->parts), V) * V;
        s->parts = (int)ceil_div(p->vocab, s->part_len);
    };
    if (p->vocab <= 8 * 8 - V) parts_of(8, 8);
    else if (p->vocab <= 64 * 32 - V || (int64_t)p->rows * p->vocab < (int64_t)512 * 8192) parts_of(64, 32);
    else parts_of(512, 64);
    if (s->parts > 1) {
        s->stats_bytes = (size_t)p->rows * s->parts * 16;
        s->bytes = s->stats_bytes + (size_t)p->rows * s->parts * p->top * 8;
    }
    return true;
}

template <class T>
static void launch_logprobs(const LogprobsArgs& a, int lanes, hipStream_t st) {
    const int64_t units = (int64_t)a.rows * a.parts;
    if (lanes == 8) hipLaunchKernelGGL((logprobs_part_kernel<T, 8, 8, 256>), grid_of(ceil_div(units, 32)), dim3(256), 0, st, a);
    else if (lanes == 64) hipLaunchKernelGGL((logprobs_part_kernel<T, 64, 32, 64>), grid_of(units), dim3(64), 0, st, a);
    else hipLaunchKernelGGL((logprobs_part_kernel<T, 512, 64, 512>), grid_of(units), dim3(512), 0, st, a);
    if (a.parts > 1) hipLaunchKernelGGL((logprobs_join_kernel<T>), grid_of(a.rows), dim3(64), 0, st, a);
}

}  // namespace seq
}  // namespace tae

extern "C" {

size_t tae_token_logprobs_workspace(const tae_logprobs_args* p) {
    using namespace tae::seq;
    LogprobsPlan s;
    if (!p || p->struct_size != (int32_t)sizeof(tae_logprobs_args) || !plan_logprobs(p, &s)) return 0;
    return s.bytes;
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
    if (!aligned(p->logits, dtype_bytes(p->dtype)) || !aligned(p->tokens, p->token_bytes)) return fail_msg(TAE_EINVAL, "token_logprobs: a pointer is not aligned to its elements");
    LogprobsPlan s;
    if (!plan_logprobs(p, &s)) return fail_msg(TAE_EINVAL, "token_logprobs: bad sizes");
    if (s.bytes && (!p->workspace || p->workspace_bytes < s.bytes || !aligned(p->workspace, 16)))
        return fail_msg(TAE_EINVAL, "token_logprobs: the workspace is missing, misaligned or smaller than tae_token_logprobs_workspace");
    LogprobsArgs a{p->logits, p->tokens, p->logp, p->entropy, p->top_logp, p->top_ids, s.bytes ? (float*)p->workspace : nullptr,
                   s.bytes ? (u64*)((char*)p->workspace + s.stats_bytes) : nullptr, p->logits_row, p->rows, p->vocab, p->top, s.parts, s.part_len, p->token_bytes};
    return guarded([&] {
        hipStream_t st = (hipStream_t)stream;
        switch (p->dtype) {
            case TAE_DTYPE_F32: launch_logprobs<float>(a, s.lanes, st); break;
            case TAE_DTYPE_F16: launch_logprobs<f16>(a, s.lanes, st); break;
            default: launch_logprobs<bf16>(a, s.lanes, st); break;
        }
        return (int)TAE_OK;
    });
}

}  // extern "C"
