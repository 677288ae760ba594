// tae_norm_residual: the norms before and after a block fused with its gate and residual scale.
//
//     p = post ? norm(block) w + b : block,   r = residual + alpha scale act(gate) p,   normed = norm(r) w' + b'
//
// Bound by memory: a row is read once and stays in registers (TPR lanes hold V adjacent elements in each of NV steps); mean and variance are
// two sums over those registers, the second of the squares of what is left of the first, so that a large mean costs no digits.  Measured:
// 8192 x 4096 in bf16 with gates and an fp32 residual, both norms (470 MB) 94 us, 5.0 TB/s, what a large copy reaches (5.2); 50000 x 100 in
// fp32 (80 MB) 15.4 us, 5.2 TB/s; 16 x 2048 4.4 us, most of it starting up.  EDGE: rows of any width on any element, in loads of four that
// need no alignment, the last one of a row moved back inside it: 8192 x 4095 104 us (single elements: 130).
#include "turboae_seq.hpp"

namespace tae {
namespace seq {

struct NormArgs {
    const void *residual, *block, *gate;
    const float *scale, *post_w, *post_b, *pre_w, *pre_b;
    void *out, *normed;
    int64_t rs_b, rs_r, bl_b, bl_r, ga_b, ga_r, ou_b, ou_r;
    int rows, dim, center, gate_act;
    Divisor by_len;
    float eps, alpha;
};

// 1 - 2 / (1 + e^2g) of the magnitude, and next to 0, where that loses digits, the series up to g^9: what is left out is below 2^-26 of the value
__device__ __forceinline__ float tanh_of(float g) {
    const float s = g * g, series = g * __builtin_fmaf(s, __builtin_fmaf(s, __builtin_fmaf(s, __builtin_fmaf(s, 62.0f / 2835.0f, -17.0f / 315.0f), 2.0f / 15.0f), -1.0f / 3.0f), 1.0f);
    return fabsf(g) < 0.25f ? series : copysignf(1.0f - 2.0f * sigmoid(-2.0f * fabsf(g)), g);
}
__device__ __forceinline__ float gate_value(float g, int act) {
    switch (act) {
        case TAE_ACT_TANH: return tanh_of(g);
        case TAE_ACT_SIGMOID: return sigmoid(g);
        case TAE_ACT_SILU: return silu(g);
        default: return g;
    }
}

// Sum over the TPR lanes of a row; every lane gets it.
template <int TPR, int THREADS>
__device__ __forceinline__ float row_sum(float v, float* lds) {
    v = lanes_sum<(TPR < 64 ? TPR : 64)>(v);
    if constexpr (TPR > 64) {
        const int w = threadIdx.x >> 6;
        __syncthreads();                        // the last sum has been read
        if ((threadIdx.x & 63) == 0) lds[w] = v;
        __syncthreads();
        v = 0.0f;
#pragma unroll
        for (int i = 0; i < TPR / 64; ++i) v += lds[i];
    }
    return v;
}

template <class T, class R, int V, int NV, int TPR, int THREADS, bool EDGE>
__global__ __launch_bounds__(THREADS) void norm_residual_kernel(NormArgs a) {
    __shared__ float lds[16];
    const int lane = threadIdx.x % TPR;
    const int64_t row = block_index() * (THREADS / TPR) + threadIdx.x / TPR;
    if (row >= a.rows) return;                  // whole workgroups, or with TPR <= 64 all lanes of a row, which meet no barrier
    int64_t b;
    int t;
    a.by_len.split(row, b, t);
    const R* rs = (const R*)a.residual + b * a.rs_b + t * a.rs_r;
    const T* bl = (const T*)a.block + b * a.bl_b + t * a.bl_r;
    const T* ga = (const T*)a.gate + b * a.ga_b + t * a.ga_r;
    const float inv = 1.0f / (float)a.dim;
    // All of the row is on its way before any of it is used; lanes behind the row repeat its last elements.  Only with 32 elements for each
    // of 1024 lanes (128 registers for each) the gate would not fit beside the rest: there it is loaded where it is used.
    constexpr bool GATE_AHEAD = NV * V < 32;
    Raw<R, V> raw_r[NV];
    Raw<T, V> raw_p[NV], raw_g[GATE_AHEAD ? NV : 1];
    const int over = EDGE ? (a.dim + V - 1) / V * V - a.dim : 0;            // by how much the last V reach past the row
    auto fetch = [&](auto& raw, const auto* from, int e) {
        if constexpr (EDGE) raw.from_any(from + min(e, a.dim - V));
        else raw.from(from + min(e, a.dim - V));
    };
    auto settle = [&](auto& raw, int e) {       // EDGE: the last V of a row were loaded `over` elements early
        if constexpr (EDGE) raw.drop(e < a.dim && e + V > a.dim ? over : 0);
    };
    auto place = [&](int j) { return (j * TPR + lane) * V; };
#pragma unroll
    for (int j = 0; j < NV; ++j) fetch(raw_r[j], rs, place(j));
    if (a.block) {
#pragma unroll
        for (int j = 0; j < NV; ++j) fetch(raw_p[j], bl, place(j));
        if (GATE_AHEAD && a.gate) {
#pragma unroll
            for (int j = 0; j < NV; ++j) fetch(raw_g[GATE_AHEAD ? j : 0], ga, place(j));
        }
    }
    auto vector = [&](const float* from, int e) {
        Raw<float, V> w;
        fetch(w, from, e);
        settle(w, e);
        return w;
    };
    auto put = [&](auto* to, const auto& x, int e) {
        if constexpr (EDGE) {
            if (e + V <= a.dim) {
                store_any(to + e, x);
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i)
                    if (e + i < a.dim) to[e + i] = x.v[i];
            }
        } else {
            store(to + e, x);
        }
    };
    float r[NV][V];
    auto norm_of = [&](const float (&v)[NV][V], float& mean, float& rstd) {
        mean = 0.0f;
        float s = 0.0f;
        if (a.center) {
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int i = 0; i < V; ++i) s += v[j][i];
            mean = row_sum<TPR, THREADS>(s, lds) * inv;
            s = 0.0f;
        }
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int e = place(j);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float d = e + (EDGE ? i : 0) < a.dim ? v[j][i] - mean : 0.0f;
                s = __builtin_fmaf(d, d, s);
            }
        }
        rstd = __builtin_amdgcn_rsqf(row_sum<TPR, THREADS>(s, lds) * inv + a.eps);
    };
    auto unpack = [&](float (&v)[NV][V], auto& raw) {        // zeros behind the row
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            settle(raw[j], place(j));
#pragma unroll
            for (int i = 0; i < V; ++i) v[j][i] = place(j) < a.dim ? raw[j][i] : 0.0f;
        }
    };
    if (a.block) {
        float p[NV][V];
        unpack(p, raw_p);
        float mean = 0.0f, rstd = 1.0f;
        if (a.post_w) norm_of(p, mean, rstd);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int e = place(j);
            if (e >= a.dim) continue;
            float f[V];
#pragma unroll
            for (int i = 0; i < V; ++i) f[i] = p[j][i];
            if (a.post_w) {
                const Raw<float, V> w = vector(a.post_w, e);
#pragma unroll
                for (int i = 0; i < V; ++i) f[i] = (f[i] - mean) * rstd * w[i];
                if (a.post_b) {
                    const Raw<float, V> c = vector(a.post_b, e);
#pragma unroll
                    for (int i = 0; i < V; ++i) f[i] += c[i];
                }
            }
            if (a.scale) {
                const Raw<float, V> w = vector(a.scale, e);
#pragma unroll
                for (int i = 0; i < V; ++i) f[i] *= w[i];
            }
            if (a.gate) {
                Raw<T, V>& g = raw_g[GATE_AHEAD ? j : 0];
                if (!GATE_AHEAD) fetch(g, ga, e);
                settle(g, e);
#pragma unroll
                for (int i = 0; i < V; ++i) f[i] *= gate_value(g[i], a.gate_act);
            }
#pragma unroll
            for (int i = 0; i < V; ++i) p[j][i] = f[i];
        }
        unpack(r, raw_r);
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < V; ++i) r[j][i] = __builtin_fmaf(a.alpha, p[j][i], r[j][i]);
    } else {
        unpack(r, raw_r);
    }
    if (a.out) {
        R* o = (R*)a.out + b * a.ou_b + t * a.ou_r;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int e = place(j);
            if (e >= a.dim) continue;
            Pack<R, V> x;
#pragma unroll
            for (int i = 0; i < V; ++i) x.v[i] = (R)r[j][i];
            put(o, x, e);
        }
    }
    if (a.normed) {
        float mean, rstd;
        norm_of(r, mean, rstd);
        T* o = (T*)a.normed + row * a.dim;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int e = place(j);
            if (e >= a.dim) continue;
            const Raw<float, V> w = vector(a.pre_w, e);
            float f[V];
#pragma unroll
            for (int i = 0; i < V; ++i) f[i] = (r[j][i] - mean) * rstd * w[i];
            if (a.pre_b) {
                const Raw<float, V> c = vector(a.pre_b, e);
#pragma unroll
                for (int i = 0; i < V; ++i) f[i] += c[i];
            }
            Pack<T, V> x;
#pragma unroll
            for (int i = 0; i < V; ++i) x.v[i] = (T)f[i];
            put(o, x, e);
        }
    }
}

template <class T, class R, int V, int NV, int TPR, int THREADS, bool EDGE>
static void launch_norm_as(const NormArgs& a, hipStream_t st) {
    hipLaunchKernelGGL((norm_residual_kernel<T, R, V, NV, TPR, THREADS, EDGE>), grid_of(ceil_div(a.rows, THREADS / TPR)), dim3(THREADS), 0, st, a);
}

// Lanes and steps of V that hold a row: part of a wave for short rows, then a wave, then a workgroup, so that few of them stay empty.
// Measured in us: 20736 rows of 1152 in bf16 43 (a workgroup of 256, one step: 50), of 1149 58 (256 lanes, two steps: 69; a wave, five: 61),
// 10000 of 2000 36 (a wave, four steps: 44), 8192 of 4096 94 (128 lanes, four steps: 113).
template <class T, class R, int V, bool EDGE>
static void launch_norm_width(const NormArgs& a, hipStream_t st) {
    const int vecs = (int)ceil_div(a.dim, V);
    if (vecs <= 16) launch_norm_as<T, R, V, 1, 16, 256, EDGE>(a, st);
    else if (vecs <= 32) launch_norm_as<T, R, V, 1, 32, 256, EDGE>(a, st);
    else if (vecs <= 64) launch_norm_as<T, R, V, 1, 64, 256, EDGE>(a, st);
    else if (vecs <= 128) launch_norm_as<T, R, V, 2, 64, 256, EDGE>(a, st);
    else if (vecs <= 192) launch_norm_as<T, R, V, 3, 64, 256, EDGE>(a, st);
    else if (vecs <= 256) launch_norm_as<T, R, V, 1, 256, 256, EDGE>(a, st);
    else if (vecs <= 384) launch_norm_as<T, R, V, 3, 128, 128, EDGE>(a, st);
    else if (vecs <= 512) launch_norm_as<T, R, V, 2, 256, 256, EDGE>(a, st);
    else if (vecs <= 768) launch_norm_as<T, R, V, 3, 256, 256, EDGE>(a, st);
    else if (vecs <= 1024) launch_norm_as<T, R, V, 4, 256, 256, EDGE>(a, st);
    else if (vecs <= 2048) launch_norm_as<T, R, V, 2, 1024, 1024, EDGE>(a, st);
    else if (V == 8 || vecs <= 4096) launch_norm_as<T, R, V, 4, 1024, 1024, EDGE>(a, st);
    else if constexpr (V < 8) launch_norm_as<T, R, V, 8, 1024, 1024, EDGE>(a, st);
}

template <class T, class R>
static void launch_norm(const NormArgs& a, int width, hipStream_t st) {
    if (width == 8) launch_norm_width<T, R, 8, false>(a, st);
    else if (width == 4) launch_norm_width<T, R, 4, false>(a, st);
    else if (a.dim >= 4) launch_norm_width<T, R, 4, true>(a, st);
    else launch_norm_as<T, R, 1, 1, 16, 256, false>(a, st);
}

}  // namespace seq
}  // namespace tae

extern "C" int tae_norm_residual(const tae_norm_args* p, void* stream) {
    using namespace tae;
    using namespace tae::seq;
    if (!p || p->struct_size != (int32_t)sizeof(tae_norm_args)) return fail_msg(TAE_EINVAL, "tae_norm_args: NULL or struct_size mismatch (ABI)");
    if (!dtype_ok(p->dtype)) return fail_msg(TAE_EINVAL, "norm_residual: dtype must be a TAE_DTYPE_* code");
    if (p->residual_dtype != p->dtype && p->residual_dtype != TAE_DTYPE_F32) return fail_msg(TAE_EINVAL, "norm_residual: the residual has the block's type or fp32");
    if (p->batch < 1 || p->len < 1 || (int64_t)p->batch * p->len > INT32_MAX) return fail_msg(TAE_EINVAL, "norm_residual: batch and len must be >= 1, their product below 2^31");
    if (p->dim < 1 || p->dim > 32768) return fail_msg(TAE_EINVAL, "norm_residual: dim must be in 1..32768");
    if (!(p->eps >= 0x1p-126f)) return fail_msg(TAE_EINVAL, "norm_residual: eps must be > 0, and no subnormal number");
    if (p->gate_act != TAE_ACT_LINEAR && p->gate_act != TAE_ACT_TANH && p->gate_act != TAE_ACT_SIGMOID && p->gate_act != TAE_ACT_SILU)
        return fail_msg(TAE_EINVAL, "norm_residual: gate_act must be linear, tanh, sigmoid or silu");
    if (!p->residual) return fail_msg(TAE_EINVAL, "norm_residual: residual is NULL");
    if (p->block && !p->residual_out) return fail_msg(TAE_EINVAL, "norm_residual: a block needs residual_out");
    if (!p->block && (p->gate || p->scale || p->post_weight)) return fail_msg(TAE_EINVAL, "norm_residual: gate, scale and post_weight need a block");
    if ((p->post_bias && !p->post_weight) || (p->pre_bias && !p->pre_weight)) return fail_msg(TAE_EINVAL, "norm_residual: a bias needs its weight");
    if ((p->normed != nullptr) != (p->pre_weight != nullptr)) return fail_msg(TAE_EINVAL, "norm_residual: normed and pre_weight come together");
    if (!p->residual_out && !p->normed) return fail_msg(TAE_EINVAL, "norm_residual: nothing to write");
    if (p->residual_out == p->residual && p->residual && (p->out_batch != p->residual_batch || p->out_row != p->residual_row))
        return fail_msg(TAE_EINVAL, "norm_residual: an in-place residual_out has the residual's strides");
    const size_t tb = dtype_bytes(p->dtype), rb = dtype_bytes(p->residual_dtype);
    if (!elements_aligned(tb, p->block, p->gate, p->normed) || !elements_aligned(rb, p->residual, p->residual_out) ||
        !elements_aligned(4, p->scale, p->post_weight, p->post_bias, p->pre_weight, p->pre_bias))
        return fail_msg(TAE_EINVAL, "norm_residual: a pointer is not aligned to its elements");
    Width wt(tb), wr(rb), wf(4);
    wt.elements(p->dim).pointer(p->normed);
    if (p->block) wt.pointer(p->block).elements(p->block_batch).elements(p->block_row);
    if (p->gate) wt.pointer(p->gate).elements(p->gate_batch).elements(p->gate_row);
    wr.elements(p->dim).pointer(p->residual).elements(p->residual_batch).elements(p->residual_row);
    if (p->residual_out) wr.pointer(p->residual_out).elements(p->out_batch).elements(p->out_row);
    wf.elements(p->dim).pointer(p->scale).pointer(p->post_weight).pointer(p->post_bias).pointer(p->pre_weight).pointer(p->pre_bias);
    int width = 1;
    for (int v : {8, 4})
        if (width == 1 && p->dim % v == 0 && wt.fits(v * tb < 16 ? v * tb : 16) && wr.fits(v * rb < 16 ? v * rb : 16) && wf.fits(16)) width = v;
    NormArgs a{p->residual, p->block, p->gate, p->scale, p->post_weight, p->post_bias, p->pre_weight, p->pre_bias, p->residual_out, p->normed,
               p->residual_batch, p->residual_row, p->block_batch, p->block_row, p->gate_batch, p->gate_row, p->out_batch, p->out_row,
               p->batch * p->len, p->dim, p->center ? 1 : 0, p->gate_act, Divisor(p->len), p->eps, p->alpha};
    return guarded([&] {
        hipStream_t st = (hipStream_t)stream;
        const bool same = p->residual_dtype == p->dtype;
        switch (p->dtype) {
            case TAE_DTYPE_F32: launch_norm<float, float>(a, width, st); break;
            case TAE_DTYPE_F16: same ? launch_norm<f16, f16>(a, width, st) : launch_norm<f16, float>(a, width, st); break;
            default: same ? launch_norm<bf16, bf16>(a, width, st) : launch_norm<bf16, float>(a, width, st); break;
        }
        return (int)TAE_OK;
    });
}
