// tae_causal_conv: y[t] = act(bias + sum_k weight[k] x[t - K + 1 + k]) of each channel, with the last K - 1 inputs as state.
//
// Bound by memory.  A lane owns V adjacent channels and walks kSteps positions with the window in registers: x is read once, plus the K - 1
// positions in front of its piece (which its neighbour has just read, so they come from L2).
#include "turboae_seq.hpp"

namespace tae {
namespace seq {

struct ConvArgs {
    const void* x;
    const float *weight, *bias;
    const void* state;
    const int32_t* lengths;
    void *y, *state_out;
    int64_t x_b, x_r;
    int len, channels, groups, pieces, act;      // groups: lanes that cover the channels; pieces: of kSteps positions
    int64_t lanes;                               // batch * pieces * groups
};

constexpr int kSteps = 16;

template <class T, int V, int K>
__global__ __launch_bounds__(256) void causal_conv_kernel(ConvArgs a) {
    const int64_t id = block_index() * 256 + threadIdx.x;
    if (id >= a.lanes) return;
    const int g = (int)(id % a.groups);
    const int64_t rest = id / a.groups;
    const int piece = (int)(rest % a.pieces);
    const int64_t b = rest / a.pieces;
    const int e = g * V, t0 = piece * kSteps, E = a.channels;
    const int n = a.lengths ? min(max(a.lengths[b], 0), a.len) : a.len;
    const T* x = (const T*)a.x + b * a.x_b + e;
    const T* before = a.state ? (const T*)a.state + b * (K - 1) * E + e : nullptr;
    T* y = (T*)a.y + b * a.len * E + e;
    // input i of the sequence, the state's in front of it at i < 0
    auto input = [&](int i) {
        if (i >= 0) return load<T, V>(x + (int64_t)i * a.x_r);
        if (before) return load<T, V>(before + (int64_t)(i + K - 1) * E);
        Pack<T, V> zero;
#pragma unroll
        for (int v = 0; v < V; ++v) zero.v[v] = (T)0.0f;
        return zero;
    };
    float w[K][V], c[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        c[v] = a.bias ? a.bias[e + v] : 0.0f;
#pragma unroll
        for (int k = 0; k < K; ++k) w[k][v] = a.weight[(int64_t)(e + v) * K + k];
    }
    float win[K - 1 + kSteps][V];
    const int steps = min(kSteps, n - t0);       // of valid positions; may be negative
#pragma unroll
    for (int i = 0; i < K - 1 + kSteps; ++i) {
        const bool need = i < K - 1 ? steps > 0 : i - (K - 1) < steps;
        if (need) {
            const Pack<T, V> p = input(t0 + i - (K - 1));
#pragma unroll
            for (int v = 0; v < V; ++v) win[i][v] = (float)p.v[v];
        } else {
#pragma unroll
            for (int v = 0; v < V; ++v) win[i][v] = 0.0f;
        }
    }
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
        if (t0 + i >= a.len) break;
        Pack<T, V> out;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float s = c[v];
#pragma unroll
            for (int k = 0; k < K; ++k) s = __builtin_fmaf(w[k][v], win[i + k][v], s);
            if (a.act == TAE_ACT_SILU) s = silu(s);
            out.v[v] = (T)(i < steps ? s : 0.0f);
        }
        store<T, V>(y + (int64_t)(t0 + i) * E, out);
    }
    // Only this lane reads the state of these channels (a later piece starts at least K - 1 positions in), and it has read all of it before
    // it writes: state_out may be the state.
    if (piece == 0 && a.state_out && K > 1) {
        T* o = (T*)a.state_out + b * (K - 1) * E + e;
        Pack<T, V> last[K > 1 ? K - 1 : 1];
#pragma unroll
        for (int j = 0; j < K - 1; ++j) last[j] = input(n + j - (K - 1));
#pragma unroll
        for (int j = 0; j < K - 1; ++j) store<T, V>(o + (int64_t)j * E, last[j]);
    }
}

template <class T, int V>
static void launch_conv(const ConvArgs& a, int taps, hipStream_t st) {
    const dim3 grid = grid_of(ceil_div(a.lanes, 256));
    switch (taps) {
        case 1: hipLaunchKernelGGL((causal_conv_kernel<T, V, 1>), grid, dim3(256), 0, st, a); break;
        case 2: hipLaunchKernelGGL((causal_conv_kernel<T, V, 2>), grid, dim3(256), 0, st, a); break;
        case 3: hipLaunchKernelGGL((causal_conv_kernel<T, V, 3>), grid, dim3(256), 0, st, a); break;
        case 4: hipLaunchKernelGGL((causal_conv_kernel<T, V, 4>), grid, dim3(256), 0, st, a); break;
        case 5: hipLaunchKernelGGL((causal_conv_kernel<T, V, 5>), grid, dim3(256), 0, st, a); break;
        case 6: hipLaunchKernelGGL((causal_conv_kernel<T, V, 6>), grid, dim3(256), 0, st, a); break;
        case 7: hipLaunchKernelGGL((causal_conv_kernel<T, V, 7>), grid, dim3(256), 0, st, a); break;
        default: hipLaunchKernelGGL((causal_conv_kernel<T, V, 8>), grid, dim3(256), 0, st, a); break;
    }
}

}  // namespace seq
}  // namespace tae

extern "C" int tae_causal_conv(const tae_conv_args* p, void* stream) {
    using namespace tae;
    using namespace tae::seq;
    if (!p || p->struct_size != (int32_t)sizeof(tae_conv_args)) return fail_msg(TAE_EINVAL, "tae_conv_args: NULL or struct_size mismatch (ABI)");
    if (!dtype_ok(p->dtype)) return fail_msg(TAE_EINVAL, "causal_conv: dtype must be a TAE_DTYPE_* code");
    if (p->batch < 1 || p->len < 1 || p->channels < 1) return fail_msg(TAE_EINVAL, "causal_conv: batch, len and channels must be >= 1");
    if (p->len > INT32_MAX - 64 || p->channels > INT32_MAX - 64) return fail_msg(TAE_EINVAL, "causal_conv: len and channels must stay below 2^31 - 64");
    if (p->taps < 1 || p->taps > 8) return fail_msg(TAE_EINVAL, "causal_conv: taps must be in 1..8");
    if (p->act != TAE_ACT_LINEAR && p->act != TAE_ACT_SILU) return fail_msg(TAE_EINVAL, "causal_conv: act must be linear or silu");
    if (!p->x || !p->weight || !p->y) return fail_msg(TAE_EINVAL, "causal_conv: x, weight and y must not be NULL");
    const size_t tb = dtype_bytes(p->dtype);
    Width w(tb);
    w.elements(p->channels).elements(p->x_batch).elements(p->x_row).pointer(p->x).pointer(p->y).pointer(p->state).pointer(p->state_out);
    const int vec = w.fits(16) ? (int)(16 / tb) : w.fits(4) ? (int)(4 / tb) : 1;
    ConvArgs a{p->x, p->weight, p->bias, p->state, p->lengths, p->y, p->state_out, p->x_batch, p->x_row, p->len, p->channels,
               p->channels / vec, (int)ceil_div(p->len, kSteps), p->act, 0};
    a.lanes = (int64_t)p->batch * a.pieces * a.groups;
    if (ceil_div(a.lanes, 256) > ((int64_t)kGridX << 15)) return fail_msg(TAE_EINVAL, "causal_conv: the batch is too large for one call");
    return guarded([&] {
        hipStream_t st = (hipStream_t)stream;
        switch (p->dtype) {
            case TAE_DTYPE_F32: vec == 4 ? launch_conv<float, 4>(a, p->taps, st) : launch_conv<float, 1>(a, p->taps, st); break;
            case TAE_DTYPE_F16: vec == 8 ? launch_conv<f16, 8>(a, p->taps, st) : vec == 2 ? launch_conv<f16, 2>(a, p->taps, st) : launch_conv<f16, 1>(a, p->taps, st); break;
            default: vec == 8 ? launch_conv<bf16, 8>(a, p->taps, st) : vec == 2 ? launch_conv<bf16, 2>(a, p->taps, st) : launch_conv<bf16, 1>(a, p->taps, st); break;
        }
        return (int)TAE_OK;
    });
}
