// tae_causal_conv: y[t] = act(bias + sum_k weight[k] x[t - K + 1 + k]) of each channel, with the last K - 1 inputs as state.
//
// Bound by memory.  A lane owns V adjacent channels and walks a piece of the positions with the window in registers: x is read once, plus the
// K - 1 positions in front of its piece.  Rows are loaded in blocks, the next block while this one is worked on.  Measured, bf16, 4 x 2048 x
// 4096 with 4 taps (134 MB): 32.2 us, 4.2 TB/s; two waves for each SIMD, 66 % of their time issuing (window, products, silu).  Pieces of 16
// positions 38.8 us, of 64 38.2, blocks of eight rows 34.7, workgroups of four waves 33.7, of eight 38.2.  A single position of 64
// sequences x 4096 channels: 4.7 us (workgroups of four waves: 5.8), most of it starting up.
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
    int len, channels, act;
    Divisor groups, pieces;                      // lanes that cover the channels; pieces of the positions
    int64_t lanes;                               // batch * pieces * groups
};

constexpr int kBlock = 4, kBlocks = 8;           // rows loaded together, blocks of a piece (a single position: 1 of each)
constexpr int kThreads = 64;                     // single waves: they spread evenly over the CUs

template <class T, int V, int K, int ROWS, int BLOCKS>
__global__ __launch_bounds__(kThreads) void causal_conv_kernel(ConvArgs a) {
    constexpr int PIECE = ROWS * BLOCKS;
    const int64_t id = block_index() * kThreads + threadIdx.x;
    if (id >= a.lanes) return;
    int64_t rest, b;
    int g, piece;
    a.groups.split(id, rest, g);
    a.pieces.split(rest, b, piece);
    const int e = g * V, t0 = piece * PIECE, E = a.channels;
    const int n = a.lengths ? min(max(a.lengths[b], 0), a.len) : a.len;
    const int steps = min(PIECE, n - t0), total = min(PIECE, a.len - t0);        // valid positions (may be none), all positions
    const T* x = (const T*)a.x + b * a.x_b + e;
    const T* before = a.state ? (const T*)a.state + b * (K - 1) * E + e : nullptr;
    T* y = (T*)a.y + (b * a.len + t0) * E + e;
    float w[K][V], c[V], win[K][V];              // win: the last K inputs, oldest first
#pragma unroll
    for (int v = 0; v < V; ++v) {
        c[v] = a.bias ? a.bias[e + v] : 0.0f;
#pragma unroll
        for (int k = 0; k < K; ++k) w[k][v] = a.weight[(int64_t)(e + v) * K + k];
    }
    Raw<T, V> now[ROWS], next[ROWS];
    auto fetch = [&](Raw<T, V>(&r)[ROWS], int at) {          // rows behind the last valid one repeat it
#pragma unroll
        for (int i = 0; i < ROWS; ++i) r[i].from(x + (int64_t)(t0 + min(at + i, steps - 1)) * a.x_r);
    };
    if (steps > 0) fetch(now, 0);
    // inputs in front of the piece: of the sequence (a later piece starts at least K - 1 positions in), or of the state
    const bool inside = piece > 0 && steps > 0;
    const T* old = inside ? x + (int64_t)(t0 - (K - 1)) * a.x_r : before;
    const int64_t old_r = inside ? a.x_r : E;
#pragma unroll
    for (int k = 0; k < K - 1; ++k) {
        Pack<T, V> p{};
        if (inside || (piece == 0 && before)) p = load<T, V>(old + k * old_r);
#pragma unroll
        for (int v = 0; v < V; ++v) win[k + 1][v] = (float)p.v[v];
    }
#pragma unroll
    for (int block = 0; block < BLOCKS; ++block) {
        const int at = block * ROWS;
        if (at >= total) break;
        if (block + 1 < BLOCKS && at + ROWS < steps) fetch(next, at + ROWS);
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            if (at + i < total) {
                Pack<T, V> out;
#pragma unroll
                for (int v = 0; v < V; ++v) {
#pragma unroll
                    for (int k = 0; k < K - 1; ++k) win[k][v] = win[k + 1][v];
                    win[K - 1][v] = now[i][v];
                    float s = c[v];
#pragma unroll
                    for (int k = 0; k < K; ++k) s = __builtin_fmaf(w[k][v], win[k][v], s);
                    if (a.act == TAE_ACT_SILU) s = silu(s);
                    out.v[v] = (T)(at + i < steps ? s : 0.0f);
                }
                store<T, V>(y + (int64_t)(at + i) * E, out);
            }
        }
        if constexpr (BLOCKS > 1) {
#pragma unroll
            for (int i = 0; i < ROWS; ++i) now[i] = next[i];
        }
    }
    // Only this lane reads the state of these channels, and it has read all of it before it writes: state_out may be the state.
    if (piece == 0 && a.state_out && K > 1) {
        T* o = (T*)a.state_out + b * (K - 1) * E + e;
        Pack<T, V> last[K > 1 ? K - 1 : 1];
#pragma unroll
        for (int j = 0; j < K - 1; ++j) {
            const int i = n + j - (K - 1);
            last[j] = Pack<T, V>{};
            if (i >= 0) last[j] = load<T, V>(x + (int64_t)i * a.x_r);
            else if (before) last[j] = load<T, V>(before + (int64_t)(i + K - 1) * E);
        }
#pragma unroll
        for (int j = 0; j < K - 1; ++j) store<T, V>(o + (int64_t)j * E, last[j]);
    }
}

template <class T, int V, int K>
static void launch_conv_taps(const ConvArgs& a, hipStream_t st) {
    const dim3 grid = grid_of(ceil_div(a.lanes, kThreads));
    if (a.len == 1) hipLaunchKernelGGL((causal_conv_kernel<T, V, K, 1, 1>), grid, dim3(kThreads), 0, st, a);
    else hipLaunchKernelGGL((causal_conv_kernel<T, V, K, kBlock, kBlocks>), grid, dim3(kThreads), 0, st, a);
}

template <class T, int V>
static void launch_conv(const ConvArgs& a, int taps, hipStream_t st) {
    switch (taps) {
        case 1: launch_conv_taps<T, V, 1>(a, st); break;
        case 2: launch_conv_taps<T, V, 2>(a, st); break;
        case 3: launch_conv_taps<T, V, 3>(a, st); break;
        case 4: launch_conv_taps<T, V, 4>(a, st); break;
        case 5: launch_conv_taps<T, V, 5>(a, st); break;
        case 6: launch_conv_taps<T, V, 6>(a, st); break;
        case 7: launch_conv_taps<T, V, 7>(a, st); break;
        default: launch_conv_taps<T, V, 8>(a, st); break;
    }
}

}  // namespace seq
}  // namespace tae

extern "C" int tae_causal_conv(const tae_conv_args* p, void* stream) {
    using namespace tae;
    using namespace tae::seq;
    if (!p || p->struct_size != (int32_t)sizeof(tae_conv_args)) return fail_msg(TAE_EINVAL, "tae_conv_args: NULL or struct_size mismatch (ABI)");
    if (p->reserved) return fail_msg(TAE_EINVAL, "causal_conv: reserved must be 0");
    if (!dtype_ok(p->dtype)) return fail_msg(TAE_EINVAL, "causal_conv: dtype must be a TAE_DTYPE_* code");
    if (p->batch < 1 || p->len < 1 || p->channels < 1) return fail_msg(TAE_EINVAL, "causal_conv: batch, len and channels must be >= 1");
    if (p->len > INT32_MAX - 64 || p->channels > INT32_MAX - 64) return fail_msg(TAE_EINVAL, "causal_conv: len and channels must stay below 2^31 - 64");
    if (p->taps < 1 || p->taps > 8) return fail_msg(TAE_EINVAL, "causal_conv: taps must be in 1..8");
    if (p->act != TAE_ACT_LINEAR && p->act != TAE_ACT_SILU) return fail_msg(TAE_EINVAL, "causal_conv: act must be linear or silu");
    if (!p->x || !p->weight || !p->y) return fail_msg(TAE_EINVAL, "causal_conv: x, weight and y must not be NULL");
    const size_t tb = dtype_bytes(p->dtype);
    if (!elements_aligned(tb, p->x, p->state, p->y, p->state_out) || !elements_aligned(4, p->weight, p->bias, p->lengths))
        return fail_msg(TAE_EINVAL, "causal_conv: a pointer is not aligned to its elements");
    Width w(tb);
    w.elements(p->channels).elements(p->x_batch).elements(p->x_row).pointer(p->x).pointer(p->y).pointer(p->state).pointer(p->state_out);
    const int vec = w.fits(16) ? (int)(16 / tb) : w.fits(4) ? (int)(4 / tb) : 1;
    const int64_t groups = p->channels / vec, pieces = p->len == 1 ? 1 : ceil_div(p->len, kBlock * kBlocks);
    const ConvArgs a{p->x, p->weight, p->bias, p->state, p->lengths, p->y, p->state_out, p->x_batch, p->x_row, p->len, p->channels, p->act,
                     Divisor(groups), Divisor(pieces), p->batch * pieces * groups};
    if (ceil_div(a.lanes, kThreads) > ((int64_t)kGridX << 15)) return fail_msg(TAE_EINVAL, "causal_conv: the batch is too large for one call");
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
