// tae_selective_scan: h[t] = exp(d[t] A) h[t-1] + d[t] B[t] x[t],  y[t] = (C[t] . h[t] + D x[t]) z[t] sigmoid(z[t]).
#include "turboae_seq.hpp"

namespace tae {
namespace seq {

struct ScanArgs {
    const void *x, *dt, *b, *c, *z;
    const float *a, *d, *dt_bias, *state;
    const int32_t* lengths;
    void* y;
    float* state_out;
    float *steps, *states;                       // workspace: (batch, pieces, channels) sums of d; (batch, pieces + 1, channels, states)
    int64_t x_b, x_r, dt_b, dt_r, b_b, b_r, c_b, c_r, z_b, z_r;
    int len, channels, n, softplus, groups, pieces, piece_len;      // groups of CW channels; pieces of piece_len positions
    int64_t blocks;
};

constexpr int kScanThreads = 256;
constexpr int kTile = 32;                        // positions staged in LDS at once

// P adjacent lanes share a channel, each holds S of its states.  ENDS: only the state behind a piece, started from zero (the first piece: from
// `state`), and the sum of its steps, whose exponential carries a state across the piece.
template <class T, int S, int P, bool ENDS>
__global__ __launch_bounds__(kScanThreads) void selective_scan_kernel(ScanArgs q) {
    constexpr int CW = kScanThreads / P, N = S * P, DS = kTile + 4;
    __shared__ float sd[CW * DS], sx[CW * DS], sb[kTile * N], sc[ENDS ? 1 : kTile * N];
    int64_t id = block_index();
    if (id >= q.blocks) return;
    const int group = (int)(id % q.groups);
    id /= q.groups;
    const int piece = (int)(id % q.pieces);
    const int64_t b = id / q.pieces;
    const int tid = threadIdx.x, ch = tid / P, p = tid % P;
    const int e0 = group * CW, e = e0 + ch, E = q.channels;
    const bool mine = e < E;
    const int n = q.lengths ? min(max(q.lengths[b], 0), q.len) : q.len;
    const int begin = piece * q.piece_len, end = min(begin + q.piece_len, q.len), stop = min(end, n);
    const int last_piece = n > 0 ? (n - 1) / q.piece_len : 0;
    float a2[S], h[S];
#pragma unroll
    for (int s = 0; s < S; ++s) {
        const int k = p * S + s;
        a2[s] = mine && k < q.n ? q.a[(int64_t)e * q.n + k] * kLog2e : 0.0f;
        h[s] = 0.0f;
    }
    float* kept = q.pieces > 1 ? q.states + ((b * (q.pieces + 1)) * E + e) * q.n : nullptr;     // [0]: the start, [k + 1]: behind piece k
    const int64_t kept_step = (int64_t)E * q.n;
    if (mine && piece == 0 && q.state && (ENDS || q.pieces == 1)) {
#pragma unroll
        for (int s = 0; s < S; ++s)
            if (p * S + s < q.n) h[s] = q.state[(b * E + e) * q.n + p * S + s];
    }
    if (ENDS && mine && piece == 0) {            // the start is kept: state_out may be the state
#pragma unroll
        for (int s = 0; s < S; ++s)
            if (p * S + s < q.n) kept[p * S + s] = h[s];
    }
    if (!ENDS && q.pieces > 1 && mine && (stop > begin || piece == last_piece)) {
        if (piece == 0) {
#pragma unroll
            for (int s = 0; s < S; ++s)
                if (p * S + s < q.n) h[s] = kept[p * S + s];
        }
        for (int k = 0; k < piece; ++k) {
            const float sum = q.steps[(b * q.pieces + k) * E + e];
#pragma unroll
            for (int s = 0; s < S; ++s)
                if (p * S + s < q.n) h[s] = __builtin_fmaf(__builtin_amdgcn_exp2f(sum * a2[s]), h[s], kept[(k + 1) * kept_step + p * S + s]);
        }
    }
    float sum = 0.0f;
    const T* x = (const T*)q.x + b * q.x_b;
    const T* dt = (const T*)q.dt + b * q.dt_b;
    const T* bm = (const T*)q.b + b * q.b_b;
    const T* cm = (const T*)q.c + b * q.c_b;
    const T* z = q.z ? (const T*)q.z + b * q.z_b : nullptr;
    T* y = (T*)q.y + b * q.len * (int64_t)E;
    for (int t0 = begin; t0 < (ENDS ? stop : end); t0 += kTile) {
        __syncthreads();
        if (t0 < stop) {
            for (int i = tid; i < kTile * CW; i += kScanThreads) {
                const int t = i / CW, c = i % CW;
                float d = 0.0f, dx = 0.0f;
                if (t0 + t < stop && e0 + c < E) {
                    d = (float)dt[(t0 + t) * q.dt_r + e0 + c] + (q.dt_bias ? q.dt_bias[e0 + c] : 0.0f);
                    if (q.softplus) d = softplus(d);
                    dx = d * (float)x[(t0 + t) * q.x_r + e0 + c];
                }
                sd[c * DS + t] = d;
                sx[c * DS + t] = dx;
            }
            for (int i = tid; i < kTile * N; i += kScanThreads) {
                const int t = i / N, k = i % N;
                const bool in = t0 + t < stop && k < q.n;
                sb[i] = in ? (float)bm[(t0 + t) * q.b_r + k] : 0.0f;
                if constexpr (!ENDS) sc[i] = in ? (float)cm[(t0 + t) * q.c_r + k] : 0.0f;
            }
            __syncthreads();
            // positions behind `stop` have step 0: they keep the state
            for (int t = 0; t < kTile; t += 4) {
                const Pack<float, 4> d4 = load<float, 4>(&sd[ch * DS + t]), x4 = load<float, 4>(&sx[ch * DS + t]);
                float out[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float o = 0.0f;
#pragma unroll
                    for (int s = 0; s < S; ++s) {
                        const float g = __builtin_amdgcn_exp2f(d4.v[i] * a2[s]);
                        h[s] = __builtin_fmaf(g, h[s], x4.v[i] * sb[(t + i) * N + p * S + s]);
                        if constexpr (!ENDS) o = __builtin_fmaf(h[s], sc[(t + i) * N + p * S + s], o);
                    }
                    if constexpr (ENDS) sum += d4.v[i];
                    else out[i] = lanes_sum<P>(o);
                }
                if constexpr (!ENDS) {
                    if (p == 0) store<float, 4>(&sx[ch * DS + t], Pack<float, 4>{out[0], out[1], out[2], out[3]});
                }
            }
        }
        if constexpr (!ENDS) {
            __syncthreads();
            for (int i = tid; i < kTile * CW; i += kScanThreads) {
                const int t = i / CW, c = i % CW, at = t0 + t;
                if (at >= end || e0 + c >= E) continue;
                float o = 0.0f;
                if (at < stop) {
                    o = sx[c * DS + t];
                    if (q.d) o = __builtin_fmaf(q.d[e0 + c], (float)x[at * q.x_r + e0 + c], o);
                    if (z) o *= silu((float)z[at * q.z_r + e0 + c]);
                }
                y[(int64_t)at * E + e0 + c] = (T)o;
            }
        }
    }
    if (!mine) return;
    if constexpr (ENDS) {
#pragma unroll
        for (int s = 0; s < S; ++s)
            if (p * S + s < q.n) kept[(piece + 1) * kept_step + p * S + s] = h[s];
        if (p == 0) q.steps[(b * q.pieces + piece) * E + e] = sum;
    } else if (piece == last_piece) {
#pragma unroll
        for (int s = 0; s < S; ++s)
            if (p * S + s < q.n) q.state_out[(b * E + e) * q.n + p * S + s] = h[s];
    }
}

// How a call is cut: pieces of piece_len positions (a multiple of kTile).
struct ScanPlan {
    int lanes = 1, per_lane = 4, groups = 1, pieces = 1, piece_len = 0;
    size_t steps_bytes = 0, bytes = 0;
};

static bool plan_scan(const tae_scan_args* p, ScanPlan* s) {
    if (p->batch < 1 || p->len < 1 || p->channels < 1 || p->states < 1 || p->states > 64) return false;
    while (s->per_lane * s->lanes < p->states) s->lanes *= 2;
    s->groups = (int)ceil_div(p->channels, kScanThreads / s->lanes);
    const int64_t wgs = (int64_t)p->batch * s->groups;
    int64_t pieces = 1;
    if (wgs < 128) pieces = std::min<int64_t>(ceil_div(256, wgs), ceil_div(p->len, 4 * kTile));
    s->piece_len = (int)(ceil_div(ceil_div(p->len, pieces), kTile) * kTile);
    s->pieces = (int)ceil_div(p->len, s->piece_len);
    if (s->pieces > 1) {
        s->steps_bytes = ((size_t)p->batch * s->pieces * p->channels * 4 + 255) / 256 * 256;
        s->bytes = s->steps_bytes + (size_t)p->batch * (s->pieces + 1) * p->channels * p->states * 4;
    }
    return true;
}

template <class T, int P>
static void launch_scan(const ScanArgs& a, hipStream_t st) {
    if (a.pieces > 1) hipLaunchKernelGGL((selective_scan_kernel<T, 4, P, true>), grid_of(a.blocks), dim3(kScanThreads), 0, st, a);
    hipLaunchKernelGGL((selective_scan_kernel<T, 4, P, false>), grid_of(a.blocks), dim3(kScanThreads), 0, st, a);
}

template <class T>
static void launch_scan_lanes(const ScanArgs& a, int lanes, hipStream_t st) {
    switch (lanes) {
        case 1: launch_scan<T, 1>(a, st); break;
        case 2: launch_scan<T, 2>(a, st); break;
        case 4: launch_scan<T, 4>(a, st); break;
        case 8: launch_scan<T, 8>(a, st); break;
        default: launch_scan<T, 16>(a, st); break;
    }
}

}  // namespace seq
}  // namespace tae

extern "C" {

size_t tae_selective_scan_workspace(const tae_scan_args* p) {
    using namespace tae::seq;
    ScanPlan s;
    if (!p || p->struct_size != (int32_t)sizeof(tae_scan_args) || !plan_scan(p, &s)) return 0;
    return s.bytes;
}

int tae_selective_scan(const tae_scan_args* p, void* stream) {
    using namespace tae;
    using namespace tae::seq;
    if (!p || p->struct_size != (int32_t)sizeof(tae_scan_args)) return fail_msg(TAE_EINVAL, "tae_scan_args: NULL or struct_size mismatch (ABI)");
    if (!dtype_ok(p->dtype)) return fail_msg(TAE_EINVAL, "selective_scan: dtype must be a TAE_DTYPE_* code");
    if (p->states < 1 || p->states > 64) return fail_msg(TAE_EINVAL, "selective_scan: states must be in 1..64");
    if (p->batch < 1 || p->len < 1 || p->channels < 1) return fail_msg(TAE_EINVAL, "selective_scan: batch, len and channels must be >= 1");
    if (p->len > (1 << 30) || p->channels > (1 << 30)) return fail_msg(TAE_EINVAL, "selective_scan: len and channels must be at most 2^30");
    if (!p->x || !p->dt || !p->a || !p->b || !p->c || !p->y || !p->state_out) return fail_msg(TAE_EINVAL, "selective_scan: x, dt, a, b, c, y and state_out must not be NULL");
    ScanPlan s;
    if (!plan_scan(p, &s)) return fail_msg(TAE_EINVAL, "selective_scan: bad sizes");
    if (s.bytes && (!p->workspace || p->workspace_bytes < s.bytes || !aligned(p->workspace, 16)))
        return fail_msg(TAE_EINVAL, "selective_scan: the workspace is missing, misaligned or smaller than tae_selective_scan_workspace");
    ScanArgs a{p->x, p->dt, p->b, p->c, p->z, p->a, p->d, p->dt_bias, p->state, p->lengths, p->y, p->state_out,
               s.bytes ? (float*)p->workspace : nullptr, s.bytes ? (float*)((char*)p->workspace + s.steps_bytes) : nullptr,
               p->x_batch, p->x_row, p->dt_batch, p->dt_row, p->b_batch, p->b_row, p->c_batch, p->c_row, p->z_batch, p->z_row,
               p->len, p->channels, p->states, p->softplus ? 1 : 0, s.groups, s.pieces, s.piece_len, (int64_t)p->batch * s.groups * s.pieces};
    if (a.blocks > ((int64_t)kGridX << 15)) return fail_msg(TAE_EINVAL, "selective_scan: the batch is too large for one call");
    return guarded([&] {
        hipStream_t st = (hipStream_t)stream;
        switch (p->dtype) {
            case TAE_DTYPE_F32: launch_scan_lanes<float>(a, s.lanes, st); break;
            case TAE_DTYPE_F16: launch_scan_lanes<f16>(a, s.lanes, st); break;
            default: launch_scan_lanes<bf16>(a, s.lanes, st); break;
        }
        return (int)TAE_OK;
    });
}

}  // extern "C"
