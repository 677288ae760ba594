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
    float *steps, *states;                       // workspace: (batch, pieces, channels) sums of d; (batch, pieces + 1, states, channels)
    int64_t x_b, x_r, dt_b, dt_r, b_b, b_r, c_b, c_r, z_b, z_r;
    int len, channels, n, softplus, gate, pieces, piece_len;       // pieces of piece_len positions
    Divisor by_groups, by_pieces;                                  // groups of channels; pieces
    int64_t blocks;
};

// Elements of a row as they were loaded, in whole registers and taken out only when they are used, so that a load stays in flight until
// then.  V = 4: four adjacent ones, aligned to them; V = 1: four on any element, those of the row's end moved back inside it until `settle`;
// V = 0: one, those behind the row repeat its last.
template <class T, int V>
struct Loaded {
    uint32_t w[V ? sizeof(T) : 1];
    __device__ __forceinline__ static uint32_t one(const T* p) {
        if constexpr (sizeof(T) == 4) return *reinterpret_cast<const uint32_t*>(p);
        else return *reinterpret_cast<const uint16_t*>(p);
    }
    __device__ __forceinline__ void from(const T* row, int at, int width) {
        if constexpr (V == 4 && sizeof(T) == 4) {
            const uint4 u = *reinterpret_cast<const uint4*>(row + min(at, width - 4));
            w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
        } else if constexpr (V == 4) {
            const uint2 u = *reinterpret_cast<const uint2*>(row + min(at, width - 4));
            w[0] = u.x, w[1] = u.y;
        } else if constexpr (V == 1) {
            if (width >= 4) {
                __builtin_memcpy(w, row + min(at, width - 4), 4 * sizeof(T));
            } else if constexpr (sizeof(T) == 4) {
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = one(row + min(at + i, width - 1));
            } else {
#pragma unroll
                for (int i = 0; i < 2; ++i) w[i] = one(row + min(at + 2 * i, width - 1)) | one(row + min(at + 2 * i + 1, width - 1)) << 16;
            }
        } else {
            w[0] = one(row + min(at, width - 1));
        }
    }
    __device__ __forceinline__ void settle(int at, int width) {
        if constexpr (V == 1) {
            if (width >= 4) drop_first<T>(w, min(max(at + 4 - width, 0), 3));
        }
    }
    __device__ __forceinline__ float operator[](int i) const {
        if constexpr (sizeof(T) == 4) {
            return __uint_as_float(w[i]);
        } else {
            const uint32_t u = i & 1 ? w[i / 2] >> 16 : w[i / 2] & 0xFFFFu;
            return (float)__builtin_bit_cast(T, (uint16_t)u);
        }
    }
};

// Sum over the P adjacent lanes of a channel for four positions at once.  Lanes that hold the same sum twice are put to use: in P = 16 the
// first exchange leaves positions 0 | 1 (2 | 3) in the two halves of a row and the second 0, 2, 1, 3 in its four quads - 11 instructions
// instead of 16.  The position whose sum a lane ends up with is `reduced_position`.
template <int CTRL>
__device__ __forceinline__ float dpp_add(float v) { return v + dpp<CTRL>(v); }
template <int CTRL>
__device__ __forceinline__ float dpp_choose(bool second, float v0, float v1) {
    const float a = dpp_add<CTRL>(v0), b = dpp_add<CTRL>(v1);      // by all lanes, before the choice
    return second ? b : a;
}

template <int P>
__device__ __forceinline__ int reduced_position(int lane) {
    if constexpr (P == 16) return ((lane >> 3) & 1) | ((lane >> 1) & 2);
    return (lane >> 2) & 1;                     // P = 8: pairs 0 | 1 and 2 | 3
}

// P lanes share a channel, each holds S of its states (n = s P + p).  A workgroup takes 256 / P channels and walks the positions of its
// piece in tiles of TT: steps d and d x (once for each channel and position), B and C go through LDS as rows over the positions, so that a
// lane reads four positions with one 16-byte load; two buffers, one barrier for each tile; the next tile's loads are in flight meanwhile.
// ENDS: only the state behind a piece, started from zero (the first piece: from `state`), and the sum of its steps, whose exponential
// carries a state across the piece.  V: 4 where rows allow loads of four channels, else 1.  FILLED: some states only fill lanes up.  Their B and C
// are 0, but an infinite step or input makes NaN of them, so they are left out of the sums by choice.
//
// Bound by issuing: with 16 states in P = 8, S = 2 a wave takes 45 ns for a position of its 8 channels, of which 26 are the states' 12 issue
// slots (two products, exp of two slots, two fused) and the rest sums over lanes, LDS, softplus and gate.  More lanes for a channel spread few
// channels over the chip and share softplus and gate, for longer sums over lanes; what each split takes stands at kForms.  Measured, bf16:
// 2048 x 512 channels x 16 states 10 us and 9 for the ends, 8 x 512 x 256 x 64 34 and 17, 256 x 2048 x 16 in one piece 15.
template <class T, int S, int P, int TT, int V, bool ENDS, bool FILLED>
__global__ __launch_bounds__(kScanThreads) void selective_scan_kernel(ScanArgs q) {
    constexpr int CW = kScanThreads / P, N = S * P, DS = TT + 4;
    constexpr int R = TT * CW / 4 / kScanThreads, RB = (TT * N + kScanThreads - 1) / kScanThreads;      // groups of four, elements for each thread
    static_assert(P == 4 || P == 8 || P == 16, "sums over lanes");
    static_assert(R >= 1 && TT * CW % (4 * kScanThreads) == 0, "a tile is whole groups of four for every thread");
    __shared__ float sd[2][CW * DS], sx[2][CW * DS], sb[2][N * DS], sc[ENDS ? 1 : 2][ENDS ? 4 : N * DS], sy[ENDS ? 1 : 2][ENDS ? 4 : CW * DS];
    const int64_t id = block_index();
    if (id >= q.blocks) return;
    int64_t rest, b;
    int group, piece;
    q.by_groups.split(id, rest, group);
    q.by_pieces.split(rest, b, piece);
    if (ENDS && piece + 1 == q.pieces) return;   // nothing starts from there
    const int tid = threadIdx.x, ch = tid / P, p = tid % P;
    const int e0 = group * CW, e = e0 + ch, E = q.channels;
    const bool mine = e < E;
    const int n = q.lengths ? min(max(q.lengths[b], 0), q.len) : q.len;
    const int begin = piece * q.piece_len, end = min(begin + q.piece_len, q.len), stop = min(end, n);
    const int last_piece = n > 0 ? (n - 1) / q.piece_len : 0;
    float a2[S], h[S];
#pragma unroll
    for (int s = 0; s < S; ++s) {
        const int k = s * P + p;
        a2[s] = mine && k < q.n ? q.a[(int64_t)e * q.n + k] * kLog2e : 0.0f;
        h[s] = 0.0f;
    }
    if (mine && (ENDS || q.pieces == 1) && piece == 0 && q.state) {
#pragma unroll
        for (int s = 0; s < S; ++s)
            if (s * P + p < q.n) h[s] = q.state[(b * E + e) * q.n + s * P + p];
    }
    if (!ENDS && mine && q.pieces > 1) {
        const float* kept = q.states + (b * (q.pieces + 1) + piece) * q.n * (int64_t)E + e;
#pragma unroll
        for (int s = 0; s < S; ++s)
            if (s * P + p < q.n) h[s] = kept[(int64_t)(s * P + p) * E];
    }
    float sum = 0.0f;
    const T* x = (const T*)q.x + b * q.x_b;
    const T* dt = (const T*)q.dt + b * q.dt_b;
    const T* bm = (const T*)q.b + b * q.b_b;
    const T* cm = (const T*)q.c + b * q.c_b;
    const T* z = (const T*)q.z + b * q.z_b;          // without a gate: x again, unused
    T* y = (T*)q.y + b * q.len * (int64_t)E;

    using Raw4 = Loaded<T, V>;
    using Raw1 = Loaded<T, 0>;
    constexpr int CQ = CW / 4;
    float bias[4];                               // of this thread's channels: the same four in every group, because CQ divides 256
    const int cq = (tid % CQ) * 4;
#pragma unroll
    for (int i = 0; i < 4; ++i) bias[i] = q.dt_bias && e0 + cq + i < E ? q.dt_bias[e0 + cq + i] : 0.0f;
    float dcoef[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) dcoef[i] = !ENDS && q.d && e0 + cq + i < E ? q.d[e0 + cq + i] : 0.0f;
    // Where this thread's groups of four lie in a tile: rows at or behind `rows` repeat the last one in front of it, as elements behind a row
    // repeat its last ones, so that every load is unconditional and stays in flight until `stage` uses it.
    struct Offsets {
        int64_t x[R], dt[R], z[R], b[RB], c[RB];
    };
    auto offsets = [&](int rows) {
        Offsets o;
#pragma unroll
        for (int j = 0; j < R; ++j) {
            const int64_t t = min((j * kScanThreads + tid) / CQ, rows - 1);
            o.x[j] = t * q.x_r;
            o.dt[j] = t * q.dt_r;
            o.z[j] = t * q.z_r;
        }
#pragma unroll
        for (int j = 0; j < RB; ++j) {
            const int64_t t = min((j * kScanThreads + tid) / N, rows - 1);
            o.b[j] = t * q.b_r;
            o.c[j] = t * q.c_r;
        }
        return o;
    };
    struct Raw {
        Raw4 x[R], dt[R], z[R];
        Raw1 b[RB], c[RB];
    };
    Offsets off;
    auto fetch = [&](Raw& r, int t0) {
        if (t0 + TT > stop) off = offsets(stop - t0);        // the last one
        const int64_t t = t0;
#pragma unroll
        for (int j = 0; j < R; ++j) {
            r.x[j].from(x + t * q.x_r + off.x[j], e0 + cq, E);
            r.dt[j].from(dt + t * q.dt_r + off.dt[j], e0 + cq, E);
            if constexpr (!ENDS) r.z[j].from(z + t * q.z_r + off.z[j], e0 + cq, E);
        }
#pragma unroll
        for (int j = 0; j < RB; ++j) {
            const int k = (j * kScanThreads + tid) % N;
            r.b[j].from(bm + t * q.b_r + off.b[j], k, q.n);
            if constexpr (!ENDS) r.c[j].from(cm + t * q.c_r + off.c[j], k, q.n);
        }
    };
    // positions at or behind `stop` get step 0: they keep the state.  What was repeated is replaced, not multiplied by 0: it may be infinite
    auto stage = [&](Raw& r, int t0, int buf) {
#pragma unroll
        for (int j = 0; j < R; ++j) {
            r.x[j].settle(e0 + cq, E);
            r.dt[j].settle(e0 + cq, E);
            if constexpr (!ENDS) r.z[j].settle(e0 + cq, E);
            const int t = (j * kScanThreads + tid) / CQ;
            const bool in = t0 + t < stop;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float d = r.dt[j][i] + bias[i];
                if (q.softplus) d = softplus(d);
                const float dx = d * r.x[j][i];
                sd[buf][(cq + i) * DS + t] = in ? d : 0.0f;
                sx[buf][(cq + i) * DS + t] = in ? dx : 0.0f;
            }
        }
#pragma unroll
        for (int j = 0; j < RB; ++j) {
            const int i = j * kScanThreads + tid, t = i / N, k = i % N;
            if (TT * N % kScanThreads == 0 || i < TT * N) {
                const bool in = t0 + t < stop && k < q.n;
                sb[buf][k * DS + t] = in ? r.b[j][0] : 0.0f;
                if constexpr (!ENDS) sc[buf][k * DS + t] = in ? r.c[j][0] : 0.0f;
            }
        }
    };
    const int first = begin, behind = ENDS ? stop : end;
    Raw now, next;
    int tile = 0;
    // what the loop uses has arrived before it: a wait inside would wait for the loads in flight too
#pragma unroll
    for (int s = 0; s < S; ++s) asm volatile("" : "+v"(h[s]), "+v"(a2[s]));
#pragma unroll
    for (int i = 0; i < 4; ++i) asm volatile("" : "+v"(bias[i]), "+v"(dcoef[i]));
    if (first < stop) {
        off = offsets(TT);
        fetch(now, first);
        stage(now, first, 0);
        __syncthreads();
    }
    for (int t0 = first; t0 < behind; t0 += TT, ++tile) {
        const int buf = tile & 1;
        const bool more = t0 + TT < stop;
        if (more) fetch(next, t0 + TT);
        if (t0 < stop) {
            const float* pd = &sd[buf][ch * DS];
            const float* px = &sx[buf][ch * DS];
            Pack<float, 4> d4 = load<float, 4>(pd), x4 = load<float, 4>(px), b4[S], c4[S];
#pragma unroll
            for (int s = 0; s < S; ++s) {
                b4[s] = load<float, 4>(&sb[buf][(s * P + p) * DS]);
                if constexpr (!ENDS) c4[s] = load<float, 4>(&sc[buf][(s * P + p) * DS]);
            }
            auto four = [&](int t) {
                // the next four positions' operands are read while these are worked on (at the last, four floats of padding)
                const Pack<float, 4> dn = load<float, 4>(pd + t + 4), xn = load<float, 4>(px + t + 4);
                Pack<float, 4> bn[S], cn[S];
#pragma unroll
                for (int s = 0; s < S; ++s) {
                    bn[s] = load<float, 4>(&sb[buf][(s * P + p) * DS + t + 4]);
                    if constexpr (!ENDS) cn[s] = load<float, 4>(&sc[buf][(s * P + p) * DS + t + 4]);
                }
                float out[4];
#pragma unroll
                for (int s = 0; s < S; ++s) {
                    float at[4];                 // the state behind each position
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float g = __builtin_amdgcn_exp2f(d4.v[i] * a2[s]);
                        at[i] = h[s] = __builtin_fmaf(g, h[s], x4.v[i] * b4[s].v[i]);
                        if (!ENDS && (!FILLED || S == 1 || 2 * s < S)) out[i] = s == 0 ? at[i] * c4[s].v[i] : __builtin_fmaf(at[i], c4[s].v[i], out[i]);
                    }
                    if constexpr (!ENDS && FILLED) {
                        if constexpr (S == 1) {
#pragma unroll
                            for (int i = 0; i < 4; ++i) out[i] = p < q.n ? out[i] : 0.0f;
                        } else if (2 * s >= S) {         // more than half of all states are in use
                            if (s * P + p < q.n) {
                                asm volatile("");            // a branch: with four choices 50 x 410 x 480 x 12 takes 57 us, so 54
#pragma unroll
                                for (int i = 0; i < 4; ++i) out[i] = __builtin_fmaf(at[i], c4[s].v[i], out[i]);
                            }
                        }
                    }
                }
                if constexpr (ENDS) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) sum += d4.v[i];
                } else {
                    float* py = &sy[buf][ch * DS + t];
                    if constexpr (P == 16) {
                        const bool up8 = (tid & 8) != 0, up4 = (tid & 4) != 0;
                        const float a = dpp_choose<kRor8>(up8, out[0], out[1]), c = dpp_choose<kRor8>(up8, out[2], out[3]);
                        const float v = dpp_choose<kHalfMirror>(up4, a, c);
                        py[reduced_position<16>(tid)] = dpp_add<kXor2>(dpp_add<kXor1>(v));
                    } else if constexpr (P == 8) {
                        const bool up4 = (tid & 4) != 0;
                        const float a = dpp_choose<kHalfMirror>(up4, out[0], out[1]), c = dpp_choose<kHalfMirror>(up4, out[2], out[3]);
                        py[reduced_position<8>(tid)] = dpp_add<kXor2>(dpp_add<kXor1>(a));
                        py[2 + reduced_position<8>(tid)] = dpp_add<kXor2>(dpp_add<kXor1>(c));
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            out[i] = dpp_add<kXor1>(out[i]);
                            out[i] = dpp_add<kXor2>(out[i]);
                        }
                        store<float, 4>(py, Pack<float, 4>{out[0], out[1], out[2], out[3]});
                    }
                }
                d4 = dn;
                x4 = xn;
#pragma unroll
                for (int s = 0; s < S; ++s) {
                    b4[s] = bn[s];
                    if constexpr (!ENDS) c4[s] = cn[s];
                }
            };
            if (stop - t0 >= TT) {
#pragma unroll 4
                for (int t = 0; t < TT; t += 4) four(t);
            } else {                             // no more than there are, rounded up: steps behind them are 0
#pragma unroll 1
                for (int t = 0; t < stop - t0; t += 4) four(t);
            }
        }
        if (more) stage(next, t0 + TT, buf ^ 1);
        __syncthreads();
        if constexpr (!ENDS) {
#pragma unroll
            for (int j = 0; j < R; ++j) {
                const int tt = (j * kScanThreads + tid) / CQ, at = t0 + tt;
                if (at >= end || e0 + cq >= E) continue;
                Pack<T, 4> o;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float v = 0.0f;
                    if (at < stop) {
                        v = sy[buf][(cq + i) * DS + tt];
                        if (q.d) v = __builtin_fmaf(dcoef[i], now.x[j][i], v);         // not 0 times an infinite x
                        if (q.gate) v *= silu(now.z[j][i]);
                    }
                    o.v[i] = (T)v;
                }
                T* to = y + (int64_t)at * E + e0 + cq;
                if constexpr (V == 4) {
                    store<T, 4>(to, o);
                } else if (e0 + cq + 4 <= E) {
                    store_any(to, o);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (e0 + cq + i < E) to[i] = o.v[i];
                }
            }
        }
        now = next;
    }
    if (!mine) return;
    if constexpr (ENDS) {
#pragma unroll
        for (int s = 0; s < S; ++s)
            if (s * P + p < q.n) q.states[((b * (q.pieces + 1) + piece + 1) * q.n + s * P + p) * E + e] = h[s];
        if (p == 0) q.steps[(b * q.pieces + piece) * E + e] = sum;
    } else if (piece == last_piece) {
#pragma unroll
        for (int s = 0; s < S; ++s)
            if (s * P + p < q.n) q.state_out[(b * E + e) * q.n + s * P + p] = h[s];
    }
}

// A lane owns a channel with its N states; a wave walks the positions of its piece by itself.  B[t] and C[t] are the same for all channels and
// come from LDS, so that a state costs five instructions (two products, exp, two fused) and no sum crosses lanes.  All loads are kAhead
// positions ahead; each wave has LDS of its own, so no barrier is needed.
//
// Bound by issuing: 119 vector instructions (20 of them exp, log and rcp at half rate) for each position of 64 channels with 16 states.
// Eight waves make a workgroup so that they are dealt out evenly over a CU's SIMDs, two each (waves w and w + 4), and know of each other:
// left alone the older of two gets most of the issue slots and the younger runs by itself at the end, at half the rate (61 and 83 us of a
// wave's life where both should take 72).  So whichever has more positions left goes first.  Measured, bf16, 4096 positions x 4096 channels
// x 16 states in 32 pieces: 90 us, ends pass 65 (four waves, no priorities: 90 and 68); fp32, 500 x 100 x 200 x 16: 48 (57).  More pieces,
// so more waves, are no faster (48: 94 + 69, 64: 92 + 71), fewer are slower (16: 129 + 84).  FILLED: as above.
constexpr int kAhead = 8;

template <class T, int N, bool ENDS, bool FILLED>
__global__ __launch_bounds__(kLaneWaves * 64) void scan_lane_kernel(ScanArgs q) {
    constexpr int W = ENDS ? N : 2 * N, RB = (kAhead * W + 63) / 64;       // values of B (and C) for each position; loads of each lane
    __shared__ alignas(16) float lds[kLaneWaves][2][kAhead * W];
    __shared__ int left[kLaneWaves];    // positions; read without a barrier, for priorities only
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    auto report = [&](int positions) { if ((threadIdx.x & 63) == 0) __hip_atomic_store(&left[wave], positions, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP); };
    report(0);
    float(*rows)[kAhead * W] = lds[wave];
    const int64_t id = block_index() * (kLaneWaves) + wave;
    if (id >= q.blocks) return;
    int64_t rest, b;
    int group, piece;
    q.by_groups.split(id, rest, group);
    q.by_pieces.split(rest, b, piece);
    if (ENDS && piece + 1 == q.pieces) return;   // nothing starts from there
    const int lane = threadIdx.x & 63, E = q.channels, e = group * 64 + lane, ec = min(e, E - 1);
    const bool mine = e < E;
    const int n = q.lengths ? min(max(q.lengths[b], 0), q.len) : q.len;
    const int begin = piece * q.piece_len, end = min(begin + q.piece_len, q.len), stop = min(end, n);
    const int last_piece = n > 0 ? (n - 1) / q.piece_len : 0;
    float a2[N], h[N];
    const float* start = ENDS || q.pieces == 1 ? (piece == 0 ? q.state : nullptr) : nullptr;
    const float* kept = q.pieces > 1 ? q.states + ((b * (q.pieces + 1) + piece) * q.n) * E + ec : nullptr;
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const int kc = min(k, q.n - 1);
        const bool real = k < q.n;
        a2[k] = real ? q.a[(int64_t)ec * q.n + kc] * kLog2e : 0.0f;
        h[k] = 0.0f;
        if (start) h[k] = real ? start[(b * E + ec) * q.n + kc] : 0.0f;
        if (!ENDS && kept) h[k] = real ? kept[(int64_t)kc * E] : 0.0f;
    }
    const float bias = q.dt_bias ? q.dt_bias[ec] : 0.0f, dcoef = !ENDS && q.d ? q.d[ec] : 0.0f;
    float sum = 0.0f;
    const T* x = (const T*)q.x + b * q.x_b;
    const T* dt = (const T*)q.dt + b * q.dt_b;
    const T* z = (const T*)q.z + b * q.z_b;
    const T* bm = (const T*)q.b + b * q.b_b;
    const T* cm = (const T*)q.c + b * q.c_b;
    T* y = (T*)q.y + b * q.len * (int64_t)E;
    struct Raw {
        Loaded<T, 0> x[kAhead], dt[kAhead], z[kAhead], bc[RB];
    };
    auto fetch = [&](Raw& r, int t0) {           // rows at or behind `stop` repeat the last one in front of it
        const T *px = x + t0 * q.x_r, *pd = dt + t0 * q.dt_r, *pz = z + t0 * q.z_r;
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            r.x[i].from(px, ec, E);
            r.dt[i].from(pd, ec, E);
            if constexpr (!ENDS) {
                if (q.gate) r.z[i].from(pz, ec, E);
            }
            if (t0 + i + 1 < stop) {
                px += q.x_r;
                pd += q.dt_r;
                pz += q.z_r;
            }
        }
#pragma unroll
        for (int j = 0; j < RB; ++j) {
            const int i = j * 64 + lane, k = i % N;
            const int64_t t = min(t0 + min(i / W, kAhead - 1), stop - 1);
            const T* row = !ENDS && i / N % 2 ? cm + t * q.c_r : bm + t * q.b_r;
            r.bc[j].from(row, k, q.n);
        }
    };
    // Lanes read what others of the wave wrote.  Its LDS instructions are carried out in the order of the program; the fences, no instructions
    // themselves, keep that order the one written here: reads of this buffer's last use, writes, reads.
    auto stage = [&](const Raw& r, int buf) {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int j = 0; j < RB; ++j) {
            const int i = j * 64 + lane;
            if (kAhead * W % 64 == 0 || i < kAhead * W) rows[buf][i] = i % N < q.n ? r.bc[j][0] : 0.0f;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    };
    Raw now, next;
#pragma unroll
    for (int k = 0; k < N; ++k) asm volatile("" : "+v"(h[k]), "+v"(a2[k]));
    // `count` positions from t0 on: steps and gates first, then the states without a branch between positions, then the results
    auto block = [&](int t0, int count, int buf) {
        float d[kAhead], dx[kAhead], out[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) d[i] = now.dt[i][0] + bias;
        if (q.softplus) {
#pragma unroll
            for (int i = 0; i < kAhead; ++i) d[i] = softplus(d[i]);
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const float xv = now.x[i][0];
            dx[i] = d[i] * xv;
            out[i] = q.d ? dcoef * xv : 0.0f;    // not 0 times an infinite x
            if constexpr (ENDS) sum += i < count ? d[i] : 0.0f;
        }
        // G states at a time: their products, exps, products and fused adds each as G instructions in a row, so that none waits for the one in
        // front of it; the next group's B and C are read meanwhile.  The fences keep the compiler from mixing them again.
        constexpr int G = N < 8 ? N : 8, GROUPS = N / G;
        float bv[2][G], cv[2][G];
        auto read = [&](int at, int to) {
            const float* row = &rows[buf][at / GROUPS * W + at % GROUPS * G];
#pragma unroll
            for (int k = 0; k < G; k += 4) {
                const Pack<float, 4> p = load<float, 4>(row + k);
#pragma unroll
                for (int c = 0; c < 4; ++c) bv[to][k + c] = p.v[c];
                if constexpr (!ENDS) {
                    const Pack<float, 4> r = load<float, 4>(row + N + k);
#pragma unroll
                    for (int c = 0; c < 4; ++c) cv[to][k + c] = r.v[c];
                }
            }
        };
        read(0, 0);
#pragma unroll
        for (int at = 0; at < kAhead * GROUPS; ++at) {
            const int i = at / GROUPS, k0 = at % GROUPS * G;
            if (i >= count) break;
            if (at + 1 < kAhead * GROUPS) read(at + 1, (at + 1) & 1);
            float g[G], u[G];
#pragma unroll
            for (int k = 0; k < G; ++k) g[k] = d[i] * a2[k0 + k];
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int k = 0; k < G; ++k) g[k] = __builtin_amdgcn_exp2f(g[k]);
#pragma unroll
            for (int k = 0; k < G; ++k) u[k] = dx[i] * bv[at & 1][k];
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int k = 0; k < G; ++k) h[k0 + k] = __builtin_fmaf(g[k], h[k0 + k], u[k]);
            if constexpr (!ENDS) {
#pragma unroll
                for (int k = 0; k < (FILLED && k0 ? G / 2 : G); ++k)
                    if (!FILLED || k0 + k <= N / 2 || k0 + k < q.n) out[i] = __builtin_fmaf(h[k0 + k], cv[at & 1][k], out[i]);      // more than half are in use
                if (FILLED && k0 && k0 + G / 2 < q.n) {
                    asm volatile("");            // a branch for all lanes: up to 12 states pay three choices and save four products
#pragma unroll
                    for (int k = G / 2; k < G; ++k)
                        if (k0 + k < q.n) out[i] = __builtin_fmaf(h[k0 + k], cv[at & 1][k], out[i]);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (!ENDS) {
            if (q.gate) {
#pragma unroll
                for (int i = 0; i < kAhead; ++i) out[i] *= silu(now.z[i][0]);
            }
            if (mine) {
#pragma unroll
                for (int i = 0; i < kAhead; ++i)
                    if (i < count) y[(int64_t)(t0 + i) * E + e] = (T)out[i];
            }
        }
    };
    int buf = 0;
    if (begin < stop) {
        fetch(now, begin);
        stage(now, 0);
    }
    int t0 = begin;
    for (; t0 + kAhead <= stop; t0 += kAhead) {
        const bool more = t0 + kAhead < stop;
        report(stop - t0);
        if (__builtin_amdgcn_readfirstlane(__hip_atomic_load(&left[wave ^ 4], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP)) < stop - t0) __builtin_amdgcn_s_setprio(1);
        else __builtin_amdgcn_s_setprio(0);
        if (more) fetch(next, t0 + kAhead);
        block(t0, kAhead, buf);
        if (more) stage(next, buf ^ 1);
        buf ^= 1;
        now = next;
    }
    if (t0 < stop) block(t0, stop - t0, buf);
    if (!mine) return;
    if constexpr (ENDS) {
        float* to = q.states + ((b * (q.pieces + 1) + piece + 1) * q.n) * E + e;
#pragma unroll
        for (int k = 0; k < N; ++k)
            if (k < q.n) to[(int64_t)k * E] = h[k];
        q.steps[(b * q.pieces + piece) * E + e] = sum;
    } else {
        for (int t = max(begin, stop); t < end; ++t) y[(int64_t)t * E + e] = (T)0.0f;
        if (piece == last_piece) {
#pragma unroll
            for (int k = 0; k < N; ++k)
                if (k < q.n) q.state_out[(b * E + e) * q.n + k] = h[k];
        }
    }
}

// The state in front of every piece from those behind them: slot k of `states` holds what piece k - 1 left (slot 0 nothing yet), and gets
// what piece k starts from.  The first piece has started from `state`.  One lane for a state; bound by waiting for its loads, 8 pieces at a
// time (7.1 us for 32 pieces of 65536 states; 16 or 32 at a time the same).
__global__ __launch_bounds__(kScanThreads) void scan_join_kernel(ScanArgs q, int64_t count) {
    const int64_t i = block_index() * kScanThreads + threadIdx.x;
    if (i >= count) return;
    const int E = q.channels, e = (int)(i % E), k = (int)(i / E % q.n);
    const int64_t b = i / E / q.n, step = (int64_t)E * q.n;
    const float a2 = q.a[(int64_t)e * q.n + k] * kLog2e;
    float* slot = q.states + (b * (q.pieces + 1) * q.n + k) * E + e;
    const float* sums = q.steps + b * q.pieces * E + e;
    float h = q.state ? q.state[(b * E + e) * q.n + k] : 0.0f;
    slot[0] = h;
    h = slot[step];
    constexpr int A = 8;
    for (int j0 = 1; j0 < q.pieces; j0 += A) {
        float sum[A], part[A];
#pragma unroll
        for (int j = 0; j < A; ++j) {
            const int64_t at = min(j0 + j, q.pieces - 1);
            sum[j] = sums[at * E];
            part[j] = slot[(at + 1) * step];
        }
#pragma unroll
        for (int j = 0; j < A; ++j) {
            if (j0 + j < q.pieces) {
                slot[(j0 + j) * step] = h;
                // by its root twice: the whole factor may be infinite (a growing state) where its product is not; a state of 0 stays one.  A root
                // of finite steps is 2^-126 at least: 2^-252 of a state is nothing, but an infinite one, which no position makes finite, stays one
                const float exponent = 0.5f * sum[j] * a2;
                const float root = __builtin_amdgcn_exp2f(exponent < -126.0f && exponent > -__builtin_inff() ? -126.0f : exponent);
                h = h == 0.0f ? part[j] : __builtin_fmaf(root, root * h, part[j]);
            }
        }
    }
}

// One position: bound by reading and writing the states.  P lanes share a channel, each holds V adjacent states; they keep A in registers
// for EACH sequences, whose operands are all on their way before the first is worked on.  Measured, bf16, 64 sequences x 4096 channels x 16
// states (36 MB): 9.8 us, 3.7 TB/s with start and drain (against one sequence at a time whole calls took 17 instead of 21 us).
template <class T, int P, int V, int EACH>
__global__ __launch_bounds__(kScanThreads) void scan_step_kernel(ScanArgs q, int batch) {
    constexpr int CW = kScanThreads / P;
    const int64_t id = block_index();
    if (id >= q.blocks) return;
    int64_t row;
    int group;
    q.by_groups.split(id, row, group);
    const int tid = threadIdx.x, p = tid % P, e = group * CW + tid / P, E = q.channels, b0 = (int)row * EACH;
    const int k = p * V;                         // V = 4: states are whole groups of four
    const int ec = min(e, E - 1), kc = min(k, q.n - V);      // lanes without a channel or a state stay for the sums over lanes
    const bool mine = e < E && k < q.n;
    const Pack<float, V> a = load<float, V>(q.a + (int64_t)ec * q.n + kc);
    const float bias = q.dt_bias ? q.dt_bias[ec] : 0.0f, dcoef = q.d ? q.d[ec] : 0.0f;
    Pack<float, V> h[EACH];
    Raw<T, 1> x[EACH], dt[EACH], z[EACH];
    Raw<T, V> bm[EACH], cm[EACH];
    bool on[EACH];
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        const int64_t b = min(b0 + i, batch - 1);
        on[i] = !q.lengths || q.lengths[b] > 0;
        if (q.state) h[i] = load<float, V>(q.state + (b * E + ec) * q.n + kc);
        else h[i] = Pack<float, V>{};
        if (on[i]) {                             // what is padding is not read
            x[i].from((const T*)q.x + b * q.x_b + ec);
            dt[i].from((const T*)q.dt + b * q.dt_b + ec);
            z[i].from((const T*)q.z + b * q.z_b + ec);
            bm[i].from_any((const T*)q.b + b * q.b_b + kc);
            cm[i].from_any((const T*)q.c + b * q.c_b + kc);
        }
    }
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        const int64_t b = b0 + i;
        float out = 0.0f;
        if (on[i]) {
            float d = dt[i][0] + bias;
            if (q.softplus) d = softplus(d);
            const float dx = d * x[i][0];
#pragma unroll
            for (int j = 0; j < V; ++j) {
                h[i].v[j] = __builtin_fmaf(__builtin_amdgcn_exp2f(d * (a.v[j] * kLog2e)), h[i].v[j], dx * bm[i][j]);
                if (mine) out = __builtin_fmaf(h[i].v[j], cm[i][j], out);
            }
            out = lanes_sum<P>(out);
            if (q.d) out = __builtin_fmaf(dcoef, x[i][0], out);
            if (q.gate) out *= silu(z[i][0]);
        }
        if (b < batch && e < E) {
            if (p == 0) ((T*)q.y)[b * E + e] = (T)out;
            if (mine) store<float, V>(q.state_out + (b * E + e) * q.n + k, h[i]);
        }
    }
}

template <class T, int V, int EACH>
static int launch_step(ScanArgs a, int batch, hipStream_t st) {
    const int lanes = state_lanes(a.n, V);
    const int64_t groups = ceil_div(a.channels, kScanThreads / lanes);
    a.by_groups = Divisor(groups);
    a.blocks = groups * ceil_div(batch, EACH);
    if (a.blocks > ((int64_t)kGridX << 15)) return fail_msg(TAE_EINVAL, "selective_scan: the batch is too large for one call");
    const dim3 grid = grid_of(a.blocks), block(kScanThreads);
    switch (lanes) {
        case 1: hipLaunchKernelGGL((scan_step_kernel<T, 1, V, EACH>), grid, block, 0, st, a, batch); break;
        case 2: hipLaunchKernelGGL((scan_step_kernel<T, 2, V, EACH>), grid, block, 0, st, a, batch); break;
        case 4: hipLaunchKernelGGL((scan_step_kernel<T, 4, V, EACH>), grid, block, 0, st, a, batch); break;
        case 8: hipLaunchKernelGGL((scan_step_kernel<T, 8, V, EACH>), grid, block, 0, st, a, batch); break;
        case 16: hipLaunchKernelGGL((scan_step_kernel<T, 16, V, EACH>), grid, block, 0, st, a, batch); break;
        case 32: hipLaunchKernelGGL((scan_step_kernel<T, 32, V, EACH>), grid, block, 0, st, a, batch); break;
        default: hipLaunchKernelGGL((scan_step_kernel<T, 64, V, EACH>), grid, block, 0, st, a, batch); break;
    }
    return TAE_OK;
}

template <class T, int V>
static int launch_steps(const ScanArgs& a, int batch, hipStream_t st) {
    return step_sequences(batch, a.channels, a.n, V) == 4 ? launch_step<T, V, 4>(a, batch, st) : launch_step<T, V, 1>(a, batch, st);
}

// Few positions: as one position, P lanes for a channel with V adjacent states each, and all operands straight from memory, kNear positions
// ahead: no tile to fill, no LDS that few workgroups of a CU share.  Measured, bf16, against the tiles: 100 sequences x 2048 channels x 16
// states 14 us for 2 positions (33), 30 for 12 (37), 99 for 50 (87); x 64 states 36 for 2 (225), 172 for 24 (317); one sequence x 4096 x 16
// 6 to 14 us up to 12 positions (7 to 9), 12 for 24 (7).
constexpr int kNear = 4;

template <class T, int P, int V>
__global__ __launch_bounds__(kScanThreads) void scan_short_kernel(ScanArgs q) {
    constexpr int CW = kScanThreads / P;
    const int64_t id = block_index();
    if (id >= q.blocks) return;
    int64_t b;
    int group;
    q.by_groups.split(id, b, group);
    const int tid = threadIdx.x, p = tid % P, E = q.channels, e = group * CW + tid / P, ec = min(e, E - 1), k = p * V, kc = min(k, q.n - V);
    const bool mine = e < E && k < q.n;
    const int n = q.lengths ? min(max(q.lengths[b], 0), q.len) : q.len;
    const float bias = q.dt_bias ? q.dt_bias[ec] : 0.0f, dcoef = q.d ? q.d[ec] : 0.0f;
    Pack<float, V> a = load<float, V>(q.a + (int64_t)ec * q.n + kc), h{};
    if (q.state) h = load<float, V>(q.state + (b * E + ec) * q.n + kc);
#pragma unroll
    for (int j = 0; j < V; ++j) a.v[j] *= kLog2e;
    const T* x = (const T*)q.x + b * q.x_b + ec;
    const T* dt = (const T*)q.dt + b * q.dt_b + ec;
    const T* z = (const T*)q.z + b * q.z_b + ec;
    const T* bm = (const T*)q.b + b * q.b_b + kc;
    const T* cm = (const T*)q.c + b * q.c_b + kc;
    T* y = (T*)q.y + b * q.len * (int64_t)E + e;
    struct Rows {
        Raw<T, 1> x[kNear], dt[kNear], z[kNear];
        Raw<T, V> b[kNear], c[kNear];
    } now, next;
    auto fetch = [&](Rows& r, int t0) {          // rows behind the last valid one repeat it
#pragma unroll
        for (int i = 0; i < kNear; ++i) {
            const int64_t t = min(t0 + i, n - 1);
            r.x[i].from(x + t * q.x_r);
            r.dt[i].from(dt + t * q.dt_r);
            if (q.gate) r.z[i].from(z + t * q.z_r);
            r.b[i].from_any(bm + t * q.b_r);
            r.c[i].from_any(cm + t * q.c_r);
        }
    };
    if (n > 0) fetch(now, 0);
    for (int t0 = 0; t0 < n; t0 += kNear) {
        if (t0 + kNear < n) fetch(next, t0 + kNear);
#pragma unroll
        for (int i = 0; i < kNear; ++i) {
            if (t0 + i >= n) break;
            float d = now.dt[i][0] + bias, out = 0.0f;
            if (q.softplus) d = softplus(d);
            const float dx = d * now.x[i][0];
#pragma unroll
            for (int j = 0; j < V; ++j) {
                h.v[j] = __builtin_fmaf(__builtin_amdgcn_exp2f(d * a.v[j]), h.v[j], dx * now.b[i][j]);
                if (mine) out = __builtin_fmaf(h.v[j], now.c[i][j], out);
            }
            out = lanes_sum<P>(out);
            if (q.d) out = __builtin_fmaf(dcoef, now.x[i][0], out);
            if (q.gate) out *= silu(now.z[i][0]);
            if (p == 0 && e < E) y[(int64_t)(t0 + i) * E] = (T)out;
        }
        now = next;
    }
    if (e < E) {
        for (int t = n + p; t < q.len; t += P) y[(int64_t)t * E] = (T)0.0f;
        if (mine) store<float, V>(q.state_out + (b * E + e) * q.n + k, h);
    }
}

template <class T, int V>
static int launch_short(ScanArgs a, int64_t batch, hipStream_t st) {
    const int lanes = state_lanes(a.n, V);
    const int64_t groups = ceil_div(a.channels, kScanThreads / lanes);
    a.by_groups = Divisor(groups);
    a.blocks = groups * batch;
    if (a.blocks > ((int64_t)kGridX << 15)) return fail_msg(TAE_EINVAL, "selective_scan: the batch is too large for one call");
    const dim3 grid = grid_of(a.blocks), block(kScanThreads);
    switch (lanes) {
        case 1: hipLaunchKernelGGL((scan_short_kernel<T, 1, V>), grid, block, 0, st, a); break;
        case 2: hipLaunchKernelGGL((scan_short_kernel<T, 2, V>), grid, block, 0, st, a); break;
        case 4: hipLaunchKernelGGL((scan_short_kernel<T, 4, V>), grid, block, 0, st, a); break;
        case 8: hipLaunchKernelGGL((scan_short_kernel<T, 8, V>), grid, block, 0, st, a); break;
        case 16: hipLaunchKernelGGL((scan_short_kernel<T, 16, V>), grid, block, 0, st, a); break;
        case 32: hipLaunchKernelGGL((scan_short_kernel<T, 32, V>), grid, block, 0, st, a); break;
        default: hipLaunchKernelGGL((scan_short_kernel<T, 64, V>), grid, block, 0, st, a); break;
    }
    return TAE_OK;
}

static void launch_join(const ScanArgs& a, int64_t batch, hipStream_t st) {
    const int64_t count = batch * a.n * a.channels;
    hipLaunchKernelGGL(scan_join_kernel, grid_of(ceil_div(count, kScanThreads)), dim3(kScanThreads), 0, st, a, count);
}

template <class T, int S, int P, int TT, int V>
static void launch_scan_as(const ScanArgs& a, int64_t batch, hipStream_t st) {
    if (a.pieces > 1) {
        hipLaunchKernelGGL((selective_scan_kernel<T, S, P, TT, V, true, false>), grid_of(a.blocks), dim3(kScanThreads), 0, st, a);
        launch_join(a, batch, st);
    }
    if (a.n == S * P) hipLaunchKernelGGL((selective_scan_kernel<T, S, P, TT, V, false, false>), grid_of(a.blocks), dim3(kScanThreads), 0, st, a);
    else hipLaunchKernelGGL((selective_scan_kernel<T, S, P, TT, V, false, true>), grid_of(a.blocks), dim3(kScanThreads), 0, st, a);
}

template <class T, int S, int P, int TT>
static int launch_scan(const ScanArgs& a, bool vector, int64_t batch, hipStream_t st) {
    vector ? launch_scan_as<T, S, P, TT, 4>(a, batch, st) : launch_scan_as<T, S, P, TT, 1>(a, batch, st);
    return TAE_OK;
}

template <class T, int N>
static int launch_lane(const ScanArgs& a, int64_t batch, hipStream_t st) {
    const dim3 grid = grid_of(ceil_div(a.blocks, kLaneWaves)), block(kLaneWaves * 64);
    if (a.pieces > 1) {
        hipLaunchKernelGGL((scan_lane_kernel<T, N, true, false>), grid, block, 0, st, a);
        launch_join(a, batch, st);
    }
    if (a.n == N) hipLaunchKernelGGL((scan_lane_kernel<T, N, false, false>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((scan_lane_kernel<T, N, false, true>), grid, block, 0, st, a);
    return TAE_OK;
}

template <class T>
static int launch_scan_plan(const ScanArgs& a, const ScanPlan& s, bool v, int batch, hipStream_t st) {
    if (a.len == 1) return v ? launch_steps<T, 4>(a, batch, st) : launch_steps<T, 1>(a, batch, st);
    if (s.lanes == 0) return v ? launch_short<T, 4>(a, batch, st) : launch_short<T, 1>(a, batch, st);
    switch (s.lanes * 100 + s.per_lane) {
        case 116: return launch_lane<T, 16>(a, batch, st);
        case 401: return launch_scan<T, 1, 4, 32>(a, v, batch, st);
        case 801: return launch_scan<T, 1, 8, 32>(a, v, batch, st);
        case 802: return launch_scan<T, 2, 8, 32>(a, v, batch, st);
        case 804: return launch_scan<T, 4, 8, 32>(a, v, batch, st);
        case 1601: return launch_scan<T, 1, 16, 64>(a, v, batch, st);
        case 1602: return launch_scan<T, 2, 16, 64>(a, v, batch, st);
        case 1604: return launch_scan<T, 4, 16, 64>(a, v, batch, st);
    }
    return fail_msg(TAE_EINVAL, "internal: selective_scan has no kernel for this plan");
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
    if (p->reserved) return fail_msg(TAE_EINVAL, "selective_scan: reserved must be 0");
    if (!dtype_ok(p->dtype)) return fail_msg(TAE_EINVAL, "selective_scan: dtype must be a TAE_DTYPE_* code");
    if (p->states < 1 || p->states > 64) return fail_msg(TAE_EINVAL, "selective_scan: states must be in 1..64");
    if (p->batch < 1 || p->len < 1 || p->channels < 1) return fail_msg(TAE_EINVAL, "selective_scan: batch, len and channels must be >= 1");
    if (p->len > (1 << 30) || p->channels > (1 << 30)) return fail_msg(TAE_EINVAL, "selective_scan: len and channels must be at most 2^30");
    if (!p->x || !p->dt || !p->a || !p->b || !p->c || !p->y || !p->state_out) return fail_msg(TAE_EINVAL, "selective_scan: x, dt, a, b, c, y and state_out must not be NULL");
    if (!elements_aligned(dtype_bytes(p->dtype), p->x, p->dt, p->b, p->c, p->z, p->y) || !elements_aligned(4, p->a, p->d, p->dt_bias, p->state, p->lengths, p->state_out))
        return fail_msg(TAE_EINVAL, "selective_scan: a pointer is not aligned to its elements");
    ScanPlan s;
    if (!plan_scan(p, &s)) return fail_msg(TAE_EINVAL, "selective_scan: bad sizes");
    if (s.bytes && (!p->workspace || p->workspace_bytes < s.bytes || !aligned(p->workspace, 16)))
        return fail_msg(TAE_EINVAL, "selective_scan: the workspace is missing, misaligned or smaller than tae_selective_scan_workspace");
    ScanArgs a{p->x, p->dt, p->b, p->c, p->z ? p->z : p->x, p->a, p->d, p->dt_bias, p->state, p->lengths, p->y, p->state_out,
               s.bytes ? (float*)p->workspace : nullptr, s.bytes ? (float*)((char*)p->workspace + s.steps_bytes) : nullptr,
               p->x_batch, p->x_row, p->dt_batch, p->dt_row, p->b_batch, p->b_row, p->c_batch, p->c_row, p->z ? p->z_batch : p->x_batch, p->z ? p->z_row : p->x_row,
               p->len, p->channels, p->states, p->softplus ? 1 : 0, p->z ? 1 : 0, s.pieces, s.piece_len, Divisor(s.groups), Divisor(s.pieces), (int64_t)p->batch * s.groups * s.pieces};
    const size_t four = 4 * dtype_bytes(p->dtype);
    Width w(dtype_bytes(p->dtype));
    w.elements(p->channels).pointer(p->x).pointer(p->dt).pointer(p->z).pointer(p->y).elements(p->x_batch).elements(p->x_row).elements(p->dt_batch).elements(p->dt_row);
    if (p->z) w.elements(p->z_batch).elements(p->z_row);
    Width w4(4);
    w4.elements(p->states).pointer(p->a).pointer(p->state).pointer(p->state_out);
    const bool vector = s.lanes ? w.fits(four) : w4.fits(16);         // loads of four channels; few positions: of four states
    if (a.blocks > ((int64_t)kGridX << 15)) return fail_msg(TAE_EINVAL, "selective_scan: the batch is too large for one call");
    return guarded([&] {
        hipStream_t st = (hipStream_t)stream;
        switch (p->dtype) {
            case TAE_DTYPE_F32: return launch_scan_plan<float>(a, s, vector, p->batch, st);
            case TAE_DTYPE_F16: return launch_scan_plan<f16>(a, s, vector, p->batch, st);
            default: return launch_scan_plan<bf16>(a, s, vector, p->batch, st);
        }
    });
}

}  // extern "C"
