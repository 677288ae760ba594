// tae_quantize_int8 and tae_int8_linear: products of 8-bit whole numbers with one scale for each token and each output channel.
//
//     scale = max|x| / 127,  q = round(127 x / max|x|),  y[m][n] = (sum_k q[m][k] w[n][k]) scale[m] weight_scale[n] + bias[n]
//
// The sums are exact (|sum| <= 131072 * 127 * 127 < 2^31), so every split of k gives the same result.  127 x is exact for 16-bit x and the
// division is correctly rounded: a quotient half way between two whole numbers is met exactly and goes to the even one.
#include "turboae_seq.hpp"

namespace tae {
namespace seq {

using i32x4 = __attribute__((ext_vector_type(4))) int;

struct QuantArgs {
    const void* x;
    int8_t* q;
    float* scale;
    int64_t x_r, q_r;
    int rows, cols;
};

// V whole numbers of a row with the largest magnitude `most`.  127 x / most is first taken with one reciprocal for the row, off by at most
// 127 * 2^-23; only where that could move it across the middle of two whole numbers is it divided as it is defined.  Adding 1.5 * 2^23 rounds
// halves to even and leaves the whole number in the low bits.
template <class T, int V>
__device__ __forceinline__ Pack<int8_t, V> whole_numbers(const Pack<T, V>& p, float by, float reciprocal) {
    constexpr float kMagic = 12582912.0f;
    Pack<int8_t, V> o;
    bool near = false;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const float t = (float)p.v[i] * reciprocal, r = t + kMagic;
        near = near || !(fabsf(t - (r - kMagic)) < 0.4995f);         // also where the reciprocal of a tiny magnitude is infinite
        o.v[i] = (int8_t)__float_as_int(r);
    }
    if (near) {
        const float down = by > 1e36f ? 0x1p-10f : 1.0f;         // where 127 x would overflow
#pragma unroll
        for (int i = 0; i < V; ++i) o.v[i] = (int8_t)__float_as_int((float)p.v[i] * down * 127.0f / (by * down) + kMagic);
    }
    return o;
}

// The largest magnitude by its bits, which are ordered as the magnitudes are, two 16-bit ones at once; an infinity or NaN is infinite.
template <class T>
struct Largest {
    using Halves = __attribute__((ext_vector_type(2))) uint16_t;
    uint32_t bits = 0;
    template <int V>
    __device__ __forceinline__ void look(const Pack<T, V>& p) {
        uint32_t w[sizeof(p) / 4];
        __builtin_memcpy(w, &p, sizeof(p));
#pragma unroll
        for (int i = 0; i < (int)sizeof(p) / 4; ++i) {
            if constexpr (sizeof(T) == 4) bits = max(bits, w[i] & 0x7FFFFFFFu);
            else bits = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(Halves, bits), __builtin_bit_cast(Halves, w[i] & 0x7FFF7FFFu)));
        }
    }
    __device__ __forceinline__ float value() const {
        float v;
        if constexpr (sizeof(T) == 4) v = __uint_as_float(bits);
        else v = (float)__builtin_bit_cast(T, (uint16_t)max(bits & 0xFFFFu, bits >> 16));
        return v < __builtin_inff() ? v : __builtin_inff();
    }
};

// One workgroup for each row, which stays in registers (KEEP groups of V for each lane; a row holds one at least) or, with KEEP = 0, is read
// twice.  Rows may start on any element: wide loads need no more here.  Bound by memory and by issuing at once: 8192 x 4096 in bf16 (101 MB)
// 22 us, 4.5 TB/s, vector instructions 95 % of the time when magnitudes were compared as floats, by bits 21; 4 x 4096 3.2 us, most of it starting up.
template <class T, int V, int KEEP>
__global__ __launch_bounds__(256) void quantize_int8_kernel(QuantArgs a) {
    __shared__ float lds[4];
    const int64_t row = block_index();
    if (row >= a.rows) return;
    const int tid = threadIdx.x;
    const T* x = (const T*)a.x + row * a.x_r;
    Largest<T> largest;
    auto edge = [&](int e) {                     // the last group of a row, zeros behind it
        Pack<T, V> p;
#pragma unroll
        for (int i = 0; i < V; ++i) p.v[i] = e + i < a.cols ? x[e + i] : (T)0.0f;
        return p;
    };
    Pack<T, V> kept[KEEP > 0 ? KEEP : 1];
    if constexpr (KEEP > 0) {
#pragma unroll
        for (int j = 0; j < KEEP; ++j) kept[j] = load_any<T, V>(x + min((j * 256 + tid) * V, a.cols - V));
#pragma unroll
        for (int j = 0; j < KEEP; ++j) {
            const int e = (j * 256 + tid) * V;
            if (e < a.cols && e + V > a.cols) kept[j] = edge(e);
            largest.look(kept[j]);
        }
    } else {
        int e = tid * V;
        for (; e + V <= a.cols; e += 256 * V) largest.look(load_any<T, V>(x + e));
        if (e < a.cols) largest.look(edge(e));
    }
    float most = lanes_max<64>(largest.value());
    if ((tid & 63) == 0) lds[tid >> 6] = most;
    __syncthreads();
    most = fmaxf(fmaxf(lds[0], lds[1]), fmaxf(lds[2], lds[3]));
    const bool fine = most < __builtin_inff();
    if (tid == 0) a.scale[row] = fine ? most / 127.0f : __builtin_nanf("");
    // a row of zeros: 0; one with an infinity or NaN: 0 too, whatever it holds
    const float by = most > 0.0f ? most : 1.0f, reciprocal = 127.0f / by;
    int8_t* q = a.q + row * a.q_r;
    const Pack<int8_t, V> zeros{};
    if constexpr (KEEP > 0) {
#pragma unroll
        for (int j = 0; j < KEEP; ++j) {
            const int e = (j * 256 + tid) * V;
            if (e < a.q_r) store<int8_t, V>(q + e, fine && e < a.cols ? whole_numbers<T, V>(kept[j], by, reciprocal) : zeros);
        }
        for (int e = (KEEP * 256 + tid) * V; e < a.q_r; e += 256 * V) store<int8_t, V>(q + e, zeros);
    } else {
        int e = tid * V;
        if (fine) {
            for (; e + V <= a.cols; e += 256 * V) store<int8_t, V>(q + e, whole_numbers<T, V>(load_any<T, V>(x + e), by, reciprocal));
            if (e < a.cols) store<int8_t, V>(q + e, whole_numbers<T, V>(edge(e), by, reciprocal)), e += 256 * V;
        }
        for (; e < a.q_r; e += 256 * V) store<int8_t, V>(q + e, zeros);
    }
}

template <class T>
static void launch_quantize(const QuantArgs& a, hipStream_t st) {
    constexpr int V = 16 / sizeof(T);
    const dim3 grid = grid_of(a.rows), block(256);
    if (a.cols >= V && a.cols <= 256 * V) hipLaunchKernelGGL((quantize_int8_kernel<T, V, 1>), grid, block, 0, st, a);
    else if (a.cols >= V && a.cols <= 512 * V) hipLaunchKernelGGL((quantize_int8_kernel<T, V, 2>), grid, block, 0, st, a);
    else if (a.cols >= V && a.cols <= 1024 * V) hipLaunchKernelGGL((quantize_int8_kernel<T, V, 4>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((quantize_int8_kernel<T, V, 0>), grid, block, 0, st, a);
}

static void launch_quantize_dtype(const QuantArgs& a, int32_t dtype, hipStream_t st) {
    switch (dtype) {
        case TAE_DTYPE_F32: launch_quantize<float>(a, st); break;
        case TAE_DTYPE_F16: launch_quantize<f16>(a, st); break;
        default: launch_quantize<bf16>(a, st); break;
    }
}

struct Int8Args {
    const int8_t *q, *w;                         // (rows, q_r) zero behind k; (outputs, w_r)
    const float *scale, *w_scale, *bias;
    void* y;
    int64_t q_r, w_r;
    int m, k, n, tiles_n, wide;                  // wide: rows of y start on 16-byte boundaries
    int64_t tiles_m, blocks;
};

// Products of 16 rows of weights with 16 rows of x over 64 inputs: lane l hands over 16 adjacent inputs of row l % 16, from input 16 (l / 16),
// for both, and holds the sums of weight rows 4 (l / 16) .. + 3 with x row l % 16.
__device__ __forceinline__ i32x4 mfma64(i32x4 w, i32x4 q, i32x4 c) { return __builtin_amdgcn_mfma_i32_16x16x64_i8(w, q, c, 0, 0, 0); }

// COUNT adjacent outputs from n on: their scales and biases once, then row by row.
template <class T, int COUNT>
struct Outputs {
    float scale[COUNT], bias[COUNT];
    int n;
    __device__ __forceinline__ Outputs(const Int8Args& a, int n0) : n(n0) {
#pragma unroll
        for (int i = 0; i < COUNT; ++i) {
            const int at = min(n + i, a.n - 1);
            scale[i] = a.w_scale[at];
            bias[i] = a.bias ? a.bias[at] : 0.0f;
        }
    }
    __device__ __forceinline__ Pack<T, COUNT> row(const int (&sum)[COUNT], float sm) const {
        Pack<T, COUNT> out;
#pragma unroll
        for (int i = 0; i < COUNT; ++i) out.v[i] = (T)__builtin_fmaf((float)sum[i], sm * scale[i], bias[i]);
        return out;
    }
};

// 32 bytes that are not read again soon and leave the operands in L2 alone; 64 of them, 4 x 16 apart, are put together there first (measured,
// 2396 x 2188 x 7244 in fp32: 123 us past L2, 78 through it)
template <class T>
__device__ __forceinline__ void store_once(T* to, const Pack<T, 16>& p) {
    i32x4 part[sizeof(p) / 16];
    __builtin_memcpy(part, &p, sizeof(p));
#pragma unroll
    for (int i = 0; i < (int)sizeof(p) / 16; ++i) {
        i32x4* at = reinterpret_cast<i32x4*>(to) + i;
        if constexpr (sizeof(T) == 4) *at = part[i];
        else __builtin_nontemporal_store(part[i], at);
    }
}

// Copies 16 bytes for each lane from a buffer to LDS without registers, to `to` + 16 lane; counted by vmcnt.  Offsets outside the buffer
// give zeros.
using LdsPtr = __attribute__((address_space(3))) void*;
__device__ __forceinline__ void copy_to_lds(__amdgpu_buffer_rsrc_t buffer, LdsPtr to, uint32_t offset) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(buffer, to, 16, offset, 0, 0, 0);
}
template <int LEFT>
__device__ __forceinline__ void wait_copies() {             // all but the last LEFT of this wave's copies have arrived, for every wave
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(LEFT) : "memory");
}

// BM x BN outputs at a time for each workgroup of WM x WN waves, 64 weight rows for each wave.
//
// Bound by the matrix instructions.  A workgroup takes tile after tile without a break: the slabs of 128 inputs of all its tiles are one
// stream through STAGES LDS buffers, copied directly, whole 128-byte lines at a time.  The one barrier of a slab stands behind its last
// fragment reads, a quarter of its products before its end: there the next slab has arrived, this slab's buffer is free for the one
// STAGES further, and the next slab's first fragments are read during the rest of the products.  A tile's results are stored while the next tile is
// under way.  A row's eight 16-byte pieces are permuted by its number (by which piece a lane copies), so that the 16 lanes which read LDS
// together touch all banks.  Weight rows are dealt to fragments such that a lane ends up with 16 adjacent outputs.  Workgroups of one XCD
// (every eighth) take adjacent tiles, eight rows of tiles high, and share operands in its L2.
//
// Measured, bf16, 8192 x 4096 x 8192 (550 G operations): 230 us among other work and 263 to 285 in a row, by the power that is left: 1.9 to 2.4 POP/s.
// A stream of nothing but these matrix instructions on such numbers reaches 3.7, a large library product 1.8.  The matrix pipes are busy half
// of the cycles; the rest are waits for fragments and copies at 61 bytes a clock for each CU.  Slower: a ring of five buffers of 64 inputs
// (requests of half a line), waves of 128 x 128 (spills), 128 x 128 tiles (4096 x 4096 x 4096: 91 us, these 83).
template <class T, int BM, int BN, int WM, int WN, int STAGES>
__global__ __launch_bounds__(WM * WN * 64, BM / WM * (BN / WN) > 8192 ? 1 : 2) void int8_linear_kernel(Int8Args a) {
    constexpr int WAVES = WM * WN, MF = BM / WM / 16, NF = BN / WN / 16, ROWS = BM + BN, PIECES = ROWS / 8 / WAVES, STAGE = ROWS * 128;
    static_assert(BN / WN % 64 == 0 && ROWS % (8 * WAVES) == 0 && BM % (8 * PIECES) == 0, "whole pieces of one operand for each wave");
    extern __shared__ char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / WN, wn = wave % WN;
    // this workgroup's tiles: of its XCD's share, every (workgroups of the XCD)-th
    const int64_t xcd = blockIdx.x % 8, each = a.blocks / 8, more = a.blocks % 8, stride_tiles = (gridDim.x - xcd + 7) / 8;
    const int64_t share = each + (xcd < more), begin = xcd * each + min(xcd, more), slot = blockIdx.x / 8;
    const int tiles = (int)(slot < share ? (share - slot + stride_tiles - 1) / stride_tiles : 0);
    if (tiles == 0) return;
    auto place = [&](int i, int& m0, int& n0) {
        const int64_t tile = begin + slot + i * stride_tiles, band = tile / (8 * (int64_t)a.tiles_n), first = band * 8;
        const int64_t high = min((int64_t)8, a.tiles_m - first), in = tile - first * a.tiles_n;
        m0 = (int)(first + in % high) * BM;
        n0 = (int)(in / high) * BN;
    };
    const int slabs = (a.k + 127) / 128;

    // the copying end of the stream: its tile, slab and buffer; this wave copies rows 8 PIECES wave .. of x (rows 0 .. BM - 1), then of the weights
    const bool weights = wave * PIECES * 8 >= BM;
    const int64_t stride = weights ? a.w_r : a.q_r;
    __amdgpu_buffer_rsrc_t buffer;
    uint32_t offset[PIECES];
    auto open = [&](int i) {
        int m0, n0;
        place(i, m0, n0);
        const int rows = weights ? min(a.n - n0, BN) : min(a.m - m0, BM);
        const int8_t* from = weights ? a.w + (int64_t)n0 * a.w_r : a.q + (int64_t)m0 * a.q_r;
        buffer = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(from), 0, (int)((rows - 1) * stride) + ((a.k + 15) & ~15), 0x00020000);
#pragma unroll
        for (int j = 0; j < PIECES; ++j) {
            const int r = (wave * PIECES + j) * 8 + lane / 8;        // row of the stage
            int row = weights ? r - BM : r;
            if (weights) row = (row & ~63) + (row / 4 % 4) * 16 + (row / 16 % 4) * 4 + row % 4;
            offset[j] = (uint32_t)min(row, rows - 1) * (uint32_t)stride + ((lane ^ r) & 7) * 16;
        }
    };
    int to_tile = 0, to_slab = 0;
    auto copy = [&](int stage) {                 // behind the end the last slab again
#pragma unroll
        for (int j = 0; j < PIECES; ++j) copy_to_lds(buffer, (LdsPtr)(lds + stage * STAGE + (wave * PIECES + j) * 1024), offset[j] + (uint32_t)to_slab * 128);
        if (to_slab + 1 < slabs) {
            ++to_slab;
        } else if (to_tile + 1 < tiles) {
            open(++to_tile);
            to_slab = 0;
        }
    };

    // pieces q and 4 + q of row r16 for the two halves of a slab
    const int r16 = lane & 15, half[2] = {r16 * 128 + (((lane >> 4) ^ r16) & 7) * 16, r16 * 128 + (((lane >> 4 | 4) ^ r16) & 7) * 16};
    i32x4 wf[NF], wf_next[NF], qf[MF], qf_next[2], acc[NF][MF] = {};
    auto weight = [&](const char* p, int f) { return *(const i32x4*)(p + (BM + (wn * NF + f) * 16) * 128); };
    auto x = [&](const char* p, int f) { return *(const i32x4*)(p + (wm * MF + f) * 2048); };
    int tile = 0, slab = 0, stage = 0, m0, n0;
    auto results = [&]() {
        float sm[MF];
#pragma unroll
        for (int i = 0; i < MF; ++i) sm[i] = a.scale[min(m0 + (wm * MF + i) * 16 + r16, a.m - 1)];
        const bool whole = a.wide && n0 + BN <= a.n;
#pragma unroll
        for (int block = 0; block < NF / 4; ++block) {
            const int n = n0 + (wn * NF / 4 + block) * 64 + (lane >> 4) * 16;
            const Outputs<T, 16> outputs(a, n);
#pragma unroll
            for (int i = 0; i < MF; ++i) {
                const int m = m0 + (wm * MF + i) * 16 + r16;
                int sum[16];
#pragma unroll
                for (int f = 0; f < 4; ++f)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        sum[f * 4 + r] = acc[block * 4 + f][i][r];
                        acc[block * 4 + f][i][r] = 0;
                    }
                const Pack<T, 16> out = outputs.row(sum, sm[i]);
                T* y = (T*)a.y + (int64_t)m * a.n + n;
                if (whole) {
                    if (m < a.m) store_once(y, out);
                } else if (n + 16 <= a.n) {
                    if (m < a.m) store_any(y, out);
                } else {
#pragma unroll
                    for (int c = 0; c < 16; ++c)
                        if (m < a.m && n + c < a.n) y[c] = out.v[c];
                }
            }
        }
    };
    constexpr int EARLY = MF * 3 / 4;            // of the second half's products, in front of the barrier: what needs no more fragments
    auto multiply = [&](int from, int to) {
#pragma unroll
        for (int i = from; i < to; ++i)
#pragma unroll
            for (int f = 0; f < NF; ++f) acc[f][i] = mfma64(wf[f], qf[i], acc[f][i]);
    };
    auto advance = [&]() {
#pragma unroll
        for (int f = 0; f < NF; ++f) wf[f] = wf_next[f];
        qf[0] = qf_next[0];
        qf[1] = qf_next[1];
    };
    auto first = [&](const char* p) {            // the fragments that a half starts with
#pragma unroll
        for (int f = 0; f < NF; ++f) wf_next[f] = weight(p, f);
        qf_next[0] = x(p, 0);
        qf_next[1] = x(p, 1);
    };
    place(0, m0, n0);
    open(0);
#pragma unroll
    for (int s = 0; s < STAGES; ++s) copy(s);
    wait_copies<(STAGES - 1) * PIECES>();
    first(lds + half[0]);
    advance();
    for (;;) {
        const char* here = lds + stage * STAGE;
#pragma unroll
        for (int i = 2; i < MF; ++i) qf[i] = x(here + half[0], i);
        first(here + half[1]);
        multiply(0, MF);
        // issue order: one fragment read for every second or third product
#pragma unroll
        for (int f = 0; f < NF + MF; ++f) {
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x008, MF * NF / (NF + MF), 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, MF * NF - MF * NF / (NF + MF) * (NF + MF), 0);
        __builtin_amdgcn_sched_barrier(0);
        advance();
#pragma unroll
        for (int i = 2; i < MF; ++i) qf[i] = x(here + half[1], i);
        multiply(0, EARLY);
#pragma unroll
        for (int f = 2; f < MF; ++f) {
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 1);
            __builtin_amdgcn_sched_group_barrier(0x008, EARLY * NF / (MF - 2), 1);
        }
        // all fragments of this slab have been read, by every wave, and all copies of the next one have arrived
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        wait_copies<(STAGES - 2) * PIECES>();
        copy(stage);
        stage = stage + 1 == STAGES ? 0 : stage + 1;
        first(lds + stage * STAGE + half[0]);
        multiply(EARLY, MF);
        advance();
        if (++slab < slabs) continue;
        results();
        slab = 0;
        if (++tile == tiles) break;
        place(tile, m0, n0);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");         // no copy is under way when the workgroup's LDS is given away
}

// Few rows of x: bound by reading the weights.  16 NF weight rows and up to 16 MF rows of x for each workgroup; its eight waves share the
// inputs and join their sums, exact in any order, in LDS.  Both operands come straight from memory (x from L2), DEEP slabs of 64 in flight.
// Measured: 4 x 4096 x 4096 6.1 us, 2.8 TB/s of weights with start and drain.
template <class T, int MF, int NF, int DEEP>
__global__ __launch_bounds__(512) void int8_few_kernel(Int8Args a) {
    constexpr int FRAGMENTS = MF * NF, ROUND = FRAGMENTS < 8 ? FRAGMENTS : 8;          // joined at once
    __shared__ i32x4 part[8][ROUND][64];
    const int64_t id = block_index();
    if (id >= a.blocks) return;
    const int n0 = (int)(id % a.tiles_n) * 16 * NF, m0 = (int)(id / a.tiles_n) * 16 * MF;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r16 = lane & 15, kk = (lane >> 4) * 16;
    const int slabs = (a.k + 63) / 64, each = (slabs + 7) / 8, begin = wave * each, end = min(begin + each, slabs);
    const int8_t *w[NF], *q[MF];
#pragma unroll
    for (int f = 0; f < NF; ++f) w[f] = a.w + (int64_t)min(n0 + f * 16 + r16, a.n - 1) * a.w_r;
#pragma unroll
    for (int i = 0; i < MF; ++i) q[i] = a.q + (int64_t)min(m0 + i * 16 + r16, a.m - 1) * a.q_r;
    i32x4 acc[NF][MF] = {};
    const int last = (a.k - 1) & ~15;            // the last 16 bytes of a row that may be read; q is zero where they repeat
    for (int s0 = begin; s0 < end; s0 += DEEP) {
        i32x4 wv[DEEP][NF], qv[DEEP][MF];
#pragma unroll
        for (int d = 0; d < DEEP; ++d) {
            const int k = min(s0 + d, end - 1) * 64 + kk;
#pragma unroll
            for (int f = 0; f < NF; ++f) wv[d][f] = *(const i32x4*)(w[f] + min(k, last));
#pragma unroll
            for (int i = 0; i < MF; ++i) qv[d][i] = *(const i32x4*)(q[i] + k);
        }
#pragma unroll
        for (int d = 0; d < DEEP; ++d) {
            if (s0 + d < end) {
#pragma unroll
                for (int i = 0; i < MF; ++i)
#pragma unroll
                    for (int f = 0; f < NF; ++f) acc[f][i] = mfma64(wv[d][f], qv[d][i], acc[f][i]);
            }
        }
    }
    // fragment f, i is number f + NF i; a wave finishes those whose number is its own modulo 8
#pragma unroll
    for (int first = 0; first < FRAGMENTS; first += ROUND) {
        if (first > 0) __syncthreads();          // the last round has been read
#pragma unroll
        for (int j = 0; j < ROUND; ++j) part[wave][j][lane] = acc[(first + j) % NF][(first + j) / NF];
        __syncthreads();
        if (wave >= ROUND) continue;
        i32x4 sum = part[0][wave][lane];
#pragma unroll
        for (int u = 1; u < 8; ++u) sum += part[u][wave][lane];
        const int m = m0 + (first + wave) / NF * 16 + r16, n = n0 + (first + wave) % NF * 16 + (lane >> 4) * 4;
        if (m >= a.m || n >= a.n) continue;
        const Pack<T, 4> out = Outputs<T, 4>(a, n).row({sum[0], sum[1], sum[2], sum[3]}, a.scale[m]);
        T* y = (T*)a.y + (int64_t)m * a.n + n;
        if (n + 4 <= a.n) {
            store_any(y, out);
        } else {
#pragma unroll
            for (int c = 0; c < 4; ++c)
                if (n + c < a.n) y[c] = out.v[c];
        }
    }
}

// Up to 8 rows of x in one launch: every workgroup quantises all of them itself, into LDS, with its first weights under way, and goes on like
// int8_few_kernel with 16 weight rows.  `share` waves share a row.  Measured in bf16 in a graph, then eagerly, against two launches: 4 x 1024 x
// 1024 5.8 and 9.8 us (7.5 and 13.9), 1 x 4096 x 4096 7.7 and 9.7 (9.0 and 14.4), 4 x 4096 x 4096 9.3 and 9.8 (9.6 and 14.6).  More rows or
// inputs take longer to quantise again and again than a launch (with 8 groups a lane, 8 x 4096 x 4096: 16.1 where two launches take 9.9), and
// so do more workgroups than the CUs hold at once (1 x 1024 x 51200: 33 where two take 16).
template <class T>
__global__ __launch_bounds__(512) void int8_rows_kernel(Int8Args a, const T* x, int64_t x_r, int share) {
    constexpr int V = 16 / sizeof(T), DEEP = 8;
    __shared__ i32x4 part[8][64];
    __shared__ float most_of[8], scale_of[8];
    extern __shared__ char lds[];                // (m, q_r) whole numbers, zero behind k
    const int64_t id = block_index();
    if (id >= a.blocks) return;
    const int n0 = (int)id * 16, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r16 = lane & 15, kk = (lane >> 4) * 16;
    const int slabs = (a.k + 63) / 64, each = (slabs + 7) / 8, begin = wave * each, end = min(begin + each, slabs), last = (a.k - 1) & ~15;
    const int8_t* w = a.w + (int64_t)min(n0 + r16, a.n - 1) * a.w_r;
    i32x4 wv[DEEP];
    auto fetch = [&](int s0) {
#pragma unroll
        for (int d = 0; d < DEEP; ++d) wv[d] = *(const i32x4*)(w + min(min(s0 + d, slabs - 1) * 64 + kk, last));
    };
    fetch(begin);
    const int step = 64 * V * share, from = (wave % share * 64 + lane) * V, m = wave / share;
    const T* row = x + m * x_r;
    Pack<T, V> kept[kRowsGroups];
    Largest<T> largest;
    if (m < a.m) {
        if (a.k >= V) {
#pragma unroll
            for (int i = 0; i < kRowsGroups; ++i) kept[i] = load_any<T, V>(row + min(from + i * step, a.k - V));
        }
#pragma unroll
        for (int i = 0; i < kRowsGroups; ++i) {
            const int e = from + i * step;
            if (a.k < V || (e < a.k && e + V > a.k)) {            // the last group of the row, zeros behind it
#pragma unroll
                for (int c = 0; c < V; ++c) kept[i].v[c] = e + c < a.k ? row[e + c] : (T)0.0f;
            }
            largest.look(kept[i]);
        }
    }
    float most = lanes_max<64>(largest.value());
    if (lane == 0) most_of[wave] = most;
    __syncthreads();
    if (m < a.m) {
        for (int i = 0; i < share; ++i) most = fmaxf(most, most_of[m * share + i]);
        const bool fine = most < __builtin_inff();
        if (lane == 0) scale_of[m] = fine ? most / 127.0f : __builtin_nanf("");
        const float by = most > 0.0f ? most : 1.0f, reciprocal = 127.0f / by;
        int8_t* q = (int8_t*)lds + m * (int)a.q_r;
#pragma unroll
        for (int i = 0; i < kRowsGroups; ++i) {
            const int e = from + i * step;
            if (e < slabs * 64) store<int8_t, V>(q + e, fine && e < a.k ? whole_numbers<T, V>(kept[i], by, reciprocal) : Pack<int8_t, V>{});
        }
    }
    __syncthreads();
    const char* q = lds + min(r16, a.m - 1) * (int)a.q_r + kk;
    i32x4 acc = {};
    for (int s0 = begin; s0 < end; s0 += DEEP) {
        if (s0 > begin) fetch(s0);
#pragma unroll
        for (int d = 0; d < DEEP; ++d)
            if (s0 + d < end) acc = mfma64(wv[d], *(const i32x4*)(q + (s0 + d) * 64), acc);
    }
    part[wave][lane] = acc;
    __syncthreads();
    if (wave > 0) return;
    i32x4 sum = part[0][lane];
#pragma unroll
    for (int u = 1; u < 8; ++u) sum += part[u][lane];
    const int n = n0 + (lane >> 4) * 4;
    if (r16 >= a.m || n >= a.n) return;
    const Pack<T, 4> out = Outputs<T, 4>(a, n).row({sum[0], sum[1], sum[2], sum[3]}, scale_of[r16]);
    T* y = (T*)a.y + (int64_t)r16 * a.n + n;
    if (n + 4 <= a.n) {
        store_any(y, out);
    } else {
#pragma unroll
        for (int c = 0; c < 4; ++c)
            if (n + c < a.n) y[c] = out.v[c];
    }
}

template <class T, int BM, int BN, int WM, int WN, int STAGES>
static hipError_t launch_tiles(Int8Args a, hipStream_t st) {
    constexpr int bytes = STAGES * (BM + BN) * 128;
    a.tiles_m = ceil_div(a.m, BM);
    a.tiles_n = (int)ceil_div(a.n, BN);
    a.blocks = a.tiles_m * a.tiles_n;
    const void* kernel = reinterpret_cast<const void*>(int8_linear_kernel<T, BM, BN, WM, WN, STAGES>);
    const hipError_t e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);        // of the current device
    if (e != hipSuccess) return e;
    const int64_t resident = 256 * (160 * 1024 / bytes);     // workgroups that 256 CUs hold at once
    hipLaunchKernelGGL((int8_linear_kernel<T, BM, BN, WM, WN, STAGES>), dim3((uint32_t)std::min(a.blocks, resident)), dim3(WM * WN * 64), bytes, st, a);
    return hipSuccess;
}

template <class T, int MF, int NF, int DEEP>
static hipError_t launch_few(Int8Args a, hipStream_t st) {
    a.tiles_m = ceil_div(a.m, 16 * MF);
    a.tiles_n = (int)ceil_div(a.n, 16 * NF);
    a.blocks = a.tiles_m * a.tiles_n;
    hipLaunchKernelGGL((int8_few_kernel<T, MF, NF, DEEP>), grid_of(a.blocks), dim3(512), 0, st, a);
    return hipSuccess;
}

template <class T>
static hipError_t launch_int8(const Int8Args& a, Int8Form form, hipStream_t st) {
    switch (form) {
        case Int8Form::tiles256: return launch_tiles<T, 256, 256, 2, 4, 2>(a, st);
        case Int8Form::tiles128_two: return launch_tiles<T, 128, 128, 2, 2, 2>(a, st);
        case Int8Form::few16: return launch_few<T, 1, 1, 8>(a, st);
        case Int8Form::few32: return launch_few<T, 2, 2, 4>(a, st);
        case Int8Form::few64: return launch_few<T, 4, 2, 4>(a, st);
        default: return launch_tiles<T, 128, 128, 2, 2, 4>(a, st);
    }
}

template <class T>
static void launch_rows(Int8Args a, const tae_int8_args* p, hipStream_t st) {
    a.q_r = ceil_div(p->inputs, 64) * 64 + 16;
    a.blocks = ceil_div(a.n, 16);
    hipLaunchKernelGGL((int8_rows_kernel<T>), dim3((uint32_t)a.blocks), dim3(512), a.m * a.q_r, st, a, (const T*)p->x, p->x_row, rows_share(p));
}

// Rows 1024 bytes and multiples apart would send a slab's lines of all rows to few channels of L2.
static int64_t q_stride(int32_t k) {
    const int64_t r = ceil_div(k, 128) * 128;
    return r % 1024 ? r : r + 128;
}

}  // namespace seq
}  // namespace tae

extern "C" {

int tae_quantize_int8(int32_t dtype, const void* x, int64_t x_row, int32_t rows, int32_t cols, int8_t* q, int64_t q_row, float* scale, void* stream) {
    using namespace tae;
    using namespace tae::seq;
    if (!dtype_ok(dtype)) return fail_msg(TAE_EINVAL, "quantize_int8: dtype must be a TAE_DTYPE_* code");
    if (!x || !q || !scale) return fail_msg(TAE_EINVAL, "quantize_int8: x, q and scale must not be NULL");
    if (rows < 1 || cols < 1 || cols > (1 << 30)) return fail_msg(TAE_EINVAL, "quantize_int8: rows must be >= 1, cols in 1..2^30");
    if (q_row < cols || q_row % 16 || q_row > (1 << 30) + 1024 || !aligned(q, 16)) return fail_msg(TAE_EINVAL, "quantize_int8: q rows start on 16-byte boundaries and hold cols values");
    if (!elements_aligned(dtype_bytes(dtype), x) || !elements_aligned(4, scale)) return fail_msg(TAE_EINVAL, "quantize_int8: a pointer is not aligned to its elements");
    return guarded([&] {
        launch_quantize_dtype(QuantArgs{x, q, scale, x_row, q_row, rows, cols}, dtype, (hipStream_t)stream);
        return (int)TAE_OK;
    });
}

size_t tae_int8_linear_workspace(const tae_int8_args* p) {
    using namespace tae::seq;
    if (!p || p->struct_size != (int32_t)sizeof(tae_int8_args) || !int8_sizes(p) || !dtype_ok(p->dtype) || int8_in_one(p)) return 0;
    return (size_t)p->rows * q_stride(p->inputs) + (size_t)p->rows * 4;
}

int tae_int8_linear(const tae_int8_args* p, void* stream) {
    using namespace tae;
    using namespace tae::seq;
    if (!p || p->struct_size != (int32_t)sizeof(tae_int8_args)) return fail_msg(TAE_EINVAL, "tae_int8_args: NULL or struct_size mismatch (ABI)");
    if (p->reserved) return fail_msg(TAE_EINVAL, "int8_linear: reserved must be 0");
    if (!dtype_ok(p->dtype)) return fail_msg(TAE_EINVAL, "int8_linear: dtype must be a TAE_DTYPE_* code");
    if (!int8_sizes(p)) return fail_msg(TAE_EINVAL, "int8_linear: inputs must be in 1..131072, rows and outputs in 1..2^30");
    if (!p->x || !p->weight || !p->weight_scale || !p->y) return fail_msg(TAE_EINVAL, "int8_linear: x, weight, weight_scale and y must not be NULL");
    if (!aligned(p->weight, 16) || p->weight_row % 16 || p->weight_row < p->inputs || p->weight_row > (1 << 23)) return fail_msg(TAE_EINVAL, "int8_linear: weight rows start on 16-byte boundaries (quantize_int8 lays them so), at most 2^23 bytes apart");
    const size_t need = tae_int8_linear_workspace(p);         // 0: in one launch
    if (need && (!p->workspace || p->workspace_bytes < need || !aligned(p->workspace, 16))) return fail_msg(TAE_EINVAL, "int8_linear: the workspace is missing, misaligned or smaller than tae_int8_linear_workspace");
    if (!elements_aligned(dtype_bytes(p->dtype), p->x, p->y) || !elements_aligned(4, p->weight_scale, p->bias)) return fail_msg(TAE_EINVAL, "int8_linear: a pointer is not aligned to its elements");
    const int64_t qr = q_stride(p->inputs);
    int8_t* q = (int8_t*)p->workspace;
    float* scale = need ? (float*)(q + (size_t)p->rows * qr) : nullptr;
    Width wy(dtype_bytes(p->dtype));
    wy.elements(p->outputs).pointer(p->y);
    const Int8Args a{q, p->weight, scale, p->weight_scale, p->bias, p->y, qr, p->weight_row, p->rows, p->inputs, p->outputs, 0, wy.fits(16), 0, 0};
    return guarded([&] {
        hipStream_t st = (hipStream_t)stream;
        if (!need) {
            switch (p->dtype) {
                case TAE_DTYPE_F32: launch_rows<float>(a, p, st); break;
                case TAE_DTYPE_F16: launch_rows<f16>(a, p, st); break;
                default: launch_rows<bf16>(a, p, st); break;
            }
            return (int)TAE_OK;
        }
        launch_quantize_dtype(QuantArgs{p->x, q, scale, p->x_row, qr, p->rows, p->inputs}, p->dtype, st);
        hipError_t e;
        const Int8Form form = int8_form(p);
        switch (p->dtype) {
            case TAE_DTYPE_F32: e = launch_int8<float>(a, form, st); break;
            case TAE_DTYPE_F16: e = launch_int8<f16>(a, form, st); break;
            default: e = launch_int8<bf16>(a, form, st); break;
        }
        if (e != hipSuccess) return fail_msg(TAE_EHIP, hipGetErrorString(e));
        return (int)TAE_OK;
    });
}

}  // extern "C"
