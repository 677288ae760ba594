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

// One workgroup for each row: its largest magnitude, then its whole numbers (the second reading comes from L2).
template <class T, int V>
__global__ __launch_bounds__(256) void quantize_int8_kernel(QuantArgs a) {
    __shared__ float lds[4];
    const int64_t row = block_index();
    if (row >= a.rows) return;
    const int tid = threadIdx.x;
    const T* x = (const T*)a.x + row * a.x_r;
    float most = 0.0f;
    bool bad = false;
    for (int e = tid * V; e < a.cols; e += 256 * V) {
        const Pack<T, V> p = load<T, V>(x + e);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float v = fabsf((float)p.v[i]);
            bad = bad || !(v < __builtin_inff());
            most = fmaxf(most, v);
        }
    }
    if (__any(bad)) most = __builtin_inff();
    most = lanes_max<64>(most);
    if ((tid & 63) == 0) lds[tid >> 6] = most;
    __syncthreads();
    most = fmaxf(fmaxf(lds[0], lds[1]), fmaxf(lds[2], lds[3]));
    const bool fine = most < __builtin_inff();
    if (tid == 0) a.scale[row] = fine ? most / 127.0f : __builtin_nanf("");
    const float by = most > 0.0f ? most : 1.0f;
    int8_t* q = a.q + row * a.q_r;
    for (int e = tid * V; e < a.q_r; e += 256 * V) {
        Pack<int8_t, V> o;
        Pack<T, V> p;
        if (e < a.cols) p = load<T, V>(x + e);
#pragma unroll
        for (int i = 0; i < V; ++i) o.v[i] = fine && e < a.cols ? (int8_t)(int)rintf((float)p.v[i] * 127.0f / by) : (int8_t)0;
        store<int8_t, V>(q + e, o);
    }
}

template <class T>
static void launch_quantize(const QuantArgs& a, hipStream_t st) {
    constexpr int V = 16 / sizeof(T);
    Width w(sizeof(T));
    w.elements(a.cols).elements(a.x_r).pointer(a.x);
    if (w.fits(16)) hipLaunchKernelGGL((quantize_int8_kernel<T, V>), grid_of(a.rows), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((quantize_int8_kernel<T, 1>), grid_of(a.rows), dim3(256), 0, st, a);
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
    int m, k, n, tiles_n;
    int64_t blocks;
};

// 64 x 64 outputs for each workgroup, 32 x 32 for each wave.  LDS holds 16 x 64 pieces of both operands in the order in which a wave's lanes
// hand them to the matrix instruction: lane l has 16 adjacent k of row l % 16, from k = 16 (l / 16).
template <class T>
__global__ __launch_bounds__(256) void int8_linear_kernel(Int8Args a) {
    __shared__ i32x4 lw[256], lq[256];
    const int64_t id = block_index();
    if (id >= a.blocks) return;
    const int n0 = (int)(id % a.tiles_n) * 64;
    const int m0 = (int)(id / a.tiles_n) * 64;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int row = (tid >> 6) * 16 + (lane & 15), kk = (lane >> 4) * 16;
    const int8_t* w = a.w + (int64_t)min(n0 + row, a.n - 1) * a.w_r;
    const int8_t* q = a.q + (int64_t)min(m0 + row, a.m - 1) * a.q_r;
    i32x4 acc[2][2] = {};
    for (int k0 = 0; k0 < a.k; k0 += 64) {
        i32x4 vw{}, vq{};
        if (k0 + kk < a.k) {
            vw = *(const i32x4*)(w + k0 + kk);
            vq = *(const i32x4*)(q + k0 + kk);
        }
        __syncthreads();
        lw[tid] = vw;
        lq[tid] = vq;
        __syncthreads();
        const int tn = (wave & 1) * 2, tm = (wave >> 1) * 2;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
                acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(lw[(tn + i) * 64 + lane], lq[(tm + j) * 64 + lane], acc[i][j], 0, 0, 0);
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int m = m0 + (wave >> 1) * 32 + j * 16 + (lane & 15);
        if (m >= a.m) continue;
        const float sm = a.scale[m];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int n = n0 + (wave & 1) * 32 + i * 16 + (lane >> 4) * 4 + r;
                if (n >= a.n) continue;
                float v = (float)acc[i][j][r] * (sm * a.w_scale[n]);
                if (a.bias) v += a.bias[n];
                ((T*)a.y)[(int64_t)m * a.n + n] = (T)v;
            }
    }
}

template <class T>
static void launch_int8(const Int8Args& a, hipStream_t st) {
    hipLaunchKernelGGL((int8_linear_kernel<T>), grid_of(a.blocks), dim3(256), 0, st, a);
}

static int64_t q_stride(int32_t k) { return ceil_div(k, 64) * 64; }

static bool int8_sizes(const tae_int8_args* p) {
    return p->rows >= 1 && p->inputs >= 1 && p->inputs <= 131072 && p->outputs >= 1 && p->rows <= (1 << 30) && p->outputs <= (1 << 30);
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
    return guarded([&] {
        launch_quantize_dtype(QuantArgs{x, q, scale, x_row, q_row, rows, cols}, dtype, (hipStream_t)stream);
        return (int)TAE_OK;
    });
}

size_t tae_int8_linear_workspace(const tae_int8_args* p) {
    using namespace tae::seq;
    if (!p || p->struct_size != (int32_t)sizeof(tae_int8_args) || !int8_sizes(p)) return 0;
    return (size_t)p->rows * q_stride(p->inputs) + (size_t)p->rows * 4;
}

int tae_int8_linear(const tae_int8_args* p, void* stream) {
    using namespace tae;
    using namespace tae::seq;
    if (!p || p->struct_size != (int32_t)sizeof(tae_int8_args)) return fail_msg(TAE_EINVAL, "tae_int8_args: NULL or struct_size mismatch (ABI)");
    if (!dtype_ok(p->dtype)) return fail_msg(TAE_EINVAL, "int8_linear: dtype must be a TAE_DTYPE_* code");
    if (!int8_sizes(p)) return fail_msg(TAE_EINVAL, "int8_linear: inputs must be in 1..131072, rows and outputs in 1..2^30");
    if (!p->x || !p->weight || !p->weight_scale || !p->y) return fail_msg(TAE_EINVAL, "int8_linear: x, weight, weight_scale and y must not be NULL");
    if (!aligned(p->weight, 16) || p->weight_row % 16 || p->weight_row < p->inputs) return fail_msg(TAE_EINVAL, "int8_linear: weight rows start on 16-byte boundaries (quantize_int8 lays them so)");
    const size_t need = tae_int8_linear_workspace(p);
    if (!p->workspace || p->workspace_bytes < need || !aligned(p->workspace, 16)) return fail_msg(TAE_EINVAL, "int8_linear: the workspace is missing, misaligned or smaller than tae_int8_linear_workspace");
    const int64_t qr = q_stride(p->inputs);
    int8_t* q = (int8_t*)p->workspace;
    float* scale = (float*)(q + (size_t)p->rows * qr);
    const int tiles_n = (int)ceil_div(p->outputs, 64);
    Int8Args a{q, p->weight, scale, p->weight_scale, p->bias, p->y, qr, p->weight_row, p->rows, p->inputs, p->outputs, tiles_n, tiles_n * ceil_div(p->rows, 64)};
    if (a.blocks > ((int64_t)kGridX << 15)) return fail_msg(TAE_EINVAL, "int8_linear: the product is too large for one call");
    return guarded([&] {
        hipStream_t st = (hipStream_t)stream;
        launch_quantize_dtype(QuantArgs{p->x, q, scale, p->x_row, qr, p->rows, p->inputs}, p->dtype, st);
        switch (p->dtype) {
            case TAE_DTYPE_F32: launch_int8<float>(a, st); break;
            case TAE_DTYPE_F16: launch_int8<f16>(a, st); break;
            default: launch_int8<bf16>(a, st); break;
        }
        return (int)TAE_OK;
    });
}

}  // extern "C"
