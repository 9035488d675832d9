// Row-wise operators around a matrix product: root-mean-square norm with the residual's addition (16-bit, FP32 or 8-bit result)
// and its gradients, e4m3 quantisation of rows and of a weight matrix, and the gradient of a product's epilogue.
//
// All are bound by HBM: every input is read once and every output written once.
//
//   norm      h = x + residual;  r_i = 1 / sqrt(mean_k h_ik^2 + eps);  y = h r w.  A row belongs to one CTA (or one warp) whose threads
//             hold it in registers as 32-bit floats between the sum of squares and the result, so nothing is read twice.  For an
//             e4m3 result the row's scale is amax_k |y_ik| / 448, found by a second reduction over the same registers.
//   gradient  with xhat = h r and g = dout w:  dh = r (g - xhat mean_k(g xhat)) + (gradient arriving at h),  dw_k = sum_i dout xhat.
//             CTAs stay on the GPU and take rows in turn; a thread keeps its columns' sums of dw in registers over all of its
//             rows, the next row's loads are under way during the reduction of the current one, and one partial row of dw per CTA
//             is added up by a second kernel in a fixed order: two calls give the same bits.
//   epilogue  C = act(Z + bias) + residual:  dZ = dC act'(Z + bias), dbias_j = sum_i dZ_ij (from the unrounded products), summed the
//             same way.
//
// Rows that are no whole 16-byte vectors (or buffers that do not start on 16 bytes) are accessed element by element by the same
// kernels; rows longer than a CTA's registers hold go through a form that reads them again from L2 instead.
#include <algorithm>
#include <cstring>

#include "esmm_dtypes.cuh"

namespace esmm {

constexpr int ROWS_MAX_PARTIALS = 592;   // rows of partial column sums that a backward pass may write (4 CTAs per SM)

// ---- access to VEC elements of T at a time -----------------------------------------------------------------------------
template <typename T, int VEC> struct Raw;
template <> struct Raw<float, 4> { typedef uint4 type; };
template <> struct Raw<__half, 8> { typedef uint4 type; };
template <> struct Raw<__nv_bfloat16, 8> { typedef uint4 type; };
template <typename T> struct Raw<T, 1> { typedef T type; };

template <typename T, int VEC>
__device__ __forceinline__ void unpack(const typename Raw<T, VEC>::type &raw, float (&v)[VEC])
{
    if constexpr (VEC == 1) {
        v[0] = to_float<T>(raw);
    } else {
        const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 4) {
                v[i] = __uint_as_float(w[i]);
            } else {
                const float2 f = std::is_same<T, __half>::value ? unpack_f16(w[i]) : unpack_bf16(w[i]);
                v[2 * i] = f.x;
                v[2 * i + 1] = f.y;
            }
        }
    }
}

template <typename T, int VEC>
__device__ __forceinline__ typename Raw<T, VEC>::type pack(const float (&v)[VEC])
{
    if constexpr (VEC == 1) {
        return from_float<T>(v[0]);
    } else {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 4) w[i] = __float_as_uint(v[i]);
            else w[i] = std::is_same<T, __half>::value ? pack_f16(v[2 * i], v[2 * i + 1]) : pack_bf16(v[2 * i], v[2 * i + 1]);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
}

template <typename T, int VEC>
__device__ __forceinline__ typename Raw<T, VEC>::type load_raw(const T *p)
{
    return *reinterpret_cast<const typename Raw<T, VEC>::type *>(p);
}

template <typename T, int VEC>
__device__ __forceinline__ void store_raw(T *p, const float (&v)[VEC])
{
    *reinterpret_cast<typename Raw<T, VEC>::type *>(p) = pack<T, VEC>(v);
}

template <int VEC>
__device__ __forceinline__ void store_e4m3(uint8_t *p, const float (&v)[VEC])
{
    if constexpr (VEC == 1) {
        *p = (uint8_t)pack_e4m3(v[0], 0.0f);
    } else {
        uint32_t w[VEC / 4];
#pragma unroll
        for (int i = 0; i < VEC / 4; ++i) w[i] = pack_e4m3(v[4 * i], v[4 * i + 1]) | (pack_e4m3(v[4 * i + 2], v[4 * i + 3]) << 16);
        if constexpr (VEC == 8) *reinterpret_cast<uint2 *>(p) = make_uint2(w[0], w[VEC / 4 - 1]);
        else *reinterpret_cast<uint32_t *>(p) = w[0];
    }
}

// ---- reductions over the threads of a row -------------------------------------------------------------------------------
__device__ __forceinline__ float warp_sum(float v)
{
#pragma unroll
    for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, d);
    return v;
}

__device__ __forceinline__ float warp_max(float v)
{
#pragma unroll
    for (int d = 16; d; d >>= 1) v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, d));
    return v;
}

// Over all warps of the CTA (one row per CTA) or, with one warp per row, over the warp.  `slots`: 32 floats of shared memory that no
// other reduction of the same row uses.
template <bool MAX>
__device__ __forceinline__ float row_reduce(float v, float *slots)
{
    v = MAX ? warp_max(v) : warp_sum(v);
    if (blockDim.x > 32) {
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
        if (lane == 0) slots[warp] = v;
        __syncthreads();
        v = lane < warps ? slots[lane] : 0.0f;
        v = MAX ? warp_max(v) : warp_sum(v);
    }
    return v;
}

struct NormParams {
    int M, K;
    float eps;
    const void *x, *residual, *weight;
    void *sum, *out;
    float *scale, *rstd;
    int *status;
};

// One row per blockDim.x threads (blockDim.y rows per CTA where a warp has a row of its own).  NORM = false: the rows themselves, only
// quantised.
template <typename T, int VEC, int NV, bool OUT8, bool NORM>
__global__ void __launch_bounds__(1024)
esmm_rmsnorm_kernel(const NormParams p)
{
    grid_dependency_wait();
    __shared__ float slots[64];
    typedef typename Raw<T, VEC>::type raw_t;
    const size_t row = (size_t)blockIdx.x * blockDim.y + threadIdx.y;
    if (row >= (size_t)p.M) return;              // (a whole warp; one row per CTA never leaves here)
    const size_t base = row * (size_t)p.K, end = (size_t)p.M * p.K;
    const T *x = static_cast<const T *>(p.x) + base;
    const T *res = p.residual ? static_cast<const T *>(p.residual) + base : nullptr;
    const T *weight = static_cast<const T *>(p.weight);
    float h[NV][VEC];
    raw_t w[NV];
    float ss = 0.0f;
    {
        raw_t xr[NV], rr[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (threadIdx.x + i * blockDim.x) * VEC;
            if (c < p.K) {
                xr[i] = load_raw<T, VEC>(x + c);
                if (res) rr[i] = load_raw<T, VEC>(res + c);
            }
        }
        if (NORM && weight) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = (threadIdx.x + i * blockDim.x) * VEC;
                if (c < p.K) w[i] = load_raw<T, VEC>(weight + c);
            }
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (threadIdx.x + i * blockDim.x) * VEC;
#pragma unroll
            for (int j = 0; j < VEC; ++j) h[i][j] = 0.0f;
            if (c < p.K) {
                unpack<T, VEC>(xr[i], h[i]);
                if (res) {
                    float r[VEC];
                    unpack<T, VEC>(rr[i], r);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) h[i][j] += r[j];
                }
                if (NORM && p.sum && bounds_ok(base + c + VEC <= end, p.status, 60)) store_raw<T, VEC>(static_cast<T *>(p.sum) + base + c, h[i]);   // checked build: site 60
            }
#pragma unroll
            for (int j = 0; j < VEC; ++j) ss = fmaf(h[i][j], h[i][j], ss);
        }
    }
    if (NORM) {
        ss = row_reduce<false>(ss, slots);
        const float rstd = __frsqrt_rn(ss / (float)p.K + p.eps);
        if (p.rstd && threadIdx.x == 0) p.rstd[row] = rstd;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float f[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) f[j] = 1.0f;
            if (weight && (threadIdx.x + i * blockDim.x) * VEC < p.K) unpack<T, VEC>(w[i], f);
#pragma unroll
            for (int j = 0; j < VEC; ++j) h[i][j] = h[i][j] * rstd * f[j];
        }
    }
    float inv = 1.0f;
    if (OUT8) {
        float amax = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < VEC; ++j) amax = fmaxf(amax, fabsf(h[i][j]));   // (NaN does not count)
        amax = row_reduce<true>(amax, slots + 32);
        const float scale = e4m3_scale(amax);
        inv = 1.0f / scale;
        if (threadIdx.x == 0) p.scale[row] = scale;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (threadIdx.x + i * blockDim.x) * VEC;
        if (c < p.K && bounds_ok(base + c + VEC <= end, p.status, 61)) {
            if constexpr (OUT8) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) h[i][j] *= inv;
                store_e4m3<VEC>(static_cast<uint8_t *>(p.out) + base + c, h[i]);
            } else {
                store_raw<T, VEC>(static_cast<T *>(p.out) + base + c, h[i]);
            }
        }
    }
}

// Rows longer than a CTA's registers: the statistics first, over rows that are read again (from L2) for the result.  Nothing is
// written before the last pass, in which every element is read and written by one thread, so the outputs may lie over the inputs here too.
template <typename T, bool OUT8, bool NORM>
__global__ void __launch_bounds__(1024)
esmm_rmsnorm_long_kernel(const NormParams p)
{
    grid_dependency_wait();
    __shared__ float slots[64];
    const size_t base = (size_t)blockIdx.x * (size_t)p.K;
    const T *x = static_cast<const T *>(p.x) + base;
    const T *res = p.residual ? static_cast<const T *>(p.residual) + base : nullptr;
    const T *weight = static_cast<const T *>(p.weight);
    auto h_at = [&](int c) { return to_float<T>(x[c]) + (res ? to_float<T>(res[c]) : 0.0f); };
    float rstd = 1.0f;
    if (NORM) {
        float ss = 0.0f;
        for (int c = threadIdx.x; c < p.K; c += blockDim.x) ss = fmaf(h_at(c), h_at(c), ss);
        ss = row_reduce<false>(ss, slots);
        rstd = __frsqrt_rn(ss / (float)p.K + p.eps);
        if (p.rstd && threadIdx.x == 0) p.rstd[blockIdx.x] = rstd;
    }
    auto y_at = [&](float h, int c) { return NORM ? h * rstd * (weight ? to_float<T>(weight[c]) : 1.0f) : h; };
    float inv = 1.0f;
    if (OUT8) {
        float amax = 0.0f;
        for (int c = threadIdx.x; c < p.K; c += blockDim.x) amax = fmaxf(amax, fabsf(y_at(h_at(c), c)));
        amax = row_reduce<true>(amax, slots + 32);
        const float scale = e4m3_scale(amax);
        inv = 1.0f / scale;
        if (threadIdx.x == 0) p.scale[blockIdx.x] = scale;
    }
    for (int c = threadIdx.x; c < p.K; c += blockDim.x) {
        const float h = h_at(c), y = y_at(h, c);
        if (NORM && p.sum) static_cast<T *>(p.sum)[base + c] = from_float<T>(h);
        if (OUT8) static_cast<uint8_t *>(p.out)[base + c] = (uint8_t)pack_e4m3(y * inv, 0.0f);
        else static_cast<T *>(p.out)[base + c] = from_float<T>(y);
    }
}

// ---- the norm's gradients -----------------------------------------------------------------------------------------------
struct NormGradParams {
    int M, K;
    const void *dout, *h, *weight, *dsum;
    const float *rstd;
    void *dx;
    float *partial;      // one row of K sums per CTA
    int *status;
};

template <typename T, int VEC, int NV>
__global__ void __launch_bounds__(1024)
esmm_rmsnorm_backward_kernel(const NormGradParams p)
{
    grid_dependency_wait();
    __shared__ float slots[64];
    typedef typename Raw<T, VEC>::type raw_t;
    const T *weight = static_cast<const T *>(p.weight);
    const T *dout = static_cast<const T *>(p.dout), *h = static_cast<const T *>(p.h), *dsum = static_cast<const T *>(p.dsum);
    float dw[NV][VEC];
    raw_t w[NV], g_raw[NV], h_raw[NV], s_raw[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (threadIdx.x + i * blockDim.x) * VEC;
#pragma unroll
        for (int j = 0; j < VEC; ++j) dw[i][j] = 0.0f;
        if (weight && c < p.K) w[i] = load_raw<T, VEC>(weight + c);
    }
    float rstd_next = 0.0f;
    auto load_row = [&](size_t row) {
        const size_t base = row * (size_t)p.K;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (threadIdx.x + i * blockDim.x) * VEC;
            if (c < p.K) {
                g_raw[i] = load_raw<T, VEC>(dout + base + c);
                h_raw[i] = load_raw<T, VEC>(h + base + c);
                if (dsum) s_raw[i] = load_raw<T, VEC>(dsum + base + c);
            }
        }
        rstd_next = p.rstd[row];
    };
    load_row(blockIdx.x);
    int turn = 0;
    for (size_t row = blockIdx.x; row < (size_t)p.M; row += gridDim.x, turn ^= 32) {
        const size_t base = row * (size_t)p.K;
        const float rstd = rstd_next;
        float gw[NV][VEC], xh[NV][VEC], add[NV][VEC], dot = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (threadIdx.x + i * blockDim.x) * VEC;
#pragma unroll
            for (int j = 0; j < VEC; ++j) gw[i][j] = xh[i][j] = add[i][j] = 0.0f;
            if (c < p.K) {
                unpack<T, VEC>(g_raw[i], gw[i]);
                unpack<T, VEC>(h_raw[i], xh[i]);
                if (dsum) unpack<T, VEC>(s_raw[i], add[i]);
                float f[VEC];
#pragma unroll
                for (int j = 0; j < VEC; ++j) f[j] = 1.0f;
                if (weight) unpack<T, VEC>(w[i], f);
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    xh[i][j] *= rstd;
                    dw[i][j] = fmaf(gw[i][j], xh[i][j], dw[i][j]);
                    gw[i][j] *= f[j];
                    dot = fmaf(gw[i][j], xh[i][j], dot);
                }
            }
        }
        if (row + gridDim.x < (size_t)p.M) load_row(row + gridDim.x);
        // (two sets of slots in turn: a warp may be a row ahead of the slowest one's reads)
        dot = row_reduce<false>(dot, slots + turn) / (float)p.K;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (threadIdx.x + i * blockDim.x) * VEC;
            if (c < p.K && bounds_ok(base + c + VEC <= (size_t)p.M * p.K, p.status, 62)) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) gw[i][j] = fmaf(rstd, fmaf(-xh[i][j], dot, gw[i][j]), add[i][j]);
                store_raw<T, VEC>(static_cast<T *>(p.dx) + base + c, gw[i]);
            }
        }
    }
    if (p.partial) {
        float *to = p.partial + (size_t)blockIdx.x * p.K;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (threadIdx.x + i * blockDim.x) * VEC;
            if (c < p.K)
#pragma unroll
                for (int j = 0; j < VEC; ++j) to[c + j] = dw[i][j];
        }
    }
}

// Rows longer than a CTA's registers: read twice, the sums of dw in the CTA's row of the workspace.
template <typename T>
__global__ void __launch_bounds__(1024)
esmm_rmsnorm_backward_long_kernel(const NormGradParams p)
{
    grid_dependency_wait();
    __shared__ float slots[64];
    const T *weight = static_cast<const T *>(p.weight);
    float *to = p.partial ? p.partial + (size_t)blockIdx.x * p.K : nullptr;
    int turn = 0;
    for (size_t row = blockIdx.x; row < (size_t)p.M; row += gridDim.x, turn ^= 32) {
        const size_t base = row * (size_t)p.K;
        const T *dout = static_cast<const T *>(p.dout) + base, *h = static_cast<const T *>(p.h) + base;
        const T *dsum = p.dsum ? static_cast<const T *>(p.dsum) + base : nullptr;
        const float rstd = p.rstd[row];
        float dot = 0.0f;
        for (int c = threadIdx.x; c < p.K; c += blockDim.x)
            dot = fmaf(to_float<T>(dout[c]) * (weight ? to_float<T>(weight[c]) : 1.0f), to_float<T>(h[c]) * rstd, dot);
        dot = row_reduce<false>(dot, slots + turn) / (float)p.K;
        for (int c = threadIdx.x; c < p.K; c += blockDim.x) {
            const float g = to_float<T>(dout[c]), xh = to_float<T>(h[c]) * rstd;
            if (to) to[c] = row == blockIdx.x ? g * xh : fmaf(g, xh, to[c]);
            const float gw = g * (weight ? to_float<T>(weight[c]) : 1.0f);
            static_cast<T *>(p.dx)[base + c] = from_float<T>(fmaf(rstd, fmaf(-xh, dot, gw), dsum ? to_float<T>(dsum[c]) : 0.0f));
        }
    }
}

// out[c] = sum over `rows` rows of partial[r][c], in a fixed order: 32 columns per CTA, thread row y takes rows y, y + 32, ..., the 32
// sums are added as a tree.
template <typename T>
__global__ void __launch_bounds__(1024)
esmm_column_sum_kernel(const float *partial, int rows, int K, T *out)
{
    grid_dependency_wait();
    __shared__ float sums[32][33];
    const int c = blockIdx.x * 32 + threadIdx.x;
    float s0 = 0.0f, s1 = 0.0f, s2 = 0.0f, s3 = 0.0f;
    if (c < K) {
        const float *at = partial + c;
        int r = threadIdx.y;
        for (; r + 96 < rows; r += 128) {
            s0 += at[(size_t)r * K];
            s1 += at[(size_t)(r + 32) * K];
            s2 += at[(size_t)(r + 64) * K];
            s3 += at[(size_t)(r + 96) * K];
        }
        for (; r < rows; r += 32) s0 += at[(size_t)r * K];
    }
    sums[threadIdx.y][threadIdx.x] = (s0 + s1) + (s2 + s3);
    __syncthreads();
    const float s = warp_sum(sums[threadIdx.x][threadIdx.y]);   // thread row y adds up column y
    if (threadIdx.x == 0 && blockIdx.x * 32 + threadIdx.y < K) out[blockIdx.x * 32 + threadIdx.y] = from_float<T>(s);
}

// ---- gradient of a product's epilogue --------------------------------------------------------------------------------------
// A CTA takes 32 * VEC columns and a run of rows, eight rows at a time (one per warp); its sums of dZ go to one partial row.
struct EpiGradParams {
    int M, N, activation, rows_per;
    const void *dc, *pre;
    void *dz;
    float *partial;
    int *status;
};

template <typename T>
__global__ void __launch_bounds__(256)
esmm_epilogue_backward_kernel(const EpiGradParams p)
{
    grid_dependency_wait();
    constexpr int VEC = 16 / sizeof(T), U = 4;         // rows in flight per warp
    typedef typename Raw<T, VEC>::type raw_t;
    __shared__ float sums[8][32 * VEC];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int col = (blockIdx.x * 32 + lane) * VEC;
    const int r0 = blockIdx.y * p.rows_per, r1 = min(p.M, r0 + p.rows_per);
    const T *dc = static_cast<const T *>(p.dc), *pre = static_cast<const T *>(p.pre);
    float acc[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[j] = 0.0f;
    if (col < p.N) {
        for (int r = r0 + warp; r < r1; r += 8 * U) {
            raw_t g[U], z[U];
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (r + 8 * u < r1) {
                    g[u] = load_raw<T, VEC>(dc + (size_t)(r + 8 * u) * p.N + col);
                    if (pre) z[u] = load_raw<T, VEC>(pre + (size_t)(r + 8 * u) * p.N + col);
                }
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (r + 8 * u < r1) {
                    float gf[VEC];
                    unpack<T, VEC>(g[u], gf);
                    if (pre) {
                        float zf[VEC];
                        unpack<T, VEC>(z[u], zf);
                        with_activation(p.activation, [&](auto tag) {
#pragma unroll
                            for (int j = 0; j < VEC; ++j) gf[j] *= activate_grad<decltype(tag)::value>(zf[j]);
                        });
                    }
#pragma unroll
                    for (int j = 0; j < VEC; ++j) acc[j] += gf[j];
                    const size_t off = (size_t)(r + 8 * u) * p.N + col;
                    if (p.dz && bounds_ok(off + VEC <= (size_t)p.M * p.N, p.status, 63)) store_raw<T, VEC>(static_cast<T *>(p.dz) + off, gf);
                }
        }
    }
    if (p.partial) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) sums[warp][lane * VEC + j] = acc[j];
        __syncthreads();
        for (int c = threadIdx.x; c < 32 * VEC; c += 256) {
            const int to = blockIdx.x * 32 * VEC + c;
            float s = 0.0f;
#pragma unroll
            for (int w = 0; w < 8; ++w) s += sums[w][c];
            if (to < p.N) p.partial[(size_t)blockIdx.y * p.N + to] = s;
        }
    }
}

// ---- a weight matrix in e4m3, transposed ------------------------------------------------------------------------------------
// scale[n] = amax_k |B[k][n]| / 448: 32 columns per CTA, 32 rows at a time.
template <typename T>
__global__ void __launch_bounds__(1024)
esmm_column_scale_kernel(const T *B, int K, int N, float *scale)
{
    grid_dependency_wait();
    __shared__ float part[32][33];
    const int n = blockIdx.x * 32 + threadIdx.x;
    float amax = 0.0f;
    if (n < N)
        for (int k = threadIdx.y; k < K; k += 32) amax = fmaxf(amax, fabsf(to_float<T>(B[(size_t)k * N + n])));
    part[threadIdx.y][threadIdx.x] = amax;
    __syncthreads();
    amax = warp_max(part[threadIdx.x][threadIdx.y]);
    const int to = blockIdx.x * 32 + threadIdx.y;
    if (threadIdx.x == 0 && to < N) scale[to] = e4m3_scale(amax);
}

// bt[n][k] = e4m3(B[k][n] / scale[n]): tiles of 128 k x 32 n through shared memory, four codes of a row per store
template <typename T>
__global__ void __launch_bounds__(256)
esmm_quantize_transpose_kernel(const T *B, int K, int N, const float *scale, uint8_t *bt)
{
    grid_dependency_wait();
    __shared__ float tile[128][33];
    const int k0 = blockIdx.y * 128, n0 = blockIdx.x * 32;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const float inv = n0 + lane < N ? 1.0f / scale[n0 + lane] : 0.0f;
    for (int r = warp; r < 128; r += 8)
        tile[r][lane] = k0 + r < K && n0 + lane < N ? to_float<T>(B[(size_t)(k0 + r) * N + n0 + lane]) * inv : 0.0f;
    __syncthreads();
    for (int c = warp; c < 32; c += 8) {
        const int n = n0 + c, k = k0 + lane * 4;
        if (n < N && k < K)   // (K is a multiple of 16)
            *reinterpret_cast<uint32_t *>(bt + (size_t)n * K + k) =
                pack_e4m3(tile[lane * 4][c], tile[lane * 4 + 1][c]) | (pack_e4m3(tile[lane * 4 + 2][c], tile[lane * 4 + 3][c]) << 16);
    }
}

// ---- launches -------------------------------------------------------------------------------------------------------------------
static bool aligned16(std::initializer_list<const void *> ptrs)
{
    uintptr_t bits = 0;
    for (const void *q : ptrs) bits |= (uintptr_t)q;
    return (bits & 15) == 0;
}

// Rows of more than this many per SM are taken with several vectors per thread: fewer threads per row, so that more rows are in
// flight and a thread has more loads of its own under way.  Fewer rows get one vector per thread: a row alone on its SM is
// through sooner the more warps load it.
constexpr int NORM_ROWS_PER_SM = 8;

static int sm_count(int *sms)
{
    int dev = 0;
    ESMM_CUDA_TRY(cudaGetDevice(&dev));
    ESMM_CUDA_TRY(cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev));
    return ESMM_OK;
}

template <typename T, bool OUT8, bool NORM>
static int norm_launch_type(const NormParams &p, bool vectors, int sms, cudaStream_t stream)
{
    constexpr int VEC = 16 / (int)sizeof(T);
    const bool many = (long)p.M > (long)NORM_ROWS_PER_SM * sms;
    auto go = [&](auto kernel, int vec, int nv) -> int {
        const int warps = ceil_div(ceil_div(p.K, vec * nv), 32);
        const int rows = warps == 1 ? 8 : 1;
        ESMM_CUDA_TRY(launch_dependent(kernel, dim3((unsigned)ceil_div(p.M, rows)), dim3(warps * 32, rows), 0, stream, p));
        return ESMM_OK;
    };
    const int units = vectors ? ceil_div(p.K, VEC) : p.K;
    if (vectors) {
        if (units > 1024 * 4 || (many && units > 32 * 2)) {
            if (units <= 1024 * 4) return go(esmm_rmsnorm_kernel<T, VEC, 4, OUT8, NORM>, VEC, 4);
        } else {
            if (units <= (many ? 32 : 1024)) return go(esmm_rmsnorm_kernel<T, VEC, 1, OUT8, NORM>, VEC, 1);
            if (units <= 1024 * 2) return go(esmm_rmsnorm_kernel<T, VEC, 2, OUT8, NORM>, VEC, 2);
            return go(esmm_rmsnorm_kernel<T, VEC, 4, OUT8, NORM>, VEC, 4);
        }
    } else {
        if (units <= 32 * 4 || (!many && units <= 1024 * 4)) return go(esmm_rmsnorm_kernel<T, 1, 4, OUT8, NORM>, 1, 4);
        if (units <= 1024 * 16) return go(esmm_rmsnorm_kernel<T, 1, 16, OUT8, NORM>, 1, 16);
    }
    ESMM_CUDA_TRY(launch_dependent(esmm_rmsnorm_long_kernel<T, OUT8, NORM>, dim3((unsigned)p.M), dim3(1024), 0, stream, p));
    return ESMM_OK;
}

template <bool NORM>
static int norm_launch(const NormParams &p, int dtype, bool out8, bool vectors, cudaStream_t stream)
{
    int sms = 0;
    const int st = sm_count(&sms);
    if (st != ESMM_OK) return st;
    if (out8) {
        if (dtype == ESMM_F32) return norm_launch_type<float, true, NORM>(p, vectors, sms, stream);
        if (dtype == ESMM_F16) return norm_launch_type<__half, true, NORM>(p, vectors, sms, stream);
        return norm_launch_type<__nv_bfloat16, true, NORM>(p, vectors, sms, stream);
    }
    if constexpr (NORM) {
        if (dtype == ESMM_F32) return norm_launch_type<float, false, true>(p, vectors, sms, stream);
        if (dtype == ESMM_F16) return norm_launch_type<__half, false, true>(p, vectors, sms, stream);
        return norm_launch_type<__nv_bfloat16, false, true>(p, vectors, sms, stream);
    }
    return ESMM_ERR_UNSUPPORTED;
}

static bool row_dtype(int dtype) { return dtype == ESMM_F32 || dtype == ESMM_F16 || dtype == ESMM_BF16; }

static bool element_aligned(const void *p, int bytes) { return ((uintptr_t)p & (uintptr_t)(bytes - 1)) == 0; }

template <typename T>
static int norm_backward_type(const NormGradParams &p, bool vectors, int sms, int *ctas, cudaStream_t stream)
{
    constexpr int VEC = 16 / (int)sizeof(T);
    auto go = [&](auto kernel, int threads) -> int {
        int per_sm = 0;
        ESMM_CUDA_TRY(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, threads, 0));
        *ctas = std::max(1, std::min(std::min(p.M, ROWS_MAX_PARTIALS), sms * std::max(1, std::min(per_sm, 4))));
        ESMM_CUDA_TRY(launch_dependent(kernel, dim3((unsigned)*ctas), dim3(threads), 0, stream, p));
        return ESMM_OK;
    };
    auto threads_for = [&](int vec, int nv) { return ceil_div(ceil_div(p.K, vec * nv), 32) * 32; };
    if (vectors) {
        const int units = ceil_div(p.K, VEC);
        if (units <= 512) return go(esmm_rmsnorm_backward_kernel<T, VEC, 1>, threads_for(VEC, 1));
        if (units <= 2048) return go(esmm_rmsnorm_backward_kernel<T, VEC, 2>, threads_for(VEC, 2));
    } else {
        if (p.K <= 2048) return go(esmm_rmsnorm_backward_kernel<T, 1, 4>, threads_for(1, 4));
        if (p.K <= 8192) return go(esmm_rmsnorm_backward_kernel<T, 1, 8>, threads_for(1, 8));
    }
    return go(esmm_rmsnorm_backward_long_kernel<T>, 1024);
}

static int column_sum(const float *partial, int rows, int K, int dtype, void *out, cudaStream_t stream)
{
    auto go = [&](auto tag) -> int {
        typedef decltype(tag) T;
        ESMM_CUDA_TRY(launch_dependent(esmm_column_sum_kernel<T>, dim3((unsigned)ceil_div(K, 32)), dim3(32, 32), 0, stream, partial, rows, K,
                                       static_cast<T *>(out)));
        return ESMM_OK;
    };
    return dtype == ESMM_F32 ? go(float()) : dtype == ESMM_F16 ? go(__half()) : go(__nv_bfloat16());
}

}  // namespace esmm

extern "C" {

int esmm_rmsnorm(int M, int K, int dtype, const void *d_x, const void *d_residual, const void *d_weight, float eps, void *d_sum,
                 int out_dtype, void *d_out, float *d_scale, float *d_rstd, void *stream)
{
    using namespace esmm;
    const bool out8 = out_dtype == ESMM_E4M3;
    if (!d_x || !d_out || (out8 && !d_scale)) return ESMM_ERR_NULL;
    if (M <= 0 || K <= 0) return ESMM_ERR_SHAPE;
    if (!row_dtype(dtype) || (!out8 && out_dtype != dtype)) return ESMM_ERR_UNSUPPORTED;
    const int size = dtype_bytes(dtype);
    for (const void *q : {d_x, d_residual, d_weight, (const void *)d_sum, (const void *)(out8 ? nullptr : d_out)})
        if (!element_aligned(q, size)) return ESMM_ERR_ALIGN;
    if (!element_aligned(d_scale, 4) || !element_aligned(d_rstd, 4)) return ESMM_ERR_ALIGN;
    NormParams p;
    memset(&p, 0, sizeof p);
    p.M = M;
    p.K = K;
    p.eps = eps;
    p.x = d_x;
    p.residual = d_residual;
    p.weight = d_weight;
    p.sum = d_sum;
    p.out = d_out;
    p.scale = d_scale;
    p.rstd = d_rstd;
    p.status = device_status_ptr();
    if (!p.status) return ESMM_ERR_CUDA;
    const bool vectors = K % (16 / size) == 0 && aligned16({d_x, d_residual, d_weight, d_sum, d_out});
    return norm_launch<true>(p, dtype, out8, vectors, (cudaStream_t)stream);
}

int esmm_quantize_rows(int M, int K, int dtype, const void *d_x, void *d_out, float *d_scale, void *stream)
{
    using namespace esmm;
    if (!d_x || !d_out || !d_scale) return ESMM_ERR_NULL;
    if (M <= 0 || K <= 0) return ESMM_ERR_SHAPE;
    if (!row_dtype(dtype)) return ESMM_ERR_UNSUPPORTED;
    const int size = dtype_bytes(dtype);
    if (!element_aligned(d_x, size) || !element_aligned(d_scale, 4)) return ESMM_ERR_ALIGN;
    NormParams p;
    memset(&p, 0, sizeof p);
    p.M = M;
    p.K = K;
    p.x = d_x;
    p.out = d_out;
    p.scale = d_scale;
    p.status = device_status_ptr();
    if (!p.status) return ESMM_ERR_CUDA;
    return norm_launch<false>(p, dtype, true, K % (16 / size) == 0 && aligned16({d_x, d_out}), (cudaStream_t)stream);
}

size_t esmm_rmsnorm_backward_workspace_bytes(int M, int K)
{
    if (M <= 0 || K <= 0) return 0;
    return (size_t)std::min(M, esmm::ROWS_MAX_PARTIALS) * K * sizeof(float);
}

int esmm_rmsnorm_backward(int M, int K, int dtype, const void *d_dout, const void *d_h, const void *d_weight, const float *d_rstd,
                          const void *d_dsum, void *d_dx, void *d_dweight, void *d_workspace, void *stream_)
{
    using namespace esmm;
    cudaStream_t stream = (cudaStream_t)stream_;
    if (!d_dout || !d_h || !d_rstd || !d_dx || (d_dweight && !d_workspace)) return ESMM_ERR_NULL;
    if (M <= 0 || K <= 0) return ESMM_ERR_SHAPE;
    if (!row_dtype(dtype)) return ESMM_ERR_UNSUPPORTED;
    const int size = dtype_bytes(dtype);
    for (const void *q : {d_dout, d_h, d_weight, d_dsum, (const void *)d_dx, (const void *)d_dweight})
        if (!element_aligned(q, size)) return ESMM_ERR_ALIGN;
    if (!element_aligned(d_rstd, 4) || ((uintptr_t)d_workspace & 15)) return ESMM_ERR_ALIGN;
    NormGradParams p;
    memset(&p, 0, sizeof p);
    p.M = M;
    p.K = K;
    p.dout = d_dout;
    p.h = d_h;
    p.weight = d_weight;
    p.dsum = d_dsum;
    p.rstd = d_rstd;
    p.dx = d_dx;
    p.partial = d_dweight ? static_cast<float *>(d_workspace) : nullptr;
    p.status = device_status_ptr();
    if (!p.status) return ESMM_ERR_CUDA;
    int sms = 0, ctas = 0;
    int st = sm_count(&sms);
    if (st != ESMM_OK) return st;
    const bool vectors = K % (16 / size) == 0 && aligned16({d_dout, d_h, d_weight, d_dsum, d_dx});
    if (dtype == ESMM_F32) st = norm_backward_type<float>(p, vectors, sms, &ctas, stream);
    else if (dtype == ESMM_F16) st = norm_backward_type<__half>(p, vectors, sms, &ctas, stream);
    else st = norm_backward_type<__nv_bfloat16>(p, vectors, sms, &ctas, stream);
    if (st != ESMM_OK || !d_dweight) return st;
    return column_sum(p.partial, ctas, K, dtype, d_dweight, stream);
}

size_t esmm_epilogue_backward_workspace_bytes(int M, int N)
{
    if (M <= 0 || N <= 0) return 0;
    return (size_t)std::min(esmm::ceil_div(M, 8), esmm::ROWS_MAX_PARTIALS) * N * sizeof(float);
}

int esmm_epilogue_backward(int M, int N, int dtype, const void *d_dC, const void *d_pre, int activation, void *d_dZ, void *d_dbias,
                           void *d_workspace, void *stream_)
{
    using namespace esmm;
    cudaStream_t stream = (cudaStream_t)stream_;
    if (!d_dC || (!d_dZ && !d_dbias) || (d_dbias && !d_workspace)) return ESMM_ERR_NULL;
    if (activation_known(activation) && activation != ESMM_ACT_NONE && !d_pre) return ESMM_ERR_NULL;
    if (!row_dtype(dtype) || !activation_known(activation)) return ESMM_ERR_UNSUPPORTED;
    const int vec = 16 / dtype_bytes(dtype);
    if (M <= 0 || N <= 0 || N % vec) return ESMM_ERR_SHAPE;
    if (!aligned16({d_dC, d_pre, d_dZ, d_workspace}) || !element_aligned(d_dbias, dtype_bytes(dtype))) return ESMM_ERR_ALIGN;
    EpiGradParams p;
    memset(&p, 0, sizeof p);
    p.M = M;
    p.N = N;
    p.activation = activation;
    p.dc = d_dC;
    p.pre = activation == ESMM_ACT_NONE ? nullptr : d_pre;
    p.dz = d_dZ;
    p.partial = d_dbias ? static_cast<float *>(d_workspace) : nullptr;
    p.status = device_status_ptr();
    if (!p.status) return ESMM_ERR_CUDA;
    int sms = 0;
    const int st = sm_count(&sms);
    if (st != ESMM_OK) return st;
    // about eight CTAs per SM, eight rows at least for each
    const int across = ceil_div(N, 32 * vec);
    const int down = std::max(1, std::min(std::min(ceil_div(M, 8), ROWS_MAX_PARTIALS), ceil_div(8 * sms, across)));
    p.rows_per = ceil_div(M, down);
    const int runs = ceil_div(M, p.rows_per);
    auto go = [&](auto kernel) -> int {
        ESMM_CUDA_TRY(launch_dependent(kernel, dim3((unsigned)across, (unsigned)runs), dim3(256), 0, stream, p));
        return ESMM_OK;
    };
    const int lst = dtype == ESMM_F32   ? go(esmm_epilogue_backward_kernel<float>)
                    : dtype == ESMM_F16 ? go(esmm_epilogue_backward_kernel<__half>)
                                        : go(esmm_epilogue_backward_kernel<__nv_bfloat16>);
    if (lst != ESMM_OK || !d_dbias) return lst;
    return column_sum(p.partial, runs, N, dtype, d_dbias, stream);
}

int esmm_quantize_b(int K, int N, int dtype, const void *d_B, void *d_bt, float *d_scale, void *stream_)
{
    using namespace esmm;
    cudaStream_t stream = (cudaStream_t)stream_;
    if (!d_B || !d_bt || !d_scale) return ESMM_ERR_NULL;
    if (K <= 0 || N <= 0 || K % 16) return ESMM_ERR_SHAPE;
    if (!row_dtype(dtype)) return ESMM_ERR_UNSUPPORTED;
    if (!element_aligned(d_B, dtype_bytes(dtype)) || ((uintptr_t)d_bt & 15) || !element_aligned(d_scale, 4)) return ESMM_ERR_ALIGN;
    if (ceil_div(K, 128) > 65535) return ESMM_ERR_TOO_LARGE;
    auto go = [&](auto tag) -> int {
        typedef decltype(tag) T;
        const T *B = static_cast<const T *>(d_B);
        ESMM_CUDA_TRY(launch_dependent(esmm_column_scale_kernel<T>, dim3((unsigned)ceil_div(N, 32)), dim3(32, 32), 0, stream, B, K, N, d_scale));
        ESMM_CUDA_TRY(launch_dependent(esmm_quantize_transpose_kernel<T>, dim3((unsigned)ceil_div(N, 32), (unsigned)ceil_div(K, 128)), dim3(256),
                                       0, stream, B, K, N, (const float *)d_scale, static_cast<uint8_t *>(d_bt)));
        return ESMM_OK;
    };
    return dtype == ESMM_F32 ? go(float()) : dtype == ESMM_F16 ? go(__half()) : go(__nv_bfloat16());
}

}  // extern "C"
