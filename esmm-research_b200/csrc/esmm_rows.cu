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
//             rows, rows come some ahead as bulk copies, and one partial row of dw per CTA is added up by a second kernel in a fixed
//             order: two calls give the same bits.
//   epilogue  C = act(Z + bias) + residual:  dZ = dC act'(Z + bias), dbias_j = sum_i dZ_ij (from the unrounded products), summed the
//             same way.
//
// Rows that are no whole 16-byte vectors, and buffers that do not start on 16 bytes, have forms of their own; rows longer than a CTA's
// registers hold go through a form that reads them again from L2 instead.
//
// Measured, of HBM's copy rate (one B200): norm with residual 8192 x 4096 bf16 41.8 us (98 %), to e4m3 37.1 (97 %); its gradients 46.6 (88 %:
// 3.5 us for adding up dw); rows to e4m3 18.5 (83 %); epilogue's gradient with silu and bias 2048 x 11008 bf16 27.8 (74 %, the exponentials).
#include <algorithm>
#include <atomic>
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
    grid_launch_dependents();
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
            if (c < p.K && bounds_ok(base + c + VEC <= end, p.status, 59)) {   // checked build: site 59
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
    float inv = 1.0f, scale = 1.0f;
    if (OUT8) {
        float amax = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < VEC; ++j) amax = fmaxf(amax, fabsf(h[i][j]));   // (NaN does not count)
        amax = row_reduce<true>(amax, slots + 32);
        scale = e4m3_scale(amax);
        inv = 1.0f / scale;
        if (threadIdx.x == 0) p.scale[row] = scale;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (threadIdx.x + i * blockDim.x) * VEC;
        if (c < p.K && bounds_ok(base + c + VEC <= end, p.status, 61)) {
            if constexpr (OUT8) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) h[i][j] = e4m3_quotient(h[i][j], scale, inv);
                store_e4m3<VEC>(static_cast<uint8_t *>(p.out) + base + c, h[i]);
            } else {
                store_raw<T, VEC>(static_cast<T *>(p.out) + base + c, h[i]);
            }
        }
    }
}

// Rows that are no whole vectors, in buffers that start on 16 bytes: a thread takes aligned vectors of the matrix as it lies, which hold the
// end of the row before and the start of the row after at the row's two ends.  Those elements count for nothing, and such vectors are
// written element by element (8192 x 1021 of bf16 with a residual, element by element throughout 32.6 us, so 20.8; HBM alone 10.2).
template <typename T, int VEC, int NV, bool OUT8, bool NORM>
__global__ void __launch_bounds__(1024)
esmm_rmsnorm_ragged_kernel(const NormParams p)
{
    grid_launch_dependents();
    grid_dependency_wait();
    __shared__ float slots[64];
    typedef typename Raw<T, VEC>::type raw_t;
    const size_t row = (size_t)blockIdx.x * blockDim.y + threadIdx.y;
    if (row >= (size_t)p.M) return;              // (a whole warp; one row per CTA never leaves here)
    const size_t begin = row * (size_t)p.K;
    const int lead = (int)(begin % VEC);                             // elements of the row before in the first vector
    const size_t first = begin - lead, left = (size_t)p.M * p.K - first;
    const T *x = static_cast<const T *>(p.x) + first, *res = static_cast<const T *>(p.residual), *weight = static_cast<const T *>(p.weight);
    if (res) res += first;
    // vector i of this thread starts at element off(i) from `first`, which is column off(i) - lead of the row; here(i): it holds some of the
    // row, whole(i): nothing else; in(i, j): its element j belongs to the row
    auto off = [&](int i) { return (int)(threadIdx.x + i * blockDim.x) * VEC; };
    auto here = [&](int i) { return off(i) < p.K + lead; };
    auto whole = [&](int i) { return off(i) >= lead && off(i) + VEC <= p.K + lead; };
    auto in = [&](int i, int j) { return off(i) + j >= lead && off(i) + j < p.K + lead; };
    auto loadable = [&](int i) { return (size_t)(off(i) + VEC) <= left; };   // the matrix does not end inside it
    // checked build, sites 67 (vectors), 68 (elements), 69 (weights), 70 (results): `n` elements from element j of vector i lie in the row, or, with their neighbours, in the matrix
    auto in_row = [&](int i, int j, int n, int site) {
        if constexpr (kCheckedBuild) return bounds_ok(first + off(i) + j >= begin && first + off(i) + j + n <= begin + p.K && row < (size_t)p.M, p.status, site);
        return true;
    };
    auto in_matrix = [&](int i) {
        if constexpr (kCheckedBuild) return bounds_ok(first + off(i) + VEC <= (size_t)p.M * p.K, p.status, 67);
        return true;
    };
    float h[NV][VEC];
    float ss = 0.0f;
    {
        raw_t xr[NV], rr[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (here(i) && loadable(i) && in_matrix(i)) {
                xr[i] = load_raw<T, VEC>(x + off(i));
                if (res) rr[i] = load_raw<T, VEC>(res + off(i));
            }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) h[i][j] = 0.0f;
            if (!here(i)) continue;
            if (loadable(i)) {
                unpack<T, VEC>(xr[i], h[i]);
                if (res) {
                    float r[VEC];
                    unpack<T, VEC>(rr[i], r);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) h[i][j] += r[j];
                }
            } else {
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    if (in(i, j) && in_row(i, j, 1, 68)) h[i][j] = to_float<T>(x[off(i) + j]) + (res ? to_float<T>(res[off(i) + j]) : 0.0f);
            }
            T *to = static_cast<T *>(p.sum) + first + off(i);
            if (whole(i)) {
                if (NORM && p.sum && in_row(i, 0, VEC, 70)) store_raw<T, VEC>(to, h[i]);
            } else {
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    if (NORM && p.sum && in(i, j) && in_row(i, j, 1, 70)) to[j] = from_float<T>(h[i][j]);
                    if (!in(i, j)) h[i][j] = 0.0f;                   // (counts for nothing from here on)
                }
            }
#pragma unroll
            for (int j = 0; j < VEC; ++j) ss = fmaf(h[i][j], h[i][j], ss);
        }
    }
    if (NORM) {
        float w[NV][VEC];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) w[i][j] = 1.0f;
            if (!weight || !here(i)) continue;
            const T *from = weight + (off(i) - lead);
            if (whole(i)) {
                if (!in_row(i, 0, VEC, 69)) continue;
                if (VEC == 8 && (lead & 1) == 0) {                   // pairs on their own alignment
                    const uint32_t *pairs = reinterpret_cast<const uint32_t *>(from);
#pragma unroll
                    for (int j = 0; j < VEC; j += 2) {
                        const float2 f = std::is_same<T, __half>::value ? unpack_f16(pairs[j / 2]) : unpack_bf16(pairs[j / 2]);
                        w[i][j] = f.x, w[i][j + 1] = f.y;
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < VEC; ++j) w[i][j] = to_float<T>(from[j]);
                }
            } else {
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    if (in(i, j) && in_row(i, j, 1, 69)) w[i][j] = to_float<T>(from[j]);
            }
        }
        ss = row_reduce<false>(ss, slots);
        const float rstd = __frsqrt_rn(ss / (float)p.K + p.eps);
        if (p.rstd && threadIdx.x == 0) p.rstd[row] = rstd;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < VEC; ++j) h[i][j] = h[i][j] * rstd * w[i][j];
    }
    float inv = 1.0f, scale = 1.0f;
    if (OUT8) {
        float amax = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (here(i)) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) amax = fmaxf(amax, whole(i) || in(i, j) ? fabsf(h[i][j]) : 0.0f);
            }
        amax = row_reduce<true>(amax, slots + 32);
        scale = e4m3_scale(amax);
        inv = 1.0f / scale;
        if (threadIdx.x == 0) p.scale[row] = scale;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        if (!here(i)) continue;
        if constexpr (OUT8) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) h[i][j] = e4m3_quotient(h[i][j], scale, inv);
            uint8_t *to = static_cast<uint8_t *>(p.out) + first + off(i);
            if (whole(i)) {
                if (in_row(i, 0, VEC, 70)) store_e4m3<VEC>(to, h[i]);
            } else {
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    if (in(i, j) && in_row(i, j, 1, 70)) to[j] = (uint8_t)pack_e4m3(h[i][j], 0.0f);
            }
        } else {
            T *to = static_cast<T *>(p.out) + first + off(i);
            if (whole(i)) {
                if (in_row(i, 0, VEC, 70)) store_raw<T, VEC>(to, h[i]);
            } else {
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    if (in(i, j) && in_row(i, j, 1, 70)) to[j] = from_float<T>(h[i][j]);
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
    grid_launch_dependents();
    grid_dependency_wait();
    __shared__ float slots[64];
    const size_t base = (size_t)blockIdx.x * (size_t)p.K;
    const T *x = static_cast<const T *>(p.x) + base;
    const T *res = p.residual ? static_cast<const T *>(p.residual) + base : nullptr;
    const T *weight = static_cast<const T *>(p.weight);
    auto inside = [&](int c) { return bounds_ok(base + c < (size_t)p.M * p.K && c < p.K, p.status, 71); };   // checked build: site 71
    auto h_at = [&](int c) { return inside(c) ? to_float<T>(x[c]) + (res ? to_float<T>(res[c]) : 0.0f) : 0.0f; };
    float rstd = 1.0f;
    if (NORM) {
        float ss = 0.0f;
        for (int c = threadIdx.x; c < p.K; c += blockDim.x) ss = fmaf(h_at(c), h_at(c), ss);
        ss = row_reduce<false>(ss, slots);
        rstd = __frsqrt_rn(ss / (float)p.K + p.eps);
        if (p.rstd && threadIdx.x == 0) p.rstd[blockIdx.x] = rstd;
    }
    auto y_at = [&](float h, int c) { return NORM ? h * rstd * (weight ? to_float<T>(weight[c]) : 1.0f) : h; };
    float inv = 1.0f, scale = 1.0f;
    if (OUT8) {
        float amax = 0.0f;
        for (int c = threadIdx.x; c < p.K; c += blockDim.x) amax = fmaxf(amax, fabsf(y_at(h_at(c), c)));
        amax = row_reduce<true>(amax, slots + 32);
        scale = e4m3_scale(amax);
        inv = 1.0f / scale;
        if (threadIdx.x == 0) p.scale[blockIdx.x] = scale;
    }
    for (int c = threadIdx.x; c < p.K; c += blockDim.x) {
        const float h = h_at(c), y = y_at(h, c);
        if (!inside(c)) continue;
        if (NORM && p.sum) static_cast<T *>(p.sum)[base + c] = from_float<T>(h);
        if (OUT8) static_cast<uint8_t *>(p.out)[base + c] = (uint8_t)pack_e4m3(e4m3_quotient(y, scale, inv), 0.0f);
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
    int stages, row_bytes, bar_off;
    int *status;
};

// The rows come as bulk copies into a ring of `stages` rows of dout, h and dsum, some rows ahead: what is under way does not depend
// on the registers of the threads that wait for a row's reduction.  KEEP: a thread keeps its part of a row between the row's two passes,
// and the row's slot is free at once; for the longest rows it reads the slot again.  us without dw, rows through registers one ahead / so /
// HBM alone: 8192 x 4096 of bf16 54.3 / 42.5 / 41.0, 2048 x 11008 75 / 36 / 27.5.
template <typename T, int VEC, int NV, int THREADS, bool KEEP>
__global__ void __launch_bounds__(THREADS)
esmm_rmsnorm_backward_kernel(const NormGradParams p)
{
    extern __shared__ __align__(16) char smem[];   // per group: [stage][dout, h, dsum][row_bytes]; from bar_off one barrier per group and stage
    __shared__ float slots[64];
    __shared__ int abort_word;
    volatile int *abort_flag = &abort_word;
    typedef typename Raw<T, VEC>::type raw_t;
    // blockDim.y groups of blockDim.x threads have a row each (several only where a group is one warp)
    const int groups = blockDim.y, group = threadIdx.y;
    const char *ring = smem + (size_t)group * p.stages * 3 * p.row_bytes;
    const uint32_t ring0 = smem_u32(ring), bars = smem_u32(smem) + (uint32_t)(p.bar_off + group * p.stages * 8);
    const T *weight = static_cast<const T *>(p.weight);
    if (threadIdx.x == 0) {
        for (int i = 0; i < p.stages; ++i) mbar_init(bars + 8 * i, 1);
        abort_word = 0;
        fence_barrier_init();
        fence_proxy_async();
    }
    __syncthreads();
    grid_launch_dependents();
    grid_dependency_wait();
    const bool adds = p.dsum != nullptr;
    const uint32_t bytes = (uint32_t)p.row_bytes;
    auto fetch = [&](size_t row, int slot) {
        const size_t from = row * bytes;
        const uint32_t to = ring0 + (uint32_t)slot * 3u * bytes, bar = bars + 8 * slot;
        mbar_arrive_expect_tx(bar, bytes * (adds ? 3u : 2u));
        bulk_load(to, static_cast<const char *>(p.dout) + from, bytes, bar);
        bulk_load(to + bytes, static_cast<const char *>(p.h) + from, bytes, bar);
        if (adds) bulk_load(to + 2u * bytes, static_cast<const char *>(p.dsum) + from, bytes, bar);
    };
    const size_t first = (size_t)blockIdx.x * groups + group, stride = (size_t)gridDim.x * groups;
    if (threadIdx.x == 0)
        for (int i = 0; i < p.stages; ++i)
            if (first + i * stride < (size_t)p.M) fetch(first + i * stride, i);
    float dw[NV][VEC];
    raw_t w[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (threadIdx.x + i * blockDim.x) * VEC;
#pragma unroll
        for (int j = 0; j < VEC; ++j) dw[i][j] = 0.0f;
        if (weight && c < p.K) w[i] = load_raw<T, VEC>(weight + c);
    }
    bool ok = true;
    int slot = 0, turn = 0;
    uint32_t phase = 0;
    float rstd = first < (size_t)p.M ? p.rstd[first] : 0.0f;
    for (size_t row = first; row < (size_t)p.M; row += stride, turn ^= 32) {
        const size_t base = row * (size_t)p.K, next = row + stride;
        const float rstd_next = next < (size_t)p.M ? p.rstd[next] : 0.0f;
        const char *g_at = ring + (size_t)slot * 3 * p.row_bytes;
        const char *h_at = g_at + p.row_bytes, *s_at = h_at + p.row_bytes;
        ok = mbar_wait(bars + 8 * slot, phase, abort_flag) && ok;
        auto element = [&](const char *at, int c) { return *reinterpret_cast<const raw_t *>(at + (size_t)c * sizeof(T)); };
        raw_t s_raw[KEEP ? NV : 1];
        float gw[KEEP ? NV : 1][VEC], xh[KEEP ? NV : 1][VEC], dot[2] = {0.0f, 0.0f};
        auto products = [&](int i, int c, float (&gwi)[VEC], float (&xhi)[VEC], bool sums) {
            float f[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) f[j] = 1.0f;
            unpack<T, VEC>(element(g_at, c), gwi);
            unpack<T, VEC>(element(h_at, c), xhi);
            if (weight) unpack<T, VEC>(w[i], f);
#pragma unroll
            for (int j = 0; j < VEC; j += 2) {
                const float2 g2 = make_float2(gwi[j], gwi[j + 1]), x2 = __fmul2_rn(make_float2(xhi[j], xhi[j + 1]), make_float2(rstd, rstd));
                const float2 p2 = __fmul2_rn(g2, make_float2(f[j], f[j + 1]));
                if (sums) {
                    const float2 d2 = __ffma2_rn(g2, x2, make_float2(dw[i][j], dw[i][j + 1])), s2 = __ffma2_rn(p2, x2, make_float2(dot[0], dot[1]));
                    dw[i][j] = d2.x, dw[i][j + 1] = d2.y;
                    dot[0] = s2.x, dot[1] = s2.y;
                }
                xhi[j] = x2.x, xhi[j + 1] = x2.y;
                gwi[j] = p2.x, gwi[j + 1] = p2.y;
            }
        };
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (threadIdx.x + i * blockDim.x) * VEC;
            if (c < p.K) {
                if (KEEP && adds) s_raw[KEEP ? i : 0] = element(s_at, c);
                products(i, c, gw[KEEP ? i : 0], xh[KEEP ? i : 0], true);
            }
        }
        const float mean = row_reduce<false>(dot[0] + dot[1], slots + turn) / (float)p.K;
        // every thread has the row in its registers (or, !KEEP, is through with the row before it): that slot takes the next row
        if (blockDim.x == 32) __syncwarp();
        if (threadIdx.x == 0) {
            const size_t ahead = row + (KEEP ? p.stages : p.stages - 1) * stride;
            if (ahead < (size_t)p.M && (KEEP || row != first)) fetch(ahead, KEEP ? slot : slot ? slot - 1 : p.stages - 1);
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (threadIdx.x + i * blockDim.x) * VEC;
            if (c < p.K && ok && bounds_ok(base + c + VEC <= (size_t)p.M * p.K, p.status, 62)) {
                float add[VEC];
#pragma unroll
                for (int j = 0; j < VEC; ++j) add[j] = 0.0f;
                const int at = KEEP ? i : 0;
                if constexpr (KEEP) {
                    if (adds) unpack<T, VEC>(s_raw[at], add);
                } else {
                    if (adds) unpack<T, VEC>(element(s_at, c), add);
                    products(i, c, gw[0], xh[0], false);
                }
#pragma unroll
                for (int j = 0; j < VEC; j += 2) {
                    const float2 g2 = __ffma2_rn(make_float2(-mean, -mean), make_float2(xh[at][j], xh[at][j + 1]), make_float2(gw[at][j], gw[at][j + 1]));
                    const float2 o2 = __ffma2_rn(make_float2(rstd, rstd), g2, make_float2(add[j], add[j + 1]));
                    gw[at][j] = o2.x, gw[at][j + 1] = o2.y;
                }
                store_raw<T, VEC>(static_cast<T *>(p.dx) + base + c, gw[at]);
            }
        }
        rstd = rstd_next;
        if (++slot == p.stages) {
            slot = 0;
            phase ^= 1;
        }
    }
    if (!ok) {
        settle_after_timeout();
        if ((threadIdx.x & 31) == 0) atomicExch(p.status, (int)ESMM_ERR_TIMEOUT);
    }
    if (!p.partial || !bounds_ok((int)blockIdx.x < min(p.M, ROWS_MAX_PARTIALS), p.status, 72)) return;   // checked build: site 72
    float *to = p.partial + (size_t)blockIdx.x * p.K;
    float *mine = groups == 1 ? to : reinterpret_cast<float *>(smem) + (size_t)group * (blockDim.x * NV * VEC);
    if (groups > 1) __syncthreads();               // (every group's rows are through: the rings' memory is free)
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (threadIdx.x + i * blockDim.x) * VEC;
        if (c < p.K) {
#pragma unroll
            for (int j = 0; j < VEC; j += 4) *reinterpret_cast<float4 *>(mine + c + j) = make_float4(dw[i][j], dw[i][j + 1], dw[i][j + 2], dw[i][j + 3]);
        }
    }
    if (groups > 1) {
        __syncthreads();
        const float *all = reinterpret_cast<const float *>(smem);
        for (int c = threadIdx.y * blockDim.x + threadIdx.x; c < p.K; c += blockDim.x * groups) {
            float sum = 0.0f;
            for (int g = 0; g < groups; ++g) sum += all[(size_t)g * (blockDim.x * NV * VEC) + c];
            to[c] = sum;
        }
    }
}

// Rows that are no whole vectors, or buffers that do not start on 16 bytes: element by element through registers, one row ahead.  (Through
// the ring 1003 x 1509 of fp32 took 12.7 us instead of 9, 8192 x 1021 of bf16 39 instead of 30.)
template <typename T, int NV>
__global__ void __launch_bounds__(512)
esmm_rmsnorm_backward_ragged_kernel(const NormGradParams p)
{
    grid_launch_dependents();
    grid_dependency_wait();
    __shared__ float slots[64];
    const T *weight = static_cast<const T *>(p.weight);
    const T *dout = static_cast<const T *>(p.dout), *h = static_cast<const T *>(p.h), *dsum = static_cast<const T *>(p.dsum);
    float dw[NV];
    T w[NV], g_raw[NV], h_raw[NV], s_raw[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = threadIdx.x + i * blockDim.x;
        dw[i] = 0.0f;
        w[i] = weight && c < p.K ? weight[c] : from_float<T>(1.0f);
    }
    float rstd_next = 0.0f;
    auto load_row = [&](size_t row) {
        const size_t base = row * (size_t)p.K;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = threadIdx.x + i * blockDim.x;
            if (c < p.K && bounds_ok(base + c < (size_t)p.M * p.K, p.status, 73)) {   // checked build: site 73
                g_raw[i] = dout[base + c];
                h_raw[i] = h[base + c];
                if (dsum) s_raw[i] = dsum[base + c];
            }
        }
        rstd_next = p.rstd[row];
    };
    load_row(blockIdx.x);
    int turn = 0;
    for (size_t row = blockIdx.x; row < (size_t)p.M; row += gridDim.x, turn ^= 32) {
        const size_t base = row * (size_t)p.K;
        const float rstd = rstd_next;
        float gw[NV], xh[NV], add[NV], dot = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            gw[i] = xh[i] = add[i] = 0.0f;
            if (threadIdx.x + i * blockDim.x < (unsigned)p.K) {
                const float g = to_float<T>(g_raw[i]);
                xh[i] = to_float<T>(h_raw[i]) * rstd;
                if (dsum) add[i] = to_float<T>(s_raw[i]);
                dw[i] = fmaf(g, xh[i], dw[i]);
                gw[i] = g * to_float<T>(w[i]);
                dot = fmaf(gw[i], xh[i], dot);
            }
        }
        if (row + gridDim.x < (size_t)p.M) load_row(row + gridDim.x);
        // (two sets of slots in turn: a warp may be a row ahead of the slowest one's reads)
        const float mean = row_reduce<false>(dot, slots + turn) / (float)p.K;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = threadIdx.x + i * blockDim.x;
            if (c < p.K && bounds_ok(base + c < (size_t)p.M * p.K, p.status, 62))
                static_cast<T *>(p.dx)[base + c] = from_float<T>(fmaf(rstd, fmaf(-mean, xh[i], gw[i]), add[i]));
        }
    }
    if (p.partial) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = threadIdx.x + i * blockDim.x;
            if (c < p.K && bounds_ok((int)blockIdx.x < min(p.M, ROWS_MAX_PARTIALS), p.status, 72)) p.partial[(size_t)blockIdx.x * p.K + c] = dw[i];
        }
    }
}

// Rows longer than a CTA's registers: read twice, the sums of dw in the CTA's row of the workspace.
template <typename T>
__global__ void __launch_bounds__(1024)
esmm_rmsnorm_backward_long_kernel(const NormGradParams p)
{
    grid_launch_dependents();
    grid_dependency_wait();
    __shared__ float slots[64];
    const T *weight = static_cast<const T *>(p.weight);
    float *to = p.partial && bounds_ok((int)blockIdx.x < min(p.M, ROWS_MAX_PARTIALS), p.status, 72) ? p.partial + (size_t)blockIdx.x * p.K : nullptr;
    auto inside = [&](size_t base, int c) { return bounds_ok(base + c < (size_t)p.M * p.K && c < p.K, p.status, 71); };
    int turn = 0;
    for (size_t row = blockIdx.x; row < (size_t)p.M; row += gridDim.x, turn ^= 32) {
        const size_t base = row * (size_t)p.K;
        const T *dout = static_cast<const T *>(p.dout) + base, *h = static_cast<const T *>(p.h) + base;
        const T *dsum = p.dsum ? static_cast<const T *>(p.dsum) + base : nullptr;
        const float rstd = p.rstd[row];
        float dot = 0.0f;
        for (int c = threadIdx.x; c < p.K && inside(base, c); c += blockDim.x)
            dot = fmaf(to_float<T>(dout[c]) * (weight ? to_float<T>(weight[c]) : 1.0f), to_float<T>(h[c]) * rstd, dot);
        dot = row_reduce<false>(dot, slots + turn) / (float)p.K;
        for (int c = threadIdx.x; c < p.K && inside(base, c); c += blockDim.x) {
            const float g = to_float<T>(dout[c]), xh = to_float<T>(h[c]) * rstd;
            if (to) to[c] = row == blockIdx.x ? g * xh : fmaf(g, xh, to[c]);
            const float gw = g * (weight ? to_float<T>(weight[c]) : 1.0f);
            static_cast<T *>(p.dx)[base + c] = from_float<T>(fmaf(rstd, fmaf(-xh, dot, gw), dsum ? to_float<T>(dsum[c]) : 0.0f));
        }
    }
}

// out[c] = sum over `rows` rows of partial[r][c], in a fixed order: 32 columns per CTA, four per thread, thread row y takes rows y, y + 64,
// ..., the 64 sums are added as a tree.
template <typename T>
__global__ void __launch_bounds__(512)
esmm_column_sum_kernel(const float *partial, int rows, int K, T *out, int *status)
{
    grid_launch_dependents();
    grid_dependency_wait();
    __shared__ float sums[64][33];
    const int c = blockIdx.x * 32 + threadIdx.x * 4;
    const bool vectors = K % 4 == 0;
    float4 s[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) s[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    auto take = [&](float4 &sum, int r) {
        const float *at = partial + (size_t)r * K + c;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        if (!bounds_ok(r < min(rows, ROWS_MAX_PARTIALS), status, 74)) return;   // checked build: site 74
        if (vectors) {
            if (c < K) v = *reinterpret_cast<const float4 *>(at);
        } else {
            if (c < K) v.x = at[0];
            if (c + 1 < K) v.y = at[1];
            if (c + 2 < K) v.z = at[2];
            if (c + 3 < K) v.w = at[3];
        }
        sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
    };
    int r = threadIdx.y;
    for (; r + 192 < rows; r += 256) {
#pragma unroll
        for (int i = 0; i < 4; ++i) take(s[i], r + 64 * i);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (r + 64 * i < rows) take(s[i], r + 64 * i);
    float *mine = &sums[threadIdx.y][threadIdx.x * 4];
    mine[0] = (s[0].x + s[1].x) + (s[2].x + s[3].x);
    mine[1] = (s[0].y + s[1].y) + (s[2].y + s[3].y);
    mine[2] = (s[0].z + s[1].z) + (s[2].z + s[3].z);
    mine[3] = (s[0].w + s[1].w) + (s[2].w + s[3].w);
    __syncthreads();
    const int warp = (threadIdx.y * 8 + threadIdx.x) >> 5, lane = (threadIdx.y * 8 + threadIdx.x) & 31;
#pragma unroll
    for (int i = 0; i < 2; ++i) {                 // a warp adds up two of the 32 columns
        const int col = warp * 2 + i;
        const float v = warp_sum(sums[lane][col] + sums[lane + 32][col]);
        if (lane == 0 && blockIdx.x * 32 + col < K && bounds_ok((size_t)blockIdx.x * 32 + col < (size_t)K, status, 74)) out[blockIdx.x * 32 + col] = from_float<T>(v);
    }
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
    grid_launch_dependents();
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
                if (r + 8 * u < r1 && bounds_ok((size_t)(r + 8 * u) * p.N + col + VEC <= (size_t)p.M * p.N, p.status, 63)) {
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
            if (to < p.N && bounds_ok((int)blockIdx.y < min((p.M + 7) / 8, ROWS_MAX_PARTIALS), p.status, 72)) p.partial[(size_t)blockIdx.y * p.N + to] = s;
        }
    }
}

// ---- a weight matrix in e4m3, transposed ------------------------------------------------------------------------------------
// scale[n] = amax_k |B[k][n]| / 448: 32 columns per CTA, 32 rows at a time.
template <typename T>
__global__ void __launch_bounds__(1024)
esmm_column_scale_kernel(const T *B, int K, int N, float *scale, int *status)
{
    grid_launch_dependents();
    grid_dependency_wait();
    __shared__ float part[32][33];
    const int n = blockIdx.x * 32 + threadIdx.x;
    float amax = 0.0f;
    if (n < N)
        for (int k = threadIdx.y; k < K && bounds_ok((size_t)k * N + n < (size_t)K * N, status, 75); k += 32) amax = fmaxf(amax, fabsf(to_float<T>(B[(size_t)k * N + n])));
    part[threadIdx.y][threadIdx.x] = amax;
    __syncthreads();
    amax = warp_max(part[threadIdx.x][threadIdx.y]);
    const int to = blockIdx.x * 32 + threadIdx.y;
    if (threadIdx.x == 0 && to < N && bounds_ok(to >= 0, status, 75)) scale[to] = e4m3_scale(amax);   // checked build: site 75
}

// bt[n][k] = e4m3(B[k][n] / scale[n]): tiles of 128 k x 32 n through shared memory, four codes of a row per store
template <typename T>
__global__ void __launch_bounds__(256)
esmm_quantize_transpose_kernel(const T *B, int K, int N, const float *scale, uint8_t *bt, int *status)
{
    grid_launch_dependents();
    grid_dependency_wait();
    __shared__ float tile[128][33];
    const int k0 = blockIdx.y * 128, n0 = blockIdx.x * 32;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const float sc = n0 + lane < N ? scale[n0 + lane] : 1.0f, inv = 1.0f / sc;
    for (int r = warp; r < 128; r += 8)
        tile[r][lane] = k0 + r < K && n0 + lane < N && bounds_ok((size_t)(k0 + r) * N + n0 + lane < (size_t)K * N, status, 76) ? e4m3_quotient(to_float<T>(B[(size_t)(k0 + r) * N + n0 + lane]), sc, inv) : 0.0f;
    __syncthreads();
    for (int c = warp; c < 32; c += 8) {
        const int n = n0 + c, k = k0 + lane * 4;
        if (n < N && k < K && bounds_ok((size_t)n * K + k + 4 <= (size_t)N * K, status, 76))   // (K is a multiple of 16; checked build: site 76)
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

// With more 16-byte vectors than this per SM, rows are taken with up to four vectors per thread: fewer threads per row, so that more rows
// are in flight and a thread has more loads of its own under way.  With fewer, one vector per thread: a row that has its SM nearly to itself is
// through sooner the more warps load it.  One / up to four vectors, us: 16 x 4096 bf16 2.0 / 2.5, 512 x 4096 bf16 3.7 / 4.7, 2048 x 1024 bf16
// 3.9 / 4.6; on the other side 1024 x 4096 bf16 to e4m3 7.4 / 6.7, 512 x 4096 fp32 7.4 / 6.3, 2048 x 11008 bf16 43 / 32.
constexpr int NORM_VECTORS_PER_SM = 2560;

static int sm_count(int *sms)
{
    static std::atomic<int> known[64];
    int dev = 0;
    ESMM_CUDA_TRY(cudaGetDevice(&dev));
    int n = dev >= 0 && dev < 64 ? known[dev].load(std::memory_order_relaxed) : 0;
    if (!n) {
        ESMM_CUDA_TRY(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev));
        if (dev >= 0 && dev < 64) known[dev].store(n, std::memory_order_relaxed);
    }
    *sms = n;
    return ESMM_OK;
}

template <typename T, bool OUT8, bool NORM>
static int norm_launch_type(const NormParams &p, bool aligned, int sms, cudaStream_t stream)
{
    constexpr int VEC = 16 / (int)sizeof(T);
    const bool many = (long)p.M * ceil_div(p.K, VEC) > (long)NORM_VECTORS_PER_SM * sms, vectors = aligned && p.K % VEC == 0;
    // a vector's worth of elements for every `nv`-th thread and its row
    auto go = [&](auto kernel, int units, int nv) -> int {
        const int warps = ceil_div(ceil_div(units, nv), 32);
        const int rows = warps == 1 ? 8 : 1;
        ESMM_CUDA_TRY(launch_dependent(kernel, dim3((unsigned)ceil_div(p.M, rows)), dim3(warps * 32, rows), 0, stream, p));
        return ESMM_OK;
    };
    const int units = vectors ? p.K / VEC : aligned ? p.K / VEC + 2 : p.K;
    const int nv = units <= (many ? 32 : 1024) ? 1 : units <= (many ? 64 : 2048) ? 2 : 4;
    if (vectors && units <= 4096)
        return nv == 1   ? go(esmm_rmsnorm_kernel<T, VEC, 1, OUT8, NORM>, units, 1)
               : nv == 2 ? go(esmm_rmsnorm_kernel<T, VEC, 2, OUT8, NORM>, units, 2)
                         : go(esmm_rmsnorm_kernel<T, VEC, 4, OUT8, NORM>, units, 4);
    if (!vectors && aligned && units <= 2048)
        return units <= (many ? 32 : 1024) ? go(esmm_rmsnorm_ragged_kernel<T, VEC, 1, OUT8, NORM>, units, 1)
                                           : go(esmm_rmsnorm_ragged_kernel<T, VEC, 2, OUT8, NORM>, units, 2);
    // (of 16-bit values four vectors a thread are more than its registers hold; 2139 x 13966 of fp32 to e4m3 143 -> 90 us)
    if constexpr (VEC == 4) {
        if (!vectors && aligned && units <= 4096) return go(esmm_rmsnorm_ragged_kernel<T, VEC, 4, OUT8, NORM>, units, 4);
    }
    if (!aligned && units <= 4096) return go(esmm_rmsnorm_kernel<T, 1, 4, OUT8, NORM>, units, 4);
    ESMM_CUDA_TRY(launch_dependent(esmm_rmsnorm_long_kernel<T, OUT8, NORM>, dim3((unsigned)p.M), dim3(1024), 0, stream, p));
    return ESMM_OK;
}

template <bool NORM>
static int norm_launch(const NormParams &p, int dtype, bool out8, bool aligned, cudaStream_t stream)
{
    int sms = 0;
    const int st = sm_count(&sms);
    if (st != ESMM_OK) return st;
    if (out8) {
        if (dtype == ESMM_F32) return norm_launch_type<float, true, NORM>(p, aligned, sms, stream);
        if (dtype == ESMM_F16) return norm_launch_type<__half, true, NORM>(p, aligned, sms, stream);
        return norm_launch_type<__nv_bfloat16, true, NORM>(p, aligned, sms, stream);
    }
    if constexpr (NORM) {
        if (dtype == ESMM_F32) return norm_launch_type<float, false, true>(p, aligned, sms, stream);
        if (dtype == ESMM_F16) return norm_launch_type<__half, false, true>(p, aligned, sms, stream);
        return norm_launch_type<__nv_bfloat16, false, true>(p, aligned, sms, stream);
    }
    return ESMM_ERR_UNSUPPORTED;
}

template <int N> struct Num { static constexpr int value = N; };

// Rows and columns are counted in int, in steps of up to a CTA's threads.
constexpr int MAX_EXTENT = 0x7FFFFFFF - 65536;

static bool row_dtype(int dtype) { return dtype == ESMM_F32 || dtype == ESMM_F16 || dtype == ESMM_BF16; }

static bool element_aligned(const void *p, int bytes) { return ((uintptr_t)p & (uintptr_t)(bytes - 1)) == 0; }

constexpr int RING_BYTES = 200 * 1024;   // of a backward pass's rows under way, per SM

// Raises a kernel's shared-memory allowance to the device's maximum, once per device.
template <auto KERNEL>
static int allow_ring()
{
    static std::atomic<bool> done[64];
    int dev = 0;
    ESMM_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !done[dev].load(std::memory_order_acquire)) {
        ESMM_CUDA_TRY(cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, RING_BYTES + 1024));
        if (dev >= 0 && dev < 64) done[dev].store(true, std::memory_order_release);
    }
    return ESMM_OK;
}

template <typename T>
static int norm_backward_type(NormGradParams p, bool aligned, int sms, int *ctas, cudaStream_t stream)
{
    constexpr int VEC = 16 / (int)sizeof(T);
    const bool vectors = aligned && p.K % VEC == 0;
    p.row_bytes = p.K <= 2048 * VEC ? p.K * (int)sizeof(T) : 0;
    auto go = [&](auto nv, auto most, auto keep) -> int {
        constexpr int N = decltype(nv)::value;
        constexpr auto kernel = &esmm_rmsnorm_backward_kernel<T, VEC, N, decltype(most)::value, decltype(keep)::value != 0>;
        const int threads = ceil_div(ceil_div(p.K, VEC * N), 32) * 32;
        const int groups = threads == 32 ? std::min(4, p.M) : 1;
        // As many rows under way as the SM's shared memory holds, two per group at least, in one to four CTAs per SM.  More CTAs leave
        // more partial rows of dw to add up; they pay for short rows where each has many (one / two / four CTAs per SM, us: 8192 x 4096
        // bf16 67 / 46 / 52, 8192 x 1024 fp32 60 / 35 / 28, 4096 x 4096 fp32 45 / 48.5 / 48.5).
        int per_sm = threads > 256 ? 1 : threads <= 128 && groups == 1 && p.M >= 32 * sms ? 4 : 2;
        while (per_sm > 1 && RING_BYTES / per_sm < 2 * groups * 3 * p.row_bytes) --per_sm;
        *ctas = std::max(1, std::min(std::min(ceil_div(p.M, groups), ROWS_MAX_PARTIALS), sms * per_sm));
        p.stages = std::max(1, std::min({8, RING_BYTES / per_sm / (groups * 3 * p.row_bytes), ceil_div(p.M, *ctas * groups)}));
        // (the groups' sums of dw are added up where the rings were)
        p.bar_off = std::max(groups * p.stages * 3 * p.row_bytes, groups > 1 ? groups * threads * N * VEC * 4 : 0);
        const size_t smem = (size_t)p.bar_off + groups * p.stages * 8;
        const int st = allow_ring<kernel>();
        if (st != ESMM_OK) return st;
        ESMM_CUDA_TRY(launch_dependent(kernel, dim3((unsigned)*ctas), dim3(threads, groups), smem, stream, p));
        return ESMM_OK;
    };
    if (vectors && p.K <= 2048 * VEC && 2 * 3 * p.row_bytes <= RING_BYTES) {
        if (p.K <= 32 * VEC) return go(Num<1>(), Num<128>(), Num<1>());
        if (p.K <= 64 * VEC) return go(Num<2>(), Num<128>(), Num<1>());
        if (VEC == 8 && p.K <= 128 * VEC) return go(Num<4>(), Num<128>(), Num<1>());
        if (p.K <= 512 * VEC) return go(Num<2>(), Num<256>(), Num<1>());
        if (p.K <= 1024 * VEC) return go(Num<2>(), Num<512>(), Num<1>());
        return go(Num<4>(), Num<512>(), Num<0>());
    }
    auto ragged = [&](auto nv) -> int {
        constexpr int N = decltype(nv)::value;
        auto *kernel = esmm_rmsnorm_backward_ragged_kernel<T, N>;
        const int threads = ceil_div(ceil_div(p.K, N), 32) * 32;
        // (1024 threads of an SM: what a kernel of up to 64 registers has room for; sixteen elements need more, 60 bytes a thread beyond the 128
        // there are, and their 512 threads are alone)
        *ctas = std::max(1, std::min(std::min(p.M, ROWS_MAX_PARTIALS), sms * std::max(1, std::min((N > 8 ? 512 : 1024) / threads, 4))));
        ESMM_CUDA_TRY(launch_dependent(kernel, dim3((unsigned)*ctas), dim3(threads), 0, stream, p));
        return ESMM_OK;
    };
    // us with 1024 threads of at most 64 registers / so: 1000 x 4001 bf16 28.3 / 18.3, 1090 x 6091 bf16 49.7 / 48.5, 3231 x 5029 fp32
    // 134 / 98; eight elements a thread for short rows too: 1003 x 1509 fp32 12.8 instead of 10.0.
    if (!vectors && p.K <= 512 * 4) return ragged(Num<4>());
    if (!vectors && p.K <= 512 * 8) return ragged(Num<8>());
    if (!vectors && p.K <= 512 * 16) return ragged(Num<16>());
    *ctas = std::max(1, std::min(std::min(p.M, ROWS_MAX_PARTIALS), 2 * sms));
    ESMM_CUDA_TRY(launch_dependent(esmm_rmsnorm_backward_long_kernel<T>, dim3((unsigned)*ctas), dim3(1024), 0, stream, p));
    return ESMM_OK;
}

static int column_sum(const float *partial, int rows, int K, int dtype, void *out, int *status, cudaStream_t stream)
{
    auto go = [&](auto tag) -> int {
        typedef decltype(tag) T;
        ESMM_CUDA_TRY(launch_dependent(esmm_column_sum_kernel<T>, dim3((unsigned)ceil_div(K, 32)), dim3(8, 64), 0, stream, partial, rows, K,
                                       static_cast<T *>(out), status));
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
    if (M > MAX_EXTENT || K > MAX_EXTENT) return ESMM_ERR_TOO_LARGE;
    if (!row_dtype(dtype) || (!out8 && out_dtype != dtype)) return ESMM_ERR_UNSUPPORTED;
    const int size = dtype_bytes(dtype);
    for (const void *q : {d_x, d_residual, d_weight, (const void *)d_sum, (const void *)(out8 ? nullptr : d_out)})
        if (!element_aligned(q, size)) return ESMM_ERR_ALIGN;
    if ((out8 && !element_aligned(d_scale, 4)) || !element_aligned(d_rstd, 4)) return ESMM_ERR_ALIGN;
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
    return norm_launch<true>(p, dtype, out8, aligned16({d_x, d_residual, d_weight, d_sum, d_out}), (cudaStream_t)stream);
}

int esmm_quantize_rows(int M, int K, int dtype, const void *d_x, void *d_out, float *d_scale, void *stream)
{
    using namespace esmm;
    if (!d_x || !d_out || !d_scale) return ESMM_ERR_NULL;
    if (M <= 0 || K <= 0) return ESMM_ERR_SHAPE;
    if (M > MAX_EXTENT || K > MAX_EXTENT) return ESMM_ERR_TOO_LARGE;
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
    return norm_launch<false>(p, dtype, true, aligned16({d_x, d_out}), (cudaStream_t)stream);
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
    if (M > MAX_EXTENT || K > MAX_EXTENT) return ESMM_ERR_TOO_LARGE;
    if (!row_dtype(dtype)) return ESMM_ERR_UNSUPPORTED;
    const int size = dtype_bytes(dtype);
    for (const void *q : {d_dout, d_h, d_weight, d_dsum, (const void *)d_dx, (const void *)d_dweight})
        if (!element_aligned(q, size)) return ESMM_ERR_ALIGN;
    if (!element_aligned(d_rstd, 4) || (d_dweight && ((uintptr_t)d_workspace & 15))) return ESMM_ERR_ALIGN;
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
    const bool aligned = aligned16({d_dout, d_h, d_weight, d_dsum, d_dx});
    if (dtype == ESMM_F32) st = norm_backward_type<float>(p, aligned, sms, &ctas, stream);
    else if (dtype == ESMM_F16) st = norm_backward_type<__half>(p, aligned, sms, &ctas, stream);
    else st = norm_backward_type<__nv_bfloat16>(p, aligned, sms, &ctas, stream);
    if (st != ESMM_OK || !d_dweight) return st;
    return column_sum(p.partial, ctas, K, dtype, d_dweight, p.status, stream);
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
    if (M > MAX_EXTENT || N > MAX_EXTENT) return ESMM_ERR_TOO_LARGE;
    if (!aligned16({d_dC, activation == ESMM_ACT_NONE ? nullptr : d_pre, d_dZ, d_dbias ? d_workspace : nullptr}) || !element_aligned(d_dbias, dtype_bytes(dtype)))
        return ESMM_ERR_ALIGN;
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
    return column_sum(p.partial, runs, N, dtype, d_dbias, p.status, stream);
}

int esmm_quantize_b(int K, int N, int dtype, const void *d_B, void *d_bt, float *d_scale, void *stream_)
{
    using namespace esmm;
    cudaStream_t stream = (cudaStream_t)stream_;
    if (!d_B || !d_bt || !d_scale) return ESMM_ERR_NULL;
    if (K <= 0 || N <= 0 || K % 16) return ESMM_ERR_SHAPE;
    if (!row_dtype(dtype)) return ESMM_ERR_UNSUPPORTED;
    if (!element_aligned(d_B, dtype_bytes(dtype)) || ((uintptr_t)d_bt & 15) || !element_aligned(d_scale, 4)) return ESMM_ERR_ALIGN;
    if (K / 128 >= 65535 || N > MAX_EXTENT) return ESMM_ERR_TOO_LARGE;
    int *status = device_status_ptr();
    if (!status) return ESMM_ERR_CUDA;
    auto go = [&](auto tag) -> int {
        typedef decltype(tag) T;
        const T *B = static_cast<const T *>(d_B);
        ESMM_CUDA_TRY(launch_dependent(esmm_column_scale_kernel<T>, dim3((unsigned)ceil_div(N, 32)), dim3(32, 32), 0, stream, B, K, N, d_scale, status));
        ESMM_CUDA_TRY(launch_dependent(esmm_quantize_transpose_kernel<T>, dim3((unsigned)ceil_div(N, 32), (unsigned)ceil_div(K, 128)), dim3(256),
                                       0, stream, B, K, N, (const float *)d_scale, static_cast<uint8_t *>(d_bt), status));
        return ESMM_OK;
    };
    return dtype == ESMM_F32 ? go(float()) : dtype == ESMM_F16 ? go(__half()) : go(__nv_bfloat16());
}

}  // extern "C"
