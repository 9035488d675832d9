// Dense matrix product with its epilogue on the 5th-generation tensor cores (tcgen05, sm_100a), for 16-bit and 8-bit operands:
//
//   C = act(a_scale_i b_scale_j sum_k op(A)_ik op(B)_kj + bias_j) + residual_ij,   FP32 accumulation in tensor memory, one rounding.
//
// Operands are read as they lie.  A K step is 128 bytes of K (64 16-bit or 128 e4m3 values).  An operand whose K runs along
// memory (A of M x K, B stored transposed as N x K) comes as boxes of 128 bytes x rows with the 128-byte swizzle, the canonical K-major
// layout; one whose other index does (A stored as K x M, B of K x N, 16-bit only) as boxes of 64 values x 64 k, the canonical
// MN-major layout: eight k of 64 values are 1024 bytes, the next 64 values follow a box later.  So neither the forward product nor
// its gradients (dA = dZ B^T, dB = A^T dZ) need a transposed copy of anything.
//
// Two kernels:
//   esmm_linear_pair_kernel           large products.  Persistent, a cluster of two CTAs per 256 x 64 .. 256 tile (cta_group::2 MMAs): each CTA
//       fetches its 128 rows of A and half the columns of B into a ring, one thread of the even CTA issues the MMAs, eight
//       epilogue warps per CTA drain one of two accumulators in tensor memory while the other is filled.  Where tiles of 288 .. 512 columns make
//       one round of what would be a round and a bit, both accumulators belong to one tile (two MMAs a step side by side).
//   esmm_linear_split_kernel<NB, F8>  few rows or few tiles: one CTA per 128 x NB tile and part of K, the parts of a tile being one
//       cluster.  The CTAs add up their accumulators through distributed shared memory in a fixed order, each of them finishing a
//       share of the tile's outputs: no workspace, no atomics, the same bits on every call.  Its cost is the operands' bytes: all
//       SMs stream the weights whatever the number of tokens, and rows of A that do not exist are not fetched.
// What bounds them: large products the tensor pipe at the clock that the power cap leaves (2048 x 4096 x 11008 bf16 118 us = 1.57 PFLOP/s
// in bursts, 146 in a loop of seconds, where cuBLAS's plain product takes 152; 2048 x 11008 x 4096 e4m3 65 us = 2.8 PFLOP/s, 79 in a loop); products of
// few rows HBM and a launch's start and end (16 x 4096 x 11008 bf16 16.8 us for 13.8 us of bytes, 1 x 11008 x 4096 e4m3 10.0 for 6.9); small
// ones that start and end (1024 x 64 x 1536 4.1 us: 0.9 until a dependent launch may read, 1.1 for the first copies, 0.8 epilogue, 0.8 to leave).
// Every wait is bounded, as in the other kernels; tensor memory is freed on every path out.
#include <algorithm>
#include <cstring>
#include <mutex>
#include <type_traits>

#include "esmm_dtypes.cuh"
#include "esmm_gemm_shared.cuh"

namespace esmm {

// What depends on a tile's width
struct LinearTile {
    int nb, width, tiles_n;              // columns of an MMA and of a tile, tiles across
    int b_boxes, b_box_cols, b_box_bytes;   // copies of B per stage (K-major: one), columns and bytes of one
    int stage_bytes;                     // pair kernel: bytes that a CTA copies per stage
    uint32_t b_desc_hi, b_lbo, b_step;   // B's descriptors: high word, leading byte offset in place, from one MMA to the next
    uint32_t idesc;
};

struct LinearParams {
    int M, N, ksteps;                    // K in steps of 128 bytes
    int tiles_m, num_tiles;
    // pair kernel: the first `wide_tiles` tiles cover the columns before `wide_cols` in the first width, the rest the others in the second
    // (joined: a tile is as wide as both together, the accumulators side by side, and there is one tile per pair)
    LinearTile kind[2];
    int joined;
    int wide_tiles, wide_cols;
    int group_m;
    int a_boxes;                         // copies of A per stage
    int a_k_major, b_k_major;
    int k_elems;                         // elements of K per step
    int stages;
    int a_stage_bytes;                   // split kernel: of A's part of a stage
    int slot_bytes;                      // pair kernel: from one ring slot to the next
    int boxes, box_off;                  // pair kernel: staging boxes per epilogue warp, the first one's place
    int column_off;                      // pair kernel: place of the tile's scales and biases by column
    uint32_t a_lbo;                      // leading byte offset of A's descriptors, in place
    uint32_t a_step;                     // from one MMA to the next along K, in 16-byte units
    int bf16;                            // type of C, bias, residual and pre: bfloat16 or float16
    int activation, has_pre, has_residual;
    const float *a_scale, *b_scale;
    const void *bias;
    const void *residual;                // split kernel
    void *pre, *C;                       // split kernel
    // pair kernel, relu with the values before it kept: those nearer to zero than this share of their size are summed again, from A and B as
    // they are stored, with the strides of their two indices
    float border;
    int K;
    const void *A, *B;
    size_t a_row, a_k, b_col, b_k;
    int *status;
};

struct LinearMaps {
    CUtensorMap a, b[2];                 // (b by the tiles' width)
    CUtensorMap c, residual, pre;        // pair kernel: boxes of 64 columns x 32 rows, 128-byte swizzle
};

constexpr int L_KBYTES = 128;            // bytes of K per step
// Warps that issue copies, K steps in turn.  (In order of K overall: a step's slot was last used by a step that every earlier wait of the same
// warp has seen pass, as long as the ring has as many slots as there are such warps.)
constexpr int L_PRODUCERS = 3;
constexpr uint32_t L_DESC_HI = 64u | (1u << 14) | (2u << 29);   // eight rows (or k) of 128 bytes every 1024 bytes, version 1, 128-byte swizzle
constexpr uint32_t L_DESC_HI_64 = 32u | (1u << 14) | (4u << 29);   // eight k of 64 bytes every 512 bytes, 64-byte swizzle

template <bool PAIR, bool F8>
__device__ __forceinline__ void linear_mma(uint32_t tmem_d, uint32_t a_lo, uint32_t b_lo, uint32_t b_hi, uint32_t idesc, uint32_t accumulate)
{
#define ESMM_LINEAR_MMA(GROUP, KIND)                                                                                     \
    asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"                                                         \
                 "mov.b64 da, {%1, %5};\n\tmov.b64 db, {%2, %6};\n\tsetp.ne.b32 p, %4, 0;\n\t"                         \
                 "tcgen05.mma.cta_group::" GROUP ".kind::" KIND " [%0], da, db, %3, p;\n\t}\n" ::"r"(tmem_d),             \
                 "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(accumulate), "r"(L_DESC_HI), "r"(b_hi)                             \
                 : "memory")
    if constexpr (PAIR && F8) ESMM_LINEAR_MMA("2", "f8f6f4");
    else if constexpr (PAIR) ESMM_LINEAR_MMA("2", "f16");
    else if constexpr (F8) ESMM_LINEAR_MMA("1", "f8f6f4");
    else ESMM_LINEAR_MMA("1", "f16");
#undef ESMM_LINEAR_MMA
}

// true in one lane of the warp, the same one every time
__device__ __forceinline__ bool linear_elect()
{
    uint32_t on;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(on));
    return on != 0;
}

// The MMAs of one K step by the elected lane.  The loops around it are run by the whole warp, so that the descriptors are computed in
// uniform registers, where the instruction wants them: from a lane's own branch every MMA took 68 cycles to issue, more
// than an MMA of 64 columns runs.
template <bool PAIR, bool F8>
__device__ __forceinline__ void linear_mma_step(const LinearParams &p, const LinearTile &t, uint32_t d, uint32_t a, uint32_t b, bool more, bool elected)
{
    if (elected) {
        linear_mma<PAIR, F8>(d, a, b, t.b_desc_hi, t.idesc, more ? 1u : 0u);
#pragma unroll
        for (uint32_t j = 1; j < 4; ++j) linear_mma<PAIR, F8>(d, a + j * p.a_step, b + j * t.b_step, t.b_desc_hi, t.idesc, 1u);
    }
    __syncwarp();
}

// arrives on the barrier (at this offset in both CTAs of a pair) once the MMAs issued so far are complete
template <bool PAIR>
__device__ __forceinline__ void linear_commit(uint32_t bar)
{
    if constexpr (PAIR) {
        const uint16_t mask = 3;
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
                     "h"(mask)
                     : "memory");
    } else {
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
    }
}

__device__ __forceinline__ void linear_tmem_ld(uint32_t taddr, float *v)
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
          "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]),
          "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]),
          "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
        : "r"(taddr));
}

// the loads before it have arrived in their registers (z: what they write, so that no use of it is moved ahead)
template <int COUNT>
__device__ __forceinline__ void linear_tmem_wait(float (&z)[COUNT])
{
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < COUNT; ++i) asm volatile("" : "+f"(z[i]));
}

__device__ __forceinline__ void linear_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void linear_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

__device__ __forceinline__ uint32_t linear_cta_rank()
{
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}

__device__ __forceinline__ void linear_cluster_sync()
{
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// The same without ordering memory: for the barriers' set-up (fenced by itself) and the end of the kernel, where no data passes.
__device__ __forceinline__ void linear_cluster_meet()
{
    asm volatile("barrier.cluster.arrive.relaxed.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}

__device__ __forceinline__ uint32_t linear_map_to_cta(uint32_t addr, uint32_t rank)
{
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}

template <bool PAIR>
__device__ __forceinline__ void linear_load(uint32_t dst, const CUtensorMap *map, int x, int y, uint32_t bar)
{
    if constexpr (PAIR)   // the bytes are counted on a barrier that may lie in the pair's other CTA
        asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
                     "l"(map), "r"(x), "r"(y), "r"(bar)
                     : "memory");
    else
        tma_load_2d(dst, map, x, y, bar);
}

__device__ __forceinline__ void linear_prefetch(const CUtensorMap *map, int x, int y)
{
    asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global [%0, {%1, %2}];" ::"l"(map), "r"(x), "r"(y) : "memory");
}

// The copies of one K step: lanes 0 .. a_boxes - 1 fetch A, lanes 4 .. 4 + b_boxes - 1 fetch B.  row_a, row_b: first row of op(A) and
// column of op(B) of this CTA's part of the tile.
template <bool PAIR>
__device__ __forceinline__ void linear_load_step(const LinearParams &p, const LinearTile &t, const LinearMaps &maps, const CUtensorMap *b_map, int lane, int step, int row_a, int row_b,
                                                 uint32_t dst_a, uint32_t dst_b, uint32_t bar)
{
    const bool is_b = lane >= 4;
    const int i = lane & 3;
    if (lane >= 8 || i >= (is_b ? t.b_boxes : p.a_boxes)) return;
    const int k = step * p.k_elems, r = is_b ? row_b + t.b_box_cols * i : row_a + 64 * i;
    const bool k_major = is_b ? p.b_k_major : p.a_k_major;
    linear_load<PAIR>(is_b ? dst_b + (uint32_t)(t.b_box_bytes * i) : dst_a + 8192u * (uint32_t)i, is_b ? b_map : &maps.a, k_major ? k : r, k_major ? r : k, bar);
}

// ----------------------------------------------------------------------------------------------------------------------------
// Pair kernel
// ----------------------------------------------------------------------------------------------------------------------------
constexpr int LP_EPI_WARPS = 8;
constexpr int LP_THREADS = (4 + LP_EPI_WARPS) * 32;
constexpr int LP_BOX = 4096;                      // staging box of an epilogue warp: 32 rows x 64 16-bit columns
constexpr int LP_MAX_STAGES = 8;
constexpr int LP_MAX_NB = 256;
constexpr int LP_A_BYTES = 128 * L_KBYTES;
// shared memory: ring, staging boxes (one or two per epilogue warp) | the tile's scales and biases by column | barriers, flags | lists of elements
constexpr int LP_COLUMN_OFF = 224 * 1024;
constexpr int LP_BAR_OFF = LP_COLUMN_OFF + 2 * LP_MAX_NB * 4;
constexpr int LP_LIST = 12;                       // elements next to relu's border that an epilogue warp notes
constexpr int LP_LIST_OFF = LP_BAR_OFF + (2 * LP_MAX_STAGES + 4 + LP_EPI_WARPS) * 8 + 16;
constexpr int LP_SMEM = LP_LIST_OFF + LP_EPI_WARPS * LP_LIST * 8;
constexpr int LP_TMEM_COLS = 2 * LP_MAX_NB;
constexpr int LP_JOINED_OFF = LP_A_BYTES + LP_MAX_NB / 2 * L_KBYTES;   // joined tiles: place of the second MMA's columns of B in a slot
static_assert(LP_SMEM <= SMEM_LIMIT, "shared memory of a CTA");

// ---- relu's border -----------------------------------------------------------------------------------------------------------------
// relu's slope jumps at zero, so where the values before it are kept for the backward pass the sign of a small one has to be the sum's and not the
// accumulation's.  The tensor cores cut every addition to the accumulator's 24 bits.  Their error next to zero, in units of Z's
// standard deviation: 16-bit operands rms 5.8e-10 K, largest of some 690 elements 1.9e-6, 8.2e-6, 2.3e-5 at K = 784, 4096, 11008 (an FP32 FMA sum of
// cuBLAS: 1.1e-6, 3.7e-6, 6.2e-6); e4m3 rms up to 2.7e-11 K.  So an element below ten times the rms, two of 2^19 at K = 784, is summed again in 64 bits (of 8000
// sums that cancel halfway the largest error was 5.5 times it, and the next line's estimate may be a third too small).
// The standard deviation is taken as (row's norm) (column's norm) / (norm) over a 32 x 64 piece, so that a column of small weights is not all border; a sum
// that is exactly zero counts where it is the only one of its row and of its column in the piece (others are sums of zeros, as of pruned blocks).
// An epilogue warp notes such elements of its pieces, as they lie rounded in its staging box, and the CTA sums them when its tiles are through, all epilogue
// warps with a part of K each.  us with the values kept, silu / relu: 520 x 776 x 1032 fp16 8.7 / 9.9 (13 where an element is found), 2048 x 4096 x 11008 131 / 209
// (some 800 elements, a column of B being 4096 lines of memory); summed by the warp alone within the piece 418, by a kernel of its own 220, and 17.5 for the small one.
constexpr float LB_SHARE = 6e-9f, LB_SHARE_F8 = 3e-10f;
constexpr float LB_WIDEST = 1e-3f;            // (from K = 167 thousand on, where 64-bit sums of all that may be off would take longer than the product)
constexpr int LB_MOST = LP_LIST / 2;          // elements per piece: more are no coincidence, and a bound on the time
constexpr int LB_ROWS = 8;                    // in fewer rows a column's size does not show: the row's is taken alone

template <bool F8, bool BF16> struct LinearOperand { typedef __half type; };
template <> struct LinearOperand<false, true> { typedef __nv_bfloat16 type; };
template <bool BF16> struct LinearOperand<true, BF16> { typedef uint8_t type; };
__device__ __forceinline__ float linear_to_float(uint8_t v) { return e4m3_to_float(v); }
__device__ __forceinline__ float linear_to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float linear_to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

// Sum of op(A)_row,k op(B)_k,col in 64 bits over k = first, first + step, ... of the warp's lanes, in every lane; the order is fixed.  (Loads past K are of the
// last k, so that none waits for a branch: all of a round are under way together.)
template <bool F8, bool BF16>
__device__ __noinline__ double linear_sum64(const LinearParams &p, int row, int col, int first, int step)
{
    typedef typename LinearOperand<F8, BF16>::type operand_t;
    constexpr int U = 16;
    double sum = 0.0, other = 0.0;
    if (bounds_ok(row < p.M && col < p.N, p.status, 66)) {   // checked build: site 66
        const operand_t *a = static_cast<const operand_t *>(p.A) + (size_t)row * p.a_row, *b = static_cast<const operand_t *>(p.B) + (size_t)col * p.b_col;
        for (long k0 = first; k0 < p.K; k0 += (long)step * U) {
            operand_t x[U], y[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const size_t k = (size_t)min(k0 + (long)step * u, (long)p.K - 1);
                x[u] = a[k * p.a_k];
                y[u] = b[k * p.b_k];
            }
#pragma unroll
            for (int u = 0; u < U; u += 2) {
                sum = fma(k0 + (long)step * u < p.K ? (double)linear_to_float(x[u]) : 0.0, (double)linear_to_float(y[u]), sum);
                other = fma(k0 + (long)step * (u + 1) < p.K ? (double)linear_to_float(x[u + 1]) : 0.0, (double)linear_to_float(y[u + 1]), other);
            }
        }
    }
    sum += other;
#pragma unroll
    for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, d);
    return sum;
}

// the value before the activation from its 64-bit sum, over the one that is there
template <bool BF16>
__device__ __forceinline__ void linear_put(const LinearParams &p, int2 at, double sum)
{
    typedef typename std::conditional<BF16, __nv_bfloat16, __half>::type out_t;
    if (!bounds_ok(at.x < p.M && at.y < p.N, p.status, 66)) return;
    if (p.a_scale) sum *= (double)p.a_scale[at.x];
    if (p.b_scale) sum *= (double)p.b_scale[at.y];
    if (p.bias) sum += (double)to_float<out_t>(static_cast<const out_t *>(p.bias)[at.y]);
    static_cast<out_t *>(p.pre)[(size_t)at.x * p.N + at.y] = from_float<out_t>((float)sum);
}

// Notes the elements of a staged piece (a row per lane from row0 on, columns from col0 on) that lie below the border.  cb: the columns' biases; reach: the share of the norm
// of this lane's row of sums.  The warp's whole list is summed first where it has no room for a piece's.  Returns how many the list holds.  (Little code: fetching
// it is what its first call in an SM takes.  With the norms of all rows and columns unrolled 520 x 776 x 1032 took 12.3 us.)
template <bool F8, bool BF16>
__device__ __noinline__ int linear_note_border(const LinearParams &p, const char *box, const float *cb, int row0, int col0, float reach, int2 *list, int noted)
{
    constexpr unsigned all = 0xFFFFFFFFu;
    typedef typename std::conditional<BF16, __nv_bfloat16, __half>::type out_t;
    const int lane = threadIdx.x & 31;
    const char *mine = box + lane * 128;
    const int there = min(64, p.N - col0);
    auto value = [&](int j) { return to_float<out_t>(*reinterpret_cast<const out_t *>(mine + (((j >> 3) ^ (lane & 7)) << 4) + 2 * (j & 7))); };
    unsigned long long hit = 0, zero = 0;
#pragma unroll 1
    for (int x = 0; x < there; x += 8) {
        const uint4 raw = *reinterpret_cast<const uint4 *>(mine + (((x >> 3) ^ (lane & 7)) << 4));
        const uint32_t words[4] = {raw.x, raw.y, raw.z, raw.w};
        unsigned below = 0, none = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 z = BF16 ? unpack_bf16(words[j]) : unpack_f16(words[j]), b = *reinterpret_cast<const float2 *>(cb + x + 2 * j);
            below |= (unsigned)(fabsf(z.x) < reach) << (2 * j) | (unsigned)(fabsf(z.y) < reach) << (2 * j + 1);
            none |= (unsigned)(z.x == b.x) << (2 * j) | (unsigned)(z.y == b.y) << (2 * j + 1);
        }
        hit |= (unsigned long long)below << x;
        zero |= (unsigned long long)(below & none) << x;   // (only there: beside a bias of size one many a sum is lost in the rounding)
    }
    if (zero & (zero - 1)) hit &= ~zero;                         // not the only one of its row
    float whole = reach * reach;
#pragma unroll
    for (int d = 16; d; d >>= 1) whole += __shfl_xor_sync(all, whole, d);
    const float inv = rsqrtf(whole) * p.border, alone = rsqrtf((float)there);
    unsigned long long columns = (unsigned long long)__reduce_or_sync(all, (unsigned)hit) | (unsigned long long)__reduce_or_sync(all, (unsigned)(hit >> 32)) << 32;
    int left = LB_MOST;
    while (columns && left > 0) {
        const int j = __ffsll((long long)columns) - 1;
        columns &= columns - 1;
        const float z = value(j), v = row0 + lane < p.M ? z - cb[j] : 0.0f;
        float down = v * v;
#pragma unroll
        for (int d = 16; d; d >>= 1) down += __shfl_xor_sync(all, down, d);
        const bool single = __popc(__ballot_sync(all, zero >> j & 1)) == 1;
        unsigned rows = __ballot_sync(all, (hit >> j & 1) && (v != 0.0f || single) && fabsf(z) < reach * (p.M - row0 < LB_ROWS ? alone : sqrtf(down) * inv));
        if (rows && noted > LP_LIST - LB_MOST && left == LB_MOST) {
            if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");   // the pieces are in place
            __syncwarp();
            for (int e = 0; e < noted; ++e) {
                const double sum = linear_sum64<F8, BF16>(p, list[e].x, list[e].y, lane, 32);
                if (lane == 0) linear_put<BF16>(p, list[e], sum);
            }
            __syncwarp();
            noted = 0;
        }
        for (; rows && left > 0; rows &= rows - 1, --left, ++noted)
            if (lane == 0 && bounds_ok(noted < LP_LIST, p.status, 66)) list[noted] = make_int2(row0 + __ffs((int)rows) - 1, col0 + j);
    }
    return noted;
}

// By all epilogue warps when the CTA's tiles are through: every warp a part of K of all elements that they have noted, then the parts in their order.  (The ring is
// free then: the copies of these tiles have landed and been read.)
template <bool F8, bool BF16>
__device__ __noinline__ void linear_sum_border(const LinearParams &p, char *smem, int tid, int noted)
{
    constexpr int ENTRIES = LP_EPI_WARPS * LP_LIST;
    const int lane = tid & 31, w = tid >> 5;
    int2 *lists = reinterpret_cast<int2 *>(smem + LP_LIST_OFF);
    double *parts = reinterpret_cast<double *>(smem);
    if (lane < LP_LIST && lane >= noted) lists[w * LP_LIST + lane].x = -1;
    unsigned any;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.s32 q, %1, 0;\n\tbarrier.cta.red.or.pred p, 1, 256, q;\n\tselp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(any) : "r"(noted) : "memory");
    if (!any) return;
#pragma unroll 1
    for (int e0 = 0; e0 < ENTRIES; e0 += 32) {
        unsigned there = __ballot_sync(0xFFFFFFFFu, lists[e0 + lane].x >= 0);
        for (; there; there &= there - 1) {
            const int e = e0 + __ffs((int)there) - 1;
            const double sum = linear_sum64<F8, BF16>(p, lists[e].x, lists[e].y, tid, 32 * LP_EPI_WARPS);
            if (lane == 0) parts[e * LP_EPI_WARPS + w] = sum;
        }
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");   // the pieces are in place
    asm volatile("bar.sync 1, 256;" ::: "memory");
    if (tid < ENTRIES && lists[tid].x >= 0) {
        double sum = 0.0;
        for (int i = 0; i < LP_EPI_WARPS; ++i) sum += parts[tid * LP_EPI_WARPS + i];
        linear_put<BF16>(p, lists[tid], sum);
    }
}
static_assert(LP_EPI_WARPS * LP_LIST % 32 == 0, "lists are looked through 32 elements at a time");

// Tile `item` of the launch: its width, tile row and first column.
__device__ __forceinline__ const LinearTile &linear_tile(const LinearParams &p, int item, int &second, int &tm, int &col)
{
    second = item >= p.wide_tiles;
    const LinearTile &t = p.kind[second];
    int tn;
    tile_coords(second ? item - p.wide_tiles : item, p.tiles_m, t.tiles_n, tm, tn, p.group_m);
    col = (second ? p.wide_cols : 0) + tn * t.width;
    return t;
}

// BORDER: with relu's border, apart from the others because its code in the epilogue costs them registers (2048 x 2048 x 4096 of bf16 27.6 us instead of 29.2).
template <bool F8, bool BF16, bool BORDER>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(LP_THREADS, 1)
esmm_linear_pair_kernel(const __grid_constant__ LinearMaps maps, const __grid_constant__ LinearParams p)
{
    extern __shared__ __align__(1024) char smem[];
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + LP_BAR_OFF);
    const uint32_t full0 = smem_u32(bars), empty0 = smem_u32(bars + LP_MAX_STAGES), accf0 = smem_u32(bars + 2 * LP_MAX_STAGES),
                   acce0 = smem_u32(bars + 2 * LP_MAX_STAGES + 2), res0 = smem_u32(bars + 2 * LP_MAX_STAGES + 4);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(bars + 2 * LP_MAX_STAGES + 4 + LP_EPI_WARPS);
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(const_cast<int *>(abort_flag + 1));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = linear_cta_rank();
    const bool leader = rank == 0;
    const int pair = blockIdx.x >> 1, num_pairs = gridDim.x >> 1;

    if (warp == 0) {                                           // a barrier per lane
        if (lane < p.stages) {
            mbar_init(full0 + 8 * lane, 1);                    // (even CTA) its producers; bytes of both CTAs' copies
            mbar_init(empty0 + 8 * lane, 1);                   // one commit per stage, delivered to both CTAs
        } else if (lane >= 16 && lane < 16 + LP_EPI_WARPS) {
            mbar_init(res0 + 8 * (lane - 16), 1);
        } else if (lane >= 24 && lane < 26) {
            mbar_init(accf0 + 8 * (lane - 24), 1);
            mbar_init(acce0 + 8 * (lane - 24), 2 * LP_EPI_WARPS);   // (even CTA) the epilogue warps of both CTAs
        }
        if (lane == 26) *abort_flag = 0;
        fence_barrier_init();
        fence_proxy_async();
    } else if (warp == 1 && lane == 0) {
        tma_prefetch_descriptor(&maps.a);
        tma_prefetch_descriptor(&maps.b[0]);
        tma_prefetch_descriptor(&maps.c);
    }
    if (warp == L_PRODUCERS) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                     "r"(LP_TMEM_COLS));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::);
    }
    linear_fence_before();
    __syncthreads();
    linear_cluster_meet();
    linear_fence_after();
    grid_launch_dependents();
    grid_dependency_wait();
    const uint32_t tmem = *tmem_slot;
    bool ok = true;

    if (warp < L_PRODUCERS) {
        // ---------------- producers: K steps in turn ----------------
        int slot = warp, first = warp;                     // the slot of this warp's next step, and that step's index in the tile
        uint32_t phase = 0;
        for (int tile = pair; tile < p.num_tiles && ok; tile += num_pairs) {
            int second, tm, col;
            const LinearTile &t = linear_tile(p, tile, second, tm, col);
            const int row_a = tm * 256 + (int)rank * 128, row_b = col + (int)rank * (t.nb / 2);
            int step = first;
            for (; step < p.ksteps; step += L_PRODUCERS) {
                ok = mbar_wait(empty0 + 8 * slot, phase ^ 1, abort_flag);
                ok = __all_sync(0xFFFFFFFFu, ok);
                if (!ok) break;
                if (leader && lane == 0) mbar_arrive_expect_tx(full0 + 8 * slot, 2u * (uint32_t)t.stage_bytes);
                __syncwarp();
                const uint32_t dst = smem_u32(smem) + (uint32_t)(slot * p.slot_bytes);
                const uint32_t bar = linear_map_to_cta(full0 + 8 * slot, 0);
                linear_load_step<true>(p, t, maps, &maps.b[second], lane, step, row_a, row_b, dst, dst + LP_A_BYTES, bar);
                if (p.joined && lane >= 8 && lane - 8 < p.kind[1].b_boxes) {
                    const LinearTile &u = p.kind[1];
                    const int i = lane - 8, k = step * p.k_elems, r = col + t.nb + (int)rank * (u.nb / 2) + u.b_box_cols * i;
                    linear_load<true>(dst + (uint32_t)(LP_JOINED_OFF + u.b_box_bytes * i), &maps.b[1], p.b_k_major ? k : r, p.b_k_major ? r : k, bar);
                }
                slot += L_PRODUCERS;
                if (slot >= p.stages) {
                    slot -= p.stages;
                    phase ^= 1;
                }
            }
            first = step - p.ksteps;
        }
    } else if (warp == L_PRODUCERS) {
        // ---------------- MMA issue: one thread of the even CTA, for both CTAs ----------------
        if (leader) {
            const bool elected = linear_elect();
            int slot = 0;
            uint32_t phase = 0, turn = 0;
            bool landed = false;
            const uint32_t ring = (smem_u32(smem) & 0x3FFFFu) >> 4;
            for (int tile = pair; tile < p.num_tiles && ok; tile += num_pairs, ++turn) {
                const uint32_t ab = turn & 1u;
                ok = mbar_wait(acce0 + 8 * ab, ((turn >> 1) & 1u) ^ 1u, abort_flag);   // drained in both CTAs
                ok = __all_sync(0xFFFFFFFFu, ok);
                if (!ok) break;
                linear_fence_after();
                const LinearTile &t = p.kind[tile >= p.wide_tiles];
                const uint32_t d = tmem + ab * (uint32_t)LP_MAX_NB;
                for (int step = 0; step < p.ksteps; ++step) {
                    if (!landed) ok = mbar_wait(full0 + 8 * slot, phase, abort_flag);
                    ok = __all_sync(0xFFFFFFFFu, ok);
                    if (!ok) break;
                    const uint32_t at = ring + (uint32_t)(slot * (p.slot_bytes >> 4));
                    const int nslot = slot + 1 == p.stages ? 0 : slot + 1;
                    // (a wait costs time even where the data is there: ask for the next step's while this one's MMAs are issued)
                    landed = mbar_test_wait(full0 + 8 * nslot, nslot ? phase : phase ^ 1u);
                    linear_mma_step<true, F8>(p, t, d, at | p.a_lbo, (at + (LP_A_BYTES >> 4)) | t.b_lbo, step != 0, elected);
                    if (p.joined)
                        linear_mma_step<true, F8>(p, p.kind[1], d + (uint32_t)LP_MAX_NB, at | p.a_lbo, (at + (LP_JOINED_OFF >> 4)) | p.kind[1].b_lbo,
                                                  step != 0, elected);
                    if (elected) linear_commit<true>(empty0 + 8 * slot);
                    landed = __all_sync(0xFFFFFFFFu, landed);
                    if (++slot == p.stages) {
                        slot = 0;
                        phase ^= 1;
                    }
                }
                if (!ok) break;
                if (elected) linear_commit<true>(accf0 + 8 * ab);
                __syncwarp();
            }
        }
    } else if (warp >= 4) {
        // ---------------- epilogue: a row per thread, 64 columns at a time through the warp's staging boxes ----------------
        const int w = warp - 4, q = w & 3, half = w >> 2;         // TMEM lanes 32 q .., columns 64 (half + 2 c) ..
        const int tid = threadIdx.x - 128;
        char *boxes = smem + p.box_off + w * p.boxes * LP_BOX;
        typedef typename std::conditional<BF16, __nv_bfloat16, __half>::type out_t;
        const int columns = p.joined ? 2 * LP_MAX_NB : LP_MAX_NB;
        float *col_scale = reinterpret_cast<float *>(smem + p.column_off), *col_bias = col_scale + columns;
        const uint32_t res_bar = res0 + 8 * w;
        const bool scaled = F8 || p.a_scale != nullptr || p.b_scale != nullptr;
        auto unpack2 = [](uint32_t v) { return BF16 ? unpack_bf16(v) : unpack_f16(v); };
        auto pack2 = [](float lo, float hi) { return BF16 ? pack_bf16(lo, hi) : pack_f16(lo, hi); };
        // The warp's boxes are taken in turn, whatever tile a piece is of.  With two, the residual of the piece after the current one is fetched as
        // soon as the current one's has been read, into the other box (4096 x 512 x 4096 25.0 -> 23.9 us); with one, when its turn comes.
        const bool ahead = p.boxes == 2;
        int noted = 0;                                            // elements next to relu's border in this warp's list
        uint32_t turn = 0, res_phase = 0;
        int which = 0;                                            // the current piece's box
        // (lane 0) residual of piece c of a tile to a box, if any of it lies inside C
        auto fetch_residual = [&](int tile, int c, int to) {
            int second, tm, col;
            const LinearTile &t = linear_tile(p, tile, second, tm, col);
            col += half * 64 + 128 * c;
            const int row = tm * 256 + (int)rank * 128 + q * 32;
            if (half * 64 + 128 * c + 64 > t.width || row >= p.M || col >= p.N) return;   // (not a narrow piece's, which has no box)
            mbar_arrive_expect_tx(res_bar, (uint32_t)LP_BOX);
            tma_load_2d(smem_u32(boxes) + (uint32_t)(to * LP_BOX), &maps.residual, col, row, res_bar);
        };
        if (lane == 0 && p.has_residual && ahead && pair < p.num_tiles) fetch_residual(pair, 0, 0);
        // (after a wait that ran out these warps go on through all tiles, doing nothing, so that none is missing at their barrier; the waits return
        // at once then)
        for (int tile = pair; tile < p.num_tiles; tile += num_pairs, ++turn) {
            int second, tm, tile_col;
            const LinearTile &t = linear_tile(p, tile, second, tm, tile_col);
            const int chunks = ((t.width + 63) / 64 - half + 1) / 2;   // of the tile's 64-column pieces, every other one: none to four
            const int row0 = tm * 256 + (int)rank * 128 + q * 32, col0 = tile_col + half * 64;
            const uint32_t ab = turn & 1u;
            if (lane == 0 && ok && p.has_residual && !ahead) {    // (one box: the first piece's, under the wait for the accumulator)
                asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                fetch_residual(tile, 0, 0);
            }
            // the tile's scales and biases, a column per epilogue thread, under the wait for the accumulator
            const float sa = p.a_scale && row0 + lane < p.M ? p.a_scale[row0 + lane] : 1.0f;
            float scale[2], bias[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int c = tid + i * LP_MAX_NB;
                scale[i] = 1.0f, bias[i] = 0.0f;
                if (c < t.width && tile_col + c < p.N) {
                    if (p.b_scale) scale[i] = p.b_scale[tile_col + c];
                    if (p.bias) bias[i] = to_float<out_t>(static_cast<const out_t *>(p.bias)[tile_col + c]);
                }
            }
            asm volatile("bar.sync 1, 256;" ::: "memory");        // every epilogue warp is through with the tile before
#pragma unroll
            for (int i = 0; i < 2; ++i)
                if (i * LP_MAX_NB < columns) {
                    col_scale[tid + i * LP_MAX_NB] = scale[i];
                    col_bias[tid + i * LP_MAX_NB] = bias[i];
                }
            asm volatile("bar.sync 1, 256;" ::: "memory");
            ok = __all_sync(0xFFFFFFFFu, mbar_wait(accf0 + 8 * ab, (turn >> 1) & 1u, abort_flag) && ok);
            linear_fence_after();
            // A second pass over a piece for the values before the activation, which take its box once C's have left it.  One copy of the
            // code for all pieces: with short K a tile's epilogue is what counts, and unrolled it takes as long to fetch as to run.
            const int passes = p.has_pre ? 2 : 1, steps = passes * chunks;
#pragma unroll 1
            for (int i = 0; i < steps && ok; ++i) {
                const int c = passes == 2 ? i >> 1 : i;
                const bool pre_pass = passes == 2 && (i & 1);
                const int col = col0 + 128 * c;
                char *box = boxes + which * LP_BOX, *mine = box + lane * 128;
                const bool inside = row0 < p.M && col < p.N;      // (a box wholly outside C is not stored; the rest is clipped)
                const bool narrow = half * 64 + 128 * c + 64 > t.width;   // 32 columns, the last piece of some joined tiles
                const bool adds = p.has_residual && inside && !pre_pass && !narrow;
                float z[64];
                const uint32_t from = tmem + ((uint32_t)(q * 32) << 16) + ab * (uint32_t)LP_MAX_NB + (uint32_t)(half * 64 + 128 * c);
                linear_tmem_ld(from, z);
                linear_tmem_ld(from + 32, z + 32);
                // the box is free: with two, all but the last store, which reads the other one, are over (a residual's box was waited for when it
                // was fetched); with one, and before a second pass over the same box, all of them
                if (lane == 0) {
                    if (!ahead || p.has_pre) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                    else if (!adds) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
                    if (adds && !ahead && i) fetch_residual(tile, c, which);
                }
                linear_tmem_wait(z);
                if (i == steps - 1) {                             // the accumulator is read: the next but one tile may have it
                    linear_fence_before();
                    __syncwarp();
                    if (lane == 0)
                        asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(linear_map_to_cta(acce0 + 8 * ab, 0)) : "memory");
                }
                const float *cs = col_scale + half * 64 + 128 * c, *cb = col_bias + half * 64 + 128 * c;
                if (scaled) {
#pragma unroll
                    for (int j = 0; j < 64; j += 4) {
                        const float4 s4 = *reinterpret_cast<const float4 *>(cs + j);
                        z[j] = z[j] * sa * s4.x;
                        z[j + 1] = z[j + 1] * sa * s4.y;
                        z[j + 2] = z[j + 2] * sa * s4.z;
                        z[j + 3] = z[j + 3] * sa * s4.w;
                    }
                }
                // whether an element of this row may lie below relu's border: none does that is not below the row's norm times the share, a column's norm being at
                // most the piece's
                const bool borders = BORDER && pre_pass;
                float reach = 0.0f;
                if (borders) {
                    float squares[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int j = 0; j < 64; ++j) squares[j & 3] = fmaf(z[j], z[j], squares[j & 3]);
                    reach = p.border * sqrtf((squares[0] + squares[1]) + (squares[2] + squares[3]));
                }
                if (p.bias) {
#pragma unroll
                    for (int j = 0; j < 64; j += 4) {
                        const float4 b4 = *reinterpret_cast<const float4 *>(cb + j);
                        z[j] += b4.x;
                        z[j + 1] += b4.y;
                        z[j + 2] += b4.z;
                        z[j + 3] += b4.w;
                    }
                }
                bool near = false;
                if (borders) {
#pragma unroll
                    for (int j = 0; j < 64; j += 8) {
                        float least = fabsf(z[j]);
#pragma unroll
                        for (int e = 1; e < 8; ++e) least = fminf(least, fabsf(z[j + e]));
                        near = near || (col + j < p.N && least < reach);
                    }
                }
                if (p.activation && !pre_pass)
                    with_activation(p.activation, [&](auto tag) {
#pragma unroll
                        for (int j = 0; j < 64; ++j) z[j] = activate<decltype(tag)::value>(z[j]);
                    });
                if (narrow) {                                     // 64 bytes of each row without a box, whose store would take the next tile's columns along
                    const size_t at = (size_t)(row0 + lane) * p.N + col;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        if (row0 + lane >= p.M || col + 8 * j >= p.N || !bounds_ok(at + 8 * j + 8 <= (size_t)p.M * p.N, p.status, 65)) continue;   // checked build: site 65
                        if (p.has_residual && !pre_pass) {
                            const uint4 r = *reinterpret_cast<const uint4 *>(static_cast<const out_t *>(p.residual) + at + 8 * j);
                            const uint32_t rw[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const float2 f = unpack2(rw[e]);
                                z[8 * j + 2 * e] += f.x;
                                z[8 * j + 2 * e + 1] += f.y;
                            }
                        }
                        *reinterpret_cast<uint4 *>(static_cast<out_t *>(pre_pass ? p.pre : p.C) + at + 8 * j) =
                            make_uint4(pack2(z[8 * j], z[8 * j + 1]), pack2(z[8 * j + 2], z[8 * j + 3]), pack2(z[8 * j + 4], z[8 * j + 5]), pack2(z[8 * j + 6], z[8 * j + 7]));
                    }
                    continue;                                     // (nothing follows it: a joined tile is its pair's only one)
                }
                if (adds) {
                    ok = mbar_wait(res_bar, res_phase, abort_flag);
                    res_phase ^= 1u;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {                 // 16 bytes = 8 columns; chunk x of row r lies at x ^ (r & 7)
                        const uint4 r = *reinterpret_cast<const uint4 *>(mine + ((j ^ (lane & 7)) << 4));
                        const uint32_t rw[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float2 f = unpack2(rw[e]);
                            z[8 * j + 2 * e] += f.x;
                            z[8 * j + 2 * e + 1] += f.y;
                        }
                    }
                }
                __syncwarp();                                     // (lane 0 has waited for the box, and every lane has read its residual)
                if (lane == 0 && ok && p.has_residual && ahead && !pre_pass) {
                    asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                    if (c + 1 < chunks) fetch_residual(tile, c + 1, which ^ 1);
                    else if (tile + num_pairs < p.num_tiles) fetch_residual(tile + num_pairs, 0, which ^ 1);
                }
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    *reinterpret_cast<uint4 *>(mine + ((j ^ (lane & 7)) << 4)) = make_uint4(pack2(z[8 * j], z[8 * j + 1]), pack2(z[8 * j + 2], z[8 * j + 3]),
                                                                                            pack2(z[8 * j + 4], z[8 * j + 5]), pack2(z[8 * j + 6], z[8 * j + 7]));
                fence_proxy_async();
                __syncwarp();
                ok = __all_sync(0xFFFFFFFFu, ok);
                if (lane == 0) {
                    if (inside && ok)
                        asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(pre_pass ? &maps.pre : &maps.c),
                                     "r"(col), "r"(row0), "r"(smem_u32(box))
                                     : "memory");
                    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                }
                if (BORDER && __any_sync(0xFFFFFFFFu, near))
                    noted = linear_note_border<F8, BF16>(p, box, cb, row0, col, reach, reinterpret_cast<int2 *>(smem + LP_LIST_OFF) + w * LP_LIST, noted);
                if (passes == 1 || pre_pass) which ^= p.boxes - 1;
            }
            if (chunks == 0 && lane == 0)                         // (the other four warps do all of a narrow tile)
                asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(linear_map_to_cta(acce0 + 8 * ab, 0)) : "memory");
        }
        if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");   // (what is written is there when the kernel has ended)
        if (BORDER) linear_sum_border<F8, BF16>(p, smem, tid, ok ? noted : 0);
    }

    if (!ok) {
        settle_after_timeout();
        if (lane == 0) atomicExch(p.status, (int)ESMM_ERR_TIMEOUT);
    }
    linear_fence_before();
    __syncthreads();
    linear_cluster_meet();        // nothing of the other CTA is touched after this
    if (warp == L_PRODUCERS) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(LP_TMEM_COLS));
}

// ----------------------------------------------------------------------------------------------------------------------------
// Split kernel
// ----------------------------------------------------------------------------------------------------------------------------
constexpr int LS_DRAIN_WARPS = 8;                 // half the accumulator's columns each; then warps that copy and one that issues the MMAs
constexpr int LS_THREADS = (LS_DRAIN_WARPS + L_PRODUCERS + 1) * 32;
constexpr int LS_MAX_STAGES = 16;
constexpr int LS_MAX_SPLIT = 8;
// At least so much shared memory per CTA, so that no more than four are on an SM: tensor memory has room for the accumulators of four, and
// a CTA that waited for it would hold up the rest of its cluster.
constexpr int LS_MIN_SMEM = 50 * 1024;

// shared memory: ring of A, ring of B (the sums lie over both after the last MMA) | barriers, flags
__host__ __device__ constexpr int ls_red_bytes(int rows, int nb) { return rows * (nb + 4) * 4; }

// The share of CTA `rank` of a tile's outputs, by the draining warps: four columns per thread and row, neighbouring threads on neighbouring
// columns (reads of the other CTAs' sums move 16 bytes per lane without gaps), a few rows at a time so that their loads are under way
// together.  What the epilogue reads beside the sums is fetched before the last MMA: the column's scale and bias, and for the thread's
// first rows the row's scale and the residual.
template <int NB>
struct LinearSplitEpilogue {
    static constexpr int LANES = NB / 4, ROWS = LS_DRAIN_WARPS * 32 / LANES, U = 2;
    float bias[4], sb[4];
    float sa[U];
    uint2 res[U];

    __device__ __forceinline__ static float2 unpack2(const LinearParams &p, uint32_t w) { return p.bf16 ? unpack_bf16(w) : unpack_f16(w); }
    __device__ __forceinline__ static uint32_t pack2(const LinearParams &p, float lo, float hi) { return p.bf16 ? pack_bf16(lo, hi) : pack_f16(lo, hi); }

    // rows r, r + step, ...
    __device__ __forceinline__ void fetch_rows(const LinearParams &p, int row0, int col, int r, int step, int rows)
    {
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int ri = r + i * step;
            sa[i] = 1.0f;
            if (ri < rows) {
                if (p.a_scale) sa[i] = p.a_scale[row0 + ri];
                if (p.has_residual) res[i] = *reinterpret_cast<const uint2 *>(static_cast<const char *>(p.residual) + ((size_t)(row0 + ri) * p.N + col) * 2);
            }
        }
    }

    __device__ __forceinline__ void fetch(const LinearParams &p, int rank, int split, int row0, int col0, int rows)
    {
        const int col = col0 + (threadIdx.x % LANES) * 4;
#pragma unroll
        for (int j = 0; j < 4; ++j) bias[j] = 0.0f, sb[j] = 1.0f;
        if (col >= p.N) return;
        if (p.bias) {
            const uint2 w = *reinterpret_cast<const uint2 *>(static_cast<const char *>(p.bias) + (size_t)col * 2);
            const float2 f0 = unpack2(p, w.x), f1 = unpack2(p, w.y);
            bias[0] = f0.x, bias[1] = f0.y, bias[2] = f1.x, bias[3] = f1.y;
        }
        if (p.b_scale) {   // (aligned to its elements only)
#pragma unroll
            for (int j = 0; j < 4; ++j) sb[j] = p.b_scale[col + j];
        }
        fetch_rows(p, row0, col, rank * ROWS + threadIdx.x / LANES, split * ROWS, rows);
    }

    // sums: this CTA's, at the same place in every CTA of the cluster.  (The loads from them are volatile, as the cluster barrier is, so that
    // none is moved before it.)
    template <int SPLIT>
    __device__ __forceinline__ void finish(const LinearParams &p, uint32_t sums, int rank, int row0, int col0, int rows)
    {
        uint32_t part_base[SPLIT];
#pragma unroll
        for (int part = 0; part < SPLIT; ++part) part_base[part] = SPLIT == 1 ? sums : linear_map_to_cta(sums, (uint32_t)part);
        constexpr int V = SPLIT <= 2 ? U : SPLIT <= 4 ? 2 : 1;      // rows whose sums are loaded together
        const int c = (threadIdx.x % LANES) * 4, col = col0 + c;
        if (col >= p.N) return;
        const int first = rank * ROWS + threadIdx.x / LANES;
        for (int r = first; r < rows; r += SPLIT * ROWS * U) {
            if (r != first) fetch_rows(p, row0, col, r, SPLIT * ROWS, rows);
#pragma unroll
            for (int i0 = 0; i0 < U; i0 += V) {
                float4 u[V][SPLIT];
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const int ri = r + (i0 + i) * SPLIT * ROWS;
                    if (ri >= rows) break;
#pragma unroll
                    for (int part = 0; part < SPLIT; ++part) {
                        const uint32_t at = part_base[part] + (uint32_t)((ri * (NB + 4) + c) * 4);
                        if constexpr (SPLIT == 1)
                            asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(u[i][part].x), "=f"(u[i][part].y), "=f"(u[i][part].z), "=f"(u[i][part].w) : "r"(at));
                        else
                            asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(u[i][part].x), "=f"(u[i][part].y), "=f"(u[i][part].z), "=f"(u[i][part].w) : "r"(at));
                    }
                }
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const int ri = r + (i0 + i) * SPLIT * ROWS;
                    if (ri >= rows) break;
                    const size_t off = (size_t)(row0 + ri) * p.N + col;
                    float z[4] = {u[i][0].x, u[i][0].y, u[i][0].z, u[i][0].w};
#pragma unroll
                    for (int part = 1; part < SPLIT; ++part) z[0] += u[i][part].x, z[1] += u[i][part].y, z[2] += u[i][part].z, z[3] += u[i][part].w;
#pragma unroll
                    for (int j = 0; j < 4; ++j) z[j] = fmaf(z[j] * sa[i0 + i], sb[j], bias[j]);
                    const bool inside = bounds_ok(off + 4 <= (size_t)p.M * p.N, p.status, 64);   // checked build: site 64
                    if (p.has_pre && inside) *reinterpret_cast<uint2 *>(static_cast<char *>(p.pre) + off * 2) = make_uint2(pack2(p, z[0], z[1]), pack2(p, z[2], z[3]));
                    with_activation(p.activation, [&](auto tag) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) z[j] = activate<decltype(tag)::value>(z[j]);
                    });
                    if (p.has_residual) {
                        const float2 f0 = unpack2(p, res[i0 + i].x), f1 = unpack2(p, res[i0 + i].y);
                        z[0] += f0.x, z[1] += f0.y, z[2] += f1.x, z[3] += f1.y;
                    }
                    if (inside) *reinterpret_cast<uint2 *>(static_cast<char *>(p.C) + off * 2) = make_uint2(pack2(p, z[0], z[1]), pack2(p, z[2], z[3]));
                }
            }
        }
    }
};

template <int NB, bool F8>
__global__ void __launch_bounds__(LS_THREADS, 2)
esmm_linear_split_kernel(const __grid_constant__ LinearMaps maps, const __grid_constant__ LinearParams p, const int split, const int bar_off)
{
    extern __shared__ __align__(1024) char smem[];
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + bar_off);
    const uint32_t full0 = smem_u32(bars), empty0 = smem_u32(bars + LS_MAX_STAGES), accf = smem_u32(bars + 2 * LS_MAX_STAGES);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(bars + 2 * LS_MAX_STAGES + 1);
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(const_cast<int *>(abort_flag + 1));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)linear_cta_rank();
    const int tile = blockIdx.x / split;
    int tm, tn;
    const LinearTile &t = p.kind[0];
    tile_coords(tile, p.tiles_m, t.tiles_n, tm, tn, p.group_m);
    const int s0 = (int)((long)p.ksteps * rank / split), s1 = (int)((long)p.ksteps * (rank + 1) / split);   // this CTA's K steps, one at least
    const int row0 = tm * 128, col0 = tn * NB, rows = min(128, p.M - row0);
    constexpr int B_BYTES = NB * L_KBYTES;
    const uint32_t a_ring = smem_u32(smem), b_ring = a_ring + (uint32_t)(p.stages * p.a_stage_bytes);

    // The first K steps of B are brought into L2 while the barriers are set up and the kernel before this one finishes (only there: should
    // that kernel write B, what is read after the wait below is what it wrote).  1 x 4096 x 11008, weights in HBM: 18.2 -> 17.6 us.
    if (warp >= LS_DRAIN_WARPS && warp < LS_DRAIN_WARPS + L_PRODUCERS && lane < t.b_boxes) {
        for (int step = s0 + warp - LS_DRAIN_WARPS; step < s1 && step < s0 + p.stages; step += L_PRODUCERS) {
            const int k = step * p.k_elems, r = col0 + t.b_box_cols * lane;
            linear_prefetch(&maps.b[0], p.b_k_major ? k : r, p.b_k_major ? r : k);
        }
    }
    if (warp == 1 && lane == 0) tma_prefetch_descriptor(&maps.a);
    if (warp == 0) {
        if (lane < p.stages) {
            mbar_init(full0 + 8 * lane, 1);
            mbar_init(empty0 + 8 * lane, 1);
        } else if (lane == 31) {
            mbar_init(accf, 1);
            *abort_flag = 0;
        }
        fence_barrier_init();
        fence_proxy_async();
    }
    if (warp == LS_DRAIN_WARPS + L_PRODUCERS) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(NB));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
    }
    linear_fence_before();
    __syncthreads();
    linear_fence_after();
    grid_launch_dependents();
    grid_dependency_wait();
    const uint32_t tmem = *tmem_slot;
    bool ok = true;

    if (warp >= LS_DRAIN_WARPS && warp < LS_DRAIN_WARPS + L_PRODUCERS) {
        const int turn = warp - LS_DRAIN_WARPS;
        int slot = turn % p.stages;
        uint32_t phase = (uint32_t)(turn / p.stages) & 1u;
        for (int step = s0 + turn; step < s1; step += L_PRODUCERS) {
            ok = mbar_wait(empty0 + 8 * slot, phase ^ 1, abort_flag);
            ok = __all_sync(0xFFFFFFFFu, ok);
            if (!ok) break;
            if (lane == 0) mbar_arrive_expect_tx(full0 + 8 * slot, (uint32_t)(p.a_stage_bytes + B_BYTES));
            __syncwarp();
            linear_load_step<false>(p, t, maps, &maps.b[0], lane, step, row0, col0, a_ring + (uint32_t)(slot * p.a_stage_bytes), b_ring + (uint32_t)(slot * B_BYTES),
                                    full0 + 8 * slot);
            slot += L_PRODUCERS;
            if (slot >= p.stages) {
                slot -= p.stages;
                phase ^= 1;
            }
        }
    } else if (warp == LS_DRAIN_WARPS + L_PRODUCERS) {
        const bool elected = linear_elect();
        int slot = 0;
        uint32_t phase = 0;
        bool landed = false;
        const uint32_t a0 = (a_ring & 0x3FFFFu) >> 4, b0 = (b_ring & 0x3FFFFu) >> 4;
        for (int step = s0; step < s1; ++step) {
            if (!landed) ok = mbar_wait(full0 + 8 * slot, phase, abort_flag);
            ok = __all_sync(0xFFFFFFFFu, ok);
            if (!ok) break;
            const int nslot = slot + 1 == p.stages ? 0 : slot + 1;
            landed = mbar_test_wait(full0 + 8 * nslot, nslot ? phase : phase ^ 1u);
            linear_mma_step<false, F8>(p, t, tmem, (a0 + (uint32_t)(slot * (p.a_stage_bytes >> 4))) | p.a_lbo,
                                       (b0 + (uint32_t)(slot * (B_BYTES >> 4))) | t.b_lbo, step > s0, elected);
            if (elected) linear_commit<false>(empty0 + 8 * slot);
            landed = __all_sync(0xFFFFFFFFu, landed);
            if (++slot == p.stages) {
                slot = 0;
                phase ^= 1;
            }
        }
        if (ok && elected) linear_commit<false>(accf);
        __syncwarp();
    } else {
        LinearSplitEpilogue<NB> epilogue;
        epilogue.fetch(p, rank, split, row0, col0, rows);
        // The sums of the rows that exist, to shared memory: 16 bytes apart beyond their length, so that the stores of eight threads
        // (eight rows) fall on all banks.  The ring is free: every copy has landed and every MMA has read it.
        ok = __all_sync(0xFFFFFFFFu, mbar_wait(accf, 0, abort_flag));   // (the loads from tensor memory are the whole warp's)
        const int q = warp & 3, c0 = (warp >> 2) * (NB / 2);      // TMEM lanes 32 q .., columns c0 ..
        if (ok && q * 32 < rows) {
            linear_fence_after();
            float *red = reinterpret_cast<float *>(smem) + (size_t)(q * 32 + lane) * (NB + 4) + c0;
            const bool mine = q * 32 + lane < rows;
#pragma unroll 1
            for (int c = 0; c < NB / 2; c += 32) {
                float z[32];
                linear_tmem_ld(tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(c0 + c), z);
                linear_tmem_wait(z);
                if (mine && bounds_ok(ls_red_bytes(q * 32 + lane, NB) + (c0 + c + 32) * 4 <= bar_off, p.status, 77)) {   // checked build: site 77
#pragma unroll
                    for (int j = 0; j < 32; j += 4) *reinterpret_cast<float4 *>(red + c + j) = make_float4(z[j], z[j + 1], z[j + 2], z[j + 3]);
                }
            }
            linear_fence_before();
        }
        if (!ok) settle_after_timeout();
        __syncwarp();
        linear_cluster_sync();       // all parts' sums are in their CTAs' shared memory
        if (ok) {
            const uint32_t sums = smem_u32(smem);
            switch (split) {
            case 1: epilogue.template finish<1>(p, sums, rank, row0, col0, rows); break;
            case 2: epilogue.template finish<2>(p, sums, rank, row0, col0, rows); break;
            case 3: epilogue.template finish<3>(p, sums, rank, row0, col0, rows); break;
            case 4: epilogue.template finish<4>(p, sums, rank, row0, col0, rows); break;
            case 5: epilogue.template finish<5>(p, sums, rank, row0, col0, rows); break;
            case 6: epilogue.template finish<6>(p, sums, rank, row0, col0, rows); break;
            case 7: epilogue.template finish<7>(p, sums, rank, row0, col0, rows); break;
            default: epilogue.template finish<8>(p, sums, rank, row0, col0, rows); break;
            }
        }
    }
    if (warp >= LS_DRAIN_WARPS) {
        if (!ok) settle_after_timeout();
        __syncwarp();
        linear_cluster_sync();       // (as the draining warps above)
    }
    if (!ok && lane == 0) atomicExch(p.status, (int)ESMM_ERR_TIMEOUT);
    __syncwarp();
    linear_cluster_meet();       // (the others may still read this CTA's sums)
    if (warp == LS_DRAIN_WARPS + L_PRODUCERS) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(NB));
}

// ---- launches -------------------------------------------------------------------------------------------------------------------
// Once per device: the SM count and the shared-memory allowance of every kernel.
static int linear_prepare(int dev, int *sms)
{
    static std::mutex mu;
    static int count[64];
    if (dev < 0 || dev >= 64) return record_cuda_error_text("esmm_linear: device ordinal out of range");
    std::lock_guard<std::mutex> lock(mu);
    if (!count[dev]) {
        int n = 0;
        ESMM_CUDA_TRY(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev));
        auto allow = [](auto kernel, int bytes) { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes); };
        ESMM_CUDA_TRY(allow(esmm_linear_pair_kernel<false, false, false>, SMEM_LIMIT));
        ESMM_CUDA_TRY(allow(esmm_linear_pair_kernel<false, false, true>, SMEM_LIMIT));
        ESMM_CUDA_TRY(allow(esmm_linear_pair_kernel<false, true, false>, SMEM_LIMIT));
        ESMM_CUDA_TRY(allow(esmm_linear_pair_kernel<false, true, true>, SMEM_LIMIT));
        ESMM_CUDA_TRY(allow(esmm_linear_pair_kernel<true, false, false>, SMEM_LIMIT));
        ESMM_CUDA_TRY(allow(esmm_linear_pair_kernel<true, false, true>, SMEM_LIMIT));
        ESMM_CUDA_TRY(allow(esmm_linear_pair_kernel<true, true, false>, SMEM_LIMIT));
        ESMM_CUDA_TRY(allow(esmm_linear_pair_kernel<true, true, true>, SMEM_LIMIT));
        ESMM_CUDA_TRY(allow(esmm_linear_split_kernel<64, false>, SMEM_LIMIT));
        ESMM_CUDA_TRY(allow(esmm_linear_split_kernel<64, true>, SMEM_LIMIT));
        ESMM_CUDA_TRY(allow(esmm_linear_split_kernel<128, false>, SMEM_LIMIT));
        ESMM_CUDA_TRY(allow(esmm_linear_split_kernel<128, true>, SMEM_LIMIT));
        count[dev] = n;
    }
    *sms = count[dev];
    return ESMM_OK;
}

// Row-major matrix of `outer` rows x `inner` elements of `dtype`.
static int linear_map(CUtensorMap *map, int dtype, const void *base, long inner, long outer, int box_inner, int box_outer,
                      CUtensorMapSwizzle swizzle = CU_TENSOR_MAP_SWIZZLE_128B)
{
    EncodeTiledFn enc = encode_tiled_fn();
    if (!enc) return record_cuda_error_text("cuTensorMapEncodeTiled entry point not available");
    const int size = dtype_bytes(dtype);
    cuuint64_t dims[2] = {(cuuint64_t)inner, (cuuint64_t)outer};
    cuuint64_t strides[1] = {(cuuint64_t)inner * size};
    cuuint32_t box[2] = {(cuuint32_t)box_inner, (cuuint32_t)box_outer};
    cuuint32_t estr[2] = {1, 1};
    const CUtensorMapDataType type = dtype == ESMM_F16    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                     : dtype == ESMM_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                          : CU_TENSOR_MAP_DATA_TYPE_UINT8;
    const CUresult r = enc(map, type, 2, const_cast<void *>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        char buf[96];
        snprintf(buf, sizeof buf, "cuTensorMapEncodeTiled failed with CUresult %d", (int)r);
        return record_cuda_error_text(buf);
    }
    return ESMM_OK;
}

struct LinearChoice {
    int pair_nb;          // 64, 128, 192, 256: the width of the pair kernel's tiles; 0: the split kernel
    int tail_nb, columns; // pair kernel: from this tile column on, tiles of another width; no columns: every tile is that much wider (joined)
    int nb, split;        // split kernel
};

// `border`: elements next to relu's border are to be found, which the pair kernel does in the staging boxes of its pieces (of joined tiles the last has none).
// Which kernel, tile widths and parts of K: the smallest estimated time in us.  The constants are fitted to the times of all variants on 216
// shapes (M = 1 .. 4096; K and N from 64 to 11008; 16 and 8 bits, B up to 90 MB, three sets of operands in turn): what the rule picks takes
// 0.6 % longer than the best variant on average, 11 % at most; on 663 shapes with their weights mostly in L2 1.5 %, 23 % at most.
static LinearChoice linear_choose(int M, int N, int ksteps, bool b_k_major, bool border, int sms)
{
    LinearChoice c = {0, 0, 0, 128, 1};
    const int pairs = std::max(1, sms / 2), down = ceil_div(M, 256);
    const double hbm = (((double)M + N) * ksteps * L_KBYTES + 2.0 * M * N) / 6.5e6;   // operands and C once
    double best = 1e30;
    // a K step is as long as its copies take, which are slower the more SMs copy
    auto step = [&](int nb, long tiles) { return (256 + nb) * (0.000562 + 0.000293 * (double)std::min<long>(tiles, pairs) / pairs); };
    for (int nb = 64; nb <= 256; nb += 64) {
        const int across = ceil_div(N, nb);
        const long tiles = (long)down * across, rounds = (tiles + pairs - 1) / pairs;
        const double fixed = 5.68 + 0.73 * nb / 64, t = fixed + std::max(rounds * ksteps * step(nb, tiles), hbm) + 1.5 * (rounds - 1);
        if (t < best) best = t, c.pair_nb = nb, c.columns = c.tail_nb = 0;
        // where the last round is partly filled: whole rounds of this width, the columns that are left in narrower tiles
        const int columns = (int)std::min<long>(across, tiles / pairs * pairs / down);
        if (columns < 1 || columns == across) continue;
        for (int tail = 64; tail < nb; tail += 64) {
            const long first = (long)columns * down, all = first + (long)ceil_div(N - columns * nb, tail) * down;
            const long wide = (first + pairs - 1) / pairs, narrow = (all + pairs - 1) / pairs - wide;
            const double tt = fixed + std::max(ksteps * (wide * step(nb, pairs) + narrow * step(tail, pairs)), hbm) + 1.5 * (wide + narrow - 1);
            if (tt < 0.98 * best) best = tt, c.pair_nb = nb, c.tail_nb = tail, c.columns = columns;
        }
    }
    // One tile per pair, wider than an MMA: as many columns as a single round takes.  (Two accumulators have no room beside each other then, so
    // there is no second round.)  The second MMA's columns of B come in 32s, of which a CTA has half; stored K x N in boxes of 32.  The ring is shorter
    // and nothing runs beside the epilogue: steps and fixed part are taken longer than those above, fitted to 44 shapes where this is possible
    // (us, best of the other widths / joined: 512 x 4096 x 11008 bf16 40.1 / 36.2, 256 x 4096 x 20480 bf16 43.0 / 38.4, 1536 x 11008 x 4096 e4m3 54.8 / 50.7,
    // but 2304 x 1024 x 4096 e4m3, where 512 columns are needed, 15.0 / 16.2).
    const int per_pair = b_k_major ? 32 : 64;
    auto joined_fits = [&](int extra) { return (long)down * ceil_div(N, LP_MAX_NB + extra) <= pairs; };
    for (int extra = per_pair; !border && extra <= LP_MAX_NB && (long)down * ceil_div(N, LP_MAX_NB) > pairs; extra += per_pair) {
        if (!joined_fits(extra)) continue;
        const int nb = LP_MAX_NB + extra;
        const double t = 6.68 + 0.73 * nb / 64 + std::max(1.2 * ksteps * step(nb, (long)down * ceil_div(N, nb)), hbm);
        if (t < best) best = t, c.pair_nb = LP_MAX_NB, c.tail_nb = extra, c.columns = 0;
        break;
    }
    const int rows = std::min(M, 128), box = ceil_div(rows, 8) * 8;
    for (int nb = 64; nb <= 128 && !border; nb += 64) {
        const long tiles = (long)ceil_div(M, 128) * ceil_div(N, nb);
        const double drain = (double)rows * nb / 16384;
        for (int split : {1, 2, 3, 4, 6, 8}) {
            if (split > ksteps) break;
            const long ctas = tiles * split, rounds = (ctas + 2 * sms - 1) / (2 * sms);
            const int steps = ceil_div(ksteps, split);
            const double kb = (box + nb) * (L_KBYTES / 1000.0);                // copied per step and CTA
            const double one = rounds * std::max(steps * std::max(0.412, kb / 52.5), 0.52 * drain), all = ctas * steps * kb / 11800.0;
            // (fewer CTAs than the SMs have room for have less of HBM under way)
            const double bytes = hbm * (1.0 + 0.66 * (1.0 - (double)ctas / (rounds * 2 * sms)));
            const double t = 3.42 + 5.2 * drain + std::max({one, all, bytes}) + 1.55 * ctas / (2 * sms) +
                             (split - 1) * (0.128 + (double)M * N * 4 / 2.86e6);   // sums through distributed shared memory
            if (t < best) best = t, c = {0, 0, 0, nb, split};
        }
    }
    const int forced = tuning_get("LINEAR_PAIR", -1);
    if ((forced == 0 && !border) || forced == 64 || forced == 128 || forced == 192 || forced == 256) c.pair_nb = forced, c.columns = c.tail_nb = 0;
    const int forced_tail = tuning_get("LINEAR_TAIL", 0);
    if (c.pair_nb && forced_tail > 0 && forced_tail < c.pair_nb && forced_tail % 64 == 0 && N > c.pair_nb)
        c.tail_nb = forced_tail, c.columns = (ceil_div(N, c.pair_nb) + 1) / 2;
    if (!border && forced > LP_MAX_NB && forced <= 2 * LP_MAX_NB && forced % per_pair == 0 && joined_fits(forced - LP_MAX_NB))
        c.pair_nb = LP_MAX_NB, c.tail_nb = forced - LP_MAX_NB, c.columns = 0;
    const int forced_split = tuning_get("LINEAR_SPLIT", 0);
    if (forced_split >= 1 && forced_split <= LS_MAX_SPLIT) c.split = std::min(forced_split, ksteps);
    const int forced_nb = tuning_get("LINEAR_COLUMNS", 0);
    if (forced_nb == 64 || forced_nb == 128) c.nb = forced_nb;
    return c;
}

}  // namespace esmm

extern "C" int esmm_linear(int M, int N, int K, int dtype, const void *d_A, int trans_a, const void *d_B, int trans_b, int out_dtype, void *d_C,
                           const float *d_a_scale, const float *d_b_scale, const void *d_bias, const void *d_residual, void *d_pre, int activation,
                           void *stream_)
{
    using namespace esmm;
    cudaStream_t stream = (cudaStream_t)stream_;
    if (!d_A || !d_B || !d_C) return ESMM_ERR_NULL;
    const bool f8 = dtype == ESMM_E4M3;
    if (!f8 && dtype != ESMM_F16 && dtype != ESMM_BF16) return ESMM_ERR_UNSUPPORTED;
    if (f8 ? (out_dtype != ESMM_F16 && out_dtype != ESMM_BF16) : out_dtype != dtype) return ESMM_ERR_UNSUPPORTED;
    if (f8 && (trans_a || !trans_b)) return ESMM_ERR_UNSUPPORTED;
    if (trans_a && trans_b) return ESMM_ERR_UNSUPPORTED;
    if (!activation_known(activation)) return ESMM_ERR_UNSUPPORTED;
    if (M <= 0 || N <= 0 || K <= 0 || N % 8) return ESMM_ERR_SHAPE;
    constexpr int most = 0x7FFFFFFF - 65536;   // (rows, columns and k are counted in int, in steps of tiles)
    if (M > most || N > most || K > most) return ESMM_ERR_TOO_LARGE;
    // rows of 16 bytes: A's are K (or, transposed, M) long, B's N or K
    const int per16 = f8 ? 16 : 8;
    if ((trans_a ? M : K) % per16 || (trans_b ? K % per16 : 0)) return ESMM_ERR_SHAPE;
    if (((uintptr_t)d_A | (uintptr_t)d_B | (uintptr_t)d_C | (uintptr_t)d_bias | (uintptr_t)d_residual | (uintptr_t)d_pre) & 15) return ESMM_ERR_ALIGN;
    if (((uintptr_t)d_a_scale | (uintptr_t)d_b_scale) & 3) return ESMM_ERR_ALIGN;

    int dev = 0, sms = 0;
    ESMM_CUDA_TRY(cudaGetDevice(&dev));
    int st = linear_prepare(dev, &sms);
    if (st != ESMM_OK) return st;

    LinearParams p;
    memset(&p, 0, sizeof p);
    p.M = M;
    p.N = N;
    p.k_elems = f8 ? 128 : 64;
    p.ksteps = ceil_div(K, p.k_elems);
    p.a_k_major = !trans_a;
    p.b_k_major = trans_b != 0;
    // K-major: the next MMA's 32 bytes of K lie in the same rows; MN-major: its 16 k are two groups of 1024 bytes on
    p.a_step = p.a_k_major ? 2u : 128u;
    p.a_lbo = (p.a_k_major ? 1u : 8192u >> 4) << 16;
    p.bf16 = out_dtype == ESMM_BF16;
    p.activation = activation;
    p.has_pre = d_pre != nullptr;
    p.has_residual = d_residual != nullptr;
    p.a_scale = d_a_scale;
    p.b_scale = d_b_scale;
    p.bias = d_bias;
    p.residual = d_residual;
    p.pre = d_pre;
    p.C = d_C;
    p.group_m = std::max(1, tuning_get("GROUP_M", GROUP_M));
    p.status = device_status_ptr();
    if (!p.status) return ESMM_ERR_CUDA;

    const bool border = d_pre && activation == ESMM_ACT_RELU;
    if (border) {
        p.border = std::min((float)K * (f8 ? LB_SHARE_F8 : LB_SHARE), LB_WIDEST);
        p.K = K;
        p.A = d_A;
        p.B = d_B;
        p.a_row = trans_a ? 1 : K;
        p.a_k = trans_a ? M : 1;
        p.b_col = trans_b ? K : 1;
        p.b_k = trans_b ? 1 : N;
    }
    const LinearChoice choice = linear_choose(M, N, p.ksteps, trans_b != 0, border, sms);
    const int rows_a = 128;                                                 // rows of A per CTA
    // few rows: boxes of as many as there are (what the MMA reads past them is never looked at)
    int a_box_rows = rows_a;
    if (!choice.pair_nb && p.a_k_major && M < rows_a) a_box_rows = ceil_div(M, 8) * 8;
    p.a_boxes = p.a_k_major ? 1 : rows_a / 64;
    LinearMaps maps;
    memset(&maps, 0, sizeof maps);
    st = p.a_k_major ? linear_map(&maps.a, dtype, d_A, K, M, p.k_elems, a_box_rows) : linear_map(&maps.a, dtype, d_A, M, K, 64, 64);
    if (st) return st;
    for (int i = 0; i < (choice.tail_nb ? 2 : 1); ++i) {
        LinearTile &t = p.kind[i];
        t.nb = i ? choice.tail_nb : choice.pair_nb ? choice.pair_nb : choice.nb;
        t.width = t.nb;
        const int cols = choice.pair_nb ? t.nb / 2 : t.nb;                  // columns of B per CTA
        // MN-major B in boxes of 64 columns, or of 32 with the 64-byte swizzle where a CTA's columns are no multiple of 64
        const bool wide = cols % 64 == 0;
        t.b_box_cols = p.b_k_major ? cols : wide ? 64 : 32;
        t.b_box_bytes = t.b_box_cols * 128;                                 // 128 bytes of K, or 64 k of two bytes each, per column
        t.b_boxes = cols / t.b_box_cols;
        t.stage_bytes = LP_A_BYTES + cols * L_KBYTES;
        t.b_desc_hi = p.b_k_major || wide ? L_DESC_HI : L_DESC_HI_64;
        t.b_step = p.b_k_major ? 2u : wide ? 128u : 64u;
        t.b_lbo = (p.b_k_major ? 1u : (uint32_t)t.b_box_bytes >> 4) << 16;
        // D = F32; A and B: F16 0, BF16 1, E4M3 0; bits 15, 16: MN-major; N >> 3, M >> 4
        const uint32_t ab_type = dtype == ESMM_BF16 ? 1u : 0u, mma_m = choice.pair_nb ? 256u : 128u;
        t.idesc = (1u << 4) | (ab_type << 7) | (ab_type << 10) | ((p.a_k_major ? 0u : 1u) << 15) | ((p.b_k_major ? 0u : 1u) << 16) |
                  (((uint32_t)t.nb >> 3) << 17) | ((mma_m >> 4) << 24);
        st = p.b_k_major ? linear_map(&maps.b[i], dtype, d_B, K, N, p.k_elems, cols)
                         : linear_map(&maps.b[i], dtype, d_B, N, K, t.b_box_cols, 64, wide ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B);
        if (st) return st;
    }

    if (choice.pair_nb) {
        st = linear_map(&maps.c, out_dtype, d_C, N, M, 64, 32);
        if (!st && d_residual) st = linear_map(&maps.residual, out_dtype, d_residual, N, M, 64, 32);
        if (!st && d_pre) st = linear_map(&maps.pre, out_dtype, d_pre, N, M, 64, 32);
        if (st) return st;
        p.tiles_m = ceil_div(M, 256);
        p.joined = choice.tail_nb && !choice.columns;
        if (p.joined) {
            p.kind[0].width += choice.tail_nb;
            p.kind[0].stage_bytes += p.kind[1].stage_bytes - LP_A_BYTES;
        }
        p.kind[0].tiles_n = choice.columns ? choice.columns : ceil_div(N, p.kind[0].width);
        p.wide_cols = p.kind[0].tiles_n * p.kind[0].width;
        if (choice.columns) p.kind[1].tiles_n = ceil_div(N - p.wide_cols, choice.tail_nb);
        if ((long)p.tiles_m * (p.kind[0].tiles_n + p.kind[1].tiles_n) > 0x7FFFFFFFL) return ESMM_ERR_TOO_LARGE;
        p.wide_tiles = p.tiles_m * p.kind[0].tiles_n;
        p.num_tiles = p.wide_tiles + p.tiles_m * p.kind[1].tiles_n;
        const int pairs = std::max(1, std::min(sms / 2, p.num_tiles));
        p.slot_bytes = p.kind[0].stage_bytes;
        // One box per epilogue warp leaves room for a sixth stage of the widest tiles, which long K gains from; with short K the epilogue's own
        // time counts, and the next piece's residual is under way in the second box.
        p.boxes = p.ksteps >= 16 ? 1 : 2;
        const int staging = LP_EPI_WARPS * p.boxes * LP_BOX;
        p.column_off = p.joined ? LP_BAR_OFF - 2 * 2 * LP_MAX_NB * 4 : LP_COLUMN_OFF;
        p.box_off = (p.column_off - staging) & ~1023;
        p.stages = std::min(LP_MAX_STAGES, p.box_off / p.slot_bytes);
        auto go = [&](auto kernel) -> int {
            ESMM_CUDA_TRY(launch_dependent(kernel, dim3((unsigned)(2 * pairs)), dim3(LP_THREADS), (size_t)LP_SMEM, stream, maps, p));
            return ESMM_OK;
        };
        auto by_type = [&](auto with_border) -> int {
            constexpr bool BORDER = decltype(with_border)::value;
            if (p.bf16) return f8 ? go(esmm_linear_pair_kernel<true, true, BORDER>) : go(esmm_linear_pair_kernel<false, true, BORDER>);
            return f8 ? go(esmm_linear_pair_kernel<true, false, BORDER>) : go(esmm_linear_pair_kernel<false, false, BORDER>);
        };
        return border ? by_type(std::true_type()) : by_type(std::false_type());
    }

    p.tiles_m = ceil_div(M, 128);
    p.kind[0].tiles_n = ceil_div(N, choice.nb);
    if ((long)p.tiles_m * p.kind[0].tiles_n * choice.split > 0x7FFFFFFFL) return ESMM_ERR_TOO_LARGE;
    p.num_tiles = p.tiles_m * p.kind[0].tiles_n;
    p.a_stage_bytes = a_box_rows * L_KBYTES;
    const int b_stage = choice.nb * L_KBYTES, steps = ceil_div(p.ksteps, choice.split);
    // two CTAs per SM; the MMA reads 128 rows of A from any slot, so past the last one the B ring (16 KB at least) has to follow
    p.stages = std::min({LS_MAX_STAGES, steps, (112 * 1024 - 512) / (p.a_stage_bytes + b_stage)});
    p.stages = std::max(p.stages, ceil_div(128 * L_KBYTES, b_stage));
    const int ring = p.stages * (p.a_stage_bytes + b_stage);
    const int bar_off = (std::max(ring, ls_red_bytes(std::min(M, 128), choice.nb)) + 15) & ~15;
    const size_t smem = std::max((size_t)bar_off + (2 * LS_MAX_STAGES + 1) * 8 + 16, (size_t)LS_MIN_SMEM);
    if (smem > (size_t)SMEM_LIMIT) return ESMM_ERR_TOO_LARGE;
    auto go = [&](auto kernel) -> int {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)(p.num_tiles * choice.split));
        cfg.blockDim = dim3(LS_THREADS);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = stream;
        cudaLaunchAttribute attr[2];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = (unsigned)choice.split;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[1].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = tuning_get("NO_DEPENDENT_LAUNCH", 0) ? 1 : 2;
        ESMM_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, maps, p, choice.split, bar_off));
        return ESMM_OK;
    };
    if (choice.nb == 64) return f8 ? go(esmm_linear_split_kernel<64, true>) : go(esmm_linear_split_kernel<64, false>);
    return f8 ? go(esmm_linear_split_kernel<128, true>) : go(esmm_linear_split_kernel<128, false>);
}
