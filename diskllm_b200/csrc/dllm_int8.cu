// dllm_int8.cu -- the LM-head tail with 8-bit integer weights: rows to int8 codes with a scale each,
// and the int8 matrix product with a scale for each token and channel.
//
//   codes    y = x, or x * g / sqrt(mean(x^2) + eps); s = (float)(max|y| / 127); q = rint(y / s)
//   product  out[m][n] = a_scale[m] * b_scale[n] * sum_k a[m][k] * b[n][k], the sum exact in int32
//   softcap  cap * tanhf(out / cap) when cap > 0 (src/core/context.c:873-876)
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <float.h>
#include <math.h>

#include "dllm_internal.h"

namespace dllm {
namespace {

// ----------------------------------------------------------------------------------------
// rows to int8 codes

constexpr int QZ_THREADS = 256;

template <int DT>
__device__ __forceinline__ float load_elem(const void *row, int64_t i) {
    if (DT == DLLM_DTYPE_F32) return ((const float *)row)[i];
    const unsigned short u = ((const unsigned short *)row)[i];
    if (DT == DLLM_DTYPE_BF16) return __uint_as_float((uint32_t)u << 16);
    return __half2float(__ushort_as_half(u));
}

// sum (or maximum) over the block of one double per thread
template <bool MAX>
__device__ __forceinline__ double block_reduce(double v, double *part) {
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, nw = blockDim.x >> 5;
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        const double w = __shfl_xor_sync(0xffffffffu, v, o);
        v = MAX ? fmax(v, w) : v + w;
    }
    if (lane == 0) part[wid] = v;
    __syncthreads();
    v = part[0];
    for (int i = 1; i < nw; i++) v = MAX ? fmax(v, part[i]) : v + part[i];
    __syncthreads();
    return v;
}

// One CTA per row.  The normalised value, the largest one and the quotient are formed in 64 bits:
// a quotient next to a half-integer would otherwise round to the other code.
template <int DT>
__global__ void __launch_bounds__(QZ_THREADS) quantize_rows_kernel(const void *x, int64_t x_stride, int cols, int norm,
                                                                   const float *w, float eps, int add_one, int8_t *q,
                                                                   int64_t q_stride, float *scale) {
    __shared__ double part[QZ_THREADS / 32];
    const int tid = threadIdx.x;
    const size_t esz = DT == DLLM_DTYPE_F32 ? 4 : 2;
    const unsigned char *row = (const unsigned char *)x + (size_t)blockIdx.x * x_stride * esz;
    int8_t *qrow = q + (size_t)blockIdx.x * q_stride;
    double rs = 1.0;
    if (norm) {
        double ss = 0.0;
        for (int i = tid; i < cols; i += QZ_THREADS) {
            const double v = load_elem<DT>(row, i);
            ss += v * v;
        }
        rs = 1.0 / sqrt(block_reduce<false>(ss, part) / (double)cols + (double)eps);
    }
    auto value = [&](int i) {
        double y = (double)load_elem<DT>(row, i) * rs;
        if (w) y *= (double)w[i] + (add_one ? 1.0 : 0.0);
        return y;
    };
    double big = 0.0;
    int bad = 0;
    for (int i = tid; i < cols; i += QZ_THREADS) {
        const double a = fabs(value(i));
        bad |= !(a <= DBL_MAX);
        big = fmax(big, a);
    }
    big = block_reduce<true>(big, part);
    float s = __double2float_rn(big / 127.0);
    bad = __syncthreads_or(bad | !(s <= FLT_MAX));
    if (bad) s = __int_as_float(0x7fc00000);  // NaN: every product of the row is NaN
    const bool zero = bad || !(s >= FLT_MIN);
    if (!bad && zero) s = 0.0f;
    if (tid == 0) scale[blockIdx.x] = s;
    const double sd = (double)s;
    for (int i = tid; i < cols; i += QZ_THREADS) qrow[i] = zero ? 0 : (int8_t)__double2int_rn(value(i) / sd);
}

// ----------------------------------------------------------------------------------------
// int8 product

template <int DT>
__device__ __forceinline__ void store_out(void *out, int64_t i, float v) {
    if (DT == DLLM_DTYPE_F32) ((float *)out)[i] = v;
    else if (DT == DLLM_DTYPE_BF16) ((__nv_bfloat16 *)out)[i] = __float2bfloat16_rn(v);
    else ((__half *)out)[i] = __float2half_rn(v);
}

// The product runs on the tensor cores (tcgen05.mma kind::i8, sums in tensor memory).  The channels
// (rows of b: output weights) are the instruction's 128 rows and the tokens (rows of a) its columns,
// so a few tokens cost a narrow instruction, and an accumulator lane is a channel: a warp's 32 lanes
// store 32 neighbouring outputs of one token.
constexpr int MM_ROWS = 128;                 // channels of a tile
constexpr int MM_KB = 128;                   // bytes of k in a pipeline stage (one swizzle row)
constexpr int MM_EPI_WARPS = 8;
constexpr int MM_THREADS = 64 + 32 * MM_EPI_WARPS;
constexpr int MM_MAX_STAGES = 12;
constexpr int MM_SMEM = 220 * 1024;          // stages, with 1 KB to align them

struct MmArgs {
    const float *sa, *sb;
    void *out;
    int64_t ldo;
    int32_t *status;
    int m, n, k;
    int nt;          // tokens of a tile (a multiple of 16, at most 256)
    int token_tiles;
    int stages;
    int tmem_cols;   // allocated columns: two accumulators
    float softcap;
};

__device__ __forceinline__ uint32_t smem_addr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(uint32_t bar, int count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n.reg .pred p;\n"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
        "selp.b32 %0, 1, 0, p;\n}\n"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    return done;
}
// Bounded wait: gives up after two seconds, or once another role of the CTA has.
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile int *gave_up) {
    if (mbar_try(bar, parity)) return true;
    unsigned long long t0, t;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t0));
    for (;;) {
        for (int i = 0; i < 64; i++)
            if (mbar_try(bar, parity)) return true;
        asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
        if (*gave_up || t - t0 > 2000000000ull) {
            *gave_up = 1;
            return false;
        }
    }
}
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap *map, int x, int y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(bar)
        : "memory");
}
// Operand descriptor: rows of 128 bytes, 128-byte swizzle, groups of 8 rows 1024 bytes apart.
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr) {
    return (uint64_t)((addr & 0x3ffff) >> 4) | (uint64_t)1 << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 |
           (uint64_t)2 << 61;
}
__device__ __forceinline__ void mma_i8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile(
        "{\n.reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
        : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// 16 accumulator columns of the warp's 32 lanes.  The wait is part of the statement, so that no use
// of the registers can be scheduled before it.
__device__ __forceinline__ void tmem_load16(uint32_t addr, int (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
        "[%16];\n"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(addr)
        : "memory");
}

// Persistent, one CTA per SM.  Warp 0 copies tiles (TMA), warp 1 issues the products, warps 2 to 9
// scale and store; two accumulators, so that a tile's stores run under the next tile's products.
template <int DT, bool CAP>
__global__ void __launch_bounds__(MM_THREADS, 1) matmul_i8_kernel(const __grid_constant__ CUtensorMap map_a,
                                                                  const __grid_constant__ CUtensorMap map_b, MmArgs p) {
    extern __shared__ unsigned char raw[];
    __shared__ __align__(8) uint64_t bars[2 * MM_MAX_STAGES + 5];
    __shared__ uint32_t tmem_base;
    __shared__ int gave_up;
    const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
    const uint32_t tiles = (smem_addr(raw) + 1023) & ~1023u;
    const int stage_bytes = (MM_ROWS + p.nt) * MM_KB;
    const uint32_t full = smem_addr(bars), empty = full + 8 * MM_MAX_STAGES, done = full + 16 * MM_MAX_STAGES,
                   drained = done + 16, flushed = drained + 16;
    const int64_t ntiles = (int64_t)((p.n + MM_ROWS - 1) / MM_ROWS) * p.token_tiles;
    const int kblocks = (p.k + MM_KB - 1) / MM_KB;

    if (wid == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_base)),
                     "r"(p.tmem_cols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    if (tid == 0) {
        for (int i = 0; i < p.stages; i++) {
            mbar_init(full + 8 * i, 1);
            mbar_init(empty + 8 * i, 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(done + 8 * i, 1);
            mbar_init(drained + 8 * i, MM_EPI_WARPS);
        }
        mbar_init(flushed, 1);
        gave_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = tmem_base;

    if (wid == 0) {
        if (lane == 0) {
            uint32_t step = 0;  // k blocks so far: stage step % stages, use step / stages
            bool ok = true;
            for (int64_t t = blockIdx.x; t < ntiles && ok; t += gridDim.x) {
                const int y_b = (int)(t / p.token_tiles) * MM_ROWS, y_a = (int)(t % p.token_tiles) * p.nt;
                for (int kb = 0; kb < kblocks; kb++, step++) {
                    const uint32_t s = step % p.stages, use = step / p.stages;
                    if (use > 0 && !(ok = mbar_wait(empty + 8 * s, (use - 1) & 1, &gave_up))) break;
                    const uint32_t at = tiles + s * stage_bytes, bar = full + 8 * s;
                    mbar_expect(bar, stage_bytes);
                    tma_load(at, &map_b, kb * MM_KB, y_b, bar);
                    tma_load(at + MM_ROWS * MM_KB, &map_a, kb * MM_KB, y_a, bar);
                }
            }
            // no copy may be in flight when the CTA ends, also where a wait ran out
            volatile int alone = 0;
            for (uint32_t i = step < (uint32_t)p.stages ? 0 : step - p.stages; i < step; i++)
                mbar_wait(full + 8 * (i % p.stages), (i / p.stages) & 1, &alone);
        }
        __syncwarp();
    } else if (wid == 1) {
        if (lane == 0) {
            // sums of signed 8-bit products in 32-bit integers, 128 rows by nt columns
            const uint32_t idesc = 2u << 4 | 1u << 7 | 1u << 10 | (uint32_t)(p.nt >> 3) << 17 | (MM_ROWS >> 4) << 24;
            uint32_t step = 0, it = 0;
            bool ok = true;
            for (int64_t t = blockIdx.x; t < ntiles && ok; t += gridDim.x, it++) {
                const uint32_t acc = it & 1;
                if (it >= 2 && !(ok = mbar_wait(drained + 8 * acc, ((it >> 1) - 1) & 1, &gave_up))) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                for (int kb = 0; kb < kblocks; kb++, step++) {
                    const uint32_t s = step % p.stages;
                    if (!(ok = mbar_wait(full + 8 * s, (step / p.stages) & 1, &gave_up))) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint32_t at = tiles + s * stage_bytes;
                    const uint64_t da = operand_desc(at), db = operand_desc(at + MM_ROWS * MM_KB);
#pragma unroll
                    for (int j = 0; j < MM_KB / 32; j++)  // 32 bytes of k at a time
                        mma_i8(tmem + acc * p.nt, da + 2 * j, db + 2 * j, idesc, kb > 0 || j > 0);
                    mma_commit(empty + 8 * s);
                }
                if (ok) mma_commit(done + 8 * acc);
            }
            mma_commit(flushed);  // nor any product
            volatile int alone = 0;
            mbar_wait(flushed, 0, &alone);
        }
        __syncwarp();
    } else {
        const int quarter = wid & 3, half = (wid - 2) >> 2;  // tensor memory lanes of a warp: 32 * (warp % 4)
        uint32_t it = 0;
        for (int64_t t = blockIdx.x; t < ntiles; t += gridDim.x, it++) {
            const uint32_t acc = it & 1;
            const int ch = (int)(t / p.token_tiles) * MM_ROWS + quarter * 32 + lane;
            const int t0 = (int)(t % p.token_tiles) * p.nt;
            const float sb = ch < p.n ? __ldg(p.sb + ch) : 0.0f;
            int ok = mbar_wait(done + 8 * acc, (it >> 1) & 1, &gave_up);
            if (!__all_sync(0xffffffffu, ok)) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            for (int c = half * 16; c < p.nt; c += 32) {
                int r[16];
                tmem_load16(tmem + acc * p.nt + c + ((uint32_t)quarter << 21), r);
                if (ch < p.n) {
#pragma unroll
                    for (int j = 0; j < 16; j++) {
                        const int token = t0 + c + j;
                        if (token < p.m) {
                            float v = __fmul_rn(__fmul_rn((float)r[j], __ldg(p.sa + token)), sb);
                            if (CAP) v = __fmul_rn(p.softcap, tanhf(__fdiv_rn(v, p.softcap)));
                            store_out<DT>(p.out, token * p.ldo + ch, v);
                        }
                    }
                }
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(drained + 8 * acc);
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (wid == 1) {
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(p.tmem_cols));
        if (lane == 0 && gave_up && p.status) atomicOr(p.status, DLLM_ROW_ERR_TIMEOUT);
    }
}

using EncodeTiled = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                 const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encode_tiled() {
    static const EncodeTiled f = [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult got;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &got) != cudaSuccess ||
            got != cudaDriverEntryPointSuccess)
            p = nullptr;
        return (EncodeTiled)p;
    }();
    return f;
}

// Rows of codes, copied in boxes of box_rows x 128 bytes; what lies outside reads as zero.
bool code_map(CUtensorMap *map, const int8_t *base, int rows, int cols, int64_t stride, int box_rows) {
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)stride};
    const cuuint32_t box[2] = {MM_KB, (cuuint32_t)box_rows}, one[2] = {1, 1};
    const EncodeTiled f = encode_tiled();
    return f && f(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, (void *)base, dims, strides, box, one,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int sm_count() {
    int dev = 0, n = 148;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    return n;
}

}  // namespace

dllm_status launch_quantize_i8(int rows, int cols, const void *x, int64_t x_stride, int x_dtype, int norm,
                               const float *norm_w, float eps, int add_one, int8_t *q, int64_t q_stride, float *scale,
                               cudaStream_t stream) {
    if (rows == 0) return DLLM_OK;
    auto go = [&](auto kernel) {
        kernel<<<rows, QZ_THREADS, 0, stream>>>(x, x_stride, cols, norm, norm_w, eps, add_one, q, q_stride, scale);
        return cudaGetLastError() == cudaSuccess ? DLLM_OK : DLLM_ERR_CUDA;
    };
    if (x_dtype == DLLM_DTYPE_F32) return go(quantize_rows_kernel<DLLM_DTYPE_F32>);
    if (x_dtype == DLLM_DTYPE_BF16) return go(quantize_rows_kernel<DLLM_DTYPE_BF16>);
    return go(quantize_rows_kernel<DLLM_DTYPE_F16>);
}

dllm_status launch_matmul_i8(int m, int n, int k, const int8_t *a, int64_t lda, const float *sa, const int8_t *b,
                             int64_t ldb, const float *sb, float softcap, void *out, int64_t ldo, int out_dtype,
                             int32_t *status, cudaStream_t stream) {
    if (m == 0 || n == 0) return DLLM_OK;
    MmArgs p = {};
    p.sa = sa;
    p.sb = sb;
    p.out = out;
    p.ldo = ldo;
    p.status = status;
    p.m = m;
    p.n = n;
    p.k = k;
    p.softcap = softcap;
    // token tiles of equal size, at most 256 (the widest instruction)
    p.token_tiles = (m + 255) / 256;
    p.nt = ((m + p.token_tiles - 1) / p.token_tiles + 15) / 16 * 16;
    p.stages = (MM_SMEM - 1024) / ((MM_ROWS + p.nt) * MM_KB);
    if (p.stages > MM_MAX_STAGES) p.stages = MM_MAX_STAGES;
    p.tmem_cols = 32;
    while (p.tmem_cols < 2 * p.nt) p.tmem_cols *= 2;
    CUtensorMap map_a, map_b;
    if (!code_map(&map_a, a, m, k, lda, p.nt) || !code_map(&map_b, b, n, k, ldb, MM_ROWS)) return DLLM_ERR_CUDA;
    const int64_t tiles = (int64_t)((n + MM_ROWS - 1) / MM_ROWS) * p.token_tiles;
    const int sms = sm_count(), grid = tiles < sms ? (int)tiles : sms;
    auto go = [&](auto kernel) {
        if (cudaFuncSetAttribute((const void *)kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, MM_SMEM) != cudaSuccess)
            return DLLM_ERR_CUDA;
        kernel<<<grid, MM_THREADS, MM_SMEM, stream>>>(map_a, map_b, p);
        return cudaGetLastError() == cudaSuccess ? DLLM_OK : DLLM_ERR_CUDA;
    };
    const bool cap = softcap > 0.0f;
    if (out_dtype == DLLM_DTYPE_F32)
        return cap ? go(matmul_i8_kernel<DLLM_DTYPE_F32, true>) : go(matmul_i8_kernel<DLLM_DTYPE_F32, false>);
    if (out_dtype == DLLM_DTYPE_BF16)
        return cap ? go(matmul_i8_kernel<DLLM_DTYPE_BF16, true>) : go(matmul_i8_kernel<DLLM_DTYPE_BF16, false>);
    return cap ? go(matmul_i8_kernel<DLLM_DTYPE_F16, true>) : go(matmul_i8_kernel<DLLM_DTYPE_F16, false>);
}

}  // namespace dllm
