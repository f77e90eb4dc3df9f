// dllm_int8.cu -- the LM-head tail with 8-bit integer weights: rows to int8 codes with a scale each,
// and the int8 matrix product with a scale for each token and channel.
//
//   codes    y = x, or x * g / sqrt(mean(x^2) + eps); s = (float)(max|y| / 127); q = rint(y / s)
//   product  out[m][n] = a_scale[m] * b_scale[n] * sum_k a[m][k] * b[n][k], the sum exact in int32
//   softcap  cap * tanhf(out / cap) when cap > 0 (src/core/context.c:873-876)
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

constexpr int MM_T = 64;  // output tile

template <int DT>
__global__ void __launch_bounds__(256) matmul_i8_kernel(const int8_t *a, int64_t lda, const float *sa, const int8_t *b,
                                                        int64_t ldb, const float *sb, int m, int n, int k,
                                                        float softcap, void *out, int64_t ldo) {
    __shared__ int as[16][MM_T + 1], bs[16][MM_T + 1];  // 64 bytes of k as 16 words
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const int64_t m0 = (int64_t)blockIdx.y * MM_T, n0 = (int64_t)blockIdx.x * MM_T;
    int acc[4][4] = {};
    for (int k0 = 0; k0 < k; k0 += 64) {
        for (int i = tid; i < MM_T * 16; i += 256) {
            const int r = i >> 4, wd = i & 15, at = k0 + 4 * wd;
            int av = 0, bv = 0;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if (at + j >= k) break;
                if (m0 + r < m) av |= (int)(uint8_t)a[(m0 + r) * lda + at + j] << (8 * j);
                if (n0 + r < n) bv |= (int)(uint8_t)b[(n0 + r) * ldb + at + j] << (8 * j);
            }
            as[wd][r] = av;
            bs[wd][r] = bv;
        }
        __syncthreads();
#pragma unroll
        for (int wd = 0; wd < 16; wd++)
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) acc[i][j] = __dp4a(as[wd][ty * 4 + i], bs[wd][tx * 4 + j], acc[i][j]);
        __syncthreads();
    }
    for (int i = 0; i < 4; i++)
        for (int j = 0; j < 4; j++) {
            const int64_t r = m0 + ty * 4 + i, c = n0 + tx * 4 + j;
            if (r >= m || c >= n) continue;
            float v = __fmul_rn(__fmul_rn((float)acc[i][j], sa[r]), sb[c]);
            if (softcap > 0.0f) v = __fmul_rn(softcap, tanhf(__fdiv_rn(v, softcap)));
            store_out<DT>(out, r * ldo + c, v);
        }
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
    (void)status;
    if (m == 0 || n == 0) return DLLM_OK;
    const dim3 grid((n + MM_T - 1) / MM_T, (m + MM_T - 1) / MM_T);
    auto go = [&](auto kernel) {
        kernel<<<grid, 256, 0, stream>>>(a, lda, sa, b, ldb, sb, m, n, k, softcap, out, ldo);
        return cudaGetLastError() == cudaSuccess ? DLLM_OK : DLLM_ERR_CUDA;
    };
    if (out_dtype == DLLM_DTYPE_F32) return go(matmul_i8_kernel<DLLM_DTYPE_F32>);
    if (out_dtype == DLLM_DTYPE_BF16) return go(matmul_i8_kernel<DLLM_DTYPE_BF16>);
    return go(matmul_i8_kernel<DLLM_DTYPE_F16>);
}

}  // namespace dllm
