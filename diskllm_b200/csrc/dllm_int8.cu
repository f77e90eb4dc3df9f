// dllm_int8.cu -- the LM-head tail with 8-bit integer weights: rows to int8 codes with a scale each,
// and the int8 matrix product with a scale for each token and channel.
//
//   codes    y = x, or x * g / sqrt(mean(x^2) + eps); s = (float)(max|y| / 127); q = rint(y / s)
//   product  out[m][n] = a_scale[m] * b_scale[n] * sum_k a[m][k] * b[n][k], the sum exact in int32
//   softcap  cap * tanh(out / cap) when cap > 0 (src/core/context.c:873-876)
//
// Measured on B200 (GPU time of a call, a few dozen back to back; in brackets when calls follow one another
// for seconds, so that the power cap lowers the SM clock from 1965 MHz):
//   codes of 32000 x 4096, bf16    78 us (82 at 1.9 GHz; 393 MB: 5.0 TB/s); fp16 70, fp32 110;
//     of 4 x 4096 fp32 with norm    4.5 us; of 2048 x 4096 fp32 with norm    29 us (6.4 at the copy rate): 64-bit
//     operations, two to four for each value
//     off the 16-byte path: 32000 x 4097 bf16, read by value and written by byte    378 us;
//     8192 x 28672 bf16, too long for registers    583 us (108 at the copy rate)
//   product 2048 x 8192 x 8192 to bf16    105 us (2.6e15 operations/s; 123 at 1.57 GHz);
//     16 x 4096 x 4096    8.7 us
//   LM head 1 x 4096 x 128256    85 to 89 us (91 at 1.87 GHz; 526 MB: 6.1 TB/s, 0.94 of the measured copy rate);
//     256 x 2304 x 256000 with softcap    164 to 172 us (204 at 1.25 GHz; 852 MB, 130 us at the copy rate)
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <float.h>
#include <math.h>

#include "dllm_internal.h"
#include "dllm_pair.cuh"

namespace dllm {
namespace {

// ----------------------------------------------------------------------------------------
// rows to int8 codes

template <int DT>
struct Elem {
    static constexpr int SIZE = DT == DLLM_DTYPE_F32 ? 4 : 2;
    static constexpr int VEC = 16 / SIZE;  // elements of 16 bytes
};

template <int DT>
__device__ __forceinline__ float load_elem(const void *row, int64_t i) {
    if (DT == DLLM_DTYPE_F32) return ((const float *)row)[i];
    const unsigned short u = ((const unsigned short *)row)[i];
    if (DT == DLLM_DTYPE_BF16) return __uint_as_float((uint32_t)u << 16);
    return __half2float(__ushort_as_half(u));
}

template <int DT>
__device__ __forceinline__ void unpack(const uint4 &v, float *f) {
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if (DT == DLLM_DTYPE_F32) f[i] = __uint_as_float(u[i]);
        else if (DT == DLLM_DTYPE_BF16) {
            f[2 * i] = __uint_as_float(u[i] << 16);
            f[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
        } else {
            f[2 * i] = __half2float(__ushort_as_half((unsigned short)(u[i] & 0xffffu)));
            f[2 * i + 1] = __half2float(__ushort_as_half((unsigned short)(u[i] >> 16)));
        }
    }
}

// sum (or maximum) over the TPR threads of a row, in every one of them
template <bool MAX, int TPR>
__device__ __forceinline__ double row_reduce(double v, double *part) {
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        const double w = __shfl_xor_sync(0xffffffffu, v, o);
        v = MAX ? fmax(v, w) : v + w;
    }
    if (TPR == 32) return v;
    const int lane = threadIdx.x & 31;
    if (lane == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = lane < TPR / 32 ? part[lane] : 0.0;  // sums of squares and magnitudes: zero changes neither
#pragma unroll
    for (int o = TPR / 64; o; o >>= 1) {
        const double w = __shfl_xor_sync(0xffffffffu, v, o);
        v = MAX ? fmax(v, w) : v + w;
    }
    return __shfl_sync(0xffffffffu, v, 0);
}

struct QuantArgs {
    const void *x;
    int64_t x_stride, q_stride;
    int rows, cols, norm, add_one;
    const float *w;
    float eps;
    int8_t *q;
    float *scale;
};

// A row's scale from its largest magnitude: (float)(big / 127); 0 below the smallest normal number,
// NaN for a row that is not finite (every product of the row is then NaN).
__device__ __forceinline__ float scale_of(double big) {
    if (!(big <= DBL_MAX)) return __int_as_float(0x7fc00000);
    const float s = __double2float_rn(big / 127.0);
    return s > FLT_MAX ? __int_as_float(0x7fc00000) : s >= FLT_MIN ? s : 0.0f;
}

__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if one of them is
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}

// TPR threads hold a row in registers, E elements each (vectors of 16 bytes where the rows allow it).
// A code is formed in 32 bits, x * (rs / s) * g with four roundings at most, so within
// 127.5 * 4 * 2^-24 = 3.1e-5 of the quotient, and rounded by adding 1.5 * 2^23, whose sum holds the
// code in its low byte; only where that lies within 6e-5 of a half-integer is it decided anew:
//   without norm, by the sign of x - h * s for the half-integer h, which one fused operation gives exactly
//     (a value of half the row's largest one lies there, so in 16-bit types that is no rare case);
//   with norm, by comparing y with h * s in 64 bits, where h * s is exact.
// With norm the sum of squares, the largest |x * g| and the scale are 64-bit too.  The factors' products
// stay inside the range of fp32 for scales from 1e-30 to 1e30 and factors up to 1e30; rows with
// others are divided in 64 bits.
// Without norm 64 registers, so that 1024 threads fit on an SM (32000 x 4096 bf16: 80 us, 86 with 68
// registers); with norm they would spill.
template <int DT, int TPR, int E, bool VECTORS, bool NORM>
__global__ void __launch_bounds__(TPR == 32 ? 256 : TPR, NORM ? 1 : TPR == 32 ? 4 : 1024 / TPR)
    quantize_rows_kernel(QuantArgs a) {
    constexpr int VEC = VECTORS ? Elem<DT>::VEC : 1, NV = E / VEC;
    constexpr float MAGIC = 12582912.0f;
    __shared__ double part[2][32];
    asm volatile("griddepcontrol.launch_dependents;");
    const int t = threadIdx.x % TPR, lane = threadIdx.x & 31;
    const int64_t row = TPR == 32 ? (int64_t)blockIdx.x * 8 + threadIdx.x / 32 : blockIdx.x;
    if (row >= a.rows) return;
    const unsigned char *src = (const unsigned char *)a.x + (size_t)row * a.x_stride * Elem<DT>::SIZE;
    int8_t *dst = a.q + (size_t)row * a.q_stride;
    auto place = [&](int v) { return (v * TPR + t) * VEC; };  // first element of this thread's vector v
    float x[E], g[NORM ? E : 1];
    const float one = a.w && !a.add_one ? 0.0f : 1.0f;  // the factor is w + one
#pragma unroll
    for (int v = 0; v < NV; v++) {
        const int at = place(v);
        if (VECTORS && at + VEC <= a.cols) unpack<DT>(__ldg((const uint4 *)(src + (size_t)at * Elem<DT>::SIZE)), x + v * VEC);
        else
#pragma unroll
            for (int e = 0; e < VEC; e++) x[v * VEC + e] = at + e < a.cols ? load_elem<DT>(src, at + e) : 0.0f;
        if (NORM)
#pragma unroll
            for (int e = 0; e < VEC; e++) g[v * VEC + e] = a.w && at + e < a.cols ? __ldg(a.w + at + e) : 0.0f;
    }
    double rs = 1.0;
    float s, c, gmax = 0.0f;
    if (NORM) {
        double ss = 0.0, big = 0.0;
#pragma unroll
        for (int e = 0; e < E; e++) {
            ss = fma(wide(x[e]), wide(x[e]), ss);
            const double y = fabs(wide(x[e]) * (wide(g[e]) + (double)one));
            big = y <= DBL_MAX ? fmax(big, y) : INFINITY;
            g[e] = __fadd_rn(g[e], one);
            gmax = fmaxf(gmax, fabsf(g[e]));
        }
        rs = 1.0 / sqrt(row_reduce<false, TPR>(ss, part[0]) / (double)a.cols + wide(a.eps));
        big = row_reduce<true, TPR>(big, part[1]);
        s = rs <= DBL_MAX ? scale_of(big * rs) : __int_as_float(0x7fc00000);  // else a row of zeros and eps = 0
        c = s > 0.0f ? __double2float_rn(rs / (double)s) : 0.0f;
    } else {
        float m = 0.0f;
#pragma unroll
        for (int e = 0; e < E; e++) m = max_nan(m, fabsf(x[e]));
        uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(m));  // NaN is above infinity
        if (TPR > 32) {
            uint32_t *tops = (uint32_t *)part;
            if (lane == 0) tops[threadIdx.x >> 5] = top;
            __syncthreads();
            top = __reduce_max_sync(0xffffffffu, lane < TPR / 32 ? tops[lane] : 0);
        }
        s = top < 0x7f800000u ? __fdiv_rn(__uint_as_float(top), 127.0f) : __int_as_float(0x7fc00000);
        c = s > 0.0f ? __fdiv_rn(1.0f, s) : 0.0f;
    }
    if (t == 0) a.scale[row] = s;
    const bool fast = s > 1e-30f && s < 1e30f && c > 1e-30f && c < 1e30f && gmax <= 1e30f;
#pragma unroll
    for (int v = 0; v < NV; v++) {
        const int at = place(v);
        uint32_t sum[VEC < 2 ? 2 : VEC];  // the codes are their low bytes
        float off = 0.0f;                 // how far the quotients are from integers
#pragma unroll
        for (int e = 0; e < VEC; e += 2) {
            const int i = v * VEC + e, j = VEC > 1 ? i + 1 : i;
            Pair y = mul2(Pair(x[i], x[j]), Pair(c, c));
            if (NORM) y = mul2(y, Pair(g[i], g[j]));
            const Pair m = add2(y, Pair(MAGIC, MAGIC)), r = add2(m, Pair(-MAGIC, -MAGIC));
            const Pair d = fma2(r, Pair(-1.0f, -1.0f), y);
            float da, db, ma, mb;
            d.split(da, db);
            m.split(ma, mb);
            off = fmaxf(off, fmaxf(fabsf(da), fabsf(db)));
            sum[e] = __float_as_uint(ma);
            sum[VEC > 1 ? e + 1 : 1] = __float_as_uint(mb);
        }
        if (fast && off > 0.5f - 6e-5f) {
#pragma unroll
            for (int e = 0; e < VEC; e++) {
                const int i = v * VEC + e;
                float about = __fmul_rn(x[i], c);
                if (NORM) about = __fmul_rn(about, g[i]);
                const float low = floorf(about), half = low + 0.5f;
                if (fabsf(about - half) > 1e-4f) continue;
                int code = (int)low;
                if (NORM) {
                    const double w = a.w && at + e < a.cols ? wide(__ldg(a.w + at + e)) : 0.0;
                    const double y = wide(x[i]) * rs * (w + (double)one), border = (double)half * (double)s;
                    code += y > border || (y == border && (code & 1));
                } else {
                    const float rest = __fmaf_rn(-half, s, x[i]);
                    code += rest > 0.0f || (rest == 0.0f && (code & 1));
                }
                sum[e] = (uint32_t)code;
            }
        }
        if (!fast) {  // zero rows, NaN rows, scales and factors out of range
#pragma unroll 1
            for (int e = 0; e < VEC; e++) {
                if (at + e >= a.cols) break;
                const double w = a.w ? wide(a.w[at + e]) : 0.0;
                const double y = wide(load_elem<DT>(src, at + e)) * rs * (NORM ? w + (double)one : 1.0);
                dst[at + e] = s > 0.0f ? (int8_t)__double2int_rn(y / (double)s) : 0;
            }
        } else if (VEC > 1 && at + VEC <= a.cols) {
            uint32_t word[2] = {0, 0};
#pragma unroll
            for (int w = 0; w < VEC / 4; w++)
                word[w] = __byte_perm(__byte_perm(sum[4 * w], sum[4 * w + 1], 0x0040),
                                      __byte_perm(sum[4 * w + 2], sum[4 * w + 3], 0x0040), 0x5410);
            if (VEC == 4) *(uint32_t *)(dst + at) = word[0];
            else *(uint2 *)(dst + at) = make_uint2(word[0], word[1]);
        } else {
#pragma unroll
            for (int e = 0; e < VEC; e++)
                if (at + e < a.cols) dst[at + e] = (int8_t)(sum[e] & 0xff);
        }
    }
}

// Rows too long for the registers of a CTA: read three times (from L2 after the first).
constexpr int QZ_LONG = 1024;

template <int DT>
__global__ void __launch_bounds__(QZ_LONG) quantize_long_rows_kernel(QuantArgs a) {
    __shared__ double part[2][32];
    asm volatile("griddepcontrol.launch_dependents;");
    const int t = threadIdx.x;
    const int64_t row = blockIdx.x;
    const unsigned char *src = (const unsigned char *)a.x + (size_t)row * a.x_stride * Elem<DT>::SIZE;
    int8_t *dst = a.q + (size_t)row * a.q_stride;
    double rs = 1.0, big = 0.0;
    if (a.norm) {
        double ss = 0.0;
        for (int i = t; i < a.cols; i += QZ_LONG) {
            const double v = wide(load_elem<DT>(src, i));
            ss = fma(v, v, ss);
        }
        rs = 1.0 / sqrt(row_reduce<false, QZ_LONG>(ss, part[0]) / (double)a.cols + wide(a.eps));
    }
    auto gain = [&](int i) { return a.w ? wide(a.w[i]) + (a.add_one ? 1.0 : 0.0) : 1.0; };
    for (int i = t; i < a.cols; i += QZ_LONG) {
        const double y = fabs(wide(load_elem<DT>(src, i)) * gain(i));
        big = y <= DBL_MAX ? fmax(big, y) : INFINITY;
    }
    big = row_reduce<true, QZ_LONG>(big, part[1]);
    if (!(rs <= DBL_MAX)) big = INFINITY;
    const float s = scale_of(big * rs);
    if (t == 0) a.scale[row] = s;
    for (int i = t; i < a.cols; i += QZ_LONG)
        dst[i] = s > 0.0f ? (int8_t)__double2int_rn(wide(load_elem<DT>(src, i)) * rs * gain(i) / (double)s) : 0;
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
constexpr int MM_SMEM = 216 * 1024;          // stages, with 1 KB to align them

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
    int early_b;     // a and its scales come from the kernel before, which may still run; b does not
    float softcap;
    long long fault_polls;  // test hook: the issuing thread's first wait is for something that nothing completes
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
// Test hook: a wait for a barrier that nothing completes runs out after `polls` polls.
__device__ __forceinline__ bool injected_wait(uint32_t bar, long long polls, volatile int *gave_up) {
    for (long long i = 0; i < polls; i++)
        if (mbar_try(bar, 0)) return true;
    *gave_up = 1;
    return false;
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

// tanh of both values.  Up to 1: z * (1 + z^2 Q(z^2)), Q of degree 6 fitted to tanh(z) / z by reweighted
// least squares on Chebyshev points (relative error 5e-9; evaluated in fp32, 1.8 x 2^-24).  Above:
// 1 - 2 / (e^2z + 1), whose error there is under 4 x 2^-24, for the warps that hold such a value.
__device__ __forceinline__ Pair tanh2(Pair z) {
    const Pair u = mul2(z, z);
    Pair q(-3.584515071e-04f, -3.584515071e-04f);
    q = fma2(q, u, Pair(2.301362809e-03f, 2.301362809e-03f));
    q = fma2(q, u, Pair(-7.946103811e-03f, -7.946103811e-03f));
    q = fma2(q, u, Pair(2.148665674e-02f, 2.148665674e-02f));
    q = fma2(q, u, Pair(-5.387980118e-02f, -5.387980118e-02f));
    q = fma2(q, u, Pair(1.333234459e-01f, 1.333234459e-01f));
    q = fma2(q, u, Pair(-3.333329558e-01f, -3.333329558e-01f));
    q = fma2(q, u, Pair(1.0f, 1.0f));
    return mul2(q, z);
}
__device__ __forceinline__ float tanh_above_one(float z) {
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(__fmul_rn(fabsf(z), 2.88539008177792681f)));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(__fadd_rn(e, 1.0f)));
    return copysignf(__fmaf_rn(-2.0f, r, 1.0f), z);
}

// A channel's scale over the softcap.  Above the largest number it is that number: sums of 0 stay 0, and
// others' tanh is 1.
__device__ __forceinline__ float over_cap(float sb, float cap) {
    const float q = __fdiv_rn(sb, cap);
    return fabsf(q) > FLT_MAX && fabsf(sb) <= FLT_MAX ? copysignf(FLT_MAX, q) : q;
}

// Half of a tile's 16-column groups: the warp's 32 channels, from its lanes' accumulators, scaled, capped
// and stored.
template <int DT, bool CAP>
__device__ __forceinline__ void store_tile(const MmArgs &p, uint32_t lanes, int half, int ch, int t0, const float *sa,
                               float sb) {
    for (int c = half * 16; c < p.nt; c += 32) {
        int r[16];
        __syncwarp();
        tmem_load16(lanes + c, r);
        float v[16];
        float big = 0.0f;
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
            const float4 s4 = *(const float4 *)(sa + c + j);
            Pair lo = mul2(mul2(Pair((float)r[j], (float)r[j + 1]), Pair(s4.x, s4.y)), Pair(sb, sb));
            Pair hi = mul2(mul2(Pair((float)r[j + 2], (float)r[j + 3]), Pair(s4.z, s4.w)), Pair(sb, sb));
            if (CAP) {
                float z[4];
                lo.split(z[0], z[1]);
                hi.split(z[2], z[3]);
                lo = tanh2(lo);
                hi = tanh2(hi);
                big = fmaxf(fmaxf(fabsf(z[0]), fabsf(z[1])), fmaxf(fabsf(z[2]), fabsf(z[3])));
                if (__any_sync(0xffffffffu, big > 1.0f)) {
                    float y[4];
                    lo.split(y[0], y[1]);
                    hi.split(y[2], y[3]);
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (fabsf(z[i]) > 1.0f) y[i] = tanh_above_one(z[i]);
                    lo = Pair(y[0], y[1]);
                    hi = Pair(y[2], y[3]);
                }
                lo = mul2(lo, Pair(p.softcap, p.softcap));
                hi = mul2(hi, Pair(p.softcap, p.softcap));
            }
            lo.split(v[j], v[j + 1]);
            hi.split(v[j + 2], v[j + 3]);
        }
        if (ch >= p.n) continue;
        int64_t at = (int64_t)(t0 + c) * p.ldo + ch;
        if (t0 + c + 16 <= p.m) {
#pragma unroll
            for (int j = 0; j < 16; j++, at += p.ldo) store_out<DT>(p.out, at, v[j]);
        } else {
#pragma unroll
            for (int j = 0; j < 16; j++, at += p.ldo)
                if (t0 + c + j < p.m) store_out<DT>(p.out, at, v[j]);
        }
    }
}

// Persistent, one CTA per SM.  Warp 0 copies tiles (TMA), warp 1 issues the products, warps 2 to 9
// scale and store; two accumulators, so that a tile's stores run under the next tile's products.
// With few tokens the stream of b bounds it (11 stages of 18 KB in flight on each SM); with 256, b and
// the stores together (without stores 147 of 165 us); with thousands the tensor unit (73 % busy while
// the SMs are, 86 % of the last wave of tiles filled) at the clock that the power cap leaves.  Pairs of
// CTAs on one tile (half the traffic of a from L2) were no faster, nor was asking for b in L2 ahead, nor
// a pipeline each for a and b (7 stages of b and 4 of a at 256 tokens: 167 and 168 us, at 128 tokens 111
// and 101).
template <int DT, bool CAP>
__global__ void __launch_bounds__(MM_THREADS, 1) matmul_i8_kernel(const __grid_constant__ CUtensorMap map_a,
                                                                  const __grid_constant__ CUtensorMap map_b, MmArgs p) {
    extern __shared__ unsigned char raw[];
    __shared__ __align__(8) uint64_t bars[2 * MM_MAX_STAGES + 5];
    __shared__ __align__(16) float scales[MM_EPI_WARPS][256];  // a warp's copy of its tile's token scales
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
            uint32_t step;  // k blocks so far: stage step % stages, use step / stages
            int64_t t;
            int kb, y_a, y_b;  // k block, and the tile's first token and channel
            uint32_t s;        // step % stages
            auto tile = [&] {
                y_b = (int)(t / p.token_tiles) * MM_ROWS;
                y_a = (int)(t % p.token_tiles) * p.nt;
            };
            auto begin = [&] {
                t = blockIdx.x;
                kb = 0;
                s = step = 0;
                tile();
            };
            auto advance = [&] {
                step++;
                if (++s == (uint32_t)p.stages) s = 0;
                if (++kb == kblocks) {
                    kb = 0;
                    t += gridDim.x;
                    tile();
                }
            };
            auto load_b = [&] {
                mbar_expect(full + 8 * s, stage_bytes);
                tma_load(tiles + s * stage_bytes, &map_b, kb * MM_KB, y_b, full + 8 * s);
            };
            auto load_a = [&] {
                tma_load(tiles + s * stage_bytes + MM_ROWS * MM_KB, &map_a, kb * MM_KB, y_a, full + 8 * s);
            };
            begin();
            if (p.early_b) {  // fill the pipeline with b while a is still being made
                for (; step < (uint32_t)p.stages && t < ntiles; advance()) load_b();
                const uint32_t filled = step;
                asm volatile("griddepcontrol.wait;" ::: "memory");
                for (begin(); step < filled; advance()) load_a();
            }
            for (; t < ntiles; advance()) {
                if (step >= (uint32_t)p.stages && !mbar_wait(empty + 8 * s, (step / p.stages - 1) & 1, &gave_up)) break;
                load_b();
                load_a();
            }
            // no copy may be in flight when the CTA ends, also where a wait ran out, nor a product's arrival
            const uint32_t oldest = step < (uint32_t)p.stages ? 0 : step - p.stages;
            for (uint32_t i = oldest; i < step; i++)
                if (!mbar_wait(empty + 8 * (i % p.stages), (i / p.stages) & 1, &gave_up)) break;
            volatile int alone = 0;
            for (uint32_t i = oldest; gave_up && i < step; i++)
                mbar_wait(full + 8 * (i % p.stages), (i / p.stages) & 1, &alone);
        }
        __syncwarp();
    } else if (wid == 1) {
        if (lane == 0) {
            // sums of signed 8-bit products in 32-bit integers, 128 rows by nt columns
            const uint32_t idesc = 2u << 4 | 1u << 7 | 1u << 10 | (uint32_t)(p.nt >> 3) << 17 | (MM_ROWS >> 4) << 24;
            uint32_t step = 0, it = 0;
            bool ok = !p.fault_polls || injected_wait(flushed, p.fault_polls, &gave_up);
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
        float *sa = scales[wid - 2];
        if (p.early_b) asm volatile("griddepcontrol.wait;" ::: "memory");
        uint32_t it = 0;
        for (int64_t t = blockIdx.x; t < ntiles; t += gridDim.x, it++) {
            const uint32_t acc = it & 1;
            const int ch = (int)(t / p.token_tiles) * MM_ROWS + quarter * 32 + lane;
            const int t0 = (int)(t % p.token_tiles) * p.nt;
            float sb = ch < p.n ? __ldg(p.sb + ch) : 0.0f;
            if (CAP) sb = over_cap(sb, p.softcap);
            if (it == 0 || p.token_tiles > 1) {
                __syncwarp();
                for (int i = lane; i < p.nt; i += 32) sa[i] = t0 + i < p.m ? __ldg(p.sa + t0 + i) : 0.0f;
                __syncwarp();
            }
            int ok = mbar_wait(done + 8 * acc, (it >> 1) & 1, &gave_up);
            if (!__all_sync(0xffffffffu, ok)) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            store_tile<DT, CAP>(p, tmem + acc * p.nt + ((uint32_t)quarter << 21), half, ch, t0, sa, sb);
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

// The same product for few tiles (16 x 4096 x 4096: 32 tiles on 128 CTAs take 8.8 us, on 32 CTAs
// 13.8): a cluster of CTAs per tile, each taking a part of k.  The parts' integer sums are exchanged
// through distributed shared memory (over the drained pipeline stages): every CTA adds up and stores
// 128 / cluster of the tile's channels.
template <int DT, bool CAP>
__global__ void __launch_bounds__(MM_THREADS, 1) matmul_i8_split_kernel(const __grid_constant__ CUtensorMap map_a,
                                                                        const __grid_constant__ CUtensorMap map_b,
                                                                        MmArgs p) {
    extern __shared__ unsigned char raw[];
    __shared__ __align__(8) uint64_t bars[2 * MM_MAX_STAGES + 1];
    __shared__ uint32_t tmem_base;
    __shared__ int gave_up;
    const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
    uint32_t rank, parts;
    asm("mov.u32 %0, %cluster_ctarank;" : "=r"(rank));
    asm("mov.u32 %0, %cluster_nctarank;" : "=r"(parts));
    const uint32_t pad = (1024 - (smem_addr(raw) & 1023)) & 1023, tiles = smem_addr(raw) + pad;
    const int stage_bytes = (MM_ROWS + p.nt) * MM_KB;
    const uint32_t full = smem_addr(bars), empty = full + 8 * MM_MAX_STAGES, done = full + 16 * MM_MAX_STAGES;
    const int kblocks = (p.k + MM_KB - 1) / MM_KB;
    const int k0 = (int)((int64_t)kblocks * rank / parts), n = (int)((int64_t)kblocks * (rank + 1) / parts) - k0;
    const int t = blockIdx.x / parts, y_b = t / p.token_tiles * MM_ROWS, y_a = t % p.token_tiles * p.nt;

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
        mbar_init(done, 1);
        gave_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = tmem_base;

    if (wid == 0) {
        if (lane == 0) {
            auto load_b = [&](int i) {
                const uint32_t s = i % p.stages;
                mbar_expect(full + 8 * s, stage_bytes);
                tma_load(tiles + s * stage_bytes, &map_b, (k0 + i) * MM_KB, y_b, full + 8 * s);
            };
            auto load_a = [&](int i) {
                const uint32_t s = i % p.stages;
                tma_load(tiles + s * stage_bytes + MM_ROWS * MM_KB, &map_a, (k0 + i) * MM_KB, y_a, full + 8 * s);
            };
            const int first = n < p.stages ? n : p.stages;
            int i = 0;
            for (; i < first; i++) load_b(i);
            if (p.early_b) asm volatile("griddepcontrol.wait;" ::: "memory");
            for (i = 0; i < first; i++) load_a(i);
            for (; i < n; i++) {
                if (!mbar_wait(empty + 8 * (i % p.stages), (i / p.stages - 1) & 1, &gave_up)) break;
                load_b(i);
                load_a(i);
            }
            const int oldest = i < p.stages ? 0 : i - p.stages;
            for (int j = oldest; j < i; j++)
                if (!mbar_wait(empty + 8 * (j % p.stages), (j / p.stages) & 1, &gave_up)) break;
            volatile int alone = 0;
            for (int j = oldest; gave_up && j < i; j++)
                mbar_wait(full + 8 * (j % p.stages), (j / p.stages) & 1, &alone);
        }
        __syncwarp();
    } else if (wid == 1) {
        if (lane == 0) {
            const uint32_t idesc = 2u << 4 | 1u << 7 | 1u << 10 | (uint32_t)(p.nt >> 3) << 17 | (MM_ROWS >> 4) << 24;
            if (p.fault_polls) injected_wait(done, p.fault_polls, &gave_up);
            for (int i = 0; i < n && !(p.fault_polls && gave_up); i++) {
                const uint32_t s = i % p.stages;
                if (!mbar_wait(full + 8 * s, (i / p.stages) & 1, &gave_up)) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint64_t da = operand_desc(tiles + s * stage_bytes),
                               db = operand_desc(tiles + s * stage_bytes + MM_ROWS * MM_KB);
#pragma unroll
                for (int j = 0; j < MM_KB / 32; j++) mma_i8(tmem, da + 2 * j, db + 2 * j, idesc, i > 0 || j > 0);
                mma_commit(empty + 8 * s);
            }
            mma_commit(done);
        }
        __syncwarp();
    }
    // every thread: this CTA's products are complete (bounded), then every CTA's, so that all stages are free
    volatile int alone = 0;
    if (!mbar_wait(done, 0, &alone)) gave_up = 1;
    __syncwarp();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    // channel c of the tile belongs to rank c / own; its sums lie there as [part][token][own]
    const int own = MM_ROWS / (int)parts;
    if (wid >= 2) {
        const int quarter = wid & 3, half = (wid - 2) >> 2, c = quarter * 32 + lane;
        uint32_t there;
        asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(tiles), "r"((uint32_t)(c / own)));
        there += (rank * p.nt * own + c % own) * 4;
        for (int col = half * 16; col < p.nt; col += 32) {
            int r[16];
            tmem_load16(tmem + col + ((uint32_t)quarter << 21), r);
#pragma unroll
            for (int j = 0; j < 16; j++)
                asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(there + (col + j) * own * 4), "r"(r[j]) : "memory");
        }
        __syncwarp();
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (wid == 1) {
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(p.tmem_cols));
        if (lane == 0 && gave_up && p.status) atomicOr(p.status, DLLM_ROW_ERR_TIMEOUT);
    }
    if (p.early_b) asm volatile("griddepcontrol.wait;" ::: "memory");  // the token scales
    const int *sums = (const int *)(raw + pad);
    for (int i = tid; i < own * p.nt / 2; i += MM_THREADS) {  // two tokens of a channel
        const int c = i % own, col = i / own * 2, ch = y_b + (int)rank * own + c, token = y_a + col;
        if (ch >= p.n || token >= p.m) continue;
        int a0 = 0, a1 = 0;
        for (int q = 0; q < (int)parts; q++) {
            a0 += sums[(q * p.nt + col) * own + c];
            a1 += sums[(q * p.nt + col + 1) * own + c];
        }
        float sb = __ldg(p.sb + ch), v0, v1;
        if (CAP) sb = over_cap(sb, p.softcap);
        const bool two = token + 1 < p.m;
        Pair v = mul2(mul2(Pair((float)a0, (float)a1), Pair(__ldg(p.sa + token), two ? __ldg(p.sa + token + 1) : 0.0f)),
                      Pair(sb, sb));
        if (CAP) {
            float z0, z1;
            v.split(z0, z1);
            tanh2(v).split(v0, v1);
            if (fabsf(z0) > 1.0f) v0 = tanh_above_one(z0);
            if (fabsf(z1) > 1.0f) v1 = tanh_above_one(z1);
            v = mul2(Pair(v0, v1), Pair(p.softcap, p.softcap));
        }
        v.split(v0, v1);
        store_out<DT>(p.out, (int64_t)token * p.ldo + ch, v0);
        if (two) store_out<DT>(p.out, (int64_t)(token + 1) * p.ldo + ch, v1);
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

template <auto Kernel>
dllm_status launch_product(const cudaLaunchConfig_t &cfg, const CUtensorMap &map_a, const CUtensorMap &map_b,
                           const MmArgs &p) {
    cudaError_t e = set_once<Kernel>(cudaFuncAttributeMaxDynamicSharedMemorySize, MM_SMEM);
    if (e == cudaSuccess) e = cudaLaunchKernelEx(&cfg, Kernel, map_a, map_b, p);
    return e == cudaSuccess ? DLLM_OK : cuda_failed("int8 product kernel launch", e);
}

// A warp per row up to 1024 columns; then a CTA, of 128 or 256 threads up to 8192 columns, and for the few
// rows of a decode step (fewer than SMs) of 1024, whose threads have less to do one after another.
// Both sides, in us (bf16 without norm; in brackets fp32 with norm):
//   many rows, 32 values a thread against the next larger CTA: 16384 x 1024 a warp 12.9, 128 threads 26.2;
//     16384 x 4096 128 threads 42.0, 256 84.7; 16384 x 8192 256 threads 83.7, 1024 199; 2048 x 16384 1024 threads
//     36.8, long rows 95.4 [124, 121]
//   one row of 4096: 1024 threads 2.07, 128 2.28 [4.64, 4.11]; 147 rows: 2.57, 3.61 [4.97, 4.94]
//   148 rows of 4096: 128 threads 3.37, 1024 2.48 [5.04, 4.98]; 300 rows: 3.72, 4.61 [7.92, 12.1], so the limit could lie
//     between one and two rows an SM
//   one row of 1024 or 2048: 1024 threads 2.0, 128 with 16 values 1.8 [4.5, 2.8]
template <int DT>
dllm_status quantize_typed(const QuantArgs &a, cudaStream_t stream) {
    const bool vec = (uintptr_t)a.x % 16 == 0 && (a.rows == 1 || a.x_stride * Elem<DT>::SIZE % 16 == 0);
    auto go = [&](auto kernel, int grid, int threads) {
        const cudaError_t e = launch_kernel(kernel, grid, threads, 0, stream, a);
        return e == cudaSuccess ? DLLM_OK : cuda_failed("int8 quantisation kernel launch", e);
    };
#define DLLM_QUANTIZE(TPR, E, GRID)                                                            \
    do {                                                                                       \
        const int threads = TPR == 32 ? 256 : TPR;                                             \
        if (a.norm) return vec ? go(quantize_rows_kernel<DT, TPR, E, true, true>, GRID, threads)  \
                               : go(quantize_rows_kernel<DT, TPR, E, false, true>, GRID, threads); \
        return vec ? go(quantize_rows_kernel<DT, TPR, E, true, false>, GRID, threads)          \
                   : go(quantize_rows_kernel<DT, TPR, E, false, false>, GRID, threads);        \
    } while (0)
    const int groups = (int)(((int64_t)a.rows + 7) / 8);
    const bool many = a.rows >= 148;
    if (a.cols <= 512) DLLM_QUANTIZE(32, 16, groups);
    if (a.cols <= 1024 && many) DLLM_QUANTIZE(32, 32, groups);
    if (a.cols <= 2048 && many) DLLM_QUANTIZE(128, 16, a.rows);
    if (a.cols <= 4096 && many) DLLM_QUANTIZE(128, 32, a.rows);
    if (a.cols <= 8192 && many) DLLM_QUANTIZE(256, 32, a.rows);
    if (a.cols <= 8192) DLLM_QUANTIZE(1024, 8, a.rows);
    if (a.cols <= 16384) DLLM_QUANTIZE(1024, 16, a.rows);
#undef DLLM_QUANTIZE
    return go(quantize_long_rows_kernel<DT>, a.rows, QZ_LONG);
}

}  // namespace

dllm_status launch_quantize_i8(int rows, int cols, const void *x, int64_t x_stride, int x_dtype, int norm,
                               const float *norm_w, float eps, int add_one, int8_t *q, int64_t q_stride, float *scale,
                               cudaStream_t stream) {
    if (rows == 0) return DLLM_OK;
    const QuantArgs a = {x, x_stride, q_stride, rows, cols, norm, add_one, norm_w, eps, q, scale};
    if (x_dtype == DLLM_DTYPE_F32) return quantize_typed<DLLM_DTYPE_F32>(a, stream);
    if (x_dtype == DLLM_DTYPE_BF16) return quantize_typed<DLLM_DTYPE_BF16>(a, stream);
    return quantize_typed<DLLM_DTYPE_F16>(a, stream);
}

dllm_status launch_matmul_i8(int m, int n, int k, const int8_t *a, int64_t lda, const float *sa, const int8_t *b,
                             int64_t ldb, const float *sb, float softcap, void *out, int64_t ldo, int out_dtype,
                             int32_t *status, bool early_b, cudaStream_t stream) {
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
    p.early_b = early_b;
    p.fault_polls = product_fault_polls();
    // token tiles of equal size, at most 256 (the widest instruction)
    p.token_tiles = (m + 255) / 256;
    p.nt = ((m + p.token_tiles - 1) / p.token_tiles + 15) / 16 * 16;
    const int sms = sm_count(), kblocks = (k + MM_KB - 1) / MM_KB;
    const int64_t tiles = (int64_t)((n + MM_ROWS - 1) / MM_ROWS) * p.token_tiles;
    // Few tiles: split k over a cluster of up to 8 CTAs, while the SMs suffice and a part has 4 blocks.
    // Measured with 16 tokens and k = 4096, in us with 1, 2, 4 and 8 parts: 8 tiles 13.8 11.6 8.2 6.5; 32 tiles 13.8
    // 11.8 8.8 17.6; 74 tiles 15.0 15.3 25.4 32.6.  The rule counts SMs, not the places that GPCs have for whole
    // clusters, so some sizes get a part count that runs in two rounds: 16 tiles in 8 parts 12.0 (in 4: 8.3), 36
    // tiles in 4 parts 15.5 (in 2: 11.8).  It does not look at the tokens either: with 256 of them the exchange
    // costs more than it saves at k = 1024 (32 tiles 16.5 in 2 parts, 7.8 in one) and gains at k = 14336 (25.4
    // in 4 parts, 43.7 in one).  75 to 147 tiles are not split (86 tiles 15.2, at the copy rate 7.0).
    int parts = 1;
    while (parts < 8 && tiles * parts * 2 <= sms && kblocks >= parts * 8) parts *= 2;
    p.stages = (MM_SMEM - 1024) / ((MM_ROWS + p.nt) * MM_KB);
    if (p.stages > MM_MAX_STAGES) p.stages = MM_MAX_STAGES;
    p.tmem_cols = 32;
    while (p.tmem_cols < 2 * p.nt) p.tmem_cols *= 2;
    CUtensorMap map_a, map_b;
    if (!code_map(&map_a, a, m, k, lda, p.nt) || !code_map(&map_b, b, n, k, ldb, MM_ROWS)) {
        set_last_error_message("int8 product: the driver makes no tensor map of the codes");
        return DLLM_ERR_CUDA;
    }
    cudaLaunchAttribute attr[2] = {};
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(parts > 1 ? tiles * parts : tiles < sms ? tiles : sms));
    cfg.blockDim = dim3(MM_THREADS);
    cfg.dynamicSmemBytes = MM_SMEM;
    cfg.stream = stream;
    cfg.attrs = attr;
    if (early_b) {  // launched while the kernel that makes a runs; it waits for it on the GPU
        attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (parts > 1) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
        attr[cfg.numAttrs++].val.clusterDim = {(unsigned)parts, 1, 1};
    }
    const bool cap = softcap > 0.0f;
#define DLLM_MATMUL(DT)                                                                      \
    (parts > 1 ? (cap ? launch_product<matmul_i8_split_kernel<DT, true>>(cfg, map_a, map_b, p)   \
                      : launch_product<matmul_i8_split_kernel<DT, false>>(cfg, map_a, map_b, p)) \
               : (cap ? launch_product<matmul_i8_kernel<DT, true>>(cfg, map_a, map_b, p)         \
                      : launch_product<matmul_i8_kernel<DT, false>>(cfg, map_a, map_b, p)))
    if (out_dtype == DLLM_DTYPE_F32) return DLLM_MATMUL(DLLM_DTYPE_F32);
    if (out_dtype == DLLM_DTYPE_BF16) return DLLM_MATMUL(DLLM_DTYPE_BF16);
    return DLLM_MATMUL(DLLM_DTYPE_F16);
#undef DLLM_MATMUL
}

}  // namespace dllm
