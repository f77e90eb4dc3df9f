// dllm_beam.cu -- one step of beam search: the k best continuations over beams and vocabulary
// (dllm_cuda_beam_select) and the states moved after the chosen parents (dllm_cuda_beam_reorder).
//
//   cum(b, i) = score_b + x_bi - log(sum over allowed j of exp(x_bj))
//   rank      = cum / length^alpha; order: rank desc, beam asc, logit desc, id asc
//
// Within a beam that order is the order of the logits, so a row is read once: a piece of it keeps
// its k best (logit desc, id asc) and its running maximum and exponential sum, and one CTA per
// sequence joins the pieces.
//
// Measured on B200 (GPU time of a call, several back to back):
//   64 x 8 rows of 262144 in bf16, k = 16    76 us (268 MB: 3.5 TB/s); 41 us at the measured copy rate
//   16 x 8 rows of 151936 in fp32, 2 % allowed, a quarter of the beams ended    24 us (30 MB read)
//   8 x 4 rows of 128257 in bf16    13 to 15 us;  1 x 4 rows of 32000 in fp32    9 to 12 us
//   16 x 8 rows of 151936 in fp32, k = 8: all allowed without a mask 30 us, 10 % allowed 37, 30 to 60 % 63
// What bounds the first (65 % of the issue slots taken, the special-function unit 59 % busy, DRAM 45 %):
// candidates take 13 us of it, published maxima 4, the second kernel 5; without the exponentials, but
// else whole, it is no faster, and a bare read of the rows with this layout takes 47.
// 8 x 4 rows: a piece is one tile, and a warp issues 1010 instructions for it, where a tile in the middle of a
// piece takes 361: the rest is a piece's own work (first threshold, candidates, ranking), and the second
// kernel, whose five phases depend on one another, ranks again.  1 x 4 rows: launch and dependency latency.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <float.h>
#include <math.h>

#include "dllm_internal.h"
#include "dllm_pair.cuh"

namespace dllm {
namespace {

constexpr int BS_NT = 256;
constexpr int BS_WARPS = BS_NT / 32;
constexpr int BS_U = 4;             // 16-byte vectors per thread and tile
constexpr int BS_WCAP = 512;        // candidates that a warp holds: at least k (256) and one vector of each lane
constexpr int BS_CAP = BS_WARPS * BS_WCAP;
constexpr uint32_t KEY_NINF = 0x007fffffu;  // order key of -inf

// One piece's maximum and its exponential sum, relative to sum_base(m).
struct PieceSum {
    float m;
    float pad;
    double s;
};

// Order-preserving key of a float; -0 and +0 are the same value.
__device__ __forceinline__ uint32_t okey(float x) {
    uint32_t b = __float_as_uint(x);
    if ((b << 1) == 0) b = 0;
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float okey_value(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Maximum that keeps subnormal values (the unit is built to flush them) and passes over NaN.
__device__ __forceinline__ float max_keep(float a, float b) {
    float y;
    asm("max.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}
__device__ __forceinline__ Pair exp2_approx(Pair x) {
    float a, b;
    x.split(a, b);
    return Pair(exp2_approx(a), exp2_approx(b));
}

// Exponential sums are held as sums of 2^(x * LOG2E - base(m)), m the largest x so far.  The base is
// LOG2E * m rounded to fp32, so that one fused product-and-sum forms an exponent; from 2^20 on, where
// that rounding is no longer small, it is the exact product and the exponent LOG2E * (x - m).
// log(sum of e^x) is then (log2(sum) + base) / LOG2E with this LOG2E, whose own rounding (1.3e-8 of it)
// changes the result by that much times the softmax's entropy.
constexpr float LOG2E = 1.44269504088896340736f;
constexpr float BASE_EXACT = 1048576.0f;
__device__ __forceinline__ bool beyond(float m) { return fabsf(m) >= BASE_EXACT && m > -INFINITY; }
__device__ __forceinline__ double sum_base(float m) {
    return fabsf(m) < BASE_EXACT ? (double)__fmul_rn(m, LOG2E) : (double)m * (double)LOG2E;
}
// what a sum relative to `from` is multiplied by to be one relative to `to` (>= from)
__device__ __forceinline__ double rebase(float from, float to) {
    return from == to ? 1.0 : from == -INFINITY ? 0.0 : (double)exp2_approx((float)(sum_base(from) - sum_base(to)));
}

// A candidate: (order key << 32) | ~id, so that a larger composite is (logit desc, id asc).
__device__ __forceinline__ uint64_t composite(uint32_t key, int id) { return (uint64_t)key << 32 | (uint32_t)~id; }

// A beam that offers its row's continuations: not ended, with a finite score.
__device__ __forceinline__ bool beam_live(const dllm_beam_desc &d, int64_t row) {
    if (d.finished && d.finished[row]) return false;
    return fabsf(d.scores[row]) <= FLT_MAX;
}

// Sorts buf[0, n2) descending (n2 a power of two) by `nt` threads, of which this is number `t`.
template <class Sync>
__device__ __forceinline__ void sort_desc(uint64_t *buf, int n2, int t, int nt, Sync sync) {
    for (int size = 2; size <= n2; size <<= 1)
        for (int stride = size >> 1; stride; stride >>= 1) {
            for (int i = t; i < n2 / 2; i += nt) {
                const int lo = 2 * i - (i & (stride - 1)), hi = lo + stride;
                const uint64_t a = buf[lo], b = buf[hi];
                if ((a < b) == ((lo & size) == 0)) {
                    buf[lo] = b;
                    buf[hi] = a;
                }
            }
            sync();
        }
}

// How 16 bytes hold logits.
template <int DT>
struct Vec {
    static constexpr int N = DT == DLLM_DTYPE_F32 ? 4 : 8;  // elements
    static constexpr int ESZ = DT == DLLM_DTYPE_F32 ? 4 : 2;
    static constexpr uint32_t NINF = DT == DLLM_DTYPE_F32 ? 0xff800000u : DT == DLLM_DTYPE_BF16 ? 0xff80ff80u : 0xfc00fc00u;
};

__device__ __forceinline__ uint32_t word_of(const uint4 &v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

// the two elements of word i of a 16-bit vector, or elements 2 i and 2 i + 1 of an fp32 one
template <int DT>
__device__ __forceinline__ float2 pair_of(const uint4 &v, int i) {
    if (DT == DLLM_DTYPE_F32) return make_float2(__uint_as_float(word_of(v, 2 * i)), __uint_as_float(word_of(v, 2 * i + 1)));
    const uint32_t u = word_of(v, i);
    if (DT == DLLM_DTYPE_BF16) return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
    return make_float2(__half2float(__ushort_as_half((unsigned short)(u & 0xffffu))),
                       __half2float(__ushort_as_half((unsigned short)(u >> 16))));
}

// elementwise maximum of two words of 16-bit logits
template <int DT>
__device__ __forceinline__ uint32_t max_words(uint32_t a, uint32_t b) {
    uint32_t y;
    if (DT == DLLM_DTYPE_BF16) asm("max.bf16x2 %0, %1, %2;" : "=r"(y) : "r"(a), "r"(b));
    else asm("max.f16x2 %0, %1, %2;" : "=r"(y) : "r"(a), "r"(b));
    return y;
}
// the largest element of U vectors
template <int DT, int U>
__device__ __forceinline__ float largest(const uint4 (&v)[U]) {
    if (DT == DLLM_DTYPE_F32) {
        float m = -INFINITY;
#pragma unroll
        for (int u = 0; u < U; u++)
            m = max_keep(m, max_keep(max_keep(__uint_as_float(v[u].x), __uint_as_float(v[u].y)),
                                     max_keep(__uint_as_float(v[u].z), __uint_as_float(v[u].w))));
        return m;
    }
    uint32_t m = Vec<DT>::NINF;
#pragma unroll
    for (int u = 0; u < U; u++)
        m = max_words<DT>(m, max_words<DT>(max_words<DT>(v[u].x, v[u].y), max_words<DT>(v[u].z, v[u].w)));
    const float2 p = pair_of<DT>(make_uint4(m, 0, 0, 0), 0);
    return max_keep(p.x, p.y);
}

template <int DT>
__device__ __forceinline__ uint4 ninf_vector() {
    return make_uint4(Vec<DT>::NINF, Vec<DT>::NINF, Vec<DT>::NINF, Vec<DT>::NINF);
}

// The vector of elements i0 .. of a row, of which some lie outside it: those are -inf.
template <int DT>
__device__ __noinline__ uint4 edge_vector(const unsigned char *row, int i0, int V) {
    constexpr int VEC = Vec<DT>::N;
    uint32_t x[4] = {Vec<DT>::NINF, Vec<DT>::NINF, Vec<DT>::NINF, Vec<DT>::NINF};
#pragma unroll
    for (int e = 0; e < VEC; e++) {
        if (i0 + e < 0 || e >= V - i0) continue;
        const int i = i0 + e;
        if (DT == DLLM_DTYPE_F32) x[e % 4] = ((const uint32_t *)row)[i];
        else {
            const uint32_t u = ((const unsigned short *)row)[i];
            x[e / 2] = e & 1 ? (x[e / 2] & 0xffffu) | u << 16 : (x[e / 2] & 0xffff0000u) | u;
        }
    }
    return make_uint4(x[0], x[1], x[2], x[3]);
}

// How the rows' tiles are dealt out: CTA g of `ctas` takes the tiles [g W / ctas, (g + 1) W / ctas) of all
// W = rows x per_row, so that all have the same work wherever rows begin and end.  The part of a row
// that one CTA takes is a piece; piece i of a row is that of the i-th CTA that takes some of it.
struct Split {
    int64_t all;      // W
    int ctas, per_row;
    int pieces;       // at most so many of one row
    __host__ __device__ int64_t begin(int64_t cta) const { return cta * all / ctas; }
    __host__ __device__ int cta_of(int64_t tile) const { return (int)(((tile + 1) * ctas - 1) / all); }
};

// The warps' published keys: each warp's `top` largest of its lanes' keys.  The k-th largest of them has
// k lanes' keys at or above it; 8 top >= 2 k (or all are published), so it is close to the k-th largest
// of all.  Up to 32 published keys (k <= 16) have their five lowest bits replaced by their places, so
// that all differ and one comparison with each gives a key's rank; a lower threshold only keeps more.
// A warp may publish again, higher keys, while others read: each value that k entries were seen to
// reach stays one that k lanes reach.
struct Tops {
    uint4 keys[BS_NT / 4];  // [warp][top]

    __device__ __forceinline__ static int top(int k) { return min(32, (k + 3) / 4); }
    __device__ __forceinline__ void clear() {
        if (threadIdx.x < BS_NT / 4) keys[threadIdx.x] = make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ void publish(uint32_t key, int k) {
        const int lane = threadIdx.x & 31, n = top(k);
        volatile uint32_t *mine = (volatile uint32_t *)keys + (threadIdx.x >> 5) * n;
        for (int i = 0; i < n; i++) {
            const uint32_t mx = __reduce_max_sync(0xffffffffu, key);
            const uint32_t holders = __ballot_sync(0xffffffffu, key == mx);
            if (lane == __ffs(holders) - 1) {
                mine[i] = k <= 16 ? (mx & ~31u) | (31 - ((threadIdx.x >> 5) * n + i)) : mx;
                key = 0;
            }
        }
        __syncwarp();
    }
    // the k-th largest, or 0 where none was found
    __device__ __forceinline__ uint32_t kth(int k) const {
        const int lane = threadIdx.x & 31, n = BS_WARPS * top(k);
        uint32_t found = 0;
        if (k <= 16) {
            const uint32_t v = lane < n ? ((volatile const uint32_t *)keys)[lane] : 0;
            const uint32_t at = (uint32_t)__cvta_generic_to_shared(keys);
            int above = 0;
#pragma unroll
            for (int i = 0; i < 8; i++) {  // places past the last published one hold 0
                uint4 o;
                asm volatile("ld.volatile.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                             : "=r"(o.x), "=r"(o.y), "=r"(o.z), "=r"(o.w)
                             : "r"(at + 16 * i));
                above += (o.x > v) + (o.y > v) + (o.z > v) + (o.w > v);
            }
            if (above == k - 1) found = v & ~31u;
        } else {
            volatile const uint32_t *all = (volatile const uint32_t *)keys;
            for (int at = lane; at < n; at += 32) {
                const uint32_t v = all[at];
                int above = 0, same = 0;
#pragma unroll 8
                for (int i = 0; i < n; i++) {
                    const uint32_t o = all[i];
                    above += o > v;
                    same += o == v;
                }
                if (above < k && above + same >= k) found = v;
            }
            __syncwarp();
        }
        return __reduce_max_sync(0xffffffffu, found);
    }
};

template <int DT>
__device__ __forceinline__ float load_one(const void *row, int i) {
    if (DT == DLLM_DTYPE_F32) return __ldg((const float *)row + i);
    const unsigned short u = __ldg((const unsigned short *)row + i);
    return DT == DLLM_DTYPE_BF16 ? __uint_as_float((uint32_t)u << 16) : __half2float(__ushort_as_half(u));
}

template <int DT>
__device__ __forceinline__ float load_shared(const void *elems, int i) {
    if (DT == DLLM_DTYPE_F32) return ((const float *)elems)[i];
    const unsigned short u = ((const unsigned short *)elems)[i];
    return DT == DLLM_DTYPE_BF16 ? __uint_as_float((uint32_t)u << 16) : __half2float(__ushort_as_half(u));
}

// A warp sorts its candidates, best first; the k-th.
__device__ __noinline__ uint64_t warp_sorts(uint64_t *mine, int count, int k) {
    const int lane = threadIdx.x & 31;
    for (int i = count + lane; i < BS_WCAP; i += 32) mine[i] = 0;
    __syncwarp();
    sort_desc(mine, BS_WCAP, lane, 32, [] { __syncwarp(); });
    return mine[k - 1];
}

// A CTA's shared memory for one piece of a row.
struct PieceShared {
    uint64_t buf[BS_CAP];          // [warp][BS_WCAP] candidates
    uint64_t few[BS_NT];
    Tops tops;
    uint4 held[BS_WARPS][BS_U];    // the vectors of a lane that holds a candidate
    uint32_t floor_key;
    int wcount[BS_WARPS];
    float wm[BS_WARPS];
    double ws[BS_WARPS];
};

// What a thread keeps of its piece: the running maximum and exponential sum of its elements, and its
// warp's candidates.
//
// Threshold: the k-th of the warps' published keys, of their lanes' running maxima, which are different
// elements.  While candidates are taken as they come, a warp publishes after 2^i of its tiles, and the
// first warp passes the k-th on a tile later; older values are lower, so no order between the warps is
// needed, and no barrier.  A warp whose buffer could overflow sorts it and keeps its k best: their last
// key is a threshold for all, and the warp itself then takes only what comes before the last of them.
struct Piece {
    PieceShared &sh;
    const int lane, wid, k;
    uint64_t *const mine;    // this warp's candidates
    int count = 0;           // how many they are
    uint32_t thr = KEY_NINF + 1;   // a candidate's key has to reach it
    uint64_t last = 0;             // and the candidate has to come before this one
    float m = -INFINITY;     // this thread's maximum so far
    float base = -INFINITY;  // (float)sum_base(m)
    double s = 0.0;          // its exponential sum, relative to sum_base(m)
    int tile = 0;

    __device__ __forceinline__ Piece(PieceShared &shared, int k_)
        : sh(shared), lane(threadIdx.x & 31), wid(threadIdx.x >> 5), k(k_),
          mine(shared.buf + (threadIdx.x >> 5) * BS_WCAP) {
        __syncthreads();  // the piece before is done with the shared memory
        sh.tops.clear();
        if (threadIdx.x == 0) sh.floor_key = 0;
        __syncthreads();
    }
    // keeps this warp's k best
    __device__ __forceinline__ void cut() {
        const uint64_t kth = warp_sorts(mine, count, k);
        if (count >= k) {
            count = k;
            last = kth;
            thr = max(thr, (uint32_t)(last >> 32));
            if (lane == 0) atomicMax(&sh.floor_key, (uint32_t)(last >> 32));
        }
        __syncwarp();
    }
    // the lanes' elements x, of those that have one, if they can be among the k best
    __device__ __forceinline__ void offer(bool has, float x, int id) {
        const uint32_t key = okey(x);
        const uint64_t c = composite(key, id);
        const bool take = has && x == x && key >= thr && c > last;
        const uint32_t who = __ballot_sync(0xffffffffu, take);
        if (take) mine[count + __popc(who & ((1u << lane) - 1))] = c;
        count += __popc(who);
        if (count > BS_WCAP - 32) cut();
    }
    // The maximum and the reference of the sum after a tile whose largest element is `tm`; false where some
    // lane's lies beyond the range in which sum_base is one rounded product, or did before the tile: that
    // lane's sum is relative to the exact product, of which `base` is a rounding.
    __device__ __forceinline__ bool raise(float tm) {
        const float to = max_keep(m, tm);
        const bool plain = !__any_sync(0xffffffffu, beyond(to) || beyond(m));
        if (plain) {
            if (tm > m) {
                const float b = __fmul_rn(tm, LOG2E);
                s *= (double)exp2_approx(__fsub_rn(base, b));
                base = b;
            }
        } else if (tm > m) {
            s *= rebase(m, tm);
            base = (float)sum_base(tm);
        }
        m = to;
        return plain;
    }
    __device__ __forceinline__ float plain_base() const { return m == -INFINITY ? 0.0f : base; }
    // exponent of x where raise() gave false, as x - ref and what is added to LOG2E times that
    __device__ __forceinline__ void exact_base(float *ref, float *off) const {
        *ref = m == -INFINITY ? 0.0f : m;
        *off = (float)((double)LOG2E * (double)*ref - sum_base(*ref));
    }
    // all warps, after their first tile: a threshold that k elements reach
    __device__ __forceinline__ void settle_threshold() {
        sh.tops.publish(okey(m), k);
        __syncthreads();
        thr = max(thr, sh.tops.kth(k));
    }
    // after tile number `tile` (from 1), where candidates are taken as they come: their threshold
    __device__ __forceinline__ void raise_threshold() {
        if ((tile & (tile - 1)) == 0) sh.tops.publish(okey(m), k);
        if (wid == 0 && ((tile - 1) & (tile - 2)) == 0) {  // a tile later, when the others have published too
            const uint32_t kth = sh.tops.kth(k);
            if (lane == 0) atomicMax(&sh.floor_key, kth);
        }
        thr = max(thr, *(volatile uint32_t *)&sh.floor_key);
    }
    // all warps: the piece's maximum, sum and k best
    __device__ __forceinline__ void finish(PieceSum *sum, uint64_t *out) {
        const float M_warp = okey_value(__reduce_max_sync(0xffffffffu, m == m ? okey(m) : 0xffffffffu));
        if (lane == 0) {
            sh.wm[wid] = M_warp;
            sh.wcount[wid] = count;
        }
        __syncthreads();
        float M = sh.wm[0];
        int n = 0, at = 0;
#pragma unroll
        for (int w = 0; w < BS_WARPS; w++) {
            M = max_keep(M, sh.wm[w]);
            if (w == wid) at = n;
            n += sh.wcount[w];
        }
        double S = s * rebase(m, M);
#pragma unroll
        for (int o = 16; o; o >>= 1) S += __shfl_xor_sync(0xffffffffu, S, o);
        if (lane == 0) sh.ws[wid] = S;
        if (n > BS_NT) {  // leave those that reach the last threshold
            sh.tops.publish(okey(m), k);
            __syncthreads();
            const uint64_t lowest = (uint64_t)max(sh.tops.kth(k), sh.floor_key) << 32;
            int kept = 0;
            for (int i = lane; i < (count + 31) / 32 * 32; i += 32) {  // in place: what is kept moves to the front
                const uint64_t c = i < count ? mine[i] : 0;
                const bool keep = i < count && c >= lowest;
                const uint32_t who = __ballot_sync(0xffffffffu, keep);
                if (keep) mine[kept + __popc(who & ((1u << lane) - 1))] = c;
                kept += __popc(who);
            }
            count = kept;
            if (lane == 0) sh.wcount[wid] = kept;
            __syncthreads();
            n = 0;
#pragma unroll
            for (int w = 0; w < BS_WARPS; w++) {
                if (w == wid) at = n;
                n += sh.wcount[w];
            }
        }
        const int tid = threadIdx.x;
        if (n <= BS_NT) {  // each candidate's place is the number of larger ones
            for (int i = lane; i < count; i += 32) sh.few[at + i] = mine[i];
            __syncthreads();
            for (int i0 = 0; i0 < n; i0 += BS_NT / 8) {  // eight lanes compare one with all
                const int i = i0 + tid / 8;
                const uint64_t c = sh.few[min(i, n - 1)];
                int place = 0;
#pragma unroll 4
                for (int j = tid % 8; j < n; j += 8) place += sh.few[j] > c;
#pragma unroll
                for (int o = 4; o; o >>= 1) place += __shfl_xor_sync(0xffffffffu, place, o);
                if (tid % 8 == 0 && i < n && place < k) out[place] = c;
            }
            for (int i = n + tid; i < k; i += BS_NT) out[i] = 0;
        } else {
            for (int i = count + lane; i < BS_WCAP; i += 32) mine[i] = 0;
            __syncthreads();
            sort_desc(sh.buf, BS_CAP, tid, BS_NT, [] { __syncthreads(); });
            for (int i = tid; i < k; i += BS_NT) out[i] = sh.buf[i];
        }
        if (tid == 0) {
            double total = 0.0;
#pragma unroll
            for (int w = 0; w < BS_WARPS; w++) total += sh.ws[w];
            *sum = {M, 0.0f, total};
        }
    }
};

// Pieces of rows without a mask.  A tile is BS_NT * BS_U of the row's 16-byte vectors, counted from the
// row's first byte rounded down to 16 (so any row start is served; the first and the last vector are
// read by element).  The next tile is loaded while one is worked on.
template <int DT>
__device__ __forceinline__ void dense_piece(const dllm_beam_desc &d, PieceShared &sh, int64_t row, int tile0, int ntiles,
                                            PieceSum *sum, uint64_t *out) {
    constexpr int VEC = Vec<DT>::N, TILE = BS_NT * BS_U;
    const int tid = threadIdx.x;
    const int V = d.vocab;
    const unsigned char *first = (const unsigned char *)d.logits + (size_t)row * d.row_stride * Vec<DT>::ESZ;
    const int shift = (int)((uintptr_t)first % 16 / Vec<DT>::ESZ);  // elements before the row in its first vector
    const uint4 *vecs = (const uint4 *)(first - shift * Vec<DT>::ESZ);
    const int nvec = (int)(((int64_t)V + shift + VEC - 1) / VEC), v0 = tile0 * TILE, v1 = min(v0 + ntiles * TILE, nvec);
    // vectors from here on are not wholly inside the row, or belong to the next piece
    const int v_full = min(v1, (int)(((int64_t)V + shift) / VEC));

    auto load = [&](uint4 (&x)[BS_U], int t0) {
        if (t0 + TILE <= v_full && (t0 > 0 || shift == 0)) {
#pragma unroll
            for (int u = 0; u < BS_U; u++) x[u] = __ldg(vecs + t0 + tid + u * BS_NT);
        } else {
#pragma unroll
            for (int u = 0; u < BS_U; u++) {
                const int j = t0 + tid + u * BS_NT;
                x[u] = ninf_vector<DT>();
                if (j >= v1) continue;
                if (j < v_full && (j > 0 || shift == 0)) x[u] = __ldg(vecs + j);
                else x[u] = edge_vector<DT>(first, j * VEC - shift, V);
            }
        }
    };
    uint4 x[BS_U], next[BS_U];
    load(next, v0);  // under way while the beam's state is read
    if (!beam_live(d, row)) return;
    Piece c(sh, d.k);

    auto work = [&](const uint4 (&x)[BS_U]) {
        const float tm = largest<DT, BS_U>(x);
        Pair part(0.0f, 0.0f);
        const Pair scale(LOG2E, LOG2E);
        if (c.raise(tm)) {
            const float base = c.plain_base();
            const Pair minus(-base, -base);
#pragma unroll
            for (int u = 0; u < BS_U; u++)
#pragma unroll
                for (int i = 0; i < VEC / 2; i++) {
                    const float2 xi = pair_of<DT>(x[u], i);
                    part = add2(part, exp2_approx(fma2(Pair(xi.x, xi.y), scale, minus)));
                }
        } else {
            float ref, off;
            c.exact_base(&ref, &off);
#pragma unroll 1
            for (int u = 0; u < BS_U; u++) {
                uint4 xu = x[0];
#pragma unroll
                for (int w = 1; w < BS_U; w++) xu = u == w ? x[w] : xu;
#pragma unroll
                for (int i = 0; i < VEC / 2; i++) {
                    const float2 xi = pair_of<DT>(xu, i);
                    const Pair from = add2(Pair(xi.x, xi.y), Pair(-ref, -ref));
                    part = add2(part, exp2_approx(fma2(from, scale, Pair(off, off))));
                }
            }
        }
        c.s += (double)part.sum();
        return tm;
    };
    for (int t0 = v0;;) {
#pragma unroll
        for (int u = 0; u < BS_U; u++) x[u] = next[u];
        load(next, t0 + TILE);
        const float tm = work(x);
        c.tile++;
        if (c.tile == 1) c.settle_threshold();  // with every warp's first tile
        else c.raise_threshold();
        // Lanes that hold a candidate are rare: each puts its vectors into shared memory, where the warp
        // looks at them together, an element in each lane.
        for (uint32_t who = __ballot_sync(0xffffffffu, tm >= okey_value(c.thr)); who; who &= who - 1) {
            const int holder = __ffs(who) - 1, e = c.lane % (BS_U * VEC);
            if (c.lane == holder)
#pragma unroll
                for (int u = 0; u < BS_U; u++) sh.held[c.wid][u] = x[u];
            __syncwarp();
            const float f = load_shared<DT>(sh.held[c.wid], e);
            c.offer(c.lane < BS_U * VEC, f, (t0 + e / VEC * BS_NT + c.wid * 32 + holder) * VEC - shift + e % VEC);
            __syncwarp();
        }
        t0 += TILE;
        if (t0 >= v1) break;
    }
    c.finish(sum, out);
}

// Pieces of rows with a mask.  A tile is BS_NT of the row's mask words, a warp takes 32 words (1024 ids) at
// a time, and only allowed logits are read.  Where at most a quarter of the 1024 is allowed each lane
// takes the set bits of its own word, four a round; else the warp takes four words a round, a bit of
// them each lane.  Logits are read singly, so rows may start anywhere.
template <int DT>
__device__ __forceinline__ void masked_piece(const dllm_beam_desc &d, PieceShared &sh, int64_t row, int tile0, int ntiles,
                                             PieceSum *sum, uint64_t *out) {
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
    const int V = d.vocab, words = (int)(((int64_t)V + 31) / 32), w0 = tile0 * BS_NT, w1 = min(w0 + ntiles * BS_NT, words);
    const uint32_t *mask = d.mask + row * d.mask_stride;
    const unsigned char *logits = (const unsigned char *)d.logits + (size_t)row * d.row_stride * Vec<DT>::ESZ;
    auto word_at = [&](int i) {
        if (i >= w1) return 0u;
        const uint32_t w = __ldg(mask + i);
        return i == words - 1 && (V & 31) ? w & ((1u << (V & 31)) - 1) : w;
    };
    int group = w0 + wid * 32;  // this warp's words
    uint32_t word = word_at(group + lane), next_word = word_at(group + 32 * BS_WARPS + lane);
    if (!beam_live(d, row)) return;
    Piece c(sh, d.k);

    // Four elements of a lane: element e has the id start + (places >> 8 e & 255); absent ones are -inf.
    struct Round {
        float x[4];
        int start;
        uint32_t places;
    };
    int dense_at = -1;  // word of the group that a dense group's next round starts at; -1: not dense
    bool fresh = true;
    auto fetch = [&](Round &r) {
        for (;;) {
            if (fresh) {
                fresh = false;
                dense_at = __reduce_add_sync(0xffffffffu, __popc(word)) > 256 ? 0 : -1;
            }
            if (dense_at >= 0 ? dense_at < 32 : __any_sync(0xffffffffu, word)) break;
            group += 32 * BS_WARPS;
            if (group >= w1) return false;
            word = next_word;
            next_word = word_at(group + 32 * BS_WARPS + lane);
            fresh = true;
        }
        bool has[4];
        r.places = 0;
        if (dense_at >= 0) {
            r.start = (group + dense_at) * 32 + lane;
            r.places = 0u | 32u << 8 | 64u << 16 | 96u << 24;
#pragma unroll
            for (int e = 0; e < 4; e++) has[e] = __shfl_sync(0xffffffffu, word, dense_at + e) >> lane & 1;
            dense_at += 4;
        } else {
            r.start = (group + lane) * 32;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                has[e] = word != 0;
                r.places |= (uint32_t)((__ffs(word) - 1) & 255) << (8 * e);
                word &= word - 1;
            }
        }
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int i = r.start + (int)(r.places >> (8 * e) & 255);
            r.x[e] = has[e] ? load_one<DT>(logits, i) : -INFINITY;
        }
        return true;
    };
    auto work = [&](const Round &r) {
        const float tm = max_keep(max_keep(r.x[0], r.x[1]), max_keep(r.x[2], r.x[3]));
        float part = 0.0f;
        if (c.raise(tm)) {
            const float base = c.plain_base();
#pragma unroll
            for (int e = 0; e < 4; e++) part += exp2_approx(__fmaf_rn(r.x[e], LOG2E, -base));
        } else {
            float ref, off;
            c.exact_base(&ref, &off);
#pragma unroll
            for (int e = 0; e < 4; e++) part += exp2_approx(__fmaf_rn(r.x[e] - ref, LOG2E, off));
        }
        c.s += (double)part;
        c.tile++;
        if (c.tile == 1) c.settle_threshold();  // with every warp's first round
        else c.raise_threshold();
        if (!__any_sync(0xffffffffu, tm >= okey_value(c.thr))) return;
#pragma unroll
        for (int e = 0; e < 4; e++)
            c.offer(r.x[e] >= okey_value(c.thr), r.x[e], r.start + (int)(r.places >> (8 * e) & 255));
    };
    Round a, b;
    bool more = group < w1 && fetch(a);
    if (!more) c.settle_threshold();  // no allowed id here: the warp still joins the others
    while (more) {
        more = fetch(b);
        work(a);
        if (!more) break;
        more = fetch(a);
        work(b);
    }
    c.finish(sum, out);
}

// Persistent, 4 CTAs per SM: each takes its share of the tiles, piece by piece.  (A CTA per row left
// the SMs with 4 and with 3 rows: 512 rows took as long as 592.)
template <int DT, bool MASK>
__global__ void __launch_bounds__(BS_NT, 4) beam_pieces_kernel(dllm_beam_desc d, Split split, PieceSum *sums,
                                                               uint64_t *cands) {
    __shared__ PieceShared sh;
    asm volatile("griddepcontrol.launch_dependents;");
    int64_t at = split.begin(blockIdx.x);
    const int64_t end = split.begin(blockIdx.x + 1);
    while (at < end) {
        const int64_t row = at / split.per_row;
        const int tile = (int)(at - row * split.per_row), n = (int)min((int64_t)(split.per_row - tile), end - at);
        const int64_t piece = row * split.pieces + ((int)blockIdx.x - split.cta_of(row * split.per_row));
        if (MASK) masked_piece<DT>(d, sh, row, tile, n, sums + piece, cands + piece * d.k);
        else dense_piece<DT>(d, sh, row, tile, n, sums + piece, cands + piece * d.k);
        at += n;
    }
}


struct Best {
    double rank;
    int beam;
    uint64_t comp;
};
// Order-preserving key of a double.
__device__ __forceinline__ uint64_t okey64(double x) {
    const int64_t b = __double_as_longlong(x + 0.0);
    return (uint64_t)b ^ ((uint64_t)(b >> 63) | 0x8000000000000000ull);
}
// whether a comes before b in the operator's order
__device__ __forceinline__ bool before(const Best &a, const Best &b) {
    if (a.rank != b.rank) return a.rank > b.rank;
    if (a.beam != b.beam) return a.beam < b.beam;
    return a.comp > b.comp;
}

// One CTA per sequence (about 5 us, most of it the latency of its five dependent phases): the beams'
// log-sum-exps from their pieces, then the k best of the pieces' candidates.  The same threshold as in a piece (over the threads' best ranks, rounded down to
// fp32, which keeps their order) leaves a few; each one's place is the number that comes before
// it.  Where more are left than fit, the threshold is raised to the highest that k candidates
// reach; where that still leaves too many (equal ranks), k rounds take the best candidate that
// comes after the one taken last.
constexpr int BM_LEFT = 512;
constexpr int BM_HELD = 4;  // candidates that a thread keeps in registers

__global__ void __launch_bounds__(BS_NT) beam_merge_kernel(dllm_beam_desc d, const PieceSum *sums,
                                                           const uint64_t *cands, Split split) {
    __shared__ int npieces[DLLM_BEAM_MAX];
    // log-sum-exp of a row: its maximum, and what is added to that (the sum of both would lose it where
    // logits are huge)
    __shared__ float row_max[DLLM_BEAM_MAX];
    __shared__ double log_sum[DLLM_BEAM_MAX], divisor[DLLM_BEAM_MAX], inverse[DLLM_BEAM_MAX];
    __shared__ float score_in[DLLM_BEAM_MAX];  // copies, so that the outputs may lie over the inputs
    __shared__ int length_in[DLLM_BEAM_MAX];
    __shared__ int live[DLLM_BEAM_MAX];  // 0 nothing to offer, 1 its row's continuations, 2 ended
    __shared__ Best wbest[BS_WARPS];
    __shared__ uint64_t left_key[BM_LEFT], left_comp[BM_LEFT];
    __shared__ int left_beam[BM_LEFT];
    __shared__ float left_score[BM_LEFT];
    __shared__ Tops tops;
    __shared__ int wnumber[BS_WARPS];
    __shared__ int nleft;
    const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
    const int K = d.beams, k = d.k;
    const int64_t item = blockIdx.x;
    const bool by_length = d.length_penalty != 0.0f && d.lengths;
    if (tid == 0) nleft = 0;
    tops.clear();
    // what does not come from the pieces is read while they run
    for (int b = tid; b < K; b += BS_NT) {
        const int64_t row = item * K + b;
        const float sc = d.scores[row];
        const bool ended = d.finished && d.finished[row];
        const int len_in = d.lengths ? d.lengths[row] : 0;
        const double len = fmax((double)len_in + (ended ? 0.0 : 1.0), 1.0);
        npieces[b] = split.cta_of((row + 1) * split.per_row - 1) - split.cta_of(row * split.per_row) + 1;
        length_in[b] = len_in;
        score_in[b] = sc;
        // L^alpha, kept within 1e-200 and 1e200, so that ranks stay finite; L itself where alpha is 1
        divisor[b] = !by_length                   ? 1.0
                     : d.length_penalty == 1.0f ? len
                                                : fmin(fmax(pow(len, (double)d.length_penalty), 1e-200), 1e200);
        inverse[b] = 1.0 / divisor[b];
        live[b] = !(sc >= -FLT_MAX && sc <= FLT_MAX) ? 0 : ended ? 2 : 1;
    }
    __syncthreads();
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int lists = split.pieces, per_beam = lists * k, N = K * per_beam;
    const uint64_t *mine = cands + item * N;
    // The warps take the pieces' lists in turn, so that the best are spread over them.  Candidate number q
    // of a warp is position q % k of its list q / k.
    const int warp_n = ((K * lists - wid + BS_WARPS - 1) / BS_WARPS) * k;
    auto number = [&](int q) { return q < warp_n ? ((q / k) * BS_WARPS + wid) * k + q % k : N; };
    auto comp_at = [&](int e, int b) {  // a beam that offers none, or a piece that is not there, has none
        return live[b] == 1 && e / k - b * lists < npieces[b] ? mine[e] : 0;
    };
    uint64_t held[BM_HELD];  // this thread's first candidates
    int at_e[BM_HELD];
#pragma unroll
    for (int i = 0; i < BM_HELD; i++) {
        const int e = at_e[i] = number(lane + 32 * i);
        held[i] = e < N ? comp_at(e, e / per_beam) : 0;
    }
    for (int b = wid; b < K; b += BS_WARPS) {
        const int64_t row = item * K + b;
        int st = 0, kind = live[b];
        float M = -INFINITY;
        double l = 0.0;
        if (kind == 0 && !(score_in[b] < 0.0f)) st = DLLM_ROW_ERR_NONFINITE;  // NaN or +inf
        if (kind == 1) {
            double S = 0.0;
            const PieceSum *mysums = sums + row * lists;
            if (npieces[b] <= 32) {
                const PieceSum p = lane < npieces[b] ? mysums[lane] : PieceSum{-INFINITY, 0.0f, 0.0};
                M = p.m;
#pragma unroll
                for (int o = 16; o; o >>= 1) M = max_keep(M, __shfl_xor_sync(0xffffffffu, M, o));
                S = p.s * rebase(p.m, M);
            } else {
                for (int c = lane; c < npieces[b]; c += 32) M = max_keep(M, mysums[c].m);
#pragma unroll
                for (int o = 16; o; o >>= 1) M = max_keep(M, __shfl_xor_sync(0xffffffffu, M, o));
                for (int c = lane; c < npieces[b]; c += 32) S += mysums[c].s * rebase(mysums[c].m, M);
            }
#pragma unroll
            for (int o = 16; o; o >>= 1) S += __shfl_xor_sync(0xffffffffu, S, o);
            if (S != S || M == INFINITY) {
                st = DLLM_ROW_ERR_NONFINITE;
                kind = 0;
            } else if (M > -INFINITY) l = (log2(S) + (sum_base(M) - wide(M) * (double)LOG2E)) * (1.0 / (double)LOG2E);
            else kind = 0;
        }
        __syncwarp();
        if (lane == 0) {
            row_max[b] = M;
            log_sum[b] = l;
            live[b] = kind;
            if (d.status) d.status[row] = st;
        }
    }
    __syncthreads();
    auto log_prob = [&](int b, uint64_t comp) {
        return (wide(okey_value((uint32_t)(comp >> 32))) - wide(row_max[b])) - log_sum[b];
    };
    // candidate e: position e % k of a piece's list; an ended beam offers its first position only
    auto candidate_of = [&](int e, int b, uint64_t comp, Best *c) {
        double cum = wide(score_in[b]);
        if (live[b] == 0) return false;
        if (live[b] == 2) {
            if (e != b * per_beam) return false;
            comp = composite(0, d.eos);
        } else {
            if (!comp) return false;
            cum += log_prob(b, comp);
        }
        // cum / divisor, correctly rounded (Markstein's step on the product by the rounded reciprocal): equal
        // ranks go to the lowest beam
        const double rank = cum * inverse[b];
        *c = {fma(fma(-rank, divisor[b], cum), inverse[b], rank), b, comp};
        return true;
    };
    auto candidate = [&](int e, Best *c) {
        const int b = e / per_beam;
        return candidate_of(e, b, comp_at(e, b), c);
    };
    auto score_of = [&](int b, uint64_t comp) {
        return narrow(live[b] == 1 ? wide(score_in[b]) + log_prob(b, comp) : wide(score_in[b]));
    };
    auto emit = [&](int place, const Best &c, float score, bool none) {
        d.out_score[item * k + place] = score;
        d.out_parent[item * k + place] = none ? -1 : c.beam;
        const int32_t token = none ? -1 : (int32_t)~(uint32_t)c.comp;
        const bool ended = !none && live[c.beam] == 2;
        d.out_token[item * k + place] = token;
        if (d.out_finished) d.out_finished[item * k + place] = ended || (!none && token == d.eos);
        if (d.out_lengths) d.out_lengths[item * k + place] = none ? 0 : length_in[c.beam] + (ended ? 0 : 1);
    };
    auto keep = [&](int at, const Best &c) {
        left_key[at] = okey64(c.rank);
        left_beam[at] = c.beam;
        left_comp[at] = c.comp;
        left_score[at] = score_of(c.beam, c.comp);
    };
    uint32_t mx = 0, key[BM_HELD];
#pragma unroll
    for (int i = 0; i < BM_HELD; i++) {
        const int e = at_e[i];
        Best c;
        key[i] = e < N && candidate_of(e, e / per_beam, held[i], &c) ? okey(narrow_down(c.rank)) : 0;
        mx = max(mx, key[i]);
    }
    for (int q = lane + 32 * BM_HELD; q < warp_n; q += 32) {
        Best c;
        if (candidate(number(q), &c)) mx = max(mx, okey(narrow_down(c.rank)));
    }
    tops.publish(mx, k);
    __syncthreads();
    const uint32_t lo = tops.kth(k);
#pragma unroll
    for (int i = 0; i < BM_HELD; i++) {
        if (key[i] == 0 || key[i] < lo) continue;
        const int e = at_e[i], at = atomicAdd(&nleft, 1);
        Best c;
        if (at < BM_LEFT && candidate_of(e, e / per_beam, held[i], &c)) keep(at, c);
    }
    for (int q = lane + 32 * BM_HELD; q < warp_n; q += 32) {
        Best c;
        if (!candidate(number(q), &c) || okey(narrow_down(c.rank)) < lo) continue;
        const int at = atomicAdd(&nleft, 1);
        if (at < BM_LEFT) keep(at, c);
    }
    __syncthreads();
    int n = nleft;
    if (n > BM_LEFT) {  // the largest threshold that k candidates reach, by bisection of its key
        uint32_t reached = lo, above = 0xffffffffu;
        while (above - reached > 1) {
            const uint32_t mid = reached + (above - reached) / 2;
            int c_mid = 0;
            for (int e = tid; e < N; e += BS_NT) {
                Best c;
                c_mid += candidate(e, &c) && okey(narrow_down(c.rank)) >= mid;
            }
            c_mid = __reduce_add_sync(0xffffffffu, c_mid);
            __syncthreads();
            if (lane == 0) wnumber[wid] = c_mid;
            __syncthreads();
            c_mid = 0;
#pragma unroll
            for (int w = 0; w < BS_WARPS; w++) c_mid += wnumber[w];
            if (c_mid >= k) reached = mid;
            else above = mid;
        }
        __syncthreads();
        if (tid == 0) nleft = 0;
        __syncthreads();
        for (int e = tid; e < N; e += BS_NT) {
            Best c;
            if (!candidate(e, &c) || okey(narrow_down(c.rank)) < reached) continue;
            const int at = atomicAdd(&nleft, 1);
            if (at < BM_LEFT) keep(at, c);
        }
        __syncthreads();
        n = nleft;
    }
    if (n <= BM_LEFT) {
        for (int i0 = 0; i0 < n; i0 += BS_NT / 8) {  // eight lanes compare one with all
            const int i = i0 + tid / 8;
            const int mine_at = i < n ? i : 0, beam = left_beam[mine_at];
            const uint64_t key = left_key[mine_at], comp = left_comp[mine_at];
            int place = 0;
#pragma unroll 2
            for (int j = tid % 8; j < n; j += 8) {  // no branches: equal ranks are common in 16-bit logits
                const uint64_t other = left_key[j], other_comp = left_comp[j];
                const int other_beam = left_beam[j];
                const bool earlier = (other_beam < beam) | ((other_beam == beam) & (other_comp > comp));
                place += (other > key) | ((other == key) & earlier);
            }
#pragma unroll
            for (int o = 4; o; o >>= 1) place += __shfl_xor_sync(0xffffffffu, place, o);
            if (tid % 8 || i >= n) continue;
            if (place < k) emit(place, Best{0.0, beam, comp}, left_score[i], false);
        }
        for (int i = n + tid; i < k; i += BS_NT) emit(i, Best{}, -INFINITY, true);
        return;
    }
    Best last = {INFINITY, -1, 0};
    for (int r = 0; r < k; r++) {
        Best best = {-INFINITY, 1 << 30, 0};
        for (int e = tid; e < N; e += BS_NT) {
            Best c;
            if (candidate(e, &c) && before(last, c) && before(c, best)) best = c;
        }
        for (int o = 16; o; o >>= 1) {
            Best c;
            c.rank = __shfl_xor_sync(0xffffffffu, best.rank, o);
            c.beam = __shfl_xor_sync(0xffffffffu, best.beam, o);
            c.comp = __shfl_xor_sync(0xffffffffu, best.comp, o);
            if (before(c, best)) best = c;
        }
        if (lane == 0) wbest[wid] = best;
        __syncthreads();
        best = wbest[0];
        for (int w = 1; w < BS_WARPS; w++)
            if (before(wbest[w], best)) best = wbest[w];
        __syncthreads();
        if (tid == 0) emit(r, best, score_of(best.beam, best.comp), false);  // more candidates than BM_LEFT >= k: there is one
        last = best;
    }
}

// A CTA for every tile, at most as many as fit on the GPU at once.
Split beam_split(const dllm_beam_desc *d) {
    const int vec = d->dtype == DLLM_DTYPE_F32 ? 4 : 8;
    Split s;
    // rows begin anywhere in their first vector
    if (d->mask) s.per_row = (int)((((int64_t)d->vocab + 31) / 32 + BS_NT - 1) / BS_NT);
    else s.per_row = (int)((((int64_t)d->vocab + 2 * vec - 2) / vec + BS_NT * BS_U - 1) / (BS_NT * BS_U));
    s.all = (int64_t)d->batch * d->beams * s.per_row;
    const int64_t room = (int64_t)sm_count() * 4;
    s.ctas = (int)(s.all < room ? s.all : room);
    const int64_t share = s.all / s.ctas;  // tiles of a CTA, at least
    const int64_t most = (s.per_row + share - 2) / share + 1;
    s.pieces = (int)(most < s.per_row ? most : s.per_row);
    return s;
}

// ----------------------------------------------------------------------------------------
// states after their parents, in place

constexpr int RO_NT = 256;
constexpr int RO_TENSORS = 64;  // pointers of one launch

struct ReorderArgs {
    unsigned char *tensors[RO_TENSORS];
    const int32_t *parent;
    int batch, beams, segs;
    int slices;                           // column ranges of one run
    int64_t row_stride, seg_stride, run;  // bytes
};

// 16 caches of 64 rows, 5 of 8 beams moved: 384 us for 2.3 GB (6.0 TB/s, 0.92 of the measured copy rate), 390 to
// 400 when calls follow one another for seconds; bound by HBM.  Rows that start on 4 bytes only: a quarter of
// that size 252 us (115 on 16 bytes); on 2 or 1 bytes, moved byte by byte, 905.  Runs of 256 bytes, 64 x 1024 of
// them in 4 states: 87 us (13 at the copy rate), 16 threads of a CTA with work.  A CTA owns one column range (one vector per thread) of one segment for all beams of a sequence:
// every thread first copies the vectors that others need into its own shared-memory column, then
// writes them out, so no second buffer is needed and beams that stay are neither read nor written.
template <int VB>
__global__ void __launch_bounds__(RO_NT) beam_reorder_kernel(ReorderArgs a) {
    extern __shared__ __align__(16) unsigned char stage[];  // [beams][blockDim.x][VB]
    __shared__ int from[DLLM_BEAM_MAX];    // source of a moved beam, -1 for one that stays
    __shared__ int needed[DLLM_BEAM_MAX];
    const int tid = threadIdx.x, K = a.beams;
    unsigned at = blockIdx.x;
    const int slice = at % a.slices;
    at /= a.slices;
    const int seg = at % a.segs;
    at /= a.segs;
    const int64_t item = at % a.batch;
    const int tensor = at / a.batch;
    for (int j = tid; j < K; j += blockDim.x) needed[j] = 0;
    __syncthreads();
    for (int j = tid; j < K; j += blockDim.x) {
        const int p = a.parent[item * K + j];
        const bool moved = p >= 0 && p < K && p != j;
        from[j] = moved ? p : -1;
        if (moved) needed[p] = 1;
    }
    __syncthreads();
    const int64_t col = ((int64_t)slice * blockDim.x + tid) * VB;
    if (col >= a.run) return;
    const int tail = a.run - col < VB ? (int)(a.run - col) : 0;  // bytes of a run's last, shorter vector
    unsigned char *base = a.tensors[tensor] + item * K * a.row_stride + seg * a.seg_stride + col;
    unsigned char *mine = stage + (size_t)tid * VB;
    const size_t pitch = (size_t)blockDim.x * VB;
    for (int p = 0; p < K; p++) {
        if (!needed[p]) continue;
        if (VB == 1) mine[p * pitch] = base[p * a.row_stride];
        else if (tail) for (int i = 0; i < tail; i++) mine[p * pitch + i] = base[p * a.row_stride + i];
        else {
            const uint32_t to = (uint32_t)__cvta_generic_to_shared(mine + p * pitch);
            asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(to), "l"(base + p * a.row_stride), "n"(VB < 4 ? 4 : VB)
                         : "memory");
        }
    }
    if (VB > 1) asm volatile("cp.async.wait_all;" ::: "memory");
    for (int j = 0; j < K; j++) {
        if (from[j] < 0) continue;
        const unsigned char *src = mine + from[j] * pitch;
        unsigned char *dst = base + j * a.row_stride;
        if (VB > 1 && tail) for (int i = 0; i < tail; i++) dst[i] = src[i];
        else if (VB == 16) *(uint4 *)dst = *(const uint4 *)src;
        else if (VB == 4) *(uint32_t *)dst = *(const uint32_t *)src;
        else *dst = *src;
    }
}

}  // namespace

template <auto Kernel>
static cudaError_t launch_pieces(const dllm_beam_desc &d, const Split &split, PieceSum *sums, uint64_t *cands,
                                 cudaStream_t stream) {
    // room for four CTAs' buffers on an SM
    const cudaError_t e = set_once<Kernel>(cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    return e == cudaSuccess ? launch_kernel(Kernel, split.ctas, BS_NT, 0, stream, d, split, sums, cands) : e;
}

static size_t sums_bytes(int64_t pieces) { return ((size_t)pieces * sizeof(PieceSum) + 255) / 256 * 256; }

size_t beam_ws_bytes(const dllm_beam_desc *d) {
    const int64_t n = (int64_t)d->batch * d->beams * beam_split(d).pieces;
    return sums_bytes(n) + (size_t)n * d->k * sizeof(uint64_t);
}

dllm_status launch_beam_select(const dllm_beam_desc *d, void *ws, cudaStream_t stream) {
    const Split split = beam_split(d);
    PieceSum *sums = (PieceSum *)ws;
    uint64_t *cands = (uint64_t *)((unsigned char *)ws + sums_bytes((int64_t)d->batch * d->beams * split.pieces));
#define DLLM_PIECES(DT)                                                                       \
    (d->mask ? launch_pieces<beam_pieces_kernel<DT, true>>(*d, split, sums, cands, stream)    \
             : launch_pieces<beam_pieces_kernel<DT, false>>(*d, split, sums, cands, stream))
    cudaError_t e = d->dtype == DLLM_DTYPE_F32    ? DLLM_PIECES(DLLM_DTYPE_F32)
                    : d->dtype == DLLM_DTYPE_BF16 ? DLLM_PIECES(DLLM_DTYPE_BF16)
                                                  : DLLM_PIECES(DLLM_DTYPE_F16);
#undef DLLM_PIECES
    if (e != cudaSuccess) return cuda_failed("beam selection kernel launch", e);
    // launched while the pieces run; it waits for them on the GPU
    cudaLaunchAttribute attr = {};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(d->batch);
    cfg.blockDim = dim3(BS_NT);
    cfg.stream = stream;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, beam_merge_kernel, *d, (const PieceSum *)sums, (const uint64_t *)cands, split);
    return e == cudaSuccess ? DLLM_OK : cuda_failed("beam selection kernel launch", e);
}

dllm_status launch_beam_reorder(int batch, int beams, const int32_t *parent, int ntensors, void *const *tensors,
                                int64_t row_stride, int segs, int64_t seg_stride, int64_t run, cudaStream_t stream) {
    // the widest vectors that every run's start allows
    uintptr_t bits = (uintptr_t)row_stride | (segs > 1 ? (uintptr_t)seg_stride : 0);
    for (int i = 0; i < ntensors; i++) bits |= (uintptr_t)tensors[i];
    const int vb = bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : 1;
    ReorderArgs a = {};
    a.parent = parent;
    a.batch = batch;
    a.beams = beams;
    a.segs = segs;
    a.row_stride = row_stride;
    a.seg_stride = seg_stride;
    a.run = run;
    const int nt = beams <= 32 ? RO_NT : 64;
    const int64_t slices = ((run + vb - 1) / vb + nt - 1) / nt, per_tensor = slices * segs * batch;
    if (slices > INT32_MAX || slices * segs > INT32_MAX || per_tensor > INT32_MAX) return DLLM_ERR_UNSUPPORTED;
    a.slices = (int)slices;
    const int group = (int)(INT32_MAX / per_tensor < RO_TENSORS ? INT32_MAX / per_tensor : RO_TENSORS);
    const size_t smem = (size_t)beams * nt * vb;
    auto launch = [&](auto kernel) {
        for (int t = 0; t < ntensors; t += group) {
            const int n = ntensors - t < group ? ntensors - t : group;
            for (int i = 0; i < n; i++) a.tensors[i] = (unsigned char *)tensors[t + i];
            const cudaError_t e = launch_kernel(kernel, (unsigned)(per_tensor * n), nt, smem, stream, a);
            if (e != cudaSuccess) return cuda_failed("beam reorder kernel launch", e);
        }
        return DLLM_OK;
    };
    const cudaFuncAttribute size = cudaFuncAttributeMaxDynamicSharedMemorySize;
    cudaError_t e = vb == 16  ? set_once<beam_reorder_kernel<16>>(size, 131072)
                    : vb == 4 ? set_once<beam_reorder_kernel<4>>(size, 131072)
                              : set_once<beam_reorder_kernel<1>>(size, 131072);
    if (e != cudaSuccess) return cuda_failed("beam reorder kernel set-up", e);
    return vb == 16 ? launch(beam_reorder_kernel<16>) : vb == 4 ? launch(beam_reorder_kernel<4>) : launch(beam_reorder_kernel<1>);
}

}  // namespace dllm
