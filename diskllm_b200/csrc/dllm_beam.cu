// dllm_beam.cu -- one step of beam search: the k best continuations over beams and vocabulary
// (dllm_cuda_beam_select) and the states moved after the chosen parents (dllm_cuda_beam_reorder).
//
//   cum(b, i) = score_b + x_bi - log(sum over allowed j of exp(x_bj))
//   rank      = cum / length^alpha; order: rank desc, beam asc, logit desc, id asc
//
// Within a beam that order is the order of the logits, so a row is read once: a chunk of it keeps
// its k best (logit desc, id asc) and its running maximum and exponential sum, and one CTA per
// sequence joins the chunks.
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

// One chunk's maximum and its exponential sum, relative to sum_base(m).
struct ChunkSum {
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

// The j-th largest of a warp's 32 keys (j from 1), in every lane.
__device__ __forceinline__ uint32_t warp_jth(uint32_t key, int j) {
    uint32_t mx = __reduce_max_sync(0xffffffffu, key);
    for (int i = 1; i < j; i++) {
        const uint32_t holders = __ballot_sync(0xffffffffu, key == mx);
        if ((threadIdx.x & 31) == __ffs(holders) - 1) key = 0;
        mx = __reduce_max_sync(0xffffffffu, key);
    }
    return mx;
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

// Which elements of U vectors are at or above `least`, as bits: element e of fp32 vectors at bit e;
// of 16-bit ones, the lower element of word w at bit w and the upper one at bit 16 + w.  `least` is
// rounded down to the type, so a few more may be marked.
template <int DT, int U>
__device__ __forceinline__ uint32_t reaching(const uint4 (&v)[U], float least) {
    uint32_t take = 0;
    if (DT == DLLM_DTYPE_F32) {
#pragma unroll
        for (int e = 0; e < 4 * U; e++) take |= (uint32_t)(__uint_as_float(word_of(v[e / 4], e % 4)) >= least) << e;
        return take;
    }
    uint32_t two;  // -inf is never marked
    if (DT == DLLM_DTYPE_BF16) two = __bfloat16_as_ushort(__float2bfloat16_rd(fmaxf(least, -3.38953139e38f)));
    else two = __half_as_ushort(__float2half_rd(fmaxf(least, -65504.0f)));
    two |= two << 16;
#pragma unroll
    for (int w = 0; w < 4 * U; w++) {
        uint32_t ge;
        if (DT == DLLM_DTYPE_BF16) asm("set.ge.u32.bf16x2 %0, %1, %2;" : "=r"(ge) : "r"(word_of(v[w / 4], w % 4)), "r"(two));
        else asm("set.ge.u32.f16x2 %0, %1, %2;" : "=r"(ge) : "r"(word_of(v[w / 4], w % 4)), "r"(two));
        take |= ge & (0x10001u << w);
    }
    return take;
}
// the element at a bit of reaching(), and its number in the vectors
template <int DT, int U>
__device__ __forceinline__ float element_of(const uint4 (&v)[U], int bit, int *e) {
    const int w = bit & 15;
    uint32_t word = word_of(v[0], 0);
#pragma unroll
    for (int i = 1; i < 4 * U; i++) word = w == i ? word_of(v[i / 4], i % 4) : word;
    if (DT == DLLM_DTYPE_F32) {
        *e = w;
        return __uint_as_float(word);
    }
    const float2 p = pair_of<DT>(make_uint4(word, 0, 0, 0), 0);
    *e = 2 * w + (bit >> 4);
    return bit & 16 ? p.y : p.x;
}

template <int DT>
__device__ __forceinline__ uint4 ninf_vector() {
    return make_uint4(Vec<DT>::NINF, Vec<DT>::NINF, Vec<DT>::NINF, Vec<DT>::NINF);
}

// The vector of elements i0 .. of a row, of which some lie outside it: those and masked ones are -inf.
template <int DT>
__device__ __noinline__ uint4 edge_vector(const unsigned char *row, const uint32_t *mask, int i0, int V) {
    constexpr int VEC = Vec<DT>::N;
    uint32_t x[4] = {Vec<DT>::NINF, Vec<DT>::NINF, Vec<DT>::NINF, Vec<DT>::NINF};
#pragma unroll
    for (int e = 0; e < VEC; e++) {
        if (i0 + e < 0 || e >= V - i0) continue;
        const int i = i0 + e;
        if (mask && !(mask[i >> 5] >> (i & 31) & 1)) continue;
        if (DT == DLLM_DTYPE_F32) x[e % 4] = ((const uint32_t *)row)[i];
        else {
            const uint32_t u = ((const unsigned short *)row)[i];
            x[e / 2] = e & 1 ? (x[e / 2] & 0xffffu) | u << 16 : (x[e / 2] & 0xffff0000u) | u;
        }
    }
    return make_uint4(x[0], x[1], x[2], x[3]);
}

// Grid rows x chunks.  A chunk is a range of the row's 16-byte vectors, counted from the row's
// first byte rounded down to 16 (so any row start is served; the first and the last vector are
// read by element).  Per tile a thread updates its running maximum and exponential sum, and a warp
// that holds an element at or above the threshold appends such elements to its own buffer; no
// barrier is needed between tiles.
//
// Threshold: each warp publishes the `top` largest of its lanes' running maxima, which are different
// elements; the k-th largest of what the 8 warps have published has k elements at or above it
// (8 top >= 2 k, so it is close to the k-th largest of all lanes' maxima).  A warp publishes after
// 1, 2, 3, 5, 9, ... tiles, and the first warp then passes the k-th on; older values are lower, so no
// order between the warps is needed.  A warp whose
// buffer could overflow sorts it and keeps its k best: their last key is a threshold for all, and
// what the warp meets later, with larger ids, has to be strictly above it.
template <int DT, bool MASK>
__global__ void __launch_bounds__(BS_NT, 4) beam_chunk_kernel(dllm_beam_desc d, int chunks, ChunkSum *sums,
                                                              uint64_t *cands) {
    constexpr int VEC = Vec<DT>::N;
    __shared__ uint64_t buf[BS_CAP];
    __shared__ uint64_t few[BS_NT];
    __shared__ volatile uint32_t tops[BS_NT];  // [warp][top]
    __shared__ uint32_t floor_key;
    __shared__ float wm[BS_WARPS];
    __shared__ double ws[BS_WARPS];
    __shared__ int wcount[BS_WARPS];
    asm volatile("griddepcontrol.launch_dependents;");
    const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
    const int64_t row = blockIdx.x / chunks;
    const int part_no = blockIdx.x % chunks;
    const int V = d.vocab, k = d.k, top = min(32, (k + 3) / 4);
    const unsigned char *first = (const unsigned char *)d.logits + (size_t)row * d.row_stride * Vec<DT>::ESZ;
    const int shift = (int)((uintptr_t)first % 16 / Vec<DT>::ESZ);  // elements before the row in its first vector
    const uint4 *vecs = (const uint4 *)(first - shift * Vec<DT>::ESZ);
    const uint32_t *mrow = MASK ? d.mask + row * d.mask_stride : nullptr;
    const int nvec = (int)(((int64_t)V + shift + VEC - 1) / VEC), per = (nvec + chunks - 1) / chunks;
    const int v0 = per * part_no, v1 = min(v0 + per, nvec);
    // vectors from here on are not wholly inside the row, or belong to the next chunk
    const int v_full = min(v1, (int)(((int64_t)V + shift) / VEC));

    // Vector j; masked elements and those outside the row are -inf.  A vector that is wholly masked
    // is not read.
    auto load = [&](int j) {
        if (j >= v1) return ninf_vector<DT>();
        const int i0 = j * VEC - shift;
        if (i0 < 0 || i0 > V - VEC) return edge_vector<DT>(first, mrow, i0, V);
        if (!MASK) return __ldg(vecs + j);
        const int w = i0 >> 5, o = i0 & 31;
        const uint32_t lo = __ldg(mrow + w), hi = o + VEC > 32 ? __ldg(mrow + w + 1) : 0;
        const uint32_t bits = __funnelshift_r(lo, hi, o) & ((1u << VEC) - 1);
        uint4 v = ninf_vector<DT>();
        if (bits) v = __ldg(vecs + j);
        uint32_t x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            uint32_t keep;
            if (DT == DLLM_DTYPE_F32) keep = 0u - (bits >> i & 1);
            else {
                const uint32_t two = bits >> (2 * i);
                keep = ((two | two << 15) & 0x10001u) * 0xffffu;
            }
            x[i] = (x[i] & keep) | (Vec<DT>::NINF & ~keep);
        }
        return make_uint4(x[0], x[1], x[2], x[3]);
    };
    uint4 next[BS_U];  // the next tile
    auto load_tile = [&](int t0) {
        if (!MASK && t0 + BS_U * BS_NT <= v_full && (t0 > 0 || shift == 0)) {
#pragma unroll
            for (int u = 0; u < BS_U; u++) next[u] = __ldg(vecs + t0 + tid + u * BS_NT);
        } else {
#pragma unroll
            for (int u = 0; u < BS_U; u++) next[u] = load(t0 + u * BS_NT + tid);
        }
    };
    load_tile(v0);  // under way while the beam's state is read
    if (!beam_live(d, row)) return;
    tops[tid] = 0;
    if (tid == 0) floor_key = 0;
    if (tid < BS_WARPS) wcount[tid] = 0;
    __syncthreads();

    float m = -INFINITY;   // this thread's maximum so far
    double s = 0.0;        // its exponential sum, relative to sum_base(m)
    uint32_t thr = KEY_NINF + 1;   // a candidate's key has to reach it
    int count = 0;                 // candidates in this warp's buffer
    uint64_t *mine = buf + wid * BS_WCAP;

    auto publish = [&] {
        uint32_t key = okey(m);
        for (int i = 0; i < top; i++) {
            const uint32_t mx = __reduce_max_sync(0xffffffffu, key);
            const uint32_t holders = __ballot_sync(0xffffffffu, key == mx);
            if (lane == __ffs(holders) - 1) {
                tops[wid * top + i] = mx;
                key = 0;
            }
        }
    };
    // The k-th largest published key, without its five lowest bits: they make the keys of a lane
    // group different, so that one comparison with each gives a key's place.
    auto kth_published = [&] {
        uint32_t found = 0;
        if (k <= 16) {  // 32 keys at most
            const uint32_t v = lane < BS_WARPS * top ? tops[lane] & ~31u | (31 - lane) : 0;
            int above = 0;
#pragma unroll 8
            for (int i = 0; i < BS_WARPS * top; i++) above += (tops[i] & ~31u | (31 - i)) > v;
            if (above == k - 1) found = v & ~31u;
        } else {
            for (int at = lane; at < BS_WARPS * top; at += 32) {
                const uint32_t v = tops[at];
                int above = 0, same = 0;
#pragma unroll 8
                for (int i = 0; i < BS_WARPS * top; i++) {
                    const uint32_t o = tops[i];
                    above += o > v;
                    same += o == v;
                }
                if (above < k && above + same >= k) found = v;
            }
            __syncwarp();
        }
        // warps go on publishing meanwhile, so a lane may find none, or another one; each is a key
        // that k elements reach
        return __reduce_max_sync(0xffffffffu, found);
    };
    // this warp's k best, sorted
    auto cut = [&] {
        for (int i = count + lane; i < BS_WCAP; i += 32) mine[i] = 0;
        __syncwarp();
        sort_desc(mine, BS_WCAP, lane, 32, [] { __syncwarp(); });
        if (count >= k) {
            count = k;
            const uint32_t last = (uint32_t)(mine[k - 1] >> 32);
            if (lane == 0) atomicMax(&floor_key, last);
            thr = max(thr, last + 1);
        }
        if (lane == 0) wcount[wid] = count;
        __syncwarp();
    };

    // appends the elements of a tile that reach the threshold
    auto collect = [&](const uint4 (&x)[BS_U], int t0) {
        const uint32_t all = reaching<DT, BS_U>(x, okey_value(thr));
        auto append = [&](uint32_t take) {
            while (take) {
                const int bit = __ffs(take) - 1;
                take &= take - 1;
                int e;  // element of this thread's tile: vector e / VEC, place e % VEC
                const uint32_t key = okey(element_of<DT, BS_U>(x, bit, &e));
                if (key >= thr)
                    mine[atomicAdd(&wcount[wid], 1)] =
                        composite(key, (t0 + e / VEC * BS_NT + tid) * VEC - shift + e % VEC);
            }
            __syncwarp();
            count = *(volatile int *)&wcount[wid];
        };
        if (count + __reduce_add_sync(0xffffffffu, __popc(all)) <= BS_WCAP) append(all);
        else
#pragma unroll 1
            for (int u = 0; u < BS_U; u++) {  // one vector of each lane at a time
                if (count > BS_WCAP - 32 * VEC) cut();
                append(all & (DT == DLLM_DTYPE_F32 ? 0xfu : 0xf000fu) << (4 * u));
            }
    };

    float base = -INFINITY;  // sum_base(m), for |m| < 2^20
    int tile = 0;
    for (int t0 = v0; t0 < v1; t0 += BS_NT * BS_U, tile++) {
        uint4 x[BS_U];
#pragma unroll
        for (int u = 0; u < BS_U; u++) x[u] = next[u];
        load_tile(t0 + BS_NT * BS_U);
        const float tm = largest<DT, BS_U>(x);
        Pair part(0.0f, 0.0f);
        const Pair scale(LOG2E, LOG2E);
        if (!__any_sync(0xffffffffu, fabsf(tm) >= BASE_EXACT || fabsf(m) >= BASE_EXACT)) {
            if (tm > m) {
                const float to = __fmul_rn(tm, LOG2E);
                s *= (double)exp2_approx(__fsub_rn(base, to));
                base = to;
                m = tm;
            }
            const Pair minus(-base, -base);
#pragma unroll
            for (int u = 0; u < BS_U; u++)
#pragma unroll
                for (int i = 0; i < VEC / 2; i++) {
                    const float2 xi = pair_of<DT>(x[u], i);
                    part = add2(part, exp2_approx(fma2(Pair(xi.x, xi.y), scale, minus)));
                }
        } else {  // values from 2^20 on, or nothing above -inf yet
            if (tm > m) {
                s *= rebase(m, tm);
                m = tm;
            }
            base = m == -INFINITY ? m : (float)sum_base(m);
            const float ref = m == -INFINITY ? 0.0f : m, off = (float)((double)LOG2E * (double)ref - sum_base(ref));
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
        s += (double)part.sum();

        if ((tile & (tile - 1)) == 0) {  // after 1, 2, 3, 5, 9, ... tiles
            publish();
            if (tile == 0) {  // the first threshold is taken from every warp's first tile
                __syncthreads();
                thr = max(thr, kth_published());
            } else if (wid == 0) {
                __syncwarp();
                const uint32_t kth = kth_published();
                if (lane == 0) atomicMax(&floor_key, kth);
            }
        }
        thr = max(thr, *(volatile uint32_t *)&floor_key);
        if (__any_sync(0xffffffffu, tm >= okey_value(thr))) collect(x, t0);
    }

    // the chunk's maximum and sum, and the warps' candidates that reach the last threshold
    float M = m;
#pragma unroll
    for (int o = 16; o; o >>= 1) M = max_keep(M, __shfl_xor_sync(0xffffffffu, M, o));
    publish();
    if (lane == 0) wm[wid] = M;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < BS_WARPS; w++) M = max_keep(M, wm[w]);
    double S = s * rebase(m, M);
#pragma unroll
    for (int o = 16; o; o >>= 1) S += __shfl_xor_sync(0xffffffffu, S, o);
    const uint64_t lowest = (uint64_t)max(kth_published(), floor_key) << 32;
    int kept = 0;
    for (int i = lane; i < (count + 31) / 32 * 32; i += 32) {  // in place: what is kept moves towards the front
        const uint64_t c = i < count ? mine[i] : 0;
        const bool keep = i < count && c >= lowest;
        const uint32_t who = __ballot_sync(0xffffffffu, keep);
        if (keep) mine[kept + __popc(who & ((1u << lane) - 1))] = c;
        kept += __popc(who);
    }
    if (lane == 0) {
        ws[wid] = S;
        wcount[wid] = kept;
    }
    __syncthreads();
    int n = 0, at = 0;
#pragma unroll
    for (int w = 0; w < BS_WARPS; w++) {
        if (w == wid) at = n;
        n += wcount[w];
    }
    const int64_t chunk = blockIdx.x;
    if (tid == 0) {
        double tot = 0.0;
        for (int w = 0; w < BS_WARPS; w++) tot += ws[w];
        sums[chunk] = {M, 0.0f, tot};
    }
    uint64_t *out = cands + chunk * k;
    if (n <= BS_NT) {  // each candidate's place is the number of larger ones
        for (int i = lane; i < kept; i += 32) few[at + i] = mine[i];
        __syncthreads();
        if (tid < n) {
            const uint64_t c = few[tid];
            int place = 0;
            for (int i = 0; i < n; i++) place += few[i] > c;
            if (place < k) out[place] = c;
        }
        for (int i = n + tid; i < k; i += BS_NT) out[i] = 0;
        return;
    }
    for (int i = kept + lane; i < BS_WCAP; i += 32) mine[i] = 0;
    __syncthreads();
    sort_desc(buf, BS_CAP, tid, BS_NT, [] { __syncthreads(); });
    for (int i = tid; i < k; i += BS_NT) out[i] = buf[i];
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

// One CTA per sequence: the beams' log-sum-exps from their chunks, then the k best of the chunks'
// candidates.  The same threshold as in a chunk (over the threads' best ranks, rounded down to
// fp32, which keeps their order) leaves a few; each one's place is the number that comes before
// it.  Where more are left than fit, the threshold is raised to the highest that k candidates
// reach; where that still leaves too many (equal ranks), k rounds take the best candidate that
// comes after the one taken last.
constexpr int BM_LEFT = 512;
constexpr int BM_HELD = 4;  // candidates that a thread keeps in registers

__global__ void __launch_bounds__(BS_NT) beam_merge_kernel(dllm_beam_desc d, const ChunkSum *sums,
                                                           const uint64_t *cands, int chunks) {
    __shared__ double lse[DLLM_BEAM_MAX], inv_len[DLLM_BEAM_MAX];
    __shared__ float score_in[DLLM_BEAM_MAX];  // copies, so that the outputs may lie over the inputs
    __shared__ int length_in[DLLM_BEAM_MAX];
    __shared__ int live[DLLM_BEAM_MAX];  // 0 nothing to offer, 1 its row's continuations, 2 ended
    __shared__ Best wbest[BS_WARPS];
    __shared__ uint64_t left_key[BM_LEFT], left_comp[BM_LEFT];
    __shared__ int left_beam[BM_LEFT];
    __shared__ uint32_t wkey[BS_WARPS];
    __shared__ int nleft;
    const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
    const int K = d.beams, k = d.k;
    const int64_t item = blockIdx.x;
    if (tid == 0) nleft = 0;
    // what does not come from the chunks is read while they run
    for (int b = tid; b < K; b += BS_NT) {
        const int64_t row = item * K + b;
        const float sc = d.scores[row];
        const bool ended = d.finished && d.finished[row];
        const int len_in = d.lengths ? d.lengths[row] : 0;
        const double len = fmax((double)len_in + (ended ? 0.0 : 1.0), 1.0);
        length_in[b] = len_in;
        score_in[b] = sc;
        inv_len[b] = d.length_penalty != 0.0f && d.lengths ? 1.0 / pow(len, (double)d.length_penalty) : 1.0;
        live[b] = !(sc >= -FLT_MAX && sc <= FLT_MAX) ? 0 : ended ? 2 : 1;
    }
    __syncthreads();
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int per_beam = chunks * k, N = K * per_beam;
    const uint64_t *mine = cands + item * N;
    // The warps take the chunks' lists in turn, so that each meets every beam's candidates: their
    // thresholds are then alike.  Candidate number q of a warp is position q % k of its list q / k.
    const int warp_n = ((K * chunks - wid + BS_WARPS - 1) / BS_WARPS) * k;
    auto number = [&](int q) { return q < warp_n ? ((q / k) * BS_WARPS + wid) * k + q % k : N; };
    uint64_t held[BM_HELD];  // this thread's first candidates
    int at_e[BM_HELD];
#pragma unroll
    for (int i = 0; i < BM_HELD; i++) {
        const int e = at_e[i] = number(lane + 32 * i);
        held[i] = e < N && live[e / per_beam] == 1 ? mine[e] : 0;
    }
    for (int b = wid; b < K; b += BS_WARPS) {
        const int64_t row = item * K + b;
        int st = 0, kind = live[b];
        double l = 0.0;
        if (kind == 0 && !(score_in[b] < 0.0f)) st = DLLM_ROW_ERR_NONFINITE;  // NaN or +inf
        if (kind == 1) {
            float M = -INFINITY;
            double S = 0.0;
            if (chunks <= 32) {
                const ChunkSum p = lane < chunks ? sums[row * chunks + lane] : ChunkSum{-INFINITY, 0.0f, 0.0};
                M = p.m;
#pragma unroll
                for (int o = 16; o; o >>= 1) M = max_keep(M, __shfl_xor_sync(0xffffffffu, M, o));
                S = p.s * rebase(p.m, M);
            } else {
                for (int c = lane; c < chunks; c += 32) M = max_keep(M, sums[row * chunks + c].m);
#pragma unroll
                for (int o = 16; o; o >>= 1) M = max_keep(M, __shfl_xor_sync(0xffffffffu, M, o));
                for (int c = lane; c < chunks; c += 32) {
                    const ChunkSum p = sums[row * chunks + c];
                    S += p.s * rebase(p.m, M);
                }
            }
#pragma unroll
            for (int o = 16; o; o >>= 1) S += __shfl_xor_sync(0xffffffffu, S, o);
            if (S != S || M == INFINITY) {
                st = DLLM_ROW_ERR_NONFINITE;
                kind = 0;
            } else if (M > -INFINITY) l = (sum_base(M) + log2(S)) * (1.0 / (double)LOG2E);
            else kind = 0;
        }
        __syncwarp();
        if (lane == 0) {
            lse[b] = l;
            live[b] = kind;
            if (d.status) d.status[row] = st;
        }
    }
    __syncthreads();
    // candidate e: position e % k of a chunk's list; an ended beam offers its first position only
    auto candidate_of = [&](int e, int b, uint64_t comp, Best *c) {
        double cum = (double)score_in[b];
        if (live[b] == 0) return false;
        if (live[b] == 2) {
            if (e != b * per_beam) return false;
            comp = composite(0, d.eos);
        } else {
            if (!comp) return false;
            cum += (double)okey_value((uint32_t)(comp >> 32)) - lse[b];
        }
        *c = {cum * inv_len[b], b, comp};
        return true;
    };
    auto candidate = [&](int e, Best *c) {
        const int b = e / per_beam;
        return candidate_of(e, b, live[b] == 1 ? mine[e] : 0, c);
    };
    auto emit = [&](int place, const Best &c, bool none) {
        float score = -INFINITY;
        if (!none) {
            double cum = (double)score_in[c.beam];
            if (live[c.beam] == 1) cum += (double)okey_value((uint32_t)(c.comp >> 32)) - lse[c.beam];
            score = __double2float_rn(cum);
        }
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
    };
    uint32_t mx = 0, key[BM_HELD];
#pragma unroll
    for (int i = 0; i < BM_HELD; i++) {
        const int e = at_e[i];
        Best c;
        key[i] = e < N && candidate_of(e, e / per_beam, held[i], &c) ? okey(__double2float_rd(c.rank)) : 0;
        mx = max(mx, key[i]);
    }
    for (int q = lane + 32 * BM_HELD; q < warp_n; q += 32) {
        Best c;
        if (candidate(number(q), &c)) mx = max(mx, okey(__double2float_rd(c.rank)));
    }
    const uint32_t kj = warp_jth(mx, (k + BS_WARPS - 1) / BS_WARPS);
    if (lane == 0) wkey[wid] = kj;
    __syncthreads();
    uint32_t lo = wkey[0];
#pragma unroll
    for (int w = 1; w < BS_WARPS; w++) lo = min(lo, wkey[w]);
#pragma unroll
    for (int i = 0; i < BM_HELD; i++) {
        if (key[i] == 0 || key[i] < lo) continue;
        const int e = at_e[i], at = atomicAdd(&nleft, 1);
        Best c;
        if (at < BM_LEFT && candidate_of(e, e / per_beam, held[i], &c)) keep(at, c);
    }
    for (int q = lane + 32 * BM_HELD; q < warp_n; q += 32) {
        Best c;
        if (!candidate(number(q), &c) || okey(__double2float_rd(c.rank)) < lo) continue;
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
                c_mid += candidate(e, &c) && okey(__double2float_rd(c.rank)) >= mid;
            }
            c_mid = __reduce_add_sync(0xffffffffu, c_mid);
            __syncthreads();
            if (lane == 0) wkey[wid] = c_mid;
            __syncthreads();
            c_mid = 0;
#pragma unroll
            for (int w = 0; w < BS_WARPS; w++) c_mid += wkey[w];
            if (c_mid >= k) reached = mid;
            else above = mid;
        }
        __syncthreads();
        if (tid == 0) nleft = 0;
        __syncthreads();
        for (int e = tid; e < N; e += BS_NT) {
            Best c;
            if (!candidate(e, &c) || okey(__double2float_rd(c.rank)) < reached) continue;
            const int at = atomicAdd(&nleft, 1);
            if (at < BM_LEFT) keep(at, c);
        }
        __syncthreads();
        n = nleft;
    }
    if (n <= BM_LEFT) {
        for (int i = tid; i < n; i += BS_NT) {
            const uint64_t key = left_key[i], comp = left_comp[i];
            const int beam = left_beam[i];
            int place = 0, same = 0;
#pragma unroll 4
            for (int j = 0; j < n; j++) {
                const uint64_t other = left_key[j];
                place += other > key;
                same += other == key;
            }
            if (same > 1)
                for (int j = 0; j < n; j++)
                    if (left_key[j] == key)
                        place += left_beam[j] < beam || (left_beam[j] == beam && left_comp[j] > comp);
            if (place < k) emit(place, Best{0.0, beam, comp}, false);
        }
        for (int i = n + tid; i < k; i += BS_NT) emit(i, Best{}, true);
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
        if (tid == 0) emit(r, best, false);  // more candidates than BM_LEFT >= k: there is one
        last = best;
    }
}

// Chunks per row: the count whose waves of CTAs (4 per SM) take least, a chunk's set-up and
// selection counted as two tiles.
int beam_chunks(int64_t rows, int vocab, int dtype) {
    const int vec = dtype == DLLM_DTYPE_F32 ? 4 : 8;
    const int64_t tiles = ((int64_t)vocab + BS_NT * BS_U * vec - 1) / (BS_NT * BS_U * vec), slots = 148 * 4;
    int best = 1;
    int64_t least = INT64_MAX;
    for (int c = 1; c <= tiles && c <= 64; c++) {
        const int64_t cost = (rows * c + slots - 1) / slots * ((tiles + c - 1) / c + 2);
        if (cost < least) {
            least = cost;
            best = c;
        }
    }
    return best;
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

// A CTA owns one column range (one vector per thread) of one segment for all beams of a sequence:
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
    unsigned char *base = a.tensors[tensor] + item * K * a.row_stride + seg * a.seg_stride + col;
    unsigned char *mine = stage + (size_t)tid * VB;
    const size_t pitch = (size_t)blockDim.x * VB;
    for (int p = 0; p < K; p++) {
        if (!needed[p]) continue;
        if (VB == 1) mine[p * pitch] = base[p * a.row_stride];
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
        if (VB == 16) *(uint4 *)dst = *(const uint4 *)src;
        else if (VB == 4) *(uint32_t *)dst = *(const uint32_t *)src;
        else *dst = *src;
    }
}

}  // namespace

template <auto Kernel>
static void launch_chunks(unsigned grid, const dllm_beam_desc &d, int chunks, ChunkSum *sums, uint64_t *cands,
                          cudaStream_t stream) {
    // room for four CTAs' buffers on an SM
    set_once<Kernel>(cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    Kernel<<<grid, BS_NT, 0, stream>>>(d, chunks, sums, cands);
}

size_t beam_ws_bytes(const dllm_beam_desc *d) {
    const int64_t rows = (int64_t)d->batch * d->beams;
    const size_t n = (size_t)rows * beam_chunks(rows, d->vocab, d->dtype);
    return (n * sizeof(ChunkSum) + 255) / 256 * 256 + n * d->k * sizeof(uint64_t);
}

dllm_status launch_beam_select(const dllm_beam_desc *d, void *ws, cudaStream_t stream) {
    const int64_t rows = (int64_t)d->batch * d->beams;
    const int chunks = beam_chunks(rows, d->vocab, d->dtype);
    ChunkSum *sums = (ChunkSum *)ws;
    uint64_t *cands = (uint64_t *)((unsigned char *)ws + ((size_t)rows * chunks * sizeof(ChunkSum) + 255) / 256 * 256);
    if (rows * chunks > INT32_MAX) return DLLM_ERR_UNSUPPORTED;
    const unsigned grid = (unsigned)(rows * chunks);
#define DLLM_CHUNKS(DT)                                                                                \
    (d->mask ? launch_chunks<beam_chunk_kernel<DT, true>>(grid, *d, chunks, sums, cands, stream)       \
             : launch_chunks<beam_chunk_kernel<DT, false>>(grid, *d, chunks, sums, cands, stream))
    if (d->dtype == DLLM_DTYPE_F32) DLLM_CHUNKS(DLLM_DTYPE_F32);
    else if (d->dtype == DLLM_DTYPE_BF16) DLLM_CHUNKS(DLLM_DTYPE_BF16);
    else DLLM_CHUNKS(DLLM_DTYPE_F16);
#undef DLLM_CHUNKS
    if (cudaGetLastError() != cudaSuccess) return DLLM_ERR_CUDA;
    // launched while the chunks run; it waits for them on the GPU
    cudaLaunchAttribute attr = {};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(d->batch);
    cfg.blockDim = dim3(BS_NT);
    cfg.stream = stream;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, beam_merge_kernel, *d, (const ChunkSum *)sums, (const uint64_t *)cands, chunks) ==
                   cudaSuccess
               ? DLLM_OK
               : DLLM_ERR_CUDA;
}

dllm_status launch_beam_reorder(int batch, int beams, const int32_t *parent, int ntensors, void *const *tensors,
                                int64_t row_stride, int segs, int64_t seg_stride, int64_t run, cudaStream_t stream) {
    uintptr_t bits = (uintptr_t)row_stride | (uintptr_t)run | (segs > 1 ? (uintptr_t)seg_stride : 0);
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
    const int64_t slices = (run / vb + nt - 1) / nt, per_tensor = slices * segs * batch;
    if (slices > INT32_MAX || slices * segs > INT32_MAX || per_tensor > INT32_MAX) return DLLM_ERR_UNSUPPORTED;
    a.slices = (int)slices;
    const int group = (int)(INT32_MAX / per_tensor < RO_TENSORS ? INT32_MAX / per_tensor : RO_TENSORS);
    const size_t smem = (size_t)beams * nt * vb;
    auto launch = [&](auto kernel) {
        for (int t = 0; t < ntensors; t += group) {
            const int n = ntensors - t < group ? ntensors - t : group;
            for (int i = 0; i < n; i++) a.tensors[i] = (unsigned char *)tensors[t + i];
            kernel<<<(unsigned)(per_tensor * n), nt, smem, stream>>>(a);
            if (cudaGetLastError() != cudaSuccess) return DLLM_ERR_CUDA;
        }
        return DLLM_OK;
    };
    const cudaFuncAttribute size = cudaFuncAttributeMaxDynamicSharedMemorySize;
    cudaError_t e = vb == 16  ? set_once<beam_reorder_kernel<16>>(size, 131072)
                    : vb == 4 ? set_once<beam_reorder_kernel<4>>(size, 131072)
                              : set_once<beam_reorder_kernel<1>>(size, 131072);
    if (e != cudaSuccess) return DLLM_ERR_CUDA;
    return vb == 16 ? launch(beam_reorder_kernel<16>) : vb == 4 ? launch(beam_reorder_kernel<4>) : launch(beam_reorder_kernel<1>);
}

}  // namespace dllm
