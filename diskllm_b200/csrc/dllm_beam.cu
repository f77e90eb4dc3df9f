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

namespace dllm {
namespace {

constexpr int BS_NT = 256;
constexpr int BS_WARPS = BS_NT / 32;
constexpr int BS_U = 4;             // 16-byte vectors per thread and tile
constexpr int BS_CAP = 4096;        // candidate buffer (entries of 8 bytes); a power of two
constexpr uint32_t KEY_NINF = 0x007fffffu;  // order key of -inf

// One chunk's maximum and exponential sum relative to it.
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

// A candidate: (order key << 32) | ~id, so that a larger composite is (logit desc, id asc).
__device__ __forceinline__ uint64_t composite(uint32_t key, int id) { return (uint64_t)key << 32 | (uint32_t)~id; }

// A beam that offers its row's continuations: not ended, with a finite score.
__device__ __forceinline__ bool beam_live(const dllm_beam_desc &d, int64_t row) {
    if (d.finished && d.finished[row]) return false;
    return fabsf(d.scores[row]) <= FLT_MAX;
}

// Sorts buf[0, n2) descending (n2 a power of two; entries past n are set to 0 first).
__device__ void sort_desc(uint64_t *buf, int n, int n2) {
    for (int i = n + threadIdx.x; i < n2; i += BS_NT) buf[i] = 0;
    __syncthreads();
    for (int size = 2; size <= n2; size <<= 1)
        for (int stride = size >> 1; stride; stride >>= 1) {
            for (int i = threadIdx.x; i < n2 / 2; i += BS_NT) {
                const int lo = 2 * i - (i & (stride - 1)), hi = lo + stride;
                const uint64_t a = buf[lo], b = buf[hi];
                if ((a < b) == ((lo & size) == 0)) {
                    buf[lo] = b;
                    buf[hi] = a;
                }
            }
            __syncthreads();
        }
}

__device__ __forceinline__ int pow2_at_least(int n) { return n <= 2 ? 2 : 1 << (32 - __clz(n - 1)); }

// The j-th largest of a warp's 32 keys (j from 1), in every lane.
__device__ __forceinline__ uint32_t warp_jth(uint32_t key, int j) {
    uint32_t mx = 0;
    for (int i = 0; i < j; i++) {
        mx = __reduce_max_sync(0xffffffffu, key);
        const uint32_t holders = __ballot_sync(0xffffffffu, key == mx);
        if ((threadIdx.x & 31) == __ffs(holders) - 1) key = 0;
    }
    return mx;
}

template <int DT>
struct Vec {
    static constexpr int N = DT == DLLM_DTYPE_F32 ? 4 : 8;  // elements of 16 bytes
};

template <int DT>
__device__ __forceinline__ void unpack(const uint4 &raw, float *f) {
    const uint32_t u[4] = {raw.x, raw.y, raw.z, raw.w};
    if (DT == DLLM_DTYPE_F32) {
#pragma unroll
        for (int i = 0; i < 4; i++) f[i] = __uint_as_float(u[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (DT == DLLM_DTYPE_BF16) {
                f[2 * i] = __uint_as_float(u[i] << 16);
                f[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
            } else {
                f[2 * i] = __half2float(__ushort_as_half((unsigned short)(u[i] & 0xffffu)));
                f[2 * i + 1] = __half2float(__ushort_as_half((unsigned short)(u[i] >> 16)));
            }
        }
    }
}

// Grid rows x chunks.  A chunk is a range of the row's 16-byte vectors, counted from the row's
// first byte rounded down to 16 (so any row start is served; the first and the last vector are
// read by element).  Per tile a thread keeps its elements in registers, updates its running
// maximum and sum, and appends those at or above the threshold to the candidate buffer.
//
// Threshold: after the first tile, with k <= 8 j, the smallest over the warps of the j-th largest
// thread maximum has at least k entries at or above it, all of the first tile, so with smaller
// ids than any later entry; later ones have to be strictly larger.  When the buffer could
// overflow it is sorted and cut to k, which raises the threshold the same way.
template <int DT, bool MASK>
__global__ void __launch_bounds__(BS_NT) beam_chunk_kernel(dllm_beam_desc d, int chunks, ChunkSum *sums,
                                                           uint64_t *cands) {
    constexpr int VEC = Vec<DT>::N, E = BS_U * VEC;
    constexpr float LOG2E = 1.44269504088896340736f;
    __shared__ uint64_t buf[BS_CAP];
    __shared__ int count;
    __shared__ uint32_t wkey[BS_WARPS];
    __shared__ float wm[BS_WARPS];
    __shared__ double ws[BS_WARPS];
    const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
    const int64_t row = blockIdx.x / chunks;
    const int part_no = blockIdx.x % chunks;
    if (!beam_live(d, row)) return;
    const int V = d.vocab, k = d.k;
    const size_t esz = DT == DLLM_DTYPE_F32 ? 4 : 2;
    const unsigned char *first = (const unsigned char *)d.logits + (size_t)row * d.row_stride * esz;
    const int shift = (int)((uintptr_t)first % 16 / esz);  // elements before the row in its first vector
    const uint4 *vecs = (const uint4 *)(first - shift * esz);
    const uint32_t *mrow = MASK ? d.mask + row * d.mask_stride : nullptr;
    const int64_t nvec = ((int64_t)V + shift + VEC - 1) / VEC;
    const int64_t per = (nvec + chunks - 1) / chunks;
    const int64_t v0 = per * part_no, v1 = v0 + per < nvec ? v0 + per : nvec;

    if (tid == 0) count = 0;
    __syncthreads();

    // vector j as floats; masked elements and those outside the row are -inf
    auto load = [&](int64_t j, float *f) {
        if (j >= v1) {
#pragma unroll
            for (int e = 0; e < VEC; e++) f[e] = -INFINITY;
            return;
        }
        const int64_t i0 = j * VEC - shift;
        if (i0 >= 0 && i0 + VEC <= V) {
            unpack<DT>(__ldg(vecs + j), f);
            if (MASK) {
                const int w = (int)(i0 >> 5), o = (int)(i0 & 31);
                const uint32_t lo = mrow[w], hi = o + VEC > 32 ? mrow[w + 1] : 0;
                const uint32_t bits = __funnelshift_r(lo, hi, o);
#pragma unroll
                for (int e = 0; e < VEC; e++)
                    if (!(bits >> e & 1)) f[e] = -INFINITY;
            }
        } else {
#pragma unroll
            for (int e = 0; e < VEC; e++) {
                const int64_t i = i0 + e;
                float x = -INFINITY;
                if (i >= 0 && i < V && (!MASK || (mrow[i >> 5] >> (i & 31) & 1))) {
                    if (DT == DLLM_DTYPE_F32) x = ((const float *)first)[i];
                    else {
                        const unsigned short u = ((const unsigned short *)first)[i];
                        x = DT == DLLM_DTYPE_BF16 ? __uint_as_float((uint32_t)u << 16)
                                                  : __half2float(__ushort_as_half(u));
                    }
                }
                f[e] = x;
            }
        }
    };

    float m = -INFINITY;   // this thread's maximum so far
    double s = 0.0;        // sum of exp(x - m)
    uint32_t thr = KEY_NINF + 1;  // a candidate's key has to reach it
    bool first_tile = true;
    float x[E];

    auto append = [&](int64_t j, int u) {
#pragma unroll
        for (int e = 0; e < VEC; e++) {
            const uint32_t key = okey(x[u * VEC + e]);
            if (x[u * VEC + e] == x[u * VEC + e] && key >= thr) {
                const int at = atomicAdd(&count, 1);
                if (at < BS_CAP) buf[at] = composite(key, (int)(j * VEC - shift + e));
            }
        }
    };
    // sorts the buffer, keeps the k best; the threshold is then above the last one kept
    auto cut = [&]() {
        const int n = count;
        sort_desc(buf, n, pow2_at_least(n));
        if (n >= k) thr = max(thr, (uint32_t)(buf[k - 1] >> 32) + 1);
        __syncthreads();
        if (tid == 0) count = n < k ? n : k;
        __syncthreads();
    };

    for (int64_t t0 = v0; t0 < v1; t0 += (int64_t)BS_NT * BS_U) {
#pragma unroll
        for (int u = 0; u < BS_U; u++) load(t0 + (int64_t)u * BS_NT + tid, x + u * VEC);
        float tm = x[0];
#pragma unroll
        for (int e = 1; e < E; e++) tm = fmaxf(tm, x[e]);
        const float mn = fmaxf(m, tm), ref = mn == -INFINITY ? 0.0f : mn;
        float part = 0.0f;
#pragma unroll
        for (int e = 0; e < E; e++) part += exp2_approx((x[e] - ref) * LOG2E);
        if (mn != m) s *= (double)exp2_approx((m - ref) * LOG2E);
        m = mn;
        s += (double)part;

        uint32_t lo = KEY_NINF;  // first tile: a key that k of its entries reach
        if (first_tile) {
            const uint32_t kj = warp_jth(okey(tm), (k + BS_WARPS - 1) / BS_WARPS);
            if (lane == 0) wkey[wid] = kj;
            __syncthreads();
            lo = wkey[0];
#pragma unroll
            for (int w = 1; w < BS_WARPS; w++) lo = min(lo, wkey[w]);
            thr = max(thr, lo);
        }
        const int before = count;
        __syncthreads();
        if (okey(tm) >= thr) {
#pragma unroll
            for (int u = 0; u < BS_U; u++) append(t0 + (int64_t)u * BS_NT + tid, u);
        }
        __syncthreads();
        if (count > BS_CAP) {  // too many at once: take the tile again, a vector of each thread at a time
            __syncthreads();
            if (tid == 0) count = before;
#pragma unroll
            for (int u = 0; u < BS_U; u++) {
                __syncthreads();
                const int held = count;
                __syncthreads();
                if (held > BS_CAP - BS_NT * VEC) cut();
                append(t0 + (int64_t)u * BS_NT + tid, u);
            }
            __syncthreads();
        }
        if (lo > KEY_NINF) thr = max(thr, lo + 1);
        first_tile = false;
        const int held = count;
        __syncthreads();
        if (held > BS_CAP / 2) cut();
    }

    // the chunk's maximum and sum
    float M = m;
#pragma unroll
    for (int o = 16; o; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    if (lane == 0) wm[wid] = M;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < BS_WARPS; w++) M = fmaxf(M, wm[w]);
    const float ref = M == -INFINITY ? 0.0f : M;
    double S = m == -INFINITY ? s : s * (double)expf(m - ref);
#pragma unroll
    for (int o = 16; o; o >>= 1) S += __shfl_xor_sync(0xffffffffu, S, o);
    if (lane == 0) ws[wid] = S;
    const int n = count;
    sort_desc(buf, n, pow2_at_least(n));
    const int64_t chunk = blockIdx.x;
    if (tid == 0) {
        double tot = 0.0;
        for (int w = 0; w < BS_WARPS; w++) tot += ws[w];
        sums[chunk] = {M, 0.0f, tot};
    }
    for (int i = tid; i < k; i += BS_NT) cands[chunk * k + i] = i < n ? buf[i] : 0;
}

struct Best {
    double rank;
    int beam;
    uint64_t comp;
};
// whether a comes before b in the operator's order
__device__ __forceinline__ bool before(const Best &a, const Best &b) {
    if (a.rank != b.rank) return a.rank > b.rank;
    if (a.beam != b.beam) return a.beam < b.beam;
    return a.comp > b.comp;
}

// One CTA per sequence: the beams' log-sum-exps from their chunks, then k rounds, each taking the
// best candidate that comes after the one taken last.
__global__ void __launch_bounds__(BS_NT) beam_merge_kernel(dllm_beam_desc d, const ChunkSum *sums,
                                                           const uint64_t *cands, int chunks) {
    __shared__ double lse[DLLM_BEAM_MAX], inv_len[DLLM_BEAM_MAX];
    __shared__ float score_in[DLLM_BEAM_MAX];  // copies, so that the outputs may lie over the inputs
    __shared__ int length_in[DLLM_BEAM_MAX];
    __shared__ int live[DLLM_BEAM_MAX];  // 0 nothing to offer, 1 its row's continuations, 2 ended
    __shared__ Best wbest[BS_WARPS];
    const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
    const int K = d.beams, k = d.k;
    const int64_t item = blockIdx.x;
    for (int b = tid; b < K; b += BS_NT) {
        const int64_t row = item * K + b;
        const float sc = d.scores[row];
        const bool ended = d.finished && d.finished[row];
        int st = 0, kind = 0;
        double l = 0.0;
        if (sc != sc || sc == INFINITY) st = DLLM_ROW_ERR_NONFINITE;
        else if (ended) kind = sc >= -FLT_MAX ? 2 : 0;
        else if (sc >= -FLT_MAX) {
            float M = -INFINITY;
            for (int c = 0; c < chunks; c++) M = fmaxf(M, sums[row * chunks + c].m);
            double S = 0.0;
            for (int c = 0; c < chunks; c++) {
                const ChunkSum p = sums[row * chunks + c];
                S += p.m == -INFINITY ? p.s : p.s * exp((double)p.m - (double)M);
            }
            if (S != S || M == INFINITY) st = DLLM_ROW_ERR_NONFINITE;
            else if (M > -INFINITY) {
                kind = 1;
                l = (double)M + log(S);
            }
        }
        length_in[b] = d.lengths ? d.lengths[row] : 0;
        const double len = fmax((double)length_in[b] + (ended ? 0.0 : 1.0), 1.0);
        score_in[b] = sc;
        lse[b] = l;
        inv_len[b] = d.length_penalty != 0.0f && d.lengths ? 1.0 / pow(len, (double)d.length_penalty) : 1.0;
        live[b] = kind;
        if (d.status) d.status[row] = st;
    }
    __syncthreads();
    const int64_t N = (int64_t)K * chunks * k;
    // candidate e: position e % k of a chunk's list; an ended beam offers its first position only
    auto candidate = [&](int64_t e, Best *c) {
        const int b = (int)(e / ((int64_t)chunks * k));
        if (live[b] == 0) return false;
        double cum = (double)score_in[b];
        uint64_t comp;
        if (live[b] == 2) {
            if (e % ((int64_t)chunks * k)) return false;
            comp = composite(0, d.eos);
        } else {
            comp = cands[item * N + e];
            if (!comp) return false;
            cum += (double)okey_value((uint32_t)(comp >> 32)) - lse[b];
        }
        *c = {cum * inv_len[b], b, comp};
        return true;
    };
    Best last = {INFINITY, -1, 0};
    for (int r = 0; r < k; r++) {
        Best best = {-INFINITY, 1 << 30, 0};
        for (int64_t e = tid; e < N; e += BS_NT) {
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
        const bool none = best.beam == 1 << 30;
        if (tid == 0) {
            float score = -INFINITY;
            if (!none) {
                double cum = (double)score_in[best.beam];
                if (live[best.beam] == 1) cum += (double)okey_value((uint32_t)(best.comp >> 32)) - lse[best.beam];
                score = __double2float_rn(cum);
            }
            d.out_score[item * k + r] = score;
            d.out_parent[item * k + r] = none ? -1 : best.beam;
            const int32_t token = none ? -1 : (int32_t)~(uint32_t)best.comp;
            const bool ended = !none && live[best.beam] == 2;
            d.out_token[item * k + r] = token;
            if (d.out_finished) d.out_finished[item * k + r] = ended || (!none && token == d.eos);
            if (d.out_lengths) d.out_lengths[item * k + r] = none ? 0 : length_in[best.beam] + (ended ? 0 : 1);
        }
        last = none ? Best{-INFINITY, 1 << 30, 0} : best;
    }
}

// Chunks per row: enough CTAs to fill the GPU, no chunk smaller than one tile.
int beam_chunks(int64_t rows, int vocab, int dtype) {
    const int vec = dtype == DLLM_DTYPE_F32 ? 4 : 8;
    const int64_t tile = (int64_t)BS_NT * BS_U * vec;
    int64_t most = (vocab + tile - 1) / tile, want = (148 * 6 + rows - 1) / rows;
    if (want > most) want = most;
    return (int)(want < 1 ? 1 : want);
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
    auto go = [&](auto kernel) { kernel<<<grid, BS_NT, 0, stream>>>(*d, chunks, sums, cands); };
    const bool mask = d->mask != nullptr;
    if (d->dtype == DLLM_DTYPE_F32) {
        if (mask) go(beam_chunk_kernel<DLLM_DTYPE_F32, true>);
        else go(beam_chunk_kernel<DLLM_DTYPE_F32, false>);
    } else if (d->dtype == DLLM_DTYPE_BF16) {
        if (mask) go(beam_chunk_kernel<DLLM_DTYPE_BF16, true>);
        else go(beam_chunk_kernel<DLLM_DTYPE_BF16, false>);
    } else {
        if (mask) go(beam_chunk_kernel<DLLM_DTYPE_F16, true>);
        else go(beam_chunk_kernel<DLLM_DTYPE_F16, false>);
    }
    if (cudaGetLastError() != cudaSuccess) return DLLM_ERR_CUDA;
    beam_merge_kernel<<<d->batch, BS_NT, 0, stream>>>(*d, sums, cands, chunks);
    return cudaGetLastError() == cudaSuccess ? DLLM_OK : DLLM_ERR_CUDA;
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
    auto go = [&](auto kernel) {
        if (cudaFuncSetAttribute((const void *)kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 131072) != cudaSuccess)
            return DLLM_ERR_CUDA;
        for (int t = 0; t < ntensors; t += group) {
            const int n = ntensors - t < group ? ntensors - t : group;
            for (int i = 0; i < n; i++) a.tensors[i] = (unsigned char *)tensors[t + i];
            kernel<<<(unsigned)(per_tensor * n), nt, smem, stream>>>(a);
            if (cudaGetLastError() != cudaSuccess) return DLLM_ERR_CUDA;
        }
        return DLLM_OK;
    };
    if (vb == 16) return go(beam_reorder_kernel<16>);
    if (vb == 4) return go(beam_reorder_kernel<4>);
    return go(beam_reorder_kernel<1>);
}

}  // namespace dllm
