// hx_attn.cuh — what the two decode attention kernels share: typed access, the division of the work over the
// CTAs, the join of its pieces and the argument checks.
#pragma once

#include "hx_paged.cuh"

namespace hx {

constexpr int ATTN_SMS = 148;

__device__ __forceinline__ float io_load(const void *p, int dtype, int64_t i) {
    if (dtype == F32) return static_cast<const float *>(p)[i];
    if (dtype == F16) return to_f32(static_cast<const __half *>(p)[i]);
    return to_f32(static_cast<const __nv_bfloat16 *>(p)[i]);
}
__device__ __forceinline__ void io_store(void *p, int dtype, int64_t i, float x) {
    if (dtype == F32) static_cast<float *>(p)[i] = x;
    else if (dtype == F16) static_cast<__half *>(p)[i] = from_f32<__half>(x);
    else static_cast<__nv_bfloat16 *>(p)[i] = from_f32<__nv_bfloat16>(x);
}

// 2^x to about 2^-22 relative, in one instruction; results below 2^-126 are zero.
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// ln of the weights' sum: m their largest exponent, sum relative to 2^(m - off).
__device__ __forceinline__ float lse_of(float m, float sum, float off) {
    if (sum == 0.0f) return -kv_inf();
    return ((m == -kv_inf() ? 0.0f : m) + log2f(sum) - off) * 0.693147180559945f;
}

// A sequence longer than its table cannot be read: it has no work, and the join gives NaN for it.
__device__ __forceinline__ int64_t table_capacity(const KvView &c) { return (int64_t)c.table_pages << c.pt_log2; }
__device__ __forceinline__ int units_of(const KvView &c, const int32_t *lens, int b, int unit) {
    const int n = lens[b];
    return n <= 0 || n > table_capacity(c) ? 0 : (int)(((int64_t)n + unit - 1) / unit);
}

// The calling CTA's share [cur, end) of the N = n_pairs * sum_b units_of(b) units, laid out sequence by sequence,
// pair by pair: the sequence of unit cur and the sum of the units of the sequences before it. False without a
// share. Every thread of the CTA calls it; scan: one word a warp.
template <int THREADS>
__device__ __forceinline__ bool my_units(const KvView &c, const int32_t *lens, int unit, int n_pairs, int64_t *scan, int &b,
                                         int64_t &before, int64_t &cur, int64_t &end, int64_t &total, int &ctas) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, B = c.n_seqs;
    const int per = (B + THREADS - 1) / THREADS;
    int64_t mine = 0;
    for (int i = tid * per; i < min(B, (tid + 1) * per); i++) mine += units_of(c, lens, i, unit);
    int64_t upto = mine;
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
        const int64_t x = __shfl_up_sync(0xffffffffu, upto, s);
        if (lane >= s) upto += x;
    }
    if (lane == 31) scan[warp] = upto;
    __syncthreads();
    int64_t base = 0, sum = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; w++) {
        if (w < warp) base += scan[w];
        sum += scan[w];
    }
    total = sum * n_pairs;
    ctas = (int)min((int64_t)gridDim.x, total);
    const int64_t start = base + upto - mine;             // units of the sequences before my chunk
    cur = end = 0;
    if (total) cur = blockIdx.x * total / ctas, end = (blockIdx.x + 1) * total / ctas;
    const bool none = blockIdx.x >= ctas;
    // the chunk that holds unit cur: the last one that starts at or before it
    const int chunk = __syncthreads_count(start * n_pairs <= cur) - 1;
    if (tid == chunk) scan[0] = start;
    __syncthreads();
    if (none) return false;
    b = chunk * per, before = scan[0];
    for (;;) {
        const int nu = units_of(c, lens, b, unit);
        if ((before + nu) * n_pairs > cur) break;
        before += nu, b++;
    }
    return true;
}

// One launch after the split kernel: pieces of each (sequence, head) whose work several CTAs did are joined in CTA
// order (weights 2^(m_i - max m)); empty sequences get zeros and -inf, ones longer than their table NaN.
struct JoinArgs {
    const int32_t *lens;
    const int4 *desc;       // [n_seqs][n_pairs]: first CTA, its slot, last CTA, 1 if split
    const float2 *ml;       // [CTAs][2][cols]
    const float *o;         // [CTAs][2][cols][D]
    int64_t capacity;
    int n_pairs, cols, D, max_ctas;
};

int attn_check_io(const char *who, int B, int H, const void *q, int64_t qs, int64_t qh, void *out, int64_t os, int64_t oh,
                  int od, int dtype, const int32_t *lens, float scale);

}  // namespace hx
