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

// The share [cur, end) of CTA `cta` of `grid` in the N = n_pairs * sum_b units_of(b) units, laid out sequence by
// sequence, pair by pair: the sequence of unit cur and the sum of the units of the sequences before it. False
// without a share. ctas: the CTAs that have one (the first min(grid, N)). Every thread of the CTA calls it;
// scan: one word a warp.
template <int THREADS>
__device__ __forceinline__ bool my_units(const KvView &c, const int32_t *lens, int unit, int n_pairs, int cta, int grid,
                                         int64_t *scan, int &b, int64_t &before, int64_t &cur, int64_t &end,
                                         int64_t &total, int &ctas) {
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
    ctas = (int)min((int64_t)grid, total);
    const int64_t start = base + upto - mine;             // units of the sequences before my chunk
    cur = end = 0;
    if (total) cur = cta * total / ctas, end = (cta + 1) * total / ctas;
    const bool none = cta >= ctas;
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

// Two f32 as a pair of 16-bit matrix operands of TYPE F16 or BF16 (x in the low half); what they leave stays in x, y.
template <int TYPE>
__device__ __forceinline__ uint32_t take_pair(float &x, float &y) {
    if constexpr (TYPE == F16) {
        const __half2 h = __floats2half2_rn(x, y);
        x = __fsub_rn(x, __low2float(h)), y = __fsub_rn(y, __high2float(h));
        return reinterpret_cast<const uint32_t &>(h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
        x = __fsub_rn(x, __low2float(h)), y = __fsub_rn(y, __high2float(h));
        return reinterpret_cast<const uint32_t &>(h);
    }
}

// d += A B, m16n8k16 on operands of TYPE F16 or BF16.
template <int TYPE>
__device__ __forceinline__ void mma16(float d[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (TYPE == F16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The power of two 2^k, as its exponent k, that brings a largest magnitude m to [2^13, 2^14), the upper part of f16's
// range; k <= 120, so that 2^k and 2^-k are normal, and 0 for m = 0 or not finite.
__device__ __forceinline__ int f16_lift(float m) {
    return m == 0.0f || !(m < kv_inf()) ? 0 : min(140 - (int)(__float_as_uint(m) >> 23), 120);
}
__device__ __forceinline__ float pow2i(int k) { return __uint_as_float((uint32_t)(127 + k) << 23); }

int attn_check_io(const char *who, int B, int H, const void *q, int64_t qs, int64_t qh, void *out, int64_t os, int64_t oh,
                  int od, int dtype, const int32_t *lens, float scale);

}  // namespace hx
