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

// N units in `ctas` shares that differ by at most one: the first N % ctas have one more.
struct Shares {
    int64_t each;
    int more;
    __device__ __forceinline__ Shares(int64_t total, int ctas) {
        if (total <= 0xffffffffll) each = (uint32_t)total / (uint32_t)ctas, more = (int)((uint32_t)total % (uint32_t)ctas);
        else each = total / ctas, more = (int)(total % ctas);
    }
    __device__ __forceinline__ int64_t start(int cta) const { return cta * each + min(cta, more); }
    __device__ __forceinline__ int of(int64_t unit) const {      // the share a unit is in
        const int64_t big = more * (each + 1);
        const int64_t n = unit < big ? unit : unit - big, d = unit < big ? each + 1 : each;
        const int q = ((n | d) >> 32) == 0 ? (int)((uint32_t)n / (uint32_t)d) : (int)(n / d);
        return unit < big ? q : more + q;
    }
};

// What a (sequence, pair) counts in the division: its units, and before them `extra` that stand for the beginning and the end of
// a CTA's piece of it (queries, sums out), so that a CTA with several pieces gets fewer units.
__device__ __forceinline__ int work_of(const KvView &c, const int32_t *lens, int b, int unit, int extra) {
    const int nu = units_of(c, lens, b, unit);
    return nu ? nu + extra : 0;
}

// The share [cur, end) of CTA `cta` of `grid` in the N = n_pairs * sum_b work_of(b) units, laid out sequence by
// sequence, pair by pair: the sequence of unit cur and the sum of the units of the sequences before it. False
// without a share. ctas: the CTAs that have one (the first min(grid, N)). Every thread of the CTA calls it;
// scan: one word a warp.
template <int THREADS>
__device__ __forceinline__ bool my_units(const KvView &c, const int32_t *lens, int unit, int extra, int n_pairs, int cta, int grid,
                                         int64_t *scan, int &b, int64_t &before, int64_t &cur, int64_t &end,
                                         int64_t &total, int &ctas) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, B = c.n_seqs;
    const int per = (B + THREADS - 1) / THREADS;
    int64_t mine = 0;
    for (int i = tid * per; i < min(B, (tid + 1) * per); i++) mine += work_of(c, lens, i, unit, extra);
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
    if (total) {
        const Shares sh(total, ctas);
        cur = sh.start(cta), end = sh.start(cta + 1);
    }
    const bool none = cta >= ctas;
    // the chunk that holds unit cur: the last one that starts at or before it
    const int chunk = __syncthreads_count(start * n_pairs <= cur) - 1;
    if (tid == chunk) scan[0] = start;
    __syncthreads();
    if (none) return false;
    b = chunk * per, before = scan[0];
    for (;;) {
        const int nw = work_of(c, lens, b, unit, extra);
        if ((before + nw) * n_pairs > cur) break;
        before += nw, b++;
    }
    return true;
}

// Where a (sequence, pair)'s work [unit0, unit0 + extra + nu) went, from the lengths alone: CTAs first .. last, each with one
// piece, in slot 0 but for the first CTA where the pair is not what it began with. One CTA: it wrote the result itself.
struct Span {
    int first, last, slot;
    __device__ __forceinline__ bool split() const { return first != last; }
};
__device__ __forceinline__ Span span_of(int64_t unit0, int extra, int nu, int64_t total, int grid) {
    const Shares sh(total, (int)min((int64_t)grid, total));
    Span s;
    s.first = sh.of(unit0 + extra), s.last = sh.of(unit0 + extra + nu - 1);
    s.slot = sh.start(s.first) >= unit0 ? 0 : 1;
    return s;
}
// The work of the sequences before b, and of all: the same sums my_units forms. Every thread of the CTA calls it.
template <int THREADS>
__device__ __forceinline__ void work_sums(const KvView &c, const int32_t *lens, int unit, int extra, int b, int64_t (*scratch)[2], int64_t &before, int64_t &all) {
    before = all = 0;
    for (int i = threadIdx.x; i < c.n_seqs; i += THREADS) {
        const int nw = work_of(c, lens, i, unit, extra);
        all += nw;
        if (i < b) before += nw;
    }
#pragma unroll
    for (int s = 16; s >= 1; s >>= 1) all += __shfl_xor_sync(0xffffffffu, all, s), before += __shfl_xor_sync(0xffffffffu, before, s);
    if (threadIdx.x % 32 == 0) scratch[threadIdx.x / 32][0] = before, scratch[threadIdx.x / 32][1] = all;
    __syncthreads();
    before = all = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; w++) before += scratch[w][0], all += scratch[w][1];
}

// A running softmax-weighted sum of pieces (maximum, sum, N values each): weights 2^(m_i - max m).
template <int N>
struct Joined {
    float m, l = 0.0f, o[N] = {};
    __device__ __forceinline__ Joined() : m(-kv_inf()) {}
    __device__ __forceinline__ void add(float2 ml, const float *x) {
        const float mx = fmaxf(m, ml.x), base = mx == -kv_inf() ? 0.0f : mx;
        const float f = exp2_fast(__fsub_rn(m, base)), w = exp2_fast(__fsub_rn(ml.x, base));
        l = __fmaf_rn(l, f, __fmul_rn(ml.y, w));
#pragma unroll
        for (int i = 0; i < N; i++) o[i] = __fmaf_rn(o[i], f, __fmul_rn(x[i], w));
        m = mx;
    }
};

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
