// hx_attn_decode.cu — attention of one new token a sequence over its pages (hxb_attn_decode_dev; the
// reference's engine/src/model.c:519-629 in another order of summation).
//
// o = sum_r p_r v_r, p = softmax(scale q . k_r). Each key and value is read once: a kv head's bytes
// are shared by the query heads of its group, so the work is n * 2 * row bytes of reading against
// 4 n H D operations, 1 to 16 a byte: HBM bounds it as long as the products ride on the matrix
// instructions (mma.sync m16n8k16; at 8 heads a kv head its rate is far above the reads', and the
// fifth-generation unit's 128-row tiles would be 1/16 full).
//
// Split. A unit is 64 positions of one kv head of one sequence. The grid is as many CTAs as fit
// the GPU at once, and CTA c takes units [c N / G, (c + 1) N / G) of all N, in the order (sequence, kv head,
// position), with N summed from the lengths on the device: the shares are equal whatever the lengths are, and a
// captured graph follows them. A CTA that does all of a (sequence, kv head) writes its output; otherwise it
// leaves (maximum, sum, output) in the scratch and the join kernel adds the pieces in order.
//
// A warp takes 16 positions of a unit. Keys and values go from HBM to registers in the order the
// matrix instructions want, without a stop in shared memory: S^T = K Q^T takes a 16-byte piece of a key row
// per lane as two steps' operands (the same permutation of the head's dims on both sides leaves the
// dot as it is); P^T is the accumulator transposed by movmatrix; O^T = V^T P^T takes 16-byte pieces of four
// value rows per lane, paired by byte permutes. With heads as the 8 columns nothing is padded for groups
// of 8. The next tile's rows are on their way while one is worked on: up to 8 KB a warp, 12 warps an SM.
//
// Measured: one bf16 sequence of 262147, 32 heads over 4 of 128: 95 us, 5.6 TB/s, 87 % of the copy rate (the split kernel
// alone 96 %); 48 Q8 sequences of up to 6011: 58.4 us, 3.2 TB/s, where a CTA has several pieces, each with its own queries, first
// loads and sums (some 12 us a call together), and half of the issue slots go to codes and weights; one f16 sequence of 777
// with 16 heads: 12 us on the GPU, 22 with the call.
//
// Bits. Matrix operands have the cache's type (Q8: f16, which holds the codes exactly; the scales are applied in f32, a
// value's to its weight). Queries of more bits are split into terms (bf16: 3 for f32, 2 for f16; f16: 2 for f32,
// after a power of two that puts the head's largest value at 2^13), and weights into 2 terms (bf16 for f32
// outputs: 3), since one rounding of each weight to the operand's type would be as large as the output's own.
// f16 weights carry 2^14, so that those down to 2^-38 of the largest count; Q8 ones are taken relative to the power of
// two of the largest value scale so far. Q8 keys go in as the codes themselves, one packed subtraction a pair from the form the
// bytes have under f16's exponent (1152 + code): taking 1152 times the query off the sums instead loses up to 2^-12
// of the score's terms where one large key channel leaves the others of its block codes of a few steps.
// The matrix instructions cut their sums off instead of rounding them, so that a long chain of them drifts: by 2^-18 over the
// tiles of 262147 positions. 16-bit outputs round far above that; f32 ones (WIDE) take each tile's products, and each 32 dims of a
// score, into a sum of their own and add those in f32.
#include "hx_attn.cuh"

#include <algorithm>

namespace hx {
namespace {

constexpr int AD_WARPS = 4, AD_THREADS = 32 * AD_WARPS;
// Units a piece's beginning and end count for in the division: 48 Q8 sequences of up to 6011: 61.5 us with 0, 60.1, 58.5 and 59.4
// with 1 to 3.
constexpr int AD_EXTRA = 2;

constexpr int ad_nj(int D) { return D <= 64 ? 1 : D <= 128 ? 2 : 4; }   // blocks of 64 dims, padded
// Resident CTAs an SM by registers. 16-bit rows of 128 dims: 12 warps with 168 registers each, 8 KB a warp under way (16 with
// 128 measured 68 % of the copy rate instead of 90 %). Q8 rows are half as long and cost more instructions a byte: 16
// warps (58.5 us a call on 48 sequences of up to 6011; 12: 61.4, 20: 87), whose 128 registers spill 16 bytes of stores and 24
// of loads at 128 dims (f32 queries at most 60 and 96, there and in four other instances, for 0 to 3 % of their time).
constexpr int ad_ctas(int cache, int nj, int nht) { return nj * nht <= 2 ? (cache == Q8 ? 4 : 3) : 2; }

// What the join needs beside SplitArgs.
struct JoinArgs {
    int cols, unit, ctas;   // heads of a pair's piece, positions a unit, CTAs of the split kernel
    int heads;              // heads a CTA of the join
    float off;              // exponent the weights carry
};

struct SplitArgs {
    KvView c;
    const int32_t *lens;
    const void *q;
    void *out;
    float *lse;
    int64_t qs, qh, os, oh;
    int H, group, passes, dtype, D;
    float sc2;              // scale * log2(e)
    float2 *ml;             // [CTAs][2][columns]: maximum (log2 domain), sum
    float *o;               // [CTAs][2][columns][D]
};

// ------------------------------------------------------------------------------------------- the split kernel

__device__ __forceinline__ uint32_t trans8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// Bytes 0, 1 (HI: 2, 3) of codes as an f16 pair: a byte with its sign bit flipped under 0x64 is 1152 + code, less 1152.
template <bool HI>
__device__ __forceinline__ uint32_t codes2(uint32_t flipped) {
    const uint32_t x = __byte_perm(flipped, 0x64646464u, HI ? 0x4342 : 0x4140), off = 0x64806480u;
    const __half2 r = __hsub2(reinterpret_cast<const __half2 &>(x), reinterpret_cast<const __half2 &>(off));
    return reinterpret_cast<const uint32_t &>(r);
}

template <int CACHE, int NTQ, int NTP, int NJ, int NHT>
struct SplitShape {
    static constexpr int UNIT = AD_WARPS * 16;
    static constexpr int COLS = 8 * NHT;
    static constexpr int OROW = 64 * NJ + 4;                       // floats between heads in the merge buffer
    static constexpr size_t Q_BYTES = (size_t)NTQ * NHT * 2 * NJ * 32 * 16;
    static constexpr size_t SMEM = Q_BYTES + (size_t)AD_WARPS * COLS * OROW * 4;
};

template <int CACHE, int NTQ, int NTP, int NJ, int NHT>
__global__ void __launch_bounds__(AD_THREADS, ad_ctas(CACHE, NJ, NHT)) k_attn_split(const __grid_constant__ SplitArgs a) {
    using Sh = SplitShape<CACHE, NTQ, NTP, NJ, NHT>;
    constexpr int UNIT = Sh::UNIT, COLS = Sh::COLS;
    constexpr int OT = CACHE == BF16 ? BF16 : F16;   // the operands' type
    constexpr float POFF = OT == F16 ? 14.0f : 0.0f;
    constexpr bool WIDE = NTQ == (CACHE == BF16 ? 3 : 2);   // f32 queries and outputs: sums of products rounded to nearest, see above
    extern __shared__ __align__(16) uint8_t smem[];
    uint4 *qs = reinterpret_cast<uint4 *>(smem);                    // [term][column tile][32-dim step][lane]
    float *mrg = reinterpret_cast<float *>(smem + Sh::Q_BYTES);     // [warp][column][OROW]
    __shared__ int64_t scan[AD_WARPS];
    __shared__ float wm[AD_WARPS][COLS], wl[AD_WARPS][COLS], qfac[COLS];

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int D = a.D, chunks = D / 8, n_pairs = a.c.Hkv * a.passes;
    pdl_trigger();

    // my share of the units
    int b;
    int64_t cur, end, acc, total;
    int ctas;
    if (!my_units<AD_THREADS>(a.c, a.lens, UNIT, AD_EXTRA, n_pairs, blockIdx.x, gridDim.x, scan, b, acc, cur, end, total, ctas)) return;
    const int64_t first_unit = cur;
    int nw = work_of(a.c, a.lens, b, UNIT, AD_EXTRA);
    const int64_t into = cur - acc * n_pairs;
    int pi = into <= 0xffffffffll ? (int)((uint32_t)into / (uint32_t)nw) : (int)(into / nw), at = (int)(into - (int64_t)pi * nw);

    for (int step; cur < end; cur += step, at = 0, pi++) {
        if (pi == n_pairs) {
            pi = 0;
            do nw = work_of(a.c, a.lens, ++b, UNIT, AD_EXTRA);
            while (nw == 0);
        }
        step = (int)min((int64_t)(nw - at), end - cur);
        const int n = a.lens[b], u = max(at - AD_EXTRA, 0), nseg = at + step - AD_EXTRA - u;
        if (nseg <= 0) continue;
        const int kvh = pi / a.passes, h0 = kvh * a.group + (pi - kvh * a.passes) * COLS;
        const int nh = min(COLS, (kvh + 1) * a.group - h0);

        // pages of the warp's tiles, asked for a tile ahead of their rows: one, or a lane's own where pages are under 16
        auto page_of = [&](int i) {
            const int tok = (u + i) * UNIT + warp * 16 + (a.c.pt_log2 >= 4 ? 0 : (lane & 15));
            return i < nseg && tok < n ? a.c.table[(int64_t)b * a.c.table_stride + (tok >> a.c.pt_log2)] : -1;
        };
        // row of position tok + rel of this kv head, -1: none
        auto row_at = [&](int page, int tok, int rel) -> int64_t {
            int pg = page;
            if (a.c.pt_log2 < 4) pg = __shfl_sync(0xffffffffu, page, rel);
            if (tok + rel >= n || (uint32_t)pg >= (uint64_t)a.c.n_pages) return -1;
            return (((int64_t)pg * a.c.Hkv + kvh) << a.c.pt_log2) + ((tok + rel) & ((1 << a.c.pt_log2) - 1));
        };

        constexpr int KW = CACHE == Q8 ? NJ : 2 * NJ, ES = CACHE == Q8 ? 1 : 2;
        uint4 kr[2][KW];
        float ks[2][CACHE == Q8 ? NJ : 1], vs[2][CACHE == Q8 ? NJ : 1];
        uint32_t vr[4][NJ][CACHE == Q8 ? 2 : 4];
        bool dead[2];     // a position in range without a row
        // A tile with all its positions in one page and heads of 64 NJ dims needs no checks: one address a row block. Rows of a
        // page lie D elements apart; *_lane is where a lane reads in them.
        const bool whole_d = D == 64 * NJ && a.c.pt_log2 >= 4;
        const uint32_t k_lane = (g * D) * ES + 16 * t, v_lane = (2 * t * D) * ES + g * (8 * ES);
        auto plain_tile = [&](int pg, int i) {
            return whole_d && (u + i) * UNIT + warp * 16 + 16 <= n && (uint32_t)pg < (uint64_t)a.c.n_pages;
        };
        auto block_at = [&](int page, int tok) { return (((int64_t)page * a.c.Hkv + kvh) << a.c.pt_log2) + (tok & ((1 << a.c.pt_log2) - 1)); };

        auto load_k = [&](int pg, int i, bool plain) {
            const int tok = (u + i) * UNIT + warp * 16;
            if (plain) {
                const int64_t row = block_at(pg, tok);
                const uint8_t *p = static_cast<const uint8_t *>(a.c.k) + row * (D * ES) + k_lane;
#pragma unroll
                for (int r = 0; r < 2; r++) {
                    dead[r] = false;
#pragma unroll
                    for (int j = 0; j < KW; j++) kr[r][j] = __ldg(reinterpret_cast<const uint4 *>(p + r * 8 * 64 * NJ * ES) + 4 * j);
                }
                if constexpr (CACHE == Q8) {
                    const float *kp = a.c.ks + (row + g) * NJ, *vp = a.c.vs + (row + g) * NJ;
#pragma unroll
                    for (int r = 0; r < 2; r++)
#pragma unroll
                        for (int j = 0; j < NJ; j++) ks[r][j] = __ldg(kp + r * 8 * NJ + j), vs[r][j] = __ldg(vp + r * 8 * NJ + j);
                }
                return;
            }
#pragma unroll
            for (int r = 0; r < 2; r++) {
                const int64_t row = row_at(pg, tok, g + 8 * r);
                dead[r] = row < 0 && tok + g + 8 * r < n;
                const uint8_t *p = static_cast<const uint8_t *>(a.c.k) + row * D * ES;
#pragma unroll
                for (int j = 0; j < KW; j++) {
                    const bool on = row >= 0 && (CACHE == Q8 ? 64 * j < D : 4 * j + t < chunks);
                    kr[r][j] = on ? __ldg(reinterpret_cast<const uint4 *>(p) + 4 * j + t) : make_uint4(0, 0, 0, 0);
                }
                if constexpr (CACHE == Q8) {
#pragma unroll
                    for (int j = 0; j < NJ; j++) {
                        const bool on = row >= 0 && 64 * j < D;
                        ks[r][j] = on ? __ldg(a.c.ks + row * (D / KV_BLOCK) + j) : 0.0f;
                        vs[r][j] = on ? __ldg(a.c.vs + row * (D / KV_BLOCK) + j) : 0.0f;
                    }
                }
            }
        };
        auto load_v = [&](int pg, int i, bool plain) {
            const int tok = (u + i) * UNIT + warp * 16;
            const uint8_t *base = static_cast<const uint8_t *>(a.c.v) + (plain ? block_at(pg, tok) * (D * ES) + v_lane : 0);
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int rel = (r & 1) + 8 * (r >> 1);
                const int64_t row = plain ? 0 : row_at(pg, tok, 2 * t + rel);
                const uint8_t *p = plain ? base + rel * 64 * NJ * ES : static_cast<const uint8_t *>(a.c.v) + row * D * ES + g * (8 * ES);
#pragma unroll
                for (int j = 0; j < NJ; j++) {
                    const bool on = plain || (row >= 0 && g + 8 * j < chunks);
                    if constexpr (CACHE == Q8) {
                        const uint2 x = on ? __ldg(reinterpret_cast<const uint2 *>(p) + 8 * j) : make_uint2(0, 0);
                        vr[r][j][0] = x.x, vr[r][j][1] = x.y;
                    } else {
                        const uint4 x = on ? __ldg(reinterpret_cast<const uint4 *>(p) + 8 * j) : make_uint4(0, 0, 0, 0);
                        vr[r][j][0] = x.x, vr[r][j][1] = x.y, vr[r][j][2] = x.z, vr[r][j][3] = x.w;
                    }
                }
            }
        };

        int pg = page_of(0), pg_next;
        bool plain = plain_tile(pg, 0);
        if (plain) load_k(pg, 0, true), load_v(pg, 0, true);
        else load_k(pg, 0, false), load_v(pg, 0, false);
        pg_next = page_of(1);

        // queries into shared memory as the products' column operands: a warp a head, a lane eight dims
        for (int h = warp; h < COLS; h += AD_WARPS) {
            float x[8] = {};
            if (h < nh && lane < chunks) {
                const int64_t at = b * a.qs + (int64_t)(h0 + h) * a.qh + lane * 8;
#pragma unroll
                for (int i = 0; i < 8; i++) x[i] = io_load(a.q, a.dtype, at + i);
            }
            float fac = a.sc2;
            if constexpr (OT == F16) {
                float m = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; i++) m = fmaxf(m, fabsf(x[i]));
#pragma unroll
                for (int o = 16; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
                const int k = f16_lift(m);
#pragma unroll
                for (int i = 0; i < 8; i++) x[i] = __fmul_rn(x[i], pow2i(k));
                fac = __fmul_rn(fac, pow2i(-k));
            }
            if (lane == 0) qfac[h] = fac;
            if (lane < 8 * NJ) {
                const int step = CACHE == Q8 ? 2 * (lane >> 3) + (lane & 1) : lane >> 2, tt = CACHE == Q8 ? (lane & 7) >> 1 : lane & 3;
#pragma unroll
                for (int k = 0; k < NTQ; k++) {
                    uint4 w;
                    w.x = take_pair<OT>(x[0], x[1]), w.y = take_pair<OT>(x[2], x[3]);
                    w.z = take_pair<OT>(x[4], x[5]), w.w = take_pair<OT>(x[6], x[7]);
                    qs[((k * NHT + (h >> 3)) * 2 * NJ + step) * 32 + (h & 7) * 4 + tt] = w;
                }
            }
        }
        __syncthreads();
        float fac[NHT][2];
        int ve[CACHE == Q8 ? NJ : 1] = {};      // exponents of the largest value scales so far
#pragma unroll
        for (int c = 0; c < NHT; c++) fac[c][0] = qfac[8 * c + 2 * t], fac[c][1] = qfac[8 * c + 2 * t + 1];

        float o[NHT][NJ][4][4] = {};
        float m[NHT][2], l[NHT][2];
#pragma unroll
        for (int c = 0; c < NHT; c++) m[c][0] = m[c][1] = -kv_inf(), l[c][0] = l[c][1] = 0.0f;

        // The next tile's keys are asked for once this one's scores are formed, its values after this one's.
        for (int i = 0; i < nseg; i++) {
            const int tok = (u + i) * UNIT + warp * 16, pgv = pg_next;
            const bool more = i + 1 < nseg, next_plain = more && plain_tile(pg_next, i + 1);
            // S^T = K Q^T
            float s[NHT][4];
#pragma unroll
            for (int c = 0; c < NHT; c++) {
                s[c][0] = s[c][1] = s[c][2] = s[c][3] = 0.0f;
                if constexpr (CACHE == Q8) {
#pragma unroll
                    for (int j = 0; j < NJ; j++) {
                        float p[4] = {};
                        const uint32_t w0[4] = {kr[0][j].x, kr[0][j].y, kr[0][j].z, kr[0][j].w};
                        const uint32_t w1[4] = {kr[1][j].x, kr[1][j].y, kr[1][j].z, kr[1][j].w};
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const uint32_t f0 = w0[e] ^ 0x80808080u, f1 = w1[e] ^ 0x80808080u;
                            const uint32_t a0 = codes2<false>(f0), a1 = codes2<false>(f1), a2 = codes2<true>(f0), a3 = codes2<true>(f1);
#pragma unroll
                            for (int k = NTQ - 1; k >= 0; k--) {
                                const uint4 q = qs[((k * NHT + c) * 2 * NJ + 2 * j + (e >> 1)) * 32 + lane];
                                mma16<OT>(p, a0, a1, a2, a3, e & 1 ? q.z : q.x, e & 1 ? q.w : q.y);
                            }
                        }
                        s[c][0] = __fmaf_rn(p[0], ks[0][j], s[c][0]);
                        s[c][1] = __fmaf_rn(p[1], ks[0][j], s[c][1]);
                        s[c][2] = __fmaf_rn(p[2], ks[1][j], s[c][2]);
                        s[c][3] = __fmaf_rn(p[3], ks[1][j], s[c][3]);
                    }
                } else {
                    float rest[4] = {};      // WIDE: the lower terms' products, too small for their truncation to matter
#pragma unroll
                    for (int j = 0; j < 2 * NJ; j++) {
                        float first[4] = {};
#pragma unroll
                        for (int k = NTQ - 1; k >= 0; k--) {
                            const uint4 q = qs[((k * NHT + c) * 2 * NJ + j) * 32 + lane];
                            float(&to)[4] = WIDE ? (k == 0 ? first : rest) : s[c];
                            mma16<OT>(to, kr[0][j].x, kr[1][j].x, kr[0][j].y, kr[1][j].y, q.x, q.y);
                            mma16<OT>(to, kr[0][j].z, kr[1][j].z, kr[0][j].w, kr[1][j].w, q.z, q.w);
                        }
                        if constexpr (WIDE)
#pragma unroll
                            for (int e = 0; e < 4; e++) s[c][e] = __fadd_rn(s[c][e], first[e]);
                    }
                    if constexpr (WIDE)
#pragma unroll
                        for (int e = 0; e < 4; e++) s[c][e] = __fadd_rn(s[c][e], rest[e]);
                }
            }
            // scores in the log2 domain; positions past the end have no weight, one without a row has no value
#pragma unroll
            for (int c = 0; c < NHT; c++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    s[c][e] = __fmul_rn(s[c][e], fac[c][e & 1]);
                    if (!plain) s[c][e] = dead[e >> 1] ? kv_nan() : tok + g + 8 * (e >> 1) < n ? s[c][e] : -kv_inf();
                }
            float pv[2][CACHE == Q8 ? NJ : 1];   // the values' scales of this tile, below 2 by the power of two that O carries
            if constexpr (CACHE == Q8) {
#pragma unroll
                for (int j = 0; j < NJ; j++) {
                    uint32_t top = 0;
#pragma unroll
                    for (int r = 0; r < 2; r++) {
                        const uint32_t bits = __float_as_uint(vs[r][j]);
                        top = max(top, bits < 0x7f800000u ? bits : 0u);
                    }
                    const int e = (int)(__reduce_max_sync(0xffffffffu, top) >> 23);
                    if (e > ve[j]) {      // the same in every lane
                        const float f = ve[j] == 0 ? 0.0f : exp2_fast((float)(ve[j] - e));
#pragma unroll
                        for (int c = 0; c < NHT; c++)
#pragma unroll
                            for (int k = 0; k < 4; k++)
#pragma unroll
                                for (int x = 0; x < 4; x++) o[c][j][k][x] = __fmul_rn(o[c][j][k][x], f);
                        ve[j] = e;
                    }
                    const float inv = __uint_as_float((uint32_t)max(254 - ve[j], 1) << 23);
#pragma unroll
                    for (int r = 0; r < 2; r++) pv[r][j] = ve[j] == 0 ? vs[r][j] : __fmul_rn(vs[r][j], inv);
                }
            }
            if (next_plain) load_k(pgv, i + 1, true);
            else if (more) load_k(pgv, i + 1, false);
            pg_next = page_of(i + 2);

            // running maximum and sum; the earlier sums fade together
#pragma unroll
            for (int c = 0; c < NHT; c++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    float x = fmaxf(m[c][e], fmaxf(s[c][e], s[c][e + 2]));
#pragma unroll
                    for (int w = 4; w <= 16; w <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, w));
                    const float base = x == -kv_inf() ? 0.0f : x, shift = __fsub_rn(base, POFF);
                    const float fade = exp2_fast(__fsub_rn(m[c][e], base));
                    s[c][e] = exp2_fast(__fsub_rn(s[c][e], shift));
                    s[c][e + 2] = exp2_fast(__fsub_rn(s[c][e + 2], shift));
                    l[c][e] = __fmaf_rn(l[c][e], fade, __fadd_rn(s[c][e], s[c][e + 2]));
                    m[c][e] = x;
                    if (!__all_sync(0xffffffffu, fade == 1.0f)) {
#pragma unroll
                        for (int j = 0; j < NJ; j++)
#pragma unroll
                            for (int k = 0; k < 4; k++) o[c][j][k][e] = __fmul_rn(o[c][j][k][e], fade), o[c][j][k][e + 2] = __fmul_rn(o[c][j][k][e + 2], fade);
                    }
                }

            // O^T += V^T P^T
            uint32_t bp[NHT][CACHE == Q8 ? NJ : 1][NTP][2];
#pragma unroll
            for (int c = 0; c < NHT; c++)
#pragma unroll
                for (int j = 0; j < (CACHE == Q8 ? NJ : 1); j++) {
                    float x[4] = {s[c][0], s[c][1], s[c][2], s[c][3]};
                    if constexpr (CACHE == Q8) {
                        x[0] = __fmul_rn(x[0], pv[0][j]), x[1] = __fmul_rn(x[1], pv[0][j]);
                        x[2] = __fmul_rn(x[2], pv[1][j]), x[3] = __fmul_rn(x[3], pv[1][j]);
                    }
#pragma unroll
                    for (int k = 0; k < NTP; k++) {
                        bp[c][j][k][0] = trans8x8(take_pair<OT>(x[0], x[1]));
                        bp[c][j][k][1] = trans8x8(take_pair<OT>(x[2], x[3]));
                    }
                }
#pragma unroll
            for (int j = 0; j < NJ; j++)
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    uint32_t a0, a1, a2, a3;
                    if constexpr (CACHE == Q8) {
                        const uint32_t w0 = __byte_perm(vr[0][j][k >> 1], vr[1][j][k >> 1], k & 1 ? 0x7362 : 0x5140) ^ 0x80808080u;
                        const uint32_t w1 = __byte_perm(vr[2][j][k >> 1], vr[3][j][k >> 1], k & 1 ? 0x7362 : 0x5140) ^ 0x80808080u;
                        a0 = codes2<false>(w0), a1 = codes2<true>(w0), a2 = codes2<false>(w1), a3 = codes2<true>(w1);
                    } else {
                        a0 = __byte_perm(vr[0][j][k], vr[1][j][k], 0x5410), a1 = __byte_perm(vr[0][j][k], vr[1][j][k], 0x7632);
                        a2 = __byte_perm(vr[2][j][k], vr[3][j][k], 0x5410), a3 = __byte_perm(vr[2][j][k], vr[3][j][k], 0x7632);
                    }
#pragma unroll
                    for (int c = 0; c < NHT; c++) {
                        float tile[4] = {};
                        float(&to)[4] = WIDE ? tile : o[c][j][k];
#pragma unroll
                        for (int x = NTP - 1; x >= 0; x--)
                            mma16<OT>(to, a0, a1, a2, a3, bp[c][CACHE == Q8 ? j : 0][x][0], bp[c][CACHE == Q8 ? j : 0][x][1]);
                        if constexpr (WIDE)
#pragma unroll
                            for (int e = 0; e < 4; e++) o[c][j][k][e] = __fadd_rn(o[c][j][k][e], tile[e]);
                    }
                }
            if (next_plain) load_v(pgv, i + 1, true);
            else if (more) load_v(pgv, i + 1, false);
            plain = next_plain;
        }

        // the warps' pieces into one
#pragma unroll
        for (int c = 0; c < NHT; c++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
#pragma unroll
                for (int w = 4; w <= 16; w <<= 1) l[c][e] = __fadd_rn(l[c][e], __shfl_xor_sync(0xffffffffu, l[c][e], w));
                if (g == 0) wm[warp][8 * c + 2 * t + e] = m[c][e], wl[warp][8 * c + 2 * t + e] = l[c][e];
            }
        __syncthreads();
#pragma unroll
        for (int c = 0; c < NHT; c++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int h = 8 * c + 2 * t + e;
                float x = wm[0][h];
#pragma unroll
                for (int w = 1; w < AD_WARPS; w++) x = fmaxf(x, wm[w][h]);
                const float fade = exp2_fast(__fsub_rn(m[c][e], x == -kv_inf() ? 0.0f : x));
                float *dst = mrg + (warp * COLS + h) * Sh::OROW;
#pragma unroll
                for (int j = 0; j < NJ; j++)
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        float x0 = __fmul_rn(o[c][j][k][e], fade), x1 = __fmul_rn(o[c][j][k][e + 2], fade);
                        if constexpr (CACHE == Q8) {
                            const float f = ve[j] == 0 ? 1.0f : __uint_as_float((uint32_t)ve[j] << 23);
                            x0 = __fmul_rn(x0, f), x1 = __fmul_rn(x1, f);
                        }
                        *reinterpret_cast<float2 *>(dst + 64 * j + 8 * g + 2 * k) = make_float2(x0, x1);
                    }
            }
        __syncthreads();
        const bool whole = nseg == nw - AD_EXTRA;
        const int slot = cur == first_unit ? 0 : 1;
        const int64_t piece = (int64_t)blockIdx.x * 2 + slot;
        for (int h = warp; h < nh; h += AD_WARPS) {
            float x = wm[0][h], sum = 0.0f;
#pragma unroll
            for (int w = 1; w < AD_WARPS; w++) x = fmaxf(x, wm[w][h]);
#pragma unroll
            for (int w = 0; w < AD_WARPS; w++) sum = __fmaf_rn(wl[w][h], exp2_fast(__fsub_rn(wm[w][h], x == -kv_inf() ? 0.0f : x)), sum);
            for (int d = lane; d < D; d += 32) {
                float v = mrg[h * Sh::OROW + d];
#pragma unroll
                for (int w = 1; w < AD_WARPS; w++) v = __fadd_rn(v, mrg[(w * COLS + h) * Sh::OROW + d]);
                if (whole) io_store(a.out, a.dtype, b * a.os + (int64_t)(h0 + h) * a.oh + d, sum == 0.0f ? 0.0f : __fdiv_rn(v, sum));
                else a.o[(piece * COLS + h) * D + d] = v;
            }
            if (lane == 0) {
                if (!whole) a.ml[piece * COLS + h] = make_float2(x, sum);
                else if (a.lse) a.lse[(int64_t)b * a.H + h0 + h] = lse_of(x, sum, POFF);
            }
        }
        __syncthreads();
    }
}

// ------------------------------------------------------------------------------------------- the join

constexpr int JOIN_THREADS = 512;

// The pieces of a pair that several CTAs worked on are added with weights 2^(m_i - max m), in a fixed order. A CTA takes
// `heads` heads of a pair: a thread four dims of one, every `groups`-th piece; then the groups are joined. Which pieces there
// are follows from the lengths, before the split kernel has ended; after it one round of loads is left. Empty
// sequences get zeros and -inf, ones longer than their table NaN.
__global__ void __launch_bounds__(JOIN_THREADS) k_attn_join(const __grid_constant__ SplitArgs a, const __grid_constant__ JoinArgs j) {
    __shared__ int64_t sums[JOIN_THREADS / 32][2];
    __shared__ float4 part[JOIN_THREADS];
    __shared__ float2 part_ml[JOIN_THREADS];
    const int b = blockIdx.y, tid = threadIdx.x, D = a.D, quads = D / 4, each = quads * j.heads, groups = JOIN_THREADS / each;
    const int nb = (j.cols + j.heads - 1) / j.heads, pair = blockIdx.x / nb, kvh = pair / a.passes, pass = pair - kvh * a.passes;
    const int gr = tid / each, col = (blockIdx.x - pair * nb) * j.heads + (tid - gr * each) / quads, qd = tid % quads;
    const int hg = pass * j.cols + col, h = kvh * a.group + hg;
    const bool live = gr < groups && col < j.cols && hg < a.group;
    const int n = a.lens[b], nu = units_of(a.c, a.lens, b, j.unit), n_pairs = a.c.Hkv * a.passes;
    int64_t before, all;
    work_sums<JOIN_THREADS>(a.c, a.lens, j.unit, AD_EXTRA, b, sums, before, all);
    Span sp = {};
    if (nu) sp = span_of(before * n_pairs + (int64_t)pair * (nu + AD_EXTRA), AD_EXTRA, nu, all * n_pairs, j.ctas);
    if (!nu || !sp.split()) {
        pdl_wait();      // no CTA ends before the split kernel has: the stream's next kernel waits for this one only
        if (nu || !live || gr) return;
        for (int k = 0; k < 4; k++) io_store(a.out, a.dtype, b * a.os + (int64_t)h * a.oh + 4 * qd + k, n <= 0 ? 0.0f : kv_nan());
        if (qd == 0 && a.lse) a.lse[(int64_t)b * a.H + h] = n <= 0 ? -kv_inf() : kv_nan();
        return;
    }
    const int count = sp.last - sp.first + 1;
    pdl_wait();
    Joined<4> mine;
    if (live)
#pragma unroll 8
        for (int i = gr; i < count; i += groups) {
            const int64_t at = ((int64_t)(sp.first + i) * 2 + (i == 0 ? sp.slot : 0)) * j.cols + col;
            const float2 ml = __ldcg(a.ml + at);
            const float4 x = __ldcg(reinterpret_cast<const float4 *>(a.o + at * D) + qd);
            const float v[4] = {x.x, x.y, x.z, x.w};
            mine.add(ml, v);
        }
    if (groups > 1) {
        part[tid] = make_float4(mine.o[0], mine.o[1], mine.o[2], mine.o[3]), part_ml[tid] = make_float2(mine.m, mine.l);
        __syncthreads();
        if (gr == 0)
#pragma unroll 1
            for (int k = 1; k < min(groups, count); k++) {
                const float4 x = part[k * each + tid];
                const float v[4] = {x.x, x.y, x.z, x.w};
                mine.add(part_ml[k * each + tid], v);
            }
    }
    if (!live || gr) return;
#pragma unroll 1
    for (int k = 0; k < 4; k++) {
        io_store(a.out, a.dtype, b * a.os + (int64_t)h * a.oh + 4 * qd + k, mine.l == 0.0f ? 0.0f : __fdiv_rn(mine.o[0], mine.l));
        mine.o[0] = mine.o[1], mine.o[1] = mine.o[2], mine.o[2] = mine.o[3];
    }
    if (qd == 0 && a.lse) a.lse[(int64_t)b * a.H + h] = lse_of(mine.m, mine.l, j.off);
}

// ------------------------------------------------------------------------------------------- host side

struct Plan {
    int nj, nht, passes, ctas;
    size_t ml, o, bytes;
};

Plan plan_of(const hxb_kv_cache *c, int H) {
    Plan p = {};
    const int group = H / c->n_kv_heads;
    p.nj = ad_nj(c->head_dim);
    // 16 columns halve the reads of groups over 8; at 256 dims their sums do not fit the registers
    p.nht = group > 8 && p.nj <= 2 ? 2 : 1;
    p.passes = (group + 8 * p.nht - 1) / (8 * p.nht);
    p.ctas = ATTN_SMS * ad_ctas(c->dtype, p.nj, p.nht);
    const int most = ATTN_SMS * std::max(ad_ctas(Q8, p.nj, p.nht), ad_ctas(BF16, p.nj, p.nht));      // one size for every type
    p.ml = (size_t)most * 2 * 8 * p.nht * sizeof(float2);
    p.o = (size_t)most * 2 * 8 * p.nht * c->head_dim * sizeof(float);
    p.bytes = p.ml + p.o;
    return p;
}

template <int CACHE, int NTQ, int NTP, int NJ, int NHT>
cudaError_t split(const SplitArgs &a, int ctas, cudaStream_t s) {
    using Sh = SplitShape<CACHE, NTQ, NTP, NJ, NHT>;
    auto k = k_attn_split<CACHE, NTQ, NTP, NJ, NHT>;
    static_assert(Sh::SMEM <= 46 * 1024, "dynamic shared memory without an opt-in, beside the kernel's own");
    // more heads a join CTA while there are two CTAs an SM: with many sequences the pieces of each are few
    int heads = 1;
    const int pairs = a.c.Hkv * a.passes;
    while (heads < Sh::COLS && 2 * heads * (a.D / 4) <= JOIN_THREADS &&
           (int64_t)pairs * (std::min(a.group, Sh::COLS) / (2 * heads)) * a.c.n_seqs >= 2 * ATTN_SMS)
        heads *= 2;
    const JoinArgs j = {Sh::COLS, Sh::UNIT, ctas, heads, CACHE == BF16 ? 0.0f : 14.0f};
    const cudaError_t e = launch_pdl(false, k, dim3(ctas), dim3(AD_THREADS), Sh::SMEM, s, a);
    if (e != cudaSuccess) return e;
    return launch_pdl(true, k_attn_join, dim3(pairs * ((Sh::COLS + heads - 1) / heads), a.c.n_seqs), dim3(JOIN_THREADS), 0, s, a, j);
}

template <int CACHE, int NTQ, int NTP>
cudaError_t split_shape(const SplitArgs &a, const Plan &p, cudaStream_t s) {
    if (p.nj == 1) return p.nht == 1 ? split<CACHE, NTQ, NTP, 1, 1>(a, p.ctas, s) : split<CACHE, NTQ, NTP, 1, 2>(a, p.ctas, s);
    if (p.nj == 2) return p.nht == 1 ? split<CACHE, NTQ, NTP, 2, 1>(a, p.ctas, s) : split<CACHE, NTQ, NTP, 2, 2>(a, p.ctas, s);
    return split<CACHE, NTQ, NTP, 4, 1>(a, p.ctas, s);
}

}  // namespace

int attn_check_io(const char *who, int B, int H, const void *q, int64_t qs, int64_t qh, void *out, int64_t os, int64_t oh,
                  int od, int dtype, const int32_t *lens, float scale) {
    const size_t size = dtype == F32 ? 4 : 2;
    auto off = [](const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n != 0; };
    if (!q || !out || !lens) return attn_fail(HXB_E_ARG, "%s: null pointer", who);
    if (q == out) return attn_fail(HXB_E_ARG, "%s: not in place (out is q)", who);
    if (off(q, size) || off(out, size) || off(lens, 4)) return attn_fail(HXB_E_ARG, "%s: pointer not aligned to its elements", who);
    if (qs < 0 || qh < 0 || os < 0 || oh < 0 || rows_overlap(B, os, H, oh, od))
        return attn_fail(HXB_E_ARG, "%s: bad strides", who);
    if (!(fabsf(scale) < INFINITY)) return attn_fail(HXB_E_ARG, "%s: scale is not finite", who);
    return HXB_OK;
}

}  // namespace hx

using namespace hx;

extern "C" HXB_API size_t hxb_attn_decode_workspace(const hxb_kv_cache *c, int n_heads) {
    if (!c || c->n_seqs < 0 || c->n_kv_heads < 1 || n_heads < 1 || n_heads % c->n_kv_heads || c->head_dim < 1) return 0;
    return plan_of(c, n_heads).bytes;
}

extern "C" HXB_API int hxb_attn_decode_dev(const hxb_kv_cache *c, const int32_t *lens, const void *q, int64_t q_stride,
                                           int64_t q_head_stride, int n_heads, int dtype, float scale, void *out,
                                           int64_t out_stride, int64_t out_head_stride, float *lse, void *ws,
                                           size_t ws_bytes, void *stream) {
    const char *who = "attn_decode";
    SplitArgs a = {};
    int rc = kv_view(c, who, false, &a.c);
    if (rc != HXB_OK) return rc;
    if (c->head_dim % 16 || c->head_dim > 256)
        return attn_fail(HXB_E_UNSUPPORTED, "%s: head_dim %d (a multiple of 16 up to 256)", who, c->head_dim);
    if (n_heads < 1 || n_heads > 65535 || n_heads % c->n_kv_heads || c->n_seqs > 65535)
        return attn_fail(HXB_E_ARG, "%s: %d heads over %d kv heads, %d sequences (up to 65535)", who, n_heads, c->n_kv_heads, c->n_seqs);
    if (dtype != F32 && dtype != F16 && dtype != BF16) return attn_fail(HXB_E_ARG, "%s: bad dtype", who);
    if (c->n_seqs == 0) return HXB_OK;
    rc = attn_check_io(who, c->n_seqs, n_heads, q, q_stride, q_head_stride, out, out_stride, out_head_stride, c->head_dim, dtype, lens, scale);
    if (rc != HXB_OK) return rc;
    if (reinterpret_cast<uintptr_t>(lse) % 4) return attn_fail(HXB_E_ARG, "%s: pointer not aligned to its elements", who);
    const Plan p = plan_of(c, n_heads);
    if (!ws || reinterpret_cast<uintptr_t>(ws) % 16 || ws_bytes < p.bytes)
        return attn_fail(HXB_E_ARG, "%s: workspace of %zu bytes, 16-byte aligned, needed", who, p.bytes);
    a.lens = lens, a.q = q, a.out = out, a.lse = lse, a.qs = q_stride, a.qh = q_head_stride, a.os = out_stride, a.oh = out_head_stride;
    a.H = n_heads, a.group = n_heads / c->n_kv_heads, a.passes = p.passes, a.dtype = dtype, a.D = c->head_dim;
    a.sc2 = scale * 1.44269504088896f;
    uint8_t *w = static_cast<uint8_t *>(ws);
    a.ml = reinterpret_cast<float2 *>(w), a.o = reinterpret_cast<float *>(w + p.ml);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    cudaError_t e;
    if (c->dtype == F16) e = dtype == F32 ? split_shape<F16, 2, 2>(a, p, s) : split_shape<F16, 1, 2>(a, p, s);
    else if (c->dtype == BF16)
        e = dtype == F32 ? split_shape<BF16, 3, 3>(a, p, s) : dtype == F16 ? split_shape<BF16, 2, 2>(a, p, s) : split_shape<BF16, 1, 2>(a, p, s);
    else e = dtype == F32 ? split_shape<Q8, 2, 2>(a, p, s) : split_shape<Q8, 1, 2>(a, p, s);
    if (e != cudaSuccess) return attn_fail(HXB_E_DEVICE, "%s: %s", who, cudaGetErrorString(e));
    return HXB_OK;
}
