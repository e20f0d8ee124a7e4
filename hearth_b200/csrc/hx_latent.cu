// hx_latent.cu — absorbed latent attention of one new token a sequence (hxb_latent_decode_dev; the reference's
// engine/src/model.c:739-787 in another order of summation), in three launches chained by programmatic
// dependent launch:
//
//   k_latent_absorb  qa[b][h] = [sum_d q[d] w[h][d] | q's rotated part] into the scratch (f32; for a bf16 cache rounded to the
//                    products' operands); mma.sync, a warp 64 latent dims of a head for 32 sequences, weights straight
//                    into registers.
//   k_latent_core    softmax(scale qa C^T) C over the pages, on the fifth-generation tensor cores.
//   k_latent_expand  joins the core's pieces and multiplies by w's value rows.
//
// The core. One row of 576 values (1152 bytes) serves every head as key and as value: 2 (576 + 512) H operations for
// 1152 bytes, 121 a byte at 64 heads, about half of what the machine can do per byte read: HBM bounds it while the
// tensor cores run at half their rate, so they have to be fed by the fifth-generation unit. A CTA takes up to 64
// heads and a run of 64-position tiles (the shares of all CTAs are equal, as in hx_attn_decode.cu; with more
// heads, groups of CTAs take the same runs side by side and share the rows through L2):
//
//   S [heads x 64]    = Q [64 x 576] K^T          tcgen05 M 64, N 64: both from shared memory, row-major
//   P                 = 2^(S - ref) -> shared memory, a thread a head
//   O^T [512 x heads] += V^T [512 x 64] P^T       M 128 x 4, N heads: V is the K tile itself, read column-major
//
// With O transposed its 4 x 64 columns and two S buffers take 384 of the 512 tensor-memory columns at 64 heads (O
// itself, 64 rows high, would leave half of the lanes empty), and the tile in shared memory is used twice. Shared
// memory: Q 72 KB, two tiles of 72 KB, P 8 KB. Warps 0-3 softmax, 4 issues the scores' products, 5 the values', 6-13 load:
// 16-bit rows four warps for each of the two tiles, so that the one in flight never waits for the one at work. Rows
// are fetched by 16-byte asynchronous copies: they take any page size, and rows past the end arrive as zeros
// (an unused slot may hold NaN, and 0 x NaN would reach every sum); tensor-map boxes of 64 x 64 took longer.
//
// Measured (64 heads, 512 + 64 values a row, 128 + 128 a head): 32 sequences of up to 8191, bf16: 86 us, 204 MB of
// rows and 17 MB of weights, 2.6 TB/s; one of 1531: 26 us; 4 Q8 sequences of up to 65536 with 16 heads: 62 us. Of the 86 us
// absorb takes 7, the core 68 after it and expand 10 after that. A tile of the core takes some 4500 cycles
// (72 KB: 16 bytes a cycle and SM, the copy rate is 23): its buffer waits for scores (1500), softmax (1900) and half of
// the values' products (1300) before the next rows (3000 to 4000) may follow, and there is room for two buffers. Asking for
// the next rows in L2 ahead made it slower (106 us for 99), Q8 codes asked for over a tile's end too (73 us for 66:
// the proxy fence waits for loads under way).
//
// ref is the running maximum, moved only when a score passes it by 2^7 (O^T is then rescaled in tensor memory):
// the weights relative to it stay below 2^7 (f16 operands: 2^15, lifted by 2^8), and most tiles skip the rescale.
//
// Bits. Operands have the cache's type; Q8 rows are expanded to f16 (code x scale in f32, rounded once to 11 bits; bf16's 8
// would add an error as large as the output's own). f16 queries are lifted by a power of two a head. Weights
// go in as two terms for the same reason, the second into the tile's rotated part, which S no longer needs (32 sequences of up to
// 8191 in f16: 92.6 us, 89.7 with one term and an error of 1.5 times the plain form's instead of 1.3). Over a Q8 cache they have
// one f16 term: the rows' rounding is what shows there with f16 outputs (0.0004 to the plain form's 0.0002 in 32 bits;
// with a second term 0.0004 too, and 93.0 us for 88.6); with bf16 outputs neither does. Queries have one term: a second would
// take 72 KB of shared memory from the second tile (bf16: error 0.0020 to 0.0023, the outputs' own rounding 0.0017).
#include "hx_attn.cuh"

#include <algorithm>

namespace hx {
namespace {

constexpr int LT = 64;                  // positions a tile
constexpr int LH = 64;                  // heads a CTA (rows of S)
constexpr int SEG = LT * 128;           // 64 dims of 64 rows: a 128-byte swizzled block column
constexpr int SCORE_WARP = 4, LD_WARP0 = 6, LD_WARPS = 8;       // 0-3 softmax, 4 scores, 5 values, the others load
constexpr int CORE_WARPS = LD_WARP0 + LD_WARPS, CORE_THREADS = 32 * CORE_WARPS;
// 16-bit rows: four loading warps for each of the two tile buffers, so that one in flight never waits for the other. Q8: all
// eight for one tile after the other: expanding a tile takes four warps as long as both tiles' products.
template <int CACHE> constexpr int LD_GROUPS = CACHE == Q8 ? 1 : 2;
template <int CACHE> constexpr int LD_THREADS = 32 * LD_WARPS / LD_GROUPS<CACHE>;
constexpr float REF_SLACK = 7.0f;
// Tiles a run's beginning and end count for in the division (queries and sums of 64 heads take about as long): 32 sequences of up
// to 8191: 104.4 us with 0, 102.4, 100.0, 98.7, 99.2 and 100.9 with 1 to 5.
constexpr int CORE_EXTRA = 3;

struct LatentArgs {
    KvView c;
    const int32_t *lens;
    const void *q, *w;
    void *out;
    // [n_seqs][H][R + dr] f32; for a bf16 cache the products' bf16 operands in the first half of each row. A head whose work
    // one CTA did leaves its o, maximum and sum here.
    float *qa;
    float2 *ml;             // [CTAs][2][hp]
    float *o;               // [CTAs][2][hp][R]
    int *err;
    int64_t qs, qh, os, oh;
    int H, R, dr, dn, dv, passes, hp;   // hp heads a pass
    float sc2;
};

// ------------------------------------------------------------------------------------------- absorb

// Weights from HBM bound it (8.4 MB at 64 heads of 128 + 512, 1.3 us), in practice the round trips of a CTA: queries, then two
// batches of weights; 6.8 us for 32 sequences, 5.5 for one.
constexpr int AB_WARPS = 4, AB_ROWS = 32, AB_AHEAD = 4;

template <int T, bool ROUND>
__global__ void __launch_bounds__(32 * AB_WARPS) k_latent_absorb(const __grid_constant__ LatentArgs a) {
    __shared__ uint16_t qsm[AB_ROWS][256 + 8];
    const int nc = (a.R + 64 * AB_WARPS - 1) / (64 * AB_WARPS);
    const int h = blockIdx.x / nc, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int r0 = ((blockIdx.x - h * nc) * AB_WARPS + warp) * 64, b0 = blockIdx.y * AB_ROWS, rows = min(AB_ROWS, a.c.n_seqs - b0);
    pdl_trigger();
    if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *a.err = 0;
    const uint16_t *w = static_cast<const uint16_t *>(a.w) + (int64_t)h * (a.dn + a.dv) * a.R + r0 + 8 * g;
    auto fetch = [&](uint4 v[4], int d0) {
#pragma unroll
        for (int k = 0; k < 4; k++)
            v[k] = r0 < a.R && d0 < a.dn ? __ldg(reinterpret_cast<const uint4 *>(w + (int64_t)(d0 + 2 * t + (k & 1) + 8 * (k >> 1)) * a.R)) : make_uint4(0, 0, 0, 0);
    };
    uint4 pre[AB_AHEAD][4];      // weights on their way before the queries are staged, and that far ahead from then on
#pragma unroll
    for (int i = 0; i < AB_AHEAD; i++) fetch(pre[i], 16 * i);
    const uint16_t *q = static_cast<const uint16_t *>(a.q) + h * a.qh;
    constexpr int AB_EACH = AB_ROWS / AB_WARPS;      // rows a warp stages: all its loads before their stores
    auto row_at = [&](int r, int d, int lim) -> uint16_t {
        return warp + r * AB_WARPS < rows && d < lim ? __ldg(q + (b0 + warp + r * AB_WARPS) * a.qs + d) : 0;
    };
    const int row = a.R + a.dr;
    const bool rot = blockIdx.x == h * nc;      // the rotated parts, with the head's first CTA
    uint16_t xr[2][AB_EACH];
#pragma unroll
    for (int r = 0; r < AB_EACH; r++) xr[0][r] = rot ? row_at(r, a.dn + lane, a.dn + a.dr) : 0, xr[1][r] = rot ? row_at(r, a.dn + lane + 32, a.dn + a.dr) : 0;
#pragma unroll 1
    for (int d = lane; d < a.dn; d += 128) {
        uint16_t x[4][AB_EACH];
#pragma unroll
        for (int r = 0; r < AB_EACH; r++)
#pragma unroll
            for (int e = 0; e < 4; e++) x[e][r] = row_at(r, d + 32 * e, a.dn);
#pragma unroll
        for (int r = 0; r < AB_EACH; r++)
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (d + 32 * e < a.dn) qsm[warp + r * AB_WARPS][d + 32 * e] = x[e][r];
    }
    if (rot) {
#pragma unroll
        for (int r = 0; r < AB_EACH; r++)
#pragma unroll
            for (int e = 0; e < 2; e++)
                if (warp + r * AB_WARPS < rows && lane + 32 * e < a.dr) {
                    float *dst = a.qa + ((int64_t)(b0 + warp + r * AB_WARPS) * a.H + h) * row;
                    const int d = a.R + lane + 32 * e;
                    if constexpr (ROUND) reinterpret_cast<uint16_t *>(dst)[d] = xr[e][r];
                    else dst[d] = T == F16 ? f16_to_f32_hw(xr[e][r]) : bf16_to_f32(xr[e][r]);
                }
    }
    __syncthreads();
    if (r0 >= a.R) return;
    float acc[2][8][4] = {};
    // AB_AHEAD steps of 16 dims, each with registers of its own (moving a load's registers on would wait for it)
#pragma unroll 1
    for (int d0 = 0; d0 < a.dn; d0 += 16 * AB_AHEAD) {
#pragma unroll
        for (int j = 0; j < AB_AHEAD; j++) {
            const int d = d0 + 16 * j;
            if (d >= a.dn) break;
            uint32_t f[2][4];
#pragma unroll
            for (int m = 0; m < 2; m++)
#pragma unroll
                for (int k = 0; k < 4; k++)
                    f[m][k] = *reinterpret_cast<const uint32_t *>(&qsm[16 * m + g + 8 * (k & 1)][d + 2 * t + 8 * (k >> 1)]);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t x[4] = {(&pre[j][0].x)[i], (&pre[j][1].x)[i], (&pre[j][2].x)[i], (&pre[j][3].x)[i]};
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const uint32_t p0 = __byte_perm(x[0], x[1], e ? 0x7632 : 0x5410), p1 = __byte_perm(x[2], x[3], e ? 0x7632 : 0x5410);
#pragma unroll
                    for (int m = 0; m < 2; m++) mma16<T>(acc[m][2 * i + e], f[m][0], f[m][1], f[m][2], f[m][3], p0, p1);
                }
            }
            fetch(pre[j], d + 16 * AB_AHEAD);
        }
    }
    // column n of product i is latent dim 8 n + i
#pragma unroll
    for (int m = 0; m < 2; m++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const int r = 16 * m + g + 8 * e;
            if (r >= rows) continue;
            float *dst = a.qa + ((int64_t)(b0 + r) * a.H + h) * row;
#pragma unroll
            for (int n = 0; n < 2; n++) {
                if constexpr (ROUND) {
                    uint32_t o[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        float x = acc[m][2 * i][2 * e + n], y = acc[m][2 * i + 1][2 * e + n];
                        o[i] = take_pair<T>(x, y);
                    }
                    *reinterpret_cast<uint4 *>(reinterpret_cast<uint16_t *>(dst) + r0 + 16 * t + 8 * n) = make_uint4(o[0], o[1], o[2], o[3]);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; i += 4)
                        *reinterpret_cast<float4 *>(dst + r0 + 16 * t + 8 * n + i) = make_float4(acc[m][i][2 * e + n], acc[m][i + 1][2 * e + n], acc[m][i + 2][2 * e + n], acc[m][i + 3][2 * e + n]);
                }
            }
        }
}

// ------------------------------------------------------------------------------------------- core

struct CoreShared {
    uint64_t full[2], freed[2], sfull[2], sfree[2], done[2], pready;   // freed: the first half of a buffer's dims, before done
    int64_t scan[CORE_WARPS];
    uint32_t tmem, failed;
    uint32_t dead[2][2];     // positions of a tile without a row
    float alpha[LH], fac[LH];
};

// Shared-memory matrix descriptors of 128-byte swizzled operands (8-row groups 1024 bytes apart): the high word is
// the same for all of them, the low word is the address in 16-byte units under the distance `lead` between blocks of
// 64 outer elements (column-major operands; ignored for row-major ones). Steps through an operand add to the low word.
constexpr uint32_t DESC_HI = (1024 >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_lo(uint32_t addr, uint32_t lead) { return ((addr >> 4) & 0x3fff) | ((lead >> 4) << 16); }

template <bool ACC>
__device__ __forceinline__ void umma_f16(uint32_t d, uint32_t da, uint32_t db, uint32_t idesc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tmov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\tsetp.ne.b32 p, %5, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, p;\n\t}" ::"r"(d),
        "r"(da), "r"(db), "n"(DESC_HI), "r"(idesc), "n"(ACC ? 1 : 0)
        : "memory");
}
// A pair of products with one first operand: the first keeps it in the unit, the second takes it from there.
template <bool ACC>
__device__ __forceinline__ void umma_f16_keep(uint32_t d, uint32_t da, uint32_t db, uint32_t idesc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tmov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\tsetp.ne.b32 p, %5, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16.collector::a::fill [%0], a, b, %4, p;\n\t}" ::"r"(d),
        "r"(da), "r"(db), "n"(DESC_HI), "r"(idesc), "n"(ACC ? 1 : 0)
        : "memory");
}
template <bool ACC>
__device__ __forceinline__ void umma_f16_kept(uint32_t d, uint32_t da, uint32_t db, uint32_t idesc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tmov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\tsetp.ne.b32 p, %5, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16.collector::a::lastuse [%0], a, b, %4, p;\n\t}" ::"r"(d),
        "r"(da), "r"(db), "n"(DESC_HI), "r"(idesc), "n"(ACC ? 1 : 0)
        : "memory");
}
// One lane of the calling warp, the same at every call.
__device__ __forceinline__ bool elected() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ void umma_done(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// 16 lanes by 64 columns, as the accumulators of 16 x 8 products: [8-column block][row g: 2 t, 2 t + 1; row g + 8].
__device__ __forceinline__ void tm_ld_rows16(uint32_t addr, float v[8][4]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=f"(v[0][0]), "=f"(v[0][1]), "=f"(v[0][2]), "=f"(v[0][3]), "=f"(v[1][0]), "=f"(v[1][1]), "=f"(v[1][2]), "=f"(v[1][3]), "=f"(v[2][0]), "=f"(v[2][1]), "=f"(v[2][2]), "=f"(v[2][3]), "=f"(v[3][0]), "=f"(v[3][1]), "=f"(v[3][2]), "=f"(v[3][3]), "=f"(v[4][0]), "=f"(v[4][1]), "=f"(v[4][2]), "=f"(v[4][3]), "=f"(v[5][0]), "=f"(v[5][1]), "=f"(v[5][2]), "=f"(v[5][3]), "=f"(v[6][0]), "=f"(v[6][1]), "=f"(v[6][2]), "=f"(v[6][3]), "=f"(v[7][0]), "=f"(v[7][1]), "=f"(v[7][2]), "=f"(v[7][3])
        : "r"(addr)
        : "memory");
}
__device__ __forceinline__ void tm_ld16(uint32_t addr, float v[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
          "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
        : "r"(addr)
        : "memory");
}
__device__ __forceinline__ void tm_st16(uint32_t addr, const float v[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
        "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]), "f"(v[8]), "f"(v[9]),
        "f"(v[10]), "f"(v[11]), "f"(v[12]), "f"(v[13]), "f"(v[14]), "f"(v[15])
        : "memory");
}
__device__ __forceinline__ void tm_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tm_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void arrive(uint64_t *bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// Barrier BAR of N threads, with the or of x.
template <int BAR, int N>
__device__ __forceinline__ bool any_of(bool x) {
    __syncwarp();
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\t"
        "barrier.cta.red.or.pred.aligned q, %2, %3, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(r)
        : "r"(x ? 1u : 0u), "n"(BAR), "n"(N)
        : "memory");
    return r != 0;
}
__device__ __forceinline__ bool softmax_any(bool x) { return any_of<1, 128>(x); }

__device__ __forceinline__ void cp16(uint32_t dst, const void *src, bool on) {   // zeros when off
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}

// A wait that ends: on the phase, when another role has given up, or at the spin limit (the error word, so
// that the outputs become NaN).
__device__ __forceinline__ bool core_wait(CoreShared &y, uint64_t *bar, uint32_t parity, int *err) {
    for (uint32_t i = 0; i < kSpinLimit; i++) {
        if (mbar_try_wait(bar, parity)) return true;
        if (*reinterpret_cast<volatile uint32_t *>(&y.failed)) return false;
    }
    *reinterpret_cast<volatile uint32_t *>(&y.failed) = 1;
    set_error(err, DEV_E_WAIT_TIMEOUT);
    return false;
}

// One run of tiles of a sequence; every role walks the same list.
struct Run {
    int b, u, nu, n, tiles;     // sequence, first tile, its tiles, its length, tiles of the run
};
struct Walk {
    const LatentArgs &a;
    int64_t cur, end;
    int b, u, nw;       // the sequence, where in its work, its work
    __device__ __forceinline__ Walk(const LatentArgs &a_, int b_, int64_t before, int64_t cur_, int64_t end_)
        : a(a_), cur(cur_), end(end_), b(b_), u((int)(cur_ - before)), nw(work_of(a_.c, a_.lens, b_, LT, CORE_EXTRA)) {}
    __device__ __forceinline__ bool next(Run &r) {
        while (cur < end) {
            while (u >= nw) nw = work_of(a.c, a.lens, ++b, LT, CORE_EXTRA), u = 0;
            const int step = (int)min((int64_t)(nw - u), end - cur);
            r.b = b, r.u = max(u - CORE_EXTRA, 0), r.nu = nw - CORE_EXTRA, r.n = a.lens[b], r.tiles = u + step - CORE_EXTRA - r.u;
            cur += step, u += step;
            if (r.tiles > 0) return true;
        }
        return false;
    }
};

// A loading thread's rows of a tile. 16-bit rows: eight lanes a 128-byte block row, 16 rows at once; Q8: four lanes a row.
template <int CACHE>
struct TileRows {
    static constexpr int N = CACHE == Q8 ? 1 : 4;
    int64_t row[N];
    uint32_t dead;      // positions in range that have no row
    static __device__ __forceinline__ int at(int lt, int k) { return CACHE == Q8 ? lt >> 2 : (lt >> 3) + 16 * k; }
    __device__ __forceinline__ void find(const LatentArgs &a, const Run &r, int tile, int lt) {
        dead = 0;
#pragma unroll
        for (int k = 0; k < N; k++) {
            const int pos = (r.u + tile) * LT + at(lt, k);
            row[k] = pos < r.n ? kv_row(a.c, r.b, pos) : -1;
            if (pos < r.n && row[k] < 0) dead |= 1u << k;
        }
    }
    // marks them for the softmax (bit position of the tile)
    __device__ __forceinline__ void mark(CoreShared &y, int buf, int lt) const {
        if (!dead || (lt & (CACHE == Q8 ? 3 : 7))) return;
#pragma unroll
        for (int k = 0; k < N; k++)
            if (dead >> k & 1) atomicOr(&y.dead[buf][at(lt, k) >> 5], 1u << (at(lt, k) & 31));
    }
};

// Sixteen Q8 codes of a block and their scale. The loads are volatile so that they stay where they are written: ahead of
// the wait for the buffer.
struct RawRows {
    uint4 code;
    float d;
    __device__ __forceinline__ void fetch(const LatentArgs &a, int64_t row, int s, int segs, int lt) {
        code = make_uint4(0, 0, 0, 0), d = 0.0f;
        if (row < 0 || s >= segs) return;
        const int8_t *p = static_cast<const int8_t *>(a.c.k) + row * a.c.hd + s * 64 + 16 * (lt & 3);
        asm volatile("ld.global.nc.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(code.x), "=r"(code.y), "=r"(code.z), "=r"(code.w) : "l"(p));
        asm volatile("ld.global.nc.f32 %0, [%1];" : "=f"(d) : "l"(a.c.ks + row * segs + s));
    }
};
// The codes times d as f16, into pieces 2 q and 2 q + 1 of a block row, in packed f32 pairs.
__device__ __forceinline__ void expand16(uint32_t at, int rw, int q, const RawRows &r) {
    const uint64_t d2 = (uint64_t)__float_as_uint(r.d) << 32 | __float_as_uint(r.d);
    const uint64_t off = (uint64_t)__float_as_uint(-8388736.0f) << 32 | __float_as_uint(-8388736.0f);
#pragma unroll
    for (int c = 0; c < 2; c++) {
        uint32_t o[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const uint32_t w = (c ? (e < 2 ? r.code.z : r.code.w) : (e < 2 ? r.code.x : r.code.y)) ^ 0x80808080u;
            // 2^23 + (code + 128) as a float's bits, twice
            const uint32_t lo = __byte_perm(w, 0x4b000000u, e & 1 ? 0x7542 : 0x7540), hi = __byte_perm(w, 0x4b000000u, e & 1 ? 0x7543 : 0x7541);
            uint64_t x = (uint64_t)hi << 32 | lo;
            asm("add.rn.f32x2 %0, %0, %1;" : "+l"(x) : "l"(off));
            asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(x) : "l"(d2));
            const __half2 h = __floats2half2_rn(__uint_as_float((uint32_t)x), __uint_as_float((uint32_t)(x >> 32)));
            o[e] = reinterpret_cast<const uint32_t &>(h);
        }
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at + rw * 128 + (((2 * q + c) ^ (rw & 7)) << 4)), "r"(o[0]),
                     "r"(o[1]), "r"(o[2]), "r"(o[3])
                     : "memory");
    }
}

// Query rows of a run as the S product's first operand: eight lanes a head. bf16: copies that the caller waits for (from f32 rows it
// took 7700 cycles, most of them between two round trips to L2). f16: a power of two a head, from f32.
template <int OT, int THREADS>
__device__ __forceinline__ void load_q(const LatentArgs &a, CoreShared &y, uint32_t dst, int segs, const Run &r, int h0, int nh, int lt) {
    const int c8 = lt & 7, W = a.R + a.dr;
    if constexpr (OT == BF16) {
#pragma unroll 2
        for (int h = lt >> 3; h < LH; h += THREADS / 8) {
            const uint16_t *src = reinterpret_cast<const uint16_t *>(a.qa + ((int64_t)r.b * a.H + h0 + min(h, nh - 1)) * W) + 8 * c8;
            for (int s = 0; s < segs; s++) {
                const bool on = h < nh && s * 64 + c8 * 8 < W;
                cp16(dst + s * SEG + h * 128 + ((c8 ^ (h & 7)) << 4), on ? src + s * 64 : src, on);
            }
            if (c8 == 0) y.fac[h] = a.sc2;
        }
        return;
    }
#pragma unroll 1
    for (int h = lt >> 3; h < LH; h += THREADS / 8) {
        const float4 *src = reinterpret_cast<const float4 *>(a.qa + ((int64_t)r.b * a.H + h0 + h) * W) + 2 * c8;
        float4 x[9][2];
#pragma unroll
        for (int s = 0; s < 9; s++) {
            const bool on = h < nh && s * 64 + c8 * 8 < W;
            x[s][0] = on ? __ldcg(src + 16 * s) : make_float4(0, 0, 0, 0);
            x[s][1] = on ? __ldcg(src + 16 * s + 1) : make_float4(0, 0, 0, 0);
        }
        float fac = a.sc2, up = 1.0f;
        if constexpr (OT == F16) {
            float m = 0.0f;
#pragma unroll
            for (int s = 0; s < 9; s++)
#pragma unroll
                for (int i = 0; i < 2; i++)
                    m = fmaxf(m, fmaxf(fmaxf(fabsf(x[s][i].x), fabsf(x[s][i].y)), fmaxf(fabsf(x[s][i].z), fabsf(x[s][i].w))));
#pragma unroll
            for (int o = 4; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
            const int k = f16_lift(m);
            up = pow2i(k), fac = __fmul_rn(fac, pow2i(-k));
        }
        if (c8 == 0) y.fac[h] = fac;
#pragma unroll
        for (int s = 0; s < 9; s++) {
            if (s >= segs) break;
            uint32_t o[4];
#pragma unroll
            for (int i = 0; i < 2; i++) {
                float4 v = x[s][i];
                v.x = __fmul_rn(v.x, up), v.y = __fmul_rn(v.y, up), v.z = __fmul_rn(v.z, up), v.w = __fmul_rn(v.w, up);
                o[2 * i] = take_pair<OT>(v.x, v.y), o[2 * i + 1] = take_pair<OT>(v.z, v.w);
            }
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst + s * SEG + h * 128 + ((c8 ^ (h & 7)) << 4)), "r"(o[0]),
                         "r"(o[1]), "r"(o[2]), "r"(o[3])
                         : "memory");
        }
    }
}

template <int CACHE>
__global__ void __launch_bounds__(CORE_THREADS, 1) k_latent_core(const __grid_constant__ LatentArgs a) {
    constexpr int OT = CACHE == BF16 ? BF16 : F16;
    constexpr int NTP = CACHE == Q8 ? 1 : 2;
    constexpr float POFF = OT == F16 ? 8.0f : 0.0f;
    extern __shared__ uint8_t raw[];
    uint8_t *base = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
    const int segs = a.R / 64 + 1;
    uint8_t *qb = base, *kvb = qb + segs * SEG, *pb = kvb + 2 * segs * SEG;
    CoreShared &y = *reinterpret_cast<CoreShared *>(pb + SEG);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int pass = blockIdx.x % a.passes, cta = blockIdx.x / a.passes, grid = gridDim.x / a.passes;
    const int h0 = pass * a.hp, nh = min(a.hp, a.H - h0), cols = (nh + 15) & ~15;

    pdl_trigger();
    int b0, ctas;
    int64_t before, cur, end, total;
    const bool have = my_units<CORE_THREADS>(a.c, a.lens, LT, CORE_EXTRA, 1, cta, grid, y.scan, b0, before, cur, end, total, ctas);
    if (!have) {
        pdl_wait();
        return;
    }
    if (tid == 0) {
        for (int i = 0; i < 2; i++) {
            mbar_init(&y.full[i], LD_THREADS<CACHE>);
            mbar_init(&y.freed[i], 1);
            mbar_init(&y.sfull[i], 1);
            mbar_init(&y.sfree[i], 128);
            mbar_init(&y.done[i], 1);
            y.dead[i][0] = y.dead[i][1] = 0;
        }
        mbar_init(&y.pready, 128);
        y.failed = 0;
        fence_mbar_init();
    }
    if (warp == SCORE_WARP) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&y.tmem)), "r"(512u));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    tc_before();
    __syncthreads();
    tc_after();
    const uint32_t tm = y.tmem, tm_o = tm + 128;      // S in columns 0-63 and 64-127, O^T from 128 on
    Walk walk(a, b0, before, cur, end);
    Run r;

    const int pieces = a.R / 128, half = (pieces + 1) / 2;      // blocks of 128 dims; those freed first
    if (warp >= LD_WARP0) {
        // ---- loading: a group takes every GROUPS-th tile
        constexpr int GROUPS = LD_GROUPS<CACHE>, THREADS = LD_THREADS<CACHE>;
        const int group = (tid - 32 * LD_WARP0) / THREADS, lt = (tid - 32 * LD_WARP0) % THREADS;
        TileRows<CACHE> rows, next;
        auto wait = [&](uint64_t *bar, uint32_t parity) { return __all_sync(0xffffffffu, core_wait(y, bar, parity, a.err)); };
        bool ok = true, waited = false;
        int k0 = 0;      // tiles before this run
        while (ok && walk.next(r)) {
            const int i0 = GROUPS == 1 ? 0 : (k0 ^ group) & 1;
            if (i0 < r.tiles) next.find(a, r, i0, lt);
            for (int i = i0; ok && i < r.tiles; i += GROUPS) {
                const int k = k0 + i, buf = k & 1;
                const uint32_t dst = smem_u32(kvb) + buf * segs * SEG;
                rows = next;
                if constexpr (CACHE == Q8) {
                    // all of a tile's codes into registers while the tiles before are at work; then three block columns at a time,
                    // the registers moved down in between (unrolled to nine the code was fetched slower than it ran)
                    RawRows raw[9];
#pragma unroll
                    for (int s = 0; s < 9; s++) raw[s].fetch(a, rows.row[0], s, segs, lt);
                    if (i + GROUPS < r.tiles) next.find(a, r, i + GROUPS, lt);      // the next tile's places, ahead too
                    if (k >= 2) ok = wait(&y.freed[buf], ((k >> 1) - 1) & 1);
                    bool all = k < 2;
#pragma unroll 1
                    for (int s0 = 0; ok && s0 < segs; s0 += 3) {
#pragma unroll
                        for (int e = 0; e < 3; e++) {
                            const int s = s0 + e;
                            if (s >= segs) break;
                            if (s >= 2 * half && !all) {
                                ok = wait(&y.done[buf], ((k >> 1) - 1) & 1), all = true;
                                if (!ok) break;
                            }
                            expand16(dst + s * SEG, lt >> 2, lt & 3, raw[e]);
                        }
#pragma unroll
                        for (int e = 0; e < 6; e++) raw[e] = raw[e + 3];
                    }
                    if (!ok) break;
                } else {
                    const int c8 = lt & 7, tail = a.dr / 8;
                    auto copy = [&](int s0, int s1) {
#pragma unroll
                        for (int n = 0; n < 4; n++) {
                            const int rw = (lt >> 3) + 16 * n;
                            const bool on = rows.row[n] >= 0;
                            const uint8_t *src = static_cast<const uint8_t *>(a.c.k) + (on ? rows.row[n] * a.c.hd * 2 + c8 * 16 : 0);
                            const uint32_t at = dst + rw * 128 + ((c8 ^ (rw & 7)) << 4);
                            for (int s = s0; s < s1; s++) {
                                const bool use = on && (s < segs - 1 || c8 < tail);
                                cp16(at + s * SEG, use ? src + s * 128 : src, use);
                            }
                        }
                    };
                    if (k >= 2) ok = wait(&y.freed[buf], ((k >> 1) - 1) & 1);
                    if (!ok) break;
                    copy(0, 2 * half);
                    if (k >= 2) ok = wait(&y.done[buf], ((k >> 1) - 1) & 1);
                    if (!ok) break;
                    copy(2 * half, segs);
                    if (i + GROUPS < r.tiles) next.find(a, r, i + GROUPS, lt);
                }
                rows.mark(y, buf, lt);
                if (i == 0) {     // the first tile's warps bring the queries, once the last run's products are done
                    if (!waited) pdl_wait(), waited = true;
                    if (k >= 1) ok = wait(&y.done[buf ^ 1], ((k - 1) >> 1) & 1);
                    if (!ok) break;
                    load_q<OT, THREADS>(a, y, smem_u32(qb), segs, r, h0, nh, lt);
                }
                asm volatile("cp.async.wait_all;" ::: "memory");
                fence_proxy_async();
                arrive(&y.full[buf]);
            }
            k0 += r.tiles;
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        if (!waited) pdl_wait();
    } else if (warp >= SCORE_WARP) {
        // ---- products: a warp each for scores and values walks and waits, one of its lanes issues. One warp for both spent as
        // long between its products as on them: a wait costs some 100 cycles beside a busy shared memory.
        const uint32_t fmt = OT == BF16 ? (1u << 7) | (1u << 10) : 0u;
        constexpr uint32_t SEG16 = SEG >> 4, STEP = 32 >> 4, VSTEP = 2048 >> 4;
        const bool lead = elected();
        bool ok = true;
        int k = 0;
        if (warp == SCORE_WARP) {      // S = Q K^T
            const uint32_t is = (1u << 4) | fmt | ((uint32_t)(LT >> 3) << 17) | ((uint32_t)(LH >> 4) << 24);
            const uint32_t q_lo = desc_lo(smem_u32(qb), 16), k0 = desc_lo(smem_u32(kvb), 16);
            while (ok && walk.next(r))
                for (int i = 0; ok && i < r.tiles; i++, k++) {
                    if (k >= 2) ok = core_wait(y, &y.sfree[k & 1], ((k >> 1) - 1) & 1, a.err);
                    ok = ok && core_wait(y, &y.full[k & 1], (k >> 1) & 1, a.err);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    tc_after();
                    if (lead) {
                        const uint32_t d = tm + (k & 1) * 64;
                        uint32_t da = q_lo, db = k0 + (k & 1) * segs * SEG16;
                        umma_f16<false>(d, da, db, is);
#pragma unroll
                        for (int e = 1; e < 4; e++) umma_f16<true>(d, da + e * STEP, db + e * STEP, is);
#pragma unroll 2
                        for (int s = 1; s < segs; s++) {
                            da += SEG16, db += SEG16;
#pragma unroll
                            for (int e = 0; e < 4; e++) umma_f16<true>(d, da + e * STEP, db + e * STEP, is);
                        }
                        umma_done(&y.sfull[k & 1]);
                    }
                    __syncwarp();
                }
        } else {      // O^T += V^T P^T
            const uint32_t ip = (1u << 4) | fmt | (1u << 15) | ((uint32_t)(cols >> 3) << 17) | (8u << 24);
            const uint32_t p_lo = desc_lo(smem_u32(pb), 16), v0 = desc_lo(smem_u32(kvb), SEG), r0 = desc_lo(smem_u32(kvb), 16) + (segs - 1) * SEG16;
            while (ok && walk.next(r))
                for (int i = 0; ok && i < r.tiles; i++, k++) {
                    ok = __all_sync(0xffffffffu, core_wait(y, &y.pready, k & 1, a.err));
                    if (!ok) break;
                    tc_after();
                    if (lead) {
                        uint32_t da = v0 + (k & 1) * segs * SEG16, d = tm_o;
                        const uint32_t rest = r0 + (k & 1) * segs * SEG16;
                        for (int blk = 0; blk < pieces; blk++, d += cols, da += 2 * SEG16) {
                            if constexpr (NTP == 2) {
                                if (i == 0) umma_f16_keep<false>(d, da, p_lo, ip);
                                else umma_f16_keep<true>(d, da, p_lo, ip);
                                umma_f16_kept<true>(d, da, rest, ip);
#pragma unroll
                                for (int e = 1; e < LT / 16; e++) {
                                    umma_f16_keep<true>(d, da + e * VSTEP, p_lo + e * STEP, ip);
                                    umma_f16_kept<true>(d, da + e * VSTEP, rest + e * STEP, ip);
                                }
                            } else {
                                if (i == 0) umma_f16<false>(d, da, p_lo, ip);
                                else umma_f16<true>(d, da, p_lo, ip);
#pragma unroll
                                for (int e = 1; e < LT / 16; e++) umma_f16<true>(d, da + e * VSTEP, p_lo + e * STEP, ip);
                            }
                            // a commit costs the unit about as long as five products: one half way, one at the end
                            if (blk == half - 1) umma_done(&y.freed[k & 1]);
                        }
                        umma_done(&y.done[k & 1]);
                    }
                    __syncwarp();
                }
        }
    } else {
        // ---- softmax. The 64 rows (heads) of S lie in lanes 0-15 of the four warps' quarters of tensor memory; read 16
        // lanes by 256 bits, lane (g, t) gets heads 16 w + g and + 8, columns 8 j + 2 t and + 1. O^T: a lane a dim.
        const int g = lane >> 2, t = lane & 3, hd[2] = {16 * warp + g, 16 * warp + g + 8};
        const uint32_t lanes = (uint32_t)(32 * warp) << 16;
        // where this lane's rows of 8 x 8 blocks go in P: lanes 0-7 block j, rows g; 8-15 rows g + 8; 16-31 block j + 1
        const int prow = 16 * warp + (lane & 15), pcol = lane >> 4;
        int k = 0;
        bool ok = true, up = false, dry = true;
        while (!up && walk.next(r)) {
            float ref[2] = {-kv_inf(), -kv_inf()}, sum[2] = {}, fac[2] = {};
            // One dry step while the first loads are on their way, on whatever tensor memory holds and with nothing kept: it
            // brings the code near (code that runs for the first time is fetched slower than it runs): one sequence of 1531 in 24.0 us
            // of GPU time, 24.7 without it, 4 Q8 ones of up to 65536 in 62.7 and 64.5. The same in the kernels that join cost more
            // than it gave (0.5 to 1.6 us).
            for (int i = dry ? -1 : 0; i < r.tiles; i++, k++) {
                const int buf = k & 1;
                // a wait that fails shows at the next barrier of the four warps, where all of them give up
                if (!dry) ok = core_wait(y, &y.sfull[buf], (k >> 1) & 1, a.err) && ok;
                __syncwarp();
                tc_after();
                if (i == 0) fac[0] = y.fac[hd[0]], fac[1] = y.fac[hd[1]];
                float v[8][4];
                tm_ld_rows16(tm + lanes + buf * 64, v);
                tc_before();
                if (!dry) arrive(&y.sfree[buf]);
                const int live = dry ? LT : r.n - (r.u + i) * LT;
                const uint32_t d0 = dry ? 0 : y.dead[buf][0], d1 = dry ? 0 : y.dead[buf][1];
                float mx[2] = {-kv_inf(), -kv_inf()}, fade[2] = {1.0f, 1.0f};
#pragma unroll
                for (int j = 0; j < 8; j++)
#pragma unroll
                    for (int e = 0; e < 4; e++) v[j][e] = __fmul_rn(v[j][e], fac[e >> 1]);
                if (live < LT || (d0 | d1)) {      // a sequence's last tile, or positions without a row
#pragma unroll
                    for (int j = 0; j < 8; j++)
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const int c = 8 * j + 2 * t + (e & 1);
                            if ((j < 4 ? d0 >> c : d1 >> (c - 32)) & 1) v[j][e] = kv_nan();
                            if (c >= live) v[j][e] = -kv_inf();
                        }
                }
#pragma unroll
                for (int j = 0; j < 8; j++)
#pragma unroll
                    for (int e = 0; e < 4; e++) mx[e >> 1] = fmaxf(mx[e >> 1], v[j][e]);
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 1));
                    mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 2));
                    if (mx[e] > ref[e] + REF_SLACK || ref[e] == -kv_inf()) {
                        fade[e] = exp2_fast(__fsub_rn(ref[e], mx[e] == -kv_inf() ? 0.0f : mx[e]));
                        ref[e] = mx[e];
                    }
                }
                const bool rescale = i > 0 && (fade[0] != 1.0f || fade[1] != 1.0f);
                if (softmax_any(!ok || rescale)) {
                    if (softmax_any(!ok)) { up = true; break; }
                    if (t == 0) y.alpha[hd[0]] = fade[0], y.alpha[hd[1]] = fade[1];
                    ok = core_wait(y, &y.done[buf ^ 1], ((k - 1) >> 1) & 1, a.err) && ok;
                    if (softmax_any(!ok)) { up = true; break; }
                    tc_after();
                    for (int c = 0; c < a.R / 128 * cols; c += 16) {
                        float o[16];
                        tm_ld16(tm_o + lanes + c, o);
                        tm_wait_ld();
                        const float *al = y.alpha + c % cols;
#pragma unroll
                        for (int j = 0; j < 16; j++) o[j] = __fmul_rn(o[j], al[j]);
                        tm_st16(tm_o + lanes + c, o);
                    }
                    tm_wait_st();
                }
#pragma unroll
                for (int e = 0; e < 2; e++) sum[e] = __fmul_rn(sum[e], fade[e]);
                const float shift[2] = {__fsub_rn(ref[0] == -kv_inf() ? 0.0f : ref[0], POFF), __fsub_rn(ref[1] == -kv_inf() ? 0.0f : ref[1], POFF)};
#pragma unroll
                for (int j = 0; j < 8; j++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        v[j][e] = exp2_fast(__fsub_rn(v[j][e], shift[e >> 1]));
                        sum[e >> 1] = __fadd_rn(sum[e >> 1], v[j][e]);
                    }
                // P's buffer is free once the previous values' product is done
                if (k >= 1) ok = core_wait(y, &y.done[buf ^ 1], ((k - 1) >> 1) & 1, a.err) && ok;
                __syncwarp();
                if (16 * warp < cols) {
                    const uint32_t p0 = smem_u32(pb) + prow * 128, p1 = dry ? p0 : smem_u32(kvb) + buf * segs * SEG + (segs - 1) * SEG + prow * 128;
#pragma unroll
                    for (int j = 0; j < 8; j += 2)
#pragma unroll
                        for (int x = 0; x < NTP; x++) {
                            const uint32_t m0 = take_pair<OT>(v[j][0], v[j][1]), m1 = take_pair<OT>(v[j][2], v[j][3]);
                            const uint32_t m2 = take_pair<OT>(v[j + 1][0], v[j + 1][1]), m3 = take_pair<OT>(v[j + 1][2], v[j + 1][3]);
                            asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(
                                             (x == 0 ? p0 : p1) + (((j + pcol) ^ (prow & 7)) << 4)),
                                         "r"(m0), "r"(m1), "r"(m2), "r"(m3)
                                         : "memory");
                        }
                }
                if (dry) {
                    dry = false, k--;
                    ref[0] = ref[1] = -kv_inf(), sum[0] = sum[1] = 0.0f;
                    continue;
                }
                if (tid == 0) y.dead[buf][0] = y.dead[buf][1] = 0;
                fence_proxy_async();
                tc_before();
                arrive(&y.pready);
            }
            if (up) break;
            ok = core_wait(y, &y.done[(k - 1) & 1], ((k - 1) >> 1) & 1, a.err) && ok;
            if (softmax_any(!ok)) break;
            tc_after();
            const bool whole = r.tiles == r.nu;
            const int slot = r.b == b0 ? 0 : 1, W = a.R + a.dr;
            const int64_t piece = (int64_t)blockIdx.x * 2 + slot;
            float *o0 = whole ? a.qa + ((int64_t)r.b * a.H + h0) * W : a.o + piece * a.hp * a.R;
            const int64_t pitch = whole ? W : a.R;
            // columns of 16 heads at a time, the next ones read while these are stored
            float o[2][16];
            tm_ld16(tm_o + lanes, o[0]);
#pragma unroll 1
            for (int c = 0; c < cols; c += 16) {
                float *at = o0 + (int64_t)c * pitch + 32 * warp + lane;
                const bool all = c + 16 <= nh;
#pragma unroll
                for (int blk = 0; blk < 4; blk++) {
                    if (blk >= pieces) break;
                    tm_wait_ld();
                    if (blk + 1 < pieces) tm_ld16(tm_o + lanes + (blk + 1) * cols + c, o[(blk + 1) & 1]);
                    else if (c + 16 < cols) tm_ld16(tm_o + lanes + c + 16, o[(blk + 1) & 1]);
                    float *p = at + blk * 128;
#pragma unroll
                    for (int j = 0; j < 16; j++, p += pitch)
                        if (all || c + j < nh) *p = o[blk & 1][j];
                }
                if (pieces & 1) {     // the columns after an odd number of blocks were read into the other half
#pragma unroll
                    for (int j = 0; j < 16; j++) o[0][j] = o[1][j];
                }
            }
#pragma unroll
            for (int e = 0; e < 2; e++) {
                sum[e] = __fadd_rn(sum[e], __shfl_xor_sync(0xffffffffu, sum[e], 1));
                sum[e] = __fadd_rn(sum[e], __shfl_xor_sync(0xffffffffu, sum[e], 2));
                if (t != 0 || hd[e] >= nh) continue;
                if (whole) o0[(int64_t)hd[e] * W + a.R] = ref[e], o0[(int64_t)hd[e] * W + a.R + 1] = sum[e];
                else a.ml[piece * a.hp + hd[e]] = make_float2(ref[e], sum[e]);
            }
            tc_before();
        }
    }
    __syncthreads();
    if (warp == SCORE_WARP) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tm), "r"(512u));
}

// ------------------------------------------------------------------------------------------- expand

constexpr int EX_WARPS = 16, EX_ROWS = 16, EX_KEPT = 8;

struct ExpandShared {
    uint32_t ops[2][16][2][32][4];       // [term][32-dim step][eight rows][lane]
    union {
        float join[EX_WARPS][512];
        float red[16][16 * EX_ROWS];
    };
    float2 ml[EX_WARPS];
    float fac[EX_WARPS];                 // a piece's factor in its row's o
    uint4 w[EX_KEPT][2][32 * EX_WARPS];  // the threads' first weights
    uint32_t over;                       // sequences longer than their table
    int64_t sums[EX_WARPS][2];
};

// A CTA a head and up to sixteen sequences. Warps first join the pieces (weights 2^(m_i - max m), in a fixed order) into o, as
// two terms of the weights' type in shared memory; then each multiplies 16 value rows by (a part of) o. Reads from L2 bound it:
// 128 KB of weights a head (before the core has ended where its SM is free) and 2 KB a piece. 10 us after the core
// with 32 sequences of 64 heads, 4 with one.
template <int T>
__global__ void __launch_bounds__(32 * EX_WARPS, 1) k_latent_expand(const __grid_constant__ LatentArgs a, int ex_rows, int grid) {
    extern __shared__ __align__(16) uint8_t raw[];
    ExpandShared &y = *reinterpret_cast<ExpandShared *>(raw);
    const int h = blockIdx.x, b0 = blockIdx.y * ex_rows, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int rows = min(ex_rows, a.c.n_seqs - b0), pass = h / a.hp, hc = h - pass * a.hp, W = a.R + a.dr, steps = a.R / 32;
    // warps over (16 value rows, part of the latent dims): ksplit parts where there are fewer row tiles than warps
    const int mt = a.dv / 16, ksplit = max(1, EX_WARPS / mt), items = mt * ksplit;
    const uint16_t *w = static_cast<const uint16_t *>(a.w) + ((int64_t)h * (a.dn + a.dv) + a.dn + g) * a.R + 8 * t;
    auto first = [&](int item) { return item / mt * steps / ksplit; };
    auto last = [&](int item) { return item < items ? (item / mt + 1) * steps / ksplit : 0; };      // none for a warp without an item
    auto at = [&](int item, int s, int k) { return w + (int64_t)(item % mt) * 16 * a.R + s * 32 + k * 8 * (int64_t)a.R; };
    // A warp has one item at most. Its first weights come into shared memory (places of its own) before the core has ended: an SM
    // takes 128 KB from L2 in about 5000 cycles.
    const int s_first = first(warp), s_end = last(warp);
#pragma unroll
    for (int i = 0; i < EX_KEPT; i++)
        if (s_first + i < s_end) cp16(smem_u32(&y.w[i][0][threadIdx.x]), at(warp, s_first + i, 0), true), cp16(smem_u32(&y.w[i][1][threadIdx.x]), at(warp, s_first + i, 1), true);
    for (int i = threadIdx.x; i < 2 * 16 * 2 * 32; i += 32 * EX_WARPS) reinterpret_cast<uint4 *>(&y.ops)[i] = make_uint4(0, 0, 0, 0);
    if (threadIdx.x < 32) {
        const uint32_t over = __ballot_sync(0xffffffffu, lane < rows && a.lens[b0 + min(lane, rows - 1)] > table_capacity(a.c));
        if (lane == 0) y.over = over;
    }
    // the warp's row and its pieces, from the lengths
    int wpr = EX_WARPS;                                  // warps a row
    while (wpr * rows > EX_WARPS) wpr >>= 1;
    const int row = warp / wpr, part = warp % wpr, b = b0 + min(row, rows - 1);
    int64_t before, all;
    work_sums<32 * EX_WARPS>(a.c, a.lens, LT, CORE_EXTRA, b0, y.sums, before, all);
    for (int i = b0; i < b; i++) before += work_of(a.c, a.lens, i, LT, CORE_EXTRA);
    const int n = a.lens[b], nu = units_of(a.c, a.lens, b, LT);
    Span sp = {};
    if (nu) sp = span_of(before, CORE_EXTRA, nu, all, grid);
    pdl_wait();
    __syncthreads();
    if (row < rows) {
        Joined<16> o;
        const float *whole = a.qa + ((int64_t)b * a.H + h) * W;
        const int count = !nu ? 0 : sp.split() ? sp.last - sp.first + 1 : 1;
#pragma unroll 4
        for (int i = part; i < count; i += wpr) {
            const int64_t at = ((int64_t)((sp.first + i) * a.passes + pass) * 2 + (i == 0 ? sp.slot : 0)) * a.hp + hc;
            const float *src = sp.split() ? a.o + at * a.R : whole;
            const float2 ml = sp.split() ? __ldcg(a.ml + at) : make_float2(__ldcg(whole + a.R), __ldcg(whole + a.R + 1));
            float x[16] = {};
#pragma unroll
            for (int k = 0; k < 4; k++)
                if (k < a.R / 128) {
                    const float4 v = __ldcg(reinterpret_cast<const float4 *>(src + 128 * k + 4 * lane));
                    x[4 * k] = v.x, x[4 * k + 1] = v.y, x[4 * k + 2] = v.z, x[4 * k + 3] = v.w;
                }
            o.add(ml, x);
        }
        // nothing, too long a row and a failed wait as the entry point says
        const bool bad = *reinterpret_cast<volatile int *>(a.err) || (y.over >> row & 1);
        if (wpr == 1) {     // the row is whole
            const float inv = bad ? kv_nan() : o.l == 0.0f ? 0.0f : __fdiv_rn(1.0f, o.l);
#pragma unroll
            for (int k = 0; k < 4; k++) {
                if (k >= a.R / 128) break;
                float x[4];
#pragma unroll
                for (int e = 0; e < 4; e++) x[e] = bad || o.l != 0.0f ? __fmul_rn(o.o[4 * k + e], inv) : 0.0f;
#pragma unroll
                for (int term = 0; term < 2; term++) {
                    uint2 p;
                    p.x = take_pair<T>(x[0], x[1]), p.y = take_pair<T>(x[2], x[3]);
                    *reinterpret_cast<uint2 *>(&y.ops[term][4 * k + (lane >> 3)][row >> 3][(row & 7) * 4 + ((lane >> 1) & 3)][2 * (lane & 1)]) = p;
                }
            }
        } else {
#pragma unroll
            for (int k = 0; k < 4; k++)
                *reinterpret_cast<float4 *>(&y.join[warp][128 * k + 4 * lane]) = make_float4(o.o[4 * k], o.o[4 * k + 1], o.o[4 * k + 2], o.o[4 * k + 3]);
            if (lane == 0) y.ml[warp] = make_float2(o.m, bad ? kv_nan() : o.l);
        }
    }
    if (wpr > 1) {     // a row's warps together, two dims a thread
        __syncthreads();
        if (threadIdx.x < rows * wpr) {
            const int p0 = threadIdx.x / wpr * wpr;
            float m = -kv_inf(), l = 0.0f;
            for (int p = p0; p < p0 + wpr; p++) m = fmaxf(m, y.ml[p].x);
            const float base = m == -kv_inf() ? 0.0f : m;
            for (int p = p0; p < p0 + wpr; p++) l = __fmaf_rn(y.ml[p].y, exp2_fast(__fsub_rn(y.ml[p].x, base)), l);
            y.fac[threadIdx.x] = l == 0.0f ? 0.0f : __fdiv_rn(exp2_fast(__fsub_rn(y.ml[threadIdx.x].x, base)), l);
        }
        __syncthreads();
        for (int i = threadIdx.x; i < rows * (a.R / 2); i += 32 * EX_WARPS) {
            const int rw = i / (a.R / 2), d = 2 * (i - rw * (a.R / 2));
            float x0 = 0.0f, x1 = 0.0f;
#pragma unroll 4
            for (int p = rw * wpr; p < (rw + 1) * wpr; p++) {
                const float2 v = *reinterpret_cast<const float2 *>(&y.join[p][d]);
                x0 = __fmaf_rn(v.x, y.fac[p], x0), x1 = __fmaf_rn(v.y, y.fac[p], x1);
            }
#pragma unroll
            for (int k = 0; k < 2; k++) y.ops[k][d >> 5][rw >> 3][(rw & 7) * 4 + ((d >> 3) & 3)][(d >> 1) & 3] = take_pair<T>(x0, x1);
        }
    }
    __syncthreads();
    if (warp < items) {
        float acc[2][4] = {};
        auto step = [&](int s, const uint4 &v0, const uint4 &v1) {
#pragma unroll
            for (int c = 0; c < 2; c++) {
                if (8 * c >= rows) break;
#pragma unroll
                for (int k = 1; k >= 0; k--) {
                    const uint4 x = *reinterpret_cast<const uint4 *>(y.ops[k][s][c][lane]);
                    mma16<T>(acc[c], v0.x, v1.x, v0.y, v1.y, x.x, x.y);
                    mma16<T>(acc[c], v0.z, v1.z, v0.w, v1.w, x.z, x.w);
                }
            }
        };
        asm volatile("cp.async.wait_all;" ::: "memory");
#pragma unroll 4
        for (int i = 0; i < EX_KEPT; i++)
            if (s_first + i < s_end) step(s_first + i, y.w[i][0][threadIdx.x], y.w[i][1][threadIdx.x]);
#pragma unroll 4
        for (int s = s_first + EX_KEPT; s < s_end; s++) step(s, __ldg(reinterpret_cast<const uint4 *>(at(warp, s, 0))), __ldg(reinterpret_cast<const uint4 *>(at(warp, s, 1))));
#pragma unroll
        for (int c = 0; c < 2; c++)
#pragma unroll
            for (int e = 0; e < 4; e++) y.red[warp][(g + 8 * (e >> 1)) * EX_ROWS + 8 * c + 2 * t + (e & 1)] = acc[c][e];
    }
    __syncthreads();
#pragma unroll 4
    for (int i = threadIdx.x; i < rows * a.dv; i += 32 * EX_WARPS) {
        const int rw = i / a.dv, j = i - rw * a.dv;
        float x = y.red[j >> 4][(j & 15) * EX_ROWS + rw];
        for (int k = 1; k < ksplit; k++) x = __fadd_rn(x, y.red[k * mt + (j >> 4)][(j & 15) * EX_ROWS + rw]);
        io_store(a.out, T, (b0 + rw) * a.os + h * a.oh + j, x);
    }
}

// ------------------------------------------------------------------------------------------- host side

struct Plan {
    int passes, hp, grid, segs;
    size_t qa, o, ml, bytes, smem;
};

Plan plan_of(const hxb_kv_cache *c, int H, int R) {
    Plan p = {};
    p.passes = (H + LH - 1) / LH;
    p.hp = (H + p.passes - 1) / p.passes;
    p.grid = ATTN_SMS / p.passes * p.passes;
    p.segs = R / 64 + 1;
    auto up = [](size_t n) { return (n + 15) / 16 * 16; };
    p.qa = up((size_t)c->n_seqs * H * c->head_dim * sizeof(float));
    p.o = (size_t)p.grid * 2 * p.hp * R * sizeof(float);
    p.ml = (size_t)p.grid * 2 * p.hp * sizeof(float2);
    p.bytes = p.qa + p.o + p.ml + 16;
    p.smem = 1024 + (size_t)(3 * p.segs + 1) * SEG + sizeof(CoreShared);
    return p;
}

template <int CACHE, int T>
cudaError_t launch(const LatentArgs &a, const Plan &p, cudaStream_t s) {
    cudaError_t e = cudaFuncSetAttribute(k_latent_core<CACHE>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)p.smem);
    if (e != cudaSuccess) return e;
    e = cudaFuncSetAttribute(k_latent_expand<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(ExpandShared));
    if (e != cudaSuccess) return e;
    const int nc = (a.R + 64 * AB_WARPS - 1) / (64 * AB_WARPS), B = a.c.n_seqs;
    e = launch_pdl(false, k_latent_absorb<T, CACHE == BF16>, dim3(a.H * nc, (B + AB_ROWS - 1) / AB_ROWS), dim3(32 * AB_WARPS), 0, s, a);
    if (e != cudaSuccess) return e;
    e = launch_pdl(true, k_latent_core<CACHE>, dim3(p.grid), dim3(CORE_THREADS), p.smem, s, a);
    if (e != cudaSuccess) return e;
    // sixteen sequences share a read of the value rows; fewer a CTA where that would leave SMs without one
    int rows = EX_ROWS;
    while (rows > 1 && 4 * a.H * ((B + rows - 1) / rows) < 3 * ATTN_SMS) rows /= 2;
    return launch_pdl(true, k_latent_expand<T>, dim3(a.H, (B + rows - 1) / rows), dim3(32 * EX_WARPS), sizeof(ExpandShared), s, a, rows, p.grid / p.passes);
}

}  // namespace
}  // namespace hx

using namespace hx;

extern "C" HXB_API size_t hxb_latent_decode_workspace(const hxb_kv_cache *c, int n_heads, int rank) {
    if (!c || n_heads < 1 || n_heads > 256 || rank < 1 || rank > 512 || c->n_seqs < 0 || c->head_dim < 1) return 0;
    return plan_of(c, n_heads, rank).bytes;
}

extern "C" HXB_API int hxb_latent_decode_dev(const hxb_kv_cache *c, const int32_t *lens, const void *q, int64_t q_stride,
                                             int64_t q_head_stride, const void *w, int n_heads, int rank, int nope,
                                             int v_dim, int dtype, float scale, void *out, int64_t out_stride,
                                             int64_t out_head_stride, void *ws, size_t ws_bytes, void *stream) {
    const char *who = "latent_decode";
    LatentArgs a = {};
    int rc = kv_view(c, who, true, &a.c);
    if (rc != HXB_OK) return rc;
    if (dtype != F16 && dtype != BF16) return attn_fail(HXB_E_ARG, "%s: dtype %d (F16 or BF16)", who, dtype);
    if (c->dtype != Q8 && c->dtype != dtype) return attn_fail(HXB_E_ARG, "%s: the cache is Q8 or has the type of q", who);
    const int dr = c->head_dim - rank;
    if (rank < 128 || rank > 512 || rank % 128 || dr < 16 || dr > 64 || dr % 16)
        return attn_fail(HXB_E_UNSUPPORTED, "%s: rank %d in rows of %d (rank a multiple of 128 up to 512, and 16 to 64 more)", who, rank,
                         c->head_dim);
    if (nope < 16 || nope > 256 || nope % 16 || v_dim < 16 || v_dim > 256 || v_dim % 16)
        return attn_fail(HXB_E_UNSUPPORTED, "%s: nope %d, v_dim %d (multiples of 16 up to 256)", who, nope, v_dim);
    if (n_heads < 1 || n_heads > 256 || c->n_seqs > 65535)
        return attn_fail(HXB_E_ARG, "%s: %d heads (up to 256), %d sequences (up to 65535)", who, n_heads, c->n_seqs);
    if (c->n_seqs == 0) return HXB_OK;
    rc = attn_check_io(who, c->n_seqs, n_heads, q, q_stride, q_head_stride, out, out_stride, out_head_stride, v_dim, dtype, lens, scale);
    if (rc != HXB_OK) return rc;
    if (!w || reinterpret_cast<uintptr_t>(w) % 16) return attn_fail(HXB_E_ARG, "%s: w must be 16-byte aligned", who);
    const Plan p = plan_of(c, n_heads, rank);
    if (!ws || reinterpret_cast<uintptr_t>(ws) % 16 || ws_bytes < p.bytes)
        return attn_fail(HXB_E_ARG, "%s: workspace of %zu bytes, 16-byte aligned, needed", who, p.bytes);
    uint8_t *at = static_cast<uint8_t *>(ws);
    a.qa = reinterpret_cast<float *>(at), at += p.qa;
    a.o = reinterpret_cast<float *>(at), at += p.o;
    a.ml = reinterpret_cast<float2 *>(at), at += p.ml;
    a.err = reinterpret_cast<int *>(at);
    if (!a.c.k) a.c.k = ws;      // a pool of no pages: copies of no bytes still name an address
    a.lens = lens, a.q = q, a.w = w, a.out = out, a.qs = q_stride, a.qh = q_head_stride, a.os = out_stride, a.oh = out_head_stride;
    a.H = n_heads, a.R = rank, a.dr = dr, a.dn = nope, a.dv = v_dim, a.passes = p.passes, a.hp = p.hp;
    a.sc2 = scale * 1.44269504088896f;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    cudaError_t e;
    if (c->dtype == Q8) e = dtype == F16 ? launch<Q8, F16>(a, p, s) : launch<Q8, BF16>(a, p, s);
    else e = dtype == F16 ? launch<F16, F16>(a, p, s) : launch<BF16, BF16>(a, p, s);
    if (e != cudaSuccess) return attn_fail(HXB_E_DEVICE, "%s: %s", who, cudaGetErrorString(e));
    return HXB_OK;
}
