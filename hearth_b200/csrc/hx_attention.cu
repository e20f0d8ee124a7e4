// hx_attention.cu — rotary positions and the paged key-value cache on device buffers (hxb_rope_*,
// hxb_kv_*): the reference's rope_tables / rope_apply (engine/src/model.c:386-411) and its cache rows
// (model.c:484-517), with pages, element types and Q8 blocks of their own.
#include "hx_paged.cuh"

#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdio>

namespace hx {

void set_last_error(const char *msg);

int attn_fail(int code, const char *fmt, ...) {
    char buf[320];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    set_last_error(buf);
    return code;
}

bool attn_launched(const char *who) {
    const cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess) return true;
    attn_fail(HXB_E_DEVICE, "%s: %s", who, cudaGetErrorString(e));
    return false;
}

static bool aligned(const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
static size_t elem_size(int dtype) { return dtype == F32 ? 4 : 2; }
static bool io_dtype(int dtype) { return dtype == F32 || dtype == F16 || dtype == BF16; }

int kv_view(const hxb_kv_cache *c, const char *who, bool latent, KvView *o) {
    if (!c) return attn_fail(HXB_E_ARG, "%s: null cache", who);
    if (c->dtype != F16 && c->dtype != BF16 && c->dtype != Q8)
        return attn_fail(HXB_E_UNSUPPORTED, "%s: cache dtype %d (F16, BF16 or Q8)", who, c->dtype);
    const bool q8 = c->dtype == Q8;
    if (c->n_kv_heads < 1 || c->n_kv_heads > 65535 || c->head_dim < 8 || c->head_dim > 1024 || c->head_dim % 8 ||
        (q8 && c->head_dim % KV_BLOCK))
        return attn_fail(HXB_E_ARG, "%s: %d heads of %d (head_dim a multiple of %d up to 1024)", who, c->n_kv_heads,
                         c->head_dim, q8 ? KV_BLOCK : 8);
    if (c->page_tokens < 1 || c->page_tokens > 1024 || (c->page_tokens & (c->page_tokens - 1)))
        return attn_fail(HXB_E_ARG, "%s: page_tokens %d (a power of two up to 1024)", who, c->page_tokens);
    if (c->n_pages < 0 || c->n_pages > 0x7fffffff || c->table_pages < 0 || c->n_seqs < 0 || c->table_stride < 0 ||
        (int64_t)c->table_pages * c->page_tokens > 0x7fffff00)   // positions fit an int with a tile to spare
        return attn_fail(HXB_E_ARG, "%s: bad page counts", who);
    if (c->table_stride && c->table_stride < c->table_pages)
        return attn_fail(HXB_E_ARG, "%s: table rows overlap (stride %lld, %d pages)", who, (long long)c->table_stride,
                         c->table_pages);
    if (latent && (c->n_kv_heads != 1 || c->v || c->v_scale))
        return attn_fail(HXB_E_ARG, "%s: a latent cache has one row a token and no v", who);
    if (c->n_pages && (!c->k || (!latent && !c->v) || (q8 && (!c->k_scale || (!latent && !c->v_scale)))))
        return attn_fail(HXB_E_ARG, "%s: null pool", who);
    if (!q8 && (c->k_scale || c->v_scale)) return attn_fail(HXB_E_ARG, "%s: scales with a cache that is not Q8", who);
    if (!aligned(c->k, 16) || !aligned(c->v, 16) || !aligned(c->k_scale, 4) || !aligned(c->v_scale, 4) ||
        !aligned(c->table, 4))
        return attn_fail(HXB_E_ARG, "%s: pool or table not aligned", who);
    if (c->n_seqs && c->table_pages && !c->table) return attn_fail(HXB_E_ARG, "%s: null page table", who);
    o->k = c->k, o->v = c->v, o->ks = c->k_scale, o->vs = c->v_scale;
    o->table = c->table, o->table_stride = c->table_stride, o->n_pages = c->n_pages;
    o->table_pages = c->table_pages, o->n_seqs = c->n_seqs, o->Hkv = c->n_kv_heads, o->hd = c->head_dim;
    o->pt_log2 = 0;
    while ((1 << o->pt_log2) < c->page_tokens) o->pt_log2++;
    return HXB_OK;
}

// Whether rows [T][H][n] by these strides may overlap themselves; used for outputs.
bool rows_overlap(int64_t T, int64_t ts, int H, int64_t hs, int n) {
    if (T > 1 && ts < 1) return true;
    if (H > 1 && hs < 1) return true;
    if (H > 1 && hs < n) return true;
    if (T <= 1) return false;
    if (H <= 1) return ts < n;
    return !(ts >= (H - 1) * hs + n || (hs >= (T - 1) * ts + n && ts >= n));
}

namespace {

// The row kernels (rotation, cache write and read) work on items of eight values; a thread has ROW_AHEAD of them in flight,
// a CTA takes whole tokens up to ROW_ITEMS items (one token at least).
constexpr int ROW_THREADS = 256, ROW_AHEAD = 4, ROW_ITEMS = ROW_THREADS * ROW_AHEAD;

// ------------------------------------------------------------------------------------------- rotary tables

struct FreqArg {
    double2 turns[512];  // inv_freq / (2 pi) in two terms
    float fhi, flo;      // the factor in two terms
};

constexpr int TABLE_ITEMS = 4096;   // values of a CTA, at least a row

// cs[i][j] = factor * (cos, sin)(2 pi frac(p * turns_j)). The product and its fractional part are formed in 64 bits, with what the
// quotient and the product lose there added to the fraction (without it a frequency of 1 near position 2^31 is off by
// 2^-22); the f32 part of the fraction goes through sincospif and the rest, below 2^-25 of a half turn,
// enters to first order. 131072 positions of 64 angles, 67 MB written once: 24.6 us, 2.7 TB/s. A copy without sincospif takes 18.6 us,
// one without the 64-bit fraction 18.5, one without either 18.6, and a fill with a constant 12.3: arithmetic and writes
// each hold up the other.
__global__ void __launch_bounds__(256) k_rope_table(const __grid_constant__ FreqArg f, int half, FastDiv by_half, int rows, int64_t pos0,
                                                    int64_t n_pos, float2 *__restrict__ cs) {
    __shared__ double2 turns[512];     // lanes of a warp want different ones, which the parameter bank serves one by one
    for (int j = threadIdx.x; j < half; j += 256) turns[j] = f.turns[j];
    __syncthreads();
    const int64_t r0 = (int64_t)blockIdx.x * rows;
    const int n = (int)min((int64_t)rows, n_pos - r0) * half;
#pragma unroll 2
    for (int i = threadIdx.x; i < n; i += 256) {
        const int p = (int)by_half.div(i), j = i - p * half;
        const double x = (double)(pos0 + r0 + p), t = x * turns[j].x;
        const double r = 2.0 * ((t - rint(t)) + __fma_rn(x, turns[j].y, __fma_rn(x, turns[j].x, -t)));      // half turns, in [-1, 1] or just past it
        const float hi = (float)r, lo = (float)(r - (double)hi) * 3.14159265358979f;
        float s, c;
        sincospif(hi, &s, &c);
        const float cc = __fmaf_rn(-lo, s, c), ss = __fmaf_rn(lo, c, s);
        cs[r0 * half + i] = make_float2(__fmaf_rn(cc, f.fhi, cc * f.flo), __fmaf_rn(ss, f.fhi, ss * f.flo));
    }
}

// ------------------------------------------------------------------------------------------- rotation

struct RopeView {
    const float *cs;
    int64_t n_pos;
    int half, off, style;
};

__device__ __forceinline__ void rotate(float &a, float &b, float c, float s) {
    const float na = __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s));
    b = __fadd_rn(__fmul_rn(b, c), __fmul_rn(a, s));
    a = na;
}

struct RopeArgs {
    RopeView r;
    const int32_t *pos;
    const void *x;
    void *y;
    int64_t T, xs, xh, ys, yh;
    int H, hd, tpc, in_place;
    int n_rot, n_copy;            // items of a head that are rotated, and copied
    FastDiv rot_tok, rot_head, copy_tok, copy_head;
};

// Items own what they read and write, so y may be x. VEC: an item is a chunk of eight values (halves: the pair of chunks
// j, j + half), else one pair or one copied value. A CTA takes its tokens' rotated items first, then the copied ones.
// HBM bounds it: 4099 tokens of 64 heads of 192 (64 rotated), f32 to bf16, 303 MB in 54 us, 5.7 TB/s, 88 % of the copy rate.
template <class TX, class TY, bool VEC>
__global__ void __launch_bounds__(ROW_THREADS) k_rope(const __grid_constant__ RopeArgs a) {
    const int64_t t0 = (int64_t)blockIdx.x * a.tpc;
    const int nt = (int)min((int64_t)a.tpc, a.T - t0);
    const int per = a.H * a.n_rot, rot = 2 * a.r.half;
#pragma unroll 2
    for (int i = threadIdx.x; i < nt * per; i += ROW_THREADS) {
        const int tl = (int)a.rot_tok.div(i), u0 = i - tl * per;
        const int h = (int)a.rot_head.div(u0), u = u0 - h * a.n_rot;
        const int64_t t = t0 + tl;
        const TX *x = static_cast<const TX *>(a.x) + t * a.xs + h * a.xh + a.r.off;
        TY *y = static_cast<TY *>(a.y) + t * a.ys + h * a.yh + a.r.off;
        const int p = a.pos[t];
        const bool ok = p >= 0 && p < a.r.n_pos;
        const float *cs = a.r.cs + (ok ? (int64_t)p : 0) * rot;
        const float bad = ok ? 0.0f : kv_nan();
        if constexpr (!VEC) {
            const int ia = a.r.style == 0 ? u : 2 * u, ib = a.r.style == 0 ? ia + a.r.half : ia + 1;
            float va = to_f32(x[ia]), vb = to_f32(x[ib]);
            rotate(va, vb, ok ? cs[2 * u] : bad, ok ? cs[2 * u + 1] : bad);
            y[ia] = from_f32<TY>(va);
            y[ib] = from_f32<TY>(vb);
        } else if (a.r.style == 0) {
            float va[8], vb[8], c[16];
            load8(x + 8 * u, va, true);
            load8(x + a.r.half + 8 * u, vb, true);
            load8(cs + 16 * u, c, true);
            load8(cs + 16 * u + 8, c + 8, true);
#pragma unroll
            for (int j = 0; j < 8; j++) rotate(va[j], vb[j], ok ? c[2 * j] : bad, ok ? c[2 * j + 1] : bad);
            store8(y + 8 * u, va, true);
            store8(y + a.r.half + 8 * u, vb, true);
        } else {
            float v[8], c[8];
            load8(x + 8 * u, v, true);
            load8(cs + 8 * u, c, true);
#pragma unroll
            for (int j = 0; j < 4; j++) rotate(v[2 * j], v[2 * j + 1], ok ? c[2 * j] : bad, ok ? c[2 * j + 1] : bad);
            store8(y + 8 * u, v, true);
        }
    }
    if (a.in_place || !a.n_copy) return;
    const int cper = a.H * a.n_copy;
#pragma unroll 4
    for (int i = threadIdx.x; i < nt * cper; i += ROW_THREADS) {
        const int tl = (int)a.copy_tok.div(i), u0 = i - tl * cper;
        const int h = (int)a.copy_head.div(u0);
        int e = (u0 - h * a.n_copy) * (VEC ? 8 : 1);
        if (e >= a.r.off) e += rot;
        const TX *x = static_cast<const TX *>(a.x) + (t0 + tl) * a.xs + h * a.xh + e;
        TY *y = static_cast<TY *>(a.y) + (t0 + tl) * a.ys + h * a.yh + e;
        if constexpr (VEC) {
            float v[8];
            load8(x, v, true);
            store8(y, v, true);
        } else {
            *y = from_f32<TY>(to_f32(*x));
        }
    }
}

// ------------------------------------------------------------------------------------------- cache rows

struct RowArgs {
    KvView c;
    RopeView r;              // half 0: no rotation
    const int32_t *start, *pos0;
    void *x[2];              // k, v: rows read by a write, written by a read
    int64_t T, xs[2], xh[2];
    int sides, tpc, vec, rvec;
    int step, parts;         // tokens side by side in a CTA, passes of its threads over a token
    FastDiv per_tok, per_side, per_head;
};

// The rotated values of elements e .. e + 7 of a key row (its pairs may lie in another chunk, so they are read
// again there; the cache never overlaps the row).
template <class TX>
__device__ __forceinline__ void rotated8(const RowArgs &a, const TX *row, int e, int pos, float v[8]) {
    const int rot = 2 * a.r.half, r0 = e - a.r.off;
    if (r0 + 8 <= 0 || r0 >= rot) return;
    const bool ok = pos >= 0 && pos < a.r.n_pos;
    const float *cs = a.r.cs + (ok ? (int64_t)pos : 0) * rot;
    if (a.rvec && a.r.style == 0) {
        const bool first = r0 < a.r.half;
        const int j0 = first ? r0 : r0 - a.r.half;
        float w[8], c[16];
        load8(row + (first ? e + a.r.half : e - a.r.half), w, a.vec);
        load8(cs + 2 * j0, c, true);
        load8(cs + 2 * j0 + 8, c + 8, true);
#pragma unroll
        for (int j = 0; j < 8; j++) {
            float x = first ? v[j] : w[j], y = first ? w[j] : v[j];
            rotate(x, y, ok ? c[2 * j] : kv_nan(), ok ? c[2 * j + 1] : kv_nan());
            v[j] = first ? x : y;
        }
        return;
    }
    if (a.rvec) {
        float c[8];
        load8(cs + r0, c, true);
#pragma unroll
        for (int j = 0; j < 4; j++) rotate(v[2 * j], v[2 * j + 1], ok ? c[2 * j] : kv_nan(), ok ? c[2 * j + 1] : kv_nan());
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int q = r0 + i;
        if (q < 0 || q >= rot) continue;
        const bool first = a.r.style == 0 ? q < a.r.half : !(q & 1);
        const int j = a.r.style == 0 ? (first ? q : q - a.r.half) : q >> 1;
        const int mate = a.r.style == 0 ? (first ? q + a.r.half : q - a.r.half) : q ^ 1;
        const float self = to_f32(row[a.r.off + q]), other = to_f32(row[a.r.off + mate]);
        float x = first ? self : other, y = first ? other : self;
        rotate(x, y, ok ? cs[2 * j] : kv_nan(), ok ? cs[2 * j + 1] : kv_nan());
        v[i] = first ? x : y;
    }
}

// Rows of the CTA's tokens, found once per token: the pool row of head 0 (-1: no row, -2: padding) and the position.
struct Places {
    int64_t row[ROW_ITEMS];
    int pos[ROW_ITEMS];
};
// Three rounds of loads: all of start at once (the sequence of the CTA's first token is the last that starts at or before
// it; the tokens are consecutive, so the others' follow by steps), the sequence's words, the page.
__device__ __forceinline__ void find_places(const RowArgs &a, int64_t t0, int nt, Places &p) {
    const int B = a.c.n_seqs;
    int b0 = -1;
    for (int i0 = 0; i0 < B; i0 += ROW_THREADS) {
        const int i = i0 + threadIdx.x, n = __syncthreads_count(i < B && a.start[i] <= t0);
        b0 += n;
        if (n < ROW_THREADS) break;
    }
    for (int i = threadIdx.x; i < nt; i += ROW_THREADS) {
        const int64_t t = t0 + i;
        int b = max(b0, 0);
        int lo = a.start[b], hi = a.start[b + 1];
        while (t >= hi && b + 1 < B) b++, lo = hi, hi = a.start[b + 1];
        int64_t row = -2;
        int pos = -1;
        if (t >= lo && t < hi) {
            const int64_t at = (int64_t)a.pos0[b] + (t - lo);
            pos = at < 0 || at > 0x7fffffff ? -1 : (int)at;
            row = kv_row(a.c, b, pos);
        }
        p.row[i] = row, p.pos[i] = pos;
    }
    __syncthreads();
}

// What a thread of a row kernel does: eight values of one head's key or value, the same ones of ROW_AHEAD tokens of the
// CTA (every `step`-th from `first` on), so that its addresses are formed once.
struct Share {
    int first, side, h, e;
    bool on;
};
__device__ __forceinline__ Share share_at(const RowArgs &a, int part) {
    Share s;
    const int per = (int)a.per_tok.d;
    s.first = part ? 0 : (int)a.per_tok.div(threadIdx.x);      // more parts than one: a token at a time takes all threads
    int u = threadIdx.x - s.first * per + part * ROW_THREADS;
    s.on = s.first < a.step && u < per;
    s.side = (int)a.per_side.div(u);
    u -= s.side * (int)a.per_side.d;
    s.h = (int)a.per_head.div(u), s.e = (u - s.h * (int)a.per_head.d) * 8;
    return s;
}

// A thread's rows are on their way before the places are known (write), or all at once after that (read). 22026 rows of 8
// heads of 128, keys and values, bf16 to Q8: written in 49 us, read back in 38 (138 MB each, 2.8 and 3.6 TB/s). More
// than half of the issue slots are taken (rounding and packing; finding places, once a CTA), so instructions as
// much as HBM bound them; several rounds a CTA, to find places once for more rows, measured slower.
template <class TX, int CACHE>
__global__ void __launch_bounds__(ROW_THREADS) k_kv_write(const __grid_constant__ RowArgs a) {
    __shared__ Places pl;
    const int64_t t0 = (int64_t)blockIdx.x * a.tpc;
    const int nt = (int)min((int64_t)a.tpc, a.T - t0);
    for (int part = 0; part < a.parts; part++) {
        const Share s = share_at(a, part);
        const int64_t xs = s.side ? a.xs[1] : a.xs[0];
        const TX *x = static_cast<const TX *>(s.side ? a.x[1] : a.x[0]) + (t0 + s.first) * xs + s.h * (s.side ? a.xh[1] : a.xh[0]);
        float v[ROW_AHEAD][8];
#pragma unroll
        for (int k = 0; k < ROW_AHEAD; k++) {
#pragma unroll
            for (int j = 0; j < 8; j++) v[k][j] = 0.0f;
            if (s.on && s.first + k * a.step < nt) load8(x + k * a.step * xs + s.e, v[k], a.vec);
        }
        if (part == 0) find_places(a, t0, nt, pl);
        if (s.side == 0 && a.r.half)
#pragma unroll
            for (int k = 0; k < ROW_AHEAD; k++) {
                const int tl = s.first + k * a.step;
                if (s.on && tl < nt && pl.row[tl] >= 0) rotated8(a, x + k * a.step * xs, s.e, pl.pos[tl], v[k]);
            }
        float d = 0.0f, inv = 0.0f;      // Q8: lane j of a block's eight has the scale of token j % 4 and its inverse
        if constexpr (CACHE == Q8) {
            // Eight lanes hold a block: a head's pieces are a multiple of eight, in lane order. The largest magnitude as bits, so
            // that NaN and infinities come out on top; two divisions a thread for its four tokens.
            uint32_t amax[ROW_AHEAD];
#pragma unroll
            for (int k = 0; k < ROW_AHEAD; k++) {
                amax[k] = 0;
#pragma unroll
                for (int j = 0; j < 8; j++) amax[k] = max(amax[k], __float_as_uint(v[k][j]) & 0x7fffffffu);
#pragma unroll
                for (int w = 4; w >= 1; w >>= 1) amax[k] = max(amax[k], __shfl_xor_sync(0xffffffffu, amax[k], w));
            }
            static_assert(ROW_AHEAD == 4, "a lane's share of the scales");
            const uint32_t m01 = threadIdx.x & 1 ? amax[1] : amax[0], m23 = threadIdx.x & 1 ? amax[3] : amax[2];
            const uint32_t m = threadIdx.x & 2 ? m23 : m01;
            d = __fdiv_rn(__uint_as_float(m), 127.0f);
            inv = d != 0.0f ? __fdiv_rn(1.0f, d) : 0.0f;
            if (m >= 0x7f800000u) d = inv = kv_nan();
        }
        uint8_t *pool = static_cast<uint8_t *>(s.side ? a.c.v : a.c.k);
        float *scales = (s.side ? a.c.vs : a.c.ks) + s.e / KV_BLOCK;
        const int64_t head = (int64_t)s.h << a.c.pt_log2;
#pragma unroll
        for (int k = 0; k < ROW_AHEAD; k++) {
            const float dk = CACHE == Q8 ? __shfl_sync(0xffffffffu, d, (threadIdx.x & 24) + k) : 0.0f;
            const float ik = CACHE == Q8 ? __shfl_sync(0xffffffffu, inv, (threadIdx.x & 24) + k) : 0.0f;
            const int tl = s.first + k * a.step;
            if (!s.on || tl >= nt || pl.row[tl] < 0) continue;
            const int64_t row = pl.row[tl] + head;
            if constexpr (CACHE == Q8) {
                uint32_t q[8];
                if (fabsf(ik) < kv_inf()) {      // |x * inv| < 127.5: the sum's low byte is the rounded code
#pragma unroll
                    for (int j = 0; j < 8; j++) q[j] = __float_as_uint(__fadd_rn(__fmul_rn(v[k][j], ik), 12582912.0f));
                } else {                         // 1 / scale past f32's range (or no scale): 0 and the ends
#pragma unroll
                    for (int j = 0; j < 8; j++) q[j] = v[k][j] > 0.0f ? 127u : v[k][j] < 0.0f ? 129u : 0u;
                }
                auto pack = [](uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
                    return __byte_perm(__byte_perm(a0, a1, 0x0040), __byte_perm(a2, a3, 0x0040), 0x5410);
                };
                *reinterpret_cast<uint2 *>(pool + row * a.c.hd + s.e) = make_uint2(pack(q[0], q[1], q[2], q[3]), pack(q[4], q[5], q[6], q[7]));
                if (s.e % KV_BLOCK == 0) scales[row * (a.c.hd / KV_BLOCK)] = dk;
            } else if constexpr (CACHE == F16) {
                store8(reinterpret_cast<__half *>(pool) + row * a.c.hd + s.e, v[k], true);
            } else {
                store8(reinterpret_cast<__nv_bfloat16 *>(pool) + row * a.c.hd + s.e, v[k], true);
            }
        }
    }
}

template <class TY, int CACHE>
__global__ void __launch_bounds__(ROW_THREADS) k_kv_read(const __grid_constant__ RowArgs a) {
    __shared__ Places pl;
    const int64_t t0 = (int64_t)blockIdx.x * a.tpc;
    const int nt = (int)min((int64_t)a.tpc, a.T - t0);
    find_places(a, t0, nt, pl);
    for (int part = 0; part < a.parts; part++) {
        const Share s = share_at(a, part);
        if (!s.on) continue;
        const uint8_t *pool = static_cast<const uint8_t *>(s.side ? a.c.v : a.c.k);
        const float *scales = (s.side ? a.c.vs : a.c.ks) + s.e / KV_BLOCK;
        const int64_t head = (int64_t)s.h << a.c.pt_log2;
        uint4 raw[ROW_AHEAD];
        float d[ROW_AHEAD];
#pragma unroll
        for (int k = 0; k < ROW_AHEAD; k++) {
            const int tl = s.first + k * a.step;
            raw[k] = make_uint4(0, 0, 0, 0), d[k] = kv_nan();
            if (tl >= nt || pl.row[tl] < 0) continue;
            const int64_t row = pl.row[tl] + head;
            if constexpr (CACHE == Q8) {
                const uint2 q = *reinterpret_cast<const uint2 *>(pool + row * a.c.hd + s.e);
                raw[k].x = q.x, raw[k].y = q.y;
                d[k] = scales[row * (a.c.hd / KV_BLOCK)];
            } else {
                raw[k] = *reinterpret_cast<const uint4 *>(pool + (row * a.c.hd + s.e) * 2);
            }
        }
        const int64_t xs = s.side ? a.xs[1] : a.xs[0];
        TY *y = static_cast<TY *>(s.side ? a.x[1] : a.x[0]) + (t0 + s.first) * xs + s.h * (s.side ? a.xh[1] : a.xh[0]) + s.e;
#pragma unroll
        for (int k = 0; k < ROW_AHEAD; k++) {
            const int tl = s.first + k * a.step;
            if (tl >= nt || pl.row[tl] == -2) continue;
            float v[8];
            if constexpr (CACHE == Q8) {
                codes4(raw[k].x, v);
                codes4(raw[k].y, v + 4);
#pragma unroll
                for (int j = 0; j < 8; j++) v[j] = __fmul_rn(v[j], d[k]);
            } else {
                const bool none = pl.row[tl] < 0;
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const uint32_t w = (&raw[k].x)[j >> 1], h = j & 1 ? w >> 16 : w & 0xffffu;
                    v[j] = none ? kv_nan() : CACHE == F16 ? f16_to_f32_hw(h) : bf16_to_f32(h);
                }
            }
            store8(y + k * a.step * xs, v, a.vec);
        }
    }
}

bool rope_view(const hxb_rope *r, int head_dim, const char *who, RopeView *o, int *rc) {
    if (r->rope_dim < 2 || r->rope_dim % 2 || r->rope_dim > head_dim || r->offset < 0 ||
        r->offset > head_dim - r->rope_dim || (r->style != 0 && r->style != 1)) {
        *rc = attn_fail(HXB_E_ARG, "%s: rotation of %d values at %d (style %d) in a head of %d", who, r->rope_dim,
                        r->offset, r->style, head_dim);
        return false;
    }
    if (r->n_pos < 1 || !r->cs || !aligned(r->cs, 4)) {
        *rc = attn_fail(HXB_E_ARG, "%s: bad rotary table", who);
        return false;
    }
    o->cs = r->cs, o->n_pos = r->n_pos, o->half = r->rope_dim / 2, o->off = r->offset, o->style = r->style;
    return true;
}

// Eight-element access needs 16-byte aligned rows: the base and every stride that is used.
bool vec_rows(const void *p, int dtype, int64_t T, int64_t ts, int H, int64_t hs) {
    const int64_t n = 16 / (int64_t)elem_size(dtype);
    return aligned(p, 16) && (T < 2 || ts % n == 0) && (H < 2 || hs % n == 0);
}

bool rope_vec(const RopeView &r) {
    return aligned(r.cs, 16) && r.off % 8 == 0 && (r.style == 0 ? r.half % 8 == 0 : r.half % 4 == 0);
}

template <class TX, bool VEC>
void rope_to(const RopeArgs &a, int y_dtype, int grid, cudaStream_t s) {
    if (y_dtype == F32) k_rope<TX, float, VEC><<<grid, ROW_THREADS, 0, s>>>(a);
    else if (y_dtype == F16) k_rope<TX, __half, VEC><<<grid, ROW_THREADS, 0, s>>>(a);
    else k_rope<TX, __nv_bfloat16, VEC><<<grid, ROW_THREADS, 0, s>>>(a);
}
template <bool VEC>
void rope_from(const RopeArgs &a, int x_dtype, int y_dtype, int grid, cudaStream_t s) {
    if (x_dtype == F32) rope_to<float, VEC>(a, y_dtype, grid, s);
    else if (x_dtype == F16) rope_to<__half, VEC>(a, y_dtype, grid, s);
    else rope_to<__nv_bfloat16, VEC>(a, y_dtype, grid, s);
}

template <class T>
void rows_launch(const RowArgs &a, int cache, bool write, int grid, cudaStream_t s) {
    if (write) {
        if (cache == F16) k_kv_write<T, F16><<<grid, ROW_THREADS, 0, s>>>(a);
        else if (cache == BF16) k_kv_write<T, BF16><<<grid, ROW_THREADS, 0, s>>>(a);
        else k_kv_write<T, Q8><<<grid, ROW_THREADS, 0, s>>>(a);
    } else {
        if (cache == F16) k_kv_read<T, F16><<<grid, ROW_THREADS, 0, s>>>(a);
        else if (cache == BF16) k_kv_read<T, BF16><<<grid, ROW_THREADS, 0, s>>>(a);
        else k_kv_read<T, Q8><<<grid, ROW_THREADS, 0, s>>>(a);
    }
}

int kv_rows(const char *who, const hxb_kv_cache *c, const int32_t *start, const int32_t *pos0, int64_t T, void *k,
            int64_t ks, int64_t kh, void *v, int64_t vs, int64_t vh, int dtype, const hxb_rope *rope, bool write,
            void *stream) {
    RowArgs a = {};
    if (c && c->n_pages && !c->v && v) return attn_fail(HXB_E_ARG, "%s: v rows for a cache without v", who);
    const bool latent = c && !c->v && !v && (c->n_pages || c->n_kv_heads == 1);      // a pool of no pages has no pointers
    int rc = kv_view(c, who, latent, &a.c);
    if (rc != HXB_OK) return rc;
    if (T < 0 || T > 0x7fffffff || !io_dtype(dtype)) return attn_fail(HXB_E_ARG, "%s: bad row count or dtype", who);
    if (rope && !rope_view(rope, c->head_dim, who, &a.r, &rc)) return rc;
    if (T == 0 || c->n_seqs == 0) return HXB_OK;
    if (!start || !pos0 || !k || (!latent && !v)) return attn_fail(HXB_E_ARG, "%s: null pointer", who);
    if (!aligned(start, 4) || !aligned(pos0, 4) || !aligned(k, elem_size(dtype)) || !aligned(v, elem_size(dtype)))
        return attn_fail(HXB_E_ARG, "%s: pointer not aligned to its elements", who);
    if (ks < 0 || kh < 0 || (!latent && (vs < 0 || vh < 0)) ||
        (!write && (rows_overlap(T, ks, c->n_kv_heads, kh, c->head_dim) ||
                    (!latent && rows_overlap(T, vs, c->n_kv_heads, vh, c->head_dim)))))
        return attn_fail(HXB_E_ARG, "%s: bad strides", who);
    a.start = start, a.pos0 = pos0, a.T = T;
    a.x[0] = k, a.xs[0] = ks, a.xh[0] = kh;
    a.x[1] = v, a.xs[1] = vs, a.xh[1] = vh;
    a.sides = latent ? 1 : 2;
    a.vec = vec_rows(k, dtype, T, ks, c->n_kv_heads, kh) && (latent || vec_rows(v, dtype, T, vs, c->n_kv_heads, vh));
    a.rvec = rope && rope_vec(a.r);
    const int per_head = c->head_dim / 8, per_side = per_head * c->n_kv_heads, per = per_side * a.sides;
    a.per_head = FastDiv(per_head), a.per_side = FastDiv(per_side), a.per_tok = FastDiv(per);
    a.step = std::max(1, ROW_THREADS / per), a.parts = (per + ROW_THREADS - 1) / ROW_THREADS;
    a.tpc = a.step * ROW_AHEAD;      // one round: more of them a CTA measured slower (nothing in flight between rounds)
    const int64_t grid = (T + a.tpc - 1) / a.tpc;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (dtype == F32) rows_launch<float>(a, c->dtype, write, (int)grid, s);
    else if (dtype == F16) rows_launch<__half>(a, c->dtype, write, (int)grid, s);
    else rows_launch<__nv_bfloat16>(a, c->dtype, write, (int)grid, s);
    return attn_launched(who) ? HXB_OK : HXB_E_DEVICE;
}

}  // namespace
}  // namespace hx

using namespace hx;

extern "C" HXB_API int hxb_rope_freqs(int rope_dim, double theta, int scaling, double factor, int original,
                                      double beta_fast, double beta_slow, double *inv_freq, double *attn_factor) {
    if (rope_dim < 2 || rope_dim % 2 || rope_dim > 1024 || !(theta > 1.0) || !std::isfinite(theta) || !inv_freq || !attn_factor)
        return attn_fail(HXB_E_ARG, "rope_freqs: bad rope_dim, theta or pointer");
    if (scaling < HXB_ROPE_NONE || scaling > HXB_ROPE_YARN)
        return attn_fail(HXB_E_ARG, "rope_freqs: unknown scaling %d", scaling);
    if (scaling != HXB_ROPE_NONE && (!(factor >= 1.0) || !std::isfinite(factor)))
        return attn_fail(HXB_E_ARG, "rope_freqs: factor %g (at least 1)", factor);
    if (scaling == HXB_ROPE_NTK && rope_dim == 2) return attn_fail(HXB_E_ARG, "rope_freqs: base scaling needs rope_dim over 2");
    const double pi = 3.14159265358979323846;
    double lo = 0, hi = 0;
    if (scaling == HXB_ROPE_YARN) {
        if (original < 1 || !(beta_fast > beta_slow) || !(beta_slow > 0) || !std::isfinite(beta_fast))
            return attn_fail(HXB_E_ARG, "rope_freqs: bad original, beta_fast or beta_slow");
        // the j at which a frequency makes beta turns over the original positions (hi not above 0: none makes beta_slow)
        lo = std::floor(rope_dim * std::log(original / (beta_fast * 2 * pi)) / (2 * std::log(theta)));
        hi = std::ceil(rope_dim * std::log(original / (beta_slow * 2 * pi)) / (2 * std::log(theta)));
        lo = std::max(lo, 0.0);
        hi = std::min(hi, (double)rope_dim - 1);
    }
    const double base = scaling == HXB_ROPE_NTK ? theta * std::pow(factor, (double)rope_dim / (rope_dim - 2)) : theta;
    for (int j = 0; j < rope_dim / 2; j++) {
        const double f = std::pow(base, -2.0 * j / rope_dim);
        double keep = 1.0;
        if (scaling == HXB_ROPE_LINEAR) keep = 0.0;
        if (scaling == HXB_ROPE_YARN) keep = hi <= 0 ? 0.0 : 1.0 - std::min(std::max((j - lo) / std::max(hi - lo, 0.001), 0.0), 1.0);
        inv_freq[j] = f * keep + (scaling == HXB_ROPE_NONE || scaling == HXB_ROPE_NTK ? 0.0 : f / factor * (1.0 - keep));
    }
    *attn_factor = scaling == HXB_ROPE_YARN ? 0.1 * std::log(factor) + 1.0 : 1.0;
    return HXB_OK;
}

extern "C" HXB_API int hxb_rope_table_dev(const double *inv_freq, int rope_dim, double attn_factor, int64_t pos0,
                                          int64_t n_pos, float *cs, void *stream) {
    if (rope_dim < 2 || rope_dim % 2 || rope_dim > 1024 || !inv_freq || n_pos < 0 || pos0 <= -(1ll << 31) ||
        pos0 >= (1ll << 31) || n_pos > (1ll << 31) - std::max<int64_t>(pos0, 0))
        return attn_fail(HXB_E_ARG, "rope_table: bad rope_dim, positions or frequencies");
    if (!std::isfinite((float)attn_factor)) return attn_fail(HXB_E_ARG, "rope_table: factor %g is not finite in f32", attn_factor);
    if (n_pos == 0) return HXB_OK;
    if (!cs || !aligned(cs, 8)) return attn_fail(HXB_E_ARG, "rope_table: the table must be 8-byte aligned");
    FreqArg f;
    const double turn = 2 * 3.14159265358979323846, turn_rest = 2.4492935982947064e-16;      // 2 pi in two terms
    for (int j = 0; j < rope_dim / 2; j++) {
        if (!std::isfinite(inv_freq[j])) return attn_fail(HXB_E_ARG, "rope_table: frequency %d is not finite", j);
        const double t = inv_freq[j] / turn;
        f.turns[j] = make_double2(t, (std::fma(-t, turn, inv_freq[j]) - t * turn_rest) / turn);
    }
    f.fhi = (float)attn_factor, f.flo = (float)(attn_factor - f.fhi);
    const int half = rope_dim / 2, rows = std::max(1, TABLE_ITEMS / half);
    k_rope_table<<<(int)((n_pos + rows - 1) / rows), 256, 0, static_cast<cudaStream_t>(stream)>>>(f, half, FastDiv(half), rows, pos0, n_pos,
                                                                                               reinterpret_cast<float2 *>(cs));
    return attn_launched("rope_table") ? HXB_OK : HXB_E_DEVICE;
}

extern "C" HXB_API int hxb_rope_dev(const hxb_rope *r, const int32_t *pos, int64_t T, int n_heads, int head_dim,
                                    const void *x, int x_dtype, int64_t x_stride, int64_t x_head_stride, void *y,
                                    int y_dtype, int64_t y_stride, int64_t y_head_stride, void *stream) {
    RopeArgs a = {};
    int rc = HXB_OK;
    if (!r) return attn_fail(HXB_E_ARG, "rope: null rotation");
    if (T < 0 || T > 0x7fffffff || n_heads < 1 || n_heads > 65535 || head_dim < 2 || head_dim > 1024)
        return attn_fail(HXB_E_ARG, "rope: bad shape (%lld tokens, %d heads of %d)", (long long)T, n_heads, head_dim);
    if (!io_dtype(x_dtype) || !io_dtype(y_dtype)) return attn_fail(HXB_E_ARG, "rope: bad dtype");
    if (!rope_view(r, head_dim, "rope", &a.r, &rc)) return rc;
    if (T == 0) return HXB_OK;
    if (!pos || !x || !y) return attn_fail(HXB_E_ARG, "rope: null pointer");
    if (!aligned(pos, 4) || !aligned(x, elem_size(x_dtype)) || !aligned(y, elem_size(y_dtype)))
        return attn_fail(HXB_E_ARG, "rope: pointer not aligned to its elements");
    if (x_stride < 0 || x_head_stride < 0 || rows_overlap(T, y_stride, n_heads, y_head_stride, head_dim))
        return attn_fail(HXB_E_ARG, "rope: bad strides");
    a.in_place = x == y;
    if (a.in_place && (x_dtype != y_dtype || (T > 1 && x_stride != y_stride) || (n_heads > 1 && x_head_stride != y_head_stride)))
        return attn_fail(HXB_E_ARG, "rope: in place needs one type and one set of strides");
    a.pos = pos, a.x = x, a.y = y, a.T = T, a.xs = x_stride, a.xh = x_head_stride, a.ys = y_stride, a.yh = y_head_stride;
    a.H = n_heads, a.hd = head_dim;
    const int rot = 2 * a.r.half;
    const bool vec = head_dim % 8 == 0 && rope_vec(a.r) && rot % 8 == 0 && vec_rows(x, x_dtype, T, x_stride, n_heads, x_head_stride) &&
                     vec_rows(y, y_dtype, T, y_stride, n_heads, y_head_stride);
    a.n_rot = !vec ? a.r.half : a.r.style == 0 ? a.r.half / 8 : rot / 8;
    a.n_copy = (head_dim - rot) / (vec ? 8 : 1);
    a.rot_head = FastDiv(a.n_rot), a.rot_tok = FastDiv(a.n_rot * n_heads);
    a.copy_head = FastDiv(std::max(1, a.n_copy)), a.copy_tok = FastDiv(std::max(1, a.n_copy * n_heads));
    a.tpc = std::max(1, ROW_ITEMS / ((a.n_rot + a.n_copy) * n_heads));
    const int grid = (int)((T + a.tpc - 1) / a.tpc);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (vec) rope_from<true>(a, x_dtype, y_dtype, grid, s);
    else rope_from<false>(a, x_dtype, y_dtype, grid, s);
    return attn_launched("rope") ? HXB_OK : HXB_E_DEVICE;
}

extern "C" HXB_API int hxb_kv_write_dev(const hxb_kv_cache *c, const int32_t *start, const int32_t *pos0, int64_t T,
                                        const void *k, int64_t k_stride, int64_t k_head_stride, const void *v,
                                        int64_t v_stride, int64_t v_head_stride, int dtype, const hxb_rope *rope,
                                        void *stream) {
    return kv_rows("kv_write", c, start, pos0, T, const_cast<void *>(k), k_stride, k_head_stride, const_cast<void *>(v),
                   v_stride, v_head_stride, dtype, rope, true, stream);
}

extern "C" HXB_API int hxb_kv_read_dev(const hxb_kv_cache *c, const int32_t *start, const int32_t *pos0, int64_t T,
                                       void *k_out, int64_t k_stride, int64_t k_head_stride, void *v_out,
                                       int64_t v_stride, int64_t v_head_stride, int dtype, void *stream) {
    return kv_rows("kv_read", c, start, pos0, T, k_out, k_stride, k_head_stride, v_out, v_stride, v_head_stride, dtype,
                   nullptr, false, stream);
}
