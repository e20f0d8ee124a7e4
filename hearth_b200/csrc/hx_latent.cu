// hx_latent.cu — absorbed latent attention of one new token a sequence (hxb_latent_decode_dev; the reference's
// engine/src/model.c:739-787 in another order of summation).
#include "hx_attn.cuh"

#include <algorithm>

namespace hx {
namespace {

constexpr int AD_THREADS = 128;

__device__ __forceinline__ float pool_load(const void *pool, const float *scale, int dtype, int hd, int64_t row, int e) {
    if (dtype == Q8) return (float)static_cast<const int8_t *>(pool)[row * hd + e] * scale[row * (hd / KV_BLOCK) + e / KV_BLOCK];
    return io_load(pool, dtype, row * hd + e);
}

struct CoreArgs {
    KvView c;
    const int32_t *lens;
    const void *q;
    void *out;
    float *lse;
    int64_t qs, qh, os, oh;
    int H, dtype_c, dtype_q, dtype_o, vd, latent;
    float scale;
};

// One CTA a (head, sequence): tiles of AD_THREADS positions, a thread a score, then a thread an output value.
__global__ void __launch_bounds__(AD_THREADS) k_attn_core(const __grid_constant__ CoreArgs a) {
    __shared__ float q[1024], p[AD_THREADS], red[AD_THREADS / 32];
    __shared__ int64_t rows[AD_THREADS];
    const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
    const int g = h / (a.H / a.c.Hkv);
    for (int i = tid; i < a.c.hd; i += AD_THREADS) q[i] = io_load(a.q, a.dtype_q, b * a.qs + h * a.qh + i);
    const int n = a.lens[b];
    float m = -kv_inf(), l = 0.0f, o[8] = {};
    for (int r0 = 0; r0 < n; r0 += AD_THREADS) {
        __syncthreads();
        float s = -kv_inf();
        int64_t row = -1;
        if (r0 + tid < n) {
            row = kv_row(a.c, b, r0 + tid);
            if (row >= 0) row += (int64_t)g << a.c.pt_log2;
            float d = 0.0f;
            for (int i = 0; row >= 0 && i < a.c.hd; i++) d = __fmaf_rn(q[i], pool_load(a.c.k, a.c.ks, a.dtype_c, a.c.hd, row, i), d);
            s = row < 0 ? kv_nan() : d * a.scale;
        }
        rows[tid] = row;
        float mx = s;
        for (int k = 16; k >= 1; k >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, k));
        if (tid % 32 == 0) red[tid / 32] = mx;
        __syncthreads();
        float m2 = m;
        for (int k = 0; k < AD_THREADS / 32; k++) m2 = fmaxf(m2, red[k]);
        const float base = m2 == -kv_inf() ? 0.0f : m2;
        const float fade = expf(m - base);
        p[tid] = expf(s - base);
        __syncthreads();
        l *= fade;
        for (int k = 0; k < AD_THREADS; k++) l += p[k];
        const int lim = min(AD_THREADS, n - r0);
        for (int j = 0; j < 8; j++) {
            const int e = tid + j * AD_THREADS;
            if (e >= a.vd) break;
            float x = o[j] * fade;
            for (int k = 0; k < lim; k++)
                if (rows[k] >= 0)
                    x = __fmaf_rn(p[k], a.latent ? pool_load(a.c.k, a.c.ks, a.dtype_c, a.c.hd, rows[k], e)
                                                 : pool_load(a.c.v, a.c.vs, a.dtype_c, a.c.hd, rows[k], e), x);
                else x = kv_nan();
            o[j] = x;
        }
        m = m2;
    }
    for (int j = 0; j < 8; j++) {
        const int e = tid + j * AD_THREADS;
        if (e < a.vd) io_store(a.out, a.dtype_o, b * a.os + h * a.oh + e, l == 0.0f ? 0.0f : o[j] / l);
    }
    if (a.lse && tid == 0) a.lse[(int64_t)b * a.H + h] = l == 0.0f ? -kv_inf() : (m == -kv_inf() ? 0.0f : m) + logf(l);
}

struct SideArgs {
    const void *q, *w;
    float *qa, *o;
    void *out;
    int64_t qs, qh, os, oh;
    int H, R, dr, dn, dv, dtype;
};

// qa[b][h] = [sum_d q[d] w[h][d] | q's rotated part] in f32.
__global__ void k_latent_absorb(const __grid_constant__ SideArgs a) {
    const int h = blockIdx.x, b = blockIdx.y;
    float *qa = a.qa + ((int64_t)b * a.H + h) * (a.R + a.dr);
    const int64_t q0 = b * a.qs + h * a.qh, w0 = (int64_t)h * (a.dn + a.dv) * a.R;
    for (int r = threadIdx.x; r < a.R + a.dr; r += blockDim.x) {
        float x = 0.0f;
        if (r < a.R)
            for (int d = 0; d < a.dn; d++) x = __fmaf_rn(io_load(a.q, a.dtype, q0 + d), io_load(a.w, a.dtype, w0 + (int64_t)d * a.R + r), x);
        else x = io_load(a.q, a.dtype, q0 + a.dn + r - a.R);
        qa[r] = x;
    }
}

// out[b][h][j] = o[b][h] . w[h][dn + j]
__global__ void k_latent_expand(const __grid_constant__ SideArgs a) {
    const int h = blockIdx.x, b = blockIdx.y;
    const float *o = a.o + ((int64_t)b * a.H + h) * a.R;
    for (int j = threadIdx.x; j < a.dv; j += blockDim.x) {
        const int64_t w0 = ((int64_t)h * (a.dn + a.dv) + a.dn + j) * a.R;
        float x = 0.0f;
        for (int r = 0; r < a.R; r++) x = __fmaf_rn(o[r], io_load(a.w, a.dtype, w0 + r), x);
        io_store(a.out, a.dtype, b * a.os + h * a.oh + j, x);
    }
}

bool aligned(const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

}  // namespace
}  // namespace hx

using namespace hx;

extern "C" HXB_API size_t hxb_latent_decode_workspace(const hxb_kv_cache *c, int n_heads, int rank) {
    if (!c || n_heads < 1 || rank < 1 || c->n_seqs < 0) return 0;
    return ((size_t)c->n_seqs * n_heads * ((size_t)c->head_dim + rank)) * 4 + 16;
}

extern "C" HXB_API int hxb_latent_decode_dev(const hxb_kv_cache *c, const int32_t *lens, const void *q, int64_t q_stride,
                                             int64_t q_head_stride, const void *w, int n_heads, int rank, int nope,
                                             int v_dim, int dtype, float scale, void *out, int64_t out_stride,
                                             int64_t out_head_stride, void *ws, size_t ws_bytes, void *stream) {
    CoreArgs a = {};
    int rc = kv_view(c, "latent_decode", true, &a.c);
    if (rc != HXB_OK) return rc;
    if (dtype != F16 && dtype != BF16) return attn_fail(HXB_E_ARG, "latent_decode: dtype %d (F16 or BF16)", dtype);
    if (c->dtype != Q8 && c->dtype != dtype)
        return attn_fail(HXB_E_ARG, "latent_decode: the cache is Q8 or has the type of q");
    const int dr = c->head_dim - rank;
    if (rank < 128 || rank > 512 || rank % 128 || dr < 16 || dr > 64 || dr % 16)
        return attn_fail(HXB_E_UNSUPPORTED, "latent_decode: rank %d in rows of %d (rank a multiple of 128 up to 512, 16 to 64 more)",
                         rank, c->head_dim);
    if (nope < 16 || nope > 256 || nope % 16 || v_dim < 16 || v_dim > 256 || v_dim % 16)
        return attn_fail(HXB_E_UNSUPPORTED, "latent_decode: nope %d, v_dim %d (multiples of 16 up to 256)", nope, v_dim);
    if (n_heads < 1 || n_heads > 256) return attn_fail(HXB_E_ARG, "latent_decode: %d heads (up to 256)", n_heads);
    if (c->n_seqs == 0) return HXB_OK;
    rc = attn_check_io("latent_decode", c->n_seqs, n_heads, q, q_stride, q_head_stride, out, out_stride, out_head_stride, v_dim, dtype,
                       lens, scale);
    if (rc != HXB_OK) return rc;
    if (!w || !aligned(w, 16)) return attn_fail(HXB_E_ARG, "latent_decode: w must be 16-byte aligned");
    if (!ws || !aligned(ws, 16) || ws_bytes < hxb_latent_decode_workspace(c, n_heads, rank))
        return attn_fail(HXB_E_ARG, "latent_decode: workspace of %zu bytes, 16-byte aligned, needed",
                         hxb_latent_decode_workspace(c, n_heads, rank));
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    SideArgs e = {};
    e.q = q, e.w = w, e.qa = static_cast<float *>(ws), e.o = e.qa + (size_t)c->n_seqs * n_heads * c->head_dim, e.out = out;
    e.qs = q_stride, e.qh = q_head_stride, e.os = out_stride, e.oh = out_head_stride;
    e.H = n_heads, e.R = rank, e.dr = dr, e.dn = nope, e.dv = v_dim, e.dtype = dtype;
    a.lens = lens, a.q = e.qa, a.qs = (int64_t)n_heads * c->head_dim, a.qh = c->head_dim, a.out = e.o;
    a.os = (int64_t)n_heads * rank, a.oh = rank, a.H = n_heads, a.dtype_c = c->dtype, a.dtype_q = a.dtype_o = F32;
    a.vd = rank, a.latent = 1, a.scale = scale;
    const dim3 grid(n_heads, c->n_seqs);
    k_latent_absorb<<<grid, 128, 0, s>>>(e);
    k_attn_core<<<grid, AD_THREADS, 0, s>>>(a);
    k_latent_expand<<<grid, 128, 0, s>>>(e);
    return attn_launched("latent_decode") ? HXB_OK : HXB_E_DEVICE;
}
