// hx_paged.cuh — what the paged-cache kernels share: element types, 8-element loads and stores, the
// device view of a hxb_kv_cache and its page lookups.
#pragma once

#include "../../include/hearth_b200.h"
#include "hx_device.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace hx {

constexpr int KV_BLOCK = 64;   // values under one scale in a Q8 cache (the activation blocks' size)

__device__ __forceinline__ float kv_inf() { return __uint_as_float(0x7f800000u); }
__device__ __forceinline__ float kv_nan() { return __uint_as_float(CANON_NAN); }

template <class T> __device__ __forceinline__ float to_f32(T x);
template <> __device__ __forceinline__ float to_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ float to_f32<__half>(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <class T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// Eight consecutive elements; vec: p is 16-byte aligned.
template <class T>
__device__ __forceinline__ void load8(const T *p, float x[8], bool vec) {
    if (!vec) {
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = to_f32(p[i]);
        return;
    }
    if constexpr (sizeof(T) == 4) {
        const float4 a = reinterpret_cast<const float4 *>(p)[0], b = reinterpret_cast<const float4 *>(p)[1];
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
        const uint4 a = *reinterpret_cast<const uint4 *>(p);
        const T *h = reinterpret_cast<const T *>(&a);
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = to_f32(h[i]);
    }
}

template <class T>
__device__ __forceinline__ void store8(T *p, const float x[8], bool vec) {
    if (!vec) {
#pragma unroll
        for (int i = 0; i < 8; i++) p[i] = from_f32<T>(x[i]);
        return;
    }
    if constexpr (sizeof(T) == 4) {
        reinterpret_cast<float4 *>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
        reinterpret_cast<float4 *>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
        uint4 a;
        T *h = reinterpret_cast<T *>(&a);
#pragma unroll
        for (int i = 0; i < 8; i++) h[i] = from_f32<T>(x[i]);
        *reinterpret_cast<uint4 *>(p) = a;
    }
}

// The four signed bytes of w as floats, exactly: 2^23 + (byte + 128) assembled as bits, less 2^23 + 128 (an int-to-float
// conversion runs at a quarter of the rate).
__device__ __forceinline__ void codes4(uint32_t w, float o[4]) {
    w ^= 0x80808080u;
    o[0] = __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7540)) - 8388736.0f;
    o[1] = __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7541)) - 8388736.0f;
    o[2] = __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7542)) - 8388736.0f;
    o[3] = __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7543)) - 8388736.0f;
}

// i / d for 32-bit i by one multiply: exact for i < 2^31 and 1 <= d < 2^31 (round-up magic number with
// s = ceil(log2 d), m = floor(2^32 (2^s - d) / d) + 1).
struct FastDiv {
    uint32_t d = 1, m = 0, s = 0;
    FastDiv() = default;
    explicit FastDiv(uint32_t v) : d(v) {
        while (s < 31 && (1u << s) < v) s++;
        m = (uint32_t)(((1ull << 32) * ((1ull << s) - v)) / v + 1);
    }
    __device__ __forceinline__ uint32_t div(uint32_t i) const { return (uint32_t)(__umulhi(m, i) + i) >> s; }
};

// A hxb_kv_cache as the kernels take it.
struct KvView {
    void *k, *v;
    float *ks, *vs;
    const int32_t *table;
    int64_t table_stride, n_pages;
    int table_pages, n_seqs, Hkv, hd, pt_log2;
};

// Row (head 0) of position pos of sequence b, counted in head-0 rows of the pool; heads are page_tokens rows
// apart. -1 where the page table has no page of the pool for it.
__device__ __forceinline__ int64_t kv_row(const KvView &c, int b, int pos) {
    const int pi = pos >> c.pt_log2;
    if (pos < 0 || pi >= c.table_pages) return -1;
    const int page = c.table[(int64_t)b * c.table_stride + pi];
    if (page < 0 || page >= c.n_pages) return -1;
    return (((int64_t)page * c.Hkv) << c.pt_log2) + (pos & ((1 << c.pt_log2) - 1));
}

// Fills a view from a checked hxb_kv_cache; code and message as the entry points report them (who: the entry
// point's name). With latent set the cache has one row for keys and values.
int kv_view(const hxb_kv_cache *c, const char *who, bool latent, KvView *out);

// The message hxb_last_error() returns, and the code back (hx_attention.cu).
int attn_fail(int code, const char *fmt, ...);
bool rows_overlap(int64_t T, int64_t ts, int H, int64_t hs, int n);
bool attn_launched(const char *who);   // the last launch's status; sets the message

}  // namespace hx
