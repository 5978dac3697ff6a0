// What the paged cache's kernels share: element types, the 8-bit code
// conversions, a sequence's extent as the device arrays give it, and the
// host's checks of the descriptors.
#pragma once

#include "wm_internal.h"

typedef float wm_f4 __attribute__((ext_vector_type(4)));
typedef float wm_f16v __attribute__((ext_vector_type(16)));
typedef _Float16 wm_h2 __attribute__((ext_vector_type(2)));
typedef _Float16 wm_h4 __attribute__((ext_vector_type(4)));
typedef _Float16 wm_h8 __attribute__((ext_vector_type(8)));
typedef __bf16 wm_b4 __attribute__((ext_vector_type(4)));
typedef unsigned int wm_u2 __attribute__((ext_vector_type(2)));
typedef unsigned int wm_u4 __attribute__((ext_vector_type(4)));

// ---------------------------------------------------------------------------
// elements: four at a time (16 bytes of f32, 8 of the half types)
// ---------------------------------------------------------------------------
__device__ __forceinline__ wm_f4 wm_ld4(const float *p) { return *(const wm_f4 *)p; }
__device__ __forceinline__ wm_f4 wm_ld4(const _Float16 *p) {
    return __builtin_convertvector(*(const wm_h4 *)p, wm_f4);
}
__device__ __forceinline__ wm_f4 wm_ld4(const __bf16 *p) {
    const wm_u2 u = *(const wm_u2 *)p;
    wm_f4 r;
    r.x = __uint_as_float(u.x << 16);
    r.y = __uint_as_float(u.x & 0xFFFF0000u);
    r.z = __uint_as_float(u.y << 16);
    r.w = __uint_as_float(u.y & 0xFFFF0000u);
    return r;
}
__device__ __forceinline__ void wm_st4(float *p, wm_f4 v) { *(wm_f4 *)p = v; }
__device__ __forceinline__ void wm_st4(_Float16 *p, wm_f4 v) { *(wm_h4 *)p = __builtin_convertvector(v, wm_h4); }
__device__ __forceinline__ void wm_st4(__bf16 *p, wm_f4 v) { *(wm_b4 *)p = __builtin_convertvector(v, wm_b4); }

// ---------------------------------------------------------------------------
// a sequence of the step
// ---------------------------------------------------------------------------

// The arrays are device contents that no host check has seen: tok0 and n
// always lie within the packed arrays, and a sequence with `ok` has all its
// tokens there and its positions within the bounds the grid and the page table
// were sized for.
struct wm_seq {
    int tok0, n;  // first packed token, tokens
    int start;    // position of the first (negative: that many tokens have none)
    int len;      // positions, the step's included
    bool ok;
};
__device__ __forceinline__ wm_seq wm_load_seq(const wm_paged_batch &b, uint32_t s) {
    wm_seq q;
    const int c0 = b.cu_tokens[s], c1 = b.cu_tokens[s + 1], len = b.kv_len[s];
    const int most = (int)b.n_tokens;
    q.tok0 = min(max(c0, 0), most);
    q.n = min(max(c1, q.tok0), most) - q.tok0;
    q.len = len;
    q.ok = c0 >= 0 && c1 >= c0 && c1 <= most && (s != 0 || c0 == 0) && len >= 0 && len <= (int)b.max_kv_len &&
           q.n <= (int)b.max_new;
    q.start = q.ok ? len - q.n : 0;
    return q;
}

// ---------------------------------------------------------------------------
// host checks (k_paged.hip)
// ---------------------------------------------------------------------------
size_t wm_dtype_size(int type);  // 0: none of wm_dtype
// The descriptors' own fields; `who` begins the message.
wm_status wm_paged_check(wm_ctx *ctx, const char *who, const wm_paged_kv *kv, const wm_paged_batch *b);
// One packed array: `heads` heads of head_dim values per token, tokens `stride` apart.
wm_status wm_paged_check_array(wm_ctx *ctx, const char *who, const char *name, const void *p, uint64_t stride,
                               uint32_t heads, uint32_t head_dim, size_t elem);
// An output over its own queries: only with their stride.
wm_status wm_paged_check_over(wm_ctx *ctx, const char *who, const void *q, uint64_t q_stride, const void *out,
                              uint64_t out_stride);
// Makes the context's device current for the call and the caller's again at its end.
struct wm_device_guard {
    int before = -1;
    hipError_t err;
    explicit wm_device_guard(int device) {
        err = hipGetDevice(&before);
        if (err == hipSuccess && before != device) err = hipSetDevice(device);
        else before = -1;
    }
    ~wm_device_guard() {
        if (before >= 0) (void)hipSetDevice(before);
    }
};
