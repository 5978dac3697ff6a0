// The paged 8-bit KV cache: append with the rotation applied, read back.
//
// A block is one kv head's positions in one page, with one scale for K and
// one for V.  One workgroup serves one block of one sequence: it owns the
// block for the launch (two sequences may not append into one page), so the
// maximum, the codes and the scale need no exchange between workgroups.
#include <algorithm>
#include <cstdio>
#include <cstring>
#include <new>
#include <vector>

#include "wm_paged.h"

namespace {

constexpr int NT = 256;  // threads per workgroup, four waves

// Quotient a / s of two f32 (s > 0) rounded half away from zero, within
// +-127, exactly: inv = 1 / s in f64 makes |a| * inv good to 2^-51 relative.
// A quotient that is no tie lies at least 2^-33 away from one (a and (k + .5) s
// differ by 2^-32 of either at least: both have 32 bits), so adding 2^-40
// takes the ties up and nothing else.
__device__ __forceinline__ int quotient_code(float a, double inv) {
    const double t = fabs((double)a) * inv + (0.5 + 0x1p-40);
    const int m = t < 127.0 ? (int)t : (t >= 127.0 ? 127 : 0);  // NaN: 0
    return a < 0.0f ? -m : m;
}
__device__ __forceinline__ uint32_t pack_codes(int a, int b, int c, int d) {
    return (a & 255) | (b & 255) << 8 | (c & 255) << 16 | (uint32_t)d << 24;
}
__device__ __forceinline__ uint32_t quotient4(wm_f4 v, double inv) {
    return pack_codes(quotient_code(v.x, inv), quotient_code(v.y, inv), quotient_code(v.z, inv), quotient_code(v.w, inv));
}
__device__ __forceinline__ int byte_of(uint32_t w, int i) { return (int)(w << (24 - 8 * i)) >> 24; }
// Earlier codes under a grown scale: c * s_old is exact in f32's products
// only as f64 (7 + 24 bits), so the quotient is rounded the same way.
__device__ __forceinline__ int rescale_code(int c, double ratio) {
    const double t = fabs((double)c) * ratio + (0.5 + 0x1p-40);
    const int m = t < 127.0 ? (int)t : 127;
    return c < 0 ? -m : m;
}
__device__ __forceinline__ uint32_t rescale4(uint32_t w, double ratio) {
    return pack_codes(rescale_code(byte_of(w, 0), ratio), rescale_code(byte_of(w, 1), ratio),
                      rescale_code(byte_of(w, 2), ratio), rescale_code(byte_of(w, 3), ratio));
}

// |v| where v is finite, else 0.
__device__ __forceinline__ float finite_abs(float v) {
    const float a = fabsf(v);
    return a <= 3.402823466e38f ? a : 0.0f;
}
__device__ __forceinline__ float finite_abs4(wm_f4 v) {
    return fmaxf(fmaxf(finite_abs(v.x), finite_abs(v.y)), fmaxf(finite_abs(v.z), finite_abs(v.w)));
}

// A head is taken in units of 8 dims, as two runs of 4 that hold whole
// pairs: unit u < n_rot / 8 of the half layout is (4u.., n_rot / 2 + 4u..),
// every other unit 8 dims in a row.
struct unit_dims {
    int a, b;
    bool rot;
};
__device__ __forceinline__ unit_dims dims_of(int u, int n_rot, bool half) {
    unit_dims d;
    d.rot = 8 * u < n_rot;
    const bool split = d.rot && half;
    d.a = split ? 4 * u : 8 * u;
    d.b = split ? n_rot / 2 + 4 * u : 8 * u + 4;
    return d;
}
// The rotation of one unit's four pairs: products exact in f64 (48 bits), one
// rounding of their sum to f64 and one of that to f32.
__device__ __forceinline__ float rot_lo(float x, float y, float c, float s) {
    return (float)__builtin_fma((double)x, (double)c, -((double)y * (double)s));
}
__device__ __forceinline__ float rot_hi(float x, float y, float c, float s) {
    return (float)__builtin_fma((double)y, (double)c, (double)x * (double)s);
}
__device__ __forceinline__ void rotate_unit(wm_f4 &a, wm_f4 &b, wm_f4 c, wm_f4 s, bool half) {
    if (half) {
        wm_f4 x = a, y = b;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            a[i] = rot_lo(x[i], y[i], c[i], s[i]);
            b[i] = rot_hi(x[i], y[i], c[i], s[i]);
        }
    } else {
        wm_f4 x = a, y = b;
        a[0] = rot_lo(x[0], x[1], c[0], s[0]);
        a[1] = rot_hi(x[0], x[1], c[0], s[0]);
        a[2] = rot_lo(x[2], x[3], c[1], s[1]);
        a[3] = rot_hi(x[2], x[3], c[1], s[1]);
        b[0] = rot_lo(y[0], y[1], c[2], s[2]);
        b[1] = rot_hi(y[0], y[1], c[2], s[2]);
        b[2] = rot_lo(y[2], y[3], c[3], s[3]);
        b[3] = rot_hi(y[2], y[3], c[3], s[3]);
    }
}

struct append_args {
    wm_paged_kv kv;
    wm_paged_batch b;
    wm_rope rope;  // n_rot 0: none
    const void *q, *k, *v;
    void *q_out;
    uint64_t qs, ks, vs, qos;  // elements between tokens
    uint32_t group;            // query heads per kv head (0: no queries)
    uint32_t touch;            // pages a sequence can touch, at most
    uint32_t seq0;             // the launch's first sequence
    uint32_t blocks;           // of the launch's sequences, at most
    bool by_kind;              // order of the workgroups (k_paged_append)
};

// One block's place in the step: sequence s, its page lp, kv head h, of a
// launch's id-th from sequence seq0 on.
struct block_place {
    wm_seq q;
    int lp, h, page;
    uint32_t n_pages;
    bool live;  // positions of the step lie in it
    __device__ __forceinline__ bool stored() const { return (uint32_t)page < n_pages; }  // its page is in the pool
};
__device__ __forceinline__ block_place place_block(const wm_paged_kv &kv, const wm_paged_batch &b, uint32_t touch,
                                                   uint32_t seq0, uint32_t id) {
    block_place p;
    p.h = id % kv.n_kv_heads;
    const uint32_t sm = id / kv.n_kv_heads, s = seq0 + sm / touch;
    p.q = wm_load_seq(b, s);
    p.lp = max(p.q.start, 0) / (int)kv.page_size + (int)(sm % touch);
    p.live = p.q.ok && p.q.n > 0 && (int64_t)p.lp * kv.page_size < p.q.len;
    p.page = p.live ? b.page_table[(uint64_t)s * b.table_stride + p.lp] : -1;
    p.n_pages = kv.n_pages;
    return p;
}

// Append.  Bound by the bytes of q, k, v in and q out (the codes are a
// quarter of f32's), and for a decode step by latency: the chain is lengths,
// page id, old scale, and the earlier codes of a block are loaded with the
// scale, before it is known whether they change.  A block's keys, its values
// and the queries of 16 of its positions are a workgroup each: one workgroup
// for all three left 250 long ones in a step of 24 sequences in pages of 64
// positions, 33.5 us against 19.2.
//
// Measured (20 query heads over 5, f32, pages of 16): 16 sequences of one
// token 4.9 us, a launch's length; 8 prompts of 100 to 2000 tokens 61 us, and
// 14 to read them back, the time that the 360 MB of both take at the rate of
// a large copy (4.7 TB/s).

// Queries of slots [first, hi) of 16: a thread has 8 dims of one position in
// every head of the kv head's group, so the angles are loaded once.
template <typename T, int D>
__device__ __forceinline__ void append_queries(const append_args &a, const block_place &p, int base, int first, int hi,
                                               int64_t tok) {
    const int n_rot = (int)a.rope.n_rot, slot = (int)threadIdx.x / (D / 8), u = (int)threadIdx.x % (D / 8);
    const bool half = a.rope.layout == WM_ROPE_HALF;
    for (int t = first + slot; t < hi; t += NT / (D / 8)) {
        const unit_dims d = dims_of(u, n_rot, half);
        const T *row = (const T *)a.q + (uint64_t)(tok + t) * a.qs + (uint64_t)p.h * a.group * D;
        T *out = (T *)a.q_out + (uint64_t)(tok + t) * a.qos + (uint64_t)p.h * a.group * D;
        wm_f4 c = {1, 1, 1, 1}, s = {0, 0, 0, 0};
        if (d.rot) {
            const uint64_t at = (uint64_t)(base + t) * (n_rot / 2) + 4 * u;
            c = *(const wm_f4 *)(a.rope.cos + at), s = *(const wm_f4 *)(a.rope.sin + at);
        }
        for (uint32_t g0 = 0; g0 < a.group; g0 += 4) {  // four heads' loads together
            wm_f4 x[4], y[4];
#pragma unroll
            for (int g = 0; g < 4; g++) {
                const uint32_t h = min(g0 + g, a.group - 1) * D;
                x[g] = wm_ld4(row + h + d.a), y[g] = wm_ld4(row + h + d.b);
            }
#pragma unroll
            for (int g = 0; g < 4; g++) {
                if (g0 + g >= a.group) break;
                if (d.rot) rotate_unit(x[g], y[g], c, s, half);
                wm_st4(out + (g0 + g) * D + d.a, x[g]);
                wm_st4(out + (g0 + g) * D + d.b, y[g]);
            }
        }
    }
}

// The block's new scale from its new values' maximum and its old scale, and
// what quotients by it need.
struct block_scale {
    float s;
    double inv, ratio;
    bool grew;
    __device__ __forceinline__ block_scale(float most, float old, float *red) {
        most = wm_wave_max_nonneg(most);
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = most;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < NT / 64; w++) most = fmaxf(most, red[w]);
        s = fmaxf(old, (float)((double)most / 127.0));
        inv = s > 0.0f ? 1.0 / (double)s : 0.0;
        ratio = (double)old * inv;
        grew = s > old;
    }
};

// Keys: a thread's units are 8 dims of one position.
template <typename T, int PS, int D>
__device__ __forceinline__ void append_keys(const append_args &a, const block_place &p, int base, int first, int hi,
                                            int64_t tok, float *red) {
    constexpr int N = (PS * D / 8 + NT - 1) / NT;
    const int tid = threadIdx.x, n_rot = (int)a.rope.n_rot;
    const bool half = a.rope.layout == WM_ROPE_HALF;
    const T *k = (const T *)a.k + (uint64_t)p.h * D;
    wm_f4 x[N], y[N], c[N], s[N];
    uint32_t ox[N], oy[N];
    // the new keys' loads go out before the page's id is here
#pragma unroll
    for (int i = 0; i < N; i++) {
        const int unit = tid + i * NT, slot = unit / (D / 8), u = unit % (D / 8);
        const unit_dims d = dims_of(u, n_rot, half);
        x[i] = y[i] = wm_f4{0, 0, 0, 0};
        c[i] = s[i] = wm_f4{0, 0, 0, 0};
        if (slot >= first && slot < hi) {
            const T *row = k + (uint64_t)(tok + slot) * a.ks;
            x[i] = wm_ld4(row + d.a), y[i] = wm_ld4(row + d.b);
            if (d.rot) {
                const uint64_t at = (uint64_t)(base + slot) * (n_rot / 2) + 4 * u;
                c[i] = *(const wm_f4 *)(a.rope.cos + at), s[i] = *(const wm_f4 *)(a.rope.sin + at);
            }
        }
    }
    if (!p.stored()) return;
    const uint64_t blk = (uint64_t)p.page * a.kv.n_kv_heads + p.h;
    int8_t *codes = a.kv.k_codes + blk * (PS * D);
    const float old = first > 0 ? a.kv.k_scales[blk] : 0.0f;
#pragma unroll
    for (int i = 0; i < N; i++) {
        const int unit = tid + i * NT, slot = unit / (D / 8);
        const unit_dims d = dims_of(unit % (D / 8), n_rot, half);
        ox[i] = oy[i] = 0;
        if (slot < first) {
            ox[i] = *(const uint32_t *)(codes + slot * D + d.a);
            oy[i] = *(const uint32_t *)(codes + slot * D + d.b);
        }
    }
    float most = 0.0f;
#pragma unroll
    for (int i = 0; i < N; i++) {
        const int u = (tid + i * NT) % (D / 8);
        if (8 * u < n_rot) rotate_unit(x[i], y[i], c[i], s[i], half);
        most = fmaxf(most, fmaxf(finite_abs4(x[i]), finite_abs4(y[i])));
    }
    const block_scale b(most, old, red);
#pragma unroll
    for (int i = 0; i < N; i++) {
        const int unit = tid + i * NT, slot = unit / (D / 8);
        const unit_dims d = dims_of(unit % (D / 8), n_rot, half);
        uint32_t *wx = (uint32_t *)(codes + slot * D + d.a), *wy = (uint32_t *)(codes + slot * D + d.b);
        if (slot >= hi) continue;
        if (slot >= first) {
            *wx = quotient4(x[i], b.inv);
            *wy = quotient4(y[i], b.inv);
        } else if (b.grew) {
            *wx = rescale4(ox[i], b.ratio);
            *wy = rescale4(oy[i], b.ratio);
        }
    }
    if (tid == 0) a.kv.k_scales[blk] = b.s;
}

// Values: a thread's units are 4 positions x 4 dims, so that the transposed
// codes leave as whole dwords.
template <typename T, int PS, int D>
__device__ __forceinline__ void append_values(const append_args &a, const block_place &p, int first, int hi, int64_t tok,
                                              float *red) {
    constexpr int N = (PS * D / 16 + NT - 1) / NT;
    const int tid = threadIdx.x;
    const T *v = (const T *)a.v + (uint64_t)p.h * D;
    wm_f4 x[N][4];
    uint32_t o[N][4];
    float most = 0.0f;
#pragma unroll
    for (int i = 0; i < N; i++) {
        const int unit = tid + i * NT, quad = unit / (D / 4) * 4, dim = unit % (D / 4) * 4;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            x[i][j] = wm_f4{0, 0, 0, 0};
            if (quad + j >= first && quad + j < hi) x[i][j] = wm_ld4(v + (uint64_t)(tok + quad + j) * a.vs + dim);
        }
    }
    if (!p.stored()) return;
    const uint64_t blk = (uint64_t)p.page * a.kv.n_kv_heads + p.h;
    int8_t *codes = a.kv.v_codes + blk * (PS * D);
    const float old = first > 0 ? a.kv.v_scales[blk] : 0.0f;
#pragma unroll
    for (int i = 0; i < N; i++) {
        const int unit = tid + i * NT, quad = unit / (D / 4) * 4, dim = unit % (D / 4) * 4;
        const bool part = quad < hi && (quad < first || quad + 4 > hi);  // earlier positions, or none yet
#pragma unroll
        for (int j = 0; j < 4; j++) o[i][j] = part ? *(const uint32_t *)(codes + (dim + j) * PS + quad) : 0;
    }
#pragma unroll
    for (int i = 0; i < N; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) most = fmaxf(most, finite_abs4(x[i][j]));
    const block_scale b(most, old, red);
#pragma unroll
    for (int i = 0; i < N; i++) {
        const int unit = tid + i * NT, quad = unit / (D / 4) * 4, dim = unit % (D / 4) * 4;
        if (quad >= hi || (quad + 4 <= first && !b.grew)) continue;
#pragma unroll
        for (int j = 0; j < 4; j++) {  // dim + j of four positions
            const uint32_t kept = b.grew ? rescale4(o[i][j], b.ratio) : o[i][j];
            uint32_t w = 0;
#pragma unroll
            for (int t = 0; t < 4; t++) {
                const uint32_t mask = 255u << (8 * t);
                const int slot = quad + t;
                const uint32_t fresh = (uint32_t)(quotient_code(x[i][t][j], b.inv) & 255) << (8 * t);
                w |= slot < first ? kept & mask : slot < hi ? fresh : o[i][j] & mask;
            }
            *(uint32_t *)(codes + (dim + j) * PS + quad) = w;
        }
    }
    if (tid == 0) a.kv.v_scales[blk] = b.s;
}

template <typename T, int PS, int D>
__global__ __launch_bounds__(NT) void k_paged_append(append_args a) {
    static_assert(PS * D % (16 * NT) == 0 || PS * D < 16 * NT, "whole units per thread");
    __shared__ float red[NT / 64];
    // Values, keys, queries: the longest chains first where all workgroups
    // start at about the same time, else a block's kinds side by side, which
    // read neighbouring rows.  Both ways, first and side by side, in bf16
    // pages of 64: a grid of 1440 12.1 us and 13.8, 4320 13.7 and 17.4, 7440
    // 28.8 and 31.7; in f32 pages of 16: 1920 13.2 and 12.1, 6720 34.5 and
    // 29.9, 15120 95 and 83.
    uint32_t kind, id;
    if (a.by_kind) kind = blockIdx.x / a.blocks, id = blockIdx.x % a.blocks;
    else if (a.group) kind = blockIdx.x % (2 + PS / 16), id = blockIdx.x / (2 + PS / 16);
    else kind = blockIdx.x % 2, id = blockIdx.x / 2;
    const block_place p = place_block(a.kv, a.b, a.touch, a.seq0, id);
    if (!p.live) return;
    const int base = p.lp * PS;  // first position of the page
    const int first = max(max(p.q.start, 0) - base, 0), hi = min(p.q.len - base, PS);  // its new slots
    const int64_t tok = (int64_t)p.q.tok0 + base - p.q.start;  // packed token of slot 0
    if (kind >= 2) {
        const int s0 = 16 * (int)(kind - 2);
        append_queries<T, D>(a, p, base, max(first, s0), min(hi, s0 + 16), tok);
        return;
    }
    if ((kind == 0) == a.by_kind) append_values<T, PS, D>(a, p, first, hi, tok, red);
    else append_keys<T, PS, D>(a, p, base, first, hi, tok, red);
}

struct read_args {
    wm_paged_kv kv;
    wm_paged_batch b;
    void *k, *v;
    uint64_t ks, vs;
    uint32_t touch, seq0;
};

__device__ __forceinline__ wm_f4 values4(uint32_t w, float s) {
    return wm_f4{(float)byte_of(w, 0) * s, (float)byte_of(w, 1) * s, (float)byte_of(w, 2) * s, (float)byte_of(w, 3) * s};
}

// Read back: bound by its output bytes.  A unit is 4 positions x 4 dims: K's
// rows are a dword each, V's transposed through the unit's 16 bytes.
template <typename T, int PS, int D>
__global__ __launch_bounds__(NT) void k_paged_read(read_args a) {
    const block_place p = place_block(a.kv, a.b, a.touch, a.seq0, blockIdx.x);
    if (!p.live) return;
    const int base = p.lp * PS, first = max(max(p.q.start, 0) - base, 0), hi = min(p.q.len - base, PS);
    const int64_t tok = (int64_t)p.q.tok0 + base - p.q.start;
    const bool stored = p.stored();
    const uint64_t blk = (uint64_t)(stored ? p.page : 0) * a.kv.n_kv_heads + p.h;
    const int8_t *kc = a.kv.k_codes + blk * (PS * D), *vc = a.kv.v_codes + blk * (PS * D);
    const float nan = __uint_as_float(0x7FC00000u);
    const float sk = stored ? a.kv.k_scales[blk] : nan, sv = stored ? a.kv.v_scales[blk] : nan;
    constexpr int N = (PS * D / 16 + NT - 1) / NT;
    uint32_t wk[N][4], wv[N][4];
#pragma unroll
    for (int i = 0; i < N; i++) {  // all loads together
        const int unit = threadIdx.x + i * NT, quad = unit / (D / 4) * 4, dim = unit % (D / 4) * 4;
        const bool live = quad + 4 > first && quad < hi;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            wk[i][j] = live ? *(const uint32_t *)(kc + (quad + j) * D + dim) : 0;
            wv[i][j] = live ? *(const uint32_t *)(vc + (dim + j) * PS + quad) : 0;
        }
    }
#pragma unroll
    for (int i = 0; i < N; i++) {
        const int unit = threadIdx.x + i * NT, quad = unit / (D / 4) * 4, dim = unit % (D / 4) * 4;
#pragma unroll
        for (int t = 0; t < 4; t++) {
            const int slot = quad + t;
            if (slot < first || slot >= hi) continue;
            const uint64_t row = (uint64_t)(tok + slot);
            if (a.k) wm_st4((T *)a.k + row * a.ks + (uint64_t)p.h * D + dim, values4(wk[i][t], sk));
            const uint32_t col = pack_codes(byte_of(wv[i][0], t), byte_of(wv[i][1], t), byte_of(wv[i][2], t),
                                            byte_of(wv[i][3], t));
            if (a.v) wm_st4((T *)a.v + row * a.vs + (uint64_t)p.h * D + dim, values4(col, sv));
        }
    }
}

// Pages one sequence of the step can touch, at most: its tokens and the
// positions before its first in the same page.
uint32_t touched_pages(const wm_paged_kv *kv, const wm_paged_batch *b) {
    const uint64_t most = b->max_new < b->max_kv_len ? b->max_new : b->max_kv_len;
    return most ? (uint32_t)((most + 2 * kv->page_size - 2) / kv->page_size) : 0;
}
// Sequences of one launch, which counts threads in 32 bits; an append has up
// to six workgroups a block.  Many sequences next to a long one take several
// launches: the host knows no lengths, only their bound.
wm_status launch_seqs(wm_ctx *ctx, const char *who, const wm_paged_kv *kv, const wm_paged_batch *b, uint32_t *seqs) {
    const uint64_t one = (uint64_t)touched_pages(kv, b) * kv->n_kv_heads, most = 0x7FFFFFFFull / NT / 6;
    if (one > most || (one && b->n_seqs > most))
        return wm_set_error(ctx, WM_E_SHAPE, "%s: %u sequences of up to %llu blocks", who, b->n_seqs, (unsigned long long)one);
    *seqs = one ? (uint32_t)(most / one) : 0;
    return WM_OK;
}

template <typename T, int PS, int D> struct launch_append {
    static void go(append_args a, uint32_t blocks, hipStream_t s) {
        const uint32_t grid = blocks * (a.group ? 2 + PS / 16 : 2);
        a.blocks = blocks, a.by_kind = grid <= 4096;
        k_paged_append<T, PS, D><<<grid, NT, 0, s>>>(a);
    }
};
template <typename T, int PS, int D> struct launch_read {
    static void go(const read_args &a, uint32_t grid, hipStream_t s) { k_paged_read<T, PS, D><<<grid, NT, 0, s>>>(a); }
};
template <template <typename, int, int> class L, typename T, typename A>
void by_page(uint32_t ps, uint32_t d, const A &a, uint32_t grid, hipStream_t s) {
    if (d == 64) {
        if (ps == 16) L<T, 16, 64>::go(a, grid, s);
        else if (ps == 32) L<T, 32, 64>::go(a, grid, s);
        else L<T, 64, 64>::go(a, grid, s);
    } else {
        if (ps == 16) L<T, 16, 128>::go(a, grid, s);
        else if (ps == 32) L<T, 32, 128>::go(a, grid, s);
        else L<T, 64, 128>::go(a, grid, s);
    }
}
template <template <typename, int, int> class L, typename A>
void by_shape(int type, uint32_t ps, uint32_t d, const A &a, uint32_t grid, hipStream_t s) {
    if (type == WM_DTYPE_F32) by_page<L, float>(ps, d, a, grid, s);
    else if (type == WM_DTYPE_F16) by_page<L, _Float16>(ps, d, a, grid, s);
    else by_page<L, __bf16>(ps, d, a, grid, s);
}

// The fields that need no device; the message goes to `msg`.
wm_status check_fields(const wm_paged_kv *kv, const wm_paged_batch *b, char *msg, size_t n) {
    if (!kv || !b) return snprintf(msg, n, "null descriptor"), WM_E_ARG;
    if (kv->page_size != 16 && kv->page_size != 32 && kv->page_size != 64)
        return snprintf(msg, n, "page_size %u is not 16, 32 or 64", kv->page_size), WM_E_SHAPE;
    if (kv->head_dim != 64 && kv->head_dim != 128)
        return snprintf(msg, n, "head_dim %u is not 64 or 128", kv->head_dim), WM_E_SHAPE;
    if (kv->n_kv_heads == 0 || kv->n_kv_heads > 65536)
        return snprintf(msg, n, "%u kv heads", kv->n_kv_heads), WM_E_SHAPE;
    if (kv->n_pages == 0 || kv->n_pages > 0x7FFFFFFFu)
        return snprintf(msg, n, "%u pages", kv->n_pages), WM_E_SHAPE;
    if (b->n_tokens > 0x7FFFFFFFu || b->n_seqs > 0x7FFFFFFEu || b->max_kv_len > 1u << 30)
        return snprintf(msg, n, "n_tokens %u, n_seqs %u or max_kv_len %u is too large", b->n_tokens, b->n_seqs,
                        b->max_kv_len), WM_E_SHAPE;
    if (b->max_new > b->n_tokens)
        return snprintf(msg, n, "max_new %u is above n_tokens %u", b->max_new, b->n_tokens), WM_E_SHAPE;
    if ((uint64_t)b->table_stride * kv->page_size < b->max_kv_len)
        return snprintf(msg, n, "table_stride %u pages of %u hold fewer than max_kv_len %u positions", b->table_stride,
                        kv->page_size, b->max_kv_len), WM_E_SHAPE;
    return WM_OK;
}

}  // namespace

size_t wm_dtype_size(int type) {
    return type == WM_DTYPE_F32 ? 4 : type == WM_DTYPE_F16 || type == WM_DTYPE_BF16 ? 2 : 0;
}

wm_status wm_paged_check(wm_ctx *ctx, const char *who, const wm_paged_kv *kv, const wm_paged_batch *b) {
    char msg[160];
    if (wm_status st = check_fields(kv, b, msg, sizeof msg)) return wm_set_error(ctx, st, "%s: %s", who, msg);
    if (!kv->k_codes || !kv->v_codes || !kv->k_scales || !kv->v_scales)
        return wm_set_error(ctx, WM_E_ARG, "%s: null page pool", who);
    if (((uintptr_t)kv->k_codes | (uintptr_t)kv->v_codes) % 16 || ((uintptr_t)kv->k_scales | (uintptr_t)kv->v_scales) % 4)
        return wm_set_error(ctx, WM_E_ARG, "%s: misaligned page pool", who);
    if (b->n_seqs && (!b->cu_tokens || !b->kv_len || (!b->page_table && b->max_kv_len)))
        return wm_set_error(ctx, WM_E_ARG, "%s: null lengths or page table", who);
    if (((uintptr_t)b->cu_tokens | (uintptr_t)b->kv_len | (uintptr_t)b->page_table) % 4)
        return wm_set_error(ctx, WM_E_ARG, "%s: misaligned lengths or page table", who);
    return WM_OK;
}

wm_status wm_paged_check_array(wm_ctx *ctx, const char *who, const char *name, const void *p, uint64_t stride,
                               uint32_t heads, uint32_t head_dim, size_t elem) {
    if (!p) return wm_set_error(ctx, WM_E_ARG, "%s: null %s", who, name);
    if ((uintptr_t)p % 16 || stride * elem % 16)
        return wm_set_error(ctx, WM_E_ARG, "%s: %s and its rows must be 16-byte aligned", who, name);
    if (stride < (uint64_t)heads * head_dim || stride > 1ull << 40)
        return wm_set_error(ctx, WM_E_SHAPE, "%s: %s rows of %u x %u values are %llu apart", who, name, heads, head_dim,
                            (unsigned long long)stride);
    return WM_OK;
}

wm_status wm_paged_check_over(wm_ctx *ctx, const char *who, const void *q, uint64_t q_stride, const void *out,
                              uint64_t out_stride) {
    if (q == out && q_stride != out_stride)
        return wm_set_error(ctx, WM_E_ARG, "%s: the output over q has rows %llu apart, not %llu", who,
                            (unsigned long long)out_stride, (unsigned long long)q_stride);
    return WM_OK;
}

extern "C" {

wm_status wm_paged_batch_check(const wm_paged_kv *kv, const wm_paged_batch *b, const int32_t *cu_tokens,
                               const int32_t *kv_len, const int32_t *page_table, int appends) {
    char msg[160];
    if (wm_status st = check_fields(kv, b, msg, sizeof msg)) return st;
    if (b->n_seqs == 0) return WM_OK;
    if (!cu_tokens || !kv_len || (!page_table && b->max_kv_len)) return WM_E_ARG;
    if (cu_tokens[0] != 0) return WM_E_SHAPE;
    for (uint32_t s = 0; s < b->n_seqs; s++) {
        const int64_t n = (int64_t)cu_tokens[s + 1] - cu_tokens[s];
        if (n < 0 || n > b->max_new || (uint32_t)cu_tokens[s + 1] > b->n_tokens) return WM_E_SHAPE;
        if (kv_len[s] < 0 || (uint32_t)kv_len[s] > b->max_kv_len) return WM_E_SHAPE;
    }
    // per page: 0 free, 1 read, 2 appended to
    std::vector<uint8_t> use;
    try {
        if (appends) use.assign(kv->n_pages, 0);
    } catch (const std::bad_alloc &) {
        return WM_E_OOM;
    }
    for (uint32_t s = 0; s < b->n_seqs; s++) {
        const int64_t n = (int64_t)cu_tokens[s + 1] - cu_tokens[s], len = kv_len[s];
        if (!n) continue;  // reads and writes nothing
        const int64_t start = len > n ? len - n : 0;
        for (int64_t lp = 0; lp * kv->page_size < len; lp++) {
            const int32_t page = page_table[(uint64_t)s * b->table_stride + lp];
            if (page < 0 || (uint32_t)page >= kv->n_pages) return WM_E_BOUNDS;
            if (!appends) continue;
            const bool write = (lp + 1) * kv->page_size > start;
            if (write ? use[page] != 0 : use[page] == 2) return WM_E_BOUNDS;
            use[page] = write ? 2 : 1;
        }
    }
    return WM_OK;
}

wm_status wm_paged_kv_append_dev(wm_ctx *ctx, const wm_paged_kv *kv, const wm_paged_batch *batch,
                                 const wm_rope *rope, int type, const void *d_q, uint64_t q_stride,
                                 uint32_t n_heads, const void *d_k, uint64_t k_stride, const void *d_v,
                                 uint64_t v_stride, void *d_q_out, uint64_t q_out_stride) {
    static const char who[] = "paged_kv_append";
    if (!ctx) return WM_E_ARG;
    wm_status st;
    if ((st = wm_paged_check(ctx, who, kv, batch))) return st;
    const size_t elem = wm_dtype_size(type);
    if (!elem) return wm_set_error(ctx, WM_E_UNSUPPORTED_TYPE, "%s: type %d is not F32, F16 or BF16", who, type);
    if (n_heads % kv->n_kv_heads || n_heads > 1u << 20)
        return wm_set_error(ctx, WM_E_SHAPE, "%s: %u query heads over %u kv heads", who, n_heads, kv->n_kv_heads);
    append_args a;
    memset(&a, 0, sizeof a);
    if (rope) {
        a.rope = *rope;
        if (rope->n_rot % 8 || rope->n_rot > kv->head_dim)
            return wm_set_error(ctx, WM_E_SHAPE, "%s: n_rot %u is not a multiple of 8 up to head_dim %u", who,
                                rope->n_rot, kv->head_dim);
        if (rope->layout != WM_ROPE_HALF && rope->layout != WM_ROPE_INTERLEAVED)
            return wm_set_error(ctx, WM_E_ARG, "%s: rope layout %u", who, rope->layout);
        if (rope->n_rot) {
            if (!rope->cos || !rope->sin || ((uintptr_t)rope->cos | (uintptr_t)rope->sin) % 16)
                return wm_set_error(ctx, WM_E_ARG, "%s: null or misaligned rope tables", who);
            if (rope->n_pos < batch->max_kv_len)
                return wm_set_error(ctx, WM_E_SHAPE, "%s: rope tables of %u positions for max_kv_len %u", who,
                                    rope->n_pos, batch->max_kv_len);
        }
    }
    if (batch->n_tokens == 0 || batch->n_seqs == 0) return WM_OK;
    if ((st = wm_paged_check_array(ctx, who, "k", d_k, k_stride, kv->n_kv_heads, kv->head_dim, elem))) return st;
    if ((st = wm_paged_check_array(ctx, who, "v", d_v, v_stride, kv->n_kv_heads, kv->head_dim, elem))) return st;
    if (n_heads) {
        if ((st = wm_paged_check_array(ctx, who, "q", d_q, q_stride, n_heads, kv->head_dim, elem))) return st;
        if ((st = wm_paged_check_array(ctx, who, "q_out", d_q_out, q_out_stride, n_heads, kv->head_dim, elem))) return st;
        if ((st = wm_paged_check_over(ctx, who, d_q, q_stride, d_q_out, q_out_stride))) return st;
    }
    a.kv = *kv, a.b = *batch;
    a.q = d_q, a.k = d_k, a.v = d_v, a.q_out = d_q_out;
    a.qs = q_stride, a.ks = k_stride, a.vs = v_stride, a.qos = q_out_stride;
    a.group = n_heads / kv->n_kv_heads;
    a.touch = touched_pages(kv, batch);
    uint32_t seqs;
    if ((st = launch_seqs(ctx, who, kv, batch, &seqs))) return st;
    if (!seqs) return WM_OK;
    wm_device_guard dev(ctx->device);
    WM_HIP(ctx, dev.err);
    for (uint32_t left; a.seq0 < batch->n_seqs; a.seq0 += left) {
        left = std::min(seqs, batch->n_seqs - a.seq0);
        by_shape<launch_append>(type, kv->page_size, kv->head_dim, a, left * a.touch * kv->n_kv_heads, ctx->stream);
        WM_HIP(ctx, hipGetLastError());
    }
    return WM_OK;
}

wm_status wm_paged_kv_read_dev(wm_ctx *ctx, const wm_paged_kv *kv, const wm_paged_batch *batch, int type,
                               void *d_k_out, uint64_t k_stride, void *d_v_out, uint64_t v_stride) {
    static const char who[] = "paged_kv_read";
    if (!ctx) return WM_E_ARG;
    wm_status st;
    if ((st = wm_paged_check(ctx, who, kv, batch))) return st;
    const size_t elem = wm_dtype_size(type);
    if (!elem) return wm_set_error(ctx, WM_E_UNSUPPORTED_TYPE, "%s: type %d is not F32, F16 or BF16", who, type);
    if (batch->n_tokens == 0 || batch->n_seqs == 0 || (!d_k_out && !d_v_out)) return WM_OK;
    if (d_k_out && (st = wm_paged_check_array(ctx, who, "k_out", d_k_out, k_stride, kv->n_kv_heads, kv->head_dim, elem)))
        return st;
    if (d_v_out && (st = wm_paged_check_array(ctx, who, "v_out", d_v_out, v_stride, kv->n_kv_heads, kv->head_dim, elem)))
        return st;
    read_args a{*kv, *batch, d_k_out, d_v_out, k_stride, v_stride, touched_pages(kv, batch), 0};
    uint32_t seqs;
    if ((st = launch_seqs(ctx, who, kv, batch, &seqs))) return st;
    if (!seqs) return WM_OK;
    wm_device_guard dev(ctx->device);
    WM_HIP(ctx, dev.err);
    for (uint32_t left; a.seq0 < batch->n_seqs; a.seq0 += left) {
        left = std::min(seqs, batch->n_seqs - a.seq0);
        by_shape<launch_read>(type, kv->page_size, kv->head_dim, a, left * a.touch * kv->n_kv_heads, ctx->stream);
        WM_HIP(ctx, hipGetLastError());
    }
    return WM_OK;
}

}  // extern "C"
