// Causal attention over the paged 8-bit KV cache.
//
// A block's scale factors out of its scores and of its values, so both
// products run on its codes: int8 codes are exact in f16, and
// v_mfma_f32_*_f16 multiplies them by f16 queries (weights) with f32 sums.
// A query row is scaled by a power of two to [2^14, 2^15) and taken as one
// f16 term (f16 and bf16 inputs: exact but for elements 2^-28 below the row's
// largest) or two (f32: 22 bits).  Weights e^(s - max) * v_scale are scaled
// the same way; one f16 term for half outputs (2^-12, under the output's
// own rounding), two for f32.  Maxima, sums and accumulators are f32.
//
// A wave holds scores transposed, S^T = K Q^T: lane l has query row l % 16
// and 16 positions in a row, (l / 16) * 16 .. + 15 of a 64-position tile,
// which is how the second product, O^T = V^T P^T, takes its weights: no
// value crosses lanes but the running maximum.  The tile's K rows are dealt
// to the MFMA's rows so that this holds, and V's codes lie transposed in the
// page so that a lane's 16 positions of one dim are one 16-byte load.
#include <cstdio>
#include <cstring>

#include "wm_paged.h"

namespace {

constexpr int NT = 256;    // threads per workgroup, four waves
constexpr int TILE = 64;   // positions per tile of one wave
constexpr int W_EXP = 14;  // weights are formed times 2^W_EXP
constexpr int E_NONE = -200;  // the exponent of a zero scale

struct attn_args {
    wm_paged_kv kv;
    wm_paged_batch b;
    const void *q;
    void *out;
    float *lse;
    uint64_t qs, os;
    uint32_t n_heads, group;
    int type;
    float scale_log2;  // scale * log2 e
    // the split of the positions: n_splits workgroups of split_len each, and
    // where they leave their partial rows (n_splits 1: none)
    uint32_t split_len, n_splits, row_tiles;
    float *part_o, *part_lse;
};

// Sixteen codes to f16: 0x6400 | (code + 128) is 1024 + 128 + code.
__device__ __forceinline__ void codes_to_f16(wm_u4 w, wm_h8 &lo, wm_h8 &hi) {
    const wm_h2 bias = {(_Float16)-1152.0f, (_Float16)-1152.0f};
    union {
        wm_h2 h[8];
        wm_h8 v[2];
    } r;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t u = w[i] ^ 0x80808080u;
        r.h[2 * i] = __builtin_bit_cast(wm_h2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) + bias;
        r.h[2 * i + 1] = __builtin_bit_cast(wm_h2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) + bias;
    }
    lo = r.v[0];
    hi = r.v[1];
}

// Over the four 16-lane groups (lanes l, l ^ 16, l ^ 32, l ^ 48).
__device__ __forceinline__ float group_max(float v) {
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ int group_max(int v) {
    auto a = __builtin_amdgcn_permlane32_swap((unsigned)v, (unsigned)v, false, false);
    v = max((int)a[0], (int)a[1]);
    a = __builtin_amdgcn_permlane16_swap((unsigned)v, (unsigned)v, false, false);
    return max((int)a[0], (int)a[1]);
}
__device__ __forceinline__ float group_sum(float v) {
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

// A value as one f16 term, or as two whose sum holds its upper 22 bits: the
// first is cut off, not rounded, so that both come from the same f32 value
// (a rounded one, fused with the product that made the value, could round a
// tie the other way than its copy that is subtracted).
template <int TERMS>
__device__ __forceinline__ void to_terms(float v, _Float16 *hi, _Float16 *lo) {
    if (TERMS == 1) {
        *hi = (_Float16)v;
    } else {
        const float h = __uint_as_float(__float_as_uint(v) & 0xFFFFE000u);
        *hi = (_Float16)h;
        *lo = (_Float16)(v - h);
    }
}
// f32 inputs take two terms, the half types one.
template <int TERMS>
__device__ __forceinline__ wm_f4 load_q4(const attn_args &a, uint64_t at) {
    if (TERMS > 1) return wm_ld4((const float *)a.q + at);
    if (a.type == WM_DTYPE_F16) return wm_ld4((const _Float16 *)a.q + at);
    return wm_ld4((const __bf16 *)a.q + at);
}
__device__ __forceinline__ void store_out4(const attn_args &a, uint64_t at, wm_f4 v) {
    if (a.type == WM_DTYPE_F32) wm_st4((float *)a.out + at, v);
    else if (a.type == WM_DTYPE_F16) wm_st4((_Float16 *)a.out + at, v);
    else wm_st4((__bf16 *)a.out + at, v);
}

// A row tile: rows r0 .. of one sequence and kv head, row r = token r / group
// and query head h * group + r % group.
struct row_tile {
    wm_seq q;
    uint32_t s, h;
    int rows, r0;  // rows of the sequence and head; the tile's first
    int len;       // positions that the tile's last row attends to
};
__device__ __forceinline__ row_tile load_tile(const attn_args &a, uint32_t s, uint32_t h, uint32_t t, int per) {
    row_tile r;
    r.q = wm_load_seq(a.b, s);
    r.s = s, r.h = h;
    r.rows = r.q.n * (int)a.group;
    r.r0 = (int)t * per;
    const int last = (min(r.r0 + per, r.rows) - 1) / (int)a.group;
    r.len = min(max(r.q.start + last + 1, 0), r.q.len);
    return r;
}
__device__ __forceinline__ uint64_t row_token(const attn_args &a, const row_tile &t, int r) {
    return (uint64_t)(t.q.tok0 + r / (int)a.group);
}
__device__ __forceinline__ uint64_t row_head(const attn_args &a, const row_tile &t, int r) {
    return (uint64_t)t.h * a.group + r % (int)a.group;
}

// A bad sequence's rows.
__device__ __forceinline__ void poison_rows(const attn_args &a, const row_tile &t, int per, int d) {
    const float nan = __uint_as_float(0x7FC00000u);
    const int n = min(per, t.rows - t.r0);
    for (int i = threadIdx.x; i < n * (d / 4); i += NT) {
        const int r = t.r0 + i / (d / 4);
        const uint64_t tok = row_token(a, t, r), head = row_head(a, t, r);
        store_out4(a, tok * a.os + head * d + i % (d / 4) * 4, wm_f4{nan, nan, nan, nan});
        if (a.lse && i % (d / 4) == 0) a.lse[tok * a.n_heads + head] = nan;
    }
}

// One workgroup: NR row tiles of 16 rows, one split of the positions; its
// four waves take the split's tiles in turn, each with sums of its own, and
// meet in LDS at the end.  Decode reads every code once from HBM, which is
// its bound; a tile's 16 KB are in flight per wave while the tile before is
// worked on (K's registers are loaded again as soon as the scores are out,
// V's after the second product).
template <int D, int NR, int TERMS>
__global__ __launch_bounds__(NT) void k_paged_attn_rows(attn_args a) {
    constexpr int ROWS = 16 * NR, KS = D / 32, DT = D / 16, LDO = D + 4;
    __shared__ float sh_o[4][ROWS][LDO];
    __shared__ float sh_lse[4][ROWS];
    uint32_t id = blockIdx.x;
    const uint32_t split = id % a.n_splits;
    id /= a.n_splits;
    const uint32_t rt = id % a.row_tiles;
    id /= a.row_tiles;
    const row_tile t = load_tile(a, id / a.kv.n_kv_heads, id % a.kv.n_kv_heads, rt, ROWS);
    if (t.r0 >= t.rows) return;
    if (!t.q.ok) {
        if (split == 0) poison_rows(a, t, ROWS, D);
        return;
    }
    const int p0 = (int)(split * a.split_len);
    if (split && p0 >= t.len) return;
    const int p1 = (int)min((int64_t)p0 + a.split_len, (int64_t)t.len);
    const bool whole = t.len <= (int)a.split_len;

    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, n = lane & 15, g = lane >> 4;
    // queries
    wm_h8 q[NR][KS][TERMS];
    float kfac[NR];
    int count[NR];
#pragma unroll
    for (int r = 0; r < NR; r++) {
        const int row = t.r0 + 16 * r + n;
        const bool valid = row < t.rows;
        count[r] = valid ? t.q.start + row / (int)a.group + 1 : t.len;
        float x[KS][8], m = 0.0f;
        const uint64_t at = valid ? row_token(a, t, row) * a.qs + row_head(a, t, row) * D : 0;
#pragma unroll
        for (int j = 0; j < KS; j++)
#pragma unroll
            for (int i = 0; i < 8; i += 4) {
                const wm_f4 v = valid ? load_q4<TERMS>(a, at + j / 2 * 64 + g * 16 + j % 2 * 8 + i) : wm_f4{0, 0, 0, 0};
#pragma unroll
                for (int c = 0; c < 4; c++) x[j][i + c] = v[c], m = fmaxf(m, fabsf(v[c]));
            }
        const int e = __builtin_amdgcn_frexp_expf(group_max(m));
        kfac[r] = ldexpf(a.scale_log2, e - 15);
#pragma unroll
        for (int j = 0; j < KS; j++)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                _Float16 hi, lo;
                to_terms<TERMS>(ldexpf(x[j][i], 15 - e), &hi, &lo);
                q[r][j][0][i] = hi;
                if (TERMS > 1) q[r][j][TERMS - 1][i] = lo;
            }
    }
    const int all = t.q.start + t.r0 / (int)a.group + 1;  // positions that every row attends to

    wm_f4 o[NR][DT];
    float m[NR], l[NR];
#pragma unroll
    for (int r = 0; r < NR; r++) {
        m[r] = -INFINITY, l[r] = 0.0f;
#pragma unroll
        for (int i = 0; i < DT; i++) o[r][i] = wm_f4{0, 0, 0, 0};
    }
    int e_ref = -300;

    const uint32_t ps = a.kv.page_size, ps_log = 31 - __builtin_clz(ps);
    const int32_t *table = a.b.page_table + (uint64_t)t.s * a.b.table_stride;
    const int kgrp = n >> 2;  // the 16-position group this lane's K rows are of
    const uint64_t block = (uint64_t)ps * D;
    struct pages {
        int k, v;
    };
    // pages of the lane's K rows and of its V positions (those past the
    // tile's end: any page it has)
    auto load_pages = [&](int p) {
        const int last = t.len - 1;
        return pages{table[min(p + kgrp * 16, last) >> ps_log], table[min(p + g * 16, last) >> ps_log]};
    };
    wm_u4 kr[4][D / 64], vr[DT];
    auto load_k = [&](int p, int page) {
        const uint64_t pg = (uint32_t)page < a.kv.n_pages ? (uint32_t)page : 0;
        const int8_t *src = a.kv.k_codes + (pg * a.kv.n_kv_heads + t.h) * block +
                            (((p + kgrp * 16) & (int)(ps - 1)) + (n & 3)) * D + g * 16;
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int j = 0; j < D / 64; j++) kr[i][j] = *(const wm_u4 *)(src + 4 * i * D + 64 * j);
    };
    auto load_v = [&](int p, int page) {
        const uint64_t pg = (uint32_t)page < a.kv.n_pages ? (uint32_t)page : 0;
        const int8_t *src = a.kv.v_codes + (pg * a.kv.n_kv_heads + t.h) * block + (uint64_t)n * ps +
                            ((p + g * 16) & (int)(ps - 1));
#pragma unroll
        for (int i = 0; i < DT; i++) vr[i] = *(const wm_u4 *)(src + (uint64_t)(16 * i) * ps);
    };
    struct scales {
        float k, v;
    };
    auto load_scales = [&](int page) {
        if ((uint32_t)page >= a.kv.n_pages) return scales{__uint_as_float(0x7FC00000u), 0.0f};
        const uint64_t at = (uint64_t)page * a.kv.n_kv_heads + t.h;
        return scales{a.kv.k_scales[at], a.kv.v_scales[at]};
    };

    int p = p0 + wave * TILE;
    pages pg{0, 0}, pg_next{0, 0};
    scales sc{0, 0}, sc_next{0, 0};
    if (p < p1) {
        pg = load_pages(p);
        sc = load_scales(pg.v);
        load_k(p, pg.k);
        load_v(p, pg.v);
        if (p + 4 * TILE < p1) pg_next = load_pages(p + 4 * TILE);
    }
    for (; p < p1; p += 4 * TILE) {
        const bool more = p + 4 * TILE < p1;
        wm_f4 s[NR][4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
#pragma unroll
            for (int r = 0; r < NR; r++) s[r][i] = wm_f4{0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < D / 64; j++) {
                wm_h8 k0, k1;
                codes_to_f16(kr[i][j], k0, k1);
#pragma unroll
                for (int r = 0; r < NR; r++)
#pragma unroll
                    for (int w = 0; w < TERMS; w++) {
                        s[r][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, q[r][2 * j][w], s[r][i], 0, 0, 0);
                        s[r][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, q[r][2 * j + 1][w], s[r][i], 0, 0, 0);
                    }
            }
        }
        pages pg_after{0, 0};
        if (more) {
            load_k(p + 4 * TILE, pg_next.k);
            sc_next = load_scales(pg_next.v);
            if (p + 8 * TILE < p1) pg_after = load_pages(p + 8 * TILE);
        }
        // The values' scale 2^eb * [1/2, 1) goes into the weight: the score
        // gets eb - e_ref (e_ref: the largest exponent so far, of any lane),
        // so that the running maximum is that of the products and the f16
        // weights hold their 11 bits relative to it, however the scales
        // differ; the sum of the weights is taken without it.
        const int eb0 = sc.v != 0.0f ? __builtin_amdgcn_frexp_expf(sc.v) : E_NONE;
        const int e_new = max(e_ref, group_max(eb0)), eb = max(eb0, e_new - 60);
        const float shift = (float)(eb - e_new), unshift = ldexpf(1.0f, e_new - eb), fb = ldexpf(sc.v, W_EXP - eb);
        const float dm = (float)(e_new - e_ref);
        e_ref = e_new;
        const bool masked = p + TILE > all;
        wm_h8 w[NR][2][TERMS];
#pragma unroll
        for (int r = 0; r < NR; r++) {
            const float f = kfac[r] * sc.k;
            float x[16], top = -INFINITY;
#pragma unroll
            for (int i = 0; i < 16; i++) x[i] = __builtin_fmaf(s[r][i / 4][i % 4], f, shift);
            if (masked) {
                const int left = count[r] - (p + g * 16);
#pragma unroll
                for (int i = 0; i < 16; i++) x[i] = i < left ? x[i] : -INFINITY;
            }
#pragma unroll
            for (int i = 0; i < 16; i++) top = fmaxf(top, x[i]);
            const float m_old = m[r] - dm, m_new = fmaxf(m_old, group_max(top));
            const float base = m_new == -INFINITY ? 0.0f : m_new;
            const float alpha = __builtin_amdgcn_exp2f(m_old - base);
            l[r] *= __builtin_amdgcn_exp2f(m[r] - base);
            m[r] = m_new;
            if (__ballot(alpha != 1.0f)) {
#pragma unroll
                for (int i = 0; i < DT; i++) o[r][i] *= alpha;
            }
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const float e = __builtin_amdgcn_exp2f(x[i] - base);
                sum += e;
                x[i] = e * fb;
            }
            l[r] = __builtin_fmaf(sum, unshift, l[r]);
#pragma unroll
            for (int i = 0; i < 16; i++) {
                _Float16 hi, lo;
                to_terms<TERMS>(x[i], &hi, &lo);
                w[r][i / 8][0][i % 8] = hi;
                if (TERMS > 1) w[r][i / 8][TERMS - 1][i % 8] = lo;
            }
        }
#pragma unroll
        for (int i = 0; i < DT; i++) {
            wm_h8 v0, v1;
            codes_to_f16(vr[i], v0, v1);
#pragma unroll
            for (int r = 0; r < NR; r++)
#pragma unroll
                for (int x = 0; x < TERMS; x++) {
                    o[r][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, w[r][0][x], o[r][i], 0, 0, 0);
                    o[r][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, w[r][1][x], o[r][i], 0, 0, 0);
                }
        }
        if (more) load_v(p + 4 * TILE, pg_next.v);
        pg_next = pg_after;
        sc = sc_next;
    }

    // rows of this wave, normalised, with the log2 of their sums
#pragma unroll
    for (int r = 0; r < NR; r++) {
        const float sum = group_sum(l[r]);
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
        for (int i = 0; i < DT; i++) {
            wm_f4 v = o[r][i] * inv;
#pragma unroll
            for (int c = 0; c < 4; c++) v[c] = ldexpf(v[c], e_ref - W_EXP);
            *(wm_f4 *)&sh_o[wave][16 * r + n][16 * i + 4 * g] = v;
        }
        // a sum of 0 is that of a row without positions, or without a tile
        if (g == 0) sh_lse[wave][16 * r + n] = sum == 0.0f ? -INFINITY : m[r] + __builtin_amdgcn_logf(sum);
    }
    __syncthreads();
    const int rows = min(ROWS, t.rows - t.r0);
    for (int i = tid; i < rows * (D / 4); i += NT) {
        const int row = i / (D / 4), c = i % (D / 4) * 4;
        float ls[4], top = -INFINITY;
#pragma unroll
        for (int w = 0; w < 4; w++) ls[w] = sh_lse[w][row], top = fmaxf(top, ls[w]);
        const float base = top == -INFINITY ? 0.0f : top;
        wm_f4 v = {0, 0, 0, 0};
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; w++) {
            const float e = __builtin_amdgcn_exp2f(ls[w] - base);
            sum += e;
            v += *(const wm_f4 *)&sh_o[w][row][c] * e;
        }
        if (sum != 0.0f) v *= 1.0f / sum;
        const float lse2 = sum == 0.0f ? -INFINITY : base + __builtin_amdgcn_logf(sum);
        const int r = t.r0 + row;
        const uint64_t tok = row_token(a, t, r), head = row_head(a, t, r), at = tok * a.n_heads + head;
        if (whole) {
            store_out4(a, tok * a.os + head * D + c, v);
            if (a.lse && c == 0) a.lse[at] = lse2 * 0.6931471805599453f;
        } else {
            *(wm_f4 *)(a.part_o + (at * a.n_splits + split) * D + c) = v;
            if (c == 0) a.part_lse[at * a.n_splits + split] = lse2;
        }
    }
}

// The splits' rows joined: weights 2^(lse - max), one thread per four dims.
template <int D>
__global__ __launch_bounds__(NT) void k_paged_attn_join(attn_args a, int per) {
    uint32_t id = blockIdx.x;
    const uint32_t rt = id % a.row_tiles;
    id /= a.row_tiles;
    const row_tile t = load_tile(a, id / a.kv.n_kv_heads, id % a.kv.n_kv_heads, rt, per);
    if (t.r0 >= t.rows || !t.q.ok || t.len <= (int)a.split_len) return;
    const int n = (t.len + (int)a.split_len - 1) / (int)a.split_len, rows = min(per, t.rows - t.r0);
    for (int i = threadIdx.x; i < rows * (D / 4); i += NT) {
        const int r = t.r0 + i / (D / 4), c = i % (D / 4) * 4;
        const uint64_t tok = row_token(a, t, r), head = row_head(a, t, r), at = tok * a.n_heads + head;
        const float *ls = a.part_lse + at * a.n_splits, *os = a.part_o + at * a.n_splits * D + c;
        float top = -INFINITY;
        for (int s = 0; s < n; s++) top = fmaxf(top, ls[s]);
        const float base = top == -INFINITY ? 0.0f : top;
        wm_f4 v = {0, 0, 0, 0};
        float sum = 0.0f;
        for (int s = 0; s < n; s++) {
            const float e = __builtin_amdgcn_exp2f(ls[s] - base);
            sum += e;
            v += *(const wm_f4 *)(os + (uint64_t)s * D) * e;
        }
        if (sum != 0.0f) v *= 1.0f / sum;
        store_out4(a, tok * a.os + head * D + c, v);
        if (a.lse && c == 0) a.lse[at] = sum == 0.0f ? -INFINITY : (base + __builtin_amdgcn_logf(sum)) * 0.6931471805599453f;
    }
}

// How a step is divided: from the host's bounds alone.
struct attn_plan {
    int nr;  // row tiles of 16 per workgroup
    uint32_t split_len, n_splits, row_tiles;
    uint64_t grid;
};
attn_plan make_plan(const wm_paged_kv *kv, const wm_paged_batch *b, uint32_t n_heads) {
    attn_plan p;
    const uint64_t rows = (uint64_t)b->max_new * (n_heads / kv->n_kv_heads);
    p.nr = rows > 16 ? 2 : 1;
    p.row_tiles = (uint32_t)((rows + 16 * p.nr - 1) / (16 * p.nr));
    const uint64_t units = (uint64_t)b->n_seqs * kv->n_kv_heads * p.row_tiles;
    // splits of whole rounds of the four waves' tiles
    const uint32_t round = 4 * TILE, rounds = (b->max_kv_len + round - 1) / round;
    const uint64_t want = units ? 1024 / units + 1 : 1;
    uint32_t per = rounds / (uint32_t)want;
    if (per < 1) per = 1;
    p.split_len = per * round;
    p.n_splits = rounds ? (rounds + per - 1) / per : 1;
    p.grid = units * p.n_splits;
    return p;
}

}  // namespace

extern "C" {

size_t wm_paged_attention_workspace(const wm_paged_kv *kv, const wm_paged_batch *batch, uint32_t n_heads) {
    if (!kv || !batch || !kv->n_kv_heads || n_heads % kv->n_kv_heads) return 0;
    const attn_plan p = make_plan(kv, batch, n_heads);
    if (p.n_splits <= 1) return 0;
    return (size_t)batch->n_tokens * n_heads * p.n_splits * (kv->head_dim + 1) * sizeof(float);
}

wm_status wm_paged_attention_dev(wm_ctx *ctx, const wm_paged_kv *kv, const wm_paged_batch *batch, int type,
                                 const void *d_q, uint64_t q_stride, uint32_t n_heads, float scale, void *d_out,
                                 uint64_t out_stride, float *d_lse, void *d_work, size_t work_bytes) {
    static const char who[] = "paged_attention";
    if (!ctx) return WM_E_ARG;
    wm_status st;
    if ((st = wm_paged_check(ctx, who, kv, batch))) return st;
    const size_t elem = wm_dtype_size(type);
    if (!elem) return wm_set_error(ctx, WM_E_UNSUPPORTED_TYPE, "%s: type %d is not F32, F16 or BF16", who, type);
    if (n_heads == 0 || n_heads % kv->n_kv_heads || n_heads > 1u << 20)
        return wm_set_error(ctx, WM_E_SHAPE, "%s: %u query heads over %u kv heads", who, n_heads, kv->n_kv_heads);
    if (!(scale - scale == 0.0f)) return wm_set_error(ctx, WM_E_NONFINITE, "%s: scale %g", who, (double)scale);
    if (batch->n_tokens == 0 || batch->n_seqs == 0 || batch->max_new == 0) return WM_OK;
    if ((st = wm_paged_check_array(ctx, who, "q", d_q, q_stride, n_heads, kv->head_dim, elem))) return st;
    if ((st = wm_paged_check_array(ctx, who, "out", d_out, out_stride, n_heads, kv->head_dim, elem))) return st;
    if ((uintptr_t)d_lse % 4) return wm_set_error(ctx, WM_E_ARG, "%s: misaligned lse", who);
    if ((uint64_t)batch->max_new * (n_heads / kv->n_kv_heads) > 0x7FFFFFFFull - 64)
        return wm_set_error(ctx, WM_E_SHAPE, "%s: %u tokens of %u heads in one sequence", who, batch->max_new, n_heads);
    const attn_plan p = make_plan(kv, batch, n_heads);
    if (p.grid > 0x7FFFFFFFull / NT)
        return wm_set_error(ctx, WM_E_SHAPE, "%s: %llu workgroups in one step", who, (unsigned long long)p.grid);
    const size_t need = wm_paged_attention_workspace(kv, batch, n_heads);
    if (need && (!d_work || work_bytes < need || (uintptr_t)d_work % 16))
        return wm_set_error(ctx, WM_E_ARG, "%s: workspace of %zu bytes, %zu needed, 16-byte aligned", who,
                            d_work ? work_bytes : (size_t)0, need);
    attn_args a;
    memset(&a, 0, sizeof a);
    a.kv = *kv, a.b = *batch;
    a.q = d_q, a.out = d_out, a.lse = d_lse;
    a.qs = q_stride, a.os = out_stride;
    a.n_heads = n_heads, a.group = n_heads / kv->n_kv_heads;
    a.type = type;
    a.scale_log2 = scale * 1.4426950408889634f;
    a.split_len = p.split_len, a.n_splits = p.n_splits, a.row_tiles = p.row_tiles;
    a.part_o = (float *)d_work;
    a.part_lse = a.part_o ? a.part_o + (size_t)batch->n_tokens * n_heads * p.n_splits * kv->head_dim : nullptr;
    wm_device_guard dev(ctx->device);
    WM_HIP(ctx, dev.err);
    const uint32_t grid = (uint32_t)p.grid;
    hipStream_t s = ctx->stream;
    const bool two = type == WM_DTYPE_F32;
#define WM_ROWS(D_, NR_)                                                              \
    do {                                                                              \
        if (two) k_paged_attn_rows<D_, NR_, 2><<<grid, NT, 0, s>>>(a);                 \
        else k_paged_attn_rows<D_, NR_, 1><<<grid, NT, 0, s>>>(a);                     \
    } while (0)
    if (kv->head_dim == 64) {
        if (p.nr == 1) WM_ROWS(64, 1);
        else WM_ROWS(64, 2);
    } else {
        if (p.nr == 1) WM_ROWS(128, 1);
        else WM_ROWS(128, 2);
    }
#undef WM_ROWS
    WM_HIP(ctx, hipGetLastError());
    if (p.n_splits > 1) {
        const uint32_t g = grid / p.n_splits;
        if (kv->head_dim == 64) k_paged_attn_join<64><<<g, NT, 0, s>>>(a, 16 * p.nr);
        else k_paged_attn_join<128><<<g, NT, 0, s>>>(a, 16 * p.nr);
        WM_HIP(ctx, hipGetLastError());
    }
    return WM_OK;
}

}  // extern "C"
