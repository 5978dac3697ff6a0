// Causal attention over the paged 8-bit KV cache.
//
// A block's scale factors out of its scores and of its values, so both
// products run on its codes: int8 codes are exact in f16, and
// v_mfma_f32_*_f16 multiplies them by f16 queries (weights) with f32 sums.
// A query row is scaled by a power of two to [2^14, 2^15) and taken as one
// f16 term (f16 and bf16 inputs: exact but for elements 2^-28 below the row's
// largest) or two (f32: 22 bits).  A weight 2^(s - max) * v_scale comes out of
// one exponential, the scale's logarithm in its argument: the product of
// the scores becomes the argument by one fma.  It is one f16 term for half
// outputs, two for f32, which takes the second product twice.  One term is
// rounded by up to 2^-11: an eighth of a bf16 output's own rounding (64 long
// sequences are 0.0017 off 64 bits, as their plain form in f32 is), as much as
// an f16 output's (8 prompts 0.00026, their plain form 0.00021).  Maxima, sums
// and accumulators are f32.
//
// A wave holds scores transposed, S^T = K Q^T: lane l has query row l % 16
// and 16 positions in a row, (l / 16) * 16 .. + 15 of a 64-position tile,
// which is how the second product, O^T = V^T P^T, takes its weights: no
// value crosses lanes but the running maximum.  The tile's K rows are dealt
// to the MFMA's rows so that this holds, and V's codes lie transposed in the
// page so that a lane's 16 positions of one dim are one 16-byte load.  (That
// is the kernel for few rows; the one for many does the same with 32 rows and
// the 32x32x16 product.)
//
// Measured with 20 query heads over 5 of 128 dims.  Few rows: 64 sequences of
// 2000 to 16000 positions, bf16, 138 us, 726 MB of codes at 5.2 TB/s (the
// bound; a large copy moves 4.7).  16 of 128 to 4064, f32, 18.8 us, and one of
// 1024, 10.0 us: the length of two launches' chains (lengths, page id, codes,
// scores, exponentials, the join).  Many rows: one prompt of 8192, bf16, 414
// to 426 us, 815 TFLOP/s of products: a SIMD runs vector instructions
// (exponentials, conversions, masks) for 53 % of that time and its matrix core
// for 35 %, which two waves overlap only in part.  16 sequences of 1 to 32
// tokens over up to 4064 positions, f32, 46 us.
#include <algorithm>
#include <cstdio>
#include <cstring>

#include "wm_paged.h"

namespace {

constexpr int NT = 256;    // threads per workgroup, four waves
constexpr int TILE = 64;   // positions per tile of one wave
constexpr float W_EXP = 7.0f;   // the largest weight is 2^W_EXP when the sums are scaled,
constexpr float W_MOST = 15.0f; // and may grow to this before they are scaled anew (f16 ends at 2^16)
constexpr int E_NONE = -1000;   // the exponent of a zero scale
// Rows (tokens x group) of a sequence and kv head up to which a wave takes
// them all, one tile of the matrix instruction, and rows of a workgroup beyond.
// 16 sequences over 128 to 4064 positions, f32: 16 rows each 23.1 us, 20 rows
// 35.2, 64 rows 43.1, 128 rows 47.6.
constexpr int FEW = 16;
constexpr int MANY = 128;

struct attn_args {
    wm_paged_kv kv;
    wm_paged_batch b;
    const void *q;
    void *out;
    float *lse;
    uint64_t qs, os;
    uint32_t n_heads, group;
    uint32_t few_recip;  // row * few_recip >> 16 is row / group for the first FEW rows
    int type;
    float scale_log2;  // scale * log2 e
    // Sequences of few rows: few_blocks workgroups share all their positions
    // evenly (few_share).  Those of many: up to many_n workgroups of many_len
    // positions each per row tile, many_blocks in all; many_levels row tiles of MANY and
    // contexts of as many tokens at most (many_order).
    uint32_t few_blocks, many_blocks, many_levels, many_len, many_n;
    // partial rows: FEW of each few_share::slot, then [token][head][many_n] of
    // the packed tokens or, where they are fewer, of max_new to a sequence
    float *part_o, *part_lse;
    bool parts_by_seq;
    // of each (sequence of few rows, kv head): the first workgroup that has a part of it, and how many have
    uint32_t *few_parts;
};
constexpr int ROUND = 4 * TILE;  // positions that a workgroup's four waves take at once
// Two workgroups of the kernel for few rows fit a compute unit.  Up to twice
// as many rounds are one workgroup's each; more are shared by those that fit:
// 318 rounds twice against 636 took 20.7 us against 19.5, 11400 rounds over
// 1024 workgroups 144 us against 139 over 512.
constexpr uint32_t FEW_RESIDENT = 512;
__host__ __device__ inline uint64_t few_slots(uint32_t blocks, uint32_t units) { return (uint64_t)blocks + units; }
__device__ __forceinline__ uint64_t many_part(const attn_args &a, uint32_t s, const wm_seq &q, uint64_t token, uint64_t head) {
    if (a.parts_by_seq) token = (uint64_t)s * a.b.max_new + (token - q.tok0);
    return (a.few_blocks ? few_slots(a.few_blocks, a.b.n_seqs * a.kv.n_kv_heads) * FEW : 0) +
           (token * a.n_heads + head) * a.many_n;
}

// The rounds of all sequences of few rows, (sequence, kv head, round) in
// order, dealt to the workgroups in runs of `per`: as even as lengths that
// only the device knows allow, and a workgroup has more than one (sequence,
// kv head) only where its run goes past an end.  Every wave scans the
// lengths by itself, 64 sequences at a time.
struct few_share {
    uint32_t per, total = 0;  // the host keeps the total below 2^31
    // the first 64 sequences, one to a lane, as the scan found them
    wm_seq q;
    uint32_t mine, upto;
    // the rounds of a sequence for one kv head (one to write empty or bad rows)
    static __device__ __forceinline__ uint32_t rounds(const attn_args &a, const wm_seq &q) {
        if (!q.ok) return 1;
        if (q.n == 0 || (int64_t)q.n * a.group > FEW) return 0;
        return max(1, (q.len + ROUND - 1) / ROUND);
    }
    static __device__ __forceinline__ void scan(const attn_args &a, uint32_t s0, wm_seq &q, uint32_t &mine, uint32_t &upto) {
        const uint32_t s = s0 + (threadIdx.x & 63);
        q = wm_load_seq(a.b, min(s, a.b.n_seqs - 1));
        mine = s < a.b.n_seqs ? rounds(a, q) : 0;
        upto = wm_wave_scan_i32(mine);
    }
    __device__ __forceinline__ few_share(const attn_args &a) {
        scan(a, 0, q, mine, upto);
        total = __builtin_amdgcn_readlane(upto, 63);
        for (uint32_t s = 64; s < a.b.n_seqs; s += 64) {
            wm_seq x;
            uint32_t m, u;
            scan(a, s, x, m, u);
            total += __builtin_amdgcn_readlane(u, 63);
        }
        total *= a.kv.n_kv_heads;
        per = total <= a.few_blocks ? 1 : (total + FEW_RESIDENT - 1) / FEW_RESIDENT;
    }
    // The sequence that round x is of, its rounds and the first of them; no
    // rounds where none has it, as lengths that change under the kernel leave
    // it: the search ends whatever it reads.
    struct place {
        wm_seq q;
        uint32_t s, rounds = 0, first;
    };
    __device__ __forceinline__ place find(const attn_args &a, uint32_t x) const {
        uint32_t base = 0, m = mine, u = upto;
        wm_seq at = q;
        for (uint32_t s = 0; s < a.b.n_seqs; s += 64) {
            if (s) scan(a, s, at, m, u);
            const uint64_t hit = __ballot(base + u * a.kv.n_kv_heads > x);
            if (hit) {
                const int lane = __builtin_ctzll(hit);
                const uint32_t n = __builtin_amdgcn_readlane(m, lane);
                place p;
                p.s = s + lane, p.rounds = n, p.first = base + (__builtin_amdgcn_readlane(u, lane) - n) * a.kv.n_kv_heads;
                p.q.tok0 = __builtin_amdgcn_readlane(at.tok0, lane), p.q.n = __builtin_amdgcn_readlane(at.n, lane);
                p.q.start = __builtin_amdgcn_readlane(at.start, lane), p.q.len = __builtin_amdgcn_readlane(at.len, lane);
                p.q.ok = __builtin_amdgcn_readlane(at.ok, lane);
                return p;
            }
            base += __builtin_amdgcn_readlane(u, 63) * a.kv.n_kv_heads;
        }
        return place();
    }
    // Where workgroup w leaves its part of a unit (sequence, kv head): along
    // the runs either grows by one at a time.
    static __device__ __forceinline__ uint64_t slot(uint64_t w, uint64_t unit) { return w + unit; }
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
// Over the two halves of a wave.
__device__ __forceinline__ float half_max(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float half_sum(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}
__device__ __forceinline__ float read_lane(float v, int lane) {
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane));
}
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// A value scale's exponent, and the log2 of what the exponent leaves.
__device__ __forceinline__ int scale_exponent(float v) { return v != 0.0f ? __builtin_amdgcn_frexp_expf(v) : E_NONE; }
__device__ __forceinline__ float scale_rest(float v, int e) {
    return v != 0.0f ? __builtin_amdgcn_logf(ldexpf(v, -e)) : -60.0f;
}

// A row's reference exponent, the largest of the value scales of the blocks
// that it attends to in the tiles so far (a tile's other blocks do not count:
// what a row gives must not depend on them).  What is held is O 2^-e, and the
// running maximum m is that of score + log2(scale) - e, so that the f16
// weights hold their 11 bits relative to the largest product of weight and
// scale, however the scales differ.  l = sum 2^(score - m) has no e in it.
// Until a tile is masked all rows of a wave have the same e.
struct scale_ref {
    int e = E_NONE;
    int rise = 0;  // what e has risen by for this tile
    __device__ __forceinline__ void raise(int to) {
        rise = e == E_NONE ? 0 : max(to - e, 0);  // before the first scale, O is 0
        e = max(e, to);
    }
    // log2 of a block's scale (scale_exponent, scale_rest) relative to e.  One
    // 2^60 below it, or 0, counts as 2^-60: such a weight is 0 in f16.
    __device__ __forceinline__ float part(int eb, float rest) const {
        return eb < e - 60 ? -60.0f : (float)(eb - e) + rest;
    }
};
// Under a new tile's largest relative score `top` (of the row): m, l and what
// O is to be scaled by; `from` is what the scores are relative to.  True where
// any row of the wave needs it.
struct row_max {
    float m = -INFINITY, l = 0.0f, from = 0.0f;
    // A risen reference lowers m, and l grows; where l would leave its range
    // (scales more than 2^60 apart), O falls instead, by 2^-fall.  True where
    // any row of the wave needs that.  A row's lanes hold parts of its l, but
    // one m: `row_max` takes the largest of the parts, so that all lanes of a
    // row do the same.
    template <typename F>
    __device__ __forceinline__ bool begin(const scale_ref &r, F row_max, int &fall) {
        from = m == -INFINITY ? 0.0f : m;
        if (!__ballot(r.rise != 0)) return false;
        const int down = row_max(l) > 0x1p60f ? 0 : min(r.rise, 60);
        m -= (float)down, l = ldexpf(l, down), fall = r.rise - down;
        from = m == -INFINITY ? 0.0f : m;
        return __ballot(fall > 0);
    }
    // Every lane's scores have then to be lowered by `by`, O scaled by `alpha`
    // (by 0 and 1 in rows that do not need it).
    __device__ __forceinline__ bool grows(float top, float &by, float &alpha) {
        const bool over = top > (m == -INFINITY ? -INFINITY : W_MOST);
        if (!__ballot(over)) return false;
        const float to = over ? fmaxf(m, from + top - W_EXP) : m, base = to == -INFINITY ? 0.0f : to;
        alpha = __builtin_amdgcn_exp2f(m - base);
        l *= alpha;
        m = to;
        by = base - from;
        return true;
    }
};

// O 2^e / sum: the exponents together, so that no factor leaves its range.
struct row_scale {
    float inv;
    int e;
    __device__ __forceinline__ row_scale(float sum, int ref_e) {
        const int k = __builtin_amdgcn_frexp_expf(sum);
        inv = sum == 0.0f ? 0.0f : 1.0f / ldexpf(sum, -k), e = ref_e - k;
    }
    __device__ __forceinline__ float operator()(float o) const { return ldexpf(o * inv, e); }
};
// Parts of a row are joined under weights 2^x, applied as two factors: a
// part far below the others in its sum may be as far above them in its values.
__device__ __forceinline__ float half_weight(float x) { return __builtin_amdgcn_exp2f(0.5f * x); }
// The exponent that a query row is scaled by (rows below 2^-100 are taken as
// if they reached it: the factor stays finite).
__device__ __forceinline__ int query_exponent(float most) { return max(__builtin_amdgcn_frexp_expf(most), -100); }

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
__device__ __forceinline__ row_tile make_tile(const attn_args &a, const wm_seq &q, uint32_t s, uint32_t h, uint32_t t, int per) {
    row_tile r;
    r.q = q;
    r.s = s, r.h = h;
    r.rows = r.q.ok ? r.q.n * (int)a.group : 0;
    r.r0 = (int)t * per;
    const int last = (min(r.r0 + per, r.rows) - 1) / (int)a.group;
    r.len = min(max(r.q.start + last + 1, 0), r.q.len);
    return r;
}
__device__ __forceinline__ row_tile load_tile(const attn_args &a, uint32_t s, uint32_t h, uint32_t t, int per) {
    wm_seq q = wm_load_seq(a.b, s);
    // of the whole workgroup: in scalar registers
    q.tok0 = uniform(q.tok0), q.n = uniform(q.n), q.start = uniform(q.start), q.len = uniform(q.len);
    q.ok = uniform(q.ok);
    return make_tile(a, q, s, h, t, per);
}
__device__ __forceinline__ uint64_t row_token(const attn_args &a, const row_tile &t, int r) {
    return (uint64_t)(t.q.tok0 + r / (int)a.group);
}
__device__ __forceinline__ uint64_t row_head(const attn_args &a, const row_tile &t, int r) {
    return (uint64_t)t.h * a.group + r % (int)a.group;
}

// Every row of a sequence whose lengths break their bounds, by one workgroup.
__device__ __forceinline__ void poison_sequence(const attn_args &a, const row_tile &t, int d) {
    const float nan = __uint_as_float(0x7FC00000u);
    const int64_t per = (int64_t)a.group * (d / 4), n = t.q.n * per;
    for (int64_t i = threadIdx.x; i < n; i += NT) {
        const uint64_t tok = t.q.tok0 + i / per, head = (uint64_t)t.h * a.group + i % per / (d / 4);
        store_out4(a, tok * a.os + head * d + i % (d / 4) * 4, wm_f4{nan, nan, nan, nan});
        if (a.lse && i % (d / 4) == 0) a.lse[tok * a.n_heads + head] = nan;
    }
}

// Few rows.  One workgroup: the 16 rows of one MFMA tile, some rounds of one
// sequence's positions; its four waves take a tile of each round, each with
// sums of its own, and meet in LDS at the end.  Decode reads every code once
// from HBM, which is its bound; a tile's 16 KB are in flight per wave while
// the tile before is worked on (K's registers are loaded again as soon as the
// scores are out, V's after the second product).  Registers for that leave two
// waves to a SIMD; capped for three or four they spill (204 and 450 us for
// 138).
template <int D>
struct alignas(16) few_shared {
    float o[4][FEW][D + 4];
    float lse[4][FEW];
};
template <int D, int TERMS>
__device__ __forceinline__ void attend_few_part(const attn_args &a, const wm_seq &seq, uint32_t s, uint32_t h, uint32_t k0,
                                                uint32_t k1, bool whole, uint64_t slot, few_shared<D> &sh) {
    constexpr int KS = D / 32, DT = D / 16;
    const row_tile t = make_tile(a, seq, s, h, 0, FEW);
    if (!t.q.ok) {
        poison_sequence(a, t, D);
        return;
    }
    const int p0 = (int)k0 * ROUND, p1 = min((int)k1 * ROUND, t.len);

    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, n = lane & 15, g = lane >> 4;
    wm_f4 o[DT];
    row_max sums;
    scale_ref ref;
#pragma unroll
    for (int i = 0; i < DT; i++) o[i] = wm_f4{0, 0, 0, 0};

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
        if (p + 4 * TILE < p1) pg_next = load_pages(p + 4 * TILE);
    }
    // The queries' loads go out with the page ids', in front of the codes'.
    // Rows past the last repeat it, and are not written.
    const int at_row = min(n, t.rows - 1), j_row = (int)(at_row * a.few_recip >> 16), count = t.q.start + j_row + 1;
    float x_q[KS][8], q_max = 0.0f;
    {
        const uint64_t at = (uint64_t)(t.q.tok0 + j_row) * a.qs + ((uint64_t)t.h * a.group + at_row - j_row * a.group) * D;
#pragma unroll
        for (int j = 0; j < KS; j++)
#pragma unroll
            for (int i = 0; i < 8; i += 4) {
                const wm_f4 v = load_q4<TERMS>(a, at + j / 2 * 64 + g * 16 + j % 2 * 8 + i);
#pragma unroll
                for (int c = 0; c < 4; c++) x_q[j][i + c] = v[c];
            }
    }
    if (p < p1) {
        load_k(p, pg.k);
        load_v(p, pg.v);
        sc = load_scales(pg.v);
    }
#pragma unroll
    for (int j = 0; j < KS; j++)
#pragma unroll
        for (int i = 0; i < 8; i++) q_max = fmaxf(q_max, fabsf(x_q[j][i]));
    // queries
    wm_h8 q[KS][TERMS];
    const int e = query_exponent(group_max(q_max));
    const float kfac = ldexpf(a.scale_log2, e - 15), q_scale = ldexpf(1.0f, 15 - e);
#pragma unroll
    for (int j = 0; j < KS; j++)
#pragma unroll
        for (int i = 0; i < 8; i++) {
            _Float16 hi, lo;
            to_terms<TERMS>(x_q[j][i] * q_scale, &hi, &lo);
            q[j][0][i] = hi;
            if (TERMS > 1) q[j][TERMS - 1][i] = lo;
        }
    const int all = t.q.start + t.r0 / (int)a.group + 1;  // positions that every row attends to

    for (; p < p1; p += 4 * TILE) {
        const bool more = p + 4 * TILE < p1;
        wm_f4 s[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            s[i] = wm_f4{0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < D / 64; j++) {
                wm_h8 k0, k1;
                codes_to_f16(kr[i][j], k0, k1);
#pragma unroll
                for (int w = 0; w < TERMS; w++) {
                    s[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, q[2 * j][w], s[i], 0, 0, 0);
                    s[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, q[2 * j + 1][w], s[i], 0, 0, 0);
                }
            }
        }
        pages pg_after{0, 0};
        if (more) {
            load_k(p + 4 * TILE, pg_next.k);
            sc_next = load_scales(pg_next.v);
            if (p + 8 * TILE < p1) pg_after = load_pages(p + 8 * TILE);
        }
        const bool masked = p + TILE > all;
        const int left = masked ? count - (p + g * 16) : 16;  // of the lane's positions, those that its row attends to
        const int eb = scale_exponent(sc.v);
        ref.raise(group_max(left > 0 ? eb : E_NONE));
        const float part = ref.part(eb, scale_rest(sc.v, eb)), back = __builtin_amdgcn_exp2f(-part);
        wm_h8 w[2][TERMS];
        int fall;
        if (sums.begin(ref, [](float l) { return group_max(l); }, fall))
#pragma unroll
            for (int i = 0; i < DT; i++)
#pragma unroll
                for (int c = 0; c < 4; c++) o[i][c] = ldexpf(o[i][c], -fall);
        const float f = kfac * sc.k, c = part - sums.from;
        float x[16], top = -INFINITY;
#pragma unroll
        for (int i = 0; i < 16; i++) x[i] = __builtin_fmaf(s[i / 4][i % 4], f, c);
        if (masked) {
#pragma unroll
            for (int i = 0; i < 16; i++) x[i] = i < left ? x[i] : -INFINITY;
        }
#pragma unroll
        for (int i = 0; i < 16; i++) top = fmaxf(top, x[i]);
        float by, alpha;
        if (sums.grows(group_max(top), by, alpha)) {
#pragma unroll
            for (int i = 0; i < 16; i++) x[i] -= by;
#pragma unroll
            for (int i = 0; i < DT; i++) o[i] *= alpha;
        }
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const float e = __builtin_amdgcn_exp2f(x[i]);
            sum += e;
            _Float16 hi, lo;
            to_terms<TERMS>(e, &hi, &lo);
            w[i / 8][0][i % 8] = hi;
            if (TERMS > 1) w[i / 8][TERMS - 1][i % 8] = lo;
        }
        sums.l = __builtin_fmaf(sum, back, sums.l);
#pragma unroll
        for (int i = 0; i < DT; i++) {
            wm_h8 v0, v1;
            codes_to_f16(vr[i], v0, v1);
#pragma unroll
            for (int y = 0; y < TERMS; y++) {
                o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, w[0][y], o[i], 0, 0, 0);
                o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, w[1][y], o[i], 0, 0, 0);
            }
        }
        if (more) load_v(p + 4 * TILE, pg_next.v);
        pg_next = pg_after;
        sc = sc_next;
    }

    // rows of this wave, normalised, with the log2 of their sums
    {
        const float sum = group_sum(sums.l);
        const row_scale by(sum, ref.e);
#pragma unroll
        for (int i = 0; i < DT; i++) {
            wm_f4 v;
#pragma unroll
            for (int c = 0; c < 4; c++) v[c] = by(o[i][c]);
            *(wm_f4 *)&sh.o[wave][n][16 * i + 4 * g] = v;
        }
        // a sum of 0 is that of a row without positions, or without a tile
        if (g == 0) sh.lse[wave][n] = sum == 0.0f ? -INFINITY : sums.m + __builtin_amdgcn_logf(sum);
    }
    __syncthreads();
    const int rows = t.rows;
    for (int i = tid; i < rows * (D / 4); i += NT) {
        const int row = i / (D / 4), c = i % (D / 4) * 4;
        float ls[4], top = -INFINITY;
#pragma unroll
        for (int w = 0; w < 4; w++) ls[w] = sh.lse[w][row], top = fmaxf(top, ls[w]);
        const float base = top == -INFINITY ? 0.0f : top;
        wm_f4 v = {0, 0, 0, 0};
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; w++) {
            const float e = half_weight(ls[w] - base);
            sum += e * e;
            v += *(const wm_f4 *)&sh.o[w][row][c] * e * e;
        }
        if (sum != 0.0f) v *= 1.0f / sum;
        const float lse2 = sum == 0.0f ? -INFINITY : base + __builtin_amdgcn_logf(sum);
        const int r = t.r0 + row;
        const uint64_t tok = row_token(a, t, r), head = row_head(a, t, r);
        if (whole) {
            store_out4(a, tok * a.os + head * D + c, v);
            if (a.lse && c == 0) a.lse[tok * a.n_heads + head] = lse2 * 0.6931471805599453f;
        } else {
            const uint64_t part = slot * FEW + row;
            *(wm_f4 *)(a.part_o + part * D + c) = v;
            if (c == 0) a.part_lse[part] = lse2;
        }
    }
}

template <int D, int TERMS>
__device__ __forceinline__ void attend_few(const attn_args &a, uint32_t w, few_shared<D> &sh) {
    const few_share all(a);
    const uint32_t end = uniform(min((w + 1) * all.per, all.total));
    for (uint32_t x = uniform(w * all.per); x < end;) {
        const auto f = all.find(a, x);
        if (f.rounds == 0) return;
        // its kv heads from round x on
        while (x < end && x < f.first + f.rounds * a.kv.n_kv_heads) {
            const uint32_t h = uniform((x - f.first) / f.rounds), k0 = x - f.first - h * f.rounds;
            const uint32_t k1 = min(f.rounds, k0 + (end - x));
            const uint32_t unit = f.s * a.kv.n_kv_heads + h;
            if (k0 == 0 && a.few_parts && threadIdx.x == 0)
                *(wm_u2 *)(a.few_parts + 2 * unit) = wm_u2{w, (x + f.rounds - 1) / all.per - w + 1};
            attend_few_part<D, TERMS>(a, f.q, f.s, h, k0, k1, k1 - k0 == f.rounds, few_share::slot(w, unit), sh);
            x += k1 - k0;
            if (x < end) __syncthreads();  // the next part writes where this one was joined
        }
    }
}

template <int D, int TERMS>
__global__ __launch_bounds__(NT, 2) void k_paged_attn_few(attn_args a) {
    __shared__ few_shared<D> sh;
    attend_few<D, TERMS>(a, blockIdx.x, sh);
}

// The order of the row tiles of sequences of many rows: those with the most
// positions first, so that the last workgroups to start are short, and only
// tiles that exist, so that the compute dies take equal shares (workgroup i
// runs on die i % 8; with every sequence's tiles up to the longest one's in
// the grid, one die had nine times another's work).  A tile's level is its
// number in the sequence plus the context's length in tiles; the tiles at
// level l or above are counted by a scan over the sequences, and a bisection
// finds the level of the y-th.
struct many_order {
    wm_seq q;  // the first 64 sequences, one to a lane
    uint32_t low = 0, tiles = 0;
    __device__ __forceinline__ void load(const attn_args &a, uint32_t s0) {
        const uint32_t s = s0 + (threadIdx.x & 63);
        q = wm_load_seq(a.b, min(s, a.b.n_seqs - 1));
        const int64_t rows = (int64_t)q.n * a.group;
        const bool many = s < a.b.n_seqs && q.ok && rows > FEW;
        tiles = many ? (uint32_t)((rows + MANY - 1) / MANY) : 0;
        low = many ? (uint32_t)((int64_t)max(q.start, 0) * a.group / MANY) : 0;
    }
    __device__ __forceinline__ uint32_t from_level(uint32_t l) const {
        return wm_wave_total_i32(min(low + tiles > l ? low + tiles - l : 0, tiles));
    }
    // Tile y: its sequence and row tile; false past the last (and where lengths
    // change under the kernel).
    __device__ __forceinline__ bool find(const attn_args &a, uint32_t y, wm_seq &seq, uint32_t &s, uint32_t &rt) {
        const bool one = a.b.n_seqs <= 64;
        auto count = [&](uint32_t l) {
            uint32_t n = 0;
            for (uint32_t s0 = 0; s0 < a.b.n_seqs; s0 += 64) {
                if (!one) load(a, s0);
                n += from_level(l);
            }
            return n;
        };
        if (one) load(a, 0);
        if (y >= count(0)) return false;
        uint32_t l = 0, above = a.many_levels;  // count(l) > y >= count(above)
        while (above - l > 1) {
            const uint32_t mid = (l + above) / 2;
            if (count(mid) > y) l = mid;
            else above = mid;
        }
        uint32_t left = y - count(l + 1);  // among the tiles of level l, one of a sequence at most
        for (uint32_t s0 = 0; s0 < a.b.n_seqs; s0 += 64) {
            if (!one) load(a, s0);
            const bool has = low <= l && l < low + tiles;
            const uint64_t mask = __ballot(has);
            const uint32_t n = __popcll(mask);
            if (left < n) {
                const uint64_t hit = __ballot(has && __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32),
                                                                              __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0)) == left);
                const int lane = __builtin_ctzll(hit);
                s = s0 + lane, rt = l - __builtin_amdgcn_readlane(low, lane);
                seq.tok0 = __builtin_amdgcn_readlane(q.tok0, lane), seq.n = __builtin_amdgcn_readlane(q.n, lane);
                seq.start = __builtin_amdgcn_readlane(q.start, lane), seq.len = __builtin_amdgcn_readlane(q.len, lane);
                seq.ok = true;
                return true;
            }
            left -= n;
        }
        return false;
    }
};

// What a wave of a workgroup for many rows holds: 32 rows, their sums, and a
// tile's scores on the way to weights.
template <int D, int TERMS>
struct wave_rows {
    static constexpr int KS = D / 16, DT = D / 32;
    int n, hi;            // the lane's row of the 32, and half
    bool valid;           // (rows past the last repeat it, and are not written)
    int count, all, any;  // positions that the row, all rows, and any row of the wave attend to
    uint64_t tok, head;
    wm_h8 q[KS][TERMS];
    float kfac;
    wm_f16v o[DT];
    row_max sums;
    scale_ref ref;
    // a tile's scales, K's and V's: of the lane's group of 16 positions (lane % 4)
    float ks, v_rest, part, back;
    int v_exp;

    __device__ __forceinline__ void begin(const attn_args &a, const row_tile &t, int w0) {
        const int lane = threadIdx.x & 63;
        n = lane & 31, hi = lane >> 5;
        valid = w0 + n < t.rows;
        const int row = min(w0 + n, t.rows - 1), j = row / (int)a.group;
        count = t.q.start + j + 1;
        all = t.q.start + w0 / (int)a.group + 1;
        any = w0 < t.rows ? t.q.start + (min(w0 + 32, t.rows) - 1) / (int)a.group + 1 : 0;
        tok = (uint64_t)(t.q.tok0 + j), head = (uint64_t)t.h * a.group + row - j * (int)a.group;
        float x[KS][8], m = 0.0f;
        const uint64_t at = tok * a.qs + head * D;
#pragma unroll
        for (int j = 0; j < KS; j++)
#pragma unroll
            for (int i = 0; i < 8; i += 4) {
                const wm_f4 v = load_q4<TERMS>(a, at + 16 * j + 8 * hi + i);
#pragma unroll
                for (int c = 0; c < 4; c++) x[j][i + c] = v[c], m = fmaxf(m, fabsf(v[c]));
            }
        const int e = query_exponent(half_max(m));
        kfac = ldexpf(a.scale_log2, e - 15);
        const float scale = ldexpf(1.0f, 15 - e);
#pragma unroll
        for (int j = 0; j < KS; j++)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                _Float16 h, lo;
                to_terms<TERMS>(x[j][i] * scale, &h, &lo);
                q[j][0][i] = h;
                if (TERMS > 1) q[j][TERMS - 1][i] = lo;
            }
#pragma unroll
        for (int i = 0; i < DT; i++)
#pragma unroll
            for (int c = 0; c < 16; c++) o[i][c] = 0.0f;
    }
    // The scales of the tile at p, and the rows' reference with them: the
    // scales relative to it as logarithms, and their inverses, where all rows
    // have the same (in masked tiles `weights` does that row by row).
    __device__ __forceinline__ void take_scales(const float (*scale)[2], int p) {
        const float v = scale[threadIdx.x & 3][1];
        ks = scale[threadIdx.x & 3][0], v_exp = scale_exponent(v), v_rest = scale_rest(v, v_exp);
        int e = max(v_exp, __builtin_amdgcn_mov_dpp(v_exp, 0xB1, 0xF, 0xF, true));  // over lanes l ^ 1, l ^ 2
        e = max(e, __builtin_amdgcn_mov_dpp(e, 0x4E, 0xF, 0xF, true));
        if (p + TILE > all) {
            e = E_NONE;
#pragma unroll
            for (int g = 0; g < 4; g++) e = max(e, 16 * g < count - p ? __builtin_amdgcn_readlane(v_exp, g) : E_NONE);
        }
        ref.raise(e);
        part = ref.part(v_exp, v_rest), back = __builtin_amdgcn_exp2f(-part);
        int fall;
        if (sums.begin(ref, half_max, fall))
#pragma unroll
            for (int i = 0; i < DT; i++)
#pragma unroll
                for (int c = 0; c < 16; c++) o[i][c] = ldexpf(o[i][c], -fall);
    }
    // S^T = K Q^T of a tile in LDS.
    __device__ __forceinline__ void scores(const _Float16 (*k)[D + 8], wm_f16v (&s)[2]) const {
#pragma unroll
        for (int i = 0; i < 2; i++) {
            s[i] = wm_f16v{0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < KS; j++) {
                const wm_h8 x = *(const wm_h8 *)&k[32 * i + n][16 * j + 8 * hi];
#pragma unroll
                for (int y = 0; y < TERMS; y++) s[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, q[j][y], s[i], 0, 0, 0);
            }
        }
    }
    // Scores of the tile at p to weights, relative to the maximum so far, the
    // values' scale included.
    __device__ __forceinline__ void weights(const wm_f16v (&s)[2], int p, wm_h8 (&w)[4][TERMS]) {
        const bool masked = p + TILE > all;
        float c[4], inverse[4];
#pragma unroll
        for (int g = 0; g < 4; g++) c[g] = read_lane(part, g) - sums.from, inverse[g] = read_lane(back, g);
        if (masked) {
#pragma unroll
            for (int g = 0; g < 4; g++) {
                const float of_row = ref.part(__builtin_amdgcn_readlane(v_exp, g), read_lane(v_rest, g));
                c[g] = of_row - sums.from, inverse[g] = __builtin_amdgcn_exp2f(-of_row);
            }
        }
        float x[4][8];
#pragma unroll
        for (int g = 0; g < 4; g++) {
            const float f = kfac * read_lane(ks, g);
#pragma unroll
            for (int y = 0; y < 8; y++) x[g][y] = __builtin_fmaf(s[g / 2][8 * (g % 2) + y], f, c[g]);
        }
        if (masked) {
            const int left = count - p - 4 * hi;
#pragma unroll
            for (int g = 0; g < 4; g++)
#pragma unroll
                for (int y = 0; y < 8; y++) x[g][y] = 16 * g + 8 * (y / 4) + y % 4 < left ? x[g][y] : -INFINITY;
        }
        float top = -INFINITY;
#pragma unroll
        for (int g = 0; g < 4; g++)
#pragma unroll
            for (int y = 0; y < 8; y++) top = fmaxf(top, x[g][y]);
        float by, alpha;
        if (sums.grows(half_max(top), by, alpha)) {
#pragma unroll
            for (int i = 0; i < DT; i++) o[i] *= alpha;
#pragma unroll
            for (int g = 0; g < 4; g++)
#pragma unroll
                for (int y = 0; y < 8; y++) x[g][y] -= by;
        }
#pragma unroll
        for (int g = 0; g < 4; g++) {
            float sum = 0.0f;
#pragma unroll
            for (int y = 0; y < 8; y++) {
                const float e = __builtin_amdgcn_exp2f(x[g][y]);
                sum += e;
                _Float16 h, lo;
                to_terms<TERMS>(e, &h, &lo);
                w[g][0][y] = h;
                if (TERMS > 1) w[g][TERMS - 1][y] = lo;
            }
            sums.l = __builtin_fmaf(sum, inverse[g], sums.l);
        }
    }
    // O^T += V^T P^T of a tile in LDS.
    __device__ __forceinline__ void values(const _Float16 (*v)[TILE + 8], const wm_h8 (&w)[4][TERMS]) {
#pragma unroll
        for (int i = 0; i < DT; i++)
#pragma unroll
            for (int g = 0; g < 4; g++) {
                const wm_h8 x = *(const wm_h8 *)&v[32 * i + n][16 * g + 8 * hi];
#pragma unroll
                for (int y = 0; y < TERMS; y++) o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, w[g][y], o[i], 0, 0, 0);
            }
    }
    __device__ __forceinline__ void write(const attn_args &a, const row_tile &t, bool whole, uint32_t split) const {
        if (!valid) return;
        const float sum = half_sum(sums.l);
        const row_scale by(sum, ref.e);
        const float lse2 = sum == 0.0f ? -INFINITY : sums.m + __builtin_amdgcn_logf(sum);
        const uint64_t part_at = whole ? 0 : many_part(a, t.s, t.q, tok, head) + split;
#pragma unroll
        for (int i = 0; i < DT; i++)
#pragma unroll
            for (int c = 0; c < 16; c += 4) {
                wm_f4 v;
#pragma unroll
                for (int x = 0; x < 4; x++) v[x] = by(o[i][c + x]);
                const int d = 32 * i + 2 * c + 4 * hi;
                if (whole) store_out4(a, tok * a.os + head * D + d, v);
                else *(wm_f4 *)(a.part_o + part_at * D + d) = v;
            }
        if (hi == 0) {
            if (!whole) a.part_lse[part_at] = lse2;
            else if (a.lse) a.lse[tok * a.n_heads + head] = lse2 * 0.6931471805599453f;
        }
    }
};

// A workgroup's row tile and split, of those that exist.
struct many_work {
    row_tile t;
    uint32_t split;
    int p0, p1;
    bool whole;
    __device__ __forceinline__ bool find(const attn_args &a, uint32_t id) {
        const uint32_t part_id = id % a.many_n, tile_id = id / a.many_n;
        wm_seq seq;
        uint32_t s, rt;
        if (!many_order().find(a, tile_id / a.kv.n_kv_heads, seq, s, rt)) return false;
        t = make_tile(a, seq, s, tile_id % a.kv.n_kv_heads, rt, MANY);
        split = (part_id + tile_id) % a.many_n;  // (a short tile's missing splits fall on every die)
        p0 = (int)(split * a.many_len), p1 = (int)min((int64_t)p0 + a.many_len, (int64_t)t.len);
        whole = t.len <= (int)a.many_len;
        return split == 0 || p0 < t.len;
    }
};

// A tile of 64 positions, converted once to f16 for all waves: K [position]
// [dim], V [dim][position] with each 16 positions in the order that a lane's
// half of the second product's K = 16 step takes them (0-3, 8-11 | 4-7,
// 12-15), so both operands are 16-byte reads.  Rows are padded by 16 bytes:
// 16 lanes' reads then fall into all 64 banks.
template <int D>
struct alignas(16) shared_tile {
    _Float16 k[TILE][D + 8];
    _Float16 v[D][TILE + 8];
    float scale[4][2];  // of each 16 positions, K's and V's
};

// One wave's share in making tiles, a quarter of K's codes or of V's: wave w
// of four takes what lies in the page of the tile's positions 16 w .. + 15,
// so that a page is one scalar and a lane's addresses are a scalar base and
// offsets that stay.  K: those 16 positions.  V: of a page of 16 n positions
// that n waves share, the D / n dims that are its turn's, all positions.
template <int D>
struct stager {
    static constexpr int U = D / 64;  // 16-byte units per lane
    const int8_t *codes;
    uint64_t block;
    uint32_t off[U], lds[U];
    bool is_v;
    wm_u4 raw[U];
    __device__ __forceinline__ void begin(const attn_args &a, uint32_t h, int w, bool v) {
        const int ps = (int)a.kv.page_size, ng = ps / 16, lane = threadIdx.x & 63, sub = w & (ng - 1);
        block = (uint64_t)ps * D;
        codes = (v ? a.kv.v_codes : a.kv.k_codes) + h * block;
        block *= a.kv.n_kv_heads;
        is_v = v;
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int x = lane + 64 * u;
            const int pos = x / (D / 16), kdim = x % (D / 16) * 16;
            const int grp = x & (ng - 1), dim = (sub * D + x) / ng;
            off[u] = v ? dim * ps + 16 * grp : (16 * sub + pos) * D + kdim;
            lds[u] = v ? (uint32_t)offsetof(shared_tile<D>, v) + (dim * (TILE + 8) + 16 * (w - sub + grp)) * 2
                       : ((16 * w + pos) * (D + 8) + kdim) * 2;
        }
    }
    __device__ __forceinline__ void load(uint32_t page) {
        const int8_t *base = codes + page * block;
#pragma unroll
        for (int u = 0; u < U; u++) raw[u] = *(const wm_u4 *)(base + off[u]);
    }
    __device__ __forceinline__ void put(shared_tile<D> *tile) const {
#pragma unroll
        for (int u = 0; u < U; u++) {
            wm_h8 c0, c1;
            // (V's 16 positions in a half's order)
            codes_to_f16(wm_u4{raw[u].x, is_v ? raw[u].z : raw[u].y, is_v ? raw[u].y : raw[u].z, raw[u].w}, c0, c1);
            char *to = (char *)tile + lds[u];
            *(wm_h8 *)to = c0;
            *(wm_h8 *)(to + 16) = c1;
        }
    }
};
// The page of a wave's 16 positions, tile after tile, loaded a turn ahead of
// its use, and the block's two scales (lane 0 K's, lane 1 V's).
struct page_walk {
    const int32_t *table;
    const float *scales;
    uint32_t n_pages, n_kv, ps_log;
    int last, ahead;
    uint32_t page;  // of the tile last turned to: within the pool
    bool good;      // as the table has it
    float scale;
    __device__ __forceinline__ void begin(const attn_args &a, const row_tile &t, int w) {
        table = a.b.page_table + (uint64_t)t.s * a.b.table_stride;
        scales = ((threadIdx.x & 1) ? a.kv.v_scales : a.kv.k_scales) + t.h;
        n_pages = a.kv.n_pages, n_kv = a.kv.n_kv_heads, ps_log = 31 - __builtin_clz(a.kv.page_size);
        last = t.len - 1;
    }
    // (past the last position: its page)
    __device__ __forceinline__ void look(int position) { ahead = table[min(position, last) >> ps_log]; }
    __device__ __forceinline__ void turn() {
        const uint32_t id = (uint32_t)uniform(ahead);
        good = id < n_pages;
        page = good ? id : 0;
    }
    __device__ __forceinline__ void load_scale() { scale = scales[(uint64_t)page * n_kv]; }
    __device__ __forceinline__ void put_scale(float (*to)[2], int w, bool good) const {
        const int lane = threadIdx.x & 63;
        if (lane < 2) to[w][lane] = good ? scale : lane ? 0.0f : __uint_as_float(0x7FC00000u);
    }
};

// Many rows.  One workgroup: 128 rows of one sequence and kv head, 32 to a
// wave, one split of the positions (all of them where there are workgroups
// enough).  Two buffers, one barrier per tile: the next tile's codes are
// loaded a tile ahead and converted while the matrix cores work on this one.
// 128 rows and two workgroups to a compute unit: 256 rows in eight waves of
// one, half of them at their products while the others are at their
// exponentials, took 465 us for a prompt of 8192 against 408.
template <int D>
struct alignas(16) many_shared {
    shared_tile<D> tile[2];
};
template <int D, int TERMS>
__device__ __forceinline__ void attend_many(const attn_args &a, uint32_t id, many_shared<D> &sh) {
    many_work work;
    if (!work.find(a, id)) return;
    const row_tile &t = work.t;
    wave_rows<D, TERMS> rows;
    stager<D> k, v;
    page_walk pages;
    const int wave = uniform((int)threadIdx.x >> 6);
    pages.begin(a, t, wave);
    if (work.p0 < work.p1) pages.look(work.p0 + 16 * wave);  // (rows without positions have no page)
    rows.begin(a, t, t.r0 + 32 * wave);
    k.begin(a, t.h, wave, false), v.begin(a, t.h, wave, true);
    auto load = [&](int next) {  // the tile turned to, and the page of the one behind it
        pages.turn();
        pages.look(next + 16 * wave);
        pages.load_scale();
        k.load(pages.page), v.load(pages.page);
    };
    auto put = [&](int buf) {
        k.put(&sh.tile[buf]), v.put(&sh.tile[buf]);
        pages.put_scale(sh.tile[buf].scale, wave, pages.good);
    };
    if (work.p0 < work.p1) {
        load(work.p0 + TILE);
        put(0);
    }
    int buf = 0;
    for (int p = work.p0; p < work.p1; p += TILE, buf ^= 1) {
        const bool more = p + TILE < work.p1;
        if (more) load(p + 2 * TILE);
        __syncthreads();
        rows.take_scales(sh.tile[buf].scale, p);
        const bool live = p < rows.any;
        wm_h8 w[4][TERMS];
        if (live) {
            wm_f16v s[2];
            rows.scores(sh.tile[buf].k, s);
            rows.weights(s, p, w);
        }
        if (more) put(buf ^ 1);
        if (live) rows.values(sh.tile[buf].v, w);
    }
    rows.write(a, t, work.whole, work.split);
}

// A step with sequences of many rows, whose workgroups run longer and come
// first; behind them those of few rows (in front of them, most of them
// without any, they took a ragged step from 45.8 us to 47.9).
template <int D, int TERMS>
__global__ __launch_bounds__(NT, 2) void k_paged_attn_many(attn_args a) {
    __shared__ union alignas(16) {
        few_shared<D> few;
        many_shared<D> many;
    } sh;
    if (blockIdx.x < a.many_blocks) attend_many<D, TERMS>(a, blockIdx.x, sh.many);
    else attend_few<D, TERMS>(a, blockIdx.x - a.many_blocks, sh.few);
}

// The rows' parts joined: weights 2^(lse - max), one thread per four dims;
// one workgroup per FEW rows of a sequence (of the launch's, from seq0 on) and
// kv head.
template <int D>
__global__ __launch_bounds__(NT) void k_paged_attn_join(attn_args a, uint32_t chunks, uint32_t seq0) {
    uint32_t id = blockIdx.x;
    const uint32_t chunk = id % chunks;
    id /= chunks;
    const uint32_t s = seq0 + id / a.kv.n_kv_heads, h = id % a.kv.n_kv_heads;
    const uint32_t unit = s * a.kv.n_kv_heads + h;
    const wm_u2 parts = a.few_blocks ? *(const wm_u2 *)(a.few_parts + 2 * unit) : wm_u2{0, 0};  // where its rows are few
    const row_tile t = load_tile(a, s, h, chunk / (MANY / FEW), MANY);
    const bool few = t.rows <= FEW;
    const int r0 = (int)chunk * FEW, rows = min(FEW, t.rows - r0);
    if (rows <= 0 || !t.q.ok) return;
    int n;
    uint64_t first = 0;
    if (few) {
        n = (int)parts.y;
        first = few_share::slot(parts.x, unit) * FEW;
    } else {
        n = (t.len + (int)a.many_len - 1) / (int)a.many_len;
    }
    if (n <= 1) return;  // written whole
    const uint64_t step = few ? FEW : 1;  // rows from one part of a row to its next
    for (int i = threadIdx.x; i < rows * (D / 4); i += NT) {
        const int r = r0 + i / (D / 4), c = i % (D / 4) * 4;
        const uint64_t tok = row_token(a, t, r), head = row_head(a, t, r);
        const uint64_t part = few ? first + r : many_part(a, s, t.q, tok, head);
        const float *ls = a.part_lse + part, *os = a.part_o + part * D + c;
        // eight splits at a time, their loads together
        wm_f4 v = {0, 0, 0, 0};
        float top = -INFINITY, sum = 0.0f;
        for (int s0 = 0; s0 < n; s0 += 8) {
            float z[8];
            wm_f4 x[8];
#pragma unroll
            for (int s = 0; s < 8; s++) {
                const int at = min(s0 + s, n - 1);
                z[s] = ls[at * step];
                x[s] = *(const wm_f4 *)(os + at * step * D);
            }
            float m = top;
#pragma unroll
            for (int s = 0; s < 8; s++) {
                if (s0 + s >= n) z[s] = -INFINITY;
                m = fmaxf(m, z[s]);
            }
            const float to = m == -INFINITY ? 0.0f : m, alpha = half_weight(top - to);
            sum *= alpha * alpha, v *= alpha, v *= alpha, top = m;
#pragma unroll
            for (int s = 0; s < 8; s++) {
                const float e = half_weight(z[s] - to);
                sum += e * e;
                v += x[s] * e * e;
            }
        }
        const float base = top == -INFINITY ? 0.0f : top;
        if (sum != 0.0f) v *= 1.0f / sum;
        store_out4(a, tok * a.os + head * D + c, v);
        if (a.lse && c == 0)
            a.lse[tok * a.n_heads + head] = sum == 0.0f ? -INFINITY : (base + __builtin_amdgcn_logf(sum)) * 0.6931471805599453f;
    }
}

// How a step is divided: from the host's bounds alone, of a step that has
// tokens and whose max_new times the group fits 32 bits.
struct attn_plan {
    bool many;         // a sequence may have more than FEW rows
    uint32_t many_levels, many_len, many_n;
    uint64_t few_blocks, many_blocks;
    uint32_t join_chunks;  // of a sequence and kv head
    bool join;
    size_t parts;      // partial rows
    bool parts_by_seq;
    uint64_t rounds;   // of all sequences and kv heads, at most
};
// Tokens that rows of splits are kept of: the packed ones or max_new of each
// sequence, whichever are fewer, so that padding costs none.
uint64_t kept_tokens(const wm_paged_batch *b) {
    const uint64_t by_seq = (uint64_t)b->n_seqs * b->max_new;
    return by_seq < b->n_tokens ? by_seq : b->n_tokens;
}
attn_plan make_plan(const wm_paged_kv *kv, const wm_paged_batch *b, uint32_t n_heads) {
    attn_plan p;
    const uint64_t rows = (uint64_t)b->max_new * (n_heads / kv->n_kv_heads), units = (uint64_t)b->n_seqs * kv->n_kv_heads;
    const uint32_t rounds = b->max_kv_len > ROUND ? (b->max_kv_len + ROUND - 1) / ROUND : 1;
    p.many = rows > FEW;
    p.few_blocks = units * rounds < 2 * FEW_RESIDENT ? units * rounds : 2 * FEW_RESIDENT;
    p.parts = rounds > 1 ? (size_t)few_slots((uint32_t)p.few_blocks, (uint32_t)units) * FEW : 0;
    p.join = rounds > 1;
    p.parts_by_seq = kept_tokens(b) < b->n_tokens;
    p.rounds = units * rounds;
    p.many_levels = 0, p.many_blocks = 0, p.many_len = 0, p.many_n = 1, p.join_chunks = 1;
    if (p.many) {
        const uint64_t most = (rows + MANY - 1) / MANY;  // of one sequence and kv head
        // as many row tiles as the packed tokens can fill, not as many as the longest would in every sequence
        const uint64_t full = (uint64_t)b->n_tokens * (n_heads / kv->n_kv_heads) / MANY + b->n_seqs;
        const uint64_t tiles = full < most * b->n_seqs ? full : most * b->n_seqs;
        // 512 workgroups fit the device
        const uint64_t want = (512 + tiles * kv->n_kv_heads - 1) / (tiles * kv->n_kv_heads);
        const uint32_t per = want < rounds ? (uint32_t)(rounds / want) : 1;
        p.many_len = per * ROUND;
        p.many_n = (rounds + per - 1) / per;
        p.many_blocks = tiles * kv->n_kv_heads * p.many_n;
        p.many_levels = (uint32_t)most + (uint32_t)((uint64_t)b->max_kv_len * (n_heads / kv->n_kv_heads) / MANY) + 1;
        if (p.many_n > 1) {
            p.parts = (size_t)few_slots((uint32_t)p.few_blocks, (uint32_t)units) * FEW;
            p.parts += (kept_tokens(b) * n_heads * p.many_n + 1) & ~(size_t)1;
            p.join_chunks = (uint32_t)most * (MANY / FEW);
        }
    }
    return p;
}

bool sizes_fit(const wm_paged_kv *kv, const wm_paged_batch *b, uint32_t n_heads) {
    return (uint64_t)(b->max_new > b->max_kv_len ? b->max_new : b->max_kv_len) * (n_heads / kv->n_kv_heads) <= 1u << 30;
}
// Partial rows, the log2 of their sums, and each unit's parts: of this plan
// and of those of all smaller bounds (a smaller step may have more splits).
// Of T = tiles * kv heads a split step has T < 512 and up to 2 ceil(512 / T) -
// 1 splits, so T * many_n <= 1022 + T <= 1533, and its kept tokens fill MANY
// rows of each tile at most.
constexpr uint64_t MOST_PARTS = (uint64_t)MANY * 1533;
size_t plan_bytes(const attn_plan &p, const wm_paged_kv *kv, const wm_paged_batch *b, uint32_t n_heads) {
    if (!p.join) return 0;
    const uint64_t units = (uint64_t)b->n_seqs * kv->n_kv_heads, rounds = (b->max_kv_len + ROUND - 1) / ROUND;
    uint64_t many = 0;
    if (p.many) {
        const uint64_t tokens = kept_tokens(b);
        many = tokens < MOST_PARTS ? tokens * n_heads : MOST_PARTS;
        many = many < MOST_PARTS ? (many * rounds + 1) & ~(uint64_t)1 : MOST_PARTS;
        many = many < MOST_PARTS ? many : MOST_PARTS;
    }
    return (few_slots((uint32_t)p.few_blocks, (uint32_t)units) * FEW + many) * (kv->head_dim + 1) * sizeof(float) +
           units * sizeof(wm_u2);
}

}  // namespace

extern "C" {

size_t wm_paged_attention_workspace(const wm_paged_kv *kv, const wm_paged_batch *batch, uint32_t n_heads) {
    if (!kv || !batch || !kv->n_kv_heads || n_heads % kv->n_kv_heads || !sizes_fit(kv, batch, n_heads)) return 0;
    if (batch->n_tokens == 0 || batch->n_seqs == 0 || batch->max_new == 0) return 0;
    return plan_bytes(make_plan(kv, batch, n_heads), kv, batch, n_heads);
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
    const float scale_log2 = scale * 1.4426950408889634f;
    if (!(scale_log2 - scale_log2 == 0.0f)) return wm_set_error(ctx, WM_E_NONFINITE, "%s: scale %g", who, (double)scale);
    if (batch->n_tokens == 0 || batch->n_seqs == 0 || batch->max_new == 0) return WM_OK;
    if ((st = wm_paged_check_array(ctx, who, "q", d_q, q_stride, n_heads, kv->head_dim, elem))) return st;
    if ((st = wm_paged_check_array(ctx, who, "out", d_out, out_stride, n_heads, kv->head_dim, elem))) return st;
    if ((st = wm_paged_check_over(ctx, who, d_q, q_stride, d_out, out_stride))) return st;
    if ((uintptr_t)d_lse % 4) return wm_set_error(ctx, WM_E_ARG, "%s: misaligned lse", who);
    if (!sizes_fit(kv, batch, n_heads))
        return wm_set_error(ctx, WM_E_SHAPE, "%s: max_new %u or max_kv_len %u is too large for %u heads over %u", who,
                            batch->max_new, batch->max_kv_len, n_heads, kv->n_kv_heads);
    const attn_plan p = make_plan(kv, batch, n_heads);
    // A launch counts threads in 32 bits.  The join, which has a workgroup for
    // every FEW rows that any sequence may have, takes some sequences at a time.
    const uint64_t most = 0x7FFFFFFFull / NT, blocks = p.few_blocks + p.many_blocks;
    const uint64_t seq_blocks = (uint64_t)kv->n_kv_heads * p.join_chunks, units = (uint64_t)kv->n_kv_heads * batch->n_seqs;
    if (blocks > most || p.rounds > 0x3FFFFFFF || (p.join && (seq_blocks > most || units > most)))
        return wm_set_error(ctx, WM_E_SHAPE, "%s: %llu workgroups, %llu rounds of %d positions, %u sequences of up to %llu "
                            "joins in one step", who, (unsigned long long)blocks, (unsigned long long)p.rounds, ROUND,
                            batch->n_seqs, (unsigned long long)seq_blocks);
    const size_t need = plan_bytes(p, kv, batch, n_heads);
    if (need && (!d_work || work_bytes < need || (uintptr_t)d_work % 16))
        return wm_set_error(ctx, WM_E_ARG, "%s: workspace of %zu bytes, %zu needed, 16-byte aligned", who,
                            d_work ? work_bytes : (size_t)0, need);
    attn_args a;
    memset(&a, 0, sizeof a);
    a.kv = *kv, a.b = *batch;
    a.q = d_q, a.out = d_out, a.lse = d_lse;
    a.qs = q_stride, a.os = out_stride;
    a.n_heads = n_heads, a.group = n_heads / kv->n_kv_heads;
    a.few_recip = (0x10000 + a.group - 1) / a.group;
    a.type = type;
    a.scale_log2 = scale_log2;
    a.few_blocks = (uint32_t)p.few_blocks, a.many_blocks = (uint32_t)p.many_blocks;
    a.many_levels = p.many_levels, a.many_len = p.many_len, a.many_n = p.many_n;
    a.part_o = (float *)d_work, a.parts_by_seq = p.parts_by_seq;
    if (p.join) {
        a.part_lse = a.part_o + p.parts * kv->head_dim;
        a.few_parts = (uint32_t *)(a.part_lse + p.parts);  // FEW rows to a part: an even count
    }
    wm_device_guard dev(ctx->device);
    WM_HIP(ctx, dev.err);
    const uint32_t grid = (uint32_t)blocks;
    hipStream_t s = ctx->stream;
    const bool two = type == WM_DTYPE_F32;
#define WM_ATTEND(D_)                                                                  \
    do {                                                                               \
        if (p.many && two) k_paged_attn_many<D_, 2><<<grid, NT, 0, s>>>(a);             \
        else if (p.many) k_paged_attn_many<D_, 1><<<grid, NT, 0, s>>>(a);               \
        else if (two) k_paged_attn_few<D_, 2><<<grid, NT, 0, s>>>(a);                   \
        else k_paged_attn_few<D_, 1><<<grid, NT, 0, s>>>(a);                            \
    } while (0)
    if (kv->head_dim == 64) WM_ATTEND(64);
    else WM_ATTEND(128);
#undef WM_ATTEND
    WM_HIP(ctx, hipGetLastError());
    for (uint32_t s0 = 0, n; p.join && s0 < batch->n_seqs; s0 += n) {
        n = (uint32_t)std::min<uint64_t>(batch->n_seqs - s0, most / seq_blocks);
        const uint32_t g = (uint32_t)(n * seq_blocks);
        if (kv->head_dim == 64) k_paged_attn_join<64><<<g, NT, 0, s>>>(a, p.join_chunks, s0);
        else k_paged_attn_join<128><<<g, NT, 0, s>>>(a, p.join_chunks, s0);
        WM_HIP(ctx, hipGetLastError());
    }
    return WM_OK;
}

}  // extern "C"
