// Log probabilities of given tokens, the entropy of their distribution, the
// token's rank and the top alternatives, per row of logits.
//
// With m any number near the largest logit, l = sum e^(x - m) and
// s = sum (x - m) e^(x - m):
//   logprob = x[token] - m - log l,   entropy = log l - s / l,
// and sums of two parts of a row join under the larger m.
//
// The bound is one read of the logits: a workgroup takes a part of a row into
// registers (at most 64 VGPRs a lane, all loads in flight at once), and
// maximum, sums, rank and top tokens come from there.  Lanes read whole
// 16-byte vectors wherever the row begins.  The top tokens of a part: about
// the k-th largest of the lanes' maxima is a value that at least k logits
// reach, and few more do, so those are listed and ranked by counting.  A
// second launch joins the parts of a row.
//
// Measured (f32, 512 rows of 128256, top 5): 51 us, of which 46 are the parts
// (263 MB, 5.7 TB/s; the chip's last cache holds some of it).  16-bit logits
// are nearer to the vector unit's rate: 14 instructions per logit, among them
// an exponential, take 65 % of a SIMD's time; 2047 rows of 50257 in bfloat16
// (206 MB) take 57 us.  One row of 128256, in 32 short parts, takes 12.5 us,
// the length of two launches' chains.
#include <algorithm>
#include <cstdio>
#include <cstring>

#include "wm_paged.h"

namespace {

constexpr int NT = 256;
constexpr uint32_t MAX_TOP = 64, MAX_VOCAB = 1u << 30;
constexpr int LIST = 512;   // logits that may reach the threshold before a slower way is taken
constexpr int FIRST = 128;  // a part's first ids, listed on that way

struct lp_part {  // of one part of a row; with `keys` what the join reads
    float m, l, s;
    int32_t before;
};

struct lp_args {
    const void *x;
    uint64_t stride;
    uint32_t n_rows, vocab, top_k;
    const int32_t *tokens;
    float *logprob, *entropy;
    int32_t *rank, *top_ids;
    float *top_logprobs;
    uint32_t parts, part_vecs;  // parts of a row, 16-byte vectors of each
    lp_part *part;              // [row][part]
    uint64_t *keys;             // [row][part][top_k], in order
};

// Order of (logit descending, id): the larger key comes first.  Zeros are
// one value; NaN is below every number; no logit has key 0.
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return x != x ? 1u : b ^ ((int)b < 0 ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ uint64_t key_of(float x, uint32_t id) { return (uint64_t)ordered(x) << 32 | ~id; }
__device__ __forceinline__ float key_value(uint64_t key) {
    const uint32_t o = (uint32_t)(key >> 32);
    return o <= 1 ? __uint_as_float(0x7FC00000u) : __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o);
}
// The value of lane l ^ D, by moves inside the vector unit (a few cycles; a
// shuffle through LDS takes about a hundred).
template <int D>
__device__ __forceinline__ uint32_t lane_xor(uint32_t v) {
    if (D == 1) return __builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, true);
    if (D == 2) return __builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xF, 0xF, true);
    if (D == 4) {  // lanes 0-3 and 8-11 of each 16 from four above, the others from four below
        const int up = __builtin_amdgcn_update_dpp(0, (int)v, 0x104, 0xF, 0x5, false);
        return __builtin_amdgcn_update_dpp(up, (int)v, 0x114, 0xF, 0xA, false);
    }
    if (D == 8) return __builtin_amdgcn_mov_dpp((int)v, 0x128, 0xF, 0xF, true);
    if (D == 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        return (threadIdx.x & 16) ? r[0] : r[1];
    }
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return (threadIdx.x & 32) ? r[0] : r[1];
}
template <int D> __device__ __forceinline__ float lane_xor(float v) { return __uint_as_float(lane_xor<D>(__float_as_uint(v))); }
template <int D> __device__ __forceinline__ uint64_t lane_xor(uint64_t v) {
    return (uint64_t)lane_xor<D>((uint32_t)(v >> 32)) << 32 | lane_xor<D>((uint32_t)v);
}
// f(value, value of lane l ^ D) over D = 32 .. 1.
template <typename T, typename F>
__device__ __forceinline__ T over_lanes(T v, F f) {
    v = f(v, lane_xor<32>(v));
    v = f(v, lane_xor<16>(v));
    v = f(v, lane_xor<8>(v));
    v = f(v, lane_xor<4>(v));
    v = f(v, lane_xor<2>(v));
    return f(v, lane_xor<1>(v));
}
__device__ __forceinline__ float lanes_sum(float v) {
    return over_lanes(v, [](float a, float b) { return a + b; });
}
__device__ __forceinline__ float lanes_max(float v) {
    return over_lanes(v, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ uint64_t lanes_max(uint64_t v) {
    return over_lanes(v, [](uint64_t a, uint64_t b) { return max(a, b); });
}
// One exchange of a descending bitonic sort over the wave: runs of SIZE.
template <int SIZE, int D>
__device__ __forceinline__ void exchange(float &y) {
    const float o = lane_xor<D>(y);
    const bool lower = ((threadIdx.x & D) != 0) != ((threadIdx.x & SIZE) != 0 && SIZE < 64);
    y = lower ? fminf(y, o) : fmaxf(y, o);
    if constexpr (D > 1) exchange<SIZE, D / 2>(y);
}
__device__ __forceinline__ float sorted(float y) {
    exchange<2, 1>(y);
    exchange<4, 2>(y);
    exchange<8, 4>(y);
    exchange<16, 8>(y);
    exchange<32, 16>(y);
    exchange<64, 32>(y);
    return y;
}

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

// e^(x - m) sums of two parts under their common maximum.
__device__ __forceinline__ lp_part join_parts(lp_part a, lp_part b) {
    const float m = fmaxf(a.m, b.m), base = m == -INFINITY ? 0.0f : m;
    const float da = a.m - base, db = b.m - base;
    const float ea = __builtin_amdgcn_exp2f(da * LOG2E), eb = __builtin_amdgcn_exp2f(db * LOG2E);
    return {m, a.l * ea + b.l * eb,
            ea * (a.s + a.l * fmaxf(da, -200.0f)) + eb * (b.s + b.l * fmaxf(db, -200.0f)), a.before + b.before};
}

// The same over lanes that differ in bits D and below.
template <int D>
__device__ __forceinline__ lp_part join_lanes(lp_part p) {
    p = join_parts(p, {lane_xor<D>(p.m), lane_xor<D>(p.l), lane_xor<D>(p.s), (int)lane_xor<D>((uint32_t)p.before)});
    if constexpr (D > 1) p = join_lanes<D / 2>(p);
    return p;
}

// What a finished row says.
struct row_end {
    float m, log_l;
    bool none;  // every logit -inf
};
__device__ __forceinline__ row_end end_row(const lp_part &p) {
    const bool none = p.m == -INFINITY && p.l == 0.0f;
    return {p.m, none ? 0.0f : logf(p.l), none};
}
__device__ __forceinline__ float end_logprob(const row_end &e, float x) {
    const float p = e.none ? x : (x - e.m) - e.log_l;
    return p > 0.0f ? 0.0f : p;  // (by the sum's rounding)
}
__device__ __forceinline__ void write_row(const lp_args &a, uint32_t row, const lp_part &p, const row_end &e, bool known,
                                          float xt) {
    if (a.logprob) a.logprob[row] = known ? end_logprob(e, xt) : __uint_as_float(0x7FC00000u);
    const float entropy = e.none ? 0.0f : e.log_l - p.s / p.l;
    if (a.entropy) a.entropy[row] = entropy < 0.0f ? 0.0f : entropy;
    if (a.rank) a.rank[row] = known ? p.before : -1;
}
__device__ __forceinline__ void write_top(const lp_args &a, uint32_t row, uint32_t i, const row_end &e, uint64_t key) {
    const uint64_t at = (uint64_t)row * a.top_k + i;
    if (a.top_ids) a.top_ids[at] = (int32_t)~(uint32_t)key;
    if (a.top_logprobs) a.top_logprobs[at] = end_logprob(e, key_value(key));
}

// The elements of one 16-byte vector.
template <typename T> struct vec;
template <> struct vec<float> {
    static constexpr int N = 4;
    static constexpr uint32_t LOW = 0xFF800000u;  // -inf in every element of a word
    static __device__ __forceinline__ float at(wm_u4 v, int i) { return __uint_as_float(v[i]); }
    static __device__ __forceinline__ float one(const float *p) { return *p; }
    static __device__ __forceinline__ uint32_t bits(const float *p) { return __float_as_uint(*p); }
};
template <> struct vec<_Float16> {
    static constexpr int N = 8;
    static constexpr uint32_t LOW = 0xFC00FC00u;
    static __device__ __forceinline__ float at(wm_u4 v, int i) {
        return (float)__builtin_bit_cast(wm_h2, (unsigned)v[i / 2])[i % 2];
    }
    static __device__ __forceinline__ float one(const _Float16 *p) { return (float)*p; }
    static __device__ __forceinline__ uint32_t bits(const _Float16 *p) { return *(const uint16_t *)p; }
};
template <> struct vec<__bf16> {
    static constexpr int N = 8;
    static constexpr uint32_t LOW = 0xFF80FF80u;
    static __device__ __forceinline__ float at(wm_u4 v, int i) {
        return __uint_as_float(i % 2 ? v[i / 2] & 0xFFFF0000u : v[i / 2] << 16);
    }
    static __device__ __forceinline__ float one(const __bf16 *p) { return __uint_as_float((uint32_t)bits(p) << 16); }
    static __device__ __forceinline__ uint32_t bits(const __bf16 *p) { return *(const uint16_t *)p; }
};

// In front of each use of a vector of 16-bit values in a pass over the
// registers: without it values unpacked in one pass stay alive for the next,
// or all of a pass are unpacked at its beginning, and the registers overflow.
__device__ __forceinline__ void repack(wm_u4 &v) { asm volatile("" : "+v"(v)); }

template <typename T, int NV>
__global__ __launch_bounds__(NT, 4) void k_logprobs_part(lp_args a) {
    using V = vec<T>;
    constexpr int N = V::N;
    __shared__ uint64_t sh_list[LIST];
    __shared__ lp_part sh_part[NT / 64];
    __shared__ uint64_t sh_key[NT / 64];
    __shared__ int sh_n, sh_reach;
    __shared__ float sh_thr[2][NT / 64];
    const uint32_t row = blockIdx.x / a.parts, part = blockIdx.x % a.parts;
    const T *x = (const T *)a.x + row * a.stride;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int32_t token = a.tokens ? a.tokens[row] : -1;
    const bool known = token >= 0 && (uint32_t)token < a.vocab;
    // Vectors lie on 16-byte boundaries of the address; `skew` elements of
    // the row's first are in front of it.
    const int skew = (int)((uintptr_t)x % 16 / sizeof(T));
    const int vocab = (int)a.vocab, v0 = (int)(part * a.part_vecs);
    const int v_end = min(v0 + (int)a.part_vecs, (vocab + skew + N - 1) / N);
    // All loads first, of whole vectors only (lanes without one load another's
    // and drop it), so that nothing waits between them; then the row's ends,
    // element by element.
    const int whole0 = skew ? 1 : 0, whole1 = (vocab + skew) / N;
    wm_u4 v[NV];
    if (whole1 > whole0) {
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int at = min(max(v0 + tid + i * NT, whole0), whole1 - 1);
            v[i] = __builtin_nontemporal_load((const wm_u4 *)(x + (int64_t)at * N - skew));
        }
    }
    const float xt = known ? V::one(x + token) : 0.0f;
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const int at = v0 + tid + i * NT;
        if (at < whole0 || at >= whole1 || at >= v_end) {
            v[i] = wm_u4{V::LOW, V::LOW, V::LOW, V::LOW};
            if (at < v_end) {
#pragma unroll
                for (int e = 0; e < N; e++) {
                    const int id = at * N - skew + e;
                    if (id < 0 || id >= vocab) continue;
                    const uint32_t b = V::bits(x + id), s = 16 * (e % 2);
                    if (N == 4) v[i][e] = b;
                    else v[i][e / 2] = (v[i][e / 2] & ~(0xFFFFu << s)) | b << s;
                }
            }
        }
    }
    const int rounds = (v_end - v0 + NT - 1) / NT;  // of the NV, those that hold logits
    auto maximum = [&](int n) {
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < NV; i++) {
            if (N > 4) repack(v[i]);
            if (i >= n) continue;
#pragma unroll
            for (int e = 0; e < N; e++) top = fmaxf(top, V::at(v[i], e));
        }
        return top;
    };
    auto of_all_waves = [&](float m) {
        m = lanes_max(m);
        __syncthreads();
        if (lane == 0) sh_part[wave].m = m;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < NT / 64; w++) m = fmaxf(m, sh_part[w].m);
        return m;
    };
    // The sums are relative to the maximum of the part's first round, which
    // saves a pass where no top tokens are asked for; sums that come out
    // large, whose logarithm would take the differences' digits, are formed
    // again under the part's maximum.
    const float first = maximum(1);
    float top = -INFINITY;
    if (a.top_k) {
        top = maximum(rounds);
        // The lanes' maxima in order, and two values that k of them reach: the
        // smallest of the waves' k/4-th, and the largest of their k-th (where
        // a wave holds few logits).
        const float y = sorted(top);
        const float quarter = __shfl(y, ((int)a.top_k + 3) / 4 - 1, 64), all = __shfl(y, (int)a.top_k - 1, 64);
        if (lane == 0) sh_thr[0][wave] = quarter, sh_thr[1][wave] = all;
        if (tid == 0) sh_n = 0;
    }
    float m = of_all_waves(first), thr = -INFINITY;
    if (m == -INFINITY) m = of_all_waves(a.top_k ? top : maximum(rounds));
    if (a.top_k) {
        float least = INFINITY;
#pragma unroll
        for (int w = 0; w < NT / 64; w++) thr = fmaxf(thr, sh_thr[1][w]), least = fminf(least, sh_thr[0][w]);
        thr = fmaxf(thr, least);
    }

    // Sums, and the logits before the token: x > xt, or x >= xt below its id,
    // which is x > the number before xt.  (A token at -inf or NaN: by keys.)
    const bool plain = known && xt > -INFINITY;
    const float below = xt == 0.0f ? -1.401298464e-45f : __uint_as_float(__float_as_uint(xt) + (xt > 0.0f ? -1 : 1));
    float l = 0.0f, s = 0.0f;
    int before = 0;  // of the wave
    // The exponentials' arguments in one fma, x log2 e - m log2 e; the
    // rounding of the latter is known and put back into the sums.
    auto fast = [&]() {
        const float base = m == -INFINITY ? 0.0f : m;
        const float shift = base * LOG2E, off = -__builtin_fmaf(base, LOG2E, -shift);
#pragma unroll
        for (int i = 0; i < NV; i++) {
            if (N > 4) repack(v[i]);
            if (i >= rounds) continue;
            const int id = (v0 + tid + i * NT) * N - skew;
            const float limit = id + N <= token ? below : xt;
#pragma unroll
            for (int e = 0; e < N; e++) {
                const float y = V::at(v[i], e), d = __builtin_fmaf(y, LOG2E, -shift), w = __builtin_amdgcn_exp2f(d);
                l += w;
                s = __builtin_fmaf(w, fmaxf(d, -300.0f), s);
                before += __popcll(__ballot(y > limit));
            }
            if (__ballot(id <= token && id + N > token)) {
                int same = 0;
#pragma unroll
                for (int e = 0; e < N; e++) same += id <= token && id + e < token && id + N > token && V::at(v[i], e) == xt;
                before += over_lanes((uint32_t)same, [](uint32_t a, uint32_t b) { return a + b; });
            }
        }
        s = LN2 * __builtin_fmaf(off, l, s);
        s = __builtin_fmaf(s, off * LN2, s);
        l = __builtin_fmaf(l, off * LN2, l);
    };
    fast();
    // the part's ids, for what reads them again
    const int id0 = max(v0 * N - skew, 0), id1 = min(v_end * N - skew, vocab);
    if (known && !plain) {
        const uint64_t mine = key_of(xt, token);
        before = 0;
        for (int id = id0 + tid; id < id1; id += NT) before += key_of(V::one(x + id), (uint32_t)id) > mine;
        before = over_lanes((uint32_t)before, [](uint32_t a, uint32_t b) { return a + b; });
    }
    // the logits that reach the threshold
    if (a.top_k && thr > -INFINITY && top >= thr) {
#pragma unroll
        for (int i = 0; i < NV; i++) {
            if (N > 4) repack(v[i]);
            if (i >= rounds) continue;
#pragma unroll
            for (int e = 0; e < N; e++) {
                const float y = V::at(v[i], e);
                if (y >= thr) {
                    const int n = atomicAdd(&sh_n, 1);
                    if (n < LIST) sh_list[n] = key_of(y, (uint32_t)((v0 + tid + i * NT) * N - skew + e));
                }
            }
        }
    }
    auto join_waves = [&]() {
        l = lanes_sum(l), s = lanes_sum(s);
        __syncthreads();  // sh_part's maxima are read
        if (lane == 0) sh_part[wave] = {m, l, s, before};
        __syncthreads();
        lp_part p = sh_part[0];
#pragma unroll
        for (int w = 1; w < NT / 64; w++) p.l += sh_part[w].l, p.s += sh_part[w].s, p.before += sh_part[w].before;
        return p;
    };
    lp_part p = join_waves();
    if (!(p.l <= 1e12f && fabsf(m) <= 1024.0f) && m != -INFINITY) {
        // The sums are large, or NaN, or the rounding put back is over 2^-13:
        // the same from memory, by differences to the part's maximum.
        m = -INFINITY;
        for (int id = id0 + tid; id < id1; id += NT) m = fmaxf(m, V::one(x + id));
        m = of_all_waves(m);
        const float base = m == -INFINITY ? 0.0f : m;
        l = s = 0.0f;
        for (int id = id0 + tid; id < id1; id += NT) {
            const float d = V::one(x + id) - base, w = __builtin_amdgcn_exp2f(d * LOG2E);
            l += w;
            s = __builtin_fmaf(w, fmaxf(d, -200.0f), s);
        }
        p = join_waves();
    }
    const bool whole = a.parts == 1;
    const row_end end = end_row(p);
    if (tid == 0) {
        if (whole) write_row(a, row, p, end, known, xt);
        else a.part[blockIdx.x] = p;
    }
    if (!a.top_k) return;
    auto put = [&](uint32_t i, uint64_t key) {
        if (whole) write_top(a, row, i, end, key);
        else a.keys[(uint64_t)blockIdx.x * a.top_k + i] = key;
    };
    int n = sh_n;
    bool listed = thr > -INFINITY && n <= LIST;
    if (!listed) {
        // Fewer than k lanes hold a number above -inf, or very many logits
        // are equal, as a mask leaves them: what is above the threshold, and
        // the part's first ids.  Logits at the threshold that are not listed
        // come behind those that are; if k of the listed reach it, they are it.
        __syncthreads();
        if (tid == 0) sh_n = sh_reach = 0;
        __syncthreads();
        for (int id = id0 + tid; id < id1; id += NT) {
            const float y = V::one(x + id);
            if (y > thr || id < id0 + FIRST) {
                const int at = atomicAdd(&sh_n, 1);
                if (at < LIST) sh_list[at] = key_of(y, (uint32_t)id);
                if (y >= thr) atomicAdd(&sh_reach, 1);
            }
        }
        __syncthreads();
        n = sh_n;
        listed = n <= LIST && (sh_reach >= (int)a.top_k || id1 - id0 <= FIRST);
    }
    if (listed) {
        for (int c = tid; c < n; c += NT) {
            const uint64_t mine = sh_list[c];
            uint32_t rank = 0;
#pragma unroll 8
            for (int i = 0; i < n; i++) rank += sh_list[i] > mine;
            if (rank < a.top_k) put(rank, mine);
        }
        for (uint32_t i = n + tid; i < a.top_k; i += NT) put(i, 0);  // the part has no more
        return;
    }
    // Many equal or not numbers, and not at the beginning: one more pass over
    // the part per token.
    uint64_t last = ~0ull;
    for (uint32_t k = 0; k < a.top_k; k++) {
        uint64_t best = 0;
        for (int id = id0 + tid; id < id1; id += NT) {
            const uint64_t key = key_of(V::one(x + id), (uint32_t)id);
            if (key < last && key > best) best = key;
        }
        best = lanes_max(best);
        __syncthreads();
        if (lane == 0) sh_key[wave] = best;
        __syncthreads();
        best = sh_key[0];
#pragma unroll
        for (int w = 1; w < NT / 64; w++) best = max(best, sh_key[w]);
        if (tid == 0) put(k, best);
        if (best == 0) {  // the part has no more
            for (uint32_t i = k + tid; i < a.top_k; i += NT) put(i, 0);
            return;
        }
        last = best;
    }
}

// Lane i of a wave holds the i-th of 64 keys in order; the first 64 of these
// and of another such list: the larger of a[i] and b[63 - i] are they, in an
// order that six exchanges sort.
__device__ __forceinline__ uint64_t merge64(uint64_t a, uint64_t b_reversed, int lane) {
    uint64_t v = max(a, b_reversed), o;
#define WM_MERGE(D) o = lane_xor<D>(v), v = (lane & D) ? min(v, o) : max(v, o)
    WM_MERGE(32);
    WM_MERGE(16);
    WM_MERGE(8);
    WM_MERGE(4);
    WM_MERGE(2);
    WM_MERGE(1);
#undef WM_MERGE
    return v;
}

// One workgroup per row: its parts' sums, and their lists merged.
template <typename T>
__global__ __launch_bounds__(NT) void k_logprobs_join(lp_args a) {
    __shared__ lp_part sh_part[NT / 64];
    __shared__ uint64_t sh_list[NT / 64][64];
    const uint32_t row = blockIdx.x;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int32_t token = a.tokens ? a.tokens[row] : -1;
    const bool known = token >= 0 && (uint32_t)token < a.vocab;
    const float xt = known ? vec<T>::one((const T *)a.x + row * a.stride + token) : 0.0f;
    const lp_part *part = a.part + (uint64_t)row * a.parts;
    lp_part p = {-INFINITY, 0.0f, 0.0f, 0};
    for (uint32_t i = tid; i < a.parts; i += NT) p = join_parts(p, part[i]);
    p = join_lanes<32>(p);
    if (lane == 0) sh_part[wave] = p;
    uint64_t list = 0;
    if (a.top_k) {
        // eight lists at a time, their loads ahead of the merges
        const uint64_t *keys = a.keys + (uint64_t)row * a.parts * a.top_k;
        const uint32_t j = 63 - lane;
        for (uint32_t i0 = wave; i0 < a.parts; i0 += 8 * (NT / 64)) {
            uint64_t next[8];
#pragma unroll
            for (int u = 0; u < 8; u++) {
                const uint32_t i = i0 + u * (NT / 64);
                next[u] = i < a.parts && j < a.top_k ? keys[(uint64_t)i * a.top_k + j] : 0;
            }
#pragma unroll
            for (int u = 0; u < 8; u++)
                if (i0 + u * (NT / 64) < a.parts) list = merge64(list, next[u], lane);
        }
        sh_list[wave][lane] = list;
    }
    __syncthreads();
    p = sh_part[0];
#pragma unroll
    for (int w = 1; w < NT / 64; w++) p = join_parts(p, sh_part[w]);
    const row_end end = end_row(p);
    if (tid == 0) write_row(a, row, p, end, known, xt);
    if (wave == 0 && a.top_k) {
#pragma unroll
        for (int w = 1; w < NT / 64; w++) list = merge64(list, sh_list[w][63 - lane], lane);
        if (lane < (int)a.top_k) write_top(a, row, lane, end, list);
    }
}

// The same without top tokens, of at most 16 parts: 16 lanes per row.  (Sums
// in the order of the kernel above, where the other lanes add nothing: what a
// row gives does not depend on which outputs are asked for.)
template <typename T>
__global__ __launch_bounds__(64) void k_logprobs_join_rows(lp_args a) {
    const uint32_t at = blockIdx.x * 4 + threadIdx.x / 16, i = threadIdx.x % 16, row = min(at, a.n_rows - 1);
    const int32_t token = a.tokens ? a.tokens[row] : -1;
    const bool known = token >= 0 && (uint32_t)token < a.vocab;
    lp_part p = {-INFINITY, 0.0f, 0.0f, 0};
    if (i < a.parts) p = a.part[(uint64_t)row * a.parts + i];
    const float xt = known ? vec<T>::one((const T *)a.x + row * a.stride + token) : 0.0f;
    p = join_lanes<8>(p);
    if (i == 0 && at < a.n_rows) write_row(a, row, p, end_row(p), known, xt);
}

// How a row is divided: as few parts as its lanes' registers allow, and of
// few rows parts a quarter as long.
constexpr uint32_t LONG_PART = 64 * NT, SHORT_PART = 16 * NT;  // elements, at most
// Long parts of a call up to which it takes short ones.  Long and short, f32
// rows of 128256, top 20: 8 of them 15.8 us and 12.6, 128 16.1 and 13.6, 256
// 16.4 and 15.8, 512 18.6 and 19.5, 1024 23.5 and 27.8.
constexpr uint32_t SMALL = 128;
struct lp_plan {
    bool small;
    uint32_t parts, part_vecs;
};
uint32_t most_parts(uint32_t vocab, size_t elem, uint32_t len) {
    const uint32_t per = (uint32_t)(16 / elem), vecs = (vocab + 2 * per - 2) / per;  // with any skew
    return (vecs + len / per - 1) / (len / per);
}
lp_plan make_plan(uint32_t n_rows, uint32_t vocab, size_t elem) {
    const uint32_t per = (uint32_t)(16 / elem), vecs = (vocab + 2 * per - 2) / per;  // with any skew
    lp_plan p;
    p.small = (uint64_t)n_rows * ((vocab + LONG_PART - 1) / LONG_PART) <= SMALL;
    p.parts = most_parts(vocab, elem, p.small ? SHORT_PART : LONG_PART);
    p.part_vecs = ((vecs + p.parts - 1) / p.parts + NT - 1) / NT * NT;  // of whole rounds, but for the last
    p.parts = (vecs + p.part_vecs - 1) / p.part_vecs;
    return p;
}
// Parts of a call, of any type, and of every one of fewer rows or a smaller
// vocabulary, which may take short parts where this one does not.  With c long
// parts of a row, c * n_rows <= SMALL, a row has 4 c + 1 short ones at most:
// 5 SMALL of the call.
size_t kept_parts(uint32_t n_rows, uint32_t vocab) {
    size_t n = 0;
    for (size_t elem = 2; elem <= 4; elem *= 2) {
        const size_t few = most_parts(vocab, elem, SHORT_PART), many = most_parts(vocab, elem, LONG_PART);
        if (few > 1) n = std::max(n, std::min<size_t>(n_rows * few, 5 * SMALL));
        if (many > 1) n = std::max(n, n_rows * many);
    }
    return n;
}

template <typename T>
void launch(const lp_args &a, const lp_plan &p, hipStream_t s) {
    const uint32_t grid = a.n_rows * a.parts;
    if (p.small) k_logprobs_part<T, SHORT_PART / NT / vec<T>::N><<<grid, NT, 0, s>>>(a);
    else k_logprobs_part<T, LONG_PART / NT / vec<T>::N><<<grid, NT, 0, s>>>(a);
    if (a.parts <= 1) return;
    if (!a.top_k && a.parts <= 16) k_logprobs_join_rows<T><<<(a.n_rows + 3) / 4, 64, 0, s>>>(a);
    else k_logprobs_join<T><<<a.n_rows, NT, 0, s>>>(a);
}

constexpr char who[] = "token_logprobs";
wm_status check_sizes(wm_ctx *ctx, size_t elem, uint32_t n_rows, uint32_t vocab, uint32_t top_k) {
    if (vocab == 0 || vocab > MAX_VOCAB) return wm_set_error(ctx, WM_E_SHAPE, "%s: vocabulary of %u", who, vocab);
    if ((uint64_t)n_rows * make_plan(n_rows, vocab, elem).parts > 0x7FFFFFFFu / NT)  // the launch counts threads in 32 bits
        return wm_set_error(ctx, WM_E_SHAPE, "%s: %u rows of %u", who, n_rows, vocab);
    if (top_k > MAX_TOP || top_k > vocab)
        return wm_set_error(ctx, WM_E_SHAPE, "%s: top_k %u of %u tokens, %u at most", who, top_k, vocab, MAX_TOP);
    return WM_OK;
}
wm_status check_outputs(wm_ctx *ctx, uint32_t top_k, const void *tokens, const void *logprob, const void *rank,
                        const void *top_ids, const void *top_logprobs) {
    if (!top_k && (top_ids || top_logprobs))
        return wm_set_error(ctx, WM_E_ARG, "%s: outputs for the top tokens with top_k 0", who);
    if (!tokens && (logprob || rank))
        return wm_set_error(ctx, WM_E_ARG, "%s: log probabilities or ranks of no tokens", who);
    return WM_OK;
}

}  // namespace

extern "C" {

size_t wm_token_logprobs_workspace(uint32_t n_rows, uint32_t vocab, uint32_t top_k) {
    if (n_rows == 0 || vocab == 0 || vocab > MAX_VOCAB || top_k > MAX_TOP) return 0;
    return kept_parts(n_rows, vocab) * (sizeof(lp_part) + 8 * (size_t)top_k);
}

wm_status wm_token_logprobs_dev(wm_ctx *ctx, int type, const void *d_logits, uint64_t row_stride, uint32_t n_rows,
                                uint32_t vocab, const int32_t *d_tokens, uint32_t top_k, float *d_logprob,
                                float *d_entropy, int32_t *d_rank, int32_t *d_top_ids, float *d_top_logprobs,
                                void *d_work, size_t work_bytes) {
    if (!ctx) return WM_E_ARG;
    const size_t elem = wm_dtype_size(type);
    if (!elem) return wm_set_error(ctx, WM_E_UNSUPPORTED_TYPE, "%s: type %d is not F32, F16 or BF16", who, type);
    if (wm_status st = check_sizes(ctx, elem, n_rows, vocab, top_k)) return st;
    if (n_rows > 1 && (row_stride < vocab || row_stride > 1ull << 40))
        return wm_set_error(ctx, WM_E_SHAPE, "%s: rows of %u values are %llu apart", who, vocab,
                            (unsigned long long)row_stride);
    if (wm_status st = check_outputs(ctx, top_k, d_tokens, d_logprob, d_rank, d_top_ids, d_top_logprobs)) return st;
    if (n_rows == 0) return WM_OK;
    if (!d_logits) return wm_set_error(ctx, WM_E_ARG, "%s: null logits", who);
    if ((uintptr_t)d_logits % elem ||
        ((uintptr_t)d_tokens | (uintptr_t)d_logprob | (uintptr_t)d_entropy | (uintptr_t)d_rank | (uintptr_t)d_top_ids |
         (uintptr_t)d_top_logprobs) % 4)
        return wm_set_error(ctx, WM_E_ARG, "%s: misaligned pointer", who);
    const lp_plan p = make_plan(n_rows, vocab, elem);
    const size_t need = p.parts > 1 ? wm_token_logprobs_workspace(n_rows, vocab, top_k) : 0;
    if (need && (!d_work || work_bytes < need || (uintptr_t)d_work % 16))
        return wm_set_error(ctx, WM_E_ARG, "%s: workspace of %zu bytes, %zu needed, 16-byte aligned", who,
                            d_work ? work_bytes : (size_t)0, need);
    lp_args a;
    memset(&a, 0, sizeof a);
    a.x = d_logits, a.stride = row_stride, a.n_rows = n_rows, a.vocab = vocab;
    a.top_k = d_top_ids || d_top_logprobs ? top_k : 0;
    a.tokens = d_tokens, a.logprob = d_logprob, a.entropy = d_entropy, a.rank = d_rank;
    a.top_ids = d_top_ids, a.top_logprobs = d_top_logprobs;
    a.parts = p.parts, a.part_vecs = p.part_vecs;
    a.part = (lp_part *)d_work;
    a.keys = d_work ? (uint64_t *)(a.part + (size_t)n_rows * p.parts) : nullptr;
    wm_device_guard dev(ctx->device);
    WM_HIP(ctx, dev.err);
    if (type == WM_DTYPE_F32) launch<float>(a, p, ctx->stream);
    else if (type == WM_DTYPE_F16) launch<_Float16>(a, p, ctx->stream);
    else launch<__bf16>(a, p, ctx->stream);
    WM_HIP(ctx, hipGetLastError());
    return WM_OK;
}

wm_status wm_token_logprobs(wm_ctx *ctx, const float *logits, uint32_t n_rows, uint32_t vocab, const int32_t *tokens,
                            uint32_t top_k, float *logprob, float *entropy, int32_t *rank, int32_t *top_ids,
                            float *top_logprobs) {
    if (!ctx) return WM_E_ARG;
    if (n_rows == 0 || !logits)  // the device form's words for these
        return wm_token_logprobs_dev(ctx, WM_DTYPE_F32, logits, vocab, n_rows, vocab, tokens, top_k, logprob, entropy,
                                     rank, top_ids, top_logprobs, nullptr, 0);
    // (before anything is allocated or copied)
    if (wm_status st = check_sizes(ctx, sizeof(float), n_rows, vocab, top_k)) return st;
    if (wm_status st = check_outputs(ctx, top_k, tokens, logprob, rank, top_ids, top_logprobs)) return st;
    wm_device_guard dev(ctx->device);
    WM_HIP(ctx, dev.err);
    // one block of the context's scratch: logits, tokens, outputs, workspace
    const size_t n = n_rows, word = (n * 4 + 255) & ~(size_t)255, top = (n * top_k * 4 + 255) & ~(size_t)255;
    const size_t in = (n * vocab * 4 + 255) & ~(size_t)255, ws = wm_token_logprobs_workspace(n_rows, vocab, top_k);
    void *scratch;
    if (wm_status st = wm_ctx_scratch(ctx, in + 4 * word + 2 * top + ws, &scratch)) return st;
    uint8_t *at = (uint8_t *)scratch;
    float *d_x = (float *)at;
    int32_t *d_tok = (int32_t *)(at += in);
    float *d_lp = (float *)(at += word), *d_en = (float *)(at += word);
    int32_t *d_rk = (int32_t *)(at += word), *d_ti = (int32_t *)(at += word);
    float *d_tl = (float *)(at += top);
    at += top;
    hipStream_t s = ctx->stream;
    WM_HIP(ctx, hipMemcpyAsync(d_x, logits, n * vocab * 4, hipMemcpyHostToDevice, s));
    if (tokens) WM_HIP(ctx, hipMemcpyAsync(d_tok, tokens, n * 4, hipMemcpyHostToDevice, s));
    wm_status st = wm_token_logprobs_dev(ctx, WM_DTYPE_F32, d_x, vocab, n_rows, vocab, tokens ? d_tok : nullptr, top_k,
                                         logprob ? d_lp : nullptr, entropy ? d_en : nullptr, rank ? d_rk : nullptr,
                                         top_ids ? d_ti : nullptr, top_logprobs ? d_tl : nullptr, ws ? at : nullptr, ws);
    if (st) {
        WM_HIP(ctx, hipStreamSynchronize(s));
        return st;
    }
    if (logprob) WM_HIP(ctx, hipMemcpyAsync(logprob, d_lp, n * 4, hipMemcpyDeviceToHost, s));
    if (entropy) WM_HIP(ctx, hipMemcpyAsync(entropy, d_en, n * 4, hipMemcpyDeviceToHost, s));
    if (rank) WM_HIP(ctx, hipMemcpyAsync(rank, d_rk, n * 4, hipMemcpyDeviceToHost, s));
    if (top_ids) WM_HIP(ctx, hipMemcpyAsync(top_ids, d_ti, n * top_k * 4, hipMemcpyDeviceToHost, s));
    if (top_logprobs) WM_HIP(ctx, hipMemcpyAsync(top_logprobs, d_tl, n * top_k * 4, hipMemcpyDeviceToHost, s));
    WM_HIP(ctx, hipStreamSynchronize(s));
    return WM_OK;
}

}  // extern "C"
