// Log probabilities of given tokens, the entropy of their distribution, the
// token's rank and the top alternatives, per row of logits.
#include <cstdio>
#include <cstring>

#include "wm_paged.h"

namespace {

constexpr int NT = 1024;
constexpr uint32_t MAX_TOP = 64;

struct lp_args {
    const void *x;
    uint64_t stride;
    uint32_t n_rows, vocab, top_k;
    const int32_t *tokens;
    float *logprob, *entropy;
    int32_t *rank, *top_ids;
    float *top_logprobs;
};

// Order of (logit descending, id): the larger key comes first.  Zeros are
// one value; NaN is below every number.
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return x != x ? 0u : b ^ ((int)b < 0 ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ uint64_t key_of(float x, uint32_t id) { return (uint64_t)ordered(x) << 32 | ~id; }
__device__ __forceinline__ float key_value(uint64_t key) {
    const uint32_t o = (uint32_t)(key >> 32);
    return o == 0 ? __uint_as_float(0x7FC00000u) : __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o);
}

// Sum of e^(x - m) and of e^(x - m) (x - m) under the running maximum m.
struct stats {
    float m, l, s;
};
__device__ __forceinline__ void add(stats &a, float x) {
    if (x > a.m) {
        const float d = a.m - x, e = expf(d);
        a.s = e * (a.s + a.l * fmaxf(d, -200.0f));
        a.l *= e;
        a.m = x;
    }
    const float d = a.m == -INFINITY ? x : x - a.m, e = expf(d);
    a.l += e;
    a.s += e * fmaxf(d, -200.0f);
}
__device__ __forceinline__ stats join(stats a, stats b) {
    const float m = fmaxf(a.m, b.m), base = m == -INFINITY ? 0.0f : m;
    const float da = a.m - base, db = b.m - base, ea = expf(da), eb = expf(db);
    return {m, a.l * ea + b.l * eb,
            ea * (a.s + a.l * fmaxf(da, -200.0f)) + eb * (b.s + b.l * fmaxf(db, -200.0f))};
}
__device__ __forceinline__ float read(const float *x, uint64_t i) { return x[i]; }
__device__ __forceinline__ float read(const _Float16 *x, uint64_t i) { return (float)x[i]; }
__device__ __forceinline__ float read(const __bf16 *x, uint64_t i) { return (float)x[i]; }

__device__ __forceinline__ uint64_t shfl_xor64(uint64_t v, int o) {
    return (uint64_t)__shfl_xor((int)(v >> 32), o, 64) << 32 | (uint32_t)__shfl_xor((int)v, o, 64);
}

template <typename T>
__global__ __launch_bounds__(NT) void k_token_logprobs(lp_args a) {
    __shared__ stats sh[NT / 64];
    __shared__ uint64_t sh_key[NT / 64];
    __shared__ int sh_n[NT / 64];
    const T *x = (const T *)a.x + blockIdx.x * a.stride;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int32_t token = a.tokens ? a.tokens[blockIdx.x] : -1;
    const bool known = token >= 0 && (uint32_t)token < a.vocab;
    const uint64_t mine = known ? key_of(read(x, token), token) : 0;
    stats st = {-INFINITY, 0.0f, 0.0f};
    int before = 0;
    for (uint64_t i = tid; i < a.vocab; i += NT) {
        const float v = read(x, i);
        add(st, v);
        before += key_of(v, (uint32_t)i) > mine;
    }
    for (int o = 32; o; o >>= 1) {
        st = join(st, stats{__shfl_xor(st.m, o, 64), __shfl_xor(st.l, o, 64), __shfl_xor(st.s, o, 64)});
        before += __shfl_xor(before, o, 64);
    }
    if (lane == 0) sh[wave] = st, sh_n[wave] = before;
    __syncthreads();
    st = sh[0], before = sh_n[0];
    for (int w = 1; w < NT / 64; w++) st = join(st, sh[w]), before += sh_n[w];
    const float log_l = logf(st.l);
    auto logprob = [&](float v) {
        // every logit -inf: its sum is 0 (log -inf), which only takes NaN or
        // +inf to leave NaN
        return st.m == -INFINITY && st.l == 0.0f ? v : (v - st.m) - log_l;
    };
    if (tid == 0) {
        const bool none = st.m == -INFINITY && st.l == 0.0f;
        if (a.logprob) a.logprob[blockIdx.x] = known ? logprob(read(x, token)) : __uint_as_float(0x7FC00000u);
        if (a.entropy) a.entropy[blockIdx.x] = none ? 0.0f : log_l - st.s / st.l;
        if (a.rank) a.rank[blockIdx.x] = known ? before : -1;
    }
    uint64_t last = ~0ull;
    for (uint32_t k = 0; k < a.top_k; k++) {
        uint64_t best = 0;
        for (uint64_t i = tid; i < a.vocab; i += NT) {
            const uint64_t key = key_of(read(x, i), (uint32_t)i);
            if (key < last && key > best) best = key;
        }
        for (int o = 32; o; o >>= 1) best = max(best, shfl_xor64(best, o));
        __syncthreads();
        if (lane == 0) sh_key[wave] = best;
        __syncthreads();
        best = sh_key[0];
        for (int w = 1; w < NT / 64; w++) best = max(best, sh_key[w]);
        last = best;
        if (tid == 0) {
            const uint64_t at = (uint64_t)blockIdx.x * a.top_k + k;
            if (a.top_ids) a.top_ids[at] = (int32_t)~(uint32_t)best;
            if (a.top_logprobs) a.top_logprobs[at] = logprob(key_value(best));
        }
    }
}

}  // namespace

extern "C" {

size_t wm_token_logprobs_workspace(uint32_t n_rows, uint32_t vocab, uint32_t top_k) {
    (void)n_rows, (void)vocab, (void)top_k;
    return 0;
}

wm_status wm_token_logprobs_dev(wm_ctx *ctx, int type, const void *d_logits, uint64_t row_stride, uint32_t n_rows,
                                uint32_t vocab, const int32_t *d_tokens, uint32_t top_k, float *d_logprob,
                                float *d_entropy, int32_t *d_rank, int32_t *d_top_ids, float *d_top_logprobs,
                                void *d_work, size_t work_bytes) {
    static const char who[] = "token_logprobs";
    if (!ctx) return WM_E_ARG;
    const size_t elem = wm_dtype_size(type);
    if (!elem) return wm_set_error(ctx, WM_E_UNSUPPORTED_TYPE, "%s: type %d is not F32, F16 or BF16", who, type);
    if (vocab == 0 || vocab > 0x7FFFFFFFu) return wm_set_error(ctx, WM_E_SHAPE, "%s: vocabulary of %u", who, vocab);
    if (n_rows > 0x7FFFFFFFu / NT) return wm_set_error(ctx, WM_E_SHAPE, "%s: %u rows", who, n_rows);
    if (top_k > MAX_TOP || top_k > vocab)
        return wm_set_error(ctx, WM_E_SHAPE, "%s: top_k %u of %u tokens, %u at most", who, top_k, vocab, MAX_TOP);
    if (n_rows > 1 && (row_stride < vocab || row_stride > 1ull << 40))
        return wm_set_error(ctx, WM_E_SHAPE, "%s: rows of %u values are %llu apart", who, vocab,
                            (unsigned long long)row_stride);
    if (!top_k && (d_top_ids || d_top_logprobs))
        return wm_set_error(ctx, WM_E_ARG, "%s: outputs for the top tokens with top_k 0", who);
    if (!d_tokens && (d_logprob || d_rank))
        return wm_set_error(ctx, WM_E_ARG, "%s: log probabilities or ranks of no tokens", who);
    if (n_rows == 0) return WM_OK;
    if (!d_logits) return wm_set_error(ctx, WM_E_ARG, "%s: null logits", who);
    if ((uintptr_t)d_logits % elem ||
        ((uintptr_t)d_tokens | (uintptr_t)d_logprob | (uintptr_t)d_entropy | (uintptr_t)d_rank | (uintptr_t)d_top_ids |
         (uintptr_t)d_top_logprobs) % 4)
        return wm_set_error(ctx, WM_E_ARG, "%s: misaligned pointer", who);
    const size_t need = wm_token_logprobs_workspace(n_rows, vocab, top_k);
    if (need && (!d_work || work_bytes < need || (uintptr_t)d_work % 16))
        return wm_set_error(ctx, WM_E_ARG, "%s: workspace of %zu bytes, %zu needed, 16-byte aligned", who,
                            d_work ? work_bytes : (size_t)0, need);
    lp_args a{d_logits, row_stride, n_rows, vocab, top_k, d_tokens, d_logprob, d_entropy, d_rank, d_top_ids, d_top_logprobs};
    if (!d_top_ids && !d_top_logprobs) a.top_k = 0;
    wm_device_guard dev(ctx->device);
    WM_HIP(ctx, dev.err);
    if (type == WM_DTYPE_F32) k_token_logprobs<float><<<n_rows, NT, 0, ctx->stream>>>(a);
    else if (type == WM_DTYPE_F16) k_token_logprobs<_Float16><<<n_rows, NT, 0, ctx->stream>>>(a);
    else k_token_logprobs<__bf16><<<n_rows, NT, 0, ctx->stream>>>(a);
    WM_HIP(ctx, hipGetLastError());
    return WM_OK;
}

wm_status wm_token_logprobs(wm_ctx *ctx, const float *logits, uint32_t n_rows, uint32_t vocab, const int32_t *tokens,
                            uint32_t top_k, float *logprob, float *entropy, int32_t *rank, int32_t *top_ids,
                            float *top_logprobs) {
    static const char who[] = "token_logprobs";
    if (!ctx) return WM_E_ARG;
    if (n_rows == 0 || vocab == 0 || !logits)  // the device form's words for these
        return wm_token_logprobs_dev(ctx, WM_DTYPE_F32, logits, vocab, n_rows, vocab, tokens, top_k, logprob, entropy,
                                     rank, top_ids, top_logprobs, nullptr, 0);
    if (top_k > MAX_TOP) return wm_set_error(ctx, WM_E_SHAPE, "%s: top_k %u, %u at most", who, top_k, MAX_TOP);
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
