// Log probabilities of given tokens for gfx950, with the entropy of the distribution and its best alternatives, and the
// gradient to the logits.  Row r of the logits x, z = x * inv_temperature (rounded to fp32; the order of the alternatives
// is the order of z, equal values by the lower token):
//   m = max z,  L = log sum exp(z - m),  log p_j = (z_j - m) - L,  entropy = L - sum exp(z_j - m) (z_j - m) / sum exp(z - m)
//   d(log p_t)/dz_j = [j = t] - p_j,  d(entropy)/dz_j = -p_j (log p_j + entropy)
// A term of weight zero adds nothing to the entropy (z_j = -inf: a blocked token).
#include "common.h"

namespace {

constexpr int MAX_TOP = 64;

__device__ __forceinline__ float scaled(const float x, const float t) { return x * t + 0.0f; }   // + 0: the two zeros are one value

// The order of the alternatives as one integer: larger value first, of equal values the lower token; NaN behind -inf.
__device__ __forceinline__ unsigned long long order_key(const float z, const unsigned token) {
    unsigned u = __float_as_uint(z);
    u = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
    if (z != z) u = 0;
    return ((unsigned long long)u << 32) | (0xFFFFFFFFu - token);
}

__device__ __forceinline__ float block_reduce(float v, float *sm, const bool max) {
    for (int o = 32; o; o >>= 1) {
        const float w = __shfl_xor(v, o, 64);
        v = max ? fmaxf(v, w) : v + w;
    }
    if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = v;
    __syncthreads();
    v = sm[0];
    for (int w = 1; w < 4; ++w) v = max ? fmaxf(v, sm[w]) : v + sm[w];
    __syncthreads();
    return v;
}

// One workgroup per row: maximum, sums, then the alternatives one by one (the largest key below the last one).
__global__ __launch_bounds__(256) void token_logprobs_f32(const float *__restrict__ x, long long n, long long stride, float t,
                                                           const int *__restrict__ targets, int ignore, float *__restrict__ logprobs,
                                                           float *__restrict__ entropy, float *__restrict__ stats, int top,
                                                           float *__restrict__ top_logprobs, int *__restrict__ top_tokens) {
    __shared__ float sm[4];
    __shared__ unsigned long long sk[4];
    const long long row = blockIdx.x;
    const float *xr = x + row * stride;
    const int tid = threadIdx.x;
    float m = -INFINITY;
    bool nan = false;
    for (long long j = tid; j < n; j += 256) { const float z = scaled(xr[j], t); m = fmaxf(m, z); nan |= z != z; }
    m = block_reduce(m, sm, true);
    if (__syncthreads_or(nan)) m = __builtin_nanf("");
    float l = 0.f, u = 0.f;
    for (long long j = tid; j < n; j += 256) {
        const float y = scaled(xr[j], t) - m, e = expf(y);
        l += e;
        if (e != 0.f) u += e * y;
    }
    l = block_reduce(l, sm, false);
    u = block_reduce(u, sm, false);
    const float L = logf(l), H = L - u / l;
    if (tid == 0) {
        if (targets && logprobs) {
            const int g = targets[row];
            logprobs[row] = g == ignore ? 0.f : (g < 0 || g >= n ? __builtin_nanf("") : (scaled(xr[g], t) - m) - L);
        }
        if (entropy) entropy[row] = H;
        if (stats) { stats[3 * row] = m; stats[3 * row + 1] = L; stats[3 * row + 2] = H; }
    }
    unsigned long long below = ~0ull;
    for (int i = 0; i < top; ++i) {
        unsigned long long best = 0;
        for (long long j = tid; j < n; j += 256) {
            const unsigned long long key = order_key(scaled(xr[j], t), (unsigned)j);
            if (key < below && key > best) best = key;
        }
        for (int o = 32; o; o >>= 1) { const unsigned long long w = __shfl_xor(best, o, 64); best = w > best ? w : best; }
        if ((tid & 63) == 0) sk[tid >> 6] = best;
        __syncthreads();
        for (int w = 0; w < 4; ++w) best = sk[w] > best ? sk[w] : best;
        __syncthreads();
        if (tid == 0) {
            const unsigned token = 0xFFFFFFFFu - (unsigned)best;
            top_tokens[row * top + i] = (int)token;
            top_logprobs[row * top + i] = (scaled(xr[token], t) - m) - L;
        }
        below = best;
    }
}

__global__ __launch_bounds__(256) void token_logprobs_bwd_f32(const float *x, long long n, long long stride, float t,
                                                               const int *__restrict__ targets, int ignore,
                                                               const float *__restrict__ stats, const float *__restrict__ dlogprobs,
                                                               const float *__restrict__ dentropy, float *dx) {
    const long long row = blockIdx.x;
    const float m = stats[3 * row], L = stats[3 * row + 1], H = stats[3 * row + 2];
    const int g = targets ? targets[row] : ignore;
    const float gl = (dlogprobs && g != ignore) ? (g < 0 || g >= n ? __builtin_nanf("") : dlogprobs[row]) : 0.f;
    const float ge = dentropy ? dentropy[row] : 0.f;
    for (long long j = threadIdx.x; j < n; j += 256) {
        const float lp = (scaled(x[row * stride + j], t) - m) - L, p = expf(lp);
        float r = -p * gl;
        if (p != 0.f) r -= ge * p * (lp + H);
        if (j == g) r += gl;
        dx[row * stride + j] = r * t;
    }
}

int logprob_checks(const char *what, int64_t rows, int64_t n, int64_t stride, const float *logits) {
    DL4S_REQUIRE(rows >= 0 && n >= 0, DL4S_HIP_EINVALID_ARG, "%s: negative extent", what);
    if (rows == 0) return DL4S_HIP_OK;
    DL4S_REQUIRE(logits, DL4S_HIP_EINVALID_ARG, "%s: NULL logits", what);
    DL4S_REQUIRE(n >= 1 && n < (int64_t(1) << 31) && rows < (int64_t(1) << 31), DL4S_HIP_EUNSUPPORTED,
                 "%s: %lld rows of %lld tokens (rows of 1 to 2^31 - 1 tokens are implemented)", what, (long long)rows, (long long)n);
    DL4S_REQUIRE(stride >= n, DL4S_HIP_ESHAPE, "%s: rows of %lld tokens every %lld floats", what, (long long)n, (long long)stride);
    return DL4S_HIP_OK;
}

}  // namespace

extern "C" {

int dl4s_hip_token_logprobs_f32(dl4s_hip_ctx *ctx, const float *logits, int64_t rows, int64_t n, int64_t row_stride,
                                float inv_temperature, const int32_t *targets, int32_t ignore_index, float *logprobs, float *entropy,
                                float *stats, int64_t top_k, float *top_logprobs, int32_t *top_tokens) {
    DL4S_CHECK_CTX(ctx);
    const int rc = logprob_checks("token_logprobs", rows, n, row_stride, logits);
    if (rc || rows == 0) return rc;
    DL4S_REQUIRE((targets != nullptr) == (logprobs != nullptr), DL4S_HIP_EINVALID_ARG,
                 "token_logprobs: targets and logprobs come together");
    DL4S_REQUIRE(top_k >= 0 && top_k <= MAX_TOP, DL4S_HIP_EUNSUPPORTED, "token_logprobs: %lld alternatives (up to %d are implemented)",
                 (long long)top_k, MAX_TOP);
    DL4S_REQUIRE(top_k <= n, DL4S_HIP_ESHAPE, "token_logprobs: %lld alternatives of %lld tokens", (long long)top_k, (long long)n);
    DL4S_REQUIRE(top_k == 0 || (top_logprobs && top_tokens), DL4S_HIP_EINVALID_ARG, "token_logprobs: NULL output for the alternatives");
    hipLaunchKernelGGL(token_logprobs_f32, dim3((unsigned)rows), dim3(256), 0, ctx->stream, logits, (long long)n, (long long)row_stride,
                       inv_temperature, targets, ignore_index, logprobs, entropy, stats, (int)top_k, top_logprobs, top_tokens);
    return dl4s::launch_status("token_logprobs_f32");
}

int dl4s_hip_token_logprobs_bwd_f32(dl4s_hip_ctx *ctx, const float *logits, int64_t rows, int64_t n, int64_t row_stride,
                                    float inv_temperature, const int32_t *targets, int32_t ignore_index, const float *stats,
                                    const float *dlogprobs, const float *dentropy, float *dlogits) {
    DL4S_CHECK_CTX(ctx);
    const int rc = logprob_checks("token_logprobs_bwd", rows, n, row_stride, logits);
    if (rc || rows == 0) return rc;
    DL4S_REQUIRE(stats && dlogits, DL4S_HIP_EINVALID_ARG, "token_logprobs_bwd: NULL pointer");
    DL4S_REQUIRE(!dlogprobs || targets, DL4S_HIP_EINVALID_ARG, "token_logprobs_bwd: a gradient of the log probabilities without targets");
    hipLaunchKernelGGL(token_logprobs_bwd_f32, dim3((unsigned)rows), dim3(256), 0, ctx->stream, logits, (long long)n,
                       (long long)row_stride, inv_temperature, targets, ignore_index, stats, dlogprobs, dentropy, dlogits);
    return dl4s::launch_status("token_logprobs_bwd_f32");
}

}  // extern "C"
