// Log probabilities of given tokens for gfx950, with the entropy of the distribution and its best alternatives, and the
// gradient to the logits.  Row r of the logits x, z = x * inv_temperature (rounded to fp32; the order of the alternatives
// is the order of z, equal values by the lower token):
//   m = max z,  L = log sum exp(z - m),  log p_j = (z_j - m) - L,  entropy = L - sum exp(z_j - m) (z_j - m) / sum exp(z - m)
//   d(log p_t)/dz_j = [j = t] - p_j,  d(entropy)/dz_j = -p_j (log p_j + entropy)
// A term of weight zero adds nothing to the entropy (z_j = -inf: a blocked token).
//
// Bound: reading the logits once from HBM (the gradient: reading and writing them once).  token_logprobs_f32 makes one pass:
// every lane keeps a running maximum m, l = sum exp(z - m) and u = sum exp(z - m) (z - m) of its own values, in fp32, and a
// wavefront keeps the alternatives it met as one sorted list, the i-th best in lane i.  A value and its token are one 64-bit
// integer that orders them, so the result is exact and does not depend on who was ready first.  Only values above a bound
// are looked at: the k-th largest of the maxima that 128 groups of lanes have seen so far, k values that are really there.  The
// workgroup renews it after 1, 2, 4, 8 ... tiles, so about k values per doubling of what has been read come through; each is
// found by a ballot and inserted by shifting the lanes behind it.  What is left at the end, a few more than k values, is put in
// order by counting.
// Measured: 4096 rows of 100000 tokens with 20 alternatives 267 us (6.1 TB/s; without alternatives 250 us = 6.5 TB/s, a plain
// read of as much reaches 6.6 to 6.9), 2048 rows of 50257 63 us, their gradient 130 us (6.3 TB/s read and written).
#include "common.h"

#include <algorithm>

namespace {

constexpr int MAX_TOP = 64;
constexpr int MERGE_KEYS = 1024;     // alternatives that one merge ranks
constexpr float LOG2E = 1.44269504088896340736f;
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned long long u64;

__device__ __forceinline__ float scaled(const float x, const float t) { return x * t + 0.0f; }   // + 0: the two zeros are one value
__device__ __forceinline__ float exp_fast(const float y) { return __builtin_amdgcn_exp2f(y * LOG2E); }
// With what the change of base rounds off put back (|y| <= 1e4): a far y's exponential is off by a step, not by |y| steps.
__device__ __forceinline__ float exp_near(const float y) {
    const float t = y * LOG2E, r = __builtin_fmaf(y, 1.925963033500702e-8f, __builtin_fmaf(y, LOG2E, -t));
    return __builtin_amdgcn_exp2f(t) * __builtin_fmaf(r, 0.69314718055994530942f, 1.0f);
}

// The order of the alternatives as one integer: larger value first, of equal values the lower token; NaN behind -inf.  0 is no token.
__device__ __forceinline__ u64 order_key(const float z, const unsigned token) {
    unsigned u = __float_as_uint(z);
    u = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
    if (z != z) u = 0;
    return ((u64)u << 32) | (0xFFFFFFFFu - token);
}
__device__ __forceinline__ float key_value(const u64 key) {
    const unsigned u = (unsigned)(key >> 32);
    if (u == 0) return __builtin_nanf("");
    return __uint_as_float((u & 0x80000000u) ? (u & 0x7FFFFFFFu) : ~u);
}
__device__ __forceinline__ int key_token(const u64 key) { return (int)(0xFFFFFFFFu - (unsigned)key); }

__device__ __forceinline__ u64 lane_key(const u64 key, const int lane) {
    return ((u64)(unsigned)__builtin_amdgcn_readlane((int)(key >> 32), lane) << 32) | (unsigned)__builtin_amdgcn_readlane((int)(unsigned)key, lane);
}
__device__ __forceinline__ u64 key_before(const u64 key) {       // the key of the lane before (lane 0: its own)
    const unsigned lo = (unsigned)__builtin_amdgcn_update_dpp((int)(unsigned)key, (int)(unsigned)key, 0x138, 0xF, 0xF, false);
    const unsigned hi = (unsigned)__builtin_amdgcn_update_dpp((int)(key >> 32), (int)(key >> 32), 0x138, 0xF, 0xF, false);
    return ((u64)hi << 32) | lo;
}

// Running maximum and sums of one lane, wavefront or part of a row.
struct Sums {
    float m, l, u;
};
// s with M in place of its maximum.  Far below M the weight f is zero, and the distance is held at -1e4 as it is for a token's value:
// a masked value's distance times the number of such values is past fp32's range (where it is NaN, so is f).
__device__ __forceinline__ Sums rescaled(const Sums s, const float M) {
    const float f = s.m == -INFINITY ? 0.f : exp_fast(s.m - M), d = s.m == -INFINITY ? 0.f : fmaxf(s.m - M, -1e4f);
    Sums r;
    r.m = M;
    r.l = s.m == -INFINITY ? s.l : s.l * f;
    r.u = s.m == -INFINITY ? s.u : f * (s.u + s.l * d);
    return r;
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    return v;
}

// What a row's sums and alternatives become.
struct Outputs {
    const int *targets;
    int ignore;
    float *logprobs, *entropy, *stats, *top_logprobs;
    int *top_tokens;
    int top;
};
__device__ __forceinline__ void row_results(const Outputs &o, const long long row, const float *xr, const long long n, const float t,
                                            const Sums s) {
    const float L = logf(s.l), H = L - s.u / s.l;
    if (o.targets) {
        const int g = o.targets[row];
        o.logprobs[row] = g == o.ignore ? 0.f : (g < 0 || g >= n ? __builtin_nanf("") : (scaled(xr[g], t) - s.m) - L);
    }
    if (o.entropy) o.entropy[row] = H;
    if (o.stats) { o.stats[3 * row] = s.m; o.stats[3 * row + 1] = s.l; o.stats[3 * row + 2] = H; }
}
// The `top` largest of `count` keys in LDS (0 = none) as outputs, or as keys: each is put where its rank says.  The keys are
// read in pieces of eight: the list is filled up with zeros.
__device__ __forceinline__ void rank_keys(u64 *keys, const int count, const int top, const Outputs *o, const long long row, const Sums s,
                                          u64 *to) {
    if (threadIdx.x < 8) keys[count + threadIdx.x] = 0;
    __syncthreads();
    for (int e = threadIdx.x; e < count; e += blockDim.x) {
        const u64 key = keys[e];
        if (key == 0) continue;
        int rank = 0;
        for (int j = 0; j < count; j += 8) {
#pragma unroll
            for (int i = 0; i < 8; ++i) rank += keys[j + i] > key;
        }
        if (rank >= top) continue;
        if (to) to[rank] = key;
        else {
            o->top_tokens[row * top + rank] = key_token(key);
            o->top_logprobs[row * top + rank] = (key_value(key) - s.m) - logf(s.l);
        }
    }
}

// Largest of the GS lanes (2 or 8, consecutive) that hold the lane.
template <int CTRL>
__device__ __forceinline__ float max_lanes(const float v) {
    return fmaxf(v, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xF, 0xF, true)));
}
template <int GS>
__device__ __forceinline__ float group_max(float v) {
    v = max_lanes<0xB1>(v);            // quad_perm [1,0,3,2]
    if (GS == 8) {
        v = max_lanes<0x4E>(v);        // quad_perm [2,3,0,1]
        v = max_lanes<0x141>(v);       // row_half_mirror
    }
    return v;
}
// A key below which no key of the `top` largest lies, from 128 values of different tokens (-inf: no token), two per lane: the
// upper 16 bits of the top-th largest, found bit by bit.
__device__ __forceinline__ u64 lower_bound(const float v, const float w, const int top) {
    const unsigned u = (unsigned)(order_key(v, 0) >> 32), y = (unsigned)(order_key(w, 0) >> 32);
    unsigned prefix = 0;
#pragma unroll
    for (int bit = 31; bit >= 16; --bit) {
        const unsigned with = prefix | (1u << bit);
        if (__popcll(__ballot(u >= with)) + __popcll(__ballot(y >= with)) >= top) prefix = with;
    }
    return prefix <= 0x007FFFFFu ? 0 : ((u64)prefix << 32) - 1;          // not above -inf: no bound
}

// One workgroup per row, or per part of a row (blockIdx.x); parts leave [top keys][m, l, u] in scratch for the merge.
template <int NW, bool TOP>
__global__ __launch_bounds__(NW * 64) void token_logprobs_f32(const float *__restrict__ x, const long long n, const long long stride,
                                                               const float t, const Outputs out, const int parts, u64 *partial) {
    constexpr int GS = NW / 2, GROUPS = 64 / GS;                         // groups of lanes: 128 in the workgroup
    __shared__ Sums sums[NW];
    __shared__ u64 keys[TOP ? NW * MAX_TOP + 8 : 1], bar;
    __shared__ float seen[2][TOP ? 128 : 1];
    __shared__ int kept;
    const long long row = blockIdx.y + (long long)blockIdx.z * 65535;
    const int part = blockIdx.x;
    const float *xr = x + row * stride;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (TOP && threadIdx.x == 0) { bar = 0; kept = 0; }

    // granules of 16 bytes: granule g holds elements 4 g - before .. + 3 of the row
    const int before = (int)((reinterpret_cast<uintptr_t>(xr) >> 2) & 3);
    const long long granules = (n + before + 3) / 4, share = ((granules + parts - 1) / parts + 255) / 256 * 256;
    const long long g0 = part * share, g1 = min(granules, g0 + share);
    const float *xg = xr - before;
    const int tiles = (int)((max(g1 - g0, 0ll) + 256 * NW - 1) / (256 * NW));

    // sixteen values of the lane; what lies outside the row is -inf
    auto load = [&](const long long base, f32x4 (&v)[4]) {
        if (base >= g1) {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = f32x4{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        } else if (4 * base >= before && 4 * (base + 256) - before <= n) {   // no granule is cut by the row's ends
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = __builtin_nontemporal_load(reinterpret_cast<const f32x4 *>(xg + 4 * (base + 64 * i + lane)));
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const long long j = 4 * (base + 64 * i + lane) - before + c;
                    v[i][c] = j >= 0 && j < n ? xr[j] : (t < 0.f ? INFINITY : -INFINITY);
                }
        }
    };

    Sums s = {-INFINITY, 0.f, 0.f};
    u64 list = 0, tau = 0;                                               // keys above tau are wanted
    f32x4 next[4];
    if (TOP) load(g0 + 256 * wave, next);                                // (the other form has nothing to do that would hold up its loads)
    for (int tile = 0; tile < tiles; ++tile) {
        const long long base = g0 + 256 * (wave + (long long)NW * tile);
        float z[16], mx = -INFINITY;
        if (!TOP) load(base, next);
#pragma unroll
        for (int e = 0; e < 16; ++e) z[e] = scaled(next[e >> 2][e & 3], t);
        if (base >= g1) {
#pragma unroll
            for (int e = 0; e < 16; ++e) z[e] = -INFINITY;
        }
        if (TOP) load(base + 256 * NW, next);
#pragma unroll
        for (int e = 0; e < 16; e += 2) mx = fmaxf(fmaxf(mx, z[e]), z[e + 1]);
        const float M = fmaxf(s.m, mx);
        const float mu = M == -INFINITY ? 0.f : M;
        s = rescaled(s, M);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const float y = z[e] - mu, p = exp_fast(y);
            s.l += p;
            s.u += p * fmaxf(y, -1e4f);                                      // p = 0 far below: 0 * -inf is no term
        }
        if (TOP) {
            if ((tile & (tile - 1)) == 0) {                                  // the same tiles for every wavefront
                const int turn = (tile == 0 ? 0 : __builtin_ctz(tile) + 1) & 1;
                const float gm = group_max<GS>(s.m);
                if (lane % GS == 0) seen[turn][wave * GROUPS + lane / GS] = gm;
                __syncthreads();
                const u64 low = lower_bound(seen[turn][lane], seen[turn][64 + lane], out.top);
                tau = low > tau ? low : tau;
            }
            float tau_value = (tau >> 32) == 0 ? -INFINITY : key_value(tau);
            if (__any(!(mx < tau_value)) && base < g1) {
                const u64 others = __hip_atomic_load(&bar, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
                if (others > tau) { tau = others; tau_value = key_value(tau); }
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    if (!__any(!(z[e] < tau_value))) continue;               // (a NaN passes: its key decides)
                    const long long j = 4 * (base + 64 * (e >> 2) + lane) - before + (e & 3);
                    const u64 key = j >= 0 && j < n ? order_key(z[e], (unsigned)j) : 0;
                    u64 better = __ballot(key > tau);
                    while (better) {
                        const int from = __builtin_ctzll(better);
                        const u64 add = lane_key(key, from);
                        const int pos = __popcll(__ballot(list > add));
                        const u64 shifted = key_before(list);
                        list = lane < pos ? list : (lane == pos ? add : shifted);
                        const u64 kth = lane_key(list, out.top - 1);
                        if (kth > tau) { tau = kth; tau_value = key_value(tau); }
                        better &= __ballot(key > tau) & ~(1ull << from);
                    }
                }
                if (lane == 0) __hip_atomic_fetch_max(&bar, tau, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
            }
        }
    }

    const float M = wave_max(s.m);
    s = rescaled(s, M);
    s.l = dl4s::wave_sum(s.l);
    s.u = dl4s::wave_sum(s.u);
    if (lane == 0) sums[wave] = s;
    __syncthreads();
    int count = 0;
    if (TOP) {
        // bar is at most the top-th largest key of the row: what is not below it goes on
        const bool keep = lane < out.top && list != 0 && list >= bar;
        const u64 keeping = __ballot(keep);
        int at = 0;
        if (lane == 0) at = atomicAdd(&kept, __popcll(keeping));
        at = __builtin_amdgcn_readfirstlane(at) + __popcll(keeping & ((1ull << lane) - 1));
        if (keep) keys[at] = list;
        __syncthreads();
        count = kept;
    }
    float Mall = sums[0].m;
#pragma unroll
    for (int w = 1; w < NW; ++w) Mall = fmaxf(Mall, sums[w].m);
    Sums all = rescaled(sums[0], Mall);
#pragma unroll
    for (int w = 1; w < NW; ++w) {
        const Sums r = rescaled(sums[w], Mall);
        all.l += r.l;
        all.u += r.u;
    }
    u64 *rec = parts > 1 ? partial + (row * parts + part) * (out.top + 2) : nullptr;
    if (threadIdx.x == 0) {
        if (rec) {
            float *f = reinterpret_cast<float *>(rec + out.top);
            f[0] = all.m; f[1] = all.l; f[2] = all.u;
        } else {
            row_results(out, row, xr, n, t, all);
        }
    }
    if (TOP) {
        if (rec)                       // a part may hold fewer keys than asked for
            for (int e = threadIdx.x; e < out.top; e += NW * 64) rec[e] = 0;
        rank_keys(keys, count, out.top, &out, row, all, rec);
    }
}

// Joins the parts of a row: one workgroup per row.
__global__ __launch_bounds__(256) void token_logprobs_merge_f32(const float *__restrict__ x, const long long n, const long long stride,
                                                                 const float t, const Outputs out, const int parts, const u64 *partial) {
    __shared__ u64 keys[MERGE_KEYS + 8];
    const long long row = blockIdx.x;
    const u64 *rec = partial + row * parts * (out.top + 2);
    Sums all = {-INFINITY, 0.f, 0.f};
    float M = -INFINITY;
    for (int p = 0; p < parts; ++p) M = fmaxf(M, reinterpret_cast<const float *>(rec + p * (out.top + 2) + out.top)[0]);
    for (int p = 0; p < parts; ++p) {
        const float *f = reinterpret_cast<const float *>(rec + p * (out.top + 2) + out.top);
        const Sums r = rescaled(Sums{f[0], f[1], f[2]}, M);
        all.l += r.l;
        all.u += r.u;
    }
    all.m = M;
    if (threadIdx.x == 0) row_results(out, row, x + row * stride, n, t, all);
    for (int e = threadIdx.x; e < parts * out.top; e += 256) keys[e] = rec[e / out.top * (out.top + 2) + e % out.top];
    __syncthreads();
    rank_keys(keys, parts * out.top, out.top, &out, row, all, nullptr);
}

// One workgroup per 4096 elements of a row.
__global__ __launch_bounds__(256) void token_logprobs_bwd_f32(const float *x, const long long n, const long long stride, const float t,
                                                               const int *__restrict__ targets, const int ignore,
                                                               const float *__restrict__ stats, const float *__restrict__ dlogprobs,
                                                               const float *__restrict__ dentropy, float *dx) {
    const long long row = blockIdx.y + (long long)blockIdx.z * 65535;
    const float m = stats[3 * row], l = stats[3 * row + 1], L = logf(l), inv = 1.0f / l;
    const int g = targets ? targets[row] : ignore;
    const float gl = (dlogprobs && g != ignore) ? (g < 0 || g >= n ? __builtin_nanf("") : dlogprobs[row]) : 0.f;
    // (the entropy enters only where it has a gradient: zero times what may stand there is not always zero)
    const float ge = dentropy ? dentropy[row] : 0.f, H = ge == 0.f ? 0.f : stats[3 * row + 2];
    const float *xr = x + row * stride;
    float *dr = dx + row * stride;
    // A row that no gradient reaches gets zeros, whatever stands in it (padding: an ignored target, tokens that are all blocked).
    const bool none = gl == 0.f && ge == 0.f;
    auto gradient = [&](const float v, const long long j) {
        if (none) return 0.f;
        float y = scaled(v, t) - m;
        y = y < -1e4f ? -1e4f : y;                                     // (a NaN stays)
        // (not from log p: the subtraction of L rounds by as much as a far z)
        float r = -(exp_near(y) * inv) * (gl + ge * ((y - L) + H));
        if (j == g) r += gl;
        return r * t;
    };
    const int before = (int)((reinterpret_cast<uintptr_t>(xr) >> 2) & 3);
    const bool alike = ((reinterpret_cast<uintptr_t>(dr) ^ reinterpret_cast<uintptr_t>(xr)) & 15) == 0;
    const long long base = (long long)blockIdx.x * 1024;
    if (alike && 4 * base >= before && 4 * (base + 1024) - before <= n) {
        f32x4 v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = __builtin_nontemporal_load(reinterpret_cast<const f32x4 *>(xr - before + 4 * (base + 256 * i + threadIdx.x)));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const long long j = 4 * (base + 256 * i + threadIdx.x) - before;
#pragma unroll
            for (int c = 0; c < 4; ++c) v[i][c] = gradient(v[i][c], j + c);
            __builtin_nontemporal_store(v[i], reinterpret_cast<f32x4 *>(dr + j));
        }
    } else {
        for (int i = 0; i < 16; ++i) {
            const long long j = 4 * base - before + 256 * i + threadIdx.x;
            if (j >= 0 && j < n) dr[j] = gradient(xr[j], j);
        }
    }
}

int logprob_checks(const char *what, int64_t rows, int64_t n, int64_t stride, const float *logits, float t) {
    DL4S_REQUIRE(rows >= 0 && n >= 0, DL4S_HIP_EINVALID_ARG, "%s: negative extent", what);
    if (rows == 0) return DL4S_HIP_OK;
    DL4S_REQUIRE(logits, DL4S_HIP_EINVALID_ARG, "%s: NULL logits", what);
    DL4S_REQUIRE(n >= 1 && n < (int64_t(1) << 31) && rows < (int64_t(1) << 31), DL4S_HIP_EUNSUPPORTED,
                 "%s: %lld rows of %lld tokens (rows of 1 to 2^31 - 1 tokens are implemented)", what, (long long)rows, (long long)n);
    DL4S_REQUIRE(t > 0.f || t < 0.f, DL4S_HIP_EINVALID_ARG, "%s: inv_temperature %g (it may not be zero)", what, (double)t);
    DL4S_REQUIRE(stride >= n, DL4S_HIP_ESHAPE, "%s: rows of %lld tokens every %lld floats", what, (long long)n, (long long)stride);
    return DL4S_HIP_OK;
}

// Rows on the grid's second and third axis (65535 at most on the second).  The caller splits launches of partly filled layers.
template <typename F>
int over_rows(int64_t rows, F launch) {
    const int64_t whole = rows / 65535 * 65535;
    if (whole) {
        const int rc = launch(int64_t(0), dim3(0, 65535, (unsigned)(whole / 65535)));
        if (rc) return rc;
    }
    return rows > whole ? launch(whole, dim3(0, (unsigned)(rows - whole), 1)) : DL4S_HIP_OK;
}

}  // namespace

extern "C" {

int dl4s_hip_token_logprobs_f32(dl4s_hip_ctx *ctx, const float *logits, int64_t rows, int64_t n, int64_t row_stride,
                                float inv_temperature, const int32_t *targets, int32_t ignore_index, float *logprobs, float *entropy,
                                float *stats, int64_t top_k, float *top_logprobs, int32_t *top_tokens) {
    DL4S_CHECK_CTX(ctx);
    int rc = logprob_checks("token_logprobs", rows, n, row_stride, logits, inv_temperature);
    if (rc || rows == 0) return rc;
    DL4S_REQUIRE((targets != nullptr) == (logprobs != nullptr), DL4S_HIP_EINVALID_ARG,
                 "token_logprobs: targets and logprobs come together");
    DL4S_REQUIRE(top_k >= 0 && top_k <= MAX_TOP, DL4S_HIP_EUNSUPPORTED, "token_logprobs: %lld alternatives (up to %d are implemented)",
                 (long long)top_k, MAX_TOP);
    DL4S_REQUIRE(top_k <= n, DL4S_HIP_ESHAPE, "token_logprobs: %lld alternatives of %lld tokens", (long long)top_k, (long long)n);
    DL4S_REQUIRE(top_k == 0 || (top_logprobs && top_tokens), DL4S_HIP_EINVALID_ARG, "token_logprobs: NULL output for the alternatives");
    // 16 wavefronts to a row up to one row to a compute unit, otherwise four (256 rows of 50000 tokens 10.9 us and 16.1, with 8
    // alternatives 19.4 and 29.9; 1000 rows of 5000 tokens 11.1 us and 6.7, with 8 alternatives 27.7 and 13.5: the renewed bound
    // has the wavefronts wait for each other).  Then long rows come in parts, too, of at least 16384 tokens, a tile for each
    // wavefront (8 rows of 150000 tokens 9.5 us, in one part 17.2, in parts of 4096 11.9).
    const bool few = rows <= ctx->cu_count;
    int64_t parts = 1;
    if (few) {
        parts = std::min<int64_t>(n / 16384, ctx->cu_count / rows);
        parts = std::min<int64_t>(parts, top_k ? MERGE_KEYS / top_k : 64);
        parts = std::max<int64_t>(parts, 1);
    }
    std::unique_lock<std::mutex> scratch_lock(ctx->scratch_mu, std::defer_lock);
    u64 *partial = nullptr;
    if (parts > 1) {
        scratch_lock.lock();
        rc = dl4s::ensure_scratch(ctx, (size_t)rows * parts * (top_k + 2) * sizeof(u64));
        if (rc) return rc;
        partial = reinterpret_cast<u64 *>(ctx->scratch);
    }
    rc = over_rows(rows, [&](const int64_t from, dim3 grid) {
        grid.x = (unsigned)parts;
        const Outputs out = {targets ? targets + from : nullptr, ignore_index, logprobs ? logprobs + from : nullptr,
                             entropy ? entropy + from : nullptr, stats ? stats + 3 * from : nullptr,
                             top_k ? top_logprobs + from * top_k : nullptr, top_k ? top_tokens + from * top_k : nullptr, (int)top_k};
        const float *x = logits + from * row_stride;
#define DL4S_LOGPROBS(NW, TOP)                                                                                                     \
    hipLaunchKernelGGL((token_logprobs_f32<NW, TOP>), grid, dim3(NW * 64), 0, ctx->stream, x, (long long)n, (long long)row_stride, \
                       inv_temperature, out, (int)parts, partial)
        if (few && top_k) DL4S_LOGPROBS(16, true);
        else if (few) DL4S_LOGPROBS(16, false);
        else if (top_k) DL4S_LOGPROBS(4, true);
        else DL4S_LOGPROBS(4, false);
#undef DL4S_LOGPROBS
        return dl4s::launch_status("token_logprobs_f32");
    });
    if (rc || parts == 1) return rc;
    const Outputs out = {targets, ignore_index, logprobs, entropy, stats, top_logprobs, top_tokens, (int)top_k};
    hipLaunchKernelGGL(token_logprobs_merge_f32, dim3((unsigned)rows), dim3(256), 0, ctx->stream, logits, (long long)n, (long long)row_stride,
                       inv_temperature, out, (int)parts, (const u64 *)partial);
    return dl4s::launch_status("token_logprobs_merge_f32");
}

int dl4s_hip_token_logprobs_bwd_f32(dl4s_hip_ctx *ctx, const float *logits, int64_t rows, int64_t n, int64_t row_stride,
                                    float inv_temperature, const int32_t *targets, int32_t ignore_index, const float *stats,
                                    const float *dlogprobs, const float *dentropy, float *dlogits) {
    DL4S_CHECK_CTX(ctx);
    const int rc = logprob_checks("token_logprobs_bwd", rows, n, row_stride, logits, inv_temperature);
    if (rc || rows == 0) return rc;
    DL4S_REQUIRE(stats && dlogits, DL4S_HIP_EINVALID_ARG, "token_logprobs_bwd: NULL pointer");
    DL4S_REQUIRE(!dlogprobs || targets, DL4S_HIP_EINVALID_ARG, "token_logprobs_bwd: a gradient of the log probabilities without targets");
    return over_rows(rows, [&](const int64_t from, dim3 grid) {
        grid.x = (unsigned)((n + 3 + 4095) / 4096);                    // (up to three elements of the first granule lie before the row)
        hipLaunchKernelGGL(token_logprobs_bwd_f32, grid, dim3(256), 0, ctx->stream, logits + from * row_stride, (long long)n,
                           (long long)row_stride, inv_temperature, targets ? targets + from : nullptr, ignore_index, stats + 3 * from,
                           dlogprobs ? dlogprobs + from : nullptr, dentropy ? dentropy + from : nullptr, dlogits + from * row_stride);
        return dl4s::launch_status("token_logprobs_bwd_f32");
    });
}

}  // extern "C"
