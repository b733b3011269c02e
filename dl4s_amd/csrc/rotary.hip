// Rotary positions for gfx950: pairs of columns of every query and key head turn by an angle that grows with the token's
// position, pair i by turns[i] full turns per position:
//   y_a = amplitude (x_a cos - x_b sin),  y_b = amplitude (x_a sin + x_b cos),  angle = 2 pi frac(position * turns[i])
// with (a, b) = (i, i + rot/2) or, interleaved, (2i, 2i + 1); columns from rot on are copied.  The inverse turns by the
// negative angle: it is the transposed map, so it is also the gradient.
//
// Bound: HBM, every element read and written once.  A workgroup takes a few tokens: it forms their cosines and sines once
// (64-bit reduction, one angle per pair and token) in LDS, then turns all query and key heads of those tokens, and in the
// appending form copies the values, in pieces of four columns (eight with the partner columns of the half layout).
// Measured: 2 x 8192 tokens, 32 + 8 heads of 128 columns, 64 of them turned: 131 us with inputs that change from call to call (5.1
// TB/s; a copy of 2 GiB reaches 5.4); appending 16 tokens of 16 + 16 heads of 64: 4.1 us, a launch.
#include "common.h"

#include <algorithm>

#include <cmath>

namespace {

// cos and sin of turns * position turns.  The whole turns and quarters are taken off in 64 bits, where a far position's
// product still has its fraction; what is left, at most an eighth of a turn, goes through the Taylor series (next terms
// x^11 / 11! and x^12 / 12!: below 2^-28 at an eighth of a turn).
__device__ __forceinline__ void turn(const double turns, const long long position, float &c, float &s) {
    double t = turns * (double)position;
    t -= floor(t);
    const double quarters = rint(4.0 * t);
    const float x = (float)((t - 0.25 * quarters) * 6.283185307179586476925286766559), z = x * x;
    const float sn = x + x * z * (-1.0f / 6 + z * (1.0f / 120 + z * (-1.0f / 5040 + z * (1.0f / 362880))));
    const float cs = 1.0f + z * (-0.5f + z * (1.0f / 24 + z * (-1.0f / 720 + z * (1.0f / 40320 + z * (-1.0f / 3628800)))));
    const int k = (int)quarters & 3;
    const float a = k & 1 ? sn : cs, b = k & 1 ? cs : sn;
    c = (k == 1 || k == 2) ? -a : a;
    s = k >= 2 ? -b : b;
}

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

struct RotaryArgs {
    int B, L, H, Hkv, d, rot;
    const double *turns;
    const int *positions;      // rotary: [B, L]; append: [B]; or NULL
    long long position0;
    const int *counts;         // append: new rows of each batch element, or NULL
    float amplitude;
    int interleaved, inverse, token_major;
    long long Tcap;            // append only
    int tokens, per_wg;        // B * L, tokens of a workgroup
};

__device__ __forceinline__ long long element(const RotaryArgs &a, const int heads, const int b, const int l, const int h) {
    return a.token_major ? (((long long)b * a.L + l) * heads + h) * a.d : (((long long)b * heads + h) * a.L + l) * a.d;
}

// VEC: pieces of four columns (d and rot multiples of 4, in the half layout rot a multiple of 8, rows on 16 bytes); otherwise a
// piece is one pair, or one column that is copied.
template <bool APPEND, bool VEC>
__global__ __launch_bounds__(256) void rotary_f32(const float *q, float *q_out, const float *k, float *k_out, const float *v,
                                                   float *v_out, const RotaryArgs a) {
    extern __shared__ __align__(16) f32x2 rotary_lds[];                    // [token][pair] cosine, sine
    const int half = a.rot / 2, t0 = blockIdx.x * a.per_wg, nt = min(a.per_wg, a.tokens - t0);
    auto position = [&](const int t) -> long long {                        // of token t = b L + l
        if (!a.positions) return a.position0 + t % a.L;
        return APPEND ? (long long)a.positions[t / a.L] + t % a.L : a.positions[t];
    };
    for (int e = threadIdx.x; e < nt * half; e += 256) {
        float c, s;
        turn(a.turns[e % half], position(t0 + e / half), c, s);
        rotary_lds[e] = f32x2{c * a.amplitude, a.inverse ? -s * a.amplitude : s * a.amplitude};
    }
    __syncthreads();
    // pieces of a head: those that turn, then those that are copied; of a token: the heads', then (append) the values'
    const int turned = VEC ? (a.interleaved ? a.rot / 4 : a.rot / 8) : half;
    const int piece = turned + (VEC ? (a.d - a.rot) / 4 : a.d - a.rot), values = APPEND ? (VEC ? a.d / 4 : a.d) : 0;
    const int turning = (a.H + a.Hkv) * piece, all = turning + a.Hkv * values;
    const bool in_place = !APPEND && q == q_out && k == k_out;
    for (int e = threadIdx.x; e < nt * all; e += 256) {
        // head-major tensors: the tokens of one head lie together, so they are the inner index over a head's pieces
        int tt, i, h;
        bool value = false;
        if (a.token_major) {
            tt = e / all;
            i = e % all;
            if (APPEND && i >= turning) { value = true; i -= turning; h = a.H + i / values; i %= values; }
            else { h = i / piece; i %= piece; }
        } else {
            i = e;
            if (APPEND && i >= nt * turning) { value = true; i -= nt * turning; h = a.H + i / (nt * values); i %= nt * values; tt = i / values; i %= values; }
            else { h = i / (nt * piece); i %= nt * piece; tt = i / piece; i %= piece; }
        }
        const int t = t0 + tt, b = t / a.L, l = t % a.L;
        const bool key = h >= a.H;
        const int hh = key ? h - a.H : h;
        const long long at = element(a, key ? a.Hkv : a.H, b, l, hh);
        long long to = at;
        if (APPEND && key) {
            const long long pos = position(t);
            if (pos < 0 || pos >= a.Tcap || (a.counts && l >= a.counts[b])) continue;
            to = (((long long)b * a.Hkv + hh) * a.Tcap + pos) * a.d;
        }
        const float *x = (value ? v : (key ? k : q)) + at;
        float *y = (value ? v_out : (key ? k_out : q_out)) + to;
        if (value || i >= turned) {
            const int c = value ? i : (i - turned);
            if (VEC) {
                const int at4 = (value ? 0 : a.rot) + 4 * c;
                if (!in_place) *reinterpret_cast<f32x4 *>(y + at4) = *reinterpret_cast<const f32x4 *>(x + at4);
            } else {
                y[(value ? 0 : a.rot) + c] = x[(value ? 0 : a.rot) + c];
            }
            continue;
        }
        const f32x2 *cs = rotary_lds + tt * half;
        if (VEC && a.interleaved) {
            const f32x4 z = *reinterpret_cast<const f32x4 *>(x + 4 * i);
            const f32x2 u = cs[2 * i], w = cs[2 * i + 1];
            *reinterpret_cast<f32x4 *>(y + 4 * i) = f32x4{z.x * u.x - z.y * u.y, z.x * u.y + z.y * u.x, z.z * w.x - z.w * w.y, z.z * w.y + z.w * w.x};
        } else if (VEC) {
            const f32x4 xa = *reinterpret_cast<const f32x4 *>(x + 4 * i), xb = *reinterpret_cast<const f32x4 *>(x + half + 4 * i);
            f32x4 ya, yb;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const f32x2 u = cs[4 * i + c];
                ya[c] = xa[c] * u.x - xb[c] * u.y;
                yb[c] = xa[c] * u.y + xb[c] * u.x;
            }
            *reinterpret_cast<f32x4 *>(y + 4 * i) = ya;
            *reinterpret_cast<f32x4 *>(y + half + 4 * i) = yb;
        } else {
            const int ca = a.interleaved ? 2 * i : i, cb = a.interleaved ? 2 * i + 1 : i + half;
            const float xa = x[ca], xb = x[cb];
            const f32x2 u = cs[i];
            y[ca] = xa * u.x - xb * u.y;
            y[cb] = xa * u.y + xb * u.x;
        }
    }
}

constexpr int MAX_ROTARY_DIM = 4096;       // a token's cosines and sines: 16 KiB of LDS

template <bool APPEND>
int launch_rotary(dl4s_hip_ctx *ctx, const float *q, float *q_out, const float *k, float *k_out, const float *v, float *v_out, RotaryArgs &a) {
    uintptr_t bits = 0;
    for (const void *p : {(const void *)q, (const void *)q_out, (const void *)k, (const void *)k_out, (const void *)v, (const void *)v_out})
        bits |= reinterpret_cast<uintptr_t>(p);
    const bool vec = (bits & 15) == 0 && a.d % 4 == 0 && a.rot % (a.interleaved ? 4 : 8) == 0;
    // About 8192 columns a workgroup (one token each: 8 x 2048 tokens of 4 heads of 32 11.6 us against 5.0; 32768 columns: 2 x 8192
    // tokens of 40 heads of 128 151 us against 122), while there are four workgroups to a compute unit (otherwise 4 x 2048 tokens
    // of 5 heads of 64 6.6 us against 5.5), and at most 32 KiB of LDS.
    const int columns = (a.H + a.Hkv) * a.d;
    a.tokens = a.B * a.L;
    a.per_wg = std::max(1, std::min(8192 / columns, a.tokens / (4 * ctx->cu_count)));
    if (a.rot) a.per_wg = std::max(1, std::min(a.per_wg, 32768 / (a.rot * 4)));
    const size_t lds = (size_t)a.per_wg * (a.rot / 2) * sizeof(f32x2);
    const dim3 grid((a.tokens + a.per_wg - 1) / a.per_wg);
    DL4S_REQUIRE(grid.x < (1u << 24), DL4S_HIP_EUNSUPPORTED, "rotary: %u workgroups of 256 threads", grid.x);
    if (vec) hipLaunchKernelGGL((rotary_f32<APPEND, true>), grid, dim3(256), lds, ctx->stream, q, q_out, k, k_out, v, v_out, a);
    else hipLaunchKernelGGL((rotary_f32<APPEND, false>), grid, dim3(256), lds, ctx->stream, q, q_out, k, k_out, v, v_out, a);
    return dl4s::launch_status("rotary_f32");
}

int rotary_checks(const char *what, int64_t B, int64_t L, int64_t H, int64_t Hkv, int64_t d, int64_t rot_dim, int64_t position0,
                  uint32_t flags, uint32_t known) {
    DL4S_REQUIRE(B >= 0 && L >= 0 && H >= 0 && Hkv >= 0, DL4S_HIP_EINVALID_ARG, "%s: negative extent", what);
    DL4S_REQUIRE(!(flags & ~known), DL4S_HIP_EINVALID_ARG, "%s: unknown flags %#x", what, flags);
    DL4S_REQUIRE(d >= 1 && d <= MAX_ROTARY_DIM, DL4S_HIP_EUNSUPPORTED, "%s: head dim %lld (1 to %d are implemented)", what, (long long)d,
                 MAX_ROTARY_DIM);
    DL4S_REQUIRE(rot_dim >= 0 && rot_dim <= d && rot_dim % 2 == 0, DL4S_HIP_ESHAPE, "%s: %lld turned columns of %lld (an even number is needed)", what,
                 (long long)rot_dim, (long long)d);
    const int64_t big = int64_t(1) << 30;
    DL4S_REQUIRE(B < big && L < big && H < big && Hkv < big && position0 > -big && position0 < big, DL4S_HIP_EUNSUPPORTED,
                 "%s: an extent or the first position above 2^30", what);
    DL4S_REQUIRE(B * L < big && (H + Hkv) * d < big / 2, DL4S_HIP_EUNSUPPORTED, "%s: more than 2^30 tokens or 2^29 columns of a token", what);
    return DL4S_HIP_OK;
}

}  // namespace

extern "C" {

int dl4s_hip_rotary_frequencies(int64_t rot_dim, double base, int scaling, double factor, double low, double high,
                                int64_t original_length, double *out_turns) {
    DL4S_REQUIRE(out_turns || rot_dim == 0, DL4S_HIP_EINVALID_ARG, "rotary_frequencies: out_turns is NULL");
    DL4S_REQUIRE(rot_dim >= 0 && rot_dim % 2 == 0, DL4S_HIP_ESHAPE, "rotary_frequencies: %lld turned columns (an even number is needed)",
                 (long long)rot_dim);
    DL4S_REQUIRE(scaling >= DL4S_ROTARY_UNSCALED && scaling <= DL4S_ROTARY_SCALE_BY_PARTS, DL4S_HIP_EINVALID_ARG,
                 "rotary_frequencies: unknown scaling %d", scaling);
    DL4S_REQUIRE(base > 0 && (scaling == DL4S_ROTARY_UNSCALED || factor > 0), DL4S_HIP_EINVALID_ARG,
                 "rotary_frequencies: base and factor must be positive");
    DL4S_REQUIRE(scaling != DL4S_ROTARY_SCALE_BY_PARTS || (high > low && original_length > 0), DL4S_HIP_EINVALID_ARG,
                 "rotary_frequencies: scaling by parts needs high > low and an original length");
    if (scaling == DL4S_ROTARY_SCALE_BASE && rot_dim > 2) base *= pow(factor, (double)rot_dim / (double)(rot_dim - 2));
    for (int64_t i = 0; i < rot_dim / 2; ++i) {
        double f = pow(base, -2.0 * (double)i / (double)rot_dim) / 6.283185307179586476925286766559;
        if (scaling == DL4S_ROTARY_SCALE_POSITIONS) f /= factor;
        if (scaling == DL4S_ROTARY_SCALE_BY_PARTS) {
            double keep = ((double)original_length * f - low) / (high - low);
            keep = keep < 0 ? 0 : (keep > 1 ? 1 : keep);
            f *= keep + (1 - keep) / factor;
        }
        out_turns[i] = f;
    }
    return DL4S_HIP_OK;
}

int dl4s_hip_rotary_f32(dl4s_hip_ctx *ctx, const float *q, float *q_out, const float *k, float *k_out, int64_t B, int64_t L, int64_t H,
                        int64_t Hkv, int64_t d, int64_t rot_dim, const double *turns, const int32_t *positions, int64_t position0,
                        float amplitude, uint32_t flags) {
    DL4S_CHECK_CTX(ctx);
    const int rc = rotary_checks("rotary", B, L, H, Hkv, d, rot_dim, position0, flags,
                                 DL4S_ROTARY_INTERLEAVED | DL4S_ROTARY_INVERSE | DL4S_ROTARY_TOKEN_MAJOR);
    if (rc) return rc;
    if (B * L == 0 || H + Hkv == 0) return DL4S_HIP_OK;
    DL4S_REQUIRE((H == 0 || (q && q_out)) && (Hkv == 0 || (k && k_out)) && (rot_dim == 0 || turns), DL4S_HIP_EINVALID_ARG,
                 "rotary: NULL pointer");
    RotaryArgs a = {(int)B, (int)L, (int)H, (int)Hkv, (int)d, (int)rot_dim, turns, positions, position0, nullptr, amplitude,
                    (flags & DL4S_ROTARY_INTERLEAVED) != 0, (flags & DL4S_ROTARY_INVERSE) != 0, (flags & DL4S_ROTARY_TOKEN_MAJOR) != 0, 0, 0, 0};
    return launch_rotary<false>(ctx, H ? q : nullptr, H ? q_out : nullptr, Hkv ? k : nullptr, Hkv ? k_out : nullptr, nullptr, nullptr, a);
}

int dl4s_hip_rotary_append_f32(dl4s_hip_ctx *ctx, const float *q, const float *k_new, const float *v_new, float *q_out, float *kcache,
                               float *vcache, int64_t B, int64_t L, int64_t H, int64_t Hkv, int64_t Tcap, int64_t d, int64_t rot_dim,
                               const double *turns, const int32_t *positions, int64_t position0, const int32_t *counts, float amplitude,
                               uint32_t flags) {
    DL4S_CHECK_CTX(ctx);
    const int rc = rotary_checks("rotary_append", B, L, H, Hkv, d, rot_dim, position0, flags,
                                 DL4S_ROTARY_INTERLEAVED | DL4S_ROTARY_TOKEN_MAJOR);
    if (rc) return rc;
    DL4S_REQUIRE(Tcap >= 0 && Tcap < (int64_t(1) << 30), DL4S_HIP_EUNSUPPORTED, "rotary_append: cache capacity %lld", (long long)Tcap);
    if (B * L == 0 || H + Hkv == 0) return DL4S_HIP_OK;
    DL4S_REQUIRE((H == 0 || (q && q_out)) && (Hkv == 0 || (k_new && v_new && kcache && vcache)) && (rot_dim == 0 || turns),
                 DL4S_HIP_EINVALID_ARG, "rotary_append: NULL pointer");
    RotaryArgs a = {(int)B, (int)L, (int)H, (int)Hkv, (int)d, (int)rot_dim, turns, positions, position0, counts, amplitude,
                    (flags & DL4S_ROTARY_INTERLEAVED) != 0, 0, (flags & DL4S_ROTARY_TOKEN_MAJOR) != 0, Tcap, 0, 0};
    return launch_rotary<true>(ctx, H ? q : nullptr, H ? q_out : nullptr, Hkv ? k_new : nullptr, Hkv ? kcache : nullptr, Hkv ? v_new : nullptr,
                               Hkv ? vcache : nullptr, a);
}

}  // extern "C"
