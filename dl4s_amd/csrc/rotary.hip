// Rotary positions for gfx950: pairs of columns of every query and key head turn by an angle that grows with the token's
// position, pair i by turns[i] full turns per position:
//   y_a = amplitude (x_a cos - x_b sin),  y_b = amplitude (x_a sin + x_b cos),  angle = 2 pi frac(position * turns[i])
// with (a, b) = (i, i + rot/2) or, interleaved, (2i, 2i + 1); columns from rot on are copied.  The inverse turns by the
// negative angle: it is the transposed map, so it is also the gradient.
#include "common.h"

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

struct RotaryArgs {
    int B, L, H, Hkv, d, rot;
    const double *turns;
    const int *positions;      // rotary: [B, L]; append: [B]; or NULL
    long long position0;
    const int *counts;         // append: new rows of each batch element, or NULL
    float amplitude;
    int interleaved, inverse, token_major;
    long long Tcap;            // append only
};

__device__ __forceinline__ long long element(const RotaryArgs &a, const int heads, const int b, const int l, const int h) {
    return a.token_major ? (((long long)b * a.L + l) * heads + h) * a.d : (((long long)b * heads + h) * a.L + l) * a.d;
}

// One thread per (token, head, pair or copied column); APPEND writes the turned keys and the values into cache rows.
template <bool APPEND>
__global__ __launch_bounds__(256) void rotary_f32(const float *q, float *q_out, const float *k, float *k_out, const float *v,
                                                   float *v_out, RotaryArgs a, long long n) {
    const int heads = a.H + a.Hkv, half = a.rot / 2, per = half + (a.d - a.rot);
    for (long long e = (long long)blockIdx.x * 256 + threadIdx.x; e < n; e += (long long)gridDim.x * 256) {
        const int c = (int)(e % per);
        long long t = e / per;
        const int h = (int)(t % heads);
        t /= heads;
        const int l = (int)(t % a.L), b = (int)(t / a.L);
        long long pos = a.position0 + l;
        if (a.positions) pos = APPEND ? (long long)a.positions[b] + l : a.positions[(long long)b * a.L + l];
        const bool key = h >= a.H;
        const float *x = key ? k + element(a, a.Hkv, b, l, h - a.H) : q + element(a, a.H, b, l, h);
        float *y = key ? k_out + element(a, a.Hkv, b, l, h - a.H) : q_out + element(a, a.H, b, l, h);
        if (APPEND && key) {
            if (pos < 0 || pos >= a.Tcap || (a.counts && l >= a.counts[b])) continue;
            y = k_out + (((long long)b * a.Hkv + (h - a.H)) * a.Tcap + pos) * a.d;
        }
        if (c < half) {
            const int i = a.interleaved ? 2 * c : c, j = a.interleaved ? 2 * c + 1 : c + half;
            float co, si;
            turn(a.turns[c], pos, co, si);
            co *= a.amplitude;
            si *= a.inverse ? -a.amplitude : a.amplitude;
            const float xa = x[i], xb = x[j];
            y[i] = xa * co - xb * si;
            y[j] = xa * si + xb * co;
        } else {
            y[a.rot + c - half] = x[a.rot + c - half];
        }
        if (APPEND && key) {
            const float *vx = v + element(a, a.Hkv, b, l, h - a.H);
            float *vy = v_out + (((long long)b * a.Hkv + (h - a.H)) * a.Tcap + pos) * a.d;
            if (c < half) {
                vy[c] = vx[c];
                vy[c + half] = vx[c + half];
            } else {
                vy[a.rot + c - half] = vx[a.rot + c - half];
            }
        }
    }
}

int rotary_checks(const char *what, int64_t B, int64_t L, int64_t H, int64_t Hkv, int64_t d, int64_t rot_dim, int64_t position0,
                  uint32_t flags, uint32_t known) {
    DL4S_REQUIRE(B >= 0 && L >= 0 && H >= 0 && Hkv >= 0, DL4S_HIP_EINVALID_ARG, "%s: negative extent", what);
    DL4S_REQUIRE(!(flags & ~known), DL4S_HIP_EINVALID_ARG, "%s: unknown flags %#x", what, flags);
    DL4S_REQUIRE(d >= 1 && d <= (int64_t(1) << 20), DL4S_HIP_EUNSUPPORTED, "%s: head dim %lld", what, (long long)d);
    DL4S_REQUIRE(rot_dim >= 0 && rot_dim <= d && rot_dim % 2 == 0, DL4S_HIP_ESHAPE, "%s: %lld turned columns of %lld (an even number is needed)", what,
                 (long long)rot_dim, (long long)d);
    const int64_t big = int64_t(1) << 30;
    DL4S_REQUIRE(B < big && L < big && H < big && Hkv < big && position0 > -big && position0 < big, DL4S_HIP_EUNSUPPORTED,
                 "%s: an extent or the first position above 2^30", what);
    DL4S_REQUIRE(B * L < big && (H + Hkv) * d < big, DL4S_HIP_EUNSUPPORTED, "%s: more than 2^30 tokens or columns of a token", what);
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
    const long long n = (long long)B * L * (H + Hkv) * (rot_dim / 2 + (d - rot_dim));
    if (n == 0) return DL4S_HIP_OK;
    DL4S_REQUIRE((H == 0 || (q && q_out)) && (Hkv == 0 || (k && k_out)) && (rot_dim == 0 || turns), DL4S_HIP_EINVALID_ARG,
                 "rotary: NULL pointer");
    const RotaryArgs a = {(int)B, (int)L, (int)H, (int)Hkv, (int)d, (int)rot_dim, turns, positions, position0, nullptr, amplitude,
                          (flags & DL4S_ROTARY_INTERLEAVED) != 0, (flags & DL4S_ROTARY_INVERSE) != 0, (flags & DL4S_ROTARY_TOKEN_MAJOR) != 0, 0};
    const long long blocks = (n + 255) / 256;
    hipLaunchKernelGGL((rotary_f32<false>), dim3((unsigned)(blocks < 65536 ? blocks : 65536)), dim3(256), 0, ctx->stream, q, q_out, k, k_out,
                       (const float *)nullptr, (float *)nullptr, a, n);
    return dl4s::launch_status("rotary_f32");
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
    const long long n = (long long)B * L * (H + Hkv) * (rot_dim / 2 + (d - rot_dim));
    if (n == 0) return DL4S_HIP_OK;
    DL4S_REQUIRE((H == 0 || (q && q_out)) && (Hkv == 0 || (k_new && v_new && kcache && vcache)) && (rot_dim == 0 || turns),
                 DL4S_HIP_EINVALID_ARG, "rotary_append: NULL pointer");
    const RotaryArgs a = {(int)B, (int)L, (int)H, (int)Hkv, (int)d, (int)rot_dim, turns, positions, position0, counts, amplitude,
                          (flags & DL4S_ROTARY_INTERLEAVED) != 0, 0, (flags & DL4S_ROTARY_TOKEN_MAJOR) != 0, Tcap};
    const long long blocks = (n + 255) / 256;
    hipLaunchKernelGGL((rotary_f32<true>), dim3((unsigned)(blocks < 65536 ? blocks : 65536)), dim3(256), 0, ctx->stream, q, q_out, k_new,
                       kcache, v_new, vcache, a, n);
    return dl4s::launch_status("rotary_f32");
}

}  // extern "C"
