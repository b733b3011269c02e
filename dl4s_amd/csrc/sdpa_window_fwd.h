// Forward kernel of the windowed attention for head dims up to 128.
//
// One workgroup = 4 wavefronts of 32 query rows each, over one key head: with shared key heads the wavefronts take `hp`
// query heads of the group (hp = 1, 2 or 4), so that the workgroup's queries lie closer together, its keys are staged for
// all of them and fewer tiles are cut by the window's edges.  Per tile of BN keys:
//   S^T[key, query] = K . Q^T (K from LDS, Q in registers), mask and online softmax in the accumulators (a lane holds one
//   query), O^T[column, query] += V^T . P^T with P^T the accumulators themselves as the second operand.
// Bound: the matrix instructions (two products of six each), beside which softmax and the splitting into planes run.
#pragma once
#include "sdpa_window_common.h"

namespace {

struct WindowGeometry {
    int H, Hkv, group, hp, Lq, Lk, d;
    int nqb;                 // query blocks of 128 / hp rows
    int units, per_xcd;      // workgroups with work; consecutive units run on one XCD (workgroup ids go round the 8 XCDs)
    float rT;
    int vec;
    Layout lq, lk;
    WindowArgs w;
};

// Keys of a 32-query wavefront at positions [p0, p1] against a 32-key tile: nothing visible / everything visible.
__device__ __forceinline__ bool tile_hidden(const WindowArgs &w, const long long p0, const long long p1, const int k0, const int len) {
    return k0 > p1 || k0 >= len || ((long long)k0 + 31 <= p0 - w.window && k0 >= w.sinks);
}
__device__ __forceinline__ bool tile_open(const WindowArgs &w, const long long p0, const long long p1, const int k0, const int len) {
    return k0 + 31 <= p0 && k0 + 32 <= len && (k0 > p1 - w.window || k0 + 32 <= w.sinks);
}

template <int DT, int BN>
__global__ __launch_bounds__(256, 2) void sdpa_window_fwd_f32(const float *__restrict__ q, const float *__restrict__ k,
                                                               const float *__restrict__ v, float *__restrict__ out,
                                                               float *__restrict__ stats, const WindowGeometry g) {
    typedef Tile<BN, DT> T;
    extern __shared__ __align__(16) u16 window_lds[];
    u16 *Ks = window_lds, *Vs = window_lds + 3 * T::ROWS_PLANE;

    const int unit = (blockIdx.x & 7) * g.per_xcd + (blockIdx.x >> 3);
    if (unit >= g.units) return;
    const int qb = unit % g.nqb, pair = unit / g.nqb;                  // pair: (batch, key head, part of the group)
    const int parts = g.group / g.hp;
    const int part = pair % parts, hk = (pair / parts) % g.Hkv, b = pair / parts / g.Hkv;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, half = lane >> 5, ln = lane & 31;
    const int h = hk * g.group + part * g.hp + wave % g.hp;
    const int rows = 128 / g.hp;
    const int q0 = qb * rows + wave / g.hp * 32, qi = q0 + ln, qc = qi < g.Lq ? qi : g.Lq - 1;
    const int len = valid_keys(g.w, b, g.Lk);

    // tiles of the workgroup: [0, first) and [lo, end)
    const long long wp0 = g.w.q_offset + qb * rows, wp1 = g.w.q_offset + min(qb * rows + rows, g.Lq) - 1;
    const int end = (int)((min(wp1 + 1, (long long)len) + BN - 1) / BN);
    const long long low = wp0 - g.w.window + 1;
    const int lo = (int)min((long long)end, low > 0 ? low / BN : 0), first = min(lo, (g.w.sinks + BN - 1) / BN);
    const int tiles = first + (end - lo);

    const float *kp = k + b * g.lk.b + hk * g.lk.h, *vp = v + b * g.lk.b + hk * g.lk.h;
    f32x4 kst[T::NROW], vst[4];
    auto load = [&](const int i) {
        const int k0 = (i < first ? i : lo + i - first) * BN;
        T::load_rows(kst, kp, g.lk.l, k0, len, g.d, g.vec);
        T::load_quad(vst, vp, g.lk.l, k0, len, g.d, g.vec);
    };
    if (tiles > 0) load(0);

    Frag qf[DT / 16];
    {
        const float *qp = q + b * g.lq.b + h * g.lq.h + qc * g.lq.l;
#pragma unroll
        for (int s = 0; s < DT / 16; ++s) {
            const f32x4 x = load4(qp, 16 * s + 8 * half, g.d, g.vec), y = load4(qp, 16 * s + 8 * half + 4, g.d, g.vec);
            float z[8];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                z[e] = (x[e] * g.rT) * LOG2E;              // scores in the base-2 exponent domain
                z[4 + e] = (y[e] * g.rT) * LOG2E;
            }
            qf[s] = split8(z);
        }
    }
    const long long p0 = g.w.q_offset + q0, p1 = g.w.q_offset + min(q0 + 31, g.Lq - 1), p = g.w.q_offset + qi;
    const bool idle = q0 >= g.Lq;

    f32x16 o[DT / 32];
#pragma unroll
    for (int t = 0; t < DT / 32; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[t][r] = 0.f;
    float m_run = -INFINITY, m_use = 0.f, l_run = 0.f;

    for (int i = 0; i < tiles; ++i) {
        __syncthreads();
        T::store_rows(Ks, kst);
        T::store_cols(Vs, vst);
        __syncthreads();
        if (i + 1 < tiles) load(i + 1);
        const int t0 = (i < first ? i : lo + i - first) * BN;
#pragma unroll
        for (int sub = 0; sub < BN / 32; ++sub) {
            const int k0 = t0 + 32 * sub;
            if (idle || tile_hidden(g.w, p0, p1, k0, len)) continue;
            f32x16 s;
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = 0.f;
#pragma unroll
            for (int st = 0; st < DT / 16; ++st) s = mma6(T::rows_frag(Ks, sub, st), qf[st], s);
            if (!tile_open(g.w, p0, p1, k0, len)) {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int j = k0 + acc_row(r) + 4 * half;
                    if (!(j <= p && j < len && (j > p - g.w.window || j < g.w.sinks))) s[r] = -INFINITY;
                }
            }
            float tmax = s[0];
#pragma unroll
            for (int r = 1; r < 16; ++r) tmax = fmaxf(tmax, s[r]);
            tmax = max_halves(tmax);
            // the reference maximum moves, and the sums are rescaled, only when a weight would pass 2^8: any factor left in the
            // weights of a row cancels in the division by their sum
            if (__any(tmax - m_run > 8.0f)) {
                const float m_new = fmaxf(m_run, tmax);
                const float alpha = m_run == m_new ? 1.0f : exp2_fast(m_run - m_new);
                m_run = m_new;
                m_use = m_new == -INFINITY ? 0.f : m_new;
                l_run *= alpha;
#pragma unroll
                for (int t = 0; t < DT / 32; ++t)
#pragma unroll
                    for (int r = 0; r < 16; ++r) o[t][r] *= alpha;
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                s[r] = exp2_fast(s[r] - m_use);
                l_run += s[r];
            }
#pragma unroll
            for (int st = 0; st < 2; ++st) {
                const Frag pf = acc_frag(s, st);
#pragma unroll
                for (int t = 0; t < DT / 32; ++t) o[t] = mma6(T::cols_frag(Vs, t, 2 * sub + st), pf, o[t]);
            }
        }
    }

    if (qi >= g.Lq) return;
    const float l = sum_halves(l_run);
    // a row that saw no key: zeros
    const Range see = visible_keys(g.w, b, qi, g.Lk);
    const float inv = see.first + (see.hi - see.lo) > 0 ? 1.0f / l : 0.f;
    float *op = out + b * g.lq.b + h * g.lq.h + qi * g.lq.l;
#pragma unroll
    for (int t = 0; t < DT / 32; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r)
            store4(op, 32 * t + 8 * r + 4 * half, g.d, g.vec,
                   f32x4{o[t][4 * r] * inv, o[t][4 * r + 1] * inv, o[t][4 * r + 2] * inv, o[t][4 * r + 3] * inv});
    if (stats && half == 0) {
        const long long at = 2 * (((long long)b * g.H + h) * g.Lq + qi);
        stats[at] = m_use;
        stats[at + 1] = inv;
    }
}

}  // namespace
