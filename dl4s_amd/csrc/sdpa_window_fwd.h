// Forward kernel of the windowed attention for head dims up to 128.
//
// One workgroup = 4 wavefronts of 32 query rows each, over one key head: with shared key heads the wavefronts take `hp`
// query heads of the group (hp = 1, 2 or 4), so that the workgroup's queries lie closer together, its keys are staged for
// all of them and fewer tiles are cut by the window's edges.  Per tile of BN keys:
//   S^T[key, query] = K . Q^T (K from LDS, Q in registers), mask and online softmax in the accumulators (a lane holds one
//   query), O^T[column, query] += V^T . P^T with P^T the accumulators themselves as the second operand.
// In small launches eight wavefronts share the 128 rows, four to a half of the tile's keys (KS = 2), and are merged at the end.
// Weights carry a factor 2^7, which cancels against their sum: up to 2^15 they fit fp16, and from 2^-14 down they lose bits
// that are 2^-31 of the row's sum or less.
// Bound: the issue of vector instructions (12 for every matrix instruction) and the matrix instructions (two products of three
// each) beside them, in turns between barriers.  Measured: B8 H16 L2048 d64 window 512 160 us (190 TFLOP/s on the visible pairs,
// 157 is the peak of the fp32 instructions; matrix pipe 26 % busy, vector issue about 40 %), B1 H16/4 L8192 d128 window 1024
// 250 us (260 TFLOP/s, 34 %).  Left out for a timing only: the splitting into planes 27 and 54 us, the softmax 22 and 26, the loads
// of the next tile 16 and 28.
#pragma once
#include "sdpa_window_common.h"

namespace {

struct WindowGeometry {
    int H, Hkv, group, hp, Lq, Lk, d;
    int nqb;                 // query blocks of 128 / hp rows
    int units, per_xcd;      // workgroups with work; consecutive units run on one XCD (workgroup ids go round the 8 XCDs)
    float rT;
    Layout lq, lk;
    WindowArgs w;
};

// Keys of a 32-query wavefront at positions [p0, p1] against a 32-key tile: nothing visible / everything visible.
__device__ __forceinline__ bool tile_hidden(const WindowArgs &w, const int p0, const int p1, const int k0, const int len) {
    return k0 > p1 || k0 >= len || (k0 + 31 <= p0 - w.window && k0 >= w.sinks);
}
__device__ __forceinline__ bool tile_open(const WindowArgs &w, const int p0, const int p1, const int k0, const int len) {
    return k0 + 31 <= p0 && k0 + 32 <= len && (k0 > p1 - w.window || k0 + 32 <= w.sinks);
}

// The workgroup's place: 128 rows of one key head, hp query heads x 128 / hp queries, and the key tiles they see.  Wavefronts
// 4 .. 7, where there are that many, have the rows of 0 .. 3.
template <int BN>
struct Place {
    int qb, part, hk, b, h, rows, q0, qi, qc, len;
    int wp0, wp1;            // first and last position of the workgroup's queries
    int first, lo, tiles;    // tiles [0, first) and [lo, lo + tiles - first)
    __device__ __forceinline__ Place(const WindowGeometry &g, const int unit) {
        qb = unit % g.nqb;
        const int pair = unit / g.nqb, parts = g.group / g.hp;
        part = pair % parts;
        hk = pair / parts % g.Hkv;
        b = pair / parts / g.Hkv;
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) & 3;
        h = hk * g.group + part * g.hp + wave % g.hp;
        rows = 128 / g.hp;
        q0 = qb * rows + wave / g.hp * 32;
        qi = q0 + (threadIdx.x & 31);
        qc = min(qi, g.Lq - 1);
        len = valid_keys(g.w, b, g.Lk);
        wp0 = g.w.q_offset + qb * rows;
        wp1 = g.w.q_offset + min(qb * rows + rows, g.Lq) - 1;
        const int end = (min(wp1 + 1, len) + BN - 1) / BN;
        lo = min(end, max(wp0 - g.w.window + 1, 0) / BN);
        first = min(lo, (g.w.sinks + BN - 1) / BN);
        tiles = first + end - lo;
    }
    __device__ __forceinline__ int key0(const int i) const { return (i < first ? i : lo + i - first) * BN; }
};

template <int DT, int BN, int KS, bool VEC>
__global__ __launch_bounds__(256 * KS, DT <= 64 && KS == 1 ? 3 : 2) void sdpa_window_fwd_f32(const float *__restrict__ q, const float *__restrict__ k,
                                                                             const float *__restrict__ v, float *__restrict__ out,
                                                                             float *__restrict__ stats, const WindowGeometry g) {
    typedef Tile<BN, DT> T;
    extern __shared__ __align__(16) u16 window_lds[];
    u16 *Ks = window_lds, *Vc = Ks + 2 * T::ROWS_PLANE;
    __shared__ __align__(16) int powers[2][BN / 8];        // [K, V]

    const int unit = (blockIdx.x & 7) * g.per_xcd + (blockIdx.x >> 3);
    if (unit >= g.units) return;
    const Place<BN> at(g, unit);
    const int half = (threadIdx.x & 63) >> 5, part = KS == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);

    const float *kp = k + at.b * g.lk.b + at.hk * g.lk.h, *vp = v + at.b * g.lk.b + at.hk * g.lk.h;
    const int ks = (int)g.lk.l, hide0 = g.w.sinks, hide1 = at.wp0 - g.w.window + 1;      // keys between them no query here sees
    Stage<BN, DT, VEC, 256 * KS> kv(ks, g.d, threadIdx.x);
    const int keys = min(at.len, at.wp1 + 1);
    auto load = [&](const int i) {
        const int k0 = at.key0(i);
        kv.load(kp + (long long)k0 * ks, vp + (long long)k0 * ks, ks, k0, keys - k0, g.d, hide0, hide1);
    };
    if (at.tiles > 0) load(0);

    // scores in the base-2 exponent domain
    Frag qf[DT / 16];
    const float *qp = q + at.b * g.lq.b + at.h * g.lq.h + at.qc * g.lq.l;
    const float unq = pow2(-row_operand<DT>(qf, [&](const int c) { return load4(qp, c, g.d, VEC); }, g.rT * LOG2E));
    const int p0 = g.w.q_offset + at.q0, p1 = g.w.q_offset + min(at.q0 + 31, g.Lq - 1), p = g.w.q_offset + at.qi;
    const bool idle = at.q0 >= g.Lq;

    f32x16 o[DT / 32];
#pragma unroll
    for (int t = 0; t < DT / 32; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[t][r] = 0.f;
    float m_run = -INFINITY, m_use = 0.f, l_run = 0.f;
    int nv = -MOST_POWER, nv_most = -MOST_POWER;          // o is in units of 2^nv; the largest of them so far

    for (int i = 0; i < at.tiles; ++i) {
        __syncthreads();
        kv.template store<true, false, false, true>(Ks, nullptr, nullptr, Vc, &powers[0][0]);
        __syncthreads();
        if (i + 1 < at.tiles) load(i + 1);
        const int t0 = at.key0(i);
#pragma unroll
        for (int step = 0; step < BN / 32 / KS; ++step) {
            const int sub = KS == 1 ? step : BN / 32 / KS * part + step, k0 = t0 + 32 * sub;
            if (idle || tile_hidden(g.w, p0, p1, k0, at.len)) continue;
            f32x16 s;
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = 0.f;
#pragma unroll
            for (int st = 0; st < DT / 16; ++st) s = mma3(T::rows_frag(Ks, sub, st), qf[st], s);
            const i32x4 nk = *reinterpret_cast<const i32x4 *>(&powers[0][4 * sub]);
            const Powers vs(&powers[1][4 * sub]);
            settle(s);
            if (!tile_open(g.w, p0, p1, k0, at.len)) {
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] = sees(g.w, p, k0 + acc_row(r) + 4 * half, at.len) ? s[r] : -INFINITY;
            }
            // scores = accumulators * f, one factor for every eight keys (not zero, for those at -inf)
            float f[4], tmax = -INFINITY;
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                f[x] = fmaxf(__builtin_ldexpf(unq, nk[x]), 1.17549435e-38f);
                tmax = fmaxf(tmax, max3(max3(s[4 * x], s[4 * x + 1], s[4 * x + 2]), s[4 * x + 3], s[4 * x + 3]) * f[x]);
            }
            // the reference maximum moves, and the sums are rescaled, only when a weight would pass 2^8 (x 2^7): any factor
            // left in the weights of a row cancels in the division by their sum
            if (__any(tmax - m_run > 8.0f)) {
                tmax = max_halves(tmax);
                const float m_new = tmax - m_run > 8.0f ? tmax : m_run;
                const float alpha = m_run == m_new ? 1.0f : exp2_fast(m_run - m_new);
                m_run = m_new;
                m_use = m_new == -INFINITY ? 0.f : m_new - 7.0f;
                l_run *= alpha;
#pragma unroll
                for (int t = 0; t < DT / 32; ++t) o[t] *= alpha;
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                s[r] = exp2_fast(__builtin_fmaf(s[r], f[r >> 2], -m_use));
                l_run += s[r];
            }
            if (vs.lo != nv || vs.hi != nv) {
                const float unit = to_unit_of_tile(vs, nv, nv_most, s);
#pragma unroll
                for (int t = 0; t < DT / 32; ++t) o[t] *= unit;
            }
#pragma unroll
            for (int st = 0; st < 2; ++st) {
                const Frag pf = acc_frag(s, st);
                Frag vf[DT / 32];
#pragma unroll
                for (int t = 0; t < DT / 32; ++t) vf[t] = T::cols_frag(Vc, t, 2 * sub + st);
                mma3(o, vf, pf);
            }
        }
    }

#pragma unroll
    for (int t = 0; t < DT / 32; ++t) settle(o[t]);
    if (KS == 2) {
        // the second four wavefronts hand what they have to the first
        f32x4 *sums = reinterpret_cast<f32x4 *>(window_lds);             // [wavefront][DT / 8][lane], over the tiles
        __shared__ float rest[3][4][64];
        __shared__ int units[4];
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) & 3, lane = threadIdx.x & 63;
        __syncthreads();
        if (part) {
#pragma unroll
            for (int t = 0; t < DT / 32; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    sums[(wave * (DT / 8) + 4 * t + r) * 64 + lane] = f32x4{o[t][4 * r], o[t][4 * r + 1], o[t][4 * r + 2], o[t][4 * r + 3]};
            rest[0][wave][lane] = m_run;
            rest[1][wave][lane] = m_use;
            rest[2][wave][lane] = l_run;
            units[wave] = nv;
        }
        __syncthreads();
        if (part) return;
        const float m1 = rest[0][wave][lane], u1 = rest[1][wave][lane];
        const int n1 = __builtin_amdgcn_readfirstlane(units[wave]), n = max(nv, n1);
        // (what saw no finite score holds zeros, or NaN, which must survive)
        const float u = m_run == -INFINITY ? (m1 == -INFINITY ? 0.f : u1) : (m1 == -INFINITY ? m_use : fmaxf(m_use, u1));
        const float f0 = m_run == -INFINITY ? 1.0f : exp2_fast(m_use - u), f1 = m1 == -INFINITY ? 1.0f : exp2_fast(u1 - u);
        l_run = l_run * f0 + rest[2][wave][lane] * f1;
        const float g0 = f0 * pow2(max(nv - n, -200)), g1 = f1 * pow2(max(n1 - n, -200));
#pragma unroll
        for (int t = 0; t < DT / 32; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const f32x4 x = sums[(wave * (DT / 8) + 4 * t + r) * 64 + lane];
#pragma unroll
                for (int e = 0; e < 4; ++e) o[t][4 * r + e] = o[t][4 * r + e] * g0 + x[e] * g1;
            }
        m_use = u;
        nv = n;
    }
    if (at.qi >= g.Lq) return;
    const float l = sum_halves(l_run);
    // a row that saw no key: zeros
    const Range see = visible_keys(g.w, at.b, at.qi, g.Lk);
    const float inv = see.first + (see.hi - see.lo) > 0 ? 1.0f / l : 0.f;
    const float unscale = pow2(nv);
    float *op = out + at.b * g.lq.b + at.h * g.lq.h + at.qi * g.lq.l;
#pragma unroll
    for (int t = 0; t < DT / 32; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            f32x4 x = {o[t][4 * r], o[t][4 * r + 1], o[t][4 * r + 2], o[t][4 * r + 3]};
            x = (x * inv) * unscale;
            store4(op, 32 * t + 8 * r + 4 * half, g.d, VEC, x);
        }
    if (stats && half == 0) {
        const long long row = 2 * (((long long)at.b * g.H + at.h) * g.Lq + at.qi);
        stats[row] = m_use;
        stats[row + 1] = inv;
    }
}

}  // namespace
