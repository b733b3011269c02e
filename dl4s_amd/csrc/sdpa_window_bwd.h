// Gradient kernels of the windowed attention for head dims up to 128.  The scores are formed again from q, k and the row
// statistics (m, 1 / l) of the forward pass, w = 2^(s - m) / l, once in each of the two kernels:
//   sdpa_window_dq_f32   workgroups, tiles and operand order of the forward kernel:
//     S^T = K . Q^T, dP^T = V . dO^T, dS^T = w (dP^T - delta), dQ^T += K^T . dS^T; it also forms delta = dO . out per row
//     and leaves it in scratch for the other kernel.
//   sdpa_window_dkv_f32  one workgroup = 8 wavefronts = 128 keys of a key head over 32-row query tiles of all query heads of the
//     group.  Two wavefronts share 32 keys (the columns of their accumulators): one holds K and forms S = Q . K^T, the weights
//     w, and dV^T += dO^T . w, the other holds V and forms dP = dO . V^T and, with the weights it gets through LDS,
//     dK^T += Q^T . dS.  That halves what a wavefront keeps in registers, so two run on a SIMD at every head dim (one
//     wavefront for both, alone on its SIMD above 64 columns, took 655 us where this takes 395 us at B2 H16/4 L4096 d96 window 777).
//     Shared key heads are summed in the accumulators, in a fixed order, without atomics.  Key blocks that hold visible
//     first keys are seen by every later query: their query tiles are dealt to several workgroups whose partial sums a
//     last kernel adds up in order; so are all blocks where that shortens the longest queue of a compute unit.
// The size of dS, and of the weights a key gets, is not known beforehand: as operands they carry a power of two per column
// (query or key), set by the first tile so that the largest value there is 2^8 and lowered, with the accumulators, when a
// later one, weighed with the size of the rows it is multiplied with, would pass 2^15.
// Seven products for the five of the gradient, each three matrix instructions per 16-deep step, and the vector instructions of
// the splitting, which every tile goes through in both forms, rows and columns: their issue bounds both kernels (B2 H16/4 L4096
// d96 window 777: dq 230 us with the matrix pipe 31 % busy, dk/dv 395 us, 23 %).
#pragma once
#include "sdpa_window_fwd.h"

namespace {

// The unit 2^u of the sums in a lane's column.  A tile's operand is x * factor, factor = base * 2^(hi - u), where 2^hi is the unit of
// the planes that it is multiplied with.  fit and fit_tiny look at a tile's x before they are multiplied, whose size is that of
// fp32 numbers, and return whether any lane's unit rose; acc_factor is then the lane's factor for what it has accumulated.  A unit
// rises by what the column itself meets (x and the planes' size together): large rows that only other columns meet leave it alone.
struct ColumnUnit {
    const float base;
    float factor;
    int u = 0;
    bool fresh = true;                                     // nothing but zeros so far
    __device__ __forceinline__ explicit ColumnUnit(const float b) : base(b), factor(b) {}

    __device__ __forceinline__ void move(const int to, const int hi, float &acc_factor) {
        acc_factor = pow2(max(min(u - to, 0), -200));      // (fresh columns, which may go down, hold zeros)
        u = to;
        set(hi);
    }
    // (a column of zeros may be any number of steps from the tile's unit: 0 times a finite factor)
    __device__ __forceinline__ void set(const int hi) { factor = fminf(__builtin_ldexpf(base, hi - u), 3.40282347e38f); }
    // the unit that takes m to 2^8
    __device__ __forceinline__ int unit_for(const float m, const int hi) const {
        return hi - min(max(135 - (int)(__float_as_uint(m * base) >> 23), -126), 126);
    }
    __device__ __forceinline__ bool fit(const f32x16 &x, const int hi, float &acc_factor) {
        float m = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) m = fmaxf(m, fabsf(x[r]));
        const float f = __builtin_ldexpf(base, hi - u);
        factor = fminf(f, 3.40282347e38f);
        if (!__any(m * f > 32768.0f || (fresh && m > 0.f))) return false;
        m = max_halves(m);
        const bool moves = m * f > 32768.0f || (fresh && m > 0.f);
        fresh = fresh && !(m > 0.f);
        move(moves ? unit_for(m, hi) : u, hi, acc_factor);
        return true;
    }
    // For weights, which are at most 2^13: a column takes the tile's unit where its largest is 2^-3 or more.
    __device__ __forceinline__ bool fit_tiny(const f32x16 &w, const int hi, float &acc_factor) {
        float m = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) m = fmaxf(m, w[r]);
        m = max_halves(m);
        int to = u;
        if (m >= 0.125f) to = fresh ? hi : max(u, hi);
        else if (m > 0.f && (fresh || __builtin_ldexpf(m, hi - u) > 32768.0f)) to = unit_for(m, hi);
        const bool rises = !fresh && to > u;
        fresh = fresh && !(m > 0.f);
        move(to, hi, acc_factor);
        return __any(rises);
    }
};

// (delta may be NULL: another kernel has formed it)
template <int DT, int KS, bool VEC>
__device__ __forceinline__ void window_dq(const float *__restrict__ q, const float *__restrict__ k, const float *__restrict__ v,
                                          const float *__restrict__ out, const float *__restrict__ stats,
                                          const float *__restrict__ dout, float *__restrict__ dq, float *__restrict__ delta,
                                          const WindowGeometry &g, const int workgroup) {
    constexpr int BN = 32 * KS;
    typedef Tile<BN, DT> T;
    extern __shared__ __align__(16) u16 window_lds[];
    u16 *Ks = window_lds, *Vs = Ks + 2 * T::ROWS_PLANE, *Kc = Vs + 2 * T::ROWS_PLANE;
    __shared__ __align__(16) int powers[2][BN / 8];        // [K, V]

    const int place = (workgroup & 7) * g.per_xcd + (workgroup >> 3);
    if (place >= g.units) return;
    const Place<BN> at(g, place);
    const int half = (threadIdx.x & 63) >> 5, part = KS == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);

    const float *kp = k + at.b * g.lk.b + at.hk * g.lk.h, *vp = v + at.b * g.lk.b + at.hk * g.lk.h;
    const int ks = (int)g.lk.l, hide0 = g.w.sinks, hide1 = at.wp0 - g.w.window + 1;
    Stage<BN, DT, VEC, 256 * KS> kv(ks, g.d, threadIdx.x);
    const int keys = min(at.len, at.wp1 + 1);
    auto load = [&](const int i) {
        const int k0 = at.key0(i);
        kv.load(kp + (long long)k0 * ks, vp + (long long)k0 * ks, ks, k0, keys - k0, g.d, hide0, hide1);
    };
    if (at.tiles > 0) load(0);

    const long long el = at.b * g.lq.b + at.h * g.lq.h + at.qc * g.lq.l, row = ((long long)at.b * g.H + at.h) * g.Lq + at.qc;
    Frag qf[DT / 16], gf[DT / 16];
    const float unq = pow2(-row_operand<DT>(qf, [&](const int c) { return load4(q + el, c, g.d, VEC); }, g.rT * LOG2E));
    float del = 0.f;
    const float ung = pow2(-row_operand<DT>(gf, [&](const int c) {
        const f32x4 x = load4(dout + el, c, g.d, VEC), o = load4(out + el, c, g.d, VEC);
#pragma unroll
        for (int e = 0; e < 4; ++e) del += x[e] * o[e];
        return x;
    }, 1.0f));
    del = sum_halves(del);
    const float m = stats[2 * row], inv = stats[2 * row + 1];
    if (delta && half == 0 && part == 0 && at.qi < g.Lq) delta[row] = del;
    const int p0 = g.w.q_offset + at.q0, p1 = g.w.q_offset + min(at.q0 + 31, g.Lq - 1), p = g.w.q_offset + at.qi;
    const bool idle = at.q0 >= g.Lq;

    f32x16 acc[DT / 32];
#pragma unroll
    for (int t = 0; t < DT / 32; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[t][r] = 0.f;
    ColumnUnit unit(inv);                                  // dS = 2^(s - m) (dP - delta) / l

    for (int i = 0; i < at.tiles; ++i) {
        __syncthreads();
        kv.template store<true, true, true, false>(Ks, Kc, Vs, nullptr, &powers[0][0]);
        __syncthreads();
        if (i + 1 < at.tiles) load(i + 1);
        const int k0 = at.key0(i) + 32 * part;
        if (idle || tile_hidden(g.w, p0, p1, k0, at.len)) continue;
        f32x16 s, dp;
#pragma unroll
        for (int r = 0; r < 16; ++r) { s[r] = 0.f; dp[r] = 0.f; }
#pragma unroll
        for (int st = 0; st < DT / 16; ++st)
            mma3x2(s, T::rows_frag(Ks, part, st), qf[st], dp, T::rows_frag(Vs, part, st), gf[st]);
        const Powers kn(&powers[0][4 * part]);
        const i32x4 vn = *reinterpret_cast<const i32x4 *>(&powers[1][4 * part]);
        settle(s, dp);
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const float f = __builtin_ldexpf(unq, kn.n[x]), fp = __builtin_ldexpf(ung, vn[x]);
#pragma unroll
            for (int r = 4 * x; r < 4 * x + 4; ++r) s[r] = exp2_fast(__builtin_fmaf(s[r], f, -m)) * __builtin_fmaf(dp[r], fp, -del);
        }
        if (!tile_open(g.w, p0, p1, k0, at.len)) {
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = sees(g.w, p, k0 + acc_row(r) + 4 * half, at.len) ? s[r] : 0.f;
        }
        if (kn.lo != kn.hi) to_one_unit(kn, s);
        float shrink;
        if (unit.fit(s, kn.hi, shrink)) {
#pragma unroll
            for (int t = 0; t < DT / 32; ++t) acc[t] *= shrink;
        }
#pragma unroll
        for (int st = 0; st < 2; ++st) {
            const Frag df = acc_frag(s, st, unit.factor);
            Frag kc[DT / 32];
#pragma unroll
            for (int t = 0; t < DT / 32; ++t) kc[t] = T::cols_frag(Kc, t, 2 * part + st);
            mma3(acc, kc, df);
        }
    }

#pragma unroll
    for (int t = 0; t < DT / 32; ++t) settle(acc[t]);
    const int power = unit.u;
    f32x4 *sums = reinterpret_cast<f32x4 *>(window_lds);                 // KS = 2: [wavefront][DT / 8][lane], over the tiles
    const int at_sums = ((threadIdx.x >> 6) & 3) * (DT / 8) * 64 + (threadIdx.x & 63);
    if (KS == 2) {
        // the second four wavefronts hand what they have to the first
        __syncthreads();
        if (part) {
#pragma unroll
            for (int t = 0; t < DT / 32; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    f32x4 x;
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[e] = __builtin_ldexpf(acc[t][4 * r + e], power);
                    sums[at_sums + 64 * (4 * t + r)] = x;
                }
        }
        __syncthreads();
        if (part) return;
    }
    if (at.qi >= g.Lq) return;
    const bool empty = inv == 0.f;                         // saw no key: no gradient, whatever stands in its rows
#pragma unroll
    for (int t = 0; t < DT / 32; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            f32x4 x = {acc[t][4 * r], acc[t][4 * r + 1], acc[t][4 * r + 2], acc[t][4 * r + 3]};
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = __builtin_ldexpf(x[e], power);
            if (KS == 2) x += sums[at_sums + 64 * (4 * t + r)];
            x *= g.rT;
            if (empty) x = f32x4{0.f, 0.f, 0.f, 0.f};
            store4(dq + el, 32 * t + 8 * r + 4 * half, g.d, VEC, x);
        }
}

template <int DT, int KS, bool VEC>
__global__ __launch_bounds__(256 * KS, DT <= 96 ? 2 : 1) void sdpa_window_dq_f32(const float *__restrict__ q, const float *__restrict__ k,
                                                                                 const float *__restrict__ v, const float *__restrict__ out,
                                                                                 const float *__restrict__ stats,
                                                                                 const float *__restrict__ dout, float *__restrict__ dq,
                                                                                 float *__restrict__ delta, const WindowGeometry g) {
    window_dq<DT, KS, VEC>(q, k, v, out, stats, dout, dq, delta, g, blockIdx.x);
}

// How the key blocks (128 keys) of all (batch, key head) pairs are dealt to workgroups: class 0 are those that hold visible
// first keys, class 1 the others; each in `chunks` equal pieces of its query tiles.  The pieces of class 1 are started
// first, the shorter ones of class 0 fill up.  Workgroup ids of a class go round the XCDs so that consecutive pieces of
// work share one XCD's L2.
struct KeyBlocks {
    int pairs, blocks, sink_blocks;
    int chunks[2];                   // [0] blocks with first keys, [1] the others
    int units[2], per_xcd[2];
    float *partial;                  // [pair][block][chunk][dk, dv][128][d], blocks with one chunk have none
    long long class1;                // element offset of the second class's partial sums
};
__device__ __forceinline__ float *partial_sums(const KeyBlocks &kb, const int pair, const int block, const int chunk, const int d) {
    const int c = block >= kb.sink_blocks;
    const long long slot = c ? ((long long)pair * (kb.blocks - kb.sink_blocks) + block - kb.sink_blocks) * kb.chunks[1] + chunk
                             : ((long long)pair * kb.sink_blocks + block) * kb.chunks[0] + chunk;
    return kb.partial + (c ? kb.class1 : 0) + slot * 256 * d;
}

template <int DT, bool VEC>
__device__ __forceinline__ void window_dkv(const float *__restrict__ q, const float *__restrict__ k, const float *__restrict__ v,
                                           const float *__restrict__ stats, const float *__restrict__ dout,
                                           const float *__restrict__ delta, float *__restrict__ dk, float *__restrict__ dv,
                                           const WindowGeometry &g, const KeyBlocks &kb, const int workgroup) {
    typedef Tile<32, DT> T;
    extern __shared__ __align__(16) u16 window_lds[];
    constexpr int BUF = 4 * (T::ROWS_PLANE + T::COLS_PLANE);     // [Q rows][dO rows][Q columns][dO columns]
    f32x4 *weights = reinterpret_cast<f32x4 *>(window_lds + 2 * BUF);      // [pair of wavefronts][4][lane]
    __shared__ __align__(16) float row_values[2][96];      // [buffer][3][32]: m, 2^13 / l, delta of the tile's queries
    __shared__ __align__(16) int powers[2][2][4];          // [buffer][Q, dO]

    int id = workgroup, cl = 1;
    if (id >= 8 * kb.per_xcd[1]) { id -= 8 * kb.per_xcd[1]; cl = 0; }
    const int unit = (id & 7) * kb.per_xcd[cl] + (id >> 3);
    if (unit >= kb.units[cl]) return;
    const int chunk = unit % kb.chunks[cl], in_class = cl ? kb.blocks - kb.sink_blocks : kb.sink_blocks;
    const int block = unit / kb.chunks[cl] % in_class + (cl ? kb.sink_blocks : 0), pair = unit / kb.chunks[cl] / in_class;
    const int hk = pair % g.Hkv, b = pair / g.Hkv;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, half = lane >> 5, ln = lane & 31;
    const int two = wave & 3;
    const bool values = wave >= 4;                         // holds V, forms dP and dK; the other holds K, forms w and dV
    const int b0 = block * 128, k0 = b0 + two * 32, key = k0 + ln;
    const int len = valid_keys(g.w, b, g.Lk);

    // query tiles that can see the block: from the first key's position to the window's end behind the last key.  Queries that
    // see no key at all (their window lies behind the last valid one, and no first keys) are taken as rows of zeros.
    const int rows = min(len, g.w.sinks) > 0 ? g.Lq : min(g.Lq, max(len + g.w.window - 1 - g.w.q_offset, 0));
    const int i1 = min(rows, b0 < g.w.sinks ? g.Lq : max(b0 + 127 + g.w.window - g.w.q_offset, 0));
    const int t0 = max(b0 - g.w.q_offset, 0) / 32, t1 = (i1 + 31) / 32;
    const int per_head = b0 < len && t1 > t0 ? t1 - t0 : 0;
    const int all = per_head * g.group, from = (int)((long long)all * chunk / kb.chunks[cl]), to = (int)((long long)all * (chunk + 1) / kb.chunks[cl]);

    // (wavefronts take pieces of the tiles in the order 0, 4, 1, 5, ...: where there are fewer pieces, both kinds get some)
    Stage<32, DT, VEC, 512> qg((int)g.lq.l, g.d, (two * 2 + values) * 64 + lane);
    float sv = 0.f;
    // the next tile to be loaded: its place, and where it lies
    int next = t0 + (per_head ? from % per_head : 0);
    const int head0 = hk * g.group + (per_head ? from / per_head : 0), qs = (int)g.lq.l;
    const float *qp = q + b * g.lq.b + head0 * g.lq.h + (long long)next * 32 * qs, *gp = dout + (qp - q);
    long long row0 = ((long long)b * g.H + head0) * g.Lq;
    auto load = [&]() {
        const int r0 = next * 32;
        qg.load(qp, gp, qs, r0, rows - r0, g.d);
        if (threadIdx.x < 96) {
            const int which = threadIdx.x >> 5, r = r0 + (threadIdx.x & 31);
            sv = 0.f;
            if (r < rows) sv = which == 2 ? delta[row0 + r] : stats[2 * (row0 + r) + which];
            if (which == 1) sv *= 8192.0f;
        }
        if (++next == t1) {                                // on to the group's next head
            next = t0;
            qp += g.lq.h - (long long)(t1 - 1 - t0) * 32 * qs;
            gp += g.lq.h - (long long)(t1 - 1 - t0) * 32 * qs;
            row0 += g.Lq;
        } else {
            qp += 32 * qs;
            gp += 32 * qs;
        }
    };
    auto stage = [&](const int e) {
        const int buf = (e - from) & 1;
        u16 *Qs = window_lds + buf * BUF, *Gs = Qs + 2 * T::ROWS_PLANE, *Qc = Gs + 2 * T::ROWS_PLANE, *Gc = Qc + 2 * T::COLS_PLANE;
        qg.template store<true, true, true, true>(Qs, Qc, Gs, Gc, &powers[buf][0][0], g.rT * LOG2E);
        if (threadIdx.x < 96) row_values[buf][threadIdx.x] = sv;
        if (e + 1 < to) load();
    };
    int now = next;                                        // the tile that is worked on
    if (from < to) load();

    Frag mine[DT / 16];                                    // the key rows, or the value rows
    const long long el = b * g.lk.b + hk * g.lk.h + key * g.lk.l;
    const float *mrow = (values ? v : k) + el;
    const bool seen = key < len && key < g.w.q_offset + g.Lq && (key < g.w.sinks || key > g.w.q_offset - g.w.window);   // by any query
    const float unscale = pow2(-row_operand<DT>(mine, [&](const int c) { return seen ? load4(mrow, c, g.d, VEC) : f32x4{0.f, 0.f, 0.f, 0.f}; }, 1.0f));

    f32x16 acc[DT / 32];
#pragma unroll
    for (int t = 0; t < DT / 32; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[t][r] = 0.f;
    // The operands are 2^13 w, and w (dP - delta).
    ColumnUnit column(values ? 1.0f / 8192 : 1.0f);
    bool plain = false;                                    // every column is in units of 2^plain_unit, and its weights need no factor there
    int plain_unit = 0;

    // Two buffers: behind the exchange of the weights one wavefront of a pair multiplies and then stages its share of the next
    // tile, the other stages first, so that on their SIMD one's vector work runs beside the other's matrix instructions.
    if (from < to) {
        stage(from);
        __syncthreads();
    }
    for (int e = from; e < to; ++e) {
        const int buf = (e - from) & 1;
        const u16 *rows_at = window_lds + buf * BUF, *cols_at = rows_at + 4 * T::ROWS_PLANE;
        const u16 *first = rows_at + (values ? 2 * T::ROWS_PLANE : 0), *then = cols_at + (values ? 0 : 2 * T::COLS_PLANE);
        const float *rowv = row_values[buf];
        const int q0 = now * 32;
        now = now + 1 == t1 ? t0 : now + 1;
        const int p0 = g.w.q_offset + q0, p1 = g.w.q_offset + min(q0 + 31, g.Lq - 1);
        const bool hidden = tile_hidden(g.w, p0, p1, k0, len), open = tile_open(g.w, p0, p1, k0, len) && q0 + 32 <= g.Lq;
        f32x16 s;
        if (!hidden) {
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = 0.f;
#pragma unroll
            for (int st = 0; st < DT / 16; ++st) s = mma3(T::rows_frag(first, 0, st), mine[st], s);
            const i32x4 n = *reinterpret_cast<const i32x4 *>(powers[buf][values]);
            settle(s);
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const float f = __builtin_ldexpf(unscale, n[x]);
                const f32x4 m = *reinterpret_cast<const f32x4 *>(rowv + (values ? 64 : 0) + 8 * x + 4 * half);
#pragma unroll
                for (int y = 0; y < 4; ++y) s[4 * x + y] = __builtin_fmaf(s[4 * x + y], f, -m[y]);     // s - m, or dP - delta
            }
            if (!values) {
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const f32x4 inv = *reinterpret_cast<const f32x4 *>(rowv + 32 + 8 * x + 4 * half);
#pragma unroll
                    for (int y = 0; y < 4; ++y) s[4 * x + y] = exp2_fast(s[4 * x + y]) * inv[y];
                }
                if (!open) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int i = q0 + acc_row(r) + 4 * half;
                        s[r] = ((i < g.Lq) & sees(g.w, g.w.q_offset + i, key, len)) ? s[r] : 0.f;
                    }
                }
#pragma unroll
                for (int x = 0; x < 4; ++x) weights[(two * 4 + x) * 64 + lane] = f32x4{s[4 * x], s[4 * x + 1], s[4 * x + 2], s[4 * x + 3]};
            }
        }
        __syncthreads();
        if (!values && e + 1 < to) stage(e + 1);
        if (!hidden) {
            if (values) {
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const f32x4 w = weights[(two * 4 + x) * 64 + lane];
#pragma unroll
                    for (int y = 0; y < 4; ++y) s[4 * x + y] *= w[y];
                }
            }
            const Powers pw(powers[buf][!values]);
            if (pw.lo != pw.hi) to_one_unit(pw, s);
            if (values || !plain || pw.lo != plain_unit || pw.hi != plain_unit) {
                float shrink;
                if (values ? column.fit(s, pw.hi, shrink) : column.fit_tiny(s, pw.hi, shrink)) {
#pragma unroll
                    for (int t = 0; t < DT / 32; ++t) acc[t] *= shrink;
                }
                s *= column.factor;
                plain = !__any(column.fresh || column.u != pw.hi);
                plain_unit = pw.hi;
            }
#pragma unroll
            for (int st = 0; st < 2; ++st) {
                const Frag f = acc_frag(s, st);
                Frag c[DT / 32];
#pragma unroll
                for (int t = 0; t < DT / 32; ++t) c[t] = T::cols_frag(then, t, st);
                mma3(acc, c, f);
            }
        }
        if (values && e + 1 < to) stage(e + 1);
        __syncthreads();
    }

#pragma unroll
    for (int t = 0; t < DT / 32; ++t) settle(acc[t]);
    if (key >= g.Lk) return;
    // q was staged as q rT log2(e): dk = rT sum dS q = ln(2) of what was summed
    const int power = column.u - (values ? 0 : 13);
    const float factor_out = values ? 0.69314718055994530942f : 1.0f;
    float *to_row = (values ? dk : dv) + el;
    if (kb.chunks[cl] > 1) to_row = partial_sums(kb, pair, block, chunk, g.d) + (values ? 0 : 128ll * g.d) + (two * 32 + ln) * (long long)g.d;
#pragma unroll
    for (int t = 0; t < DT / 32; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            f32x4 x = {acc[t][4 * r], acc[t][4 * r + 1], acc[t][4 * r + 2], acc[t][4 * r + 3]};
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = __builtin_ldexpf(x[e] * factor_out, power);
            store4(to_row, 32 * t + 8 * r + 4 * half, g.d, VEC, x);
        }
}

template <int DT, bool VEC>
__global__ __launch_bounds__(512, 2) void sdpa_window_dkv_f32(const float *__restrict__ q, const float *__restrict__ k,
                                                              const float *__restrict__ v, const float *__restrict__ stats,
                                                              const float *__restrict__ dout, const float *__restrict__ delta,
                                                              float *__restrict__ dk, float *__restrict__ dv, const WindowGeometry g,
                                                              const KeyBlocks kb) {
    window_dkv<DT, VEC>(q, k, v, stats, dout, delta, dk, dv, g, kb, blockIdx.x);
}

// Both at once, where all their workgroups find a compute unit of their own: side by side they take as long as the longer one.
// delta has been formed before.
template <int DT, bool VEC>
__global__ __launch_bounds__(512, 2) void sdpa_window_dq_dkv_f32(const float *__restrict__ q, const float *__restrict__ k,
                                                                 const float *__restrict__ v, const float *__restrict__ out,
                                                                 const float *__restrict__ stats, const float *__restrict__ dout,
                                                                 const float *__restrict__ delta, float *__restrict__ dq,
                                                                 float *__restrict__ dk, float *__restrict__ dv, const WindowGeometry g,
                                                                 const KeyBlocks kb) {
    const int first = 8 * (kb.per_xcd[0] + kb.per_xcd[1]), workgroup = blockIdx.x;
    if (workgroup < first) window_dkv<DT, VEC>(q, k, v, stats, dout, delta, dk, dv, g, kb, workgroup);
    else window_dq<DT, 2, VEC>(q, k, v, out, stats, dout, dq, nullptr, g, workgroup - first);
}

// Adds up the partial sums of the key blocks that were dealt to several workgroups, chunk after chunk.  One thread per
// element of dk and dv of such a block.
__global__ __launch_bounds__(256) void sdpa_window_join_f32(float *__restrict__ dk, float *__restrict__ dv, const WindowGeometry g,
                                                             const KeyBlocks kb, const int block0) {
    const int block = block0 + blockIdx.y, pair = blockIdx.z, chunks = kb.chunks[block >= kb.sink_blocks];
    const int e = blockIdx.x * 256 + threadIdx.x;                        // over [dk, dv][128][d]
    const int which = e / (128 * g.d), r = e / g.d % 128, c = e % g.d, key = block * 128 + r;
    if (which > 1 || key >= g.Lk) return;
    float s = 0.f;
    for (int x = 0; x < chunks; ++x) s += partial_sums(kb, pair, block, x, g.d)[e];
    (which ? dv : dk)[(pair / g.Hkv) * g.lk.b + (pair % g.Hkv) * g.lk.h + key * g.lk.l + c] = s;
}

}  // namespace
