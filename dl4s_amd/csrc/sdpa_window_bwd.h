// Gradient kernels of the windowed attention for head dims up to 128.  The scores are formed again from q, k and the row
// statistics (m, 1 / l) of the forward pass, w = 2^(s - m) / l, once in each of the two kernels:
//   sdpa_window_dq_f32   workgroups, tiles and operand order of the forward kernel:
//     S^T = K . Q^T, dP^T = V . dO^T, dS^T = w (dP^T - delta), dQ^T += K^T . dS^T; it also forms delta = dO . out per row
//     and leaves it in scratch for the other kernel.
//   sdpa_window_dkv_f32  one workgroup = 128 keys of a key head (a wavefront holds 32 keys as columns, K and V in registers)
//     over 32-row query tiles of all query heads of the group:
//     S = Q . K^T, dP = dO . V^T, dV^T += dO^T . w, dK^T += Q^T . dS
//     so shared key heads are summed in the accumulators, in a fixed order, without atomics.  Key blocks that hold visible
//     first keys are seen by every later query: their query tiles are dealt to several workgroups whose partial sums a
//     last kernel adds up in order; so are all blocks when there are too few of them to fill the GPU.
// Seven products for the five of the gradient, each six matrix instructions per 16-deep step: that is what bounds them.
#pragma once
#include "sdpa_window_fwd.h"

namespace {

// Two 32 x C tiles staged together: a thread loads 4 x 4 pieces, splits them once and writes them in row form and, exchanged
// pairwise, in column form.  C / 4 * 8 pieces a tile are a whole number of wavefronts, so which tile a thread serves is
// uniform over its wavefront.
template <int C>
struct Pair {
    typedef Tile<32, C> T;
    static constexpr int QUADS = 8 * (C / 4), NP = (2 * QUADS + 255) / 256;
    f32x4 x[NP][4];

    __device__ static __forceinline__ int piece(const int i) { return threadIdx.x + 256 * i; }
    __device__ static __forceinline__ bool has(const int i) { return piece(i) < 2 * QUADS; }
    __device__ static __forceinline__ int second(const int i) { return piece(i) >= QUADS; }
    __device__ static __forceinline__ int row(const int i) { return (piece(i) - second(i) * QUADS) / (C / 4) * 4; }
    __device__ static __forceinline__ int col(const int i) { return (piece(i) - second(i) * QUADS) % (C / 4) * 4; }

    __device__ __forceinline__ void load(const float *a, const float *b, const long long stride, const int r0, const int rows, const int d,
                                         const bool vec) {
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const float *base = second(i) ? b : a;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int r = r0 + row(i) + j;
                x[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
                if (has(i) && r < rows) x[i][j] = load4(base + r * stride, col(i), d, vec);
            }
        }
    }
    // scale: of the first tile's values (two factors, rounded one after the other); the column form of a tile only where asked
    template <bool COLS_A, bool COLS_B>
    __device__ __forceinline__ void store(u16 *rows_a, u16 *cols_a, u16 *rows_b, u16 *cols_b, const float f0, const float f1) const {
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            if (!has(i)) continue;
            const bool b = second(i);
            u16 *tr = (b ? rows_b : rows_a) + row(i) * (C + 8) + col(i);
            Planes w[4][2];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                f32x4 v = x[i][j];
                if (!b) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = (v[e] * f0) * f1;
                }
                w[j][0] = split2(v.x, v.y);
                w[j][1] = split2(v.z, v.w);
                *reinterpret_cast<u32x2 *>(tr + j * (C + 8)) = u32x2{w[j][0].h, w[j][1].h};
                *reinterpret_cast<u32x2 *>(tr + j * (C + 8) + T::ROWS_PLANE) = u32x2{w[j][0].m, w[j][1].m};
                *reinterpret_cast<u32x2 *>(tr + j * (C + 8) + 2 * T::ROWS_PLANE) = u32x2{w[j][0].l, w[j][1].l};
            }
            if (b ? !COLS_B : !COLS_A) continue;
            const int kq = row(i) >> 2, at = 2 * (kq >> 2) + (kq & 1), sub = 4 * ((kq >> 1) & 1);
            u16 *tc = b ? cols_b : cols_a;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                u16 *p = tc + (col(i) + c) * 32 + ((at ^ T::swap(col(i) + c)) << 3) + sub;
                // low or high halves of two rows' words, side by side
                const unsigned pick = c & 1 ? 0x07060302u : 0x05040100u;
                auto turn = [&](const unsigned r0, const unsigned r1) { return __builtin_amdgcn_perm(r1, r0, pick); };
                *reinterpret_cast<u32x2 *>(p) = u32x2{turn(w[0][c >> 1].h, w[1][c >> 1].h), turn(w[2][c >> 1].h, w[3][c >> 1].h)};
                *reinterpret_cast<u32x2 *>(p + T::COLS_PLANE) = u32x2{turn(w[0][c >> 1].m, w[1][c >> 1].m), turn(w[2][c >> 1].m, w[3][c >> 1].m)};
                *reinterpret_cast<u32x2 *>(p + 2 * T::COLS_PLANE) = u32x2{turn(w[0][c >> 1].l, w[1][c >> 1].l), turn(w[2][c >> 1].l, w[3][c >> 1].l)};
            }
        }
    }
};

template <int DT>
__global__ __launch_bounds__(256, DT <= 64 ? 2 : 1) void sdpa_window_dq_f32(const float *__restrict__ q, const float *__restrict__ k,
                                                                            const float *__restrict__ v, const float *__restrict__ out,
                                                                            const float *__restrict__ stats,
                                                                            const float *__restrict__ dout, float *__restrict__ dq,
                                                                            float *__restrict__ delta, const WindowGeometry g) {
    typedef Tile<32, DT> T;
    extern __shared__ __align__(16) u16 window_lds[];
    u16 *Ks = window_lds, *Vs = Ks + 3 * T::ROWS_PLANE, *Kc = Vs + 3 * T::ROWS_PLANE;

    const int unit = (blockIdx.x & 7) * g.per_xcd + (blockIdx.x >> 3);
    if (unit >= g.units) return;
    const int qb = unit % g.nqb, pair = unit / g.nqb;
    const int parts = g.group / g.hp;
    const int part = pair % parts, hk = (pair / parts) % g.Hkv, b = pair / parts / g.Hkv;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, half = lane >> 5, ln = lane & 31;
    const int h = hk * g.group + part * g.hp + wave % g.hp;
    const int rows = 128 / g.hp;
    const int q0 = qb * rows + wave / g.hp * 32, qi = q0 + ln, qc = qi < g.Lq ? qi : g.Lq - 1;
    const int len = valid_keys(g.w, b, g.Lk);

    const long long wp0 = g.w.q_offset + qb * rows, wp1 = g.w.q_offset + min(qb * rows + rows, g.Lq) - 1;
    const int end = (int)((min(wp1 + 1, (long long)len) + 31) / 32);
    const long long low = wp0 - g.w.window + 1;
    const int lo = (int)min((long long)end, low > 0 ? low / 32 : 0), first = min(lo, (g.w.sinks + 31) / 32);
    const int tiles = first + (end - lo);

    const float *kp = k + b * g.lk.b + hk * g.lk.h, *vp = v + b * g.lk.b + hk * g.lk.h;
    Pair<DT> kv;
    if (tiles > 0) kv.load(kp, vp, g.lk.l, (0 < first ? 0 : lo) * 32, len, g.d, g.vec);

    const long long at = b * g.lq.b + h * g.lq.h + qc * g.lq.l, row = ((long long)b * g.H + h) * g.Lq + qc;
    Frag qf[DT / 16], gf[DT / 16];
    float del = 0.f;
#pragma unroll
    for (int s = 0; s < DT / 16; ++s) {
        float z[8], y[8];
#pragma unroll
        for (int e = 0; e < 8; e += 4) {
            const f32x4 a = load4(q + at, 16 * s + 8 * half + e, g.d, g.vec), c = load4(dout + at, 16 * s + 8 * half + e, g.d, g.vec),
                        o = load4(out + at, 16 * s + 8 * half + e, g.d, g.vec);
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                z[e + x] = (a[x] * g.rT) * LOG2E;
                y[e + x] = c[x];
                del += c[x] * o[x];
            }
        }
        qf[s] = split8(z);
        gf[s] = split8(y);
    }
    del = sum_halves(del);
    const float m = stats[2 * row], inv = stats[2 * row + 1];
    if (half == 0 && qi < g.Lq) delta[row] = del;
    const long long p0 = g.w.q_offset + q0, p1 = g.w.q_offset + min(q0 + 31, g.Lq - 1), p = g.w.q_offset + qi;
    const bool idle = q0 >= g.Lq;

    f32x16 acc[DT / 32];
#pragma unroll
    for (int t = 0; t < DT / 32; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[t][r] = 0.f;

    for (int i = 0; i < tiles; ++i) {
        __syncthreads();
        kv.template store<true, false>(Ks, Kc, Vs, nullptr, 1.0f, 1.0f);
        __syncthreads();
        if (i + 1 < tiles) kv.load(kp, vp, g.lk.l, (i + 1 < first ? i + 1 : lo + i + 1 - first) * 32, len, g.d, g.vec);
        const int k0 = (i < first ? i : lo + i - first) * 32;
        if (idle || tile_hidden(g.w, p0, p1, k0, len)) continue;
        f32x16 s, dp;
#pragma unroll
        for (int r = 0; r < 16; ++r) { s[r] = 0.f; dp[r] = 0.f; }
#pragma unroll
        for (int st = 0; st < DT / 16; ++st) {
            s = mma6(T::rows_frag(Ks, 0, st), qf[st], s);
            dp = mma6(T::rows_frag(Vs, 0, st), gf[st], dp);
        }
        if (!tile_open(g.w, p0, p1, k0, len)) {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int j = k0 + acc_row(r) + 4 * half;
                if (!(j <= p && j < len && (j > p - g.w.window || j < g.w.sinks))) s[r] = -INFINITY;
            }
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = (exp2_fast(s[r] - m) * inv) * (dp[r] - del);
#pragma unroll
        for (int st = 0; st < 2; ++st) {
            const Frag f = acc_frag(s, st);
#pragma unroll
            for (int t = 0; t < DT / 32; ++t) acc[t] = mma6(T::cols_frag(Kc, t, st), f, acc[t]);
        }
    }

    if (qi >= g.Lq) return;
#pragma unroll
    for (int t = 0; t < DT / 32; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r)
            store4(dq + at, 32 * t + 8 * r + 4 * half, g.d, g.vec,
                   f32x4{acc[t][4 * r] * g.rT, acc[t][4 * r + 1] * g.rT, acc[t][4 * r + 2] * g.rT, acc[t][4 * r + 3] * g.rT});
}

// How the key blocks (128 keys) of all (batch, key head) pairs are dealt to workgroups: those that hold visible first keys,
// then the others; each in `chunks` equal pieces of its query tiles.  Workgroup ids of a class go round the XCDs so that
// consecutive pieces of work share one XCD's L2.
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

template <int DT>
__global__ __launch_bounds__(256, DT <= 64 ? 2 : 1) void sdpa_window_dkv_f32(const float *__restrict__ q, const float *__restrict__ k,
                                                                             const float *__restrict__ v,
                                                                             const float *__restrict__ stats,
                                                                             const float *__restrict__ dout,
                                                                             const float *__restrict__ delta, float *__restrict__ dk,
                                                                             float *__restrict__ dv, const WindowGeometry g,
                                                                             const KeyBlocks kb) {
    typedef Tile<32, DT> T;
    extern __shared__ __align__(16) u16 window_lds[];
    u16 *Qs = window_lds, *Gs = Qs + 3 * T::ROWS_PLANE, *Qc = Gs + 3 * T::ROWS_PLANE, *Gc = Qc + 3 * T::COLS_PLANE;
    float *rowv = reinterpret_cast<float *>(Gc + 3 * T::COLS_PLANE);            // [3][32]: m, 1 / l, delta of the tile's queries

    int id = blockIdx.x, cl = 0;
    if (id >= 8 * kb.per_xcd[0]) { id -= 8 * kb.per_xcd[0]; cl = 1; }
    const int unit = (id & 7) * kb.per_xcd[cl] + (id >> 3);
    if (unit >= kb.units[cl]) return;
    const int chunk = unit % kb.chunks[cl], in_class = cl ? kb.blocks - kb.sink_blocks : kb.sink_blocks;
    const int block = unit / kb.chunks[cl] % in_class + (cl ? kb.sink_blocks : 0), pair = unit / kb.chunks[cl] / in_class;
    const int hk = pair % g.Hkv, b = pair / g.Hkv;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, half = lane >> 5, ln = lane & 31;
    const int b0 = block * 128, k0 = b0 + wave * 32, key = k0 + ln;
    const int len = valid_keys(g.w, b, g.Lk);

    // query tiles that can see the block: from the first key's position to the window's end behind the last key
    const long long i0 = b0 - g.w.q_offset, i1 = b0 < g.w.sinks ? g.Lq : b0 + 127ll + g.w.window - g.w.q_offset;
    const int t0 = i0 > 0 ? (int)min((long long)g.Lq, i0) / 32 : 0, t1 = (int)((max(0ll, min(i1, (long long)g.Lq)) + 31) / 32);
    const int per_head = b0 < len && t1 > t0 ? t1 - t0 : 0;
    const int all = per_head * g.group, from = (int)((long long)all * chunk / kb.chunks[cl]), to = (int)((long long)all * (chunk + 1) / kb.chunks[cl]);

    Pair<DT> qg;
    float sv = 0.f;
    auto load = [&](const int e) {
        const int h = hk * g.group + e / per_head, r0 = (t0 + e % per_head) * 32;
        qg.load(q + b * g.lq.b + h * g.lq.h, dout + b * g.lq.b + h * g.lq.h, g.lq.l, r0, g.Lq, g.d, g.vec);
        if (threadIdx.x < 96) {
            const int which = threadIdx.x >> 5, r = r0 + (threadIdx.x & 31);
            const long long row = ((long long)b * g.H + h) * g.Lq + r;
            sv = r < g.Lq ? (which == 2 ? delta[row] : stats[2 * row + which]) : 0.f;
        }
    };
    if (from < to) load(from);

    Frag kf[DT / 16], vf[DT / 16];
    {
        const long long at = b * g.lk.b + hk * g.lk.h + key * g.lk.l;
#pragma unroll
        for (int s = 0; s < DT / 16; ++s) {
            float z[8], y[8];
#pragma unroll
            for (int e = 0; e < 8; e += 4) {
                f32x4 a = {0.f, 0.f, 0.f, 0.f}, c = a;
                if (key < len) {
                    a = load4(k + at, 16 * s + 8 * half + e, g.d, g.vec);
                    c = load4(v + at, 16 * s + 8 * half + e, g.d, g.vec);
                }
#pragma unroll
                for (int x = 0; x < 4; ++x) { z[e + x] = a[x]; y[e + x] = c[x]; }
            }
            kf[s] = split8(z);
            vf[s] = split8(y);
        }
    }

    f32x16 ak[DT / 32], av[DT / 32];
#pragma unroll
    for (int t = 0; t < DT / 32; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) { ak[t][r] = 0.f; av[t][r] = 0.f; }

    for (int e = from; e < to; ++e) {
        __syncthreads();
        qg.template store<true, true>(Qs, Qc, Gs, Gc, g.rT, LOG2E);
        if (threadIdx.x < 96) rowv[threadIdx.x] = sv;
        __syncthreads();
        if (e + 1 < to) load(e + 1);
        const int q0 = (t0 + e % per_head) * 32;
        const long long p0 = g.w.q_offset + q0, p1 = g.w.q_offset + min(q0 + 31, g.Lq - 1);
        if (tile_hidden(g.w, p0, p1, k0, len)) continue;
        f32x16 s, dp;
#pragma unroll
        for (int r = 0; r < 16; ++r) { s[r] = 0.f; dp[r] = 0.f; }
#pragma unroll
        for (int st = 0; st < DT / 16; ++st) {
            s = mma6(T::rows_frag(Qs, 0, st), kf[st], s);
            dp = mma6(T::rows_frag(Gs, 0, st), vf[st], dp);
        }
        const bool open = tile_open(g.w, p0, p1, k0, len) && q0 + 32 <= g.Lq;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const f32x4 m = *reinterpret_cast<const f32x4 *>(rowv + 8 * x + 4 * half), inv = *reinterpret_cast<const f32x4 *>(rowv + 32 + 8 * x + 4 * half),
                        del = *reinterpret_cast<const f32x4 *>(rowv + 64 + 8 * x + 4 * half);
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                const int r = 4 * x + y;
                float w = exp2_fast(s[r] - m[y]) * inv[y];
                if (!open) {
                    const int i = q0 + 8 * x + 4 * half + y;
                    const long long p = g.w.q_offset + i;
                    if (!(i < g.Lq && key <= p && key < len && (key > p - g.w.window || key < g.w.sinks))) w = 0.f;
                }
                s[r] = w;
                dp[r] = w * (dp[r] - del[y]);
            }
        }
#pragma unroll
        for (int st = 0; st < 2; ++st) {
            const Frag wf = acc_frag(s, st), df = acc_frag(dp, st);
#pragma unroll
            for (int t = 0; t < DT / 32; ++t) {
                av[t] = mma6(T::cols_frag(Gc, t, st), wf, av[t]);
                ak[t] = mma6(T::cols_frag(Qc, t, st), df, ak[t]);
            }
        }
    }

    if (key >= g.Lk) return;
    // q was staged as q rT log2(e): dk = rT sum dS q = ln(2) of what was summed
    constexpr float LN2 = 0.69314718055994530942f;
    const bool whole = kb.chunks[cl] == 1;
    const long long at = b * g.lk.b + hk * g.lk.h + key * g.lk.l;
    float *part = whole ? nullptr : partial_sums(kb, pair, block, chunk, g.d) + (wave * 32 + ln) * (long long)g.d;
    float *ok = whole ? dk + at : part, *ov = whole ? dv + at : part + 128ll * g.d;
#pragma unroll
    for (int t = 0; t < DT / 32; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            store4(ok, 32 * t + 8 * r + 4 * half, g.d, g.vec,
                   f32x4{ak[t][4 * r] * LN2, ak[t][4 * r + 1] * LN2, ak[t][4 * r + 2] * LN2, ak[t][4 * r + 3] * LN2});
            store4(ov, 32 * t + 8 * r + 4 * half, g.d, g.vec, f32x4{av[t][4 * r], av[t][4 * r + 1], av[t][4 * r + 2], av[t][4 * r + 3]});
        }
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
