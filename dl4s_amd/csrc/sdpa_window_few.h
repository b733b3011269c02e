// Windowed attention for few query rows: a decoding step over a cache, the last rows of a prompt, short prompts; and the forward
// pass above 128 columns.
//
// What bounds it is reading the visible keys and values once from HBM.  One wavefront takes 16 keys at a time for up to 16
// query rows of one key head (the heads of a group, and their rows): S[key, row] = K . Q^T and O[column, row] += V^T . P on
// v_mfma_f32_16x16x4_f32, whose layouts let K and V come straight from memory into the operands, four floats per lane, and
// the weights pass from the first product's accumulators into the second as they are:
//   A of S:  lane l holds key l % 16, columns 16 s + 4 (l / 16) .. + 3     (any order of the contraction serves, Q has the same)
//   S:       lane l holds row l % 16, keys 4 (l / 16) + r
//   A of O:  step r contracts over the keys 4 (l / 16) + r; lane l holds columns 64 j + 4 (l % 16) + e, e = 0 .. 3
// At 32 cycles per instruction a wavefront needs 4 cycles for 16 bytes of K or V whatever the number of rows (up to 16), about
// 16 TB/s over the chip: well above what HBM delivers.  Vector-ALU dot products would need as much for two rows.
// Measured: B32 H32/8 T30001 d128 window 4096 176 us (6.1 TB/s over the visible rows; a plain read reaches 6.6 to 6.9), B16 H16 T4096
// d64 window 1024 27 us (4.9 TB/s; some 6 us of it are the launch, the first loads and the merge).
// Wavefronts and, where (batch, key head) pairs do not fill the GPU, workgroups share the keys; partial results are merged
// with the usual softmax rescaling, in LDS and by a second small kernel.
#pragma once
#include "sdpa_window_common.h"

namespace {

struct FewArgs {
    int H, Hkv, group, Lq, Lk, d, cols;      // cols = group * Lq query rows of a key head: row c = query c / group, head c % group
    float rT;
    int vec;
    Layout lq, lk;
    WindowArgs w;
    int nsplit, chunk;                       // visible keys per workgroup (a multiple of 16)
    int pair0;                               // (batch, key head) pair of blockIdx.y = 0
    float *partial;                          // [pair][split][cols][d + 2], with nsplit > 1
};

template <int DT, int NW>
__global__ __launch_bounds__(NW * 64, DT <= 64 ? 3 : (DT <= 128 ? 2 : 1)) void sdpa_window_few_f32(
    const float *__restrict__ q, const float *__restrict__ k, const float *__restrict__ v, float *__restrict__ out,
    float *__restrict__ stats, const FewArgs a) {
    extern __shared__ __align__(16) float few_lds[];
    const int split = blockIdx.x % a.nsplit, c0 = blockIdx.x / a.nsplit * 16, nc = min(16, a.cols - c0), pair = a.pair0 + blockIdx.y;
    const int hk = pair % a.Hkv, b = pair / a.Hkv;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, ln = lane & 15, quad = lane >> 4;
    const int len = valid_keys(a.w, b, a.Lk);

    // the keys any of these rows sees: [0, first) and [lo, hi); x counts through both
    const Range r0 = visible_keys(a.w, b, c0 / a.group, a.Lk), r1 = visible_keys(a.w, b, (c0 + nc - 1) / a.group, a.Lk);
    const int lo = r0.lo, first = min(a.w.sinks, lo), hi = r1.hi, seen = first + max(0, hi - lo);
    const int x0 = split * a.chunk, x1 = min(seen, x0 + a.chunk);

    const int col = c0 + min(ln, nc - 1), hq = hk * a.group + col % a.group, iq = col / a.group;
    const int p = a.w.last_key ? len - 1 : a.w.q_offset + iq;
    float qf[DT / 4];
    {
        const float *qp = q + b * a.lq.b + hq * a.lq.h + iq * a.lq.l;
#pragma unroll
        for (int s = 0; s < DT / 16; ++s) {
            const f32x4 x = load4(qp, 16 * s + 4 * quad, a.d, a.vec);
#pragma unroll
            for (int e = 0; e < 4; ++e) qf[4 * s + e] = (x[e] * a.rT) * LOG2E;
        }
    }
    const float *kp = k + b * a.lk.b + hk * a.lk.h, *vp = v + b * a.lk.b + hk * a.lk.h;

    f32x4 o[DT / 64][4];
#pragma unroll
    for (int j = 0; j < DT / 64; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[j][e] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m_run = -INFINITY, m_use = 0.f, l_run = 0.f;

    // a row's four floats: this workgroup does not read them again (others of the same key head do, if it has more than 16 query rows)
    auto stream4 = [&](const float *row, const int c) -> f32x4 {
        if (!a.vec) return load4(row, c, a.d, false);
        return c < a.d ? __builtin_nontemporal_load(reinterpret_cast<const f32x4 *>(row + c)) : f32x4{0.f, 0.f, 0.f, 0.f};
    };
    struct Keys {
        f32x4 k[DT / 16], v[4][DT / 64];
    };
    auto key_at = [&](const int i) { const int y = min(i, x1 - 1); return y < first ? y : lo + y - first; };
    auto fetch = [&](Keys &f, const int x) {
        const float *kr = kp + key_at(x + ln) * a.lk.l;
#pragma unroll
        for (int s = 0; s < DT / 16; ++s) f.k[s] = stream4(kr, 16 * s + 4 * quad);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float *vr = vp + key_at(x + 4 * quad + r) * a.lk.l;
#pragma unroll
            for (int j = 0; j < DT / 64; ++j) f.v[r][j] = stream4(vr, 64 * j + 4 * ln);
        }
    };
    auto attend = [&](const Keys &f, const int x) {
        f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int t = 0; t < DT / 16; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) s = __builtin_amdgcn_mfma_f32_16x16x4f32(f.k[t][e], qf[4 * t + e], s, 0, 0, 0);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int j = key_at(x + 4 * quad + r);
            s[r] = ((x + 4 * quad + r < x1) & sees(a.w, p, j, len)) ? s[r] : -INFINITY;
        }
        const float tmax = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
        // the reference maximum, one per row and shared by its four lanes, moves only when a weight would pass 2^8
        if (__any(tmax - m_run > 8.0f)) {
            float m_new = fmaxf(m_run, tmax);
            m_new = fmaxf(m_new, __shfl_xor(m_new, 16, 64));
            m_new = fmaxf(m_new, __shfl_xor(m_new, 32, 64));
            const float alpha = m_run == m_new ? 1.0f : exp2_fast(m_run - m_new);
            m_run = m_new;
            m_use = m_new == -INFINITY ? 0.f : m_new;
            l_run *= alpha;
#pragma unroll
            for (int j = 0; j < DT / 64; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[j][e] *= alpha;
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            s[r] = exp2_fast(s[r] - m_use);
            l_run += s[r];
#pragma unroll
            for (int j = 0; j < DT / 64; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[j][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(f.v[r][j][e], s[r], o[j][e], 0, 0, 0);
        }
    };
    // the next 16 keys are on their way while these are worked on (rows above 128 columns: no registers for that)
    constexpr int STEP = 16 * NW;
    int x = x0 + 16 * wave;
    if (DT <= 128) {
        Keys f0, f1;
        if (x < x1) fetch(f0, x);
        for (; x < x1; x += 2 * STEP) {
            fetch(f1, x + STEP);
            attend(f0, x);
            if (x + STEP >= x1) break;
            fetch(f0, x + 2 * STEP);
            attend(f1, x + STEP);
        }
    } else {
        Keys f;
        for (; x < x1; x += STEP) {
            fetch(f, x);
            attend(f, x);
        }
    }
    l_run += __shfl_xor(l_run, 16, 64);
    l_run += __shfl_xor(l_run, 32, 64);

    // merge the wavefronts: [wave][row][DT + 4], the last four: m, l
    constexpr int STR = DT + 4;
    if (ln < nc) {
        float *w = few_lds + (wave * nc + ln) * STR;
#pragma unroll
        for (int j = 0; j < DT / 64; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                *reinterpret_cast<f32x4 *>(w + 64 * j + 4 * (4 * quad + r)) = f32x4{o[j][0][r], o[j][1][r], o[j][2][r], o[j][3][r]};
        if (quad == 0) { w[DT] = m_run; w[DT + 1] = l_run; }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < nc * DT; e += NW * 64) {
        const int c = e / DT, x = e % DT;
        if (x >= a.d) continue;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < NW; ++w) M = fmaxf(M, few_lds[(w * nc + c) * STR + DT]);
        const float Mu = M == -INFINITY ? 0.f : M;
        float L = 0.f, O = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float *part = few_lds + (w * nc + c) * STR;
            // a part that saw no finite score holds zeros, or NaN, which must survive
            const float f = part[DT] == -INFINITY ? 1.0f : exp2_fast(part[DT] - Mu);
            L += part[DT + 1] * f;
            O += part[x] * f;
        }
        const int row = c0 + c;
        if (a.nsplit > 1) {
            float *rec = a.partial + (((long long)pair * a.nsplit + split) * a.cols + row) * (a.d + 2);
            rec[x] = O;
            if (x == 0) { rec[a.d] = M; rec[a.d + 1] = L; }
        } else {
            const int h = hk * a.group + row % a.group, i = row / a.group;
            const Range r = visible_keys(a.w, b, i, a.Lk);
            const float inv = r.first + (r.hi - r.lo) > 0 ? 1.0f / L : 0.f;
            out[b * a.lq.b + h * a.lq.h + i * a.lq.l + x] = O * inv;
            if (stats && x == 0) {
                const long long at = 2 * (((long long)b * a.H + h) * a.Lq + i);
                stats[at] = Mu;
                stats[at + 1] = inv;
            }
        }
    }
}

constexpr int MAX_SPLIT = 256;

// Merges the partial results of one query row: one workgroup per row.  A thread has one part's maximum and sum, then one column of
// all parts, whose loads do not wait for each other.
__global__ __launch_bounds__(MAX_SPLIT) void sdpa_window_merge_f32(float *__restrict__ out, float *__restrict__ stats, const FewArgs a) {
    __shared__ float factor[MAX_SPLIT], most[4], total[4];
    const int row = blockIdx.x, pair = a.pair0 + blockIdx.y, x = threadIdx.x, wave = x >> 6;
    const int hk = pair % a.Hkv, b = pair / a.Hkv, h = hk * a.group + row % a.group, i = row / a.group;
    const long long step = (long long)a.cols * (a.d + 2);
    const float *rec = a.partial + ((long long)pair * a.nsplit * a.cols + row) * (a.d + 2);
    const float m = x < a.nsplit ? rec[x * step + a.d] : -INFINITY, l = x < a.nsplit ? rec[x * step + a.d + 1] : 0.f;
    float M = m;
#pragma unroll
    for (int o = 32; o; o >>= 1) M = fmaxf(M, __shfl_xor(M, o, 64));
    if ((x & 63) == 0) most[wave] = M;
    __syncthreads();
    M = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3]));
    const float Mu = M == -INFINITY ? 0.f : M, f = m == -INFINITY ? 1.0f : exp2_fast(m - Mu);
    factor[x] = f;
    const float part = dl4s::wave_sum(l * f);
    if ((x & 63) == 0) total[wave] = part;
    __syncthreads();
    const float L = (total[0] + total[1]) + (total[2] + total[3]);
    const Range r = visible_keys(a.w, b, i, a.Lk);
    const float inv = r.first + (r.hi - r.lo) > 0 ? 1.0f / L : 0.f;
    if (x < a.d) {
        float O = 0.f;
        int s = 0;
        for (; s + 8 <= a.nsplit; s += 8) {
            float p[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) p[e] = rec[(s + e) * step + x];
#pragma unroll
            for (int e = 0; e < 8; ++e) O += p[e] * factor[s + e];
        }
        for (; s < a.nsplit; ++s) O += rec[s * step + x] * factor[s];
        out[b * a.lq.b + h * a.lq.h + i * a.lq.l + x] = O * inv;
    }
    if (stats && x == 0) {
        const long long at = 2 * (((long long)b * a.H + h) * a.Lq + i);
        stats[at] = Mu;
        stats[at + 1] = inv;
    }
}

}  // namespace
