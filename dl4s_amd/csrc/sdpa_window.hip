// Attention with a sliding window and visible first keys for gfx950: forward, gradients, one decoding step over a cache.
//
// Query i of batch element b stands at position p = q_offset + i and sees the keys
//   V(i) = { j : j <= p,  j > p - window or j < sinks,  j < lengths[b] }
//   s_ij = (q_i * rT) . k_j,   w_ij = exp(s_ij) / sum over V(i) of exp(s_ij'),   out_i = sum over V(i) of w_ij v_j
// and a row that sees no key has weights and output zero.  H / Hkv consecutive query heads share a key head.  Gradients:
//   dv_j = sum_i w_ij dout_i,  dS_ij = w_ij (dout_i . v_j - dout_i . out_i),  dq_i = rT sum_j dS_ij k_j,
//   dk_j = rT sum_i dS_ij q_i  (dk, dv summed over the query heads of the group)
#include <algorithm>
#include <initializer_list>

#include "sdpa_window_bwd.h"
#include "sdpa_window_few.h"

namespace {

// delta_i = dout_i . out_i, one wavefront per row
__global__ __launch_bounds__(256) void window_delta_f32(const float *__restrict__ dout, const float *__restrict__ out,
                                                         float *__restrict__ delta, int H, int Lq, int d, Layout lq, long long rows) {
    const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= rows) return;
    const int lane = threadIdx.x & 63;
    const long long bh = row / Lq, at = (bh / H) * lq.b + (bh % H) * lq.h + (row % Lq) * lq.l;
    float s = 0.f;
    for (int c = lane; c < d; c += 64) s += dout[at + c] * out[at + c];
    s = dl4s::wave_sum(s);
    if (lane == 0) delta[row] = s;
}

// dq: one wavefront per query row, the walk of the forward kernel
__global__ __launch_bounds__(256) void sdpa_window_dq_rows_f32(const float *__restrict__ q, const float *__restrict__ k,
                                                                const float *__restrict__ v, const float *__restrict__ dout,
                                                                const float *__restrict__ stats, const float *__restrict__ delta,
                                                                float *__restrict__ dq, int H, int group, int Lq, int Lk, int d,
                                                                float rT, WindowArgs w, Layout lq, Layout lk, long long rows) {
    __shared__ float qs[4][MAXD], gs[4][MAXD], ps[4][64];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const long long row = (long long)blockIdx.x * 4 + wave;
    if (row >= rows) return;
    const int i = (int)(row % Lq);
    const long long bh = row / Lq;
    const int h = (int)(bh % H), b = (int)(bh / H);
    const long long at = b * lq.b + h * lq.h + i * lq.l;
    const float *kp = k + b * lk.b + (h / group) * lk.h, *vp = v + b * lk.b + (h / group) * lk.h;
    for (int c = lane; c < d; c += 64) {
        qs[wave][c] = q[at + c] * rT;
        gs[wave][c] = dout[at + c];
    }
    const Range r = visible_keys(w, b, i, Lk);
    const float m = stats[2 * row], inv = stats[2 * row + 1], del = delta[row];
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    for (int part = 0; part < 2; ++part) {
        const int end = part ? r.hi : r.first;
        for (int j0 = part ? r.lo : 0; j0 < end; j0 += 64) {
            const int n = min(64, end - j0);
            float ds = 0.f;
            if (lane < n) {
                const float *kr = kp + (long long)(j0 + lane) * lk.l, *vr = vp + (long long)(j0 + lane) * lk.l;
                float s = 0.f, g = 0.f;
                for (int c = 0; c < d; ++c) { s += qs[wave][c] * kr[c]; g += gs[wave][c] * vr[c]; }
                ds = __builtin_amdgcn_exp2f(s * LOG2E - m) * inv * (g - del);
            }
            ps[wave][lane] = ds;
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const int c = lane + 64 * t;
                if (c >= d) break;
                for (int x = 0; x < n; ++x) acc[t] += ps[wave][x] * kp[(long long)(j0 + x) * lk.l + c];
            }
        }
    }
#pragma unroll
    for (int t = 0; t < 4; ++t)
        if (lane + 64 * t < d) dq[at + lane + 64 * t] = acc[t] * rT;
}

// dk, dv: one wavefront per key row, over the queries of the group's heads that can see it, 64 at a time
__global__ __launch_bounds__(256) void sdpa_window_dkv_rows_f32(const float *__restrict__ q, const float *__restrict__ k,
                                                                 const float *__restrict__ v, const float *__restrict__ dout,
                                                                 const float *__restrict__ stats, const float *__restrict__ delta,
                                                                 float *__restrict__ dk, float *__restrict__ dv, int H, int Hkv,
                                                                 int Lq, int Lk, int d, float rT, WindowArgs w, Layout lq, Layout lk,
                                                                 long long rows) {
    __shared__ float ks[4][MAXD], vs[4][MAXD], ps[4][64], ss[4][64];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const long long row = (long long)blockIdx.x * 4 + wave;
    if (row >= rows) return;
    const int j = (int)(row % Lk), group = H / Hkv;
    const long long bh = row / Lk;
    const int hk = (int)(bh % Hkv), b = (int)(bh / Hkv);
    const long long at = b * lk.b + hk * lk.h + j * lk.l;
    for (int c = lane; c < d; c += 64) {
        ks[wave][c] = k[at + c];
        vs[wave][c] = v[at + c];
    }
    int len = w.lengths ? w.lengths[b] : Lk;
    len = len > Lk ? Lk : len;
    // positions that see key j: from j on, to the window's end unless the key is one of the first
    long long i0 = (long long)j - w.q_offset, i1 = j < w.sinks ? Lq : (long long)j + w.window - w.q_offset;
    if (i0 < 0) i0 = 0;
    if (i1 > Lq) i1 = Lq;
    if (j >= len) i1 = i0;
    float ak[4] = {0.f, 0.f, 0.f, 0.f}, av[4] = {0.f, 0.f, 0.f, 0.f};
    for (int h = hk * group; h < (hk + 1) * group; ++h) {
        const long long base = b * lq.b + h * lq.h, srow = ((long long)b * H + h) * Lq;
        for (int q0 = (int)i0; q0 < i1; q0 += 64) {
            const int n = (int)min(64ll, i1 - q0);
            float p = 0.f, ds = 0.f;
            if (lane < n) {
                const float *qr = q + base + (long long)(q0 + lane) * lq.l, *gr = dout + base + (long long)(q0 + lane) * lq.l;
                float s = 0.f, g = 0.f;
                for (int c = 0; c < d; ++c) { s += qr[c] * rT * ks[wave][c]; g += gr[c] * vs[wave][c]; }
                const long long sr = srow + q0 + lane;
                p = __builtin_amdgcn_exp2f(s * LOG2E - stats[2 * sr]) * stats[2 * sr + 1];
                ds = p * (g - delta[sr]);
            }
            ps[wave][lane] = p;
            ss[wave][lane] = ds;
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const int c = lane + 64 * t;
                if (c >= d) break;
                for (int x = 0; x < n; ++x) {
                    const long long a = base + (long long)(q0 + x) * lq.l + c;
                    av[t] += ps[wave][x] * dout[a];
                    ak[t] += ss[wave][x] * q[a];
                }
            }
        }
    }
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        const int c = lane + 64 * t;
        if (c < d) { dk[at + c] = ak[t] * rT; dv[at + c] = av[t]; }
    }
}

inline Layout layout(bool token_major, int64_t heads, int64_t L, int64_t d) {
    return token_major ? Layout{L * heads * d, d, heads * d} : Layout{heads * L * d, L * d, d};
}
inline dim3 row_grid(long long rows) { return dim3((unsigned)((rows + 3) / 4)); }
// A launch has fewer than 2^32 threads along its first axis: refused before anything is launched.
inline int fits_a_launch(const char *what, long long workgroups, int threads) {
    DL4S_REQUIRE(workgroups < (1ll << 32) / threads, DL4S_HIP_EUNSUPPORTED, "%s: %lld workgroups of %d threads", what, workgroups, threads);
    return DL4S_HIP_OK;
}

inline bool on_16_bytes(std::initializer_list<const void *> ps) {
    uintptr_t bits = 0;
    for (const void *p : ps) bits |= reinterpret_cast<uintptr_t>(p);
    return (bits & 15) == 0;
}

// Query heads of a group that one workgroup takes together, and the rest of the launch.
WindowGeometry geometry(int64_t B, int64_t H, int64_t Hkv, int64_t Lq, int64_t Lk, int64_t d, float rT, bool token_major, const WindowArgs &w) {
    WindowGeometry g;
    g.H = (int)H; g.Hkv = (int)Hkv; g.group = (int)(H / Hkv); g.Lq = (int)Lq; g.Lk = (int)Lk; g.d = (int)d;
    g.hp = g.group % 4 == 0 ? 4 : (g.group % 2 == 0 ? 2 : 1);
    g.nqb = (int)((Lq + 128 / g.hp - 1) / (128 / g.hp));
    g.units = (int)(B * Hkv * (g.group / g.hp) * g.nqb);
    g.per_xcd = (g.units + 7) / 8;
    g.rT = rT;
    g.lq = layout(token_major, H, Lq, d);
    g.lk = layout(token_major, Hkv, Lk, d);
    g.w = w;
    return g;
}

// Kernels with more than 64 KiB of LDS have their limit raised once per device.
template <typename K>
int lds_limit(dl4s_hip_ctx *ctx, int family, int kind, K kernel, size_t bytes) {
    if (bytes > 65536 && dl4s::lds_limit_pending(ctx, family, kind)) {
        DL4S_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
        dl4s::lds_limit_done(ctx, family, kind);
    }
    return DL4S_HIP_OK;
}

// Whether eight wavefronts share a workgroup's rows, four to a half of every tile of 64 keys (KS = 2), or four have them alone.
// They do while a compute unit has no second workgroup to run beside the first, and where there are more than three tiles
// (d 64, B1 H8 L1024 window 1024, 64 workgroups: forward 46 us with four, 36 with eight, gradients 106 and 89; window 128: 17
// and 16, 54 and 50; B4 H8 L2048, 512 workgroups: 73 and 81, 285 and 293; d 96, L64: gradients 27 and 28).
inline bool share_rows(const dl4s_hip_ctx *ctx, const WindowGeometry &g) {
    return g.units <= ctx->cu_count && std::min<long long>(g.Lk, (long long)g.w.window + g.w.sinks + 128 / g.hp - 1) > 192;
}

template <int DT, int BN, int KS, bool VEC>
int launch_fwd(dl4s_hip_ctx *ctx, const float *q, const float *k, const float *v, float *out, float *stats, const WindowGeometry &g) {
    typedef Tile<BN, DT> T;
    constexpr size_t lds = 2 * 2 * (T::ROWS_PLANE + T::COLS_PLANE);
    const int rc = lds_limit(ctx, dl4s::LDS_WINDOW_FWD, 2 * (DT / 32 - 1) + VEC, sdpa_window_fwd_f32<DT, BN, KS, VEC>, lds);
    if (rc) return rc;
    hipLaunchKernelGGL((sdpa_window_fwd_f32<DT, BN, KS, VEC>), dim3(8 * g.per_xcd), dim3(256 * KS), lds, ctx->stream, q, k, v, out, stats, g);
    return dl4s::launch_status("sdpa_window_fwd_f32");
}
template <bool VEC>
int launch_fwd_width(dl4s_hip_ctx *ctx, const float *q, const float *k, const float *v, float *out, float *stats, const WindowGeometry &g) {
    if (share_rows(ctx, g)) {
        if (g.d <= 32) return launch_fwd<32, 64, 2, VEC>(ctx, q, k, v, out, stats, g);
        if (g.d <= 64) return launch_fwd<64, 64, 2, VEC>(ctx, q, k, v, out, stats, g);
        if (g.d <= 96) return launch_fwd<96, 64, 2, VEC>(ctx, q, k, v, out, stats, g);
        return launch_fwd<128, 64, 2, VEC>(ctx, q, k, v, out, stats, g);
    }
    if (g.d <= 32) return launch_fwd<32, 64, 1, VEC>(ctx, q, k, v, out, stats, g);
    if (g.d <= 64) return launch_fwd<64, 64, 1, VEC>(ctx, q, k, v, out, stats, g);
    if (g.d <= 96) return launch_fwd<96, 32, 1, VEC>(ctx, q, k, v, out, stats, g);
    return launch_fwd<128, 32, 1, VEC>(ctx, q, k, v, out, stats, g);
}

// Deals the key blocks to workgroups, of which a compute unit has one at a time.  The blocks without first keys are cut into as
// many pieces as make the longest queue of a compute unit shortest (in query tiles: a workgroup costs about one more, a
// second launch that adds up partial sums about three, and their way through memory); those with first keys, which
// every later query sees, into enough pieces to give every compute unit one.  At most 2048 workgroups leave partial sums.
// beside: the workgroups share the GPU with those of dq; they are to be no more than the compute units that those leave.
// *partial_bytes: what the partial sums take (1 KiB of d for each workgroup that leaves some); kb.partial is set by the caller.
KeyBlocks key_blocks(const dl4s_hip_ctx *ctx, const WindowGeometry &g, int64_t B, bool beside, size_t *partial_bytes) {
    KeyBlocks kb;
    kb.pairs = (int)(B * g.Hkv);
    kb.blocks = (g.Lk + 127) / 128;
    kb.sink_blocks = std::min(kb.blocks, (g.w.sinks + 127) / 128);
    const long long cus = ctx->cu_count - (beside ? g.units : 0), tiles = (g.Lq + 31) / 32, near = std::min<long long>(tiles, (g.w.window + 127ll + 31) / 32 + 1);
    const long long n[2] = {tiles * g.group, near * g.group}, count[2] = {(long long)kb.pairs * kb.sink_blocks, (long long)kb.pairs * (kb.blocks - kb.sink_blocks)};
    for (int c = 1; c >= 0; --c) {
        const long long most = std::max(1ll, std::min(n[c] / 4, 2048 / std::max(1ll, count[c])));
        long long chunks = 1;
        if (c == 0) {
            const long long left = beside ? cus - kb.units[1] : cus + count[0] - 1;
            chunks = std::min(most, std::max(1ll, left / std::max(1ll, count[0])));
        } else {
            double best = 0;
            for (long long x = 1; x <= std::min(most, 8ll); ++x) {
                const double queue = (double)((count[1] * x + cus - 1) / cus) * (double)((n[1] + x - 1) / x + 1);
                const double cost = queue + (x > 1 ? 3.0 + (double)(count[1] * x) * g.d * 2e-4 : 0.0);   // 2 KiB of d, at 5 TB/s and 2 us a tile
                if (x == 1 || cost < best) { best = cost; chunks = x; }
            }
        }
        kb.chunks[c] = (int)chunks;
        kb.units[c] = (int)(count[c] * chunks);
        kb.per_xcd[c] = (kb.units[c] + 7) / 8;
    }
    const long long floats0 = kb.chunks[0] > 1 ? kb.units[0] * 256ll * g.d : 0, floats1 = kb.chunks[1] > 1 ? kb.units[1] * 256ll * g.d : 0;
    kb.class1 = floats0;
    kb.partial = nullptr;
    *partial_bytes = (size_t)(floats0 + floats1) * sizeof(float);
    return kb;
}

template <int DT, int KS, bool VEC>
int launch_dq(dl4s_hip_ctx *ctx, const float *q, const float *k, const float *v, const float *out, const float *stats, const float *dout,
              float *dq, float *delta, const WindowGeometry &g) {
    typedef Tile<32 * KS, DT> T;
    const size_t lds = 2 * 2 * (2 * T::ROWS_PLANE + T::COLS_PLANE);
    const int rc = lds_limit(ctx, KS == 2 ? dl4s::LDS_WINDOW_DQ_SHARED : dl4s::LDS_WINDOW_DQ, 2 * (DT / 32 - 1) + VEC, sdpa_window_dq_f32<DT, KS, VEC>, lds);
    if (rc) return rc;
    hipLaunchKernelGGL((sdpa_window_dq_f32<DT, KS, VEC>), dim3(8 * g.per_xcd), dim3(256 * KS), lds, ctx->stream, q, k, v, out, stats, dout, dq, delta, g);
    return dl4s::launch_status("sdpa_window_dq_f32");
}

template <int DT, bool VEC>
int launch_bwd(dl4s_hip_ctx *ctx, const float *q, const float *k, const float *v, const float *out, const float *stats, const float *dout,
               float *dq, float *dk, float *dv, float *delta, const WindowGeometry &g, const KeyBlocks &kb, const bool beside) {
    typedef Tile<32, DT> T;
    const size_t lds_k = 2 * 2 * 4 * (T::ROWS_PLANE + T::COLS_PLANE) + 16384;
    int rc = DL4S_HIP_OK;
    if constexpr (DT <= 96) {
        typedef Tile<64, DT> T2;
        if (beside) {
            const size_t lds = std::max(lds_k, (size_t)(2 * 2 * (2 * T2::ROWS_PLANE + T2::COLS_PLANE)));
            rc = lds_limit(ctx, dl4s::LDS_WINDOW_DQ_DKV, 2 * (DT / 32 - 1) + VEC, sdpa_window_dq_dkv_f32<DT, VEC>, lds);
            if (rc) return rc;
            const long long rows = (long long)kb.pairs * g.group * g.Lq;
            hipLaunchKernelGGL(window_delta_f32, row_grid(rows), dim3(256), 0, ctx->stream, dout, out, delta, g.H, g.Lq, g.d, g.lq, rows);
            hipLaunchKernelGGL((sdpa_window_dq_dkv_f32<DT, VEC>), dim3(8 * (kb.per_xcd[0] + kb.per_xcd[1] + g.per_xcd)), dim3(512), lds, ctx->stream,
                               q, k, v, out, stats, dout, delta, dq, dk, dv, g, kb);
            rc = dl4s::launch_status("sdpa_window_dq_dkv_f32");
        }
    }
    if (!rc && !beside) rc = lds_limit(ctx, dl4s::LDS_WINDOW_DKV, 2 * (DT / 32 - 1) + VEC, sdpa_window_dkv_f32<DT, VEC>, lds_k);
    if (rc) return rc;
    if (!beside && g.units) {
        // (128 columns: two such wavefronts do not fit the registers of a SIMD)
        rc = DT <= 96 && share_rows(ctx, g) ? launch_dq<DT, DT <= 96 ? 2 : 1, VEC>(ctx, q, k, v, out, stats, dout, dq, delta, g)
                                                           : launch_dq<DT, 1, VEC>(ctx, q, k, v, out, stats, dout, dq, delta, g);
        if (rc) return rc;
    }
    if (kb.pairs && kb.blocks) {
        if (!beside) {
            hipLaunchKernelGGL((sdpa_window_dkv_f32<DT, VEC>), dim3(8 * (kb.per_xcd[0] + kb.per_xcd[1])), dim3(512), lds_k, ctx->stream, q, k, v, stats,
                               dout, delta, dk, dv, g, kb);
            rc = dl4s::launch_status("sdpa_window_dkv_f32");
        }
        for (int c = 0; c < 2 && !rc; ++c) {
            const int first = c ? kb.sink_blocks : 0, n = c ? kb.blocks - kb.sink_blocks : kb.sink_blocks;
            if (kb.chunks[c] == 1 || n == 0) continue;
            hipLaunchKernelGGL(sdpa_window_join_f32, dim3(g.d, n, kb.pairs), dim3(256), 0, ctx->stream, dk, dv, g, kb, first);
            rc = dl4s::launch_status("sdpa_window_join_f32");
        }
    }
    return rc;
}

template <bool VEC>
int launch_bwd_width(dl4s_hip_ctx *ctx, const float *q, const float *k, const float *v, const float *out, const float *stats,
                     const float *dout, float *dq, float *dk, float *dv, float *delta, const WindowGeometry &g, const KeyBlocks &kb,
                     const bool beside) {
    if (g.d <= 32) return launch_bwd<32, VEC>(ctx, q, k, v, out, stats, dout, dq, dk, dv, delta, g, kb, beside);
    if (g.d <= 64) return launch_bwd<64, VEC>(ctx, q, k, v, out, stats, dout, dq, dk, dv, delta, g, kb, beside);
    if (g.d <= 96) return launch_bwd<96, VEC>(ctx, q, k, v, out, stats, dout, dq, dk, dv, delta, g, kb, beside);
    return launch_bwd<128, VEC>(ctx, q, k, v, out, stats, dout, dq, dk, dv, delta, g, kb, beside);
}

// Few query rows: the workgroups and the split of the keys.  Lk is the number of rows that can be visible at all (T of a cache).
FewArgs few_args(int64_t B, int64_t H, int64_t Hkv, int64_t Lq, int64_t Lk, int64_t d, float rT, const WindowArgs &w, Layout lq, Layout lk,
                 int cus) {
    FewArgs a;
    a.H = (int)H; a.Hkv = (int)Hkv; a.group = (int)(H / Hkv); a.Lq = (int)Lq; a.Lk = (int)Lk; a.d = (int)d;
    a.cols = a.group * a.Lq;
    a.rT = rT;
    a.lq = lq; a.lk = lk; a.w = w;
    // Workgroups of 8 wavefronts and 16 rows.  Enough of them that every compute unit has one; a split costs a second launch, so
    // up to 512 keys one workgroup reads them all, and a workgroup has at least 256 keys.
    const int64_t queries = std::min<int64_t>(Lq, 14 / a.group + 2);         // of a workgroup's rows
    const int64_t most = std::min<int64_t>(Lk, (int64_t)w.window + queries - 1 + w.sinks), blocks = B * Hkv * ((a.cols + 15) / 16);
    const int64_t ns = most <= 512 ? 1 : std::min<int64_t>(MAX_SPLIT, std::min((cus + blocks - 1) / blocks, (most + 255) / 256));
    a.chunk = (int)std::max<int64_t>(16, ((most + ns - 1) / ns + 15) / 16 * 16);
    a.nsplit = (int)std::max<int64_t>(1, (most + a.chunk - 1) / a.chunk);
    a.partial = nullptr;
    a.pair0 = 0;
    return a;
}

template <int DT>
int launch_few_rows(dl4s_hip_ctx *ctx, const float *q, const float *k, const float *v, float *out, float *stats, FewArgs &a, int64_t pairs) {
    constexpr int NW = 8;
    const size_t of_row = (size_t)NW * (DT + 4) * sizeof(float), lds = std::min(16, a.cols) * of_row;
    const long long workgroups = (long long)a.nsplit * ((a.cols + 15) / 16);
    int rc = fits_a_launch("sdpa_window", workgroups, NW * 64);
    if (!rc) rc = lds_limit(ctx, dl4s::LDS_WINDOW_FEW, DT == 64 ? 0 : (DT == 128 ? 1 : 2), sdpa_window_few_f32<DT, NW>, 16 * of_row);
    for (int64_t from = 0; from < pairs && !rc; from += 65535) {
        const unsigned n = (unsigned)std::min<int64_t>(pairs - from, 65535);
        a.pair0 = (int)from;
        hipLaunchKernelGGL((sdpa_window_few_f32<DT, NW>), dim3((unsigned)workgroups, n), dim3(NW * 64), lds, ctx->stream, q, k, v, out, stats, a);
        rc = dl4s::launch_status("sdpa_window_few_f32");
        if (rc || a.nsplit == 1) continue;
        hipLaunchKernelGGL(sdpa_window_merge_f32, dim3(a.cols, n), dim3(MAX_SPLIT), 0, ctx->stream, out, stats, a);
        rc = dl4s::launch_status("sdpa_window_merge_f32");
    }
    return rc;
}

int few_rows(dl4s_hip_ctx *ctx, const float *q, const float *k, const float *v, float *out, float *stats, FewArgs &a, int64_t pairs) {
    a.vec = a.d % 4 == 0 && on_16_bytes({q, k, v});
    std::unique_lock<std::mutex> scratch_lock(ctx->scratch_mu, std::defer_lock);
    if (a.nsplit > 1) {
        scratch_lock.lock();
        const int rc = dl4s::ensure_scratch(ctx, (size_t)pairs * a.nsplit * a.cols * (a.d + 2) * sizeof(float));
        if (rc) return rc;
        a.partial = reinterpret_cast<float *>(ctx->scratch);
    }
    if (a.d <= 64) return launch_few_rows<64>(ctx, q, k, v, out, stats, a, pairs);
    if (a.d <= 128) return launch_few_rows<128>(ctx, q, k, v, out, stats, a, pairs);
    return launch_few_rows<256>(ctx, q, k, v, out, stats, a, pairs);
}

// What the three entry points check alike.  Returns a status; *w is filled in.
int window_checks(const char *what, int64_t B, int64_t H, int64_t Hkv, int64_t Lq, int64_t Lk, int64_t d, const dl4s_window_desc *desc,
                  uint32_t flags, WindowArgs *w) {
    DL4S_REQUIRE(B >= 0 && H >= 0 && Hkv >= 0 && Lq >= 0 && Lk >= 0, DL4S_HIP_EINVALID_ARG, "%s: negative extent", what);
    DL4S_REQUIRE(desc, DL4S_HIP_EINVALID_ARG, "%s: NULL window descriptor", what);
    DL4S_REQUIRE(desc->window >= 1 && desc->sinks >= 0 && desc->q_offset >= 0, DL4S_HIP_EINVALID_ARG,
                 "%s: window %lld must be at least 1, sinks %lld and q_offset %lld at least 0", what, (long long)desc->window,
                 (long long)desc->sinks, (long long)desc->q_offset);
    DL4S_REQUIRE(!(flags & ~DL4S_SDPA_TOKEN_MAJOR), DL4S_HIP_EINVALID_ARG, "%s: flags %#x (only DL4S_SDPA_TOKEN_MAJOR is known here)", what, flags);
    DL4S_REQUIRE(H == 0 || (Hkv > 0 && H % Hkv == 0), DL4S_HIP_ESHAPE, "%s: %lld query heads do not share %lld key heads evenly", what,
                 (long long)H, (long long)Hkv);
    DL4S_REQUIRE(d >= 1 && d <= MAXD, DL4S_HIP_EUNSUPPORTED, "%s: head dim %lld (1 to %d are implemented)", what, (long long)d, MAXD);
    const int64_t big = int64_t(1) << 30, most = big - 256;
    DL4S_REQUIRE(Lq <= most && Lk <= most && B < big && H < big && Hkv < big && B * H < big && B * Hkv < big && desc->q_offset <= most - Lq,
                 DL4S_HIP_EUNSUPPORTED, "%s: more than 2^30 heads, or a position above 2^30 - 256", what);
    DL4S_REQUIRE(H * d <= (int64_t(1) << 22), DL4S_HIP_EUNSUPPORTED, "%s: %lld heads of %lld: a token's heads above 2^22 values", what,
                 (long long)H, (long long)d);
    DL4S_REQUIRE(B * H * Lq < big * 4 && B * Hkv * Lk < big * 4, DL4S_HIP_EUNSUPPORTED, "%s: more than 2^32 rows", what);
    w->window = (int)(desc->window < big ? desc->window : big);
    w->sinks = (int)(desc->sinks < Lk ? desc->sinks : Lk);
    w->q_offset = (int)desc->q_offset;
    w->lengths = desc->lengths;
    w->last_key = 0;
    return DL4S_HIP_OK;
}

}  // namespace

extern "C" {

int dl4s_hip_sdpa_window_fwd_f32(dl4s_hip_ctx *ctx, const float *q, const float *k, const float *v, float *out, float *stats,
                                 int64_t B, int64_t H, int64_t Hkv, int64_t Lq, int64_t Lk, int64_t d, float inv_temperature,
                                 const dl4s_window_desc *window, uint32_t flags) {
    DL4S_CHECK_CTX(ctx);
    WindowArgs w;
    const int rc = window_checks("sdpa_window_fwd", B, H, Hkv, Lq, Lk, d, window, flags, &w);
    if (rc) return rc;
    const long long rows = (long long)B * H * Lq;
    if (rows == 0) return DL4S_HIP_OK;
    DL4S_REQUIRE(q && out && (Lk == 0 || (k && v)), DL4S_HIP_EINVALID_ARG, "sdpa_window_fwd: NULL tensor pointer");
    const bool tm = flags & DL4S_SDPA_TOKEN_MAJOR;
    const Layout lq = layout(tm, H, Lq, d), lk = layout(tm, Hkv, Lk, d);
    // The kernel for few rows takes 16 to a workgroup and shares their keys among wavefronts and workgroups; the other takes 128
    // and walks their keys in turn, on faster instructions.  While a compute unit gets at most one workgroup of the former it
    // is the faster one (d 64: 8 heads L 512 window 256 11 us against 22, 64 rows over 4096 keys 17 against 165, 512 workgroups
    // of a group of four 19 against 19, 1024 of them 36 against 19), as for 16 rows to a key head over long stretches (1024
    // key heads, 2048 keys: 180 us against 219, 500 keys: 64 against 60).  Above 128 columns it is the only one.
    const int64_t cols = H / Hkv * Lq, blocks = (cols + 15) / 16, most = std::min<int64_t>(Lk, (int64_t)w.window + w.sinks);
    if (d > 128 || B * Hkv * blocks <= ctx->cu_count || (cols <= 16 && most > 1024)) {
        if (const int bad = fits_a_launch("sdpa_window_fwd", blocks, 512)) return bad;
        FewArgs few = few_args(B, H, Hkv, Lq, Lk, d, inv_temperature, w, lq, lk, ctx->cu_count);
        return few_rows(ctx, q, k, v, out, stats, few, B * Hkv);
    }
    const WindowGeometry g = geometry(B, H, Hkv, Lq, Lk, d, inv_temperature, tm, w);
    if (const int bad = fits_a_launch("sdpa_window_fwd", 8ll * g.per_xcd, 256)) return bad;
    return d % 4 == 0 && on_16_bytes({q, k, v, out}) ? launch_fwd_width<true>(ctx, q, k, v, out, stats, g)
                                                     : launch_fwd_width<false>(ctx, q, k, v, out, stats, g);
}

int dl4s_hip_sdpa_window_bwd_f32(dl4s_hip_ctx *ctx, const float *q, const float *k, const float *v, const float *out,
                                 const float *stats, const float *dout, float *dq, float *dk, float *dv, int64_t B, int64_t H,
                                 int64_t Hkv, int64_t Lq, int64_t Lk, int64_t d, float inv_temperature, const dl4s_window_desc *window,
                                 uint32_t flags) {
    DL4S_CHECK_CTX(ctx);
    WindowArgs w;
    int rc = window_checks("sdpa_window_bwd", B, H, Hkv, Lq, Lk, d, window, flags, &w);
    if (rc) return rc;
    const long long rows = (long long)B * H * Lq, krows = (long long)B * Hkv * Lk;
    if (rows == 0 && krows == 0) return DL4S_HIP_OK;
    DL4S_REQUIRE((rows == 0 || (q && out && stats && dout && dq)) && (krows == 0 || (k && v && dk && dv)), DL4S_HIP_EINVALID_ARG,
                 "sdpa_window_bwd: NULL tensor pointer");
    const bool tm = flags & DL4S_SDPA_TOKEN_MAJOR;
    const Layout lq = layout(tm, H, Lq, d), lk = layout(tm, Hkv, Lk, d);
    std::unique_lock<std::mutex> scratch_lock(ctx->scratch_mu);
    const size_t delta_bytes = ((size_t)rows * sizeof(float) + 255) / 256 * 256;
    if (d <= 128 && H > 0) {
        const WindowGeometry g = geometry(B, H, Hkv, Lq, Lk, d, inv_temperature, tm, w);
        // dq and dk/dv run side by side, behind a small kernel for delta, where all their workgroups find a compute unit of
        // their own (d 64, one after the other and side by side: B4 H8 L512 window 128 50 us and 33, B1 H8 L2048 window 1024 117
        // and 94, L64 21 and 13; d 96: 67 and 42, 153 and 117, 26 and 16; with two workgroups to a compute unit, B4 H8 L1024
        // window 128, 53 and 57); above 96 columns dq needs a SIMD's registers alone
        bool beside = d <= 96 && rows && krows && 2 * g.units <= ctx->cu_count;
        size_t partial_bytes = 0;
        KeyBlocks kb = krows ? key_blocks(ctx, g, B, beside, &partial_bytes) : KeyBlocks{};
        if (beside && g.units + kb.units[0] + kb.units[1] > ctx->cu_count) {
            beside = false;
            kb = key_blocks(ctx, g, B, false, &partial_bytes);
        }
        rc = fits_a_launch("sdpa_window_bwd", std::max(8ll * g.per_xcd, 16ll * (kb.per_xcd[0] + kb.per_xcd[1])), 256);
        if (rc) return rc;
        rc = dl4s::ensure_scratch(ctx, delta_bytes + partial_bytes);
        if (rc) return rc;
        float *delta = reinterpret_cast<float *>(ctx->scratch);
        kb.partial = delta + delta_bytes / sizeof(float);
        return d % 4 == 0 && on_16_bytes({q, k, v, out, dout, dq, dk, dv})
                   ? launch_bwd_width<true>(ctx, q, k, v, out, stats, dout, dq, dk, dv, delta, g, kb, beside)
                   : launch_bwd_width<false>(ctx, q, k, v, out, stats, dout, dq, dk, dv, delta, g, kb, beside);
    }
    rc = fits_a_launch("sdpa_window_bwd", std::max(rows + 3, krows + 3) / 4, 256);
    if (!rc) rc = dl4s::ensure_scratch(ctx, delta_bytes);
    if (rc) return rc;
    float *delta = reinterpret_cast<float *>(ctx->scratch);
    if (rows) {
        hipLaunchKernelGGL(window_delta_f32, row_grid(rows), dim3(256), 0, ctx->stream, dout, out, delta, (int)H, (int)Lq, (int)d, lq, rows);
        hipLaunchKernelGGL(sdpa_window_dq_rows_f32, row_grid(rows), dim3(256), 0, ctx->stream, q, k, v, dout, stats, delta, dq, (int)H,
                           (int)(H / Hkv), (int)Lq, (int)Lk, (int)d, inv_temperature, w, lq, lk, rows);
        rc = dl4s::launch_status("sdpa_window_dq_rows_f32");
        if (rc) return rc;
    }
    if (krows)
        hipLaunchKernelGGL(sdpa_window_dkv_rows_f32, row_grid(krows), dim3(256), 0, ctx->stream, q, k, v, dout, stats, delta, dk, dv,
                           (int)H, (int)Hkv, (int)Lq, (int)Lk, (int)d, inv_temperature, w, lq, lk, krows);
    return dl4s::launch_status("sdpa_window_dkv_rows_f32");
}

int dl4s_hip_sdpa_window_decode_f32(dl4s_hip_ctx *ctx, const float *q, const float *kcache, const float *vcache, float *out, int64_t B,
                                    int64_t H, int64_t Hkv, int64_t T, int64_t Tcap, int64_t d, float inv_temperature, int64_t window,
                                    int64_t sinks, const int32_t *lengths) {
    DL4S_CHECK_CTX(ctx);
    const dl4s_window_desc desc = {window, sinks, 0, lengths};
    WindowArgs w;
    const int rc = window_checks("sdpa_window_decode", B, H, Hkv, 1, Tcap, d, &desc, 0, &w);
    if (rc) return rc;
    if (B * H == 0) return DL4S_HIP_OK;
    DL4S_REQUIRE(q && kcache && vcache && out, DL4S_HIP_EINVALID_ARG, "sdpa_window_decode: NULL tensor pointer");
    DL4S_REQUIRE(T >= 1 && T <= Tcap, DL4S_HIP_ESHAPE, "sdpa_window_decode: T=%lld must be in [1, Tcap=%lld]", (long long)T, (long long)Tcap);
    w.last_key = 1;
    FewArgs a = few_args(B, H, Hkv, 1, T, d, inv_temperature, w, layout(false, H, 1, d), layout(false, Hkv, Tcap, d), ctx->cu_count);
    return few_rows(ctx, q, kcache, vcache, out, nullptr, a, B * Hkv);
}

}  // extern "C"
