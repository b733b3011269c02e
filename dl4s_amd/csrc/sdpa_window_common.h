// Shared by the windowed attention kernels: which keys a query sees, and fp32 products on the bf16 matrix instructions.
//
// A value x is held as three bf16 planes, x = h + m + l: h = bf16(x), m = bf16(x - h), l = bf16(x - h - m), each rounded to
// nearest, so that h, m, l carry 8 + 8 + 8 significant bits and what is dropped is below 2^-27 |x|.  A product is six matrix
// instructions (l.h + h.l + m.m + m.h + h.m + h.h, the small ones first); the three left out are below 2^-25 |x y|, less than
// the rounding of one fp32 product, and the accumulators are fp32.  Measured against 64 bits, sums of 64 products of normal
// values are off by 1.2e-7 of their size this way, 1.5e-7 through v_mfma_f32_32x32x2_f32.  Why: a 32 x 32 x 16 step costs
// 6 x 36 = 216 SIMD cycles (measured) where eight fp32 steps cost 8 x 66 = 525, and the vector ALU runs beside the bf16
// instructions (up to six vector instructions per matrix instruction cost nothing), not beside the fp32 ones.
// An infinity has no such planes (inf - inf): it turns the sums it enters into NaN.
#pragma once
#include "common.h"

namespace {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned short u16;

constexpr float LOG2E = 1.44269504088896340736f;
constexpr int MAXD = 256;

__device__ __forceinline__ float exp2_fast(const float x) { return __builtin_amdgcn_exp2f(x); }

struct WindowArgs {
    int window, sinks;      // clamped to [1, 2^30] and [0, Lk]
    long long q_offset;
    const int *lengths;
    int last_key;           // decode: the query of batch element b stands at position lengths[b] - 1 (or Lk - 1)
};

// The keys a query sees, as two ranges [0, first) and [lo, hi) with first <= lo.
struct Range {
    int first, lo, hi;
};
__device__ __forceinline__ int valid_keys(const WindowArgs &w, const int b, const int Lk) {
    const int len = w.lengths ? w.lengths[b] : Lk;
    return len < 0 ? 0 : (len > Lk ? Lk : len);
}
__device__ __forceinline__ Range visible_keys(const WindowArgs &w, const int b, const int i, const int Lk) {
    const int len = valid_keys(w, b, Lk);
    const long long p = w.last_key ? (long long)len - 1 : w.q_offset + i;
    Range r;
    const long long lo = p - w.window + 1;
    r.hi = (int)(p + 1 < len ? p + 1 : len);
    r.lo = lo < 0 ? 0 : (int)(lo > r.hi ? r.hi : lo);
    r.first = w.sinks < r.lo ? w.sinks : r.lo;
    return r;
}

struct Layout {             // element strides of [B, heads, L, d] tensors in either layout
    long long b, h, l;
};

// Four consecutive columns of a row; columns at or beyond d are zeros.  vec: d is a multiple of 4 and rows start on 16 bytes.
__device__ __forceinline__ f32x4 load4(const float *row, const int col, const int d, const bool vec) {
    f32x4 r = {0.f, 0.f, 0.f, 0.f};
    if (vec) {
        if (col < d) r = *reinterpret_cast<const f32x4 *>(row + col);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (col + e < d) r[e] = row[col + e];
    }
    return r;
}
__device__ __forceinline__ void store4(float *row, const int col, const int d, const bool vec, const f32x4 v) {
    if (vec) {
        if (col < d) *reinterpret_cast<f32x4 *>(row + col) = v;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (col + e < d) row[col + e] = v[e];
    }
}

// The planes of a pair of values, the first in the low half of each word.
struct Planes {
    unsigned h, m, l;
};
__device__ __forceinline__ unsigned round2(const float a, const float b) {
    return __builtin_bit_cast(unsigned, __builtin_convertvector((f32x2){a, b}, bf16x2));
}
__device__ __forceinline__ Planes split2(const float a, const float b) {
    Planes p;
    p.h = round2(a, b);
    const float a1 = a - __uint_as_float(p.h << 16), b1 = b - __uint_as_float(p.h & 0xffff0000u);
    p.m = round2(a1, b1);
    p.l = round2(a1 - __uint_as_float(p.m << 16), b1 - __uint_as_float(p.m & 0xffff0000u));
    return p;
}

// One lane's share of an operand of a 32 x 32 x 16 step: eight values along the contraction, as planes.
struct Frag {
    bf16x8 h, m, l;
};
__device__ __forceinline__ Frag split8(const float (&x)[8]) {
    u32x4 h, m, l;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const Planes p = split2(x[2 * i], x[2 * i + 1]);
        h[i] = p.h; m[i] = p.m; l[i] = p.l;
    }
    return Frag{__builtin_bit_cast(bf16x8, h), __builtin_bit_cast(bf16x8, m), __builtin_bit_cast(bf16x8, l)};
}
__device__ __forceinline__ f32x16 mma6(const Frag &a, const Frag &b, f32x16 c) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.l, b.h, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.h, b.l, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.m, b.m, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.m, b.h, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.h, b.m, c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.h, b.h, c, 0, 0, 0);
}

// Tiles of R rows x C columns in LDS as planes, written by a workgroup of 256 from fp32 rows in global memory.
//   Rows: [plane][row][C + 8]: a lane's eight columns are one 128-bit read, eight rows fall on distinct banks.
//   Columns (the transposed tile): [plane][column][R], the rows of each 16 in the order 0-3, 8-11, 4-7, 12-15, so that the
//   eight rows a lane needs against an accumulator's register order are one 128-bit read; 16-byte pieces of a column
//   are exchanged by a function of the column that spreads both the reads (32 columns, one piece) and the writes (every
//   fourth column, a few pieces) over the banks.
template <int R, int C>
struct Tile {
    static constexpr int ROWS_PLANE = R * (C + 8), COLS_PLANE = C * R;     // 16-bit elements
    static constexpr int NROW = R * C / 1024;                              // float4 pieces per thread
    static constexpr int QUADS = (R / 4) * (C / 4);                        // 4 x 4 pieces, at most one per thread
    static_assert(R * C % 1024 == 0 && QUADS <= 256 && (R == 32 || R == 64) && C % 32 == 0, "tile");

    __device__ static __forceinline__ int swap(const int col) {
        return R == 64 ? ((col >> 2) & 7) ^ ((col & 3) << 1) : ((col >> 1) ^ (col >> 3)) & 3;
    }
    // thread's piece i of the row form: row, column
    __device__ static __forceinline__ int row_of(const int i) { return (threadIdx.x + 256 * i) / (C / 4); }
    __device__ static __forceinline__ int col_of(const int i) { return (threadIdx.x + 256 * i) % (C / 4) * 4; }
    __device__ static __forceinline__ void load_rows(f32x4 (&x)[NROW], const float *base, const long long stride, const int r0,
                                                     const int rows, const int d, const bool vec) {
#pragma unroll
        for (int i = 0; i < NROW; ++i) {
            const int r = r0 + row_of(i);
            x[i] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (r < rows) x[i] = load4(base + r * stride, col_of(i), d, vec);
        }
    }
    __device__ static __forceinline__ void store_rows(u16 *t, const f32x4 (&x)[NROW]) {
#pragma unroll
        for (int i = 0; i < NROW; ++i) {
            const Planes a = split2(x[i].x, x[i].y), b = split2(x[i].z, x[i].w);
            u16 *p = t + row_of(i) * (C + 8) + col_of(i);
            *reinterpret_cast<u32x2 *>(p) = u32x2{a.h, b.h};
            *reinterpret_cast<u32x2 *>(p + ROWS_PLANE) = u32x2{a.m, b.m};
            *reinterpret_cast<u32x2 *>(p + 2 * ROWS_PLANE) = u32x2{a.l, b.l};
        }
    }
    // thread's 4 x 4 piece of the column form
    __device__ static __forceinline__ int quad_row() { return threadIdx.x / (C / 4) * 4; }
    __device__ static __forceinline__ int quad_col() { return threadIdx.x % (C / 4) * 4; }
    __device__ static __forceinline__ bool has_quad() { return QUADS == 256 || threadIdx.x < QUADS; }
    __device__ static __forceinline__ void load_quad(f32x4 (&x)[4], const float *base, const long long stride, const int r0,
                                                     const int rows, const int d, const bool vec) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = r0 + quad_row() + i;
            x[i] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (has_quad() && r < rows) x[i] = load4(base + r * stride, quad_col(), d, vec);
        }
    }
    __device__ static __forceinline__ void store_cols(u16 *t, const f32x4 (&x)[4]) {
        if (!has_quad()) return;
        const int kq = quad_row() >> 2;
        const int piece = 2 * (kq >> 2) + (kq & 1), sub = 4 * ((kq >> 1) & 1);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int col = quad_col() + j;
            const Planes a = split2(x[0][j], x[1][j]), b = split2(x[2][j], x[3][j]);
            u16 *p = t + col * R + ((piece ^ swap(col)) << 3) + sub;
            *reinterpret_cast<u32x2 *>(p) = u32x2{a.h, b.h};
            *reinterpret_cast<u32x2 *>(p + COLS_PLANE) = u32x2{a.m, b.m};
            *reinterpret_cast<u32x2 *>(p + 2 * COLS_PLANE) = u32x2{a.l, b.l};
        }
    }
    // operand of rows [32 sub, 32 sub + 32), columns [16 step, 16 step + 16): lane = row, eight columns
    __device__ static __forceinline__ Frag rows_frag(const u16 *t, const int sub, const int step) {
        const int lane = threadIdx.x & 63;
        const u16 *p = t + (32 * sub + (lane & 31)) * (C + 8) + 16 * step + 8 * (lane >> 5);
        return Frag{*reinterpret_cast<const bf16x8 *>(p), *reinterpret_cast<const bf16x8 *>(p + ROWS_PLANE),
                    *reinterpret_cast<const bf16x8 *>(p + 2 * ROWS_PLANE)};
    }
    // operand of columns [32 part, 32 part + 32), rows [16 step, 16 step + 16): lane = column, eight rows in accumulator order
    __device__ static __forceinline__ Frag cols_frag(const u16 *t, const int part, const int step) {
        const int lane = threadIdx.x & 63, col = 32 * part + (lane & 31);
        const u16 *p = t + col * R + (((2 * step + (lane >> 5)) ^ swap(col)) << 3);
        return Frag{*reinterpret_cast<const bf16x8 *>(p), *reinterpret_cast<const bf16x8 *>(p + COLS_PLANE),
                    *reinterpret_cast<const bf16x8 *>(p + 2 * COLS_PLANE)};
    }
};

// Row of register r of a 32 x 32 accumulator in the lane's half of the wavefront (the column is lane % 32).
__device__ __forceinline__ constexpr int acc_row(const int r) { return 8 * (r >> 2) + (r & 3); }

__device__ __forceinline__ float max_halves(const float v) { return fmaxf(v, __shfl_xor(v, 32, 64)); }
__device__ __forceinline__ float sum_halves(const float v) { return v + __shfl_xor(v, 32, 64); }

// The registers [8 step, 8 step + 8) of an accumulator as the other operand of a product that contracts over its rows.
__device__ __forceinline__ Frag acc_frag(const f32x16 &s, const int step) {
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = s[8 * step + e];
    return split8(x);
}

}  // namespace
