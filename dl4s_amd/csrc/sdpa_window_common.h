// Shared by the windowed attention kernels: which keys a query sees, and fp32 products on the fp16 matrix instructions.
//
// A value x is held as two fp16 planes of x times a power of two, x 2^a = h + l with h = fp16(x 2^a), l = fp16(x 2^a - h),
// each rounded to nearest: 11 + 11 significant bits.  A product is three matrix instructions, l.h + h.l + h.h (the small ones
// first), summed in fp32; the one left out is below 2^-22 of the product.  The power of two is shared: by a row for an operand
// in registers, whose largest finite value it puts at 2^14 or more, and by the 8, 16 or 32 neighbouring rows (above 64, above 32, up to 32
// columns) that a wavefront stages at a time for one in LDS: 2^11 or more, or 2^7 where rows up to 2^8 times as large were staged
// before.  Nothing overflows, and what a value loses is 2^-23 of it or, where that is more, 2^-39 (2^-36, 2^-32) of that
// largest: neighbouring rows that differ by up to 2^13 (2^9) in size are as exact as in fp32 row by row.  Measured
// against 64 bits, sums of 64 (512) products of normal values are off by 1.2e-7 (2.5e-7) of their size this way, 1.5e-7
// (3.8e-7) through v_mfma_f32_32x32x2_f32.  Why: a 32 x 32 x 16 step costs 3 x 39 SIMD cycles (measured) where eight fp32
// steps cost 8 x 66, and the vector ALU runs beside the fp16 instructions, not beside the fp32 ones.  Three bf16 planes
// need no power of two, but six instructions and half as much again of registers and LDS (the forward pass of B8 H16 L2048
// d64 window 512 took 244 us that way).
// An infinity has no such planes (inf - inf): it turns the sums it enters into NaN.
#pragma once
#include "common.h"

namespace {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned short u16;

constexpr float LOG2E = 1.44269504088896340736f;
constexpr int MAXD = 256;

__device__ __forceinline__ float exp2_fast(const float x) { return __builtin_amdgcn_exp2f(x); }

// Positions and extents are below 2^30, so that a position and a window add up in 32 bits.
struct WindowArgs {
    int window, sinks;      // clamped to [1, 2^30] and [0, Lk]
    int q_offset;
    const int *lengths;
    int last_key;           // decode: the query of batch element b stands at position lengths[b] - 1 (or Lk - 1)
};
__device__ __forceinline__ bool sees(const WindowArgs &w, const int p, const int j, const int len) {
    return (j <= p) & (j < len) & ((j > p - w.window) | (j < w.sinks));
}

// The keys a query sees, as two ranges [0, first) and [lo, hi) with first <= lo.
struct Range {
    int first, lo, hi;
};
__device__ __forceinline__ int valid_keys(const WindowArgs &w, const int b, const int Lk) {
    const int len = w.lengths ? w.lengths[b] : Lk;
    return len < 0 ? 0 : (len > Lk ? Lk : len);
}
__device__ __forceinline__ Range visible_keys(const WindowArgs &w, const int b, const int i, const int Lk) {
    const int len = valid_keys(w, b, Lk), p = w.last_key ? len - 1 : w.q_offset + i;
    Range r;
    r.hi = min(p + 1, len);
    r.lo = min(max(p - w.window + 1, 0), r.hi);
    r.first = min(w.sinks, r.lo);
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

// ---- powers of two
__device__ __forceinline__ float pow2(const int a) { return __builtin_ldexpf(1.0f, a); }
// The power that puts m (>= 0, finite) into [2^14, 2^15).  m below 2^-112 stays below, so that the power and its inverse are
// normal numbers: what is lost there are bits below 2^-136.
__device__ __forceinline__ int scale_of(const float m) {
    const int e = (int)(__float_as_uint(m) >> 23);
    return 141 - min(max(e, 15), 254);
}
// The same in steps of 2^4 ([2^11, 2^15)): neighbouring rows of like size then mostly have the same power.
__device__ __forceinline__ int coarse_scale_of(const float m) {
    return 139 - ((max((int)(__float_as_uint(m) >> 23), 15) + 1) & ~3);
}
constexpr int MOST_POWER = 123;                            // the largest of these
__device__ __forceinline__ float finite_abs(const float x) { return fabsf(x) < INFINITY ? fabsf(x) : 0.f; }
template <int CTRL>
__device__ __forceinline__ unsigned max_lanes(const unsigned u) {
    return max(u, (unsigned)__builtin_amdgcn_update_dpp(0, (int)u, CTRL, 0xF, 0xF, true));
}
// Largest of the 64 lanes' values (>= 0, so their bits are in the same order), uniform.
__device__ __forceinline__ float wave_max_abs(const float v) {
    unsigned u = __float_as_uint(v);
    u = max_lanes<0xB1>(u);
    u = max_lanes<0x4E>(u);
    u = max_lanes<0x141>(u);
    u = max_lanes<0x140>(u);
    const unsigned r0 = __builtin_amdgcn_readlane(u, 0), r1 = __builtin_amdgcn_readlane(u, 16), r2 = __builtin_amdgcn_readlane(u, 32),
                   r3 = __builtin_amdgcn_readlane(u, 48);
    return __uint_as_float(max(max(r0, r1), max(r2, r3)));
}
// Maxima without the quieting of signalling NaNs that fmaxf brings along (a NaN is passed over)
__device__ __forceinline__ float max3(const float a, const float b, const float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}
__device__ __forceinline__ float max_abs(const float m, const float a, const float b) {
    float r;
    asm("v_max3_f32 %0, %1, |%2|, |%3|" : "=v"(r) : "v"(m), "v"(a), "v"(b));
    return r;
}
template <int N>
__device__ __forceinline__ float largest(const f32x4 (&x)[N], float m = 0.f) {
#pragma unroll
    for (int i = 0; i < N; ++i) m = max_abs(max_abs(m, x[i].x, x[i].y), x[i].z, x[i].w);
    return m;
}
// Infinities do not set the scale of their neighbours: the largest finite value, for the rare case that `largest` met one.
template <int N>
__device__ __forceinline__ float largest_finite(const f32x4 (&x)[N]) {
    float m = 0.f;
    asm volatile("" ::: "memory");                 // (not to be formed ahead of the question whether it is needed)
#pragma unroll
    for (int i = 0; i < N; ++i) m = fmaxf(fmaxf(m, fmaxf(finite_abs(x[i].x), finite_abs(x[i].y))), fmaxf(finite_abs(x[i].z), finite_abs(x[i].w)));
    return m;
}

// The planes of a pair of values, the first in the low half of each word.
struct Planes {
    unsigned h, l;
};
// v_fma_mixlo_f16 / v_fma_mixhi_f16 round an fp32 multiply-add to fp16 into the low / high half of their result.  A half that was
// moved up may be read one wait state later at the earliest, and a matrix instruction reads what a vector instruction wrote
// two wait states later; the compiler does not look into the statement, so it ends with these two.
__device__ __forceinline__ unsigned round2(const float a, const float b) {
    return __builtin_bit_cast(unsigned, __builtin_convertvector((f32x2){a, b}, f16x2));
}
// The planes of four values times s.
__device__ __forceinline__ void split4(const f32x4 v, const float s, Planes &p, Planes &q) {
    asm("v_fma_mixlo_f16 %0, %4, %8, 0\n\t"
        "v_fma_mixhi_f16 %0, %5, %8, 0\n\t"
        "v_fma_mixlo_f16 %2, %6, %8, 0\n\t"
        "v_fma_mixhi_f16 %2, %7, %8, 0\n\t"
        "v_fma_mixlo_f16 %1, %4, %8, -%0 op_sel:[0,0,0] op_sel_hi:[0,0,1]\n\t"
        "v_fma_mixhi_f16 %1, %5, %8, -%0 op_sel:[0,0,1] op_sel_hi:[0,0,1]\n\t"
        "v_fma_mixlo_f16 %3, %6, %8, -%2 op_sel:[0,0,0] op_sel_hi:[0,0,1]\n\t"
        "v_fma_mixhi_f16 %3, %7, %8, -%2 op_sel:[0,0,1] op_sel_hi:[0,0,1]\n\t"
        "s_nop 1"
        : "=&v"(p.h), "=&v"(p.l), "=&v"(q.h), "=&v"(q.l)
        : "v"(v.x), "v"(v.y), "v"(v.z), "v"(v.w), "v"(s));
}

// One lane's share of an operand of a 32 x 32 x 16 step: eight values along the contraction, as planes.
struct Frag {
    f16x8 h, l;
};
__device__ __forceinline__ Frag split8(const float (&x)[8]) {
    u32x4 h, l;
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = round2(x[2 * i], x[2 * i + 1]);
    unsigned l0, l1, l2, l3;
    asm("v_fma_mixlo_f16 %0, %4, 1.0, -%12 op_sel:[0,0,0] op_sel_hi:[0,0,1]\n\t"
        "v_fma_mixlo_f16 %1, %6, 1.0, -%13 op_sel:[0,0,0] op_sel_hi:[0,0,1]\n\t"
        "v_fma_mixlo_f16 %2, %8, 1.0, -%14 op_sel:[0,0,0] op_sel_hi:[0,0,1]\n\t"
        "v_fma_mixlo_f16 %3, %10, 1.0, -%15 op_sel:[0,0,0] op_sel_hi:[0,0,1]\n\t"
        "v_fma_mixhi_f16 %0, %5, 1.0, -%12 op_sel:[0,0,1] op_sel_hi:[0,0,1]\n\t"
        "v_fma_mixhi_f16 %1, %7, 1.0, -%13 op_sel:[0,0,1] op_sel_hi:[0,0,1]\n\t"
        "v_fma_mixhi_f16 %2, %9, 1.0, -%14 op_sel:[0,0,1] op_sel_hi:[0,0,1]\n\t"
        "v_fma_mixhi_f16 %3, %11, 1.0, -%15 op_sel:[0,0,1] op_sel_hi:[0,0,1]\n\t"
        "s_nop 1"
        : "=&v"(l0), "=&v"(l1), "=&v"(l2), "=&v"(l3)
        : "v"(x[0]), "v"(x[1]), "v"(x[2]), "v"(x[3]), "v"(x[4]), "v"(x[5]), "v"(x[6]), "v"(x[7]), "v"(h.x), "v"(h.y), "v"(h.z), "v"(h.w));
    l = u32x4{l0, l1, l2, l3};
    return Frag{__builtin_bit_cast(f16x8, h), __builtin_bit_cast(f16x8, l)};
}
__device__ __forceinline__ f32x16 mma3(const Frag &a, const Frag &b, f32x16 c) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_f16(a.l, b.h, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_f16(a.h, b.l, c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a.h, b.h, c, 0, 0, 0);
}
// The three instructions of a product go to an accumulator one after the other; the accumulators c[0 .. N) take turns, because
// an instruction that adds to the accumulator of the one before it waits for it.
template <int N>
__device__ __forceinline__ void mma3(f32x16 (&c)[N], const Frag (&a)[N], const Frag &b) {
#pragma unroll
    for (int n = 0; n < N; ++n) c[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[n].l, b.h, c[n], 0, 0, 0);
#pragma unroll
    for (int n = 0; n < N; ++n) c[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[n].h, b.l, c[n], 0, 0, 0);
#pragma unroll
    for (int n = 0; n < N; ++n) c[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[n].h, b.h, c[n], 0, 0, 0);
}
// Two products at once, each with operands of its own.
__device__ __forceinline__ void mma3x2(f32x16 &c0, const Frag &a0, const Frag &b0, f32x16 &c1, const Frag &a1, const Frag &b1) {
    c0 = __builtin_amdgcn_mfma_f32_32x32x16_f16(a0.l, b0.h, c0, 0, 0, 0);
    c1 = __builtin_amdgcn_mfma_f32_32x32x16_f16(a1.l, b1.h, c1, 0, 0, 0);
    c0 = __builtin_amdgcn_mfma_f32_32x32x16_f16(a0.h, b0.l, c0, 0, 0, 0);
    c1 = __builtin_amdgcn_mfma_f32_32x32x16_f16(a1.h, b1.l, c1, 0, 0, 0);
    c0 = __builtin_amdgcn_mfma_f32_32x32x16_f16(a0.h, b0.h, c0, 0, 0, 0);
    c1 = __builtin_amdgcn_mfma_f32_32x32x16_f16(a1.h, b1.h, c1, 0, 0, 0);
}

// The vector ALU may read an accumulator 12 wait states after the last matrix instruction that wrote it.  The compiler puts
// them in, but not on a path that branches right behind the instructions (its assembly had one state there, and wrong
// sums): results that a branch follows are waited for explicitly.
__device__ __forceinline__ void settle(f32x16 &a) { asm volatile("s_nop 11" : "+v"(a)); }
__device__ __forceinline__ void settle(f32x16 &a, f32x16 &b) { asm volatile("s_nop 11" : "+v"(a), "+v"(b)); }

// With the value of lane ^ 32: both lanes end up with the same.
__device__ __forceinline__ f32x2 both_halves(const float v) {
    const u32x2 r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return f32x2{__uint_as_float(r.x), __uint_as_float(r.y)};
}
__device__ __forceinline__ float max_halves(const float v) { const f32x2 r = both_halves(v); return fmaxf(r.x, r.y); }
__device__ __forceinline__ float sum_halves(const float v) { const f32x2 r = both_halves(v); return r.x + r.y; }

// A row of up to DT columns times a factor, one row per lane of a half wavefront (lane and lane ^ 32 share it), as the operand
// whose contraction runs along the row.  The factor goes into the splitting: a plane is rounded from the exact product.
// Returns the row's power of two.
template <int DT, typename Load>
__device__ __forceinline__ int row_operand(Frag (&f)[DT / 16], const Load load, const float factor) {
    const int half = (threadIdx.x & 63) >> 5;
    f32x4 x[DT / 8];
#pragma unroll
    for (int s = 0; s < DT / 16; ++s) {
        x[2 * s] = load(16 * s + 8 * half);
        x[2 * s + 1] = load(16 * s + 8 * half + 4);
    }
    float top = max_halves(largest(x));
    if (__any(top == INFINITY)) top = max_halves(largest_finite(x));
    const int a = scale_of(top * fabsf(factor));
    const float p = pow2(a) * factor;
#pragma unroll
    for (int s = 0; s < DT / 16; ++s) {
        Planes w[4];
        split4(x[2 * s], p, w[0], w[1]);
        split4(x[2 * s + 1], p, w[2], w[3]);
        f[s] = Frag{__builtin_bit_cast(f16x8, (u32x4){w[0].h, w[1].h, w[2].h, w[3].h}), __builtin_bit_cast(f16x8, (u32x4){w[0].l, w[1].l, w[2].l, w[3].l})};
    }
    return a;
}

// Rows of a tile of an fp32 tensor through a buffer descriptor made per tile (base: the tile's first row): rows from `rows` on,
// and columns at or beyond d (whose offset lies outside every descriptor), read as zeros without a branch.
constexpr unsigned NOWHERE = 0x80000000u;
__device__ __forceinline__ __amdgpu_buffer_rsrc_t tile_rows(const float *base, const int stride, const int rows, const int d) {
    return __builtin_amdgcn_make_buffer_rsrc((void *)base, 0, rows > 0 ? ((rows - 1) * stride + d) * 4 : 0, 0x00020000);
}
// at: byte offset of the piece's first column, NOWHERE (or above) where the piece lies outside; left: columns from it to d
template <bool VEC>
__device__ __forceinline__ f32x4 tile_load4(const __amdgpu_buffer_rsrc_t rsrc, const unsigned at, const int left) {
    if (VEC) return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rsrc, (int)at, 0, 0));
    f32x4 r;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        r[e] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rsrc, (int)(e < left ? at + 4u * e : NOWHERE), 0, 0));
    return r;
}

// Tiles of R rows x C columns in LDS as planes.
//   Rows: [plane][row][C + 8]: a lane's eight columns are one 128-bit read, eight rows fall on distinct banks.
//   Columns (the transposed tile): [plane][column][R], the rows of each 16 in the order 0-3, 8-11, 4-7, 12-15, so that the
//   eight rows a lane needs against an accumulator's register order are one 128-bit read; 16-byte pieces of a column
//   are exchanged by a function of the column that spreads both the reads (32 columns, one piece) and the writes (every
//   fourth column, a few pieces) over the banks.
template <int R, int C>
struct Tile {
    static constexpr int ROWS_PLANE = R * (C + 8), COLS_PLANE = C * R;     // 16-bit elements
    static_assert((R == 32 || R == 64) && C % 32 == 0, "tile");

    __device__ static __forceinline__ int swap(const int col) {
        return R == 64 ? ((col >> 2) & 7) ^ ((col & 3) << 1) : ((col >> 1) ^ (col >> 3)) & 3;
    }
    // operand of rows [32 sub, 32 sub + 32), columns [16 step, 16 step + 16): lane = row, eight columns
    __device__ static __forceinline__ Frag rows_frag(const u16 *t, const int sub, const int step) {
        const int lane = threadIdx.x & 63;
        const u16 *p = t + (32 * sub + (lane & 31)) * (C + 8) + 16 * step + 8 * (lane >> 5);
        return Frag{*reinterpret_cast<const f16x8 *>(p), *reinterpret_cast<const f16x8 *>(p + ROWS_PLANE)};
    }
    // operand of columns [32 part, 32 part + 32), rows [16 step, 16 step + 16): lane = column, eight rows in accumulator order
    __device__ static __forceinline__ Frag cols_frag(const u16 *t, const int part, const int step) {
        const int lane = threadIdx.x & 63, col = 32 * part + (lane & 31);
        const u16 *p = t + col * R + (((2 * step + (lane >> 5)) ^ swap(col)) << 3);
        return Frag{*reinterpret_cast<const f16x8 *>(p), *reinterpret_cast<const f16x8 *>(p + COLS_PLANE)};
    }
};

// Two R x C tiles (A, B) staged together by NT threads: a thread loads 4 x 4 pieces, splits them and writes them in row form
// and / or, exchanged pairwise, in column form.  The pieces that a wavefront handles at a time are whole rows of one tile
// (C is rounded up to a power of two for that), so it finds their largest value and their power of two by itself; the
// powers go to LDS with the tile, one for every eight rows.
template <int R, int C, bool VEC, int NT = 256>
struct Stage {
    typedef Tile<R, C> T;
    static constexpr int GROUPS = (C <= 32 ? 32 : (C <= 64 ? 64 : 128)) / 4;      // of four columns
    static constexpr int QUADS = (R / 4) * GROUPS, NP = (2 * QUADS + NT - 1) / NT, WAVE_ROWS = 256 / GROUPS;
    static_assert(QUADS % 64 == 0 && WAVE_ROWS >= 8, "pieces");
    f32x4 x[NP][4];
    unsigned from[NP];       // byte offset of the thread's piece in its tensor's tile
    int to_row[NP], to_col[NP];
    // The power of the rows that this wavefront staged last of either tile, as the bits of the least number that keeps it: numbers from
    // there up to 2^8 times as much do.
    unsigned kept[2] = {least_of(MOST_POWER), least_of(MOST_POWER)};
    __device__ static __forceinline__ constexpr unsigned least_of(const int a) { return (unsigned)(134 - a) << 23; }
    __device__ static __forceinline__ int power_of(const unsigned least) { return 134 - (int)(least >> 23); }
    // The power of rows whose largest value is m behind rows with the power `last`.  Rows that would take a power one step (2^4) above
    // the last one take the last one: sizes that lie about a step's border then keep one power.  Smaller rows get their own, so
    // that no row is rounded to the size of one that was staged long before it.
    __device__ static __forceinline__ int next_power(const int last, const float m) {
        const int own = coarse_scale_of(m);
        return own <= last + 4 ? min(last, own) : own;
    }

    const int tid, wave0;    // the thread's number, and its wavefront's first, in the order in which wavefronts are given pieces

    __device__ __forceinline__ int piece(const int i) const { return tid + NT * i; }
    __device__ __forceinline__ bool has(const int i) const { return NT * (i + 1) <= 2 * QUADS || wave0 + NT * i < 2 * QUADS; }
    __device__ __forceinline__ bool second(const int i) const { return QUADS % NT == 0 ? NT * i >= QUADS : wave0 + NT * i >= QUADS; }
    __device__ __forceinline__ int row(const int i) const { return (piece(i) - second(i) * QUADS) / GROUPS * 4; }
    __device__ __forceinline__ int col(const int i) const { return piece(i) % GROUPS * 4; }
    __device__ __forceinline__ bool inside(const int i) const { return C == 4 * GROUPS || col(i) < C; }

    __device__ __forceinline__ Stage(const int stride, const int d, const int thread)
        : tid(thread), wave0(__builtin_amdgcn_readfirstlane(thread)) {
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            from[i] = col(i) < d ? (unsigned)(row(i) * stride + col(i)) * 4u : NOWHERE;
            to_row[i] = row(i) * (C + 8) + col(i);
            // column form: four rows of a column are one 8-byte write; the piece's exchange takes in the column's low bits by
            // an exclusive or with a constant
            const int kq = row(i) >> 2, at = 2 * (kq >> 2) + (kq & 1), sub = 4 * ((kq >> 1) & 1);
            to_col[i] = col(i) * R + ((at ^ T::swap(col(i))) << 3) + sub;
        }
    }
    // a, b: row r0 of either tensor; of its next R rows `rows` are valid, and those that are [hide0, hide1) of the tensor are taken
    // as zeros
    __device__ __forceinline__ void load(const float *a, const float *b, const int stride, const int r0, const int rows, const int d,
                                         const int hide0 = 0, const int hide1 = 0) {
        const __amdgpu_buffer_rsrc_t ra = tile_rows(a, stride, min(rows, R), d), rb = tile_rows(b, stride, min(rows, R), d);
        const bool cut = r0 < hide1 && r0 + R > hide0;
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            if (!has(i)) continue;
            unsigned at[4] = {from[i], from[i] + 4u * stride, from[i] + 8u * stride, from[i] + 12u * stride};
            if (__builtin_expect(cut, 0)) {
                asm volatile("" : "+v"(at[0]), "+v"(at[1]), "+v"(at[2]), "+v"(at[3]));     // (keeps this a branch)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int r = r0 + row(i) + j;
                    if (r >= hide0 && r < hide1) at[j] = NOWHERE;
                }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) x[i][j] = tile_load4<VEC>(second(i) ? rb : ra, at[j], VEC ? 0 : d - col(i));
        }
    }
    // fa: a factor of tile A's values.  powers: [A, B][R / 8], negated.
    template <bool ROWS_A, bool COLS_A, bool ROWS_B, bool COLS_B>
    __device__ __forceinline__ void store(u16 *rows_a, u16 *cols_a, u16 *rows_b, u16 *cols_b, int *powers, const float fa = 1.0f) {
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            if (!has(i)) continue;
            const bool b = second(i);
            const float f = b ? 1.0f : fa;
            unsigned &keeps = QUADS % NT == 0 ? kept[b] : kept[0];       // (a wavefront has either pieces of one tile only, or these in turn)
            float m = wave_max_abs(largest(x[i]));
            int a = power_of(keeps);
            if (__builtin_expect(__builtin_amdgcn_readfirstlane(__float_as_uint(m * fabsf(f))) - keeps >= 8u << 23, 0)) {
                if (m == INFINITY) m = wave_max_abs(largest_finite(x[i]));
                // (rows of zeros, a tile's missing ones among them, have no size that their neighbours would be weighed with)
                if (m * fabsf(f) == 0.f) a = MOST_POWER;
                else keeps = least_of(a = next_power(a, m * fabsf(f)));
            }
            const int lane = threadIdx.x & 63;
            if (lane < WAVE_ROWS / 8) powers[(b ? R / 8 : 0) + ((wave0 + NT * i - b * QUADS) / GROUPS >> 1) + lane] = -a;
            if (b) put<ROWS_B, COLS_B>(i, rows_b, cols_b, pow2(a));
            else put<ROWS_A, COLS_A>(i, rows_a, cols_a, pow2(a) * f);
        }
    }
    // scale: a power of two times the factor
    template <bool ROWS, bool COLS>
    __device__ __forceinline__ void put(const int i, u16 *rows, u16 *cols, const float scale) const {
        if (!inside(i)) return;
        Planes w[4][2];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            split4(x[i][j], scale, w[j][0], w[j][1]);
            if (ROWS) {
                u16 *tr = rows + to_row[i] + j * (C + 8);
                *reinterpret_cast<u32x2 *>(tr) = u32x2{w[j][0].h, w[j][1].h};
                *reinterpret_cast<u32x2 *>(tr + T::ROWS_PLANE) = u32x2{w[j][0].l, w[j][1].l};
            }
        }
        if (COLS) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                u16 *p = cols + (to_col[i] ^ (T::swap(c) << 3)) + c * R;
                // the low or high halves of two rows' words, side by side
                const unsigned pick = c & 1 ? 0x07060302u : 0x05040100u;
                auto turn = [&](const unsigned r0, const unsigned r1) { return __builtin_amdgcn_perm(r1, r0, pick); };
                *reinterpret_cast<u32x2 *>(p) = u32x2{turn(w[0][c >> 1].h, w[1][c >> 1].h), turn(w[2][c >> 1].h, w[3][c >> 1].h)};
                *reinterpret_cast<u32x2 *>(p + T::COLS_PLANE) = u32x2{turn(w[0][c >> 1].l, w[1][c >> 1].l), turn(w[2][c >> 1].l, w[3][c >> 1].l)};
            }
        }
    }
};
// The negated powers of two of 32 rows, one for every eight: 2^n undoes them.
typedef int i32x4 __attribute__((ext_vector_type(4)));
struct Powers {
    i32x4 n;
    int lo, hi;              // uniform
    __device__ __forceinline__ explicit Powers(const int *p) : n(*reinterpret_cast<const i32x4 *>(p)) {
        lo = __builtin_amdgcn_readfirstlane(min(min(n.x, n.y), min(n.z, n.w)));
        hi = __builtin_amdgcn_readfirstlane(max(max(n.x, n.y), max(n.z, n.w)));
    }
};
// The operand's registers r stand for rows with powers of their own: those that stand for smaller ones are taken down to 2^hi.
__device__ __forceinline__ void to_one_unit(const Powers &p, f32x16 &operand) {
#pragma unroll
    for (int r = 0; r < 16; ++r) operand[r] *= __builtin_ldexpf(1.0f, p.n[r >> 2] - p.hi);
}
// The same for sums that are kept in units of 2^n for all columns alike; returns the factor for what has been summed before.  n
// follows the tiles down as well, so that a column that met none of the large rows does not have its operand taken down: it is
// the tile's 2^hi, or 2^-60 of the largest so far.  What has been summed is then at most 2^120 units (operands and planes of up
// to 2^15, 2^30 rows, 2^60 of a step down), which fp32 holds.
__device__ __forceinline__ float to_unit_of_tile(const Powers &p, int &n, int &most, f32x16 &operand) {
    const int was = n;
    most = max(most, p.hi);
    n = max(p.hi, most - 60);
#pragma unroll
    for (int r = 0; r < 16; ++r) operand[r] *= __builtin_ldexpf(1.0f, p.n[r >> 2] - n);
    return pow2(max(was - n, -200));
}

// Row of register r of a 32 x 32 accumulator in the lane's half of the wavefront (the column is lane % 32).
__device__ __forceinline__ constexpr int acc_row(const int r) { return 8 * (r >> 2) + (r & 3); }

// The registers [8 step, 8 step + 8) of an accumulator as the other operand of a product that contracts over its rows; in the
// second form times a factor.
__device__ __forceinline__ Frag acc_frag(const f32x16 &s, const int step) {
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = s[8 * step + e];
    return split8(x);
}
__device__ __forceinline__ Frag acc_frag(const f32x16 &s, const int step, const float factor) {
    Planes w[4];
#pragma unroll
    for (int e = 0; e < 2; ++e)
        split4(f32x4{s[8 * step + 4 * e], s[8 * step + 4 * e + 1], s[8 * step + 4 * e + 2], s[8 * step + 4 * e + 3]}, factor, w[2 * e], w[2 * e + 1]);
    return Frag{__builtin_bit_cast(f16x8, (u32x4){w[0].h, w[1].h, w[2].h, w[3].h}), __builtin_bit_cast(f16x8, (u32x4){w[0].l, w[1].l, w[2].l, w[3].l})};
}

}  // namespace
