// w4.hip -- weights in 4 bits with a bf16 scale per group: quantize, dequantize, and products of a few rows with them.
//
// No counterpart in the reference (fp32 cuBLAS only).  Codes are the small floats 0, 0.5, 1, 1.5, 2, 3, 4, 6 with a
// sign, which gfx950 converts two at a time (v_cvt_scalef32_pk_f32_fp4); rows are row-major, two codes to a byte and
// padded to 16 bytes, so 16 bytes are 32 consecutive columns: one "unit".
#include "common.hpp"
#include "../../include/nerf_amd.h"

#include <math.h>

#include <algorithm>
#include <type_traits>

#pragma clang fp contract(off)

namespace nerf {
namespace {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

__device__ __forceinline__ float bf16_to_f32(unsigned short b) { return __builtin_bit_cast(float, (unsigned)b << 16); }
__device__ __forceinline__ unsigned short f32_to_bf16(float x) { return __builtin_bit_cast(unsigned short, (__bf16)x); }

template <int CTRL>
__device__ __forceinline__ unsigned max_dpp(unsigned x) {
    const unsigned y = (unsigned)__builtin_amdgcn_update_dpp((int)x, (int)x, CTRL, 0xf, 0xf, false);
    return max(x, y);
}

// the eight values of a dword of codes, times two: whole numbers, whose products with fp32 numbers are multiples of 2^-149
__device__ __forceinline__ void doubles8(unsigned c, float* v) {
    const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 2.0f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 2.0f, 1);
    const f32x2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 2.0f, 2), e = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 2.0f, 3);
    v[0] = a[0]; v[1] = a[1]; v[2] = b[0]; v[3] = b[1];
    v[4] = d[0]; v[5] = d[1]; v[6] = e[0]; v[7] = e[1];
}

// ---- quantize and dequantize ----------------------------------------------------------------------------
constexpr unsigned SLAB = 0x40000000u;  // pieces of a slab of rows (gridDim.y of them): their numbers fit 32 bits

// piece number `id` of a slab: its row (of all), or rows if there is none, and its place in the row; `per_row` to a row
__device__ __forceinline__ long piece_of(unsigned id, unsigned per_row, int rows, unsigned& place) {
    const unsigned in_slab = id / per_row, slab_rows = SLAB / per_row;
    place = id - in_slab * per_row;
    const long row = (long)blockIdx.y * slab_rows + in_slab;
    return in_slab < slab_rows && row < rows ? row : rows;
}

// A thread takes eight consecutive columns of a row; the 4, 8 or 16 threads of a group are neighbours in a row of sixteen
// lanes (a row of W has whole groups of threads).  Bound by memory: 8192 x 8192 53.6 us = 5.7 TB/s; two such pieces to a
// thread 56, four columns to a thread, so that a load takes whole lines in a row, 63 (57.5 with two pieces), reads past the
// caches 55.  Vector work is next (seven comparisons to a weight instead of a quotient: 57.5).
template <int GROUP>
__global__ __launch_bounds__(256) void quantize_w4_kernel(const float* __restrict__ src, long ld, int rows, int cols,
                                                          unsigned per_row, unsigned char* __restrict__ codes,
                                                          long row_bytes, unsigned short* __restrict__ scales, int groups) {
    unsigned place;
    const long row = piece_of(blockIdx.x * 256 + threadIdx.x, per_row, rows, place);
    const int col = (int)place * 8;
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (row < rows) {
        const float* p = src + row * ld + col;
        if (col + 8 <= cols) {
            const f32x4u a = *reinterpret_cast<const f32x4u*>(p), b = *reinterpret_cast<const f32x4u*>(p + 4);
#pragma unroll
            for (int k = 0; k < 4; k++) { x[k] = a[k]; x[k + 4] = b[k]; }
        } else {
#pragma unroll
            for (int k = 0; k < 7; k++)
                if (col + k < cols) x[k] = p[k];
        }
    }
    unsigned top = 0;  // of the magnitudes' bits: infinities and NaN come out on top
#pragma unroll
    for (int k = 0; k < 8; k++) top = max(top, __builtin_bit_cast(unsigned, fabsf(x[k])));
    top = max_dpp<0xB1>(top);
    top = max_dpp<0x4E>(top);
    if (GROUP >= 64) top = max_dpp<0x141>(top);
    if (GROUP >= 128) top = max_dpp<0x140>(top);
    // the smallest bf16 s with 6 s >= top: a sixth cut to 16 bits, or the next one (6 s has 10 bits and is exact)
    const float largest = __builtin_bit_cast(float, top);
    unsigned s = __builtin_bit_cast(unsigned, largest * (1.0f / 6.0f)) >> 16;
    s += 6.0f * bf16_to_f32((unsigned short)s) < largest;
    const bool bad = top >= 0x7F800000u;
    if (row >= rows) return;
    // The quotient by the scale, as its fp32 rounding, and the conversion to nearest with ties to even decide as the weights
    // themselves do: a weight that is not on a border between codes (a multiple of the scale with 12 bits at most) is a step
    // of its own away from it, 2^-24 and more, and the scale's 8 bits leave the quotient 2^-32 farther from the border than
    // half a step of fp32.  One correction of a product with the reciprocal is as near as 2^-45.  Powers of two are taken out
    // first, for scales whose reciprocal would leave fp32's range.
    const float scale = bf16_to_f32((unsigned short)s), part = __builtin_amdgcn_frexp_mantf(scale);
    const int exponent = __builtin_amdgcn_frexp_expf(scale);
    const float inverse = top == 0 ? 0.0f : __builtin_amdgcn_rcpf(part);
    float q[8];
#pragma unroll
    for (int k = 0; k < 8; k++) {
        const float w = __builtin_amdgcn_ldexpf(x[k], -exponent), near = w * inverse;
        q[k] = __builtin_fmaf(__builtin_fmaf(-near, part, w), inverse, near);
    }
    unsigned word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, q[0], q[1], 1.0f, 0);
    word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, q[2], q[3], 1.0f, 1);
    word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, q[4], q[5], 1.0f, 2);
    word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, q[6], q[7], 1.0f, 3);
    const unsigned some = (word | word >> 1 | word >> 2) & 0x11111111u;  // codes that are not zero: only they keep a sign
    word = bad ? 0u : word & (0x77777777u | some << 3);
    if ((long)place * 4 < row_bytes) *reinterpret_cast<unsigned*>(codes + row * row_bytes + (long)place * 4) = word;
    if (place % (GROUP / 8) == 0) scales[row * groups + place / (GROUP / 8)] = bad ? 0x7FC0 : (unsigned short)s;
}

// A thread does two pieces of four consecutive columns, so that a wavefront writes whole lines, and past the caches: a
// half-written line does not wait for its other half (8192 x 8192: 42 us = 7.2 TB/s; through the caches 62, and 104 where a
// thread's eight columns went out in two halves past them).
__global__ __launch_bounds__(256) void dequantize_w4_kernel(const unsigned char* __restrict__ codes, long row_bytes,
                                                            const unsigned short* __restrict__ scales, int groups, int group,
                                                            int rows, int cols, unsigned per_row, float* __restrict__ dst, long ld) {
#pragma unroll
    for (int u = 0; u < 2; u++) {
        unsigned place;
        const long row = piece_of(blockIdx.x * 512 + u * 256 + threadIdx.x, per_row, rows, place);
        if (row >= rows) continue;
        const int col = (int)place * 4;
        const float scale = bf16_to_f32(scales[row * groups + col / group]);
        const unsigned c = *reinterpret_cast<const unsigned short*>(codes + row * row_bytes + (long)place * 2);
        const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 1);
        const f32x4u v = {a[0] * scale, a[1] * scale, b[0] * scale, b[1] * scale};
        float* p = dst + row * ld + col;
        if (col + 4 <= cols) __builtin_nontemporal_store(v, reinterpret_cast<f32x4u*>(p));
        else
#pragma unroll
            for (int k = 0; k < 3; k++)
                if (col + k < cols) p[k] = v[k];
    }
}

// ---- products -------------------------------------------------------------------------------------------
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x2u __attribute__((ext_vector_type(2), aligned(2)));
typedef unsigned u32u __attribute__((aligned(2)));
typedef unsigned u32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned u32x4u2 __attribute__((ext_vector_type(4), aligned(2)));

constexpr int WAVES = 8;  // of a workgroup

struct W4Args {
    const void* X;
    const unsigned char* codes;
    const unsigned short* scales;
    void* Y;
    long ldx, ldy, row_bytes;
    int M, N, K, group, groups, x_bf16, y_bf16, epilogue;
};

__device__ __forceinline__ void store_y(const W4Args& a, long at, float y) {
    // sigmoid through the hardware exp2 and reciprocal, as in the other products' epilogues
    if (a.epilogue == 1) y = y * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(y * -1.44269504088896340736f));
    if (a.y_bf16) ((unsigned short*)a.Y)[at] = f32_to_bf16(y);
    else ((float*)a.Y)[at] = y;
}

// ---- one or two rows ------------------------------------------------------------------------------------
// A lane keeps the X of one unit (32 columns) of each row in registers as fp32 and walks down the rows of W: 16 bytes of
// codes and a scale per row, converted two at a time and multiplied by fused multiply-adds.  Sixty-four lanes are 2048
// columns: `kw` wavefronts lie side by side along K (a longer K takes several rounds), a shorter K has `lanes` lanes to
// a row and several rows to a wavefront.  B loads of W are on their way while the B before are worked on.  Bound by memory:
// 1 x 16384 x 8192 in bf16 12.6 us = 5.5 TB/s, in fp32 14.4.  Matrix instructions, which round up to 16 rows, took 17.5; from
// three rows on they are the faster ones (4 x 16384 x 8192 20.6 us here 31.6, 3 x 4096 x 4096 6.1 and 6.5).
template <int CTRL>
__device__ __forceinline__ float add_dpp(float x) {
    const int y = __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true);
    return x + __builtin_bit_cast(float, y);
}
// a + b where the lower half of the result is the sum of a's halves and the upper half that of b's; and for every two
// rows of sixteen lanes alike
__device__ __forceinline__ float fold32(float a, float b) {
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, a), __builtin_bit_cast(unsigned, b), false, false);
    const unsigned lo = r[0], hi = r[1];  // (a bit cast of r[1] itself reads r[0])
    return __builtin_bit_cast(float, lo) + __builtin_bit_cast(float, hi);
}
__device__ __forceinline__ float fold16(float a, float b) {
    const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, a), __builtin_bit_cast(unsigned, b), false, false);
    const unsigned lo = r[0], hi = r[1];  // (a bit cast of r[1] itself reads r[0])
    return __builtin_bit_cast(float, lo) + __builtin_bit_cast(float, hi);
}
__device__ __forceinline__ float sum16(float x) {
    return add_dpp<0x140>(add_dpp<0x141>(add_dpp<0x4E>(add_dpp<0xB1>(x))));
}

constexpr int GEMV_LOADS = 2;  // of W on their way, and as many worked on

struct GemvShape {
    int log_lanes;  // 2^log_lanes lanes to a row: 64, or less where that is all of K
    int log_kw;     // 2^log_kw wavefronts along K (of WAVES)
    int loads;      // of W per wavefront and round, a multiple of B
    int stride;     // bytes between a unit's pieces of an fp32 X in LDS: 128 past a multiple of 256
};

template <int M, bool XBF>
__global__ __launch_bounds__(64 * WAVES) void gemv_w4_kernel(const W4Args a, const GemvShape g) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    constexpr int B = GEMV_LOADS;
    // LDS: an fp32 X as [row][piece of four columns in a unit][unit], so that it is read from memory and from LDS in runs
    // (a lane's unit is 128 bytes, and as many lines as lanes are slow to look up; a bf16 unit is half of that and is
    // read directly); then the sums [M][kw][rows of the workgroup]
    float* sums = reinterpret_cast<float*>(lds + (XBF ? 0 : M * 8 * g.stride));
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lanes = 1 << g.log_lanes, kw = 1 << g.log_kw;
    const int wk = wave & (kw - 1), wn = wave >> g.log_kw;
    const int at_once = 64 >> g.log_lanes;       // rows of a load
    const int wave_rows = g.loads * at_once, block_rows = wave_rows * (WAVES >> g.log_kw);
    const int sub = lane >> g.log_lanes;         // the lane's row of a load
    const int units = (a.K + 31) / 32, shift = a.group == 32 ? 0 : a.group == 64 ? 1 : 2;
    const long n0 = (long)blockIdx.x * block_rows + wn * wave_rows;
    for (int round = 0; round * kw * 64 < units; round++) {
        const int unit = (round * kw + wk) * 64 + (lane & (lanes - 1));
        const bool live = unit < units;
        const int held = min(unit, units - 1);
        const unsigned char* codes = a.codes + (long)held * 16;
        const unsigned short* scales = a.scales + (held >> shift);
        u32x4 next[B];
        unsigned short next_scale[B];
        auto load = [&](int first) {
#pragma unroll
            for (int b = 0; b < B; b++) {  // rows past the end repeat the last one; what they give is not stored
                const long n = min(n0 + (first + b) * at_once + sub, (long)a.N - 1);
                next[b] = *reinterpret_cast<const u32x4*>(codes + n * a.row_bytes);
                next_scale[b] = scales[n * a.groups];
            }
        };
        load(0);
        float x[M][32];
        if constexpr (XBF) {
#pragma unroll
            for (int m = 0; m < M; m++)
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    const int col = unit * 32 + q * 8;
                    const unsigned short* from = (const unsigned short*)a.X + m * a.ldx + col;
                    u32x4 v = {0, 0, 0, 0};
                    if (col + 8 <= a.K) v = *reinterpret_cast<const u32x4u2*>(from);
                    else if (col < a.K)
#pragma unroll
                        for (int k = 0; k < 7; k++)
                            if (col + k < a.K) v[k / 2] |= (unsigned)from[k] << (16 * (k & 1));
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const unsigned word = v[e];
                        x[m][q * 8 + 2 * e] = __builtin_bit_cast(float, word << 16);
                        x[m][q * 8 + 2 * e + 1] = __builtin_bit_cast(float, word & 0xFFFF0000u);
                    }
                }
        } else {
            if (round) __syncthreads();
            const int width = kw << g.log_lanes, base = round * kw * 64;  // units of a round, and the first one
            for (int p = threadIdx.x; p < M * width * 8; p += 64 * WAVES) {
                const int m = M == 1 ? 0 : p >= width * 8, at = p - m * width * 8;
                const int col = base * 32 + at * 4;
                const float* from = (const float*)a.X + m * a.ldx + col;
                f32x4 v = {0.f, 0.f, 0.f, 0.f};
                if (col + 4 <= a.K) v = *reinterpret_cast<const f32x4u*>(from);
                else
                    for (int k = 0; k < 3; k++)
                        if (col + k < a.K) v[k] = from[k];
                *reinterpret_cast<f32x4*>(lds + (m * 8 + at % 8) * g.stride + at / 8 * 16) = v;
            }
            __syncthreads();
#pragma unroll
            for (int m = 0; m < M; m++)
#pragma unroll
                for (int q = 0; q < 8; q++) {
                    const f32x4 v = *reinterpret_cast<const f32x4*>(lds + (m * 8 + q) * g.stride + (unit - base) * 16);
#pragma unroll
                    for (int e = 0; e < 4; e++) x[m][q * 4 + e] = v[e];
                }
        }
        for (int first = 0; first < g.loads; first += B) {
            u32x4 c[B];
            float scale[B], y[M][B];
#pragma unroll
            for (int b = 0; b < B; b++) {
                c[b] = next[b];
                scale[b] = live ? bf16_to_f32(next_scale[b]) * 0.5f : 0.0f;
            }
            if (first + B < g.loads) load(first + B);
            asm volatile("" ::: "memory");  // the loads stay here, B rows ahead of their use
#pragma unroll
            for (int b = 0; b < B; b++) {
                float part[M];
#pragma unroll
                for (int m = 0; m < M; m++) part[m] = 0.0f;
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    float v[8];
                    doubles8(c[b][q], v);
#pragma unroll
                    for (int m = 0; m < M; m++)
#pragma unroll
                        for (int k = 0; k < 8; k++) part[m] = __builtin_fmaf(x[m][q * 8 + k], v[k], part[m]);
                }
#pragma unroll
                for (int m = 0; m < M; m++) y[m][b] = part[m] * scale[b];
            }
            // sums over a row's lanes, and who holds which row of this turn
            int row = first * at_once + sub, count = B;
            bool writes = (lane & (lanes - 1)) == 0;
            if (g.log_lanes == 6) {
#pragma unroll
                for (int m = 0; m < M; m++) {  // two rows go to the two halves
                    const float z = fold32(y[m][0], y[m][1]);
                    y[m][0] = sum16(fold16(z, z));
                }
                row = first + (lane >> 5);
                writes = (lane & 31) == 0;
                count = 1;
            } else {
#pragma unroll
                for (int m = 0; m < M; m++)
#pragma unroll
                    for (int b = 0; b < B; b++) {
                        float t = y[m][b];
                        if (g.log_lanes > 0) t = add_dpp<0xB1>(t);
                        if (g.log_lanes > 1) t = add_dpp<0x4E>(t);
                        if (g.log_lanes > 2) t = add_dpp<0x141>(t);
                        if (g.log_lanes > 3) t = add_dpp<0x140>(t);
                        if (g.log_lanes > 4) t = fold16(t, t);
                        y[m][b] = t;
                    }
            }
            if (writes) {
#pragma unroll
                for (int m = 0; m < M; m++) {
                    float* to = sums + (m * kw + wk) * block_rows + wn * wave_rows + row;
#pragma unroll
                    for (int b = 0; b < B; b++)
                        if (b < count) to[b * at_once] = round ? to[b * at_once] + y[m][b] : y[m][b];
                }
            }
        }
    }
    __syncthreads();
    for (int r = threadIdx.x; r < block_rows * M; r += 64 * WAVES) {
        const int m = r / block_rows, row = r - m * block_rows;
        const long n = (long)blockIdx.x * block_rows + row;
        if (n >= a.N) continue;
        float y = 0.0f;
        for (int k = 0; k < kw; k++) y += sums[(m * kw + k) * block_rows + row];
        store_y(a, m * a.ldy + n, y);
    }
}

// ---- many rows ------------------------------------------------------------------------------------------
// One product for any number of rows.  A workgroup of eight wavefronts takes R MT rows of X and 16 NT columns of Y (rows
// of W) for each of `8 / kw` wavefronts; `kw` wavefronts share the same columns and split the contraction, which goes in
// chunks of 128 columns.
//   X: a slice of the rows' columns is put in LDS as matrix operands, once for all wavefronts: bf16 as it is, fp32 as
// three bf16 numbers that add up to it exactly (its upper, middle and lower 8 significant bits, cut off), with one matrix
// instruction each.  What these leave over of a number below 2^-110 is seen as it is put there, and multiplied after the rest
// (add_left_over).  Codes are bf16 numbers exactly, so products are exact and sums are fp32.  The slice after the next is
// on its way in registers while one is worked on.
//   W: per chunk a lane loads 16 bytes (one unit of 32 columns) of one of 16 rows straight to registers, DEPTH chunks
// ahead; four lane swaps turn the four units that four lanes hold of a row into the four steps of a matrix instruction
// (16 x 16 x 32), so that a step's 32 columns lie in one group and the sum over a group takes one scale.  Columns of
// workgroups start at different chunks of a slice: rows of W are often a power of two apart, and workgroups that walk
// them in step would all ask the same few memory channels.
//   Times (groups of 64): 16 x 16384 x 8192 24.4 us = 2.9 TB/s of W; left out by turns, X costs 7 us of it, matrix instructions
// and conversions 4.5, and W, two launches and the join the rest.  24 x 4100 x 4090 13.9 us: X 4, the second
// launch and the join 4.5, the rest a chain that is too short to overlap.  64 x 16384 x 8192 58 us, in bf16 33 = 520 TFLOP/s.
// Scales that each wavefront loads for itself, chunk by chunk (16 lines for 64 bytes of each row), had cost 5 us of
// 8 x 16384 x 8192 in bf16 (17.6 us); sixteen wavefronts to a workgroup, or a whole slice of W ahead, gained nothing.
// eight codes as eight bf16
__device__ __forceinline__ bf16x8 values8_bf16(unsigned c) {
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, 1.0f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, 1.0f, 1);
    const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, 1.0f, 2), e = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, 1.0f, 3);
    return bf16x8{a[0], a[1], b[0], b[1], d[0], d[1], e[0], e[1]};
}

// upper halves of two words, the first one below
__device__ __forceinline__ unsigned upper_halves(unsigned lo, unsigned hi) { return __builtin_amdgcn_perm(hi, lo, 0x07060302); }

// the upper, middle and lower 8 significant bits of an fp32 number, each as the upper half of a word (a bf16 number)
__device__ __forceinline__ void split3(unsigned x, unsigned& hi, unsigned& mid, unsigned& lo) {
    const float rest = __builtin_bit_cast(float, x) - __builtin_bit_cast(float, x & 0xFFFF0000u);
    hi = x;
    mid = __builtin_bit_cast(unsigned, rest);
    lo = __builtin_bit_cast(unsigned, rest - __builtin_bit_cast(float, mid & 0xFFFF0000u));
}
// the same for a number that may not be finite: infinity less itself would be NaN, and a NaN cut off could read as infinity,
// so these go in the first part alone
__device__ __forceinline__ void split3_any(unsigned x, unsigned& hi, unsigned& mid, unsigned& lo) {
    split3(x, hi, mid, lo);
    if ((x & 0x7F800000u) != 0x7F800000u) return;
    hi = (x & 0x7FFFFFFFu) > 0x7F800000u ? 0x7FC00000u : x;
    mid = lo = 0;
}

// A bf16 number has no bit below 2^-133, so the parts of a number below 2^-110 may leave something over, then the lower half of
// `lo`: this much, times 2^32
__device__ __forceinline__ float left_over(unsigned x) {
    if ((x & 0x7FFFFFFFu) >= 0x08800000u) return 0.0f;  // 2^-110 and above, and what is not finite
    unsigned hi, mid, lo;
    split3(x, hi, mid, lo);
    return (__builtin_bit_cast(float, lo) - __builtin_bit_cast(float, lo & 0xFFFF0000u)) * 0x1p32f;
}

// Eight consecutive values of a row of X as they lie in memory, and as one or three operands of eight bf16
template <bool XBF>
struct Piece {
    u32x4 v[XBF ? 1 : 2];

    __device__ __forceinline__ void load(const void* row, int col) {
        if constexpr (XBF) {
            v[0] = *reinterpret_cast<const u32x4u2*>((const unsigned short*)row + col);
        } else {
            v[0] = *reinterpret_cast<const u32x4u*>((const unsigned*)row + col);
            v[1] = *reinterpret_cast<const u32x4u*>((const unsigned*)row + col + 4);
        }
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int k = 0; k < (XBF ? 1 : 2); k++) v[k] = u32x4{0, 0, 0, 0};
    }
    // the answer's lower half is not zero if the parts leave something over
    __device__ __forceinline__ unsigned operands(u32x4* o) const {
        if constexpr (XBF) {
            o[0] = v[0];
            return 0;
        } else {
            unsigned hi[8], mid[8], lo[8], left = 0;
            auto pack = [&] {
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    o[0][k] = upper_halves(hi[2 * k], hi[2 * k + 1]);
                    o[1][k] = upper_halves(mid[2 * k], mid[2 * k + 1]);
                    o[2][k] = upper_halves(lo[2 * k], lo[2 * k + 1]);
                }
            };
#pragma unroll
            for (int k = 0; k < 8; k++) split3(v[k / 4][k % 4], hi[k], mid[k], lo[k]);
            pack();
            float none = 0.0f;  // lo times zero: a NaN if any number is not finite
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const unsigned two = o[2][k];  // (a bit cast of the element itself reads the first one)
                none = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, two), bf16x2{0, 0}, none, false);
            }
            if (none != 0.0f) {
#pragma unroll
                for (int k = 0; k < 8; k++) split3_any(v[k / 4][k % 4], hi[k], mid[k], lo[k]);
                pack();
            }
#pragma unroll
            for (int k = 0; k < 8; k++) left |= lo[k];
            return left;
        }
    }
};

// d[s] of lane group j (16 lanes each) becomes what d[j] of lane group s was
__device__ __forceinline__ u32x4 transpose4(u32x4 d) {
    auto a = __builtin_amdgcn_permlane32_swap(d[0], d[2], false, false);
    auto b = __builtin_amdgcn_permlane32_swap(d[1], d[3], false, false);
    auto c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
    auto e = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
    return u32x4{c[0], c[1], e[0], e[1]};
}

// Up to eight consecutive scales of a row of W, from `first` on, as they lie in memory; the row has `groups`.  At the row's
// end they are its last COUNT ones, and the shift is left to put(): nothing is done to what is loaded before it is used, or
// the load would be waited for.  Groups past the end have the scale zero.
template <int COUNT>
struct Scales {
    unsigned v[COUNT <= 2 ? 1 : COUNT / 2];

    __device__ __forceinline__ void load(const unsigned short* row, int first, int groups) {
        if (groups >= COUNT) {
            const unsigned short* p = row + min(first, groups - COUNT);
            if constexpr (COUNT == 8) {
                const u32x4u2 x = *reinterpret_cast<const u32x4u2*>(p);
#pragma unroll
                for (int k = 0; k < 4; k++) v[k] = x[k];
            } else if constexpr (COUNT == 4) {
                const u32x2u x = *reinterpret_cast<const u32x2u*>(p);
                v[0] = x[0];
                v[1] = x[1];
            } else {
                v[0] = *reinterpret_cast<const u32u*>(p);
            }
        } else {
#pragma unroll
            for (int k = 0; k < COUNT / 2; k++)
                v[k] = (2 * k < groups ? row[2 * k] : 0u) | (2 * k + 1 < groups ? (unsigned)row[2 * k + 1] << 16 : 0u);
        }
    }
    __device__ __forceinline__ void put(char* at, int first, int groups) const {
        if (first + COUNT <= max(groups, COUNT)) {
            if constexpr (COUNT == 8) *reinterpret_cast<u32x4*>(at) = u32x4{v[0], v[1], v[2], v[3]};
            else
#pragma unroll
                for (int k = 0; k < COUNT / 2; k++) reinterpret_cast<unsigned*>(at)[k] = v[k];
            return;
        }
        const int past = first - max(0, groups - COUNT);  // places too far up
#pragma unroll
        for (int k = 0; k < COUNT; k++) {
            const unsigned short x = (unsigned short)(v[k / 2] >> (16 * (k & 1)));
            unsigned short* to = reinterpret_cast<unsigned short*>(at);
            if (k >= past) to[k - past] = x;
            if (COUNT - 1 - k < past) to[k] = 0;
        }
    }
};

struct GemmShape {
    int log_kw;        // 2^log_kw wavefronts split the contraction: 1, 2, 4 or 8
    int split_chunks;  // chunks of one part of the contraction (gridDim.z parts), a multiple of a slice
    int scales_at;     // bytes of a slice in LDS before its scales
    int slice_bytes;   // bytes from one slice to the other where there are two, else 0
    float* partial;    // [parts][M][N], or null: one part, stored to Y
};

constexpr int CUS = 256;
// Chunks of W on their way to a wavefront: 4 x 16384 x 8192 23.9, 20.5 and 21.0 us with 1, 2 and 4, 8 x 16384 x 8192 in bf16
// 18.2, 17.6 and 20.1, 16 x 512 x 512 4.06, 4.14 and 4.58: the loop is as many chunks long, and small products also wait for code.
constexpr int DEPTH = 2;

// Chunks of a slice, of X in R MT rows and of the scales.  LDS holds two slices where it has room: the next one is put there
// by some wavefronts while others still work on this one, and a slice costs one barrier instead of two (against one slice
// of twice the length: 8 x 16384 x 8192 in bf16 17.9 us for 18.8, 32 x 16384 x 8192 37 for 39, 16 x 512 x 512 4.2 for 4.9, but
// 6 x 200 x 16000 9.6 for 8.8).  Up to four rows in fp32 their eight wavefronts along the contraction need long slices.
constexpr int slice_chunks(int r, int mt, bool x_bf16) { return r == 4 ? 16 : mt == 1 ? (x_bf16 ? 8 : 4) : x_bf16 ? 4 : 2; }
// whether LDS has room for two slices
constexpr bool two_slices(int r, int mt, bool x_bf16) { return r == 16 && (x_bf16 || mt <= 2); }
// scales of a row in a slice; bytes from row to row in LDS
constexpr int slice_scales(int slice, int group) { return slice * (128 / group); }
constexpr int scales_pitch(int slice, int group) { return slice_scales(slice, group) * 2 + 16; }

struct GemmArguments {  // as they lie in memory
    W4Args a;
    GemmShape g;
};

// The products with what the parts of X leave over, its 16 bits as two parts, slice by slice and nothing ahead: rare.  It
// reads the arguments again, so that its needs take no registers from what runs before it: inside the main loop, as its second
// time round, it cost every call 1 us.  Seeing that there is something costs 0.1 to 0.2 us (16 x 512 x 512 4.15 us without and
// 4.28 with, 24 x 4100 x 4090 13.8 and 14.1, 64 x 16384 x 8192 57.8 and 59.3); where a workgroup's X has such numbers the call
// takes 2.4 to 4 times as long (10.3, 33 and 230).
template <int R, int MT, int NT, int GROUP>
__device__ __forceinline__ void add_left_over(char* lds, f32x4 (&acc)[MT][NT]) {
    constexpr int SLICE = slice_chunks(R, MT, false), TILE_BYTES = R * 64, PART_BYTES = MT * TILE_BYTES, STEP_BYTES = 2 * PART_BYTES + 16;
    auto memory = (__attribute__((address_space(4))) const GemmArguments*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(memory));
    const auto& a = memory->a;
    const unsigned thread = threadIdx.x;
    const int lane = thread & 63, wave = __builtin_amdgcn_readfirstlane(thread >> 6), ln = lane & 15, lj = lane >> 4;
    const int log_kw = memory->g.log_kw, kw = 1 << log_kw, wk = wave & (kw - 1);
    const long n0 = ((long)blockIdx.x * (WAVES >> log_kw) + (wave >> log_kw)) * (16 * NT), m0 = (long)blockIdx.y * (R * MT);
    const int rows = (int)min((long)(R * MT), a.M - m0), chunks = (a.K + 127) / 128, units = (a.K + 31) / 32;
    const int first = blockIdx.z * memory->g.split_chunks, end = min(chunks, first + memory->g.split_chunks);
#pragma unroll 1
    for (int base = first; base < end; base += SLICE) {
        const int width = min(SLICE, end - base) * 128;
        __syncthreads();
#pragma unroll 1
        for (int q = thread; q < rows * width; q += 64 * WAVES) {
            const int r = q / width, p = q % width, col = base * 128 + p;
            const float x = col < a.K ? left_over(((const unsigned*)a.X)[(m0 + r) * a.ldx + col]) : 0.0f;
            unsigned h[3];
            split3(__builtin_bit_cast(unsigned, x), h[0], h[1], h[2]);
            char* at = lds + (p / 32) * STEP_BYTES + (r / R) * TILE_BYTES + (p % 32 / 8 * R + r % R) * 16 + p % 8 * 2;
            reinterpret_cast<unsigned short*>(at)[0] = h[0] >> 16;
            reinterpret_cast<unsigned short*>(at + PART_BYTES)[0] = h[1] >> 16;
        }
        __syncthreads();
#pragma unroll 1
        for (int c = base + wk; c < min(end, base + SLICE); c += kw) {
            const char* xs = lds + (c - base) * (4 * STEP_BYTES) + (lj * R + min(ln, R - 1)) * 16;
#pragma unroll
            for (int t = 0; t < NT; t++) {
                const long n = min(n0 + t * 16 + ln, (long)a.N - 1);
                const u32x4 codes = transpose4(*reinterpret_cast<const u32x4*>(a.codes + n * a.row_bytes + (long)min(c * 4 + lj, units - 1) * 16));
#pragma unroll
                for (int s = 0; s < 4; s++) {
                    float scale = c * 4 + s < units ? bf16_to_f32(a.scales[n * a.groups + (c * 4 + s) / (GROUP / 32)]) : 0.0f;
                    if (!(fabsf(scale) < INFINITY)) scale = 0.0f;  // the sum has what it makes of it
                    scale *= 0x1p-32f;  // loses bits where these products are below 2^-200
                    const bf16x8 v = values8_bf16(codes[s]);
#pragma unroll
                    for (int i = 0; i < MT; i++) {
                        const char* at = xs + s * STEP_BYTES + i * TILE_BYTES;
                        f32x4 part = {0.f, 0.f, 0.f, 0.f};
                        part = __builtin_amdgcn_mfma_f32_16x16x32_bf16(*reinterpret_cast<const bf16x8*>(at + PART_BYTES), v, part, 0, 0, 0);
                        part = __builtin_amdgcn_mfma_f32_16x16x32_bf16(*reinterpret_cast<const bf16x8*>(at), v, part, 0, 0, 0);
                        asm volatile("" ::: "memory");  // one at a time: few registers
#pragma unroll
                        for (int r = 0; r < 4; r++) acc[i][t][r] = __builtin_fmaf(part[r], scale, acc[i][t][r]);
                    }
                }
            }
        }
    }
}

// X in fp32 leaves room in LDS for one workgroup on a CU, two wavefronts to a SIMD: said here, the compiler spends the registers
// (16 x 16384 x 8192 24.1 us for 24.9, 24 x 4100 x 4090 14.3 for 14.6)
template <int R, int MT, int NT, bool XBF, int GROUP>
__global__ __launch_bounds__(64 * WAVES) __attribute__((amdgpu_waves_per_eu(2, XBF || R == 4 ? 8 : 2))) void gemm_w4_kernel(const W4Args a, const GemmShape g) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    __shared__ unsigned leaves[XBF ? 1 : WAVES];  // whether a wavefront's X leaves something over
    constexpr int PARTS = XBF ? 1 : 3, STEPS = GROUP / 32, SLICE = slice_chunks(R, MT, XBF), PIECES = R * MT * SLICE / 32;
    constexpr int SCALES = slice_scales(SLICE, GROUP), COUNT = SCALES < 8 ? SCALES : 8, RUNS = SCALES / COUNT, PITCH = scales_pitch(SLICE, GROUP);
    constexpr int SCALE_TURNS = (16 * NT * WAVES * RUNS + 64 * WAVES - 1) / (64 * WAVES);
    // LDS: [step of 32 columns][part][tile of R rows][unit of 8 columns][row], 16 bytes each: a wavefront reads an operand as
    // one run; the steps are 16 bytes further apart, and the upper two units' rows in another order (row ^ 4), so that a run of
    // a row's pieces is written to different banks (half of the conflicts: 64 x 16384 x 8192 59 -> 55.5 us).  An order that differs
    // in each unit makes reads collide, and threads that take pieces below each other read rows that are often a power of
    // two apart: both slower
    constexpr int TILE_BYTES = R * 64, PART_BYTES = MT * TILE_BYTES, STEP_BYTES = PARTS * PART_BYTES + 16, SWIZZLE = R == 16 ? 4 : 0;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int ln = lane & 15, lj = lane >> 4;
    const int kw = 1 << g.log_kw, columns = WAVES >> g.log_kw;  // wavefronts along the contraction, along N
    const int wk = wave & (kw - 1), wn = wave >> g.log_kw;
    const long n0 = ((long)blockIdx.x * columns + wn) * (16 * NT);
    const long m0 = (long)blockIdx.y * (R * MT);
    const int rows = (int)min((long)(R * MT), a.M - m0);
    const int chunks = (a.K + 127) / 128, units = (a.K + 31) / 32;
    const int first = blockIdx.z * g.split_chunks, end = min(chunks, first + g.split_chunks);
    const unsigned char* wrow[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) {  // rows past the end repeat the last one; what they give is not stored
        const long n = min(n0 + t * 16 + ln, (long)a.N - 1);
        wrow[t] = a.codes + n * a.row_bytes;
    }
    // A wavefront's turns: SLICE / kw in each slice but the last, which has what is left.  Within a slice they begin at
    // a place that differs from workgroup to workgroup.
    const int log_turns = __builtin_ctz(SLICE) - g.log_kw;
    const unsigned place = (blockIdx.x * 0x9E3779B1u) >> 16;
    const int turns_all = end - first > wk ? (end - first - wk + kw - 1) >> g.log_kw : 0;
    auto chunk_of = [&](int turn) {  // of turns_all
        const int slice = turn >> log_turns, in_slice = turn - (slice << log_turns);
        const int count = min(1 << log_turns, turns_all - (slice << log_turns));
        int i = in_slice + (int)((place * (unsigned)count) >> 16);
        if (i >= count) i -= count;
        return first + slice * SLICE + wk + (i << g.log_kw);
    };
    auto load = [&](u32x4* w, int turn) {
        const int c = chunk_of(min(turn, turns_all - 1));  // past the end: the last one again
#pragma unroll
        for (int t = 0; t < NT; t++) w[t] = *reinterpret_cast<const u32x4*>(wrow[t] + (long)min(c * 4 + lj, units - 1) * 16);
    };
    f32x4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
        for (int t = 0; t < NT; t++) acc[i][t] = f32x4{0.f, 0.f, 0.f, 0.f};

    // A thread's pieces of a slice: SLICE * 16 pieces in a row, R MT SLICE * 16 = PIECES * 512 of them.  A piece that holds the
    // row's last columns and others past them is put together by itself.
    Piece<XBF> piece[PIECES];
    auto at_piece = [&](char* to, int r, int p) { return to + (p / 4) * STEP_BYTES + (r / R) * TILE_BYTES + ((p % 4) * R + (r % R ^ (p % 4 / 2 * SWIZZLE))) * 16; };
    auto load_x = [&](int base) {
#pragma unroll
        for (int k = 0; k < PIECES; k++) {
            const int q = threadIdx.x + k * 64 * WAVES, r = q / (SLICE * 16), col = base * 128 + q % (SLICE * 16) * 8;
            piece[k].zero();
            if (r < rows && col + 8 <= a.K) piece[k].load((const char*)a.X + (m0 + r) * a.ldx * (XBF ? 2 : 4), col);
        }
    };
    auto stage_x = [&](char* to, int base) {
        unsigned left = 0;
        const int width = min(SLICE, end - base) * 16;  // pieces of a row that are looked at
#pragma unroll
        for (int k = 0; k < PIECES; k++) {
            const int q = threadIdx.x + k * 64 * WAVES, r = q / (SLICE * 16), p = q % (SLICE * 16), col = base * 128 + p * 8;
            if (r < rows && p < width && (col + 8 <= a.K || col >= a.K)) {
                u32x4 o[PARTS];
                left |= piece[k].operands(o);
                char* at = at_piece(to, r, p);
#pragma unroll
                for (int part = 0; part < PARTS; part++) *reinterpret_cast<u32x4*>(at + part * PART_BYTES) = o[part];
            }
        }
        const int ragged = a.K / 8 * 8;
        if (ragged != a.K && ragged >= base * 128 && ragged < (base + SLICE) * 128 && ragged < end * 128) {
#pragma unroll 1
            for (int q = threadIdx.x; q < rows * 8; q += 64 * WAVES) {
                const int r = q / 8, col = ragged + q % 8;
                unsigned h[3] = {0, 0, 0};
                if (col < a.K) {
                    const long from = (m0 + r) * a.ldx + col;
                    if constexpr (XBF) h[0] = (unsigned)((const unsigned short*)a.X)[from] << 16;
                    else split3_any(((const unsigned*)a.X)[from], h[0], h[1], h[2]);
                    left |= XBF ? 0 : h[2];
                }
                char* at = at_piece(to, r, ragged / 8 - base * 16) + (q % 8) * 2;
#pragma unroll
                for (int part = 0; part < PARTS; part++) *reinterpret_cast<unsigned short*>(at + part * PART_BYTES) = h[part] >> 16;
            }
        }
        if constexpr (!XBF) {
            if ((left & 0xFFFFu) != 0) leaves[wave] = 1;
        }
    };
    // rows past the end are read as what LDS holds there, or as the last row where R < 16: their sums are not stored
    const int xlane = (lj * R + (min(ln, R - 1) ^ (lj / 2 * SWIZZLE))) * 16;

    // the scales of the slice, of all rows of W of the workgroup: read in runs along a row, once for the wavefronts that
    // split the contraction, and one slice ahead like X
    Scales<COUNT> scales[SCALE_TURNS];
    auto scales_of = [&](int k, int& row, int& run) {
        const int q = threadIdx.x + k * 64 * WAVES;
        row = q / RUNS, run = q % RUNS;
        return row < columns * 16 * NT;
    };
    auto load_scales = [&](int base) {
#pragma unroll
        for (int k = 0; k < SCALE_TURNS; k++) {
            int row, run;
            if (scales_of(k, row, run)) {
                const long n = min((long)blockIdx.x * (columns * 16 * NT) + row, (long)a.N - 1);
                scales[k].load(a.scales + n * a.groups, base * (128 / GROUP) + run * COUNT, a.groups);
            }
        }
    };
    auto stage_scales = [&](char* to, int base) {
#pragma unroll
        for (int k = 0; k < SCALE_TURNS; k++) {
            int row, run;
            if (scales_of(k, row, run)) scales[k].put(to + g.scales_at + row * PITCH + run * COUNT * 2, base * (128 / GROUP) + run * COUNT, a.groups);
        }
    };
    const int slane = g.scales_at + (wn * 16 * NT + ln) * PITCH;

    u32x4 w[DEPTH][NT];
    load_scales(first);
    load_x(first);  // before W: loads come back in their order, and X is waited for first
    if (turns_all) {
#pragma unroll
        for (int d = 0; d < DEPTH; d++) load(w[d], d);
    }
    auto chunk = [&](const char* slice, const u32x4* w, int turn, int base) {
        const int at = chunk_of(turn) - base;
        const char* xs = slice + xlane + at * (4 * STEP_BYTES);
        u32x4 codes[NT];
        float scales[NT][128 / GROUP];
#pragma unroll
        for (int t = 0; t < NT; t++) {
            codes[t] = transpose4(w[t]);
            const char* from = slice + slane + t * 16 * PITCH + at * (256 / GROUP);
            if constexpr (GROUP == 128) {
                scales[t][0] = bf16_to_f32(*reinterpret_cast<const unsigned short*>(from));
            } else {
#pragma unroll
                for (int k = 0; k < 64 / GROUP; k++) {
                    const unsigned two = reinterpret_cast<const unsigned*>(from)[k];
                    scales[t][2 * k] = __builtin_bit_cast(float, two << 16);
                    scales[t][2 * k + 1] = __builtin_bit_cast(float, two & 0xFFFF0000u);
                }
            }
        }
        f32x4 part[MT][NT];
#pragma unroll
        for (int s = 0; s < 4; s++) {
            bf16x8 x[MT][PARTS];
#pragma unroll
            for (int i = 0; i < MT; i++)
#pragma unroll
                for (int k = 0; k < PARTS; k++)
                    x[i][k] = *reinterpret_cast<const bf16x8*>(xs + s * STEP_BYTES + k * PART_BYTES + i * TILE_BYTES);
#pragma unroll
            for (int t = 0; t < NT; t++) {
                const bf16x8 v = values8_bf16(codes[t][s]);
                const float scale = scales[t][s / STEPS];
#pragma unroll
                for (int i = 0; i < MT; i++) {
                    if (s % STEPS == 0) part[i][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int k = PARTS - 1; k >= 0; k--)
                        part[i][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[i][k], v, part[i][t], 0, 0, 0);
                    if (s % STEPS == STEPS - 1) {
#pragma unroll
                        for (int r = 0; r < 4; r++) acc[i][t][r] = __builtin_fmaf(part[i][t][r], scale, acc[i][t][r]);
                    }
                }
            }
        }
    };
    // what leaves something over is told of in LDS before a slice's barrier, and looked up well before it is asked for
    unsigned some_leave = 0;  // one wavefront's to a lane
    auto look = [&] {
        if constexpr (!XBF) some_leave = leaves[lane % WAVES];
    };
    if constexpr (!XBF) leaves[wave] = 0;
    int turn = 0;
    auto work_on = [&](const char* slice, int base) {
        const int stop = min(turns_all, turn + (1 << log_turns));
        // a whole slice that others follow has a multiple of DEPTH turns
        for (; turn < stop; turn += DEPTH) {
#pragma unroll
            for (int d = 0; d < DEPTH; d++) {
                if (turn + d < stop) chunk(slice, w[d], turn + d, base);
                load(w[d], turn + d + DEPTH);
                asm volatile("" ::: "memory");  // the loads stay here, turns ahead of their use
            }
        }
    };
    // the first time round there is no slice to work on yet
    if constexpr (two_slices(R, MT, XBF)) {
        int here = g.slice_bytes, other = 0;
        for (int base = first - SLICE; base < end; base += SLICE) {
            if (base + SLICE < end) {
                stage_scales(lds + other, base + SLICE);
                stage_x(lds + other, base + SLICE);
            }
            if (base + 2 * SLICE < end) {
                load_scales(base + 2 * SLICE);
                load_x(base + 2 * SLICE);
            }
            look();
            if (base >= first) work_on(lds + here, base);
            __syncthreads();
            const int before = here;
            here = other;
            other = before;
        }
    } else {
        for (int base = first - SLICE; base < end; base += SLICE) {
            const bool more = base + SLICE < end;
            if (more && base >= first) {
                load_scales(base + SLICE);
                load_x(base + SLICE);
            }
            if (base >= first) {
                look();
                work_on(lds, base);
                __syncthreads();
            }
            if (more) {
                stage_scales(lds, base + SLICE);
                stage_x(lds, base + SLICE);
                __syncthreads();
            }
        }
    }

    // lane (ln, lj) holds column ln, rows 4 lj .. 4 lj + 3 of each 16 x 16 tile; the wavefronts of a column add up
    f32x4* sums = reinterpret_cast<f32x4*>(lds);  // [wavefronts][NT][64]
    auto put_sums = [&](int i) {
#pragma unroll
        for (int t = 0; t < NT; t++) sums[(wave * NT + t) * 64 + lane] = acc[i][t];
    };
    put_sums(0);
    __syncthreads();
    if constexpr (!XBF) {
        if (__builtin_expect(__any(some_leave != 0), 0)) {
            add_left_over<R, MT, NT, GROUP>(lds, acc);
            __syncthreads();
            put_sums(0);
            __syncthreads();
        }
    }
#pragma unroll
    for (int i = 0; i < MT; i++) {
        if (i) {
            __syncthreads();
            put_sums(i);
            __syncthreads();
        }
        for (int e = threadIdx.x; e < columns * NT * 64; e += 64 * WAVES) {
            const int group = e / (NT * 64), rest = e % (NT * 64);
            f32x4 y = sums[group * kw * NT * 64 + rest];
            for (int k = 1; k < kw; k++) {
                const f32x4 z = sums[(group * kw + k) * NT * 64 + rest];
#pragma unroll
                for (int r = 0; r < 4; r++) y[r] += z[r];
            }
            const long n = ((long)blockIdx.x * columns + group) * (16 * NT) + (rest >> 6) * 16 + (rest & 15);
            const int at = ((rest & 63) >> 4) * 4;  // row in the tile
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const long m = m0 + i * R + at + r;
                if (n >= a.N || at + r >= R || m >= a.M) continue;
                if (g.partial) g.partial[((long)blockIdx.z * a.M + m) * a.N + n] = y[r];
                else store_y(a, m * a.ldy + n, y[r]);
            }
        }
    }
}

// the parts of a split contraction, added in their order; four columns to a thread, a row of Y to gridDim.y
__global__ __launch_bounds__(256) void join_w4_kernel(const W4Args a, const float* partial, int parts) {
    const int n = (blockIdx.x * 256 + threadIdx.x) * 4;
    const long m = blockIdx.y, size = (long)a.M * a.N;
    if (n >= a.N) return;
    const float* p = partial + m * a.N + n;
    const int columns = min(4, a.N - n);
    f32x4 y = {0.f, 0.f, 0.f, 0.f};
    if (columns == 4) {
        y = *reinterpret_cast<const f32x4u*>(p);
#pragma unroll 4
        for (int k = 1; k < parts; k++) {
            const f32x4 z = *reinterpret_cast<const f32x4u*>(p + k * size);
#pragma unroll
            for (int r = 0; r < 4; r++) y[r] += z[r];
        }
    } else {
        for (int k = 0; k < parts; k++)
#pragma unroll
            for (int r = 0; r < 3; r++)
                if (r < columns) y[r] = k ? y[r] + p[k * size + r] : p[r];
    }
#pragma unroll
    for (int r = 0; r < 4; r++)
        if (r < columns) store_y(a, m * a.ldy + n + r, y[r]);
}

struct Costs {
    float x, weight, product, read, slice, join, part, value;
};
constexpr Costs F32_COSTS = {7.5e-5f, 7.7e-6f, 1.14e-5f, 0.0f, 0.44f, 2.3f, 0.075f, 2.7e-6f};
constexpr Costs BF16_COSTS = {2.1e-5f, 5.5e-6f, 7.6e-6f, 4.4e-6f, 0.36f, 2.36f, 0.07f, 1.4e-6f};

struct GemmPlan {
    int r, mt, nt, log_kw, parts, split_chunks;
};

// The shape of a launch is the one whose estimated time is least (us on 256 CUs, a workgroup at a time on each): so much for
// a value of X (brought in, split, put in LDS), for a weight (brought in and converted), for a weight and a tile of rows
// (multiplied), for a tile of X read from LDS for 16 NT columns, for a slice, for the second kernel that joins parts, for a part,
// and for a value of one (written and read).  The numbers are fitted to 3600 measured launches of 41 shapes (3 to 200
// rows, 200 to 32768 columns, K from 500 to 16384) so that the shapes they find are the fastest ones measured: they
// were within 5 % of those for 36 of them and within 10 % for all.  (That was before the present order of X in LDS, and before
// what is left over of X was looked for.)  What decides, with both sides measured on the code as it is (X in fp32); the shapes
// found are the fastest of these or within 1 %:
//   rows to a workgroup: 64 x 16384 x 8192 58.2 us with 64, 58.1 with 32 and 64.6 with 16, but 64 x 512 x 512 4.3 with 16 and 7.4
// with 32
//   columns of a wavefront, 16 or 32: 16 x 16384 x 8192 28.0 and 25.0 us, but 64 x 512 x 512 4.3 and 5.2
//   wavefronts along the contraction: 3 x 4096 x 4096 6.3, 7.7, 10.7 and 16.7 us with 8, 4, 2 and 1; 16 x 16384 x 8192 25.0 with 1
// and 27.6 with 2
//   parts: 24 x 4100 x 4090 37.2, 23.6, 14.0 and 18.2 us with 1, 2, 6 and 12
GemmPlan plan_gemm(int M, int N, int K, bool x_bf16) {
    GemmPlan best = {};
    const int chunks = K / 128 + (K % 128 != 0), r = M <= 4 ? 4 : 16;
    const Costs& of = x_bf16 ? BF16_COSTS : F32_COSTS;
    float least = INFINITY;
    for (int mt = 1; mt == 1 || (mt <= 4 && 8 * mt < M); mt *= 2) {
        const int slice = slice_chunks(r, mt, x_bf16);
        const long m_blocks = (M + r * mt - 1L) / (r * mt);
        for (int nt = 1; nt <= 2; nt++)
            for (int log_kw = 0; log_kw <= 3 && slice >> log_kw && chunks >> log_kw; log_kw++) {
                const int columns = 16 * nt * (WAVES >> log_kw);
                const long n_blocks = ((long)N + columns - 1) / columns, blocks = n_blocks * m_blocks;
                if (n_blocks >= 1L << 23) continue;  // a launch has fewer than 2^32 threads in a row; 256 columns always do
                // as many parts as there are CUs for, half or a quarter of them, and one
                for (long want = std::min(std::min(64L, (long)chunks), std::max(1L, CUS / blocks)), turn = 0; turn < 4; turn++) {
                    const int parts = turn == 3 ? 1 : (int)(want >> turn);
                    if (parts < 1 || (parts == 1 && turn < 3)) continue;
                    int split = (chunks + parts - 1) / parts;
                    if (parts > 1 && split > slice) split = (split + slice - 1) / slice * slice;
                    if (split > slice && slice >> log_kw < DEPTH) continue;
                    const int used = (chunks + split - 1) / split;
                    const float depth = (float)std::min(split * 128L, (long)K), slices = (float)((split + slice - 1) / slice);
                    const float work = depth * (of.x * std::min(M, r * mt) + columns * (of.weight + mt * (of.product + of.read / nt))) + of.slice * slices;
                    float cost = (float)((blocks * used + CUS - 1) / CUS) * work;
                    if (used > 1) cost += of.join + used * (of.part + of.value * M * N);
                    if (cost < least) {
                        least = cost;
                        best = {r, mt, nt, log_kw, used, split};
                    }
                }
            }
    }
    return best;
}

template <int R, int MT, int NT, bool XBF, int GROUP>
hipError_t launch_gemm(const W4Args& a, const GemmPlan& p, float* partial) {
    constexpr int PARTS = XBF ? 1 : 3, SLICE = slice_chunks(R, MT, XBF);
    const size_t x_bytes = (size_t)std::min(SLICE, p.split_chunks) * 4 * (PARTS * MT * R * 64 + 16);
    const long columns = 16L * NT * (WAVES >> p.log_kw);
    const size_t slice_bytes = x_bytes + (size_t)columns * scales_pitch(SLICE, GROUP);
    const bool two = two_slices(R, MT, XBF) && p.split_chunks > SLICE;
    const size_t bytes = std::max(slice_bytes * (two ? 2 : 1), (size_t)WAVES * NT * 64 * 16);
    const GemmShape shape = {p.log_kw, p.split_chunks, (int)x_bytes, two ? (int)slice_bytes : 0, p.parts > 1 ? partial : nullptr};
    constexpr long MOST = 65535L * R * MT;  // rows of a launch: gridDim.y has 16 bits
    for (long m = 0; m < a.M; m += MOST) {
        W4Args some = a;
        some.M = (int)std::min(MOST, a.M - m);
        some.X = (const char*)a.X + m * a.ldx * (XBF ? 2 : 4);
        some.Y = (char*)a.Y + m * a.ldy * (a.y_bf16 ? 2 : 4);
        const dim3 grid((unsigned)((a.N + columns - 1) / columns), (unsigned)((some.M + R * MT - 1L) / (R * MT)), (unsigned)p.parts);
        hipLaunchKernelGGL((gemm_w4_kernel<R, MT, NT, XBF, GROUP>), grid, dim3(64 * WAVES), bytes, stream(), some, shape);
    }
    if (p.parts > 1)
        hipLaunchKernelGGL(join_w4_kernel, dim3((unsigned)((a.N + 1023L) / 1024), (unsigned)a.M), dim3(256), 0, stream(), a, partial, p.parts);
    return hipGetLastError();
}
template <int R, int MT, int NT>
hipError_t launch_gemm(const W4Args& a, const GemmPlan& p, float* partial) {
    if (a.x_bf16) {
        if (a.group == 32) return launch_gemm<R, MT, NT, true, 32>(a, p, partial);
        if (a.group == 64) return launch_gemm<R, MT, NT, true, 64>(a, p, partial);
        return launch_gemm<R, MT, NT, true, 128>(a, p, partial);
    }
    if (a.group == 32) return launch_gemm<R, MT, NT, false, 32>(a, p, partial);
    if (a.group == 64) return launch_gemm<R, MT, NT, false, 64>(a, p, partial);
    return launch_gemm<R, MT, NT, false, 128>(a, p, partial);
}
template <int R, int MT>
hipError_t launch_gemm(const W4Args& a, const GemmPlan& p, float* partial) {
    return p.nt == 1 ? launch_gemm<R, MT, 1>(a, p, partial) : launch_gemm<R, MT, 2>(a, p, partial);
}

template <int M>
hipError_t launch_gemv(const W4Args& a) {
    const int units = a.K / 32 + (a.K % 32 != 0);
    GemvShape g = {0, 0, GEMV_LOADS, 0};
    while (g.log_lanes < 6 && (1 << g.log_lanes) < units) g.log_lanes++;
    while (g.log_kw < 3 && (64 << g.log_kw) < units) g.log_kw++;
    g.stride = std::max(16, 1 << (g.log_lanes + g.log_kw)) * 16 + 128;
    // As few rows to a wavefront as leave one workgroup per CU, or two where X takes no LDS: 1 x 16384 x 8192 in bf16
    // takes 23.1, 16.5, 13.8, 13.0 and 13.9 us with 2, 4, 8, 16 and 32 loads (512 workgroups with 16), in fp32 14.6 us with 32
    // (256 workgroups) and 15.1 with 16; 1 x 512 x 512 takes 3.1 us with 2 and 5.0 with 8.
    const long row = (64 >> g.log_lanes) * (WAVES >> g.log_kw);
    while (g.loads < 32 && g.loads * row < 4096 && a.N / (g.loads * row) >= (a.x_bf16 ? 512 : 256) + 1) g.loads *= 2;
    const long block_rows = g.loads * row;
    const dim3 grid((unsigned)((a.N + block_rows - 1) / block_rows));
    const size_t bytes = (a.x_bf16 ? 0 : (size_t)M * 8 * g.stride) + (size_t)block_rows * (M << g.log_kw) * sizeof(float);
    if (a.x_bf16) hipLaunchKernelGGL((gemv_w4_kernel<M, true>), grid, dim3(64 * WAVES), bytes, stream(), a, g);
    else hipLaunchKernelGGL((gemv_w4_kernel<M, false>), grid, dim3(64 * WAVES), bytes, stream(), a, g);
    return hipGetLastError();
}

bool group_ok(int group) { return group == 32 || group == 64 || group == 128; }
bool type_ok(int t) { return t == NERF_TYPE_F32 || t == NERF_TYPE_BF16; }
int ceil_div(int a, int b) { return a / b + (a % b != 0); }

// launch shape of the two conversions, `block` pieces to a workgroup
dim3 piece_grid(int rows, unsigned per_row, unsigned block) {
    const unsigned slab = SLAB / per_row;
    const unsigned in_slab = std::min((unsigned)rows, slab);
    return dim3((unsigned)(((unsigned long long)in_slab * per_row + block - 1) / block), ((unsigned)rows + slab - 1) / slab);
}

}  // namespace
}  // namespace nerf

using namespace nerf;

extern "C" {

size_t nerf_w4_row_bytes(int cols) { return cols > 0 ? ((size_t)cols + 31) / 32 * 16 : 0; }

int nerf_quantize_w4(const float* d_src, long ld_src, int rows, int cols, int group, unsigned char* d_codes,
                     unsigned short* d_scales) {
    if (!d_src || !d_codes || !d_scales || rows <= 0 || cols <= 0 || cols > NERF_W4_MAX_DIM || ld_src < cols || !group_ok(group) ||
        ((uintptr_t)d_src & 3) || ((uintptr_t)d_codes & 15) || ((uintptr_t)d_scales & 1))
        return NERF_ERR_ARG;
    const int groups = ceil_div(cols, group);
    const unsigned per_row = (unsigned)groups * (unsigned)(group / 8);
    const long row_bytes = (long)nerf_w4_row_bytes(cols);
    ProfScope prof(K_QUANTIZE_W4, (double)rows * cols * 4.5);
    const auto kernel = group == 32 ? quantize_w4_kernel<32> : group == 64 ? quantize_w4_kernel<64> : quantize_w4_kernel<128>;
    hipLaunchKernelGGL(kernel, piece_grid(rows, per_row, 256), dim3(256), 0, stream(), d_src, ld_src, rows, cols, per_row, d_codes, row_bytes,
                       d_scales, groups);
    return hipGetLastError() == hipSuccess ? NERF_OK : NERF_ERR_HIP;
}

int nerf_dequantize_w4(const unsigned char* d_codes, const unsigned short* d_scales, int rows, int cols, int group,
                       float* d_dst, long ld_dst) {
    if (!d_dst || !d_codes || !d_scales || rows <= 0 || cols <= 0 || cols > NERF_W4_MAX_DIM || ld_dst < cols || !group_ok(group) ||
        ((uintptr_t)d_dst & 3) || ((uintptr_t)d_codes & 15) || ((uintptr_t)d_scales & 1))
        return NERF_ERR_ARG;
    const unsigned per_row = (unsigned)ceil_div(cols, 4);
    ProfScope prof(K_QUANTIZE_W4, (double)rows * cols * 4.5);
    hipLaunchKernelGGL(dequantize_w4_kernel, piece_grid(rows, per_row, 512), dim3(256), 0, stream(), d_codes, (long)nerf_w4_row_bytes(cols),
                       d_scales, ceil_div(cols, group), group, rows, cols, per_row, d_dst, ld_dst);
    return hipGetLastError() == hipSuccess ? NERF_OK : NERF_ERR_HIP;
}

size_t nerf_gemm_w4_workspace(int M, int N, int K) {
    const int chunks = ceil_div(std::max(K, 0), 128);
    if (M <= 2 || N <= 0 || chunks < 2) return 0;
    // Fewer rows may be split into more parts, and a workspace for many rows has to serve fewer: so this is not the plan's own
    // size but a bound that grows with each of the three.  A plan has at most min(64, chunks) parts; where it has several,
    // its workgroups times its parts are at most CUS, and a workgroup has at most 64 x 256 values.
    const size_t workgroups = (size_t)CUS * std::min(M, 64) * std::min(N, 256), parts = std::min(64, chunks);
    const size_t values = (size_t)M * N;  // below 2^61
    return sizeof(float) * (values > workgroups / parts ? workgroups : values * parts);
}

int nerf_gemm_w4(const void* d_X, int x_type, long ldx, const unsigned char* d_codes, const unsigned short* d_scales,
                 int group, void* d_Y, int y_type, long ldy, int M, int N, int K, int epilogue, void* d_workspace,
                 size_t workspace_bytes) {
    if (!d_X || !d_codes || !d_scales || !d_Y || M <= 0 || N <= 0 || K <= 0 || N > NERF_W4_MAX_DIM || K > NERF_W4_MAX_DIM || ldx < K || ldy < N || !group_ok(group) ||
        !type_ok(x_type) || !type_ok(y_type) || (epilogue != 0 && epilogue != 1) || ((uintptr_t)d_codes & 15) ||
        ((uintptr_t)d_scales & 1) || ((uintptr_t)d_X & (x_type == NERF_TYPE_BF16 ? 1 : 3)) ||
        ((uintptr_t)d_Y & (y_type == NERF_TYPE_BF16 ? 1 : 3)) || ((uintptr_t)d_workspace & 15))
        return NERF_ERR_ARG;
    GemmPlan p = {};
    if (M > 2) p = plan_gemm(M, N, K, x_type == NERF_TYPE_BF16);
    const size_t need = nerf_gemm_w4_workspace(M, N, K);
    if (workspace_bytes < need || (need && !d_workspace)) return NERF_ERR_ARG;
    W4Args a = {};
    a.X = d_X; a.codes = d_codes; a.scales = d_scales; a.Y = d_Y;
    a.ldx = ldx; a.ldy = ldy; a.row_bytes = (long)nerf_w4_row_bytes(K);
    a.M = M; a.N = N; a.K = K; a.group = group; a.groups = ceil_div(K, group);
    a.x_bf16 = x_type == NERF_TYPE_BF16; a.y_bf16 = y_type == NERF_TYPE_BF16; a.epilogue = epilogue;
    ProfScope prof(K_GEMM_W4, 2.0 * M * N * K);
    float* partial = (float*)d_workspace;
    hipError_t rc;
    if (M == 1) rc = launch_gemv<1>(a);
    else if (M == 2) rc = launch_gemv<2>(a);
    else if (p.mt == 4) rc = launch_gemm<16, 4>(a, p, partial);
    else if (p.mt == 2) rc = launch_gemm<16, 2>(a, p, partial);
    else rc = p.r == 16 ? launch_gemm<16, 1>(a, p, partial) : launch_gemm<4, 1>(a, p, partial);
    return rc == hipSuccess ? NERF_OK : NERF_ERR_HIP;
}

}  // extern "C"
