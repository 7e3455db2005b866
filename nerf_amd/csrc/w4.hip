// w4.hip -- weights in 4 bits with a bf16 scale per group: quantize, dequantize, and products of a few rows with them.
//
// No counterpart in the reference (fp32 cuBLAS only).  Codes are the small floats 0, 0.5, 1, 1.5, 2, 3, 4, 6 with a
// sign, which gfx950 converts two at a time (v_cvt_scalef32_pk_f32_fp4); rows are row-major, two codes to a byte and
// padded to 16 bytes, so 16 bytes are 32 consecutive columns: one "unit".
#include "common.hpp"
#include "../../include/nerf_amd.h"

#include <algorithm>

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

// the eight values of a dword of codes
__device__ __forceinline__ void values8(unsigned c, float* v) {
    const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 1);
    const f32x2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 2), e = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 3);
    v[0] = a[0]; v[1] = a[1]; v[2] = b[0]; v[3] = b[1];
    v[4] = d[0]; v[5] = d[1]; v[6] = e[0]; v[7] = e[1];
}

// ---- quantize -------------------------------------------------------------------------------------------
// A thread takes eight consecutive columns of a row; the 4, 8 or 16 threads of a group are neighbours in a row of
// sixteen lanes.  `per_row` threads (whole groups) belong to a row.
template <int GROUP>
__global__ __launch_bounds__(256) void quantize_w4_kernel(const float* __restrict__ src, long ld, int rows, int cols,
                                                          unsigned per_row, unsigned char* __restrict__ codes,
                                                          long row_bytes, unsigned short* __restrict__ scales, int groups) {
    const unsigned id = blockIdx.x * 256 + threadIdx.x;
    const unsigned slab_row = id / per_row, piece = id - slab_row * per_row;
    const long row = (long)blockIdx.y * (0x40000000u / per_row) + slab_row;
    const bool live = row < rows && slab_row < 0x40000000u / per_row;
    const int col = (int)piece * 8;
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (live) {
        const float* p = src + row * ld + col;
        if (col + 8 <= cols) {
            const f32x4u a = *reinterpret_cast<const f32x4u*>(p), b = *reinterpret_cast<const f32x4u*>(p + 4);
#pragma unroll
            for (int k = 0; k < 4; k++) { x[k] = a[k]; x[k + 4] = b[k]; }
        } else {
            for (int k = 0; k < 8 && col + k < cols; k++) x[k] = p[k];
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
    const float scale = bad ? 0.0f : bf16_to_f32((unsigned short)s);
    if (!live) return;
    // steps between codes, where the value of the border (a multiple of the scale) is exact; a tie takes the even code
    unsigned word = 0;
#pragma unroll
    for (int k = 0; k < 8; k++) {
        const float a = fabsf(x[k]);
        unsigned c = (a > 0.25f * scale) + (a >= 0.75f * scale) + (a > 1.25f * scale) + (a >= 1.75f * scale) +
                     (a > 2.5f * scale) + (a >= 3.5f * scale) + (a > 5.0f * scale);
        if (bad || top == 0) c = 0;
        if (c && x[k] < 0.0f) c |= 8;
        word |= c << (4 * k);
    }
    if ((long)piece * 4 < row_bytes) *reinterpret_cast<unsigned*>(codes + row * row_bytes + (long)piece * 4) = word;
    if (piece % (GROUP / 8) == 0) scales[row * groups + piece / (GROUP / 8)] = bad ? 0x7FC0 : (unsigned short)s;
}

__global__ __launch_bounds__(256) void dequantize_w4_kernel(const unsigned char* __restrict__ codes, long row_bytes,
                                                            const unsigned short* __restrict__ scales, int groups, int group,
                                                            int rows, int cols, unsigned per_row, float* __restrict__ dst, long ld) {
    const unsigned id = blockIdx.x * 256 + threadIdx.x;
    const unsigned slab_row = id / per_row, piece = id - slab_row * per_row;
    const long row = (long)blockIdx.y * (0x40000000u / per_row) + slab_row;
    if (row >= rows || slab_row >= 0x40000000u / per_row) return;
    const int col = (int)piece * 8;
    const float scale = bf16_to_f32(scales[row * groups + col / group]);
    float v[8];
    values8(*reinterpret_cast<const unsigned*>(codes + row * row_bytes + (long)piece * 4), v);
    float* p = dst + row * ld + col;
    if (col + 8 <= cols) {
        *reinterpret_cast<f32x4u*>(p) = f32x4u{v[0] * scale, v[1] * scale, v[2] * scale, v[3] * scale};
        *reinterpret_cast<f32x4u*>(p + 4) = f32x4u{v[4] * scale, v[5] * scale, v[6] * scale, v[7] * scale};
    } else {
        for (int k = 0; k < 8 && col + k < cols; k++) p[k] = v[k] * scale;
    }
}

// ---- products -------------------------------------------------------------------------------------------
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

// One product for any number of rows: a workgroup takes 16 NT columns of Y (rows of W) and 16 MT rows of X; its
// wavefronts share out the contraction in chunks of 128 columns and add up in LDS at the end, so no piece of W or X is
// read twice in a workgroup.  Per chunk a lane loads 16 bytes (one unit of 32 columns) of one of 16 rows of W; four
// lane swaps turn the four units that four lanes hold of a row into the four steps of a matrix instruction
// (16 x 16 x 32, both operands bf16), so that a step's 32 columns lie in one group and its sum takes one scale.
//   Codes are bf16 numbers exactly.  An fp32 x goes as three bf16 numbers that add up to it exactly (its upper, middle
// and lower 8 significant bits, cut off), with one instruction each: products are exact, sums are fp32.
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x2u __attribute__((ext_vector_type(2), aligned(2)));
typedef unsigned u32u __attribute__((aligned(2)));
typedef unsigned u32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned u32x4u2 __attribute__((ext_vector_type(4), aligned(2)));

// eight codes as eight bf16
__device__ __forceinline__ bf16x8 values8_bf16(unsigned c) {
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, 1.0f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, 1.0f, 1);
    const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, 1.0f, 2), e = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, 1.0f, 3);
    return bf16x8{a[0], a[1], b[0], b[1], d[0], d[1], e[0], e[1]};
}

// upper halves of two words, the first one below
__device__ __forceinline__ unsigned upper_halves(unsigned lo, unsigned hi) { return __builtin_amdgcn_perm(hi, lo, 0x07060302); }

// what eight consecutive values of X are as matrix operands
template <bool XBF>
struct Operand;
template <>
struct Operand<true> {
    static constexpr int PARTS = 1;
    u32x4 p[1];
};
template <>
struct Operand<false> {
    static constexpr int PARTS = 3;
    u32x4 p[3];
};

template <bool XBF>
struct Raw {  // as loaded
    u32x4 a, b;  // eight fp32; bf16: a alone
};

template <bool XBF>
__device__ __forceinline__ Raw<XBF> load_raw(const void* row, int col, int K, bool whole) {
    Raw<XBF> r = {};
    if (XBF) {
        const unsigned short* p = (const unsigned short*)row + col;
        if (whole) r.a = *reinterpret_cast<const u32x4u2*>(p);
        else
#pragma unroll
            for (int k = 0; k < 8; k++)
                if (col + k < K) r.a[k / 2] |= (unsigned)p[k] << (16 * (k & 1));
    } else {
        const unsigned* p = (const unsigned*)row + col;
        if (whole) {
            r.a = *reinterpret_cast<const u32x4u*>(p);
            r.b = *reinterpret_cast<const u32x4u*>(p + 4);
        } else {
#pragma unroll
            for (int k = 0; k < 4; k++) {
                if (col + k < K) r.a[k] = p[k];
                if (col + 4 + k < K) r.b[k] = p[k + 4];
            }
        }
    }
    return r;
}

template <bool XBF>
__device__ __forceinline__ void split(const Raw<XBF>& r, Operand<XBF>& o) {
    if constexpr (XBF) {
        o.p[0] = r.a;
    } else {
        unsigned hi[8], mid[8], lo[8];
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const unsigned x = k < 4 ? r.a[k] : r.b[k - 4];
            hi[k] = x & 0xFFFF0000u;
            // infinity less itself would be NaN: what is not finite goes in the first part alone
            const float rest = __builtin_bit_cast(float, x) - __builtin_bit_cast(float, hi[k]);
            const unsigned m = (x & 0x7F800000u) == 0x7F800000u ? 0u : __builtin_bit_cast(unsigned, rest);
            mid[k] = m & 0xFFFF0000u;
            lo[k] = __builtin_bit_cast(unsigned, __builtin_bit_cast(float, m) - __builtin_bit_cast(float, mid[k]));
            // a NaN whose upper half alone would read as infinity stays a NaN
            if ((x & 0x7FFFFFFFu) > 0x7F800000u) hi[k] = 0x7FC00000u;
        }
#pragma unroll
        for (int k = 0; k < 4; k++) {
            o.p[0][k] = upper_halves(hi[2 * k], hi[2 * k + 1]);
            o.p[1][k] = upper_halves(mid[2 * k], mid[2 * k + 1]);
            o.p[2][k] = upper_halves(lo[2 * k], lo[2 * k + 1]);
        }
    }
}

// d[s] of lane group j (16 lanes each) becomes what d[j] of lane group s was
__device__ __forceinline__ void transpose4(u32x4& d) {
    auto a = __builtin_amdgcn_permlane32_swap(d[0], d[2], false, false);
    auto b = __builtin_amdgcn_permlane32_swap(d[1], d[3], false, false);
    auto c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
    auto e = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
    d = u32x4{c[0], c[1], e[0], e[1]};
}

template <int GROUP>
__device__ __forceinline__ void load_scales(const unsigned short* row, int chunk, int K, bool whole, float* s) {
    const int first = chunk * 128 / GROUP;
    if (whole) {
        if (GROUP == 32) {
            const u32x2u w = *reinterpret_cast<const u32x2u*>(row + first);
            s[0] = __builtin_bit_cast(float, w[0] << 16);
            s[1] = __builtin_bit_cast(float, w[0] & 0xFFFF0000u);
            s[2] = __builtin_bit_cast(float, w[1] << 16);
            s[3] = __builtin_bit_cast(float, w[1] & 0xFFFF0000u);
        } else if (GROUP == 64) {
            const unsigned w = *reinterpret_cast<const u32u*>(row + first);
            s[0] = s[1] = __builtin_bit_cast(float, w << 16);
            s[2] = s[3] = __builtin_bit_cast(float, w & 0xFFFF0000u);
        } else {
            s[0] = s[1] = s[2] = s[3] = bf16_to_f32(row[first]);
        }
    } else {
#pragma unroll
        for (int k = 0; k < 4; k++) s[k] = chunk * 128 + 32 * k < K ? bf16_to_f32(row[(chunk * 128 + 32 * k) / GROUP]) : 0.0f;
    }
}

template <int MT, int NT, bool XBF, int GROUP>
__global__ __launch_bounds__(512) void gemm_w4_kernel(const W4Args a) {
    extern __shared__ __attribute__((aligned(16))) f32x4 sums[];  // [wavefronts][NT][64]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    const int ln = lane & 15, lj = lane >> 4;
    const long n0 = (long)blockIdx.x * (16 * NT);
    const long m0 = (long)blockIdx.y * (16 * MT);
    const unsigned char* wrow[NT];
    const unsigned short* srow[NT];
    const char* xrow[MT];
#pragma unroll
    for (int t = 0; t < NT; t++) {  // rows past the end repeat the last one; what they give is not stored
        const long n = min(n0 + t * 16 + ln, (long)a.N - 1);
        wrow[t] = a.codes + n * a.row_bytes + lj * 16;
        srow[t] = a.scales + n * a.groups;
    }
#pragma unroll
    for (int t = 0; t < MT; t++)
        xrow[t] = (const char*)a.X + min(m0 + t * 16 + ln, (long)a.M - 1) * a.ldx * (XBF ? 2 : 4);
    f32x4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
        for (int t = 0; t < NT; t++) acc[i][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int chunks = (a.K + 127) / 128, units = (a.K + 31) / 32;
    for (int c = wave; c < chunks; c += waves) {
        const bool whole = c * 128 + 128 <= a.K;
        u32x4 d[NT];
        float scale[NT][4];
#pragma unroll
        for (int t = 0; t < NT; t++) {
            d[t] = u32x4{0, 0, 0, 0};
            if (whole || c * 4 + lj < units) d[t] = *reinterpret_cast<const u32x4*>(wrow[t] + (long)c * 64);
            load_scales<GROUP>(srow[t], c, a.K, whole, scale[t]);
        }
        Raw<XBF> raw[MT][4];
#pragma unroll
        for (int i = 0; i < MT; i++)
#pragma unroll
            for (int s = 0; s < 4; s++) raw[i][s] = load_raw<XBF>(xrow[i], c * 128 + 32 * s + 8 * lj, a.K, whole);
#pragma unroll
        for (int t = 0; t < NT; t++) transpose4(d[t]);
#pragma unroll
        for (int s = 0; s < 4; s++) {
            Operand<XBF> x[MT];
#pragma unroll
            for (int i = 0; i < MT; i++) split<XBF>(raw[i][s], x[i]);
#pragma unroll
            for (int t = 0; t < NT; t++) {
                const bf16x8 w = values8_bf16(d[t][s]);
#pragma unroll
                for (int i = 0; i < MT; i++) {
                    f32x4 part = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int q = Operand<XBF>::PARTS - 1; q >= 0; q--)
                        part = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x[i].p[q]), w, part, 0, 0, 0);
#pragma unroll
                    for (int r = 0; r < 4; r++) acc[i][t][r] = __builtin_fmaf(part[r], scale[t][s], acc[i][t][r]);
                }
            }
        }
    }
    // lane (ln, lj) holds column ln, rows 4 lj .. 4 lj + 3 of each 16 x 16 tile
#pragma unroll
    for (int i = 0; i < MT; i++) {
        if (i) __syncthreads();
#pragma unroll
        for (int t = 0; t < NT; t++) sums[(wave * NT + t) * 64 + lane] = acc[i][t];
        __syncthreads();
        for (int e = threadIdx.x; e < NT * 64; e += blockDim.x) {
            f32x4 y = sums[e];
            for (int w = 1; w < waves; w++) {
                const f32x4 z = sums[w * NT * 64 + e];
#pragma unroll
                for (int r = 0; r < 4; r++) y[r] += z[r];
            }
            const long n = n0 + (e >> 6) * 16 + (e & 15);
            const long m = m0 + i * 16 + ((e & 63) >> 4) * 4;
#pragma unroll
            for (int r = 0; r < 4; r++)
                if (n < a.N && m + r < a.M) store_y(a, (m + r) * a.ldy + n, y[r]);
        }
    }
}

template <int MT, int NT, bool XBF, int GROUP>
void launch_gemm(const W4Args& a) {
    const int chunks = (a.K + 127) / 128;
    int waves = 8;
    while (waves > 1 && waves / 2 >= chunks) waves /= 2;
    hipLaunchKernelGGL((gemm_w4_kernel<MT, NT, XBF, GROUP>),
                       dim3((unsigned)((a.N + 16L * NT - 1) / (16 * NT)), (unsigned)((a.M + 16L * MT - 1) / (16 * MT))),
                       dim3(64 * waves), waves * NT * 64 * sizeof(f32x4), stream(), a);
}
template <int MT, int NT>
void launch_gemm(const W4Args& a) {
    if (a.x_bf16) {
        if (a.group == 32) launch_gemm<MT, NT, true, 32>(a);
        else if (a.group == 64) launch_gemm<MT, NT, true, 64>(a);
        else launch_gemm<MT, NT, true, 128>(a);
    } else {
        if (a.group == 32) launch_gemm<MT, NT, false, 32>(a);
        else if (a.group == 64) launch_gemm<MT, NT, false, 64>(a);
        else launch_gemm<MT, NT, false, 128>(a);
    }
}

bool group_ok(int group) { return group == 32 || group == 64 || group == 128; }
bool type_ok(int t) { return t == NERF_TYPE_F32 || t == NERF_TYPE_BF16; }
int ceil_div(int a, int b) { return a / b + (a % b != 0); }

// launch shape of the two conversions: rows in slabs whose threads fit 32 bits
dim3 piece_grid(int rows, unsigned per_row) {
    const unsigned slab = 0x40000000u / per_row;
    const unsigned in_slab = std::min((unsigned)rows, slab);
    return dim3((unsigned)(((unsigned long long)in_slab * per_row + 255) / 256), ((unsigned)rows + slab - 1) / slab);
}

}  // namespace
}  // namespace nerf

using namespace nerf;

extern "C" {

size_t nerf_w4_row_bytes(int cols) { return cols > 0 ? ((size_t)cols + 31) / 32 * 16 : 0; }

int nerf_quantize_w4(const float* d_src, long ld_src, int rows, int cols, int group, unsigned char* d_codes,
                     unsigned short* d_scales) {
    if (!d_src || !d_codes || !d_scales || rows <= 0 || cols <= 0 || ld_src < cols || !group_ok(group) ||
        ((uintptr_t)d_src & 3) || ((uintptr_t)d_codes & 15) || ((uintptr_t)d_scales & 1))
        return NERF_ERR_ARG;
    const int groups = ceil_div(cols, group);
    const unsigned per_row = (unsigned)groups * (unsigned)(group / 8);
    const long row_bytes = (long)nerf_w4_row_bytes(cols);
    ProfScope prof(K_QUANTIZE_W4, (double)rows * cols * 4.5);
#define QUANTIZE(G)                                                                                                        \
    hipLaunchKernelGGL((quantize_w4_kernel<G>), piece_grid(rows, per_row), dim3(256), 0, stream(), d_src, ld_src, rows, cols, \
                       per_row, d_codes, row_bytes, d_scales, groups)
    if (group == 32) QUANTIZE(32);
    else if (group == 64) QUANTIZE(64);
    else QUANTIZE(128);
#undef QUANTIZE
    return hipGetLastError() == hipSuccess ? NERF_OK : NERF_ERR_HIP;
}

int nerf_dequantize_w4(const unsigned char* d_codes, const unsigned short* d_scales, int rows, int cols, int group,
                       float* d_dst, long ld_dst) {
    if (!d_dst || !d_codes || !d_scales || rows <= 0 || cols <= 0 || ld_dst < cols || !group_ok(group) ||
        ((uintptr_t)d_dst & 3) || ((uintptr_t)d_codes & 15) || ((uintptr_t)d_scales & 1))
        return NERF_ERR_ARG;
    const unsigned per_row = (unsigned)ceil_div(cols, 8);
    ProfScope prof(K_QUANTIZE_W4, (double)rows * cols * 4.5);
    hipLaunchKernelGGL(dequantize_w4_kernel, piece_grid(rows, per_row), dim3(256), 0, stream(), d_codes,
                       (long)nerf_w4_row_bytes(cols), d_scales, ceil_div(cols, group), group, rows, cols, per_row, d_dst, ld_dst);
    return hipGetLastError() == hipSuccess ? NERF_OK : NERF_ERR_HIP;
}

size_t nerf_gemm_w4_workspace(int M, int N, int K) {
    (void)M; (void)N; (void)K;
    return 0;
}

int nerf_gemm_w4(const void* d_X, int x_type, long ldx, const unsigned char* d_codes, const unsigned short* d_scales,
                 int group, void* d_Y, int y_type, long ldy, int M, int N, int K, int epilogue, void* d_workspace,
                 size_t workspace_bytes) {
    if (!d_X || !d_codes || !d_scales || !d_Y || M <= 0 || N <= 0 || K <= 0 || ldx < K || ldy < N || !group_ok(group) ||
        !type_ok(x_type) || !type_ok(y_type) || (epilogue != 0 && epilogue != 1) || ((uintptr_t)d_codes & 15) ||
        ((uintptr_t)d_scales & 1) || ((uintptr_t)d_X & (x_type == NERF_TYPE_BF16 ? 1 : 3)) ||
        ((uintptr_t)d_Y & (y_type == NERF_TYPE_BF16 ? 1 : 3)) || ((uintptr_t)d_workspace & 15))
        return NERF_ERR_ARG;
    const size_t need = nerf_gemm_w4_workspace(M, N, K);
    if (workspace_bytes < need || (need && !d_workspace)) return NERF_ERR_ARG;
    W4Args a = {};
    a.X = d_X; a.codes = d_codes; a.scales = d_scales; a.Y = d_Y;
    a.ldx = ldx; a.ldy = ldy; a.row_bytes = (long)nerf_w4_row_bytes(K);
    a.M = M; a.N = N; a.K = K; a.group = group; a.groups = ceil_div(K, group);
    a.x_bf16 = x_type == NERF_TYPE_BF16; a.y_bf16 = y_type == NERF_TYPE_BF16; a.epilogue = epilogue;
    ProfScope prof(K_GEMM_W4, 2.0 * M * N * K);
    if (M <= 16) {
        if (N >= 8192) launch_gemm<1, 4>(a);
        else launch_gemm<1, 1>(a);
    } else if (M <= 32) {
        launch_gemm<2, 2>(a);
    } else {
        launch_gemm<4, 2>(a);
    }
    return hipGetLastError() == hipSuccess ? NERF_OK : NERF_ERR_HIP;
}

}  // extern "C"
