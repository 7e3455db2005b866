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

__device__ __forceinline__ float load_x(const W4Args& a, long at) {
    return a.x_bf16 ? bf16_to_f32(((const unsigned short*)a.X)[at]) : ((const float*)a.X)[at];
}
__device__ __forceinline__ void store_y(const W4Args& a, long at, float y) {
    // sigmoid through the hardware exp2 and reciprocal, as in the other products' epilogues
    if (a.epilogue == 1) y = y * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(y * -1.44269504088896340736f));
    if (a.y_bf16) ((unsigned short*)a.Y)[at] = f32_to_bf16(y);
    else ((float*)a.Y)[at] = y;
}

// One wavefront per (row of W, row of X): a lane takes every 64th unit.
__global__ __launch_bounds__(256) void gemv_w4_kernel(const W4Args a) {
    const int lane = threadIdx.x & 63;
    const long n = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (n >= a.N) return;
    const int m = blockIdx.y;
    const int units = (a.K + 31) / 32;
    float acc = 0.0f;
    for (int u = lane; u < units; u += 64) {
        const u32x4 c = *reinterpret_cast<const u32x4*>(a.codes + n * a.row_bytes + (long)u * 16);
        const float scale = bf16_to_f32(a.scales[n * a.groups + u * 32 / a.group]);
        float part = 0.0f;
#pragma unroll
        for (int q = 0; q < 4; q++) {
            float v[8];
            values8(c[q], v);
            for (int k = 0; k < 8; k++) {
                const int col = u * 32 + q * 8 + k;
                if (col < a.K) part = __builtin_fmaf(load_x(a, (long)m * a.ldx + col), v[k], part);
            }
        }
        acc = __builtin_fmaf(part, scale, acc);
    }
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) acc += __shfl_xor(acc, d, 64);
    if (lane == 0) store_y(a, (long)m * a.ldy + n, acc);
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
    if (M > 65535) return NERF_ERR_ARG;
    ProfScope prof(K_GEMM_W4, 2.0 * M * N * K);
    hipLaunchKernelGGL(gemv_w4_kernel, dim3((unsigned)ceil_div(N, 4), (unsigned)M), dim3(256), 0, stream(), a);
    return hipGetLastError() == hipSuccess ? NERF_OK : NERF_ERR_HIP;
}

}  // extern "C"
