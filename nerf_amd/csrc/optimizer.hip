// optimizer.hip -- one AdamW step over many tensors, its 8-bit states, and the global gradient norm.
//
// No counterpart in the reference, which updates each matrix of its two MLPs on its own
// (update_weights_mlp, train.c:219-220).  A plan (NerfAdamw) holds a table of chunks -- a chunk is a run of up to
// 4096 elements of one tensor, the work of four workgroups -- so a step over any number of tensors is ONE launch.
// A chunk's record holds its addresses themselves: one dependent read in front of the data.
//
// Everything here waits for memory.  A workgroup takes 1024 elements, four to a thread: all it reads is asked for
// before the first use, and there are always others to take over while it waits (134 million elements, bf16 gradients
// and copy, 28 bytes an element: 593 us = 6.3 TB/s, 580 to 645 over cards; on one card 623 us, and with 2048, 4096 and 8192
// elements to a workgroup 658, 671 and 684; a loop over the pieces does not overlap them as well as the scheduler does).
#include "common.hpp"
#include "../../include/nerf_amd.h"

#include <math.h>

#include <algorithm>
#include <new>
#include <vector>

#pragma clang fp contract(off)

namespace nerf {
namespace {

// Elements that share an exponent in the 8-bit states: one wavefront's four consecutive elements per lane.
constexpr unsigned BLOCK = 256;
constexpr unsigned NORM_BLOCKS = 512, NORM_WAVES = 16;  // workgroups, and partial sums, of the norm; wavefronts of one
constexpr unsigned CHUNK = 4096, PIECE = 1024, PIECES = CHUNK / PIECE;  // elements of a record, of a workgroup

// pieces of elements at any element-aligned address
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned short u16x4u __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned short u16x8u __attribute__((ext_vector_type(8), aligned(2)));
typedef unsigned u32u __attribute__((aligned(1)));
// Pointers out of the plan's table are to device memory: saying so keeps their loads off the generic path
#define GLOBAL __attribute__((address_space(1)))
typedef GLOBAL const f32x4u* LoadF32x4;
typedef GLOBAL f32x4u* StoreF32x4;
typedef GLOBAL const u16x4u* LoadU16x4;
typedef GLOBAL u16x4u* StoreU16x4;
typedef GLOBAL const u16x8u* LoadU16x8;
typedef GLOBAL const u32u* LoadU32;
typedef GLOBAL u32u* StoreU32;
typedef GLOBAL const float* LoadF32;
typedef GLOBAL float* StoreF32;
typedef GLOBAL const unsigned short* LoadU16;
typedef GLOBAL unsigned short* StoreU16;
typedef GLOBAL const unsigned char* LoadU8;
typedef GLOBAL unsigned char* StoreU8;

struct Chunk {
    float* w;  // the chunk's first elements
    const void* g;
    void* m;
    void* v;
    unsigned char* m_exp;
    unsigned char* v_exp;
    unsigned short* w_bf16;
    size_t first;    // elements of the whole list before it
    unsigned count;  // elements, at most the plan's chunk
    unsigned tensor, block;  // place in the list; blocks of the tensor before it
    float lr_scale, weight_decay;
    int g_bf16;
};

struct StepArgs {
    const Chunk* chunks;
    float lr, root_c2t, c1t;      // learning rate, sqrt(1 - beta2^t), 1 - beta1^t
    float grad_div, grad_mul;     // grad_mul: 1 / grad_div where that is exact, else 0
    float beta1, beta2, eps;
    const float* norm;
    float max_norm;
    unsigned key;
};

__device__ __forceinline__ float bf16_to_f32(unsigned short b) { return __builtin_bit_cast(float, (unsigned)b << 16); }
__device__ __forceinline__ unsigned short f32_to_bf16(float x) {
    return __builtin_bit_cast(unsigned short, (__bf16)x);  // to nearest, ties to even
}

// a 32-bit mixing function, xor-shifts and two odd multipliers: the published integer hash lowbias32
__host__ __device__ __forceinline__ unsigned mix32(unsigned x) {
    x ^= x >> 16;
    x *= 0x7FEB352Du;
    x ^= x >> 15;
    x *= 0x846CA68Bu;
    return x ^ (x >> 16);
}

// Up to four consecutive elements; `left` of them exist.  STREAM: past the caches, for data that is larger than they are.
template <bool STREAM>
__device__ __forceinline__ f32x4u load4(const float* p, unsigned left) {
    if (left >= 4) return STREAM ? __builtin_nontemporal_load((LoadF32x4)p) : *(LoadF32x4)p;
    f32x4u x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (unsigned k = 0; k < 3; k++)
        if (k < left) x[k] = ((LoadF32)p)[k];
    return x;
}
template <bool STREAM>
__device__ __forceinline__ f32x4u load4(const unsigned short* p, unsigned left) {
    u16x4u b = {0, 0, 0, 0};
    if (left >= 4) b = STREAM ? __builtin_nontemporal_load((LoadU16x4)p) : *(LoadU16x4)p;
    else
#pragma unroll
        for (unsigned k = 0; k < 3; k++)
            if (k < left) b[k] = ((LoadU16)p)[k];
    f32x4u x;
#pragma unroll
    for (int k = 0; k < 4; k++) x[k] = bf16_to_f32(b[k]);
    return x;
}
template <bool STREAM>
__device__ __forceinline__ unsigned load4(const unsigned char* p, unsigned left) {
    if (left >= 4) return STREAM ? __builtin_nontemporal_load((LoadU32)p) : *(LoadU32)p;
    unsigned x = 0;
#pragma unroll
    for (unsigned k = 0; k < 3; k++)
        if (k < left) x |= (unsigned)((LoadU8)p)[k] << (8 * k);
    return x;
}
template <bool STREAM>
__device__ __forceinline__ void store4(float* p, f32x4u x, unsigned left) {
    if (left < 4) {
#pragma unroll
        for (unsigned k = 0; k < 3; k++)
            if (k < left) ((StoreF32)p)[k] = x[k];
    } else if (STREAM) {
        __builtin_nontemporal_store(x, (StoreF32x4)p);
    } else {
        *(StoreF32x4)p = x;
    }
}
template <bool STREAM>
__device__ __forceinline__ void store4_bf16(unsigned short* p, f32x4u x, unsigned left) {
    u16x4u b;
#pragma unroll
    for (int k = 0; k < 4; k++) b[k] = f32_to_bf16(x[k]);
    if (left < 4) {
#pragma unroll
        for (unsigned k = 0; k < 3; k++)
            if (k < left) ((StoreU16)p)[k] = b[k];
    } else if (STREAM) {
        __builtin_nontemporal_store(b, (StoreU16x4)p);
    } else {
        *(StoreU16x4)p = b;
    }
}
template <bool STREAM>
__device__ __forceinline__ void store4(unsigned char* p, unsigned x, unsigned left) {
    if (left < 4) {
#pragma unroll
        for (unsigned k = 0; k < 3; k++)
            if (k < left) ((StoreU8)p)[k] = (unsigned char)(x >> (8 * k));
    } else if (STREAM) {
        __builtin_nontemporal_store(x, (StoreU32)p);
    } else {
        *(StoreU32)p = x;
    }
}

// What an element's gradient is multiplied by beyond the divisor; false: the step is left out (the norm is not
// finite, so some gradient is not)
__device__ __forceinline__ bool clip_factor(const StepArgs& a, float& factor) {
    factor = 1.0f;
    if (!a.norm) return true;
    const float norm = *a.norm;
    if (!(norm < INFINITY)) return false;
    if (norm > a.max_norm) factor = __fdiv_rn(a.max_norm, norm);
    return true;
}

// a / b for b a power of two is a * (1 / b) exactly: the usual divisor (points of a batch) saves the division
__device__ __forceinline__ float gradient(const StepArgs& a, float g, float factor) {
    const float x = a.grad_mul != 0.0f ? __fmul_rn(g, a.grad_mul) : __fdiv_rn(g, a.grad_div);
    return __fmul_rn(x, factor);
}

template <bool STREAM>
__device__ __forceinline__ f32x4u load_g(const Chunk& c, unsigned i, unsigned left) {
    return c.g_bf16 ? load4<STREAM>((const unsigned short*)c.g + i, left) : load4<STREAM>((const float*)c.g + i, left);
}

// The chunk of a workgroup, and the step's factors for its tensor; false: nothing to do
struct Piece {
    Chunk c;
    float factor, alpha, decay;

    __device__ __forceinline__ bool of(const StepArgs& a) {
        c = a.chunks[blockIdx.x / PIECES];
        if (!clip_factor(a, factor) || blockIdx.x % PIECES * PIECE >= c.count) return false;
        const float lr = __fmul_rn(a.lr, c.lr_scale);
        alpha = __fdiv_rn(__fmul_rn(lr, a.root_c2t), a.c1t);
        decay = __fsub_rn(1.0f, __fmul_rn(lr, c.weight_decay));
        return true;
    }
};

// ---- 32-bit states --------------------------------------------------------------------------------------
// The operations of adamw_element (mlp.hip) in the same order: the same bits as nerf_trainer_update.
template <bool STREAM>
__device__ __forceinline__ void adamw32_four(const StepArgs& a, const Piece& p, unsigned i, unsigned left) {
    const Chunk& c = p.c;
    const float c1 = __fsub_rn(1.0f, a.beta1), c2 = __fsub_rn(1.0f, a.beta2);
    f32x4u w = load4<STREAM>(c.w + i, left), m = load4<STREAM>((float*)c.m + i, left), v = load4<STREAM>((float*)c.v + i, left);
    const f32x4u g = load_g<STREAM>(c, i, left);
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const float gi = gradient(a, g[k], p.factor);
        m[k] = __fadd_rn(__fmul_rn(a.beta1, m[k]), __fmul_rn(c1, gi));
        v[k] = __fadd_rn(__fmul_rn(a.beta2, v[k]), __fmul_rn(__fmul_rn(c2, gi), gi));
        const float up = __fdiv_rn(__fmul_rn(p.alpha, m[k]), __fadd_rn(sqrtf(v[k]), a.eps));
        w[k] = __fsub_rn(__fmul_rn(w[k], p.decay), up);
    }
    store4<STREAM>((float*)c.m + i, m, left);
    store4<STREAM>((float*)c.v + i, v, left);
    store4<STREAM>(c.w + i, w, left);
    if (c.w_bf16) store4_bf16<STREAM>(c.w_bf16 + i, w, left);
}

template <bool STREAM>
__global__ __launch_bounds__(256) void adamw32_kernel(const StepArgs a) {
    Piece p;
    if (!p.of(a)) return;
    const unsigned begin = blockIdx.x % PIECES * PIECE, i = begin + threadIdx.x * 4;
    if (begin + PIECE <= p.c.count) adamw32_four<STREAM>(a, p, i, 4);
    else if (i < p.c.count) adamw32_four<STREAM>(a, p, i, min(4u, p.c.count - i));
}

// ---- 8-bit states ---------------------------------------------------------------------------------------
// A block of 256 elements shares one exponent byte E (a biased fp32 exponent, 16..254).  A code is a small float
// with a 4-bit exponent field and gradual underflow, its top binade at 2^(E-127):
//   m         sign, 4 exponent bits, 3 mantissa bits
//   sqrt(v)   4 exponent bits, 4 mantissa bits (the root halves the range that v needs, and what the update
//             divides by keeps 5 significant bits)
// An fp32 number whose exponent field is 0..15 holds such a code in its upper bits, so a value becomes a code by
// scaling it with 2^(15-E) and rounding off the lower mantissa bits, carry and underflow included.
// A root's code is zero only where v is, or was not finite; v is zero only where every gradient so far was, or next to it (or
// beta2 forgets it at once).  An m beside such a code counts as zero, whatever its own code: what the update divides it by
// is gone (the step after a gradient of 1e21 would divide 1e20 by eps).  This costs the step of 134 million elements 1.4 %
// (371 and 376 us; a test of four codes at once before the selections costs as much, and half of the read of states).
__device__ __forceinline__ float decode(unsigned code, int low, int exponent) {
    return __builtin_amdgcn_ldexpf(__builtin_bit_cast(float, code << low), exponent - 15);
}
__device__ __forceinline__ float decode_m(unsigned code, unsigned root_code, int exponent) {
    const float x = root_code ? decode(code & 127, 20, exponent) : 0.0f;
    return code & 128 ? -x : x;
}
__device__ __forceinline__ unsigned encode(float x, int low, int exponent, unsigned noise) {
    return (__builtin_bit_cast(unsigned, __builtin_amdgcn_ldexpf(x, 15 - exponent)) + noise) >> low;
}

template <int CTRL>
__device__ __forceinline__ unsigned max_dpp(unsigned x) {
    const unsigned y = (unsigned)__builtin_amdgcn_update_dpp((int)x, (int)x, CTRL, 0xf, 0xf, false);
    return max(x, y);
}
// the largest of a wavefront's 64 values, the same in every lane
__device__ __forceinline__ unsigned wave_max(unsigned x) {
    x = max_dpp<0xB1>(x);   // the neighbour in the pair
    x = max_dpp<0x4E>(x);   // the other pair of the quad
    x = max_dpp<0x141>(x);  // the other quad of eight lanes
    x = max_dpp<0x140>(x);  // the other eight lanes of the row
    x = max_dpp<0x142>(x);  // rows 1 and 3 take in lane 15 and 47
    x = max_dpp<0x143>(x);  // rows 2 and 3 take in lane 31
    return (unsigned)__builtin_amdgcn_readlane((int)x, 63);
}
// The exponent byte whose top binade holds the largest value once it is rounded up
__device__ __forceinline__ int block_exponent(unsigned top, int low) {
    const int e = (int)((top + (1u << low) - 1) >> 23);
    return min(max(e, 16), 254);
}

// A wavefront takes a whole block, four consecutive elements to a lane; every lane stays, those past the end with nothing
// `left`.
template <bool STOCHASTIC, bool STREAM>
__device__ __forceinline__ void adamw8_block(const StepArgs& a, const Piece& p, unsigned i, unsigned left) {
    const Chunk& c = p.c;
    const float c1 = __fsub_rn(1.0f, a.beta1), c2 = __fsub_rn(1.0f, a.beta2);
    const int lane = threadIdx.x & 63;
    const unsigned block = __builtin_amdgcn_readfirstlane(i / BLOCK);
    unsigned char *mc = (unsigned char*)c.m + i, *vc = (unsigned char*)c.v + i;
    f32x4u w = load4<STREAM>(c.w + i, left);
    const f32x4u g = load_g<STREAM>(c, i, left);
    const unsigned m_old = load4<STREAM>(mc, left), v_old = load4<STREAM>(vc, left);
    const int m_e = ((LoadU8)c.m_exp)[block], v_e = ((LoadU8)c.v_exp)[block];
    float m[4], r[4];
    unsigned m_top = 0, r_top = 0;
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const unsigned mb = (m_old >> (8 * k)) & 255, vb = (v_old >> (8 * k)) & 255;
        const float m0 = decode_m(mb, vb, m_e);
        const float r0 = decode(vb, 19, v_e);
        const float gi = gradient(a, g[k], p.factor);
        m[k] = __fadd_rn(__fmul_rn(a.beta1, m0), __fmul_rn(c1, gi));
        r[k] = sqrtf(__fadd_rn(__fmul_rn(a.beta2, __fmul_rn(r0, r0)), __fmul_rn(__fmul_rn(c2, gi), gi)));
        const float up = __fdiv_rn(__fmul_rn(p.alpha, m[k]), __fadd_rn(r[k], a.eps));
        w[k] = __fsub_rn(__fmul_rn(w[k], p.decay), up);
        // a state that is not finite is held as zero and leaves the block's exponent alone
        if (!(fabsf(m[k]) < INFINITY)) m[k] = 0.0f;
        if (!(r[k] < INFINITY)) r[k] = 0.0f;
        m_top = max(m_top, __builtin_bit_cast(unsigned, fabsf(m[k])));
        r_top = max(r_top, __builtin_bit_cast(unsigned, r[k]));
    }
    if (left) store4<STREAM>(c.w + i, w, left);
    if (left && c.w_bf16) store4_bf16<STREAM>(c.w_bf16 + i, w, left);
    const int m_new = block_exponent(wave_max(m_top), 20), v_new = block_exponent(wave_max(r_top), 19);
    const unsigned block_key = mix32(mix32(a.key + c.tensor * 0x9E3779B9u) + (c.block + block) * 0x85EBCA6Bu);
    unsigned m_codes = 0, v_codes = 0;
#pragma unroll
    for (int k = 0; k < 4; k++) {
        unsigned m_noise = 1u << 19, r_noise = 1u << 18;  // half a step: to nearest
        if (STOCHASTIC) {
            const unsigned h = mix32(block_key ^ (unsigned)(lane * 4 + k));
            m_noise = (h & 0xFFFF) << 4;
            r_noise = (h >> 16) << 3;
        }
        unsigned mq = min(encode(fabsf(m[k]), 20, m_new, m_noise), 127u);
        if (m[k] < 0.0f && mq) mq |= 128;
        unsigned rq = min(encode(r[k], 19, v_new, r_noise), 255u);
        // a second moment that is not zero does not become zero: the update divides by its root
        if (rq == 0 && r[k] > 0.0f) rq = 1;
        m_codes |= mq << (8 * k);
        v_codes |= rq << (8 * k);
    }
    if (left) {
        store4<STREAM>(mc, m_codes, left);
        store4<STREAM>(vc, v_codes, left);
    }
    if (lane == 0) {
        ((StoreU8)c.m_exp)[block] = (unsigned char)m_new;
        ((StoreU8)c.v_exp)[block] = (unsigned char)v_new;
    }
}

template <bool STOCHASTIC, bool STREAM>
__global__ __launch_bounds__(256) void adamw8_kernel(const StepArgs a) {
    Piece p;
    if (!p.of(a)) return;
    const unsigned begin = blockIdx.x % PIECES * PIECE, i = begin + threadIdx.x * 4;
    if (begin + PIECE <= p.c.count) adamw8_block<STOCHASTIC, STREAM>(a, p, i, 4);
    else if (i / BLOCK * BLOCK < p.c.count) adamw8_block<STOCHASTIC, STREAM>(a, p, i, i < p.c.count ? min(4u, p.c.count - i) : 0);
}

// the values that 8-bit states stand for, as bf16 (every one is exact: at most 5 significant bits)
template <bool STREAM>
__global__ __launch_bounds__(256) void read_states_kernel(const Chunk* chunks, unsigned short* m_out, unsigned short* r_out) {
    const Chunk c = chunks[blockIdx.x];
    auto four = [&](unsigned i, unsigned left) {
        const unsigned mc = load4<STREAM>((const unsigned char*)c.m + i, left), vc = load4<STREAM>((const unsigned char*)c.v + i, left);
        const int m_e = ((LoadU8)c.m_exp)[i / BLOCK], v_e = ((LoadU8)c.v_exp)[i / BLOCK];
        f32x4u m, r;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const unsigned mb = (mc >> (8 * k)) & 255, vb = (vc >> (8 * k)) & 255;
            m[k] = decode_m(mb, vb, m_e);
            r[k] = decode(vb, 19, v_e);
        }
        if (m_out) store4_bf16<STREAM>(m_out + c.first + i, m, left);
        if (r_out) store4_bf16<STREAM>(r_out + c.first + i, r, left);
    };
    const unsigned whole = c.count & ~1023u;
    unsigned i = threadIdx.x * 4;
    for (; i < whole; i += 1024) four(i, 4);
    if (i < c.count) four(i, min(4u, c.count - i));
}

// ---- global norm ----------------------------------------------------------------------------------------
// Squares are added in 64 bits, so neither the range of the squares nor the length of the sum costs anything
// (the kernel waits for memory).  Each wavefront walks the pieces at a fixed stride, each workgroup leaves one partial sum;
// the workgroup that draws the last ticket adds the partial sums in their order: the same bits on every call.
//
// A partial sum is all that passes between workgroups, and it says itself that it is there: its place holds NO_SUM until then,
// and again as soon as it is taken.  So nothing hangs on the order in which operations on different places are seen, only
// on one place's own: no fence is needed, which would write the caches back.  The last one's loads nearly always come
// after all sums; where one does not, it asks again, and the sum it asks for is on its way: its workgroup sent it before it drew
// its ticket.  (Two calls at once on one plan, which are not allowed, could take each other's sums, so the asking ends.)
constexpr unsigned long long NO_SUM = ~0ull;  // a NaN that no sum of squares is: its lower bits come from doubles made of floats
constexpr int MOST_TURNS = 1 << 16;
__device__ __forceinline__ double block_sum(double x, double* shared) {
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) x += __shfl_xor(x, d, 64);
    if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = x;
    __syncthreads();
    x = 0.0;
#pragma unroll
    for (int w = 0; w < NORM_WAVES; w++) x += shared[w];
    __syncthreads();
    return x;
}

// a wavefront's part of the sum of the squares of a chunk's elements from `begin` on, PIECE of them or to the end
__device__ __forceinline__ double squares(const Chunk& c, unsigned begin) {
    double sum[4] = {0.0, 0.0, 0.0, 0.0};
    const unsigned lane = threadIdx.x & 63;
    auto add = [&](f32x4u g) {
#pragma unroll
        for (int k = 0; k < 4; k++) sum[k] += (double)g[k] * (double)g[k];
    };
    if (begin + PIECE > c.count) {
        for (unsigned i = begin + lane * 4; i < c.count; i += 256) add(load_g<false>(c, i, min(4u, c.count - i)));
    } else if (c.g_bf16) {  // 16 bytes to a lane
        u16x8u g[2];
#pragma unroll
        for (int u = 0; u < 2; u++) g[u] = *(LoadU16x8)((const unsigned short*)c.g + begin + lane * 8 + u * 512);
#pragma unroll
        for (int u = 0; u < 2; u++) {
            add(f32x4u{bf16_to_f32(g[u][0]), bf16_to_f32(g[u][1]), bf16_to_f32(g[u][2]), bf16_to_f32(g[u][3])});
            add(f32x4u{bf16_to_f32(g[u][4]), bf16_to_f32(g[u][5]), bf16_to_f32(g[u][6]), bf16_to_f32(g[u][7])});
        }
    } else {
        f32x4u g[4];
#pragma unroll
        for (int u = 0; u < 4; u++) g[u] = load4<false>((const float*)c.g + begin + lane * 4 + u * 256, 4);
#pragma unroll
        for (int u = 0; u < 4; u++) add(g[u]);
    }
    return (sum[0] + sum[1]) + (sum[2] + sum[3]);
}

__global__ __launch_bounds__(64 * NORM_WAVES) void grad_norm_kernel(const Chunk* chunks, unsigned count, unsigned long long* partial, unsigned* ticket,
                                                        float grad_div, float* norm) {
    __shared__ double shared[NORM_WAVES];
    __shared__ bool last;
    double sum = 0.0;
    for (unsigned b = blockIdx.x * NORM_WAVES + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); b < count; b += gridDim.x * NORM_WAVES) {
        const Chunk c = chunks[b / PIECES];
        if (b % PIECES * PIECE < c.count) sum += squares(c, b % PIECES * PIECE);
    }
    sum = block_sum(sum, shared);
    if (threadIdx.x == 0) {
        __hip_atomic_store(partial + blockIdx.x, __builtin_bit_cast(unsigned long long, sum), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        last = atomicInc(ticket, gridDim.x - 1) == gridDim.x - 1;  // the last one takes it back to 0 for the next call
    }
    __syncthreads();
    if (!last) return;
    sum = 0.0;
    for (unsigned b = threadIdx.x; b < gridDim.x; b += 64 * NORM_WAVES) {
        unsigned long long bits = NO_SUM;
        for (int turn = 0; bits == NO_SUM && turn < MOST_TURNS; turn++) bits = __hip_atomic_load(partial + b, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __hip_atomic_store(partial + b, NO_SUM, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        sum += __builtin_bit_cast(double, bits);
    }
    sum = block_sum(sum, shared);
    if (threadIdx.x == 0) *norm = (float)(sqrt(sum) / (double)grad_div);
}

bool finite_not_negative(float x) { return x >= 0.0f && x < INFINITY; }

// Whether a buffer may be handed to a kernel on a device: inside one allocation, and not pageable host memory or
// another GPU's.  Tensors mostly come out of a few allocations: the last one found is kept.
class DevicePointers {
public:
    explicit DevicePointers(int device) : device_(device) {}
    bool holds(const void* p, size_t bytes) {
        const uintptr_t at = (uintptr_t)p;
        if (at >= begin_ && at - begin_ < size_) return bytes <= size_ - (at - begin_);
        hipPointerAttribute_t info;
        if (hipPointerGetAttributes(&info, p) != hipSuccess) {
            (void)hipGetLastError();
            return false;
        }
        if (info.type == hipMemoryTypeDevice ? info.device != device_ : info.type != hipMemoryTypeHost && info.type != hipMemoryTypeManaged)
            return false;
        hipDeviceptr_t base = nullptr;
        size_t size = 0;
        if (hipMemGetAddressRange(&base, &size, (hipDeviceptr_t)p) != hipSuccess) {
            (void)hipGetLastError();
            return true;  // known to the runtime, but not as one allocation
        }
        begin_ = (uintptr_t)base;
        size_ = size;
        return at >= begin_ && at - begin_ < size_ && bytes <= size_ - (at - begin_);
    }

private:
    int device_;
    uintptr_t begin_ = 1;
    size_t size_ = 0;
};

struct Range {
    uintptr_t begin, end;
    bool written;
};

// No buffer that a step writes may overlap another one of the list
bool disjoint(std::vector<Range>& r) {
    std::sort(r.begin(), r.end(), [](const Range& a, const Range& b) { return a.begin < b.begin; });
    uintptr_t read_to = 0, written_to = 0;
    for (const Range& x : r) {
        if (x.begin < written_to || (x.written && x.begin < read_to)) return false;
        uintptr_t& to = x.written ? written_to : read_to;
        to = std::max(to, x.end);
    }
    return true;
}

int check_tensors(const NerfAdamwTensor* tensors, int count, int state_bits) {
    if (!tensors || count < 1 || (state_bits != 0 && state_bits != 8 && state_bits != 32)) return NERF_ERR_ARG;
    std::vector<Range> ranges;
    size_t chunks = 0;
    for (int k = 0; k < count; k++) {
        const NerfAdamwTensor& t = tensors[k];
        if (t.n == 0) continue;
        if (t.n > NERF_ADAMW_MAX_ELEMENTS) return NERF_ERR_ARG;
        chunks += t.n / CHUNK + (t.n % CHUNK != 0);
        if (chunks > NERF_ADAMW_MAX_ELEMENTS / CHUNK || (t.grad_type != NERF_TYPE_F32 && t.grad_type != NERF_TYPE_BF16)) return NERF_ERR_ARG;
        const size_t g_item = t.grad_type == NERF_TYPE_BF16 ? 2 : 4;
        auto add = [&](const void* p, size_t items, size_t item, bool written) {
            const uintptr_t at = (uintptr_t)p;
            if (!p || at % item || at + items * item < at) return false;
            ranges.push_back(Range{at, at + items * item, written});
            return true;
        };
        if (!add(t.g, t.n, g_item, false)) return NERF_ERR_ARG;
        if (state_bits == 0) continue;
        if (!finite_not_negative(t.lr_scale) || !finite_not_negative(t.weight_decay)) return NERF_ERR_ARG;
        const size_t item = state_bits == 8 ? 1 : 4, blocks = nerf_adamw_state_blocks(t.n);
        if (!add(t.w, t.n, 4, true) || !add(t.m, t.n, item, true) || !add(t.v, t.n, item, true)) return NERF_ERR_ARG;
        if (state_bits == 8 && (!add(t.m_exp, blocks, 1, true) || !add(t.v_exp, blocks, 1, true))) return NERF_ERR_ARG;
        if (t.w_bf16 && !add(t.w_bf16, t.n, 2, true)) return NERF_ERR_ARG;
    }
    return disjoint(ranges) ? NERF_OK : NERF_ERR_ARG;
}

}  // namespace
}  // namespace nerf

using namespace nerf;

// Bytes of a step beyond which it streams past the caches (256 MB on the memory side).  Three lists in turn, each with
// and without: 4 million elements in 32 bits (112 MB) 19.8 and 18.1 us, 8 million (224 MB) 37.7 and 43.3 us, 134 million with
// bf16 gradients and copy (3.8 GB) 623 and 739 us (one card).
constexpr double STREAM_BYTES = 160e6;

struct NerfAdamw {
    int device, state_bits;
    float beta1, beta2, eps;
    unsigned chunks;
    double bytes, grad_bytes;  // of one step, of one norm
    void* memory;              // one allocation: partial sums, ticket, chunks
    unsigned long long* d_partial;
    unsigned* d_ticket;
    Chunk* d_chunks;
};

extern "C" {

size_t nerf_adamw_state_blocks(size_t n) { return n / BLOCK + (n % BLOCK != 0); }

// NERF_OK, or NERF_ERR_ARG while the library's stream is being captured into a graph, or is the default one and another
// stream that waits for it is captured: the runtime answers that with an error, which is not left for a later call to report
static int not_capturing() {
    hipStreamCaptureStatus capturing = hipStreamCaptureStatusNone;
    const hipError_t rc = hipStreamIsCapturing(stream(), &capturing);
    if (rc != hipSuccess) {
        (void)hipGetLastError();
        return rc == hipErrorStreamCaptureImplicit ? NERF_ERR_ARG : NERF_ERR_HIP;
    }
    return capturing == hipStreamCaptureStatusNone ? NERF_OK : NERF_ERR_ARG;
}

static int build_plan(const NerfAdamwTensor* tensors, int count, int state_bits, NerfAdamw* plan) {
    static_assert(NERF_ADAMW_MAX_ELEMENTS % CHUNK == 0 && NERF_ADAMW_MAX_ELEMENTS / PIECE * 256 < 1ull << 32, "a launch has fewer than 2^32 threads");
    size_t pieces = 0;
    for (int k = 0; k < count; k++) pieces += tensors[k].n / CHUNK + (tensors[k].n % CHUNK != 0);
    constexpr size_t HEAD = NORM_BLOCKS * sizeof(unsigned long long) + 256;
    std::vector<char> image(HEAD + pieces * sizeof(Chunk));
    std::fill_n(reinterpret_cast<unsigned long long*>(image.data()), NORM_BLOCKS, NO_SUM);
    Chunk* table = reinterpret_cast<Chunk*>(image.data() + HEAD);
    DevicePointers known(plan->device);
    size_t first = 0;
    for (int k = 0; k < count; k++) {
        const NerfAdamwTensor& s = tensors[k];
        if (s.n == 0) continue;
        const bool bf = s.grad_type == NERF_TYPE_BF16;
        const size_t state = state_bits == 8 ? 1 : 4, blocks = nerf_adamw_state_blocks(s.n);
        bool ok = known.holds(s.g, s.n * (bf ? 2 : 4));
        if (state_bits) ok = ok && known.holds(s.w, s.n * 4) && known.holds(s.m, s.n * state) && known.holds(s.v, s.n * state);
        if (state_bits == 8) ok = ok && known.holds(s.m_exp, blocks) && known.holds(s.v_exp, blocks);
        if (state_bits && s.w_bf16) ok = ok && known.holds(s.w_bf16, s.n * 2);
        if (!ok) return NERF_ERR_ARG;
        const double g_item = bf ? 2.0 : 4.0;
        plan->grad_bytes += (double)s.n * g_item;
        plan->bytes += (double)s.n * (8.0 + g_item + 4.0 * (double)state + (s.w_bf16 ? 2.0 : 0.0));
        for (size_t at = 0; at < s.n; at += CHUNK) {
            Chunk c = {};
            c.g = (const char*)s.g + at * (bf ? 2 : 4);
            c.g_bf16 = bf;
            c.count = (unsigned)std::min((size_t)CHUNK, s.n - at);
            if (state_bits) {
                c.w = s.w + at;
                c.m = (char*)s.m + at * state;
                c.v = (char*)s.v + at * state;
                c.w_bf16 = s.w_bf16 ? s.w_bf16 + at : nullptr;
                c.lr_scale = s.lr_scale;
                c.weight_decay = s.weight_decay;
            }
            if (state_bits == 8) {
                c.m_exp = s.m_exp + at / BLOCK;
                c.v_exp = s.v_exp + at / BLOCK;
            }
            c.first = first + at;
            c.tensor = (unsigned)k;
            c.block = (unsigned)(at / BLOCK);
            *table++ = c;
        }
        first += s.n;
    }
    plan->chunks = (unsigned)pieces;
    const int rc = not_capturing();  // the wait below would end the capture
    if (rc != NERF_OK) return rc;
    if (hipMalloc(&plan->memory, image.size()) != hipSuccess) return NERF_ERR_HIP;
    plan->d_partial = (unsigned long long*)plan->memory;
    plan->d_ticket = (unsigned*)((char*)plan->memory + NORM_BLOCKS * sizeof(unsigned long long));
    plan->d_chunks = (Chunk*)((char*)plan->memory + HEAD);
    if (hipMemcpyAsync(plan->memory, image.data(), image.size(), hipMemcpyHostToDevice, stream()) != hipSuccess ||
        hipStreamSynchronize(stream()) != hipSuccess)
        return NERF_ERR_HIP;
    return NERF_OK;
}

int nerf_adamw_create(const NerfAdamwTensor* tensors, int count, int state_bits, float beta1, float beta2, float eps,
                      NerfAdamw** out) {
    if (!out) return NERF_ERR_ARG;
    *out = nullptr;
    if (!(beta1 >= 0.0f && beta1 < 1.0f && beta2 >= 0.0f && beta2 < 1.0f && eps > 0.0f && eps < INFINITY)) return NERF_ERR_ARG;
    NerfAdamw* plan = nullptr;
    int rc = NERF_ERR_HIP;
    try {
        rc = check_tensors(tensors, count, state_bits);
        if (rc != NERF_OK) return rc;
        rc = NERF_ERR_HIP;
        plan = new NerfAdamw();
        plan->state_bits = state_bits;
        plan->beta1 = beta1;
        plan->beta2 = beta2;
        plan->eps = eps;
        if (hipGetDevice(&plan->device) == hipSuccess) rc = build_plan(tensors, count, state_bits, plan);
    } catch (const std::bad_alloc&) {
        rc = NERF_ERR_HIP;
    }
    if (rc != NERF_OK) {
        nerf_adamw_destroy(plan);
        (void)hipGetLastError();
        return rc;
    }
    *out = plan;
    return NERF_OK;
}

void nerf_adamw_destroy(NerfAdamw* plan) {
    if (!plan) return;
    if (plan->memory) (void)hipFree(plan->memory);  // of none, too, it would end another stream's capture
    delete plan;
}

// the plan's buffers belong to the device it was made on
static bool plan_usable(const NerfAdamw* plan) {
    int device = -1;
    return plan && hipGetDevice(&device) == hipSuccess && device == plan->device;
}

int nerf_adamw_step(NerfAdamw* plan, int step, float learning_rate, float grad_div, const float* d_norm, float max_norm,
                    unsigned long long seed) {
    if (!plan || !plan->state_bits || step < 1 || !finite_not_negative(learning_rate) || !(grad_div > 0.0f && grad_div < INFINITY) ||
        (d_norm && (((uintptr_t)d_norm & 3) || !(max_norm > 0.0f && max_norm < INFINITY))) || !plan_usable(plan))
        return NERF_ERR_ARG;
    const int rc = not_capturing();  // a graph would repeat this step number and learning rate for ever
    if (rc != NERF_OK) return rc;
    if (!plan->chunks) return NERF_OK;
    StepArgs a = {};
    a.chunks = plan->d_chunks;
    a.lr = learning_rate;
    a.root_c2t = sqrtf(1.0f - powf(plan->beta2, (float)step));
    a.c1t = 1.0f - powf(plan->beta1, (float)step);
    a.grad_div = grad_div;
    int exponent = 0;
    if (frexpf(grad_div, &exponent) == 0.5f && exponent > -120 && exponent < 120) a.grad_mul = 1.0f / grad_div;
    a.beta1 = plan->beta1;
    a.beta2 = plan->beta2;
    a.eps = plan->eps;
    a.norm = d_norm;
    a.max_norm = max_norm;
    // one 32-bit key per (seed, step): a 64-bit mixing function (splitmix64), its halves folded
    unsigned long long z = seed + (unsigned long long)step * 0x9E3779B97F4A7C15ull;
    z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
    z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
    z ^= z >> 31;
    a.key = (unsigned)(z ^ (z >> 32));
    ProfScope prof(K_ADAMW, plan->bytes);
    const dim3 grid(plan->chunks * PIECES), block(256);
    const bool stream_past = plan->bytes > STREAM_BYTES;
#define STEP(KERNEL) hipLaunchKernelGGL(KERNEL, grid, block, 0, stream(), a)
    if (plan->state_bits == 32) {
        if (stream_past) STEP(adamw32_kernel<true>);
        else STEP(adamw32_kernel<false>);
    } else if (seed) {
        if (stream_past) STEP((adamw8_kernel<true, true>));
        else STEP((adamw8_kernel<true, false>));
    } else {
        if (stream_past) STEP((adamw8_kernel<false, true>));
        else STEP((adamw8_kernel<false, false>));
    }
#undef STEP
    return hipGetLastError() == hipSuccess ? NERF_OK : NERF_ERR_HIP;
}

int nerf_adamw_read_states(NerfAdamw* plan, unsigned short* d_m, unsigned short* d_root_v) {
    if (!plan || plan->state_bits != 8 || (!d_m && !d_root_v) || (((uintptr_t)d_m | (uintptr_t)d_root_v) & 1) || !plan_usable(plan))
        return NERF_ERR_ARG;
    if (!plan->chunks) return NERF_OK;
    if (plan->bytes > STREAM_BYTES)
        hipLaunchKernelGGL(read_states_kernel<true>, dim3(plan->chunks), dim3(256), 0, stream(), plan->d_chunks, d_m, d_root_v);
    else
        hipLaunchKernelGGL(read_states_kernel<false>, dim3(plan->chunks), dim3(256), 0, stream(), plan->d_chunks, d_m, d_root_v);
    return hipGetLastError() == hipSuccess ? NERF_OK : NERF_ERR_HIP;
}

int nerf_grad_norm(NerfAdamw* plan, float grad_div, float* d_norm) {
    if (!plan || !d_norm || ((uintptr_t)d_norm & 3) || !(grad_div > 0.0f && grad_div < INFINITY) || !plan_usable(plan)) return NERF_ERR_ARG;
    // A piece to a wavefront up to one workgroup per CU, two workgroups for long lists: every workgroup adds 10 ns for its
    // ticket, every further round of pieces the time of a read.  134 million bf16 elements take 94.9, 55.5, 46.9 and 49.7 us
    // with at most 128, 256, 512 and 1024 workgroups (5.7 TB/s), 16 million in fp32 13.2, 13.8, 15.4 and 19.3 us, 603 136
    // (37 workgroups) 4.9 us; workgroups of four wavefronts took 60 and 16.7 us at their best.  (Then a workgroup still waited for
    // its sum to arrive before it drew its ticket; without that 46.8, 13.4 and 4.5 us.)
    const unsigned pieces = plan->chunks * PIECES, most = pieces < 65536 ? 256 : NORM_BLOCKS;
    const unsigned blocks = std::max(1u, std::min((pieces + NORM_WAVES - 1) / NORM_WAVES, most));
    ProfScope prof(K_GRAD_NORM, plan->grad_bytes);
    hipLaunchKernelGGL(grad_norm_kernel, dim3(blocks), dim3(64 * NORM_WAVES), 0, stream(), plan->d_chunks, plan->chunks * PIECES, plan->d_partial,
                       plan->d_ticket, grad_div, d_norm);
    return hipGetLastError() == hipSuccess ? NERF_OK : NERF_ERR_HIP;
}

}  // extern "C"
