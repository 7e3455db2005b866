// optimizer.hip -- one AdamW step over many tensors, its 8-bit states, and the global gradient norm.
//
// No counterpart in the reference, which updates each matrix of its two MLPs on its own
// (update_weights_mlp, train.c:219-220).  A plan (NerfAdamw) holds a table of the tensors and a table of
// chunks -- a chunk is a run of elements of one tensor, the work of one workgroup -- so a step over any
// number of tensors is ONE launch.
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
constexpr unsigned NORM_BLOCKS = 1024;  // workgroups, and partial sums, of the norm

// pieces of four elements at any element-aligned address
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned short u16x4u __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned u32u __attribute__((aligned(1)));

struct Tensor {
    float* w;
    const void* g;
    void* m;
    void* v;
    unsigned char* m_exp;
    unsigned char* v_exp;
    unsigned short* w_bf16;
    size_t n;
    size_t first;  // elements of the tensors before this one
    float lr_scale, weight_decay;
    int g_bf16;
    unsigned index;
};
struct Chunk {
    unsigned tensor, number;  // elements [number * chunk, (number + 1) * chunk) of the tensor
};

struct StepArgs {
    const Tensor* tensors;
    const Chunk* chunks;
    unsigned chunk;  // elements, a multiple of 1024
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

// a 32-bit mixing function: xor-shifts and two odd multipliers
__host__ __device__ __forceinline__ unsigned mix32(unsigned x) {
    x ^= x >> 16;
    x *= 0x7FEB352Du;
    x ^= x >> 15;
    x *= 0x846CA68Bu;
    return x ^ (x >> 16);
}

// up to four consecutive elements; `left` of them exist
__device__ __forceinline__ f32x4u load4(const float* p, unsigned left) {
    if (left >= 4) return *reinterpret_cast<const f32x4u*>(p);
    f32x4u x = {0.f, 0.f, 0.f, 0.f};
    for (unsigned k = 0; k < left; k++) x[k] = p[k];
    return x;
}
__device__ __forceinline__ f32x4u load4(const unsigned short* p, unsigned left) {
    u16x4u b = {0, 0, 0, 0};
    if (left >= 4) b = *reinterpret_cast<const u16x4u*>(p);
    else
        for (unsigned k = 0; k < left; k++) b[k] = p[k];
    f32x4u x;
    for (int k = 0; k < 4; k++) x[k] = bf16_to_f32(b[k]);
    return x;
}
__device__ __forceinline__ unsigned load4(const unsigned char* p, unsigned left) {
    if (left >= 4) return *reinterpret_cast<const u32u*>(p);
    unsigned x = 0;
    for (unsigned k = 0; k < left; k++) x |= (unsigned)p[k] << (8 * k);
    return x;
}
__device__ __forceinline__ void store4(float* p, f32x4u x, unsigned left) {
    if (left >= 4) *reinterpret_cast<f32x4u*>(p) = x;
    else
        for (unsigned k = 0; k < left; k++) p[k] = x[k];
}
__device__ __forceinline__ void store4_bf16(unsigned short* p, f32x4u x, unsigned left) {
    u16x4u b;
    for (int k = 0; k < 4; k++) b[k] = f32_to_bf16(x[k]);
    if (left >= 4) *reinterpret_cast<u16x4u*>(p) = b;
    else
        for (unsigned k = 0; k < left; k++) p[k] = b[k];
}
__device__ __forceinline__ void store4(unsigned char* p, unsigned x, unsigned left) {
    if (left >= 4) *reinterpret_cast<u32u*>(p) = x;
    else
        for (unsigned k = 0; k < left; k++) p[k] = (unsigned char)(x >> (8 * k));
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

// ---- 32-bit states --------------------------------------------------------------------------------------
// The operations of adamw_element (mlp.hip) in the same order: the same bits as nerf_trainer_update.
__global__ __launch_bounds__(256) void adamw32_kernel(const StepArgs a) {
    const Chunk c = a.chunks[blockIdx.x];
    const Tensor t = a.tensors[c.tensor];
    float factor;
    if (!clip_factor(a, factor)) return;
    const float lr = __fmul_rn(a.lr, t.lr_scale);
    const float alpha = __fdiv_rn(__fmul_rn(lr, a.root_c2t), a.c1t);
    const float decay = __fsub_rn(1.0f, __fmul_rn(lr, t.weight_decay));
    const float c1 = __fsub_rn(1.0f, a.beta1), c2 = __fsub_rn(1.0f, a.beta2);
    const size_t begin = (size_t)c.number * a.chunk;
    const size_t end = min(t.n, begin + a.chunk);
    for (size_t i = begin + threadIdx.x * 4; i < end; i += 1024) {
        const unsigned left = (unsigned)min((size_t)4, end - i);
        f32x4u w = load4(t.w + i, left), m = load4((float*)t.m + i, left), v = load4((float*)t.v + i, left);
        const f32x4u g = t.g_bf16 ? load4((const unsigned short*)t.g + i, left) : load4((const float*)t.g + i, left);
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const float gi = gradient(a, g[k], factor);
            m[k] = __fadd_rn(__fmul_rn(a.beta1, m[k]), __fmul_rn(c1, gi));
            v[k] = __fadd_rn(__fmul_rn(a.beta2, v[k]), __fmul_rn(__fmul_rn(c2, gi), gi));
            const float up = __fdiv_rn(__fmul_rn(alpha, m[k]), __fadd_rn(sqrtf(v[k]), a.eps));
            w[k] = __fsub_rn(__fmul_rn(w[k], decay), up);
        }
        store4((float*)t.m + i, m, left);
        store4((float*)t.v + i, v, left);
        store4(t.w + i, w, left);
        if (t.w_bf16) store4_bf16(t.w_bf16 + i, w, left);
    }
}

// ---- 8-bit states ---------------------------------------------------------------------------------------
// A block of 256 elements shares one exponent byte E (a biased fp32 exponent, 16..254).  A code is a small float
// with a 4-bit exponent field and gradual underflow, its top binade at 2^(E-127):
//   m         sign, 4 exponent bits, 3 mantissa bits
//   sqrt(v)   4 exponent bits, 4 mantissa bits (the root halves the range that v needs, and what the update
//             divides by keeps 5 significant bits)
// An fp32 number whose exponent field is 0..15 holds such a code in its upper bits, so a value becomes a code by
// scaling it with 2^(15-E) and rounding off the lower mantissa bits, carry and underflow included.
__device__ __forceinline__ float decode(unsigned code, int low, int exponent) {
    return __builtin_amdgcn_ldexpf(__builtin_bit_cast(float, code << low), exponent - 15);
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

__global__ __launch_bounds__(256) void adamw8_kernel(const StepArgs a, const int stochastic) {
    const Chunk c = a.chunks[blockIdx.x];
    const Tensor t = a.tensors[c.tensor];
    float factor;
    if (!clip_factor(a, factor)) return;
    const float lr = __fmul_rn(a.lr, t.lr_scale);
    const float alpha = __fdiv_rn(__fmul_rn(lr, a.root_c2t), a.c1t);
    const float decay = __fsub_rn(1.0f, __fmul_rn(lr, t.weight_decay));
    const float c1 = __fsub_rn(1.0f, a.beta1), c2 = __fsub_rn(1.0f, a.beta2);
    const unsigned tensor_key = mix32(a.key + t.index * 0x9E3779B9u);
    unsigned char *mc = (unsigned char*)t.m, *vc = (unsigned char*)t.v;
    const size_t begin = (size_t)c.number * a.chunk;
    const size_t end = min(t.n, begin + a.chunk);
    const int lane = threadIdx.x & 63;
    // a wavefront takes a whole block: every lane stays in the loop, those past the end with nothing left
    for (size_t b0 = begin + (threadIdx.x >> 6) * BLOCK; b0 < end; b0 += 1024) {
        const size_t block = b0 / BLOCK;
        const size_t i = b0 + lane * 4;
        const unsigned left = i < end ? (unsigned)min((size_t)4, end - i) : 0;
        f32x4u w = {0.f, 0.f, 0.f, 0.f}, g = {0.f, 0.f, 0.f, 0.f};
        unsigned m_old = 0, v_old = 0;
        if (left) {
            w = load4(t.w + i, left);
            m_old = load4(mc + i, left);
            v_old = load4(vc + i, left);
            g = t.g_bf16 ? load4((const unsigned short*)t.g + i, left) : load4((const float*)t.g + i, left);
        }
        const int m_e = t.m_exp[block], v_e = t.v_exp[block];
        float m[4], r[4];
        unsigned m_top = 0, r_top = 0;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const unsigned mb = (m_old >> (8 * k)) & 255, vb = (v_old >> (8 * k)) & 255;
            const float m0 = decode(mb & 127, 20, m_e);
            const float r0 = decode(vb, 19, v_e);
            const float gi = gradient(a, g[k], factor);
            m[k] = __fadd_rn(__fmul_rn(a.beta1, mb & 128 ? -m0 : m0), __fmul_rn(c1, gi));
            r[k] = sqrtf(__fadd_rn(__fmul_rn(a.beta2, __fmul_rn(r0, r0)), __fmul_rn(__fmul_rn(c2, gi), gi)));
            const float up = __fdiv_rn(__fmul_rn(alpha, m[k]), __fadd_rn(r[k], a.eps));
            w[k] = __fsub_rn(__fmul_rn(w[k], decay), up);
            // a state that is not finite is held as zero and leaves the block's exponent alone
            if (!(fabsf(m[k]) < INFINITY)) m[k] = 0.0f;
            if (!(r[k] < INFINITY)) r[k] = 0.0f;
            m_top = max(m_top, __builtin_bit_cast(unsigned, fabsf(m[k])));
            r_top = max(r_top, __builtin_bit_cast(unsigned, r[k]));
        }
        const int m_new = block_exponent(wave_max(m_top), 20), v_new = block_exponent(wave_max(r_top), 19);
        const unsigned block_key = mix32(tensor_key + (unsigned)block * 0x85EBCA6Bu);
        unsigned m_codes = 0, v_codes = 0;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            unsigned m_noise = 1u << 19, r_noise = 1u << 18;  // half a step: to nearest
            if (stochastic) {
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
            store4(t.w + i, w, left);
            store4(mc + i, m_codes, left);
            store4(vc + i, v_codes, left);
            if (t.w_bf16) store4_bf16(t.w_bf16 + i, w, left);
        }
        if (lane == 0) {
            t.m_exp[block] = (unsigned char)m_new;
            t.v_exp[block] = (unsigned char)v_new;
        }
    }
}

// the values that 8-bit states stand for, as bf16 (every one is exact: at most 5 significant bits)
__global__ __launch_bounds__(256) void read_states_kernel(const Tensor* tensors, const Chunk* chunks, unsigned chunk,
                                                          unsigned short* m_out, unsigned short* r_out) {
    const Chunk c = chunks[blockIdx.x];
    const Tensor t = tensors[c.tensor];
    const size_t begin = (size_t)c.number * chunk;
    const size_t end = min(t.n, begin + chunk);
    for (size_t i = begin + threadIdx.x * 4; i < end; i += 1024) {
        const unsigned left = (unsigned)min((size_t)4, end - i);
        const unsigned mc = load4((const unsigned char*)t.m + i, left), vc = load4((const unsigned char*)t.v + i, left);
        const int m_e = t.m_exp[i / BLOCK], v_e = t.v_exp[i / BLOCK];
        f32x4u m, r;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const unsigned mb = (mc >> (8 * k)) & 255, vb = (vc >> (8 * k)) & 255;
            const float x = decode(mb & 127, 20, m_e);
            m[k] = mb & 128 ? -x : x;
            r[k] = decode(vb, 19, v_e);
        }
        if (m_out) store4_bf16(m_out + t.first + i, m, left);
        if (r_out) store4_bf16(r_out + t.first + i, r, left);
    }
}

// ---- global norm ----------------------------------------------------------------------------------------
// Squares are added in 64 bits, so neither the range of the squares nor the length of the sum costs anything
// (the kernel waits for memory).  Each workgroup walks the chunks at a fixed stride and leaves one partial sum;
// the workgroup that finishes last adds the partial sums in their order: the same bits on every call.
__device__ __forceinline__ double block_sum(double x, double* shared) {
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) x += __shfl_xor(x, d, 64);
    if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = x;
    __syncthreads();
    x = shared[0] + shared[1] + shared[2] + shared[3];
    __syncthreads();
    return x;
}

__global__ __launch_bounds__(256) void grad_norm_kernel(const Tensor* tensors, const Chunk* chunks, unsigned count,
                                                        unsigned chunk, double* partial, unsigned* ticket,
                                                        float grad_div, float* norm) {
    __shared__ double shared[4];
    __shared__ bool last;
    double sum = 0.0;
    for (unsigned b = blockIdx.x; b < count; b += gridDim.x) {
        const Chunk c = chunks[b];
        const Tensor t = tensors[c.tensor];
        const size_t begin = (size_t)c.number * chunk;
        const size_t end = min(t.n, begin + chunk);
        for (size_t i = begin + threadIdx.x * 4; i < end; i += 1024) {
            const unsigned left = (unsigned)min((size_t)4, end - i);
            const f32x4u g = t.g_bf16 ? load4((const unsigned short*)t.g + i, left) : load4((const float*)t.g + i, left);
#pragma unroll
            for (int k = 0; k < 4; k++) sum += (double)g[k] * (double)g[k];
        }
    }
    sum = block_sum(sum, shared);
    if (threadIdx.x == 0) {
        partial[blockIdx.x] = sum;
        __threadfence();
        last = atomicInc(ticket, gridDim.x - 1) == gridDim.x - 1;  // wraps to 0 for the next call
    }
    __syncthreads();
    if (!last) return;
    __threadfence();
    sum = 0.0;
    for (unsigned b = threadIdx.x; b < gridDim.x; b += 256) sum += partial[b];
    sum = block_sum(sum, shared);
    if (threadIdx.x == 0) *norm = (float)(sqrt(sum) / (double)grad_div);
}

bool finite_not_negative(float x) { return x >= 0.0f && x < INFINITY; }

// Whether `p` may be handed to a kernel on `device`: not pageable host memory, not another GPU's
bool on_device(const void* p, int device) {
    hipPointerAttribute_t at;
    if (hipPointerGetAttributes(&at, p) != hipSuccess) {
        (void)hipGetLastError();
        return false;
    }
    if (at.type == hipMemoryTypeDevice) return at.device == device;
    return at.type == hipMemoryTypeHost || at.type == hipMemoryTypeManaged;
}

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
    for (int k = 0; k < count; k++) {
        const NerfAdamwTensor& t = tensors[k];
        if (t.n == 0) continue;
        if (t.n > NERF_ADAMW_MAX_ELEMENTS || (t.grad_type != NERF_TYPE_F32 && t.grad_type != NERF_TYPE_BF16)) return NERF_ERR_ARG;
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

struct NerfAdamw {
    int device, state_bits;
    float beta1, beta2, eps;
    unsigned chunk, chunks;
    size_t elements;
    double bytes, grad_bytes;  // of one step, of one norm
    Tensor* d_tensors;
    Chunk* d_chunks;
    double* d_partial;
    unsigned* d_ticket;
};

extern "C" {

size_t nerf_adamw_state_blocks(size_t n) { return n / BLOCK + (n % BLOCK != 0); }

static int build_plan(const NerfAdamwTensor* tensors, int count, int state_bits, NerfAdamw* plan) {
    std::vector<Tensor> table((size_t)count);
    std::vector<Chunk> chunks;
    size_t elements = 0;
    for (int k = 0; k < count; k++) elements += tensors[k].n;
    plan->elements = elements;
    // Up to a million elements a chunk is one piece per thread, so that the few workgroups there are spread over
    // the chip; beyond that, four
    plan->chunk = elements <= (1u << 20) ? 1024 : 4096;
    size_t first = 0;
    for (int k = 0; k < count; k++) {
        const NerfAdamwTensor& s = tensors[k];
        if (s.n) {
            const void* all[] = {s.g, s.w, s.m, s.v, s.m_exp, s.v_exp, s.w_bf16};
            const int used = state_bits == 0 ? 1 : state_bits == 32 ? 4 : 6;
            for (int p = 0; p < 7; p++)
                if ((p < used || (p == 6 && state_bits && s.w_bf16)) && !on_device(all[p], plan->device)) return NERF_ERR_ARG;
        }
        table[k] = Tensor{s.w, s.g, s.m, s.v, s.m_exp, s.v_exp, s.w_bf16, s.n, first, s.lr_scale, s.weight_decay,
                          s.grad_type == NERF_TYPE_BF16, (unsigned)k};
        const double g_item = s.grad_type == NERF_TYPE_BF16 ? 2.0 : 4.0;
        plan->grad_bytes += (double)s.n * g_item;
        plan->bytes += (double)s.n * (8.0 + g_item + (state_bits == 8 ? 4.0 : 16.0) + (s.w_bf16 ? 2.0 : 0.0));
        first += s.n;
        const size_t pieces = s.n / plan->chunk + (s.n % plan->chunk != 0);
        if (chunks.size() + pieces > 0xffffffu) return NERF_ERR_ARG;  // a launch has fewer than 2^32 threads
        for (size_t p = 0; p < pieces; p++) chunks.push_back(Chunk{(unsigned)k, (unsigned)p});
    }
    plan->chunks = (unsigned)chunks.size();
    if (hipMalloc((void**)&plan->d_tensors, table.size() * sizeof(Tensor)) != hipSuccess) return NERF_ERR_HIP;
    if (hipMalloc((void**)&plan->d_chunks, (chunks.size() + 1) * sizeof(Chunk)) != hipSuccess) return NERF_ERR_HIP;
    if (hipMalloc((void**)&plan->d_partial, NORM_BLOCKS * sizeof(double)) != hipSuccess) return NERF_ERR_HIP;
    if (hipMalloc((void**)&plan->d_ticket, sizeof(unsigned)) != hipSuccess) return NERF_ERR_HIP;
    const unsigned zero = 0;
    if (hipMemcpyAsync(plan->d_tensors, table.data(), table.size() * sizeof(Tensor), hipMemcpyHostToDevice, stream()) != hipSuccess ||
        (plan->chunks && hipMemcpyAsync(plan->d_chunks, chunks.data(), chunks.size() * sizeof(Chunk), hipMemcpyHostToDevice,
                                        stream()) != hipSuccess) ||
        hipMemcpyAsync(plan->d_ticket, &zero, sizeof(zero), hipMemcpyHostToDevice, stream()) != hipSuccess ||
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
        (void)hipGetLastError();
        nerf_adamw_destroy(plan);
        return rc;
    }
    *out = plan;
    return NERF_OK;
}

void nerf_adamw_destroy(NerfAdamw* plan) {
    if (!plan) return;
    (void)hipFree(plan->d_tensors);
    (void)hipFree(plan->d_chunks);
    (void)hipFree(plan->d_partial);
    (void)hipFree(plan->d_ticket);
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
        (d_norm && !(max_norm > 0.0f && max_norm < INFINITY)) || !plan_usable(plan))
        return NERF_ERR_ARG;
    // a graph would repeat this step number and learning rate for ever
    hipStreamCaptureStatus capturing = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing(stream(), &capturing) != hipSuccess) return NERF_ERR_HIP;
    if (capturing != hipStreamCaptureStatusNone) return NERF_ERR_ARG;
    if (!plan->chunks) return NERF_OK;
    StepArgs a = {};
    a.tensors = plan->d_tensors;
    a.chunks = plan->d_chunks;
    a.chunk = plan->chunk;
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
    // one 32-bit key per (seed, step): a 64-bit mixing function, its halves folded
    unsigned long long z = seed + (unsigned long long)step * 0x9E3779B97F4A7C15ull;
    z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
    z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
    z ^= z >> 31;
    a.key = (unsigned)(z ^ (z >> 32));
    ProfScope prof(K_ADAMW, plan->bytes);
    if (plan->state_bits == 8)
        hipLaunchKernelGGL(adamw8_kernel, dim3(plan->chunks), dim3(256), 0, stream(), a, seed != 0);
    else
        hipLaunchKernelGGL(adamw32_kernel, dim3(plan->chunks), dim3(256), 0, stream(), a);
    return hipGetLastError() == hipSuccess ? NERF_OK : NERF_ERR_HIP;
}

int nerf_adamw_read_states(NerfAdamw* plan, unsigned short* d_m, unsigned short* d_root_v) {
    if (!plan || plan->state_bits != 8 || (!d_m && !d_root_v) || (((uintptr_t)d_m | (uintptr_t)d_root_v) & 1) || !plan_usable(plan))
        return NERF_ERR_ARG;
    if (!plan->chunks) return NERF_OK;
    hipLaunchKernelGGL(read_states_kernel, dim3(plan->chunks), dim3(256), 0, stream(), plan->d_tensors, plan->d_chunks,
                       plan->chunk, d_m, d_root_v);
    return hipGetLastError() == hipSuccess ? NERF_OK : NERF_ERR_HIP;
}

int nerf_grad_norm(NerfAdamw* plan, float grad_div, float* d_norm) {
    if (!plan || !d_norm || ((uintptr_t)d_norm & 3) || !(grad_div > 0.0f && grad_div < INFINITY) || !plan_usable(plan)) return NERF_ERR_ARG;
    const unsigned blocks = std::max(1u, std::min(plan->chunks, NORM_BLOCKS));
    ProfScope prof(K_GRAD_NORM, plan->grad_bytes);
    hipLaunchKernelGGL(grad_norm_kernel, dim3(blocks), dim3(256), 0, stream(), plan->d_tensors, plan->d_chunks, plan->chunks,
                       plan->chunk, plan->d_partial, plan->d_ticket, grad_div, d_norm);
    return hipGetLastError() == hipSuccess ? NERF_OK : NERF_ERR_HIP;
}

}  // extern "C"
