// The norms around a sublayer in one pass: what the sublayer left (a stack of partial sums) is gated, normed, scaled
// and added to the residual stream, and the row that the next sublayer reads is normed while it is still on the chip.
//
//   u  =  (sum_s y[s] + y_bias) * sigmoid(sum_s g[s] + g_bias)        (the gate is optional)
//   x <-  x + mult * scale * N1(u)                                    (N1 and the vector scale are optional)
//   h  =  N2(x)                                                       (optional)
//
// Every product and sum is rounded by itself and the norms' factor is one reciprocal root, so that the steps one by one give
// the same values up to their sums' order: what is left of a difference decides how often the 4-bit form of h falls on the
// other side of a border.
//
// N: a layer norm (t - mean) / sqrt(var + eps) * w + b, var the mean of the squared deviations, or with `rms`
// t / sqrt(mean(t^2) + eps) * w + b.  h is float32, bfloat16 or microscaled 4-bit floats (mx4.cuh).
//
// Bound by instructions and memory, and for few rows by the chain of sums.  A block per row, which stays in registers between
// the sums, two groups of four values a thread (2,048 rows of 2,560 with a gate: 31 us from memory and 21 from the L2, where
// the bytes take 14; with five groups and a quarter of the warps 42 from memory, with one group 37, though 8 rows then take
// 3.5 instead of 4.2; with each block's next row prefetched into shared memory 36, into the L2 31).  Rows that whole 16-byte
// loads do not fit, or longer ones, stay in shared memory.
// How a row is shared out among the threads depends on its length and on whether whole 16-byte loads fit (every address, the
// stacks' strides, the gate's width and first column), so its bits are the same in any batch that is laid out alike, as a
// layer's are from step to step; rows that start elsewhere in memory may differ in their sums' order.
#include "kernels.h"
#include "mx4.cuh"

namespace jb {

constexpr int OUT_F32 = 0, OUT_BF16 = 1, OUT_MX4 = 4;

struct NormsArgs {
    float *x;
    const float *y, *y_bias, *g, *g_bias, *w1, *b1, *scale, *w2, *b2;
    int Sy, Sg, g_ld, g_col0, rms, out_kind, dm;
    size_t y_stride, g_stride;
    float eps1, mult, eps2, inv_dm;
    void *out;
    uint8_t *scales;
};

__device__ __forceinline__ float gated(float v, float z) { return __fmul_rn(v, __frcp_rn(1.0f + expf(-z))); }
// t inv w (+ b), and x + c t
__device__ __forceinline__ float normed(float t, float inv, float w, const float *b)
{
    const float v = __fmul_rn(__fmul_rn(t, inv), w);
    return b ? __fadd_rn(v, *b) : v;
}
__device__ __forceinline__ float added(float x, float c, float t) { return __fadd_rn(x, __fmul_rn(c, t)); }

// mean (0 with rms) and 1 / sqrt(var + eps) of a row in shared memory
__device__ __forceinline__ void row_moments(const float *row, int dm, float inv_dm, float sum, bool rms, float eps, float *red,
                                            float &mean, float &inv)
{
    mean = rms ? 0.0f : block_sum(sum, red) * inv_dm;
    float sq = 0.0f;
    for (int i = threadIdx.x; i < dm; i += blockDim.x) {
        const float d = row[i] - mean;
        sq = fmaf(d, d, sq);
    }
    inv = rsqrtf(block_sum(sq, red) * inv_dm + eps);
}

// The sum of v over a block of at most W warps: every thread adds up all warps' sums, in order, from slots that no other sum
// uses (zeros where there is no warp), so one barrier is enough.
template <int W>
__device__ __forceinline__ float slot_sum(float v, float *slots)
{
    v = warp_sum(v);
    if ((threadIdx.x & 31) == 0)
        slots[threadIdx.x >> 5] = v;
    __syncthreads();
    float t = 0.0f;
#pragma unroll
    for (int w = 0; w < W; w += 4) {
        const float4 u = load4(slots + w);
        t += (u.x + u.y) + (u.z + u.w);
    }
    return t;
}

__device__ __forceinline__ float sum4(const float4 &v) { return (v.x + v.y) + (v.z + v.w); }

// The norm of a row in registers: t <- (t - mean) / sqrt(var + eps) * w + b.  Values past the row's end are zeros before
// and whatever comes out after.
template <int NV, int W>
__device__ __forceinline__ void norm_row(float4 *t, int dm, float inv_dm, bool rms, float eps, const float *w, const float *b, float *slots)
{
    float mean = 0.0f;
    if (!rms) {
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < NV; j++)
            sum += sum4(t[j]);
        mean = slot_sum<W>(sum, slots) * inv_dm;
    }
    float sq = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; j++) {
        if (4 * (int)(threadIdx.x + j * blockDim.x) < dm) {
            t[j].x -= mean, t[j].y -= mean, t[j].z -= mean, t[j].w -= mean;
            sq += (t[j].x * t[j].x + t[j].y * t[j].y) + (t[j].z * t[j].z + t[j].w * t[j].w);
        }
    }
    const float inv = rsqrtf(slot_sum<W>(sq, slots + W) * inv_dm + eps);
#pragma unroll
    for (int j = 0; j < NV; j++) {
        const int i = 4 * (threadIdx.x + j * blockDim.x);
        if (i < dm) {
            const float4 u = load4(w + i);
            t[j] = make_float4(normed(t[j].x, inv, u.x, nullptr), normed(t[j].y, inv, u.y, nullptr),
                               normed(t[j].z, inv, u.z, nullptr), normed(t[j].w, inv, u.w, nullptr));
            if (b) {
                const float4 c = load4(b + i);
                t[j] = make_float4(__fadd_rn(t[j].x, c.x), __fadd_rn(t[j].y, c.y), __fadd_rn(t[j].z, c.z), __fadd_rn(t[j].w, c.w));
            }
        }
    }
}

// The sum of four columns over a stack, after a vector or nothing.
__device__ __forceinline__ float4 sum_stack(const float *bias, const float *p, int S, size_t stride)
{
    float4 v = load4(p);
    if (bias) {
        const float4 c = load4(bias);
        v.x += c.x, v.y += c.y, v.z += c.z, v.w += c.w;
    }
    for (int s = 1; s < S; s++) {
        const float4 u = load4(p + s * stride);
        v.x += u.x, v.y += u.y, v.z += u.z, v.w += u.w;
    }
    return v;
}

// From the gated sums t and the old x of a row: x and h.
template <int NV, int W>
__device__ __forceinline__ void finish_row(const NormsArgs &a, size_t r, float4 *t, const float4 *old, float (*slots)[W])
{
    const int dm = a.dm;
    float *x = a.x + r * dm;
    if (a.w1)
        norm_row<NV, W>(t, dm, a.inv_dm, a.rms, a.eps1, a.w1, a.b1, slots[0]);
#pragma unroll
    for (int j = 0; j < NV; j++) {
        const int i = 4 * (threadIdx.x + j * blockDim.x);
        if (i < dm) {
            const float4 c = a.scale ? load4(a.scale + i) : make_float4(1.f, 1.f, 1.f, 1.f);
            t[j] = make_float4(added(old[j].x, a.mult * c.x, t[j].x), added(old[j].y, a.mult * c.y, t[j].y),
                               added(old[j].z, a.mult * c.z, t[j].z), added(old[j].w, a.mult * c.w, t[j].w));
            store4(x + i, t[j]);
        }
    }
    if (!a.w2)
        return;
    norm_row<NV, W>(t, dm, a.inv_dm, a.rms, a.eps2, a.w2, a.b2, slots[2]);
    const int blocks = (dm + 31) / 32, chunks = mx4_chunks(dm);
#pragma unroll
    for (int j = 0; j < NV; j++) {
        const int g = threadIdx.x + j * blockDim.x, i = 4 * g;
        if (a.out_kind == OUT_MX4) {
            // eight lanes have a block; what lies past the row's end in its last one is zero
            uint32_t code;
            const uint32_t packed = mx4_pack4(i < dm ? t[j] : make_float4(0.f, 0.f, 0.f, 0.f), code);
            if (g < 8 * blocks)
                *reinterpret_cast<uint16_t *>((uint8_t *)a.out + r * mx4_row_bytes(dm) + 2 * g) = (uint16_t)packed;
            const int b = g >> 3;
            if ((g & 7) == 0 && b < blocks)
                a.scales[mx4_scale_at(r, b >> 3, chunks, (b >> 2) & 1) + (b & 3)] = (uint8_t)code;
        } else if (i < dm) {
            if (a.out_kind == OUT_BF16)
                store4((bf16 *)a.out + r * dm + i, t[j]);
            else
                store4((float *)a.out + r * dm + i, t[j]);
        }
    }
    if (a.out_kind == OUT_MX4) {
        const int b = blocks + threadIdx.x;         // the last chunk's blocks past the row's end
        if (b < 8 * chunks)
            a.scales[mx4_scale_at(r, b >> 3, chunks, (b >> 2) & 1) + (b & 3)] = 0;
    }
}

__device__ __forceinline__ float4 gated4(const float4 &v, const float4 &z)
{
    return make_float4(gated(v.x, z.x), gated(v.y, z.y), gated(v.z, z.z), gated(v.w, z.w));
}

// NV groups of four values a thread, at most W warps; every address at a 16-byte boundary.
template <int NV, int W>
__global__ void __maxnreg__(NV == 2 ? 48 : 64)
sublayer_norms_vec_kernel(const NormsArgs a)
{
    __shared__ __align__(16) float slots[4][W];
    if (threadIdx.x < 4 * W)
        slots[0][threadIdx.x] = 0.0f;
    pdl_trigger();
    __syncthreads();
    pdl_wait();
    const size_t r = blockIdx.x;
    float4 t[NV], old[NV];
#pragma unroll
    for (int j = 0; j < NV; j++) {
        const int i = 4 * (threadIdx.x + j * blockDim.x);
        t[j] = old[j] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (i < a.dm) {
            old[j] = load4(a.x + r * a.dm + i);
            t[j] = sum_stack(a.y_bias ? a.y_bias + i : nullptr, a.y + r * a.dm + i, a.Sy, a.y_stride);
            if (a.g)
                t[j] = gated4(t[j], sum_stack(a.g_bias ? a.g_bias + i : nullptr, a.g + r * a.g_ld + a.g_col0 + i, a.Sg, a.g_stride));
        }
    }
    finish_row<NV, W>(a, r, t, old, slots);
}

__global__ void __launch_bounds__(256)
sublayer_norms_kernel(const NormsArgs a)
{
    extern __shared__ float row[];
    __shared__ float red[32];
    pdl_trigger();
    pdl_wait();
    const size_t r = blockIdx.x;
    const int dm = a.dm;
    float *x = a.x + r * dm;
    float sum = 0.0f;
    for (int i = threadIdx.x; i < dm; i += blockDim.x) {
        float v = add_partials(a.y_bias ? a.y_bias[i] : 0.0f, a.y + r * dm + i, a.Sy, a.y_stride);
        if (a.g) {
            const float z = add_partials(a.g_bias ? a.g_bias[i] : 0.0f, a.g + r * a.g_ld + a.g_col0 + i, a.Sg, a.g_stride);
            v = gated(v, z);
        }
        row[i] = v;
        sum += v;
    }
    float mean = 0.0f, inv = 1.0f;
    if (a.w1)
        row_moments(row, dm, a.inv_dm, sum, a.rms, a.eps1, red, mean, inv);
    sum = 0.0f;
    for (int i = threadIdx.x; i < dm; i += blockDim.x) {
        float v = row[i];
        if (a.w1)
            v = normed(v - mean, inv, a.w1[i], a.b1 ? a.b1 + i : nullptr);
        v = added(x[i], a.scale ? a.mult * a.scale[i] : a.mult, v);
        x[i] = v;
        row[i] = v;
        sum += v;
    }
    if (!a.w2)
        return;
    row_moments(row, dm, a.inv_dm, sum, a.rms, a.eps2, red, mean, inv);
    if (a.out_kind == OUT_MX4) {
        const int lane = threadIdx.x & 31, chunks = mx4_chunks(dm);
        __syncthreads();
        for (int c = threadIdx.x >> 5; c < chunks; c += blockDim.x >> 5) {
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int i = c * MX4_CHUNK + 8 * lane + j;
                v[j] = i < dm ? normed(row[i] - mean, inv, a.w2[i], a.b2 ? a.b2 + i : nullptr) : 0.0f;
            }
            uint32_t code;
            const uint32_t packed = mx4_pack_chunk(v, code);
            mx4_store_chunk(packed, code, r, c, dm, (uint8_t *)a.out, a.scales);
        }
        return;
    }
    for (int i = threadIdx.x; i < dm; i += blockDim.x) {
        const float v = normed(row[i] - mean, inv, a.w2[i], a.b2 ? a.b2 + i : nullptr);
        if (a.out_kind == OUT_BF16)
            ((bf16 *)a.out)[r * dm + i] = from_f<bf16>(v);
        else
            ((float *)a.out)[r * dm + i] = v;
    }
}

}  // namespace jb

using namespace jb;

// y: a stack [Sy, n, dm]; g: a stack [Sg, n, g_ld] whose columns g_col0 .. g_col0 + dm - 1 are the gate, or null; biases,
// weights and scale float32 [dm] or null (w1 null: no norm of the result; w2 null: no h).  out_kind: 0 float32, 1
// bfloat16, 4 microscaled 4-bit floats (out the codes, at an address that 16 divides, out_scales the scales).
extern "C" int jb_norm_residual_norm(float *x, const float *y, int Sy, long long y_stride, const float *y_bias,
                                     const float *g, int Sg, long long g_stride, int g_ld, int g_col0, const float *g_bias,
                                     const float *w1, const float *b1, float eps1, const float *scale, float mult,
                                     const float *w2, const float *b2, float eps2, int rms, void *out, void *out_scales,
                                     int out_kind, int n, int dm, cudaStream_t st)
{
    if (n == 0 && dm > 0 && dm <= jb_norm_residual_norm_most())
        return JB_OK;
    if (n < 0 || dm < 1 || Sy < 1 || (g && (Sg < 1 || g_col0 < 0 || g_ld - g_col0 < dm)) || dm > jb_norm_residual_norm_most() ||
        (w2 && !out) || (out_kind != OUT_F32 && out_kind != OUT_BF16 && out_kind != OUT_MX4) ||
        (w2 && out_kind == OUT_MX4 && (!out_scales || (uintptr_t)out % 16 != 0)))
        return JB_EINVAL;
    NormsArgs a{x, y, y_bias, g, g_bias, w1, b1, scale, w2, b2, Sy, Sg, g_ld, g_col0, rms, out_kind, dm,
                (size_t)y_stride, (size_t)g_stride, eps1, mult, eps2, 1.0f / dm, out, (uint8_t *)out_scales};
    const uintptr_t all = (uintptr_t)x | (uintptr_t)y | (uintptr_t)y_bias | (uintptr_t)g | (uintptr_t)g_bias | (uintptr_t)w1 |
                          (uintptr_t)b1 | (uintptr_t)scale | (uintptr_t)w2 | (uintptr_t)b2 | (uintptr_t)out;
    if (dm % 4 == 0 && dm <= 16384 && all % 16 == 0 && y_stride % 4 == 0 && (!g || (g_stride % 4 == 0 && g_ld % 4 == 0 && g_col0 % 4 == 0))) {
        #define JB_ROW(NV, W)                                                                          \
    if (dm <= 128 * W * NV) {                                                                  \
        launch(sublayer_norms_vec_kernel<NV, W>, (unsigned)n, 32 * ((dm + 128 * NV - 1) / (128 * NV)), 0, st, a); \
        return launch_status();                                                                \
    }
        JB_ROW(2, 4) JB_ROW(2, 8) JB_ROW(2, 12) JB_ROW(2, 16) JB_ROW(2, 32) JB_ROW(4, 32)
#undef JB_ROW
    }
    static unsigned long long allowed = 0;
    if (!allow_dynamic_smem(sublayer_norms_kernel, jb_norm_residual_norm_most() * 4, allowed))
        return JB_ELAUNCH;
    launch(sublayer_norms_kernel, (unsigned)n, 256, (size_t)dm * 4, st, a);
    return launch_status();
}

// The longest row that the kernel keeps in shared memory.
extern "C" int jb_norm_residual_norm_most(void) { return 32768; }
