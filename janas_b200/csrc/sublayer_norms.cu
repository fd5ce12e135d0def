// The norms around a sublayer in one pass: what the sublayer left (a stack of partial sums) is gated, normed, scaled
// and added to the residual stream, and the row that the next sublayer reads is normed while it is still on the chip.
//
//   u  =  (sum_s y[s] + y_bias) * sigmoid(sum_s g[s] + g_bias)        (the gate is optional)
//   x <-  x + mult * scale * N1(u)                                    (N1 and the vector scale are optional)
//   h  =  N2(x)                                                       (optional)
//
// N: a layer norm (t - mean) / sqrt(var + eps) * w + b, var the mean of the squared deviations, or with `rms`
// t / sqrt(mean(t^2) + eps) * w + b.  h is float32, bfloat16 or microscaled 4-bit floats (mx4.cuh).
//
// Bound by memory.  A block per row, which stays in shared memory between the passes.
#include "kernels.h"
#include "mx4.cuh"

namespace jb {

constexpr int OUT_F32 = 0, OUT_BF16 = 1, OUT_MX4 = 4;

struct NormsArgs {
    float *x;
    const float *y, *y_bias, *g, *g_bias, *w1, *b1, *scale, *w2, *b2;
    int Sy, Sg, g_ld, g_col0, rms, out_kind, dm;
    size_t y_stride, g_stride;
    float eps1, mult, eps2;
    void *out;
    uint8_t *scales;
};

// mean (0 with rms) and 1 / sqrt(var + eps) of a row in shared memory
__device__ __forceinline__ void row_moments(const float *row, int dm, float sum, bool rms, float eps, float *red,
                                            float &mean, float &inv)
{
    mean = rms ? 0.0f : block_sum(sum, red) / (float)dm;
    float sq = 0.0f;
    for (int i = threadIdx.x; i < dm; i += blockDim.x) {
        const float d = row[i] - mean;
        sq = fmaf(d, d, sq);
    }
    inv = 1.0f / sqrtf(block_sum(sq, red) / (float)dm + eps);
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
            v = v / (1.0f + expf(-z));
        }
        row[i] = v;
        sum += v;
    }
    float mean = 0.0f, inv = 1.0f;
    if (a.w1)
        row_moments(row, dm, sum, a.rms, a.eps1, red, mean, inv);
    sum = 0.0f;
    for (int i = threadIdx.x; i < dm; i += blockDim.x) {
        float v = row[i];
        if (a.w1)
            v = fmaf((v - mean) * inv, a.w1[i], a.b1 ? a.b1[i] : 0.0f);
        v = fmaf(a.scale ? a.mult * a.scale[i] : a.mult, v, x[i]);
        x[i] = v;
        row[i] = v;
        sum += v;
    }
    if (!a.w2)
        return;
    row_moments(row, dm, sum, a.rms, a.eps2, red, mean, inv);
    if (a.out_kind == OUT_MX4) {
        const int lane = threadIdx.x & 31, chunks = mx4_chunks(dm);
        __syncthreads();
        for (int c = threadIdx.x >> 5; c < chunks; c += blockDim.x >> 5) {
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int i = c * MX4_CHUNK + 8 * lane + j;
                v[j] = i < dm ? fmaf((row[i] - mean) * inv, a.w2[i], a.b2 ? a.b2[i] : 0.0f) : 0.0f;
            }
            mx4_store_chunk(v, r, c, dm, (uint8_t *)a.out, a.scales);
        }
        return;
    }
    for (int i = threadIdx.x; i < dm; i += blockDim.x) {
        const float v = fmaf((row[i] - mean) * inv, a.w2[i], a.b2 ? a.b2[i] : 0.0f);
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
// bfloat16, 4 microscaled 4-bit floats (out the codes, out_scales the scales).
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
        (w2 && out_kind == OUT_MX4 && !out_scales))
        return JB_EINVAL;
    static unsigned long long allowed = 0;
    if (!allow_dynamic_smem(sublayer_norms_kernel, jb_norm_residual_norm_most() * 4, allowed))
        return JB_ELAUNCH;
    NormsArgs a{x, y, y_bias, g, g_bias, w1, b1, scale, w2, b2, Sy, Sg, g_ld, g_col0, rms, out_kind, dm,
                (size_t)y_stride, (size_t)g_stride, eps1, mult, eps2, out, (uint8_t *)out_scales};
    launch(sublayer_norms_kernel, (unsigned)n, 256, (size_t)dm * 4, st, a);
    return launch_status();
}

// The longest row that the kernel keeps in shared memory.
extern "C" int jb_norm_residual_norm_most(void) { return 32768; }
