// Products of microscaled 4-bit floats (mx4.cuh):
//
//     out[r, f] = sum over blocks b of 2^(sa[r, b] + sw[f, b]) * sum over i in b of pa[r, i] pw[f, i]
//
// A thread per output.  Twice a 4-bit number is a whole number up to 12, so a block's sum is exact in integers; the
// blocks' sums are added in float32, in order.
#include "kernels.h"
#include "mx4.cuh"

namespace jb {

// twice the numbers of the low halves of four bytes, as four signed bytes
__device__ __forceinline__ int mx4_twice(uint32_t nibbles)
{
    const uint32_t m = nibbles & 0x07070707u, s = (nibbles >> 3) & 0x01010101u;
    const uint32_t sel = (m & 7) | (m >> 4 & 0x70) | (m >> 8 & 0x700) | (m >> 12 & 0x7000);
    const uint32_t v = __byte_perm(0x03020100u, 0x0c080604u, sel);
    const uint32_t neg = s * 255u;
    return (int)__vsub4(v ^ neg, neg);
}

template <typename TO>
__global__ void __launch_bounds__(256)
mx4_product_kernel(const uint8_t *ac, const uint8_t *as, const uint8_t *wc, const uint8_t *ws, TO *__restrict__ out, int n,
                   int m, int k)
{
    pdl_trigger();
    pdl_wait();
    const int f = blockIdx.y * 32 + (threadIdx.x & 31);
    const size_t r = (size_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (f >= m || r >= (size_t)n)
        return;
    const size_t row_bytes = mx4_row_bytes(k);
    const int chunks = mx4_chunks(k), blocks = (k + 31) / 32;
    float sum = 0.0f;
    for (int b = 0; b < blocks; b++) {
        const uint4 a = *reinterpret_cast<const uint4 *>(ac + r * row_bytes + (size_t)b * 16);
        const uint4 w = *reinterpret_cast<const uint4 *>(wc + (size_t)f * row_bytes + (size_t)b * 16);
        const uint32_t av[4] = {a.x, a.y, a.z, a.w}, wv[4] = {w.x, w.y, w.z, w.w};
        int dot = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            dot = __dp4a(mx4_twice(av[i]), mx4_twice(wv[i]), dot);
            dot = __dp4a(mx4_twice(av[i] >> 4), mx4_twice(wv[i] >> 4), dot);
        }
        const int half = (b >> 2) & 1, q = b & 3;
        const float sa = mx4_scale(as[mx4_scale_at(r, b >> 3, chunks, half) + q]);
        const float sw = mx4_scale(ws[mx4_scale_at(f, b >> 3, chunks, half) + q]);
        sum += 0.25f * (float)dot * sa * sw;
    }
    out[r * m + f] = from_f<TO>(sum);
}

}  // namespace jb

using namespace jb;

// out [n, m] (out_dt 0 float32, 1 bfloat16) = a [n, k] . w [m, k]^T, both as codes and scales.
extern "C" int jb_linear_mx4(const void *a_codes, const void *a_scales, const void *w_codes, const void *w_scales, void *out,
                             int out_dt, int n, int m, int k, cudaStream_t st)
{
    if (n < 0 || m < 0 || k < 1 || (out_dt != 0 && out_dt != 1) || (uintptr_t)a_codes % 16 || (uintptr_t)w_codes % 16 ||
        (uintptr_t)a_scales % 16 || (uintptr_t)w_scales % 16 || (m + 31) / 32 > 65535)
        return JB_EINVAL;
    if (n == 0 || m == 0)
        return JB_OK;
    const dim3 grid((unsigned)((n + 7) / 8), (unsigned)((m + 31) / 32));
    if (out_dt == 1)
        launch(mx4_product_kernel<bf16>, grid, 256, 0, st, (const uint8_t *)a_codes, (const uint8_t *)a_scales,
               (const uint8_t *)w_codes, (const uint8_t *)w_scales, (bf16 *)out, n, m, k);
    else
        launch(mx4_product_kernel<float>, grid, 256, 0, st, (const uint8_t *)a_codes, (const uint8_t *)a_scales,
               (const uint8_t *)w_codes, (const uint8_t *)w_scales, (float *)out, n, m, k);
    return launch_status();
}
