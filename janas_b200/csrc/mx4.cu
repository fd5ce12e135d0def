// Rows and matrices brought to microscaled 4-bit floats (mx4.cuh), and back.
//
// A warp takes a chunk of 256 values of a row, eight to a lane: four lanes make a block, whose largest magnitude they
// find by two shuffles; the lane's codes are one word.  Bound by memory: a value read, 17 / 32 of a byte written.
//
// The kernel that quantizes a caller's rows may be followed by a product that reads them as its weights ahead of its
// dependency wait, so unless `early` is set it lets no kernel behind it start before it has ended, and its stores stand
// before a device-wide fence.
#include "kernels.h"
#include "mx4.cuh"

namespace jb {

// Eight consecutive values of a row from column col0 on; zeros past the row's end.
template <typename T, bool VEC> struct RowSource {
    const T *x;
    int k;
    __device__ __forceinline__ void load(size_t r, int col0, float *v) const
    {
        const T *p = x + r * (size_t)k + col0;
        if (VEC) {
            float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
            if (col0 < k) {
                a = load4(p);
                b = load4(p + 4);
            }
            v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
            v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++)
                v[i] = col0 + i < k ? to_f(p[i]) : 0.0f;
        }
    }
};

// The gated unit of the sums [S, n, 2 k]: columns [0, k) the gate, [k, 2 k) the up side.
struct UnitSource {
    const float *z;
    int S;
    size_t stride;
    int k;
    GatedUnit unit;
    __device__ __forceinline__ void load(size_t r, int col0, float *v) const
    {
        const float *g = z + r * 2 * (size_t)k + col0, *u = g + k;
#pragma unroll
        for (int i = 0; i < 8; i++)
            v[i] = col0 + i < k ? gated_unit(add_partials(0.0f, g + i, S, stride), add_partials(0.0f, u + i, S, stride), unit)
                                : 0.0f;
    }
};

template <typename Source>
__global__ void __launch_bounds__(256)
mx4_quantize_kernel(const Source src, uint8_t *__restrict__ codes, uint8_t *__restrict__ scales, int n, int k, int early)
{
    if (early)
        pdl_trigger();
    pdl_wait();
    const int chunks = mx4_chunks(k);
    const size_t total = (size_t)n * chunks, step = (size_t)gridDim.x * (blockDim.x >> 5);
    for (size_t i = (size_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); i < total; i += step) {
        const size_t r = i / chunks;
        const int c = (int)(i - r * chunks);
        float v[8];
        src.load(r, c * MX4_CHUNK + 8 * (threadIdx.x & 31), v);
        mx4_store_chunk(v, r, c, k, codes, scales);
    }
    if (!early)
        __threadfence();
}

template <typename T>
__global__ void __launch_bounds__(256)
mx4_values_kernel(const uint8_t *codes, const uint8_t *scales, T *__restrict__ out, int n, int k)
{
    pdl_trigger();
    pdl_wait();
    const int chunks = mx4_chunks(k), lane = threadIdx.x & 31;
    const size_t total = (size_t)n * chunks, step = (size_t)gridDim.x * (blockDim.x >> 5), row_bytes = mx4_row_bytes(k);
    for (size_t i = (size_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); i < total; i += step) {
        const size_t r = i / chunks;
        const int c = (int)(i - r * chunks), col0 = c * MX4_CHUNK + 8 * lane;
        if (col0 >= k)
            continue;
        float v[8];
        mx4_unpack8(*reinterpret_cast<const uint32_t *>(codes + r * row_bytes + col0 / 2), v);
        const float s = mx4_scale(scales[mx4_scale_at(r, c, chunks, lane >> 4) + ((lane >> 2) & 3)]);
        T *o = out + r * (size_t)k + col0;
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (col0 + j < k)
                o[j] = from_f<T>(v[j] * s);
    }
}

static unsigned warps_grid(size_t chunks)
{
    const size_t blocks = (chunks + 7) / 8, most = (size_t)sm_count() * 8;
    return (unsigned)(blocks < most ? blocks : most);
}

}  // namespace jb

using namespace jb;

extern "C" long long jb_mx4_code_bytes(int rows, int k) { return rows < 0 || k < 1 ? 0 : (long long)(mx4_row_bytes(k) * (size_t)rows); }
extern "C" long long jb_mx4_scale_bytes(int rows, int k)
{
    return rows < 0 || k < 1 ? 0 : (long long)((size_t)((rows + 127) / 128) * mx4_chunks(k) * MX4_TILE);
}

static bool bad_target(const void *codes, const void *scales, int n, int k)
{
    return n < 0 || k < 1 || (uintptr_t)codes % 16 != 0 || (uintptr_t)scales % 16 != 0;
}

// x [n, k] -> codes and scales.  early: kernels behind this one may start before it has ended (they must then not
// read the result ahead of their dependency wait).
extern "C" int jb_mx4_quantize(const void *x, int dt, void *codes, void *scales, int n, int k, int early, cudaStream_t st)
{
    if (bad_target(codes, scales, n, k) || (dt != 0 && dt != 1))
        return JB_EINVAL;
    if (n == 0)
        return JB_OK;
    const bool vec = k % 8 == 0 && (uintptr_t)x % 16 == 0;
    const unsigned grid = warps_grid((size_t)n * mx4_chunks(k));
#define JB_Q(T, V) \
    launch(mx4_quantize_kernel<RowSource<T, V>>, grid, 256, 0, st, RowSource<T, V>{(const T *)x, k}, (uint8_t *)codes, \
           (uint8_t *)scales, n, k, early)
    if (dt == 1)
        vec ? JB_Q(bf16, true) : JB_Q(bf16, false);
    else
        vec ? JB_Q(float, true) : JB_Q(float, false);
#undef JB_Q
    return launch_status();
}

// The gated unit (see jb_gated_unit) of z, a stack [S, n, 2 ff] of sums, in 4 bits.
extern "C" int jb_mx4_gated_unit(const float *z, int S, long long stride, void *codes, void *scales, int n, int ff,
                                 float alpha, float limit, float shift, cudaStream_t st)
{
    if (bad_target(codes, scales, n, ff) || S < 1 || ff > 0x3fffffff)
        return JB_EINVAL;
    if (n == 0)
        return JB_OK;
    launch(mx4_quantize_kernel<UnitSource>, warps_grid((size_t)n * mx4_chunks(ff)), 256, 0, st,
           UnitSource{z, S, (size_t)stride, ff, GatedUnit{alpha, limit, shift}}, (uint8_t *)codes, (uint8_t *)scales, n, ff, 1);
    return launch_status();
}

// What codes and scales stand for, as [n, k].
extern "C" int jb_mx4_values(const void *codes, const void *scales, void *out, int out_dt, int n, int k, cudaStream_t st)
{
    if (bad_target(codes, scales, n, k) || (out_dt != 0 && out_dt != 1))
        return JB_EINVAL;
    if (n == 0)
        return JB_OK;
    const unsigned grid = warps_grid((size_t)n * mx4_chunks(k));
    if (out_dt == 1)
        launch(mx4_values_kernel<bf16>, grid, 256, 0, st, (const uint8_t *)codes, (const uint8_t *)scales, (bf16 *)out, n, k);
    else
        launch(mx4_values_kernel<float>, grid, 256, 0, st, (const uint8_t *)codes, (const uint8_t *)scales, (float *)out, n, k);
    return launch_status();
}
