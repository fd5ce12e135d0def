// Rows and matrices brought to microscaled 4-bit floats (mx4.cuh), and back.
//
// Rows that whole 16-byte loads fit: a warp takes 512 values of a row, sixteen to a lane, so two lanes make a block and one
// shuffle finds its largest magnitude.  Others, and the gated unit: 256 values, eight to a lane.  Bound by the instructions
// it takes to scale, round and pack (and for the unit by its exponential and division), close to what memory takes.
//
// The kernel that quantizes a caller's rows may be followed by a product that reads them as its weights ahead of its
// dependency wait, so unless `early` is set it lets no kernel behind it start before it has ended, and its stores stand
// before a device-wide fence.
#include "kernels.h"
#include "mx4.cuh"

namespace jb {

template <typename T> struct RowSource {
    const T *x;
    int k;
    struct Values {
        float v[8];
    };
    __device__ __forceinline__ void load(size_t r, int col0, Values &t) const
    {
        load8<T, false>(x + r * (size_t)k + col0, k - col0, t.v);
    }
    __device__ __forceinline__ uint32_t pack(Values &t, uint32_t &code) const { return mx4_pack_chunk(t.v, code); }
};

// The gated unit of the sums [S, n, 2 k]: columns [0, k) the gate, [k, 2 k) the up side.
template <bool VEC> struct UnitSource {
    const float *z;
    int S;
    size_t stride;
    int k;
    GatedUnit unit;
    struct Values {
        float v[16];
    };
    __device__ __forceinline__ void load(size_t r, int col0, Values &to) const
    {
        float *v = to.v;
        const float *g = z + r * 2 * (size_t)k + col0, *u = g + k;
        load8<float, VEC>(g, k - col0, v);
        load8<float, VEC>(u, k - col0, v + 8);
        for (int s = 1; s < S; s++) {
            float t[16];
            load8<float, VEC>(g + s * stride, k - col0, t);
            load8<float, VEC>(u + s * stride, k - col0, t + 8);
#pragma unroll
            for (int i = 0; i < 16; i++)
                v[i] += t[i];
        }
    }
    __device__ __forceinline__ uint32_t pack(Values &t, uint32_t &code) const
    {
#pragma unroll
        for (int i = 0; i < 8; i++)
            t.v[i] = gated_unit(t.v[i], t.v[8 + i], unit);
        return mx4_pack_chunk(t.v, code);
    }
};

// total: n times the spans of 512 values of a row.  A warp takes U spans at a time, all read before the first is packed.
template <typename T, typename Values, int U>
__global__ void __launch_bounds__(256)
mx4_rows_kernel(const T *x, uint8_t *__restrict__ codes, uint8_t *__restrict__ scales, unsigned total, int k, int early)
{
    if (early)
        pdl_trigger();
    pdl_wait();
    constexpr int SPAN = 2 * MX4_CHUNK;
    const int lane = threadIdx.x & 31, chunks = mx4_chunks(k);
    const unsigned spans = (unsigned)(chunks + 1) / 2, step = gridDim.x * (blockDim.x >> 5) * U;
    const size_t row_bytes = mx4_row_bytes(k);
    for (unsigned first = (blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5)) * U; first < total;) {
        Values v[U];
        unsigned r = first / spans, c = first - r * spans, r0 = r, q0 = c;
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int col0 = (int)c * SPAN + 16 * lane;
            if (first + u < total)
                v[u].load(x + r * (size_t)k + col0, k - col0);
            if (++c == spans)
                c = 0, r++;
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (first + u < total) {
                uint32_t code;
                const uint2 packed = v[u].pack(code);
                const unsigned at = q0 * (SPAN / 2) + 8 * lane;
                if (at < row_bytes)
                    *reinterpret_cast<uint2 *>(codes + r0 * row_bytes + at) = packed;
                const int ch = 2 * (int)q0 + (lane >> 4);
                if ((lane & 1) == 0 && ch < chunks)
                    scales[mx4_scale_at(r0, ch, chunks, (lane >> 3) & 1) + ((lane >> 1) & 3)] = (uint8_t)code;
            }
            if (++q0 == spans)
                q0 = 0, r0++;
        }
        if (total - first <= step)
            break;
        first += step;
    }
    if (!early)
        __threadfence();
}

// A warp takes a chunk at a time.  total: n times the chunks of a row.
template <typename Source>
__global__ void __launch_bounds__(256)
mx4_quantize_kernel(const Source src, uint8_t *__restrict__ codes, uint8_t *__restrict__ scales, unsigned total, int k, int early)
{
    if (early)
        pdl_trigger();
    pdl_wait();
    const unsigned chunks = mx4_chunks(k), step = gridDim.x * (blockDim.x >> 5);
    for (unsigned i = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); i < total;) {
        typename Source::Values v;
        const unsigned r = i / chunks, c = i - r * chunks;
        uint32_t code;
        src.load(r, c * MX4_CHUNK + 8 * (threadIdx.x & 31), v);
        const uint32_t packed = src.pack(v, code);
        mx4_store_chunk(packed, code, r, c, k, codes, scales);
        if (total - i <= step)
            break;
        i += step;
    }
    if (!early)
        __threadfence();
}

template <typename T, int U, bool VEC>
__global__ void __launch_bounds__(256)
mx4_values_kernel(const uint8_t *codes, const uint8_t *scales, T *__restrict__ out, unsigned total, int k)
{
    pdl_trigger();
    pdl_wait();
    const unsigned chunks = mx4_chunks(k), first = (blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5)) * U;
    const int lane = threadIdx.x & 31;
    const size_t row_bytes = mx4_row_bytes(k);
    uint32_t word[U], scale[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const unsigned i = first + u, r = i / chunks, c = i - r * chunks;
        const int col0 = c * MX4_CHUNK + 8 * lane;
        if (i < total && col0 < k) {
            word[u] = *reinterpret_cast<const uint32_t *>(codes + r * row_bytes + col0 / 2);
            scale[u] = scales[mx4_scale_at(r, c, chunks, lane >> 4) + ((lane >> 2) & 3)];
        }
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        const unsigned i = first + u, r = i / chunks, c = i - r * chunks;
        const int col0 = c * MX4_CHUNK + 8 * lane;
        if (i >= total || col0 >= k)
            continue;
        float v[8];
        mx4_unpack8(word[u], v);
        const float s = mx4_scale(scale[u]);
        T *o = out + r * (size_t)k + col0;
        if (VEC) {
            store4(o, make_float4(v[0] * s, v[1] * s, v[2] * s, v[3] * s));
            store4(o + 4, make_float4(v[4] * s, v[5] * s, v[6] * s, v[7] * s));
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (col0 + j < k)
                    o[j] = from_f<T>(v[j] * s);
        }
    }
}

// Chunks that a warp takes: four once that leaves all SMs 32 warps.
static int mx4_unroll(size_t total) { return total >= (size_t)sm_count() * 32 * 4 ? 4 : 1; }
static unsigned mx4_grid(size_t total, int unroll) { return (unsigned)((total + 8 * unroll - 1) / (8 * unroll)); }

template <typename Source>
static int quantize(const Source &src, void *codes, void *scales, int n, int k, int early, cudaStream_t st)
{
    const size_t total = (size_t)n * mx4_chunks(k);
    if (total > 0xffffff00u)
        return JB_EINVAL;
    const unsigned most = (unsigned)sm_count() * 8, grid = mx4_grid(total, 1);
    launch(mx4_quantize_kernel<Source>, grid < most ? grid : most, 256, 0, st, src, (uint8_t *)codes, (uint8_t *)scales,
           (unsigned)total, k, early);
    return launch_status();
}

template <typename T, typename Values>
static int quantize_rows(const T *x, void *codes, void *scales, int n, int k, int early, cudaStream_t st)
{
    const size_t total = (size_t)n * ((mx4_chunks(k) + 1) / 2);
    if (total > 0xffffff00u)
        return JB_EINVAL;
    const int u = mx4_unroll(total) > 1 ? 2 : 1;
    const unsigned most = (unsigned)sm_count() * 8, grid = mx4_grid(total, u);
    launch(u > 1 ? mx4_rows_kernel<T, Values, 2> : mx4_rows_kernel<T, Values, 1>, grid < most ? grid : most, 256, 0, st, x,
           (uint8_t *)codes, (uint8_t *)scales, (unsigned)total, k, early);
    return launch_status();
}

template <typename T, bool VEC>
static int values(const void *codes, const void *scales, T *out, int n, int k, cudaStream_t st)
{
    const size_t total = (size_t)n * mx4_chunks(k);
    if (total > 0xffffff00u)
        return JB_EINVAL;
    const int u = mx4_unroll(total);
    launch(u == 4 ? mx4_values_kernel<T, 4, VEC> : mx4_values_kernel<T, 1, VEC>, mx4_grid(total, u), 256, 0, st,
           (const uint8_t *)codes, (const uint8_t *)scales, out, (unsigned)total, k);
    return launch_status();
}

}  // namespace jb

using namespace jb;

static bool bad_size(int n, int k) { return n < 0 || k < 1 || n > MX4_MOST || k > MX4_MOST; }

extern "C" long long jb_mx4_code_bytes(int rows, int k)
{
    return bad_size(rows, k) ? 0 : (long long)(mx4_row_bytes(k) * (size_t)rows);
}
extern "C" long long jb_mx4_scale_bytes(int rows, int k)
{
    return bad_size(rows, k) ? 0 : (long long)((size_t)((rows + 127) / 128) * mx4_chunks(k) * MX4_TILE);
}

static bool bad_target(const void *codes, const void *scales, int n, int k)
{
    return bad_size(n, k) || (uintptr_t)codes % 16 != 0 || (uintptr_t)scales % 16 != 0;
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
    if (dt == 1)
        return vec ? quantize_rows<bf16, SixteenBf16>((const bf16 *)x, codes, scales, n, k, early, st)
                   : quantize(RowSource<bf16>{(const bf16 *)x, k}, codes, scales, n, k, early, st);
    return vec ? quantize_rows<float, Sixteen>((const float *)x, codes, scales, n, k, early, st)
               : quantize(RowSource<float>{(const float *)x, k}, codes, scales, n, k, early, st);
}

// The gated unit (see jb_gated_unit) of z, a stack [S, n, 2 ff] of sums, in 4 bits.
extern "C" int jb_mx4_gated_unit(const float *z, int S, long long stride, void *codes, void *scales, int n, int ff,
                                 float alpha, float limit, float shift, cudaStream_t st)
{
    if (bad_target(codes, scales, n, ff) || S < 1 || ff > 0x3fffffff)
        return JB_EINVAL;
    if (n == 0)
        return JB_OK;
    const GatedUnit unit{alpha, limit, shift};
    if (ff % 8 == 0 && (uintptr_t)z % 16 == 0 && stride % 4 == 0)
        return quantize(UnitSource<true>{z, S, (size_t)stride, ff, unit}, codes, scales, n, ff, 1, st);
    return quantize(UnitSource<false>{z, S, (size_t)stride, ff, unit}, codes, scales, n, ff, 1, st);
}

// What codes and scales stand for, as [n, k].
extern "C" int jb_mx4_values(const void *codes, const void *scales, void *out, int out_dt, int n, int k, cudaStream_t st)
{
    if (bad_target(codes, scales, n, k) || (out_dt != 0 && out_dt != 1))
        return JB_EINVAL;
    if (n == 0)
        return JB_OK;
    const bool vec = k % 8 == 0 && (uintptr_t)out % 16 == 0;
    if (out_dt == 1)
        return vec ? values<bf16, true>(codes, scales, (bf16 *)out, n, k, st)
                   : values<bf16, false>(codes, scales, (bf16 *)out, n, k, st);
    return vec ? values<float, true>(codes, scales, (float *)out, n, k, st)
               : values<float, false>(codes, scales, (float *)out, n, k, st);
}
