// Microscaled 4-bit floats: a block of 32 values along a row stands for 2^s times 32 numbers of one sign, two
// exponent and one mantissa bit (0, 0.5, 1, 1.5, 2, 3, 4, 6).
//
//   s = max(floor(log2 max |x|) - 2, -127),   number = x / 2^s rounded to nearest, ties to even, at most 6
//
// so the block's largest value lies in [4, 8) before the rounding and what lies above 6 becomes 6.  A block with a NaN
// or an infinity stands for NaNs.  The last block of a row is filled up with zeros.
//
// In memory: codes [rows, 16 ceil(k / 32)] bytes, value 2i in the low half of byte i; scales [ceil(rows / 128),
// ceil(k / 256), 1024] bytes, s + 127 (255: NaN), a chunk of 256 values of 128 rows together: in the order in which the
// tensor cores take them (four consecutive blocks of row r at 16 (r % 32) + 4 (r / 32 % 4), the other four 512 behind).
#pragma once

#include "common.cuh"

namespace jb {

constexpr int MX4_CHUNK = 256;              // values of a row that a chunk of scales is for
constexpr int MX4_TILE = 1024;              // its bytes, for 128 rows
constexpr int MX4_MOST = 0x7fffff00;        // most rows, and values of a row: padded to a chunk or tile they are an int

__host__ __device__ inline size_t mx4_row_bytes(int k) { return (size_t)((k + 31) / 32) * 16; }
__host__ __device__ inline int mx4_chunks(int k) { return (k + MX4_CHUNK - 1) / MX4_CHUNK; }
// the place of the first four (half 0) or last four (half 1) scales of row r's chunk c
__host__ __device__ inline size_t mx4_scale_at(size_t r, int c, int chunks, int half)
{
    return ((r >> 7) * (size_t)chunks + (size_t)c) * MX4_TILE + half * 512 + (r & 31) * 16 + ((r >> 5) & 3) * 4;
}

// s + 127 of a block from the bits of its largest magnitude
__device__ __forceinline__ uint32_t mx4_scale_code(uint32_t top)
{
    if (top >= 0x7f800000u)
        return 255u;
    uint32_t e = top >> 23;
    return e > 2u ? e - 2u : 0u;
}

// 2^-s of a scale's code (0 .. 252); the products with it are exact
__device__ __forceinline__ float mx4_inverse(uint32_t code)
{
    return __uint_as_float((254u - min(code, 252u)) << 23);
}

// 2^s (a subnormal float for the code 0, NaN for 255)
__device__ __forceinline__ float mx4_scale(uint32_t code)
{
    return __uint_as_float(code == 255u ? 0x7fffffffu : code == 0u ? 0x00400000u : code << 23);
}

// Eight values rounded to 4 bits: value i in bits 4 i.
__device__ __forceinline__ uint32_t mx4_pack8(const float *v)
{
    uint32_t r;
    asm("{\n\t"
        ".reg .b8 a, b, c, d;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
        "mov.b32 %0, {a, b, c, d};\n\t"
        "}\n"
        : "=r"(r)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return r;
}
// The same of the values times inv, a power of two.
__device__ __forceinline__ uint32_t mx4_pack8(const float *v, float inv)
{
    float t[8];
#pragma unroll
    for (int i = 0; i < 8; i++)
        t[i] = v[i] * inv;
    return mx4_pack8(t);
}

// The larger of two magnitudes; a NaN is larger than all.
__device__ __forceinline__ float mx4_larger(float a, float b)
{
    float m;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
    return m;
}

__device__ __forceinline__ float mx4_largest(float a, float b, float c)
{
    float m;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(a), "f"(b), "f"(c));
    return m;
}

// The bits of the largest magnitude among eight values.
__device__ __forceinline__ uint32_t mx4_top8(const float *v)
{
    const float a = mx4_largest(fabsf(v[0]), fabsf(v[1]), fabsf(v[2])), b = mx4_largest(fabsf(v[3]), fabsf(v[4]), fabsf(v[5]));
    return __float_as_uint(mx4_larger(mx4_largest(a, b, fabsf(v[6])), fabsf(v[7])));
}

// Eight consecutive floats of which `left` exist; zeros for the others.  VEC: all eight or none, at a 16-byte boundary.
template <typename T, bool VEC> __device__ __forceinline__ void load8(const T *p, int left, float *v)
{
    if (VEC) {
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
        if (left > 0) {
            if (sizeof(T) == 2) {
                const uint4 u = *reinterpret_cast<const uint4 *>(p);
                a = make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16),
                                __uint_as_float(u.y & 0xffff0000u));
                b = make_float4(__uint_as_float(u.z << 16), __uint_as_float(u.z & 0xffff0000u), __uint_as_float(u.w << 16),
                                __uint_as_float(u.w & 0xffff0000u));
            } else {
                a = load4(p);
                b = load4(p + 4);
            }
        }
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
        v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++)
            v[i] = i < left ? to_f(p[i]) : 0.0f;
    }
}

// A warp packs a chunk of 256 values, eight to a lane (zeros past the row's end): the lane's codes, and its block's scale's
// code, which the four lanes of a block share.
__device__ __forceinline__ uint32_t mx4_pack_chunk(const float *v, uint32_t &code)
{
    uint32_t top = mx4_top8(v);
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    code = mx4_scale_code(top);
    return mx4_pack8(v, mx4_inverse(code));
}

// Sixteen values of a lane, half a block: two words of codes, and the block's scale's code, which two lanes share.
__device__ __forceinline__ uint2 mx4_pack16(const float *v, uint32_t &code)
{
    uint32_t top = max(mx4_top8(v), mx4_top8(v + 8));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    code = mx4_scale_code(top);
    const float inv = mx4_inverse(code);
    return make_uint2(mx4_pack8(v, inv), mx4_pack8(v + 8, inv));
}

// Eight bfloat16 times a power of two (in both halves of inv), in 4 bits.
__device__ __forceinline__ uint32_t mx4_pack8(const uint4 &x, uint32_t inv)
{
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
    float v[8];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        uint32_t p;
        asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(p) : "r"(w[i]), "r"(inv));
        v[2 * i] = __uint_as_float(p << 16);
        v[2 * i + 1] = __uint_as_float(p & 0xffff0000u);
    }
    return mx4_pack8(v);
}

// The same for sixteen bfloat16 as they lie in memory: magnitudes and the products with a power of two two at a time.
__device__ __forceinline__ uint2 mx4_pack16(const uint4 *x, uint32_t &code)
{
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 2; i++)
        top = __vmaxu2(top, __vmaxu2(__vmaxu2(x[i].x & 0x7fff7fffu, x[i].y & 0x7fff7fffu),
                                     __vmaxu2(x[i].z & 0x7fff7fffu, x[i].w & 0x7fff7fffu)));
    top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top & 0xffff0000u, top << 16);
    code = mx4_scale_code(top);
    const uint32_t inv = (254u - min(code, 252u)) * 0x00800080u;
    return make_uint2(mx4_pack8(x[0], inv), mx4_pack8(x[1], inv));
}

// Sixteen values of a lane as they are packed: floats, or bfloat16 as they lie in memory; zeros past the row's end.
struct Sixteen {
    float v[16];
    __device__ __forceinline__ void load(const float *p, int left)
    {
        load8<float, true>(p, left, v);
        load8<float, true>(p + 8, left - 8, v + 8);
    }
    __device__ __forceinline__ uint2 pack(uint32_t &code) const { return mx4_pack16(v, code); }
};
struct SixteenBf16 {
    uint4 v[2];
    __device__ __forceinline__ void load(const bf16 *p, int left)
    {
        const uint4 *q = reinterpret_cast<const uint4 *>(p);
        v[0] = left > 0 ? q[0] : make_uint4(0, 0, 0, 0);
        v[1] = left > 8 ? q[1] : make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ uint2 pack(uint32_t &code) const { return mx4_pack16(v, code); }
};

// A lane's four values of a block that eight lanes share, in 16 bits, and the block's scale's code.
__device__ __forceinline__ uint32_t mx4_pack4(const float4 &x, uint32_t &code)
{
    float t = mx4_larger(mx4_larger(fabsf(x.x), fabsf(x.y)), mx4_larger(fabsf(x.z), fabsf(x.w)));
    uint32_t top = __float_as_uint(t);
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 4));
    code = mx4_scale_code(top);
    const float inv = mx4_inverse(code);
    uint32_t r;
    asm("{\n\t"
        ".reg .b8 a, b;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
        "mov.b32 %0, {a, b, a, b};\n\t"
        "}\n"
        : "=r"(r)
        : "f"(x.x * inv), "f"(x.y * inv), "f"(x.z * inv), "f"(x.w * inv));
    return r;
}

// Packed values to memory: chunk c of row r.
__device__ __forceinline__ void mx4_store_chunk(uint32_t packed, uint32_t code, size_t r, int c, int k,
                                                uint8_t *__restrict__ codes, uint8_t *__restrict__ scales)
{
    const int lane = threadIdx.x & 31;
    const size_t row_bytes = mx4_row_bytes(k), at = (size_t)c * (MX4_CHUNK / 2) + lane * 4;
    if (at < row_bytes)
        *reinterpret_cast<uint32_t *>(codes + r * row_bytes + at) = packed;
    if ((lane & 3) == 0)
        scales[mx4_scale_at(r, c, mx4_chunks(k), lane >> 4) + ((lane >> 2) & 3)] = (uint8_t)code;
}

// The numbers that the 8 codes of a word stand for.
__device__ __forceinline__ void mx4_unpack8(uint32_t word, float *v)
{
    uint32_t h[4];
    asm("{\n\t"
        ".reg .b8 a, b, c, d;\n\t"
        "mov.b32 {a, b, c, d}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, a;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, b;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, c;\n\t"
        "cvt.rn.f16x2.e2m1x2 %3, d;\n\t"
        "}\n"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
        : "r"(word));
#pragma unroll
    for (int i = 0; i < 4; i++) {
        asm("{\n\t"
            ".reg .b16 lo, hi;\n\t"
            "mov.b32 {lo, hi}, %2;\n\t"
            "cvt.f32.f16 %0, lo;\n\t"
            "cvt.f32.f16 %1, hi;\n\t"
            "}\n"
            : "=f"(v[2 * i]), "=f"(v[2 * i + 1])
            : "r"(h[i]));
    }
}

}  // namespace jb
