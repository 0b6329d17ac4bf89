// Microscaled 4-bit floating point (MXFP4): quantisation and its inverse.
//
// A block is 32 consecutive values along the last axis sharing one E8M0 scale
// byte b (2^(b - 127)); a value is an E2M1 code (sign, 2 exponent bits, 1
// mantissa bit: 0, .5, 1, 1.5, 2, 3, 4, 6), two codes per byte, the even
// element in the low nibble.  With m = max |x| of the block
//   b = max(floor(log2 m) - 2 + 127, 0),   code = rne_e2m1(x * 2^(127 - b)), |code| <= 6,
// so the largest value lands in [4, 8) and saturates at 6.  A block holding an
// infinity or NaN gets b = 255 (NaN), which reads back as NaN throughout.
#include <cuda_fp16.h>

#include "pdx_common.cuh"

namespace pdx {

constexpr int kMxBlock = 32;
constexpr int kMxThreads = 256;

__device__ __forceinline__ float mx_scale(uint32_t b) {  // 2^(b - 127); 255 = NaN
    return __uint_as_float(b == 255u ? 0x7FC00000u : (b ? b << 23 : 0x00400000u));
}

// Eight floats -> eight E2M1 codes, element 0 in the lowest nibble (round to
// nearest even, saturating).
__device__ __forceinline__ uint32_t e2m1x8(const float* v) {
    uint32_t r;
    asm("{\n\t.reg .b8 c0, c1, c2, c3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c0, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c1, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c2, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c3, %8, %7;\n\t"
        "mov.b32 %0, {c0, c1, c2, c3};\n\t}"
        : "=r"(r)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return r;
}

// Eight E2M1 codes -> floats (exact).
__device__ __forceinline__ void e2m1x8_to_float(uint32_t codes, float* v) {
    uint32_t h[4];
    asm("{\n\t.reg .b8 c0, c1, c2, c3;\n\t"
        "mov.b32 {c0, c1, c2, c3}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, c0;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, c1;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, c2;\n\t"
        "cvt.rn.f16x2.e2m1x2 %3, c3;\n\t}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
        : "r"(codes));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}

template <typename T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_float<bf16>(bf16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ bf16 from_float<bf16>(float v) { return __float2bfloat16_rn(v); }

// Eight values of type T at p, 16-byte accesses where ALIGNED.
template <typename T, bool ALIGNED>
__device__ __forceinline__ void load8(const T* p, float* v) {
    alignas(16) T t[8];
    if (ALIGNED) {
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i)
            reinterpret_cast<uint4*>(t)[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) t[i] = p[i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_float<T>(t[i]);
}

template <typename T, bool ALIGNED>
__device__ __forceinline__ void store8(T* p, const float* v) {
    alignas(16) T t[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = from_float<T>(v[i]);
    if (ALIGNED) {
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i)
            reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(t)[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = t[i];
    }
}

// Both kernels are copies with a conversion: HBM-bound.  98,304 x 2048: BF16 to
// MXFP4 96 us (5.3 TB/s), back 78 us (6.5 TB/s); half as much FP32 to MXFP4 65 us
// (7.0 TB/s).  A thread takes a few pieces of eight values, a CTA's threads
// neighbouring pieces, and issues all its loads before converting (quantising: 2
// pieces 96 us, 4 pieces 112, 1 piece 109; back: 4 pieces 78, 2 pieces 80, 1 piece
// 105).  FLAT: rows without gaps, so a piece's place needs no division by the row
// length.
constexpr int kMxUnroll = 2, kMxUnrollBack = 4;

template <bool FLAT>
__device__ __forceinline__ int64_t mx_at(int64_t c, int64_t per_row, int64_t ld) {
    if (FLAT) return c * 8;
    const int64_t row = c / per_row;
    return row * ld + (c - row * per_row) * 8;
}

// Four lanes per block, eight values each.  rows x cols values with row stride
// ld (elements), cols / 8 = per_row; codes and scales dense.  chunks is a
// multiple of 4, so the four lanes of a block are in range together.
template <typename T, bool ALIGNED, bool FLAT>
__global__ void __launch_bounds__(kMxThreads) k_mx4_quantize(const T* __restrict__ x, int64_t chunks, int64_t per_row,
                                                             int64_t ld, uint32_t* __restrict__ codes,
                                                             uint8_t* __restrict__ scales) {
    griddep_wait();
    griddep_launch();
    const int64_t c0 = static_cast<int64_t>(blockIdx.x) * (kMxThreads * kMxUnroll) + threadIdx.x;
    float v[kMxUnroll][8];
#pragma unroll
    for (int j = 0; j < kMxUnroll; ++j) {
        const int64_t c = c0 + j * kMxThreads;
        if (c < chunks) load8<T, ALIGNED>(x + mx_at<FLAT>(c, per_row, ld), v[j]);
    }
#pragma unroll
    for (int j = 0; j < kMxUnroll; ++j) {
        const int64_t c = c0 + j * kMxThreads;
        if (c >= chunks) return;
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[j][i]) & 0x7FFFFFFFu);
        const uint32_t mask = 0xFu << (lane_id() & 28u);
        m = max(m, __shfl_xor_sync(mask, m, 1));
        m = max(m, __shfl_xor_sync(mask, m, 2));
        const uint32_t exp = m >> 23;
        const uint32_t b = exp == 255u ? 255u : (exp > 2u ? exp - 2u : 0u);
        const float inv = __uint_as_float((254u - min(b, 254u)) << 23);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[j][i] *= inv;
        codes[c] = b == 255u ? 0u : e2m1x8(v[j]);
        if ((c & 3) == 0) scales[c >> 2] = static_cast<uint8_t>(b);
    }
}

template <typename T, bool ALIGNED, bool FLAT>
__global__ void __launch_bounds__(kMxThreads) k_mx4_dequantize(const uint32_t* __restrict__ codes,
                                                               const uint8_t* __restrict__ scales, int64_t chunks,
                                                               int64_t per_row, int64_t ld, T* __restrict__ out) {
    griddep_wait();
    griddep_launch();
    const int64_t c0 = static_cast<int64_t>(blockIdx.x) * (kMxThreads * kMxUnrollBack) + threadIdx.x;
    uint32_t code[kMxUnrollBack], scale[kMxUnrollBack];
#pragma unroll
    for (int j = 0; j < kMxUnrollBack; ++j) {
        const int64_t c = c0 + j * kMxThreads;
        if (c < chunks) {
            code[j] = __ldg(codes + c);
            scale[j] = __ldg(scales + (c >> 2));
        }
    }
#pragma unroll
    for (int j = 0; j < kMxUnrollBack; ++j) {
        const int64_t c = c0 + j * kMxThreads;
        if (c >= chunks) return;
        const float s = mx_scale(scale[j]);
        float v[8];
        e2m1x8_to_float(code[j], v);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] *= s;
        store8<T, ALIGNED>(out + mx_at<FLAT>(c, per_row, ld), v);
    }
}

}  // namespace pdx
