// Microscaled 4-bit floating point: a block of 32 consecutive elements of a row holds 32 E2M1
// codes (sign, two exponent bits of bias 1, one mantissa bit: 0, .5, 1, 1.5, 2, 3, 4, 6) and
// one power-of-two scale, a byte b that stands for 2^(b - 127) (255: NaN).  No counterpart in
// the reference, whose packers stop at 8 bits (feather/packers/fp8.py).
//
// Storage: two codes to a byte, the even element in the low half; a row of n elements takes
// ceil(n / 32) blocks = 16 bytes of codes and one scale byte each, a short last block is
// filled up with zero codes.
//
// Quantising a block: b = max(E - 2, 0) with E the FP32 exponent field of max |x| (the largest
// element then lies in [4, 8) scales, above 6 it saturates), codes = round to nearest even of
// x 2^(127 - b), which FP32 multiplies exactly wherever the code is not zero.  A block with an
// infinity or a NaN has no such scale: its byte is 255 and its codes are 0, so it decodes to NaN.
#pragma once
#include <cuda_bf16.h>

#include "fp8_codec.cuh"

namespace feather {

constexpr int kMxBlock = 32;

enum : int { kSrcF16 = 0, kSrcF32 = 1, kSrcBF16 = 2, kSrcMxfp4 = 3 };

template <int T> struct MxElem;
template <> struct MxElem<kSrcF16> {
    typedef unsigned short type;
    static __device__ __forceinline__ float get(unsigned short x) { return __half2float(__ushort_as_half(x)); }
    static __device__ __forceinline__ unsigned short put(float x) { return __half_as_ushort(__float2half_rn(x)); }
};
template <> struct MxElem<kSrcBF16> {
    typedef unsigned short type;
    static __device__ __forceinline__ float get(unsigned short x) { return __uint_as_float((uint32_t)x << 16); }
    static __device__ __forceinline__ unsigned short put(float x) { return __bfloat16_as_ushort(__float2bfloat16_rn(x)); }
};
template <> struct MxElem<kSrcF32> {
    typedef float type;
    static __device__ __forceinline__ float get(float x) { return x; }
    static __device__ __forceinline__ float put(float x) { return x; }
};

// Scale byte of a block whose largest |x| has this FP32 bit pattern (sign cleared).
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t amax_bits) {
    const int e = (int)(amax_bits >> 23);
    return e == 255 ? 255u : (uint32_t)max(e - 2, 0);
}
// 2^(127 - b), the factor that takes the block's values to the grid of the codes; 0 for b = 255.
__device__ __forceinline__ float mx_to_grid(uint32_t b) {
    return __uint_as_float(b == 255u ? 0u : (254u - b) << 23);
}
// 2^(b - 127), NaN for b = 255, exact at b = 0 too (2^-127 is an FP32 subnormal).
__device__ __forceinline__ float mx_scale_value(uint32_t b) {
    const uint32_t bits = b == 0u ? 0x00400000u : b << 23;
    return __uint_as_float(b == 255u ? 0x7FC00000u : bits);
}
// Eight values on the grid to eight codes, element 0 in the low four bits (round to nearest
// even, saturating: the conversion instruction's own definition).
__device__ __forceinline__ uint32_t mx_encode8(const float (&y)[8]) {
    uint32_t w;
    asm("{ .reg .b8 a, b, c, d;\n"
        "  cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n"
        "  cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n"
        "  cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n"
        "  cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n"
        "  mov.b32 %0, {a, b, c, d}; }"
        : "=r"(w)
        : "f"(y[0]), "f"(y[1]), "f"(y[2]), "f"(y[3]), "f"(y[4]), "f"(y[5]), "f"(y[6]), "f"(y[7]));
    return w;
}
// Eight codes to four FP16 pairs in element order; every code is an FP16 number.
__device__ __forceinline__ void mx_decode8(uint32_t w, uint32_t (&h)[4]) {
    asm("{ .reg .b8 a, b, c, d;\n"
        "  mov.b32 {a, b, c, d}, %4;\n"
        "  cvt.rn.f16x2.e2m1x2 %0, a;\n"
        "  cvt.rn.f16x2.e2m1x2 %1, b;\n"
        "  cvt.rn.f16x2.e2m1x2 %2, c;\n"
        "  cvt.rn.f16x2.e2m1x2 %3, d; }"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
        : "r"(w));
}

// First thing in a kernel launched ahead of its turn (programmatic stream serialisation): lets
// the next kernel do the same, and waits for the one in front before memory is touched.
__device__ __forceinline__ void in_turn() {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
}

// The largest |x| of eight values as an FP32 bit pattern, and the values.
template <int T>
__device__ __forceinline__ uint32_t mx_load8(const void* src, long long e, float (&x)[8]) {
    uint32_t top = 0u;
    if constexpr (T == kSrcF32) {
        const float4* p = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(src) + e);
        const float4 a = __ldcs(p), b = __ldcs(p + 1);
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
        x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
#pragma unroll
        for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7FFFFFFFu);
    } else {
        const uint4 w = __ldcs(reinterpret_cast<const uint4*>(reinterpret_cast<const unsigned short*>(src) + e));
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
        uint32_t m = 0u;   // the larger of each half: 16-bit magnitudes order like the values
#pragma unroll
        for (int i = 0; i < 4; ++i) m = __vmaxu2(m, u[i] & 0x7FFF7FFFu);
        const uint32_t h = max(m & 0xFFFFu, m >> 16);
        top = __float_as_uint(MxElem<T>::get((unsigned short)h));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = MxElem<T>::get((unsigned short)(u[i] & 0xFFFFu));
            x[2 * i + 1] = MxElem<T>::get((unsigned short)(u[i] >> 16));
        }
    }
    return top;
}

// ------------------------------------------------------------ quantise -----
// Rows of whole blocks, 16-byte aligned: the matrix is a flat run of blocks.  Four threads
// take a block, eight elements each (16- or 2 x 16-byte loads), and agree on the block's
// maximum with two shuffles; a warp takes kMxSteps runs of 256 elements per trip.  Bound by
// HBM: it reads every element once and writes 17/32 byte for each; 16384 x 8192 FP16 56.7 us
// (6.0 TB/s).
constexpr int kMxSteps = 4;
template <int T>
__global__ void __launch_bounds__(256)
mx_encode_kernel(const void* __restrict__ src, uint32_t* __restrict__ codes, unsigned char* __restrict__ scales,
                 long long n_words) {
    in_turn();
    const int lane = threadIdx.x & 31;
    const long long warps = ((long long)gridDim.x * blockDim.x) >> 5;
    const long long warp = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
    for (long long base = warp * (32 * kMxSteps); base < n_words; base += warps * (32 * kMxSteps)) {
        float x[kMxSteps][8];
        uint32_t top[kMxSteps];
#pragma unroll
        for (int u = 0; u < kMxSteps; ++u) {
            const long long w = base + 32 * u + lane;
            top[u] = 0u;
            if (w < n_words) {
                top[u] = mx_load8<T>(src, w * 8, x[u]);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) x[u][i] = 0.f;
            }
        }
#pragma unroll
        for (int u = 0; u < kMxSteps; ++u) {
            const long long w = base + 32 * u + lane;
            uint32_t m = top[u];
            m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, 1));
            m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, 2));
            const uint32_t b = mx_scale_byte(m);
            const float f = mx_to_grid(b);
            float y[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = x[u][i] * f;
            const uint32_t c = mx_encode8(y);
            if (w < n_words) {
                codes[w] = b == 255u ? 0u : c;
                if ((lane & 3) == 0) scales[w >> 2] = (unsigned char)b;
            }
        }
    }
}

// Any row length and alignment: the same four threads to a block, each finding its row by a division
// and loading its eight elements W bytes at a time (what the rows' alignment allows); the
// loads of a warp touch the same lines one after the other and hit in L1.  5001 x 2050 FP16 10.8
// us; a warp per block with one element per lane took 26.7 (three quarters of it instructions).
template <int T, int W>
__global__ void __launch_bounds__(256)
mx_encode_rows_kernel(const typename MxElem<T>::type* __restrict__ src, uint32_t* __restrict__ codes,
                      unsigned char* __restrict__ scales, long long n_words, long long cols, uint32_t words_row) {
    in_turn();
    const int lane = threadIdx.x & 31;
    const long long warps = ((long long)gridDim.x * blockDim.x) >> 5;
    const long long warp = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
    constexpr int kPer = W / (int)sizeof(typename MxElem<T>::type);   // elements of a load
    for (long long base = warp * (32 * kMxSteps); base < n_words; base += warps * (32 * kMxSteps)) {
        float x[kMxSteps][8];
#pragma unroll
        for (int u = 0; u < kMxSteps; ++u) {
            const long long w = min(base + 32 * u + lane, n_words - 1);
            const long long row = n_words >> 32 ? w / words_row : (uint32_t)w / words_row;
            const long long col = (w - row * words_row) * 8;
            const typename MxElem<T>::type* p = src + row * cols + col;
            if (col + 8 <= cols) {
#pragma unroll
                for (int k = 0; k < 8; k += kPer) {
                    if constexpr (kPer == 1) {
                        x[u][k] = MxElem<T>::get(p[k]);
                    } else {
                        const uint32_t pair = *reinterpret_cast<const uint32_t*>(p + k);
                        x[u][k] = MxElem<T>::get((unsigned short)(pair & 0xFFFFu));
                        x[u][k + 1] = MxElem<T>::get((unsigned short)(pair >> 16));
                    }
                }
            } else {
#pragma unroll
                for (int k = 0; k < 8; ++k) x[u][k] = col + k < cols ? MxElem<T>::get(p[k]) : 0.f;
            }
        }
#pragma unroll
        for (int u = 0; u < kMxSteps; ++u) {
            const long long w = base + 32 * u + lane;
            uint32_t m = 0u;
#pragma unroll
            for (int k = 0; k < 8; ++k) m = max(m, __float_as_uint(x[u][k]) & 0x7FFFFFFFu);
            m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, 1));
            m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, 2));
            const uint32_t b = mx_scale_byte(m);
            const float f = mx_to_grid(b);
            float y[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) y[k] = x[u][k] * f;
            const uint32_t c = mx_encode8(y);
            if (w < n_words) {
                codes[w] = b == 255u ? 0u : c;
                if ((lane & 3) == 0) scales[w >> 2] = (unsigned char)b;
            }
        }
    }
}

// ---------------------------------------------------------- dequantise -----
// value = code * scale, one rounding to the output type (none for BF16 and FP32 down to their
// subnormals: a code has two significant bits).
template <int T>
__device__ __forceinline__ uint32_t mx_put2(float lo, float hi) {
    return (uint32_t)MxElem<T>::put(lo) | ((uint32_t)MxElem<T>::put(hi) << 16);
}

// Rows of whole blocks, 16-byte aligned output.  A lane loads one word (eight codes) per
// step; for 16-bit outputs it writes its own 16 bytes, for FP32 the words change hands inside
// the warp so that each store instruction writes 512 consecutive bytes.  Bound by HBM: 8192 x
// 8192 to FP32 48.2 us (6.3 TB/s), 16384 x 8192 to BF16 55.0 (6.2).
template <int T>
__global__ void __launch_bounds__(256)
mx_decode_kernel(const uint32_t* __restrict__ codes, const unsigned char* __restrict__ scales, void* __restrict__ dst,
                 long long n_words) {
    in_turn();
    const int lane = threadIdx.x & 31;
    const long long warps = ((long long)gridDim.x * blockDim.x) >> 5;
    const long long warp = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
    for (long long base = warp * (32 * kMxSteps); base < n_words; base += warps * (32 * kMxSteps)) {
        uint32_t c[kMxSteps];
        float f[kMxSteps];
#pragma unroll
        for (int u = 0; u < kMxSteps; ++u) {
            const long long w = base + 32 * u + lane;
            c[u] = w < n_words ? __ldcs(codes + w) : 0u;
            f[u] = mx_scale_value(w < n_words ? scales[w >> 2] : 0u);
        }
#pragma unroll
        for (int u = 0; u < kMxSteps; ++u) {
            const long long w0 = base + 32 * u;
            if constexpr (T == kSrcF32) {
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int from = 16 * half + (lane >> 1);
                    const uint32_t cw = __shfl_sync(0xFFFFFFFFu, c[u], from);
                    const float fw = __shfl_sync(0xFFFFFFFFu, f[u], from);
                    uint32_t h[4];
                    mx_decode8(lane & 1 ? cw >> 16 : cw, h);
                    const float2 a = h2_to_f2(h[0]), b = h2_to_f2(h[1]);
                    if (w0 + from < n_words)
                        __stcs(reinterpret_cast<float4*>(dst) + 2 * w0 + 32 * half + lane,
                               make_float4(a.x * fw, a.y * fw, b.x * fw, b.y * fw));
                }
            } else {
                uint32_t h[4], o[4];
                mx_decode8(c[u], h);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 a = h2_to_f2(h[i]);
                    o[i] = mx_put2<T>(a.x * f[u], a.y * f[u]);
                }
                if (w0 + lane < n_words)
                    __stcs(reinterpret_cast<uint4*>(dst) + w0 + lane, make_uint4(o[0], o[1], o[2], o[3]));
            }
        }
    }
}

// Any row length and alignment: a warp takes kMxRun consecutive pairs of blocks of a row, a lane two
// consecutive elements (a byte) of each, so that its stores are consecutive; PAIRED: rows of
// an even number of 16-bit elements, stored two at a time.  5001 x 2050 to FP16 11.4 us (one element
// per lane 18.3).
constexpr int kMxRun = 4;            // as many as mx_decode8 takes
template <int T, bool PAIRED>
__global__ void __launch_bounds__(256)
mx_decode_rows_kernel(const unsigned char* __restrict__ codes, const unsigned char* __restrict__ scales,
                      typename MxElem<T>::type* __restrict__ dst, long long rows, long long cols, int blocks_row,
                      int runs_row) {
    in_turn();
    const int lane = threadIdx.x & 31;
    const long long warps = ((long long)gridDim.x * blockDim.x) >> 5, runs = rows * runs_row;
    for (long long run = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 5; run < runs; run += warps) {
        const long long row = runs >> 32 ? run / runs_row : (uint32_t)run / (uint32_t)runs_row;
        const int b0 = (int)(run - row * runs_row) * (2 * kMxRun) + (lane >> 4);
        const long long blk = row * blocks_row + b0;
        uint32_t pairs = 0u, h[4], s[kMxRun];
#pragma unroll
        for (int u = 0; u < kMxRun; ++u) {
            const bool there = b0 + 2 * u < blocks_row;
            pairs |= (there ? (uint32_t)codes[(blk + 2 * u) * 16 + (lane & 15)] : 0u) << (8 * u);
            s[u] = there ? scales[blk + 2 * u] : 0u;
        }
        mx_decode8(pairs, h);
#pragma unroll
        for (int u = 0; u < kMxRun; ++u) {
            const long long col = (long long)(b0 + 2 * u) * kMxBlock + 2 * (lane & 15);
            const float2 x = h2_to_f2(h[u]);
            const float f = mx_scale_value(s[u]);
            typename MxElem<T>::type* to = dst + row * cols + col;
            if constexpr (PAIRED) {
                if (col < cols) *reinterpret_cast<uint32_t*>(to) = mx_put2<T>(x.x * f, x.y * f);
            } else {
                if (col < cols) to[0] = MxElem<T>::put(x.x * f);
                if (col + 1 < cols) to[1] = MxElem<T>::put(x.y * f);
            }
        }
    }
}

}  // namespace feather
