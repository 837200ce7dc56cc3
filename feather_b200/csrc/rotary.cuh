// Rotary positions: the first R of a head's D elements are R/2 pairs (a, b), and pair i of a
// token at position p is turned by the angle p * inv_freq[i]:
//
//   (a, b) -> scale * (a cos - b sin, a sin + b cos)
//
// half layout: a = x[i], b = x[i + R/2]; interleaved: a = x[2i], b = x[2i + 1]; elements from
// R on pass through.  The result has the input's type, or is packed to FP8 codes in the
// packer's rounding (fp8_codec.cuh), one head after the other -- which is what the packed
// attention takes, a head's (tokens, D) codes in one piece.  No counterpart in the reference.
//
// Angles: far into a context p * inv_freq has lost its fraction in FP32 (at p = 10^6 one ulp is
// 1/16 of a radian), so the product and its reduction to a fraction of a turn are done in
// 64 bits; the remaining angle, below half a turn, takes FP32 sine and cosine (absolute error
// about 1e-7).  The angles of a token are computed once and shared by its heads.
//
// Bound by HBM for prompts (every element is read and written once): 8192 x 32 x 128 FP16, half of
// each head interleaved, 23.1 us = 5.8 TB/s.  By latency for a token: 1 x 36 x 64 takes 1.9 us.
#pragma once
#include "mxfp4_codec.cuh"

namespace feather {

constexpr int kRotThreads = 256;
constexpr int kRotMaxPairs = 512;    // R <= 1024
constexpr int kRotAngles = 2048;     // of a CTA's tokens, in shared memory
constexpr int kRotTile = 8;          // tokens of a CTA, at most
constexpr int kRotBatch = 4;         // of them in flight per thread

__device__ __forceinline__ float2 rotary_turn(double position, double inv_freq) {
    const double turns = position * inv_freq * 0.15915494309189533577;   // 1 / (2 pi)
    const float part = (float)(turns - rint(turns));                     // [-1/2, 1/2]
    float s, c;
    sincospif(2.0f * part, &s, &c);
    return make_float2(c, s);
}

// V consecutive elements as loaded, and widened: what waits for its turn takes few registers.
template <int T, int V>
struct RotaryRaw {
    static constexpr int kBytes = V * (int)sizeof(typename MxElem<T>::type);   // 16, 8, or one element's
    uint32_t w[kBytes < 4 ? 1 : kBytes / 4];
    __device__ __forceinline__ void load(const typename MxElem<T>::type* p) {
        if constexpr (kBytes == 16) {
            const uint4 a = *reinterpret_cast<const uint4*>(p);
            w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
        } else if constexpr (kBytes == 8) {
            const uint2 a = *reinterpret_cast<const uint2*>(p);
            w[0] = a.x; w[1] = a.y;
        } else if constexpr (T == kSrcF32) {
            w[0] = __float_as_uint(*p);
        } else {
            w[0] = *p;
        }
    }
    __device__ __forceinline__ void widen(float (&x)[V]) const {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            if constexpr (T == kSrcF32) x[i] = __uint_as_float(w[i]);
            else x[i] = MxElem<T>::get((unsigned short)(w[i / 2] >> (16 * (i & 1))));
        }
    }
};

// Eight (four) values to FP8 codes.  Inside the format's finite range the conversion instruction
// rounds as the packer does (to nearest even, subnormals kept); it saturates where the packer
// overflows, so a vector with a larger value or a NaN takes the packer's arithmetic.  Measured at
// 8192 x 32 x 128 FP16 to E5M2: 34.5 us with the packer's integer arithmetic throughout, 28.0 us so (with
// the vectors dealt as below 25.9 in the half layout, 21.8 interleaved).
template <int MODE, int V>
__device__ __forceinline__ void rotary_encode(const float (&y)[V], uint32_t (&w)[V / 4]) {
    uint32_t top = 0u;
#pragma unroll
    for (int i = 0; i < V; ++i) top = max(top, __float_as_uint(y[i]) & 0x7FFFFFFFu);
    if (top <= (MODE == kE5M2 ? 0x47600000u : 0x43E00000u)) {      // 57344, 448: the largest codes
#pragma unroll
        for (int i = 0; i < V / 4; ++i) {
            if constexpr (MODE == kE5M2)
                asm("{ .reg .b16 a, b;\n  cvt.rn.satfinite.e5m2x2.f32 a, %2, %1;\n  cvt.rn.satfinite.e5m2x2.f32 b, %4, %3;\n"
                    "  mov.b32 %0, {a, b}; }" : "=r"(w[i]) : "f"(y[4 * i]), "f"(y[4 * i + 1]), "f"(y[4 * i + 2]), "f"(y[4 * i + 3]));
            else
                asm("{ .reg .b16 a, b;\n  cvt.rn.satfinite.e4m3x2.f32 a, %2, %1;\n  cvt.rn.satfinite.e4m3x2.f32 b, %4, %3;\n"
                    "  mov.b32 %0, {a, b}; }" : "=r"(w[i]) : "f"(y[4 * i]), "f"(y[4 * i + 1]), "f"(y[4 * i + 2]), "f"(y[4 * i + 3]));
        }
    } else {
#pragma unroll
        for (int i = 0; i < V / 4; ++i)
            w[i] = encode_f32<MODE>(y[4 * i]) | (encode_f32<MODE>(y[4 * i + 1]) << 8) |
                   (encode_f32<MODE>(y[4 * i + 2]) << 16) | (encode_f32<MODE>(y[4 * i + 3]) << 24);
    }
}

// V consecutive results at element `at`: in the input's type (MODE < 0) or as FP8 codes.
template <int T, int MODE, int V>
__device__ __forceinline__ void rotary_store(void* out, long long at, const float (&y)[V]) {
    if constexpr (MODE >= 0) {
        unsigned char* p = reinterpret_cast<unsigned char*>(out) + at;
        if constexpr (V == 1) {
            *p = (unsigned char)encode_f32<MODE>(y[0]);
        } else {
            uint32_t w[V / 4];
            rotary_encode<MODE, V>(y, w);
            if constexpr (V == 8) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
            else *reinterpret_cast<uint32_t*>(p) = w[0];
        }
    } else {
        typename MxElem<T>::type* p = reinterpret_cast<typename MxElem<T>::type*>(out) + at;
        if constexpr (V == 1) *p = MxElem<T>::put(y[0]);
        else if constexpr (T == kSrcF32) *reinterpret_cast<float4*>(p) = make_float4(y[0], y[1], y[2], y[3]);
        else if constexpr (V == 4) *reinterpret_cast<uint2*>(p) = make_uint2(mx_put2<T>(y[0], y[1]), mx_put2<T>(y[2], y[3]));
        else *reinterpret_cast<uint4*>(p) = make_uint4(mx_put2<T>(y[0], y[1]), mx_put2<T>(y[2], y[3]),
                                                       mx_put2<T>(y[4], y[5]), mx_put2<T>(y[6], y[7]));
    }
}

struct RotaryArgs {
    const void* x;
    const void* positions;      // int32 or int64, one per token
    const double* inv_freq;     // R / 2
    void* out;
    long long tokens, token_stride, head_stride;   // strides of x in elements
    int heads, dim, rotated, wide_positions, interleaved;
    int tile, items_each;       // tokens, and items of each, per CTA
    float scale;
};

// A CTA takes `tile` consecutive tokens (blockIdx.x) and a share of their heads (blockIdx.y): first the
// tile's angles, then, without another barrier, items of two V-element vectors -- a pair of vectors
// that turn into each other, or 2 V elements that pass through -- kRotBatch tokens of an item in
// flight per thread.  V = 16 bytes of the input type
// where sizes, strides and addresses allow, else (16-bit types) 8 bytes, else 1.
template <int T, int MODE, int V>
__global__ void __launch_bounds__(kRotThreads, 4)
rotary_kernel(const RotaryArgs a) {
    typedef typename MxElem<T>::type E;
    __shared__ float2 turns[kRotAngles];
    in_turn();
    const int half = a.rotated / 2;
    const int turned = half / V;                                   // items of a head that turn
    const int still = (a.dim - a.rotated + 2 * V - 1) / (2 * V);   // items that pass through
    const int items = turned + still;
    const long long t0 = (long long)blockIdx.x * a.tile;
    const int n = (int)min((long long)a.tile, a.tokens - t0);
    for (int i = threadIdx.x; i < n * half; i += kRotThreads) {
        const int tok = i / half, p = i - tok * half;
        const double at = a.wide_positions ? (double)reinterpret_cast<const long long*>(a.positions)[t0 + tok]
                                           : (double)reinterpret_cast<const int*>(a.positions)[t0 + tok];
        float2 cs = rotary_turn(at, a.inv_freq[p]);
        cs.x *= a.scale;
        cs.y *= a.scale;
        turns[i] = cs;
    }
    __syncthreads();
    const int j_end = min(((int)blockIdx.y + 1) * a.items_each, a.heads * items);
    for (int j = (int)blockIdx.y * a.items_each + (int)threadIdx.x; j < j_end; j += kRotThreads) {
        const int h = j / items, k = j - h * items;
        // The two vectors' first elements: neighbouring items take neighbouring vectors, whether a
        // vector's pairs are in it (interleaved; one pair per item where V is 1) or in the other one.
        int at_u, at_v;
        if (k >= turned) {
            at_u = a.rotated + (k - turned) * V;
            at_v = at_u + still * V;
        } else if (V == 1 && a.interleaved) {
            at_u = 2 * k;
            at_v = at_u + 1;
        } else {
            at_u = k * V;
            at_v = at_u + half;
        }
        const bool two = at_v < a.dim;
        const E* x = reinterpret_cast<const E*>(a.x) + t0 * a.token_stride + h * a.head_stride;
        const long long step = MODE >= 0 ? a.dim : (long long)a.heads * a.dim;
        const long long o = MODE >= 0 ? ((long long)h * a.tokens + t0) * a.dim : (t0 * a.heads + h) * a.dim;
        for (int tok = 0; tok < n; tok += kRotBatch) {
            // (loaded ahead of the angles, the first batch spilled: 37 us at 8192 x 32 x 128 FP16 against 27.6)
            RotaryRaw<T, V> ru[kRotBatch], rv[kRotBatch];
#pragma unroll
            for (int b = 0; b < kRotBatch; ++b) {
                const E* from = x + (long long)min(tok + b, n - 1) * a.token_stride;
                ru[b].load(from + at_u);
                rv[b].load(from + (two ? at_v : at_u));
            }
#pragma unroll
            for (int b = 0; b < kRotBatch; ++b) {
                if (tok + b >= n) break;
                float u[V], v[V];
                ru[b].widen(u);
                rv[b].widen(v);
                if (k < turned) {
                    const float2* turn = turns + (tok + b) * half + (a.interleaved && V > 1 ? k * V / 2 : k * V);
                    if (!a.interleaved || V == 1) {
#pragma unroll
                        for (int e = 0; e < V; ++e) {
                            const float2 cs = turn[e];
                            const float p0 = u[e], p1 = v[e];
                            u[e] = p0 * cs.x - p1 * cs.y;
                            v[e] = p0 * cs.y + p1 * cs.x;
                        }
                    } else if constexpr (V > 1) {
#pragma unroll
                        for (int e = 0; e < V; e += 2) {
                            const float2 c0 = turn[e / 2], c1 = turn[half / 2 + e / 2];
                            const float p0 = u[e], p1 = u[e + 1], q0 = v[e], q1 = v[e + 1];
                            u[e] = p0 * c0.x - p1 * c0.y;
                            u[e + 1] = p0 * c0.y + p1 * c0.x;
                            v[e] = q0 * c1.x - q1 * c1.y;
                            v[e + 1] = q0 * c1.y + q1 * c1.x;
                        }
                    }
                }
                const long long to = o + (tok + b) * step;
                rotary_store<T, MODE, V>(a.out, to + at_u, u);
                if (two) rotary_store<T, MODE, V>(a.out, to + at_v, v);
            }
        }
    }
}

}  // namespace feather
