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
// Bound by HBM for prompts (every element is read and written once), by latency for a token.
#pragma once
#include "mxfp4_codec.cuh"

namespace feather {

constexpr int kRotThreads = 256;
constexpr int kRotMaxPairs = 512;   // R <= 1024: the angles of a token in shared memory

__device__ __forceinline__ float2 rotary_turn(double position, double inv_freq) {
    const double turns = position * inv_freq * 0.15915494309189533577;   // 1 / (2 pi)
    const float part = (float)(turns - rint(turns));                     // [-1/2, 1/2]
    float s, c;
    sincospif(2.0f * part, &s, &c);
    return make_float2(c, s);
}

template <int T, int V>
__device__ __forceinline__ void rotary_load(const typename MxElem<T>::type* p, float (&x)[V]) {
    if constexpr (V == 1) {
        x[0] = MxElem<T>::get(*p);
    } else if constexpr (T == kSrcF32) {
        static_assert(T != kSrcF32 || V == 4 || V == 1, "16-byte accesses");
        const float4 a = *reinterpret_cast<const float4*>(p);
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    } else {
        const uint4 a = *reinterpret_cast<const uint4*>(p);
        const uint32_t u[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = MxElem<T>::get((unsigned short)(u[i] & 0xFFFFu));
            x[2 * i + 1] = MxElem<T>::get((unsigned short)(u[i] >> 16));
        }
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
#pragma unroll
            for (int i = 0; i < V / 4; ++i)
                w[i] = encode_f32<MODE>(y[4 * i]) | (encode_f32<MODE>(y[4 * i + 1]) << 8) |
                       (encode_f32<MODE>(y[4 * i + 2]) << 16) | (encode_f32<MODE>(y[4 * i + 3]) << 24);
            if constexpr (V == 8) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
            else *reinterpret_cast<uint32_t*>(p) = w[0];
        }
    } else {
        typename MxElem<T>::type* p = reinterpret_cast<typename MxElem<T>::type*>(out) + at;
        if constexpr (V == 1) {
            *p = MxElem<T>::put(y[0]);
        } else if constexpr (T == kSrcF32) {
            *reinterpret_cast<float4*>(p) = make_float4(y[0], y[1], y[2], y[3]);
        } else {
            *reinterpret_cast<uint4*>(p) = make_uint4(mx_put2<T>(y[0], y[1]), mx_put2<T>(y[2], y[3]),
                                                      mx_put2<T>(y[4], y[5]), mx_put2<T>(y[6], y[7]));
        }
    }
}

struct RotaryArgs {
    const void* x;
    const void* positions;      // int32 or int64, one per token
    const double* inv_freq;     // R / 2
    void* out;
    long long tokens, token_stride, head_stride;   // strides of x in elements
    int heads, dim, rotated, wide_positions, interleaved;
    int items_each;             // items of a token per CTA
    float scale;
};

// A CTA takes a token (blockIdx.x + k gridDim.x) and a share of its heads (blockIdx.y) at a time, in
// items of two V-element vectors: a pair of vectors that turn into each other, or 2 V elements
// that pass through; V = 16 bytes of the input type where sizes, strides and addresses allow, else
// 1.  The next token's angles are computed and its first items loaded while this one's items turn.
template <int T, int MODE, int V>
__global__ void __launch_bounds__(kRotThreads)
rotary_kernel(const RotaryArgs a) {
    typedef typename MxElem<T>::type E;
    __shared__ float2 turns[2][kRotMaxPairs];
    const int half = a.rotated / 2;
    const int turned = half / V;                                   // items of a head that turn
    const int still = (a.dim - a.rotated + 2 * V - 1) / (2 * V);   // items that pass through
    const int items = turned + still;
    const int j_begin = (int)blockIdx.y * a.items_each, j_end = min(j_begin + a.items_each, a.heads * items);
    auto angles = [&](long long t, float2* turn) {
        const double p = a.wide_positions ? (double)reinterpret_cast<const long long*>(a.positions)[t]
                                          : (double)reinterpret_cast<const int*>(a.positions)[t];
        for (int i = threadIdx.x; i < half; i += kRotThreads) {
            float2 cs = rotary_turn(p, a.inv_freq[i]);
            cs.x *= a.scale;
            cs.y *= a.scale;
            turn[i] = cs;
        }
    };
    // an item's place in its head: the two vectors' first elements, and the first pair
    auto place = [&](int k, int& at_u, int& at_v) {
        if (k < turned) {
            at_u = a.interleaved ? 2 * k * V : k * V;
            at_v = a.interleaved ? at_u + V : at_u + half;
        } else {
            at_u = a.rotated + (k - turned) * 2 * V;
            at_v = at_u + V;
        }
    };
    const int j0 = j_begin + (int)threadIdx.x, h0 = j0 / items, k0 = j0 - h0 * items;   // this thread's first item of every token
    int u0, v0;
    place(k0, u0, v0);
    float u[V], v[V];
    auto fetch = [&](long long t) {
        if (j0 >= j_end) return;
        const E* x = reinterpret_cast<const E*>(a.x) + t * a.token_stride + h0 * a.head_stride;
        rotary_load<T, V>(x + u0, u);
        if (v0 < a.dim) rotary_load<T, V>(x + v0, v);
    };
    long long t = blockIdx.x;
    if (t >= a.tokens) return;
    fetch(t);
    angles(t, turns[0]);
    __syncthreads();
    for (int buf = 0; t < a.tokens; t += gridDim.x, buf ^= 1) {
        const float2* turn = turns[buf];
        const bool more = t + gridDim.x < a.tokens;
        for (int j = j0; j < j_end; j += kRotThreads) {
            int h = h0, k = k0, at_u = u0, at_v = v0;
            if (j != j0) {
                h = j / items;
                k = j - h * items;
                place(k, at_u, at_v);
                const E* x = reinterpret_cast<const E*>(a.x) + t * a.token_stride + h * a.head_stride;
                rotary_load<T, V>(x + at_u, u);
                if (at_v < a.dim) rotary_load<T, V>(x + at_v, v);
            }
            if (k < turned) {
                const int i = k * V;
                if (!a.interleaved || V == 1) {
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        const float2 cs = turn[i + e];
                        const float p0 = u[e], p1 = v[e];
                        u[e] = p0 * cs.x - p1 * cs.y;
                        v[e] = p0 * cs.y + p1 * cs.x;
                    }
                } else if constexpr (V > 1) {
#pragma unroll
                    for (int e = 0; e < V; e += 2) {
                        const float2 c0 = turn[i + e / 2], c1 = turn[i + V / 2 + e / 2];
                        const float p0 = u[e], p1 = u[e + 1], q0 = v[e], q1 = v[e + 1];
                        u[e] = p0 * c0.x - p1 * c0.y;
                        u[e + 1] = p0 * c0.y + p1 * c0.x;
                        v[e] = q0 * c1.x - q1 * c1.y;
                        v[e + 1] = q0 * c1.y + q1 * c1.x;
                    }
                }
            }
            const long long o = MODE >= 0 ? ((long long)h * a.tokens + t) * a.dim : (t * a.heads + h) * a.dim;
            rotary_store<T, MODE, V>(a.out, o + at_u, u);
            if (at_v < a.dim) rotary_store<T, MODE, V>(a.out, o + at_v, v);
        }
        if (more) {
            fetch(t + gridDim.x);
            angles(t + gridDim.x, turns[buf ^ 1]);
        }
        __syncthreads();
    }
}

}  // namespace feather
