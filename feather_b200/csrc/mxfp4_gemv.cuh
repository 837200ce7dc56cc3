// Microscaled 4-bit matrix times up to eight vectors:
//
//   out[b][r] = sum_j value(m[r][j]) * v[b][j]        FP32 accumulation
//
// value() as in mxfp4_codec.cuh; a vector is FP16, BF16 or FP32, or packed like the matrix.
// No counterpart in the reference (its GEMV multiplies packed FP8, feather/routines/gemv.py).
//
// The bytes (17/32 per element) want 44 codes per clock and SM at the HBM rate.  A decode and
// an FMA for each on the FP32 pipe is more than an SM issues, so the products go through
// mma.sync m16n8k16 (FP16 operands, FP32 accumulator): a code is an FP16 number, and the
// vector is brought to FP16 block by block.
//
// Block-diagonal B.  The scales differ from row to row and block to block, so the sums of
// different blocks must not meet before they are scaled.  A lane loads 16 bytes of a row: one
// whole block.  The four lanes of a row hold four neighbouring blocks, and a product adds
// over all four -- but it has eight columns: column 2 t and 2 t + 1 hold the vector for lane
// t's block and zeros for the other three lanes' slots.  The accumulator that lane t gets
// back for its row is then the sum of ITS block alone, so it multiplies it with its own scale,
// and nothing moves between lanes until the row's end.  The two columns per block hold the
// two halves of an FP32 vector, or two vectors.
//
// The vector.  A block is scaled by a power of two so that its largest finite element lies in
// [2^14, 2^15), and rounded to FP16: FP16, BF16 and packed values are exact (elements 2^-39 of
// the block's largest and below lose bits that an FP32 sum would not keep either); FP32
// values are split in two, x = hi + lo, each rounded to nearest, which leaves an error of at
// most 2^-24 of the element -- one FP32 rounding.  The block sum (FP32) is multiplied by
// the vector block's power of two and then, in an FMA, by the matrix block's.
//
// Work split.  A CTA per SM owns a range of 16-row groups; its 16 warps split the row's tiles of
// 128 codes (and, for short rows, the groups): a warp keeps its range of columns for all
// groups and leaves a partial sum per row in shared memory, so there is no barrier until
// the CTA's rows are done; then the partials are added in warp order (same bits every run).
// Loads go to registers, kMgDepth tiles of two groups ahead.
#pragma once
#include "gemv_common.cuh"
#include "mxfp4_codec.cuh"

namespace feather {

constexpr int kMgWarps = 16;
constexpr int kMgThreads = kMgWarps * 32;
constexpr int kMgTile = 128;                    // codes of a row per tile: four lanes x one block
constexpr int kMgPartFloats = 12288;            // partial sums held in shared memory
constexpr int kMgVecHalfs = 49152;              // vector columns held in shared memory, all of them together

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                        uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

struct MxGemvArgs {
    const unsigned char* codes;
    const unsigned char* scales;
    const void* v;                   // nv vectors, N elements (or packed rows) apart
    const unsigned char* v_scales;   // packed vectors only
    float* out;                      // nv x M
    long long M, N;
    int blocks;                      // per row
    int nv;                          // vectors of this launch
    int chunk_blocks;                // blocks of the vector in shared memory at a time, a multiple of 4
    int slots;                       // tasks whose partial sums fit
    int col_warps;                   // warps that split a row's columns: a power of two, at most the first chunk's tiles
};

// Layout of dynamic shared memory: columns of halfs [2 P][chunk + 8], block scales
// [nv][chunk_blocks], 64 bytes of zeros, partial sums.
template <int P>
__host__ __device__ constexpr int mg_column(int chunk_blocks) { return chunk_blocks * kMxBlock + 8; }
template <int P>
__host__ __device__ constexpr int mg_smem_bytes(int chunk_blocks, int nv) {
    return 2 * P * mg_column<P>(chunk_blocks) * 2 + 4 * nv * chunk_blocks + 64 + 4 * kMgPartFloats;
}

// VT: type of the vector (kSrc...); P: pairs of columns, 2 P columns in all; R: 16-row groups
// a warp multiplies with the same vector registers.
template <int VT, int P, int R>
__global__ void __launch_bounds__(kMgThreads, 1)
mx_gemv_kernel(const MxGemvArgs a) {
    constexpr int kParts = VT == kSrcF32 ? 2 : 1;      // columns per vector
    constexpr int kAcc = P * (kParts == 2 ? 1 : 2);    // vectors a launch can take
    constexpr int kBuf = 3;                            // tiles in flight
    extern __shared__ __align__(16) unsigned char mg_smem[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int column = mg_column<P>(a.chunk_blocks);
    __half* vec = reinterpret_cast<__half*>(mg_smem);
    float* vscale = reinterpret_cast<float*>(mg_smem + 2 * P * column * 2);
    unsigned char* zeros = mg_smem + 2 * P * column * 2 + 4 * a.nv * a.chunk_blocks;
    float* part = reinterpret_cast<float*>(zeros + 64);

    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");

    const long long groups = (a.M + 15) / 16;
    const long long g_begin = groups * blockIdx.x / gridDim.x, g_end = groups * (blockIdx.x + 1) / gridDim.x;
    const int my_groups = (int)(g_end - g_begin);
    const int tasks = (my_groups + R - 1) / R;
    const long long row_bytes = (long long)a.blocks * 16;
    if (tid < 16) reinterpret_cast<uint32_t*>(zeros)[tid] = 0u;

    const int chunks = (a.blocks + a.chunk_blocks - 1) / a.chunk_blocks;
    // warps over columns (wk of them) and tasks (wr of them)
    const int wk = a.col_warps, wr = kMgWarps / wk, my_k = warp & (wk - 1), my_r = warp / wk;
    for (int first = 0; first < tasks; first += a.slots) {
        const int n_tasks = min(a.slots, tasks - first);
        for (int ch = 0; ch < chunks; ++ch) {
            const int blk0 = ch * a.chunk_blocks, n_blk = min(a.chunk_blocks, a.blocks - blk0);
            const int tiles = (n_blk + 3) / 4;
            const int tile_begin = tiles * my_k / wk, my_tiles = tiles * (my_k + 1) / wk - tile_begin;
            const int my_tasks = my_r < n_tasks ? (n_tasks - my_r + wr - 1) / wr : 0;
            const int steps = my_tasks * my_tiles;

            // the matrix loads: tile `step` of this warp's walk (its tasks, inside them its tiles)
            uint4 m[kBuf][R][2];
            uint32_t s[kBuf][R][2];
            int l_tile = 0, l_task = my_r;
            auto load = [&](int buf) {
                const int blk = blk0 + (tile_begin + l_tile) * 4 + t;
                const bool in_row = blk < blk0 + n_blk;
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const int grp = (first + l_task) * R + r;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const long long row = (g_begin + grp) * 16 + g + 8 * h;
                        const bool ok = in_row && grp < my_groups && row < a.M;
                        m[buf][r][h] = make_uint4(0u, 0u, 0u, 0u);
                        s[buf][r][h] = 0u;
                        if (ok) {
                            m[buf][r][h] = ldg_stream(reinterpret_cast<const uint4*>(a.codes + row * row_bytes) + blk);
                            s[buf][r][h] = __ldg(a.scales + row * a.blocks + blk);
                        }
                    }
                }
                if (++l_tile == my_tiles) l_tile = 0, l_task += wr;
            };
#pragma unroll
            for (int i = 0; i < kBuf - 1; ++i)
                if (i < steps) load(i);

            // the vector chunk: four threads per block, eight elements each
            if (ch > 0 || first > 0 ? chunks > 1 : true) {
                if (ch > 0 || first > 0) __syncthreads();   // the previous chunk's readers are done
                const int pad_blk = tiles * 4;
                const int quads = a.nv * pad_blk;
                for (int i0 = warp * 32; i0 < quads * 4; i0 += kMgThreads) {   // whole warps: the lanes shuffle
                    const int i = i0 + lane, q = i & 3, b = (i >> 2) % pad_blk;
                    const bool mine = (i >> 2) < quads;
                    const int n = mine ? (i >> 2) / pad_blk : 0;
                    const long long e0 = (long long)(blk0 + b) * kMxBlock + q * 8;
                    float x[8];
                    uint32_t hi[4] = {0u, 0u, 0u, 0u}, lo[4] = {0u, 0u, 0u, 0u};
                    float sv = 1.f;
                    if constexpr (VT == kSrcMxfp4) {
                        if (b < n_blk) {
                            const long long at = (long long)n * a.blocks + blk0 + b;
                            mx_decode8(__ldg(reinterpret_cast<const uint32_t*>(a.v) + at * 4 + q), hi);
                            sv = mx_scale_value(__ldg(a.v_scales + at));
                        }
                    } else {
                        typedef typename MxElem<VT>::type E;
                        const E* p = reinterpret_cast<const E*>(a.v) + (long long)n * a.N + e0;
                        uint32_t top = 0u;
                        if (e0 + 8 <= a.N && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
                            mx_load8<VT>(p, 0, x);
                        } else {
#pragma unroll
                            for (int k = 0; k < 8; ++k) x[k] = e0 + k < a.N ? MxElem<VT>::get(p[k]) : 0.f;
                        }
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            const uint32_t u = __float_as_uint(x[k]) & 0x7FFFFFFFu;
                            if (u < 0x7F800000u) top = max(top, u);
                        }
                        top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
                        top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
                        const uint32_t f = min(268u - (top >> 23), 253u);   // exponent field of the factor
                        const float factor = __uint_as_float(f << 23);
                        sv = __uint_as_float((254u - f) << 23);
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            float y[2], z[2];
                            unsigned short w[2], l[2];
#pragma unroll
                            for (int j = 0; j < 2; ++j) {
                                y[j] = x[2 * k + j] * factor;
                                w[j] = __half_as_ushort(__float2half_rn(y[j]));
                                z[j] = y[j] - __half2float(__ushort_as_half(w[j]));
                                l[j] = (w[j] & 0x7C00u) == 0x7C00u ? 0 : __half_as_ushort(__float2half_rn(z[j]));
                            }
                            hi[k] = w[0] | ((uint32_t)w[1] << 16);
                            lo[k] = l[0] | ((uint32_t)l[1] << 16);
                        }
                    }
                    if (!mine) continue;
                    __half* d = vec + (long long)n * kParts * column + b * kMxBlock + q * 8;
                    *reinterpret_cast<uint4*>(d) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                    if (kParts == 2) *reinterpret_cast<uint4*>(d + column) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                    if (q == 0) vscale[n * a.chunk_blocks + b] = sv;
                }
                __syncthreads();
            }

            // the products
            const int n_col = a.nv * kParts;
            float acc[R][2][kAcc];
            int tile = 0, task = my_r;
            const bool diag = (g >> 1) == t;        // this lane's column belongs to its own block
            auto multiply = [&](int buf) {
                if (tile == 0) {
#pragma unroll
                    for (int r = 0; r < R; ++r)
#pragma unroll
                        for (int h = 0; h < 2; ++h)
#pragma unroll
                            for (int n = 0; n < kAcc; ++n) acc[r][h][n] = 0.f;
                }
                const int b = (tile_begin + tile) * 4 + t;      // block inside the chunk
#pragma unroll
                for (int p = 0; p < P; ++p) {
                    const int col = 2 * p + (g & 1);
                    const uint4* src = reinterpret_cast<const uint4*>(
                        diag && col < n_col ? reinterpret_cast<const unsigned char*>(vec + col * column + b * kMxBlock) : zeros);
                    float c[R][4];
#pragma unroll
                    for (int r = 0; r < R; ++r) c[r][0] = c[r][1] = c[r][2] = c[r][3] = 0.f;
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const uint4 bv = src[w];
#pragma unroll
                        for (int r = 0; r < R; ++r) {
                            uint32_t x[4], y[4];
                            mx_decode8((&m[buf][r][0].x)[w], x);
                            mx_decode8((&m[buf][r][1].x)[w], y);
                            mma_f16(c[r], x[0], y[0], x[1], y[1], bv.x, bv.y);
                            mma_f16(c[r], x[2], y[2], x[3], y[3], bv.z, bv.w);
                        }
                    }
#pragma unroll
                    for (int r = 0; r < R; ++r)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const float sw = mx_scale_value(s[buf][r][h]);
                            if constexpr (kParts == 2) {
                                const float sv = p < a.nv ? vscale[p * a.chunk_blocks + b] : 0.f;
                                acc[r][h][p] = fmaf((c[r][2 * h] + c[r][2 * h + 1]) * sv, sw, acc[r][h][p]);
                            } else {
#pragma unroll
                                for (int e = 0; e < 2; ++e) {
                                    const int n = 2 * p + e;
                                    const float sv = n < a.nv ? vscale[n * a.chunk_blocks + b] : 0.f;
                                    acc[r][h][n] = fmaf(c[r][2 * h + e] * sv, sw, acc[r][h][n]);
                                }
                            }
                        }
                }
                if (++tile == my_tiles) {
                    // the row's partial sums: over the four lanes, then one slot per warp
#pragma unroll
                    for (int r = 0; r < R; ++r)
#pragma unroll
                        for (int h = 0; h < 2; ++h)
#pragma unroll
                            for (int n = 0; n < kAcc; ++n) {
                                float x = acc[r][h][n];
                                x += __shfl_xor_sync(0xFFFFFFFFu, x, 1);
                                x += __shfl_xor_sync(0xFFFFFFFFu, x, 2);
                                if (t == 0 && n < a.nv) {
                                    float* to = part + ((task * wk + my_k) * a.nv + n) * (16 * R) + r * 16 + h * 8 + g;
                                    *to = ch == 0 ? x : *to + x;
                                }
                            }
                    tile = 0;
                    task += wr;
                }
            };
            for (int i = 0; i < steps; i += kBuf) {
#pragma unroll
                for (int u = 0; u < kBuf; ++u) {
                    if (i + u < steps) {
                        if (i + u + kBuf - 1 < steps) load((u + kBuf - 1) % kBuf);
                        multiply(u);
                    }
                }
            }
        }
        __syncthreads();
        for (int i = tid; i < n_tasks * a.nv * 16 * R; i += kMgThreads) {
            const int r = i % (16 * R), n = (i / (16 * R)) % a.nv, task = i / (16 * R * a.nv);
            const int grp = (first + task) * R + r / 16;
            const long long row = (g_begin + grp) * 16 + (r & 15);
            float x = 0.f;
            for (int k = 0; k < wk; ++k) x += part[((task * wk + k) * a.nv + n) * (16 * R) + r];
            if (grp < my_groups && row < a.M) a.out[n * a.M + row] = x;
        }
        __syncthreads();
    }
}

}  // namespace feather
