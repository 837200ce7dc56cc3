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
// different blocks must not meet before they are scaled.  A lane holds whole blocks of a row; the
// four lanes of a row hold neighbouring ones, and a product adds over all four -- but it has
// eight columns: two columns hold the vector for lane t's block (or blocks) and zeros for the
// other three lanes' slots.  The accumulator that lane t gets back for its row is then the sum
// of ITS block alone, so it multiplies it with its own scale, and nothing moves between lanes
// until the row's end.
//
// The vector.  A block is scaled by a power of two so that its largest finite element lies in
// [2^14, 2^15), and rounded to FP16.  FP16, BF16 and packed values are exact but for what lies
// below FP16's smallest step, half of which is 2^-39 of the block's largest element -- less than
// the FP32 sum keeps.  FP32 values are split in two, x = hi + lo, each rounded to nearest: 2 x 11 bits
// and lo's sign leave at most 2^-23 of the element (a quarter of random ones lose more than 2^-24, what
// rounding to FP32 would), or that same 2^-39; a third part would cost a third column.  Blocks below
// 2^-112 stay below 2^14 (the factor ends at 2^126) and lose nothing more by it: all FP32 numbers are
// multiples of 2^-149, there 2^-23.  The block sum (FP32) is multiplied by the
// vector block's power of two and by the matrix block's, the second time in the FMA that adds it.
//
// Two kernels.  mx_gemv_ring_kernel: one or two columns per block, any size (below).
// mx_gemv_many_kernel: four or eight, for matrices that are too small to go to the tensor cores
// as digits (mxfp4_gemm.cuh); a tile is 16 rows x 128 codes, loaded to registers two tiles ahead.
//
// Work split, both.  A CTA per SM owns a range of 16-row groups; its 16 warps split the row's
// columns (and, for short rows, the groups): a warp keeps its range of columns for all groups and
// leaves a partial sum per row in shared memory, so there is no barrier until the CTA's rows are
// done; then the partials are added in warp order (same bits every run).
//
// Measured, one FP16 vector: 16384 x 16384 26.0 us (5.5 TB/s), 8192 x 8192 10.2, 32000 x 2048 9.1,
// 4096 x 4096 4.6, 256 x 2048 3.0; FP32 at 16384 x 16384 31.7, two FP16 vectors 34.5.  The first
// version (tiles of 16 x 128 loaded to registers, as the many-column kernel still does) took 43.4.
#pragma once
#include <type_traits>

#include "attention_tc.cuh"   // tensor-map copies
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

// Two scale bytes (in the low half) to their values; the conversion gives 2^-127 and NaN their due.
__device__ __forceinline__ float2 mx_scale_pair(uint32_t s) {
    uint32_t d;
    asm("{ .reg .b16 x; cvt.u16.u32 x, %1; cvt.rn.bf16x2.ue8m0x2 %0, x; }" : "=r"(d) : "r"(s));
    return make_float2(__uint_as_float(d << 16), __uint_as_float(d & 0xFFFF0000u));
}

// c x sv x sw, added to `sum`; both factors are powers of two.  c is a multiple of 2^-25 below 2^23 (of
// a packed vector a multiple of 1/4), so c x sv is exact for 2^-124 <= sv < 2^100 (for a packed one below,
// too), and always for FP16 vectors.  A vector with a block outside of that (`far`) has the factors
// taken in the order in which nothing leaves FP32's range but what the result leaves it with:
//   the larger first while it is at most 2^100: no overflow, and no bits lost below 2^-149;
//   else their product, if the smaller one is below 1 (2^-27 .. 2^127, exact);
//   else the smaller first.
// (2^124 in the vector against 2^-60 in the matrix, 2^-149 against 2^127.)  Only such vectors pay:
// FP32 at 16384 x 16384 31.7 us, some such order throughout 33.1, never 31.5.  The many-column kernel,
// short of registers, has its loop twice: 2048 x 4096 x 8 BF16 10.5 us, asked at every product 10.95.
template <bool FAR>
__device__ __forceinline__ float mx_scaled(float c, float sv, float sw, float sum) {
    if constexpr (!FAR) return fmaf(c * sv, sw, sum);
    float low, high;                                 // a NaN scale stays one
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(low) : "f"(sv), "f"(sw));
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(high) : "f"(sv), "f"(sw));
    float first = high, second = low;
    if (!(high <= 0x1p100f)) {
        first = low < 1.f ? high * low : low;
        second = low < 1.f ? 1.f : high;
    }
    return fmaf(c * first, second, sum);
}

struct MxGemvArgs {
    const unsigned char* codes;
    const unsigned char* scales;
    const void* v;                   // nv vectors, N elements apart
    const unsigned char* v_scales;   // of a packed vector (one per launch)
    float* out;                      // nv x M
    long long M, N;
    int blocks;                      // per row
    int nv;                          // vectors of this launch
    int chunk_blocks;                // blocks of the vector in shared memory at a time, a multiple of 8
    int slots;                       // tasks whose partial sums fit
    int part_floats;                 // room for partial sums
    int groups_each, groups_more;    // row groups of every CTA, and CTAs with one more
    unsigned int* status;
    int col_warps;                   // warps that split a row's columns: a power of two, at most the first chunk's tiles or spans
};

// Layout of dynamic shared memory: COLS columns of chunk + 8 halfs, block scales [nv][chunk_blocks],
// 64 bytes of zeros, partial sums.
__host__ __device__ constexpr int mg_column(int chunk_blocks) { return chunk_blocks * kMxBlock + 8; }
__host__ __device__ constexpr int mg_smem_bytes(int cols, int chunk_blocks, int nv, int part_floats) {
    return cols * mg_column(chunk_blocks) * 2 + 4 * nv * chunk_blocks + 64 + 4 * part_floats;
}

// Blocks [blk0, blk0 + pad_blk) of the vectors to shared memory, those from n_blk on as zeros: four
// threads per block, eight elements each, the loads of a few such pieces in flight.  `between` runs
// behind the first loads: what it starts overlaps their latency.  Whether one of this thread's blocks
// is far (see mx_scaled) is returned; a block of zeros is not.
template <int VT, typename F>
__device__ __forceinline__ bool mg_stage(const MxGemvArgs& a, __half* vec, float* vscale, int column, int blk0, int n_blk,
                                         int pad_blk, int tid, F&& between) {
    constexpr int kParts = VT == kSrcF32 ? 2 : 1;
    constexpr int kWords = VT == kSrcF32 ? 8 : VT == kSrcMxfp4 ? 1 : 4;   // of eight elements
    constexpr int kBatch = VT == kSrcF32 ? 2 : 4, kStep = kMgThreads / 4;
    const int q = tid & 3, pieces = a.nv * pad_blk;
    bool begun = false, far = false;
    for (int base = 0; base < pieces; base += kBatch * kStep) {
        uint32_t raw[kBatch][kWords];
        uint32_t sb[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            if (base + u * kStep >= pieces) break;           // the same for every thread
            const int i = min(base + u * kStep + (tid >> 2), pieces - 1), n = i / pad_blk, b = i - n * pad_blk;
            const long long e0 = (long long)(blk0 + b) * kMxBlock + q * 8;
#pragma unroll
            for (int k = 0; k < kWords; ++k) raw[u][k] = 0u;
            sb[u] = 127u;
            if (b >= n_blk) continue;
            if constexpr (VT == kSrcMxfp4) {
                raw[u][0] = __ldg(reinterpret_cast<const uint32_t*>(a.v) + (long long)(blk0 + b) * 4 + q);   // there is one
                sb[u] = __ldg(a.v_scales + blk0 + b);
            } else {
                typedef typename MxElem<VT>::type E;
                const E* p = reinterpret_cast<const E*>(a.v) + (long long)n * a.N + e0;
                if (e0 + 8 <= a.N && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
#pragma unroll
                    for (int k = 0; k < kWords / 4; ++k) {
                        const uint4 x = __ldg(reinterpret_cast<const uint4*>(p) + k);
                        raw[u][4 * k] = x.x; raw[u][4 * k + 1] = x.y; raw[u][4 * k + 2] = x.z; raw[u][4 * k + 3] = x.w;
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        if (e0 + k >= a.N) continue;
                        if constexpr (VT == kSrcF32) raw[u][k] = __float_as_uint(p[k]);
                        else raw[u][k / 2] |= (uint32_t)p[k] << (16 * (k & 1));
                    }
                }
            }
        }
        if (!begun) between();
        begun = true;
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            if (base + u * kStep >= pieces) break;
            const int i = base + u * kStep + (tid >> 2), n = min(i, pieces - 1) / pad_blk, b = min(i, pieces - 1) - n * pad_blk;
            uint32_t hi[4] = {0u, 0u, 0u, 0u}, lo[4] = {0u, 0u, 0u, 0u};
            float sv;
            if constexpr (VT == kSrcMxfp4) {
                mx_decode8(raw[u][0], hi);
                sv = mx_scale_value(sb[u]);
                far |= sv >= 0x1p100f;
            } else {
                float x[8];
                uint32_t top = 0u;
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    if constexpr (VT == kSrcF32) x[k] = __uint_as_float(raw[u][k]);
                    else x[k] = MxElem<VT>::get((unsigned short)(raw[u][k / 2] >> (16 * (k & 1))));
                    const uint32_t m = __float_as_uint(x[k]) & 0x7FFFFFFFu;
                    if (m < 0x7F800000u) top = max(top, m);
                }
                top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
                top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
                const uint32_t f = min(268u - (top >> 23), 253u);   // exponent field of the factor
                const float factor = __uint_as_float(f << 23);
                sv = __uint_as_float((254u - f) << 23);
                far |= sv >= 0x1p100f || (sv < 0x1p-124f && top != 0u);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    unsigned short h[2], l[2];
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const float y = x[2 * k + j] * factor;
                        h[j] = __half_as_ushort(__float2half_rn(y));
                        const float z = y - __half2float(__ushort_as_half(h[j]));
                        l[j] = (h[j] & 0x7C00u) == 0x7C00u ? 0 : __half_as_ushort(__float2half_rn(z));
                    }
                    hi[k] = h[0] | ((uint32_t)h[1] << 16);
                    lo[k] = l[0] | ((uint32_t)l[1] << 16);
                }
            }
            if (i < pieces) {
                __half* d = vec + (long long)n * kParts * column + b * kMxBlock + q * 8;
                *reinterpret_cast<uint4*>(d) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                if (kParts == 2) *reinterpret_cast<uint4*>(d + column) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                if (q == 0) vscale[n * a.chunk_blocks + b] = sv;
            }
        }
    }
    return far;
}

// Four or eight columns.  A lane takes 16 bytes of a row, one block; columns 2 t and 2 t + 1 of a product
// are two vectors, or the halves of an FP32 one, for lane t's block.  VT: type of the vector
// (kSrc..., not a packed one); COLS: columns, an FP32 vector takes two.
template <int VT, int COLS>
__global__ void __launch_bounds__(kMgThreads, 1)
mx_gemv_many_kernel(const MxGemvArgs a) {
    constexpr int kParts = VT == kSrcF32 ? 2 : 1;      // columns per vector
    constexpr int kAcc = COLS / kParts;                // vectors a launch can take
    constexpr int P = COLS / 2;                        // products per 16 codes
    static_assert(COLS % 2 == 0 && VT != kSrcMxfp4, "two columns to a product");
    constexpr int kBuf = 3;                            // tiles in flight
    extern __shared__ __align__(16) unsigned char mg_smem[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int column = mg_column(a.chunk_blocks);
    __half* vec = reinterpret_cast<__half*>(mg_smem);
    float* vscale = reinterpret_cast<float*>(mg_smem + COLS * column * 2);
    unsigned char* zeros = mg_smem + COLS * column * 2 + 4 * a.nv * a.chunk_blocks;
    float* part = reinterpret_cast<float*>(zeros + 64);

    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");

    const long long groups = (a.M + 15) / 16;
    const long long g_begin = groups * blockIdx.x / gridDim.x, g_end = groups * (blockIdx.x + 1) / gridDim.x;
    const int tasks = (int)(g_end - g_begin);          // a 16-row group each
    const int my_rows = (int)min(a.M - g_begin * 16, (long long)tasks * 16);
    const uint4* codes = reinterpret_cast<const uint4*>(a.codes) + g_begin * 16 * a.blocks;
    const unsigned char* scales = a.scales + g_begin * 16 * a.blocks;
    if (tid < 16) reinterpret_cast<uint32_t*>(zeros)[tid] = 0u;

    const int chunks = (a.blocks + a.chunk_blocks - 1) / a.chunk_blocks;
    // warps over columns (wk of them) and tasks (wr of them)
    const int wk = a.col_warps, wr = kMgWarps / wk, my_k = warp & (wk - 1), my_r = warp / wk;
    bool far = false;                                  // the chunk in shared memory has a block that mx_scaled asks about
    for (int first = 0; first < tasks; first += a.slots) {
        const int n_tasks = min(a.slots, tasks - first);
        for (int ch = 0; ch < chunks; ++ch) {
            const int blk0 = ch * a.chunk_blocks, n_blk = min(a.chunk_blocks, a.blocks - blk0);
            const int tiles = (n_blk + 3) / 4;
            const int tile_begin = tiles * my_k / wk, my_tiles = tiles * (my_k + 1) / wk - tile_begin;
            const int my_tasks = my_r < n_tasks ? (n_tasks - my_r + wr - 1) / wr : 0;
            const int steps = my_tasks * my_tiles;

            // The matrix loads, along this warp's walk (its tasks, inside them its tiles).  Offsets
            // count from the CTA's first row in 32 bits.  Rows past the last are the last row again
            // and blocks past the row's end its last block again: the former are not stored, the
            // latter meet a vector of zeros.
            uint4 m[kBuf][2];
            uint32_t s[kBuf][2];
            uint32_t row_at[2];
            int l_tile = 0, l_task = my_r;
            auto load = [&](int buf) {
                if (l_tile == 0) {
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        row_at[h] = (uint32_t)min((first + l_task) * 16 + g + 8 * h, my_rows - 1) * (uint32_t)a.blocks;
                }
                const uint32_t blk = (uint32_t)(blk0 + min((tile_begin + l_tile) * 4 + t, n_blk - 1));
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t at = row_at[h] + blk;
                    m[buf][h] = ldg_stream(codes + at);
                    s[buf][h] = __ldg(scales + at);
                }
                if (++l_tile == my_tiles) l_tile = 0, l_task += wr;
            };
#pragma unroll
            for (int i = 0; i < kBuf - 1; ++i)
                if (i < steps) load(i);

            // the vector chunk: four threads per block, eight elements each
            if (ch > 0 || first > 0 ? chunks > 1 : true) {
                if (ch > 0 || first > 0) __syncthreads();   // the previous chunk's readers are done
                far = mg_stage<VT>(a, vec, vscale, column, blk0, n_blk, tiles * 4, tid, [] {});
                if constexpr (VT == kSrcF16) __syncthreads();
                else far = __syncthreads_or(far);
            }

            // the products
            const int n_col = a.nv * kParts;
            float acc[2][kAcc];
            int tile = 0, task = my_r;
            const bool diag = (g >> 1) == t;        // this lane's column belongs to its own block
            auto multiply = [&](int buf, auto far) {
                if (tile == 0) {
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int n = 0; n < kAcc; ++n) acc[h][n] = 0.f;
                }
                const int b = (tile_begin + tile) * 4 + t;      // block inside the chunk
                const float2 sw = mx_scale_pair(s[buf][0] | (s[buf][1] << 8));
                uint32_t x[2][4][4];                    // decoded once, multiplied with every pair of columns
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    mx_decode8(m[buf][h].x, x[h][0]);
                    mx_decode8(m[buf][h].y, x[h][1]);
                    mx_decode8(m[buf][h].z, x[h][2]);
                    mx_decode8(m[buf][h].w, x[h][3]);
                }
#pragma unroll
                for (int p = 0; p < P; ++p) {
                    const int col = 2 * p + (g & 1);
                    const uint4* src = reinterpret_cast<const uint4*>(
                        diag && col < n_col ? reinterpret_cast<const unsigned char*>(vec + col * column + b * kMxBlock) : zeros);
                    float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const uint4 bv = src[w];
                        mma_f16(c, x[0][w][0], x[1][w][0], x[0][w][1], x[1][w][1], bv.x, bv.y);
                        mma_f16(c, x[0][w][2], x[1][w][2], x[0][w][3], x[1][w][3], bv.z, bv.w);
                    }
                    // (a block's sum) x (the vector block's power of two) x (the matrix block's)
                    if constexpr (kParts == 2) {
                        const float sv = p < a.nv ? vscale[p * a.chunk_blocks + b] : 0.f;
                        acc[0][p] = mx_scaled<far>(c[0] + c[1], sv, sw.x, acc[0][p]);
                        acc[1][p] = mx_scaled<far>(c[2] + c[3], sv, sw.y, acc[1][p]);
                    } else {
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const int n = 2 * p + e;
                            const float sv = n < a.nv ? vscale[n * a.chunk_blocks + b] : 0.f;
                            acc[0][n] = mx_scaled<far>(c[e], sv, sw.x, acc[0][n]);
                            acc[1][n] = mx_scaled<far>(c[2 + e], sv, sw.y, acc[1][n]);
                        }
                    }
                }
                if (++tile == my_tiles) {
                    // the row's partial sums: over the four lanes, then one slot per warp
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int n = 0; n < kAcc; ++n) {
                            float x = acc[h][n];
                            x += __shfl_xor_sync(0xFFFFFFFFu, x, 1);
                            x += __shfl_xor_sync(0xFFFFFFFFu, x, 2);
                            if (t == 0 && n < a.nv) {
                                float* to = part + ((task * wk + my_k) * a.nv + n) * 16 + h * 8 + g;
                                *to = ch == 0 ? x : *to + x;
                            }
                        }
                    tile = 0;
                    task += wr;
                }
            };
            auto walk = [&](auto far) {
                for (int i = 0; i < steps; i += kBuf) {
#pragma unroll
                    for (int u = 0; u < kBuf; ++u) {
                        if (i + u < steps) {
                            if (i + u + kBuf - 1 < steps) load((u + kBuf - 1) % kBuf);
                            multiply(u, far);
                        }
                    }
                }
            };
            if (VT != kSrcF16 && far) walk(std::true_type{});
            else walk(std::false_type{});
        }
        __syncthreads();
        for (int i = tid; i < n_tasks * a.nv * 16; i += kMgThreads) {
            const int r = i % 16, n = (i / 16) % a.nv, task = i / (16 * a.nv);
            const long long row = (g_begin + first + task) * 16 + r;
            float x = 0.f;
            for (int k = 0; k < wk; ++k) x += part[((task * wk + k) * a.nv + n) * 16 + r];
            if (row < a.M) a.out[n * a.M + row] = x;
        }
        __syncthreads();
    }
}

// One or two columns (a vector, an FP32 vector in two parts, two vectors), any size.
//
// A lane takes 32 bytes of a row, two neighbouring blocks, and the four lanes of a row a whole
// 128-byte line.  The product's rows 0-7 are the first blocks of eight rows, its rows 8-15 the
// second blocks of the same rows; column n holds the vector for block n of the line, zero but
// in the slots of lane n / 2.  Of the four sums a lane gets back, the first is its first block's
// and the last its second block's.
//
// The codes come through shared memory.  A warp owns SLOTS slots of 4 KB, 16 rows x 512 codes (two
// lines), that it fills itself with tensor-map copies (128-byte swizzle: the reads below are free of
// bank conflicts); it refills a slot as soon as it has read it, so nothing is shared and nothing
// but arrival is waited for.  Loads straight to registers reached 3.9 TB/s at 16384 x 16384 (the
// bytes in flight hang on the scoreboard), this 5.5.  The vector is loaded before the first copies are
// issued and staged while they travel: its loads behind 19 MB of copies had cost 3 us.
constexpr int kMrRows = 16, kMrLines = 2, kMrSlotBytes = kMrRows * kMrLines * 128;

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z) : "memory");
}
// The same boxes into L2 only.
__device__ __forceinline__ void tma_prefetch_3d(const CUtensorMap* map, int x, int y, int z) {
    asm volatile("cp.async.bulk.prefetch.tensor.3d.L2.global [%0, {%1, %2, %3}];"
                 ::"l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z) : "memory");
}
// Host side: rows of whole lines as {128 bytes, rows, lines} with boxes of 16 rows x 2 lines.
inline bool mr_make_map(CUtensorMap* map, const void* base, long long row_bytes, long long rows) {
    const AtcEncodeTiled encode = atc_encoder();
    if (!encode) return false;
    const cuuint64_t dims[3] = {128, (cuuint64_t)rows, (cuuint64_t)(row_bytes / 128)};
    const cuuint64_t strides[2] = {(cuuint64_t)row_bytes, 128};
    const cuuint32_t box[3] = {128, kMrRows, kMrLines};
    const cuuint32_t steps[3] = {1, 1, 1};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(base), dims, strides, box, steps,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// WHOLE: rows of whole lines, one three-dimensional copy per slot; else two two-dimensional ones.
// Shared memory: slots, then as above, then a barrier per slot.
template <int VT, int COLS, int SLOTS, bool WHOLE>
__global__ void __launch_bounds__(kMgThreads, 1)
mx_gemv_ring_kernel(const __grid_constant__ CUtensorMap map, const MxGemvArgs a) {
    constexpr int kParts = VT == kSrcF32 ? 2 : 1;
    constexpr int kAcc = COLS / kParts;
    constexpr int R = kMrRows / 8;
    extern __shared__ __align__(1024) unsigned char mr_smem[];
    unsigned char* mg_smem = mr_smem + kMgWarps * SLOTS * kMrSlotBytes;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int column = mg_column(a.chunk_blocks);
    __half* vec = reinterpret_cast<__half*>(mg_smem);
    float* vscale = reinterpret_cast<float*>(mg_smem + COLS * column * 2);
    unsigned char* zeros = mg_smem + COLS * column * 2 + 4 * a.nv * a.chunk_blocks;
    float* part = reinterpret_cast<float*>(zeros + 64);
    const uint32_t slots = smem_u32(mr_smem) + warp * (SLOTS * kMrSlotBytes);
    const uint32_t bars = smem_u32(part + a.part_floats) + warp * (SLOTS * 8);

    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (smem_u32(mr_smem) & 1023u) {                 // every CTA alike
        if (tid == 0) atomicOr(a.status, 2u);
        return;
    }
    if (lane == 0) {
        for (int i = 0; i < SLOTS; ++i) mbar_init(bars + 8 * i, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    // everything that needs no memory is behind us when the kernel before this one has ended
    const int extra = min((int)blockIdx.x, a.groups_more);
    const int g_begin = (int)blockIdx.x * a.groups_each + extra, tasks = a.groups_each + ((int)blockIdx.x < a.groups_more ? 1 : 0);
    const int my_rows = (int)min(a.M - (long long)g_begin * kMrRows, (long long)tasks * kMrRows);
    const unsigned char* scales = a.scales + (long long)g_begin * kMrRows * a.blocks;
    if (tid < 16) reinterpret_cast<uint32_t*>(zeros)[tid] = 0u;

    const int chunks = (a.blocks + a.chunk_blocks - 1) / a.chunk_blocks;
    const int wk = a.col_warps, wr = kMgWarps / wk, my_k = warp & (wk - 1), my_r = warp / wk;
    // Ask L2 for the first slots' codes while the kernel in front still runs: harmless whatever it
    // writes, because its writes land in L2 too.  (8192 x 8192 11.2 -> 10.2 us, 16384 x 16384 26.9 ->
    // 26.0, 256 x 2048 the same.)
    if (lane == 0 && my_r < tasks) {
        const int n_blk = min(a.chunk_blocks, a.blocks), spans = (n_blk + 8 * kMrLines - 1) / (8 * kMrLines);
        const int from = spans * my_k / wk, n = spans * (my_k + 1) / wk - from;
        int span = 0, task = my_r;
        for (int i = 0; i < SLOTS && task < min(a.slots, tasks) && n > 0; ++i) {
            const int y = (g_begin + task) * kMrRows, z = (from + span) * kMrLines;
            if constexpr (WHOLE) {
                tma_prefetch_3d(&map, 0, y, z);
            } else {
#pragma unroll
                for (int l = 0; l < kMrLines; ++l) tma_prefetch_2d(&map, (z + l) * 128, y);
            }
            if (++span == n) span = 0, task += wr;
        }
    }
    __syncwarp();
    asm volatile("griddepcontrol.wait;" ::: "memory");
    bool ok = true, far = false;                     // far: see mx_scaled
    int used = 0;                                    // slots read so far, over all chunks
    int filled = 0, lost = 0;                        // slots asked for, and read when a wait gave up
    for (int first = 0; first < tasks; first += a.slots) {
        const int n_tasks = min(a.slots, tasks - first);
        for (int ch = 0; ch < chunks; ++ch) {
            const int blk0 = ch * a.chunk_blocks, n_blk = min(a.chunk_blocks, a.blocks - blk0);
            const int spans = (n_blk + 8 * kMrLines - 1) / (8 * kMrLines);
            const int span_begin = spans * my_k / wk, my_spans = spans * (my_k + 1) / wk - span_begin;
            const int my_tasks = my_r < n_tasks ? (n_tasks - my_r + wr - 1) / wr : 0;
            const int steps = my_tasks * my_spans;

            int l_span = 0, l_task = my_r;
            auto fill = [&](int slot) {              // the next step of this warp's walk; one lane
                const int y = (g_begin + first + l_task) * kMrRows, z = blk0 / 8 + (span_begin + l_span) * kMrLines;
                const uint32_t to = slots + slot * kMrSlotBytes, bar = bars + 8 * slot;
                if (lane == 0 && ok) {               // after a wait that gave up nothing more is asked for
                    ++filled;
                    mbar_arrive_expect_tx(bar, kMrSlotBytes);
                    if constexpr (WHOLE) {
                        tma_load_3d(to, &map, 0, y, z, bar);
                    } else {
#pragma unroll
                        for (int i = 0; i < kMrLines; ++i) tma_load_2d(to + i * (kMrRows * 128), &map, (z + i) * 128, y, bar);
                    }
                }
                if (++l_span == my_spans) l_span = 0, l_task += wr;
            };
            auto begin = [&] {
                for (int i = 0; i < SLOTS && i < steps; ++i) fill((used + i) % SLOTS);
            };
            // scale bytes of a step, two blocks of two lines of R rows, a step ahead
            uint32_t s[kMrLines][R], s_next[kMrLines][R];
            int s_span = 0, s_task = my_r;
            auto load_scales = [&]() {
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const uint32_t row = (uint32_t)min((first + s_task) * kMrRows + r * 8 + g, my_rows - 1) * (uint32_t)a.blocks;
#pragma unroll
                    for (int l = 0; l < kMrLines; ++l) {
                        const int blk = ((span_begin + s_span) * kMrLines + l) * 8 + 2 * t;
                        if constexpr (WHOLE) {
                            const int at = min(blk, n_blk - 2);
                            s_next[l][r] = __ldg(reinterpret_cast<const unsigned short*>(scales + row + blk0 + at));
                        } else {
                            s_next[l][r] = __ldg(scales + row + blk0 + min(blk, n_blk - 1)) |
                                           ((uint32_t)__ldg(scales + row + blk0 + min(blk + 1, n_blk - 1)) << 8);
                        }
                    }
                }
                if (++s_span == my_spans) s_span = 0, s_task += wr;
            };
            if (ch > 0 || first > 0 ? chunks > 1 : true) {
                if (ch > 0 || first > 0) __syncthreads();   // the previous chunk's readers are done
                far = mg_stage<VT>(a, vec, vscale, column, blk0, n_blk, spans * 8 * kMrLines, tid, begin);
                if (steps > 0) load_scales();
                if constexpr (VT == kSrcF16) __syncthreads();
                else far = __syncthreads_or(far);
            } else {
                begin();
                if (steps > 0) load_scales();
            }

            float acc[R][kAcc];
            int span = 0, task = my_r;
            const bool diag = (g >> 1) == t;
            for (int i = 0; i < steps; ++i, ++used) {
                const int slot = used % SLOTS;
                if (span == 0) {
#pragma unroll
                    for (int r = 0; r < R; ++r)
#pragma unroll
                        for (int n = 0; n < kAcc; ++n) acc[r][n] = 0.f;
                }
#pragma unroll
                for (int l = 0; l < kMrLines; ++l)
#pragma unroll
                    for (int r = 0; r < R; ++r) s[l][r] = s_next[l][r];
                if (i + 1 < steps) load_scales();
                if (ok && !mbar_wait(bars + 8 * slot, (uint32_t)((used / SLOTS) & 1), a.status)) ok = false, lost = used;
                const unsigned char* from = mr_smem + (warp * SLOTS + slot) * kMrSlotBytes + g * 128;
#pragma unroll
                for (int l = 0; l < kMrLines; ++l) {
                    const int b = ((span_begin + span) * kMrLines + l) * 8;      // the line's first block inside the chunk
                    float c[R][COLS][4];
                    const uint4* src[COLS];
#pragma unroll
                    for (int p = 0; p < COLS; ++p) {
                        src[p] = reinterpret_cast<const uint4*>(
                            diag ? reinterpret_cast<const unsigned char*>(vec + p * column + (b + g) * kMxBlock) : zeros);
#pragma unroll
                        for (int r = 0; r < R; ++r) c[r][p][0] = c[r][p][1] = c[r][p][2] = c[r][p][3] = 0.f;
                    }
                    uint4 m[R][2];
#pragma unroll
                    for (int r = 0; r < R; ++r)
#pragma unroll
                        for (int h = 0; h < 2; ++h)      // 16-byte units of a row are swizzled with the row's number
                            m[r][h] = *reinterpret_cast<const uint4*>(from + l * (kMrRows * 128) + r * 1024 + (((2 * t + h) ^ g) << 4));
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        uint4 bv[COLS];
#pragma unroll
                        for (int p = 0; p < COLS; ++p) bv[p] = src[p][w];
#pragma unroll
                        for (int r = 0; r < R; ++r) {
                            uint32_t x[4], y[4];
                            mx_decode8(w == 0 ? m[r][0].x : w == 1 ? m[r][0].y : w == 2 ? m[r][0].z : m[r][0].w, x);
                            mx_decode8(w == 0 ? m[r][1].x : w == 1 ? m[r][1].y : w == 2 ? m[r][1].z : m[r][1].w, y);
#pragma unroll
                            for (int p = 0; p < COLS; ++p) {
                                mma_f16(c[r][p], x[0], y[0], x[1], y[1], bv[p].x, bv[p].y);
                                mma_f16(c[r][p], x[2], y[2], x[3], y[3], bv[p].z, bv[p].w);
                            }
                        }
                    }
#pragma unroll
                    for (int n = 0; n < kAcc; ++n) {
                        const float2 sv = *reinterpret_cast<const float2*>(vscale + n * a.chunk_blocks + b + 2 * t);
#pragma unroll
                        for (int r = 0; r < R; ++r) {
                            const float2 sw = mx_scale_pair(s[l][r]);
                            const float c0 = kParts == 2 ? c[r][0][0] + c[r][COLS - 1][0] : c[r][n][0];
                            const float c1 = kParts == 2 ? c[r][0][3] + c[r][COLS - 1][3] : c[r][n][3];
                            if (VT != kSrcF16 && far) {
                                acc[r][n] = mx_scaled<true>(c0, sv.x, sw.x, acc[r][n]);
                                acc[r][n] = mx_scaled<true>(c1, sv.y, sw.y, acc[r][n]);
                            } else {
                                acc[r][n] = mx_scaled<false>(c0, sv.x, sw.x, acc[r][n]);
                                acc[r][n] = mx_scaled<false>(c1, sv.y, sw.y, acc[r][n]);
                            }
                        }
                    }
                }
                __syncwarp();                        // every lane has read the slot
                if (i + SLOTS < steps) fill(slot);
                if (++span == my_spans) {
#pragma unroll
                    for (int r = 0; r < R; ++r)
#pragma unroll
                        for (int n = 0; n < kAcc; ++n) {
                            float x = acc[r][n];
                            x += __shfl_xor_sync(0xFFFFFFFFu, x, 1);
                            x += __shfl_xor_sync(0xFFFFFFFFu, x, 2);
                            if (t == 0) {
                                float* to = part + ((task * wk + my_k) * kAcc + n) * kMrRows + r * 8 + g;
                                *to = ch == 0 ? x : *to + x;
                            }
                        }
                    span = 0;
                    task += wr;
                }
            }
        }
        __syncthreads();
        for (int i = tid; i < n_tasks * kAcc * kMrRows; i += kMgThreads) {
            const int r = i % kMrRows, n = (i / kMrRows) % kAcc, task = i / (kMrRows * kAcc);
            const int row = (first + task) * kMrRows + r;
            float x = 0.f;
            for (int k = 0; k < wk; ++k) x += part[((task * wk + k) * kAcc + n) * kMrRows + r];
            if (row < my_rows) a.out[n * a.M + (long long)g_begin * kMrRows + row] = x;
        }
        __syncthreads();
    }
    if (!ok && lane == 0)                            // shared memory outlives what was asked for
        for (int i = lost; i < filled; ++i) mbar_wait(bars + 8 * (i % SLOTS), (uint32_t)((i / SLOTS) & 1), a.status);
    __syncthreads();
}

}  // namespace feather
