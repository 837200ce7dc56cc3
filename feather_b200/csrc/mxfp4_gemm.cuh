// Product of two microscaled 4-bit matrices on the fifth-generation tensor cores (sm_100a):
//
//   out[b][r] = sum_j value(m[r][j]) * value(x[b][j])     FP32 accumulation, one rounding to
//                                                         FP32, BF16 or FP16
//
// value() as in mxfp4_codec.cuh.  No counterpart in the reference.  tcgen05.mma kind::mxf4 takes
// the packed codes and the scale bytes as they are: nothing is decoded.
//
// Mapping.  A tile is 128 rows of m (the 128 lanes of tensor memory) x NT rows of x (its columns);
// a persistent CTA per SM walks the tiles.  A stage of the shared-memory ring holds 256 codes
// (128 bytes) of every row of the tile, brought by tensor-map copies in the 128-byte swizzle,
// and their eight scale bytes.  Per stage four products of 64 codes run; each names two of the
// four scale bytes of a 32-bit tensor-memory word, where tcgen05.cp puts them from shared
// memory: 128 rows x 4 scales are a 512-byte piece, row r at (r % 32) * 16 + (r / 32) * 4.  The
// scales lie row after row in global memory, so four warps load them (8 bytes per row and
// stage, four stages at a time) and store them in that order.
//
// Warps: 0 copies, 1 issues, 2-5 scales, 6-9 store finished tiles while the next one is
// multiplied (two accumulators alternate).  Every wait is bounded; a CTA that gave up
// frees its tensor memory.
//
// What it took, at 16384 x 8192 x 4096 (NT = 224): one lane of the issuing warp walking the stages
// by itself 382 us; the whole warp walking them (uniform addresses), one elected lane issuing 244;
// the result through shared memory and tensor-map copies instead of 2-byte stores 219 us = 5.0
// PFLOP/s in short runs.  Products alone, operands in place and nothing awaited, take 148 us;
// a stage needs 90 bytes per clock from L2, and only four fit.  Under load the 1000 W cap holds the
// SM at 1.43 GHz: 258 us, 4.3 PFLOP/s, 3.1 times the bf16 rate measured so.  Pairs of CTAs
// (cta_group::2, 256 x 224 tiles, 30 KB instead of 44 per CTA and stage) took 249 .. 263 us and were
// dropped; so was a split over clusters of eight (they do not all run at once).
// Small: 2048 x 5632 x 33 6.8 us (four CTAs per tile; whole 8.1), 5001 x 2050 x 200 to FP32 10.6.
// Memory-bound: 16384 x 16384 x 16 25.6 us (5.6 TB/s).
//
// Few tiles: a cluster of 2 or 4 CTAs shares one tile, each with its part of the row; the
// partial sums meet through distributed shared memory and are added in rank order, each CTA
// storing its share of the columns.  No scratch in global memory, the same bits every run.
//
// Dense vectors (DIGITS): a vector is first written as kGmDigits packed rows whose sum it is --
// each row is the quantised remainder of the ones before it (mx_digits_kernel), at least two more
// bits per row -- and its columns are added when they are stored.  With a matrix that is read
// once anyway the extra columns cost little, and nothing of the matrix is decoded.
#pragma once
#include "attention_tc.cuh"   // descriptors, tensor-map copies, tensor-memory loads
#include "mxfp4_codec.cuh"

namespace feather {

constexpr int kGmThreads = 10 * 32;
constexpr int kGmRows = 128;
constexpr int kGmBox = 128;                    // bytes of a row per stage = the swizzle width
constexpr int kGmBlocks = 8;                   // scale blocks per stage
constexpr int kGmGroup = 4;                    // stages whose scales travel together

constexpr int kGmPiece = 2048;                 // bytes of a warp's piece of the result: 32 rows of m x 32 (16-bit) or 16 of x
constexpr int kGmOutBytes = 4 * 2 * kGmPiece;  // two per storing warp

template <int NT>
struct GmLayout {
    static constexpr int kRowAtoms = NT > 128 ? 2 : 1;                     // 128-row pieces of x's scales
    static constexpr int kA = kGmRows * kGmBox, kB = NT * kGmBox;          // operand bytes of a stage
    static constexpr int kSfStage = 2 * (1 + kRowAtoms) * 512;             // scale bytes of a stage: 2 x (m, x)
    static constexpr int kSfGroup = kGmGroup * kSfStage;
    static constexpr int kMost = (227 * 1024 - 256 - 2 * kSfGroup - kGmOutBytes) / (kA + kB);
    static constexpr int kStages = kMost > 10 ? 10 : kMost;
    static constexpr int kSf = kStages * (kA + kB);                        // two groups of scales behind the operands
    static constexpr int kOut = kSf + 2 * kSfGroup;                        // pieces of the result on their way out
    static constexpr int kBar = kOut + kGmOutBytes;
    static constexpr int kBytes = kBar + 8 * (2 * kStages + 8) + 16;
    static constexpr int kSfColsA = 2 * 4, kSfColsB = 2 * 4 * kRowAtoms;   // 32-bit columns of a stage's scales
    static constexpr int kSfCol = 2 * NT;                                  // two sets alternate
    static constexpr int kCols = 512;
    static_assert(kSfCol + 2 * (kSfColsA + kSfColsB) <= kCols, "tensor memory");
    static_assert(kA % 1024 == 0 && kB % 1024 == 0, "swizzled tiles are 1 KiB aligned");
};

// Instruction descriptor of kind::mxf4: E2M1 operands (1 in bits 7-9 and 10-11), K-major, N / 8 in
// bits 17-22, power-of-two scales (bit 23), M / 16 in bits 24-28, the scale bytes' place in
// their word (0 or 2) in bits 4-5 for B and 29-30 for A.
template <int NT>
__host__ __device__ constexpr uint32_t gm_idesc(int place) {
    return ((uint32_t)place << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(NT / 8) << 17) | (1u << 23) |
           ((uint32_t)(kGmRows / 16) << 24) | ((uint32_t)place << 29);
}
__device__ __forceinline__ void gm_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                       uint32_t accumulate) {
    asm volatile("{ .reg .pred p; setp.ne.b32 p, %6, 0;\n"
                 "  tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p; }"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate) : "memory");
}
// One lane of a converged warp, the same one every time.
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{ .reg .pred p; elect.sync _|p, 0xFFFFFFFF; selp.u32 %0, 1, 0, p; }" : "=r"(p));
    return p != 0;
}
// 512 bytes (32 rows of 16) of shared memory to four columns of tensor memory, the same in
// every quarter of the lanes.
__device__ __forceinline__ void gm_copy_scales(uint32_t taddr, uint64_t desc) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

// A box of a 2-D tensor map written from shared memory, and the waits for such copies: all
// but N groups have been read / are complete.
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, uint32_t src, int x, int y) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];"
                 ::"l"(reinterpret_cast<uint64_t>(map)), "r"(src), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void bulk_wait_read() { asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory"); }
template <int N>
__device__ __forceinline__ void bulk_wait() { asm volatile("cp.async.bulk.wait_group %0;" ::"n"(N) : "memory"); }

// Host side: the result as a 2-D tensor map with boxes of 32 of m x `piece` rows of x.
inline bool gm_make_out_map(CUtensorMap* map, void* out, int out_size, bool bf16, long long M, long long batch, int piece) {
    const AtcEncodeTiled encode = atc_encoder();
    if (!encode) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)M, (cuuint64_t)batch};
    const cuuint64_t strides[1] = {(cuuint64_t)M * out_size};
    const cuuint32_t box[2] = {32, (cuuint32_t)piece};
    const cuuint32_t steps[2] = {1, 1};
    const CUtensorMapDataType type = out_size == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                     : bf16        ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                   : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    return encode(map, type, 2, out, dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
                  CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// The scale bytes of blocks [k, k + 32) of a row as eight words, those past the row's end as 0.
// `all` is one past the last scale byte of the operand.
__device__ __forceinline__ void gm_load_scales(uint32_t (&w)[8], const unsigned char* row, int k, int blocks, int align,
                                               const unsigned char* begin, const unsigned char* all) {
    if (align == 16) {                           // whole rows in steps of 16 blocks
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint4 v = k + 16 * i < blocks ? __ldg(reinterpret_cast<const uint4*>(row + k) + i) : make_uint4(0u, 0u, 0u, 0u);
            w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
        }
    } else if (align == 4) {
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = k + 4 * i < blocks ? __ldg(reinterpret_cast<const uint32_t*>(row + k) + i) : 0u;
    } else {
        // any alignment: the aligned words that cover the bytes, shifted into place
        const unsigned char* from = reinterpret_cast<const unsigned char*>(reinterpret_cast<uintptr_t>(row + k) & ~(uintptr_t)3);
        const uint32_t shift = 8u * (uint32_t)(reinterpret_cast<uintptr_t>(row + k) & 3);
        const int left = blocks - k;             // bytes of this row still wanted, at least 1
        uint32_t x[9];
        if (from >= begin && from + 36 <= all) { // no branch between the loads: they are in flight together
#pragma unroll
            for (int i = 0; i < 9; ++i) x[i] = __ldg(reinterpret_cast<const uint32_t*>(from) + i);
        } else {                                 // at an end of the operand: byte by byte, and no further
            for (int i = 0; i < 9; ++i) x[i] = 0u;
#pragma unroll
            for (int i = 0; i < 36; ++i)
                if (from + i >= begin && from + i < all) x[i / 4] |= (uint32_t)__ldg(from + i) << (8 * (i % 4));
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            w[i] = __funnelshift_r(x[i], x[i + 1], shift);
            const int over = 4 * i + 4 - left;   // bytes of this word past the row's end
            if (over > 0) w[i] = over >= 4 ? 0u : w[i] & (0xFFFFFFFFu >> (8 * over));
        }
    }
}

struct MxGemmArgs {
    const unsigned char* m_scales;
    const unsigned char* x_scales;
    void* out;                    // batch x M
    int M, batch, blocks;
    int tiles_m, tiles_x;
    int split;                    // CTAs of a cluster that share a tile
    int align;                    // of the scale rows: 16, 4 or 1
    int bulk;                     // 1: result rows are 16-byte aligned, pieces leave by tensor-map copies
    unsigned int* status;
    // dense vectors: x is their digits, batch counts digit rows; what the rare repair needs
    const unsigned char* m_codes;
    const void* v;
    int v_dtype;
    long long N;
};

constexpr int kGmDigits = 12;

// Dense vectors to digits: row kGmDigits n + d of (codes, scales) is the quantised remainder of vector
// n after d rows.  Four threads per block, eight elements each; the remainder is exact in FP32 (an
// element and its code's value are within a factor of two, or the code is zero).  A row leaves at
// most a quarter of the block's largest remainder, so after all of them 2^-24 of its largest
// element is left: one FP32 rounding of that (or 2^-129, a quarter of the smallest scale).  (16 rows: 39.6 us for 8 vectors at 16384 x
// 16384, 12 rows 38.8, before other steps.)  A block with an infinity or a NaN gets scale 255 in row 0.
template <int VT>
__global__ void __launch_bounds__(256)
mx_digits_kernel(const void* __restrict__ v, uint32_t* __restrict__ codes, unsigned char* __restrict__ scales, long long N,
                 int blocks, int vectors) {
    // The product kernel behind this one may start once everything before this one is done: it reads
    // the matrix before it waits for the digits.
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    typedef typename MxElem<VT>::type E;
    const int quads = blocks * vectors, i = blockIdx.x * blockDim.x + threadIdx.x;
    const bool mine = (i >> 2) < quads;
    const int q = i & 3, n = mine ? (i >> 2) / blocks : 0, b = mine ? (i >> 2) - n * blocks : 0;
    const long long e0 = (long long)b * kMxBlock + q * 8;
    const E* p = reinterpret_cast<const E*>(v) + n * N + e0;
    float x[8];
    if (e0 + 8 <= N && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
        mx_load8<VT>(p, 0, x);
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] = e0 + k < N ? MxElem<VT>::get(p[k]) : 0.f;
    }
#pragma unroll 4
    for (int d = 0; d < kGmDigits; ++d) {
        uint32_t top = 0u;
#pragma unroll
        for (int k = 0; k < 8; ++k) top = max(top, __float_as_uint(x[k]) & 0x7FFFFFFFu);
        top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
        top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
        const uint32_t s = mx_scale_byte(top);
        const float f = mx_to_grid(s), back = mx_scale_value(s);
        float y[8];
        uint32_t h[4];
#pragma unroll
        for (int k = 0; k < 8; ++k) y[k] = x[k] * f;
        const uint32_t c = s == 255u ? 0u : mx_encode8(y);
        mx_decode8(c, h);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float2 z = h2_to_f2(h[k]);
            x[2 * k] = s == 255u ? 0.f : x[2 * k] - z.x * back;
            x[2 * k + 1] = s == 255u ? 0.f : x[2 * k + 1] - z.y * back;
        }
        if (mine) {
            const long long at = ((long long)n * kGmDigits + d) * blocks + b;
            codes[at * 4 + q] = c;
            if (q == 0) scales[at] = (unsigned char)s;
        }
    }
}

// The digits' columns of a vector added up, the smallest digit first.
__device__ __forceinline__ float gm_add_digits(uint32_t taddr) {
    float r[16];                                 // the last four are the next vector's
    tmem_ld<16>(taddr, r);
    float x = r[kGmDigits - 1];
#pragma unroll
    for (int d = kGmDigits - 2; d >= 0; --d) x += r[d];
    return x;
}
// Bit c: vector x0 + c holds an infinity or a NaN (its first digits have a block of scale 255).
template <int VECTORS>
__device__ __forceinline__ uint32_t gm_find_not_finite(const MxGemmArgs& g, int x0, int lane) {
    uint32_t found = 0u;
    for (int c = 0; c < VECTORS && (x0 + c) * kGmDigits < g.batch; ++c) {
        const unsigned char* s = g.x_scales + (long long)(x0 + c) * kGmDigits * g.blocks;
        uint32_t top = 0u;
        for (int b0 = lane; b0 - lane < g.blocks; b0 += 32 * 16) {     // sixteen loads in flight
            uint32_t x[16];
#pragma unroll
            for (int u = 0; u < 16; ++u) x[u] = b0 + 32 * u < g.blocks ? __ldg(s + b0 + 32 * u) : 0u;
#pragma unroll
            for (int u = 0; u < 16; ++u) top = max(top, x[u]);
        }
        if (__any_sync(0xFFFFFFFFu, top == 255u)) found |= 1u << c;
    }
    return found;
}
// Row m times such a vector: the blocks that hold what is not finite decide the result.  (Not inlined,
// it gives the kernel a stack frame, and that alone cost 7 of 36 us at 16384 x 16384 x 3.)
__device__ __forceinline__ float gm_not_finite(const MxGemmArgs& g, int m, int n) {
    const unsigned char* s = g.x_scales + (long long)n * kGmDigits * g.blocks;
    float sum = 0.f;
    for (int b = 0; b < g.blocks; ++b) {
        const uint32_t ms = g.m_scales[(long long)m * g.blocks + b];
        if (ms == 255u) return __uint_as_float(0x7FC00000u);     // the row is NaN whatever the vector holds
        if (s[b] != 255) continue;
        const float scale = mx_scale_value(ms);
        for (int i = 0; i < kMxBlock && (long long)b * kMxBlock + i < g.N; ++i) {
            const long long e = n * g.N + (long long)b * kMxBlock + i;
            const float v = g.v_dtype == kSrcF32   ? reinterpret_cast<const float*>(g.v)[e]
                            : g.v_dtype == kSrcF16 ? MxElem<kSrcF16>::get(reinterpret_cast<const unsigned short*>(g.v)[e])
                                                   : MxElem<kSrcBF16>::get(reinterpret_cast<const unsigned short*>(g.v)[e]);
            const uint32_t pair = g.m_codes[((long long)m * g.blocks + b) * 16 + i / 2];
            uint32_t h[4];
            mx_decode8(i & 1 ? pair >> 4 : pair, h);
            sum = fmaf(h2_to_f2(h[0]).x * scale, v, sum);
        }
    }
    return sum;
}

template <int NT, int OUT, bool DIGITS>
__global__ void __launch_bounds__(kGmThreads, 1)
mx_gemm_kernel(const __grid_constant__ CUtensorMap map_m, const __grid_constant__ CUtensorMap map_x,
               const __grid_constant__ CUtensorMap map_out, const MxGemmArgs g) {
    typedef GmLayout<NT> L;
    extern __shared__ __align__(1024) unsigned char gm_smem[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t sbase = smem_u32(gm_smem), bars = sbase + L::kBar;
    auto full = [&](int s) { return bars + 8u * s; };
    auto empty = [&](int s) { return bars + 8u * (L::kStages + s); };
    auto acc_full = [&](int a) { return bars + 8u * (2 * L::kStages + a); };
    auto acc_empty = [&](int a) { return bars + 8u * (2 * L::kStages + 2 + a); };
    auto sf_full = [&](int a) { return bars + 8u * (2 * L::kStages + 4 + a); };
    auto sf_empty = [&](int a) { return bars + 8u * (2 * L::kStages + 6 + a); };
    const uint32_t tmem_slot = bars + 8u * (2 * L::kStages + 8);
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (sbase & 1023u) {                      // every CTA alike
        if (tid == 0) atomicOr(g.status, 2u);
        return;
    }
    if (tid == 0) {
        for (int s = 0; s < L::kStages; ++s) {
            mbar_init(full(s), 1);            // the copying lane (and its bytes)
            mbar_init(empty(s), 1);           // the tensor core's commit
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(acc_full(a), 1);
            mbar_init(acc_empty(a), 4);       // the four storing warps
            mbar_init(sf_full(a), 4);         // the four scale warps
            mbar_init(sf_empty(a), 1);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(tmem_slot), "r"((uint32_t)L::kCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(gm_smem + L::kBar + 8 * (2 * L::kStages + 8));
    const int n_tiles = g.tiles_m * g.tiles_x;
    const int all_steps = (g.blocks + kGmBlocks - 1) / kGmBlocks;
    // this CTA's tiles, and its part of their rows in stages: pairs of stages dealt to the cluster
    const int rank = (int)blockIdx.x % g.split, tile0 = (int)blockIdx.x / g.split, tile_step = (int)gridDim.x / g.split;
    const int pairs = (all_steps + 1) / 2;
    const int k_begin = 2 * (pairs * rank / g.split);
    const int n_step = min(2 * (pairs * (rank + 1) / g.split), all_steps) - k_begin;
    // Ask L2 for the first stages' rows of m while the kernel in front still runs (harmless: its writes
    // land in L2 too).  16384 x 16384 x 16 27.0 -> 25.6 us.
    if (!DIGITS && warp == 0 && lane == 0 && tile0 < n_tiles)
        for (int k = 0; k < min(L::kStages, n_step); ++k)
            tma_prefetch_2d(&map_m, (k_begin + k) * kGmBox, (tile0 / g.tiles_x) * kGmRows);
    __syncwarp();
    // Operands and result may be the previous kernel's -- but for the matrix of dense vectors: that
    // kernel is mx_digits_kernel, which starts this one when all before it is done.
    if (!DIGITS || warp != 0) asm volatile("griddepcontrol.wait;" ::: "memory");

    if (warp == 0) {
        if (lane == 0) {
            bool ok = true;
            int it = 0, early = 0;               // stages so far; those whose rows of m are on their way already
            if (DIGITS) {
                early = tile0 < n_tiles ? min(L::kStages, n_step) : 0;
                for (int k = 0; k < early; ++k) {
                    mbar_arrive_expect_tx(full(k), (uint32_t)(L::kA + L::kB));
                    tma_load_2d(sbase + k * (L::kA + L::kB), &map_m, (k_begin + k) * kGmBox, (tile0 / g.tiles_x) * kGmRows, full(k));
                }
                asm volatile("griddepcontrol.wait;" ::: "memory");
            }
            for (int tile = tile0; tile < n_tiles && ok; tile += tile_step) {
                const int m0 = (tile / g.tiles_x) * kGmRows, x0 = (tile % g.tiles_x) * NT;
                for (int k = 0; k < n_step && ok; ++k, ++it) {
                    const int s = it % L::kStages;
                    if (it >= L::kStages) ok = mbar_wait(empty(s), (uint32_t)((it / L::kStages - 1) & 1), g.status);
                    const uint32_t at = sbase + s * (L::kA + L::kB);
                    if (it >= early) {
                        mbar_arrive_expect_tx(full(s), (uint32_t)(L::kA + L::kB));
                        tma_load_2d(at, &map_m, (k_begin + k) * kGmBox, m0, full(s));
                    }
                    tma_load_2d(at + L::kA, &map_x, (k_begin + k) * kGmBox, x0, full(s));
                }
            }
            // whoever gave up: shared memory outlives what was asked for
            for (int i = max(it - L::kStages, 0); i < it; ++i)
                mbar_wait(full(i % L::kStages), (uint32_t)((i / L::kStages) & 1), g.status);
        }
        __syncwarp();
    } else if (warp == 1) {
        // The whole warp walks the stages (uniform control flow and addresses); one elected lane issues.
        const bool leader = elect_one();
        bool ok = true;
        int s = 0, done = 0, grp = 0;          // ring slot, tiles, scale groups so far
        uint32_t phase = 0;
        const uint64_t desc_a = tc_desc_swizzled(sbase, 1024, 2), desc_sf = tc_desc(sbase + L::kSf, 128, 128);
        for (int tile = tile0; tile < n_tiles && ok; tile += tile_step, ++done) {
            const int a = done & 1;
            if (done >= 2) ok = mbar_wait(acc_empty(a), (uint32_t)((done / 2 - 1) & 1), g.status);
            for (int k = 0; k < n_step && ok; ++k) {
                if (k % kGmGroup == 0) ok = mbar_wait(sf_full(grp & 1), (uint32_t)((grp / 2) & 1), g.status);
                ok = ok && mbar_wait(full(s), phase, g.status);
                tc_fence_after();
                // descriptors count in 16-byte units
                const uint64_t at = desc_a + (uint32_t)(s * ((L::kA + L::kB) / 16));
                const uint64_t sf = desc_sf + (uint32_t)((grp & 1) * (L::kSfGroup / 16) + (k % kGmGroup) * (L::kSfStage / 16));
                const uint32_t sfa = tmem + L::kSfCol + (k & 1) * (L::kSfColsA + L::kSfColsB), sfb = sfa + L::kSfColsA;
                const uint32_t d = tmem + NT * a;
                const bool last = k == n_step - 1;
                if (leader) {
#pragma unroll
                    for (int p = 0; p < 2 + 2 * L::kRowAtoms; ++p) gm_copy_scales(sfa + 4 * p, sf + 32 * p);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        gm_mma(d, at + 2 * j, at + L::kA / 16 + 2 * j, j & 1 ? gm_idesc<NT>(2) : gm_idesc<NT>(0),
                               sfa + 4 * (j / 2), sfb + 4 * L::kRowAtoms * (j / 2), k > 0 || j > 0);
                    tc_commit(empty(s));
                    if (k % kGmGroup == kGmGroup - 1 || last) tc_commit(sf_empty(grp & 1));
                    if (last) tc_commit(acc_full(a));
                }
                __syncwarp();
                if (k % kGmGroup == kGmGroup - 1 || last) ++grp;
                if (++s == L::kStages) s = 0, phase ^= 1;
            }
        }
    } else if (warp < 6) {
        // A thread takes row i of m's tile and rows i (and i + 128) of x's; the rows are dealt so that a
        // warp's words are 128 consecutive bytes of a piece.  A group's loads are issued before the
        // wait for the room of the one before it: the fence between that one's stores and the products
        // waits for loads too, and then they have arrived.
        const int i = (lane & 7) + 8 * (warp - 2) + 32 * (lane >> 3);
        const int at = (i & 31) * 16 + (i >> 5) * 4;
        const unsigned char* m_all = g.m_scales + (long long)g.M * g.blocks;
        const unsigned char* x_all = g.x_scales + (long long)g.batch * g.blocks;
        uint32_t q[2][1 + L::kRowAtoms][8];
        auto load = [&](uint32_t (&q)[1 + L::kRowAtoms][8], int tile, int k) {
            const int m = (tile / g.tiles_x) * kGmRows + i, x = (tile % g.tiles_x) * NT + i;
            const bool there = tile < n_tiles;
#pragma unroll
            for (int p = 0; p <= L::kRowAtoms; ++p) {
                const bool mine = p == 0 ? m < g.M : i + 128 * (p - 1) < NT && x + 128 * (p - 1) < g.batch;
                if (there && mine) {
                    const unsigned char* row = p == 0 ? g.m_scales + (long long)m * g.blocks
                                                      : g.x_scales + (long long)(x + 128 * (p - 1)) * g.blocks;
                    gm_load_scales(q[p], row, (k_begin + k) * kGmBlocks, g.blocks, g.align, p == 0 ? g.m_scales : g.x_scales,
                                   p == 0 ? m_all : x_all);
                } else {
#pragma unroll
                    for (int w = 0; w < 8; ++w) q[p][w] = 0u;
                }
            }
        };
        bool ok = true;
        int grp = 0, l_tile = tile0, l_k = 0;
        auto load_next = [&](uint32_t (&q)[1 + L::kRowAtoms][8]) {
            load(q, l_tile, l_k);
            if ((l_k += kGmGroup) >= n_step) l_k = 0, l_tile += tile_step;
        };
        load_next(q[0]);
        const int n_grp = tile0 < n_tiles ? ((n_tiles - tile0 - 1) / tile_step + 1) * ((n_step + kGmGroup - 1) / kGmGroup) : 0;
        for (int g0 = 0; g0 < n_grp && ok; g0 += 2) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                if (grp < n_grp && ok) {
                    load_next(q[u ^ 1]);
                    if (grp >= 2) ok = mbar_wait(sf_empty(u), (uint32_t)((grp / 2 - 1) & 1), g.status);
                    unsigned char* sf = gm_smem + L::kSf + u * L::kSfGroup + at;
#pragma unroll
                    for (int w = 0; w < 8; ++w) {    // word w: four blocks, half a stage
                        unsigned char* to = sf + (w / 2) * L::kSfStage;
                        *reinterpret_cast<uint32_t*>(to + 512 * (w & 1)) = q[u][0][w];
#pragma unroll
                        for (int p = 0; p < L::kRowAtoms; ++p)
                            *reinterpret_cast<uint32_t*>(to + 512 * (2 + L::kRowAtoms * (w & 1) + p)) = q[u][1 + p][w];
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(sf_full(u));
                    ++grp;
                }
            }
        }
    }
    typedef typename MxElem<OUT>::type E;
    constexpr int kSums = DIGITS ? NT / kGmDigits : NT;      // results of a row of m in a tile
    E* out = reinterpret_cast<E*>(g.out);
    const int w = warp & 3;                      // the quarter of tensor memory a storing warp can read
    const int sums_all = DIGITS ? g.batch / kGmDigits : g.batch;
    uint32_t repair = 0u;                        // vectors of this tile that hold an infinity or a NaN
    if (warp >= 6 && g.split == 1) {
        constexpr int kPiece = kGmPiece / (32 * (int)sizeof(E));
        int done = 0, pieces = 0;
        bool ok = true;
        for (int tile = tile0; tile < n_tiles && ok; tile += tile_step, ++done) {
            const int a = done & 1;
            const int m = (tile / g.tiles_x) * kGmRows + w * 32 + lane, x0 = (tile % g.tiles_x) * kSums;
            if (DIGITS) repair = gm_find_not_finite<kSums>(g, x0, lane);
            ok = mbar_wait(acc_full(a), (uint32_t)((done / 2) & 1), g.status);
            ok = __all_sync(0xFFFFFFFFu, ok);
            tc_fence_after();
            const uint32_t from = tmem + NT * a + ((uint32_t)(w * 32) << 16);
            if constexpr (DIGITS) {
#pragma unroll 1
                for (int c = 0; c < kSums; ++c) {
                    if (x0 + c >= sums_all) break;
                    float r = gm_add_digits(from + kGmDigits * c);
                    if (ok && m < g.M) {
                        if ((repair >> c) & 1) r = gm_not_finite(g, m, x0 + c);
                        out[(long long)(x0 + c) * g.M + m] = r;
                    }
                }
            } else {
#pragma unroll 1
                for (int c = 0; c < NT; c += kPiece) {
                    if (x0 + c >= g.batch) break;
                    float r[kPiece];
                    tmem_ld<kPiece>(from + c, r);
                    if (g.bulk) {
                        // [kPiece rows of x][32 of m] through shared memory; rows outside the result are not written
                        const uint32_t at = L::kOut + (w * 2 + (pieces & 1)) * kGmPiece;
                        E* to = reinterpret_cast<E*>(gm_smem + at) + lane;
                        if (lane == 0) bulk_wait_read<1>();      // the piece before the last has been read
                        __syncwarp();
#pragma unroll
                        for (int v = 0; v < kPiece; ++v) to[32 * v] = MxElem<OUT>::put(r[v]);
                        fence_proxy_async_smem();
                        __syncwarp();
                        if (lane == 0 && ok && m - lane < g.M) tma_store_2d(&map_out, sbase + at, m - lane, x0 + c);
                        if (lane == 0) bulk_commit();
                        ++pieces;
                    } else if (ok && m < g.M) {
                        E* to = out + (long long)(x0 + c) * g.M + m;
#pragma unroll
                        for (int v = 0; v < kPiece; ++v)
                            if (x0 + c + v < g.batch) to[(long long)v * g.M] = MxElem<OUT>::put(r[v]);
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(acc_empty(a));
        }
        if (!DIGITS && lane == 0) bulk_wait<0>();           // shared memory and the result outlive the copies
    }
    if (g.split > 1) {
        // One tile per cluster.  Column c of the result is rank c % split's: every CTA sends its partial
        // sums there, to [c / split][sender][128 rows] in the place of the operands, which
        // every CTA's products have read behind the first barrier.  Stores, not loads: nothing waits
        // for a round trip.
        const int m = (tile0 / g.tiles_x) * kGmRows + w * 32 + lane, x0 = (tile0 % g.tiles_x) * kSums;
        const int sums = min(kSums, sums_all - x0);
        const uint32_t part = sbase + (w * 32 + lane) * 4;
        bool ok = true;
        if (warp >= 6) {
            if (DIGITS) repair = gm_find_not_finite<kSums>(g, x0, lane);
            ok = mbar_wait(acc_full(0), 0u, g.status);
            ok = __all_sync(0xFFFFFFFFu, ok);
            tc_fence_after();
        }
        __syncwarp();
        cluster_sync();
        if (warp >= 6) {
            const uint32_t from = tmem + ((uint32_t)(w * 32) << 16);
            const uint32_t row = (uint32_t)rank * (kGmRows * 4), shift = (uint32_t)(31 - __clz(g.split));
            if constexpr (DIGITS) {
                for (int c = 0; c < sums; ++c)
                    st_cluster_f32(map_cluster(part + ((uint32_t)(c >> shift) << shift) * (kGmRows * 4) + row, (uint32_t)(c & (g.split - 1))),
                                   gm_add_digits(from + kGmDigits * c));
            } else {
#pragma unroll 1
                for (int c = 0; c < NT; c += 16) {
                    if (c >= sums) break;
                    float r[16];
                    tmem_ld<16>(from + c, r);
#pragma unroll
                    for (int v = 0; v < 16; ++v)
                        if (c + v < sums)
                            st_cluster_f32(map_cluster(part + ((uint32_t)((c + v) >> shift) << shift) * (kGmRows * 4) + row,
                                                       (uint32_t)((c + v) & (g.split - 1))), r[v]);
                }
            }
        }
        __syncwarp();
        cluster_sync();
        if (warp >= 6) {
            const float* mine = reinterpret_cast<const float*>(gm_smem) + w * 32 + lane;
            const int n_mine = (sums - rank + g.split - 1) / g.split;
            for (int i = 0; i < n_mine; i += 8) {        // eight columns at a time: their loads overlap
                float r[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) r[e] = i + e < n_mine ? mine[(i + e) * g.split * kGmRows] : 0.f;
                for (int p = 1; p < g.split; ++p)
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (i + e < n_mine) r[e] += mine[((i + e) * g.split + p) * kGmRows];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int c = rank + (i + e) * g.split;
                    if (i + e < n_mine && ok && m < g.M) {
                        if (DIGITS && ((repair >> c) & 1)) r[e] = gm_not_finite(g, m, x0 + c);
                        out[(long long)(x0 + c) * g.M + m] = MxElem<OUT>::put(r[e]);
                    }
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)L::kCols) : "memory");
    }
}

}  // namespace feather
