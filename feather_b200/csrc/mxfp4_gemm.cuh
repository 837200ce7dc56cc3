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

template <int NT, int CHAINS>
struct GmLayout {
    static constexpr int kRowAtoms = NT > 128 ? 2 : 1;                     // 128-row pieces of x's scales
    static constexpr int kA = kGmRows * kGmBox, kB = NT * kGmBox;          // operand bytes of a stage
    static constexpr int kSfStage = 2 * (1 + kRowAtoms) * 512;             // scale bytes of a stage: 2 x (m, x)
    static constexpr int kSfGroup = kGmGroup * kSfStage;
    static constexpr int kMost = (227 * 1024 - 256 - 2 * kSfGroup - kGmOutBytes) / (kA + kB);
    static constexpr int kStages = kMost > 8 ? 8 : kMost;
    static constexpr int kSf = kStages * (kA + kB);                        // two groups of scales behind the operands
    static constexpr int kOut = kSf + 2 * kSfGroup;                        // pieces of the result on their way out
    static constexpr int kBar = kOut + kGmOutBytes;
    static constexpr int kBytes = kBar + 8 * (2 * kStages + 8) + 16;
    static constexpr int kAccCols = NT * CHAINS;
    static constexpr int kSfColsA = 2 * 4, kSfColsB = 2 * 4 * kRowAtoms;   // 32-bit columns of a stage's scales
    static constexpr int kSfCol = 2 * kAccCols;                            // two sets alternate
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
__device__ __forceinline__ void gm_load_scales(uint32_t (&w)[8], const unsigned char* row, int k, int blocks, int align) {
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
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            w[i] = 0u;
#pragma unroll
            for (int b = 0; b < 4; ++b)
                if (k + 4 * i + b < blocks) w[i] |= (uint32_t)__ldg(row + k + 4 * i + b) << (8 * b);
        }
    }
}

struct MxGemmArgs {
    const unsigned char* m_scales;
    const unsigned char* x_scales;
    void* out;                    // batch x M
    int M, batch, blocks;
    int tiles_m, tiles_x;
    int align;                    // of the scale rows: 16, 4 or 1
    int bulk;                     // 1: result rows are 16-byte aligned, pieces leave by tensor-map copies
    unsigned int* status;
};

template <int NT, int CHAINS, int OUT>
__global__ void __launch_bounds__(kGmThreads, 1)
mx_gemm_kernel(const __grid_constant__ CUtensorMap map_m, const __grid_constant__ CUtensorMap map_x,
               const __grid_constant__ CUtensorMap map_out, const MxGemmArgs g) {
    typedef GmLayout<NT, CHAINS> L;
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
    asm volatile("griddepcontrol.wait;" ::: "memory");   // operands and result may be the previous kernel's

    const int n_tiles = g.tiles_m * g.tiles_x;
    const int n_step = (g.blocks + kGmBlocks - 1) / kGmBlocks;
    if (warp == 0) {
        if (lane == 0) {
            bool ok = true;
            int it = 0;
            for (int tile = blockIdx.x; tile < n_tiles && ok; tile += gridDim.x) {
                const int m0 = (tile / g.tiles_x) * kGmRows, x0 = (tile % g.tiles_x) * NT;
                for (int k = 0; k < n_step && ok; ++k, ++it) {
                    const int s = it % L::kStages;
                    if (it >= L::kStages) ok = mbar_wait(empty(s), (uint32_t)((it / L::kStages - 1) & 1), g.status);
                    mbar_arrive_expect_tx(full(s), (uint32_t)(L::kA + L::kB));
                    const uint32_t at = sbase + s * (L::kA + L::kB);
                    tma_load_2d(at, &map_m, k * kGmBox, m0, full(s));
                    tma_load_2d(at + L::kA, &map_x, k * kGmBox, x0, full(s));
                }
            }
        }
    } else if (warp == 1) {
        // The whole warp walks the stages (uniform control flow and addresses); one elected lane issues.
        const bool leader = elect_one();
        bool ok = true;
        int s = 0, done = 0, grp = 0;          // ring slot, tiles, scale groups so far
        uint32_t phase = 0;
        const uint64_t desc_a = tc_desc_swizzled(sbase, 1024, 2), desc_sf = tc_desc(sbase + L::kSf, 128, 128);
        for (int tile = blockIdx.x; tile < n_tiles && ok; tile += gridDim.x, ++done) {
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
                const uint32_t d = tmem + NT * (CHAINS * a + k % CHAINS);
                const bool last = k == n_step - 1;
                if (leader) {
#pragma unroll
                    for (int p = 0; p < 2 + 2 * L::kRowAtoms; ++p) gm_copy_scales(sfa + 4 * p, sf + 32 * p);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        gm_mma(d, at + 2 * j, at + L::kA / 16 + 2 * j, j & 1 ? gm_idesc<NT>(2) : gm_idesc<NT>(0),
                               sfa + 4 * (j / 2), sfb + 4 * L::kRowAtoms * (j / 2), k >= CHAINS || j > 0);
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
        // thread i: row i of m's tile, rows i (and i + 128) of x's.  The loads of the next group are
        // issued behind the fence of this one: the fence would wait for them.
        const int i = tid - 64;
        const int at = (i & 31) * 16 + (i >> 5) * 4;
        uint32_t q[1 + L::kRowAtoms][8];
        auto load = [&](int tile, int k) {
            const int m = (tile / g.tiles_x) * kGmRows + i, x = (tile % g.tiles_x) * NT + i;
            const bool there = tile < n_tiles;
#pragma unroll
            for (int p = 0; p <= L::kRowAtoms; ++p) {
                const bool mine = p == 0 ? m < g.M : i + 128 * (p - 1) < NT && x + 128 * (p - 1) < g.batch;
                if (there && mine) {
                    const unsigned char* row = p == 0 ? g.m_scales + (long long)m * g.blocks
                                                      : g.x_scales + (long long)(x + 128 * (p - 1)) * g.blocks;
                    gm_load_scales(q[p], row, k * kGmBlocks, g.blocks, g.align);
                } else {
#pragma unroll
                    for (int w = 0; w < 8; ++w) q[p][w] = 0u;
                }
            }
        };
        bool ok = true;
        int grp = 0;
        load(blockIdx.x, 0);
        for (int tile = blockIdx.x; tile < n_tiles && ok; tile += gridDim.x) {
            for (int k = 0; k < n_step && ok; k += kGmGroup, ++grp) {
                if (grp >= 2) ok = mbar_wait(sf_empty(grp & 1), (uint32_t)((grp / 2 - 1) & 1), g.status);
                unsigned char* sf = gm_smem + L::kSf + (grp & 1) * L::kSfGroup + at;
#pragma unroll
                for (int w = 0; w < 8; ++w) {    // word w: four blocks, half a stage
                    unsigned char* to = sf + (w / 2) * L::kSfStage;
                    *reinterpret_cast<uint32_t*>(to + 512 * (w & 1)) = q[0][w];
#pragma unroll
                    for (int p = 0; p < L::kRowAtoms; ++p)
                        *reinterpret_cast<uint32_t*>(to + 512 * (2 + L::kRowAtoms * (w & 1) + p)) = q[1 + p][w];
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(sf_full(grp & 1));
                if (k + kGmGroup < n_step) load(tile, k + kGmGroup);
                else load(tile + gridDim.x, 0);
            }
        }
    } else {
        const int w = warp & 3;                  // the quarter of tensor memory this warp can read
        typedef typename MxElem<OUT>::type E;
        constexpr int kPiece = kGmPiece / (32 * (int)sizeof(E));
        E* out = reinterpret_cast<E*>(g.out);
        int done = 0, pieces = 0;
        bool ok = true;
        for (int tile = blockIdx.x; tile < n_tiles && ok; tile += gridDim.x, ++done) {
            const int a = done & 1;
            const int m = (tile / g.tiles_x) * kGmRows + w * 32 + lane, x0 = (tile % g.tiles_x) * NT;
            ok = mbar_wait(acc_full(a), (uint32_t)((done / 2) & 1), g.status);
            ok = __all_sync(0xFFFFFFFFu, ok);
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < NT; c += kPiece) {
                if (x0 + c >= g.batch) break;
                float r[kPiece];
                const uint32_t from = tmem + NT * CHAINS * a + c + ((uint32_t)(w * 32) << 16);
                tmem_ld<kPiece>(from, r);
#pragma unroll
                for (int h = 1; h < CHAINS; ++h) {
                    if (h < n_step) {            // the chains that this row length reaches
                        float more[kPiece];
                        tmem_ld<kPiece>(from + NT * h, more);
#pragma unroll
                        for (int v = 0; v < kPiece; ++v) r[v] += more[v];
                    }
                }
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
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(acc_empty(a));
        }
        if (lane == 0) bulk_wait<0>();           // shared memory and the result outlive the copies
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)L::kCols) : "memory");
    }
}

}  // namespace feather
