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
// stage, kGmAhead stages ahead) and store them in that order.
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
constexpr int kGmAhead = 4;                    // stages the scale loads run ahead

template <int NT, int CHAINS>
struct GmLayout {
    static constexpr int kRowAtoms = NT > 128 ? 2 : 1;                     // 128-row pieces of x's scales
    static constexpr int kA = kGmRows * kGmBox, kB = NT * kGmBox;          // operand bytes of a stage
    static constexpr int kSfA = 2 * 512, kSfB = 2 * kRowAtoms * 512;       // scale bytes of a stage
    static constexpr int kStage = kA + kB + kSfA + kSfB;
    static constexpr int kMost = (227 * 1024 - 256) / kStage;
    static constexpr int kStages = kMost > 8 ? 8 : kMost;
    static constexpr int kSf = kStages * (kA + kB);                        // scales behind all operands
    static constexpr int kBar = kSf + kStages * (kSfA + kSfB);
    static constexpr int kBytes = kBar + 8 * (2 * kStages + 4) + 16;
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
// 512 bytes (32 rows of 16) of shared memory to four columns of tensor memory, the same in
// every quarter of the lanes.
__device__ __forceinline__ void gm_copy_scales(uint32_t taddr, uint64_t desc) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

// Eight scale bytes of blocks [k, k + 8) of a row, those past the row's end as 0.
__device__ __forceinline__ uint2 gm_load_scales(const unsigned char* row, int k, int blocks, int align) {
    uint2 r = make_uint2(0u, 0u);
    if (align == 8) {                            // whole rows in steps of 8 blocks
        r = __ldg(reinterpret_cast<const uint2*>(row + k));
    } else if (align == 4) {
        r.x = __ldg(reinterpret_cast<const uint32_t*>(row + k));
        if (k + 4 < blocks) r.y = __ldg(reinterpret_cast<const uint32_t*>(row + k) + 1);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (k + i < blocks) r.x |= (uint32_t)__ldg(row + k + i) << (8 * i);
            if (k + 4 + i < blocks) r.y |= (uint32_t)__ldg(row + k + 4 + i) << (8 * i);
        }
    }
    return r;
}

struct MxGemmArgs {
    const unsigned char* m_scales;
    const unsigned char* x_scales;
    void* out;                    // batch x M
    int M, batch, blocks;
    int tiles_m, tiles_x;
    int align;                    // of the scale rows: 8, 4 or 1
    unsigned int* status;
};

template <int NT, int CHAINS, int OUT>
__global__ void __launch_bounds__(kGmThreads, 1)
mx_gemm_kernel(const __grid_constant__ CUtensorMap map_m, const __grid_constant__ CUtensorMap map_x, const MxGemmArgs g) {
    typedef GmLayout<NT, CHAINS> L;
    extern __shared__ __align__(1024) unsigned char gm_smem[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t sbase = smem_u32(gm_smem), bars = sbase + L::kBar;
    auto full = [&](int s) { return bars + 8u * s; };
    auto empty = [&](int s) { return bars + 8u * (L::kStages + s); };
    auto acc_full = [&](int a) { return bars + 8u * (2 * L::kStages + a); };
    auto acc_empty = [&](int a) { return bars + 8u * (2 * L::kStages + 2 + a); };
    const uint32_t tmem_slot = bars + 8u * (2 * L::kStages + 4);
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (sbase & 1023u) {                      // every CTA alike
        if (tid == 0) atomicOr(g.status, 2u);
        return;
    }
    if (tid == 0) {
        for (int s = 0; s < L::kStages; ++s) {
            mbar_init(full(s), 1 + 4);        // the copying lane (and its bytes), four scale warps
            mbar_init(empty(s), 1);           // the tensor core's commit
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(acc_full(a), 1);
            mbar_init(acc_empty(a), 4);       // the four storing warps
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
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(gm_smem + L::kBar + 8 * (2 * L::kStages + 4));
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
        if (lane == 0) {
            bool ok = true;
            int it = 0, done = 0;
            for (int tile = blockIdx.x; tile < n_tiles && ok; tile += gridDim.x, ++done) {
                const int a = done & 1;
                if (done >= 2) ok = mbar_wait(acc_empty(a), (uint32_t)((done / 2 - 1) & 1), g.status);
                tc_fence_after();
                for (int k = 0; k < n_step && ok; ++k, ++it) {
                    const int s = it % L::kStages;
                    ok = mbar_wait(full(s), (uint32_t)((it / L::kStages) & 1), g.status);
                    tc_fence_after();
                    const uint32_t at = sbase + s * (L::kA + L::kB);
                    const uint32_t sf = sbase + L::kSf + s * (L::kSfA + L::kSfB);
                    const uint32_t sfa = tmem + L::kSfCol + (it & 1) * (L::kSfColsA + L::kSfColsB), sfb = sfa + L::kSfColsA;
#pragma unroll
                    for (int p = 0; p < 2; ++p) gm_copy_scales(sfa + 4 * p, tc_desc(sf + 512 * p, 128, 128));
#pragma unroll
                    for (int p = 0; p < 2 * L::kRowAtoms; ++p)
                        gm_copy_scales(sfb + 4 * p, tc_desc(sf + L::kSfA + 512 * p, 128, 128));
                    const uint32_t d = tmem + NT * (CHAINS * a + k % CHAINS);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        gm_mma(d, tc_desc_swizzled(at + 32 * j, 1024, 2), tc_desc_swizzled(at + L::kA + 32 * j, 1024, 2),
                               j & 1 ? gm_idesc<NT>(2) : gm_idesc<NT>(0), sfa + 4 * (j / 2),
                               sfb + 4 * L::kRowAtoms * (j / 2), k >= CHAINS || j > 0);
                    tc_commit(empty(s));
                }
                tc_commit(acc_full(a));
            }
        }
    } else if (warp < 6) {
        // thread i: row i of m's tile, rows i (and i + 128) of x's
        const int i = tid - 64;
        const int at = (i & 31) * 16 + (i >> 5) * 4;
        struct Cursor { int tile, k; } ahead{(int)blockIdx.x, 0}, now{(int)blockIdx.x, 0};
        auto step = [&](Cursor& c) {
            if (++c.k == n_step) c.k = 0, c.tile += gridDim.x;
        };
        uint2 q[kGmAhead][1 + L::kRowAtoms];
        auto load = [&](uint2 (&r)[1 + L::kRowAtoms]) {
            const int m = (ahead.tile / g.tiles_x) * kGmRows + i, x = (ahead.tile % g.tiles_x) * NT + i;
#pragma unroll
            for (int p = 0; p <= L::kRowAtoms; ++p) r[p] = make_uint2(0u, 0u);
            if (ahead.tile < n_tiles) {
                if (m < g.M) r[0] = gm_load_scales(g.m_scales + (long long)m * g.blocks, ahead.k * kGmBlocks, g.blocks, g.align);
#pragma unroll
                for (int p = 0; p < L::kRowAtoms; ++p)
                    if (i + 128 * p < NT && x + 128 * p < g.batch)
                        r[1 + p] = gm_load_scales(g.x_scales + (long long)(x + 128 * p) * g.blocks, ahead.k * kGmBlocks,
                                                  g.blocks, g.align);
                step(ahead);
            }
        };
#pragma unroll
        for (int u = 0; u < kGmAhead; ++u) load(q[u]);
        bool ok = true;
        for (int it = 0; now.tile < n_tiles && ok;) {
#pragma unroll
            for (int u = 0; u < kGmAhead; ++u) {
                if (now.tile < n_tiles && ok) {
                    const int s = it % L::kStages;
                    if (it >= L::kStages) ok = mbar_wait(empty(s), (uint32_t)((it / L::kStages - 1) & 1), g.status);
                    unsigned char* sf = gm_smem + L::kSf + s * (L::kSfA + L::kSfB) + at;
                    *reinterpret_cast<uint32_t*>(sf) = q[u][0].x;
                    *reinterpret_cast<uint32_t*>(sf + 512) = q[u][0].y;
#pragma unroll
                    for (int p = 0; p < L::kRowAtoms; ++p) {
                        *reinterpret_cast<uint32_t*>(sf + L::kSfA + 512 * p) = q[u][1 + p].x;
                        *reinterpret_cast<uint32_t*>(sf + L::kSfA + 512 * (L::kRowAtoms + p)) = q[u][1 + p].y;
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(full(s));
                    load(q[u]);
                    step(now);
                    ++it;
                }
            }
        }
    } else {
        const int w = warp & 3;                  // the quarter of tensor memory this warp can read
        typedef typename MxElem<OUT>::type E;
        E* out = reinterpret_cast<E*>(g.out);
        int done = 0;
        bool ok = true;
        for (int tile = blockIdx.x; tile < n_tiles && ok; tile += gridDim.x, ++done) {
            const int a = done & 1;
            const int m = (tile / g.tiles_x) * kGmRows + w * 32 + lane, x0 = (tile % g.tiles_x) * NT;
            ok = mbar_wait(acc_full(a), (uint32_t)((done / 2) & 1), g.status);
            ok = __all_sync(0xFFFFFFFFu, ok);
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < NT; c += 32) {
                if (x0 + c >= g.batch) break;
                float r[32];
                const uint32_t from = tmem + NT * CHAINS * a + c + ((uint32_t)(w * 32) << 16);
                tmem_ld<32>(from, r);
#pragma unroll
                for (int h = 1; h < CHAINS; ++h) {
                    if (h < n_step) {            // the chains that this row length reaches
                        float more[32];
                        tmem_ld<32>(from + NT * h, more);
#pragma unroll
                        for (int v = 0; v < 32; ++v) r[v] += more[v];
                    }
                }
                if (ok && m < g.M) {
                    E* to = out + (long long)(x0 + c) * g.M + m;
#pragma unroll
                    for (int v = 0; v < 32; ++v)
                        if (x0 + c + v < g.batch) to[(long long)v * g.M] = MxElem<OUT>::put(r[v]);
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(acc_empty(a));
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
