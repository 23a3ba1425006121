// Product of two operands of 8-bit floats with a power-of-two scale for each block of 128 along the sum (tab_matmul_blocks_launch):
//   y[m][n] = sum over k of  a[m][k] 2^ea(m, k/128)  b[n][k] 2^eb(n, k/128).
//
// The scales are powers of two, so the tensor cores apply them themselves: tcgen05.mma kind::mxf8f6f4 multiplies 8-bit floats with an
// e8m0 scale for each 32 of them into fp32 accumulators, and a block of 128 is four such steps under one scale.  (With scales of any
// value, every 128 terms of the sum would have to leave the tensor memory for the vector units and be scaled and added there.)
//
// The scale bytes a step reads lie in tensor memory, 32 bits for each row of an operand: row r in lane r % 32 of column r / 32, repeated
// in the four lane quarters.  The byte within the 32 bits is chosen by the instruction, so one copy of 4 bytes for each row serves four
// blocks of 128, i.e. 512 terms.
#include <algorithm>
#include <cstdio>
#include <cuda.h>
#include <mutex>
#include "blocks_common.cuh"
#include "umma_common.cuh"

namespace tab {

// ---- block-scaled 8-bit MMAs -----------------------------------------------------------------------------------------------
// D fp32, A / B e4m3 (0) or e5m2 (1), both K-major, scales ue8m0.  The byte of the scale words is bits 4-5 (B) and 29-30 (A).
__host__ __device__ constexpr uint32_t umma_idesc_f8(int m, int n, int aformat, int bformat) {
    return ((uint32_t)aformat << 7) | ((uint32_t)bformat << 10) | ((uint32_t)(n >> 3) << 17) | (1u << 23) | ((uint32_t)(m >> 4) << 24);
}
__device__ __forceinline__ uint32_t with_scale_byte(uint32_t idesc, uint32_t j) { return idesc | (j << 4) | (j << 29); }
__device__ __forceinline__ void umma_f8(uint32_t tmem_d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\t"
                 "setp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.block32 [%0], %1, %2, %3, [%5], [%6], p;\n\t}"
                 :: "r"(tmem_d), "l"(da), "l"(db), "r"(idesc), "r"(accumulate), "r"(sfa), "r"(sfb) : "memory");
}
// 512 bytes of scales, [32][4 words] as described above, from shared memory to four columns of tensor memory.  The descriptor: no
// swizzle, 8-row groups of 16-byte rows 128 bytes apart.  Copies and MMAs of one thread execute in the order of their issue.
__device__ __forceinline__ void tmem_copy_scales(uint32_t taddr, uint32_t smem_addr) {
    const uint64_t d = ((uint64_t)((128u >> 4) | (1u << 14)) << 32) | ((smem_addr & 0x3FFFFu) >> 4);
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(d) : "memory");
}
__device__ __forceinline__ float ld_cluster_f32(uint32_t addr, uint32_t rank) {
    float v;
    asm volatile("{\n\t.reg .b32 ra;\n\tmapa.shared::cluster.u32 ra, %1, %2;\n\tld.shared::cluster.f32 %0, [ra];\n\t}" : "=f"(v) : "r"(addr), "r"(rank) : "memory");
    return v;
}

// Scale words (4 blocks from kb on, 127 = 2^0 where there is no block or row) of rows lane, lane + 32, lane + 64, lane + 96 of the 128
// from row0 on.  Only blocks below kb1 are read.
__device__ __forceinline__ uint4 load_scales(const BlocksOperand& o, int row0, int kb, int kb1, int lane) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if (i > 0 && o.shift) { w[i] = w[0]; continue; }                   // one scale for all 128 rows
        const int row = row0 + i * 32 + lane;
        const bool in = (o.shift ? row0 : row) < o.rows;
        const uint8_t* s = o.s + (long long)(o.shift ? row0 >> o.shift : row) * o.sr + (long long)kb * o.sk;
        uint32_t v = 0;
#pragma unroll
        for (int j = 0; j < 4; j++) v |= (in && kb + j < kb1 ? (uint32_t)s[j * o.sk] : 127u) << (8 * j);
        w[i] = v;
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// 32 accumulators of a row (columns c0 .. c0+31 of ncols) to row-major memory.
template <typename T>
__device__ __forceinline__ void store_row32(T* y, int c0, int ncols, bool vec, const float (&v)[32]) {
#pragma unroll
    for (int j = 0; j < 32; j += 8) {
        float t[8];
#pragma unroll
        for (int i = 0; i < 8; i++) t[i] = v[j + i];
        store8(y + c0 + j, ncols - (c0 + j), vec, t);
    }
}

static constexpr int TT = 256;                           // threads of a tile CTA
static constexpr int SF_SLOTS = 4;                       // scale words of 512 terms each, in shared memory

// One CTA: 128 rows of operand R times BN rows of operand C over this rank's share of the sum.  Warp 0 copies the operands, warp 1
// issues the MMAs, warp 2 brings the scales, warps 4-7 finish.  A cluster shares out the sum: rank r of S takes blocks
// [r * per, (r+1) * per), the partial results meet in shared memory and every rank adds its share of the columns, in the order of
// the ranks.  SWAP: R is b, the tile is transposed (few rows of a: the 128-row side of the MMA takes the weights).
template <int BN, bool SWAP, int TYPE>
__global__ void __launch_bounds__(TT) matmul_blocks_tile_kernel(const __grid_constant__ CUtensorMap tmR, const __grid_constant__ CUtensorMap tmC, BlocksOperand R, BlocksOperand C,
                                                                void* yv, long long ldy, int KB, int per, int nst, int tiles_c, int split, int vec, int* status) {
    using T = typename ElemOf<TYPE>::type;
    extern __shared__ uint8_t raw[];
    constexpr int STAGE = (128 + BN) * 128;
    constexpr int CG = (BN + 127) / 128;                                   // groups of 128 rows of C
    constexpr int SFB = 512 * (1 + CG);                                    // bytes of a slot of scales
    constexpr int SFCOL = BN < 32 ? 32 : BN;                               // first tensor-memory column of the scales: two slots
    constexpr int TCOLS = SFCOL + 8 * (1 + CG) <= 64 ? 64 : SFCOL + 8 * (1 + CG) <= 128 ? 128 : SFCOL + 8 * (1 + CG) <= 256 ? 256 : 512;
    __shared__ __align__(8) uint64_t bars[16 + 2 * SF_SLOTS + 1];
    __shared__ __align__(512) uint8_t sf[SF_SLOTS * SFB];
    __shared__ uint32_t tslot;
    __shared__ int dead_flag;
    volatile int* deadp = &dead_flag;
    const uint32_t sRing = ((uint32_t)__cvta_generic_to_shared(raw) + 1023u) & ~1023u;
    const uint32_t full = (uint32_t)__cvta_generic_to_shared(bars), empty = full + 64, sfFull = full + 128, sfEmpty = sfFull + 8 * SF_SLOTS, accFull = sfEmpty + 8 * SF_SLOTS;
    const uint32_t sSF = (uint32_t)__cvta_generic_to_shared(sf), slot_addr = (uint32_t)__cvta_generic_to_shared(&tslot);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = split > 1 ? (int)cluster_ctarank() : 0;
    const unsigned tile = blockIdx.x / (unsigned)split;
    const int r0 = (int)(tile / (unsigned)tiles_c) * 128, c0 = (int)(tile % (unsigned)tiles_c) * BN;
    const int kb0 = min(KB, rank * per), kb1 = min(KB, kb0 + per);

    if (tid == 0) {
        *deadp = 0;
        for (int s = 0; s < 8; s++) { mbar_init(full + 8 * s, 1); mbar_init(empty + 8 * s, 1); }
        for (int s = 0; s < SF_SLOTS; s++) { mbar_init(sfFull + 8 * s, 1); mbar_init(sfEmpty + 8 * s, 1); }
        mbar_init(accFull, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) tmem_alloc(slot_addr, TCOLS);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *static_cast<volatile uint32_t*>(&tslot);
    pdl_wait();
    auto expire = [&](int code) { if (lane == 0) { if (status) atomicExch(status, code); *deadp = 1; } };

    if (warp == 0) {
        for (int kb = kb0, g = 0; kb < kb1; kb++, g++) {
            const int s = g % nst;
            if (g >= nst && !mbar_wait_warp(empty + 8 * s, (g / nst - 1) & 1)) { expire(31); break; }
            if (elect_one()) {
                mbar_expect_tx(full + 8 * s, STAGE);
                tma_load_2d(sRing + s * STAGE, &tmR, kb * BLK, r0, full + 8 * s);
                tma_load_2d(sRing + s * STAGE + 128 * 128, &tmC, kb * BLK, c0, full + 8 * s);
            }
            __syncwarp();
        }
    } else if (warp == 1) {
        const uint32_t idesc = umma_idesc_f8(128, BN, R.format == TAB_E5M2, C.format == TAB_E5M2);
        bool dead = false;
        for (int kb = kb0, g = 0; kb < kb1; kb++, g++) {
            const int s = g % nst, q = g >> 2, j = g & 3;
            const uint32_t sfcol = tmem + SFCOL + (q & 1) * 4 * (1 + CG);
            if (j == 0) {
                const int slot = q % SF_SLOTS;
                if (!mbar_wait_warp(sfFull + 8 * slot, (q / SF_SLOTS) & 1)) { expire(32); dead = true; break; }
                tc_fence_after();
                if (elect_one()) {
#pragma unroll
                    for (int i = 0; i < 1 + CG; i++) tmem_copy_scales(sfcol + 4 * i, sSF + slot * SFB + 512 * i);
                    umma_commit(sfEmpty + 8 * slot);
                }
                __syncwarp();
            }
            if (!mbar_wait_warp(full + 8 * s, (g / nst) & 1)) { expire(33); dead = true; break; }
            tc_fence_after();
            if (elect_one()) {
                const uint64_t da = umma_desc(sRing + s * STAGE), db = umma_desc(sRing + s * STAGE + 128 * 128);
                const uint32_t id = with_scale_byte(idesc, j);
#pragma unroll
                for (int i = 0; i < 4; i++) umma_f8(tmem, da + 2 * i, db + 2 * i, id, sfcol, sfcol + 4, (g | i) != 0);
                umma_commit(empty + 8 * s);
                if (kb == kb1 - 1) umma_commit(accFull);
            }
            __syncwarp();
        }
        (void)dead;
    } else if (warp == 2) {
        const int groups = (kb1 - kb0 + 3) / 4;
        uint4 wr, wc[CG];
        auto fetch = [&](int q) {
            wr = load_scales(R, r0, kb0 + 4 * q, kb1, lane);
#pragma unroll
            for (int i = 0; i < CG; i++) wc[i] = load_scales(C, c0 + 128 * i, kb0 + 4 * q, kb1, lane);
        };
        if (groups > 0) fetch(0);
        for (int q = 0; q < groups; q++) {
            const int slot = q % SF_SLOTS;
            if (q >= SF_SLOTS && !mbar_wait_warp(sfEmpty + 8 * slot, (q / SF_SLOTS - 1) & 1)) { expire(34); break; }
            const uint32_t at = sSF + slot * SFB + lane * 16;
            sts_v4(at, wr.x, wr.y, wr.z, wr.w);
#pragma unroll
            for (int i = 0; i < CG; i++) sts_v4(at + 512 * (1 + i), wc[i].x, wc[i].y, wc[i].z, wc[i].w);
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(sfFull + 8 * slot);
            if (q + 1 < groups) fetch(q + 1);
        }
    }
    __syncwarp();
    // All of the CTA meet here when the accumulators are complete: nothing of the sum is under way any more, and the ring is free.
    if (kb1 > kb0 && !mbar_wait_warp(accFull, 0)) expire(35);
    tc_fence_after();
    T* y = static_cast<T*>(yv);
    const int quarter = (warp & 3) * 32, row = r0 + quarter + lane;
    const uint32_t taddr = tmem + ((uint32_t)quarter << 16);
    constexpr int LC = BN < 32 ? 16 : 32;                                  // columns of a step
    if (split == 1) {
        if (warp >= 4) {
#pragma unroll 1
            for (int cb = 0; cb < BN && c0 + cb < C.rows; cb += 32) {
                uint32_t v[32];
                tmem_ld32(taddr + cb, v);                                  // BN = 16: the columns behind the tile's are read and not used
                float o[32];
#pragma unroll
                for (int j = 0; j < 32; j++) o[j] = __uint_as_float(v[j]);
                if (row < R.rows) {
                    if (SWAP) {
#pragma unroll
                        for (int j = 0; j < LC; j++) if (c0 + cb + j < C.rows) y[(long long)(c0 + cb + j) * ldy + row] = from_float<T>(o[j]);
                    } else {
                        store_row32(y + (long long)row * ldy, c0 + cb, min(C.rows, c0 + BN), vec, o);
                    }
                }
            }
        }
    } else {
        // partial results, [column][128 rows] floats, in the ring; a rank without blocks contributes zeros
        float* part = reinterpret_cast<float*>(raw + (sRing - (uint32_t)__cvta_generic_to_shared(raw)));
        if (warp >= 4) {
#pragma unroll 1
            for (int cb = 0; cb < BN; cb += 32) {
                uint32_t v[32];
                tmem_ld32(taddr + cb, v);
#pragma unroll
                for (int j = 0; j < LC; j++) part[(cb + j) * 128 + quarter + lane] = kb1 > kb0 ? __uint_as_float(v[j]) : 0.f;
            }
        }
        cluster_sync_all();
        const int share = BN / split, cfirst = rank * share;               // columns this rank finishes
        const int rl = tid & 127, rr = r0 + rl;
        for (int c = cfirst + (tid >> 7); c < cfirst + share; c += 2) {
            float sum = 0.f;
            for (int i = 0; i < split; i++) sum += ld_cluster_f32(sRing + (uint32_t)(c * 128 + rl) * 4u, (uint32_t)i);
            if (rr < R.rows && c0 + c < C.rows) {
                if (SWAP) y[(long long)(c0 + c) * ldy + rr] = from_float<T>(sum);
                else y[(long long)rr * ldy + c0 + c] = from_float<T>(sum);
            }
        }
        cluster_sync_all();                                                // nobody reads this CTA's memory any more
    }
    tc_fence_before();
    __syncthreads();
    if (*deadp != 0) {
        // a wait ran out: copies and MMAs that may still be in flight get time to land before this CTA's memory is another's
        for (int i = 0; i < 200; i++) __nanosleep(1000);
        __syncthreads();
    }
    pdl_launch_dependents();
    if (warp == 1) tmem_dealloc(tmem, TCOLS);
}

// ---- host side ----------------------------------------------------------------------------------------------------------------
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static EncodeTiledFn blocks_encode_fn() {
    static EncodeTiledFn fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* ptr = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeTiledFn>(ptr);
    });
    return fn;
}
// [rows][K] bytes with pitch ld, boxes of 128 bytes x box_rows, 128-byte swizzle; what lies outside reads as 0.
static bool blocks_map(CUtensorMap* m, const BlocksOperand& o, int K, unsigned box_rows) {
    EncodeTiledFn fn = blocks_encode_fn();
    if (!fn) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)o.rows}, strides[1] = {(cuuint64_t)o.ld};
    const cuuint32_t box[2] = {128, box_rows}, estr[2] = {1, 1};
    return fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(o.q), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

static thread_local char g_last_blocks_kernel[96] = "none";
const char* matmul_blocks_last_kernel() { return g_last_blocks_kernel; }

struct BlocksPlan { int bn; bool swap; int split, per, nst; };

template <int BN, bool SWAP, int TYPE>
static int launch_tile(const MatmulBlocksParams& p, const BlocksPlan& pl, int* status, cudaStream_t stream) {
    auto kernel = matmul_blocks_tile_kernel<BN, SWAP, TYPE>;
    const BlocksOperand &R = SWAP ? p.b : p.a, &C = SWAP ? p.a : p.b;
    alignas(64) CUtensorMap tmR, tmC;
    if (!blocks_map(&tmR, R, p.K, 128) || !blocks_map(&tmC, C, p.K, BN)) return TAB_E_TOO_LARGE;
    static std::mutex mu;
    static bool configured[64] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return record_cuda_error(e);
    const int smem = std::max(pl.nst * (128 + BN) * 128, pl.split > 1 ? BN * 512 : 0) + 1024;
    {
        std::lock_guard<std::mutex> lock(mu);
        if (dev < 0 || dev >= 64 || !configured[dev]) {
            e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 220 * 1024);
            if (e != cudaSuccess) return record_cuda_error(e);
            if (dev >= 0 && dev < 64) configured[dev] = true;
        }
    }
    const long long tiles_r = (R.rows + 127) / 128, tiles_c = ((long long)C.rows + BN - 1) / BN, grid = tiles_r * tiles_c * pl.split;
    if (grid >= (1LL << 31)) return TAB_E_TOO_LARGE;
    const int size = p.type == TAB_FP32 ? 4 : 2;
    const int vec = !(reinterpret_cast<uintptr_t>(p.y) & (8 * size - 1)) && p.ldy % 8 == 0;
    snprintf(g_last_blocks_kernel, sizeof(g_last_blocks_kernel), "matmul_blocks_tile_kernel<%d,%d> split %d stages %d", BN, (int)SWAP, pl.split, pl.nst);
    return launch_pdl_as(false, (unsigned)pl.split, kernel, dim3((unsigned)grid), dim3(TT), (size_t)smem, stream, tmR, tmC, R, C, p.y, p.ldy, blocks_of(p.K), pl.per, pl.nst,
                         (int)tiles_c, pl.split, vec, status);
}

int matmul_blocks_dispatch(const MatmulBlocksParams& p, cudaStream_t stream) {
    int* status = device_status_word();
    if (stalled(status)) return TAB_E_STALLED;
    BlocksPlan pl = {128, false, 1, blocks_of(p.K), 6};
#define TAB_MB(BN, SW) (p.type == TAB_FP32 ? launch_tile<BN, SW, TAB_FP32>(p, pl, status, stream) : p.type == TAB_BF16 ? launch_tile<BN, SW, TAB_BF16>(p, pl, status, stream) \
                                                                                                                     : launch_tile<BN, SW, TAB_FP16>(p, pl, status, stream))
    return TAB_MB(128, false);
#undef TAB_MB
}

}  // namespace tab
