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
#include <cstdlib>
#include <cuda.h>
#include <mutex>
#include <type_traits>
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
__device__ __forceinline__ void sts_b32(uint32_t at, uint32_t v) { asm volatile("st.shared.b32 [%0], %1;" ::"r"(at), "r"(v) : "memory"); }
__device__ __forceinline__ float ld_cluster_f32(uint32_t addr, uint32_t rank) {
    float v;
    asm volatile("{\n\t.reg .b32 ra;\n\tmapa.shared::cluster.u32 ra, %1, %2;\n\tld.shared::cluster.f32 %0, [ra];\n\t}" : "=f"(v) : "r"(addr), "r"(rank) : "memory");
    return v;
}

// The scales of 16 blocks from kb on of the 128 rows from row0 on, brought from memory by a warp (load), and written to shared memory as
// the tensor memory wants them, four blocks a time (store).  127 = 2^0 stands where there is no block or row; only blocks below kb1
// are read.  A load takes longer than the MMAs of four blocks when the operands' copies fill the memory system, hence 16 at a time.
//   layout 1     block by block, as the quantiser writes them (sr == 1): lane l holds rows 4l .. 4l+3, a word for each block (for the last
//                one to three rows too: their bytes one by one, or block after block, 511x777x4000 18.6 us, this way 11.6)
//   layout 16, 4 row by row (sk == 1), 16 or 4 scales of a row one aligned vector or word; 0: bytes of any strides; a square's scale serves
//                all rows.  Lane l holds rows l, l + 32, l + 64, l + 96, a word for four blocks.
struct ScaleLoader {
    int layout;
    uint32_t w[16];
    __device__ __forceinline__ ScaleLoader(const BlocksOperand& o, int kb0) {
        const uintptr_t at = reinterpret_cast<uintptr_t>(o.s);
        if (o.shift == 0 && o.sr == 1 && (at & 3) == 0 && o.sk % 4 == 0 && o.sk >= ((long long)o.rows + 3) / 4 * 4) layout = 1;
        else if (o.sk != 1) layout = 0;
        else layout = ((at | (uintptr_t)o.sr | (uintptr_t)kb0) & 15) == 0 ? 16 : ((at | (uintptr_t)o.sr | (uintptr_t)kb0) & 3) == 0 ? 4 : 0;
    }
    __device__ __forceinline__ void load(const BlocksOperand& o, int row0, int kb, int kb1, int lane) {
#pragma unroll
        for (int i = 0; i < 16; i++) w[i] = 0x7F7F7F7Fu;
        if (layout == 1) {
            const int row = row0 + 4 * lane, n = o.rows - row;
            const uint8_t* s = o.s + row + (long long)kb * o.sk;
            if (n <= 0) return;
            // A word that holds the last one to three rows reaches into the bytes before the next block's, and is cut to size; behind the last
            // block there need be none.
            const int whole = n >= 4 ? kb1 : kb1 - 1;
#pragma unroll
            for (int i = 0; i < 16; i++) if (kb + i < whole) w[i] = *reinterpret_cast<const uint32_t*>(s + i * o.sk);
            if (n >= 4) return;
            uint32_t end = 0x7F7F7F7Fu;
            if (kb1 - kb <= 16) {
                const uint8_t* e = o.s + row + (long long)whole * o.sk;
                end = (uint32_t)e[0] | (uint32_t)(n > 1 ? e[1] : 127) << 8 | (uint32_t)(n > 2 ? e[2] : 127) << 16;
            }
            const uint32_t keep = 0xFFFFFFu >> (8 * (3 - n));
#pragma unroll
            for (int i = 0; i < 16; i++) w[i] = ((kb + i == whole ? end : w[i]) & keep) | (0x7F7F7F7Fu & ~keep);
            return;
        }
        const int row = row0 + (o.shift ? 0 : lane), left = kb1 - kb, whole = layout >= 4 ? min(left >> 2, 4) : 0;      // words of four blocks that there are
        const uint8_t* s = o.s + (long long)(row >> o.shift) * o.sr + (long long)kb * o.sk;
        const long long step = 32 * o.sr;
        if (layout == 16 && whole == 4) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if ((i > 0 && o.shift) || row + 32 * i >= o.rows) continue;
                const uint4 u = *reinterpret_cast<const uint4*>(s + i * step);
                w[4 * i] = u.x; w[4 * i + 1] = u.y; w[4 * i + 2] = u.z; w[4 * i + 3] = u.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (j < whole && !(i > 0 && o.shift) && row + 32 * i < o.rows) w[4 * i + j] = reinterpret_cast<const uint32_t*>(s + i * step)[j];
            if (4 * whole < min(left, 16)) {                               // byte by byte
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    if ((i > 0 && o.shift) || row + 32 * i >= o.rows) continue;
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        if (j < whole || 4 * j >= left) continue;
                        uint32_t v = 0;
#pragma unroll
                        for (int b = 0; b < 4; b++) v |= (4 * j + b < left ? (uint32_t)s[i * step + (4 * j + b) * o.sk] : 127u) << (8 * b);
                        w[4 * i + j] = v;
                    }
                }
            }
        }
        if (o.shift)
#pragma unroll
            for (int i = 4; i < 16; i++) w[i] = w[i & 3];
    }
    // The words of blocks 4j .. 4j+3: row r at at + (r % 32) * 16 + (r / 32) * 4.
    __device__ __forceinline__ void store(uint32_t at, int j, int lane) const {
        if (layout != 1) {
            sts_v4(at + lane * 16, w[j], w[4 + j], w[8 + j], w[12 + j]);
            return;
        }
        const uint32_t a = __byte_perm(w[4 * j], w[4 * j + 1], 0x5140), b = __byte_perm(w[4 * j + 2], w[4 * j + 3], 0x5140);   // rows 0, 1 of two blocks
        const uint32_t c = __byte_perm(w[4 * j], w[4 * j + 1], 0x7362), d = __byte_perm(w[4 * j + 2], w[4 * j + 3], 0x7362);   // rows 2, 3
        const uint32_t to = at + (uint32_t)((4 * lane) & 31) * 16u + (uint32_t)(lane >> 3) * 4u;
        sts_b32(to, __byte_perm(a, b, 0x5410)); sts_b32(to + 16, __byte_perm(a, b, 0x7632));
        sts_b32(to + 32, __byte_perm(c, d, 0x5410)); sts_b32(to + 48, __byte_perm(c, d, 0x7632));
    }
};

__device__ __forceinline__ void tma_store_2d(const void* tmap, int x, int y, uint32_t src) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(tmap), "r"(src), "r"(x), "r"(y) : "memory");
}
// A warp's 32 x 32 accumulators (lane: row, columns c0 .. c0+31) to row-major memory, through 4 KB of shared memory (`stage`, this warp's
// own).  A lane that writes its own row keeps the load and store unit busy for a cycle a row, and the loads of scales wait behind it.
//   tma   (rows of y start and end on 16 bytes) boxes of 64 bytes x 32 rows, 64-byte swizzle, two buffers in turn; what lies outside y is not written
//   else  16 columns at a time are turned round (the rotation by row / 2 keeps both directions free of bank conflicts) and written by
//         16 lanes a row.
template <typename T>
__device__ __forceinline__ void store_rows32(const void* tmY, T* y, long long ldy, int row0, int nrows, int c0, int ncols, bool tma, const float (&v)[32], uint32_t stage, uint32_t& turn, int lane) {
    if (tma) {
        constexpr int E = 64 / sizeof(T);
#pragma unroll
        for (int h = 0; h < 32; h += E) {
            const uint32_t buf = stage + (turn & 1) * 2048u, row = buf + (uint32_t)lane * 64u, x = (uint32_t)(lane >> 1) & 3u;
            turn++;
            if (lane == 0) bulk_wait_read<1>();                            // the store before last has left this buffer
            __syncwarp();
#pragma unroll
            for (int c = 0; c < 4; c++) {
                if (sizeof(T) == 4) {
                    sts_v4(row + ((c ^ x) << 4), __float_as_uint(v[(h + 4 * c) & 31]), __float_as_uint(v[(h + 4 * c + 1) & 31]), __float_as_uint(v[(h + 4 * c + 2) & 31]), __float_as_uint(v[(h + 4 * c + 3) & 31]));
                } else {
                    sts_v4(row + ((c ^ x) << 4), pack2(v[8 * c], v[8 * c + 1], T()), pack2(v[8 * c + 2], v[8 * c + 3], T()), pack2(v[8 * c + 4], v[8 * c + 5], T()), pack2(v[8 * c + 6], v[8 * c + 7], T()));
                }
            }
            fence_async_smem();
            __syncwarp();
            if (lane == 0) {
                if (row0 < nrows && c0 + h < ncols) tma_store_2d(tmY, c0 + h, row0, buf);
                bulk_commit();
            }
        }
        return;
    }
#pragma unroll
    for (int h = 0; h < 32; h += 16) {
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 16; j++) asm volatile("st.shared.f32 [%0], %1;" ::"r"(stage + (uint32_t)(lane * 16 + ((j + (lane >> 1)) & 15)) * 4u), "f"(v[h + j]) : "memory");
        __syncwarp();
        const int c = c0 + h + (lane & 15);
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const int r = 2 * i + (lane >> 4);
            float f;
            asm volatile("ld.shared.f32 %0, [%1];" : "=f"(f) : "r"(stage + (uint32_t)(r * 16 + (((lane & 15) + (r >> 1)) & 15)) * 4u) : "memory");
            if (row0 + r < nrows && c < ncols) y[(long long)(row0 + r) * ldy + c] = from_float<T>(f);
        }
    }
}

static constexpr int TT = 256;                           // threads of a tile CTA
static constexpr int SF_SLOTS = 3;                       // of scale words of 16 blocks, in shared memory

// One CTA: 128 rows of operand R times BN rows of operand C over this rank's share of the sum.  Warp 0 copies the operands, warp 1
// issues the MMAs, warp 2 brings the scales, warps 4-7 finish.  A cluster shares out the sum: rank r of S takes blocks
// [r * per, (r+1) * per), the partial results meet in shared memory and every rank adds its share of the columns, in the order of
// the ranks.  SWAP: R is b, the tile is transposed (few rows of a: the 128-row side of the MMA takes the weights).  What bounds it is start
// and end (4 us of a call on next to nothing) and what an SM takes in, 43 to 64 bytes a cycle; us at sizes: see blocks_plan.
template <int BN, int KS, bool SWAP, int TYPE>
__global__ void __launch_bounds__(TT) matmul_blocks_tile_kernel(const __grid_constant__ CUtensorMap tmR, const __grid_constant__ CUtensorMap tmC, const __grid_constant__ CUtensorMap tmY, BlocksOperand R, BlocksOperand C,
                                                                void* yv, long long ldy, int KB, int per, int nst, int tiles_c, int split, int tma, int* status) {
    using T = typename ElemOf<TYPE>::type;
    extern __shared__ uint8_t raw[];
    constexpr int STAGE = KS * (128 + BN) * 128;                           // KS blocks: their rows of R, then their rows of C
    static_assert(BN <= 128, "the scales of 128 rows on either side");
    constexpr int SFB = 1024;                                              // bytes of four blocks' scales; a slot holds four of them
    constexpr int SFCOL = BN < 32 ? 32 : BN;                               // first tensor-memory column of the scales: two slots
    constexpr int TCOLS = SFCOL + 16 <= 64 ? 64 : SFCOL + 16 <= 128 ? 128 : 256;
    __shared__ __align__(8) uint64_t bars[16 + 2 * SF_SLOTS + 1];
    __shared__ __align__(512) uint8_t sf[SF_SLOTS * 4 * SFB];
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
    pdl_launch_dependents();
    auto expire = [&](int code) { if (lane == 0) { if (status) atomicExch(status, code); *deadp = 1; } };

    if (warp == 0) {
        for (int kb = kb0, g = 0; kb < kb1; kb += KS, g++) {
            const int s = g % nst, blocks = min(KS, kb1 - kb);
            if (g >= nst && !mbar_wait_warp(empty + 8 * s, (g / nst - 1) & 1)) { expire(31); break; }
            if (elect_one()) {
                mbar_expect_tx(full + 8 * s, (uint32_t)blocks * (128 + BN) * 128);
                for (int i = 0; i < blocks; i++) {
                    tma_load_2d(sRing + s * STAGE + i * 16384, &tmR, (kb + i) * BLK, r0, full + 8 * s);
                    tma_load_2d(sRing + s * STAGE + KS * 16384 + i * BN * 128, &tmC, (kb + i) * BLK, c0, full + 8 * s);
                }
            }
            __syncwarp();
        }
    } else if (warp == 1) {
        const uint32_t idesc = umma_idesc_f8(128, BN, R.format == TAB_E5M2, C.format == TAB_E5M2);
        for (int kb = kb0, g = 0; kb < kb1; kb += KS, g++) {
            const int s = g % nst, at = kb - kb0, q = at >> 4, slot = q % SF_SLOTS;
            const uint32_t sfcol = tmem + SFCOL + ((at >> 2) & 1) * 8;
            if ((at & 15) == 0) {
                if (!mbar_wait_warp(sfFull + 8 * slot, (q / SF_SLOTS) & 1)) { expire(32); break; }
                tc_fence_after();
            }
            if (!mbar_wait_warp(full + 8 * s, (g / nst) & 1)) { expire(33); break; }
            tc_fence_after();
            if (elect_one()) {
                if ((at & 3) == 0) {
#pragma unroll
                    for (int i = 0; i < 2; i++) tmem_copy_scales(sfcol + 4 * i, sSF + (slot * 4 + ((at >> 2) & 3)) * SFB + 512 * i);
                    if ((at & 12) == 12 || kb + 4 >= kb1) umma_commit(sfEmpty + 8 * slot);
                }
#pragma unroll
                for (int b = 0; b < KS; b++) {
                    if (kb + b >= kb1) break;
                    const uint64_t da = umma_desc(sRing + s * STAGE + b * 16384), db = umma_desc(sRing + s * STAGE + KS * 16384 + b * BN * 128);
                    const uint32_t id = with_scale_byte(idesc, (uint32_t)((at + b) & 3));
#pragma unroll
                    for (int i = 0; i < 4; i++) umma_f8(tmem, da + 2 * i, db + 2 * i, id, sfcol, sfcol + 4, (at | b | i) != 0);
                }
                umma_commit(empty + 8 * s);
                if (kb + KS >= kb1) umma_commit(accFull);
            }
            __syncwarp();
        }
    } else if (warp == 2) {
        ScaleLoader r(R, kb0), c(C, kb0);
        for (int kb = kb0, q = 0; kb < kb1; kb += 16, q++) {
            r.load(R, r0, kb, kb1, lane);
            c.load(C, c0, kb, kb1, lane);
            const int slot = q % SF_SLOTS;
            if (q >= SF_SLOTS && !mbar_wait_warp(sfEmpty + 8 * slot, (q / SF_SLOTS - 1) & 1)) { expire(34); break; }
#pragma unroll
            for (int j = 0; j < 4; j++) {
                r.store(sSF + (slot * 4 + j) * SFB, j, lane);
                c.store(sSF + (slot * 4 + j) * SFB + 512, j, lane);
            }
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(sfFull + 8 * slot);
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
            uint32_t turn = 0;
#pragma unroll 1
            for (int cb = 0; cb < BN && c0 + cb < C.rows; cb += 32) {
                uint32_t v[32];
                tmem_ld32(taddr + cb, v);                                  // BN = 16: the columns behind the tile's are read and not used
                float o[32];
#pragma unroll
                for (int j = 0; j < 32; j++) o[j] = __uint_as_float(v[j]);
                if (SWAP) {
                    if (row < R.rows) {
#pragma unroll
                        for (int j = 0; j < LC; j++) if (c0 + cb + j < C.rows) y[(long long)(c0 + cb + j) * ldy + row] = from_float<T>(o[j]);
                    }
                } else {
                    store_rows32(&tmY, y, ldy, r0 + quarter, R.rows, c0 + cb, C.rows, tma, o, sRing + (uint32_t)(warp - 4) * 4096u, turn, lane);
                }
            }
            if (!SWAP && tma && lane == 0) bulk_wait_all();
        }
    } else {
        // Partial results in the ring: [column][128 rows] floats, or [row][BN + 1] for a tile that is written as it is.  A rank without blocks
        // contributes zeros.  Every rank finishes its share of the rows of y, in the order of the ranks, 32 neighbours of a row a warp.
        float* part = reinterpret_cast<float*>(raw + (sRing - (uint32_t)__cvta_generic_to_shared(raw)));
        if (warp >= 4) {
#pragma unroll 1
            for (int cb = 0; cb < BN; cb += 32) {
                uint32_t v[32];
                tmem_ld32(taddr + cb, v);
#pragma unroll
                for (int j = 0; j < LC; j++) part[SWAP ? (cb + j) * 128 + quarter + lane : (quarter + lane) * (BN + 1) + cb + j] = kb1 > kb0 ? __uint_as_float(v[j]) : 0.f;
            }
        }
        cluster_sync_all();
        constexpr int YR = SWAP ? BN : 128, YC = SWAP ? 128 : BN, PITCH = SWAP ? 128 : BN + 1;   // rows and columns of y in the tile
        const int y0 = SWAP ? c0 : r0, x0 = SWAP ? r0 : c0, ylim = SWAP ? C.rows : R.rows, xlim = SWAP ? R.rows : C.rows, share = YR / split;
        for (int i = rank * share * (YC / 32) + warp, end = (rank + 1) * share * (YC / 32); i < end; i += TT / 32) {
            const int yr = i / (YC / 32), xc = i % (YC / 32) * 32 + lane;
            float sum = 0.f;
            for (int k = 0; k < split; k++) sum += ld_cluster_f32(sRing + (uint32_t)(yr * PITCH + xc) * 4u, (uint32_t)k);
            if (y0 + yr < ylim && x0 + xc < xlim) y[(long long)(y0 + yr) * ldy + x0 + xc] = from_float<T>(sum);
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
    if (warp == 1) tmem_dealloc(tmem, TCOLS);
}

// ---- CTA pairs ----------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ void umma_f8_pair(uint32_t tmem_d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\t"
                 "setp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.block32 [%0], %1, %2, %3, [%5], [%6], p;\n\t}"
                 :: "r"(tmem_d), "l"(da), "l"(db), "r"(idesc), "r"(accumulate), "r"(sfa), "r"(sfb) : "memory");
}
// The same 512 bytes of both CTAs' shared memory to the same columns of both tensor memories.
__device__ __forceinline__ void tmem_copy_scales_pair(uint32_t taddr, uint32_t smem_addr) {
    const uint64_t d = ((uint64_t)((128u >> 4) | (1u << 14)) << 32) | ((smem_addr & 0x3FFFFu) >> 4);
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(d) : "memory");
}

static constexpr int PT = 256;                           // threads of a pair's CTA: copies, MMAs, scales, -, four that finish
static constexpr int PSTAGES = 6;                        // of 128 terms: 128 rows of a and 128 of b, 32 KB
static constexpr int PSTAGE = 32768;
static constexpr int PSF = 1536;                         // scale words of 512 terms: 128 rows of a, 256 of b; a slot holds four of them
static constexpr int PSLOTS = 2;
static_assert(PSTAGES * PSTAGE + PSLOTS * 4 * PSF + 4 * 4096 + 1024 + 512 <= UMMA_SMEM_MAX, "static and dynamic shared memory");
static constexpr int PACC = 224;                         // second accumulator's first column: it shares 32 with the first
static constexpr int PSFCOL = 480;
static constexpr int PSMEM = PSTAGES * PSTAGE + PSLOTS * 4 * PSF + 4 * 4096 + 1024;

// A persistent pair of CTAs works 256 x 256 tiles: each CTA holds 128 rows of a and of b, and one MMA stream, issued by the even CTA,
// multiplies for both; each CTA's tensor memory receives the sums of its own 128 rows of a and all 256 of b.  Two accumulators, so
// that a tile's sums leave while the next tile's are made: 512 columns hold two of 256 and the scales only if the accumulators share
// some, here 32, which the finishing warps read first and release; from there on the next tile's MMAs may run.
// 4096x8192x4096 with bf16 results: 104 us in bursts (2.65 PFLOP/s; tensor pipe 68 % busy under the profiler), 127 in loops of a second, where the
// 1000 W cap sets the clock; 128 x 128 tiles of single CTAs 149.  A CTA takes in 32 KB in the 512 cycles of a stage's MMAs, about all an SM can.
// group: tiles are taken in bands of so many row blocks, column by column, so that what is in work at a time shares its operands in the L2.
template <int TYPE>
__global__ void __launch_bounds__(PT) matmul_blocks_pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const __grid_constant__ CUtensorMap tmY, BlocksOperand A, BlocksOperand B,
                                                               void* yv, long long ldy, int KB, int tiles_m, int tiles_n, int group, int tma, int* status) {
    using T = typename ElemOf<TYPE>::type;
    extern __shared__ uint8_t raw[];
    __shared__ __align__(8) uint64_t bars[2 * PSTAGES + 2 * PSLOTS + 3];
    __shared__ uint32_t tslot;
    __shared__ int dead_flag;
    volatile int* deadp = &dead_flag;
    const uint32_t sRing = ((uint32_t)__cvta_generic_to_shared(raw) + 1023u) & ~1023u, sSF = sRing + PSTAGES * PSTAGE, sStage = sSF + PSLOTS * 4 * PSF;
    const uint32_t full = (uint32_t)__cvta_generic_to_shared(bars), empty = full + 8 * PSTAGES, sfFull = empty + 8 * PSTAGES, sfEmpty = sfFull + 8 * PSLOTS,
                   accFull = sfEmpty + 8 * PSLOTS, accFree = accFull + 16;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t rank = cluster_ctarank();
    const int pair0 = (int)(blockIdx.x >> 1), pairs = (int)(gridDim.x >> 1), ntiles = tiles_m * tiles_n;

    if (tid == 0) {
        *deadp = 0;
        for (int s = 0; s < PSTAGES; s++) { mbar_init(full + 8 * s, 1); mbar_init(empty + 8 * s, 1); }
        for (int s = 0; s < PSLOTS; s++) { mbar_init(sfFull + 8 * s, 2); mbar_init(sfEmpty + 8 * s, 1); }
        mbar_init(accFull, 1); mbar_init(accFull + 8, 1); mbar_init(accFree, 8);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) tmem_alloc_pair((uint32_t)__cvta_generic_to_shared(&tslot), 512);
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();                                                    // both CTAs' barriers exist before either arrives on the other's
    tc_fence_after();
    const uint32_t tmem = *static_cast<volatile uint32_t*>(&tslot);
    pdl_wait();
    auto expire = [&](int code) { if (lane == 0) { if (status) atomicExch(status, code); *deadp = 1; } };
    auto tile_at = [&](int t, int& m0, int& n0) {
        const int band = t / (group * tiles_n), first = band * group, rows = min(group, tiles_m - first), i = t - first * tiles_n;
        m0 = (first + i % rows) * 256;
        n0 = i / rows * 256;
    };

    if (warp == 0) {
        int g = 0;
        bool dead = false;
        for (int t = pair0; t < ntiles && !dead; t += pairs) {
            int m0, n0;
            tile_at(t, m0, n0);
            m0 += (int)rank * 128; n0 += (int)rank * 128;
            for (int kb = 0; kb < KB; kb++, g++) {
                const int s = g % PSTAGES;
                if (g >= PSTAGES && !mbar_wait_cluster_warp(empty + 8 * s, (g / PSTAGES - 1) & 1)) { expire(36); dead = true; break; }
                if (elect_one()) {
                    if (rank == 0) mbar_expect_tx(full + 8 * s, 2 * PSTAGE);   // both CTAs' copies are counted on the even one's barrier
                    tma_load_2d_pair(sRing + s * PSTAGE, &tmA, kb * BLK, m0, full + 8 * s);
                    tma_load_2d_pair(sRing + s * PSTAGE + 16384, &tmB, kb * BLK, n0, full + 8 * s);
                }
                __syncwarp();
            }
        }
    } else if (warp == 1 && rank == 0) {
        const uint32_t idesc = umma_idesc_f8(256, 256, A.format == TAB_E5M2, B.format == TAB_E5M2);
        int g = 0, q = 0, a = 0;
        bool dead = false;
        for (int t = pair0; t < ntiles && !dead; t += pairs, a++) {
            const uint32_t d = tmem + (a & 1) * PACC;
            if (a >= 1 && !mbar_wait_cluster_warp(accFree, (a - 1) & 1)) { expire(37); break; }
            tc_fence_after();
            for (int kb = 0; kb < KB; kb++, g++) {
                const int s = g % PSTAGES, slot = q % PSLOTS;
                const uint32_t sfcol = tmem + PSFCOL + ((kb >> 2) & 1) * 12;
                if ((kb & 15) == 0) {
                    if (!mbar_wait_cluster_warp(sfFull + 8 * slot, (q / PSLOTS) & 1)) { expire(38); dead = true; break; }
                    tc_fence_after();
                }
                if (!mbar_wait_cluster_warp(full + 8 * s, (g / PSTAGES) & 1)) { expire(39); dead = true; break; }
                tc_fence_after();
                const bool last_scales = (kb & 3) == 0 && ((kb & 12) == 12 || kb + 4 >= KB);
                if (elect_one()) {
                    if ((kb & 3) == 0) {
#pragma unroll
                        for (int i = 0; i < 3; i++) tmem_copy_scales_pair(sfcol + 4 * i, sSF + (slot * 4 + ((kb >> 2) & 3)) * PSF + 512 * i);
                        if (last_scales) umma_commit_pair(sfEmpty + 8 * slot);
                    }
                    const uint64_t da = umma_desc(sRing + s * PSTAGE), db = umma_desc(sRing + s * PSTAGE + 16384);
                    const uint32_t id = with_scale_byte(idesc, (uint32_t)(kb & 3));
#pragma unroll
                    for (int i = 0; i < 4; i++) umma_f8_pair(d, da + 2 * i, db + 2 * i, id, sfcol, sfcol + 4, (kb | i) != 0);
                    umma_commit_pair(empty + 8 * s);
                    if (kb == KB - 1) umma_commit_pair(accFull + 8 * (a & 1));
                }
                __syncwarp();
                if (last_scales) q++;
            }
        }
    } else if (warp == 2) {
        // A chunk of 16 blocks is fetched, stored and announced before the next one is asked for: the fence and the arrival on the other
        // CTA's barrier would wait for loads under way.  Two slots, 32 blocks, keep the MMAs supplied meanwhile.
        ScaleLoader wa(A, 0), w0(B, 0), w1(B, 0);
        bool dead = false;
        int q = 0;
        for (int t = pair0; t < ntiles && !dead; t += pairs) {
            int m0, n0;
            tile_at(t, m0, n0);
            for (int kb = 0; kb < KB; kb += 16, q++) {
                wa.load(A, m0 + (int)rank * 128, kb, KB, lane);
                w0.load(B, n0, kb, KB, lane);
                w1.load(B, n0 + 128, kb, KB, lane);
                const int slot = q % PSLOTS;
                if (q >= PSLOTS && !mbar_wait_cluster_warp(sfEmpty + 8 * slot, (q / PSLOTS - 1) & 1)) { expire(40); dead = true; break; }
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const uint32_t at = sSF + (slot * 4 + j) * PSF;
                    wa.store(at, j, lane);
                    w0.store(at + 512, j, lane);
                    w1.store(at + 1024, j, lane);
                }
                fence_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster(sfFull + 8 * slot, 0u);
            }
        }
    } else if (warp >= 4) {
        T* y = static_cast<T*>(yv);
        const int quarter = (warp & 3) * 32;
        uint32_t turn = 0;
        int a = 0;
        for (int t = pair0; t < ntiles; t += pairs, a++) {
            int m0, n0;
            tile_at(t, m0, n0);
            if (!mbar_wait_cluster_warp(accFull + 8 * (a & 1), (a >> 1) & 1)) { expire(41); break; }
            tc_fence_after();
            const uint32_t taddr = tmem + (a & 1) * PACC + ((uint32_t)quarter << 16);
#pragma unroll 1
            for (int i = 0; i < 8; i++) {
                const int cb = ((a & 1) ? i : 7 - i) * 32;                 // the shared columns first: the first accumulator's last, the second's first
                uint32_t v[32];
                tmem_ld32(taddr + cb, v);
                if (i == 0) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_cluster(accFree, 0u);       // and this warp is done with the other accumulator
                }
                float o[32];
#pragma unroll
                for (int j = 0; j < 32; j++) o[j] = __uint_as_float(v[j]);
                if (n0 + cb < B.rows) store_rows32(&tmY, y, ldy, m0 + (int)rank * 128 + quarter, A.rows, n0 + cb, B.rows, tma, o, sStage + (uint32_t)(warp - 4) * 4096u, turn, lane);
            }
        }
        if (tma && lane == 0) bulk_wait_all();
    }
    tc_fence_before();
    __syncthreads();
    if (*deadp != 0) {
        for (int i = 0; i < 200; i++) __nanosleep(1000);                   // see the tile kernel
        __syncthreads();
    }
    cluster_sync_all();                                                    // the other CTA neither reads this one's memory nor arrives on its barriers any more
    pdl_launch_dependents();
    if (warp == 1) tmem_dealloc_pair(tmem, 512);
}

// ---- few rows of a ----------------------------------------------------------------------------------------------------------------
// Two 8-bit floats (low byte first) as fp16, exact for both formats.
__device__ __forceinline__ uint32_t widen2(uint32_t two, bool e5m2) {
    uint32_t h;
    if (e5m2) asm("cvt.rn.f16x2.e5m2x2 %0, %1;" : "=r"(h) : "h"((uint16_t)two));
    else asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)two));
    return h;
}
template <int FORMAT>
__device__ __forceinline__ void widen16(const uint4& u, uint32_t (&h)[8]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; i++) { h[2 * i] = widen2(w[i] & 0xFFFFu, FORMAT == TAB_E5M2); h[2 * i + 1] = widen2(w[i] >> 16, FORMAT == TAB_E5M2); }
}
// 16 values of a row from k on; those behind its end are 0 and not read.
__device__ __forceinline__ uint4 load_values16(const uint8_t* row, int k, int K) {
    if (k + 16 <= K) return *reinterpret_cast<const uint4*>(row + k);
    uint32_t w[4] = {0, 0, 0, 0};
    for (int j = 0; j < 16; j++) if (k + j < K) w[j >> 2] |= (uint32_t)row[k + j] << (8 * (j & 3));
    return make_uint4(w[0], w[1], w[2], w[3]);
}
// A load of weights that are read once.
__device__ __forceinline__ uint4 ld_stream(const uint8_t* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.L2::128B.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
// sum + v * 2^(a - 127) * 2^(b - 127) for scale bytes (255: NaN).
__device__ __forceinline__ float add_scaled(float sum, float v, int a, int b) {
    const int e = a + b - 127;
    if (e >= 1 && e <= 254 && a != 255 && b != 255) return fmaf(v, __uint_as_float((uint32_t)e << 23), sum);
    if (a == 255 || b == 255) return __uint_as_float(0x7FC00000u);
    const int h = (e - 127) >> 1;                                          // beyond fp32's exponents: in two steps
    return sum + v * exp2_int(h) * exp2_int(e - 127 - h);
}
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

static constexpr int VMOST = 8;                          // rows of a

// At most eight rows of a against all of b: every weight is read once and multiplied so few times that nothing but the reading counts,
// so there is no pipeline through shared and tensor memory, whose start and end cost more than the reading of a few megabytes.  A warp
// takes 16 rows of b and a share of the sum straight into registers, 16 bytes a lane, and multiplies in fp16, which holds every 8-bit
// float, with fp32 sums (the sum's order is free as long as both operands agree, so a lane's 16 neighbours serve four MMAs).  A block's
// sum is added under its scales; the warps' sums are added in their order.  CTAS on an SM: two with two blocks of the sum under way in each warp
// while that is all of b, else four with one, which leave fewer SMs idle at the end (cold weights, us, two / four): 1x1024x4096 4.1 / 5.4,
// 1x4096x4096 5.8 / 6.4 (the tile kernel 7.3), 1x8192x8192 16.1 / 14.7 (19.4), 1x32000x4096 28.5 / 24.8 (5.3 TB/s; 26.2), 1x6000x2000 9.3 / 7.2.
// Up to 64 rows of a this way were slower from 16 on (24x4096x4096 10.8, 8.3).
template <int FA, int FB, int CTAS>
__global__ void __launch_bounds__(256, CTAS) matmul_blocks_rows_kernel(BlocksOperand A, BlocksOperand B, void* y, long long ldy, int type, int K, int per) {
    constexpr int VAHEAD = 4 / CTAS;                                       // blocks of the sum a warp has under way
    __shared__ float part[8][16][9];
    pdl_wait();
    pdl_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, n0 = (int)blockIdx.x * 16, KB = (K + BLK - 1) / BLK;
    const int kb1 = min(KB, (warp + 1) * per);
    // rows that do not exist are read as the last one, and their results not written
    const uint8_t* b[2];
    const uint8_t* bs[2];
    const uint8_t* as[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const int row = min(n0 + g + 8 * i, B.rows - 1), m = min(2 * t + i, A.rows - 1);
        b[i] = B.q + (long long)row * B.ld;
        bs[i] = B.s + (long long)(row >> B.shift) * B.sr;
        as[i] = A.s + (long long)(m >> A.shift) * A.sr;
    }
    const uint8_t* a = A.q + (long long)min(g, A.rows - 1) * A.ld;
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
    auto block = [&](const uint4 (&w)[2][2], const uint4 (&v)[2], const int (&sa)[2], const int (&sb)[2]) {
        float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int h = 0; h < 2; h++) {
            uint32_t w0[8], w1[8], x[8];
            widen16<FB>(w[h][0], w0);
            widen16<FB>(w[h][1], w1);
            widen16<FA>(v[h], x);
#pragma unroll
            for (int j = 0; j < 4; j++) mma_f16(d, w0[2 * j], w1[2 * j], w0[2 * j + 1], w1[2 * j + 1], x[2 * j], x[2 * j + 1]);
        }
#pragma unroll
        for (int j = 0; j < 4; j++) sum[j] = add_scaled(sum[j], d[j], sa[j & 1], sb[j >> 1]);
    };
    const int whole = min(kb1, K / BLK);                                   // blocks that are not cut short by the row's end
    int kb = warp * per;
    auto several = [&](auto count) {
        constexpr int N = decltype(count)::value;
        uint4 w[N][2][2], v[N][2];
        int sb[N][2], sa[N][2];
#pragma unroll
        for (int i = 0; i < N; i++) {
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int k = (kb + i) * BLK + h * 64 + t * 16;
#pragma unroll
                for (int r = 0; r < 2; r++) w[i][h][r] = ld_stream(b[r] + k);
                v[i][h] = *reinterpret_cast<const uint4*>(a + k);
            }
#pragma unroll
            for (int r = 0; r < 2; r++) {
                sb[i][r] = bs[r][(long long)(kb + i) * B.sk];
                sa[i][r] = as[r][(long long)(kb + i) * A.sk];
            }
        }
#pragma unroll
        for (int i = 0; i < N; i++) block(w[i], v[i], sa[i], sb[i]);
        kb += N;
    };
    while (kb + VAHEAD <= whole) several(std::integral_constant<int, VAHEAD>());
    if (VAHEAD > 1) while (kb < whole) several(std::integral_constant<int, 1>());
    if (kb < kb1) {                                                        // the row's last, short block
        uint4 w[2][2], v[2];
        int sb[2], sa[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int k = kb * BLK + h * 64 + t * 16;
#pragma unroll
            for (int r = 0; r < 2; r++) w[h][r] = load_values16(b[r], k, K);
            v[h] = load_values16(a, k, K);
        }
#pragma unroll
        for (int r = 0; r < 2; r++) {
            sb[r] = bs[r][(long long)kb * B.sk];
            sa[r] = as[r][(long long)kb * A.sk];
        }
        block(w, v, sa, sb);
    }
#pragma unroll
    for (int j = 0; j < 4; j++) part[warp][g + 8 * (j >> 1)][2 * t + (j & 1)] = sum[j];
    __syncthreads();
    if (threadIdx.x < 128) {
        const int n = threadIdx.x & 15, m = threadIdx.x >> 4;
        if (n0 + n < B.rows && m < A.rows) {
            float s = 0.f;
            for (int i = 0; i < (int)blockDim.x / 32; i++) s += part[i][n][m];
            const long long at = (long long)m * ldy + n0 + n;
            if (type == TAB_FP32) static_cast<float*>(y)[at] = s;
            else if (type == TAB_BF16) static_cast<__nv_bfloat16*>(y)[at] = __float2bfloat16_rn(s);
            else static_cast<__half*>(y)[at] = __float2half_rn(s);
        }
    }
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

// y as store_rows32 writes it; false where its rows do not start, or do not end, on 16 bytes: a store is cut off at multiples of 16 bytes
// only, and would write up to 12 bytes behind a row.
static bool blocks_result_map(CUtensorMap* m, const MatmulBlocksParams& p) {
    const cuuint64_t size = (cuuint64_t)type_bytes(p.type);
    EncodeTiledFn fn = blocks_encode_fn();
    if (!fn || (reinterpret_cast<uintptr_t>(p.y) & 15) || p.ldy * size % 16 || p.b.rows * size % 16 || p.ldy * size >= (1ULL << 40)) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)p.b.rows, (cuuint64_t)p.a.rows}, strides[1] = {p.ldy * size};
    const cuuint32_t box[2] = {(cuuint32_t)(64 / size), 32}, estr[2] = {1, 1};
    const CUtensorMapDataType type = p.type == TAB_FP32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : p.type == TAB_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    return fn(m, type, 2, p.y, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct BlocksPlan { int bn; bool swap; int split, per, nst, ks; };

// What the thread launched last, put into words when somebody asks.
static thread_local struct { int kind; BlocksPlan plan; } g_last = {0, {}};
const char* matmul_blocks_last_kernel() {
    static thread_local char text[96];
    const BlocksPlan& p = g_last.plan;
    if (g_last.kind == 0) return "none";
    if (g_last.kind == 1) return "matmul_blocks_rows_kernel";
    if (g_last.kind == 3) return "matmul_blocks_pair_kernel";
    snprintf(text, sizeof(text), "matmul_blocks_tile_kernel<%d,%d,%d> split %d stages %d", p.bn, p.ks, (int)p.swap, p.split, p.nst);
    return text;
}

template <int BN, int KS, bool SWAP, int TYPE>
static int launch_tile(const MatmulBlocksParams& p, const BlocksPlan& pl, int* status, cudaStream_t stream) {
    auto kernel = matmul_blocks_tile_kernel<BN, KS, SWAP, TYPE>;
    const BlocksOperand &R = SWAP ? p.b : p.a, &C = SWAP ? p.a : p.b;
    alignas(64) CUtensorMap tmR, tmC;
    if (!blocks_map(&tmR, R, p.K, 128) || !blocks_map(&tmC, C, p.K, BN)) return TAB_E_TOO_LARGE;
    static std::mutex mu;
    static bool configured[64] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return record_cuda_error(e);
    const int smem = std::max(pl.nst * KS * (128 + BN) * 128, pl.split > 1 ? 128 * (BN + 1) * 4 : 0) + 1024;
    {
        std::lock_guard<std::mutex> lock(mu);
        if (dev < 0 || dev >= 64 || !configured[dev]) {
            e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 208 * 1024);
            if (e != cudaSuccess) return record_cuda_error(e);
            if (dev >= 0 && dev < 64) configured[dev] = true;
        }
    }
    const long long tiles_r = (R.rows + 127) / 128, tiles_c = ((long long)C.rows + BN - 1) / BN, grid = tiles_r * tiles_c * pl.split;
    if (grid >= (1LL << 31)) return TAB_E_TOO_LARGE;
    alignas(64) CUtensorMap tmY = tmR;                                     // a stand-in where it is not used
    const int tma = !SWAP && pl.split == 1 && blocks_result_map(&tmY, p);
    g_last.kind = 2; g_last.plan = pl;
    return launch_pdl_as(false, (unsigned)pl.split, kernel, dim3((unsigned)grid), dim3(TT), (size_t)smem, stream, tmR, tmC, tmY, R, C, p.y, p.ldy, blocks_of(p.K), pl.per, pl.nst,
                         (int)tiles_c, pl.split, tma, status);
}

// How many pairs the device holds at once (0: none), asked of the occupancy calculator once per device.
static int matmul_pairs() {
    static std::mutex mu;
    static int known[64] = {};                                             // 0 unknown, else pairs + 1
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
    std::lock_guard<std::mutex> lock(mu);
    if (!known[dev]) {
        int clusters = 0;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(2); cfg.blockDim = dim3(PT); cfg.dynamicSmemBytes = PSMEM;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = 2; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr; cfg.numAttrs = 1;
        bool ok = true;
        for (auto kernel : {matmul_blocks_pair_kernel<TAB_FP32>, matmul_blocks_pair_kernel<TAB_BF16>, matmul_blocks_pair_kernel<TAB_FP16>})
            ok = ok && cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, PSMEM) == cudaSuccess &&
                 cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg) == cudaSuccess && clusters >= 1;
        if (!ok) { cudaGetLastError(); return 0; }                         // (asked again by the next call)
        known[dev] = clusters + 1;
    }
    return known[dev] - 1;
}

static int launch_pair(const MatmulBlocksParams& p, int pairs, int* status, cudaStream_t stream) {
    alignas(64) CUtensorMap tmA, tmB;
    if (!blocks_map(&tmA, p.a, p.K, 128) || !blocks_map(&tmB, p.b, p.K, 128)) return TAB_E_TOO_LARGE;
    const long long tiles_m = ((long long)p.a.rows + 255) / 256, tiles_n = ((long long)p.b.rows + 255) / 256, ntiles = tiles_m * tiles_n;
    if (ntiles >= (1LL << 30)) return TAB_E_TOO_LARGE;
    alignas(64) CUtensorMap tmY = tmA;
    const int tma = blocks_result_map(&tmY, p);
    const unsigned grid = 2u * (unsigned)std::min<long long>(ntiles, pairs);
    g_last.kind = 3;
    auto kernel = p.type == TAB_FP32 ? matmul_blocks_pair_kernel<TAB_FP32> : p.type == TAB_BF16 ? matmul_blocks_pair_kernel<TAB_BF16> : matmul_blocks_pair_kernel<TAB_FP16>;
    return launch_pdl_as(false, 2u, kernel, dim3(grid), dim3(PT), (size_t)PSMEM, stream, tmA, tmB, tmY, p.a, p.b, p.y, p.ldy, blocks_of(p.K), (int)tiles_m, (int)tiles_n, 8, tma, status);
}

static int launch_rows(const MatmulBlocksParams& p, cudaStream_t stream) {
    const int KB = blocks_of(p.K);
    const unsigned grid = (unsigned)(((long long)p.b.rows + 15) / 16);
    const int warps = 8;
    const int per = (KB + warps - 1) / warps;
    g_last.kind = 1;
    const bool one_round = (long long)grid <= 2LL * blocks_sms();
#define TAB_MR(FA, FB) (one_round ? launch_pdl(matmul_blocks_rows_kernel<FA, FB, 2>, dim3(grid), dim3(32 * warps), 0, stream, p.a, p.b, p.y, p.ldy, p.type, p.K, per) \
                                  : launch_pdl(matmul_blocks_rows_kernel<FA, FB, 4>, dim3(grid), dim3(32 * warps), 0, stream, p.a, p.b, p.y, p.ldy, p.type, p.K, per))
    if (p.a.format == TAB_E5M2) return p.b.format == TAB_E5M2 ? TAB_MR(TAB_E5M2, TAB_E5M2) : TAB_MR(TAB_E5M2, TAB_E4M3);
    return p.b.format == TAB_E5M2 ? TAB_MR(TAB_E4M3, TAB_E5M2) : TAB_MR(TAB_E4M3, TAB_E4M3);
#undef TAB_MR
}

template <int BN, int KS, bool SWAP>
static int launch_tile_type(const MatmulBlocksParams& p, const BlocksPlan& pl, int* status, cudaStream_t stream) {
    return p.type == TAB_FP32 ? launch_tile<BN, KS, SWAP, TAB_FP32>(p, pl, status, stream) : p.type == TAB_BF16 ? launch_tile<BN, KS, SWAP, TAB_BF16>(p, pl, status, stream)
                                                                                                                : launch_tile<BN, KS, SWAP, TAB_FP16>(p, pl, status, stream);
}

// Tile, split and stages where there are too few tiles for the pairs.  Measured with cold operands (us, bf16 result, square scales of b):
//   columns   Waits and issues cost the MMA warp about 300 cycles a stage whatever it holds, so a stage holds four blocks where a CTA has
//             the SM to itself: 256x4096x4096, 128 x 64 tiles, stages of 1 / 2 / 4 blocks 17.4 / 12.5 / 10.6; of 128 x 128: 18.6 / 13.5.
//             64 columns while that makes at most a tile an SM (1024x1024x8192 16.9, 128 columns 22.8), then 128 (1024x2048x2048 9.4,
//             64 columns 10.0), and with two CTAs an SM small stages (2048x2048x2048 13.0, stages of two blocks 17.8; pairs 14.1).
//   swap      At most 64 rows of a: the 128-row side takes the weights (16x8192x2048 6.9, else 9.7; 40x8192x2048 8.9 / 9.7).
//   split     Meeting in shared memory costs about 1.2 us, a block of the sum 0.2: ranks keep eight blocks, and sums of fewer than 32 are
//             not split (12x4096x4096: 1 / 4 / 8 ranks 11.7 / 8.0 / 8.3; 16x8192x2048 1 / 2 / 4 ranks 6.9 / 8.1 / 8.3; 128x128x8192: 8 ranks
//             8.2, 4 9.9); wide tiles only while most SMs would idle (100x4096x4096, 64 tiles: 1 / 4 ranks 10.4 / 12.1).
static BlocksPlan blocks_plan(int M, int N, int KB, int sms) {
    const long long rows = ((long long)M + 127) / 128, tiles64 = rows * (((long long)N + 63) / 64), tiles128 = rows * (((long long)N + 127) / 128);
    BlocksPlan pl = {64, M <= 64, 1, KB, 2, 4};
    long long tiles = tiles64;
    if (pl.swap) {
        pl.bn = M <= 16 ? 16 : M <= 32 ? 32 : 64;
        tiles = ((long long)N + 127) / 128;
    } else if (tiles64 > sms) {
        pl.bn = 128; pl.nst = 3; pl.ks = tiles128 <= sms ? 2 : 1;
        tiles = tiles128;
    }
    while (pl.split < 8 && KB >= 32 && KB >= 16 * pl.split && tiles * 2 * pl.split <= (pl.swap ? 2 * sms : sms / 2)) pl.split *= 2;
    if (pl.swap && tiles * pl.split > sms) { pl.ks = 2; pl.nst = pl.bn == 64 ? 2 : 3; }      // (room for a second CTA on an SM, or nearly)
    pl.per = (KB + pl.split - 1) / pl.split;
#ifdef TAB_TUNE
    // Build-time diagnostic (-DTAB_TUNE, never in the shipped library): "columns,swap,split,stages,blocks" from the environment.
    if (const char* env = getenv("TAB_MATMUL")) {
        int swap = 0;
        if (sscanf(env, "%d,%d,%d,%d,%d", &pl.bn, &swap, &pl.split, &pl.nst, &pl.ks) == 5) { pl.swap = swap != 0; pl.per = (KB + pl.split - 1) / pl.split; return pl; }
    }
#endif
    return pl;
}

int matmul_blocks_dispatch(const MatmulBlocksParams& p, cudaStream_t stream) {
    int* status = device_status_word();
    if (stalled(status)) return TAB_E_STALLED;
    const int sms = blocks_sms();
    // pairs from two rounds of 128 x 128 tiles on: 1536x4096x1024 (384 of them) 15.8, single CTAs 17.1; 4096x1024x1024 (256) 12.4 / 9.9; 129x20000x4096
    // 41 / 47, 200x40000x4096 57 / 81.  The count alone decides, so 65 to 128 rows against more than 37888 columns take them too, whose tiles are half
    // padding then: 100x40000x4096 57 / 53, 128x65536x4096 76 / 65, 128x40000x512 22 / 16.
    const long long tiles128 = ((long long)p.a.rows + 127) / 128 * (((long long)p.b.rows + 127) / 128);
    const int pairs = matmul_pairs();
    bool few = p.a.rows <= VMOST, pair = pairs > 0 && p.a.rows > 64 && tiles128 > 2LL * sms;
#ifdef TAB_TUNE
    if (const char* env = getenv("TAB_MATMUL")) { few = env[0] == 'v' && p.a.rows <= VMOST; pair = env[0] == 'p'; }
#endif
    if (few) return launch_rows(p, stream);
    if (pair) return launch_pair(p, pairs, status, stream);
    const BlocksPlan pl = blocks_plan(p.a.rows, p.b.rows, blocks_of(p.K), sms);
#define TAB_BT(BN, KS, SW) if (pl.bn == BN && pl.ks == KS && pl.swap == SW) return launch_tile_type<BN, KS, SW>(p, pl, status, stream)
    TAB_BT(16, 2, true); TAB_BT(32, 2, true); TAB_BT(64, 2, true);
    TAB_BT(16, 4, true); TAB_BT(32, 4, true); TAB_BT(64, 4, true);
    TAB_BT(64, 4, false); TAB_BT(128, 2, false); TAB_BT(128, 1, false);
#undef TAB_BT
    return TAB_E_TOO_LARGE;
}

}  // namespace tab
