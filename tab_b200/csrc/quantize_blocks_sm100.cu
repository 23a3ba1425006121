// fp32 / bf16 / fp16 values -> 8-bit floats with one power-of-two scale for each block of 128 (tab_quantize_blocks_launch).
//
// A block's scale is s = 2^e, e the least integer with max|x| <= F * 2^e (F the type's largest value), and its values are x / s
// rounded to nearest even.  x / s is exact (s is a power of two), so a value is rounded once, and the result does not depend on how
// the work is split.  Bytes are what bounds both kernels; every value is read once, whichever of the outputs are asked for:
//   rows     blocks along the rows only.  16 lanes hold a block, 8 values each; the maximum takes four shuffles.
//   tiles    blocks along rows and along columns, or squares of 128 x 128 and their transpose.  A CTA takes a square of 128 x 128 into
//            registers (8 rows x 8 columns a thread), finds its maxima, and turns the transposed bytes round in 16 KB of shared memory.
#include "blocks_common.cuh"

namespace tab {

static constexpr int QROWS = 4;              // blocks a half-warp of the rows kernel has in flight

// hk half-warps of the sixteen lie along K, the others along M.
template <int TYPE, int FORMAT>
__global__ void __launch_bounds__(256) quantize_rows_kernel(QuantBlocksParams p, int KB, int hk_log2, int chunks, int vec, int qvec) {
    using T = typename ElemOf<TYPE>::type;
    pdl_wait();
    const int half = threadIdx.x >> 4, l = threadIdx.x & 15;
    const int hk = 1 << hk_log2, rstep = 16 >> hk_log2;
    const int kb = (int)(blockIdx.x % (unsigned)chunks) * hk + (half & (hk - 1));
    const long long row0 = (long long)(blockIdx.x / (unsigned)chunks) * (rstep * QROWS) + (half >> hk_log2);
    const int k0 = kb * BLK + l * 8, n = kb < KB ? p.K - k0 : 0;
    float v[QROWS][8];
#pragma unroll
    for (int i = 0; i < QROWS; i++) {
        const long long m = row0 + i * rstep;
        load8(static_cast<const T*>(p.x) + m * p.ldx + k0, m < p.M ? n : 0, vec, v[i]);
    }
    pdl_launch_dependents();
#pragma unroll
    for (int i = 0; i < QROWS; i++) {
        const long long m = row0 + i * rstep;
        uint32_t a = 0;
#pragma unroll
        for (int j = 0; j < 8; j++) a = max(a, finite_bits(v[i][j]));
        const int e = scale_exponent(half_warp_max(a), FORMAT);
        if (m >= p.M || kb >= KB) continue;                                // (no shuffles below)
        store_bytes8(p.q + m * p.ldq + k0, n, qvec, narrow8<FORMAT>(v[i], exp2_int(-e)));
        if (l == 0) p.s[m * KB + kb] = (uint8_t)(e + 127);
    }
}

// 128 x 128 values: half-warp h holds rows 8h .. 8h+7, its lane l columns 8l .. 8l+7.
template <int TYPE, int FORMAT, bool SQUARE>
__global__ void __launch_bounds__(256, 2) quantize_tiles_kernel(QuantBlocksParams p, int KB, int MB, int vec, int qvec, int qtvec) {
    using T = typename ElemOf<TYPE>::type;
    __shared__ uint32_t colmax[16][BLK];
    __shared__ uint32_t colexp[BLK];
    __shared__ __align__(16) uint2 turned[BLK * 16];                       // [column][8 rows], chunks of a column permuted
    pdl_wait();
    const int half = threadIdx.x >> 4, l = threadIdx.x & 15;
    const int kb = (int)(blockIdx.x % (unsigned)KB);
    const long long mb = blockIdx.x / (unsigned)KB;
    const long long m0 = mb * BLK + half * 8;
    const int k0 = kb * BLK + l * 8, n = p.K - k0;
    float v[8][8];
#pragma unroll
    for (int r = 0; r < 8; r++) load8(static_cast<const T*>(p.x) + (m0 + r) * p.ldx + k0, m0 + r < p.M ? n : 0, vec, v[r]);
    pdl_launch_dependents();
    int ecol[8];
    if (SQUARE) {
        uint32_t a = 0;
#pragma unroll
        for (int r = 0; r < 8; r++)
#pragma unroll
            for (int c = 0; c < 8; c++) a = max(a, finite_bits(v[r][c]));
        a = half_warp_max(a);
        if (l == 0) colmax[0][half] = a;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 16; i++) a = max(a, colmax[0][i]);
        const int e = scale_exponent(a, FORMAT);
        if (threadIdx.x == 0) {
            if (p.s) p.s[mb * KB + kb] = (uint8_t)(e + 127);
            if (p.st) p.st[(long long)kb * MB + mb] = (uint8_t)(e + 127);
        }
        const float inv = exp2_int(-e);
        if (p.q) {
#pragma unroll
            for (int r = 0; r < 8; r++)
                if (m0 + r < p.M) store_bytes8(p.q + (m0 + r) * p.ldq + k0, n, qvec, narrow8<FORMAT>(v[r], inv));
        }
#pragma unroll
        for (int c = 0; c < 8; c++) ecol[c] = e;
    } else {
        uint32_t a[8];
#pragma unroll
        for (int c = 0; c < 8; c++) a[c] = 0;
#pragma unroll
        for (int r = 0; r < 8; r++) {
            uint32_t row = 0;
#pragma unroll
            for (int c = 0; c < 8; c++) {
                const uint32_t b = finite_bits(v[r][c]);
                row = max(row, b);
                a[c] = max(a[c], b);
            }
            const int e = scale_exponent(half_warp_max(row), FORMAT);
            if (m0 + r < p.M) {
                store_bytes8(p.q + (m0 + r) * p.ldq + k0, n, qvec, narrow8<FORMAT>(v[r], exp2_int(-e)));
                if (l == 0) p.s[(m0 + r) * KB + kb] = (uint8_t)(e + 127);
            }
        }
#pragma unroll
        for (int c = 0; c < 8; c++) colmax[half][l * 8 + c] = a[c];
        __syncthreads();
        if (threadIdx.x < BLK) {
            uint32_t b = 0;
#pragma unroll
            for (int i = 0; i < 16; i++) b = max(b, colmax[i][threadIdx.x]);
            const int e = scale_exponent(b, FORMAT);
            colexp[threadIdx.x] = (uint32_t)e;
            const long long k = (long long)kb * BLK + threadIdx.x;
            if (k < p.K) p.st[k * MB + mb] = (uint8_t)(e + 127);
        }
        __syncthreads();
#pragma unroll
        for (int c = 0; c < 8; c++) ecol[c] = (int)colexp[l * 8 + c];
    }
    if (SQUARE && !p.qt) return;
    // Chunk h of column c lies at place h ^ (c / 8): the sixteen lanes that write different columns, and the sixteen that read
    // different chunks, each meet all banks.
#pragma unroll
    for (int c = 0; c < 8; c++) {
        float t[8];
#pragma unroll
        for (int r = 0; r < 8; r++) t[r] = v[r][c];
        turned[(l * 8 + c) * 16 + (half ^ l)] = narrow8<FORMAT>(t, exp2_int(-ecol[c]));
    }
    __syncthreads();
    const long long mt = mb * BLK + l * 8;
    const int nt = (int)min((long long)8, p.M - mt);
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int c = half * 8 + i;
        const long long k = (long long)kb * BLK + c;
        if (k < p.K && nt > 0) store_bytes8(p.qt + k * p.ldqt + mt, nt, qtvec, turned[c * 16 + (l ^ half)]);
    }
}

template <int TYPE, int FORMAT>
static int launch_quantize_blocks(const QuantBlocksParams& p, bool square, cudaStream_t stream) {
    using T = typename ElemOf<TYPE>::type;
    const int KB = blocks_of(p.K);
    const uintptr_t xmask = 8 * sizeof(T) - 1;
    const int vec = !(reinterpret_cast<uintptr_t>(p.x) & xmask) && p.ldx % 8 == 0;
    const int qvec = !(reinterpret_cast<uintptr_t>(p.q) & 7) && p.ldq % 8 == 0, qtvec = !(reinterpret_cast<uintptr_t>(p.qt) & 7) && p.ldqt % 8 == 0;
    if (!square && !p.qt) {
        int hl = 0;
        while (hl < 4 && (1 << hl) < KB) hl++;
        const long long chunks = (KB + (1 << hl) - 1) >> hl, rows = (16 >> hl) * QROWS, grid = chunks * ((p.M + rows - 1) / rows);
        if (grid >= (1LL << 31)) return TAB_E_TOO_LARGE;
        return launch_pdl(quantize_rows_kernel<TYPE, FORMAT>, dim3((unsigned)grid), dim3(256), 0, stream, p, KB, hl, (int)chunks, vec, qvec);
    }
    const long long MB = (p.M + BLK - 1) / BLK, grid = MB * KB;
    if (grid >= (1LL << 31)) return TAB_E_TOO_LARGE;
    if (square) return launch_pdl(quantize_tiles_kernel<TYPE, FORMAT, true>, dim3((unsigned)grid), dim3(256), 0, stream, p, KB, (int)MB, vec, qvec, qtvec);
    return launch_pdl(quantize_tiles_kernel<TYPE, FORMAT, false>, dim3((unsigned)grid), dim3(256), 0, stream, p, KB, (int)MB, vec, qvec, qtvec);
}

int quantize_blocks_dispatch(const QuantBlocksParams& p, int type, bool square, cudaStream_t stream) {
#define TAB_QB(T) (p.format == TAB_E5M2 ? launch_quantize_blocks<T, TAB_E5M2>(p, square, stream) : launch_quantize_blocks<T, TAB_E4M3>(p, square, stream))
    return type == TAB_FP32 ? TAB_QB(TAB_FP32) : type == TAB_BF16 ? TAB_QB(TAB_BF16) : TAB_QB(TAB_FP16);
#undef TAB_QB
}

}  // namespace tab
