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

// Eight values as they are loaded, so that 16-bit types take half of the registers; their magnitudes are compared as integers, two at a
// time (the order of the bits is that of the values).
template <int TYPE>
struct Eight {
    static constexpr int W = TYPE == TAB_FP32 ? 8 : 4;                     // words
    static constexpr uint32_t SIGNS = TYPE == TAB_FP32 ? 0x7FFFFFFFu : 0x7FFF7FFFu;
    static constexpr uint32_t INF = TYPE == TAB_FP32 ? 0x7F800000u : TYPE == TAB_BF16 ? 0x7F80u : 0x7C00u;
    uint32_t w[W];
    template <typename T>
    __device__ __forceinline__ void load(const T* p, int n, bool vec) {
        if (vec && n >= 8) {
            if (TYPE == TAB_FP32) {
                asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4 % W]), "=r"(w[5 % W]), "=r"(w[6 % W]), "=r"(w[7 % W]) : "l"(p));
            } else {
                const uint4 u = *reinterpret_cast<const uint4*>(p);
                w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
            }
            return;
        }
#pragma unroll
        for (int i = 0; i < W; i++) w[i] = 0;
        if (n <= 0) return;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            if (i >= n) continue;
            if (TYPE == TAB_FP32) w[i % W] = reinterpret_cast<const uint32_t*>(p)[i];
            else w[i / 2 % W] |= (uint32_t)reinterpret_cast<const uint16_t*>(p)[i] << (16 * (i & 1));
        }
    }
    __device__ __forceinline__ float at(int i) const {
        if (TYPE == TAB_FP32) return __uint_as_float(w[i % W]);
        const uint32_t u = w[i / 2 % W];
        if (TYPE == TAB_BF16) return __uint_as_float(i & 1 ? u & 0xFFFF0000u : u << 16);
        return __half2float(__ushort_as_half((unsigned short)(i & 1 ? u >> 16 : u & 0xFFFFu)));
    }
    // Word i's magnitudes; with `odd` those of NaN and infinities are 0 (they keep to their own element).
    __device__ __forceinline__ uint32_t size(int i, bool odd) const {
        uint32_t u = w[i] & SIGNS;
        if (odd) {
            if (TYPE == TAB_FP32) u = u < INF ? u : 0u;
            else u = ((u & 0xFFFFu) < INF ? u & 0xFFFFu : 0u) | ((u >> 16) < INF ? u & 0xFFFF0000u : 0u);
        }
        return u;
    }
    static __device__ __forceinline__ uint32_t most(uint32_t a, uint32_t b) { return TYPE == TAB_FP32 ? max(a, b) : __vmaxu2(a, b); }
    // The larger of a word's magnitudes, in the type's bits; and those bits as the bits of a float.
    static __device__ __forceinline__ uint32_t one(uint32_t a) { return TYPE == TAB_FP32 ? a : max(a & 0xFFFFu, a >> 16); }
    static __device__ __forceinline__ uint32_t float_bits(uint32_t a) {
        return TYPE == TAB_FP32 ? a : TYPE == TAB_BF16 ? a << 16 : __float_as_uint(__half2float(__ushort_as_half((unsigned short)a)));
    }
    __device__ __forceinline__ uint32_t largest(bool odd) const {
        uint32_t m = size(0, odd);
#pragma unroll
        for (int i = 1; i < W; i++) m = most(m, size(i, odd));
        return one(m);
    }
};
// narrow8 of eight floats where `odd` says that there may be infinities among them.
template <int FORMAT>
__device__ __forceinline__ uint2 narrow8_of(const float (&v)[8], float inv, bool odd) {
    if (odd) return narrow8<FORMAT>(v, inv);
    uint2 r;
    r.x = narrow2<FORMAT>(v[0] * inv, v[1] * inv) | narrow2<FORMAT>(v[2] * inv, v[3] * inv) << 16;
    r.y = narrow2<FORMAT>(v[4] * inv, v[5] * inv) | narrow2<FORMAT>(v[6] * inv, v[7] * inv) << 16;
    return r;
}

static constexpr int QROWS = 2;              // blocks a half-warp of the rows kernel has in flight

// Half-warps take blocks of two neighbouring columns of blocks (of one, where there is no more), the others rows; scales are gathered so
// that those of a column of blocks leave side by side.
template <int TYPE, int FORMAT>
__global__ void __launch_bounds__(256) quantize_rows_kernel(QuantBlocksParams p, int KB, int two, int chunks, int vec, int qvec) {
    using T = typename ElemOf<TYPE>::type;
    using E = Eight<TYPE>;
    __shared__ uint8_t scales[16 * QROWS];
    pdl_wait();
    const int half = threadIdx.x >> 4, l = threadIdx.x & 15;
    const int hr = half >> two, rstep = 16 >> two, rows = rstep * QROWS;
    const int kb = (int)(blockIdx.x % (unsigned)chunks << two) + (half & two);
    const long long row0 = (long long)(blockIdx.x / (unsigned)chunks) * rows;
    const int k0 = kb * BLK + l * 8, n = kb < KB ? p.K - k0 : 0;
    E v[QROWS];
#pragma unroll
    for (int i = 0; i < QROWS; i++) {
        const long long m = row0 + i * rstep + hr;
        v[i].load(static_cast<const T*>(p.x) + m * p.ldx + k0, m < p.M ? n : 0, vec);
    }
    pdl_launch_dependents();
    uint32_t high = 0;
#pragma unroll
    for (int i = 0; i < QROWS; i++) high = max(high, v[i].largest(false));
    const bool odd = __any_sync(0xFFFFFFFFu, high >= E::INF);
#pragma unroll
    for (int i = 0; i < QROWS; i++) {
        const long long m = row0 + i * rstep + hr;
        const int e = scale_exponent(E::float_bits(half_warp_max(v[i].largest(odd))), FORMAT);
        if (l == 0) scales[(half & two) * rows + i * rstep + hr] = (uint8_t)(e + 127);
        float f[8];
#pragma unroll
        for (int j = 0; j < 8; j++) f[j] = v[i].at(j);
        if (m < p.M && kb < KB) store_bytes8(p.q + m * p.ldq + k0, n, qvec, narrow8_of<FORMAT>(f, exp2_int(-e), odd));
    }
    __syncthreads();
    if ((int)threadIdx.x < rows << two) {
        const int r = threadIdx.x % rows, c = (int)(blockIdx.x % (unsigned)chunks << two) + threadIdx.x / rows;
        if (row0 + r < p.M && c < KB) p.s[c * p.lds + row0 + r] = scales[threadIdx.x];
    }
}

// 128 x 128 values: half-warp h holds rows 8h .. 8h+7, its lane l columns 8l .. 8l+7.
template <int TYPE, int FORMAT, bool SQUARE>
__global__ void __launch_bounds__(256, TYPE == TAB_FP32 ? 2 : SQUARE ? 4 : 3) quantize_tiles_kernel(QuantBlocksParams p, int KB, int vec, int qvec, int qtvec) {
    using T = typename ElemOf<TYPE>::type;
    using E = Eight<TYPE>;
    __shared__ uint32_t colmax[16][16 * E::W];                             // word i of lane l at [i * 16 + l]; a square's maxima: word 0
    __shared__ int colexp[BLK];                                            // of column 8l + c at [c * 16 + l]
    __shared__ __align__(16) uint2 turned[BLK * 16];                       // [column][8 rows], chunks of a column permuted
    pdl_wait();
    const int half = threadIdx.x >> 4, l = threadIdx.x & 15;
    const int kb = (int)(blockIdx.x % (unsigned)KB);
    const long long mb = blockIdx.x / (unsigned)KB;
    const long long m0 = mb * BLK + half * 8;
    const int k0 = kb * BLK + l * 8, n = p.K - k0;
    E v[8];
#pragma unroll
    for (int r = 0; r < 8; r++) v[r].load(static_cast<const T*>(p.x) + (m0 + r) * p.ldx + k0, m0 + r < p.M ? n : 0, vec);
    pdl_launch_dependents();
    uint32_t a[E::W];
    auto maxima = [&](bool odd) {
#pragma unroll
        for (int i = 0; i < E::W; i++) a[i] = v[0].size(i, odd);
#pragma unroll
        for (int r = 1; r < 8; r++)
#pragma unroll
            for (int i = 0; i < E::W; i++) a[i] = E::most(a[i], v[r].size(i, odd));
        uint32_t m = a[0];
#pragma unroll
        for (int i = 1; i < E::W; i++) m = E::most(m, a[i]);
        return E::one(m);
    };
    uint32_t high = maxima(false);
    const bool odd = __any_sync(0xFFFFFFFFu, high >= E::INF);
    if (odd) high = maxima(true);
    int e = 0;                                                             // a square's scale
    if (SQUARE) {
        high = half_warp_max(high);
        if (l == 0) colmax[half][0] = high;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 16; i++) high = max(high, colmax[i][0]);
        e = scale_exponent(E::float_bits(high), FORMAT);
        if (threadIdx.x == 0) {
            if (p.s) p.s[mb * p.lds + kb] = (uint8_t)(e + 127);
            if (p.st) p.st[kb * p.ldst + mb] = (uint8_t)(e + 127);
        }
    } else {
#pragma unroll
        for (int i = 0; i < E::W; i++) colmax[half][i * 16 + l] = a[i];
        __syncthreads();
        if (threadIdx.x < 16 * E::W) {                                     // a thread: the columns of one word
            uint32_t b = 0;
#pragma unroll
            for (int i = 0; i < 16; i++) b = E::most(b, colmax[i][threadIdx.x]);
#pragma unroll
            for (int c = 0; c < 8 / E::W; c++) {
                const int in8 = half * (8 / E::W) + c;                     // of the lane's eight columns
                const int ec = scale_exponent(E::float_bits(TYPE == TAB_FP32 ? b : b >> (16 * c) & 0xFFFFu), FORMAT);
                colexp[in8 * 16 + l] = ec;
            }
        }
    }
    int mine = e;                                                          // the scale of row 8h + l / 2 of this half-warp, in lane l
    if (!SQUARE) {
        // Eight rows' maxima over sixteen lanes: in every step a lane hands half of its rows to its neighbour and keeps the others, eight
        // shuffles instead of 32, and each lane then finds one row's scale instead of eight.
        uint32_t m[8];
#pragma unroll
        for (int r = 0; r < 8; r++) m[r] = v[r].largest(odd);
#pragma unroll
        for (int o = 8; o > 1; o >>= 1) {
            const bool upper = l & o;
#pragma unroll
            for (int r = 0; r < o / 2; r++) {
                const uint32_t give = upper ? m[r] : m[r + o / 2], keep = upper ? m[r + o / 2] : m[r];
                m[r] = max(keep, __shfl_xor_sync(0xFFFFFFFFu, give, o));
            }
        }
        m[0] = max(m[0], __shfl_xor_sync(0xFFFFFFFFu, m[0], 1));
        mine = scale_exponent(E::float_bits(m[0]), FORMAT);
        if (!(l & 1) && m0 + l / 2 < p.M) p.s[kb * p.lds + m0 + l / 2] = (uint8_t)(mine + 127);
    }
    if (!SQUARE || p.q) {
#pragma unroll
        for (int r = 0; r < 8; r++) {
            const int er = SQUARE ? e : __shfl_sync(0xFFFFFFFFu, mine, (threadIdx.x & 16) + 2 * r);
            float f[8];
#pragma unroll
            for (int c = 0; c < 8; c++) f[c] = v[r].at(c);
            if (m0 + r < p.M) store_bytes8(p.q + (m0 + r) * p.ldq + k0, n, qvec, narrow8_of<FORMAT>(f, exp2_int(-er), odd));
        }
    }
    if (SQUARE && !p.qt) return;
    __syncthreads();
    if (!SQUARE && threadIdx.x < BLK && kb * BLK + (int)threadIdx.x < p.K)
        p.st[mb * p.ldst + kb * BLK + threadIdx.x] = (uint8_t)(colexp[(threadIdx.x & 7) * 16 + (threadIdx.x >> 3)] + 127);
    // Chunk h of column c lies at place h ^ (c / 8): the sixteen lanes that write different columns, and the sixteen that read
    // different chunks, each meet all banks.
#pragma unroll
    for (int c = 0; c < 8; c++) {
        float f[8];
#pragma unroll
        for (int r = 0; r < 8; r++) f[r] = v[r].at(c);
        turned[(l * 8 + c) * 16 + (half ^ l)] = narrow8_of<FORMAT>(f, exp2_int(SQUARE ? -e : -colexp[c * 16 + l]), odd);
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
        const int two = KB > 1;
        const long long chunks = (KB + two) >> two, rows = (16 >> two) * QROWS, grid = chunks * ((p.M + rows - 1) / rows);
        if (grid >= (1LL << 31)) return TAB_E_TOO_LARGE;
        return launch_pdl(quantize_rows_kernel<TYPE, FORMAT>, dim3((unsigned)grid), dim3(256), 0, stream, p, KB, two, (int)chunks, vec, qvec);
    }
    const long long MB = (p.M + BLK - 1) / BLK, grid = MB * KB;
    if (grid >= (1LL << 31)) return TAB_E_TOO_LARGE;
    if (square) return launch_pdl(quantize_tiles_kernel<TYPE, FORMAT, true>, dim3((unsigned)grid), dim3(256), 0, stream, p, KB, vec, qvec, qtvec);
    return launch_pdl(quantize_tiles_kernel<TYPE, FORMAT, false>, dim3((unsigned)grid), dim3(256), 0, stream, p, KB, vec, qvec, qtvec);
}

int quantize_blocks_dispatch(const QuantBlocksParams& p, int type, bool square, cudaStream_t stream) {
#define TAB_QB(T) (p.format == TAB_E5M2 ? launch_quantize_blocks<T, TAB_E5M2>(p, square, stream) : launch_quantize_blocks<T, TAB_E4M3>(p, square, stream))
    return type == TAB_FP32 ? TAB_QB(TAB_FP32) : type == TAB_BF16 ? TAB_QB(TAB_BF16) : TAB_QB(TAB_FP16);
#undef TAB_QB
}

}  // namespace tab
