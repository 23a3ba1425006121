// fp32 / bf16 / fp16 values -> 8-bit floats with one power-of-two scale for each block of 128 (tab_quantize_blocks_launch).
//
// A block's scale is s = 2^e, e the least integer with max|x| <= F * 2^e (F the type's largest value), and its values are x / s
// rounded to nearest even.  x / s is exact (s is a power of two), so a value is rounded once, and the result does not depend on how
// the work is split.  Bytes are what bounds both kernels; every value is read once, whichever of the outputs are asked for:
//   rows     blocks along the rows only.  16 lanes hold a block, 8 values each; the maximum takes four shuffles.
//   tiles    blocks along rows and along columns, or squares of 128 x 128 and their transpose.  A CTA takes a square of 128 x 128 into
//            registers (8 rows x 8 columns a thread), finds its maxima, and turns the transposed bytes round in 16 KB of shared memory.
// us (TB/s of bytes that have to move), bf16: 8192x4096 rows 17.5 (5.8), both axes 25.1 (5.35), squares 15.6 (6.5), with their transpose 21.9 (6.1);
// 16384x8192 63 (6.4), 90 (6.0), 59 (6.8), 84 (6.4).  Both axes at half the instructions of the first form of these kernels (70 us).
#include <type_traits>
#include "blocks_common.cuh"
#include "umma_common.cuh"

namespace tab {

// Both kernels meet the memory's rate only if they spend few instructions on a value, hence: magnitudes of 16-bit types are compared two at
// a time as integers (the order of the bits is that of the values); NaN and infinities are looked for once and dealt with on a path of
// their own; bf16 is scaled two at a time, exactly, before it is widened; a block that lies inside x is worked without bounds.
template <int TYPE>
struct Eight {
    static constexpr int W = TYPE == TAB_FP32 ? 8 : 4;                     // words
    static constexpr uint32_t SIGNS = TYPE == TAB_FP32 ? 0x7FFFFFFFu : 0x7FFF7FFFu;
    static constexpr uint32_t INF = TYPE == TAB_FP32 ? 0x7F800000u : TYPE == TAB_BF16 ? 0x7F80u : 0x7C00u;
    uint32_t w[W];
    __device__ __forceinline__ void load_all(const void* p) {
        if (TYPE == TAB_FP32) {
            asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4 % W]), "=r"(w[5 % W]), "=r"(w[6 % W]), "=r"(w[7 % W]) : "l"(p));
        } else {
            const uint4 u = *static_cast<const uint4*>(p);
            w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
        }
    }
    // The first n of them exist; vec: aligned.
    __device__ __forceinline__ void load(const void* p, int n, bool vec) {
        if (vec && n >= 8) { load_all(p); return; }
#pragma unroll
        for (int i = 0; i < W; i++) w[i] = 0;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            if (i >= n) continue;
            if (TYPE == TAB_FP32) w[i % W] = static_cast<const uint32_t*>(p)[i];
            else w[i / 2 % W] |= (uint32_t)static_cast<const uint16_t*>(p)[i] << (16 * (i & 1));
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
    // All eight times a power of two, given as the bits of a float (for two columns' own factors: at even and at odd places).
    __device__ __forceinline__ void scaled(const uint32_t (&inv)[8], float (&v)[8]) const {
#pragma unroll
        for (int i = 0; i < W; i++) {
            if (TYPE == TAB_BF16) {
                const uint32_t f = __byte_perm(inv[2 * i % 8], inv[(2 * i + 1) % 8], 0x7632);    // their upper halves: two bf16
                const __nv_bfloat162 h = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&w[i]), *reinterpret_cast<const __nv_bfloat162*>(&f));
                const uint32_t u = *reinterpret_cast<const uint32_t*>(&h);
                v[2 * i % 8] = __uint_as_float(u << 16); v[(2 * i + 1) % 8] = __uint_as_float(u & 0xFFFF0000u);
            } else if (TYPE == TAB_FP32) {
                v[i] = at(i) * __uint_as_float(inv[i]);
            } else {
                v[2 * i % 8] = at(2 * i) * __uint_as_float(inv[2 * i % 8]); v[(2 * i + 1) % 8] = at(2 * i + 1) * __uint_as_float(inv[(2 * i + 1) % 8]);
            }
        }
    }
};

// Eight scaled values as bytes; `odd`: infinities may be among them.
template <int FORMAT>
__device__ __forceinline__ uint2 bytes8(const float (&v)[8], bool odd) {
    uint2 r;
    r.x = __byte_perm(narrow2<FORMAT>(v[0], v[1]), narrow2<FORMAT>(v[2], v[3]), 0x5410);
    r.y = __byte_perm(narrow2<FORMAT>(v[4], v[5]), narrow2<FORMAT>(v[6], v[7]), 0x5410);
    if (odd) r = narrow8<FORMAT>(v, 1.f);
    return r;
}

// Half-warps take blocks of two neighbouring columns of blocks (of one, where there is no more), the others rows, QROWS blocks each;
// scales are gathered so that those of a column of blocks leave side by side.
template <int TYPE, int FORMAT, int QROWS>
__global__ void __launch_bounds__(256) quantize_rows_kernel(QuantBlocksParams p, int KB, int two, FastDiv chunks, int vec, int qvec) {
    using T = typename ElemOf<TYPE>::type;
    using E = Eight<TYPE>;
    __shared__ uint8_t scales[16 * QROWS];
    const int half = threadIdx.x >> 4, l = threadIdx.x & 15;
    const int hr = half >> two, rstep = 16 >> two, rows = rstep * QROWS;
    const unsigned band = chunks.div(blockIdx.x), chunk = blockIdx.x - band * chunks.d;
    const int kb = (int)(chunk << two) + (half & two);
    const long long row0 = (long long)band * rows, m = row0 + hr;
    const int k0 = kb * BLK + l * 8, n = kb < KB ? p.K - k0 : 0;
    const T* x = static_cast<const T*>(p.x) + m * p.ldx + k0;
    uint8_t* q = p.q + m * p.ldq + k0;
    pdl_wait();
    auto work = [&](auto inside) {
        constexpr bool IN = decltype(inside)::value;
        E v[QROWS];
#pragma unroll
        for (int i = 0; i < QROWS; i++) {
            if (IN) v[i].load_all(x + i * rstep * p.ldx);
            else v[i].load(x + i * rstep * p.ldx, m + i * rstep < p.M ? n : 0, vec);
        }
        pdl_launch_dependents();
        uint32_t a[QROWS], high = 0;
#pragma unroll
        for (int i = 0; i < QROWS; i++) { a[i] = v[i].largest(false); high = max(high, a[i]); }
        const bool odd = __any_sync(0xFFFFFFFFu, high >= E::INF);
        if (odd)
#pragma unroll
            for (int i = 0; i < QROWS; i++) a[i] = v[i].largest(true);
#pragma unroll
        for (int i = 0; i < QROWS; i++) {
            const uint32_t s = scale_byte<FORMAT>(E::float_bits(half_warp_max(a[i])));
            if (l == 0) scales[(half & two) * rows + i * rstep + hr] = (uint8_t)s;
            const uint32_t f = inverse_bits(s), inv[8] = {f, f, f, f, f, f, f, f};
            float y[8];
            v[i].scaled(inv, y);
            const uint2 o = bytes8<FORMAT>(y, odd);
            if (IN) *reinterpret_cast<uint2*>(q + i * rstep * p.ldq) = o;
            else if (m + i * rstep < p.M && kb < KB) store_bytes8(q + i * rstep * p.ldq, n, qvec, o);
        }
    };
    if (vec && qvec && row0 + rows <= p.M && (int)((chunk + 1) << two) * BLK <= p.K) work(std::true_type());
    else work(std::false_type());
    __syncthreads();
    if ((int)threadIdx.x < rows << two) {
        const int r = threadIdx.x % rows, c = (int)(chunk << two) + threadIdx.x / rows;
        if (row0 + r < p.M && c < KB) p.s[c * p.lds + row0 + r] = scales[threadIdx.x];
    }
}

// 128 x 128 values: half-warp h holds rows 8h .. 8h+7, its lane l columns 8l .. 8l+7.
template <int TYPE, int FORMAT, bool SQUARE>
__global__ void __launch_bounds__(256, TYPE == TAB_FP32 ? 2 : SQUARE ? 4 : 3) quantize_tiles_kernel(QuantBlocksParams p, FastDiv KB, int vec, int qvec, int qtvec) {
    using T = typename ElemOf<TYPE>::type;
    using E = Eight<TYPE>;
    __shared__ uint32_t colmax[16][16 * E::W];                             // word i of lane l at [i * 16 + l]; a square's maxima: word 0
    __shared__ uint32_t colscale[BLK];                                     // of column 8l + c at [c * 16 + l]
    __shared__ __align__(16) uint2 turned[BLK * 16];                       // [column][8 rows], chunks of a column permuted
    const int half = threadIdx.x >> 4, l = threadIdx.x & 15;
    const long long mb = KB.div(blockIdx.x);
    const int kb = (int)(blockIdx.x - (unsigned)mb * KB.d);
    const long long m0 = mb * BLK + half * 8;
    const int k0 = kb * BLK + l * 8, n = p.K - k0;
    const T* x = static_cast<const T*>(p.x) + m0 * p.ldx + k0;
    pdl_wait();
    auto work = [&](auto inside) {
        constexpr bool IN = decltype(inside)::value;
        E v[8];
#pragma unroll
        for (int r = 0; r < 8; r++) {
            if (IN) v[r].load_all(x + r * p.ldx);
            else v[r].load(x + r * p.ldx, m0 + r < p.M ? n : 0, vec);
        }
        pdl_launch_dependents();
        uint32_t a[E::W], m[8];                                            // magnitudes of the columns, word by word; of the rows
        auto maxima = [&](bool odd) {
            uint32_t high = 0;
#pragma unroll
            for (int r = 0; r < 8; r++) {
                uint32_t row = 0;
#pragma unroll
                for (int i = 0; i < E::W; i++) {
                    const uint32_t u = v[r].size(i, odd);
                    row = i ? E::most(row, u) : u;
                    if (!SQUARE) a[i] = r ? E::most(a[i], u) : u;
                }
                if (!SQUARE) m[r] = E::one(row);
                high = r ? E::most(high, row) : row;
            }
            return E::one(high);
        };
        uint32_t high = maxima(false);
        const bool odd = __any_sync(0xFFFFFFFFu, high >= E::INF);
        if (odd) high = maxima(true);
        uint32_t mine;                                                     // the scale of row 8h + l / 2 of this half-warp, or the square's
        if (SQUARE) {
            high = half_warp_max(high);
            if (l == 0) colmax[half][0] = high;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 16; i++) high = max(high, colmax[i][0]);
            mine = scale_byte<FORMAT>(E::float_bits(high));
            if (threadIdx.x == 0) {
                if (p.s) p.s[mb * p.lds + kb] = (uint8_t)mine;
                if (p.st) p.st[kb * p.ldst + mb] = (uint8_t)mine;
            }
        } else {
#pragma unroll
            for (int i = 0; i < E::W; i++) colmax[half][i * 16 + l] = a[i];
            // Eight rows' maxima over sixteen lanes: in every step a lane hands half of its rows to its neighbour and keeps the others, eight
            // shuffles instead of 32, and each lane then finds one row's scale instead of eight.
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
            mine = scale_byte<FORMAT>(E::float_bits(m[0]));
            if (!(l & 1) && m0 + l / 2 < p.M) p.s[kb * p.lds + m0 + l / 2] = (uint8_t)mine;
            __syncthreads();
            if (threadIdx.x < 16 * E::W) {                                 // a thread: the columns of one word
                uint32_t b = 0;
#pragma unroll
                for (int i = 0; i < 16; i++) b = E::most(b, colmax[i][threadIdx.x]);
#pragma unroll
                for (int c = 0; c < 8 / E::W; c++)
                    colscale[(half * (8 / E::W) + c) * 16 + l] = scale_byte<FORMAT>(E::float_bits(TYPE == TAB_FP32 ? b : b >> (16 * c) & 0xFFFFu));
            }
        }
        if (!SQUARE || p.q) {
            uint8_t* q = p.q + m0 * p.ldq + k0;
#pragma unroll
            for (int r = 0; r < 8; r++) {
                const uint32_t f = inverse_bits(SQUARE ? mine : __shfl_sync(0xFFFFFFFFu, mine, (threadIdx.x & 16) + 2 * r)), inv[8] = {f, f, f, f, f, f, f, f};
                float y[8];
                v[r].scaled(inv, y);
                const uint2 o = bytes8<FORMAT>(y, odd);
                if (IN) *reinterpret_cast<uint2*>(q + r * p.ldq) = o;
                else if (m0 + r < p.M) store_bytes8(q + r * p.ldq, n, qvec, o);
            }
        }
        if (SQUARE && !p.qt) return;
        if (!SQUARE) __syncthreads();
        // Chunk h of column c lies at place h ^ (c / 8): the sixteen lanes that write different columns, and the sixteen that read
        // different chunks, each meet all banks.  The values are scaled pair by pair of columns and written column by column.
        uint32_t inv[8];
#pragma unroll
        for (int c = 0; c < 8; c++) inv[c] = inverse_bits(SQUARE ? mine : colscale[c * 16 + l]);
#pragma unroll
        for (int c = 0; c < 8; c += 8 / E::W) {
            float y[8 / E::W][8];
#pragma unroll
            for (int r = 0; r < 8; r++) {
                if (TYPE == TAB_BF16) {
                    const uint32_t f = __byte_perm(inv[c], inv[c + 1], 0x7632);
                    const __nv_bfloat162 h = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&v[r].w[c / 2 % E::W]), *reinterpret_cast<const __nv_bfloat162*>(&f));
                    const uint32_t u = *reinterpret_cast<const uint32_t*>(&h);
                    y[0][r] = __uint_as_float(u << 16); y[8 / E::W - 1][r] = __uint_as_float(u & 0xFFFF0000u);
                } else {
#pragma unroll
                    for (int i = 0; i < 8 / E::W; i++) y[i][r] = v[r].at(c + i) * __uint_as_float(inv[c + i]);
                }
            }
#pragma unroll
            for (int i = 0; i < 8 / E::W; i++) turned[(l * 8 + c + i) * 16 + (half ^ l)] = bytes8<FORMAT>(y[i], odd);
        }
        __syncthreads();
        const long long mt = mb * BLK + l * 8;
        uint8_t* qt = p.qt + (kb * BLK + half * 8) * p.ldqt + mt;
        const int nt = (int)min((long long)8, p.M - mt);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const uint2 o = turned[(half * 8 + i) * 16 + (l ^ half)];
            if (IN) *reinterpret_cast<uint2*>(qt + i * p.ldqt) = o;
            else if (kb * BLK + half * 8 + i < p.K && nt > 0) store_bytes8(qt + i * p.ldqt, nt, qtvec, o);
        }
        if (!SQUARE && threadIdx.x < BLK && kb * BLK + (int)threadIdx.x < p.K)
            p.st[mb * p.ldst + kb * BLK + threadIdx.x] = (uint8_t)colscale[(threadIdx.x & 7) * 16 + (threadIdx.x >> 3)];
    };
    if (vec && qvec && qtvec && (mb + 1) * BLK <= p.M && (kb + 1) * BLK <= p.K) work(std::true_type());
    else work(std::false_type());
}

template <int TYPE, int FORMAT>
static int launch_quantize_blocks(const QuantBlocksParams& p, bool square, cudaStream_t stream) {
    using T = typename ElemOf<TYPE>::type;
    const int KB = blocks_of(p.K);
    const uintptr_t xmask = 8 * sizeof(T) - 1;
    const int vec = !(reinterpret_cast<uintptr_t>(p.x) & xmask) && p.ldx % 8 == 0;
    const int qvec = !(reinterpret_cast<uintptr_t>(p.q) & 7) && p.ldq % 8 == 0, qtvec = !(reinterpret_cast<uintptr_t>(p.qt) & 7) && p.ldqt % 8 == 0;
    const long long MB = (p.M + BLK - 1) / BLK;
    if (MB * KB >= (1LL << 27)) return TAB_E_TOO_LARGE;                    // 2^41 values, and grids of CTAs of 16 blocks below 2^31
    if (!square && !p.qt) {
        // four blocks a half-warp where that leaves every SM several CTAs (8192x4096: 17.4 us, one 23.1), one where there is little to do (64x4096: 1.6, four 2.2)
        const int two = KB > 1;
        const long long chunks = (KB + two) >> two, blocks = p.M * KB;
        const FastDiv by = make_fastdiv((uint32_t)chunks);
#define TAB_QR(N) launch_pdl(quantize_rows_kernel<TYPE, FORMAT, N>, dim3((unsigned)(chunks * ((p.M + (16 >> two) * N - 1) / ((16 >> two) * N)))), dim3(256), 0, stream, p, KB, two, by, vec, qvec)
        return blocks >= 1 << 16 ? TAB_QR(4) : TAB_QR(1);
#undef TAB_QR
    }
    const FastDiv by = make_fastdiv((uint32_t)KB);
    if (square) return launch_pdl(quantize_tiles_kernel<TYPE, FORMAT, true>, dim3((unsigned)(MB * KB)), dim3(256), 0, stream, p, by, vec, qvec, qtvec);
    return launch_pdl(quantize_tiles_kernel<TYPE, FORMAT, false>, dim3((unsigned)(MB * KB)), dim3(256), 0, stream, p, by, vec, qvec, qtvec);
}

int quantize_blocks_dispatch(const QuantBlocksParams& p, int type, bool square, cudaStream_t stream) {
#define TAB_QB(T) (p.format == TAB_E5M2 ? launch_quantize_blocks<T, TAB_E5M2>(p, square, stream) : launch_quantize_blocks<T, TAB_E4M3>(p, square, stream))
    return type == TAB_FP32 ? TAB_QB(TAB_FP32) : type == TAB_BF16 ? TAB_QB(TAB_BF16) : TAB_QB(TAB_FP16);
#undef TAB_QB
}

}  // namespace tab
