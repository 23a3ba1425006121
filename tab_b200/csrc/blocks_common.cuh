// 8-bit floats in blocks of 128 with one power-of-two scale each, and the operators around them: types, scales and element access
// shared by the kernels behind tab_quantize_blocks_launch, tab_matmul_blocks_launch and tab_residual_norm_launch.
#pragma once
#include <atomic>
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "tab_kernels.cuh"

namespace tab {

constexpr int BLK = 128;                     // values that share a scale

inline int blocks_of(long long n) { return (int)((n + BLK - 1) / BLK); }
// SMs of the current device.
inline int blocks_sms() {
    static std::atomic<int> known[64];
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
    n = known[dev].load(std::memory_order_relaxed);
    if (n == 0) {
        if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) { cudaGetLastError(); n = 148; }
        known[dev].store(n, std::memory_order_relaxed);
    }
    return n;
}
inline int type_bytes(int type) { return type == TAB_FP32 ? 4 : 2; }

// What the quantiser is given.  Pitches are in elements; a null output is not written.
struct QuantBlocksParams {
    const void* x;
    long long ldx, M;
    int K;
    int format;                              // TAB_E4M3 or TAB_E5M2
    uint8_t* q;                              // [M][K], row pitch ldq
    long long ldq;
    uint8_t* s;                              // rows: [ceil(K/128)][M], pitch lds; squares: [ceil(M/128)][ceil(K/128)]
    long long lds;
    uint8_t* qt;                             // [K][M], row pitch ldqt
    long long ldqt;
    uint8_t* st;                             // columns: [ceil(M/128)][K], pitch ldst; squares: the transpose of s
    long long ldst;
};
int quantize_blocks_dispatch(const QuantBlocksParams& p, int type, bool square, cudaStream_t stream);

// One operand of the product: values [rows][K] with pitch ld (bytes), scale of (row, k) at s[(row >> shift) * sr + (k / 128) * sk].
struct BlocksOperand {
    const uint8_t* q;
    long long ld;
    const uint8_t* s;
    long long sr, sk;
    int shift;                               // 0: a scale for each row, 7: for each 128 rows
    int rows;
    int format;
};
struct MatmulBlocksParams {
    BlocksOperand a, b;
    void* y;
    long long ldy;                           // elements
    int type;                                // of y
    int K;
};
int matmul_blocks_dispatch(const MatmulBlocksParams& p, cudaStream_t stream);

using NormParams = tab_norm_t;
using NormBackwardParams = tab_norm_backward_t;
int residual_norm_dispatch(const NormParams& p, int type, cudaStream_t stream);
int residual_norm_backward_dispatch(const NormBackwardParams& p, int type, cudaStream_t stream);
size_t residual_norm_partial_bytes(long long M, int C);
constexpr int NORM_MAX = 16384;              // elements of a row
const char* matmul_blocks_last_kernel();

#ifdef __CUDACC__

template <int TYPE> struct ElemOf { using type = float; };
template <> struct ElemOf<TAB_BF16> { using type = __nv_bfloat16; };
template <> struct ElemOf<TAB_FP16> { using type = __half; };

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

// Eight consecutive elements as floats.  n: how many of them exist (the others read as 0); vec: they start on a boundary of their
// own size (32 or 16 bytes) wherever all eight exist.
__device__ __forceinline__ void widen8(const uint4& u, float (&v)[8], __nv_bfloat16) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; i++) { v[2 * i] = __uint_as_float(w[i] << 16); v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u); }
}
__device__ __forceinline__ void widen8(const uint4& u, float (&v)[8], __half) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        v[2 * i] = f.x; v[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ void load8(const float* p, int n, bool vec, float (&v)[8]) {
    if (vec && n >= 8) {
        asm volatile("ld.global.v8.f32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                     : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]) : "l"(p));
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = i < n ? p[i] : 0.f;
}
template <typename T>
__device__ __forceinline__ void load8(const T* p, int n, bool vec, float (&v)[8]) {
    if (vec && n >= 8) {
        widen8(*reinterpret_cast<const uint4*>(p), v, T());
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = i < n ? to_float(p[i]) : 0.f;
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __half) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(float a, float, float) { return __float_as_uint(a); }   // (fp32 has nothing to pack)
__device__ __forceinline__ void store8(float* p, int n, bool vec, const float (&v)[8]) {
    if (vec && n >= 8) {
        asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
                     :: "l"(p), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]) : "memory");
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; i++) if (i < n) p[i] = v[i];
}
template <typename T>
__device__ __forceinline__ void store8(T* p, int n, bool vec, const float (&v)[8]) {
    if (vec && n >= 8) {
        *reinterpret_cast<uint4*>(p) = make_uint4(pack2(v[0], v[1], T()), pack2(v[2], v[3], T()), pack2(v[4], v[5], T()), pack2(v[6], v[7], T()));
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; i++) if (i < n) p[i] = from_float<T>(v[i]);
}

// ---- scales ------------------------------------------------------------------------------------------------------------------
// Magnitude bits of v for the block's maximum: NaN and infinities do not count (they keep to their own element).
__device__ __forceinline__ uint32_t finite_bits(float v) {
    const uint32_t b = __float_as_uint(v) & 0x7FFFFFFFu;
    return b < 0x7F800000u ? b : 0u;
}
// e + 127 of the block's scale 2^e, e the least with amax <= F * 2^e for F = 1.75 * 2^8 (e4m3) or 1.75 * 2^15 (e5m2), from the bits of amax = m * 2^k:
// k - 8 (k - 15), one more where m > 1.75, which the addition carries into the exponent; at least 0, the least a byte holds (which subnormal
// maxima fall below); 127 for a block of zeros.
template <int FORMAT>
__device__ __forceinline__ uint32_t scale_byte(uint32_t bits) {
    const int b = (int)((bits + 0x1FFFFFu) >> 23) - (FORMAT == TAB_E5M2 ? 15 : 8);
    return bits == 0 ? 127u : (uint32_t)max(b, 0);
}
// 2^-e as the bits of a float: e + 127 is at most 247, so this is a normal number.
__device__ __forceinline__ uint32_t inverse_bits(uint32_t scale) { return (254u - scale) << 23; }
// 2^n for -127 <= n <= 127.
__device__ __forceinline__ float exp2_int(int n) { return __uint_as_float(n == -127 ? 0x00400000u : (uint32_t)(n + 127) << 23); }

// Two values, already divided by their scale, to the nearest 8-bit floats (ties to even): a in the low byte.  The scale keeps finite
// values within the type's range, so the conversion's saturation never acts on one of them; it does on infinities, which mend8 puts right.
template <int FORMAT>
__device__ __forceinline__ uint32_t narrow2(float a, float b) {
    uint16_t r;
    if (FORMAT == TAB_E5M2) asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
    else asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
    return r;
}
// The byte of an infinity: e5m2 has infinities, e4m3 has not and takes its NaN.
template <int FORMAT>
__device__ __forceinline__ uint32_t infinity8(float v) { return FORMAT == TAB_E5M2 ? (v < 0 ? 0xFCu : 0x7Cu) : 0x7Fu; }
// Eight values of one block as bytes.
template <int FORMAT>
__device__ __forceinline__ uint2 narrow8(const float (&v)[8], float inv) {
    uint2 r;
    r.x = narrow2<FORMAT>(v[0] * inv, v[1] * inv) | narrow2<FORMAT>(v[2] * inv, v[3] * inv) << 16;
    r.y = narrow2<FORMAT>(v[4] * inv, v[5] * inv) | narrow2<FORMAT>(v[6] * inv, v[7] * inv) << 16;
    uint32_t high = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) high = max(high, __float_as_uint(v[i]) & 0x7FFFFFFFu);
    if (high >= 0x7F800000u) {
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (isinf(v[i])) {
                uint32_t& w = i < 4 ? r.x : r.y;
                w = (w & ~(0xFFu << (8 * (i & 3)))) | infinity8<FORMAT>(v[i]) << (8 * (i & 3));
            }
    }
    return r;
}
// Eight bytes of which the first n exist.
__device__ __forceinline__ void store_bytes8(uint8_t* p, int n, bool vec, uint2 v) {
    if (vec && n >= 8) {
        *reinterpret_cast<uint2*>(p) = v;
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; i++) if (i < n) p[i] = (uint8_t)((i < 4 ? v.x : v.y) >> (8 * (i & 3)));
}
// Maximum over the 16 lanes of a half-warp.
__device__ __forceinline__ uint32_t half_warp_max(uint32_t v) {
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
    return v;
}

#endif  // __CUDACC__

}  // namespace tab
