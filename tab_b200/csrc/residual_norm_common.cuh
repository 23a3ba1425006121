// The norm after a block with its gate, the scaled residual, and the norm before the next block in one pass over the rows
// (tab_residual_norm_launch), and the gradients of all of it in one pass and a short sum (tab_residual_norm_backward_launch).
//
// With v^ = (v - mean) / sqrt(var + eps) (centred), or v / sqrt(mean v^2 + eps):
//   u = y^ w1 + b1,  r = alpha x + g u  (kept in the type of y; what is normalised is what is kept),  h = r^ w2 + b2;
//   dr = gr + D(gh w2; r),  dx = alpha dr,  dg = dr u,  du = g dr,  dy = D(du w1; y),  dw = sum over rows of (gradient) v^,  db = sum of (gradient),
//   D(t; v) = (t - v^ mean(t v^) - [centred: mean t]) / deviation.
// Bytes bound both.  A row lies in the registers of 32 to 1024 threads, eight consecutive elements at a time, and is read once; sums
// over a row go through shuffles and one exchange in shared memory, in fp32, a variance as the mean of squared differences from the
// mean.  Sums over rows (weights', shifts' and channel gate's gradients) stay in the registers of the threads that own the columns
// while a CTA walks through its rows; the CTAs' sums are added in a fixed order by a second launch: no atomics, the same bits every time.
#pragma once
#include <algorithm>
#include <mutex>
#include <type_traits>
#include "blocks_common.cuh"
#include "umma_common.cuh"

namespace tab {

__device__ __forceinline__ void load8_any(const void* p, int type, long long at, int n, bool vec, float (&v)[8]) {
    if (type == TAB_FP32) load8(static_cast<const float*>(p) + at, n, vec, v);
    else if (type == TAB_BF16) load8(static_cast<const __nv_bfloat16*>(p) + at, n, vec, v);
    else load8(static_cast<const __half*>(p) + at, n, vec, v);
}
__device__ __forceinline__ float load_any(const void* p, int type, long long at) {
    return type == TAB_FP32 ? static_cast<const float*>(p)[at] : type == TAB_BF16 ? to_float(static_cast<const __nv_bfloat16*>(p)[at]) : to_float(static_cast<const __half*>(p)[at]);
}
__device__ __forceinline__ void store8_any(void* p, int type, long long at, int n, bool vec, const float (&v)[8]) {
    if (type == TAB_FP32) store8(static_cast<float*>(p) + at, n, vec, v);
    else if (type == TAB_BF16) store8(static_cast<__nv_bfloat16*>(p) + at, n, vec, v);
    else store8(static_cast<__half*>(p) + at, n, vec, v);
}
__device__ __forceinline__ void store_any(void* p, int type, long long at, float v) {
    if (type == TAB_FP32) static_cast<float*>(p)[at] = v;
    else if (type == TAB_BF16) static_cast<__nv_bfloat16*>(p)[at] = __float2bfloat16_rn(v);
    else static_cast<__half*>(p)[at] = __float2half_rn(v);
}

// Which tensors' rows start on the boundary of eight elements (host side fills it in).
enum { V_Y = 1, V_X = 2, V_R = 4, V_H = 8, V_Q = 16, V_W1 = 32, V_B1 = 64, V_W2 = 128, V_B2 = 256, V_G = 512, V_GR = 1024, V_GH = 2048, V_DY = 4096, V_DX = 8192, V_DG = 16384 };

// The columns of a thread, NV times eight of them.  VEC: eight neighbours, which move as one vector (all rows start on eight elements and
// have a multiple of them); else every 32nd of a warp's 256, so that a warp's single elements lie side by side.
template <int GT, int NV, bool VEC>
struct Columns {
    int g, C;
    __device__ __forceinline__ int at(int i, int j) const { return VEC ? (i * GT + g) * 8 + j : (i * GT + (g & ~31)) * 8 + j * 32 + (g & 31); }
    __device__ __forceinline__ bool in(int i, int j) const { return at(i, VEC ? 0 : j) < C; }
    template <typename T>
    __device__ __forceinline__ void singles(const T* p, int n, float (&v)[8]) const {
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = 32 * j < n ? to_float(p[32 * j]) : 0.f;
    }
    template <typename T>
    __device__ __forceinline__ void put(T* p, int n, const float (&v)[8]) const {
#pragma unroll
        for (int j = 0; j < 8; j++) if (32 * j < n) p[32 * j] = from_float<T>(v[j]);
    }
    __device__ __forceinline__ void load(const void* p, int type, long long row, int i, float (&v)[8]) const {
        const int c = at(i, 0);
        if (VEC) load8_any(p, type, row + c, c < C ? 8 : 0, true, v);
        else if (type == TAB_FP32) singles(static_cast<const float*>(p) + row + c, C - c, v);
        else if (type == TAB_BF16) singles(static_cast<const __nv_bfloat16*>(p) + row + c, C - c, v);
        else singles(static_cast<const __half*>(p) + row + c, C - c, v);
    }
    __device__ __forceinline__ void store(void* p, int type, long long row, int i, const float (&v)[8]) const {
        const int c = at(i, 0);
        if (VEC) store8_any(p, type, row + c, c < C ? 8 : 0, true, v);
        else if (type == TAB_FP32) put(static_cast<float*>(p) + row + c, C - c, v);
        else if (type == TAB_BF16) put(static_cast<__nv_bfloat16*>(p) + row + c, C - c, v);
        else put(static_cast<__half*>(p) + row + c, C - c, v);
    }
};

// Sums of N values over the GT threads of a row, the same in all of them.  `bank` alternates between two exchange buffers, so that one
// barrier a sum is enough: a buffer is written again only behind the barrier of the sum in between.
template <int GT, int N>
__device__ __forceinline__ void row_sums(float (&v)[N], float (*exchange)[32][N], int& bank) {
#pragma unroll
    for (int i = 0; i < N; i++)
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v[i] += __shfl_xor_sync(0xFFFFFFFFu, v[i], o);
    if (GT == 32) return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0)
#pragma unroll
        for (int i = 0; i < N; i++) exchange[bank][warp][i] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; i++) {
        float t = lane < GT / 32 ? exchange[bank][lane][i] : 0.f;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xFFFFFFFFu, t, o);
        v[i] = t;
    }
    bank ^= 1;
}

// ---- what the kernels for many rows share ---------------------------------------------------------------------------------------
// A row's copy into shared memory, counted on a barrier; address and size are multiples of 16 bytes.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t mbar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(mbar) : "memory");
}
// Two floats an instruction.
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 r;
    asm("{.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;}" : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 r;
    asm("{.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;}" : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 r;
    asm("{.reg .b64 x, y, w, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 w, {%6, %7};\n\tfma.rn.f32x2 z, x, y, w;\n\tmov.b64 {%0, %1}, z;}"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return r;
}
__device__ __forceinline__ float2 both(float a) { return make_float2(a, a); }
using Pairs = float2[4];                                                   // a thread's eight columns
__device__ __forceinline__ void to_pairs(const float (&v)[8], Pairs& p) {
#pragma unroll
    for (int i = 0; i < 4; i++) p[i] = make_float2(v[2 * i], v[2 * i + 1]);
}
__device__ __forceinline__ float sum_of(const Pairs& p) {
    const float2 s = add2(add2(p[0], p[1]), add2(p[2], p[3]));
    return s.x + s.y;
}
// Sum of a[i] * b[i].
__device__ __forceinline__ float dot_of(const Pairs& a, const Pairs& b) {
    const float2 s = fma2(a[0], b[0], mul2(a[1], b[1])), t = fma2(a[2], b[2], mul2(a[3], b[3])), u = add2(s, t);
    return u.x + u.y;
}
__device__ __forceinline__ void pairs_any(const void* p, int type, long long at, Pairs& v) {
    float f[8];
    load8_any(p, type, at, 8, true, f);
    to_pairs(f, v);
}
// Eight values of a row in shared memory.
template <int TYPE>
__device__ __forceinline__ void lds_pairs(uint32_t row, int c, Pairs& v) {
    using T = typename ElemOf<TYPE>::type;
    if constexpr (TYPE == TAB_FP32) {
        const int4 a = lds_v4(row + c * 4), b = lds_v4(row + c * 4 + 16);
        v[0] = make_float2(__int_as_float(a.x), __int_as_float(a.y)); v[1] = make_float2(__int_as_float(a.z), __int_as_float(a.w));
        v[2] = make_float2(__int_as_float(b.x), __int_as_float(b.y)); v[3] = make_float2(__int_as_float(b.z), __int_as_float(b.w));
    } else {
        const int4 a = lds_v4(row + c * 2);
        float f[8];
        widen8(make_uint4((uint32_t)a.x, (uint32_t)a.y, (uint32_t)a.z, (uint32_t)a.w), f, T());
        to_pairs(f, v);
    }
}
// Eight results to memory; `kept`: they become what was stored.
template <int TYPE>
__device__ __forceinline__ void store_pairs(void* p, long long at, Pairs& v, bool kept) {
    using T = typename ElemOf<TYPE>::type;
    if constexpr (TYPE == TAB_FP32) {
        const float f[8] = {v[0].x, v[0].y, v[1].x, v[1].y, v[2].x, v[2].y, v[3].x, v[3].y};
        if (p) store8(static_cast<float*>(p) + at, 8, true, f);
    } else {
        const uint4 u = make_uint4(pack2(v[0].x, v[0].y, T()), pack2(v[1].x, v[1].y, T()), pack2(v[2].x, v[2].y, T()), pack2(v[3].x, v[3].y, T()));
        if (p) *reinterpret_cast<uint4*>(static_cast<T*>(p) + at) = u;
        if (kept) {
            float f[8];
            widen8(u, f, T());
            to_pairs(f, v);
        }
    }
}
// Sums over the CTA, the same in all threads; `bank` alternates as in row_sums.
template <int WARPS, int N>
__device__ __forceinline__ void cta_sums(float (&v)[N], float (*exchange)[N][WARPS < 4 ? 4 : WARPS], int& bank) {
#pragma unroll
    for (int i = 0; i < N; i++)
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v[i] += __shfl_xor_sync(0xFFFFFFFFu, v[i], o);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0)
#pragma unroll
        for (int i = 0; i < N; i++) exchange[bank][i][warp] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; i++) {
        if (WARPS == 1) {
        } else if (WARPS < 4) {
            v[i] = exchange[bank][i][0] + exchange[bank][i][WARPS - 1];
        } else if (WARPS <= 8) {
            float s = 0.f;
#pragma unroll
            for (int w = 0; w < WARPS; w += 4) {
                const float4 e = *reinterpret_cast<const float4*>(&exchange[bank][i][w]);
                s += (e.x + e.y) + (e.z + e.w);
            }
            v[i] = s;
        } else {
            float s = exchange[bank][i][lane & (WARPS - 1)];
#pragma unroll
            for (int o = WARPS / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
            v[i] = s;
        }
    }
    bank ^= 1;
}

// ---- host side ----------------------------------------------------------------------------------------------------------------
static bool on8(const void* p, long long ld, int size) { return p && !(reinterpret_cast<uintptr_t>(p) & (8 * size - 1)) && ld % 8 == 0; }
static int norm_flags(const NormParams& p, int type) {
    const int b = type_bytes(type), w = type_bytes(p.ptype), g = type_bytes(p.gtype);
    return (on8(p.y, p.ldy, b) ? V_Y : 0) | (on8(p.x, p.ldx, b) ? V_X : 0) | (on8(p.r, p.ldr, b) ? V_R : 0) | (on8(p.h, p.ldh, b) ? V_H : 0) |
           (on8(p.q, p.ldq, 1) ? V_Q : 0) | (on8(p.w1, 0, w) ? V_W1 : 0) | (on8(p.b1, 0, w) ? V_B1 : 0) | (on8(p.w2, 0, w) ? V_W2 : 0) |
           (on8(p.b2, 0, w) ? V_B2 : 0) | (on8(p.gate, p.gkind == TAB_GATE_FULL ? p.ldg : 0, g) ? V_G : 0);
}
static constexpr int NORM_CTAS = 16 * 148;                                 // most CTAs of a stream kernel
static bool rows16(const void* p, long long ld, int size) { return !p || (!(reinterpret_cast<uintptr_t>(p) & 15) && ld * size % 16 == 0); }
// Whether all tensors that are there have rows that move eight elements at a time.
static bool norm_vectors(const NormParams& p, int type, int flags) {
    return p.C % 8 == 0 && (!p.y || (flags & V_Y)) && (!p.x || (flags & V_X)) && (!p.r || (flags & V_R)) && (!p.h || (flags & V_H)) && (!p.q || (flags & V_Q)) && (!p.w1 || (flags & V_W1)) &&
           (!p.b1 || (flags & V_B1)) && (!p.w2 || (flags & V_W2)) && (!p.b2 || (flags & V_B2)) && (p.gkind < TAB_GATE_CHANNEL || (flags & V_G));
}

// What a stream kernel is launched with: CTAs that are all resident, and rows in flight.
struct StreamPlan { int ctas, stages; size_t smem; };
// each: CTAs an SM holds by its registers; rows: least rows of a CTA (fewer CTAs than fit, but one an SM); row_bytes: of one row's tensors;
// fixed: bytes besides the ring.  0 stages: it does not fit.
template <auto KERNEL>
static StreamPlan stream_plan(int each, long long M, int rows, size_t row_bytes, size_t fixed) {
    StreamPlan pl = {0, 0, 0};
    int dev = 0;
    const int sms = blocks_sms();
    if (cudaGetDevice(&dev) != cudaSuccess) return pl;
    const size_t room = 226 * 1024;
    for (int n = each; n >= 1 && !pl.stages; n--) {
        const size_t share = std::min<size_t>(room, 228 * 1024 / n - 1536);    // less a kilobyte that every CTA is charged and what is static
        const long long stages = share > fixed ? (long long)((share - fixed) / row_bytes) : 0;
        if (stages >= 2) {
            pl.stages = (int)std::min<long long>(stages, 4);
            pl.ctas = (int)std::min<long long>(std::min(n * sms, NORM_CTAS), std::max<long long>(sms, M / rows));
        }
    }
    if (!pl.stages) return pl;
    pl.smem = pl.stages * row_bytes + fixed;
    static std::mutex mu;
    static bool configured[64] = {};
    std::lock_guard<std::mutex> lock(mu);
    if (dev < 0 || dev >= 64 || !configured[dev]) {
        if (cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)room) != cudaSuccess) { cudaGetLastError(); pl.stages = 0; return pl; }
        if (dev >= 0 && dev < 64) configured[dev] = true;
    }
    return pl;
}

#define TAB_NORM_SIZES(F, C, ARG) \
    if (C <= 256) return F(32, 1)(ARG, stream); \
    if (C <= 1024) return F(128, 1)(ARG, stream); \
    if (C <= 2048) return F(128, 2)(ARG, stream); \
    if (C <= 4096) return F(256, 2)(ARG, stream); \
    if (C <= 8192) return F(512, 2)(ARG, stream); \
    return F(1024, 2)(ARG, stream)

}  // namespace tab
