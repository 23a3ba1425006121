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

// Mean (0 where not centred) and 1 / deviation of the row in v.
template <int GT, int NV, bool VEC, bool LAYER>
__device__ __forceinline__ float2 row_stats(const float (&v)[NV][8], const Columns<GT, NV, VEC>& col, float eps, float (*exchange)[32][1], int& bank) {
    float s[1] = {0.f}, mean = 0.f;
    if (LAYER) {
#pragma unroll
        for (int i = 0; i < NV; i++)
#pragma unroll
            for (int j = 0; j < 8; j++) s[0] += v[i][j];                   // elements behind the row's end are 0
        row_sums<GT, 1>(s, exchange, bank);
        mean = s[0] / (float)col.C;
        s[0] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < NV; i++)
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float d = LAYER ? (col.in(i, j) ? v[i][j] - mean : 0.f) : v[i][j];
            s[0] += d * d;
        }
    row_sums<GT, 1>(s, exchange, bank);
    return make_float2(mean, 1.f / sqrtf(s[0] / (float)col.C + eps));
}

// A row by GT threads, at once.
template <int TYPE, int GT, int NV, bool VEC, bool LAYER>
__global__ void __launch_bounds__(GT < 128 ? 128 : GT) residual_norm_kernel(NormParams p) {
    using T = typename ElemOf<TYPE>::type;
    __shared__ float exchange[2][32][1];
    constexpr int G = GT < 128 ? 128 / GT : 1;
    const Columns<GT, NV, VEC> col = {(int)threadIdx.x % GT, p.C};
    const int g = col.g;
    const long long m = (long long)blockIdx.x * G + threadIdx.x / GT;
    int bank = 0;
    pdl_wait();
    if (G > 1 && m >= p.M) return;                                         // a row is one warp's here: no barrier below
    float v[NV][8], xv[NV][8];
#pragma unroll
    for (int i = 0; i < NV; i++) {
        col.load(p.y, TYPE, m * p.ldy, i, v[i]);
        if (p.x) col.load(p.x, TYPE, m * p.ldx, i, xv[i]);
    }
    pdl_launch_dependents();
    float4 st = make_float4(0.f, 1.f, 0.f, 1.f);
    if (p.w1) {
        const float2 s = row_stats<GT, NV, VEC, LAYER>(v, col, p.eps, exchange, bank);
        st.x = s.x; st.y = s.y;
    }
    const float gtoken = p.gkind == TAB_GATE_TOKEN ? load_any(p.gate, p.gtype, m * p.ldg) : 1.f;
#pragma unroll
    for (int i = 0; i < NV; i++) {
        float t[8];
        if (p.w1) {
            col.load(p.w1, p.ptype, 0, i, t);
#pragma unroll
            for (int j = 0; j < 8; j++) v[i][j] = (v[i][j] - st.x) * st.y * t[j];
            if (p.b1) {
                col.load(p.b1, p.ptype, 0, i, t);
#pragma unroll
                for (int j = 0; j < 8; j++) v[i][j] += t[j];
            }
        }
        if (p.gkind == TAB_GATE_CHANNEL || p.gkind == TAB_GATE_FULL) {
            col.load(p.gate, p.gtype, p.gkind == TAB_GATE_FULL ? m * p.ldg : 0, i, t);
#pragma unroll
            for (int j = 0; j < 8; j++) v[i][j] *= t[j];
        } else if (p.gkind == TAB_GATE_TOKEN) {
#pragma unroll
            for (int j = 0; j < 8; j++) v[i][j] *= gtoken;
        }
        if (p.x) {
#pragma unroll
            for (int j = 0; j < 8; j++) v[i][j] = fmaf(p.alpha, xv[i][j], v[i][j]);
        }
        if (p.r) col.store(p.r, TYPE, m * p.ldr, i, v[i]);
        // r is what is kept: the norm below is that of the rounded values (elements behind the row's end stay 0 for its sums)
#pragma unroll
        for (int j = 0; j < 8; j++) v[i][j] = col.in(i, j) ? to_float(from_float<T>(v[i][j])) : 0.f;
    }
    if (p.w2) {
        const float2 s = row_stats<GT, NV, VEC, LAYER>(v, col, p.eps, exchange, bank);
        st.z = s.x; st.w = s.y;
#pragma unroll
        for (int i = 0; i < NV; i++) {
            float t[8];
            col.load(p.w2, p.ptype, 0, i, t);
#pragma unroll
            for (int j = 0; j < 8; j++) v[i][j] = (v[i][j] - st.z) * st.w * t[j];
            if (p.b2) {
                col.load(p.b2, p.ptype, 0, i, t);
#pragma unroll
                for (int j = 0; j < 8; j++) v[i][j] += t[j];
            }
            if (p.h) col.store(p.h, TYPE, m * p.ldh, i, v[i]);
            if (!p.q) continue;
            uint8_t* q = static_cast<uint8_t*>(p.q) + m * p.ldq;
            uint32_t a[2] = {0, 0};                                        // VEC: sixteen threads hold a block; else a warp holds two, four columns a lane of each
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const uint32_t b = col.in(i, j) ? finite_bits(v[i][j]) : 0u;
                a[VEC ? 0 : j >> 2] = max(a[VEC ? 0 : j >> 2], b);
            }
            if (VEC) {
                const int e = scale_exponent(half_warp_max(a[0]), p.format), c = col.at(i, 0);
                const float inv = exp2_int(-e);
                if (c < p.C) {
                    *reinterpret_cast<uint2*>(q + c) = p.format == TAB_E5M2 ? narrow8<TAB_E5M2>(v[i], inv) : narrow8<TAB_E4M3>(v[i], inv);
                    if ((g & 15) == 0) p.s[(long long)(c / BLK) * p.lds + m] = (uint8_t)(e + 127);
                }
            } else {
                float sc[8];
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const uint32_t top = half_warp_max(max(a[h], __shfl_xor_sync(0xFFFFFFFFu, a[h], 16)));
                    const int e = scale_exponent(top, p.format), c = col.at(i, 4 * h);
#pragma unroll
                    for (int j = 0; j < 4; j++) sc[4 * h + j] = exp2_int(-e);
                    if ((g & 31) == 0 && c < p.C) p.s[(long long)(c / BLK) * p.lds + m] = (uint8_t)(e + 127);
                }
                float y[8];
#pragma unroll
                for (int j = 0; j < 8; j++) y[j] = v[i][j] * sc[j];
                const uint2 o = p.format == TAB_E5M2 ? narrow8<TAB_E5M2>(y, 1.f) : narrow8<TAB_E4M3>(y, 1.f);
#pragma unroll
                for (int j = 0; j < 8; j++) if (col.in(i, j)) q[col.at(i, j)] = (uint8_t)((j < 4 ? o.x : o.y) >> (8 * (j & 3)));
            }
        }
    }
    if (p.stats && g == 0) *reinterpret_cast<float4*>(p.stats + 4 * m) = st;
}

// Sums over rows that a thread keeps: of w2, w1, the channel gate, and with shifts of b2, b1.
template <bool LAYER> constexpr int NORM_SUMS = LAYER ? 5 : 3;

// rows_each rows by GT threads, one after the other.
template <int TYPE, int GT, int NV, bool VEC, bool LAYER>
__global__ void __launch_bounds__(GT < 128 ? 128 : GT) residual_norm_backward_kernel(NormBackwardParams b, long long rows_each) {
    const NormParams& p = b.f;
    constexpr int G = GT < 128 ? 128 / GT : 1, NS = NORM_SUMS<LAYER>;
    __shared__ float exchange[2][32][3];
    const Columns<GT, NV, VEC> col = {(int)threadIdx.x % GT, p.C};
    const int g = col.g;
    const long long part = (long long)blockIdx.x * G + threadIdx.x / GT, m0 = part * rows_each, m1 = min(p.M, m0 + rows_each);
    int bank = 0;
    float sum[NS][NV][8];
#pragma unroll
    for (int k = 0; k < NS; k++)
#pragma unroll
        for (int i = 0; i < NV; i++)
#pragma unroll
            for (int j = 0; j < 8; j++) sum[k][i][j] = 0.f;
    pdl_wait();
    const float inv_c = 1.f / (float)p.C;
    const bool pre = p.w2 && b.gh, post = p.w1 != nullptr, want_u = post || p.gkind != TAB_GATE_NONE;
    for (long long m = m0; m < m1; m++) {
        const float4 st = p.stats ? *reinterpret_cast<const float4*>(p.stats + 4 * m) : make_float4(0.f, 1.f, 0.f, 1.f);
        float dr[NV][8], yv[NV][8];
        float red[3] = {0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < NV; i++) {
            if (b.gr) col.load(b.gr, TYPE, m * b.ldgr, i, dr[i]);
            else
#pragma unroll
                for (int j = 0; j < 8; j++) dr[i][j] = 0.f;
            if (want_u) col.load(p.y, TYPE, m * p.ldy, i, yv[i]);
        }
        if (pre) {
            float t[NV][8], rh[NV][8];
#pragma unroll
            for (int i = 0; i < NV; i++) {
                col.load(b.gh, TYPE, m * b.ldgh, i, t[i]);
                col.load(p.r, TYPE, m * p.ldr, i, rh[i]);
                float w[8];
                col.load(p.w2, p.ptype, 0, i, w);
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    rh[i][j] = (rh[i][j] - st.z) * st.w;
                    sum[0][i][j] += t[i][j] * rh[i][j];
                    if (LAYER) sum[NS - 2][i][j] += t[i][j];
                    t[i][j] *= w[j];
                    red[0] += t[i][j] * rh[i][j];
                    if (LAYER) red[1] += t[i][j];
                }
            }
            row_sums<GT, 3>(red, exchange, bank);
            const float c1 = red[0] * inv_c, c2 = LAYER ? red[1] * inv_c : 0.f;
#pragma unroll
            for (int i = 0; i < NV; i++)
#pragma unroll
                for (int j = 0; j < 8; j++) dr[i][j] += st.w * (t[i][j] - rh[i][j] * c1 - c2);
        }
        const float gtoken = p.gkind == TAB_GATE_TOKEN ? load_any(p.gate, p.gtype, m * p.ldg) : 1.f;
        red[0] = red[1] = red[2] = 0.f;
        float t[NV][8];
#pragma unroll
        for (int i = 0; i < NV; i++) {
            if (b.dx) {
                float d[8];
#pragma unroll
                for (int j = 0; j < 8; j++) d[j] = p.alpha * dr[i][j];
                col.store(b.dx, TYPE, m * b.lddx, i, d);
            }
            if (!want_u) {
#pragma unroll
                for (int j = 0; j < 8; j++) t[i][j] = dr[i][j];
                continue;
            }
            float w[8], gv[8], u[8];
#pragma unroll
            for (int j = 0; j < 8; j++) { w[j] = 1.f; gv[j] = gtoken; if (!col.in(i, j)) dr[i][j] = 0.f; }
            if (post) col.load(p.w1, p.ptype, 0, i, w);
            if (p.gkind == TAB_GATE_CHANNEL || p.gkind == TAB_GATE_FULL) col.load(p.gate, p.gtype, p.gkind == TAB_GATE_FULL ? m * p.ldg : 0, i, gv);
#pragma unroll
            for (int j = 0; j < 8; j++) {
                yv[i][j] = (yv[i][j] - st.x) * st.y;                       // y itself without a norm: mean 0, deviation 1
                u[j] = yv[i][j] * w[j];
            }
            if (p.gkind != TAB_GATE_NONE && p.b1) {
                float s[8];
                col.load(p.b1, p.ptype, 0, i, s);
#pragma unroll
                for (int j = 0; j < 8; j++) u[j] += s[j];
            }
            if (p.gkind == TAB_GATE_FULL && b.dgate) {
                float d[8];
#pragma unroll
                for (int j = 0; j < 8; j++) d[j] = dr[i][j] * u[j];
                col.store(b.dgate, p.gtype, m * p.C, i, d);
            }
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float dg = dr[i][j] * u[j], du = dr[i][j] * gv[j];
                if (p.gkind == TAB_GATE_CHANNEL) sum[2][i][j] += dg;
                red[2] += dg;
                t[i][j] = du * w[j];
                if (post) {
                    sum[1][i][j] += du * yv[i][j];
                    if (LAYER) sum[NS - 1][i][j] += du;
                    red[0] += t[i][j] * yv[i][j];
                    if (LAYER) red[1] += t[i][j];
                }
            }
        }
        float c1 = 0.f, c2 = 0.f;
        if (post || p.gkind == TAB_GATE_TOKEN) {
            row_sums<GT, 3>(red, exchange, bank);
            if (post) { c1 = red[0] * inv_c; c2 = LAYER ? red[1] * inv_c : 0.f; }
            if (p.gkind == TAB_GATE_TOKEN && b.dgate && g == 0) store_any(b.dgate, p.gtype, m, red[2]);
        }
        if (b.dy) {
#pragma unroll
            for (int i = 0; i < NV; i++) {
                if (post) {
#pragma unroll
                    for (int j = 0; j < 8; j++) t[i][j] = st.y * (t[i][j] - yv[i][j] * c1 - c2);
                }
                col.store(b.dy, TYPE, m * b.lddy, i, t[i]);
            }
        }
    }
    pdl_launch_dependents();
    if (b.partial == nullptr) return;
#pragma unroll
    for (int k = 0; k < NS; k++)
#pragma unroll
        for (int i = 0; i < NV; i++) col.store(b.partial, TAB_FP32, (part * NS + k) * p.C, i, sum[k][i]);
}

// ---- many rows ------------------------------------------------------------------------------------------------------------------
// The same with CTAs that stay: rows come by bulk copies into a ring in shared memory, a few rows ahead, so that the memory is asked for the
// next rows while the threads meet over this one; a thread keeps its eight columns' weights (forward) or their sums (backward) in
// registers from row to row, so that weights are read once a CTA and not once a row.  Rows and their pitches are multiples of 16 bytes
// and eight elements here; the kernels above take everything else.
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

// A thread has NV times eight columns, THREADS * 8 apart; what a row costs whatever its length (waits, meetings, addresses) is most of a
// row's instructions at one.  FAST: both norms, a residual and no gate or one of channels, known when the kernel is compiled.
constexpr int forward_threads(bool layer, bool fast) { return fast && !layer ? 640 : 512; }              // an SM holds, by registers
template <int TYPE, int THREADS, int NV, bool LAYER, bool QUANT, bool FAST>
__global__ void __launch_bounds__(THREADS, forward_threads(LAYER, FAST) / THREADS) residual_norm_stream_kernel(NormParams p, int stages, int* status) {
    using T = typename ElemOf<TYPE>::type;
    extern __shared__ __align__(128) uint8_t ring[];
    __shared__ __align__(8) uint64_t bars[8];
    constexpr int WARPS = THREADS / 32;
    __shared__ __align__(16) float exchange[2][1][WARPS < 4 ? 4 : WARPS];
    const int g = threadIdx.x;
    const uint32_t row_bytes = (uint32_t)p.C * sizeof(T), sRing = (uint32_t)__cvta_generic_to_shared(ring), full = (uint32_t)__cvta_generic_to_shared(bars);
    const float inv_c = 1.f / (float)p.C;
    const bool post = FAST || p.w1, has_x = FAST || p.x, pre = FAST || p.w2;
    const int gkind = FAST ? (int)TAB_GATE_CHANNEL : p.gkind;
    int bank = 0;
    bool dead = false;
    if (g == 0) {
        for (int s = 0; s < stages; s++) mbar_init(full + 8 * s, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    pdl_wait();
    auto request = [&](long long m, int s) {
        const uint32_t at = sRing + (uint32_t)s * 2 * row_bytes;
        mbar_expect_tx(full + 8 * s, has_x ? 2 * row_bytes : row_bytes);
        bulk_load(at, static_cast<const T*>(p.y) + m * p.ldy, row_bytes, full + 8 * s);
        if (has_x) bulk_load(at + row_bytes, static_cast<const T*>(p.x) + m * p.ldx, row_bytes, full + 8 * s);
    };
    const long long step = gridDim.x;
    if (g == 0)
        for (int s = 0; s < stages; s++)
            if (blockIdx.x + s * step < p.M) request(blockIdx.x + s * step, s);
    bool mine[NV];
    Pairs w1[NV], w2[NV], gate[NV];
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const int c = (i * THREADS + g) * 8;
        mine[i] = c < p.C;
#pragma unroll
        for (int j = 0; j < 4; j++) { w1[i][j] = w2[i][j] = both(0.f); gate[i][j] = both(1.f); }
        if (!mine[i]) continue;
        if (p.w1) pairs_any(p.w1, p.ptype, c, w1[i]);
        if (p.w2) pairs_any(p.w2, p.ptype, c, w2[i]);
        if (p.gkind == TAB_GATE_CHANNEL) pairs_any(p.gate, p.gtype, c, gate[i]);
        if (!LAYER && post && gkind == TAB_GATE_CHANNEL)                   // no shift between the two: one factor
#pragma unroll
            for (int j = 0; j < 4; j++) w1[i][j] = mul2(w1[i][j], gate[i][j]);
    }
    const bool gate_now = gkind == TAB_GATE_CHANNEL && (LAYER || !post);
    int slot = 0, turn = 0;
    for (long long m = blockIdx.x; m < p.M; m += step) {
        if (!dead && !mbar_wait(full + 8 * slot, turn & 1)) { dead = true; if (status) atomicExch(status, 42); }
        const uint32_t at = sRing + (uint32_t)slot * 2 * row_bytes;
        Pairs v[NV], x[NV];
#pragma unroll
        for (int i = 0; i < NV; i++) {
#pragma unroll
            for (int j = 0; j < 4; j++) v[i][j] = x[i][j] = both(0.f);
            if (!mine[i]) continue;
            lds_pairs<TYPE>(at, (i * THREADS + g) * 8, v[i]);
            if (has_x) lds_pairs<TYPE>(at + row_bytes, (i * THREADS + g) * 8, x[i]);
        }
        // The first barrier of a row also says that everybody has read it, and its place is filled again.
        bool open = true;
        auto refill = [&]() {
            if (open && g == 0 && m + stages * step < p.M) request(m + stages * step, slot);
            open = false;
        };
        auto normalise = [&](float& mean, float& inverse) {
            float s[1];
            mean = 0.f;
            if (LAYER) {
                s[0] = sum_of(v[0]);
#pragma unroll
                for (int i = 1; i < NV; i++) s[0] += sum_of(v[i]);
                cta_sums<WARPS, 1>(s, exchange, bank);
                refill();
                mean = s[0] * inv_c;
#pragma unroll
                for (int i = 0; i < NV; i++)
                    if (mine[i])
#pragma unroll
                        for (int j = 0; j < 4; j++) v[i][j] = add2(v[i][j], both(-mean));
            }
            s[0] = dot_of(v[0], v[0]);
#pragma unroll
            for (int i = 1; i < NV; i++) s[0] += dot_of(v[i], v[i]);
            cta_sums<WARPS, 1>(s, exchange, bank);
            refill();
            inverse = 1.f / sqrtf(s[0] * inv_c + p.eps);
        };
        auto shift = [&](const void* b) {
#pragma unroll
            for (int i = 0; i < NV; i++) {
                Pairs f;
                if (!mine[i]) continue;
                pairs_any(b, p.ptype, (i * THREADS + g) * 8, f);
#pragma unroll
                for (int j = 0; j < 4; j++) v[i][j] = add2(v[i][j], f[j]);
            }
        };
        float4 st = make_float4(0.f, 1.f, 0.f, 1.f);
        if (post) {
            normalise(st.x, st.y);
#pragma unroll
            for (int i = 0; i < NV; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) v[i][j] = mul2(mul2(v[i][j], both(st.y)), w1[i][j]);
            if (LAYER && p.b1) shift(p.b1);
        }
        if (gate_now) {
#pragma unroll
            for (int i = 0; i < NV; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) v[i][j] = mul2(v[i][j], gate[i][j]);
        } else if (gkind == TAB_GATE_FULL) {
#pragma unroll
            for (int i = 0; i < NV; i++) {
                Pairs f;
                if (!mine[i]) continue;
                pairs_any(p.gate, p.gtype, m * p.ldg + (i * THREADS + g) * 8, f);
#pragma unroll
                for (int j = 0; j < 4; j++) v[i][j] = mul2(v[i][j], f[j]);
            }
        } else if (gkind == TAB_GATE_TOKEN) {
            const float one = load_any(p.gate, p.gtype, m * p.ldg);
#pragma unroll
            for (int i = 0; i < NV; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) v[i][j] = mul2(v[i][j], both(one));
        }
#pragma unroll
        for (int i = 0; i < NV; i++) {
            if (has_x) {
#pragma unroll
                for (int j = 0; j < 4; j++) v[i][j] = fma2(both(p.alpha), x[i][j], v[i][j]);
            }
            store_pairs<TYPE>(mine[i] ? p.r : nullptr, m * p.ldr + (i * THREADS + g) * 8, v[i], true);     // v: r as it is kept
        }
        if (pre) {
            normalise(st.z, st.w);
#pragma unroll
            for (int i = 0; i < NV; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) v[i][j] = mul2(mul2(v[i][j], both(st.w)), w2[i][j]);
            if (LAYER && p.b2) shift(p.b2);
            if (!QUANT) {
#pragma unroll
                for (int i = 0; i < NV; i++)
                    if (mine[i]) store_pairs<TYPE>(p.h, m * p.ldh + (i * THREADS + g) * 8, v[i], false);
            } else {
                // The larger magnitudes, which fmaxf takes past NaN; rows with an infinity are looked at again.
                float a[NV], most = 0.f;
#pragma unroll
                for (int i = 0; i < NV; i++) {
                    a[i] = fmaxf(fmaxf(fmaxf(fabsf(v[i][0].x), fabsf(v[i][0].y)), fmaxf(fabsf(v[i][1].x), fabsf(v[i][1].y))),
                                 fmaxf(fmaxf(fabsf(v[i][2].x), fabsf(v[i][2].y)), fmaxf(fabsf(v[i][3].x), fabsf(v[i][3].y))));
                    most = fmaxf(most, a[i]);
                }
                const bool odd = __any_sync(0xFFFFFFFFu, isinf(most));
#pragma unroll
                for (int i = 0; i < NV; i++) {
                    const int c = (i * THREADS + g) * 8;
                    const float f[8] = {v[i][0].x, v[i][0].y, v[i][1].x, v[i][1].y, v[i][2].x, v[i][2].y, v[i][3].x, v[i][3].y};
                    uint32_t bits = __float_as_uint(a[i]);
                    if (odd) {
                        bits = 0;
#pragma unroll
                        for (int j = 0; j < 8; j++) bits = max(bits, finite_bits(f[j]));
                    }
                    bits = half_warp_max(bits);
                    uint2 o;
                    uint32_t s;
                    auto round = [&](auto format) {
                        constexpr int F = decltype(format)::value;
                        s = scale_byte<F>(bits);
                        const float inv = __uint_as_float(inverse_bits(s));
                        if (odd) {
                            o = narrow8<F>(f, inv);
                            return;
                        }
                        Pairs y;
#pragma unroll
                        for (int j = 0; j < 4; j++) y[j] = mul2(v[i][j], both(inv));
                        o.x = __byte_perm(narrow2<F>(y[0].x, y[0].y), narrow2<F>(y[1].x, y[1].y), 0x5410);
                        o.y = __byte_perm(narrow2<F>(y[2].x, y[2].y), narrow2<F>(y[3].x, y[3].y), 0x5410);
                    };
                    if (p.format == TAB_E5M2) round(std::integral_constant<int, TAB_E5M2>());
                    else round(std::integral_constant<int, TAB_E4M3>());
                    if (mine[i]) {
                        *reinterpret_cast<uint2*>(static_cast<uint8_t*>(p.q) + m * p.ldq + c) = o;
                        if ((g & 15) == 0) p.s[(long long)(c / BLK) * p.lds + m] = (uint8_t)s;
                    }
                }
            }
        }
        if (open) { __syncthreads(); refill(); }
        if (p.stats && g == 0) *reinterpret_cast<float4*>(p.stats + 4 * m) = st;
        if (++slot == stages) { slot = 0; turn++; }
    }
    pdl_launch_dependents();
    if (dead) for (int i = 0; i < 200; i++) __nanosleep(1000);             // copies that may still be under way land before this memory is another's
}

// What a row's sums are needed for is read from the ring again behind the meeting instead of being kept: registers are what the sums
// over rows leave.  FAST: both norms and all gradients, and no gate or one of channels.
constexpr int backward_threads(int nv, bool layer) { return nv == 1 && !layer ? 1024 : 512; }    // an SM holds, by registers
template <int TYPE, int THREADS, int NV, bool LAYER, bool TOKEN, bool FAST>
__global__ void __launch_bounds__(THREADS, backward_threads(NV, LAYER) / THREADS) residual_norm_backward_stream_kernel(NormBackwardParams b, int stages, int* status) {
    using T = typename ElemOf<TYPE>::type;
    const NormParams& p = b.f;
    constexpr int NS = NORM_SUMS<LAYER>, N1 = LAYER ? 2 : 1, N2 = N1 + (TOKEN ? 1 : 0), WARPS = THREADS / 32;
    extern __shared__ __align__(128) uint8_t ring[];
    __shared__ __align__(8) uint64_t bars[8];
    __shared__ __align__(16) float exchange1[2][N1][WARPS < 4 ? 4 : WARPS];
    __shared__ __align__(16) float exchange2[2][N2][WARPS < 4 ? 4 : WARPS];
    const int g = threadIdx.x;
    const uint32_t row_bytes = (uint32_t)p.C * sizeof(T), sRing = (uint32_t)__cvta_generic_to_shared(ring), full = (uint32_t)__cvta_generic_to_shared(bars);
    const uint32_t plane = (uint32_t)p.C * 2u, sPar = sRing + (uint32_t)stages * 4 * row_bytes;   // fp32: w2, w1, gate, each a plane of the first four of eight and one of the others
    const float inv_c = 1.f / (float)p.C;
    const bool pre = FAST || (p.w2 && b.gh), post = FAST || p.w1, has_gr = FAST || b.gr, channel = p.gkind == TAB_GATE_CHANNEL;
    const bool want_u = post || p.gkind != TAB_GATE_NONE;
    int bank1 = 0, bank2 = 0;
    bool dead = false;
    if (g == 0) {
        for (int s = 0; s < stages; s++) mbar_init(full + 8 * s, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    pdl_wait();
    auto request = [&](long long m, int s) {
        const uint32_t at = sRing + (uint32_t)s * 4 * row_bytes;
        mbar_expect_tx(full + 8 * s, row_bytes * ((pre ? 2u : 0u) + (has_gr ? 1u : 0u) + (want_u ? 1u : 0u)));
        if (pre) {
            bulk_load(at, static_cast<const T*>(b.gh) + m * b.ldgh, row_bytes, full + 8 * s);
            bulk_load(at + row_bytes, static_cast<const T*>(p.r) + m * p.ldr, row_bytes, full + 8 * s);
        }
        if (has_gr) bulk_load(at + 2 * row_bytes, static_cast<const T*>(b.gr) + m * b.ldgr, row_bytes, full + 8 * s);
        if (want_u) bulk_load(at + 3 * row_bytes, static_cast<const T*>(p.y) + m * p.ldy, row_bytes, full + 8 * s);
    };
    const long long step = gridDim.x;
    if (g == 0)
        for (int s = 0; s < stages; s++)
            if (blockIdx.x + s * step < p.M) request(blockIdx.x + s * step, s);
    bool mine[NV];
#pragma unroll
    for (int i = 0; i < NV; i++) {                                         // a thread reads back what it wrote itself
        const int c = (i * THREADS + g) * 8;
        mine[i] = c < p.C;
        if (!mine[i]) continue;
        Pairs w;
        auto keep = [&](int k) {
            const uint32_t to = sPar + (uint32_t)k * 2 * plane + (uint32_t)c * 2u;
            sts_v4(to, __float_as_uint(w[0].x), __float_as_uint(w[0].y), __float_as_uint(w[1].x), __float_as_uint(w[1].y));
            sts_v4(to + plane, __float_as_uint(w[2].x), __float_as_uint(w[2].y), __float_as_uint(w[3].x), __float_as_uint(w[3].y));
        };
        if (pre) { pairs_any(p.w2, p.ptype, c, w); keep(0); }
        if (post) { pairs_any(p.w1, p.ptype, c, w); keep(1); }
        if (channel) { pairs_any(p.gate, p.gtype, c, w); keep(2); }
    }
    auto param = [&](int k, int c, Pairs& w) {
        const int4 u = lds_v4(sPar + (uint32_t)k * 2 * plane + (uint32_t)c * 2u), v = lds_v4(sPar + (uint32_t)k * 2 * plane + plane + (uint32_t)c * 2u);
        w[0] = make_float2(__int_as_float(u.x), __int_as_float(u.y)); w[1] = make_float2(__int_as_float(u.z), __int_as_float(u.w));
        w[2] = make_float2(__int_as_float(v.x), __int_as_float(v.y)); w[3] = make_float2(__int_as_float(v.z), __int_as_float(v.w));
    };
    float2 sum[NS][NV][4];
#pragma unroll
    for (int k = 0; k < NS; k++)
#pragma unroll
        for (int i = 0; i < NV; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) sum[k][i][j] = both(0.f);
    float4 next = make_float4(0.f, 1.f, 0.f, 1.f);
    if (p.stats && blockIdx.x < p.M) next = *reinterpret_cast<const float4*>(p.stats + 4 * (long long)blockIdx.x);
    int slot = 0, turn = 0;
    for (long long m = blockIdx.x; m < p.M; m += step) {
        const float4 st = next;
        if (p.stats && m + step < p.M) next = *reinterpret_cast<const float4*>(p.stats + 4 * (m + step));
        if (!dead && !mbar_wait(full + 8 * slot, turn & 1)) { dead = true; if (status) atomicExch(status, 43); }
        const uint32_t at = sRing + (uint32_t)slot * 4 * row_bytes;
        // r^ and gh w2 of eight columns
        auto upper = [&](int c, Pairs& rh, Pairs& t, Pairs& gh) {
            Pairs w;
            lds_pairs<TYPE>(at, c, gh);
            lds_pairs<TYPE>(at + row_bytes, c, rh);
            param(0, c, w);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                rh[j] = LAYER ? mul2(add2(rh[j], both(-st.z)), both(st.w)) : mul2(rh[j], both(st.w));
                t[j] = mul2(gh[j], w[j]);
            }
        };
        Pairs dr[NV];
        float c1 = 0.f, c2 = 0.f;
        if (pre) {
            float red[N1];
#pragma unroll
            for (int n = 0; n < N1; n++) red[n] = 0.f;
#pragma unroll
            for (int i = 0; i < NV; i++) {
                if (!mine[i]) continue;
                Pairs rh, t, gh;
                upper((i * THREADS + g) * 8, rh, t, gh);
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    sum[0][i][j] = fma2(gh[j], rh[j], sum[0][i][j]);
                    if (LAYER) sum[NS - 2][i][j] = add2(sum[NS - 2][i][j], gh[j]);
                }
                red[0] += dot_of(t, rh);
                if (LAYER) red[N1 - 1] += sum_of(t);
            }
            cta_sums<WARPS, N1>(red, exchange1, bank1);
            c1 = -red[0] * inv_c;
            c2 = LAYER ? -red[N1 - 1] * inv_c : 0.f;
        }
        // y^ of eight columns
        auto lower = [&](int c, Pairs& yv) {
            lds_pairs<TYPE>(at + 3 * row_bytes, c, yv);
            if (post)
#pragma unroll
                for (int j = 0; j < 4; j++) yv[j] = LAYER ? mul2(add2(yv[j], both(-st.x)), both(st.y)) : mul2(yv[j], both(st.y));
        };
        const float one = TOKEN ? load_any(p.gate, p.gtype, m * p.ldg) : 1.f;
        float red[N2];
#pragma unroll
        for (int n = 0; n < N2; n++) red[n] = 0.f;
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int c = (i * THREADS + g) * 8;
#pragma unroll
            for (int j = 0; j < 4; j++) dr[i][j] = both(0.f);
            if (!mine[i]) continue;
            if (has_gr) lds_pairs<TYPE>(at + 2 * row_bytes, c, dr[i]);
            if (pre) {
                Pairs rh, t, gh;
                upper(c, rh, t, gh);
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    t[j] = fma2(rh[j], both(c1), t[j]);
                    if (LAYER) t[j] = add2(t[j], both(c2));
                    dr[i][j] = fma2(t[j], both(st.w), dr[i][j]);
                }
            }
            if (FAST || b.dx) {
                Pairs d;
#pragma unroll
                for (int j = 0; j < 4; j++) d[j] = mul2(dr[i][j], both(p.alpha));
                store_pairs<TYPE>(b.dx, m * b.lddx + c, d, false);
            }
            if (!want_u) continue;
            Pairs yv, w, gv;
            lower(c, yv);
            if (post) param(1, c, w);
            else
#pragma unroll
                for (int j = 0; j < 4; j++) w[j] = both(1.f);
            if (channel) {
                param(2, c, gv);
            } else if (!FAST && p.gkind == TAB_GATE_FULL) {
                pairs_any(p.gate, p.gtype, m * p.ldg + c, gv);
            } else {
#pragma unroll
                for (int j = 0; j < 4; j++) gv[j] = both(one);
            }
            if (channel || (!FAST && p.gkind != TAB_GATE_NONE)) {
                Pairs u;
#pragma unroll
                for (int j = 0; j < 4; j++) u[j] = mul2(yv[j], w[j]);
                if (LAYER && p.b1) {
                    Pairs s;
                    pairs_any(p.b1, p.ptype, c, s);
#pragma unroll
                    for (int j = 0; j < 4; j++) u[j] = add2(u[j], s[j]);
                }
                if (channel) {
#pragma unroll
                    for (int j = 0; j < 4; j++) sum[2][i][j] = fma2(u[j], dr[i][j], sum[2][i][j]);
                } else if (TOKEN) {
                    red[N2 - 1] += dot_of(u, dr[i]);
                } else if (b.dgate) {
                    float d[8];
#pragma unroll
                    for (int j = 0; j < 4; j++) { d[2 * j] = u[j].x * dr[i][j].x; d[2 * j + 1] = u[j].y * dr[i][j].y; }
                    store8_any(b.dgate, p.gtype, m * p.C + c, 8, true, d);
                }
            }
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float2 du = mul2(dr[i][j], gv[j]);
                if (post) {
                    sum[1][i][j] = fma2(du, yv[j], sum[1][i][j]);
                    if (LAYER) sum[NS - 1][i][j] = add2(sum[NS - 1][i][j], du);
                }
                dr[i][j] = mul2(du, w[j]);                                 // from here on the gradient at y^
            }
            if (post) {
                red[0] += dot_of(dr[i], yv);
                if (LAYER) red[1 % N2] += sum_of(dr[i]);
            }
        }
        if (post || TOKEN) cta_sums<WARPS, N2>(red, exchange2, bank2);
        if (TOKEN && b.dgate && g == 0) store_any(b.dgate, p.gtype, m, red[N2 - 1]);
        if (FAST || b.dy) {
            c1 = -red[0] * inv_c;
            c2 = LAYER ? -red[1 % N2] * inv_c : 0.f;
#pragma unroll
            for (int i = 0; i < NV; i++) {
                const int c = (i * THREADS + g) * 8;
                if (!mine[i]) continue;
                if (post) {
                    Pairs yv;
                    lower(c, yv);
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        dr[i][j] = fma2(yv[j], both(c1), dr[i][j]);
                        if (LAYER) dr[i][j] = add2(dr[i][j], both(c2));
                        dr[i][j] = mul2(dr[i][j], both(st.y));
                    }
                }
                store_pairs<TYPE>(b.dy, m * b.lddy + c, dr[i], false);
            }
        }
        __syncthreads();                                                   // everybody has read the row
        if (g == 0 && m + stages * step < p.M) request(m + stages * step, slot);
        if (++slot == stages) { slot = 0; turn++; }
    }
    pdl_launch_dependents();
    if (b.partial)
#pragma unroll
        for (int i = 0; i < NV; i++)
            if (mine[i])
#pragma unroll
                for (int k = 0; k < NS; k++) {
                    const float2(&s)[4] = sum[k][i];
                    const float f[8] = {s[0].x, s[0].y, s[1].x, s[1].y, s[2].x, s[2].y, s[3].x, s[3].y};
                    store8(b.partial + ((long long)blockIdx.x * NS + k) * p.C + (i * THREADS + g) * 8, 8, true, f);
                }
    if (dead) for (int i = 0; i < 200; i++) __nanosleep(1000);
}

// The CTAs' sums of a column, in a fixed order: 32 warps take every 32nd of them, four columns a lane (one where rows of sums do not start
// on 16 bytes), and one warp adds theirs.
template <int V>
__global__ void __launch_bounds__(1024) norm_sums_kernel(const float* partial, int parts, int NS, int C, int type, void* o0, void* o1, void* o2, int gtype, void* o3, void* o4) {
    __shared__ float acc[32][32 * V + 1];
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5, c0 = blockIdx.x * 32 * V, k = blockIdx.y;
    void* out = k == 0 ? o0 : k == 1 ? o1 : k == 2 ? o2 : k == 3 ? o3 : o4;
    if (!out) return;
    float s[V];
#pragma unroll
    for (int j = 0; j < V; j++) s[j] = 0.f;
    if (c0 + lane * V < C) {                                               // (C is a multiple of V)
        const float* from = partial + (long long)k * C + c0 + lane * V;
        const long long pitch = (long long)NS * C;
#pragma unroll 8
        for (int i = slice; i < parts; i += 32) {
            if (V == 4) {
                const float4 f = *reinterpret_cast<const float4*>(from + i * pitch);
                s[0] += f.x; s[1 % V] += f.y; s[2 % V] += f.z; s[3 % V] += f.w;
            } else {
                s[0] += from[i * pitch];
            }
        }
    }
#pragma unroll
    for (int j = 0; j < V; j++) acc[slice][lane * V + j] = s[j];
    __syncthreads();
    if ((int)threadIdx.x >= 32 * V) return;
    float v = 0.f;
#pragma unroll
    for (int i = 0; i < 32; i++) v += acc[i][threadIdx.x];
    if (c0 + (int)threadIdx.x < C) store_any(out, k == 2 ? gtype : type, c0 + threadIdx.x, v);
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
// How many parts of the rows the general kernel sums on their own (one for each group of threads): some rows for each, since the sums of
// a part are as many bytes as the rows of one.
static int norm_groups(int C) { return C <= 256 ? 4 : 1; }
static long long norm_parts(long long M, int C) {
    const int G = norm_groups(C);
    const long long most = 148LL * G * (C <= 2048 ? 4 : C <= 4096 ? 2 : 1), wanted = std::min(most, std::min(M, std::max(148LL * G, M / 4)));
    return (wanted + G - 1) / G * G;
}
size_t residual_norm_partial_bytes(long long M, int C) { return (size_t)std::max(norm_parts(M, C), std::min<long long>(M, NORM_CTAS)) * 5 * (size_t)C * sizeof(float); }
static bool rows16(const void* p, long long ld, int size) { return !p || (!(reinterpret_cast<uintptr_t>(p) & 15) && ld * size % 16 == 0); }
// Whether all tensors that are there have rows that move eight elements at a time.
static bool norm_vectors(const NormParams& p, int type, int flags) {
    return p.C % 8 == 0 && (!p.y || (flags & V_Y)) && (!p.x || (flags & V_X)) && (!p.r || (flags & V_R)) && (!p.h || (flags & V_H)) && (!p.q || (flags & V_Q)) && (!p.w1 || (flags & V_W1)) &&
           (!p.b1 || (flags & V_B1)) && (!p.w2 || (flags & V_W2)) && (!p.b2 || (flags & V_B2)) && (p.gkind < TAB_GATE_CHANNEL || (flags & V_G));
}
static bool wants_sums(const NormBackwardParams& b) { return b.dw1 || b.db1 || b.dw2 || b.db2 || (b.f.gkind == TAB_GATE_CHANNEL && b.dgate); }
static int backward_flags(const NormBackwardParams& b, int type) {
    const int s = type_bytes(type);
    return norm_flags(b.f, type) | (on8(b.gr, b.ldgr, s) ? V_GR : 0) | (on8(b.gh, b.ldgh, s) ? V_GH : 0) | (on8(b.dy, b.lddy, s) ? V_DY : 0) |
           (on8(b.dx, b.lddx, s) ? V_DX : 0) | (on8(b.dgate, b.f.C, type_bytes(b.f.gtype)) ? V_DG : 0);
}
static bool backward_vectors(const NormBackwardParams& b, int type) {
    NormParams f = b.f;
    const int flags = backward_flags(b, type);
    if (!(f.w2 && b.gh)) f.w2 = f.b2 = f.r = nullptr;                      // not looked at
    if (!f.w1 && f.gkind == TAB_GATE_NONE) f.y = nullptr;
    f.x = f.h = f.q = nullptr;
    return norm_vectors(f, type, flags) && (!(f.w2 && b.gh) || (flags & V_GH)) && (!b.gr || (flags & V_GR)) && (!b.dy || (flags & V_DY)) && (!b.dx || (flags & V_DX)) &&
           (!(f.gkind == TAB_GATE_FULL && b.dgate) || (flags & V_DG));
}

template <int TYPE, int GT, int NV>
static int launch_norm(const NormParams& p, cudaStream_t stream) {
    constexpr int G = GT < 128 ? 128 / GT : 1;
    const long long grid = (p.M + G - 1) / G;
    if (grid >= (1LL << 31)) return TAB_E_TOO_LARGE;
#define TAB_NK(V, L) launch_pdl(residual_norm_kernel<TYPE, GT, NV, V, L>, dim3((unsigned)grid), dim3(GT < 128 ? 128 : GT), 0, stream, p)
    if (norm_vectors(p, TYPE, norm_flags(p, TYPE))) return p.layer ? TAB_NK(true, true) : TAB_NK(true, false);
    return p.layer ? TAB_NK(false, true) : TAB_NK(false, false);
#undef TAB_NK
}
// What a stream kernel is launched with: CTAs that are all resident, and rows in flight.
struct StreamPlan { int ctas, stages; size_t smem; };
// row_bytes: of one row's tensors; fixed: bytes besides the ring.  0 stages: it does not fit, or there are too few rows to stay for.
template <auto KERNEL>
static StreamPlan stream_plan(int each, long long M, size_t row_bytes, size_t fixed) {
    StreamPlan pl = {0, 0, 0};
    int dev = 0;
    const int sms = blocks_sms();
    if (M < 2LL * sms || cudaGetDevice(&dev) != cudaSuccess) return pl;
    const size_t room = 226 * 1024;
    for (int n = each; n >= 1 && !pl.stages; n--) {                        // each: CTAs an SM holds by its registers
        const size_t share = std::min<size_t>(room, 228 * 1024 / n - 1536);    // less a kilobyte that every CTA is charged and what is static
        const long long stages = share > fixed ? (long long)((share - fixed) / row_bytes) : 0;
        if (stages >= 2 && M >= 2LL * n * sms) { pl.stages = (int)std::min<long long>(stages, 4); pl.ctas = std::min(n * sms, NORM_CTAS); }
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
// TAB_E_TOO_LARGE: the stream kernel does not take the problem.
template <int TYPE, int THREADS, int NV, bool LAYER, bool QUANT, bool FAST>
static int launch_norm_stream_as(const NormParams& p, cudaStream_t stream) {
    constexpr auto kernel = residual_norm_stream_kernel<TYPE, THREADS, NV, LAYER, QUANT, FAST>;
    const StreamPlan pl = stream_plan<kernel>(forward_threads(LAYER, FAST) / THREADS, p.M, 2 * (size_t)p.C * type_bytes(TYPE), 0);
    if (!pl.stages) return TAB_E_TOO_LARGE;
    int* status = device_status_word();
    if (stalled(status)) return TAB_E_STALLED;
    return launch_pdl(kernel, dim3((unsigned)std::min<long long>(p.M, pl.ctas)), dim3(THREADS), pl.smem, stream, p, pl.stages, status);
}
template <int TYPE, int THREADS, int NV>
static int launch_norm_stream(const NormParams& p, cudaStream_t stream) {
    const int s = type_bytes(TYPE);
    if (!norm_vectors(p, TYPE, norm_flags(p, TYPE)) || !rows16(p.y, p.ldy, s) || !rows16(p.x, p.ldx, s) || (!p.h && !p.q && p.w2)) return TAB_E_TOO_LARGE;
    const bool fast = p.w1 && p.x && p.w2 && p.r && (p.gkind == TAB_GATE_NONE || p.gkind == TAB_GATE_CHANNEL);
    if (p.h && p.q) return TAB_E_TOO_LARGE;
#define TAB_NS(L, Q) (fast ? launch_norm_stream_as<TYPE, THREADS, NV, L, Q, true>(p, stream) : launch_norm_stream_as<TYPE, THREADS, NV, L, Q, false>(p, stream))
    return p.layer ? (p.q ? TAB_NS(true, true) : TAB_NS(true, false)) : (p.q ? TAB_NS(false, true) : TAB_NS(false, false));
#undef TAB_NS
}
static int launch_norm_sums(const NormBackwardParams& b, int parts, cudaStream_t stream) {
    const NormParams& p = b.f;
    const int NS = p.layer ? NORM_SUMS<true> : NORM_SUMS<false>;
    void *dgate = p.gkind == TAB_GATE_CHANNEL ? b.dgate : nullptr, *db2 = p.layer ? b.db2 : nullptr, *db1 = p.layer ? b.db1 : nullptr;
    if (p.C % 4 == 0)
        return launch_pdl(norm_sums_kernel<4>, dim3((unsigned)((p.C + 127) / 128), (unsigned)NS), dim3(1024), 0, stream, (const float*)b.partial, parts, NS, p.C, p.ptype, b.dw2, b.dw1, dgate,
                          p.gtype, db2, db1);
    return launch_pdl(norm_sums_kernel<1>, dim3((unsigned)((p.C + 31) / 32), (unsigned)NS), dim3(1024), 0, stream, (const float*)b.partial, parts, NS, p.C, p.ptype, b.dw2, b.dw1, dgate, p.gtype,
                      db2, db1);
}
template <int TYPE, int THREADS, int NV, bool LAYER, bool TOKEN, bool FAST>
static int launch_norm_backward_stream_as(NormBackwardParams b, cudaStream_t stream) {
    const NormParams& p = b.f;
    constexpr auto kernel = residual_norm_backward_stream_kernel<TYPE, THREADS, NV, LAYER, TOKEN, FAST>;
    const StreamPlan pl = stream_plan<kernel>(backward_threads(NV, LAYER) / THREADS, p.M, 4 * (size_t)p.C * type_bytes(TYPE), (p.gkind == TAB_GATE_CHANNEL ? 12 : 8) * (size_t)p.C);
    if (!pl.stages) return TAB_E_TOO_LARGE;
    int* status = device_status_word();
    if (stalled(status)) return TAB_E_STALLED;
    const bool sums = wants_sums(b);
    if (!sums) b.partial = nullptr;
    const int ctas = (int)std::min<long long>(p.M, pl.ctas);
    const int rc = launch_pdl(kernel, dim3((unsigned)ctas), dim3(THREADS), pl.smem, stream, b, pl.stages, status);
    return rc != TAB_OK || !sums ? rc : launch_norm_sums(b, ctas, stream);
}
template <int TYPE, int THREADS, int NV, bool LAYER>
static int launch_norm_backward_stream(const NormBackwardParams& b, cudaStream_t stream) {
    const NormParams& f = b.f;
    const bool pre = f.w2 && b.gh, want_u = f.w1 || f.gkind != TAB_GATE_NONE, token = f.gkind == TAB_GATE_TOKEN;
    if (!backward_vectors(b, TYPE) || (!pre && !b.gr && !want_u)) return TAB_E_TOO_LARGE;
    if (token) return launch_norm_backward_stream_as<TYPE, THREADS, NV, LAYER, true, false>(b, stream);
    if (pre && f.w1 && b.gr && b.dx && b.dy && f.gkind != TAB_GATE_FULL) return launch_norm_backward_stream_as<TYPE, THREADS, NV, LAYER, false, true>(b, stream);
    return launch_norm_backward_stream_as<TYPE, THREADS, NV, LAYER, false, false>(b, stream);
}
template <int TYPE, int GT, int NV>
static int launch_norm_backward(NormBackwardParams b, cudaStream_t stream) {
    constexpr int G = GT < 128 ? 128 / GT : 1;
    const NormParams& p = b.f;
    const long long parts = norm_parts(p.M, p.C), rows_each = (p.M + parts - 1) / parts;
    const bool sums = wants_sums(b);
    if (!sums) b.partial = nullptr;
    const dim3 grid((unsigned)(parts / G)), block(GT < 128 ? 128 : GT);
#define TAB_NK(V, L) launch_pdl(residual_norm_backward_kernel<TYPE, GT, NV, V, L>, grid, block, 0, stream, b, rows_each)
    const int rc = backward_vectors(b, TYPE) ? (p.layer ? TAB_NK(true, true) : TAB_NK(true, false)) : (p.layer ? TAB_NK(false, true) : TAB_NK(false, false));
#undef TAB_NK
    return rc != TAB_OK || !sums ? rc : launch_norm_sums(b, (int)parts, stream);
}

#define TAB_NORM_SIZES(F, C, ARG) \
    if (C <= 256) return F(32, 1)(ARG, stream); \
    if (C <= 1024) return F(128, 1)(ARG, stream); \
    if (C <= 2048) return F(128, 2)(ARG, stream); \
    if (C <= 4096) return F(256, 2)(ARG, stream); \
    if (C <= 8192) return F(512, 2)(ARG, stream); \
    return F(1024, 2)(ARG, stream)

template <int TYPE>
static int norm_sizes(const NormParams& p, cudaStream_t stream) {
    int rc = TAB_E_TOO_LARGE;
    if (p.C > 256 && p.C <= 512) rc = launch_norm_stream<TYPE, 64, 1>(p, stream);
    else if (p.C > 512 && p.C <= 1024) rc = launch_norm_stream<TYPE, 64, 2>(p, stream);
    else if (p.C > 1024 && p.C <= 2048) rc = launch_norm_stream<TYPE, 128, 2>(p, stream);
    else if (p.C > 2048 && p.C <= 4096) rc = launch_norm_stream<TYPE, 256, 2>(p, stream);
    else if (p.C > 4096 && p.C <= 8192) rc = launch_norm_stream<TYPE, 512, 2>(p, stream);
    if (rc != TAB_E_TOO_LARGE) return rc;
#define TAB_NORM_F(GT, NV) launch_norm<TYPE, GT, NV>
    TAB_NORM_SIZES(TAB_NORM_F, p.C, p);
#undef TAB_NORM_F
}
template <int TYPE>
static int norm_backward_sizes(const NormBackwardParams& b, cudaStream_t stream) {
    // Centred norms have five sums over rows instead of three to hold: twice the registers, half the threads.
    int rc = TAB_E_TOO_LARGE;
    const int C = b.f.C;
    if (b.f.layer) {
        if (C > 256 && C <= 512) rc = launch_norm_backward_stream<TYPE, 64, 1, true>(b, stream);
        else if (C > 512 && C <= 1024) rc = launch_norm_backward_stream<TYPE, 128, 1, true>(b, stream);
        else if (C > 1024 && C <= 2048) rc = launch_norm_backward_stream<TYPE, 256, 1, true>(b, stream);
        else if (C > 2048 && C <= 4096) rc = launch_norm_backward_stream<TYPE, 512, 1, true>(b, stream);
        else if (C > 4096 && C <= 8192) rc = launch_norm_backward_stream<TYPE, 512, 2, true>(b, stream);
    } else {
        if (C > 256 && C <= 512) rc = launch_norm_backward_stream<TYPE, 32, 2, false>(b, stream);
        else if (C > 512 && C <= 1024) rc = launch_norm_backward_stream<TYPE, 64, 2, false>(b, stream);
        else if (C > 1024 && C <= 2048) rc = launch_norm_backward_stream<TYPE, 128, 2, false>(b, stream);
        else if (C > 2048 && C <= 4096) rc = launch_norm_backward_stream<TYPE, 256, 2, false>(b, stream);
        else if (C > 4096 && C <= 8192) rc = launch_norm_backward_stream<TYPE, 512, 2, false>(b, stream);
    }
    if (rc != TAB_E_TOO_LARGE) return rc;
#define TAB_NORM_B(GT, NV) launch_norm_backward<TYPE, GT, NV>
    TAB_NORM_SIZES(TAB_NORM_B, b.f.C, b);
#undef TAB_NORM_B
}
int residual_norm_dispatch(const NormParams& p, int type, cudaStream_t stream) {
    return type == TAB_FP32 ? norm_sizes<TAB_FP32>(p, stream) : type == TAB_BF16 ? norm_sizes<TAB_BF16>(p, stream) : norm_sizes<TAB_FP16>(p, stream);
}
int residual_norm_backward_dispatch(const NormBackwardParams& p, int type, cudaStream_t stream) {
    return type == TAB_FP32 ? norm_backward_sizes<TAB_FP32>(p, stream) : type == TAB_BF16 ? norm_backward_sizes<TAB_BF16>(p, stream) : norm_backward_sizes<TAB_FP16>(p, stream);
}

}  // namespace tab
