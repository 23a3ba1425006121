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
#include "blocks_common.cuh"

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
template <int GT, int NV, bool LAYER>
__device__ __forceinline__ float2 row_stats(const float (&v)[NV][8], int C, int g, float eps, float (*exchange)[32][1], int& bank) {
    float s[1] = {0.f}, mean = 0.f;
    if (LAYER) {
#pragma unroll
        for (int i = 0; i < NV; i++)
#pragma unroll
            for (int j = 0; j < 8; j++) s[0] += v[i][j];                   // elements behind the row's end are 0
        row_sums<GT, 1>(s, exchange, bank);
        mean = s[0] / (float)C;
        s[0] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const int n = C - (i * GT + g) * 8;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float d = LAYER ? (j < n ? v[i][j] - mean : 0.f) : v[i][j];
            s[0] += d * d;
        }
    }
    row_sums<GT, 1>(s, exchange, bank);
    return make_float2(mean, 1.f / sqrtf(s[0] / (float)C + eps));
}

template <int TYPE, int GT, int NV, bool LAYER>
__global__ void __launch_bounds__(GT < 128 ? 128 : GT) residual_norm_kernel(NormParams p, int flags) {
    using T = typename ElemOf<TYPE>::type;
    __shared__ float exchange[2][32][1];
    constexpr int G = GT < 128 ? 128 / GT : 1;
    const int g = threadIdx.x % GT;
    const long long m = (long long)blockIdx.x * G + threadIdx.x / GT;
    int bank = 0;
    pdl_wait();
    if (G > 1 && m >= p.M) return;                                         // a row is one warp's here: no barrier below
    const T *y = static_cast<const T*>(p.y) + m * p.ldy, *x = static_cast<const T*>(p.x) + m * p.ldx;
    float v[NV][8], xv[NV][8];
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const int c = (i * GT + g) * 8;
        load8(y + c, p.C - c, flags & V_Y, v[i]);
        if (p.x) load8(x + c, p.C - c, flags & V_X, xv[i]);
    }
    pdl_launch_dependents();
    float4 st = make_float4(0.f, 1.f, 0.f, 1.f);
    if (p.w1) {
        const float2 s = row_stats<GT, NV, LAYER>(v, p.C, g, p.eps, exchange, bank);
        st.x = s.x; st.y = s.y;
    }
    const float gtoken = p.gkind == TAB_GATE_TOKEN ? load_any(p.gate, p.gtype, m * p.ldg) : 1.f;
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const int c = (i * GT + g) * 8, n = p.C - c;
        float t[8];
        if (p.w1) {
            load8_any(p.w1, p.ptype, c, n, flags & V_W1, t);
#pragma unroll
            for (int j = 0; j < 8; j++) v[i][j] = (v[i][j] - st.x) * st.y * t[j];
            if (p.b1) {
                load8_any(p.b1, p.ptype, c, n, flags & V_B1, t);
#pragma unroll
                for (int j = 0; j < 8; j++) v[i][j] += t[j];
            }
        }
        if (p.gkind != TAB_GATE_NONE) {
            if (p.gkind == TAB_GATE_TOKEN) {
#pragma unroll
                for (int j = 0; j < 8; j++) v[i][j] *= gtoken;
            } else {
                load8_any(p.gate, p.gtype, (p.gkind == TAB_GATE_FULL ? m * p.ldg : 0) + c, n, flags & V_G, t);
#pragma unroll
                for (int j = 0; j < 8; j++) v[i][j] *= t[j];
            }
        }
        if (p.x) {
#pragma unroll
            for (int j = 0; j < 8; j++) v[i][j] = fmaf(p.alpha, xv[i][j], v[i][j]);
        }
        if (p.r) store8(static_cast<T*>(p.r) + m * p.ldr + c, n, flags & V_R, v[i]);
        // r is what is kept: the norm below is that of the rounded values (elements behind the row's end stay 0 for its sums)
#pragma unroll
        for (int j = 0; j < 8; j++) v[i][j] = j < n ? to_float(from_float<T>(v[i][j])) : 0.f;
    }
    if (p.w2) {
        const float2 s = row_stats<GT, NV, LAYER>(v, p.C, g, p.eps, exchange, bank);
        st.z = s.x; st.w = s.y;
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int c = (i * GT + g) * 8, n = p.C - c;
            float t[8];
            load8_any(p.w2, p.ptype, c, n, flags & V_W2, t);
#pragma unroll
            for (int j = 0; j < 8; j++) v[i][j] = (v[i][j] - st.z) * st.w * t[j];
            if (p.b2) {
                load8_any(p.b2, p.ptype, c, n, flags & V_B2, t);
#pragma unroll
                for (int j = 0; j < 8; j++) v[i][j] += t[j];
            }
            if (p.h) store8(static_cast<T*>(p.h) + m * p.ldh + c, n, flags & V_H, v[i]);
            if (p.q) {                                                     // sixteen threads hold a block
                uint32_t a = 0;
#pragma unroll
                for (int j = 0; j < 8; j++) a = max(a, j < n ? finite_bits(v[i][j]) : 0u);
                const int e = scale_exponent(half_warp_max(a), p.format);
                const float inv = exp2_int(-e);
                store_bytes8(static_cast<uint8_t*>(p.q) + m * p.ldq + c, n, flags & V_Q, p.format == TAB_E5M2 ? narrow8<TAB_E5M2>(v[i], inv) : narrow8<TAB_E4M3>(v[i], inv));
                if ((g & 15) == 0 && n > 0) p.s[(long long)(c / BLK) * p.lds + m] = (uint8_t)(e + 127);
            }
        }
    }
    if (p.stats && g == 0) *reinterpret_cast<float4*>(p.stats + 4 * m) = st;
}

// Sums over rows that a thread keeps: of w2, w1, the channel gate, and with shifts of b2, b1.
template <bool LAYER> constexpr int NORM_SUMS = LAYER ? 5 : 3;

template <int TYPE, int GT, int NV, bool LAYER>
__global__ void __launch_bounds__(GT < 128 ? 128 : GT) residual_norm_backward_kernel(NormBackwardParams b, int flags, long long rows_each) {
    using T = typename ElemOf<TYPE>::type;
    const NormParams& p = b.f;
    constexpr int G = GT < 128 ? 128 / GT : 1, NS = NORM_SUMS<LAYER>;
    __shared__ float exchange[2][32][3];
    const int g = threadIdx.x % GT;
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
            const int c = (i * GT + g) * 8, n = p.C - c;
            if (b.gr) load8(static_cast<const T*>(b.gr) + m * b.ldgr + c, n, flags & V_GR, dr[i]);
            else
#pragma unroll
                for (int j = 0; j < 8; j++) dr[i][j] = 0.f;
            if (want_u) load8(static_cast<const T*>(p.y) + m * p.ldy + c, n, flags & V_Y, yv[i]);
        }
        if (pre) {
            float t[NV][8], rh[NV][8];
#pragma unroll
            for (int i = 0; i < NV; i++) {
                const int c = (i * GT + g) * 8, n = p.C - c;
                load8(static_cast<const T*>(b.gh) + m * b.ldgh + c, n, flags & V_GH, t[i]);
                load8(static_cast<const T*>(p.r) + m * p.ldr + c, n, flags & V_R, rh[i]);
                float w[8];
                load8_any(p.w2, p.ptype, c, n, flags & V_W2, w);
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
            const int c = (i * GT + g) * 8, n = p.C - c;
            if (b.dx) {
                float d[8];
#pragma unroll
                for (int j = 0; j < 8; j++) d[j] = p.alpha * dr[i][j];
                store8(static_cast<T*>(b.dx) + m * b.lddx + c, n, flags & V_DX, d);
            }
            if (!want_u) {
#pragma unroll
                for (int j = 0; j < 8; j++) t[i][j] = dr[i][j];
                continue;
            }
            float w[8], gv[8], u[8];
#pragma unroll
            for (int j = 0; j < 8; j++) { w[j] = 1.f; gv[j] = gtoken; if (j >= n) dr[i][j] = 0.f; }
            if (post) load8_any(p.w1, p.ptype, c, n, flags & V_W1, w);
            if (p.gkind == TAB_GATE_CHANNEL || p.gkind == TAB_GATE_FULL) load8_any(p.gate, p.gtype, (p.gkind == TAB_GATE_FULL ? m * p.ldg : 0) + c, n, flags & V_G, gv);
#pragma unroll
            for (int j = 0; j < 8; j++) {
                yv[i][j] = (yv[i][j] - st.x) * st.y;                       // y itself without a norm: mean 0, deviation 1
                u[j] = yv[i][j] * w[j];
            }
            if (p.gkind != TAB_GATE_NONE && p.b1) {
                float s[8];
                load8_any(p.b1, p.ptype, c, n, flags & V_B1, s);
#pragma unroll
                for (int j = 0; j < 8; j++) u[j] += s[j];
            }
            if (p.gkind == TAB_GATE_FULL && b.dgate) {
                float d[8];
#pragma unroll
                for (int j = 0; j < 8; j++) d[j] = dr[i][j] * u[j];
                store8_any(b.dgate, p.gtype, m * p.C + c, n, flags & V_DG, d);
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
                const int c = (i * GT + g) * 8, n = p.C - c;
                if (post) {
#pragma unroll
                    for (int j = 0; j < 8; j++) t[i][j] = st.y * (t[i][j] - yv[i][j] * c1 - c2);
                }
                store8(static_cast<T*>(b.dy) + m * b.lddy + c, n, flags & V_DY, t[i]);
            }
        }
    }
    pdl_launch_dependents();
    if (b.partial == nullptr) return;
#pragma unroll
    for (int k = 0; k < NS; k++)
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int c = (i * GT + g) * 8;
            store8(b.partial + (part * NS + k) * p.C + c, p.C - c, p.C % 8 == 0, sum[k][i]);
        }
}

// The CTAs' sums of a column, in their order: eight threads take every eighth of them, then one adds the eight.
__global__ void __launch_bounds__(256) norm_sums_kernel(const float* partial, int parts, int NS, int C, int type, void* o0, void* o1, void* o2, int gtype, void* o3, void* o4) {
    __shared__ float acc[8][33];
    pdl_wait();
    const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5, c = blockIdx.x * 32 + lane, k = blockIdx.y;
    void* out = k == 0 ? o0 : k == 1 ? o1 : k == 2 ? o2 : k == 3 ? o3 : o4;
    float s = 0.f;
    if (out && c < C)
        for (int i = slice; i < parts; i += 8) s += partial[((long long)i * NS + k) * C + c];
    acc[slice][lane] = s;
    __syncthreads();
    if (slice == 0 && out && c < C) {
        for (int i = 1; i < 8; i++) s += acc[i][lane];
        store_any(out, k == 2 ? gtype : type, c, s);
    }
    pdl_launch_dependents();
}

// ---- host side ----------------------------------------------------------------------------------------------------------------
static bool on8(const void* p, long long ld, int size) { return p && !(reinterpret_cast<uintptr_t>(p) & (8 * size - 1)) && ld % 8 == 0; }
static int norm_flags(const NormParams& p, int type) {
    const int b = type_bytes(type), w = type_bytes(p.ptype), g = type_bytes(p.gtype);
    return (on8(p.y, p.ldy, b) ? V_Y : 0) | (on8(p.x, p.ldx, b) ? V_X : 0) | (on8(p.r, p.ldr, b) ? V_R : 0) | (on8(p.h, p.ldh, b) ? V_H : 0) |
           (on8(p.q, p.ldq, 1) ? V_Q : 0) | (on8(p.w1, 0, w) ? V_W1 : 0) | (on8(p.b1, 0, w) ? V_B1 : 0) | (on8(p.w2, 0, w) ? V_W2 : 0) |
           (on8(p.b2, 0, w) ? V_B2 : 0) | (on8(p.gate, p.gkind == TAB_GATE_FULL ? p.ldg : 0, g) ? V_G : 0);
}
// How many parts of the rows are summed on their own (one for each group of threads of the backward kernel).
static int norm_groups(int C) { return C <= 1024 ? 4 : 1; }
static long long norm_parts(long long M, int C) {
    const int G = norm_groups(C), ctas = 148 * (C <= 2048 ? 4 : C <= 4096 ? 2 : 1);
    const long long wanted = std::min<long long>((long long)ctas * G, M);
    return (wanted + G - 1) / G * G;
}
size_t residual_norm_partial_bytes(long long M, int C) { return (size_t)norm_parts(M, C) * 5 * (size_t)C * sizeof(float); }

template <int TYPE, int GT, int NV>
static int launch_norm(const NormParams& p, cudaStream_t stream) {
    constexpr int G = GT < 128 ? 128 / GT : 1;
    const long long grid = (p.M + G - 1) / G;
    if (grid >= (1LL << 31)) return TAB_E_TOO_LARGE;
    const int flags = norm_flags(p, TYPE);
    if (p.layer) return launch_pdl(residual_norm_kernel<TYPE, GT, NV, true>, dim3((unsigned)grid), dim3(GT < 128 ? 128 : GT), 0, stream, p, flags);
    return launch_pdl(residual_norm_kernel<TYPE, GT, NV, false>, dim3((unsigned)grid), dim3(GT < 128 ? 128 : GT), 0, stream, p, flags);
}
template <int TYPE, int GT, int NV>
static int launch_norm_backward(NormBackwardParams b, cudaStream_t stream) {
    constexpr int G = GT < 128 ? 128 / GT : 1;
    const NormParams& p = b.f;
    const int s = type_bytes(TYPE);
    const int flags = norm_flags(p, TYPE) | (on8(b.gr, b.ldgr, s) ? V_GR : 0) | (on8(b.gh, b.ldgh, s) ? V_GH : 0) | (on8(b.dy, b.lddy, s) ? V_DY : 0) |
                      (on8(b.dx, b.lddx, s) ? V_DX : 0) | (on8(b.dgate, p.C, type_bytes(p.gtype)) ? V_DG : 0);
    const long long parts = norm_parts(p.M, p.C), rows_each = (p.M + parts - 1) / parts;
    void* dgate = p.gkind == TAB_GATE_CHANNEL ? b.dgate : nullptr;
    const bool sums = b.dw1 || b.db1 || b.dw2 || b.db2 || dgate;
    if (!sums) b.partial = nullptr;
    const dim3 grid((unsigned)(parts / G)), block(GT < 128 ? 128 : GT);
    const int rc = p.layer ? launch_pdl(residual_norm_backward_kernel<TYPE, GT, NV, true>, grid, block, 0, stream, b, flags, rows_each)
                           : launch_pdl(residual_norm_backward_kernel<TYPE, GT, NV, false>, grid, block, 0, stream, b, flags, rows_each);
    if (rc != TAB_OK || !sums) return rc;
    const int NS = p.layer ? NORM_SUMS<true> : NORM_SUMS<false>;
    return launch_pdl(norm_sums_kernel, dim3((unsigned)((p.C + 31) / 32), (unsigned)NS), dim3(256), 0, stream, (const float*)b.partial, (int)parts, NS, p.C, p.ptype, b.dw2, b.dw1, dgate, p.gtype,
                      p.layer ? b.db2 : nullptr, p.layer ? b.db1 : nullptr);
}

#define TAB_NORM_SIZES(F, C, ARG) \
    if (C <= 256) return F(32, 1)(ARG, stream); \
    if (C <= 1024) return F(32, 4)(ARG, stream); \
    if (C <= 2048) return F(128, 2)(ARG, stream); \
    if (C <= 4096) return F(256, 2)(ARG, stream); \
    if (C <= 8192) return F(512, 2)(ARG, stream); \
    return F(1024, 2)(ARG, stream)

template <int TYPE>
static int norm_sizes(const NormParams& p, cudaStream_t stream) {
#define TAB_NORM_F(GT, NV) launch_norm<TYPE, GT, NV>
    TAB_NORM_SIZES(TAB_NORM_F, p.C, p);
#undef TAB_NORM_F
}
template <int TYPE>
static int norm_backward_sizes(const NormBackwardParams& b, cudaStream_t stream) {
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
