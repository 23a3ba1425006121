// Gradients of the residual stream between two blocks (tab_residual_norm_backward_launch); the mathematics stand in
// residual_norm_common.cuh.
#include "residual_norm_common.cuh"

namespace tab {

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

// ---- many rows -------------------------------------------------------------------------------------------------------------------
// CTAs that stay and a ring of rows as in the forward pass.  The weights and the gate of channels lie in shared memory as fp32; the registers hold the
// sums over rows of a thread's NV times eight columns.  Rows of 257 to 8192 elements as there, if shared memory holds two of them: 16-bit types always,
// fp32 up to 5256 elements with a gate of channels and 5784 without (4096x5248 92 us, 5.6 TB/s; 4096x5264 by the kernel above 150).  Beyond, that
// kernel's registers spill: us at 2048x8192 fp32 99, 2048x16384 bf16 235 (1.7 TB/s), centred 380, fp32 362 (2.2 TB/s).
// us with weights, gate, residual, bf16: 8192x4096 71 with the sums' launch (403 MB: 5.7 TB/s), 4096x8192 75; centred 130 (five sums over rows leave one
// CTA of 512 threads on an SM).  One vector a thread and twice the warps: 90.
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

// ---- sums over rows --------------------------------------------------------------------------------------------------------------
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

// ---- host side -------------------------------------------------------------------------------------------------------------------
// How many parts of the rows the general kernel sums on their own (one for each group of threads): some rows for each, since the sums of
// a part are as many bytes as the rows of one.
static int norm_groups(int C) { return C <= 256 ? 4 : 1; }
static long long norm_parts(long long M, int C) {
    const int G = norm_groups(C);
    const long long most = 148LL * G * (C <= 2048 ? 4 : C <= 4096 ? 2 : 1), wanted = std::min(most, std::min(M, std::max(148LL * G, M / 4)));
    return (wanted + G - 1) / G * G;
}
// The most CTAs of the stream kernel, each of which sums its rows on its own: what an SM holds by registers of those the row's length chooses
// (norm_backward_sizes), and some rows for each.  0: rows that it does not take.
static int stream_rows(int C) { return C <= 2048 ? 4 : 2; }
static long long stream_parts(long long M, int C, bool layer) {
    if (C <= 256 || C > 8192) return 0;
    const int wide = C <= 512 ? 512 : C <= 1024 ? 1024 : C <= 2048 ? 2048 : C <= 4096 ? 4096 : 8192, each = layer ? std::max(1, 4096 / wide) : 8192 / wide;
    return std::min({M, 148LL * each, std::max(148LL, M / stream_rows(C))});
}
// Neither the kernel nor the number of sums is known here: room for whichever needs most.
size_t residual_norm_partial_bytes(long long M, int C) {
    const long long rows = std::max({norm_parts(M, C) * NORM_SUMS<true>, stream_parts(M, C, true) * NORM_SUMS<true>, stream_parts(M, C, false) * NORM_SUMS<false>});
    return (size_t)rows * (size_t)C * sizeof(float);
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
    // Below two rows an SM the general kernel is as fast (148x4096 8.9 us, this one 10.3; 296: 11.6 / 12.2; 444: 14.2 / 13.9; 2048: 72 / 26); a
    // CTA has some rows to itself, since its sums are as many bytes as some of them (us at 592x4096 / 2048x1024: 1 row 14.5 / 18.1, 4 rows 16.4 / 15.6).
    if (p.M < 2LL * blocks_sms()) return TAB_E_TOO_LARGE;
    const StreamPlan pl = stream_plan<kernel>(backward_threads(NV, LAYER) / THREADS, p.M, stream_rows(p.C), 4 * (size_t)p.C * type_bytes(TYPE), (p.gkind == TAB_GATE_CHANNEL ? 12 : 8) * (size_t)p.C);
    if (!pl.stages) return TAB_E_TOO_LARGE;
    int* status = device_status_word();
    if (stalled(status)) return TAB_E_STALLED;
    const bool sums = wants_sums(b);
    if (!sums) b.partial = nullptr;
    const int ctas = (int)std::min<long long>(stream_parts(p.M, p.C, LAYER), pl.ctas);
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
int residual_norm_backward_dispatch(const NormBackwardParams& p, int type, cudaStream_t stream) {
    return type == TAB_FP32 ? norm_backward_sizes<TAB_FP32>(p, stream) : type == TAB_BF16 ? norm_backward_sizes<TAB_BF16>(p, stream) : norm_backward_sizes<TAB_FP16>(p, stream);
}

}  // namespace tab
