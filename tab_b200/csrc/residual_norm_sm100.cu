// The norm after a block with its gate, the scaled residual, and the norm before the next block in one pass over the rows
// (tab_residual_norm_launch); the mathematics stand in residual_norm_common.cuh.
#include "residual_norm_common.cuh"

namespace tab {

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

// A row by GT threads, at once: rows that are not aligned, of at most 256 elements or of more than 8192.  (Aligned ones the kernel below takes, single
// rows too: 1x4096 2.9 us, 3.9 here; 4096x8192 45.7 / 61.5.)
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
            auto scale = [&](uint32_t bits) { return p.format == TAB_E5M2 ? scale_byte<TAB_E5M2>(bits) : scale_byte<TAB_E4M3>(bits); };
            uint32_t a[2] = {0, 0};                                        // VEC: sixteen threads hold a block; else a warp holds two, four columns a lane of each
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const uint32_t b = col.in(i, j) ? finite_bits(v[i][j]) : 0u;
                a[VEC ? 0 : j >> 2] = max(a[VEC ? 0 : j >> 2], b);
            }
            if (VEC) {
                const uint32_t sb = scale(half_warp_max(a[0]));
                const int c = col.at(i, 0);
                const float inv = __uint_as_float(inverse_bits(sb));
                if (c < p.C) {
                    *reinterpret_cast<uint2*>(q + c) = p.format == TAB_E5M2 ? narrow8<TAB_E5M2>(v[i], inv) : narrow8<TAB_E4M3>(v[i], inv);
                    if ((g & 15) == 0) p.s[(long long)(c / BLK) * p.lds + m] = (uint8_t)sb;
                }
            } else {
                float sc[8];
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const uint32_t top = half_warp_max(max(a[h], __shfl_xor_sync(0xFFFFFFFFu, a[h], 16)));
                    const uint32_t sb = scale(top);
                    const int c = col.at(i, 4 * h);
#pragma unroll
                    for (int j = 0; j < 4; j++) sc[4 * h + j] = __uint_as_float(inverse_bits(sb));
                    if ((g & 31) == 0 && c < p.C) p.s[(long long)(c / BLK) * p.lds + m] = (uint8_t)sb;
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

// ---- many rows -------------------------------------------------------------------------------------------------------------------
// CTAs that stay: rows come by bulk copies into a ring in shared memory, a few rows ahead, so that the memory is asked for the next rows while
// the threads meet over this one.  Weights and a gate of channels stay in registers from row to row, so that they are read once a CTA; shifts
// and other gates are loaded for every row.  Rows of 257 to 8192 elements that start, and are spaced, on 16 bytes and eight elements; wider ones and all
// others take the kernel above, without a row in flight (2048x16384 bf16 77 us, 3.5 TB/s, centred 110; fp32 106, 5.1 TB/s).
// us with weights, gate and residual, bf16: 8192x4096 46.4 (268 MB: 5.8 TB/s), 4096x8192 45.8, to blocks 57.2; bound by instructions between the
// meetings of a row (23 M warp instructions at 8192x4096, 1.9 a cycle and SM), with one vector a thread 58, not FAST and without pairs 61.
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
                // The larger magnitudes, which fmaxf takes past NaN, from 0 on, so that eight NaN leave 0; rows with an infinity are looked at again.
                float a[NV], most = 0.f;
#pragma unroll
                for (int i = 0; i < NV; i++) {
                    a[i] = fmaxf(fmaxf(fmaxf(fmaxf(0.f, fabsf(v[i][0].x)), fabsf(v[i][0].y)), fmaxf(fabsf(v[i][1].x), fabsf(v[i][1].y))),
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

// ---- host side -------------------------------------------------------------------------------------------------------------------
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

// TAB_E_TOO_LARGE: the stream kernel does not take the problem.
template <int TYPE, int THREADS, int NV, bool LAYER, bool QUANT, bool FAST>
static int launch_norm_stream_as(const NormParams& p, cudaStream_t stream) {
    constexpr auto kernel = residual_norm_stream_kernel<TYPE, THREADS, NV, LAYER, QUANT, FAST>;
    const StreamPlan pl = stream_plan<kernel>(forward_threads(LAYER, FAST) / THREADS, p.M, 1, 2 * (size_t)p.C * type_bytes(TYPE), 0);
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
int residual_norm_dispatch(const NormParams& p, int type, cudaStream_t stream) {
    return type == TAB_FP32 ? norm_sizes<TAB_FP32>(p, stream) : type == TAB_BF16 ? norm_sizes<TAB_BF16>(p, stream) : norm_sizes<TAB_FP16>(p, stream);
}

}  // namespace tab
