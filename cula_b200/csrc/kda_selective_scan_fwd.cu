// Selective scan, forward (definition and layout: selective_scan.cuh). One CTA walks a segment of a sequence for a tile of channels, LC
// tokens at a time. Four warps scan: every (token, channel, state) costs one exponential and four multiply-adds (packed in pairs) on
// states that stay in registers. Four others serve them: they fetch the rows of the tiles ahead, make the steps and their products with x,
// once per token and channel, for the next tile, and turn the sums of the tile before into outputs. One barrier per tile.
//
// What it cannot do without at 4 x 2048 tokens x 4096 channels x 16 states in bf16 with a gate (268 MB): 42 us of HBM traffic, 115 us of
// exponentials (16 per clock and SM), 137 with the three of softplus and silu per token and channel. Measured: 524 us with every thread staging, scanning and writing
// in turn (B and C rows waited for in registers, 16-byte loads of 32 lanes to 32 lines for the kept states), 219 us so; 235 with the
// states kept for a backward pass. The unit of the exponentials is 66 % busy: 256 CTAs leave 40 of 148 SMs with one CTA in place of two
// (86 %), and of a pair's time it is busy for three quarters; the data path of shared memory is half busy beside it. An eighth or a quarter
// of the exponentials as polynomials on the multiply-add units made it 6 and 9 us slower.
#include "selective_scan.cuh"

namespace kda {

constexpr int SEL_AHEAD = 4;                   // tiles of rows: the one that outputs are made of, the one that is scanned, two ahead
constexpr int SEL_FWD_THREADS = 2 * SEL_THREADS;

__device__ __forceinline__ void sel_barrier() { asm volatile("bar.sync 1, %0;" :: "n"(SEL_FWD_THREADS) : "memory"); }

template <int SL, typename T>
struct SelFwdSmem {
    using G = SelShape<SL>;
    static constexpr int Q = SelVec<T>::Q;
    float4 dx[2][G::LC][G::CH / 2];                                  // two channels' steps, and their products with x
    float4 b[2][G::LC][G::SL], c[2][G::LC][G::SL];
    float2 y[2][G::LC][G::CH / 2 + 2];                               // rows shifted against each other: no bank conflicts of the writers
    T raw_b[SEL_AHEAD][G::UNITS][4], raw_c[SEL_AHEAD][G::UNITS][4];                  // B and C rows as they are
    uint4 raw[SEL_AHEAD][3][Q][G::ITEMS];                                    // x, dt, z rows as they are: [stage][which][piece][thread]
};

// STATE_ONLY: what each segment adds to the state that enters it, and the sum of its steps; nothing else
template <int SL, typename T, bool STATE_ONLY>
__global__ void __launch_bounds__(SEL_FWD_THREADS, 2) kda_selective_scan_fwd_kernel(const SelScanArgs a, const int tiles_per_group) {
    using G = SelShape<SL>;
    using V = SelVec<T>;
    constexpr int LC = G::LC, CH = G::CH, SP = G::SP, Q = V::Q;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    SelFwdSmem<SL, T>& sm = *reinterpret_cast<SelFwdSmem<SL, T>*>(smem_raw);
    const int tid = threadIdx.x % SEL_THREADS, lane = tid & 31, warp = tid >> 5;
    const bool scans = threadIdx.x < SEL_THREADS;
    const int tiles = tiles_per_group * a.G, tile = blockIdx.x % tiles;
    const int group = tile / tiles_per_group, per_group = a.D / a.G;
    const int d0 = group * per_group + (tile % tiles_per_group) * CH, d_end = (group + 1) * per_group;
    pdl_wait();
    SelItem it;
    if (!sel_item(a, blockIdx.x / tiles, it)) return;
    if (STATE_ONLY && it.seg == it.segs - 1) return;                 // nothing comes after it

    const int n_tiles = (it.t1 - it.t0 + LC - 1) / LC;

    if (!scans) {
        // ---- the thread's piece of a staged tile: token `tt` of it, channels dv..dv+7 ----
        const int tt = tid / G::VECS, dv = d0 + 8 * (tid % G::VECS);
        const bool item = tid < G::ITEMS && dv < d_end;
        const int batch = a.cu_seqlens ? 0 : it.seq;
        const long long first = a.cu_seqlens ? it.row0 : 0;              // token of the sequence's row in its tensors
        const T* xp = static_cast<const T*>(a.x) + batch * a.x_seq + first * a.x_row + dv;
        const T* dtp = static_cast<const T*>(a.dt) + batch * a.dt_seq + first * a.dt_row + dv;
        const T* zp = static_cast<const T*>(a.z) + batch * a.z_seq + first * a.z_row + dv;
        const T* bp = static_cast<const T*>(a.Bm) + batch * a.b_seq + first * a.b_row + group * a.S;
        const T* cp = static_cast<const T*>(a.Cm) + batch * a.c_seq + first * a.c_row + group * a.S;
        const bool gate = !STATE_ONLY && a.z != nullptr;
        const int x_row = (int)a.x_row, dt_row = (int)a.dt_row, z_row = (int)a.z_row, b_row = (int)a.b_row, c_row = (int)a.c_row;
        auto fetch = [&](int k) {                                        // tile k into its stage
            const int t = it.t0 + k * LC + tt;
            if (item && k < n_tiles && t < it.t1) {
                uint4(*to)[Q][G::ITEMS] = sm.raw[k % SEL_AHEAD];
#pragma unroll
                for (int q = 0; q < Q; ++q) {
                    sel_copy16(&to[0][q][tid], xp + (long long)t * x_row + q * (8 / Q));
                    sel_copy16(&to[1][q][tid], dtp + (long long)t * dt_row + q * (8 / Q));
                    if (gate) sel_copy16(&to[2][q][tid], zp + (long long)t * z_row + q * (8 / Q));
                }
            }
#pragma unroll
            for (int u = 0; u < G::UB; ++u) {
                const int i = u * SEL_THREADS + tid, t = it.t0 + k * LC + i / SL;
                if (i < G::UNITS && k < n_tiles && t < it.t1) {
                    sel_fetch4(sm.raw_b[k % SEL_AHEAD][i], bp + (long long)t * b_row, 4 * (i % SL), a.S, a.vec_bc);
                    if (!STATE_ONLY) sel_fetch4(sm.raw_c[k % SEL_AHEAD][i], cp + (long long)t * c_row, 4 * (i % SL), a.S, a.vec_bc);
                }
            }
            sel_commit();
        };
        float2 bias[4], skip[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            bias[e] = item && a.dt_bias ? make_float2(a.dt_bias[dv + 2 * e], a.dt_bias[dv + 2 * e + 1]) : make_float2(0.f, 0.f);
            skip[e] = !STATE_ONLY && item && a.skip ? make_float2(a.skip[dv + 2 * e], a.skip[dv + 2 * e + 1]) : make_float2(0.f, 0.f);
        }
        auto stage = [&](int k) {                                        // tile k, arrived, as the scan takes it; zeros past the end change no state
            const int buf = k & 1, slot = k % SEL_AHEAD;
            if (tid < G::ITEMS) {
                const uint4(*from)[Q][G::ITEMS] = sm.raw[slot];
                float2 x[4], d[4];
                V::unpack(&from[0][0][tid], G::ITEMS, x);
                V::unpack(&from[1][0][tid], G::ITEMS, d);
#pragma unroll
                for (int e = 0; e < 4; ++e) d[e] = add2(d[e], bias[e]);
                if (a.softplus) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) d[e] = sel_softplus2(d[e]);
                }
                if (!(item && it.t0 + k * LC + tt < it.t1)) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) d[e] = x[e] = make_float2(0.f, 0.f);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float2 p = mul2(d[e], x[e]);
                    sm.dx[buf][tt][e * G::VECS + tid % G::VECS] = make_float4(d[e].x, d[e].y, p.x, p.y);
                }
            }
#pragma unroll
            for (int u = 0; u < G::UB; ++u) {
                const int i = u * SEL_THREADS + tid;
                if (i < G::UNITS) {
                    const bool live = it.t0 + k * LC + i / SL < it.t1;
                    const float4 rb = V::four(sm.raw_b[slot][i]);
                    sm.b[buf][i / SL][i % SL] = live ? rb : make_float4(0.f, 0.f, 0.f, 0.f);
                    if (!STATE_ONLY) {
                        const float4 rc = V::four(sm.raw_c[slot][i]);
                        sm.c[buf][i / SL][i % SL] = live ? rc : make_float4(0.f, 0.f, 0.f, 0.f);
                    }
                }
            }
        };

        auto finish = [&](int k) {                                       // the outputs of tile k
            const int t = it.t0 + k * LC + tt;
            if (item && t < it.t1) {
                const uint4(*from)[Q][G::ITEMS] = sm.raw[k % SEL_AHEAD];
                float2 x[4], o[4];
                V::unpack(&from[0][0][tid], G::ITEMS, x);
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = fma2(skip[e], x[e], sm.y[k & 1][tt][e * G::VECS + tid % G::VECS]);
                const size_t at = (size_t)(it.row0 + t) * a.D + dv;
                if (gate) {
                    if (a.y_pre) SelVec<float>::store(a.y_pre + at, o);
                    float2 z[4];
                    V::unpack(&from[2][0][tid], G::ITEMS, z);
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[e] = mul2(mul2(o[e], z[e]), sel_sigmoid2(z[e]));
                }
                V::store(static_cast<T*>(a.y) + at, o);
            }
        };
        if (n_tiles > 0) {
            fetch(0);
            fetch(1);
            fetch(2);
            sel_wait<2>();
            stage(0);
            sel_barrier();
        }
        for (int k = 0; k < n_tiles; ++k) {
            if (k + 1 < n_tiles) {
                sel_wait<1>();                                       // tile k + 1 is here, k + 2 on its way
                stage(k + 1);
            }
            if (!STATE_ONLY && k > 0) finish(k - 1);
            fetch(k + 3);                                            // where tile k - 1 was
            sel_barrier();
        }
        if (!STATE_ONLY && n_tiles > 0) finish(n_tiles - 1);
        sel_wait<0>();
        return;
    }

    // ---- what the thread holds: states n0..n0+3 of channels dc, dc+1 ----
    const int cl = lane & (G::CL - 1), s = lane / G::CL, n0 = 4 * s, pair = warp * G::CL + cl, dc = d0 + 8 * cl + 2 * warp;
    const bool own = dc < d_end;                                     // tiles and groups are whole pieces of 8 channels
    float2 A2[2][2], h[2][2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        h[c][0] = h[c][1] = A2[c][0] = A2[c][1] = make_float2(0.f, 0.f);
        if (own) {
            sel_load_rates(a.A + (size_t)(dc + c) * a.S, n0, a.S, A2[c]);
            if (!STATE_ONLY && a.h0) sel_load4(a.h0 + ((size_t)it.seq * a.D + dc + c) * a.S, n0, a.S, h[c]);
        }
    }
    if constexpr (!STATE_ONLY) {
        if (it.seg && own) {                                         // the segments before this one
#pragma unroll 4
            for (int q = 0; q < it.seg; ++q) {
                const size_t at = (size_t)(it.slot0 + q) * a.D + dc;
                const float2 sum = *reinterpret_cast<const float2*>(a.seg_dt + at);
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const float4 add = *reinterpret_cast<const float4*>(a.seg_state + (at + c) * SP + n0);
                    const float2 d = splat2(c ? sum.y : sum.x);
                    h[c][0] = fma2(decay2(d, A2[c][0]), h[c][0], make_float2(add.x, add.y));
                    h[c][1] = fma2(decay2(d, A2[c][1]), h[c][1], make_float2(add.z, add.w));
                }
            }
        }
    }

    float2 sum_dt = make_float2(0.f, 0.f);
    if (n_tiles > 0) sel_barrier();
    for (int k = 0; k < n_tiles; ++k) {
        const int buf = k & 1;
        // The sums over states come after the tile's last token: everything before is independent of their exchanges, and no shared store
        // stands between its loads. A warp alone on its scheduler takes 125 cycles per token, two of them 103 each; 65 are exponentials.
        float v[2 * LC];
#pragma unroll
        for (int u = 0; u < LC; ++u) {
            if (!STATE_ONLY && u % SEL_KEEP == 0 && a.states && it.t0 + k * LC + u < it.t1) {
                float4* to = sel_kept<SL>(a, it.chunk0, it.t0 + k * LC + u, tile, tiles) + warp * 64 + lane;
#pragma unroll
                for (int c = 0; c < 2; ++c) to[c * 32] = make_float4(h[c][0].x, h[c][0].y, h[c][1].x, h[c][1].y);
            }
            const float4 dx = sm.dx[buf][u][pair], b = sm.b[buf][u][s];
            if (STATE_ONLY) sum_dt = add2(sum_dt, make_float2(dx.x, dx.y));
            float4 cc;
            if (!STATE_ONLY) cc = sm.c[buf][u][s];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const float2 d = splat2(c ? dx.y : dx.x), p = splat2(c ? dx.w : dx.z);
                h[c][0] = fma2(p, make_float2(b.x, b.y), mul2(decay2(d, A2[c][0]), h[c][0]));
                h[c][1] = fma2(p, make_float2(b.z, b.w), mul2(decay2(d, A2[c][1]), h[c][1]));
                if (!STATE_ONLY) {
                    const float2 q = fma2(make_float2(cc.z, cc.w), h[c][1], mul2(make_float2(cc.x, cc.y), h[c][0]));
                    v[2 * u + c] = q.x + q.y;
                }
            }
        }
        if constexpr (!STATE_ONLY) {
            sel_reduce<2 * LC, SL>(v, lane, G::CL);
            constexpr int LEFT = LC / SL;                            // tokens whose sums each lane is left with
#pragma unroll
            for (int u = 0; u < LEFT; ++u) sm.y[buf][s * LEFT + u][pair] = make_float2(v[2 * u], v[2 * u + 1]);
        }
        sel_barrier();
    }
    // Not before: what follows in the stream would take places beside CTAs that run for long, and leave other SMs empty.
    pdl_launch_dependents();
    if (!own) return;
    if constexpr (STATE_ONLY) {
        const size_t at = (size_t)(it.slot0 + it.seg) * a.D + dc;
#pragma unroll
        for (int c = 0; c < 2; ++c)
            *reinterpret_cast<float4*>(a.seg_state + (at + c) * SP + n0) = make_float4(h[c][0].x, h[c][0].y, h[c][1].x, h[c][1].y);
        if (s == 0) *reinterpret_cast<float2*>(a.seg_dt + at) = sum_dt;
    } else if (a.hT && it.seg == it.segs - 1) {
#pragma unroll
        for (int c = 0; c < 2; ++c) sel_store4(a.hT + ((size_t)it.seq * a.D + dc + c) * a.S, n0, a.S, h[c]);
    }
}

template <int SL, typename T>
static int launch_sel_fwd(const SelScanArgs& a, cudaStream_t stream) {
    using G = SelShape<SL>;
    const int tpg = (a.D / a.G + G::CH - 1) / G::CH;
    const long long items = sel_items(a);
    const long long blocks = items * tpg * a.G;
    if (blocks == 0) return 0;
    if (blocks > 0x7fffffffLL) return -1;
    static_assert(sizeof(SelFwdSmem<SL, T>) <= 227 * 1024, "");
    constexpr int smem = sizeof(SelFwdSmem<SL, T>);
    static std::atomic<unsigned long long> done[2];
    if (a.seg_chunks) {
        if (const cudaError_t e = allow_smem(kda_selective_scan_fwd_kernel<SL, T, true>, smem, done[1]); e != cudaSuccess) return (int)launched(e);
        if (const cudaError_t e = sel_launch(sel_long(a), kda_selective_scan_fwd_kernel<SL, T, true>, blocks, SEL_FWD_THREADS, smem, stream, a, tpg);
            e != cudaSuccess)
            return (int)e;
    }
    if (const cudaError_t e = allow_smem(kda_selective_scan_fwd_kernel<SL, T, false>, smem, done[0]); e != cudaSuccess) return (int)launched(e);
    return (int)sel_launch(sel_long(a), kda_selective_scan_fwd_kernel<SL, T, false>, blocks, SEL_FWD_THREADS, smem, stream, a, tpg);
}

}  // namespace kda

extern "C" int kda_launch_selective_scan_fwd(const kda::SelScanArgs* a, int state_lanes, cudaStream_t stream) {
    using namespace kda;
    switch (state_lanes) {
        case 2: return a->fp32 ? launch_sel_fwd<2, float>(*a, stream) : launch_sel_fwd<2, __nv_bfloat16>(*a, stream);
        case 4: return a->fp32 ? launch_sel_fwd<4, float>(*a, stream) : launch_sel_fwd<4, __nv_bfloat16>(*a, stream);
        case 8: return a->fp32 ? launch_sel_fwd<8, float>(*a, stream) : launch_sel_fwd<8, __nv_bfloat16>(*a, stream);
        case 16: return a->fp32 ? launch_sel_fwd<16, float>(*a, stream) : launch_sel_fwd<16, __nv_bfloat16>(*a, stream);
    }
    return -1;
}
