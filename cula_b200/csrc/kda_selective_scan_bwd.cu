// Selective scan, backward (definition and layout: selective_scan.cuh). With g_t the gradient of h_t,
//     g_t = dy_t C_t + a_{t+1} g_{t+1},     a_t = exp(dt_t A),     dy_t = dout_t silu(z_t)
//     dC_t = sum_d dy_t h_t            dB_t = sum_d g_t dt_t x_t         dA = sum_t w_t dt_t,   w_t = a_t g_t h_{t-1}
//     dx_t = dt_t sum_n g_t B_t + skip dy_t                              ddt_t = x_t sum_n g_t B_t + sum_n w_t A
//     dz_t = dout_t y_t silu'(z_t)     dskip = sum_t dy_t x_t            dh0 = a_1 g_1
// One CTA walks a segment of a sequence backwards for a tile of channels. The states between are made again, eight tokens at a time, from
// those that the forward pass kept, and stay in registers together with the a_t until the way back has used them. Sums over states go over
// the lanes of a channel, sums over channels over the lanes of a state and the warps; the tiles' shares of dB and dC and the CTAs' shares
// of dA, dskip and dbias are added up by a second kernel in a fixed order, so that every gradient is the same from run to run.
//
// Four warps scan, with the 136 registers that eight tokens' states and factors take, and four serve them as in the forward pass: rows two
// tiles ahead, operands of the next tile, gradients of the tile before. Per element one exponential, eleven multiply-adds (packed in
// pairs) and two sums over lanes, which go as half of the values per step. At 4 x 2048 x 4096 x 16 in bf16 with a gate: 473 MB of inputs and
// gradients (73 us) and 536 of kept states, y before the gate and shares of dB and dC there and back (83 us more), 115 us of the recurrence's
// exponentials (165 with softplus and three sigmoids per token and channel), 184 us of multiply-adds at their rate. Measured: 1040 us with
// every thread doing everything, 567 so (lone CTAs 345). Nothing is saturated: issue slots 58 %, of which packed multiply-adds take two each, shared memory's data path 53 %
// of the launch; 22 % of the warps that would fit are resident, since registers and shared memory hold two CTAs per SM. Tried: sums over
// channels by tensor-core products with ones (590: fewer exchanges, no less time), packed pairs over channels in place of states (689: B
// and C twice in shared memory), eight scanning warps and four serving ones in one CTA per SM (617), other register splits (176 + 80: 592).
#include "selective_scan.cuh"

namespace kda {

constexpr int SEL_BWD_THREADS = 2 * SEL_THREADS;
constexpr int SEL_SCAN_REGS = 184, SEL_SERVE_REGS = 72;             // of a thread of either kind; the block is launched with their mean

__device__ __forceinline__ void sel_bwd_barrier() { asm volatile("bar.sync 1, %0;" :: "n"(SEL_BWD_THREADS) : "memory"); }

template <int SL, typename T>
struct SelBwdSmem {
    using G = SelShape<SL>;
    // tiles of rows: of the gradients that are made, of the next tile, and one more where the rows are of 16 bits and two CTAs share an SM all
    // the same (64 states, 4 x 2048 x 4096: 2.88 ms with three, 2.13 with two). With 64 states in fp32 one CTA has the SM either way.
    static constexpr int Q = SelVec<T>::Q, RING = Q == 1 && SL < 16 ? 3 : 2;
    float4 dx[2][G::LC][G::CH / 2];                                  // two channels' steps, and their products with x
    float2 dy[2][G::LC][G::CH / 2];
    float4 b[2][G::LC][SL], c[2][G::LC][SL];
    float4 sums[2][G::LC][G::CH / 2];                                // two channels' sum_n g B, sum_n w A (log2 units)
    float bc[2][SEL_WARPS][G::LC][2 * G::SP];                        // per warp: dB, dC
    float2 par[2][4][G::VECS];                                       // dt_bias, skip: [which][pair of a piece][piece]
    T raw_b[RING][G::UNITS][4], raw_c[RING][G::UNITS][4];            // B and C rows as they are
    uint4 raw[RING][4][Q][G::ITEMS];                                 // x, dt, z, dout rows as they are
    union {
        float4 kept[G::LC / SEL_KEEP][2][SEL_THREADS];               // each thread's states before every eighth token
        float4 acc[4][G::ITEMS];                                     // at the end: the serving threads' sums for dskip and dbias
    };
    static_assert(sizeof(acc) <= 2 * sizeof(kept), "");
};
static_assert(sizeof(SelBwdSmem<16, __nv_bfloat16>) <= 113 * 1024 && sizeof(SelBwdSmem<4, float>) <= 113 * 1024, "two CTAs per SM");

// What the serving warps do for an item: rows of the tiles to come, operands of the next tile, gradients of the one before.
template <int SL, typename T, bool STATE_ONLY>
__device__ __forceinline__ void sel_bwd_serve(const SelScanArgs& a, SelBwdSmem<SL, T>& sm, const SelItem& it, int d0, int d_end, int group, int share,
                                              float2 (&acc)[2][4]) {
    using G = SelShape<SL>;
    using V = SelVec<T>;
    constexpr int LC = G::LC, SP = G::SP, Q = V::Q, RING = SelBwdSmem<SL, T>::RING;
    const int tid = threadIdx.x % SEL_THREADS, tt = tid / G::VECS, vec = tid % G::VECS, dv = d0 + 8 * vec;
    const bool item = tid < G::ITEMS && dv < d_end, gate = a.z != nullptr;
    const int batch = a.cu_seqlens ? 0 : it.seq, n_tiles = (it.t1 - it.t0 + LC - 1) / LC;
    const long long first = a.cu_seqlens ? it.row0 : 0;
    const T* xp = static_cast<const T*>(a.x) + batch * a.x_seq + first * a.x_row + dv;
    const T* dtp = static_cast<const T*>(a.dt) + batch * a.dt_seq + first * a.dt_row + dv;
    const T* zp = static_cast<const T*>(a.z) + batch * a.z_seq + first * a.z_row + dv;
    const T* dop = static_cast<const T*>(a.dy) + (size_t)it.row0 * a.D + dv;
    const T* bp = static_cast<const T*>(a.Bm) + batch * a.b_seq + first * a.b_row + group * a.S;
    const T* cp = static_cast<const T*>(a.Cm) + batch * a.c_seq + first * a.c_row + group * a.S;
    const int x_row = (int)a.x_row, dt_row = (int)a.dt_row, z_row = (int)a.z_row, b_row = (int)a.b_row, c_row = (int)a.c_row;
    // tiles are taken from the last to the first; the j-th taken is tile n_tiles - 1 - j
    auto fetch = [&](int j) {
        const int t_first = it.t0 + (n_tiles - 1 - j) * LC, t = t_first + tt, slot = j % RING;
        if (item && j < n_tiles && t < it.t1) {
            uint4(*to)[Q][G::ITEMS] = sm.raw[slot];
#pragma unroll
            for (int q = 0; q < Q; ++q) {
                sel_copy16(&to[0][q][tid], xp + (long long)t * x_row + q * (8 / Q));
                sel_copy16(&to[1][q][tid], dtp + (long long)t * dt_row + q * (8 / Q));
                if (gate) sel_copy16(&to[2][q][tid], zp + (long long)t * z_row + q * (8 / Q));
                sel_copy16(&to[3][q][tid], dop + (size_t)t * a.D + q * (8 / Q));
            }
        }
#pragma unroll
        for (int u = 0; u < G::UB; ++u) {
            const int i = u * SEL_THREADS + tid, tb = t_first + i / SL;
            if (i < G::UNITS && j < n_tiles && tb < it.t1) {
                if (!STATE_ONLY) sel_fetch4(sm.raw_b[slot][i], bp + (long long)tb * b_row, 4 * (i % SL), a.S, a.vec_bc);
                sel_fetch4(sm.raw_c[slot][i], cp + (long long)tb * c_row, 4 * (i % SL), a.S, a.vec_bc);
            }
        }
        sel_commit();
    };
    auto stage = [&](int j) {
        const int buf = j & 1, t_first = it.t0 + (n_tiles - 1 - j) * LC, slot = j % RING;
        if (tid < G::ITEMS) {                                        // zeros for channels past the tile: they add nothing to dB and dC
            const bool live = item && t_first + tt < it.t1;
            const uint4(*from)[Q][G::ITEMS] = sm.raw[slot];
            float2 x[4], d[4];
            V::unpack(&from[1][0][tid], G::ITEMS, d);
#pragma unroll
            for (int e = 0; e < 4; ++e) d[e] = add2(d[e], sm.par[0][e][vec]);
            if (a.softplus) {
#pragma unroll
                for (int e = 0; e < 4; ++e) d[e] = sel_softplus2(d[e]);
            }
            V::unpack(&from[0][0][tid], G::ITEMS, x);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float2 p = mul2(d[e], x[e]);
                sm.dx[buf][tt][e * G::VECS + vec] = live ? make_float4(d[e].x, d[e].y, p.x, p.y) : make_float4(0.f, 0.f, 0.f, 0.f);
            }
            float2 o[4];
            V::unpack(&from[3][0][tid], G::ITEMS, o);
            if (gate) {
                float2 z[4];
                V::unpack(&from[2][0][tid], G::ITEMS, z);
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = mul2(mul2(o[e], z[e]), sel_sigmoid2(z[e]));
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) sm.dy[buf][tt][e * G::VECS + vec] = live ? o[e] : make_float2(0.f, 0.f);
        }
#pragma unroll
        for (int u = 0; u < G::UB; ++u) {
            const int i = u * SEL_THREADS + tid;
            if (i < G::UNITS) {
                const bool live = t_first + i / SL < it.t1;
                if (!STATE_ONLY) {
                    const float4 rb = V::four(sm.raw_b[slot][i]);
                    sm.b[buf][i / SL][i % SL] = live ? rb : make_float4(0.f, 0.f, 0.f, 0.f);
                }
                const float4 rc = V::four(sm.raw_c[slot][i]);
                sm.c[buf][i / SL][i % SL] = live ? rc : make_float4(0.f, 0.f, 0.f, 0.f);
            }
        }
    };
    auto finish = [&](int j) {
        const int buf = j & 1, t_first = it.t0 + (n_tiles - 1 - j) * LC, t = t_first + tt;
        if (item && t < it.t1) {
            const uint4(*from)[Q][G::ITEMS] = sm.raw[j % RING];
            const size_t at = (size_t)(it.row0 + t) * a.D + dv;
            float4 y0, y1;
            if (gate) {                                              // on its way while dx and ddt are made
                y0 = reinterpret_cast<const float4*>(a.y_pre + at)[0];
                y1 = reinterpret_cast<const float4*>(a.y_pre + at)[1];
            }
            float2 x[4], d[4], sg[4];
            V::unpack(&from[1][0][tid], G::ITEMS, d);
            if (a.softplus) {
#pragma unroll
                for (int e = 0; e < 4; ++e) sg[e] = sel_sigmoid2(add2(d[e], sm.par[0][e][vec]));
            } else sg[0] = sg[1] = sg[2] = sg[3] = splat2(1.f);
            V::unpack(&from[0][0][tid], G::ITEMS, x);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float4 sums = sm.sums[buf][tt][e * G::VECS + vec], step = sm.dx[buf][tt][e * G::VECS + vec];
                const float2 gB = make_float2(sums.x, sums.z), dy = sm.dy[buf][tt][e * G::VECS + vec];
                d[e] = mul2(fma2(x[e], gB, mul2(make_float2(sums.y, sums.w), splat2(0.6931471805599453f))), sg[e]);      // A is held times log2(e)
                acc[0][e] = fma2(dy, x[e], acc[0][e]);
                acc[1][e] = add2(acc[1][e], d[e]);
                x[e] = fma2(make_float2(step.x, step.y), gB, mul2(sm.par[1][e][vec], dy));
            }
            V::store(static_cast<T*>(a.ddt) + at, d);
            V::store(static_cast<T*>(a.dx) + at, x);
            if (gate) {
                float2 z[4], o[4];
                V::unpack(&from[2][0][tid], G::ITEMS, z);
                V::unpack(&from[3][0][tid], G::ITEMS, o);
                const float2 y[4] = {make_float2(y0.x, y0.y), make_float2(y0.z, y0.w), make_float2(y1.x, y1.y), make_float2(y1.z, y1.w)};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float2 s = sel_sigmoid2(z[e]);             // silu' = s (1 + z (1 - s))
                    o[e] = mul2(mul2(o[e], y[e]), mul2(s, fma2(z[e], fma2(s, splat2(-1.f), splat2(1.f)), splat2(1.f))));
                }
                V::store(static_cast<T*>(a.dz) + at, o);
            }
        }
        // this tile of channels' share of dB and dC
        for (int i = tid; i < LC * SP / 2; i += SEL_THREADS) {
            const int u = i / (SP / 2), n = 4 * (i % (SP / 2));
            if (t_first + u < it.t1) {
                float4 sum = *reinterpret_cast<const float4*>(&sm.bc[buf][0][u][n]);
#pragma unroll
                for (int w = 1; w < SEL_WARPS; ++w) {
                    const float4 r = *reinterpret_cast<const float4*>(&sm.bc[buf][w][u][n]);
                    sum.x += r.x; sum.y += r.y; sum.z += r.z; sum.w += r.w;
                }
                const size_t at = (((size_t)share * a.rows + it.row0 + t_first + u) * a.G + group) * (2 * SP) + n;
                *reinterpret_cast<float4*>(a.part_bc + at) = sum;
            }
        }
    };
    if (n_tiles == 0) return;
#pragma unroll
    for (int j = 0; j < RING - 1; ++j) fetch(j);
    sel_wait<RING - 2>();
    stage(0);
    sel_bwd_barrier();
    for (int j = 0; j < n_tiles; ++j) {
        if (!STATE_ONLY && j > 0) finish(j - 1);
        fetch(j + RING - 1);                                         // where tile j - 1 was
        sel_wait<RING - 2>();                                        // tile j + 1 is here
        if (j + 1 < n_tiles) stage(j + 1);
        sel_bwd_barrier();
    }
    if (!STATE_ONLY) finish(n_tiles - 1);
    sel_wait<0>();
}

// STATE_ONLY: what each segment adds to the gradient of the state that leaves it, and the sum of its steps
template <int SL, typename T, bool STATE_ONLY>
__global__ void __launch_bounds__(SEL_BWD_THREADS, 2) kda_selective_scan_bwd_kernel(const SelScanArgs a, const int tiles_per_group, const long long items) {
    using G = SelShape<SL>;
    constexpr int LC = G::LC, CH = G::CH, CL = G::CL, SP = G::SP, KEEP = SEL_KEEP, SUBS = LC / KEEP;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    SelBwdSmem<SL, T>& sm = *reinterpret_cast<SelBwdSmem<SL, T>*>(smem_raw);
    const int tid = threadIdx.x % SEL_THREADS, lane = tid & 31, warp = tid >> 5;
    const int tiles = tiles_per_group * a.G, tile = blockIdx.x % tiles, row = blockIdx.x / tiles;
    const int group = tile / tiles_per_group, per_group = a.D / a.G, share = tile % tiles_per_group;
    const int d0 = group * per_group + share * CH, d_end = (group + 1) * per_group;
    pdl_wait();

    if (threadIdx.x >= SEL_THREADS) {
        // Of the 128 registers per thread that the block starts with, the serving warps give up what the scanning ones need
        if constexpr (!STATE_ONLY) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" :: "n"(SEL_SERVE_REGS));
        for (int i = tid; i < CH; i += SEL_THREADS) {
            const bool in = d0 + i < d_end;
            (&sm.par[0][i / 2 % 4][i / 8].x)[i & 1] = in && a.dt_bias ? a.dt_bias[d0 + i] : 0.f;
            (&sm.par[1][i / 2 % 4][i / 8].x)[i & 1] = in && a.skip ? a.skip[d0 + i] : 0.f;
        }
        asm volatile("bar.sync 2, %0;" :: "n"(SEL_THREADS) : "memory");
        float2 acc[2][4];                                            // dskip and dbias of the thread's 8 channels
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[0][e] = acc[1][e] = make_float2(0.f, 0.f);
        for (long long i = row; i < items; i += a.cta_rows) {
            SelItem it;
            if (!sel_item(a, i, it) || (STATE_ONLY && it.seg == 0)) continue;
            sel_bwd_serve<SL, T, STATE_ONLY>(a, sm, it, d0, d_end, group, share, acc);
        }
        if constexpr (!STATE_ONLY) {
            sel_bwd_barrier();                                       // the scanning warps have read their last states
            if (tid < G::ITEMS) {
#pragma unroll
                for (int e = 0; e < 4; ++e) sm.acc[e][tid] = make_float4(acc[e / 2][2 * (e & 1)].x, acc[e / 2][2 * (e & 1)].y, acc[e / 2][2 * (e & 1) + 1].x, acc[e / 2][2 * (e & 1) + 1].y);
            }
            asm volatile("bar.sync 2, %0;" :: "n"(SEL_THREADS) : "memory");
            // dskip and dbias: the threads that stood at the same channels, in order
            for (int i = tid; i < 4 * G::VECS; i += SEL_THREADS) {
                const int v = i % G::VECS, e = i / G::VECS;
                if (d0 + 8 * v < d_end) {
                    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
                    for (int k = v; k < G::ITEMS; k += G::VECS) {
                        const float4 r = sm.acc[e][k];
                        sum.x += r.x; sum.y += r.y; sum.z += r.z; sum.w += r.w;
                    }
                    float* to = e < 2 ? a.part_skip : a.part_bias;
                    if (to) *reinterpret_cast<float4*>(to + (size_t)row * a.D + d0 + 8 * v + 4 * (e & 1)) = sum;
                }
            }
        }
        return;
    }
    if constexpr (!STATE_ONLY) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" :: "n"(SEL_SCAN_REGS));

    const int cl = lane & (CL - 1), s = lane / CL, n0 = 4 * s, pair = warp * CL + cl, dc = d0 + 8 * cl + 2 * warp;
    const bool own = dc < d_end;
    float2 A2[2][2], dA[2][2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        dA[c][0] = dA[c][1] = A2[c][0] = A2[c][1] = make_float2(0.f, 0.f);
        if (own) {
            sel_load_rates(a.A + (size_t)(dc + c) * a.S, n0, a.S, A2[c]);
        }
    }

    for (long long i = row; i < items; i += a.cta_rows) {
        SelItem it;
        if (!sel_item(a, i, it) || (STATE_ONLY && it.seg == 0)) continue;        // nothing comes before a first segment
        const int n_tiles = (it.t1 - it.t0 + LC - 1) / LC;
        // the kept states of place `sub` of the j-th tile taken
        auto fetch = [&](int j, int sub) {
            const int at = it.t0 + (n_tiles - 1 - j) * LC + sub * KEEP;
            if (j < n_tiles && at < it.t1) {
                const float4* from = sel_kept<SL>(a, it.chunk0, at, tile, tiles) + warp * 64 + lane;
                sel_copy16(&sm.kept[sub][0][tid], from);
                sel_copy16(&sm.kept[sub][1][tid], from + 32);
            }
            sel_commit();
        };
        if constexpr (!STATE_ONLY) {
#pragma unroll
            for (int sub = SUBS - 1; sub >= 0; --sub) fetch(0, sub);
        }

        float2 gh[2][2];                                             // a_{t+1} g_{t+1}: the gradient of h_t through what comes after
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            gh[c][0] = gh[c][1] = make_float2(0.f, 0.f);
            if (!STATE_ONLY && own && a.dhT) sel_load4(a.dhT + ((size_t)it.seq * a.D + dc + c) * a.S, n0, a.S, gh[c]);
        }
        if constexpr (!STATE_ONLY) {
            if (own) {                                               // the segments after this one
#pragma unroll 4
                for (int q = it.segs - 1; q > it.seg; --q) {
                    const size_t at = (size_t)(it.slot0 + q) * a.D + dc;
                    const float2 sum = *reinterpret_cast<const float2*>(a.seg_dt + at);
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const float4 add = *reinterpret_cast<const float4*>(a.seg_state + (at + c) * SP + n0);
                        const float2 d = splat2(c ? sum.y : sum.x);
                        gh[c][0] = fma2(decay2(d, A2[c][0]), gh[c][0], make_float2(add.x, add.y));
                        gh[c][1] = fma2(decay2(d, A2[c][1]), gh[c][1], make_float2(add.z, add.w));
                    }
                }
            }
        }

        float2 sum_dt = make_float2(0.f, 0.f);
        if (n_tiles > 0) sel_bwd_barrier();
        for (int j = 0; j < n_tiles; ++j) {
            const int buf = j & 1, tile_t0 = it.t0 + (n_tiles - 1 - j) * LC;
            if constexpr (STATE_ONLY) {
#pragma unroll
                for (int u = LC - 1; u >= 0; --u) {
                    const float4 dx = sm.dx[buf][u][pair], cc = sm.c[buf][u][s];
                    const float2 dy = sm.dy[buf][u][pair];
                    sum_dt = add2(sum_dt, make_float2(dx.x, dx.y));
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const float2 d = splat2(c ? dx.y : dx.x), o = splat2(c ? dy.y : dy.x);
                        gh[c][0] = mul2(decay2(d, A2[c][0]), fma2(o, make_float2(cc.x, cc.y), gh[c][0]));
                        gh[c][1] = mul2(decay2(d, A2[c][1]), fma2(o, make_float2(cc.z, cc.w), gh[c][1]));
                    }
                }
            } else {
#pragma unroll 1
                for (int sub = SUBS - 1; sub >= 0; --sub) {
                    const int tb = sub * KEEP;
                    float2 st[KEEP + 1][2][2], av[KEEP][2][2];       // states before and after each token; a_t
                    sel_wait<SUBS - 1>();
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const float4 r = sm.kept[sub][c][tid];
                        st[0][c][0] = make_float2(r.x, r.y);
                        st[0][c][1] = make_float2(r.z, r.w);
                    }
                    fetch(j + 1, sub);
                    if (tile_t0 + tb >= it.t1) continue;             // past the end: nothing in it
#pragma unroll
                    for (int u = 0; u < KEEP; ++u) {
                        const float4 dx = sm.dx[buf][tb + u][pair], b = sm.b[buf][tb + u][s];
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            const float2 d = splat2(c ? dx.y : dx.x), p = splat2(c ? dx.w : dx.z);
                            av[u][c][0] = decay2(d, A2[c][0]);
                            av[u][c][1] = decay2(d, A2[c][1]);
                            st[u + 1][c][0] = fma2(p, make_float2(b.x, b.y), mul2(av[u][c][0], st[u][c][0]));
                            st[u + 1][c][1] = fma2(p, make_float2(b.z, b.w), mul2(av[u][c][1], st[u][c][1]));
                        }
                    }
                    constexpr int TB = SL > 4 ? SL / 4 : 2;          // tokens whose sums over states are added up together
                    float v[4 * TB];
                    // the next token's rows are asked for before this one's sums are stored: no load waits behind a store
                    float4 dx_n = sm.dx[buf][tb + KEEP - 1][pair], b_n = sm.b[buf][tb + KEEP - 1][s], c_n = sm.c[buf][tb + KEEP - 1][s];
                    float2 dy_n = sm.dy[buf][tb + KEEP - 1][pair];
#pragma unroll
                    for (int u = KEEP - 1; u >= 0; --u) {
                        const float4 dx = dx_n, b = b_n, cc = c_n;
                        const float2 dy = dy_n;
                        if (u > 0) {
                            dx_n = sm.dx[buf][tb + u - 1][pair];
                            b_n = sm.b[buf][tb + u - 1][s];
                            c_n = sm.c[buf][tb + u - 1][s];
                            dy_n = sm.dy[buf][tb + u - 1][pair];
                        }
                        float2 dB0 = make_float2(0.f, 0.f), dB1 = dB0, dC0 = dB0, dC1 = dB0;
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            const float2 d = splat2(c ? dx.y : dx.x), p = splat2(c ? dx.w : dx.z), o = splat2(c ? dy.y : dy.x);
                            const float2 g0 = fma2(o, make_float2(cc.x, cc.y), gh[c][0]), g1 = fma2(o, make_float2(cc.z, cc.w), gh[c][1]);
                            dC0 = c ? fma2(o, st[u + 1][c][0], dC0) : mul2(o, st[u + 1][c][0]);
                            dC1 = c ? fma2(o, st[u + 1][c][1], dC1) : mul2(o, st[u + 1][c][1]);
                            dB0 = c ? fma2(g0, p, dB0) : mul2(g0, p);
                            dB1 = c ? fma2(g1, p, dB1) : mul2(g1, p);
                            const float2 s1 = fma2(g1, make_float2(b.z, b.w), mul2(g0, make_float2(b.x, b.y)));
                            gh[c][0] = mul2(av[u][c][0], g0);
                            gh[c][1] = mul2(av[u][c][1], g1);
                            const float2 w0 = mul2(gh[c][0], st[u][c][0]), w1 = mul2(gh[c][1], st[u][c][1]);
                            const float2 s2 = fma2(w1, A2[c][1], mul2(w0, A2[c][0]));
                            dA[c][0] = fma2(w0, d, dA[c][0]);
                            dA[c][1] = fma2(w1, d, dA[c][1]);
                            v[4 * (u % TB) + 2 * c] = s1.x + s1.y;
                            v[4 * (u % TB) + 2 * c + 1] = s2.x + s2.y;
                        }
                        if (u % TB == 0) {                           // values: (token, channel, which sum)
                            float r[4 * TB];
#pragma unroll
                            for (int k = 0; k < 4 * TB; ++k) r[k] = v[k];
                            sel_reduce<4 * TB, SL>(r, lane, CL);
                            constexpr int LEFT = 4 * TB / SL;        // values that each lane is left with
                            const int tok = s * LEFT / 4, at = s * LEFT % 4;
                            float* to = reinterpret_cast<float*>(&sm.sums[buf][tb + u + tok][pair]) + at;
                            if constexpr (LEFT == 4) *reinterpret_cast<float4*>(to) = make_float4(r[0], r[1], r[2], r[3]);
                            else if constexpr (LEFT == 2) *reinterpret_cast<float2*>(to) = make_float2(r[0], r[1]);
                            else *to = r[0];
                        }
                        float r[8] = {dB0.x, dB0.y, dB1.x, dB1.y, dC0.x, dC0.y, dC1.x, dC1.y};
                        sel_reduce<8, CL>(r, lane, 1);
                        if constexpr (CL >= 8) {
                            constexpr int REP = CL / 8;          // lanes left with the same value
                            if (REP == 1 || cl % REP == 0) {
                                const int id = cl / REP;
                                sm.bc[buf][warp][tb + u][(id >> 2) * SP + n0 + (id & 3)] = r[0];
                            }
                        } else {
                            constexpr int LEFT = 8 / CL;         // neighbours
                            const int id = cl * LEFT;
                            float* to = &sm.bc[buf][warp][tb + u][(id >> 2) * SP + n0 + (id & 3)];
                            if constexpr (LEFT == 4) *reinterpret_cast<float4*>(to) = make_float4(r[0], r[1], r[2], r[3]);
                            else *reinterpret_cast<float2*>(to) = make_float2(r[0], r[1]);
                        }
                    }
                }
            }
            sel_bwd_barrier();
        }
        sel_wait<0>();
        if (own) {
            if constexpr (STATE_ONLY) {
                const size_t at = (size_t)(it.slot0 + it.seg) * a.D + dc;
#pragma unroll
                for (int c = 0; c < 2; ++c)
                    *reinterpret_cast<float4*>(a.seg_state + (at + c) * SP + n0) = make_float4(gh[c][0].x, gh[c][0].y, gh[c][1].x, gh[c][1].y);
                if (s == 0) *reinterpret_cast<float2*>(a.seg_dt + at) = sum_dt;
            } else if (a.dh0 && it.seg == 0) {
#pragma unroll
                for (int c = 0; c < 2; ++c) sel_store4(a.dh0 + ((size_t)it.seq * a.D + dc + c) * a.S, n0, a.S, gh[c]);
            }
        }
    }
    // Not before: what follows in the stream would take places beside CTAs that run for long, and leave other SMs empty.
    pdl_launch_dependents();
    if constexpr (!STATE_ONLY) {
        sel_bwd_barrier();
        if (own) {
#pragma unroll
            for (int c = 0; c < 2; ++c)
                *reinterpret_cast<float4*>(a.part_A + ((size_t)row * a.D + dc + c) * SP + n0) = make_float4(dA[c][0].x, dA[c][0].y, dA[c][1].x, dA[c][1].y);
        }
    }
}

// ---- the shares added up: dB and dC (four threads per token row, group and four states, one after the other's part of the shares), then dA,
//      dskip, dbias (one thread per value) ----
template <typename T>
__global__ void __launch_bounds__(256) kda_selective_scan_sum_kernel(const SelScanArgs a, const int tiles_per_group, const int SP, const unsigned bc_blocks) {
    __shared__ float4 part[3][64];
    pdl_launch_dependents();
    pdl_wait();
    if (blockIdx.x < bc_blocks) {
        const int me = threadIdx.x & 63, quarter = threadIdx.x >> 6, per = (tiles_per_group + 3) / 4;
        const long long i = (long long)blockIdx.x * 64 + me, quads = SP / 2, rg = i / quads;
        const int q = (int)(i - rg * quads), isC = q >= SP / 4, n = 4 * (q % (SP / 4));
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
        if (rg < a.rows * a.G && (!a.cu_seqlens || rg / a.G < a.total_tokens)) {       // rows past the packed tokens have zero gradients
#pragma unroll 8
            for (int k = quarter * per; k < min(tiles_per_group, (quarter + 1) * per); ++k) {
                const float4 r = *reinterpret_cast<const float4*>(a.part_bc + ((size_t)k * a.rows * a.G + rg) * (2 * SP) + 4 * q);
                sum.x += r.x; sum.y += r.y; sum.z += r.z; sum.w += r.w;
            }
        }
        if (quarter) part[quarter - 1][me] = sum;
        __syncthreads();
        if (quarter || rg >= a.rows * a.G) return;
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            const float4 r = part[k][me];
            sum.x += r.x; sum.y += r.y; sum.z += r.z; sum.w += r.w;
        }
        T* to = static_cast<T*>(isC ? a.dCm : a.dBm) + rg * a.S;
        const float f[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (n + k < a.S) {
                if constexpr (sizeof(T) == 4) to[n + k] = f[k];
                else to[n + k] = __float2bfloat16_rn(f[k]);
            }
        }
    } else {
        const long long i = (long long)(blockIdx.x - bc_blocks) * 256 + threadIdx.x, nA = (long long)a.D * SP;
        const float* from = i < nA ? a.part_A + i : i < nA + a.D ? a.part_skip + (i - nA) : a.part_bias + (i - nA - a.D);
        const long long stride = i < nA ? nA : a.D;
        if (i >= nA + 2LL * a.D) return;
        if ((i >= nA && i < nA + a.D && !a.dskip) || (i >= nA + a.D && !a.dbias)) return;
        float sum = 0.f;
#pragma unroll 8
        for (int k = 0; k < a.cta_rows; ++k) sum += from[k * stride];
        if (i < nA) {
            const int n = (int)(i % SP);
            if (n < a.S) a.dA[i / SP * a.S + n] = sum;
        } else if (i < nA + a.D) a.dskip[i - nA] = sum;
        else a.dbias[i - nA - a.D] = sum;
    }
}

template <int SL, typename T>
static int launch_sel_bwd(const SelScanArgs& a, cudaStream_t stream) {
    using G = SelShape<SL>;
    const int tpg = (a.D / a.G + G::CH - 1) / G::CH;
    const long long items = sel_items(a);
    const long long blocks = (long long)a.cta_rows * tpg * a.G;
    if (blocks <= 0 || blocks > 0x7fffffffLL) return -1;
    static_assert(sizeof(SelBwdSmem<SL, T>) <= 227 * 1024, "");
    constexpr int smem = sizeof(SelBwdSmem<SL, T>);
    static std::atomic<unsigned long long> done[2];
    if (a.seg_chunks) {
        if (const cudaError_t e = allow_smem(kda_selective_scan_bwd_kernel<SL, T, true>, smem, done[1]); e != cudaSuccess) return (int)launched(e);
        if (const cudaError_t e = sel_launch(sel_long(a), kda_selective_scan_bwd_kernel<SL, T, true>, blocks, SEL_BWD_THREADS, smem, stream, a, tpg, items);
            e != cudaSuccess)
            return (int)e;
    }
    if (const cudaError_t e = allow_smem(kda_selective_scan_bwd_kernel<SL, T, false>, smem, done[0]); e != cudaSuccess) return (int)launched(e);
    // the scanning warps would wait for ever for registers that the block was not launched with
    static const bool enough = [] {
        cudaFuncAttributes f{};
        return cudaFuncGetAttributes(&f, kda_selective_scan_bwd_kernel<SL, T, false>) == cudaSuccess && 2 * f.numRegs >= SEL_SCAN_REGS + SEL_SERVE_REGS;
    }();
    if (!enough) return (int)cudaErrorLaunchOutOfResources;
    if (const cudaError_t e = sel_launch(sel_long(a), kda_selective_scan_bwd_kernel<SL, T, false>, blocks, SEL_BWD_THREADS, smem, stream, a, tpg, items);
        e != cudaSuccess)
        return (int)e;
    const long long bc_blocks = (a.rows * a.G * (G::SP / 2) + 63) / 64, rest = ((long long)a.D * (G::SP + 2) + 255) / 256;
    if (bc_blocks + rest > 0x7fffffffLL) return -1;
    return (int)launch_early(kda_selective_scan_sum_kernel<T>, dim3((unsigned)(bc_blocks + rest)), 256, 0, stream, a, tpg, G::SP, (unsigned)bc_blocks);
}

}  // namespace kda

// what a caller has to provide for part_bc: channel tiles per group
extern "C" int kda_selective_scan_tiles(int D, int groups, int state_lanes) {
    const int ch = 256 / state_lanes;
    return (D / groups + ch - 1) / ch;
}

extern "C" int kda_launch_selective_scan_bwd(const kda::SelScanArgs* a, int state_lanes, cudaStream_t stream) {
    using namespace kda;
    switch (state_lanes) {
        case 2: return a->fp32 ? launch_sel_bwd<2, float>(*a, stream) : launch_sel_bwd<2, __nv_bfloat16>(*a, stream);
        case 4: return a->fp32 ? launch_sel_bwd<4, float>(*a, stream) : launch_sel_bwd<4, __nv_bfloat16>(*a, stream);
        case 8: return a->fp32 ? launch_sel_bwd<8, float>(*a, stream) : launch_sel_bwd<8, __nv_bfloat16>(*a, stream);
        case 16: return a->fp32 ? launch_sel_bwd<16, float>(*a, stream) : launch_sel_bwd<16, __nv_bfloat16>(*a, stream);
    }
    return -1;
}
