// Single tokens of a selective state space block against pools that are updated in place:
//   selective scan:     h <- exp(dt A) h + dt x B,   y = (sum_n C[n] h[n] + skip x) silu(z)        [D, S] fp32 states per slot
//   short convolution:  window <- (window without its oldest, x),   y = act(sum_i w[i] window[i] + bias)        [D, W] fp32 per slot
// Both stream their pool rows once each way (8 S and 8 W bytes per channel against a few bytes of everything else), so they are laid out
// for wide accesses with several in flight per thread. Negative slots skip a row (zero output, no access to the pool); slots past the
// pool do the same and are reported.
#include "kda_common.cuh"
#include "kda_params.h"

namespace kda {

constexpr int STEP_THREADS = 128;

template <typename T> __device__ __forceinline__ float step_load(const T* p);
template <> __device__ __forceinline__ float step_load<float>(const float* p) { return *p; }
template <> __device__ __forceinline__ float step_load<__nv_bfloat16>(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void step_store(float* p, float v) { *p = v; }
__device__ __forceinline__ void step_store(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ float4 step_load4(const float* p) { return *reinterpret_cast<const float4*>(p); }
__device__ __forceinline__ float4 step_load4(const __nv_bfloat16* p) {
    const uint2 r = *reinterpret_cast<const uint2*>(p);
    const float2 a = unpack_bf16(r.x), b = unpack_bf16(r.y);
    return make_float4(a.x, a.y, b.x, b.y);
}
template <typename T>
__device__ __forceinline__ float4 step_four(const T* row, int n, int S, int vec) {
    if (vec) return n < S ? step_load4(row + n) : make_float4(0.f, 0.f, 0.f, 0.f);
    float4 r;
    r.x = n < S ? step_load(row + n) : 0.f;
    r.y = n + 1 < S ? step_load(row + n + 1) : 0.f;
    r.z = n + 2 < S ? step_load(row + n + 2) : 0.f;
    r.w = n + 3 < S ? step_load(row + n + 3) : 0.f;
    return r;
}
// the pool slot of a row, or -1
__device__ __forceinline__ int step_slot(const int* indices, int row, int pool, int* status) {
    if (!indices) return row;
    const int slot = indices[row];
    if (slot >= pool) {
        if (threadIdx.x == 0) report_status(status, STATUS_BAD_INDEX);
        return -1;
    }
    return slot;
}

// SL lanes (four states each) share a channel; a thread does NI channels, STEP_THREADS / SL apart, whose states are all asked for first
template <int SL, int NI, typename T>
__global__ void __launch_bounds__(STEP_THREADS) kda_selective_step_kernel(const SelStepArgs a, const int tiles) {
    constexpr int CH = STEP_THREADS / SL;
    const int row = blockIdx.x / tiles, d0 = (blockIdx.x % tiles) * (CH * NI) + threadIdx.x / SL, n0 = 4 * (threadIdx.x % SL);
    pdl_launch_dependents();
    pdl_wait();
    const int slot = step_slot(a.indices, row, a.pool, a.status);
    T* y = static_cast<T*>(a.y) + (size_t)row * a.D;
    if (slot < 0) {
        for (int i = 0; i < NI; ++i) {
            const int d = d0 + i * CH;
            if (d < a.D && n0 == 0) step_store(y + d, 0.f);
        }
        return;
    }
    float* st = a.state + (size_t)slot * a.D * a.S;
    const int per_group = a.D / a.G;
    float4 h[NI], A[NI], B[NI], C[NI];
    float x[NI], dt[NI], z[NI], skip[NI];
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        const int d = min(d0 + i * CH, a.D - 1), g = d / per_group;      // clamped: surplus channels are not stored
        h[i] = step_four(st + (size_t)d * a.S, n0, a.S, a.vec);
        x[i] = step_load(static_cast<const T*>(a.x) + row * a.x_row + d);
        dt[i] = step_load(static_cast<const T*>(a.dt) + row * a.dt_row + d) + (a.dt_bias ? a.dt_bias[d] : 0.f);
        z[i] = a.z ? step_load(static_cast<const T*>(a.z) + row * a.z_row + d) : 0.f;
        skip[i] = a.skip ? a.skip[d] : 0.f;
        A[i] = step_four(a.A + (size_t)d * a.S, n0, a.S, a.vec);
        B[i] = step_four(static_cast<const T*>(a.Bm) + row * a.b_row + g * a.S, n0, a.S, a.vec);
        C[i] = step_four(static_cast<const T*>(a.Cm) + row * a.c_row + g * a.S, n0, a.S, a.vec);
    }
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        const int d = d0 + i * CH;
        const float step = a.softplus ? softplus2(splat2(dt[i])).x : dt[i], p = step * x[i], s2 = step * RCP_LN2;
        h[i].x = fmaf(fast_exp2(s2 * A[i].x), h[i].x, p * B[i].x);
        h[i].y = fmaf(fast_exp2(s2 * A[i].y), h[i].y, p * B[i].y);
        h[i].z = fmaf(fast_exp2(s2 * A[i].z), h[i].z, p * B[i].z);
        h[i].w = fmaf(fast_exp2(s2 * A[i].w), h[i].w, p * B[i].w);
        float o = fmaf(h[i].x, C[i].x, h[i].y * C[i].y) + fmaf(h[i].z, C[i].z, h[i].w * C[i].w);
#pragma unroll
        for (int m = SL / 2; m; m >>= 1) o += __shfl_xor_sync(0xffffffffu, o, m);
        if (d >= a.D) continue;
        float* to = st + (size_t)d * a.S + n0;
        if (a.vec) {
            if (n0 < a.S) *reinterpret_cast<float4*>(to) = h[i];
        } else {
            const float f[4] = {h[i].x, h[i].y, h[i].z, h[i].w};
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (n0 + k < a.S) to[k] = f[k];
        }
        if (n0 == 0) {
            o = fmaf(skip[i], x[i], o);
            if (a.z) o = o * z[i] * fast_rcp(1.f + fast_exp2(-RCP_LN2 * z[i]));
            step_store(y + d, o);
        }
    }
}

// two channels per thread and place, NI places STEP_THREADS pairs apart
template <int W, int NI>
__global__ void __launch_bounds__(STEP_THREADS) kda_conv_step_kernel(const ConvStepArgs a, const int tiles) {
    const int row = blockIdx.x / tiles, d0 = 2 * ((blockIdx.x % tiles) * (STEP_THREADS * NI) + threadIdx.x);
    pdl_launch_dependents();
    pdl_wait();
    const int slot = step_slot(a.indices, row, a.pool, a.status);
    __nv_bfloat16* y = static_cast<__nv_bfloat16*>(a.y) + (size_t)row * a.D;
    if (slot < 0) {
        for (int i = 0; i < NI; ++i) {
            const int d = d0 + 2 * STEP_THREADS * i;
            if (d < a.D) *reinterpret_cast<uint32_t*>(y + d) = 0u;
        }
        return;
    }
    float* cache = a.cache + (size_t)slot * a.D * W;
    float win[NI][2][W], w[NI][2][W];
    float2 x[NI], b[NI];
    auto load = [&](const float* p, float (&v)[2][W]) {
        if constexpr (W % 2 == 0) {
#pragma unroll
            for (int q = 0; q < 2 * W / 4; ++q) {
                const float4 r = reinterpret_cast<const float4*>(p)[q];
                v[4 * q / W][4 * q % W] = r.x;
                v[(4 * q + 1) / W][(4 * q + 1) % W] = r.y;
                v[(4 * q + 2) / W][(4 * q + 2) % W] = r.z;
                v[(4 * q + 3) / W][(4 * q + 3) % W] = r.w;
            }
        } else {
#pragma unroll
            for (int q = 0; q < 2 * W; ++q) v[q / W][q % W] = p[q];
        }
    };
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        const int d = min(d0 + 2 * STEP_THREADS * i, a.D - 2);
        load(cache + (size_t)d * W, win[i]);
        load(a.w + (size_t)d * W, w[i]);
        x[i] = unpack_bf16(*reinterpret_cast<const uint32_t*>(static_cast<const __nv_bfloat16*>(a.x) + row * a.x_row + d));
        b[i] = a.bias ? make_float2(a.bias[d], a.bias[d + 1]) : make_float2(0.f, 0.f);
    }
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        const int d = d0 + 2 * STEP_THREADS * i;
        float o[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
            for (int k = 0; k + 1 < W; ++k) win[i][c][k] = win[i][c][k + 1];
            win[i][c][W - 1] = c ? x[i].y : x[i].x;
            o[c] = c ? b[i].y : b[i].x;
#pragma unroll
            for (int k = 0; k < W; ++k) o[c] = fmaf(w[i][c][k], win[i][c][k], o[c]);
            if (a.silu) o[c] = o[c] * fast_rcp(1.f + fast_exp2(-RCP_LN2 * o[c]));
        }
        if (d >= a.D) continue;
        float* to = cache + (size_t)d * W;
        if constexpr (W % 2 == 0) {
#pragma unroll
            for (int q = 0; q < 2 * W / 4; ++q)
                reinterpret_cast<float4*>(to)[q] = make_float4(win[i][4 * q / W][4 * q % W], win[i][(4 * q + 1) / W][(4 * q + 1) % W],
                                                               win[i][(4 * q + 2) / W][(4 * q + 2) % W], win[i][(4 * q + 3) / W][(4 * q + 3) % W]);
        } else {
#pragma unroll
            for (int q = 0; q < 2 * W; ++q) to[q] = win[i][q / W][q % W];
        }
        *reinterpret_cast<uint32_t*>(y + d) = pack_bf16(o[0], o[1]);
    }
}

template <int SL, typename T>
static int launch_sel_step(const SelStepArgs& a, cudaStream_t stream) {
    constexpr int CH = STEP_THREADS / SL;
    // four channels per thread where that leaves a block for every place of the GPU, one where blocks are few
    const bool many = (long long)a.rows * ((a.D + 4 * CH - 1) / (4 * CH)) >= 4LL * sm_count();
    const int tiles = (a.D + CH * (many ? 4 : 1) - 1) / (CH * (many ? 4 : 1));
    const long long blocks = (long long)a.rows * tiles;
    if (blocks > 0x7fffffffLL) return -1;
    return (int)launch_early(many ? kda_selective_step_kernel<SL, 4, T> : kda_selective_step_kernel<SL, 1, T>, dim3((unsigned)blocks), STEP_THREADS, 0,
                             stream, a, tiles);
}

}  // namespace kda

extern "C" int kda_launch_selective_step(const kda::SelStepArgs* a, cudaStream_t stream) {
    using namespace kda;
    if (a->rows == 0) return 0;
#define KDA_STEP(SL) return a->fp32 ? launch_sel_step<SL, float>(*a, stream) : launch_sel_step<SL, __nv_bfloat16>(*a, stream)
    if (a->S <= 4) KDA_STEP(1);
    if (a->S <= 8) KDA_STEP(2);
    if (a->S <= 16) KDA_STEP(4);
    if (a->S <= 32) KDA_STEP(8);
    if (a->S <= 64) KDA_STEP(16);
#undef KDA_STEP
    return -1;
}

extern "C" int kda_launch_conv_step(const kda::ConvStepArgs* a, cudaStream_t stream) {
    using namespace kda;
    if (a->rows == 0) return 0;
    const int pairs = a->D / 2;
    const bool many = (long long)a->rows * ((pairs + 2 * STEP_THREADS - 1) / (2 * STEP_THREADS)) >= 4LL * sm_count();
    const int per = STEP_THREADS * (many ? 2 : 1), tiles = (pairs + per - 1) / per;
    const long long blocks = (long long)a->rows * tiles;
    if (blocks > 0x7fffffffLL) return -1;
    void (*kernel)(const ConvStepArgs, const int) = nullptr;
    switch (a->W) {
        case 1: kernel = many ? kda_conv_step_kernel<1, 2> : kda_conv_step_kernel<1, 1>; break;
        case 2: kernel = many ? kda_conv_step_kernel<2, 2> : kda_conv_step_kernel<2, 1>; break;
        case 3: kernel = many ? kda_conv_step_kernel<3, 2> : kda_conv_step_kernel<3, 1>; break;
        case 4: kernel = many ? kda_conv_step_kernel<4, 2> : kda_conv_step_kernel<4, 1>; break;
        default: return -1;
    }
    return (int)launch_early(kernel, dim3((unsigned)blocks), STEP_THREADS, 0, stream, *a, tiles);
}
