// Single tokens of a selective state space block against pools that are updated in place:
//   selective scan:     h <- exp(dt A) h + dt x B,   y = (sum_n C[n] h[n] + skip x) silu(z)        [D, S] fp32 states per slot
//   short convolution:  window <- (window without its oldest, x),   y = act(sum_i w[i] window[i] + bias)        [D, W] fp32 per slot
// Both stream their pool rows once each way (8 S and 8 W bytes per channel against a few bytes of everything else). A warp keeps its
// channels, with their parameters in registers, and walks the rows of the batch, asking for the next row's states before it works on this
// one's. Negative slots skip a row (zero output, no access to the pool); slots past the pool do the same and are reported.
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
// Values as they are, to be converted when they are needed: whatever is done to them where they are loaded, taking a word apart among it,
// waits for the load (256 rows x 4096 channels x 8 states in bf16: 27 us so, 20 without)
__device__ __forceinline__ uint32_t step_raw(const float* p) { return *reinterpret_cast<const uint32_t*>(p); }
__device__ __forceinline__ uint32_t step_raw(const __nv_bfloat16* p) { return *reinterpret_cast<const unsigned short*>(p); }
template <typename T> __device__ __forceinline__ float step_value(uint32_t r) { return __uint_as_float(sizeof(T) == 2 ? r << 16 : r); }
template <typename T> struct Raw4 {                                 // four values: two words of bf16, four of fp32
    uint32_t v[sizeof(T)];
    __device__ __forceinline__ void load(const T* row, int n, int S, int vec) {
        if constexpr (sizeof(T) == 2) {
            if (vec) {
                const uint2 r = n < S ? *reinterpret_cast<const uint2*>(row + n) : make_uint2(0u, 0u);
                v[0] = r.x; v[1] = r.y;
            } else {
#pragma unroll
                for (int k = 0; k < 2; ++k)
                    v[k] = (n + 2 * k < S ? step_raw(row + n + 2 * k) : 0u) | (n + 2 * k + 1 < S ? step_raw(row + n + 2 * k + 1) : 0u) << 16;
            }
        } else if (vec) {
            const uint4 r = n < S ? *reinterpret_cast<const uint4*>(row + n) : make_uint4(0u, 0u, 0u, 0u);
            v[0] = r.x; v[1] = r.y; v[2] = r.z; v[3] = r.w;
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = n + k < S ? step_raw(row + n + k) : 0u;
        }
    }
    __device__ __forceinline__ float4 get() const {
        if constexpr (sizeof(T) == 2) {
            const float2 a = unpack_bf16(v[0]), b = unpack_bf16(v[1]);
            return make_float4(a.x, a.y, b.x, b.y);
        } else return make_float4(__uint_as_float(v[0]), __uint_as_float(v[1]), __uint_as_float(v[2]), __uint_as_float(v[3]));
    }
};
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

// SL lanes (four states each) share a channel, NI channels a lane: channel c of lane (g, s) is the warp's c (32 / SL) + g. What concerns a
// channel as a whole (step, gate, output) is done by one lane, its owner, and handed to the others. The next row's states are on their way to
// shared memory, each thread's to a place of its own, while a row is worked on; everything else is asked for one row ahead too.
// Bound by memory: 256 rows x 4096 channels x 16 states in bf16 (143 MB, 22 us at the copy rate) take 65 us with a block per row and tile
// and 28 to 29 so (5.0 TB/s, launch and ramp included; 512 rows 5.6). The next row in registers: 29.3, and 46 in the place of 28 where 64 states
// leave none. Two rows ahead: 28.6; other numbers of blocks per SM: 30 to 35.
constexpr int STEP_RING = 2;
// Blocks that an SM holds: those of few states per channel need more of them for as many bytes on their way (8 states: 23 -> 19 us)
constexpr int step_resident(int SL) { return SL == 1 ? 8 : SL == 2 ? 6 : 5; }

template <int SL, typename T>
__global__ void __launch_bounds__(STEP_THREADS, step_resident(SL)) kda_selective_step_kernel(const SelStepArgs a, const int tiles, const int row_step) {
    constexpr int CG = 32 / SL, NI = SL < 4 ? SL : 4, SHARE = SL / NI;      // SHARE: lanes that are left with a channel's sum
    __shared__ float4 ring[STEP_RING][NI][STEP_THREADS];
    const int tid = threadIdx.x, lane = tid & 31, s = lane % SL, g = lane / SL, n0 = 4 * s, c_own = s / SHARE;
    const int d0 = ((blockIdx.x % tiles) * blockDim.x + (tid & ~31)) / 32 * (CG * NI), mine = d0 + c_own * CG + g;
    const bool owner = s % SHARE == 0 && mine < a.D;
    pdl_launch_dependents();
    pdl_wait();
    const int dm = min(mine, a.D - 1), per_group = a.D / a.G;        // surplus channels are computed and not stored
    auto channel = [&](int c) { return min(d0 + c * CG + g, a.D - 1); };
    const float bias = a.dt_bias ? a.dt_bias[dm] : 0.f, skip = a.skip ? a.skip[dm] : 0.f;
    float4 A[NI];
#pragma unroll
    for (int c = 0; c < NI; ++c) A[c] = step_four(a.A + (size_t)channel(c) * a.S, n0, a.S, a.vec);
    // B and C of a row: asked for ahead where the warp's channels have one group
    const int group0 = min(d0, a.D - 1) / per_group;
    const bool one_group = group0 == min(d0 + CG * NI - 1, a.D - 1) / per_group;

    auto slot_of = [&](int r) { return r < a.rows ? step_slot(a.indices, r, a.pool, a.status) : -1; };
    auto fetch_state = [&](int k, int at) {
        if (at >= 0) {
            const float* st = a.state + (size_t)at * a.D * a.S;
#pragma unroll
            for (int c = 0; c < NI; ++c) {
                float4* to = &ring[k][c][tid];
                const float* from = st + (size_t)channel(c) * a.S;
                if (a.vec) {
                    if (n0 < a.S) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" :: "r"(smem_u32(to)), "l"(from + n0) : "memory");
                    else *to = make_float4(0.f, 0.f, 0.f, 0.f);
                } else *to = step_four(from, n0, a.S, 0);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    uint32_t raw[3];
    Raw4<T> Bn, Cn;                                                  // x, dt, z, B, C of the row to come
    auto fetch = [&](int r, int at) {
        if (at < 0) return;
        raw[0] = step_raw(static_cast<const T*>(a.x) + r * a.x_row + dm);
        raw[1] = step_raw(static_cast<const T*>(a.dt) + r * a.dt_row + dm);
        if (a.z) raw[2] = step_raw(static_cast<const T*>(a.z) + r * a.z_row + dm);
        if (one_group) {
            Bn.load(static_cast<const T*>(a.Bm) + r * a.b_row + group0 * a.S, n0, a.S, a.vec);
            Cn.load(static_cast<const T*>(a.Cm) + r * a.c_row + group0 * a.S, n0, a.S, a.vec);
        }
    };
    int row = blockIdx.x / tiles, slots[STEP_RING + 1];              // of this row and the ones to come
#pragma unroll
    for (int k = 0; k <= STEP_RING; ++k) slots[k] = slot_of(row + k * row_step);
#pragma unroll
    for (int k = 0; k < STEP_RING - 1; ++k) fetch_state(k, slots[k]);
    fetch(row, slots[0]);
    for (int k = 0; row < a.rows; row += row_step, k = k + 1 == STEP_RING ? 0 : k + 1) {
        const int at = slots[0];
        fetch_state(k == 0 ? STEP_RING - 1 : k - 1, slots[STEP_RING - 1]);
        const float4 B0 = Bn.get(), C0 = Cn.get();
        const float x = step_value<T>(raw[0]), dt = step_value<T>(raw[1]) + bias, z = a.z ? step_value<T>(raw[2]) : 0.f;
#pragma unroll
        for (int i = 0; i < STEP_RING; ++i) slots[i] = slots[i + 1];
        slots[STEP_RING] = slot_of(row + (STEP_RING + 1) * row_step);
        fetch(row + row_step, slots[0]);
        asm volatile("cp.async.wait_group %0;" :: "n"(STEP_RING - 1) : "memory");
        T* y = static_cast<T*>(a.y) + (size_t)row * a.D;
        if (at < 0) {
            if (owner) step_store(y + mine, 0.f);
            continue;
        }
        float* st = a.state + (size_t)at * a.D * a.S;
        const float step = a.softplus ? softplus2(splat2(dt)).x : dt, step2 = step * RCP_LN2, prod = step * x;
        float v[NI];
#pragma unroll
        for (int c = 0; c < NI; ++c) {
            const int d = channel(c);
            const float e = __shfl_sync(0xffffffffu, step2, g * SL + c * SHARE), p = __shfl_sync(0xffffffffu, prod, g * SL + c * SHARE);
            float4 B = B0, C = C0, h = ring[k][c][tid];
            if (!one_group) {
                const int group = d / per_group;
                B = step_four(static_cast<const T*>(a.Bm) + row * a.b_row + group * a.S, n0, a.S, a.vec);
                C = step_four(static_cast<const T*>(a.Cm) + row * a.c_row + group * a.S, n0, a.S, a.vec);
            }
            h.x = fmaf(decay(e, A[c].x), h.x, p * B.x);
            h.y = fmaf(decay(e, A[c].y), h.y, p * B.y);
            h.z = fmaf(decay(e, A[c].z), h.z, p * B.z);
            h.w = fmaf(decay(e, A[c].w), h.w, p * B.w);
            v[c] = fmaf(h.x, C.x, h.y * C.y) + fmaf(h.z, C.z, h.w * C.w);
            if (d0 + c * CG + g < a.D) {
                float* to = st + (size_t)d * a.S + n0;
                if (a.vec) {
                    if (n0 < a.S) *reinterpret_cast<float4*>(to) = h;
                } else {
                    const float f[4] = {h.x, h.y, h.z, h.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (n0 + i < a.S) to[i] = f[i];
                }
            }
        }
        // each channel's sum goes to its owner: half of a lane's sums are handed over per step
#pragma unroll
        for (int n = NI, m = SL / 2; m; m >>= 1) {
            if (n > 1) {
                n >>= 1;
#pragma unroll
                for (int i = 0; i < n; ++i) {
                    const float give = (s & m) ? v[i] : v[i + n], keep = (s & m) ? v[i + n] : v[i];
                    v[i] = keep + __shfl_xor_sync(0xffffffffu, give, m);
                }
            } else v[0] += __shfl_xor_sync(0xffffffffu, v[0], m);
        }
        if (owner) {
            float o = fmaf(skip, x, v[0]);
            if (a.z) o = o * z * fast_rcp(1.f + fast_exp2(-RCP_LN2 * z));
            step_store(y + mine, o);
        }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// two neighbouring channels per thread; 256 rows x 12288 channels x 4 (113 MB, 17.6 us at the copy rate): 20.5 us
template <int W>
__global__ void __launch_bounds__(STEP_THREADS) kda_conv_step_kernel(const ConvStepArgs a, const int tiles, const int row_step) {
    const int d0 = 2 * ((blockIdx.x % tiles) * blockDim.x + threadIdx.x);
    const bool live = d0 < a.D;
    const int d = live ? d0 : a.D - 2;
    pdl_launch_dependents();
    pdl_wait();
    auto load = [&](const float* p, float (&v)[2 * W]) {
        if constexpr (W % 2 == 0) {
#pragma unroll
            for (int q = 0; q < W / 2; ++q) {
                const float4 r = reinterpret_cast<const float4*>(p)[q];
                v[4 * q] = r.x; v[4 * q + 1] = r.y; v[4 * q + 2] = r.z; v[4 * q + 3] = r.w;
            }
        } else {
#pragma unroll
            for (int q = 0; q < 2 * W; ++q) v[q] = p[q];
        }
    };
    float w[2 * W], next[2 * W];
    load(a.w + (size_t)d * W, w);
    const float2 b = a.bias ? make_float2(a.bias[d], a.bias[d + 1]) : make_float2(0.f, 0.f);
    int row = blockIdx.x / tiles, slot = step_slot(a.indices, row, a.pool, a.status);
    int slot_next = row + row_step < a.rows ? step_slot(a.indices, row + row_step, a.pool, a.status) : -1;
    uint32_t raw = 0;
    auto fetch = [&](int r, int at) {
        if (at < 0) return;
        load(a.cache + ((size_t)at * a.D + d) * W, next);
        raw = *reinterpret_cast<const uint32_t*>(static_cast<const __nv_bfloat16*>(a.x) + r * a.x_row + d);
    };
    fetch(row, slot);
    while (row < a.rows) {
        const int r = row, at = slot;
        float win[2 * W];
        const float2 x = unpack_bf16(raw);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
            for (int k = 0; k + 1 < W; ++k) win[c * W + k] = next[c * W + k + 1];
            win[c * W + W - 1] = c ? x.y : x.x;
        }
        row += row_step;
        if (row < a.rows) {
            slot = slot_next;
            fetch(row, slot);
            if (row + row_step < a.rows) slot_next = step_slot(a.indices, row + row_step, a.pool, a.status);
        }
        uint32_t* y = reinterpret_cast<uint32_t*>(static_cast<__nv_bfloat16*>(a.y) + (size_t)r * a.D + d);
        if (at < 0) {
            if (live) *y = 0u;
            continue;
        }
        float o[2] = {b.x, b.y};
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
            for (int k = 0; k < W; ++k) o[c] = fmaf(w[c * W + k], win[c * W + k], o[c]);
            if (a.silu) o[c] = o[c] * fast_rcp(1.f + fast_exp2(-RCP_LN2 * o[c]));
        }
        if (!live) continue;
        float* to = a.cache + ((size_t)at * a.D + d) * W;
        if constexpr (W % 2 == 0) {
#pragma unroll
            for (int q = 0; q < W / 2; ++q) reinterpret_cast<float4*>(to)[q] = make_float4(win[4 * q], win[4 * q + 1], win[4 * q + 2], win[4 * q + 3]);
        } else {
#pragma unroll
            for (int q = 0; q < 2 * W; ++q) to[q] = win[q];
        }
        *y = pack_bf16(o[0], o[1]);
    }
}

// Blocks of 128 threads walk several rows each, as many blocks as the SMs hold; where rows and channels are few, blocks of a warp with one row.
struct StepGrid { int threads, tiles, row_step; };
static StepGrid step_grid(int rows, int units, int resident) {       // units: threads that a row takes
    StepGrid g;
    g.threads = (long long)rows * units >= 128LL * 2 * sm_count() ? STEP_THREADS : 32;
    g.tiles = (units + g.threads - 1) / g.threads;
    const long long most = (long long)sm_count() * resident * (STEP_THREADS / g.threads) / g.tiles;
    g.row_step = (int)(most < 1 ? 1 : most < rows ? most : rows);
    return g;
}
template <int SL, typename T>
static int launch_sel_step(const SelStepArgs& a, cudaStream_t stream) {
    constexpr int channels = 32 / SL * (SL < 4 ? SL : 4);            // of a warp
    const StepGrid g = step_grid(a.rows, (a.D + channels - 1) / channels * 32, step_resident(SL));
    return (int)launch_early(kda_selective_step_kernel<SL, T>, dim3((unsigned)(g.tiles * g.row_step)), g.threads, 0, stream, a, g.tiles, g.row_step);
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
    const StepGrid g = step_grid(a->rows, a->D / 2, 16);
    void (*kernel)(const ConvStepArgs, const int, const int) = a->W == 1 ? kda_conv_step_kernel<1> : a->W == 2 ? kda_conv_step_kernel<2>
                                                             : a->W == 3 ? kda_conv_step_kernel<3> : kda_conv_step_kernel<4>;
    return (int)launch_early(kernel, dim3((unsigned)(g.tiles * g.row_step)), g.threads, 0, stream, *a, g.tiles, g.row_step);
}
