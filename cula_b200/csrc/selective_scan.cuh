// Shared by the forward and the backward kernel of the selective scan: how states and channels lie over a warp, the work items (a
// sequence or a segment of one, times a tile of channels), and the staging of token rows.
//
//     h_t = exp(dt_t A) h_{t-1} + dt_t x_t B_t     (per channel d and state n; dt_t = softplus(raw_t + bias))
//     y_t = sum_n C_t[n] h_t[n] + skip x_t,   out_t = y_t silu(z_t)
//
// A thread holds two channels times four states; SL lanes share the states of a channel (SP = 4 SL of them, the ones past S are zero),
// CL = 32 / SL lanes stand side by side over channels. The lanes of one state quad are neighbours, since a 16-byte shared load whose
// neighbouring lanes ask for the same address takes 2.3 cycles of the SM instead of 4. Lane cl of warp w has channels 8 cl + 2 w and the
// next: what one thread stages, a piece of 8 channels, is a pair for each warp, and both sides touch shared memory in order.
#pragma once
#include <cfloat>

#include "kda_common.cuh"
#include "kda_params.h"

namespace kda {

constexpr int SEL_THREADS = 128, SEL_WARPS = SEL_THREADS / 32;
constexpr int SEL_KEEP = 8;                    // a state is kept for the backward pass before every eighth token

template <int SL_>
struct SelShape {
    static constexpr int SL = SL_, SP = 4 * SL;                     // lanes over states, padded states
    static constexpr int CL = 32 / SL, CW = 2 * CL, CH = SEL_WARPS * CW;      // lanes over channels, channels of a warp, of a CTA
    static constexpr int LC = SL == 2 ? 8 : 16;                     // tokens staged at a time (a divisor of 64)
    static constexpr int VECS = CH / 8;                             // 8-channel pieces of a token row
    static constexpr int ITEMS = LC * VECS;                         // pieces of a staged tile: one per thread, or fewer
    static constexpr int UNITS = LC * SL, UB = (UNITS + SEL_THREADS - 1) / SEL_THREADS;       // 4-state pieces of its B (or C) rows
    static_assert(ITEMS <= SEL_THREADS && BT % LC == 0 && LC % SEL_KEEP == 0, "");
};

// A segment of a sequence: tokens [t0, t1) of `len`, counted inside the sequence. There are sel_items() numbers for them.
inline long long sel_items(const SelScanArgs& a) {
    const long long cps = (a.T + BT - 1) / BT, K = a.seg_chunks;
    if (!K) return a.n_seqs;
    return a.cu_seqlens ? a.num_chunks / K + a.n_seqs : a.n_seqs * ((cps + K - 1) / K);
}
struct SelItem {
    int seq, t0, t1, len, seg, segs;
    long long slot0;              // of its sequence's first segment
    long long chunk0;             // its sequence's first chunk
    long long row0;               // its sequence's first row in the contiguous tensors
};
__device__ __forceinline__ bool sel_item(const SelScanArgs& a, long long i, SelItem& it) {
    const int K = a.seg_chunks;
    if (!a.cu_seqlens) {
        const int cps = (a.T + BT - 1) / BT, segs = K ? (cps + K - 1) / K : 1;
        it.seq = (int)(i / segs);
        it.seg = (int)(i - (long long)it.seq * segs);
        it.segs = segs;
        it.len = a.T;
        it.slot0 = (long long)it.seq * segs;
        it.chunk0 = (long long)it.seq * cps;
        it.row0 = (long long)it.seq * a.T;
    } else {
        // Segments of a packed batch are numbered chunk_offsets[seq] / K + seq + seg: one more per sequence keeps those of all of them
        // apart, at the price of at most one number per sequence that stands for none.
        int lo = 0;
        if (!K) lo = a.seq_order[i];
        else
            for (int hi = a.n_seqs; hi - lo > 1;) {
                const int mid = (lo + hi) >> 1;
                if (a.chunk_offsets[mid] / K + mid <= i) lo = mid;
                else hi = mid;
            }
        it.seq = lo;
        it.chunk0 = a.chunk_offsets[lo];
        it.slot0 = K ? it.chunk0 / K + lo : lo;
        const int bos = a.cu_seqlens[lo];
        it.len = a.cu_seqlens[lo + 1] - bos;
        const int cps = (it.len + BT - 1) / BT;
        it.segs = K ? max(1, (cps + K - 1) / K) : 1;
        it.seg = K ? (int)(i - it.slot0) : 0;
        if (it.seg >= it.segs) return false;
        it.row0 = bos;
    }
    it.t0 = K ? it.seg * K * BT : 0;
    it.t1 = K ? min(it.len, it.t0 + K * BT) : it.len;
    return true;
}

// ---- 8 channels of a token row ----
template <typename T> struct SelVec;
template <> struct SelVec<__nv_bfloat16> {
    static constexpr int Q = 1;                                     // 16-byte pieces
    __device__ static void unpack(const uint4* p, int step, float2 (&v)[4]) {
        const uint4 r = p[0];
        v[0] = unpack_bf16(r.x); v[1] = unpack_bf16(r.y); v[2] = unpack_bf16(r.z); v[3] = unpack_bf16(r.w);
    }
    __device__ static void store(__nv_bfloat16* p, const float2 (&v)[4]) {
        *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16(v[0].x, v[0].y), pack_bf16(v[1].x, v[1].y), pack_bf16(v[2].x, v[2].y), pack_bf16(v[3].x, v[3].y));
    }
    __device__ static float4 four(const __nv_bfloat16* p) {
        const uint2 r = *reinterpret_cast<const uint2*>(p);
        const float2 a = unpack_bf16(r.x), b = unpack_bf16(r.y);
        return make_float4(a.x, a.y, b.x, b.y);
    }
};
template <> struct SelVec<float> {
    static constexpr int Q = 2;
    __device__ static void unpack(const uint4* p, int step, float2 (&v)[4]) {
        const float4 r = *reinterpret_cast<const float4*>(p), s = *reinterpret_cast<const float4*>(p + step);
        v[0] = make_float2(r.x, r.y); v[1] = make_float2(r.z, r.w); v[2] = make_float2(s.x, s.y); v[3] = make_float2(s.z, s.w);
    }
    __device__ static void store(float* p, const float2 (&v)[4]) {
        reinterpret_cast<float4*>(p)[0] = make_float4(v[0].x, v[0].y, v[1].x, v[1].y);
        reinterpret_cast<float4*>(p)[1] = make_float4(v[2].x, v[2].y, v[3].x, v[3].y);
    }
    __device__ static float4 four(const float* p) { return *reinterpret_cast<const float4*>(p); }
};
// Each thread copies the pieces that it will use itself, so their arrival concerns no other thread.
__device__ __forceinline__ void sel_copy16(void* dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" :: "r"(smem_u32(dst)), "l"(src) : "memory");
}
template <int BYTES>
__device__ __forceinline__ void sel_copy(void* dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" :: "r"(smem_u32(dst)), "l"(src), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void sel_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void sel_wait() { asm volatile("cp.async.wait_group %0;" :: "n"(N) : "memory"); }

// Four states of a B or C row, as they are, into the thread's own place: one copy where rows allow it, else element by element (zeros past
// the last of S).
template <typename T>
__device__ __forceinline__ void sel_fetch4(T* to, const T* row, int n, int S, int vec) {
    if (vec && n + 3 < S) sel_copy<4 * sizeof(T)>(to, row + n);
    else {
#pragma unroll
        for (int k = 0; k < 4; ++k) to[k] = n + k < S ? row[n + k] : T(0.f);
    }
}
// Where the states that are kept for the backward pass stand: a thread's two times four of them as two 16-byte pieces, those of a warp in
// order. Returned is the first piece of lane 0 of a CTA's warp 0; pieces follow as [warp][channel of two][lane].
template <int SL>
__device__ __forceinline__ float4* sel_kept(const SelScanArgs& a, long long chunk0, int t, int tile, int tiles) {
    return reinterpret_cast<float4*>(a.states) + ((size_t)(chunk0 * (BT / SEL_KEEP) + t / SEL_KEEP) * tiles + tile) * (SEL_WARPS * 2 * 32);
}
// four states of a [.., S] fp32 row
__device__ __forceinline__ void sel_load4(const float* row, int n, int S, float2 (&v)[2]) {
    float f[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) f[k] = n + k < S ? row[n + k] : 0.f;
    v[0] = make_float2(f[0], f[1]); v[1] = make_float2(f[2], f[3]);
}
// four rates, for exponents of two. One of minus infinity is held as the lowest number: tokens past the end of a tile have steps of zero, which
// change no state, while zero times infinity would
__device__ __forceinline__ void sel_load_rates(const float* row, int n, int S, float2 (&v)[2]) {
    float f[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float r = n + k < S ? row[n + k] * RCP_LN2 : 0.f;
        f[k] = r == -INFINITY ? -FLT_MAX : r;
    }
    v[0] = make_float2(f[0], f[1]); v[1] = make_float2(f[2], f[3]);
}
__device__ __forceinline__ void sel_store4(float* row, int n, int S, const float2 (&v)[2]) {
    const float f[4] = {v[0].x, v[0].y, v[1].x, v[1].y};
#pragma unroll
    for (int k = 0; k < 4; ++k)
        if (n + k < S) row[n + k] = f[k];
}

// softplus(x) = max(x, 0) + log1p(e), e = exp(-|x|), with log1p(e) = e q(e): q by Remez exchange for the least relative error on [0, 1]
// (4.7e-9 before rounding, 1.7e-7 in fp32 arithmetic). One exponential and no reciprocal: the exponentials' unit bounds the scan.
__device__ __forceinline__ float2 sel_softplus2(float2 x) {
    const float2 e = ex2_2(make_float2(-RCP_LN2 * fabsf(x.x), -RCP_LN2 * fabsf(x.y)));
    float2 q = fma2(e, splat2(-0.00324402517f), splat2(0.0198514629f));
    q = fma2(e, q, splat2(-0.0569595359f));
    q = fma2(e, q, splat2(0.106036551f));
    q = fma2(e, q, splat2(-0.153055921f));
    q = fma2(e, q, splat2(0.196759388f));
    q = fma2(e, q, splat2(-0.249541342f));
    q = fma2(e, q, splat2(0.333299637f));
    q = fma2(e, q, splat2(-0.499999017f));
    q = fma2(e, q, splat2(1.f));
    return fma2(e, q, make_float2(fmaxf(x.x, 0.f), fmaxf(x.y, 0.f)));
}
__device__ __forceinline__ float2 sel_sigmoid2(float2 x) {
    return make_float2(fast_rcp(1.f + fast_exp2(-RCP_LN2 * x.x)), fast_rcp(1.f + fast_exp2(-RCP_LN2 * x.y)));
}

// Sums of V values over the N lanes whose numbers differ in the bits from `low` up, each lane left with V / N of them (one where N > V):
// half of the values are handed over per step instead of all of them. Value i ends with the lane (of those N) number i / (V / N).
template <int V, int N>
__device__ __forceinline__ void sel_reduce(float (&v)[V], int lane, int low) {
    if constexpr (N > 1) {
        const bool up = lane & (low * (N / 2));
        if constexpr (V > 1) {
            float w[V / 2];
#pragma unroll
            for (int i = 0; i < V / 2; ++i) {
                const float give = up ? v[i] : v[i + V / 2], keep = up ? v[i + V / 2] : v[i];
                w[i] = keep + __shfl_xor_sync(0xffffffffu, give, low * (N / 2));
            }
            sel_reduce<V / 2, N / 2>(w, lane, low);
#pragma unroll
            for (int i = 0; i < V / 2; ++i) v[i] = w[i];
        } else {
            v[0] += __shfl_xor_sync(0xffffffffu, v[0], low * (N / 2));
            sel_reduce<1, N / 2>(v, lane, low);
        }
    }
}

// Long scans are not launched while the kernel before them drains: their CTAs would stand two to an SM wherever that one's had gone first,
// and leave other SMs empty for all of their time (128 CTAs of 4096 tokens: 429 us that way, 263 this way).
inline bool sel_long(const SelScanArgs& a) { return (a.seg_chunks ? a.seg_chunks : a.num_chunks / max(1, a.n_seqs)) >= 8; }
template <typename... P, typename... A>
inline cudaError_t sel_launch(bool whole, void (*kernel)(P...), long long blocks, int threads, int smem, cudaStream_t stream, const A&... args) {
    if (!whole) return launch_early(kernel, dim3((unsigned)blocks), threads, smem, stream, args...);
    kernel<<<dim3((unsigned)blocks), threads, smem, stream>>>(static_cast<P>(args)...);
    return launched(cudaGetLastError());
}

}  // namespace kda
