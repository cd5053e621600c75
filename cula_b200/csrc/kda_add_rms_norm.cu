// RMS norm with the addition to the residual stream before it, forward and backward, and with an 8-bit output:
//     v = x + r, rounded to the stream's type (what the next block adds to, and what is normalised);  n = v rsqrt(mean(v^2) + eps);  y = n w
//     8 bits: per row or per group of columns, scale = max(amax|y| / 448, 2^-126), q = e4m3(y / scale)
//     dv = rstd (dn - n mean(dn n)) + dr_out with dn = dy w;  dx, dr = dv;  dw = sum over rows of dy n
// Everything is read and written once: TPR threads hold a row in registers, VPT pieces of 8 columns each, and ask for their next row before
// they sum, scale and store this one. Bound by memory: 8192 x 4096 in bf16 forward 40 us (268 MB: 6.6 TB/s), backward 44 (268 MB), 8-bit output
// beside an fp32 stream at 16384 x 4096 112 to 117 us (738 MB: 6.3 to 6.6 TB/s), the same with a scale per 128 columns.
#include <cuda_fp8.h>

#include "kda_common.cuh"
#include "kda_params.h"

namespace kda {

enum { RES_NONE = 0, RES_BF16 = 1, RES_FP32 = 2 };
constexpr float E4M3_MAX = 448.f, SCALE_MIN = 1.17549435e-38f;

template <typename T> struct Oct;                                   // 8 columns
template <> struct Oct<__nv_bfloat16> {
    uint4 r;
    __device__ void load(const __nv_bfloat16* p) { r = *reinterpret_cast<const uint4*>(p); }
    __device__ void get(float2 (&v)[4]) const { v[0] = unpack_bf16(r.x); v[1] = unpack_bf16(r.y); v[2] = unpack_bf16(r.z); v[3] = unpack_bf16(r.w); }
    __device__ void set(const float2 (&v)[4]) {
        r = make_uint4(pack_bf16(v[0].x, v[0].y), pack_bf16(v[1].x, v[1].y), pack_bf16(v[2].x, v[2].y), pack_bf16(v[3].x, v[3].y));
    }
    __device__ void store(__nv_bfloat16* p) const { *reinterpret_cast<uint4*>(p) = r; }
};
template <> struct Oct<float> {
    float4 a, b;
    __device__ void load(const float* p) { a = reinterpret_cast<const float4*>(p)[0]; b = reinterpret_cast<const float4*>(p)[1]; }
    __device__ void get(float2 (&v)[4]) const {
        v[0] = make_float2(a.x, a.y); v[1] = make_float2(a.z, a.w); v[2] = make_float2(b.x, b.y); v[3] = make_float2(b.z, b.w);
    }
    __device__ void set(const float2 (&v)[4]) { a = make_float4(v[0].x, v[0].y, v[1].x, v[1].y); b = make_float4(v[2].x, v[2].y, v[3].x, v[3].y); }
    __device__ void store(float* p) const { reinterpret_cast<float4*>(p)[0] = a; reinterpret_cast<float4*>(p)[1] = b; }
};
template <int RES, typename T> struct StreamOf { using type = T; };
template <typename T> struct StreamOf<RES_BF16, T> { using type = __nv_bfloat16; };
template <typename T> struct StreamOf<RES_FP32, T> { using type = float; };

constexpr int norm_threads(int TPR) { return TPR < 64 ? 128 : TPR; }

// the sum (or the maximum of bit patterns) over the TPR threads of a row, a part of a warp or whole warps; `slot` is theirs for this call and
// not written again before another barrier has passed
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* slot) {
#pragma unroll
    for (int o = (TPR < 32 ? TPR : 32) / 2; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if constexpr (TPR > 32) {
        const int warp = threadIdx.x >> 5;
        if ((threadIdx.x & 31) == 0) slot[warp] = v;
        __syncthreads();
        v = 0.f;
#pragma unroll
        for (int w = 0; w < TPR / 32; ++w) v += slot[w];
    }
    return v;
}
template <int TPR>
__device__ __forceinline__ int row_max(int v, int* slot) {
    if constexpr (TPR < 32) {
#pragma unroll
        for (int o = TPR / 2; o; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    } else v = __reduce_max_sync(0xffffffffu, v);
    if constexpr (TPR > 32) {
        const int warp = threadIdx.x >> 5;
        if ((threadIdx.x & 31) == 0) slot[warp] = v;
        __syncthreads();
        v = slot[0];
#pragma unroll
        for (int w = 1; w < TPR / 32; ++w) v = max(v, slot[w]);
    }
    return v;
}

// v / scale, as exact as a division: a product with the reciprocal alone is off by a rounding more, and puts twice as many values on the
// other side of a boundary between two 8-bit values. The reciprocal has a second part, its own rounding. Of 2^26 values 35 to 48 are then not
// the nearest to 64 bits' quotient, and 46 to 64 of plain fp32; with products and factor in two parts none would be, for twice the time of a
// norm without a stream (46 -> 88 us at 16384 x 4096), or 63 us where only quotients beside a boundary are done so.
struct Quotient {
    float inv, rest;
    __device__ Quotient(float scale) : inv(1.f / scale), rest(scale < INFINITY ? fmaf(-scale, inv, 1.f) * inv : 0.f) {}
    __device__ float2 of(float2 v) const { return fma2(v, splat2(inv), mul2(v, splat2(rest))); }
};

// Blocks that an SM holds where the registers allow it: of the rows that are on their way, the narrow ones are the fewest bytes
// (4096 x 8192 in bf16, no residual: 36 -> 30 us)
constexpr int norm_fwd_blocks(int RES, bool FP8, bool fp32, int TPR, int VPT) {
    return TPR == 512 && VPT == 2 && !fp32 && (RES == RES_NONE || (RES == RES_BF16 && !FP8)) ? 2 : 1;
}
template <typename T, int RES, bool FP8, int TPR, int VPT>
__global__ void __launch_bounds__(norm_threads(TPR), norm_fwd_blocks(RES, FP8, sizeof(T) == 4, TPR, VPT)) kda_add_rms_norm_fwd_kernel(const AddNormArgs a) {
    using R = typename StreamOf<RES, T>::type;
    constexpr int GROUPS = norm_threads(TPR) / TPR, WARPS = TPR <= 32 ? 1 : TPR / 32;
    __shared__ float s_sum[2][WARPS];
    __shared__ int s_max[2][WARPS];
    const int lane = threadIdx.x % TPR, nv = a.D / 8;
    pdl_launch_dependents();
    pdl_wait();
    Oct<float> w[VPT];
#pragma unroll
    for (int v = 0; v < VPT; ++v)
        if (const int c = lane + v * TPR; c < nv) w[v].load(a.w + 8 * c);
    int parity = 0;
    Oct<T> rx[VPT];
    Oct<R> rr[VPT];
    auto fetch = [&](long long row) {
#pragma unroll
        for (int v = 0; v < VPT; ++v) {
            const int c = lane + v * TPR;
            if (row < a.R && c < nv) {
                rx[v].load(static_cast<const T*>(a.x) + row * a.x_row + 8 * c);
                if (RES != RES_NONE) rr[v].load(static_cast<const R*>(a.r) + row * a.r_row + 8 * c);
            }
        }
    };
    const long long row0 = (long long)blockIdx.x * GROUPS + threadIdx.x / TPR, step = (long long)gridDim.x * GROUPS;
    fetch(row0);
    for (long long row = row0; row - threadIdx.x / TPR < a.R; row += step, parity ^= 1) {
        const bool live = row < a.R;
        float2 val[VPT][4], ss = make_float2(0.f, 0.f);
#pragma unroll
        for (int v = 0; v < VPT; ++v) {
            const int c = lane + v * TPR;
            if (live && c < nv) {
                rx[v].get(val[v]);
                if constexpr (RES != RES_NONE) {
                    float2 r[4];
                    rr[v].get(r);
#pragma unroll
                    for (int e = 0; e < 4; ++e) val[v][e] = add2(val[v][e], r[e]);
                    rr[v].set(val[v]);                               // the one rounding of the stream: what is kept is what is normalised
                    rr[v].store(static_cast<R*>(a.r_out) + (size_t)row * a.D + 8 * c);
                    rr[v].get(val[v]);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) ss = fma2(val[v][e], val[v][e], ss);
            }
        }
        fetch(row + step);                                           // on its way while this row is summed, scaled and stored
        const float rstd = rsqrtf(row_sum<TPR>(ss.x + ss.y, s_sum[parity]) * (1.f / a.D) + a.eps);
        if (a.rstd && live && lane == 0) a.rstd[row] = rstd;
#pragma unroll
        for (int v = 0; v < VPT; ++v) {
            const int c = lane + v * TPR;
            if (live && c < nv) {
                float2 wv[4];
                if constexpr (TPR * VPT > 1024) w[v].load(a.w + 8 * c);          // too many to be held
                w[v].get(wv);
#pragma unroll
                for (int e = 0; e < 4; ++e) val[v][e] = mul2(mul2(val[v][e], splat2(rstd)), wv[e]);
                if constexpr (!FP8) {
                    Oct<T> o;
                    o.set(val[v]);
                    o.store(static_cast<T*>(a.y) + (size_t)row * a.D + 8 * c);
                }
            }
        }
        if constexpr (FP8) {
            int m[VPT];                                              // bits of the largest |y| of a piece: a NaN is larger than anything
#pragma unroll
            for (int v = 0; v < VPT; ++v) {
                m[v] = 0;
                if (live && lane + v * TPR < nv) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) m[v] = max(m[v], max(__float_as_int(fabsf(val[v][e].x)), __float_as_int(fabsf(val[v][e].y))));
                }
            }
            auto scale_of = [](int bits) {
                const float s = __int_as_float(bits) / E4M3_MAX;
                return s < SCALE_MIN ? SCALE_MIN : s;
            };
            if (a.group) {                                           // the threads of a group are neighbours in one warp
                for (int o = a.group / 16; o; o >>= 1)
#pragma unroll
                    for (int v = 0; v < VPT; ++v) m[v] = max(m[v], __shfl_xor_sync(0xffffffffu, m[v], o));
                const int pieces = 31 - __clz(a.group / 8);          // log2 of a group's threads
#pragma unroll
                for (int v = 0; v < VPT; ++v) {
                    const int c = lane + v * TPR;
                    if (live && c < nv) {
                        const float scale = scale_of(m[v]);
                        const Quotient by(scale);
                        if (c == c >> pieces << pieces) a.scale[row * (nv >> pieces) + (c >> pieces)] = scale;
#pragma unroll
                        for (int e = 0; e < 4; ++e) val[v][e] = by.of(val[v][e]);
                    }
                }
            } else {
                int top = m[0];
#pragma unroll
                for (int v = 1; v < VPT; ++v) top = max(top, m[v]);
                const float scale = scale_of(row_max<TPR>(top, s_max[parity]));
                const Quotient by(scale);
                if (live && lane == 0) a.scale[row] = scale;
#pragma unroll
                for (int v = 0; v < VPT; ++v)
#pragma unroll
                    for (int e = 0; e < 4; ++e) val[v][e] = by.of(val[v][e]);
            }
#pragma unroll
            for (int v = 0; v < VPT; ++v) {
                const int c = lane + v * TPR;
                if (live && c < nv) {
                    uint32_t q[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) q[e] = __nv_cvt_float2_to_fp8x2(val[v][e], __NV_SATFINITE, __NV_E4M3);
                    *reinterpret_cast<uint2*>(static_cast<unsigned char*>(a.y) + (size_t)row * a.D + 8 * c) = make_uint2(q[0] | q[1] << 16, q[2] | q[3] << 16);
                }
            }
        }
    }
}

// Blocks that an SM holds: two rows' loads of two pieces per thread fit 128 registers, so that there are 512 threads (60 -> 45 us at 8192 x 4096);
// those of one piece fit 64, or 100 in fp32
constexpr int norm_bwd_resident(bool fp32, int TPR, int VPT) { return (VPT == 2 ? 512 : fp32 ? 640 : 1024) / norm_threads(TPR); }
template <typename T, int RES, int TPR, int VPT>
__global__ void __launch_bounds__(norm_threads(TPR), norm_bwd_resident(RES == RES_FP32 || sizeof(T) == 4, TPR, VPT)) kda_add_rms_norm_bwd_kernel(const AddNormArgs a) {
    using R = typename StreamOf<RES, T>::type;
    constexpr int GROUPS = norm_threads(TPR) / TPR, WARPS = TPR <= 32 ? 1 : TPR / 32;
    __shared__ float s_sum[2][WARPS];
    const int lane = threadIdx.x % TPR, nv = a.D / 8;
    const long long group = (long long)blockIdx.x * GROUPS + threadIdx.x / TPR;
    pdl_launch_dependents();
    pdl_wait();
    float2 dw[VPT][4];
    Oct<float> w[VPT];
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
        const int c = lane + v * TPR;
#pragma unroll
        for (int e = 0; e < 4; ++e) dw[v][e] = make_float2(0.f, 0.f);
        if (c < nv) w[v].load(a.w + 8 * c);
    }
    int parity = 0;
    Oct<R> rv[VPT], rd[VPT], cd[VPT];
    Oct<T> ry[VPT];
    float next_rstd = 0.f;
    auto fetch = [&](long long row) {
        if (row < a.R) next_rstd = a.rstd[row];
#pragma unroll
        for (int v = 0; v < VPT; ++v) {
            const int c = lane + v * TPR;
            if (row < a.R && c < nv) {
                const size_t at = (size_t)row * a.D + 8 * c;
                rv[v].load(static_cast<const R*>(a.v) + (RES == RES_NONE ? row * a.x_row + 8 * c : at));
                ry[v].load(static_cast<const T*>(a.dy) + at);
                if (RES != RES_NONE && a.dr_out) rd[v].load(static_cast<const R*>(a.dr_out) + at);
            }
        }
    };
    const long long step = (long long)gridDim.x * GROUPS;
    fetch(group);
    for (long long row = group; row - threadIdx.x / TPR < a.R; row += step, parity ^= 1) {
        const bool live = row < a.R;
        const float rstd = next_rstd;
        float2 n[VPT][4], dn[VPT][4], dot = make_float2(0.f, 0.f);
#pragma unroll
        for (int v = 0; v < VPT; ++v) {
            const int c = lane + v * TPR;
            if (live && c < nv) {
                float2 dy[4], wv[4];
                w[v].get(wv);
                rv[v].get(n[v]);
                ry[v].get(dy);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    n[v][e] = mul2(n[v][e], splat2(rstd));
                    dw[v][e] = fma2(dy[e], n[v][e], dw[v][e]);
                    dn[v][e] = mul2(dy[e], wv[e]);
                    dot = fma2(dn[v][e], n[v][e], dot);
                }
            }
        }
#pragma unroll
        for (int v = 0; v < VPT; ++v) cd[v] = rd[v];
        fetch(row + step);                                           // on its way while this row is summed and stored
        const float m = -row_sum<TPR>(dot.x + dot.y, s_sum[parity]) * (1.f / a.D);
#pragma unroll
        for (int v = 0; v < VPT; ++v) {
            const int c = lane + v * TPR;
            if (live && c < nv) {
                const size_t at = (size_t)row * a.D + 8 * c;
                float2 dv[4], d[4];
                if (RES != RES_NONE && a.dr_out) cd[v].get(d);
                else d[0] = d[1] = d[2] = d[3] = make_float2(0.f, 0.f);
#pragma unroll
                for (int e = 0; e < 4; ++e) dv[e] = fma2(splat2(rstd), fma2(n[v][e], splat2(m), dn[v][e]), d[e]);
                Oct<T> ox;
                ox.set(dv);
                ox.store(static_cast<T*>(a.dx) + at);
                if (RES != RES_NONE && a.dr) {
                    Oct<R> orr;
                    orr.set(dv);
                    orr.store(static_cast<R*>(a.dr) + at);
                }
            }
        }
    }
    if constexpr (GROUPS > 1) {                                      // the CTA's rows side by side first, one after the other
        __shared__ float4 s_dw[GROUPS - 1][2 * TPR * VPT];
        const int mine = threadIdx.x / TPR;
        if (mine > 0) {
#pragma unroll
            for (int v = 0; v < VPT; ++v) {
                s_dw[mine - 1][2 * (lane + v * TPR)] = make_float4(dw[v][0].x, dw[v][0].y, dw[v][1].x, dw[v][1].y);
                s_dw[mine - 1][2 * (lane + v * TPR) + 1] = make_float4(dw[v][2].x, dw[v][2].y, dw[v][3].x, dw[v][3].y);
            }
        }
        __syncthreads();
        if (mine > 0) return;
#pragma unroll
        for (int k = 0; k < GROUPS - 1; ++k)
#pragma unroll
            for (int v = 0; v < VPT; ++v) {
                const float4 p = s_dw[k][2 * (lane + v * TPR)], q = s_dw[k][2 * (lane + v * TPR) + 1];
                dw[v][0] = add2(dw[v][0], make_float2(p.x, p.y));
                dw[v][1] = add2(dw[v][1], make_float2(p.z, p.w));
                dw[v][2] = add2(dw[v][2], make_float2(q.x, q.y));
                dw[v][3] = add2(dw[v][3], make_float2(q.z, q.w));
            }
    }
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
        const int c = lane + v * TPR;
        if (c < nv) {
            Oct<float> o;
            o.set(dw[v]);
            o.store(a.part_w + (size_t)blockIdx.x * a.D + 8 * c);
        }
    }
}

// Rows that registers do not hold (D > 8192) are read once for the sum and once more, out of L2, for the gradients: 2730 x 12288 beside an fp32
// stream takes 112 us (floor 83), and 287 with a thousand bytes of spilled registers per thread
template <typename T, int RES, int TPR, int VPT>
__global__ void __launch_bounds__(TPR, 2) kda_add_rms_norm_bwd_wide_kernel(const AddNormArgs a) {
    using R = typename StreamOf<RES, T>::type;
    __shared__ float s_sum[2][TPR / 32];
    const int lane = threadIdx.x, nv = a.D / 8;
    pdl_launch_dependents();
    pdl_wait();
    float2 dw[VPT][4];
#pragma unroll
    for (int v = 0; v < VPT; ++v)
#pragma unroll
        for (int e = 0; e < 4; ++e) dw[v][e] = make_float2(0.f, 0.f);
    int parity = 0;
    for (long long row = blockIdx.x; row < a.R; row += gridDim.x, parity ^= 1) {
        const R* vp = static_cast<const R*>(a.v) + (RES == RES_NONE ? row * a.x_row : row * a.D);
        const T* yp = static_cast<const T*>(a.dy) + row * a.D;
        const float rstd = a.rstd[row];
        auto piece = [&](int c, float2 (&n)[4], float2 (&dy)[4], float2 (&dn)[4]) {
            Oct<R> rv;
            Oct<T> ry;
            Oct<float> rw;
            rv.load(vp + 8 * c);
            ry.load(yp + 8 * c);
            rw.load(a.w + 8 * c);
            rv.get(n);
            ry.get(dy);
            rw.get(dn);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                n[e] = mul2(n[e], splat2(rstd));
                dn[e] = mul2(dy[e], dn[e]);
            }
        };
        float2 dot = make_float2(0.f, 0.f);
#pragma unroll
        for (int v = 0; v < VPT; ++v)
            if (const int c = lane + v * TPR; c < nv) {
                float2 n[4], dy[4], dn[4];
                piece(c, n, dy, dn);
#pragma unroll
                for (int e = 0; e < 4; ++e) dot = fma2(dn[e], n[e], dot);
            }
        const float m = -row_sum<TPR>(dot.x + dot.y, s_sum[parity]) * (1.f / a.D);
#pragma unroll
        for (int v = 0; v < VPT; ++v)
            if (const int c = lane + v * TPR; c < nv) {
                const size_t at = (size_t)row * a.D + 8 * c;
                float2 n[4], dy[4], dn[4], d[4];
                if (RES != RES_NONE && a.dr_out) {
                    Oct<R> rd;
                    rd.load(static_cast<const R*>(a.dr_out) + at);
                    rd.get(d);
                } else d[0] = d[1] = d[2] = d[3] = make_float2(0.f, 0.f);
                piece(c, n, dy, dn);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    dw[v][e] = fma2(dy[e], n[e], dw[v][e]);
                    d[e] = fma2(splat2(rstd), fma2(n[e], splat2(m), dn[e]), d[e]);
                }
                Oct<T> ox;
                ox.set(d);
                ox.store(static_cast<T*>(a.dx) + at);
                if (RES != RES_NONE && a.dr) {
                    Oct<R> orr;
                    orr.set(d);
                    orr.store(static_cast<R*>(a.dr) + at);
                }
            }
    }
#pragma unroll
    for (int v = 0; v < VPT; ++v)
        if (const int c = lane + v * TPR; c < nv) {
            Oct<float> o;
            o.set(dw[v]);
            o.store(a.part_w + (size_t)blockIdx.x * a.D + 8 * c);
        }
}

// the shares of dw added up in a fixed order: 32 columns per block with 32 threads each, or 8 with 128 where 32 would leave SMs without a block
template <int COLS>
__global__ void __launch_bounds__(1024) kda_add_rms_norm_sum_kernel(const float* part, float* dw, int D, int rows) {
    __shared__ float s[32][COLS + 1];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, col = blockIdx.x * COLS + threadIdx.x % COLS;
    pdl_launch_dependents();
    pdl_wait();
    float sum = 0.f;
    if (col < D) {
#pragma unroll 8
        for (int k = threadIdx.x / COLS; k < rows; k += 1024 / COLS) sum += part[(size_t)k * D + col];
    }
#pragma unroll
    for (int o = COLS; o < 32; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane < COLS) s[warp][lane] = sum;
    __syncthreads();
    if (warp >= COLS) return;
    sum = s[lane][warp];                                             // a warp per column
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0 && blockIdx.x * COLS + warp < D) dw[blockIdx.x * COLS + warp] = sum;
}

// Threads and pieces for a row: as many threads as it has pieces, or pairs of pieces, in steps of some warps; idle threads cost loads that could
// be on their way (2560 columns, backward, fp32 stream: 113 -> 101 us with 160 threads in the place of 256; 64 columns 182 -> 93 with 8 in
// the place of 32). Where rows are few, one piece per thread (forward): a row's latency is then the call's.
struct NormShape { int tpr, vpt; };
static NormShape norm_shape(int D, long long R, bool backward) {
    const int nv = D / 8;
    if (nv <= 32) return {nv <= 8 ? 8 : nv <= 16 ? 16 : 32, 1};
    if (backward && nv <= 128) return {nv <= 64 ? 64 : nv <= 96 ? 96 : 128, 1};
    if (nv <= 128) return {32, nv <= 64 ? 2 : 4};
    if (nv <= 512 && R <= 2LL * sm_count() && !backward) return {512, 1};
    if (nv <= 768) return {nv <= 256 ? 128 : nv <= 320 ? 160 : nv <= 384 ? 192 : nv <= 512 ? 256 : nv <= 640 ? 320 : 384, 2};
    return {512, nv <= 1024 ? 2 : 4};
}
// f<TPR, VPT>() for a shape of either direction
#define KDA_NORM_SHAPES(s, KERNEL)                                                                                              \
    ((s).tpr == 8 ? KERNEL(8, 1) : (s).tpr == 16 ? KERNEL(16, 1)                                                                    \
     : (s).tpr == 128 ? KERNEL(128, 2) : (s).tpr == 160 ? KERNEL(160, 2) : (s).tpr == 192 ? KERNEL(192, 2)                          \
     : (s).tpr == 256 ? KERNEL(256, 2) : (s).tpr == 320 ? KERNEL(320, 2) : (s).tpr == 384 ? KERNEL(384, 2) : KERNEL(512, 2))

template <typename T, int RES, bool FP8>
static int launch_norm_fwd(const AddNormArgs& a, cudaStream_t stream) {
    const NormShape s = norm_shape(a.D, a.R, false);
#define KDA_NORM_FWD(TPR, VPT) kda_add_rms_norm_fwd_kernel<T, RES, FP8, TPR, VPT>
    void (*kernel)(const AddNormArgs) = s.tpr == 32 ? (s.vpt == 1 ? KDA_NORM_FWD(32, 1) : s.vpt == 2 ? KDA_NORM_FWD(32, 2) : KDA_NORM_FWD(32, 4))
                                        : s.tpr == 512 && s.vpt != 2 ? (s.vpt == 1 ? KDA_NORM_FWD(512, 1) : KDA_NORM_FWD(512, 4))
                                                                     : KDA_NORM_SHAPES(s, KDA_NORM_FWD);
#undef KDA_NORM_FWD
    const int threads = norm_threads(s.tpr), groups = threads / s.tpr;
    const long long want = (a.R + groups - 1) / groups, cap = sm_count() * (2048LL / threads);
    return (int)launch_early(kernel, dim3((unsigned)(want < cap ? want : cap)), threads, 0, stream, a);
}
static long long norm_bwd_blocks(int D, long long R, bool fp32, NormShape s) {
    const int groups = norm_threads(s.tpr) / s.tpr;
    const long long want = (R + groups - 1) / groups, cap = (long long)sm_count() * (s.vpt == 4 ? 2 : norm_bwd_resident(fp32, s.tpr, s.vpt));
    return want < cap ? want : cap;
}
template <typename T, int RES>
static int launch_norm_bwd(const AddNormArgs& a, cudaStream_t stream) {
    const NormShape s = norm_shape(a.D, a.R, true);
#define KDA_NORM_BWD(TPR, VPT) kda_add_rms_norm_bwd_kernel<T, RES, TPR, VPT>
    void (*kernel)(const AddNormArgs) = s.vpt == 4 ? kda_add_rms_norm_bwd_wide_kernel<T, RES, 512, 4> : s.tpr == 32 ? KDA_NORM_BWD(32, 1)
                                        : s.tpr == 64 ? KDA_NORM_BWD(64, 1) : s.tpr == 96 ? KDA_NORM_BWD(96, 1)
                                        : s.vpt == 1 && s.tpr == 128 ? KDA_NORM_BWD(128, 1) : KDA_NORM_SHAPES(s, KDA_NORM_BWD);
#undef KDA_NORM_BWD
    const long long blocks = norm_bwd_blocks(a.D, a.R, RES == RES_FP32 || sizeof(T) == 4, s);
    if (const cudaError_t e = launch_early(kernel, dim3((unsigned)blocks), norm_threads(s.tpr), 0, stream, a); e != cudaSuccess) return (int)e;
    return (int)(a.D <= 1024 ? launch_early(kda_add_rms_norm_sum_kernel<8>, dim3(a.D / 8), 1024, 0, stream, (const float*)a.part_w, a.dw, a.D, (int)blocks)
                             : launch_early(kda_add_rms_norm_sum_kernel<32>, dim3((a.D + 31) / 32), 1024, 0, stream, (const float*)a.part_w, a.dw, a.D, (int)blocks));
}

}  // namespace kda

// rows of `part_w` that the backward pass writes at most
extern "C" int kda_add_rms_norm_shares(int D, long long R) {
    using namespace kda;
    const NormShape s = norm_shape(D, R, true);
    return (int)norm_bwd_blocks(D, R, false, s);                     // of the type that takes the most
}

extern "C" int kda_launch_add_rms_norm(const kda::AddNormArgs* a, int backward, cudaStream_t stream) {
    using namespace kda;
    using bf16 = __nv_bfloat16;
    if (a->R <= 0) return 0;
    if (a->D % 8 || a->D > 16384) return -1;
#define KDA_NORM(T, RES) return backward ? launch_norm_bwd<T, RES>(*a, stream) : a->fp8 ? launch_norm_fwd<T, RES, true>(*a, stream) : launch_norm_fwd<T, RES, false>(*a, stream)
    if (!a->fp32) {
        if (a->res == RES_NONE) KDA_NORM(bf16, RES_NONE);
        if (a->res == RES_BF16) KDA_NORM(bf16, RES_BF16);
        KDA_NORM(bf16, RES_FP32);
    }
    if (a->res == RES_NONE) KDA_NORM(float, RES_NONE);
    if (a->res == RES_FP32) KDA_NORM(float, RES_FP32);
#undef KDA_NORM
    return -1;
}
