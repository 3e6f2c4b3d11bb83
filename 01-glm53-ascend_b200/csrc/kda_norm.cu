// Root-mean-square norms of the attention layer on sm_100a: the input norm
// with the residual's addition (kda_rmsnorm_launch) and the per-head output
// norm with its gate (kda_gated_rmsnorm_launch), each with an optional e4m3
// output and one scale per row.
//
// Both read every input once and write every output once (5 to 7 bytes an
// element against ~10 operations), so HBM bounds them, or latency when there
// are few rows: 33,494 rows of 4,096 with an e4m3 output take 156 us (rmsnorm
// with residual, 6.2 TB/s) and 114 us (gated, 6.0 TB/s; its two special-function
// operations an element keep that unit 63% busy), 256 rows 3 to 4 us.
// Rows off 16 bytes miss the ring, whose copies start on 16 bytes, and read their
// weights singly: 33,494 x 1,001 fp16 take 53 us (2.5 TB/s).
// A row belongs to a group of 1..32 warps that keeps all of it in registers;
// the statistics cross lanes by shuffles and warps by one exchange through
// shared memory. The e4m3 scale needs max|y| = max|s w| / rms, so rmsnorm
// takes the sum of squares and max|s w| in the same exchange. The gated norm's
// statistics are per head, D / 8 neighbouring lanes, and only its scale
// crosses warps.

#include <type_traits>

#include "kda_host.cuh"
#include "kda_ring.cuh"
#include "kda_rows.cuh"

namespace kda {
namespace norm {

constexpr int kMaxThreads = 1024;
constexpr int kLongThreads = 256;

template <typename T>
__device__ __forceinline__ float weight_at(const void *w, bool fp32, int64_t i) {
    return fp32 ? static_cast<const float *>(w)[i] : to_f32(static_cast<const T *>(w)[i]);
}

// Sum or maximum over `warps` warps of this thread's row (group `slot` of the
// block), given the warp's own value in every lane.
struct Stats {
    float sum, top;
};
__device__ __forceinline__ Stats across_warps(Stats v, int warps, bool both, float2 *part) {
    const int warp = threadIdx.x >> 5;
    if ((threadIdx.x & 31) == 0) part[warp] = make_float2(v.sum, v.top);
    __syncthreads();
    const int first = warp / warps * warps;
    Stats r = {0.0f, 0.0f};
    for (int i = 0; i < warps; ++i) {
        const float2 q = part[first + i];
        if (both) r.sum += q.x;
        r.top = max_nan(r.top, q.y);
    }
    return r;
}

template <typename T>
__device__ __forceinline__ void unpack8(uint4 r, float2 (&v)[4]) {
    v[0] = unpack2<T>(r.x), v[1] = unpack2<T>(r.y), v[2] = unpack2<T>(r.z), v[3] = unpack2<T>(r.w);
}
// Eight neighbouring elements of a row as four pairs; one 16-byte access where the row allows it.
template <typename T>
__device__ __forceinline__ void load8(const T *p, bool aligned, float2 (&v)[4]) {
    if (aligned) {
        unpack8<T>(*reinterpret_cast<const uint4 *>(p), v);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = make_float2(to_f32(p[2 * i]), to_f32(p[2 * i + 1]));
    }
}
template <typename T>
__device__ __forceinline__ void store8(T *p, bool aligned, const float2 (&v)[4]) {
    if (aligned) {
        *reinterpret_cast<uint4 *>(p) = make_uint4(pack2<T>(v[0].x, v[0].y), pack2<T>(v[1].x, v[1].y),
                                                   pack2<T>(v[2].x, v[2].y), pack2<T>(v[3].x, v[3].y));
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) p[2 * i] = from_f32<T>(v[i].x), p[2 * i + 1] = from_f32<T>(v[i].y);
    }
}
__device__ __forceinline__ void store8(__nv_fp8_e4m3 *p, bool aligned, const float2 (&v)[4]) {
    if (aligned) {
        *reinterpret_cast<uint2 *>(p) =
            make_uint2(pack4_e4m3(v[0].x, v[0].y, v[1].x, v[1].y), pack4_e4m3(v[2].x, v[2].y, v[3].x, v[3].y));
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) p[2 * i] = from_f32<__nv_fp8_e4m3>(v[i].x), p[2 * i + 1] = from_f32<__nv_fp8_e4m3>(v[i].y);
    }
}
__device__ __forceinline__ float max8(float top, const float2 (&v)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) top = max_abs_nan(top, v[i].x, v[i].y);
    return top;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// The 8 weights from column e on, which are on 16 bytes.
template <typename T>
__device__ __forceinline__ void vector_weights(const KdaNormArgs &p, int e, float2 (&w)[4]) {
    if (p.weight_fp32) {
        const float4 *q = reinterpret_cast<const float4 *>(static_cast<const float *>(p.weight) + e);
        const float4 a = q[0], b = q[1];
        w[0] = make_float2(a.x, a.y), w[1] = make_float2(a.z, a.w);
        w[2] = make_float2(b.x, b.y), w[3] = make_float2(b.z, b.w);
    } else {
        load8(static_cast<const T *>(p.weight) + e, true, w);
    }
}

// The scale of a row whose largest |y| is `top`; thread `lead` writes it. Returns its inverse.
__device__ __forceinline__ float e4m3_inverse(float top, float *scale, int64_t row, bool lead) {
    const float s = max_nan(top * (1.0f / kE4m3Max), KDA_E4M3_SCALE_FLOOR);
    if (lead) scale[row] = s;
    return reciprocal(s);
}

// How a row lies in memory. ALIGNED: vectors of 8 elements on 16 bytes. SHIFTED:
// the rows of every tensor start the same `shift` elements past 16 bytes (as
// contiguous rows of an odd length do), so vectors on 16 bytes cover them with a
// part of one at either end. LOOSE: single elements, side by side.
enum Rows { ALIGNED = KDA_NORM_ALIGNED, SHIFTED = KDA_NORM_SHIFTED, LOOSE = KDA_NORM_LOOSE };

// Elements [e, e + 8) of a row of `columns`, those inside it; zeros for the rest.
template <typename T>
__device__ __forceinline__ void load8_part(const T *row, int e, int columns, float2 (&v)[4]) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int a = e + 2 * k;
        v[k].x = a >= 0 && a < columns ? to_f32(row[a]) : 0.0f;
        v[k].y = a + 1 >= 0 && a + 1 < columns ? to_f32(row[a + 1]) : 0.0f;
    }
}
template <typename T>
__device__ __forceinline__ void store8_part(T *row, int e, int columns, const float2 (&v)[4]) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int a = e + 2 * k;
        if (a >= 0 && a < columns) row[a] = from_f32<T>(v[k].x);
        if (a + 1 >= 0 && a + 1 < columns) row[a + 1] = from_f32<T>(v[k].y);
    }
}

// The products s w for the e4m3 scale's maximum come ahead of the root. They are
// held 2^32 times smaller: a row whose sum of squares is finite has |s| < 2^64, so
// with weights below 2^96 none passes fp32's range unless y does, and a row
// whose sum is infinite (root 0) gives zeros with weights below 2^32. What this takes
// from the small end, |s w| < 2^-94, is far below the scale's floor for any eps
// above 2^-112. A 16-bit output multiplies s by the root first, and loses nothing.
constexpr float kDown = 0x1p-32f, kUp = 0x1p32f;

// V units of 8 elements per thread: vectors, or (LOOSE) single elements
// `threads` apart, which keeps a warp's 2-byte accesses side by side. The sum
// with the residual is stored as soon as it is known; until the row's
// statistics have met, s w is held for an e4m3 output, and s otherwise, with
// the weights beside it, loaded first, where they are few (loaded afterwards they cost
// a row alone their latency). Rows off 16 bytes get one block of 1024 threads as their
// bound: left to itself the compiler takes 32 registers for some and spills (1,021 x
// 1,001 fp16 5.0 us against 3.8).
template <typename T, bool FP8, bool RESIDUAL, Rows ROWS, int V>
__global__ void __launch_bounds__(kMaxThreads, ROWS == ALIGNED ? 0 : 1) rmsnorm_kernel(const KdaNormArgs p, const int warps) {
    using Out = typename std::conditional<FP8, __nv_fp8_e4m3, T>::type;
    __shared__ float2 part[kMaxThreads / 32];
    let_next_start();
    wait_for_previous();
    const int threads = warps * 32, tid = threadIdx.x % threads;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * (blockDim.x / threads) + threadIdx.x / threads;
    const bool live = row < p.num_tokens;
    const int columns = live ? p.hidden : 0;
    const int shift = ROWS == SHIFTED ? static_cast<int>(row * p.x_row_stride & 7) : 0;
    const T *x = static_cast<const T *>(p.x) + row * p.x_row_stride;
    const T *res = static_cast<const T *>(p.residual) + (RESIDUAL ? row * p.residual_row_stride : 0);
    T *res_out = static_cast<T *>(p.residual_out) + (RESIDUAL ? row * p.residual_out_row_stride : 0);
    Out *out = static_cast<Out *>(p.out) + row * p.out_row_stride;
    float2 v[V][4], sum = make_float2(0.0f, 0.0f);
    // Unit j of this thread: its first element, or (LOOSE) that of its k-th pair's first half.
    const auto first = [&](int j) { return (j * threads + tid) * 8 - shift; };
    const auto loose = [&](int j, int e) { return (j * 8 + e) * threads + tid; };
    // The weights of unit j; zeros, or (SHIFTED) some weight, past the row's ends. ALIGNED units lie inside it.
    const auto weights = [&](int j, float2 (&w)[4]) {
        if constexpr (ROWS == ALIGNED) {
            vector_weights<T>(p, first(j), w);
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int a = ROWS == LOOSE ? loose(j, 2 * k) : first(j) + 2 * k, b = ROWS == LOOSE ? loose(j, 2 * k + 1) : a + 1;
                if (ROWS == LOOSE)
                    w[k] = make_float2(a < columns ? weight_at<T>(p.weight, p.weight_fp32, a) : 0.0f,
                                       b < columns ? weight_at<T>(p.weight, p.weight_fp32, b) : 0.0f);
                else
                    w[k] = make_float2(weight_at<T>(p.weight, p.weight_fp32, min(max(a, 0), p.hidden - 1)),
                                       weight_at<T>(p.weight, p.weight_fp32, min(max(b, 0), p.hidden - 1)));
            }
        }
    };
    constexpr bool kHeld = !FP8 && V <= 2;
    float2 held[kHeld ? V : 1][4];
#pragma unroll
    for (int j = 0; j < V; ++j)
        if (kHeld && (ROWS != ALIGNED || first(j) < columns)) weights(j, held[j]);
#pragma unroll
    for (int j = 0; j < V; ++j) {
        if (ROWS == LOOSE) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int a = loose(j, 2 * k), b = loose(j, 2 * k + 1);
                v[j][k] = make_float2(a < columns ? to_f32(x[a]) : 0.0f, b < columns ? to_f32(x[b]) : 0.0f);
                if (RESIDUAL)
                    v[j][k] = add2(v[j][k], make_float2(a < columns ? to_f32(res[a]) : 0.0f, b < columns ? to_f32(res[b]) : 0.0f));
            }
            continue;
        }
        const int e = first(j);
        const bool whole = ROWS == ALIGNED ? e < columns : e >= 0 && e + 8 <= columns;
        if (whole) {
            load8(x + e, true, v[j]);
        } else if (ROWS == SHIFTED && e < columns) {
            load8_part(x, e, columns, v[j]);
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) v[j][k] = make_float2(0.0f, 0.0f);
        }
        if (RESIDUAL && (whole || (ROWS == SHIFTED && e < columns))) {
            float2 r[4];
            whole ? load8(res + e, true, r) : load8_part(res, e, columns, r);
#pragma unroll
            for (int k = 0; k < 4; ++k) v[j][k] = add2(v[j][k], r[k]);
        }
    }
    float top = 0.0f;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        if (ROWS == ALIGNED && first(j) >= columns) continue;
        if (RESIDUAL && p.residual_out != nullptr) {
            if (ROWS == LOOSE) {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int a = loose(j, 2 * k), b = loose(j, 2 * k + 1);
                    if (a < columns) res_out[a] = from_f32<T>(v[j][k].x);
                    if (b < columns) res_out[b] = from_f32<T>(v[j][k].y);
                }
            } else {
                const int e = first(j);
                if (ROWS == ALIGNED || (e >= 0 && e + 8 <= columns))
                    store8(res_out + e, true, v[j]);
                else
                    store8_part(res_out, e, columns, v[j]);
            }
        }
        float2 w[4];
        if (FP8) weights(j, w);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            sum = fma2(v[j][k], v[j][k], sum);
            if (!FP8) continue;
            v[j][k] = make_float2(v[j][k].x * kDown * w[k].x, v[j][k].y * kDown * w[k].y);   // singly: pairs spill
            if (ROWS == SHIFTED) {   // a weight of infinity or NaN must not reach the maximum from past the ends
                const int a = first(j) + 2 * k;
                v[j][k] = make_float2(a >= 0 && a < columns ? v[j][k].x : 0.0f, a + 1 >= 0 && a + 1 < columns ? v[j][k].y : 0.0f);
            }
        }
        if (FP8) top = max8(top, v[j]);
    }
    Stats st = {warp_sum(sum.x + sum.y), FP8 ? warp_max_nan(top) : 0.0f};
    if (warps > 1) st = across_warps(st, warps, true, part);
    if (!live) return;
    float m = rsqrtf(st.sum / p.hidden + p.eps);
    if (FP8) {
        m *= kUp;
        m *= e4m3_inverse(st.top * m, p.scale, row, tid == 0);
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
#pragma unroll
        for (int k = 0; k < 4; ++k) v[j][k] = mul2(v[j][k], make_float2(m, m));
        if (ROWS == ALIGNED && first(j) >= columns) continue;
        if (!FP8) {
            float2 w[4];
            if (!kHeld) weights(j, w);
#pragma unroll
            for (int k = 0; k < 4; ++k) v[j][k] = mul2(v[j][k], kHeld ? held[j][k] : w[k]);
        }
        if (ROWS == LOOSE) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int a = loose(j, 2 * k), b = loose(j, 2 * k + 1);
                if (a < columns) out[a] = from_f32<Out>(v[j][k].x);
                if (b < columns) out[b] = from_f32<Out>(v[j][k].y);
            }
            continue;
        }
        const int e = first(j);
        if (ROWS == ALIGNED || (e >= 0 && e + 8 <= columns))
            store8(out + e, true, v[j]);
        else
            store8_part(out, e, columns, v[j]);
    }
}

// Rows too long for the registers of 1024 threads: read twice.
template <typename T, bool FP8>
__global__ void __launch_bounds__(kLongThreads) rmsnorm_long_kernel(const KdaNormArgs p) {
    __shared__ float2 part[kLongThreads / 32];
    let_next_start();
    wait_for_previous();
    const int64_t row = blockIdx.x;
    const T *x = static_cast<const T *>(p.x) + row * p.x_row_stride;
    const T *res = p.residual != nullptr ? static_cast<const T *>(p.residual) + row * p.residual_row_stride : nullptr;
    T *rout = p.residual_out != nullptr ? static_cast<T *>(p.residual_out) + row * p.residual_out_row_stride : nullptr;
    Stats st = {0.0f, 0.0f};
    for (int64_t i = threadIdx.x; i < p.hidden; i += kLongThreads) {
        float s = to_f32(x[i]);
        if (res != nullptr) s += to_f32(res[i]);
        st.sum = fmaf(s, s, st.sum);
        if (FP8) st.top = max_nan(st.top, fabsf(s * kDown * weight_at<T>(p.weight, p.weight_fp32, i)));
    }
    st = {warp_sum(st.sum), warp_max_nan(st.top)};
    st = across_warps(st, kLongThreads / 32, true, part);
    const float rstd = rsqrtf(st.sum / p.hidden + p.eps);
    const float inv = FP8 ? e4m3_inverse(st.top * (rstd * kUp), p.scale, row, threadIdx.x == 0) : 1.0f;
    for (int64_t i = threadIdx.x; i < p.hidden; i += kLongThreads) {
        float s = to_f32(x[i]);
        if (res != nullptr) s += to_f32(res[i]);
        const float y = s * rstd * weight_at<T>(p.weight, p.weight_fp32, i);
        if (FP8)
            static_cast<__nv_fp8_e4m3 *>(p.out)[row * p.out_row_stride + i] = from_f32<__nv_fp8_e4m3>(y * inv);
        else
            static_cast<T *>(p.out)[row * p.out_row_stride + i] = from_f32<T>(y);
        if (rout != nullptr) rout[i] = from_f32<T>(s);
    }
}

// The channels of a thread's vectors are the same in every head, since a row's
// threads are a multiple of a head's vectors: their weights are loaded once.
template <typename T, int D>
__device__ __forceinline__ void gated_weights(const KdaGatedNormArgs &p, int tid, float2 (&w)[4]) {
    const int c = tid % (D / 8) * 8;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        w[e] = make_float2(weight_at<T>(p.weight, p.weight_fp32, c + 2 * e), weight_at<T>(p.weight, p.weight_fp32, c + 2 * e + 1));
}

// Vector i (8 channels) of a row: its head's values normalised, weighted and gated.
template <typename T, int D>
__device__ __forceinline__ void gated_load8(const KdaGatedNormArgs &p, int64_t row, int64_t i, bool in, bool aligned,
                                            float2 (&y)[4], float2 (&g)[4]) {
    if (in) {
        const int64_t h = i / (D / 8);
        const int c = static_cast<int>(i % (D / 8)) * 8;
        load8(static_cast<const T *>(p.o) + row * p.o_stride[0] + h * p.o_stride[1] + c, aligned, y);
        load8(static_cast<const T *>(p.gate) + row * p.gate_row_stride + i * 8, aligned, g);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = g[e] = make_float2(0.0f, 0.0f);
    }
}
template <int D, int ACT>
__device__ __forceinline__ void gated8(const KdaGatedNormArgs &p, const float2 (&w)[4], const float2 (&g)[4], float2 (&y)[4]) {
    float2 square = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int e = 0; e < 4; ++e) square = fma2(y[e], y[e], square);
    float sum = square.x + square.y;
#pragma unroll
    for (int o = D / 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const float rstd = rsqrtf(sum * (1.0f / D) + p.eps);
#pragma unroll
    for (int e = 0; e < 4; ++e)   // from the left: w act(g) alone may pass fp32's range where y does not
        y[e] = mul2(mul2(mul2(y[e], make_float2(rstd, rstd)), w[e]), activate2<ACT>(g[e]));
}

template <typename T, bool FP8, int D, int ACT, int V>
__global__ void __launch_bounds__(kMaxThreads) gated_rmsnorm_kernel(const KdaGatedNormArgs p, const int warps,
                                                                    const bool aligned) {
    __shared__ float2 part[kMaxThreads / 32];
    let_next_start();
    wait_for_previous();
    const int threads = warps * 32, tid = threadIdx.x % threads;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * (blockDim.x / threads) + threadIdx.x / threads;
    const bool live = row < p.num_tokens;
    const int vectors = live ? p.num_heads * (D / 8) : 0;
    float2 y[V][4], g[V][4], w[4];
#pragma unroll
    for (int j = 0; j < V; ++j) gated_load8<T, D>(p, row, j * threads + tid, j * threads + tid < vectors, aligned, y[j], g[j]);
    gated_weights<T, D>(p, tid, w);
    Stats st = {0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < V; ++j) {
        gated8<D, ACT>(p, w, g[j], y[j]);
        if (FP8) st.top = max8(st.top, y[j]);
    }
    float inv = 1.0f;
    if (FP8) {
        st.top = warp_max_nan(st.top);
        if (warps > 1) st = across_warps(st, warps, false, part);
        if (live) inv = e4m3_inverse(st.top, p.scale, row, tid == 0);
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int i = j * threads + tid;
        if (i >= vectors) continue;
        if (FP8) {
#pragma unroll
            for (int e = 0; e < 4; ++e) y[j][e] = mul2(y[j][e], make_float2(inv, inv));
            store8(static_cast<__nv_fp8_e4m3 *>(p.out) + row * p.out_row_stride + i * 8, aligned, y[j]);
        } else {
            store8(static_cast<T *>(p.out) + row * p.out_row_stride + i * 8, aligned, y[j]);
        }
    }
}

// Rows of more vectors than 1024 threads hold: read twice for the scale.
template <typename T, bool FP8, int D, int ACT>
__global__ void __launch_bounds__(kLongThreads) gated_rmsnorm_long_kernel(const KdaGatedNormArgs p, const bool aligned) {
    __shared__ float2 part[kLongThreads / 32];
    let_next_start();
    wait_for_previous();
    const int64_t row = blockIdx.x, vectors = static_cast<int64_t>(p.num_heads) * (D / 8);
    float2 y[4], g[4], w[4];
    float inv = 1.0f;
    gated_weights<T, D>(p, threadIdx.x, w);
    if (FP8) {
        Stats st = {0.0f, 0.0f};
        for (int64_t i0 = 0; i0 < vectors; i0 += kLongThreads) {
            gated_load8<T, D>(p, row, i0 + threadIdx.x, i0 + threadIdx.x < vectors, aligned, y, g);
            gated8<D, ACT>(p, w, g, y);
            st.top = max8(st.top, y);
        }
        st.top = warp_max_nan(st.top);
        st = across_warps(st, kLongThreads / 32, false, part);
        inv = e4m3_inverse(st.top, p.scale, row, threadIdx.x == 0);
    }
    for (int64_t i0 = 0; i0 < vectors; i0 += kLongThreads) {
        const int64_t i = i0 + threadIdx.x;
        gated_load8<T, D>(p, row, i, i < vectors, aligned, y, g);
        gated8<D, ACT>(p, w, g, y);
        if (i >= vectors) continue;
        if (FP8) {
            for (int e = 0; e < 4; ++e) y[e] = mul2(y[e], make_float2(inv, inv));
            store8(static_cast<__nv_fp8_e4m3 *>(p.out) + row * p.out_row_stride + i * 8, aligned, y);
        } else {
            store8(static_cast<T *>(p.out) + row * p.out_row_stride + i * 8, aligned, y);
        }
    }
}

// ---------------------------------------------------------------------------
// Many rows: persistent CTAs fed by a ring of bulk copies
// ---------------------------------------------------------------------------

// A stage holds `rows` rows of each input. The rows are copied by bulk TMA, so
// how much is in flight does not depend on the registers or on when a warp gets
// to it; the barrier that a row's statistics need anyway also frees its stage.
struct RingPlan {
    int32_t warps;       // per row
    int32_t rows;        // per stage
    int32_t stages;
    int32_t row_bytes;   // of one input
};

struct Ring {
    uint64_t *full;      // one barrier per stage
    uint8_t *data;
    RingPlan plan;
    int32_t inputs;
    __device__ __forceinline__ uint8_t *row(int stage, int r, int input) const {
        return data + (static_cast<int64_t>(stage) * plan.rows + r) * inputs * plan.row_bytes + input * plan.row_bytes;
    }
};

// The whole warp 0: lane r copies row `first + r` of each input into `stage`.
__device__ __forceinline__ void ring_fill(const Ring &ring, int stage, int64_t first, int64_t tokens, const uint8_t *a,
                                          int64_t a_stride, const uint8_t *b, int64_t b_stride) {
    const int lane = threadIdx.x;
    const int64_t left = tokens - first;
    if (left <= 0) return;
    const int rows = left < ring.plan.rows ? static_cast<int>(left) : ring.plan.rows;
    if (lane == 0) mbar_arrive_expect_tx(&ring.full[stage], rows * ring.inputs * ring.plan.row_bytes);
    __syncwarp();
    if (lane < rows) {
        bulk_g2s(ring.row(stage, lane, 0), a + (first + lane) * a_stride, ring.plan.row_bytes, &ring.full[stage]);
        if (ring.inputs == 2)
            bulk_g2s(ring.row(stage, lane, 1), b + (first + lane) * b_stride, ring.plan.row_bytes, &ring.full[stage]);
    }
}

template <typename T>
__device__ __forceinline__ void load8_shared(const uint8_t *p, float2 (&v)[4]) {
    unpack8<T>(*reinterpret_cast<const uint4 *>(p), v);
}

// What the warps of a CTA tell one another, double-buffered by turn so that
// one barrier a turn is enough; the barrier also says that the stage was read.
struct Exchange {
    float sum[2][32], top[2][32];
};
template <bool SUM, bool TOP>
__device__ __forceinline__ Stats ring_exchange(Stats v, int warps, Exchange &part, int turn) {
    const int warp = threadIdx.x >> 5;
    if (warps > 1 && (threadIdx.x & 31) == 0) {
        if (SUM) part.sum[turn][warp] = v.sum;
        if (TOP) part.top[turn][warp] = v.top;
    }
    __syncthreads();
    if (warps == 1 || !(SUM || TOP)) return v;
    Stats r = {0.0f, 0.0f};
    const int first = warp / warps * warps;
    if (warps == 4) {   // a row's place is then a multiple of 16 bytes
        if (SUM) {
            const float4 q = *reinterpret_cast<const float4 *>(&part.sum[turn][first]);
            r.sum = (q.x + q.y) + (q.z + q.w);
        }
        if (TOP) {
            const float4 q = *reinterpret_cast<const float4 *>(&part.top[turn][first]);
            r.top = max_nan(max_nan(q.x, q.y), max_nan(q.z, q.w));
        }
        return r;
    }
    for (int i = 0; i < warps; ++i) {
        if (SUM) r.sum += part.sum[turn][first + i];
        if (TOP) r.top = max_nan(r.top, part.top[turn][first + i]);
    }
    return r;
}

extern __shared__ __align__(128) uint8_t ring_smem[];

// Sets the ring up and fills it; returns it ready. All threads.
template <typename Fill>
__device__ __forceinline__ Ring ring_start(const RingPlan &plan, int inputs, uint64_t *full, volatile int32_t *abort_word,
                                           Fill fill) {
    const Ring ring = {full, ring_smem, plan, inputs};
    let_next_start();
    if (threadIdx.x == 0) {
        for (int i = 0; i < plan.stages; ++i) mbar_init(&full[i], 1);
        *abort_word = 0;
        fence_mbar_init();
    }
    __syncthreads();
    wait_for_previous();
    if (threadIdx.x < 32)
        for (int i = 0; i < plan.stages; ++i) fill(ring, i, i);
    return ring;
}

// A warp that does not meet a turn's copies leaves the loop, so that no stage is
// filled or counted again whose copies have not landed; a block barrier goes on
// without the warps that have left. What warp 0 had asked for gets one more wait
// to land before the shared memory goes away (thread 0, having left at `turn`).
template <typename First>
__device__ __forceinline__ void ring_drain(const Ring &ring, int turn, int64_t rows, First first_row, int32_t *status) {
    const RingTurns turns = {ring.plan.stages};
    int32_t gave_up = 0;
    for (const int end = turns.end_in_flight(turn); turn < end && first_row(turn) < rows; ++turn)
        mbar_wait(&ring.full[turns.stage(turn)], turns.parity(turn), status, &gave_up);
}

// 80 registers let 24 warps of 4 vectors a thread be resident; with 16 at 104
// registers the gated norm of 33,494 rows of 4,096 took 134 us against 125.
constexpr int kRingRegisters = 80, kRingWarps = 24, kRingBytes = 200 * 1024, kMaxStages = 16;

template <typename T, bool FP8, bool RESIDUAL, int V>
__global__ void __maxnreg__(kRingRegisters) rmsnorm_ring_kernel(const KdaNormArgs p, const RingPlan plan) {
    __shared__ uint64_t full[kMaxStages];
    __shared__ __align__(16) Exchange part;
    __shared__ int32_t abort_word;
    const int threads = plan.warps * 32, tid = threadIdx.x % threads, sub = threadIdx.x / threads;
    const auto first_row = [&](int turn) { return (static_cast<int64_t>(turn) * gridDim.x + blockIdx.x) * plan.rows; };
    const auto fill = [&](const Ring &ring, int stage, int turn) {
        ring_fill(ring, stage, first_row(turn), p.num_tokens, static_cast<const uint8_t *>(p.x), p.x_row_stride * 2,
                  static_cast<const uint8_t *>(p.residual), p.residual_row_stride * 2);
    };
    const Ring ring = ring_start(plan, RESIDUAL ? 2 : 1, full, &abort_word, fill);
    int stage = 0;
    uint32_t phase = 0;
    int turn = 0;
    for (; first_row(turn) < p.num_tokens; ++turn) {
        const int64_t row = first_row(turn) + sub;
        const bool live = row < p.num_tokens;
        if (!__all_sync(0xffffffffu, mbar_wait(&full[stage], phase, p.status, &abort_word))) break;
        const uint8_t *x = ring.row(stage, sub, 0), *res = ring.row(stage, sub, RESIDUAL ? 1 : 0);
        float2 v[V][4], sum = make_float2(0.0f, 0.0f);
        // A 16-bit output's first weights, ahead of the exchange; the others come after it. 33,494 rows of 4,096 with
        // residual 176 us, 8,000 of 8,192 86; none ahead 177 and 90; two, packed, 186 and 90.
        float2 ahead[4];
        float top = 0.0f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int i = (j * threads + tid) * 8;
            if (live && i < p.hidden) {
                float2 w[4];
                if (FP8) vector_weights<T>(p, i, w);   // ahead of the store, which no load passes
                load8_shared<T>(x + i * 2, v[j]);
                if (RESIDUAL) {
                    float2 r[4];
                    load8_shared<T>(res + i * 2, r);
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[j][e] = add2(v[j][e], r[e]);
                    if (p.residual_out != nullptr)
                        store8(static_cast<T *>(p.residual_out) + row * p.residual_out_row_stride + i, true, v[j]);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) sum = fma2(v[j][e], v[j][e], sum);
                if (FP8) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[j][e] = mul2(mul2(v[j][e], make_float2(kDown, kDown)), w[e]);
                    top = max8(top, v[j]);
                }
            }
        }
        if (!FP8 && tid * 8 < p.hidden) vector_weights<T>(p, tid * 8, ahead);
        Stats st = {warp_sum(sum.x + sum.y), FP8 ? warp_max_nan(top) : 0.0f};
        st = ring_exchange<true, FP8>(st, plan.warps, part, turn & 1);
        if (threadIdx.x < 32) fill(ring, stage, turn + plan.stages);
        if (++stage == plan.stages) stage = 0, phase ^= 1;
        if (!live) continue;
        float m = rsqrtf(st.sum / p.hidden + p.eps);
        if (FP8) {
            m *= kUp;
            m *= e4m3_inverse(st.top * m, p.scale, row, tid == 0);
        }
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int i = (j * threads + tid) * 8;
            if (i >= p.hidden) continue;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[j][e] = mul2(v[j][e], make_float2(m, m));
            if (!FP8) {
                float2 w[4];
                if (j > 0) vector_weights<T>(p, i, w);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[j][e] = mul2(v[j][e], j > 0 ? w[e] : ahead[e]);
            }
            if (FP8)
                store8(static_cast<__nv_fp8_e4m3 *>(p.out) + row * p.out_row_stride + i, true, v[j]);
            else
                store8(static_cast<T *>(p.out) + row * p.out_row_stride + i, true, v[j]);
        }
    }
    if (threadIdx.x == 0) ring_drain(ring, turn, p.num_tokens, first_row, p.status);
}

// What a turn adds to an address stays in registers here (64-bit products of
// rows and strides, and checks of the columns, took a fifth of the kernel's
// instructions, which bound it with its exponentials: 124 us -> 116). The kernel
// above is bound by HBM and 2% slower that way.
template <typename T, bool FP8, int D, int ACT, int V>
__global__ void __maxnreg__(kRingRegisters) gated_rmsnorm_ring_kernel(const KdaGatedNormArgs p, const RingPlan plan) {
    using Out = typename std::conditional<FP8, __nv_fp8_e4m3, T>::type;
    __shared__ uint64_t full[kMaxStages];
    __shared__ __align__(16) Exchange part;
    __shared__ int32_t abort_word;
    const int threads = plan.warps * 32, tid = threadIdx.x % threads, sub = threadIdx.x / threads;
    const int vectors = p.num_heads * (D / 8);
    const int64_t step = static_cast<int64_t>(gridDim.x) * plan.rows;
    const auto first_row = [&](int turn) { return turn * step + static_cast<int64_t>(blockIdx.x) * plan.rows; };
    const auto fill = [&](const Ring &ring, int stage, int turn) {
        ring_fill(ring, stage, first_row(turn), p.num_tokens, static_cast<const uint8_t *>(p.o), p.o_stride[0] * 2,
                  static_cast<const uint8_t *>(p.gate), p.gate_row_stride * 2);
    };
    int64_t first = first_row(0);
    const Ring ring = ring_start(plan, 2, full, &abort_word, fill);
    const int stage_bytes = plan.rows * 2 * plan.row_bytes, hop = threads * 8;
    const uint8_t *source = ring.row(0, sub, 0);
    Out *out = static_cast<Out *>(p.out) + (first + sub) * p.out_row_stride + tid * 8;
    float2 w[4];
    gated_weights<T, D>(p, tid, w);
    // Vectors past the row's end read its first one: it meets no other head's, is not stored, and its
    // maximum is not taken. A row past the last reads what its stage holds, for nothing.
    bool in[V];
    int offset[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        in[j] = j * threads + tid < vectors;
        offset[j] = in[j] ? (j * threads + tid) * 16 : 0;
    }
    int stage = 0;
    uint32_t phase = 0;
    int turn = 0;
    for (; first < p.num_tokens; ++turn, first += step) {
        const bool live = first + sub < p.num_tokens;
        if (!__all_sync(0xffffffffu, mbar_wait(&full[stage], phase, p.status, &abort_word))) break;
        const uint8_t *o = source + stage * stage_bytes, *gate = o + plan.row_bytes;
        float2 y[V][4];
        Stats st = {0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < V; ++j) {
            float2 g[4];
            load8_shared<T>(o + offset[j], y[j]);
            load8_shared<T>(gate + offset[j], g);
            gated8<D, ACT>(p, w, g, y[j]);
            if (FP8 && in[j]) st.top = max8(st.top, y[j]);
        }
        if (FP8) st.top = warp_max_nan(st.top);
        st = ring_exchange<false, FP8>(st, plan.warps, part, turn & 1);
        if (threadIdx.x < 32) fill(ring, stage, turn + plan.stages);
        if (++stage == plan.stages) stage = 0, phase ^= 1;
        if (live) {
            float inv = 1.0f;
            if (FP8) inv = e4m3_inverse(st.top, p.scale, first + sub, tid == 0);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                if (!in[j]) continue;
                if (FP8)
#pragma unroll
                    for (int e = 0; e < 4; ++e) y[j][e] = mul2(y[j][e], make_float2(inv, inv));
                store8(out + j * hop, true, y[j]);
            }
        }
        out += step * p.out_row_stride;
    }
    if (threadIdx.x == 0) ring_drain(ring, turn, p.num_tokens, first_row, p.status);
}

// How rows of `units` (vectors, or 8 single elements) are laid over a launch.
struct Layout {
    int v;          // units per thread: 1, 2 or 4; 0 where the row does not fit
    int warps;      // per row
    int rows;       // per CTA
    unsigned grid;
};
Layout layout(int64_t units, int64_t rows, int64_t sms, int most = 4) {
    Layout l = {};
    // As many threads as the rows have units while they fit the GPU at half
    // occupancy, for latency; beyond that more units per thread, which leaves
    // fewer warps to meet (rmsnorm, 4,096 columns: 256 rows 4.3 us with one
    // unit against 6.3 with four; 1,000 rows 8.3 against 6.4).
    int v = 1;
    while (v < 4 && (units > static_cast<int64_t>(v) * kMaxThreads ||
                     (v < most && units * rows > static_cast<int64_t>(v) * 1024 * sms)))
        v *= 2;
    if (units > static_cast<int64_t>(v) * kMaxThreads) return l;
    while (v > 1 && units <= static_cast<int64_t>(v / 2) * 32) v /= 2;   // one warp, no idle vectors
    l.v = v;
    l.warps = static_cast<int>((units + 32 * v - 1) / (32 * v));
    l.rows = l.warps >= 4 || rows <= 4 * sms ? 1 : 4 / l.warps;
    l.grid = static_cast<unsigned>((rows + l.rows - 1) / l.rows);
    return l;
}

// The ring's layout, or v == 0 where the direct kernel is taken: rows that
// fill the resident CTAs fewer than three times (its start costs more than it
// hides: 1,000 rows of 4,096 8.6 us against 6.4; 8,256 rows 44 against 47,
// 33,494 rows 156 against 170, gated 125 against 191), or longer than 16,384.
struct RingLayout {
    int v, threads, bytes;
    unsigned grid;
    RingPlan plan;
};
RingLayout ring_layout(int64_t units, int64_t rows, int inputs, int64_t sms) {
    RingLayout l = {};
    int v = 4;
    while (v > 1 && units <= static_cast<int64_t>(v / 2) * 32) v /= 2;
    const int64_t warps = (units + 32 * v - 1) / (32 * v);
    if (warps > 16) return l;
    l.plan.warps = static_cast<int>(warps);
    l.plan.rows = warps >= 4 ? 1 : static_cast<int>(4 / warps);
    const int per_sm = kRingWarps / (l.plan.warps * l.plan.rows) > 0 ? kRingWarps / (l.plan.warps * l.plan.rows) : 1;
    const int64_t grid = per_sm * sms;
    if (rows < 3 * grid * l.plan.rows) return l;
    l.plan.row_bytes = static_cast<int32_t>(units * 16);
    const int stage = l.plan.rows * inputs * l.plan.row_bytes;
    const int stages = kRingBytes / (per_sm * stage);
    l.plan.stages = stages < kMaxStages ? stages : kMaxStages;   // 16 warps: 64 KB a stage, 3 of them
    l.bytes = l.plan.stages * stage;
    l.threads = l.plan.warps * l.plan.rows * 32;
    l.grid = static_cast<unsigned>(grid);
    l.v = v;
    return l;
}

bool aligned(const void *p, int64_t stride, int64_t rows, int bytes) {
    return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && (rows <= 1 || stride * bytes % 16 == 0);
}
bool aligned_out(const void *p, int64_t stride, int64_t rows, bool fp8) {
    // 8 values: 16 bytes, or 8 in e4m3
    return (reinterpret_cast<uintptr_t>(p) & (fp8 ? 7u : 15u)) == 0 && (rows <= 1 || stride % 8 == 0);
}

template <typename T, bool FP8, bool RESIDUAL, Rows ROWS>
cudaError_t launch_rows(const KdaNormArgs &a, const Layout &l, cudaStream_t st) {
    const auto kernel = l.v == 1   ? rmsnorm_kernel<T, FP8, RESIDUAL, ROWS, 1>
                        : l.v == 2 ? rmsnorm_kernel<T, FP8, RESIDUAL, ROWS, 2>
                                   : rmsnorm_kernel<T, FP8, RESIDUAL, ROWS, 4>;
    return launch_overlapped(kernel, dim3(l.grid), l.warps * 32 * l.rows, 0, 1, st, a, l.warps);
}
template <typename T, bool FP8, bool RESIDUAL>
cudaError_t launch_rows(Rows rows, const KdaNormArgs &a, const Layout &l, cudaStream_t st) {
    return rows == ALIGNED   ? launch_rows<T, FP8, RESIDUAL, ALIGNED>(a, l, st)
           : rows == SHIFTED ? launch_rows<T, FP8, RESIDUAL, SHIFTED>(a, l, st)
                             : launch_rows<T, FP8, RESIDUAL, LOOSE>(a, l, st);
}
template <typename T, bool FP8, bool RESIDUAL, int V>
cudaError_t launch_ring_v(const KdaNormArgs &a, const RingLayout &r, cudaStream_t st) {
    static OptIn opted;
    if (!opt_in(rmsnorm_ring_kernel<T, FP8, RESIDUAL, V>, opted, r.bytes)) return cudaErrorInvalidValue;
    return launch_overlapped(rmsnorm_ring_kernel<T, FP8, RESIDUAL, V>, dim3(r.grid), r.threads, r.bytes, 1, st, a, r.plan);
}
template <typename T, bool FP8, bool RESIDUAL>
cudaError_t launch_ring(const KdaNormArgs &a, const RingLayout &r, cudaStream_t st) {
    return r.v == 1   ? launch_ring_v<T, FP8, RESIDUAL, 1>(a, r, st)
           : r.v == 2 ? launch_ring_v<T, FP8, RESIDUAL, 2>(a, r, st)
                      : launch_ring_v<T, FP8, RESIDUAL, 4>(a, r, st);
}
// What a launch takes: the ring (ring.v != 0), the direct kernel (direct.v != 0), or neither: rows read twice.
struct Plan {
    Rows rows;
    RingLayout ring;
    Layout direct;
};
Plan plan_of(const KdaNormArgs &a, int64_t sms) {
    const int64_t T_ = a.num_tokens;
    const bool res = a.residual != nullptr, res_out = res && a.residual_out != nullptr;
    // Bases on 16 bytes (8 for e4m3), and the rows' distances alike modulo 8 elements.
    const bool based = aligned(a.x, 0, 1, 2) && (!res || aligned(a.residual, 0, 1, 2)) &&
                       (!res_out || aligned(a.residual_out, 0, 1, 2)) && aligned_out(a.out, 0, 1, a.scale != nullptr);
    const int64_t stride = T_ > 1 ? a.x_row_stride : 0;
    const auto alike = [&](int64_t other) { return T_ <= 1 || (stride - other) % 8 == 0; };
    const bool same = based && alike(a.out_row_stride) && (!res || alike(a.residual_row_stride)) &&
                      (!res_out || alike(a.residual_out_row_stride));
    Plan p = {};
    p.rows = !same ? LOOSE : a.hidden % 8 == 0 && stride % 8 == 0 && aligned(a.weight, 0, 1, 4) ? ALIGNED : SHIFTED;
    const int64_t units = (static_cast<int64_t>(a.hidden) + 7) / 8 + (p.rows == SHIFTED ? 1 : 0);   // a part at either end
    if (p.rows == ALIGNED) p.ring = ring_layout(units, T_, res ? 2 : 1, sms);
    if (p.ring.v == 0) p.direct = layout(units, T_, sms, p.rows == ALIGNED ? 4 : 2);   // the other forms hold more registers per unit
    if (p.ring.v == 0 && p.direct.v == 0) p.rows = LOOSE;
    return p;
}
template <typename T, bool FP8>
cudaError_t launch(const KdaNormArgs &a, cudaStream_t st) {
    const bool res = a.residual != nullptr;
    const Plan p = plan_of(a, sm_count());
    if (p.ring.v != 0) return res ? launch_ring<T, FP8, true>(a, p.ring, st) : launch_ring<T, FP8, false>(a, p.ring, st);
    if (p.direct.v == 0)
        return launch_overlapped(rmsnorm_long_kernel<T, FP8>, dim3(static_cast<unsigned>(a.num_tokens)), kLongThreads, 0, 1, st, a);
    return res ? launch_rows<T, FP8, true>(p.rows, a, p.direct, st) : launch_rows<T, FP8, false>(p.rows, a, p.direct, st);
}

Plan plan_of(const KdaGatedNormArgs &a, int64_t sms) {
    const int64_t T_ = a.num_tokens, units = static_cast<int64_t>(a.num_heads) * (a.head_dim / 8);
    const bool vec = aligned(a.o, a.o_stride[0], T_, 2) && aligned(a.o, a.o_stride[1], a.num_heads, 2) &&
                     aligned(a.gate, a.gate_row_stride, T_, 2) && aligned_out(a.out, a.out_row_stride, T_, a.scale != nullptr);
    Plan p = {};
    p.rows = vec ? ALIGNED : LOOSE;
    // The ring copies a token's heads as one row.
    if (vec && (a.num_heads == 1 || a.o_stride[1] == a.head_dim)) p.ring = ring_layout(units, T_, 2, sms);
    if (p.ring.v == 0) p.direct = layout(units, T_, sms);
    return p;
}
KdaNormForm form_of(const Plan &p) {
    if (p.ring.v != 0) return {KDA_NORM_RING, p.rows, p.ring.v, p.ring.plan.warps};
    if (p.direct.v != 0) return {KDA_NORM_DIRECT, p.rows, p.direct.v, p.direct.warps};
    return {KDA_NORM_LONG, p.rows, 0, kLongThreads / 32};
}

template <typename T, bool FP8, int D, int ACT, int V>
cudaError_t launch_gated_ring(const KdaGatedNormArgs &a, const RingLayout &r, cudaStream_t st) {
    static OptIn opted;
    if (!opt_in(gated_rmsnorm_ring_kernel<T, FP8, D, ACT, V>, opted, r.bytes)) return cudaErrorInvalidValue;
    return launch_overlapped(gated_rmsnorm_ring_kernel<T, FP8, D, ACT, V>, dim3(r.grid), r.threads, r.bytes, 1, st, a, r.plan);
}
template <typename T, bool FP8, int D, int ACT>
cudaError_t launch_gated(const KdaGatedNormArgs &a, cudaStream_t st) {
    const Plan p = plan_of(a, sm_count());
    const bool vec = p.rows == ALIGNED;
    if (p.ring.v == 1) return launch_gated_ring<T, FP8, D, ACT, 1>(a, p.ring, st);
    if (p.ring.v == 2) return launch_gated_ring<T, FP8, D, ACT, 2>(a, p.ring, st);
    if (p.ring.v == 4) return launch_gated_ring<T, FP8, D, ACT, 4>(a, p.ring, st);
    const Layout &l = p.direct;
    if (l.v == 0)
        return launch_overlapped(gated_rmsnorm_long_kernel<T, FP8, D, ACT>, dim3(static_cast<unsigned>(a.num_tokens)),
                                 kLongThreads, 0, 1, st, a, vec);
    const auto kernel = l.v == 1   ? gated_rmsnorm_kernel<T, FP8, D, ACT, 1>
                        : l.v == 2 ? gated_rmsnorm_kernel<T, FP8, D, ACT, 2>
                                   : gated_rmsnorm_kernel<T, FP8, D, ACT, 4>;
    return launch_overlapped(kernel, dim3(l.grid), l.warps * 32 * l.rows, 0, 1, st, a, l.warps, vec);
}
template <typename T, int D>
cudaError_t launch_gated(const KdaGatedNormArgs &a, cudaStream_t st) {
    const bool silu = a.activation == KDA_ACT_SILU;
    if (a.scale != nullptr)
        return silu ? launch_gated<T, true, D, KDA_ACT_SILU>(a, st) : launch_gated<T, true, D, KDA_ACT_SIGMOID>(a, st);
    return silu ? launch_gated<T, false, D, KDA_ACT_SILU>(a, st) : launch_gated<T, false, D, KDA_ACT_SIGMOID>(a, st);
}

bool stride_ok(int64_t stride, int64_t columns, int64_t rows) { return rows <= 1 || stride >= columns; }

// Argument checks of the two launchers: KDA_OK, or the code to return.
int check(const KdaNormArgs *args) {
    if (args == nullptr) return KDA_ERR_INVALID_ARGUMENT;
    const KdaNormArgs &a = *args;
    if (a.num_tokens < 0 || a.hidden <= 0) return KDA_ERR_INVALID_ARGUMENT;
    if (a.dtype != KDA_DTYPE_BF16 && a.dtype != KDA_DTYPE_FP16) return KDA_ERR_UNSUPPORTED;
    if (a.num_tokens == 0) return KDA_OK;
    if (a.x == nullptr || a.weight == nullptr || a.out == nullptr) return KDA_ERR_INVALID_ARGUMENT;
    if (!stride_ok(a.out_row_stride, a.hidden, a.num_tokens) ||
        (a.residual_out != nullptr && !stride_ok(a.residual_out_row_stride, a.hidden, a.num_tokens)))
        return KDA_ERR_INVALID_ARGUMENT;
    return KDA_OK;
}
int check(const KdaGatedNormArgs *args) {
    if (args == nullptr) return KDA_ERR_INVALID_ARGUMENT;
    const KdaGatedNormArgs &a = *args;
    if (a.num_tokens < 0 || a.num_heads <= 0) return KDA_ERR_INVALID_ARGUMENT;
    if (a.head_dim != 64 && a.head_dim != 128) return KDA_ERR_UNSUPPORTED;
    if (a.num_heads > (1 << 30) / a.head_dim) return KDA_ERR_TOO_LARGE;
    if (a.dtype != KDA_DTYPE_BF16 && a.dtype != KDA_DTYPE_FP16) return KDA_ERR_UNSUPPORTED;
    if (a.activation != KDA_ACT_SIGMOID && a.activation != KDA_ACT_SILU) return KDA_ERR_UNSUPPORTED;
    if (a.num_tokens == 0) return KDA_OK;
    if (a.o == nullptr || a.gate == nullptr || a.weight == nullptr || a.out == nullptr) return KDA_ERR_INVALID_ARGUMENT;
    if (!stride_ok(a.out_row_stride, static_cast<int64_t>(a.num_heads) * a.head_dim, a.num_tokens))
        return KDA_ERR_INVALID_ARGUMENT;
    return KDA_OK;
}
template <typename Args>
int form_of(const Args *args, int32_t sms, KdaNormForm *form) {
    const int rc = check(args);
    if (rc != KDA_OK) return rc;
    if (sms < 0 || form == nullptr || args->num_tokens == 0) return KDA_ERR_INVALID_ARGUMENT;
    *form = form_of(plan_of(*args, sms > 0 ? sms : sm_count()));
    return KDA_OK;
}

}  // namespace norm
}  // namespace kda

extern "C" int kda_rmsnorm_launch(const KdaNormArgs *args, void *stream) {
    using namespace kda::norm;
    const int rc = check(args);
    if (rc != KDA_OK || args->num_tokens == 0) return rc;
    const KdaNormArgs &a = *args;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool fp8 = a.scale != nullptr;
    const cudaError_t e = a.dtype == KDA_DTYPE_BF16
                              ? (fp8 ? launch<__nv_bfloat16, true>(a, st) : launch<__nv_bfloat16, false>(a, st))
                              : (fp8 ? launch<__half, true>(a, st) : launch<__half, false>(a, st));
    return e == cudaSuccess ? KDA_OK : KDA_ERR_LAUNCH;
}

extern "C" int kda_gated_rmsnorm_launch(const KdaGatedNormArgs *args, void *stream) {
    using namespace kda::norm;
    const int rc = check(args);
    if (rc != KDA_OK || args->num_tokens == 0) return rc;
    const KdaGatedNormArgs &a = *args;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool bf16 = a.dtype == KDA_DTYPE_BF16;
    const cudaError_t e =
        a.head_dim == 128 ? (bf16 ? launch_gated<__nv_bfloat16, 128>(a, st) : launch_gated<__half, 128>(a, st))
                          : (bf16 ? launch_gated<__nv_bfloat16, 64>(a, st) : launch_gated<__half, 64>(a, st));
    return e == cudaSuccess ? KDA_OK : KDA_ERR_LAUNCH;
}

extern "C" int kda_rmsnorm_form(const KdaNormArgs *args, int32_t sms, KdaNormForm *form) {
    return kda::norm::form_of(args, sms, form);
}

extern "C" int kda_gated_rmsnorm_form(const KdaGatedNormArgs *args, int32_t sms, KdaNormForm *form) {
    return kda::norm::form_of(args, sms, form);
}
