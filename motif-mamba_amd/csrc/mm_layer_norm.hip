// mm_layer_norm.hip -- gfx950 residual add with layer norm or RMS norm, channels last, forward and backward (mm_layer_norm.h has
// the formulas).
//
// HBM-bound: every tensor is read once and written once. A row stays in the registers of the threads that loaded it, one wave's up
// to 4,096 channels, four waves' beyond (and where rows are few), so that the mean, the squares of the differences from it and the
// results need no second read. Pieces of 16 bytes of x at any alignment; weight and bias come from the cache row by row. The backward
// adds its rows' dweight and dbias in registers, one partial row per block, which a second kernel sums in order (no atomics: the same
// bits on every call).
//
// 16,384 rows of 2,560, bfloat16 with a float32 residual: forward 89 us (5.6 TB/s, x and residual in part from the last-level cache; 96.5
// in calls of their own, a large copy's rate), backward 145 (4.6 TB/s: the rows' sums, with two blocks per CU), ln_sum 5. 64 rows: 3.6 us.
// Wider rows of as many elements: 10,240 of 4,096 backward 176 us (3.8 TB/s; eight pieces of a thread take 314 registers, with dbias 378, so
// that a SIMD holds one wave and half the blocks wait for the other half), 8,192 of 5,120 146, 2,560 of 16,384 with mean and dbias 196.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "mm_common.h"
#include "mm_internal.h"
#include "mm_layer_norm.h"

namespace mm {
namespace ln {

__device__ __forceinline__ float load_w(const void *p, mm_dtype dt, int64_t i) {
    switch (dt) {
        case MM_FLOAT32: return reinterpret_cast<const float *>(p)[i];
        case MM_FLOAT16: return to_f32(reinterpret_cast<const f16_t *>(p)[i]);
        default: return to_f32(reinterpret_cast<const bf16_t *>(p)[i]);
    }
}
__device__ __forceinline__ void store_w(void *p, mm_dtype dt, int64_t i, float x) {
    switch (dt) {
        case MM_FLOAT32: reinterpret_cast<float *>(p)[i] = x; break;
        case MM_FLOAT16: reinterpret_cast<f16_t *>(p)[i] = from_f32<f16_t>(x); break;
        default: reinterpret_cast<bf16_t *>(p)[i] = from_f32<bf16_t>(x);
    }
}

// A row's channels among its threads: `full` pieces of VE elements, one every 64 W pieces of a thread, and the few behind the last whole
// piece (fewer than VE), one each of the first threads.
template <int W, int VE>
struct Split {
    int lane, full, tail;   // tail: this thread's channel behind the pieces, or -1

    __device__ __forceinline__ Split(int lane_, int size) : lane(lane_), full(unsigned(size) / VE), tail(-1) {
        if (full * VE + lane < size) tail = full * VE + lane;
        if (lane >= VE) tail = -1;
    }
    __device__ __forceinline__ bool has(int v) const { return v * 64 * W + lane < full; }
    __device__ __forceinline__ int at(int v) const { return (v * 64 * W + lane) * VE; }
};

template <typename T, int VE>
__device__ __forceinline__ RawVec<T, VE> load_piece(const T *row, int c) {
    return load_any<T, VE>(reinterpret_cast<const char *>(row), uint32_t(c) * uint32_t(sizeof(T)));
}
template <typename T, int VE>
__device__ __forceinline__ void store_piece(T *row, int c, const float *x) {
    store_any<T, VE>(reinterpret_cast<char *>(row), uint32_t(c) * uint32_t(sizeof(T)), x);
}
// Four or eight weights.
template <int VE>
__device__ __forceinline__ void weight_piece(const void *p, mm_dtype dt, int c, float other, float *w) {
#pragma unroll
    for (int e = 0; e < VE; ++e) w[e] = other;
    if (!p) return;
    if (dt == MM_FLOAT32) unpack_raw(load_piece<float, VE>(static_cast<const float *>(p), c), w);
    else if (dt == MM_FLOAT16) unpack_raw(load_piece<f16_t, VE>(static_cast<const f16_t *>(p), c), w);
    else unpack_raw(load_piece<bf16_t, VE>(static_cast<const bf16_t *>(p), c), w);
}

// Sums of one or two values over a row's threads: W waves, in the same order in every thread; `buf` (4 W floats) alternates between two
// halves, which lie alike for one value and two: no wave writes where another may still read, with one barrier per sum.
template <int W, int N>
__device__ __forceinline__ void row_sum(float (&x)[N], float *buf, int &half) {
    static_assert(N <= 2, "a half has 2 W floats");
#pragma unroll
    for (int i = 0; i < N; ++i) {
        x[i] = group_sum<16>(x[i]);
        x[i] += __shfl_xor(x[i], 16);
        x[i] += __shfl_xor(x[i], 32);
    }
    if constexpr (W > 1) {
        float *b = buf + half * 2 * W;
        half ^= 1;
        if (threadIdx.x % 64 == 0)
#pragma unroll
            for (int i = 0; i < N; ++i) b[threadIdx.x / 64 * N + i] = x[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            x[i] = 0.f;
#pragma unroll
            for (int w = 0; w < W; ++w) x[i] += b[w * N + i];
        }
    }
}

constexpr int kThreads = 256;

// A thread's elements of h, and the row's mean and 1 / sqrt(var + eps).
template <int W, int VE, int NV>
struct Row {
    float h[NV][VE], ht;
    float mean, rstd;

    template <typename T, typename R>
    __device__ __forceinline__ void load(const T *x, const R *res, const Split<W, VE> &s) {
        RawVec<T, VE> rx[NV] = {};
        RawVec<R, VE> rr[NV] = {};
#pragma unroll
        for (int v = 0; v < NV; ++v)
            if (s.has(v)) {
                if (x) rx[v] = load_piece<T, VE>(x, s.at(v));
                if (res) rr[v] = load_piece<R, VE>(res, s.at(v));
            }
        ht = 0.f;
        if (s.tail >= 0) ht = (x ? to_f32(x[s.tail]) : 0.f) + (res ? to_f32(res[s.tail]) : 0.f);
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            float a[VE], b[VE];
            unpack_raw(rx[v], a);
            unpack_raw(rr[v], b);
#pragma unroll
            for (int e = 0; e < VE; ++e) h[v][e] = a[e] + b[e];
        }
    }
    __device__ __forceinline__ void stats(bool rms, float eps, int size, const Split<W, VE> &s, float *buf, int &half) {
        float sum[1] = {ht};
        mean = 0.f;
        if (!rms) {
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int e = 0; e < VE; ++e) sum[0] += h[v][e];
            row_sum<W>(sum, buf, half);
            mean = sum[0] / float(size);
        }
        sum[0] = s.tail >= 0 ? (ht - mean) * (ht - mean) : 0.f;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            float q = 0.f;
#pragma unroll
            for (int e = 0; e < VE; ++e) q = __builtin_fmaf(h[v][e] - mean, h[v][e] - mean, q);
            sum[0] += s.has(v) ? q : 0.f;
        }
        row_sum<W>(sum, buf, half);
        rstd = 1.f / sqrtf(sum[0] / float(size) + eps);
    }
};

template <typename T, typename R, int W, int VE, int NV>
__global__ void __launch_bounds__(kThreads) ln_fwd(const mm_layer_norm_params p) {
    __shared__ float buf[4 * W];
    const int size = int(p.channels);
    const int64_t row = int64_t(blockIdx.x) * (4 / W) + threadIdx.x / (64 * W);
    if (row >= p.rows) return;   // whole waves, and whole blocks where they meet at a barrier
    const Split<W, VE> s(threadIdx.x % (64 * W), size);
    int half = 0;
    Row<W, VE, NV> r;
    r.load(static_cast<const T *>(p.x) + row * p.x_row_stride, p.residual ? static_cast<const R *>(p.residual) + row * p.residual_row_stride : nullptr, s);
    if (p.residual_out) {
        R *to = static_cast<R *>(p.residual_out) + row * p.channels;
#pragma unroll
        for (int v = 0; v < NV; ++v)
            if (s.has(v)) store_piece<R, VE>(to, s.at(v), r.h[v]);
        if (s.tail >= 0) to[s.tail] = from_f32<R>(r.ht);
    }
    r.stats(p.is_rms, p.eps, size, s, buf, half);
    T *out = static_cast<T *>(p.out) + row * p.channels;
#pragma unroll
    for (int v = 0; v < NV; ++v)
        if (s.has(v)) {
            float w[VE], b[VE];
            weight_piece<VE>(p.weight, p.wtype, s.at(v), 1.f, w);
            weight_piece<VE>(p.bias, p.wtype, s.at(v), 0.f, b);
#pragma unroll
            for (int e = 0; e < VE; ++e) w[e] = __builtin_fmaf((r.h[v][e] - r.mean) * r.rstd, w[e], b[e]);
            store_piece<T, VE>(out, s.at(v), w);
        }
    if (s.tail >= 0) {
        const float w = p.weight ? load_w(p.weight, p.wtype, s.tail) : 1.f, b = p.bias ? load_w(p.bias, p.wtype, s.tail) : 0.f;
        out[s.tail] = from_f32<T>(__builtin_fmaf((r.ht - r.mean) * r.rstd, w, b));
    }
}

// With y the normed values and dn = dout weight:
//   dh = rstd (dn - mean(dn) - y mean(dn y)) + dresidual_out          (is_rms: without mean(dn))
// Waves (W = 4: blocks) take every gridDim.x-th row; part: [block][2][channels].
template <typename T, typename R, int W, int VE, int NV, bool DB>
__global__ void __launch_bounds__(kThreads) ln_bwd(const mm_layer_norm_params p, float *part) {
    __shared__ float buf[4 * W], sums[W == 1 ? 3 * 64 * VE : 1];
    const int size = int(p.channels);
    const Split<W, VE> s(threadIdx.x % (64 * W), size);
    int half = 0;
    float dw[NV][VE], db[DB ? NV : 1][VE], dwt = 0.f, dbt = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int e = 0; e < VE; ++e) {
            dw[v][e] = 0.f;
            if constexpr (DB) db[v][e] = 0.f;
        }
    const float wt = s.tail >= 0 && p.weight ? load_w(p.weight, p.wtype, s.tail) : 1.f;
#pragma unroll 1
    for (int64_t row = int64_t(blockIdx.x) * (4 / W) + threadIdx.x / (64 * W); row < p.rows; row += int64_t(gridDim.x) * (4 / W)) {
        Row<W, VE, NV> r;
        RawVec<T, VE> rd[NV] = {};
        const T *dout = static_cast<const T *>(p.dout) + row * p.dout_row_stride;
#pragma unroll
        for (int v = 0; v < NV; ++v)
            if (s.has(v)) rd[v] = load_piece<T, VE>(dout, s.at(v));
        const float dt = s.tail >= 0 ? to_f32(dout[s.tail]) : 0.f;
        r.load(p.x ? static_cast<const T *>(p.x) + row * p.x_row_stride : nullptr,
               p.residual ? static_cast<const R *>(p.residual) + row * p.residual_row_stride : nullptr, s);
        r.stats(p.is_rms, p.eps, size, s, buf, half);
        const float yt = (r.ht - r.mean) * r.rstd;
        dwt = __builtin_fmaf(dt, yt, dwt);
        dbt += dt;
        float sum[2] = {dt * wt * yt, dt * wt};
#pragma unroll
        for (int v = 0; v < NV; ++v)
            if (s.has(v)) {
                float d[VE], w[VE];
                unpack_raw(rd[v], d);
                weight_piece<VE>(p.weight, p.wtype, s.at(v), 1.f, w);
#pragma unroll
                for (int e = 0; e < VE; ++e) {
                    const float y = (r.h[v][e] - r.mean) * r.rstd, dn = d[e] * w[e];
                    dw[v][e] = __builtin_fmaf(d[e], y, dw[v][e]);
                    if constexpr (DB) db[v][e] += d[e];
                    sum[0] = __builtin_fmaf(dn, y, sum[0]);
                    sum[1] += dn;
                }
            }
        row_sum<W>(sum, buf, half);
        const float m1 = sum[0] / float(size), m0 = p.is_rms ? 0.f : sum[1] / float(size);
        const R *dres = p.dresidual_out ? static_cast<const R *>(p.dresidual_out) + row * p.dresidual_out_row_stride : nullptr;
        T *dx = p.dx ? static_cast<T *>(p.dx) + row * p.channels : nullptr;
        R *dr = p.dresidual ? static_cast<R *>(p.dresidual) + row * p.channels : nullptr;
#pragma unroll
        for (int v = 0; v < NV; ++v)
            if (s.has(v)) {
                float d[VE], w[VE], a[VE];
                unpack_raw(rd[v], d);
                weight_piece<VE>(p.weight, p.wtype, s.at(v), 1.f, w);   // once more, from the cache: held it would take too many registers
                if (dres) unpack_raw(load_piece<R, VE>(dres, s.at(v)), a);
#pragma unroll
                for (int e = 0; e < VE; ++e) {
                    const float y = (r.h[v][e] - r.mean) * r.rstd;
                    d[e] = r.rstd * (d[e] * w[e] - m0 - y * m1);
                    if (dres) d[e] += a[e];
                }
                if (dx) store_piece<T, VE>(dx, s.at(v), d);
                if (dr) store_piece<R, VE>(dr, s.at(v), d);
            }
        if (s.tail >= 0) {
            float d = r.rstd * (dt * wt - m0 - yt * m1);
            if (dres) d += to_f32(dres[s.tail]);
            if (dx) dx[s.tail] = from_f32<T>(d);
            if (dr) dr[s.tail] = from_f32<R>(d);
        }
    }
    if (!part) return;
    float *pw = part + int64_t(blockIdx.x) * 2 * p.channels, *pb = pw + p.channels;
    // The four waves' rows of a block, in order.
    auto add = [&](float *x, int n) {
        if constexpr (W == 1) {
            const int l = threadIdx.x % 64, wave = threadIdx.x / 64;
            __syncthreads();
            if (wave > 0)
                for (int e = 0; e < n; ++e) sums[((wave - 1) * VE + e) * 64 + l] = x[e];
            __syncthreads();
            if (wave == 0)
                for (int e = 0; e < n; ++e)
#pragma unroll
                    for (int w = 0; w < 3; ++w) x[e] += sums[(w * VE + e) * 64 + l];
            return wave == 0;
        }
        return true;
    };
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const bool mine = add(dw[v], VE) && s.has(v);
        if (mine) store_piece<float, VE>(pw, s.at(v), dw[v]);
        if constexpr (DB) {
            const bool too = add(db[v], VE) && s.has(v);
            if (too) store_piece<float, VE>(pb, s.at(v), db[v]);
        }
    }
    if (add(&dwt, 1) && s.tail >= 0) pw[s.tail] = dwt;
    if constexpr (DB)
        if (add(&dbt, 1) && s.tail >= 0) pb[s.tail] = dbt;
}

// dweight and dbias: the blocks' partial rows summed in order, 32 columns and 32 runs of rows per block.
__global__ void __launch_bounds__(1024) ln_sum(const mm_layer_norm_params p, const float *part, int64_t n) {
    __shared__ float buf[2][32][33];
    const int x = threadIdx.x % 32, run = threadIdx.x / 32;
    const int64_t c = int64_t(blockIdx.x) * 32 + x;
    float w = 0.f, b = 0.f;
    if (c < p.channels)
#pragma unroll 4
        for (int64_t r = run; r < n; r += 32) {
            w += part[2 * r * p.channels + c];
            if (p.dbias) b += part[(2 * r + 1) * p.channels + c];
        }
    buf[0][run][x] = w;
    buf[1][run][x] = b;
    __syncthreads();
    // The runs' sums of a column by 32 lanes of one wave.
    w = buf[0][x][run];
    b = buf[1][x][run];
    for (int d = 16; d > 0; d /= 2) {
        w += __shfl_xor(w, d);
        b += __shfl_xor(b, d);
    }
    const int64_t out = int64_t(blockIdx.x) * 32 + run;
    if (x == 0 && out < p.channels) {
        if (p.dweight) store_w(p.dweight, p.wtype, out, w);
        if (p.dbias) store_w(p.dbias, p.wtype, out, b);
    }
}

struct Plan {
    int waves, nv;        // waves of a row, pieces of a thread
    int64_t blocks;
};
static Plan plan(const mm_layer_norm_params &p, bool bwd) {
    Plan k;
    const int64_t ve = p.itype == MM_FLOAT32 ? 4 : 8, pieces = p.channels / ve, cus = device_simds() / 4;
    // One wave per row while that takes at most 64 elements of a thread, but for forwards of so few rows that they do not fill the
    // card: there four waves shorten a row's time.
    k.waves = p.channels > 4096 || (!bwd && p.rows <= cus * 4 && pieces > 64) ? 4 : 1;
    k.nv = std::max(1, int((pieces + 64 * k.waves - 1) / (64 * k.waves)));
    const int64_t per = 4 / k.waves;
    k.blocks = (p.rows + per - 1) / per;
    // Two blocks per CU, and a partial row for each.
    if (bwd) k.blocks = std::min<int64_t>(k.blocks, cus * 2);
    return k;
}

template <typename T, typename R, int W, int VE, int NV>
static int launch_nv(const mm_layer_norm_params &p, const Plan &k, bool bwd, hipStream_t s) {
    const dim3 grid{unsigned(k.blocks)}, block{unsigned(kThreads)};
    if (!bwd) {
        hipLaunchKernelGGL((ln_fwd<T, R, W, VE, NV>), grid, block, 0, s, p);
        return launch_status("ln_fwd");
    }
    float *part = p.dweight || p.dbias ? static_cast<float *>(p.workspace) : nullptr;
    if (p.dbias) hipLaunchKernelGGL((ln_bwd<T, R, W, VE, NV, true>), grid, block, 0, s, p, part);
    else hipLaunchKernelGGL((ln_bwd<T, R, W, VE, NV, false>), grid, block, 0, s, p, part);
    if (const int rc = launch_status("ln_bwd")) return rc;
    if (!part) return MM_OK;
    hipLaunchKernelGGL(ln_sum, dim3(unsigned((p.channels + 31) / 32)), dim3(1024), 0, s, p, part, k.blocks);
    return launch_status("ln_sum");
}

// NV: the numbers of pieces that kernels are built for, ascending.
template <typename T, typename R, int W, int VE, int... NV>
static int launch(const mm_layer_norm_params &p, const Plan &k, bool bwd, hipStream_t s) {
    int rc = MM_OK;
    (void)((k.nv <= NV && (rc = launch_nv<T, R, W, VE, NV>(p, k, bwd, s), true)) || ...);
    return rc;
}

template <typename T, typename R>
static int run_r(const mm_layer_norm_params &p, bool bwd, hipStream_t s) {
    const Plan k = plan(p, bwd);
    constexpr int VE = 16 / sizeof(T);
    if constexpr (sizeof(T) == 2) return k.waves == 1 ? launch<T, R, 1, VE, 1, 2, 3, 4, 5, 6, 8>(p, k, bwd, s) : launch<T, R, 4, VE, 1, 2, 4, 8>(p, k, bwd, s);
    else return k.waves == 1 ? launch<T, R, 1, VE, 1, 2, 4, 6, 8, 12, 16>(p, k, bwd, s) : launch<T, R, 4, VE, 1, 2, 4, 8, 16>(p, k, bwd, s);
}
static int run(const mm_layer_norm_params &p, bool bwd, hipStream_t s) {
    const bool wide = p.rtype == MM_FLOAT32;
    switch (p.itype) {
        case MM_FLOAT32: return run_r<float, float>(p, bwd, s);
        case MM_FLOAT16: return wide ? run_r<f16_t, float>(p, bwd, s) : run_r<f16_t, f16_t>(p, bwd, s);
        default: return wide ? run_r<bf16_t, float>(p, bwd, s) : run_r<bf16_t, bf16_t>(p, bwd, s);
    }
}

static int64_t bwd_bytes(const mm_layer_norm_params &p) {
    return p.dweight || p.dbias ? plan(p, true).blocks * 2 * p.channels * 4 : 0;
}

static int check(const mm_layer_norm_params &p) {
    auto ok = [](mm_dtype t) { return t == MM_FLOAT32 || t == MM_FLOAT16 || t == MM_BFLOAT16; };
    if (!ok(p.itype) || !ok(p.rtype) || !ok(p.wtype)) return set_error(MM_ERR_INVALID_ARGUMENT, "layer norm: unknown dtype");
    if (p.rtype != p.itype && p.rtype != MM_FLOAT32) return set_error(MM_ERR_UNSUPPORTED, "layer norm: the residual must have x's dtype or float32");
    if (p.rows < 0 || p.channels < 0) return set_error(MM_ERR_INVALID_ARGUMENT, "layer norm: negative size");
    if (p.channels > MM_LAYER_NORM_MAX_CHANNELS) return set_error(MM_ERR_UNSUPPORTED, "layer norm: a row must have at most 16384 channels");
    // A block for each row, or for four.
    if (p.rows >= int64_t(1) << 24) return set_error(MM_ERR_UNSUPPORTED, "layer norm: at most 2^24 - 1 rows");
    if (!(p.eps >= 0.f)) return set_error(MM_ERR_INVALID_ARGUMENT, "layer norm: eps must be >= 0");
    return MM_OK;
}

}  // namespace ln
}  // namespace mm

using namespace mm;

extern "C" int mm_layer_norm_fwd(const mm_layer_norm_params *params, void *stream) {
    if (!params) return set_error(MM_ERR_INVALID_ARGUMENT, "mm_layer_norm_fwd: params is NULL");
    const mm_layer_norm_params &p = *params;
    if (const int rc = ln::check(p)) return rc;
    if (p.rows == 0 || p.channels == 0) return MM_OK;
    if (!p.x || !p.out) return set_error(MM_ERR_INVALID_ARGUMENT, "mm_layer_norm_fwd: x and out are required");
    return ln::run(p, false, reinterpret_cast<hipStream_t>(stream));
}

extern "C" int64_t mm_layer_norm_bwd_workspace_size(const mm_layer_norm_params *p) {
    if (!p || p->rows <= 0 || p->channels <= 0) return 0;
    return ln::bwd_bytes(*p);
}

extern "C" int mm_layer_norm_bwd(const mm_layer_norm_params *params, void *stream) {
    if (!params) return set_error(MM_ERR_INVALID_ARGUMENT, "mm_layer_norm_bwd: params is NULL");
    const mm_layer_norm_params &p = *params;
    if (const int rc = ln::check(p)) return rc;
    if (p.channels == 0) return MM_OK;
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    if (p.rows == 0) {   // empty sums
        if (p.dweight || p.dbias) hipLaunchKernelGGL(ln::ln_sum, dim3(unsigned((p.channels + 31) / 32)), dim3(1024), 0, s, p, nullptr, int64_t(0));
        return p.dweight || p.dbias ? launch_status("ln_sum") : MM_OK;
    }
    if ((!p.x && !p.residual) || !p.dout) return set_error(MM_ERR_INVALID_ARGUMENT, "mm_layer_norm_bwd: x or residual, and dout, are required");
    const int64_t need = ln::bwd_bytes(p);
    if (need > 0 && (!p.workspace || p.workspace_bytes < need))
        return set_error(MM_ERR_INVALID_ARGUMENT, "mm_layer_norm_bwd: the workspace is smaller than mm_layer_norm_bwd_workspace_size()");
    return ln::run(p, true, s);
}
