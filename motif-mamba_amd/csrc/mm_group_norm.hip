// mm_group_norm.hip -- gfx950 group norm of a row's channel groups with a gate or an activation, channels
// last, forward and backward (mm_group_norm.h has the formulas).
//
// HBM-bound: every tensor is read once and written once. A group's elements stay with the `lanes` threads that
// loaded them until the store, so that the mean, the squares of the differences from it and the outputs
// need no second read. They lie in registers, but for large groups: a block of 1,024 threads has 128 for each and spills
// the rest to scratch (backward: 16-bit groups past 8,192 channels some 290, float32 past 4,096 39 and past 8,192 327, element
// by element up to 395; forward: float32 past 8,192 36, element by element up to 157). Sums over a group's threads
// are taken by lane swaps, past 64 threads through LDS. A thread keeps its columns over the rows of its block: it
// reads weight and bias once, and the backward adds its rows' dweight and dbias in registers, one partial row per
// block, which a second kernel sums in order (no atomics: the same bits on every call).
// Measured, bfloat16 (a large copy reaches 4.9 TB/s): 16,384 x 5,120 in one group, gated, forward 140 us (3.6 TB/s); 16,384 x
// 1,536 in 24 groups, forward 36 us (4.2 TB/s), backward 84 us + 7 us for the sums (2.8 TB/s; blocks of 32 groups, so that a
// quarter of their lanes have none).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "mm_common.h"
#include "mm_group_norm.h"
#include "mm_internal.h"

namespace mm {
namespace gn {

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
// 1 / (1 + exp(-x)) on v_exp_f32 and v_rcp_f32 (about 1 ulp each).
__device__ __forceinline__ float sigmoid(float x) {
    return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-x * kLog2e));
}

// NV pieces of VE consecutive elements (16 bytes, or 1) on their way from memory, one every `lanes` pieces.
template <typename T, int VE, int NV>
struct Raw {
    typedef typename std::conditional<VE == 1, T, uint4>::type V;
    V v[NV];

    __device__ __forceinline__ void load(const T *p, int lane, int lanes, int size, bool live) {
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            const int c = (n * lanes + lane) * VE;
            v[n] = V{};
            if (live && c < size) v[n] = *reinterpret_cast<const V *>(p + c);
        }
    }
    __device__ __forceinline__ void get(int n, float *x) const {
        if constexpr (VE == 1) {
            x[0] = to_f32(v[n]);
        } else {
            const uint32_t w[4] = {v[n].x, v[n].y, v[n].z, v[n].w};
#pragma unroll
            for (int e = 0; e < VE; ++e) x[e] = elem_f32<T>(sizeof(T) == 4 ? w[e] : (w[e / 2] >> (16 * (e % 2))) & 0xffffu);
        }
    }
};
template <typename T, int VE>
__device__ __forceinline__ void store(T *p, const float *x) {
    if constexpr (VE == 1) {
        p[0] = from_f32<T>(x[0]);
    } else {
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if constexpr (sizeof(T) == 4) w[k] = __float_as_uint(x[k]);
            else w[k] = std::is_same_v<T, bf16_t> ? pack_bf16x2(x[2 * k], x[2 * k + 1]) : pack_f16x2(x[2 * k], x[2 * k + 1]);
        }
        *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// Sums of N values over a group's `lanes` threads (a power of two up to 64, then whole waves), by lane swaps in a wave and
// through `buf` past it, in the same order in every thread; `buf` alternates between two halves so that one barrier per sum
// is enough.
template <int N>
__device__ __forceinline__ void group_sums(float (&x)[N], int lanes, float *buf, int &half) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if (lanes > 1) x[i] = dpp_add<0xB1>(x[i]);    // quad_perm [1,0,3,2]
        if (lanes > 2) x[i] = dpp_add<0x4E>(x[i]);    // quad_perm [2,3,0,1]
        if (lanes > 4) x[i] = dpp_add<0x141>(x[i]);   // row_half_mirror: the other quad of 8 lanes
        if (lanes > 8) x[i] = dpp_add<0x140>(x[i]);   // row_mirror: the other half of 16 lanes
        if (lanes > 16) x[i] += __shfl_xor(x[i], 16);
        if (lanes > 32) x[i] += __shfl_xor(x[i], 32);
    }
    if (lanes <= 64) return;
    float *b = buf + half * 32;
    half ^= 1;
    if (threadIdx.x % 64 == 0)
#pragma unroll
        for (int i = 0; i < N; ++i) b[threadIdx.x / 64 * N + i] = x[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        float s = 0.f;
        for (int w = 0; w < lanes / 64; ++w) s += b[w * N + i];
        x[i] = s;
    }
}

struct Plan {
    int lanes, threads, nv;      // threads per group, per block; vectors per thread
    int64_t col_blocks, row_blocks, per;   // rows per block
};

// One row's group: h (the normed input), its mean and 1 / sqrt(var + eps).
template <typename T, int VE, int NV>
struct Group {
    float x[NV][VE], s[NV][VE], z[NV][VE];   // x, sigmoid(z), z
    float mean, rstd;

    __device__ __forceinline__ float h(int v, int e, bool before) const {
        return before ? x[v][e] * (z[v][e] * s[v][e]) : x[v][e];
    }
    __device__ __forceinline__ void take(const Raw<T, VE, NV> &rx, const Raw<T, VE, NV> &rz) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            rx.get(v, x[v]);
            rz.get(v, z[v]);
        }
    }
    __device__ __forceinline__ void stats(const mm_group_norm_params &p, int lane, int lanes, int size, float *buf, int &half) {
        const bool before = p.gate == MM_GATE_BEFORE;
        if (p.z)
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int e = 0; e < VE; ++e) s[v][e] = sigmoid(z[v][e]);
        float sum[1] = {0.f};
        mean = 0.f;
        if (!p.is_rms) {
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int e = 0; e < VE; ++e) sum[0] += h(v, e, before);
            group_sums<1>(sum, lanes, buf, half);
            mean = sum[0] / float(size);
        }
        sum[0] = 0.f;
#pragma unroll
        for (int v = 0; v < NV; ++v)
            if ((v * lanes + lane) * VE < size)
#pragma unroll
                for (int e = 0; e < VE; ++e) {
                    const float d = h(v, e, before) - mean;
                    sum[0] = __builtin_fmaf(d, d, sum[0]);
                }
        group_sums<1>(sum, lanes, buf, half);
        rstd = 1.f / sqrtf(sum[0] / float(size) + p.eps);
    }
};

template <int VE, int NV>
__device__ __forceinline__ void read_weights(const mm_group_norm_params &p, float (&w)[NV][VE], float (&b)[NV][VE], int64_t c0, int lane,
                                             int lanes, int size, bool live) {
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int e = 0; e < VE; ++e) {
            const int c = (v * lanes + lane) * VE + e;
            w[v][e] = p.weight && live && c < size ? load_w(p.weight, p.wtype, c0 + c) : 1.f;
            b[v][e] = p.bias && live && c < size ? load_w(p.bias, p.wtype, c0 + c) : 0.f;
        }
}

template <typename T, int VE, int NV, int NT>
__global__ void __launch_bounds__(NT) gn_fwd(const mm_group_norm_params p, const Plan k) {
    __shared__ float buf[64];
    const int lane = threadIdx.x % k.lanes, size = int(p.channels / p.n_groups);
    const int64_t grp = int64_t(blockIdx.x) * (k.threads / k.lanes) + threadIdx.x / k.lanes, c0 = grp * size;
    const bool live = grp < p.n_groups;
    float w[NV][VE], b[NV][VE];
    read_weights<VE, NV>(p, w, b, c0, lane, k.lanes, size, live);
    int half = 0;
    const int64_t r0 = int64_t(blockIdx.y) * k.per, r1 = min(p.rows, r0 + k.per);
    // The next row is on its way while a row is worked on.
    Raw<T, VE, NV> rx, rz = {};
    auto read = [&](int64_t row) {
        rx.load(reinterpret_cast<const T *>(p.x) + row * p.x_row_stride + c0, lane, k.lanes, size, live);
        if (p.z) rz.load(reinterpret_cast<const T *>(p.z) + row * p.z_row_stride + c0, lane, k.lanes, size, live);
    };
    if (r0 < r1) read(r0);
    for (int64_t row = r0; row < r1; ++row) {
        Group<T, VE, NV> g;
        g.take(rx, rz);
        if (row + 1 < r1) read(row + 1);
        g.stats(p, lane, k.lanes, size, buf, half);
        T *out = reinterpret_cast<T *>(p.out) + row * p.channels + c0;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int c = (v * k.lanes + lane) * VE;
            float y[VE];
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                const float a = __builtin_fmaf((g.h(v, e, p.gate == MM_GATE_BEFORE) - g.mean) * g.rstd, w[v][e], b[v][e]);
                y[e] = p.gate == MM_GATE_AFTER ? a * (g.z[v][e] * g.s[v][e]) : p.gate == MM_GATE_ACT ? a * sigmoid(a) : a;
            }
            if (live && c < size) store<T, VE>(out + c, y);
        }
    }
}

// With y the normed values, da the gradient of a and dn = da weight:
//   dh = rstd (dn - mean(dn) - y mean(dn y))          (is_rms: without mean(dn))
// dx = dh, times silu(z) where the gate comes before; dz = the gate's gradient times silu'(z).
template <typename T, int VE, int NV, int NT>
__global__ void __launch_bounds__(NT) gn_bwd(const mm_group_norm_params p, const Plan k, float *part) {
    __shared__ float buf[64];
    const int lane = threadIdx.x % k.lanes, size = int(p.channels / p.n_groups);
    const int64_t grp = int64_t(blockIdx.x) * (k.threads / k.lanes) + threadIdx.x / k.lanes, c0 = grp * size;
    const bool live = grp < p.n_groups, before = p.gate == MM_GATE_BEFORE;
    float w[NV][VE], b[NV][VE], dw[NV][VE], db[NV][VE];
    read_weights<VE, NV>(p, w, b, c0, lane, k.lanes, size, live);
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int e = 0; e < VE; ++e) dw[v][e] = db[v][e] = 0.f;
    int half = 0;
    const int64_t r0 = int64_t(blockIdx.y) * k.per, r1 = min(p.rows, r0 + k.per);
    Raw<T, VE, NV> rx, rd, rz = {};
    auto read = [&](int64_t row) {
        rx.load(reinterpret_cast<const T *>(p.x) + row * p.x_row_stride + c0, lane, k.lanes, size, live);
        rd.load(reinterpret_cast<const T *>(p.dout) + row * p.dout_row_stride + c0, lane, k.lanes, size, live);
        if (p.z) rz.load(reinterpret_cast<const T *>(p.z) + row * p.z_row_stride + c0, lane, k.lanes, size, live);
    };
    if (r0 < r1) read(r0);
    for (int64_t row = r0; row < r1; ++row) {
        Group<T, VE, NV> g;
        float d[NV][VE];
        g.take(rx, rz);
#pragma unroll
        for (int v = 0; v < NV; ++v) rd.get(v, d[v]);
        if (row + 1 < r1) read(row + 1);
        g.stats(p, lane, k.lanes, size, buf, half);
        float sum[2] = {0.f, 0.f};
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int c = (v * k.lanes + lane) * VE;
            float dz[VE];
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                const float y = (g.h(v, e, before) - g.mean) * g.rstd;
                const float a = __builtin_fmaf(y, w[v][e], b[v][e]);
                float da = d[v][e];
                if (p.gate == MM_GATE_AFTER) {
                    const float s = g.s[v][e], z = g.z[v][e];
                    dz[e] = da * a * (s * (1.f + z * (1.f - s)));
                    da *= z * s;
                } else if (p.gate == MM_GATE_ACT) {
                    const float s = sigmoid(a);
                    da *= s * (1.f + a * (1.f - s));
                }
                if (c < size) {   // elements past the group have y = -mean rstd
                    dw[v][e] = __builtin_fmaf(da, y, dw[v][e]);
                    db[v][e] += da;
                    const float dn = da * w[v][e];
                    sum[0] = __builtin_fmaf(dn, y, sum[0]);
                    sum[1] += dn;
                    d[v][e] = dn;
                }
            }
            if (p.gate == MM_GATE_AFTER && live && c < size) store<T, VE>(reinterpret_cast<T *>(p.dz) + row * p.channels + c0 + c, dz);
        }
        group_sums<2>(sum, k.lanes, buf, half);
        const float m1 = sum[0] / float(size), m0 = p.is_rms ? 0.f : sum[1] / float(size);
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int c = (v * k.lanes + lane) * VE;
            float dx[VE], dz[VE];
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                const float y = (g.h(v, e, before) - g.mean) * g.rstd;
                dx[e] = g.rstd * (d[v][e] - m0 - y * m1);
                if (before) {
                    const float s = g.s[v][e], z = g.z[v][e];
                    dz[e] = dx[e] * g.x[v][e] * (s * (1.f + z * (1.f - s)));
                    dx[e] *= z * s;
                }
            }
            if (live && c < size) {
                store<T, VE>(reinterpret_cast<T *>(p.dx) + row * p.channels + c0 + c, dx);
                if (before) store<T, VE>(reinterpret_cast<T *>(p.dz) + row * p.channels + c0 + c, dz);
            }
        }
    }
    if (!part || !live) return;
    float *pw = part + (int64_t(blockIdx.y) * 2) * p.channels + c0, *pb = pw + p.channels;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int e = 0; e < VE; ++e) {
            const int c = (v * k.lanes + lane) * VE + e;
            if (c < size) {
                pw[c] = dw[v][e];
                pb[c] = db[v][e];
            }
        }
}

// dweight and dbias: the blocks' partial rows summed in order, 32 columns and 32 runs of rows per block.
__global__ void __launch_bounds__(1024) gn_sum(const mm_group_norm_params p, const float *part, int64_t n) {
    __shared__ float buf[2][32][33];
    const int x = threadIdx.x % 32, run = threadIdx.x / 32;
    const int64_t c = int64_t(blockIdx.x) * 32 + x;
    float w = 0.f, b = 0.f;
    if (c < p.channels)
#pragma unroll 4
        for (int64_t r = run; r < n; r += 32) {
            w += part[2 * r * p.channels + c];
            b += part[(2 * r + 1) * p.channels + c];
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

static int64_t elem(mm_dtype t) { return t == MM_FLOAT32 ? 4 : 2; }

// 16-byte accesses where every row and group starts on 16 bytes.
static bool vectors(const mm_group_norm_params &p, bool bwd) {
    const int64_t e = elem(p.itype);
    uint64_t all = (p.channels / p.n_groups * e) | (p.x_row_stride * e) | reinterpret_cast<uintptr_t>(p.x);
    if (p.z) all |= (p.z_row_stride * e) | reinterpret_cast<uintptr_t>(p.z);
    if (!bwd) all |= reinterpret_cast<uintptr_t>(p.out);
    else all |= (p.dout_row_stride * e) | reinterpret_cast<uintptr_t>(p.dout) | reinterpret_cast<uintptr_t>(p.dx) | reinterpret_cast<uintptr_t>(p.dz);
    return all % 16 == 0;
}

static Plan plan(const mm_group_norm_params &p, bool bwd) {
    Plan k = {};
    const int64_t size = p.channels / p.n_groups, ve = vectors(p, bwd) ? 16 / elem(p.itype) : 1, vecs = (size + ve - 1) / ve;
    // A wave or less per group while that takes at most `most` pieces per thread, else as many waves as that takes, up to 16.
    const int most = ve == 1 ? 4 : 2, all = ve == 1 ? 16 : 4;
    if (vecs <= 64 * most) {
        k.lanes = 1;
        while (k.lanes < vecs && k.lanes < 64) k.lanes *= 2;
    } else {
        const int per = vecs <= 1024 * most ? most : all;
        k.lanes = int((vecs + 64 * per - 1) / (64 * per)) * 64;
    }
    k.nv = int((vecs + k.lanes - 1) / k.lanes);
    k.threads = k.lanes > 64 ? k.lanes : 256;
    k.col_blocks = (p.n_groups + k.threads / k.lanes - 1) / (k.threads / k.lanes);
    // Blocks for 8 waves per SIMD, half as many in the backward, which writes a partial row per block (norm of 16,384 x 5,120: 139 us,
    // 164 with half as many, 141 with twice as many).
    const int64_t want = std::max<int64_t>(1, device_simds() * 8 / ((k.threads + 63) / 64) / k.col_blocks / (bwd ? 2 : 1));
    k.per = std::max<int64_t>(1, (p.rows + std::min<int64_t>(want, 65535) - 1) / std::min<int64_t>(want, 65535));
    k.row_blocks = (p.rows + k.per - 1) / k.per;
    return k;
}

template <typename T, int VE, int NV, int NT>
static int launch_nt(const mm_group_norm_params &p, const Plan &k, bool bwd, hipStream_t s) {
    const dim3 grid{unsigned(k.col_blocks), unsigned(k.row_blocks)};
    const dim3 block{unsigned(k.threads)};
    if (!bwd) {
        hipLaunchKernelGGL((gn_fwd<T, VE, NV, NT>), grid, block, 0, s, p, k);
        return launch_status("gn_fwd");
    }
    float *part = p.dweight || p.dbias ? static_cast<float *>(p.workspace) : nullptr;
    hipLaunchKernelGGL((gn_bwd<T, VE, NV, NT>), grid, block, 0, s, p, k, part);
    if (const int rc = launch_status("gn_bwd")) return rc;
    if (!part) return MM_OK;
    hipLaunchKernelGGL(gn_sum, dim3(unsigned((p.channels + 31) / 32)), dim3(1024), 0, s, p, part, k.row_blocks);
    return launch_status("gn_sum");
}

// NT: the block sizes that plan() takes with these pieces, ascending.
template <typename T, int VE, int NV, int... NT>
static int launch(const mm_group_norm_params &p, const Plan &k, bool bwd, hipStream_t s) {
    int rc = MM_OK;
    (void)((k.threads <= NT && (rc = launch_nt<T, VE, NV, NT>(p, k, bwd, s), true)) || ...);
    return rc;
}

template <typename T>
static int run(const mm_group_norm_params &p, bool bwd, hipStream_t s) {
    const Plan k = plan(p, bwd);
    constexpr int V = 16 / sizeof(T);
    if (vectors(p, bwd)) {
        if (k.nv == 1) return launch<T, V, 1, 256>(p, k, bwd, s);
        if constexpr (sizeof(T) == 4)   // 16,384 16-bit channels are two pieces of 1,024 threads
            if (k.nv > 2) return launch<T, V, 4, 1024>(p, k, bwd, s);
        return launch<T, V, 2, 256, 512, 1024>(p, k, bwd, s);
    }
    if (k.nv <= 2) return launch<T, 1, 2, 256>(p, k, bwd, s);
    if (k.nv <= 4) return launch<T, 1, 4, 256, 512, 1024>(p, k, bwd, s);
    return launch<T, 1, 16, 512, 1024>(p, k, bwd, s);
}

static int64_t bwd_bytes(const mm_group_norm_params &p) {
    return p.dweight || p.dbias ? plan(p, true).row_blocks * 2 * p.channels * 4 : 0;
}

static int check(const mm_group_norm_params &p) {
    auto ok = [](mm_dtype t) { return t == MM_FLOAT32 || t == MM_FLOAT16 || t == MM_BFLOAT16; };
    if (!ok(p.itype) || !ok(p.wtype)) return set_error(MM_ERR_INVALID_ARGUMENT, "group norm: unknown dtype");
    if (p.rows < 0 || p.channels < 0) return set_error(MM_ERR_INVALID_ARGUMENT, "group norm: negative size");
    if (p.n_groups < 1 || p.channels % p.n_groups) return set_error(MM_ERR_INVALID_ARGUMENT, "group norm: channels must be a multiple of n_groups");
    if (p.channels / p.n_groups > MM_GROUP_NORM_MAX_GROUP)
        return set_error(MM_ERR_UNSUPPORTED, "group norm: a group must have at most 16384 channels");
    if (!(p.eps >= 0.f)) return set_error(MM_ERR_INVALID_ARGUMENT, "group norm: eps must be >= 0");
    const bool gated = p.gate == MM_GATE_AFTER || p.gate == MM_GATE_BEFORE;
    if (p.gate < MM_GATE_NONE || p.gate > MM_GATE_ACT) return set_error(MM_ERR_INVALID_ARGUMENT, "group norm: unknown gate");
    if (p.rows && p.channels && gated != (p.z != nullptr)) return set_error(MM_ERR_INVALID_ARGUMENT, "group norm: z goes with MM_GATE_AFTER or MM_GATE_BEFORE");
    return MM_OK;
}

}  // namespace gn
}  // namespace mm

using namespace mm;

extern "C" int mm_group_norm_fwd(const mm_group_norm_params *params, void *stream) {
    if (!params) return set_error(MM_ERR_INVALID_ARGUMENT, "mm_group_norm_fwd: params is NULL");
    const mm_group_norm_params &p = *params;
    if (const int rc = gn::check(p)) return rc;
    if (p.rows == 0 || p.channels == 0) return MM_OK;
    if (!p.x || !p.out) return set_error(MM_ERR_INVALID_ARGUMENT, "mm_group_norm_fwd: x and out are required");
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    switch (p.itype) {
        case MM_FLOAT32: return gn::run<float>(p, false, s);
        case MM_FLOAT16: return gn::run<f16_t>(p, false, s);
        default: return gn::run<bf16_t>(p, false, s);
    }
}

extern "C" int64_t mm_group_norm_bwd_workspace_size(const mm_group_norm_params *p) {
    if (!p || p->rows <= 0 || p->channels <= 0 || p->n_groups < 1) return 0;
    return gn::bwd_bytes(*p);
}

extern "C" int mm_group_norm_bwd(const mm_group_norm_params *params, void *stream) {
    if (!params) return set_error(MM_ERR_INVALID_ARGUMENT, "mm_group_norm_bwd: params is NULL");
    const mm_group_norm_params &p = *params;
    if (const int rc = gn::check(p)) return rc;
    if (p.channels == 0) return MM_OK;
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    if (p.rows == 0) {   // empty sums
        if (p.dweight || p.dbias) hipLaunchKernelGGL(gn::gn_sum, dim3(unsigned((p.channels + 31) / 32)), dim3(1024), 0, s, p, nullptr, int64_t(0));
        return p.dweight || p.dbias ? launch_status("gn_sum") : MM_OK;
    }
    if (!p.x || !p.dout || !p.dx || (p.z && !p.dz)) return set_error(MM_ERR_INVALID_ARGUMENT, "mm_group_norm_bwd: x, dout, dx and, with z, dz are required");
    const int64_t need = gn::bwd_bytes(p);
    if (need > 0 && (!p.workspace || p.workspace_bytes < need))
        return set_error(MM_ERR_INVALID_ARGUMENT, "mm_group_norm_bwd: the workspace is smaller than mm_group_norm_bwd_workspace_size()");
    switch (p.itype) {
        case MM_FLOAT32: return gn::run<float>(p, true, s);
        case MM_FLOAT16: return gn::run<f16_t>(p, true, s);
        default: return gn::run<bf16_t>(p, true, s);
    }
}
