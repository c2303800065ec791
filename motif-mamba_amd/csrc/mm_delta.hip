// mm_delta.hip -- gfx950 gated delta rule: chunked forward and backward on the matrix cores. The single-token step and the plan of
// a call are in mm_delta_api.hip; operand layouts, planes and decays are the linear attention's (mm_linattn_dev.h).
//
// The mathematics. A chunk of C tokens starts from the state S (dk x dv). With c_i the sum of log_decay up to token i, c_end its
// total, D_ij = exp(c_i - c_j) for i >= j, B = diag(beta), N the strict lower triangle of K K^T . D and M the lower one of
// scale Q K^T . D:
//     X = V - diag(e^c) K S            what the tokens would correct if they did not see each other
//     (I + N B) Z = X,  U = B Z        z_i = v_i - S'^T k_i
//     O = scale diag(e^c) Q S + M U,   S' = e^c_end S + K^T diag(e^(c_end - c)) U
// P = -(I + N B)^-1 N is strictly lower triangular and gives Z = X + P B X, without a division by beta, and the gradient's
// transposed system as well: with R the gradient of S',
//     dU = M^T dO + diag(e^(c_end - c)) K R,   G = dU + P^T B dU,   dV = dX = B G,   dbeta_i = G_i . Z_i
//     R' = e^c_end R + scale Q^T diag(e^c) dO - K^T diag(e^c) dV
//     dQ = scale diag(e^c) dO S^T + A K,                    A = the lower triangle of scale dO U^T . D
//     dK = A^T Q + E K + E^T K - diag(e^c) dV S^T + diag(e^(c_end - c)) U R^T,   E = minus the strict one of dV U^T . D
// P and M need no state: dr_prep makes them for all chunks at once, dr_walk carries the state through a row's chunks, dr_back the
// state's gradient back, and dr_grad takes dQ and dK chunk by chunk from the kept S, R, Z and dV, again all chunks at once. Rows of few heads
// run in segments: a first walk finds what each adds to the state and what it makes of it, dr_join the states that they start from.
//
// Exactness: every float32 factor (S, R, P, M, U, dV and the decayed scores) enters its product as three bfloat16 planes (2^-25), for
// every input type: two would be 2^-17 per factor, and errors of the state add up over the chunks. 16-bit results are rounded once.
//
// Built once per input type: this file for float32, mm_delta_f16.hip / mm_delta_bf16.hip, which set MM_DELTA_TYPE.
#ifndef MM_DELTA_TYPE
#define MM_DELTA_TYPE float
#endif

#include <algorithm>

#include "mm_delta_host.h"
#include "mm_linattn_dev.h"

namespace mm {
namespace dr {

using namespace la;

constexpr int kWaves = 4, kThreads = 64 * kWaves;

// ---- triangles as operands -----------------------------------------------------------------------

// The 32-wide A operands of a triangle of 16 x 16 tiles: row tile t, columns 32 j .. 32 j + 31, those that hold a tile of it. LOWER:
// 2 j <= t, its transpose 2 j + 1 >= t.
template <int C> constexpr int kFrags = C == 64 ? 6 : 2;
template <int C, bool LOWER>
constexpr bool has_frag(int t, int j) { return LOWER ? 2 * j <= t : 2 * j + 1 >= t; }
template <int C, bool LOWER>
constexpr int frag_at(int t, int j) { return LOWER ? (t < 2 ? t : 2 * t - 2 + j) : (C == 32 ? t : t < 2 ? 2 * t + j : t + 2); }
template <int C> constexpr int kImage = kFrags<C> * kPlanes * 512;   // elements

__device__ __forceinline__ bf16x8 image_frag(const u16 *img, int frag, int plane, int lane) {
    return *reinterpret_cast<const bf16x8 *>(img + (frag * kPlanes + plane) * 512 + lane * 8);
}

// ---- a workgroup's place -------------------------------------------------------------------------

struct Spot {
    int b, h, bh;
};
template <typename A>
__device__ __forceinline__ Spot spot_of(const A &a, unsigned pair) {
    Spot p;
    p.bh = afresh(int(pair));
    p.h = afresh(int(pair % unsigned(a.heads)));
    p.b = afresh(int(pair / unsigned(a.heads)));
    return p;
}
__device__ __forceinline__ Gates gates_of(const Gate &g, const Spot &p) {
    const int64_t size = g.type == MM_FLOAT32 ? 4 : 2;
    return Gates{g.p ? afresh(static_cast<const char *>(g.p) + (p.b * g.batch + p.h * g.head) * size) : nullptr, afresh(g.seq * size), mm_dtype(afresh(int(g.type)))};
}
template <int C>
__device__ __forceinline__ uint32_t load_gate(const Gates &g, int t0, int end, int lane) {
    return g.p ? g.template load<C>(t0, end, lane) : 0u;
}
__device__ __forceinline__ float decode_beta(uint32_t w, mm_dtype t) {
    return t == MM_FLOAT32 ? __uint_as_float(w) : t == MM_BFLOAT16 ? __uint_as_float(w << 16) : elem_f32<f16_t>(w);
}

// A chunk's decays (without the scale), beta, and scale e^c.
template <int C>
struct Chunk {
    Decays<C> d;
    float beta[C], inq[C];
};
// One wave makes them; g and b: the lane's token's bits.
template <int C>
__device__ __forceinline__ void make_chunk(Chunk<C> &k, uint32_t g, mm_dtype gtype, uint32_t b, mm_dtype btype, float scale, int lane) {
    make_decays<C>(k.d, decode_g(g, gtype), 1.f, lane);
    if (C == 64 || lane < C) {
        k.beta[lane] = decode_beta(b, btype);
        k.inq[lane] = k.d.in[lane] * scale;
    }
}

// What a walk needs of it: no factors between two tokens. It lies behind the chunk's images (dr_prep).
template <int C>
struct __attribute__((aligned(16))) Steps {
    float in[C], out[C], beta[C], inq[C];   // e^c, e^(c_end - c), beta, scale e^c
    float hi[C], lo[C];                     // c
    float all;                              // e^c_end
};
static_assert(sizeof(Steps<64>) == steps_bytes(64) && sizeof(Steps<32>) == steps_bytes(32), "the plan's bytes");
template <int C>
__device__ __forceinline__ void write_steps(char *dst, const Chunk<C> &k, int tid) {
    float *to = reinterpret_cast<float *>(dst);
    for (int x = tid; x < 6 * C + 1; x += kThreads) {
        const int n = x / C, t = x % C;
        to[x] = n == 0 ? k.d.in[t] : n == 1 ? k.d.out[t] : n == 2 ? k.beta[t] : n == 3 ? k.inq[t] : n == 4 ? k.d.hi[t] : n == 5 ? k.d.lo[t] : k.d.all;
    }
}
// A chunk's record: N images, then its steps.
template <int C, int N> constexpr int kRecord = N * kImage<C> * 2 + int(sizeof(Steps<C>));

// ---- products ------------------------------------------------------------------------------------

// s += the tiles L of X Y^T, X in PX planes and Y in PY: column i the row token 16 O + i of X, rows 4g + r the tokens of Y.
template <int PX, int PY, int C, int D, typename L>
__device__ __forceinline__ void tile_products(f32x4 *s, const u16 *X, const u16 *Y, int lane) {
    constexpr int PL = kTile<C, D>;
    const int g = lane >> 4, i = lane & 15;
    constexpr int B = PY > 1 ? 3 : 4;   // tiles whose operands are held at once
#pragma unroll
    for (int k = 0; k < D / 32; ++k) {
#pragma unroll
        for (int j0 = 0; j0 < L::N; j0 += B) {
            bf16x8 a[B][PY], b[B][PX];
#pragma unroll
            for (int j = 0; j < B && j0 + j < L::N; ++j) {
#pragma unroll
                for (int p = 0; p < PX; ++p) {
                    if (j > 0 && L::O(j0 + j) == L::O(j0 + j - 1)) b[j][p] = b[j - 1][p];
                    else b[j][p] = frag_row<D>(X + p * PL, 16 * L::O(j0 + j), k, g, i);
                }
#pragma unroll
                for (int p = 0; p < PY; ++p) a[j][p] = frag_row<D>(Y + p * PL, 16 * L::n(j0 + j), k, g, i);
            }
#pragma unroll
            for (int p = 0; p < PY; ++p)
#pragma unroll
                for (int q = 0; q < PX; ++q)
                    if (p + q < kPlanes)
#pragma unroll
                        for (int j = 0; j < B && j0 + j < L::N; ++j) s[j0 + j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[j][p], b[j][q], s[j0 + j], 0, 0, 0);
        }
        if (k % 2) __builtin_amdgcn_sched_barrier(0);   // (no more than two steps' operands held)
    }
}
// The waves' shares of a chunk's lower triangle of tiles.
template <int C, typename F>
__device__ __forceinline__ void each_tile(int wave, F &&f) {
    if constexpr (C == 64) {
        switch (wave) {
            case 0: f(Tiles<3, 0, 3, 1, 3, 2>{}); break;
            case 1: f(Tiles<2, 0, 2, 1, 2, 2>{}); break;
            case 2: f(Tiles<1, 0, 1, 1, 3, 3>{}); break;
            default: f(Tiles<0, 0>{});
        }
    } else {
        switch (wave) {
            case 0: f(Tiles<1, 0>{}); break;
            case 1: f(Tiles<1, 1>{}); break;
            case 2: f(Tiles<0, 0>{});
        }
    }
}

// Rows of accumulators times w as B operands in three planes: f[j] holds the tokens 32 j .. 32 j + 31.
template <int C, int NC>
__device__ __forceinline__ void split_rows(bf16x8 (&f)[C / 32][NC][kPlanes], const f32x4 (&x)[C / 16][NC], const float *w, int lane) {
    const int g = lane >> 4;
#pragma unroll
    for (int j = 0; j < C / 32; ++j) {
        const f32x4 w0 = *reinterpret_cast<const f32x4 *>(w + 32 * j + 4 * g), w1 = *reinterpret_cast<const f32x4 *>(w + 32 * j + 16 + 4 * g);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            float y[8];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                y[r] = x[2 * j][c][r] * w0[r];
                y[4 + r] = x[2 * j + 1][c][r] * w1[r];
            }
            split8(y, f[j][c]);
        }
    }
}
// O += T f, T a triangle's image.
template <int C, int NC, bool LOWER, int PF>
__device__ __forceinline__ void triangle(f32x4 (&O)[C / 16][NC], const u16 *img, const bf16x8 (&f)[C / 32][NC][PF], int lane) {
#pragma unroll
    for (int j = 0; j < C / 32; ++j) {
        bf16x8 a[C / 16][kPlanes];
#pragma unroll
        for (int t = 0; t < C / 16; ++t)
            if (has_frag<C, LOWER>(t, j))
#pragma unroll
                for (int p = 0; p < kPlanes; ++p) a[t][p] = image_frag(img, frag_at<C, LOWER>(t, j), p, lane);
#pragma unroll
        for (int p = 0; p < kPlanes; ++p)
#pragma unroll
            for (int q = 0; q < PF; ++q)
                if (p + q < kPlanes)
#pragma unroll
                    for (int t = 0; t < C / 16; ++t)
                        if (has_frag<C, LOWER>(t, j))
#pragma unroll
                            for (int c = 0; c < NC; ++c)
                                O[t][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[t][p], f[j][c][q], O[t][c], 0, 0, 0);
    }
}
// S += Y^T f, Y a tile of the inputs' rows.
template <typename T, int C, int KD, int NC>
__device__ __forceinline__ void add_rows(f32x4 (&S)[KD / 16][NC], const u16 *Y, const bf16x8 (&f)[C / 32][NC][kPlanes], int lane) {
    constexpr int PL = kTile<C, KD>, PI = Cfg<T>::in, KB = PI > 1 ? 2 : 4;
    const int g = lane >> 4, i = lane & 15;
#pragma unroll
    for (int j = 0; j < C / 32; ++j)
#pragma unroll
        for (int b = 0; b < KD / 16; b += KB) {
            bf16x8 a[KB][PI];
#pragma unroll
            for (int k = 0; k < KB; ++k)
#pragma unroll
                for (int p = 0; p < PI; ++p) a[k][p] = frag_tr<KD>(Y + p * PL, 32 * j, 16 * (b + k), g, i);
#pragma unroll
            for (int p = 0; p < PI; ++p)
#pragma unroll
                for (int q = 0; q < kPlanes; ++q)
                    if (p + q < kPlanes)
#pragma unroll
                        for (int k = 0; k < KB; ++k)
#pragma unroll
                            for (int c = 0; c < NC; ++c)
                                S[b + k][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[k][p], f[j][c][q], S[b + k][c], 0, 0, 0);
        }
}
// A tile of the inputs' rows in the accumulators' layout, from the wave's columns.
template <typename T, int C, int NC, int LDV, typename F>
__device__ __forceinline__ void tile_columns(const u16 *V, int col, int lane, F &&f) {
    constexpr int PL = kTile<C, LDV>, PI = Cfg<T>::in;
    const int g = lane >> 4, i = lane & 15;
#pragma unroll
    for (int j = 0; j < C / 32; ++j)
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            float x[8], y[8];
            unpack_frag(frag_tr<LDV>(V + (PI - 1) * PL, 32 * j, col + 16 * c, g, i), x);
#pragma unroll
            for (int p = PI - 2; p >= 0; --p) {
                unpack_frag(frag_tr<LDV>(V + p * PL, 32 * j, col + 16 * c, g, i), y);
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] += y[e];
            }
            f(j, c, x);
        }
}

// ---- P and M -------------------------------------------------------------------------------------

// Row pitch of the float32 triangles in LDS: rows of one column lie 4 banks apart.
template <int C> constexpr int kPitch = C + 4;

// A triangle in `f` (row-major, pitch kPitch; 0 above the diagonal in the tiles on it, tiles above it not written) as operands, TR: its
// transpose. NW waves share it.
template <int C, bool TR, int NW = kWaves>
__device__ __forceinline__ void write_image(char *dst, const float *f, int wave, int lane) {
    const int g = lane >> 4, i = lane & 15;
#pragma unroll
    for (int t = 0; t < C / 16; ++t)
#pragma unroll
        for (int j = 0; j < C / 32; ++j)
            if (has_frag<C, !TR>(t, j)) {
                const int n = frag_at<C, !TR>(t, j);
                if (n % NW != wave) continue;
                float x[8];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int o = 2 * j + h;   // tile o
                    f32x4 y = {0.f, 0.f, 0.f, 0.f};
                    if constexpr (TR) {
                        if (o >= t)
#pragma unroll
                            for (int r = 0; r < 4; ++r) y[r] = f[(16 * o + 4 * g + r) * kPitch<C> + 16 * t + i];
                    } else {
                        if (o <= t) y = *reinterpret_cast<const f32x4 *>(&f[(16 * t + i) * kPitch<C> + 16 * o + 4 * g]);
                    }
#pragma unroll
                    for (int r = 0; r < 4; ++r) x[4 * h + r] = y[r];
                }
                bf16x8 p[kPlanes];
                split8(x, p);
#pragma unroll
                for (int q = 0; q < kPlanes; ++q)
                    *reinterpret_cast<bf16x8 *>(dst + ((n * kPlanes + q) * 64 + lane) * 16) = p[q];
            }
}

// The records of every chunk: the images of P and M; REV, for the backward: that of P, and those of P^T and M^T. One workgroup per chunk. The
// triangles are made in float32: the diagonal tiles of P by substitution, row by row, those of a column block below by 16 x 16 products on
// v_mfma_f32_16x16x4_f32, which keeps them float32. Bound by what it stores (38 KB for a chunk of 64, 57 with REV) and by the substitution's
// latency, which the workgroups on a CU hide for each other: 10,240 chunks at dk 128, 384 MB of operands, 134 us (2.9 TB/s). Two on a CU, as
// with M in LDS of its own, took 180, and so did three with spills; M lies in P's place, and waves that do not substitute write its image.
// A workgroup that takes several chunks and loads ahead was slower: the loads' wait is one for the stores before them too.
template <typename T, int KD> constexpr int kPrepGroups = KD == 64 || sizeof(T) == 2 ? 4 : 3;   // on a CU, by registers
template <typename T, int KD, bool REV, bool VEC>
__global__ void __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(kPrepGroups<T, KD>, kPrepGroups<T, KD>))) dr_prep(const Args) {
    constexpr int C = Cfg<T>::C, PI = Cfg<T>::in, CT = C / 16, LD = kPitch<C>;
    typedef Stage<T, C, KD, kThreads, VEC> SX;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    u16 *K = reinterpret_cast<u16 *>(smem), *Q = K + PI * kTile<C, KD>;
    float *N = reinterpret_cast<float *>(smem), *P = N + C * LD, *M = P;   // over K and Q, once those are read; P over M
    constexpr int kTiles = 2 * 2 * PI * kTile<C, KD>, kTri = 2 * C * LD * 4;
    Chunk<C> *ck = reinterpret_cast<Chunk<C> *>(smem + (kTiles > kTri ? kTiles : kTri));
    auto args = [] { return own_args<Args>(); };
    int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, i = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(tid / 64);
    auto fresh = [&] {   // (no addresses of later steps held from here)
        tid = afresh_lane(tid);
        lane = tid & 63;
        g = lane >> 4;
        i = lane & 15;
    };
    const int64_t total = [&] { const Args a = args(); return a.batch * a.heads * a.chunks; }();
    for (int64_t id = blockIdx.x; id < total; id += gridDim.x) {
        // Heads next to each other: those of a group read the same rows of q and k.
        int chunk;
        Spot p;
        {
            const Args a = args();
            const int64_t bc = id / a.heads;
            chunk = afresh(int(bc % a.chunks));
            p = spot_of(a, unsigned(bc / a.chunks * a.heads + id % a.heads));
        }
        const int t0 = chunk * C, rows = min(C, afresh(int(args().seqlen)) - t0);
        uint32_t gbits = 0, bbits = 0;
        __syncthreads();
        fresh();
        {
            SX sk, sq;
            {
                const Args a = args();
                sk.load(rows_of<T>(a.k, p.b, p.h, a.dk), t0, rows, tid);
            }
            {
                const Args a = args();
                sq.load(rows_of<T>(a.q, p.b, p.h, a.dk), t0, rows, tid);
            }
            if (wave == kWaves - 1) {
                const Args a = args();
                gbits = load_gate<C>(gates_of(a.g, p), t0, t0 + rows, lane);
                bbits = load_gate<C>(gates_of(a.beta, p), t0, t0 + rows, lane);
            }
            sk.store(K, tid);
            sq.store(Q, tid);
        }
        __syncthreads();
        fresh();
        f32x4 n[3], m[3];
        each_tile<C>(wave, [&](auto Lc) {
            typedef decltype(Lc) L;
#pragma unroll
            for (int j = 0; j < L::N; ++j) n[j] = m[j] = f32x4{0.f, 0.f, 0.f, 0.f};
            tile_products<PI, PI, C, KD, L>(n, K, K, lane);
            tile_products<PI, PI, C, KD, L>(m, Q, K, lane);
        });
        if (wave == kWaves - 1) {   // which has the fewest tiles
            const Args a = args();
            make_chunk<C>(*ck, gbits, a.g.type, bbits, a.beta.type, a.scale, lane);
        }
        __syncthreads();
        fresh();
        const float scale = args().scale;
        each_tile<C>(wave, [&](auto Lc) {
            typedef decltype(Lc) L;
            static_for<0, L::N>([&](auto Jc) {
                constexpr int j = decltype(Jc)::value, O = L::O(j), o = L::n(j);
                const f32x4 f = tile_decay<C, false, O, o>(ck->d, 1.f, lane);
                f32x4 x, y;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    x[r] = O != o || 4 * g + r < i ? n[j][r] * f[r] : 0.f;
                    y[r] = O != o || 4 * g + r <= i ? m[j][r] * (f[r] * scale) : 0.f;
                }
                *reinterpret_cast<f32x4 *>(&N[(16 * O + i) * LD + 16 * o + 4 * g]) = x;
                *reinterpret_cast<f32x4 *>(&M[(16 * O + i) * LD + 16 * o + 4 * g]) = y;
            });
        });
        __syncthreads();
        fresh();
        char *ra, *rb;
        {
            const Args a = args();
            const int64_t at = p.bh * a.chunks + chunk;
            ra = afresh(a.rec_a) + at * kRecord<C, REV ? 1 : 2>;
            rb = REV ? afresh(a.rec_b) + at * kRecord<C, 2> : nullptr;
        }
        // Diagonal tiles, one per 16 lanes: a lane has a column. N is 0 from the diagonal on, and so is x. M's image by the other waves
        // meanwhile.
        float x[16], w[16];   // P and B P
        if (wave > 0) {
            write_image<C, REV, kWaves - 1>((REV ? rb : ra) + kImage<C> * 2, M, wave - 1, lane);
        } else if (g < CT) {
            const float *Nd = N + 16 * g * LD + 16 * g, *bt = ck->beta + 16 * g;
            f32x4 n4[2][4];
            float own[2], bs[2];
            auto read = [&](int r) {
#pragma unroll
                for (int k = 0; k < (r + 3) / 4; ++k) n4[r % 2][k] = *reinterpret_cast<const f32x4 *>(Nd + r * LD + 4 * k);
                own[r % 2] = Nd[r * LD + i];
                bs[r % 2] = bt[r];
            };
            read(0);
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                if (r < 15) read(r + 1);
                __builtin_amdgcn_sched_barrier(0);
                float s = -own[r % 2], s2 = 0.f;
#pragma unroll
                for (int k = 0; k < r; ++k) {
                    if (k % 2) s2 = __builtin_fmaf(-n4[r % 2][k / 4][k % 4], w[k], s2);
                    else s = __builtin_fmaf(-n4[r % 2][k / 4][k % 4], w[k], s);
                }
                x[r] = s + s2;
                w[r] = bs[r % 2] * x[r];
            }
        }
        __syncthreads();
        fresh();
        if (wave == 0 && g < CT)
#pragma unroll
            for (int r = 0; r < 16; ++r) P[(16 * g + r) * LD + 16 * g + i] = x[r];
        __syncthreads();
        fresh();
        // The tiles below them, a wave its column block J: P_IJ = (1 + P_II B_I) Y, Y = -(N_IJ + sum over K of N_IK B_K P_KJ).
        auto column = [&](auto Jc) {
            constexpr int J = decltype(Jc)::value;
            auto rows4 = [&](const float *f, int I, int K2) { return *reinterpret_cast<const f32x4 *>(&f[(16 * I + i) * LD + 16 * K2 + 4 * g]); };   // as an A operand
            auto tile = [&](const float *f, int I) {
                f32x4 x;
#pragma unroll
                for (int r = 0; r < 4; ++r) x[r] = f[(16 * I + 4 * g + r) * LD + 16 * J + i];
                return x;
            };
            f32x4 w[CT], bt[CT], y[CT], nn[CT][CT], pp[CT];   // w: B_K P_KJ
#pragma unroll
            for (int I = J; I < CT; ++I) {
                bt[I] = *reinterpret_cast<const f32x4 *>(ck->beta + 16 * I + 4 * g);
                y[I] = tile(I == J ? P : N, I);
                if (I > J) pp[I] = rows4(P, I, I);
#pragma unroll
                for (int K2 = J; K2 < I; ++K2) nn[I][K2] = rows4(N, I, K2);
            }
            w[J] = bt[J] * y[J];
#pragma unroll
            for (int I = J + 1; I < CT; ++I) {
#pragma unroll
                for (int K2 = J; K2 < I; ++K2)
#pragma unroll
                    for (int r = 0; r < 4; ++r) y[I] = __builtin_amdgcn_mfma_f32_16x16x4f32(nn[I][K2][r], w[K2][r], y[I], 0, 0, 0);
                f32x4 z = -y[I];
                const f32x4 v = bt[I] * z;
#pragma unroll
                for (int r = 0; r < 4; ++r) z = __builtin_amdgcn_mfma_f32_16x16x4f32(pp[I][r], v[r], z, 0, 0, 0);
                w[I] = bt[I] * z;
#pragma unroll
                for (int r = 0; r < 4; ++r) P[(16 * I + 4 * g + r) * LD + 16 * J + i] = z[r];
            }
        };
        switch (wave) {
            case 0: column(std::integral_constant<int, 0>{}); break;
            case 1: if constexpr (CT > 2) column(std::integral_constant<int, 1>{}); break;
            case 2: if constexpr (CT > 2) column(std::integral_constant<int, 2>{});
        }
        __syncthreads();
        fresh();
        write_image<C, false>(ra, P, wave, lane);
        write_steps<C>(ra + (REV ? 1 : 2) * kImage<C> * 2, *ck, tid);
        if constexpr (REV) {
            write_image<C, true>(rb, P, wave, lane);
            write_steps<C>(rb + 2 * kImage<C> * 2, *ck, tid);
        }
    }
}

// ---- walks ---------------------------------------------------------------------------------------

// Stage with its pieces' halves swapped by selects, and one address and constants for all pieces of a thread (they are whole blocks of
// 16 rows apart): 100 vector instructions of a walk's chunk less (bfloat16; the other types' stores are the base's).
template <typename T, int C, int D, int NT, bool VEC>
struct Staged : Stage<T, C, D, NT, VEC> {
    typedef Stage<T, C, D, NT, VEC> S;
    __device__ __forceinline__ void store(u16 *tile, int tid) const {
        if constexpr (std::is_same_v<T, bf16_t> && S::RS % 16 == 0 && S::kEven) {
            static_assert(S::VE == 8, "two units of four elements");
            const int row = unsigned(tid) / S::VR, col = unsigned(tid) % S::VR * 8, sw = swizzle(row);
            u16 *dst = tile + row * D + (row >> 4) * 8 + ((((col >> 2) ^ sw) & ~1) << 2);
#pragma unroll
            for (int n = 0; n < S::N; ++n) {
                const uint4 r = S::r[n];
                const uint64_t lo = uint64_t(r.y) << 32 | r.x, hi = uint64_t(r.w) << 32 | r.z, x = sw & 1 ? hi : lo, y = sw & 1 ? lo : hi;
                *reinterpret_cast<uint4 *>(dst + n * (S::RS * D + S::RS / 16 * 8)) = make_uint4(uint32_t(x), uint32_t(x >> 32), uint32_t(y), uint32_t(y >> 32));
            }
        } else {
            S::store(tile, tid);
        }
    }
};
// A record on its way from memory to LDS.
template <int BYTES>
struct StageRecord {
    static constexpr int N = (BYTES / 16 + kThreads - 1) / kThreads;
    uint4 r[N];
    __device__ __forceinline__ void load(const char *src, int tid) {
        const __amdgpu_buffer_rsrc_t buf = buffer(src);
#pragma unroll
        for (int n = 0; n < N; ++n) {
            uint32_t at = uint32_t((n * kThreads + tid) * 16);
            if ((n + 1) * kThreads * 16 > BYTES && at >= uint32_t(BYTES)) at = kNone;
            asm("" : "+v"(at));
            r[n] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(buf, at, 0, 0));
        }
    }
    // The first image and the last `STEPS` bytes of a record of `size` bytes.
    template <int STEPS>
    __device__ __forceinline__ void load_ends(const char *src, int size, int tid) {
        const __amdgpu_buffer_rsrc_t buf = buffer(src);
#pragma unroll
        for (int n = 0; n < N; ++n) {
            uint32_t at = uint32_t((n * kThreads + tid) * 16);
            if ((n + 1) * kThreads * 16 > BYTES - STEPS) at = at < uint32_t(BYTES - STEPS) ? at : at < uint32_t(BYTES) ? at + uint32_t(size - BYTES) : kNone;
            asm("" : "+v"(at));
            r[n] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(buf, at, 0, 0));
        }
    }
    __device__ __forceinline__ void store(char *dst, int tid) const {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int at = (n * kThreads + tid) * 16;
            if ((n + 1) * kThreads * 16 <= BYTES || at < BYTES) *reinterpret_cast<uint4 *>(dst + at) = r[n];
        }
    }
};

// A workgroup's (pair, segment, slice). Slices of one segment read the same q, k and records: they are 8 ids apart, which is one XCD and
// its L2.
struct Unit {
    unsigned pair, seg, slice;
    bool live;
};
__device__ __forceinline__ Unit unit_of(const Args &a, unsigned slices) {
    const unsigned id = blockIdx.x, per = 8u * slices, in = id % per, ps = id / per * 8u + in % 8u;
    Unit u;
    u.pair = ps / unsigned(a.segs);
    u.seg = ps % unsigned(a.segs);
    u.slice = in / 8u;
    u.live = ps < unsigned(a.batch * a.heads) * unsigned(a.segs);
    return u;
}
inline int64_t unit_grid(const Args &a, int slices) { return (a.batch * a.heads * a.segs + 7) / 8 * 8 * slices; }

// Two workgroups on a CU: of two waves that could issue the older one does, so that one workgroup runs ahead and leaves the other its CU
// alone at the end. A wave gives way with every quarter of its chunks that it has done (of `n`): 64 pairs of 128 x 128 in four segments of
// 1,024 tokens, two groups on every CU: 142 us where the older one's way took 153, prompts of 160 pairs in one piece 491 and 523.
struct Turns {
    int quarter, left;
    __device__ __forceinline__ void start(int n) {
        quarter = afresh((n + 3) / 4);
        left = 4 * quarter;
        __builtin_amdgcn_s_setprio(3);
    }
    __device__ __forceinline__ void step() {
        --left;
        if (left == 3 * quarter) __builtin_amdgcn_s_setprio(2);
        if (left == 2 * quarter) __builtin_amdgcn_s_setprio(1);
        if (left == quarter) __builtin_amdgcn_s_setprio(0);
    }
};

// The wave's outputs of a chunk. Whole 16-byte pieces leave by way of its own columns of V, which no other wave reads (see
// store_out); they are held until the next chunk's rows are staged, so that those wait for no store.
template <typename T, int C, int LDV, bool VEC>
struct HeldOut {
    static constexpr bool kPieces = VEC && sizeof(T) == 2;
    static constexpr int CT = C / 16, NP = kPieces ? C * 2 / 64 : 1;
    u32x4 w[NP];
    f32x4 o[kPieces ? 1 : CT];
    int rows;

    __device__ __forceinline__ void take(const f32x4 (&O)[CT][1], u16 *tile, int r, int col, int lane) {
        rows = r;
        if constexpr (kPieces) {
            const int g = lane >> 4, i = lane & 15;
            wave_fence();
#pragma unroll
            for (int t = 0; t < CT; ++t)
#pragma unroll
                for (int e = 0; e < 4; e += 2) {
                    const uint32_t x = std::is_same_v<T, bf16_t> ? pack_bf16x2(O[t][0][e], O[t][0][e + 1]) : pack_f16x2(O[t][0][e], O[t][0][e + 1]);
                    tile[block<LDV>(16 * t) + at<LDV>(4 * g + e, col + i)] = u16(x);
                    tile[block<LDV>(16 * t) + at<LDV>(4 * g + e + 1, col + i)] = u16(x >> 16);
                }
            wave_fence();
#pragma unroll
            for (int n = 0; n < NP; ++n) {
                const u16 *src = tile + block<LDV>(32 * n);
                const int row = lane / 2, c = lane % 2 * 8;
                const uint2 a = *reinterpret_cast<const uint2 *>(src + at<LDV>(row, col + c)), b = *reinterpret_cast<const uint2 *>(src + at<LDV>(row, col + c + 4));
                w[n] = u32x4{a.x, a.y, b.x, b.y};
            }
        } else {
#pragma unroll
            for (int t = 0; t < CT; ++t) o[t] = O[t][0];
        }
    }
    // The rows from token t0 on; stride in elements, `cols` of the row exist.
    __device__ __forceinline__ void flush(char *out, uint32_t stride, int t0, int cols, int col, int lane) const {
        const __amdgpu_buffer_rsrc_t buf = buffer(out + uint64_t(unsigned(t0)) * stride * sizeof(T));
        if constexpr (kPieces) {
#pragma unroll
            for (int n = 0; n < NP; ++n) {
                const int row = 32 * n + lane / 2, c = col + lane % 2 * 8;
                __builtin_amdgcn_raw_buffer_store_b128(w[n], buf, row < rows && c < cols ? uint32_t(row) * stride * 2 + uint32_t(c) * 2 : kNone, 0, 0);
            }
        } else {
            const int g = lane >> 4, x = col + (lane & 15);
#pragma unroll
            for (int t = 0; t < CT; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int n = 16 * t + 4 * g + r;
                    store_element<T, false>(o[t][r], buf, n < rows && x < cols ? uint32_t(n) * stride + uint32_t(x) : kNone);
                }
        }
    }
};

// X = diag(wx) A S and, with TWO, O = diag(wo) B S for the wave's columns; the state is split once for both.
template <typename T, int C, int KD, bool TWO>
__device__ __forceinline__ void state_products(f32x4 (&X)[C / 16][1], f32x4 (&O)[C / 16][1], const f32x4 (&S)[KD / 16][1], const u16 *A, const u16 *B,
                                               const float *wx, const float *wo, int lane) {
    constexpr int PL = kTile<C, KD>, PI = Cfg<T>::in, CT = C / 16, STEPS = KD / 32 * (TWO ? 2 : 1);
    const int g = lane >> 4, i = lane & 15;
#pragma unroll
    for (int t = 0; t < CT; ++t) X[t][0] = O[t][0] = f32x4{0.f, 0.f, 0.f, 0.f};
    // The next step's rows are read while the products of this one run.
    bf16x8 a[2][CT][PI];
    auto read = [&](int n) {
        const u16 *tile = TWO && n % 2 ? B : A;
        const int k = TWO ? n / 2 : n;
#pragma unroll
        for (int t = 0; t < CT; ++t)
#pragma unroll
            for (int p = 0; p < PI; ++p) a[n % 2][t][p] = frag_row<KD>(tile + p * PL, 16 * t, k, g, i);
    };
    auto split = [&](int k, bf16x8 (&s)[kPlanes]) {
        float x[8];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            x[r] = S[2 * k][0][r];
            x[4 + r] = S[2 * k + 1][0][r];
        }
        split8(x, s);
    };
    read(0);
    bf16x8 s[2][kPlanes];
    split(0, s[0]);
#pragma unroll
    for (int n = 0; n < STEPS; ++n) {
        const int k = TWO ? n / 2 : n;
        if (n + 1 < STEPS) read(n + 1);
        const bool ahead = k + 1 < KD / 32 && (!TWO || n % 2 == 0);
        if (ahead) split(k + 1, s[(k + 1) % 2]);
#pragma unroll
        for (int p = 0; p < PI; ++p)
#pragma unroll
            for (int q = 0; q < kPlanes; ++q)
                if (p + q < kPlanes)
#pragma unroll
                    for (int t = 0; t < CT; ++t) {
                        f32x4 &to = TWO && n % 2 ? O[t][0] : X[t][0];
                        to = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[n % 2][t][p], s[k % 2][q], to, 0, 0, 0);
                    }
        // The next operands' reads first; then the products with the state's next split between them, a product's time each.
        __builtin_amdgcn_sched_group_barrier(0x100, 4 * CT * PI, 0);
#pragma unroll
        for (int m = 0; m < CT * (PI == 1 ? 3 : PI == 2 ? 5 : 6); ++m) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x002, 4, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int t = 0; t < CT; ++t) {
        const f32x4 f = *reinterpret_cast<const f32x4 *>(wx + 16 * t + 4 * g);
#pragma unroll
        for (int r = 0; r < 4; ++r) X[t][0][r] *= f[r];
        if constexpr (TWO) {
            const f32x4 h = *reinterpret_cast<const f32x4 *>(wo + 16 * t + 4 * g);
#pragma unroll
            for (int r = 0; r < 4; ++r) O[t][0][r] *= h[r];
        }
    }
}

// A chunk's tokens one by one, as the recurrence says. out(t, c, the column's q S) in every lane.
template <typename T, int C, int KD, int NC, int LDV, typename F>
__device__ __forceinline__ void recur_delta(f32x4 (&S)[KD / 16][NC], const u16 *Q, const u16 *K, const u16 *V, const Steps<C> &ck, int rows, int kdim,
                                            int col, int lane, F &&out) {
#pragma unroll 1
    for (int t = 0; t < rows; ++t) {
        lane = afresh_lane(lane);
        const int g = lane >> 4, i = lane & 15;
        const float e = exp_f32(t ? (ck.hi[t] - ck.hi[t - 1]) + (ck.lo[t] - ck.lo[t - 1]) : ck.hi[0] + ck.lo[0]);
        float z[NC], o[NC];
#pragma unroll
        for (int c = 0; c < NC; ++c) z[c] = o[c] = 0.f;
#pragma unroll
        for (int k = 0; k < KD / 16; ++k) {
            kdim = afresh(kdim);   // (no masks of all rows held at once)
            float y[4];
            tile_row4<T, C, KD>(y, K, t, 16 * k + 4 * g);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const bool in = 16 * k + 4 * g + r < kdim;
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    S[k][c][r] = in ? e * S[k][c][r] : 0.f;
                    z[c] += in ? y[r] * S[k][c][r] : 0.f;
                }
            }
        }
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            z[c] += __shfl_xor(z[c], 16);
            z[c] += __shfl_xor(z[c], 32);
            z[c] = (tile_at<T, C, LDV>(V, t, col + 16 * c + i) - z[c]) * ck.beta[t];
        }
#pragma unroll
        for (int k = 0; k < KD / 16; ++k) {
            kdim = afresh(kdim);
            float y[4], x[4];
            tile_row4<T, C, KD>(y, K, t, 16 * k + 4 * g);
            tile_row4<T, C, KD>(x, Q, t, 16 * k + 4 * g);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const bool in = 16 * k + 4 * g + r < kdim;
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    S[k][c][r] = in ? __builtin_fmaf(y[r], z[c], S[k][c][r]) : 0.f;
                    o[c] += in ? x[r] * S[k][c][r] : 0.f;
                }
            }
        }
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            o[c] += __shfl_xor(o[c], 16);
            o[c] += __shfl_xor(o[c], 32);
            out(t, c, o[c]);
        }
    }
}

// The state that a unit starts from.
template <int KD>
__device__ __forceinline__ void start_state(f32x4 (&S)[KD / 16][1], const Args &a, const Spot &p, int seg, int col0, int col, int lane) {
    if (a.segs > 1) {
        const int vd = 64 * a.slices;
        load_state<KD, 1>(S, Mat{a.starts + (int64_t(p.bh) * a.segs + seg) * KD * vd + col0, vd, 1}, KD, 64, col, lane);
    } else {
        load_state<KD, 1>(S, Mat{const_cast<float *>(a.s0 ? a.s0 + int64_t(p.bh) * a.dk * a.dv + col0 : nullptr), a.dv, 1}, a.dk, a.dv - col0, col, lane);
    }
}

// What an infinity or NaN reaches is not what the chunks' products make of it (their planes and masked zeros make NaN of more). A walk
// that met one is followed by this: the recurrence once more from its start, whose outputs from the wave's first such chunk on (`first`),
// and state, take the others' place. Its arguments are read again, so that nothing of it takes registers while the products run.
template <typename T, int KD, bool VEC>
__device__ __forceinline__ void infinite_rows(f32x4 (&S)[KD / 16][1], char *smem, int beg, int end, int first) {
    constexpr int C = Cfg<T>::C, PI = Cfg<T>::in, W = 64;
    auto args = [] { return own_args<Args>(); };
    u16 *K = reinterpret_cast<u16 *>(smem), *Q = K + PI * kTile<C, KD>, *V = Q + PI * kTile<C, KD>;
    Steps<C> &ck = *reinterpret_cast<Steps<C> *>(V + PI * kTile<C, W>);
    const int tid = afresh_lane(threadIdx.x), wave = __builtin_amdgcn_readfirstlane(tid / 64), lane = tid & 63, col = wave * 16;
    const Unit u = unit_of(args(), args().slices);
    const Spot p = spot_of(args(), u.pair);
    const int col0 = int(u.slice) * W;
    f32x4 R[KD / 16][1];
    start_state<KD>(R, args(), p, u.seg, col0, col, lane);
    __threadfence();   // the outputs that are stored once more
#pragma unroll 1
    for (int t0 = beg; t0 < end; t0 += C) {
        const Args a = args();
        const int rows = min(C, end - t0);
        __syncthreads();
        {
            Stage<T, C, KD, kThreads, VEC> s;
            s.load(rows_of<T>(a.k, p.b, p.h, a.dk), t0, rows, tid);
            s.store(K, tid);
            s.load(rows_of<T>(a.q, p.b, p.h, a.dk), t0, rows, tid);
            s.store(Q, tid);
        }
        {
            Stage<T, C, W, kThreads, VEC> s;
            s.load(rows_of<T>(a.v, p.b, p.h, a.dv, col0), t0, rows, tid);
            s.store(V, tid);
        }
        const float *steps = reinterpret_cast<const float *>(a.rec_a + (int64_t(p.bh) * a.chunks + t0 / C + 1) * kRecord<C, 2> - sizeof(Steps<C>));
        for (int x = tid; x < int(sizeof(Steps<C>)) / 4; x += kThreads) reinterpret_cast<float *>(&ck)[x] = steps[x];
        __syncthreads();
        const __amdgpu_buffer_rsrc_t to = buffer(static_cast<char *>(a.out) + (p.b * a.out_batch + p.h * a.out_head + t0 * a.out_seq + col0) * int64_t(sizeof(T)));
        recur_delta<T, C, KD, 1, W>(R, Q, K, V, ck, rows, a.dk, col, lane, [&](int t, int, float x) {
            const int at = col + (lane & 15);
            store_element<T, false>(x * a.scale, to, t0 >= first && lane < 16 && at < a.dv - col0 ? uint32_t(t) * uint32_t(a.out_seq) + uint32_t(at) : kNone);
        });
        // A state that is NaN throughout stays so, and so did the walk's.
        bool lost = true;
        const int dk = afresh(a.dk), g = lane >> 4;
#pragma unroll
        for (int k = 0; k < KD / 16; ++k)
#pragma unroll
            for (int r = 0; r < 4; ++r) lost &= R[k][0][r] != R[k][0][r] || 16 * k + 4 * g + r >= dk;
        if (__syncthreads_and(lost || first >= end || col + (lane & 15) >= a.dv - col0)) break;
    }
    if (first < end)
#pragma unroll
        for (int k = 0; k < KD / 16; ++k) S[k][0] = R[k][0];
}

// What a walk leaves.
enum Leaves {
    kOutputs,   // outputs, and the last state
    kStates,    // the state before every chunk, and Z (the backward's)
    kMaps       // of a segment: what it adds to the state (V's columns) and what it makes of it (as many columns as rows, from the identity)
};

// The state's way through a segment's chunks, a workgroup 64 columns of it, a wave 16. A chunk's steps hang on each other (split the state,
// K S and Q S, split, P, split, M, the update), so that latency bounds it: at dk 128 in bfloat16 4.6 us per chunk where a workgroup is alone on its
// CU (10,300 cycles, the matrix cores busy for 3,456), 7.7 to 8.9 where two are; 160 pairs of 128 x 128, L 4,096: 491 us. Both
// 64-column halves of a head in one workgroup of eight waves, with one staging: at most 8 % less, 2 % of a training step.
template <typename T, int KD, Leaves L, bool VEC>
__global__ void __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(2, 2))) dr_walk(const Args) {
    constexpr int C = Cfg<T>::C, PI = Cfg<T>::in, W = 64, NC = 1, CT = C / 16;
    constexpr bool kOut = L == kOutputs;
    constexpr int kLoaded = kRecord<C, kOut ? 2 : 1>;
    typedef Staged<T, C, KD, kThreads, VEC> SX;
    typedef Staged<T, C, W, kThreads, VEC> SV;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    u16 *K = reinterpret_cast<u16 *>(smem), *Q = K + PI * kTile<C, KD>, *V = kOut ? Q + PI * kTile<C, KD> : Q;
    u16 *img = V + PI * kTile<C, W>;
    const Steps<C> &ck = *reinterpret_cast<const Steps<C> *>(img + (kOut ? 2 : 1) * kImage<C>);

    int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid / 64), col = wave * 16 * NC;
    auto fresh = [&] {
        tid = afresh_lane(tid);
        lane = tid & 63;
    };
    auto args = [] { return own_args<Args>(); };
    const Unit u = unit_of(args(), L == kMaps ? args().slices + KD / 64 : args().slices);
    if (!u.live) return;
    const Spot p = spot_of(args(), u.pair);
    const int col0 = afresh(int(u.slice) * W);
    int beg, end;
    {
        const Args a = args();
        beg = afresh(int(u.seg) * int(a.seg_len));
        end = afresh(min(int(a.seqlen), beg + int(a.seg_len)));
        if constexpr (kOut) {
            // A state that is not finite goes through its row in one piece, as the recurrence does.
            if (a.segs > 1 && a.flags[p.bh]) {
                if (u.seg) return;
                end = afresh(int(a.seqlen));
            }
        }
        // What the last segment adds is nobody's start; what it makes of the state is, in the backward.
        if (L == kMaps && u.seg + 1 == unsigned(a.segs) && (!a.last_map || int(u.slice) < a.slices)) return;
    }
    f32x4 S[KD / 16][NC];
    {
        const Args a = args();
        if (L == kMaps) {
            const int j0 = col0 - 64 * a.slices + col;
#pragma unroll
            for (int k = 0; k < KD / 16; ++k)
#pragma unroll
                for (int r = 0; r < 4; ++r) S[k][0][r] = j0 >= 0 && 16 * k + 4 * (lane >> 4) + r == j0 + (lane & 15) ? 1.f : 0.f;
        } else {
            start_state<KD>(S, a, p, u.seg, col0, col, lane);
        }
    }
    auto tensor = [&](auto of) { const Args a = args(); return of(a); };
    const Rows<T> rk = tensor([&](const Args &a) { return rows_of<T>(a.k, p.b, p.h, a.dk); });
    const Rows<T> rq = kOut ? tensor([&](const Args &a) { return rows_of<T>(a.q, p.b, p.h, a.dk); }) : rk;
    const Rows<T> rv = tensor([&](const Args &a) { return rows_of<T>(a.v, p.b, p.h, a.dv, col0); });
    const int stride = kOut ? kRecord<C, 2> : afresh(args().rec_a_step);
    const char *records = tensor([&](const Args &a) { return afresh(a.rec_a + int64_t(p.bh) * a.chunks * a.rec_a_step); });
    char *const out = tensor([&](const Args &a) {
        return kOut ? afresh(static_cast<char *>(a.out) + (p.b * a.out_batch + p.h * a.out_head + col0) * int64_t(sizeof(T))) : nullptr;
    });
    const uint32_t out_stride = uint32_t(afresh(int(args().out_seq)));

    SX sk, sq;
    SV sv;
    StageRecord<kLoaded> si;
    auto load_rows = [&](int t0) {
        const int rows = min(C, end - t0);
        sk.load(rk, t0, rows, tid);
        if constexpr (kOut) sq.load(rq, t0, rows, tid);
        sv.load(rv, t0, rows, tid);
    };
    auto load_record = [&](int t0) {
        // P and the steps; in the forward's records M lies between.
        if constexpr (kOut) si.load(records + int64_t(t0 / C) * stride, tid);
        else si.template load_ends<int(sizeof(Steps<C>))>(records + int64_t(t0 / C) * stride, stride, tid);
    };
    load_record(beg);
    load_rows(beg);
    HeldOut<T, C, W, VEC> held;
    int first_odd = 0x7fffffff;   // the first chunk with something not finite in it
    Turns turns;   // (of aligned rows: the element-wise loads have no scalars left for it)
    if constexpr (VEC) turns.start((end - beg + C - 1) / C);
    for (int t0 = beg; t0 < end; t0 += C) {
        const int rows = min(C, end - t0);
        if constexpr (VEC) turns.step();
        __syncthreads();
        fresh();
        sk.store(K, tid);
        if constexpr (kOut) sq.store(Q, tid);
        sv.store(V, tid);
        si.store(reinterpret_cast<char *>(img), tid);
        if constexpr (kOut)
            if (t0 > beg) held.flush(out, out_stride, t0 - C, rv.d, col, lane);
        if (t0 + C < end) load_rows(t0 + C);
        __syncthreads();
        fresh();
        if constexpr (L == kStates) {
            const Args a = args();
            const int vd = 64 * a.slices;
            store_state<KD, NC>(S, Mat{a.states + (int64_t(p.bh) * a.chunks + t0 / C) * KD * vd + col0, vd, 1}, KD, W, col, lane);
        }
        f32x4 X[CT][NC], O[CT][NC];
        state_products<T, C, KD, kOut>(X, O, S, K, Q, ck.in, ck.inq, lane);
        tile_columns<T, C, NC, W>(V, col, lane, [&](int j, int c, const float *v) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                X[2 * j][c][r] = v[r] - X[2 * j][c][r];
                X[2 * j + 1][c][r] = v[4 + r] - X[2 * j + 1][c][r];
            }
        });
        fresh();
        bf16x8 f[C / 32][NC][kPlanes];
        split_rows<C, NC>(f, X, ck.beta, lane);
        triangle<C, NC, true, kPlanes>(X, img, f, lane);   // Z
        const int g = lane >> 4;
        if constexpr (L == kStates) {
            const Args a = args();
            const int vd = 64 * a.slices;
            const __amdgpu_buffer_rsrc_t to = buffer(a.z + (int64_t(p.bh) * a.chunks * C + t0) * vd + col0 + col);
#pragma unroll
            for (int t = 0; t < CT; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(X[t][0][r]), to, uint32_t((16 * t + 4 * g + r) * vd + (lane & 15)) * 4, 0, 0);
        }
#pragma unroll
        for (int t = 0; t < CT; ++t) {
            const f32x4 b = *reinterpret_cast<const f32x4 *>(ck.beta + 16 * t + 4 * g);
            X[t][0] *= b;   // U
        }
        if constexpr (kOut) {
            bf16x8 w[C / 32][NC][kPlanes];
#pragma unroll
            for (int j = 0; j < C / 32; ++j) {
                float y[8];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    y[r] = X[2 * j][0][r];
                    y[4 + r] = X[2 * j + 1][0][r];
                }
                split8(y, w[j][0]);
            }
            triangle<C, NC, true, kPlanes>(O, img + kImage<C>, w, lane);
            // 0 times what is not finite is not 0. (A row of U that is not finite is in its own row tile's products, and makes NaN of them.)
            float nan = 0.f;
#pragma unroll
            for (int t = 0; t < CT; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) nan = __builtin_fmaf(O[t][0][r], 0.f, nan);
            if (first_odd > t0 && __any(!(nan == 0.f))) first_odd = t0;
        }
        if (t0 + C < end) load_record(t0 + C);
        split_rows<C, NC>(f, X, ck.out, lane);
        const float all = ck.all;
#pragma unroll
        for (int k = 0; k < KD / 16; ++k) S[k][0] *= all;
        add_rows<T, C, KD, NC>(S, K, f, lane);
        fresh();
        if constexpr (kOut) held.take(O, V, rows, col, lane);
    }
    if constexpr (kOut) {
        held.flush(out, out_stride, beg + (end - 1 - beg) / C * C, rv.d, col, lane);
        if (__syncthreads_or(first_odd < end)) infinite_rows<T, KD, VEC>(S, smem, beg, end, first_odd);
    }
    const Args a = args();
    if constexpr (kOut) {
        if (a.s1 && end == int(a.seqlen)) store_state<KD, NC>(S, Mat{a.s1 + int64_t(p.bh) * a.dk * a.dv + col0, a.dv, 1}, a.dk, a.dv - col0, col, lane);
    }
    if constexpr (L == kMaps) {
        const int md = 64 * a.slices + KD;
        store_state<KD, NC>(S, Mat{a.maps + (int64_t(p.bh) * a.segs + u.seg) * KD * md + col0, md, 1}, KD, W, col, lane);
        if (u.seg == 0 && u.slice == 0 && tid == 0) a.flags[p.bh] = 0;
    }
}

// The state's gradient R back through a segment's chunks: dV, dbeta's shares, R at every chunk's end, and the first state's gradient.
// MAPS: what a segment adds to R alone. Bound as dr_walk is, with the states' gradients and dV's float32 rows stored beside it: 64 pairs of
// 128 x 128, L 4,096, four segments, bfloat16: 216 us, the maps 143.
template <typename T, int KD, bool MAPS, bool VEC>
__global__ void __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(2, 2))) dr_back(const Args) {
    constexpr int C = Cfg<T>::C, PI = Cfg<T>::in, W = 64, NC = 1, CT = C / 16;
    constexpr int kRec = kRecord<C, 2>;
    typedef Staged<T, C, KD, kThreads, VEC> SX;
    typedef Staged<T, C, W, kThreads, VEC> SV;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    u16 *K = reinterpret_cast<u16 *>(smem), *Q = K + PI * kTile<C, KD>, *V = Q + PI * kTile<C, KD>;
    u16 *img = V + PI * kTile<C, W>;
    const Steps<C> &ck = *reinterpret_cast<const Steps<C> *>(img + 2 * kImage<C>);
    float *part = reinterpret_cast<float *>(reinterpret_cast<char *>(img) + kRec);   // [wave][C]

    int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid / 64), col = wave * 16 * NC;
    auto fresh = [&] {
        tid = afresh_lane(tid);
        lane = tid & 63;
    };
    auto args = [] { return own_args<Args>(); };
    const Unit u = unit_of(args(), args().slices);
    if (!u.live || (MAPS && u.seg == 0)) return;
    const Spot p = spot_of(args(), u.pair);
    const int col0 = afresh(int(u.slice) * W);
    int beg, end;
    {
        const Args a = args();
        beg = afresh(int(u.seg) * int(a.seg_len));
        end = afresh(min(int(a.seqlen), beg + int(a.seg_len)));
    }
    const int first = beg / C, last = (end - 1) / C;
    f32x4 R[KD / 16][NC];
    {
        const Args a = args();
        if (MAPS) {
            load_state<KD, NC>(R, Mat{nullptr, 0, 1}, 0, 0, col, lane);
        } else if (a.segs > 1) {
            const int vd = 64 * a.slices;
            load_state<KD, NC>(R, Mat{a.back_starts + (int64_t(p.bh) * a.segs + u.seg) * KD * vd + col0, vd, 1}, KD, W, col, lane);
        } else {
            load_state<KD, NC>(R, Mat{const_cast<float *>(a.dlast ? a.dlast + int64_t(p.bh) * a.dk * a.dv + col0 : nullptr), a.dv, 1}, a.dk, a.dv - col0, col, lane);
        }
    }
    auto tensor = [&](auto of) { const Args a = args(); return of(a); };
    const Rows<T> rk = tensor([&](const Args &a) { return rows_of<T>(a.k, p.b, p.h, a.dk); });
    const Rows<T> rq = tensor([&](const Args &a) { return rows_of<T>(a.q, p.b, p.h, a.dk); });
    const Rows<T> rd = tensor([&](const Args &a) { return rows_of<T>(a.dout, p.b, p.h, a.dv, col0); });
    const char *records = tensor([&](const Args &a) { return afresh(a.rec_b + int64_t(p.bh) * a.chunks * kRec); });
    char *const out = tensor([&](const Args &a) {
        return afresh(static_cast<char *>(a.out) + (p.b * a.out_batch + p.h * a.out_head + col0) * int64_t(sizeof(T)));
    });
    const uint32_t out_stride = uint32_t(afresh(int(args().out_seq)));
    SX sk, sq;
    SV sd;
    StageRecord<kRec> si;
    auto load = [&](int n) {
        const int t0 = n * C, rows = min(C, end - t0);
        sk.load(rk, t0, rows, tid);
        si.load(records + int64_t(n) * kRec, tid);
        sq.load(rq, t0, rows, tid);
        sd.load(rd, t0, rows, tid);
    };
    load(last);
    HeldOut<T, C, W, VEC> held;
    Turns turns;
    if constexpr (VEC) turns.start(last - first + 1);
    for (int n = last; n >= first; --n) {
        const int t0 = n * C, rows = min(C, end - t0);
        if constexpr (VEC) turns.step();
        __syncthreads();
        fresh();
        sk.store(K, tid);
        si.store(reinterpret_cast<char *>(img), tid);
        sq.store(Q, tid);
        sd.store(V, tid);
        f32x4 Z[CT][NC];
        const int g = lane >> 4;
        if constexpr (!MAPS) {
            const Args a = args();
            const int vd = 64 * a.slices;
            const __amdgpu_buffer_rsrc_t from = buffer(a.z + (int64_t(p.bh) * a.chunks * C + t0) * vd + col0 + col);
#pragma unroll
            for (int t = 0; t < CT; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    Z[t][0][r] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(from, uint32_t((16 * t + 4 * g + r) * vd + (lane & 15)) * 4, 0, 0));
            if (n < last) held.flush(out, out_stride, t0 + C, rd.d, col, lane);
            store_state<KD, NC>(R, Mat{a.r + (int64_t(p.bh) * a.chunks + n) * KD * vd + col0, vd, 1}, KD, W, col, lane);
        }
        if (n > first) load(n - 1);
        __syncthreads();
        fresh();
        f32x4 G[CT][NC], none[CT][NC];
        state_products<T, C, KD, false>(G, none, R, K, K, ck.out, ck.out, lane);
        bf16x8 d[C / 32][NC][PI];
        load_v<T, C, NC, W>(d, V, col, lane);
        triangle<C, NC, false, PI>(G, img + kImage<C>, d, lane);   // dU
        fresh();
        bf16x8 f[C / 32][NC][kPlanes];
        split_rows<C, NC>(f, G, ck.beta, lane);
        triangle<C, NC, false, kPlanes>(G, img, f, lane);          // G
#pragma unroll
        for (int t = 0; t < CT; ++t) {
            const f32x4 b = *reinterpret_cast<const f32x4 *>(ck.beta + 16 * t + 4 * g);
            if constexpr (!MAPS) {
                f32x4 s = G[t][0] * Z[t][0];
#pragma unroll
                for (int r = 0; r < 4; ++r) s[r] = group_sum<16>(s[r]);
                if ((lane & 15) == 0) *reinterpret_cast<f32x4 *>(part + wave * C + 16 * t + 4 * g) = s;
            }
            G[t][0] *= b;   // dV
        }
        if constexpr (!MAPS) {
            const Args a = args();
            const int vd = 64 * a.slices;
            const __amdgpu_buffer_rsrc_t to = buffer(a.dx + (int64_t(p.bh) * a.chunks * C + t0) * vd + col0 + col);
#pragma unroll
            for (int t = 0; t < CT; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(G[t][0][r]), to, uint32_t((16 * t + 4 * g + r) * vd + (lane & 15)) * 4, 0, 0);
        }
        // R = e^c_end R + Q^T (scale e^c dO) - K^T (e^c dV)
        update<T, C, KD, NC>(R, d, Q, ck.inq, ck.all, lane);
        {
            f32x4 y[CT][NC];
#pragma unroll
            for (int t = 0; t < CT; ++t) y[t][0] = -G[t][0];
            split_rows<C, NC>(f, y, ck.in, lane);
        }
        add_rows<T, C, KD, NC>(R, K, f, lane);
        fresh();
        if constexpr (!MAPS) {
            held.take(G, V, rows, col, lane);
            __syncthreads();
            if (tid < C) {
                float s = 0.f;
#pragma unroll
                for (int w = 0; w < kWaves; ++w) s += part[w * C + tid];
                const Args a = args();
                a.pbeta[(int64_t(u.slice) * a.batch * a.heads + p.bh) * a.chunks * C + t0 + tid] = s;
            }
        }
    }
    const Args a = args();
    if constexpr (MAPS) {
        const int vd = 64 * a.slices;
        store_state<KD, NC>(R, Mat{a.back_maps + (int64_t(p.bh) * a.segs + u.seg) * KD * vd + col0, vd, 1}, KD, W, col, lane);
    } else {
        held.flush(out, out_stride, first * C, rd.d, col, lane);
        if (a.ds0 && u.seg == 0) store_state<KD, NC>(R, Mat{a.ds0 + int64_t(p.bh) * a.dk * a.dv + col0, a.dv, 1}, a.dk, a.dv - col0, col, lane);
    }
}

// The segments' maps (B | A: what they add, what they make of the state) into the states that they start from; BACK: into R at their ends,
// by the transposes of A. One workgroup per 32 columns of a (batch row, head); its waves split the rows, in float32 on
// v_mfma_f32_16x16x4_f32, the next segment's map on its way meanwhile. A row that holds something not finite is flagged. A chain of one step per
// segment, whatever the pairs: some 6 us a step at dk 128 (four segments of 64 pairs: 22 us), 1.6 at 64 (21 segments of 24 pairs: 35 us);
// three or five maps on their way took as long.
template <int KD, bool BACK>
__global__ void __launch_bounds__(kThreads) dr_join(const Args) {
    constexpr int NT = KD / 64, NC = 2;   // tiles of 16 rows, of 16 columns per wave
    __shared__ float S[2][KD][16 * NC + 4];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / 64), lane = tid & 63, g = lane >> 4, i = lane & 15;
    const Args a = own_args<Args>();
    const int vd = 64 * a.slices, md = vd + KD, segs = a.segs, groups = vd / (16 * NC), row0 = 16 * wave * NT;
    const int64_t bh = blockIdx.x / groups;
    const int col = int(blockIdx.x % groups) * 16 * NC;
    const float *edge = BACK ? a.dlast : a.s0;
    float *starts = (BACK ? a.back_starts : a.starts) + bh * segs * KD * vd;
    const float *maps = a.maps + bh * segs * KD * md, *adds = BACK ? a.back_maps + bh * segs * KD * vd : maps;
    const int ad = BACK ? vd : md;
    float nan = 0.f;
    f32x4 x[NT][NC], add[NT][NC], ma[NT][KD / 16];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int row = row0 + 16 * t + 4 * g + r, v = col + 16 * c + i;
                x[t][c][r] = edge && row < a.dk && v < a.dv ? edge[bh * a.dk * a.dv + int64_t(row) * a.dv + v] : 0.f;
            }
    auto load = [&](int seg) {
        const float *m = maps + int64_t(seg) * KD * md + vd, *b = adds + int64_t(seg) * KD * ad + col;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int at = row0 + 16 * t;
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int r = 0; r < 4; ++r) add[t][c][r] = b[(at + 4 * g + r) * ad + 16 * c + i];
#pragma unroll
            for (int k = 0; k < KD / 16; ++k) {
                if constexpr (BACK) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) ma[t][k][r] = m[(16 * k + 4 * g + r) * md + at + i];
                } else {
                    ma[t][k] = *reinterpret_cast<const f32x4 *>(m + (at + i) * md + 16 * k + 4 * g);
                }
            }
        }
    };
    load(BACK ? segs - 1 : 0);
    for (int n = 0; n < segs; ++n) {
        const int seg = BACK ? segs - 1 - n : n;
        auto s = S[n % 2];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int row = row0 + 16 * t + 4 * g + r;
                    s[row][16 * c + i] = x[t][c][r];
                    starts[(int64_t(seg) * KD + row) * vd + col + 16 * c + i] = x[t][c][r];
                    nan = __builtin_fmaf(x[t][c][r], 0.f, nan);
                }
        if (n + 1 == segs) break;
        f32x4 m[NT][KD / 16];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
#pragma unroll
            for (int c = 0; c < NC; ++c) x[t][c] = add[t][c];
#pragma unroll
            for (int k = 0; k < KD / 16; ++k) m[t][k] = ma[t][k];
        }
        if (n + 2 < segs) load(BACK ? seg - 1 : seg + 1);
        __syncthreads();
#pragma unroll
        for (int k = 0; k < KD / 16; ++k)
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    const float b = s[16 * k + 4 * g + r][16 * c + i];
#pragma unroll
                    for (int t = 0; t < NT; ++t) x[t][c] = __builtin_amdgcn_mfma_f32_16x16x4f32(m[t][k][r], b, x[t][c], 0, 0, 0);
                }
    }
    if (!BACK && !(nan == 0.f)) a.flags[bh] = 1;
}

// ---- dQ, dK, dbeta and the decays' gradient ------------------------------------------------------

// A C x 64 tile whose rows are only ever read as operands lies in their order, 1,024 bytes for 16 rows and 32 columns of a plane: one
// 16-byte read per lane without bank conflicts. Element (row, x), x a multiple of 4, of the first of P planes, 512 elements apart:
template <int P>
__device__ __forceinline__ int operand_at(int row, int x) {
    return ((row >> 4) * 2 + (x >> 5)) * P * 512 + ((x >> 2 & 3) * 16 + (row & 15)) * 8 + (x >> 4 & 1) * 4;
}
template <int P>
__device__ __forceinline__ bf16x8 operand(const u16 *img, int t, int k, int plane, int lane) {
    return *reinterpret_cast<const bf16x8 *>(img + ((t * 2 + k) * P + plane) * 512 + lane * 8);
}
// Eight (four) consecutive elements of a row in P planes, each the nearest of what is left.
template <int P, int N = 8>
__device__ __forceinline__ void put_operand(u16 *img, int row, int x, const float (&y)[8]) {
    bf16x8 p[kPlanes];
    split8(y, p);
#pragma unroll
    for (int q = 0; q < P; ++q) {
        const u32x4 v = __builtin_bit_cast(u32x4, p[q]);
        *reinterpret_cast<uint2 *>(img + q * 512 + operand_at<P>(row, x)) = make_uint2(v.x, v.y);
        if constexpr (N == 8) *reinterpret_cast<uint2 *>(img + q * 512 + operand_at<P>(row, x + 4)) = make_uint2(v.z, v.w);
    }
}

// 64 columns of a chunk's float32 rows (pitch vd) on their way into a tile's planes, 8 of a row per thread and step.
template <int C, int NT>
struct StageF32 {
    static constexpr int N = (C * 8 + NT - 1) / NT;
    float4 r[N][2];

    __device__ __forceinline__ void load(const float *src, int vd, int tid) {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int at = n * NT + tid;
            if (C * 8 % NT != 0 && at >= C * 8) break;
            const float *p = src + (at / 8) * vd + at % 8 * 8;
            r[n][0] = *reinterpret_cast<const float4 *>(p);
            r[n][1] = *reinterpret_cast<const float4 *>(p + 4);
        }
    }
    // Rows times w (NULL: 1).
    __device__ __forceinline__ void store(u16 *img, const float *w, int tid) const {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int at = n * NT + tid, row = at / 8, x = at % 8 * 8;
            if (C * 8 % NT != 0 && at >= C * 8) break;
            const float s = w ? w[row] : 1.f;
            const float4 a = r[n][0], b = r[n][1];
            const float y[8] = {a.x * s, a.y * s, a.z * s, a.w * s, b.x * s, b.y * s, b.z * s, b.w * s};
            put_operand<kPlanes>(img, row, x, y);
        }
    }
};
// The same of a tensor's own rows (64 of their columns).
template <typename T, int C, int NT, bool VEC>
__device__ __forceinline__ void store_operand(const Stage<T, C, 64, NT, VEC> &s, u16 *img, int tid) {
    typedef Stage<T, C, 64, NT, VEC> S;
#pragma unroll
    for (int n = 0; n < S::N; ++n) {
        const int row = tid / S::VR + n * S::RS, x = tid % S::VR * S::VE;
        if (!S::kEven && row >= C) break;
        const uint32_t w[4] = {s.r[n].x, s.r[n].y, s.r[n].z, s.r[n].w};
        if constexpr (std::is_same_v<T, bf16_t>) {
            *reinterpret_cast<uint2 *>(img + operand_at<1>(row, x)) = make_uint2(w[0], w[1]);
            *reinterpret_cast<uint2 *>(img + operand_at<1>(row, x + 4)) = make_uint2(w[2], w[3]);
        } else {
            float y[8] = {};
#pragma unroll
            for (int e = 0; e < S::VE; ++e) y[e] = elem_f32<T>(sizeof(T) == 4 ? w[e] : (w[e / 2] >> (16 * (e % 2))) & 0xffffu);
            put_operand<Cfg<T>::in, S::VE>(img, row, x, y);
        }
    }
}

// O[t] += A(t, k) f for one 32-wide step k of rows in PA planes.
template <int C, int PA>
__device__ __forceinline__ void row_products(f32x4 (&O)[C / 16][1], const u16 *A, int k, const bf16x8 (&f)[kPlanes], int lane) {
    bf16x8 a[C / 16][PA];
#pragma unroll
    for (int t = 0; t < C / 16; ++t)
#pragma unroll
        for (int p = 0; p < PA; ++p) a[t][p] = operand<PA>(A, t, k, p, lane);
#pragma unroll
    for (int p = 0; p < PA; ++p)
#pragma unroll
        for (int q = 0; q < kPlanes; ++q)
            if (p + q < kPlanes)
#pragma unroll
                for (int t = 0; t < C / 16; ++t) O[t][0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[t][p], f[q], O[t][0], 0, 0, 0);
}
// tile_products of two such tiles.
template <int PX, int PY, typename L>
__device__ __forceinline__ void operand_products(f32x4 *s, const u16 *X, const u16 *Y, int lane) {
    constexpr int B = PX > 1 ? 3 : 4;   // tiles whose operands are held at once
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int j0 = 0; j0 < L::N; j0 += B) {
            bf16x8 a[B][PY], b[B][PX];
#pragma unroll
            for (int j = 0; j < B && j0 + j < L::N; ++j) {
#pragma unroll
                for (int p = 0; p < PX; ++p) {
                    if (j > 0 && L::O(j0 + j) == L::O(j0 + j - 1)) b[j][p] = b[j - 1][p];
                    else b[j][p] = operand<PX>(X, L::O(j0 + j), k, p, lane);
                }
#pragma unroll
                for (int p = 0; p < PY; ++p) a[j][p] = operand<PY>(Y, L::n(j0 + j), k, p, lane);
            }
#pragma unroll
            for (int p = 0; p < PY; ++p)
#pragma unroll
                for (int q = 0; q < PX; ++q)
                    if (p + q < kPlanes)
#pragma unroll
                        for (int j = 0; j < B && j0 + j < L::N; ++j) s[j0 + j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[j][p], b[j][q], s[j0 + j], 0, 0, 0);
        }
}

// part[n] = sum over the wave's columns of A[n][x] Y[n][x] + B[n][x] Z[n][x] (B may be NULL).
template <typename T, int C, int NC, int LD, bool TWO>
__device__ __forceinline__ void dot_two(const f32x4 (&A)[C / 16][NC], const u16 *Y, const f32x4 (&B)[C / 16][NC], const u16 *Z, int col, float *part, int lane) {
    float s[C / 32][8] = {};
    tile_columns<T, C, NC, LD>(Y, col, lane, [&](int j, int c, const float *y) {
#pragma unroll
        for (int e = 0; e < 8; ++e) s[j][e] = __builtin_fmaf(A[2 * j + e / 4][c][e % 4], y[e], s[j][e]);
    });
    if constexpr (TWO)
        tile_columns<T, C, NC, LD>(Z, col, lane, [&](int j, int c, const float *y) {
#pragma unroll
            for (int e = 0; e < 8; ++e) s[j][e] = __builtin_fmaf(B[2 * j + e / 4][c][e % 4], y[e], s[j][e]);
        });
#pragma unroll
    for (int j = 0; j < C / 32; ++j) {
#pragma unroll
        for (int e = 0; e < 8; ++e) s[j][e] = group_sum<16>(s[j][e]);
        if ((lane & 15) == 0) {
            *reinterpret_cast<f32x4 *>(part + 32 * j + 4 * (lane >> 4)) = f32x4{s[j][0], s[j][1], s[j][2], s[j][3]};
            *reinterpret_cast<f32x4 *>(part + 32 * j + 16 + 4 * (lane >> 4)) = f32x4{s[j][4], s[j][5], s[j][6], s[j][7]};
        }
    }
}

__device__ __forceinline__ void store_gate(void *p, mm_dtype t, int64_t i, float x) {
    switch (t) {
        case MM_FLOAT32: reinterpret_cast<float *>(p)[i] = x; break;
        case MM_FLOAT16: reinterpret_cast<f16_t *>(p)[i] = from_f32<f16_t>(x); break;
        default: reinterpret_cast<bf16_t *>(p)[i] = from_f32<bf16_t>(x);
    }
}

// The waves' shares of the lower triangles of tiles of dO U^T (f's first list; PI planes by 3) and of dV U^T (its second one; 3 by 3,
// twice the products).
template <int C, int NW, typename F>
__device__ __forceinline__ void each_tile_of_two(int wave, F &&f) {
    typedef Tiles<> None;
    if constexpr (C == 64 && NW == 8) {
        switch (wave) {
            case 0: f(None{}, Tiles<3, 0, 3, 1>{}); break;
            case 1: f(None{}, Tiles<3, 2, 3, 3>{}); break;
            case 2: f(None{}, Tiles<2, 0, 2, 1>{}); break;
            case 3: f(None{}, Tiles<2, 2, 1, 0>{}); break;
            case 4: f(None{}, Tiles<1, 1, 0, 0>{}); break;
            case 5: f(Tiles<3, 0, 3, 1, 3, 2, 3, 3>{}, None{}); break;
            case 6: f(Tiles<2, 0, 2, 1, 2, 2>{}, None{}); break;
            default: f(Tiles<1, 0, 1, 1, 0, 0>{}, None{});
        }
    } else if constexpr (C == 64) {
        switch (wave) {
            case 0: f(None{}, Tiles<3, 0, 3, 1, 3, 2, 3, 3>{}); break;
            case 1: f(None{}, Tiles<2, 0, 2, 1, 2, 2, 1, 0>{}); break;
            case 2: f(Tiles<3, 0, 3, 1, 3, 2, 3, 3>{}, Tiles<1, 1, 0, 0>{}); break;
            default: f(Tiles<2, 0, 2, 1, 2, 2, 1, 0, 1, 1, 0, 0>{}, None{});
        }
    } else if constexpr (NW == 8) {
        switch (wave) {
            case 0: f(None{}, Tiles<1, 0>{}); break;
            case 1: f(None{}, Tiles<1, 1>{}); break;
            case 2: f(None{}, Tiles<0, 0>{}); break;
            case 3: f(Tiles<1, 0>{}, None{}); break;
            case 4: f(Tiles<1, 1>{}, None{}); break;
            case 5: f(Tiles<0, 0>{}, None{});
        }
    } else {
        switch (wave) {
            case 0: f(None{}, Tiles<1, 0>{}); break;
            case 1: f(None{}, Tiles<1, 1>{}); break;
            case 2: f(None{}, Tiles<0, 0>{}); break;
            default: f(Tiles<1, 0, 1, 1, 0, 0>{}, None{});
        }
    }
}

// One workgroup per chunk; its waves split the columns of dQ and dK, 16 each. dO, U and dV pass through LDS 64 columns at a time; S and
// R come from memory as B operands, each wave its own rows of them.
//
// A log decay's gradient is the sum over the pairs (i, j) that it lies between, j < t <= i, of W_ij = A_ij (q_i . k_j) + E_ij (k_i . k_j),
// of what enters the chunk (S) and of what leaves it (R). Row sums of W with the entering terms are q_i . dQ_i + k_i . dKr_i (dKr: dK's
// terms with E and S), column sums with the leaving ones, f_j, are k_j . dKc_j. So, summed from t on to the chunk's end or to the next
// forgotten state, which no pair crosses,
//     dg_t = sum of (row sum - column sum without f) + sum over j < t of f_j + e^c_end <R, S>.
// A's diagonal would be in a row sum and in a column sum alike; it is added to dQ and dK behind them.
//
// Bound by the LDS's latency at two waves per SIMD (138 KB at dk 128, one workgroup on a CU): 64 pairs of 128 x 128, L 4,096, bfloat16, heads of
// 4 sharing q and k: 420 us, matrix cores 21 % and vector units 40 % busy, a third of the LDS cycles conflicts, in the transposed
// triangles' reads; 192 pairs of 64 x 64, L 2,048: 260 us. dO, U and dV in the order of their operands took 498 to 422 and 294 to 260.
template <typename T, int KD, bool VEC, bool F32>
__global__ void __launch_bounds__(KD * 4) __attribute__((amdgpu_waves_per_eu(2, 2))) dr_grad(const Args) {
    constexpr int C = Cfg<T>::C, PI = Cfg<T>::in, CT = C / 16, NC = 1, NW = KD / 16, NT = 64 * NW, PM = kTile<C, kScoreRow>;
    typedef Stage<T, C, KD, NT, VEC> SX;
    typedef Stage<T, C, 64, NT, VEC> SV;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    u16 *K = reinterpret_cast<u16 *>(smem), *Q = K + PI * kTile<C, KD>, *D = Q + PI * kTile<C, KD>;
    u16 *U = D + PI * kTile<C, 64>, *X = U + kPlanes * kTile<C, 64>;
    u16 *MA = U, *ME = X;   // the triangles, once U and dV are read (kTile<C, 64> is kTile<C, kScoreRow>)
    Chunk<C> *ck = reinterpret_cast<Chunk<C> *>(X + kPlanes * kTile<C, 64>);
    float *row = reinterpret_cast<float *>(ck + 1), *cols = row + NW * C, *fs = cols + NW * C, *diag = fs + NW * C, *rs = diag + C;   // [wave][C]; diag [C], rs [wave]
    auto args = [] { return own_args<Args>(); };
    int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, i = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(tid / 64), col = wave * 16;
    auto fresh = [&] {
        tid = afresh_lane(tid);
        lane = tid & 63;
        g = lane >> 4;
        i = lane & 15;
    };
    const int64_t total = [&] { const Args a = args(); return a.batch * a.heads * a.chunks; }();
    struct Where {
        Spot p;
        int64_t at;
        int t0, rows;
    };
    auto where = [&](int64_t id) {
        const Args a = args();
        const int64_t bc = id / a.heads;
        const int chunk = int(bc % a.chunks);
        Where w;
        w.p = spot_of(a, unsigned(bc / a.chunks * a.heads + id % a.heads));
        w.at = afresh(w.p.bh * a.chunks + chunk);
        w.t0 = afresh(chunk * C);
        w.rows = afresh(min(C, int(a.seqlen) - w.t0));
        return w;
    };
    const int vd = afresh(64 * args().slices);
    SX sk, sq;
    SV sd;
    StageF32<C, NT> su, sx;
    float4 sr[2][2][2];   // [k][S, R][half of 8]
    uint32_t gbits = 0, bbits = 0;
    auto load = [&](const Where &w, int h0) {
        {
            const Args a = args();
            sd.load(rows_of<T>(a.dout, w.p.b, w.p.h, a.dv, h0), w.t0, w.rows, tid);
        }
        const Args a = args();
        su.load(a.z + w.at * C * vd + h0, vd, tid);
        sx.load(a.dx + w.at * C * vd + h0, vd, tid);
    };
    auto load_states = [&](const Where &w, int h0) {
        const Args a = args();
        const float *S = a.states + w.at * KD * vd + h0, *R = a.r + w.at * KD * vd + h0;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int o = (col + i) * vd + 32 * k + 4 * g;
            sr[k][0][0] = *reinterpret_cast<const float4 *>(S + o);
            sr[k][0][1] = *reinterpret_cast<const float4 *>(S + o + 16);
            sr[k][1][0] = *reinterpret_cast<const float4 *>(R + o);
            sr[k][1][1] = *reinterpret_cast<const float4 *>(R + o + 16);
        }
    };
    auto load_first = [&](const Where &w) {
        if (wave == NW - 1) {
            const Args a = args();
            gbits = load_gate<C>(gates_of(a.g, w.p), w.t0, w.t0 + w.rows, lane);
            bbits = load_gate<C>(gates_of(a.beta, w.p), w.t0, w.t0 + w.rows, lane);
        }
        {
            const Args a = args();
            sk.load(rows_of<T>(a.k, w.p.b, w.p.h, a.dk), w.t0, w.rows, tid);
        }
        {
            const Args a = args();
            sq.load(rows_of<T>(a.q, w.p.b, w.p.h, a.dk), w.t0, w.rows, tid);
        }
        load(w, 0);
        load_states(w, 0);
    };
    // At dk 128 a group takes several chunks, the next one's first loads on their way while it ends one (465 us where a group for each
    // took 508, 64 pairs, L 4,096, dv 128). At 64 two groups are on a CU, which do the same for each other and have no registers for it
    // (312 and 363 us, 192 pairs, L 2,048, dv 64).
    constexpr bool kAhead = KD == 128;
    Where next = where(blockIdx.x);
    if constexpr (kAhead) load_first(next);
    for (int64_t id = blockIdx.x; id < total; id += gridDim.x) {
        if constexpr (!kAhead) {
            if (id != blockIdx.x) next = where(id);
            load_first(next);
        }
        const Where w = next;
        const Spot p = w.p;
        const int t0 = w.t0, rows = w.rows;
        __syncthreads();
        fresh();
        if (wave == NW - 1) {
            const Args a = args();
            make_chunk<C>(*ck, gbits, a.g.type, bbits, a.beta.type, a.scale, lane);
        }
        sk.store(K, tid);
        sq.store(Q, tid);
        constexpr int kScores = C == 64 && NW == 4 ? 6 : C == 64 ? 4 : 3;
        f32x4 sc[kScores], dq[CT][NC], dr[CT][NC], dc[CT][NC];   // sc: the tiles of both lists
        float rdots = 0.f;
#pragma unroll
        for (int j = 0; j < kScores; ++j) sc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int t = 0; t < CT; ++t) dq[t][0] = dr[t][0] = dc[t][0] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
        for (int h0 = 0; h0 < vd; h0 += 64) {
            __syncthreads();
            fresh();
            store_operand<T, C, NT, VEC>(sd, D, tid);
            su.store(U, ck->beta, tid);
            sx.store(X, nullptr, tid);
            if (h0 + 64 < vd) load(w, h0 + 64);
            __syncthreads();
            fresh();
            each_tile_of_two<C, NW>(wave, [&](auto L1, auto L2) {
                if constexpr (decltype(L1)::N > 0) operand_products<PI, kPlanes, decltype(L1)>(sc, D, U, lane);
                if constexpr (decltype(L2)::N > 0) operand_products<kPlanes, kPlanes, decltype(L2)>(sc + decltype(L1)::N, X, U, lane);
            });
            fresh();
            bf16x8 f[2][2][kPlanes];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                float y[2][8];
#pragma unroll
                for (int m = 0; m < 2; ++m)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        y[m][4 * e] = sr[k][m][e].x;
                        y[m][4 * e + 1] = sr[k][m][e].y;
                        y[m][4 * e + 2] = sr[k][m][e].z;
                        y[m][4 * e + 3] = sr[k][m][e].w;
                    }
#pragma unroll
                for (int e = 0; e < 8; ++e) rdots = __builtin_fmaf(y[0][e], y[1][e], rdots);
                split8(y[0], f[k][0]);
                split8(y[1], f[k][1]);
            }
            if (h0 + 64 < vd) load_states(w, h0 + 64);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                row_products<C, PI>(dq, D, k, f[k][0], lane);
                row_products<C, kPlanes>(dr, X, k, f[k][0], lane);
                row_products<C, kPlanes>(dc, U, k, f[k][1], lane);
            }
        }
        if constexpr (kAhead) {
            if (id + gridDim.x < total) {
                next = where(id + gridDim.x);
                load_first(next);
            }
        }
        // The state terms' row factors.
#pragma unroll
        for (int t = 0; t < CT; ++t) {
            const f32x4 fq = *reinterpret_cast<const f32x4 *>(ck->inq + 16 * t + 4 * g), fi = *reinterpret_cast<const f32x4 *>(ck->d.in + 16 * t + 4 * g),
                        fo = *reinterpret_cast<const f32x4 *>(ck->d.out + 16 * t + 4 * g);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                dq[t][0][r] *= fq[r];
                dr[t][0][r] *= -fi[r];
                dc[t][0][r] *= fo[r];
            }
        }
        const bool want_g = args().dg || args().dg_sum;
        if (want_g) {
            dot_two<T, C, NC, KD, false>(dc, K, dc, K, col, fs + wave * C, lane);
            rdots = wave_sum(rdots);
            if (lane == 0) rs[wave] = rdots;
        }
        __syncthreads();
        fresh();
        // The triangles.
        const float scale = args().scale;
        each_tile_of_two<C, NW>(wave, [&](auto L1, auto L2) {
            typedef decltype(L1) A;
            typedef decltype(L2) E;
            static_for<0, A::N>([&](auto Jc) {
                constexpr int j = decltype(Jc)::value, O = A::O(j), o = A::n(j);
                const f32x4 w = tile_decay<C, false, O, o>(ck->d, 1.f, lane);
                float x[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    x[r] = sc[j][r] * (w[r] * scale);
                    if constexpr (O == o) {
                        if (4 * g + r == i) diag[16 * O + i] = x[r];
                        x[r] = 4 * g + r < i ? x[r] : 0.f;
                    }
                }
                store_scores<C>(MA, x, O, o, lane);
            });
            static_for<0, E::N>([&](auto Jc) {
                constexpr int j = decltype(Jc)::value, O = E::O(j), o = E::n(j);
                const f32x4 w = tile_decay<C, false, O, o>(ck->d, 1.f, lane);
                float x[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) x[r] = O != o || 4 * g + r < i ? -(sc[A::N + j][r] * w[r]) : 0.f;
                store_scores<C>(ME, x, O, o, lane);
            });
        });
        zero_masked_scores<C>(MA, false, tid, NT);
        zero_masked_scores<C>(ME, false, tid, NT);
        __syncthreads();
        fresh();
#pragma unroll
        for (int j = 0; j < C / 32; ++j) {
            bf16x8 k[PI], q[PI];
#pragma unroll
            for (int x = 0; x < PI; ++x) {
                k[x] = frag_tr<KD>(K + x * kTile<C, KD>, 32 * j, col, g, i);
                q[x] = frag_tr<KD>(Q + x * kTile<C, KD>, 32 * j, col, g, i);
            }
            // dQ += A K, dKr += E K, dKc += A^T Q + E^T K: a plane's products of all row tiles, then the next plane's.
#pragma unroll
            for (int x = 0; x < kPlanes; ++x) {
                bf16x8 ma[CT], me[CT], ta[CT], te[CT];
#pragma unroll
                for (int t = 0; t < CT; ++t) {
                    if (has_frag<C, true>(t, j)) {
                        ma[t] = frag_row<kScoreRow>(MA + x * PM, 16 * t, j, g, i);
                        me[t] = frag_row<kScoreRow>(ME + x * PM, 16 * t, j, g, i);
                    }
                    if (has_frag<C, false>(t, j)) {
                        ta[t] = frag_tr<kScoreRow>(MA + x * PM, 32 * j, 16 * t, g, i);
                        te[t] = frag_tr<kScoreRow>(ME + x * PM, 32 * j, 16 * t, g, i);
                    }
                }
#pragma unroll
                for (int y = 0; y < PI; ++y)
                    if (x + y < kPlanes) {
#pragma unroll
                        for (int t = 0; t < CT; ++t) {
                            if (has_frag<C, true>(t, j)) {
                                dq[t][0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ma[t], k[y], dq[t][0], 0, 0, 0);
                                dr[t][0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(me[t], k[y], dr[t][0], 0, 0, 0);
                            }
                            if (has_frag<C, false>(t, j)) dc[t][0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ta[t], q[y], dc[t][0], 0, 0, 0);
                        }
#pragma unroll
                        for (int t = 0; t < CT; ++t)
                            if (has_frag<C, false>(t, j)) dc[t][0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(te[t], k[y], dc[t][0], 0, 0, 0);
                    }
            }
        }
        fresh();
        if (want_g) {
            dot_two<T, C, NC, KD, true>(dq, Q, dr, K, col, row + wave * C, lane);
            dot_two<T, C, NC, KD, false>(dc, K, dc, K, col, cols + wave * C, lane);
        }
        // A's diagonal, which is in no decay's sum: dQ_i += A_ii k_i, dK_i += A_ii q_i.
        auto add_diagonal = [&](f32x4 (&x)[CT][NC], const u16 *rows_) {
            tile_columns<T, C, NC, KD>(rows_, col, lane, [&](int j, int, const float *y) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const f32x4 d = *reinterpret_cast<const f32x4 *>(diag + 32 * j + 16 * h + 4 * g);
#pragma unroll
                    for (int r = 0; r < 4; ++r) x[2 * j + h][0][r] = __builtin_fmaf(d[r], y[4 * h + r], x[2 * j + h][0][r]);
                }
            });
        };
#pragma unroll
        for (int t = 0; t < CT; ++t) dr[t][0] += dc[t][0];
        add_diagonal(dq, K);
        add_diagonal(dr, Q);
        {
            const Args a = args();
            const int64_t ob = (p.b * a.seqlen * a.heads + p.h) * a.dk * int64_t(F32 ? 4 : sizeof(T));
            const uint32_t stride = uint32_t(a.heads * a.dk);
            store_out<T, C, NC, KD, VEC, F32>(dq, static_cast<char *>(a.dq) + ob, stride, t0, rows, a.dk, Q, col, lane);
            store_out<T, C, NC, KD, VEC, F32>(dr, static_cast<char *>(a.dk_out) + ob, stride, t0, rows, a.dk, K, col, lane);
        }
        __syncthreads();
        if (wave == 0 && lane < rows) {
            const Args a = args();
            float s = 0.f;
            for (int x = 0; x < a.slices; ++x) s += a.pbeta[(int64_t(x) * a.batch * a.heads + p.bh) * a.chunks * C + t0 + lane];
            store_gate(a.dbeta, a.beta.type, (p.b * a.seqlen + t0 + lane) * a.heads + p.h, s);
        }
        if (want_g && wave == 1) {
            const Args a = args();
            const bool forgets = lane < rows && decode_g(load_gate<C>(gates_of(a.g, p), t0, t0 + rows, lane), a.g.type) == -128.f;
            const uint64_t all = __ballot(forgets);
            float e = 0.f, f = 0.f;
            if (lane < C) {
#pragma unroll
                for (int w = 0; w < NW; ++w) {
                    const float left = fs[w * C + lane];
                    e += row[w * C + lane] - (cols[w * C + lane] - left);
                    f += left;
                }
            }
            // e from here to the chunk's end or the next forgotten state, f of the tokens before.
            const uint64_t behind = all >> lane >> 1;
            const int last = min(rows, lane + 1 + (behind ? __builtin_ctzll(behind) : 64));
            float before = f;
#pragma unroll
            for (int d = 1; d < C; d *= 2) {
                const float x = __shfl_down(e, d), y = __shfl_up(before, d);
                if (lane + d < last) e += x;
                if (lane >= d) before += y;
            }
            before = __shfl_up(before, 1);
            if (lane < rows) {
                float s = 0.f;
#pragma unroll
                for (int w = 0; w < NW; ++w) s += rs[w];
                s = forgets ? 0.f : ck->d.all * s + (lane ? before : 0.f) + e;
                if (a.dg_sum) a.dg_sum[p.bh * a.seqlen + t0 + lane] = s;
                else store_gate(a.dg, a.g.type, (p.b * a.seqlen + t0 + lane) * a.heads + p.h, s);
            }
        }
    }
}

// ---- launches ------------------------------------------------------------------------------------

constexpr int64_t kMostGroups = int64_t(1) << 17;   // of a launch that loops over chunks

template <typename T, int KD, bool REV, bool VEC>
static int prep_t(const Args &a, hipStream_t s) {
    constexpr int C = Cfg<T>::C, PI = Cfg<T>::in;
    constexpr int tiles = 2 * 2 * PI * kTile<C, KD>, tri = 2 * C * kPitch<C> * 4, bytes = (tiles > tri ? tiles : tri) + int(sizeof(Chunk<C>));
    static std::atomic<uint64_t> done{0};
    return launch_kernel(dr_prep<T, KD, REV, VEC>, bytes, done, std::min<int64_t>(a.batch * a.heads * a.chunks, kMostGroups), kThreads, a, s, "dr_prep");
}
template <typename T, int KD, Leaves L, bool VEC>
static int walk_t(const Args &a, hipStream_t s) {
    constexpr int C = Cfg<T>::C, PI = Cfg<T>::in;
    constexpr int bytes = 2 * ((L == kOutputs ? 2 : 1) * PI * kTile<C, KD> + PI * kTile<C, 64>) + kRecord<C, L == kOutputs ? 2 : 1>;
    static_assert(bytes <= 80 * 1024, "two workgroups on a CU");
    static std::atomic<uint64_t> done{0};
    return launch_kernel(dr_walk<T, KD, L, VEC>, bytes, done, unit_grid(a, L == kMaps ? a.slices + KD / 64 : a.slices), kThreads, a, s, "dr_walk");
}
template <typename T, int KD, bool MAPS, bool VEC>
static int back_t(const Args &a, hipStream_t s) {
    constexpr int C = Cfg<T>::C, PI = Cfg<T>::in;
    constexpr int bytes = 2 * (2 * PI * kTile<C, KD> + PI * kTile<C, 64>) + kRecord<C, 2> + 4 * kWaves * C;
    static_assert(bytes <= 160 * 1024, "LDS");
    static std::atomic<uint64_t> done{0};
    return launch_kernel(dr_back<T, KD, MAPS, VEC>, bytes, done, unit_grid(a, a.slices), kThreads, a, s, "dr_back");
}
template <int KD, bool BACK>
static int join_t(const Args &a, hipStream_t s) {
    hipLaunchKernelGGL((dr_join<KD, BACK>), dim3(unsigned(a.batch * a.heads * a.slices * 2)), dim3(kThreads), 0, s, a);
    return launch_status("dr_join");
}
template <typename T, int KD, bool VEC, bool F32>
static int grad_t(const Args &a, hipStream_t s) {
    constexpr int C = Cfg<T>::C, PI = Cfg<T>::in;
    constexpr int NW = KD / 16;
    constexpr int bytes = 2 * (2 * PI * kTile<C, KD> + PI * kTile<C, 64> + 2 * kPlanes * kTile<C, 64>) + int(sizeof(Chunk<C>)) + 4 * ((3 * NW + 1) * C + NW);
    static_assert(bytes <= (KD == 64 ? 80 : 160) * 1024, "two workgroups on a CU at KD 64, one at 128");
    static std::atomic<uint64_t> done{0};
    return launch_kernel(dr_grad<T, KD, VEC, F32>, bytes, done, std::min<int64_t>(a.batch * a.heads * a.chunks, KD == 64 ? kMostGroups : device_simds() / 4), 64 * NW, a, s, "dr_grad");
}

template <typename T>
int launch_prep(const Args &a, bool rev, hipStream_t s) {
    const bool vec = a.q.vec && a.k.vec;
    auto go = [&](auto kd, auto r) {
        constexpr int KD = decltype(kd)::value;
        constexpr bool REV = decltype(r)::value;
        return vec ? prep_t<T, KD, REV, true>(a, s) : prep_t<T, KD, REV, false>(a, s);
    };
    typedef std::integral_constant<int, 64> K64;
    typedef std::integral_constant<int, 128> K128;
    if (rev) return a.dk <= 64 ? go(K64{}, std::true_type{}) : go(K128{}, std::true_type{});
    return a.dk <= 64 ? go(K64{}, std::false_type{}) : go(K128{}, std::false_type{});
}
template <typename T>
int launch_walk(const Args &a, bool states, hipStream_t s) {
    const bool maps = a.k.vec && a.v.vec, vec = maps && (states || (a.q.vec && a.out_vec));
    auto go = [&](auto kd) {
        constexpr int KD = decltype(kd)::value;
        if (a.segs > 1 && !a.kept_starts) {
            if (const int rc = maps ? walk_t<T, KD, kMaps, true>(a, s) : walk_t<T, KD, kMaps, false>(a, s)) return rc;
            if (const int rc = join_t<KD, false>(a, s)) return rc;
        }
        if (states) return vec ? walk_t<T, KD, kStates, true>(a, s) : walk_t<T, KD, kStates, false>(a, s);
        return vec ? walk_t<T, KD, kOutputs, true>(a, s) : walk_t<T, KD, kOutputs, false>(a, s);
    };
    return a.dk <= 64 ? go(std::integral_constant<int, 64>{}) : go(std::integral_constant<int, 128>{});
}
template <typename T>
int launch_back(const Args &a, hipStream_t s) {
    const bool maps = a.q.vec && a.k.vec && a.dout.vec, vec = maps && a.out_vec;
    auto go = [&](auto kd) {
        constexpr int KD = decltype(kd)::value;
        if (a.segs > 1) {
            if (const int rc = maps ? back_t<T, KD, true, true>(a, s) : back_t<T, KD, true, false>(a, s)) return rc;
            if (const int rc = join_t<KD, true>(a, s)) return rc;
        }
        return vec ? back_t<T, KD, false, true>(a, s) : back_t<T, KD, false, false>(a, s);
    };
    return a.dk <= 64 ? go(std::integral_constant<int, 64>{}) : go(std::integral_constant<int, 128>{});
}
template <typename T>
int launch_grad(const Args &a, hipStream_t s) {
    const bool vec = a.q.vec && a.k.vec && a.dout.vec && a.dqk_vec;
    auto go = [&](auto kd) {
        constexpr int KD = decltype(kd)::value;
        if constexpr (sizeof(T) == 2)
            if (!a.dqk_f32) return vec ? grad_t<T, KD, true, false>(a, s) : grad_t<T, KD, false, false>(a, s);
        return vec ? grad_t<T, KD, true, true>(a, s) : grad_t<T, KD, false, true>(a, s);
    };
    return a.dk <= 64 ? go(std::integral_constant<int, 64>{}) : go(std::integral_constant<int, 128>{});
}

template int launch_prep<MM_DELTA_TYPE>(const Args &, bool, hipStream_t);
template int launch_walk<MM_DELTA_TYPE>(const Args &, bool, hipStream_t);
template int launch_back<MM_DELTA_TYPE>(const Args &, hipStream_t);
template int launch_grad<MM_DELTA_TYPE>(const Args &, hipStream_t);

}  // namespace dr
}  // namespace mm
