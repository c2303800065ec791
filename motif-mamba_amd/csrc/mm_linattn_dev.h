// mm_linattn_dev.h -- device pieces of the chunked linear attention with one decay for each head
// (mm_linattn.hip): the operand planes, the tiles' staging, and a chunk's steps.
//
// The mathematics. With c_i the sum of log_decay over a chunk's tokens up to i (c_end its total), a chunk
// of C tokens that starts from the state S (dk x dv) gives
//     o_i  = exp(c_i) q_i S + sum_{j <= i} exp(c_i - c_j) (q_i . k_j) v_j
//     S'   = exp(c_end) S + sum_j k_j (exp(c_end - c_j) v_j)^T
// and each of the three gradients of q, k and v is a walk of the same form: dq_i the forward one with
// (do, v, k) in the place of (q, k, v), dv_j and dk_j the one from the end with (k, q, do) and (v, do, q),
// whose row factor is exp(c_end - c_j) and whose update factor exp(c_i). A walk is named here by its
// tiles: X (C x KD, the rows' factor), Y (C x KD, what the state is built from), V (C x columns).
//
// Exactness. Products run on v_mfma_f32_16x16x32_bf16, which multiplies bfloat16 exactly and adds in
// float32. Every other number is carried as a sum of bfloat16 planes: float16 inputs as two and float32
// inputs as three (both exact), and every float32 factor, the state, the decayed scores and the decayed rows
// that the state is built from, as three (relative error 2^-25, for every input type). So all of them are
// float32 from end to end and 16-bit outputs are rounded once. (Two planes, 2^-17, for the state and the scores of 16-bit
// inputs took 316 us where three take 361, 4 x 4,096 tokens of 80 heads at 128 x 64 in bfloat16, and moved outputs near the
// middle of two 16-bit numbers to the wrong one.)
//
// Lane layouts (l the lane, g = l / 16, i = l % 16; checked on the card): an accumulator tile holds column
// i, rows 4g .. 4g + 3. An operand holds row (A) or column (B) i and eight of 32 contraction indices; the
// order of those is free as long as A and B agree, and here it is {4g .. 4g + 3, 16 + 4g .. 16 + 4g + 3}:
// two accumulator tiles, one below the other, ARE a B operand, so the state goes from the accumulators of
// its update into the product with X without leaving the registers.
#pragma once

#include <hip/hip_runtime.h>

#include "mm_common.h"
#include "mm_internal.h"
#include "mm_linattn.h"

namespace mm {
namespace la {

typedef uint16_t u16;
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// Planes of an input; tokens of a chunk.
template <typename T> struct Cfg;
template <> struct Cfg<bf16_t> { static constexpr int in = 1, C = 64; };
template <> struct Cfg<f16_t> { static constexpr int in = 2, C = 32; };
template <> struct Cfg<float> { static constexpr int in = 3, C = 32; };
constexpr int kPlanes = 3;       // of a float32 factor

constexpr int kBlock = 256;      // tokens between two kept states (see the decays' gradient)

// Tiles in LDS are rows of D elements (64 or 128; 64 scores), cut into units of 4 (8 bytes). Both ways that operands
// are read, 16 rows of one unit (frag_row) and 4 rows of 4 units (frag_tr), should touch the 16 units of a 128-byte
// line each once, so unit u of row r lies at u ^ swizzle(r): r's low two bits move a unit between the line's quarters,
// its next two within one. Bank conflicts are still 31 % of the walks' LDS cycles (rows padded by 16 bytes instead: 42 %); which
// access makes them has not been told apart.
__device__ __forceinline__ constexpr int swizzle(int row) { return (row & 3) << 2 | (row >> 2 & 3); }
// 16 bytes stand between blocks of 16 rows: two blocks' reads at one lane's address are then no constant distance apart that one
// instruction could span. (The compiler would join them, and move every half into its operand afterwards.)
template <int D>
__device__ __forceinline__ constexpr int block(int row) { return row * D + row / 16 * 8; }   // row: a multiple of 16
template <int D>
__device__ __forceinline__ constexpr int at(int row, int col) {
    return row * D + (row >> 4) * 8 + (((col >> 2) ^ swizzle(row)) << 2) + (col & 3);
}
template <int C, int D>
constexpr int kTile = C * D + C / 16 * 8;   // elements of a tile's plane
constexpr int kScoreRow = 64;

// A log decay's bits (converted when used, so that the load is waited for there).
__device__ __forceinline__ uint32_t load_g_raw(const void *p, mm_dtype t, int64_t i) {
    if (t == MM_FLOAT32) return reinterpret_cast<const uint32_t *>(p)[i];
    return reinterpret_cast<const u16 *>(p)[i];
}
__device__ __forceinline__ float decode_g(uint32_t w, mm_dtype t) {
    const float x = t == MM_FLOAT32 ? __uint_as_float(w) : t == MM_BFLOAT16 ? __uint_as_float(w << 16) : elem_f32<f16_t>(w);
    // exp(-128) is 0 in float32 as every smaller decay is, and exp(128) infinite; a finite sum keeps the
    // differences of two sums defined. The comparisons are false for NaN, which stays.
    return x < -128.f ? -128.f : x > 128.f ? 128.f : x;
}

__device__ __forceinline__ bool finite(float x) { return __builtin_fabsf(x) <= 3.402823466e38f; }

// exp(x): 2^(x log2 e) with the product's rounding error and log2 e's own taken back in (v_exp_f32 is within 1 ulp). An infinite
// result has no correction: infinity less a part of itself is NaN.
__device__ __forceinline__ float exp_f32(float x) {
    const float p = x * kLog2e;
    const float e = __builtin_fmaf(x, 1.925963033e-8f, __builtin_fmaf(x, kLog2e, -p));
    const float r = __builtin_amdgcn_exp2f(p);
    return p < 128.f ? __builtin_fmaf(r, e * kLn2, r) : r;
}

// A number that the compiler does not know to be the one it was: what is computed from it is computed where it is used,
// not once and held in registers through the walk (the walks would not fit their registers otherwise).
__device__ __forceinline__ int afresh(int x) {
    asm volatile("" : "+s"(x));
    return x;
}
__device__ __forceinline__ int64_t afresh(int64_t x) {
    asm volatile("" : "+s"(x));
    return x;
}
__device__ __forceinline__ float afresh(float x) {
    asm volatile("" : "+s"(x));
    return x;
}
template <typename T>
__device__ __forceinline__ T *afresh(T *p) {
    typedef __attribute__((address_space(1))) T *Global;
    Global x = (Global)p;
    asm volatile("" : "+s"(x));
    return (T *)x;
}
__device__ __forceinline__ int afresh_lane(int x) {
    asm volatile("" : "+v"(x));
    return x;
}

// ---- planes --------------------------------------------------------------------------------------

// x as a sum of bfloat16 planes, each the nearest of what is left.
__device__ __forceinline__ void split8(const float *x, bf16x8 *out) {
    float r[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = x[i];
#pragma unroll
    for (int p = 0; p < kPlanes; ++p) {
        u32x4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = pack_bf16x2(r[2 * i], r[2 * i + 1]);
        out[p] = __builtin_bit_cast(bf16x8, w);
        if (p + 1 < kPlanes) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                r[2 * i] -= __uint_as_float(w[i] << 16);
                r[2 * i + 1] -= __uint_as_float(w[i] & 0xffff0000u);
            }
        }
    }
}

__device__ __forceinline__ bf16x8 join(uint2 a, uint2 b) {
    return __builtin_bit_cast(bf16x8, u32x4{a.x, a.y, b.x, b.y});
}
// Operand whose row or column is tile row r0 + i (r0 a multiple of 16) and whose contraction runs over tile columns 32 k .. 32 k + 31.
template <int D>
__device__ __forceinline__ bf16x8 frag_row(const u16 *tile, int r0, int k, int g, int i) {
    const u16 *row = tile + block<D>(r0) + i * D + (k / 2) * 64;
    const int u = (8 * (k % 2) + g) ^ swizzle(i);
    return join(*reinterpret_cast<const uint2 *>(row + 4 * u), *reinterpret_cast<const uint2 *>(row + 4 * (u ^ 4)));
}
// Operand whose row or column is tile column col + i and whose contraction runs over tile rows r0 .. r0 + 31
// (r0 and col multiples of 16).
template <int D>
__device__ __forceinline__ bf16x8 frag_tr(const u16 *tile, int r0, int col, int g, int i) {
    const int u = ((col / 16 % 4) ^ (i >> 2)) << 2 | ((i & 3) ^ g);
    const u16 *a = tile + block<D>(r0) + (4 * g + (i >> 2)) * D + col / 64 * 64 + 4 * u;
    typedef __attribute__((address_space(3))) s16x4 *lds_ptr;
    const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)a);
    const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(a + block<D>(16)));
    return join(__builtin_bit_cast(uint2, x), __builtin_bit_cast(uint2, y));
}

__device__ __forceinline__ void unpack_frag(const bf16x8 &f, float *x) {
    const u32x4 w = __builtin_bit_cast(u32x4, f);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        x[2 * k] = __uint_as_float(w[k] << 16);
        x[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
    }
}

// ---- staging -------------------------------------------------------------------------------------

// Buffer accesses: offsets below 2^31 from a uniform base; kNone reads 0 and drops a store.
constexpr uint32_t kNone = 0x80000000u;
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer(const void *base) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(base), (short)0, int(kNone), 0x00020000);
}

// A tensor's rows of one (batch row, head): token t at p + t * stride. The host takes care that 64 rows span less
// than 2^31 bytes.
template <typename T> struct Rows {
    const T *p;
    uint32_t stride; // bytes
    int d;           // elements of a row that exist
};

// A C x D tile on its way from memory to LDS, 16 bytes per thread and step, in registers. VEC: rows and d are
// multiples of 16 bytes; else element by element. Rows and columns that do not exist are 0.
template <typename T, int C, int D, int NT, bool VEC>
struct Stage {
    static constexpr int VE = 16 / sizeof(T), VR = D / VE, RS = NT / VR, N = (C + RS - 1) / RS;
    static constexpr int PLANE = kTile<C, D>;
    static_assert(NT % VR == 0, "a row's threads");
    static constexpr bool kEven = C % RS == 0;
    uint4 r[N];

    __device__ __forceinline__ void load(const Rows<T> &s, int t0, int rows, int tid) {
        const __amdgpu_buffer_rsrc_t buf = buffer(reinterpret_cast<const char *>(s.p) + uint64_t(unsigned(t0)) * s.stride);
        const int row = unsigned(tid) / VR, col = unsigned(tid) % VR * VE;
        const uint32_t stride = s.stride, off = uint32_t(row) * stride + uint32_t(col) * uint32_t(sizeof(T));
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const bool live = row + n * RS < (kEven ? rows : min(rows, C));
            const uint32_t at = off + uint32_t(n * RS) * stride;
            if constexpr (VEC) {
                uint32_t a = live && col < s.d ? at : kNone;
                asm("" : "+v"(a));   // the offset is selected, the load not branched over
                r[n] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(buf, a, 0, 0));
            } else {
                uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
                for (int e = 0; e < VE; ++e) {
                    const uint32_t a = live && col + e < s.d ? at + e * uint32_t(sizeof(T)) : kNone;
                    if constexpr (sizeof(T) == 4) w[e] = __builtin_amdgcn_raw_buffer_load_b32(buf, a, 0, 0);
                    else w[e / 2] |= uint32_t(u16(__builtin_amdgcn_raw_buffer_load_b16(buf, a, 0, 0))) << (16 * (e % 2));
                }
                r[n] = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
    }

    // Into the tile's planes. float16 and float32 are cut after 8 significant bits per plane, which is exact;
    // an infinity or NaN stands in the first plane alone.
    __device__ __forceinline__ void store(u16 *tile, int tid) const {
        const int row0 = unsigned(tid) / VR, col = unsigned(tid) % VR * VE;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int row = row0 + n * RS;
            if (!kEven && row >= C) break;
            // Two units of 4 elements (one of float32), next to each other but in the order of the row's swizzle.
            const int sw = swizzle(row);
            const bool flip = VE == 8 && (sw & 1);
            u16 *dst = tile + row * D + (row >> 4) * 8 + ((((col >> 2) ^ sw) & (VE == 8 ? ~1 : ~0)) << 2);
            const uint32_t w[4] = {r[n].x, r[n].y, r[n].z, r[n].w};
            if constexpr (std::is_same_v<T, bf16_t>) {
                *reinterpret_cast<uint4 *>(dst) = flip ? make_uint4(w[2], w[3], w[0], w[1]) : r[n];
            } else {
                constexpr int P = Cfg<T>::in;
                uint32_t o[P][VE / 2];
                float x[VE];
#pragma unroll
                for (int e = 0; e < VE; ++e) x[e] = elem_f32<T>(sizeof(T) == 4 ? w[e] : (w[e / 2] >> (16 * (e % 2))) & 0xffffu);
#pragma unroll
                for (int e = 0; e < VE; ++e) {
                    const uint32_t b = __float_as_uint(x[e]);
                    const bool fin = (b & 0x7f800000u) != 0x7f800000u;
                    uint32_t h = b & 0xffff0000u;
                    if (!fin && (b & 0x007fffffu)) h |= 0x00400000u;   // NaN whatever its payload
                    float rest = fin ? x[e] - __uint_as_float(h) : 0.f;
#pragma unroll
                    for (int p = 0; p < P; ++p) {
                        if (e % 2 == 0) o[p][e / 2] = h >> 16;
                        else o[p][e / 2] |= h;
                        h = __float_as_uint(rest) & 0xffff0000u;
                        rest -= __uint_as_float(h);
                    }
                }
#pragma unroll
                for (int p = 0; p < P; ++p) {
                    if constexpr (VE == 8) *reinterpret_cast<uint4 *>(dst + p * PLANE) = flip ? make_uint4(o[p][2], o[p][3], o[p][0], o[p][1]) : make_uint4(o[p][0], o[p][1], o[p][2], o[p][3]);
                    else *reinterpret_cast<uint2 *>(dst + p * PLANE) = make_uint2(o[p][0], o[p][1]);
                }
            }
        }
    }
};

// ---- decays of a chunk ---------------------------------------------------------------------------

// All from sums taken in float64 over the chunk's tokens, so that a difference of two sums is as good as
// its own sum: scores of 16-token tiles off the diagonal take the product of three factors, each the
// exponential of a sum of log decays (at most 1 where those are at most 0: nothing overflows, and a
// forgotten state gives 0, never 0 times infinity), tiles on the diagonal exp(c_i - c_j) itself.
template <int C>
struct __attribute__((aligned(16))) Decays {
    float in[C];           // scale exp(c_t): from the chunk's start, t's own decay included
    float out[C];          // exp(c_end - c_t)
    float from[C];         // scale exp(c_t - the sum before t's tile)
    float to[C];           // exp(the sum up to the end of t's tile - c_t)
    float hi[C], lo[C];    // c_t
    float mid[C / 16][C / 16];   // [I][J], J < I: from the end of tile J to the start of tile I
    float all;             // exp(c_end)
};

template <int CTRL>
__device__ __forceinline__ double dpp_add_f64(double x, int row_mask) {
    const uint64_t b = __builtin_bit_cast(uint64_t, x);
    uint32_t lo, hi;
    if (row_mask == 0xf) {
        lo = __builtin_amdgcn_update_dpp(0, int(uint32_t(b)), CTRL, 0xf, 0xf, false);
        hi = __builtin_amdgcn_update_dpp(0, int(uint32_t(b >> 32)), CTRL, 0xf, 0xf, false);
    } else if (row_mask == 0xa) {
        lo = __builtin_amdgcn_update_dpp(0, int(uint32_t(b)), CTRL, 0xa, 0xf, false);
        hi = __builtin_amdgcn_update_dpp(0, int(uint32_t(b >> 32)), CTRL, 0xa, 0xf, false);
    } else {
        lo = __builtin_amdgcn_update_dpp(0, int(uint32_t(b)), CTRL, 0xc, 0xf, false);
        hi = __builtin_amdgcn_update_dpp(0, int(uint32_t(b >> 32)), CTRL, 0xc, 0xf, false);
    }
    return x + __builtin_bit_cast(double, uint64_t(lo) | uint64_t(hi) << 32);
}
__device__ __forceinline__ double readlane_f64(double x, int lane) {
    const uint64_t b = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = __builtin_amdgcn_readlane(int(uint32_t(b)), lane);
    const uint32_t hi = __builtin_amdgcn_readlane(int(uint32_t(b >> 32)), lane);
    return __builtin_bit_cast(double, uint64_t(lo) | uint64_t(hi) << 32);
}
// Sum over the lanes up to and including this one.
__device__ __forceinline__ double prefix_f64(double x) {
    x = dpp_add_f64<0x111>(x, 0xf);   // row_shr 1, 2, 4, 8: within 16 lanes
    x = dpp_add_f64<0x112>(x, 0xf);
    x = dpp_add_f64<0x114>(x, 0xf);
    x = dpp_add_f64<0x118>(x, 0xf);
    x = dpp_add_f64<0x142>(x, 0xa);   // row_bcast 15 into rows 1 and 3
    x = dpp_add_f64<0x143>(x, 0xc);   // row_bcast 31 into rows 2 and 3
    return x;
}

__device__ __forceinline__ double shfl_f64(double x, int lane) {
    const uint64_t b = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = __builtin_amdgcn_ds_bpermute(lane * 4, int(uint32_t(b))), hi = __builtin_amdgcn_ds_bpermute(lane * 4, int(uint32_t(b >> 32)));
    return __builtin_bit_cast(double, uint64_t(lo) | uint64_t(hi) << 32);
}

// One wave; g: the lane's token's log decay, 0 behind the last token and in lanes past C. Returns the chunk's total.
template <int C>
__device__ __forceinline__ double make_decays(Decays<C> &d, float g, float scale, int lane) {
    const double c = prefix_f64(double(g));
    const double all = readlane_f64(c, C - 1);
    const int tile = (lane >> 4);
    const double end = shfl_f64(c, 16 * tile + 15), before = shfl_f64(c, 16 * tile - 1 & 63);
    // lane 4 I + J of the first 16: from the end of tile J to the start of tile I (J < I)
    const int I = lane >> 2 & 3, J = lane & 3;
    const double mid = shfl_f64(c, 16 * I - 1 & 63) - shfl_f64(c, 16 * J + 15);
    const float hi = float(c);
    const float in = exp_f32(hi), out = exp_f32(float(all - c)), from = exp_f32(float(c - (tile ? before : 0.0))),
                to = exp_f32(float(end - c)), m = exp_f32(float(mid));
    if (C == 64 || lane < C) {
        d.in[lane] = in * scale;
        d.out[lane] = out;
        d.from[lane] = from * scale;
        d.to[lane] = to;
        d.hi[lane] = hi;
        d.lo[lane] = float(c - double(hi));
        if (lane == C - 1) d.all = in;
    }
    if (lane < 16 && I < C / 16 && J < I) d.mid[I][J] = m;
    return all;
}

// ---- a chunk's steps -----------------------------------------------------------------------------

// A list of 16 x 16 score tiles: row token tiles O and tiles n of the tokens they see.
template <int... ON>
struct Tiles {
    static constexpr int N = sizeof...(ON) / 2;
    static constexpr int on[2 * N] = {ON...};
    static constexpr int O(int j) { return on[2 * j]; }
    static constexpr int n(int j) { return on[2 * j + 1]; }
};

// Their scores, side by side: column i the row token 16 O + i of X, rows 4g + r the tokens 16 n + 4g + r of Y.
template <typename T, int C, int KD, typename L>
__device__ __forceinline__ void score_tiles(f32x4 (&s)[L::N], const u16 *X, const u16 *Y, int lane) {
    constexpr int PL = kTile<C, KD>, P = Cfg<T>::in, N = L::N;
    const int g = (lane >> 4), i = (lane & 15);
#pragma unroll
    for (int j = 0; j < N; ++j) s[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < KD / 32; k += 2) {
        bf16x8 a[2][N][P], b[2][N][P];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int p = 0; p < P; ++p)
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    if (j > 0 && L::O(j) == L::O(j - 1)) b[h][j][p] = b[h][j - 1][p];
                    else b[h][j][p] = frag_row<KD>(X + p * PL, 16 * L::O(j), k + h, g, i);
                    a[h][j][p] = frag_row<KD>(Y + p * PL, 16 * L::n(j), k + h, g, i);
                }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int p = 0; p < P; ++p)
#pragma unroll
                for (int q = 0; q < P; ++q)
                    if (p + q < 3)
#pragma unroll
                        for (int j = 0; j < N; ++j) s[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[h][j][p], b[h][j][q], s[j], 0, 0, 0);
    }
}

// The decay factors of the tile (O, n) times `scale`, 0 where the token does not see the other. REV: row tokens see later
// ones. One factor per accumulator element.
template <int C, bool REV, int O, int n>
__device__ __forceinline__ f32x4 tile_decay(const Decays<C> &d, float scale, int lane) {
    const int g = (lane >> 4), i = (lane & 15);
    constexpr int o = 16 * O, m = 16 * n;
    f32x4 f;
    if constexpr (O != n) {
        const float row = REV ? d.to[o + i] * d.mid[n][O] : d.from[o + i] * d.mid[O][n];
        const f32x4 col = *reinterpret_cast<const f32x4 *>(REV ? &d.from[m + 4 * g] : &d.to[m + 4 * g]);
#pragma unroll
        for (int r = 0; r < 4; ++r) f[r] = row * col[r];
    } else {
        const f32x4 hi = *reinterpret_cast<const f32x4 *>(&d.hi[m + 4 * g]), lo = *reinterpret_cast<const f32x4 *>(&d.lo[m + 4 * g]);
        const float h = d.hi[o + i], l = d.lo[o + i];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            float x = (h - hi[r]) + (l - lo[r]);
            if (REV) x = -x;
            f[r] = exp_f32((REV ? 4 * g + r >= i : 4 * g + r <= i) ? x : -1e30f) * scale;
        }
    }
    return f;
}

// Four consecutive scores of row token 16 ot + i into the score tile's planes ([row token][other token]).
template <int C>
__device__ __forceinline__ void store_scores(u16 *M, const float *x, int ot, int nt, int lane) {
    constexpr int PL = kTile<C, kScoreRow>;
    u16 *dst = M + block<kScoreRow>(16 * ot) + at<kScoreRow>((lane & 15), 16 * nt + 4 * ((lane >> 4)));
    float r[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
    for (int p = 0; p < kPlanes; ++p) {
        const uint2 w = make_uint2(pack_bf16x2(r[0], r[1]), pack_bf16x2(r[2], r[3]));
        *reinterpret_cast<uint2 *>(dst + p * PL) = w;
        r[0] -= __uint_as_float(w.x << 16);
        r[1] -= __uint_as_float(w.x & 0xffff0000u);
        r[2] -= __uint_as_float(w.y << 16);
        r[3] -= __uint_as_float(w.y & 0xffff0000u);
    }
}

// The forward walk's decayed, masked scores of the tiles L into M. True where a row of X or Y holds an infinity or NaN: the
// product of a token's own two rows then is neither finite, and the tiles on the diagonal hold those.
template <typename T, int C, int KD, typename L>
__device__ __forceinline__ bool scores(const Decays<C> &d, const u16 *X, const u16 *Y, u16 *M, float scale, int lane) {
    f32x4 s[L::N];
    score_tiles<T, C, KD, L>(s, X, Y, lane);
    bool special = false;
    static_for<0, L::N>([&](auto Nc) {
        constexpr int j = decltype(Nc)::value, O = L::O(j), n = L::n(j);
        if constexpr (O == n) special |= !finite((s[j][0] + s[j][1]) + (s[j][2] + s[j][3]));
        const f32x4 f = tile_decay<C, false, O, n>(d, scale, lane);
        float x[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) x[r] = n == O && 4 * ((lane >> 4)) + r > (lane & 15) ? 0.f : s[j][r] * f[r];
        store_scores<C>(M, x, O, n, lane);
    });
    return special;
}

// The backward walk's, of both products (K Q^T into M1, V dO^T into M2, row token tile O), and with `sums` the tiles' sums of
// w = both scores times the decay, the diagonal left out: over the seen tokens for each seeing one (rowp) and over the seeing
// tokens for each seen one (colp).
template <typename T, int C, int KD, int VD, typename L>
__device__ __forceinline__ void scores_bwd(const Decays<C> &d, const u16 *Q, const u16 *K, const u16 *V, const u16 *G, u16 *M1, u16 *M2, float scale,
                                           bool sums, float *rowp, float *colp, int lane) {
    f32x4 p[L::N], dp[L::N];
    score_tiles<T, C, KD, L>(p, K, Q, lane);
    score_tiles<T, C, VD, L>(dp, V, G, lane);
    static_for<0, L::N>([&](auto Nc) {
        constexpr int j = decltype(Nc)::value, O = L::O(j), m = L::n(j);
        const f32x4 f = tile_decay<C, true, O, m>(d, scale, lane);
        const int i = (lane & 15), ii = 4 * ((lane >> 4));
        float s1[4], s2[4], w[4], cs = 0.f;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const bool sees = m != O || ii + r >= i;
            s1[r] = sees ? p[j][r] * f[r] : 0.f;
            s2[r] = sees ? dp[j][r] * f[r] : 0.f;
            w[r] = m != O || ii + r > i ? p[j][r] * s2[r] : 0.f;
            cs += w[r];
        }
        store_scores<C>(M1, s1, O, m, lane);
        store_scores<C>(M2, s2, O, m, lane);
        if (sums) {
            f32x4 rs;
#pragma unroll
            for (int r = 0; r < 4; ++r) rs[r] = group_sum<16>(w[r]);
            cs += __shfl_xor(cs, 16);
            cs += __shfl_xor(cs, 32);
            if (i == 0) *reinterpret_cast<f32x4 *>(&rowp[O * C + 16 * m + ii]) = rs;
            if (lane < 16) colp[m * C + 16 * O + i] = cs;
        }
    });
}

// The tiles on the masked side of the diagonal that share a 32-wide contraction with a diagonal tile are 0
// (written once; the chunks write the other tiles only).
template <int C>
__device__ __forceinline__ void zero_masked_scores(u16 *M, bool rev, int tid, int nt) {
    constexpr int PL = kTile<C, kScoreRow>;
    for (int x = tid; x < C / 32 * 16 * 16 * kPlanes; x += nt) {
        const int p = x / (C / 32 * 256), y = x % (C / 32 * 256), pair = y / 256, r = y % 256 / 16, c = y % 16;
        const int row = 32 * pair + (rev ? 16 : 0) + r, col = 32 * pair + (rev ? 0 : 16) + c;
        M[p * PL + at<kScoreRow>(row, col)] = 0;
    }
}

// O = diag(row) X S for the wave's columns, from the state S before (after, REV) the chunk.
template <typename T, int C, int KD, int NC>
__device__ __forceinline__ void inter(f32x4 (&O)[C / 16][NC], const f32x4 (&S)[KD / 16][NC], const u16 *X, const float *row,
                                      int lane) {
    constexpr int PL = kTile<C, KD>, PI = Cfg<T>::in;
    const int g = (lane >> 4), i = (lane & 15);
#pragma unroll
    for (int t = 0; t < C / 16; ++t)
#pragma unroll
        for (int c = 0; c < NC; ++c) O[t][c] = f32x4{0.f, 0.f, 0.f, 0.f};
    // The rows of the next 32 columns are read while the products of these run.
    bf16x8 a[2][C / 16][PI];
    auto read = [&](int k) {
#pragma unroll
        for (int t = 0; t < C / 16; ++t)
#pragma unroll
            for (int p = 0; p < PI; ++p) a[k % 2][t][p] = frag_row<KD>(X + p * PL, 16 * t, k, g, i);
    };
    read(0);
#pragma unroll
    for (int k = 0; k < KD / 32; ++k) {
        if (k + 1 < KD / 32) read(k + 1);
        __builtin_amdgcn_sched_barrier(0);
        bf16x8 s[NC][kPlanes];
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            float x[8];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                x[r] = S[2 * k][c][r];
                x[4 + r] = S[2 * k + 1][c][r];
            }
            split8(x, s[c]);
        }
#pragma unroll
        for (int p = 0; p < PI; ++p)
#pragma unroll
            for (int q = 0; q < kPlanes; ++q)
                if (p + q < kPlanes)
#pragma unroll
                    for (int t = 0; t < C / 16; ++t)
#pragma unroll
                        for (int c = 0; c < NC; ++c)
                            O[t][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[k % 2][t][p], s[c][q], O[t][c], 0, 0, 0);
    }
#pragma unroll
    for (int t = 0; t < C / 16; ++t) {
        const f32x4 f = *reinterpret_cast<const f32x4 *>(row + 16 * t + 4 * g);
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int c = 0; c < NC; ++c) O[t][c][r] *= f[r];
    }
}

// S = all S + Y^T diag(w) V for the wave's columns (V's operands in v).
template <typename T, int C, int KD, int NC>
__device__ __forceinline__ void update(f32x4 (&S)[KD / 16][NC], const bf16x8 (&v)[C / 32][NC][Cfg<T>::in], const u16 *Y,
                                       const float *w, float all, int lane) {
    constexpr int PL = kTile<C, KD>, PI = Cfg<T>::in;
    const int g = (lane >> 4), i = (lane & 15);
#pragma unroll
    for (int k = 0; k < KD / 16; ++k)
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int r = 0; r < 4; ++r) S[k][c][r] *= all;
#pragma unroll
    for (int j = 0; j < C / 32; ++j) {
        const f32x4 w0 = *reinterpret_cast<const f32x4 *>(w + 32 * j + 4 * g);
        const f32x4 w1 = *reinterpret_cast<const f32x4 *>(w + 32 * j + 16 + 4 * g);
        bf16x8 u[NC][kPlanes];
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            float x[8], y[8];
            unpack_frag(v[j][c][PI - 1], x);
#pragma unroll
            for (int p = PI - 2; p >= 0; --p) {
                unpack_frag(v[j][c][p], y);
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] += y[e];
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x[e] *= w0[e];
                x[4 + e] *= w1[e];
            }
            split8(x, u[c]);
        }
        constexpr int KB = PI > 1 ? 2 : 4;   // rows of tiles read ahead
        bf16x8 a[2][KB][PI];
        auto read = [&](int b) {
#pragma unroll
            for (int k = 0; k < KB; ++k)
#pragma unroll
                for (int p = 0; p < PI; ++p)
                    if (b * KB + k < KD / 16) a[b % 2][k][p] = frag_tr<KD>(Y + p * PL, 32 * j, 16 * (b * KB + k), g, i);
        };
        read(0);
#pragma unroll
        for (int b = 0; b * KB < KD / 16; ++b) {
            if ((b + 1) * KB < KD / 16) read(b + 1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int p = 0; p < PI; ++p)
#pragma unroll
                for (int q = 0; q < kPlanes; ++q)
                    if (p + q < kPlanes)
#pragma unroll
                        for (int k = 0; k < KB; ++k)
#pragma unroll
                            for (int c = 0; c < NC; ++c)
                                if (b * KB + k < KD / 16)
                                    S[b * KB + k][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[b % 2][k][p], u[c][q], S[b * KB + k][c], 0, 0, 0);
        }
    }
}

template <typename T, int C, int NC, int LDV>
__device__ __forceinline__ void load_v(bf16x8 (&v)[C / 32][NC][Cfg<T>::in], const u16 *V, int col, int lane) {
    constexpr int PL = kTile<C, LDV>;
#pragma unroll
    for (int j = 0; j < C / 32; ++j)
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int p = 0; p < Cfg<T>::in; ++p)
                v[j][c][p] = frag_tr<LDV>(V + p * PL, 32 * j, col + 16 * c, (lane >> 4), (lane & 15));
}

// O += M V, M the masked scores. A masked score is 0, and 0 times an infinity or NaN of a token that the row
// does not see would be NaN: where V holds one, its elements leave the product and are added one by one.
template <typename T, int C, int NC, int LDV, bool REV>
__device__ __forceinline__ void intra(f32x4 (&O)[C / 16][NC], const bf16x8 (&v0)[C / 32][NC][Cfg<T>::in], const u16 *M,
                                      const u16 *V, int col, int lane) {
    constexpr int PL = kTile<C, kScoreRow>, PI = Cfg<T>::in;
    const int g = (lane >> 4), i = (lane & 15);
    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
    u16x2 most = {0, 0};
#pragma unroll
    for (int j = 0; j < C / 32; ++j)
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const u32x4 w = __builtin_bit_cast(u32x4, v0[j][c][0]);
#pragma unroll
            for (int k = 0; k < 4; ++k) most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, w[k] & 0x7fff7fffu));
        }
    const bool odd = most[0] >= 0x7f80 || most[1] >= 0x7f80;
    auto product = [&](const bf16x8 (&v)[C / 32][NC][PI]) {
#pragma unroll
        for (int j = 0; j < C / 32; ++j) {
            bf16x8 a[C / 16][kPlanes];
#pragma unroll
            for (int t = 0; t < C / 16; ++t)
                if (REV ? 2 * j + 1 >= t : 2 * j <= t)
#pragma unroll
                    for (int p = 0; p < kPlanes; ++p) a[t][p] = frag_row<kScoreRow>(M + p * PL, 16 * t, j, g, i);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int p = 0; p < kPlanes; ++p)
#pragma unroll
                for (int q = 0; q < PI; ++q)
                    if (p + q < kPlanes)
#pragma unroll
                        for (int t = 0; t < C / 16; ++t)
#pragma unroll
                            for (int c = 0; c < NC; ++c)
                                if (REV ? 2 * j + 1 >= t : 2 * j <= t)
                                    O[t][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[t][p], v[j][c][q], O[t][c], 0, 0, 0);
        }
    };
    if (!__any(odd)) {
        product(v0);
        return;
    }
    bf16x8 v[C / 32][NC][PI];
#pragma unroll
    for (int j = 0; j < C / 32; ++j)
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            u32x4 w = __builtin_bit_cast(u32x4, v0[j][c][0]);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if ((w[k] & 0x7f80u) == 0x7f80u) w[k] &= 0xffff0000u;
                if ((w[k] & 0x7f800000u) == 0x7f800000u) w[k] &= 0xffffu;
            }
            v[j][c][0] = __builtin_bit_cast(bf16x8, w);
#pragma unroll
            for (int p = 1; p < PI; ++p) v[j][c][p] = v0[j][c][p];
        }
    product(v);
    for (int n = 0; n < C; ++n)
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const float x = __uint_as_float(uint32_t(V[at<LDV>(n, col + 16 * c + i)]) << 16);
            const bool bad = (__float_as_uint(x) & 0x7f800000u) == 0x7f800000u;
            if (!__any(bad)) continue;
#pragma unroll
            for (int t = 0; t < C / 16; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int o = 16 * t + 4 * g + r;
                    if (!bad || (REV ? n < o : n > o)) continue;
                    float m = 0.f;
#pragma unroll
                    for (int p = kPlanes - 1; p >= 0; --p) m += __uint_as_float(uint32_t(M[p * PL + at<kScoreRow>(o, n)]) << 16);
                    O[t][c][r] += m * x;
                }
        }
}

// ---- infinite values -----------------------------------------------------------------------------

// An infinity has no planes behind the first (their rest would be infinity - infinity), and a plane that is 0 times an infinity
// is NaN. So the products above make NaN of every output and state element that an infinity reaches, and of those alone. Which of
// them the recurrence makes +-infinity is found by running it, token by token in float32, behind the walk over a row that holds
// one, and what is not finite there is written over the NaN. The finite results stay as they are, and so does a row of finite
// values and NaN. Such a row takes some six times as long.

// Whether there are infinities and NaNs among the values that this lane was shown.
struct Kinds {
    bool inf, nan;

    __device__ __forceinline__ void add(float x) {
        inf |= __builtin_fabsf(x) == __builtin_inff();
        nan |= x != x;
    }
    template <int C, int D>
    __device__ __forceinline__ void tile(const u16 *tile, int lane) {   // the first plane; the lane's share
        for (int x = lane; x < C * D / 4; x += 64) {
            const int row = x / (D / 4);
            const uint2 w = *reinterpret_cast<const uint2 *>(tile + row * D + row / 16 * 8 + x % (D / 4) * 4);
            add(__uint_as_float(w.x << 16));
            add(__uint_as_float(w.x & 0xffff0000u));
            add(__uint_as_float(w.y << 16));
            add(__uint_as_float(w.y & 0xffff0000u));
        }
    }
};
template <int KD, int NC>
__device__ __forceinline__ Kinds kinds(const f32x4 (&S)[KD / 16][NC]) {
    Kinds k = {false, false};
#pragma unroll
    for (int y = 0; y < KD / 16; ++y)
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int r = 0; r < 4; ++r) k.add(S[y][c][r]);
    return k;
}
template <int KD, int NC>
__device__ __forceinline__ bool finite_state(const f32x4 (&S)[KD / 16][NC]) {
    const Kinds k = kinds<KD, NC>(S);
    return !k.inf && !k.nan;
}
// Four consecutive elements of a tile's row, and one.
template <typename T, int C, int D>
__device__ __forceinline__ void tile_row4(float (&x)[4], const u16 *tile, int row, int col) {
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = 0.f;
#pragma unroll
    for (int p = Cfg<T>::in - 1; p >= 0; --p) {
        const uint2 w = *reinterpret_cast<const uint2 *>(tile + p * kTile<C, D> + at<D>(row, col));
        x[0] += __uint_as_float(w.x << 16);
        x[1] += __uint_as_float(w.x & 0xffff0000u);
        x[2] += __uint_as_float(w.y << 16);
        x[3] += __uint_as_float(w.y & 0xffff0000u);
    }
}
template <typename T, int C, int D>
__device__ __forceinline__ float tile_at(const u16 *tile, int row, int col) {
    float x = 0.f;
#pragma unroll
    for (int p = Cfg<T>::in - 1; p >= 0; --p) x += __uint_as_float(uint32_t(tile[p * kTile<C, D> + at<D>(row, col)]) << 16);
    return x;
}

// A chunk's first `rows` tokens one by one: S = exp(g) S + y v^T; out(t, c, the column's x S without the scale) in every lane (OUT).
// kdim: the rows' length; beyond it S stays 0.
template <typename T, int C, int KD, int NC, int LDV, bool OUT, typename F>
__device__ __forceinline__ void recur(f32x4 (&S)[KD / 16][NC], const u16 *X, const u16 *Y, const u16 *V, const Decays<C> &d, int rows, int kdim,
                                      int col, int lane, F &&out) {
    const int g = (lane >> 4), i = (lane & 15);
#pragma unroll 1
    for (int t = 0; t < rows; ++t) {
        const float e = exp_f32(t ? (d.hi[t] - d.hi[t - 1]) + (d.lo[t] - d.lo[t - 1]) : d.hi[0] + d.lo[0]);
        float v[NC], o[NC];
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            v[c] = tile_at<T, C, LDV>(V, t, col + 16 * c + i);
            o[c] = 0.f;
        }
#pragma unroll
        for (int k = 0; k < KD / 16; ++k) {
            float y[4], x[4];
            tile_row4<T, C, KD>(y, Y, t, 16 * k + 4 * g);
            if constexpr (OUT) tile_row4<T, C, KD>(x, X, t, 16 * k + 4 * g);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const bool in = 16 * k + 4 * g + r < kdim;
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    S[k][c][r] = in ? __builtin_fmaf(e, S[k][c][r], y[r] * v[c]) : 0.f;
                    if constexpr (OUT) o[c] += in ? x[r] * S[k][c][r] : 0.f;
                }
            }
        }
        if constexpr (OUT) {
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                o[c] += __shfl_xor(o[c], 16);
                o[c] += __shfl_xor(o[c], 32);
                out(t, c, o[c]);
            }
        }
    }
}

// A float32 matrix of a (batch row, head): rows x cols, with its strides (spans less than 2^31 bytes).
struct Mat {
    float *p;
    int64_t row, col;
};
// Byte offset of the state's element (16 k + 4 g + r, col + 16 c + i), kNone outside.
__device__ __forceinline__ uint32_t state_at(const Mat &m, int rows, int cols, int y, int x) {
    return y < rows && x < cols ? (uint32_t(y) * uint32_t(m.row) + uint32_t(x) * uint32_t(m.col)) * 4 : kNone;
}
template <int KD, int NC>
__device__ __forceinline__ void load_state(f32x4 (&S)[KD / 16][NC], const Mat &m, int rows, int cols, int col, int lane) {
    const int g = (lane >> 4), i = (lane & 15);
    rows = m.p ? afresh(rows) : 0;
    cols = afresh(cols);
    const __amdgpu_buffer_rsrc_t buf = buffer(m.p);
#pragma unroll
    for (int k = 0; k < KD / 16; ++k)
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                uint32_t at = state_at(m, rows, cols, 16 * k + 4 * g + r, col + 16 * c + i);
                asm("" : "+v"(at));
                S[k][c][r] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(buf, at, 0, 0));
            }
}
// ODD: only the elements that are not finite.
template <int KD, int NC, bool ODD = false>
__device__ __forceinline__ void store_state(const f32x4 (&S)[KD / 16][NC], const Mat &m, int rows, int cols, int col, int lane) {
    const int g = (lane >> 4), i = (lane & 15);
    rows = afresh(rows);
    cols = afresh(cols);
    const __amdgpu_buffer_rsrc_t buf = buffer(m.p);
#pragma unroll
    for (int k = 0; k < KD / 16; ++k)
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                uint32_t at = state_at(m, rows, cols, 16 * k + 4 * g + r, col + 16 * c + i);
                if (ODD && finite(S[k][c][r])) at = kNone;
                asm("" : "+v"(at));
                __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(S[k][c][r]), buf, at, 0, 0);
            }
}
// The wave's share of <S, m>.
template <int KD, int NC>
__device__ __forceinline__ float dot_state(const f32x4 (&S)[KD / 16][NC], const Mat &m, int rows, int cols, int col, int lane) {
    const int g = (lane >> 4), i = (lane & 15);
    rows = afresh(rows);
    cols = afresh(cols);
    const __amdgpu_buffer_rsrc_t buf = buffer(m.p);
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < KD / 16; ++k)
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            float w[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                uint32_t at = state_at(m, rows, cols, 16 * k + 4 * g + r, col + 16 * c + i);
                asm("" : "+v"(at));
                w[r] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(buf, at, 0, 0));
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                // Outside the matrix the state is 0, whatever its accumulator holds.
                const bool in = 16 * k + 4 * g + r < rows && col + 16 * c + i < cols;
                sum = __builtin_fmaf(in ? S[k][c][r] : 0.f, w[r], sum);
            }
        }
    return sum;
}

// Orders a wave's LDS accesses of different types around it (they are in order in the hardware; the compiler may take a store
// of one type and a load of another for independent).
__device__ __forceinline__ void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// One output element; `at` counts elements, kNone drops it.
template <typename T, bool F32>
__device__ __forceinline__ void store_element(float x, const __amdgpu_buffer_rsrc_t &buf, uint32_t at) {
    constexpr uint32_t ES = F32 ? 4 : sizeof(T);
    at = at == kNone ? kNone : at * ES;
    if constexpr (ES == 4) __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(x), buf, at, 0, 0);
    else if constexpr (std::is_same_v<T, bf16_t>) __builtin_amdgcn_raw_buffer_store_b16(short(pack_bf16x2(x, 0.f)), buf, at, 0, 0);
    else __builtin_amdgcn_raw_buffer_store_b16(short(pack_f16x2(x, 0.f)), buf, at, 0, 0);
}

// The wave's C x 16 NC outputs to rows of T, or of float32 (F32). In 16-byte pieces (VEC) they go
// through the wave's own columns of a tile that no other wave reads any more: 16-bit rows as they lie there, the 16-bit types'
// float32 shares half a chunk at a time, each row in the place of two rows of the tile. float32 tensors' rows go out by the lane, in
// 64-byte runs (through LDS 3 % slower on one card, 65,536 tokens of 40 heads; cards differ by as much).
template <typename T, int C, int NC, int LDV, bool VEC, bool F32>
__device__ __forceinline__ void store_out(const f32x4 (&O)[C / 16][NC], void *out, uint32_t stride, int t0, int rows, int cols,
                                          u16 *tile, int col, int lane) {
    const int g = (lane >> 4), i = (lane & 15);
    constexpr uint32_t ES = F32 ? 4 : sizeof(T);
    const __amdgpu_buffer_rsrc_t buf = buffer(static_cast<char *>(out) + uint64_t(unsigned(t0)) * stride * ES);
    const uint32_t step = stride * ES;
    if constexpr (VEC && sizeof(T) == 2) wave_fence();
    if constexpr (VEC && !F32 && sizeof(T) == 2) {
#pragma unroll
        for (int t = 0; t < C / 16; ++t)
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int r = 0; r < 4; r += 2) {
                    const uint32_t w = std::is_same_v<T, bf16_t> ? pack_bf16x2(O[t][c][r], O[t][c][r + 1]) : pack_f16x2(O[t][c][r], O[t][c][r + 1]);
                    tile[block<LDV>(16 * t) + at<LDV>(4 * g + r, col + 16 * c + i)] = u16(w);
                    tile[block<LDV>(16 * t) + at<LDV>(4 * g + r + 1, col + 16 * c + i)] = u16(w >> 16);
                }
        wave_fence();
        constexpr int PR = 2 * NC;   // pieces of a row
#pragma unroll
        for (int n = 0; n < C * PR / 64; ++n) {
            const int row = n * (64 / PR) + int(unsigned(lane) / PR), c = int(unsigned(lane) % PR) * 8;
            const u16 *src = tile + block<LDV>(n * (64 / PR));   // whole tiles of 16 rows down
            const uint2 w0 = *reinterpret_cast<const uint2 *>(src + at<LDV>(int(unsigned(lane) / PR), col + c)),
                        w1 = *reinterpret_cast<const uint2 *>(src + at<LDV>(int(unsigned(lane) / PR), col + c + 4));
            const u32x4 w = {w0.x, w0.y, w1.x, w1.y};
            const bool live = row < rows && col + c < cols;
            __builtin_amdgcn_raw_buffer_store_b128(w, buf, live ? uint32_t(row) * step + uint32_t(col + c) * 2 : kNone, 0, 0);
        }
    } else if constexpr (VEC && sizeof(T) == 2) {
        constexpr int PR = 4 * NC, TH = C / 32;   // pieces of a row, row tiles of half a chunk
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int t = 0; t < TH; ++t)
#pragma unroll
                for (int c = 0; c < NC; ++c)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        // element x of row n: row 2 n + x / (8 NC), column 2 (x mod 8 NC) of the tile
                        const int n = 4 * g + r, x = 16 * c + i;
                        *reinterpret_cast<float *>(tile + block<LDV>(32 * t) + at<LDV>(2 * n + x / (8 * NC), col + x % (8 * NC) * 2)) =
                            O[h * TH + t][c][r];
                    }
            wave_fence();
#pragma unroll
            for (int m = 0; m < C / 2 * PR / 64; ++m) {
                const int q = m * 64 + lane, n = q / PR, x = q % PR * 4;
                const int row = 2 * n + x / (8 * NC), cc = col + x % (8 * NC) * 2;
                const uint2 w0 = *reinterpret_cast<const uint2 *>(tile + at<LDV>(row, cc)), w1 = *reinterpret_cast<const uint2 *>(tile + at<LDV>(row, cc + 4));
                const u32x4 w = {w0.x, w0.y, w1.x, w1.y};
                const int to = h * (C / 2) + n;
                const bool live = to < rows && col + x < cols;
                __builtin_amdgcn_raw_buffer_store_b128(w, buf, live ? uint32_t(to) * step + uint32_t(col + x) * 4 : kNone, 0, 0);
            }
            wave_fence();
        }
    } else {
#pragma unroll
        for (int t = 0; t < C / 16; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int n = 16 * t + 4 * g + r;
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    const int x = col + 16 * c + i;
                    store_element<T, F32>(O[t][c][r], buf, n < rows && x < cols ? uint32_t(n) * stride + uint32_t(x) : kNone);
                }
            }
    }
}

// dot[n] = sum over the wave's columns of O[n][x] Z[n][x], into part[n] (lanes i == 0 write). A transposed read of Z has O's layout.
template <typename T, int C, int NC, int LDZ>
__device__ __forceinline__ void dot_rows(const f32x4 (&O)[C / 16][NC], const u16 *Z, int col, float *part, int lane) {
    constexpr int PL = kTile<C, LDZ>, PI = Cfg<T>::in;
    const int g = (lane >> 4), i = (lane & 15);
#pragma unroll
    for (int j = 0; j < C / 32; ++j) {
        float s[8] = {};
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            float z[8], y[8];
            unpack_frag(frag_tr<LDZ>(Z + (PI - 1) * PL, 32 * j, col + 16 * c, g, i), z);
#pragma unroll
            for (int p = PI - 2; p >= 0; --p) {
                unpack_frag(frag_tr<LDZ>(Z + p * PL, 32 * j, col + 16 * c, g, i), y);
#pragma unroll
                for (int e = 0; e < 8; ++e) z[e] += y[e];
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) s[e] = __builtin_fmaf(O[2 * j + e / 4][c][e % 4], z[e], s[e]);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) s[e] = group_sum<16>(s[e]);
        if (i == 0) {
            *reinterpret_cast<f32x4 *>(part + 32 * j + 4 * g) = f32x4{s[0], s[1], s[2], s[3]};
            *reinterpret_cast<f32x4 *>(part + 32 * j + 16 + 4 * g) = f32x4{s[4], s[5], s[6], s[7]};
        }
    }
}

__device__ __forceinline__ float wave_sum(float x) {
    x = group_sum<16>(x);
    x += __shfl_xor(x, 16);
    x += __shfl_xor(x, 32);
    return x;
}

}  // namespace la
}  // namespace mm
