// mm_linattn.hip -- gfx950 linear attention with one decay for each head: chunked forward and backward
// (mm_linattn_dev.h has the mathematics and the operands' layouts). The single-token step and the plan of a call are
// in mm_linattn_api.hip.
//
// A walk takes one (batch row, head), or a segment of it, through its chunks in order, the state in the
// accumulators of its waves: every tensor is read once and every output written once. Rows with too few
// (batch row, head) pairs for the card are cut into segments; a first pass then gathers what each segment
// adds to the state, a second joins those, and the walks start from the joined states.
//
// Built once per input type: this file for float32, mm_linattn_f16.hip / mm_linattn_bf16.hip, which set
// MM_LINATTN_TYPE, for the 16-bit types.
#ifndef MM_LINATTN_TYPE
#define MM_LINATTN_TYPE float
#define MM_LINATTN_COMMON
#endif

#include <algorithm>
#include <atomic>

#include "mm_linattn_dev.h"
#include "mm_linattn_host.h"

namespace mm {
namespace la {

constexpr int kWaves = 4, kThreads = 64 * kWaves;

// The kernel's only argument, read where this stands. A walk keeps the few numbers that every chunk needs (a tensor's first
// row and stride, 3 scalars each) and reads the others when it needs them: all of them, some 60, do not fit the scalar registers, and a
// build that spilled them lost the low word of an output's address (a tuple of arguments was overwritten in part before it was
// spilled; one instance of 144 stored to wrong addresses).
template <typename A>
__device__ __forceinline__ A own_args() {
    typedef const __attribute__((address_space(4))) A *Args;
    Args args = (Args)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(args));
    return *(const A *)args;
}

template <typename T>
__device__ __forceinline__ Rows<T> rows_of(const View &v, int b, int h, int d, int col0 = 0) {
    return Rows<T>{afresh(reinterpret_cast<const T *>(v.p) + b * v.batch + int64_t(unsigned(h) / unsigned(v.share)) * v.head + col0), uint32_t(afresh(int(v.seq) * int(sizeof(T)))), afresh(d - col0)};
}
// A workgroup's place: its batch row, head and segment, and the segment's tokens.
struct Place {
    int slice, seg, b, h, beg, end;
};
template <typename A>
__device__ __forceinline__ Place place_of(const A &a, int slices) {
    const unsigned id = unsigned(afresh(int(blockIdx.x))), seg = id / unsigned(slices), pair = seg / unsigned(a.segs);
    Place p;
    p.slice = afresh(int(id % unsigned(slices)));
    p.seg = afresh(int(seg % unsigned(a.segs)));
    p.h = afresh(int(pair % unsigned(a.heads)));
    p.b = afresh(int(pair / unsigned(a.heads)));
    p.beg = afresh(p.seg * int(a.seg_len));
    p.end = afresh(min(int(a.seqlen), p.beg + int(a.seg_len)));
    return p;
}
// The log decays of a (batch row, head).
struct Gates {
    const char *p;
    int64_t stride;   // bytes
    mm_dtype type;

    // A lane's token's bits in the chunk at t0, 0 past `end`; see decode_g.
    template <int C>
    __device__ __forceinline__ uint32_t load(int t0, int end, int lane) const {
        const int t = t0 + lane;
        return lane < C && t < end ? load_g_raw(p + t * stride, type, 0) : 0u;
    }
};
template <typename A>
__device__ __forceinline__ Gates gates_of(const A &a, const Place &p) {
    const int64_t size = a.gtype == MM_FLOAT32 ? 4 : 2;
    return Gates{afresh(static_cast<const char *>(a.g) + (p.b * a.g_batch + p.h * a.g_head) * size), afresh(a.g_seq * size), mm_dtype(afresh(int(a.gtype)))};
}

// The walk once more by the recurrence, for what is not finite in it (see mm_linattn_dev.h). Its arguments are read again, so that
// nothing of it takes registers while the products run.
template <typename T, int KD, int NC, bool DOT, bool VEC, bool F32>
__device__ __forceinline__ void infinite_rows(char *smem) {
    constexpr int C = Cfg<T>::C, PI = Cfg<T>::in, W = 64 * NC, ES = F32 ? 4 : sizeof(T);
    auto args = [] { return own_args<WalkArgs>(); };
    u16 *X = reinterpret_cast<u16 *>(smem), *Y = X + PI * kTile<C, KD>, *V = Y + PI * kTile<C, KD>;
    Decays<C> *dec = reinterpret_cast<Decays<C> *>(V + (DOT ? 2 : 1) * PI * kTile<C, W> + kPlanes * kTile<C, kScoreRow>);
    const int tid = afresh_lane(threadIdx.x), wave = __builtin_amdgcn_readfirstlane(tid / 64), lane = tid & 63, col = wave * 16 * NC;
    const Place p = place_of(args(), 1);
    f32x4 S[KD / 16][NC];
    auto begin = [&] {
        const WalkArgs a = args();
        const int64_t bh = int64_t(p.b) * a.heads + p.h;
        load_state<KD, NC>(S, Mat{a.s0.p ? a.s0.p + (bh * a.segs + p.seg) * a.s0_step : nullptr, a.s0.row, a.s0.col}, a.kdim, a.cdim, col, lane);
    };
    auto stage = [&](int t0) {
        const WalkArgs a = args();
        const int rows = min(C, p.end - t0);
        __syncthreads();
        {
            Stage<T, C, KD, kThreads, VEC> s;
            s.load(rows_of<T>(a.x, p.b, p.h, a.kdim), t0, rows, tid);
            s.store(X, tid);
            s.load(rows_of<T>(a.y, p.b, p.h, a.kdim), t0, rows, tid);
            s.store(Y, tid);
        }
        {
            Stage<T, C, W, kThreads, VEC> s;
            s.load(rows_of<T>(a.v, p.b, p.h, a.cdim), t0, rows, tid);
            s.store(V, tid);
        }
        if (wave == 0) make_decays<C>(dec[0], decode_g(gates_of(a, p).template load<C>(t0, p.end, lane), a.gtype), a.scale, lane);
        __syncthreads();
    };
    // NaN alone needs no second look.
    begin();
    Kinds seen = kinds<KD, NC>(S);
#pragma unroll 1
    for (int t0 = p.beg; t0 < p.end; t0 += C) {
        stage(t0);
        seen.tile<C, KD>(X, lane);
        seen.tile<C, KD>(Y, lane);
        seen.tile<C, W>(V, lane);
        seen.add(dec[0].hi[C - 1]);
    }
    const bool inf = __syncthreads_or(seen.inf), nan = __syncthreads_or(seen.nan);
    if (nan && !inf) return;
    begin();
    auto keep = [&](const WalkArgs &a, int64_t block) {
        const int64_t bh = int64_t(p.b) * a.heads + p.h;
        store_state<KD, NC, true>(S, Mat{a.ck + (bh * a.blocks + block) * a.kdim * a.cdim, a.cdim, 1}, a.kdim, a.cdim, col, lane);
    };
#pragma unroll 1
    for (int t0 = p.beg; t0 < p.end; t0 += C) {
        if constexpr (DOT) {
            const WalkArgs a = args();
            if (a.ck && t0 > 0 && t0 % kBlock == 0) keep(a, t0 / kBlock - 1);
        }
        stage(t0);
        const WalkArgs a = args();
        const __amdgpu_buffer_rsrc_t to = buffer(static_cast<char *>(a.out) + (p.b * a.out_batch + p.h * a.out_head + t0 * a.out_seq) * ES);
        recur<T, C, KD, NC, W, true>(S, X, Y, V, dec[0], min(C, p.end - t0), a.kdim, col, lane, [&](int t, int c, float x) {
            x *= a.scale;
            const int at = col + 16 * c + (lane & 15);
            store_element<T, F32>(x, to, !finite(x) && lane < 16 && at < a.cdim ? uint32_t(t) * uint32_t(a.out_seq) + uint32_t(at) : kNone);
        });
    }
    const WalkArgs a = args();
    if (a.s1.p && p.seg == a.segs - 1)
        store_state<KD, NC, true>(S, Mat{a.s1.p + (int64_t(p.b) * a.heads + p.h) * a.kdim * a.cdim, a.s1.row, a.s1.col}, a.kdim, a.cdim, col, lane);
    if constexpr (DOT) {
        if (a.ck && a.ck_last && p.seg == a.segs - 1) keep(a, a.blocks - 1);
    }
}

// Forward walk: out = scale (masked X Y^T) V + ..., KD the padded length of X's rows, 64 NC that of V's,
// 16 NC columns per wave. DOT: also e[t] = (the product with the state alone) . Z_t, and the state at every
// kBlock-th token into ck (the decays' gradient).
//
// Per chunk: stage X, Y and V; scores (each wave its tiles, into M) and the product with the state; the product of M and V,
// the state's update, the outputs. The waves share X, Y and M through LDS and split V's columns, so that a wave's part of the
// state never leaves its accumulators. At dk 128, dv 64, bfloat16 a wave issues 124 matrix and some 940 other vector
// instructions per 64 tokens and the LDS works 3,200 cycles, a third of them bank conflicts; with 2 workgroups on a CU (203
// registers, 69 KB) a chunk of both takes 5.6 us, of one alone 4.2. While a CU has work its vector units are busy 44 % of the
// time, its matrix cores 23 %, its LDS 38 %: with one or two waves per SIMD nothing covers a wave's latencies between the three
// barriers. 4 x 4,096 tokens, 80 heads: 361 us, 1.0 TB/s of its 360 MB and 460 TFLOP/s on the matrix cores, split planes counted.
// With two planes of the state, three workgroups at 168 registers spilled (457 us for 128 heads against 365) and chunks of 32
// tokens gained nothing (394). Rows of 128 x 128 spill 8 to 13 registers, with DOT 38 to 43.
// 64 x 64 has the registers and the LDS of three workgroups on a CU (with DOT the LDS of two, but for float16).
template <typename T, int KD, int NC, bool DOT, bool VEC, bool F32>
__global__ void __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(KD * NC == 64 ? 3 : 2, KD * NC == 64 ? 3 : 2))) la_walk(const WalkArgs) {
    constexpr int C = Cfg<T>::C, PI = Cfg<T>::in, W = 64 * NC;
    constexpr int LDX = KD, LDV = W, LDM = kScoreRow;
    typedef Stage<T, C, KD, kThreads, VEC> SX;
    typedef Stage<T, C, W, kThreads, VEC> SV;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    u16 *X = reinterpret_cast<u16 *>(smem), *Y = X + PI * kTile<C, LDX>, *V = Y + PI * kTile<C, LDX>;
    u16 *M = V + PI * kTile<C, LDV>, *Z = M + kPlanes * kTile<C, LDM>;
    Decays<C> *dec = reinterpret_cast<Decays<C> *>(Z + (DOT ? PI * kTile<C, LDV> : 0));
    float *part = reinterpret_cast<float *>(dec + 2);

    int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid / 64);
    auto fresh = [&] {
        tid = afresh_lane(tid);
        lane = tid & 63;
    };
    auto args = [] { return own_args<WalkArgs>(); };
    const Place p = place_of(args(), 1);
    const int col = wave * 16 * NC;

    f32x4 S[KD / 16][NC];
    {
        const WalkArgs a = args();
        const int64_t bh = int64_t(p.b) * a.heads + p.h;
        load_state<KD, NC>(S, Mat{a.s0.p ? a.s0.p + (bh * a.segs + p.seg) * a.s0_step : nullptr, a.s0.row, a.s0.col}, a.kdim, a.cdim, col, lane);
    }
    zero_masked_scores<C>(M, false, tid, kThreads);
    bool special = false;   // something in X or Y was not finite
    // One after the other: arguments that are read together are held together.
    auto tensor = [&](auto of) { const WalkArgs a = args(); return of(a); };
    const Rows<T> rx = tensor([&](const WalkArgs &a) { return rows_of<T>(a.x, p.b, p.h, a.kdim); });
    const Rows<T> ry = tensor([&](const WalkArgs &a) { return rows_of<T>(a.y, p.b, p.h, a.kdim); });
    const Rows<T> rv = tensor([&](const WalkArgs &a) { return rows_of<T>(a.v, p.b, p.h, a.cdim); });
    const Rows<T> rz = DOT ? tensor([&](const WalkArgs &a) { return rows_of<T>(a.z, p.b, p.h, a.cdim); }) : rv;
    const Gates gates = tensor([&](const WalkArgs &a) { return gates_of(a, p); });
    const float scale = afresh(args().scale);
    char *const out = tensor([&](const WalkArgs &a) {
        return afresh(static_cast<char *>(a.out) + (p.b * a.out_batch + p.h * a.out_head) * int64_t(F32 ? 4 : sizeof(T)));
    });
    const uint32_t out_stride = uint32_t(afresh(int(args().out_seq)));
    float *const e_out = DOT ? tensor([&](const WalkArgs &a) { return afresh(a.e + (int64_t(p.b) * a.heads + p.h) * a.seqlen); }) : nullptr;

    SX sx, sy;
    SV sv, sz;
    auto load = [&](int t0) {
        const int rows = min(C, p.end - t0);
        sx.load(rx, t0, rows, tid);
        sy.load(ry, t0, rows, tid);
        sv.load(rv, t0, rows, tid);
        if constexpr (DOT) sz.load(rz, t0, rows, tid);
    };
    auto make = [&](int buf, uint32_t g) { make_decays<C>(dec[buf], decode_g(g, gates.type), scale, lane); };
    auto keep = [&](const WalkArgs &a, int64_t block) {
        const int64_t bh = int64_t(p.b) * a.heads + p.h;
        store_state<KD, NC>(S, Mat{a.ck + (bh * a.blocks + block) * a.kdim * a.cdim, a.cdim, 1}, a.kdim, a.cdim, col, lane);
    };
    const int dwave = kWaves - 1;
    uint32_t gnext = 0;
    load(p.beg);
    if (wave == dwave) {
        make(0, gates.template load<C>(p.beg, p.end, lane));
        if (p.beg + C < p.end) gnext = gates.template load<C>(p.beg + C, p.end, lane);
    }
    int buf = 0;
    for (int t0 = p.beg; t0 < p.end; t0 += C, buf ^= 1) {
        const int rows = min(C, p.end - t0);
        if constexpr (DOT) {
            if (t0 > 0 && t0 % kBlock == 0) {
                const WalkArgs a = args();
                if (a.ck) keep(a, t0 / kBlock - 1);
            }
        }
        __syncthreads();
        fresh();
        sx.store(X, tid);
        sy.store(Y, tid);
        sv.store(V, tid);
        if constexpr (DOT) sz.store(Z, tid);
        const bool more = t0 + C < p.end;
        const int next = min(C, p.end - t0 - C);
        // The next chunk's loads go out between the steps, a tensor at a time (float32: at once, its walk is bound elsewhere).
        constexpr bool kSpread = sizeof(T) == 2;
        if (!kSpread && more) load(t0 + C);
        __syncthreads();
        fresh();
        const Decays<C> &d = dec[buf];
        // The score tiles, static for each wave; the last one, which also makes the next chunk's decays, has the fewest.
        auto tiles = [&](auto L) { special |= scores<T, C, KD, decltype(L)>(d, X, Y, M, scale, lane); };
        if constexpr (C == 64) {
            switch (wave) {
                case 0: tiles(Tiles<3, 0, 3, 1, 3, 2>{}); break;
                case 1: tiles(Tiles<2, 0, 2, 1, 2, 2>{}); break;
                case 2: tiles(Tiles<1, 0, 1, 1, 3, 3>{}); break;
                default: tiles(Tiles<0, 0>{});
            }
        } else {
            switch (wave) {
                case 0: tiles(Tiles<1, 0>{}); break;
                case 1: tiles(Tiles<1, 1>{}); break;
                case 2: tiles(Tiles<0, 0>{});
            }
        }
        if (kSpread && more) sx.load(rx, t0 + C, next, tid);
        f32x4 O[C / 16][NC];
        fresh();
        inter<T, C, KD, NC>(O, S, X, d.in, lane);
        if constexpr (DOT) dot_rows<T, C, NC, LDV>(O, Z, col, part + wave * C, lane);
        if (kSpread && more) sy.load(ry, t0 + C, next, tid);
        if (wave == dwave && more) {
            make(buf ^ 1, gnext);
            if (t0 + 2 * C < p.end) gnext = gates.template load<C>(t0 + 2 * C, p.end, lane);
        }
        __syncthreads();
        fresh();
        if constexpr (DOT) {
            if (tid < rows) {
                float e = 0.f;
#pragma unroll
                for (int w = 0; w < kWaves; ++w) e += part[w * C + tid];
                e_out[t0 + tid] = e;
            }
        }
        if (kSpread && more) {
            sv.load(rv, t0 + C, next, tid);
            if constexpr (DOT) sz.load(rz, t0 + C, next, tid);
        }
        bf16x8 v[C / 32][NC][PI];
        load_v<T, C, NC, LDV>(v, V, col, lane);
        intra<T, C, NC, LDV, false>(O, v, M, V, col, lane);
        update<T, C, KD, NC>(S, v, Y, d.out, d.all, lane);
        fresh();
        store_out<T, C, NC, LDV, VEC, F32>(O, out, out_stride, t0, rows, rv.d, V, col, lane);
    }
    {
        const WalkArgs a = args();
        if (a.s1.p && p.seg == a.segs - 1)
            store_state<KD, NC>(S, Mat{a.s1.p + (int64_t(p.b) * a.heads + p.h) * a.kdim * a.cdim, a.s1.row, a.s1.col}, a.kdim, a.cdim, col, lane);
        if constexpr (DOT) {
            // The state after the last token, for the product with the last state's gradient.
            if (a.ck && a.ck_last && p.seg == a.segs - 1) keep(a, a.blocks - 1);
        }
    }

    // A state that is not finite stays so: what made it so is seen at the end.
    if (__syncthreads_or(special || !finite_state<KD, NC>(S))) infinite_rows<T, KD, NC, DOT, VEC, F32>(smem);
}

// What each segment but the last one (REV: the first one) of a row adds to the state: sum of y_t (decay to the
// segment's end) v_t^T into st[bh][seg], and the segment's own decay into decay[bh][seg]. About 2 us per chunk and CU at
// dk 128 (7 of 8 segments of 64 pairs, dv 128, L 4,096: 52 us).
template <typename T, int KD, bool REV, bool VEC>
__global__ void __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(sizeof(T) == 2 ? 3 : 2, sizeof(T) == 2 ? 3 : 2))) la_segments(const WalkArgs) {
    constexpr int C = Cfg<T>::C, PI = Cfg<T>::in, W = 64;
    constexpr int LDX = KD, LDV = W;
    typedef Stage<T, C, KD, kThreads, VEC> SX;
    typedef Stage<T, C, W, kThreads, VEC> SV;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    u16 *Y = reinterpret_cast<u16 *>(smem), *V = Y + PI * kTile<C, LDX>;
    Decays<C> *dec = reinterpret_cast<Decays<C> *>(V + PI * kTile<C, LDV>);
    int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid / 64);
    auto args = [] { return own_args<WalkArgs>(); };
    const Place p = place_of(args(), args().slices);
    if (p.seg == (REV ? 0 : args().segs - 1)) return;
    const int chunks = (p.end - p.beg + C - 1) / C;
    const int col0 = p.slice * W, col = wave * 16;
    auto tensor = [&](auto of) { const WalkArgs a = args(); return of(a); };
    const Rows<T> ry = tensor([&](const WalkArgs &a) { return rows_of<T>(a.y, p.b, p.h, a.kdim); });
    const Rows<T> rv = tensor([&](const WalkArgs &a) { return rows_of<T>(a.v, p.b, p.h, a.cdim, col0); });
    const Gates gates = tensor([&](const WalkArgs &a) { return gates_of(a, p); });
    const float scale = afresh(args().scale);
    f32x4 S[KD / 16][1];
    load_state<KD, 1>(S, Mat{nullptr, 0, 0}, 0, 0, 0, lane);
    SX sy;
    SV sv;
    auto start = [&](int n) { return p.beg + (REV ? chunks - 1 - n : n) * C; };
    auto load = [&](int n) {
        const int t0 = start(n), rows = min(C, p.end - t0);
        sy.load(ry, t0, rows, tid);
        sv.load(rv, t0, rows, tid);
    };
    auto decay = [&](int n) { return gates.template load<C>(start(n), p.end, lane); };
    // The next chunk's decays are made by one wave while the others work on this one's state.
    double total = 0.0;
    bool cut = false;   // a token's own decay is 0
    auto decays = [&](int buf, uint32_t w) {
        const float g = decode_g(w, gates.type);
        total += make_decays<C>(dec[buf], g, scale, lane);
        cut |= exp_f32(g) == 0.f;
    };
    uint32_t gnext = 0;
    load(0);
    if (wave == 0) {
        decays(0, decay(0));
        if (chunks > 1) gnext = decay(1);
    }
    int buf = 0;
    for (int n = 0; n < chunks; ++n, buf ^= 1) {
        __syncthreads();
        tid = afresh_lane(tid);
        lane = tid & 63;
        sy.store(Y, tid);
        sv.store(V, tid);
        if (n + 1 < chunks) load(n + 1);
        __syncthreads();
        const Decays<C> &d = dec[buf];
        bf16x8 v[C / 32][1][PI];
        load_v<T, C, 1, LDV>(v, V, col, lane);
        update<T, C, KD, 1>(S, v, Y, REV ? d.in : d.out, d.all, lane);
        if (wave == 0 && n + 1 < chunks) {
            decays(buf ^ 1, gnext);
            if (n + 2 < chunks) gnext = decay(n + 2);
        }
    }
    if constexpr (!REV) {
        // What an infinity reached, by the recurrence, as behind the walk.
        if (__syncthreads_or(!finite_state<KD, 1>(S))) {
            auto again = [&](int n) {
                __syncthreads();
                load(n);
                sy.store(Y, tid);
                sv.store(V, tid);
                if (wave == 0) make_decays<C>(dec[0], decode_g(decay(n), gates.type), scale, lane);
                __syncthreads();
            };
            Kinds seen = {false, false};
#pragma unroll 1
            for (int n = 0; n < chunks; ++n) {
                again(n);
                seen.tile<C, KD>(Y, lane);
                seen.tile<C, W>(V, lane);
                seen.add(dec[0].hi[C - 1]);
            }
            const bool inf = __syncthreads_or(seen.inf), nan = __syncthreads_or(seen.nan);
            if (inf || !nan) {
                f32x4 R[KD / 16][1];
                load_state<KD, 1>(R, Mat{nullptr, 0, 0}, 0, 0, 0, lane);
#pragma unroll 1
                for (int n = 0; n < chunks; ++n) {
                    again(n);
                    recur<T, C, KD, 1, LDV, false>(R, nullptr, Y, V, dec[0], min(C, p.end - start(n)), args().kdim, col, lane,
                                                   [](int, int, float) {});
                }
#pragma unroll
                for (int k = 0; k < KD / 16; ++k)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (!finite(S[k][0][r])) S[k][0][r] = R[k][0][r];
            }
        }
    }
    const WalkArgs a = args();
    const int64_t at = (int64_t(p.b) * a.heads + p.h) * a.segs + p.seg;
    store_state<KD, 1>(S, Mat{a.st + at * a.kdim * a.cdim, a.cdim, 1}, a.kdim, a.cdim, col0 + col, lane);
    // A decay that no token's own makes 0 is not 0: an infinite state stays infinite in any number of segments. (Nothing finite
    // changes by 2^-126 of a state.)
    cut = __any(cut);
    if (p.slice == 0 && tid == 0) {
        const float d = exp_f32(float(total));
        a.seg_decay[at] = !cut && d < 1.17549435e-38f ? 1.17549435e-38f : d;
    }
}

// Backward walk from the end: dv, dk, the scores' part of the decays' gradient (a), the state's part (f), and at
// every kBlock-th token the product of the state there with its gradient (y). Waves 0 to 3 hold the gradient R of the
// state for dv (rows dk, columns dv), waves 4 to 7 its transpose for dk: two walks over the same tiles, each in code of
// its own with the same barriers.
//
// Every q, k, v and dout row is read once for both. One workgroup of 8 waves per CU (102 KB of LDS and 224 registers at dk 128,
// dv 64; 118 KB, 256 registers and 6 to 12 spilled at 128 x 128), 7.2 us per 64 tokens with dv 64. A wave issues 130 matrix and some 1,135
// other vector instructions per chunk, two waves per SIMD: the vector units are busy 55 % of the time, the matrix cores 25 %, the LDS
// 38 % (a third of it conflicts), and a wave waits a third of its own. 8 x 2,048 tokens, 24 heads, 229 us; 4 x 4,096 tokens, 16 heads
// with dv 128, 181 us.
//
// FOR_K: the walk of dk, X = v, Y = do, V = q; else that of dv, X = k, Y = q, V = do. KX: X's padded row length, KV: V's.
template <typename T, int KD, int VD, bool VEC, bool F32, bool FOR_K>
__device__ __forceinline__ void bwd_walk(char *smem, int tid, int wave, int lane) {
    auto args = [] { return own_args<BwdArgs>(); };
    constexpr bool kTight = KD + VD > 128;   // registers
    auto fresh = [&] {
        if constexpr (kTight) {
            tid = afresh_lane(tid);
            lane = tid & 63;
        }
    };
    constexpr int C = Cfg<T>::C, PI = Cfg<T>::in, NT2 = 2 * kThreads;
    constexpr int LDK = KD, LDV = VD, LDM = kScoreRow, CT = C / 16;
    constexpr int KX = FOR_K ? VD : KD, NC = (FOR_K ? KD : VD) / 64, LDC = FOR_K ? LDK : LDV;
    typedef Stage<T, C, KD, NT2, VEC> SK;
    typedef Stage<T, C, VD, NT2, VEC> SV;
    u16 *Q = reinterpret_cast<u16 *>(smem), *K = Q + PI * kTile<C, LDK>, *V = K + PI * kTile<C, LDK>, *G = V + PI * kTile<C, LDV>;
    u16 *M1 = G + PI * kTile<C, LDV>, *M2 = M1 + kPlanes * kTile<C, LDM>;
    Decays<C> *dec = reinterpret_cast<Decays<C> *>(M2 + kPlanes * kTile<C, LDM>);
    float *rowp = reinterpret_cast<float *>(dec + 2), *colp = rowp + CT * C, *part = colp + CT * C;

    const Place p = place_of(args(), 1);
    const int chunks = (p.end - p.beg + C - 1) / C, col = (wave % kWaves) * 16 * NC;
    auto pair = [&](const BwdArgs &a) { return int64_t(p.b) * a.heads + p.h; };

    // R (or its transpose) at the segment's end.
    f32x4 S[KX / 16][NC];
    {
        const BwdArgs a = args();
        load_state<KX, NC>(S, Mat{a.r0 ? const_cast<float *>(a.r0) + (pair(a) * a.segs + p.seg) * a.dk * a.dv : nullptr, FOR_K ? 1 : a.dv,
                                  FOR_K ? a.dv : 1}, FOR_K ? a.dv : a.dk, FOR_K ? a.dk : a.dv, col, lane);
    }
    // <R, state> at a kept boundary, each wave's share.
    auto boundary = [&](const BwdArgs &a, int m) {
        const int64_t at = pair(a) * a.blocks + m;
        const Mat ck{const_cast<float *>(a.ck) + at * a.dk * a.dv, a.dk, 1};   // rows dv, columns dk
        float sum = dot_state<KX, NC>(S, ck, a.dv, a.dk, col, lane);
        sum = wave_sum(sum);
        if (lane == 0) a.y[at * kWaves + wave - kWaves] = sum;
    };
    if constexpr (FOR_K) {
        const BwdArgs a = args();
        if (a.ck && a.has_last && p.seg == a.segs - 1) boundary(a, int(a.blocks) - 1);
    }

    // One after the other: arguments that are read together are held together.
    auto tensor = [&](auto of) { const BwdArgs a = args(); return of(a); };
    const Rows<T> rq = tensor([&](const BwdArgs &a) { return rows_of<T>(a.q, p.b, p.h, a.dk); });
    const Rows<T> rk = tensor([&](const BwdArgs &a) { return rows_of<T>(a.k, p.b, p.h, a.dk); });
    const Rows<T> rv = tensor([&](const BwdArgs &a) { return rows_of<T>(a.v, p.b, p.h, a.dv); });
    const Rows<T> rd = tensor([&](const BwdArgs &a) { return rows_of<T>(a.dout, p.b, p.h, a.dv); });
    const float scale = afresh(args().scale);
    const bool want_g = args().a != nullptr;
    char *const out = tensor([&](const BwdArgs &a) {
        return afresh(static_cast<char *>(FOR_K ? a.dk_out : a.dv_out) +
                      (p.b * a.seqlen * a.heads + p.h) * (FOR_K ? a.dk : a.dv) * int64_t(FOR_K && F32 ? 4 : sizeof(T)));
    });
    const uint32_t out_stride = tensor([&](const BwdArgs &a) { return uint32_t(afresh(int(a.heads) * (FOR_K ? a.dk : a.dv))); });
    zero_masked_scores<C>(M1, true, tid, NT2);
    zero_masked_scores<C>(M2, true, tid, NT2);
    SK sq, sk;
    SV sv, sd;
    auto start = [&](int n) { return p.beg + (chunks - 1 - n) * C; };
    // (dk's walk alone makes the decays.)
    const Gates gates = FOR_K ? tensor([&](const BwdArgs &a) { return gates_of(a, p); }) : Gates{nullptr, 0, MM_FLOAT32};
    auto make = [&](int buf, uint32_t g) { make_decays<C>(dec[buf], decode_g(g, gates.type), scale, lane); };
    const bool dwave = FOR_K && wave == 2 * kWaves - 1;
    uint32_t gnext = 0;
    {
        const int t0 = start(0), rows = min(C, p.end - t0);
        sq.load(rq, t0, rows, tid);
        sk.load(rk, t0, rows, tid);
        sv.load(rv, t0, rows, tid);
        sd.load(rd, t0, rows, tid);
    }
    if (dwave) {
        make(0, gates.template load<C>(start(0), p.end, lane));
        if (chunks > 1) gnext = gates.template load<C>(start(1), p.end, lane);
    }
    int buf = 0;
    for (int n = 0; n < chunks; ++n, buf ^= 1) {
        const int t0 = start(n), rows = min(C, p.end - t0);
        __syncthreads();
        fresh();
        sq.store(Q, tid);
        sk.store(K, tid);
        sv.store(V, tid);
        sd.store(G, tid);
        const bool more = n + 1 < chunks;
        const int tn = t0 - C;   // the next chunk is a whole one
        __syncthreads();
        fresh();
        const Decays<C> &d = dec[buf];
        auto tiles = [&](auto L) { scores_bwd<T, C, KD, VD, decltype(L)>(d, Q, K, V, G, M1, M2, scale, want_g, rowp, colp, lane); };
        if constexpr (C == 64) {
            switch (wave) {
                case 0: tiles(Tiles<0, 0, 0, 1>{}); break;
                case 1: tiles(Tiles<0, 2, 0, 3>{}); break;
                case 2: tiles(Tiles<1, 1, 1, 2>{}); break;
                case 3: tiles(Tiles<3, 3>{}); break;
                case 4: tiles(Tiles<1, 3>{}); break;
                case 5: tiles(Tiles<2, 2>{}); break;
                case 6: tiles(Tiles<2, 3>{});
            }
        } else {
            switch (wave) {
                case 0: tiles(Tiles<0, 0>{}); break;
                case 1: tiles(Tiles<0, 1>{}); break;
                case kWaves: tiles(Tiles<1, 1>{});
            }
        }
        if (more) sq.load(rq, tn, C, tid);
        f32x4 O[CT][NC];
        fresh();
        inter<T, C, KX, NC>(O, S, FOR_K ? V : K, d.out, lane);
        if constexpr (FOR_K) {
            if (want_g) dot_rows<T, C, NC, LDK>(O, K, col, part + (wave - kWaves) * C, lane);
        }
        if (more) sk.load(rk, tn, C, tid);
        if (dwave && more) {
            make(buf ^ 1, gnext);
            if (n + 2 < chunks) gnext = gates.template load<C>(start(n + 2), p.end, lane);
        }
        __syncthreads();
        fresh();
        if constexpr (!FOR_K) {
            if (want_g && tid < rows) {
                const int t = tid / 16;
                float sum = 0.f, f = 0.f;
                for (int o = 0; o <= t; ++o) sum += rowp[o * C + tid];
                for (int m = t; m < CT; ++m) sum -= colp[m * C + tid];
#pragma unroll
                for (int w = 0; w < kWaves; ++w) f += part[w * C + tid];
                const BwdArgs a = args();
                const int64_t at = pair(a) * a.seqlen + t0 + tid;
                a.a[at] = sum;
                a.f[at] = f;
            }
        }
        if (more) {
            sv.load(rv, tn, C, tid);
            sd.load(rd, tn, C, tid);
        }
        const u16 *VT = FOR_K ? Q : G;
        bf16x8 v[C / 32][NC][PI];
        load_v<T, C, NC, LDC>(v, VT, col, lane);
        intra<T, C, NC, LDC, true>(O, v, FOR_K ? M2 : M1, VT, col, lane);
        update<T, C, KX, NC>(S, v, FOR_K ? G : Q, d.in, d.all, lane);
        fresh();
        store_out<T, C, NC, LDC, VEC, FOR_K && F32>(O, out, out_stride, t0, rows, FOR_K ? rk.d : rv.d, FOR_K ? K : V, col, lane);
        if constexpr (FOR_K) {
            if (want_g && t0 > 0 && t0 % kBlock == 0) boundary(args(), t0 / kBlock - 1);
        }
    }
    if constexpr (!FOR_K) {
        const BwdArgs a = args();
        if (a.dr && p.seg == 0) store_state<KX, NC>(S, Mat{a.dr + pair(a) * a.dk * a.dv, a.dv, 1}, a.dk, a.dv, col, lane);
    }
}

template <typename T, int KD, int VD, bool VEC, bool F32>
__global__ void __launch_bounds__(2 * kThreads) __attribute__((amdgpu_waves_per_eu(2, 2))) la_bwd(const BwdArgs) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / 64), lane = tid & 63;
    if (wave < kWaves) bwd_walk<T, KD, VD, VEC, F32, false>(smem, tid, wave, lane);
    else bwd_walk<T, KD, VD, VEC, F32, true>(smem, tid, wave, lane);
}

// Launches with `bytes` of dynamic LDS, which a kernel is allowed once per device (`done`: a bit per device).
template <typename K, typename A>
static int launch_kernel(K kernel, int bytes, std::atomic<uint64_t> &done, int64_t grid, int threads, const A &a, hipStream_t s,
                         const char *what) {
    int dev = 0;
    if (const hipError_t e = hipGetDevice(&dev)) return set_error(int(e), "linear attention: hipGetDevice failed");
    const uint64_t bit = uint64_t(1) << (dev & 63);
    if (!(done.load(std::memory_order_relaxed) & bit)) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (e != hipSuccess) return set_error(int(e), "linear attention: hipFuncSetAttribute failed");
        done.fetch_or(bit, std::memory_order_relaxed);
    }
    hipLaunchKernelGGL(kernel, dim3(unsigned(grid)), dim3(unsigned(threads)), bytes, s, a);
    return launch_status(what);
}

template <typename T, int KD, int NC, bool DOT, bool VEC, bool F32>
static int launch_walk_t(const WalkArgs &a, hipStream_t s) {
    constexpr int C = Cfg<T>::C, PI = Cfg<T>::in;
    constexpr int bytes = 2 * (2 * PI * kTile<C, KD> + (DOT ? 2 : 1) * PI * kTile<C, 64 * NC> + kPlanes * kTile<C, kScoreRow>) +
                          2 * int(sizeof(Decays<C>)) + (DOT ? 4 * kWaves * C : 0);
    static_assert(bytes <= 160 * 1024, "LDS");
    const auto kernel = la_walk<T, KD, NC, DOT, VEC, F32>;
    static std::atomic<uint64_t> done{0};
    return launch_kernel(kernel, bytes, done, a.batch * a.heads * a.segs, kThreads, a, s, "la_walk");
}
template <typename T, int KD, int NC, bool DOT>
static int launch_walk_k(const WalkArgs &a, hipStream_t s) {
    const bool vec = a.x.vec && a.y.vec && a.v.vec && (!DOT || a.z.vec) && a.out_vec;
    if constexpr (sizeof(T) == 4) {
        return vec ? launch_walk_t<T, KD, NC, DOT, true, true>(a, s) : launch_walk_t<T, KD, NC, DOT, false, true>(a, s);
    } else {
        if (a.out_f32) return vec ? launch_walk_t<T, KD, NC, DOT, true, true>(a, s) : launch_walk_t<T, KD, NC, DOT, false, true>(a, s);
        return vec ? launch_walk_t<T, KD, NC, DOT, true, false>(a, s) : launch_walk_t<T, KD, NC, DOT, false, false>(a, s);
    }
}

template <typename T, int KD, bool REV, bool VEC>
static int launch_segments_t(const WalkArgs &a0, hipStream_t s) {
    constexpr int C = Cfg<T>::C, PI = Cfg<T>::in;
    constexpr int bytes = 2 * (PI * kTile<C, KD> + PI * kTile<C, 64>) + 2 * int(sizeof(Decays<C>));
    static_assert(bytes <= 160 * 1024, "LDS");
    const auto kernel = la_segments<T, KD, REV, VEC>;
    static std::atomic<uint64_t> done{0};
    WalkArgs a = a0;
    a.slices = (a.cdim + 63) / 64;
    return launch_kernel(kernel, bytes, done, a.batch * a.heads * a.segs * a.slices, kThreads, a, s, "la_segments");
}
template <typename T, int KD>
static int launch_segments_k(const WalkArgs &a, bool rev, hipStream_t s) {
    if (a.y.vec && a.v.vec) return rev ? launch_segments_t<T, KD, true, true>(a, s) : launch_segments_t<T, KD, false, true>(a, s);
    return rev ? launch_segments_t<T, KD, true, false>(a, s) : launch_segments_t<T, KD, false, false>(a, s);
}

template <typename T, int KD, int VD, bool VEC, bool F32>
static int launch_bwd_t(const BwdArgs &a, hipStream_t s) {
    constexpr int C = Cfg<T>::C, PI = Cfg<T>::in;
    constexpr int bytes = 2 * (2 * PI * kTile<C, KD> + 2 * PI * kTile<C, VD> + 2 * kPlanes * kTile<C, kScoreRow>) +
                          2 * int(sizeof(Decays<C>)) + 4 * (2 * (C / 16) * C + kWaves * C);
    static_assert(bytes <= 160 * 1024, "LDS");
    const auto kernel = la_bwd<T, KD, VD, VEC, F32>;
    static std::atomic<uint64_t> done{0};
    return launch_kernel(kernel, bytes, done, a.batch * a.heads * a.segs, 2 * kThreads, a, s, "la_bwd");
}
template <typename T, int KD, int VD, bool F32>
static int launch_bwd_f(const BwdArgs &a, hipStream_t s) {
    const bool vec = a.q.vec && a.k.vec && a.v.vec && a.dout.vec && a.out_vec;
    return vec ? launch_bwd_t<T, KD, VD, true, F32>(a, s) : launch_bwd_t<T, KD, VD, false, F32>(a, s);
}
template <typename T, int KD, int VD>
static int launch_bwd_k(const BwdArgs &a, hipStream_t s) {
    if constexpr (sizeof(T) == 4) return launch_bwd_f<T, KD, VD, true>(a, s);
    else return a.dk_f32 ? launch_bwd_f<T, KD, VD, true>(a, s) : launch_bwd_f<T, KD, VD, false>(a, s);
}

template <typename T>
int launch_walk(const WalkArgs &a, bool dot, hipStream_t s) {
    const bool wide = a.cdim > 64;
    if (dot) {
        if (a.kdim <= 64) return wide ? launch_walk_k<T, 64, 2, true>(a, s) : launch_walk_k<T, 64, 1, true>(a, s);
        return wide ? launch_walk_k<T, 128, 2, true>(a, s) : launch_walk_k<T, 128, 1, true>(a, s);
    }
    if (a.kdim <= 64) return wide ? launch_walk_k<T, 64, 2, false>(a, s) : launch_walk_k<T, 64, 1, false>(a, s);
    return wide ? launch_walk_k<T, 128, 2, false>(a, s) : launch_walk_k<T, 128, 1, false>(a, s);
}

template <typename T>
int launch_segments(const WalkArgs &a, bool rev, hipStream_t s) {
    return a.kdim <= 64 ? launch_segments_k<T, 64>(a, rev, s) : launch_segments_k<T, 128>(a, rev, s);
}

template <typename T>
int launch_bwd(const BwdArgs &a, hipStream_t s) {
    if (a.dk <= 64) return a.dv <= 64 ? launch_bwd_k<T, 64, 64>(a, s) : launch_bwd_k<T, 64, 128>(a, s);
    return a.dv <= 64 ? launch_bwd_k<T, 128, 64>(a, s) : launch_bwd_k<T, 128, 128>(a, s);
}

template int launch_walk<MM_LINATTN_TYPE>(const WalkArgs &, bool, hipStream_t);
template int launch_segments<MM_LINATTN_TYPE>(const WalkArgs &, bool, hipStream_t);
template int launch_bwd<MM_LINATTN_TYPE>(const BwdArgs &, hipStream_t);

#ifdef MM_LINATTN_COMMON
// ---- joins and sums ------------------------------------------------------------------------------

// The segments' shares in st[bh][seg] become the states the segments start from (rev: end with).
__global__ void __launch_bounds__(256) la_join(float *st, const float *decay, const float *edge, int segs, int64_t size, bool rev) {
    const int64_t bh = blockIdx.x, x = int64_t(blockIdx.y) * 256 + threadIdx.x;
    if (x >= size) return;
    float cur = edge ? edge[bh * size + x] : 0.f;
    float *p = st + bh * segs * size + x;
    for (int n = 0; n < segs; ++n) {
        const int seg = rev ? segs - 1 - n : n;
        const float add = n + 1 < segs ? p[seg * size] : 0.f;
        p[seg * size] = cur;
        if (n + 1 < segs) cur = __builtin_fmaf(decay[bh * segs + seg], cur, add);
    }
}

// out[row][x] = sum over the group's heads of part[row][head][x], in order; W consecutive x per thread. HBM-bound: 201 MB of
// 24 heads' gradients in 31 us (6.5 TB/s, part of them from the last-level cache), 59 with one element per thread.
template <typename T, int W>
__global__ void __launch_bounds__(256) la_head_sum(const float *part, T *out, int64_t n, int heads, int share, int d) {
    for (int64_t id = (int64_t(blockIdx.x) * 256 + threadIdx.x) * W; id < n; id += int64_t(gridDim.x) * 256 * W) {
        const int64_t x = id % d, rg = id / d, groups = heads / share, row = rg / groups, grp = rg % groups;
        const float *p = part + (row * heads + grp * share) * d + x;
        float s[W] = {};
#pragma unroll 8
        for (int r = 0; r < share; ++r) {
            if constexpr (W == 4) {
                const f32x4 y = *reinterpret_cast<const f32x4 *>(p + int64_t(r) * d);
#pragma unroll
                for (int e = 0; e < 4; ++e) s[e] += y[e];
            } else {
                s[0] += p[int64_t(r) * d];
            }
        }
#pragma unroll
        for (int e = 0; e < W; ++e) out[id + e] = from_f32<T>(s[e]);
    }
}

__device__ __forceinline__ void store_g(void *p, mm_dtype t, int64_t i, float x) {
    switch (t) {
        case MM_FLOAT32: reinterpret_cast<float *>(p)[i] = x; break;
        case MM_FLOAT16: reinterpret_cast<f16_t *>(p)[i] = from_f32<f16_t>(x); break;
        default: reinterpret_cast<bf16_t *>(p)[i] = from_f32<bf16_t>(x);
    }
}

// The gradient of a log decay is the sum of W_ij = scale exp(c_i - c_j) (q_i . k_j) (do_i . v_j) over the pairs that it
// lies between, j < t <= i. Cut at t's chunk, with S the state before and R the state's gradient after the chunk: pairs
// inside it (a holds each token's row sum less its column sum, the diagonal left out; summed from t on), pairs from before into
// it (e_i), pairs from it to behind (f_j), and pairs around it, Z = exp(c_end) <R, S>, which is <R, S'> less the chunk's f; <R, S'>
// is taken from the states themselves every kBlock tokens. Two of these are differences: a pair that lies wholly behind t is in
// a's sum once with each sign, and Z is what is left of <R, S'>. So a result's error is a fraction (2^-24 and the sums' depth) of the
// terms of its chunk's tokens behind it and of its block's. A forgotten state (-inf) ends both: no pair crosses it, so a's sum stops
// there and Z is 0, and a document's results have nothing of another one's rounding. One workgroup per block and
// (batch row, head); C: the chunk's tokens.
__global__ void __launch_bounds__(kBlock) la_decay_grad(const float *a, const float *e, const float *f, const float *y, int64_t seqlen,
                                                        int64_t blocks, int heads, int C, bool has_last, const void *g, int64_t g_batch,
                                                        int64_t g_seq, int64_t g_head, float *tmp, void *out, mm_dtype gtype) {
    __shared__ float sa[kBlock], sf[kBlock], se[kBlock], zc[kBlock / 16];
    __shared__ int chunk_forgets[kBlock / 32];
    const int64_t blk = blockIdx.y, bh = blockIdx.x, t = blk * kBlock + threadIdx.x;
    const int tid = threadIdx.x, chunks = kBlock / C;
    const bool live = t < seqlen;
    const float ae = live ? e[bh * seqlen + t] : 0.f;
    sa[tid] = (live ? a[bh * seqlen + t] : 0.f) + ae;
    sf[tid] = live ? f[bh * seqlen + t] : 0.f;
    se[tid] = ae;
    const bool forgets = live && decode_g(load_g_raw(g, gtype, bh / heads * g_batch + t * g_seq + bh % heads * g_head), gtype) == -128.f;
    const uint64_t all_forgets = __ballot(forgets);   // of 64 tokens: one chunk or two
    if (tid % C == 0) chunk_forgets[tid / C] = (all_forgets >> tid % 64 & (C == 64 ? ~uint64_t(0) : (uint64_t(1) << C) - 1)) != 0;
    __syncthreads();
    if (tid < chunks) {   // the chunks' totals
        float E = 0.f, F = 0.f;
        for (int n = 0; n < C; ++n) {
            E += se[tid * C + n];
            F += sf[tid * C + n];
        }
        zc[tid] = E;
        zc[chunks + tid] = F;
    }
    __syncthreads();
    if (tid == 0) {
        float Y = 0.f;
        if (blk + 1 < blocks || has_last)
            for (int w = 0; w < 4; ++w) Y += y[(bh * blocks + blk) * 4 + w];
        for (int c = chunks - 1; c >= 0; --c) {
            const float Z = chunk_forgets[c] ? 0.f : Y - zc[chunks + c];
            Y = Z + zc[c];
            zc[c] = Z;
        }
    }
    __syncthreads();
    if (!live) return;
    const int c0 = tid / C * C;
    float s = zc[tid / C];
    for (int n = c0; n < tid; ++n) s += sf[n];
    const uint64_t behind = all_forgets >> tid % 64 >> 1;
    const int end = min(c0 + C, tid + 1 + (behind ? __builtin_ctzll(behind) : 64));
    for (int n = end - 1; n >= tid; --n) s += sa[n];
    if (forgets) s = 0.f;
    if (tmp) tmp[bh * seqlen + t] = s;
    else store_g(out, gtype, (bh / heads * seqlen + t) * heads + bh % heads, s);
}

// dlog_decay[h] = sum over batch rows and tokens, one workgroup per head.
__global__ void __launch_bounds__(256) la_decay_sum(const float *tmp, int64_t batch, int64_t heads, int64_t seqlen, void *out, mm_dtype gtype) {
    __shared__ float part[256];
    const int64_t h = blockIdx.x;
    float s = 0.f;
    for (int64_t b = 0; b < batch; ++b)
        for (int64_t t = threadIdx.x; t < seqlen; t += 256) s += tmp[(b * heads + h) * seqlen + t];
    part[threadIdx.x] = s;
    for (int n = 128; n > 0; n /= 2) {
        __syncthreads();
        if (int(threadIdx.x) < n) part[threadIdx.x] += part[threadIdx.x + n];
    }
    if (threadIdx.x == 0) store_g(out, gtype, h, part[0]);
}

__global__ void __launch_bounds__(256) la_copy(float *dst, const float *src, int64_t n) {
    for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < n; i += int64_t(gridDim.x) * 256) dst[i] = src ? src[i] : 0.f;
}
__global__ void __launch_bounds__(256) la_zero_g(void *dst, mm_dtype t, int64_t n) {
    for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < n; i += int64_t(gridDim.x) * 256) store_g(dst, t, i, 0.f);
}

// Blocks of 256 for n elements, each thread taking one at a time until none is left: a launch holds less than 2^32 threads.
static unsigned blocks_of(int64_t n) { return unsigned(std::min<int64_t>((n + 255) / 256, 1 << 23)); }

int launch_join(float *st, const float *decay, const float *edge, int segs, int64_t size, int64_t bh, bool rev, hipStream_t s) {
    hipLaunchKernelGGL(la_join, dim3(unsigned(bh), blocks_of(size)), dim3(256), 0, s, st, decay, edge, segs, size, rev);
    return launch_status("la_join");
}

int launch_head_sum(const float *part, void *out, mm_dtype t, int64_t rows, int heads, int share, int d, hipStream_t s) {
    const int64_t n = rows * (heads / share) * d;
    const bool vec = d % 4 == 0;
    const dim3 grid(blocks_of(vec ? n / 4 : n)), blk(256);
    auto go = [&](auto *to) {
        typedef std::remove_pointer_t<decltype(to)> O;
        if (vec) hipLaunchKernelGGL((la_head_sum<O, 4>), grid, blk, 0, s, part, to, n, heads, share, d);
        else hipLaunchKernelGGL((la_head_sum<O, 1>), grid, blk, 0, s, part, to, n, heads, share, d);
    };
    if (t == MM_FLOAT32) go(static_cast<float *>(out));
    else if (t == MM_FLOAT16) go(static_cast<f16_t *>(out));
    else go(static_cast<bf16_t *>(out));
    return launch_status("la_head_sum");
}

int launch_decay_grad(const BwdArgs &a, const float *e, int C, bool per_head, void *out, mm_dtype gtype, hipStream_t s) {
    // The sums over a head's tokens go through f's place, which a block reads before it writes.
    hipLaunchKernelGGL(la_decay_grad, dim3(unsigned(a.batch * a.heads), unsigned(a.blocks)), dim3(kBlock), 0, s, a.a, e, a.f, a.y, a.seqlen,
                       a.blocks, int(a.heads), C, a.has_last != 0, a.g, a.g_batch, a.g_seq, a.g_head, per_head ? a.f : nullptr, out, gtype);
    if (const int rc = launch_status("la_decay_grad")) return rc;
    if (!per_head) return MM_OK;
    hipLaunchKernelGGL(la_decay_sum, dim3(unsigned(a.heads)), dim3(256), 0, s, a.f, a.batch, a.heads, a.seqlen, out, gtype);
    return launch_status("la_decay_sum");
}

int launch_copy(float *dst, const float *src, int64_t n, hipStream_t s) {
    hipLaunchKernelGGL(la_copy, dim3(blocks_of(n)), dim3(256), 0, s, dst, src, n);
    return launch_status("la_copy");
}
int launch_zero_g(void *dst, mm_dtype t, int64_t n, hipStream_t s) {
    hipLaunchKernelGGL(la_zero_g, dim3(blocks_of(n)), dim3(256), 0, s, dst, t, n);
    return launch_status("la_zero_g");
}
#endif  // MM_LINATTN_COMMON

}  // namespace la
}  // namespace mm
