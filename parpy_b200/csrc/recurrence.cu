// Gated linear recurrence over sequences for sm_100a, its gradient, and its single-token step:
//
//   f_t = sigmoid(g_t),   h_t = f_t h_{t-1} + (1 - f_t) x_t        (channel by channel)
//
// A run of steps maps the state that enters it to the state that leaves it by h -> A h + B with A = prod f, and two
// runs in a row compose: (A2, B2) o (A1, B1) = (A1 A2, A2 B1 + B2). So a tile of 128 steps is cut into one run per
// warp, kept in registers: every warp forms its (A, B), the runs of a tile are folded through shared memory, those of
// the tiles that a cluster works on at the same time through distributed shared memory, and each warp then steps
// through its run again from the state it now knows. Every value is read and written once; the order of all sums is
// fixed. The gradient runs the same fold from the other end, for the quantity c_t = f_t r_t that step t hands to the
// step before it (r_t = dL/dh_t = dh_t + c_{t+1}):
//
//   c_t = f_t (dh_t + c_{t+1}),  dx_t = (1 - f_t) r_t,  dg_t = r_t (h_{t-1} - x_t) f_t (1 - f_t),  dh0 = c_1
//
// and rebuilds the states in 32 bits from the one that the forward kernel stored at the start of every tile (1/128 of
// their bytes) instead of reading back h, which has been rounded to the output type.
//
// An infinite or NaN state, input or gate reaches every later step of its channel (and every earlier one's gradient) as an
// infinity or NaN, and no other channel. Which of the two is not the stepwise definition's: a run's A that has underflowed to
// 0 makes NaN of an infinity.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <climits>

#include "../../include/parpy_b200.h"
#include "common.cuh"
#include "cluster.cuh"

namespace {

constexpr int kTile = PARPY_B200_SCAN_TILE;   // steps per tile, and per stored state
constexpr int kMaxRanks = 8;
constexpr int kStages = 3;                    // rounds of inputs in shared memory in the staged kernels

// ---- four bytes of a row: the channels of one lane ------------------------------------------------------
// kCap: the lowest gate value that is told apart, exact in its type (see gate()).
template <typename T>
struct Word;
template <>
struct Word<float> {
    static constexpr int CH = 1;
    static constexpr float kCap = -87.0f;
    __device__ static void unpack(unsigned w, float (&v)[1]) { v[0] = __uint_as_float(w); }
    __device__ static unsigned cap(unsigned w) {        // max(v, kCap), NaN for NaN
        float r;
        asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(__uint_as_float(w)), "f"(kCap));
        return __float_as_uint(r);
    }
    __device__ static unsigned pack(const float (&v)[1]) { return __float_as_uint(v[0]); }
};
template <>
struct Word<__nv_bfloat16> {
    static constexpr int CH = 2;
    static constexpr float kCap = -41.5f;
    __device__ static void unpack(unsigned w, float (&v)[2]) {
        v[0] = __uint_as_float(w << 16);
        v[1] = __uint_as_float(w & 0xffff0000u);
    }
    __device__ static unsigned cap(unsigned w) {
        const __nv_bfloat162 r = __hmax2_nan(*reinterpret_cast<const __nv_bfloat162 *>(&w), __float2bfloat162_rn(kCap));
        return *reinterpret_cast<const unsigned *>(&r);
    }
    __device__ static unsigned pack(const float (&v)[2]) {
        const __nv_bfloat162 p = __floats2bfloat162_rn(v[0], v[1]);
        return *reinterpret_cast<const unsigned *>(&p);
    }
};
template <>
struct Word<__half> {
    static constexpr int CH = 2;
    static constexpr float kCap = -41.5f;
    __device__ static void unpack(unsigned w, float (&v)[2]) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w));
        v[0] = f.x;
        v[1] = f.y;
    }
    __device__ static unsigned cap(unsigned w) {
        const __half2 r = __hmax2_nan(*reinterpret_cast<const __half2 *>(&w), __float2half2_rn(kCap));
        return *reinterpret_cast<const unsigned *>(&r);
    }
    __device__ static unsigned pack(const float (&v)[2]) {
        const __half2 p = __floats2half2_rn(v[0], v[1]);
        return *reinterpret_cast<const unsigned *>(&p);
    }
};

// A lane's channels within a block of 32 CH are neighbours, read as one word where rows allow 4-byte access (VEC) and one
// by one where they start at any element.
template <typename T, bool VEC>
__device__ __forceinline__ unsigned load_word(const T *p, int lane, int n) {
    if constexpr (VEC) {
        unsigned w = 0;
        if (lane * Word<T>::CH < n)
            asm volatile("ld.global.L1::no_allocate.u32 %0, [%1];" : "=r"(w) : "l"(p + lane * Word<T>::CH));
        return w;
    } else {
        const unsigned short *q = reinterpret_cast<const unsigned short *>(p) + 2 * lane;
        const unsigned lo = 2 * lane < n ? q[0] : 0, hi = 2 * lane + 1 < n ? q[1] : 0;
        return lo | (hi << 16);
    }
}
template <typename T, bool VEC>
__device__ __forceinline__ void store_word(T *p, int lane, int n, unsigned w) {
    if constexpr (VEC) {
        if (lane * Word<T>::CH < n) __stcs(reinterpret_cast<unsigned *>(p + lane * Word<T>::CH), w);
    } else {
        unsigned short *q = reinterpret_cast<unsigned short *>(p) + 2 * lane;
        if (2 * lane < n) q[0] = (unsigned short)w;
        if (2 * lane + 1 < n) q[1] = (unsigned short)(w >> 16);
    }
}

// ---- the CH channels of a lane as one value: a register, or a pair with one instruction for both -----------------
// Nothing is contracted behind the source's back, so that all layouts give the same bits.
template <int CH>
struct Lanes;
template <>
struct Lanes<1> {
    float v;
    __device__ static Lanes of(float a) { return {a}; }
    __device__ static Lanes of(const float (&a)[1]) { return {a[0]}; }
    __device__ void get(float (&a)[1]) const { a[0] = v; }
};
template <>
struct Lanes<2> {
    unsigned long long v;
    __device__ static Lanes of(float a, float b) {
        Lanes r;
        asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
        return r;
    }
    __device__ static Lanes of(float a) { return of(a, a); }
    __device__ static Lanes of(const float (&a)[2]) { return of(a[0], a[1]); }
    __device__ void get(float (&a)[2]) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(a[0]), "=f"(a[1]) : "l"(v)); }
};
__device__ __forceinline__ Lanes<1> operator+(Lanes<1> a, Lanes<1> b) { return {__fadd_rn(a.v, b.v)}; }
__device__ __forceinline__ Lanes<1> operator*(Lanes<1> a, Lanes<1> b) { return {__fmul_rn(a.v, b.v)}; }
__device__ __forceinline__ Lanes<1> fma(Lanes<1> a, Lanes<1> b, Lanes<1> c) { return {fmaf(a.v, b.v, c.v)}; }
__device__ __forceinline__ Lanes<2> operator+(Lanes<2> a, Lanes<2> b) {
    Lanes<2> r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ Lanes<2> operator*(Lanes<2> a, Lanes<2> b) {
    Lanes<2> r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ Lanes<2> fma(Lanes<2> a, Lanes<2> b, Lanes<2> c) {
    Lanes<2> r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}

// f = sigmoid(g) and 1 - f, each to its own relative precision: with e = exp(-g), f = 1 / (1 + e) and 1 - f = e f. g is capped
// from below so that e and f stay normal numbers: at -87 (f = 1.6e-38) where a channel has a reciprocal of its own. Two
// 16-bit channels share one, f_0 = d_1 / (d_0 d_1) with d = 1 + e (the special unit takes 16 a clock and SM, and two of
// these for every value would be half of its time): there at -41.5, where f = 2^-60 is nothing beside 1 - f = 1, so that the
// product stays finite; a NaN gate, whose d the minimum leaves out of the product, stays in its own channel.
__device__ __forceinline__ float reciprocal(float d) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d));
    return r;
}
__device__ __forceinline__ void gate(const float (&g)[1], Lanes<1> &f, Lanes<1> &keep) {
    const float e = pb::ex2_approx(-1.4426950408889634f * g[0]);
    f = Lanes<1>::of(reciprocal(1.0f + e));
    keep = Lanes<1>::of(e) * f;
}
__device__ __forceinline__ void gate(const float (&g)[2], Lanes<2> &f, Lanes<2> &keep) {
    float t[2], d[2];
    (Lanes<2>::of(g) * Lanes<2>::of(-1.4426950408889634f)).get(t);
    const Lanes<2> e = Lanes<2>::of(pb::ex2_approx(t[0]), pb::ex2_approx(t[1]));
    (e + Lanes<2>::of(1.0f)).get(d);
    d[0] = fminf(d[0], 0x1p62f);
    d[1] = fminf(d[1], 0x1p62f);
    const float r = reciprocal(__fmul_rn(d[0], d[1]));
    f = fma(e, Lanes<2>::of(0.0f), Lanes<2>::of(__fmul_rn(r, d[1]), __fmul_rn(r, d[0])));
    keep = e * f;
}

__device__ __forceinline__ void st_cluster_f32x2(unsigned addr, float a, float b) {
    asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(addr), "f"(a), "f"(b) : "memory");
}

// Arrival at the cluster's barrier by a warp that has written nothing the others read: no fence, which would wait for
// the warp's stores of results.
__device__ __forceinline__ void cluster_arrive_relaxed() {
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
}

struct Walk {        // one [B, T, D] array: elements between sequences and between steps
    void *p;
    long long sb, st;
};

struct ScanArgs {
    Walk g, x, h, dh, dg, dx;
    const float *h0, *dlast;
    float *last, *carry, *dh0;
    const void *lens;
    int wide_lens, B, T, D, blocks;   // blocks: channel blocks per sequence
};

__device__ __forceinline__ int length_of(const ScanArgs &a, int b) {
    if (!a.lens) return a.T;
    const long long n = a.wide_lens ? static_cast<const long long *>(a.lens)[b]
                                    : (long long)static_cast<const int *>(a.lens)[b];
    return (int)pb::ll_max(0, pb::ll_min(n, a.T));
}

template <typename T>
__device__ __forceinline__ T *start_of(const Walk &w, int b, int c0) {
    return static_cast<T *>(w.p) + b * w.sb + c0;
}

// The steps of a warp's run, a fixed number of rows apart. The warp's number is broadcast so that addresses and bounds
// are known to be the same for all lanes.
template <typename T, bool VEC, int S>
__device__ __forceinline__ void load_run(unsigned (&w)[S], const T *p, long long st, int steps, int lane, int n) {
    if (steps >= S) {
#pragma unroll
        for (int s = 0; s < S; ++s) w[s] = load_word<T, VEC>(p + s * st, lane, n);
    } else {
#pragma unroll
        for (int s = 0; s < S; ++s) w[s] = s < steps ? load_word<T, VEC>(p + s * st, lane, n) : 0u;
    }
}

// grid.x = sequences x channel blocks x C; a cluster of C CTAs works on C tiles of one sequence at a time. A round: every
// warp folds its run; one warp per channel plane folds the tile's runs, exchanges the tile's (A, B) within the cluster
// and leaves the state that enters each run; every warp steps through its run. The next round's inputs are in
// registers before the exchange begins.
template <typename T, bool VEC, int S, int W>
__global__ void __launch_bounds__(W * 32, 2) scan_forward(const ScanArgs a, const int C) {
    static_assert(S * W == kTile, "one stored state per tile");
    constexpr int CH = Word<T>::CH;
    using L = Lanes<CH>;
    __shared__ float2 s_run[W][CH][32];              // (A, B) of each run
    __shared__ float s_in[W][CH][32];                // state entering each run
    __shared__ float2 s_tile[2][kMaxRanks][CH][32];  // (A, B) of the cluster's tiles, by round parity
    const int lane = threadIdx.x & 31, warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
    const int rank = C > 1 ? (int)cluster_ctarank() : 0;
    const int item = blockIdx.x / C, b = item / a.blocks, c0 = (item % a.blocks) * 32 * CH;
    const int n = min(a.D - c0, 32 * CH), len = length_of(a, b);
    const T *g = start_of<T>(a.g, b, c0), *x = start_of<T>(a.x, b, c0);
    T *h = start_of<T>(a.h, b, c0);

    float state = 0.0f;   // of a plane's warp: entering the cluster's tiles of this turn
    const int mine = lane * CH + warp;
    if (warp < CH && a.h0 && mine < n) state = a.h0[(long long)b * a.D + c0 + mine];
    if (C > 1) {          // every CTA runs before the first store into its shared memory
        cluster_arrive();
        cluster_wait();
    }
    const int stride = C * kTile, rounds = (len + stride - 1) / stride;
    int t0 = rank * kTile + warp * S;
    unsigned gw[S], xw[S];
    load_run<T, VEC, S>(gw, g + t0 * a.g.st, a.g.st, len - t0, lane, n);
    load_run<T, VEC, S>(xw, x + t0 * a.x.st, a.x.st, len - t0, lane, n);
    for (int round = 0; round < rounds; ++round, t0 += stride) {
        const int par = round & 1;
        L f[S], u[S], A, B;
#pragma unroll
        for (int s = 0; s < S; ++s) {
            float gv[CH], xv[CH];
            Word<T>::unpack(Word<T>::cap(gw[s]), gv);
            Word<T>::unpack(xw[s], xv);
            gate(gv, f[s], u[s]);
            u[s] = u[s] * L::of(xv);
        }
        if (t0 + S > len) {           // behind the end the state is held
#pragma unroll
            for (int s = 0; s < S; ++s)
                if (t0 + s >= len) {
                    f[s] = L::of(1.0f);
                    u[s] = L::of(0.0f);
                }
        }
        A = L::of(1.0f);
        B = L::of(0.0f);
#pragma unroll
        for (int s = 0; s < S; ++s) {
            A = A * f[s];
            B = fma(f[s], B, u[s]);
        }
        {
            float av[CH], bv[CH];
            A.get(av);
            B.get(bv);
#pragma unroll
            for (int j = 0; j < CH; ++j) s_run[warp][j][lane] = make_float2(av[j], bv[j]);
        }
        if (round + 1 < rounds) {
            const long long t = t0 + stride;
            load_run<T, VEC, S>(gw, g + t * a.g.st, a.g.st, len - (int)t, lane, n);
            load_run<T, VEC, S>(xw, x + t * a.x.st, a.x.st, len - (int)t, lane, n);
        }
        __syncthreads();
        float2 run[W];
        if (warp < CH) {
#pragma unroll
            for (int w = 0; w < W; ++w) run[w] = s_run[w][warp][lane];
        }
        if (C > 1) {
            if (warp < CH) {
                float ta = 1.0f, tb = 0.0f;
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    ta *= run[w].x;
                    tb = fmaf(run[w].x, tb, run[w].y);
                }
                const unsigned at = smem_u32(&s_tile[par][rank][warp][lane]);
                for (int r = 0; r < C; ++r) st_cluster_f32x2(map_to_rank(at, r), ta, tb);
            }
            cluster_arrive();
            cluster_wait();
        }
        if (warp < CH) {
            float in = state;
            if (C > 1) {
                for (int r = 0; r < C; ++r) {
                    if (r == rank) in = state;
                    const float2 v = s_tile[par][r][warp][lane];
                    state = fmaf(v.x, state, v.y);
                }
            }
            const int tile = round * C + rank;
            if (a.carry && mine < n && tile * kTile < len)
                a.carry[((long long)b * ((a.T + kTile - 1) / kTile) + tile) * a.D + c0 + mine] = in;
#pragma unroll
            for (int w = 0; w < W; ++w) {
                s_in[w][warp][lane] = in;
                in = fmaf(run[w].x, in, run[w].y);
            }
            if (C == 1) state = in;
        }
        __syncthreads();
        float v[CH];
#pragma unroll
        for (int j = 0; j < CH; ++j) v[j] = s_in[warp][j][lane];
        L hs = L::of(v);
        T *out = h + t0 * a.h.st;
        if (t0 + S <= len) {
#pragma unroll
            for (int s = 0; s < S; ++s) {
                hs = fma(f[s], hs, u[s]);
                hs.get(v);
                store_word<T, VEC>(out + s * a.h.st, lane, n, Word<T>::pack(v));
            }
        } else {
#pragma unroll
            for (int s = 0; s < S; ++s) {
                hs = fma(f[s], hs, u[s]);
                hs.get(v);
                if (t0 + s < a.T) store_word<T, VEC>(out + s * a.h.st, lane, n, t0 + s < len ? Word<T>::pack(v) : 0u);
            }
        }
    }
    for (; t0 < a.T; t0 += stride)     // behind the end
        for (int s = 0; s < S && t0 + s < a.T; ++s) store_word<T, VEC>(h + (t0 + s) * a.h.st, lane, n, 0u);
    if (a.last && rank == 0 && warp < CH && mine < n) a.last[(long long)b * a.D + c0 + mine] = state;
}

template <typename T, bool VEC, int S, int W>
__global__ void __launch_bounds__(W * 32) scan_backward(const ScanArgs a, const int C) {
    static_assert(S * W == kTile, "one stored state per tile");
    constexpr int CH = Word<T>::CH;
    using L = Lanes<CH>;
    __shared__ float2 s_run[W][CH][32];              // (A, B) of each run's states
    __shared__ float s_back[W][CH][32];              // B of each run's gradients; their A is the same product
    __shared__ float s_in[W][CH][32], s_out[W][CH][32];     // state entering each run; c entering it from behind
    __shared__ float2 s_tile[2][kMaxRanks][CH][32];
    const int lane = threadIdx.x & 31, warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
    const int rank = C > 1 ? (int)cluster_ctarank() : 0;
    const int item = blockIdx.x / C, b = item / a.blocks, c0 = (item % a.blocks) * 32 * CH;
    const int n = min(a.D - c0, 32 * CH), len = length_of(a, b);
    const T *g = start_of<T>(a.g, b, c0), *x = start_of<T>(a.x, b, c0), *dh = start_of<T>(a.dh, b, c0);
    T *dg = start_of<T>(a.dg, b, c0), *dx = start_of<T>(a.dx, b, c0);
    const int plane = warp < CH ? warp : warp - CH, mine = lane * CH + plane;
    const float *carry = a.carry + (long long)b * ((a.T + kTile - 1) / kTile) * a.D + c0 + mine;

    float back = 0.0f;    // of a plane's warp: c entering the cluster's tiles of this turn from behind
    if (warp < CH && a.dlast && mine < n) back = a.dlast[(long long)b * a.D + c0 + mine];
    if (C > 1) {
        cluster_arrive();
        cluster_wait();
    }
    const int stride = C * kTile, rounds = (len + stride - 1) / stride;
    for (int t = rounds * stride + rank * kTile + warp * S; t < a.T; t += stride)     // behind the end
        for (int s = 0; s < S && t + s < a.T; ++s) {
            store_word<T, VEC>(dg + (t + s) * a.dg.st, lane, n, 0u);
            store_word<T, VEC>(dx + (t + s) * a.dx.st, lane, n, 0u);
        }
    int t0 = (rounds - 1) * stride + rank * kTile + warp * S;
    unsigned gw[S], xw[S], dw[S];
    float stored = 0.0f;  // of the second set of planes' warps: the state at the start of the tile
    auto fetch = [&](long long t, int tile) {
        load_run<T, VEC, S>(gw, g + t * a.g.st, a.g.st, len - (int)t, lane, n);
        load_run<T, VEC, S>(xw, x + t * a.x.st, a.x.st, len - (int)t, lane, n);
        load_run<T, VEC, S>(dw, dh + t * a.dh.st, a.dh.st, a.dh.p ? len - (int)t : 0, lane, n);
        if (warp >= CH && warp < 2 * CH) stored = mine < n && tile * kTile < len ? carry[(long long)tile * a.D] : 0.0f;
    };
    if (rounds > 0) fetch(t0, (rounds - 1) * C + rank);
    for (int round = rounds - 1; round >= 0; --round, t0 -= stride) {
        const int par = round & 1;
        L f[S], keep[S], A, B, R = L::of(0.0f);
        unsigned xn[S], dn[S];
        const float entering = stored;
#pragma unroll
        for (int s = 0; s < S; ++s) {
            float gv[CH];
            Word<T>::unpack(Word<T>::cap(gw[s]), gv);
            gate(gv, f[s], keep[s]);
            xn[s] = xw[s];
            dn[s] = dw[s];
        }
        if (t0 + S > len) {
#pragma unroll
            for (int s = 0; s < S; ++s)
                if (t0 + s >= len) {
                    f[s] = L::of(1.0f);
                    keep[s] = L::of(0.0f);
                }
        }
        A = L::of(1.0f);
        B = L::of(0.0f);
#pragma unroll
        for (int s = 0; s < S; ++s) {
            float xv[CH];
            Word<T>::unpack(xn[s], xv);
            A = A * f[s];
            B = fma(f[s], B, keep[s] * L::of(xv));
        }
#pragma unroll
        for (int s = S - 1; s >= 0; --s) {       // r_s = dh_s + f_{s+1} r_{s+1}
            float dv[CH];
            Word<T>::unpack(dn[s], dv);
            R = s == S - 1 ? L::of(dv) : fma(f[s + 1 < S ? s + 1 : s], R, L::of(dv));
        }
        R = f[0] * R;
        {
            float av[CH], bv[CH], rv[CH];
            A.get(av);
            B.get(bv);
            R.get(rv);
#pragma unroll
            for (int j = 0; j < CH; ++j) {
                s_run[warp][j][lane] = make_float2(av[j], bv[j]);
                s_back[warp][j][lane] = rv[j];
            }
        }
        if (round > 0) fetch(t0 - stride, (round - 1) * C + rank);
        __syncthreads();
        if (warp >= CH && warp < 2 * CH) {
            float in = entering;
#pragma unroll
            for (int w = 0; w < W; ++w) {
                const float2 r = s_run[w][plane][lane];
                s_in[w][plane][lane] = in;
                in = fmaf(r.x, in, r.y);
            }
        }
        if (C > 1) {
            if (warp < CH) {
                float qa = 1.0f, qb = 0.0f;
#pragma unroll
                for (int w = W - 1; w >= 0; --w) {
                    const float aw = s_run[w][plane][lane].x;
                    qa *= aw;
                    qb = fmaf(aw, qb, s_back[w][plane][lane]);
                }
                const unsigned at = smem_u32(&s_tile[par][rank][plane][lane]);
                for (int r = 0; r < C; ++r) st_cluster_f32x2(map_to_rank(at, r), qa, qb);
            }
            cluster_arrive();
            cluster_wait();
        }
        if (warp < CH) {
            float out = back;
            if (C > 1) {
                for (int r = C - 1; r >= 0; --r) {
                    if (r == rank) out = back;
                    const float2 v = s_tile[par][r][plane][lane];
                    back = fmaf(v.x, back, v.y);
                }
            }
#pragma unroll
            for (int w = W - 1; w >= 0; --w) {
                s_out[w][plane][lane] = out;
                out = fmaf(s_run[w][plane][lane].x, out, s_back[w][plane][lane]);
            }
            if (C == 1) back = out;
        }
        __syncthreads();
        // the states before each step, then backwards through the run
        float v[CH];
        L before[S];
#pragma unroll
        for (int j = 0; j < CH; ++j) v[j] = s_in[warp][j][lane];
        L hs = L::of(v);
#pragma unroll
        for (int s = 0; s < S; ++s) {
            float xv[CH];
            Word<T>::unpack(xn[s], xv);
            before[s] = hs;
            hs = fma(f[s], hs, keep[s] * L::of(xv));
        }
#pragma unroll
        for (int j = 0; j < CH; ++j) v[j] = s_out[warp][j][lane];
        L r = L::of(v);
        T *const ox = dx + t0 * a.dx.st, *const og = dg + t0 * a.dg.st;
#pragma unroll
        for (int s = S - 1; s >= 0; --s) {
            float xv[CH], dv[CH], gx[CH], gg[CH];
            Word<T>::unpack(xn[s], xv);
            Word<T>::unpack(dn[s], dv);
            r = s == S - 1 ? L::of(dv) + r : fma(f[s + 1 < S ? s + 1 : s], r, L::of(dv));
            const L kr = keep[s] * r, gl = kr * (f[s] * fma(L::of(xv), L::of(-1.0f), before[s]));
            kr.get(gx);
            gl.get(gg);
            if (t0 + s < a.T) {
                const bool alive = t0 + s < len;
                store_word<T, VEC>(ox + s * a.dx.st, lane, n, alive ? Word<T>::pack(gx) : 0u);
                store_word<T, VEC>(og + s * a.dg.st, lane, n, alive ? Word<T>::pack(gg) : 0u);
            }
        }
    }
    if (a.dh0 && rank == 0 && warp < CH && mine < n) a.dh0[(long long)b * a.D + c0 + mine] = back;
}

// ---- the same two kernels where rows allow 16-byte access ----------------------------------------------------------
// A warp's run of S steps x 128 bytes of channels lies in S rows of shared memory that only this warp uses: fetched
// with 16-byte asynchronous copies up to kStages - 1 rounds ahead, read with 4-byte loads at constant offsets, overwritten
// in place by the results, and written back 16 bytes a lane during the next round's exchange.
//
// Measured (bf16): 1 x 65536 x 2048 in 195 us (4.1 TB/s, 63 % of the measured copy rate), 16 x 1000..4000 x 2048 forward in
// 110 us (78 %) and backward in 225 us (66 %); fp32, 16 x 1000..4000 x 1024, in 105 us (82 %) and 180 us (82 %). What bounds them: a round is a chain of barriers (fold, exchange,
// step), and the two CTAs of an SM (one, backward) do not fill each other's waits; without the exchange between
// the cluster's CTAs the long sequence would take 164 us, without the gates 176 us, without both 143 us. Loading and
// storing 4 bytes a lane and step straight from global memory spends two thirds of the instructions on addresses (270 us,
// and 176 + 314 us); folding all runs in every warp instead of in one warp per channel plane cost 356 us. Eight steps a
// warp and 16 warps forward (64 registers) cost 577 us, two stages and three CTAs an SM 234 us.
__device__ __forceinline__ void copy16(unsigned to, const void *from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// One array's rows of a warp's runs: 128 bytes of each step, a lane moving 16 bytes of every fourth row. `at` is the
// lane's place in the run that comes next; a round moves it by `round` elements.
template <typename T, int S>
struct Rows {
    T *at;
    long long four, round;
    bool in;            // the lane's channels exist
    int sub;            // its row within four
    __device__ Rows(const Walk &w, int b, int c0, int n, int lane, int t, int stride) {
        constexpr int E = 16 / sizeof(T);
        sub = lane >> 3;
        at = start_of<T>(w, b, c0) + (lane & 7) * E + (t + sub) * w.st;
        four = 4 * w.st;
        round = stride * w.st;
        in = w.p && (lane & 7) * E < n;
    }
    // `left`: steps from the run's first to the end; whole runs, which all but a sequence's last are, need no comparison
    __device__ void fetch(unsigned to, int left) {
        const T *q = at;
        if (in) {
            if (left >= S) {
#pragma unroll
                for (int i = 0; i < S / 4; ++i, q += four) copy16(to + i * 512, q);
            } else {
#pragma unroll
                for (int i = 0; i < S / 4; ++i, q += four)
                    if (sub + 4 * i < left) copy16(to + i * 512, q);
            }
        }
        at += round;
    }
    __device__ void store(const uint4 *from, int left, int until) {     // zeros in [left, until)
        T *q = at;
        if (in) {
            if (left >= S) {
#pragma unroll
                for (int i = 0; i < S / 4; ++i, q += four) __stcs(reinterpret_cast<uint4 *>(q), from[i * 32]);
            } else {
#pragma unroll
                for (int i = 0; i < S / 4; ++i, q += four)
                    if (sub + 4 * i < until)
                        __stcs(reinterpret_cast<uint4 *>(q), sub + 4 * i < left ? from[i * 32] : make_uint4(0, 0, 0, 0));
            }
        }
        at += round;
    }
};

template <typename T, int S, int W, int NST>
__global__ void __launch_bounds__(W * 32, 2) scan_forward_staged(const ScanArgs a, const int C) {
    static_assert(S * W == kTile, "one stored state per tile");
    constexpr int CH = Word<T>::CH, kRun = S * 128;       // bytes of one array's run
    using L = Lanes<CH>;
    extern __shared__ __align__(128) unsigned char s_rows[];
    __shared__ float2 s_run[W][CH][32];              // (A, B) of each run
    __shared__ float s_in[W][CH][32];                // state entering each run
    __shared__ float2 s_tile[2][kMaxRanks][CH][32];  // (A, B) of the cluster's tiles, by round parity
    const int lane = threadIdx.x & 31, warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
    const int rank = C > 1 ? (int)cluster_ctarank() : 0;
    const int item = blockIdx.x / C, b = item / a.blocks, c0 = (item % a.blocks) * 32 * CH;
    const int n = min(a.D - c0, 32 * CH), len = length_of(a, b);
    const int stride = C * kTile, rounds = (len + stride - 1) / stride;
    int t0 = rank * kTile + warp * S, fill = 0, ahead = t0;
    Rows<T, S> g(a.g, b, c0, n, lane, t0, stride), x(a.x, b, c0, n, lane, t0, stride), h(a.h, b, c0, n, lane, t0, stride);
    unsigned char *const mine_rows = s_rows + warp * (NST * 2 * kRun);
    const uint4 *const lane_rows = reinterpret_cast<const uint4 *>(mine_rows) + lane;
    const unsigned rows = smem_u32(mine_rows) + lane * 16;

    float state = 0.0f;   // of a plane's warp: entering the cluster's tiles of this turn
    const int mine = lane * CH + warp;
    if (warp < CH && a.h0 && mine < n) state = a.h0[(long long)b * a.D + c0 + mine];
    auto fetch = [&]() {
        if (ahead < len) {
            g.fetch(rows + fill, len - ahead);
            x.fetch(rows + fill + kRun, len - ahead);
        }
        ahead += stride;
        copy_commit();
        fill = fill == (NST - 1) * 2 * kRun ? 0 : fill + 2 * kRun;
    };
#pragma unroll
    for (int i = 0; i < NST - 1; ++i) fetch();
    if (C > 1) {          // every CTA runs before the first store into its shared memory
        cluster_arrive();
        cluster_wait();
    }
    int slot = 0;
    for (int round = 0; round < rounds; ++round, t0 += stride) {
        const int par = round & 1;
        copy_wait<NST - 2>();
        __syncwarp();
        unsigned *const gr = reinterpret_cast<unsigned *>(mine_rows + slot) + lane, *const xr = gr + kRun / 4;
        const int before = slot == 0 ? (NST - 1) * 2 * kRun : slot - 2 * kRun;
        slot = slot == (NST - 1) * 2 * kRun ? 0 : slot + 2 * kRun;
        L f[S], u[S], A, B;
#pragma unroll
        for (int s = 0; s < S; ++s) {
            float gv[CH], xv[CH];
            Word<T>::unpack(Word<T>::cap(gr[s * 32]), gv);
            Word<T>::unpack(xr[s * 32], xv);
            gate(gv, f[s], u[s]);
            u[s] = u[s] * L::of(xv);
        }
        if (t0 + S > len) {                  // behind the end the state is held
#pragma unroll
            for (int s = 0; s < S; ++s)
                if (t0 + s >= len) {
                    f[s] = L::of(1.0f);
                    u[s] = L::of(0.0f);
                }
        }
        A = L::of(1.0f);
        B = L::of(0.0f);
#pragma unroll
        for (int s = 0; s < S; ++s) {
            A = A * f[s];
            B = fma(f[s], B, u[s]);
        }
        {
            float av[CH], bv[CH];
            A.get(av);
            B.get(bv);
#pragma unroll
            for (int j = 0; j < CH; ++j) s_run[warp][j][lane] = make_float2(av[j], bv[j]);
        }
        __syncthreads();
        float2 run[W];
        if (warp < CH) {
#pragma unroll
            for (int w = 0; w < W; ++w) run[w] = s_run[w][warp][lane];
        }
        if (C > 1) {
            if (warp < CH) {
                float ta = 1.0f, tb = 0.0f;
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    ta *= run[w].x;
                    tb = fmaf(run[w].x, tb, run[w].y);
                }
                const unsigned at = smem_u32(&s_tile[par][rank][warp][lane]);
                for (int r = 0; r < C; ++r) st_cluster_f32x2(map_to_rank(at, r), ta, tb);
                cluster_arrive();
            } else {
                cluster_arrive_relaxed();
            }
        }
        // while the exchange is under way: the round before goes out, and its rows take the inputs of a later one
        if (round > 0) h.store(lane_rows + (before + kRun) / 16, len - t0 + stride, a.T - t0 + stride);
        __syncwarp();
        fetch();
        if (C > 1) cluster_wait();
        if (warp < CH) {
            float in = state;
            if (C > 1) {
                for (int r = 0; r < C; ++r) {
                    if (r == rank) in = state;
                    const float2 v = s_tile[par][r][warp][lane];
                    state = fmaf(v.x, state, v.y);
                }
            }
            const int tile = round * C + rank;
            if (a.carry && mine < n && tile * kTile < len)
                a.carry[((long long)b * ((a.T + kTile - 1) / kTile) + tile) * a.D + c0 + mine] = in;
#pragma unroll
            for (int w = 0; w < W; ++w) {
                s_in[w][warp][lane] = in;
                in = fmaf(run[w].x, in, run[w].y);
            }
            if (C == 1) state = in;
        }
        __syncthreads();
        float v[CH];
#pragma unroll
        for (int j = 0; j < CH; ++j) v[j] = s_in[warp][j][lane];
        L hs = L::of(v);
#pragma unroll
        for (int s = 0; s < S; ++s) {
            hs = fma(f[s], hs, u[s]);
            hs.get(v);
            xr[s * 32] = Word<T>::pack(v);
        }
        __syncwarp();
    }
    copy_wait<0>();
    if (rounds > 0) {
        const int last = slot == 0 ? (NST - 1) * 2 * kRun : slot - 2 * kRun;
        h.store(lane_rows + (last + kRun) / 16, len - t0 + stride, a.T - t0 + stride);
    }
    for (; t0 < a.T; t0 += stride) h.store(lane_rows, 0, a.T - t0);     // behind the end
    if (a.last && rank == 0 && warp < CH && mine < n) a.last[(long long)b * a.D + c0 + mine] = state;
}

template <typename T, int S, int W, int NST>
__global__ void __launch_bounds__(W * 32) scan_backward_staged(const ScanArgs a, const int C) {
    static_assert(S * W == kTile, "one stored state per tile");
    constexpr int CH = Word<T>::CH, kRun = S * 128;
    using L = Lanes<CH>;
    extern __shared__ __align__(128) unsigned char s_rows[];
    __shared__ float2 s_run[W][CH][32];              // (A, B) of each run's states
    __shared__ float s_back[W][CH][32];              // B of each run's gradients; their A is the same product
    __shared__ float s_in[W][CH][32], s_out[W][CH][32];     // state entering each run; c entering it from behind
    __shared__ float2 s_tile[2][kMaxRanks][CH][32];
    const int lane = threadIdx.x & 31, warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
    const int rank = C > 1 ? (int)cluster_ctarank() : 0;
    const int item = blockIdx.x / C, b = item / a.blocks, c0 = (item % a.blocks) * 32 * CH;
    const int n = min(a.D - c0, 32 * CH), len = length_of(a, b);
    const int stride = C * kTile, rounds = (len + stride - 1) / stride;
    unsigned char *const mine_rows = s_rows + warp * (NST * 3 * kRun);
    const uint4 *const lane_rows = reinterpret_cast<const uint4 *>(mine_rows) + lane;
    const unsigned rows = smem_u32(mine_rows) + lane * 16;
    const int plane = warp < CH ? warp : warp - CH, mine = lane * CH + plane;
    const float *carry = a.carry + (long long)b * ((a.T + kTile - 1) / kTile) * a.D + c0 + mine;

    float back = 0.0f;    // of a plane's warp: c entering the cluster's tiles of this turn from behind
    if (warp < CH && a.dlast && mine < n) back = a.dlast[(long long)b * a.D + c0 + mine];
    {
        int t = rounds * stride + rank * kTile + warp * S;      // behind the end
        Rows<T, S> dg(a.dg, b, c0, n, lane, t, stride), dx(a.dx, b, c0, n, lane, t, stride);
        for (; t < a.T; t += stride) {
            dg.store(lane_rows, 0, a.T - t);
            dx.store(lane_rows, 0, a.T - t);
        }
    }
    int t0 = (rounds - 1) * stride + rank * kTile + warp * S, fill = 0, ahead = t0;
    Rows<T, S> g(a.g, b, c0, n, lane, t0, -stride), x(a.x, b, c0, n, lane, t0, -stride), dh(a.dh, b, c0, n, lane, t0, -stride);
    Rows<T, S> dg(a.dg, b, c0, n, lane, t0, -stride), dx(a.dx, b, c0, n, lane, t0, -stride);
    auto fetch = [&]() {
        if (ahead >= 0) {
            g.fetch(rows + fill, len - ahead);
            x.fetch(rows + fill + kRun, len - ahead);
            dh.fetch(rows + fill + 2 * kRun, len - ahead);
        }
        ahead -= stride;
        copy_commit();
        fill = fill == (NST - 1) * 3 * kRun ? 0 : fill + 3 * kRun;
    };
    auto put = [&](int slot_at, int t) {
        dg.store(lane_rows + slot_at / 16, len - t, a.T - t);
        dx.store(lane_rows + (slot_at + kRun) / 16, len - t, a.T - t);
    };
    // a second set of planes' warps holds the state at the start of the tile, one round ahead
    auto state_of = [&](int round) {
        const int tile = round * C + rank;
        return round >= 0 && warp >= CH && warp < 2 * CH && mine < n && tile * kTile < len ? carry[(long long)tile * a.D]
                                                                                           : 0.0f;
    };
    float stored = state_of(rounds - 1);
#pragma unroll
    for (int i = 0; i < NST - 1; ++i) fetch();
    if (C > 1) {
        cluster_arrive();
        cluster_wait();
    }
    int slot = 0;
    for (int round = rounds - 1; round >= 0; --round, t0 -= stride) {
        const int par = round & 1;
        const float entering = stored;
        stored = state_of(round - 1);
        copy_wait<NST - 2>();
        __syncwarp();
        const int before = slot == 0 ? (NST - 1) * 3 * kRun : slot - 3 * kRun;
        unsigned *const gr = reinterpret_cast<unsigned *>(mine_rows + slot) + lane, *const xr = gr + kRun / 4,
                       *const dr = xr + kRun / 4;
        slot = slot == (NST - 1) * 3 * kRun ? 0 : slot + 3 * kRun;
        L f[S], keep[S], xl[S], dl[S], A, B, R = L::of(0.0f);
#pragma unroll
        for (int s = 0; s < S; ++s) {
            float gv[CH], xv[CH], dv[CH];
            Word<T>::unpack(Word<T>::cap(gr[s * 32]), gv);
            Word<T>::unpack(xr[s * 32], xv);
            Word<T>::unpack(dr[s * 32], dv);
            gate(gv, f[s], keep[s]);
            xl[s] = L::of(xv);
            dl[s] = L::of(dv);
        }
        const bool cut = t0 + S > len;
        if (cut) {                           // behind the end: held, and no gradient
#pragma unroll
            for (int s = 0; s < S; ++s)
                if (t0 + s >= len) {
                    f[s] = L::of(1.0f);
                    keep[s] = L::of(0.0f);
                    xl[s] = dl[s] = L::of(0.0f);
                }
        }
        if (!a.dh.p) {
#pragma unroll
            for (int s = 0; s < S; ++s) dl[s] = L::of(0.0f);
        }
        A = L::of(1.0f);
        B = L::of(0.0f);
#pragma unroll
        for (int s = 0; s < S; ++s) {
            A = A * f[s];
            B = fma(f[s], B, keep[s] * xl[s]);
        }
#pragma unroll
        for (int s = S - 1; s >= 0; --s) {       // r_s = dh_s + f_{s+1} r_{s+1}
            R = s == S - 1 ? dl[s] : fma(f[s + 1 < S ? s + 1 : s], R, dl[s]);
        }
        R = f[0] * R;
        {
            float av[CH], bv[CH], rv[CH];
            A.get(av);
            B.get(bv);
            R.get(rv);
#pragma unroll
            for (int j = 0; j < CH; ++j) {
                s_run[warp][j][lane] = make_float2(av[j], bv[j]);
                s_back[warp][j][lane] = rv[j];
            }
        }
        __syncthreads();
        if (warp >= CH && warp < 2 * CH) {
            float in = entering;
#pragma unroll
            for (int w = 0; w < W; ++w) {
                const float2 r = s_run[w][plane][lane];
                s_in[w][plane][lane] = in;
                in = fmaf(r.x, in, r.y);
            }
        }
        if (C > 1) {
            if (warp < CH) {
                float qa = 1.0f, qb = 0.0f;
#pragma unroll
                for (int w = W - 1; w >= 0; --w) {
                    const float aw = s_run[w][plane][lane].x;
                    qa *= aw;
                    qb = fmaf(aw, qb, s_back[w][plane][lane]);
                }
                const unsigned at = smem_u32(&s_tile[par][rank][plane][lane]);
                for (int r = 0; r < C; ++r) st_cluster_f32x2(map_to_rank(at, r), qa, qb);
                cluster_arrive();
            } else {
                cluster_arrive_relaxed();
            }
        }
        // while the exchange is under way: the round before goes out, and its rows take the inputs of a later one
        if (round < rounds - 1) put(before, t0 + stride);
        __syncwarp();
        fetch();
        if (C > 1) cluster_wait();
        if (warp < CH) {
            float out = back;
            if (C > 1) {
                for (int r = C - 1; r >= 0; --r) {
                    if (r == rank) out = back;
                    const float2 v = s_tile[par][r][plane][lane];
                    back = fmaf(v.x, back, v.y);
                }
            }
#pragma unroll
            for (int w = W - 1; w >= 0; --w) {
                s_out[w][plane][lane] = out;
                out = fmaf(s_run[w][plane][lane].x, out, s_back[w][plane][lane]);
            }
            if (C == 1) back = out;
        }
        __syncthreads();
        // f (h_{t-1} - x) of each step, then backwards through the run
        float v[CH];
        L q[S];
#pragma unroll
        for (int j = 0; j < CH; ++j) v[j] = s_in[warp][j][lane];
        L hs = L::of(v);
#pragma unroll
        for (int s = 0; s < S; ++s) {
            q[s] = f[s] * fma(xl[s], L::of(-1.0f), hs);
            hs = fma(f[s], hs, keep[s] * xl[s]);
        }
#pragma unroll
        for (int j = 0; j < CH; ++j) v[j] = s_out[warp][j][lane];
        L r = L::of(v);
#pragma unroll
        for (int s = S - 1; s >= 0; --s) {
            float gx[CH], gg[CH];
            r = s == S - 1 ? dl[s] + r : fma(f[s + 1 < S ? s + 1 : s], r, dl[s]);
            const L kr = keep[s] * r, gl = kr * q[s];
            kr.get(gx);
            gl.get(gg);
            xr[s * 32] = Word<T>::pack(gx);
            gr[s * 32] = Word<T>::pack(gg);
        }
        __syncwarp();
    }
    copy_wait<0>();
    if (rounds > 0) put(slot == 0 ? (NST - 1) * 3 * kRun : slot - 3 * kRun, t0 + stride);
    if (a.dh0 && rank == 0 && warp < CH && mine < n) a.dh0[(long long)b * a.D + c0 + mine] = back;
}

// ---- one token for every row (bounded by memory: 2048 x 8192 bf16 in 38 us, 93 % of the measured copy rate) --------
// 8 channels per thread where the rows allow 16-byte access, else 2 (2, because a pair of 16-bit channels shares its
// reciprocal: the step then has the scan's bits).
template <typename T, int VN>
__global__ void __launch_bounds__(256) scan_step(const T *g, const T *x, const float *state, T *h, float *last,
                                                 long long N, int D, long long ldg, long long ldx, long long ldh) {
    constexpr int CH = Word<T>::CH;
    const int per = (D + VN - 1) / VN;
    const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= N * per) return;
    const long long row = i / per;
    const int c = (int)(i % per) * VN;
    const long long at = row * D + c;
    __align__(16) T gv[VN];
    __align__(16) T xv[VN];
    __align__(16) T hv[VN];
    __align__(16) float sv[VN];
    __align__(16) float lv[VN];
    if constexpr (VN == 2) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const bool in = c + k < D;
            gv[k] = in ? g[row * ldg + c + k] : (T)0.0f;
            xv[k] = in ? x[row * ldx + c + k] : (T)0.0f;
            sv[k] = in ? state[at + k] : 0.0f;
        }
    } else {
        constexpr int NV = VN * sizeof(T) / 16, NS = VN / 4;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            reinterpret_cast<uint4 *>(gv)[k] = reinterpret_cast<const uint4 *>(g + row * ldg + c)[k];
            reinterpret_cast<uint4 *>(xv)[k] = reinterpret_cast<const uint4 *>(x + row * ldx + c)[k];
        }
#pragma unroll
        for (int k = 0; k < NS; ++k)
            reinterpret_cast<float4 *>(sv)[k] = reinterpret_cast<const float4 *>(state + at)[k];
    }
#pragma unroll
    for (int k = 0; k < VN; k += CH) {
        float gk[CH], xk[CH], sk[CH];
#pragma unroll
        for (int j = 0; j < CH; ++j) {
            const float v = (float)gv[k + j];
            gk[j] = v < Word<T>::kCap ? Word<T>::kCap : v;
            xk[j] = (float)xv[k + j];
            sk[j] = sv[k + j];
        }
        Lanes<CH> f, keep;
        gate(gk, f, keep);
        fma(f, Lanes<CH>::of(sk), keep * Lanes<CH>::of(xk)).get(sk);
#pragma unroll
        for (int j = 0; j < CH; ++j) {
            lv[k + j] = sk[j];
            hv[k + j] = (T)sk[j];
        }
    }
    if constexpr (VN == 2) {
#pragma unroll
        for (int k = 0; k < 2; ++k)
            if (c + k < D) {
                h[row * ldh + c + k] = hv[k];
                last[at + k] = lv[k];
            }
    } else {
        constexpr int NV = VN * sizeof(T) / 16, NS = VN / 4;
#pragma unroll
        for (int k = 0; k < NV; ++k) reinterpret_cast<uint4 *>(h + row * ldh + c)[k] = reinterpret_cast<uint4 *>(hv)[k];
#pragma unroll
        for (int k = 0; k < NS; ++k) reinterpret_cast<float4 *>(last + at)[k] = reinterpret_cast<float4 *>(lv)[k];
    }
}

// ---- host side ---------------------------------------------------------------------------------------------
size_t bytes_of(int32_t dtype) { return dtype == PARPY_B200_F32 ? 4 : 2; }

int32_t check_scan(const char *what, int32_t dtype, int64_t B, int64_t T, int64_t D) {
    PB_REQUIRE(dtype == PARPY_B200_F32 || dtype == PARPY_B200_BF16 || dtype == PARPY_B200_F16,
               "%s: unknown element type %d", what, dtype);
    PB_REQUIRE(B >= 0 && T >= 0 && D >= 0 && B <= INT_MAX && T <= INT_MAX - (1 << 16) && D <= INT_MAX - 64,
               "%s: shape (%lld, %lld, %lld) is not supported", what, (long long)B, (long long)T, (long long)D);
    return PB_OK;
}

// strides must reach the next row, and every row must start at an element
int32_t check_walk(const char *what, const char *name, const Walk &w, int32_t dtype, int64_t B, int64_t T, int64_t D,
                   bool output) {
    PB_REQUIRE(w.p, "%s: null pointer (%s)", what, name);
    PB_REQUIRE(reinterpret_cast<uintptr_t>(w.p) % bytes_of(dtype) == 0, "%s: misaligned %s", what, name);
    PB_REQUIRE(w.sb >= 0 && w.st >= 0, "%s: negative strides of %s", what, name);
    if (output) {
        const bool steps_inside = B <= 1 || (T <= 1 ? w.sb >= D : w.sb >= w.st && w.sb >= (T - 1) * w.st + D);
        const bool rows_inside = T <= 1 || (B <= 1 ? w.st >= D : w.st >= w.sb && w.st >= (B - 1) * w.sb + D);
        const bool apart = (B <= 1 && T <= 1) || (B <= 1 ? rows_inside : T <= 1 ? steps_inside
                           : (w.st >= D && steps_inside) || (w.sb >= D && rows_inside));
        PB_REQUIRE(apart, "%s: rows of %s overlap", what, name);
    }
    return PB_OK;
}

// whether every row of an array starts on a 16-byte boundary
bool wide_rows(const Walk &w, int32_t dtype) {
    const int64_t e = 16 / (int64_t)bytes_of(dtype);
    return !w.p || (pb::aligned16(w.p) && w.sb % e == 0 && w.st % e == 0);
}

bool words(const Walk &w, int32_t dtype) {
    return !w.p || dtype == PARPY_B200_F32 ||
           (reinterpret_cast<uintptr_t>(w.p) % 4 == 0 && w.sb % 2 == 0 && w.st % 2 == 0);
}

template <typename K>
int32_t launch_scan(K kernel, const char *what, ScanArgs &a, int channels, int threads, size_t smem, int C,
                    cudaStream_t stream) {
    if (smem) PB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    a.blocks = (a.D + channels - 1) / channels;
    const long long grid = (long long)a.B * a.blocks * C;
    PB_REQUIRE(grid <= INT_MAX, "%s: shape (%d, %d, %d) needs too many blocks", what, a.B, a.T, a.D);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim = {(unsigned)C, 1, 1};
    cfg.attrs = attr;
    cfg.numAttrs = C > 1 ? 1 : 0;
    const ScanArgs &args = a;
    PB_CUDA(cudaLaunchKernelEx(&cfg, kernel, args, C));
    return PB_OK;
}

// CTAs of a cluster, which share a sequence's tiles: one where the channel blocks alone occupy two thirds of the SMs, else
// as many as are resident at once (two an SM forward, one backward). An exchange a round costs more than idle SMs or
// a second wave: bf16, 2048 channels, 2000 steps a sequence, for 1 / 2 / 4 / 8 CTAs a cluster, forward 29 / 33 / 35 / 41 us at 128
// blocks, 49 / 41 / 33 / 37 at 64 (twice the steps), 90 / 72 / 41 / 33 at 32 (four times); backward 45 / 70 / 78 / 98,
// 82 / 68 / 72 / 94 and 156 / 119 / 68 / 100 us.
int cluster_of(const ScanArgs &a, int channels, int sms, int per_sm) {
    const long long blocks = (long long)a.B * ((a.D + channels - 1) / channels);
    int C = 1;
    if (3 * blocks < 2LL * sms)
        while (C < kMaxRanks && 2 * C * blocks <= (long long)per_sm * sms && (long long)C * kTile < a.T) C *= 2;
    return C;
}

enum Access { kElements, kWords, kWide };     // how rows are read: 2 or 4 bytes a lane, or staged 16 bytes a lane

template <typename T, Access ACC>
int32_t run_forward(ScanArgs &a, const pb::DeviceInfo &dev, cudaStream_t stream) {
    constexpr int channels = 32 * Word<T>::CH;
    const int C = cluster_of(a, channels, dev.sm_count, 2);
    if constexpr (ACC == kWide)
        return launch_scan(scan_forward_staged<T, 16, 8, kStages>, "gated_scan", a, channels, 256,
                           kStages * 2 * kTile * 128, C, stream);
    return launch_scan(scan_forward<T, ACC != kElements, 16, 8>, "gated_scan", a, channels, 256, 0, C, stream);
}
template <typename T, Access ACC>
int32_t run_backward(ScanArgs &a, const pb::DeviceInfo &dev, cudaStream_t stream) {
    constexpr int channels = 32 * Word<T>::CH;
    const int C = cluster_of(a, channels, dev.sm_count, 1);
    if constexpr (ACC == kWide)
        return launch_scan(scan_backward_staged<T, 8, 16, kStages>, "gated_scan_grad", a, channels, 512,
                           kStages * 3 * kTile * 128, C, stream);
    return launch_scan(scan_backward<T, ACC != kElements, 8, 16>, "gated_scan_grad", a, channels, 512, 0, C, stream);
}
template <typename T>
int32_t run_step(const void *g, const void *x, const float *state, void *h, float *last, int64_t N, int64_t D,
                 int64_t ldg, int64_t ldx, int64_t ldh, cudaStream_t stream) {
    constexpr int E = 16 / sizeof(T);
    const bool wide = D % 8 == 0 && ldg % E == 0 && ldx % E == 0 && ldh % E == 0 && pb::aligned16(g) &&
                      pb::aligned16(x) && pb::aligned16(state) && pb::aligned16(h) && pb::aligned16(last);
    const long long work = N * (wide ? D / 8 : (D + 1) / 2), blocks = (work + 255) / 256;
    PB_REQUIRE(blocks <= INT_MAX, "gated_step: shape (%lld, %lld) is too large", (long long)N, (long long)D);
    const T *gt = static_cast<const T *>(g), *xt = static_cast<const T *>(x);
    if (wide) scan_step<T, 8><<<(unsigned)blocks, 256, 0, stream>>>(gt, xt, state, static_cast<T *>(h), last, N, (int)D, ldg, ldx, ldh);
    else scan_step<T, 2><<<(unsigned)blocks, 256, 0, stream>>>(gt, xt, state, static_cast<T *>(h), last, N, (int)D, ldg, ldx, ldh);
    PB_CUDA(cudaGetLastError());
    return PB_OK;
}

Walk walk(const void *p, int64_t sb, int64_t st) { return Walk{const_cast<void *>(p), sb, st}; }

}  // namespace

extern "C" {

int32_t parpy_b200_gated_scan(int32_t dtype, int64_t B, int64_t T, int64_t D, const void *g, int64_t g_sb,
                              int64_t g_st, const void *x, int64_t x_sb, int64_t x_st, const float *h0,
                              const void *lens, int32_t wide_lens, void *h, int64_t h_sb, int64_t h_st, float *last,
                              float *carry, void *stream) {
    const char *what = "gated_scan";
    int32_t rc = check_scan(what, dtype, B, T, D);
    if (rc || B == 0 || D == 0) return rc;
    ScanArgs a = {};
    if (T > 0) {
        a.g = walk(g, g_sb, g_st);
        a.x = walk(x, x_sb, x_st);
        a.h = walk(h, h_sb, h_st);
        rc = check_walk(what, "g", a.g, dtype, B, T, D, false);
        if (!rc) rc = check_walk(what, "x", a.x, dtype, B, T, D, false);
        if (!rc) rc = check_walk(what, "h", a.h, dtype, B, T, D, true);
        if (rc) return rc;
    }
    a.h0 = h0;
    a.last = last;
    a.carry = carry;
    a.lens = lens;
    a.wide_lens = wide_lens;
    a.B = (int)B;
    a.T = (int)T;
    a.D = (int)D;
    pb::DeviceInfo dev;
    rc = pb::device_info(&dev);
    if (rc) return rc;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool wide = D % (16 / (int64_t)bytes_of(dtype)) == 0 && wide_rows(a.g, dtype) && wide_rows(a.x, dtype) &&
                      wide_rows(a.h, dtype);
    const bool vec = D % 2 == 0 && words(a.g, dtype) && words(a.x, dtype) && words(a.h, dtype);
    if (dtype == PARPY_B200_F32) return wide ? run_forward<float, kWide>(a, dev, s) : run_forward<float, kWords>(a, dev, s);
    if (dtype == PARPY_B200_BF16)
        return wide ? run_forward<__nv_bfloat16, kWide>(a, dev, s)
               : vec ? run_forward<__nv_bfloat16, kWords>(a, dev, s)
                     : run_forward<__nv_bfloat16, kElements>(a, dev, s);
    return wide ? run_forward<__half, kWide>(a, dev, s)
           : vec ? run_forward<__half, kWords>(a, dev, s)
                 : run_forward<__half, kElements>(a, dev, s);
}

int32_t parpy_b200_gated_scan_grad(int32_t dtype, int64_t B, int64_t T, int64_t D, const void *g, int64_t g_sb,
                                   int64_t g_st, const void *x, int64_t x_sb, int64_t x_st, const void *lens,
                                   int32_t wide_lens, const float *carry, const void *dh, int64_t dh_sb, int64_t dh_st,
                                   const float *dlast, void *dg, int64_t dg_sb, int64_t dg_st, void *dx, int64_t dx_sb,
                                   int64_t dx_st, float *dh0, void *stream) {
    const char *what = "gated_scan_grad";
    int32_t rc = check_scan(what, dtype, B, T, D);
    if (rc || B == 0 || D == 0) return rc;
    ScanArgs a = {};
    if (T > 0) {
        PB_REQUIRE(carry, "%s: null pointer (carry)", what);
        a.g = walk(g, g_sb, g_st);
        a.x = walk(x, x_sb, x_st);
        a.dh = walk(dh, dh_sb, dh_st);
        a.dg = walk(dg, dg_sb, dg_st);
        a.dx = walk(dx, dx_sb, dx_st);
        rc = check_walk(what, "g", a.g, dtype, B, T, D, false);
        if (!rc) rc = check_walk(what, "x", a.x, dtype, B, T, D, false);
        if (!rc && dh) rc = check_walk(what, "dh", a.dh, dtype, B, T, D, false);
        if (!rc) rc = check_walk(what, "dg", a.dg, dtype, B, T, D, true);
        if (!rc) rc = check_walk(what, "dx", a.dx, dtype, B, T, D, true);
        if (rc) return rc;
    }
    a.carry = const_cast<float *>(carry);
    a.dlast = dlast;
    a.dh0 = dh0;
    a.lens = lens;
    a.wide_lens = wide_lens;
    a.B = (int)B;
    a.T = (int)T;
    a.D = (int)D;
    pb::DeviceInfo dev;
    rc = pb::device_info(&dev);
    if (rc) return rc;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool wide = D % (16 / (int64_t)bytes_of(dtype)) == 0 && wide_rows(a.g, dtype) && wide_rows(a.x, dtype) &&
                      wide_rows(a.dh, dtype) && wide_rows(a.dg, dtype) && wide_rows(a.dx, dtype);
    const bool vec = D % 2 == 0 && words(a.g, dtype) && words(a.x, dtype) && words(a.dh, dtype) &&
                     words(a.dg, dtype) && words(a.dx, dtype);
    if (dtype == PARPY_B200_F32)
        return wide ? run_backward<float, kWide>(a, dev, s) : run_backward<float, kWords>(a, dev, s);
    if (dtype == PARPY_B200_BF16)
        return wide ? run_backward<__nv_bfloat16, kWide>(a, dev, s)
               : vec ? run_backward<__nv_bfloat16, kWords>(a, dev, s)
                     : run_backward<__nv_bfloat16, kElements>(a, dev, s);
    return wide ? run_backward<__half, kWide>(a, dev, s)
           : vec ? run_backward<__half, kWords>(a, dev, s)
                 : run_backward<__half, kElements>(a, dev, s);
}

int32_t parpy_b200_gated_step(int32_t dtype, int64_t N, int64_t D, const void *g, int64_t ldg, const void *x,
                              int64_t ldx, const float *state, void *h, int64_t ldh, float *last, void *stream) {
    const char *what = "gated_step";
    int32_t rc = check_scan(what, dtype, N, 1, D);
    if (rc || N == 0 || D == 0) return rc;
    PB_REQUIRE(g && x && state && h && last, "%s: null pointer", what);
    PB_REQUIRE(reinterpret_cast<uintptr_t>(g) % bytes_of(dtype) == 0 && reinterpret_cast<uintptr_t>(x) % bytes_of(dtype) == 0 &&
                   reinterpret_cast<uintptr_t>(h) % bytes_of(dtype) == 0, "%s: misaligned array", what);
    PB_REQUIRE(ldg >= 0 && ldx >= 0 && (ldh >= D || N <= 1), "%s: rows of h overlap, or a negative pitch", what);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (dtype == PARPY_B200_F32) return run_step<float>(g, x, state, h, last, N, D, ldg, ldx, ldh, s);
    if (dtype == PARPY_B200_BF16) return run_step<__nv_bfloat16>(g, x, state, h, last, N, D, ldg, ldx, ldh, s);
    return run_step<__half>(g, x, state, h, last, N, D, ldg, ldx, ldh, s);
}

}  // extern "C"
