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

// ---- four bytes of a row: the channels of one lane ------------------------------------------------------
template <typename T>
struct Word;
template <>
struct Word<float> {
    static constexpr int CH = 1;
    __device__ static void unpack(unsigned w, float (&v)[1]) { v[0] = __uint_as_float(w); }
    __device__ static unsigned pack(const float (&v)[1]) { return __float_as_uint(v[0]); }
};
template <>
struct Word<__nv_bfloat16> {
    static constexpr int CH = 2;
    __device__ static void unpack(unsigned w, float (&v)[2]) {
        v[0] = __uint_as_float(w << 16);
        v[1] = __uint_as_float(w & 0xffff0000u);
    }
    __device__ static unsigned pack(const float (&v)[2]) {
        const __nv_bfloat162 p = __floats2bfloat162_rn(v[0], v[1]);
        return *reinterpret_cast<const unsigned *>(&p);
    }
};
template <>
struct Word<__half> {
    static constexpr int CH = 2;
    __device__ static void unpack(unsigned w, float (&v)[2]) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w));
        v[0] = f.x;
        v[1] = f.y;
    }
    __device__ static unsigned pack(const float (&v)[2]) {
        const __half2 p = __floats2half2_rn(v[0], v[1]);
        return *reinterpret_cast<const unsigned *>(&p);
    }
};

// A lane's channels within a block of 32 CH: neighbours where rows allow 4-byte access (VEC), 32 apart where they
// start at any element.
template <typename T, bool VEC>
__device__ __forceinline__ int channel(int lane, int j) {
    return VEC ? lane * Word<T>::CH + j : lane + 32 * j;
}
template <typename T, bool VEC>
__device__ __forceinline__ unsigned load_word(const T *p, int lane, int n) {
    if constexpr (VEC) {
        unsigned w = 0;
        if (lane * Word<T>::CH < n)
            asm volatile("ld.global.L1::no_allocate.u32 %0, [%1];" : "=r"(w) : "l"(p + lane * Word<T>::CH));
        return w;
    } else {
        const unsigned short *q = reinterpret_cast<const unsigned short *>(p);
        const unsigned lo = lane < n ? q[lane] : 0, hi = lane + 32 < n ? q[lane + 32] : 0;
        return lo | (hi << 16);
    }
}
template <typename T, bool VEC>
__device__ __forceinline__ void store_word(T *p, int lane, int n, unsigned w) {
    if constexpr (VEC) {
        if (lane * Word<T>::CH < n) __stcs(reinterpret_cast<unsigned *>(p + lane * Word<T>::CH), w);
    } else {
        unsigned short *q = reinterpret_cast<unsigned short *>(p);
        if (lane < n) q[lane] = (unsigned short)w;
        if (lane + 32 < n) q[lane + 32] = (unsigned short)(w >> 16);
    }
}

// f = sigmoid(g) and 1 - f, each to its own relative precision: with e = exp(-g), f = 1 / (1 + e) and 1 - f = e f.
// The exponent is capped so that e f stays 1 for g far below zero; a NaN passes.
__device__ __forceinline__ void gate(float g, float &f, float &keep) {
    float t = -1.4426950408889634f * g;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(t) : "f"(t), "f"(126.0f));
    const float e = pb::ex2_approx(t);
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(f) : "f"(1.0f + e));
    keep = e * f;
}

__device__ __forceinline__ void st_cluster_f32x2(unsigned addr, float a, float b) {
    asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(addr), "f"(a), "f"(b) : "memory");
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

// grid.x = sequences x channel blocks x C; a cluster of C CTAs works on C tiles of one sequence at a time.
template <typename T, bool VEC, int S, int W>
__global__ void __launch_bounds__(W * 32, 2) scan_forward(const ScanArgs a, const int C) {
    static_assert(S * W == kTile, "one stored state per tile");
    constexpr int CH = Word<T>::CH;
    __shared__ float2 s_run[2][W][CH][32];
    __shared__ float2 s_tile[2][kMaxRanks][CH][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int rank = C > 1 ? (int)cluster_ctarank() : 0;
    const int item = blockIdx.x / C, b = item / a.blocks, c0 = (item % a.blocks) * 32 * CH;
    const int n = min(a.D - c0, 32 * CH), len = length_of(a, b);
    const T *g = start_of<T>(a.g, b, c0), *x = start_of<T>(a.x, b, c0);
    T *h = start_of<T>(a.h, b, c0);

    float state[CH];      // entering the cluster's tiles of this round
#pragma unroll
    for (int j = 0; j < CH; ++j) {
        const int c = channel<T, VEC>(lane, j);
        state[j] = a.h0 && c < n ? a.h0[(long long)b * a.D + c0 + c] : 0.0f;
    }
    if (C > 1) {          // every CTA runs before the first store into its shared memory
        cluster_arrive();
        cluster_wait();
    }
    const int stride = C * kTile, rounds = (len + stride - 1) / stride;
    int t0 = rank * kTile + warp * S;
    unsigned gw[S], xw[S];
    auto fetch = [&](int t) {
#pragma unroll
        for (int s = 0; s < S; ++s) {
            gw[s] = xw[s] = 0;
            if (t + s < len) {
                gw[s] = load_word<T, VEC>(g + (t + s) * a.g.st, lane, n);
                xw[s] = load_word<T, VEC>(x + (t + s) * a.x.st, lane, n);
            }
        }
    };
    fetch(t0);
    for (int round = 0; round < rounds; ++round, t0 += stride) {
        const int par = round & 1;
        float f[S][CH], u[S][CH], A[CH], Bv[CH];
#pragma unroll
        for (int j = 0; j < CH; ++j) {
            A[j] = 1.0f;
            Bv[j] = 0.0f;
        }
#pragma unroll
        for (int s = 0; s < S; ++s) {
            float gv[CH], xv[CH];
            Word<T>::unpack(gw[s], gv);
            Word<T>::unpack(xw[s], xv);
            const bool in = t0 + s < len;
#pragma unroll
            for (int j = 0; j < CH; ++j) {
                float keep;
                gate(gv[j], f[s][j], keep);
                u[s][j] = keep * xv[j];
                if (!in) {            // behind the end the state is held
                    f[s][j] = 1.0f;
                    u[s][j] = 0.0f;
                }
                A[j] *= f[s][j];
                Bv[j] = fmaf(f[s][j], Bv[j], u[s][j]);
            }
        }
        if (round + 1 < rounds) fetch(t0 + stride);
#pragma unroll
        for (int j = 0; j < CH; ++j) s_run[par][warp][j][lane] = make_float2(A[j], Bv[j]);
        __syncthreads();
        float pa[CH], pb[CH], ta[CH], tb[CH];    // runs before this warp's, and the whole tile
#pragma unroll
        for (int j = 0; j < CH; ++j) {
            ta[j] = 1.0f;
            tb[j] = 0.0f;
#pragma unroll
            for (int w = 0; w < W; ++w) {
                if (w == warp) {
                    pa[j] = ta[j];
                    pb[j] = tb[j];
                }
                const float2 r = s_run[par][w][j][lane];
                ta[j] *= r.x;
                tb[j] = fmaf(r.x, tb[j], r.y);
            }
        }
        float in[CH];
        if (C > 1) {
            if (warp == 0) {
                for (int r = 0; r < C; ++r)
#pragma unroll
                    for (int j = 0; j < CH; ++j)
                        st_cluster_f32x2(map_to_rank(smem_u32(&s_tile[par][rank][j][lane]), r), ta[j], tb[j]);
            }
            cluster_arrive();
            cluster_wait();
#pragma unroll
            for (int j = 0; j < CH; ++j) {
                for (int r = 0; r < C; ++r) {
                    if (r == rank) in[j] = state[j];
                    const float2 v = s_tile[par][r][j][lane];
                    state[j] = fmaf(v.x, state[j], v.y);
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < CH; ++j) {
                in[j] = state[j];
                state[j] = fmaf(ta[j], state[j], tb[j]);
            }
        }
        const int tile = round * C + rank;
        if (a.carry && warp == 0 && tile * kTile < len) {
            const long long at = ((long long)b * ((a.T + kTile - 1) / kTile) + tile) * a.D + c0;
#pragma unroll
            for (int j = 0; j < CH; ++j)
                if (channel<T, VEC>(lane, j) < n) a.carry[at + channel<T, VEC>(lane, j)] = in[j];
        }
        float v[CH];
#pragma unroll
        for (int j = 0; j < CH; ++j) v[j] = fmaf(pa[j], in[j], pb[j]);
#pragma unroll
        for (int s = 0; s < S; ++s) {
            const bool alive = t0 + s < len;
#pragma unroll
            for (int j = 0; j < CH; ++j) v[j] = fmaf(f[s][j], v[j], u[s][j]);
            if (t0 + s < a.T) store_word<T, VEC>(h + (t0 + s) * a.h.st, lane, n, alive ? Word<T>::pack(v) : 0u);
        }
    }
    for (; t0 < a.T; t0 += stride)     // behind the end
        for (int s = 0; s < S && t0 + s < a.T; ++s) store_word<T, VEC>(h + (t0 + s) * a.h.st, lane, n, 0u);
    if (a.last && rank == 0 && warp == 0) {
#pragma unroll
        for (int j = 0; j < CH; ++j)
            if (channel<T, VEC>(lane, j) < n) a.last[(long long)b * a.D + c0 + channel<T, VEC>(lane, j)] = state[j];
    }
}

template <typename T, bool VEC, int S, int W>
__global__ void __launch_bounds__(W * 32) scan_backward(const ScanArgs a, const int C) {
    static_assert(S * W == kTile, "one stored state per tile");
    constexpr int CH = Word<T>::CH;
    __shared__ float2 s_run[2][W][CH][32];      // (A, B) of the states
    __shared__ float s_back[2][W][CH][32];      // B of the gradients; their A is the same product
    __shared__ float2 s_tile[2][kMaxRanks][CH][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int rank = C > 1 ? (int)cluster_ctarank() : 0;
    const int item = blockIdx.x / C, b = item / a.blocks, c0 = (item % a.blocks) * 32 * CH;
    const int n = min(a.D - c0, 32 * CH), len = length_of(a, b);
    const T *g = start_of<T>(a.g, b, c0), *x = start_of<T>(a.x, b, c0), *dh = a.dh.p ? start_of<T>(a.dh, b, c0) : nullptr;
    T *dg = start_of<T>(a.dg, b, c0), *dx = start_of<T>(a.dx, b, c0);
    const float *carry = a.carry + (long long)b * ((a.T + kTile - 1) / kTile) * a.D + c0;

    float back[CH];       // c entering the cluster's tiles of this round from behind
#pragma unroll
    for (int j = 0; j < CH; ++j) {
        const int c = channel<T, VEC>(lane, j);
        back[j] = a.dlast && c < n ? a.dlast[(long long)b * a.D + c0 + c] : 0.0f;
    }
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
    float cv[CH];         // the stored state of the tile
    auto fetch = [&](int t, int tile) {
#pragma unroll
        for (int s = 0; s < S; ++s) {
            gw[s] = xw[s] = dw[s] = 0;
            if (t + s < len) {
                gw[s] = load_word<T, VEC>(g + (t + s) * a.g.st, lane, n);
                xw[s] = load_word<T, VEC>(x + (t + s) * a.x.st, lane, n);
                if (dh) dw[s] = load_word<T, VEC>(dh + (t + s) * a.dh.st, lane, n);
            }
        }
#pragma unroll
        for (int j = 0; j < CH; ++j) {
            const int c = channel<T, VEC>(lane, j);
            cv[j] = c < n && tile * kTile < len ? carry[(long long)tile * a.D + c] : 0.0f;
        }
    };
    if (rounds > 0) fetch(t0, (rounds - 1) * C + rank);
    for (int round = rounds - 1; round >= 0; --round, t0 -= stride) {
        const int par = round & 1;
        float f[S][CH], keep[S][CH], xv[S][CH], d[S][CH], hp[CH], A[CH], Bv[CH], Rv[CH];
#pragma unroll
        for (int j = 0; j < CH; ++j) {
            A[j] = 1.0f;
            Bv[j] = Rv[j] = 0.0f;
            hp[j] = cv[j];
        }
#pragma unroll
        for (int s = 0; s < S; ++s) {
            float gv[CH];
            Word<T>::unpack(gw[s], gv);
            Word<T>::unpack(xw[s], xv[s]);
            Word<T>::unpack(dw[s], d[s]);
            const bool in = t0 + s < len;
#pragma unroll
            for (int j = 0; j < CH; ++j) {
                gate(gv[j], f[s][j], keep[s][j]);
                if (!in) {
                    f[s][j] = 1.0f;
                    keep[s][j] = 0.0f;
                }
                A[j] *= f[s][j];
                Bv[j] = fmaf(f[s][j], Bv[j], keep[s][j] * xv[s][j]);
            }
        }
#pragma unroll
        for (int s = S - 1; s >= 0; --s)
#pragma unroll
            for (int j = 0; j < CH; ++j) Rv[j] = f[s][j] * (d[s][j] + Rv[j]);
        if (round > 0) fetch(t0 - stride, (round - 1) * C + rank);
#pragma unroll
        for (int j = 0; j < CH; ++j) {
            s_run[par][warp][j][lane] = make_float2(A[j], Bv[j]);
            s_back[par][warp][j][lane] = Rv[j];
        }
        __syncthreads();
        float qa[CH], qb[CH];      // the runs behind this warp's, then the whole tile
        float ra[CH], rb[CH];
#pragma unroll
        for (int j = 0; j < CH; ++j) {
#pragma unroll
            for (int w = 0; w < W; ++w)
                if (w < warp) {
                    const float2 r = s_run[par][w][j][lane];
                    hp[j] = fmaf(r.x, hp[j], r.y);
                }
            qa[j] = 1.0f;
            qb[j] = 0.0f;
#pragma unroll
            for (int w = W - 1; w >= 0; --w) {
                if (w == warp) {
                    ra[j] = qa[j];
                    rb[j] = qb[j];
                }
                const float aw = s_run[par][w][j][lane].x;
                qa[j] *= aw;
                qb[j] = fmaf(aw, qb[j], s_back[par][w][j][lane]);
            }
        }
        float in[CH];
        if (C > 1) {
            if (warp == 0) {
                for (int r = 0; r < C; ++r)
#pragma unroll
                    for (int j = 0; j < CH; ++j)
                        st_cluster_f32x2(map_to_rank(smem_u32(&s_tile[par][rank][j][lane]), r), qa[j], qb[j]);
            }
            cluster_arrive();
            cluster_wait();
#pragma unroll
            for (int j = 0; j < CH; ++j) {
                for (int r = C - 1; r >= 0; --r) {
                    if (r == rank) in[j] = back[j];
                    const float2 v = s_tile[par][r][j][lane];
                    back[j] = fmaf(v.x, back[j], v.y);
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < CH; ++j) {
                in[j] = back[j];
                back[j] = fmaf(qa[j], back[j], qb[j]);
            }
        }
        // the states before each step, then backwards through the run
        float before[S][CH], c[CH];
#pragma unroll
        for (int s = 0; s < S; ++s)
#pragma unroll
            for (int j = 0; j < CH; ++j) {
                before[s][j] = hp[j];
                hp[j] = fmaf(f[s][j], hp[j], keep[s][j] * xv[s][j]);
            }
#pragma unroll
        for (int j = 0; j < CH; ++j) c[j] = fmaf(ra[j], in[j], rb[j]);
#pragma unroll
        for (int s = S - 1; s >= 0; --s) {
            float gx[CH], gg[CH];
#pragma unroll
            for (int j = 0; j < CH; ++j) {
                const float r = d[s][j] + c[j];
                gx[j] = keep[s][j] * r;
                gg[j] = gx[j] * f[s][j] * (before[s][j] - xv[s][j]);
                c[j] = f[s][j] * r;
            }
            if (t0 + s < a.T) {
                const bool alive = t0 + s < len;
                store_word<T, VEC>(dx + (t0 + s) * a.dx.st, lane, n, alive ? Word<T>::pack(gx) : 0u);
                store_word<T, VEC>(dg + (t0 + s) * a.dg.st, lane, n, alive ? Word<T>::pack(gg) : 0u);
            }
        }
    }
    if (a.dh0 && rank == 0 && warp == 0) {
#pragma unroll
        for (int j = 0; j < CH; ++j)
            if (channel<T, VEC>(lane, j) < n) a.dh0[(long long)b * a.D + c0 + channel<T, VEC>(lane, j)] = back[j];
    }
}

// ---- one token for every row: 8 channels per thread where the rows allow 16-byte access, else one ------------
template <typename T, int VN>
__global__ void __launch_bounds__(256) scan_step(const T *g, const T *x, const float *state, T *h, float *last,
                                                 long long N, int D, long long ldg, long long ldx, long long ldh) {
    const int per = D / VN;
    const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= N * per) return;
    const long long row = i / per, at = row * D + (i % per) * VN;
    const int c = (int)(i % per) * VN;
    __align__(16) T gv[VN];
    __align__(16) T xv[VN];
    __align__(16) T hv[VN];
    __align__(16) float sv[VN];
    __align__(16) float lv[VN];
    if constexpr (VN == 1) {
        gv[0] = g[row * ldg + c];
        xv[0] = x[row * ldx + c];
        sv[0] = state[at];
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
    for (int k = 0; k < VN; ++k) {
        float f, keep;
        gate((float)gv[k], f, keep);
        lv[k] = fmaf(f, sv[k], keep * (float)xv[k]);
        hv[k] = (T)lv[k];
    }
    if constexpr (VN == 1) {
        h[row * ldh + c] = hv[0];
        last[at] = lv[0];
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

bool words(const Walk &w, int32_t dtype) {
    return !w.p || dtype == PARPY_B200_F32 ||
           (reinterpret_cast<uintptr_t>(w.p) % 4 == 0 && w.sb % 2 == 0 && w.st % 2 == 0);
}

template <typename K>
int32_t launch_scan(K kernel, const char *what, ScanArgs &a, int channels, int threads, int C, cudaStream_t stream) {
    a.blocks = (a.D + channels - 1) / channels;
    const long long grid = (long long)a.B * a.blocks * C;
    PB_REQUIRE(grid <= INT_MAX, "%s: shape (%d, %d, %d) needs too many blocks", what, a.B, a.T, a.D);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3((unsigned)threads);
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

int cluster_of(const ScanArgs &a, int channels, int sms) {
    const long long blocks = (long long)a.B * ((a.D + channels - 1) / channels);
    int C = 1;
    while (C < kMaxRanks && blocks * C < 2LL * sms && (long long)C * kTile < a.T) C *= 2;
    return C;
}

template <typename T, bool VEC>
int32_t run_forward(ScanArgs &a, const pb::DeviceInfo &dev, cudaStream_t stream) {
    constexpr int channels = 32 * Word<T>::CH;
    return launch_scan(scan_forward<T, VEC, 16, 8>, "gated_scan", a, channels, 256, cluster_of(a, channels, dev.sm_count),
                       stream);
}
template <typename T, bool VEC>
int32_t run_backward(ScanArgs &a, const pb::DeviceInfo &dev, cudaStream_t stream) {
    constexpr int channels = 32 * Word<T>::CH;
    return launch_scan(scan_backward<T, VEC, 8, 16>, "gated_scan_grad", a, channels, 512,
                       cluster_of(a, channels, dev.sm_count), stream);
}

template <typename T>
int32_t run_step(const void *g, const void *x, const float *state, void *h, float *last, int64_t N, int64_t D,
                 int64_t ldg, int64_t ldx, int64_t ldh, cudaStream_t stream) {
    constexpr int E = 16 / sizeof(T);
    const bool wide = D % 8 == 0 && ldg % E == 0 && ldx % E == 0 && ldh % E == 0 && pb::aligned16(g) &&
                      pb::aligned16(x) && pb::aligned16(state) && pb::aligned16(h) && pb::aligned16(last);
    const long long work = N * (wide ? D / 8 : D), blocks = (work + 255) / 256;
    PB_REQUIRE(blocks <= INT_MAX, "gated_step: shape (%lld, %lld) is too large", (long long)N, (long long)D);
    const T *gt = static_cast<const T *>(g), *xt = static_cast<const T *>(x);
    if (wide) scan_step<T, 8><<<(unsigned)blocks, 256, 0, stream>>>(gt, xt, state, static_cast<T *>(h), last, N, (int)D, ldg, ldx, ldh);
    else scan_step<T, 1><<<(unsigned)blocks, 256, 0, stream>>>(gt, xt, state, static_cast<T *>(h), last, N, (int)D, ldg, ldx, ldh);
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
    if (dtype == PARPY_B200_F32) return run_forward<float, true>(a, dev, s);
    const bool vec = D % 2 == 0 && words(a.g, dtype) && words(a.x, dtype) && words(a.h, dtype);
    if (dtype == PARPY_B200_BF16)
        return vec ? run_forward<__nv_bfloat16, true>(a, dev, s) : run_forward<__nv_bfloat16, false>(a, dev, s);
    return vec ? run_forward<__half, true>(a, dev, s) : run_forward<__half, false>(a, dev, s);
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
    if (dtype == PARPY_B200_F32) return run_backward<float, true>(a, dev, s);
    const bool vec = D % 2 == 0 && words(a.g, dtype) && words(a.x, dtype) && words(a.dh, dtype) &&
                     words(a.dg, dtype) && words(a.dx, dtype);
    if (dtype == PARPY_B200_BF16)
        return vec ? run_backward<__nv_bfloat16, true>(a, dev, s) : run_backward<__nv_bfloat16, false>(a, dev, s);
    return vec ? run_backward<__half, true>(a, dev, s) : run_backward<__half, false>(a, dev, s);
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
