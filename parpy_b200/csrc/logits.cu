// Operators on rows of vocabulary logits for sm_100a: log-probabilities of given tokens with the row's entropy and
// its K best alternatives, distillation from a teacher's K best logits, and both gradients.
//
// With z = x / temperature and a row's log-sum-exp lse = log sum_j exp(z_j), p_j = exp(z_j - lse):
//
//   token_logprobs   logp = z_t - lse,  entropy = -sum_j p_j log p_j,  the K largest x_j (ties to the lowest column)
//     gradient       dx_j = (dlogp ([j = t] - p_j) - dentropy p_j (log p_j + entropy)) / temperature
//   distill_topk     loss = sum_k q_k (log q_k - (z_{i_k} - lse)), q the teacher's renormalised probabilities; with a
//                    tail q_k = exp(v_k) and one more term for the bucket of all other columns:
//                    left (log left - (rest - lse)), left = 1 - sum q, rest = log sum over the other columns exp(z)
//     gradient       dz_j = W p_j - q_j [j listed] - left exp(z_j - rest) [j not listed],  W = sum q (+ left)
//
// The forward kernels read every logit once: a thread keeps a reference value `ref`, S = sum exp2((x - ref) c) and
// E = sum exp2(t) t with t = (x - ref) c, c = log2(e) / temperature, and moves `ref` up only when a value exceeds it
// by more than 8 powers of two (floating-point sums lose nothing by a reference that is not the exact maximum). x - ref
// is formed before the scaling, so that rows of large offsets or of the type's lowest value stay exact. The triples of
// threads, warps and the CTAs of a cluster are joined by the same rescaling.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <cfloat>
#include <climits>
#include <cmath>

#include "../../include/parpy_b200.h"
#include "common.cuh"
#include "cluster.cuh"

namespace {

constexpr double kLn2 = 0.693147180559945309417;
constexpr double kLog2eD = 1.44269504088896340736;
constexpr int kTopMax = 128;         // alternatives a row can ask for
constexpr int kListMax = 1024;       // entries of a teacher's list
constexpr int kGroups = 128;         // most thread groups whose best values give the first bound
constexpr int kMaxCluster = 8;

using u64 = unsigned long long;

// ---- element types: 32 bytes of a row, the widest load there is ------------------------------------------
struct Vec {
    unsigned w[8];
};

template <typename T>
struct Elem;
template <>
struct Elem<float> {
    static constexpr int VE = 8;
    static constexpr unsigned kFill = 0xff800000u;   // -inf
    __device__ static float to_float(float v) { return v; }
    __device__ static float from_float(float v) { return v; }
    // elements 2 i and 2 i + 1
    __device__ static void pair(const Vec &r, int i, float &a, float &b) {
        a = __uint_as_float(r.w[2 * i]);
        b = __uint_as_float(r.w[2 * i + 1]);
    }
    __device__ static void set_pair(Vec &r, int i, float a, float b) {
        r.w[2 * i] = __float_as_uint(a);
        r.w[2 * i + 1] = __float_as_uint(b);
    }
    __device__ static float vmax(const Vec &r) {
        float m = __uint_as_float(r.w[0]);
#pragma unroll
        for (int i = 1; i < 8; ++i) m = fmaxf(m, __uint_as_float(r.w[i]));
        return m;
    }
};
template <>
struct Elem<__nv_bfloat16> {
    static constexpr int VE = 16;
    static constexpr unsigned kFill = 0xff80ff80u;
    __device__ static float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
    __device__ static __nv_bfloat16 from_float(float v) { return __float2bfloat16_rn(v); }
    __device__ static void pair(const Vec &r, int i, float &a, float &b) {
        a = __uint_as_float(r.w[i] << 16);
        b = __uint_as_float(r.w[i] & 0xffff0000u);
    }
    __device__ static void set_pair(Vec &r, int i, float a, float b) {
        const __nv_bfloat162 p = __floats2bfloat162_rn(a, b);
        r.w[i] = *reinterpret_cast<const unsigned *>(&p);
    }
    __device__ static float vmax(const Vec &r) {
        const __nv_bfloat162 *p = reinterpret_cast<const __nv_bfloat162 *>(r.w);
        const __nv_bfloat162 m = __hmax2(__hmax2(__hmax2(p[0], p[1]), __hmax2(p[2], p[3])),
                                         __hmax2(__hmax2(p[4], p[5]), __hmax2(p[6], p[7])));
        return fmaxf(__low2float(m), __high2float(m));
    }
};
template <>
struct Elem<__half> {
    static constexpr int VE = 16;
    static constexpr unsigned kFill = 0xfc00fc00u;
    __device__ static float to_float(__half v) { return __half2float(v); }
    __device__ static __half from_float(float v) { return __float2half_rn(v); }
    __device__ static void pair(const Vec &r, int i, float &a, float &b) {
        const float2 f = __half22float2(reinterpret_cast<const __half2 *>(r.w)[i]);
        a = f.x;
        b = f.y;
    }
    __device__ static void set_pair(Vec &r, int i, float a, float b) {
        const __half2 p = __floats2half2_rn(a, b);
        r.w[i] = *reinterpret_cast<const unsigned *>(&p);
    }
    __device__ static float vmax(const Vec &r) {
        const __half2 *p = reinterpret_cast<const __half2 *>(r.w);
        const __half2 m = __hmax2(__hmax2(__hmax2(p[0], p[1]), __hmax2(p[2], p[3])),
                                  __hmax2(__hmax2(p[4], p[5]), __hmax2(p[6], p[7])));
        return fmaxf(__low2float(m), __high2float(m));
    }
};
template <typename T>
__device__ __forceinline__ float element(const Vec &r, int i) {
    float a, b;
    Elem<T>::pair(r, i >> 1, a, b);
    return i & 1 ? b : a;
}

// Rounding can take a probability a little past 1: its logarithm, and an entropy, stop at 0. A NaN stays.
__device__ __forceinline__ float at_most_zero(double v) { return v > 0.0 ? 0.0f : (float)v; }
__device__ __forceinline__ float at_least_zero(double v) { return v < 0.0 ? 0.0f : (float)v; }

// ---- packed fp32 pairs (two lanes of one 64-bit register, one instruction each) ------------------------
__device__ __forceinline__ u64 pack2(float a, float b) {
    u64 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpack2(u64 p, float &a, float &b) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p));
}
__device__ __forceinline__ u64 add2(u64 a, u64 b) {
    u64 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ u64 mul2(u64 a, u64 b) {
    u64 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ u64 fma2(u64 a, u64 b, u64 c) {
    u64 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

// ---- a row as 32-byte vectors -----------------------------------------------------------------------------
// Vector v of a row holds the columns [v VE - mis, v VE - mis + VE), where mis is the number of elements between the
// last 32-byte boundary and the row's start: rows may start at any element. Only the first and the last vector can
// be partial; they are fetched element by element and filled up with -inf, so nothing outside the row is read.
template <typename T>
struct Row {
    const T *p;
    int M, mis, nvec, v0, v1;   // vectors [v0, v1) are whole
    __device__ Row(const T *row, int m) : p(row), M(m) {
        constexpr int VE = Elem<T>::VE;
        mis = (int)((reinterpret_cast<uintptr_t>(row) & 31u) / sizeof(T));
        nvec = (int)(((long long)M + mis + VE - 1) / VE);
        v0 = mis ? 1 : 0;
        v1 = (int)(((long long)M + mis) / VE);
    }
    __device__ bool whole(int v) const { return v >= v0 && v < v1; }
    __device__ bool tail() const { return nvec > v1 && (nvec > 1 || !v0); }   // vector v1 is partial and not the first
    __device__ int first(int v) const { return v * Elem<T>::VE - mis; }
    __device__ const T *at(int v) const { return p + (long long)v * Elem<T>::VE - mis; }
    __device__ Vec edge(int v) const {
        constexpr int VE = Elem<T>::VE;
        Vec r;
#pragma unroll
        for (int i = 0; i < 8; ++i) r.w[i] = Elem<T>::kFill;
        T *e = reinterpret_cast<T *>(r.w);
        const int c0 = first(v);
#pragma unroll
        for (int i = 0; i < VE; ++i)
            if (c0 + i >= 0 && c0 + i < M) e[i] = p[c0 + i];
        return r;
    }
};

// The forward pass may read through the non-coherent path; a gradient written over its own logits may not.
__device__ __forceinline__ Vec ld_const(const void *p) {
    Vec r;
    asm volatile("ld.global.nc.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r.w[0]), "=r"(r.w[1]), "=r"(r.w[2]), "=r"(r.w[3]), "=r"(r.w[4]), "=r"(r.w[5]), "=r"(r.w[6]),
                   "=r"(r.w[7])
                 : "l"(p));
    return r;
}
__device__ __forceinline__ Vec ld_stream(const void *p) {
    Vec r;
    asm volatile("ld.global.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r.w[0]), "=r"(r.w[1]), "=r"(r.w[2]), "=r"(r.w[3]), "=r"(r.w[4]), "=r"(r.w[5]), "=r"(r.w[6]),
                   "=r"(r.w[7])
                 : "l"(p)
                 : "memory");
    return r;
}
__device__ __forceinline__ void st_stream(void *p, const Vec &r) {
    asm volatile("st.global.cs.v8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::"r"(r.w[0]), "r"(r.w[1]), "r"(r.w[2]),
                 "r"(r.w[3]), "r"(r.w[4]), "r"(r.w[5]), "r"(r.w[6]), "r"(r.w[7]), "l"(p)
                 : "memory");
}

// ---- the order of (value, lowest column) as one 64-bit key: larger is better, 0 is "none" ------------------
__device__ __forceinline__ unsigned order_of(float f) {
    const unsigned u = __float_as_uint(f + 0.0f);   // -0 counts as 0
    return u ^ ((unsigned)((int)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(unsigned o) {
    return __uint_as_float((o & 0x80000000u) ? o ^ 0x80000000u : ~o);
}
__device__ __forceinline__ u64 key_of(float f, int column) {
    return ((u64)order_of(f) << 32) | (0xffffffffu - (unsigned)column);
}

// ---- running softmax sums of one thread ------------------------------------------------------------------------
struct Sums {
    float ref, S, E;   // S = 0: nothing finite seen
};

template <bool ENT>
__device__ __forceinline__ Sums join(Sums a, float R, float c) {
    // the sums of `a` relative to the reference R >= a.ref
    const float r = a.S == 0.0f ? 0.0f : pb::ex2_approx((a.ref - R) * c);
    Sums o;
    o.ref = R;
    o.S = a.S == 0.0f ? 0.0f : a.S * r;
    o.E = 0.0f;
    if (ENT) o.E = a.S == 0.0f ? 0.0f : r * (a.E + fmaxf((a.ref - R) * c, -1e30f) * a.S);
    return o;
}
__device__ __forceinline__ float ref_of(const Sums &a) { return a.S == 0.0f ? -INFINITY : a.ref; }

template <bool ENT>
__device__ __forceinline__ Sums warp_join(Sums a, float c) {
    const float R = pb::warp_max(ref_of(a));
    Sums o = join<ENT>(a, R, c);
    o.S = pb::warp_sum(o.S);
    if (ENT) o.E = pb::warp_sum(o.E);
    return o;
}

enum ListMode { kNone = 0, kRenorm = 1, kTail = 2 };

struct RowArgs {
    const void *x;
    long long ldx, N;
    int M, K;
    double inv_t;            // 1 / temperature
    const void *tokens;      // token_logprobs: [N] or null
    const void *index;       // distill: [N, K]
    const void *values;      // distill: [N, K]
    int wide, value_type;    // 64-bit tokens / index; dtype of values
    float *logp, *lse, *entropy, *top;   // top_logp
    void *at;                // top_index
    int at_wide;
    float *loss, *rest;
};

__device__ __forceinline__ long long load_index(const void *p, long long i, int wide) {
    return wide ? static_cast<const long long *>(p)[i] : (long long)static_cast<const int *>(p)[i];
}
__device__ __forceinline__ float load_value(const void *p, long long i, int type) {
    return type == PARPY_B200_F32    ? static_cast<const float *>(p)[i]
           : type == PARPY_B200_BF16 ? __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i])
                                     : __half2float(static_cast<const __half *>(p)[i]);
}

// A teacher's list in shared memory. Negative columns and second mentions of a column are not used; a column past the
// vocabulary makes the row `bad`.
struct List {
    int col[kListMax];
    unsigned char used[kListMax];
    float v[kListMax], x[kListMax];
    int bad;
};

// Every thread of the CTA takes part. Second mentions are found by whole warps: an entry against the lanes' share of
// the entries before it.
template <typename T>
__device__ void load_list(List &l, const RowArgs &a, long long row, const T *xr) {
    const int lane = threadIdx.x & 31;
    if (threadIdx.x == 0) l.bad = 0;
    __syncthreads();
    for (int k = threadIdx.x; k < a.K; k += blockDim.x) {
        const long long i = load_index(a.index, row * a.K + k, a.wide);
        const bool in = i >= 0 && i < a.M;
        if (i >= a.M) l.bad = 1;
        l.col[k] = in ? (int)i : -1;
        l.v[k] = load_value(a.values, row * a.K + k, a.value_type);
        l.x[k] = in ? Elem<T>::to_float(xr[i]) : 0.0f;
    }
    __syncthreads();
    for (int k = threadIdx.x >> 5; k < a.K; k += blockDim.x >> 5) {
        const int c = l.col[k];
        bool seen = false;
        for (int j = lane; j < k; j += 32) seen |= l.col[j] == c;
        const bool again = __any_sync(0xffffffffu, seen);
        if (lane == 0) l.used[k] = c >= 0 && !again;
    }
    __syncthreads();
}

// The logarithm of a sum of exp(z) over some columns, as its reference logit and what is left: ref / temperature + log. A
// logit is compared with it through the difference to ref, so that a row's common offset (a mask of the type's lowest value
// over every column has 3.4e38) costs nothing. log = -inf: no column.
struct Mass {
    double ref, log;
    __device__ double value(double inv_t) const { return log == -INFINITY ? log : ref * inv_t + log; }
    // log of exp(x / temperature) relative to the sum
    __device__ double below(float x, double inv_t) const {
        return x == -INFINITY ? (double)x : ((double)x - ref) * inv_t - log;
    }
};
__device__ __forceinline__ Mass join_mass(const Mass &a, const Mass &b, double inv_t) {
    if (a.log == -INFINITY) return b;
    if (b.log == -INFINITY) return a;
    const double ref = fmax(a.ref, b.ref), la = (a.ref - ref) * inv_t + a.log, lb = (b.ref - ref) * inv_t + b.log;
    const double m = fmax(la, lb);
    return {ref, m + log(exp(la - m) + exp(lb - m))};     // NaN stays NaN
}
// The 32-bit output of a sum that exists is finite: it stops at the type's range. A NaN stays.
__device__ __forceinline__ float limited(double v) {
    const float f = (float)v;
    return isinf(f) && !isinf(v) ? copysignf(FLT_MAX, f) : f;
}

// What one warp derives from a list: the teacher's normaliser and mass, the student's listed sum (natural logs).
struct Teacher {
    float vref;       // log q_k = (v_k - vref) - norm: an offset common to the teacher's logits costs nothing
    double norm;
    double mass;      // sum q (before `left`), in 64 bits: 1 - mass is next to a border
    Mass listed;      // log sum over the listed columns exp(z)
    int any;          // entries in use
    __device__ double log_q(float v) const { return ((double)v - (double)vref) - norm; }
};

template <bool TAIL, bool STUDENT>
__device__ Teacher warp_teacher(const List &l, int K, double inv_t) {
    const int lane = threadIdx.x & 31;
    float vm = -INFINITY, xm = -INFINITY;
    int n = 0;
    for (int k = lane; k < K; k += 32)
        if (l.used[k]) {
            vm = fmaxf(vm, l.v[k]);
            xm = fmaxf(xm, l.x[k]);
            ++n;
        }
    if (!TAIL) vm = pb::warp_max(vm);
    if (STUDENT) xm = pb::warp_max(xm);
    const float vref = isinf(vm) ? 0.0f : vm, xref = isinf(xm) ? 0.0f : xm;
    double sv = 0.0, sx = 0.0;
    for (int k = lane; k < K; k += 32)
        if (l.used[k]) {
            sv += TAIL ? exp((double)l.v[k]) : (double)expf(l.v[k] - vref);
            if (STUDENT) sx += (double)expf((float)(((double)l.x[k] - (double)xref) * inv_t));
        }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        sv += __shfl_xor_sync(0xffffffffu, sv, o);
        if (STUDENT) sx += __shfl_xor_sync(0xffffffffu, sx, o);
        n += __shfl_xor_sync(0xffffffffu, n, o);
    }
    Teacher t;
    t.any = n;
    t.vref = TAIL ? 0.0f : vref;
    t.norm = TAIL || sv == 0.0 ? 0.0 : log(sv);      // no entry with mass: every q is exp(-inf) = 0
    t.mass = !isfinite(sv) ? (double)NAN : TAIL ? sv : sv == 0.0 ? 0.0 : 1.0;
    // a sum that is not finite holds a NaN or +inf (finite columns are taken relative to their largest): the row is broken
    t.listed = {(double)xref, !STUDENT || sx == 0.0 ? -INFINITY : isfinite(sx) ? log(sx) : NAN};
    return t;
}

// mass of the bucket of all other columns: none where every column is listed
__device__ __forceinline__ double left_of(const Teacher &t, int M) {
    const double left = 1.0 - t.mass;
    return t.any >= M || left < 0.0 ? 0.0 : left;
}

// Shared memory of the forward kernel. Selection and list parts exist only where they are used.
template <int THREADS, bool TOP>
struct TopSmem {};
template <int THREADS>
struct TopSmem<THREADS, true> {
    // a warp that has a row to itself is one of 32 on its SM, and never in a cluster
    static constexpr int kCand = THREADS == 32 ? 128 : 512;
    u64 group[kGroups];
    u64 cand[kCand];
    u64 merge[THREADS == 32 ? 1 : kMaxCluster * kTopMax];
    int sel[THREADS];
    u64 tau;
    int nsel, ncand;
};
template <int THREADS, int LIST>
struct ListSmem {};
template <int THREADS>
struct ListSmem<THREADS, kRenorm> {
    List l;
};
template <int THREADS>
struct ListSmem<THREADS, kTail> {
    List l;
    int head[THREADS];          // a thread's listed columns as a chain: first entry, -1 for none
    short link[kListMax];       // the entry after this one
};

__device__ __forceinline__ void st_cluster_u64(unsigned addr, u64 v) {
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}

// Rows dealt to clusters of C CTAs, vectors of a row round robin to the cluster's threads; with C = 1 as many CTAs as are
// resident take rows in turn, and a row's first vectors and token are asked for before the row before it is joined.
//
// What bounds it: a 16-bit logit costs one exp2 of the special unit (16 a clock and SM: 60 us for 4096 x 65536, of the
// 82 us that reading them takes at the measured copy rate) and 7 to 8 instructions, so memory, special unit and issue are
// all above half; the rest is a row's end, where its CTA loads nothing. Measured: 4096 x 131072 bf16 without entropy
// 194 us (84 % of the copy rate), 4096 x 65536 with entropy 117 us (70 %), 4096 x 131072 with entropy and 20 alternatives
// 256 us (64 %). 128 threads a row keep more rows apart in their phases than 256 (distillation 194 against 211 us); the
// selection's end and a tail's list are shared by 256 (257 against 300 us; 45 against 53 us). The second look of a
// selection costs 16 % of the row's bytes again (1184 rows: 360 MB read for 310), in pieces of 32 bytes of the few threads
// that pass the bound; a row's end keeps one vector a thread in flight. 64 registers leave 28 to 76 bytes of spills in
// most instances with entropy or alternatives (one warp a row with both: 276), none without. Held in registers two
// stages deep: loads that pass through shared memory (cp.async, four stages) cost 218 instead of 209 us, in 16-byte
// pieces of a lane's own vector 322 us; scalar arithmetic instead of packed pairs 132 instead of 120 us.
template <typename T, int THREADS, bool ENT, bool TOP, int LIST>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) row_stats(const RowArgs a, const int C) {
    constexpr int VE = Elem<T>::VE, NW = THREADS / 32, U = ENT && sizeof(T) == 2 ? 1 : 2;
    __shared__ Sums s_warp[NW];
    __shared__ Sums s_rank[kMaxCluster];
    __shared__ double s_ref, s_log;     // the row's reference value and log(S): lse = ref / temperature + log(S)
    __shared__ TopSmem<THREADS, TOP> s_top;
    __shared__ ListSmem<THREADS, LIST> s_list;

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rank = C > 1 ? (int)cluster_ctarank() : 0;
    const long long rows_apart = gridDim.x / C;
    const int total = C * THREADS, me = rank * THREADS + tid;
    const float c = (float)(kLog2eD * a.inv_t);
    const float slack = 8.0f / c;
    const int reach = (U - 1) * total;
    Vec r0[U], r1[U];
    auto load = [&](Vec (&r)[U], const Row<T> &rv, int at) {
#pragma unroll
        for (int u = 0; u < U; ++u) r[u] = ld_const(rv.at(at + u * total));
    };
    auto open_row = [&](long long row) {     // a row's first vectors, before anything else of it
        const Row<T> rv(static_cast<const T *>(a.x) + row * a.ldx, a.M);
        const int v = me < rv.v0 ? me + total : me;
        if (v + reach < rv.v1) load(r0, rv, v);
    };
    open_row(blockIdx.x / C);

    if constexpr (TOP) {
        if (C > 1 && rank == 0)
            for (int i = tid; i < C * a.K; i += THREADS) s_top.merge[i] = 0;
    }
    if (C > 1) cluster_arrive();     // matched before the first store into rank 0's shared memory

    int token_ahead = -1;            // of the thread that writes the results: the next row's token, M for one past the row
    auto look_ahead = [&](long long row) {
        if (LIST == kNone && rank == 0 && tid == 0 && a.tokens && row < a.N)
            token_ahead = (int)pb::ll_max(-1, pb::ll_min(load_index(a.tokens, row, a.wide), a.M));
    };
    look_ahead(blockIdx.x / C);
    // with C > 1 every cluster has one row
    for (long long row = blockIdx.x / C; row < a.N; row += rows_apart) {
        const T *xr = static_cast<const T *>(a.x) + row * a.ldx;
        const Row<T> rv(xr, a.M);
        if constexpr (TOP) {
            if (tid == 0) {
                s_top.tau = 0;
                s_top.nsel = 0;
                s_top.ncand = 0;
            }
        }
        const int token = token_ahead;
        T x_token = Elem<T>::from_float(0.0f);
        if (token >= 0 && token < a.M) x_token = xr[token];
        look_ahead(row + rows_apart);
        int next = INT_MAX;              // tail: the next vector of this thread that holds a listed column
        if constexpr (LIST == kTail) {
            s_list.head[tid] = -1;
            load_list(s_list.l, a, row, xr);
            {
                for (int k = tid; k < a.K; k += THREADS)
                    if (s_list.l.used[k]) {
                        const int owner = ((s_list.l.col[k] + rv.mis) / VE) % total;
                        if (owner / THREADS == rank)
                            s_list.link[k] = (short)atomicExch(&s_list.head[owner % THREADS], k);
                    }
                __syncthreads();
                for (int k = s_list.head[tid]; k >= 0; k = s_list.link[k]) next = min(next, (s_list.l.col[k] + rv.mis) / VE);
            }
        }

        float ref = 0.0f, lim = -INFINITY, best = -INFINITY;
        int best_v = me < rv.nvec ? me : -1;
        u64 S2 = 0, E2 = 0;
        const u64 c2 = pack2(c, c);

        auto take = [&](const Vec &got, int at) {
            Vec r = got;
            if constexpr (LIST == kTail) {
                if (at == next) {         // listed columns are summed apart: read as masked here
                    T *e = reinterpret_cast<T *>(r.w);
                    const unsigned fill = Elem<T>::kFill;
                    next = INT_MAX;
                    for (int k = s_list.head[tid]; k >= 0; k = s_list.link[k]) {
                        const int col = s_list.l.col[k] + rv.mis, w = col / VE;
                        if (w == at) {
#pragma unroll
                            for (int i = 0; i < VE; ++i)
                                if (i == col % VE) e[i] = *reinterpret_cast<const T *>(&fill);
                        } else if (w > at) {
                            next = min(next, w);
                        }
                    }
                }
            }
            const float vm = Elem<T>::vmax(r);
            if constexpr (TOP) {
                if (vm > best) {
                    best = vm;
                    best_v = at;
                }
            }
            if (vm > lim) {
                const bool fresh = lim == -INFINITY;         // nothing summed yet: ref means nothing
                const float sh = fresh ? 0.0f : (ref - vm) * c;
                const float f = fresh ? 0.0f : pb::ex2_approx(sh);
                float s0, s1;
                unpack2(S2, s0, s1);
                if constexpr (ENT) {
                    float e0, e1;
                    unpack2(E2, e0, e1);
                    const float k = fmaxf(sh, -1e30f);
                    E2 = pack2(f * (e0 + k * s0), f * (e1 + k * s1));
                }
                S2 = pack2(f * s0, f * s1);
                ref = vm;
                lim = vm + slack;
            }
            const u64 nref = pack2(-ref, -ref), before = E2;
#pragma unroll
            for (int i = 0; i < VE / 2; ++i) {
                float x0, x1, t0, t1;
                Elem<T>::pair(r, i, x0, x1);
                const u64 t = mul2(add2(pack2(x0, x1), nref), c2);
                unpack2(t, t0, t1);
                const u64 e = pack2(pb::ex2_approx(t0), pb::ex2_approx(t1));
                S2 = add2(S2, e);
                if constexpr (ENT) E2 = fma2(e, t, E2);
            }
            if constexpr (ENT) {
                // a masked column adds 0 times -inf: seen by the NaN it leaves, and added again with t kept finite
                float e0, e1;
                unpack2(E2, e0, e1);
                if (isnan(e0 + e1)) {
                    E2 = before;
#pragma unroll
                    for (int i = 0; i < VE / 2; ++i) {
                        float x0, x1, t0, t1;
                        Elem<T>::pair(r, i, x0, x1);
                        unpack2(mul2(add2(pack2(x0, x1), nref), c2), t0, t1);
                        const u64 e = pack2(pb::ex2_approx(t0), pb::ex2_approx(t1));
                        E2 = fma2(e, pack2(fmaxf(t0, -1e30f), fmaxf(t1, -1e30f)), E2);
                    }
                }
            }
        };
        auto take_all = [&](const Vec (&r)[U], int at) {
#pragma unroll
            for (int u = 0; u < U; ++u) take(r[u], at + u * total);
        };
        if (rv.v0 && me == 0) take(rv.edge(0), 0);
        // at most 2^28 + 1 vectors and 2^12 threads: no sum of them leaves 32 bits
        int v = me < rv.v0 ? me + total : me;
        bool more = v + reach < rv.v1;
        while (more) {                   // the next vectors are on their way while these are summed
            int then = v + U * total;
            more = then + reach < rv.v1;
            if (more) load(r1, rv, then);
            take_all(r0, v);
            v = then;
            if (!more) break;
            then = v + U * total;
            more = then + reach < rv.v1;
            if (more) load(r0, rv, then);
            take_all(r1, v);
            v = then;
        }
        for (; v < rv.v1; v += total) take(ld_const(rv.at(v)), v);
        if (rv.tail() && me == rv.v1 % total) take(rv.edge(rv.v1), rv.v1);

        if (row + rows_apart < a.N) open_row(row + rows_apart);
        if constexpr (LIST == kRenorm) load_list(s_list.l, a, row, xr);      // needed at the end only
        Sums mine;
        {
            float s0, s1, e0, e1;
            unpack2(S2, s0, s1);
            unpack2(E2, e0, e1);
            mine = {ref, s0 + s1, e0 + e1};
        }
        mine = warp_join<ENT>(mine, c);
        if (lane == 0) s_warp[warp] = mine;

        // A group's best value is one of the row's elements, so the K-th best of the groups' values bounds the K-th best
        // element from below: only threads whose own best reaches it can hold one of the K. Few groups rank fast, many bound
        // well: with 64 groups and K = 20 about 24 elements pass, with 128 about 22. A vector's place stands for its
        // columns; the bound takes the vector's last column, so that it never cuts off a tie.
        u64 key = 0, group_key = 0;
        const int sample = max(64, 2 * a.K);
        const int groups = min(a.K <= 32 ? kGroups / 2 : kGroups, THREADS), GL = THREADS / groups, sub = tid & (GL - 1);
        if constexpr (TOP) {
            key = best_v < 0 ? 0 : key_of(best, max(rv.first(best_v), 0));
            group_key = key;
            for (int o = GL >> 1; o > 0; o >>= 1) {
                const u64 other = __shfl_xor_sync(0xffffffffu, group_key, o);
                group_key = other > group_key ? other : group_key;
            }
            if (sub == 0) s_top.group[tid / GL] = group_key;
        }
        __syncthreads();
        if (warp == 0) {
            Sums w = lane < NW ? s_warp[lane] : Sums{0.0f, 0.0f, 0.0f};
            w = warp_join<ENT>(w, c);
            if (lane == 0) s_warp[0] = w;
            __syncwarp();
        }

        int n_local = 0;
        if constexpr (TOP) {
            int above = 0;
#pragma unroll 4
            for (int j = sub; j < groups; j += GL) above += s_top.group[j] > group_key;
            for (int o = GL >> 1; o > 0; o >>= 1) above += __shfl_xor_sync(0xffffffffu, above, o);
            if (sub == 0 && above == a.K - 1 && group_key != 0) s_top.tau = group_key - (VE - 1);
            __syncthreads();
            u64 tau = s_top.tau;
            if (key != 0 && key >= tau) s_top.sel[atomicAdd(&s_top.nsel, 1)] = tid;
            __syncthreads();
            const int nsel = s_top.nsel, per = (rv.nvec + total - 1) / total;
            while (true) {
                for (int it = tid; it < nsel * per; it += THREADS) {
                    const int s = it / per, at = rank * THREADS + s_top.sel[s] + (it - s * per) * total;
                    if (at >= rv.nvec) continue;
                    const Vec r = rv.whole(at) ? ld_const(rv.at(at)) : rv.edge(at);
                    const int c0 = rv.first(at);
                    if (order_of(Elem<T>::vmax(r)) < (unsigned)(tau >> 32)) continue;
#pragma unroll
                    for (int e = 0; e < VE; ++e) {
                        const u64 k = key_of(element<T>(r, e), c0 + e);
                        if (k >= tau && c0 + e >= 0 && c0 + e < a.M) {
                            const int p = atomicAdd(&s_top.ncand, 1);
                            if (p < s_top.kCand) s_top.cand[p] = k;
                        }
                    }
                }
                __syncthreads();
                n_local = s_top.ncand;
                if (n_local <= 2 * sample) break;
                // too many to rank, or more than there is room for: the K-th best of any `sample` of them is a higher bound,
                // which drops sample - K of them at least
                for (int i = tid; i < sample; i += THREADS) {
                    const u64 k = s_top.cand[i];
                    int n = 0;
#pragma unroll 4
                    for (int j = 0; j < sample; ++j) n += s_top.cand[j] > k;
                    if (n == a.K - 1) s_top.tau = k;
                }
                __syncthreads();
                tau = s_top.tau;
                if (tid == 0) s_top.ncand = 0;
                __syncthreads();
            }
        }

        if (C > 1) {
            cluster_wait();
            if (tid == 0) {
                const unsigned to = map_to_rank(smem_u32(&s_rank[rank]), 0);
                st_cluster_f32(to, s_warp[0].ref);
                st_cluster_f32(to + 4, s_warp[0].S);
                st_cluster_f32(to + 8, s_warp[0].E);
            }
            if constexpr (TOP) {
                for (int i = tid; i < n_local; i += THREADS) {
                    const u64 k = s_top.cand[i];
                    int n = 0;
#pragma unroll 4
                    for (int j = 0; j < n_local; ++j) n += s_top.cand[j] > k;
                    if (n < a.K) st_cluster_u64(map_to_rank(smem_u32(&s_top.merge[rank * a.K + n]), 0), k);
                }
            }
            cluster_arrive();
            cluster_wait();
            if (rank != 0) return;
        }

        if (warp == 0) {
            Sums w = C > 1 ? (lane < C ? s_rank[lane] : Sums{0.0f, 0.0f, 0.0f}) : s_warp[0];
            if (C > 1) w = warp_join<ENT>(w, c);
            const float logS = logf(w.S);       // -inf for 0
            const Mass rest{(double)w.ref, (double)logS};
            if constexpr (LIST != kNone) {
                const Teacher t = warp_teacher<LIST == kTail, LIST == kTail>(s_list.l, a.K, a.inv_t);
                const Mass lse = LIST == kTail ? join_mass(rest, t.listed, a.inv_t) : rest;
                double loss = 0.0;
                for (int k = lane; k < a.K; k += 32)
                    if (s_list.l.used[k]) {
                        const double logq = t.log_q(s_list.l.v[k]);
                        const double q = (double)expf((float)logq);
                        if (!(q <= 0.0)) loss += q * (logq - lse.below(s_list.l.x[k], a.inv_t));
                    }
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) loss += __shfl_xor_sync(0xffffffffu, loss, o);
                if (lane == 0) {
                    if (LIST == kTail) {
                        const double left = left_of(t, a.M);
                        if (left > 0.0)
                            loss += left * (log(left) - (rest.log == -INFINITY
                                                             ? rest.log
                                                             : (rest.ref - lse.ref) * a.inv_t + rest.log - lse.log));
                    }
                    if (s_list.l.bad || isnan(t.mass) || isnan(lse.log)) loss = NAN;
                    a.loss[row] = (float)loss;
                    a.lse[row] = limited(lse.value(a.inv_t));
                    if (a.rest) a.rest[row] = limited(rest.value(a.inv_t));
                }
            } else if (lane == 0) {
                a.lse[row] = limited(rest.value(a.inv_t));
                const float x = Elem<T>::to_float(x_token);
                if (a.logp)
                    a.logp[row] = token < 0        ? 0.0f
                                  : token >= a.M   ? NAN
                                  : x == -INFINITY ? (isnan(logS) ? NAN : -INFINITY)
                                                   : at_most_zero(rest.below(x, a.inv_t));
                if (ENT) a.entropy[row] = w.S == 0.0f ? 0.0f : at_least_zero((double)logS - kLn2 * (double)(w.E / w.S));
                s_ref = w.S == 0.0f ? 0.0 : (double)w.ref;
                s_log = (double)logS;
            }
        }
        if constexpr (TOP) {
            __syncthreads();
            const double row_ref = s_ref, row_log = s_log;
            const bool broken = isnan(row_ref * 0.0 + row_log);     // S = 0 (log -inf) is an empty row, not a broken one
            auto put = [&](int place, float logp, long long column) {
                const long long o = row * a.K + place;
                a.top[o] = logp;
                if (a.at_wide) static_cast<long long *>(a.at)[o] = column;
                else static_cast<int *>(a.at)[o] = (int)column;
            };
            const u64 *from = C > 1 ? s_top.merge : s_top.cand;
            const int n = broken ? 0 : C > 1 ? C * a.K : n_local;
            if (broken)          // a NaN may stand anywhere in the order, and fewer than K may have passed
                for (int i = tid; i < a.K; i += THREADS) put(i, NAN, -1);
            for (int i = tid; i < n; i += THREADS) {
                const u64 k = from[i];
                if (k == 0) continue;
                int above = 0;
#pragma unroll 4
                for (int j = 0; j < n; ++j) above += from[j] > k;
                if (above >= a.K) continue;
                const float x = value_of((unsigned)(k >> 32));
                put(above, x == -INFINITY ? x : at_most_zero(((double)x - row_ref) * a.inv_t - row_log),
                    (long long)(0xffffffffu - (unsigned)k));
            }
        }
        __syncthreads();     // before the next row's values come into the shared memory that this one's are read from
    }
}

// ---- gradients -------------------------------------------------------------------------------------------
struct GradArgs {
    RowArgs r;
    void *dx;
    long long lddx;
    const float *lse, *entropy, *rest, *dlogp, *dentropy, *dloss;
};

// The sums of a gradient's row from the logits themselves, over vectors from, from + step, ... and all threads of the CTA; with
// MASK the listed columns are left out. A vector of a list is found by a bit of its number (false hits cost a look).
template <typename T, int THREADS, bool MASK>
__device__ Sums row_sums(const Row<T> rv, const float c, const int from, const int step, const List *l,
                                      const int K) {
    constexpr int VE = Elem<T>::VE, NW = THREADS / 32, kMarks = 8192;
    __shared__ Sums s_warp[NW];
    __shared__ unsigned s_marks[MASK ? kMarks / 32 : 1];
    const int tid = threadIdx.x, lane = tid & 31;
    if constexpr (MASK) {
        for (int i = tid; i < kMarks / 32; i += THREADS) s_marks[i] = 0;
        __syncthreads();
        for (int k = tid; k < K; k += THREADS)
            if (l->used[k]) {
                const int m = ((l->col[k] + rv.mis) / VE) % kMarks;
                atomicOr(&s_marks[m >> 5], 1u << (m & 31));
            }
        __syncthreads();
    }
    Sums a{-INFINITY, 0.0f, 0.0f};
    for (int v = from; v < rv.nvec; v += step) {
        Vec r = rv.whole(v) ? ld_stream(rv.at(v)) : rv.edge(v);
        if constexpr (MASK) {
            const int m = v % kMarks;
            if (s_marks[m >> 5] >> (m & 31) & 1u) {
                T *e = reinterpret_cast<T *>(r.w);
                const unsigned fill = Elem<T>::kFill;
                for (int k = 0; k < K; ++k) {
                    const int col = l->col[k] + rv.mis;
                    if (!l->used[k] || col / VE != v) continue;
#pragma unroll
                    for (int i = 0; i < VE; ++i)
                        if (i == col % VE) e[i] = *reinterpret_cast<const T *>(&fill);
                }
            }
        }
        const float vm = Elem<T>::vmax(r);
        if (vm > a.ref) {
            a.S = a.S == 0.0f ? 0.0f : a.S * pb::ex2_approx((a.ref - vm) * c);
            a.ref = vm;
        }
        if (a.ref == -INFINITY) continue;
#pragma unroll
        for (int i = 0; i < VE / 2; ++i) {
            float x0, x1;
            Elem<T>::pair(r, i, x0, x1);
            a.S += pb::ex2_approx((x0 - a.ref) * c) + pb::ex2_approx((x1 - a.ref) * c);
        }
    }
    a = warp_join<false>(a, c);
    if (lane == 0) s_warp[tid >> 5] = a;
    __syncthreads();
    return warp_join<false>(lane < NW ? s_warp[lane] : Sums{0.0f, 0.0f, 0.0f}, c);
}

// Whether `given`, in 32 bits, is this sum's rounding: half a step of it, and what two sums of a row may differ by. A sum over
// more columns than the row's (a vocabulary in parts) is not, and is then taken as it was given.
__device__ __forceinline__ bool same_sum(float given, const Mass &m, double inv_t) {
    if (m.log == -INFINITY) return given == -INFINITY;
    return fabs((double)limited(m.value(inv_t)) - (double)given) <= 0x1p-23 * fabs((double)given) + 0x1p-10;
}

// What bounds it: memory. One exp2, 10 instructions and 4 bytes a 16-bit logit; 4096 x 131072 bf16 with a list in 350 us is
// 6.1 TB/s, 93 % of the measured copy rate, 4096 x 65536 with the entropy's term in 178 us 92 %. A list's columns are written by a
// second, short pass over what the first one wrote: to look for them within the first cost 1141 us.
// grid.x = rows x parts; the vectors of a row are dealt round robin to the threads of its parts. Every element is
// read and written by the same thread, so dx may be x itself (a list's logits are read before the first store only
// within a CTA: in place needs parts = 1 there).
//
// lse (and rest) come in 32 bits: their rounding, up to 2^-24 |lse|, scales every probability of the row. Up to |lse| = 64 for
// fp32 and 1024 for 16-bit gradients that is 2^-18 and 2^-14 (a value's own rounding: 2^-24; 2^-9 and 2^-12). Rows beyond,
// whose logits share a large offset, lie under a mask of the type's lowest value, or meet a small temperature, are summed
// again here in a pass of their own before the first store. `together`: the parts of a row are a cluster and share that
// pass, because in place another part's stores would be under way.
template <typename T, int THREADS, int LIST>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) row_grad(const GradArgs g, const int parts, const bool together) {
    constexpr int VE = Elem<T>::VE, U = 2;
    __shared__ ListSmem<THREADS, LIST == kNone ? kNone : kRenorm> s_list;
    __shared__ Teacher s_teacher;
    __shared__ Sums s_part[LIST == kNone ? kMaxCluster : 1];
    const RowArgs &a = g.r;
    const int tid = threadIdx.x;
    const int part = blockIdx.x % parts;
    const long long row = blockIdx.x / parts;
    const int total = parts * THREADS, me = part * THREADS + tid;
    const T *xr = static_cast<const T *>(a.x) + row * a.ldx;
    T *dr = static_cast<T *>(g.dx) + row * g.lddx;
    const Row<T> rv(xr, a.M);
    const unsigned apart = (unsigned)((reinterpret_cast<uintptr_t>(xr) ^ reinterpret_cast<uintptr_t>(dr)) & 31u);
    const float c = (float)(kLog2eD * a.inv_t);

    // dx_j = e_j (al + be t_j), t_j = (x_j - ref) c, e_j = exp2(t_j), for every column but the token's
    // (gamma more) and the listed ones (written last). ref is lse (or rest) in units of x, as a high and a
    // low part, because its rounding would scale the whole row.
    const float lse = g.lse[row];
    double base = (double)lse;
    float al = 0.0f, be = 0.0f, gamma = 0.0f;
    long long token = -1;                     // its column, where this thread writes it
    float x_token = 0.0f;
    double w = 0.0, W = 0.0;
    Mass row_lse{0.0, base};
    bool broken = false;
    const bool dead = base == -INFINITY;      // no finite logit in the row: no gradient
    auto far_off = [&](float v) { return isfinite(v) && fabsf(v) > (sizeof(T) == 4 ? 64.0f : 1024.0f); };
    float far_ref = 0.0f, far_log2 = 0.0f;    // of a row that is summed again
    bool again = false;
    if constexpr (LIST == kNone) {
        if (a.tokens) token = load_index(a.tokens, row, a.wide);
        const double dl = g.dlogp && token >= 0 ? (double)g.dlogp[row] : 0.0;
        const double de = g.dentropy ? (double)g.dentropy[row] : 0.0;
        if (!dead) {
            al = (float)((-dl - (g.dentropy ? de * (double)g.entropy[row] : 0.0)) * a.inv_t);
            be = (float)(-de * kLn2 * a.inv_t);
            gamma = (float)(dl * a.inv_t);
        }
        if (token >= a.M) al = NAN;
        if (token >= 0 && token < a.M && !dead && (int)((token + rv.mis) / VE) % total == me)
            x_token = Elem<T>::to_float(xr[token]);      // before it may be written over
        else
            token = -1;
        if (far_off(lse)) {
            Sums s = together ? row_sums<T, THREADS, false>(rv, c, me, total, nullptr, 0)
                              : row_sums<T, THREADS, false>(rv, c, tid, THREADS, nullptr, 0);
            if (together) {
                cluster_arrive();             // every part runs before the first store into its shared memory
                cluster_wait();
                if (tid < parts) {
                    const unsigned to = map_to_rank(smem_u32(&s_part[part]), tid);
                    st_cluster_f32(to, s.ref);
                    st_cluster_f32(to + 4, s.S);
                }
                cluster_arrive();
                cluster_wait();
                const int lane = tid & 31;
                s = lane < parts ? Sums{s_part[lane].ref, s_part[lane].S, 0.0f} : Sums{0.0f, 0.0f, 0.0f};
                s = warp_join<false>(s, c);
            }
            again = same_sum(lse, Mass{(double)s.ref, (double)logf(s.S)}, a.inv_t);
            far_ref = s.ref;
            far_log2 = log2f(s.S);
        }
    } else {
        load_list(s_list.l, a, row, xr);
        const bool far_row = far_off(lse) || (LIST == kTail && !dead && far_off(g.rest[row]));
        if (tid < 32) {
            const Teacher t = LIST == kTail && far_row ? warp_teacher<LIST == kTail, true>(s_list.l, a.K, a.inv_t)
                                                       : warp_teacher<LIST == kTail, false>(s_list.l, a.K, a.inv_t);
            if (tid == 0) s_teacher = t;
        }
        __syncthreads();
        const Teacher t = s_teacher;
        Mass rest{0.0, LIST == kTail ? (double)g.rest[row] : 0.0};
        if (far_row) {
            const Sums s = row_sums<T, THREADS, LIST == kTail>(rv, c, tid, THREADS, &s_list.l, a.K);
            const Mass found{(double)s.ref, (double)logf(s.S)};
            const Mass all = LIST == kTail ? join_mass(found, t.listed, a.inv_t) : found;
            again = same_sum(lse, all, a.inv_t) && (LIST != kTail || same_sum(g.rest[row], found, a.inv_t));
            if (again) {
                row_lse = all;
                rest = found;
            }
            far_ref = s.ref;
            far_log2 = log2f(s.S);
        }
        const double left = LIST == kTail ? left_of(t, a.M) : 0.0;
        w = (double)g.dloss[row] * a.inv_t;
        W = t.mass + left;
        broken = s_list.l.bad || isnan(t.mass) || isnan(base);
        if (broken) {
            al = NAN;
        } else if (!dead && LIST == kTail) {
            // exp(z - rest) cannot overflow where it is used, however little the student has there
            base = (double)g.rest[row];
            al = rest.log == -INFINITY
                     ? 0.0f
                     : (float)(w * (W * exp((rest.ref - row_lse.ref) * a.inv_t + rest.log - row_lse.log) - left));
        } else if (!dead) {
            al = (float)(w * W);
        }
    }
    if (base == -INFINITY) base = 0.0;        // every x it meets is -inf: exp2(-inf) = 0
    base /= a.inv_t;
    again = again && far_log2 != -INFINITY;
    const float hi = again ? far_ref : (float)base;
    const float lo = again ? far_log2 : (float)((base - (double)hi) * (double)c);

    auto slope = [&](float x) {
        const float t = fmaf(x - hi, c, -lo);
        const float e = pb::ex2_approx(t);
        return LIST == kNone ? e * fmaf(be, fmaxf(t, -1024.0f), al) : e * al;      // e = 0 long before
    };
    auto put = [&](const Vec &r, int at, bool whole) {
        Vec o;
#pragma unroll
        for (int i = 0; i < VE / 2; ++i) {
            float x0, x1;
            Elem<T>::pair(r, i, x0, x1);
            Elem<T>::set_pair(o, i, slope(x0), slope(x1));
        }
        const int c0 = rv.first(at);
        if (whole && apart == 0) {
            st_stream(dr + c0, o);
        } else if (whole && (apart & 3u) == 0) {       // rows of x and dx at different places of 32 bytes
            unsigned *w = reinterpret_cast<unsigned *>(dr + c0);
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = o.w[i];
        } else {
            const T *e = reinterpret_cast<const T *>(o.w);
#pragma unroll
            for (int i = 0; i < VE; ++i)
                if (c0 + i >= 0 && c0 + i < a.M) dr[c0 + i] = e[i];
        }
    };

    if (rv.v0 && me == 0) put(rv.edge(0), 0, false);
    {
        int v = me < rv.v0 ? me + total : me;
        for (; v + (U - 1) * total < rv.v1; v += U * total) {
            Vec r[U];
#pragma unroll
            for (int u = 0; u < U; ++u) r[u] = ld_stream(rv.at(v + u * total));
#pragma unroll
            for (int u = 0; u < U; ++u) put(r[u], v + u * total, true);
        }
        for (; v < rv.v1; v += total) put(ld_stream(rv.at(v)), v, true);
    }
    if (rv.tail() && me == rv.v1 % total) put(rv.edge(rv.v1), rv.v1, false);
    if constexpr (LIST == kNone) {
        if (token >= 0) dr[token] = Elem<T>::from_float(slope(x_token) + gamma);     // over this thread's own value
    } else {
        // the listed columns of this part's vectors, over what the pass wrote there (each column is listed once)
        __syncthreads();
        const Teacher teacher = s_teacher;
        for (int k = tid; k < a.K; k += THREADS)
            if (s_list.l.used[k] && ((s_list.l.col[k] + rv.mis) / VE) % total / THREADS == part) {
                const float p = expf((float)row_lse.below(s_list.l.x[k], a.inv_t));
                const float q = expf((float)teacher.log_q(s_list.l.v[k]));
                dr[s_list.l.col[k]] =
                    Elem<T>::from_float(broken ? NAN : dead ? 0.0f : (float)(w * (W * (double)p - (double)q)));
            }
    }
}

// ---- host side ---------------------------------------------------------------------------------------------
size_t size_of(int32_t dtype) { return dtype == PARPY_B200_F32 ? 4 : 2; }

int32_t check_rows(const char *what, const void *x, int32_t dtype, int64_t ldx, int64_t N, int64_t M,
                   double temperature) {
    PB_REQUIRE(dtype == PARPY_B200_F32 || dtype == PARPY_B200_BF16 || dtype == PARPY_B200_F16,
               "%s: unknown element type %d", what, dtype);
    PB_REQUIRE(N >= 0 && M >= 1 && M <= INT_MAX - 64, "%s: shape (%lld, %lld) is not supported", what, (long long)N,
               (long long)M);
    PB_REQUIRE(ldx >= M || N <= 1, "%s: row pitch %lld is smaller than a row of %lld", what, (long long)ldx,
               (long long)M);
    PB_REQUIRE(temperature >= 1e-4 && temperature <= 1e4, "%s: temperature %g is outside [1e-4, 1e4]", what,
               temperature);
    PB_REQUIRE(N == 0 || x, "%s: null pointer", what);
    PB_REQUIRE(reinterpret_cast<uintptr_t>(x) % size_of(dtype) == 0, "%s: misaligned logits", what);
    return PB_OK;
}

template <typename T, int THREADS, bool ENT, bool TOP, int LIST>
int32_t launch_row_stats(const char *what, const RowArgs &a, int C, const pb::DeviceInfo &dev, cudaStream_t stream) {
    auto kernel = row_stats<T, THREADS, ENT, TOP, LIST>;
    static std::atomic<int> resident{0};      // the same on every device the library runs on
    int per_sm = resident.load(std::memory_order_relaxed);
    if (per_sm == 0) {
        PB_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, THREADS, 0));
        resident.store(std::max(per_sm, 1), std::memory_order_relaxed);
    }
    // a row for each cluster, or as many CTAs as are resident, which take rows in turn
    const long long grid = C > 1 ? a.N * C : std::min<long long>(a.N, (long long)std::max(per_sm, 1) * dev.sm_count);
    PB_REQUIRE(grid <= INT_MAX, "%s: %lld rows are too many", what, a.N);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(THREADS);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim = {(unsigned)C, 1, 1};
    cfg.attrs = attr;
    cfg.numAttrs = C > 1 ? 1 : 0;
    PB_CUDA(cudaLaunchKernelEx(&cfg, kernel, a, C));
    return PB_OK;
}

template <typename T, bool ENT, bool TOP, int LIST>
int32_t launch_stats(const char *what, const RowArgs &a, cudaStream_t stream) {
    pb::DeviceInfo dev;
    const int32_t rc = pb::device_info(&dev);
    if (rc) return rc;
    const long long bytes = (long long)a.M * sizeof(T);
    constexpr int kBig = TOP || LIST == kTail ? 256 : 128;
    const bool big = bytes >= 4 * kBig * 32;
    const int threads = big ? kBig : 128;
    int C = 1;
    while (C < kMaxCluster && a.N * C < 2LL * dev.sm_count && bytes / (2 * C) >= (long long)threads * 32) C *= 2;
    if constexpr (LIST == kNone) {
        // a row that gives a lane four vectors at most is one warp's (32 groups bound up to 32 alternatives)
        if (bytes <= 4 * 32 * 32 && a.K <= 32) return launch_row_stats<T, 32, ENT, TOP, LIST>(what, a, 1, dev, stream);
    }
    return big ? launch_row_stats<T, kBig, ENT, TOP, LIST>(what, a, C, dev, stream)
               : launch_row_stats<T, 128, ENT, TOP, LIST>(what, a, C, dev, stream);
}

template <typename T>
int32_t launch_logprobs(const RowArgs &a, cudaStream_t stream) {
    const char *what = "token_logprobs";
    if (a.entropy)
        return a.K ? launch_stats<T, true, true, kNone>(what, a, stream)
                   : launch_stats<T, true, false, kNone>(what, a, stream);
    return a.K ? launch_stats<T, false, true, kNone>(what, a, stream)
               : launch_stats<T, false, false, kNone>(what, a, stream);
}

template <typename T, int LIST>
int32_t launch_grad(const char *what, const GradArgs &g, cudaStream_t stream) {
    pb::DeviceInfo dev;
    const int32_t rc = pb::device_info(&dev);
    if (rc) return rc;
    const long long bytes = (long long)g.r.M * sizeof(T);
    // small CTAs keep more rows apart in their phases (8192 x 16384: 113 us with 128 threads, 190 us with 512; with a list),
    // large ones have less of a row's constants to make (4096 x 131072: 358 and 342 us)
    const bool big = bytes >= 192 * 1024, in_place = g.r.x == g.dx;
    const int threads = big ? 512 : 128;
    // in place, a row's parts are a cluster, or one where there is a list
    const int most = !in_place ? INT_MAX : LIST == kNone ? kMaxCluster : 1;
    int parts = 1;
    while (parts < most && g.r.N * parts < 4LL * dev.sm_count && bytes / (2 * parts) >= (long long)threads * 16) parts *= 2;
    PB_REQUIRE(g.r.N * parts <= INT_MAX, "%s: %lld rows are too many", what, g.r.N);
    const bool together = in_place && parts > 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(g.r.N * parts));
    cfg.blockDim = dim3((unsigned)threads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim = {(unsigned)parts, 1, 1};
    cfg.attrs = attr;
    cfg.numAttrs = together ? 1 : 0;
    auto kernel = big ? row_grad<T, 512, LIST> : row_grad<T, 128, LIST>;
    PB_CUDA(cudaLaunchKernelEx(&cfg, kernel, g, parts, together));
    return PB_OK;
}

int32_t check_gradient(const char *what, const void *x, int32_t dtype, int64_t ldx, int64_t N, int64_t M, void *dx,
                       int64_t lddx) {
    PB_REQUIRE(N == 0 || dx, "%s: null pointer", what);
    PB_REQUIRE(lddx >= M || N <= 1, "%s: row pitch %lld is smaller than a row of %lld", what, (long long)lddx,
               (long long)M);
    PB_REQUIRE(reinterpret_cast<uintptr_t>(dx) % size_of(dtype) == 0, "%s: misaligned gradient", what);
    PB_REQUIRE(x != dx || ldx == lddx || N <= 1, "%s: in place needs equal row pitches", what);
    return PB_OK;
}

int32_t check_list(const char *what, const void *index, const void *values, int32_t value_dtype, int64_t K) {
    PB_REQUIRE(index && values, "%s: null pointer", what);
    PB_REQUIRE(K >= 1 && K <= kListMax, "%s: K=%lld is outside [1, %d]", what, (long long)K, kListMax);
    PB_REQUIRE(value_dtype == PARPY_B200_F32 || value_dtype == PARPY_B200_BF16 || value_dtype == PARPY_B200_F16,
               "%s: unknown element type %d", what, value_dtype);
    return PB_OK;
}

#define PB_BY_TYPE(dtype, expr)                                    \
    switch (dtype) {                                               \
        case PARPY_B200_F32: { using T = float; return expr; }     \
        case PARPY_B200_BF16: { using T = __nv_bfloat16; return expr; } \
        default: { using T = __half; return expr; }                \
    }

}  // namespace

extern "C" {

int32_t parpy_b200_token_logprobs(const void *x, int32_t dtype, int64_t ldx, int64_t N, int64_t M, const void *tokens,
                                  int32_t wide_tokens, double temperature, int64_t K, float *logp, float *lse,
                                  float *entropy, float *top_logp, void *top_index, int32_t wide_index, void *stream) {
    const int32_t rc = check_rows("token_logprobs", x, dtype, ldx, N, M, temperature);
    if (rc) return rc;
    PB_REQUIRE(K >= 0 && K <= kTopMax && K <= M, "token_logprobs: K=%lld is outside [0, min(M, %d)]", (long long)K,
               kTopMax);
    if (N == 0) return PB_OK;
    PB_REQUIRE(lse && (!logp || tokens) && (K == 0 || (top_logp && top_index)), "token_logprobs: null pointer");
    RowArgs a = {};
    a.x = x;
    a.ldx = ldx;
    a.N = N;
    a.M = (int)M;
    a.K = (int)K;
    a.inv_t = 1.0 / temperature;
    a.tokens = logp ? tokens : nullptr;
    a.wide = wide_tokens;
    a.logp = logp;
    a.lse = lse;
    a.entropy = entropy;
    a.top = top_logp;
    a.at = top_index;
    a.at_wide = wide_index;
    PB_BY_TYPE(dtype, launch_logprobs<T>(a, static_cast<cudaStream_t>(stream)))
}

int32_t parpy_b200_token_logprobs_grad(const void *x, int32_t dtype, int64_t ldx, int64_t N, int64_t M,
                                       const void *tokens, int32_t wide_tokens, double temperature, const float *lse,
                                       const float *entropy, const float *dlogp, const float *dentropy, void *dx,
                                       int64_t lddx, void *stream) {
    int32_t rc = check_rows("token_logprobs_grad", x, dtype, ldx, N, M, temperature);
    if (!rc) rc = check_gradient("token_logprobs_grad", x, dtype, ldx, N, M, dx, lddx);
    if (rc || N == 0) return rc;
    PB_REQUIRE(lse && (!dlogp || tokens) && (!dentropy || entropy), "token_logprobs_grad: null pointer");
    GradArgs g = {};
    g.r.x = x;
    g.r.ldx = ldx;
    g.r.N = N;
    g.r.M = (int)M;
    g.r.inv_t = 1.0 / temperature;
    g.r.tokens = dlogp ? tokens : nullptr;
    g.r.wide = wide_tokens;
    g.dx = dx;
    g.lddx = lddx;
    g.lse = lse;
    g.entropy = entropy;
    g.dlogp = dlogp;
    g.dentropy = dentropy;
    PB_BY_TYPE(dtype, (launch_grad<T, kNone>("token_logprobs_grad", g, static_cast<cudaStream_t>(stream))))
}

int32_t parpy_b200_distill_topk(const void *x, int32_t dtype, int64_t ldx, int64_t N, int64_t M, const void *index,
                                int32_t wide_index, const void *values, int32_t value_dtype, int64_t K,
                                double temperature, int32_t tail, float *loss, float *lse, float *rest, void *stream) {
    int32_t rc = check_rows("distill_topk", x, dtype, ldx, N, M, temperature);
    if (rc || N == 0) return rc;
    rc = check_list("distill_topk", index, values, value_dtype, K);
    if (rc) return rc;
    PB_REQUIRE(loss && lse && (!tail || rest), "distill_topk: null pointer");
    RowArgs a = {};
    a.x = x;
    a.ldx = ldx;
    a.N = N;
    a.M = (int)M;
    a.K = (int)K;
    a.inv_t = 1.0 / temperature;
    a.index = index;
    a.values = values;
    a.wide = wide_index;
    a.value_type = value_dtype;
    a.lse = lse;
    a.loss = loss;
    a.rest = tail ? rest : nullptr;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    PB_BY_TYPE(dtype, (tail ? launch_stats<T, false, false, kTail>("distill_topk", a, s)
                            : launch_stats<T, false, false, kRenorm>("distill_topk", a, s)))
}

int32_t parpy_b200_distill_topk_grad(const void *x, int32_t dtype, int64_t ldx, int64_t N, int64_t M,
                                     const void *index, int32_t wide_index, const void *values, int32_t value_dtype,
                                     int64_t K, double temperature, int32_t tail, const float *lse, const float *rest,
                                     const float *dloss, void *dx, int64_t lddx, void *stream) {
    int32_t rc = check_rows("distill_topk_grad", x, dtype, ldx, N, M, temperature);
    if (!rc) rc = check_gradient("distill_topk_grad", x, dtype, ldx, N, M, dx, lddx);
    if (rc || N == 0) return rc;
    rc = check_list("distill_topk_grad", index, values, value_dtype, K);
    if (rc) return rc;
    PB_REQUIRE(lse && dloss && (!tail || rest), "distill_topk_grad: null pointer");
    GradArgs g = {};
    g.r.x = x;
    g.r.ldx = ldx;
    g.r.N = N;
    g.r.M = (int)M;
    g.r.K = (int)K;
    g.r.inv_t = 1.0 / temperature;
    g.r.index = index;
    g.r.values = values;
    g.r.wide = wide_index;
    g.r.value_type = value_dtype;
    g.dx = dx;
    g.lddx = lddx;
    g.lse = lse;
    g.rest = rest;
    g.dloss = dloss;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    PB_BY_TYPE(dtype, (tail ? launch_grad<T, kTail>("distill_topk_grad", g, s)
                            : launch_grad<T, kRenorm>("distill_topk_grad", g, s)))
}

}  // extern "C"
