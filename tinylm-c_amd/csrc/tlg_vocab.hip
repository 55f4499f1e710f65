// tlg_vocab.hip -- operators over rows of logits [N][V] besides softmax-CE and
// argmax: log probabilities of given tokens with entropy and top alternatives,
// their gradient, and distillation from a teacher's top log probabilities.
//
// For one row x[0..V) and a scale s = 1 / temperature:
//   m = max x,  S = sum_v e^(s (x_v - m)),  log p_v = s (x_v - m) - log S
//   H = -sum_v p_v log p_v = log S - s sum_v (x_v - m) e^(s (x_v - m)) / S
// All of them are bound by HBM: a logit is read once (and its gradient written
// once) per call, and the work on it (one or two exponentials, a maximum, two or
// three sums) fits in the time its bytes take.  Sums are fp32, joined over
// threads in a fixed order, and fp64 where K terms cancel; 16-bit outputs are rounded
// once.  Times in this file are of calls within a graph, over several sets of rows in
// turn, which together do not fit the last-level cache where a set is 50 MB or more.
#include "tlg_internal.h"
#include "tlg_rows.h"
#include "../../include/tltrain.h"
#include <float.h>
#include <math.h>

#define ST(s) ((hipStream_t)(s))
#define LAUNCH_CHECK() TLG_HIP(hipGetLastError())

typedef unsigned long long u64;
__device__ __forceinline__ u64 lane_u64(u64 v, int lane)
{
    const unsigned lo = __builtin_amdgcn_readlane((unsigned)v, lane);
    const unsigned hi = __builtin_amdgcn_readlane((unsigned)(v >> 32), lane);
    return (u64)hi << 32 | lo;
}

// A total order of values (equal for -0 and +0) in the high half and the lower
// position first in the low half; 0 for -inf, which is no alternative.
__device__ __forceinline__ u64 vb_key(float x, int g)
{
    const unsigned b = __float_as_uint(x + 0.0f);
    const unsigned o = b & 0x80000000u ? ~b : b | 0x80000000u;
    return x == -INFINITY ? 0ull : (u64)o << 32 | (unsigned)~g;
}
__device__ __forceinline__ float vb_key_value(u64 k)
{
    const unsigned o = (unsigned)(k >> 32);
    return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}

// -------------------------------------------------------------- one pass --
// Running sums of a thread's part of a row in base 2: with c = scale log2 e
// rounded and a reference R = m c rounded, m the part's maximum so far,
//   t_v = x_v c - R (one fused product),  s = sum 2^t,  u = sum t 2^t.
// R is exact as the reference it is, whatever its distance from m c, so parts
// join by the differences of their references, and
//   rho = R - m c,  log sum e^(scale (x - m)) = ln 2 rho + log(s + kappa u),
// with kappa = ln 2 (scale log2 e - c) / c for the rounding of c, to first order.
// NaN and +inf make s NaN.  Exponents are clamped at -200, where 2^t is 0, in the
// factor of the products only: 0 * -inf must not be NaN, NaN must stay.  R is kept
// at -ACC_FAR or above, so that a part of nothing but masked values, -inf or large
// finite ones, has s = 0 or one of its size; a row whose maximum is farther than
// that from 0, where the rounding of m c would reach the exponents, has its sums
// formed from differences (sums_apart).
#define ACC_FAR 1e6f
struct Acc { float R, s, u; };
#define ACC0 {-ACC_FAR, 0.f, 0.f}
__device__ __forceinline__ float acc_ref(float m, float c) { return fmaxf(m * c, -ACC_FAR); }
__device__ __forceinline__ void acc_shift(Acc &a, float R)                    // to a reference R >= a.R
{
    const float d = a.R - R, f = __builtin_amdgcn_exp2f(d);
    a.u = f * fmaf(fmaxf(d, -200.f), a.s, a.u);
    a.s *= f;
    a.R = R;
}
// A sum loses what is below half its last place: an element at a time, the many
// small terms of a long row (the mean of log S was off by -1.1e-7 for 30000 values of
// deviation 2.5 at scale 1 / 0.7, by -4e-6 for 2^20 of them).  So a vector's sums are
// formed by themselves, then a round's, then the thread's.
template <int TYPE> __device__ __forceinline__ Acc acc_vector(const u32x4 &q, float R, float c)
{
    Acc a;
#pragma unroll
    for (int e = 0; e < El<TYPE>::VE; e++) {
        const float t = fmaf(el_at<TYPE>(q, e), c, -R), v = __builtin_amdgcn_exp2f(t), l = fmaxf(t, -200.f);
        a.s = e ? a.s + v : v;
        a.u = e ? fmaf(v, l, a.u) : v * l;
    }
    return a;
}
// all lanes' parts in every lane, m the wave's maximum; the order of additions is fixed
__device__ __forceinline__ Acc acc_wave(Acc a, float m, float c)
{
    acc_shift(a, acc_ref(m, c));
    return Acc{a.R, wave_sum(a.s), wave_sum(a.u)};
}
// parts {s, u, m} relative to their own references
__device__ __forceinline__ Acc acc_join(const f32x4 *p, int n, float c, float &m)
{
    m = p[0][2];
    for (int w = 1; w < n; w++) m = fmaxf(m, p[w][2]);
    Acc r = {acc_ref(m, c), 0.f, 0.f};
    for (int w = 0; w < n; w++) {
        Acc a = {acc_ref(p[w][2], c), p[w][0], p[w][1]};
        acc_shift(a, r.R);
        r.s += a.s;
        r.u += a.u;
    }
    return r;
}
__device__ __forceinline__ bool acc_far(float m, float c) { return fabsf(m * c) > ACC_FAR && m > -INFINITY; }
// What is asked of a row: m its maximum, ls = log sum e^(scale (x - m)), H the
// entropy; NaN and -inf mark rows without a distribution.
struct Sums { float m, ls, H; };
template <int TYPE, int W>
__device__ __noinline__ Acc sums_apart(const Row<TYPE> x, float m, float c, int t, f32x4 *part)
{
    constexpr int VE = El<TYPE>::VE;
    Acc a = {0.f, 0.f, 0.f};                            // R is not used: rho = 0
    for (int j = t; j < x.nv; j += 64 * W) {
        const u32x4 q = x.any(j);
        float s = 0.f, u = 0.f;
#pragma unroll
        for (int e = 0; e < VE; e++) {
            const float d = (el_at<TYPE>(q, e) - m) * c, f = __builtin_amdgcn_exp2f(d);
            s += f;
            u = fmaf(f, fmaxf(d, -200.f), u);
        }
        a.s += s;
        a.u += u;
    }
    a.s = wave_sum(a.s);
    a.u = wave_sum(a.u);
    if constexpr (W > 1) {
        row_sync<W>();
        if (t % 64 == 0) part[t / 64] = f32x4{a.s, a.u, 0.f, 0.f};
        row_sync<W>();
        a.s = a.u = 0.f;
        for (int w = 0; w < W; w++) {
            a.s += part[w][0];
            a.u += part[w][1];
        }
        row_sync<W>();
    }
    return a;
}
__device__ __forceinline__ Sums sums_of(float m, const Acc &a, float c, float kappa)
{
    if (a.s != a.s) return Sums{NAN, NAN, NAN};
    if (m == -INFINITY) return Sums{-INFINITY, -INFINITY, 0.f};
    const float rho = acc_far(m, c) ? 0.f : -fmaf(m, c, -a.R), ls = fmaf(0.69314718056f, rho, logf(fmaf(kappa, a.u, a.s)));
    return Sums{m, ls, ls - 0.69314718056f * fmaf(a.u, __builtin_amdgcn_rcpf(a.s), rho)};
}

// --------------------------------------------------------- log probabilities --
// The K largest of a row beside its sums.  Every thread keeps its own maximum v1.
// These are different elements, so a bound T that enough of them reach (J =
// ceil(K / waves) lanes of every wave) is reached by K elements of the row at
// least, in a row of random order by little more.  They go to a list, which is
// ranked by counting.  A row of at most U vectors a thread (RES) is still in
// registers then.  Of longer rows the pass leaves line maxima in LDS, for less than
// an operation per element: eight neighbouring lanes' vectors are a line of 128
// bytes (2^q lines U 64 W vectors apart, in rows of more than LP_LINES lines per
// wave); the lines that reach T are read again, by all threads evenly.  A list that
// overflows, from many equal values or large values that lie together, raises T by
// the same argument over what it holds, and is made again.
struct LpArgs {
    const void *logits;
    long long ld;
    int N, V, S;                 // S segments of a row, joined by k_logprobs_join
    float scale, c, kappa;       // c = scale log2 e rounded, kappa = ln 2 (scale log2 e - c) / c
    const int *ids;
    int M;
    float *logp, *lse2, *entropy;
    int K;
    int *top_ids;
    float *top_logp;
    float *part;                 // S > 1: [N][S][4]
    u64 *keys;                   // S > 1: [N][K][S], descending over K
};

// What a row's threads share.
#define LP_LINES 512
template <int W, bool LINES, bool TOP> struct LpShared {
    static constexpr int CAP = W < 4 ? 256 * W : 1024;
    f32x4 part[W];               // a wave's sums, maximum and bound
    u64 t[W];
    int n, lines;
    union {
        alignas(16) float max[LINES ? LP_LINES * W : 1];         // until the lines are chosen
        u64 cand[TOP ? CAP : 1];
    };
    unsigned short line[LINES ? LP_LINES * W : 1];
};

// A value that at least J lanes of the wave reach, and not many more; the lowest
// finite one if there is no such value.  Pivots are lanes' values; each step drops
// the pivot's lane at least.
__device__ __forceinline__ float wave_bound(float v, int J)
{
    float T = -FLT_MAX;
    u64 open = ~0ull;
    while (open) {
        const float p = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), __ffsll((long long)open) - 1));
        const u64 reach = __ballot(v >= p);
        const int n = __popcll(reach);
        if (n >= J) {
            T = fmaxf(T, p);
            if (n <= J + J / 4 + 1) break;
            open &= __ballot(v > p);
        } else
            open &= ~reach & ~(1ull << (__ffsll((long long)open) - 1));
    }
    return T;
}
// the same for the list's keys, exactly J lanes
__device__ __forceinline__ u64 wave_bound_key(u64 v, int J)
{
    u64 T = 0, open = ~0ull;
    while (open) {
        const int l = __ffsll((long long)open) - 1;
        const u64 p = lane_u64(v, l), reach = __ballot(v >= p);
        if (__popcll(reach) >= J) {
            T = p;
            open &= __ballot(v > p);
        } else
            open &= ~reach;
    }
    return T;
}

// The lanes' elements with `take` to the wave's list, whose length is n.
template <typename E> __device__ __forceinline__ void wave_push(bool take, E v, E *list, int &n, int cap)
{
    const u64 m = __ballot(take);
    const int at = n + __builtin_amdgcn_mbcnt_hi((unsigned)(m >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)m, 0));
    if (take && at < cap) list[at] = v;
    n += __popcll(m);
}
// element e, any e, of a raw vector
template <int TYPE> __device__ __forceinline__ float el_any(const u32x4 &r, int e)
{
    constexpr int P = El<TYPE>::VE / 4;                  // elements of a register
    const int k = e / P;
    const unsigned a = k & 1 ? r[1] : r[0], b = k & 1 ? r[3] : r[2], w = k & 2 ? b : a;
    return el_float<TYPE>(P == 1 ? w : w >> (e & 1) * 16 & 0xffffu);
}
// all elements of a vector at place j that reach T (by value, then by key)
template <int TYPE, int W>
__device__ __forceinline__ void lp_list(const u32x4 &q, int j, float T, u64 Tkey, u64 *cand, int &n, int cap)
{
    if constexpr (W == 1) {                              // all lanes at once: most elements reach T in none
#pragma unroll
        for (int e = 0; e < El<TYPE>::VE; e++) {
            const float x = el_at<TYPE>(q, e);
            if (__ballot(x >= T)) {
                const u64 key = vb_key(x, j * El<TYPE>::VE + e);
                wave_push(x >= T && key >= Tkey, key, cand, n, cap);
            }
        }
    } else {
        unsigned hit = 0;
#pragma unroll
        for (int e = El<TYPE>::VE - 1; e >= 0; e--) hit = hit * 2 + (el_at<TYPE>(q, e) >= T);
        while (hit) {
            const int e = __ffs(hit) - 1;
            hit &= hit - 1;
            const u64 key = vb_key(el_any<TYPE>(q, e), j * El<TYPE>::VE + e);
            if (key >= Tkey) {
                const int at = atomicAdd(&n, 1);
                if (at < cap) cand[at] = key;
            }
        }
    }
}

// a given token of a row and its logit, loaded ahead of the row's sums
struct Given { int id; float x; };
template <int TYPE> __device__ __forceinline__ Given lp_given(const LpArgs &a, size_t r, const char *x, int t)
{
    Given g = {-1, 0.f};
    if (t < a.M) {
        g.id = a.ids[r * a.M + t];
        if (g.id >= 0 && g.id < a.V) g.x = el_load<TYPE>(x, g.id);
    }
    return g;
}
__device__ __forceinline__ void lp_finish(const LpArgs &a, size_t r, const Given &g, const Sums &s, int t)
{
    if (t < a.M) {
        float o = lp_scaled(g.x, s.m, a.scale) - s.ls;
        if (s.m == -INFINITY) o = -INFINITY;
        a.logp[r * a.M + t] = g.id >= a.V ? NAN : g.id < 0 ? 0.f : o;
    }
    if (t == 0) {
        if (a.lse2) {
            a.lse2[2 * r] = s.m;
            a.lse2[2 * r + 1] = s.ls;
        }
        if (a.entropy) a.entropy[r] = s.H;
    }
}

__device__ __forceinline__ void lp_put(const LpArgs &a, size_t r, int k, u64 key, int sh, const Sums &s)
{
    const bool bad = s.ls != s.ls;
    a.top_ids[r * a.K + k] = key && !bad ? (int)~(unsigned)key - sh : -1;
    a.top_logp[r * a.K + k] = bad ? NAN : key ? lp_scaled(vb_key_value(key), s.m, a.scale) - s.ls : -INFINITY;
}

// W waves on a row, or on one of its S segments (W > 1); 4 rows of one wave per
// workgroup.  TOP: K > 0.
template <int TYPE, int W, int U, bool RES, bool TOP>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W) void k_logprobs(LpArgs a)
{
    constexpr int VE = El<TYPE>::VE, TPR = 64 * W;
    constexpr bool LINES = TOP && !RES;
    typedef LpShared<W, LINES, TOP> Sh;
    constexpr int CAP = Sh::CAP;
    __shared__ Sh shared[W == 1 ? 4 : 1];
    const int lane = threadIdx.x & 63, wave = W == 1 ? 0 : threadIdx.x >> 6, t = W == 1 ? lane : threadIdx.x;
    Sh &sh = shared[W == 1 ? threadIdx.x >> 6 : 0];
    size_t r;
    int seg = 0;
    if constexpr (W == 1) {
        r = (size_t)blockIdx.x * 4 + (threadIdx.x >> 6);
        if (r >= (size_t)a.N) return;                    // whole waves: no barrier follows for W == 1
    } else {
        r = blockIdx.x / (unsigned)a.S;
        seg = blockIdx.x % (unsigned)a.S;
    }
    const Row<TYPE> x(a.logits, a.ld, r, a.V);
    // the segment's vectors [j0, j1)
    const int per = a.S > 1 ? ((x.nv + a.S - 1) / a.S + TPR - 1) / TPR * TPR : x.nv;
    const int j0 = min(seg * per, x.nv), j1 = min(j0 + per, x.nv);
    u32x4 raw[U];
    auto load = [&](int j) {
        if (j >= x.f0 && j + (U - 1) * TPR < min(x.f1, j1)) {
#pragma unroll
            for (int k = 0; k < U; k++) raw[k] = __builtin_nontemporal_load(x.v + j + k * TPR);
        } else {
#pragma unroll
            for (int k = 0; k < U; k++) raw[k] = x.any(j + k * TPR < j1 ? j + k * TPR : x.nv);
        }
    };

    // lines are joined over 2^q rounds; every wave takes part in every round, so that
    // all lines up to the last round's are written
    int q = 0;
    if constexpr (LINES)
        while (LP_LINES * 8 * W << q < j1 - j0) q++;
    const Given given = lp_given<TYPE>(a, r, x.x, t);
    Acc A = ACC0;
    float v1 = -INFINITY;
    for (int j = j0 + t, l = (wave * 8 + lane / 8) * U; RES || j - t < j1; l += U * 8 * W) {
        float lm[U];
#pragma unroll
        for (int k = 0; k < U; k++) lm[k] = -INFINITY;
        for (int i = 0; i < 1 << q && (RES || j - t < j1); i++, j += U * TPR) {
            load(j);
            float gm = -INFINITY;
#pragma unroll
            for (int k = 0; k < U; k++) {
                float vm = el_at<TYPE>(raw[k], 0);
#pragma unroll
                for (int e = 1; e < VE; e++) vm = fmaxf(vm, el_at<TYPE>(raw[k], e));
                gm = fmaxf(gm, vm);
                if constexpr (LINES) lm[k] = fmaxf(lm[k], vm);
            }
            v1 = fmaxf(v1, gm);
            acc_shift(A, acc_ref(v1, a.c));
            Acc round;
#pragma unroll
            for (int k = 0; k < U; k++) {
                if (RES) keep_packed(raw[k]);
                const Acc v = acc_vector<TYPE>(raw[k], A.R, a.c);
                round.s = k ? round.s + v.s : v.s;
                round.u = k ? round.u + v.u : v.u;
                if (RES) keep_packed(raw[k]);
            }
            A.s += round.s;
            A.u += round.u;
        }
        if constexpr (LINES) {
#pragma unroll
            for (int k = 0; k < U; k++) {               // over 8 lanes
                lm[k] = fmaxf(lm[k], lane_move<0xB1>(lm[k]));
                lm[k] = fmaxf(lm[k], lane_move<0x4E>(lm[k]));
                lm[k] = fmaxf(lm[k], lane_move<0x141>(lm[k]));
            }
            if (lane % 8 == 0) *(f32x4 *)(sh.max + l) = f32x4{lm[0], lm[1], lm[2], lm[3]};
        }
        if (RES) break;
    }

    // the row's sums, maximum and bound
    float m = wave_max(v1), T = -FLT_MAX;
    A = acc_wave(A, m, a.c);
    if constexpr (TOP) {
        const int full = min(W, (j1 - j0) / 64);        // waves whose lanes all have a vector
        const int J = full ? (a.K + full - 1) / full : 65;
        T = wave >= (full ? full : 1) ? FLT_MAX : wave_bound(v1, J);
        if (W > 1 && t == 0) sh.n = sh.lines = 0;
    }
    if constexpr (W > 1) {
        if (lane == 0) sh.part[wave] = f32x4{A.s, A.u, m, T};
    }
    row_sync<W>();
    if constexpr (W > 1) {
        A = acc_join(sh.part, W, a.c, m);
        for (int w = 0; w < W; w++) T = fminf(T, sh.part[w][3]);
        if (a.S > 1 && t == 0) ((f32x4 *)a.part)[r * a.S + seg] = f32x4{A.s, A.u, m, 0.f};
    }
    const bool whole = W == 1 || a.S == 1;
    if (whole && acc_far(m, a.c)) A = sums_apart<TYPE, W>(x, m, a.c, t, sh.part);
    if constexpr (!TOP) {
        if (whole && wave == 0) lp_finish(a, r, given, sums_of(m, A, a.c, a.kappa), t);
        return;
    }

    // The lines that reach T, then the elements that do.  Line l is the lanes 8 o ..
    // 8 o + 7 of wave w in load k of the rounds i 2^q ..., from l's digits.
    int n1 = 0, lines1 = 0;                             // the lists' lengths, for one wave
    int &n = W == 1 ? n1 : sh.n, &lines = W == 1 ? lines1 : sh.lines;
    auto first = [&](int l) {
        const int k = l % U, o = l / U % 8, w = l / (U * 8) % W, i = l / (U * 8 * W);
        return j0 + (((i << q) * U + k) * W + w) * 64 + o * 8;
    };
    int items = 0;
    if constexpr (LINES) {
        const int rounds = (j1 - j0 + U * TPR - 1) / (U * TPR), all = ((rounds + (1 << q) - 1) >> q) * (U * 8 * W);
        for (int l = 4 * t; l - 4 * lane < all; l += 4 * TPR) {          // all is a multiple of 32
            const f32x4 v = l < all ? *(const f32x4 *)(sh.max + l) : f32x4{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int e = 0; e < 4; e++) {
                if constexpr (W == 1) wave_push(v[e] >= T, (unsigned short)(l + e), sh.line, lines, LP_LINES);
                else if (v[e] >= T) sh.line[atomicAdd(&lines, 1)] = l + e;
            }
        }
        row_sync<W>();
        items = lines * 8 << q;
    }
    // A list that has overflowed takes no more (4096 rows of 131072 equal bf16 values:
    // 2.4 -> 0.8 ms); rows in registers or of one wave are too short to gain by it.
    auto over = [&] {
        if constexpr (W > 1) return *(volatile int *)&sh.n > CAP;
        else return false;
    };
    auto list = [&](u64 Tkey) {
        if constexpr (RES) {
#pragma unroll
            for (int k = 0; k < U; k++) lp_list<TYPE, W>(raw[k], j0 + t + k * TPR, T, Tkey, sh.cand, n, CAP);
        } else
            for (int i = t; i - lane < items && !over(); i += TPR) {
                int j = x.nv;
                if (i < items)
                    j = first(sh.line[i >> (3 + q)]) + (i >> 3 & ((1 << q) - 1)) * (U * TPR) + i % 8;
                lp_list<TYPE, W>(x.any(j < j1 ? j : x.nv), j, T, Tkey, sh.cand, n, CAP);
            }
        row_sync<W>();
    };
    list(0);
    while (n > CAP) {
        u64 b = 0;
        for (int i = t; i < CAP; i += TPR) b = sh.cand[i] > b ? sh.cand[i] : b;
        b = wave_bound_key(b, (a.K + W - 1) / W);
        if constexpr (W > 1) {
            if (lane == 0) sh.t[wave] = b;
            row_sync<W>();
            for (int w = 0; w < W; w++) b = sh.t[w] < b ? sh.t[w] : b;
            if (t == 0) n = 0;
        } else
            n = 0;
        if (W > 1) T = fmaxf(T, vb_key_value(b));
        row_sync<W>();
        list(b);
    }
    const int got = n;
    u64 *out = a.keys + r * a.K * a.S + seg;             // S > 1
    if (wave > 0 && 64 * wave >= max(got, a.K)) return;  // nothing of the rest is this wave's
    Sums sum = {0.f, 0.f, 0.f};
    if (whole) {
        sum = sums_of(m, A, a.c, a.kappa);
        if (wave == 0) lp_finish(a, r, given, sum, t);
    }
    for (int i = t; i < got; i += TPR) {
        const u64 key = sh.cand[i];
        int rank = 0;
#pragma unroll 8
        for (int o = 0; o < got; o++) rank += sh.cand[o] > key;
        if (rank < a.K) {
            if (W > 1 && a.S > 1) out[(size_t)rank * a.S] = key;
            else lp_put(a, r, rank, key, x.sh, sum);
        }
    }
    for (int k = got + t; k < a.K; k += TPR) {
        if (W > 1 && a.S > 1) out[(size_t)k * a.S] = 0;
        else lp_put(a, r, k, 0, x.sh, sum);
    }
}

// Joins the S segments of a row: one workgroup per row.  Their K largest come
// sorted; the same bound and list pick the row's K from them, and the list can
// hold all of them.
#define LP_JOIN 4096                                     // S K at most
template <int TYPE, bool TOP> __global__ __launch_bounds__(256) void k_logprobs_join(LpArgs a)
{
    __shared__ f32x4 part[64];
    __shared__ float tw[4];
    __shared__ u64 cand[TOP ? LP_JOIN : 1];
    __shared__ int cnt;
    const size_t r = blockIdx.x;
    const int t = threadIdx.x, lane = t & 63, n = a.S * a.K;
    const Row<TYPE> x(a.logits, a.ld, r, a.V);
    const Given given = lp_given<TYPE>(a, r, x.x, t);
    if (t < a.S) part[t] = ((const f32x4 *)a.part)[r * a.S + t];
    float T = -FLT_MAX;
    const u64 *keys = a.keys + r * n;
    u64 held[2] = {0, 0};
    if constexpr (TOP) {
        u64 b = 0;
#pragma unroll
        for (int k = 0; k < 2; k++) {                    // most are held from the first reading
            held[k] = t + 256 * k < n ? keys[t + 256 * k] : 0;
            b = held[k] > b ? held[k] : b;
        }
        for (int i = t + 512; i < n; i += 256) b = keys[i] > b ? keys[i] : b;
        const int full = min(4, n / 64), J = full ? (a.K + full - 1) / full : 65;
        T = t / 64 >= (full ? full : 1) ? FLT_MAX : wave_bound(b ? vb_key_value(b) : -FLT_MAX, J);
        if (lane == 0) tw[t >> 6] = T;
        if (t == 0) cnt = 0;
    }
    __syncthreads();
    float m;
    Acc A = acc_join(part, a.S, a.c, m);
    __syncthreads();
    if (acc_far(m, a.c)) A = sums_apart<TYPE, 4>(x, m, a.c, t, part);
    const Sums sum = sums_of(m, A, a.c, a.kappa);
    lp_finish(a, r, given, sum, t);
    if constexpr (!TOP) return;
    for (int w = 0; w < 4; w++) T = fminf(T, tw[w]);
    auto put = [&](u64 key) {
        if (key && vb_key_value(key) >= T) cand[atomicAdd(&cnt, 1)] = key;
    };
    put(held[0]);
    put(held[1]);
    for (int i = t + 512; i < n; i += 256) put(keys[i]);
    __syncthreads();
    const int got = cnt;
    for (int i = t; i < got; i += 256) {
        const u64 q = cand[i];
        int rank = 0;
        for (int o = 0; o < got; o++) rank += cand[o] > q;
        if (rank < a.K) lp_put(a, r, rank, q, x.sh, sum);
    }
    for (int k = got + t; k < a.K; k += 256) lp_put(a, r, k, 0, x.sh, sum);
}

// Writing: vector j of row x's grid, one element at a time where the row's ends
// or a different alignment of the written row ask for it.
template <int TYPE>
__device__ __forceinline__ void row_store(const Row<TYPE> &x, const Row<TYPE> &d, int j, const float *g)
{
    constexpr int VE = El<TYPE>::VE;
    if (j >= x.f0 && j < x.f1 && d.sh == x.sh) {
        u32x4 q;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            if constexpr (TYPE == TLG_F32) q[k] = __float_as_uint(g[k]);
            else q[k] = el_bits<TYPE>(g[2 * k]) | el_bits<TYPE>(g[2 * k + 1]) << 16;
        }
        __builtin_nontemporal_store(q, const_cast<u32x4 *>(d.v) + j);
        return;
    }
#pragma unroll
    for (int e = 0; e < VE; e++) {
        const int i = j * VE + e - x.sh;
        if (i >= 0 && i < x.V) el_store<TYPE>(const_cast<char *>(d.x), i, g[e]);
    }
}

// ------------------------------------------------- log probabilities' gradient --
// dz_v = p_v (c0 - c1 (log p_v + H)) + the given tokens' own terms, with t_v =
// (x_v - m) c:  p_v = 2^t_v / S and log p_v = ln 2 t_v - log S, so a logit costs one
// exponential and two products.  One workgroup writes a segment of up to BW_SEG
// vectors of a row, then once more the given tokens among them; their logits are
// read before the first write, which may go to the same place.  4096 rows of 131072 in
// bf16 take 370 us, 5.8 TB/s of reads and writes.
#define BW_SEG 2048
struct LpBwdArgs {
    const void *logits;
    long long ld;
    int V, S;
    float scale, c;
    const int *ids;
    int M;
    const float *lse2, *entropy, *dlogp, *dlse, *dent;
    void *dlogits;
    long long ldd;
};

template <int TYPE> __global__ __launch_bounds__(256) void k_logprobs_bwd(LpBwdArgs a)
{
    constexpr int VE = El<TYPE>::VE, U = 4;
    __shared__ int si[TLG_VOCAB_IDS];
    __shared__ float sg[TLG_VOCAB_IDS];
    const size_t r = blockIdx.x / (unsigned)a.S;
    const int seg = blockIdx.x % (unsigned)a.S, t = threadIdx.x;
    const Row<TYPE> x(a.logits, a.ld, r, a.V), d(a.dlogits, a.ldd, r, a.V);
    const int j0 = seg * BW_SEG, j1 = min(j0 + BW_SEG, x.nv);
    float xv = 0.f;
    bool mine = false;
    if (t < a.M) {
        const int id = a.ids[r * a.M + t];
        si[t] = id;
        sg[t] = id >= a.V ? NAN : id >= 0 ? a.dlogp[r * a.M + t] : 0.f;
        const int j = (id + x.sh) / VE;
        mine = id >= 0 && id < a.V && j >= j0 && j < j1;
        if (mine) xv = el_load<TYPE>(x.x, id);
    }
    __syncthreads();
    float c0 = a.dlse ? a.dlse[r] : 0.f;
    bool some = c0 != 0.f;                               // any coefficient: those that cancel are no padding
    for (int j = 0; j < a.M; j++) {
        c0 -= sg[j];
        some |= sg[j] != 0.f;
    }
    const float c1 = a.dent ? a.dent[r] : 0.f, H = a.dent ? a.entropy[r] : 0.f;
    const float m = a.lse2[2 * r], ls = a.lse2[2 * r + 1];
    const bool empty = m == -INFINITY && c0 == c0;
    const bool zero = empty || (c0 == 0.f && c1 == 0.f && !(some && ls != ls));
    const float rs = a.scale * __expf(-ls), k1 = -0.69314718056f * c1, k0 = c0 - c1 * (H - ls);
    auto grad = [&](float v) -> float {
        const float e = (v - m) * a.c;
        return __builtin_amdgcn_exp2f(e) * rs * fmaf(k1, fmaxf(e, -200.f), k0);
    };
    for (int j = j0 + t; j < j1; j += U * 256) {
        u32x4 raw[U];
        float g[U][VE];
        if (zero) {
#pragma unroll
            for (int k = 0; k < U; k++)
#pragma unroll
                for (int e = 0; e < VE; e++) g[k][e] = 0.f;
        } else {
            if (j >= x.f0 && j + (U - 1) * 256 < min(x.f1, j1)) {
#pragma unroll
                for (int k = 0; k < U; k++) raw[k] = __builtin_nontemporal_load(x.v + j + k * 256);
            } else {
#pragma unroll
                for (int k = 0; k < U; k++) raw[k] = x.any(j + k * 256 < j1 ? j + k * 256 : x.nv);
            }
#pragma unroll
            for (int k = 0; k < U; k++)
#pragma unroll
                for (int e = 0; e < VE; e++) g[k][e] = grad(el_at<TYPE>(raw[k], e));
        }
#pragma unroll
        for (int k = 0; k < U; k++)
            if (j + k * 256 < j1) row_store<TYPE>(x, d, j + k * 256, g[k]);
    }
    __syncthreads();
    if (mine && !empty) {
        float g = 0.f;
        for (int j = 0; j < a.M; j++) g += si[j] == si[t] ? sg[j] : 0.f;
        el_store<TYPE>(const_cast<char *>(d.x), si[t], (zero ? 0.f : grad(xv)) + a.scale * g);
    }
}

// -------------------------------------------------------------- distillation --
// With S the teacher's ids, m_o and s_o the maximum and sum over the tokens
// outside S (over all of them when there is no remainder), M and s the whole
// row's, every token outside S has
//   d / dx_v = E_v (w_kd tau (Q F / s - q_r / s_o) + w_ce F / s),  E_v = 2^((x_v - m_o) c),
//   F = 2^((m_o - M) c)
// (one exponential; a second one where the cross-entropy has another temperature).
// The reference m_o keeps the remainder exact however little the student gives
// it, and summing it without the ids' terms, which a bitmap in LDS marks, keeps it
// from being a difference.  The ids and the target are written again afterwards.
// The teacher's side and the logarithms are in 64 bits, by one wave.
struct KdArgs {
    const void *logits;
    long long ld;
    int N, V, S, K, tail;
    float tau, w_kd, w_ce, scale;
    float c, c_lo;                // log2 e / tau = c + c_lo, c_lo > 0
    double inv;                   // 1 / tau
    int two;                      // the cross-entropy needs sums of its own: w_ce != 0 and tau != 1
    const int *t_ids;
    const float *t_logp;
    const int *tgt;
    float *rows;
    void *dlogits;
    long long ldd;
    int words;                    // tail: 32-bit words of a row's (or segment's) bitmap, a multiple of 4
    int keep;                     // first rounds of a row read twice that stay in LDS, behind the bitmap
    float *part;                  // S > 1: [N][S][4] sums, then [N][KD_XS] logits of ids and target
};
#define KD_XS (TLG_VOCAB_TOP + 1)
#define KD_C1 1.44269502162933349609375f       // log2 e = KD_C1 + KD_C1_LO
#define KD_C1_LO 1.925963033500e-8f

// 2^((x - m) (c + lo)): the small product first, so that the fused one rounds the
// whole exponent once (added to a rounded d c it would always be lost, and sums be off
// by the rounding of c in one direction).  lo > 0, so that -inf stays -inf.
__device__ __forceinline__ float kd_exp(float d, float c, float lo)
{
    return __builtin_amdgcn_exp2f(fmaf(d, c, d * lo));
}
// sums of a part at temperature tau and, with TWO, at the cross-entropy's 1
struct Kd { float m, s, s1; };
#define KD0 {-FLT_MAX, 0.f, 0.f}
template <bool TWO> __device__ __forceinline__ void kd_shift(Kd &a, float m, const KdArgs &k)
{
    const float d = a.m - m;
    a.s *= kd_exp(d, k.c, k.c_lo);
    if (TWO) a.s1 *= kd_exp(d, KD_C1, KD_C1_LO);
    a.m = m;
}
template <bool TWO> __device__ __forceinline__ Kd kd_wave(Kd a, const KdArgs &k)
{
    kd_shift<TWO>(a, wave_max(a.m), k);
    return Kd{a.m, wave_sum(a.s), TWO ? wave_sum(a.s1) : 0.f};
}
template <bool TWO> __device__ __forceinline__ Kd kd_join(const f32x4 *p, int n, const KdArgs &k)
{
    Kd r = {p[0][0], 0.f, 0.f};
#pragma unroll 4
    for (int w = 1; w < n; w++) r.m = fmaxf(r.m, p[w][0]);
#pragma unroll 4
    for (int w = 0; w < n; w++) {
        Kd a = {p[w][0], p[w][1], p[w][2]};
        kd_shift<TWO>(a, r.m, k);
        r.s += a.s;
        r.s1 += a.s1;
    }
    return r;
}
__device__ __forceinline__ double lane_double(double v, int lane)
{
    return __builtin_bit_cast(double, lane_u64(__builtin_bit_cast(u64, v), lane));
}
template <int CTRL> __device__ __forceinline__ double lane_move64(double v)
{
    const u64 b = __builtin_bit_cast(u64, v);
    const unsigned lo = __float_as_uint(lane_move<CTRL>(__uint_as_float((unsigned)b)));
    const unsigned hi = __float_as_uint(lane_move<CTRL>(__uint_as_float((unsigned)(b >> 32))));
    return __builtin_bit_cast(double, (u64)hi << 32 | lo);
}
__device__ __forceinline__ double wave_sum64(double v)          // as wave_sum
{
    v += lane_move64<0xB1>(v);
    v += lane_move64<0x4E>(v);
    v += lane_move64<0x141>(v);
    v += lane_move64<0x140>(v);
    return (lane_double(v, 0) + lane_double(v, 16)) + (lane_double(v, 32) + lane_double(v, 48));
}

// What a row's threads share: the waves' sums, the ids' sums, and the teacher's
// entries (id, logit, q, log q before normalising) between the first wave's two turns.
#define KD_HASH 128
template <int W> struct KdShared {
    f32x4 part[W], in;
    double Q, qr, lq0;            // sum q + q_r, q_r, what log q subtracts
    int flags, tgt;
    float xt;
    double q[TLG_VOCAB_TOP];
    float x[TLG_VOCAB_TOP], l[TLG_VOCAB_TOP];
    union {
        int id[TLG_VOCAB_TOP];
        unsigned seen[KD_HASH];
    };
};
// entries at all; the target among them; an id or target past V, an entry of NaN
// or +inf (which a maximum would not show); a target
enum { KD_ANY = 1, KD_HIT = 2, KD_BAD = 4, KD_CE = 8 };

// Rounds before the last one that a row read twice keeps in registers between its
// reads (4096 rows of 131072 in bf16: 468 us with none, 444 with 1, 436 with 2; a
// third takes the kernel past 64 registers, 457).
#define KD_HOLD 2
enum { KD_WHOLE = 0, KD_SUMS = 1, KD_GRAD = 2 };
// W waves on a row (PHASE KD_WHOLE) or on one of its S segments: KD_SUMS leaves
// the segment's sums, KD_GRAD joins them and writes the segment.  RES: a thread's
// part, at most U vectors, stays in registers, as exponentials, from the sums to
// the gradient; longer rows are read twice.  TWO: a cross-entropy at another
// temperature than the teacher's.
template <int TYPE, int W, int U, bool RES, bool TWO, int PHASE>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W, RES ? 4 : 8) void k_distill(KdArgs a)
{
    constexpr int VE = El<TYPE>::VE, TPR = 64 * W;
    __shared__ KdShared<W> shared[W == 1 ? 4 : 1];
    // tail: the support, a bit for each element; then the rounds kept
    extern __shared__ __attribute__((aligned(16))) unsigned all_bits[];
    const int lane = threadIdx.x & 63, wave = W == 1 ? 0 : threadIdx.x >> 6, t = W == 1 ? lane : threadIdx.x;
    const int slot = W == 1 ? threadIdx.x >> 6 : 0;
    KdShared<W> &sh = shared[slot];
    size_t r;
    int seg = 0;
    if constexpr (W == 1) {
        r = (size_t)blockIdx.x * 4 + slot;
        if (r >= (size_t)a.N) return;
    } else if constexpr (PHASE == KD_WHOLE)
        r = blockIdx.x;
    else {
        r = blockIdx.x / (unsigned)a.S;
        seg = blockIdx.x % (unsigned)a.S;
    }
    const Row<TYPE> x(a.logits, a.ld, r, a.V);
    const int per = PHASE == KD_WHOLE ? x.nv : ((x.nv + a.S - 1) / a.S + TPR - 1) / TPR * TPR;
    const int j0 = PHASE == KD_WHOLE ? 0 : min(seg * per, x.nv), j1 = PHASE == KD_WHOLE ? x.nv : min(j0 + per, x.nv);
    const float c = a.c;

    u32x4 raw[U];
    auto load = [&](int j, bool last) {
        if (j >= x.f0 && j + (U - 1) * TPR < min(x.f1, j1)) {
#pragma unroll
            for (int k = 0; k < U; k++) raw[k] = last ? __builtin_nontemporal_load(x.v + j + k * TPR) : x.v[j + k * TPR];
        } else {
#pragma unroll
            for (int k = 0; k < U; k++) raw[k] = x.any(j + k * TPR < j1 ? j + k * TPR : x.nv);
        }
    };
    // The first wave's loads of the teacher's entries, lane and lane + 64, go ahead of
    // the row's, so that the entries' logits are on their way while the row arrives.
    const int K = a.K;
    int id[2] = {-1, -1}, tgt = -1;
    float tl[2] = {-INFINITY, -INFINITY};
    if (wave == 0) {
        if (lane < K) {
            id[0] = a.t_ids[r * K + lane];
            tl[0] = a.t_logp[r * K + lane];
        }
        if (lane + 64 < K) {
            id[1] = a.t_ids[r * K + lane + 64];
            tl[1] = a.t_logp[r * K + lane + 64];
        }
        if (a.w_ce != 0.f) tgt = a.tgt[r];
    }
    if (PHASE != KD_GRAD) load(j0 + t, RES);

    unsigned *bits = all_bits + slot * a.words;
    float *xs = a.part + (size_t)a.N * a.S * 4 + r * KD_XS;              // S > 1
    if (PHASE != KD_GRAD && a.tail)
        for (int i = t; i < a.words; i += TPR) bits[i] = 0;
    if (wave == 0) {
        float xk[2] = {-INFINITY, -INFINITY}, xt = 0.f;
        for (int i = lane; i < KD_HASH; i += 64) sh.seen[i] = 0;
        int flags = __ballot(tgt >= a.V || id[0] >= a.V || id[1] >= a.V) ? KD_BAD : 0;
        if (tgt >= 0) flags |= KD_CE;
        if (__ballot(tgt >= 0 && (id[0] == tgt || id[1] == tgt))) flags |= KD_HIT;
        if (id[0] >= a.V) id[0] = -1;
        if (id[1] >= a.V) id[1] = -1;
#pragma unroll
        for (int k = 0; k < 2; k++)
            if (id[k] >= 0) xk[k] = PHASE == KD_GRAD ? xs[lane + 64 * k] : el_load<TYPE>(x.x, id[k]);
        if (tgt >= 0 && tgt < a.V) xt = PHASE == KD_GRAD ? xs[KD_XS - 1] : el_load<TYPE>(x.x, tgt);
        // A repeated id counts at its first place: looked for only where a set of
        // 32 KD_HASH bits says that there may be one.
        row_sync<1>();
        bool twice = false;
#pragma unroll
        for (int k = 0; k < 2; k++)
            if (id[k] >= 0) {
                const unsigned h = (unsigned)id[k] % (32 * KD_HASH);
                twice |= atomicOr(&sh.seen[h / 32], 1u << h % 32) >> h % 32 & 1;
            }
        if (__ballot(twice)) {
            const int was[2] = {id[0], id[1]};
            for (int j = 0; j < K; j++) {
                const int o = __builtin_amdgcn_readlane(j < 64 ? was[0] : was[1], j % 64);
                if (o == was[0] && j < lane) id[0] = -1;
                if (o == was[1] && j < lane + 64) id[1] = -1;
            }
#pragma unroll
            for (int k = 0; k < 2; k++)
                if (id[k] < 0) xk[k] = -INFINITY;
        }
        const int some = __popcll(__ballot(id[0] >= 0)) + __popcll(__ballot(id[1] >= 0));
        if (some) flags |= KD_ANY;
        if (__ballot((id[0] >= 0 && !(tl[0] < INFINITY)) || (id[1] >= 0 && !(tl[1] < INFINITY)))) flags |= KD_BAD;
        row_sync<1>();
        if constexpr (PHASE == KD_SUMS) {
            if (seg == 0) {
                xs[lane] = xk[0];
                xs[lane + 64] = xk[1];
                if (lane == 0) xs[KD_XS - 1] = xt;
            }
        } else {
            // q, its sum and the remainder; the ids' part of the sums, which the bitmap leaves out
            if (id[0] < 0) tl[0] = -INFINITY;
            if (id[1] < 0) tl[1] = -INFINITY;
            const float tm = a.tail ? 0.f : wave_max(fmaxf(tl[0], tl[1]));
            double q[2] = {0.0, 0.0};
            if (tm > -INFINITY) {
                q[0] = exp((double)tl[0] - tm);
                if (K > 64) q[1] = exp((double)tl[1] - tm);
            }
            double Q = wave_sum64(q[0] + q[1]), qr = 0.0, lq0 = 0.0;
            if (a.tail) {
                if (some && some < a.V && Q < 1.0) qr = 1.0 - Q;
                Q += qr;
            } else if (Q > 0.0) {
                const double n = 1.0 / Q;
                q[0] *= n;
                q[1] *= n;
                lq0 = Q;
                Q = 1.0;
            }
            Kd B = KD0;
            if (a.tail) {
                B.m = fmaxf(fmaxf(xk[0], xk[1]), -FLT_MAX);
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    B.s += kd_exp(xk[k] - B.m, c, a.c_lo);
                    if (TWO) B.s1 += kd_exp(xk[k] - B.m, KD_C1, KD_C1_LO);
                }
                B = kd_wave<TWO>(B, a);
            }
            if (lane == 0) {
                sh.Q = Q;
                sh.qr = qr;
                sh.lq0 = lq0;
                sh.in = f32x4{B.m, B.s, B.s1, 0.f};
                sh.xt = xt;
            }
#pragma unroll
            for (int k = 0; k < 2; k++)
                if (lane + 64 * k < K) {
                    sh.q[lane + 64 * k] = q[k];
                    sh.x[lane + 64 * k] = xk[k];
                    sh.l[lane + 64 * k] = tl[k] - tm;
                }
        }
        if (lane == 0) {
            sh.flags = flags;
            sh.tgt = tgt;
        }
        if (lane < K) sh.id[lane] = id[0];
        if (lane + 64 < K) sh.id[lane + 64] = id[1];
    }
    if (PHASE != KD_GRAD && a.tail) {
        row_sync<W>();
        for (int k = t; k < a.K; k += TPR) {
            const int g = sh.id[k] + x.sh - j0 * VE;
            if (sh.id[k] >= 0 && g >= 0 && g < a.words * 32) atomicOr(&bits[g >> 5], 1u << (g & 31));
        }
        row_sync<W>();
    }

    // sums
    Kd A = KD0;
    constexpr bool EXP = RES && U * VE <= 32 * (VE == 4 ? 2 : 1);      // kept as exponentials, else as they came
    float ex[EXP ? U * VE : 1], ex1[EXP && TWO ? U * VE : 1];
    int jl = j0 + t, round = 0;                         // the last round's vector; rounds
    u32x4 *kept = (u32x4 *)(all_bits + a.words);
    // rounds before the last whose vectors stay, as far as registers reach
    constexpr int HOLD = RES || PHASE != KD_WHOLE ? 0 : KD_HOLD;
    u32x4 hold[HOLD ? HOLD : 1][U];
    if constexpr (HOLD > 0)
#pragma unroll
        for (int h = 0; h < HOLD; h++)
#pragma unroll
            for (int k = 0; k < U; k++) hold[h][k] = raw[k];
    if constexpr (PHASE != KD_GRAD) {
        for (int j = j0 + t; RES ? j == j0 + t : j < j1; j += U * TPR) {
            if (!RES && j != j0 + t) {
                if constexpr (HOLD > 0)
#pragma unroll
                    for (int k = 0; k < U; k++) {
#pragma unroll
                        for (int h = HOLD - 1; h > 0; h--) hold[h][k] = hold[h - 1][k];
                        hold[0][k] = raw[k];
                    }
                load(j, false);
            }
            if (a.tail)
#pragma unroll
                for (int k = 0; k < U; k++) {
                    const int g = (j + k * TPR - j0) * VE;           // VE divides 32
                    unsigned b = j + k * TPR < j1 ? bits[g >> 5] >> (g & 31) & ((1u << VE) - 1) : 0;
                    if (b)
#pragma unroll
                        for (int e = 0; e < VE; e++)
                            if (b >> e & 1) {
                                if constexpr (TYPE == TLG_F32) raw[k][e] = El<TYPE>::NEG;
                                else raw[k][e >> 1] = e & 1 ? (raw[k][e >> 1] & 0xffffu) | El<TYPE>::NEG << 16
                                                            : (raw[k][e >> 1] & 0xffff0000u) | El<TYPE>::NEG;
                            }
                }
            if constexpr (HOLD > 0) {
                jl = j;
                if (round < a.keep)
#pragma unroll
                    for (int k = 0; k < U; k++) kept[(round * U + k) * TPR + t] = raw[k];
                round++;
            }
            float m = A.m;
#pragma unroll
            for (int k = 0; k < U; k++)
#pragma unroll
                for (int e = 0; e < VE; e++) m = fmaxf(m, el_at<TYPE>(raw[k], e));
            kd_shift<TWO>(A, m, a);
            if constexpr (RES && !EXP)
#pragma unroll
                for (int k = 0; k < U; k++) keep_packed(raw[k]);
            float rs = 0.f, rs1 = 0.f;                  // a vector's sums, then the round's, as in acc_vector
#pragma unroll
            for (int k = 0; k < U; k++) {
                float vs = 0.f, vs1 = 0.f;
#pragma unroll
                for (int e = 0; e < VE; e++) {
                    const float d = el_at<TYPE>(raw[k], e) - A.m, v = kd_exp(d, c, a.c_lo);
                    const float v1 = TWO ? kd_exp(d, KD_C1, KD_C1_LO) : 0.f;
                    vs = e ? vs + v : v;
                    if (TWO) vs1 = e ? vs1 + v1 : v1;
                    if constexpr (EXP) ex[k * VE + e] = v;
                    if constexpr (EXP && TWO) ex1[k * VE + e] = v1;
                    if constexpr (RES && !EXP)
                        if (e == VE - 1) keep_packed(raw[k]);
                }
                rs = k ? rs + vs : vs;
                if (TWO) rs1 = k ? rs1 + vs1 : vs1;
            }
            A.s += rs;
            if (TWO) A.s1 += rs1;
        }
    }
    const float mine = A.m;                             // the reference of ex, ex1
    if constexpr (PHASE != KD_GRAD) {
        A = kd_wave<TWO>(A, a);
        if (W > 1 && lane == 0) sh.part[wave] = f32x4{A.m, A.s, A.s1, 0.f};
    }
    row_sync<W>();
    if constexpr (W > 1) {
        if constexpr (PHASE == KD_GRAD) A = kd_join<TWO>((const f32x4 *)a.part + r * a.S, a.S, a);
        else A = kd_join<TWO>(sh.part, W, a);
    }
    if constexpr (PHASE == KD_SUMS) {
        if (t == 0) ((f32x4 *)a.part)[r * a.S + seg] = f32x4{A.m, A.s, A.s1, 0.f};
        return;
    }

    // the row's sums and coefficients
    const Kd B = {sh.in[0], sh.in[1], sh.in[2]};
    const float Q = (float)sh.Q, qr = (float)sh.qr;
    const int flags = sh.flags;
    const bool any = flags & KD_ANY, bad_id = flags & KD_BAD, ce = flags & KD_CE;
    const float M = fmaxf(A.m, B.m);
    const float F = kd_exp(A.m - M, c, a.c_lo), s = A.s * F + B.s * kd_exp(B.m - M, c, a.c_lo);
    float s1 = s;
    if (TWO) s1 = A.s1 * kd_exp(A.m - M, KD_C1, KD_C1_LO) + B.s1 * kd_exp(B.m - M, KD_C1, KD_C1_LO);
    const bool empty = s == 0.f, nothing = !any && !ce && !bad_id;
    const float ck = any ? a.w_kd * a.tau * a.scale : 0.f, cc = ce ? a.w_ce * a.scale : 0.f;
    const float rs = empty ? 0.f : __builtin_amdgcn_rcpf(s), r1 = empty ? 0.f : __builtin_amdgcn_rcpf(s1);
    const float kin = ck * Q * rs;                                         // inside S, reference M
    float kout = kin * F;                                                  // outside, reference m_o
    if (qr > 0.f && A.s > 0.f) kout -= ck * qr * __builtin_amdgcn_rcpf(A.s);
    if (!TWO) kout += cc * r1 * F;
    const float k1 = TWO ? cc * r1 : 0.f;                                  // of the second exponential, reference M
    if (bad_id) kout = NAN;
    auto outside = [&](float v) -> float {
        float g = kout * __builtin_amdgcn_exp2f((v - A.m) * c);
        if (TWO) g = fmaf(k1, __builtin_amdgcn_exp2f((v - M) * KD_C1), g);
        return g;
    };
    if (a.dlogits) {
        const Row<TYPE> d(a.dlogits, a.ldd, r, a.V);
        const bool zero = nothing || (empty && !bad_id);
        // of exponentials with a thread's own reference
        const float fk = kout * kd_exp(mine - A.m, c, a.c_lo), f1 = TWO ? k1 * kd_exp(mine - M, KD_C1, KD_C1_LO) : 0.f;
        // backwards: the sums' last rounds are here or the likeliest to be in the caches still
        if (PHASE == KD_GRAD) jl = j0 + t + (max(j1 - j0 - t, 1) - 1) / (U * TPR) * (U * TPR);
        for (int j = jl, i = 0; j >= j0; j -= U * TPR, i++) {
            if (!RES && !zero) {
                if (HOLD && i > HOLD && round - 1 - i < a.keep)
#pragma unroll
                    for (int k = 0; k < U; k++) raw[k] = kept[((round - 1 - i) * U + k) * TPR + t];
                else if (!HOLD || i > HOLD) load(j, true);
                else if (i > 0)
#pragma unroll
                    for (int k = 0; k < U; k++) {
                        raw[k] = hold[0][k];
#pragma unroll
                        for (int h = 0; h + 1 < HOLD; h++) hold[h][k] = hold[h + 1][k];
                    }
            }
#pragma unroll
            for (int k = 0; k < U; k++) {
                float g[VE];
#pragma unroll
                for (int e = 0; e < VE; e++) {
                    if constexpr (EXP) {
                        g[e] = fk * ex[k * VE + e];
                        if constexpr (TWO) g[e] = fmaf(f1, ex1[k * VE + e], g[e]);
                    } else
                        g[e] = outside(el_at<TYPE>(raw[k], e));
                    if (zero) g[e] = 0.f;
                }
                if (j + k * TPR < j1) row_store<TYPE>(x, d, j + k * TPR, g);
            }
            if (RES) break;
        }
        row_sync<W>();
        if (wave == 0 && !zero && !bad_id) {
            const int tgt = sh.tgt;
            for (int k = lane; k < K; k += 64) {
                const int id = sh.id[k], j = (id + x.sh) / VE;
                if (id >= 0 && j >= j0 && j < j1) {
                    const float p = kd_exp(sh.x[k] - M, c, a.c_lo);
                    const float p1 = TWO ? kd_exp(sh.x[k] - M, KD_C1, KD_C1_LO) : p;
                    float g = kin * p - ck * (float)sh.q[k] + (ce ? cc * (p1 * r1) : 0.f);
                    if (id == tgt) g -= cc;
                    el_store<TYPE>(const_cast<char *>(d.x), id, g);
                }
            }
            const int j = (tgt + x.sh) / VE;
            if (lane == 0 && ce && !(flags & KD_HIT) && j >= j0 && j < j1)
                el_store<TYPE>(const_cast<char *>(d.x), tgt, outside(sh.xt) - cc);
        }
    }
    if (!a.rows || seg != 0 || wave != 0) return;
    // The row's loss: log p_k = (x_k - M) / tau - log s, log q_k = l_k - log of their
    // sum.  One logarithm, of s, s_o, s1, q_r and that sum in lanes of their own.
    const double arg = lane == 0 ? (double)s : lane == 1 ? (double)A.s : lane == 2 ? (double)s1
                     : lane == 3 ? sh.qr : sh.lq0 > 0.0 ? sh.lq0 : 1.0;
    const double logs = log(arg), ls = lane_double(logs, 0), lo = lane_double(logs, 1), ls1 = lane_double(logs, 2),
                 lr = lane_double(logs, 3), lq = lane_double(logs, 4);
    double kl = 0.0;
    for (int k = lane; k < a.K; k += 64) {
        const double q = sh.q[k];
        if (q > 0.0 || q != q)
            kl += empty ? INFINITY : q * (((double)sh.l[k] - lq) - (((double)sh.x[k] - M) * a.inv - ls));
    }
    kl = wave_sum64(kl);
    if (lane != 0) return;
    if (sh.qr > 0.0) kl += empty ? INFINITY : sh.qr * (lr - (((double)A.m - M) * a.inv + lo - ls));
    double L = 0.0;
    if (any && a.w_kd != 0.f) L = (double)a.w_kd * a.tau * a.tau * kl;
    if (ce) L += (double)a.w_ce * (empty ? INFINITY : ls1 - ((double)sh.xt - M));
    if (s != s) L = NAN;
    a.rows[r] = bad_id ? NAN : nothing ? 0.f : (float)L;
}

// The mean of the row losses, summed in double in a fixed order by one workgroup:
// eight loads in flight a thread, one barrier.
__global__ __launch_bounds__(1024) void k_rows_mean(const float *__restrict__ rows, int n, float *__restrict__ out)
{
    __shared__ double s[16];
    const int t = threadIdx.x;
    double a = 0.0;
    for (int i = t; i < n; i += 8 * 1024) {
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; k++) v[k] = i + 1024 * k < n ? rows[i + 1024 * k] : 0.f;
#pragma unroll
        for (int k = 0; k < 8; k++) a += (double)v[k];
    }
    a = wave_sum64(a);
    if (t % 64 == 0) s[t / 64] = a;
    __syncthreads();
    if (t >= 64) return;
    a = wave_sum64(t < 16 ? s[t] : 0.0);
    if (t == 0) out[0] = (float)(a / n);
}

// -------------------------------------------------------------------- entries --
static int vb_check_out(const char *who, const void *logits, long long ld, const void *dlogits, int type,
                        long long ldd, int N, int V)
{
    if (ldd < V || (uintptr_t)dlogits % vb_size(type))
        return tlg_fail(TLG_EINVAL, "%s: dlogits %p ldd=%lld", who, dlogits, ldd);
    const uintptr_t b = vb_size(type), a0 = (uintptr_t)logits, d0 = (uintptr_t)dlogits;
    const uintptr_t a1 = a0 + ((uintptr_t)(N - 1) * ld + V) * b, d1 = d0 + ((uintptr_t)(N - 1) * ldd + V) * b;
    if (a0 < d1 && d0 < a1 && !(a0 == d0 && ld == ldd))
        return tlg_fail(TLG_EINVAL, "%s: dlogits overlaps logits without being the same rows", who);
    return TLG_OK;
}
static float f_of(double v) { return (float)v; }

// vectors of the longest row of a call: one more where rows do not all start on
// the 16-byte grid
static int vb_vectors(int type, const void *logits, long long ld, int V)
{
    const int b = (int)vb_size(type), ve = 16 / b;
    const bool on_grid = (uintptr_t)logits % 16 == 0 && ld * b % 16 == 0;
    return (V + (on_grid ? 0 : ve - 1) + ve - 1) / ve;
}
// Segments of a row.  A workgroup alone takes 12 us for a row of 8192 vectors and
// 19 for one of 16384 (log probabilities, 20 alternatives); from 8192 vectors on, few
// rows are cut into pieces of 2048 until 512 workgroups work (one row of 16384: 12.5
// us, 128 of them 27.8 -> 20.2).  Shorter rows and 512 of them are not: the second
// launch costs more than it saves (48 rows of 4000 vectors: 11.3 us whole, 12.4 cut).
// Pieces of 1024, 2048 and 4096 vectors: one row of 16384 takes 13.0, 12.3 and 13.5 us,
// 64 take 16.3, 16.3 and 16.6; distillation 12.3, 13.9, 18.2 and 20.9, 20.8, 23.1.
#define VB_CUT 8192
#define VB_PIECE 2048
#define VB_FILL 512
static int vb_segments(int type, int N, int V, int most)
{
    const int ve = type == TLG_F32 ? 4 : 8;
    if (V / ve < VB_CUT) return 1;
    const long long by_rows = (VB_FILL + N - 1) / N, by_size = (V / ve + VB_PIECE - 1) / VB_PIECE;
    const long long s = by_rows < by_size ? by_rows : by_size;
    return s > most ? most : (int)s;
}

#define BY_TYPE(grid, block, lds, a, K0, ...)                                                                       \
    do {                                                                                                            \
        if (type == TLG_F32) hipLaunchKernelGGL((K0<TLG_F32 __VA_ARGS__>), dim3(grid), dim3(block), lds, st, a);    \
        else if (type == TLG_F16) hipLaunchKernelGGL((K0<TLG_F16 __VA_ARGS__>), dim3(grid), dim3(block), lds, st, a); \
        else hipLaunchKernelGGL((K0<TLG_BF16 __VA_ARGS__>), dim3(grid), dim3(block), lds, st, a);                   \
    } while (0)

#define BY_16(grid, block, lds, a, K0, ...)                                                                         \
    do {                                                                                                            \
        if (type == TLG_F16) hipLaunchKernelGGL((K0<TLG_F16 __VA_ARGS__>), dim3(grid), dim3(block), lds, st, a);    \
        else hipLaunchKernelGGL((K0<TLG_BF16 __VA_ARGS__>), dim3(grid), dim3(block), lds, st, a);                   \
    } while (0)

static int lp_segments(int type, int N, int V, int K)
{
    const int most = K > 0 && LP_JOIN / K < 64 ? LP_JOIN / K : 64;
    return vb_segments(type, N, V, most);
}

extern "C" size_t tlg_logprobs_ws_bytes(int type, int N, int V, int K)
{
    if (N <= 0 || V <= 0 || K < 0) return 0;
    const size_t S = lp_segments(type, N, V, K);
    return S > 1 ? (size_t)N * S * (16 + 8 * (size_t)K) : 0;
}

// One wave per row where the rows are short and many: no barriers, and a lane's
// four (or, of fp32, eight) vectors stay in registers; 4096 rows of 2048 fp32 values
// with 8 alternatives take 11.2 us so, 13.2 with the rows read again, 16.5 with four
// waves each.  Four waves win for fewer rows (2048 columns, 8 alternatives, fp32: 512
// rows 5.8 against 7.1 us, 1024 equal at 7.5, 2048 11.0 against 8.7; bf16: 6.7 equal at
// 512, 8.4 against 7.3 at 1024) and for many alternatives, whose bound one wave finds
// lane by lane and whose list overflows near 48 (fp32: 20 of 1024 rows 7.9 against 8.4,
// of 1536 9.5 against 9.2; 32 of 1024 8.3 against 10.1, of 2048 12.0 against 11.5; 40
// of 2048 12.7 against 13.9, of 4096 19.5 against 17.9; 48 of 4096 20.4 against 26.9).
// Rows that one wave reads again need more of all that (4096 rows of 2800 fp32 values: 8
// alternatives 16.0 us, four waves 17.9; 20: 18.3, 18.8; 32: 22.0, 20.5; 2048 such
// rows with 20: 14.0, 12.4; 4096 of 16384 fp32 values: 58, 49).  Four waves too keep four
// vectors a thread (900 rows of 4000 fp32 values: 8.2 us, 9.1 read again).
template <bool TOP> static void lp_launch(const LpArgs &a, int type, int nv, hipStream_t st)
{
    const unsigned rows = (unsigned)a.N;
    const bool wave = a.K <= 40 && rows >= 1024 && rows >= 64u * a.K;
    if (a.S > 1) {
        BY_TYPE(rows * a.S, 256, 0, a, k_logprobs, , 4, 4, false, TOP);
        BY_TYPE(rows, 256, 0, a, k_logprobs_join, , TOP);
    } else if (wave && nv <= 256)
        BY_TYPE((rows + 3) / 4, 256, 0, a, k_logprobs, , 1, 4, true, TOP);
    else if (wave && nv <= 512 && type == TLG_F32)
        hipLaunchKernelGGL((k_logprobs<TLG_F32, 1, 8, true, TOP>), dim3((rows + 3) / 4), dim3(256), 0, st, a);
    else if (wave && nv <= 1024 && rows >= 2 * (unsigned)nv && rows >= 192u * a.K)
        BY_TYPE((rows + 3) / 4, 256, 0, a, k_logprobs, , 1, 4, false, TOP);
    else if (nv <= 1024)
        BY_TYPE(rows, 256, 0, a, k_logprobs, , 4, 4, true, TOP);
    else
        BY_TYPE(rows, 256, 0, a, k_logprobs, , 4, 4, false, TOP);
}

extern "C" int tlg_dev_logprobs(const void *logits, int type, long long ld, int N, int V, float scale, const int *ids,
                                int M, float *logp, float *lse2, float *entropy, int K, int *top_ids, float *top_logp,
                                void *ws, size_t ws_bytes, void *stream)
{
    int rc;
    if ((rc = vb_check("logprobs", logits, type, ld, N, V))) return rc;
    if (!vb_positive(scale)) return tlg_fail(TLG_EINVAL, "logprobs: scale %g", scale);
    if (M < 0 || M > TLG_VOCAB_IDS || K < 0 || K > TLG_VOCAB_TOP)
        return tlg_fail(TLG_EINVAL, "logprobs: M=%d K=%d", M, K);
    if (N == 0) return TLG_OK;
    if ((M && (!ids || !logp)) || (K && (!top_ids || !top_logp)))
        return tlg_fail(TLG_EINVAL, "logprobs: NULL ids, logp, top_ids or top_logp");
    if ((rc = vb_check_ws("logprobs", ws, ws_bytes, tlg_logprobs_ws_bytes(type, N, V, K)))) return rc;
    if ((rc = tlg_ensure_init())) return rc;
    const double c = (double)scale * 1.4426950408889634;
    LpArgs a = {logits, ld, N, V, lp_segments(type, N, V, K), scale, f_of(c), 0.f, ids, M, logp, lse2, entropy, K,
                top_ids, top_logp, (float *)ws, nullptr};
    a.kappa = f_of(0.6931471805599453 * (c - (double)a.c) / c);
    a.keys = (u64 *)(a.part + (size_t)N * a.S * 4);
    hipStream_t st = ST(stream);
    const int nv = vb_vectors(type, logits, ld, V);
    if (K) lp_launch<true>(a, type, nv, st);
    else lp_launch<false>(a, type, nv, st);
    LAUNCH_CHECK();
    return TLG_OK;
}

extern "C" int tlg_dev_logprobs_bwd(const void *logits, int type, long long ld, int N, int V, float scale,
                                    const int *ids, int M, const float *lse2, const float *entropy,
                                    const float *dlogp, const float *dlse, const float *dentropy, void *dlogits,
                                    long long ldd, void *stream)
{
    int rc;
    if ((rc = vb_check("logprobs_bwd", logits, type, ld, N, V))) return rc;
    if (!vb_positive(scale)) return tlg_fail(TLG_EINVAL, "logprobs_bwd: scale %g", scale);
    if (M < 0 || M > TLG_VOCAB_IDS) return tlg_fail(TLG_EINVAL, "logprobs_bwd: M=%d", M);
    if (N == 0) return TLG_OK;
    if (!lse2 || !dlogits || (M && (!ids || !dlogp)) || (dentropy && !entropy))
        return tlg_fail(TLG_EINVAL, "logprobs_bwd: NULL lse2, dlogits, ids, dlogp or entropy");
    if ((rc = vb_check_out("logprobs_bwd", logits, ld, dlogits, type, ldd, N, V))) return rc;
    if ((rc = tlg_ensure_init())) return rc;
    const int S = (vb_vectors(type, logits, ld, V) + BW_SEG - 1) / BW_SEG;
    const LpBwdArgs a = {logits, ld, V, S, scale, f_of((double)scale * 1.4426950408889634), ids, M, lse2, entropy,
                         dlogp, dlse, dentropy, dlogits, ldd};
    hipStream_t st = ST(stream);
    BY_TYPE((unsigned)N * S, 256, 0, a, k_logprobs_bwd, );
    LAUNCH_CHECK();
    return TLG_OK;
}

// Distillation's uncut rows have up to sixteen waves each, so that only fewer or
// longer rows gain by a second launch: 16384 vectors take 12.8 us cut and 17.6 whole for
// one row, 19.1 and 20.6 for 64, 24.4 and 23.0 for 128.
static int kd_segments(int type, int N, int V)
{
    return (long long)N * 256 <= V / (type == TLG_F32 ? 4 : 8) ? vb_segments(type, N, V, 64) : 1;
}

// The first rounds (of U vectors a thread) of a row read twice that fit a workgroup's
// share of the LDS, 2048 threads on a CU of 160 KB, beside the bitmap and the shared rest
// (4096 rows of 65536 fp32 values, two temperatures: 428 us without, 406; 301 rows of
// 50021: 37.6, 35.9; of 65536 in bf16, where the caches hold them too, 221, 226).
static int kd_keep(int threads, int U, size_t bits)
{
    static_assert(sizeof(KdShared<16>) <= 4096 && sizeof(KdShared<8>) <= 4096, "the shared rest");
    const size_t share = 160 * 1024 / (2048 / threads), rest = bits + 4096;
    return rest < share ? (int)((share - rest) / ((size_t)threads * U * 16)) : 0;
}

// Rows of up to 4096 vectors (of 2048, with 16-bit types and two temperatures) stay in
// registers between sums and gradient, on as few waves as hold them: 4096 rows of 2048
// fp32 values take 19.7 us on one wave and 25.0 read twice by four, of 16384 101 against
// 110, of 32768 in bf16 107 against 131, but of 20000 in bf16 with two temperatures 115
// against 104.  In longer ones a row's waves wait for each other with nothing else to
// work on their CU (256 rows of 50021 fp32 values: 30.9 us, 26.5 read twice).  These
// are read twice, by sixteen waves, so that the rows in work (two on a CU) fit the
// last-level cache (4096 rows of 131072 in bf16: 468 us, with eight waves 502, with four
// 583), the last rounds in registers (436) and the first in LDS (430).  With two
// temperatures and 16-bit types eight waves are faster (501 against 521 us).
// Borders: one wave a row against four at 1536, 2048 and 4096 rows of 2048 fp32 values
// 11.1, 11.9, 19.2 and 10.6, 12.1, 21.2 us (bf16 10.0, 10.6, 15.6 and 9.8, 10.8, 17.1); two
// vectors a thread against four at 512 vectors 6.0 and 6.5 us for 64 rows, 10.7 and 11.0
// for 1500; eight a thread on four waves, on eight waves, and read twice at 2048 vectors
// of fp32 8.9, 9.2, 9.1 for 64 rows, 10.5, 11.4, 11.9 for 300 and 53, 62, 64 for 4096.
template <bool TWO> static void kd_launch(KdArgs a, int type, int nv, size_t lds, hipStream_t st)
{
    const unsigned rows = a.N;
    const bool f32 = type == TLG_F32;
    if (a.S > 1) {
        BY_TYPE(rows * a.S, 256, lds, a, k_distill, , 4, 4, false, TWO, KD_SUMS);
        BY_TYPE(rows * a.S, 256, 0, a, k_distill, , 4, 4, false, TWO, KD_GRAD);
    } else if (nv <= 256 && rows >= 2048)
        BY_TYPE((rows + 3) / 4, 256, 4 * lds, a, k_distill, , 1, 4, true, TWO, KD_WHOLE);
    else if (nv <= 512 && f32 && rows >= 2048)
        hipLaunchKernelGGL((k_distill<TLG_F32, 1, 8, true, TWO, KD_WHOLE>), dim3((rows + 3) / 4), dim3(256), 4 * lds,
                           st, a);
    else if (nv <= 512)
        BY_TYPE(rows, 256, lds, a, k_distill, , 4, 2, true, TWO, KD_WHOLE);
    else if (nv <= 1024)
        BY_TYPE(rows, 256, lds, a, k_distill, , 4, 4, true, TWO, KD_WHOLE);
    else if (nv <= 2048)
        BY_TYPE(rows, 256, lds, a, k_distill, , 4, 8, true, TWO, KD_WHOLE);
    else if (nv <= 4096 && f32)
        hipLaunchKernelGGL((k_distill<TLG_F32, 8, 8, true, TWO, KD_WHOLE>), dim3(rows), dim3(512), lds, st, a);
    else if (nv <= 4096 && !TWO)
        BY_16(rows, 512, lds, a, k_distill, , 8, 8, true, false, KD_WHOLE);
    else if (TWO && !f32) {
        a.keep = kd_keep(512, 2, lds);
        BY_16(rows, 512, lds + a.keep * 16384, a, k_distill, , 8, 2, false, TWO, KD_WHOLE);
    } else {
        a.keep = kd_keep(1024, 2, lds);
        if (f32)
            hipLaunchKernelGGL((k_distill<TLG_F32, 16, 2, false, TWO, KD_WHOLE>), dim3(rows), dim3(1024),
                               lds + a.keep * 32768, st, a);
        else
            BY_16(rows, 1024, lds + a.keep * 32768, a, k_distill, , 16, 2, false, false, KD_WHOLE);
    }
}

extern "C" size_t tlg_distill_ws_bytes(int type, int N, int V)
{
    if (N <= 0 || V <= 0) return 0;
    const size_t S = kd_segments(type, N, V);
    return S > 1 ? (size_t)N * (S * 16 + KD_XS * 4) : 0;
}

extern "C" int tlg_dev_distill(const void *logits, int type, long long ld, int N, int V, const int *t_ids,
                               const float *t_logp, int K, int tail, float temp, float w_kd, const int *tgt,
                               float w_ce, float *rows, float *loss, void *dlogits, long long ldd, float scale,
                               void *ws, size_t ws_bytes, void *stream)
{
    int rc;
    if ((rc = vb_check("distill", logits, type, ld, N, V))) return rc;
    if (!vb_positive(temp) || !isfinite(w_kd) || !isfinite(w_ce) || !isfinite(scale))
        return tlg_fail(TLG_EINVAL, "distill: temp %g w_kd %g w_ce %g scale %g", temp, w_kd, w_ce, scale);
    if (K < 0 || K > TLG_VOCAB_TOP) return tlg_fail(TLG_EINVAL, "distill: K=%d", K);
    if (N == 0) return TLG_OK;
    if ((K && (!t_ids || !t_logp)) || (w_ce != 0.f && !tgt))
        return tlg_fail(TLG_EINVAL, "distill: NULL t_ids, t_logp or tgt");
    if ((!rows && !dlogits) || (loss && !rows)) return tlg_fail(TLG_EINVAL, "distill: NULL rows");
    if (dlogits && (rc = vb_check_out("distill", logits, ld, dlogits, type, ldd, N, V))) return rc;
    if ((rc = vb_check_ws("distill", ws, ws_bytes, tlg_distill_ws_bytes(type, N, V)))) return rc;
    if ((rc = tlg_ensure_init())) return rc;
    const double c = 1.4426950408889634 / (double)temp;
    const int nv = vb_vectors(type, logits, ld, V), ve = type == TLG_F32 ? 4 : 8, S = kd_segments(type, N, V);
    float hi = f_of(c);                                  // below c, so that what is left is positive
    if ((double)hi >= c) hi = nextafterf(hi, 0.f);
    KdArgs a = {logits, ld, N, V, S, K, tail ? 1 : 0, temp, w_kd, w_ce, scale, hi, f_of(c - (double)hi),
                1.0 / (double)temp, w_ce != 0.f && temp != 1.f, t_ids, t_logp, tgt, rows, dlogits, ldd, 0, 0,
                (float *)ws};
    hipStream_t st = ST(stream);
    // a segment is a multiple of 256 vectors, see the kernel
    const int per = S > 1 ? ((nv + S - 1) / S + 255) / 256 * 256 : nv;
    a.words = tail ? ((per * ve + 31) / 32 + 3) & ~3 : 0;
    const size_t lds = (size_t)a.words * 4;
    if (a.two) kd_launch<true>(a, type, nv, lds, st);
    else kd_launch<false>(a, type, nv, lds, st);
    if (loss) hipLaunchKernelGGL(k_rows_mean, dim3(1), dim3(1024), 0, st, (const float *)rows, N, loss);
    LAUNCH_CHECK();
    return TLG_OK;
}
