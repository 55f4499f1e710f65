// tlg_verify.hip -- verification of drafted tokens by sampling (include/tlserve.h).
//
// With p = softmax(s x) of the target's row and q of the draft model's, row i
// keeps its draft d iff u q(d) < p(d), which happens with probability min(1, p /
// q); the first row that does not gives the token argmax_v w_v / e_v over
// independent exponentials e, w = max(0, p - q).  The smallest of the times e_v /
// w_v belongs to v with probability w_v / sum w, so that no sum over the vocabulary
// stands between the numbers given and the token: one token's rounding cannot
// shift the borders of all later ones, as it does in a cumulative sum.
//
// Two launches: the sums of every row (bound by HBM, each logit read once), then
// for each sequence the tests of its rows, a scalar each, and the race over the one
// row that ends it; a third joins races that are cut over workgroups.  Short rows: one.
// Measured: 898 rows of 131072 bf16 logits, 674 of them with the draft model's, 118 to 125 us (sums 72
// us for 412 MB, 5.7 TB/s; races 44 us, whose rows are read again; join 4 us); 168 rows of 32003 fp16
// logits 22 us, three launches of a few rounds of loads each.
#include "tlg_internal.h"
#include "tlg_rows.h"
#include "../../include/tlserve.h"
#include <float.h>

#define ST(s) ((hipStream_t)(s))
#define LAUNCH_CHECK() TLG_HIP(hipGetLastError())
#define SV_THREADS 256

// VE elements from any element of a row (16 bytes of the elements' alignment)
typedef unsigned u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
template <int TYPE> __device__ __forceinline__ u32x4 sv_load(const char *x, int i)
{
    return *(const u32x4_any *)(x + (size_t)i * El<TYPE>::SZ);
}

struct SvSum { float m, s; };         // maximum, sum e^(scale (x - m)); s = 0: nothing but -inf, NaN: NaN or +inf in it
struct SvArgs {
    const void *x, *y;
    long long ld, ldy, ldn;
    float scale, c, dscale, dc;       // c = scale log2 e
    int N, V, B, S, T;                // S segments of a row's sums, T of a race
    const int *row0, *draft;
    const float *u, *noise;
    int *tokens, *accepted;
    float *logp;
    SvSum *part;                      // [N][2][S]
    f32x4 *best, *info;               // [B][T] keys and tokens of both races, [B] of the row that ends a sequence
};

// 2^((x - m) c): the difference first, so that any logits and scales do
__device__ __forceinline__ float sv_term(float x, float m, float c) { return __builtin_amdgcn_exp2f((x - m) * c); }
// a maximum that differences can be formed with
__device__ __forceinline__ float sv_ref(float m) { return fmaxf(m, -FLT_MAX); }

__device__ __forceinline__ SvSum sv_join(const SvSum *p, int n, float c)
{
    SvSum r = p[0];
    for (int k = 1; k < n; k++) r.m = fmaxf(r.m, p[k].m);
    r.s = 0.f;
    const float ref = sv_ref(r.m);
    for (int k = 0; k < n; k++) r.s += p[k].s * sv_term(sv_ref(p[k].m), ref, c);
    return r;
}

// ---------------------------------------------------------------- row sums --
// The sums of vectors [lo, hi) of row x over TH threads, and, with the flag, of the
// elements behind the last vector; the thread's own, t of TH.
template <int TYPE, int TH>
__device__ __forceinline__ SvSum sv_some(const char *x, int V, int lo, int hi, bool tail, float c, int t)
{
    constexpr int VE = El<TYPE>::VE, U = 4;
    float m = -INFINITY, s = 0.f;
    for (int j = lo + t; j < hi; j += U * TH) {
        u32x4 q[U];
#pragma unroll
        for (int k = 0; k < U; k++) {
            const int i = j + k * TH;
            q[k] = sv_load<TYPE>(x, (i < hi ? i : j) * VE);      // beyond the end: a vector taken already, left out below
        }
        float n = m;
#pragma unroll
        for (int k = 0; k < U; k++)
#pragma unroll
            for (int e = 0; e < VE; e++) n = fmaxf(n, el_at<TYPE>(q[k], e));
        const float ref = sv_ref(n);
        float sum = 0.f;
#pragma unroll
        for (int k = 0; k < U; k++) {
            float v[VE];
#pragma unroll
            for (int e = 0; e < VE; e++) v[e] = sv_term(el_at<TYPE>(q[k], e), ref, c);
#pragma unroll
            for (int w = VE / 2; w; w /= 2)
#pragma unroll
                for (int e = 0; e < w; e++) v[e] += v[e + w];
            sum += j + k * TH < hi ? v[0] : 0.f;
        }
        s = s * sv_term(sv_ref(m), ref, c) + sum;
        m = n;
    }
    if (tail && t < V % VE) {
        const float v = el_load<TYPE>(x, V / VE * VE + t), n = fmaxf(m, v), ref = sv_ref(n);
        s = s * sv_term(sv_ref(m), ref, c) + sv_term(v, ref, c);
        m = n;
    }
    return SvSum{m, s};
}
__device__ __forceinline__ SvSum sv_wave(SvSum p, float c)
{
    const float M = wave_max(p.m);
    return SvSum{M, wave_sum(p.s * sv_term(sv_ref(p.m), sv_ref(M), c))};
}
// Segment blockIdx.x % S of row blockIdx.x / S; blockIdx.y 1: of the draft model's.
template <int TYPE> __global__ __launch_bounds__(SV_THREADS) void k_sv_sums(SvArgs a)
{
    const int r = blockIdx.x / a.S, seg = blockIdx.x % a.S, of = blockIdx.y, t = threadIdx.x;
    if (of && a.draft[r] < 0) return;
    const char *x = (const char *)(of ? a.y : a.x) + (long long)r * (of ? a.ldy : a.ld) * El<TYPE>::SZ;
    const float c = of ? a.dc : a.c;
    const int nv = a.V / El<TYPE>::VE, lo = (int)((long long)nv * seg / a.S), hi = (int)((long long)nv * (seg + 1) / a.S);
    const SvSum p = sv_wave(sv_some<TYPE, SV_THREADS>(x, a.V, lo, hi, seg == a.S - 1, c, t), c);
    __shared__ SvSum part[SV_THREADS / 64];
    if (t % 64 == 0) part[t / 64] = p;
    __syncthreads();
    if (t == 0) a.part[((size_t)r * 2 + of) * a.S + seg] = sv_join(part, SV_THREADS / 64, c);
}

// -------------------------------------------------------------------- tests --
__device__ __forceinline__ bool sv_none(const SvSum &s) { return !(s.s > 0.f && s.s < INFINITY); }
__device__ __forceinline__ float sv_logp(float x, const SvSum &s, float scale)
{
    return x == -INFINITY ? x : lp_scaled(x, s.m, scale) - logf(s.s);
}
enum { SV_KEEP = 0, SV_PLAIN = 1, SV_REFUSED = 2, SV_NONE = 3 };
// What row r does with its draft: u q(d) < p(d) as u sum_p < sum_q e^(s (x_d - m) - s' (y_d -
// m')), whose exponent needs 64 bits where the logits are far apart.
struct SvTest { int how; float lp; SvSum p, q; };
template <int TYPE> __device__ __forceinline__ SvTest sv_test(const SvArgs &a, int r, bool last)
{
    SvTest o = {SV_NONE, 0.f, sv_join(a.part + (size_t)r * 2 * a.S, a.S, a.c), {0.f, 1.f}};
    const int d = last ? -1 : a.draft[r];
    const float u = a.u[r];
    if (sv_none(o.p)) return o;
    o.how = SV_PLAIN;
    if (d < 0) return o;
    const float x = d < a.V ? el_load<TYPE>((const char *)a.x + (long long)r * a.ld * El<TYPE>::SZ, d) : -INFINITY;
    double z = ((double)x - (double)o.p.m) * a.scale, sq = 1.0;
    if (a.y) {
        const float y = d < a.V ? el_load<TYPE>((const char *)a.y + (long long)r * a.ldy * El<TYPE>::SZ, d) : -INFINITY;
        o.q = sv_join(a.part + ((size_t)r * 2 + 1) * a.S, a.S, a.dc);
        if (!(o.q.s >= 0.f && o.q.s < INFINITY)) {
            o.how = SV_NONE;
            return o;
        }
        z -= o.q.s == 0.f ? -INFINITY : ((double)y - (double)o.q.m) * a.dscale;
        if (o.q.s > 0.f) sq = o.q.s;
    }
    o.lp = sv_logp(x, o.p, a.scale);
    const bool keep = u == 0.f ? x > -INFINITY : (double)u * o.p.s < sq * exp(z);
    o.how = keep ? SV_KEEP : SV_REFUSED;
    return o;
}

// ---------------------------------------------------------------------- race --
struct SvBest { float k, kp; int v, vp; };             // the race of w and, for no w at all, of p
__device__ __forceinline__ void sv_better(SvBest &a, const SvBest &b)
{
    if (b.k > a.k || (b.k == a.k && b.v < a.v)) a.k = b.k, a.v = b.v;
    if (b.kp > a.kp || (b.kp == a.kp && b.vp < a.vp)) a.kp = b.kp, a.vp = b.vp;
}
__device__ __forceinline__ SvBest sv_lane(const SvBest &b, int o)
{
    return SvBest{__shfl_xor(b.k, o), __shfl_xor(b.kp, o), __shfl_xor(b.v, o), __shfl_xor(b.vp, o)};
}
struct SvRow {                                         // the row that ends a sequence
    const char *x, *y;                                 // y NULL: q is no distribution, or is left out
    const float *e;
    SvSum p, q;
    float c, dc, rp, rq;
    int point;                                         // a token of weight 0, or -1
};
__device__ __forceinline__ void sv_try(SvBest &b, const SvRow &w, float x, float y, float e, int v)
{
    const float p = sv_term(x, w.p.m, w.c) * w.rp;
    float g = p;
    if (w.y) g = p - sv_term(y, sv_ref(w.q.m), w.dc) * w.rq;
    if (v == w.point) g = 0.f;
    const float r = e >= 1e-30f && e <= 1e30f ? __builtin_amdgcn_rcpf(e) : 0.f, k = g * r, kp = p * r;
    if (k > b.k) b.k = k, b.v = v;
    if (kp > b.kp) b.kp = kp, b.vp = v;
}
// U vectors of each row in flight
template <int TYPE, int TH> __device__ __forceinline__ SvBest sv_race(const SvRow &w, int V, int seg, int T)
{
    constexpr int VE = El<TYPE>::VE, U = 2;
    const int nv = V / VE, lo = (int)((long long)nv * seg / T), hi = (int)((long long)nv * (seg + 1) / T), t = threadIdx.x;
    SvBest b = {0.f, 0.f, V, V};
    for (int j = lo + t; j < hi; j += U * TH) {
        u32x4 x[U], y[U];
        f32x4 e[U][VE / 4];
#pragma unroll
        for (int k = 0; k < U; k++) {
            const int i = j + k * TH < hi ? j + k * TH : j;
            x[k] = sv_load<TYPE>(w.x, i * VE);
            y[k] = w.y ? sv_load<TYPE>(w.y, i * VE) : x[k];
#pragma unroll
            for (int n = 0; n < VE / 4; n++) e[k][n] = *(const f32x4_any *)(w.e + i * VE + 4 * n);
        }
#pragma unroll
        for (int k = 0; k < U; k++)
            if (j + k * TH < hi) {
#pragma unroll
                for (int i = 0; i < VE; i++)
                    sv_try(b, w, el_at<TYPE>(x[k], i), el_at<TYPE>(y[k], i), e[k][i / 4][i % 4], (j + k * TH) * VE + i);
            }
    }
    if (seg == T - 1 && t < V % VE) {
        const int v = nv * VE + t;
        sv_try(b, w, el_load<TYPE>(w.x, v), w.y ? el_load<TYPE>(w.y, v) : 0.f, w.e[v], v);
    }
    return b;
}
// the token, its log p and how many drafts were kept; n is the row's place in its sequence
template <int TYPE>
__device__ __forceinline__ void sv_put(const SvArgs &a, int b, int r, int n, const SvBest &w, float m, float s)
{
    const int v = (unsigned)w.v < (unsigned)a.V ? w.v : (unsigned)w.vp < (unsigned)a.V ? w.vp : -1;
    a.tokens[r] = v;
    if (a.logp)
        a.logp[r] = v < 0 ? NAN : sv_logp(el_load<TYPE>((const char *)a.x + (long long)r * a.ld * El<TYPE>::SZ, v),
                                                 SvSum{m, s}, a.scale);
    if (a.accepted) a.accepted[b] = n;
}
__device__ __forceinline__ void sv_rows(const SvArgs &a, int b, int &lo, int &hi)
{
    lo = min(max(a.row0[b], 0), a.N);
    hi = min(max(a.row0[b + 1], lo), a.N);
}

// Segment seg of the race of sequence b, TH threads; segment 0 writes the rows besides the
// one that ends the sequence.
template <int TYPE, int TH> __device__ __forceinline__ void sv_pick(const SvArgs &a, int b, int seg)
{
    const int t = threadIdx.x;
    __shared__ int stop;
    __shared__ SvTest at_stop;
    __shared__ SvBest part[TH / 64];
    int lo, hi;
    sv_rows(a, b, lo, hi);
    if (lo == hi) {
        if (seg == 0 && t == 0 && a.accepted) a.accepted[b] = 0;
        if (seg == 0 && t == 0 && a.T > 1) a.info[b] = f32x4{__int_as_float(-1), 0.f, 0.f, 0.f};
        return;
    }
    if (t == 0) stop = hi;
    __syncthreads();
    for (int r0 = lo; r0 < hi; r0 += TH) {
        const int r = r0 + t;
        SvTest h = {SV_KEEP, 0.f, {0.f, 1.f}, {0.f, 1.f}};
        if (r < hi) h = sv_test<TYPE>(a, r, r == hi - 1);
        if (h.how != SV_KEEP) atomicMin(&stop, r);
        __syncthreads();
        const int at = stop;
        if (r == at) at_stop = h;
        if (seg == 0 && r < hi && r != at) {
            a.tokens[r] = r < at ? a.draft[r] : -1;
            if (a.logp) a.logp[r] = r < at ? h.lp : 0.f;
        }
        __syncthreads();
    }
    // the last row keeps nothing, so stop < hi
    const int r = stop, h = at_stop.how;
    SvRow w;
    w.x = (const char *)a.x + (long long)r * a.ld * El<TYPE>::SZ;
    w.y = nullptr;
    w.e = a.noise + (long long)b * a.ldn;
    w.p = at_stop.p;
    w.q = SvSum{0.f, 1.f};
    w.c = a.c;
    w.dc = a.dc;
    w.rp = 1.f / w.p.s;
    w.rq = 0.f;
    w.point = -1;
    if (h == SV_REFUSED) {
        if (!a.y) w.point = a.draft[r];
        else {
            w.q = at_stop.q;
            if (w.q.s > 0.f) {
                w.y = (const char *)a.y + (long long)r * a.ldy * El<TYPE>::SZ;
                w.rq = 1.f / w.q.s;
            }
        }
    }
    SvBest k = {0.f, 0.f, a.V, a.V};
    if (h != SV_NONE) k = sv_race<TYPE, TH>(w, a.V, seg, a.T);
#pragma unroll
    for (int o = 32; o; o /= 2) sv_better(k, sv_lane(k, o));
    if (t % 64 == 0) part[t / 64] = k;
    __syncthreads();
    if (t) return;
    for (int i = 1; i < TH / 64; i++) sv_better(k, part[i]);
    if (a.T == 1) {
        sv_put<TYPE>(a, b, r, r - lo, k, w.p.m, w.p.s);
        return;
    }
    a.best[(size_t)b * a.T + seg] = f32x4{k.k, k.kp, __int_as_float(k.v), __int_as_float(k.vp)};
    if (seg == 0) a.info[b] = f32x4{__int_as_float(r), __int_as_float(r - lo), w.p.m, w.p.s};
}

// Segment blockIdx.x % T of a sequence's race, the last sequences first: their rows are
// those that the sums read last.
template <int TYPE> __global__ __launch_bounds__(SV_THREADS) void k_sv_pick(SvArgs a)
{
    sv_pick<TYPE, SV_THREADS>(a, a.B - 1 - blockIdx.x / a.T, blockIdx.x % a.T);
}
// Short rows: a workgroup does all of a sequence, a wave the sums of a row.
template <int TYPE> __global__ __launch_bounds__(1024) void k_sv_short(SvArgs a)
{
    const int b = blockIdx.x, wave = threadIdx.x >> 6, lane = threadIdx.x & 63, two = a.y ? 2 : 1;
    int lo, hi;
    sv_rows(a, b, lo, hi);
    for (int i = wave; i < (hi - lo) * two; i += 16) {
        const int r = lo + i / two, of = i % two;
        if (of && a.draft[r] < 0) continue;
        const char *x = (const char *)(of ? a.y : a.x) + (long long)r * (of ? a.ldy : a.ld) * El<TYPE>::SZ;
        const float c = of ? a.dc : a.c;
        const SvSum p = sv_wave(sv_some<TYPE, 64>(x, a.V, 0, a.V / El<TYPE>::VE, true, c, lane), c);
        if (lane == 0) a.part[(size_t)r * 2 + of] = p;
    }
    __syncthreads();
    sv_pick<TYPE, 1024>(a, b, 0);
}

// The winners of a race's segments (T <= 64), one wave a sequence.
template <int TYPE> __global__ __launch_bounds__(64) void k_sv_join(SvArgs a)
{
    const int b = blockIdx.x, t = threadIdx.x;
    const f32x4 i = a.info[b];
    const int r = __float_as_int(i[0]);
    if ((unsigned)r >= (unsigned)a.N) return;            // none, or another call wrote to this workspace
    SvBest k = {0.f, 0.f, a.V, a.V};
    if (t < a.T) {
        const f32x4 p = a.best[(size_t)b * a.T + t];
        k = SvBest{p[0], p[1], __float_as_int(p[2]), __float_as_int(p[3])};
    }
#pragma unroll
    for (int o = 32; o; o /= 2) sv_better(k, sv_lane(k, o));
    if (t == 0) sv_put<TYPE>(a, b, r, __float_as_int(i[1]), k, i[2], i[3]);
}

// -------------------------------------------------------------------- entries --
// Rows of up to SV_SHORT vectors are one workgroup's a sequence, twice as long ones from
// SV_CROWD sequences on, where there are no more sequences than CUs and a sequence has SV_SUMS sums
// (rows, twice with a draft model) in the mean, one of each wave, or from SV_CROWD on four.  In a
// graph that gains where sequences fill the chip (256 of 5 rows of 4096 fp32 values 14.8 us, in two
// launches 18.0; of 2048 values 11.7 and 12.4, of 32 rows 24.5 and 24.7) and costs little where they do
// not (one of 3 rows of 2048 8.8 and 8.7, of 16 rows 10.0 and 9.1; 16 of 16 rows 11.5 and 9.9); a call from
// the host saves the second launch, 2.8 us.  More rows leave the chip idle (one sequence of 64 rows
// 18.5 and 10.0, of 2048 285 and 34; 128 of 256 rows of both models 127 and 104), more sequences
// wait for each other's barriers (384 of 5 rows 17.6 and 13.6, 2048 64 and 35).  Longer rows are cut
// until enough workgroups work: a race's threads wait for every round of loads, so its pieces
// are smaller.
#define SV_SHORT 512
#define SV_CROWD 128
#define SV_MOST 256
#define SV_SUMS 16
static bool sv_short(int type, int N, int V, int B, int drafted)
{
    const int nv = V / (type == TLG_F32 ? 4 : 8);
    const bool crowd = B >= SV_CROWD;
    return nv <= (crowd ? 2 : 1) * SV_SHORT && B <= SV_MOST &&
           (long long)N * (drafted ? 2 : 1) <= (long long)B * SV_SUMS * (crowd ? 4 : 1);
}
static int sv_cut(int type, long long rows, int V, int piece, int fill)
{
    const long long nv = V / (type == TLG_F32 ? 4 : 8), by_size = nv / piece, by_rows = fill / rows;
    const long long s = by_size < by_rows ? by_size : by_rows;
    return s < 1 ? 1 : s > 64 ? 64 : (int)s;
}
static size_t sv_layout(int type, int N, int V, int B, int drafted, int *S, int *T, size_t *best, size_t *info)
{
    const bool one = sv_short(type, N, V, B, drafted);
    *S = one ? 1 : sv_cut(type, (long long)N * (drafted ? 2 : 1), V, 1024, 1024);
    *T = one ? 1 : sv_cut(type, B, V, 512, 1024);
    *best = ((size_t)N * 2 * *S * sizeof(SvSum) + 15) & ~(size_t)15;
    *info = *best + (*T > 1 ? (size_t)B * *T * 16 : 0);
    return *info + (*T > 1 ? (size_t)B * 16 : 0);
}

extern "C" size_t tlg_spec_verify_ws_bytes(int type, int N, int V, int B, int drafted)
{
    if (N <= 0 || V <= 0 || B <= 0) return 0;
    int S, T;
    size_t best, info;
    return sv_layout(type, N, V, B, drafted, &S, &T, &best, &info);
}

template <int TYPE> static void sv_launch(const SvArgs &a, hipStream_t st)
{
    if (sv_short(TYPE, a.N, a.V, a.B, a.y != nullptr)) {
        hipLaunchKernelGGL((k_sv_short<TYPE>), dim3((unsigned)a.B), dim3(1024), 0, st, a);
        return;
    }
    hipLaunchKernelGGL((k_sv_sums<TYPE>), dim3((unsigned)a.N * a.S, a.y ? 2 : 1), dim3(SV_THREADS), 0, st, a);
    hipLaunchKernelGGL((k_sv_pick<TYPE>), dim3((unsigned)a.B * a.T), dim3(SV_THREADS), 0, st, a);
    if (a.T > 1) hipLaunchKernelGGL((k_sv_join<TYPE>), dim3(a.B), dim3(64), 0, st, a);
}

extern "C" int tlg_dev_spec_verify(const void *logits, int type, long long ld, float scale, const void *draft_logits,
                                   long long ldd, float dscale, int N, int V, const int *row0, int B, const int *draft,
                                   const float *u, const float *noise, long long ldn, int *tokens, float *logp,
                                   int *accepted, void *ws, size_t ws_bytes, void *stream)
{
    int rc;
    if ((rc = vb_check("spec_verify", logits, type, ld, N, V))) return rc;
    if (draft_logits && (rc = vb_check("spec_verify", draft_logits, type, ldd, N, V))) return rc;
    if (!vb_positive(scale) || (draft_logits && !vb_positive(dscale)))
        return tlg_fail(TLG_EINVAL, "spec_verify: scale %g, dscale %g", scale, dscale);
    if (B < 0 || B > TLG_PAGED_SEQS) return tlg_fail(TLG_EINVAL, "spec_verify: B=%d", B);
    if (B == 0) return TLG_OK;
    if (!row0 || (uintptr_t)row0 % 4) return tlg_fail(TLG_EINVAL, "spec_verify: row0 %p", (const void *)row0);
    if (N > 0 && (!draft || !u || !noise || !tokens || ldn < V))
        return tlg_fail(TLG_EINVAL, "spec_verify: NULL draft, u, noise or tokens, or ldn=%lld", ldn);
    if (((uintptr_t)draft | (uintptr_t)u | (uintptr_t)noise | (uintptr_t)tokens | (uintptr_t)logp | (uintptr_t)accepted) % 4)
        return tlg_fail(TLG_EINVAL, "spec_verify: draft, u, noise, tokens, logp or accepted not aligned");
    if ((rc = vb_check_ws("spec_verify", ws, ws_bytes, tlg_spec_verify_ws_bytes(type, N, V, B, draft_logits != nullptr))))
        return rc;
    if (N == 0 && !accepted) return TLG_OK;
    if ((rc = tlg_ensure_init())) return rc;
    SvArgs a = {logits, draft_logits, ld, ldd, ldn, scale, (float)((double)scale * 1.4426950408889634), dscale,
                (float)((double)dscale * 1.4426950408889634), N, V, B, 1, 1, row0, draft, u, noise, tokens, accepted, logp,
                (SvSum *)ws, nullptr, nullptr};
    hipStream_t st = ST(stream);
    if (N == 0) {
        hipLaunchKernelGGL((k_sv_pick<TLG_F32>), dim3(B), dim3(SV_THREADS), 0, st, a);
        LAUNCH_CHECK();
        return TLG_OK;
    }
    size_t best, info;
    sv_layout(type, N, V, B, draft_logits != nullptr, &a.S, &a.T, &best, &info);
    a.best = (f32x4 *)((char *)ws + best);
    a.info = (f32x4 *)((char *)ws + info);
    if (type == TLG_F32) sv_launch<TLG_F32>(a, st);
    else if (type == TLG_F16) sv_launch<TLG_F16>(a, st);
    else sv_launch<TLG_BF16>(a, st);
    LAUNCH_CHECK();
    return TLG_OK;
}
