// tlg_vocab.hip -- operators over rows of logits [N][V] besides softmax-CE and
// argmax: log probabilities of given tokens with entropy and top alternatives,
// their gradient, and distillation from a teacher's top log probabilities.
//
// For one row x[0..V) and a scale s = 1 / temperature:
//   m = max x,  S = sum_v e^(s (x_v - m)),  log p_v = s (x_v - m) - log S
//   H = -sum_v p_v log p_v = log S - s sum_v (x_v - m) e^(s (x_v - m)) / S
// Sums are fp32 (and fp64 where K terms cancel), outputs are rounded once.
#include "tlg_internal.h"
#include "../../include/tltrain.h"
#include <math.h>

#define ST(s) ((hipStream_t)(s))
#define LAUNCH_CHECK() TLG_HIP(hipGetLastError())
#define VB 256

// ------------------------------------------------------------- elements --
template <int TYPE> struct El;
template <> struct El<TLG_F32> { typedef float t; };
template <> struct El<TLG_F16> { typedef _Float16 t; };
template <> struct El<TLG_BF16> { typedef __bf16 t; };

__device__ __forceinline__ float vb_max(float v, float *sh)
{
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    return fmaxf(fmaxf(sh[0], sh[1]), fmaxf(sh[2], sh[3]));
}
template <typename F> __device__ __forceinline__ F vb_sum(F v, F *sh)
{
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    return (sh[0] + sh[1]) + (sh[2] + sh[3]);
}

// A total order of values (equal for -0 and +0) in the high half and the lower
// index first in the low half; 0 for -inf, which is no alternative.
__device__ __forceinline__ unsigned long long vb_key(float x, int i)
{
    const unsigned b = __float_as_uint(x + 0.0f);
    const unsigned o = b & 0x80000000u ? ~b : b | 0x80000000u;
    return x == -INFINITY ? 0ull : (unsigned long long)o << 32 | (unsigned)~i;
}
__device__ __forceinline__ float vb_key_value(unsigned long long k)
{
    const unsigned o = (unsigned)(k >> 32);
    return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}

// --------------------------------------------------------- log probabilities --
// One workgroup per row.
template <int TYPE>
__global__ __launch_bounds__(VB) void k_logprobs(const void *__restrict__ logits, long long ld, int V, float scale,
                                                 const int *__restrict__ ids, int M, float *__restrict__ logp,
                                                 float *__restrict__ lse2, float *__restrict__ entropy, int K,
                                                 int *__restrict__ top_ids, float *__restrict__ top_logp)
{
    typedef typename El<TYPE>::t T;
    __shared__ float sh[4];
    __shared__ unsigned long long shk[4];
    const size_t r = blockIdx.x;
    const int t = threadIdx.x;
    const T *x = (const T *)logits + r * ld;
    float m = -INFINITY;
    for (int i = t; i < V; i += VB) m = fmaxf(m, (float)x[i]);
    m = vb_max(m, sh);
    const bool empty = m == -INFINITY;
    float s = 0.f, u = 0.f;
    for (int i = t; i < V; i += VB) {
        const float d = ((float)x[i] - m) * scale, e = expf(d);
        s += empty ? 0.f : e;
        u += e > 0.f || e != e ? e * d : 0.f;
    }
    s = vb_sum(s, sh);
    u = vb_sum(u, sh);
    const bool bad = s != s;
    if (empty) u = 0.f;
    // a row with NaN or +inf has no distribution
    const float ls = bad ? NAN : empty ? -INFINITY : logf(s);
    for (int j = t; j < M; j += VB) {
        const int id = ids[r * M + j];
        float o = 0.f;
        if (id >= V) o = NAN;
        else if (id >= 0) o = empty ? -INFINITY : ((float)x[id] - m) * scale - ls;
        logp[r * M + j] = o;
    }
    if (t == 0) {
        if (lse2) { lse2[2 * r] = bad ? NAN : m; lse2[2 * r + 1] = ls; }
        if (entropy) entropy[r] = empty ? 0.f : ls - u / s;
    }
    unsigned long long last = ~0ull;
    for (int k = 0; k < K; k++) {
        unsigned long long b = 0;
        if (last && !bad)
            for (int i = t; i < V; i += VB) {
                const unsigned long long c = vb_key((float)x[i], i);
                if (c < last && c > b) b = c;
            }
        for (int o = 32; o > 0; o >>= 1) {
            const unsigned long long c = __shfl_xor(b, o);
            if (c > b) b = c;
        }
        __syncthreads();
        if ((t & 63) == 0) shk[t >> 6] = b;
        __syncthreads();
        for (int w = 0; w < 4; w++) b = shk[w] > b ? shk[w] : b;
        last = b;
        if (t == 0) {
            top_ids[r * K + k] = b ? ~(unsigned)b : -1;
            top_logp[r * K + k] = bad ? NAN : b ? (vb_key_value(b) - m) * scale - ls : -INFINITY;
        }
    }
}

// dlogits of logp, lse and entropy: dz_v = sum_j g_j (1{v = id_j} - p_v) +
// g_lse p_v - g_H p_v (log p_v + H).  One workgroup per row; the rows of the
// ids are written again after the others.
#define VB_IDS 64
template <int TYPE>
__global__ __launch_bounds__(VB) void k_logprobs_bwd(const void *logits, long long ld, int V, float scale,
                                                     const int *__restrict__ ids, int M,
                                                     const float *__restrict__ lse2,
                                                     const float *__restrict__ entropy,
                                                     const float *__restrict__ dlogp, const float *__restrict__ dlse,
                                                     const float *__restrict__ dent, void *dlogits, long long ldd)
{
    typedef typename El<TYPE>::t T;
    __shared__ int si[VB_IDS];
    __shared__ float sg[VB_IDS];
    const size_t r = blockIdx.x;
    const int t = threadIdx.x;
    const T *x = (const T *)logits + r * ld;
    T *d = (T *)dlogits + r * ldd;
    float xv = 0.f;
    if (t < M) {
        const int id = ids[r * M + t];
        si[t] = id;
        sg[t] = id >= V ? NAN : id >= 0 ? dlogp[r * M + t] : 0.f;
        if (id >= 0 && id < V) xv = (float)x[id];
    }
    __syncthreads();
    float c0 = dlse ? dlse[r] : 0.f;
    for (int j = 0; j < M; j++) c0 -= sg[j];
    const float c1 = dent ? dent[r] : 0.f, H = dent ? entropy[r] : 0.f;
    const float m = lse2[2 * r], ls = lse2[2 * r + 1];
    const bool empty = m == -INFINITY, zero = empty || (c0 == 0.f && c1 == 0.f);
    auto grad = [&](float v) -> float {
        if (zero) return 0.f;
        const float lp = (v - m) * scale - ls, p = expf(lp);
        return c0 * p - (p == 0.f ? 0.f : c1 * p * (lp + H));
    };
    for (int i = t; i < V; i += VB) d[i] = (T)(scale * grad(zero ? 0.f : (float)x[i]));
    __syncthreads();
    if (t < M && !empty && si[t] >= 0 && si[t] < V) {
        float g = 0.f;
        for (int j = 0; j < M; j++) g += si[j] == si[t] ? sg[j] : 0.f;
        d[si[t]] = (T)(scale * (grad(xv) + g));
    }
}

// -------------------------------------------------------------- distillation --
struct DistillArgs {
    const void *logits;
    long long ld;
    int V, K, tail;
    float tau, w_kd, w_ce, scale;
    const int *t_ids;
    const float *t_logp;
    const int *tgt;
    float *rows;
    void *dlogits;
    long long ldd;
};

#define VB_TOP 128
template <int TYPE> __global__ __launch_bounds__(VB) void k_distill(DistillArgs a)
{
    typedef typename El<TYPE>::t T;
    __shared__ float sh[4];
    __shared__ double shd[4];
    __shared__ int si[VB_TOP];
    __shared__ int sflag;
    extern __shared__ unsigned bits[];              // tail: the support as a set
    const size_t r = blockIdx.x;
    const int t = threadIdx.x, V = a.V, K = a.K;
    const T *x = (const T *)a.logits + r * a.ld;
    T *d = a.dlogits ? (T *)a.dlogits + r * a.ldd : nullptr;
    const int tgt = a.w_ce != 0.f ? a.tgt[r] : -1;
    if (t == 0) sflag = tgt >= V;
    if (t < K) si[t] = a.t_ids[r * K + t];
    if (a.tail)
        for (int i = t; i < (V + 31) / 32; i += VB) bits[i] = 0;
    __syncthreads();
    // the teacher's entry of thread t: an id counts once, at its first place
    int id = -1;
    double tl = -INFINITY;
    if (t < K) {
        id = si[t];
        if (id >= V) sflag = 1;
        for (int j = 0; j < t; j++)
            if (si[j] == id) id = -1;
        if (id >= V) id = -1;
        if (id >= 0) {
            tl = a.t_logp[r * K + t];
            if (a.tail) atomicOr(&bits[id >> 5], 1u << (id & 31));
        }
    }
    __syncthreads();
    const bool bad_id = sflag;
    const int some = (int)vb_sum(id >= 0 ? 1.f : 0.f, sh);
    if (!some && tgt < 0) {                       // nothing to learn from: the logits are not read
        if (d)
            for (int i = t; i < V; i += VB) d[i] = (T)0.f;
        if (a.rows && t == 0) a.rows[r] = bad_id ? NAN : 0.f;
        return;
    }
    const float inv = 1.0f / a.tau;
    float xk = 0.f, xt = 0.f;
    if (id >= 0) xk = (float)x[id];
    if (tgt >= 0 && tgt < V) xt = (float)x[tgt];
    float m = -INFINITY;
    for (int i = t; i < V; i += VB) m = fmaxf(m, (float)x[i]);
    m = vb_max(m, sh);
    const bool empty = m == -INFINITY;
    float s1 = 0.f, so = 0.f, si_ = 0.f;            // CE; outside and inside the support
    for (int i = t; i < V; i += VB) {
        const float v = empty ? -INFINITY : (float)x[i] - m, e = expf(v * inv);
        s1 += expf(v);
        if (a.tail && (bits[i >> 5] >> (i & 31) & 1)) si_ += e;
        else so += e;
    }
    s1 = vb_sum(s1, sh);
    so = vb_sum(so, sh);
    si_ = vb_sum(si_, sh);
    const float s = so + si_;
    // the teacher's distribution
    double q, Q, qr = 0.0;
    if (a.tail) {
        q = id >= 0 ? exp(tl) : 0.0;
        Q = vb_sum(q, shd);
        if (some && some < V && Q < 1.0) qr = 1.0 - Q;
        Q += qr;
    } else {
        const float tm = vb_max((float)tl, sh);
        q = id >= 0 && tm > -INFINITY ? exp(tl - tm) : 0.0;
        if (tl != tl) q = tl;
        Q = vb_sum(q, shd);
        q = Q > 0.0 || Q != Q ? q / Q : 0.0;
        Q = Q > 0.0 ? 1.0 : Q;
    }
    const double ls = log((double)s), ls1 = log((double)s1);
    double kl = 0.0;
    if (q > 0.0 || q != q) kl = empty ? INFINITY : q * (log(q) - ((double)(xk - m) * inv - ls));
    kl = vb_sum(kl, shd);
    if (qr > 0.0) kl += empty ? INFINITY : qr * (log(qr) - (log((double)so) - ls));
    if (a.rows && t == 0) {
        double L = (double)a.w_kd * a.tau * a.tau * kl;
        if (a.w_kd == 0.f || !some) L = 0.0;
        if (tgt >= 0) L += (double)a.w_ce * (empty ? INFINITY : ls1 - (double)(xt - m));
        if (s != s) L = NAN;
        a.rows[r] = bad_id ? NAN : (float)L;
    }
    if (!d) return;
    const float rs = 1.0f / s, rs1 = 1.0f / s1;
    const float ck = some ? a.w_kd * a.tau * a.scale : 0.f, cc = tgt >= 0 ? a.w_ce * a.scale : 0.f;
    const float in = (float)Q, out = qr > 0.0 && so > 0.f ? (float)(Q - qr * s / so) : in;
    auto grad = [&](float v, float mass) -> float {
        if (bad_id) return NAN;
        if (empty) return 0.f;
        const float g = v - m;
        return ck * mass * (expf(g * inv) * rs) + (cc != 0.f ? cc * (expf(g) * rs1) : 0.f);
    };
    __syncthreads();                              // every read of x[id] precedes the writes (in place)
    for (int i = t; i < V; i += VB) d[i] = (T)grad((float)x[i], out);
    __syncthreads();
    bool hit = false;                             // is the target one of the teacher's ids?
    for (int j = 0; j < K; j++) hit |= si[j] == tgt;
    if (empty || bad_id) return;
    if (id >= 0) d[id] = (T)(grad(xk, in) - ck * (float)q - (id == tgt ? cc : 0.f));
    if (t == 0 && tgt >= 0 && tgt < V && !hit) d[tgt] = (T)(grad(xt, out) - cc);
}

// the mean of the row losses, summed in double in a fixed order
__global__ __launch_bounds__(1024) void k_rows_mean(const float *__restrict__ rows, int n, float *__restrict__ out)
{
    __shared__ double s[1024];
    double a = 0.0;
    for (int i = threadIdx.x; i < n; i += 1024) a += (double)rows[i];
    s[threadIdx.x] = a;
    __syncthreads();
    for (int o = 512; o > 0; o >>= 1) {
        if ((int)threadIdx.x < o) s[threadIdx.x] += s[threadIdx.x + o];
        __syncthreads();
    }
    if (threadIdx.x == 0) out[0] = (float)(s[0] / n);
}

// -------------------------------------------------------------------- entries --
static size_t vb_size(int type) { return type == TLG_F32 ? 4 : 2; }

// what every entry asks of its logits; `who` names the entry in the error
static int vb_check(const char *who, const void *logits, int type, long long ld, int N, int V)
{
    if (type != TLG_F32 && type != TLG_F16 && type != TLG_BF16) return tlg_fail(TLG_EINVAL, "%s: type %d", who, type);
    if (N < 0 || V <= 0 || V > TLG_VOCAB_MAX || ld < V)
        return tlg_fail(TLG_EINVAL, "%s: N=%d V=%d ld=%lld", who, N, V, ld);
    if (N > 0 && (!logits || (uintptr_t)logits % vb_size(type)))
        return tlg_fail(TLG_EINVAL, "%s: logits %p", who, logits);
    return TLG_OK;
}
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
static bool vb_positive(float s) { return s > 0.f && s <= 3.4028234e38f; }

#define BY_TYPE(kernel, grid, lds, ...)                                                                          \
    do {                                                                                                         \
        if (type == TLG_F32) hipLaunchKernelGGL(kernel<TLG_F32>, grid, dim3(VB), lds, st, __VA_ARGS__);          \
        else if (type == TLG_F16) hipLaunchKernelGGL(kernel<TLG_F16>, grid, dim3(VB), lds, st, __VA_ARGS__);     \
        else hipLaunchKernelGGL(kernel<TLG_BF16>, grid, dim3(VB), lds, st, __VA_ARGS__);                         \
    } while (0)

extern "C" size_t tlg_logprobs_ws_bytes(int type, int N, int V, int K)
{
    (void)type; (void)N; (void)V; (void)K;
    return 0;
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
    if (ws_bytes < tlg_logprobs_ws_bytes(type, N, V, K))
        return tlg_fail(TLG_EINVAL, "logprobs: workspace of %zu bytes", ws_bytes);
    (void)ws;
    if ((rc = tlg_ensure_init())) return rc;
    hipStream_t st = ST(stream);
    BY_TYPE(k_logprobs, dim3(N), 0, logits, ld, V, scale, ids, M, logp, lse2, entropy, K, top_ids, top_logp);
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
    hipStream_t st = ST(stream);
    BY_TYPE(k_logprobs_bwd, dim3(N), 0, logits, ld, V, scale, ids, M, lse2, entropy, dlogp, dlse, dentropy, dlogits,
            ldd);
    LAUNCH_CHECK();
    return TLG_OK;
}

extern "C" size_t tlg_distill_ws_bytes(int type, int N, int V)
{
    (void)type; (void)N; (void)V;
    return 0;
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
    if (ws_bytes < tlg_distill_ws_bytes(type, N, V))
        return tlg_fail(TLG_EINVAL, "distill: workspace of %zu bytes", ws_bytes);
    (void)ws;
    if ((rc = tlg_ensure_init())) return rc;
    hipStream_t st = ST(stream);
    const DistillArgs a = {logits, ld, V, K, tail, temp, w_kd, w_ce, scale, t_ids, t_logp, tgt, rows, dlogits, ldd};
    BY_TYPE(k_distill, dim3(N), tail ? (size_t)(V + 31) / 32 * 4 : 0, a);
    if (loss) hipLaunchKernelGGL(k_rows_mean, dim3(1), dim3(1024), 0, st, (const float *)rows, N, loss);
    LAUNCH_CHECK();
    return TLG_OK;
}
