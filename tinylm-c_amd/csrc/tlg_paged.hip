// tlg_paged.hip -- a paged KV cache and the attention over it (include/tlserve.h).
#include "tlg_internal.h"
#include "../../include/tlserve.h"
#include <math.h>
#include <float.h>

#define ST(s) ((hipStream_t)(s))
#define LAUNCH_CHECK() TLG_HIP(hipGetLastError())

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 h16;
typedef __bf16 b16;

template <int T> struct ElT;
template <> struct ElT<TLG_F32> { typedef float E; };
template <> struct ElT<TLG_F16> { typedef h16 E; };
template <> struct ElT<TLG_BF16> { typedef b16 E; };

// ----------------------------------------------------------------- batches --
// What the kernels know of a batch and its cache.  Page numbers, rows and lengths
// come from device memory and are cut to what the buffers hold where they are read.
struct PgBatch {
    const int *row0, *len, *table;
    int B, N, ldt;
    int page, n_pages;
    unsigned magic;              // ceil(2^32 / page)
    long long page_ld, tok_ld, head_ld;
};
// t / page for 0 <= t < 2^31: the product is t / page or one more (its error is below t / 2^32)
__device__ __forceinline__ int pg_of(const PgBatch &b, int t)
{
    if (b.page == 1) return t;
    int g = (int)__umulhi((unsigned)t, b.magic);
    return g - (g * b.page > t);
}
__device__ __forceinline__ int pg_row0(const PgBatch &b, int i) { return min(max(b.row0[i], 0), b.N); }

// The last i in [0, n) with start(i) <= x (0 if there is none), all lanes of a wave
// at once: 64 probes a step; start must not decrease.
template <typename F> __device__ __forceinline__ int pg_search(int n, long long x, F start)
{
    const int lane = threadIdx.x & 63;
    int lo = 0;
    while (n > 1) {
        const int step = (n + 63) / 64, i = lane * step;
        const bool in = i < n && (i == 0 || start(lo + i) <= x);
        const int k = __popcll(__ballot(in));            // probes at or below x are the first ones
        lo += (k - 1) * step;
        n = min(step, n - (k - 1) * step);
    }
    return lo;
}

// ------------------------------------------------------------------- store --
struct StoreArgs {
    PgBatch b;
    char *K, *V;
    int KV, H, hd;
    const char *q, *k, *v;
    char *qo;
    long long ldq, ldqo, ldk, ldv;
    const float *cs, *sn;
    int maxpos;
};
template <int T> __device__ __forceinline__ void st_get(const char *p, float *x)       // 8 elements
{
    if constexpr (T == TLG_F32) {
        const f32x4 a = *(const f32x4 *)p, b = *(const f32x4 *)(p + 16);
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = a[i], x[4 + i] = b[i];
    } else {
        typedef typename ElT<T>::E e8 __attribute__((ext_vector_type(8)));
        const e8 a = *(const e8 *)p;
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = (float)a[i];
    }
}
template <int T> __device__ __forceinline__ void st_put(char *p, const float *x)
{
    if constexpr (T == TLG_F32) {
        *(f32x4 *)p = f32x4{x[0], x[1], x[2], x[3]};
        *(f32x4 *)(p + 16) = f32x4{x[4], x[5], x[6], x[7]};
    } else {
        typedef typename ElT<T>::E e8 __attribute__((ext_vector_type(8)));
        e8 a;
#pragma unroll
        for (int i = 0; i < 8; i++) a[i] = (typename ElT<T>::E)x[i];
        *(e8 *)p = a;
    }
}

// A workgroup takes R consecutive rows; a thread eight pairs (i, i + hd/2) of a head.
#define ST_ROWS 4
template <int T, int C> __global__ __launch_bounds__(256) void k_paged_store(StoreArgs a)
{
    constexpr int ts = T == TLG_F32 ? 4 : 2, cs = C == TLG_F32 ? 4 : 2;
    const int lane = threadIdx.x & 63, r0 = blockIdx.x * ST_ROWS, half = a.hd >> 1, per = half >> 3;
    __shared__ int pos[ST_ROWS];                      // position, -1 none: no such row
    __shared__ long long at[ST_ROWS];                 // the token's elements in the cache, -1: not stored
    for (int k = threadIdx.x >> 6; k < ST_ROWS; k += 4) {
        const int r = r0 + k;
        int p = INT_MIN;
        long long to = -1;
        if (r < a.b.N) {
            const int s = pg_search(a.b.B, r, [&](int i) { return pg_row0(a.b, i); });
            const int lo = pg_row0(a.b, s), hi = pg_row0(a.b, s + 1);
            if (r >= lo && r < hi) {
                p = max(a.b.len[s], 0) - (hi - r);
                if (p >= 0) {
                    const int g = pg_of(a.b, p), n = g < a.b.ldt ? a.b.table[(long long)s * a.b.ldt + g] : -1;
                    if (n >= 0 && n < a.b.n_pages) to = n * a.b.page_ld + (p - g * a.b.page) * a.b.tok_ld;
                }
            }
        }
        if (lane == 0) {
            pos[k] = p;
            at[k] = to;
        }
    }
    __syncthreads();
    const int heads = a.H + 2 * a.KV, items = heads * per;
    for (int q = threadIdx.x; q < ST_ROWS * items; q += 256) {
        const int k = q / items, rem = q - k * items, h = rem / per, i = (rem - h * per) * 8, p = pos[k];
        if (p == INT_MIN) continue;
        const long long r = r0 + k;
        const bool isq = h < a.H, isv = h >= a.H + a.KV;
        const int hh = isq ? h : isv ? h - a.H - a.KV : h - a.H;
        if (!isq && at[k] < 0) continue;
        const char *src = isq ? a.q + r * a.ldq * ts : isv ? a.v + r * a.ldv * ts : a.k + r * a.ldk * ts;
        src += (hh * a.hd + i) * ts;
        float x[8], y[8], u[8], w[8];
        st_get<T>(src, x);
        st_get<T>(src + half * ts, y);
        if (!isv && a.cs) {
            if (p < 0 || p >= a.maxpos) {
#pragma unroll
                for (int e = 0; e < 8; e++) u[e] = w[e] = NAN;
            } else {
                float c[8], s[8];
                st_get<TLG_F32>((const char *)(a.cs + (long long)p * half + i), c);
                st_get<TLG_F32>((const char *)(a.sn + (long long)p * half + i), s);
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    u[e] = x[e] * c[e] - y[e] * s[e];
                    w[e] = y[e] * c[e] + x[e] * s[e];
                }
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) u[e] = x[e], w[e] = y[e];
        }
        if (isq) {
            char *d = a.qo + (r * a.ldqo + hh * a.hd + i) * ts;
            st_put<T>(d, u);
            st_put<T>(d + half * ts, w);
        } else {
            char *d = (isv ? a.V : a.K) + (at[k] + hh * a.b.head_ld + i) * cs;
            st_put<C>(d, u);
            st_put<C>(d + half * cs, w);
        }
    }
}

// --------------------------------------------------------------- attention --
struct AttnArgs {
    PgBatch b;
    const char *K, *V, *q;
    char *out;
    float *lse;
    long long ldq, ldo;
    int H, KV, G, hd, win, sinks;
    float c;                     // scale log2 e
};

// One wave a row and head, tokens over the lanes; then elements over the lanes.
template <int T, int C> __global__ __launch_bounds__(64) void k_paged_attn_plain(AttnArgs a)
{
    typedef typename ElT<T>::E Q;
    typedef typename ElT<C>::E E;
    __shared__ float w[64];
    __shared__ long long off[64];
    const int r = blockIdx.x, h = blockIdx.y, lane = threadIdx.x, kvh = h / a.G;
    const int s = pg_search(a.b.B, r, [&](int i) { return pg_row0(a.b, i); });
    const int lo = pg_row0(a.b, s), hi = pg_row0(a.b, s + 1);
    if (r < lo || r >= hi) return;
    const int cap = a.b.ldt * a.b.page;
    const int p = min(max(a.b.len[s], 0) - (hi - r), cap);              // token `cap` stands for all without a page
    const int from = a.win > 0 ? max(0, p - a.win + 1) : 0;
    const Q *q = (const Q *)a.q + (long long)r * a.ldq + h * a.hd;
    float m = -INFINITY, l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
    for (int t0 = 0; t0 <= p; t0 += 64) {
        if (t0 < from && t0 + 63 < from && t0 >= a.sinks) continue;
        const int t = t0 + lane;
        const bool see = t <= p && (t >= from || t < a.sinks);
        float z = -INFINITY;
        long long o = -1;
        if (see) {
            const int g = pg_of(a.b, t), n = g < a.b.ldt ? a.b.table[(long long)s * a.b.ldt + g] : -1;
            if (n >= 0 && n < a.b.n_pages) {
                o = n * a.b.page_ld + (t - g * a.b.page) * a.b.tok_ld + kvh * a.b.head_ld;
                const E *k = (const E *)a.K + o;
                z = 0.f;
                for (int d = 0; d < a.hd; d++) z = fmaf((float)q[d], (float)k[d], z);
            } else z = NAN;
        }
        float n = z;
        for (int x = 32; x; x /= 2) n = fmaxf(n, __shfl_xor(n, x));
        n = fmaxf(m, n);
        const float ref = n == -INFINITY ? 0.f : n * a.c, f = exp2f((m == -INFINITY ? -INFINITY : m * a.c) - ref);
        const float e = see ? exp2f(fmaf(z, a.c, -ref)) : 0.f;
        __syncthreads();
        w[lane] = e;
        off[lane] = see ? o : -2;
        __syncthreads();
        l = l * f + e;
        m = n;
        for (int j = 0; j < a.hd / 64 + (a.hd % 64 != 0); j++) {
            const int d = j * 64 + lane;
            if (d >= a.hd) continue;
            float x = acc[j] * f;
            for (int i = 0; i < 64; i++)
                if (off[i] >= 0) x = fmaf(w[i], (float)((const E *)a.V)[off[i] + d], x);
            acc[j] = x;
        }
    }
    for (int x = 32; x; x /= 2) l += __shfl_xor(l, x);
    for (int j = 0; j < a.hd / 64 + (a.hd % 64 != 0); j++) {
        const int d = j * 64 + lane;
        if (d < a.hd) ((Q *)a.out)[(long long)r * a.ldo + h * a.hd + d] = (Q)(l == 0.f ? 0.f : acc[j] / l + 0.f * l);
    }
    if (a.lse && lane == 0)
        a.lse[(long long)r * a.H + h] = l == 0.f ? -INFINITY : (m == -INFINITY ? 0.f : m * a.c * 0.69314718056f) + logf(l);
}

// -------------------------------------------------------------------- entries --
static size_t pg_size(int type) { return type == TLG_F32 ? 4 : 2; }
static bool pg_type(int type) { return type == TLG_F32 || type == TLG_F16 || type == TLG_BF16; }
static bool pg_al(const void *p, size_t n) { return p && (uintptr_t)p % n == 0; }

// what both entries ask of cache and batch; *ok 0: nothing to do
static int pg_check(const char *who, const TlgPages *c, const TlgBatch *b, int type, PgBatch *o, int *work)
{
    *work = 0;
    if (!c || !b) return tlg_fail(TLG_EINVAL, "%s: NULL cache or batch", who);
    if (!pg_type(type) || !pg_type(c->type) || (type != TLG_F32 && type != c->type))
        return tlg_fail(TLG_EINVAL, "%s: rows of type %d, a cache of type %d", who, type, c->type);
    if (c->hd != 32 && c->hd != 64 && c->hd != 96 && c->hd != 128 && c->hd != 256)
        return tlg_fail(TLG_EINVAL, "%s: hd=%d", who, c->hd);
    if (c->KV <= 0 || c->KV > TLG_PAGED_HEADS || c->page <= 0 || c->page > TLG_PAGED_PAGE || c->n_pages < 0)
        return tlg_fail(TLG_EINVAL, "%s: KV=%d page=%d n_pages=%d", who, c->KV, c->page, c->n_pages);
    const long long e = 16 / (long long)pg_size(c->type), far = 1ll << 40;
    if (c->page_ld < 0 || c->tok_ld < 0 || c->head_ld < 0 || c->page_ld > far || c->tok_ld > far || c->head_ld > far ||
        c->page_ld % e || c->tok_ld % e || c->head_ld % e)
        return tlg_fail(TLG_EINVAL, "%s: page_ld=%lld tok_ld=%lld head_ld=%lld", who, c->page_ld, c->tok_ld, c->head_ld);
    if (c->n_pages > 0 && (!pg_al(c->K, 16) || !pg_al(c->V, 16)))
        return tlg_fail(TLG_EINVAL, "%s: cache %p, %p", who, c->K, c->V);
    if (b->B < 0 || b->B > TLG_PAGED_SEQS || b->N < 0 || b->N > TLG_PAGED_ROWS || b->ldt < 0 ||
        (long long)b->ldt * c->page > TLG_PAGED_LEN || b->max_rows < 0 || b->max_len < 0)
        return tlg_fail(TLG_EINVAL, "%s: B=%d N=%d ldt=%d max_rows=%d max_len=%d", who, b->B, b->N, b->ldt, b->max_rows,
                        b->max_len);
    if (b->B == 0 || b->N == 0) return TLG_OK;
    if (!pg_al(b->row0, 4) || !pg_al(b->len, 4) || (b->ldt && !pg_al(b->table, 4)))
        return tlg_fail(TLG_EINVAL, "%s: row0 %p len %p table %p", who, (const void *)b->row0, (const void *)b->len,
                        (const void *)b->table);
    *o = PgBatch{b->row0, b->len, b->table, b->B, b->N, b->ldt, c->page, c->n_pages,
                 (unsigned)(((1ull << 32) + c->page - 1) / c->page), c->page_ld, c->tok_ld, c->head_ld};
    *work = 1;
    return TLG_OK;
}
static bool pg_rows(const void *p, long long ld, long long width, int type)
{
    return pg_al(p, 16) && ld >= width && ld <= 1ll << 40 && ld % (16 / (long long)pg_size(type)) == 0;
}

extern "C" int tlg_dev_paged_store(const TlgPages *c, const TlgBatch *b, const void *q, long long ldq, void *q_out,
                                   long long ldqo, int H, const void *k, long long ldk, const void *v, long long ldv,
                                   int type, const float *cos_t, const float *sin_t, int maxpos, void *stream)
{
    StoreArgs a;
    int rc, work;
    if ((rc = pg_check("paged_store", c, b, type, &a.b, &work))) return rc;
    if (q && (H <= 0 || H > TLG_PAGED_HEADS)) return tlg_fail(TLG_EINVAL, "paged_store: H=%d", H);
    if (!cos_t != !sin_t || (cos_t && (!pg_al(cos_t, 16) || !pg_al(sin_t, 16) || maxpos < 0)))
        return tlg_fail(TLG_EINVAL, "paged_store: tables %p, %p of %d positions", (const void *)cos_t, (const void *)sin_t,
                        maxpos);
    if (!work) return TLG_OK;
    const long long wq = (long long)H * c->hd, wk = (long long)c->KV * c->hd;
    if (!pg_rows(k, ldk, wk, type) || !pg_rows(v, ldv, wk, type))
        return tlg_fail(TLG_EINVAL, "paged_store: k %p ldk=%lld v %p ldv=%lld", k, ldk, v, ldv);
    if (q && (!pg_rows(q, ldq, wq, type) || !pg_rows(q_out, ldqo, wq, type)))
        return tlg_fail(TLG_EINVAL, "paged_store: q %p ldq=%lld q_out %p ldqo=%lld", q, ldq, q_out, ldqo);
    if ((rc = tlg_ensure_init())) return rc;
    a.K = (char *)c->K;
    a.V = (char *)c->V;
    a.KV = c->KV;
    a.H = q ? H : 0;
    a.hd = c->hd;
    a.q = (const char *)q;
    a.k = (const char *)k;
    a.v = (const char *)v;
    a.qo = (char *)q_out;
    a.ldq = ldq;
    a.ldqo = ldqo;
    a.ldk = ldk;
    a.ldv = ldv;
    a.cs = cos_t;
    a.sn = sin_t;
    a.maxpos = maxpos;
    const dim3 grid((b->N + ST_ROWS - 1) / ST_ROWS), block(256);
    hipStream_t st = ST(stream);
    if (type == TLG_F16) hipLaunchKernelGGL((k_paged_store<TLG_F16, TLG_F16>), grid, block, 0, st, a);
    else if (type == TLG_BF16) hipLaunchKernelGGL((k_paged_store<TLG_BF16, TLG_BF16>), grid, block, 0, st, a);
    else if (c->type == TLG_F32) hipLaunchKernelGGL((k_paged_store<TLG_F32, TLG_F32>), grid, block, 0, st, a);
    else if (c->type == TLG_F16) hipLaunchKernelGGL((k_paged_store<TLG_F32, TLG_F16>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((k_paged_store<TLG_F32, TLG_BF16>), grid, block, 0, st, a);
    LAUNCH_CHECK();
    return TLG_OK;
}

extern "C" size_t tlg_paged_attn_ws_bytes(const TlgPages *c, const TlgBatch *b, int type, int H)
{
    (void)c, (void)b, (void)type, (void)H;
    return 0;
}

extern "C" int tlg_dev_paged_attn(const TlgPages *c, const TlgBatch *b, const void *q, int type, long long ldq, int H,
                                  float scale, int win, int sinks, void *out, long long ldo, float *lse, void *ws,
                                  size_t ws_bytes, void *stream)
{
    AttnArgs a;
    int rc, work;
    if ((rc = pg_check("paged_attn", c, b, type, &a.b, &work))) return rc;
    if (H <= 0 || H > TLG_PAGED_HEADS || H % c->KV)
        return tlg_fail(TLG_EINVAL, "paged_attn: H=%d KV=%d", H, c->KV);
    if (!(scale >= 1e-30f && scale <= 1e30f) || win < 0 || sinks < 0)
        return tlg_fail(TLG_EINVAL, "paged_attn: scale=%g win=%d sinks=%d", scale, win, sinks);
    if (!work) return TLG_OK;
    const long long w = (long long)H * c->hd;
    if (!pg_rows(q, ldq, w, type) || !pg_rows(out, ldo, w, type) || (lse && !pg_al(lse, 4)))
        return tlg_fail(TLG_EINVAL, "paged_attn: q %p ldq=%lld out %p ldo=%lld lse %p", q, ldq, out, ldo, (void *)lse);
    const size_t need = tlg_paged_attn_ws_bytes(c, b, type, H);
    if (need && (ws_bytes < need || !pg_al(ws, 16)))
        return tlg_fail(TLG_EINVAL, "paged_attn: workspace %p of %zu bytes, %zu needed", ws, ws_bytes, need);
    if ((rc = tlg_ensure_init())) return rc;
    a.K = (const char *)c->K;
    a.V = (const char *)c->V;
    a.q = (const char *)q;
    a.out = (char *)out;
    a.lse = lse;
    a.ldq = ldq;
    a.ldo = ldo;
    a.H = H;
    a.KV = c->KV;
    a.G = H / c->KV;
    a.hd = c->hd;
    a.win = win;
    a.sinks = sinks;
    a.c = (float)((double)scale * 1.4426950408889634);
    hipStream_t st = ST(stream);
    const dim3 grid(b->N, H), block(64);
    if (type == TLG_F16) hipLaunchKernelGGL((k_paged_attn_plain<TLG_F16, TLG_F16>), grid, block, 0, st, a);
    else if (type == TLG_BF16) hipLaunchKernelGGL((k_paged_attn_plain<TLG_BF16, TLG_BF16>), grid, block, 0, st, a);
    else if (c->type == TLG_F32) hipLaunchKernelGGL((k_paged_attn_plain<TLG_F32, TLG_F32>), grid, block, 0, st, a);
    else if (c->type == TLG_F16) hipLaunchKernelGGL((k_paged_attn_plain<TLG_F32, TLG_F16>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((k_paged_attn_plain<TLG_F32, TLG_BF16>), grid, block, 0, st, a);
    LAUNCH_CHECK();
    return TLG_OK;
}
