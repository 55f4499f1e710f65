// tlg_paged.hip -- a paged KV cache and the attention over it (include/tlserve.h).
#include "tlg_paged.h"

#define ST(s) ((hipStream_t)(s))
#define LAUNCH_CHECK() TLG_HIP(hipGetLastError())

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
// Scores are formed transposed, S^T = K Q^T, 32 tokens by 32 columns (rows times query
// heads of one KV head, so that a key is read once for all heads that share it): a lane
// then has 16 of a column's 32 scores, its softmax needs one exchange between the halves
// of the wave, and the weights are already the operand of O^T = V^T P^T, whose sums
// the lane rescales by its own column's factor.  Which token stands at which place of
// an operand's reduction is free as long as both operands agree, so nothing moves
// between lanes.
//
// k_paged_direct works from global memory: a lane reads its token's key (one row of the
// first operand) in pieces of 16 bytes.  For 16-bit rows the values go through LDS, each
// wave's own 32 tokens, and are read back transposed; fp32 products (two tokens at a
// time) take them as they are, element 32 m.. of lane m being whatever is contiguous.
// !ROWS: few columns (a decoded token, a drafted chunk), bound by the cache's bytes: the
// four waves of a workgroup take every fourth tile of the tokens and join their sums,
// and S workgroups share a long sequence.  ROWS (fp32): every wave 32 columns of its
// own, whose keys the waves of a workgroup find in the CU's cache.
template <int T, int C, int HD, bool ROWS>
__global__ __launch_bounds__(256, (T == TLG_F32 && HD >= 128) || HD == 256 ? 1 : 2) void k_paged_direct(AttnArgs a)
{
    constexpr bool F = T == TLG_F32;
    constexpr int NB = HD / 32, ts = F ? 4 : 2, cs = C == TLG_F32 ? 4 : 2;
    constexpr int NK = F ? HD / 8 : HD / 16, KW = F ? cs : 4;           // pieces of a key and their registers
    constexpr int NV = F ? 16 : HD / 16, VW = F ? (NB * cs + 3) / 4 : 4;
    constexpr int VST = (HD / 2) % 64 == 16 || (HD / 2) % 64 == 48 ? HD : HD + 32;   // elements between tokens in LDS
    constexpr int VB = F ? 0 : 4 * 32 * VST * 2, MB = ROWS ? 0 : 4 * 32 * 36 * 4;
    typedef typename ElT<C>::E E;
    __shared__ __align__(16) char mem[VB > MB ? VB : MB ? MB : 16];
    __shared__ long long toff[4][2][32];
    __shared__ float red[4][2][32];

    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 31, h = lane >> 5;
    const int kvh = blockIdx.x % a.KV, s = blockIdx.x / a.KV % a.S, y = blockIdx.x / a.KV / a.S;
    int b = y, base = blockIdx.y * 32;
    if (ROWS) {
        auto start = [&](int i) { return (long long)pg_row0(a.b, i) * a.G / 128 + i; };
        b = pg_search(a.b.B, y, start);
        base = (int)(y - start(b)) * 128 + 32 * wave;
    }
    const Seq q = pg_seq(a.b, b);
    const int cols = q.n * a.G;
    if (base < 0 || base >= cols || cols <= a.few || cols > a.many) return;
    const int *table = a.b.table + (long long)b * a.b.ldt;
    const long long head = kvh * a.b.head_ld;
    const E *Kc = (const E *)a.K + head, *Vc = (const E *)a.V + head;
    AttnArgs av = a;                                                    // pg_special reads V from the head on
    av.V = (const char *)Vc;
    auto at = [](int blk, int m) { return F ? NB * m + blk : 32 * blk + m; };
    E *vs = (E *)mem + wave * 32 * VST;

    for (int rh0 = base; rh0 < cols; rh0 += 32 * gridDim.y) {
        const Range rg = pg_range<32>(a, q, rh0, min(rh0 + 32, cols));
        const int parts = pg_parts<32>(a.S, rg.total);
        if (s >= parts) {
            if (ROWS) return;
            continue;
        }
        const int j0 = (int)((long long)rg.total * s / parts), j1 = (int)((long long)rg.total * (s + 1) / parts);
        const int step = ROWS ? 1 : 4;
        // the lane's column
        const int rh = rh0 + col, ci = min(rh, cols - 1) / a.G, g = min(rh, cols - 1) - ci * a.G;
        const bool live = rh < cols;
        const int r = q.lo + ci, p = live ? pg_pos(a, q, ci) : -1, from = pg_from(a, p);
        u32x4 qf[NK];
        {
            const char *qp = a.q + ((long long)r * a.ldq + (kvh * a.G + g) * HD + (F ? 4 : 8) * h) * ts;
#pragma unroll
            for (int i = 0; i < NK; i++) {
                qf[i] = *(const u32x4 *)(qp + i * (F ? 8 : 16) * ts);
                if (!live) qf[i] = u32x4{0, 0, 0, 0};
            }
        }
        f32x16 o[NB];
#pragma unroll
        for (int i = 0; i < NB; i++)
#pragma unroll
            for (int k = 0; k < 16; k++) o[i][k] = 0.f;
        float R = -INFINITY, l = 0.f;

        unsigned kr[NK][KW], vr[NV][VW];
        // the page of the lane's token of tile j, then its elements
        auto page = [&](int j) {
            const int t = pg_tile<32>(rg, j) + col, n = pg_of(a.b, t);
            return j < j1 && t <= rg.pmax && n < a.b.ldt ? table[n] : -1;
        };
        auto elems = [&](int j, int n) {
            const int t = pg_tile<32>(rg, j) + col;
            return n >= 0 && n < a.b.n_pages ? n * a.b.page_ld + (t - pg_of(a.b, t) * a.b.page) * a.b.tok_ld : -1ll;
        };
        auto loadK = [&](long long off) {
            const E *k = Kc + max(off, 0ll) + (F ? 4 : 8) * h;
#pragma unroll
            for (int i = 0; i < NK; i++) __builtin_memcpy(kr[i], __builtin_assume_aligned(k + i * (F ? 8 : 16), 4 * KW), 4 * KW);
        };
        auto loadV = [&](int buf, long long off) {
            if (h == 0) toff[wave][buf][col] = off;
            pg_wave_sync();
            if constexpr (F) {
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const E *v = Vc + max(toff[wave][buf][pg_at(i, h)], 0ll) + NB * col;
                    vr[i][VW - 1] = 0;
                    __builtin_memcpy(vr[i], v, NB * cs);
                }
            } else {
#pragma unroll
                for (int i = 0; i < NV; i++) {
                    const int ch = lane + 64 * i, t = ch / (HD / 8), d = ch % (HD / 8) * 8;
                    __builtin_memcpy(vr[i], __builtin_assume_aligned(Vc + max(toff[wave][buf][t], 0ll) + d, 16), 16);
                }
            }
        };
        int j = j0 + (ROWS ? 0 : wave), buf = 0, ahead = page(j + step);
        long long off = elems(j, page(j));
        if (j < j1) {
            loadK(off);
            loadV(0, off);
        }
        for (; j < j1; j += step, buf ^= 1) {
            const int t0 = pg_tile<32>(rg, j);
            const bool more = j + step < j1;
            const long long next = elems(j + step, ahead);
            ahead = page(j + 2 * step);
            // scores
            f32x16 z;
#pragma unroll
            for (int i = 0; i < 16; i++) z[i] = 0.f;
            if (off < 0) kr[0][0] = ~0u;
            if constexpr (F) {
#pragma unroll
                for (int i = 0; i < NK; i++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        float k;
                        if constexpr (C == TLG_F32) k = __uint_as_float(kr[i][e]);
                        else k = (float)__builtin_bit_cast(E, (unsigned short)(kr[i][e / 2] >> (e & 1) * 16));
                        z = __builtin_amdgcn_mfma_f32_32x32x2f32(k, __uint_as_float(qf[i][e]), z, 0, 0, 0);
                    }
            } else {
#pragma unroll
                for (int i = 0; i < NK; i++) z = pg_mfma<T>(u32x4{kr[i][0], kr[i][1], kr[i][2], kr[i][3]}, qf[i], z);
            }
            if (more) loadK(next);
            // weights
            const bool full = t0 + 31 <= rg.pmin && (rg.lomax <= t0 || t0 + 31 < a.sinks);
            float e[16];
#pragma unroll
            for (int i = 0; i < 16; i++) e[i] = full || pg_sees(a, t0 + pg_at(i, h), p, from) ? z[i] : -INFINITY;
            pg_weights<16, NB>(e, a.c, R, l, o);
            bool odd = false;
            if (!full) {
#pragma unroll
                for (int i = 0; i < NV; i++) {
                    bool hit = false;
#pragma unroll
                    for (int k = 0; k < VW; k++) hit |= pg_clean<C>(vr[i][k]);
                    const int t = F ? pg_at(i, h) : (lane + 64 * i) / (HD / 8);
                    odd |= hit && t0 + t <= rg.pmax;
                }
                odd = __any(odd);
            }
            // values
            if constexpr (F) {
#pragma unroll
                for (int i = 0; i < 16; i++)
#pragma unroll
                    for (int k = 0; k < NB; k++) {
                        float v;
                        if constexpr (C == TLG_F32) v = __uint_as_float(vr[i][k]);
                        else v = (float)__builtin_bit_cast(E, (unsigned short)(vr[i][k / 2] >> (k & 1) * 16));
                        o[k] = __builtin_amdgcn_mfma_f32_32x32x2f32(v, e[i], o[k], 0, 0, 0);
                    }
                if (more) loadV(buf ^ 1, next);
            } else {
                pg_wave_sync();
#pragma unroll
                for (int i = 0; i < NV; i++) {
                    const int ch = lane + 64 * i, t = ch / (HD / 8), d = ch % (HD / 8) * 8;
                    *(u32x4 *)(vs + t * VST + d) = u32x4{vr[i][0], vr[i][1], vr[i][2], vr[i][3]};
                }
                if (more) loadV(buf ^ 1, next);
                pg_wave_sync();
                u32x4 pf[2];
#pragma unroll
                for (int i = 0; i < 8; i++) pf[i / 4][i & 3] = pg_pack<T>(e[2 * i], e[2 * i + 1]);
                typedef short s16x4 __attribute__((ext_vector_type(4)));
                typedef __attribute__((address_space(3))) s16x4 *lds;
                const E *vt = vs + (4 * h + (lane >> 2 & 3)) * VST + 16 * (lane >> 4 & 1) + 4 * (lane & 3);
#pragma unroll
                for (int k = 0; k < NB; k++)
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        const u32x2 v0 = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds)(vt + 16 * i * VST + 32 * k)));
                        const u32x2 v1 = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds)(vt + (16 * i + 8) * VST + 32 * k)));
                        o[k] = pg_mfma<T>(u32x4{v0[0], v0[1], v1[0], v1[1]}, pf[i], o[k]);
                    }
            }
            if (odd) pg_special<C, NB>(av, o, e, t0, rg.pmax, p, from, [&](int k) { return toff[wave][buf][k]; }, at);
            off = next;
        }
        l = pg_both_sum(l);
        if constexpr (ROWS) {
            if (!live) return;
            if constexpr (F) {
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    float x[NB];
#pragma unroll
                    for (int k = 0; k < NB; k++) x[k] = o[k][i];
                    pg_out<T, NB>(a, HD, s, parts, r, kvh * a.G + g, NB * pg_at(i, h), l, x);
                }
            } else {
#pragma unroll
                for (int k = 0; k < NB; k++)
#pragma unroll
                    for (int i = 0; i < 16; i += 4) {
                        float x[4] = {o[k][i], o[k][i + 1], o[k][i + 2], o[k][i + 3]};
                        pg_out<T, 4>(a, HD, s, parts, r, kvh * a.G + g, 32 * k + pg_at(i, h), l, x);
                    }
            }
            if (h == 0) pg_out_sums(a, s, parts, r, kvh * a.G + g, R, l);
            return;
        } else {
            // the waves' sums against the largest of their references
            if (h == 0) {
                red[wave][0][col] = R;
                red[wave][1][col] = l;
            }
            __syncthreads();
            auto top = [&](int c) { return fmaxf(fmaxf(red[0][0][c], red[1][0][c]), fmaxf(red[2][0][c], red[3][0][c])); };
            const float mine = top(col), f = __builtin_amdgcn_exp2f(R - (mine == -INFINITY ? 0.f : mine));
            const int oc = threadIdx.x >> 3, om = threadIdx.x & 7;     // the thread's column and four rows of each block
            const float Rt = top(oc);
            float lt = 0.f, x[4 * NB];
#pragma unroll
            for (int w = 0; w < 4; w++)
                lt += red[w][1][oc] * __builtin_amdgcn_exp2f(red[w][0][oc] - (Rt == -INFINITY ? 0.f : Rt));
            float *mg = (float *)mem;
#pragma unroll
            for (int k = 0; k < NB; k++) {
#pragma unroll
                for (int i = 0; i < 4; i++)
                    *(f32x4 *)(mg + (wave * 32 + col) * 36 + 8 * i + 4 * h) =
                        f32x4{o[k][4 * i], o[k][4 * i + 1], o[k][4 * i + 2], o[k][4 * i + 3]} * f;
                __syncthreads();
                f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int w = 0; w < 4; w++) v += *(const f32x4 *)(mg + (w * 32 + oc) * 36 + 4 * om);
#pragma unroll
                for (int i = 0; i < 4; i++) x[F ? i * NB + k : 4 * k + i] = v[i];
                __syncthreads();
            }
            const int orh = rh0 + oc;
            if (orh < cols) {
                const int oi = orh / a.G, hq = kvh * a.G + orh - oi * a.G;
                if constexpr (F) pg_out<T, 4 * NB>(a, HD, s, parts, q.lo + oi, hq, 4 * om * NB, lt, x);
                else {
#pragma unroll
                    for (int k = 0; k < NB; k++) pg_out<T, 4>(a, HD, s, parts, q.lo + oi, hq, 32 * k + 4 * om, lt, x + 4 * k);
                }
                if (om == 0) pg_out_sums(a, s, parts, q.lo + oi, hq, Rt, lt);
            }
        }
    }
}

// The sums of the workgroups that shared a row's tokens: one wave a row and head.  Tiles
// of sequences of at most `few` columns had 32 of them, others `big` (their tokens in
// tiles of 32 or, with the flag, 64).
template <int T> __global__ __launch_bounds__(256) void k_paged_join(AttnArgs a, int hd, int few, int big, int by64)
{
    const int lane = threadIdx.x & 63;
    const long long rhd = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int r = (int)(rhd / a.H), head = (int)(rhd - (long long)r * a.H);
    if (r >= a.b.N) return;
    const int b = pg_search(a.b.B, r, [&](int i) { return pg_row0(a.b, i); });
    const Seq q = pg_seq(a.b, b);
    if (r < q.lo || r >= q.lo + q.n) return;
    const int cols = q.n * a.G, rh = (r - q.lo) * a.G + head % a.G, w = cols <= few ? 32 : big;
    const int rh0 = rh / w * w, rh1 = min(rh0 + w, cols);
    const int parts = cols > few && by64 ? pg_parts<64>(a.S, pg_range<64>(a, q, rh0, rh1).total)
                                         : pg_parts<32>(a.S, pg_range<32>(a, q, rh0, rh1).total);
    if (parts < 2) return;
    const long long row = (long long)r * a.H + head, all = (long long)a.b.N * a.H;
    float R = -INFINITY, l = 0.f;
    if (lane < parts) {
        const float2 m = *(const float2 *)(a.pm + (row + lane * all) * 2);
        R = m.x;
        l = m.y;
    }
    float top = R;
#pragma unroll
    for (int o = 32; o; o /= 2) top = fmaxf(top, __shfl_xor(top, o));
    const float f = __builtin_amdgcn_exp2f(R - (top == -INFINITY ? 0.f : top));
    l *= f;
#pragma unroll
    for (int o = 32; o; o /= 2) l += __shfl_xor(l, o);
    const float *po = a.po + row * hd;
    float x[4] = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < parts; s++) {
        const float fs = __shfl(f, s);
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (i * 64 + lane < hd) x[i] = fmaf(fs, po[s * all * hd + i * 64 + lane], x[i]);
    }
    const float inv = pg_inverse(l);
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (i * 64 + lane < hd)
            ((typename ElT<T>::E *)a.out)[(long long)r * a.ldo + (long long)head * hd + i * 64 + lane] =
                (typename ElT<T>::E)(l == 0.f ? 0.f : x[i] * inv);
    if (a.lse && lane == 0) a.lse[row] = pg_lse(top, l);
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

// How a call is launched: the columns (rows times heads of a KV head) of a sequence
// decide.  few: only k_paged_direct with workgroups of 32 columns; else the rows' kernel,
// and, where the numbers of rows differ, the former for the sequences of few.
#define PG_FEW 32
#define PG_FILL 1024                 /* workgroups wanted */
struct Plan {
    bool few, both;
    unsigned tiles, slots;           // of 32 columns of a sequence, of 128 of all
    int S;
    size_t sums;                     // bytes of the partial sums, before their references
};
static Plan pg_plan(const TlgPages *c, const TlgBatch *b, int H)
{
    Plan p = {};
    const int G = H / c->KV, rows = b->max_rows && b->max_rows < b->N ? b->max_rows : b->N;
    const long long cols = (long long)rows * G, room = (long long)b->ldt * c->page,
                    len = b->max_len && b->max_len < room ? b->max_len : room;
    p.few = cols <= PG_FEW;
    p.tiles = p.few ? (unsigned)((cols + 31) / 32) : 1;
    p.slots = (unsigned)((long long)b->N * G / 128 + b->B);
    p.both = !p.few && (long long)b->B * rows > b->N;
    const long long groups = p.few ? (long long)b->B * p.tiles * c->KV : (long long)p.slots * c->KV,
                    row = (long long)b->N * H * (c->hd + 2) * 4;
    long long S = PG_FILL / groups;
    if (S > len / PG_MIN) S = len / PG_MIN;
    if (S > (128ll << 20) / row) S = (128ll << 20) / row;
    p.S = S < 1 ? 1 : S > 64 ? 64 : (int)S;
    p.sums = p.S > 1 ? (size_t)p.S * b->N * H * c->hd * 4 : 0;
    return p;
}

extern "C" size_t tlg_paged_attn_ws_bytes(const TlgPages *c, const TlgBatch *b, int type, int H)
{
    (void)type;
    if (!c || !b || c->KV <= 0 || H < c->KV || b->N <= 0 || b->B <= 0 || c->hd <= 0 || c->page <= 0 || b->ldt < 0 ||
        b->max_rows < 0 || b->max_len < 0)
        return 0;
    const Plan p = pg_plan(c, b, H);
    return p.sums ? p.sums + (size_t)p.S * b->N * H * 8 : 0;
}

template <int T, int C, bool ROWS> static void pg_direct(const AttnArgs &a, int hd, dim3 grid, hipStream_t st)
{
    if (hd == 32) hipLaunchKernelGGL((k_paged_direct<T, C, 32, ROWS>), grid, dim3(256), 0, st, a);
    else if (hd == 64) hipLaunchKernelGGL((k_paged_direct<T, C, 64, ROWS>), grid, dim3(256), 0, st, a);
    else if (hd == 96) hipLaunchKernelGGL((k_paged_direct<T, C, 96, ROWS>), grid, dim3(256), 0, st, a);
    else if (hd == 128) hipLaunchKernelGGL((k_paged_direct<T, C, 128, ROWS>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((k_paged_direct<T, C, 256, ROWS>), grid, dim3(256), 0, st, a);
}
template <bool ROWS> static void pg_direct(const AttnArgs &a, int type, int kv, int hd, dim3 grid, hipStream_t st)
{
    if (type == TLG_F16) pg_direct<TLG_F16, TLG_F16, ROWS>(a, hd, grid, st);
    else if (type == TLG_BF16) pg_direct<TLG_BF16, TLG_BF16, ROWS>(a, hd, grid, st);
    else if (kv == TLG_F32) pg_direct<TLG_F32, TLG_F32, ROWS>(a, hd, grid, st);
    else if (kv == TLG_F16) pg_direct<TLG_F32, TLG_F16, ROWS>(a, hd, grid, st);
    else pg_direct<TLG_F32, TLG_BF16, ROWS>(a, hd, grid, st);
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
    if ((long long)b->N * H > 1 << 30) return tlg_fail(TLG_EINVAL, "paged_attn: N=%d H=%d", b->N, H);
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
    a.win = win < TLG_PAGED_LEN + 1 ? win : 0;            // a longer one hides nothing
    a.sinks = sinks < TLG_PAGED_LEN ? sinks : TLG_PAGED_LEN;
    a.c = (float)((double)scale * 1.4426950408889634);
    if (c->n_pages == 0) {               // no token has a page: any readable memory stands for the first
        a.K = a.V = a.q;
        a.b.head_ld = 0;
    }
    const Plan p = pg_plan(c, b, H);
    a.S = p.S;
    a.few = 0;
    a.many = p.few ? INT_MAX : PG_FEW;
    a.po = (float *)ws;
    a.pm = (float *)((char *)ws + p.sums);
    hipStream_t st = ST(stream);
    if (p.few || p.both)
        pg_direct<false>(a, type, c->type, c->hd, dim3((unsigned)b->B * c->KV * p.S, p.tiles), st);
    if (!p.few) {
        a.few = p.both ? PG_FEW : 0;
        a.many = INT_MAX;
        pg_direct<true>(a, type, c->type, c->hd, dim3(p.slots * c->KV * p.S), st);
    }
    if (p.S > 1) {
        const int big = 32, by64 = 0;
        const dim3 grid((unsigned)(((long long)b->N * H + 3) / 4));
        if (type == TLG_F32) hipLaunchKernelGGL((k_paged_join<TLG_F32>), grid, dim3(256), 0, st, a, c->hd, a.few, big, by64);
        else if (type == TLG_F16)
            hipLaunchKernelGGL((k_paged_join<TLG_F16>), grid, dim3(256), 0, st, a, c->hd, a.few, big, by64);
        else hipLaunchKernelGGL((k_paged_join<TLG_BF16>), grid, dim3(256), 0, st, a, c->hd, a.few, big, by64);
    }
    LAUNCH_CHECK();
    return TLG_OK;
}
