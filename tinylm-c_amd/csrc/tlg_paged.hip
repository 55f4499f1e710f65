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
// Scores are formed transposed, S^T = K Q^T, tokens by columns (rows times query heads
// of one KV head, so that a key is read once for all heads that share it): a lane then
// has a share of one column's scores, its softmax needs exchanges between the two or
// four lanes of a column only, and the weights are already the operand of O^T = V^T
// P^T, whose sums the lane rescales by its own column's factor.  Which token stands at
// which place of an operand's reduction is free as long as both operands agree, so
// nothing moves between lanes.
//
// k_paged_direct works from global memory, on 32 tokens at a time: a lane reads its
// tokens' keys (rows of the first operand) in pieces of 16 bytes.  For 16-bit rows the values
// go through LDS, each wave's own tokens, and are read back transposed; fp32 products
// take them as they are, rows of V^T being dealt out so that a lane's are contiguous.
// !ROWS: few columns (a decoded token, a drafted chunk), bound by the cache's bytes: the
// four waves of a workgroup take every fourth tile of the tokens and join their sums,
// and S workgroups share a long sequence.  Blocks of W = 16 columns where there are no
// more: half the registers of 32.  ROWS (fp32): every wave 32 columns of its own,
// whose keys the waves of a workgroup find in the CU's cache.
template <int T, int C, int HD, int W, bool ROWS>
__global__ __launch_bounds__(256, (T == TLG_F32 && HD >= 128 && W == 32) || HD == 256 ? 1 : 2) void k_paged_direct(AttnArgs a)
{
    typedef typename ElT<C>::E E;
    typedef typename AccT<W>::A Acc;
    constexpr bool F = T == TLG_F32;
    constexpr int G = 64 / W, TB = 32 / W;                              // groups of lanes, blocks of tokens
    constexpr int NB = HD / W, NR = W * W / 64, NE = W / 2;             // blocks of a value, registers of a block, weights
    constexpr int ts = F ? 4 : 2, cs = C == TLG_F32 ? 4 : 2;
    constexpr int PE = F ? 4 : 8, NQ = HD / (PE * G), NK = NQ * TB, KW = PE * cs / 4;  // a key's pieces: elements, number, registers
    constexpr int NV = F ? NE : HD / 16, VW = F ? (NB * cs + 3) / 4 : 4;
    constexpr int VST = (HD / 2) % 64 == 16 || (HD / 2) % 64 == 48 ? HD : HD + 32;     // elements between tokens in LDS
    constexpr int MS = W + 4, BS = NB % 4 ? 2 : 4, MB = W == 32 ? 1 : BS;              // the sums' blocks joined at once
    constexpr int V1 = F ? 0 : 32 * VST * 2, M1 = MB * W * MS * 4, P1 = 1024;
    constexpr int PW = V1 > M1 ? (V1 > P1 ? V1 : P1) : (M1 > P1 ? M1 : P1);            // LDS of a wave
    __shared__ __align__(16) char mem[4 * PW];
    __shared__ long long toff[4][2][32];
    __shared__ float red[4][2][W];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane % W, g = lane / W;
    const int kvh = blockIdx.x % a.KV, s = blockIdx.x / a.KV % a.S, y = blockIdx.x / a.KV / a.S;
    int b = y, base = blockIdx.y * W;
    if (ROWS) {
        auto start = [&](int i) { return (long long)pg_row0(a.b, i) * a.G / 128 + i; };
        b = pg_search(a.b.B, y, start);
        base = (int)(y - start(b)) * 128 + 32 * wave;
    }
    const Seq q = pg_seq(a.b, b);
    const int cols = q.n * a.G;
    if (base < 0 || base >= cols || cols <= a.few || cols > a.many) return;
    const int *table = a.b.table + (long long)b * a.b.ldt;
    const E *Kc = (const E *)a.K + kvh * a.b.head_ld, *Vc = (const E *)a.V + kvh * a.b.head_ld;
    auto at = [](int blk, int m) { return F ? NB * m + blk : W * blk + m; };
    E *vs = (E *)(mem + wave * PW);

    for (int rh0 = base; rh0 < cols; rh0 += W * gridDim.y) {
        const Range rg = pg_range<32>(a, q, rh0, min(rh0 + W, cols));
        const int parts = pg_parts<32>(a, rg.total);
        if (s >= parts) {
            if (ROWS) return;
            continue;
        }
        const int j0 = (int)((long long)rg.total * s / parts), j1 = (int)((long long)rg.total * (s + 1) / parts);
        const int step = ROWS ? 1 : 4;
        // the lane's column
        const int rh = rh0 + col, ci = min(rh, cols - 1) / a.G, gq = min(rh, cols - 1) - ci * a.G;
        const bool live = rh < cols;
        const int r = q.lo + ci, p = live ? pg_pos(a, q, ci) : -1, from = pg_from(a, p);
        u32x4 qf[NQ];
        {
            const char *qp = a.q + ((long long)r * a.ldq + (kvh * a.G + gq) * HD + PE * g) * ts;
#pragma unroll
            for (int i = 0; i < NQ; i++) {
                qf[i] = *(const u32x4 *)(qp + i * PE * G * ts);
                if (!live) qf[i] = u32x4{0, 0, 0, 0};
            }
        }
        Acc o[NB];
#pragma unroll
        for (int i = 0; i < NB; i++)
#pragma unroll
            for (int k = 0; k < NR; k++) o[i][k] = 0.f;
        float R = -INFINITY, l = 0.f;

        unsigned kr[NK][KW], vr[NV][VW];
        // the page of token lane % 32 of tile j, then its elements
        auto page = [&](int j) {
            const int t = pg_tile<32>(rg, j) + (lane & 31), n = pg_of(a.b, t);
            return j < j1 && t <= rg.pmax && n < a.b.ldt ? table[n] : -1;
        };
        auto elems = [&](int j, int n) {
            const int t = pg_tile<32>(rg, j) + (lane & 31);
            return n >= 0 && n < a.b.n_pages ? n * a.b.page_ld + (t - pg_of(a.b, t) * a.b.page) * a.b.tok_ld : -1ll;
        };
        // a key that has no page is NaN in its first element of the lane's, and so are its scores
        bool lost[TB];
        auto loadK = [&](int buf, long long off) {
            if (lane < 32) toff[wave][buf][lane] = off;
            pg_wave_sync();
#pragma unroll
            for (int t = 0; t < TB; t++) {
                const long long k0 = toff[wave][buf][W * t + col];
                lost[t] = k0 < 0;
                const E *k = Kc + max(k0, 0ll) + PE * g;
#pragma unroll
                for (int i = 0; i < NQ; i++)
                    __builtin_memcpy(kr[t * NQ + i], __builtin_assume_aligned(k + i * PE * G, 4 * KW), 4 * KW);
            }
        };
        auto loadV = [&](int buf) {
            if constexpr (F) {
#pragma unroll
                for (int i = 0; i < NV; i++) {
                    const E *v = Vc + max(toff[wave][buf][pg_at<W>(i, g)], 0ll) + NB * col;
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
        if (j < j1) {
            loadK(0, elems(j, page(j)));
            loadV(0);
        }
        for (; j < j1; j += step, buf ^= 1) {
            const int t0 = pg_tile<32>(rg, j);
            const bool more = j + step < j1;
            const long long next = elems(j + step, ahead);
            ahead = page(j + 2 * step);
            // scores
            float e[NE];
#pragma unroll
            for (int t = 0; t < TB; t++) {
                Acc z;
#pragma unroll
                for (int i = 0; i < NR; i++) z[i] = 0.f;
                if (lost[t]) kr[t * NQ][0] = ~0u;
#pragma unroll
                for (int i = 0; i < NQ; i++) {
                    unsigned *k = kr[t * NQ + i];
                    if constexpr (!F) z = pg_mfma<T, W>(u32x4{k[0], k[1], k[2], k[3]}, qf[i], z);
                    else {
#pragma unroll
                        for (int x = 0; x < 4; x++) {
                            float f;
                            if constexpr (C == TLG_F32) f = __uint_as_float(k[x]);
                            else f = (float)__builtin_bit_cast(E, (unsigned short)(k[x / 2] >> (x & 1) * 16));
                            z = pg_mfma32<W>(f, __uint_as_float(qf[i][x]), z);
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < NR; i++) e[t * NR + i] = z[i];
            }
            if (more) loadK(buf ^ 1, next);
            // weights
            const bool full = t0 + 31 <= rg.pmin && (rg.lomax <= t0 || t0 + 31 < a.sinks);
            if (!full) {
#pragma unroll
                for (int i = 0; i < NE; i++) e[i] = pg_sees(a, t0 + pg_at<W>(i, g), p, from) ? e[i] : -INFINITY;
            }
            pg_weights<W, NE, NB>(e, a.c, R, l, o);
            bool odd = false;
            if (!full) {
#pragma unroll
                for (int i = 0; i < NV; i++) {
                    bool hit = false;
#pragma unroll
                    for (int k = 0; k < VW; k++) hit |= pg_clean<C>(vr[i][k]);
                    const int t = F ? pg_at<W>(i, g) : (lane + 64 * i) / (HD / 8);
                    odd |= hit && t0 + t <= rg.pmax;
                }
                odd = __any(odd);
            }
            // values
            if constexpr (F) {
#pragma unroll
                for (int i = 0; i < NV; i++)
#pragma unroll
                    for (int k = 0; k < NB; k++) {
                        float v;
                        if constexpr (C == TLG_F32) v = __uint_as_float(vr[i][k]);
                        else v = (float)__builtin_bit_cast(E, (unsigned short)(vr[i][k / 2] >> (k & 1) * 16));
                        o[k] = pg_mfma32<W>(v, e[i], o[k]);
                    }
                if (more) loadV(buf ^ 1);
            } else {
                pg_wave_sync();
#pragma unroll
                for (int i = 0; i < NV; i++) {
                    const int ch = lane + 64 * i, t = ch / (HD / 8), d = ch % (HD / 8) * 8;
                    *(u32x4 *)(vs + t * VST + d) = u32x4{vr[i][0], vr[i][1], vr[i][2], vr[i][3]};
                }
                if (more) loadV(buf ^ 1);
                pg_wave_sync();
                u32x4 pf[NE / 8];
#pragma unroll
                for (int i = 0; i < NE / 2; i++) pf[i / 4][i & 3] = pg_pack<T>(e[2 * i], e[2 * i + 1]);
                // sixteen lanes read four tokens of sixteen elements and get a column of them each
                const E *vt = vs + (4 * g + (lane >> 2 & 3)) * VST + (W == 32 ? 16 * (lane >> 4 & 1) : 0) + 4 * (lane & 3);
#pragma unroll
                for (int k = 0; k < NB; k++)
#pragma unroll
                    for (int i = 0; i < NE / 8; i++) {
                        const E *v = vt + 16 * i * VST + W * k;
                        const u32x2 v0 = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)v));
                        const u32x2 v1 =
                            __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(v + 4 * G * VST)));
                        o[k] = pg_mfma<T, W>(u32x4{v0[0], v0[1], v1[0], v1[1]}, pf[i], o[k]);
                    }
            }
            if (odd)
                pg_special<C, W, NB>(a, o, e, (float *)(mem + wave * PW), (const char *)Vc, t0, rg.pmax, p, from,
                                     [&](int k) { return toff[wave][buf][k]; }, at);
        }
        l = pg_gsum<W>(l);
        if constexpr (ROWS) {
            if (!live) return;
#pragma unroll
            for (int i = 0; i < NR; i++) {
                float x[NB];
#pragma unroll
                for (int k = 0; k < NB; k++) x[k] = o[k][i];
                pg_out<T, NB>(a, HD, s, parts, r, kvh * a.G + gq, NB * pg_at<W>(i, g), l, x);
            }
            if (g == 0) pg_out_sums(a, s, parts, r, kvh * a.G + gq, R, l);
            return;
        } else {
            // the waves' sums against the largest of their references
            if (g == 0) {
                red[wave][0][col] = R;
                red[wave][1][col] = l;
            }
            __syncthreads();
            auto top = [&](int c) { return fmaxf(fmaxf(red[0][0][c], red[1][0][c]), fmaxf(red[2][0][c], red[3][0][c])); };
            const float mine = top(col), f = __builtin_amdgcn_exp2f(R - (mine == -INFINITY ? 0.f : mine));
            // the thread's column, four rows of a block, and which of MB blocks
            const int ob = threadIdx.x / (W * W / 4), oc = threadIdx.x / (W / 4) % W, om = threadIdx.x % (W / 4) * 4;
            const float Rt = top(oc);
            float lt = 0.f;
#pragma unroll
            for (int w = 0; w < 4; w++)
                lt += red[w][1][oc] * __builtin_amdgcn_exp2f(red[w][0][oc] - (Rt == -INFINITY ? 0.f : Rt));
            const int orh = rh0 + oc, oi = min(orh, cols - 1) / a.G, hq = kvh * a.G + min(orh, cols - 1) - oi * a.G;
            float *mg = (float *)mem;
#pragma unroll
            for (int k0 = 0; k0 < NB; k0 += MB) {
                if (k0) __syncthreads();
#pragma unroll
                for (int k = 0; k < MB; k++)
#pragma unroll
                    for (int i = 0; i < NR; i += 4)
                        *(f32x4 *)(mg + ((wave * MB + k) * W + col) * MS + pg_at<W>(i, g)) =
                            f32x4{o[k0 + k][i], o[k0 + k][i + 1], o[k0 + k][i + 2], o[k0 + k][i + 3]} * f;
                __syncthreads();
                if (ob < MB && orh < cols) {
                    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int w = 0; w < 4; w++) v += *(const f32x4 *)(mg + ((w * MB + ob) * W + oc) * MS + om);
                    float x[4] = {v[0], v[1], v[2], v[3]};
                    if constexpr (F) {
#pragma unroll
                        for (int i = 0; i < 4; i++) pg_out<T, 1>(a, HD, s, parts, q.lo + oi, hq, at(k0 + ob, om + i), lt, x + i);
                    } else pg_out<T, 4>(a, HD, s, parts, q.lo + oi, hq, at(k0 + ob, om), lt, x);
                }
            }
            if (ob == 0 && om == 0 && orh < cols) pg_out_sums(a, s, parts, q.lo + oi, hq, Rt, lt);
            __syncthreads();                             // before another tile's waves write here
        }
    }
}

// The sums of the workgroups that shared a row's tokens: one wave a row and head.  Tiles
// of sequences of at most `few` columns had `small` of them, others `big` (their tokens in
// tiles of 32 or, with the flag, 64).
template <int T, int U> __global__ __launch_bounds__(256) void k_paged_join(AttnArgs a, int hd, int few, int small, int big, int by64)
{
    const int lane = threadIdx.x & 63;
    const long long rhd = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int r = __builtin_amdgcn_readfirstlane((int)(rhd / a.H)), head = __builtin_amdgcn_readfirstlane((int)(rhd % a.H));
    if (r >= a.b.N) return;
    const int b = pg_search(a.b.B, r, [&](int i) { return pg_row0(a.b, i); });
    const Seq q = pg_seq(a.b, b);
    if (r < q.lo || r >= q.lo + q.n) return;
    const int cols = q.n * a.G, rh = (r - q.lo) * a.G + head % a.G, w = cols <= few ? small : big;
    const int rh0 = rh / w * w, rh1 = min(rh0 + w, cols);
    const int parts = cols > few && by64 ? pg_parts<64>(a, pg_range<64>(a, q, rh0, rh1).total)
                                         : pg_parts<32>(a, pg_range<32>(a, q, rh0, rh1).total);
    if (parts < 2) return;
    const long long row = (long long)r * a.H + head, all = (long long)a.b.N * a.H;
    float R = -INFINITY, l = 0.f;
    if (lane < parts) {
        const float2 m = *(const float2 *)(a.pm + (row + lane * all) * 2);
        R = m.x;
        l = m.y;
    }
    // U workgroups' sums in flight at a time, four elements a lane (lanes beyond hd: none)
    const float *po = a.po + row * hd + 4 * lane;
    const bool in = 4 * lane < hd;
    f32x4 x = {0.f, 0.f, 0.f, 0.f}, v[U];
#pragma unroll
    for (int i = 0; i < U; i++) v[i] = in ? *(const f32x4 *)(po + min(i, parts - 1) * all * hd) : x;
    float top = R;
#pragma unroll
    for (int o = 32; o; o /= 2) top = fmaxf(top, __shfl_xor(top, o));
    const float f = __builtin_amdgcn_exp2f(R - (top == -INFINITY ? 0.f : top));
    l *= f;
#pragma unroll
    for (int o = 32; o; o /= 2) l += __shfl_xor(l, o);
    for (int s = 0; s < parts; s += U) {
#pragma unroll
        for (int i = 0; i < U; i++) {
            const float fs = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(f), min(s + i, 63)));
            if (s + i < parts) x += fs * v[i];
            if (s + U < parts) v[i] = in ? *(const f32x4 *)(po + min(s + U + i, parts - 1) * all * hd) : x;
        }
    }
    float y[4] = {x[0], x[1], x[2], x[3]};
    AttnArgs one = a;
    one.lse = nullptr;
    if (in) pg_out<T, 4>(one, hd, 0, 1, r, head, 4 * lane, l, y);
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
                 0xffffffffu / (unsigned)c->page, c->page_ld, c->tok_ld, c->head_ld};
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
#define PG_MIN 8                     /* tiles of 32 tokens of a workgroup, at least */
struct Plan {
    bool few, both;
    int W;                           // columns of a workgroup of few
    unsigned tiles, slots;           // of W columns of a sequence, of 128 of all
    int S, per;
    size_t sums;                     // bytes of the partial sums, before their references
};
static Plan pg_plan(const TlgPages *c, const TlgBatch *b, int H)
{
    Plan p = {};
    const int G = H / c->KV, rows = b->max_rows && b->max_rows < b->N ? b->max_rows : b->N;
    const long long cols = (long long)rows * G, room = (long long)b->ldt * c->page,
                    len = b->max_len && b->max_len < room ? b->max_len : room;
    p.few = cols <= PG_FEW;
    p.W = cols <= 16 ? 16 : 32;
    p.tiles = p.few ? (unsigned)((cols + p.W - 1) / p.W) : 1;
    p.slots = (unsigned)((long long)b->N * G / 128 + b->B);
    p.both = !p.few && (long long)b->B * rows > b->N;
    const long long groups = p.few ? (long long)b->B * p.tiles * c->KV : (long long)p.slots * c->KV,
                    row = (long long)b->N * H * (c->hd + 2) * 4, tiles = (len + 31) / 32;
    long long S = PG_FILL / groups;
    if (S > tiles / PG_MIN) S = tiles / PG_MIN;
    if (S > (128ll << 20) / row) S = (128ll << 20) / row;
    p.S = S < 1 ? 1 : S > 64 ? 64 : (int)S;
    p.per = (int)((tiles + p.S - 1) / p.S);
    if (p.per < PG_MIN) p.per = PG_MIN;
    p.per += p.per & 1;
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

template <int T, int C, int W, bool ROWS> static void pg_direct(const AttnArgs &a, int hd, dim3 grid, hipStream_t st)
{
    if (hd == 32) hipLaunchKernelGGL((k_paged_direct<T, C, 32, W, ROWS>), grid, dim3(256), 0, st, a);
    else if (hd == 64) hipLaunchKernelGGL((k_paged_direct<T, C, 64, W, ROWS>), grid, dim3(256), 0, st, a);
    else if (hd == 96) hipLaunchKernelGGL((k_paged_direct<T, C, 96, W, ROWS>), grid, dim3(256), 0, st, a);
    else if (hd == 128) hipLaunchKernelGGL((k_paged_direct<T, C, 128, W, ROWS>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((k_paged_direct<T, C, 256, W, ROWS>), grid, dim3(256), 0, st, a);
}
template <int W> static void pg_few(const AttnArgs &a, int type, int kv, int hd, dim3 grid, hipStream_t st)
{
    if (type == TLG_F16) pg_direct<TLG_F16, TLG_F16, W, false>(a, hd, grid, st);
    else if (type == TLG_BF16) pg_direct<TLG_BF16, TLG_BF16, W, false>(a, hd, grid, st);
    else if (kv == TLG_F32) pg_direct<TLG_F32, TLG_F32, W, false>(a, hd, grid, st);
    else if (kv == TLG_F16) pg_direct<TLG_F32, TLG_F16, W, false>(a, hd, grid, st);
    else pg_direct<TLG_F32, TLG_BF16, W, false>(a, hd, grid, st);
}
template <int T> static void pg_join(const AttnArgs &a, int hd, int few, int small, int big, int by64, dim3 grid, hipStream_t st)
{
    if (a.S <= 4) hipLaunchKernelGGL((k_paged_join<T, 4>), grid, dim3(256), 0, st, a, hd, few, small, big, by64);
    else hipLaunchKernelGGL((k_paged_join<T, 16>), grid, dim3(256), 0, st, a, hd, few, small, big, by64);
}
static void pg_rows32(const AttnArgs &a, int kv, int hd, dim3 grid, hipStream_t st)
{
    if (kv == TLG_F32) pg_direct<TLG_F32, TLG_F32, 32, true>(a, hd, grid, st);
    else if (kv == TLG_F16) pg_direct<TLG_F32, TLG_F16, 32, true>(a, hd, grid, st);
    else pg_direct<TLG_F32, TLG_BF16, 32, true>(a, hd, grid, st);
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
    a.per = p.per;
    a.few = 0;
    a.many = p.few ? INT_MAX : PG_FEW;
    a.po = (float *)ws;
    a.pm = (float *)((char *)ws + p.sums);
    hipStream_t st = ST(stream);
    if (p.few || p.both) {
        const dim3 grid((unsigned)b->B * c->KV * p.S, p.tiles);
        if (p.W == 16) pg_few<16>(a, type, c->type, c->hd, grid, st);
        else pg_few<32>(a, type, c->type, c->hd, grid, st);
    }
    if (!p.few) {
        a.few = p.both ? PG_FEW : 0;
        a.many = INT_MAX;
        if (type == TLG_F32) pg_rows32(a, c->type, c->hd, dim3(p.slots * c->KV * p.S), st);
        else pg_tile_launch(a, type, c->hd, p.slots * c->KV * p.S, st);
    }
    if (p.S > 1) {
        // few: every tile's columns were p.W, else those of the rows' kernel
        const int few = p.few ? INT_MAX : a.few, big = type == TLG_F32 ? 32 : PGT_ROWS,
                  by64 = type != TLG_F32 && PGT_TOKENS(c->hd) == 64;
        const dim3 grid((unsigned)(((long long)b->N * H + 3) / 4));
        if (type == TLG_F32) pg_join<TLG_F32>(a, c->hd, few, p.W, big, by64, grid, st);
        else if (type == TLG_F16) pg_join<TLG_F16>(a, c->hd, few, p.W, big, by64, grid, st);
        else pg_join<TLG_BF16>(a, c->hd, few, p.W, big, by64, grid, st);
    }
    LAUNCH_CHECK();
    return TLG_OK;
}
