// tlg_paged.hip -- a paged KV cache and the attention over it (include/tlserve.h): rows
// into the cache, attention of few rows a sequence and of fp32 rows, the joins of shared
// sums, and the entries.  tlg_paged_tile.hip has the attention of many 16-bit rows.
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
    int maxpos, per;             // rows of a workgroup
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

// A workgroup takes up to ST_ROWS consecutive rows; a thread eight pairs (i, i + hd/2) of
// a head.  Bound by the bytes of many rows (16384 rows of 48 heads of 128 bf16 values: 71
// us, 5.7 TB/s, a copy reaches 5.4), by the chain sequence - page - row of few, which one row
// a workgroup keeps shortest (300 such rows: 6.1 us, 9.7 with four; 16384 71 and 74).  Only many
// rows that leave half of a workgroup's threads without work are taken in fours: 24 heads of 64 fp16
// values, one / four: 300 rows 3.7 / 4.4 us, 1024 5.2 / 6.0, 4000 10.4 / 9.2, 16384 29.9 / 26.7; 18 of
// 32 fp32 3.7 / 3.8, 4.9 / 4.9, 8.7 / 7.9, 26.4 / 22.8; 48 of 64 bf16 4.0 / 5.7, 6.1 / 7.4, 15.9 / 15.4, 42.5 / 42.4.
#define ST_ROWS 4
#define ST_MANY 4096
template <int T, int C> __global__ __launch_bounds__(256) void k_paged_store(StoreArgs a)
{
    constexpr int ts = T == TLG_F32 ? 4 : 2, cs = C == TLG_F32 ? 4 : 2;
    const int lane = threadIdx.x & 63, r0 = blockIdx.x * a.per, half = a.hd >> 1, per = half >> 3;
    __shared__ int pos[ST_ROWS];                      // position, -1 none: no such row
    __shared__ long long at[ST_ROWS];                 // the token's elements in the cache, -1: not stored
    for (int k = threadIdx.x >> 6; k < a.per; k += 4) {
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
    for (int q = threadIdx.x; q < a.per * items; q += 256) {
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
// Units of a sequence's tiles of W columns (of each of them), 0 where a launch leaves it out.
__device__ __forceinline__ int pg_units(const AttnArgs &a, const Seq &q)
{
    const int cols = q.n * a.G;
    return cols > a.few && cols <= a.many ? max(1, pg_range<32>(a, q, 0, cols).total) : 0;
}
// Where each sequence's units start, [B + 1] in LDS; the workgroups that take part, each with
// PG_UNITS at least.  B <= PG_EVEN, 256 threads.  The units number less than 2^31, the host
// sees to it, unless row0 decreases and sequences share rows: then none takes part.
#define PG_EVEN 1024
#define PG_UNITS 4
template <int W> __device__ __forceinline__ int pg_places(const AttnArgs &a, int *place)
{
    __shared__ unsigned part[4];
    __shared__ int with[4];
    auto add = [](unsigned x, unsigned y) { return __builtin_elementwise_add_sat(x, y); };
    const int t = threadIdx.x, per = (a.b.B + 255) / 256, lane = t & 63;
    unsigned n[PG_EVEN / 256], sum = 0;
    int some = 0;
#pragma unroll
    for (int i = 0; i < PG_EVEN / 256; i++) {
        n[i] = 0;
        if (i < per && t * per + i < a.b.B) {
            const Seq q = pg_seq(a.b, t * per + i);
            n[i] = pg_units(a, q) * ((q.n * a.G + W - 1) / W);
        }
        sum = add(sum, n[i]);
        some += __popcll(__ballot(n[i] > 0));
    }
    unsigned upto = sum;
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
        const unsigned v = __shfl_up(upto, o);
        upto = add(upto, lane >= o ? v : 0);
    }
    if (lane == 63) {
        part[t >> 6] = upto;
        with[t >> 6] = some;
    }
    __syncthreads();
    unsigned all = 0;
#pragma unroll
    for (int w = 0; w < 4; w++) {
        if (w == t >> 6) upto = add(upto, all);
        all = add(all, part[w]);
    }
    if (all > INT_MAX) return 0;
    upto -= sum;
#pragma unroll
    for (int i = 0; i < PG_EVEN / 256; i++) {
        if (i < per && t * per + i < a.b.B) place[t * per + i] = upto;
        upto += n[i];
    }
    if (t == 0) place[a.b.B] = all;
    __syncthreads();
    // Small shares of equal sequences are cut alike: a second sequence in a share costs its
    // workgroup about 4 us, as much as 8 tiles or more.
    const int seqs = with[0] + with[1] + with[2] + with[3], P = min(a.P, max((int)all / PG_UNITS, all > 0 ? 1 : 0));
    return P > seqs && (int)all < 32 * P ? P / seqs * seqs : P;
}
// Share y of T units over P: the first T % P have one more.
__device__ __forceinline__ int pg_share(int T, int P, int y) { return T / P * y + min(y, T % P); }
__device__ __forceinline__ int pg_share_of(int T, int P, int u)
{
    const int n = T / P, more = T % P, k = u / (n + 1);
    return k < more ? k : more + (u - more * (n + 1)) / n;
}

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
// !ROWS: few columns (a decoded token, a drafted chunk), bound by the cache's bytes.  The
// tokens of all sequences, tile after tile, are dealt out evenly to the workgroups of a
// KV head, so that ragged lengths leave none idle; the four waves of a workgroup take
// every fourth of its tiles and join their sums.  Blocks of W = 16 columns where there
// are no more: half the registers of 32.  ROWS (fp32): every wave a block of columns of its
// own, whose keys the waves of a workgroup find in the CU's cache.
// Measured: 56 sequences of 1024 to 4096 tokens, 32 query and 8 KV heads of 128 bf16
// values, 118 us for 602 MB of cache (5.1 TB/s; a plain read reaches 7.1), one row over 131072
// tokens 102 us (5.2); 2000 sequences of up to 1024 tokens 5.3 TB/s.  256 to 512 workgroups
// are best; with three waves a SIMD or 1024 workgroups the same bytes take 8 to 12 % longer.
// fp32 prompts reach 70 to 93 TFLOP/s of 142.
// One workgroup a CU where two would spill (fp32 rows of 96 elements on, 256 elements).
template <int T, int C, int HD, int W, bool ROWS>
__global__ __launch_bounds__(256, (T == TLG_F32 && HD * (W == 32 || C == TLG_F32 ? 4 : 3) >= 384) || HD == 256 ? 1 : 2) void k_paged_direct(AttnArgs a)
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
    constexpr bool LATE = F && HD == 256;                               // keys and values do not fit the registers at once
    constexpr int MS = W + 4, BS = NB % 4 ? 2 : 4, MB = W == 32 ? 1 : BS;              // the sums' blocks joined at once
    constexpr int V1 = F ? 0 : 32 * VST * 2, M1 = MB * W * MS * 4, P1 = 1024;
    constexpr int PW = V1 > M1 ? (V1 > P1 ? V1 : P1) : (M1 > P1 ? M1 : P1);            // LDS of a wave
    __shared__ __align__(16) char mem[4 * PW];
    __shared__ long long toff[4][2][32];
    __shared__ float red[4][2][W];
    __shared__ int place[ROWS ? 1 : PG_EVEN + 1];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane % W, g = lane / W;
    const int kvh = blockIdx.x % a.KV, y = blockIdx.x / a.KV;
    const E *Kc = (const E *)a.K + kvh * a.b.head_ld, *Vc = (const E *)a.V + kvh * a.b.head_ld;
    auto at = [](int blk, int m) { return F ? NB * m + blk : W * blk + m; };
    E *vs = (E *)(mem + wave * PW);

    // the workgroup's share: units [u, u1) of the sequences' tiles of W columns by 32 tokens
    int b = y;
    int u = 0, u1 = 0;
    if constexpr (ROWS) {
        auto start = [&](int i) { return (long long)pg_row0(a.b, i) * a.G / (4 * W) + i; };
        b = pg_search(a.b.B, y / a.S, start);
        u = (int)(y / a.S - start(b));
    } else if (a.P) {
        const int P = pg_places<W>(a, place);
        if (blockIdx.x == 0)
            for (int i = threadIdx.x; i <= a.b.B + 1; i += 256) a.place[i] = i <= a.b.B ? place[i] : P;
        if (y >= P) return;
        u = pg_share(place[a.b.B], P, y);
        u1 = pg_share(place[a.b.B], P, y + 1);
        b = pg_search(a.b.B, u, [&](int i) { return place[i]; });       // the last that starts there: it has units
    } else b = y / a.S;
    const int s = ROWS || !a.P ? y % a.S : 0;
    for (bool first = true; first || (!ROWS && u < u1); first = false) {   // `continue` below: !P, u counts on
        const Seq q = pg_seq(a.b, b);
        const int cols = q.n * a.G;
        int rh0, t0seg = 0, t1seg = 0;
        bool only = true;
        if constexpr (ROWS) {
            rh0 = (4 * u + wave) * W;
            if (u < 0 || rh0 >= cols || cols <= a.few || cols > a.many) return;
        } else {
            const int tot = pg_units(a, q);
            if (tot == 0) return;                        // without places only: a sequence of no rows, or not this launch's
            if (a.P) {
                const int in = u - place[b], k = in / tot;
                rh0 = k * W;
                t0seg = in - k * tot;
                t1seg = min(tot, t0seg + u1 - u);
                only = t0seg == 0 && t1seg == tot;
                u += t1seg - t0seg;
            } else {                                     // its tiles of columns one after the other
                rh0 = u * W;
                u++;
                u1 = (cols + W - 1) / W;
            }
        }
        const Range rg = pg_range<32>(a, q, rh0, min(rh0 + W, cols));
        int parts = 1, j0, j1;
        if (ROWS || !a.P) {
            parts = pg_parts<32>(a, rg.total);
            if (s >= parts) {
                if (ROWS) return;
                continue;
            }
            j0 = (int)((long long)rg.total * s / parts);
            j1 = (int)((long long)rg.total * (s + 1) / parts);
        } else {
            j0 = min(t0seg, rg.total);
            j1 = min(t1seg, rg.total);
        }
        constexpr int step = ROWS ? 1 : 4;
        const int *table = a.b.table + (long long)b * a.b.ldt;
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
            if (!LATE) loadV(0);
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
            if (LATE) loadV(buf);
            else if (more) loadK(buf ^ 1, next);
            // weights
            const bool full = t0 + 31 <= rg.pmin && (rg.lomax <= t0 || t0 + 31 < a.sinks);
            if (!full) {
#pragma unroll
                for (int i = 0; i < NE; i++) e[i] = pg_sees(a, t0 + pg_at<W>(i, g), p, from) ? e[i] : -INFINITY;
            }
            pg_weights<T, W, NE, NB>(e, a.c, R, l, o);
            // 16-bit rows: in every tile, for an infinite value times a weight's second piece is none
            bool odd = !full;
            if constexpr (!F) odd = __any(pg_odd<C, NV, VW>(vr));
            if (odd) {
                odd = false;
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
                if (more && LATE) loadK(buf ^ 1, next);
                if (more && !LATE) loadV(buf ^ 1);
            } else {
                pg_wave_sync();
#pragma unroll
                for (int i = 0; i < NV; i++) {
                    const int ch = lane + 64 * i, t = ch / (HD / 8), d = ch % (HD / 8) * 8;
                    *(u32x4 *)(vs + t * VST + d) = u32x4{vr[i][0], vr[i][1], vr[i][2], vr[i][3]};
                }
                if (more) loadV(buf ^ 1);
                pg_wave_sync();
                // weights in two pieces, what rounding takes from the first one and that: the products
                // then keep 16 (bf16) or 22 bits of them (small fp16 ones fewer, PG_LIFT), in time that the cache's
                // bytes take anyway
                u32x4 pf[NE / 8], pr[NE / 8];
#pragma unroll
                for (int i = 0; i < NE / 2; i++) pg_split<T>(e[2 * i], e[2 * i + 1], pf[i / 4], pr[i / 4], i & 3);
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
                        const u32x4 vf = {v0[0], v0[1], v1[0], v1[1]};
                        o[k] = pg_mfma<T, W>(vf, pf[i], o[k]);
                        o[k] = pg_mfma<T, W>(vf, pr[i], o[k]);
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
                pg_out<T, NB>(a, HD, pg_part(a, a.po, HD, s, parts, r, kvh * a.G + gq), r, kvh * a.G + gq, NB * pg_at<W>(i, g), l,
                              x);
            }
            if (g == 0) pg_out_sums(a, pg_part(a, a.pm, 2, s, parts, r, kvh * a.G + gq), r, kvh * a.G + gq, R, l);
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
            // a tile that goes on from another workgroup's, and one that another goes on with, have places of their own
            const long long slot = (((long long)y * a.KV + kvh) * 2 + (t0seg == 0)) * W + oc;
            float *eo = only ? nullptr : a.eo + slot * HD, *em = only ? nullptr : a.em + slot * 2;
            if (!a.P) {
                eo = pg_part(a, a.po, HD, s, parts, q.lo + oi, hq);
                em = pg_part(a, a.pm, 2, s, parts, q.lo + oi, hq);
            }
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
                        for (int i = 0; i < 4; i++) pg_out<T, 1>(a, HD, eo, q.lo + oi, hq, at(k0 + ob, om + i), lt, x + i);
                    } else pg_out<T, 4>(a, HD, eo, q.lo + oi, hq, at(k0 + ob, om), lt, x);
                }
            }
            if (ob == 0 && om == 0 && orh < cols) pg_out_sums(a, em, q.lo + oi, hq, Rt, lt);
            __syncthreads();                             // before another tile's waves write here
            if (a.P)
                while (u < u1 && place[b + 1] <= u) b++;
        }
    }
}

// The sums of the workgroups that shared a row's tokens: one wave a row and head, or, for
// few rows, four that take a quarter of the sums each (64 sums of 128 elements: 6.7 us
// against 21; 1792 rows with four sums: 8.5 against 5).  EVEN:
// those of k_paged_direct in tiles of `w` columns; else of the rows' kernels, whose tiles of `w`
// columns had their tokens in tiles of 32 or, with the flag, 64.
template <int T, bool EVEN, int WV>
__device__ __forceinline__ void pg_join_row(const AttnArgs &a, int hd, int w, int by64, int rhd)
{
    constexpr int U = 8;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int part = WV == 4 ? wave : 0, r = rhd / a.H, head = rhd - r * a.H;
    const int b = pg_search(a.b.B, r, [&](int i) { return pg_row0(a.b, i); });
    const Seq q = pg_seq(a.b, b);
    if (r < q.lo || r >= q.lo + q.n) return;
    const int cols = q.n * a.G, rh = (r - q.lo) * a.G + head % a.G, kvh = head / a.G;
    if (cols <= a.few || cols > a.many) return;
    int parts;
    long long first, second, apart;                      // places (columns) of the first sums, the second, and from one to the next
    const float *po, *pm;
    if constexpr (EVEN) {
        // cut to what there is, should another call have written to this workspace
        const int all = a.place[a.b.B], P = min(a.place[a.b.B + 1], a.P), from = a.place[b], tiles = (cols + w - 1) / w,
                  tot = (a.place[b + 1] - from) / tiles, u = from + rh / w * tot;
        if (P < 1 || all < P || tot < 1) return;
        const long long i0 = min(max(pg_share_of(all, P, u), 0), P - 1), i1 = min(max(pg_share_of(all, P, u + tot - 1), (int)i0), P - 1);
        parts = (int)(i1 - i0 + 1);
        first = ((i0 * a.KV + kvh) * 2 + 1) * w + rh % w;
        second = ((i0 + 1) * a.KV + kvh) * 2 * w + rh % w;
        apart = 2ll * a.KV * w;
        po = a.eo;
        pm = a.em;
    } else {
        const int rh0 = rh / w * w, rh1 = min(rh0 + w, cols);
        parts = by64 ? pg_parts<64>(a, pg_range<64>(a, q, rh0, rh1).total) : pg_parts<32>(a, pg_range<32>(a, q, rh0, rh1).total);
        first = (long long)r * a.H + head;
        apart = (long long)a.b.N * a.H;
        second = first + apart;
        po = a.po;
        pm = a.pm;
    }
    if (parts < 2) return;
    auto where = [&](int p) { return p == 0 ? first : second + (p - 1) * apart; };
    float top = -INFINITY;
    for (int p = lane; p < parts; p += 64) top = fmaxf(top, pm[where(p) * 2]);
#pragma unroll
    for (int o = 32; o; o /= 2) top = fmaxf(top, __shfl_xor(top, o));
    // U workgroups' sums in flight at a time, four elements a lane (lanes beyond hd: none)
    const bool in = 4 * lane < hd;
    const float *e = po + 4 * lane;
    f32x4 x = {0.f, 0.f, 0.f, 0.f};
    float l = 0.f;
    for (int p0 = U * part; p0 < parts; p0 += WV * U) {
        f32x4 v[U];
        float f = 0.f;
#pragma unroll
        for (int i = 0; i < U; i++) v[i] = in ? *(const f32x4 *)(e + where(min(p0 + i, parts - 1)) * hd) : f32x4{0.f, 0.f, 0.f, 0.f};
        if (lane < U && p0 + lane < parts) {
            const float2 m = *(const float2 *)(pm + where(p0 + lane) * 2);
            f = __builtin_amdgcn_exp2f(m.x - (top == -INFINITY ? 0.f : top));
            l += f * m.y;
        }
#pragma unroll
        for (int i = 0; i < U; i++) {
            const float fi = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(f), i));
            if (p0 + i < parts) x += fi * v[i];
        }
    }
#pragma unroll
    for (int o = 32; o; o /= 2) l += __shfl_xor(l, o);
    if constexpr (WV == 4) {
        __shared__ f32x4 xs[4][64];
        __shared__ float ls[4];
        xs[wave][lane] = x;
        if (lane == 0) ls[wave] = l;
        __syncthreads();
        if (wave) return;
        x = (xs[0][lane] + xs[1][lane]) + (xs[2][lane] + xs[3][lane]);
        l = (ls[0] + ls[1]) + (ls[2] + ls[3]);
    }
    float y[4] = {x[0], x[1], x[2], x[3]};
    if (in) pg_out<T, 4>(a, hd, nullptr, r, head, 4 * lane, l, y);
    if (lane == 0) pg_out_sums(a, nullptr, r, head, top, l);
}
template <int T, bool EVEN, int WV> __global__ __launch_bounds__(256) void k_paged_join(AttnArgs a, int hd, int w, int by64)
{
    if constexpr (WV == 4) pg_join_row<T, EVEN, 4>(a, hd, w, by64, blockIdx.x);
    else
        for (int i = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6)); i < a.b.N * a.H; i += gridDim.x * 4)
            pg_join_row<T, EVEN, 1>(a, hd, w, by64, i);
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
    // without columns the table is not looked at, but a first entry of it may be read
    *o = PgBatch{b->row0, b->len, b->ldt ? b->table : b->row0, b->B, b->N, b->ldt, c->page, c->n_pages,
                 0xffffffffu / (unsigned)c->page, c->page_ld, c->tok_ld, c->head_ld};
    *work = 1;
    return TLG_OK;
}
static bool pg_rows(const void *p, long long ld, long long width, int type)
{
    return pg_al(p, 16) && ld >= width && ld <= 1ll << 40 && ld % (16 / (long long)pg_size(type)) == 0;
}

// memory from the first to the last element of two sets of N rows meets
static bool pg_meet(const void *a, long long lda, const void *b, long long ldb, long long width, int type, int N)
{
    const uintptr_t e = pg_size(type), a0 = (uintptr_t)a, b0 = (uintptr_t)b;
    return a0 < b0 + ((uintptr_t)(N - 1) * ldb + width) * e && b0 < a0 + ((uintptr_t)(N - 1) * lda + width) * e;
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
    if (q && !(q == q_out && ldq == ldqo) && pg_meet(q, ldq, q_out, ldqo, wq, type, b->N))
        return tlg_fail(TLG_EINVAL, "paged_store: q_out overlaps q without being the same rows");
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
    a.per = b->N >= ST_MANY && (a.H + 2 * a.KV) * (a.hd / 16) <= 128 ? ST_ROWS : 1;
    const dim3 grid((b->N + a.per - 1) / a.per), block(256);
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
// decide.  few: only k_paged_direct; else the rows' kernel, and, where that helps (both) and the
// numbers of rows differ, the former for the sequences of few.
// 16-bit rows are few up to PG_FEW.  us by k_paged_direct / by the rows' kernel, 32 / 8 heads:
//   columns                         24         32         36         48
//   8 x 8192 tokens, 128 bf16   65.3/88.2  66.5/64.2  79.6/67.5  80.5/68.0
//   32 x 1024                   43.3/44.0  46.8/46.7  66.4/54.8  70.0/55.3
//   4 x 300                     13.0/18.5  13.2/18.5  22.1/18.7  22.5/18.7
//   8 x 8192, 64 fp16           43.5/44.7  44.1/38.6  54.6/44.7  55.2/48.4
//   32 x 1024                   31.7/33.2  34.3/35.4  45.6/37.8  48.6/37.9
//   8 x 8192, 32 fp16           34.5/36.2  34.8/33.2  40.4/37.8  40.8/40.2
//   8 x 8192, 256 bf16           138/236    138/181    257/186    255/186
// fp32 rows up to twice that, over sequences of more than PG_SHORT tiles:
//   columns                         36         64         68        128
//   32 x 1024, 128 fp32          148/219    163/236    219/288    301/442
//   8 x 1000                      55/62      62/65      79/67     111/76
//   4 x 300                       49/60      51/61      72/61      96/63
//   8 x 8192, 32 over fp16        71/80      72/91     101/109    129/157
//   8 x 1000                      25/28      27/30      34/30      46/33
//   4 x 300                       23/20      24/21      33/20      43/21
// both: over more than PG_SHORT tiles, for a row over many tokens must not be left to one of the
// rows' kernel's workgroups.  us in two launches / by the rows' kernel alone, 32 / 8 heads:
//   tokens of each                   256       512      1024       4000
//   4 x 60 rows, 60 x 1, 128 bf16   39/32     58/49     97/84    291/263
//                        64 fp16    27/18     40/26     64/42    185/141
//                        256 bf16   71/84    109/141   189/253   536/798
//                        128 fp32  102/147   137/253   203/458
//                        32 fp32    38/32     59/56     80/86              (over fp16)
//   2048 rows, 1 row over 8192 and 65536, 128 bf16: 129/284, 170/2110; 64 fp16 92/183, 113/1356
// k_paged_direct's workgroups share the batch's tokens evenly from PG_LONG tiles of a
// sequence on (64 sequences of 1024 to 4096 tokens: 139 us against 148 where each is cut
// alike; of 525 to 2100 74 and 72), up to PG_MANY sequences times KV heads (200 of 525 to 2100: 227 and
// 207, the price of batches of one long sequence among short ones; 512 547 and 500) and PG_EVEN
// sequences, what the table of places holds; below PG_LONG, where looking up the batch costs
// more than that gains, each is cut alike (32 sequences of 5 rows that see 1028 tokens: 18 us against 24).
// fp32 rows take blocks of 16 columns a wave where those of 32 do not fill the chip (4
// prompts of 256 rows, 8 heads of 32: 14 us, 18 in blocks of 32; of 128 elements 68 and 58, so not there).
// Many rows' partial sums cost more than their tokens' division gains, unless the
// chip is not filled or every part is long (4 prompts of 300 rows, 32 heads of 128 bf16: 28 us
// whole, 68 in two parts; 512 rows over 8192 tokens 120 us in seven parts, 129 in five; before weights
// were in two pieces).
#define PG_FEW 32
#define PG_FILL 512                  /* workgroups wanted of k_paged_direct: two a CU */
#define PG_FILL_TILE 384             /* of k_paged_tile                     */
#define PG_FILL_ROWS 1024            /* of k_paged_direct for fp32 rows: short waves, one SIMD each */
#define PG_LONG 64                   /* tiles of 32 tokens                  */
#define PG_SHORT 16                  /* tiles up to which the rows' kernels take sequences of few rows too */
#define PG_MANY 2048                 /* sequences times KV heads that need no sharing */
struct Plan {
    bool few, both;
    int border;                      // columns of the sequences that are k_paged_direct's
    int W;                           // columns of a workgroup of few
    int wide;                        // of a workgroup of the rows' kernel
    unsigned slots;                  // and how many
    int P, Sf, perf, S, per;         // few: shares, or parts of a sequence; the rows' kernel's parts
    size_t po, pm, place, eo, em, bytes;
};
// Parts of a sequence: until `fill` workgroups work, with 8 tiles at least each.
static int pg_cut(long long groups, long long fill, long long tiles, long long row)
{
    long long S = fill / groups;
    if (S > tiles / 8) S = tiles / 8;
    if (S > (128ll << 20) / row) S = (128ll << 20) / row;
    return S < 1 ? 1 : S > 64 ? 64 : (int)S;
}
static int pg_per(long long tiles, int S)
{
    const long long n = (tiles + S - 1) / S;
    return (int)(n < 8 ? 8 : n + (n & 1));
}
static Plan pg_plan(const TlgPages *c, const TlgBatch *b, int type, int H, int win, int sinks, bool alike)
{
    Plan p = {};
    const int G = H / c->KV, rows = b->max_rows && b->max_rows < b->N ? b->max_rows : b->N;
    const long long cols = (long long)rows * G, room = (long long)b->ldt * c->page,
                    most = b->max_len && b->max_len < room ? b->max_len : room,
                    seen = win ? (long long)win + rows + (sinks < most ? sinks : most) + 64 : most,
                    tiles = ((seen < most ? seen : most) + 31) / 32, row = (long long)b->N * H * (c->hd + 2) * 4;
    // by the tokens that there are, not those in a window: the workspace is sized without one
    p.border = type == TLG_F32 && most > 32 * PG_SHORT ? 2 * PG_FEW : PG_FEW;
    p.few = cols <= p.border;
    p.W = cols <= 16 || c->hd == 256 ? 16 : 32;            // 32 of 256 elements do not fit the registers
    p.wide = PGT_ROWS;
    if (type == TLG_F32 && (c->hd == 256 || (c->hd <= 64 && ((long long)b->N * G / 128 + b->B) * c->KV < PG_FILL))) p.wide = 64;
    p.both = !p.few && (long long)b->B * rows > b->N && tiles > PG_SHORT;
    p.slots = (unsigned)((long long)b->N * G / p.wide + b->B);
    p.S = p.Sf = 1;
    if (p.few || p.both) {
        // units that the batch may hold, whatever the hints say
        const double units = ((double)b->N * G / p.W + b->B) * (room / 32 + 2);
        if (!alike && tiles > PG_LONG && b->B <= PG_EVEN && (long long)b->B * c->KV < PG_MANY && units < 2e9) {
            p.P = PG_FILL / c->KV;
            if (p.P < b->B) p.P = b->B;
        } else p.Sf = pg_cut((long long)b->B * c->KV, PG_FILL, tiles, row);
    }
    if (!p.few) {
        // the tiles that there are: of each sequence's last, half, in the mean
        const long long groups = ((long long)b->N * G / p.wide + (b->B + 1) / 2) * c->KV;
        const int fill = type == TLG_F32 ? PG_FILL_ROWS : PG_FILL_TILE, one = pg_cut(groups, fill, tiles, row),
                  two = pg_cut(groups, 2 * fill, tiles / 4, row);
        p.S = one > two ? one : two;
    }
    p.perf = pg_per(tiles, p.Sf);
    p.per = pg_per(tiles, p.S);
    const int S = p.S > p.Sf ? p.S : p.Sf;
    const size_t parts = S > 1 ? (size_t)S * b->N * H : 0, even = (size_t)p.P * c->KV * 2 * p.W;
    p.pm = parts * c->hd * 4;
    p.place = (p.pm + parts * 8 + 15) & ~(size_t)15;
    p.eo = (p.place + (p.P ? (b->B + 2) * 4 : 0) + 15) & ~(size_t)15;
    p.em = p.eo + even * c->hd * 4;
    p.bytes = p.em + even * 8;
    return p;
}

extern "C" size_t tlg_paged_attn_ws_bytes(const TlgPages *c, const TlgBatch *b, int type, int H)
{
    if (!c || !b || c->KV <= 0 || H < c->KV || b->N <= 0 || b->B <= 0 || c->hd <= 0 || c->page <= 0 || b->ldt < 0 ||
        b->max_rows < 0 || b->max_len < 0)
        return 0;
    // whatever the window leaves of the tokens: fewer are cut into fewer parts
    const size_t even = pg_plan(c, b, type, H, 0, 0, false).bytes, alike = pg_plan(c, b, type, H, 0, 0, true).bytes;
    return even > alike ? even : alike;
}

template <int T, int C, int W> static void pg_few(const AttnArgs &a, int hd, dim3 grid, hipStream_t st)
{
    if (hd == 32) hipLaunchKernelGGL((k_paged_direct<T, C, 32, W, false>), grid, dim3(256), 0, st, a);
    else if (hd == 64) hipLaunchKernelGGL((k_paged_direct<T, C, 64, W, false>), grid, dim3(256), 0, st, a);
    else if (hd == 96) hipLaunchKernelGGL((k_paged_direct<T, C, 96, W, false>), grid, dim3(256), 0, st, a);
    else if (hd == 128) hipLaunchKernelGGL((k_paged_direct<T, C, 128, W, false>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((k_paged_direct<T, C, 256, 16, false>), grid, dim3(256), 0, st, a);
}
template <int W> static void pg_few(const AttnArgs &a, int type, int kv, int hd, dim3 grid, hipStream_t st)
{
    if (type == TLG_F16) pg_few<TLG_F16, TLG_F16, W>(a, hd, grid, st);
    else if (type == TLG_BF16) pg_few<TLG_BF16, TLG_BF16, W>(a, hd, grid, st);
    else if (kv == TLG_F32) pg_few<TLG_F32, TLG_F32, W>(a, hd, grid, st);
    else if (kv == TLG_F16) pg_few<TLG_F32, TLG_F16, W>(a, hd, grid, st);
    else pg_few<TLG_F32, TLG_BF16, W>(a, hd, grid, st);
}
template <bool EVEN, int WV> static void pg_join(const AttnArgs &a, int type, int hd, int w, int by64, hipStream_t st)
{
    const long long groups = ((long long)a.b.N * a.H * WV + 3) / 4;
    const dim3 grid((unsigned)(groups < 1 << 16 ? groups : 1 << 16));
    if (type == TLG_F32) hipLaunchKernelGGL((k_paged_join<TLG_F32, EVEN, WV>), grid, dim3(256), 0, st, a, hd, w, by64);
    else if (type == TLG_F16) hipLaunchKernelGGL((k_paged_join<TLG_F16, EVEN, WV>), grid, dim3(256), 0, st, a, hd, w, by64);
    else hipLaunchKernelGGL((k_paged_join<TLG_BF16, EVEN, WV>), grid, dim3(256), 0, st, a, hd, w, by64);
}
template <bool EVEN> static void pg_join(const AttnArgs &a, int type, int hd, int w, int by64, hipStream_t st)
{
    if ((long long)a.b.N * a.H < 512) pg_join<EVEN, 4>(a, type, hd, w, by64, st);
    else pg_join<EVEN, 1>(a, type, hd, w, by64, st);
}
template <int C, int W> static void pg_rows32(const AttnArgs &a, int hd, dim3 grid, hipStream_t st)
{
    if (hd == 32) hipLaunchKernelGGL((k_paged_direct<TLG_F32, C, 32, W, true>), grid, dim3(256), 0, st, a);
    else if (hd == 64) hipLaunchKernelGGL((k_paged_direct<TLG_F32, C, 64, W, true>), grid, dim3(256), 0, st, a);
    else if (hd == 96) hipLaunchKernelGGL((k_paged_direct<TLG_F32, C, 96, W, true>), grid, dim3(256), 0, st, a);
    else if (hd == 128) hipLaunchKernelGGL((k_paged_direct<TLG_F32, C, 128, W, true>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((k_paged_direct<TLG_F32, C, 256, 16, true>), grid, dim3(256), 0, st, a);
}
template <int C> static void pg_rows32(const AttnArgs &a, int wide, int hd, dim3 grid, hipStream_t st)
{
    if (wide == 64) pg_rows32<C, 16>(a, hd, grid, st);
    else pg_rows32<C, 32>(a, hd, grid, st);
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
    if ((long long)b->N * H > 1 << 29 || (long long)b->B * c->KV > 1 << 22)           // what a grid takes
        return tlg_fail(TLG_EINVAL, "paged_attn: N=%d H=%d B=%d KV=%d", b->N, H, b->B, c->KV);
    if (!(scale >= 1e-30f && scale <= 1e30f) || win < 0 || sinks < 0)
        return tlg_fail(TLG_EINVAL, "paged_attn: scale=%g win=%d sinks=%d", scale, win, sinks);
    if (!work) return TLG_OK;
    const long long w = (long long)H * c->hd;
    if (!pg_rows(q, ldq, w, type) || !pg_rows(out, ldo, w, type) || (lse && !pg_al(lse, 4)))
        return tlg_fail(TLG_EINVAL, "paged_attn: q %p ldq=%lld out %p ldo=%lld lse %p", q, ldq, out, ldo, (void *)lse);
    if (pg_meet(q, ldq, out, ldo, w, type, b->N)) return tlg_fail(TLG_EINVAL, "paged_attn: out overlaps q");
    a.win = win < TLG_PAGED_LEN + 1 ? win : 0;            // a longer one hides nothing
    a.sinks = sinks < TLG_PAGED_LEN ? sinks : TLG_PAGED_LEN;
    const Plan p = pg_plan(c, b, type, H, a.win, a.sinks, false);
    size_t need = tlg_paged_attn_ws_bytes(c, b, type, H);
    if (p.bytes > need) need = p.bytes;                  // never: a window only lessens the plan's parts
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
    a.c = (float)((double)scale * 1.4426950408889634);
    if (c->n_pages == 0) {               // no token has a page: any readable memory stands for the first
        a.K = a.V = a.q;
        a.b.head_ld = 0;
    }
    a.P = p.P;
    a.po = (float *)ws;
    a.pm = (float *)((char *)ws + p.pm);
    a.place = (int *)((char *)ws + p.place);
    a.eo = (float *)((char *)ws + p.eo);
    a.em = (float *)((char *)ws + p.em);
    hipStream_t st = ST(stream);
    if (p.few || p.both) {
        a.few = 0;
        a.many = p.few ? INT_MAX : p.border;
        a.S = p.Sf;
        a.per = p.perf;
        const dim3 grid((unsigned)(p.P ? p.P : b->B * p.Sf) * c->KV);
        if (p.W == 16) pg_few<16>(a, type, c->type, c->hd, grid, st);
        else pg_few<32>(a, type, c->type, c->hd, grid, st);
        if (p.P) pg_join<true>(a, type, c->hd, p.W, 0, st);
        else if (p.Sf > 1) pg_join<false>(a, type, c->hd, p.W, 0, st);
    }
    if (!p.few) {
        a.few = p.both ? p.border : 0;
        a.many = INT_MAX;
        a.S = p.S;
        a.per = p.per;
        const dim3 grid(p.slots * c->KV * p.S);
        if (type == TLG_F32 && c->type == TLG_F32) pg_rows32<TLG_F32>(a, p.wide, c->hd, grid, st);
        else if (type == TLG_F32 && c->type == TLG_F16) pg_rows32<TLG_F16>(a, p.wide, c->hd, grid, st);
        else if (type == TLG_F32) pg_rows32<TLG_BF16>(a, p.wide, c->hd, grid, st);
        else pg_tile_launch(a, type, c->hd, grid.x, st);
        if (p.S > 1) pg_join<false>(a, type, c->hd, type == TLG_F32 ? p.wide / 4 : PGT_ROWS, type != TLG_F32 && PGT_TOKENS(c->hd) == 64, st);
    }
    LAUNCH_CHECK();
    return TLG_OK;
}
