// tlg_paged.h -- batches of sequences over a paged KV cache, as the kernels of
// tlg_paged.hip and tlg_paged_tile.hip see them.
#pragma once
#include "tlg_internal.h"
#include "../../include/tlserve.h"
#include <math.h>
#include <limits.h>

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
    unsigned magic;              // floor((2^32 - 1) / page)
    long long page_ld, tok_ld, head_ld;
};
// t / page for 0 <= t < 2^31: the product is t / page or one less (its error is below t / 2^32 + 1)
__device__ __forceinline__ int pg_of(const PgBatch &b, int t)
{
    const int g = (int)__umulhi((unsigned)t, b.magic);
    return g + (t - g * b.page >= b.page);
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

// --------------------------------------------------------------- attention --
struct AttnArgs {
    PgBatch b;
    const char *K, *V, *q;
    char *out;
    float *lse;
    long long ldq, ldo;
    int H, KV, G, win, sinks;
    int few, many;               // columns (rows times heads of a KV head) of the sequences that a launch takes: more than few, many at most
    float c;                     // scale log2 e
    // S workgroups share a tile's tokens, `per` tiles of 32 tokens each; S > 1: their sums
    // [S][N][H][hd] and references and weights [S][N][H][2]
    int S, per;
    float *po, *pm;
    // k_paged_direct, P > 0: P workgroups of a KV head share the tokens of all sequences evenly
    // instead, with the place of each sequence [B + 1] and the number that took part, and
    // the sums of tiles that are not one workgroup's, [P][KV][2][W][hd] and [..][2]
    int P;
    int *place;
    float *eo, *em;
};

// Base-2 scores against a reference: with R the largest c (q . k) of a row so far less PG_LIFT,
// rounded once, a weight is 2^(c (q . k) - R), one fused product, and whatever R is
// exactly, it is the same for all of a row's tokens.  R stays while the largest weight stays below
// 2^(PG_LIFT + PG_SLACK), so that the sums are rarely rescaled; weights up to 2^8 lose nothing in
// bf16 or fp32.  fp16's smallest step is 2^-24: with largest weights of 2^11 to 2^15 two pieces
// keep 22 bits of weights above 2^-14 of the row's largest and are off by 2^-36 of that at most
// below, which many small equal weights may add up to.
template <int T> constexpr float PG_LIFT = T == TLG_F16 ? 11.0f : 0.0f;
template <int T> constexpr float PG_SLACK = T == TLG_F16 ? 4.0f : 8.0f;

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 *lds_s16x4;
template <int T> struct Vec8 { typedef typename ElT<T>::E E; typedef E e8 __attribute__((ext_vector_type(8))); };
// Products of W x W blocks (W 32 or 16): the lane's column is lane % W, its group lane
// / W; register i of a result is row pg_at<W>(i, group).  16-bit operands have eight
// reduction elements a lane, fp32 ones one.
template <int W> struct AccT;
template <> struct AccT<32> { typedef f32x16 A; };
template <> struct AccT<16> { typedef f32x4 A; };
template <int W> __device__ __forceinline__ int pg_at(int i, int group) { return 256 / W * (i >> 2) + 4 * group + (i & 3); }
template <int T, int W>
__device__ __forceinline__ typename AccT<W>::A pg_mfma(u32x4 a, u32x4 b, typename AccT<W>::A c)
{
    typedef typename Vec8<T>::e8 e8;
    const e8 x = __builtin_bit_cast(e8, a), y = __builtin_bit_cast(e8, b);
    if constexpr (T == TLG_F16 && W == 32) return __builtin_amdgcn_mfma_f32_32x32x16_f16(x, y, c, 0, 0, 0);
    else if constexpr (T == TLG_F16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(x, y, c, 0, 0, 0);
    else if constexpr (W == 32) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, y, c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, y, c, 0, 0, 0);
}
template <int W> __device__ __forceinline__ typename AccT<W>::A pg_mfma32(float a, float b, typename AccT<W>::A c)
{
    if constexpr (W == 32) return __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}
template <int T> __device__ __forceinline__ unsigned pg_pack(float lo, float hi)      // rounded to nearest even
{
    typedef typename ElT<T>::E e2 __attribute__((ext_vector_type(2)));
    const e2 v = {(typename ElT<T>::E)lo, (typename ElT<T>::E)hi};
    return __builtin_bit_cast(unsigned, v);
}
// Two weights as register k of two operands whose sum they are to twice the type's bits: rounded, and
// what that took from them (exact in fp32), rounded.  (The barrier: the compiler would round each
// weight by itself a second time to have it as a float.)
template <int T> __device__ __forceinline__ void pg_split(float x, float y, u32x4 &hi, u32x4 &lo, int k)
{
    unsigned w = pg_pack<T>(x, y);
    asm("" : "+v"(w));
    typedef typename ElT<T>::E e2 __attribute__((ext_vector_type(2)));
    const e2 back = __builtin_bit_cast(e2, w);
    hi[k] = w;
    lo[k] = pg_pack<T>(x - (float)back[0], y - (float)back[1]);
}
// Sum and maximum over the groups of lanes that share a column, in every lane.
template <int W, typename OP> __device__ __forceinline__ float pg_groups(float v, OP op)
{
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = op(__uint_as_float(r[0]), __uint_as_float(r[1]));
    if constexpr (W == 16) {
        const auto q = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = op(__uint_as_float(q[0]), __uint_as_float(q[1]));
    }
    return v;
}
template <int W> __device__ __forceinline__ float pg_gmax(float v)
{
    return pg_groups<W>(v, [](float a, float b) { return fmaxf(a, b); });
}
template <int W> __device__ __forceinline__ float pg_gsum(float v)
{
    return pg_groups<W>(v, [](float a, float b) { return a + b; });
}

// A sequence of the batch, and the column of a tile that a lane has: the row i and
// query head g of its KV head, rh = i G + g of n G.
struct Seq { int lo, n, len; };
__device__ __forceinline__ Seq pg_seq(const PgBatch &b, int s)
{
    Seq q;
    q.lo = pg_row0(b, s);
    q.n = max(pg_row0(b, s + 1) - q.lo, 0);
    q.len = max(b.len[s], 0);
    return q;
}
// Positions are cut to `cap`, the first token that no table has a column for: it
// stands for all of them, as a token without a page.
__device__ __forceinline__ int pg_pos(const AttnArgs &a, const Seq &q, int i)
{
    return min(q.len - q.n + i, a.b.ldt * a.b.page);
}
__device__ __forceinline__ int pg_from(const AttnArgs &a, int p) { return a.win ? max(0, p - a.win + 1) : 0; }

// The tokens that columns [rh0, rh1) of a sequence see, in tiles of TT: `sink` tiles
// from 0 on, then those from tile `first` on, `total` in all.
struct Range { int pmin, pmax, lomax, sink, first, total; };
template <int TT> __device__ __forceinline__ Range pg_range(const AttnArgs &a, const Seq &q, int rh0, int rh1)
{
    Range r;
    r.pmin = pg_pos(a, q, rh0 / a.G);
    r.pmax = pg_pos(a, q, (rh1 - 1) / a.G);
    r.lomax = pg_from(a, r.pmax);
    r.first = pg_from(a, r.pmin) / TT;
    r.sink = min((a.sinks + TT - 1) / TT, r.first);
    r.total = r.pmax < 0 ? 0 : r.sink + r.pmax / TT - r.first + 1;
    return r;
}
template <int TT> __device__ __forceinline__ int pg_tile(const Range &r, int j)
{
    return (j < r.sink ? j : r.first + j - r.sink) * TT;
}
// The workgroups that share a tile's tokens: one for every `per` tiles of 32 tokens, S at most.
template <int TT> __device__ __forceinline__ int pg_parts(const AttnArgs &a, int total)
{
    const int per = a.per * 32 / TT;
    return max(1, min(a.S, (total + per - 1) / per));
}

// A token's elements in the cache, -1 without a page.  Loads of such a token go to the
// first page, and a key of it is made NaN, which its scores then are.
__device__ __forceinline__ long long pg_token(const PgBatch &b, const int *table, int t)
{
    const int g = pg_of(b, t), n = g < b.ldt ? table[g] : -1;
    return n >= 0 && n < b.n_pages ? n * b.page_ld + (t - g * b.page) * b.tok_ld : -1;
}

// What is not finite in a register of cache elements becomes 0; true if anything was.
template <int C> __device__ __forceinline__ bool pg_clean(unsigned &w)
{
    bool hit = false;
    if constexpr (C == TLG_F32) {
        hit = (w & 0x7f800000u) == 0x7f800000u;
        w = hit ? 0u : w;
    } else {
        constexpr unsigned X = C == TLG_F16 ? 0x7c00u : 0x7f80u;
        const bool l = (w & X) == X, h = (w & X << 16) == X << 16;
        w &= (l ? 0xffff0000u : ~0u) & (h ? 0x0000ffffu : ~0u);
        hit = l || h;
    }
    return hit;
}
// true if anything in these registers of 16-bit elements is not finite
template <int C, int N, int M> __device__ __forceinline__ bool pg_odd(const unsigned (&w)[N][M])
{
    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
    constexpr unsigned short X = C == TLG_F16 ? 0x7c00 : 0x7f80;
    u16x2 m = {0, 0};
#pragma unroll
    for (int i = 0; i < N; i++)
#pragma unroll
        for (int k = 0; k < M; k++) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, w[i][k] & 0x7fff7fffu));
    return m[0] >= X || m[1] >= X;
}
__device__ __forceinline__ bool pg_finite(float v) { return fabsf(v) < INFINITY; }

__device__ __forceinline__ bool pg_sees(const AttnArgs &a, int t, int p, int from)
{
    return (t <= p) & ((t >= from) | (t < a.sinks));
}
// Orders a wave's own reads and writes of LDS.
__device__ __forceinline__ void pg_wave_sync()
{
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// Values that are not finite would reach, through products with a weight of 0, columns
// that do not see their tokens.  In tiles that some column sees in part they are 0 in
// the products, and come here, from the cache, to the columns that do see them: one
// token at a time, for it is rare.  e: the weights of the 32 tokens from t0 on in the
// product's layout, w: 1 KB of LDS of the wave's own; off(i): token i's elements of V, the
// same in all lanes; at(b, m): the element that row m of block b stands for.
template <int C, int W, int NB, typename OFF, typename AT>
__device__ __forceinline__ void pg_special(const AttnArgs &a, typename AccT<W>::A (&o)[NB], const float *e, float *w,
                                           const char *V, int t0, int pmax, int p, int from, OFF off, AT at)
{
    typedef typename ElT<C>::E E;
    const int lane = threadIdx.x & 63, col = lane % W, g = lane / W;
#pragma unroll
    for (int i = 0; i < W / 2; i += 4) {
        const int tb = pg_at<W>(i, 0);                   // the 256 / W tokens of four registers
        pg_wave_sync();
#pragma unroll
        for (int j = 0; j < 4; j++) w[(4 * g + j) * W + col] = e[i + j];
        pg_wave_sync();
#pragma unroll 1
        for (int k = 0; k < 256 / W && t0 + tb + k <= pmax; k++) {
            const long long at0 = off(tb + k);
            if (at0 < 0) continue;
            const float f = w[k * W + col];
            const bool see = pg_sees(a, t0 + tb + k, p, from);
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int j = 0; j < W * W / 64; j++) {
                    const float v = (float)((const E *)V)[at0 + at(b, pg_at<W>(j, g))];
                    if (see && !pg_finite(v)) o[b][j] = fmaf(f, v, o[b][j]);
                }
        }
    }
    pg_wave_sync();
}

// The running maximum of a column and what it does to its sums: z the scores of N
// registers (hidden ones -inf), which become weights.
template <int T, int W, int N, int NB>
__device__ __forceinline__ void pg_weights(float (&z)[N], float c, float &R, float &l, typename AccT<W>::A (&o)[NB])
{
    float m[4] = {z[0], z[1], z[2], z[3]};
#pragma unroll
    for (int i = 4; i < N; i++) m[i & 3] = fmaxf(m[i & 3], z[i]);
    const float mx = pg_gmax<W>(fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]))) * c;
    if (__any(mx > R + (PG_LIFT<T> + PG_SLACK<T>))) {
        const float n = fmaxf(R, mx - PG_LIFT<T>), f = __builtin_amdgcn_exp2f(R - (n == -INFINITY ? 0.f : n));
        R = n;
        l *= f;
#pragma unroll
        for (int b = 0; b < NB; b++) o[b] *= f;
    }
    const float ref = R == -INFINITY ? 0.f : R;
    float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < N; i++) {
        z[i] = __builtin_amdgcn_exp2f(fmaf(z[i], c, -ref));
        s[i & 3] += z[i];
    }
    l += (s[0] + s[1]) + (s[2] + s[3]);
}

// K consecutive elements of a row of out, weighted by 1 / l.
__device__ __forceinline__ float pg_inverse(float l) { return l == 0.f ? 0.f : 1.f / l; }
template <int T, int K> __device__ __forceinline__ void pg_put(char *p, const float *x)
{
    typedef typename ElT<T>::E E;
    E v[K];
#pragma unroll
    for (int i = 0; i < K; i++) v[i] = (E)x[i];
    __builtin_memcpy(__builtin_assume_aligned(p, K * sizeof(E) % 16 == 0 ? 16 : K * sizeof(E) % 8 == 0 ? 8 : 4), v, sizeof v);
}
__device__ __forceinline__ float pg_lse(float R, float l)
{
    return l == 0.f ? -INFINITY : ((R == -INFINITY ? 0.f : R) + __builtin_amdgcn_logf(l)) * 0.69314718056f;
}
// (sums: where they go if they are not the row's only ones)
template <int T, int K>
__device__ __forceinline__ void pg_out(const AttnArgs &a, int hd, float *sums, int r, int head, int d, float l, float *x)
{
    if (sums) {
        pg_put<TLG_F32, K>((char *)(sums + d), x);
        return;
    }
    const float f = pg_inverse(l);
#pragma unroll
    for (int i = 0; i < K; i++) x[i] = l == 0.f ? 0.f : x[i] * f;
    pg_put<T, K>(a.out + ((long long)r * a.ldo + (long long)head * hd + d) * (T == TLG_F32 ? 4 : 2), x);
}
__device__ __forceinline__ void pg_out_sums(const AttnArgs &a, float *sums, int r, int head, float R, float l)
{
    if (sums) *(float2 *)sums = float2{R, l};
    else if (a.lse) a.lse[(long long)r * a.H + head] = pg_lse(R, l);
}
// the rows' kernels' sums of workgroup s of several
__device__ __forceinline__ float *pg_part(const AttnArgs &a, float *p, int w, int s, int parts, int r, int head)
{
    return parts > 1 ? p + (((long long)s * a.b.N + r) * a.H + head) * w : nullptr;
}

// What the launches of tlg_paged_tile.hip take (tlg_paged.hip decides).
#define PGT_ROWS 128                 /* columns (rows times heads) of a workgroup */
#define PGT_TOKENS(hd) ((hd) == 256 ? 32 : 64)
void pg_tile_launch(const AttnArgs &a, int type, int hd, unsigned grid, hipStream_t st);
