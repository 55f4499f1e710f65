// tlg_paged_tile.hip -- attention of many rows over a paged KV cache, 16-bit
// (include/tlserve.h): prompts and long chunks, bound by the matrix cores.
//
// A workgroup has 128 columns (rows times query heads of one KV head), 32 a wave, and
// walks over the tokens that any of them sees in tiles of 64, which its threads
// bring from the pages into LDS, rows as they lie in the cache, while the waves work on
// the tile before: two buffers, one barrier a tile.  The products are those of
// k_paged_direct (scores transposed, weights staying in their lanes).  Rows in LDS are
// apart by what makes the reads free of bank conflicts: keys are read 16 bytes a lane
// down 16 tokens (row lengths 4 modulo 64 banks), values four tokens by 32 elements
// (16 modulo 32 banks).
// Measured: 4096 rows over 16384 tokens, 32 query and 8 KV heads of 128 bf16 values, 1.45 to 1.5
// ms, 640 to 662 TFLOP/s of the operator's own products (a large library product: 1210); matrix cores 47 %
// busy, vector ALUs 42 %, which follow each other within a wave.  The weights are in two pieces as
// k_paged_direct's, half of the products again: rounded to bf16 once they took 1.16 to 1.18
// ms and left a norm error of 0.0023, where the output's own rounding is 0.0017.  Exponentials and splits
// dealt out between the products, by hand or by scheduling barriers, were no faster (1.47
// to 1.53 ms against 1.48).
#include "tlg_paged.h"
#include <type_traits>

// ALIKE: the 16 bytes that a wave brings in one go, up to 16 tokens' in a row, lie on one page (pages
// of a multiple of 16 tokens): their address is then one scalar and an offset that the
// lane keeps (with weights in one piece: 207 M vector instructions in place of 343 M, 1276 -> 1162 us).
template <int T, int HD, bool ALIKE> __global__ __launch_bounds__(256, HD == 256 ? 1 : 2) void k_paged_tile(AttnArgs a)
{
    typedef typename ElT<T>::E E;
    constexpr int TT = PGT_TOKENS(HD), NB = HD / 32, NT = TT / 32, CH = HD / 8, NL = TT * CH / 256;
    constexpr int KST = HD + 8, VST = (HD / 2) % 64 == 16 || (HD / 2) % 64 == 48 ? HD : HD + 32;
    __shared__ __align__(16) E ks[2][TT * KST], vs[2][TT * VST];
    __shared__ float scratch[4][256];

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 31, h = lane >> 5;
    const int kvh = blockIdx.x % a.KV, s = blockIdx.x / a.KV % a.S, y = blockIdx.x / a.KV / a.S;
    auto start = [&](int i) { return (long long)pg_row0(a.b, i) * a.G / PGT_ROWS + i; };
    const int b = pg_search(a.b.B, y, start), base = (int)(y - start(b)) * PGT_ROWS;
    const Seq q = pg_seq(a.b, b);
    const int cols = q.n * a.G;
    if (base < 0 || base >= cols || cols <= a.few) return;
    const Range rg = pg_range<TT>(a, q, base, min(base + PGT_ROWS, cols));
    const int parts = pg_parts<TT>(a, rg.total);
    if (s >= parts) return;
    const int j0 = (int)((long long)rg.total * s / parts), j1 = (int)((long long)rg.total * (s + 1) / parts);
    const int *table = a.b.table + (long long)b * a.b.ldt;
    const E *Kc = (const E *)a.K + kvh * a.b.head_ld, *Vc = (const E *)a.V + kvh * a.b.head_ld;

    // the wave's and the lane's columns
    const int rh0 = min(base + 32 * wave, cols - 1), rh = base + 32 * wave + col;
    const bool some = base + 32 * wave < cols, live = rh < cols;
    const Range rw = pg_range<TT>(a, q, rh0, min(rh0 + 32, cols));
    const int lomin = pg_from(a, rw.pmin);
    const int ci = min(rh, cols - 1) / a.G, g = min(rh, cols - 1) - ci * a.G;
    const int r = q.lo + ci, p = live ? pg_pos(a, q, ci) : -1, from = pg_from(a, p);
    u32x4 qf[HD / 16];
    {
        const E *qp = (const E *)a.q + (long long)r * a.ldq + (kvh * a.G + g) * HD + 8 * h;
#pragma unroll
        for (int i = 0; i < HD / 16; i++) {
            qf[i] = *(const u32x4 *)(qp + 16 * i);
            if (!live) qf[i] = u32x4{0, 0, 0, 0};
        }
    }
    // the thread's pieces of a tile: token (tid + 256 i) / CH, elements 8 ((tid + 256 i) % CH)
    int pg[NL], in[NL];                                  // its page, and its place there
    u32x4 kr[NL], vr[NL];
    bool lost[NL];
    const unsigned mine = ALIKE ? (unsigned)(lane / CH * (int)a.b.tok_ld + lane % CH * 8) * 2 : 0;
    auto page = [&](int j) {
#pragma unroll
        for (int i = 0; i < NL; i++) {
            const int t = pg_tile<TT>(rg, j) + ((ALIKE ? 64 * wave : tid) + 256 * i) / CH, n = pg_of(a.b, t);
            pg[i] = table[max(min(n, a.b.ldt - 1), 0)];
            in[i] = n < a.b.ldt ? t - n * a.b.page : -1;
        }
    };
    auto load = [&]() {
#pragma unroll
        for (int i = 0; i < NL; i++) {
            const int n = ALIKE ? __builtin_amdgcn_readfirstlane(pg[i]) : pg[i];
            lost[i] = n < 0 || n >= a.b.n_pages || in[i] < 0;
            const long long off = lost[i] ? 0ll : n * a.b.page_ld + in[i] * a.b.tok_ld;
            if constexpr (ALIKE) {
                kr[i] = *(const u32x4 *)((const char *)(Kc + off) + (lost[i] ? 0u : mine));
                vr[i] = *(const u32x4 *)((const char *)(Vc + off) + (lost[i] ? 0u : mine));
            } else {
                kr[i] = *(const u32x4 *)(Kc + off + (tid + 256 * i) % CH * 8);
                vr[i] = *(const u32x4 *)(Vc + off + (tid + 256 * i) % CH * 8);
            }
        }
    };
    auto whole = [&](const Range &x, int t0) { return t0 + TT - 1 <= x.pmin && (x.lomax <= t0 || t0 + TT - 1 < a.sinks); };
    // to LDS; true if values of a tile had to be cleaned: one that some column sees in part, or any
    auto put = [&](int j, int buf, auto every) {
        bool odd = false;
        const int t0 = pg_tile<TT>(rg, j);
        if (every || !whole(rg, t0)) {
#pragma unroll
            for (int i = 0; i < NL; i++) {
                bool hit = false;
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    unsigned w = vr[i][k];
                    hit |= pg_clean<T>(w);
                    vr[i][k] = w;
                }
                odd |= hit && t0 + (tid + 256 * i) / CH <= rg.pmax;
            }
        }
#pragma unroll
        for (int i = 0; i < NL; i++) {
            const int ch = tid + 256 * i, t = ch / CH, d = ch % CH * 8;
            if (lost[i]) kr[i][0] = ~0u;
            *(u32x4 *)(ks[buf] + t * KST + d) = kr[i];
            *(u32x4 *)(vs[buf] + t * VST + d) = vr[i];
        }
        return odd;
    };
    // An infinite value times a weight's second piece, which may be 0 or negative, is no infinity.  Sums
    // that are not finite are therefore formed once more, with every tile's values cleaned.
    f32x16 o[NB];
    float R, l;
    auto walk = [&](auto every) {
#pragma unroll
        for (int k = 0; k < NB; k++)
#pragma unroll
            for (int i = 0; i < 16; i++) o[k][i] = 0.f;
        R = -INFINITY;
        l = 0.f;
        bool odd = false;
        if (j0 < j1) {
            page(j0);
            load();
            page(j0 + 1);
            odd = __syncthreads_or(put(j0, 0, every));
        }
        for (int j = j0, buf = 0; j < j1; j++, buf ^= 1) {
            const bool more = j + 1 < j1;
            if (more) {
                load();
                page(j + 2);
            }
            const int t0 = pg_tile<TT>(rg, j);
            if (some && t0 <= rw.pmax && (t0 + TT > lomin || t0 < a.sinks)) {
                float e[16 * NT];
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    f32x16 z;
#pragma unroll
                    for (int i = 0; i < 16; i++) z[i] = 0.f;
#pragma unroll
                    for (int i = 0; i < HD / 16; i++)
                        z = pg_mfma<T, 32>(*(const u32x4 *)(ks[buf] + (32 * t + col) * KST + 16 * i + 8 * h), qf[i], z);
#pragma unroll
                    for (int i = 0; i < 16; i++) e[16 * t + i] = z[i];
                }
                const bool full = whole(rw, t0);
                if (!full) {
#pragma unroll
                    for (int t = 0; t < NT; t++)
#pragma unroll
                        for (int i = 0; i < 16; i++)
                            e[16 * t + i] = pg_sees(a, t0 + 32 * t + pg_at<32>(i, h), p, from) ? e[16 * t + i] : -INFINITY;
                }
                pg_weights<T, 32, 16 * NT, NB>(e, a.c, R, l, o);
                const E *vt = vs[buf] + (4 * h + (lane >> 2 & 3)) * VST + 16 * (lane >> 4 & 1) + 4 * (lane & 3);
#pragma unroll
                for (int i = 0; i < 2 * NT; i++) {
                    // weights in two pieces, as k_paged_direct's
                    u32x4 pf, pr;
#pragma unroll
                    for (int k = 0; k < 4; k++) pg_split<T>(e[8 * i + 2 * k], e[8 * i + 2 * k + 1], pf, pr, k);
#pragma unroll
                    for (int k = 0; k < NB; k++) {
                        const E *v = vt + 16 * i * VST + 32 * k;
                        const u32x2 v0 = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)v));
                        const u32x2 v1 = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(v + 8 * VST)));
                        const u32x4 vf = {v0[0], v0[1], v1[0], v1[1]};
                        o[k] = pg_mfma<T, 32>(vf, pf, o[k]);
                        o[k] = pg_mfma<T, 32>(vf, pr, o[k]);
                    }
                }
                if (odd) {                               // also where this wave's columns see all of the tile
#pragma unroll
                    for (int t = 0; t < NT; t++)
                        pg_special<T, 32, NB>(a, o, e + 16 * t, scratch[wave], (const char *)Vc, t0 + 32 * t, rg.pmax, p, from,
                                              [&](int k) { return pg_token(a.b, table, t0 + 32 * t + k); },
                                              [](int blk, int m) { return 32 * blk + m; });
                }
            }
            if (more) {
                const bool hit = put(j + 1, buf ^ 1, every);
                if (!every && whole(rg, pg_tile<TT>(rg, j + 1))) {
                    odd = false;
                    __syncthreads();
                } else odd = __syncthreads_or(hit);
            }
        }
        l = pg_gsum<32>(l);
    };
    walk(std::false_type());
    bool again = false;
#pragma unroll
    for (int k = 0; k < NB; k++)
#pragma unroll
        for (int i = 0; i < 16; i++) again |= !pg_finite(o[k][i]);
    if (__syncthreads_or(again && live && pg_finite(l))) walk(std::true_type());
    if (!live) return;
    const int head = kvh * a.G + g;
    float *sums = pg_part(a, a.po, HD, s, parts, r, head);
#pragma unroll
    for (int k = 0; k < NB; k++)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            float x[4] = {o[k][i], o[k][i + 1], o[k][i + 2], o[k][i + 3]};
            pg_out<T, 4>(a, HD, sums, r, head, 32 * k + pg_at<32>(i, h), l, x);
        }
    if (h == 0) pg_out_sums(a, pg_part(a, a.pm, 2, s, parts, r, head), r, head, R, l);
}

template <int T, bool ALIKE> static void launch(const AttnArgs &a, int hd, unsigned grid, hipStream_t st)
{
    if (hd == 32) hipLaunchKernelGGL((k_paged_tile<T, 32, ALIKE>), dim3(grid), dim3(256), 0, st, a);
    else if (hd == 64) hipLaunchKernelGGL((k_paged_tile<T, 64, ALIKE>), dim3(grid), dim3(256), 0, st, a);
    else if (hd == 96) hipLaunchKernelGGL((k_paged_tile<T, 96, false>), dim3(grid), dim3(256), 0, st, a);
    else if (hd == 128) hipLaunchKernelGGL((k_paged_tile<T, 128, ALIKE>), dim3(grid), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((k_paged_tile<T, 256, ALIKE>), dim3(grid), dim3(256), 0, st, a);
}
void pg_tile_launch(const AttnArgs &a, int type, int hd, unsigned grid, hipStream_t st)
{
    // 16 tokens' offsets in 32 bits
    const bool alike = a.b.page % 16 == 0 && a.b.tok_ld < 1 << 24;
    if (type == TLG_F16 && alike) launch<TLG_F16, true>(a, hd, grid, st);
    else if (type == TLG_F16) launch<TLG_F16, false>(a, hd, grid, st);
    else if (alike) launch<TLG_BF16, true>(a, hd, grid, st);
    else launch<TLG_BF16, false>(a, hd, grid, st);
}
