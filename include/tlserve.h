/* tlserve.h -- serving a batch of sequences over a paged KV cache, on device
 * pointers (libtlgemm.so, gfx950): the new rows' keys and values into the
 * cache's pages, the attention of ragged chunks over them (one token of each
 * sequence, drafted chunks, prompts), and the verification of drafted tokens by
 * sampling.  They are to a batch what tldecode.h's ring store, attention and
 * argmax are to one sequence; tinylm.c serves one sequence over a ring, so they
 * have no reference counterpart as calls.
 *
 * Conventions as tltrain.h's operators over rows of logits: asynchronous on
 * `stream`, TLG_OK or an error code with tlg_last_error() set; only the caller's
 * buffers are used, so calls may overlap on any streams as long as their outputs
 * and workspaces differ, and any call can be captured into a graph (after
 * tlg_init).  Equal calls give equal bits.  Element types are TLG_F32, TLG_F16
 * and TLG_BF16 (tltrain.h); sums are fp32 or wider.
 *
 * What lies in device memory (row0, len, table, tokens) is not looked at on the
 * host.  Values out of range never make a kernel read or write outside the
 * buffers described: rows are cut to [0, N), and what a page number outside
 * [0, n_pages) or a table too short for the sequence leads to is said at each
 * call. */
#ifndef TLSERVE_H
#define TLSERVE_H
#include <stddef.h>
#include "tltrain.h"
#ifdef __cplusplus
extern "C" {
#endif

#define TLG_PAGED_PAGE (1 << 16)    /* tokens of a page                       */
#define TLG_PAGED_LEN (1 << 30)     /* tokens of a sequence (ldt * page)       */
#define TLG_PAGED_ROWS (1 << 21)    /* rows of a call                          */
#define TLG_PAGED_SEQS (1 << 16)    /* sequences of a call                     */
#define TLG_PAGED_HEADS 1024        /* query heads; N * H of an attention is at
                                       most 2^29, B * KV at most 2^22          */

/* One layer's cache: n_pages pages of `page` tokens; the hd elements of page g,
 * token t and head h start at g * page_ld + t * tok_ld + h * head_ld elements of
 * K and of V (so [pages][page][KV][hd] and [pages][KV][page][hd] are both
 * described).  hd is 32, 64, 96, 128 or 256; K, V and the three distances are
 * multiples of 16 bytes, and distances reach from 0 to 2^40. */
typedef struct {
    void *K, *V;
    int type;                /* TLG_F32, TLG_F16, TLG_BF16 */
    int KV, hd;
    int page, n_pages;
    long long page_ld, tok_ld, head_ld;
} TlgPages;

/* A batch: sequence b has the rows row0[b] .. row0[b + 1] - 1 of the call's N
 * rows (its new tokens, in order; any number, none too) and len[b] tokens, the
 * new ones among them, so its row i of n is at position len[b] - n + i.  Token t
 * lies on page table[b * ldt + t / page].  row0 must not decrease; rows in no
 * sequence (before row0[0], from row0[B] on) are neither read nor written.
 * max_rows and max_len are what no sequence exceeds, as far as the host knows (0:
 * not known): they choose the launch, and results are right, only later, where
 * a sequence does exceed them. */
typedef struct {
    int B, N;
    const int *row0;         /* [B + 1] */
    const int *len;          /* [B]     */
    const int *table;        /* [B][ldt] */
    int ldt;
    int max_rows, max_len;
} TlgBatch;

/* The new rows into the cache: with the position p of every row,
 *   K[page of p][p % page] = rope(k), V[..] = v, q_out = rope(q)
 * rope as tlg_dev_rope (tinylm.c:630-651: the pairs (i, i + hd/2) of a head turned
 * by the angles of cos_t / sin_t [maxpos][hd/2], 16-byte aligned; a position outside
 * them gives NaN), computed in fp32 and rounded once.  cos_t and sin_t NULL:
 * no rotation.  q (rows of H heads; q_out its rows, which may be the same memory
 * with the same ldq, else the memory from its first to its last element must not overlap
 * q's) may be NULL, then H is ignored.  Rows are `type` elements, row
 * r of q at q + r * ldq and so on, 16-byte aligned with distances that are
 * multiples of 16 bytes (slices of one fused projection, for instance).  The cache is
 * of the rows' type, or of any type for fp32 rows.
 * A row with a negative position or no valid page is not stored (its q_out is
 * written); where tokens share a page and slot, either may win. */
int tlg_dev_paged_store(const TlgPages *c, const TlgBatch *b, const void *q, long long ldq, void *q_out,
                        long long ldqo, int H, const void *k, long long ldk, const void *v, long long ldv, int type,
                        const float *cos_t, const float *sin_t, int maxpos, void *stream);

/* Attention of the new rows over their sequences' pages (attn_body,
 * tinylm.c:3639-3715, for a batch): the row at position p sees the tokens t <= p
 * and, with win > 0, of those only t > p - win and t < sinks (a sliding window and
 * the first tokens, which stay visible; cfg_lwin, :64-68, has the window).  Head h
 * reads KV head h / (H / KV):
 *   out[r][h] = sum_t softmax_t(scale q . k_t) v_t,   lse[r][h] = log sum_t e^(scale q . k_t)
 * q and out have rows of H * hd elements of `type`, ldq and ldo apart (16-byte
 * aligned; the memory from out's first to its last element must not overlap q's, nor
 * the cache); lse [N][H] may be NULL.  The
 * cache is of that type, or of any type for fp32 rows.  scale lies in 1e-30 ..
 * 1e30.  Scores, softmax and sums are fp32.  For 16-bit rows the weights e^(s - max)
 * are rounded to twice that type's bits before they meet v (fp16: or by 2^-36 of the row's largest,
 * whichever is more); fp32 rows keep fp32 products.
 * Sums of weights of up to 2^8 (fp16: 2^15) times values are formed before they are divided, so that
 * values up to 1e27 cannot overflow.
 * A row that sees nothing (or only scores of -inf) is 0, its lse -inf.  A row
 * that sees a token without a valid page is NaN.  Tokens that a row does not see
 * cannot reach it, whatever their slots hold, NaN and infinities too.
 * A value that is not finite reaches its own element of the rows that see it: NaN, an infinity as
 * it is (NaN where its weight lies below fp32's range, or against one of the other sign).
 * ws: tlg_paged_attn_ws_bytes(c, b, type, H) bytes, 16-byte aligned, of any
 * content (NULL when that is 0; it depends on B, N, ldt, max_rows and max_len, on no
 * device memory). */
size_t tlg_paged_attn_ws_bytes(const TlgPages *c, const TlgBatch *b, int type, int H);
int tlg_dev_paged_attn(const TlgPages *c, const TlgBatch *b, const void *q, int type, long long ldq, int H, float scale,
                       int win, int sinks, void *out, long long ldo, float *lse, void *ws, size_t ws_bytes,
                       void *stream);

/* Verification of drafted tokens by sampling (of what tl_decode_generate_spec
 * does greedily, tinylm.c:3985-4001).  The rows of sequence b, row0[b] ..
 * row0[b + 1] - 1, are the target model's next-token logits after its last
 * token and after each drafted one: row i judges the token draft[i], drawn
 * from the draft model's logits of the same row of draft_logits, or chosen
 * without chance where draft_logits is NULL.  With p = softmax(scale x) and q =
 * softmax(dscale y), or q = 1 at draft[i]:
 *   row i keeps its draft  iff  u[i] q(draft) < p(draft)
 * up to the sequence's first row that does not, or has no draft (a negative
 * one; the last row's is not looked at).  That row gives one more token, by an
 * exponential race over the noise e of its sequence (noise[b * ldn + v], v < V):
 *   token = argmax_v w_v / e_v,  w_v = max(0, p_v - q_v) if a draft was refused
 *                                      (p_v if that is 0 everywhere), else p_v
 * the lowest v among equals.  With u uniform in [0, 1) and e independent
 * exponentials (-log of uniforms) the kept tokens and this one are distributed as
 * samples of p, whatever the drafts.  Tokens whose noise lies outside 1e-30 .. 1e30
 * are not chosen.
 *   tokens[r]   the kept drafts, then the chosen token; -1 in the rows after it
 *   logp[r]     their log p (0 in the rows after); may be NULL
 *   accepted[b] how many drafts were kept; may be NULL
 * A row without a distribution (all -inf, a NaN or +inf in it or in its draft
 * row where it has a draft) or without a token to choose ends its sequence with
 * token -1 and logp NaN.  A draft from V on has p = q = 0; a draft row of
 * nothing but -inf has q = 0 everywhere.  A sequence without rows has accepted 0;
 * rows in no sequence are left alone.
 * Logits as in tltrain.h's operators over rows of logits (both of `type`, rows ld and
 * ldd apart, V <= TLG_VOCAB_MAX, N <= TLG_VOCAB_ROWS); scale and dscale (1 /
 * temperature) lie in 1e-30 .. 1e30.  ws: tlg_spec_verify_ws_bytes(type, N, V, B,
 * draft_logits != NULL) bytes, 16-byte aligned, of any content. */
size_t tlg_spec_verify_ws_bytes(int type, int N, int V, int B, int drafted);
int tlg_dev_spec_verify(const void *logits, int type, long long ld, float scale, const void *draft_logits,
                        long long ldd, float dscale, int N, int V, const int *row0, int B, const int *draft,
                        const float *u, const float *noise, long long ldn, int *tokens, float *logp, int *accepted,
                        void *ws, size_t ws_bytes, void *stream);

#ifdef __cplusplus
}
#endif
#endif
