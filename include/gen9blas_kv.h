/* gen9blas_kv.h -- a key-value cache in pages and the operators that write, read, search and thin it, for serving
 * (an addition of the B200 build: the reference's lib/gen9blas_ml.h keeps one contiguous cache per stream). Conventions
 * (results, threads, streams, no-wait mode) as in gen9blas.h and gen9blas_ml.h; gen9blas_flush waits
 * for the stream of gen9blas_set_stream only.
 *
 * The cache: a pool of pages of `page` slots for each of HKV key-value heads, keys and values FP16, shared by ns streams
 * through a table of page numbers: slot k of stream s is slot k % page of page table[s·ts + k / page], for k below
 * mp·page. A page number outside [0, n_pages) (use -1) means "no page": its slots are never read or written, attention
 * does not see them. Streams may share pages they only read; a page that is written, counted or evicted from belongs to
 * one stream.
 *
 * Memory: every operand is device or managed memory of the current device (GEN9BLAS_ERR_INVALID_ARG otherwise); lengths,
 * counts and tables are read on the device, so that a captured call follows them at each replay. Calls are queued;
 * sync = 1 waits (not while the stream is being captured: GEN9BLAS_ERR_INVALID_ARG). Operands of one call that are
 * written overlap no other operand, unless said, nor themselves: the strides of K, V, acc and pos nest where a call writes
 * them, each at least what the dimensions with smaller ones span (GEN9BLAS_ERR_INVALID_ARG otherwise).
 *
 * Shapes: D a multiple of 8 up to 256, H a multiple of HKV (gen9blas_kv_supported; other shapes return
 * GEN9BLAS_DECLINED, nothing written); K, V and bounds 16-byte aligned, their strides multiples of 8 elements. kv_append and
 * attn_paged with acc take up to 65535 streams, and as many heads or (stream, head) rows (GEN9BLAS_ERR_INVALID_ARG past that). */
#pragma once
#include "gen9blas_ml.h"
#ifdef __cplusplus
extern "C" {
#endif

typedef struct gen9blas_kv_cache {
    int D, HKV;              /* head size, key-value heads */
    int page, n_pages;       /* slots per page, pages in the pool */
    uint16_t *K;             /* element d of (page p, slot i, head g) at K[p·kp + i·kk + g·kh + d], in k_bytes bytes */
    int64_t kp, kk, kh;
    size_t k_bytes;
    uint16_t *V;
    int64_t vp, vk, vh;
    size_t v_bytes;
    uint16_t *bounds;        /* NULL or [n_pages][HKV][2][D]: least and largest value of each key element in a page */
    const int *table;        /* page numbers, mp per stream, streams ts apart */
    int64_t ts;
    int mp, ns;
    void *stream;            /* cudaStream_t of the calls on this cache; NULL: as for every other call (gen9blas_set_stream) */
} gen9blas_kv_cache;

GEN9BLAS_API int gen9blas_kv_supported(int D, int H, int HKV);

/* Workspace of attn_paged, kv_select and kv_evict. NULL in a call means the library's own one of the device: calls that
 * share a workspace run one after the other (one on another stream than the last first waits for the device; that, and the
 * allocation when a workspace grows, would end a capture under way on some other stream: beside one, call with a workspace that
 * the call's stream has used before). A call
 * that is captured into a CUDA graph needs a workspace of its own here, large enough from an earlier call of the same
 * shape outside the capture (GEN9BLAS_ERR_INVALID_ARG otherwise); a replay must not run at the same time as another
 * replay or call that uses its workspace: the library does not see replays, so that order is the caller's.
 * kv_ws_free waits for the device; the graphs that use the workspace must not run after it. */
typedef struct gen9blas_kv_ws gen9blas_kv_ws;
GEN9BLAS_API gen9blas_kv_ws *gen9blas_kv_ws_create(void);
GEN9BLAS_API void gen9blas_kv_ws_free(gen9blas_kv_ws *ws);

/* Writes nt new tokens per stream: slots len[s] + t, t < min(cnt[s], nt) (cnt NULL: nt; a negative len or cnt counts as
 * 0). K and V: F32, element d of (token t, head g, stream s) at K[t·kt + g·kh + s·ks + d], rounded to FP16 (nearest
 * even). With bounds in the cache, the bounds of the pages written are set (slot 0 of the page among the new ones) or
 * widened, NaN elements left out (+inf and -inf if there is no other). acc and pos (each NULL or element k of (s, g) at
 * acc[s·ms + g·mh + k]): acc = 0, pos = pos0[s] + t (pos0 NULL: the slot's number) for the new slots. Tokens past mp·page
 * or without a page are dropped; with sync = 1, *bad (NULL allowed) = 1 if there were any, else 0. len is not changed. */
GEN9BLAS_API int gen9blas_kv_append(const gen9blas_kv_cache *c, int nt, const float *K, int64_t kt, int64_t kh, int64_t ks,
                                    const float *V, int64_t vt, int64_t vh, int64_t vs, const int *len, const int *cnt,
                                    float *acc, int *pos, int64_t ms, int64_t mh, const int *pos0, int sync, int *bad);

/* Attention of nq tokens per stream over the cache: O F32 [s][t][h][D] = softmax(scale·q·k) v over the slots that token t
 * of stream s sees: k < vt = min(vis[s] + dvis·t, mp·page), and k >= vt - window if window > 0. Q F32, element d of (t, h, s)
 * at Q[t·qt + h·qh + s·qs + d]; query head h reads key-value head h / (H / HKV). lse (NULL or [s][t][h]): log of the sum of
 * exp(score). A token that sees nothing gets O = 0, lse = -inf. dvis and window >= 0.
 * What lies in slots that a token does not see (NaN, infinities) does not enter its result; a seen key or value that is
 * not finite enters as the formula has it, for the heads that see it only: NaN, as a rule (where the formula gives an infinite
 * output, NaN may stand for it); a score of -inf has no weight.
 * sel (NULL or int [s][t][HKV][nsel]): only the slots of the listed pages, given by their place k / page in the stream,
 * ascending; an entry that is negative or not below mp is skipped, and so is one that is not above every earlier entry that
 * was not (a page counts once). Not with window > 0.
 * acc (NULL or as in kv_append): acc[k] += the softmax weights that slot k got from all tokens and query heads of the
 * key-value head (sums in a fixed order: the same bits each time). Meant for few tokens (decoding, drafts); any nq >= 1
 * works. */
GEN9BLAS_API int gen9blas_attn_paged(const gen9blas_kv_cache *c, int H, int nq, const float *Q, int64_t qt, int64_t qh,
                                     int64_t qs, const int *vis, int dvis, int window, const int *sel, int nsel, float scale,
                                     float *O, float *lse, float *acc, int64_t ms, int64_t mh, gen9blas_kv_ws *ws, int sync);

/* Pages for the attention above: for each (s, t, g), sel[s][t][g][0 .. nsel) = places of the pages that count among those
 * holding visible slots (vt as above): the first `first` and the last `last` of them, then those with the largest score
 * max over the head's queries of sum_d max(q_d·lo_d, q_d·hi_d) -- no key of the page has a larger q·k -- ties to the
 * lowest place; ascending, -1 behind if there are fewer than nsel. The sums are taken in 64 bits; lo <= hi in bounds that
 * are finite. A NaN score and a place
 * without a page rank last. first, last >= 0; if they are more than nsel, the lowest places among them. Needs bounds. */
GEN9BLAS_API int gen9blas_kv_select(const gen9blas_kv_cache *c, int H, int nq, const float *Q, int64_t qt, int64_t qh,
                                    int64_t qs, const int *vis, int dvis, int first, int last, int nsel, int *sel,
                                    gen9blas_kv_ws *ws, int sync);

/* Thins each stream with len[s] > keep slots down to `keep`, separately for each head: the slots with pos < first or pos
 * among the `recent` newest (pos > newest pos - recent) stay, then those with the largest acc (ties: the lowest slot; NaN
 * last). A staying slot at or above `keep` moves (K, V, acc, pos) into a slot below that was given up, the j-th such slot
 * into the j-th free one: the order of the cache changes, its positions are in pos. pos NULL: the slot's number is its
 * position. Bounds of the pages that changed are taken anew. len_out[s] (may be len itself) = min(len[s], keep). Slots at
 * and above `keep` and all else stay as they were. keep >= 1, first, recent >= 0, first + recent <= keep; acc is needed.
 * A slot without a page (see the table) is given up only by its rank, and its row moves nowhere. */
GEN9BLAS_API int gen9blas_kv_evict(const gen9blas_kv_cache *c, const int *len, int keep, int first, int recent, float *acc,
                                   int *pos, int64_t ms, int64_t mh, int *len_out, gen9blas_kv_ws *ws, int sync);

#ifdef __cplusplus
}
#endif
