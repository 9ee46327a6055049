/* gsk.h: C ABI of libgse.so's operators over a paged cache of keys and values, and of beam search over it (gfx950).
 *
 * A step's new keys and values written to their cache slots (as they are or in 8 bits), cached tokens read back as contiguous
 * rows, attention of a step's new tokens over the cache, the best continuations over a request's beams and the vocabulary, and
 * the beams' cached tokens moved to the beams that continue them. They follow gse.h and gsp.h: the handle is a gse_handle,
 * structs are size-first, errors are negative GSE_E_* codes with the text in gse_last_error(h), every data pointer is a device
 * pointer, every call is asynchronous on the caller's stream and allocates nothing, so a graph can capture it. Slots, tables and
 * lengths are those of gsp_pages_step. Part of the library since ABI 1.7.
 *
 * gsk_attend and gsk_beam use the handle's tickets (calls of one handle must not overlap on the device) and scratch memory that
 * the caller passes; gsk_write, gsk_read and gsk_reorder use none.
 */
#ifndef GSK_H
#define GSK_H

#include "gse.h"

#ifdef __cplusplus
extern "C" {
#endif

enum { GSK_BF16 = 0, GSK_F16 = 1, GSK_F32 = 2, GSK_E4M3 = 3, GSK_I8 = 4 };

/* One layer's cache: keys and values of one type and layout, dim elements of a token's head lying together; strides in
 * elements. In 8 bits (GSK_E4M3: 8-bit floats of 4 exponent and 3 mantissa bits, largest 448, no infinities; GSK_I8: whole
 * numbers, -127 .. 127) a token's head has a scale, finite or NaN, and stands for its elements times that. dim is a multiple of 8, at
 * most GSK_MAX_DIM; the arrays' addresses are multiples of 8 elements, as are the strides. */
#define GSK_MAX_DIM 256
typedef struct gsk_cache {
  uint32_t size;
  uint32_t type;            /* GSK_BF16, GSK_F16, GSK_E4M3, GSK_I8 */
  uint32_t pages;
  uint32_t page;            /* tokens per page; pages * page < 2^32 */
  uint32_t heads;           /* at most 2^12 */
  uint32_t dim;
  void *keys;
  void *values;
  int64_t page_stride;
  int64_t token_stride;
  int64_t head_stride;
  float *key_scales;        /* 8 bits: the scales, by their own strides (in elements); else NULL */
  float *value_scales;
  int64_t scale_page_stride;
  int64_t scale_token_stride;
  int64_t scale_head_stride;
} gsk_cache;

/* The new tokens' rows [tokens][heads][dim], GSK_BF16, GSK_F16 or GSK_F32; addresses and strides (in elements) multiples of 8.
 * Token i goes to slot[i] (page * tokens per page + offset); a negative slot, or one past the cache, is skipped. A slot belongs
 * to one token of the call. */
typedef struct gsk_rows {
  uint32_t size;
  uint32_t tokens;
  uint32_t type;
  uint32_t reserved;
  const void *k;
  const void *v;
  int64_t k_token_stride;
  int64_t k_head_stride;
  int64_t v_token_stride;
  int64_t v_head_stride;
  const int64_t *slot;      /* [tokens] */
  void *stream;
} gsk_rows;

/* Cached tokens as rows: row begin[r] + i (begin[r] <= row < begin[r + 1]) is request r's token first[r] + i. Rows from
 * begin[requests] on are left as they were; a row whose token or page is out of range is zero. */
typedef struct gsk_read_rows {
  uint32_t size;
  uint32_t requests;
  uint32_t rows;            /* of k and v */
  uint32_t type;            /* GSK_BF16, GSK_F16, GSK_F32 */
  void *k;                  /* [rows][heads][dim], addresses multiples of 16 */
  void *v;
  const int32_t *table;     /* [requests][table_ld]: gsp_pages' */
  int64_t table_ld;
  uint32_t max_pages;       /* entries of a table row */
  uint32_t reserved;
  const int32_t *begin;     /* [requests + 1] */
  const int32_t *first;     /* [requests], or NULL: 0 */
  void *stream;
} gsk_read_rows;

/* Attention of a step's new tokens. Request r's new tokens are rows begin[r] .. begin[r + 1] - 1 of q and out, the last ones of
 * its seq_len[r] cached tokens (they are in the cache already). A new token sees the tokens before its request's new ones, and
 * of those itself and the earlier ones; with parent: itself, parent[row], that one's parent and so on (entries that are no
 * earlier row of the request end the path). Query head h reads head h / (heads / cache heads). Where nothing is seen, or every
 * score is -inf, the result is 0, as it is for a request with status[r] != 0 or with numbers out of range; cached tokens
 * whose page is out of range are not seen. A NaN or an infinity reaches the rows that see its token, whatever the token's weight (a
 * value's may stay out where its score is -inf), and no other. Rows from begin[requests] on are left as they were. */
typedef struct gsk_attention {
  uint32_t size;
  uint32_t requests;
  uint32_t tokens;          /* rows of q and out */
  uint32_t heads;           /* of q: a multiple of the cache's */
  uint32_t type;            /* of q and out: GSK_BF16, GSK_F16; the cache's own where that is not in 8 bits */
  uint32_t max_new;         /* >= every request's new tokens (later ones are left out); with parent: at most GSK_MAX_TREE */
  const void *q;            /* [tokens][heads][dim]; address and strides multiples of 8 elements */
  int64_t q_token_stride;
  int64_t q_head_stride;
  void *out;                /* [tokens][heads][dim], without gaps; address a multiple of 16 */
  const int32_t *table;
  int64_t table_ld;
  uint32_t max_pages;       /* entries of a table row; max_pages * page < 2^31 */
  float scale;              /* of the scores; at most 2^127 in size */
  const int32_t *begin;     /* [requests + 1], or NULL: one new token a request, row r */
  const int32_t *seq_len;   /* [requests] */
  const uint32_t *status;   /* [requests] gsp_step's, or NULL: every request is served */
  const int32_t *parent;    /* [tokens] a draft tree's (gse_tree.parent, its rows being these), or NULL: chains */
  void *work;               /* gsk_attention_work() bytes, a multiple of 16; not read before the call writes it */
  int64_t work_bytes;
  void *stream;
} gsk_attention;
#define GSK_MAX_TREE 64

/* One step of beam search over [requests * beams][ld] logits: for each request the n largest of
 *   scores[b] + x[b][t] - log(sum over u of exp(x[b][u]))
 * over its beams b and tokens t, in descending order; ties go to the lower beam, then to the lower token. A NaN logit counts as
 * -inf, as tokens of -inf are never taken; a beam whose score is not finite, whose logits hold +inf or nothing above -inf, gives
 * no continuation. Places without one hold -1, -1 and -inf. */
typedef struct gsk_beams {
  uint32_t size;
  uint32_t requests;
  uint32_t beams;           /* at most GSK_MAX_BEAMS */
  uint32_t n;               /* at most GSK_MAX_KEEP */
  uint32_t vocab;
  uint32_t type;            /* GSK_BF16, GSK_F16, GSK_F32 */
  const void *logits;
  int64_t ld;
  const float *scores;      /* [requests][beams] */
  int32_t *tokens;          /* [requests][n] */
  int32_t *parents;         /* [requests][n] the beam continued, 0 .. beams - 1 */
  float *out_scores;        /* [requests][n] */
  void *work;               /* gsk_beams_work() bytes */
  int64_t work_bytes;
  void *stream;
} gsk_beams;
#define GSK_MAX_BEAMS 32
#define GSK_MAX_KEEP 64

/* The cached tokens first[g] <= t < seq_len of each beam's row replaced by those of the beam that it continues, for every beam
 * of a group at once (as they were before the call): beam b of group g is table row g * beams + b, its source parent[g * beams +
 * b] in 0 .. beams - 1 (another value: left as it is). A token past either beam's length stays, as does a group whose first is
 * negative. Caches, strides and chunks as in gsp_path; pages belong to one row. */
typedef struct gsk_reorder_beams {
  uint32_t size;
  uint32_t groups;
  uint32_t beams;           /* at most GSK_MAX_BEAMS */
  uint32_t caches;
  const int32_t *table;     /* [groups * beams][table_ld] */
  int64_t table_ld;
  uint32_t max_pages;
  uint32_t page;
  const int32_t *seq_len;   /* [groups * beams] */
  const int32_t *parent;    /* [groups * beams] */
  const int32_t *first;     /* [groups], or NULL: 0 */
  void *cache;
  int64_t cache_stride;     /* bytes */
  void *const *cache_ptrs;
  uint32_t align;
  uint32_t pages;
  uint32_t chunks;
  uint32_t chunk_bytes;
  int64_t page_stride;      /* bytes */
  int64_t token_stride;
  int64_t chunk_stride;
  void *stream;
} gsk_reorder_beams;

/* Writes the rows to the cache. In 8 bits, with M = 448 (GSK_E4M3) or 127 (GSK_I8) and every operation rounded to fp32: scale =
 * max(max |x| * (1 / M), 2^-126), the element x * (1 / scale) rounded to nearest, ties to even. A row with a NaN or an infinity
 * gets the scale NaN and zeros: it reads as NaN. (The reference keeps its cache inside its packs, behind abi/gc.h: these calls
 * have no counterpart there.) */
GSE_API int gsk_write(gse_handle *h, const gsk_cache *cache, const gsk_rows *in);

/* Reads cached tokens back as rows, rounded to the rows' type. */
GSE_API int gsk_read(gse_handle *h, const gsk_cache *cache, const gsk_read_rows *in);

/* Attention of new tokens, in one launch. gsk_attention_work: the scratch bytes that it needs for these sizes on this device
 * (0: none; negative: an error); of the structs no pointer is read, and neither q's strides nor the scales'. Up to 2^37 tokens in all:
 * requests * (16 + max_pages * page / 32) < 2^32, and so much times the tiles of min(max_new, tokens) * heads / cache heads rows (of
 * 48; 32 where there are no more or dim > 128; 16), and fewer than 2^32 - 48 such rows a request: longer prompts go in parts. */
GSE_API int64_t gsk_attention_work(gse_handle *h, const gsk_cache *cache, const gsk_attention *in);
GSE_API int gsk_attend(gse_handle *h, const gsk_cache *cache, const gsk_attention *in);

/* One step of beam search, in one launch for up to 65535 rows and as many requests as the handle has tickets (its rows, 4096 at
 * least), in as many as that takes otherwise; its scratch bytes likewise. */
GSE_API int64_t gsk_beams_work(gse_handle *h, const gsk_beams *in);
GSE_API int gsk_beam(gse_handle *h, const gsk_beams *in);

/* Moves the beams' cached tokens, in one launch for up to 65535 groups. */
GSE_API int gsk_reorder(gse_handle *h, const gsk_reorder_beams *in);

#ifdef __cplusplus
}
#endif

#endif /* GSK_H */
