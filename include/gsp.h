/* gsp.h: C ABI of libgse.so's operators around a verify round whose numbers stay on the device (gfx950).
 *
 * Drafted chains verified against the target's probability rows, the paged cache's block tables and slot maps made from
 * the lengths that a round leaves on the device, and the accepted path of a draft tree moved to the cache slots that the
 * next step reads. They follow gse.h: the handle is a gse_handle, structs are size-first, errors are negative GSE_E_*
 * codes with the text in gse_last_error(h), every data pointer is a device pointer, every call is asynchronous on the
 * caller's stream and allocates nothing, so a graph can capture it. Part of the library since ABI 1.5.
 *
 * gsp_verify_chains uses the handle's workspace, like the calls of gse.h (calls of one handle must not overlap on the
 * device); gsp_pages_step and gsp_keep_path use none.
 */
#ifndef GSP_H
#define GSP_H

#include "gse.h"

#ifdef __cplusplus
extern "C" {
#endif

enum { GSP_F64 = 0, GSP_F32 = 1, GSP_BF16 = 2, GSP_F16 = 3 }; /* types of probability rows */

/* Chains of drafted tokens, one per request (speculative sampling with one draft per position). Request r's drafts are
 * token[begin[r], begin[r + 1]); a draft outside [0, vocab) ends its chain there (a padded batch pads with -1). The chain
 * of n drafts has n + 1 target rows, row begin[r] + r + i the distribution after its first i drafts, and n draft rows,
 * row begin[r] + i the distribution that draft i was drawn from. */
typedef struct gsp_chains {
  uint32_t size;
  uint32_t requests;
  uint32_t vocab;
  uint32_t max_drafts;      /* >= every chain's drafts; emit rows hold max_drafts + 1 tokens */
  uint32_t drafts;          /* entries of token and coin, rows of draft; target has drafts + requests rows */
  uint32_t target_type;     /* GSP_* */
  uint32_t draft_type;
  uint32_t u_rows;          /* 0: u has one draw per request; 1: one per target row, and the row drawn from says which */
  const void *target;       /* [drafts + requests][target_ld]: weights, each row of any positive sum */
  int64_t target_ld;
  const void *draft;        /* [drafts][draft_ld], or NULL: every draft one-hot (a deterministic drafter) */
  int64_t draft_ld;
  const int32_t *begin;     /* [requests + 1] */
  const int32_t *token;     /* [drafts] */
  const double *coin;       /* [drafts] in [0, 1): draft i is accepted iff q_i(x_i) > 0 and coin q_i(x_i) < p_i(x_i) */
  const double *u;          /* [requests], or [drafts + requests], in [0, 1): the draw of the token after the accepted drafts */
  int32_t *emit_len;        /* [requests] accepted drafts + 1 (GSE_WALK_ERROR: without the token that could not be drawn) */
  int32_t *emit_tokens;     /* [requests][emit_ld]: columns [0, max_drafts] written, -1 past the emitted tokens */
  float *emit_probs;        /* [requests][emit_ld] the target's weight of each emitted token; 0 past them; or NULL */
  int64_t emit_ld;          /* >= max_drafts + 1 */
  uint32_t *status;         /* [requests] GSE_WALK_OK, or GSE_WALK_ERROR: the weights to draw from hold a NaN or an
                             * infinity or none above zero (or sum to an infinity), or begin is not in order (nothing
                             * emitted). A rejected one-hot draft's own entry is a weight only where no other is above zero */
  void *stream;
} gsp_chains;

/* A paged cache's bookkeeping, in the caller's device arrays: which pages each request holds (a page belongs to one), and the
 * free pages as a ring (a queue: steps take from its head and give back at its tail, so that neither writes what the other
 * reads). Steps over the same arrays must follow one another on the device. */
typedef struct gsp_pages {
  uint32_t size;
  uint32_t requests;
  uint32_t page;            /* tokens per page, >= 1 */
  uint32_t pool;            /* pages of the cache: entries of ring */
  uint32_t max_pages;       /* pages a request can hold; max_pages * page < 2^31 */
  uint32_t reserved;
  int32_t *table;           /* [requests][table_ld]: request r's pages, in order; entries past held[r] are not read */
  int64_t table_ld;         /* >= max_pages */
  int32_t *ring;            /* [pool] free pages: entries head .. head + free - 1 (mod pool) */
  const int32_t *counters;  /* [2 + 2 requests]: head, free, then length[requests], held[requests] */
  int32_t *counters_out;    /* the same after the step; may be counters itself */
} gsp_pages;

enum {
  GSP_STEP_OK = 0,
  GSP_STEP_FULL = 1, /* not enough free pages for this request (in request order), more than max_pages, or more
                      * tokens than max_tokens: its kept tokens count, nothing is added, its slots are -1; it gives no
                      * page back unless it ends (keep < 0), and then every one */
  GSP_STEP_BAD = 2   /* keep, add, length or held (for every request: head or free) out of range: the request is left as it
                      * was, its slots are -1 */
};

typedef struct gsp_step {
  uint32_t size;
  uint32_t max_tokens;      /* entries of slot, pos, req */
  const int32_t *keep;      /* [requests] tokens of the pages held that the step before filled and that stay (an accepted
                             * path), < 0: the request ends and gives back every page, whether or not add fits (not when
                             * it is GSP_STEP_BAD); NULL: none */
  const int32_t *add;       /* [requests] new tokens >= 0 */
  const int32_t *depth;     /* [max_tokens] a new token's distance from its request's first (a tree node's depth), or
                             * NULL: its index among the request's new tokens */
  int32_t *begin;           /* [requests + 1] offsets of the requests' new tokens */
  int64_t *slot;            /* [max_tokens] cache slot of each new token (page * tokens per page + offset), -1 past them */
  int32_t *pos;             /* [max_tokens] its position (length + depth), 0 past them; or NULL */
  int32_t *req;             /* [max_tokens] its request, -1 past them; or NULL */
  int32_t *seq_len;         /* [requests] tokens of the request with the new ones */
  uint32_t *status;         /* [requests] GSP_STEP_* */
  void *stream;
  const uint32_t *laid;     /* [requests] the status of the step that added the tokens which keep counts (not this step's status
                             * array): a request that it did not serve had no slots, so a keep > 0 counts as 0 there; or
                             * NULL: it served every request. Since ABI 1.6 */
} gsp_step;

/* The accepted paths of draft trees whose nodes were written to the cache in node order: entry i of request r's path,
 * i = 1 .. emit_len[r] - 1, moves from slot[emit_nodes[r][i]] to slot[anchor[r] + i], in every cache. Nodes ascend along a
 * path (a parent comes before its children), and requests share no slots. Entries whose node, place or slot is out of range
 * are not moved, nor is any entry of a request whose anchor is negative (a padded one). */
typedef struct gsp_path {
  uint32_t size;
  uint32_t requests;
  uint32_t tokens;          /* entries of slot */
  uint32_t caches;          /* arrays of the same shape (keys and values of every layer) */
  const int64_t *slot;      /* [tokens] gsp_step.slot of the round; a negative slot is not moved */
  const int32_t *anchor;    /* [requests] gse_tree.anchor */
  const int32_t *emit_len;  /* [requests] gse_tree_out's */
  const int32_t *emit_nodes; /* [requests][emit_ld] */
  int64_t emit_ld;
  void *cache;              /* the first cache; cache k starts cache_stride * k bytes after it ... */
  int64_t cache_stride;
  void *const *cache_ptrs;  /* ... or [caches] their addresses (a device array; then cache is not read) */
  uint32_t align;           /* a power of two that every address of cache_ptrs is a multiple of */
  uint32_t page;            /* tokens per page */
  uint32_t pages;           /* pages of a cache: a slot past them is not moved */
  uint32_t chunks;          /* a token's data: chunks of chunk_bytes, chunk_stride bytes apart */
  uint32_t chunk_bytes;
  uint32_t reserved;
  int64_t page_stride;      /* bytes */
  int64_t token_stride;     /* bytes between tokens of a page */
  int64_t chunk_stride;
  void *stream;
} gsp_path;

/* Verifies every chain, in one launch where the handle's workspace holds the call: up to 4096 requests (or the handle's
 * rows, if more) whose rows' segment sums fit it (fp64 rows of 128256 tokens through a handle of 64 such rows: 1040
 * requests); in as many as that takes otherwise. With a the first draft that is not accepted (its distributions p, q): the
 * token is drawn from max(p - q, 0), one-hot: p without the draft; where that leaves nothing, from p. After n accepted drafts
 * it is drawn from the last row. The draw takes the first token with a positive weight whose inclusive sum in vocabulary order
 * reaches u times the row's sum (negative weights count as 0). One chain of one draft is gse_mss with a single kid.
 * Replaces: dist + mss per node of a chain, goethe_engine/engine.py:278-283, spec.py:88-103, on rows already computed. */
GSE_API int gsp_verify_chains(gse_handle *h, const gsp_chains *in);

/* One step of the bookkeeping: length' = length + keep (0 when keep < 0), pages for length' + add tokens taken from the
 * ring or given back to it, in request order; the pages given back are free from the next step on. One launch, two when
 * counters_out is counters. Replaces: goethe_engine/kv.py:287-303's commit on the host, for lengths on the device. */
GSE_API int gsp_pages_step(gse_handle *h, const gsp_pages *pages, const gsp_step *step);

/* Moves the accepted paths, in one launch for up to 65535 requests. Replaces: goethe_engine/engine.py:299-305's commit of
 * each path one request at a time (gc_c.py:302-303, gc_commit of abi/gc.h:212), for a cache whose arrays are the caller's. */
GSE_API int gsp_keep_path(gse_handle *h, const gsp_path *in);

#ifdef __cplusplus
}
#endif

#endif /* GSP_H */
