/* femtochat_cache.h — C ABI of text generation in libfemtochat_attn.so (gfx950):
 * a cache of keys and values, attention of new tokens over it, and the
 * verification of drafted tokens.
 *
 * Conventions are those of femtochat_attn.h: every entry point returns an
 * fc_status (message in fc_last_error()), all pointers are device pointers,
 * launches are asynchronous on the caller's HIP stream, and the library
 * allocates nothing.  No reference counterpart.
 *
 * The cache holds tokens in pages (C row-major index expressions):
 *   k, v              : x[(((layer*pages + page)*Hkv + h)*page_size + place)*D + d]
 *   k_scale, v_scale  : s[((layer*pages + page)*Hkv + h)*page_size + place], float32 (8-bit types)
 *   table             : t[b*max_pages + i], the page of sequence b's tokens
 *                       i*page_size .. (i+1)*page_size - 1 (int32)
 * Without a table (max_pages 0) page b is sequence b's own.  A sequence's
 * capacity is max_pages*page_size tokens (page_size without a table).
 *
 * Types: bfloat16, or 8 bits with one scale per token and KV head: for the D
 * values x of a token's head and a = max |x|,
 *   int8   code = round(x * (127 / a)) (ties to even), scale a / 127;
 *   float8 code = x * (448 / a) rounded to e4m3 (ties to even), scale a / 448;
 * and a value reads back as code * scale, every operation in float32.  Heads
 * with a below 2^-100 are held as zeros; one with an infinity or a NaN reads
 * back as NaN.
 *
 * What the host cannot check, as it lies on the device, is safe: tokens
 * beyond the capacity or on a page that is not in the pool are not written, and
 * read as NaN.
 *
 * Tensors of tokens (K, V, Q, O) are those of femtochat_attn.h, B sequences of
 * T (N) tokens, and must be 16-byte aligned, as k, v and their scales.  lengths
 * (B int32): the tokens that each sequence's cache holds before the call (not
 * below 0); counts (B int32 or null): how many of the call's T (N) tokens each
 * sequence has, null for all of them. */
#ifndef FEMTOCHAT_CACHE_H
#define FEMTOCHAT_CACHE_H

#include <stddef.h>
#include <stdint.h>

#include "femtochat_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef enum { FC_CACHE_BF16 = 1, FC_CACHE_I8 = 2, FC_CACHE_F8 = 3 } fc_cache_type;

typedef struct {
  int32_t D, Hkv;     /* head_dim (a multiple of 16 up to 128), KV heads */
  int32_t B;          /* sequences */
  int32_t layers;     /* layers that k and v hold; fc_cached_attn takes one */
  int32_t pages;      /* pages of the pool (of each layer); B without a table */
  int32_t page_size;  /* tokens, a multiple of 16; a power of two with a table */
  int32_t max_pages;  /* entries of a sequence's row of the table, 0: no table */
  int32_t type;       /* fc_cache_type */
} fc_cache_desc;

typedef struct {
  void *k, *v;
  float *k_scale, *v_scale; /* null for bfloat16 */
  const int32_t* table;     /* null without a table */
} fc_cache;

/* Writes K and V (layers, B, T, Hkv, D; float32 or bfloat16) as tokens
   lengths[b] .. lengths[b] + counts[b] - 1 of each sequence. */
fc_status fc_cache_write(const fc_cache_desc* desc, const fc_cache* cache, const void* K, const void* V,
                         int32_t in_dtype, int32_t T, const int32_t* lengths, const int32_t* counts, void* stream);

/* Reads tokens starts[b] (null: 0) .. starts[b] + counts[b] - 1 into K and V
   (layers, B, T, Hkv, D; float32 or bfloat16), with zeros behind them. */
fc_status fc_cache_read(const fc_cache_desc* desc, const fc_cache* cache, void* K, void* V, int32_t out_dtype, int32_t T,
                        const int32_t* starts, const int32_t* counts, void* stream);

/* Moves the tokens lengths[b] + path[b*N + j] to lengths[b] + j, for j below
   counts[b], in every layer: a path of accepted nodes, in increasing order, to the
   end of the sequence.  What is in between the kept tokens is lost. */
fc_status fc_cache_keep(const fc_cache_desc* desc, const fc_cache* cache, int32_t N, const int32_t* lengths,
                        const int32_t* path, const int32_t* counts, void* stream);

typedef struct {
  int32_t H;        /* query heads, a multiple of Hkv */
  int32_t N;        /* new tokens per sequence, 1 to 64 */
  int32_t left;     /* a token sees the left tokens before it (and itself); -1: all */
  int32_t tree;     /* parents: 0 none, 1 one row for all sequences, 2 (B, N) */
  float softcap;    /* fc_attn_score */
  const float* slopes;
} fc_cached_attn_options;

/* Attention of the newest tokens, whose keys and values fc_cache_write has put at
   lengths[b] .. lengths[b] + counts[b] - 1, over the cache: Q and O (B, N, H, D)
   bfloat16.  Without parents node i follows node i - 1.  With them the nodes are a
   tree: parents[i] is a node before i, or -1 where i follows the sequence itself;
   a node sees the sequence, its ancestors and itself, and its position in the text
   (for the window and slopes) is lengths[b] plus the number of its ancestors.
   O is 0 for nodes from counts[b] on and NaN for a node whose parents are not so,
   or that lies beyond the capacity.  A value in the cache that is not finite (bf16,
   or a NaN among a caller's own float8 codes) is what O has in its column at the
   nodes that see it, and reaches no other.  Sums are float32 (of values beyond 2^120
   over the number of keys they may overflow).  workspace:
   fc_cached_attn_workspace_bytes (0 is possible), 256-byte aligned. */
fc_status fc_cached_attn_workspace_bytes(const fc_cache_desc* desc, const fc_cached_attn_options* options, size_t* bytes);
fc_status fc_cached_attn(const fc_cache_desc* desc, const fc_cache* cache, const fc_cached_attn_options* options,
                         const void* Q, void* O, const int32_t* lengths, const int32_t* counts,
                         const int32_t* parents, void* workspace, size_t workspace_bytes, void* stream);

/* Verification of drafted tokens against the target's logits.  Node 0 is the
   last token of the text, the nodes after it are drafted ones, as in
   fc_cached_attn; logits (B, N, V) holds at node i the model's logits behind it,
   p = softmax(logits / temperature).
   Draws (draft_logits, without parents): node i was drawn from q, the softmax of
     draft_logits (B, N - 1, V) at i - 1.  It is accepted if u[i] q(x) < p(x), p at
     its parent; the first that is not ends the run, and the next token is drawn
     from max(p - q, 0), or from p behind the last node and where less than 2^-40
     of that is left.
   Candidates (no draft_logits): a node's children are tried in order; x is accepted
     if u[i] (1 - what those before it have of p) < p(x), and a token tried before is
     not; the next token is drawn from p without the tried ones.
   A token outside the vocabulary is neither accepted nor refused: as if there were
     no node, the next token is drawn from p without the tried ones.
   A draw takes the first token whose cumulative weight is above u[0] of the whole.
   At temperature 0 a child that is the largest logit (the first of several) is
   accepted, and the next token is the largest; draft_logits and u are not read.
   Out: path (B, N) the accepted nodes from node 0 on, -1 behind them; kept (B)
   their number; next (B) the next token.  A row of logits with a NaN or +infinity,
   or without a finite value, accepts nothing and has the next token -1; so has a
   sequence with counts[b] = 0, which keeps nothing.  Weights and their sums are
   float64, but for the denominator of an acceptance's p(x) and q(x), which beyond 2048
   tokens is a sum of float32 exponentials (within 2^-17 of itself); a weight of less
   than 2^-1000 of the row's largest is none.  workspace: fc_verify_workspace_bytes
   (0 for a small vocabulary), 256-byte aligned. */
typedef struct {
  int32_t B, N, V;      /* sequences, nodes (1 to 64), vocabulary */
  int32_t dtype;        /* FC_F32 or FC_BF16: logits and draft_logits */
  int32_t index_type;   /* tokens: 0 int32, 1 int64 (fc_index_type) */
  int32_t tree;         /* parents: 0 none, 1 one row for all sequences, 2 (B, N) */
  int32_t has_draft;    /* draft_logits is given */
  double temperature;   /* 0, or from 2^-10 to 2^10 */
} fc_verify_desc;
fc_status fc_verify_workspace_bytes(const fc_verify_desc* desc, size_t* bytes);
fc_status fc_verify_drafts(const fc_verify_desc* desc, const void* logits, const void* draft_logits, const void* tokens,
                           const float* u, const int32_t* parents, const int32_t* counts, int32_t* path, int32_t* kept,
                           int32_t* next, void* workspace, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* FEMTOCHAT_CACHE_H */
