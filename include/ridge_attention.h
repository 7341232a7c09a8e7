/*
 * ridge_attention.h -- C ABI of the MI355X (gfx950) operators around a cache of keys and
 * values in 8 bits: the norm and rotation of query and key heads, rows written to and read
 * from the cache, and the attention of each sequence's newest token over it.
 *
 * The cache is paged. A page holds pageSize tokens (a multiple of 16) of every key head; a
 * token's row of a head is `dim` 8-bit values q with one f32 scale, which stand for q * scale
 * (ridge_int8.h has the rounding: the whole number next to 127 value / largest, halves to
 * even, the scale at least the smallest normal f32). A slot is a token's place in the cache:
 * page * pageSize + offset.
 *
 * Conventions, those of ridge_int8.h: the caller allocates everything on the device; a call
 * neither allocates nor synchronises and is asynchronous on `stream` (NULL: the default
 * stream); errors come back as hipError_t values, and a refused call
 * (hipErrorInvalidValue, 1) enqueues nothing. Types are RIDGE_F16, RIDGE_BF16 or RIDGE_F32,
 * and need the alignment of their type only. What a call writes shares no byte with anything
 * else of the call, heads that are rotated in place excepted; this is not checked here. No
 * tokens and no sequences are calls that do nothing.
 *
 * What device memory says is not known on the host, so it cannot be refused: a position
 * outside the table and a page or a length outside the cache make NaNs of the rows that ask
 * for them, and nothing is read or written outside the buffers.
 */
#ifndef RIDGE_ATTENTION_H
#define RIDGE_ATTENTION_H

#include <stddef.h>
#include <stdint.h>

#include "ridge_int8.h" /* the types */

#ifdef __cplusplus
extern "C" {
#endif

/* Most columns of a head, axes of a rotation, and tokens that a cache holds. */
enum { RIDGE_ATTENTION_MAX_DIM = 256, RIDGE_ATTENTION_MAX_AXES = 4, RIDGE_ATTENTION_MAX_SLOTS = 0x7fff0000 };

/* Heads of tokens: element (t, h, d) is at[t * token + h * head + d]. */
typedef struct {
    void* at;
    int64_t token, head;
    int32_t heads;
} ridge_attention_heads_t;

/* The cache: k's byte (page, h, t, d) is k[page * pageStride + h * headStride + t * tokenStride
 * + d], its scale kScale[page * scalePage + h * scaleHead + t], and v's likewise. Strides of
 * rows are in bytes and multiples of 16, tokenStride below 2^27, those of scales in elements and multiples of 4, and
 * all four pointers multiples of 16. A row's last 16 bytes are readable. */
typedef struct {
    int8_t* k;
    int8_t* v;
    float* kScale;
    float* vScale;
    int64_t pageStride, headStride, tokenStride, scalePage, scaleHead;
    int64_t pages;
    int32_t pageSize, heads, dim;
} ridge_attention_cache_t;

/* How heads are turned. Columns p and p + pairs of a head (interleaved: 2p and 2p + 1) turn by
 * the angle whose cosine and sine are table[row * stride + p] and [... + pairs + p], row being
 * the token's position on the axis that pair p belongs to: axis 0 turns the first sections[0]
 * pairs, axis 1 the next sections[1], and so on; the sections add up to pairs. Columns from
 * 2 pairs on keep their values. The table is less than 4 GiB. positions is [tokens, axes], its rows positionStride apart. */
typedef struct {
    const float* table;
    int64_t tableStride, tableRows;
    const int32_t* positions;
    int64_t positionStride;
    int32_t pairs, axes, interleaved;
    int32_t sections[RIDGE_ATTENTION_MAX_AXES];
} ridge_attention_rotation_t;

/* qOut, kOut <- the heads of q and of k, each normed (x / sqrt(mean(x^2) + eps) * weight, where
 * its weight is not null) and turned, in f32, rounded once to `type`. Weights are `dim`
 * contiguous values of `type` or RIDGE_F32. qOut and kOut have q's and k's heads; each may be
 * what it is made of, with the same strides. k->heads may be 0. */
int ridge_attention_norm_rope(const ridge_attention_heads_t* q, const ridge_attention_heads_t* k, int type,
                              const void* qWeight, const void* kWeight, int weightType, float eps,
                              const ridge_attention_rotation_t* rotation, const ridge_attention_heads_t* qOut,
                              const ridge_attention_heads_t* kOut, int64_t tokens, int32_t dim, void* stream);

/* cache <- the heads of k and of v (of `type`; as many as the cache has), token t at slots[t]. A
 * slot that is negative or behind the cache is not written. Slots of one call differ: a slot
 * that comes twice holds the bytes of one of the two and perhaps the scale of the other. */
int ridge_attention_write(const ridge_attention_cache_t* cache, const int32_t* slots, const ridge_attention_heads_t* k,
                          const ridge_attention_heads_t* v, int type, int64_t tokens, void* stream);

/* k, v <- the values at slots[t], in f32, rounded once to `type`. A negative slot reads as
 * zeros, one behind the cache as NaNs. */
int ridge_attention_read(const ridge_attention_cache_t* cache, const int32_t* slots, const ridge_attention_heads_t* k,
                         const ridge_attention_heads_t* v, int type, int64_t tokens, void* stream);

/* The bytes of workspace that an attend of these sizes takes; negative for sizes that it
 * refuses. No device is touched. */
int64_t ridge_attention_workspace(int64_t batch, int32_t heads, int32_t kvHeads, int32_t dim, int64_t pagesEach,
                                  int32_t pageSize);

/* out[b, h] <- the sum over t of p_t v_t, p the softmax over t of scale * (q[b, h] . k_t), where
 * t are the last `window` tokens (all of them for window 0) of the lengths[b] that sequence b
 * has in the cache, page i of them in pages[b * pagesStride + i]. Key head h / (heads /
 * cache->heads) serves query head h. lse (or null) [b * heads + h] <- log of the sum over t of
 * exp(scale * (q . k_t)). A sequence of no tokens gives zeros, and -inf in lse. A length that is
 * negative or past pagesEach pages, and a page that is none of the cache's where it is read,
 * give NaN. scale is FLT_MAX / 2 at the most, 2^118 for RIDGE_F16 (of which small columns lose
 * bits beside scales below 2^-135). q and out are of `type`; nothing but out is rounded to fewer
 * bits than f32's, whatever the sizes of queries and values (a p below 2^-126 of the largest may
 * count nothing, and below 2^-47 where values' scales up to 2^-40 and past 2^88 meet).
 *
 * All sequences' tokens are shared evenly by the workgroups that run at a time, so a result's
 * last bits go by the other sequences' lengths; where
 * pagesEach pages are 512 tokens or fewer, each sequence's key heads have a workgroup each, and its
 * result depends on nothing but its own operands. workspace is ridge_attention_workspace bytes, at
 * a multiple of 16, and needs no values; calls that may run at the same time take one each. */
int ridge_attention_attend(const ridge_attention_heads_t* q, const ridge_attention_cache_t* cache, const int32_t* pages,
                           int64_t pagesStride, int64_t pagesEach, const int32_t* lengths, float scale, int64_t window,
                           const ridge_attention_heads_t* out, float* lse, int type, int64_t batch, void* workspace,
                           int64_t workspaceBytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* RIDGE_ATTENTION_H */
