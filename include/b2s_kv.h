/* b2s_kv.h -- the key/value cache of a served decoder on B200 (C ABI of libb2s.so).
 *
 * The decoder layers of the reference attend over the tokens of one call only (src/models/pi0/vlm.cpp:217-240);
 * these entry points keep keys and values between calls, in 8 bits:
 *   1. b2s_rope_axes      rotates the new tokens' query and key heads (positions with one to four axes);
 *   2. b2s_kv_write       quantises the new tokens' keys and values into the cache's pages;
 *   3. b2s_attention_kv   attention of the new tokens of a batch of sequences over their cached tokens,
 *      b2s_attention_kv_prefix   the same for sequences that share a prefix, which is read once for all of them;
 *   4. b2s_kv_read        reads cached tokens back.
 * The conventions are those of b2s.h: device pointers of the current device, a cudaStream_t, b2s_status codes,
 * b2s_last_error(). Arguments are checked before the device is, and everything that the host can see is refused
 * before anything is launched. Indices that live in device memory are checked by the kernels: one that is out of
 * range is never followed, sets bit 2 of b2s_device_error()'s word, and what it stands for is left out.
 *
 * Activations are f32 or bf16 (B2S_TYPE_F32, B2S_TYPE_BF16), rows of heads side by side, 16-byte aligned with a row
 * stride that is a multiple of 16 bytes.
 */
#ifndef B2S_KV_H
#define B2S_KV_H

#include "b2s.h"

#ifdef __cplusplus
extern "C" {
#endif

/* A paged cache. Slot s is token s % page_size of page s / page_size. One code row of head_dim bytes and one fp32
 * scale for each token and head, for keys and for values:
 *   codes [n_pages][n_kv_heads][page_size][head_dim], scales [n_pages][n_kv_heads][page_size]
 * type: B2S_TYPE_I8 (codes -127..127) or B2S_TYPE_F8_E4M3 (finite codes); the value is code * scale. head_dim is a
 * multiple of 16 up to 128, page_size a power of two from 16 to 1024, codes are 16-byte aligned. The caller owns the
 * four buffers. */
typedef struct b2s_kv_cache {
    int32_t type;
    int32_t n_kv_heads, head_dim, page_size;
    int64_t n_pages;
    void *k, *v;
    float *k_scale, *v_scale;
} b2s_kv_cache;

/* The sequences of one attention call. Sequence b has query rows q_start[b] .. q_start[b + 1] - 1 (none is allowed)
 * and kv_len[b] cached tokens (zero is allowed); its token j is in page pages[b * ld_pages + j / page_size] at
 * j % page_size. Its n query rows stand for its last n tokens. All three arrays are device memory, read when the
 * kernels run, so a captured call can be replayed with other contents. max_q bounds the query rows of a sequence and
 * max_pages * page_size its tokens. batch <= 16384. */
typedef struct b2s_kv_batch {
    int32_t batch;
    int32_t max_q;
    const int32_t *q_start; /* [batch + 1] */
    const int32_t *kv_len;  /* [batch] */
    const int32_t *pages;   /* [batch][max_pages], row stride ld_pages */
    int64_t max_pages, ld_pages;
} b2s_kv_batch;

/* Rotary embedding, NEOX pairs, with several position axes (time, height and width of an image patch, say):
 *   (y[i], y[i + hd/2]) = (x[i] cos t - x[i + hd/2] sin t, x[i] sin t + x[i + hd/2] cos t),
 *   t = pos[m][axis(i)] * theta_base^(-2 i / hd)
 * for each of M rows of n_heads heads of head_dim = hd values. pos [M][n_axes] int32 (device, row stride ldpos).
 * sections (host, n_axes counts that add up to hd / 2) says how many pairs each axis turns: in blocks, axis 0's pairs
 * first, or, with interleaved != 0, dealt to the axes in turn, passing over those that have their share. The angle is
 * formed and reduced in double precision, its cosine and sine are fp32 (within 1.5 * 2^-24), and the result is rounded
 * once to `type`. One axis is b2s_rope_neox to those roundings. y may be x (other overlaps are not allowed); M = 0 is
 * allowed; head_dim is even and at most 256, a row has fewer than 2^32 - 512 values; any row alignment that the type allows. */
int b2s_rope_axes(int32_t type, const void *x, int64_t ldx, int64_t M, int n_heads, int head_dim, const int32_t *pos,
                  int64_t ldpos, int n_axes, const int32_t *sections, int interleaved, float theta_base, void *y,
                  int64_t ldy, void *stream);

/* Quantises M tokens' keys and values (rows of n_kv_heads * head_dim values of `type`) into slots[m] (device, int64).
 * A negative slot skips its token (padding); the others have to differ. For each token and head, with TOP = 127
 * (B2S_TYPE_I8) or 448 (B2S_TYPE_F8_E4M3) and a = max(max |x|, 2^-100):
 *   code = round(x * (TOP / a)), scale = a / TOP   (fp32 quotients and product)
 * where round is to the nearest integer, halves away from zero, as in b2s_act_quant, or to the nearest e4m3 value,
 * ties to even. A head with an infinity or a NaN gets codes 0 and scale NaN: it reads back as NaN, and the rows that
 * attend to it are NaN. */
int b2s_kv_write(const b2s_kv_cache *cache, int32_t type, const void *k, int64_t ldk, const void *v, int64_t ldv,
                 int64_t M, const int64_t *slots, void *stream);

/* Reads M tokens back: row m of k and v = code * scale of slots[m], rounded once to `type`; zeros for a negative slot.
 * A slot may be read more than once. k or v may be NULL. */
int b2s_kv_read(const b2s_kv_cache *cache, const int64_t *slots, int64_t M, int32_t type, void *k, int64_t ldk, void *v,
                int64_t ldv, void *stream);

/* Workspace bytes of the attention calls for these shapes (M = rows of q; prefix_len = 0 for b2s_attention_kv) and for
 * calls on the same cache and n_heads whose M, batch, max_q, max_pages and prefix_len are no larger; 0 if they are not
 * valid. It is scratch of one call: nothing is kept in it, and calls that may overlap need one each. */
size_t b2s_attention_kv_workspace_size(const b2s_kv_cache *cache, const b2s_kv_batch *batch, int64_t M, int n_heads,
                                       int64_t prefix_len);

/* o = softmax(scale * q K^T) V of every sequence's query rows over its cached tokens; q and o [M][n_heads * head_dim]
 * of `type`, query head h reads key/value head h / (n_heads / n_kv_heads). With causal != 0 query row i of n sees the
 * tokens j <= kv_len - n + i, else all. A row that sees nothing is written as zeros; rows of o outside
 * [q_start[0], q_start[batch]) are left as they were. o may be q, with the same row stride (other overlaps are
 * not allowed). scale is finite and below 2^127.
 * Scores, softmax and sums are fp32, products run on the tensor cores, where the 8-bit codes are exact. fp32 queries
 * and probabilities are taken as two fp16 parts (error 2^-22 of the element, or of its row's largest one: 2^-38 where few
 * rows share a key/value head; where many do, 2^-33 for queries and 2^-32 for probabilities times their value scales), or,
 * queries of few rows on int8 codes, as integers of 24 bits under the row's largest element or 2^-100, if that is larger; bf16
 * queries likewise or exactly, their probabilities as fp32 ones. Where many rows share a head, the tensor cores cut sums off
 * below their last bit: about 2^-31 for each key that one block takes (5e-6 of an output over 8192 keys).
 * A query head with an infinity or a NaN is NaN; no other one is, as long as scores are within fp32's range. */
int b2s_attention_kv(const b2s_kv_cache *cache, const b2s_kv_batch *batch, int32_t type, const void *q, int64_t ldq,
                     int64_t M, int n_heads, float scale, int causal, void *o, int64_t ldo, void *workspace,
                     size_t workspace_bytes, void *stream);

/* The same with prefix_len tokens in front of every sequence that all of them share: token j of the prefix is in page
 * prefix_pages[j / page_size] (device, ceil(prefix_len / page_size) entries). kv_len counts the sequence's own tokens
 * behind it; every query row sees the whole prefix. The prefix is read once for the batch and joined with the own
 * tokens by the two parts' maxima and sums. (A short prefix is read by each sequence instead, where that takes less time.)
 * Where q_start[batch] is below a sequence's rows, that sequence may be left out too. prefix_len = 0 is b2s_attention_kv. */
int b2s_attention_kv_prefix(const b2s_kv_cache *cache, const b2s_kv_batch *batch, const int32_t *prefix_pages,
                            int64_t prefix_len, int32_t type, const void *q, int64_t ldq, int64_t M, int n_heads,
                            float scale, int causal, void *o, int64_t ldo, void *workspace, size_t workspace_bytes,
                            void *stream);

#ifdef __cplusplus
}
#endif
#endif /* B2S_KV_H */
