/*
 * marathon_kvstep.h -- C ABI of an engine step's operators around the block-scaled 8-bit KV
 * cache on MI355X (gfx950): heads normalised and turned to their positions, the same on their
 * way into the cache, and attention of a batch whose requests share what they begin with.
 *
 * Conventions are marathon_kvscaled.h's: device pointers, work enqueued on `stream`, nothing
 * allocated or synchronised, strides in ELEMENTS, rows and their strides aligned to 16 bytes,
 * MKV_OK or an MKV_ERR_* code with mkv_last_error(), indices in device memory checked on the
 * device.  A step's requests are described by its starts, lens and block_tables.
 *
 * No counterpart in the reference, whose engine does these itself (the rotation that its keys
 * come with is src/marathon/kvshift.py:44-61).
 */
#ifndef MARATHON_KVSTEP_H
#define MARATHON_KVSTEP_H

#include <stdint.h>

#include "marathon_kvscaled.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Heads x[0..D) of a token at position p become
 *     y = x / sqrt(mean(x^2) + eps) * weight            (norm 0: y = x)
 *     out[i]     = y[i] cos(a_i) - y[i + R/2] sin(a_i),
 *     out[i+R/2] = y[i+R/2] cos(a_i) + y[i] sin(a_i),    a_i = p * inv_freq[i],  i < R/2
 *     out[i]     = y[i],                                                         i >= R
 * (R = rotary) in fp32, the angles reduced in 64 bits (|a_i| below 2^50), rounded once.  The
 * squares are summed in 32 bits: a head whose squares pass fp32's range comes out as zeros,
 * or NaN where it holds an infinity.
 *
 *   inv_freq : fp32 [rotary / 2]; NULL for rotary 0.  rotary: a multiple of 32, at most
 *              head_size.
 *   q_weight, k_weight : [head_size] of weight_dtype (MKV_BF16, MKV_F16 or MKV_F32), 16-byte
 *              aligned, or NULL: ones.  NULL for norm 0.
 *   eps      : at least 0, finite.
 */
typedef struct mkv_turn {
  const float* inv_freq;
  const void* q_weight;
  const void* k_weight;
  int32_t rotary;
  int32_t weight_dtype;
  float eps;
  int32_t norm;
} mkv_turn_t;

/* [tokens, heads, head_size] in, and out; contiguous in the last dimension. */
typedef struct mkv_head_rows {
  const void* x;
  void* out;
  int64_t token_stride, head_stride;
  int64_t out_token_stride, out_head_stride;
  int32_t heads;
  int32_t reserved;
} mkv_head_rows_t;

/*
 * Query and key heads of a step, one launch.
 *   q, k      : of one dtype, MKV_BF16, MKV_F16 or MKV_F32; head_size 64, 128 or 256.  A row may
 *               be written where it was read (out = x, equal strides); otherwise no row of an
 *               output shares memory with another or with an input.
 *   positions : [tokens] of int32 or int64 (position_bytes 4 or 8); NULL for rotary 0.
 */
typedef struct mkv_norm_rotate_desc {
  mkv_head_rows_t q;
  mkv_head_rows_t k;
  mkv_turn_t turn;
  const void* positions;
  int64_t tokens;
  int32_t position_bytes;
  int32_t head_size;
  int32_t dtype;
  int32_t reserved;
} mkv_norm_rotate_desc_t;

int mkv_norm_rotate(const mkv_norm_rotate_desc_t* desc, void* stream);

/*
 * A step's projections: query heads normalised and turned as above, key heads too and, with the
 * values, into their blocks as mkv_store_scaled stores them; one launch.  A token's position is
 * its place in its request.  Keys are rounded once, from fp32 to their codes.
 *   q    : heads and rows of the queries; out's rows share no memory with the cache, k, v or,
 *          unless out = x with equal strides, with q.
 *   k, v : [tokens, cache heads, head_size], all of q's dtype.
 * Rows of no request are neither read nor written.
 */
typedef struct mkv_store_rotated_desc {
  mkv_scaled_cache_t cache;
  mkv_head_rows_t q;
  mkv_turn_t turn;
  const void* k;
  const void* v;
  int64_t k_token_stride, k_head_stride;
  int64_t v_token_stride, v_head_stride;
  const int32_t* block_tables;
  const int32_t* starts;
  const int32_t* lens;
  int32_t* error_flags;
  int64_t table_stride;
  int64_t tokens;
  int32_t table_width;
  int32_t requests;
  int32_t dtype;
  int32_t reserved;
} mkv_store_rotated_desc_t;

int mkv_store_rotated(const mkv_store_rotated_desc_t* desc, void* stream);

/*
 * mkv_attend_scaled for a batch whose requests begin, in groups, with the same cached tokens.
 *   groups : int32 [n_groups + 1], 0 <= n_groups <= MKV_MAX_REQUESTS: requests [groups[g],
 *            groups[g + 1]) begin alike; groups[0] >= 0, not descending.  A request in no group
 *            shares nothing.
 *   shared : int32 [n_groups]: how many tokens; of them the whole blocks, shared[g] / block_size,
 *            are read through block_tables' row groups[g] for the whole group, and its other
 *            requests' entries for them are not read.  A row sees of them what stands before it.
 *   attend : as mkv_attend_scaled takes it, but for
 *            max_len    the most tokens that a request has behind what its group shares (0: not
 *                       known), and
 *            workspace  mkv_attend_shared_workspace_size() bytes.
 *   max_shared : the most tokens that a group shares, where the caller knows it (0: not known).
 * Where the tables of a group agree, the result is mkv_attend_scaled's but for the order of sums
 * and p's roundings: over both ranges p is held in two bf16 terms (off by at most 2^-17) for every
 * request whose p mkv_attend_scaled holds in two, by the same max_new, however many rows share; for
 * the others in one (off by 2^-8) or two.  The hints change a result by this and by the order of sums
 * alone.
 * Groups that leave the requests or descend, and shared tokens below zero, raise MKV_FLAG_SPAN
 * and share nothing: their requests' own tables are read from the first token on.  The others share
 * what they share, but for those that a descending group reaches into.  More shared tokens than a
 * table has raise MKV_FLAG_SRC_RANGE, and are cut.
 */
typedef struct mkv_attend_shared_desc {
  mkv_attend_desc_t attend;
  const int32_t* groups;
  const int32_t* shared;
  int32_t n_groups;
  int32_t max_shared;
} mkv_attend_shared_desc_t;

int mkv_attend_shared(const mkv_attend_shared_desc_t* desc, void* stream);

/* Workspace bytes of that call (it reads no device memory); -1 where it would be refused. */
int64_t mkv_attend_shared_workspace_size(const mkv_attend_shared_desc_t* desc);

#ifdef __cplusplus
}
#endif

#endif /* MARATHON_KVSTEP_H */
