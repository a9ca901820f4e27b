/*
 * marathon_kvscaled.h -- C ABI of the block-scaled 8-bit KV cache on MI355X (gfx950).
 *
 * The cache is paged as the other entry points' caches are (blocks of block_size tokens,
 * rows K[head_size] and V[head_size] per token and KV head) and holds OCP e4m3fn codes.
 * Each (block, KV head) has two scales, one for K and one for V, held as their exponents
 * in OCP e8m0 (byte b stands for 2^(b - 127)):
 *
 *     x = decode(code) * 2^e,      e in [MKV_SCALE_MIN_EXP, MKV_SCALE_MAX_EXP]
 *
 * A byte outside that range is read as the nearer end of it.  A power of two loses nothing
 * against a free scale, e4m3 being a floating-point format itself, and buys three things:
 * every product code * 2^e is exact in bf16 and fp32, a row encoded again under a larger
 * scale keeps its value exactly wherever the code does not become subnormal, and gfx950's
 * conversions apply the scale as they decode.
 *
 * A block's scale is the smallest that fits its rows (the largest finite |x| <= 448 * 2^e;
 * MKV_SCALE_MIN_EXP for rows of zeros).  Encoding is
 *     code = e4m3fn_RNE(clamp(x * 2^-e, -448, 448)),      NaN -> 0x7F
 * with x the input in fp32: infinities saturate, and neither they nor NaNs enter the scale.
 *
 * A request's tokens fill its blocks in order: position p is row p % block_size of block
 * block_table[request][p / block_size].  Rows of a block behind the last written one hold
 * anything, and no entry point looks at them.  A block belongs to one request: calls that
 * write it from two at once leave it undefined.
 *
 * Conventions are marathon_kvshift.h's: device pointers, work enqueued on `stream`, nothing
 * allocated or synchronised, strides in ELEMENTS, cache bases and strides aligned to 16
 * bytes, MKV_OK or an MKV_ERR_* code with mkv_last_error(), and every index that lies in
 * device memory checked on the device: what fails is neither read nor written and sets
 * MKV_FLAG_* bits in `error_flags` (device int32 [1], or NULL).
 *
 * A step's requests are described by three device arrays:
 *   starts        int32 [requests + 1]: request r's new tokens are rows [starts[r],
 *                 starts[r + 1]) of the step's token arrays; starts[0] >= 0, not descending.
 *                 Rows at or behind starts[requests] belong to nobody.
 *   lens          int32 [requests]: tokens each request holds WITH its new ones, so row i
 *                 of request r is position lens[r] - (starts[r + 1] - starts[r]) + i.
 *   block_tables  int32 [requests, table_width], rows table_stride apart; at most 2^30 tokens
 *                 a request.
 * A request whose starts leave the token arrays is skipped; where starts descend, rows stay
 * untouched or go to a neighbouring request.  Both raise MKV_FLAG_SPAN, as does, in a store, a
 * request with more new tokens than tokens, which is skipped.
 *
 * No counterpart in the reference, whose caches are bf16 and whose slots are made on the
 * host (src/marathon/shift_store.py:56-60).
 */
#ifndef MARATHON_KVSCALED_H
#define MARATHON_KVSCALED_H

#include <stdint.h>

#include "marathon_kvshift.h"

#ifdef __cplusplus
extern "C" {
#endif

#define MKV_SCALE_MIN_EXP (-100)
#define MKV_SCALE_MAX_EXP 100
#define MKV_MAX_REQUESTS 4096

/*
 * One layer's cache.
 *   k_base, v_base : element 0 of K and V; fused rows have v_base = k_base + head_size.
 *   scales         : device [num_blocks, heads, 2] e8m0 bytes, contiguous: K's, then V's.
 *   block_stride, head_stride, token_stride : bytes (= elements), multiples of 16.
 *                    No row of K or V lies in another.
 *   block_size     : 16, 32, 64 or 128.   head_size : 64, 128 or 256.
 */
typedef struct mkv_scaled_cache {
  void* k_base;
  void* v_base;
  uint8_t* scales;
  int64_t num_blocks;
  int64_t block_stride;
  int64_t head_stride;
  int64_t token_stride;
  int32_t block_size;
  int32_t heads;
  int32_t head_size;
  int32_t reserved;
} mkv_scaled_cache_t;

/*
 * Block tables and slot map of one step, from the requests' lengths: one launch.
 *   held, fresh   : int32 [requests], tokens each request holds and its new ones (>= 0);
 *                   0 <= requests <= MKV_MAX_REQUESTS.
 *   block_tables  : extended in place: request r's entries for blocks
 *                   [ceil(held / bs), ceil((held + fresh) / bs)) are taken from the free
 *                   list, requests in order; no other entry is touched.
 *   free_blocks   : int32 [free_len], ids of free blocks; those from free_at[0] on are free.
 *   starts, lens  : out, as above.
 *   slots         : out int64 [max_tokens]: block * block_size + row of every new token, -1
 *                   behind the last one and where a block's id is negative (ids are not checked
 *                   otherwise: what takes them knows their cache).  positions: out int32
 *                   [max_tokens], 0 behind the last one.
 *   free_at_out   : out int32 [1]: where the free list begins now.  Not free_at itself; nor
 *                   does another output share memory with an input.
 * All or nothing: where a length is negative, the new tokens exceed max_tokens, a request
 * exceeds its table or the free list runs out, MKV_FLAG_DST_RANGE is raised, no table entry
 * changes, lens = held, starts and positions are 0, slots are -1 and free_at_out = free_at.
 * Exact integers; any block_size > 0.
 */
int mkv_step_slots(const int32_t* held, const int32_t* fresh, int32_t requests,
                   int32_t* block_tables, int64_t table_stride, int32_t table_width,
                   const int32_t* free_blocks, int64_t free_len, const int32_t* free_at,
                   int32_t block_size, int32_t* starts, int32_t* lens, int64_t* slots,
                   int32_t* positions, int64_t max_tokens, int32_t* free_at_out,
                   int32_t* error_flags, void* stream);

/*
 * New K and V rows into their blocks: one launch.
 *   k, v : [tokens, heads, head_size] of dtype MKV_BF16, MKV_F16 or MKV_F32, contiguous in the
 *          last dimension, token and head strides given, aligned to 16 bytes.
 * A block that its request begins here gets the scale of its new rows.  A block begun before
 * keeps its rows [0, p) and at least its scale: where the new rows need a larger one, the
 * rows [0, p) are encoded again under it.
 */
int mkv_store_scaled(const mkv_scaled_cache_t* cache, const void* k, int64_t k_token_stride,
                     int64_t k_head_stride, const void* v, int64_t v_token_stride,
                     int64_t v_head_stride, int64_t tokens, int32_t dtype,
                     const int32_t* block_tables, int64_t table_stride, int32_t table_width,
                     const int32_t* starts, const int32_t* lens, int32_t requests,
                     int32_t* error_flags, void* stream);

/*
 * Causal grouped-query attention over the cache.
 *   q, out : [tokens, q_heads, head_size] of dtype MKV_BF16 or MKV_F16, contiguous in the
 *            last dimension, aligned to 16 bytes; q_heads a multiple of the cache's heads,
 *            query head h reads KV head h / (q_heads / heads).  out's rows do not overlap
 *            each other, q or the cache.
 *   out[i] = sum_j p_j V[j],  p = softmax over j <= position(i), j < lens[r], of
 *            softmax_scale * q[i] . K[j]
 * computed with fp32 sums and softmax statistics.  Where it meets V, p is held in two bf16 terms,
 * off by at most 2^-17 of itself; in one, off by 2^-8, in the kernel of more than 32 rows for bf16
 * queries (rows: max_new, or without it the tokens, times the query heads of a KV head).
 * A row that sees no key is zeros; rows that belong to no request are left as they were.  Tokens
 * of a block whose id is out of range are not seen (MKV_FLAG_SRC_RANGE), nor are those behind
 * the block table.  What lies in rows that a query does not see has no effect, NaNs included.
 *   max_new, max_len : the largest number of new tokens and of tokens of a request, where the
 *            caller knows them (0: not known).  They choose launch shapes; wrong ones cost
 *            time, and change a result by the order of its sums and by p's roundings alone.
 *   workspace : device, mkv_attend_workspace_size() bytes for the same arguments, 16-byte
 *            aligned; overwritten, so calls that overlap on one workspace race.  May be NULL
 *            where that size is 0.
 */
typedef struct mkv_attend_desc {
  mkv_scaled_cache_t cache;
  const void* q;
  void* out;
  const int32_t* block_tables;
  const int32_t* starts;
  const int32_t* lens;
  int32_t* error_flags;
  void* workspace;
  int64_t workspace_bytes;
  int64_t q_token_stride;
  int64_t q_head_stride;
  int64_t out_token_stride;
  int64_t out_head_stride;
  int64_t table_stride;
  int64_t tokens;
  int32_t table_width;
  int32_t requests;
  int32_t q_heads;
  int32_t dtype;
  int32_t max_new;
  int32_t max_len;
  float softmax_scale;
  int32_t reserved;
} mkv_attend_desc_t;

int mkv_attend_scaled(const mkv_attend_desc_t* desc, void* stream);

/* Workspace bytes of that call (it reads no device memory); -1 where it would be refused. */
int64_t mkv_attend_workspace_size(const mkv_attend_desc_t* desc);

/*
 * Spans moved between block-scaled caches, every layer at once: mkv_shift_spans for
 * this cache.  Row i of span s is read at source position src_pos + i through src_table and
 * written at dst_pos + i through dst_table, K re-rotated by delta as marathon_kvshift.h says
 * (fp32, no fused multiply-add); the destination blocks are encoded anew, each under the
 * scale of the rows that it receives.  Of rows behind a span's last one the codes stay, but
 * the block's scale is the new rows': their values are undefined until they are written.
 * A block is written with all of its rows or, where a source block of one is out of range,
 * left as it was, its scales among it.
 * Destination blocks are distinct and no source blocks of the call, in any layer.
 *
 * mkv_scaled_units (a host function, no GPU call; every pointer a HOST one) resolves spans
 * into units, one for each destination block:
 *   spans  : [n_spans], 0 <= n_spans <= MKV_MAX_SPANS; src_index and dst_index are added to
 *            the block numbers in the tables; groups are not read.  A span whose dst_pos is
 *            not a multiple of the destination's block size, or with a negative position or
 *            length, gets no units (MKV_FLAG_SPAN): a block is written by one span.
 *   src, dst : geometry (block_size and num_blocks; the rest is not read).  A block that is a
 *            destination twice is refused (MKV_ERR_ARG); within one cache, which is said by
 *            one pointer for both, so is a source block that is a destination too.
 *   units  : out, room for max_units of them; at least the sum of ceil(n_tokens / dst
 *            block_size) is never too little (MKV_ERR_ARG otherwise).  A unit is
 *            MKV_UNIT_WORDS(src block_size, dst block_size) words, int32:
 *              0  destination block         1  rows, 1 to its block size
 *              2  span, whose rotation table it takes; -1: delta 0
 *              3  row 0's place in the first source block
 *              4..  source blocks, in order; -1: out of range; then zeros
 *   *n_units : out.
 *   *flags : out (or NULL), MKV_FLAG bits: a block whose id is out of range gets no unit
 *            (DST_RANGE); a unit one of whose source blocks is leaves its block as it was
 *            (SRC_RANGE).
 */
#define MKV_UNIT_SOURCES(src_bs, dst_bs) ((dst_bs) > (src_bs) ? (dst_bs) / (src_bs) + 1 : 2)
#define MKV_UNIT_WORDS(src_bs, dst_bs) ((4 + MKV_UNIT_SOURCES(src_bs, dst_bs) + 3) / 4 * 4)

int mkv_scaled_units(const mkv_span_t* spans, int32_t n_spans, const int32_t* src_table,
                     int64_t src_table_len, const int32_t* dst_table, int64_t dst_table_len,
                     const mkv_scaled_cache_t* src, const mkv_scaled_cache_t* dst,
                     int32_t* units, int64_t max_units, int64_t* n_units, int32_t* flags);

/*
 *   units        : device [n_units], 16-byte aligned, made by mkv_scaled_units; ids in them
 *                  are checked again.
 *   tables       : device fp32 [n_spans][2][rotary], mkv_rope_tables' layout; NULL for
 *                  rotary 0.  rotary: a multiple of 32, at most head_size.
 *   src_layers, dst_layers : device [layers][3]: k_base, v_base and scales of each layer.
 *   src, dst     : geometry of every layer (their base and scale pointers are not read).
 *   on_host      : 1 if units and tables are host memory.  They are read before the call
 *                  returns and passed on in the arguments of launches that each take
 *                  MKV_SHIFT_HOST_BYTES of both (MKV_ERR_ARG for a unit of no span).
 */
#define MKV_SHIFT_HOST_BYTES 3584

typedef struct mkv_scaled_shift_desc {
  mkv_scaled_cache_t src;
  mkv_scaled_cache_t dst;
  const uint64_t* src_layers;
  const uint64_t* dst_layers;
  const int32_t* units;
  const float* tables;
  int64_t n_units;
  int32_t n_spans;
  int32_t layers;
  int32_t rotary;
  int32_t on_host;
} mkv_scaled_shift_desc_t;

int mkv_shift_scaled(const mkv_scaled_shift_desc_t* desc, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* MARATHON_KVSCALED_H */
