/*
 * pad_b200.h -- C ABI of the B200 (sm_100a) paged-attention decode library
 * (libpad_b200.so).
 *
 * Every entry point takes plain pointers, sizes and strides (in ELEMENTS),
 * never framework types, and returns a pad_status code. Pointers to tensors
 * are device pointers on the device that is current when the call is made.
 * Calls are asynchronous on the given CUDA stream (a cudaStream_t passed as
 * void*; NULL means the legacy default stream) and never synchronise the
 * device.
 *
 * The decode entry point replaces, as one C call, the reference project's
 * pybind binding ``forward_v4(q, k_cache, v_cache, block_table, seq_lens,
 * scale, gqa_ratio, head_dim, page_size, num_splits)`` (cuda/binding.cpp:13-14,
 * declared at cuda/kernels.h:60-70) and the launcher behind it
 * (cuda/kernel_v4_split_k.cu:205-268). Differences, by design:
 *   - the caller owns `out` and a reusable `workspace` (the reference
 *     allocated both with torch on every call, cuda/kernel_v4_split_k.cu:228-232);
 *   - the stream is explicit (the reference launched on the legacy default
 *     stream, cuda/kernel_v4_split_k.cu:238,257);
 *   - argument errors come back as status codes instead of TORCH_CHECK
 *     exceptions (cuda/kernel_v4_split_k.cu:216-223).
 *
 * Tensor layouts (the reference's, README.md:38-44):
 *   q, out       [batch, num_q_heads, head_dim]            fp16
 *   k/v_cache    [num_pages, page_size, num_kv_heads, head_dim] fp16
 *   block_table  [batch, max_pages_per_seq]                int32
 *   seq_lens     [batch]                                   int32
 * The last dimension of q, out, k_cache and v_cache must be contiguous
 * (stride 1); the other strides of q/k_cache/v_cache must be multiples of
 * 8 elements (16 bytes, a TMA requirement) and the base pointers 16-byte
 * aligned. block_table's inner stride must be 1.
 */
#ifndef PAD_B200_H_
#define PAD_B200_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef enum pad_status {
  PAD_OK = 0,
  PAD_ERR_INVALID_ARGUMENT = 1, /* a shape, size or pointer is invalid      */
  PAD_ERR_UNSUPPORTED = 2,      /* valid but outside what the kernels cover */
  PAD_ERR_WORKSPACE = 3,        /* workspace missing or too small           */
  PAD_ERR_CUDA = 4,             /* a CUDA runtime/driver call failed        */
} pad_status;

/* Bits OR-ed into *error_flags by the kernels (value checks the reference's
 * oracle performs on the host, src/reference.py:40-41,107-112, done here on
 * the device without a host sync). */
#define PAD_FLAG_BAD_PAGE_ID 0x1     /* a block_table entry outside [0, num_pages) */
#define PAD_FLAG_SEQ_LEN_RANGE 0x2   /* seq_len < 0 or > max_pages_per_seq * page_size */
#define PAD_FLAG_BAD_SEQ_ID 0x4      /* a seq_ids entry outside [0, batch) */
#define PAD_FLAG_SHARED_PAGE 0x8     /* more tokens than the pool's pages hold: sequences share pages */
#define PAD_FLAG_SCALE_RANGE 0x10    /* a V scale of a 4-bit cache above 2^13 */
#define PAD_FLAG_WAIT_TIMEOUT 0x100  /* an in-kernel wait gave up (never expected) */

/* Human-readable text for a status code (static storage). */
const char* pad_status_string(int status);

/* Text of the last error on the calling thread (static thread-local storage). */
const char* pad_last_error(void);

/* Library version as MAJOR*10000 + MINOR*100 + PATCH. */
int pad_version(void);

/* Number of SMs of `device` and how many decode CTAs one SM holds for the
 * given head_dim / gqa_ratio (the inputs of the split heuristic). */
int pad_device_info(int device, int64_t head_dim, int64_t gqa_ratio, int* num_sms, int* ctas_per_sm);

/* Number of persistent decode CTAs (work partitions) the decode call will
 * launch for this problem on `device`.
 *   num_splits <= 0 : heuristic -- one partition per resident CTA slot
 *                     (num_sms * ctas_per_sm), capped by the number of
 *                     tiles the batch can hold (a tile is 128 (token,
 *                     KV head) rows: 128 / HG tokens of HG KV heads, HG the
 *                     largest of 8, 4, 2, 1 dividing num_kv_heads, at most
 *                     4 when gqa_ratio > 8);
 *   num_splits >= 1 : num_splits partitions per (sequence, KV head) pair,
 *                     i.e. num_splits * batch * num_kv_heads partitions. */
int pad_decode_partitions(int device, int64_t batch, int64_t num_kv_heads, int64_t gqa_ratio,
                          int64_t head_dim, int64_t page_size, int64_t max_pages_per_seq,
                          int64_t num_splits, int64_t* partitions);

/* Bytes of device workspace pad_paged_attention_decode needs for this
 * problem (same arguments as pad_decode_partitions). The workspace holds the
 * fp32 split partials (O, m, l) and per-partition merge descriptors; it
 * needs no initialisation and may be reused by consecutive calls on one
 * stream (calls that overlap in time must use distinct workspaces). */
int pad_decode_workspace_bytes(int device, int64_t batch, int64_t num_kv_heads, int64_t gqa_ratio,
                               int64_t head_dim, int64_t page_size, int64_t max_pages_per_seq,
                               int64_t num_splits, size_t* bytes);

/* Decode attention over a paged fp16 KV cache with GQA.
 *
 *   out[b, h, :] = softmax(scale * q[b, h, :] . K_b[h / G]^T) @ V_b[h / G]
 *
 * where K_b/V_b are the first seq_lens[b] token rows of the pages
 * block_table[b, 0 .. ceil(seq_lens[b] / page_size) - 1] and
 * G = num_q_heads / num_kv_heads. A sequence with seq_len == 0 yields a zero
 * row (src/reference.py:32-34). Entries of block_table past a sequence's
 * last page are never read.
 *
 * Strides are in elements: q_strides[3], k_strides[4], v_strides[4],
 * out_strides[3]; block_table_stride is the row stride of block_table.
 * error_flags (device int32, optional) receives PAD_FLAG_* bits; it is
 * OR-ed into, never cleared.
 *
 * Invalid values are flagged, never faulted on: a block_table entry outside
 * [0, num_pages) sets PAD_FLAG_BAD_PAGE_ID and the tokens it addresses are
 * read as zero K/V rows (the tensor copy zero-fills out-of-range boxes); a
 * seq_len outside [0, max_pages_per_seq * page_size] sets
 * PAD_FLAG_SEQ_LEN_RANGE and is clamped into that range. When either flag is
 * set the output of the call is undefined (the reference oracle raises
 * ValueError instead, src/reference.py:40-41,107-112).
 *
 * The library caches per-device facts (kernel attributes, occupancy, the
 * no-alloc scratch address) for the life of the process; it must not be used
 * across a cudaDeviceReset of a device it has run on.
 */
int pad_paged_attention_decode(const void* q, const void* k_cache, const void* v_cache,
                               const int32_t* block_table, const int32_t* seq_lens, void* out,
                               int64_t batch, int64_t num_q_heads, int64_t num_kv_heads,
                               int64_t head_dim, int64_t num_pages, int64_t page_size,
                               int64_t max_pages_per_seq, const int64_t* q_strides,
                               const int64_t* k_strides, const int64_t* v_strides,
                               int64_t block_table_stride, const int64_t* out_strides, float scale,
                               int64_t num_splits, void* workspace, size_t workspace_bytes,
                               void* stream, int32_t* error_flags);

/* Decode with a CSR page index instead of a dense block table -- the
 * (indptr, indices, last_page_len) layout the reference's FlashInfer adapter
 * builds from a block table (src/flashinfer_adapter.py:40-65):
 *   pages of sequence b = kv_indices[kv_indptr[b] .. kv_indptr[b+1])
 *   seq_len of b        = (pages - 1) * page_size + kv_last_page_len[b]
 *                         (0 when the sequence has no pages)
 * nnz_pages is the length of kv_indices. Everything else -- strides, scale,
 * num_splits, workspace (sized by pad_decode_csr_workspace_bytes), stream,
 * error flags -- is as for pad_paged_attention_decode. */
int pad_decode_csr_workspace_bytes(int device, int64_t batch, int64_t num_kv_heads, int64_t gqa_ratio,
                                   int64_t head_dim, int64_t page_size, int64_t nnz_pages,
                                   int64_t num_splits, size_t* bytes);
int pad_paged_attention_decode_csr(const void* q, const void* k_cache, const void* v_cache,
                                   const int32_t* kv_indptr, const int32_t* kv_indices,
                                   const int32_t* kv_last_page_len, void* out, int64_t batch,
                                   int64_t num_q_heads, int64_t num_kv_heads, int64_t head_dim,
                                   int64_t num_pages, int64_t page_size, int64_t nnz_pages,
                                   const int64_t* q_strides, const int64_t* k_strides,
                                   const int64_t* v_strides, const int64_t* out_strides, float scale,
                                   int64_t num_splits, void* workspace, size_t workspace_bytes,
                                   void* stream, int32_t* error_flags);

/* Write one new token's K and V per sequence into the paged cache (the step
 * before decode; the reference fixes this cache layout, README.md:38-44, but
 * has no writer). Token positions[b] of sequence b goes to page
 * block_table[b, positions[b] / page_size], row positions[b] % page_size,
 * for every KV head; positions[b] < 0 skips sequence b.
 * k_new / v_new are [batch, num_kv_heads, head_dim] fp16 with strides
 * k_new_strides[3] / v_new_strides[3]; caches as for decode. A position past
 * the block table sets PAD_FLAG_SEQ_LEN_RANGE, a bad page id
 * PAD_FLAG_BAD_PAGE_ID (nothing is written for that row). */
int pad_paged_kv_append(const void* k_new, const void* v_new, void* k_cache, void* v_cache,
                        const int32_t* block_table, const int32_t* positions, int64_t batch,
                        int64_t num_kv_heads, int64_t head_dim, int64_t num_pages, int64_t page_size,
                        int64_t max_pages_per_seq, const int64_t* k_new_strides,
                        const int64_t* v_new_strides, const int64_t* k_strides, const int64_t* v_strides,
                        int64_t block_table_stride, void* stream, int32_t* error_flags);

/* Decode without any device allocation, for callers that cannot call
 * cudaMalloc: code running inside a CUDA stream capture they do not own,
 * embedders whose memory is owned by a custom allocator or a fixed arena,
 * and real-time paths where an allocation could block. It behaves exactly
 * like pad_paged_attention_decode (same arguments minus the workspace) but
 * keeps the split partials in a scratch array built into the library,
 * PAD_STATIC_SCRATCH_BYTES (16 MiB) per GPU, which every GPU that loads the
 * library holds until the process exits. Problems whose workspace
 * (pad_decode_workspace_bytes) exceeds that size are rejected with
 * PAD_ERR_WORKSPACE. The first call on a device looks up the scratch
 * array's device address (cudaGetSymbolAddress) with that device current,
 * so make that first call before any stream capture. All calls on a device
 * share the one array: calls that overlap on the GPU (different streams, no
 * ordering between them) race and must be avoided. Nothing in the array has
 * to start zeroed; each call rewrites what it reads.
 * No counterpart in the reference. */
#define PAD_STATIC_SCRATCH_BYTES ((size_t)16 << 20)
int pad_paged_attention_decode_noalloc(const void* q, const void* k_cache, const void* v_cache,
                                       const int32_t* block_table, const int32_t* seq_lens, void* out,
                                       int64_t batch, int64_t num_q_heads, int64_t num_kv_heads,
                                       int64_t head_dim, int64_t num_pages, int64_t page_size,
                                       int64_t max_pages_per_seq, const int64_t* q_strides,
                                       const int64_t* k_strides, const int64_t* v_strides,
                                       int64_t block_table_stride, const int64_t* out_strides,
                                       float scale, int64_t num_splits, void* stream,
                                       int32_t* error_flags);

/* ---------------------------------------------------------------------------
 * The 4-bit cache. A token's row of one KV head is head_dim/2 code bytes and
 * 4 scale bytes, for K and for V (head_dim 32, 64 or 128):
 *   k/v_cache    [num_pages, page_size, num_kv_heads, head_dim / 2]  uint8
 *   k/v_scales   [num_pages, page_size, num_kv_heads, 4]             uint8
 * Code byte i holds dims 2i (low nibble) and 2i + 1 as e2m1 (0 0.5 1 1.5 2 3 4
 * 6 and their negatives); scale byte j is the power of two 2^(byte - 127) of
 * dims [32j, 32j + 32), 255 meaning NaN. Scale bytes past head_dim / 32 are
 * written as 0 and never read. Codes must be 16-byte aligned with strides that
 * are multiples of 16 bytes, scales 4-byte aligned with strides that are
 * multiples of 4; last axes contiguous. Strides of uint8 tensors are bytes.
 *
 * pad_paged_kv_append_fp4 quantises and writes `tokens` new rows: row t of
 * k_new / v_new [tokens, num_kv_heads, head_dim] fp16 becomes token
 * positions[t] of sequence seq_ids[t] (seq_ids NULL: of sequence t, and tokens
 * <= batch). Per block of 32 with a = max |x|: E = max(floor(log2 a) - 2, -24),
 * scale byte E + 127, codes round(x / 2^E) to nearest even, saturated at 6. A
 * block with an Inf or NaN gets scale 255 and zero codes. positions[t] < 0
 * skips t. A position past the block table sets PAD_FLAG_SEQ_LEN_RANGE, a bad
 * page id PAD_FLAG_BAD_PAGE_ID, a seq_ids entry outside [0, batch)
 * PAD_FLAG_BAD_SEQ_ID; nothing is written for that token. One call must not
 * name the same (sequence, position) twice.
 *
 * pad_paged_kv_read_fp4 gives the rows back as fp16 [tokens, num_kv_heads,
 * head_dim] (exactly what the codes of an appended row stand for); a token
 * that is skipped or flagged reads as zeros. No counterpart in the reference. */
int pad_paged_kv_append_fp4(const void* k_new, const void* v_new, void* k_cache, void* k_scales, void* v_cache,
                            void* v_scales, const int32_t* block_table, const int32_t* positions,
                            const int32_t* seq_ids, int64_t tokens, int64_t batch, int64_t num_kv_heads,
                            int64_t head_dim, int64_t num_pages, int64_t page_size, int64_t max_pages_per_seq,
                            const int64_t* k_new_strides, const int64_t* v_new_strides, const int64_t* k_strides,
                            const int64_t* ks_strides, const int64_t* v_strides, const int64_t* vs_strides,
                            int64_t block_table_stride, void* stream, int32_t* error_flags);
int pad_paged_kv_read_fp4(const void* k_cache, const void* k_scales, const void* v_cache, const void* v_scales,
                          const int32_t* block_table, const int32_t* positions, const int32_t* seq_ids, void* k_out,
                          void* v_out, int64_t tokens, int64_t batch, int64_t num_kv_heads, int64_t head_dim,
                          int64_t num_pages, int64_t page_size, int64_t max_pages_per_seq, const int64_t* k_strides,
                          const int64_t* ks_strides, const int64_t* v_strides, const int64_t* vs_strides,
                          const int64_t* k_out_strides, const int64_t* v_out_strides, int64_t block_table_stride,
                          void* stream, int32_t* error_flags);

/* Decode attention over the 4-bit cache: pad_paged_attention_decode with K and
 * V what their codes and scales stand for. V's scales may lie in 2^-24 .. 2^13,
 * which is all that the append writes, where code x scale is an fp16 value;
 * smaller ones count as 0 (the output moves by less than 6 x 2^-25), and one above
 * 2^13 that a sequence attends to sets PAD_FLAG_SCALE_RANGE and leaves that
 * sequence's output undefined (Inf or NaN). K's scales are applied in fp32 and
 * have no such bound. A NaN scale makes the sequences that attend to it NaN. head_dim 32, 64 or 128, gqa_ratio up to 16. q must be
 * 16-byte aligned with strides that are multiples of 8 elements, out 4-byte
 * aligned with even strides. weights, slot_positions, total_lens and num_new
 * are those of pad_paged_attention_decode_weights below; weights NULL leaves
 * them out. num_splits >= 1: partitions per (sequence, group of up to 4 KV
 * heads). The workspace (pad_decode_fp4_workspace_bytes; with_weights 0 or
 * 1; num_pages matters with weights alone) needs no initialisation. A bad page
 * id reads as zero rows. */
int pad_decode_fp4_workspace_bytes(int device, int64_t batch, int64_t num_kv_heads, int64_t gqa_ratio,
                                   int64_t head_dim, int64_t num_pages, int64_t page_size,
                                   int64_t max_pages_per_seq, int64_t num_splits, int with_weights, size_t* bytes);
int pad_paged_attention_decode_fp4(const void* q, const void* k_cache, const void* k_scales, const void* v_cache,
                                   const void* v_scales, const int32_t* block_table, const int32_t* seq_lens,
                                   void* out, float* weights, int32_t* slot_positions, const int32_t* total_lens,
                                   int64_t num_new, int64_t batch, int64_t num_q_heads, int64_t num_kv_heads,
                                   int64_t head_dim, int64_t num_pages, int64_t page_size, int64_t max_pages_per_seq,
                                   const int64_t* q_strides, const int64_t* k_strides, const int64_t* ks_strides,
                                   const int64_t* v_strides, const int64_t* vs_strides, int64_t block_table_stride,
                                   const int64_t* out_strides, const int64_t* weight_strides,
                                   const int64_t* position_strides, float scale, int64_t num_splits, void* workspace,
                                   size_t workspace_bytes, void* stream, int32_t* error_flags);
int pad_paged_attention_decode_fp4_by_seq(
    const void* q, const void* k_cache, const void* k_scales, const void* v_cache, const void* v_scales,
    const int32_t* block_table, const int32_t* seq_lens, void* out, float* weights, int32_t* slot_positions,
    const int32_t* total_lens, const int32_t* num_new, int64_t batch, int64_t num_q_heads, int64_t num_kv_heads,
    int64_t head_dim, int64_t num_pages, int64_t page_size, int64_t max_pages_per_seq, const int64_t* q_strides,
    const int64_t* k_strides, const int64_t* ks_strides, const int64_t* v_strides, const int64_t* vs_strides,
    int64_t block_table_stride, const int64_t* out_strides, const int64_t* weight_strides,
    const int64_t* position_strides, float scale, int64_t num_splits, void* workspace, size_t workspace_bytes,
    void* stream, int32_t* error_flags);

/* ---------------------------------------------------------------------------
 * Eviction by accumulated attention weight. Beside a paged cache live
 *   weights         [num_pages, num_kv_heads, page_size]  fp32
 *   slot_positions  [num_pages, num_kv_heads, page_size]  int32 (optional)
 * addressed through the same block table: what a slot's token has received, and
 * the token's position in its sequence (after an eviction a slot no longer
 * tells it). Any strides (in elements). A page belongs to one sequence.
 *
 * pad_paged_attention_decode_weights is pad_paged_attention_decode and then,
 * for every slot t < seq_lens[b] and KV head,
 *   weights = (t >= seq_lens[b] - num_new ? 0 : weights) + the softmax
 *             probabilities of the token, summed over the KV head's query heads
 * so that slots of the num_new newest tokens need no clearing; with
 * slot_positions these slots also get total_lens[b] - seq_lens[b] + t. num_new is
 * one number for all sequences, or, with pad_paged_attention_decode_weights_by_seq
 * (and pad_paged_attention_decode_fp4_by_seq), a device array [batch] int32 of
 * each one's, for batches that a sequence joins with its prompt; a negative entry
 * counts as 0. The
 * workspace (pad_decode_weights_workspace_bytes) also holds the call's scores,
 * 4 bytes per query head and token that the batch can hold: of min(batch *
 * max_pages_per_seq, num_pages) pages. Each weight has one writer, so results
 * are repeatable. Sequences that share pages break that: their weights lose
 * additions, other ones from run to run, and a move of one overwrites rows of the
 * other. PAD_FLAG_SHARED_PAGE is set only when they hold more tokens than the
 * pool; the Python calls refuse any shared page with PAD_B200_CHECK=1.
 *
 * pad_paged_kv_evict_plan chooses, for every sequence b with seq_lens[b] >
 * budget and every KV head, the `budget` slots to keep: first those that are
 * recent (slot_positions >= total_lens[b] - recent), then by weight descending
 * (NaN above all), ties to the lower slot. Kept slots at or above `budget` move
 * to the slots below it that are not kept:
 *   src, dst  [batch, num_kv_heads, max_moves] int32, both ascending, -1 behind
 *             the last move; max_moves = pad_evict_max_moves(...)
 *   counts    [batch, num_kv_heads] int32, moves of each
 *   new_lens  [batch] int32, min(seq_lens, budget)
 * recent > 0 needs slot_positions and total_lens ([batch] int32, tokens each
 * sequence has seen). Nothing of the cache is touched.
 *
 * pad_paged_kv_move copies row src -> row dst of 1 to 4 caches [num_pages,
 * page_size, num_kv_heads, row] (row_bytes[c] contiguous bytes; cache_strides
 * [num_caches][3]: page, row and head strides in BYTES), of weights and of
 * slot_positions (each optional). Within one (sequence, KV head) no dst may be
 * a src or occur twice, as in a plan. Entries outside the block table set
 * PAD_FLAG_SEQ_LEN_RANGE and are skipped. No counterpart in the reference. */
int pad_decode_weights_workspace_bytes(int device, int64_t batch, int64_t num_kv_heads, int64_t gqa_ratio,
                                       int64_t head_dim, int64_t num_pages, int64_t page_size,
                                       int64_t max_pages_per_seq, int64_t num_splits, size_t* bytes);
int pad_paged_attention_decode_weights(const void* q, const void* k_cache, const void* v_cache,
                                       const int32_t* block_table, const int32_t* seq_lens, void* out,
                                       float* weights, int32_t* slot_positions, const int32_t* total_lens,
                                       int64_t num_new, int64_t batch, int64_t num_q_heads, int64_t num_kv_heads,
                                       int64_t head_dim, int64_t num_pages, int64_t page_size,
                                       int64_t max_pages_per_seq, const int64_t* q_strides, const int64_t* k_strides,
                                       const int64_t* v_strides, int64_t block_table_stride,
                                       const int64_t* out_strides, const int64_t* weight_strides,
                                       const int64_t* position_strides, float scale, int64_t num_splits,
                                       void* workspace, size_t workspace_bytes, void* stream, int32_t* error_flags);
int pad_paged_attention_decode_weights_by_seq(
    const void* q, const void* k_cache, const void* v_cache, const int32_t* block_table, const int32_t* seq_lens,
    void* out, float* weights, int32_t* slot_positions, const int32_t* total_lens, const int32_t* num_new,
    int64_t batch, int64_t num_q_heads, int64_t num_kv_heads, int64_t head_dim, int64_t num_pages, int64_t page_size,
    int64_t max_pages_per_seq, const int64_t* q_strides, const int64_t* k_strides, const int64_t* v_strides,
    int64_t block_table_stride, const int64_t* out_strides, const int64_t* weight_strides,
    const int64_t* position_strides, float scale, int64_t num_splits, void* workspace, size_t workspace_bytes,
    void* stream, int32_t* error_flags);
int pad_evict_max_moves(int64_t budget, int64_t page_size, int64_t max_pages_per_seq, int64_t* max_moves);
int pad_paged_kv_evict_plan(const float* weights, const int32_t* slot_positions, const int32_t* block_table,
                            const int32_t* seq_lens, const int32_t* total_lens, int32_t* src, int32_t* dst,
                            int32_t* counts, int32_t* new_lens, int64_t batch, int64_t num_kv_heads,
                            int64_t num_pages, int64_t page_size, int64_t max_pages_per_seq, int64_t budget,
                            int64_t recent, const int64_t* weight_strides, const int64_t* position_strides,
                            int64_t block_table_stride, void* stream, int32_t* error_flags);
int pad_paged_kv_move(int64_t num_caches, void* const* caches, const int64_t* row_bytes, const int64_t* cache_strides,
                      const int32_t* block_table, const int32_t* src, const int32_t* dst, const int32_t* counts,
                      float* weights, int32_t* slot_positions, int64_t batch, int64_t num_kv_heads, int64_t num_pages,
                      int64_t page_size, int64_t max_pages_per_seq, int64_t max_moves, const int64_t* weight_strides,
                      const int64_t* position_strides, int64_t block_table_stride, void* stream,
                      int32_t* error_flags);

#ifdef __cplusplus
}
#endif

#endif /* PAD_B200_H_ */
