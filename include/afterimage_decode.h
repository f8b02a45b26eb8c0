/*
 * afterimage_decode.h -- C ABI of the MI355X (gfx950) lossless BF16 weight decoder.
 *
 * The decoder rebuilds BF16 tensors from Afterimage's compressed-store format:
 *   - a raw sign/mantissa byte per weight: (sign << 7) | mantissa
 *     (afterimage/runtime/compressed_store.py:78-88);
 *   - the exponent byte, canonical-Huffman coded in fixed-symbol-count chunks.
 *     Each chunk is its own MSB-first byte-aligned bitstream, located by
 *     chunk_offsets / chunk_nbytes (afterimage/runtime/huffman_chunked.py:151-207).
 *     The code is described by the stored flat LUT: sym_lut[2^max_bits] and
 *     len_lut[2^max_bits] (afterimage/runtime/huffman.py:128-150).
 *
 * The reference has no C layer; its decode API is Python
 * (afterimage/runtime/gpu_decode_v2.py, afterimage/runtime/compressed_store.py).
 * Each entry point below names the Python function whose work it replaces.
 * An FFI binding (ctypes) calls these with plain pointers and sizes.
 *
 * Conventions:
 *   - Every function returns AIMG_OK (0) or a positive AIMG_ERR_* code.
 *     aimg_last_error() returns the calling thread's last message.
 *   - Pointers named "device" are HIP device pointers. Streams are hipStream_t
 *     passed as void* (NULL = the null stream). Launches are asynchronous and
 *     ordered on the given stream. Nothing here synchronises the device.
 *   - No entry point allocates device memory. bf16 and exponent-byte decodes of
 *     chunks of 65536 symbols or more may split the launch's last chunks in two
 *     halves that hand over through a static 64 KiB device array (one per GPU,
 *     held until the process ends); launches that overlap on one GPU stay exact.
 *   - Functions are re-entrant.
 */
#ifndef AFTERIMAGE_DECODE_H
#define AFTERIMAGE_DECODE_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define AIMG_OK 0
#define AIMG_ERR_INVALID_ARGUMENT 1 /* bad size, null pointer, too many tensors */
#define AIMG_ERR_BAD_TABLE 2        /* LUT is not a prefix-code table with byte symbols */
#define AIMG_ERR_HIP 3              /* a HIP runtime call failed */
#define AIMG_ERR_UNSUPPORTED 4      /* valid request that this build does not serve */

/* Most tensors one aimg_decode_* call accepts (kernel-argument descriptors). */
#define AIMG_MAX_TENSORS 32

/* Library ABI version (bumped on any signature or table-layout change). */
int aimg_abi_version(void);

/* Message for the last non-OK status returned on this thread. */
const char* aimg_last_error(void);

/* ------------------------------------------------------------------------- */
/* Decode tables.                                                            */
/* Replaces prepare_decode_tables (afterimage/runtime/gpu_decode_v2.py:71-76), */
/* which copies sym_lut / len_lut to the device as two int32 tensors. Here    */
/* the stored LUT is turned on the host into one self-contained table blob:  */
/* a 4096-entry multi-symbol window table (up to 4 codewords per 12-bit      */
/* window) plus 16-entry escape blocks for codewords of 13..16 bits. The     */
/* caller copies the blob to device memory once per codebook and may share   */
/* it across every tensor with the same codebook.                            */
/* ------------------------------------------------------------------------- */

/* Size in bytes of the table blob for a LUT of 2^max_bits entries (1..16). */
int aimg_table_nbytes(int max_bits, size_t* nbytes);

/*
 * Build the table blob into host memory `out` (out_nbytes >= aimg_table_nbytes).
 * sym_lut: int32[2^max_bits], len_lut: int8[2^max_bits], as stored by
 * build_decode_lut (afterimage/runtime/huffman.py:128-150).
 * Fails with AIMG_ERR_BAD_TABLE when a symbol is outside 0..255 (the
 * reference asserts this, gpu_decode_v2.py:73-74), a length is outside
 * 0..max_bits, or an entry is not replicated over its whole prefix span.
 */
int aimg_build_table(const int32_t* sym_lut, const int8_t* len_lut, int max_bits,
                     void* out, size_t out_nbytes);

/* ------------------------------------------------------------------------- */
/* Decode.                                                                   */
/* ------------------------------------------------------------------------- */

/* One tensor's device-resident compressed form (a ChunkedEncoded plus its
 * sign/mantissa stream, huffman_chunked.py:135-148, compressed_store.py:28-42). */
typedef struct aimg_tensor {
    const uint8_t* packed;         /* device: chunk bitstreams, as stored       */
    const int32_t* chunk_offsets;  /* device: byte offset of each chunk         */
    const int32_t* chunk_nbytes;   /* device: byte length of each chunk         */
    const uint8_t* sign_mantissa;  /* device: n_symbols bytes (bf16 only)       */
    void* out;                     /* device: uint16 bf16 bits, or uint8        */
    const void* table;             /* device: blob from aimg_build_table        */
    void* index;                   /* device: segment index, or NULL (below)    */
    int64_t index_nbytes;          /* bytes at `index`                          */
    int64_t packed_nbytes;         /* bytes readable at `packed`                */
    int64_t n_symbols;             /* elements to write (below 2^31)            */
    int32_t chunk_size;            /* symbols per chunk                         */
    int32_t n_chunks;              /* chunks described by offsets / nbytes      */
} aimg_tensor;

/*
 * Decode n_tensors tensors to BF16 in one launch: the Huffman decode of
 * decode_gpu_v2 (gpu_decode_v2.py:79-117) fused with _recombine
 * (compressed_store.py:94-114). out[i] = ((sm[i] & 0x80) << 8) | (exp[i] << 7)
 * | (sm[i] & 0x7F) for i < n_symbols, where n_symbols <= n_chunks*chunk_size.
 * Replaces the body of decompress_layer_gpu (compressed_store.py:186-240) for
 * device-resident inputs; one call covers a whole decoder block of tensors.
 * A tensor of 2^31 or more symbols fails with AIMG_ERR_UNSUPPORTED.
 */
int aimg_decode_bf16(const aimg_tensor* tensors, int n_tensors, void* stream);

/*
 * Decode n_tensors exponent streams to uint8 symbols: decode_gpu_v2
 * (gpu_decode_v2.py:79-117). sign_mantissa is ignored. Positions past a
 * chunk's coded symbols decode as if the chunk's bytes were followed by zero
 * bits, as the bounded CPU reader does (huffman_chunked.py:230-235).
 */
int aimg_decode_u8(const aimg_tensor* tensors, int n_tensors, void* stream);

/*
 * Fused decode -> GEMV: y[b][r] += sum_c W[r][c] * x[b][c] in fp32 for the
 * rows x cols row-major bf16 matrix W held compressed in *t
 * (t->n_symbols == rows * cols) and b < batch (1..4). W is never written;
 * t->out is ignored. x: bf16 [batch][cols] (device). y: float [batch][rows]
 * (device), which the caller zeroes first: the kernel adds to it with
 * atomics, so the order of the fp32 additions is not fixed. The reference
 * computes this as decompress_rows_gpu (compressed_store.py:254-303) followed
 * by a matmul in its chunked lm_head (streaming_engine.py:2271-2335).
 * cols % 8 == 0 with a 16-byte-aligned x takes the vector path; other
 * shapes are correct but add every product with its own atomic.
 */
int aimg_decode_gemv_bf16(const aimg_tensor* t, int64_t rows, int64_t cols, const void* x,
                          int batch, float* y, void* stream);

/*
 * Fused decode -> GEMM for 1..16 rows of x: y[t][r] += sum_c W[r][c] * x[t][c]
 * in fp32 for t < n_x, W as in aimg_decode_gemv_bf16 (never written; t->out
 * ignored), on the matrix cores (bf16 products, fp32 sums). x: bf16
 * [n_x][cols], 16-byte aligned (device); y: float [n_x][rows] (device),
 * zeroed by the caller and added to with atomics (the order of the fp32
 * additions is not fixed). This is the chunked lm_head's speculative-verify
 * forward (streaming_engine.py:2307-2332, called with step_k + 1 positions
 * at :2554-2556: decompress_rows_gpu per row block, then F.linear) in one
 * launch that writes no weights. Needs cols % 8 == 0, chunk_size a multiple
 * of 8 in 1024 .. 2^24 and n_x * cols * 2 < 2^32; other shapes fail with
 * AIMG_ERR_UNSUPPORTED (the caller then takes the blocked decode and GEMM).
 */
int aimg_decode_gemm_bf16(const aimg_tensor* t, int64_t rows, int64_t cols, const void* x,
                          int n_x, float* y, void* stream);

/*
 * aimg_decode_gemm_bf16 with device scratch memory: the exponent bytes of up
 * to 16 rows of W a workgroup (and what one round of it decodes beyond them)
 * pass through `workspace`, so that x is read once per 16 rows of W; up to 3
 * times faster. zero_y: y is set, not added to. aimg_gemm_workspace_nbytes
 * gives the bytes it takes on the current device for n_x rows of x (of *t,
 * n_symbols and chunk_size are read; 170 MB for a large matrix of 17408
 * columns, 66 MB of 5120, at most 512 MiB and 16 packed rows of x), or 0 where
 * the call without a workspace is as fast or no workspace serves the shape
 * (n_x 0: the bytes for up to 16 rows, whichever is faster). A null,
 * misaligned (16 bytes) or smaller workspace fails with
 * AIMG_ERR_INVALID_ARGUMENT. Its contents need no initialisation and mean
 * nothing afterwards; launches that may overlap need a workspace each.
 */
int aimg_gemm_workspace_nbytes(const aimg_tensor* t, int64_t rows, int64_t cols, int n_x,
                               size_t* nbytes);
int aimg_decode_gemm_bf16_ws(const aimg_tensor* t, int64_t rows, int64_t cols, const void* x,
                             int n_x, float* y, int zero_y, void* workspace,
                             size_t workspace_nbytes, void* stream);

/*
 * out[i] = ((sm[i] & 0x80) << 8) | (exponent[i] << 7) | (sm[i] & 0x7F) for
 * i < n, on the GPU (all three pointers device memory; out is uint16 bf16
 * bits). Replaces recombine_exponent_and_sign_mantissa and _recombine
 * (afterimage/runtime/compressed_store.py:94-130) for device tensors: one
 * kernel instead of a chain of elementwise torch kernels. 16-byte aligned
 * pointers take the vector path; any alignment is correct.
 */
int aimg_recombine_bf16(const uint8_t* exponent, const uint8_t* sign_mantissa, void* out,
                        int64_t n, void* stream);

/* ------------------------------------------------------------------------- */
/* Segment index (optional; no counterpart in the reference, whose decoder    */
/* runs one chunk per lane and needs none).                                  */
/* The decode kernels split each chunk into segments of a fixed number of     */
/* bits, one per thread, and find where each segment's first codeword starts */
/* by decoding ahead of it and checking agreement with the thread before.    */
/* A segment index records, once per resident tensor, each segment's first   */
/* codeword boundary, its chunk and where its symbols go in a round of 512   */
/* segments (4 bytes per segment of 168 bits for bf16 exponent codes: about  */
/* 4.7% of a compressed layer). A decode given the index runs in rounds of   */
/* 512 segments across chunk boundaries with no look-ahead, agreement check, */
/* scan or compaction, and writes each segment's symbols straight to their   */
/* place. It is used for tensors whose chunks hold 1024 symbols or more and  */
/* that take the vector path (16-byte aligned output, chunk_size % 8 == 0);  */
/* other tensors decode without it. Decoding without an index (index ==      */
/* NULL) gives the same result.                                              */
/* An index describes one tensor's packed bytes, chunk offsets and lengths   */
/* and table: the decoders use it only with the table it was built with      */
/* (checked by checksum) and otherwise ignore it; with other packed bytes or */
/* offsets than it was built from the output is unspecified (memory stays    */
/* in bounds).                                                               */
/* ------------------------------------------------------------------------- */

/*
 * Bytes of the segment index for a tensor of packed_nbytes packed bytes in
 * n_chunks chunks whose chunks lie back to back in `packed` (as the
 * encoder writes them, huffman_chunked.py:204-205), for the table whose
 * host blob (from aimg_build_table) is host_table.
 */
int aimg_index_nbytes(const void* host_table, int64_t packed_nbytes, int32_t n_chunks,
                      size_t* nbytes);

/*
 * Build the segment index of each tensor into its `index` (device memory of
 * index_nbytes >= aimg_index_nbytes bytes; tensors with a NULL index are
 * skipped; index must be 16-byte aligned). Four launches on `stream`
 * (segment numbering, the raw entries, a walk that fixes each chunk's
 * counts at its real end and writes the round starts, then each round's
 * chunk numbers and output places); the decoders that follow on the stream
 * use the index. When the chunks' segments do not fit index_nbytes (chunks
 * not back to back) or a chunk does not hold its symbols, the index is
 * marked unusable and decoders ignore it. Other fields as for
 * aimg_decode_u8.
 */
int aimg_build_index(const aimg_tensor* tensors, int n_tensors, void* stream);

/* ------------------------------------------------------------------------- */
/* Host decode (CPU threads).                                                */
/* Replaces the reference's CPU path: _decode_exponent with device "cpu"     */
/* (afterimage/runtime/compressed_store.py:161-183) over decode_chunks_numba */
/* (afterimage/runtime/cpu_decode.py:67-113), and _recombine on the CPU.     */
/* Every pointer of the aimg_tensor descriptors is HOST memory here, and     */
/* `table` is the host blob of aimg_build_table. The result equals the GPU   */
/* entry points' on every input. n_threads <= 0 uses every hardware thread.  */
/* The call returns when the work is done.                                   */
/* ------------------------------------------------------------------------- */

/* BF16 rebuild, as aimg_decode_bf16 (no size limit on n_symbols). */
int aimg_cpu_decode_bf16(const aimg_tensor* tensors, int n_tensors, int n_threads);

/* Exponent bytes only, as aimg_decode_u8. */
int aimg_cpu_decode_u8(const aimg_tensor* tensors, int n_tensors, int n_threads);

/* Host recombine, as aimg_recombine_bf16 (one thread). */
int aimg_cpu_recombine_bf16(const uint8_t* exponent, const uint8_t* sign_mantissa, void* out,
                            int64_t n);

/* ------------------------------------------------------------------------- */
/* Encoder support (host).                                                   */
/* ------------------------------------------------------------------------- */

/*
 * Pack symbols[0..n) chunk by chunk into MSB-first byte-aligned bitstreams:
 * the packer of encode_chunked (huffman_chunked.py:41-78, :101-109).
 * code_of[256] / len_of[256] give each symbol's canonical code and length
 * (lengths 1..16; symbols that occur must have len_of > 0).
 * Writes chunk_nbytes[ceil(n/chunk_size)] and the packed bytes into out
 * (capacity out_cap); *total receives the packed byte count (no slack tail).
 */
int aimg_pack_chunked(const uint8_t* symbols, int64_t n, const uint32_t* code_of,
                      const uint8_t* len_of, int32_t chunk_size, uint8_t* out,
                      int64_t out_cap, int32_t* chunk_nbytes, int64_t* total);

/* ------------------------------------------------------------------------- */
/* Attention.                                                                */
/* The products between the projections of a decoder layer and its output    */
/* projection (the reference leaves them to the model's own forward pass).   */
/* Elements are bf16 or fp16; scores, softmax statistics and sums are fp32.  */
/* ------------------------------------------------------------------------- */

#define AIMG_BF16 0
#define AIMG_FP16 1

/* Rows of heads: element (row, head, x) is data[row * row_stride + head *
 * head_stride + x], strides in elements. dim is a multiple of 8 up to 256.
 * Inputs need 16-byte aligned data and strides of whole 16 bytes, outputs 8.
 * Rows of keys and values are at most 2^24 elements apart. */
typedef struct aimg_heads {
    void* data;          /* device                                    */
    int64_t n_rows;
    int64_t row_stride;
    int64_t head_stride;
    int32_t heads;
    int32_t dim;
} aimg_heads;

/*
 * Causal attention of n_seqs packed prompts: rows q_offsets[b] ..
 * q_offsets[b+1] - 1 of q (int32[n_seqs + 1], device) attend over rows
 * k_offsets[b] .. of k and v. The last query row sees every key, the one
 * before it all but the last, and so on (a prompt that continues a context
 * has more keys than rows); a row that sees no key gives zeros. Head h of q
 * reads head h / (q->heads / k->heads) of k and v, which have fewer than
 * 2^31 - 64 rows.
 * out has q's shape; rows outside every sequence are not written. lse: NULL,
 * or float[q->n_rows][q->heads] (device) for log(sum(exp(scale * q.k))), -inf
 * for a row that sees no key. scale > 0. Offsets outside the rows are bounded
 * to them; keys that a row does not see never reach it, whatever they hold.
 * aimg_prompt_workspace_nbytes gives the device scratch memory a call of these
 * sizes needs (16-byte aligned; 0, for most: none): few rows over many keys are
 * split along the keys and joined in order. Results do not vary between calls.
 */
int aimg_prompt_workspace_nbytes(int64_t n_rows, int64_t n_keys, int heads, int kv_heads, int dim, int n_seqs,
                                 size_t* nbytes);
int aimg_prompt_attention(const aimg_heads* q, const aimg_heads* k, const aimg_heads* v, const aimg_heads* out,
                          const int32_t* q_offsets, const int32_t* k_offsets, int n_seqs, int type,
                          float scale, float* lse, void* workspace, size_t workspace_nbytes, void* stream);

/* The keys and values of one layer in a paged cache: position j of sequence
 * slot s is row j % page_size of page page_table[s * table_stride + j /
 * page_size]; element x of head h there is k[page * page_stride + row *
 * slot_stride + h * head_stride + x], and v's likewise (strides in elements,
 * whole 16 bytes, the same for both, slot_stride at most 2^24). lengths[s]
 * positions are held before the drafted ones. Page numbers outside
 * 0..n_pages-1 read page 0. */
typedef struct aimg_pages {
    void* k;                      /* device */
    void* v;                      /* device */
    const int32_t* page_table;    /* device: [max_seqs][table_stride] */
    const int32_t* lengths;       /* device: [max_seqs] */
    int64_t page_stride;
    int64_t slot_stride;
    int64_t head_stride;
    int32_t table_stride;
    int32_t n_pages;
    int32_t page_size;
    int32_t kv_heads;
    int32_t dim;
    int32_t max_seqs;
    int32_t max_pages;            /* of a sequence (<= table_stride) */
} aimg_pages;

/*
 * Attention of drafted tokens over a paged cache: the verification forward
 * pass of a drafted tree, and plain decoding with one token a sequence. Rows
 * draft_offsets[b] .. draft_offsets[b+1] - 1 of q (int32[n_seqs + 1], device;
 * at most max_drafts rows each) are the drafted tokens of slot seqs[b]. Their
 * keys and values are in the cache at positions lengths[slot], lengths[slot] +
 * 1, ... Token t sees the positions before those, and drafted token j where
 * bit j % 64 of masks[row * mask_words + j / 64] is set (masks NULL: the
 * tokens up to itself). A row that sees nothing gives zeros; so do the rows of
 * a slot outside 0..max_seqs-1.
 * max_context: the longest lengths[slot] the caller expects; it only decides
 * how the work is split. aimg_tree_workspace_nbytes gives the device scratch
 * memory a call needs (16-byte aligned; 0: none), its contents mean nothing
 * before or after. Parts are joined in their order: results do not vary
 * between calls. lse: NULL or float[q->n_rows][q->heads], as above.
 */
int aimg_tree_workspace_nbytes(int64_t n_rows, int heads, int kv_heads, int dim, int n_seqs, int max_drafts,
                               int64_t max_context, size_t* nbytes);
int aimg_tree_attention(const aimg_heads* q, const aimg_pages* pages, const aimg_heads* out, const int32_t* seqs,
                        const int32_t* draft_offsets, int n_seqs, const int64_t* masks, int mask_words, int max_drafts,
                        int64_t max_context, int type, float scale, float* lse, void* workspace,
                        size_t workspace_nbytes, void* stream);

/* The factors of pages of 8-bit elements (see the cache below): positions
 * 16 i .. 16 i + 15 of head h of a page share k[page * page_stride + h *
 * head_stride + i], and v's likewise (strides in floats, the same for both). */
typedef struct aimg_page_scales {
    const float* k;       /* device */
    const float* v;
    int64_t page_stride;
    int64_t head_stride;
} aimg_page_scales;

/*
 * aimg_tree_attention over a cache in 8 bits: pages of e4m3 elements (strides
 * in elements, whole 16 bytes; dim and page_size multiples of 16), the factors
 * powers of two. q and out are bf16 or fp16 (type). Keys enter the first
 * product exactly; probabilities are rounded to bf16 for the second where q is
 * bf16, to a sum of two bf16 numbers (16 bits) where it is fp16.
 */
int aimg_tree8_workspace_nbytes(int64_t n_rows, int heads, int kv_heads, int dim, int n_seqs, int max_drafts,
                                int64_t max_context, size_t* nbytes);
int aimg_tree8_attention(const aimg_heads* q, const aimg_pages* pages, const aimg_page_scales* scales, const aimg_heads* out,
                         const int32_t* seqs, const int32_t* draft_offsets, int n_seqs, const int64_t* masks, int mask_words,
                         int max_drafts, int64_t max_context, int type, float scale, float* lse, void* workspace,
                         size_t workspace_nbytes, void* stream);

/*
 * masks[row * mask_words + w] for n_rows drafted tokens from their parents:
 * parents[row] is the index, within its sequence, of an earlier drafted token,
 * and any other number for a token that follows the context directly. The bits
 * are the token's own and its ancestors'.
 */
int aimg_tree_masks(const int32_t* parents, const int32_t* draft_offsets, int n_seqs, int64_t n_rows, int mask_words,
                    int64_t* masks, void* stream);

/* ------------------------------------------------------------------------- */
/* Pages of a key/value cache.                                               */
/* The pool holds every layer's keys and values, [n_layers][2][n_pages]      */
/* [kv_heads][page_size][dim] in elements of two bytes. Slot s of max_seqs   */
/* holds held[s] pages, page_table[s][0 .. held[s]-1], for lengths[s]        */
/* positions and those to come; refs[p] sequences hold page p, none a free   */
/* one. All of it is device memory and every call works there, on `stream`.  */
/* Positions at or past a length lie in pages that only their sequence holds: */
/* fork shares full pages alone. A call names a slot once.                   */
/* What a call finds wrong on the GPU it leaves undone and says in *status   */
/* (bits, or-ed in): 1 no free pages (nothing was reserved or forked), 2 a   */
/* sequence's row of the table or its pages end before the positions asked   */
/* for, 4 a slot, page, source or number of rows that does not exist. (Rows  */
/* of a table entry that is no page are neither copied nor moved; the rest   */
/* of such a sequence is.)                                                   */
/* ------------------------------------------------------------------------- */

#define AIMG_CACHE_NO_PAGES 1
#define AIMG_CACHE_ROW_FULL 2
#define AIMG_CACHE_BAD_INDEX 4

typedef struct aimg_cache {
    void* pool;           /* 16-byte aligned; dim a multiple of 8 */
    int32_t* page_table;  /* [max_seqs][max_pages] */
    int32_t* lengths;     /* [max_seqs] */
    int32_t* held;        /* [max_seqs] */
    int32_t* refs;        /* [n_pages] */
    int32_t* status;      /* [1] */
    int32_t n_layers;
    int32_t n_pages;
    int32_t kv_heads;
    int32_t page_size;
    int32_t dim;
    int32_t max_seqs;
    int32_t max_pages;
} aimg_cache;

/* Writes rows offsets[b] .. offsets[b+1] - 1 of k and v into slot seqs[b]'s
 * pages of one layer, from its length on. Lengths do not change. */
int aimg_cache_append(const aimg_cache* cache, int layer, const aimg_heads* k, const aimg_heads* v, const int32_t* seqs,
                      const int32_t* offsets, int n_seqs, void* stream);

/*
 * A cache in 8 bits: the pool holds e4m3 elements (one byte: 4 bits of
 * exponent, 3 of mantissa, no infinity), dim a multiple of 16 up to 256,
 * page_size one of 16, and scales[n_layers][2][n_pages][kv_heads][page_size /
 * 16] (floats, device) one factor for each 16 positions of a page and head: an
 * element stands for its value times the factor. Factors are powers of two from
 * 2^-100 to 2^119: the smallest that brings the largest of the block's rows to
 * at most 448 (past that at the highest one, elements are held as 448 of it).
 * Infinities and NaN are held as NaN and do not count. A block that a call adds
 * rows to is formed anew from what its rows below the length stand for and
 * those, rounded to nearest even: where its factor rises, elements of earlier
 * rows below 2^-6 of it change by up to 2^-10 of it, and stay so if the rows
 * are drafts that no commit accepts. Where `scales` is an argument of a call for
 * either, NULL means a cache in 16 bits.
 */

/* Tables of a rotation: element i < half of a position's row turns, with the
 * element it is paired with, by the angle whose cosine and sine are
 * cos[position * half + i] and sin[...]: (a, b) becomes (a c - b s, b c + a s).
 * Pairs are i and i + half, or 2 i and 2 i + 1 where interleaved is not 0; the
 * elements from 2 * half on stay. */
typedef struct aimg_rotary {
    const float* cos;     /* device: [n_positions][half] */
    const float* sin;
    int32_t n_positions;
    int32_t half;         /* 1 .. dim / 2 */
    int32_t interleaved;
} aimg_rotary;

/*
 * aimg_cache_append with the rotation of q and k on the way (rotary NULL:
 * none), into a cache in 16 bits or 8 (type: that of q, k and v; in 16 bits
 * the pool's too). Row r turns by positions[r] (int32, device), by its position in
 * the cache where positions is NULL; the turned q goes to q_out, which may be
 * q (q NULL: none). Products and sums are fp32, rounded once. A row whose
 * position the tables do not hold is left out and recorded (4); rows of no
 * sequence are left out. Rows, heads and 16-byte pieces as for aimg_heads'
 * inputs, q_out too; dim up to 256.
 */
int aimg_cache_append_rotated(const aimg_cache* cache, float* scales, int layer, const aimg_heads* q, const aimg_heads* k,
                              const aimg_heads* v, const aimg_heads* q_out, const int32_t* seqs, const int32_t* offsets,
                              int n_seqs, const aimg_rotary* rotary, const int32_t* positions, int type, void* stream);

/*
 * Rows offsets[b] .. offsets[b+1] - 1 of k and v (written, in 16 bits of the
 * given type, which is the pool's where that has 16) become positions starts[b]
 * .. (0 .. where starts is NULL) of slot seqs[b]. Positions past its length, in
 * pages it holds, are read too; rows of no sequence, or of positions that no
 * page holds (recorded), are left as they are.
 */
int aimg_cache_read(const aimg_cache* cache, float* scales, int layer, const int32_t* seqs, const int32_t* offsets,
                    const int32_t* starts, int n_seqs, const aimg_heads* k, const aimg_heads* v, int type, void* stream);

/* aimg_cache_fork, aimg_cache_commit and aimg_cache_compact of a cache in 8
 * bits, with the same workspaces. A block into which an accepted row moves is
 * formed anew; the others stay. */
int aimg_cache8_fork(const aimg_cache* cache, float* scales, const int32_t* src, const int32_t* dst, int n_seqs,
                     void* workspace, size_t workspace_nbytes, void* stream);
int aimg_cache8_commit(const aimg_cache* cache, float* scales, const int32_t* seqs, const int32_t* accepted, int max_accepted,
                       const int32_t* counts, int n_seqs, int32_t* new_lengths, void* stream);
int aimg_cache8_compact(const aimg_cache* cache, float* scales, int32_t* new_table, int32_t* new_refs, int32_t* used,
                        void* workspace, size_t workspace_nbytes, void* stream);

/* Adds offsets[b+1] - offsets[b] to slot seqs[b]'s length: the rows that every
 * layer has appended (a difference below 0 is an error, 4). */
int aimg_cache_advance(const aimg_cache* cache, const int32_t* seqs, const int32_t* offsets, int n_seqs, void* stream);

/* Pages for tokens[b] positions past slot seqs[b]'s length, for all sequences
 * or none: the lowest free pages, in the order of the call. At most 8192
 * sequences a call, here and below. */
int aimg_cache_reserve(const aimg_cache* cache, const int32_t* seqs, const int32_t* tokens, int n_seqs, void* stream);

/* Empties the slots: their references go, pages without any are free. */
int aimg_cache_release(const aimg_cache* cache, const int32_t* seqs, int n_seqs, void* stream);

/*
 * Slot dst[i] becomes a branch of slot src[i], whatever it held before, for
 * all pairs at once (a source may be another pair's branch; src[i] == dst[i]
 * stays as it is): it shares the source's full pages, and the rows of its last
 * one, in every layer, are copied to a free page, the lowest ones in the
 * order of the call. Pages that branches gave up are free after the call.
 * Nothing changes where free pages are too few. Pages reserved past the
 * source's length are not passed on.
 */
int aimg_cache_fork_workspace_nbytes(const aimg_cache* cache, int n_seqs, size_t* nbytes);
int aimg_cache_fork(const aimg_cache* cache, const int32_t* src, const int32_t* dst, int n_seqs, void* workspace,
                    size_t workspace_nbytes, void* stream);

/*
 * Keeps the accepted tokens of verified trees: rows lengths[slot] +
 * accepted[b * max_accepted + i] of every layer become rows lengths[slot] + i,
 * i < counts[b] <= max_accepted (a count outside 0..max_accepted is an error,
 * 4). Accepted indices rise (a path from the root, parents before children).
 * new_lengths[slot] = lengths[slot] + counts[b]; it may be cache->lengths, and
 * is written for the call's slots only.
 */
int aimg_cache_commit(const aimg_cache* cache, const int32_t* seqs, const int32_t* accepted, int max_accepted,
                      const int32_t* counts, int n_seqs, int32_t* new_lengths, void* stream);

/*
 * Moves pages so that the *used pages in use are 0 .. *used - 1: the i-th one
 * at or past *used goes to the i-th free one before it, in every layer.
 * new_table and new_refs (which may be the cache's own) get the page table and
 * the counts after the moves. The pages moved from keep their bytes.
 */
int aimg_cache_compact_workspace_nbytes(const aimg_cache* cache, size_t* nbytes);
int aimg_cache_compact(const aimg_cache* cache, int32_t* new_table, int32_t* new_refs, int32_t* used, void* workspace,
                       size_t workspace_nbytes, void* stream);

/* ------------------------------------------------------------------------- */
/* Tokens from logits.                                                       */
/* ------------------------------------------------------------------------- */

#define AIMG_FP32 2

/* A row's settings: its entry of an array (device), or the number below for
 * every row where the array is NULL. temperature: 0 (or less, or NaN) takes the
 * largest logit's first token. top_k: 0 (or less) for none. top_p: 1 (or more)
 * for none. min_p: 0 (or less) for none. */
typedef struct aimg_sampling {
    const float* temperatures;
    const int32_t* top_ks;
    const float* top_ps;
    const float* min_ps;
    double temperature;
    double top_p;
    double min_p;
    int32_t top_k;
} aimg_sampling;

/*
 * A token for each of n_rows (at most 2^21) rows of `vocab` logits (at most
 * 2^18), row_stride elements apart, of type bf16, fp16 or fp32. A row's tokens stand
 * in the order of falling logits, equal ones by rising index; with w = exp((x -
 * max x) / temperature) those are kept that are among the first top_k, in the
 * shortest prefix whose weights reach top_p times the first top_k's, and
 * weigh at least min_p; one at least. tokens[row] is the first whose weights,
 * summed along the order, pass uniforms[row] (in [0, 1); other numbers as the
 * nearest there) times those of all that are kept, and logprobs[row] (where not
 * NULL) the logarithm of its share of them: 0 at temperature 0. Logits of -inf or
 * NaN are no tokens; a row without any other gives -1 and -inf. Weights below
 * 2^-64 of the largest (at any temperature those of logits 2^128 below it) count
 * as nothing, the others are sums of 2^-26 of themselves, in integers and
 * doubles: results do not vary between calls. (A bf16 logit 2^16 times smaller
 * or larger in size than the largest, or an fp16 one 2^13 times, weighs besides
 * by up to 2^-24 (max x - x) / temperature of itself more or less.)
 * aimg_sample_workspace_nbytes gives the device scratch memory that a call of
 * these sizes needs for logits of any type (8-byte aligned; 0 for many rows or
 * few logits): few long rows are dealt out to several workgroups each.
 */
int aimg_sample_workspace_nbytes(int64_t n_rows, int vocab, size_t* nbytes);
int aimg_sample(const void* logits, int64_t n_rows, int64_t row_stride, int vocab, int type, const float* uniforms,
                const aimg_sampling* settings, int64_t* tokens, float* logprobs, void* workspace, size_t workspace_nbytes,
                void* stream);

#ifdef __cplusplus
}
#endif

#endif /* AFTERIMAGE_DECODE_H */
