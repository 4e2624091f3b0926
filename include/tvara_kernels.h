/*
 * tvara_kernels -- kernel-level C ABI of the B200 engine (device pointers).
 *
 * These expose single hot-path kernels without a model handle, for callers
 * that manage their own device memory (and for the standalone GEMV and
 * attention benchmarks).  Pointers marked "device" are CUDA device memory of
 * the current device; `stream` is a cudaStream_t (NULL = legacy default).
 * Every function returns 0 on success and -1 on failure, with the message in
 * tvara_last_error() (include/tvara_capi.h).  Launches are asynchronous.
 */
#ifndef TVARA_KERNELS_H
#define TVARA_KERNELS_H
#include <stddef.h>
#include <stdint.h>

#include "tvara_capi.h"

#ifdef __cplusplus
extern "C" {
#endif

/* GGUF storage types (reference core/include/tvara/gguf.hpp:152-170). */
enum { TVARA_F32 = 0, TVARA_F16 = 1, TVARA_Q4_0 = 2, TVARA_Q8_0 = 8, TVARA_Q4_K = 12 };

/* Replaces quant::dequantize_q8_0 / q4_0 / q4_k and half_to_float
 * (core/include/tvara/quant.hpp:14-84): `blocks` GGUF blocks (device) ->
 * F32 (device), bit-identical to the reference. */
TVARA_API int tvara_dequantize(int type, const void* blocks, size_t nblocks, float* out, void* stream);

/* Bytes of the engine's packed layout for a [rows][cols] matrix: the codes of
 * every row (16-byte aligned rows), then the block headers, then one signed
 * byte per row (the power-of-two scale of the tensor-core path), each part at
 * a 256-byte aligned offset.  Q4_K rows (width a multiple of 256) are
 * followed by the side arrays the tensor-core path reads
 * beside the packed codes (sub-block scales, block scales, the split minima:
 * about 0.16 bytes per weight). */
TVARA_API size_t tvara_packed_bytes(int type, size_t rows, size_t cols);
/* GGUF rows (device) -> engine layout (device, tvara_packed_bytes long). */
TVARA_API int tvara_pack(int type, const void* gguf_rows, size_t rows, size_t cols, void* packed, void* stream);

/* Logit post-processing on the device (the sampler of
 * python/tvara/native.py:301-336 up to its random draw, for many rows):
 * logits F32 [rows][vocab] (device); the token history of row r is
 * history[history_offsets[r] .. history_offsets[r+1]) (history device,
 * offsets host, at most 16384 tokens a row); per-row repetition / frequency /
 * presence (host, NULL = 1, 0, 0); allowed (device [rows][ceil(vocab/32)]
 * bitmask, NULL = all).  Outputs on the device: argmax [rows] of the
 * adjusted, masked float64 logits, status [rows] (bit 1: non-finite model
 * logits, 2: non-finite adjusted logits, 4: no allowed token), and the
 * top_k (<= 64) largest values with their ids [rows][top_k] (value
 * descending, ties by index).  `workspace` of tvara_sample_workspace bytes. */
TVARA_API size_t tvara_sample_workspace(size_t rows, size_t max_history);
TVARA_API int tvara_sample_logits(const float* logits, size_t rows, size_t vocab, const int32_t* history,
                                  const uint64_t* history_offsets, const double* repetition, const double* frequency,
                                  const double* presence, const uint32_t* allowed, uint32_t top_k, uint32_t* argmax,
                                  int32_t* status, double* top_values, uint32_t* top_ids, void* workspace,
                                  size_t workspace_bytes, void* stream);

/* The int8 KV encode of TVARA_KV_I8 pools (python/tvara/quantized_kv.py:
 * 21-30, QuantizedKV.encode): rows F32 [n][dim] (device) -> codes int8
 * [n][dim] and scales F32 [n] (device).  A non-finite row fails with
 * "Nonfinite KV input" (the call synchronises the stream to report it). */
TVARA_API int tvara_kv_quantize(const float* rows, size_t n, size_t dim, int8_t* codes, float* scales, void* stream);

/* Device scratch tvara_quant_matmul needs for `tokens` rows of width `cols`
 * (0 when the call runs on the CUDA-core path, at most 4 tokens). */
TVARA_API size_t tvara_quant_matmul_workspace(size_t cols, size_t tokens);
/* Replaces quant::matvec_f32 over dequantised weights / Matrix::multiply and
 * prefill_reference (quant.hpp:163-196, prefill.hpp:12-18):
 * y[t][r] = sum_k W[r][k] * x[t][k] for t < tokens, W packed (device), x and y
 * F32 row-major (device).  Up to 4 tokens: CUDA-core GEMV with the weights
 * dequantised in registers.  More: tcgen05 tensor cores on an exact hi+lo
 * FP16 split of both operands (F32 accumulation); needs `workspace`, and x
 * 16-byte aligned (cols is a multiple of 32 there). */
TVARA_API int tvara_quant_matmul(int type, const void* packed, size_t rows, size_t cols, const float* x,
                                 size_t tokens, float* y, void* workspace, size_t workspace_bytes, void* stream);

/* Paged GQA attention, replacing fused_paged_attention /
 * fused_prompt_attention (core/include/tvara/attention.hpp:57-89) for many
 * query rows at once.  Query row i attends to positions [0, visible[i]) of its
 * block list tables[table_offset[i] ..]; query head h reads KV head
 * h / (heads / kv_heads).  Pool layout (elements of kv_dtype): block b, layer
 * l, kind (0 K, 1 V), KV head g, slot s, element e at
 *   ((((b*layers + l)*2 + kind)*kv_heads + g)*block_tokens + s)*head_dim + e. */
typedef struct tvara_attention_args {
    uint32_t struct_size;       /* sizeof(tvara_attention_args) */
    uint32_t kv_dtype;          /* TVARA_KV_F32, TVARA_KV_F16 or TVARA_KV_I8 (needs kv_scales) */
    uint32_t heads, kv_heads, head_dim, block_tokens;
    uint32_t layers, layer;
    size_t max_blocks;
    size_t n_queries;
    const float* q;             /* device [n_queries][heads*head_dim] */
    float* out;                 /* device [n_queries][heads*head_dim] */
    const void* pool;           /* device KV pool */
    const int32_t* tables;      /* host: concatenated block ids */
    size_t tables_len;
    const uint32_t* table_offset; /* host [n_queries] */
    const uint32_t* visible;      /* host [n_queries], each >= 1 */
    /* TVARA_KV_I8: device F32 scale of each pool row (element offset / head_dim);
     * callers of the shorter struct (struct_size up to `visible`) get F32/F16 only */
    const float* kv_scales;
} tvara_attention_args;

/* Device scratch (bytes) tvara_paged_attention needs for these arguments;
 * 0 with an error for invalid arguments, including a block id outside
 * [0, max_blocks) in any block a query reads. */
TVARA_API size_t tvara_paged_attention_workspace(const tvara_attention_args* args);
/* Runs the attention; workspace is device memory of at least the size above.
 * The call uploads the block tables and work list from host memory and, after
 * the kernels, reads their error word back, so it returns only when the
 * attention has finished on `stream`; a device-side error (a copy wait that
 * timed out) returns -1 with its text.  Not capturable into a CUDA graph: a
 * capturing stream is refused with an error before anything is enqueued. */
TVARA_API int tvara_paged_attention(const tvara_attention_args* args, void* workspace, size_t workspace_bytes,
                                    void* stream);

/* No counterpart in the reference (its attention runs on the CPU).  The same
 * attention as tvara_paged_attention, with its scratch in a fixed area inside
 * this library (tvara_paged_attention_noalloc_max() bytes per device, 16 MiB)
 * instead of caller memory, for callers that cannot allocate device memory at
 * the call: FFI hosts with no device allocator, code whose device memory
 * belongs to another framework's allocator, code that must not pay
 * cudaMalloc's device-wide synchronisation.  It allocates nothing.  Arguments
 * needing more scratch than the maximum (tvara_paged_attention_workspace) are
 * rejected with an error and nothing is launched.  The first call on a device,
 * with that device current, resolves the scratch address.  Synchronous on
 * `stream` and not capturable, as tvara_paged_attention; device-side errors
 * are returned the same way.  One scratch per device: calls overlapping on one
 * device (other streams or threads) race and must be serialised by the
 * caller. */
TVARA_API size_t tvara_paged_attention_noalloc_max(void);
TVARA_API int tvara_paged_attention_noalloc(const tvara_attention_args* args, void* stream);

/* ---- drafted-token trees over the paged KV cache ------------------------
 *
 * The reference verifies one chain of drafted tokens at a time (a
 * tvara_sequence_decode_batch, then tvara_sequence_truncate;
 * python/tvara/speculative.py:255-295).  These three calls verify a *tree* of
 * drafted tokens per sequence for a batch of sequences, with every length,
 * table and choice on the device: nothing is copied to or from the host, the
 * launches are asynchronous on `stream`, and all three can be captured into a
 * CUDA graph.  A step is
 *   tvara_tree_plan       blocks, slots, positions and masks of the drafts,
 *   (per layer)           the drafts' K and V written to their slots, then
 *   tvara_tree_attention  every draft over its sequence's cache and ancestors,
 *   tvara_tree_commit     the walk along the model's choices; accepted rows
 *                         move to where the sequence continues.
 *
 * Shared conventions.  Sequence s has lengths[s] cached positions and drafts
 * the rows [cu_nodes[s], cu_nodes[s+1]) of the flat row arrays, its nodes
 * (none is allowed); cu_nodes has n_seq + 1 entries, the first 0.  Node i's
 * parent is a node of the same sequence with a smaller index, or -1 for a
 * child of the last cached position.  The row arrays have room for `capacity`
 * rows; rows from cu_nodes[n_seq] on are neither read nor written.  A slot is
 * block * block_tokens + offset in the pool layout described above.  Table
 * row s starts at tables + s * table_stride.  At most 8192 sequences and 1024
 * nodes a sequence (max_nodes, the width the ancestor masks are laid out for:
 * ceil(max_nodes / 64) words a row).
 *
 * Arrays are aligned to their types, the workspace to 16 bytes.  Heads of at
 * most 128 values, with rows of q, out and pool that are multiples of 16 bytes
 * at 16-byte addresses, run on the tensor cores; others are much slower.
 *
 * What the host can check is refused as by the calls above.  What only the
 * device sees sets bits of *status (device, one word, never cleared by these
 * calls: zero it once and look when convenient), and nothing outside the
 * caller's arrays is touched. */
enum {
    TVARA_TREE_BAD_BLOCK = 1,   /* a block id or slot outside the pool; its row is not read or written (in the
                                   attention it counts as masked) */
    TVARA_TREE_BAD_LENGTHS = 2, /* cu_nodes that are negative, decrease or do not begin with 0, more rows than
                                   capacity, more nodes than max_nodes, a negative length, a sequence longer than
                                   its table row (with or without rows of its own), a count of free blocks outside
                                   [0, free_capacity], or held blocks that are fewer than the cached positions need:
                                   the plan writes nothing, the other calls skip the sequence */
    TVARA_TREE_NO_BLOCKS = 4,   /* the plan needs more blocks than are free: it writes nothing */
    TVARA_TREE_BAD_PARENT = 8,  /* a parent that is not an earlier node: the plan treats the node as a root, the
                                   commit never accepts it */
    TVARA_TREE_TIMEOUT = 16     /* a bounded wait inside the attention ran out: its output is incomplete */
};

/* Block tables, slot maps, positions and ancestor masks of a step from the
 * request lengths (for trees, and with parents NULL for prompt chunks or
 * plain appends, where a sequence's rows are consecutive positions).
 * Sequence s holds held[s] blocks in its table row.  If its lengths[s] + n
 * positions need more, blocks are taken from the end of the free list,
 * free_blocks[*free_count - 1] first, in sequence order, and appended to the
 * row; row i gets the slot of position lengths[s] + i.  positions[i] is
 * lengths[s] + depth of node i (roots have depth 0) and bit j of row i of
 * ancestors says that node j is node i or one of its ancestors.  held_out and
 * free_left may be held and free_count themselves (a second small launch then
 * writes them); no output may overlap another array otherwise.  The free list
 * is only read, its first *free_left entries stay free. */
typedef struct tvara_tree_plan_args {
    uint32_t struct_size;         /* sizeof(tvara_tree_plan_args) */
    uint32_t block_tokens;
    size_t n_seq, capacity, max_nodes, max_blocks, table_stride, free_capacity;
    const int32_t* lengths;       /* device [n_seq] */
    const int32_t* held;          /* device [n_seq] */
    const int32_t* cu_nodes;      /* device [n_seq + 1] */
    const int32_t* parents;       /* device [capacity], or NULL: rows are consecutive positions, any number of
                                     them (max_nodes is not looked at) */
    const int32_t* free_blocks;   /* device [free_capacity]; may be NULL if free_capacity is 0 */
    const int32_t* free_count;    /* device, one entry */
    int32_t* tables;              /* device [n_seq][table_stride], appended to */
    int64_t* slots;               /* out, device [capacity] */
    int32_t* positions;           /* out, device [capacity] */
    uint64_t* ancestors;          /* out, device [capacity][ceil(max_nodes / 64)]; with parents only (else NULL) */
    int32_t* held_out;            /* out, device [n_seq] */
    int32_t* free_left;           /* out, device, one entry */
    int32_t* status;              /* device, one word */
} tvara_tree_plan_args;
TVARA_API int tvara_tree_plan(const tvara_tree_plan_args* args, void* stream);

/* Attention of drafted tokens over a paged cache: row i of sequence s attends
 * to the cached positions [0, lengths[s]) through the table row of s and to
 * the nodes j of its sequence whose bit is set in row i of ancestors (any
 * mask; NULL: j <= i, a chain), their K and V at slots[cu_nodes[s] + j].
 * Scores are q.k / sqrt(head_dim), query head h reads KV head
 * h / (heads / kv_heads), arithmetic and outputs are F32 to within rounding
 * for every pool type (as tvara_paged_attention; F16 pools: weights down to
 * 2^-36 of a row's largest).  A row that attends to
 * nothing is zero; masked K and V may hold anything, NaN included.  Rows of
 * out may not meet rows of q (column slices of one buffer are fine), and out,
 * workspace and status no other array.  One workspace serves one call at a
 * time. */
typedef struct tvara_tree_attention_args {
    uint32_t struct_size;         /* sizeof(tvara_tree_attention_args) */
    uint32_t kv_dtype;            /* TVARA_KV_F32, TVARA_KV_F16 or TVARA_KV_I8 (needs kv_scales) */
    uint32_t heads, kv_heads, head_dim, block_tokens; /* head_dim 1..256 */
    uint32_t layers, layer;
    size_t n_seq, capacity, max_nodes, max_blocks, table_stride;
    size_t q_stride, out_stride;  /* elements from row to row, at least heads * head_dim */
    const float* q;               /* device [capacity][q_stride] */
    float* out;                   /* device [capacity][out_stride] */
    const void* pool;             /* device KV pool */
    const float* kv_scales;       /* TVARA_KV_I8: device row scales (element offset / head_dim) */
    const int32_t* tables;        /* device [n_seq][table_stride] */
    const int32_t* lengths;       /* device [n_seq] */
    const int32_t* cu_nodes;      /* device [n_seq + 1] */
    const int64_t* slots;         /* device [capacity] */
    const uint64_t* ancestors;    /* device [capacity][ceil(max_nodes / 64)], or NULL */
    int32_t* status;              /* device, one word */
} tvara_tree_attention_args;
/* Device scratch (bytes) for these sizes; 0 with an error for invalid ones. */
TVARA_API size_t tvara_tree_attention_workspace(const tvara_tree_attention_args* args);
TVARA_API int tvara_tree_attention(const tvara_tree_attention_args* args, void* workspace, size_t workspace_bytes,
                                   void* stream);

/* Acceptance and commit.  choices[i] is the token the model chose after node
 * i (its argmax, or a draw from its distribution: accepting the drafts that
 * equal such choices keeps the model's distribution), first[s] the one after
 * the last cached position.  The walk starts at the last cached position with
 * first[s]; it goes to the child whose token equals the choice (the lowest
 * index if several do) and on with that child's choice, until no child
 * matches.  With first NULL, node 0 is accepted as it is (the token already
 * emitted, its K and V not yet in the cache).  path[cu_nodes[s] + k] is the
 * k-th accepted node, -1 behind the last; accepted[s] counts them; next[s] is
 * the choice the walk ended with (0xFFFFFFFF when there is none), and may be
 * first itself; lengths_out[s] = lengths[s] + accepted[s], and may be lengths
 * itself (with next over first and a pool, a second small launch writes the
 * answers).  No output, the pool among them, may overlap another array
 * otherwise.
 * With a pool, the K and V rows of the k-th accepted node (every layer and KV
 * head, int8 scales too) are copied from its slot to dest[cu_nodes[s] + k];
 * dest NULL means slots: the drafts were written behind the cached positions,
 * and the accepted ones close up in place.  Other dest slots must not be
 * slots of drafted rows of this call, and no two rows may share one. */
typedef struct tvara_tree_commit_args {
    uint32_t struct_size;         /* sizeof(tvara_tree_commit_args) */
    uint32_t kv_dtype;            /* TVARA_KV_F32, TVARA_KV_F16 or TVARA_KV_I8 (needs kv_scales) */
    uint32_t kv_heads, head_dim, block_tokens, layers;
    size_t n_seq, capacity, max_nodes, max_blocks;
    const int32_t* lengths;       /* device [n_seq] */
    const int32_t* cu_nodes;      /* device [n_seq + 1] */
    const int32_t* parents;       /* device [capacity] */
    const uint32_t* tokens;       /* device [capacity] drafted token of each node */
    const uint32_t* choices;      /* device [capacity]; 0xFFFFFFFF matches nothing */
    const uint32_t* first;        /* device [n_seq], or NULL */
    const int64_t* slots;         /* device [capacity]; with a pool */
    const int64_t* dest;          /* device [capacity], or NULL */
    void* pool;                   /* device KV pool, or NULL: nothing moves */
    float* kv_scales;             /* TVARA_KV_I8: device row scales */
    int32_t* path;                /* out, device [capacity] */
    int32_t* accepted;            /* out, device [n_seq] */
    uint32_t* next;               /* out, device [n_seq] */
    int32_t* lengths_out;         /* out, device [n_seq] */
    int32_t* status;              /* device, one word */
} tvara_tree_commit_args;
TVARA_API int tvara_tree_commit(const tvara_tree_commit_args* args, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* TVARA_KERNELS_H */
