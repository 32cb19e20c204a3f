/* Paged batch operators: a step of many requests behind one shared prefix.
 *
 * No counterpart in the reference, which serves one request at a time. A
 * server that batches translation requests behind a common prompt (the
 * template, an instruction, a document) keeps every layer's keys and values
 * in one pool of pages and runs three operators per step, all on device
 * buffers of the context's GPU and all asynchronous on one stream of it:
 *
 *   plamo_paged_plan       page tables and slot maps from the requests' row
 *                          counts (once per step);
 *   plamo_paged_store      per layer, between the QKV projection and
 *                          attention: normalises and rotates the query and
 *                          key heads, puts keys and values into their slots;
 *   plamo_paged_attention  per layer: every query over the shared prefix and
 *                          over its own request's rows. The prefix is read
 *                          once for up to 256 (row, head) pairs of the
 *                          requests that add few rows (BF16; FP32, and short
 *                          prefixes: for eight), and once for each of the
 *                          tiles of those that add many.
 *
 * Pool: [pages][2][64][kv_heads][128] elements of BF16 or FP32, 16-byte
 * aligned: a page holds 64 key rows, then 64 value rows, as the token loop's
 * own KV pages do (there FP32 and unrotated; here keys are stored rotated).
 * A slot is page * 64 + row in the page. The prefix's rows fill the pages
 * named by its own table, from row 0; a request's own rows fill the pages of
 * its table, from row 0 of its first page, whatever the prefix's length.
 *
 * A step adds rows to some requests: request r has the batch's rows
 * [starts[r], starts[r + 1]). Its own length after the step is lengths[r], so
 * its i-th new row is own row lengths[r] - (starts[r+1] - starts[r]) + i, at
 * position prefix_rows + that. Rows of the batch from starts[requests] up are
 * padding (a step captured in a CUDA graph keeps its row count): they get
 * slot -1, are stored nowhere and come out of attention as zeros.
 *
 * Return convention, as plamo_cuda.h: 1 enqueued; 0 declined, nothing
 * enqueued (the reason is in plamo_cuda_info.note); -1 a launch failed.
 * What only the device can see is reported there: rows whose slot or position
 * lies outside its array are left out, a page outside the pool reads as rows
 * of zeros, nothing out of range is read or written, and `status` (a device
 * word) gets a PLAMO_PAGED_* bit; where it is NULL a word of the context does,
 * which plamo_paged_status reads. Buffers must stay valid until
 * the stream has run the call; calls with a workspace of their own may overlap
 * on different streams. Every call can be captured in a CUDA graph: none
 * allocates, waits or reads a length on the host.
 */
#ifndef PLAMO_PAGED_H
#define PLAMO_PAGED_H
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum { PLAMO_PAGED_ROWS = 64, PLAMO_PAGED_DIM = 128 };
enum { PLAMO_PAGED_BF16 = 0, PLAMO_PAGED_FP32 = 1 };

/* Status bits. The first four make a plan decline the step as a whole. */
enum {
    PLAMO_PAGED_NO_PAGES = 1,   /* plan: the free list does not hold the pages the step needs */
    PLAMO_PAGED_TABLE = 2,      /* a request's rows do not fit its page table */
    PLAMO_PAGED_BATCH_ROWS = 4, /* the new rows exceed the batch's row count, or starts are out of order */
    PLAMO_PAGED_COUNT = 8,      /* a negative row count, or one past 2^31 - 1 */
    PLAMO_PAGED_PAGE = 16,      /* a page id or slot outside the pool */
    PLAMO_PAGED_POSITION = 32,  /* a position outside the rotation table */
    PLAMO_PAGED_FAILED = 64     /* a bounded wait of a kernel ran out: its results are not valid */
};

struct plamo_cuda;

/* Where to run. NULL means the context's own stream; the legacy default
   stream is (void *)1, as in the CUDA runtime. */

struct plamo_paged_plan_args {
    const int32_t *held;       /* [requests] own rows held before the step */
    const int32_t *added;      /* [requests] rows the step adds (0 and up) */
    int32_t *tables;           /* [requests][table_stride] page ids; the new pages' entries are written */
    const int32_t *free_pages; /* [free_count] ids of free pages, taken from the front */
    const int32_t *head;       /* NULL, or where to begin in free_pages: &summary[2] of an earlier plan */
    int32_t *lengths;          /* [requests] out: held + added */
    int32_t *starts;           /* [requests + 1] out: first batch row of each request */
    int32_t *slots;            /* [rows] out: slot of each new row, -1 for padding, -2 where the table or the free
                                  list has a negative page id or one from 2^25 up (the store reports the row) */
    int32_t *positions;        /* [rows] out: base + own row, 0 for padding */
    int32_t *summary;          /* [4] out: status bits, new rows, free-list entries used so far
                                  (head + pages taken), longest length */
    uint64_t requests, table_stride, free_count, rows;
    int64_t base;              /* position of own row 0: the prefix's rows */
    void *stream;
};
/* Pages go to requests in order, to each request's rows in order: the result
   depends on the inputs alone. A request takes a page when a row reaches it.
   A step that cannot be taken as a whole (status bits 1, 2, 4, 8) changes
   nothing: lengths = held, starts = 0, every slot -1, no table entry or page
   taken, so that a captured step's following operators do nothing. `lengths`
   may be `held` itself, to advance a step in place; buffers that overlap in
   any other way are declined. */
int plamo_paged_plan(struct plamo_cuda *, const struct plamo_paged_plan_args *);

struct plamo_paged_store_args {
    const void *qkv;          /* [rows][(query_heads + 2 * kv_heads) * 128], rows qkv_stride elements apart */
    void *pool;
    void *q;                  /* [rows][query_heads][128] of the pool's type, rows q_stride elements apart */
    const int32_t *slots;     /* [rows], all different; -1: padding (its q row is zeroed) */
    const int32_t *positions; /* [rows] */
    const uint16_t *q_norm, *k_norm; /* [128] BF16 norm weights */
    const float *table;       /* [positions_count][128]: cos[64] | sin[64] of a position, concentration applied */
    uint32_t *status;
    uint64_t rows, qkv_stride, q_stride, pages, positions_count;
    uint32_t query_heads, kv_heads, qkv_type, pool_type;
    void *stream;
};
/* head <- rotate(head / sqrt(mean(head^2) + 1e-6) * (norm + 1)) for query and
   key heads, in FP32, rounded once to the pool's type; values are rounded to
   it as they are. rotate pairs dimension d with d + 64: the lower becomes
   a*cos - b*sin, the upper b*cos + a*sin. */
int plamo_paged_store(struct plamo_cuda *, const struct plamo_paged_store_args *);

/* The PLAMO_PAGED_* bits that store and attention calls without a word of their
   own have set since it was last asked; they are then clear. Waits for the
   context's own stream: a call on another one counts once that has run it
   (synchronise it first). PLAMO_PAGED_FAILED also where the word cannot be
   read. Not while a stream is being captured. */
uint32_t plamo_paged_status(struct plamo_cuda *);

struct plamo_paged_attention_args {
    const void *q;           /* [rows][query_heads][128] of the pool's type, rows q_stride elements apart */
    const void *pool;
    void *out;               /* as q, rows out_stride elements apart */
    const int32_t *starts;   /* [requests + 1] */
    const int32_t *lengths;  /* [requests] own rows, those of this step included */
    const int32_t *tables;   /* [requests][table_stride] */
    const int32_t *prefix_pages; /* [ceil(prefix_rows / 64)], may be NULL when prefix_rows is 0 */
    void *workspace;         /* plamo_paged_attention_workspace() bytes, 256-byte aligned */
    uint64_t workspace_bytes;
    uint32_t *status;
    uint64_t rows, q_stride, out_stride, requests, table_stride, prefix_rows, pages;
    uint64_t window;         /* rows a query sees, itself included (a sliding layer's window + 1); 0: all before it */
    uint32_t query_heads, kv_heads, type;
    float scale;             /* of the scores, 1 / sqrt(128) as a rule */
    void *stream;
    uint64_t most_new;       /* rows of the request that adds most (1 in a decode step), 0: not known. It chooses the
                                kernels, where `rows` counts padding or `requests` idle slots that hide it; every row
                                gets its result whatever it says. The workspace's size depends on it. */
};
/* Device bytes a call with these shapes needs (its pointers are not read);
   0 when the shapes would be declined. The prefix and a request's page table
   hold at most 2^30 rows each; requests, and rows times query heads, are at
   most 2^30. */
uint64_t plamo_paged_attention_workspace(struct plamo_cuda *, const struct plamo_paged_attention_args *);
/* out = sum over the rows j it sees of softmax_j(scale * q . k_j) v_j, for
   every new row and query head (head h reads KV head h / (query_heads /
   kv_heads)). The row at position p sees the prefix's rows and its request's
   own rows up to itself, of these the last `window` when there is one. A row
   that sees nothing gets zeros: padding, rows before starts[0], and rows whose
   request holds fewer rows (lengths) than it adds, before the first held one.
   Where the starts do not rise from 0 to at most `rows`, `status` gets
   PLAMO_PAGED_BATCH_ROWS; where they decrease, every row gets zeros. So
   reported, and without results, is a batch whose (row, head) pairs times the
   pages that they see pass 2^34. A row
   that sees a score of NaN, or scores of -infinity only, gets NaN. Rows past a request's length, of other
   requests and after a query's own never reach its result, whatever they
   hold. Scores, softmax sums and products are FP32 for both types (against
   a BF16 pool's values the softmax weights go in as two BF16 terms, 16 bits). */
int plamo_paged_attention(struct plamo_cuda *, const struct plamo_paged_attention_args *);

#ifdef __cplusplus
}
#endif
#endif
