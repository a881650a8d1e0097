/*
 * b200exec.h -- C ABI of libb200exec.so, the B200 (sm_100a) backend for the
 * compiled executor of lets-build-a-runtime.
 *
 * The reference runs a planned graph with ONE call,
 *     void execute(OpNode* nodes, int n_nodes)          (csrc/executor.c:458)
 * bound from Python by ctypes (runtime/executor/common.py:148-163) over an
 * OpNode array built by CompiledExecutor.compile (runtime/executor/
 * compiled.py:34-70).  This library exports the same symbol with the same
 * struct, op codes and extra[] encodings.  What changes is where memory
 * lives: every pointer in the node array is a DEVICE address (arena,
 * weights and input staging allocated through rt_alloc below, or any other
 * device allocation of the current device), and execution happens on the
 * GPU.  The reference's C side never allocates (the caller owns arena,
 * weights, inputs); here the caller still owns them, but allocates them
 * through this library so that they are device memory.
 *
 * Error convention: the reference aborts on an unknown op
 * (csrc/executor.c:461-464) and checks nothing else.  This library never
 * aborts: every entry point that can fail returns an RT_* status and
 * records it for rt_last_error()/rt_last_error_message(); `execute`, which
 * must keep its void signature for ctypes compatibility, only records it.
 *
 * Threading: like the reference, one call at a time per process; all work
 * runs on one library-owned CUDA stream of the device given to rt_init.
 */
#ifndef B200EXEC_H
#define B200EXEC_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define RT_MAX_INPUTS 12   /* csrc/runtime.h:57  MAX_INPUTS */
#define RT_MAX_DIMS 24     /* csrc/runtime.h:58  MAX_DIMS   */

/* Byte-identical to OpNode (csrc/runtime.h:60-69) and COpNode
 * (runtime/executor/common.py:125-141). */
typedef struct OpNode {
    int op;
    int n_inputs;
    void* inputs[RT_MAX_INPUTS];
    void* output;
    int out_shape[RT_MAX_DIMS];
    int n_dims;
    int elem_size;
    int extra[RT_MAX_DIMS];
} OpNode;

/* Op codes: enum OpType of csrc/runtime.h:11-55 (= runtime/ir.py:36-78). */
enum RtOpType {
    RT_OP_RELU = 100, RT_OP_EXP = 101, RT_OP_TANH = 102, RT_OP_POW = 103,
    RT_OP_GELU = 104, RT_OP_RSQRT = 105, RT_OP_SILU = 106, RT_OP_NEG = 107,
    RT_OP_COS = 108, RT_OP_SIN = 109,
    RT_OP_ADD = 200, RT_OP_SUB = 201, RT_OP_MUL = 202, RT_OP_DIV = 203,
    RT_OP_MAX = 300, RT_OP_SUM = 301, RT_OP_SOFTMAX = 302,
    RT_OP_MATMUL = 400,
    RT_OP_RESHAPE = 500, RT_OP_TRANSPOSE = 501, RT_OP_PERMUTE = 502,
    RT_OP_SLICE = 503, RT_OP_EMBEDDING = 504, RT_OP_CAT = 505,
    RT_OP_LAYERNORM = 600, RT_OP_RMSNORM = 601,
    RT_OP_MATMUL_ADD = 1000, RT_OP_FUSED_BIAS_RELU = 1001,
    RT_OP_ATTENTION = 1002, RT_OP_GATED_ACT = 1003
};

/* Status codes. */
enum RtStatus {
    RT_OK = 0,
    RT_ERR_NOT_INITIALIZED = 1,
    RT_ERR_BAD_OP = 2,          /* op code with no dispatch entry (incl. PERMUTE) */
    RT_ERR_BAD_NODE = 3,        /* malformed node: dims, n_inputs, extras */
    RT_ERR_NULL_POINTER = 4,
    RT_ERR_HOST_POINTER = 5,    /* pointer is not device memory of this device */
    RT_ERR_OUT_OF_RANGE = 6,    /* buffer extent leaves its allocation */
    RT_ERR_UNSUPPORTED = 7,     /* valid reference node this build cannot run */
    RT_ERR_CUDA = 8,            /* a CUDA runtime/driver call failed */
    RT_ERR_OOM = 9,
    RT_ERR_ARGUMENT = 10,
    RT_ERR_KERNEL_TIMEOUT = 11  /* a kernel gave up a bounded wait (it recorded a code and returned) */
};

/* Execution flags for rt_execute. */
#define RT_FLAG_EAGER 1   /* launch node by node, no CUDA graph */
#define RT_FLAG_ASYNC 2   /* do not synchronise before returning */

/* One host<->device copy for rt_execute_io. */
typedef struct RtCopy {
    void* dst;
    const void* src;
    size_t bytes;
} RtCopy;

/* ---- lifecycle ---------------------------------------------------------- */
/* Select the device, create the stream.  Idempotent for the same device. */
int rt_init(int device);
/* Wait for the device, free every allocation, cached plan and graph; the
 * library may be re-inited.  A caller's CUDA graphs that hold serving calls
 * are not to be launched any more. */
int rt_destroy(void);
const char* rt_version(void);

/* ---- memory (replaces the host arena of runtime/executor/common.py:83-87
 *      and the numpy weight buffers) ------------------------------------- */
void* rt_alloc(size_t bytes);             /* device, 256-B aligned, zeroed; NULL on failure */
int rt_free(void* dev);
void* rt_host_alloc(size_t bytes);        /* pinned host memory; NULL on failure */
int rt_host_free(void* host);
int rt_upload(void* dst_dev, const void* src_host, size_t bytes);
int rt_download(void* dst_host, const void* src_dev, size_t bytes);
/* Declare [dev, dev+bytes) immutable (graph constants).  The library may
 * then cache derived forms of it (split matrix operands) across calls.
 * Writing to the range afterwards requires rt_reset_plans(). */
int rt_mark_constant(void* dev, size_t bytes);

/* ---- execution ---------------------------------------------------------- */
/* Drop-in for csrc/executor.c:458.  First call with a given node array
 * validates it, prepares derived operands and captures the launch sequence
 * into a CUDA graph; later calls with identical contents replay the graph.
 * Returns after the GPU finished.  Errors: see rt_last_error(). */
void execute(OpNode* nodes, int n_nodes);
/* Same, returning the status; flags = RT_FLAG_*. */
int rt_execute(const OpNode* nodes, int n_nodes, int flags);
/* End to end: n_in host->device copies, the graph of `nodes`, n_out
 * device->host copies, all on the library stream, then one synchronise. */
int rt_execute_io(const OpNode* nodes, int n_nodes,
                  const RtCopy* h2d, int n_in, const RtCopy* d2h, int n_out);
/* One batch as independent chunks (no counterpart in the reference): chunk c
 * runs its own node array -- the graph planned for that chunk's rows, with
 * its own arena -- between its host-to-device and device-to-host copies, on
 * its own stream, so one chunk's copies overlap another chunk's kernels.
 * Only valid when the chunks share no intermediate memory and the model
 * treats batch rows independently.  Synchronous, like rt_execute_io. */
typedef struct RtChunk {
    const OpNode* nodes;
    int n_nodes;
    const RtCopy* h2d;
    int n_in;
    const RtCopy* d2h;
    int n_out;
} RtChunk;
int rt_execute_chunks(const RtChunk* chunks, int n_chunks);
/* Validate and prepare (capture) without running. */
int rt_prepare(const OpNode* nodes, int n_nodes);
/* Kernel launches one execute of this node array issues (after prepare). */
int rt_kernel_launches(const OpNode* nodes, int n_nodes);
/* Per-node device time: runs the array `reps` times eagerly with CUDA
 * events around each node on the library stream; ms_per_node[i] receives
 * the mean over reps.  This fills RunProfile.op_timings
 * (runtime/executor/common.py:24-63) for the compiled path. */
int rt_profile(const OpNode* nodes, int n_nodes, int reps, float* ms_per_node);
/* Drop cached plans, graphs and derived constant forms. */
int rt_reset_plans(void);
/* Drop the cached plan (captured graph, scratch) of this node array only --
 * what an executor releases when it is closed while others keep theirs.
 * rt_plan_count() = plans currently cached (one per distinct node array). */
int rt_release(const OpNode* nodes, int n_nodes);
int rt_plan_count(void);
int rt_synchronize(void);
/* The library stream (a cudaStream_t), for callers that order work on it. */
void* rt_stream(void);
/* Declare [ptr, ptr+bytes) a graph output: plan-time layout fusion never
 * folds away a node that writes into it.  The output of the last node of an
 * array is always treated as a graph output; callers whose graphs return
 * more than that register the other outputs here before the first execute
 * (no counterpart in the reference, whose C side computes every node).
 * A registration lasts until rt_unprotect_all or until the rt_alloc memory
 * holding `ptr` is released with rt_free. */
int rt_protect(const void* ptr, size_t bytes);
int rt_unprotect_all(void);
/* Plan-time fusion, as execute would apply it to this node array:
 * flags[i] = 1 when node i is folded into another node and not launched (a
 * SLICE / TRANSPOSE around attention, a GELU after a GEMM), 2 for an
 * attention node launched with strided operands, 3 for a GEMM that applies a
 * folded activation and/or writes the split A operand of a later GEMM in its
 * epilogue (its A may arrive split as well), 4 for a GEMM whose only fusion is
 * that its A operand arrives split (no split pass),
 * 5 for the last node of a folded RMSNorm + rotary-embedding chain (it runs
 * the fused kernel), 6 for a gated activation reading its inputs through
 * strided views of the tensor its folded SLICEs took them from, 8 for a
 * LAYERNORM / RMSNORM writing the split A operand of the GEMM reading it
 * (that GEMM: 4), 7 for a GEMM whose epilogue applies a folded gated
 * activation (SLICE, SLICE, GATED_ACT of its output: 1 each), 0 otherwise.  Returns the number of folded nodes.  Host only: needs no
 * device and no rt_init.  RT_FUSE=0 turns all fusion off. */
int rt_fusion_report(const OpNode* nodes, int n_nodes, int* flags);

/* ---- allocation-free GEMM ------------------------------------------------ */
/* No counterpart in the reference.  C[M,N] = alpha * A[M,K] . op(B) + bias
 * (bias may be NULL; op(B) = B^T when trans_b, B stored [N,K], else B [K,N]),
 * computed by the same split-operand tensor-core kernel as MATMUL/MATMUL_ADD
 * (tf32 hi.hi product plus bf16 cross terms), for callers that may not
 * allocate device memory: plugins whose host application owns every device
 * allocation through its own pool, and processes that must not grow their
 * device footprint after start-up.  It allocates nothing and needs no
 * rt_init: it runs on the current device and `stream` (a cudaStream_t;
 * NULL = legacy default stream).  It is synchronous: it waits for `stream`
 * and returns after C is written, so it is a host-thread call, not one for a
 * CUDA host callback (which may not call CUDA).  Scratch: a fixed
 * RT_NOALLOC_SCRATCH_BYTES device array inside the library (held by every
 * GPU that loads it), so 8*(M*K + N*K) bytes must fit: larger problems
 * return RT_ERR_OUT_OF_RANGE; K % 4 != 0 returns RT_ERR_UNSUPPORTED.  A C
 * or bias off a 16-byte boundary is written / read with scalar accesses.
 * The first call on each device performs a one-time set-up (symbol address,
 * kernel attribute): make it before any stream capture.  All calls share
 * the scratch: calls that overlap on the GPU race.  Launches are checked
 * with cudaGetLastError, so an error left pending by earlier CUDA work of
 * the caller is reported as this call's RT_ERR_CUDA.  Returns an RT_*
 * status (not recorded in rt_last_error). */
#define RT_NOALLOC_SCRATCH_BYTES (32u << 20)
int rt_matmul_noalloc(const float* a, const float* b, const float* bias, float* c,
                      int M, int N, int K, int trans_b, float alpha, void* stream);

/* ---- serving: paged key/value cache ------------------------------------- */
/* No counterpart in the reference, whose text generation re-plans and re-runs
 * the whole prefix for every token (run_gpt2.py:92-113).  These calls are what
 * a decoder runs beside its planned graph instead: they store the keys and
 * values of new tokens in the pages of a cache, attend over them, read them
 * back, and verify drafted tokens.
 *
 * All of them need rt_init, enqueue on the caller's `stream` (a cudaStream_t
 * of that device; NULL = legacy default stream) and return without waiting;
 * they allocate nothing and may be captured into a CUDA graph.  Arguments are
 * checked on the host before anything is enqueued.  What only the device can
 * see (slots, page numbers, lengths, offsets) is bounds-checked by the
 * kernels: an entry out of range is treated as absent and reported as
 * RT_ERR_OUT_OF_RANGE by the next rt_check_stream (of whichever stream: the
 * serving calls share one error word, which planned graphs do not see). */
enum RtDtype { RT_F32 = 0, RT_BF16 = 1, RT_F8E4M3 = 2, RT_I8 = 3 };
/* The caller has established that every pointer of the call is memory of the
 * library's device and spans what the sizes and strides say (a tensor library
 * knows): the library then skips its own query of each pointer, which costs
 * more than the launch for the smallest calls. */
#define RT_POINTERS_CHECKED 1

/* One layer's cache, owned by the caller.  Element d of head h in slot s of
 * page p is k[p*stride[0] + s*stride[1] + h*stride[2] + d] (v alike); the
 * features are contiguous, k, v and the strides (in bytes) multiples of 16,
 * the strides the same for k and v, head_dim a multiple of 16 up to 128.  RT_F32 / RT_BF16 hold the values;
 * RT_F8E4M3 / RT_I8 hold codes, and the value is code * scale with one scale
 * per (page, slot, head) at k_scale[p*scale_stride[0] + s*scale_stride[1] +
 * h*scale_stride[2]] (NULL otherwise). */
typedef struct RtKvCache {
    void* k;
    void* v;
    float* k_scale;
    float* v_scale;
    int64_t stride[3];
    int64_t scale_stride[3];
    int dtype;
    int n_pages;
    int page_size;
    int n_heads;
    int head_dim;
    int flags;   /* RT_POINTERS_CHECKED, for all pointers of the call */
} RtKvCache;

/* Stores n_tokens rows of k and v (dtype RT_F32 / RT_BF16; element (token,
 * head, d) at token*stride[0] + head*stride[1] + d) into the cache: token i
 * goes to slot slots[i] = page * page_size + position in the page; a negative
 * slot skips the token.  Two tokens of one call must not share a slot.  For 8
 * bits, with a = max |x| over the token's head and M = 127 (I8) or 448
 * (F8E4M3), in fp32 with every step rounded: scale = a * (1/M), code = x *
 * ((1/a) * M) to the nearest code, ties to even; a < 2^-100 stores zeros with
 * scale 0, a non-finite value in the head stores zeros with scale NaN (the
 * head reads back as NaN). */
typedef struct RtKvWrite {
    RtKvCache cache;
    const void* k;
    const void* v;
    int64_t k_stride[2];
    int64_t v_stride[2];
    const int64_t* slots;
    int dtype;
    int n_tokens;
} RtKvWrite;
int rt_kv_write(const RtKvWrite* w, void* stream);

/* Reads cached positions back as dense rows: row cu[b] + i of k_out / v_out
 * (dtype RT_F32 / RT_BF16, element (row, head, d) at row*stride[0] +
 * head*stride[1] + d) is position start[b] + i of sequence b, i < cu[b+1] -
 * cu[b] (start NULL: 0).  Position j of sequence b lies in page
 * page_table[b*table_stride + j / page_size].  n_rows rows are written: those
 * from cu[n_seqs] on, and those whose position has no page, are zero. */
typedef struct RtKvRead {
    RtKvCache cache;
    void* k_out;
    void* v_out;
    int64_t k_stride[2];
    int64_t v_stride[2];
    const int* page_table;
    int64_t table_stride;
    const int* start;
    const int* cu;
    int dtype;
    int n_seqs;
    int table_width;
    int n_rows;
} RtKvRead;
int rt_kv_read(const RtKvRead* r, void* stream);

/* Attention of new tokens over the cache.  Sequence b brings the tokens
 * cu_new[b] .. cu_new[b+1]-1 of q (element (token, head, d) at token*stride[0]
 * + head*stride[1] + d; out alike) and has kv_lens[b] cached positions, the
 * new tokens' own (written before this call) included.  The new token i of n
 * stands at position P = kv_lens[b] - n + i and sees positions j <= P (causal)
 * or all of them, and with window > 0 only j > P - window.  out = softmax(q.k
 * * scale) v with query head h reading cache head h / (n_q_heads / n_heads);
 * lse (may be NULL, [tokens][n_q_heads]) = log of the softmax's sum.  A token
 * that sees nothing gets out = 0, lse = -inf, and so does a row of q that
 * belongs to no sequence (before cu_new[0], from cu_new[n_seqs] on, or of a
 * sequence whose offsets are refused).  What a position holds that a token
 * does not see never enters its result.
 * A call's work is counted in tiles of at least 8 rows (new token, query head
 * of a cache head) x 32 positions, fewer than 2^31 of them.
 * max_new / max_kv: the host's bounds on the per-sequence counts; they choose
 * how the work is split, not what is computed.  `ws` holds
 * rt_paged_attention_workspace(p) bytes of device memory, 16-byte aligned, used by
 * this call alone until it has run. */
typedef struct RtPagedAttention {
    RtKvCache cache;
    const void* q;
    void* out;
    float* lse;
    int64_t q_stride[2];
    int64_t out_stride[2];
    const int* page_table;
    int64_t table_stride;
    const int* kv_lens;
    const int* cu_new;
    float scale;
    int dtype;
    int n_seqs;
    int table_width;
    int n_q_heads;
    int total_new;
    int max_new;
    int max_kv;
    int causal;
    int window;
} RtPagedAttention;
size_t rt_paged_attention_workspace(const RtPagedAttention* p);
int rt_paged_attention(const RtPagedAttention* p, void* ws, size_t ws_bytes, void* stream);

/* Verification of drafted tokens (speculative sampling).  Row (b, i) of the
 * target's probabilities (dtype RT_F32 / RT_BF16, vocabulary contiguous, at
 * b*target_stride[0] + i*target_stride[1]) is the distribution of the token at
 * draft position i, row n_drafts the one after all drafts; draft holds the
 * draft's rows (NULL: every draft was proposed with probability 1).  Draft i
 * is accepted when accept_u[b*n_drafts + i] * draft(x_i) < target(x_i) and all
 * before it were; draft_lens[b] (NULL: n_drafts) of them exist.  The next
 * token is sampled from max(target - draft, 0) of the first refused row (from
 * target if nothing is left of it), or from the target's row after the last
 * draft: weights w become integers floor(min(w, 1) * 2^40) (negative or NaN:
 * 0), and the token is the lowest one whose running sum exceeds
 * floor(floor(u * 2^24) * total / 2^24), u = sample_u[b] in [0, 1).
 * tokens[b*(n_drafts+1) ..]: the accepted drafts, the sampled token (-1: the
 * row has no mass), then -1; accepted[b]: how many drafts were accepted. */
typedef struct RtVerifyDraft {
    const void* target;
    const void* draft;
    int64_t target_stride[2];
    int64_t draft_stride[2];
    const int* draft_tokens;
    const int* draft_lens;
    const float* accept_u;
    const float* sample_u;
    int* tokens;
    int* accepted;
    int dtype;
    int n_seqs;
    int n_drafts;
    int vocab;
    int flags;   /* RT_POINTERS_CHECKED */
} RtVerifyDraft;
int rt_verify_draft(const RtVerifyDraft* v, void* stream);

/* Waits for `stream` and returns what its kernels reported. */
int rt_check_stream(void* stream);

/* ---- errors ------------------------------------------------------------- */
/* No counterpart in the reference (which never waits on the device).  Runs
 * one kernel whose single bounded mbarrier wait is never satisfied, with a
 * limit of limit_ns (0 < limit_ns <= 1 s), through the same bounded-wait code
 * as the tensor-core kernels.  Returns RT_ERR_KERNEL_TIMEOUT (and records
 * it) when the timeout path works: the kernel records a code, returns, and
 * the context stays usable.  No fault, trap or hang is involved. */
int rt_check_wait_timeout(unsigned long long limit_ns);

int rt_last_error(void);                  /* status of the last failing call; 0 if none */
const char* rt_last_error_message(void);
void rt_clear_error(void);

#ifdef __cplusplus
}
#endif

#endif /* B200EXEC_H */
