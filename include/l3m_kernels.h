// l3m matvec entry points, B200 build. The host-pointer table keeps the reference's kernel-table
// shape (fpedd/l3m src/kernels.h:24-52) so its kernel tests drive the GPU kernels unchanged; the
// *_dev entry points take device pointers and a CUDA stream (passed as void *) and return 0 or a
// negative error (message from l3m_cuda_error()). No CUDA or torch types appear in any signature.
//
// Tile layout (the reference's, src/kernels.h:1-10, byte for byte): L3M_TILE = 16 outputs x K inputs,
//   f32   [K][16] float
//   bf16  [K/2][16][2] bf16
//   q8_0  per 32 inputs: d[16] f16, q[8][16][4] u8 = value + 128                 544 bytes
//   q4_0  per 32 inputs: d[16] f16, q[4][16][4] nibbles, value = nibble - 8     288 bytes
//   mxfp4 per 32 inputs: e[16] e8m0, the same nibbles, value = LUT[nibble]       272 bytes
// Each 64-byte line holds one 4-byte group of all 16 outputs, so a warp's 16-byte loads of a
// block are fully coalesced and every block starts 16-byte aligned.
#pragma once
#include <stddef.h>
#include <stdint.h>

#define L3M_API __attribute__((visibility("default")))
#define L3M_TILE   16
#define L3M_QBLOCK 32

#ifdef __cplusplus
extern "C" {
#endif

enum { L3M_DT_F32, L3M_DT_BF16, L3M_DT_Q8_0, L3M_DT_Q4_0, L3M_DT_MXFP4, L3M_DT_COUNT };

// The prepared activation (reference src/kernels.h:24-30): bf16 copy, or q8 with a per-32 scale and sum.
typedef struct {
    const float    *f32;
    const uint16_t *bf16;
    const int8_t   *q8;     // x[i] ~= q8[i] * scale[i/32]
    const float    *scale;  // n/32 entries
    const int32_t  *sum;    // n/32 entries: sum of q8 over the block
} l3m_vec;

// y[0 .. ntiles*16) = tiles . x, all host pointers (reference src/kernels.h:33). The GPU tables copy
// in, launch on the current device and copy out: a test and drop-in shim, not the fast path.
typedef void (*l3m_gemv_fn)(float *y, const void *tiles, int ntiles, int k, const l3m_vec *x);

typedef struct {                                   // reference src/kernels.h:35-40
    const char *name;
    l3m_gemv_fn gemv[L3M_DT_COUNT];
    void (*attend)(float *out, const float *q, const uint16_t *k, const uint16_t *v, int pos, int head_dim, int stride);
} l3m_kernels;

// "sm100a": results bit-identical to the reference's scalar table (src/kernels_scalar.c) for every
// dtype. "sm100a-fast": quantised dtypes identical as well; f32 and bf16 reassociate the sum over
// K across threads (tolerance-checked, like the reference's AVX tables).
L3M_API extern const l3m_kernels l3m_kernels_sm100a, l3m_kernels_sm100a_fast;

// Replaces reference src/dispatch.c:28-36: L3M_ISA=sm100a|sm100a-fast selects a table; anything else
// is reported and the default (sm100a) is used. There is no CPU table: without a usable B200 the
// engine's load fails with a message.
L3M_API const l3m_kernels *l3m_kernels_pick(void);
L3M_API int                l3m_kernels_usable(const l3m_kernels *k);   // 1 when a CUDA device of compute capability 10.x is present

// Layout helpers (reference src/kernels.h:48-52), host code.
L3M_API size_t l3m_row_bytes(int dtype, int k);
L3M_API size_t l3m_tile_bytes(int dtype, int k);
L3M_API void   l3m_pack_tile(void *dst, int dtype, const void *const rows[L3M_TILE], int k);   // NULL row = zeros
L3M_API void   l3m_dequant_row(float *out, int dtype, const void *row, int k);
L3M_API void   l3m_vec_prepare(l3m_vec *v, int dtype, const float *x, int n, void *scratch);    // scratch >= 2n + n/4 bytes

// ---- device entry points (no counterpart in the reference: the GPU-resident forms of the above)

// y = tiles . x on the device. exact bit 0: 1 the sm100a table's order, 0 sm100a-fast. exact bit 1
// (L3M_GEMV_CONST_TILES): the caller guarantees that no work issued earlier on the stream writes the
// tiles (model weights), so the streamed kernel may start reading them before that work has finished
// (x and y keep the stream order); successive calls then overlap.
#define L3M_GEMV_CONST_TILES 2
L3M_API int l3m_gemv_dev(int exact, int dtype, float *y, const void *tiles, int ntiles, int k, const l3m_vec *x, void *stream);
// The exact quantised matvec (the same y as l3m_gemv_dev with exact = 1, bit for bit) for callers
// that must not allocate device memory, such as a host whose framework owns the device's memory
// pool, or a decode loop where the implicit device synchronisation of cudaMalloc/cudaFree would
// stall other streams. No counterpart in the reference. K is split across every SM through one
// fixed 4 MiB device buffer inside this library: q8_0/q4_0/mxfp4 only, at most 524,288 block
// results per call (ntiles*16*k/32), larger calls return -1 and launch nothing. The buffer is
// shared by all calls on a device, so overlapping calls (two streams or threads) race and must be
// serialised. The first call on each device looks the buffer's address up and keeps it for the
// process's life, so do not reset a device this entry has used.
// Pointers must be 4-byte aligned (refused with -1 otherwise).
L3M_API int l3m_gemv_splitk_dev(int dtype, float *y, const void *tiles, int ntiles, int k, const l3m_vec *x, void *stream);
// One draw of the reference's temperature sampler (src/engine.c:98-101, 283-287, 370-384, one
// rank) over logits[0..vocab) on the device: weights expf((l - max) / temperature) (0 below -16),
// the first index whose running double sum exceeds u * (the whole sum), u the next xorshift64*
// draw of *rng_state (advanced); the last index when none does. rng_state, token: device memory;
// scratch: vocab floats of device memory. temperature must be > 0. Tests use it; l3m_generate
// samples inside its own kernel with the same code.
L3M_API int l3m_sample_dev(const float *logits, int vocab, float temperature, uint64_t *rng_state, int32_t *token, float *scratch,
                           void *stream);
// Prepare x[0..n) for dtype on the device, as l3m_vec_prepare. scratch (device) >= 2n + n/4 bytes.
L3M_API int l3m_vec_prepare_dev(int dtype, l3m_vec *out, const float *x, int n, void *scratch, void *stream);
// The exact integer part of each quantised kernel: dots[(t*16 + c)*(k/32) + b] = sum_i w*q8_x over block b
// of output c in tile t, the dtype's offset already removed (the value the epilogue converts to float).
L3M_API int l3m_block_dots_dev(int dtype, int32_t *dots, const void *tiles, int ntiles, int k, const l3m_vec *x, void *stream);
// Unpack quantised tiles on the device: integer weights q[(t*16+c)*k + i] and block scales d[(t*16+c)*(k/32) + b].
L3M_API int l3m_unpack_dev(int dtype, int8_t *q, float *d, const void *tiles, int ntiles, int k, void *stream);
// One head of causal attention over a bf16 KV cache (reference src/ops.h:14-16), device pointers.
L3M_API int l3m_attend_dev(float *out, const float *q, const uint16_t *k, const uint16_t *v, int pos, int head_dim, int stride, void *stream);
// y[i] = expf(x[i]) for i < n on the device, bit for bit the host C library's expf (the function the
// reference's softmax, SiLU and sampler call, src/ops.c:45, 50; the kernels above use the same code).
// x, y: device memory.
L3M_API int l3m_expf_dev(const float *x, float *y, int n, void *stream);
// Diagnostics: the SM cycles per step of a dependent fp32 fma chain (operands in registers), timed
// on the current device over `steps` steps (64 .. 2^24) by one warp; synchronous. The decode's
// chain-latency bound is its dependent steps per token times this.
L3M_API int l3m_chain_cycles_dev(int steps, double *cycles_per_step);
// ---- a paged key/value cache in 4 bits: its bookkeeping, its writer and its reader (no counterpart
// in the reference, whose one sequence has one bf16 cache). Keys and values are held in the file
// formats' 4-bit blocks, q4_0 or mxfp4, 32 values of one head of one token to a block; head_dim is
// rounded up to whole blocks (the padding holds zeros). The unit is a tile of 16 tokens of one
// head; with NG = ceil(head_dim / 32) it holds, in this order,
//   key codes     [16 tokens][4 parts t][NG blocks j][4 bytes]: nibble i (low one first) is value 32*j + 8*t + i
//   value codes   [16 tokens][8 parts g][NG blocks j][2 bytes]: nibble i is value 32*j + 4*g + i
//   key scales    [16 tokens][NG] and value scales [16 tokens][NG]: f16 (q4_0) or e8m0 (mxfp4)
// and tiles lie [page][kv head][page / 16]. value = (nibble - 8) * scale, or e2m1 * 2^(scale - 127).
// A slot is page id * page + offset. Slots, lengths and positions are int32, addresses 64-bit.
// All calls are asynchronous on the stream, allocate nothing, may be captured into a graph, and
// read every length on the device. They return 0, or -1 with nothing launched.
typedef struct {
    void *data;                  // n_pages * l3m_kv4_page_bytes() bytes of device memory, 16-byte aligned
    int   dtype;                 // L3M_DT_Q4_0 or L3M_DT_MXFP4
    int   n_pages;               // n_pages * page < 2^31, n_pages * n_kv_heads * page / 16 < 2^31
    int   page;                  // tokens per page, a multiple of 16, at most 4096
    int   n_kv_heads, head_dim;  // head_dim a multiple of 8, 8 .. 256
} l3m_kv4;
L3M_API size_t l3m_kv4_page_bytes(int dtype, int n_kv_heads, int head_dim, int page);   // 0: no such cache

// Bits that the calls below OR into their *status (device memory, NULL: not reported). The caller zeroes it.
enum {
    L3M_KV4_NO_PAGES = 1,        // plan: the free list ran out
    L3M_KV4_BAD_LENGTH = 2,      // plan: a negative kv_len, a length beyond max_blocks * page or 2^31 - page, or a bad n_free
    L3M_KV4_NO_ROOM = 4,         // plan: more new tokens than max_tokens
    L3M_KV4_BAD_PAGE = 8,        // a page id or slot outside the cache was left out (plan: slot -1)
    L3M_KV4_BAD_POS = 16,        // qkv: a position outside the rotation table; its row was left out
    L3M_KV4_TIMEOUT = 32,        // attend: a wait inside the kernel gave up; the rows concerned are NaN
};

// One step's bookkeeping. Request r holds kv_len[r] tokens in the pages tables[r][0 .. ceil(kv_len/page))
// and brings new_len[r] tokens (0: it waits; below 0: it has ended and its pages return to the free list,
// in request order, its table row left as it is). free_pages[0 .. *n_free) is a stack: new pages
// come off its top, in request order. Writes the new table entries, the free list, *n_free_out,
// q_start[0 .. n_req] (running sum of the new tokens), kv_total[r] (the length with the new tokens), and
// for each new token its position and slot; rows behind the last one get -1. A request is left out (kv_total 0,
// slots and positions -1, no pages taken) when its lengths are bad, when the pages wanted by it and the
// requests before it exceed the free list and it wants some, or when its rows pass max_tokens; a status bit says so. q_start counts its
// rows all the same, so it can pass max_tokens: l3m_kv4_attend's max_rows = max_tokens keeps the attention inside its tensors then.
typedef struct {
    int n_req;                   // 0 .. 16384
    int max_blocks;              // entries of a table row
    int max_tokens;              // entries of slot and pos, at most 2^30
    int page, n_pages;
    const int32_t *kv_len, *new_len;
    int32_t *tables;             // [n_req][max_blocks]
    int32_t *free_pages;         // [n_pages]
    const int32_t *n_free;       // device memory, one value
    int32_t *n_free_out;         // another one: it must not be n_free
    int32_t *q_start;            // [n_req + 1]
    int32_t *kv_total;           // [n_req], not kv_len
    int32_t *slot, *pos;         // [max_tokens]
    int32_t *status;
} l3m_kv4_plan;
L3M_API int l3m_kv4_plan_dev(const l3m_kv4_plan *a, void *stream);

// The prelude of attention, one pass over q, k and v: RMS norm of each query and key head over head_dim
// (q_norm, k_norm: weights, NULL = no norm; x * w / sqrt(mean x^2 + eps)), then the rotation of its first rot_dim
// values by pos[token] (rope_table[n_pos][rot_dim / 2][2]: cos, sin). Queries go to q_out. Keys go to
// k_out (may be NULL) and, with a cache, keys and values to the cache's slot[token] in 4 bits (a negative slot:
// not stored). A token with pos < 0 is padding: nothing of it is read or written. Tensors are
// [n_tokens][heads][head_dim], heads contiguous, ld elements from token to token, so slices of one qkv matrix serve; q_out may be q
// and k_out may be k, at the same stride; otherwise results overlap no input. Codes and scales are those of exact arithmetic: as ggml's rule gives them for the
// normed, rotated values in 64 bits (scales in f16: rounded to f32 first, at most 65504); a NaN is stored as 0. The tokens of a call
// have different slots (the plan's do): where two share one, its row holds a mixture of both.
typedef struct {
    int   dtype;                 // of q, k, v, q_out and k_out: L3M_DT_F32 or L3M_DT_BF16
    int   n_tokens, n_heads, n_kv_heads, head_dim;
    int   rope;                  // 0 none, 1 adjacent pairs (2i, 2i + 1), 2 halves (i, i + rot_dim / 2)
    int   rot_dim;               // even, at most head_dim
    int   n_pos;
    float eps;
    const float *q_norm, *k_norm, *rope_table;
    const int32_t *pos, *slot;   // slot: read with a cache only
    const void *q, *k, *v;       // q with n_heads > 0; k; v with a cache only
    int64_t q_ld, k_ld, v_ld;
    void *q_out, *k_out;
    int64_t q_out_ld, k_out_ld;
    int32_t *status;
} l3m_qkv;
L3M_API int l3m_qkv_rope_dev(const l3m_kv4 *cache, const l3m_qkv *a, void *stream);   // cache may be NULL
// Reads cache rows back: k[i], v[i] ([n][n_kv_heads][head_dim], dtype L3M_DT_F32 or L3M_DT_BF16, either may be NULL) =
// the values at slots[i]. A row whose slot lies outside the cache is left as it was.
L3M_API int l3m_kv4_load_dev(const l3m_kv4 *cache, int dtype, void *k, void *v, const int32_t *slots, int n, void *stream);

// Causal attention of a batch over the cache: request r's queries are rows q_start[r] .. q_start[r+1) of q, the
// newest tokens of its kv_len[r] cached ones (kv_total of the plan, after l3m_qkv_rope_dev stored them). The query at position p sees
// positions 0 .. p, with a window only those above p - window. A query that sees nothing (kv_len 0) gets
// zeros; rows outside q_start's range stay as they were. Positions in pages with an id outside the cache are not seen. Scales that are
// not finite (the store writes none) leave queries alone that do not see them; what sees them is not defined. Sums are held in 32 bits: a value
// below 2^-100 of the largest that any of the request's new tokens sees in its block of 32 dims may count as 0, and scores are defined where sum |q| |k| |scale|
// over a head's dims, a key of q4_0 taken as 8 of its scales, stays below 2^20 (beyond it a score's rounding is that of a factor in its probability),
// a key's scale below 2^100. Where that sum is small (5 or so), f32 results are within 2^-16 of sum p |v| of exact arithmetic, bf16 results within their
// rounding and 2^-10 of sum p |v| (over q4_0 of sum p (|v| + |scale|)), both within 2^-32 of the block's largest scale a token beside. out may not overlap q.
typedef struct {
    int   dtype;                 // of q and out: L3M_DT_F32 or L3M_DT_BF16
    int   n_heads;               // a multiple of n_kv_heads: query head h reads kv head h / (n_heads / n_kv_heads)
    int   n_req, max_blocks;
    int   max_q;                 // at least every request's number of queries (more are not looked at); max_q * n_heads <= 2^30. The bounds, not the
                                 // lengths, choose the kernel: single tokens beside a prompt, or under a prompt's max_q, take a prompt's time each
    int   max_kv;                // at least every kv_len; at most max_blocks * page
    int   window;                // 0: none
    float scale;                 // of the scores, below 2^127 in magnitude
    const void *q;
    void *out;
    int64_t q_ld, out_ld;        // elements from token to token
    const int32_t *q_start, *kv_len, *tables;
    void  *scratch;              // l3m_kv4_attend_scratch() bytes of device memory, 16-byte aligned, in any state;
    size_t scratch_bytes;        // calls that overlap need one each
    int32_t *status;
    int   max_rows;              // rows that q and out have: queries of rows behind them are not looked at and nothing is written there.
                                 // 0: not stated, q_start never passes them (the plan's does where it reports L3M_KV4_NO_ROOM)
} l3m_kv4_attend;
L3M_API size_t l3m_kv4_attend_scratch(const l3m_kv4 *cache, const l3m_kv4_attend *a);   // from the integer fields alone
L3M_API int    l3m_kv4_attend_dev(const l3m_kv4 *cache, const l3m_kv4_attend *a, void *stream);

// The last CUDA error this library saw, as text ("" if none).
L3M_API const char *l3m_cuda_error(void);

#ifdef __cplusplus
}
#endif
