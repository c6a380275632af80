/* splathip kernel-level entry points: single launches of the hot-path kernels on device
 * buffers, for parity tests and roofline micro-benchmarks. They have no counterpart in the
 * reference (whose kernels are candle's un-vendored matmul and sdpa, called from
 * depthanything3-rs/src/vit_block.rs:49-67 and mapanything-rs/src/vit_block.rs:29-38).
 * All pointers are device pointers; the launch is enqueued on the context's stream. */
#ifndef SPLATHIP_KERNELS_H
#define SPLATHIP_KERNELS_H

#include "splathip.h"

#ifdef __cplusplus
extern "C" {
#endif

/* `dtype` of every entry point below: SPLAT_F32, SPLAT_BF16 or SPLAT_F16 (the storage type of
 * the 16-bit or fp32 operands named as "in `dtype`"); accumulation is fp32 in all three.
 *
 * C[M, N] = act(A[M, K] W[N, K]^T + bias) ; A, W in `dtype`, W with
 * row stride ldw (a multiple of 64, columns K..ldw-1 zero), C fp32 when out_f32 else `dtype`.
 * act: 0 none, 1 relu, 2 gelu (erf). */
int splat_kernel_gemm(splat_ctx* ctx, int dtype, const void* A, int M, int K, const void* W, int N, int ldw,
                      const float* bias, int act, void* C, int out_f32);

/* The pre-norm block's GEMMs with its LayerNorm folded in (depthanything3-rs/src/vit_block.rs:151,165;
 * mapanything-rs/src/vit_block.rs:99,105: norm1 -> qkv, norm2 -> fc1), as the forwards run them.
 * Row statistics: (sum, sum of squares) of each row per group of `group` (64 or 128) columns.
 *  ln_in != NULL (consumer): A [M, K] holds the rows before the norm, ln_in [M, K/group, 2] their
 *    statistics; W and c1 the folded weights (W = gamma (.) W_lin along K, c1[n] = sum_k W[n, k])
 *    and bias = b_lin + W_lin beta; out = act(rstd * (acc - mean * c1[n]) + bias[n]) with each
 *    row's mean and rstd over K (biased variance, eps inside the root); K/group <= 16.
 *  res != NULL (producer, the residual epilogue of proj / fc2): out = res + gamma[n] * (acc +
 *    bias[n]), res and out fp32 [M, N]; with ln_out != NULL also the statistics of the output
 *    rows [M, N/group, 2] and, with copy != NULL, the rows in `dtype` [M, N] (the consumer's A).
 *  Otherwise as splat_kernel_gemm. */
int splat_kernel_gemm_ln(splat_ctx* ctx, int dtype, const void* A, int M, int K, const void* W, int N, int ldw,
                         const float* bias, int act, const float* ln_in, const float* c1, float eps,
                         const float* gamma, const float* res, float* ln_out, void* copy, int group, void* out,
                         int out_f32);

/* Row statistics of fp32 rows x [rows, n] (n a multiple of group, 64 or 128) in the layout above,
 * and the rows converted to `dtype` into copy [rows, n] when copy != NULL. */
int splat_kernel_ln_stats(splat_ctx* ctx, const float* x, int rows, int n, int group, float* stats, int dtype,
                          void* copy);

/* out[s*L + t, h*64 + e] = softmax(q k^T / 8) v for every sequence s < S and head h < heads,
 * reading q, k and v from a [S*L, 3*heads*64] qkv matrix (q | k | v column blocks). In bf16
 * and f16 the kernel multiplies q by log2(e)/8 and rounds it to that type before the products
 * (the networks' qkv GEMMs store q already scaled, rounding once); the weights P go to the
 * matrix cores rounded to the same type. */
int splat_kernel_attention(splat_ctx* ctx, int dtype, const void* qkv, void* out, int S, int L, int heads);

/* splat_kernel_attention that allocates nothing. It has no counterpart in the reference; it is
 * for callers that cannot allocate device memory (code under HIP graph capture, tight serving
 * loops, harnesses that forbid hipMalloc). Same kernels and key-slice plan; the fp32 partials
 * of a key-sliced launch (long sequences) live in a statically allocated scratch of 64 MiB per
 * GPU (ATTN_SCRATCH_BYTES, held by every GPU the library runs on until the process ends)
 * instead of the context's workspace. A launch whose partials would need more than that (e.g.
 * 24889 tokens x 12 heads: 236 MB; 6223 x 12 needs 59 MB and fits) runs as one key slice, with
 * no partials: the same softmax, not bit-identical to the sliced result. Every call on one GPU
 * shares that scratch, which keeps the last call's contents. Eager calls are ordered by the
 * library (each waits, on its stream, for the previous call's kernels on any context of that GPU,
 * through an event; no allocation); calls under stream capture are not, so captured graphs that
 * replay concurrently on one GPU race. Profiling records are not taken. */
int splat_kernel_attention_noalloc(splat_ctx* ctx, int dtype, const void* qkv, void* out, int S, int L, int heads);

/* Convolution (zero padding ks/2) on NHWC maps as an implicit GEMM:
 * out[V, Ho, Wo, Cout] = act(conv(relu_in ? relu(in) : in, w) + bias) + res, with
 * w [Cout, ldw] holding k = (ky*ks + kx)*Cin + ci (candle/PyTorch weight [Cout, Cin, ks, ks]
 * permuted), ldw a multiple of 64 with zero columns past ks*ks*Cin; res NHWC like out or NULL. */
int splat_kernel_conv2d(splat_ctx* ctx, int dtype, const void* in, int V, int H, int W, int Cin, const void* w,
                        int Cout, int ldw, int ks, int stride, const float* bias, int relu_in, int act,
                        const void* res, void* out);

/* Transposed convolution with kernel == stride s on NHWC maps: out[V, R*s, C*s, Cout];
 * w [s*s*Cout, ldw] with row (dy*s + dx)*Cout + co = weight[:, co, dy, dx] (PyTorch weight
 * [Cin, Cout, s, s]); bias [s*s*Cout] (the Cout biases repeated per (dy, dx)). */
int splat_kernel_conv_transpose2d(splat_ctx* ctx, int dtype, const void* in, int V, int R, int C, int Cin,
                                  const void* w, int Cout, int ldw, int s, const float* bias, void* out);

/* Per-kernel-class timing of the following forwards: HIP events around every launch on the
 * context's stream, with each launch's algorithmic work. Graph replay is bypassed while on. The lengths in a paged
 * cache are not known to the host: its calls count every sequence as long as the call allows, an upper bound. */
typedef struct splat_kernel_stat {
  char name[32];
  int launches;
  double ms;     /* summed launch durations */
  double flops;  /* summed algorithmic flops (2 * multiply-adds) */
  double bytes;  /* summed algorithmic bytes (inputs read once + outputs written once) */
} splat_kernel_stat;
int splat_profile_begin(splat_ctx* ctx);
/* Synchronises, stops recording and writes up to `max` classes (largest time first). */
int splat_profile_end(splat_ctx* ctx, splat_kernel_stat* stats, int max, int* count);

/* Bilinear resize with align_corners=True (torch upsample_bilinear2d) of NHWC maps. */
int splat_kernel_resize_bilinear(splat_ctx* ctx, int dtype, const void* in, int V, int Hi, int Wi, int C, void* out,
                                 int Ho, int Wo);

/* The device geometry of splat_da3_reconstruct / splat_ma_reconstruct on given network outputs
 * (all device pointers, fp32 unless noted): DA3 mode when depth != NULL (depth [V,H,W],
 * pose_encoding [V,9]); MapAnything mode otherwise (points_in_camera [V,H,W,3], quaternion
 * [V,4] xyzw, translation [V,3], mask [V,H,W] u8 unambiguous). conf [V,H,W]; foreground
 * [V,H,W] u8 or NULL. Out: cameras [V,16] f64 (R row-major, t, fx, fy, cx, cy, view 0's
 * frame), points [V,H,W,3], conf_out [V,H,W]. An input may share memory with an output (conf
 * cleaned in place, say): it is read from a copy that the context keeps. */
int splat_kernel_reconstruct(splat_ctx* ctx, int V, int H, int W, const float* depth, const float* pose_encoding,
                             const float* points_in_camera, const float* quaternion, const float* translation,
                             const float* conf, const uint8_t* mask, const uint8_t* foreground, double* cameras,
                             float* points, float* conf_out);

/* --- a paged cache of keys and values ------------------------------------------------------------
 * For networks of the caller's in which a token's keys and values stay as they are when others come: they are kept in pages,
 * and in each call one token of each sequence attends to those of its sequence. The two networks of this library are none: in
 * their global blocks every token sees every other, so that a new view changes the keys of all of them behind the first such
 * block, and no forward here uses the cache. Many tokens of one view are many sequences to these calls, each of which reads the whole
 * cache; splat_kernel_attention is for whole views. No counterpart in the reference. Heads of 64 channels, as in
 * splat_kernel_attention.
 *
 * Position p of sequence i lies in row p % page_size of page table[i * width + p / page_size]; a slot is
 * page * page_size + row. Lengths, tables and slots are device arrays: nothing here waits for the host. Table entries
 * outside [0, pages) hold no keys (their positions are left out), slots outside [0, pages * page_size) are not
 * written, lengths are clamped to what the table's row (1 to 2^30 positions) and max_len hold, negative ones to 0.
 * Outputs and workspaces overlap no other argument but where a call says so. Limits of one call: 2^25 tokens,
 * 2^21 query rows (n * heads), 2^25 sequences times kv_heads, 2^30 scored pages; beyond them it is refused.
 *
 * These calls allocate nothing and wait for nothing, so they may be captured into a HIP graph on the context's
 * stream. Calls that may run at the same time need workspaces of their own. */

/* The pools [pages][kv_heads][page_size][64] in `dtype`, 16-byte aligned; page_stride elements from one page to
 * the next in both (at least kv_heads * page_size * 64, a multiple of 8, at most 2^31; 0: exactly that). page_size is
 * a power of two from 8 to 256, pages * page_size below 2^31. */
typedef struct splat_kv_cache {
  int32_t dtype;
  int32_t pages;
  int32_t page_size;
  int32_t kv_heads;
  int64_t page_stride;
  void* k;
  void* v;
} splat_kv_cache;

/* Status that splat_kernel_block_tables leaves on the device. */
typedef enum splat_table_status {
  SPLAT_TABLE_OK = 0,
  SPLAT_TABLE_BAD_LENGTH = 1, /* a negative length, one past the table's width, or `used` outside the pool */
  SPLAT_TABLE_POOL_EMPTY = 2, /* the pool holds fewer pages than are needed */
  SPLAT_TABLE_SLOTS_FULL = 3  /* more than `cap` new tokens */
} splat_table_status;

/* Block tables and slot maps of n requests that hold past[i] positions and get add[i] new ones. The pages that
 * request i lacks are the next of pool [pool_size] behind the *used that are taken, requests in order; they go
 * into table [n, width] behind its ceil(past[i] / page_size) pages. Out: lens[i] = past[i] + add[i]; starts [n + 1],
 * the first new token of each request and their number; slots [cap] and positions [cap] (NULL: not wanted) of the new
 * tokens, requests in order, -1 and 0 behind the last; *used_out = pages taken now. lens may be past and used_out
 * used; other outputs overlap nothing. If *status is not SPLAT_TABLE_OK nothing was taken: the table, lens and
 * used stay, starts are 0 and slots -1. An entry of the pool or table below 0 gives slots of -1. n up to 65536. */
int splat_kernel_block_tables(splat_ctx* ctx, int n, const int32_t* past, const int32_t* add, int page_size,
                              const int32_t* pool, int pool_size, const int32_t* used, int32_t* table, int width,
                              int32_t* lens, int32_t* starts, int32_t* slots, int32_t* positions, int cap,
                              int32_t* used_out, int32_t* status);

/* Norms of the queries' and keys' heads and the position rotation in one pass over qkv [tokens, (heads + 2 *
 * kv_heads) * 64] (q | k | v, row stride ld) in `dtype`; statistics and angles in fp32 or more, rounded once.
 * norm: per head over its 64 channels, SPLAT_NORM_LAYER (x - mean) / sqrt(var + eps) * w + b (biased variance) or
 * SPLAT_NORM_RMS x / sqrt(mean(x^2) + eps) * w + b, with w and b fp32 [64] (qw, qb for queries, kw, kb for keys, 16-byte
 * aligned; NULL: left out). rope: SPLAT_ROPE_LINE turns channels (c, c + 32) by positions[t] * rope_base^(-c / 32); SPLAT_ROPE_GRID
 * turns (c, c + 16) of channels 0-31 by positions[t][0] and of channels 32-63 by positions[t][1], times
 * rope_base^(-c / 16) (depthanything3-rs/src/rope.rs:57-73, with base 100). q_out [tokens, heads * 64] and k_out
 * [tokens, kv_heads * 64] (NULL: not wanted) have row strides ldq and ldk; they may be qkv's own q and k blocks, and
 * overlap it nowhere else. With cache and slots [tokens] (both or neither) keys and values also go to the cache;
 * a slot outside the pool (-1: padding) stores nothing. The slots of one call are distinct. Row strides are multiples
 * of 8 elements and at most 2^31, rows 16-byte aligned. */
typedef enum splat_norm { SPLAT_NORM_NONE = 0, SPLAT_NORM_LAYER = 1, SPLAT_NORM_RMS = 2 } splat_norm;
typedef enum splat_rope { SPLAT_ROPE_NONE = 0, SPLAT_ROPE_LINE = 1, SPLAT_ROPE_GRID = 2 } splat_rope;
int splat_kernel_qk_norm_rope(splat_ctx* ctx, int dtype, const void* qkv, int64_t ld, int tokens, int heads,
                              int kv_heads, int norm, const float* qw, const float* qb, const float* kw,
                              const float* kb, float eps, int rope, double rope_base, const int32_t* positions,
                              void* q_out, int64_t ldq, void* k_out, int64_t ldk, const splat_kv_cache* cache,
                              const int32_t* slots);

/* Per page and head the lowest and the highest key of each channel, bounds [pages][kv_heads][2][64] in the cache's
 * dtype, over the page's positions below lens[i]: of the pages that hold the last add[i] positions of each
 * sequence (add NULL: all of its pages). max_add: about the largest add, which sizes the launch; any value is
 * right. NaN in a channel gives NaN. A page that two tables share has to be full, or as full in both. */
int splat_kernel_page_bounds(splat_ctx* ctx, const splat_kv_cache* cache, int n, const int32_t* table, int width,
                             const int32_t* lens, const int32_t* add, int max_add, void* bounds);

/* Attention of one token a sequence over its lens[i] cached positions: out[i, h] = softmax(scale q[i, h] K^T) V with
 * the keys and values of head h / (heads / kv_heads); zeros for a sequence without keys. q and out [n, heads * 64] in the
 * cache's dtype, row strides ldq and ldo (multiples of 8 elements up to 2^31, rows 16-byte aligned, not overlapping). max_len: an
 * upper bound of the lengths that the host knows, for the launch (longer ones are cut there). In bf16 and f16 a
 * weight goes to the matrix cores as two numbers of that type, the second what the first leaves: 16 bits of it in bf16, 22 in
 * f16 (the first alone for a sequence whose sums hold a NaN, as beside an infinite value).
 * workspace: device memory of at least splat_paged_attention_workspace's bytes, 16-byte aligned. One for the largest n, max_len (and
 * topk) serves every smaller call. */
int splat_paged_attention_workspace(const splat_kv_cache* cache, int n, int heads, int max_len, size_t* bytes);
int splat_kernel_paged_attention(splat_ctx* ctx, const splat_kv_cache* cache, const void* q, int64_t ldq, int n,
                                 int heads, const int32_t* table, int width, const int32_t* lens, int max_len,
                                 float scale, void* out, int64_t ldo, void* workspace, size_t workspace_bytes);

/* splat_kernel_paged_attention over the topk pages of each (sequence, key head) with the largest scores, the newest
 * page always among them. A page's score is a sum over the heads of the group, in 64 bits: of each head the most that its
 * query's product with a key between the page's bounds (splat_kernel_page_bounds) can be, each head with a key of its own, so that
 * no key of the page gives the heads more. The lower page comes first where scores are equal, NaN above all (a NaN bound or
 * query, or a query of 0 beside an infinite bound; an infinite bound that a query's sign does not choose takes no part).
 * selected [n, kv_heads, topk]: the pages' places in the table's row, ascending, -1 behind the last. topk is at most 2^27;
 * scale must be positive. */
int splat_sparse_attention_workspace(const splat_kv_cache* cache, int n, int heads, int max_len, int topk,
                                     size_t* bytes);
int splat_kernel_sparse_attention(splat_ctx* ctx, const splat_kv_cache* cache, const void* bounds, const void* q,
                                  int64_t ldq, int n, int heads, const int32_t* table, int width,
                                  const int32_t* lens, int max_len, int topk, float scale, void* out, int64_t ldo,
                                  int32_t* selected, void* workspace, size_t workspace_bytes);

#ifdef __cplusplus
}
#endif

#endif /* SPLATHIP_KERNELS_H */
