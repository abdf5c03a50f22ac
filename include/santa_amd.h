/*
 * santa_amd.h -- C ABI of the MI355X (gfx950) S^2ANTA sampled-attention
 * decode library (libsanta_amd.so).
 *
 * Plain pointers, sizes and a hipStream_t; no torch types.  All device
 * pointers are device memory on the current HIP device; every launch is
 * asynchronous on `stream` and nothing here synchronizes the device or reads
 * device memory on the host.  Inputs are never written.
 *
 * Reference interfaces replaced (upstream paths, with
 *   flash/ = flash_style_fused_santa_fixed_tile_budgets/,
 *   prop/  = santa_fused_proportional_tile_budgets/):
 *   santa_flash_plan          <- flash/santa_cuda.cpp:36-44,188-210 (block_n, T_c, S_per_tile)
 *   santa_flash_fused_tiles   <- launch_fused_tiles_vec_gqa_gh4_d128_bn{32,64,256}_{bf16,f16}
 *                                flash/santa_cuda.cpp:56-96, flash/santa_cuda_kernel.cu:514-626
 *   santa_flash_finalize      <- launch_finalize_weighted_{bf16,f16} + launch_reduce_vrows
 *                                flash/santa_cuda.cpp:98-120, flash/santa_cuda_kernel.cu:628-681
 *   santa_flash_decode        <- the launch sequence of decode_systematic_scalar,
 *   (+ _decode_tiles/_merge)     flash/santa_cuda.cpp:174-343 (minus the torch allocations)
 *   santa_prop_plan           <- prop/santa_cuda.cpp:39-77,188-229 (block_n, T_c, pass-1 path)
 *   santa_prop_pass1          <- launch_pass1_tiles_{vec,wmma}_gqa_{bf16,f16}
 *                                prop/santa_cuda.cpp:81-101, prop/santa_cuda_kernel.cu:445-519
 *   santa_prop_tile_budgets   <- launch_tile_budgets, prop/santa_cuda.cpp:108-112,
 *                                prop/santa_cuda_kernel.cu:904-915
 *   santa_prop_pass2          <- launch_pass2_grouped_fused_atomic_{bf16,f16} +
 *                                launch_cast_scale_out_{bf16,f16} + launch_reduce_vrows,
 *                                prop/santa_cuda.cpp:114-138, prop/santa_cuda_kernel.cu:917-1005
 *   santa_prop_decode         <- the launch sequence of decode_systematic_scalar,
 *                                prop/santa_cuda.cpp:270-352
 *
 * The stage entry points keep the reference launchers' split of the work and
 * their argument meaning, with these deviations:
 *   - no q_scale / scale argument (santa_flash_fused_tiles, santa_prop_pass1):
 *     the scale is computed inside from D exactly as the reference's host
 *     computes the value it passes, 1.0f / sqrtf((float)D) (flash: D = 128,
 *     bits 0x3DB504F3, flash/santa_cuda.cpp:210; prop/santa_cuda.cpp:208);
 *   - santa_flash_fused_tiles writes emit_cnt [B,KVH,T_c] (rows emitted per
 *     tile) where launch_fused_tiles_* writes rowmask [B,KVH,L]
 *     (flash/santa_cuda_kernel.cu:514-519), and santa_flash_finalize derives
 *     vrows from it (the reference's launch_reduce_vrows sums the rowmask);
 *   - one entry point per stage takes dtype, block_n and the pass-1 path as
 *     arguments where the reference has one launcher per (dtype, block_n,
 *     path) instantiation;
 *   - santa_prop_pass2 also casts and scales the output (the reference's
 *     launch_cast_scale_out_* is a separate launcher).
 *
 * Layouts (row-major, contiguous):
 *   q   [B, H, D]            (B = 1 for the single-request form [H, D])
 *   K,V [B, L_storage, KVH, D]  (NHD cache; prop: [L, KVH, D])
 *   out [B, H, D] in the input dtype, m_star [B, H] f32, vrows [B, KVH] i32.
 */
#ifndef SANTA_AMD_H_
#define SANTA_AMD_H_

#include <stddef.h>
#include <stdint.h>
#include <hip/hip_runtime_api.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Element type of q, K, V and out (the reference accepts bf16 or f16,
 * flash/santa_cuda.cpp:128-133). */
enum santa_dtype {
  SANTA_BF16 = 0,
  SANTA_F16 = 1,
  SANTA_F32 = 2 /* where an entry says so */
};

/* Return codes.  On failure santa_last_error() holds a message whose text
 * follows the reference's TORCH_CHECK messages where one exists. */
enum santa_status {
  SANTA_OK = 0,
  SANTA_ERR_INVALID = 1,     /* bad shape / argument */
  SANTA_ERR_UNSUPPORTED = 2, /* shape outside what the kernels implement */
  SANTA_ERR_WORKSPACE = 3,   /* workspace too small */
  SANTA_ERR_HIP = 4          /* a HIP launch failed */
};

/* Message of the last failure on the calling thread ("" if none). */
const char* santa_last_error(void);

/* Library version string. */
const char* santa_version(void);

/* ------------------------------------------------------------- flash */

/* Host planning.  L = valid_len > 0 ? valid_len : L_storage; block_n <= 0
 * selects 32 (L <= 1536), 64 (L <= 3072) or 256; T_c = ceil(L / block_n);
 * S_per_tile = S > 0 ? max(1, S / T_c) : 0. */
int santa_flash_plan(int64_t L_storage, int64_t valid_len, int64_t block_n, int64_t S, int* L_out,
                     int* block_n_out, int* T_c_out, int* S_per_tile_out);

/* One fused pass over every (b, kv, tile): scores, tile max / mass, seeded
 * systematic counts, emission compaction and the count-weighted V sum.
 * Outputs (device): m_tiles, ell_tiles [B,H,T_c] f32; out_tiles [B,H,T_c,D]
 * f32; emit_cnt [B,KVH,T_c] i32 (rows emitted per tile; replaces the
 * reference's rowmask); counts [B,H,T_c,block_n] i16 (may be NULL). */
int santa_flash_fused_tiles(const void* q, const void* K, const void* V, int dtype, int B, int H, int KVH,
                            int D, int L_valid, int L_storage, int block_n, int S_per_tile, uint64_t seed,
                            float* m_tiles, float* ell_tiles, float* out_tiles, int* emit_cnt, int16_t* counts,
                            hipStream_t stream);

/* Split-KV merge across tiles: m* = max_t m_t, w_t = exp(m_t - m*) ell_t,
 * out = (sum_t w_t out_t) / (Z S_per_tile) cast to dtype; vrows (may be
 * NULL) = distinct sampled rows per (b, kv). */
int santa_flash_finalize(const float* m_tiles, const float* ell_tiles, const float* out_tiles,
                         const int* emit_cnt, int dtype, int B, int H, int KVH, int D, int T_c, int S_per_tile,
                         void* out, float* m_star, int* vrows, hipStream_t stream);

/* Bytes of device workspace santa_flash_decode needs for this shape on the
 * current device (it depends on the device's compute-unit count). */
size_t santa_flash_workspace_size(int B, int H, int KVH, int D, int T_c);

/* Whole decode step (the production path).  Same results as
 * santa_flash_fused_tiles + santa_flash_finalize for m_star, vrows and every
 * sampled count; the output sum is merged per chunk of tiles with a running
 * max, so `out` agrees with the reference-order merge to rounding.
 * workspace >= santa_flash_workspace_size bytes, 256-B aligned; its contents
 * need no initialization. */
int santa_flash_decode(const void* q, const void* K, const void* V, int dtype, int B, int H, int KVH, int D,
                       int L_valid, int L_storage, int block_n, int S_per_tile, uint64_t seed, void* out,
                       float* m_star, int* vrows, void* workspace, size_t workspace_bytes, hipStream_t stream);

/* The two launches of santa_flash_decode, for callers that schedule them
 * separately: the tile pass writes chunk partials into the workspace, the
 * merge pass reads them. */
int santa_flash_decode_tiles(const void* q, const void* K, const void* V, int dtype, int B, int H, int KVH, int D,
                             int L_valid, int L_storage, int block_n, int S_per_tile, uint64_t seed, void* workspace,
                             size_t workspace_bytes, hipStream_t stream);
int santa_flash_decode_merge(const void* workspace, size_t workspace_bytes, int dtype, int B, int H, int KVH, int D,
                             int T_c, int S_per_tile, void* out, float* m_star, int* vrows, hipStream_t stream);

/* santa_flash_decode without a workspace argument, for callers that cannot
 * allocate device memory (code under HIP graph capture, tight serving
 * loops, harnesses that forbid hipMalloc).  No counterpart in the reference.
 * The workspace lives in a static device array of 16 MiB (16,777,216
 * bytes) that each device holds until the process ends; shapes whose
 * santa_flash_workspace_size exceeds it are rejected with
 * SANTA_ERR_WORKSPACE before anything is launched.  The call makes no hipMalloc / hipFree or other allocation.
 * The array needs no initialisation (every kernel writes what a later one
 * reads).  Every call on a device shares that device's array: calls that
 * overlap on one device (different streams, or host threads) race and must
 * be ordered by the caller.  Results are bit-identical to santa_flash_decode
 * on the same arguments.  Under HIP graph capture: make one uncaptured call
 * on each device first (it takes the scratch array's device address with
 * hipGetSymbolAddress); captured calls then record kernel launches only (no
 * memset or copy nodes), and their replays give the direct call's bits. */
int santa_flash_decode_noalloc(const void* q, const void* K, const void* V, int dtype, int B, int H, int KVH, int D,
                               int L_valid, int L_storage, int block_n, int S_per_tile, uint64_t seed, void* out,
                               float* m_star, int* vrows, hipStream_t stream);

/* Ragged flash (no counterpart in the reference, whose batched call takes
 * one valid_len for every sequence, flash/santa_cuda.cpp:188): sequence b of
 * a [B, L_storage, KVH, D] cache is decoded on its first seq_lens[b] tokens
 * with S_per_tile = S > 0 ? max(1, S / ceil(seq_lens[b] / block_n)) : 0 and
 * RNG key b*H + h -- exactly what the uniform call does when every length
 * equals seq_lens[b].  seq_lens: device int array [B]; max_len = max
 * seq_lens (<= L_storage) and total_tiles = sum over b of
 * ceil(seq_lens[b] / block_n), from the host; one block_n (32, 64 or 256)
 * for every sequence.  out [B,H,D], m_star [B,H], vrows [B,KVH] (may be
 * NULL).  Lengths are clamped on the device to [1, max_len].  Workspace:
 * santa_flash_ragged_workspace_size with max_tiles = ceil(max_len / block_n). */
size_t santa_flash_ragged_workspace_size(int B, int H, int KVH, int D, int max_tiles, long long total_tiles);
int santa_flash_decode_ragged(const void* q, const void* K, const void* V, int dtype, int B, int H, int KVH, int D,
                              int L_storage, const int* seq_lens, int max_len, long long total_tiles, int block_n,
                              int64_t S, uint64_t seed, void* out, float* m_star, int* vrows, void* workspace,
                              size_t workspace_bytes, hipStream_t stream);

/* Paged flash (no counterpart in the reference, which reads contiguous NHD
 * caches only, README.md:257 and tutorial_code/runtime_common.py:340-397):
 * santa_flash_decode_ragged over a page pool K_pages / V_pages
 * [num_pages, page_size, KVH, D] in place of the contiguous cache.  Token n
 * of sequence b is row n % page_size of page
 * block_table[b * table_stride + n / page_size]; block_table is a device int
 * array [B, table_stride] with table_stride >= ceil(max_len / page_size).
 * page_size is a power of two in [8, 2^20].  Page ids are clamped to
 * [0, num_pages) on the device.  Results are bit-identical to the ragged call
 * on the same tokens stored contiguously.  Workspace:
 * santa_flash_ragged_workspace_size(B, H, KVH, D, ceil(max_len / block_n),
 * total_tiles). */
int santa_flash_decode_paged(const void* q, const void* K_pages, const void* V_pages, int dtype, int B, int H, int KVH,
                             int D, int num_pages, int page_size, const int* block_table, int table_stride,
                             const int* seq_lens, int max_len, long long total_tiles, int block_n, int64_t S,
                             uint64_t seed, void* out, float* m_star, int* vrows, void* workspace,
                             size_t workspace_bytes, hipStream_t stream);

/* -------------------------------------------------------------- prop */

/* Host planning.  block_n <= 0 selects 256 when pass1_env is "vec"/"gqa_vec",
 * else the flash heuristic; pass1_path_out = 0 (exact vec path: GH=4, D=128,
 * block_n=256) or 1 (general MFMA path).  pass1_env may be NULL. */
int santa_prop_plan(int L, int H, int KVH, int D, int64_t block_n, const char* pass1_env, int* block_n_out,
                    int* T_c_out, int* pass1_path_out);

/* Pass 1 for one sequence: per-tile max / mass and the u stash [L, H]
 * (16-bit, index n*H + h).  m_tiles, ell_tiles [H, T_c] f32. */
int santa_prop_pass1(const void* q, const void* K, int dtype, int H, int KVH, int D, int L, int block_n,
                     int pass1_path, float* m_tiles, float* ell_tiles, void* u_stash, hipStream_t stream);

/* Largest-remainder tile budgets per head (deterministic Z order):
 * m_star [H]; S_tiles [H,T_c] i32; invdelta, a0 [H,T_c] f32. */
int santa_prop_tile_budgets(const float* m_tiles, const float* ell_tiles, int H, int T_c, int S, uint64_t seed,
                            float* m_star, int* S_tiles, float* invdelta, float* a0, hipStream_t stream);

/* Pass 2 + cast: counts from the stash, count-weighted V sums summed per
 * chunk of tiles in a fixed order (deterministic), out = dtype(sum / S)
 * (0 when S <= 0).  counts [H,T_c,block_n] i16 and vrows [KVH] may be NULL.
 * workspace >= santa_prop_workspace_size bytes (its chunk-partial region is
 * used; contents need no initialization). */
int santa_prop_pass2(const void* V, const void* u_stash, int dtype, int H, int KVH, int D, int L, int block_n,
                     int S, const float* invdelta, const float* a0, int16_t* counts, void* out, int* vrows,
                     void* workspace, size_t workspace_bytes, hipStream_t stream);

/* Bytes of device workspace santa_prop_decode / santa_prop_pass2 need on the
 * current device (m, ell, budgets, the u stash and chunk partials). */
size_t santa_prop_workspace_size(int H, int KVH, int D, int L, int T_c);

/* Whole single-sequence prop decode with the caller's workspace. */
int santa_prop_decode(const void* q, const void* K, const void* V, int dtype, int H, int KVH, int D, int L,
                      int block_n, int pass1_path, int S, uint64_t seed, void* out, float* m_star, int* vrows,
                      void* workspace, size_t workspace_bytes, hipStream_t stream);

/* Batched, ragged santa_prop (no counterpart in the reference, whose adapter
 * loops over sequences, tutorial_code/attention_backends.py:491-500): B
 * sequences of a [B, L_storage, KVH, D] cache, sequence b decoded exactly as
 * santa_prop_decode on its first seq_lens[b] tokens with budget seq_S[b]
 * (RNG key h, as in the per-sequence calls).  seq_lens, seq_S: device int
 * arrays [B]; max_len = max seq_lens; total_tiles = sum over b of
 * ceil(seq_lens[b] / block_n); every sequence uses the same block_n and
 * pass-1 path.  out [B,H,D], m_star [B,H], vrows [B,KVH] (may be NULL). */
size_t santa_prop_batched_workspace_size(int B, int H, int KVH, int D, int L_storage, int max_tiles,
                                         long long total_tiles);
int santa_prop_decode_batched(const void* q, const void* K, const void* V, int dtype, int B, int H, int KVH, int D,
                              int L_storage, const int* seq_lens, const int* seq_S, int max_len, long long total_tiles,
                              int block_n, int pass1_path, uint64_t seed, void* out, float* m_star, int* vrows,
                              void* workspace, size_t workspace_bytes, hipStream_t stream);

/* Paged santa_prop (no counterpart in the reference, which reads contiguous
 * NHD caches only, README.md:257): santa_prop_decode_batched over a page
 * pool K_pages / V_pages [num_pages, page_size, KVH, D], with the block table
 * and page geometry of santa_flash_decode_paged.  Results are bit-identical
 * to the batched call on the same tokens stored contiguously.  Workspace:
 * santa_prop_batched_workspace_size(B, H, KVH, D, max_len, ceil(max_len /
 * block_n), total_tiles). */
int santa_prop_decode_paged(const void* q, const void* K_pages, const void* V_pages, int dtype, int B, int H, int KVH,
                            int D, int num_pages, int page_size, const int* block_table, int table_stride,
                            const int* seq_lens, const int* seq_S, int max_len, long long total_tiles, int block_n,
                            int pass1_path, uint64_t seed, void* out, float* m_star, int* vrows, void* workspace,
                            size_t workspace_bytes, hipStream_t stream);

/* ------------------------------------------------- model-level decode */

/* Fused elementwise steps of the model-level decode loop
 * (santa_amd/runtime.py); the reference runs them as separate torch
 * kernels inside the HF decoder layer (tutorial_code/runtime_common.py:
 * 501-571).  bf16 tensors, rows contiguous.
 *
 * santa_rt_add_rms_norm: per row of h [rows, hidden], h = bf16(h + a) when a
 * is not null, then x = bf16(float(h) * rsqrt(mean(float(h)^2) + eps) *
 * float(w)).
 * santa_rt_rope_write: qkv [B, H + 2 KVH, D] (the fused projection's
 * output); q heads rotated into q_out [B, H, D], k heads rotated into
 * k_cache[b, pos] and v heads copied into v_cache[b, pos] of caches
 * [B, storage, KVH, D]; RoPE in the rotate-half convention with cos, sin
 * [D] and bf16 rounding of each product and of the sum.
 * santa_rt_rope_table: cos_, sin_ [D] bf16 of position pos, the angle of
 * dims i and i + D/2 being pos / theta^(2i / D).
 * santa_rt_rope_write_rows: santa_rt_rope_write for a prefill's P positions
 * pos .. pos + P - 1: qkv [B, P, H + 2 KVH, D], cos, sin [P, D], q_out
 * [B, P, H, D]; D a multiple of 16, every tensor 16-byte aligned.
 * santa_rt_silu_mul: out [rows, inter] = bf16(bf16(silu(gate)) * up), gate
 * and up the two halves of gu [rows, 2 inter].
 * santa_rt_linear: the decode step's weight products (the HF layers'
 * nn.Linear, bf16, no bias): y [M, N] = bf16(x [M, K] . w [N, K]^T),
 * float32 accumulation, for 1 <= M <= 8, K a multiple of 8, M rounded up to
 * 1, 2, 4 or 8 times K rounded up to 2048 at most 65536, x and w 16-byte
 * aligned.  swiglu != 0: w is [2N, K] (gate rows, then up rows) and
 * y [M, N] = bf16(bf16(silu(bf16(g))) * bf16(u)), silu_mul of the product.
 * The weights are read once at the HBM bound.
 * santa_rt_linear_f32: santa_rt_linear's product with its float32 sums as the
 * output, y [M, N] float32 (the logits of the head).
 * santa_rt_linear_rope: the fused q/k/v projection of rows x [M, K] by
 * w [(H + 2 KVH) D, K] (head by head) with santa_rt_rope_write's epilogue
 * applied to the bf16 products: q heads rotated into q_out [M, H, D], k heads
 * rotated into k_cache[b, pos], v heads into v_cache[b, pos] (caches
 * [M, storage, KVH, D]); bit for bit santa_rt_rope_write of santa_rt_linear's
 * output, without writing that output.  D even; the santa_rt_linear limits
 * on M and K.
 * santa_rt_causal_attention: exact causal GQA attention of a prefill, D = 128
 * (the HF model's own attention in the reference's prefill,
 * tutorial_code/runtime_common.py:501-571): q [B, P, H, D], k, v [B, P, KVH,
 * D], out [B, P, H, D] of one 16-bit type (enum santa_dtype); strides: 12 host
 * values, the batch, position and head strides in elements of q, k, v, out
 * (multiples of 8, positions at least D apart, the last dimension contiguous,
 * the tensors 16-byte aligned).  Scores, softmax and sums in float32, the probabilities rounded
 * to the 16-bit type for the second product.
 * santa_rt_exact_decode: exact decode attention in float32, D = 128: q, out
 * [B, H, D] contiguous, k, v [B, L.., KVH, D] of which the first L positions
 * count, one 16-bit type (enum santa_dtype); strides: 6 host values, the
 * batch, position and head strides in elements of k and v (multiples of 8,
 * positions at least D apart, the last dimension contiguous, the tensors
 * 16-byte aligned).  workspace:
 * santa_rt_exact_decode_workspace_size bytes, 16-byte aligned, needing no
 * initialization.
 * santa_rt_argmax: out[r] (int64) = the index of the maximum of row r of
 * x [rows, n] (float32), torch.argmax's choice: NaN above any number, the
 * first index among equal values; the greedy step's token choice
 * (tutorial_code/runtime_common.py:574-675). */
int santa_rt_add_rms_norm(void* h, const void* a, const void* w, void* x, int rows, int hidden, float eps,
                          hipStream_t stream);
int santa_rt_rope_write(const void* qkv, const void* cos_, const void* sin_, void* q_out, void* k_cache, void* v_cache,
                        int B, int H, int KVH, int D, long long storage, int pos, hipStream_t stream);
int santa_rt_rope_table(int pos, float theta, int D, void* cos_, void* sin_, hipStream_t stream);
int santa_rt_rope_write_rows(const void* qkv, const void* cos_, const void* sin_, void* q_out, void* k_cache,
                             void* v_cache, int B, int P, int H, int KVH, int D, long long storage, int pos,
                             hipStream_t stream);
int santa_rt_silu_mul(const void* gu, void* out, int rows, int inter, hipStream_t stream);
int santa_rt_linear(const void* x, const void* w, void* y, int M, int N, int K, int swiglu, hipStream_t stream);
int santa_rt_linear_f32(const void* x, const void* w, float* y, int M, int N, int K, hipStream_t stream);
int santa_rt_linear_rope(const void* x, const void* w, int M, int K, const void* cos_, const void* sin_, void* q_out,
                         void* k_cache, void* v_cache, int H, int KVH, int D, long long storage, int pos,
                         hipStream_t stream);
int santa_rt_argmax(const float* x, int rows, int n, long long* out, hipStream_t stream);
int santa_rt_causal_attention(const void* q, const void* k, const void* v, void* out, int dtype, int B, int P, int H,
                              int KVH, int D, const long long* strides, hipStream_t stream);
size_t santa_rt_exact_decode_workspace_size(int B, int L, int H, int KVH);
int santa_rt_exact_decode(const void* q, const void* k, const void* v, void* out, int dtype, int B, int L, int H,
                          int KVH, int D, const long long* strides, void* workspace, size_t workspace_bytes,
                          hipStream_t stream);

/* ------------------------------------------------------- shared paged caches */

/* A paged KV cache that sequences share, and the exact attention that reads it
 * (santa_amd/paged.py).  No counterpart in the reference, whose caches are
 * contiguous and one per sequence (tutorial_code/runtime_common.py:340-397).
 * Pages and block tables are those of santa_flash_decode_paged: K and V pools
 * [num_pages, page_size, KVH, D], token n of sequence s in row n % page_size of
 * page table[s][n / page_size], page_size a power of two in [8, 2^20].
 *
 * santa_pages: host bookkeeping of max_seqs sequences over num_pages pages, a
 * sequence holding at most row_pages of them.  An object is used by one host
 * thread at a time.  Every call either does all it is asked or fails and
 * changes nothing.
 *   _add: n new sequences of lengths[i] tokens, in the lowest free rows of the
 *     table, written to seqs; pages are taken lowest number first.
 *   _extend: tokens[i] more tokens for seqs[i] (each named once).  A last page
 *     that is partly filled and held by other sequences too is replaced by a
 *     copy.
 *   _shrink: the last tokens[i] tokens of seqs[i] (each named once) leave it, and
 *     it gives up the pages that hold none of those left.
 *   _keep: of the last new_tokens[i] tokens of seqs[i] (each named once) the
 *     counts[i] of those numbers stay that kept names (one sequence's after the
 *     other's, ascending), and move up behind the tokens before; the others leave.
 *     What moves must not be in pages that other sequences hold.
 *   _fork: n new sequences that hold every page of seq.
 *   _free: the sequences end; a page that none holds is free.
 *   _compact: with n pages in use, those numbered n and above move to the
 *     numbers below n that are free, both in ascending order.
 * What a call asks of the device is returned by _changes until the next call:
 * page copies [n][2] (source, destination), edits of the block table [n][4]
 * (row, first entry, count, value: entry first + i becomes value + i or, for a
 * negative value, entry first + i of row -1 - value), and whether every table
 * entry that is a copy's source becomes its destination.  _moves: the rows that
 * _keep moves, [n][5]: page and row of the source, page and row of the destination,
 * the sequence's number (0, 1, ...); those of a sequence are carried out in order.
 * _length: tokens of a sequence (-1: no such sequence); _page_size: as created;
 * _used: pages in use;
 * _row: a sequence's pages, returns how many.
 * _shared: groups of the sequences seqs whose first tokens lie in the same pages,
 * the last own[i] >= 0 tokens of each apart: group[i] is a group or -1, shared[g] the
 * tokens that group g has in common (shared: room for n / 2). */
typedef struct santa_pages santa_pages;
int santa_pages_create(int num_pages, int page_size, int max_seqs, int row_pages, santa_pages** out);
void santa_pages_destroy(santa_pages* p);
int santa_pages_add(santa_pages* p, const int* lengths, int n, int* seqs);
int santa_pages_extend(santa_pages* p, const int* seqs, const int* tokens, int n);
int santa_pages_shrink(santa_pages* p, const int* seqs, const int* tokens, int n);
int santa_pages_keep(santa_pages* p, const int* seqs, const int* new_tokens, const int* kept, const int* counts, int n);
int santa_pages_moves(const santa_pages* p, const int** moves, int* n);
int santa_pages_page_size(const santa_pages* p);
int santa_pages_fork(santa_pages* p, int seq, int n, int* seqs);
int santa_pages_free(santa_pages* p, const int* seqs, int n);
int santa_pages_compact(santa_pages* p);
int santa_pages_changes(const santa_pages* p, const int** copies, int* n_copies, const int** edits, int* n_edits,
                        int* remap);
int santa_pages_length(const santa_pages* p, int seq);
int santa_pages_used(const santa_pages* p);
int santa_pages_row(const santa_pages* p, int seq, const int** pages);
int santa_pages_shared(const santa_pages* p, const int* seqs, const int* own, int n, int* group, int* shared,
                       int* n_groups);

/* Page copies: in each of n_pools pools (page i page_stride bytes from page
 * i - 1), pairs[j][0] to pairs[j][1] for j < n.  pools and pairs are host
 * arrays, read before the call returns.  No page is written twice or both read
 * and written; page_bytes, page_stride and the pools' addresses are multiples
 * of 16. */
int santa_paged_copy(const void* const* pools, int n_pools, long long page_bytes, long long page_stride, int num_pages,
                     const int* pairs, int n, hipStream_t stream);
/* The last call's page copies in the pools and its edits in the device block
 * table [max_seqs, table_stride], on `stream`. */
int santa_pages_apply(const santa_pages* p, const void* const* pools, int n_pools, long long page_bytes,
                      long long page_stride, int* table, long long table_stride, int max_seqs, hipStream_t stream);
/* The rows that the last call, santa_pages_keep, moves, in every pool (whose
 * pages are rows of page_bytes / page_size bytes). */
int santa_pages_apply_moves(const santa_pages* p, const void* const* pools, int n_pools, long long page_bytes,
                            long long page_stride, hipStream_t stream);

/* Attention plan: how the work of santa_paged_attention is cut up for one set
 * of lengths, built on the host once and used by every layer.  Sequence b
 * holds lens[b] tokens, the last new_tokens[b] of which have queries, in block
 * table row rows[b] (rows NULL: b).  The sequences with group[b] = g >= 0
 * (group NULL: none) have their first shared[g] tokens in common, no more than
 * precede every member's queries; the pages of one of the members are
 * read for all.  fixed != 0: items and the workspace are sized so that any
 * other lengths with the same new_tokens and groups give a plan of the same
 * info but for max_len (for captured graphs whose plan changes between replays,
 * up to the lengths that the captured calls' block tables have room for).  info is
 * always written; plan (info->ints ints, 16-byte aligned, to be copied to the
 * device as it is) where it is not NULL.  Workgroups are planned for the current
 * device. */
typedef struct santa_paged_plan_info {
  int tokens;       /* queries: the sum of new_tokens */
  int groups;       /* workgroups per KV head, and the items they work through */
  int items;
  int merge_tokens; /* tokens whose output is joined from parts */
  int max_len, max_row; /* what the block table has to hold */
  int heads, kv_heads;
  long long records; /* parts: rows of the workspace */
  long long ints, pos_at, merge_at, parts_at, list_at; /* ints of the plan, and where its sections start */
  int rounded; /* 0, 1 or 2: how probabilities enter the second product (santa_paged_attention) */
  int tree_ints;     /* of a token's record in a plan with trees, 0 in others */
  long long tree_at; /* where the records start */
} santa_paged_plan_info;
int santa_paged_plan(const int* lens, const int* new_tokens, const int* rows, int B, const int* group,
                     const int* shared, int n_groups, int heads, int kv_heads, int fixed, santa_paged_plan_info* info,
                     int* plan, long long plan_ints);
/* The same where the new tokens of sequences b with trees[b] != 0 are drafts that
 * follow one another as trees, up to 8192 each: parents (one int per new token of
 * the batch, those of other sequences not read) names the earlier new token of the
 * sequence that a token follows, -1: the context (the tokens before the new ones),
 * -2: not in use, and followed by none.  A token attends to the context, the
 * tokens that it follows up to there, and itself; one that is not in use is not
 * written, attends to nothing and gives zeros, as all do of a sequence shorter
 * than its tree.  Tokens lie in the cache one after the other; a token's position
 * is the context's length and one for every drafted token that it follows.
 * A token's record is tree_ints ints from plan[tree_at + token * tree_ints] on: the context
 * tokens it attends to, its position (-1: not in use), and a bit for each place
 * from the last multiple of 64 up to the context's end on (bit n % 32 of int
 * n / 32 behind): whether it attends to that token. */
int santa_paged_tree_plan(const int* lens, const int* new_tokens, const int* rows, int B, const int* group,
                          const int* shared, int n_groups, int heads, int kv_heads, int fixed, const int* trees,
                          const int* parents, santa_paged_plan_info* info, int* plan, long long plan_ints);

/* Exact attention over pages, D = 64 or 128: query i of sequence b (row
 * sum of the earlier new_tokens + i of q [tokens, H, D]) attends to the tokens
 * 0 .. lens[b] - new_tokens[b] + i of its sequence; one that has none gives
 * zeros.  out [tokens, H, D] contiguous.  strides: 8 host values, q's token and
 * head strides, K's page, row and head strides and V's, in elements (multiples
 * of 8, the last dimension contiguous, the tensors 16-byte aligned).  plan: the
 * device copy of a plan with this info.  scale: positive and finite.  Page
 * numbers are clamped to the pool.
 * Scores, softmax and sums in float32.  The probabilities enter the second
 * product as the sum of two values of the 16-bit type, with a product each, or,
 * where info->rounded is 1 and more than 16 rows share a pass over a KV head's
 * tokens, rounded to one.  A plan sets rounded to 1 where a sequence has several new
 * tokens and more than 32 rows (tokens x query heads per KV head), and a plan with
 * trees to 2 then: those of trees are not rounded (but a tree that is one chain and
 * shares no prefix is the sequence that it is without a tree), and the other sequences'
 * are where one of these has that many rows.  A copy of info with 0 or 1 may be given to
 * any call.  workspace:
 * santa_paged_workspace_size(info, D) bytes, 16-byte aligned, no initialization
 * needed. */
size_t santa_paged_workspace_size(const santa_paged_plan_info* info, int D);
int santa_paged_attention(const void* q, const void* k_pages, const void* v_pages, void* out, int dtype, int D,
                          int num_pages, int page_size, const long long* strides, const int* table,
                          long long table_stride, int table_rows, const santa_paged_plan_info* info, const int* plan,
                          float scale, void* workspace, size_t workspace_bytes, hipStream_t stream);

/* RoPE of new tokens with their write into pages: qkv [tokens, H + 2 KVH, D]
 * contiguous, cos_, sin_ [tokens, D], one 16-bit type; q heads rotated into
 * q_out [tokens, H, D], k heads rotated and v heads copied into the pages of
 * their tokens (tokens of a plan; strides: K's page, row and head strides and
 * V's, as above).  Rotate-half convention, float32, rounded once.  D a multiple of 16, every
 * tensor 16-byte aligned.  A token of a negative position is not written. */
int santa_paged_rope_append(const void* qkv, const void* cos_, const void* sin_, void* q_out, void* k_pages,
                            void* v_pages, int dtype, int D, int num_pages, int page_size, const long long* strides,
                            const int* table, long long table_stride, int table_rows,
                            const santa_paged_plan_info* info, const int* plan, hipStream_t stream);

/* The same for heads that are normed first, and rotated in part or in the other
 * layout: with q_norm, k_norm (NULL: none; q_norm_heads rows of D, one or H, and
 * k_norm_heads, one or KVH), x / sqrt(mean(x^2) + eps) * w over the D dims of every q
 * and k head; then a rotation of its first R dims, R even, by cos_, sin_ [tokens, R]:
 * dims d and d + R / 2 or, interleaved, 2d and 2d + 1 belong together.  float32,
 * rounded once.  D up to 512. */
int santa_paged_heads_append(const void* qkv, const void* cos_, const void* sin_, int R, int interleaved,
                             const void* q_norm, int q_norm_heads, const void* k_norm, int k_norm_heads, float eps,
                             void* q_out, void* k_pages, void* v_pages, int dtype, int D, int num_pages, int page_size,
                             const long long* strides, const int* table, long long table_stride, int table_rows,
                             const santa_paged_plan_info* info, const int* plan, hipStream_t stream);
/* magnitude times cos and sin of 2 pi x positions[i * stride] x turns[p], i < n, p <
 * pairs (up to 256; turns: host array, read before the call returns), to dims p and
 * p + pairs of cos_, sin_ [n, 2 pairs] or, interleaved, 2p and 2p + 1.  positions: int
 * or, wide, 64-bit.  dtype: bf16, f16 or float32; tables 16-byte aligned.  Angles in
 * float64. */
int santa_rope_tables(const void* positions, int wide, long long stride, long long n, const double* turns, int pairs,
                      float magnitude, int interleaved, int dtype, void* cos_, void* sin_, hipStream_t stream);

/* ----------------------------------------------------------- rules on logits */

/* What santa_adjust_logits applies to row r of sequence s (the block table row that
 * a plan's token r belongs to; without a plan s = r).  NULL pointers: not applied.
 *   tokens [tokens_rows, tokens_len] (int, or 64-bit where tokens_wide; rows
 *     tokens_stride entries apart): the tokens of every sequence.  A row has seen
 *     those that its token of the plan attends to.
 *   prompts[s]: how many of a sequence's first tokens are its prompt's (NULL: 0);
 *     the others and all drafted ones are the answer's.
 *   repetition, frequency, presence: [s], or where NULL the values _all.
 *   bias_ids, bias: biases entries of sequence s from entry s * bias_stride on (0:
 *     the same for all); ids outside of the vocabulary count for nothing, and of a
 *     token named twice the last entry counts.  Up to 2046.
 *   allowed: bit v % 32 of int r * allowed_stride + v / 32 (0: the same for all rows):
 *     whether token v may come. */
typedef struct santa_logit_rules {
  const void* tokens;
  int tokens_wide, tokens_rows, tokens_len;
  long long tokens_stride;
  const int* prompts;
  const float *repetition, *frequency, *presence;
  float repetition_all, frequency_all, presence_all;
  const int* bias_ids;
  const float* bias;
  int biases;
  long long bias_stride;
  const int* allowed;
  long long allowed_stride;
  int sequences; /* how many sequences the rows are of, 0: as many as rows; how the work is cut up goes by it */
} santa_logit_rules;

/* Row by row of x [N, V] (bf16, f16 or float32, rows stride elements apart), in
 * float32: a token that the row has seen has its logit divided by the repetition
 * penalty where it is positive and multiplied by it elsewhere; one that is in the
 * answer c > 0 times loses c times the frequency penalty and once the presence
 * penalty; then the bias is added; one that may not come is -inf.  Either out [N, V]
 * (float32, contiguous) is written or token [N]: the index of the row's maximum, NaN
 * above any number, the first one among equal values.  info, plan: those of a
 * santa_paged_plan of N tokens, plan 16-byte aligned, or NULL; all other arrays are
 * aligned to their elements.  At most 2^19 - 1 tokens are counted.
 * workspace (for token): santa_adjust_logits_workspace_size bytes for these N, V and
 * rules->sequences, 8-byte aligned, no initialization needed. */
size_t santa_adjust_logits_workspace_size(int N, int V, int sequences);
int santa_adjust_logits(const void* x, int dtype, long long stride, int N, int V, const santa_logit_rules* rules,
                        const santa_paged_plan_info* info, const int* plan, float* out, long long* token,
                        void* workspace, size_t workspace_bytes, hipStream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* SANTA_AMD_H_ */
