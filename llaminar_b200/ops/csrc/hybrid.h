// Launchers of the hybrid family's blocks: the gated delta rule over several rows of every sequence (gdn_rows.cu, gdn_chunk.cu),
// the rotation of a part of every head with the append to the paged cache (rope_part.cu); and decode attention of a batch behind a shared prefix
// (attn_shared.cu).
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace llm {

// The gated delta rule over packed rows.  Row r of `in` holds q | k | v in columns [0, C), the gate z from z_off and (alpha | beta) from
// ab_off; C = (2 n_k + n_v) d.  Rows cu[b] .. cu[b + 1] are sequence b's (cu nullptr: `rows_per_seq` rows each), its state the slot
// slots[b] of conv [n_slots, C, K - 1] and rec [n_slots, n_v, d, d]; a sequence whose first row has position 0 starts from zeros
// (positions nullptr: none does).
struct GdnParams {
    const __nv_bfloat16* in; size_t in_row;
    int C, z_off, ab_off, K, n_k, n_v, d, v_head_offset;
    const float *conv_w, *ssm_a, *dt_bias, *norm_w;          // [C, K], [n_v], [n_v], [d]
    float *conv, *rec;
    const int *positions, *cu, *slots;
    int n_seqs, rows_per_seq, n_slots, n_rows;               // n_rows: rows of `in` and `out`
    __nv_bfloat16* out; size_t out_row;                      // [rows, n_v d]
    float eps;
    // what a pass that leaves the state alone keeps for gdn_commit, all [n_seqs, rows_per_seq, ...]: decay [n_v], key [n_v, d], correction [n_v, d]
    // and the convolution's inputs [C]
    float *keep_a, *keep_k, *keep_u;
    __nv_bfloat16* keep_x;
    int* status;                                             // drafted rows: receives STATUS_TIMEOUT if a wait gave up
};
// rows one after the other, any number of them; d of 32, 64 or 128.  With keep_*: the state stays as it is.
cudaError_t launch_gdn_rows(const GdnParams& p, cudaStream_t st);
// the convolution windows behind the sequences' rows; to run after everything that reads the old ones
cudaError_t launch_gdn_windows(const GdnParams& p, cudaStream_t st);
// states and windows advanced by the first accepted[b] of the kept rows (0: as they were)
cudaError_t launch_gdn_commit(const GdnParams& p, const int* accepted, cudaStream_t st);

// the same for prompts, chunk-parallel on the tensor cores; d = 128.  `workspace` (1024-byte aligned) holds as many chunks as it has room for, at
// least one; `status` receives STATUS_TIMEOUT if a wait gave up.  (Windows are left to launch_gdn_windows here too.)
size_t gdn_chunk_bytes(int units, int n_k, int n_v);
cudaError_t launch_gdn_chunk(const GdnParams& p, void* workspace, size_t bytes, int* status, int& launches, cudaStream_t st);

// Rows [(query, gate) per head | keys | values] -> normed and rotated queries, and the tokens' entries of the paged cache (bf16: [n_pages, 2, n_kv_heads, 64, head_dim];
// 8-bit: as in AttnDecodeParams, ops.h)
struct RopePartParams {
    const __nv_bfloat16* rows; size_t row;                   // first row, values from one to the next
    int whole;                                               // a lane's values may be loaded at once
    int q_stride;                                            // values from a query head to the next: head_dim, or twice that with gates
    const float *q_norm, *k_norm;                            // [head_dim] or nullptr
    const double* freqs;                                     // [rot / 2], angle per position
    float magnitude;
    int rot, interleaved;
    const int *positions, *seq_ids, *block_table;
    int n_tokens, n_heads, n_kv_heads, head_dim, max_pages, n_seqs, n_pages;
    __nv_bfloat16* q_out;                                    // [n_tokens, n_heads, head_dim]
    uint8_t* kv; size_t page_bytes, scale_off;
    int q8;
    float eps;
    int parts;                                               // warps that share a token (the launcher's choice)
};
cudaError_t launch_rope_part(const RopePartParams& p, cudaStream_t st);

struct AttnSharedParams {
    const __nv_bfloat16 *q, *kv;   // [n_seqs * rows_per_seq, n_heads, head_dim], [n_pages, 2, n_kv_heads, 64, head_dim]
    __nv_bfloat16* out;            // as q
    const int *block_table, *seq_lens, *shared_len;          // [n_seqs, max_pages], [n_seqs], one number
    int n_seqs, rows_per_seq, n_heads, n_kv_heads, head_dim, max_pages, n_pages;
    int prefix_row;                // row of block_table whose first pages are the prefix
    float scale;
    const __nv_bfloat16* gate; size_t gate_token, gate_head;         // optional: values from a token / a head to the next
    int splits, tail_splits;       // parts of the prefix's keys (0: no prefix) and of a tail's
    float *part_o, *part_ml, *tail_o, *tail_ml;              // rows of the plan: head_dim values; maximum and sum
    unsigned* tickets;             // [n_seqs * n_kv_heads], zero between calls (more than one part)
};
struct AttnSharedPlan { int splits, tail_splits; long long prefix_rows, tail_rows; };
AttnSharedPlan attn_shared_plan(int n_seqs, int rows_per_seq, int n_heads, int n_kv_heads, int head_dim, int max_shared, int max_tail, int max_tickets);
cudaError_t launch_attn_shared(const AttnSharedParams& p, int* status, cudaStream_t st);

int bounds_status_attn_shared(bool reset);
int bounds_status_rope_part(bool reset);
int bounds_status_gdn_rows(bool reset);
int bounds_status_gdn_chunk(bool reset);

}  // namespace llm
