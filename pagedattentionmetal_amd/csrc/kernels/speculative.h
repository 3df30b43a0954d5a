// speculative.h - launch interface of the kernels of a speculative-decoding step:
// batch plans, norm and rotation of query and key heads with their gradients,
// attention of drafted trees and the commit of an accepted path.
#pragma once
#include "kernels.h"

namespace pam {

// ------------------------------------------------------------------ batch plan

constexpr int kPlanMaxNodes = 1024;  // drafted tokens of one tree (its parents lie in LDS)

// bits of BatchPlanParams::status
enum PlanStatus : int32_t {
    kPlanRows = 1,      // more rows than max_rows
    kPlanBlocks = 2,    // a sequence needs more blocks than the table's width or the block list holds
    kPlanLength = 4,    // a negative length (taken as 0)
    kPlanTree = 8,      // a parent that is not an earlier node (taken as -1), or a tree past its limits
};

struct BatchPlanParams {
    const int32_t *context_lens, *query_lens;  // [num_seqs]
    const int32_t *block_list;                 // the sequences' blocks, one after another
    const int32_t *parents;                    // [parents_len] or null (chains)
    int64_t block_list_len, parents_len;
    int32_t num_seqs, block_size, max_num_blocks, max_rows, mask_words;
    int32_t seqs_per_group;
    int32_t *cu_queries;       // [num_seqs + 1]
    uint32_t *seq_lengths;     // [num_seqs]
    int32_t *block_tables;     // [num_seqs][max_num_blocks]
    int32_t *positions;        // [max_rows]
    int64_t *slot_mapping;     // [max_rows]
    uint64_t *tree_mask;       // [max_rows][mask_words] or null
    int32_t *status;           // or null
};
hipError_t launch_batch_plan(const BatchPlanParams &p, hipStream_t stream);

// ------------------------------------------------------------------ norm and rotation

constexpr int kMaxRotaryPairs = 128;

struct NormRopeParams {
    // rows of heads; row strides in elements, heads contiguous
    const void *q, *k, *v;
    void *q_out, *k_out;         // k_out may be null (keys go to the pool alone)
    const void *dq_out, *dk_out; // backward: the outputs' gradients
    const void *q_weight, *k_weight;  // [head_dim] or null (ones)
    const int32_t *positions;
    const int64_t *slot_mapping; // with the pools: the slot of each token, < 0: none
    void *k_pool, *v_pool;       // or null
    float *partial;              // backward: [groups][2][head_dim] weight-gradient sums
    float *d_q_weight, *d_k_weight;
    int64_t q_stride, k_stride, v_stride, q_out_stride, k_out_stride, dq_stride, dk_stride;
    int64_t pool_slots;          // slots of the pools (0: not known)
    int32_t num_tokens, num_heads, num_kv_heads, head_dim, rotary_dim, interleaved, normalize;
    int32_t groups;              // backward: workgroups
    float eps;
    // a pair's turns per position, as a 64-bit binary fraction: position * freq wraps
    // to the fraction of a turn without rounding
    uint64_t freq[kMaxRotaryPairs];
};
hipError_t launch_norm_rope(const NormRopeParams &p, int32_t dtype, int32_t cus, hipStream_t stream);
// Workgroups of the backward (each leaves one partial sum of both weights' gradients).
int32_t norm_rope_backward_groups(const NormRopeParams &p, int32_t dtype, int32_t cus);
hipError_t launch_norm_rope_backward(const NormRopeParams &p, int32_t dtype, hipStream_t stream);

// ------------------------------------------------------------------ tree attention

struct TreeParams {
    AttnParams a;                 // queries, pools, tables, shapes, scale, partials
    const int32_t *context_lens;  // [num_seqs]
    const int32_t *cu_queries;    // [num_seqs + 1]
    const uint64_t *tree_mask;    // [total_rows][mask_words] or null (chains)
    int32_t mask_words, num_seqs, max_queries, total_rows;
    int32_t pool_blocks;          // blocks of the pools: table entries are held below it
    // the split (tree_plan): `groups` workgroups share all units equally
    int32_t form, block_rows, rows_log2, keys_log2, groups;
};
enum TreeForm : int32_t { kTreeRow = 0, kTreeRowBlocks = 1, kTreeMfma = 2 };
// Chooses the kernel and the split; returns the bytes of partials it needs (a.part_o,
// 16-byte aligned), 0: none.
int64_t tree_plan(TreeParams &p, int32_t dtype, int32_t cus);
hipError_t launch_tree_attention(const TreeParams &p, int32_t dtype, hipStream_t stream);

// ------------------------------------------------------------------ commit

struct TreeCommitParams {
    void *k_pool, *v_pool;
    uint16_t *k_scale, *v_scale;
    const int32_t *block_tables, *context_lens, *query_lens, *paths;
    int32_t *new_lengths;         // or null
    int32_t num_seqs, max_num_blocks, max_path, num_kv_heads, head_dim, block_size, pool_blocks;
};
hipError_t launch_tree_commit(const TreeCommitParams &p, int32_t dtype, hipStream_t stream);

}  // namespace pam
