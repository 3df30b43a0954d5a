// batch_plan.hip - block tables, slot maps, positions and tree masks of a ragged
// batch, built on the GPU from the sequences' lengths (gfx950).
//
// Sequence s holds c_s cached tokens and gets n_s new ones.  With L_s = c_s + n_s and
// ceil(L_s / bs) blocks, taken from the flat block list one sequence after another:
//   cu[s] = sum_{t < s} n_t,   first_s = sum_{t < s} ceil(L_t / bs)
//   table[s][j] = list[first_s + j]  (0 behind the sequence's blocks)
//   row cu[s] + i:  slot = table[s][(c_s + i) / bs] * bs + (c_s + i) % bs,
//                   position = c_s + depth(i), mask bit j: node j is on node i's path
// A chain's depth is i; a tree's is found by walking its parents, which lie in LDS.
// Parents come before their children, so the walk meets the path's bits in falling
// order and leaves every mask word once.
//
// What bounds it: latency (launch, the lengths' loads, one reduction, the block list's
// loads); a serving batch is under 1 MB (8 sequences: 3.9 us; 256 with trees of 8 to 64 nodes,
// 0.67 MB: 5.6 us).  A workgroup takes a few consecutive sequences
// and adds up the lengths before them itself, so the whole plan is one launch: 1024
// groups at most read 1024 / 2 times the lengths, from L2.
#include <algorithm>

#include "speculative.h"

namespace pam {

constexpr int kPlanThreads = 256;
constexpr int kPlanGroups = 1024;  // most workgroups along the sequences

// sums of both values over the workgroup's threads, the same in every thread
__device__ __forceinline__ void plan_sum(int64_t &a, int64_t &b, int64_t (*red)[2]) {
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) {
        a += __shfl_xor(a, m, 64);
        b += __shfl_xor(b, m, 64);
    }
    const int wave = threadIdx.x >> 6;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[wave][0] = a, red[wave][1] = b;
    __syncthreads();
    a = b = 0;
#pragma unroll
    for (int w = 0; w < kPlanThreads / 64; w++) a += red[w][0], b += red[w][1];
}

struct PlanSeq {
    int64_t c, n, blocks;
    int32_t bad;
};
__device__ __forceinline__ PlanSeq plan_seq(const BatchPlanParams &p, int s) {
    PlanSeq q;
    q.c = p.context_lens[s], q.n = p.query_lens[s];
    q.bad = (q.c < 0 || q.n < 0) ? kPlanLength : 0;
    if (q.c < 0) q.c = 0;
    if (q.n < 0) q.n = 0;
    q.blocks = (q.c + q.n + p.block_size - 1) / p.block_size;
    return q;
}

// grid: x = groups of seqs_per_group sequences, y = pieces of every sequence's work
__global__ __launch_bounds__(kPlanThreads) void batch_plan_kernel(BatchPlanParams p) {
    __shared__ int64_t red[kPlanThreads / 64][2];
    __shared__ int32_t par[kPlanMaxNodes];
    const int tid = threadIdx.x, bs = p.block_size, W = p.max_num_blocks, words = p.mask_words;
    const int s0 = blockIdx.x * p.seqs_per_group;
    const int s1 = s0 + p.seqs_per_group < p.num_seqs ? s0 + p.seqs_per_group : p.num_seqs;
    const bool lead = blockIdx.y == 0 && tid == 0;
    const int first = blockIdx.y * kPlanThreads + tid, step = gridDim.y * kPlanThreads;
    int32_t flags = 0;

    int64_t rows = 0, blocks = 0;  // before the sequence at hand
    for (int s = tid; s < s0; s += kPlanThreads) {
        const PlanSeq q = plan_seq(p, s);
        rows += q.n;
        blocks += q.blocks;
    }
    plan_sum(rows, blocks, red);

    for (int s = s0; s < s1; s++) {
        const PlanSeq q = plan_seq(p, s);
        flags |= q.bad;
        if (q.blocks > W || blocks + q.blocks > p.block_list_len) flags |= kPlanBlocks;
        if (rows + q.n > p.max_rows) flags |= kPlanRows;
        // blocks that both the table and the list hold
        int64_t held = q.blocks < W ? q.blocks : W;
        if (held > p.block_list_len - blocks) held = p.block_list_len > blocks ? p.block_list_len - blocks : 0;
        if (lead) {
            p.cu_queries[s] = (int32_t)(rows < p.max_rows ? rows : p.max_rows);
            const int64_t len = q.c + q.n, cap = (int64_t)W * bs;
            p.seq_lengths[s] = (uint32_t)(len < cap ? len : cap);
        }
        int32_t *bt = p.block_tables + (int64_t)s * W;
        for (int j = first; j < W; j += step) bt[j] = j < held ? p.block_list[blocks + j] : 0;

        // drafted trees: the sequence's parents in LDS, -1 for a root
        const int64_t limit = p.tree_mask ? (int64_t)words * 64 : (int64_t)1 << 40;
        const int64_t nodes = p.parents ? (q.n < kPlanMaxNodes ? q.n : kPlanMaxNodes) : q.n;
        if (q.n > nodes || q.n > limit) flags |= kPlanTree;
        if (p.parents) {
            __syncthreads();
            for (int i = tid; i < (int)nodes; i += kPlanThreads) {
                const int64_t at = rows + i;
                int32_t v = at < p.parents_len ? p.parents[at] : -2;
                if (v < -1 || v >= i) flags |= kPlanTree, v = -1;
                par[i] = v;
            }
            __syncthreads();
        }
        const int64_t end = rows + q.n < p.max_rows ? rows + q.n : p.max_rows;
        for (int64_t r = rows + first; r < end; r += step) {
            const int64_t i = r - rows, tok = q.c + i, lb = tok / bs;
            uint64_t *mask = p.tree_mask ? p.tree_mask + r * words : nullptr;
            const bool in = i < nodes && i < limit;
            int64_t depth = p.parents ? 0 : i;
            if (mask && (!in || !p.parents)) {
                for (int w = 0; w < words; w++) {
                    const int64_t below = in ? i + 1 - (int64_t)w * 64 : 0;  // a chain's bits of this word
                    mask[w] = below <= 0 ? 0ull : (below >= 64 ? ~0ull : (1ull << below) - 1);
                }
            } else if (p.parents && in) {
                int w = mask ? words - 1 : 0;
                uint64_t bits = 0;
                depth = -1;
                for (int node = (int)i; node >= 0; node = par[node]) {
                    depth++;
                    if (mask) {
                        for (; w > node >> 6; w--) mask[w] = bits, bits = 0;
                        bits |= 1ull << (node & 63);
                    }
                }
                if (mask)
                    for (; w >= 0; w--) mask[w] = bits, bits = 0;
            }
            p.positions[r] = (int32_t)(q.c + depth);
            p.slot_mapping[r] = in && lb < held ? (int64_t)p.block_list[blocks + lb] * bs + tok % bs : -1;
        }
        rows += q.n;
        blocks += q.blocks;
    }

    if (s1 == p.num_seqs) {  // the last group: the total, and the rows behind it
        if (lead) p.cu_queries[p.num_seqs] = (int32_t)(rows < p.max_rows ? rows : p.max_rows);
        for (int64_t r = rows + first; r < p.max_rows; r += step) {
            p.positions[r] = 0;
            p.slot_mapping[r] = -1;
            if (p.tree_mask)
                for (int w = 0; w < words; w++) p.tree_mask[r * words + w] = 0;
        }
    }
    if (p.status && flags) atomicOr(p.status, flags);
}

hipError_t launch_batch_plan(const BatchPlanParams &p_in, hipStream_t stream) {
    BatchPlanParams p = p_in;
    if (p.num_seqs <= 0 || p.block_size <= 0 || p.max_num_blocks <= 0 || p.max_rows <= 0 ||
        (p.tree_mask && (p.mask_words <= 0 || p.mask_words > kPlanMaxNodes / 64)))
        return hipErrorInvalidValue;
    p.seqs_per_group = (p.num_seqs + kPlanGroups - 1) / kPlanGroups;
    const int groups = (p.num_seqs + p.seqs_per_group - 1) / p.seqs_per_group;
    // long tables and prompts: several workgroups a sequence, a few thousand in all
    const int64_t longest = std::max<int64_t>(p.max_num_blocks, (p.max_rows + groups - 1) / groups);
    int64_t pieces = (longest + 4 * kPlanThreads - 1) / (4 * kPlanThreads);
    pieces = std::max<int64_t>(1, std::min<int64_t>(pieces, 2048 / groups));
    hipLaunchKernelGGL(batch_plan_kernel, dim3(groups, (unsigned)pieces), dim3(kPlanThreads), 0, stream, p);
    return hipGetLastError();
}

}  // namespace pam
