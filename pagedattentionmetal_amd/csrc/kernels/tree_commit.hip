// tree_commit.hip - the accepted path of a drafted tree moved to the end of its
// sequence (gfx950).
//
// Node i of a tree over c cached tokens lies at position c + i.  The accepted path
// path[0] < path[1] < .. becomes positions c, c + 1, ..: the token of path[k] moves to
// c + k.  As path[k] >= k, no move writes a token that a later move reads, so a thread
// may read a chunk of the path's pieces before it writes them.
//
// f32 and f16 are copied.  e4m3 pools keep one scale per block: the moved tokens are
// appended with the append's own rule (scale = max(largest magnitude / 448, the block's
// scale)) from the values that their codes stand for.  A destination block's sources
// lie in it or in later blocks, so blocks are done in order with every scale still the
// one its codes were written with.
//
// What bounds it: latency (the path, the table's entries, one trip for the tokens and
// one for the stores): a path is a few tokens of 2 Hkv d elements (16 sequences, f16: 7.8 us,
// 0.4 MB; 128, f32: 9.0 us, 7.5 MB).
#include <algorithm>

#include "append_body.h"
#include "speculative.h"

namespace pam {

// A sequence's accepted tokens: entries rise and name new tokens; the path ends at the
// first that does not.
struct CommitSeq {
    const int32_t *bt, *path;
    int64_t c, n, cap;
};
__device__ __forceinline__ CommitSeq commit_seq(const TreeCommitParams &p, int s) {
    CommitSeq q;
    q.bt = p.block_tables + (int64_t)s * p.max_num_blocks;
    q.path = p.paths + (int64_t)s * p.max_path;
    q.cap = (int64_t)p.max_num_blocks * p.block_size;
    q.c = p.context_lens[s] > 0 ? p.context_lens[s] : 0;
    q.n = p.query_lens[s];
    if (q.n > q.cap - q.c) q.n = q.cap - q.c;
    return q;
}

// the path's length, by one wave: entries 64 at a time
__device__ __forceinline__ int commit_count(const TreeCommitParams &p, const CommitSeq &q) {
    const int lane = threadIdx.x & 63;
    for (int k0 = 0; k0 < p.max_path; k0 += 64) {
        const int k = k0 + lane;
        bool ok = false;
        if (k < p.max_path) {
            const int32_t v = q.path[k], before = k ? q.path[k - 1] : -1;
            ok = v > before && v < q.n && v >= 0;
        }
        const uint64_t bad = ~__ballot(ok);
        if (bad) return k0 + __builtin_ctzll(bad);
    }
    return p.max_path;
}

// pool slot of position pos of the sequence; -1: its block lies outside the pools
__device__ __forceinline__ int64_t commit_slot(const TreeCommitParams &p, const CommitSeq &q, int64_t pos) {
    const int64_t b = pos / p.block_size;
    const int32_t blk = q.bt[b];
    return (uint32_t)blk < (uint32_t)p.pool_blocks ? (int64_t)blk * p.block_size + (pos - b * p.block_size) : -1;
}

constexpr int kCommitChunk = 8;  // pieces of a path that a thread has in flight

// grid: x = sequence, y = slices of a token's pieces, z = pool
template <typename CH>
__global__ __launch_bounds__(256) void tree_commit_kernel(TreeCommitParams p, int64_t pieces) {
    const int s = blockIdx.x;
    const CommitSeq q = commit_seq(p, s);
    const int count = commit_count(p, q);
    if (p.new_lengths && blockIdx.y == 0 && blockIdx.z == 0 && threadIdx.x == 0) p.new_lengths[s] = (int32_t)(q.c + count);
    CH *pool = static_cast<CH *>(blockIdx.z ? p.v_pool : p.k_pool);
    const int64_t c = (int64_t)blockIdx.y * blockDim.x + threadIdx.x;
    if (c >= pieces) return;
    for (int k0 = 0; k0 < count; k0 += kCommitChunk) {
        CH v[kCommitChunk];
        int64_t to[kCommitChunk];
#pragma unroll
        for (int i = 0; i < kCommitChunk; i++) {
            const int k = k0 + i;
            to[i] = -1;
            if (k >= count) continue;
            const int32_t node = q.path[k];
            if (node == k) continue;  // already there
            const int64_t from = commit_slot(p, q, q.c + node);
            if (from < 0) continue;
            to[i] = commit_slot(p, q, q.c + k);
            v[i] = pool[from * pieces + c];
        }
#pragma unroll
        for (int i = 0; i < kCommitChunk; i++)
            if (to[i] >= 0) pool[to[i] * pieces + c] = v[i];
    }
}

constexpr int kCommitFp8Threads = 1024;

// grid: x = sequence, y = pool; 4 codes a thread and step
__global__ __launch_bounds__(kCommitFp8Threads) void tree_commit_fp8_kernel(TreeCommitParams p) {
    __shared__ float red[kCommitFp8Threads / 64];
    const int s = blockIdx.x;
    const CommitSeq q = commit_seq(p, s);
    const int count = commit_count(p, q);
    if (p.new_lengths && blockIdx.y == 0 && threadIdx.x == 0) p.new_lengths[s] = (int32_t)(q.c + count);
    if (count == 0) return;
    uint32_t *pool = static_cast<uint32_t *>(blockIdx.y ? p.v_pool : p.k_pool);
    uint16_t *scales = blockIdx.y ? p.v_scale : p.k_scale;
    const int64_t words = (int64_t)p.num_kv_heads * p.head_dim / 4;
    const int bs = p.block_size;
    for (int64_t lb = q.c / bs; lb <= (q.c + count - 1) / bs; lb++) {
        const int k0 = (int)(lb * bs > q.c ? lb * bs - q.c : 0);
        const int k1 = (int)((lb + 1) * bs - q.c < count ? (lb + 1) * bs - q.c : count);
        const int32_t blk = q.bt[lb];
        if ((uint32_t)blk >= (uint32_t)p.pool_blocks) continue;  // the same for every thread
        const f16 old = bits_to_f16(scales[blk]);
        auto source = [&](int k, int64_t &from, f16 &sc) {
            from = commit_slot(p, q, q.c + q.path[k]);
            if (from >= 0) sc = bits_to_f16(scales[from / bs]);
            return from >= 0;
        };
        float mx = 0.0f;
        for (int k = k0; k < k1; k++) {
            int64_t from;
            f16 sc;
            if (!source(k, from, sc)) continue;
            for (int64_t e = threadIdx.x; e < words; e += kCommitFp8Threads) {
                const uint32_t w = pool[from * words + e];
#pragma unroll
                for (int i = 0; i < 4; i++) mx = fmaxf(mx, fabsf((float)fp8_dequant((w >> (8 * i)) & 0xFFu, sc)));
            }
        }
        mx = wave_max_xor(mx, 1, 64);
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = mx;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kCommitFp8Threads / 64; w++) mx = fmaxf(mx, red[w]);
        const f16 ns = fp8_scale_rule(mx, old);
        for (int k = k0; k < k1; k++) {
            int64_t from;
            f16 sc;
            if (!source(k, from, sc)) continue;
            const int64_t to = commit_slot(p, q, q.c + k);
            for (int64_t e = threadIdx.x; e < words; e += kCommitFp8Threads) {
                const uint32_t w = pool[from * words + e];
                uint32_t o = 0;
#pragma unroll
                for (int i = 0; i < 4; i++) o |= fp8_quantize(fp8_dequant((w >> (8 * i)) & 0xFFu, sc), ns) << (8 * i);
                pool[to * words + e] = o;
            }
        }
        __syncthreads();  // every scale read above is the old one
        if (threadIdx.x == 0) scales[blk] = f16_to_bits(ns);
        __syncthreads();
    }
}

hipError_t launch_tree_commit(const TreeCommitParams &p, int32_t dtype, hipStream_t stream) {
    if (p.num_seqs <= 0 || p.max_path <= 0) return hipErrorInvalidValue;
    if (dtype == kFP8) {
        hipLaunchKernelGGL(tree_commit_fp8_kernel, dim3((unsigned)p.num_seqs, 2), dim3(kCommitFp8Threads), 0, stream, p);
        return hipGetLastError();
    }
    const int64_t row = (int64_t)p.num_kv_heads * p.head_dim * (dtype == kF32 ? 4 : 2);
    const uintptr_t at = (uintptr_t)p.k_pool | (uintptr_t)p.v_pool | (uintptr_t)row;
    const int64_t w = at % 16 == 0 ? 16 : (at % 8 == 0 ? 8 : (at % 4 == 0 ? 4 : 2));
    const int64_t pieces = row / w;
    const dim3 grid((unsigned)p.num_seqs, (unsigned)((pieces + 255) / 256), 2);
    if (w == 16)
        hipLaunchKernelGGL(tree_commit_kernel<uint4>, grid, dim3(256), 0, stream, p, pieces);
    else if (w == 8)
        hipLaunchKernelGGL(tree_commit_kernel<uint2>, grid, dim3(256), 0, stream, p, pieces);
    else if (w == 4)
        hipLaunchKernelGGL(tree_commit_kernel<uint32_t>, grid, dim3(256), 0, stream, p, pieces);
    else
        hipLaunchKernelGGL(tree_commit_kernel<uint16_t>, grid, dim3(256), 0, stream, p, pieces);
    return hipGetLastError();
}

}  // namespace pam
