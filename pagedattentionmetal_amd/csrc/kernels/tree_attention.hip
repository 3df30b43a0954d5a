// tree_attention.hip - attention of drafted trees over a paged cache (gfx950).
#include <algorithm>

#include "tree_body.h"

namespace pam {

// ------------------------------------------------------------------ one row a workgroup
// Any head size (a multiple of 4), group and alignment: a workgroup serves one (row,
// head); lanes split a key's row into 4-element slices, lane groups and waves take keys
// in turn, each with its own running maximum and sum, and merge in LDS.
template <typename KV, typename QT>
__global__ __launch_bounds__(256) void tree_row_kernel(TreeParams p, int lanes_per_key) {
    __shared__ float merge[256 / 1][6];
    const AttnParams &a = p.a;
    const int h = blockIdx.x, i = blockIdx.y, s = blockIdx.z;
    const TreeSeq q = tree_seq(p, s);
    if (i >= q.n) return;
    const int H = a.num_heads, K = a.num_kv_heads, d = a.head_dim, kvh = h / (H / K), bs = a.block_size;
    const int LPK = lanes_per_key, group = threadIdx.x / LPK, groups = 256 / LPK, d0 = threadIdx.x % LPK * 4;
    const bool ok = d0 < d;
    TreeRow row;
    row.init(p, q, i);
    const int64_t at = ((int64_t)(q.row0 + i) * H + h) * d + d0;
    float qv[4] = {0.f, 0.f, 0.f, 0.f}, acc[4] = {0.f, 0.f, 0.f, 0.f};
    if (ok) load4<QT>(static_cast<const QT *>(a.q) + at, qv);
    float m = -INFINITY, l = 0.0f;
    for (int j = row.lo + group; j < q.hi; j += groups) {
        if (!row.sees(j, q.c)) continue;
        const int32_t blk = tree_block(p, q.bt[j / bs]);
        const int64_t off = ((int64_t)blk * bs + j % bs) * ((int64_t)K * d) + (int64_t)kvh * d + d0;
        float kv[4] = {0.f, 0.f, 0.f, 0.f}, vv[4] = {0.f, 0.f, 0.f, 0.f};
        if (ok) {
            f16 ks = (f16)1.0f, vs = (f16)1.0f;
            if constexpr (sizeof(KV) == 1) ks = bits_to_f16(a.k_scale[blk]), vs = bits_to_f16(a.v_scale[blk]);
            load_kv4<KV>(static_cast<const KV *>(a.k_pool) + off, ks, kv);
            load_kv4<KV>(static_cast<const KV *>(a.v_pool) + off, vs, vv);
        }
        float x = qv[0] * kv[0] + qv[1] * kv[1] + qv[2] * kv[2] + qv[3] * kv[3];
        x = wave_sum_xor(x, 1, LPK) * a.scale_log2;
        const float mn = fmaxf(m, x), mu = mn == -INFINITY ? 0.0f : mn;
        const float corr = exp2f(m - mu), pj = exp2f(x - mu);
        l = l * corr + pj;
#pragma unroll
        for (int e = 0; e < 4; e++) acc[e] = acc[e] * corr + pj * vv[e];
        m = mn;
    }
    float *mine = merge[threadIdx.x];
#pragma unroll
    for (int e = 0; e < 4; e++) mine[e] = acc[e];
    mine[4] = m, mine[5] = l;
    __syncthreads();
    if (group != 0 || !ok) return;
    float M = -INFINITY, den = 0.0f, o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int g = 0; g < groups; g++) M = fmaxf(M, merge[g * LPK + threadIdx.x][4]);
    const float mu = M == -INFINITY ? 0.0f : M;
    for (int g = 0; g < groups; g++) {
        const float *x = merge[g * LPK + threadIdx.x];
        const float w = exp2f(x[4] - mu);
        den += w * x[5];
#pragma unroll
        for (int e = 0; e < 4; e++) o[e] += w * x[e];
    }
    const float inv = den == 0.0f ? 0.0f : 1.0f / den;
#pragma unroll
    for (int e = 0; e < 4; e++) o[e] *= inv;
    store4<QT>(static_cast<QT *>(a.out) + at, o);
}

template <typename KV, typename QT>
static hipError_t launch_tree_row(const TreeParams &p, hipStream_t stream) {
    int lpk = 1;
    while (lpk * 4 < p.a.head_dim) lpk *= 2;
    const dim3 grid((unsigned)p.a.num_heads, (unsigned)p.max_queries, (unsigned)p.num_seqs);
    hipLaunchKernelGGL((tree_row_kernel<KV, QT>), grid, dim3(256), 0, stream, p, lpk);
    return hipGetLastError();
}

hipError_t launch_tree_attention(const TreeParams &p, int32_t dtype, hipStream_t stream) {
    switch (dtype) {
        case kF32: return launch_tree_row<float, float>(p, stream);
        case kF16: return launch_tree_row<f16, f16>(p, stream);
        case kFP8: return launch_tree_row<uint8_t, f16>(p, stream);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace pam
