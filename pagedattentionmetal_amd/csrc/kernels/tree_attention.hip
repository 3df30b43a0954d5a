// tree_attention.hip - attention of drafted trees over a paged cache (gfx950): the kernels
// and their choice.
//   tree_mfma_kernel   f16 and e4m3 pools, head sizes up to 128 (tree_mfma.h)
//   tree_rows_kernel   f32 pools and larger heads: f32 probabilities on the matrix units
//                      (RowTiles, rows_body.h)
//   tree_row_kernel    what has no whole 16-byte (e4m3: 8-byte) pieces
// The first two share the chip by equal counts of units and leave partials that
// tree_reduce_kernel merges (tree_body.h).
#include <algorithm>

#include "tree_mfma.h"

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

// ------------------------------------------------------------------ row blocks

template <typename Tiles, int RB>
struct TreeSee {
    const TreeParams &p;
    const TreeRow (&row)[RB];
    int c, all;
    __device__ __forceinline__ bool sees(int b, int j) const { return row[b].sees(j, c); }
    __device__ __forceinline__ int32_t block(int32_t entry) const { return tree_block(p, entry); }
    __device__ __forceinline__ int lo_all(const TileKeys &) const { return all; }
};

template <typename KV, typename QT, int NT, int RB>
__global__ __launch_bounds__(64 * kRowsWaves, (NT <= 4 ? 2 : 1)) void tree_rows_kernel(TreeParams p) {
    typedef RowTiles<KV, QT, NT, RB> Tiles;
    constexpr int LS = Tiles::LS, RN = 16 * RB;
    __shared__ __attribute__((aligned(16))) float lds[kRowsLds<NT, RB>];
    const AttnParams &a = p.a;
    const int wave = threadIdx.x >> 6, H = a.num_heads, G = H / a.num_kv_heads, d = a.head_dim;
    const int64_t group = (blockIdx.x % kXcds) * (int64_t)(gridDim.x / kXcds) + blockIdx.x / kXcds;
    const TreeWork w = tree_work(p);
    int64_t u = group * w.per;
    const int64_t end = u + w.per < w.units ? u + w.per : w.units;
    if (u >= end) return;
    TreeItem it;
    tree_find(p, u, it);
    for (;;) {
        const int64_t item_end = it.first + it.tiles, u1 = item_end < end ? item_end : end;
        const TreeRows tr = tree_rows(p, it, 16);
        TileKeys keys;
        keys.bt = it.q.bt;
        keys.block_size = a.block_size;
        keys.shift = block_shift(a.block_size);
        keys.key0 = (it.tile0 + (int)(u - it.first)) * p.unit_keys;
        keys.lo = tree_first_key(p, it.q);
        keys.hi = it.q.hi;
        keys.hi_all = it.q.c;
        const int64_t all = (int64_t)it.q.c + it.q.n - a.window;
        const int lo_all = a.window > 0 && all > 0 ? (int)(all < it.q.c ? all : it.q.c) : 0;
        const int key_end = (it.tile0 + (int)(u1 - it.first)) * p.unit_keys;
        const int ntiles = keys.hi > keys.lo ? ((key_end < keys.hi ? key_end : keys.hi) - keys.key0 + 15) / 16 : 0;

        Tiles x;
        x.init(a, it.kvh);
        TreeRow rows[RB];
#pragma unroll
        for (int b = 0; b < RB; b++) {
            const int rho = tr.row0 + (16 * b + x.n < tr.rows ? 16 * b + x.n : tr.rows - 1), node = rho / G;
            rows[b].init(p, it.q, node);
            x.load_q(b, static_cast<const QT *>(a.q) +
                            ((int64_t)(it.q.row0 + node) * H + it.kvh * G + (rho - node * G)) * d);
        }
        const TreeSee<Tiles, RB> see{p, rows, it.q.c, lo_all};
        x.run(a, keys, see, wave, ntiles, kRowsWaves);

        float *ml = lds + kRowsWaves * RN * LS;
        const bool any_odd = __syncthreads_or(x.odd);
#pragma unroll
        for (int b = 0; b < RB; b++) {
            if (x.g == 0) {
                ml[(wave * RN + 16 * b + x.n) * 2] = x.m[b];
                ml[(wave * RN + 16 * b + x.n) * 2 + 1] = x.l[b];
            }
            x.put(b, 1.0f, lds + (wave * RN + 16 * b + x.n) * LS);
        }
        __syncthreads();
        tree_write<KV, QT, LS>(p, it, tr, w, group, u, u1, lds, (int64_t)RN * LS, ml, RN * 2, kRowsWaves, any_odd, lo_all);
        u = u1;
        if (u >= end) break;
        tree_next(p, it);
        __syncthreads();
    }
}

// ------------------------------------------------------------------ merge

// The partials of the items that several workgroups share, in order.  grid: x = row block
// and slice of its rows, y = kv head, z = sequence
constexpr int kTreeReduceRows = 8;
template <typename QT>
__global__ __launch_bounds__(256) void tree_reduce_kernel(TreeParams p) {
    const int slices = (p.block_rows + kTreeReduceRows - 1) / kTreeReduceRows;
    TreeItem it;
    tree_enter(p, blockIdx.z, it);
    it.rb = blockIdx.x / slices;
    it.kvh = blockIdx.y;
    if (it.rb >= it.blocks) return;
    int64_t before = 0, t = 0;
    for (int s = threadIdx.x & 63; s < p.num_seqs; s += 64) {
        const int64_t v = tree_units(p, s);
        t += v;
        before += s < it.s ? v : 0;
    }
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) t += __shfl_xor(t, m, 64), before += __shfl_xor(before, m, 64);
    TreeWork w;
    w.units = t;
    w.per = (t + p.groups - 1) / p.groups;
    if (w.per < p.min_units) w.per = p.min_units;
    it.first = before + ((int64_t)it.kvh * it.blocks + it.rb) * it.tiles;
    const int64_t g0 = it.first / w.per, g1 = (it.first + it.tiles - 1) / w.per;
    if (g0 == g1) return;  // one workgroup wrote its rows
    const TreeRows tr = tree_rows(p, it, p.form == kTreeMfma ? 32 : 16);
    const int d = p.a.head_dim, pieces = d / 4, r0 = (int)(blockIdx.x % slices) * kTreeReduceRows;
    const int rn = tr.rows - r0 < kTreeReduceRows ? tr.rows - r0 : kTreeReduceRows;
    // slot of group g0 by where the item begins; those of the others are their first
    const float *o0 = tree_part_o(p, tree_slot(w, g0, it.first)), *ml0 = tree_part_ml(p, tree_slot(w, g0, it.first));
    const float *o1 = tree_part_o(p, 2 * (g0 + 1)), *ml1 = tree_part_ml(p, 2 * (g0 + 1));
    const int64_t step = 2 * (int64_t)p.block_rows * (d + 2);
    const int n = (int)(g1 - g0);
    for (int i = threadIdx.x; i < rn * pieces; i += 256) {
        const int r = r0 + i / pieces, e0 = i % pieces * 4;
        float M = ml0[2 * r];
        for (int k = 0; k < n; k++) M = fmaxf(M, ml1[k * step + 2 * r]);
        const float mu = M == -INFINITY ? 0.0f : M;
        const float w0 = exp2f(ml0[2 * r] - mu);
        const float4 v0 = *reinterpret_cast<const float4 *>(o0 + (int64_t)r * d + e0);
        TreeSum s{{w0 * v0.x, w0 * v0.y, w0 * v0.z, w0 * v0.w}, w0 * ml0[2 * r + 1], M};
#pragma unroll 4
        for (int k = 0; k < n; k++) {
            const float wk = exp2f(ml1[k * step + 2 * r] - mu);
            const float4 v = *reinterpret_cast<const float4 *>(o1 + k * step + (int64_t)r * d + e0);
            s.den += wk * ml1[k * step + 2 * r + 1];
            s.a[0] += wk * v.x, s.a[1] += wk * v.y, s.a[2] += wk * v.z, s.a[3] += wk * v.w;
        }
        tree_out<QT>(p, it, tr.row0 + r, e0, s);
    }
}

// ------------------------------------------------------------------ choice

static int tree_dim_slot(int32_t head_dim) {
    const int nt = (head_dim + 31) / 32;
    return nt <= 4 ? nt - 1 : 4;
}

int64_t tree_plan(TreeParams &p, int32_t dtype, int32_t cus) {
    const AttnParams &a = p.a;
    const int64_t G = a.num_heads / a.num_kv_heads, rows = (int64_t)p.max_queries * G;
    p.form = kTreeRow;
    if (!rows_supported(a, dtype)) return 0;
    const bool mfma = dtype != kF32 && a.head_dim <= 128;
    p.form = mfma ? kTreeMfma : kTreeRowBlocks;
    if (mfma) {
        p.block_rows = rows <= 32 ? 32 : (rows <= 64 ? 64 : 128);
        p.unit_keys = rows <= 32 ? 128 : 64;
    } else {
        const bool one = rows <= 16 || (dtype == kF32 && a.head_dim > 128);
        p.block_rows = one ? 16 : 32;
        p.unit_keys = 16 * kRowsWaves;
    }
    // two workgroups a CU (a multiple of the XCDs), fewer when the batch can hold no more units
    const int64_t tiles = ((int64_t)a.max_num_blocks * a.block_size + p.unit_keys - 1) / p.unit_keys + 1;
    const int64_t most = (int64_t)p.num_seqs * a.num_kv_heads * ((rows + p.block_rows - 1) / p.block_rows) * tiles;
    p.min_units = 1;
    int64_t groups = std::min<int64_t>(2 * (int64_t)(cus > 0 ? cus : 1), most);
    groups = (groups + kXcds - 1) / kXcds * kXcds;
    p.groups = (int32_t)groups;
    return 2 * groups * p.block_rows * (a.head_dim + 2) * 4;
}

template <typename KV, int HD>
static void launch_tree_mfma(const TreeParams &p, hipStream_t stream) {
    const dim3 grid((unsigned)p.groups), block(256);
    if (p.block_rows == 32)
        hipLaunchKernelGGL((tree_mfma_kernel<KV, HD, 1>), grid, block, 0, stream, p);
    else if (p.block_rows == 64)
        hipLaunchKernelGGL((tree_mfma_kernel<KV, HD, 2>), grid, block, 0, stream, p);
    else
        hipLaunchKernelGGL((tree_mfma_kernel<KV, HD, 4>), grid, block, 0, stream, p);
}

template <typename KV, typename QT, int NT>
static void launch_tree_rows(const TreeParams &p, hipStream_t stream) {
    const dim3 grid((unsigned)p.groups), block(64 * kRowsWaves);
    if constexpr (kPrefillRowsRB<KV, NT> > 1) {
        if (p.block_rows == 32) {
            hipLaunchKernelGGL((tree_rows_kernel<KV, QT, NT, 2>), grid, block, 0, stream, p);
            return;
        }
    }
    hipLaunchKernelGGL((tree_rows_kernel<KV, QT, NT, 1>), grid, block, 0, stream, p);
}

hipError_t launch_tree_attention(const TreeParams &p, int32_t dtype, hipStream_t stream) {
    if (p.form == kTreeRow) {
        switch (dtype) {
            case kF32: return launch_tree_row<float, float>(p, stream);
            case kF16: return launch_tree_row<f16, f16>(p, stream);
            case kFP8: return launch_tree_row<uint8_t, f16>(p, stream);
            default: return hipErrorInvalidValue;
        }
    }
    if (p.a.part_o == nullptr || p.a.zero_page == nullptr) return hipErrorInvalidValue;
    if (p.form == kTreeMfma) {
        if (dtype == kF16) {
            p.a.head_dim <= 64 ? launch_tree_mfma<f16, 64>(p, stream) : launch_tree_mfma<f16, 128>(p, stream);
        } else {
            p.a.head_dim <= 64 ? launch_tree_mfma<uint8_t, 64>(p, stream) : launch_tree_mfma<uint8_t, 128>(p, stream);
        }
    } else if (dtype == kF32) {
        switch (tree_dim_slot(p.a.head_dim)) {
            case 0: launch_tree_rows<float, float, 1>(p, stream); break;
            case 1: launch_tree_rows<float, float, 2>(p, stream); break;
            case 2: launch_tree_rows<float, float, 3>(p, stream); break;
            case 3: launch_tree_rows<float, float, 4>(p, stream); break;
            default: launch_tree_rows<float, float, 8>(p, stream); break;
        }
    } else if (dtype == kF16) {
        launch_tree_rows<f16, f16, 8>(p, stream);
    } else {
        launch_tree_rows<uint8_t, f16, 8>(p, stream);
    }
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const int G = p.a.num_heads / p.a.num_kv_heads;
    const int blocks = (int)(((int64_t)p.max_queries * G + p.block_rows - 1) / p.block_rows);
    const dim3 grid((unsigned)(blocks * ((p.block_rows + kTreeReduceRows - 1) / kTreeReduceRows)),
                    (unsigned)p.a.num_kv_heads, (unsigned)p.num_seqs);
    if (dtype == kF32)
        hipLaunchKernelGGL(tree_reduce_kernel<float>, grid, dim3(256), 0, stream, p);
    else
        hipLaunchKernelGGL(tree_reduce_kernel<f16>, grid, dim3(256), 0, stream, p);
    return hipGetLastError();
}

}  // namespace pam
