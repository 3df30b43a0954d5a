// tree_attention.hip - attention of drafted trees over a paged cache (gfx950): the kernels
// and their choice.
//   tree_mfma_kernel   f16 and e4m3 pools, head sizes up to 128 (tree_mfma.h)
//   tree_rows_kernel   f32 pools, larger heads, odd or small blocks: f32 probabilities on the
//                      matrix units (RowTiles, rows_body.h)
//   tree_row_kernel    what has no whole 16-byte (e4m3: 8-byte) pieces
// The first two share the chip by equal counts of units (tree_body.h) and tree_reduce_kernel
// merges what they leave.
#include <algorithm>

#include "tree_mfma.h"

namespace pam {


// ------------------------------------------------------------------ one row a workgroup
// Any head size (a multiple of 4), group and alignment: a workgroup serves one (row,
// head); lanes split a key's row into 4-element slices, lane groups and waves take keys
// in turn, each with its own running maximum and sum, and merge in LDS.  What bounds it: a
// chain of loads a lane, and keys read again for every row (f16 heads of 20, 16 sequences of 1000
// tokens, 8 nodes: 29 us; heads of 24 on the matrix kernel 13).
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

// What bounds them: few rows, memory (f32, 8 heads of 128, 16 sequences of 4096 tokens, 8 nodes:
// 102 us, 5.3 TB/s); many, f32 matrix products (8 heads on 2 of 64, 64 nodes: 126 us, 68 TFLOP/s);
// short sequences, the latency of two launches (11 and 4 us).
constexpr int kTreeRowKeys = 16 * kRowsWaves;  // keys of a unit: a tile for every wave

template <typename KV, typename QT, int NT, int RB>
__global__ __launch_bounds__(64 * kRowsWaves, (NT <= 4 ? 2 : 1)) void tree_rows_kernel(TreeParams p) {
    typedef RowTiles<KV, QT, NT, RB> Tiles;
    constexpr int LS = Tiles::LS, RN = 16 * RB, KEYS = kTreeRowKeys;
    __shared__ __attribute__((aligned(16))) float lds[kRowsLds<NT, RB>];
    __shared__ int odd_lds[kRowsWaves];
    const AttnParams &a = p.a;
    const int wave = threadIdx.x >> 6, H = a.num_heads, G = H / a.num_kv_heads, d = a.head_dim;
    TreeWork w;
    TreeItem it;
    if (!tree_start(p, w, it)) return;
    int u = w.group * w.per;
    const int end = u + w.per < w.units ? u + w.per : w.units;
    for (;;) {
        const int u1 = tree_item_end(it, end);
        const TreeRows tr = tree_rows<16>(p, it);
        TileKeys keys;
        keys.bt = it.q.bt;
        keys.block_size = a.block_size;
        keys.shift = block_shift(a.block_size);
        keys.key0 = (it.tile0 + u - it.first) * KEYS;
        keys.lo = tree_first_key(p, it.q);
        keys.hi = it.q.hi;
        keys.hi_all = it.q.c;
        const int64_t all = (int64_t)it.q.c + it.q.n - a.window;
        const int lo_all = a.window > 0 && all > 0 ? (int)(all < it.q.c ? all : it.q.c) : 0;
        const int key_end = (it.tile0 + u1 - it.first) * KEYS;
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
        const bool wave_odd = __any(x.odd);
        if ((threadIdx.x & 63) == 0) odd_lds[wave] = wave_odd;
#pragma unroll
        for (int b = 0; b < RB; b++) {
            if (x.g == 0) {
                ml[(wave * RN + 16 * b + x.n) * 2] = x.m[b];
                ml[(wave * RN + 16 * b + x.n) * 2 + 1] = x.l[b];
            }
            x.put(b, 1.0f, lds + (wave * RN + 16 * b + x.n) * LS);
        }
        __syncthreads();
        const bool any_odd = tree_any<kRowsWaves>(odd_lds);
        tree_write<KV, QT, LS, 8 * NT, kRowsWaves, 64 * kRowsWaves>(p, it, tr, w, u, u1, lds, RN * LS, ml, RN * 2, any_odd,
                                                                    lo_all);
        u = u1;
        if (tree_last(w, u, end)) break;
        tree_next(p, it);
        __syncthreads();
    }
}

// ------------------------------------------------------------------ merge

// The partials of the items that several workgroups share, in order.  grid: x = slice of
// slice_rows rows of a row block, y = kv head, z = sequence; or, by_share, x = slice and share
// boundary, for a batch with more items than shares, few of which are split (166 sequences, 8 kv
// heads: 20 us, by item 36).  A thread adds 4 dims of a row;
// with `ways` > 1 so many threads share the row's partials.  What bounds it: few
// partials, their bytes; else the latency of the lengths and the partials behind one another,
// so a thread asks for 8 partials and their states at once.
constexpr int kTreeReduceThreads = 512;
template <typename QT>
__global__ __launch_bounds__(kTreeReduceThreads) void tree_reduce_kernel(TreeParams p, int slice_rows, int ways, bool by_share) {
    __shared__ float sums[kTreeReduceThreads][6];
    const int slices = ((1 << p.rows_log2) + slice_rows - 1) / slice_rows;
    const int lane = threadIdx.x & 63;
    TreeItem it;
    TreeSeq own{};
    TreeWork w;
    const TreeCount mine = tree_count(p, lane, own);
    tree_share(p, mine, w);
    if (by_share) {
        // the item that the boundary cuts, if no boundary before cuts it
        const int g = (int)(blockIdx.x / slices) + 1, u = g * w.per;
        if (u >= w.units) return;
        tree_find(p, w, u, mine, own, it);
        if (it.first == u || it.first < (g - 1) * w.per) return;
    } else {
        it.s = blockIdx.z;
        it.kvh = blockIdx.y;
        it.rb = blockIdx.x / slices;
        it.q = tree_seq(p, it.s);
        tree_shape(p, it);
        if (it.rb >= it.blocks) return;
        int before = 0;
        for (int s = lane; s < it.s; s += 64) {
            const TreeCount n = tree_count(p, s, own);
            before += n.items * tree_padded(n.tiles, w.pad);
        }
        it.first = tree_wave_sum(before) + (it.kvh * it.blocks + it.rb) * tree_padded(it.tiles, w.pad);
    }
    const int g0 = (int)((uint32_t)it.first / (uint32_t)w.per);
    const int np = (int)((uint32_t)(it.first + it.tiles - 1) / (uint32_t)w.per) - g0 + 1;
    if (np == 1) return;  // one workgroup wrote its rows
    const TreeRows tr = p.form == kTreeMfma ? tree_rows<32>(p, it) : tree_rows<16>(p, it);
    const int d = p.a.head_dim, pieces = d / 4, r0 = (int)(blockIdx.x % slices) * slice_rows;
    const int rn = tr.rows - r0 < slice_rows ? tr.rows - r0 : slice_rows;
    const int share = kTreeReduceThreads / ways, way = threadIdx.x / share, me = threadIdx.x % share;
    const float *first_part = tree_part(p, 2 * g0);
    const int64_t stride = 2 * (int64_t)((d + 2) << p.rows_log2);  // a workgroup's two places
    // rounds of equal length in all threads: the sums below meet at a barrier
    for (int i0 = 0; i0 < rn * pieces; i0 += share) {
        const int i = i0 + me, x = i / pieces, e0 = (i - x * pieces) * 4;
        const bool on = x < rn;
        TreeSum s{{0.f, 0.f, 0.f, 0.f}, 0.0f, -INFINITY};
        for (int k0 = way; on && k0 < np; k0 += 8 * ways) {
            float4 v[8];
            float2 ml[8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int k = k0 + j * ways;
                ml[j] = make_float2(-INFINITY, 0.0f);
                v[j] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (k < np) {
                    // tree_slot: the item is the second of its first workgroup only
                    const float *part = first_part + k * stride;
                    if (k == 0 && it.first > g0 * w.per) part += stride / 2;
                    ml[j] = *reinterpret_cast<const float2 *>(part + (d << p.rows_log2) + 2 * (r0 + x));
                    v[j] = *reinterpret_cast<const float4 *>(part + (r0 + x) * d + e0);
                }
            }
            float top = s.M;
#pragma unroll
            for (int j = 0; j < 8; j++) top = fmaxf(top, ml[j].x);
            const float mu = top == -INFINITY ? 0.0f : top, old = __builtin_amdgcn_exp2f(s.M - mu);
            s.M = top;
            s.den *= old;
#pragma unroll
            for (int e = 0; e < 4; e++) s.a[e] *= old;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float wk = __builtin_amdgcn_exp2f(ml[j].x - mu);
                s.den += wk * ml[j].y;
                s.a[0] += wk * v[j].x, s.a[1] += wk * v[j].y, s.a[2] += wk * v[j].z, s.a[3] += wk * v[j].w;
            }
        }
        if (ways > 1) {
            float *mine = sums[threadIdx.x];
#pragma unroll
            for (int e = 0; e < 4; e++) mine[e] = s.a[e];
            mine[4] = s.M, mine[5] = s.den;
            __syncthreads();
            if (way == 0) {
                for (int k = 1; k < ways; k++) s.M = fmaxf(s.M, sums[k * share + me][4]);
                const float mu = s.M == -INFINITY ? 0.0f : s.M, own = __builtin_amdgcn_exp2f(mine[4] - mu);
                s.den *= own;
#pragma unroll
                for (int e = 0; e < 4; e++) s.a[e] *= own;
                for (int k = 1; k < ways; k++) {
                    const float *o = sums[k * share + me];
                    const float wk = __builtin_amdgcn_exp2f(o[4] - mu);
                    s.den += wk * o[5];
#pragma unroll
                    for (int e = 0; e < 4; e++) s.a[e] += wk * o[e];
                }
            }
            __syncthreads();
        }
        if (on && way == 0) tree_out<QT>(p, it, tr.row0 + r0 + x, e0, s);
    }
}

// ------------------------------------------------------------------ choice

static int tree_dim_slot(int32_t head_dim) {
    const int nt = (head_dim + 31) / 32;
    return nt <= 4 ? nt - 1 : 4;
}

// workgroups of a CU and keys of a unit of the matrix kernel for `rows` query rows a block
template <typename KV, int HD, int RW>
static void tree_mfma_shape(int *per_cu, int *keys) {
    *per_cu = TreeMfma<KV, HD, RW>::PER_CU;
    *keys = TreeMfma<KV, HD, RW>::KEYS;
}
template <typename KV, int HD>
static void tree_mfma_shape(int rows, int *per_cu, int *keys) {
    switch (rows) {
        case 32: tree_mfma_shape<KV, HD, 1>(per_cu, keys); break;
        case 64: tree_mfma_shape<KV, HD, 2>(per_cu, keys); break;
        case 128: tree_mfma_shape<KV, HD, 4>(per_cu, keys); break;
        default:
            if constexpr (sizeof(KV) == 1) tree_mfma_shape<KV, HD, 8>(per_cu, keys);
            break;
    }
}

int64_t tree_plan(TreeParams &p, int32_t dtype, int32_t cus) {
    const AttnParams &a = p.a;
    const int64_t G = a.num_heads / a.num_kv_heads, rows = (int64_t)p.max_queries * G;
    p.form = kTreeRow;
    if (!rows_supported(a, dtype) || rows >= ((int64_t)1 << 31) - 256) return 0;
    int per_cu = 2, keys = kTreeRowKeys;
    // a request of the matrix kernel takes 64 pieces of the rows of one block: 16 bytes of each, or,
    // e4m3 through registers, 8
    const int64_t elem = dtype == kFP8 ? 1 : 2, block = (int64_t)a.num_kv_heads * a.head_dim * elem * a.block_size;
    const int64_t head_block = (a.head_dim <= 64 ? 64 : 128) * elem * a.block_size;  // of one head, whole pieces
    if (dtype != kF32 && a.head_dim <= 128 && (a.block_size & (a.block_size - 1)) == 0 &&
        head_block >= (dtype == kFP8 ? 512 : 1024) && block < ((int64_t)1 << 31)) {
        p.form = kTreeMfma;
        // Blocks of 256 rows dequantise a key once for 256 rows, those of 128 twice, but a block with
        // few rows leaves its waves idle, so only sequences that fill three quarters of one take it
        // (e4m3, 4 sequences of 48000 tokens and 256 rows: 331 us and 354; 16 of 128 to 4096 tokens and
        // 64 to 256 rows, 160 in the mean: 93 us and 72).  f16 has nothing to dequantise: blocks of 256
        // rows took 350 us and 358 there, and 96 us and 76, so it has none.
        const int64_t mean = p.total_rows * G / std::max(p.num_seqs, 1);  // rows of a sequence
        p.block_rows = rows <= 32 ? 32 : (rows <= 64 ? 64 : (rows <= 128 || dtype == kF16 || mean < 192 ? 128 : 256));
        // the ring of codes takes whole 16-byte pieces of aligned rows, 64 of a block
        const uintptr_t pools = (uintptr_t)a.k_pool | (uintptr_t)a.v_pool;
        if (dtype == kFP8 && p.block_rows > 64 && (a.head_dim % 16 != 0 || pools % 16 != 0 || head_block < 1024))
            p.block_rows = 64;
        if (dtype == kF16)
            a.head_dim <= 64 ? tree_mfma_shape<f16, 64>(p.block_rows, &per_cu, &keys)
                             : tree_mfma_shape<f16, 128>(p.block_rows, &per_cu, &keys);
        else
            a.head_dim <= 64 ? tree_mfma_shape<uint8_t, 64>(p.block_rows, &per_cu, &keys)
                             : tree_mfma_shape<uint8_t, 128>(p.block_rows, &per_cu, &keys);
    } else {
        p.form = kTreeRowBlocks;
        // f32, 8 heads on 2 of 64, 16 sequences of 4096 tokens: 16 rows 24 us and 31 in a block of 32;
        // 64 rows 47 us in blocks of 16 and 44
        p.block_rows = rows <= 16 || (dtype == kF32 && a.head_dim > 128) ? 16 : 32;
    }
    // the workgroups that fit the CUs (a multiple of the XCDs), fewer when the batch can hold no
    // more units; a batch of more units than 31 bits count keeps the row kernel
    const int64_t tiles = ((int64_t)a.max_num_blocks * a.block_size + keys - 1) / keys + 1;
    const int64_t most = (int64_t)p.num_seqs * a.num_kv_heads * ((rows + p.block_rows - 1) / p.block_rows) * tiles;
    if (most >= (int64_t)1 << 30) {
        p.form = kTreeRow;
        return 0;
    }
    p.rows_log2 = __builtin_ctz((unsigned)p.block_rows);
    p.keys_log2 = __builtin_ctz((unsigned)keys);
    int64_t groups = std::min<int64_t>(per_cu * (int64_t)(cus > 0 ? cus : 1), most);
    groups = (groups + kXcds - 1) / kXcds * kXcds;
    p.groups = (int32_t)groups;
    return 2 * groups * p.block_rows * (a.head_dim + 2) * 4;
}

template <typename KV, int HD, int RW>
static void launch_tree_mfma(const TreeParams &p, hipStream_t stream) {
    hipLaunchKernelGGL((tree_mfma_kernel<KV, HD, RW>), dim3((unsigned)p.groups), dim3(64 * TreeMfma<KV, HD, RW>::WAVES), 0,
                       stream, p);
}
template <typename KV, int HD>
static void launch_tree_mfma(const TreeParams &p, hipStream_t stream) {
    switch (p.block_rows) {
        case 32: launch_tree_mfma<KV, HD, 1>(p, stream); break;
        case 64: launch_tree_mfma<KV, HD, 2>(p, stream); break;
        case 128: launch_tree_mfma<KV, HD, 4>(p, stream); break;
        default:
            if constexpr (sizeof(KV) == 1) launch_tree_mfma<KV, HD, 8>(p, stream);
            break;
    }
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
        if (dtype == kF16)
            p.a.head_dim <= 64 ? launch_tree_mfma<f16, 64>(p, stream) : launch_tree_mfma<f16, 128>(p, stream);
        else
            p.a.head_dim <= 64 ? launch_tree_mfma<uint8_t, 64>(p, stream) : launch_tree_mfma<uint8_t, 128>(p, stream);
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
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const int64_t G = p.a.num_heads / p.a.num_kv_heads, blocks = ((int64_t)p.max_queries * G + p.block_rows - 1) / p.block_rows;
    const int64_t items = blocks * p.a.num_kv_heads * p.num_seqs;  // at most
    const bool by_share = items > p.groups;
    // rows of a workgroup, by the batch's 16-row slices: a full chip takes many, so that few
    // workgroups wait for the lengths (2048 slices: 13.7 us with 64 rows, 18.8 with 16); an idle one
    // few, and 4 threads a row's piece (16 slices, 33 partials: 5.0 us, 7.0 with 16 rows; but 256
    // slices: 11 us, 6 with 16 rows)
    const int64_t slices = (by_share ? p.groups : items) * p.block_rows / 16;
    const int slice_rows = slices <= 64 ? 4 : (slices <= 1024 ? 16 : 64), ways = slices <= 64 ? 4 : 1;
    const unsigned of_block = (unsigned)((p.block_rows + slice_rows - 1) / slice_rows);
    const dim3 grid = by_share ? dim3((unsigned)p.groups * of_block)
                               : dim3((unsigned)blocks * of_block, (unsigned)p.a.num_kv_heads, (unsigned)p.num_seqs);
    if (dtype == kF32)
        hipLaunchKernelGGL(tree_reduce_kernel<float>, grid, dim3(kTreeReduceThreads), 0, stream, p, slice_rows, ways, by_share);
    else
        hipLaunchKernelGGL(tree_reduce_kernel<f16>, grid, dim3(kTreeReduceThreads), 0, stream, p, slice_rows, ways, by_share);
    return hipGetLastError();
}

}  // namespace pam
