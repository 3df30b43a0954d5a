// tree_body.h - attention of drafted trees over a paged cache (gfx950): which keys a
// row sees, shared by the kernels of tree_attention.hip.
//
// Sequence s holds c cached tokens and n drafted ones at positions c .. c + n - 1
// (appended to its blocks before the call).  Row (s, i) sees the cached tokens and
// the drafted tokens whose bits its mask has set; with a window W, the last W of the keys
// it sees, in order of position.  A row that sees no key is zeros.
#pragma once
#include "prefill_body.h"
#include "rows_body.h"
#include "speculative.h"

namespace pam {

struct TreeSeq {
    const int32_t *bt;
    int c, n, hi;  // cached tokens, rows, end of the keys (c + n, within the table)
    int row0;      // first row of the batch
};
__device__ __forceinline__ TreeSeq tree_seq(const TreeParams &p, int s) {
    TreeSeq q;
    const int64_t cap = (int64_t)p.a.max_num_blocks * p.a.block_size;
    int64_t c = p.context_lens[s];
    c = c < 0 ? 0 : (c < cap ? c : cap);
    int r0 = p.cu_queries[s], r1 = p.cu_queries[s + 1];
    r0 = r0 < 0 ? 0 : (r0 < p.total_rows ? r0 : p.total_rows);
    r1 = r1 < r0 ? r0 : (r1 < p.total_rows ? r1 : p.total_rows);
    q.n = r1 - r0 < p.max_queries ? r1 - r0 : p.max_queries;
    q.bt = p.a.block_tables + (int64_t)s * p.a.bt_stride;
    q.c = (int)c;
    q.hi = (int)(c + q.n < cap ? c + q.n : cap);
    q.row0 = r0;
    return q;
}

// a table entry, held inside the pools
__device__ __forceinline__ int32_t tree_block(const TreeParams &p, int32_t entry) {
    const uint32_t last = (uint32_t)p.pool_blocks - 1;
    return (int32_t)((uint32_t)entry < last ? (uint32_t)entry : last);
}

// The keys of one row: cached keys from lo on, and drafted ones by word of 64 bits.
struct TreeRow {
    const uint64_t *mask;  // null: a chain
    int i, n, words;
    int lo;                // first cached key inside the window
    int drop;              // bits of the path, from the lowest, that lie before the window

    __device__ __forceinline__ uint64_t raw(int w) const {
        if (w < 0 || w >= words) return 0ull;
        const int live = n - 64 * w;  // nodes of the word
        if (live <= 0) return 0ull;
        uint64_t m;
        if (mask) {
            m = mask[w];
        } else {
            const int below = i + 1 - 64 * w;
            m = below <= 0 ? 0ull : (below >= 64 ? ~0ull : (1ull << below) - 1);
        }
        return live >= 64 ? m : m & ((1ull << live) - 1);
    }
    __device__ __forceinline__ void init(const TreeParams &p, const TreeSeq &q, int node) {
        words = p.tree_mask ? p.mask_words : (q.n + 63) / 64;
        mask = p.tree_mask ? p.tree_mask + (int64_t)(q.row0 + node) * p.mask_words : nullptr;
        i = node;
        n = q.hi - q.c;
        lo = drop = 0;
        const int W = p.a.window;
        if (W > 0) {
            int path = 0;
            for (int w = 0; 64 * w < n; w++) path += __popcll(raw(w));
            drop = path > W ? path - W : 0;
            const int64_t first = (int64_t)q.c + path - W;
            lo = first > 0 ? (int)(first < q.c ? first : q.c) : 0;
        }
    }
    __device__ __forceinline__ uint64_t word(int w) const {
        uint64_t m = raw(w);
        if (drop > 0) {
            int skip = drop;
            for (int u = 0; u < w; u++) skip -= __popcll(raw(u));
            for (; skip > 0 && m; skip--) m &= m - 1;
        }
        return m;
    }
    // bits of the 64 keys from kb on (c: the sequence's cached tokens)
    __device__ __forceinline__ uint64_t keys(int kb, int c) const {
        uint64_t see = 0;
        if (kb < c) {
            const int a = lo - kb, b = c - kb;  // cached keys [a, b) of the 64
            const uint64_t upto = b >= 64 ? ~0ull : (1ull << b) - 1;
            see = a <= 0 ? upto : (a >= 64 ? 0ull : upto & ~((1ull << a) - 1));
        }
        const int off = kb - c;
        if (off > -64) {
            if (off < 0) {
                see |= word(0) << -off;
            } else {
                const int w = off >> 6, sh = off & 63;
                see |= word(w) >> sh;
                if (sh) see |= word(w + 1) << (64 - sh);
            }
        }
        return see;
    }
    __device__ __forceinline__ bool sees(int j, int c) const {
        if (j < c) return j >= lo;
        return (word((j - c) >> 6) >> ((j - c) & 63)) & 1;
    }
};

// first key that some row of a sequence may see
__device__ __forceinline__ int tree_first_key(const TreeParams &p, const TreeSeq &q) {
    const int64_t first = (int64_t)q.c - p.a.window;
    return p.a.window > 0 && first > 0 ? (int)first : 0;
}

// ------------------------------------------------------------------ the split
// The work is cut into units: a block of 2^rows_log2 query rows (token, head) of one kv head
// and 2^keys_log2 keys.  An item is a row block with all its keys; items lie one behind the other
// (sequence, kv head, block), and every workgroup takes a share of `per` units.  Lengths are
// known on the device alone, so each workgroup adds them up itself (64 sequences a step).
// Workgroups that share an item leave a partial each, which tree_reduce_kernel merges in
// order.
//
// Beginning and ending an item takes about 5 us, and its partial as many bytes as its rows,
// so a share holds units of one item (items then begin at multiples of per: `pad`) where that
// costs a workgroup at most a quarter and 4 more units.  One sequence of 4133 tokens, 264 units
// on 256 workgroups: 18 us, and 22 when a share of 2 runs on into the next item; 16 ragged ones
// (tree_mfma.h) 65 us and 72.  But 4 e4m3 sequences of 16384 to 65536 tokens, 150 units a
// workgroup: 306 us with a quarter more, 281 with 4 at most.
struct TreeWork {
    int units, per, group;  // all units, units of a workgroup, this workgroup's place
    int pad;                // items begin at multiples of it
};
struct TreeItem {
    TreeSeq q;
    int s, kvh, rb;     // sequence, kv head, row block
    int blocks;         // row blocks of a kv head
    int tile0, tiles;   // first key's unit and units of the item
    int first;          // its first unit
};

__device__ __forceinline__ int tree_row_blocks(const TreeParams &p, int n) {
    return (n * (p.a.num_heads / p.a.num_kv_heads) + (1 << p.rows_log2) - 1) >> p.rows_log2;
}
__device__ __forceinline__ void tree_tiles(const TreeParams &p, const TreeSeq &q, int &tile0, int &tiles) {
    tile0 = tree_first_key(p, q) >> p.keys_log2;
    tiles = ((q.hi + (1 << p.keys_log2) - 1) >> p.keys_log2) - tile0;
    if (tiles < 1) tiles = 1;  // a row without keys is written too
}
__device__ __forceinline__ void tree_shape(const TreeParams &p, TreeItem &it) {
    it.blocks = tree_row_blocks(p, it.q.n);
    tree_tiles(p, it.q, it.tile0, it.tiles);
}
// shares of `per` units that an item fills
__device__ __forceinline__ int tree_shares(int tiles, int per) {
    return (int)(((uint32_t)tiles + (uint32_t)per - 1) / (uint32_t)per);
}
// units that an item takes, with those left empty behind it
__device__ __forceinline__ int tree_padded(int tiles, int pad) { return tree_shares(tiles, pad) * pad; }
// a sequence's items and units of one (no items past the last sequence)
struct TreeCount {
    int items, tiles;
};
__device__ __forceinline__ TreeCount tree_count(const TreeParams &p, int s, TreeSeq &q) {
    if (s >= p.num_seqs) return {0, 0};
    q = tree_seq(p, s);
    TreeCount n;
    int tile0;
    tree_tiles(p, q, tile0, n.tiles);
    n.items = tree_row_blocks(p, q.n) * p.a.num_kv_heads;
    return n;
}
// Sums over the lanes up to each: DPP moves (row_shr 1, 2, 4, 8, then row_bcast 15 and 31), as a
// chain of 6 shuffles through LDS takes 0.35 us and a workgroup needs three
__device__ __forceinline__ int tree_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
    return v;
}
__device__ __forceinline__ int tree_wave_sum(int v) { return __builtin_amdgcn_readlane(tree_scan(v), 63); }
// The split of the batch; `n`, `q`: the lane's own of the first 64 sequences
__device__ __forceinline__ void tree_share(const TreeParams &p, const TreeCount &n, TreeWork &w) {
    const int lane = threadIdx.x & 63;
    auto shares = [&](int per) {  // at most as many as units
        int sum = n.items * tree_shares(n.tiles, per);
        for (int s = lane + 64; s < p.num_seqs; s += 64) {
            TreeSeq q;
            const TreeCount o = tree_count(p, s, q);
            sum += o.items * tree_shares(o.tiles, per);
        }
        return tree_wave_sum(sum);
    };
    w.units = shares(1);
    w.per = (int)((uint32_t)(w.units + p.groups - 1) / (uint32_t)p.groups);
    w.pad = 1;
    if (w.per <= 1) return;
    const int more = w.per < 16 ? (w.per + 3) / 4 : 4;
    for (int per = w.per; per <= w.per + more; per += more) {
        const int used = shares(per);
        if (used <= p.groups) {
            w.units = used * per;
            w.per = w.pad = per;
            return;
        }
    }
}
// The item that holds unit u; `n`, `q`: the lane's own of the first 64 sequences
__device__ __forceinline__ void tree_find(const TreeParams &p, const TreeWork &w, int u, TreeCount n, TreeSeq q, TreeItem &it) {
    const int lane = threadIdx.x & 63;
    int base = 0, s0 = 0;
    for (;;) {
        const int mine = n.items * tree_padded(n.tiles, w.pad);
        const int upto = tree_scan(mine);
        const uint64_t past = __ballot(base + upto > u);
        if (past) {
            const int at = __builtin_ctzll(past);
            base += __builtin_amdgcn_readlane(upto - mine, at);
            it.s = s0 + at;
            it.q.c = __builtin_amdgcn_readlane(q.c, at);
            it.q.n = __builtin_amdgcn_readlane(q.n, at);
            it.q.hi = __builtin_amdgcn_readlane(q.hi, at);
            it.q.row0 = __builtin_amdgcn_readlane(q.row0, at);
            break;
        }
        base += __builtin_amdgcn_readlane(upto, 63);
        s0 += 64;
        n = tree_count(p, s0 + lane, q);
    }
    it.q.bt = p.a.block_tables + (int64_t)it.s * p.a.bt_stride;
    tree_shape(p, it);
    const int padded = tree_padded(it.tiles, w.pad);
    const int k = (int)((uint32_t)(u - base) / (uint32_t)padded);  // item of the sequence
    it.kvh = (int)((uint32_t)k / (uint32_t)it.blocks);
    it.rb = k - it.kvh * it.blocks;
    it.first = base + k * padded;
}
// This workgroup's share, and the item that holds its first unit (false: it has none)
__device__ __forceinline__ bool tree_start(const TreeParams &p, TreeWork &w, TreeItem &it) {
    TreeSeq q{};
    const TreeCount n = tree_count(p, threadIdx.x & 63, q);
    tree_share(p, n, w);
    // consecutive shares on one XCD, as row blocks of a kv head read the same keys, and as many
    // shares on each
    const int shares = (int)((uint32_t)(w.units + w.per - 1) / (uint32_t)w.per), of_xcd = (shares + kXcds - 1) / kXcds;
    const int place = blockIdx.x / kXcds;
    w.group = (int)(blockIdx.x % kXcds) * of_xcd + place;
    const int u = w.group * w.per;
    if (place >= of_xcd || u >= w.units) return false;
    tree_find(p, w, u, n, q, it);
    return true;
}
// the end of the share's units of an item, and whether others follow in the share
__device__ __forceinline__ int tree_item_end(const TreeItem &it, int end) {
    const int item_end = it.first + it.tiles;
    return item_end < end ? item_end : end;
}
__device__ __forceinline__ bool tree_last(const TreeWork &w, int u, int end) { return w.pad > 1 || u >= end; }
// the item behind it, when there is one (items without padding)
__device__ __forceinline__ void tree_next(const TreeParams &p, TreeItem &it) {
    it.first += it.tiles;
    if (++it.rb < it.blocks) return;
    it.rb = 0;
    if (++it.kvh < p.a.num_kv_heads) return;
    it.kvh = 0;
    do {
        if (++it.s >= p.num_seqs) return;
        it.q = tree_seq(p, it.s);
        tree_shape(p, it);
    } while (it.blocks == 0);
}
// The rows of a block, of the sequence's n G rows of the kv head: parts of PART rows are
// dealt evenly over the item's blocks
struct TreeRows {
    int row0, rows;
};
template <int PART>
__device__ __forceinline__ TreeRows tree_rows(const TreeParams &p, const TreeItem &it) {
    const int n = it.q.n * (p.a.num_heads / p.a.num_kv_heads);
    const int parts = (n + PART - 1) / PART, per = (int)((uint32_t)(parts + it.blocks - 1) / (uint32_t)it.blocks) * PART;
    TreeRows r;
    r.row0 = it.rb * per;
    r.rows = n - r.row0 < per ? n - r.row0 : per;
    if (r.rows < 0) r.rows = 0;
    return r;
}
// A group leaves at most two partials: of the item that its share begins in, and of the one
// that it ends in.
__device__ __forceinline__ int tree_slot(const TreeWork &w, int group, int first) {
    return 2 * group + (first <= group * w.per ? 0 : 1);
}

// 4 dims of a row from N states of it: O at o + i o_stride (unscaled, reference max m),
// (m, l) at ml + i ml_stride
struct TreeSum {
    float a[4], den, M;
};
template <int N>
__device__ __forceinline__ TreeSum tree_sum(const float *o, int o_stride, const float *ml, int ml_stride) {
    TreeSum s{{0.f, 0.f, 0.f, 0.f}, 0.0f, -INFINITY};
#pragma unroll
    for (int i = 0; i < N; i++) s.M = fmaxf(s.M, ml[i * ml_stride]);
    const float mu = s.M == -INFINITY ? 0.0f : s.M;
#pragma unroll
    for (int i = 0; i < N; i++) {
        const float w = __builtin_amdgcn_exp2f(ml[i * ml_stride] - mu);  // 0 for a state without keys
        const float4 v = *reinterpret_cast<const float4 *>(o + i * o_stride);
        s.den += w * ml[i * ml_stride + 1];
        s.a[0] += w * v.x, s.a[1] += w * v.y, s.a[2] += w * v.z, s.a[3] += w * v.w;
    }
    return s;
}
template <typename QT>
__device__ __forceinline__ void tree_out(const TreeParams &p, const TreeItem &it, int row, int e0, TreeSum &s) {
    const int H = p.a.num_heads, G = H / p.a.num_kv_heads, node = (int)((uint32_t)row / (uint32_t)G);
    const float inv = s.den == 0.0f ? 0.0f : 1.0f / s.den;
#pragma unroll
    for (int e = 0; e < 4; e++) s.a[e] *= inv;
    const int64_t at = ((int64_t)(it.q.row0 + node) * H + it.kvh * G + (row - node * G)) * p.a.head_dim + e0;
    store4<QT>(static_cast<QT *>(p.a.out) + at, s.a);
}

// The V elements left out of the products: not finite, of keys [j0, j1) outside [lo_all,
// c), which some rows do not see.  Adds p v to 4 dims of a row that sees them.
template <typename KV, typename QT>
__device__ __forceinline__ void tree_odd(const TreeParams &p, const TreeItem &it, int row, int e0, int j0, int j1,
                                         int lo_all, TreeSum &s) {
    const AttnParams &a = p.a;
    const int G = a.num_heads / a.num_kv_heads, d = a.head_dim, bs = a.block_size;
    TreeRow r;
    r.init(p, it.q, row / G);
    const QT *qr = static_cast<const QT *>(a.q) +
                   ((int64_t)(it.q.row0 + row / G) * a.num_heads + it.kvh * G + row % G) * d;
    const float mu = s.M == -INFINITY ? 0.0f : s.M;
    for (int j = j0; j < j1; j++) {
        if (j >= lo_all && j < it.q.c) {
            j = it.q.c - 1;
            continue;
        }
        if (!r.sees(j, it.q.c)) continue;
        const int blk = tree_block(p, it.q.bt[j / bs]);
        const int64_t off = (pool_slot(blk, bs, j % bs) * a.num_kv_heads + it.kvh) * d;
        f16 ks = (f16)1.0f, vs = (f16)1.0f;
        if constexpr (sizeof(KV) == 1) ks = bits_to_f16(a.k_scale[blk]), vs = bits_to_f16(a.v_scale[blk]);
        float v[4];
        load_kv4<KV>(static_cast<const KV *>(a.v_pool) + off + e0, vs, v);
        if (__builtin_isfinite(v[0]) && __builtin_isfinite(v[1]) && __builtin_isfinite(v[2]) && __builtin_isfinite(v[3]))
            continue;
        float sd = 0.0f;
        for (int e = 0; e < d; e += 4) {
            float kv[4], qv[4];
            load_kv4<KV>(static_cast<const KV *>(a.k_pool) + off + e, ks, kv);
            load4<QT>(qr + e, qv);
            sd += qv[0] * kv[0] + qv[1] * kv[1] + qv[2] * kv[2] + qv[3] * kv[3];
        }
        const float pj = exp2f(sd * a.scale_log2 - mu);
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (!__builtin_isfinite(v[e])) s.a[e] += pj * v[e];
    }
}

__device__ __forceinline__ float *tree_part(const TreeParams &p, int slot) {
    return p.a.part_o + (int64_t)slot * ((p.a.head_dim + 2) << p.rows_log2);  // [rows][d], then [rows] (m, l)
}

// Whether some wave left an element out: `flags`, written before a barrier by each wave (no LDS
// clear, and two barriers fewer than __syncthreads_or)
template <int WAVES>
__device__ __forceinline__ bool tree_any(const int *flags) {
    int any = 0;
#pragma unroll
    for (int w = 0; w < WAVES; w++) any |= flags[w];
    return __builtin_amdgcn_readfirstlane(any) != 0;
}

// A workgroup's rows in LDS (STATES a row: O at o, (m, l) at ml) as outputs, or as its
// partial of an item that others share.  u0, u1: the units of the item that it did.  A row has
// PIECES places for 4 dims.
template <typename KV, typename QT, int ROW_STRIDE, int PIECES, int STATES, int THREADS>
__device__ __forceinline__ void tree_write(const TreeParams &p, const TreeItem &it, const TreeRows &tr, const TreeWork &w,
                                           int u0, int u1, const float *o, int o_stride, const float *ml, int ml_stride,
                                           bool any_odd, int lo_all) {
    const int d = p.a.head_dim;
    const bool whole = u0 == it.first && u1 == it.first + it.tiles;
    float *part = tree_part(p, tree_slot(w, w.group, u0)), *part_ml = part + (d << p.rows_log2);
    const int j0 = (it.tile0 + u0 - it.first) << p.keys_log2, j1 = (it.tile0 + u1 - it.first) << p.keys_log2;
    auto put = [&](int i, bool odd) {
        const int r = i / PIECES, e0 = (i - r * PIECES) * 4;
        if (e0 >= d) return;
        TreeSum s = tree_sum<STATES>(o + r * ROW_STRIDE + e0, o_stride, ml + r * 2, ml_stride);
        if (odd) tree_odd<KV, QT>(p, it, tr.row0 + r, e0, j0, j1 < it.q.hi ? j1 : it.q.hi, lo_all, s);
        if (whole) {
            tree_out<QT>(p, it, tr.row0 + r, e0, s);
        } else {
            store4<float>(part + r * d + e0, s.a);
            if (e0 == 0) *reinterpret_cast<float2 *>(part_ml + 2 * r) = make_float2(s.M, s.den);
        }
    };
    if (!any_odd) {
#pragma unroll 2
        for (int i = threadIdx.x; i < tr.rows * PIECES; i += THREADS) put(i, false);
    } else {
#pragma unroll 1
        for (int i = threadIdx.x; i < tr.rows * PIECES; i += THREADS) put(i, true);
    }
}

}  // namespace pam
