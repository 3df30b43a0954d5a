// tree_body.h - attention of drafted trees over a paged cache (gfx950): which keys a
// row sees, shared by the kernels of tree_attention.hip.
//
// Sequence s holds c cached tokens and n drafted ones at positions c .. c + n - 1
// (appended to its blocks before the call).  Row (s, i) sees the cached tokens and
// the drafted tokens whose bits its mask has set; with a window W, the last W of the keys
// it sees, in order of position.  A row that sees no key is zeros.
#pragma once
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

}  // namespace pam
