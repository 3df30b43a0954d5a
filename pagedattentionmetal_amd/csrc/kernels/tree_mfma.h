// tree_mfma.h - attention of drafted trees with f16 matrix products (gfx950): f16 and e4m3
// pools, head sizes up to 128, blocks of a power of two tokens.  Included by
// tree_attention.hip.
//
// A workgroup holds up to 32 RW query rows (token, head) of one kv head, RW = 1, 2, 4 or (e4m3)
// 8: RW waves with 32 rows each, and KG = 4 / RW key groups, at least one, each with a ring of
// 32-key tiles in LDS that its RW waves fill.  S^T = K Q^T and O^T += V^T P^T run on
// v_mfma_f32_32x32x16_f16: the S^T accumulator is P^T's operand as it stands, and V^T is read with
// the transposing LDS load.  Running maxima (moved only past a factor of 2^8) and sums are f32;
// probabilities are rounded to f16 for the second product, and the sums add the rounded
// ones, so a row's weights still add up to one.
//
// Rows go from the pools to LDS without registers, several tiles ahead: a tile's 128- or
// 256-byte rows lie all over memory, and it is the bytes under way that give the rate.  e4m3
// codes wait in a ring of their own and are dequantised into the f16 ring two tiles before
// their use (RW <= 2: in registers, one tile ahead).  A tile's row r has its 16-byte piece x at
// x ^ swizzle(r), so that neither the operand loads nor the transposed ones conflict.  The
// block table's entries of a range of tiles (and, e4m3, the blocks' scales) lie in LDS, and a
// request's rows in one block, so its address is a sum of scalars and one constant register:
// 64-bit products in every lane cost 30% of the vector unit's time (f16, 16384 tokens and 256
// rows: 455 us with them, 420 without).
//
// What bounds it (16 sequences, 32 heads on 8, head 128, with the merge): few rows, memory (f16,
// 16384 tokens: 8 nodes 205 us, 5.3 TB/s of KV; 32 nodes 239 us, 4.5 TB/s; e4m3, 8 nodes 129 us,
// 4.2 TB/s); many, the matrix and the vector units, which take turns more than they overlap (f16,
// 64 nodes: 412 us, 0.67 PFLOP/s, matrix units busy a third of the time; the softmax's exponentials
// alone take half as long as the products); one short sequence, latency: 12 us of a 4133-token
// call are the lengths, the table's entries, the tiles, the merge of key groups and the store, one
// behind the other.
#pragma once
#include "tree_body.h"

namespace pam {

template <typename KV, int HD, int RW>
struct TreeMfma {
    static constexpr bool FP8 = sizeof(KV) == 1;
    static constexpr int KG = RW < 4 ? 4 / RW : 1, WAVES = RW * KG;
    static constexpr int ROWS = 32 * RW, KEYS = 32 * KG;    // of a unit
    // the waves on one ring: tile t's weights beside the products of tile t + 1
    static constexpr bool PIPE = RW >= 4;
    static_assert(RW <= 4 || FP8, "f16: at most 128 rows");
    static constexpr int BUFS = PIPE ? (FP8 ? 3 : 4) : (FP8 && RW == 1 ? 1 : 2);  // f16 tiles of a ring
    static constexpr int RAWS = PIPE && FP8 ? (RW == 8 ? 10 : 3) : 0;              // e4m3 tiles
    static constexpr int LS = HD + 4;                       // floats of an output row in LDS
    static constexpr int RING = KG * BUFS * 2 * 32 * HD * 2, RAW = RAWS * 2 * 32 * HD;
    static constexpr int BT = FP8 ? 768 : 1024;             // block-table entries in LDS
    static constexpr int OUT = WAVES * 32 * (LS + 2) * 4, IN = RING + RAW + BT * (FP8 ? 8 : 4);
    static constexpr int LDS = IN > OUT ? IN : OUT;
    static constexpr int PER_CU = RW < 8 && LDS + 512 <= 80 * 1024 ? 2 : 1;  // workgroups of a CU
    static constexpr int EU_WAVES = PER_CU * WAVES / 4;
};

// places of a tile's row: its 16-byte piece x lies at x ^ swizzle
template <int HD>
__device__ __forceinline__ int tree_k_swizzle(int row) { return HD == 128 ? row & 15 : (row >> 1) & 7; }
template <int HD>
__device__ __forceinline__ int tree_v_swizzle(int row) { return HD == 128 ? (row & 3) << 2 : ((row >> 1) & 1) << 2; }

// at most N of the wave's requests to memory are still under way
template <int N>
__device__ __forceinline__ void tree_wait() {
    static_assert(N >= 0 && N < 64, "vmcnt has six bits");
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
// 16 bytes of every lane straight into LDS, at lds_base (a byte offset) + 16 lane: from g, or
// from base + off with base the same in all lanes
__device__ __forceinline__ void tree_dma16(const void *g, uint32_t lds_base) {
    asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds_base), "v"(g) : "memory", "m0");
}
__device__ __forceinline__ void tree_dma16(const void *base, uint32_t off, uint32_t lds_base) {
    asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds_base), "v"(off), "s"(base) : "memory", "m0");
}
// LDS alone: what is under way from memory stays so
__device__ __forceinline__ void tree_lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

template <typename KV, int HD, int RW>
__global__ __launch_bounds__((64 * TreeMfma<KV, HD, RW>::WAVES), (TreeMfma<KV, HD, RW>::EU_WAVES)) void
tree_mfma_kernel(TreeParams p) {
    typedef TreeMfma<KV, HD, RW> Shape;
    constexpr bool FP8 = Shape::FP8;
    constexpr int KG = Shape::KG, KEYS = Shape::KEYS, KEYS_LOG2 = KG == 4 ? 7 : (KG == 2 ? 6 : 5), BUFS = Shape::BUFS, RAWS = Shape::RAWS;
    constexpr int LS = Shape::LS;
    constexpr int DC = HD / 16, DT = HD / 32, TILE = 32 * HD;  // halves of a K or V tile
    // A request takes 64 pieces: RPR rows of K (x even) or V.  A tile has RIN of them, wave rw the
    // RQ from x = rw RQ on, which lie in NG groups of rows.  On a ring, and f16, pieces of 16
    // bytes go to LDS; else of 8 bytes to registers, each request both K and V.
    constexpr bool DMA = !FP8 || RAWS > 0;
    constexpr int PIECE = DMA ? 16 : 8, PIECES = HD * (int)sizeof(KV) / PIECE, RPR = 64 / PIECES;
    constexpr int RIN = 2 * 32 / RPR, RQ = RIN / RW > 0 ? RIN / RW : 1, NG = RQ / 2 > 0 ? RQ / 2 : 1;
    __shared__ __attribute__((aligned(16))) char smem[Shape::LDS];
    __shared__ int odd_lds[Shape::WAVES];
    f16 *ring = reinterpret_cast<f16 *>(smem);
    uint8_t *raw = reinterpret_cast<uint8_t *>(smem + Shape::RING);
    int32_t *bt_lds = reinterpret_cast<int32_t *>(smem + Shape::RING + Shape::RAW);  // FP8: {block, K and V scale}
    float *o_lds = reinterpret_cast<float *>(smem), *ml_lds = o_lds + Shape::WAVES * 32 * LS;

    const AttnParams &a = p.a;
    const int tid = threadIdx.x, lane = tid & 63, n = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int rw = wave % RW, kg = wave / RW;
    const int G = a.num_heads / a.num_kv_heads, H = a.num_heads, d = a.head_dim;
    const int shift = __builtin_ctz((unsigned)a.block_size), bmask = a.block_size - 1;
    const float sl2 = a.scale_log2, inv_sl2 = 1.0f / sl2;
    const f16x2 ones = {(f16)1.0f, (f16)1.0f};
    const uint32_t row_bytes = (uint32_t)(a.num_kv_heads * d * (int)sizeof(KV)), block_bytes = row_bytes << shift;
    const bool whole = d == HD;              // else pieces behind a head's end are zeros
    const uint32_t lds0 = lds_addr(smem);
    const int my_row = lane / PIECES, my_place = lane % PIECES;  // of a request
    const int g0 = rw * RQ / 2;                                  // the wave's first group of rows

    TreeWork w;
    TreeItem it;
    if (!tree_start(p, w, it)) return;
    int u = w.group * w.per;
    const int end = u + w.per < w.units ? u + w.per : w.units;

    // V^T operands: lane (o, hh, h) reads rows 4h + o / 4 (+ 8) of a 16-key chunk at dims 32
    // dt + 16 hh + 4 (o % 4), which gives it keys 4h + {0..3, 8..11} of dim 32 dt + 16 hh + o
    int v_rd[DT];
    {
        const int o = lane & 15, hh = (lane >> 4) & 1, row = 4 * h + (o >> 2);
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
            v_rd[dt] = row * HD + (((4 * dt + 2 * hh + ((o & 3) >> 1)) ^ tree_v_swizzle<HD>(row)) << 3) + 4 * (o & 1);
    }
    const int k_rd = n * HD, k_sw = tree_k_swizzle<HD>(n);

    for (;;) {
        const int u1 = tree_item_end(it, end);
        const TreeRows tr = tree_rows<32>(p, it);
        const TreeSeq &q = it.q;
        const int first = tree_first_key(p, q), hi = q.hi;
        const int64_t all = (int64_t)q.c + q.n - a.window;
        const int lo_all = a.window > 0 && all > 0 ? (int)(all < q.c ? all : q.c) : 0;
        const bool active = rw * 32 < tr.rows;  // a wave without rows computes the last one again, unwritten
        const int rho = tr.row0 + (rw * 32 + n < tr.rows ? rw * 32 + n : tr.rows - 1), node = rho / G;
        f16x8 qv[DC];
        {
            const f16 *qp = static_cast<const f16 *>(a.q) +
                            ((int64_t)(q.row0 + node) * H + it.kvh * G + (rho - node * G)) * d + 8 * h;
#pragma unroll
            for (int c = 0; c < DC; c++)
                qv[c] = 16 * c + 8 * h < d ? *reinterpret_cast<const f16x8 *>(qp + 16 * c) : (f16x8)(f16)0.0f;
        }

        const char *kpool = static_cast<const char *>(a.k_pool) + (int64_t)it.kvh * d * (int)sizeof(KV);
        const char *vpool = static_cast<const char *>(a.v_pool) + (int64_t)it.kvh * d * (int)sizeof(KV);
        const int blk_first = first >> shift, blk_last = (hi - 1) >> shift;  // of the item's keys
        int blk0 = 0;                                                       // first block in bt_lds
        bool odd = false;
        auto k_tile = [&](int buf) { return ring + ((kg * BUFS + buf) * 2) * TILE; };
        // the group's tiles whose keys all rows see: [full0, full0 + fulls)
        const int full0 = (lo_all - kg * 32 + KEYS - 1) >> KEYS_LOG2, full1 = ((q.c - kg * 32 - 32) >> KEYS_LOG2) + 1;
        const uint32_t fulls = full1 > full0 ? full1 - full0 : 0;
        auto full = [&](int t) { return (uint32_t)(t - full0) < fulls; };
        // first key of row group g of the group's tile t, and the place of its block's entry (a
        // group lies in one block).  A group without keys takes the rows of a block that has some:
        // what lies there is masked (K) or hidden (V).
        auto key0 = [&](int t, int g) { return t * KEYS + kg * 32 + g * RPR; };
        auto entry = [&](int j0) {
            const int b = j0 >> shift, c = b < blk_last ? b : blk_last;
            return ((c > blk_first ? c : blk_first) - blk0) * (FP8 ? 2 : 1);
        };
        // lane i: the entry of the wave's row group g0 + i
        const int lane_key = key0(0, g0 + (lane & (NG - 1)));
        struct Entry {
            int32_t block, scales;
            uint32_t row;  // of the block, in bytes
        };
        auto lookup = [&](int t) {
            const int j0 = t * KEYS + lane_key, at = entry(j0);
            Entry e{bt_lds[at], 0, (uint32_t)(j0 & bmask) * row_bytes};
            if constexpr (FP8 && !DMA) e.scales = bt_lds[at + 1];
            return e;
        };
        // bytes before row group g0 + i, the same in all lanes
        auto offset = [&](int i, uint64_t lanes) {
            return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)lanes, i) |
                   (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(lanes >> 32), i) << 32;
        };
        auto offsets = [&](const Entry &e) { return (uint64_t)(uint32_t)e.block * block_bytes + e.row; };
        // V of keys that some row must not see: not there, or finite (0 * Inf would reach the
        // rows that mask it; tree_odd gives it to the others)
        auto hide = [&](int j, f16x8 &x) {
            const bool none = j < first || j >= hi, part = !(j >= lo_all && j < q.c);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const bool bad = part && !__builtin_isfinite((float)x[e]);
                odd |= bad && !none;
                x[e] = none || bad ? (f16)0.0f : x[e];
            }
        };
        // --- the wave's requests of tile t on their way to a ring place: f16 in the places of
        // their swizzle, codes in order
        auto request = [&](int t, int place, const Entry &e) {
            const uint32_t half = 32 * HD * sizeof(KV);
            const uint32_t to = lds0 + (FP8 ? Shape::RING : 0) + (uint32_t)(kg * BUFS + place) * 2 * half;
            const uint64_t lanes = offsets(e);
            if (RIN < RW && rw >= RIN) return;
#pragma unroll
            for (int i = 0; i < RQ; i++) {
                const int x = rw * RQ + i, g = x >> 1, r = g * RPR + my_row;
                const bool v = RQ > 1 ? i & 1 : x & 1;
                const int piece = FP8 ? my_place : my_place ^ (v ? tree_v_swizzle<HD>(r) : tree_k_swizzle<HD>(r));
                const char *base = (v ? vpool : kpool) + offset(RQ > 1 ? i >> 1 : 0, lanes);
                const uint32_t off = (uint32_t)my_row * row_bytes + piece * 16, dst = to + v * half + g * 1024;
                if (whole)
                    tree_dma16(base, off, dst);
                else
                    tree_dma16(piece * 16 < d * (int)sizeof(KV) ? base + off : static_cast<const char *>(a.zero_page), dst);
            }
        };
        // a wave cleans the V rows that it asked for
        auto clean = [&](int t, int buf) {
            if (full(t) || (RIN < RW && rw >= RIN) || (RQ == 1 && !(rw & 1))) return;
            f16 *vt = k_tile(buf) + TILE + lane * 8;
#pragma unroll 2
            for (int g = g0; g < g0 + NG; g++) {
                f16x8 x = *reinterpret_cast<const f16x8 *>(vt + g * 512);
                hide(key0(t, g) + my_row, x);
                *reinterpret_cast<f16x8 *>(vt + g * 512) = x;
            }
        };
        // --- e4m3 on few waves: a tile's codes in registers, dequantised to their ring place
        struct Regs {
            uint2 k[NG], v[NG];
            uint32_t s[NG];
        };
        auto fetch = [&](int t, Regs &x) {
            const Entry e = lookup(t);
            const uint64_t lanes = offsets(e);
#pragma unroll
            for (int i = 0; i < NG; i++) {
                const int r = (g0 + i) * RPR + my_row;
                const int kx = my_place ^ tree_k_swizzle<HD>(r), vx = my_place ^ tree_v_swizzle<HD>(r);
                const uint64_t off = offset(i, lanes);
                const uint32_t row = (uint32_t)my_row * row_bytes;
                const char *ka = kpool + off, *va = vpool + off;
                if (whole) {
                    x.k[i] = *reinterpret_cast<const uint2 *>(ka + (row + kx * 8));
                    x.v[i] = *reinterpret_cast<const uint2 *>(va + (row + vx * 8));
                } else {
                    const char *zero = static_cast<const char *>(a.zero_page);
                    x.k[i] = *reinterpret_cast<const uint2 *>(kx * 8 < d ? ka + (row + kx * 8) : zero);
                    x.v[i] = *reinterpret_cast<const uint2 *>(vx * 8 < d ? va + (row + vx * 8) : zero);
                }
                x.s[i] = (uint32_t)__builtin_amdgcn_readlane(e.scales, i);
            }
        };
        auto stage = [&](int t, int buf, const Regs &x) {
            const bool all = full(t);
#pragma unroll
            for (int i = 0; i < NG; i++) {
                f16 *kt = k_tile(buf) + (g0 + i) * RPR * HD + lane * 8;
                *reinterpret_cast<f16x8 *>(kt) =
                    e4m3x8_to_f16x8(x.k[i].x, x.k[i].y) * (f16x8)bits_to_f16((uint16_t)x.s[i]);
                f16x8 v = e4m3x8_to_f16x8(x.v[i].x, x.v[i].y) * (f16x8)bits_to_f16((uint16_t)(x.s[i] >> 16));
                if (!all) hide(key0(t, g0 + i) + my_row, v);
                *reinterpret_cast<f16x8 *>(kt + TILE) = v;
            }
        };
        // --- e4m3 on a ring: a wave dequantises the codes that it asked for
        auto dequant = [&](int t, int place, int buf) {
            if (RIN < RW && rw >= RIN) return;
#pragma unroll
            for (int i = 0; i < RQ; i++) {
                const int x = rw * RQ + i, g = x >> 1, r = g * RPR + my_row;
                const bool v = RQ > 1 ? i & 1 : x & 1;
                const uint4 c = *reinterpret_cast<const uint4 *>(raw + (place * 2 + v) * 32 * HD + g * 1024 + lane * 16);
                const uint32_t s = (uint32_t)bt_lds[entry(key0(t, g)) + 1];
                const f16x8 sc = (f16x8)bits_to_f16((uint16_t)(v ? s >> 16 : s));
                f16x8 lo = e4m3x8_to_f16x8(c.x, c.y) * sc, up = e4m3x8_to_f16x8(c.z, c.w) * sc;
                if (v && !full(t)) {
                    hide(key0(t, g) + my_row, lo);
                    hide(key0(t, g) + my_row, up);
                }
                f16 *row = k_tile(buf) + (v ? TILE : 0) + r * HD;
                const int sw = v ? tree_v_swizzle<HD>(r) : tree_k_swizzle<HD>(r);
                *reinterpret_cast<f16x8 *>(row + (((2 * my_place) ^ sw) << 3)) = lo;
                *reinterpret_cast<f16x8 *>(row + (((2 * my_place + 1) ^ sw) << 3)) = up;
            }
        };

        float m_use = -INFINITY, m_thr = -INFINITY, l_run = 0.0f;
        f32x16 o[DT];
#pragma unroll
        for (int dt = 0; dt < DT; dt++) o[dt] = (f32x16)0.0f;

        // S^T of the wave's 32 keys of a tile: accumulator register r is key
        // 8 (r / 4) + 4 h + r % 4 of row n
        auto load_k = [&](int buf, f16x8 (&kf)[DC]) {
            const f16 *kt = k_tile(buf) + k_rd;
#pragma unroll
            for (int c = 0; c < DC; c++) kf[c] = *reinterpret_cast<const f16x8 *>(kt + (((2 * c + h) ^ k_sw) << 3));
        };
        auto score = [&](const f16x8 (&kf)[DC], f32x16 &s) {
            s = (f32x16)0.0f;
#pragma unroll
            for (int c = 0; c < DC; c++) s = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[c], qv[c], s, 0, 0, 0);
        };
        // masks, and the reference maximum raised where a score passes it by 2^8
        auto settle = [&](int tile, f32x16 &s) {
            if (!full(tile)) {
                TreeRow row;
                row.init(p, q, node);
                const uint32_t see = (uint32_t)row.keys(tile * KEYS + kg * 32, q.c) >> (4 * h);
#pragma unroll
                for (int r = 0; r < 16; r++) s[r] = (see >> (8 * (r >> 2) + (r & 3))) & 1 ? s[r] : -INFINITY;
            }
            float mx = vmax3(s[0], s[1], s[2]);
#pragma unroll
            for (int r = 3; r < 15; r += 2) mx = vmax3(mx, s[r], s[r + 1]);
            mx = __builtin_elementwise_maximum(mx, s[15]);
            if (__any(mx > m_thr)) {
                const float mt = fmaxf(mx, shfl_xor(mx, 32)) * sl2;
                const float m_new = fmaxf(m_use, mt);
                const float corr = m_new == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m_use - m_new);
                l_run *= corr;
#pragma unroll
                for (int dt = 0; dt < DT; dt++) o[dt] *= corr;
                m_use = m_new;
                m_thr = (m_new + kRescaleLog2) * inv_sl2;
            }
        };
        // P^T in f16, as the second product's operand, and the sum of what it holds
        auto weigh = [&](const f32x16 &s, f16x8 (&pb)[2]) {
            const float mref = m_use == -INFINITY ? 0.0f : m_use;
#pragma unroll
            for (int r = 0; r < 16; r++) pb[r >> 3][r & 7] = (f16)__builtin_amdgcn_exp2f(fmaf(s[r], sl2, -mref));
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const f16x2 pr = {pb[k >> 2][2 * (k & 3)], pb[k >> 2][2 * (k & 3) + 1]};
                l_run = __builtin_amdgcn_fdot2(pr, ones, l_run, false);
            }
        };
        auto load_v = [&](int buf, f16x8 (&vf)[2][DT]) {
            const f16 *vt = k_tile(buf) + TILE;
#pragma unroll
            for (int c = 0; c < 2; c++)
#pragma unroll
                for (int dt = 0; dt < DT; dt++) {
                    const f16x4 lo = lds_read_tr16(vt + v_rd[dt] + 16 * c * HD);
                    const f16x4 up = lds_read_tr16(vt + v_rd[dt] + (16 * c + 8) * HD);
                    vf[c][dt] = (f16x8){lo[0], lo[1], lo[2], lo[3], up[0], up[1], up[2], up[3]};
                }
        };
        auto value = [&](const f16x8 (&vf)[2][DT], const f16x8 (&pb)[2]) {
#pragma unroll
            for (int c = 0; c < 2; c++)
#pragma unroll
                for (int dt = 0; dt < DT; dt++)
                    o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[c][dt], pb[c], o[dt], 0, 0, 0);
        };
        // N products in order, each followed by its share of other work: a product takes the
        // matrix unit 32 cycles, in which the vector unit is free (the compiler would put the
        // products side by side)
        auto slots = [&](auto count, auto &&product, auto &&work) {
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < decltype(count)::value; i++) {
                product(i);
                __builtin_amdgcn_sched_barrier(0);
                work(i);
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        auto score_part = [&](int c, const f16x8 (&kf)[DC], f32x16 &s) {
            s = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[c], qv[c], c ? s : (f32x16)0.0f, 0, 0, 0);
        };
        // weigh in N shares: share i takes the exponentials [16 i / N, 16 (i + 1) / N) and packs
        // those of share i - 1; share N packs the last
        auto weigh_part = [&](int i, auto count, float mref, f32x16 &s, f16x8 (&pb)[2]) {
            constexpr int N = decltype(count)::value, E = 16 / N;
            if (i < N) {
#pragma unroll
                for (int e = 0; e < E; e++) s[i * E + e] = __builtin_amdgcn_exp2f(fmaf(s[i * E + e], sl2, -mref));
            }
#pragma unroll
            for (int r = (i - 1) * E; r < i * E; r++)
                if (r > 0 && r % 2 == 1) {
                    const f16x2 x = {(f16)s[r - 1], (f16)s[r]};
                    pb[r >> 3][(r & 7) - 1] = x[0];
                    pb[r >> 3][r & 7] = x[1];
                    l_run = __builtin_amdgcn_fdot2(x, ones, l_run, false);
                }
        };
        auto reference = [&]() { return m_use == -INFINITY ? 0.0f : m_use; };
        auto load_v_part = [&](int buf, int x, f16x8 (&vf)[2][DT]) {
            const f16 *vt = k_tile(buf) + TILE + v_rd[x % DT] + 16 * (x / DT) * HD;
            const f16x4 lo = lds_read_tr16(vt), up = lds_read_tr16(vt + 8 * HD);
            vf[x / DT][x % DT] = (f16x8){lo[0], lo[1], lo[2], lo[3], up[0], up[1], up[2], up[3]};
        };

        const int t0 = it.tile0 + u - it.first, t1 = it.tile0 + u1 - it.first;
        // ranges of tiles whose block-table entries fit bt_lds
        const int64_t fit = ((int64_t)(Shape::BT - 1) << shift) / KEYS;
        const int range = fit < t1 - t0 ? (int)fit : t1 - t0;
        for (int c0 = t0; hi > first && c0 < t1; c0 += range) {
            const int c1 = c0 + range < t1 ? c0 + range : t1;
            const int j0 = c0 * KEYS > first ? c0 * KEYS : first, j1 = c1 * KEYS < hi ? c1 * KEYS : hi;
            blk0 = j0 >> shift;
            const int entries = ((j1 - 1) >> shift) - blk0 + 1;
            if (c0 != t0) __syncthreads();
            for (int i = tid; i < entries; i += 64 * Shape::WAVES) {
                const int32_t block = tree_block(p, q.bt[blk0 + i]);
                if constexpr (FP8)
                    *reinterpret_cast<int2 *>(bt_lds + 2 * i) =
                        make_int2(block, (int)((uint32_t)a.k_scale[block] | (uint32_t)a.v_scale[block] << 16));
                else
                    bt_lds[i] = block;
            }
            __syncthreads();
            // the queries have arrived: no wait for them, and for the requests behind them, in the loop
#pragma unroll
            for (int c = 0; c < DC; c++) asm volatile("" : "+v"(qv[c]));
            f32x16 s;
            f16x8 kf[DC], vf[2][DT], pb[2];
            if constexpr (Shape::PIPE) {
                // Turn t: tile t's weights beside the scores of tile t + 1, then its values.  By
                // its end tile t + 2 is whole in the ring.  f16: tile t + BUFS - 1 is asked for
                // into the place that tile t - 1 has left.  e4m3: tile t + 2 is dequantised, and
                // its place among the codes takes tile t + 2 + RAWS.
                constexpr int AHEAD = FP8 ? RAWS : BUFS - 1, PER = RQ;
                f32x16 sn;
                Entry e;
                int b0 = 0, b1 = 1, b2 = 2, rp = 0;  // places of tiles t, t + 1, t + 2; e4m3: of t + 2's codes
                auto rp_next = [&]() { rp = rp + 1 < RAWS ? rp + 1 : 0; };
                auto last = [&](int t) { return t < c1 ? t : c1 - 1; };
                if constexpr (FP8) {
                    for (int i = 0; i < RAWS && c0 + i < c1; i++) request(c0 + i, i, lookup(c0 + i));
#pragma unroll 1
                    for (int i = 0; i < 2 && c0 + i < c1; i++) {
                        if (c0 + i + RAWS - 1 < c1)
                            tree_wait<(AHEAD - 1) * PER>();
                        else
                            tree_wait<0>();
                        dequant(c0 + i, rp, i);
                        if (c0 + i + RAWS < c1) request(c0 + i + RAWS, rp, lookup(c0 + i + RAWS));
                        rp_next();
                    }
                } else {
#pragma unroll 1
                    for (int i = 0; i < AHEAD && c0 + i < c1; i++) request(c0 + i, i, lookup(c0 + i));
                    if (c0 + AHEAD - 1 < c1)
                        tree_wait<(AHEAD - 2) * PER>();
                    else
                        tree_wait<0>();
                    clean(c0, 0);
                    if (c0 + 1 < c1) clean(c0 + 1, 1);
                }
                e = lookup(last(c0 + (FP8 ? 2 : 0) + AHEAD));
                __syncthreads();
                if (active) {
                    load_k(0, kf);
                    score(kf, s);
                }
                int bn = BUFS - 1;  // f16: the place that takes tile t + BUFS - 1
#pragma unroll 1
                for (int t = c0; t < c1; t++) {
                    if (active) load_k(b1, kf);  // behind the last tile: not used
                    if constexpr (FP8) {
                        if (t + 2 < c1) {
                            if (t + 2 + RAWS - 1 < c1)
                                tree_wait<(AHEAD - 1) * PER>();
                            else
                                tree_wait<0>();
                            dequant(t + 2, rp, b2);
                            if (t + 2 + RAWS < c1) request(t + 2 + RAWS, rp, e);
                            rp_next();
                        }
                    } else if (t + AHEAD < c1) {
                        request(t + AHEAD, bn, e);
                    }
                    if (active) {
                        settle(t, s);
                        constexpr std::integral_constant<int, DC> products{};
                        const float mref = reference();
                        slots(products, [&](int i) { score_part(i, kf, sn); },
                              [&](int i) {
                                  weigh_part(i, products, mref, s, pb);
                                  load_v_part(b0, i, vf);
                              });
                        weigh_part(products, products, mref, s, pb);
                        value(vf, pb);
                        s = sn;
                    }
                    bn = b0;
                    b0 = b1, b1 = b2;
                    if constexpr (FP8) {
                        b2 = bn;
                    } else {
                        b2 = b2 + 1 < BUFS ? b2 + 1 : 0;
                        if (t + AHEAD < c1)
                            tree_wait<(AHEAD - 2) * PER>();
                        else
                            tree_wait<0>();
                        if (t + 2 < c1) clean(t + 2, b1);
                    }
                    e = lookup(last(t + 1 + (FP8 ? 2 : 0) + AHEAD));
                    tree_lds_barrier();
                }
            } else {
                Regs g;
                if constexpr (FP8)
                    fetch(c0, g);
                else
                    request(c0, 0, lookup(c0));
                int b = 0;
#pragma unroll 1
                for (int t = c0; t < c1; t++) {
                    const int b_next = b + 1 < BUFS ? b + 1 : 0;
                    if constexpr (RW > 1) __syncthreads();  // the other place has been read
                    if constexpr (FP8) {
                        stage(t, b, g);
                        if (t + 1 < c1) fetch(t + 1, g);
                    } else if (t + 1 < c1) {
                        // one wave has no barrier above: its own reads of the place are done
                        if constexpr (RW == 1) asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                        request(t + 1, b_next, lookup(t + 1));
                        tree_wait<RQ>();
                    } else {
                        tree_wait<0>();
                    }
                    if constexpr (!FP8) clean(t, b);
                    if constexpr (RW > 1) tree_lds_barrier();
                    if (active) {
                        load_k(b, kf);
                        score(kf, s);
                        load_v(b, vf);
                        settle(t, s);
                        weigh(s, pb);
                        value(vf, pb);
                    }
                    b = b_next;
                }
            }
        }

        // the waves' rows in LDS, row-major, then out
        __syncthreads();
        {
            const float l = l_run + shfl_xor(l_run, 32);
            float *row = o_lds + (wave * 32 + n) * LS;
#pragma unroll
            for (int dt = 0; dt < DT; dt++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const f32x4 x = {o[dt][4 * r], o[dt][4 * r + 1], o[dt][4 * r + 2], o[dt][4 * r + 3]};
                    *reinterpret_cast<f32x4 *>(row + 32 * dt + 8 * r + 4 * h) = x;
                }
            if (h == 0) *reinterpret_cast<float2 *>(ml_lds + (wave * 32 + n) * 2) = make_float2(m_use, l);
            const bool wave_odd = __any(odd);
            if (lane == 0) odd_lds[wave] = wave_odd;
        }
        __syncthreads();
        const bool any_odd = tree_any<Shape::WAVES>(odd_lds);
        tree_write<KV, f16, LS, HD / 4, KG, 64 * Shape::WAVES>(p, it, tr, w, u, u1, o_lds, RW * 32 * LS, ml_lds, RW * 64,
                                                               any_odd, lo_all);
        u = u1;
        if (tree_last(w, u, end)) break;
        tree_next(p, it);
        __syncthreads();
    }
}

}  // namespace pam
