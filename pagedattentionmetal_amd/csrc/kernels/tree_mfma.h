// tree_mfma.h - attention of drafted trees with f16 matrix products (gfx950): f16 and e4m3
// pools, head sizes up to 128.  Included by tree_attention.hip.
//
// A workgroup of 4 waves holds up to 32 RW query rows (token, head) of one kv head: RW
// row parts of 32 rows, and KG = 4 / RW key groups that share a part's keys.  Tiles of KT
// keys go through LDS; S^T = K Q^T and O^T += V^T P^T run on v_mfma_f32_32x32x16_f16: the
// S^T accumulator is P^T's operand as it stands, and V^T is read with the transposing LDS
// load.  Running maxima (moved only past a factor of 2^8) and sums are f32; probabilities
// are rounded to f16 for the second product, and the sums add the rounded ones, so a
// row's weights still add up to one.
#pragma once
#include "prefill_body.h"
#include "tree_body.h"

namespace pam {

template <int HD, int RW>
struct TreeMfma {
    static constexpr int KG = 4 / RW, TS = RW == 4 ? 2 : 1, KT = 32 * KG * TS;
    static constexpr int BUFS = RW == 1 ? 1 : 2;
    static constexpr int LS = HD + 4;                       // floats of an output row in LDS
    static constexpr int RING = BUFS * KT * (pf_kl<HD>() + HD) * 2;
    static constexpr int OUT = 4 * 32 * (LS + 2) * 4;
    static constexpr int LDS = RING > OUT ? RING : OUT;
};

template <typename KV, int HD, int RW>
__global__ __launch_bounds__(256, 2) void tree_mfma_kernel(TreeParams p) {
    typedef TreeMfma<HD, RW> Shape;
    constexpr bool FP8 = sizeof(KV) == 1;
    constexpr int KG = Shape::KG, TS = Shape::TS, KT = Shape::KT, BUFS = Shape::BUFS, LS = Shape::LS;
    constexpr int KL = pf_kl<HD>(), VL = HD, DC = HD / 16, DT = HD / 32, PIECES = HD / 8;
    constexpr int KPP = 256 / PIECES, NP = KT / KPP;  // keys of a staging pass, passes
    __shared__ __attribute__((aligned(16))) char smem[Shape::LDS];
    f16 *k_lds = reinterpret_cast<f16 *>(smem), *v_lds = k_lds + BUFS * KT * KL;
    float *o_lds = reinterpret_cast<float *>(smem), *ml_lds = o_lds + 4 * 32 * LS;

    const AttnParams &a = p.a;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, n = lane & 31, h = lane >> 5;
    const int rw = wave % RW, kg = wave / RW;
    const int G = a.num_heads / a.num_kv_heads, H = a.num_heads, d = a.head_dim, bs = a.block_size;
    const int shift = block_shift(bs);
    const float sl2 = a.scale_log2;
    const f16x2 ones = {(f16)1.0f, (f16)1.0f};
    const int my_piece = tid % PIECES, my_key = tid / PIECES;
    const bool piece_ok = my_piece * 8 < d;
    const uint32_t row_elems = (uint32_t)a.num_kv_heads * d;

    // consecutive ranges of units on one XCD: blocks of a kv head read the same keys
    const int64_t group = (blockIdx.x % kXcds) * (int64_t)(gridDim.x / kXcds) + blockIdx.x / kXcds;
    const TreeWork w = tree_work(p);
    int64_t u = group * w.per;
    const int64_t end = u + w.per < w.units ? u + w.per : w.units;
    if (u >= end) return;
    TreeItem it;
    tree_find(p, u, it);

    // V^T operands: as in the dense prefill (prefill_body.h)
    int v_rd[DT];
    {
        const int o = lane & 15, hh = (lane >> 4) & 1, row = 4 * h + (o >> 2);
#pragma unroll
        for (int dt = 0; dt < DT; dt++) v_rd[dt] = v_lds_at<HD>(row, 4 * dt + 2 * hh + ((o & 3) >> 1)) + 4 * (o & 1);
    }
    const int k_rd = k_lds_at<HD>(n, h);

    for (;;) {
        const int64_t item_end = it.first + it.tiles, u1 = item_end < end ? item_end : end;
        const TreeRows tr = tree_rows(p, it, 32);
        const TreeSeq &q = it.q;
        const int first = tree_first_key(p, q), hi = q.hi;
        const int64_t all = (int64_t)q.c + q.n - a.window;
        const int lo_all = a.window > 0 && all > 0 ? (int)(all < q.c ? all : q.c) : 0;
        const bool active = rw * 32 < tr.rows;
        const int rho = tr.row0 + (rw * 32 + n < tr.rows ? rw * 32 + n : tr.rows - 1), node = rho / G;
        f16x8 qv[DC];
        {
            const f16 *qp = static_cast<const f16 *>(a.q) +
                            ((int64_t)(q.row0 + node) * H + it.kvh * G + (rho - node * G)) * d + 8 * h;
#pragma unroll
            for (int c = 0; c < DC; c++)
                qv[c] = 16 * c + 8 * h < d ? *reinterpret_cast<const f16x8 *>(qp + 16 * c) : (f16x8)(f16)0.0f;
        }

        using Raw = typename std::conditional<FP8, uint2, f16x8>::type;
        Raw rk[NP], rv[NP];
        uint16_t sk[NP], sv[NP];
        int32_t blk[NP];
        const KV *kpool = static_cast<const KV *>(a.k_pool) + (int64_t)it.kvh * d + my_piece * 8;
        const KV *vpool = static_cast<const KV *>(a.v_pool) + (int64_t)it.kvh * d + my_piece * 8;
        auto key_of = [&](int tile, int i) {
            const int j = tile * KT + my_key + i * KPP;
            return j < first ? first : (j < hi ? j : hi - 1);
        };
        auto lookup = [&](int tile) {
#pragma unroll
            for (int i = 0; i < NP; i++) {
                const int j = key_of(tile, i);
                blk[i] = q.bt[shift >= 0 ? j >> shift : j / bs];
            }
        };
        auto fetch = [&](int tile) {
#pragma unroll
            for (int i = 0; i < NP; i++) {
                const int j = key_of(tile, i), b = shift >= 0 ? j >> shift : j / bs;
                const int32_t block = tree_block(p, blk[i]);
                const int64_t off = pool_slot(block, bs, j - b * bs) * row_elems;
                if (piece_ok) {
                    rk[i] = *reinterpret_cast<const Raw *>(kpool + off);
                    rv[i] = *reinterpret_cast<const Raw *>(vpool + off);
                } else {
                    rk[i] = Raw{};
                    rv[i] = Raw{};
                }
                if constexpr (FP8) sk[i] = a.k_scale[block], sv[i] = a.v_scale[block];
            }
        };
        bool odd = false;
        auto stage = [&](int tile, int buf) {
            const bool full = tile * KT >= lo_all && (tile + 1) * KT <= q.c;
#pragma unroll
            for (int i = 0; i < NP; i++) {
                const int key = my_key + i * KPP;
                f16x8 kx, vx;
                if constexpr (FP8) {
                    kx = e4m3x8_to_f16x8(rk[i].x, rk[i].y) * (f16x8)bits_to_f16(sk[i]);
                    vx = e4m3x8_to_f16x8(rv[i].x, rv[i].y) * (f16x8)bits_to_f16(sv[i]);
                } else {
                    kx = rk[i];
                    vx = rv[i];
                }
                if (!full) {
                    // V of keys that some row must not see: not there, or finite (0 * Inf
                    // would reach the rows that mask it; tree_odd gives it to the others)
                    const int j = tile * KT + key;
                    const bool none = j < first || j >= hi, part = !(j >= lo_all && j < q.c);
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const bool bad = part && !__builtin_isfinite((float)vx[e]);
                        odd |= bad && !none;
                        vx[e] = none || bad ? (f16)0.0f : vx[e];
                    }
                }
                *reinterpret_cast<f16x8 *>(k_lds + buf * KT * KL + k_lds_at<HD>(key, my_piece)) = kx;
                *reinterpret_cast<f16x8 *>(v_lds + buf * KT * VL + v_lds_at<HD>(key, my_piece)) = vx;
            }
        };

        float m_use = -INFINITY, m_thr = -INFINITY, l_run = 0.0f;
        f32x16 o[DT];
#pragma unroll
        for (int dt = 0; dt < DT; dt++) o[dt] = (f32x16)0.0f;

        auto compute = [&](int tile, int buf) {
            const f16 *kt = k_lds + buf * KT * KL + kg * TS * 32 * KL, *vt = v_lds + buf * KT * VL + kg * TS * 32 * VL;
            const int kb = tile * KT + kg * TS * 32;
            f32x16 s[TS];
#pragma unroll
            for (int e = 0; e < TS; e++) s[e] = (f32x16)0.0f;
#pragma unroll
            for (int c = 0; c < DC; c++)
#pragma unroll
                for (int e = 0; e < TS; e++) {
                    const f16x8 ka = *reinterpret_cast<const f16x8 *>(&kt[k_rd + 32 * e * KL + 16 * c]);
                    s[e] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ka, qv[c], s[e], 0, 0, 0);
                }
            if (!(kb >= lo_all && kb + 32 * TS <= q.c)) {
                TreeRow row;
                row.init(p, q, node);
                const uint64_t see = row.keys(kb, q.c) >> (4 * h);
#pragma unroll
                for (int e = 0; e < TS; e++)
#pragma unroll
                    for (int r = 0; r < 16; r++)
                        s[e][r] = (see >> (32 * e + 8 * (r >> 2) + (r & 3))) & 1 ? s[e][r] : -INFINITY;
            }
            float mx = -INFINITY;
#pragma unroll
            for (int e = 0; e < TS; e++)
#pragma unroll
                for (int r = 0; r < 16; r += 2) mx = vmax3(mx, s[e][r], s[e][r + 1]);
            if (__any(mx > m_thr)) {
                const float mt = fmaxf(mx, shfl_xor(mx, 32)) * sl2;
                const float m_new = fmaxf(m_use, mt);
                const float corr = m_new == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m_use - m_new);
                l_run *= corr;
#pragma unroll
                for (int dt = 0; dt < DT; dt++) o[dt] *= corr;
                m_use = m_new;
                m_thr = (m_new + kRescaleLog2) / sl2;
            }
            const float mref = m_use == -INFINITY ? 0.0f : m_use;
            f16x8 pb[2 * TS];
#pragma unroll
            for (int e = 0; e < TS; e++)
#pragma unroll
                for (int r = 0; r < 16; r++)
                    pb[2 * e + (r >> 3)][r & 7] = (f16)__builtin_amdgcn_exp2f(fmaf(s[e][r], sl2, -mref));
#pragma unroll
            for (int k = 0; k < 8 * TS; k++) {
                const f16x2 pr = {pb[k >> 2][2 * (k & 3)], pb[k >> 2][2 * (k & 3) + 1]};
                l_run = __builtin_amdgcn_fdot2(pr, ones, l_run, false);
            }
#pragma unroll
            for (int c = 0; c < 2 * TS; c++)
#pragma unroll
                for (int dt = 0; dt < DT; dt++) {
                    const f16x4 lo = lds_read_tr16(vt + v_rd[dt] + 16 * c * VL);
                    const f16x4 up = lds_read_tr16(vt + v_rd[dt] + (16 * c + 8) * VL);
                    const f16x8 va = {lo[0], lo[1], lo[2], lo[3], up[0], up[1], up[2], up[3]};
                    o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va, pb[c], o[dt], 0, 0, 0);
                }
        };

        const int t0 = it.tile0 + (int)(u - it.first), t1 = it.tile0 + (int)(u1 - it.first);
        if (hi > first) {
            lookup(t0);
            fetch(t0);
            if (t0 + 1 < t1) lookup(t0 + 1);
            if constexpr (BUFS == 2) {
                stage(t0, 0);
                __syncthreads();
                for (int t = t0; t < t1; t++) {
                    const int buf = (t - t0) & 1;
                    if (t + 1 < t1) fetch(t + 1);
                    if (t + 2 < t1) lookup(t + 2);
                    __builtin_amdgcn_sched_barrier(0);
                    if (active) compute(t, buf);
                    __builtin_amdgcn_sched_barrier(0);
                    if (t + 1 < t1) stage(t + 1, buf ^ 1);
                    __syncthreads();
                }
            } else {
                for (int t = t0; t < t1; t++) {
                    stage(t, 0);
                    __syncthreads();
                    if (t + 1 < t1) fetch(t + 1);
                    if (t + 2 < t1) lookup(t + 2);
                    __builtin_amdgcn_sched_barrier(0);
                    if (active) compute(t, 0);
                    __syncthreads();
                }
            }
        }

        // the waves' rows in LDS, row-major, then out
        const float l = l_run + shfl_xor(l_run, 32);
        const bool any_odd = __syncthreads_or(odd);
        float *row = o_lds + (wave * 32 + n) * LS;
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const f32x4 x = {o[dt][4 * r], o[dt][4 * r + 1], o[dt][4 * r + 2], o[dt][4 * r + 3]};
                *reinterpret_cast<f32x4 *>(row + 32 * dt + 8 * r + 4 * h) = x;
            }
        if (h == 0) *reinterpret_cast<float2 *>(ml_lds + (wave * 32 + n) * 2) = make_float2(m_use, l);
        __syncthreads();
        tree_write<KV, f16, LS>(p, it, tr, w, group, u, u1, o_lds, (int64_t)RW * 32 * LS, ml_lds, RW * 64, KG, any_odd, lo_all);
        u = u1;
        if (u >= end) break;
        tree_next(p, it);
        __syncthreads();
    }
}

}  // namespace pam
