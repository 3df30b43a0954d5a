// qk_norm_rope.hip - RMS norm of every query and key head with the position rotation
// in the same pass, and its gradients (gfx950).
//
//   y = R(pos) (x r w),  r = 1 / sqrt(mean(x^2) + eps)
// R turns the pairs (i, i + D/2) or, interleaved, (2i, 2i + 1) of the first D dims by
// pos * f_i.  With g = R^T dy:
//   dw = sum over rows of g x r,   dx = r (g w - x r^2 mean(g w x))
//
// The angle.  pos * f_i reaches far past what binary32 holds, so f_i comes as a 64-bit
// binary fraction of a turn per position (NormRopeParams::freq): the product modulo
// 2^64 is the exact fraction of a turn of that frequency, whatever the position.  Its
// upper 32 bits give the quarter turn and a remainder of at most pi / 4, whose sine and
// cosine are Taylor sums (largest error 2e-9).
//
// Layout.  A lane group of LPR lanes holds one head's row; a lane's unit is V pairs:
// elements uV .. uV + V - 1 and D/2 + uV .. (or 2uV .. 2uV + 2V - 1), so a pair never
// leaves its lane and the only exchange is the row's sum of squares.  V is 8 halves or 4
// floats where rows, strides and pointers are whole 16-byte pieces, 1 otherwise.  A
// workgroup takes a few tokens: every angle is computed once into LDS and serves all
// heads of its token.
//
// What bounds it: the rows' bytes, each read and written once (4133 f32 tokens of 16 + 4 heads:
// 18.4 us, 4.6 TB/s; the gradients of 8192 f16 tokens of 32 + 8:
// 46 us, 5.4 TB/s); a decode batch, the
// launch and one trip to memory (64 f16 tokens: 4.9 us).
#include <algorithm>

#include "pam_device.h"
#include "speculative.h"

namespace pam {

constexpr int kRopeThreads = 256;

// cosine and sine of a binary fraction of a turn
__device__ __forceinline__ float2 turn_cos_sin(uint64_t turn) {
    const uint32_t hi = (uint32_t)(turn >> 32);
    const uint32_t quarter = (hi + 0x20000000u) >> 30;
    const float x = (float)(int32_t)(hi - (quarter << 30)) * 1.46291807926715968e-9f;  // 2 pi / 2^32
    const float x2 = x * x;
    const float s = x + x * x2 * (-1.0f / 6 + x2 * (1.0f / 120 + x2 * (-1.0f / 5040 + x2 * (1.0f / 362880))));
    const float c =
        1.0f + x2 * (-0.5f + x2 * (1.0f / 24 + x2 * (-1.0f / 720 + x2 * (1.0f / 40320 + x2 * (-1.0f / 3628800)))));
    float cc = quarter & 1 ? s : c, ss = quarter & 1 ? c : s;
    if (quarter == 1 || quarter == 2) cc = -cc;
    if (quarter & 2) ss = -ss;
    return make_float2(cc, ss);
}

template <typename T, int V>
struct RopeVec {
    typedef T Raw __attribute__((ext_vector_type(V)));
    static __device__ __forceinline__ void load(const T *p, float *x) {
        const Raw r = *reinterpret_cast<const Raw *>(p);
#pragma unroll
        for (int i = 0; i < V; i++) x[i] = (float)r[i];
    }
    static __device__ __forceinline__ void store(T *p, const float *x) {
        Raw r;
#pragma unroll
        for (int i = 0; i < V; i++) r[i] = (T)x[i];
        // past the L2's lines: what stays dirty there is written back when the kernel ends, and the
        // next waits for it (4133 f32 prompt tokens: 18.4 us, with plain stores 19.6)
        __builtin_nontemporal_store(r, reinterpret_cast<Raw *>(p));
    }
};
template <typename T>
struct RopeVec<T, 1> {
    static __device__ __forceinline__ void load(const T *p, float *x) { x[0] = (float)*p; }
    static __device__ __forceinline__ void store(T *p, const float *x) { *p = (T)x[0]; }
};

// A lane's unit u of a row: two pieces of V elements at a0 and a1, rotated when `turned`
// (pair indices pair0 .. pair0 + V - 1)
struct RopeUnit {
    int a0, a1, pair0;
    bool turned;
};
template <int V>
__device__ __forceinline__ RopeUnit rope_unit(const NormRopeParams &p, int u) {
    RopeUnit r;
    const int half = p.rotary_dim / 2;
    r.pair0 = u * V;
    r.turned = r.pair0 < half;
    if (r.turned && !p.interleaved)
        r.a0 = u * V, r.a1 = half + u * V;
    else
        r.a0 = 2 * u * V, r.a1 = r.a0 + V;
    return r;
}

// the cosines and sines of a token's pairs that a unit needs (LDS row of float2)
template <int V>
__device__ __forceinline__ void rope_turn(const float2 *cs, const RopeUnit &u, bool interleaved, bool back, float *a, float *b) {
    if (!u.turned) return;
    if (!interleaved) {
#pragma unroll
        for (int i = 0; i < V; i++) {
            const float2 t = cs[u.pair0 + i];
            const float s = back ? -t.y : t.y, x = a[i], y = b[i];
            a[i] = x * t.x - y * s;
            b[i] = y * t.x + x * s;
        }
    } else if constexpr (V == 1) {
        const float2 t = cs[u.pair0];
        const float s = back ? -t.y : t.y, x = a[0], y = b[0];
        a[0] = x * t.x - y * s;
        b[0] = y * t.x + x * s;
    } else {
#pragma unroll
        for (int i = 0; i < V; i++) {
            float *e = i < V / 2 ? a + 2 * i : b + 2 * (i - V / 2);
            const float2 t = cs[u.pair0 + i];
            const float s = back ? -t.y : t.y, x = e[0], y = e[1];
            e[0] = x * t.x - y * s;
            e[1] = y * t.x + x * s;
        }
    }
}

// the angles of tokens t0 .. t1 - 1 into cs ([token][rotary_dim / 2])
__device__ __forceinline__ void rope_angles(const NormRopeParams &p, int t0, int t1, float2 *cs) {
    const int half = p.rotary_dim / 2;
    for (int i = threadIdx.x; i < (t1 - t0) * half; i += blockDim.x) {
        const int t = i / half, f = i - t * half;
        cs[i] = turn_cos_sin((uint64_t)(int64_t)p.positions[t0 + t] * p.freq[f]);
    }
}

// grid: x = groups of `tokens` tokens, y = slices of the heads
template <typename T, int V, int LPR, int NU>
__global__ __launch_bounds__(kRopeThreads) void norm_rope_kernel(NormRopeParams p, int tokens) {
    extern __shared__ float2 cs[];
    const int d = p.head_dim, H = p.num_heads, K = p.num_kv_heads, half = p.rotary_dim / 2;
    const int t0 = blockIdx.x * tokens, t1 = t0 + tokens < p.num_tokens ? t0 + tokens : p.num_tokens;
    rope_angles(p, t0, t1, cs);
    __syncthreads();
    constexpr int GROUPS = kRopeThreads / LPR;
    const int u0 = threadIdx.x % LPR, group = threadIdx.x / LPR;
    const bool pool = p.k_pool != nullptr;
    const int heads = H + K + (pool ? K : 0);  // queries, keys, values to copy
    const int per = (heads + gridDim.y - 1) / gridDim.y, h_lo = blockIdx.y * per;
    const int h_n = h_lo + per < heads ? per : heads - h_lo;
    const int units = d / (2 * V);
    for (int r = group; r < (t1 - t0) * h_n; r += GROUPS) {
        const int tl = r / h_n, head = h_lo + r - tl * h_n, t = t0 + tl;
        const bool is_q = head < H, is_v = head >= H + K;
        const int kh = is_q ? 0 : (is_v ? head - H - K : head - H);
        int64_t slot = -1;
        if (pool && !is_q) {
            slot = p.slot_mapping[t];
            if (p.pool_slots && slot >= p.pool_slots) slot = -1;
            if (is_v && slot < 0) continue;
        }
        const T *in = is_q ? static_cast<const T *>(p.q) + t * p.q_stride + head * d
                           : (is_v ? static_cast<const T *>(p.v) + t * p.v_stride + kh * d
                                   : static_cast<const T *>(p.k) + t * p.k_stride + kh * d);
        float a[NU][V], b[NU][V];
        float ss = 0.0f;
#pragma unroll
        for (int n = 0; n < NU; n++) {
            const int u = u0 + n * LPR;
            if (u < units) {
                const RopeUnit ru = rope_unit<V>(p, u);
                RopeVec<T, V>::load(in + ru.a0, a[n]);
                RopeVec<T, V>::load(in + ru.a1, b[n]);
            } else {
#pragma unroll
                for (int i = 0; i < V; i++) a[n][i] = b[n][i] = 0.0f;
            }
#pragma unroll
            for (int i = 0; i < V; i++) ss += a[n][i] * a[n][i] + b[n][i] * b[n][i];
        }
        ss = wave_sum_xor(ss, 1, LPR);
        const float rs = p.normalize ? 1.0f / sqrtf(ss / (float)d + p.eps) : 1.0f;
        const T *w = static_cast<const T *>(is_q ? p.q_weight : p.k_weight);
#pragma unroll
        for (int n = 0; n < NU; n++) {
            const int u = u0 + n * LPR;
            if (u >= units) continue;
            const RopeUnit ru = rope_unit<V>(p, u);
            if (!is_v) {
                float wa[V], wb[V];
                if (w) {
                    RopeVec<T, V>::load(w + ru.a0, wa);
                    RopeVec<T, V>::load(w + ru.a1, wb);
                }
#pragma unroll
                for (int i = 0; i < V; i++) {
                    a[n][i] *= rs * (w ? wa[i] : 1.0f);
                    b[n][i] *= rs * (w ? wb[i] : 1.0f);
                }
                rope_turn<V>(cs + tl * half, ru, p.interleaved, false, a[n], b[n]);
            }
            if (is_q) {
                T *o = static_cast<T *>(p.q_out) + t * p.q_out_stride + head * d;
                RopeVec<T, V>::store(o + ru.a0, a[n]);
                RopeVec<T, V>::store(o + ru.a1, b[n]);
                continue;
            }
            if (!is_v && p.k_out) {
                T *o = static_cast<T *>(p.k_out) + t * p.k_out_stride + kh * d;
                RopeVec<T, V>::store(o + ru.a0, a[n]);
                RopeVec<T, V>::store(o + ru.a1, b[n]);
            }
            if (slot >= 0) {
                T *o = static_cast<T *>(is_v ? p.v_pool : p.k_pool) + (slot * K + kh) * d;
                RopeVec<T, V>::store(o + ru.a0, a[n]);
                RopeVec<T, V>::store(o + ru.a1, b[n]);
            }
        }
    }
}

// Gradients.  A workgroup takes tokens blockIdx.x, + gridDim.x, ..; queries and keys in
// turn, so that a lane's 2 V sums of a weight's gradient stay in registers; the lane
// groups' sums join over the wave, then over the waves in LDS, in a fixed order, and
// the workgroup leaves them in `partial`.
constexpr int kRopeBackTokens = 4;
template <typename T, int V, int LPR, int NU>
__global__ __launch_bounds__(kRopeThreads) void norm_rope_backward_kernel(NormRopeParams p) {
    extern __shared__ float2 cs[];
    constexpr int GROUPS = kRopeThreads / LPR, WAVES = kRopeThreads / 64;
    const int d = p.head_dim, H = p.num_heads, K = p.num_kv_heads, half = p.rotary_dim / 2;
    float *sums = reinterpret_cast<float *>(cs + kRopeBackTokens * half);  // [WAVES][2][d]
    const int u0 = threadIdx.x % LPR, group = threadIdx.x / LPR;
    const int units = d / (2 * V);
    float gw[2][NU][2][V];
#pragma unroll
    for (int w = 0; w < 2; w++)
#pragma unroll
        for (int n = 0; n < NU; n++)
#pragma unroll
            for (int i = 0; i < V; i++) gw[w][n][0][i] = gw[w][n][1][i] = 0.0f;
    const float inv_d = 1.0f / (float)d;
    for (int64_t t0 = (int64_t)blockIdx.x * kRopeBackTokens; t0 < p.num_tokens; t0 += (int64_t)gridDim.x * kRopeBackTokens) {
        const int t1 = (int)(t0 + kRopeBackTokens < p.num_tokens ? t0 + kRopeBackTokens : p.num_tokens);
        __syncthreads();
        rope_angles(p, (int)t0, t1, cs);
        __syncthreads();
#pragma unroll
        for (int part = 0; part < 2; part++) {
            const int heads = part == 0 ? H : K;
            const T *x_base = static_cast<const T *>(part == 0 ? p.q : p.k);
            const T *g_base = static_cast<const T *>(part == 0 ? p.dq_out : p.dk_out);
            T *o_base = static_cast<T *>(part == 0 ? p.q_out : p.k_out);
            const int64_t xs = part == 0 ? p.q_stride : p.k_stride, gs = part == 0 ? p.dq_stride : p.dk_stride;
            const int64_t os = part == 0 ? p.q_out_stride : p.k_out_stride;
            const T *w = static_cast<const T *>(part == 0 ? p.q_weight : p.k_weight);
            for (int r = group; r < (t1 - (int)t0) * heads; r += GROUPS) {
                const int tl = r / heads, head = r - tl * heads;
                const int64_t t = t0 + tl;
                const T *x = x_base + t * xs + head * d, *g = g_base + t * gs + head * d;
                float xa[NU][V], xb[NU][V], ga[NU][V], gb[NU][V], wa[NU][V], wb[NU][V];
                float ss = 0.0f, dot = 0.0f;
#pragma unroll
                for (int n = 0; n < NU; n++) {
                    const int u = u0 + n * LPR;
                    const RopeUnit ru = rope_unit<V>(p, u);
                    if (u < units) {
                        RopeVec<T, V>::load(x + ru.a0, xa[n]);
                        RopeVec<T, V>::load(x + ru.a1, xb[n]);
                        RopeVec<T, V>::load(g + ru.a0, ga[n]);
                        RopeVec<T, V>::load(g + ru.a1, gb[n]);
                        if (w) {
                            RopeVec<T, V>::load(w + ru.a0, wa[n]);
                            RopeVec<T, V>::load(w + ru.a1, wb[n]);
                        }
                        rope_turn<V>(cs + tl * half, ru, p.interleaved, true, ga[n], gb[n]);
                    } else {
#pragma unroll
                        for (int i = 0; i < V; i++) xa[n][i] = xb[n][i] = ga[n][i] = gb[n][i] = 0.0f;
                    }
#pragma unroll
                    for (int i = 0; i < V; i++) {
                        if (!w || u >= units) wa[n][i] = wb[n][i] = 1.0f;
                        ss += xa[n][i] * xa[n][i] + xb[n][i] * xb[n][i];
                        dot += ga[n][i] * wa[n][i] * xa[n][i] + gb[n][i] * wb[n][i] * xb[n][i];
                    }
                }
                ss = wave_sum_xor(ss, 1, LPR);
                dot = wave_sum_xor(dot, 1, LPR);
                const float rs = p.normalize ? 1.0f / sqrtf(ss * inv_d + p.eps) : 1.0f;
                const float c = p.normalize ? dot * inv_d * rs * rs : 0.0f;
#pragma unroll
                for (int n = 0; n < NU; n++) {
                    const int u = u0 + n * LPR;
                    if (u >= units) continue;
                    const RopeUnit ru = rope_unit<V>(p, u);
                    T *o = o_base + t * os + head * d;
#pragma unroll
                    for (int i = 0; i < V; i++) {
                        gw[part][n][0][i] += ga[n][i] * (xa[n][i] * rs);
                        gw[part][n][1][i] += gb[n][i] * (xb[n][i] * rs);
                        xa[n][i] = rs * (ga[n][i] * wa[n][i] - xa[n][i] * c);
                        xb[n][i] = rs * (gb[n][i] * wb[n][i] - xb[n][i] * c);
                    }
                    RopeVec<T, V>::store(o + ru.a0, xa[n]);
                    RopeVec<T, V>::store(o + ru.a1, xb[n]);
                }
            }
        }
    }
    if (!p.partial) return;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
#pragma unroll
    for (int w = 0; w < 2; w++)
#pragma unroll
        for (int n = 0; n < NU; n++) {
            const int u = u0 + n * LPR;
            const RopeUnit ru = rope_unit<V>(p, u);
#pragma unroll
            for (int s = 0; s < 2; s++)
#pragma unroll
                for (int i = 0; i < V; i++) {
                    const float v = wave_sum_xor(gw[w][n][s][i], LPR, 64);
                    if (lane < LPR && u < units) sums[(wave * 2 + w) * d + (s == 0 ? ru.a0 : ru.a1) + i] = v;
                }
        }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * d; i += kRopeThreads) {
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < WAVES; w++) v += sums[w * 2 * d + i];
        p.partial[(int64_t)blockIdx.x * 2 * d + i] = v;
    }
}

// The workgroups' sums, added in a fixed order: a workgroup takes 4 columns of the
// [groups][2 d] partials, a thread every 256th row of them.  What bounds it: one trip to
// memory (1024 rows of 256 columns: 4.8 us; with 16 columns a workgroup, 64 threads each, 6.9).
__global__ __launch_bounds__(256) void norm_rope_weight_kernel(NormRopeParams p) {
    __shared__ float4 red[4];
    const int col = blockIdx.x * 4, n = 2 * p.head_dim, lane = threadIdx.x & 63;
    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (int g = threadIdx.x; g < p.groups; g += 256) {
        const float4 x = *reinterpret_cast<const float4 *>(p.partial + (int64_t)g * n + col);
        v[0] += x.x, v[1] += x.y, v[2] += x.z, v[3] += x.w;
    }
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] = wave_sum_xor(v[e], 1, 64);
    if (lane == 0) red[threadIdx.x >> 6] = make_float4(v[0], v[1], v[2], v[3]);
    __syncthreads();
    if (threadIdx.x >= 4) return;
    const float *r = reinterpret_cast<const float *>(red) + threadIdx.x;
    const int c = col + threadIdx.x;
    float *out = c < p.head_dim ? p.d_q_weight : p.d_k_weight;
    if (out) out[c < p.head_dim ? c : c - p.head_dim] = (r[0] + r[4]) + (r[8] + r[12]);
}

// ------------------------------------------------------------------ launchers

// Whole 16-byte pieces everywhere: rows, halves of the rotated part, strides, pointers.
static bool rope_wide(const NormRopeParams &p, int32_t dtype, bool backward) {
    const int v = dtype == kF32 ? 4 : 8, half = p.rotary_dim / 2;
    if (p.head_dim % (2 * v) || half % v) return false;
    uintptr_t ptrs = (uintptr_t)p.q | (uintptr_t)p.k | (uintptr_t)p.q_out | (uintptr_t)p.k_out |
                     (uintptr_t)p.q_weight | (uintptr_t)p.k_weight;
    int64_t strides = p.q_stride | p.k_stride | p.q_out_stride | (p.k_out ? p.k_out_stride : 0);
    if (p.k_pool) ptrs |= (uintptr_t)p.k_pool | (uintptr_t)p.v_pool | (uintptr_t)p.v, strides |= p.v_stride;
    if (backward) ptrs |= (uintptr_t)p.dq_out | (uintptr_t)p.dk_out, strides |= p.dq_stride | p.dk_stride;
    return (ptrs & 15) == 0 && strides % v == 0;
}

// lanes of a row (a power of two) and units of a lane
static int rope_lanes(const NormRopeParams &p, int v) {
    const int units = p.head_dim / (2 * v);
    int l = 4;
    while (l < units && l < 64) l *= 2;
    return l;
}

#define PAM_ROPE_SWITCH(CALL, T, W)                                                        \
    if (wide) {                                                                            \
        switch (rope_lanes(p, W)) {                                                        \
            case 4: CALL(T, W, 4, 1); break;                                               \
            case 8: CALL(T, W, 8, 1); break;                                               \
            case 16: CALL(T, W, 16, 1); break;                                             \
            default: CALL(T, W, 32, 1); break;                                             \
        }                                                                                  \
    } else {                                                                               \
        switch (rope_lanes(p, 1)) {                                                        \
            case 4: CALL(T, 1, 4, 1); break;                                               \
            case 8: CALL(T, 1, 8, 1); break;                                               \
            case 16: CALL(T, 1, 16, 1); break;                                             \
            case 32: CALL(T, 1, 32, 1); break;                                             \
            default: CALL(T, 1, 64, 2); break;                                             \
        }                                                                                  \
    }

hipError_t launch_norm_rope(const NormRopeParams &p, int32_t dtype, int32_t cus, hipStream_t stream) {
    if (p.num_tokens <= 0) return hipSuccess;
    const bool wide = rope_wide(p, dtype, false);
    // about four workgroups a CU, then 2 tokens each (16384 f16 tokens: 53.6 us, with one 58.5, with
    // up to 8 59.9); few tokens: the heads in slices (64 f16 tokens: 4.9 us)
    const int64_t want = 4 * (int64_t)(cus > 0 ? cus : 1);
    const int tokens = (int)std::max<int64_t>(1, std::min<int64_t>(2, p.num_tokens / want));
    const int64_t gx = (p.num_tokens + tokens - 1) / tokens;
    const int heads = p.num_heads + p.num_kv_heads * (p.k_pool ? 2 : 1);
    const int rows = kRopeThreads / rope_lanes(p, wide ? (dtype == kF32 ? 4 : 8) : 1);  // rows at once
    const int slices = (int)std::max<int64_t>(1, std::min<int64_t>((heads + rows - 1) / rows, want / gx));
    const dim3 grid((unsigned)gx, (unsigned)slices);
    const size_t lds = (size_t)tokens * (p.rotary_dim / 2) * sizeof(float2);
#define PAM_ROPE_CALL(T, W, L, NU) hipLaunchKernelGGL((norm_rope_kernel<T, W, L, NU>), grid, dim3(kRopeThreads), lds, stream, p, tokens)
    if (dtype == kF32) {
        PAM_ROPE_SWITCH(PAM_ROPE_CALL, float, 4)
    } else {
        PAM_ROPE_SWITCH(PAM_ROPE_CALL, f16, 8)
    }
    return hipGetLastError();
}

int32_t norm_rope_backward_groups(const NormRopeParams &p, int32_t dtype, int32_t cus) {
    (void)dtype;
    const int64_t n = ((int64_t)p.num_tokens + kRopeBackTokens - 1) / kRopeBackTokens;
    // two a CU (8192 f16 tokens, the call: 50 us; one 67, four 56)
    return (int32_t)std::max<int64_t>(1, std::min<int64_t>(n, 2 * (int64_t)(cus > 0 ? cus : 1)));
}

hipError_t launch_norm_rope_backward(const NormRopeParams &p, int32_t dtype, hipStream_t stream) {
    const bool wide = rope_wide(p, dtype, true);
    const dim3 grid((unsigned)p.groups);
    const size_t lds = (size_t)kRopeBackTokens * (p.rotary_dim / 2) * sizeof(float2) +
                       (size_t)(kRopeThreads / 64) * 2 * p.head_dim * sizeof(float);
#define PAM_ROPE_BACK(T, W, L, NU) hipLaunchKernelGGL((norm_rope_backward_kernel<T, W, L, NU>), grid, dim3(kRopeThreads), lds, stream, p)
    if (dtype == kF32) {
        PAM_ROPE_SWITCH(PAM_ROPE_BACK, float, 4)
    } else {
        PAM_ROPE_SWITCH(PAM_ROPE_BACK, f16, 8)
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || !p.partial) return e;
    hipLaunchKernelGGL(norm_rope_weight_kernel, dim3((unsigned)(p.head_dim / 2)), dim3(256), 0, stream, p);
    return hipGetLastError();
}

}  // namespace pam
