// speculative.cpp - the engine's speculative-decoding calls: batch plans, norm and
// rotation of query and key heads with their gradients, tree attention and the commit of
// an accepted path.  No counterpart in the reference.
#include <algorithm>
#include <cmath>
#include <limits>

#include "engine_util.h"

namespace pam {

namespace {

// The calls run on the context's device; the caller's current device comes back after.
struct DeviceGuard {
    int before = -1;
    explicit DeviceGuard(int device) {
        int now = -1;
        if (hipGetDevice(&now) == hipSuccess && now != device) {
            hip_check(hipSetDevice(device), "hipSetDevice");
            before = now;
        }
    }
    ~DeviceGuard() {
        if (before >= 0) (void)hipSetDevice(before);
    }
};

void need(bool ok, const char *what) {
    if (!ok) throw invalid_configuration(what);
}

// products of request fields, which may be any
int64_t times(int64_t a, int64_t b) {
    int64_t r;
    if (__builtin_mul_overflow(a, b, &r)) throw invalid_configuration("sizes overflow 64 bits.");
    return r;
}

int32_t blocks_of(size_t k_bytes, size_t v_bytes, const pam_layer_spec &l) {
    need(k_bytes != 0 && v_bytes != 0, "the pools' sizes are needed.");
    const int64_t block = times(l.block_size, kv_bytes_per_token(l)), n = (int64_t)(std::min(k_bytes, v_bytes) / (size_t)block);
    if (n < 1) throw buffer_too_small("K pool", block, (int64_t)std::min(k_bytes, v_bytes));
    return (int32_t)std::min<int64_t>(n, std::numeric_limits<int32_t>::max());
}

// bytes of rows `stride` elements apart, `row` elements used of each
int64_t span(int64_t rows, int64_t stride, int64_t row, int32_t elem) {
    // row <= stride: the sum fits when `rows` whole strides do
    (void)times(times(rows, stride), elem);
    return ((rows - 1) * stride + row) * elem;
}

int64_t stride_of(int64_t stride, int64_t row, const char *name) {
    if (stride == 0) return row;
    if (stride < row) throw invalid_configuration(std::string(name) + " rows overlap.");
    return stride;
}

// inv_freq / 2 pi turns per position as a 64-bit binary fraction
void set_rotation(const pam_rotary_spec &r, const pam_layer_spec &l, NormRopeParams &p) {
    need(r.rotary_dim >= 0 && r.rotary_dim <= l.head_dim && r.rotary_dim % 2 == 0,
         "rotaryDim must be even and at most headDim.");
    need(r.rotary_dim == 0 || r.inv_freq || (r.base > 0.0 && std::isfinite(r.base)), "the rotation's base must be positive.");
    p.rotary_dim = r.rotary_dim;
    p.interleaved = r.interleaved ? 1 : 0;
    const long double turn = 0.15915494309189533576888376337251L;  // 1 / 2 pi
    for (int32_t i = 0; i < r.rotary_dim / 2; i++) {
        const double f = r.inv_freq ? r.inv_freq[i] : std::pow(r.base, -2.0 * i / r.rotary_dim);
        need(std::isfinite(f), "the rotation's frequencies must be finite.");
        long double t = (long double)f * turn;
        if (t < 0.0L || t >= 1.0L) t -= std::floor(t);
        const long double scaled = t * 18446744073709551616.0L + 0.5L;
        p.freq[i] = scaled >= 18446744073709551616.0L ? 0 : (uint64_t)scaled;
    }
}

void check_norm(const pam_layer_spec &l, const pam_rotary_spec &rotary, int32_t num_tokens, float eps, bool normalize,
                const void *qw, const void *kw, const int32_t *positions, size_t positions_bytes) {
    validate_layer(l);
    need(num_tokens > 0, "numTokens must be positive.");
    need(normalize || rotary.rotary_dim > 0, "neither norm nor rotation is asked for.");
    need(normalize || (!qw && !kw), "weights go with the norm.");
    need(!normalize || (eps >= 0.0f && std::isfinite(eps)), "eps must not be negative.");
    need(rotary.rotary_dim == 0 || positions, "the rotation needs positions.");
    require(positions_bytes, "positions", (int64_t)num_tokens * 4);
}

}  // namespace

// Before a call's work: the device is set up and current, a strict code object refuses.
// Returns whether the stream is being captured.
bool Context::begin_spec() {
    if (ktab() && ktab()->strict)
        throw PamError("Unsupported paged attention path: the speculative-decoding kernels are not in the code object.");
    hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing(stream(), &st) != hipSuccess) {
        (void)hipGetLastError();
        st = hipStreamCaptureStatusNone;
    }
    const bool capturing = st == hipStreamCaptureStatusActive;
    if (capturing && synchronous)
        throw invalid_configuration("a captured call needs an asynchronous context (pam_set_synchronous).");
    return capturing;
}

// The split workspace at `bytes` at least.  A captured call may not allocate, and the
// workspace whose address it records stays until the context is destroyed.
void Context::spec_workspace(size_t bytes, bool capturing) {
    if (bytes == 0) return;
    if (capturing && bytes > workspace_.bytes)
        throw invalid_configuration("a captured call needs " + std::to_string(bytes) +
                                    " bytes of workspace: make the call once before, or pam_reserve_workspace.");
    reserve_workspace(bytes);
    if (capturing) workspace_captured_ = true;
}

// ------------------------------------------------------------------ batch plan

void Context::batch_plan(const pam_batch_plan_request &r) {
    need(r.num_seqs > 0, "numSeqs must be positive.");
    need(r.block_size > 0, "blockSize must be positive.");
    need(r.max_num_blocks > 0, "maxNumBlocks must be positive.");
    need(r.max_rows > 0, "maxRows must be positive.");
    need((int64_t)r.max_num_blocks * r.block_size <= std::numeric_limits<int32_t>::max(),
         "a sequence has at most 2^31 - 1 tokens.");
    need(r.block_list_len >= 0 && r.parents_len >= 0, "lengths must not be negative.");
    need(!r.tree_mask || (r.mask_words >= 1 && r.mask_words <= kPlanMaxNodes / 64), "maskWords must be 1 to 16.");
    need(r.context_lens && r.query_lens && (r.block_list || r.block_list_len == 0) && r.cu_queries && r.seq_lengths &&
             r.block_tables && r.positions && r.slot_mapping,
         "batch plan request has a null buffer.");
    ensure_device();
    const DeviceGuard guard(device_);
    const bool capturing = begin_spec();
    BatchPlanParams p{};
    p.context_lens = r.context_lens;
    p.query_lens = r.query_lens;
    p.block_list = r.block_list;
    p.parents = r.parents;
    p.block_list_len = r.block_list_len;
    p.parents_len = r.parents ? r.parents_len : 0;
    p.num_seqs = r.num_seqs;
    p.block_size = r.block_size;
    p.max_num_blocks = r.max_num_blocks;
    p.max_rows = r.max_rows;
    p.mask_words = r.tree_mask ? r.mask_words : 0;
    p.cu_queries = r.cu_queries;
    p.seq_lengths = r.seq_lengths;
    p.block_tables = r.block_tables;
    p.positions = r.positions;
    p.slot_mapping = r.slot_mapping;
    p.tree_mask = r.tree_mask;
    p.status = r.status;
    run_spec("batchPlan", PAM_OP_BATCH_PLAN, r.num_seqs, r.max_rows, 0, capturing,
             [&] { return launch_batch_plan(p, stream()); });
}

// ------------------------------------------------------------------ norm and rotation

void Context::qk_norm_rope(const pam_qk_norm_rope_request &r) {
    const pam_layer_spec &l = r.layer;
    check_norm(l, r.rotary, r.num_tokens, r.eps, r.normalize, r.q_weight, r.k_weight, r.positions, r.positions_bytes);
    const bool pool = r.k_pool || r.v_pool || r.slot_mapping || r.values;
    need(r.q && r.k && r.q_out && (r.k_out || pool), "norm request has a null buffer.");
    need(!pool || (r.k_pool && r.v_pool && r.slot_mapping && r.values),
         "the pools, the slot mapping and the values go together.");
    if (pool && l.data_type == kFP8)
        throw PamError("Unsupported paged attention path: FP8 pools are appended to with a block table, not a slot mapping.");
    const int64_t qrow = (int64_t)l.num_heads * l.head_dim, krow = (int64_t)l.num_kv_heads * l.head_dim;
    const int32_t e = io_bytes(l.data_type);
    NormRopeParams p{};
    p.q_stride = stride_of(r.q_stride, qrow, "Q");
    p.k_stride = stride_of(r.k_stride, krow, "K");
    p.q_out_stride = stride_of(r.q_out_stride, qrow, "Q output");
    p.k_out_stride = stride_of(r.k_out_stride, krow, "K output");
    p.v_stride = stride_of(r.v_stride, krow, "V");
    need(r.q_out != r.q || p.q_out_stride == p.q_stride, "a Q output in place has Q's stride.");
    need(r.k_out != r.k || p.k_out_stride == p.k_stride, "a K output in place has K's stride.");
    require(r.q_bytes, "Q", span(r.num_tokens, p.q_stride, qrow, e));
    require(r.k_bytes, "K", span(r.num_tokens, p.k_stride, krow, e));
    require(r.q_out_bytes, "Q output", span(r.num_tokens, p.q_out_stride, qrow, e));
    if (r.k_out) require(r.k_out_bytes, "K output", span(r.num_tokens, p.k_out_stride, krow, e));
    if (pool) {
        require(r.values_bytes, "values", span(r.num_tokens, p.v_stride, krow, e));
        require(r.slot_mapping_bytes, "slotMapping", (int64_t)r.num_tokens * 8);
        if (r.k_pool_bytes && r.v_pool_bytes)
            p.pool_slots = (int64_t)blocks_of(r.k_pool_bytes, r.v_pool_bytes, l) * l.block_size;
    }
    set_rotation(r.rotary, l, p);
    ensure_device();
    const DeviceGuard guard(device_);
    const bool capturing = begin_spec();
    p.q = r.q;
    p.k = r.k;
    p.v = r.values;
    p.q_out = r.q_out;
    p.k_out = r.k_out;
    p.q_weight = r.q_weight;
    p.k_weight = r.k_weight;
    p.positions = r.positions;
    p.slot_mapping = r.slot_mapping;
    p.k_pool = r.k_pool;
    p.v_pool = r.v_pool;
    p.num_tokens = r.num_tokens;
    p.num_heads = l.num_heads;
    p.num_kv_heads = l.num_kv_heads;
    p.head_dim = l.head_dim;
    p.normalize = r.normalize ? 1 : 0;
    p.eps = r.eps;
    run_spec("qkNormRope", PAM_OP_QK_NORM_ROPE, 1, r.num_tokens, 0, capturing,
             [&] { return launch_norm_rope(p, l.data_type, cus_, stream()); });
}

void Context::qk_norm_rope_backward(const pam_qk_norm_rope_backward_request &r) {
    const pam_layer_spec &l = r.layer;
    check_norm(l, r.rotary, r.num_tokens, r.eps, r.normalize, r.q_weight, r.k_weight, r.positions, r.positions_bytes);
    need(r.q && r.k && r.d_q_out && r.d_k_out && r.d_q && r.d_k, "norm gradient request has a null buffer.");
    need(r.normalize || (!r.d_q_weight && !r.d_k_weight), "weights go with the norm.");
    const int64_t qrow = (int64_t)l.num_heads * l.head_dim, krow = (int64_t)l.num_kv_heads * l.head_dim;
    const int32_t e = io_bytes(l.data_type);
    NormRopeParams p{};
    p.q_stride = stride_of(r.q_stride, qrow, "Q");
    p.k_stride = stride_of(r.k_stride, krow, "K");
    p.dq_stride = stride_of(r.d_q_out_stride, qrow, "Q output gradient");
    p.dk_stride = stride_of(r.d_k_out_stride, krow, "K output gradient");
    p.q_out_stride = stride_of(r.d_q_stride, qrow, "Q gradient");
    p.k_out_stride = stride_of(r.d_k_stride, krow, "K gradient");
    need(r.d_q != r.q && r.d_k != r.k && r.d_q != r.d_q_out && r.d_k != r.d_k_out,
         "the gradients need buffers of their own.");
    require(r.q_bytes, "Q", span(r.num_tokens, p.q_stride, qrow, e));
    require(r.k_bytes, "K", span(r.num_tokens, p.k_stride, krow, e));
    require(r.d_q_out_bytes, "Q output gradient", span(r.num_tokens, p.dq_stride, qrow, e));
    require(r.d_k_out_bytes, "K output gradient", span(r.num_tokens, p.dk_stride, krow, e));
    require(r.d_q_bytes, "Q gradient", span(r.num_tokens, p.q_out_stride, qrow, e));
    require(r.d_k_bytes, "K gradient", span(r.num_tokens, p.k_out_stride, krow, e));
    set_rotation(r.rotary, l, p);
    ensure_device();
    const DeviceGuard guard(device_);
    const bool capturing = begin_spec();
    p.q = r.q;
    p.k = r.k;
    p.dq_out = r.d_q_out;
    p.dk_out = r.d_k_out;
    p.q_out = r.d_q;
    p.k_out = r.d_k;
    p.q_weight = r.q_weight;
    p.k_weight = r.k_weight;
    p.d_q_weight = r.d_q_weight;
    p.d_k_weight = r.d_k_weight;
    p.positions = r.positions;
    p.num_tokens = r.num_tokens;
    p.num_heads = l.num_heads;
    p.num_kv_heads = l.num_kv_heads;
    p.head_dim = l.head_dim;
    p.normalize = r.normalize ? 1 : 0;
    p.eps = r.eps;
    p.groups = norm_rope_backward_groups(p, l.data_type, cus_);
    int64_t tmp = 0;
    if (r.d_q_weight || r.d_k_weight) {
        tmp = (int64_t)p.groups * 2 * l.head_dim * 4;
        spec_workspace((size_t)tmp, capturing);
        p.partial = static_cast<float *>(workspace_.ptr);
    }
    run_spec("qkNormRopeBackward", PAM_OP_QK_NORM_ROPE_BACKWARD, 1, r.num_tokens, tmp, capturing,
             [&] { return launch_norm_rope_backward(p, l.data_type, stream()); });
}

// ------------------------------------------------------------------ tree attention

void Context::tree_attention(const pam_tree_attention_request &r) {
    const pam_layer_spec &l = r.layer;
    validate_layer(l);
    need(r.num_seqs > 0, "numSeqs must be positive.");
    need(r.max_num_blocks > 0, "maxNumBlocks must be positive.");
    need(r.max_queries > 0, "maxQueries must be positive.");
    need(r.total_rows > 0, "totalRows must be positive.");
    need(r.num_seqs <= kMaxGridYZ && r.max_queries <= kMaxGridYZ, "at most 65535 sequences and queries of a sequence.");
    need(l.num_kv_heads <= kMaxGridYZ, "at most 65535 key heads.");
    need((int64_t)r.max_num_blocks * l.block_size + r.max_queries <= std::numeric_limits<int32_t>::max() - 4096,
         "a sequence has at most 2^31 - 4096 tokens.");
    need(!r.tree_mask || (r.mask_words > 0 && r.max_queries <= 64 * (int64_t)r.mask_words),
         "maxQueries exceeds the tree mask's bits.");
    need(r.q && r.output && r.k_pool && r.v_pool && r.block_tables && r.context_lens && r.cu_queries,
         "tree attention request has a null buffer.");
    if (l.data_type == kFP8 && (!r.k_scale || !r.v_scale))
        throw invalid_configuration("FP8 tree attention needs the K and V scale pools.");
    // whole 4-element slices of every row
    const uintptr_t kv = (uintptr_t)r.k_pool | (uintptr_t)r.v_pool, io = (uintptr_t)r.q | (uintptr_t)r.output;
    need(kv % (4 * elem_bytes(l.data_type)) == 0 && io % (4 * io_bytes(l.data_type)) == 0,
         "buffers must be aligned to 4 elements.");
    require(r.q_bytes, "Q", times(r.total_rows, q_bytes_per_token(l)));
    require(r.output_bytes, "output", times(r.total_rows, q_bytes_per_token(l)));
    require(r.block_tables_bytes, "blockTables", times((int64_t)r.num_seqs * r.max_num_blocks, 4));
    require(r.context_lens_bytes, "contextLens", (int64_t)r.num_seqs * 4);
    require(r.cu_queries_bytes, "cuQueries", ((int64_t)r.num_seqs + 1) * 4);
    if (r.tree_mask) require(r.tree_mask_bytes, "treeMask", times((int64_t)r.total_rows * r.mask_words, 8));
    TreeParams p{};
    p.pool_blocks = blocks_of(r.k_pool_bytes, r.v_pool_bytes, l);
    need(r.output != r.q, "the output needs a buffer of its own.");
    ensure_device();
    const DeviceGuard guard(device_);
    const bool capturing = begin_spec();
    AttnParams &a = p.a;
    a.q = r.q;
    a.out = r.output;
    a.k_pool = r.k_pool;
    a.v_pool = r.v_pool;
    a.k_scale = r.k_scale;
    a.v_scale = r.v_scale;
    a.block_tables = r.block_tables;
    a.rows = r.total_rows;
    a.bt_stride = r.max_num_blocks;
    a.max_num_blocks = r.max_num_blocks;
    a.num_heads = l.num_heads;
    a.num_kv_heads = l.num_kv_heads;
    a.head_dim = l.head_dim;
    a.block_size = l.block_size;
    a.window = l.window_size;
    a.mode = kRowRagged;
    a.scale_log2 = kLog2eHost / std::sqrt((float)l.head_dim);
    a.zero_page = zero_page_;
    p.context_lens = r.context_lens;
    p.cu_queries = r.cu_queries;
    p.tree_mask = r.tree_mask;
    p.mask_words = r.tree_mask ? r.mask_words : 0;
    p.num_seqs = r.num_seqs;
    p.max_queries = r.max_queries;
    p.total_rows = r.total_rows;
    const int64_t tmp = tree_plan(p, l.data_type, cus_);
    spec_workspace((size_t)tmp, capturing);
    a.part_o = static_cast<float *>(workspace_.ptr);
    run_spec("treeAttention", PAM_OP_TREE_ATTENTION, r.num_seqs, r.total_rows, tmp, capturing,
             [&] { return launch_tree_attention(p, l.data_type, stream()); });
}

// ------------------------------------------------------------------ commit

void Context::tree_commit(const pam_tree_commit_request &r) {
    const pam_layer_spec &l = r.layer;
    validate_layer(l);
    need(r.num_seqs > 0, "numSeqs must be positive.");
    need(r.max_num_blocks > 0, "maxNumBlocks must be positive.");
    need(r.max_path > 0, "maxPath must be positive.");
    need((int64_t)r.max_num_blocks * l.block_size <= std::numeric_limits<int32_t>::max(),
         "a sequence has at most 2^31 - 1 tokens.");
    need(r.k_pool && r.v_pool && r.block_tables && r.context_lens && r.query_lens && r.paths,
         "tree commit request has a null buffer.");
    need(r.new_lengths != r.context_lens && r.new_lengths != r.query_lens, "newLengths needs a buffer of its own.");
    if (l.data_type == kFP8 && (!r.k_scale || !r.v_scale))
        throw invalid_configuration("FP8 tree commit needs the K and V scale pools.");
    need(((uintptr_t)r.k_pool | (uintptr_t)r.v_pool) % (l.data_type == kF16 ? 2 : 4) == 0, "pools must be aligned.");
    require(r.block_tables_bytes, "blockTables", times((int64_t)r.num_seqs * r.max_num_blocks, 4));
    require(r.context_lens_bytes, "contextLens", (int64_t)r.num_seqs * 4);
    require(r.query_lens_bytes, "queryLens", (int64_t)r.num_seqs * 4);
    require(r.paths_bytes, "paths", times((int64_t)r.num_seqs * r.max_path, 4));
    TreeCommitParams p{};
    p.pool_blocks = blocks_of(r.k_pool_bytes, r.v_pool_bytes, l);
    ensure_device();
    const DeviceGuard guard(device_);
    const bool capturing = begin_spec();
    p.k_pool = r.k_pool;
    p.v_pool = r.v_pool;
    p.k_scale = r.k_scale;
    p.v_scale = r.v_scale;
    p.block_tables = r.block_tables;
    p.context_lens = r.context_lens;
    p.query_lens = r.query_lens;
    p.paths = r.paths;
    p.new_lengths = r.new_lengths;
    p.num_seqs = r.num_seqs;
    p.max_num_blocks = r.max_num_blocks;
    p.max_path = r.max_path;
    p.num_kv_heads = l.num_kv_heads;
    p.head_dim = l.head_dim;
    p.block_size = l.block_size;
    run_spec("treeCommit", PAM_OP_TREE_COMMIT, r.num_seqs, r.max_path, 0, capturing,
             [&] { return launch_tree_commit(p, l.data_type, stream()); });
}

}  // namespace pam
