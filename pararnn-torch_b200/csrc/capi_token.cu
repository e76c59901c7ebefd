// extern "C" entry points of the token-model operators (linear attention with a decay for each head,
// group norm with an activation, embedding lookup): argument checks, workspace layout and the
// sequence of launches.  The kernels live in linattn_*.cu, groupnorm.cu and embedding.cu.
#include "../../include/pararnn_b200.h"
#include "embedding.cuh"
#include "groupnorm.cuh"
#include "linattn.cuh"

using namespace prb;

namespace {

// the sort adds a piece's or a block's length to counts of tokens and ids in 32 bits
constexpr long long kMaxSorted = 0x7fff0000;

bool bad_type(int dtype) { return dtype != PRB_F32 && dtype != PRB_BF16; }
int done(cudaError_t e) { return e == cudaSuccess ? PRB_OK : PRB_ERR_LAUNCH; }
HeadView view(const prb_heads* h) { return HeadView{h->data, h->stride_b, h->stride_t, h->stride_h}; }

struct AttnShape {
    int dtype, rows, time, n_seq, max_len, hq, hkv, dk, dv;
};

// Segments of the time axis.  One CTA walks a segment of one head (and of one block of 64 value channels on
// the CUDA cores), so few (sequence, head) pairs leave SMs idle; cutting costs a second read of two
// inputs (the state sweep) and two more launches, some 12 us.  So nothing up to 8 chunks of 128 (fp32: 2) is
// cut, and a segment has at least 2 (fp32: 1; there two CTAs share an SM up to 64 channels).  Forward, 8 heads:
// 2048 tokens of 64 channels uncut 39.7 us, in pieces of at least 8 chunks 38.5, of 4 27.8, of 2 22.6; 4096 of
// 128: 100, 65.6, 50.6, 46.7; 32768 of 128: 772 uncut, 117 cut; 5 packed prompts of 739 tokens with their
// states: 22 uncut, 34 cut; fp32 2 x 1021 in 4 pieces 73, in 8 60.
SegMap plan_segments(const AttnShape& s, const int* cu, bool backward) {
    SegMap m{};
    m.cu = cu;
    m.n_seq = s.n_seq;
    m.time = s.time;
    const bool simt = s.dtype == PRB_F32, narrow = s.dk <= 64 && (s.dv <= 64 || !backward);
    const int chunk = 128, sm = sm_count() * (simt && narrow ? 2 : 1), least = simt ? chunk : 2 * chunk;
    const int blocks_v = simt ? (s.dv + 63) / 64 : 1, blocks_k = simt ? (s.dk + 63) / 64 : 1;
    const long long jobs =
        backward ? (long long)s.hq * blocks_k + s.hkv * (blocks_k + blocks_v) : (long long)s.hq * blocks_v;
    const long long tokens = cu ? s.time : (long long)s.rows * s.time;
    long long len = s.max_len;
    if (s.max_len > (simt ? 2 : 8) * chunk && (long long)s.n_seq * jobs < sm) {
        // rectangular: as many equal segments as one wave holds; packed: an even share of all tokens
        const long long cuts = sm / (s.n_seq * jobs);
        len = cu ? (tokens * jobs + sm - 1) / sm : (s.time + cuts - 1) / cuts;
        len = (len + chunk - 1) / chunk * chunk;
        if (len < least) len = least;
    }
    if (len >= s.max_len) {
        m.seg_len = s.max_len;
        m.n_seg = 1;
        m.n_items = s.n_seq;
        return m;
    }
    m.seg_len = (int)len;
    m.n_seg = (int)((s.time + len - 1) / len);
    m.n_items = cu ? s.n_seq + (int)(s.time / len) : s.n_seq * m.n_seg;
    return m;
}
bool segmented(const SegMap& m) { return m.n_items > m.n_seq; }

size_t attn_bytes(const AttnShape& s, bool packed, bool backward) {
    static const int dummy = 0;
    const SegMap m = plan_segments(s, packed ? &dummy : nullptr, backward);
    if (!segmented(m)) return 0;
    return sizeof(float) * (size_t)m.n_items * s.hkv * s.dk * s.dv * (backward ? 2 : 1);
}

int check_attn(const AttnShape& s) {
    if (s.rows < 1 || s.time < 1 || s.n_seq < 1 || s.hq < 1 || s.hkv < 1 || s.dk < 1 || s.dv < 1 || s.max_len < 1 ||
        s.max_len > s.time || bad_type(s.dtype))
        return PRB_ERR_BAD_ARG;
    if (s.hq % s.hkv || s.dk > kMaxHeadDim || s.dv > kMaxHeadDim) return PRB_ERR_UNSUPPORTED;
    if (s.hq > 8192 || s.hkv > 8192) return PRB_ERR_UNSUPPORTED;  // grid.y = heads x channel blocks x jobs
    if (s.time > (1 << 30)) return PRB_ERR_UNSUPPORTED;  // a length and a segment are added in 32 bits
    return PRB_OK;
}

// bf16 goes to the tensor cores wherever TMA can address its tensors; fp32 and the rest to the CUDA cores
cudaError_t launch_mix(const MixParams& p, const AttnShape& a, bool state_only, cudaStream_t s) {
    if (options().kernel_family != 0 && mix_tc_usable(p, a.dtype)) return launch_mix_tc(p, a.rows, state_only, s);
    return launch_mix_simt(p, a.dtype, state_only, s);
}

// the state sweep of (b, c) and its fold; leaves the states entering the segments in `dst`
cudaError_t segment_states(MixParams p, const HeadView& b, const HeadView& c, int share, int reverse, float upd,
                           const AttnShape& a, float* dst, const float* s_in, float* s_out, cudaStream_t s) {
    MixJob& j = p.job[0];
    j = MixJob{};
    j.a = j.b = b;
    j.c = c;
    j.s_out = dst;
    j.da = a.dk;
    j.dc = a.dv;
    j.s_row = a.dv;
    j.s_col = 1;
    j.heads = a.hkv;
    j.share_a = 1;
    j.share_b = share;
    j.reverse = reverse;
    j.upd_scale = upd;
    j.exact = s_out != nullptr;
    p.n_jobs = 1;
    cudaError_t e = launch_mix(p, a, true, s);
    if (e != cudaSuccess) return e;
    return launch_fold_states(p, dst, s_in, s_out, reverse != 0, s);
}

MixParams attn_params(const AttnShape& a, const SegMap& m, const float* log_decay) {
    MixParams p{};
    p.log_decay = log_decay;
    p.state_heads = a.hkv;
    p.state_elems = a.dk * a.dv;
    p.map = m;
    return p;
}

}  // namespace

extern "C" {

size_t prb_linear_attention_workspace_bytes(int rows, int time, int n_seq, int max_len, int q_heads, int kv_heads,
                                            int dk, int dv, int dtype, int packed, int backward) {
    const AttnShape a{dtype, rows, time, n_seq, max_len, q_heads, kv_heads, dk, dv};
    if (check_attn(a) != PRB_OK) return 0;
    return attn_bytes(a, packed != 0, backward != 0);
}

int prb_linear_attention(const prb_heads* q, const prb_heads* k, const prb_heads* v, const float* log_decay,
                         const float* state_in, const int* cu_seqlens, void* out, float* state_out, int rows,
                         int time, int n_seq, int max_len, int q_heads, int kv_heads, int dk, int dv, int dtype,
                         float scale, void* workspace, size_t workspace_bytes, prb_stream_t stream) {
    const AttnShape a{dtype, rows, time, n_seq, max_len, q_heads, kv_heads, dk, dv};
    if (!q || !k || !v || !q->data || !k->data || !v->data || !log_decay || !out) return PRB_ERR_BAD_ARG;
    if (const int rc = check_attn(a)) return rc;
    if (cu_seqlens ? rows != 1 : rows != n_seq) return PRB_ERR_BAD_ARG;
    // one of the query heads of a state writes it while the others may not have read it yet
    if (state_out && state_out == state_in && q_heads != kv_heads) return PRB_ERR_BAD_ARG;
    const SegMap m = plan_segments(a, cu_seqlens, false);
    const bool seg = segmented(m);
    if (seg && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255) ||
                workspace_bytes < attn_bytes(a, cu_seqlens != nullptr, false)))
        return PRB_ERR_WORKSPACE;
    cudaStream_t s = (cudaStream_t)stream;
    MixParams p = attn_params(a, m, log_decay);
    float* ws = reinterpret_cast<float*>(workspace);
    if (seg) {
        const cudaError_t e = segment_states(p, view(k), view(v), 1, 0, 1.f, a, ws, state_in, state_out, s);
        if (e != cudaSuccess) return PRB_ERR_LAUNCH;
    }
    MixJob& j = p.job[0];
    j.a = view(q);
    j.b = view(k);
    j.c = view(v);
    j.out = out;
    j.s_in = seg ? ws : state_in;
    j.s_out = seg ? nullptr : state_out;
    j.da = dk;
    j.dc = dv;
    j.s_row = dv;
    j.s_col = 1;
    j.heads = q_heads;
    j.share_a = q_heads / kv_heads;
    j.share_b = 1;
    j.p_scale = j.row_scale = scale;
    j.upd_scale = 1.f;
    j.exact = j.s_out != nullptr;
    p.n_jobs = 1;
    return done(launch_mix(p, a, false, s));
}

int prb_bwd_linear_attention(const prb_heads* q, const prb_heads* k, const prb_heads* v, const prb_heads* grad_out,
                             const float* log_decay, const float* state_in, const float* grad_state_out,
                             const int* cu_seqlens, void* g_q, void* g_k, void* g_v, float* g_state, int rows,
                             int time, int n_seq, int max_len, int q_heads, int kv_heads, int dk, int dv, int dtype,
                             float scale, void* workspace, size_t workspace_bytes, prb_stream_t stream) {
    const AttnShape a{dtype, rows, time, n_seq, max_len, q_heads, kv_heads, dk, dv};
    if (!q || !k || !v || !grad_out || !q->data || !k->data || !v->data || !grad_out->data || !log_decay || !g_q ||
        !g_k || !g_v)
        return PRB_ERR_BAD_ARG;
    if (const int rc = check_attn(a)) return rc;
    if (cu_seqlens ? rows != 1 : rows != n_seq) return PRB_ERR_BAD_ARG;
    // the jobs of dq and dk read these while the job of dv writes
    if (g_state && (g_state == state_in || g_state == grad_state_out)) return PRB_ERR_BAD_ARG;
    const SegMap m = plan_segments(a, cu_seqlens, true);
    const bool seg = segmented(m);
    if (seg && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255) ||
                workspace_bytes < attn_bytes(a, cu_seqlens != nullptr, true)))
        return PRB_ERR_WORKSPACE;
    cudaStream_t s = (cudaStream_t)stream;
    MixParams p = attn_params(a, m, log_decay);
    const int share = q_heads / kv_heads;
    float* fwd_states = reinterpret_cast<float*>(workspace);
    float* bwd_states = fwd_states + (size_t)m.n_items * kv_heads * dk * dv;
    if (seg) {
        cudaError_t e = segment_states(p, view(k), view(v), 1, 0, 1.f, a, fwd_states, state_in, nullptr, s);
        if (e == cudaSuccess)
            e = segment_states(p, view(q), view(grad_out), share, 1, scale, a, bwd_states, grad_state_out, g_state, s);
        if (e != cudaSuccess) return PRB_ERR_LAUNCH;
    }
    MixJob& jq = p.job[0];  // dq: forwards, state transposed
    jq.a = view(grad_out);
    jq.b = view(v);
    jq.c = view(k);
    jq.out = g_q;
    jq.s_in = seg ? fwd_states : state_in;
    jq.da = dv;
    jq.dc = dk;
    jq.s_row = 1;
    jq.s_col = dv;
    jq.heads = q_heads;
    jq.share_a = share;
    jq.share_b = 1;
    jq.p_scale = jq.row_scale = scale;
    jq.upd_scale = 1.f;
    MixJob& jk = p.job[1];  // dk: backwards, state transposed
    jk.a = view(v);
    jk.b = view(grad_out);
    jk.c = view(q);
    jk.out = g_k;
    jk.s_in = seg ? bwd_states : grad_state_out;
    jk.da = dv;
    jk.dc = dk;
    jk.s_row = 1;
    jk.s_col = dv;
    jk.heads = kv_heads;
    jk.share_a = 1;
    jk.share_b = share;
    jk.reverse = 1;
    jk.p_scale = scale;
    jk.row_scale = 1.f;
    jk.upd_scale = scale;
    MixJob& jv = p.job[2];  // dv: backwards
    jv = jk;
    jv.a = view(k);
    jv.b = view(q);
    jv.c = view(grad_out);
    jv.out = g_v;
    jv.s_out = seg ? nullptr : g_state;
    jv.exact = jv.s_out != nullptr;
    jv.da = dk;
    jv.dc = dv;
    jv.s_row = dv;
    jv.s_col = 1;
    p.n_jobs = 3;
    return done(launch_mix(p, a, false, s));
}

int prb_linear_attention_status(int clear) { return linattn_status(clear); }
int prb_linear_attention_poll(int clear) { return linattn_poll(clear); }

int prb_linear_attention_step(const void* q, const void* k, const void* v, const float* log_decay, float* state,
                              const void* block_table, int table_is_int64, void* out, int rows, int slots, int q_heads,
                              int kv_heads, int dk, int dv, int dtype, float scale, prb_stream_t stream) {
    if (!q || !k || !v || !log_decay || !state || !out || rows < 1 || slots < 1 || q_heads < 1 || kv_heads < 1 ||
        dk < 1 || dv < 1 || bad_type(dtype))
        return PRB_ERR_BAD_ARG;
    if (!block_table && rows != slots) return PRB_ERR_BAD_ARG;
    if (q_heads % kv_heads || dk > kMaxHeadDim || dv > kMaxHeadDim || kv_heads > 65535) return PRB_ERR_UNSUPPORTED;
    // every CTA looks for other rows of its slot: the time of a table grows with the square of its rows
    if (rows > (block_table ? 1 << 20 : 1 << 30)) return PRB_ERR_UNSUPPORTED;
    StepArgs a{q, k, v, log_decay, state, block_table, out, rows, slots, q_heads, kv_heads, dk, dv, table_is_int64,
               scale};
    return done(launch_linattn_step(a, dtype, (cudaStream_t)stream));
}

size_t prb_group_norm_workspace_bytes(long long samples, int positions, int channels, int groups, int dtype,
                                      int backward) {
    if (samples < 1 || positions < 1 || channels < 1 || groups < 1 || channels % groups || bad_type(dtype)) return 0;
    const GroupNormPlan pl = groupnorm_plan(dtype, samples, positions, channels, groups, backward != 0);
    return (pl.group_floats + (backward ? 2 * (size_t)pl.part_rows * channels : 0)) * sizeof(float);
}

static int group_norm(GroupNormArgs& a, int dtype, int weight_dtype, bool backward, void* ws, size_t ws_bytes,
                      prb_stream_t stream) {
    if (a.samples < 1 || a.positions < 1 || a.channels < 1 || a.groups < 1 || a.channels % a.groups ||
        bad_type(dtype) || bad_type(weight_dtype) || a.act < kActNone || a.act > kActGelu)
        return PRB_ERR_BAD_ARG;
    // 16-byte vectors: a group is a whole number of them or they are not used, so the base decides
    const uintptr_t bits = reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.dy) |
                           reinterpret_cast<uintptr_t>(a.y) | reinterpret_cast<uintptr_t>(a.dx);
    if (bits & 15) return PRB_ERR_BAD_ARG;
    if ((long long)a.channels > 256ll * 65535 || a.channels > (1 << 30)) return PRB_ERR_UNSUPPORTED;
    // the kernels step over up to kT x 8 positions at once and count them in 32 bits
    if (a.positions > 0x7fffffff - 4096) return PRB_ERR_UNSUPPORTED;
    const size_t need = prb_group_norm_workspace_bytes(a.samples, a.positions, a.channels, a.groups, dtype, backward);
    if (need && (!ws || (reinterpret_cast<uintptr_t>(ws) & 255) || ws_bytes < need)) return PRB_ERR_WORKSPACE;
    const GroupNormPlan pl = groupnorm_plan(dtype, a.samples, a.positions, a.channels, a.groups, backward);
    a.group_part = reinterpret_cast<float*>(ws);
    a.partial = a.group_part + pl.group_floats;
    a.w_f32 = weight_dtype == PRB_F32;
    return done(launch_groupnorm(a, dtype, backward, (cudaStream_t)stream));
}

int prb_group_norm(const void* x, const void* weight, const void* bias, void* y, float* stats, long long samples,
                   int positions, int channels, int groups, float eps, int activation, int dtype, int weight_dtype,
                   void* workspace, size_t workspace_bytes, prb_stream_t stream) {
    if (!x || !y) return PRB_ERR_BAD_ARG;
    GroupNormArgs a{};
    a.x = x;
    a.w = weight;
    a.b = bias;
    a.y = y;
    a.stats = reinterpret_cast<float2*>(stats);
    a.samples = samples;
    a.positions = positions;
    a.channels = channels;
    a.groups = groups;
    a.act = activation;
    a.eps = eps;
    return group_norm(a, dtype, weight_dtype, false, workspace, workspace_bytes, stream);
}

int prb_bwd_group_norm(const void* x, const void* grad_y, const void* weight, const void* bias, const float* stats,
                       void* g_x, void* g_weight, void* g_bias, long long samples, int positions, int channels,
                       int groups, int activation, int dtype, int weight_dtype, void* workspace,
                       size_t workspace_bytes, prb_stream_t stream) {
    if (!x || !grad_y || !stats || !g_x) return PRB_ERR_BAD_ARG;
    GroupNormArgs a{};
    a.x = x;
    a.dy = grad_y;
    a.w = weight;
    a.b = bias;
    a.dx = g_x;
    a.dw = g_weight;
    a.db = g_bias;
    a.stats = reinterpret_cast<float2*>(const_cast<float*>(stats));
    a.samples = samples;
    a.positions = positions;
    a.channels = channels;
    a.groups = groups;
    a.act = activation;
    return group_norm(a, dtype, weight_dtype, true, workspace, workspace_bytes, stream);
}

int prb_embedding(const void* ids, int ids_is_int64, const void* table, void* out, long long tokens, int vocab,
                  int channels, int dtype, float scale, prb_stream_t stream) {
    if (!ids || !table || !out || tokens < 1 || vocab < 1 || channels < 1 || bad_type(dtype)) return PRB_ERR_BAD_ARG;
    if (tokens > 0x7fffffffLL) return PRB_ERR_UNSUPPORTED;
    EmbedArgs a{ids, table, nullptr, out, tokens, vocab, channels, ids_is_int64, scale};
    return done(launch_embedding(a, dtype, (cudaStream_t)stream));
}

size_t prb_bwd_embedding_workspace_bytes(long long tokens, int vocab, int channels) {
    if (tokens < 1 || tokens > kMaxSorted || vocab < 1 || vocab > kMaxSorted || channels < 1) return 0;
    return embedding_plan(tokens, vocab, channels).total;
}

int prb_bwd_embedding(const void* ids, int ids_is_int64, const void* grad_out, void* g_table, long long tokens,
                      int vocab, int channels, int dtype, float scale, void* workspace, size_t workspace_bytes,
                      prb_stream_t stream) {
    if (!ids || !grad_out || !g_table || tokens < 1 || vocab < 1 || channels < 1 || bad_type(dtype))
        return PRB_ERR_BAD_ARG;
    if (tokens > kMaxSorted || vocab > kMaxSorted) return PRB_ERR_UNSUPPORTED;
    if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255) ||
        workspace_bytes < embedding_plan(tokens, vocab, channels).total)
        return PRB_ERR_WORKSPACE;
    EmbedArgs a{ids, nullptr, grad_out, g_table, tokens, vocab, channels, ids_is_int64, scale};
    return done(launch_embedding_grad(a, dtype, workspace, (cudaStream_t)stream));
}

}  // extern "C"
