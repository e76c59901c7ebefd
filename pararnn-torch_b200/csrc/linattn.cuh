// Linear attention with a decay for each head: what the kernels of this family share.
//
//   S_t = w S_{t-1} + k_t v_t^T,   o_t = s q_t S_t,   w = exp(log_decay) of the head
//
// The forward pass and all three gradients are ONE operator, a causal (or anti-causal) mix
//
//   out_i = ps sum_{j before i, j = i} w^|i-j| (a_i . b_j) c_j  +  rs w^pos(i) a_i S_in
//   S_out = w^n S_in + us sum_j w^pos'(j) b_j c_j^T
//
// with (a, b, c) = (q, k, v) for o, (dO, v, k) for dq (state transposed), and, walking the time axis
// backwards with E = dL/dS in the place of S, (v, dO, q) for dk and (k, q, dO) for dv.  Forwards
// pos(i) = i + 1 and pos'(j) = n - 1 - j inside a piece of n tokens; backwards the two change places.
// So one kernel template serves every direction, and a backward pass is one launch of three jobs
// that share their inputs in L2.
//
// Work items: a sequence is cut into segments of seg_len tokens when there are too few (sequence,
// head) pairs to fill the GPU.  Then a state-only sweep leaves every segment's own contribution
// to the state in the workspace, fold_states_kernel turns them into the states entering the
// segments, and the output sweep starts each segment from its own.
#pragma once
#include <math.h>

#include "kernels.h"

namespace prb {

constexpr int kMaxHeadDim = 128;

// (rows, time, heads, channels) array with unit channel stride; strides in elements
struct HeadView {
    const void* p;
    long long sb, st, sh;
};

struct MixJob {
    HeadView a, b, c;
    void* out;           // (rows, time, heads, dc) contiguous, I/O dtype
    const float* s_in;   // [segment][state head][dk*dv] or null = zeros
    float* s_out;        // same layout, or null
    int da, dc;          // channels of a and b, of c and out
    int s_row, s_col;    // strides of the (da, dc) state inside its dk*dv block
    int heads;           // heads of a and out
    int share_a;         // heads of a that read one state head
    int share_b;         // heads of b and c that one head of a sums over
    int reverse;
    int exact;           // the state is an output, not only an operand (tensor cores)
    float p_scale, row_scale, upd_scale;
};

// Where a work item lies: rectangular batches by division, packed ones by a search over cu_seqlens.
struct SegMap {
    const int* cu;  // device, n_seq + 1 offsets, or null
    int n_seq;      // sequences (= rows when rectangular)
    int time;       // tokens of a row
    int seg_len;    // multiple of the chunk
    int n_seg;      // segments of a row (rectangular)
    int n_items;    // grid bound: n_seq * n_seg, or n_seq + time / seg_len when packed
};

struct MixParams {
    MixJob job[3];
    int n_jobs;
    const float* log_decay;
    int state_heads;
    int state_elems;  // dk * dv
    SegMap map;

};

struct Seg {
    int row, seq, t0, len, first, last;
};

// Sequences s0 .. s0 + 31 of a packed batch, one for each lane of a warp (empty behind the last one).  `end` is where
// the sequence before s0 ends; it is moved on.  An offset counts as the largest one up to it, within the row: no
// table can send an access out of range or give a token to two sequences.
__device__ __forceinline__ int first_token(const SegMap& m) { return min(max(m.cu[0], 0), m.time); }
__device__ __forceinline__ void seq_spans(const SegMap& m, int s0, int& end, int& lo, int& hi) {
    const int lane = threadIdx.x & 31;
    hi = end;
    if (s0 + lane < m.n_seq) hi = max(hi, min(m.cu[s0 + lane + 1], m.time));
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, hi, o);
        if (lane >= o) hi = max(hi, v);
    }
    lo = __shfl_up_sync(0xffffffffu, hi, 1);
    if (lane == 0) lo = end;
    end = __shfl_sync(0xffffffffu, hi, 31);
}

// Item x of the grid (whole warp calls it); false when the packed batch has fewer items.
__device__ inline bool locate(const SegMap& m, int x, Seg& s) {
    if (!m.cu) {
        s.seq = s.row = x / m.n_seg;
        const int seg = x - s.seq * m.n_seg;
        s.t0 = seg * m.seg_len;
        s.len = min(m.seg_len, m.time - s.t0);
        s.first = seg == 0;
        s.last = seg == m.n_seg - 1;
        return true;
    }
    const int lane = threadIdx.x & 31;
    int base = 0, end = first_token(m);
    for (int s0 = 0; s0 < m.n_seq; s0 += 32) {
        int lo, hi, cnt = 0;
        seq_spans(m, s0, end, lo, hi);
        if (s0 + lane < m.n_seq) cnt = max(1, (hi - lo + m.seg_len - 1) / m.seg_len);
        int inc = cnt;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += v;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, cnt > 0 && x < base + inc);
        if (hit) {
            const int src = __ffs(hit) - 1;
            const int seg = x - base - (inc - cnt);
            s.row = 0;
            s.seq = s0 + src;
            const int myt0 = lo + seg * m.seg_len;
            s.t0 = __shfl_sync(0xffffffffu, myt0, src);
            s.len = __shfl_sync(0xffffffffu, max(0, min(m.seg_len, hi - myt0)), src);
            s.first = __shfl_sync(0xffffffffu, seg == 0, src);
            s.last = __shfl_sync(0xffffffffu, seg == cnt - 1, src);
            return true;
        }
        base += __shfl_sync(0xffffffffu, inc, 31);
    }
    return false;
}

// w^n; w^0 = 1 also for log_decay = -inf.  In double: the exponent n * log_decay is the only place
// where a long stretch of time could lose accuracy.
__device__ __forceinline__ float decay_pow(double g, int n) { return n == 0 ? 1.0f : (float)exp(g * n); }

cudaError_t launch_mix_simt(const MixParams& p, int dtype, bool state_only, cudaStream_t s);
bool mix_tc_usable(const MixParams& p, int dtype);
cudaError_t launch_mix_tc(const MixParams& p, int rows, bool state_only, cudaStream_t s);
// 0, or kErrChainTimeout when a bounded wait of a tensor-core sweep has run out on this device: of all sweeps
// so far (waits for the device), of those that have reported by now
int linattn_status(int clear);
int linattn_poll(int clear);
// states [item][head] from per-segment contributions (in place); s_out = state behind the last segment
cudaError_t launch_fold_states(const MixParams& p, float* seg_states, const float* s_in, float* s_out,
                               bool reverse, cudaStream_t s);

struct StepArgs {
    const void *q, *k, *v;  // (rows, heads, channels) contiguous
    const float* log_decay;
    float* state;            // (slots, state_heads, dk, dv)
    const void* table;       // (rows,) slot of each row, or null = its own index
    void* out;               // (rows, q heads, dv)
    int rows, slots, hq, hkv, dk, dv, table64;
    float scale;
};
cudaError_t launch_linattn_step(const StepArgs& a, int dtype, cudaStream_t s);

}  // namespace prb
