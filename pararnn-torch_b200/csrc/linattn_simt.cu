// Linear attention with a decay for each head on the CUDA cores: every type and every head size up
// to 128, all arithmetic in fp32.  One CTA walks a segment of one head in chunks of 64 tokens and
// owns 64 of the output channels; its (da, 64) slice of the state stays in shared memory.  Per
// chunk: scores P = a b^T (decayed, causal), out = P c + diag(w^pos) a S, S = w^n S + (w^pos' b)^T c.
//
// This is the fp32 path: the four products are FFMA work (4 x 4 outputs per thread, operands as
// float4 from shared memory), which bounds it; tensor cores would round the operands to fewer bits
// than an fp32 caller asked for.  The next chunk travels from global memory to registers while a
// chunk is worked on, and with da <= 64 two CTAs share an SM.  2 x 1021 tokens, 8 query and 2 key heads of
// 64 / 96 channels: 60 us in 8 segments (kernels traced one by one: state sweep 11, fold 3, outputs 47).
#include "linattn.cuh"

namespace prb {

namespace {

constexpr int kC = 64;      // tokens per chunk
constexpr int kN = 64;      // output channels per CTA
constexpr int kPitch = 68;  // floats per shared-memory row: float4-aligned, rows 4 banks apart
constexpr int kThreads = 256;

template <int D>
struct Smem {
    float at[D][kPitch];  // a, transposed: [channel][token]
    float bt[D][kPitch];
    float c[kC][kPitch];
    float s[D][kPitch];   // state slice
    float pt[kC][kPitch];           // scores, transposed: [key][query]
    float pw[kC + 1];
};

// A 64-token tile of one head on its way through registers: warp w holds tokens w, w + 8, ..., lane l
// the channels l, l + 32, ...; zeros outside.
template <typename TIO, int D>
struct Tile {
    float v[kC / 8][D / 32];
    __device__ __forceinline__ void fetch(const HeadView& view, int row, int t0, int n, int h, int c0, int d) {
        const TIO* base = reinterpret_cast<const TIO*>(view.p) + row * view.sb + (long long)t0 * view.st + h * view.sh + c0;
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
        for (int i = 0; i < kC / 8; ++i)
#pragma unroll
            for (int k = 0; k < D / 32; ++k) {
                const int t = warp + 8 * i, ch = lane + 32 * k;
                v[i][k] = (t < n && ch < d) ? ld_f(base + (long long)t * view.st + ch) : 0.f;
            }
    }
    __device__ __forceinline__ void put_t(float (*dst)[kPitch]) const {
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
        for (int i = 0; i < kC / 8; ++i)
#pragma unroll
            for (int k = 0; k < D / 32; ++k) dst[lane + 32 * k][warp + 8 * i] = v[i][k];
    }
    __device__ __forceinline__ void put(float (*dst)[kPitch]) const {
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
        for (int i = 0; i < kC / 8; ++i)
#pragma unroll
            for (int k = 0; k < D / 32; ++k) dst[warp + 8 * i][lane + 32 * k] = v[i][k];
    }
};

// acc[r][q] += sum_k x[k][r] y[k][q], 4 x 4
__device__ __forceinline__ void mma44(float (&acc)[4][4], const float* x, const float* y) {
    const float4 u = *reinterpret_cast<const float4*>(x), w = *reinterpret_cast<const float4*>(y);
    const float a[4] = {u.x, u.y, u.z, u.w}, b[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int q = 0; q < 4; ++q) acc[r][q] = fmaf(a[r], b[q], acc[r][q]);
}

template <typename TIO, bool STATE_ONLY, int D>
__global__ void __launch_bounds__(kThreads, D == 64 ? 2 : 1) mix_simt_kernel(const __grid_constant__ MixParams p) {
    extern __shared__ __align__(16) unsigned char raw[];
    Smem<D>& sm = *reinterpret_cast<Smem<D>*>(raw);
    int y = blockIdx.y, ji = 0;
    for (; ji + 1 < p.n_jobs; ++ji) {
        const int n = p.job[ji].heads * ((p.job[ji].dc + kN - 1) / kN);
        if (y < n) break;
        y -= n;
    }
    const MixJob& jb = p.job[ji];
    const int n_col = (jb.dc + kN - 1) / kN;
    const int head = y / n_col, c0 = (y % n_col) * kN, dcw = min(kN, jb.dc - c0);
    const int da = jb.da, da_pad = (da + 7) & ~7;
    const int hs = head / jb.share_a;
    Seg seg;
    if (!locate(p.map, blockIdx.x, seg)) return;
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const double g = p.log_decay[hs];
    if (tid <= kC) sm.pw[tid] = decay_pow(g, tid);
    const size_t sbase = ((size_t)blockIdx.x * p.state_heads + hs) * p.state_elems;
    for (int i = tid; i < da_pad * kN; i += kThreads) {
        const int r = i / kN, q = i % kN;
        sm.s[r][q] = (jb.s_in && !STATE_ONLY && r < da && q < dcw)
                         ? jb.s_in[sbase + (size_t)r * jb.s_row + (size_t)(c0 + q) * jb.s_col]
                         : 0.f;
    }
    __syncthreads();
    const int n_chunk = (seg.len + kC - 1) / kC;
    Tile<TIO, D> ra, rb;
    Tile<TIO, kN> rc;
    auto fetch = [&](int m, int gi) {
        if (m >= n_chunk) return;
        const int off = (jb.reverse ? n_chunk - 1 - m : m) * kC;
        const int n = min(kC, seg.len - off), t0 = seg.t0 + off;
        const int hb = jb.share_b > 1 ? head * jb.share_b + gi : hs;
        if (!STATE_ONLY && gi == 0) ra.fetch(jb.a, seg.row, t0, n, head, 0, da);
        rb.fetch(jb.b, seg.row, t0, n, hb, 0, da);
        rc.fetch(jb.c, seg.row, t0, n, hb, c0, dcw);
    };
    fetch(0, 0);
    for (int m = 0; m < n_chunk; ++m) {
        const int off = (jb.reverse ? n_chunk - 1 - m : m) * kC;
        const int n = min(kC, seg.len - off), t0 = seg.t0 + off;
        float acc[4][4] = {};
        for (int gi = 0; gi < jb.share_b; ++gi) {
            if (!STATE_ONLY && gi == 0) ra.put_t(sm.at);
            rb.put_t(sm.bt);
            rc.put(sm.c);
            __syncthreads();
            if (gi + 1 < jb.share_b) fetch(m, gi + 1);
            else fetch(m + 1, 0);
            if (!STATE_ONLY) {
                float pr[4][4] = {};
                for (int d = 0; d < da_pad; ++d) mma44(pr, &sm.at[d][ty * 4], &sm.bt[d][tx * 4]);
                if (gi == 0) {
                    for (int d = 0; d < da_pad; ++d) mma44(acc, &sm.at[d][ty * 4], &sm.s[d][tx * 4]);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int i = ty * 4 + r, e = jb.reverse ? n - 1 - i : i + 1;
                        const float f = i < n ? jb.row_scale * sm.pw[e] : 0.f;
#pragma unroll
                        for (int q = 0; q < 4; ++q) acc[r][q] = i < n ? f * acc[r][q] : 0.f;
                    }
                }
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const int i = ty * 4 + r, j = tx * 4 + q, e = jb.reverse ? j - i : i - j;
                        sm.pt[j][i] = (e >= 0 && j < n && i < n) ? pr[r][q] * (jb.p_scale * sm.pw[e]) : 0.f;
                    }
            }
            __syncthreads();
            if (!STATE_ONLY) {
                float in[4][4] = {};
                for (int j = 0; j < kC; ++j) mma44(in, &sm.pt[j][ty * 4], &sm.c[j][tx * 4]);
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        float v = in[r][q];
                        if (!(fabsf(v) < CUDART_INF_F)) {
                            // a masked score is 0, and 0 x inf = NaN: sum again over the positions
                            // that this row may see, so that what it may not see cannot reach it
                            const int i = ty * 4 + r;
                            v = 0.f;
                            for (int j = jb.reverse ? i : 0; jb.reverse ? j < n : (j <= i && j < n); ++j)
                                v = fmaf(sm.pt[j][i], sm.c[j][tx * 4 + q], v);
                        }
                        acc[r][q] += v;
                    }
            }
            // state: rows 4 ty + 64 r2, columns 4 tx
            const float wn = gi == 0 ? sm.pw[n] : 1.f;
            for (int r0 = ty * 4; r0 < da_pad; r0 += kC) {
                float u[4][4] = {};
                for (int j = 0; j < n; ++j) {
                    const float f = jb.upd_scale * sm.pw[jb.reverse ? j + 1 : n - 1 - j];
                    const float4 cv = *reinterpret_cast<const float4*>(&sm.c[j][tx * 4]);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float b = f * sm.bt[r0 + r][j];
                        u[r][0] = fmaf(b, cv.x, u[r][0]);
                        u[r][1] = fmaf(b, cv.y, u[r][1]);
                        u[r][2] = fmaf(b, cv.z, u[r][2]);
                        u[r][3] = fmaf(b, cv.w, u[r][3]);
                    }
                }
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int q = 0; q < 4; ++q) sm.s[r0 + r][tx * 4 + q] = fmaf(wn, sm.s[r0 + r][tx * 4 + q], u[r][q]);
            }
            __syncthreads();
        }
        if (!STATE_ONLY) {
            TIO* out = reinterpret_cast<TIO*>(jb.out);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int i = ty * 4 + r;
                if (i >= n) continue;
                const size_t at = (((size_t)seg.row * p.map.time + t0 + i) * jb.heads + head) * jb.dc + c0;
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    if (tx * 4 + q < dcw) st_f(out + at + tx * 4 + q, acc[r][q]);
            }
        }
    }
    if (jb.s_out && head % jb.share_a == 0) {
        for (int i = tid; i < da * kN; i += kThreads) {
            const int r = i / kN, q = i % kN;
            if (q < dcw) jb.s_out[sbase + (size_t)r * jb.s_row + (size_t)(c0 + q) * jb.s_col] = sm.s[r][q];
        }
    }
}

template <typename TIO, bool STATE_ONLY, int D>
cudaError_t launch_t(const MixParams& p, cudaStream_t s) {
    int ny = 0;
    for (int j = 0; j < p.n_jobs; ++j) ny += p.job[j].heads * ((p.job[j].dc + kN - 1) / kN);
    cudaError_t e = cudaFuncSetAttribute(mix_simt_kernel<TIO, STATE_ONLY, D>,
                                         cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(Smem<D>));
    if (e != cudaSuccess) return e;
    mix_simt_kernel<TIO, STATE_ONLY, D><<<dim3(p.map.n_items, ny), kThreads, sizeof(Smem<D>), s>>>(p);
    return cudaGetLastError();
}
template <typename TIO>
cudaError_t launch_d(const MixParams& p, bool state_only, cudaStream_t s) {
    bool wide = false;
    for (int j = 0; j < p.n_jobs; ++j) wide |= p.job[j].da > 64;
    if (wide) return state_only ? launch_t<TIO, true, 128>(p, s) : launch_t<TIO, false, 128>(p, s);
    return state_only ? launch_t<TIO, true, 64>(p, s) : launch_t<TIO, false, 64>(p, s);
}

// One thread per state element and (sequence, head): walks the sequence's segments in order.
__global__ void fold_states_kernel(const __grid_constant__ MixParams p, float* seg_states, const float* s_in,
                                   float* s_out, int reverse) {
    const int seq = blockIdx.y, hs = blockIdx.z;
    const int e = blockIdx.x * blockDim.x + threadIdx.x;
    const SegMap& m = p.map;
    int lo = 0, hi = m.time, base = seq * m.n_seg, n = m.n_seg;
    if (m.cu) {
        base = 0;
        const int lane = threadIdx.x & 31;
        int end = first_token(m);
        for (int s0 = 0; s0 <= seq; s0 += 32) {
            int l, h;
            seq_spans(m, s0, end, l, h);
            if (s0 + lane < seq) base += max(1, (h - l + m.seg_len - 1) / m.seg_len);
            if (s0 + 32 > seq) {
                lo = __shfl_sync(0xffffffffu, l, seq - s0);
                hi = __shfl_sync(0xffffffffu, h, seq - s0);
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) base += __shfl_xor_sync(0xffffffffu, base, o);
        n = max(1, (hi - lo + m.seg_len - 1) / m.seg_len);
        n = max(0, min(n, m.n_items - base));
    }
    __shared__ float w[2];  // decay over a full segment and over the last one
    if (threadIdx.x < 2)
        w[threadIdx.x] = decay_pow(p.log_decay[hs], threadIdx.x ? max(0, hi - lo - (n - 1) * m.seg_len) : m.seg_len);
    __syncthreads();
    if (e >= p.state_elems) return;
    const float w_full = w[0], w_last = w[1];
    const size_t own = ((size_t)seq * p.state_heads + hs) * p.state_elems + e;
    float run = s_in ? s_in[own] : 0.f;
    constexpr int kAhead = 8;  // loads in flight
    for (int i0 = 0; i0 < n; i0 += kAhead) {
        float u[kAhead];
        float* at[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const int i = min(i0 + k, n - 1), seg = reverse ? n - 1 - i : i;
            at[k] = seg_states + ((size_t)(base + seg) * p.state_heads + hs) * p.state_elems + e;
            u[k] = *at[k];
        }
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            if (i0 + k >= n) break;
            *at[k] = run;
            run = fmaf((reverse ? i0 + k == 0 : i0 + k == n - 1) ? w_last : w_full, run, u[k]);
        }
    }
    if (s_out) s_out[own] = run;
}

}  // namespace

cudaError_t launch_mix_simt(const MixParams& p, int dtype, bool state_only, cudaStream_t s) {
    return dtype == kF32 ? launch_d<float>(p, state_only, s) : launch_d<__nv_bfloat16>(p, state_only, s);
}

cudaError_t launch_fold_states(const MixParams& p, float* seg_states, const float* s_in, float* s_out, bool reverse,
                               cudaStream_t s) {
    const dim3 grid((p.state_elems + 255) / 256, p.map.n_seq, p.state_heads);
    fold_states_kernel<<<grid, 256, 0, s>>>(p, seg_states, s_in, s_out, reverse ? 1 : 0);
    return cudaGetLastError();
}

}  // namespace prb
