// One token of linear attention with a decay for each head: S = w S + k v^T, o = s q S, in place on a
// pool of fp32 states.  The state is read once and written once (8 bytes per element against 2 - 4
// flops), so the kernel is HBM-bound: a CTA owns a (row, state head) and a slice of the value
// channels, issues all its state loads before anything else and keeps the slice in registers for the
// update and for every query head that reads this state.  With few (row, head) pairs a slice is 32
// channels instead of all, which puts four times as many CTAs on the wires: 8 heads of 128 x 128 take
// 3.2 us for one row (4.8 in whole rows) and 5.0 for 16 (5.4), but 8.0 for 32 rows (7.1).  192 rows of a pool
// take 40.8 us, 4.9 TB/s or 76 % of the copy rate.
#include "linattn.cuh"

namespace prb {

namespace {

constexpr int kThreads = 256;

template <typename TIO, int VEC, int LANES>
__global__ void __launch_bounds__(kThreads) linattn_step_kernel(const StepArgs p) {
    constexpr int R = kThreads / LANES;          // state rows in flight per pass
    constexpr int NR = (kMaxHeadDim + R - 1) / R;  // rows per thread
    constexpr int SL = LANES * VEC;
    __shared__ float sk[kMaxHeadDim], sq[kMaxHeadDim], red[R][SL];
    __shared__ int s_next;
    const int row0 = blockIdx.x, hs = blockIdx.y, c0 = blockIdx.z * SL;
    const int tid = threadIdx.x, lane = tid % LANES, rg = tid / LANES, col = c0 + lane * VEC;
    const bool live = col < p.dv;
    auto entry = [&](int r) -> long long {
        return p.table64 ? reinterpret_cast<const long long*>(p.table)[r]
                         : (long long)reinterpret_cast<const int*>(p.table)[r];
    };
    const int share = p.hq / p.hkv;
    TIO* out = reinterpret_cast<TIO*>(p.out);
    const long long slot = p.table ? entry(row0) : row0;
    if (slot < 0 || slot >= p.slots) {
        // padding row: no state is touched, its outputs are zero
        for (int i = tid; i < share * SL; i += kThreads) {
            const int g = i / SL, c = c0 + i % SL;
            if (c < p.dv) st_f(out + ((size_t)row0 * p.hq + hs * share + g) * p.dv + c, 0.f);
        }
        return;
    }
    float* state = p.state + ((size_t)slot * p.hkv + hs) * p.dk * p.dv + col;
    float s[NR][VEC];
    bool loaded = false;
    const float w = decay_pow(p.log_decay[hs], 1);
    auto load_state = [&]() {
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            const int r = rg + i * R;
            if (r < p.dk && live) {
                if constexpr (VEC == 4) {
                    const float4 v = *reinterpret_cast<const float4*>(state + (size_t)r * p.dv);
                    s[i][0] = v.x, s[i][1] = v.y, s[i][2] = v.z, s[i][3] = v.w;
                } else {
                    s[i][0] = state[(size_t)r * p.dv];
                }
            } else {
#pragma unroll
                for (int q = 0; q < VEC; ++q) s[i][q] = 0.f;
            }
        }
    };
    // the first row that names a slot applies all rows that name it, in row order; the others leave
    if (tid == 0) s_next = p.rows;
    __syncthreads();
    int row = row0;
    while (row < p.rows) {
        const size_t kh = (size_t)row * p.hkv + hs;
        float vv[VEC];
#pragma unroll
        for (int q = 0; q < VEC; ++q)
            vv[q] = live ? ld_f(reinterpret_cast<const TIO*>(p.v) + kh * p.dv + col + q) : 0.f;
        if (tid < p.dk) sk[tid] = ld_f(reinterpret_cast<const TIO*>(p.k) + kh * p.dk + tid);
        if (!loaded) {
            load_state();
            loaded = true;
        }
        bool earlier = false;
        if (p.table) {
            int next = p.rows;
            for (int r = tid; r < p.rows; r += kThreads) {
                if (r != row && entry(r) == slot) {
                    if (r < row0) earlier = true;
                    else if (r > row) next = min(next, r);
                }
            }
            if (next < p.rows) atomicMin(&s_next, next);
        }
        if (__syncthreads_or(earlier)) return;
        const int next = s_next;
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            const int r = rg + i * R;
            const float kr = r < p.dk ? sk[r] : 0.f;
#pragma unroll
            for (int q = 0; q < VEC; ++q) s[i][q] = fmaf(kr, vv[q], w * s[i][q]);
        }
        for (int g = 0; g < share; ++g) {
            const size_t qh = (size_t)row * p.hq + hs * share + g;
            if (tid < p.dk) sq[tid] = p.scale * ld_f(reinterpret_cast<const TIO*>(p.q) + qh * p.dk + tid);
            __syncthreads();
            float o[VEC] = {};
#pragma unroll
            for (int i = 0; i < NR; ++i) {
                const int r = rg + i * R;
                if (r < p.dk) {
                    const float qr = sq[r];
#pragma unroll
                    for (int q = 0; q < VEC; ++q) o[q] = fmaf(qr, s[i][q], o[q]);
                }
            }
#pragma unroll
            for (int q = 0; q < VEC; ++q) red[rg][lane * VEC + q] = o[q];
            __syncthreads();
            if (tid < SL && c0 + tid < p.dv) {
                float t = 0.f;
#pragma unroll
                for (int r = 0; r < R; ++r) t += red[r][tid];
                st_f(out + qh * p.dv + c0 + tid, t);
            }
        }
        __syncthreads();
        if (tid == 0) s_next = p.rows;
        __syncthreads();
        row = next;
    }
#pragma unroll
    for (int i = 0; i < NR; ++i) {
        const int r = rg + i * R;
        if (r < p.dk && live) {
            if constexpr (VEC == 4)
                *reinterpret_cast<float4*>(state + (size_t)r * p.dv) = make_float4(s[i][0], s[i][1], s[i][2], s[i][3]);
            else
                state[(size_t)r * p.dv] = s[i][0];
        }
    }
}

template <typename TIO>
cudaError_t launch_t(const StepArgs& a, cudaStream_t s) {
    if (a.dv % 4 || (reinterpret_cast<uintptr_t>(a.state) & 15))
        linattn_step_kernel<TIO, 1, 32><<<dim3(a.rows, a.hkv, (a.dv + 31) / 32), kThreads, 0, s>>>(a);
    else if (a.dv <= 32 || 2ll * a.rows * a.hkv < 3ll * sm_count())
        linattn_step_kernel<TIO, 4, 8><<<dim3(a.rows, a.hkv, (a.dv + 31) / 32), kThreads, 0, s>>>(a);
    else
        linattn_step_kernel<TIO, 4, 32><<<dim3(a.rows, a.hkv, 1), kThreads, 0, s>>>(a);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_linattn_step(const StepArgs& a, int dtype, cudaStream_t s) {
    return dtype == kF32 ? launch_t<float>(a, s) : launch_t<__nv_bfloat16>(a, s);
}

}  // namespace prb
