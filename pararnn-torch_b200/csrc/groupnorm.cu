// Group norm with an activation over channel-last tensors (samples, positions, channels), forward and
// backward:  y = act(xhat w + b),  xhat = (x - mean) rstd,  statistics of a group of channels over all
// positions of a sample.  With one position per sample this is the norm over each head's channels
// behind a sequence mixer.
//
//   du = dy act'(xhat w + b);  dx = rstd (w du - mean(w du) - xhat mean(w du xhat));
//   dw = sum du xhat;  db = sum du
//
// Everything is HBM-bound (2 resp. 3 passes over the data against some 30 flops per element), so the
// kernels are about touching memory once:
//   rows   one position, groups up to 32 lanes x 4 vectors: a group sits in the registers of 1 - 32
//          lanes, mean and variance are two register passes, the data moves exactly once.
//   slabs  everything else: a first launch leaves each slab's (mean, M2) or (sum du, sum du xhat) per
//          group, a second one merges them and writes the result; it finds the data still in L2
//          because the host walks the samples in pieces of at most kPieceBytes.  Backwards a CTA of the
//          first launch walks several samples, so that dw and db need as many partial rows as CTAs.
// Squares are only ever summed about the mean of their own batch of positions, never about zero or about a chosen
// value; batches, threads, slabs and channel blocks are joined as (count, mean, M2).  All partial sums are added
// in a fixed order, so results repeat bit for bit.
#include <type_traits>

#include "groupnorm.cuh"

namespace prb {

namespace {

constexpr int kT = 256;
// CTAs per SM of the persistent row kernels (one vector per lane) and of the slab kernels; the grids are
// whole waves of them.  Few CTAs with many loads in flight per thread beat many with few: on 32768 x 1024
// bf16 the forward takes 31.6 us at 4 CTAs, 34 at 5, 37 at 6 and 44 at 8 (spills); on 16 x 4096 x 256 the
// slab kernels take 77 us (forward and backward) at 2 CTAs and 8 loads, 86 at 4 and 4, 115 at 6 and 4.
constexpr int kRowCtasFwd = 4, kRowCtasBwd = 3, kSlabCtas = 2;
constexpr int kMaxLocal = kT + 2;  // groups that one CTA's channels can touch
constexpr int kBatch = 8, kPair = 8;  // positions whose loads a thread issues together (one input, two inputs)

// V neighbouring channels as they lie in memory; loads are issued well before their conversion
template <typename T, int V>
struct __align__(sizeof(T) * V) Pack {
    T v[V];
};
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_raw(const T* p) {
    return *reinterpret_cast<const Pack<T, V>*>(p);
}
// V channels in fp32; pairs go through the packed fp32 instructions, which halves the issue slots that
// bound these kernels (28 instructions per element without them, HBM needs about 10)
template <int V>
struct Vals {
    float2 a[V / 2];
};
template <>
struct Vals<1> {
    float a[1];
};
__device__ __forceinline__ float2 op_add(float2 x, float2 y) { return __fadd2_rn(x, y); }
__device__ __forceinline__ float2 op_mul(float2 x, float2 y) { return __fmul2_rn(x, y); }
__device__ __forceinline__ float2 op_fma(float2 x, float2 y, float2 z) { return __ffma2_rn(x, y, z); }
__device__ __forceinline__ float op_add(float x, float y) { return x + y; }
__device__ __forceinline__ float op_mul(float x, float y) { return x * y; }
__device__ __forceinline__ float op_fma(float x, float y, float z) { return fmaf(x, y, z); }
__device__ __forceinline__ float2 op_ex2(float2 x) { return ex2_2(x); }
__device__ __forceinline__ float op_ex2(float x) { return ex2_approx(x); }
__device__ __forceinline__ float2 op_rcp(float2 x) { return rcp_2(x); }
__device__ __forceinline__ float op_rcp(float x) { return rcp_f(x); }
template <typename E>
__device__ __forceinline__ E all(float x);
template <>
__device__ __forceinline__ float all<float>(float x) { return x; }
template <>
__device__ __forceinline__ float2 all<float2>(float x) { return make_float2(x, x); }
__device__ __forceinline__ float total(float x) { return x; }
__device__ __forceinline__ float total(float2 x) { return x.x + x.y; }
template <int V>
constexpr int kN = V == 1 ? 1 : V / 2;  // elements of Vals
template <int V>
using Elem = std::conditional_t<V == 1, float, float2>;

template <typename T, int V>
__device__ __forceinline__ void unpack(Vals<V>& r, const Pack<T, V>& u) {
    if constexpr (V == 1) {
        r.a[0] = static_cast<float>(u.v[0]);
    } else if constexpr (sizeof(T) == 2) {
        const uint32_t* w = reinterpret_cast<const uint32_t*>(&u);
#pragma unroll
        for (int i = 0; i < V / 2; ++i)
            r.a[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
    } else {
#pragma unroll
        for (int i = 0; i < V / 2; ++i) r.a[i] = make_float2(u.v[2 * i], u.v[2 * i + 1]);
    }
}
template <typename T, int V>
__device__ __forceinline__ void store_v(T* p, const Vals<V>& r) {
    Pack<T, V> u;
    if constexpr (V == 1) {
        st_f(&u.v[0], r.a[0]);
    } else if constexpr (sizeof(T) == 2) {
        __nv_bfloat162* w = reinterpret_cast<__nv_bfloat162*>(&u);
#pragma unroll
        for (int i = 0; i < V / 2; ++i) w[i] = __floats2bfloat162_rn(r.a[i].x, r.a[i].y);
    } else {
#pragma unroll
        for (int i = 0; i < V / 2; ++i) u.v[2 * i] = r.a[i].x, u.v[2 * i + 1] = r.a[i].y;
    }
    *reinterpret_cast<Pack<T, V>*>(p) = u;
}
__device__ __forceinline__ float affine(const void* p, int f32, int i, float none) {
    if (!p) return none;
    return f32 ? __ldg(reinterpret_cast<const float*>(p) + i)
               : __bfloat162float(__ldg(reinterpret_cast<const __nv_bfloat16*>(p) + i));
}

__device__ __forceinline__ float gelu_cdf(float u) { return normcdff(u); }
__device__ __forceinline__ float2 gelu_cdf(float2 u) { return make_float2(normcdff(u.x), normcdff(u.y)); }
__device__ __forceinline__ float gelu_pdf(float u) { return 0.3989422804014327f * expf(-0.5f * u * u); }
__device__ __forceinline__ float2 gelu_pdf(float2 u) { return make_float2(gelu_pdf(u.x), gelu_pdf(u.y)); }
template <typename E>
__device__ __forceinline__ E sigmoid_e(E u) {
    return op_rcp(op_add(op_ex2(op_mul(u, all<E>(-1.4426950216293335f))), all<E>(1.f)));
}
template <int ACT, typename E>
__device__ __forceinline__ E act(E u) {
    if constexpr (ACT == kActSilu) return op_mul(u, sigmoid_e(u));
    if constexpr (ACT == kActGelu) return op_mul(u, gelu_cdf(u));
    return u;
}
template <int ACT, typename E>
__device__ __forceinline__ E act_slope(E u) {
    if constexpr (ACT == kActSilu) {
        const E s = sigmoid_e(u);
        return op_mul(s, op_fma(u, op_fma(s, all<E>(-1.f), all<E>(1.f)), all<E>(1.f)));
    }
    if constexpr (ACT == kActGelu) return op_fma(u, gelu_pdf(u), gelu_cdf(u));
    return all<E>(1.f);
}
// weight or bias of V channels from c on
template <int V>
__device__ __forceinline__ Vals<V> affine_v(const void* p, int f32, int c, float none, bool in) {
    Vals<V> r;
    if constexpr (V == 1) {
        r.a[0] = in ? affine(p, f32, c, none) : 0.f;
    } else {
#pragma unroll
        for (int i = 0; i < V / 2; ++i)
            r.a[i] = in ? make_float2(affine(p, f32, c + 2 * i, none), affine(p, f32, c + 2 * i + 1, none))
                        : make_float2(0.f, 0.f);
    }
    return r;
}
template <int V>
__device__ __forceinline__ float at(const Vals<V>& r, int i) {
    if constexpr (V == 1) return r.a[0];
    else return i & 1 ? r.a[i / 2].y : r.a[i / 2].x;
}

template <int LANES>
__device__ __forceinline__ float lane_sum(float v) {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// ---------------------------------------------------------------------------------------- rows
// Thread slots: LANES lanes per group, NV vectors of V channels per lane; a CTA holds kT / slots
// rows at a time (or a 256-slot piece of a wide row, blockIdx.y).
struct RowSlot {
    int g, sub, lane, rows;
    bool live;
};
template <int LANES>
__device__ __forceinline__ RowSlot row_slot(int groups) {
    RowSlot r;
    const int slots = groups * LANES;
    const int wide = slots > kT;
    const int per = wide ? kT : slots;
    r.rows = kT / per;
    r.sub = threadIdx.x / per;
    const int slot = threadIdx.x % per + blockIdx.y * kT;
    r.g = slot / LANES;
    r.lane = slot % LANES;
    r.live = r.sub < r.rows && r.g < groups;
    return r;
}

template <typename T, int V, int NV, int LANES, int ACT>
__global__ void __launch_bounds__(kT, NV == 1 ? kRowCtasFwd : 2) gn_rows_fwd(const __grid_constant__ GroupNormArgs p) {
    const RowSlot rs = row_slot<LANES>(p.groups);
    const int cg = p.channels / p.groups;
    using E = Elem<V>;
    constexpr int N = kN<V>;
    Vals<V> w[NV], b[NV];
    bool in[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        in[j] = rs.live && (j * LANES + rs.lane) * V < cg;
        const int c = rs.g * cg + (j * LANES + rs.lane) * V;
        w[j] = affine_v<V>(p.w, p.w_f32, c, 1.f, in[j]);
        b[j] = affine_v<V>(p.b, p.w_f32, c, 0.f, in[j]);
    }
    const float inv = 1.f / cg;
    const size_t step = (size_t)gridDim.x * rs.rows;
    const size_t col = (size_t)rs.g * cg + rs.lane * V;
    size_t row = (size_t)blockIdx.x * rs.rows + rs.sub;
    Pack<T, V> raw[NV] = {};
    auto fetch = [&](size_t r) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (in[j] && r < (size_t)p.samples)
                raw[j] = load_raw<T, V>(reinterpret_cast<const T*>(p.x) + r * p.channels + col + j * LANES * V);
    };
    fetch(row);
    // all threads of a CTA take the same number of turns: the shuffles need whole warps
    for (size_t r0 = (size_t)blockIdx.x * rs.rows; r0 < (size_t)p.samples; r0 += step, row += step) {
        Vals<V> x[NV];
        E s = all<E>(0.f);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            unpack<T, V>(x[j], raw[j]);
            if (in[j]) {
#pragma unroll
                for (int i = 0; i < N; ++i) s = op_add(s, x[j].a[i]);
            }
        }
        fetch(row + step);
        const float mean = lane_sum<LANES>(total(s)) * inv;
        E m2 = all<E>(0.f);
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (in[j]) {
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    x[j].a[i] = op_add(x[j].a[i], all<E>(-mean));
                    m2 = op_fma(x[j].a[i], x[j].a[i], m2);
                }
            }
        const float rstd = rsqrtf(lane_sum<LANES>(total(m2)) * inv + p.eps);
        if (!rs.live || row >= (size_t)p.samples) continue;
        if (rs.lane == 0 && p.stats) p.stats[row * p.groups + rs.g] = make_float2(mean, rstd);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            if (!in[j]) continue;
#pragma unroll
            for (int i = 0; i < N; ++i)
                x[j].a[i] = act<ACT>(op_fma(op_mul(x[j].a[i], all<E>(rstd)), w[j].a[i], b[j].a[i]));
            store_v<T, V>(reinterpret_cast<T*>(p.y) + row * p.channels + col + j * LANES * V, x[j]);
        }
    }
}

template <typename T, int V, int NV, int LANES, int ACT>
__global__ void __launch_bounds__(kT, NV == 1 ? kRowCtasBwd : 1) gn_rows_bwd(const __grid_constant__ GroupNormArgs p) {
    const RowSlot rs = row_slot<LANES>(p.groups);
    const int cg = p.channels / p.groups;
    using E = Elem<V>;
    constexpr int N = kN<V>;
    Vals<V> w[NV], b[NV], dw[NV], db[NV];
    bool in[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        in[j] = rs.live && (j * LANES + rs.lane) * V < cg;
        const int c = rs.g * cg + (j * LANES + rs.lane) * V;
        w[j] = affine_v<V>(p.w, p.w_f32, c, 1.f, in[j]);
        b[j] = affine_v<V>(p.b, p.w_f32, c, 0.f, in[j]);
#pragma unroll
        for (int i = 0; i < N; ++i) dw[j].a[i] = db[j].a[i] = all<E>(0.f);
    }
    const float inv = 1.f / cg;
    const size_t step = (size_t)gridDim.x * rs.rows;
    const size_t col = (size_t)rs.g * cg + rs.lane * V;
    size_t row = (size_t)blockIdx.x * rs.rows + rs.sub;
    Pack<T, V> raw_x[NV] = {}, raw_d[NV] = {};
    float2 st = make_float2(0.f, 0.f);
    auto fetch = [&](size_t r) {
        if (!rs.live || r >= (size_t)p.samples) return;
        st = p.stats[r * p.groups + rs.g];
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (in[j]) {
                const size_t at = r * p.channels + col + j * LANES * V;
                raw_x[j] = load_raw<T, V>(reinterpret_cast<const T*>(p.x) + at);
                raw_d[j] = load_raw<T, V>(reinterpret_cast<const T*>(p.dy) + at);
            }
    };
    fetch(row);
    for (size_t r0 = (size_t)blockIdx.x * rs.rows; r0 < (size_t)p.samples; r0 += step, row += step) {
        const bool live = rs.live && row < (size_t)p.samples;
        const float2 ms = st;
        Vals<V> h[NV], d[NV];  // xhat, then w du
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            unpack<T, V>(h[j], raw_x[j]);
            unpack<T, V>(d[j], raw_d[j]);
        }
        fetch(row + step);
        E s1 = all<E>(0.f), s2 = all<E>(0.f);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            if (live && in[j]) {
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const E x = op_mul(op_add(h[j].a[i], all<E>(-ms.x)), all<E>(ms.y));
                    const E du = op_mul(d[j].a[i], act_slope<ACT>(op_fma(x, w[j].a[i], b[j].a[i])));
                    dw[j].a[i] = op_fma(du, x, dw[j].a[i]);
                    db[j].a[i] = op_add(db[j].a[i], du);
                    h[j].a[i] = x;
                    d[j].a[i] = op_mul(du, w[j].a[i]);
                    s1 = op_add(s1, d[j].a[i]);
                    s2 = op_fma(d[j].a[i], x, s2);
                }
            }
        }
        const float m1 = lane_sum<LANES>(total(s1)) * inv, m2 = lane_sum<LANES>(total(s2)) * inv;
        if (!live) continue;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            if (!in[j]) continue;
#pragma unroll
            for (int i = 0; i < N; ++i)
                d[j].a[i] = op_mul(all<E>(ms.y),
                                   op_fma(h[j].a[i], all<E>(-m2), op_add(d[j].a[i], all<E>(-m1))));
            store_v<T, V>(reinterpret_cast<T*>(p.dx) + row * p.channels + col + j * LANES * V, d[j]);
        }
    }
    // one row of partial sums per CTA: its rows in order of `sub`
    __shared__ float red[2][kT][V];
    const int slots = min(kT, p.groups * LANES);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < V; ++i) {
            red[0][threadIdx.x][i] = at(dw[j], i);
            red[1][threadIdx.x][i] = at(db[j], i);
        }
        __syncthreads();
        if (rs.sub == 0 && in[j]) {
            float* dst = p.partial + (size_t)blockIdx.x * 2 * p.channels + col + j * LANES * V;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                float a0 = 0.f, a1 = 0.f;
                for (int k = 0; k < rs.rows; ++k) {
                    a0 += red[0][threadIdx.x + k * slots][i];
                    a1 += red[1][threadIdx.x + k * slots][i];
                }
                dst[i] = a0;
                dst[p.channels + i] = a1;
            }
        }
    }
}

// --------------------------------------------------------------------------------------- slabs
// blockIdx = (slab of positions, sample, block of kT * V channels).  A thread keeps one vector of V
// channels (all of one group) and walks the slab's positions.
struct SlabSlot {
    int c, g, sub, rows, p0, p1;
    bool live;
};
template <int V>
__device__ __forceinline__ SlabSlot slab_slot(const GroupNormArgs& p) {
    SlabSlot s;
    const int slots = p.channels / V;
    const int per = min(slots, kT);
    s.rows = kT / per;
    s.sub = threadIdx.x / per;
    const int slot = threadIdx.x % per + blockIdx.z * kT;
    s.c = slot * V;
    s.live = s.sub < s.rows && slot < slots;
    s.g = s.live ? s.c / (p.channels / p.groups) : 0;
    s.p0 = (int)((long long)blockIdx.x * p.positions / p.slabs);
    s.p1 = (int)((long long)(blockIdx.x + 1) * p.positions / p.slabs);
    return s;
}
// Joins (count, mean, M2) entries over a warp without a division per pair: the common mean first, then
// every entry's M2 and its distance from that mean.  `entry(t)` gives entry t of `total`.
template <typename F>
__device__ __forceinline__ float3 warp_join(int total, const F& entry) {
    const int lane = threadIdx.x & 31;
    float n = 0.f, sum = 0.f;
    for (int t = lane; t < total; t += 32) {
        const float3 u = entry(t);
        n += u.x;
        sum = fmaf(u.x, u.y, sum);
    }
    n = lane_sum<32>(n);
    const float mean = n > 0.f ? lane_sum<32>(sum) / n : 0.f;
    float m2 = 0.f;
    for (int t = lane; t < total; t += 32) {
        const float3 u = entry(t);
        const float d = u.y - mean;
        m2 += u.x > 0.f ? fmaf(u.x * d, d, u.z) : 0.f;
    }
    return make_float3(n, mean, lane_sum<32>(m2));
}
// groups that this CTA's channels touch
template <int V>
__device__ __forceinline__ void local_groups(const GroupNormArgs& p, int& lo, int& n) {
    const int cg = p.channels / p.groups;
    lo = blockIdx.z * kT * V / cg;
    n = (min(p.channels, (int)(blockIdx.z + 1) * kT * V) - 1) / cg - lo + 1;
}
// channel blocks that hold a piece of group g
template <int V>
__device__ __forceinline__ void group_blocks(const GroupNormArgs& p, int g, int& lo, int& n) {
    const int cg = p.channels / p.groups;
    lo = g * cg / (kT * V);
    n = (g * cg + cg - 1) / (kT * V) - lo + 1;
}

// a group's sums over one slab and one of the channel blocks that it touches; samples count from the piece's first
__device__ __forceinline__ float4* group_entry(const GroupNormArgs& p, size_t sample, int slab, int g, int block) {
    return reinterpret_cast<float4*>(p.group_part) + ((sample * p.slabs + slab) * p.groups + g) * p.span + block;
}

template <typename T, int V>
__global__ void __launch_bounds__(kT, kSlabCtas) gn_slab_stats(const __grid_constant__ GroupNormArgs p) {
    __shared__ float sn[kT], sm[kT], sv[kT];
    const SlabSlot s = slab_slot<V>(p);
    const size_t n = p.sample0 + blockIdx.y;
    const T* x = reinterpret_cast<const T*>(p.x) + n * p.positions * p.channels + s.c;
    // each batch's mean first, then its squares about that mean; batches are joined as (count, mean, M2)
    using E = Elem<V>;
    float cnt = 0.f, mean = 0.f, m2 = 0.f;
    if (s.live) {
        for (int q0 = s.p0 + s.sub; q0 < s.p1; q0 += kBatch * s.rows) {
            Pack<T, V> raw[kBatch];
#pragma unroll
            for (int e = 0; e < kBatch; ++e) {
                const int q = min(q0 + e * s.rows, s.p1 - 1);
                raw[e] = load_raw<T, V>(x + (size_t)q * p.channels);
            }
            const int here = min(kBatch, (s.p1 - q0 + s.rows - 1) / s.rows);
            E t1 = all<E>(0.f), t2 = all<E>(0.f);
#pragma unroll
            for (int e = 0; e < kBatch; ++e) {
                if (e >= here) break;
                Vals<V> v;
                unpack<T, V>(v, raw[e]);
#pragma unroll
                for (int i = 0; i < kN<V>; ++i) t1 = op_add(t1, v.a[i]);
            }
            const float n = (float)(here * V), m = total(t1) / n;
#pragma unroll
            for (int e = 0; e < kBatch; ++e) {
                if (e >= here) break;
                Vals<V> v;
                unpack<T, V>(v, raw[e]);
#pragma unroll
                for (int i = 0; i < kN<V>; ++i) {
                    const E d = op_add(v.a[i], all<E>(-m));
                    t2 = op_fma(d, d, t2);
                }
            }
            const float d = m - mean, part = n / (cnt + n);
            m2 += fmaf(d * (cnt * part), d, total(t2));
            mean = fmaf(d, part, mean);
            cnt += n;
        }
    }
    sn[threadIdx.x] = cnt;
    sm[threadIdx.x] = mean;
    sv[threadIdx.x] = m2;
    __syncthreads();
    int g0, ng;
    local_groups<V>(p, g0, ng);
    const int cg = p.channels / p.groups, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int per = min(p.channels / V, kT);
    for (int k = warp; k < ng; k += kT / 32) {
        const int g = g0 + k;
        const int lo = max(0, g * cg / V - (int)blockIdx.z * kT), hi = min(per, (g + 1) * cg / V - (int)blockIdx.z * kT);
        const int width = hi - lo, total = width * s.rows;
        const float3 j = warp_join(total, [&](int t) {
            const int id = (t / width) * per + lo + t % width;
            return make_float3(sn[id], sm[id], sv[id]);
        });
        int b0, nb;
        group_blocks<V>(p, g, b0, nb);
        if (lane == 0)
            *group_entry(p, blockIdx.y, blockIdx.x, g, blockIdx.z - b0) = make_float4(j.x, j.y, j.z, 0.f);
    }
}

template <typename T, int V, int ACT>
__global__ void __launch_bounds__(kT, kSlabCtas) gn_slab_fwd(const __grid_constant__ GroupNormArgs p) {
    __shared__ float2 st[kMaxLocal];
    const SlabSlot s = slab_slot<V>(p);
    const size_t n = p.sample0 + blockIdx.y;
    int g0, ng;
    local_groups<V>(p, g0, ng);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int k = warp; k < ng; k += kT / 32) {
        int b0, nb;
        group_blocks<V>(p, g0 + k, b0, nb);
        const float3 j = warp_join(p.slabs * nb, [&](int t) {
            const float4 u = *group_entry(p, blockIdx.y, t / nb, g0 + k, t % nb);
            return make_float3(u.x, u.y, u.z);
        });
        if (lane == 0) {
            const float2 r = make_float2(j.y, rsqrtf(j.z / j.x + p.eps));
            st[k] = r;
            if (blockIdx.x == 0 && p.stats && b0 == (int)blockIdx.z) p.stats[n * p.groups + g0 + k] = r;
        }
    }
    __syncthreads();
    if (!s.live) return;
    const float2 ms = st[s.g - g0];
    using E = Elem<V>;
    Vals<V> w = affine_v<V>(p.w, p.w_f32, s.c, 1.f, true);
    const Vals<V> b = affine_v<V>(p.b, p.w_f32, s.c, 0.f, true);
#pragma unroll
    for (int i = 0; i < kN<V>; ++i) w.a[i] = op_mul(w.a[i], all<E>(ms.y));
    const size_t base = n * p.positions * p.channels + s.c;
    for (int q0 = s.p0 + s.sub; q0 < s.p1; q0 += kBatch * s.rows) {
        Pack<T, V> raw[kBatch];
#pragma unroll
        for (int e = 0; e < kBatch; ++e) {
            const int q = min(q0 + e * s.rows, s.p1 - 1);
            raw[e] = load_raw<T, V>(reinterpret_cast<const T*>(p.x) + base + (size_t)q * p.channels);
        }
#pragma unroll
        for (int e = 0; e < kBatch; ++e) {
            const int q = q0 + e * s.rows;
            if (q >= s.p1) break;
            Vals<V> v;
            unpack<T, V>(v, raw[e]);
#pragma unroll
            for (int i = 0; i < kN<V>; ++i)
                v.a[i] = act<ACT>(op_fma(op_add(v.a[i], all<E>(-ms.x)), w.a[i], b.a[i]));
            store_v<T, V>(reinterpret_cast<T*>(p.y) + base + (size_t)q * p.channels, v);
        }
    }
}

// Narrow vectors leave registers for more CTAs: 1000000 x 2 x 2 bf16 backward 15.1 ms at 3, 20.6 at 2.
constexpr int sum_ctas(int vec) { return vec > 2 ? kSlabCtas : vec == 2 ? 3 : 4; }
// A CTA walks the samples blockIdx.y, blockIdx.y + gridDim.y, ... of the piece and adds its channels' sums over them,
// so that there are as many rows of partial sums as CTAs in a wave, however many samples there are.
template <typename T, int V, int ACT>
__global__ void __launch_bounds__(kT, sum_ctas(V)) gn_slab_sums(const __grid_constant__ GroupNormArgs p) {
    __shared__ float red[2][kT][V];
    __shared__ float gs[2][kT];
    const SlabSlot s = slab_slot<V>(p);
    using E = Elem<V>;
    const Vals<V> w = affine_v<V>(p.w, p.w_f32, s.c, 1.f, s.live), b = affine_v<V>(p.b, p.w_f32, s.c, 0.f, s.live);
    const int per = min(p.channels / V, kT), cg = p.channels / p.groups, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int g0, ng;
    local_groups<V>(p, g0, ng);
    float run0[V], run1[V];
#pragma unroll
    for (int i = 0; i < V; ++i) run0[i] = run1[i] = 0.f;
    for (size_t n = p.sample0 + blockIdx.y; n < (size_t)p.sample1; n += gridDim.y) {
        Vals<V> dw, db;
#pragma unroll
        for (int i = 0; i < kN<V>; ++i) dw.a[i] = db.a[i] = all<E>(0.f);
        const size_t base = n * p.positions * p.channels + s.c;
        if (s.live) {
            const float2 ms = p.stats[n * p.groups + s.g];
            for (int q0 = s.p0 + s.sub; q0 < s.p1; q0 += kPair * s.rows) {
                Pack<T, V> raw_x[kPair], raw_d[kPair];
#pragma unroll
                for (int e = 0; e < kPair; ++e) {
                    const size_t at = base + (size_t)min(q0 + e * s.rows, s.p1 - 1) * p.channels;
                    raw_x[e] = load_raw<T, V>(reinterpret_cast<const T*>(p.x) + at);
                    raw_d[e] = load_raw<T, V>(reinterpret_cast<const T*>(p.dy) + at);
                }
#pragma unroll
                for (int e = 0; e < kPair; ++e) {
                    if (q0 + e * s.rows >= s.p1) break;
                    Vals<V> h, d;
                    unpack<T, V>(h, raw_x[e]);
                    unpack<T, V>(d, raw_d[e]);
#pragma unroll
                    for (int i = 0; i < kN<V>; ++i) {
                        const E x = op_mul(op_add(h.a[i], all<E>(-ms.x)), all<E>(ms.y));
                        const E du = op_mul(d.a[i], act_slope<ACT>(op_fma(x, w.a[i], b.a[i])));
                        dw.a[i] = op_fma(du, x, dw.a[i]);
                        db.a[i] = op_add(db.a[i], du);
                    }
                }
            }
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
            red[0][threadIdx.x][i] = at(dw, i);
            red[1][threadIdx.x][i] = at(db, i);
        }
        __syncthreads();
        float t1 = 0.f, t2 = 0.f;  // sum of w du, of w du xhat over this thread's channels
        if (s.live && s.sub == 0) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                float a0 = 0.f, a1 = 0.f;
                for (int k = 0; k < s.rows; ++k) {
                    a0 += red[0][threadIdx.x + k * per][i];
                    a1 += red[1][threadIdx.x + k * per][i];
                }
                run0[i] += a0;
                run1[i] += a1;
                t1 = fmaf(at(w, i), a1, t1);
                t2 = fmaf(at(w, i), a0, t2);
            }
        }
        gs[0][threadIdx.x] = t1;
        gs[1][threadIdx.x] = t2;
        __syncthreads();  // also before the next sample's `red`; its `gs` is behind the barrier after that
        for (int k = warp; k < ng; k += kT / 32) {
            const int g = g0 + k;
            const int lo = max(0, g * cg / V - (int)blockIdx.z * kT), hi = min(per, (g + 1) * cg / V - (int)blockIdx.z * kT);
            float a = 0.f, c = 0.f;
            for (int t = lo + lane; t < hi; t += 32) {
                a += gs[0][t];
                c += gs[1][t];
            }
            a = lane_sum<32>(a);
            c = lane_sum<32>(c);
            int b0, nb;
            group_blocks<V>(p, g, b0, nb);
            if (lane == 0)
                *group_entry(p, n - p.sample0, blockIdx.x, g, blockIdx.z - b0) = make_float4(a, c, 0.f, 0.f);
        }
    }
    if (s.live && s.sub == 0) {
        // the pieces before this one have left their sums here
        float* dst = p.partial + ((size_t)blockIdx.y * p.slabs + blockIdx.x) * 2 * p.channels + s.c;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            dst[i] = p.sample0 ? dst[i] + run0[i] : run0[i];
            dst[p.channels + i] = p.sample0 ? dst[p.channels + i] + run1[i] : run1[i];
        }
    }
}

template <typename T, int V, int ACT>
__global__ void __launch_bounds__(kT, kSlabCtas) gn_slab_bwd(const __grid_constant__ GroupNormArgs p) {
    __shared__ float2 st[kMaxLocal];
    const SlabSlot s = slab_slot<V>(p);
    const size_t n = p.sample0 + blockIdx.y;
    int g0, ng;
    local_groups<V>(p, g0, ng);
    const int cg = p.channels / p.groups, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const float inv = 1.f / ((float)cg * (float)p.positions);
    for (int k = warp; k < ng; k += kT / 32) {
        int b0, nb;
        group_blocks<V>(p, g0 + k, b0, nb);
        float a = 0.f, c = 0.f;
        for (int t = lane; t < p.slabs * nb; t += 32) {
            const float4 u = *group_entry(p, blockIdx.y, t / nb, g0 + k, t % nb);
            a += u.x;
            c += u.y;
        }
        a = lane_sum<32>(a);
        c = lane_sum<32>(c);
        if (lane == 0) st[k] = make_float2(a * inv, c * inv);
    }
    __syncthreads();
    if (!s.live) return;
    const float2 ms = p.stats[n * p.groups + s.g], sums = st[s.g - g0];
    using E = Elem<V>;
    const Vals<V> w = affine_v<V>(p.w, p.w_f32, s.c, 1.f, true), b = affine_v<V>(p.b, p.w_f32, s.c, 0.f, true);
    const size_t base = n * p.positions * p.channels + s.c;
    for (int q0 = s.p0 + s.sub; q0 < s.p1; q0 += kPair * s.rows) {
        Pack<T, V> raw_x[kPair], raw_d[kPair];
#pragma unroll
        for (int e = 0; e < kPair; ++e) {
            const size_t at = base + (size_t)min(q0 + e * s.rows, s.p1 - 1) * p.channels;
            raw_x[e] = load_raw<T, V>(reinterpret_cast<const T*>(p.x) + at);
            raw_d[e] = load_raw<T, V>(reinterpret_cast<const T*>(p.dy) + at);
        }
#pragma unroll
        for (int e = 0; e < kPair; ++e) {
            const int q = q0 + e * s.rows;
            if (q >= s.p1) break;
            Vals<V> h, d;
            unpack<T, V>(h, raw_x[e]);
            unpack<T, V>(d, raw_d[e]);
#pragma unroll
            for (int i = 0; i < kN<V>; ++i) {
                const E x = op_mul(op_add(h.a[i], all<E>(-ms.x)), all<E>(ms.y));
                const E du = op_mul(d.a[i], act_slope<ACT>(op_fma(x, w.a[i], b.a[i])));
                d.a[i] = op_mul(all<E>(ms.y), op_fma(x, all<E>(-sums.y), op_fma(du, w.a[i], all<E>(-sums.x))));
            }
            store_v<T, V>(reinterpret_cast<T*>(p.dx) + base + (size_t)q * p.channels, d);
        }
    }
}

// dw, db: sums of the partial rows, 32 channels x 32 strides of rows per CTA, added in a fixed order
__global__ void __launch_bounds__(1024) gn_reduce(const float* part, long long rows, int channels, void* dw, void* db,
                                                  int w_f32) {
    __shared__ float red[32][33];
    const int lane = threadIdx.x & 31, c = blockIdx.x * 32 + lane, k = threadIdx.x >> 5;
    const float* src = part + (size_t)blockIdx.y * channels;
    float s = 0.f;
    if (c < channels) {
#pragma unroll 8
        for (long long r = k; r < rows; r += 32) s += src[(size_t)r * 2 * channels + c];
    }
    red[k][lane] = s;
    __syncthreads();
    void* dst = blockIdx.y == 0 ? dw : db;
    if (k != 0 || c >= channels || !dst) return;
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) t += red[i][lane];
    if (w_f32) reinterpret_cast<float*>(dst)[c] = t;
    else st_f(reinterpret_cast<__nv_bfloat16*>(dst) + c, t);
}

// ---------------------------------------------------------------------------------------- host
constexpr long long kPieceBytes = 72ll << 20;  // what a second pass still finds in the 126 MB of L2

template <typename T, int V, int NV, int LANES, int ACT>
cudaError_t rows_t(const GroupNormArgs& a, bool backward, cudaStream_t s) {
    const dim3 grid(a.slabs, (a.groups * LANES + kT - 1) / kT);
    if (backward) gn_rows_bwd<T, V, NV, LANES, ACT><<<grid, kT, 0, s>>>(a);
    else gn_rows_fwd<T, V, NV, LANES, ACT><<<grid, kT, 0, s>>>(a);
    return cudaGetLastError();
}
template <typename T, int V, int ACT>
cudaError_t rows_v(const GroupNormArgs& a, const GroupNormPlan& pl, bool backward, cudaStream_t s) {
    if constexpr (V > 1) {
        if (pl.nv == 4) return rows_t<T, V, 4, 32, ACT>(a, backward, s);
        if (pl.nv == 2) return rows_t<T, V, 2, 32, ACT>(a, backward, s);
    }
    switch (pl.lanes) {
        case 1: return rows_t<T, V, 1, 1, ACT>(a, backward, s);
        case 2: return rows_t<T, V, 1, 2, ACT>(a, backward, s);
        case 4: return rows_t<T, V, 1, 4, ACT>(a, backward, s);
        case 8: return rows_t<T, V, 1, 8, ACT>(a, backward, s);
        case 16: return rows_t<T, V, 1, 16, ACT>(a, backward, s);
        default: return rows_t<T, V, 1, 32, ACT>(a, backward, s);
    }
}
template <typename T, int V, int ACT>
cudaError_t slabs_v(GroupNormArgs a, const GroupNormPlan& pl, bool backward, cudaStream_t s) {
    a.span = pl.span;
    for (long long n0 = 0; n0 < a.samples; n0 += pl.piece) {
        const long long n = a.samples - n0 < pl.piece ? a.samples - n0 : pl.piece;
        const dim3 grid(a.slabs, (unsigned)n, pl.blocks);
        a.sample0 = n0;
        a.sample1 = n0 + n;
        if (backward) {
            const dim3 walk(a.slabs, (unsigned)(n < pl.walkers ? n : pl.walkers), pl.blocks);
            gn_slab_sums<T, V, ACT><<<walk, kT, 0, s>>>(a);
            gn_slab_bwd<T, V, ACT><<<grid, kT, 0, s>>>(a);
        } else {
            gn_slab_stats<T, V><<<grid, kT, 0, s>>>(a);
            gn_slab_fwd<T, V, ACT><<<grid, kT, 0, s>>>(a);
        }
    }
    return cudaGetLastError();
}
template <typename T, int V>
cudaError_t run_v(const GroupNormArgs& a, const GroupNormPlan& pl, bool backward, cudaStream_t s) {
    if (pl.rows) {
        if (a.act == kActSilu) return rows_v<T, V, kActSilu>(a, pl, backward, s);
        if (a.act == kActGelu) return rows_v<T, V, kActGelu>(a, pl, backward, s);
        return rows_v<T, V, kActNone>(a, pl, backward, s);
    }
    if (a.act == kActSilu) return slabs_v<T, V, kActSilu>(a, pl, backward, s);
    if (a.act == kActGelu) return slabs_v<T, V, kActGelu>(a, pl, backward, s);
    return slabs_v<T, V, kActNone>(a, pl, backward, s);
}

}  // namespace

// A pure function of the shape, so that the size query and the launch agree.
GroupNormPlan groupnorm_plan(int dtype, long long samples, int positions, int channels, int groups, bool backward) {
    GroupNormPlan pl{};
    const int cg = channels / groups, most = dtype == kF32 ? 4 : 8;
    // vectors of 16 bytes where a group holds whole ones, else of 2, else single channels
    pl.vec = cg % most == 0 ? most : cg % 2 == 0 ? 2 : 1;
    const int sm = sm_count();
    const int need = (cg + pl.vec - 1) / pl.vec;
    pl.lanes = 1;
    while (pl.lanes < need && pl.lanes < 32) pl.lanes *= 2;
    const long long row_slots = (long long)groups * pl.lanes, wide = (row_slots + kT - 1) / kT;
    // a row is at most as wide as the grid's second axis
    if (positions == 1 && cg <= pl.vec * 32 * (pl.vec > 1 ? 4 : 1) && wide <= 65535) {
        pl.rows = 1;
        pl.nv = need <= 32 ? 1 : need <= 64 ? 2 : 4;
        const long long at_once = row_slots >= kT ? 1 : kT / row_slots;
        // one wave of persistent CTAs, each with one row of partial sums
        const int per_sm = pl.nv > 1 ? (backward ? 1 : 2) : backward ? kRowCtasBwd : kRowCtasFwd;
        long long ctas = (long long)sm * per_sm / wide;
        const long long full = (samples + at_once - 1) / at_once;
        ctas = ctas < 1 ? 1 : ctas > full ? full : ctas;
        pl.slabs = (int)ctas;
        pl.blocks = (int)wide;
        pl.part_rows = ctas;
        return pl;
    }
    const int slots = channels / pl.vec, per = slots < kT ? slots : kT;
    pl.blocks = (slots + kT - 1) / kT;
    const int at_once = kT / per;
    // one wave of CTAs over the piece of samples that one launch covers, 8 positions a thread at least
    const long long bytes = (long long)positions * channels * (dtype == kF32 ? 4 : 2);
    long long n = kPieceBytes / (backward ? 2 * bytes : bytes);
    n = n < 1 ? 1 : n > samples ? samples : n;
    long long want = (long long)sm * kSlabCtas / (n * pl.blocks);
    const long long room = (positions + 8ll * at_once - 1) / (8ll * at_once);
    want = want < 1 ? 1 : want > room ? room : want;
    pl.slabs = (int)want;
    // channel blocks of kT vectors that a group touches at most
    const int block = kT * pl.vec;
    pl.span = block % cg == 0 ? 1 : (cg + block - 2) / block + 1;
    if (pl.span > pl.blocks) pl.span = pl.blocks;
    // the workspace holds one piece: neither its group sums nor the rows of partial sums grow with the samples
    const long long entries = want * groups * pl.span;
    const long long fit = kPieceBytes / (16 * entries);
    n = fit < 1 ? 1 : n > fit ? fit : n;
    pl.piece = n > 65535 ? 65535 : n;
    const long long walkers = (long long)sm * sum_ctas(pl.vec) / (want * pl.blocks);  // one wave shares the samples
    pl.walkers = (int)(walkers < 1 ? 1 : walkers > pl.piece ? pl.piece : walkers);
    pl.part_rows = pl.walkers * want;
    pl.group_floats = (size_t)pl.piece * entries * 4;
    return pl;
}

cudaError_t launch_groupnorm(const GroupNormArgs& args, int dtype, bool backward, cudaStream_t s) {
    GroupNormPlan pl = groupnorm_plan(dtype, args.samples, args.positions, args.channels, args.groups, backward);
    GroupNormArgs a = args;
    a.slabs = pl.slabs;
    cudaError_t e;
    if (dtype == kF32)
        e = pl.vec == 4 ? run_v<float, 4>(a, pl, backward, s)
                        : pl.vec == 2 ? run_v<float, 2>(a, pl, backward, s) : run_v<float, 1>(a, pl, backward, s);
    else
        e = pl.vec == 8 ? run_v<__nv_bfloat16, 8>(a, pl, backward, s)
                        : pl.vec == 2 ? run_v<__nv_bfloat16, 2>(a, pl, backward, s)
                                      : run_v<__nv_bfloat16, 1>(a, pl, backward, s);
    if (e != cudaSuccess || !backward || (!a.dw && !a.db)) return e;
    gn_reduce<<<dim3((a.channels + 31) / 32, 2), 1024, 0, s>>>(a.partial, pl.part_rows, a.channels, a.dw, a.db, a.w_f32);
    return cudaGetLastError();
}

}  // namespace prb
