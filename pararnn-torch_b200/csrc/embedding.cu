// Embedding lookup with scaling, out_t = s W[id_t], and its gradient dW[v] = s sum_{id_t = v} dy_t.
//
// Both are HBM-bound copies.  The gradient is a sum by sorted tokens: a counting sort groups the
// positions of each id, every row of dW is written exactly once (zeros included) and each row's terms
// are added in fp32 in the order of their positions, so the result repeats bit for bit although
// the sort itself uses integer atomics:
//   count   rank_t = atomicAdd(count[id_t])                       (arrival order, arbitrary)
//   alloc   a block of ids takes room for its lists from one cursor; lists of more than kShort
//           positions also get a segment entry
//   place   pos[offset[id_t] + rank_t] = t
//   order   one CTA per long list: a bitmap over the positions puts them in order
//   sums    a warp per row sorts its <= 32 positions with shuffles and adds; a long list is cut into
//           pieces of max(128, sqrt n) positions, a CTA each, whose sums go to the workspace
//   join    the pieces of a long list, in order
// 32768 natural-text ids into 50304 x 768 bf16: 61 us, of which the one pass over the 127 MB takes 35 and the
// six short launches around it the rest; the lookup itself takes 12 us (8.4 TB/s, part of it from L2).
// Frequent tokens (a padding id, the head of a natural-text distribution) are thereby spread over
// many CTAs instead of queueing on one row.
#include "embedding.cuh"

namespace prb {

namespace {

constexpr int kT = 256;
constexpr int kShort = 32;
constexpr int kPiece = 128;  // 32768 natural-text ids, 768 channels: 61 us, 65 with pieces of 64
constexpr int kOrderT = 512;
constexpr int kWindowWords = 8192;  // 262144 positions per bitmap
constexpr int kFew = 2048, kFewRows = 4;  // tokens, and rows per CTA, up to which one launch does it all

struct LongSeg {
    int id, off, n, piece0, piece_len;
};

template <typename T, int V>
struct __align__(sizeof(T) * V) Vec {
    T v[V];
};

__device__ __forceinline__ long long id_at(const EmbedArgs& a, long long t) {
    return a.ids64 ? __ldg(reinterpret_cast<const long long*>(a.ids) + t)
                   : (long long)__ldg(reinterpret_cast<const int*>(a.ids) + t);
}

// a warp per token; ids outside the table give rows of zeros
template <typename T, int V>
__global__ void __launch_bounds__(kT) embed_fwd(const __grid_constant__ EmbedArgs a) {
    const long long t = (long long)blockIdx.x * (kT / 32) + (threadIdx.x >> 5);
    if (t >= a.tokens) return;
    const long long id = id_at(a, t);
    const bool in = id >= 0 && id < a.vocab;
    const int nv = a.channels / V;
    const Vec<T, V>* src = reinterpret_cast<const Vec<T, V>*>(a.table) + (in ? id : 0) * nv;
    Vec<T, V>* dst = reinterpret_cast<Vec<T, V>*>(a.out) + t * nv;
#pragma unroll 4
    for (int i = threadIdx.x & 31; i < nv; i += 32) {
        Vec<T, V> x;
        if (in) x = src[i];
#pragma unroll
        for (int k = 0; k < V; ++k) st_f(&x.v[k], in ? a.scale * static_cast<float>(x.v[k]) : 0.f);
        dst[i] = x;
    }
}

// one atomic for all lanes of a warp that hold the same id: frequent tokens queue 32 times less
__global__ void __launch_bounds__(kT) embed_count(const __grid_constant__ EmbedArgs a, int* counts, int* rank) {
    const long long t = (long long)blockIdx.x * kT + threadIdx.x;
    const long long id = t < a.tokens ? id_at(a, t) : -1;
    const bool in = id >= 0 && id < a.vocab;
    const int key = in ? (int)id : -1;
    const unsigned peers = __match_any_sync(0xffffffffu, key);
    const int lane = threadIdx.x & 31, leader = __ffs(peers) - 1;
    int first = 0;
    if (in && lane == leader) first = atomicAdd(counts + key, __popc(peers));
    first = __shfl_sync(0xffffffffu, first, leader);
    if (t < a.tokens) rank[t] = in ? first + __popc(peers & ((1u << lane) - 1)) : -1;
}

// counters: [0] list cursor, [1] long segments, [2] pieces
__global__ void __launch_bounds__(kT) embed_alloc(int vocab, const int* counts, int* offsets, int* counters,
                                                  LongSeg* segs) {
    __shared__ int warp_sum[kT / 32], base;
    const int v = blockIdx.x * kT + threadIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int n = v < vocab ? counts[v] : 0;
    int inc = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += u;
    }
    if (lane == 31) warp_sum[warp] = inc;
    __syncthreads();
    if (threadIdx.x == 0) {
        int s = 0;
        for (int i = 0; i < kT / 32; ++i) {
            const int u = warp_sum[i];
            warp_sum[i] = s;
            s += u;
        }
        base = s ? atomicAdd(counters, s) : 0;
    }
    __syncthreads();
    if (v >= vocab) return;
    const int off = base + warp_sum[warp] + inc - n;
    offsets[v] = off;
    if (n > kShort) {
        LongSeg sg;
        sg.id = v;
        sg.off = off;
        sg.n = n;
        sg.piece_len = max(kPiece, (int)ceilf(sqrtf((float)n)));
        sg.piece0 = atomicAdd(counters + 2, (n + sg.piece_len - 1) / sg.piece_len);
        segs[atomicAdd(counters + 1, 1)] = sg;
    }
}

__global__ void __launch_bounds__(kT) embed_place(const __grid_constant__ EmbedArgs a, const int* offsets,
                                                  const int* rank, int* pos) {
    const long long t = (long long)blockIdx.x * kT + threadIdx.x;
    if (t >= a.tokens) return;
    const int r = rank[t];
    if (r >= 0) pos[offsets[id_at(a, t)] + r] = (int)t;
}

__global__ void __launch_bounds__(kOrderT) embed_order(long long tokens, const int* counters, const LongSeg* segs,
                                                       const int* pos, int* sorted, int* piece_seg) {
    if ((int)blockIdx.x >= counters[1]) return;
    __shared__ unsigned bits[kWindowWords];
    __shared__ int warp_sum[kOrderT / 32];
    const LongSeg sg = segs[blockIdx.x];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int pieces = (sg.n + sg.piece_len - 1) / sg.piece_len;
    for (int i = threadIdx.x; i < pieces; i += kOrderT) piece_seg[sg.piece0 + i] = blockIdx.x;
    constexpr int kWindow = kWindowWords * 32;
    int done = 0;
    for (long long w0 = 0; w0 < tokens; w0 += kWindow) {
        const int words = (int)min((long long)kWindowWords, (tokens - w0 + 31) / 32);
        for (int i = threadIdx.x; i < words; i += kOrderT) bits[i] = 0u;
        __syncthreads();
        for (int i = threadIdx.x; i < sg.n; i += kOrderT) {
            const long long t = pos[sg.off + i] - w0;
            if (t >= 0 && t < kWindow) atomicOr(&bits[t >> 5], 1u << (t & 31));
        }
        __syncthreads();
        // each thread owns a run of words
        const int per = (words + kOrderT - 1) / kOrderT, i0 = min(words, (int)threadIdx.x * per),
                  i1 = min(words, i0 + per);
        int mine = 0;
        for (int i = i0; i < i1; ++i) mine += __popc(bits[i]);
        int inc = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += u;
        }
        if (lane == 31) warp_sum[warp] = inc;
        __syncthreads();
        int before = 0, total = 0;
        for (int i = 0; i < kOrderT / 32; ++i) {
            if (i < warp) before += warp_sum[i];
            total += warp_sum[i];
        }
        int at = sg.off + done + before + inc - mine;
        for (int i = i0; i < i1; ++i)
            for (unsigned b = bits[i]; b; b &= b - 1) sorted[at++] = (int)w0 + i * 32 + __ffs(b) - 1;
        done += total;
        __syncthreads();
    }
}

// One row of the gradient from a list of at most 32 positions held by the lanes of a warp.
template <typename T, int V>
__device__ __forceinline__ void row_sum(const EmbedArgs& a, int v, int n, int mine) {
    // odd-even merge of the lanes' positions (bitonic, ascending); empty lanes sort last
    const int lane = threadIdx.x & 31;
    if (n > 1) {
#pragma unroll
        for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
            for (int j = k >> 1; j > 0; j >>= 1) {
                const int other = __shfl_xor_sync(0xffffffffu, mine, j);
                const bool up = (lane & k) == 0, low = (lane & j) == 0;
                mine = (low == up) ? min(mine, other) : max(mine, other);
            }
    }
    const int nv = a.channels / V;
    const Vec<T, V>* src = reinterpret_cast<const Vec<T, V>*>(a.dy);
    Vec<T, V>* dst = reinterpret_cast<Vec<T, V>*>(a.out) + (size_t)v * nv;
    constexpr int kCols = V == 8 ? 3 : 4;  // vectors of a lane per turn: their loads are in flight together
    for (int i0 = 0; i0 < nv; i0 += 32 * kCols) {
        float acc[kCols][V] = {};
#pragma unroll 2
        for (int j = 0; j < n; ++j) {
            const Vec<T, V>* from = src + (long long)__shfl_sync(0xffffffffu, mine, j) * nv + i0 + lane;
            Vec<T, V> x[kCols];
#pragma unroll
            for (int c = 0; c < kCols; ++c)
                if (i0 + c * 32 + lane < nv) x[c] = from[c * 32];
#pragma unroll
            for (int c = 0; c < kCols; ++c)
                if (i0 + c * 32 + lane < nv) {
#pragma unroll
                    for (int k = 0; k < V; ++k) acc[c][k] += static_cast<float>(x[c].v[k]);
                }
        }
#pragma unroll
        for (int c = 0; c < kCols; ++c) {
            const int i = i0 + c * 32 + lane;
            if (i >= nv) break;
            Vec<T, V> y;
#pragma unroll
            for (int k = 0; k < V; ++k) st_f(&y.v[k], a.scale * acc[c][k]);
            dst[i] = y;
        }
    }
}

template <typename T, int V>
__global__ void __launch_bounds__(kT) embed_sums(const __grid_constant__ EmbedArgs a, const int* counters,
                                                 const int* counts, const int* offsets, const LongSeg* segs,
                                                 const int* pos, const int* sorted, const int* piece_seg,
                                                 float* partial, int piece_blocks) {
    if ((int)blockIdx.x < piece_blocks) {
        if ((int)blockIdx.x >= counters[2]) return;
        const LongSeg sg = segs[piece_seg[blockIdx.x]];
        const int k0 = (blockIdx.x - sg.piece0) * sg.piece_len, k1 = min(sg.n, k0 + sg.piece_len);
        const int nv = a.channels / V;
        const Vec<T, V>* src = reinterpret_cast<const Vec<T, V>*>(a.dy);
        for (int i = threadIdx.x; i < nv; i += kT) {
            float acc[V] = {};
#pragma unroll 8
            for (int k = k0; k < k1; ++k) {
                const Vec<T, V> x = src[(size_t)sorted[sg.off + k] * nv + i];
#pragma unroll
                for (int q = 0; q < V; ++q) acc[q] += static_cast<float>(x.v[q]);
            }
#pragma unroll
            for (int q = 0; q < V; ++q) partial[(size_t)blockIdx.x * a.channels + i * V + q] = acc[q];
        }
        return;
    }
    const int v = (blockIdx.x - piece_blocks) * (kT / 32) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (v >= a.vocab) return;
    const int n = counts[v];
    if (n > kShort) return;
    row_sum<T, V>(a, v, n, lane < n ? pos[offsets[v] + lane] : 0x7fffffff);
}

template <typename T>
__global__ void __launch_bounds__(kT) embed_join(const __grid_constant__ EmbedArgs a, const int* counters,
                                                 const LongSeg* segs, const float* partial) {
    const int longs = counters[1];
    for (int i = blockIdx.x; i < longs; i += gridDim.x) {
        const LongSeg sg = segs[i];
        const int pieces = (sg.n + sg.piece_len - 1) / sg.piece_len;
        T* dst = reinterpret_cast<T*>(a.out) + (size_t)sg.id * a.channels;
        for (int c = blockIdx.y * kT + threadIdx.x; c < a.channels; c += kT * gridDim.y) {
            float s = 0.f;
#pragma unroll 8
            for (int k = 0; k < pieces; ++k) s += partial[(size_t)(sg.piece0 + k) * a.channels + c];
            st_f(dst + c, a.scale * s);
        }
    }
}

// Few tokens: every CTA reads all ids, keeps those of its own rows in the order of their positions, and writes
// its rows.  One launch instead of seven short ones: 1531 tokens, 997 x 257 fp32 take 6.7 us against 17.5.
// With many rows per CTA the lists are walked too often (2048 tokens, 50304 rows: 39 us against 30).  A
// row with many positions is split over the CTA's warps in order, the parts are added in order.
template <typename T, int V>
__global__ void __launch_bounds__(kT) embed_few(const __grid_constant__ EmbedArgs a, int rows_per_cta) {
    __shared__ int list_pos[kFew], list_row[kFew], warp_sum[kT / 32];
    __shared__ int mine[kFew];
    __shared__ float part[kT / 32][32 * V];
    const int v0 = blockIdx.x * rows_per_cta, v1 = min(a.vocab, v0 + rows_per_cta);
    const int n_tok = (int)a.tokens, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    constexpr int kPer = kFew / kT;  // neighbouring tokens of a thread
    int row[kPer], cnt = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int t = threadIdx.x * kPer + i;
        const long long id = t < n_tok ? id_at(a, t) : -1;
        row[i] = id >= v0 && id < v1 ? (int)id : -1;
        cnt += row[i] >= 0;
    }
    int inc = cnt;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += u;
    }
    if (lane == 31) warp_sum[warp] = inc;
    __syncthreads();
    int at = inc - cnt, n_list = 0;
    for (int i = 0; i < kT / 32; ++i) {
        if (i < warp) at += warp_sum[i];
        n_list += warp_sum[i];
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i)
        if (row[i] >= 0) {
            list_row[at] = row[i];
            list_pos[at++] = threadIdx.x * kPer + i;
        }
    __syncthreads();
    const int nv = a.channels / V;
    const Vec<T, V>* src = reinterpret_cast<const Vec<T, V>*>(a.dy);
    for (int v = v0; v < v1; ++v) {
        // positions of the row, in order; every warp counts, one writes
        int n = 0;
        for (int i0 = 0; i0 < n_list; i0 += 32) {
            const bool hit = i0 + lane < n_list && list_row[i0 + lane] == v;
            const unsigned b = __ballot_sync(0xffffffffu, hit);
            if (hit && warp == 0) mine[n + __popc(b & ((1u << lane) - 1))] = list_pos[i0 + lane];
            n += __popc(b);
        }
        __syncthreads();
        Vec<T, V>* dst = reinterpret_cast<Vec<T, V>*>(a.out) + (size_t)v * nv;
        if (n <= kShort) {
            for (int i = threadIdx.x; i < nv; i += kT) {
                float acc[V] = {};
#pragma unroll 4
                for (int k = 0; k < n; ++k) {
                    const Vec<T, V> x = src[(size_t)mine[k] * nv + i];
#pragma unroll
                    for (int q = 0; q < V; ++q) acc[q] += static_cast<float>(x.v[q]);
                }
                Vec<T, V> y;
#pragma unroll
                for (int q = 0; q < V; ++q) st_f(&y.v[q], a.scale * acc[q]);
                dst[i] = y;
            }
        } else {
            const int k0 = n * warp / (kT / 32), k1 = n * (warp + 1) / (kT / 32);
            for (int i0 = 0; i0 < nv; i0 += 32) {
                float acc[V] = {};
                if (i0 + lane < nv) {
#pragma unroll 8
                    for (int k = k0; k < k1; ++k) {
                        const Vec<T, V> x = src[(size_t)mine[k] * nv + i0 + lane];
#pragma unroll
                        for (int q = 0; q < V; ++q) acc[q] += static_cast<float>(x.v[q]);
                    }
                }
#pragma unroll
                for (int q = 0; q < V; ++q) part[warp][lane * V + q] = acc[q];
                __syncthreads();
                if (warp == 0 && i0 + lane < nv) {
                    Vec<T, V> y;
#pragma unroll
                    for (int q = 0; q < V; ++q) {
                        float s = 0.f;
#pragma unroll
                        for (int w = 0; w < kT / 32; ++w) s += part[w][lane * V + q];
                        st_f(&y.v[q], a.scale * s);
                    }
                    dst[i0 + lane] = y;
                }
                __syncthreads();
            }
        }
        __syncthreads();
    }
}

template <typename T>
int vec_of(const EmbedArgs& a, const void* p, const void* q) {
    const uintptr_t bits = reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(q);
    const int most = 16 / (int)sizeof(T);
    if (a.channels % most == 0 && bits % 16 == 0) return most;
    if (a.channels % 2 == 0 && bits % (2 * sizeof(T)) == 0) return 2;
    return 1;
}

template <typename T, int V>
cudaError_t fwd_t(const EmbedArgs& a, cudaStream_t s) {
    embed_fwd<T, V><<<(unsigned)((a.tokens + kT / 32 - 1) / (kT / 32)), kT, 0, s>>>(a);
    return cudaGetLastError();
}

template <typename T, int V>
cudaError_t grad_t(const EmbedArgs& a, const EmbedPlan& pl, char* ws, cudaStream_t s) {
    const int ctas = 4 * sm_count(), per = (a.vocab + ctas - 1) / ctas;
    if (a.tokens <= kFew && per <= kFewRows) {
        embed_few<T, V><<<(a.vocab + per - 1) / per, kT, 0, s>>>(a, per);
        return cudaGetLastError();
    }
    int* counters = reinterpret_cast<int*>(ws + pl.counters);
    int* counts = reinterpret_cast<int*>(ws + pl.counts);
    int* offsets = reinterpret_cast<int*>(ws + pl.offsets);
    int* rank = reinterpret_cast<int*>(ws + pl.rank);
    int* pos = reinterpret_cast<int*>(ws + pl.pos);
    int* sorted = reinterpret_cast<int*>(ws + pl.sorted);
    LongSeg* segs = reinterpret_cast<LongSeg*>(ws + pl.segs);
    int* piece_seg = reinterpret_cast<int*>(ws + pl.piece_seg);
    float* partial = reinterpret_cast<float*>(ws + pl.partial);
    // counters and counts lie side by side
    cudaError_t e = cudaMemsetAsync(counters, 0, pl.counts - pl.counters + sizeof(int) * a.vocab, s);
    if (e != cudaSuccess) return e;
    const unsigned tb = (unsigned)((a.tokens + kT - 1) / kT);
    embed_count<<<tb, kT, 0, s>>>(a, counts, rank);
    embed_alloc<<<(a.vocab + kT - 1) / kT, kT, 0, s>>>(a.vocab, counts, offsets, counters, segs);
    embed_place<<<tb, kT, 0, s>>>(a, offsets, rank, pos);
    const int longs = (int)pl.max_segs, pieces = (int)pl.max_pieces;
    if (longs) embed_order<<<longs, kOrderT, 0, s>>>(a.tokens, counters, segs, pos, sorted, piece_seg);
    const int rows = (a.vocab + kT / 32 - 1) / (kT / 32);
    embed_sums<T, V><<<pieces + rows, kT, 0, s>>>(a, counters, counts, offsets, segs, pos, sorted, piece_seg, partial,
                                                  pieces);
    if (longs) {
        const int cols = (a.channels + kT - 1) / kT;
        const dim3 grid(longs < 2 * sm_count() ? longs : 2 * sm_count(), cols < 64 ? cols : 64);
        embed_join<T><<<grid, kT, 0, s>>>(a, counters, segs, partial);
    }
    return cudaGetLastError();
}

}  // namespace

EmbedPlan embedding_plan(long long tokens, int vocab, int channels) {
    EmbedPlan p{};
    size_t off = 0;
    auto take = [&](size_t bytes) {
        const size_t at = off;
        off = (off + bytes + 255) & ~size_t(255);
        return at;
    };
    // a long list has more than kShort positions, and ceil(n / piece length) pieces
    p.max_segs = tokens / (kShort + 1);
    p.max_pieces = p.max_segs ? tokens / kPiece + p.max_segs : 0;
    p.counters = take(256);
    p.counts = take(sizeof(int) * (size_t)vocab);
    p.offsets = take(sizeof(int) * (size_t)vocab);
    p.rank = take(sizeof(int) * (size_t)tokens);
    p.pos = take(sizeof(int) * (size_t)tokens);
    p.sorted = take(sizeof(int) * (size_t)tokens);
    p.segs = take(sizeof(LongSeg) * (size_t)p.max_segs);
    p.piece_seg = take(sizeof(int) * (size_t)p.max_pieces);
    p.partial = take(sizeof(float) * (size_t)p.max_pieces * channels);
    p.total = off;
    return p;
}

cudaError_t launch_embedding(const EmbedArgs& a, int dtype, cudaStream_t s) {
    if (dtype == kF32) {
        const int v = vec_of<float>(a, a.table, a.out);
        return v == 4 ? fwd_t<float, 4>(a, s) : v == 2 ? fwd_t<float, 2>(a, s) : fwd_t<float, 1>(a, s);
    }
    const int v = vec_of<__nv_bfloat16>(a, a.table, a.out);
    return v == 8 ? fwd_t<__nv_bfloat16, 8>(a, s)
                  : v == 2 ? fwd_t<__nv_bfloat16, 2>(a, s) : fwd_t<__nv_bfloat16, 1>(a, s);
}

cudaError_t launch_embedding_grad(const EmbedArgs& a, int dtype, void* ws, cudaStream_t s) {
    const EmbedPlan pl = embedding_plan(a.tokens, a.vocab, a.channels);
    char* w = reinterpret_cast<char*>(ws);
    if (dtype == kF32) {
        const int v = vec_of<float>(a, a.dy, a.out);
        return v == 4 ? grad_t<float, 4>(a, pl, w, s)
                      : v == 2 ? grad_t<float, 2>(a, pl, w, s) : grad_t<float, 1>(a, pl, w, s);
    }
    const int v = vec_of<__nv_bfloat16>(a, a.dy, a.out);
    return v == 8 ? grad_t<__nv_bfloat16, 8>(a, pl, w, s)
                  : v == 2 ? grad_t<__nv_bfloat16, 2>(a, pl, w, s) : grad_t<__nv_bfloat16, 1>(a, pl, w, s);
}

}  // namespace prb
