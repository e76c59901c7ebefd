// Linear attention with a decay for each head on the tensor cores (bf16 inputs, head sizes that are
// multiples of 8 up to 128).  One CTA walks a segment of one head in chunks of 128 tokens:
//
//   P  = a b^T            (128 x 128 x da)   a, b from shared memory             -> TMEM, fp32
//   X  = (w^|i-j| P) c    (128 x dc x 128)   scores as a bf16 TMEM operand       -> TMEM
//   I  = a S              (128 x dc x da)    S as a bf16 shared-memory operand   -> TMEM
//   U  = (w^pos' b)^T c   (da x dc x 128)    decayed b^T as a TMEM operand       -> TMEM
//   out = X + w^pos I,   S = w^n S + U       S itself stays in fp32 registers
//
// Roles: warp 8 keeps a ring of (a, b, c) chunk tiles full with TMA; one thread of warp 9 issues the
// tcgen05.mma; warps 0-3 own a query row per thread (mask and decay of the scores, epilogue); warps
// 4-7 own a state row per thread (b^T decayed and moved to TMEM, S update); warp 10 stores the output
// tile with TMA out of the stage whose a and b it has replaced.
//
// b^T reaches TMEM through transposing ldmatrix loads: a fragment of 8 x 8 holds token pairs of one
// channel, which is what a 16x128b TMEM store wants, so a warp moves its 32 x 128 piece in some 750
// instructions (reading single bf16 values down the columns took 16,000 cycles per chunk).  The
// decay of a score off the diagonal 32 x 32 blocks is a product of a row and a column factor.
//
// Roundings: the scores and the state are rounded to bf16 once as operands, 2^-9 each, which is
// what the bf16 output loses anyway.  The decayed b^T is split into two bf16 halves (2^-17): the state
// it builds is returned in fp32 and may be read by thousands of later tokens.  The two halves cost
// a second pass of U's matrix product, and keep the tile of b itself untouched in shared memory.
//
// TMEM columns: scores 0-127 (fp32, then bf16 in place), I 128-255, U and then X 256-383, decayed b^T
// 384-511 (two halves).  U is read into registers before X overwrites it.
//
// A masked score is 0, and 0 x inf = NaN: a row whose X is not finite is summed again over the
// positions that it may see (row_scores / row_mix), so that nothing behind the mask can reach it.
//
// Every wait has a limit; a CTA whose wait runs out raises g_status, lets its copies and matrix
// products in flight end, frees its TMEM and leaves.
#include <cuda_bf16.h>

#include "linattn.cuh"
#include "tma.cuh"

namespace prb {

namespace {

constexpr int kC = 128;        // tokens per chunk
constexpr int kThreads = 352;  // 4 output warps, 4 state warps, TMA, MMA and store warp
constexpr uint32_t kPanel = kC * 128;  // bytes of a 128-token x 64-channel bf16 panel
constexpr uint32_t kWaitLimit = 1u << 22;

constexpr uint32_t kColP = 0, kColI = 128, kColX = 256, kColB = 384;

__device__ int g_status;

// ------------------------------------------------------------------------------- tcgen05 wrappers
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)acc)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)acc)
        : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(addr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}

__device__ __forceinline__ void tmem_st_16x128b_x2(uint32_t addr, uint32_t r0, uint32_t r1, uint32_t r2, uint32_t r3) {
    asm volatile("tcgen05.st.sync.aligned.16x128b.x2.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(r0), "r"(r1),
                 "r"(r2), "r"(r3)
                 : "memory");
}
// four 8 x 8 bf16 matrices, transposed; lane l gives the address of row l % 8 of matrix l / 8
__device__ __forceinline__ void ldmatrix_t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}

// Shared-memory operand in 128-byte-swizzled panels of 64 bf16 channels.  Read along the channels
// (K-major) only the stride between groups of 8 rows matters; read along the rows (MN-major) `lead`
// is the stride between panels.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lead) {
    return (uint64_t)((addr & 0x3ffff) >> 4) | ((uint64_t)(lead >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
           (1ull << 46) | (2ull << 61);
}
// bf16 x bf16 -> fp32, 128 rows, n columns; trans_b: B is MN-major
__device__ __forceinline__ constexpr uint32_t instr_desc(int n, bool trans_b) {
    return (1u << 4) | (1u << 7) | (1u << 10) | ((trans_b ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) |
           ((uint32_t)(kC >> 4) << 24);
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z,
                                            int w) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
        : "memory");
}
__device__ __forceinline__ void tma_store_4d(const CUtensorMap* map, uint32_t src, int x, int y, int z, int w) {
    asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4, %5}], [%1];" ::"l"(
                     reinterpret_cast<uint64_t>(map)),
                 "r"(src), "r"(x), "r"(y), "r"(z), "r"(w)
                 : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

struct TcParams {
    MixParams p;
    CUtensorMap map[3][4];  // [job][a, b, c, out]
    int units;              // heads of all jobs per state head
};

constexpr uint32_t kCtlBytes = 1536;

template <int DA, int DC, bool STATE_ONLY>
struct Layout {
    static constexpr uint32_t kA = STATE_ONLY ? 0 : DA / 64 * kPanel;
    static constexpr uint32_t kB = DA / 64 * kPanel;
    static constexpr uint32_t kCc = DC / 64 * kPanel;
    static constexpr uint32_t kStage = kA + kB + kCc;
    static constexpr uint32_t kS = STATE_ONLY ? 0 : DA * DC * 2;
    static constexpr int kStages = (int)((224 * 1024 - kS) / kStage) < 4 ? (int)((224 * 1024 - kS) / kStage) : 4;
    static constexpr uint32_t kOffS = kStages * kStage;
    static constexpr uint32_t kOffCtl = kOffS + kS;
    static constexpr uint32_t kBytes = kOffCtl + kCtlBytes + 1024;  // alignment slack
};

struct Control {
    uint64_t full[4], empty[4];
    uint64_t p_full, p_ready, b_ready, u_full, u_free, s_ready, o_full, x_free, staged, drain;
    uint32_t tmem;
    int dead;
    float pw[kC + 1];  // w^0 .. w^128
    alignas(8) float wb[kC];  // w^pos' of a full chunk, read in pairs
};
static_assert(sizeof(Control) <= kCtlBytes, "control block");

// false: the limit ran out, or another warp's did
__device__ __forceinline__ bool wait(Control& ct, uint64_t* bar, uint32_t parity) {
    for (uint32_t i = 0; i < kWaitLimit; ++i) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((i & 255) == 255 && *reinterpret_cast<volatile int*>(&ct.dead)) return false;
    }
    *reinterpret_cast<volatile int*>(&ct.dead) = 1;
    g_status = kErrChainTimeout;
    return false;
}

// for whole warps: all lanes leave together
__device__ __forceinline__ bool wait_warp(Control& ct, uint64_t* bar, uint32_t parity) {
    return __all_sync(0xffffffffu, wait(ct, bar, parity));
}

// The rows that hold something not finite read their operands again from global memory.
__device__ __forceinline__ const __nv_bfloat16* token(const HeadView& v, int row, long long t, int h) {
    return reinterpret_cast<const __nv_bfloat16*>(v.p) + row * v.sb + t * v.st + h * v.sh;
}
__device__ __forceinline__ void load8(const __nv_bfloat16* at, float (&v)[8]) {
    const uint4 u = *reinterpret_cast<const uint4*>(at);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}
// the scores of row i over the positions [j0, j1) that it may see, rounded as the operand is
__device__ __noinline__ void row_scores(const MixJob& jb, int row, long long t0, int head, int hb, int i, int j0,
                                        int j1, const float* pw, float* p) {
    const __nv_bfloat16* a = token(jb.a, row, t0 + i, head);
    for (int j = j0; j < j1; ++j) {
        const __nv_bfloat16* b = token(jb.b, row, t0 + j, hb);
        float s = 0.f, x[8], y[8];
        for (int d = 0; d < jb.da; d += 8) {
            load8(a + d, x);
            load8(b + d, y);
#pragma unroll
            for (int k = 0; k < 8; ++k) s = fmaf(x[k], y[k], s);
        }
        p[j] = __bfloat162float(__float2bfloat16_rn(s * (jb.p_scale * pw[j < i ? i - j : j - i])));
    }
}
__device__ __noinline__ void row_mix(const MixJob& jb, int row, long long t0, int hb, const float* p, int j0, int j1,
                                     int c0, float* out) {
    float acc[32] = {};
    for (int j = j0; j < j1; ++j) {
        const __nv_bfloat16* c = token(jb.c, row, t0 + j, hb) + c0;
#pragma unroll
        for (int k = 0; k < 32; k += 8) {
            if (c0 + k >= jb.dc) break;
            float v[8];
            load8(c + k, v);
#pragma unroll
            for (int q = 0; q < 8; ++q) acc[k + q] = fmaf(p[j], v[q], acc[k + q]);
        }
    }
#pragma unroll
    for (int k = 0; k < 32; ++k) out[k] = acc[k];
}

template <int DA, int DC, bool STATE_ONLY, bool GROUPED>
__global__ void __launch_bounds__(kThreads, 1) mix_tc_kernel(const __grid_constant__ TcParams tp) {
    using L = Layout<DA, DC, STATE_ONLY>;
    extern __shared__ unsigned char raw[];
    const uint32_t raw_at = smem_u32(raw), base = (raw_at + 1023) & ~1023u;
    unsigned char* smem = raw + (base - raw_at);
    Control& ct = *reinterpret_cast<Control*>(smem + L::kOffCtl);
    const MixParams& p = tp.p;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    // unit fastest: the jobs and heads that read the same tokens run side by side and share them in L2
    const int unit = blockIdx.x % tp.units, rest = blockIdx.x / tp.units;
    const int item = rest % p.map.n_items, hs = rest / p.map.n_items;
    int ji = 0, u = unit;
    for (; ji + 1 < p.n_jobs; ++ji) {
        const int n = p.job[ji].heads / p.state_heads;
        if (u < n) break;
        u -= n;
    }
    const MixJob& jb = p.job[ji];
    const int head = hs * (jb.heads / p.state_heads) + u;
    Seg seg;
    if (!locate(p.map, item, seg)) return;

    if (tid == 0) {
        for (int i = 0; i < L::kStages; ++i) {
            mbar_init(&ct.full[i], 1);
            mbar_init(&ct.empty[i], STATE_ONLY ? 5 : 6);
        }
        mbar_init(&ct.p_full, 1);
        mbar_init(&ct.p_ready, 4);
        mbar_init(&ct.b_ready, 4);
        mbar_init(&ct.u_full, 1);
        mbar_init(&ct.u_free, 4);
        mbar_init(&ct.s_ready, 4);
        mbar_init(&ct.o_full, 1);
        mbar_init(&ct.x_free, 4);
        mbar_init(&ct.staged, 4);
        mbar_init(&ct.drain, 1);
        ct.dead = 0;
        mbar_fence_init();
    }
    if (tid < kC + 1) {
        const float w = decay_pow(p.log_decay[hs], tid);
        ct.pw[tid] = w;
        if (jb.reverse) {
            if (tid > 0) ct.wb[tid - 1] = w;
        } else if (tid < kC) {
            ct.wb[kC - 1 - tid] = w;
        }
    }
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&ct.tmem))
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
        tc_fence_before();
    }
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = ct.tmem;

    const int n_chunk = (seg.len + kC - 1) / kC, share = GROUPED ? jb.share_b : 1, n_it = n_chunk * share;
    const int reverse = jb.reverse;
    auto chunk_off = [&](int it) {
        const int m = GROUPED ? it / share : it;
        return (reverse ? n_chunk - 1 - m : m) * kC;
    };
    const size_t sbase = ((size_t)item * p.state_heads + hs) * p.state_elems;

    if (warp == 8) {
        // ---- TMA
        if (lane == 0) {
            const CUtensorMap* ma = &tp.map[ji][0];
            const CUtensorMap* mb = &tp.map[ji][1];
            const CUtensorMap* mc = &tp.map[ji][2];
            int it = 0;
            for (; it < n_it; ++it) {
                const int st = it % L::kStages;
                if (it >= L::kStages && !wait(ct, &ct.empty[st], (it / L::kStages - 1) & 1)) break;
                const uint32_t at = base + st * L::kStage;
                const int t = seg.t0 + chunk_off(it), hb = share > 1 ? head * share + it % share : hs;
                mbar_expect_tx(&ct.full[st], L::kStage);
                // b first: the state warps start on it
                for (int q = 0; q < DA / 64; ++q)
                    tma_load_4d(at + L::kA + q * kPanel, mb, &ct.full[st], q * 64, hb, t, seg.row);
                if (!STATE_ONLY)
                    for (int q = 0; q < DA / 64; ++q)
                        tma_load_4d(at + q * kPanel, ma, &ct.full[st], q * 64, head, t, seg.row);
                for (int q = 0; q < DC / 64; ++q)
                    tma_load_4d(at + L::kA + L::kB + q * kPanel, mc, &ct.full[st], q * 64, hb, t, seg.row);
            }
            if (it < n_it) drain_ring(ct.full, L::kStages, it, kDrainLimit);
        }
    } else if (warp == 9) {
        // ---- MMA
        if (lane == 0) {
            constexpr uint32_t kScores = instr_desc(kC, false), kOut = instr_desc(DC, true);
            bool ok = true;
            for (int it = 0; it < n_it; ++it) {
                const int st = it % L::kStages, g = GROUPED ? it % share : 0;
                const uint32_t at = base + st * L::kStage, par = it & 1;
                const uint32_t sa = at, sb = at + L::kA, sc = at + L::kA + L::kB;
                if (!(ok = wait(ct, &ct.full[st], (it / L::kStages) & 1))) break;
                if (!STATE_ONLY) {
                    tc_fence_after();
#pragma unroll
                    for (int k = 0; k < DA / 16; ++k) {
                        const uint32_t off = (k >> 2) * kPanel + (k & 3) * 32;
                        mma_ss(tmem + kColP, smem_desc(sa + off, 16), smem_desc(sb + off, 16), kScores, k > 0);
                    }
                    tc_commit(&ct.p_full);
                    if (g == 0) {
                        const int m = GROUPED ? it / share : it;
                        if (!(ok = wait(ct, &ct.s_ready, m & 1))) break;
                        if (it > 0 && !(ok = wait(ct, &ct.x_free, (it - 1) & 1))) break;
                        tc_fence_after();
                        const uint32_t ss = base + L::kOffS;
#pragma unroll
                        for (int k = 0; k < DA / 16; ++k) {
                            const uint32_t off = (k >> 2) * kPanel + (k & 3) * 32;
                            mma_ss(tmem + kColI, smem_desc(sa + off, 16), smem_desc(ss + k * 2048, DA * 128), kOut,
                                   k > 0);
                        }
                    } else if (!(ok = wait(ct, &ct.x_free, (it - 1) & 1))) {
                        break;
                    }
                } else if (it > 0 && !(ok = wait(ct, &ct.u_free, (it - 1) & 1))) {
                    break;
                }
                if (!(ok = wait(ct, &ct.b_ready, par))) break;
                tc_fence_after();
#pragma unroll
                for (int k = 0; k < 2 * kC / 16; ++k)
                    mma_ts(tmem + kColX, tmem + kColB + k * 8, smem_desc(sc + (k & 7) * 2048, kPanel), kOut, k > 0);
                tc_commit(&ct.u_full);
                if (!STATE_ONLY) {
                    if (!(ok = wait(ct, &ct.p_ready, par)) || !(ok = wait(ct, &ct.u_free, par))) break;
                    tc_fence_after();
#pragma unroll
                    for (int k = 0; k < kC / 16; ++k)
                        mma_ts(tmem + kColX, tmem + kColP + (k >> 1) * 32 + (k & 1) * 8,
                               smem_desc(sc + k * 2048, kPanel), kOut, k > 0);
                    tc_commit(&ct.o_full);
                    // the next scores overwrite the operand that these products read
                    tc_commit(&ct.empty[st]);
                    if (!(ok = wait(ct, &ct.o_full, par))) break;
                } else {
                    tc_commit(&ct.empty[st]);
                }
            }
            tc_commit(&ct.drain);
            mbar_wait_bounded(&ct.drain, 0, kWaitLimit);
        }
    } else if (warp == 10) {
        // ---- store: whole chunks leave through TMA, ragged ones the output warps have written themselves
        if (!STATE_ONLY && lane == 0) {
            for (int it = 0; it < n_it; ++it) {
                const int st = it % L::kStages, off = chunk_off(it);
                if (!wait(ct, &ct.staged, it & 1)) break;
                if (seg.len - off >= kC && (!GROUPED || it % share == share - 1)) {
                    for (int q = 0; q < DC / 64; ++q)
                        if (q * 64 < jb.dc)
                            tma_store_4d(&tp.map[ji][3], base + st * L::kStage + q * kPanel, q * 64, head,
                                         seg.t0 + off, seg.row);
                    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                    asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                }
                mbar_arrive(&ct.empty[st]);
            }
            asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
        }
    } else if (warp >= 4) {
        // ---- state: thread r owns row r of S
        const int r = tid - 128;
        const uint32_t lanes = tmem + ((uint32_t)(warp & 3) << 21);  // lane 32 * (warp % 4) in bits 31-16
        const bool mine = (warp & 3) * 32 < DA;
        float S[DC];
#pragma unroll
        for (int c = 0; c < DC; ++c)
            S[c] = (!STATE_ONLY && jb.s_in && r < jb.da && c < jb.dc)
                       ? jb.s_in[sbase + (size_t)r * jb.s_row + (size_t)c * jb.s_col]
                       : 0.f;
        unsigned char* ss = smem + L::kOffS;
        auto publish = [&]() {
            if (mine) {
#pragma unroll
                for (int c = 0; c < DC; c += 8) {
                    uint4 v;
                    v.x = pack_bf16(S[c], S[c + 1]);
                    v.y = pack_bf16(S[c + 2], S[c + 3]);
                    v.z = pack_bf16(S[c + 4], S[c + 5]);
                    v.w = pack_bf16(S[c + 6], S[c + 7]);
                    *reinterpret_cast<uint4*>(ss + (c >> 6) * (DA * 128) + r * 128 +
                                              (((c & 63) * 2) ^ ((r & 7) << 4))) = v;
                }
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(&ct.s_ready);
        };
        if (!STATE_ONLY && n_it > 0) publish();
        for (int it = 0; it < n_it; ++it) {
            const int st = it % L::kStages, g = GROUPED ? it % share : 0;
            const int n = min(kC, seg.len - chunk_off(it));
            if (!wait_warp(ct, &ct.full[st], (it / L::kStages) & 1)) break;
            unsigned char* tile = smem + st * L::kStage + L::kA;
            if (n < kC) {
                // tokens of the next sequence behind the last one of this: no value of theirs may reach a
                // product, not even as 0 x inf
                unsigned char* tc = tile + L::kB;
                for (int i = n * 8 + r; i < kC * 8; i += 128)
#pragma unroll
                    for (int q = 0; q < DC / 64; ++q)
                        *reinterpret_cast<uint4*>(tc + q * kPanel + i * 16) = make_uint4(0, 0, 0, 0);
                fence_proxy_async();
            }
            if (mine) {
                const int d0 = (warp & 3) * 32, t2 = 2 * (lane & 3);
                const uint32_t from = smem_u32(tile) + (d0 >> 6) * kPanel + (lane & 7) * 128 +
                                      ((((d0 & 63) + 8 * (lane >> 3)) * 2) ^ ((lane & 7) << 4));
#pragma unroll 1
                for (int tg = 0; tg < kC / 8; tg += 2) {
                    uint32_t hi[2][4], lo[2][4];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        uint32_t f[4];
                        ldmatrix_t(from + (tg + e) * 1024, f);
                        const int t = (tg + e) * 8 + t2;
                        float2 w = *reinterpret_cast<const float2*>(&ct.wb[t]);
                        if (n < kC) {
                            w.x = t < n ? ct.pw[reverse ? t + 1 : n - 1 - t] : 0.f;
                            w.y = t + 1 < n ? ct.pw[reverse ? t + 2 : n - 2 - t] : 0.f;
                            const uint32_t keep = (t < n ? 0xffffu : 0u) | (t + 1 < n ? 0xffff0000u : 0u);
#pragma unroll
                            for (int q = 0; q < 4; ++q) f[q] &= keep;
                        }
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            const float2 v = __fmul2_rn(
                                make_float2(__uint_as_float(f[q] << 16), __uint_as_float(f[q] & 0xffff0000u)), w);
                            const uint32_t h = pack_bf16(v.x, v.y);
                            hi[e][q] = h;
                            lo[e][q] = pack_bf16(v.x - __uint_as_float(h << 16),
                                                 v.y - __uint_as_float(h & 0xffff0000u));
                        }
                    }
                    const uint32_t col = lanes + kColB + tg * 4, low16 = 16u << 16;
                    tmem_st_16x128b_x2(col, hi[0][0], hi[0][1], hi[1][0], hi[1][1]);
                    tmem_st_16x128b_x2(col + low16, hi[0][2], hi[0][3], hi[1][2], hi[1][3]);
                    tmem_st_16x128b_x2(col + 64, lo[0][0], lo[0][1], lo[1][0], lo[1][1]);
                    tmem_st_16x128b_x2(col + 64 + low16, lo[0][2], lo[0][3], lo[1][2], lo[1][3]);
                }
                tc_wait_st();
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&ct.b_ready);
                mbar_arrive(&ct.empty[st]);
            }
            if (!wait_warp(ct, &ct.u_full, it & 1)) break;
            tc_fence_after();
            const float wn = g == 0 ? ct.pw[n] : 1.f, us = jb.upd_scale;
            if (mine) {
#pragma unroll
                for (int c0 = 0; c0 < DC; c0 += 32) {
                    uint32_t v[32];
                    tmem_ld32(lanes + kColX + c0, v);
                    tc_wait_ld();
#pragma unroll
                    for (int k = 0; k < 32; ++k) S[c0 + k] = fmaf(wn, S[c0 + k], us * __uint_as_float(v[k]));
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&ct.u_free);
            // I = a S of this chunk has ended (committed before U): the operand may be replaced
            if (!STATE_ONLY && g == share - 1 && it + 1 < n_it) publish();
        }
        if (jb.s_out && head % jb.share_a == 0 && r < jb.da) {
#pragma unroll
            for (int c = 0; c < DC; ++c)
                if (c < jb.dc) jb.s_out[sbase + (size_t)r * jb.s_row + (size_t)c * jb.s_col] = S[c];
        }
    } else if (!STATE_ONLY) {
        // ---- output: thread i owns row i of the chunk
        const int i = tid;
        const uint32_t lanes = tmem + ((uint32_t)warp << 21);
        float acc[GROUPED ? DC : 1];
        __nv_bfloat16* out = reinterpret_cast<__nv_bfloat16*>(jb.out);
        // column factors of the blocks off the diagonal: forwards w^(31 - k), backwards w^k
        float2 colw[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            colw[k].x = jb.p_scale * ct.pw[reverse ? 2 * k : 31 - 2 * k];
            colw[k].y = jb.p_scale * ct.pw[reverse ? 2 * k + 1 : 30 - 2 * k];
        }
        for (int it = 0; it < n_it; ++it) {
            const int st = it % L::kStages, g = GROUPED ? it % share : 0;
            const int off = chunk_off(it), n = min(kC, seg.len - off);
            const uint32_t par = it & 1;
            if (!wait_warp(ct, &ct.p_full, par)) break;
            tc_fence_after();
#pragma unroll 1
            for (int jc = 0; jc < 4; ++jc) {
                uint32_t v[32], h[16];
                if (reverse ? jc < warp : jc > warp) {
#pragma unroll
                    for (int k = 0; k < 16; ++k) h[k] = 0u;
                } else {
                    tmem_ld32(lanes + kColP + jc * 32, v);
                    const float row = ct.pw[jc == warp ? 0 : reverse ? jc * 32 - i : i - jc * 32 - 31];
                    tc_wait_ld();
                    if (jc != warp) {
                        const float2 row2 = make_float2(row, row);
#pragma unroll
                        for (int k = 0; k < 16; ++k) {
                            const float2 f = __fmul2_rn(
                                make_float2(__uint_as_float(v[2 * k]), __uint_as_float(v[2 * k + 1])),
                                __fmul2_rn(colw[k], row2));
                            h[k] = pack_bf16(f.x, f.y);
                        }
                    } else {
                        // a masked score is replaced, not multiplied by 0: it may be inf or NaN
                        const float* pw = reverse ? ct.pw - lane : ct.pw + lane;
#pragma unroll
                        for (int k = 0; k < 32; k += 2) {
                            float f[2];
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                const bool in = reverse ? k + e >= lane : k + e <= lane;
                                f[e] = 0.f;
                                if (in)
                                    f[e] = __uint_as_float(v[k + e]) *
                                           (jb.p_scale * (reverse ? pw[k + e] : pw[-(k + e)]));
                            }
                            h[k >> 1] = pack_bf16(f[0], f[1]);
                        }
                    }
                    if (reverse && n < kC) {
#pragma unroll
                        for (int k = 0; k < 16; ++k) {
                            const int j = jc * 32 + 2 * k;
                            h[k] &= (j < n ? 0xffffu : 0u) | (j + 1 < n ? 0xffff0000u : 0u);
                        }
                    }
                }
                tmem_st16(lanes + kColP + jc * 32, h);
            }
            tc_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&ct.p_ready);
            if (!wait_warp(ct, &ct.o_full, par)) break;
            tc_fence_after();
            const float rw = i < n ? jb.row_scale * ct.pw[reverse ? n - 1 - i : i + 1] : 0.f;
            const float2 rw2 = make_float2(rw, rw);
            const bool whole = n == kC, final = g == share - 1;
            __nv_bfloat16* dst = out + (((size_t)seg.row * p.map.time + seg.t0 + off + i) * jb.heads + head) * jb.dc;
            unsigned char* tile = smem + st * L::kStage + i * 128;
            float again[kC];
            bool have = false;
#pragma unroll
            for (int c0 = 0; c0 < DC; c0 += 32) {
                uint32_t x[32], in[32];
                tmem_ld32(lanes + kColX + c0, x);
                if (g == 0) tmem_ld32(lanes + kColI + c0, in);
                tc_wait_ld();
                float2 o[16], bad = make_float2(0.f, 0.f);
                const float2 zero = make_float2(0.f, 0.f);
#pragma unroll
                for (int k = 0; k < 16; ++k) {
                    o[k] = make_float2(__uint_as_float(x[2 * k]), __uint_as_float(x[2 * k + 1]));
                    bad = __ffma2_rn(o[k], zero, bad);
                }
                if (!(bad.x + bad.y == 0.f) && i < n) {  // NaN: some o[k] is not finite
                    const int j0 = reverse ? i : 0, j1 = reverse ? n : i + 1;
                    const int hb = share > 1 ? head * share + g : hs;
                    if (!have) row_scores(jb, seg.row, seg.t0 + off, head, hb, i, j0, j1, ct.pw, again);
                    have = true;
                    float t[32];
                    row_mix(jb, seg.row, seg.t0 + off, hb, again, j0, j1, c0, t);
#pragma unroll
                    for (int k = 0; k < 16; ++k) o[k] = make_float2(t[2 * k], t[2 * k + 1]);
                }
#pragma unroll
                for (int k = 0; k < 16; ++k) {
                    if (g == 0)
                        o[k] = __ffma2_rn(rw2, make_float2(__uint_as_float(in[2 * k]), __uint_as_float(in[2 * k + 1])),
                                          o[k]);
                    if (GROUPED) {
                        if (g > 0) o[k] = __fadd2_rn(o[k], make_float2(acc[c0 + 2 * k], acc[c0 + 2 * k + 1]));
                        acc[c0 + 2 * k] = o[k].x;
                        acc[c0 + 2 * k + 1] = o[k].y;
                    }
                }
                if (!final) continue;
#pragma unroll
                for (int k = 0; k < 16; k += 4) {
                    uint4 w;
                    w.x = pack_bf16(o[k].x, o[k].y);
                    w.y = pack_bf16(o[k + 1].x, o[k + 1].y);
                    w.z = pack_bf16(o[k + 2].x, o[k + 2].y);
                    w.w = pack_bf16(o[k + 3].x, o[k + 3].y);
                    const int c = c0 + 2 * k;
                    if (whole)
                        *reinterpret_cast<uint4*>(tile + (c >> 6) * kPanel + (((c & 63) * 2) ^ ((i & 7) << 4))) = w;
                    else if (i < n && c < jb.dc)
                        *reinterpret_cast<uint4*>(dst + c) = w;
                }
            }
            tc_fence_before();
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&ct.x_free);
                mbar_arrive(&ct.staged);
            }
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 9) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
    }
}

typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                             const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                             CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

bool head_map(CUtensorMap* out, const HeadView& v, int d, int heads, int time, int rows) {
    const EncodeFn fn = reinterpret_cast<EncodeFn>(tensor_map_encoder());
    if (!fn) return false;
    const cuuint64_t dims[4] = {(cuuint64_t)d, (cuuint64_t)heads, (cuuint64_t)time, (cuuint64_t)rows};
    const cuuint64_t strides[3] = {(cuuint64_t)v.sh * 2, (cuuint64_t)v.st * 2, (cuuint64_t)v.sb * 2};
    const cuuint32_t box[4] = {64, 1, kC, 1}, one[4] = {1, 1, 1, 1};
    return fn(out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(v.p), dims, strides, box, one,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int DA, int DC, bool STATE_ONLY, bool GROUPED>
cudaError_t launch_g(const TcParams& tp, cudaStream_t s) {
    using L = Layout<DA, DC, STATE_ONLY>;
    auto* fn = mix_tc_kernel<DA, DC, STATE_ONLY, GROUPED>;
    const cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)L::kBytes);
    if (e != cudaSuccess) return e;
    const long long grid = (long long)tp.units * tp.p.map.n_items * tp.p.state_heads;
    if (grid > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
    fn<<<(unsigned)grid, kThreads, L::kBytes, s>>>(tp);
    return cudaGetLastError();
}
template <int DA, int DC>
cudaError_t launch_d(const TcParams& tp, bool state_only, bool grouped, cudaStream_t s) {
    if (state_only)
        return grouped ? launch_g<DA, DC, true, true>(tp, s) : launch_g<DA, DC, true, false>(tp, s);
    return grouped ? launch_g<DA, DC, false, true>(tp, s) : launch_g<DA, DC, false, false>(tp, s);
}
cudaError_t launch_set(const TcParams& tp, bool state_only, cudaStream_t s) {
    bool grouped = false;
    for (int j = 0; j < tp.p.n_jobs; ++j) grouped |= tp.p.job[j].share_b > 1;
    const bool a = tp.p.job[0].da > 64, c = tp.p.job[0].dc > 64;
    if (a) return c ? launch_d<128, 128>(tp, state_only, grouped, s) : launch_d<128, 64>(tp, state_only, grouped, s);
    return c ? launch_d<64, 128>(tp, state_only, grouped, s) : launch_d<64, 64>(tp, state_only, grouped, s);
}

}  // namespace

// TMA's rules on addresses and strides, 8-channel vectors in the epilogue, and the head sizes
bool mix_tc_usable(const MixParams& p, int dtype) {
    if (dtype != kBF16 || !tensor_map_encoder()) return false;
    for (int j = 0; j < p.n_jobs; ++j) {
        const MixJob& jb = p.job[j];
        if (jb.da % 8 || jb.dc % 8 || (reinterpret_cast<uintptr_t>(jb.out) & 15)) return false;
        for (const HeadView* v : {&jb.a, &jb.b, &jb.c}) {
            if (reinterpret_cast<uintptr_t>(v->p) & 15) return false;
            for (long long st : {v->sb, v->st, v->sh})
                if (st <= 0 || st % 8 || st >= (1ll << 38)) return false;
        }
    }
    return true;
}

cudaError_t launch_mix_tc(const MixParams& p, int rows, bool state_only, cudaStream_t s) {
    // the tensor-map encoder is a driver call: a thread that has made no runtime call of its own yet (a
    // fresh autograd worker) gets the device's context bound here
    int dev = 0;
    cudaError_t bound = cudaGetDevice(&dev);
    if (bound == cudaSuccess) bound = cudaSetDevice(dev);
    if (bound != cudaSuccess) return bound;
    // jobs of one tile shape share a launch (dq, dk and dv all do when dk and dv round up alike)
    bool left[3] = {false, false, false};
    for (int j = 0; j < p.n_jobs; ++j) left[j] = true;
    for (int j0 = 0; j0 < p.n_jobs; ++j0) {
        if (!left[j0]) continue;
        TcParams tp;
        tp.p = p;
        tp.p.n_jobs = 0;
        tp.units = 0;
        for (int j = j0; j < p.n_jobs; ++j) {
            const MixJob& jb = p.job[j];
            if (!left[j] || (jb.da > 64) != (p.job[j0].da > 64) || (jb.dc > 64) != (p.job[j0].dc > 64)) continue;
            left[j] = false;
            const int k = tp.p.n_jobs++;
            tp.p.job[k] = jb;
            tp.units += jb.heads / p.state_heads;
            const int hb = jb.share_b > 1 ? jb.heads * jb.share_b : p.state_heads;
            if (!head_map(&tp.map[k][0], jb.a, jb.da, jb.heads, p.map.time, rows) ||
                !head_map(&tp.map[k][1], jb.b, jb.da, hb, p.map.time, rows) ||
                !head_map(&tp.map[k][2], jb.c, jb.dc, hb, p.map.time, rows))
                return cudaErrorInvalidValue;
            const HeadView o{jb.out, (long long)p.map.time * jb.heads * jb.dc, (long long)jb.heads * jb.dc, jb.dc};
            if (!state_only && !head_map(&tp.map[k][3], o, jb.dc, jb.heads, p.map.time, rows))
                return cudaErrorInvalidValue;
        }
        const cudaError_t e = launch_set(tp, state_only, s);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

int linattn_status(int clear) {
    int v = 0;
    if (cudaMemcpyFromSymbol(&v, g_status, sizeof(int)) != cudaSuccess) return kErrLaunch;
    if (v && clear) {
        const int zero = 0;
        if (cudaMemcpyToSymbol(g_status, &zero, sizeof(int)) != cudaSuccess) return kErrLaunch;
    }
    return v;
}

}  // namespace prb
