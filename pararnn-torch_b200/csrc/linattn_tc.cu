// Linear attention with a decay for each head on the tensor cores (bf16 inputs, head sizes that are
// multiples of 8 up to 128).  One CTA walks a segment of one head in chunks of 128 tokens:
//
//   P = a b^T                 (128 x 128 x da)   a, b from shared memory             -> TMEM, fp32
//   X = a S                   (128 x dc x da)    S as a bf16 shared-memory operand   -> TMEM
//   X = w^pos X + (w^|i-j| P) c                  scores as a bf16 TMEM operand       -> TMEM
//   U = (w^pos' b)^T c        (da x dc x 128)    decayed b^T as a TMEM operand       -> TMEM
//   out = X,   S = w^n S + U                     S itself stays in fp32 registers
//
// With share_b > 1 (gradients of shared heads) a chunk is visited once per query head; X and U add up
// in TMEM and the epilogue and the state update run at the last visit.
//
// Roles: warps 0-3 own a state row per thread (b^T decayed and moved to TMEM, S update); warps 4-11 own
// half a query row per thread (mask and decay of the scores, row factor of X, epilogue); warp 12 keeps
// a ring of (a, b, c) tiles full with TMA; one thread of warp 13 issues the tcgen05.mma; warp 14
// stores the output tile with TMA out of the stage whose a and b it has replaced; warp 15 looks for
// inf and NaN in c.  The state rows take up to 128 registers a thread, so the warpgroups trade
// registers (setmaxnreg).
// The compiler still plans with the 128 registers of the launch: 8 of the 12 instances spill 40 - 112 bytes.
//
// Roundings: the scores and the state are rounded to bf16 once as operands, 2^-9 each, which is
// what the bf16 output loses anyway.  The decayed b^T is split into two bf16 parts (2^-17), since the state
// that it builds is read by thousands of later tokens, and into three (2^-24) where the state is returned
// in fp32 (MixJob::exact): two parts leave an error of 1.3e-6, three 3e-7.  With da = 128 the
// first two parts follow one another along K; with da = 64 they fill the two halves of the 128 TMEM
// lanes, so that the second costs no further matrix instructions: threads 64-127 then carry the
// state of the low parts, and S is the sum of the two.  The third part is one more piece behind them.
//
// b^T reaches TMEM through transposing ldmatrix loads: a fragment of 8 x 8 holds token pairs of one
// channel, which is what a 16x128b TMEM store wants.  With da = 128 it is made in two halves of 64 tokens, so
// that one half is written while the matrix unit reads the other.  The decay of a score off the diagonal
// 32 x 32 blocks is a product of a row and a column factor.
//
// With da = dc = 64 there is room for the scores and X twice (kTwice): the scores of visit i + 1 are made
// and converted while the matrix unit works on X of visit i.  With 128 channels the four
// regions fill all 512 columns.  The state warps publish S, read U and write b^T in program order, so
// one barrier (b_ready) tells the MMA thread all three; every further barrier would cost it 200 -
// 230 cycles a visit (read from clocks in the loop, which add to what they time).
//
// A masked score is 0, and 0 x inf = NaN: a chunk whose c holds an inf or a NaN skips the product with c
// on the tensor cores; its rows are summed over the positions that they may see (row_mix),
// so that nothing behind the mask can reach them.
//
// Measured: forward 16 x 4096, 8 heads of 64: 77 us, 16 x 2048, 8 heads of 128: 60 us, against 41 us of memory traffic
// at the copy rate for both; with backward 294 and 226 against 82 (its three jobs read 9 inputs where one
// pass would read 4).  A chunk takes 2.4 resp. 3.7 us (time over chunks, start-up included) where the copy rate
// would allow 1.3 resp. 2.6: the MMA warp's walk over the barriers, with the tensor pipe active for 22
// resp. 40 % of the cycles.  128 tokens per chunk because tcgen05 works on 128 rows;
// one CTA per SM because the TMEM regions and two to four stages of tiles fill one.
//
// Every wait has a limit; a CTA whose wait runs out sets the device's status word, lets its copies and matrix
// products in flight end, frees its TMEM and leaves.
#include <cuda_bf16.h>

#include <atomic>

#include "linattn.cuh"
#include "tma.cuh"

namespace prb {

namespace {

constexpr int kC = 128;        // tokens per chunk
constexpr int kThreads = 512;  // 4 state warps, 8 output warps, TMA, MMA, store and scan warp
constexpr uint32_t kPanel = kC * 128;  // bytes of a 128-token x 64-channel bf16 panel
constexpr uint32_t kWaitLimit = 1u << 22;

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

__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(addr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
        "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
        "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
// 16 lanes x 16 columns: pairs (r[2j], r[2j+1]) are the rows l / 4 and l / 4 + 8 of columns 4j ...
__device__ __forceinline__ void tmem_st_16x128b_x4(uint32_t addr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.16x128b.x4.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(addr),
                 "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
__device__ __forceinline__ void tmem_ld8(uint32_t addr, uint32_t (&r)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(addr));
}
__device__ __forceinline__ void tmem_st8(uint32_t addr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(addr), "r"(r[0]),
                 "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
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
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}
// registers per thread of the calling warpgroup, up or down from the 128 of the launch
template <int N>
__device__ __forceinline__ void set_regs() {
    if constexpr (N > 128) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
    else asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
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

__device__ __forceinline__ __nv_bfloat162 as_bf162(uint32_t x) { return *reinterpret_cast<__nv_bfloat162*>(&x); }
__device__ __forceinline__ uint32_t as_u32(__nv_bfloat162 x) { return *reinterpret_cast<uint32_t*>(&x); }

struct TcParams {
    MixParams p;
    CUtensorMap map[3][4];  // [job][a, b, c, out]
    int units;              // heads of all jobs per state head
    uint32_t wait_limit;    // polls after which a wait gives up
    int* status;            // word of the device in host memory
};

constexpr uint32_t kCtlBytes = 2048, kMaxSmem = 227 * 1024;

// ------------------------------------------------------------------------------ decayed b^T
// Weights of tokens 2 i and 2 i + 1 of a chunk of n tokens, 0 behind its end.
__device__ __forceinline__ float2 weight_f32(const float* pw, int i, int n, int reverse, float scale) {
    const int t = 2 * i;
    return make_float2(t < n ? scale * pw[reverse ? t + 1 : n - 1 - t] : 0.f,
                       t + 1 < n ? scale * pw[reverse ? t + 2 : n - 2 - t] : 0.f);
}
// the same as bf16 pairs: high and low parts
__device__ __forceinline__ uint2 weight_pair(const float* pw, int i, int n, int reverse, float scale) {
    const float2 w = weight_f32(pw, i, n, reverse, scale);
    const uint32_t h = pack_bf16(w.x, w.y);
    return make_uint2(h, pack_bf16(w.x - __uint_as_float(h << 16), w.y - __uint_as_float(h & 0xffff0000u)));
}
// Part 0, 1 or 2 of b w for a pair of tokens: high = rn(b wh), low = rn((b wh - high) + b wl), the bracket
// exact; third = rn(b w - high - low) with b w in fp32 and exact differences.
__device__ __forceinline__ uint32_t b_part(uint32_t b_bits, uint2 w, float2 wf, int kind) {
    const __nv_bfloat162 b = as_bf162(b_bits), wh = as_bf162(w.x), h = __hmul2_rn(b, wh);
    if (kind == 0) return as_u32(h);
    const __nv_bfloat162 l = __hfma2(b, as_bf162(w.y), __hfma2(b, wh, __hneg2(h)));
    if (kind == 1) return as_u32(l);
    const float2 x = __bfloat1622float2(b), hf = __bfloat1622float2(h), lf = __bfloat1622float2(l);
    return pack_bf16((x.x * wf.x - hf.x) - lf.x, (x.y * wf.y - hf.y) - lf.y);
}

template <int DA, int DC>
struct Layout {
    static constexpr uint32_t kA = DA / 64 * kPanel;
    static constexpr uint32_t kB = DA / 64 * kPanel;
    static constexpr uint32_t kCc = DC / 64 * kPanel;
    static constexpr uint32_t kStage = kA + kB + kCc;
    static constexpr uint32_t kS = 128 * DC * 2;  // 128 state rows (da = 64: high and low halves)
    static constexpr int kStages = (int)((224 * 1024 - kS) / kStage) < 4 ? (int)((224 * 1024 - kS) / kStage) : 4;
    static constexpr uint32_t kOffS = kStages * kStage;
    static constexpr uint32_t kOffCtl = kOffS + kS;
    static constexpr uint32_t kBytes = kOffCtl + kCtlBytes + 1024;  // alignment slack
    static_assert(kBytes <= kMaxSmem && kStages >= 2, "shared memory");
    // TMEM columns: scores (fp32, then bf16 in place), X, U, decayed b^T
    static constexpr bool kTwice = DA == 64 && DC == 64;
    static constexpr int kHalves = DA == 64 ? 1 : 2;  // pieces in which b^T is made
    static constexpr uint32_t kColP = 0, kColX = kTwice ? 256 : 128, kColU = kTwice ? 384 : 256,
                              kColB = kTwice ? 448 : 384;
};

struct Control {
    // one per stage: their producers may be several visits ahead of (or behind) the others
    uint64_t full[4], empty[4], scanned[4], staged[4];
    // one visit or chunk at a time
    uint64_t p_full[2], p_ready, b_ready[3], b_free[3], i_full, o_full, x_free, drain, group;
    uint32_t tmem;
    int dead;
    int dirty[4];
    float pw[kC + 1];              // w^0 .. w^128
    float wd[64];                  // scores on the diagonal: p_scale times the factor of key - query + 31
    alignas(8) uint2 wb[kC / 2];   // upd_scale w^pos' of a token pair: bf16 pairs, high and low parts
    alignas(16) float wc[32];      // p_scale times the column factors of the score blocks off the diagonal
};
static_assert(sizeof(Control) <= kCtlBytes, "control block");

// false: the limit ran out.  One compact loop: the roles' code shares the instruction cache, and every
// visit passes a dozen waits.  The roles stop one after the other, each at its own wait.
template <typename C>
__device__ __forceinline__ bool wait(C& ct, uint32_t limit, uint64_t* bar, uint32_t parity) {
    uint32_t left = limit;
#pragma unroll 1
    while (!mbar_try_wait(bar, parity))
        if (--left == 0) {
            ct.dead = 1;
            return false;
        }
    return true;
}
// for whole warps: all lanes leave together
template <typename C>
__device__ __forceinline__ bool wait_warp(C& ct, uint32_t limit, uint64_t* bar, uint32_t parity) {
    return __all_sync(0xffffffffu, wait(ct, limit, bar, parity));
}
// The four warps of a group meet inside their loop, which one of them may have left after a wait of its own
// that ran out: a barrier with the same limit in the place of bar.sync, which would wait for that warp for ever.
template <typename C>
__device__ __forceinline__ bool meet(C& ct, uint32_t limit, uint64_t* bar) {
    __syncwarp();
    int ok = 1;
    if ((threadIdx.x & 31) == 0) {
        uint64_t phase;
        asm volatile("mbarrier.arrive.shared::cta.b64 %0, [%1];" : "=l"(phase) : "r"(smem_u32(bar)) : "memory");
        uint32_t left = limit;
#pragma unroll 1
        do {
            asm volatile(
                "{\n\t.reg .pred p;\n\t"
                "mbarrier.try_wait.shared::cta.b64 p, [%1], %2;\n\t"
                "selp.u32 %0, 1, 0, p;\n\t}"
                : "=r"(ok)
                : "r"(smem_u32(bar)), "l"(phase)
                : "memory");
        } while (!ok && --left);
        if (!ok) ct.dead = 1;
    }
    ok = __shfl_sync(0xffffffffu, ok, 0);
    __syncwarp();
    return ok != 0;
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
// acc (8 channels from c0 of row i): the row's scores, rounded as the operand is, times c
__device__ __forceinline__ void row_mix(const MixJob& jb, int row, long long t0, int head, int hb, int i, int j0,
                                        int j1, int c0, const float* pw, float (&acc)[8]) {
    const __nv_bfloat16* a = token(jb.a, row, t0 + i, head);
#pragma unroll 1
    for (int j = j0; j < j1; ++j) {
        const __nv_bfloat16* b = token(jb.b, row, t0 + j, hb);
        float s = 0.f, y[8], z[8];
#pragma unroll 1
        for (int d = 0; d < jb.da; d += 8) {
            load8(a + d, y);
            load8(b + d, z);
#pragma unroll
            for (int q = 0; q < 8; ++q) s = fmaf(y[q], z[q], s);
        }
        s = __bfloat162float(__float2bfloat16_rn(s * (jb.p_scale * pw[j < i ? i - j : j - i])));
        load8(token(jb.c, row, t0 + j, hb) + c0, y);
#pragma unroll
        for (int q = 0; q < 8; ++q) acc[q] = fmaf(s, y[q], acc[q]);
    }
}

// EXACT: some job of the launch returns its state (the third part costs the others instruction cache)
template <int DA, int DC, bool EXACT>
__global__ void __launch_bounds__(kThreads, 1) mix_tc_kernel(const __grid_constant__ TcParams tp) {
    using L = Layout<DA, DC>;
    constexpr bool kSplit = DA == 64;  // low halves of b^T in lanes 64-127
    extern __shared__ unsigned char raw[];
    const uint32_t raw_at = smem_u32(raw), base = (raw_at + 1023) & ~1023u;
    unsigned char* smem = raw + (base - raw_at);
    Control& ct = *reinterpret_cast<Control*>(smem + L::kOffCtl);
    const MixParams& p = tp.p;
    const uint32_t limit = tp.wait_limit;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    // shares of the 512 x 128 registers of the launch: 128 S + 256 O + 128 M <= 65536
    constexpr int kRegS = DC == 64 ? 152 : 208, kRegO = DC == 64 ? 144 : 112, kRegM = 64;
    static_assert(128 * kRegS + 256 * kRegO + 128 * kRegM <= kThreads * 128, "register shares");

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
    const bool exact = EXACT && jb.exact;
    const int head = hs * (jb.heads / p.state_heads) + u;
    Seg seg;
    if (!locate(p.map, item, seg)) return;

    if (tid == 0) {
        for (int i = 0; i < L::kStages; ++i) {
            mbar_init(&ct.full[i], 1);
            mbar_init(&ct.empty[i], 2);
            mbar_init(&ct.scanned[i], 1);
            mbar_init(&ct.staged[i], 8);
        }
        mbar_init(&ct.p_ready, 8);
        mbar_init(&ct.p_full[0], 1);
        mbar_init(&ct.p_full[1], 1);
        for (int i = 0; i < 3; ++i) {
            mbar_init(&ct.b_ready[i], 4);
            mbar_init(&ct.b_free[i], 1);
        }
        mbar_init(&ct.i_full, 1);
        mbar_init(&ct.o_full, 1);
        mbar_init(&ct.x_free, 8);
        mbar_init(&ct.drain, 1);
        mbar_init(&ct.group, 4);
        ct.dead = 0;
        mbar_fence_init();
    }
    if (tid < kC + 1) {
        const float w = decay_pow(p.log_decay[hs], tid);
        ct.pw[tid] = w;
        // forwards w^(31 - j), backwards w^(j - 31); the other half lies behind the mask
        if (tid < 32) {
            ct.wd[jb.reverse ? 31 + tid : 31 - tid] = jb.p_scale * w;
            ct.wd[jb.reverse ? 31 - tid : 31 + tid] = jb.p_scale * w;
        }
        // forwards w^(31 - k), backwards w^k
        if (tid < 32) ct.wc[jb.reverse ? tid : 31 - tid] = jb.p_scale * w;
    }
    if (warp == 13) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&ct.tmem))
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
        tc_fence_before();
    }
    __syncthreads();
    tc_fence_after();
    constexpr uint32_t tmem = 0;  // all 512 columns are this CTA's: they start at 0

    const int n_chunk = (seg.len + kC - 1) / kC, share = jb.share_b, n_it = n_chunk * share;
    const int reverse = jb.reverse;
    const size_t sbase = ((size_t)item * p.state_heads + hs) * p.state_elems;
    // visit `it` = (chunk m of the walk, query head g of the group); advanced without divisions
    struct Visit {
        int m = 0, g = 0, st = 0;
        uint32_t lap = 0;  // parity of the ring
    };
    auto next = [&](Visit& v) {
        if (++v.st == L::kStages) v.st = 0, v.lap ^= 1;
        if (++v.g == share) v.g = 0, ++v.m;
    };
    // the scores of visit `it`: their TMEM region, their barrier and its parity
    constexpr bool kTwice = L::kTwice;
    auto p_buf = [&](int it) { return kTwice ? it & 1 : 0; };
    auto p_par = [&](int it) { return kTwice ? (it >> 1) & 1 : it & 1; };
    auto x_col = [&](const Visit& v) { return tmem + L::kColX + (kTwice ? (v.m & 1) * 64 : 0); };
    auto offset = [&](const Visit& v) { return (reverse ? n_chunk - 1 - v.m : v.m) * kC; };

    if (warp >= 12) set_regs<kRegM>();
    if (warp == 12) {
        // ---- TMA
        if (lane == 0) {
            const CUtensorMap* ma = &tp.map[ji][0];
            const CUtensorMap* mb = &tp.map[ji][1];
            const CUtensorMap* mc = &tp.map[ji][2];
            int it = 0;
            for (Visit v; it < n_it; ++it, next(v)) {
                if (it >= L::kStages && !wait(ct, limit, &ct.empty[v.st], v.lap ^ 1)) break;
                const uint32_t at = base + v.st * L::kStage;
                const int t = seg.t0 + offset(v), hb = share > 1 ? head * share + v.g : hs;
                uint64_t* full = &ct.full[v.st];
                mbar_expect_tx(full, L::kStage);
                // b first: the state warps start on it
                for (int q = 0; q < DA / 64; ++q)
                    tma_load_4d(at + L::kA + q * kPanel, mb, full, q * 64, hb, t, seg.row);
                for (int q = 0; q < DA / 64; ++q) tma_load_4d(at + q * kPanel, ma, full, q * 64, head, t, seg.row);
                for (int q = 0; q < DC / 64; ++q)
                    tma_load_4d(at + L::kA + L::kB + q * kPanel, mc, full, q * 64, hb, t, seg.row);
            }
            // also when another role gave up: no copy may land after the CTA has left
            drain_ring(ct.full, L::kStages, it, kDrainLimit);
        }
    } else if (warp == 13) {
        // ---- MMA: the whole warp walks and waits, so that addresses and descriptors stay in uniform registers;
        // one elected lane issues
        constexpr uint32_t kScores = instr_desc(kC, false), kOut = instr_desc(DC, true);
        // scores of visit it (stage v.st); false: a wait ran out
        auto scores = [&](int it, const Visit& v) {
            if (!wait_warp(ct, limit, &ct.full[v.st], v.lap)) return false;
            tc_fence_after();
            const uint32_t sa = base + v.st * L::kStage;
            const uint64_t da = smem_desc(sa, 16), db = smem_desc(sa + L::kA, 16);
            const uint32_t to = tmem + L::kColP + p_buf(it) * 128;
            if (elect_one()) {
#pragma unroll
                for (int k = 0; k < DA / 16; ++k) {
                    const uint64_t off = ((k >> 2) * kPanel + (k & 3) * 32) >> 4;
                    mma_ss(to, da + off, db + off, kScores, k > 0);
                }
                tc_commit(&ct.p_full[p_buf(it)]);
            }
            __syncwarp();
            return true;
        };
        Visit v, ahead;
        for (int it = kTwice ? -1 : 0; it < n_it; ++it) {
            const uint32_t par = it & 1, mpar = v.m & 1;
            if (kTwice) {
                // one visit ahead; the region is free when the product of visit it - 1 has ended
                if (it + 1 < n_it) {
                    if (it > 0 && !wait_warp(ct, limit, &ct.o_full, par ^ 1)) break;
                    if (!scores(it + 1, ahead)) break;
                    next(ahead);
                }
                if (it < 0) continue;
            } else {
                if (it > 0 && !wait_warp(ct, limit, &ct.o_full, par ^ 1)) break;
                if (!scores(it, v)) break;
            }
            const uint32_t sa = base + v.st * L::kStage;
            const uint64_t dcd = smem_desc(sa + L::kA + L::kB, kPanel);
            bool ok = true;
#pragma unroll
            for (int hf = 0; hf < L::kHalves; ++hf) {
                if (!(ok = wait_warp(ct, limit, &ct.b_ready[hf], par))) break;
                const bool first = hf == 0 && v.g == 0;
                // twice: p_ready of the last chunk told that the epilogue before it has read this X
                if (first && !kTwice && v.m > 0 && !(ok = wait_warp(ct, limit, &ct.x_free, mpar ^ 1))) break;
                tc_fence_after();
                if (elect_one()) {
                    if (first) {
                        const uint64_t da = smem_desc(sa, 16), ds = smem_desc(base + L::kOffS, 128 * 128);
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            const uint64_t off = kSplit ? (k & 3) * 32 >> 4 : ((k >> 2) * kPanel + (k & 3) * 32) >> 4;
                            mma_ss(x_col(v), da + off, ds + (k * 2048 >> 4), kOut, k > 0);
                        }
                        tc_commit(&ct.i_full);
                    }
#pragma unroll
                    for (int k = 0; k < 8 / L::kHalves; ++k) {
                        const uint64_t c = dcd + ((hf * 4 + k) * 2048 >> 4);
                        const uint32_t bt = tmem + L::kColB + hf * 32 + k * 8;
                        mma_ts(tmem + L::kColU, bt, c, kOut, (v.g > 0 && !exact) || hf > 0 || k > 0);
                        if (!kSplit) mma_ts(tmem + L::kColU, bt + 64, c, kOut, true);
                    }
                    tc_commit(&ct.b_free[hf]);
                }
                __syncwarp();
            }
            if (!ok) break;
            if (exact) {
                if (!wait_warp(ct, limit, &ct.b_ready[2], par)) break;
                tc_fence_after();
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        mma_ts(tmem + L::kColU, tmem + L::kColB + (kSplit || k < 4 ? k * 8 : 64 + (k - 4) * 8),
                               dcd + (k * 2048 >> 4), kOut, true);
                    tc_commit(&ct.b_free[2]);
                }
                __syncwarp();
            }
            if (!wait_warp(ct, limit, &ct.p_ready, par)) break;
            tc_fence_after();
            const bool skip = *reinterpret_cast<volatile int*>(&ct.dirty[v.st]) != 0;
            if (elect_one()) {
                if (!skip) {
                    const uint32_t from = tmem + L::kColP + p_buf(it) * 128;
#pragma unroll
                    for (int k = 0; k < kC / 16; ++k)
                        mma_ts(x_col(v), from + (k >> 1) * 32 + (k & 1) * 8, dcd + (k * 2048 >> 4), kOut, true);
                }
                tc_commit(&ct.o_full);
                tc_commit(&ct.empty[v.st]);
            }
            __syncwarp();
            next(v);
        }
        if (elect_one()) tc_commit(&ct.drain);
        __syncwarp();
        mbar_wait_bounded(&ct.drain, 0, kWaitLimit);
    } else if (warp == 14) {
        // ---- store: whole chunks leave through TMA, ragged ones the output warps have written themselves
        if (lane == 0) {
            Visit v;
            for (int it = 0; it < n_it; ++it, next(v)) {
                if (!wait(ct, limit, &ct.staged[v.st], v.lap)) break;
                const int off = offset(v);
                if (v.g == share - 1 && seg.len - off >= kC) {
                    for (int q = 0; q < DC / 64; ++q)
                        if (q * 64 < jb.dc)
                            tma_store_4d(&tp.map[ji][3], base + v.st * L::kStage + q * kPanel, q * 64, head,
                                         seg.t0 + off, seg.row);
                    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                    asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                }
                mbar_arrive(&ct.empty[v.st]);
            }
            asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
        }
    } else if (warp == 15) {
        // ---- scan of c
        Visit v;
        for (int it = 0; it < n_it; ++it, next(v)) {
            if (!wait_warp(ct, limit, &ct.full[v.st], v.lap)) break;
            const int rows = min(kC, seg.len - offset(v));
            const unsigned char* tc = smem + v.st * L::kStage + L::kA + L::kB;
            // 0 x inf and 0 x NaN are NaN
            __nv_bfloat162 zero = __float2bfloat162_rn(0.f), sum[4] = {zero, zero, zero, zero};
#pragma unroll 1
            for (int q = 0; q < DC / 64; ++q)
#pragma unroll 4
                for (int i = lane; i < rows * 8; i += 32) {
                    const uint4 x = *reinterpret_cast<const uint4*>(tc + q * kPanel + i * 16);
                    sum[0] = __hfma2(as_bf162(x.x), zero, sum[0]);
                    sum[1] = __hfma2(as_bf162(x.y), zero, sum[1]);
                    sum[2] = __hfma2(as_bf162(x.z), zero, sum[2]);
                    sum[3] = __hfma2(as_bf162(x.w), zero, sum[3]);
                }
            const float2 f = __bfloat1622float2(__hadd2(__hadd2(sum[0], sum[1]), __hadd2(sum[2], sum[3])));
            bool bad = !(f.x + f.y == 0.f);
            bad = __any_sync(0xffffffffu, bad);
            if (lane == 0) {
                ct.dirty[v.st] = bad;
                mbar_arrive(&ct.scanned[v.st]);
            }
        }
    } else if (warp < 4) {
        // ---- state: thread r owns row r of S (da = 64: row r - 64 of the low halves from thread 64 on)
        set_regs<kRegS>();
        const int r = tid;
        const uint32_t lanes = tmem + ((uint32_t)warp << 21);  // lane 32 * warp in bits 31-16
        float S[DC];
        {
            const bool given = jb.s_in && r < jb.da;
            const float* from = given ? jb.s_in + sbase + (size_t)r * jb.s_row : nullptr;
            const int n_col = given ? jb.dc : 0;
#pragma unroll
            for (int c = 0; c < DC; ++c) {
                S[c] = 0.f;
                if (c < n_col) S[c] = __ldg(from);
                from += jb.s_col;
            }
        }
        unsigned char* ss = smem + L::kOffS;
        // channels of this warp's fragments, and whether it makes the low halves
        const int d0 = (kSplit ? warp & 1 : warp) * 32;
        const bool low = kSplit && warp >= 2;
        const uint32_t from = base + L::kA + (d0 >> 6) * kPanel + (lane & 7) * 128 +
                              ((((d0 & 63) + 8 * (lane >> 3)) * 2) ^ ((lane & 7) << 4));
        bool ok = true;
        Visit v;
        // the table of the first chunk; no warp has passed a wait yet, so all four reach this barrier
        int table_n = min(kC, seg.len - offset(v));
        if (r < kC / 2) ct.wb[r] = weight_pair(ct.pw, r, table_n, reverse, jb.upd_scale);
        asm volatile("bar.sync 1, 128;" ::: "memory");
        for (int it = 0; it < n_it; ++it, next(v)) {
            const int n = min(kC, seg.len - offset(v));
            const uint32_t par = it & 1;
            if (v.g == 0) {
                // S enters the chunk; the product with the last chunk's operand ended before that chunk's U
#pragma unroll
                for (int c = 0; c < DC; c += 8) {
                    uint4 w;
                    w.x = pack_bf16(S[c], S[c + 1]);
                    w.y = pack_bf16(S[c + 2], S[c + 3]);
                    w.z = pack_bf16(S[c + 4], S[c + 5]);
                    w.w = pack_bf16(S[c + 6], S[c + 7]);
                    *reinterpret_cast<uint4*>(ss + (c >> 6) * (128 * 128) + r * 128 +
                                              (((c & 63) * 2) ^ ((r & 7) << 4))) = w;
                }
                fence_proxy_async();
            }
            if (!wait_warp(ct, limit, &ct.full[v.st], v.lap)) break;
            if (n < kC) {
                // tokens of the next sequence behind the last one of this: no value of theirs may reach a
                // product, not even as 0 x inf
                unsigned char* tb = smem + v.st * L::kStage + L::kA;
                for (int i = n * 8 + r; i < kC * 8; i += 128)
#pragma unroll
                    for (int q = 0; q < (DA + DC) / 64; ++q)
                        *reinterpret_cast<uint4*>(tb + q * kPanel + i * 16) = make_uint4(0, 0, 0, 0);
                fence_proxy_async();
            }
            // every warp reads all rows of its channels below: the zeroes of the other warps have to be there, in
            // each visit of a ragged chunk (share_b > 1 visits it once for each query head)
            if ((n < kC || n != table_n) && !meet(ct, limit, &ct.group)) break;
            if (n != table_n) {
                // the decays of this chunk length (all chunks but the ragged one have the same)
                if (r < kC / 2) ct.wb[r] = weight_pair(ct.pw, r, n, reverse, jb.upd_scale);
                if (!meet(ct, limit, &ct.group)) break;
                table_n = n;
            }
            const uint32_t tile = from + v.st * L::kStage;
#pragma unroll 1
            for (int hf = 0; hf < L::kHalves; ++hf) {
                // the third part of the last visit lay where the first piece goes
                if (it > 0 && !(ok = wait_warp(ct, limit, &ct.b_free[exact && hf == 0 ? 2 : hf], par ^ 1))) break;
                tc_fence_after();
                constexpr int kGroups = kC / 8 / L::kHalves;
#pragma unroll 1
                for (int tg = hf * kGroups; tg < hf * kGroups + kGroups; tg += 4) {
                    // registers of lanes 0-15 and 16-31 of the warp's 32 channels, token groups tg .. tg+3
                    const float2 none = make_float2(0.f, 0.f);
                    uint32_t f[4][4], hi[2][8], lo[2][8];
                    uint2 w[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        ldmatrix_t(tile + (tg + e) * 1024, f[e]);
                        w[e] = ct.wb[(tg + e) * 4 + (lane & 3)];
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e)
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            const int at = 2 * e + (q & 1);
                            hi[q >> 1][at] = b_part(f[e][q], w[e], none, 0);
                            if (!kSplit) lo[q >> 1][at] = b_part(f[e][q], w[e], none, 1);
                            else if (low) hi[q >> 1][at] = b_part(f[e][q], w[e], none, 1);
                        }
                    const uint32_t col = lanes + L::kColB + tg * 4, low16 = 16u << 16;
                    tmem_st_16x128b_x4(col, hi[0]);
                    tmem_st_16x128b_x4(col + low16, hi[1]);
                    if (!kSplit) {
                        tmem_st_16x128b_x4(col + 64, lo[0]);
                        tmem_st_16x128b_x4(col + 64 + low16, lo[1]);
                    }
                }
                tc_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&ct.b_ready[hf]);
            }
            if (!ok) break;
            if (exact) {
                // third part: b w in fp32 less the two parts, both differences exact
                if (!wait_warp(ct, limit, &ct.b_free[0], par)) break;
                tc_fence_after();
#pragma unroll 1
                for (int tg = 0; tg < kC / 8; tg += 4) {
                    uint32_t rest[2][8] = {};
                    if (!low) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            uint32_t f[4];
                            ldmatrix_t(tile + (tg + e) * 1024, f);
                            const uint2 w = ct.wb[(tg + e) * 4 + (lane & 3)];
                            const float2 wf = weight_f32(ct.pw, (tg + e) * 4 + (lane & 3), n, reverse, jb.upd_scale);
#pragma unroll
                            for (int q = 0; q < 4; ++q) rest[q >> 1][2 * e + (q & 1)] = b_part(f[q], w, wf, 2);
                        }
                    }
                    const uint32_t col = lanes + L::kColB + (kSplit || tg < 8 ? tg * 4 : 64 + (tg - 8) * 4);
                    tmem_st_16x128b_x4(col, rest[0]);
                    tmem_st_16x128b_x4(col + (16u << 16), rest[1]);
                }
                tc_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&ct.b_ready[2]);
            }
            // U of the chunk is complete (or of the visit: the tensor core truncates when it adds up, so an exact
            // state takes its visits one by one)
            if (v.g < share - 1 && !exact) continue;
            if (!wait_warp(ct, limit, &ct.b_free[exact ? 2 : L::kHalves - 1], par)) break;
            tc_fence_after();
            const float decay = v.g == 0 || !exact ? ct.pw[n] : 1.f;
            const float2 wn = make_float2(decay, decay);
#pragma unroll
            for (int c0 = 0; c0 < DC; c0 += 32) {
                uint32_t x[32];
                tmem_ld32(lanes + L::kColU + c0, x);
                tc_wait_ld();
#pragma unroll
                for (int k = 0; k < 32; k += 2) {
                    const float2 s2 = __ffma2_rn(wn, make_float2(S[c0 + k], S[c0 + k + 1]),
                                                 make_float2(__uint_as_float(x[k]), __uint_as_float(x[k + 1])));
                    S[c0 + k] = s2.x;
                    S[c0 + k + 1] = s2.y;
                }
            }
            tc_fence_before();
        }
        if (jb.s_out && head % jb.share_a == 0) {
            if (kSplit) {
                // S = high + low: the low rows pass through the operand's place, which no product reads any more
                float* ex = reinterpret_cast<float*>(ss);
                if (r >= 64) {
#pragma unroll
                    for (int c = 0; c < DC; ++c) ex[c * 64 + r - 64] = S[c];
                }
                asm volatile("bar.sync 1, 128;" ::: "memory");
                if (r < 64) {
#pragma unroll
                    for (int c = 0; c < DC; ++c) S[c] += ex[c * 64 + r];
                }
            }
            if (r < jb.da) {
                float* to = jb.s_out + sbase + (size_t)r * jb.s_row;
#pragma unroll
                for (int c = 0; c < DC; ++c) {
                    if (c < jb.dc) *to = S[c];
                    to += jb.s_col;
                }
            }
        }
    } else if (warp < 12) {
        // ---- output: threads i and i + 128 own row i of the chunk
        set_regs<kRegO>();
        const int i = (tid - 128) & 127, half = warp >= 8, w4 = warp & 3;
        const uint32_t lanes = tmem + ((uint32_t)w4 << 21);
        constexpr int kCols = DC / 2;  // output channels of a thread
        __nv_bfloat16* out = reinterpret_cast<__nv_bfloat16*>(jb.out);
        // scores of visit it: masked, decayed, to bf16 in place
        auto convert = [&](int it, const Visit& v) {
            const int n = min(kC, seg.len - offset(v));
            if (!wait_warp(ct, limit, &ct.p_full[p_buf(it)], p_par(it))) return false;
            tc_fence_after();
#pragma unroll 1
            for (int jc = half; jc < 4; jc += 2) {  // blocks alternate, so that both halves have work
                uint32_t x[32], h[16];
                if (reverse ? jc < w4 : jc > w4) {
#pragma unroll
                    for (int k = 0; k < 16; ++k) h[k] = 0u;
                } else {
                    tmem_ld32(lanes + L::kColP + p_buf(it) * 128 + jc * 32, x);
                    const float row = ct.pw[jc == w4 ? 0 : reverse ? jc * 32 - i : i - jc * 32 - 31];
                    tc_wait_ld();
                    if (jc != w4) {
                        const float2 row2 = make_float2(row, row);
#pragma unroll
                        for (int k = 0; k < 16; k += 2) {
                            const float4 w = *reinterpret_cast<const float4*>(&ct.wc[2 * k]);
                            const float2 f0 = __fmul2_rn(
                                make_float2(__uint_as_float(x[2 * k]), __uint_as_float(x[2 * k + 1])),
                                __fmul2_rn(make_float2(w.x, w.y), row2));
                            const float2 f1 = __fmul2_rn(
                                make_float2(__uint_as_float(x[2 * k + 2]), __uint_as_float(x[2 * k + 3])),
                                __fmul2_rn(make_float2(w.z, w.w), row2));
                            h[k] = pack_bf16(f0.x, f0.y);
                            h[k + 1] = pack_bf16(f1.x, f1.y);
                        }
                    } else {
                        // a masked score is replaced, not multiplied by 0: it may be inf or NaN
                        const float* wd = ct.wd + 31 - lane;
                        const uint32_t keep = reverse ? ~0u << lane : ~0u >> (31 - lane);
#pragma unroll
                        for (int k = 0; k < 32; k += 2) {
                            const float f0 = keep >> k & 1 ? __uint_as_float(x[k]) : 0.f;
                            const float f1 = keep >> (k + 1) & 1 ? __uint_as_float(x[k + 1]) : 0.f;
                            const float2 f = __fmul2_rn(make_float2(f0, f1), make_float2(wd[k], wd[k + 1]));
                            h[k >> 1] = pack_bf16(f.x, f.y);
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
                tmem_st16(lanes + L::kColP + p_buf(it) * 128 + jc * 32, h);
            }
            return true;
        };
        // X = w^pos X, and whatever keeps the matrix unit from adding the scores' product
        auto scale = [&](int it, const Visit& v) {
            const int off = offset(v), n = min(kC, seg.len - off);
            const uint32_t mpar = v.m & 1;
            if (!wait_warp(ct, limit, &ct.scanned[v.st], v.lap)) return false;
            const bool dirty = *reinterpret_cast<volatile int*>(&ct.dirty[v.st]) != 0;
            if (v.g == 0) {
                if (!wait_warp(ct, limit, &ct.i_full, mpar)) return false;
                tc_fence_after();
                const float rw = i < n ? jb.row_scale * ct.pw[reverse ? n - 1 - i : i + 1] : 0.f;
                const float2 rw2 = make_float2(rw, rw);
#pragma unroll
                for (int q = 0; q < kCols; q += 32) {
                    const uint32_t at = lanes + (x_col(v) - tmem) + half * kCols + q;
                    uint32_t x[32];
                    tmem_ld32(at, x);
                    tc_wait_ld();
#pragma unroll
                    for (int k = 0; k < 32; k += 2) {
                        const float2 f =
                            __fmul2_rn(make_float2(__uint_as_float(x[k]), __uint_as_float(x[k + 1])), rw2);
                        x[k] = __float_as_uint(f.x);
                        x[k + 1] = __float_as_uint(f.y);
                    }
                    tmem_st32(at, x);
                }
            }
            if (dirty) {
                // the products so far are in X, and the matrix unit leaves this one out
                tc_wait_st();
                tc_fence_after();
#pragma unroll 1
                for (int c0 = half * kCols; c0 < half * kCols + kCols; c0 += 8) {
                    uint32_t x[8];
                    tmem_ld8(lanes + (x_col(v) - tmem) + c0, x);
                    tc_wait_ld();
                    float acc[8] = {};
                    if (i < n && c0 < jb.dc)
                        row_mix(jb, seg.row, seg.t0 + off, head, share > 1 ? head * share + v.g : hs, i, reverse ? i : 0,
                                reverse ? n : i + 1, c0, ct.pw, acc);
                    __syncwarp();
#pragma unroll
                    for (int k = 0; k < 8; ++k) x[k] = __float_as_uint(__uint_as_float(x[k]) + acc[k]);
                    tmem_st8(lanes + (x_col(v) - tmem) + c0, x);
                }
            }
            tc_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&ct.p_ready);
                if (v.g < share - 1) mbar_arrive(&ct.staged[v.st]);
            }
            return true;
        };
        auto finish = [&](int it, const Visit& v) {
            // every visit waits: p_ready of the next one tells the MMA thread that this product has ended
            if (!wait_warp(ct, limit, &ct.o_full, it & 1)) return false;
            if (v.g < share - 1) return true;
            const int off = offset(v), n = min(kC, seg.len - off);
            tc_fence_after();
            const bool whole = n == kC;
            __nv_bfloat16* dst = out + (((size_t)seg.row * p.map.time + seg.t0 + off + i) * jb.heads + head) * jb.dc;
            unsigned char* tile = smem + v.st * L::kStage + i * 128;
#pragma unroll
            for (int q = 0; q < kCols; q += 32) {
                const int c0 = half * kCols + q;
                uint32_t x[32];
                tmem_ld32(lanes + (x_col(v) - tmem) + c0, x);
                tc_wait_ld();
#pragma unroll
                for (int k = 0; k < 32; k += 8) {
                    uint4 w;
                    w.x = pack_bf16(__uint_as_float(x[k]), __uint_as_float(x[k + 1]));
                    w.y = pack_bf16(__uint_as_float(x[k + 2]), __uint_as_float(x[k + 3]));
                    w.z = pack_bf16(__uint_as_float(x[k + 4]), __uint_as_float(x[k + 5]));
                    w.w = pack_bf16(__uint_as_float(x[k + 6]), __uint_as_float(x[k + 7]));
                    const int c = c0 + k;
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
                mbar_arrive(&ct.staged[v.st]);
            }
            return true;
        };
        Visit v, ahead;
        if (kTwice) {
            for (int it = -1; it < n_it; ++it) {
                if (it >= 0 && !scale(it, v)) break;
                if (it + 1 < n_it) {
                    if (!convert(it + 1, ahead)) break;
                    next(ahead);
                }
                if (it < 0) continue;
                if (!finish(it, v)) break;
                next(v);
            }
        } else {
            for (int it = 0; it < n_it; ++it, next(v))
                if (!convert(it, v) || !scale(it, v) || !finish(it, v)) break;
        }
        tc_wait_st();  // of a visit that was given up: nothing may be under way when TMEM is freed
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (tid == 0 && ct.dead) *(volatile int*)tp.status = kErrChainTimeout;
    if (warp == 13) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
    }
}

// The state-only sweep of a segment: U of every chunk and S = w^n S + U, from b and c alone.  Warps 4-7 and
// 8-11 take turns in making the parts of the decayed b^T (two visits in flight), warps 0-3 carry S,
// warp 12 loads, warp 13 issues the products.  TMEM columns: U 0-127, the parts of visit it from
// 128 + (it & 1) * 192 on: da = 128: high, low, third part; da = 64: high | low, third part | 0.
template <int DA, int DC>
struct StateLayout {
    static constexpr uint32_t kB = DA / 64 * kPanel, kStage = (DA + DC) / 64 * kPanel;
    static constexpr uint32_t kX = DA == 64 ? 64 * DC * 4 : 0;  // low rows on their way to the high ones
    static constexpr int kFit = (int)((kMaxSmem - kX - 4096 - 1024) / kStage), kStages = kFit < 4 ? kFit : 4;
    static constexpr uint32_t kOffX = kStages * kStage;
    static constexpr uint32_t kOffCtl = kOffX + kX;
    static constexpr uint32_t kBytes = kOffCtl + 4096 + 1024;
    static_assert(kBytes <= kMaxSmem && kStages >= 2, "shared memory");
};
struct StateControl {
    uint64_t full[4], empty[4], b_ready[2], b_free[2], u_free, drain, group[2];
    uint32_t tmem;
    int dead;
    float pw[kC + 1];
    // upd_scale w^pos' of a token pair, as bf16 pairs (high and low) and in fp32: a whole chunk, the ragged one
    alignas(16) uint2 wb[2][kC / 2];
    alignas(16) float2 wf[2][kC / 2];
};
static_assert(sizeof(StateControl) <= 4096, "control block");

template <int DA, int DC>
__global__ void __launch_bounds__(kThreads, 1) state_tc_kernel(const __grid_constant__ TcParams tp) {
    using L = StateLayout<DA, DC>;
    constexpr bool kSplit = DA == 64;
    extern __shared__ unsigned char raw[];
    const uint32_t raw_at = smem_u32(raw), base = (raw_at + 1023) & ~1023u;
    unsigned char* smem = raw + (base - raw_at);
    StateControl& ct = *reinterpret_cast<StateControl*>(smem + L::kOffCtl);
    const MixParams& p = tp.p;
    const MixJob& jb = p.job[0];
    const uint32_t limit = tp.wait_limit;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    constexpr int kRegS = DC == 64 ? 152 : 208, kRegO = DC == 64 ? 144 : 112, kRegM = 64;
    const int item = blockIdx.x % p.map.n_items, hs = blockIdx.x / p.map.n_items;
    Seg seg;
    if (!locate(p.map, item, seg)) return;
    if (tid == 0) {
        for (int i = 0; i < L::kStages; ++i) {
            mbar_init(&ct.full[i], 1);
            mbar_init(&ct.empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&ct.b_ready[i], 4);
            mbar_init(&ct.b_free[i], 1);
        }
        mbar_init(&ct.u_free, 4);
        mbar_init(&ct.drain, 1);
        mbar_init(&ct.group[0], 4);
        mbar_init(&ct.group[1], 4);
        ct.dead = 0;
        mbar_fence_init();
    }
    const int reverse = jb.reverse, exact = jb.exact;
    if (tid < kC + 1) ct.pw[tid] = decay_pow(p.log_decay[hs], tid);
    if (warp == 13) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&ct.tmem))
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
        tc_fence_before();
    }
    __syncthreads();
    tc_fence_after();
    constexpr uint32_t tmem = 0;  // all 512 columns are this CTA's: they start at 0
    const int n_chunk = (seg.len + kC - 1) / kC, share = jb.share_b, n_it = n_chunk * share;
    const size_t sbase = ((size_t)item * p.state_heads + hs) * p.state_elems;
    struct Visit {
        int m = 0, g = 0, st = 0;
        uint32_t lap = 0;
    };
    auto next = [&](Visit& v) {
        if (++v.st == L::kStages) v.st = 0, v.lap ^= 1;
        if (++v.g == share) v.g = 0, ++v.m;
    };
    auto offset = [&](const Visit& v) { return (reverse ? n_chunk - 1 - v.m : v.m) * kC; };

    if (warp >= 12) set_regs<kRegM>();
    if (warp == 12) {
        if (lane == 0) {
            int it = 0;
            for (Visit v; it < n_it; ++it, next(v)) {
                if (it >= L::kStages && !wait(ct, limit, &ct.empty[v.st], v.lap ^ 1)) break;
                const uint32_t at = base + v.st * L::kStage;
                const int t = seg.t0 + offset(v), hb = share > 1 ? hs * share + v.g : hs;
                mbar_expect_tx(&ct.full[v.st], L::kStage);
                for (int q = 0; q < DA / 64; ++q)
                    tma_load_4d(at + q * kPanel, &tp.map[0][1], &ct.full[v.st], q * 64, hb, t, seg.row);
                for (int q = 0; q < DC / 64; ++q)
                    tma_load_4d(at + L::kB + q * kPanel, &tp.map[0][2], &ct.full[v.st], q * 64, hb, t, seg.row);
            }
            drain_ring(ct.full, L::kStages, it, kDrainLimit);
        }
    } else if (warp == 13) {
        constexpr uint32_t kOut = instr_desc(DC, true);
        Visit v;
        for (int it = 0; it < n_it; ++it, next(v)) {
            const int buf = it & 1;
            if (!wait_warp(ct, limit, &ct.full[v.st], v.lap) || !wait_warp(ct, limit, &ct.b_ready[buf], (it >> 1) & 1)) break;
            if (it > 0 && !wait_warp(ct, limit, &ct.u_free, (it - 1) & 1)) break;
            tc_fence_after();
            const uint64_t c = smem_desc(base + v.st * L::kStage + L::kB, kPanel);
            const uint32_t bt = tmem + 128 + buf * 192;
            if (elect_one()) {
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    mma_ts(tmem, bt + k * 8, c + (k * 2048 >> 4), kOut, k > 0);
                    if (!kSplit) mma_ts(tmem, bt + 64 + k * 8, c + (k * 2048 >> 4), kOut, true);
                }
                if (exact) {
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        mma_ts(tmem, bt + (kSplit ? 64 : 128) + k * 8, c + (k * 2048 >> 4), kOut, true);
                }
                tc_commit(&ct.b_free[buf]);
                tc_commit(&ct.empty[v.st]);
            }
            __syncwarp();
        }
        if (elect_one()) tc_commit(&ct.drain);
        __syncwarp();
        mbar_wait_bounded(&ct.drain, 0, kWaitLimit);
    } else if (warp < 4) {
        // ---- state: thread r owns row r of S (da = 64: row r - 64 of the low parts from thread 64 on)
        set_regs<kRegS>();
        const int r = tid;
        const uint32_t lanes = tmem + ((uint32_t)warp << 21);
        float S[DC];
#pragma unroll
        for (int c = 0; c < DC; ++c) S[c] = 0.f;
        Visit v;
        for (int it = 0; it < n_it; ++it, next(v)) {
            if (!wait_warp(ct, limit, &ct.b_free[it & 1], (it >> 1) & 1)) break;
            tc_fence_after();
            const float decay = v.g == 0 ? ct.pw[min(kC, seg.len - offset(v))] : 1.f;
            const float2 wn = make_float2(decay, decay);
#pragma unroll
            for (int c0 = 0; c0 < DC; c0 += 32) {
                uint32_t x[32];
                tmem_ld32(lanes + c0, x);
                tc_wait_ld();
#pragma unroll
                for (int k = 0; k < 32; k += 2) {
                    const float2 s2 = __ffma2_rn(wn, make_float2(S[c0 + k], S[c0 + k + 1]),
                                                 make_float2(__uint_as_float(x[k]), __uint_as_float(x[k + 1])));
                    S[c0 + k] = s2.x;
                    S[c0 + k + 1] = s2.y;
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&ct.u_free);
        }
        if (kSplit) {
            float* ex = reinterpret_cast<float*>(smem + L::kOffX);
            if (r >= 64) {
#pragma unroll
                for (int c = 0; c < DC; ++c) ex[c * 64 + r - 64] = S[c];
            }
            asm volatile("bar.sync 1, 128;" ::: "memory");
            if (r < 64) {
#pragma unroll
                for (int c = 0; c < DC; ++c) S[c] += ex[c * 64 + r];
            }
        }
        if (r < jb.da) {
            float* to = jb.s_out + sbase + (size_t)r * jb.s_row;
#pragma unroll
            for (int c = 0; c < DC; ++c) {
                if (c < jb.dc) *to = S[c];
                to += jb.s_col;
            }
        }
    } else if (warp < 12) {
        // ---- parts of the decayed b^T: group 0 the even visits, group 1 the odd ones
        set_regs<kRegO>();
        const int group = warp >= 8, w4 = warp & 3, r = (tid - 128) & 127;
        const uint32_t lanes = tmem + ((uint32_t)w4 << 21);
        const int d0 = (kSplit ? w4 & 1 : w4) * 32;
        const bool low = kSplit && w4 >= 2;
        const uint32_t from = base + (d0 >> 6) * kPanel + (lane & 7) * 128 +
                              ((((d0 & 63) + 8 * (lane >> 3)) * 2) ^ ((lane & 7) << 4));
        // one table for each group to fill; no warp has passed a wait yet: all eight reach this barrier
        if (r < kC / 2) {
            const int n = group ? seg.len % kC : kC;
            ct.wb[group][r] = weight_pair(ct.pw, r, n, reverse, jb.upd_scale);
            ct.wf[group][r] = weight_f32(ct.pw, r, n, reverse, jb.upd_scale);
        }
        asm volatile("bar.sync 2, 256;" ::: "memory");
        Visit v;
        for (int it = 0; it < n_it; ++it, next(v)) {
            if ((it & 1) != group) continue;
            const int n = min(kC, seg.len - offset(v));
            if (!wait_warp(ct, limit, &ct.full[v.st], v.lap)) break;
            if (n < kC) {
                unsigned char* tb = smem + v.st * L::kStage;
                for (int i = n * 8 + r; i < kC * 8; i += 128)
#pragma unroll
                    for (int q = 0; q < (DA + DC) / 64; ++q)
                        *reinterpret_cast<uint4*>(tb + q * kPanel + i * 16) = make_uint4(0, 0, 0, 0);
                fence_proxy_async();
            }
            // as in mix_tc_kernel: no warp reads the rows before all of them are zero
            if (n < kC && !meet(ct, limit, &ct.group[group])) break;
            const int tab = n < kC;
            if (it > 1 && !wait_warp(ct, limit, &ct.b_free[group], ((it >> 1) - 1) & 1)) break;
            tc_fence_after();
            const uint32_t tile = from + v.st * L::kStage, bt = lanes + 128 + group * 192;
#pragma unroll 1
            for (int tg = 0; tg < kC / 8; tg += 4) {
                uint32_t f[4][4], part[2][8];
                uint2 w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    ldmatrix_t(tile + (tg + e) * 1024, f[e]);
                    w[e] = ct.wb[tab][(tg + e) * 4 + (lane & 3)];
                }
#pragma unroll
                for (int which = 0; which < 3; ++which) {
                    // da = 64: one store for high | low, one for the third part | 0
                    if ((kSplit && which == 1) || (which == 2 && !exact)) continue;
                    const int kind = kSplit && which == 0 && low ? 1 : which;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float2 wf = make_float2(0.f, 0.f);
                        if (which == 2) wf = ct.wf[tab][(tg + e) * 4 + (lane & 3)];
#pragma unroll
                        for (int q = 0; q < 4; ++q)
                            part[q >> 1][2 * e + (q & 1)] = kind == 2 && low ? 0u : b_part(f[e][q], w[e], wf, kind);
                    }
                    const uint32_t col = bt + (kSplit ? which / 2 : which) * 64 + tg * 4;
                    tmem_st_16x128b_x4(col, part[0]);
                    tmem_st_16x128b_x4(col + (16u << 16), part[1]);
                }
            }
            tc_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&ct.b_ready[group]);
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (tid == 0 && ct.dead) *(volatile int*)tp.status = kErrChainTimeout;
    if (warp == 13) {
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

// Status words of the devices, in page-locked host memory that kernels on any of them can write: every call can
// look at its device's word without a copy or a wait.
constexpr int kDevices = 64;
std::atomic<int*> g_status{nullptr};

int* status_word(int dev) {
    int* words = g_status.load(std::memory_order_acquire);
    if (!words) {
        // the first sweep may be one that is being captured
        cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
        cudaThreadExchangeStreamCaptureMode(&mode);
        void* p = nullptr;
        const cudaError_t e = cudaHostAlloc(&p, kDevices * sizeof(int), cudaHostAllocPortable | cudaHostAllocMapped);
        cudaThreadExchangeStreamCaptureMode(&mode);
        if (e != cudaSuccess) {
            cudaGetLastError();
            return nullptr;
        }
        for (int i = 0; i < kDevices; ++i) static_cast<int*>(p)[i] = 0;
        // of two threads that get here at once one leaves its 256 bytes unused
        if (g_status.compare_exchange_strong(words, static_cast<int*>(p))) words = static_cast<int*>(p);
    }
    return words + (dev & (kDevices - 1));
}

enum Sweep { kMix, kMixExact, kState };

template <int DA, int DC, Sweep SWEEP>
cudaError_t launch_d(const TcParams& tp, cudaStream_t s) {
    void (*fn)(TcParams) = SWEEP == kState ? state_tc_kernel<DA, DC> : mix_tc_kernel<DA, DC, SWEEP == kMixExact>;
    constexpr uint32_t bytes = SWEEP == kState ? StateLayout<DA, DC>::kBytes : Layout<DA, DC>::kBytes;
    // the attribute is a property of the function on the device: set once for each
    static bool ready[64] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64 || !ready[dev]) {
        e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
        if (e != cudaSuccess) return e;
        if (dev >= 0 && dev < 64) ready[dev] = true;
    }
    const long long grid = (long long)tp.units * tp.p.map.n_items * tp.p.state_heads;
    if (grid > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
    fn<<<(unsigned)grid, kThreads, bytes, s>>>(tp);
    return cudaGetLastError();
}
template <Sweep SWEEP>
cudaError_t launch_set(const TcParams& tp, cudaStream_t s) {
    const bool a = tp.p.job[0].da > 64, c = tp.p.job[0].dc > 64;
    if (a) return c ? launch_d<128, 128, SWEEP>(tp, s) : launch_d<128, 64, SWEEP>(tp, s);
    return c ? launch_d<64, 128, SWEEP>(tp, s) : launch_d<64, 64, SWEEP>(tp, s);
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
    int* const status = status_word(dev);
    if (!status) return cudaErrorMemoryAllocation;
    // jobs of one tile shape share a launch (dq, dk and dv all do when dk and dv round up alike)
    bool left[3] = {false, false, false};
    for (int j = 0; j < p.n_jobs; ++j) left[j] = true;
    for (int j0 = 0; j0 < p.n_jobs; ++j0) {
        if (!left[j0]) continue;
        TcParams tp;
        tp.p = p;
        tp.wait_limit = options().spin_limit < kWaitLimit ? options().spin_limit : kWaitLimit;
        tp.status = status;
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
        bool exact = false;
        for (int k = 0; k < tp.p.n_jobs; ++k) exact |= tp.p.job[k].exact != 0;
        const cudaError_t e = state_only ? launch_set<kState>(tp, s)
                              : exact    ? launch_set<kMixExact>(tp, s)
                                         : launch_set<kMix>(tp, s);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

int linattn_poll(int clear) {
    int* const words = g_status.load(std::memory_order_acquire);
    if (!words) return 0;  // no sweep has run
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return kErrLaunch;
    volatile int* word = words + (dev & (kDevices - 1));
    const int v = *word;
    if (v && clear) *word = 0;
    return v;
}

int linattn_status(int clear) {
    if (!g_status.load(std::memory_order_acquire)) return 0;
    if (cudaDeviceSynchronize() != cudaSuccess) return kErrLaunch;
    return linattn_poll(clear);
}

}  // namespace prb
