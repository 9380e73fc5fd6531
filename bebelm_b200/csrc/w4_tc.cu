// Products with 4-bit weights and group scales for many tokens, on the 5th-generation tensor cores.
//
//     y[t][n] = Σ_g s[n][g] · sx[t][g'] · Σ_{k in g} (c[n][k] - z[n][g]) · x[t][k]
//
// A = c - z (128 rows of weights, 16-bit floats, exact), B = activations (N tokens), D = the inner sum in f32
// (`tcgen05.mma kind::f16`, M 128). The scales stay out of the operands: a group's sum is read from TMEM and
// added, times its scale, to running f32 sums in registers, so nothing is rounded to 16 bits. Activations:
//   bf16: as they are (bf16 MMA), straight from the caller's rows by TMA.
//   int8: as f16 (exact).
//   f32: the sum of two f16 terms of x · 2^e, with e a token's, chosen so that its largest magnitude comes to
//        [2^14, 2^15). The terms hold x to 2^-24 of its value, half a step of f32 (and to 2^-39 of the token's
//        largest where the second term runs out of exponent). 2^-e is applied with the output.
// w4_terms_kernel writes the last two as [terms][tokens][kp].
//
// Tiles of 128 rows x N tokens, one CTA an SM that takes one tile after the other, 20 or 28 warps:
//   warps 0, 2   copies, a ring each, since they are held for different times: the activations' 128-byte-swizzled
//                tiles of 64 inputs (TMA, until their MMAs are done), the codes and zero points of 128 inputs (bulk copies:
//                they lie together, see w4.cu; until they are unpacked) and the scales (until they are applied).
//                With one ring for the three its depth bound everything: 5 stages against a stage's 6000 cycles.
//   warps 1, 3   issue the MMAs, A from TMEM, B from shared memory.
//   warps 4-11   unpack codes to A in TMEM, four buffers of 128 inputs, warps 4-7 the even and 8-11 the odd
//                ones (one set took longer than the MMAs): a warp's lanes hold (row g and g + 8, pairs 4 i + q), the
//                fragment of `tcgen05.st.16x128b`. A never passes through shared memory, whose bandwidth the
//                MMA needs for B.
//   warps 12-    read each group's sums, scale and add them; a thread has a row and 32 tokens (16 of 32). Sums go
//                over in two buffers of up to 128 columns: of few tokens' groups several at once, since a handing
//                over costs each side some 300 cycles.
// Where there are tiles for half of the SMs or less, a cluster's CTAs share a tile's inputs: each leaves its sums in
// its shared memory (where the activations' ring was) and adds up a share of the tokens, the parts in order.
// Bound: the tensor pipe for many tokens (a group of 128: 8 MMAs of N / 2 cycles each against ~N cycles of TMEM reads
// and N / 2 FMAs a thread). Measured: 2048 bf16 tokens x 8192 x 2048, groups of 128, 86.7 us: 793 TFLOP/s, 47 % of a
// library product's rate of 16-bit weights; 777 f32 tokens x 2048 x 2048, groups of 64, 24.5 us (two terms: 532 TFLOP/s
// of MMAs, a tile a CTA); 24 f32 tokens x 5003 x 2080, groups of 32, 11.3 us, three CTAs a tile.
// All waits are bounded (4 million polls, some 6 s); after one gives up the CTA waits (bounded) for its copies and MMAs
// in flight, reports kErrWaitTimeout and stores nothing more.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <atomic>
#include <cstdint>

#include "internal.h"

namespace bebelm {
namespace {

constexpr int kM = 128, kK = 128, kFixedWarps = 12;
constexpr int kConvert0 = 4, kEpi0 = kFixedWarps;  // first converter and first epilogue warp
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kColA = 256;          // four A buffers of 64 columns behind the accumulators (2 x 128 columns)
constexpr int kWaitLimit = 1 << 22;
constexpr int kRings = 225 * 1024;       // shared memory for the rings

struct TcArgs {
    W4View w;
    void* y;
    size_t tokens;
    const float* col_scale;   // [tokens]: one factor a token, or null
    const float* x_scales;    // [n_groups][tokens padded to 128]: a factor per group of inputs, or null
    size_t x_pitch, x_groups;
    int x_group, x_shift;     // inputs of a group, and their log2 (7 where a group holds 128 or more)
    int y_bf16, tiles, plane_rows;  // plane_rows: rows of B between the terms
    int split;                // CTAs of a cluster that share a tile's inputs; 1: a CTA takes tiles of its own
    int expire;               // test hook: the first CTA first waits, with a short limit, on a barrier nothing completes
    int* err;
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr) {  // 128B swizzle, K-major, SBO 1024, version 1
    return (uint64_t)((addr & 0x3FFFF) >> 4) | ((uint64_t)(16 >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
           (1ull << 46) | (2ull << 61);
}
// kind::f16, f32 accumulator, A and B both bf16 or both f16, K-major, M = 128
__host__ __device__ constexpr uint32_t instr_desc(int n, bool bf16) {
    return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kM >> 4) << 24);
}
__device__ __forceinline__ bool mbar_wait(uint32_t bar, unsigned parity, int limit = kWaitLimit) {
    for (int it = 0; it < limit; ++it) {
        uint32_t ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok)
            : "r"(bar), "r"(parity)
            : "memory");
        if (ok) return true;
    }
    return false;
}
// A try_wait takes about 280 cycles even for a phase that is complete, a test_wait 80; but polling with it slows the
// other warps down. So one test, then try_wait, which sleeps.
__device__ __forceinline__ bool mbar_ready_or_wait(uint32_t bar, unsigned parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok || mbar_wait(bar, parity);
}
__device__ __forceinline__ bool mbar_wait_warp(uint32_t bar, unsigned parity) {
    return __all_sync(0xffffffffu, mbar_ready_or_wait(bar, parity));
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
// One elected lane of a converged warp issues: with the whole warp in step, addresses and descriptors stay in
// uniform registers. (Issued by a lane in its own branch, an MMA took 130 cycles and a loop's end 250:
// 132 us against 102 for 2048 tokens x 8192 x 2048.)
__device__ __forceinline__ void commit(uint32_t bar) {
    asm volatile(
        "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar)
        : "memory");
}
__device__ __forceinline__ void expect_tx(uint32_t bar, uint32_t bytes) {
    asm volatile(
        "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
        "@e mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n\t}" ::"r"(bar), "r"(bytes)
        : "memory");
}
__device__ __forceinline__ void tma_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile(
        "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
        "@e cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];\n\t}" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void bulk(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile(
        "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
        "@e cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n\t}" ::"r"(dst), "l"(src),
        "r"(bytes), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\tsetp.ne.b32 p, %4, 0;\n\telect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
// 16 lanes x 64 columns: registers 2 i and 2 i + 1 of lane (g, q) go to column 4 i + q of lanes g and g + 8
__device__ __forceinline__ void tmem_st_tile(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.16x128b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
        "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
        "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
// 32 lanes x C columns (a multiple of 16); tmem_ld_wait() before the registers are used
template <int C>
__device__ __forceinline__ void tmem_ld(uint32_t taddr, uint32_t* r) {
#pragma unroll
    for (int i = 0; i < C; i += 16)
        asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
            "%15}, [%16];"
            : "=r"(r[i]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3]), "=r"(r[i + 4]), "=r"(r[i + 5]), "=r"(r[i + 6]),
              "=r"(r[i + 7]), "=r"(r[i + 8]), "=r"(r[i + 9]), "=r"(r[i + 10]), "=r"(r[i + 11]), "=r"(r[i + 12]),
              "=r"(r[i + 13]), "=r"(r[i + 14]), "=r"(r[i + 15])
            : "r"(taddr + i));
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// Word of 8 codes to 4 pairs of c - z, exactly (see w4.cu): 128 + c less 128 + z in bf16; in f16 1024 + c less
// 1024 + z, and 1/16 of 1024 + 16 c less 64 + z.
template <bool BF16>
__device__ __forceinline__ void pairs(uint32_t w, uint32_t za, uint32_t zb, uint32_t* o) {
    if constexpr (BF16) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t u = ((w >> (4 * j)) & 0x000f000fu) | 0x43004300u;
            const __nv_bfloat162 a = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&u), *reinterpret_cast<const __nv_bfloat162*>(&za));
            o[j] = *reinterpret_cast<const uint32_t*>(&a);
        }
    } else {
        const __half2 s16 = __float2half2_rn(0.0625f);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t v = i ? w >> 8 : w;
            const uint32_t lo = (v & 0x000f000fu) | 0x64006400u, hi = (v & 0x00f000f0u) | 0x64006400u;
            const __half2 a = __hsub2(*reinterpret_cast<const __half2*>(&lo), *reinterpret_cast<const __half2*>(&za));
            const __half2 b = __hfma2(*reinterpret_cast<const __half2*>(&hi), s16, __hneg2(*reinterpret_cast<const __half2*>(&zb)));
            o[2 * i] = *reinterpret_cast<const uint32_t*>(&a);
            o[2 * i + 1] = *reinterpret_cast<const uint32_t*>(&b);
        }
    }
}
// the pairs to take off for zero point z
template <bool BF16>
__device__ __forceinline__ void zero_pairs(uint32_t z, uint32_t& za, uint32_t& zb) {
    za = (BF16 ? 0x43004300u : 0x64006400u) + z * 0x10001u;
    if constexpr (!BF16) {
        const __half2 h = __half2half2(__ushort2half_rn((unsigned short)(64 + z)));
        zb = *reinterpret_cast<const uint32_t*>(&h);
    }
}

__device__ __forceinline__ float scale_of(uint32_t h, int bf16) {
    if (bf16) return __uint_as_float(h << 16);
    __half_raw r;
    r.x = (unsigned short)h;
    return __half2float(__half(r));
}

// two f32 operations in one instruction
__device__ __forceinline__ uint64_t pack2(uint32_t lo, uint32_t hi) {
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "r"(lo), "r"(hi));
    return v;
}
__device__ __forceinline__ void fma2(uint64_t& acc, uint64_t x, uint64_t y) {
    asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(acc) : "l"(x), "l"(y));
}
__device__ __forceinline__ uint64_t mul2(uint64_t x, uint64_t y) {
    uint64_t v;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(x), "l"(y));
    return v;
}
__device__ __forceinline__ float half_of(uint64_t v, int i) { return __uint_as_float((uint32_t)(i ? v >> 32 : v)); }

__device__ __forceinline__ void store(const TcArgs& a, size_t t, size_t r, float v) {
    if (a.col_scale) v *= __ldg(a.col_scale + t);
    if (a.y_bf16)
        static_cast<__nv_bfloat16*>(a.y)[t * a.w.n_out + r] = __float2bfloat16_rn(v);
    else
        static_cast<float*>(a.y)[t * a.w.n_out + r] = v;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// a word of CTA `rank`'s shared memory, at this CTA's address of it
__device__ __forceinline__ int ld_cluster(uint32_t addr, int rank) {
    int v;
    asm volatile(
        "{\n\t.reg .u32 p;\n\tmapa.shared::cluster.u32 p, %1, %2;\n\tld.shared::cluster.s32 %0, [p];\n\t}"
        : "=r"(v)
        : "r"(addr), "r"(rank)
        : "memory");
    return v;
}

template <int N, int TERMS, bool BF16>
struct Lay {
    static constexpr int kEpiWarps = N == 128 ? 16 : 8, kThreads = 32 * (kFixedWarps + kEpiWarps);
    static constexpr int kAtom = N * 128;                  // N tokens x 64 inputs
    static constexpr int kB = TERMS * kAtom;               // a stage: 64 inputs
    static constexpr int kW = 8192 + 512, kSW = 6;         // codes and zero points (<= 512 bytes) of 128 inputs
    static constexpr int kXs = 1024;                       // scales <= 1024 bytes, then the activations' (up to 4 x N)
    static constexpr int kS = kXs + (TERMS == 1 && !BF16 ? 4 * N * 4 : 0), kSS = 8;
    static constexpr int kOffW = 0, kOffS = kSW * kW, kOffB = (kOffS + kSS * kS + 1023) / 1024 * 1024;
    static constexpr int kSB = (kRings - kOffB) / kB < 12 ? (kRings - kOffB) / kB : 12;
    static constexpr int kSmem = kOffB + kSB * kB + 1024;
    static constexpr int kBars = 2 * (kSB + kSW + kSS) + 15;
    static_assert(kSB >= 4, "ring");  // 4 stages also hold a part's sums, N x 128 floats
};

// FB: blocks of 32 inputs whose sum is scaled together. SPLIT: the CTAs of a cluster share a tile's inputs.
template <int N, int TERMS, bool BF16, int FB, bool SPLIT>
__global__ void __launch_bounds__(Lay<N, TERMS, BF16>::kThreads, 1) w4_tc_kernel(const __grid_constant__ CUtensorMap tm_x, TcArgs a) {
    using L = Lay<N, TERMS, BF16>;
    constexpr int SB = L::kSB, SW = L::kSW, SS = L::kSS;  // ring stages
    // sums a chunk of 128 inputs, sums handed over at once, times a chunk that this happens
    constexpr int F = 4 / FB, U = F < 128 / N ? F : 128 / N, H = F / U, kIssuers = H == 1 ? 2 : 1;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* sm = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t sb = smem_u32(sm);
    __shared__ uint64_t s_bar[L::kBars];
    __shared__ uint32_t s_tmem;
    __shared__ int s_fail;
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const int chunks = (int)a.w.chunks, pc = a.w.per_chunk, row_blocks = (int)(a.w.tile_rows / 8);
    // this CTA's tiles, and its part [c_lo, c_hi) of their chunks of 128 inputs
    const int split = SPLIT ? a.split : 1, rank = SPLIT ? (int)blockIdx.x % split : 0;
    const int tile0 = SPLIT ? (int)blockIdx.x / split : (int)blockIdx.x, tile_step = SPLIT ? a.tiles : (int)gridDim.x;
    const int c_lo = SPLIT ? chunks * rank / split : 0, c_hi = SPLIT ? chunks * (rank + 1) / split : chunks;
    const int n_chunks = (a.tiles - tile0 + tile_step - 1) / tile_step * (c_hi - c_lo);
    const uint32_t bars = smem_u32(s_bar);
    auto b_full = [&](int i) { return bars + 8 * i; };
    auto b_empty = [&](int i) { return bars + 8 * (SB + i); };
    auto w_full = [&](int i) { return bars + 8 * (2 * SB + i); };
    auto w_empty = [&](int i) { return bars + 8 * (2 * SB + SW + i); };
    auto s_full = [&](int i) { return bars + 8 * (2 * (SB + SW) + i); };
    auto s_empty = [&](int i) { return bars + 8 * (2 * (SB + SW) + SS + i); };
    constexpr int R = 2 * (SB + SW + SS);
    auto a_full = [&](int i) { return bars + 8 * (R + i); };
    auto a_empty = [&](int i) { return bars + 8 * (R + 4 + i); };
    auto d_full = [&](int i) { return bars + 8 * (R + 8 + i); };
    auto d_empty = [&](int i) { return bars + 8 * (R + 10 + i); };
    const uint32_t drained = bars + 8 * (R + 12), never = bars + 8 * (R + 14);

    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "r"(kTmemCols));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    if (tid == 32) {
        auto init = [&](uint32_t b, int n) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(b), "r"(n)); };
        for (int i = 0; i < SB; ++i) init(b_full(i), 1), init(b_empty(i), 1);
        for (int i = 0; i < SW; ++i) init(w_full(i), 1), init(w_empty(i), 4);
        for (int i = 0; i < SS; ++i) init(s_full(i), 1), init(s_empty(i), L::kEpiWarps);
        for (int i = 0; i < 4; ++i) init(a_full(i), 4), init(a_empty(i), 1);
        for (int i = 0; i < 2; ++i) init(d_full(i), 1), init(d_empty(i), L::kEpiWarps);
        init(drained, 1), init(drained + 8, 1), init(never, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        s_fail = 0;
    }
    tc_before();
    __syncthreads();
    tc_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, s_tmem, 0);
    // scales and activations' terms may come from the kernel before
    asm volatile("griddepcontrol.wait;" ::: "memory");

    // A ring's position at the side that fills it: a stage is waited for, filled, and the next one is up.
    struct Fill {
        int st = 0, done = 0;
        unsigned ph = 1;  // the first round passes
    };
    auto fill = [&](Fill& r, int stages, uint32_t full0, uint32_t empty0, uint32_t bytes) -> bool {
        if (!mbar_wait_warp(empty0 + 8 * r.st, r.ph)) {
            if (lane == 0) s_fail = 1;
            return false;
        }
        expect_tx(full0 + 8 * r.st, bytes);
        r.done = min(r.done + 1, stages);
        return true;
    };
    auto next = [](Fill& r, int stages) {
        if (++r.st == stages) r.st = 0, r.ph ^= 1;
    };
    // Nothing may be in flight when the CTA exits: the last filling of each stage has to land.
    auto landed = [&](Fill& r, int stages, uint32_t full0) {
        for (; r.done > 0; --r.done) {
            if (--r.st < 0) r.st = stages - 1, r.ph ^= 1;
            mbar_wait_warp(full0 + 8 * r.st, r.ph ^ 1);
        }
    };
    if (warp == 0) {
        Fill r;
        bool ok = true;
        if (a.expire && blockIdx.x == 0 && !__all_sync(0xffffffffu, mbar_wait(never, 0, kWaitLimit >> 8)) && lane == 0) s_fail = 1;
        __syncwarp();
        for (int tile = tile0; ok && tile < a.tiles; tile += tile_step) {
            const int t0 = tile / row_blocks * N;
            for (int i = 2 * c_lo; i < 2 * c_hi; ++i) {
                ok = fill(r, SB, b_full(0), b_empty(0), L::kB);
                if (!ok) break;
#pragma unroll
                for (int p = 0; p < TERMS; ++p)
                    tma_2d(sb + L::kOffB + r.st * L::kB + p * L::kAtom, &tm_x, i * 64, t0 + p * a.plane_rows, b_full(r.st));
                next(r, SB);
            }
        }
        landed(r, SB, b_full(0));
    } else if (warp == 2) {
        const uint32_t zb = a.w.zeros ? 64u * (pc == 4 ? 8 : 4) : 0u, scb = 256u * (uint32_t)pc;
        const int xs_rows = a.x_scales ? (a.x_group < kK ? kK / a.x_group : 1) : 0;  // groups that meet 128 inputs
        Fill r, q;
        for (int tile = tile0, ok = 1; ok && tile < a.tiles; tile += tile_step) {
            const int rb = tile % row_blocks, t0 = tile / row_blocks * N;
            for (int c = c_lo; c < c_hi; ++c) {
                const size_t at = (size_t)rb * chunks + c;
                ok = fill(r, SW, w_full(0), w_empty(0), 8192u + zb);
                if (!ok) break;
                bulk(sb + L::kOffW + r.st * L::kW, reinterpret_cast<const unsigned char*>(a.w.codes) + at * 8192, 8192, w_full(r.st));
                if (zb)
                    bulk(sb + L::kOffW + r.st * L::kW + 8192, reinterpret_cast<const unsigned char*>(a.w.zeros) + at * zb, zb, w_full(r.st));
                next(r, SW);
                ok = fill(q, SS, s_full(0), s_empty(0), scb + xs_rows * N * 4u);
                if (!ok) break;
                bulk(sb + L::kOffS + q.st * L::kS, reinterpret_cast<const unsigned char*>(a.w.scales) + at * scb, scb, s_full(q.st));
                for (int j = 0; j < xs_rows; ++j) {  // behind the last group (padded inputs) the last one again
                    const size_t gr = min((size_t)c * kK / a.x_group + j, a.x_groups - 1);
                    bulk(sb + L::kOffS + q.st * L::kS + L::kXs + j * N * 4, a.x_scales + gr * a.x_pitch + t0, N * 4, s_full(q.st));
                }
                next(q, SS);
            }
        }
        landed(r, SW, w_full(0));
        landed(q, SS, s_full(0));
    } else if (warp == 1 || (warp == 3 && kIssuers == 2)) {
        // Issue is on the critical path: every offset below is a constant of the unrolled loop, ring
        // positions and phases are carried along. Four waits, four commits and eight MMAs a chunk take a warp some
        // 900 cycles, more than 128 tokens' MMAs do: where a chunk is one handing over, two warps take
        // turns, each with an accumulator and two A buffers of its own.
        constexpr uint32_t idesc = instr_desc(N, BF16);
        const int first = warp == 3;
        const uint64_t b0 = smem_desc(sb + L::kOffB);
        int st = 2 * first;  // ring stage
        uint32_t ab = first, db = first;
        unsigned b_ph = 0, a_ph = 0, d_ph = 1;  // d_ph: of the accumulators' last reads; the first round passes
        bool ok = true;
        for (int c = first; ok && c < n_chunks; c += kIssuers) {
            ok = mbar_wait_warp(a_full(0) + 8 * ab, a_ph);
            if (!ok) break;
            const uint32_t ta = tmem + kColA + 64 * ab;
            uint64_t bd = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {  // 16 inputs: 8 columns of A, 32 bytes of B
                constexpr int kUnit = 2 * FB * U;  // steps of 16 inputs between two handings over
                // The accumulator first: once it is free, every chunk before the last two is done, so the
                // stage's phase before the one waited for is over whichever warp used it.
                if (i % kUnit == 0) {
                    ok = mbar_wait_warp(d_empty(0) + 8 * db, d_ph);
                    if (!ok) break;
                }
                if (i % 4 == 0) {
                    ok = mbar_wait_warp(b_full(0) + 8 * st, b_ph);
                    if (!ok) break;
                    bd = b0 + (uint64_t)(st * (L::kB >> 4));
                }
                if (i % 4 == 0 || i % kUnit == 0) tc_after();
#pragma unroll
                for (int p = 0; p < TERMS; ++p)
                    mma_ts(tmem + db * 128 + i % kUnit / (2 * FB) * N, ta + 8 * i,
                           bd + (uint64_t)((p * L::kAtom + (i & 3) * 32) >> 4), idesc, i % (2 * FB) > 0 || p > 0);
                if ((i + 1) % kUnit == 0) {
                    commit(d_full(0) + 8 * db);
                    if (kIssuers == 2) {
                        d_ph ^= 1;
                    } else {
                        db ^= 1;
                        if (db == 0) d_ph ^= 1;
                    }
                }
                if (i % 4 == 3) {
                    commit(b_empty(0) + 8 * st);
                    if (++st == SB) st = 0, b_ph ^= 1;
                }
            }
            if (!ok) break;
            commit(a_empty(0) + 8 * ab);
            ab += kIssuers;
            if (ab >= 4) ab -= 4, a_ph ^= 1;
            if (kIssuers == 2) {  // the other warp's two stages
                st += 2;
                if (st >= SB) st -= SB, b_ph ^= 1;
            }
        }
        if (!ok && lane == 0) s_fail = 1;
        commit(drained + 8 * first);  // every MMA of this warp done, also after a failed wait
        mbar_wait_warp(drained + 8 * first, 0);
    } else if (warp >= kConvert0 && warp < kEpi0) {
        const int w = warp & 3, g = lane >> 2, rec = pc == 4 ? 8 : 4, set = (warp - kConvert0) >> 2;
        bool ok = true;
        int st = set, ab = set;
        unsigned w_ph = 0, a_ph = 1;  // the first round of A buffers passes
        for (int c = set; c < n_chunks; c += 2) {
            ok = mbar_wait_warp(w_full(st), w_ph) && mbar_wait_warp(a_empty(ab), a_ph);
            if (!ok) break;
            tc_after();
            const unsigned char* base = sm + L::kOffW + st * L::kW;
#pragma unroll 1
            for (int m = 0; m < 2; ++m) {  // tiles of 16 rows
                const int tile = 2 * w + m;
                const uint4 va = *reinterpret_cast<const uint4*>(base + tile * 1024 + lane * 16);
                const uint4 vb = *reinterpret_cast<const uint4*>(base + tile * 1024 + 512 + lane * 16);
                const uint32_t wa[4] = {va.x, va.y, va.z, va.w}, wb[4] = {vb.x, vb.y, vb.z, vb.w};
                const unsigned char* z = base + 8192 + (tile * 8 + g) * rec;
                uint32_t za = 0, za2 = 0, zb = 0, zb2 = 0;
                uint32_t r[32];
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    if (b * pc % 4 == 0) {
                        const uint32_t zz = a.w.zeros ? *reinterpret_cast<const unsigned short*>(z + 2 * (b * pc / 4)) : 0x0808u;
                        zero_pairs<BF16>(zz & 0xffu, za, za2);
                        zero_pairs<BF16>(zz >> 8, zb, zb2);
                    }
                    uint32_t pa[4], pb[4];
                    pairs<BF16>(wa[b], za, za2, pa);
                    pairs<BF16>(wb[b], zb, zb2, pb);
#pragma unroll
                    for (int j = 0; j < 4; ++j) r[2 * (4 * b + j)] = pa[j], r[2 * (4 * b + j) + 1] = pb[j];
                }
                tmem_st_tile(tmem + ((uint32_t)(32 * w + 16 * m) << 16) + kColA + 64 * ab, r);
            }
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            tc_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(a_full(ab)), mbar_arrive(w_empty(st));
            st += 2, ab += 2;
            if (st >= SW) st -= SW, w_ph ^= 1;
            if (ab >= 4) ab -= 4, a_ph ^= 1;
        }
        if (!ok && lane == 0) s_fail = 1;
    } else if (warp >= kEpi0) {
        constexpr int C = N * 4 / L::kEpiWarps;  // columns of a thread
        const int w = warp - kEpi0, part = w >> 2, row = 32 * (w & 3) + lane;
        const uint32_t t_d = tmem + ((uint32_t)(32 * (w & 3)) << 16) + part * C;
        // this row's scales in a stage: [tile][row % 8][block][row / 8]
        const int sc_at = (((row >> 4) * 8 + (row & 7)) * pc * 2 + ((row >> 3) & 1)) * 2;
        bool ok = true;
        int st = 0, db = 0;
        unsigned d_ph = 0, s_ph = 0;
        for (int tile = tile0; ok && tile < a.tiles; tile += tile_step) {
            const int rb = tile % row_blocks, t0 = tile / row_blocks * N;
            uint64_t acc[C / 2];  // pairs of neighbouring tokens
#pragma unroll
            for (int i = 0; i < C / 2; ++i) acc[i] = 0;
            for (int c = c_lo; ok && c < c_hi; ++c) {
                const unsigned char* base = sm + L::kOffS + st * L::kS;
                ok = mbar_wait_warp(s_full(st), s_ph);
#pragma unroll
                for (int h = 0; h < H; ++h) {
                    ok = ok && mbar_wait_warp(d_full(db), d_ph);
                    if (!ok) break;
                    tc_after();
#pragma unroll
                    for (int f = 0; f < U; ++f) {
                        const int sum = h * U + f;
                        const float s1 = scale_of(*reinterpret_cast<const unsigned short*>(base + sc_at + (sum * FB * pc / 4) * 4), a.w.scale_bf16);
                        const uint64_t s = pack2(__float_as_uint(s1), __float_as_uint(s1));
                        const unsigned char* xs = base + L::kXs + part * C * 4 + (sum * FB * 32 >> a.x_shift) * (N * 4);
                        constexpr int B = 16;  // columns in registers at a time
#pragma unroll
                        for (int j = 0; j < C; j += B) {
                            uint32_t d[B];
                            tmem_ld<B>(t_d + db * 128 + f * N + j, d);
                            tmem_ld_wait();
                            if (f == U - 1 && j + B == C) {
                                tc_before();
                                __syncwarp();
                                if (lane == 0) mbar_arrive(d_empty(db));
                            }
                            if (a.x_scales) {
#pragma unroll
                                for (int i = 0; i < B; i += 4) {
                                    const ulonglong2 x4 = *reinterpret_cast<const ulonglong2*>(xs + (j + i) * 4);
                                    fma2(acc[(j + i) / 2], mul2(pack2(d[i], d[i + 1]), x4.x), s);
                                    fma2(acc[(j + i) / 2 + 1], mul2(pack2(d[i + 2], d[i + 3]), x4.y), s);
                                }
                            } else {
#pragma unroll
                                for (int i = 0; i < B; i += 2) fma2(acc[(j + i) / 2], pack2(d[i], d[i + 1]), s);
                            }
                        }
                    }
                    db ^= 1;
                    if (db == 0) d_ph ^= 1;
                }
                __syncwarp();
                if (ok && lane == 0) mbar_arrive(s_empty(st));
                if (++st == SS) st = 0, s_ph ^= 1;
            }
            const size_t r = (size_t)rb * kM + row;
            if constexpr (SPLIT) {  // every MMA of this CTA is done: its activations' ring holds the part's sums
#pragma unroll
                for (int i = 0; i < C; ++i) reinterpret_cast<float*>(sm + L::kOffB)[(part * C + i) * kM + row] = half_of(acc[i / 2], i & 1);
            } else if (ok && r < a.w.n_out && !*reinterpret_cast<volatile int*>(&s_fail)) {
#pragma unroll
                for (int i = 0; i < C; ++i) {
                    const size_t t = (size_t)t0 + part * C + i;
                    if (t >= a.tokens) break;
                    store(a, t, r, half_of(acc[i / 2], i & 1));
                }
            }
        }
        if (!ok && lane == 0) s_fail = 1;
    }
    __syncwarp();
    tc_before();
    __syncthreads();
    if (tid == 0 && *reinterpret_cast<volatile int*>(&s_fail)) *reinterpret_cast<volatile int*>(a.err) = kErrWaitTimeout;
    if (warp == 0) {
        tc_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols));
    }
    if constexpr (SPLIT) {  // the parts' sums in order, a share of the tokens by each CTA
        cluster_sync();
        int fail = 0;
        for (int j = 0; j < split; ++j) fail |= ld_cluster(smem_u32(&s_fail), j);
        const int n_lo = N * rank / split, n_hi = N * (rank + 1) / split, rb = tile0 % row_blocks, t0 = tile0 / row_blocks * N;
        for (int i = n_lo * kM + tid; !fail && i < n_hi * kM; i += L::kThreads) {
            const size_t r = (size_t)rb * kM + i % kM, t = (size_t)t0 + i / kM;
            if (r >= a.w.n_out || t >= a.tokens) continue;
            float v = 0.f;
            for (int j = 0; j < split; ++j) v += __int_as_float(ld_cluster(sb + L::kOffB + 4 * i, j));
            store(a, t, r, v);
        }
        cluster_sync();  // nobody leaves while its sums are read
    }
}

// A token's row as 16-bit terms with zeros up to kp, and its factor. f32: two f16 terms of x · 2^e, factor 2^-e;
// int8: f16, factor its scale (when it has one for the row); bf16: copied. Grouped scales are transposed.
__global__ void __launch_bounds__(256) w4_terms_kernel(W4X x, size_t kp, uint16_t* out, float* col_scale, float* x_scales,
                                                       size_t x_pitch) {
    asm volatile("griddepcontrol.launch_dependents;");
    __shared__ float s_max[8];
    const size_t plane = x.tokens * kp;
    for (size_t t = blockIdx.x; t < x.tokens; t += gridDim.x) {
        uint16_t* o = out + t * kp;
        if (x.kind == kW4XF32) {
            const float* p = static_cast<const float*>(x.x) + t * x.stride;
            const bool pairs = (reinterpret_cast<uintptr_t>(p) & 7) == 0;
            auto pair = [&](size_t k) {
                if (k >= x.n_in) return make_float2(0.f, 0.f);
                return pairs ? *reinterpret_cast<const float2*>(p + k) : make_float2(p[k], p[k + 1]);
            };
            constexpr int kKeep = 8;  // pairs a thread keeps between the maximum and the terms: rows of 4096
            float2 keep[kKeep];
            float m = 0.f;
#pragma unroll
            for (int i = 0; i < kKeep; ++i) {
                keep[i] = pair(2 * threadIdx.x + 512 * i);
                m = fmaxf(m, fmaxf(fabsf(keep[i].x), fabsf(keep[i].y)));
            }
            for (size_t k = 2 * threadIdx.x + 512 * kKeep; k < x.n_in; k += 512) {
                const float2 v = pair(k);
                m = fmaxf(m, fmaxf(fabsf(v.x), fabsf(v.y)));
            }
#pragma unroll
            for (int i = 16; i > 0; i >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, i));
            __syncthreads();
            if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = m;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 8; ++i) m = fmaxf(m, s_max[i]);
            // 2^e with m 2^e in [2^14, 2^15); an infinity or only zeros: e = 0. Two factors, since 2^e may
            // itself be out of f32's range.
            const int em = (int)(__float_as_uint(m) >> 23);
            const int e = m > 0.f && em < 255 ? 14 - (max(em, 1) - 127) : 0, e1 = e / 2, e2 = e - e1;
            const float f1 = __uint_as_float((uint32_t)(127 + e1) << 23), f2 = __uint_as_float((uint32_t)(127 + e2) << 23);
            if (threadIdx.x == 0) col_scale[t] = ldexpf(1.f, -e);
            auto write = [&](size_t k, float2 u) {
                uint32_t hi = 0, lo = 0;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const float v = (j ? u.y : u.x) * f1 * f2;
                    const __half a = __float2half_rn(v);
                    const float rest = v - __half2float(a);
                    const __half b = __float2half_rn(fabsf(rest) <= 65504.f ? rest : 0.f);  // v not finite: no second term
                    hi |= (uint32_t)__half_as_ushort(a) << (16 * j), lo |= (uint32_t)__half_as_ushort(b) << (16 * j);
                }
                *reinterpret_cast<uint32_t*>(o + k) = hi;
                *reinterpret_cast<uint32_t*>(o + plane + k) = lo;
            };
#pragma unroll
            for (int i = 0; i < kKeep; ++i)
                if (const size_t k = 2 * threadIdx.x + 512 * i; k < kp) write(k, keep[i]);
            for (size_t k = 2 * threadIdx.x + 512 * kKeep; k < kp; k += 512) write(k, pair(k));
        } else {
            for (size_t k = 2 * threadIdx.x; k < kp; k += 512) {
                uint32_t v = 0;
                if (k < x.n_in) {
                    if (x.kind == kW4XInt8) {
                        const signed char* p = static_cast<const signed char*>(x.x) + t * x.stride + k;
                        v = (uint32_t)__half_as_ushort(__short2half_rn(p[0])) | (uint32_t)__half_as_ushort(__short2half_rn(p[1])) << 16;
                    } else {
                        const unsigned short* p = static_cast<const unsigned short*>(x.x) + t * x.stride + k;
                        v = (uint32_t)p[0] | (uint32_t)p[1] << 16;
                    }
                }
                *reinterpret_cast<uint32_t*>(o + k) = v;
            }
            if (x_scales)
                for (size_t j = threadIdx.x; j < x.n_groups; j += 256) x_scales[j * x_pitch + t] = x.scales[t * x.n_groups + j];
        }
    }
}

PFN_cuTensorMapEncodeTiled_v12000 map_encoder() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
    }();
    return fn;
}

// bf16 rows that TMA can read as they are
bool direct_rows(const W4X& x) {
    return x.kind == kW4XBf16 && (reinterpret_cast<uintptr_t>(x.x) & 15) == 0 && x.stride % 8 == 0;
}
size_t pad(size_t n, size_t to) { return (n + to - 1) / to * to; }
size_t terms_bytes(const W4View& w, const W4X& x) {
    return pad((x.kind == kW4XF32 ? 2 : 1) * x.tokens * w.chunks * kK * 2, 256);
}

// Clusters of k CTAs of a kernel that run at once on the device.
template <int N, int TERMS, bool BF16, int FB>
cudaError_t clusters_that_fit(int k, int num_sms, int* n) {
    static std::atomic<int> known[9];  // + 1
    *n = known[k].load(std::memory_order_relaxed) - 1;
    if (*n >= 0) return cudaSuccess;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(k * num_sms));
    cfg.blockDim = dim3(Lay<N, TERMS, BF16>::kThreads);
    cfg.dynamicSmemBytes = Lay<N, TERMS, BF16>::kSmem;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = (unsigned)k;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaOccupancyMaxActiveClusters(n, w4_tc_kernel<N, TERMS, BF16, FB, true>, &cfg);
    if (e == cudaSuccess) known[k].store(*n + 1, std::memory_order_relaxed);
    return e;
}

template <int N, int TERMS, bool BF16, int FB>
cudaError_t run(const CUtensorMap& tm, TcArgs& a, int num_sms, bool pdl, cudaStream_t s) {
    using L = Lay<N, TERMS, BF16>;
    static SmemOnce once, once_split;
    cudaError_t e = once.set(reinterpret_cast<const void*>(w4_tc_kernel<N, TERMS, BF16, FB, false>), L::kSmem);
    if (e == cudaSuccess) e = once_split.set(reinterpret_cast<const void*>(w4_tc_kernel<N, TERMS, BF16, FB, true>), L::kSmem);
    if (e != cudaSuccess) return e;
    a.tiles = (int)(a.w.tile_rows / 8 * ((a.tokens + N - 1) / N));
    // Tiles for half of the SMs or less: clusters of up to 8 share a tile's inputs, at least two chunks a CTA, if all
    // of them run at once. (24 f32 tokens, 5003 x 2080: 16.3 us with a CTA a tile, 12.4 us with three; 17 bf16 tokens,
    // 8192 x 8192: 29.7 and 20.4 us with two.)
    a.split = 1;
    for (int k = 8; k > 1 && a.split == 1; --k) {
        if ((size_t)k * 2 > a.w.chunks || (long long)a.tiles * k > num_sms) continue;
        int n;
        e = clusters_that_fit<N, TERMS, BF16, FB>(k, num_sms, &n);
        if (e != cudaSuccess) return e;
        if (a.tiles <= n) a.split = k;
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(a.split > 1 ? a.tiles * a.split : std::min(a.tiles, num_sms)));
    cfg.blockDim = dim3(L::kThreads);
    cfg.dynamicSmemBytes = L::kSmem;
    cfg.stream = s;
    cudaLaunchAttribute at[2] = {};
    if (pdl) {
        at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[0].val.programmaticStreamSerializationAllowed = 1;
        ++cfg.numAttrs;
    }
    if (a.split > 1) {
        at[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
        at[cfg.numAttrs].val.clusterDim.x = (unsigned)a.split;
        at[cfg.numAttrs].val.clusterDim.y = at[cfg.numAttrs].val.clusterDim.z = 1;
        ++cfg.numAttrs;
    }
    cfg.attrs = at;
    return a.split > 1 ? cudaLaunchKernelEx(&cfg, w4_tc_kernel<N, TERMS, BF16, FB, true>, tm, a)
                       : cudaLaunchKernelEx(&cfg, w4_tc_kernel<N, TERMS, BF16, FB, false>, tm, a);
}
template <int N, int TERMS, bool BF16>
cudaError_t run_fb(const CUtensorMap& tm, TcArgs& a, int fb, int num_sms, bool pdl, cudaStream_t s) {
    return fb == 4   ? run<N, TERMS, BF16, 4>(tm, a, num_sms, pdl, s)
           : fb == 2 ? run<N, TERMS, BF16, 2>(tm, a, num_sms, pdl, s)
                     : run<N, TERMS, BF16, 1>(tm, a, num_sms, pdl, s);
}
template <int N>
cudaError_t run_kind(const CUtensorMap& tm, TcArgs& a, int kind, int fb, int num_sms, bool pdl, cudaStream_t s) {
    return kind == kW4XBf16  ? run_fb<N, 1, true>(tm, a, fb, num_sms, pdl, s)
           : kind == kW4XF32 ? run_fb<N, 2, false>(tm, a, fb, num_sms, pdl, s)
                             : run_fb<N, 1, false>(tm, a, fb, num_sms, pdl, s);
}

}  // namespace

size_t w4_tc_workspace(const W4View& w, const W4X& x) {
    if (direct_rows(x)) return 0;
    size_t n = terms_bytes(w, x) + pad(4 * x.tokens, 256);
    if (x.group) n += 4 * x.n_groups * pad(x.tokens, 128);
    return n;
}

cudaError_t launch_w4_tc(const W4View& w, const W4X& x, void* y, int y_bf16, void* workspace, int num_sms, int* err, bool expire,
                         cudaStream_t s) {
    const auto enc = map_encoder();
    const size_t kp = w.chunks * kK, terms = x.kind == kW4XF32 ? 2 : 1;
    if (!enc || x.tokens * terms >= (1ull << 31) || w.tile_rows / 8 * (x.tokens / 32 + 1) >= (1ull << 31)) return cudaErrorNotSupported;
    TcArgs a{};
    a.w = w;
    a.y = y, a.y_bf16 = y_bf16, a.tokens = x.tokens, a.err = err, a.expire = expire;
    int fb = 4 / w.per_chunk;
    if (x.group) fb = std::min(fb, x.group / 32);
    const bool direct = direct_rows(x);
    const void* rows = x.x;
    size_t stride = x.stride, n_in = x.n_in;
    const int n_tile = x.tokens <= 32 ? 32 : x.tokens <= 64 ? 64 : 128;
    if (!direct) {
        uint16_t* t = static_cast<uint16_t*>(workspace);
        float* col = reinterpret_cast<float*>(static_cast<char*>(workspace) + terms_bytes(w, x));
        float* xs = reinterpret_cast<float*>(reinterpret_cast<char*>(col) + pad(4 * x.tokens, 256));
        a.x_pitch = pad(x.tokens, 128);
        a.x_scales = x.group ? xs : nullptr;
        a.x_group = x.group;
        a.x_shift = x.group ? std::min(x.group_shift, 7) : 7;
        a.x_groups = x.n_groups;
        a.col_scale = x.kind == kW4XF32 ? col : x.kind == kW4XInt8 && !x.group ? x.scales : nullptr;
        w4_terms_kernel<<<(unsigned)std::min<size_t>(x.tokens, 1 << 20), 256, 0, s>>>(x, kp, t, col, x.group ? xs : nullptr, a.x_pitch);
        const cudaError_t e = cudaGetLastError();
        if (e != cudaSuccess) return e;
        rows = t;
        stride = n_in = kp;
        a.plane_rows = (int)x.tokens;
    }
    CUtensorMap tm;
    const cuuint64_t dims[2] = {(cuuint64_t)n_in, (cuuint64_t)(x.tokens * terms)};
    const cuuint64_t strides[1] = {(cuuint64_t)(stride * 2)};
    const cuuint32_t box[2] = {64, (cuuint32_t)n_tile}, es[2] = {1, 1};
    if (enc(&tm, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, const_cast<void*>(rows), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        return cudaErrorInvalidValue;
    return n_tile == 32   ? run_kind<32>(tm, a, x.kind, fb, num_sms, !direct, s)
           : n_tile == 64 ? run_kind<64>(tm, a, x.kind, fb, num_sms, !direct, s)
                          : run_kind<128>(tm, a, x.kind, fb, num_sms, !direct, s);
}

}  // namespace bebelm
