// Products with 4-bit weights and group scales, few tokens (w4_stream_kernel), and the weights'
// layout (w4_pack_kernel) and the activations' (w4_planes_kernel) that the many-token kernel
// (w4_tc.cu) shares.
//
//     y[t][n] = Σ_g s[n][g] · sx[t][g'] · Σ_{k in g} (c[n][k] - z[n][g]) · x[t][k]
//
// with 4-bit codes c, a zero point z (8 when the weights have none), a scale s per group of one
// row's weights, and for int8 activations a scale sx per row or per x_group values of a token.
//
// The inner sum runs on the tensor cores in bf16 with f32 accumulation, and loses nothing there:
// c - z is an integer in [-127, 15] (zero points above 127 are refused), so a bf16; a bf16 or int8
// activation is a bf16 too; an f32 activation is the sum of three bf16 (8 + 8 + 8 significant bits, split
// by truncation, so exactly), one MMA each. Scales
// are applied in f32 to the f32 sum of each group, as the formula has it.
//
// Bound: a weight is read once, for at most 32 tokens, so HBM. What a weight costs on the way: one
// half of a logic operation and a shift to move two codes into a bf16 pair (0x4300 | c is 128 + c), one
// packed subtraction of 128 + z per pair, 1/256 of an MMA per 8 tokens and bf16 term.
//
// Layout: rows padded to 128, inputs to 128 (scale 0). A tile of 16 rows x 128 inputs is 1024 bytes,
// [row / 8][row % 8][q = 0..3][b = 0..3] words of 8 codes; the 8 tiles of 128 rows lie together, then the next 128
// inputs. Word (q, b) of a row holds inputs 32 b + 8 j + 2 q + e (j = 0..3, e = 0, 1) in nibble j + 4 e: what lane
// (g, q) of a warp gives to the A fragments of two m16n8k16 MMAs, and (w >> 4 j) & 0x000f000f is a pair of neighbours.
// A lane reads 16 bytes of its rows g and g + 8. The activations of 32 inputs are laid out alike ([q][j][e], 16 bytes a
// lane). Blocks of 32 inputs stay whole, so a group of 32 ends with an MMA. Scales [tile][row % 8][block of
// min(group, 128) inputs][row / 8], zero points the same in bytes: a lane's scales of a tile are one load.
#include <algorithm>
#include <cstdint>

#include "internal.h"

namespace bebelm {
namespace {

constexpr int kWarps = 8;    // of a CTA
constexpr int kChunk = 128;  // inputs of a tile

// How a kernel takes its activations: as they are (bf16), as three bf16 terms (f32), or as f16 (int8 with a
// scale a token, or a scale a group).
constexpr int kBf16 = 0, kF32x3 = 1, kI8Row = 2, kI8Group = 3;

// The zero points of a row as a pair to subtract: 128 + z in bf16, or, packed for f16, 1024 + z and 64 + z.
template <bool F16>
struct Zero {
    uint32_t a, b;
    __device__ __forceinline__ void set(uint32_t z) {  // z: one byte
        if constexpr (F16) {
            a = 0x64006400u + z * 0x10001u;
            // f16 of 64 + z: 10 mantissa bits below 2^6 up to 127, below 2^7 from 128 on
            const __half2 h = __half2half2(__ushort2half_rn((unsigned short)(64 + z)));
            b = *reinterpret_cast<const uint32_t*>(&h);
        } else {
            a = 0x43004300u + z * 0x10001u;
        }
    }
};

// 8 codes of a word to 4 pairs of c - z, exactly.
// bf16: 0x4300 | c is 128 + c; 128 + z is taken off. f16: two fields of a half word fit the mantissa: 0x6400 | c is
// 1024 + c, and 0x6400 | 16 c is 1024 + 16 c, 1/16 of which less 64 + z is c - z: one shift a word instead of three.
template <bool F16>
__device__ __forceinline__ void code_pairs(uint32_t w, const Zero<F16>& z, uint32_t* o) {
    if constexpr (F16) {
        const __half2 za = *reinterpret_cast<const __half2*>(&z.a), zb = *reinterpret_cast<const __half2*>(&z.b);
        const __half2 s16 = __float2half2_rn(0.0625f);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t v = i ? w >> 8 : w;
            const uint32_t lo = (v & 0x000f000fu) | 0x64006400u, hi = (v & 0x00f000f0u) | 0x64006400u;
            const __half2 a = __hsub2(*reinterpret_cast<const __half2*>(&lo), za);
            const __half2 b = __hfma2(*reinterpret_cast<const __half2*>(&hi), s16, __hneg2(zb));
            o[2 * i] = *reinterpret_cast<const uint32_t*>(&a);
            o[2 * i + 1] = *reinterpret_cast<const uint32_t*>(&b);
        }
    } else {
        const __nv_bfloat162 zz = *reinterpret_cast<const __nv_bfloat162*>(&z.a);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t u = ((w >> (4 * i)) & 0x000f000fu) | 0x43004300u;
            const __nv_bfloat162 a = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&u), zz);
            o[i] = *reinterpret_cast<const uint32_t*>(&a);
        }
    }
}

template <bool F16>
__device__ __forceinline__ void mma16816(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
    if constexpr (F16)
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float scale_of(uint32_t h, int bf16) {
    if (bf16) return __uint_as_float(h << 16);
    __half_raw r;
    r.x = (unsigned short)h;
    return __half2float(__half(r));
}

// x = p0 + p1 + p2 exactly: 8 significant bits each, cut off towards zero. A non-finite x stays in p0 alone.
__device__ __forceinline__ void split3(float x, uint32_t* p) {
    p[0] = __float_as_uint(x) & 0xffff0000u;
    float r = x - __uint_as_float(p[0]);
    if (!(fabsf(x) <= 3.4028234663852886e38f)) {  // inf or NaN (whose kept bits must not be all zero)
        if (x != x) p[0] |= 0x00400000u;
        r = 0.f;
    }
    p[1] = __float_as_uint(r) & 0xffff0000u;
    p[2] = __float_as_uint(r - __uint_as_float(p[1]));  // at most 8 bits are left
}

// Four pairs of a token's activations as P x 4 words of two 16-bit values; zeros past n_in (a multiple of 32). The pairs
// start at inputs k, k + d, k + 2 d, k + 3 d of one block of 32. f32: three bf16 terms; bf16: as they are; int8: f16.
template <int P>
__device__ __forceinline__ void x_pairs(const W4X& x, size_t t, size_t k, int d, uint32_t (*v)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        uint32_t a[3] = {0, 0, 0}, b[3] = {0, 0, 0};
        if (k < x.n_in) {
            const size_t o = t * x.stride + k + j * d;
            if (P == 3) {
                const float* p = static_cast<const float*>(x.x) + o;
                split3(p[0], a), split3(p[1], b);
            } else if (x.kind == kW4XInt8) {
                const signed char* p = static_cast<const signed char*>(x.x) + o;
                a[0] = (uint32_t)__half_as_ushort(__short2half_rn(p[0])) << 16;
                b[0] = (uint32_t)__half_as_ushort(__short2half_rn(p[1])) << 16;
            } else {
                const unsigned short* p = static_cast<const unsigned short*>(x.x) + o;
                a[0] = (uint32_t)p[0] << 16, b[0] = (uint32_t)p[1] << 16;
            }
        }
#pragma unroll
        for (int i = 0; i < P; ++i) v[i][j] = __byte_perm(a[i], b[i], 0x7632);
    }
}

// The activations in the lanes' order, [P][tokens][kp] with zeros past n_in.
template <int P>
__global__ void __launch_bounds__(256) w4_planes_kernel(W4X x, size_t kp, uint16_t* out) {
    asm volatile("griddepcontrol.launch_dependents;");
    const size_t plane = x.tokens * kp;
    for (size_t t = blockIdx.y; t < x.tokens; t += gridDim.y)
        for (size_t k = 8 * ((size_t)blockIdx.x * blockDim.x + threadIdx.x); k < kp; k += 8 * (size_t)gridDim.x * blockDim.x) {
            uint32_t v[P][4];
            x_pairs<P>(x, t, (k & ~size_t(31)) + (k >> 2 & 6), 8, v);
#pragma unroll
            for (int i = 0; i < P; ++i)
                *reinterpret_cast<uint4*>(out + i * plane + t * kp + k) = make_uint4(v[i][0], v[i][1], v[i][2], v[i][3]);
        }
}

// codes [n_out][n_in / 2], scales and zeros [n_out][n_in / group] into the layout above, a
// thread per word of 8 codes
__global__ void __launch_bounds__(256) w4_pack_kernel(const uint8_t* codes, const unsigned short* scales,
                                                      const uint8_t* zeros, W4View w, uint32_t* out_c,
                                                      unsigned short* out_s, uint8_t* out_z, int* bad) {
    const size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x;  // word of out_c
    const size_t tile = i >> 8, c = (tile >> 3) % w.chunks, tr = (tile >> 3) / w.chunks * 8 + (tile & 7);
    if (tr >= w.tile_rows) return;
    const int in = (int)(i & 255), b = in & 3, q = (in >> 2) & 3, r = in >> 4;  // r = 8 (row / 8) + row % 8
    const size_t row = tr * 16 + r, k = c * kChunk + 32 * b + 2 * q;
    uint32_t v = 0;
    if (row < w.n_out && k < w.n_in) {
        const uint8_t* p = codes + row * (w.n_in / 2) + k / 2;
        for (int j = 0; j < 4; ++j) v |= (uint32_t)(p[4 * j] & 15) << (4 * j) | (uint32_t)(p[4 * j] >> 4) << (4 * j + 16);
    }
    out_c[i] = v;
    if (q == 0 && b < w.per_chunk) {  // one scale per (row, block of min(group, 128) inputs)
        const size_t ks = c * kChunk + (size_t)b * (kChunk / w.per_chunk);
        const size_t o = ((tile * 8 + (r & 7)) * w.per_chunk + b) * 2 + (r >> 3);
        const bool in_range = row < w.n_out && ks < w.n_in;
        const size_t g = row * (w.n_in / w.group) + ks / w.group;
        out_s[o] = in_range ? scales[g] : 0;
        if (out_z) {  // a row pair's zero points take 4 bytes at least, so that a lane can copy them
            const uint8_t z = in_range ? zeros[g] : 8;
            const int rec = w.per_chunk == 4 ? 8 : 4;
            out_z[(tile * 8 + (r & 7)) * rec + 2 * b + (r >> 3)] = z;
            if (z > 127) *bad = 1;
        }
    }
}

struct StreamArgs {
    W4View w;
    W4X x;
    const uint16_t* planes;  // [P][x.tokens][ldp], 16-byte aligned rows; null: made in shared memory
    size_t ldp, plane;            // elements of a row and of a plane
    void* y;
    int y_bf16, ks, tiles;        // ks warps share a row of tiles; `tiles` groups of kWarps / ks of them
    int sums_at;                  // float offset of the warps' partial sums behind ring and planes in shared memory
};

// N bytes from global to shared memory, asynchronously; 16-byte copies pass L1 by
template <int N>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src) {
    if constexpr (N == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(N) : "memory");
}

// One ring stage of a warp: MT tiles' codes, then their scales and zero points. A lane copies exactly
// what it reads itself, so a stage needs no barrier, only its own lane's copies to have landed.
template <int MT, int PC>
struct Stage4 {
    static constexpr int kStages = MT == 1 ? 5 : 3;  // 4 KB in flight a warp while one stage is multiplied
    static constexpr int kZero = PC == 4 ? 8 : 4;  // bytes of zero points of a lane and tile (4 for PC 1: padded)
    static constexpr int kScaleAt = MT * 1024, kZeroAt = kScaleAt + MT * 32 * 4 * PC;
    static constexpr int kBytes = kZeroAt + MT * 32 * kZero;
};

// A warp: MT x 16 rows x NT x 8 tokens over its part of the inputs. PC scales of a row in 128 inputs; FB:
// blocks of 32 inputs after which a sum meets its scales.
template <int MT, int NT, int X, int PC, int FB>
__global__ void __launch_bounds__(kWarps * 32, 2) w4_stream_kernel(StreamArgs a) {
    using S = Stage4<MT, PC>;
    constexpr bool F16 = X >= kI8Row;
    constexpr int P = X == kF32x3 ? 3 : 1;
    extern __shared__ __align__(16) unsigned char s_mem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
    const int per = kWarps / a.ks, sub = warp % a.ks;
    const int chunks = (int)a.w.chunks, T = (int)a.x.tokens, rows = (int)(a.w.tile_rows / MT);
    const int c0 = (int)((long long)chunks * sub / a.ks), c1 = (int)((long long)chunks * (sub + 1) / a.ks);
    const bool zeros = a.w.zeros != nullptr;
    unsigned char* ring = s_mem + warp * S::kStages * S::kBytes;

    // The producer runs S::kStages - 1 tiles ahead of the sums, a chunk after the other.
    int p_tile = blockIdx.x, p_left = 0;
    const unsigned char *p_code = nullptr, *p_scale = nullptr, *p_zero = nullptr;
    auto p_start = [&]() {  // the pointers of the producer's next row of tiles, if there is one
        const int tr = p_tile * per + warp / a.ks;
        if (p_tile >= a.tiles || tr >= rows) return;
        const size_t at = ((size_t)(tr * MT >> 3) * chunks + c0) * 8 + (tr * MT & 7);
        p_code = reinterpret_cast<const unsigned char*>(a.w.codes) + at * 1024 + lane * 16;
        p_scale = reinterpret_cast<const unsigned char*>(a.w.scales) + (at * 8 + g) * (4 * PC);
        p_zero = reinterpret_cast<const unsigned char*>(a.w.zeros) + (at * 8 + g) * S::kZero;
        p_left = c1 - c0;
        p_tile += gridDim.x;
    };
    p_start();
    const uint32_t ring_u = (uint32_t)__cvta_generic_to_shared(ring);
    uint32_t p_dst = ring_u;
    auto produce = [&]() {
        if (p_left > 0) {
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                copy_async<16>(p_dst + m * 1024 + lane * 16, p_code + m * 1024);
                copy_async<16>(p_dst + m * 1024 + 512 + lane * 16, p_code + m * 1024 + 512);
                copy_async<4 * PC>(p_dst + S::kScaleAt + (m * 32 + lane) * 4 * PC, p_scale + m * (32 * PC));
                if (zeros) copy_async<S::kZero>(p_dst + S::kZeroAt + (m * 32 + lane) * S::kZero, p_zero + m * (8 * S::kZero));
            }
            p_code += 8192, p_scale += 256 * PC, p_zero += 64 * S::kZero;
            if (--p_left == 0) p_start();
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        p_dst = p_dst == ring_u + (S::kStages - 1) * S::kBytes ? ring_u : p_dst + S::kBytes;
    };
    // The weights do not depend on the kernel before, the activations may.
    for (int i = 0; i < S::kStages - 1; ++i) produce();
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const uint16_t* planes = a.planes;
    size_t ldp = a.ldp, plane = a.plane;
    if (!planes) {  // rows 64 bytes apart modulo 128: the 8 rows of a fragment load meet no bank twice
        uint16_t* sx = reinterpret_cast<uint16_t*>(s_mem + kWarps * S::kStages * S::kBytes);
        const int kp = chunks * kChunk;
        ldp = kp + 32;
        plane = T * ldp;
        for (int t = 0; t < T; ++t)
            for (int k = 8 * threadIdx.x; k < kp; k += 8 * kWarps * 32) {
                uint32_t v[P][4];
                x_pairs<P>(a.x, t, (k & ~31) + (k >> 2 & 6), 8, v);
#pragma unroll
                for (int p = 0; p < P; ++p)
                    *reinterpret_cast<uint4*>(sx + p * plane + t * ldp + k) = make_uint4(v[p][0], v[p][1], v[p][2], v[p][3]);
            }
        planes = sx;
        __syncthreads();
    }
    const uint16_t* xr[NT][P];  // a lane without a token repeats the last one's row: its sums are not stored
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int p = 0; p < P; ++p) xr[n][p] = planes + (size_t)min(8 * n + g, T - 1) * ldp + p * plane + 8 * q;
    const float* xs[NT][2];  // X == kI8Group: the scales of tokens 8 n + 2 q, + 1
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) xs[n][e] = a.x.scales + (size_t)min(8 * n + 2 * q + e, T - 1) * a.x.n_groups;

    const unsigned char* st = ring;
    for (int tile = blockIdx.x; tile < a.tiles; tile += gridDim.x) {
        const int tr = tile * per + warp / a.ks;
        const bool has = tr < rows;
        float acc[MT][NT][4], ga[MT][NT][4];
#pragma unroll
        for (int i = 0; i < MT * NT * 4; ++i) acc[i / (4 * NT)][i / 4 % NT][i % 4] = ga[i / (4 * NT)][i / 4 % NT][i % 4] = 0.f;
        for (int c = c0; has && c < c1; ++c) {
            asm volatile("cp.async.wait_group %0;" ::"n"(S::kStages - 2) : "memory");
            produce();  // into the stage of the tile before this one
            uint4 va[MT], vb[MT];
            uint32_t zz[MT][(PC + 1) / 2], sc[MT][PC];
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                va[m] = *reinterpret_cast<const uint4*>(st + m * 1024 + lane * 16);
                vb[m] = *reinterpret_cast<const uint4*>(st + m * 1024 + 512 + lane * 16);
#pragma unroll
                for (int i = 0; i < PC; ++i)
                    sc[m][i] = *reinterpret_cast<const uint32_t*>(st + S::kScaleAt + ((m * 32 + lane) * PC + i) * 4);
#pragma unroll
                for (int i = 0; i < (PC + 1) / 2; ++i)
                    zz[m][i] = zeros ? *reinterpret_cast<const uint32_t*>(st + S::kZeroAt + (m * 32 + lane) * S::kZero + 4 * i)
                                     : 0x08080808u;
            }
            st = st == ring + (S::kStages - 1) * S::kBytes ? ring : st + S::kBytes;
            Zero<F16> za[MT], zb[MT];
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                constexpr int kPer = 4 / PC;  // blocks of a scale
                const int blk = b / kPer;
                uint32_t f[MT][2][4];
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    if (b % kPer == 0) {
                        const uint32_t z2 = zz[m][blk / 2] >> (16 * (blk & 1));
                        za[m].set(z2 & 0xffu), zb[m].set((z2 >> 8) & 0xffu);
                    }
                    uint32_t pa[4], pb[4];
                    code_pairs<F16>(b == 0 ? va[m].x : b == 1 ? va[m].y : b == 2 ? va[m].z : va[m].w, za[m], pa);
                    code_pairs<F16>(b == 0 ? vb[m].x : b == 1 ? vb[m].y : b == 2 ? vb[m].z : vb[m].w, zb[m], pb);
#pragma unroll
                    for (int i = 0; i < 4; ++i) f[m][i >> 1][2 * (i & 1)] = pa[i], f[m][i >> 1][2 * (i & 1) + 1] = pb[i];
                }
#pragma unroll
                for (int n = 0; n < NT; ++n) {
#pragma unroll
                    for (int p = 0; p < P; ++p) {
                        const uint4 xf = *reinterpret_cast<const uint4*>(xr[n][p] + c * kChunk + 32 * b);
#pragma unroll
                        for (int m = 0; m < MT; ++m) {
                            mma16816<F16>(ga[m][n], f[m][0], xf.x, xf.y);
                            mma16816<F16>(ga[m][n], f[m][1], xf.z, xf.w);
                        }
                    }
                }
                if ((b + 1) % FB == 0) {
                    float x0[NT], x1[NT];
                    if constexpr (X == kI8Group) {
                        const int xi = (c * kChunk + 32 * b) >> a.x.group_shift;
                        const int at = min(xi, (int)a.x.n_groups - 1);  // padded inputs: the weights' scale is 0
#pragma unroll
                        for (int n = 0; n < NT; ++n) x0[n] = __ldg(xs[n][0] + at), x1[n] = __ldg(xs[n][1] + at);
                    }
#pragma unroll
                    for (int m = 0; m < MT; ++m) {
                        const float s0 = scale_of(sc[m][blk] & 0xffffu, a.w.scale_bf16), s1 = scale_of(sc[m][blk] >> 16, a.w.scale_bf16);
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            if constexpr (X == kI8Group)
                                ga[m][n][0] *= x0[n], ga[m][n][1] *= x1[n], ga[m][n][2] *= x0[n], ga[m][n][3] *= x1[n];
                            acc[m][n][0] = fmaf(ga[m][n][0], s0, acc[m][n][0]);
                            acc[m][n][1] = fmaf(ga[m][n][1], s0, acc[m][n][1]);
                            acc[m][n][2] = fmaf(ga[m][n][2], s1, acc[m][n][2]);
                            acc[m][n][3] = fmaf(ga[m][n][3], s1, acc[m][n][3]);
#pragma unroll
                            for (int e = 0; e < 4; ++e) ga[m][n][e] = 0.f;
                        }
                    }
                }
            }
        }
        if (a.ks > 1) {  // the warps of a row of tiles: their sums in order, by the first of them
            float* mine = reinterpret_cast<float*>(s_mem) + a.sums_at + (size_t)warp * 32 * 4 * NT * MT;
            if (sub) {
#pragma unroll
                for (int i = 0; i < 4 * NT * MT; ++i) mine[i * 32 + lane] = acc[i / (4 * NT)][i / 4 % NT][i % 4];
            }
            __syncthreads();
            if (!sub) {
                for (int j = 1; j < a.ks; ++j)
#pragma unroll
                    for (int i = 0; i < 4 * NT * MT; ++i)
                        acc[i / (4 * NT)][i / 4 % NT][i % 4] += mine[(size_t)j * 32 * 4 * NT * MT + i * 32 + lane];
            }
            __syncthreads();
        }
        if (has && !sub) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const size_t t = 8 * n + 2 * q + (e & 1);
                    if (t >= a.x.tokens) continue;
                    const float xscale = X == kI8Row ? a.x.scales[t] : 1.f;
#pragma unroll
                    for (int m = 0; m < MT; ++m) {
                        const size_t r = ((size_t)tr * MT + m) * 16 + g + 8 * (e >> 1);
                        if (r >= a.w.n_out) continue;
                        const float v = X == kI8Row ? acc[m][n][e] * xscale : acc[m][n][e];
                        if (a.y_bf16)
                            static_cast<__nv_bfloat16*>(a.y)[t * a.w.n_out + r] = __float2bfloat16_rn(v);
                        else
                            static_cast<float*>(a.y)[t * a.w.n_out + r] = v;
                    }
                }
        }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
}

// Shared memory for the activations' planes, beside the ring.
constexpr size_t kPlaneSmem = 48 * 1024;

struct StreamPlan {
    int num_sms;
    size_t plane_bytes;  // of the planes in shared memory
    bool pdl;            // launched as a programmatic dependent of the planes' kernel
};

template <int MT, int NT, int X, int PC, int FB>
cudaError_t run_stream(StreamArgs& a, const StreamPlan& pl, cudaStream_t s) {
    auto kernel = w4_stream_kernel<MT, NT, X, PC, FB>;
    const size_t ring = (size_t)kWarps * Stage4<MT, PC>::kStages * Stage4<MT, PC>::kBytes;
    const size_t sums = kWarps * 32 * 4 * NT * MT * sizeof(float);
    const int resident = ring + pl.plane_bytes + sums <= 112 * 1024 ? 2 : 1;
    // Warps that share a row of tiles: the split with the shortest chain of tiles for a warp, where a round
    // costs about as much as 3 tiles (its first loads, its sums joined).
    const size_t rows = a.w.tile_rows / MT, ctas = (size_t)pl.num_sms * resident;
    int ks = 1;
    size_t best = ~size_t(0);
    for (int k = 1; k <= kWarps && (size_t)k <= a.w.chunks; k *= 2) {
        const size_t tiles = (rows + kWarps / k - 1) / (kWarps / k);
        const size_t cost = (tiles + ctas - 1) / ctas * ((a.w.chunks + k - 1) / k + 3);
        if (cost < best) best = cost, ks = k;
    }
    a.ks = ks;
    a.tiles = (int)((rows + kWarps / ks - 1) / (kWarps / ks));
    a.sums_at = (int)((ring + pl.plane_bytes) / sizeof(float));
    const size_t smem = ring + pl.plane_bytes + (ks > 1 ? sums : 0);
    static SmemOnce once;  // the most this kernel is ever given
    const cudaError_t e = once.set(reinterpret_cast<const void*>(kernel), (int)(ring + kPlaneSmem + sums));
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)std::min(a.tiles, pl.num_sms * resident));
    cfg.blockDim = dim3(kWarps * 32);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &at;
    cfg.numAttrs = pl.pdl ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, a);
}
template <int MT, int NT, int X>
cudaError_t run_pc(StreamArgs& a, const StreamPlan& pl, cudaStream_t s) {
    const int pc = a.w.per_chunk;
    if constexpr (X == kI8Group)  // groups of activations smaller than the weights': scales every 32 inputs
        if (a.x.group * pc < kChunk) return pc == 1 ? run_stream<MT, NT, X, 1, 1>(a, pl, s) : run_stream<MT, NT, X, 2, 1>(a, pl, s);
    return pc == 1   ? run_stream<MT, NT, X, 1, 4>(a, pl, s)
           : pc == 2 ? run_stream<MT, NT, X, 2, 2>(a, pl, s)
                     : run_stream<MT, NT, X, 4, 1>(a, pl, s);
}
template <int X>
cudaError_t run_nt(StreamArgs& a, const StreamPlan& pl, cudaStream_t s) {
    // Two row tiles a warp share the activations' fragments and the loop's overhead; one tile a warp where
    // that would leave SMs without a full CTA.
    if (a.x.tokens <= 8)
        return a.w.tile_rows < (size_t)pl.num_sms * 2 * kWarps ? run_pc<1, 1, X>(a, pl, s) : run_pc<2, 1, X>(a, pl, s);
    return a.x.tokens <= 16 ? run_pc<2, 2, X>(a, pl, s) : run_pc<1, 4, X>(a, pl, s);
}

int terms_of(const W4X& x) { return x.kind == kW4XF32 ? 3 : 1; }
size_t plane_smem(const W4View& w, const W4X& x, size_t tokens) {
    return terms_of(x) * tokens * (w.chunks * kChunk + 32) * sizeof(uint16_t);
}
constexpr size_t kStreamTokens = 32;  // of one launch

}  // namespace

cudaError_t launch_w4_pack(const uint8_t* codes, const unsigned short* scales, const uint8_t* zeros, const W4View& w,
                           uint32_t* out_c, unsigned short* out_s, uint8_t* out_z, int* bad, cudaStream_t s) {
    const size_t words = w.tile_rows * w.chunks * 256;
    w4_pack_kernel<<<(unsigned)((words + 255) / 256), 256, 0, s>>>(codes, scales, zeros, w, out_c, out_s, out_z, bad);
    return cudaGetLastError();
}

size_t w4_stream_workspace(const W4View& w, const W4X& x) {
    if (plane_smem(w, x, std::min(x.tokens, kStreamTokens)) <= kPlaneSmem) return 0;
    return terms_of(x) * x.tokens * w.chunks * kChunk * sizeof(uint16_t);
}

cudaError_t launch_w4_stream(const W4View& w, const W4X& x, void* y, int y_bf16, void* workspace, int num_sms,
                             cudaStream_t s) {
    StreamArgs a{};
    a.w = w;
    a.y_bf16 = y_bf16;
    const bool planes = w4_stream_workspace(w, x) > 0;
    if (planes) {
        const size_t kp = w.chunks * kChunk;
        uint16_t* out = static_cast<uint16_t*>(workspace);
        const dim3 grid((unsigned)std::min<size_t>((kp / 8 + 255) / 256, 64), (unsigned)std::min<size_t>(x.tokens, 65535));
        if (x.kind == kW4XF32)
            w4_planes_kernel<3><<<grid, 256, 0, s>>>(x, kp, out);
        else
            w4_planes_kernel<1><<<grid, 256, 0, s>>>(x, kp, out);
        const cudaError_t e = cudaGetLastError();
        if (e != cudaSuccess) return e;
        a.planes = out;
        a.ldp = kp;
        a.plane = x.tokens * kp;
    }
    const size_t es = x.kind == kW4XF32 ? 4 : x.kind == kW4XBf16 ? 2 : 1;
    for (size_t t = 0; t < x.tokens; t += kStreamTokens) {
        StreamArgs b = a;
        b.x = x;
        b.x.x = static_cast<const char*>(x.x) + t * x.stride * es;
        b.x.tokens = std::min(kStreamTokens, x.tokens - t);
        b.x.scales = x.scales ? x.scales + t * x.n_groups : nullptr;
        if (a.planes) b.planes = a.planes + t * a.ldp;
        b.y = y_bf16 ? static_cast<void*>(static_cast<__nv_bfloat16*>(y) + t * w.n_out)
                     : static_cast<void*>(static_cast<float*>(y) + t * w.n_out);
        const StreamPlan pl{num_sms, a.planes ? 0 : plane_smem(w, x, b.x.tokens), planes && t == 0};
        const cudaError_t e = x.kind == kW4XF32    ? run_nt<kF32x3>(b, pl, s)
                              : x.kind == kW4XBf16 ? run_nt<kBf16>(b, pl, s)
                              : x.group > 0        ? run_nt<kI8Group>(b, pl, s)
                                                   : run_nt<kI8Row>(b, pl, s);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

}  // namespace bebelm
