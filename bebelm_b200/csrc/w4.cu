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
// Layout: rows padded to 128, inputs to 128 (scale 0). A tile of 16 rows x 128 inputs is 1024
// bytes, [row / 8][row % 8][q = 0..3][b = 0..3] words of 8 codes: word (q, b) of a row holds inputs
// 32 b + 8 q .. + 7, in the nibble order 0 2 4 6 1 3 5 7 (low first), so that (w >> 4 i) & 0x000f000f
// are inputs 2 i and 2 i + 1. Lane (g, q) of a warp reads its row's 16 bytes: for each
// 32-input block b it holds 8 inputs of rows g and g + 8, two m16n8k16 A fragments whose inputs are in
// another order than the fragment's; the activations are read in the same order, 16 bytes a
// block, and the sum does not mind. Blocks of 32 inputs stay whole, so a group of 32 ends with an MMA.
// Scales [tile row][chunk][block of min(group, 128)][row % 8][row / 8], zero points the same in bytes.
#include <algorithm>
#include <cstdint>

#include "internal.h"

namespace bebelm {
namespace {

constexpr int kWarps = 8;      // of a CTA
constexpr int kDepth = 4;      // 1 KB tiles in flight per warp
constexpr int kChunk = 128;    // inputs of a tile

__device__ __forceinline__ uint32_t code_pair(uint32_t w, int i, uint32_t zz) {
    const uint32_t u = ((w >> (4 * i)) & 0x000f000fu) | 0x43004300u;  // bf16 pair 128 + c
    __nv_bfloat162 a = *reinterpret_cast<const __nv_bfloat162*>(&u), b = *reinterpret_cast<const __nv_bfloat162*>(&zz);
    a = __hsub2(a, b);  // exact: both are integers in [128, 255]
    return *reinterpret_cast<const uint32_t*>(&a);
}

__device__ __forceinline__ void mma16816(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
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

// The activations as bf16 planes, [P][tokens][kp] with zeros past n_in.
template <int P>
__global__ void __launch_bounds__(256) w4_planes_kernel(W4X x, size_t kp, __nv_bfloat16* out) {
    asm volatile("griddepcontrol.launch_dependents;");
    const size_t plane = x.tokens * kp;
    for (size_t t = blockIdx.y; t < x.tokens; t += gridDim.y)
        for (size_t k = 2 * ((size_t)blockIdx.x * blockDim.x + threadIdx.x); k < kp; k += 2 * (size_t)gridDim.x * blockDim.x) {
            uint32_t a[3] = {0, 0, 0}, b[3] = {0, 0, 0};
            if (k < x.n_in) {  // n_in is even
                if (x.kind == kW4XF32) {
                    const float* p = static_cast<const float*>(x.x) + t * x.stride + k;
                    split3(p[0], a), split3(p[1], b);
                } else if (x.kind == kW4XInt8) {
                    const signed char* p = static_cast<const signed char*>(x.x) + t * x.stride + k;
                    a[0] = __float_as_uint((float)p[0]), b[0] = __float_as_uint((float)p[1]);
                } else {
                    const unsigned short* p = static_cast<const unsigned short*>(x.x) + t * x.stride + k;
                    a[0] = (uint32_t)p[0] << 16, b[0] = (uint32_t)p[1] << 16;
                }
            }
#pragma unroll
            for (int i = 0; i < P; ++i)
                *reinterpret_cast<uint32_t*>(out + i * plane + t * kp + k) = (a[i] >> 16) | (b[i] & 0xffff0000u);
        }
}

// codes [n_out][n_in / 2], scales and zeros [n_out][n_in / group] into the layout above, a
// thread per word of 8 codes
__global__ void __launch_bounds__(256) w4_pack_kernel(const uint8_t* codes, const unsigned short* scales,
                                                      const uint8_t* zeros, W4View w, uint32_t* out_c,
                                                      unsigned short* out_s, uint8_t* out_z, int* bad) {
    const size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x;  // word of out_c
    const size_t tile = i >> 8, tr = tile / w.chunks, c = tile % w.chunks;
    if (tr >= w.tile_rows) return;
    const int in = (int)(i & 255), b = in & 3, q = (in >> 2) & 3, r = in >> 4;  // r = 8 (row / 8) + row % 8
    const size_t row = tr * 16 + r, k = c * kChunk + 32 * b + 8 * q;
    uint32_t v = 0;
    if (row < w.n_out && k < w.n_in) {
        const uint8_t* p = codes + row * (w.n_in / 2) + k / 2;
        for (int j = 0; j < 4; ++j) v |= (uint32_t)(p[j] & 15) << (4 * j) | (uint32_t)(p[j] >> 4) << (4 * j + 16);
    }
    out_c[i] = v;
    if (q == 0 && b < w.per_chunk) {  // one scale per (row, block of min(group, 128) inputs)
        const size_t ks = c * kChunk + (size_t)b * (kChunk / w.per_chunk);
        const size_t o = (tile * w.per_chunk + b) * 16 + (r & 7) * 2 + (r >> 3);
        const bool in_range = row < w.n_out && ks < w.n_in;
        const size_t g = row * (w.n_in / w.group) + ks / w.group;
        out_s[o] = in_range ? scales[g] : 0;
        if (out_z) {
            out_z[o] = in_range ? zeros[g] : 8;
            if (out_z[o] > 127) *bad = 1;
        }
    }
}

struct StreamArgs {
    W4View w;
    W4X x;
    const __nv_bfloat16* planes;  // [P][x.tokens][ldp], 16-byte aligned rows
    size_t ldp, plane, k_end;     // elements of a plane; inputs at and past k_end count as zero
    void* y;
    int y_bf16, ks, tiles;        // ks warps share a row of tiles; `tiles` groups of kWarps / ks of them
};

// A warp: 16 rows x NT x 8 tokens over its part of the inputs.
template <int NT, int P, bool ASYM>
__global__ void __launch_bounds__(kWarps * 32) w4_stream_kernel(StreamArgs a) {
    extern __shared__ float s_red[];  // [kWarps][32][4 NT], only used when ks > 1
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
    const int per = kWarps / a.ks, sub = warp % a.ks, pc = a.w.per_chunk;
    const int chunks = (int)a.w.chunks, T = (int)a.x.tokens;
    const int c0 = (int)((long long)chunks * sub / a.ks), c1 = (int)((long long)chunks * (sub + 1) / a.ks);
    const bool grouped = a.x.kind == kW4XInt8 && a.x.group > 0;
    // blocks of 32 inputs after which a sum meets its scales
    int fb = 4 / pc;
    if (grouped) fb = min(fb, a.x.group / 32);
    const __nv_bfloat16* xr[NT];
    bool live[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        live[n] = 8 * n + g < T;
        xr[n] = a.planes + (size_t)(live[n] ? 8 * n + g : 0) * a.ldp + 8 * q;
    }
    bool waited = false;
    for (int tile = blockIdx.x; tile < a.tiles; tile += gridDim.x) {
        const size_t tr = (size_t)tile * per + warp / a.ks;
        const bool has = tr < a.w.tile_rows;
        float acc[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[n][e] = 0.f;
        if (has) {
            const uint4* wp = a.w.codes + tr * chunks * 64 + lane;
            const uint32_t* sp = a.w.scales + tr * chunks * pc * 8 + g;
            const unsigned short* zp = ASYM ? a.w.zeros + tr * chunks * pc * 8 + g : nullptr;
            uint4 wa[kDepth], wb[kDepth];
#pragma unroll
            for (int d = 0; d < kDepth; ++d)
                if (c0 + d < c1) wa[d] = __ldcs(wp + (size_t)(c0 + d) * 64), wb[d] = __ldcs(wp + (size_t)(c0 + d) * 64 + 32);
            if (!waited) {  // the weights do not depend on the kernel before, the planes may
                asm volatile("griddepcontrol.wait;" ::: "memory");
                waited = true;
            }
            float ga[NT][4];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) ga[n][e] = 0.f;
            for (int cb = c0; cb < c1; cb += kDepth) {
#pragma unroll
                for (int d = 0; d < kDepth; ++d) {
                    const int c = cb + d;
                    if (c >= c1) break;
                    const uint32_t va[4] = {wa[d].x, wa[d].y, wa[d].z, wa[d].w};
                    const uint32_t vb[4] = {wb[d].x, wb[d].y, wb[d].z, wb[d].w};
                    if (c + kDepth < c1)
                        wa[d] = __ldcs(wp + (size_t)(c + kDepth) * 64), wb[d] = __ldcs(wp + (size_t)(c + kDepth) * 64 + 32);
                    uint32_t s2 = 0, z2a = 0x43084308u, z2b = 0x43084308u;
#pragma unroll
                    for (int b = 0; b < 4; ++b) {
                        const int blk = b * pc / 4;  // scale block of the chunk
                        if (b * pc % 4 == 0) {
                            s2 = sp[((size_t)c * pc + blk) * 8];
                            if constexpr (ASYM) {
                                const uint32_t zb = zp[((size_t)c * pc + blk) * 8];
                                z2a = (0x4300u | (zb & 0xffu)) * 0x10001u;
                                z2b = (0x4300u | (zb >> 8)) * 0x10001u;
                            }
                        }
                        uint32_t pa[4], pb[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) pa[i] = code_pair(va[b], i, z2a), pb[i] = code_pair(vb[b], i, z2b);
                        const uint32_t f0[4] = {pa[0], pb[0], pa[1], pb[1]}, f1[4] = {pa[2], pb[2], pa[3], pb[3]};
                        const size_t k = (size_t)c * kChunk + 32 * b;
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
#pragma unroll
                            for (int p = 0; p < P; ++p) {
                                uint4 xf = make_uint4(0, 0, 0, 0);
                                if (live[n] && k < a.k_end) xf = *reinterpret_cast<const uint4*>(xr[n] + p * a.plane + k);
                                mma16816(ga[n], f0, xf.x, xf.y);
                                mma16816(ga[n], f1, xf.z, xf.w);
                            }
                        }
                        if ((b + 1) % fb == 0) {
                            const float s0 = scale_of(s2 & 0xffffu, a.w.scale_bf16), s1 = scale_of(s2 >> 16, a.w.scale_bf16);
#pragma unroll
                            for (int n = 0; n < NT; ++n) {
                                float x0 = 1.f, x1 = 1.f;
                                if (grouped) {  // tokens 8 n + 2 q, + 1
                                    const size_t xi = k >> a.x.group_shift;
                                    const int t0 = 8 * n + 2 * q;
                                    x0 = t0 < T && k < a.x.n_in ? a.x.scales[(size_t)t0 * a.x.n_groups + xi] : 0.f;
                                    x1 = t0 + 1 < T && k < a.x.n_in ? a.x.scales[(size_t)(t0 + 1) * a.x.n_groups + xi] : 0.f;
                                }
                                acc[n][0] = fmaf(ga[n][0] * x0, s0, acc[n][0]);
                                acc[n][1] = fmaf(ga[n][1] * x1, s0, acc[n][1]);
                                acc[n][2] = fmaf(ga[n][2] * x0, s1, acc[n][2]);
                                acc[n][3] = fmaf(ga[n][3] * x1, s1, acc[n][3]);
#pragma unroll
                                for (int e = 0; e < 4; ++e) ga[n][e] = 0.f;
                            }
                        }
                    }
                }
            }
        }
        if (a.ks > 1) {  // the warps of a row of tiles: their sums in order, by the first of them
            float* mine = s_red + (size_t)warp * 32 * 4 * NT;
            if (sub) {
#pragma unroll
                for (int i = 0; i < 4 * NT; ++i) mine[i * 32 + lane] = acc[i / 4][i % 4];
            }
            __syncthreads();
            if (!sub) {
                for (int j = 1; j < a.ks; ++j)
#pragma unroll
                    for (int i = 0; i < 4 * NT; ++i) acc[i / 4][i % 4] += mine[(size_t)j * 32 * 4 * NT + i * 32 + lane];
            }
            __syncthreads();
        }
        if (has && !sub) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const size_t t = 8 * n + 2 * q + (e & 1), r = tr * 16 + g + 8 * (e >> 1);
                    if (t >= a.x.tokens || r >= a.w.n_out) continue;
                    float v = acc[n][e];
                    if (a.x.kind == kW4XInt8 && !grouped) v *= a.x.scales[t];
                    if (a.y_bf16)
                        static_cast<__nv_bfloat16*>(a.y)[t * a.w.n_out + r] = __float2bfloat16_rn(v);
                    else
                        static_cast<float*>(a.y)[t * a.w.n_out + r] = v;
                }
        }
    }
    if (!waited) asm volatile("griddepcontrol.wait;" ::: "memory");
}

template <int NT, int P>
cudaError_t run_stream(const StreamArgs& a, int grid, bool pdl, cudaStream_t s) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(kWarps * 32);
    cfg.dynamicSmemBytes = a.ks > 1 ? kWarps * 32 * 4 * NT * sizeof(float) : 0;
    cfg.stream = s;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &at;
    cfg.numAttrs = pdl ? 1 : 0;
    return a.w.zeros ? cudaLaunchKernelEx(&cfg, w4_stream_kernel<NT, P, true>, a)
                     : cudaLaunchKernelEx(&cfg, w4_stream_kernel<NT, P, false>, a);
}

bool direct_x(const W4X& x) {  // rows that can be read as they are, 16 bytes at a time
    return x.kind == kW4XBf16 && (reinterpret_cast<uintptr_t>(x.x) & 15) == 0 && x.stride % 8 == 0;
}

}  // namespace

cudaError_t launch_w4_pack(const uint8_t* codes, const unsigned short* scales, const uint8_t* zeros, const W4View& w,
                           uint32_t* out_c, unsigned short* out_s, uint8_t* out_z, int* bad, cudaStream_t s) {
    const size_t words = w.tile_rows * w.chunks * 256;
    w4_pack_kernel<<<(unsigned)((words + 255) / 256), 256, 0, s>>>(codes, scales, zeros, w, out_c, out_s, out_z, bad);
    return cudaGetLastError();
}

cudaError_t launch_w4_planes(const W4X& x, size_t kp, __nv_bfloat16* out, cudaStream_t s) {
    const dim3 grid((unsigned)std::min<size_t>((kp / 2 + 255) / 256, 64), (unsigned)std::min<size_t>(x.tokens, 65535));
    if (x.kind == kW4XF32)
        w4_planes_kernel<3><<<grid, 256, 0, s>>>(x, kp, out);
    else
        w4_planes_kernel<1><<<grid, 256, 0, s>>>(x, kp, out);
    return cudaGetLastError();
}

size_t w4_workspace(const W4View& w, const W4X& x) {
    if (direct_x(x)) return 0;
    return (x.kind == kW4XF32 ? 3 : 1) * x.tokens * w.chunks * kChunk * sizeof(__nv_bfloat16);
}

cudaError_t launch_w4_stream(const W4View& w, const W4X& x, void* y, int y_bf16, void* workspace, int num_sms,
                             cudaStream_t s) {
    StreamArgs a{};
    a.w = w;
    a.y_bf16 = y_bf16;
    const size_t kp = w.chunks * kChunk;
    const bool direct = direct_x(x);
    if (direct) {
        a.planes = static_cast<const __nv_bfloat16*>(x.x);
        a.ldp = x.stride;
        a.k_end = w.n_in;
    } else {
        cudaError_t e = launch_w4_planes(x, kp, static_cast<__nv_bfloat16*>(workspace), s);
        if (e != cudaSuccess) return e;
        a.planes = static_cast<const __nv_bfloat16*>(workspace);
        a.ldp = kp;
        a.plane = x.tokens * kp;
        a.k_end = kp;
    }
    // warps that share a row of tiles: enough for two CTAs an SM, as long as each keeps two tiles
    int ks = 1;
    while (ks < kWarps && w.tile_rows * ks < (size_t)num_sms * 2 * kWarps && w.chunks >= (size_t)ks * 4) ks *= 2;
    a.ks = ks;
    a.tiles = (int)((w.tile_rows + kWarps / ks - 1) / (kWarps / ks));
    const int grid = std::min(a.tiles, num_sms * 4);
    for (size_t t = 0; t < x.tokens; t += 32) {
        a.x = x;
        a.x.tokens = std::min<size_t>(32, x.tokens - t);
        a.x.scales = x.scales ? x.scales + t * x.n_groups : nullptr;
        StreamArgs b = a;
        b.planes = a.planes + t * a.ldp;
        b.y = y_bf16 ? static_cast<void*>(static_cast<__nv_bfloat16*>(y) + t * w.n_out)
                     : static_cast<void*>(static_cast<float*>(y) + t * w.n_out);
        const bool pdl = !direct && t == 0;
        const size_t n = b.x.tokens;
        cudaError_t e;
        if (x.kind == kW4XF32)
            e = n <= 8 ? run_stream<1, 3>(b, grid, pdl, s) : n <= 16 ? run_stream<2, 3>(b, grid, pdl, s)
                                                                     : run_stream<4, 3>(b, grid, pdl, s);
        else
            e = n <= 8 ? run_stream<1, 1>(b, grid, pdl, s) : n <= 16 ? run_stream<2, 1>(b, grid, pdl, s)
                                                                     : run_stream<4, 1>(b, grid, pdl, s);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

}  // namespace bebelm
