// Products with 4-bit weights and group scales, few tokens (w4_stream_kernel), and the weights'
// layout (w4_pack_kernel) that the many-token kernel (w4_tc.cu) shares.
//
//     y[t][n] = Σ_g s[n][g] · sx[t][g'] · Σ_{k in g} (c[n][k] - z[n][g]) · x[t][k]
//
// with 4-bit codes c, a zero point z (8 when the weights have none), a scale s per group of one
// row's weights, and for int8 activations a scale sx per row or per x_group values of a token.
//
// The inner sum runs on the tensor cores in whole numbers (m16n8k32, u8 x s8 -> s32), exactly. int8 activations are
// one such product. bf16 and f32 activations are made whole per token and 128 inputs: X = round(x · 2^e), e chosen
// so that the largest |X| is in (2^21.99, 2^22.99), and X = 65536 d1 + 256 d2 + d3 with d in [-128, 127]: three
// products. That keeps an activation to 2^-23 of the largest of its 128 (half a step of X). Where the largest is at most
// 8 times the mean magnitude (6 standard deviations of normal values) that is 2^-20 of the mean, and a sum's error is that of f32
// sums. Where it is more, a few far larger activations would leave the rest few bits that the weights may yet see alone: there
// what rounding left is kept too, in units of 2^-15, as two more digits and products: 2^-38 of the largest. They cost 33 to
// 50 % of a call's time (2048 x 2048 4.4 -> 6.6 us, 8192 x 8192 12.3 -> 16.7 us, 128000 x 2048 32.4 -> 40.6 us, each with
// two such activations a token), and run in a loop of their own, since in one loop they took 1 us of the others' time. A chunk
// with an infinity or a NaN is a NaN.
// z is taken off as z · Σ X, also whole: the accumulators start at -z Σ d, plus the bits of 1.5 · 2^23, so that they
// are read as floats without a conversion (|Σ (c - z) d| <= 127 · 128 · 128 < 2^22). A flush per group makes a float of
// the digits and applies the scales in f32.
//
// Bound: a weight is read once, for at most 16 tokens, so HBM. On the way a weight costs 3/8 of a logic operation (two
// masks and a shift for a word of 8 codes); unpacked to 16-bit floats it cost 11/8 and the logic unit bound the
// kernel. Measured (with 16-bit floats): 128000 x 2048, 5 int8 tokens 27.7 us (44), 138 MB at 5.0 TB/s, 76 % of a
// copy's rate; 8192 x 8192, one bf16 token 12.4 us (16), 35 MB at 2.8 TB/s: every CTA makes the digits first, with the
// ring's first weights in flight; 2048 x 2048, one f32 token 4.4 us, all latency.
//
// Layout: rows padded to 128, inputs to 128 (scale 0). A tile of 16 rows x 128 inputs is 1024 bytes,
// [row / 8][row % 8][q = 0..3][b = 0..3] words of 8 codes; the 8 tiles of 128 rows lie together, then the next 128
// inputs. Word (q, b) of a row holds inputs 32 b + 8 j + 2 q + e (j = 0..3, e = 0, 1) in nibble j + 4 e. Here its low
// and high nibbles are the two words that lane (g, q) of a warp gives to an MMA for rows g (and g + 8) and 32 inputs, in
// some order of these inputs; the activations are laid out in the same order, 8 bytes a lane and 32 inputs. (w >> 4 j) &
// 0x000f000f is a pair of neighbours, which the other kernel uses.) Blocks of 32 inputs stay whole, so a
// group of 32 ends with an MMA. Scales [tile][row % 8][block of min(group, 128) inputs][row / 8], zero points the
// same in bytes: a lane's scales of a tile are one load.
#include <math_constants.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "internal.h"

namespace bebelm {
namespace {

constexpr int kWarps = 16;              // of a CTA, one an SM
constexpr int kChunk = 128;             // inputs of a tile
constexpr size_t kTokens = 16;          // the most of a call
constexpr int kMagicBits = 0x4B400000;  // 1.5 · 2^23: a float whose last bits are a whole number
constexpr float kMagic = 12582912.0f;

__device__ __forceinline__ void mma_u8s8(int* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float scale_of(uint32_t h, int bf16) {
    if (bf16) return __uint_as_float(h << 16);
    __half_raw r;
    r.x = (unsigned short)h;
    return __half2float(__half(r));
}

// The activations as digits, in shared memory or (where that is too small) the workspace: planes of rows of `row`
// bytes (1, or 3 and the 2 of the low digits), and a record per flush and token: the digits' sums and the scale,
// {Σ d, scale} or {Σ d1, Σ d2, Σ d3, scale}, and {Σ d4, Σ d5} apart. A scale below zero stands for its magnitude and
// says that the token has low digits in these 128 inputs; where it has none they are not written.
struct Digits {
    unsigned char *d, *records, *low;
    size_t row, plane;
};
constexpr int kLow = 2;  // low digits
__host__ __device__ constexpr int planes_of(int D) { return D == 3 ? 3 + kLow : D; }
__host__ __device__ inline size_t digit_row(size_t chunks) { return chunks * kChunk + 64; }  // 64 modulo 128: no bank twice
__host__ __device__ inline size_t even(size_t n) { return (n + 1) & ~size_t(1); }
__host__ __device__ inline size_t digit_bytes(int D, size_t tokens, size_t chunks, int fb) {
    return planes_of(D) * tokens * digit_row(chunks) + even(tokens) * chunks * (4 / fb) * (D == 3 ? 16 + 4 * kLow : 8);
}
__host__ __device__ inline Digits digits_at(unsigned char* p, int D, size_t tokens, size_t chunks, int fb) {
    Digits o;
    o.row = digit_row(chunks), o.plane = tokens * o.row;
    o.d = p, o.records = p + planes_of(D) * o.plane;
    o.low = o.records + even(tokens) * chunks * (4 / fb) * 16;
    return o;
}

// two neighbours; `pairs`: they are aligned to their size
__device__ __forceinline__ float2 x_pair(const W4X& x, size_t o, bool pairs) {
    if (x.kind == kW4XF32) {
        const float* p = static_cast<const float*>(x.x) + o;
        return pairs ? *reinterpret_cast<const float2*>(p) : make_float2(p[0], p[1]);
    }
    const unsigned short* p = static_cast<const unsigned short*>(x.x) + o;
    const uint32_t u = pairs ? *reinterpret_cast<const uint32_t*>(p) : (uint32_t)p[0] | (uint32_t)p[1] << 16;
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}
__device__ __forceinline__ bool x_pairs(const W4X& x) {
    const size_t to = x.kind == kW4XF32 ? 8 : 4;
    return x.stride % 2 == 0 && reinterpret_cast<uintptr_t>(x.x) % to == 0;
}

// 128 inputs of a token by half a warp: lane (b, q) the 8 of block b that lane q of an MMA gets, inputs 0, 16, 1, 17, 8,
// 24, 9, 25 from 32 b + 2 q. First the loads (of several chunks at a time), then the rest.
template <int D>
struct Eight {
    float v[D == 1 ? 1 : 8];
    uint32_t w[2];  // D = 1: the bytes
    float scale;
};
template <int D>
__device__ __forceinline__ void load_eight(Eight<D>& r, const W4X& x, bool pairs, int t, int c) {
    const int l = threadIdx.x & 15, k = c * kChunk + 32 * (l >> 2) + 2 * (l & 3);
    const bool in = (size_t)k < x.n_in;  // n_in is a multiple of 32
    const size_t base = (size_t)t * x.stride + k;
    if constexpr (D == 1) {
        constexpr int kAt[8] = {0, 16, 1, 17, 8, 24, 9, 25};
        r.w[0] = r.w[1] = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t v = in ? static_cast<const unsigned char*>(x.x)[base + kAt[i]] : 0u;
            r.w[i >> 2] |= v << (8 * (i & 3));
        }
        // padded inputs: any scale
        const int at = x.group ? min(k >> x.group_shift, (int)x.n_groups - 1) : 0;
        r.scale = x.scales[(size_t)t * x.n_groups + at];
    } else {
        constexpr int kAt[4] = {0, 16, 8, 24};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 u = in ? x_pair(x, base + kAt[i], pairs) : make_float2(0.f, 0.f);
            r.v[4 * (i >> 1) + (i & 1)] = u.x, r.v[4 * (i >> 1) + (i & 1) + 2] = u.y;
        }
    }
}
__device__ __forceinline__ float pow2(int i) { return __uint_as_float((uint32_t)(127 + i) << 23); }
// Of 128 inputs with the largest magnitude m (its bits): v -> X = round(v 2^27 2^e) if tiny, else round(v 2^e).
// 2^e takes the largest to 2^22 .. 2^23, or half of that where its digits would not fit; -105 <= e <= 122 here, up to 149
// with the 27 (2^-149 is the step of f32's smallest values, which are whole there).
struct Whole {
    int e;
    bool tiny, odd;  // odd: an infinity or a NaN among them
};
__device__ __forceinline__ Whole whole_of(uint32_t m) {
    Whole w;
    w.odd = m > 0x7f7fffffu;
    w.e = w.odd ? 0 : 22 - ((int)(m >> 23) - 127);
    w.tiny = w.e > 122;
    float most = __uint_as_float(m);
    if (w.tiny) most *= pow2(27), w.e -= 27;
    if (most * pow2(w.e) > 8355711.f) --w.e;  // 127 (65536 + 256 + 1)
    return w;
}
// Of four whole numbers, plus 128 each, the digits: byte `at` of each
__device__ __forceinline__ uint32_t bytes_of(const uint32_t* p, int at) {
    const uint32_t s = at == 2 ? 0x0062u : 0x5140u, a = __byte_perm(p[0], p[1], s), b = __byte_perm(p[2], p[3], s);
    return __byte_perm(a, b, at == 1 ? 0x7632 : 0x5410) ^ 0x80808080u;
}

// Whether the token has low digits among these 128 inputs is the answer (of half a warp).
template <int D, int FB>
__device__ __forceinline__ bool make_digits(Eight<D>& in, const W4X& x, const Digits& o, int t, int c) {
    const int l = threadIdx.x & 15, b = l >> 2, q = l & 3;
    uint32_t w[D][2];
    int sum[D];
    float scale;
    bool low = false;
    if constexpr (D == 1) {
        w[0][0] = in.w[0], w[0][1] = in.w[1], scale = in.scale;
        sum[0] = __dp4a((int)w[0][0], 0x01010101, __dp4a((int)w[0][1], 0x01010101, 0));
    } else {
        float* v = in.v;
        uint32_t m = 0;
        float total = 0.f;  // of the magnitudes, over 128
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);  // an infinity or a NaN is the largest
            total = fmaf(fabsf(v[i]), 1.f / kChunk, total);
        }
#pragma unroll
        for (int s = 8; s > 0; s >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, s)), total += __shfl_xor_sync(0xffffffffu, total, s);
        const Whole wh = whole_of(m);
        const bool odd = wh.odd, tiny = wh.tiny;
        const int e = wh.e;
        // the largest more than 8 times the mean
        low = !odd && __uint_as_float(m) * ((float)min(kChunk, (int)(x.n_in - (size_t)c * kChunk)) * (1.f / (8 * kChunk))) > total;
        if (tiny) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] *= pow2(27);
        }
        const float f = pow2(e);
        // X + 0x808080 has the digits + 128 as its bytes
        uint32_t u[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) u[i] = odd ? 0x808080u : (uint32_t)(__float2int_rn(v[i] * f) + 0x808080);
#pragma unroll
        for (int h = 0; h < 2; ++h) w[D - 1][h] = bytes_of(u + 4 * h, 0), w[D - 2][h] = bytes_of(u + 4 * h, 1), w[0][h] = bytes_of(u + 4 * h, 2);
#pragma unroll
        for (int d = 0; d < D; ++d) sum[d] = __dp4a((int)w[d][0], 0x01010101, __dp4a((int)w[d][1], 0x01010101, 0));
        scale = odd ? CUDART_NAN_F : tiny ? pow2(-e) * pow2(-27) : pow2(-e);
        if (low) scale = -scale;
    }
#pragma unroll
    for (int d = 0; d < D; ++d) {
        *reinterpret_cast<uint2*>(o.d + d * o.plane + t * o.row + c * kChunk + (b >> 1) * 64 + q * 16 + (b & 1) * 8) = make_uint2(w[d][0], w[d][1]);
#pragma unroll
        for (int s = 1; s < 4 * FB; s <<= 1) sum[d] += __shfl_xor_sync(0xffffffffu, sum[d], s);
    }
    if (l % (4 * FB) == 0) {
        unsigned char* r = o.records + ((size_t)(c * (4 / FB) + b / FB) * even(x.tokens) + t) * (D == 3 ? 16 : 8);
        if constexpr (D == 3)
            *reinterpret_cast<int4*>(r) = make_int4(sum[0], sum[1], sum[D - 1], __float_as_int(scale));
        else
            *reinterpret_cast<int2*>(r) = make_int2(sum[0], __float_as_int(scale));
    }
    return low;
}

// The low digits of the same 128 inputs, where `mine` says that the token has them: of what rounding to X left, at most 1/2, in
// units of 2^-15. By a whole warp.
template <int FB>
__device__ __forceinline__ void make_low(const Eight<3>& in, const W4X& x, const Digits& o, int t, int c, bool mine) {
    const int l = threadIdx.x & 15, b = l >> 2, q = l & 3;
    uint32_t m = 0, u[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(in.v[i]) & 0x7fffffffu);
#pragma unroll
    for (int s = 8; s > 0; s >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, s));
    const Whole wh = whole_of(m);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float y = (wh.tiny ? in.v[i] * pow2(27) : in.v[i]) * pow2(wh.e);
        u[i] = (uint32_t)(mine ? __float2int_rn((y - (float)__float2int_rn(y)) * 32768.f) + 0x8080 : 0x8080);
    }
    int sum[kLow];
#pragma unroll
    for (int d = 0; d < kLow; ++d) {
        const uint2 w = make_uint2(bytes_of(u, 1 - d), bytes_of(u + 4, 1 - d));
        sum[d] = __dp4a((int)w.x, 0x01010101, __dp4a((int)w.y, 0x01010101, 0));
#pragma unroll
        for (int s = 1; s < 4 * FB; s <<= 1) sum[d] += __shfl_xor_sync(0xffffffffu, sum[d], s);
        if (mine) *reinterpret_cast<uint2*>(o.d + (3 + d) * o.plane + t * o.row + c * kChunk + (b >> 1) * 64 + q * 16 + (b & 1) * 8) = w;
    }
    if (mine && l % (4 * FB) == 0)
        *reinterpret_cast<int2*>(o.low + ((size_t)(c * (4 / FB) + b / FB) * even(x.tokens) + t) * 8) = make_int2(sum[0], sum[1]);
}
// A record is read with its neighbour's: the one behind an odd number of tokens says that there are no low digits.
template <int FB>
__device__ __forceinline__ void end_records(const W4X& x, const Digits& o, int t, int c) {
    const int l = threadIdx.x & 15;
    if (x.tokens % 2 && t == (int)x.tokens - 1 && l < 4 / FB)
        *reinterpret_cast<float*>(o.records + ((size_t)(c * (4 / FB) + l) * even(x.tokens) + t + 1) * 16 + 12) = 0.f;
}

template <int D, int FB>
__global__ void __launch_bounds__(256) w4_digits_kernel(W4X x, int chunks, unsigned char* out) {
    asm volatile("griddepcontrol.launch_dependents;");
    const Digits o = digits_at(out, D, x.tokens, chunks, FB);
    // half a warp per 128 inputs of a token; whole warps stay in step
    const int n = (int)x.tokens * chunks;
    const bool pairs = x_pairs(x);
    for (int i = (blockIdx.x * 256 + threadIdx.x) >> 4; (i & ~1) < n; i += gridDim.x * 16) {
        const int j = min(i, n - 1);
        Eight<D> e;
        load_eight(e, x, pairs, j / chunks, j % chunks);
        const bool low = make_digits<D, FB>(e, x, o, j / chunks, j % chunks);
        if constexpr (D == 3) {
            if (__any_sync(0xffffffffu, low)) {
                load_eight(e, x, pairs, j / chunks, j % chunks);
                make_low<FB>(e, x, o, j / chunks, j % chunks, low);
            }
            end_records<FB>(x, o, j / chunks, j % chunks);
        }
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
    unsigned char* digits;   // in the workspace (WS), else made in shared memory
    void* y;
    int y_bf16, ks, tiles;   // 2^ks warps share a row of tiles; `tiles` groups of kWarps / 2^ks of them
    int digits_at, sums_at;  // in shared memory, behind the ring: the digits (bytes), the warps' partial sums (floats)
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
    static constexpr int kStages = MT == 1 ? (PC == 4 ? 4 : 5) : (PC == 4 ? 2 : 3);  // beside 60 KB of digits
    static constexpr int kZero = PC == 4 ? 8 : 4;  // bytes of zero points of a lane and tile (4 for PC 1: padded)
    static constexpr int kScaleAt = MT * 1024, kZeroAt = kScaleAt + MT * 32 * 4 * PC;
    static constexpr int kBytes = kZeroAt + MT * 32 * kZero;
};

// The producer of a warp's ring: it runs S::kStages - 1 tiles ahead of the sums, a chunk after the other.
template <int MT, int PC>
struct Producer {
    using S = Stage4<MT, PC>;
    int tile, left;
    const unsigned char *code, *scale, *zero;
    uint32_t ring, dst;

    // the pointers of the next row of tiles, if there is one
    __device__ __forceinline__ void start(const StreamArgs& a) {
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, sub = warp & ((1 << a.ks) - 1);
        const int chunks = (int)a.w.chunks, c0 = chunks * sub >> a.ks, c1 = chunks * (sub + 1) >> a.ks;
        const int tr = tile * (kWarps >> a.ks) + (warp >> a.ks);
        if (tile >= a.tiles || tr >= (int)(a.w.tile_rows / MT)) return;
        const size_t at = ((size_t)(tr * MT >> 3) * chunks + c0) * 8 + (tr * MT & 7);
        code = reinterpret_cast<const unsigned char*>(a.w.codes) + at * 1024 + lane * 16;
        scale = reinterpret_cast<const unsigned char*>(a.w.scales) + (at * 8 + g) * (4 * PC);
        zero = reinterpret_cast<const unsigned char*>(a.w.zeros) + (at * 8 + g) * S::kZero;
        left = c1 - c0;
        tile += gridDim.x;
    }
    __device__ __forceinline__ void next(const StreamArgs& a) {
        const int lane = threadIdx.x & 31;
        if (left > 0) {
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                copy_async<16>(dst + m * 1024 + lane * 16, code + m * 1024);
                copy_async<16>(dst + m * 1024 + 512 + lane * 16, code + m * 1024 + 512);
                copy_async<4 * PC>(dst + S::kScaleAt + (m * 32 + lane) * 4 * PC, scale + m * (32 * PC));
                if (a.w.zeros) copy_async<S::kZero>(dst + S::kZeroAt + (m * 32 + lane) * S::kZero, zero + m * (8 * S::kZero));
            }
            code += 8192, scale += 256 * PC, zero += 64 * S::kZero;
            if (--left == 0) start(a);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        dst = dst == ring + (S::kStages - 1) * S::kBytes ? ring : dst + S::kBytes;
    }
    __device__ __forceinline__ void fill(const StreamArgs& a, unsigned char* mem) {
        tile = blockIdx.x, left = 0, code = scale = zero = nullptr;
        ring = dst = (uint32_t)__cvta_generic_to_shared(mem);
        start(a);
        for (int i = 0; i < S::kStages - 1; ++i) next(a);
    }
};

// The tiles of a warp: MT x 16 rows x NT x 8 tokens over its part of the inputs. LOW: some token has low digits.
template <int MT, int NT, int D, int PC, int FB, bool WS, bool LOW>
__device__ __forceinline__ void stream_tiles(const StreamArgs& a, unsigned char* s_mem, unsigned char* ring, Producer<MT, PC>& p) {
    using S = Stage4<MT, PC>;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
    const int per = kWarps >> a.ks, sub = warp & ((1 << a.ks) - 1);
    const int chunks = (int)a.w.chunks, T = (int)a.x.tokens, rows = (int)(a.w.tile_rows / MT);
    const int c0 = chunks * sub >> a.ks, c1 = chunks * (sub + 1) >> a.ks;
    const bool zeros = a.w.zeros != nullptr;
    const Digits x = digits_at(WS ? a.digits : s_mem + a.digits_at, D, T, chunks, FB);
    constexpr int FL = 4 / FB, R = D == 3 ? 16 : 8;  // flushes of 128 inputs, bytes of a record
    // a lane without a token repeats the last one's row: its sums are not stored
    const unsigned char *xr[NT], *xq[NT], *xl[NT];
    const size_t step = even(T) * R;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        xr[n] = x.d + (size_t)min(8 * n + g, T - 1) * x.row + 16 * q + c0 * kChunk;
        xq[n] = x.records + min(8 * n + 2 * q, (int)even(T) - 2) * R + c0 * FL * step;
        xl[n] = x.low + min(8 * n + 2 * q, (int)even(T) - 2) * 8 + c0 * FL * (step / 2);
    }

    const unsigned char* st = ring;
    for (int tile = blockIdx.x; tile < a.tiles; tile += gridDim.x) {
        const int tr = tile * per + (warp >> a.ks);
        const bool has = tr < rows;
        float acc[MT][NT][4];
#pragma unroll
        for (int i = 0; i < MT * NT * 4; ++i) acc[i / (4 * NT)][i / 4 % NT][i % 4] = 0.f;
        for (int c = c0; has && c < c1; ++c) {
            asm volatile("cp.async.wait_group %0;" ::"n"(S::kStages - 2) : "memory");
            p.next(a);  // into the stage of the tile before this one
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
            const size_t at = (size_t)(c - c0);
            // 8 bytes for each of two blocks of 32 inputs
            uint4 xf[NT][D];
#pragma unroll
            for (int f = 0; f < FL; ++f) {
                const int blk = f * FB * PC / 4;  // scale block of the chunk
                int d[MT][NT][D][4];
                float xs[NT][2];
                int signs = 0;  // of the scales: below zero where a token has low digits here
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    int sums[2][D];  // of the digits of tokens 8 n + 2 q, + 1
                    const int4 r = *reinterpret_cast<const int4*>(xq[n] + (at * FL + f) * step);
                    if constexpr (D == 3) {
                        const int4 r1 = *reinterpret_cast<const int4*>(xq[n] + (at * FL + f) * step + 16);
                        sums[0][0] = r.x, sums[0][1] = r.y, sums[0][D - 1] = r.z, xs[n][0] = __int_as_float(r.w);
                        sums[1][0] = r1.x, sums[1][1] = r1.y, sums[1][D - 1] = r1.z, xs[n][1] = __int_as_float(r1.w);
                        signs |= r.w | r1.w;
                    } else {
                        sums[0][0] = r.x, xs[n][0] = __int_as_float(r.y);
                        sums[1][0] = r.z, xs[n][1] = __int_as_float(r.w);
                    }
#pragma unroll
                    for (int m = 0; m < MT; ++m) {
                        const uint32_t z2 = zz[m][blk / 2] >> (16 * (blk & 1));
                        const int z0 = -(int)(z2 & 0xffu), z1 = -(int)((z2 >> 8) & 0xffu);
#pragma unroll
                        for (int i = 0; i < D; ++i) {
                            d[m][n][i][0] = z0 * sums[0][i] + kMagicBits, d[m][n][i][1] = z0 * sums[1][i] + kMagicBits;
                            d[m][n][i][2] = z1 * sums[0][i] + kMagicBits, d[m][n][i][3] = z1 * sums[1][i] + kMagicBits;
                        }
                    }
                }
#pragma unroll
                for (int b = f * FB; b < (f + 1) * FB; ++b) {
                    uint32_t fr[MT][4];
#pragma unroll
                    for (int m = 0; m < MT; ++m) {
                        const uint32_t wa = b == 0 ? va[m].x : b == 1 ? va[m].y : b == 2 ? va[m].z : va[m].w;
                        const uint32_t wb = b == 0 ? vb[m].x : b == 1 ? vb[m].y : b == 2 ? vb[m].z : vb[m].w;
                        fr[m][0] = wa & 0x0f0f0f0fu, fr[m][1] = wb & 0x0f0f0f0fu;
                        fr[m][2] = (wa >> 4) & 0x0f0f0f0fu, fr[m][3] = (wb >> 4) & 0x0f0f0f0fu;
                    }
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int i = 0; i < D; ++i) {
                            if (b % 2 == 0)
                                xf[n][i] = *reinterpret_cast<const uint4*>(xr[n] + i * x.plane + at * kChunk + (b >> 1) * 64);
#pragma unroll
                            for (int m = 0; m < MT; ++m)
                                mma_u8s8(d[m][n][i], fr[m], b % 2 ? xf[n][i].z : xf[n][i].x, b % 2 ? xf[n][i].w : xf[n][i].y);
                        }
                }
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    const float s0 = scale_of(sc[m][blk] & 0xffffu, a.w.scale_bf16), s1 = scale_of(sc[m][blk] >> 16, a.w.scale_bf16);
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            float v = __int_as_float(d[m][n][0][e]) - kMagic;
#pragma unroll
                            for (int i = 1; i < D; ++i) v = fmaf(v, 256.f, __int_as_float(d[m][n][i][e]) - kMagic);
                            acc[m][n][e] = fmaf(v * (LOW ? fabsf(xs[n][e & 1]) : xs[n][e & 1]), e & 2 ? s1 : s0, acc[m][n][e]);
                        }
                }
                if constexpr (LOW) {
                    if (__any_sync(0xffffffffu, signs < 0)) {  // the same sums of the low digits
                        int l[MT][NT][kLow][4];
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            const int4 r = *reinterpret_cast<const int4*>(xl[n] + (at * FL + f) * (step / 2));
#pragma unroll
                            for (int m = 0; m < MT; ++m) {
                                const uint32_t z2 = zz[m][blk / 2] >> (16 * (blk & 1));
                                const int z0 = -(int)(z2 & 0xffu), z1 = -(int)((z2 >> 8) & 0xffu);
                                l[m][n][0][0] = z0 * r.x + kMagicBits, l[m][n][0][1] = z0 * r.z + kMagicBits;
                                l[m][n][0][2] = z1 * r.x + kMagicBits, l[m][n][0][3] = z1 * r.z + kMagicBits;
                                l[m][n][1][0] = z0 * r.y + kMagicBits, l[m][n][1][1] = z0 * r.w + kMagicBits;
                                l[m][n][1][2] = z1 * r.y + kMagicBits, l[m][n][1][3] = z1 * r.w + kMagicBits;
                            }
                        }
#pragma unroll
                        for (int b = f * FB; b < (f + 1) * FB; ++b)
#pragma unroll
                            for (int m = 0; m < MT; ++m) {
                                const uint32_t wa = b == 0 ? va[m].x : b == 1 ? va[m].y : b == 2 ? va[m].z : va[m].w;
                                const uint32_t wb = b == 0 ? vb[m].x : b == 1 ? vb[m].y : b == 2 ? vb[m].z : vb[m].w;
                                const uint32_t fr[4] = {wa & 0x0f0f0f0fu, wb & 0x0f0f0f0fu, (wa >> 4) & 0x0f0f0f0fu, (wb >> 4) & 0x0f0f0f0fu};
#pragma unroll
                                for (int n = 0; n < NT; ++n)
#pragma unroll
                                    for (int i = 0; i < kLow; ++i) {
                                        const uint2 u = *reinterpret_cast<const uint2*>(xr[n] + (D + i) * x.plane + at * kChunk + (b >> 1) * 64 + (b & 1) * 8);
                                        mma_u8s8(l[m][n][i], fr, u.x, u.y);
                                    }
                            }
#pragma unroll
                        for (int m = 0; m < MT; ++m) {
                            const float s0 = scale_of(sc[m][blk] & 0xffffu, a.w.scale_bf16), s1 = scale_of(sc[m][blk] >> 16, a.w.scale_bf16);
#pragma unroll
                            for (int n = 0; n < NT; ++n)
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    const float v = fmaf(__int_as_float(l[m][n][0][e]) - kMagic, 256.f, __int_as_float(l[m][n][1][e]) - kMagic);
                                    // a token without low digits has none written: its sums are not used
                                    if (xs[n][e & 1] < 0.f) acc[m][n][e] = fmaf(v * 0x1p-15f * -xs[n][e & 1], e & 2 ? s1 : s0, acc[m][n][e]);
                                }
                        }
                    }
                }
            }
        }
        if (a.ks > 0) {  // the warps of a row of tiles: their sums in order, by the first of them
            float* mine = reinterpret_cast<float*>(s_mem) + a.sums_at + (size_t)warp * 32 * 4 * NT * MT;
            if (sub) {
#pragma unroll
                for (int i = 0; i < 4 * NT * MT; ++i) mine[i * 32 + lane] = acc[i / (4 * NT)][i / 4 % NT][i % 4];
            }
            __syncthreads();
            if (!sub) {
                for (int j = 1; j < 1 << a.ks; ++j)
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
#pragma unroll
                    for (int m = 0; m < MT; ++m) {
                        const size_t r = ((size_t)tr * MT + m) * 16 + g + 8 * (e >> 1);
                        if (r >= a.w.n_out) continue;
                        const float v = acc[m][n][e];
                        if (a.y_bf16)
                            static_cast<__nv_bfloat16*>(a.y)[t * a.w.n_out + r] = __float2bfloat16_rn(v);
                        else
                            static_cast<float*>(a.y)[t * a.w.n_out + r] = v;
                    }
                }
        }
    }
}
// Apart from the kernel's own loop, from which these sums would take registers (in one loop 8192 x 8192 took 13.2 us
// instead of 12.3): called where some token has low digits.
template <int MT, int NT, int PC, int FB, bool WS>
__device__ __noinline__ void stream_tiles_low(const StreamArgs* args, unsigned char* s_mem, unsigned char* ring, const Producer<MT, PC>* from) {
    Producer<MT, PC> p = *from;
    stream_tiles<MT, NT, 3, PC, FB, WS, true>(*args, s_mem, ring, p);
    asm volatile("cp.async.wait_all;" ::: "memory");
}

// The forms for 9 to 16 float tokens fill the registers and spill (up to 380 bytes in groups of 32 with digits in the
// workspace, else up to 70).
// D digits an activation; PC scales of a row in 128 inputs; FB: blocks of 32 inputs after which a sum meets its scales; WS: the
// digits are in the workspace.
template <int MT, int NT, int D, int PC, int FB, bool WS>
__global__ void __launch_bounds__(kWarps * 32, 1) w4_stream_kernel(const __grid_constant__ StreamArgs a) {
    using S = Stage4<MT, PC>;
    extern __shared__ __align__(16) unsigned char s_mem[];
    const int chunks = (int)a.w.chunks, T = (int)a.x.tokens;
    unsigned char* ring = s_mem + (threadIdx.x >> 5) * S::kStages * S::kBytes;
    // The weights do not depend on the kernel before, the activations may.
    Producer<MT, PC> p;
    p.fill(a, ring);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const Digits x = digits_at(WS ? a.digits : s_mem + a.digits_at, D, T, chunks, FB);
    int more = 0;  // some token has low digits somewhere
    if constexpr (WS) {
        if constexpr (D == 3) {
            int signs = 0;
            for (int i = threadIdx.x; i < (int)even(T) * chunks * (4 / FB); i += kWarps * 32)
                signs |= *reinterpret_cast<const int*>(x.records + (size_t)i * 16 + 12);
            more = __syncthreads_or(signs < 0);
        }
    } else {
        const int n = T * chunks;
        const bool pairs = x_pairs(a.x);
        bool mine = false;
        constexpr int kU = 4;  // chunks of a half warp whose loads are under way together
        for (int i = threadIdx.x >> 4; (i & ~1) < n; i += kWarps * 2 * kU) {
            Eight<D> e[kU];
#pragma unroll
            for (int u = 0; u < kU; ++u) {
                const int j = min(i + u * kWarps * 2, n - 1), t = T == 1 ? 0 : j / chunks;
                if (((i + u * kWarps * 2) & ~1) < n) load_eight(e[u], a.x, pairs, t, j - t * chunks);
            }
#pragma unroll
            for (int u = 0; u < kU; ++u) {
                const int j = min(i + u * kWarps * 2, n - 1), t = T == 1 ? 0 : j / chunks;
                if (((i + u * kWarps * 2) & ~1) < n) mine |= make_digits<D, FB>(e[u], a.x, x, t, j - t * chunks);
            }
        }
        if constexpr (D == 3) {
            more = __syncthreads_or(mine);
            if (more) {
#pragma unroll 1
                for (int i = threadIdx.x >> 4; (i & ~1) < n; i += kWarps * 2) {
                    const int j = min(i, n - 1), t = j / chunks, c = j - t * chunks;
                    Eight<3> e;
                    load_eight(e, a.x, pairs, t, c);
                    const bool low = *reinterpret_cast<const float*>(x.records + ((size_t)c * (4 / FB) * even(T) + t) * 16 + 12) < 0.f;
                    make_low<FB>(e, a.x, x, t, c, low);
                    end_records<FB>(a.x, x, t, c);
                }
                __syncthreads();
            }
        } else {
            __syncthreads();
        }
    }
    if constexpr (D == 3) {
        if (more) {
            const Producer<MT, PC> copy = p;
            stream_tiles_low<MT, NT, PC, FB, WS>(&a, s_mem, ring, &copy);
            return;
        }
    }
    stream_tiles<MT, NT, D, PC, FB, WS, false>(a, s_mem, ring, p);
    asm volatile("cp.async.wait_all;" ::: "memory");
}

// Shared memory for the digits, beside the ring (of one row tile a warp, or of two with one tile of tokens).
constexpr size_t digit_smem(int D) { return (D == 3 ? 78 : 60) * 1024; }

int flush_blocks(const W4View& w, const W4X& x) {
    const int fb = 4 / w.per_chunk;
    return x.group && x.group / 32 < fb ? 1 : fb;  // groups of activations smaller than the weights': every 32 inputs
}
int digits_of(const W4X& x) { return x.kind == kW4XInt8 ? 1 : 3; }

template <int MT, int NT, int D, int PC, int FB, bool WS>
cudaError_t run_stream(StreamArgs& a, int num_sms, cudaStream_t s) {
    auto kernel = w4_stream_kernel<MT, NT, D, PC, FB, WS>;
    constexpr size_t ring = (size_t)kWarps * Stage4<MT, PC>::kStages * Stage4<MT, PC>::kBytes;
    constexpr size_t sums = kWarps * 32 * 4 * NT * MT * sizeof(float);
    static_assert(ring + digit_smem(D) + sums <= 227 * 1024, "shared memory");
    const size_t own = WS ? 0 : (digit_bytes(D, a.x.tokens, a.w.chunks, FB) + 15) & ~size_t(15);
    // Warps that share a row of tiles: the split with the shortest chain of tiles for a warp, where a round
    // costs about as much as 3 tiles (its first loads, its sums joined).
    const size_t rows = a.w.tile_rows / MT;
    size_t best = ~size_t(0);
    for (int k = 0; 1 << k <= kWarps && (size_t)1 << k <= a.w.chunks; ++k) {
        const size_t tiles = (rows + (kWarps >> k) - 1) / (kWarps >> k);
        const size_t cost = (tiles + num_sms - 1) / num_sms * ((a.w.chunks + (1 << k) - 1) / (1 << k) + 3);
        if (cost < best) best = cost, a.ks = k, a.tiles = (int)tiles;
    }
    a.digits_at = (int)ring;
    a.sums_at = (int)((ring + own) / sizeof(float));
    const size_t smem = ring + own + (a.ks > 0 ? sums : 0);
    static SmemOnce once;  // the most this kernel is ever given
    const cudaError_t e = once.set(reinterpret_cast<const void*>(kernel), (int)(ring + digit_smem(D) + sums));
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)std::min(a.tiles, num_sms));
    cfg.blockDim = dim3(kWarps * 32);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &at;
    cfg.numAttrs = WS ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, a);
}
template <int MT, int NT, int D, bool WS>
cudaError_t run_pc(StreamArgs& a, int num_sms, cudaStream_t s) {
    const int pc = a.w.per_chunk;
    if constexpr (D == 1)
        if (pc < 4 && flush_blocks(a.w, a.x) == 1)
            return pc == 1 ? run_stream<MT, NT, D, 1, 1, WS>(a, num_sms, s) : run_stream<MT, NT, D, 2, 1, WS>(a, num_sms, s);
    return pc == 1   ? run_stream<MT, NT, D, 1, 4, WS>(a, num_sms, s)
           : pc == 2 ? run_stream<MT, NT, D, 2, 2, WS>(a, num_sms, s)
                     : run_stream<MT, NT, D, 4, 1, WS>(a, num_sms, s);
}
template <int D, bool WS>
cudaError_t run_nt(StreamArgs& a, int num_sms, cudaStream_t s) {
    // Two row tiles a warp share the activations' fragments and the loop's overhead (128000 x 2048, 5 tokens: 28.8 ->
    // 27.8 us, 8192 x 8192 12.8 -> 12.2); one tile a warp where that would leave a warp fewer than 4 pairs (2048 x 2048: 5.3 -> 4.2), and
    // where 16 tokens' three digits fill the registers.
    if (a.x.tokens > 8) return D == 1 ? run_pc<2, 2, 1, WS>(a, num_sms, s) : run_pc<1, 2, 3, WS>(a, num_sms, s);
    return a.w.tile_rows * a.w.chunks < (size_t)num_sms * kWarps * 8 ? run_pc<1, 1, D, WS>(a, num_sms, s) : run_pc<2, 1, D, WS>(a, num_sms, s);
}

template <int D>
cudaError_t run_digits(const W4X& x, int chunks, int fb, unsigned char* out, cudaStream_t s) {
    const unsigned grid = (unsigned)std::min<size_t>((x.tokens * chunks + 15) / 16, 1024);
    if (fb == 4)
        w4_digits_kernel<D, 4><<<grid, 256, 0, s>>>(x, chunks, out);
    else if (fb == 2)
        w4_digits_kernel<D, 2><<<grid, 256, 0, s>>>(x, chunks, out);
    else
        w4_digits_kernel<D, 1><<<grid, 256, 0, s>>>(x, chunks, out);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_w4_pack(const uint8_t* codes, const unsigned short* scales, const uint8_t* zeros, const W4View& w,
                           uint32_t* out_c, unsigned short* out_s, uint8_t* out_z, int* bad, cudaStream_t s) {
    const size_t words = w.tile_rows * w.chunks * 256;
    w4_pack_kernel<<<(unsigned)((words + 255) / 256), 256, 0, s>>>(codes, scales, zeros, w, out_c, out_s, out_z, bad);
    return cudaGetLastError();
}

size_t w4_stream_workspace(const W4View& w, const W4X& x) {
    const size_t n = digit_bytes(digits_of(x), x.tokens, w.chunks, flush_blocks(w, x));
    return n <= digit_smem(digits_of(x)) ? 0 : n;
}

cudaError_t launch_w4_stream(const W4View& w, const W4X& x, void* y, int y_bf16, void* workspace, int num_sms,
                             cudaStream_t s) {
    if (x.tokens > kTokens) return cudaErrorInvalidValue;
    StreamArgs a{};
    a.w = w, a.x = x, a.y = y, a.y_bf16 = y_bf16;
    const bool three = digits_of(x) == 3;
    if (w4_stream_workspace(w, x) == 0) return three ? run_nt<3, false>(a, num_sms, s) : run_nt<1, false>(a, num_sms, s);
    a.digits = static_cast<unsigned char*>(workspace);
    const int fb = flush_blocks(w, x), chunks = (int)w.chunks;
    const cudaError_t e = three ? run_digits<3>(x, chunks, fb, a.digits, s) : run_digits<1>(x, chunks, fb, a.digits, s);
    if (e != cudaSuccess) return e;
    return three ? run_nt<3, true>(a, num_sms, s) : run_nt<1, true>(a, num_sms, s);
}

}  // namespace bebelm
