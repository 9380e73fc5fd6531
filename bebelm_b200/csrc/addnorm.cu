// Residual addition + RMS norm over the hidden size, with a float or an 8-bit output.
//
// The arithmetic is the reference's rmsnorm (src/kernels/rmsnorm.rs:10-21) behind the residual
// addition of its layer loop, each step rounded to f32 where the reference rounds:
//     h = round_T(x + residual)                       (T: the stream's type, f32 or bf16)
//     ss = Σ f64(f32(h·h)),  mean = f32(ss / n),  r = 1 / sqrt(mean + eps)
//     t = f32(f32(h·r)·gain)
//     y = t (f32 or bf16), or int8 with one scale per group of values, in the rule of the K-quant
//     products' activations (src/kernels/matmul.rs quantize_q8): a = max|t|, scale = a / 127,
//     q = round half away from zero(t·(127 / a)), 0 where a = 0.
// Every step is one IEEE operation, so the 8-bit codes are the definition's own: no code next to
// a border depends on how the sum was split. The f64 sum's order only shows when f32(ss / n) sits
// within f64 rounding of a border of f32.
//
// Bound: HBM (8 to 16 bytes an element, ~25 operations) for many rows, the latency of one load, one
// reduction and one store for few. A row stays in registers between its sum and its output, so it
// is read once. Rows of up to 1024 values take a warp each (no barrier); longer ones a CTA each with
// 8 or 16 values a thread, one barrier for the sum and one more for a scale of the whole row. Measured:
// 8192 bf16 rows of 2048 with their sum 23.4 us (134 MB at 5.7 TB/s, 87 % of a copy's rate); one row
// of 2048 to int8 2.8 us, 1037 f32 rows of 2080 5.0 us. Streaming cache hints on the loads cost 17 %, a gain read ahead of the sum 15 % (registers).
#include <algorithm>
#include <cstdint>

#include "internal.h"

namespace bebelm {
namespace {

__device__ __forceinline__ float load1(const float* p) { return *p; }
__device__ __forceinline__ float load1(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void store1(float* p, float v) { *p = v; }
__device__ __forceinline__ void store1(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ float round_as(const float*, float v) { return v; }
__device__ __forceinline__ float round_as(const __nv_bfloat16*, float v) {
    return __bfloat162float(__float2bfloat16_rn(v));
}

__device__ __forceinline__ void load8(const float* p, float* v) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}
__device__ __forceinline__ void load8(const __nv_bfloat16* p, float* v) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}
__device__ __forceinline__ void store8(float* p, const float* v) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float* v) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}

// 8 values of a row from element e; with VEC whole and aligned, else one at a time up to n
template <bool VEC, class T>
__device__ __forceinline__ void row_load(const T* p, size_t n, size_t e, float* v) {
    if constexpr (VEC) {
        load8(p + e, v);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = e + i < n ? load1(p + e + i) : 0.f;
    }
}
template <bool VEC, class T>
__device__ __forceinline__ void row_store(T* p, size_t n, size_t e, const float* v) {
    if constexpr (VEC) {
        store8(p + e, v);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (e + i < n) store1(p + e + i, v[i]);
    }
}

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
// the larger one; NaN if either is
__device__ __forceinline__ float max_nan(float a, float b) {
    float m;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
    return m;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// One row per blockDim.x threads (a warp when blockDim.y > 1 rows share the CTA); thread x holds
// the NV runs of 8 values that start at 8 (x + i blockDim.x).
// The two-run form of the bf16 stream is held to 32 registers (24 bytes of spills), which lets 2048
// threads stay on an SM: 8192 x 2048 with a bf16 output 23.4 us against 24.4 us at 40 registers. The
// f32 stream, whose runs take twice the registers, loses by it (1037 x 2080 5.4 -> 5.6 us).
template <class T, class O, int NV, bool VEC>
__global__ void __launch_bounds__(1024, VEC && sizeof(T) == 2 && sizeof(O) > 1 && NV == 2 ? 2 : 0) add_rmsnorm_kernel(AddNormArgs a) {
    __shared__ double s_part[32];
    __shared__ float s_max[32];
    const size_t row = (size_t)blockIdx.x * blockDim.y + threadIdx.y;
    if (row >= a.rows) return;  // only whole warps leave, and only where no barrier follows
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    const T* res = a.residual ? static_cast<const T*>(a.residual) + row * a.residual_stride : nullptr;
    T* sum = a.sum_out ? static_cast<T*>(a.sum_out) + row * a.sum_stride : nullptr;

    float v[NV][8];
    double ss = 0.0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const size_t e = 8 * ((size_t)threadIdx.x + (size_t)i * blockDim.x);
        if (e < a.n) {
            row_load<VEC>(x, a.n, e, v[i]);
            if (res) {
                float r[8];
                row_load<VEC>(res, a.n, e, r);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[i][j] = round_as(x, __fadd_rn(v[i][j], r[j]));
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) ss += (double)__fmul_rn(v[i][j], v[i][j]);
    }
    if (sum) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const size_t e = 8 * ((size_t)threadIdx.x + (size_t)i * blockDim.x);
            if (e < a.n) row_store<VEC>(sum, a.n, e, v[i]);
        }
    }
    ss = warp_sum(ss);
    if (warps > 1) {  // every warp adds the warps' sums itself: one barrier, not two
        if (lane == 0) s_part[warp] = ss;
        __syncthreads();
        ss = warp_sum(lane < warps ? s_part[lane] : 0.0);
    }
    const float mean = __double2float_rn(ss / (double)a.n);
    const float scale = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(mean, a.eps)));
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const size_t e = 8 * ((size_t)threadIdx.x + (size_t)i * blockDim.x);
        if (e < a.n) {
            float g[8];
            row_load<VEC>(a.gain, a.n, e, g);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] = __fmul_rn(__fmul_rn(v[i][j], scale), g[j]);
        }
        if constexpr (sizeof(O) > 1) {
            if (e < a.n) row_store<VEC>(static_cast<O*>(a.y) + row * a.n, a.n, e, v[i]);
        }
    }
    if constexpr (sizeof(O) == 1) {
        if (a.group == 0) {  // one scale for the row
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int j = 0; j < 8; ++j) amax = max_nan(amax, fabsf(v[i][j]));
            amax = warp_max(amax);
            if (warps > 1) {
                if (lane == 0) s_max[warp] = amax;
                __syncthreads();
                amax = warp_max(lane < warps ? s_max[lane] : 0.f);
            }
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const size_t e = 8 * ((size_t)threadIdx.x + (size_t)i * blockDim.x);
            if (a.group) {  // a group is group / 8 neighbouring lanes
                amax = 0.f;
#pragma unroll
                for (int j = 0; j < 8; ++j) amax = max_nan(amax, fabsf(v[i][j]));
                for (unsigned o = 1; o < a.group / 8; o <<= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
            }
            if (e >= a.n) continue;
            // 127 / a leaves f32's range below 3.8e-37: there both are formed 2^64 times as large
            const float up = amax < 0x1p-100f ? 0x1p64f : 1.f;
            const float inv = amax > 0.f ? __fdiv_rn(127.0f, __fmul_rn(amax, up)) : 0.f;
            alignas(8) signed char q[8];
#pragma unroll
            for (int j = 0; j < 8; ++j)  // |t inv| < 127.5; a NaN (0 times an infinity, or t's) gives 0
                q[j] = (signed char)__float2int_rz(roundf(__fmul_rn(__fmul_rn(v[i][j], up), inv)));
            signed char* y = static_cast<signed char*>(a.y) + row * a.n + e;
            if constexpr (VEC) {
                *reinterpret_cast<uint2*>(y) = *reinterpret_cast<const uint2*>(q);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (e + j < a.n) y[j] = q[j];
            }
            if (a.group ? e % a.group == 0 : e == 0)
                a.y_scales[a.group ? row * (a.n / a.group) + e / a.group : row] = __fadd_rn(__fdiv_rn(amax, 127.0f), __fsub_rn(amax, amax));  // an infinity: NaN
        }
    }
}

template <class T, class O>
cudaError_t launch(const AddNormArgs& a, int num_sms, cudaStream_t s) {
    // runs of 8 values a row, a multiple of 32 threads, up to 1024
    const size_t runs = (a.n + 7) / 8;
    const auto aligned = [](const void* p, size_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; };
    const size_t es = sizeof(T);
    const bool vec = a.n % 8 == 0 && aligned(a.x, 16) && a.x_stride * es % 16 == 0 &&
                     (!a.residual || (aligned(a.residual, 16) && a.residual_stride * es % 16 == 0)) &&
                     (!a.sum_out || (aligned(a.sum_out, 16) && a.sum_stride * es % 16 == 0)) && aligned(a.gain, 16) &&
                     aligned(a.y, 8 * std::min<size_t>(sizeof(O), 2)) && (sizeof(O) != 4 || aligned(a.y, 16));
    // One run a thread has the shortest chain from load to store, two a thread halve what a warp does
    // once a row (two sums, a division, a root): two where the rows fill more than half of the SMs'
    // threads. One row of 2048 takes 2.9 us with one and 3.8 us with two; 1037 f32 rows of 2080 5.9 and
    // 5.4 us, 8192 bf16 rows of 2048 26.6 and 23.4 us (5.7 TB/s; four runs 27.5 us).
    const bool many = a.rows * runs >= (size_t)num_sms * 1024;
    const int nv = runs <= 1024 && !many ? 1 : runs <= 2048 ? 2 : 4;
    dim3 block, grid;
    int nv_used = nv;
    if (runs <= 128) {  // a warp a row, 4 rows a CTA
        nv_used = runs <= 32 ? 1 : runs <= 64 ? 2 : 4;
        block = dim3(32, 4);
        grid = dim3((unsigned)((a.rows + 3) / 4));
    } else {
        block = dim3((unsigned)(((runs + nv - 1) / nv + 31) / 32 * 32), 1);
        grid = dim3((unsigned)a.rows);
    }
#define RUN(NV, V) add_rmsnorm_kernel<T, O, NV, V><<<grid, block, 0, s>>>(a)
    if (vec) {
        if (nv_used == 1) RUN(1, true);
        else if (nv_used == 2) RUN(2, true);
        else RUN(4, true);
    } else {
        if (nv_used == 1) RUN(1, false);
        else if (nv_used == 2) RUN(2, false);
        else RUN(4, false);
    }
#undef RUN
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_add_rmsnorm(const AddNormArgs& a, int num_sms, cudaStream_t s) {
    if (a.bf16) {
        if (a.out == kNormOutInt8) return launch<__nv_bfloat16, signed char>(a, num_sms, s);
        if (a.out == kNormOutBf16) return launch<__nv_bfloat16, __nv_bfloat16>(a, num_sms, s);
        return launch<__nv_bfloat16, float>(a, num_sms, s);
    }
    if (a.out == kNormOutInt8) return launch<float, signed char>(a, num_sms, s);
    if (a.out == kNormOutBf16) return launch<float, __nv_bfloat16>(a, num_sms, s);
    return launch<float, float>(a, num_sms, s);
}

}  // namespace bebelm
