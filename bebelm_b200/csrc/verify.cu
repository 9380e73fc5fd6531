// Drafted tokens checked against the target model's rows (speculative sampling), on the device.
//
// For a sequence with drafts x_0 .. x_{n-1}, target rows 0 .. n and draft rows 0 .. n-1:
//     p_i = softmax(target_i / temperature), q_i = softmax(draft_i / temperature)
//           (or the rows themselves, when they are probabilities)
//     x_i is accepted iff every draft before it was and u_i q_i(x_i) < p_i(x_i);  q_i(x_i) = 1 without
//     draft rows (a draft that was looked up, not sampled).
//     At the first refusal i the next token is drawn from max(p_i - q_i, 0) (from p_i if that is zero
//     everywhere), after n acceptances from p_n: the lowest index j with Σ_{m <= j} w_m > u Σ w.
//     Temperature 0: a draft is accepted iff it is its row's argmax (src/sampler.rs:139-149: the first
//     index of the maximum, NaN never, 0 if nothing is above -inf); the next token is an argmax.
//
// A drawn token is the place where a running sum over the vocabulary passes a border. With V entries a
// relative error e of the sums moves it with probability about V e: for 1.3e5 entries f32 is not
// enough (1e-2), so the row a token is drawn from is summed in f64 from f64 exponentials. Whether a
// draft is accepted is one comparison: its row's sum may have the 1e-7 of f32 exponentials.
//
//   verify_rows_kernel   one pass over every row that can matter: per slice the running maximum and the
//                        sum of exponentials below it (greedy: the maximum and its index). Bound: HBM.
//   verify_pick_kernel   a cluster of CTAs per sequence joins the slices, decides, and draws: each CTA
//                        holds a contiguous part of the row; the parts' sums are exchanged through distributed
//                        shared memory, and the CTA whose part the border falls into finds the place.
//   verify_greedy_kernel a warp per sequence joins the slices' maxima.
#include <cooperative_groups.h>
#include <math_constants.h>

#include <algorithm>
#include <cstdint>

#include "internal.h"

namespace cg = cooperative_groups;

namespace bebelm {
namespace {

constexpr int kRowThreads = 256, kPickThreads = 512, kMaxSlices = 64;
constexpr float kLog2e = 1.4426950408889634f;

struct RowPart {  // of one slice of a row
    float m;      // maximum (-inf: nothing above -inf)
    unsigned i;   // greedy: its first index
    double s;     // Σ exp((l - m) / temperature)
};

// a logit as it counts: NaN never wins, +inf is the largest finite value
__device__ __forceinline__ float clean(float l) { return fminf(fmaxf(l, -CUDART_INF_F), 3.402823466e38f); }
// a probability as it counts
__device__ __forceinline__ double clean_p(float p) { return p > 0.f ? (double)p : 0.0; }

__device__ __forceinline__ float ex2f(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ int drafts_of(const VerifyArgs& a, int b) {
    const int n = a.n_drafts ? a.n_drafts[b] : a.drafts;
    return min(max(n, 0), a.drafts);
}

// grid (target rows then draft rows, slices)
template <bool GREEDY, bool VEC>
__global__ void __launch_bounds__(kRowThreads) verify_rows_kernel(VerifyArgs a, RowPart* parts, int slices) {
    const int row = blockIdx.x, target_rows = a.seqs * (a.drafts + 1);
    const float* p;
    if (row < target_rows) {
        const int b = row / (a.drafts + 1), i = row % (a.drafts + 1);
        if (i > drafts_of(a, b)) return;
        p = a.target + (size_t)row * a.target_stride;
    } else {
        const int r = row - target_rows, b = r / a.drafts, i = r % a.drafts;
        if (i >= drafts_of(a, b)) return;
        p = a.draft + (size_t)r * a.draft_stride;
    }
    // whole groups of 4 values a slice
    const size_t quads = (a.vocab + 3) / 4;
    const size_t e0 = 4 * (quads * blockIdx.y / slices), e1 = min(a.vocab, 4 * (quads * (blockIdx.y + 1) / slices));
    const float c = kLog2e / a.temperature;
    float m = -CUDART_INF_F, s = 0.f;
    unsigned at = 0xffffffffu;
    constexpr int kU = 4;  // quads in flight
    for (size_t e = e0 + 4 * threadIdx.x; e < e1; e += 4 * kRowThreads * kU) {
        float v[kU][4];
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            const size_t f = e + (size_t)u * 4 * kRowThreads;
            if (VEC && f < e1) {
                const float4 t = __ldg(reinterpret_cast<const float4*>(p + f));
                v[u][0] = t.x, v[u][1] = t.y, v[u][2] = t.z, v[u][3] = t.w;
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) v[u][j] = f + j < e1 ? __ldg(p + f + j) : -CUDART_INF_F;
            }
        }
        if constexpr (GREEDY) {
#pragma unroll
            for (int u = 0; u < kU; ++u)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (v[u][j] > m) m = v[u][j], at = (unsigned)(e + (size_t)u * 4 * kRowThreads + j);
        } else {
            float mx = m;
#pragma unroll
            for (int u = 0; u < kU; ++u)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    v[u][j] = clean(v[u][j]);
                    mx = fmaxf(mx, v[u][j]);
                }
            if (mx > m) {
                s *= ex2f((m - mx) * c);  // 0 while nothing has been seen
                m = mx;
            }
            if (m > -CUDART_INF_F) {
#pragma unroll
                for (int u = 0; u < kU; ++u)
#pragma unroll
                    for (int j = 0; j < 4; ++j) s += ex2f((v[u][j] - m) * c);
            }
        }
    }
    // join the threads: maxima, then the sums below the CTA's maximum in f64
    __shared__ float s_m[kRowThreads / 32];
    __shared__ double s_s[kRowThreads / 32];
    __shared__ unsigned s_i[kRowThreads / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    float wm = m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) wm = fmaxf(wm, __shfl_xor_sync(0xffffffffu, wm, o));
    if constexpr (GREEDY) {
        unsigned wi = m == wm ? at : 0xffffffffu;
        wi = __reduce_min_sync(0xffffffffu, wi);
        if (lane == 0) s_m[warp] = wm, s_i[warp] = wi;
    } else {
        double ws = s > 0.f ? (double)(s * ex2f((m - wm) * c)) : 0.0;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) ws += __shfl_xor_sync(0xffffffffu, ws, o);
        if (lane == 0) s_m[warp] = wm, s_s[warp] = ws;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        RowPart r{-CUDART_INF_F, 0xffffffffu, 0.0};
        for (int w = 0; w < kRowThreads / 32; ++w) r.m = fmaxf(r.m, s_m[w]);
        for (int w = 0; w < kRowThreads / 32; ++w) {
            if constexpr (GREEDY) {
                if (s_m[w] == r.m) r.i = min(r.i, s_i[w]);
            } else if (s_s[w] > 0.0) {
                r.s += s_s[w] * (double)ex2f((s_m[w] - r.m) * c);
            }
        }
        parts[(size_t)row * slices + blockIdx.y] = r;
    }
}

// the slices of one row joined by a warp (every lane gets the answer)
__device__ __forceinline__ RowPart join_row(const RowPart* parts, int slices, double inv_t, bool greedy) {
    const int lane = threadIdx.x & 31;
    RowPart r{-CUDART_INF_F, 0xffffffffu, 0.0};
    for (int i = lane; i < slices; i += 32) r.m = fmaxf(r.m, parts[i].m);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) r.m = fmaxf(r.m, __shfl_xor_sync(0xffffffffu, r.m, o));
    for (int i = lane; i < slices; i += 32) {
        const RowPart p = parts[i];
        if (greedy) {
            if (p.m == r.m) r.i = min(r.i, p.i);
        } else if (p.s > 0.0) {
            r.s += p.s * exp(((double)p.m - (double)r.m) * inv_t);
        }
    }
    if (greedy) {
        r.i = __reduce_min_sync(0xffffffffu, r.i);
    } else {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) r.s += __shfl_xor_sync(0xffffffffu, r.s, o);
    }
    return r;
}

// the accepted drafts, the next token and -1 behind it
__device__ __forceinline__ void write_out(const VerifyArgs& a, int b, int n_acc, int next) {
    int* out = a.out + (size_t)b * (a.drafts + 1);
    for (int i = threadIdx.x & 31; i <= a.drafts; i += 32)
        out[i] = i < n_acc ? a.tokens[(size_t)b * a.drafts + i] : i == n_acc ? next : -1;
    if ((threadIdx.x & 31) == 0) a.accepted[b] = n_acc;
}

__global__ void __launch_bounds__(32) verify_greedy_kernel(VerifyArgs a, const RowPart* parts, int slices) {
    const int b = blockIdx.x, n = drafts_of(a, b);
    for (int i = 0;; ++i) {
        const RowPart r = join_row(parts + ((size_t)b * (a.drafts + 1) + i) * slices, slices, 0.0, true);
        const int best = r.i == 0xffffffffu ? 0 : (int)r.i;
        if (i < n && a.tokens[(size_t)b * a.drafts + i] == best) continue;
        write_out(a, b, i, best);
        return;
    }
}

__device__ __forceinline__ double block_sum(double v, double* s_part) {  // every thread gets the sum
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s_part[threadIdx.x >> 5] = v;
    __syncthreads();
    double t = 0.0;
    for (int w = 0; w < kPickThreads / 32; ++w) t += s_part[w];
    return t;
}

// One row of probabilities, of logits with a known maximum and sum, or a certain draft, as f64.
struct Row {
    const float* p;
    double m, inv_t, inv_s;
    int probs;
    __device__ __forceinline__ double raw(size_t j) const {  // before the division by the sum
        const float l = p[j];
        if (probs) return clean_p(l);
        const double d = (double)clean(l) - m;
        return exp(d * inv_t);
    }
    __device__ __forceinline__ double at(size_t j) const { return raw(j) * inv_s; }
};

__global__ void __launch_bounds__(kPickThreads) verify_pick_kernel(VerifyArgs a, const RowPart* parts, int slices) {
    cg::cluster_group cl = cg::this_cluster();
    const int ctas = (int)cl.num_blocks(), me = (int)cl.block_rank(), b = blockIdx.x / ctas;
    __shared__ double s_part[kPickThreads / 32], s_sum[3], s_m[2];
    __shared__ double s_prob[2][64];  // p_i(x_i), q_i(x_i)
    __shared__ int s_acc;
    const int n = drafts_of(a, b), warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = kPickThreads / 32;
    const int* tok = a.tokens + (size_t)b * a.drafts;
    const double inv_t = 1.0 / (double)a.temperature;
    const RowPart* tp = parts + (size_t)b * (a.drafts + 1) * slices;
    const RowPart* dp = parts + ((size_t)a.seqs * (a.drafts + 1) + (size_t)b * a.drafts) * slices;
    const float* trow = a.target + (size_t)b * (a.drafts + 1) * a.target_stride;
    const float* drow = a.draft ? a.draft + (size_t)b * a.drafts * a.draft_stride : nullptr;

    // ---- the decisions, in groups of 64 drafts (every CTA makes them for itself) ----
    int n_acc = 0;
    for (int base = 0; base < n && n_acc == base; base += 64) {
        const int cnt = min(64, n - base);
        for (int k = warp; k < 2 * cnt; k += warps) {  // a warp per value
            const int i = base + (k >> 1), side = k & 1, x = tok[i];
            double v = side ? 1.0 : 0.0;
            if (x >= 0 && (size_t)x < a.vocab && (side == 0 || drow)) {
                const float* p = side ? drow + (size_t)i * a.draft_stride : trow + (size_t)i * a.target_stride;
                if (a.probs) {
                    v = clean_p(p[x]);
                } else {
                    const RowPart r = join_row((side ? dp : tp) + (size_t)i * slices, slices, inv_t, false);
                    v = r.s > 0.0 ? exp(((double)clean(p[x]) - (double)r.m) * inv_t) / r.s : 0.0;
                }
            }
            if (lane == 0) s_prob[side][k >> 1] = v;
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            int i = 0;
            while (i < cnt && (double)a.u[(size_t)b * a.drafts + base + i] * s_prob[1][i] < s_prob[0][i]) ++i;
            s_acc = base + i;
        }
        __syncthreads();
        n_acc = s_acc;
    }

    // ---- the rows the next token is drawn from ----
    const bool refused = n_acc < n;
    const bool with_q = refused && drow;
    const int skip = refused && !drow ? tok[n_acc] : -1;  // a certain draft takes its own place away
    Row P{trow + (size_t)n_acc * a.target_stride, 0.0, inv_t, 1.0, a.probs};
    Row Q{with_q ? drow + (size_t)n_acc * a.draft_stride : nullptr, 0.0, inv_t, 1.0, a.probs};
    if (!a.probs) {
        if (warp == 0) {
            const RowPart r = join_row(tp + (size_t)n_acc * slices, slices, inv_t, false);
            if (lane == 0) s_m[0] = r.m;
        } else if (warp == 1 && with_q) {
            const RowPart r = join_row(dp + (size_t)n_acc * slices, slices, inv_t, false);
            if (lane == 0) s_m[1] = r.m;
        }
        __syncthreads();
        P.m = s_m[0];
        if (with_q) Q.m = s_m[1];
    }
    const size_t j0 = a.vocab * me / ctas, j1 = a.vocab * (me + 1) / ctas;
    const bool p_empty = !a.probs && P.m == -(double)CUDART_INF_F, q_empty = with_q && !a.probs && Q.m == -(double)CUDART_INF_F;

    // part sums of this CTA, exchanged: [0] of p, [1] of q, [2] of the weights
    auto exchange = [&](int k, double v, double* before, double* total) {
        v = block_sum(v, s_part);
        if (threadIdx.x == 0) s_sum[k] = v;
        cl.sync();
        double bf = 0.0, t = 0.0;
        for (int c = 0; c < ctas; ++c) {
            const double o = *cl.map_shared_rank(&s_sum[k], c);
            if (c < me) bf += o;
            t += o;
        }
        *before = bf;
        *total = t;
    };
    double before, total;
    if (with_q && !a.probs) {  // normalise both rows in f64 before they are compared
        double sp = 0.0, sq = 0.0, t;
        for (size_t j = j0 + threadIdx.x; j < j1; j += kPickThreads) {
            if (!p_empty) sp += P.raw(j);
            if (!q_empty) sq += Q.raw(j);
        }
        exchange(0, sp, &before, &t);
        P.inv_s = t > 0.0 ? 1.0 / t : 0.0;
        exchange(1, sq, &before, &t);
        Q.inv_s = t > 0.0 ? 1.0 / t : 0.0;
    }
    auto weight = [&](size_t j, bool plain) -> double {
        if (p_empty) return 0.0;
        const double p = P.at(j);
        if (plain) return p;
        if ((long long)j == skip) return 0.0;
        if (!with_q || q_empty) return p;
        const double w = p - Q.at(j);
        return w > 0.0 ? w : 0.0;
    };
    bool plain = !refused;
    for (int pass = 0; pass < 2; ++pass) {  // the second pass only where p - q is zero everywhere
        double w = 0.0;
        for (size_t j = j0 + threadIdx.x; j < j1; j += kPickThreads) w += weight(j, plain);
        if (pass) cl.sync();  // everyone has read the first pass's sums
        exchange(2, w, &before, &total);
        if (total > 0.0 || plain) break;
        plain = true;
    }
    // ---- the place: this CTA's, if the border lies in its part ----
    const double border = (double)a.u_sample[b] * total;
    // The first CTA whose sums pass the border; if rounding leaves none, the last one with any weight.
    int owner = -1, last = -1;
    {
        double run = 0.0;
        for (int c = 0; c < ctas; ++c) {
            const double o = *cl.map_shared_rank(&s_sum[2], c);
            run += o;
            if (o > 0.0) last = c;
            if (owner < 0 && o > 0.0 && run > border) owner = c;
        }
        if (owner < 0) owner = last;
    }
    cl.sync();  // nobody reads another CTA's memory after this
    if (owner < 0) {  // a row without any weight
        if (me == 0 && warp == 0) write_out(a, b, n_acc, 0);
        return;
    }
    if (me != owner) return;
    // tiles of 8 values a thread in order: the tile, the thread, the value
    constexpr int kPer = 8;
    __shared__ double s_scan[kPickThreads / 32];
    __shared__ int s_place, s_last;
    if (threadIdx.x == 0) s_place = INT_MAX, s_last = -1;
    __syncthreads();
    double run = before;
    for (size_t t0 = j0; t0 < j1; t0 += kPickThreads * kPer) {
        const size_t f = t0 + (size_t)threadIdx.x * kPer;
        double v[kPer], sum = 0.0;
        int lastw = -1;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            v[i] = f + i < j1 ? weight(f + i, plain) : 0.0;
            if (v[i] > 0.0) lastw = (int)(f + i);
            sum += v[i];
        }
        double inc = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double u = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += u;
        }
        if (lane == 31) s_scan[warp] = inc;
        __syncthreads();
        double at = run, all = 0.0;
        for (int w = 0; w < kPickThreads / 32; ++w) {
            if (w < warp) at += s_scan[w];
            all += s_scan[w];
        }
        at += inc - sum;
        for (int i = 0; i < kPer; ++i) {
            at += v[i];
            if (v[i] > 0.0 && at > border) {
                atomicMin(&s_place, (int)(f + i));
                break;
            }
        }
        if (lastw >= 0) atomicMax(&s_last, lastw);
        __syncthreads();
        if (s_place != INT_MAX) break;
        run += all;
        __syncthreads();
    }
    if (warp == 0) write_out(a, b, n_acc, s_place != INT_MAX ? s_place : max(s_last, 0));
}

int slices_of(const VerifyArgs& a, int num_sms) {
    // CTAs for every SM several times over, but at least 4096 values each
    const size_t rows = (size_t)a.seqs * (a.drafts + 1 + (a.draft ? a.drafts : 0));
    const size_t want = (8 * (size_t)num_sms + rows - 1) / rows, most = std::max<size_t>(1, a.vocab / 4096);
    return (int)std::max<size_t>(1, std::min<size_t>(std::min(want, most), kMaxSlices));
}

}  // namespace

size_t verify_workspace(const VerifyArgs& a, int num_sms) {
    if (a.probs && a.temperature != 0.f) return 0;
    const size_t rows = (size_t)a.seqs * (a.drafts + 1 + (a.draft ? a.drafts : 0));
    return rows * slices_of(a, num_sms) * sizeof(RowPart);
}

cudaError_t launch_verify(const VerifyArgs& a, int num_sms, cudaStream_t s) {
    const bool greedy = a.temperature == 0.f;
    RowPart* parts = static_cast<RowPart*>(a.workspace);
    const int slices = slices_of(a, num_sms);
    const auto vec4 = [](const float* p, size_t stride) {
        return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && stride % 4 == 0;
    };
    const bool vec = a.vocab % 4 == 0 && vec4(a.target, a.target_stride) &&
                     (greedy || !a.draft || vec4(a.draft, a.draft_stride));
    if (greedy || !a.probs) {
        const size_t rows = (size_t)a.seqs * (a.drafts + 1 + (!greedy && a.draft ? a.drafts : 0));
        const dim3 grid((unsigned)rows, (unsigned)slices);
        if (greedy) {
            if (vec) verify_rows_kernel<true, true><<<grid, kRowThreads, 0, s>>>(a, parts, slices);
            else verify_rows_kernel<true, false><<<grid, kRowThreads, 0, s>>>(a, parts, slices);
        } else {
            if (vec) verify_rows_kernel<false, true><<<grid, kRowThreads, 0, s>>>(a, parts, slices);
            else verify_rows_kernel<false, false><<<grid, kRowThreads, 0, s>>>(a, parts, slices);
        }
        cudaError_t e = cudaGetLastError();
        if (e != cudaSuccess) return e;
    }
    if (greedy) {
        verify_greedy_kernel<<<a.seqs, 32, 0, s>>>(a, parts, slices);
        return cudaGetLastError();
    }
    // CTAs a sequence: 8 (the portable cluster) from 16384 entries on
    const int ctas = a.vocab >= 16384 ? 8 : a.vocab >= 4096 ? 2 : 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(a.seqs * ctas));
    cfg.blockDim = dim3(kPickThreads);
    cfg.stream = s;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = (unsigned)ctas;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, verify_pick_kernel, a, (const RowPart*)parts, slices);
}

}  // namespace bebelm
