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
// draft is accepted is one comparison: its rows' sums are of f32 exponentials, a thread's in f32 (about 1e-6), unless u q
// lies so near p that their error could decide; then both rows are summed in f64 as well.
//
//   verify_rows_kernel   one pass over every row that can matter: per slice the running maximum and the
//                        sum of exponentials below it (greedy: the maximum and its index). Bound: HBM.
//   verify_pick_kernel   a cluster of CTAs per sequence joins the slices, decides, and draws: each CTA
//                        holds a contiguous part of the row; the parts' sums are exchanged through distributed
//                        shared memory, and the CTA whose part the border falls into finds the place.
//   verify_greedy_kernel a warp per sequence joins the slices' maxima.
//
// Measured (logits in f32 with draft rows, vocabulary 128000): 64 sequences of 8 drafts 132 us, of which the rows' kernel
// takes 80 (557 MB at 7 TB/s: some of it lies in L2) and the pick 48 (its f64 pass; at the f64 pipe's rate 16); one sequence of
// 4 drafts 15.4 us, a chain of latencies. 24 sequences of 5 looked-up drafts, probabilities of 32003: 7.0 us.
#include <cooperative_groups.h>
#include <math_constants.h>

#include <algorithm>
#include <atomic>
#include <cstdint>
#include <type_traits>

#include "internal.h"

namespace cg = cooperative_groups;

namespace bebelm {
namespace {

constexpr int kRowThreads = 256, kMaxSlices = 64;
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
    asm volatile("griddepcontrol.launch_dependents;");
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
                float part[kU];
#pragma unroll
                for (int u = 0; u < kU; ++u)
                    part[u] = (ex2f((v[u][0] - m) * c) + ex2f((v[u][1] - m) * c)) + (ex2f((v[u][2] - m) * c) + ex2f((v[u][3] - m) * c));
                s += (part[0] + part[1]) + (part[2] + part[3]);
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

// 2^y for -1001 <= y <= 1 to 1.1e-12: y = k + f with f in [-1/2, 1/2] (k from the rounding of 1.5 * 2^52 + y), 2^f a
// polynomial of degree 8 through 2^f at the 9 Chebyshev nodes of the interval, 2^k added to the exponent. 13 f64
// operations with the product before it: the pass over a row is bound by the f64 pipe (64 a cycle and SM), and with
// exp() and its argument formed in two steps it took 2.5 times as long.
__device__ __forceinline__ double exp2_bounded(double y) {
    const double magic = 6755399441055744.0;  // 1.5 * 2^52
    const double t = y + magic, f = y - (t - magic);
    double p = 1.3255224878668817e-06;
    p = fma(p, f, 1.5310079402249296e-05);
    p = fma(p, f, 0.00015403455852453838);
    p = fma(p, f, 0.0013333450568000645);
    p = fma(p, f, 0.009618129159402558);
    p = fma(p, f, 0.05550410941205933);
    p = fma(p, f, 0.2402265069581299);
    p = fma(p, f, 0.6931471805459335);
    p = fma(p, f, 1.0);
    return __hiloint2double(__double2hiint(p) + (__double2loint(t) << 20), __double2loint(p));
}
// the same for any y <= 1: 0 below 2^-1000
__device__ __forceinline__ double exp2_neg(double y) { return y < -1000.0 ? 0.0 : exp2_bounded(y); }

// the slices of one row joined by a warp (every lane gets the answer); scale = log2(e) / temperature
__device__ __forceinline__ RowPart join_row(const RowPart* parts, int slices, double scale, bool greedy) {
    static_assert(kMaxSlices <= 64, "a lane holds two slices");
    const int lane = threadIdx.x & 31;
    RowPart p[2], r{-CUDART_INF_F, 0xffffffffu, 0.0};
#pragma unroll
    for (int i = 0; i < 2; ++i) p[i] = lane + 32 * i < slices ? parts[lane + 32 * i] : r;
    r.m = fmaxf(p[0].m, p[1].m);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) r.m = fmaxf(r.m, __shfl_xor_sync(0xffffffffu, r.m, o));
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if (greedy) {
            if (p[i].m == r.m) r.i = min(r.i, p[i].i);
        } else if (p[i].s > 0.0) {
            r.s += p[i].s * exp2_neg(((double)p[i].m - (double)r.m) * scale);
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

// the same by one thread
__device__ __forceinline__ RowPart join_row_alone(const RowPart* parts, int slices, double scale) {
    RowPart r{-CUDART_INF_F, 0xffffffffu, 0.0};
    for (int i = 0; i < slices; ++i) r.m = fmaxf(r.m, parts[i].m);
    for (int i = 0; i < slices; ++i)
        if (parts[i].s > 0.0) r.s += parts[i].s * exp2_neg(((double)parts[i].m - (double)r.m) * scale);
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

// One row of probabilities, or of logits whose probabilities are 2^(c l + k), as f64 weights.
template <bool PROBS>
struct Row {
    const float* p;
    double c, k;
    float lim;  // logits at and below it weigh nothing (2^-1000), NaN neither
    // maximum m and sum s of exp((l - m) / temperature), scale = log2(e) / temperature
    __device__ __forceinline__ void logits(float m, double s, double scale) {
        const double mc = (double)m * scale;
        if (!(s > 0.0)) {  // nothing is above -inf
            c = k = 0.0, lim = CUDART_INF_F;
        } else if (fabs(mc) >= 1073741824.0) {
            // A step of f32 at m weighs 2^-64 or less: what is not m is nothing (and c m has no bits left for the rest)
            c = 0.0, k = -log2(s), lim = nextafterf(m, -CUDART_INF_F);
        } else {
            c = scale, k = -mc - log2(s), lim = (float)((-1000.0 - k) / scale);
            if (fma((double)lim, c, k) >= -1000.0) lim = nextafterf(lim, -CUDART_INF_F);  // rounded up: the last value below
        }
    }
    __device__ __forceinline__ double weigh(float l) const {
        if constexpr (PROBS) return clean_p(l);
        const double w = exp2_bounded(fma((double)fminf(l, 3.402823466e38f), c, k));
        return l > lim ? w : 0.0;
    }
};
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// 4 entries from j (a multiple of 4); those at and past `end` count as nothing
template <bool VEC, bool PROBS>
__device__ __forceinline__ void entries4(const Row<PROBS>& r, unsigned j, unsigned end, float* v) {
    if (VEC && j + 4 <= end) {
        const float4 t = __ldg(reinterpret_cast<const float4*>(r.p + j));
        v[0] = t.x, v[1] = t.y, v[2] = t.z, v[3] = t.w;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = j + i < end ? __ldg(r.p + j + i) : -CUDART_INF_F;
    }
}

__device__ __forceinline__ double warp_total(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ double warp_running(double v) {  // lane i: the sum of lanes 0 .. i
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const double u = __shfl_up_sync(0xffffffffu, v, o);
        if ((threadIdx.x & 31) >= o) v += u;
    }
    return v;
}

// How far sums of the rows' kernel may be off, as a part of p (and q, hence twice): 2^-24 each for a thread's additions, 16
// entries at a time (5 steps with the factor of a new maximum), and 64 steps for the exponentials, whose arguments have three
// roundings and reach some log2(vocab) where they weigh.
double near_border(size_t vocab, int slices) {
    const size_t rounds = (vocab + (size_t)slices * kRowThreads * 16 - 1) / ((size_t)slices * kRowThreads * 16);
    return (double)(5 * rounds + 64) * 0x1p-23;
}

// Whether u q(x) < p(x) for draft i and its logits, from sums of both rows in f64 by the whole cluster: p(x) is x's share of
// them. The rows' factors (the target's, and 33 behind it the draft's) are the first pass's, whose error cancels. part, all:
// shared memory of two values a warp and a CTA. One draft in some ten thousand comes here, so it is a call with few
// arguments (64 sequences 132.3 us; in line, or with the rows' pointers as arguments, 133; without it 130.4).
template <int PT, bool VEC>
__device__ __noinline__ bool accepted_in_f64(const VerifyArgs* args, const Row<false>* prow, int i, double* part, double* all) {
    const int b = blockIdx.x / (int)cg::this_cluster().num_blocks();
    const Row<false>* qrow = prow + 33;
    const float* p = args->target + ((size_t)b * (args->drafts + 1) + i) * args->target_stride;
    const float* q = args->draft ? args->draft + ((size_t)b * args->drafts + i) * args->draft_stride : nullptr;
    const int x = args->tokens[(size_t)b * args->drafts + i];
    const double u = (double)args->u[(size_t)b * args->drafts + i];
    cg::cluster_group cl = cg::this_cluster();
    const int ctas = (int)cl.num_blocks(), me = (int)cl.block_rank(), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const size_t vocab = args->vocab, quads = (vocab + 3) / 4;
    const unsigned j0 = (unsigned)(4 * (quads * me / ctas)), j1 = (unsigned)min(vocab, 4 * (quads * (me + 1) / ctas));
    for (int side = 0; side < 2; ++side) {
        double sum = 0.0;
        if (side == 0 || q) {
            Row<false> r = side ? *qrow : *prow;
            r.p = side ? q : p;
            for (unsigned j = j0 + 4 * threadIdx.x; j < j1; j += 4 * PT) {
                float v[4];
                entries4<VEC>(r, j, j1, v);
                sum += (r.weigh(v[0]) + r.weigh(v[1])) + (r.weigh(v[2]) + r.weigh(v[3]));
            }
        }
        sum = warp_total(sum);
        if (lane == 0) part[2 * warp + side] = sum;
    }
    __syncthreads();
    if (warp < 2) {  // a warp per sum, into every CTA's memory
        const double v = warp_total(lane < PT / 32 ? part[2 * lane + warp] : 0.0);
        if (lane < ctas) *cl.map_shared_rank(&all[2 * me + warp], lane) = v;
    }
    cl.sync();
    double sp = 0.0, sq = 0.0;
    for (int c = 0; c < ctas; ++c) sp += all[2 * c], sq += all[2 * c + 1];
    const double wp = prow->weigh(__ldg(p + x)) / sp, wq = q ? qrow->weigh(__ldg(q + x)) / sq : 1.0;
    cl.sync();  // read by all before anything is written there again
    return u * wq < wp;
}

// PT threads; 64 registers each, so that an SM holds 1024 of them however they are split (the forms for logits spill
// some 250 bytes).
//
// The part of a CTA is cut into blocks, a block into one cell of neighbouring entries a warp; the pass leaves every
// cell's sums, so the border is found by going from the CTA to the block to the cell to the entry, and only the last
// step computes weights again, 128 of them by one warp. What has one answer a CTA (the rows' factors, the joining of
// the CTAs' sums, the search) is done by one warp: with f64 divisions and logarithms in all 1024 threads those parts
// took 15000 of 37000 cycles of a sequence.
template <int PT, bool VEC, bool PROBS>
__global__ void __launch_bounds__(PT, 1024 / PT) verify_pick_kernel(const __grid_constant__ VerifyArgs a, const RowPart* parts, int slices, double near) {
    cg::cluster_group cl = cg::this_cluster();
    cluster_arrive();  // the others have started before their memory is written
    const int ctas = (int)cl.num_blocks(), me = (int)cl.block_rank(), b = blockIdx.x / ctas;
    constexpr int kBlocks = 64, kMaxCtas = 16, kWarps = PT / 32;
    constexpr unsigned kStep = 4 * PT;
    __shared__ double s_part[kWarps][4], s_all[2][kMaxCtas][4], s_cell[kBlocks][kWarps][2], s_block[kBlocks];
    __shared__ double s_prob[2][33];  // p_i(x_i), q_i(x_i)
    __shared__ Row<PROBS> s_row[2][33];
    __shared__ double s_before, s_border, s_fp, s_fq;
    __shared__ int s_owner;
    const int n = drafts_of(a, b), lane = threadIdx.x & 31;
    // lane 0's, which makes it the warp's for the compiler too (one sequence 16.8 -> 16.4 us, 64 134 -> 132 us)
    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0);
    const int* tok = a.tokens + (size_t)b * a.drafts;
    const double scale = 1.4426950408889634074 / (double)a.temperature;
    const RowPart* tp = parts + (size_t)b * (a.drafts + 1) * slices;
    const RowPart* dp = parts + ((size_t)a.seqs * (a.drafts + 1) + (size_t)b * a.drafts) * slices;
    const float* trow = a.target + (size_t)b * (a.drafts + 1) * a.target_stride;
    const float* drow = a.draft ? a.draft + (size_t)b * a.drafts * a.draft_stride : nullptr;
    const float u_sample = a.u_sample[b];
    asm volatile("griddepcontrol.wait;" ::: "memory");

    // ---- the decisions, in groups of 32 drafts (every CTA makes them for itself) ----
    int n_acc = 0, base = 0;
    bool others_started = false;
    for (;;) {
        const int cnt = min(32, n - base);
        const double u = lane < cnt ? (double)a.u[(size_t)b * a.drafts + base + lane] : 0.0;
        // p and q of each draft, and the factors of its rows and of the row behind the group: a warp each, or a
        // thread each where rows were cut into few slices
        auto decide = [&](int k, auto one_thread) {
            constexpr bool kAlone = decltype(one_thread)::value;
            const int at = k >> 1, i = base + at, side = k & 1, x = at < cnt ? tok[i] : -1;
            double v = side ? 1.0 : 0.0;
            if (side == 0 || drow) {
                const float* p = side ? drow + (size_t)i * a.draft_stride : trow + (size_t)i * a.target_stride;
                const bool in = x >= 0 && (size_t)x < a.vocab;
                const float l = in ? __ldg(p + x) : 0.f;
                if constexpr (PROBS) {
                    if (in) v = clean_p(l);
                } else {
                    const RowPart* rp = (side ? dp : tp) + (size_t)i * slices;
                    RowPart r;
                    if constexpr (kAlone)
                        r = join_row_alone(rp, slices, scale);
                    else
                        r = join_row(rp, slices, scale, false);
                    if (kAlone || lane == 0) {
                        if (in) v = r.s > 0.0 ? exp2_neg(((double)clean(l) - (double)r.m) * scale) / r.s : 0.0;
                        s_row[side][at].logits(r.m, r.s, scale);
                    }
                }
            }
            if (kAlone || lane == 0) s_prob[side][at] = v;
        };
        if (PROBS || slices <= 4) {
            for (int k = threadIdx.x; k <= 2 * cnt; k += PT) decide(k, std::true_type{});
        } else {
            for (int k = warp; k <= 2 * cnt; k += kWarps) decide(k, std::false_type{});
        }
        __syncthreads();
        const double uq = lane < cnt ? u * s_prob[1][lane] : 0.0, pr = lane < cnt ? s_prob[0][lane] : 0.0;
        unsigned yes = __ballot_sync(0xffffffffu, lane < cnt && uq < pr);
        if constexpr (!PROBS) {
            // the first refused draft and those before it that are near their border (the same ones in every warp and CTA)
            unsigned unsure = __ballot_sync(0xffffffffu, pr > 0.0 && fabs(uq - pr) <= near * pr);
            while (const unsigned left = unsure & (yes ^ (yes + 1))) {
                const int at = __ffs((int)left) - 1, i = base + at;
                if (!others_started) cluster_wait(), others_started = true;
                const bool ok = accepted_in_f64<PT, VEC>(&a, &s_row[0][at], i, &s_part[0][0], &s_all[0][0][0]);
                yes = ok ? yes | 1u << at : yes & ~(1u << at);
                unsure &= ~(1u << at);
            }
        }
        const int run = __ffs((int)~yes) - 1;  // drafts accepted; -1: all 32
        const int got = run < 0 ? 32 : run;
        n_acc = base + got;
        if (got < cnt || base + cnt == n) break;
        base += 32;
        __syncthreads();
    }

    // ---- the rows the next token is drawn from ----
    const bool refused = n_acc < n;
    const bool with_q = refused && drow;
    const int skip = refused && !drow ? tok[n_acc] : -1;  // a certain draft takes its own place away
    Row<PROBS> P{}, Q{};
    if constexpr (!PROBS) {  // normalised by the sums of the first pass
        P = s_row[0][n_acc - base];
        if (with_q) Q = s_row[1][n_acc - base];
    }
    P.p = trow + (size_t)n_acc * a.target_stride;
    Q.p = with_q ? drow + (size_t)n_acc * a.draft_stride : P.p;
    // this CTA's part of the row, whole groups of 4
    const size_t quads = (a.vocab + 3) / 4;
    const unsigned j0 = (unsigned)(4 * (quads * me / ctas)), j1 = (unsigned)min(a.vocab, 4 * (quads * (me + 1) / ctas));

    // The row is gone through once for all sums. p and q are normalised by the first pass's f32-grade sums, which
    // decides p > q as well as exact ones (it differs only where p - q is 1e-7 of p, and weighs as little); with the
    // sums Sp, Sq of p and q, and A, B of p and q where p > q, the weights' total is A / Sp - B / Sq.
    // Probabilities in hand are differences at once: A.
    const bool ratio = with_q && !PROBS;
    // of the entries j .. j + 3: their shares of Sp, Sq, A, B
    auto add4 = [&](auto use_q, unsigned j, bool plain, double* sums) {
        constexpr bool kQ = decltype(use_q)::value;
        float x[4], y[4];
        entries4<VEC>(P, j, j1, x);
        if constexpr (kQ) entries4<VEC>(Q, j, j1, y);
        const int sk = !plain && skip >= 0 && (unsigned)skip - j < 4 ? skip - (int)j : -1;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const double p = P.weigh(x[i]);
            if constexpr (kQ) {
                const double q = Q.weigh(y[i]);
                if constexpr (PROBS) {
                    sums[2] += fmax(p - q, 0.0);
                } else {
                    sums[0] += p, sums[1] += q;
                    if (p > q) sums[2] += p, sums[3] += q;
                }
            } else {
                if (i != sk) sums[2] += p;
            }
        }
    };
    const int steps = (int)((j1 - j0 + kStep - 1) / kStep);
    int shift = 0;  // steps of a block
    while (steps >> shift >= kBlocks) ++shift;
    const int blocks = (steps + (1 << shift) - 1) >> shift;
    const unsigned cell = 128u << shift, block_entries = cell * kWarps;
    bool plain = !refused;
    if (!others_started) cluster_wait();
    for (int slot = 0;; ++slot) {  // a second time only where p - q is zero everywhere
        double sums[4] = {0.0, 0.0, 0.0, 0.0}, all_a = 0.0, all_b = 0.0;
        auto go = [&](auto use_q) {
            constexpr bool kRatio = decltype(use_q)::value && !PROBS;
            for (int t = 0; t < blocks; ++t) {
                const unsigned c0 = j0 + t * block_entries + warp * cell + 4 * lane;
                for (int r = 0; r < 1 << shift; ++r)
                    if (c0 + 128 * r < j1) add4(use_q, c0 + 128 * r, plain, sums);
                const double u = warp_total(sums[2]);
                double v = 0.0;
                if constexpr (kRatio) v = warp_total(sums[3]);
                sums[2] = sums[3] = 0.0;
                all_a += u, all_b += v;
                if (lane == 0) s_cell[t][warp][0] = u, s_cell[t][warp][1] = v;
            }
            if constexpr (kRatio) sums[0] = warp_total(sums[0]), sums[1] = warp_total(sums[1]);
        };
        if (with_q && !plain)
            go(std::true_type{});
        else
            go(std::false_type{});
        if (lane == 0) s_part[warp][0] = sums[0], s_part[warp][1] = sums[1], s_part[warp][2] = all_a, s_part[warp][3] = all_b;
        __syncthreads();
        if (warp < 4) {  // a warp per sum, into every CTA's memory
            const double v = warp_total(lane < kWarps ? s_part[lane][warp] : 0.0);
            if (lane < ctas) *cl.map_shared_rank(&s_all[slot][me][warp], lane) = v;
        }
        cl.sync();
        if (warp == 0) {
            const bool in = lane < ctas;
            const double* c = s_all[slot][in ? lane : 0];
            double fp = 1.0, fq = 1.0, own = in ? c[2] : 0.0;
            if (ratio && !plain) {
                const double sp = warp_total(in ? c[0] : 0.0), sq = warp_total(in ? c[1] : 0.0);
                fp = sp > 0.0 ? 1.0 / sp : 0.0, fq = sq > 0.0 ? 1.0 / sq : 0.0;
                own = in ? fmax(fma(c[2], fp, -(c[3] * fq)), 0.0) : 0.0;
            }
            const double run = warp_running(own), total = __shfl_sync(0xffffffffu, run, 31);
            // The first CTA whose sum passes the border, or, if rounding leaves none, the last with any weight.
            const double border = (double)u_sample * total;
            const unsigned any = __ballot_sync(0xffffffffu, own > 0.0), over = __ballot_sync(0xffffffffu, own > 0.0 && run > border);
            const double before = __shfl_up_sync(0xffffffffu, run, 1);
            if (lane == me) s_before = me ? before : 0.0;
            if (lane == 0) {
                s_border = border, s_fp = fp, s_fq = fq;
                s_owner = over ? __ffs((int)over) - 1 : any ? 31 - __clz((int)any) : -1;
            }
        }
        __syncthreads();
        if (s_owner >= 0 || plain) break;
        plain = true;
        __syncthreads();
    }
    if (s_owner < 0) {  // a row without any weight
        if (me == 0 && warp == 0) write_out(a, b, n_acc, 0);
        return;
    }
    if (me != s_owner) return;
    const double border = s_border, fp = s_fp, fq = s_fq;
    const bool diff = ratio && !plain;
    auto weight = [&](double u, double v) { return diff ? fmax(fma(u, fp, -(v * fq)), 0.0) : u; };
    // every cell's weight and the weights of the blocks
    for (int t = warp; t < blocks; t += kWarps) {
        const double w = lane < kWarps ? weight(s_cell[t][lane][0], s_cell[t][lane][1]) : 0.0;
        if (lane < kWarps) s_cell[t][lane][0] = w;
        const double sum = warp_total(w);
        if (lane == 0) s_block[t] = sum;
    }
    __syncthreads();
    if (warp) return;
    // Of 32 weights in order behind `run`: the first whose running sum passes the border, if there is none the last
    // with any weight, -1 if there is none either; `run` becomes the sum before it (or of all).
    auto find = [&](double w, double& run, bool& passed) {
        const double inc = run + warp_running(w);
        const unsigned over = __ballot_sync(0xffffffffu, w > 0.0 && inc > border), any = __ballot_sync(0xffffffffu, w > 0.0);
        passed = over != 0;
        const int at = over ? __ffs((int)over) - 1 : any ? 31 - __clz((int)any) : -1;
        const double prev = __shfl_up_sync(0xffffffffu, inc, 1);
        run = over ? (at ? __shfl_sync(0xffffffffu, prev, at) : run) : __shfl_sync(0xffffffffu, inc, 31);
        return at;
    };
    double run = s_before, behind = 0.0;
    bool passed = false;
    int block = 0;
    for (int t = 0; t < blocks && !passed; t += 32) {
        const double w = t + lane < blocks ? s_block[t + lane] : 0.0, start = run;
        const int at = find(w, run, passed);
        if (at >= 0) block = t + at, behind = passed ? run : start + (at ? __shfl_sync(0xffffffffu, warp_running(w), at - 1) : 0.0);
    }
    run = behind;
    const double cw = lane < kWarps ? s_cell[block][lane][0] : 0.0;
    const double start = run;
    const int cat = max(find(cw, run, passed), 0);
    if (!passed) run = start + (cat ? __shfl_sync(0xffffffffu, warp_running(cw), cat - 1) : 0.0);
    // the cell's entries, 4 a lane in order
    const unsigned c0 = j0 + block * block_entries + cat * cell, c1 = min(j1, c0 + cell);
    int place = -1, last = 0;
    for (unsigned t0 = c0; t0 < c1 && place < 0; t0 += 128) {
        const unsigned j = t0 + 4 * lane;
        double v[4] = {0.0, 0.0, 0.0, 0.0};
        int mine = -1, lastw = -1;
        if (j < c1) {
            float x[4], y[4];
            entries4<VEC>(P, j, j1, x);
            if (with_q && !plain) entries4<VEC>(Q, j, j1, y);
            const int sk = !plain && skip >= 0 && (unsigned)skip - j < 4 ? skip - (int)j : -1;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[i] = P.weigh(x[i]);
                if (with_q && !plain) {
                    const double q = Q.weigh(y[i]);
                    if (v[i] > q) lastw = (int)(j + i);
                    v[i] = v[i] > q ? fmax(fma(v[i], fp, -(q * fq)), 0.0) : 0.0;
                } else if (i == sk) {
                    v[i] = 0.0;
                } else if (v[i] > 0.0) {
                    lastw = (int)(j + i);
                }
            }
        }
        const double sum = (v[0] + v[1]) + (v[2] + v[3]), inc = warp_running(sum);
        double at = run + (inc - sum);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            at += v[i];
            if (v[i] > 0.0 && at > border && mine < 0) mine = (int)(j + i);
        }
        const unsigned hit = __ballot_sync(0xffffffffu, mine >= 0);
        if (hit) place = __shfl_sync(0xffffffffu, mine, __ffs((int)hit) - 1);
        last = max(last, __reduce_max_sync(0xffffffffu, lastw));
        run += __shfl_sync(0xffffffffu, inc, 31);
    }
    write_out(a, b, n_acc, place >= 0 ? place : last);
}

// CTAs a sequence: parts of 4096 entries at least, up to the portable cluster of 8
int pick_ctas(const VerifyArgs& a) {
    int ctas = 1;
    while (ctas < 8 && a.vocab >= (size_t)ctas * 8192) ctas *= 2;
    return ctas;
}

// Whether a device runs clusters of 16 CTAs of a kernel, which have to be asked for; asked once a device. Where the
// answer is an error it is no.
bool clusters_of_16(const void* kernel, int threads, std::atomic<int>* known) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return false;
    int k = known[dev].load(std::memory_order_acquire);
    if (k) return k > 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(16);
    cfg.blockDim = dim3((unsigned)threads);
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = 16;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    int n = 0;
    const bool yes = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess &&
                     cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) == cudaSuccess && n > 0;
    if (!yes) cudaGetLastError();
    known[dev].store(yes ? 2 : 1, std::memory_order_release);
    return yes;
}

template <int PT, bool VEC, bool PROBS>
cudaError_t launch_pick(const VerifyArgs& a, const RowPart* parts, int slices, int num_sms, cudaStream_t s) {
    auto kernel = verify_pick_kernel<PT, VEC, PROBS>;
    int ctas = pick_ctas(a);
    static std::atomic<int> known[64];
    if (PT == 1024 && a.vocab >= 65536 && a.seqs * 16 <= num_sms && clusters_of_16(reinterpret_cast<const void*>(kernel), PT, known))
        ctas = 16;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(a.seqs * ctas));
    cfg.blockDim = dim3(PT);
    cfg.stream = s;
    cudaLaunchAttribute at[2] = {};
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)ctas;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // behind the rows' kernel
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = PROBS ? 1 : 2;
    return cudaLaunchKernelEx(&cfg, kernel, a, parts, slices, near_border(a.vocab, slices));
}

template <bool PROBS>
cudaError_t pick_probs(const VerifyArgs& a, const RowPart* parts, int slices, bool vec, int num_sms, cudaStream_t s) {
    // few sequences: a CTA's part of a row should be few steps; many: four CTAs an SM share its latencies
    if (a.seqs * pick_ctas(a) <= num_sms)
        return vec ? launch_pick<1024, true, PROBS>(a, parts, slices, num_sms, s)
                   : launch_pick<1024, false, PROBS>(a, parts, slices, num_sms, s);
    return vec ? launch_pick<256, true, PROBS>(a, parts, slices, num_sms, s)
               : launch_pick<256, false, PROBS>(a, parts, slices, num_sms, s);
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
    return a.probs ? pick_probs<true>(a, parts, slices, vec, num_sms, s) : pick_probs<false>(a, parts, slices, vec, num_sms, s);
}

}  // namespace bebelm
