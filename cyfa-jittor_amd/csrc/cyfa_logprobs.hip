// cyfa_logprobs.hip -- log probabilities of given tokens with the entropy and
// the most probable alternatives of each row of logits, their mean as a
// training loss, and the gradients. For a row x [V], t its token:
//   m = max x, S = sum e^(x - m), S1 = sum (x - m) e^(x - m)
//   logprob = x_t - m - log S,  entropy = log S - S1 / S
//   dx_i = p_i (A - dH (log p_i + entropy)) + sum of the cotangents of the
//          outputs that read x_i itself,  p_i = e^(x_i - m) / S,
//          A = -(sum of the cotangents of logprob and of the alternatives)
// One pass over the row each way: the forward keeps m, log S and the entropy of
// each row for the gradient, in fp32 as every sum here.
#include "cyfa_internal.h"
#include "cyfa_rows.h"

namespace cyfa {

namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kLowest = -3.402823466e38f;
constexpr int LP_NT = 256, LP_NV = 4;   // threads and vectors per thread of a tile of a row
constexpr int LP_CAP = 1024;            // candidates for the alternatives held in LDS

// The order of the alternatives as an unsigned key: larger values first (a NaN
// largest, as torch.topk has it; -0 equals +0), then the lower index.
__device__ __forceinline__ uint32_t value_key(float x) {
    x += 0.f;
    if (x != x) return 0xffffffffu;
    const uint32_t b = __builtin_bit_cast(uint32_t, x);
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}

__device__ __forceinline__ uint64_t order_key(float x, int i) { return (uint64_t)value_key(x) << 32 | (0xffffffffu - (uint32_t)i); }

__device__ __forceinline__ float key_value(uint64_t key) {
    const uint32_t k = (uint32_t)(key >> 32);
    if (k == 0xffffffffu) return __builtin_nanf("");
    return __builtin_bit_cast(float, (k & 0x80000000u) ? k ^ 0x80000000u : ~k);
}

// (m, S, S1) of a set of elements, S1 in units of log 2.
struct RowSums {
    float m, s, s1;
};

__device__ __forceinline__ void rescale(RowSums& a, float m) {
    const float d = (a.m - m) * kLog2e;  // m is finite or +inf, never below a.m
    const float f = fast_exp2(d);
    a.s1 = f * (a.s1 + fmaxf(d, -200.f) * a.s);
    a.s *= f;
    a.m = m;
}

// Adds elements x[0 .. n): -inf counts nothing (its product with t would be a NaN).
template <int n>
__device__ __forceinline__ void add_elements(RowSums& a, const float (&x)[n]) {
    float m = a.m;
#pragma unroll
    for (int i = 0; i < n; i++) m = fmaxf(m, x[i]);
    rescale(a, m);
#pragma unroll
    for (int i = 0; i < n; i++) {
        const float t = (x[i] - m) * kLog2e, e = fast_exp2(t);
        a.s += e;
        a.s1 = fmaf(fmaxf(t, -200.f), e, a.s1);
    }
}

template <class E>
__device__ __forceinline__ const E* row_of(const LogprobParams& p, long long r) {
    return static_cast<const E*>(p.x) + (r / p.inner) * p.outer_stride + (r % p.inner) * p.row_stride;
}

template <class E>
__global__ __launch_bounds__(LP_NT) void logprobs_kernel(LogprobParams p) {
    constexpr int N = RowVec<E>::N, W = LP_NT / 64;
    __shared__ RowSums red[W];
    __shared__ uint64_t keys[W][64];
    __shared__ uint64_t cand[LP_CAP];
    __shared__ uint64_t thr_s;
    __shared__ int count_s;
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const int nvec = p.V / N, tail = p.V - nvec * N;
    for (long long r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const E* x = row_of<E>(p, r);
        // Every element of this thread with its index, tile by tile.
        const auto each_vector = [&](auto&& f) {
            for (int v0 = 0; v0 < nvec; v0 += LP_NT * LP_NV) {
                typename RowVec<E>::type v[LP_NV];
#pragma unroll
                for (int j = 0; j < LP_NV; j++) {
                    const int i = v0 + j * LP_NT + tid;
                    if (i < nvec) v[j] = load_row(x + (size_t)i * N);
                }
#pragma unroll
                for (int j = 0; j < LP_NV; j++) {
                    const int i = v0 + j * LP_NT + tid;
                    if (i < nvec) {
                        float e[N];
#pragma unroll
                        for (int c = 0; c < N; c++) e[c] = (float)v[j][c];
                        f(e, i * N);
                    }
                }
            }
        };
        const float last = tid < tail ? (float)x[nvec * N + tid] : -INFINITY;
        RowSums a = {kLowest, 0.f, 0.f};
        each_vector([&](const float (&e)[N], int) { add_elements(a, e); });
        add_elements(a, {last});
        float m = wave_max(a.m);
        rescale(a, m);
        a.s = wave_sum(a.s);
        a.s1 = wave_sum(a.s1);
        if (lane == 0) red[wv] = a;
        __syncthreads();
        a = red[0];
        for (int w = 1; w < W; w++) {
            RowSums b = red[w];
            const float mm = fmaxf(a.m, b.m);
            rescale(a, mm);
            rescale(b, mm);
            a.s += b.s;
            a.s1 += b.s1;
        }
        const float ls = logf(a.s), entropy = ls - kLn2 * (a.s1 / a.s);
        if (tid == 0) {
            const long long t = p.tokens[r];
            const bool ignored = t == p.ignore;
            const float lp = t >= 0 && t < p.V ? ((float)x[t] - a.m) - ls : __builtin_nanf("");
            p.logprob[r] = ignored ? 0.f : lp;
            if (p.entropy) p.entropy[r] = entropy;
            if (p.stats) {
                p.stats[2 * r] = a.m;
                p.stats[2 * r + 1] = ls * kLog2e;
            }
        }
        if (p.k > 0) {
            // The k-th largest of the best elements of 64 sets of threads: at
            // least k elements reach it, and seldom many more.
            uint64_t best = 0;
            const auto take = [&](float e, int i) {
                const uint64_t key = order_key(e, i);
                best = key > best ? key : best;
            };
            each_vector([&](const float (&e)[N], int i) {
#pragma unroll
                for (int c = 0; c < N; c++) take(e[c], i + c);
            });
            if (tid < tail) take(last, nvec * N + tid);
            keys[wv][lane] = best;
            if (tid == 0) count_s = 0;
            __syncthreads();
            if (wv == 0) {
                for (int w = 1; w < W; w++) best = keys[w][lane] > best ? keys[w][lane] : best;
                int rank = 0;
                for (int i = 0; i < 64; i++) rank += __shfl(best, i) > best;
                const uint64_t at = __ballot(rank == p.k - 1 && best != 0);
                const uint64_t kth = __shfl(best, at ? __builtin_ctzll(at) : 0);
                if (lane == 0) thr_s = at ? kth : 1;  // (fewer than k sets hold an element: every element)
            }
            __syncthreads();
            const uint64_t thr = thr_s;
            const auto keep = [&](float e, int i) {
                const uint64_t key = order_key(e, i);
                if (key >= thr) {
                    const int n = atomicAdd(&count_s, 1);
                    if (n < LP_CAP) cand[n] = key;
                }
            };
            each_vector([&](const float (&e)[N], int i) {
#pragma unroll
                for (int c = 0; c < N; c++) keep(e[c], i + c);
            });
            if (tid < tail) keep(last, nvec * N + tid);
            __syncthreads();
            const int n = count_s;
            const auto put = [&](int rank, uint64_t key) {
                p.top_ids[r * p.k + rank] = 0xffffffffu - (uint32_t)key;
                p.top_logprobs[r * p.k + rank] = (key_value(key) - a.m) - ls;
            };
            if (n <= LP_CAP) {
                for (int c = tid; c < n; c += LP_NT) {
                    const uint64_t key = cand[c];
                    int rank = 0;
                    for (int i = 0; i < n; i++) rank += cand[i] > key;
                    if (rank < p.k) put(rank, key);
                }
            } else {  // k rounds, each the largest key below the one before
                uint64_t below = ~0ull;
                for (int rank = 0; rank < p.k; rank++) {
                    best = 0;
                    const auto next = [&](float e, int i) {
                        const uint64_t key = order_key(e, i);
                        if (key < below && key > best) best = key;
                    };
                    each_vector([&](const float (&e)[N], int i) {
#pragma unroll
                        for (int c = 0; c < N; c++) next(e[c], i + c);
                    });
                    if (tid < tail) next(last, nvec * N + tid);
                    for (int d = 32; d > 0; d >>= 1) {
                        const uint64_t o = __shfl_xor(best, d);
                        best = o > best ? o : best;
                    }
                    __syncthreads();
                    if (lane == 0) keys[wv][0] = best;
                    __syncthreads();
                    for (int w = 0; w < W; w++) best = keys[w][0] > best ? keys[w][0] : best;
                    if (tid == 0) put(rank, best);
                    below = best;
                }
            }
        }
        __syncthreads();  // red, keys, cand and count_s are free for the next row
    }
}

// loss = -(sum of logprob over the rows whose token counts) / their number, one
// workgroup, in double and in a fixed order; no rows: 0 / 0.
__global__ __launch_bounds__(1024) void loss_mean_kernel(LogprobParams p) {
    __shared__ double sums[16];
    __shared__ double counts[16];
    double s = 0., n = 0.;
    for (long long r = threadIdx.x; r < p.rows; r += 1024)
        if (p.tokens[r] != p.ignore) {
            s += (double)p.logprob[r];
            n += 1.;
        }
    s = wave_sum(s);
    n = wave_sum(n);
    if ((threadIdx.x & 63) == 0) {
        sums[threadIdx.x >> 6] = s;
        counts[threadIdx.x >> 6] = n;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        s = n = 0.;
        for (int w = 0; w < 16; w++) {
            s += sums[w];
            n += counts[w];
        }
        *p.loss = (float)(-s / n);
        *p.count = (float)n;
    }
}

template <class E>
__global__ __launch_bounds__(LP_NT) void logprobs_grad_kernel(LogprobParams p) {
    constexpr int N = RowVec<E>::N;
    const int tid = threadIdx.x;
    const int nvec = p.V / N, tail = p.V - nvec * N;
    for (long long r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const E* x = row_of<E>(p, r);
        E* dx = static_cast<E*>(p.dx) + r * p.V;
        const long long t = p.tokens[r];
        float dlp = 0.f;
        if (t != p.ignore) dlp = p.d_loss ? -*p.d_loss / *p.count : p.d_logprob ? p.d_logprob[r] : 0.f;
        if (dlp != 0.f && (t < 0 || t >= p.V)) dlp = __builtin_nanf("");
        const float dh = p.d_entropy ? p.d_entropy[r] : 0.f;
        float total = dlp;
        bool any = dlp != 0.f || dh != 0.f;
        if (p.d_top)
            for (int j = 0; j < p.k; j++) {
                const float d = p.d_top[r * p.k + j];
                total += d;
                any |= d != 0.f;
            }
        typename RowVec<E>::type o;
        if (!any) {
#pragma unroll
            for (int c = 0; c < N; c++) o[c] = (E)0.f;
            for (int i = tid; i < nvec; i += LP_NT) store_row(dx + (size_t)i * N, o);
            if (tid < tail) dx[nvec * N + tid] = (E)0.f;
            continue;
        }
        const float m = p.stats[2 * r], ls = p.stats[2 * r + 1];
        // dx = p (a + b log2 p) for the elements that no output reads by itself
        const float a = -total - (dh != 0.f ? dh * p.entropy[r] : 0.f), b = -dh * kLn2;
        const auto grad = [&](float e) {
            const float l = (e - m) * kLog2e - ls;
            const float q = fast_exp2(l);
            return q * fmaf(fmaxf(l, -200.f), b, a);
        };
        for (int i = tid; i < nvec; i += LP_NT) {
            const typename RowVec<E>::type v = load_row(x + (size_t)i * N);
#pragma unroll
            for (int c = 0; c < N; c++) o[c] = (E)grad((float)v[c]);
            store_row(dx + (size_t)i * N, o);
        }
        if (tid < tail) dx[nvec * N + tid] = (E)grad((float)x[nvec * N + tid]);
        __syncthreads();  // the elements that outputs read are written again
        const int k = p.d_top ? p.k : 0;
        if (tid <= k) {
            const auto index = [&](int j) { return j == 0 ? t : p.top_ids[r * p.k + j - 1]; };
            const auto cot = [&](int j) { return j == 0 ? dlp : p.d_top[r * p.k + j - 1]; };
            const long long i = index(tid);
            float sum = 0.f;
            bool first = i >= 0 && i < p.V;
            for (int j = 0; j <= k; j++)
                if (index(j) == i) {
                    if (j < tid) first = false;
                    sum += cot(j);
                }
            if (first) dx[i] = (E)(grad((float)x[i]) + sum);
        }
    }
}

template <class E>
void launch(const LogprobParams& p, bool grad, hipStream_t stream) {
    const dim3 grid((unsigned)min(p.rows, (long long)LOGPROBS_MAX_GRID));
    if (grad)
        hipLaunchKernelGGL(logprobs_grad_kernel<E>, grid, dim3(LP_NT), 0, stream, p);
    else
        hipLaunchKernelGGL(logprobs_kernel<E>, grid, dim3(LP_NT), 0, stream, p);
}

}  // namespace

void launch_logprobs(const LogprobParams& p, int dtype, bool grad, hipStream_t stream) {
    if (p.rows == 0)
        ;
    else if (dtype == 0)
        launch<bf16_t>(p, grad, stream);
    else if (dtype == 1)
        launch<float>(p, grad, stream);
    else
        launch<f16_t>(p, grad, stream);
    if (!grad && p.loss) hipLaunchKernelGGL(loss_mean_kernel, dim3(1), dim3(1024), 0, stream, p);
}

}  // namespace cyfa
