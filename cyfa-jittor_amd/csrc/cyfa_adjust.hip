// cyfa_adjust.hip -- logits as a sampler wants them: penalties for tokens that a
// sequence holds already, biases and a grammar's mask, and the gradient. For the
// logit x of column j, n its occurrences in the row's history and c those from
// the prompt's end on:
//   y = x > 0 ? x / repetition : x repetition                where n > 0
//   y -= c frequency + presence                              where c > 0
//   y += bias_j + the row's values for token j
//   y = -inf                                                 where j is not allowed
//   dx = dy (n > 0 ? (x > 0 ? 1 / repetition : repetition) : 1), 0 where j is not allowed
// in fp32, every product and sum rounded by itself, y rounded once.
//
// A workgroup takes a row's slice of columns: it counts the history's tokens that
// fall into the slice in LDS (a word a column: the top bit for any occurrence,
// the others count those behind the prompt; integers, so that their order does
// not matter), then passes over the slice once.
#include "cyfa_internal.h"
#include "cyfa_rows.h"

namespace cyfa {

namespace {

constexpr int AJ_NT = 256;
constexpr int AJ_NV = 4;            // vectors of a thread in flight
constexpr int AJ_COLS = 8192;       // most columns of a slice: 32 KiB of LDS, half as many where it holds the tokens' biases too
constexpr uint32_t AJ_SEEN = 0x80000000u;

template <class I>
__device__ void count_tokens(const AdjustParams& p, const I* ids, long long n, long long prompt, int c0, int cols, uint32_t* counts) {
    constexpr int U = 8;
    for (long long i0 = threadIdx.x; i0 < n; i0 += AJ_NT * U) {
        I t[U];
#pragma unroll
        for (int u = 0; u < U; u++) t[u] = ids[min(i0 + u * AJ_NT, n - 1)];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const long long i = i0 + u * AJ_NT, c = (long long)t[u] - c0;
            if (i < n && c >= 0 && c < cols) {
                if (i < prompt)
                    atomicOr(&counts[c], AJ_SEEN);
                else
                    atomicAdd(&counts[c], 1u);
            }
        }
    }
}

template <class E, bool GRAD, bool TOKENS>
__global__ __launch_bounds__(AJ_NT) void adjust_kernel(AdjustParams p) {
#pragma clang fp contract(off)
    constexpr int N = RowVec<E>::N;
    extern __shared__ uint32_t lds[];
    uint32_t* counts = lds;                                    // [p.cols] with a history
    float* values = (float*)(lds + (p.L > 0 ? p.cols : 0));    // [p.cols] with the tokens' biases
    __shared__ int ids_s[TOKENS ? ADJUST_MAX_TOKENS : 1];
    __shared__ float values_s[TOKENS ? ADJUST_MAX_TOKENS : 1];
    const int tid = threadIdx.x;
    const long long slices = (p.V + p.cols - 1) / p.cols;
    for (long long job = blockIdx.x; job < p.jobs; job += gridDim.x) {
        // The slices of a row, which read the same history, go to one XCD's L2
        // (consecutive workgroups run on the eight XCDs in turn).
        long long r, s;
        if (p.rows >= 8) {
            r = job / (8 * slices) * 8 + job % 8;
            s = job / 8 % slices;
            if (r >= p.rows) continue;
        } else {
            r = job / slices;
            s = job % slices;
        }
        const long long ro = r / p.inner, ri = r % p.inner;
        const int c0 = (int)s * p.cols, cols = min(p.cols, p.V - c0);
        const E* x = static_cast<const E*>(p.x) + ro * p.x_outer + ri * p.x_row + c0;
        const E* dy = static_cast<const E*>(p.dy) + (GRAD ? r * p.V + c0 : 0);
        E* y = static_cast<E*>(p.y) + ro * p.y_outer + ri * p.y_row + c0;
        const float repetition = p.repetitions ? p.repetitions[r] : p.repetition;
        const float presence = p.presences ? p.presences[r] : p.presence;
        const float frequency = p.frequencies ? p.frequencies[r] : p.frequency;
        const bool history = p.L > 0;
        __syncthreads();  // the row before is done with the LDS
        if (history)
            for (int c = tid; c < p.cols; c += AJ_NT) counts[c] = 0;
        if (TOKENS) {
            for (int c = tid; c < p.cols; c += AJ_NT) values[c] = 0.f;
            const long long* ids = p.token_ids + ro * p.ti_outer + ri * p.ti_row;
            const float* v = p.token_values + ro * p.tv_outer + ri * p.tv_row;
            for (int i = tid; i < p.n_tokens; i += AJ_NT) {
                const long long c = ids[i] - c0;
                ids_s[i] = c >= 0 && c < cols ? (int)c : -1;
                values_s[i] = v[i];
            }
        }
        __syncthreads();
        if (history) {
            const long long n = p.lengths ? max(0ll, min(p.L, p.lengths[r])) : p.L;
            const long long prompt = p.prompts ? p.prompts[r] : 0;
            if (p.wide)
                count_tokens(p, static_cast<const long long*>(p.history) + ro * p.h_outer + ri * p.h_row, n, prompt, c0, cols, counts);
            else
                count_tokens(p, static_cast<const int*>(p.history) + ro * p.h_outer + ri * p.h_row, n, prompt, c0, cols, counts);
        }
        if (TOKENS)
            // the first entry of a token adds all of its entries, in their order
            for (int i = tid; i < p.n_tokens; i += AJ_NT) {
                const int c = ids_s[i];
                if (c < 0) continue;
                bool first = true;
                float sum = 0.f;
                for (int j = 0; j < p.n_tokens; j++)
                    if (ids_s[j] == c) {
                        if (j < i) first = false;
                        sum += values_s[j];
                    }
                if (first) values[c] = sum;
            }
        __syncthreads();
        const float* bias = p.bias ? p.bias + ro * p.b_outer + ri * p.b_row + c0 : nullptr;
        const unsigned char* allowed = p.allowed ? static_cast<const unsigned char*>(p.allowed) + ro * p.a_outer + ri * p.a_row : nullptr;
        const auto one = [&](float e, int c, bool keep) {
            const uint32_t w = history ? counts[c] : 0;
            if (GRAD) {
                if (w && e != 0.f) {
                    const float xc = (float)x[c];
                    e *= xc > 0.f ? 1.f / repetition : repetition;
                }
                return keep ? e : 0.f;
            }
            if (w) {
                e = e > 0.f ? e / repetition : e * repetition;
                const uint32_t made = w & ~AJ_SEEN;
                if (made) e = e - ((float)made * frequency + presence);
            }
            if (bias) e = e + bias[c];
            if (TOKENS) e = e + values[c];
            return keep ? e : -INFINITY;
        };
        const auto kept = [&](int c) {
            if (!allowed) return true;
            const int j = c0 + c;
            return p.packed ? (allowed[j >> 3] >> (j & 7) & 1) != 0 : allowed[j] != 0;
        };
        const E* from = GRAD ? dy : x;
        const int nvec = cols / N, tail = cols - nvec * N;
        for (int i0 = 0; i0 < nvec; i0 += AJ_NT * AJ_NV) {
            typename RowVec<E>::type v[AJ_NV];
#pragma unroll
            for (int j = 0; j < AJ_NV; j++) v[j] = load_row(from + (size_t)min(i0 + j * AJ_NT + tid, nvec - 1) * N);
#pragma unroll
            for (int j = 0; j < AJ_NV; j++) {
                const int i = i0 + j * AJ_NT + tid;
                if (i < nvec) {
                    typename RowVec<E>::type o;
#pragma unroll
                    for (int c = 0; c < N; c++) o[c] = (E)one((float)v[j][c], i * N + c, kept(i * N + c));
                    store_row(y + (size_t)i * N, o);
                }
            }
        }
        if (tid < tail) {
            const int c = nvec * N + tid;
            y[c] = (E)one((float)from[c], c, kept(c));
        }
    }
}

template <class E>
void launch(AdjustParams p, bool grad, hipStream_t stream) {
    // Slices of a row so that some thousand workgroups fill the compute units.
    const long long want = p.rows * p.V / 1024;
    const bool tokens = !grad && p.n_tokens > 0;
    p.cols = (int)min(max((want + 31) / 32 * 32, 1024ll), (long long)(tokens ? AJ_COLS / 2 : AJ_COLS));
    const long long slices = (p.V + p.cols - 1) / p.cols;
    p.jobs = (p.rows >= 8 ? (p.rows + 7) / 8 * 8 : p.rows) * slices;
    const dim3 grid((unsigned)min(p.jobs, (long long)LOGPROBS_MAX_GRID));
    const size_t lds = (size_t)p.cols * 4 * ((p.L > 0) + tokens);
    if (grad)
        hipLaunchKernelGGL((adjust_kernel<E, true, false>), grid, dim3(AJ_NT), lds, stream, p);
    else if (tokens)
        hipLaunchKernelGGL((adjust_kernel<E, false, true>), grid, dim3(AJ_NT), lds, stream, p);
    else
        hipLaunchKernelGGL((adjust_kernel<E, false, false>), grid, dim3(AJ_NT), lds, stream, p);
}

}  // namespace

void launch_adjust(const AdjustParams& p, int dtype, bool grad, hipStream_t stream) {
    if (dtype == 0)
        launch<bf16_t>(p, grad, stream);
    else if (dtype == 1)
        launch<float>(p, grad, stream);
    else
        launch<f16_t>(p, grad, stream);
}

}  // namespace cyfa
