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
// A workgroup takes a row's slice of columns. It counts the history's tokens that
// fall into the slice in LDS (a word a column: the top bit for any occurrence,
// the low ones count those behind the prompt; integers, so that their order does
// not matter) and lists the columns that it meets, whose results it forms one by
// one; the slice itself is passed over as where nothing is repeated, and the
// listed columns are stored a second time. So the pass reads no counts, and runs
// at the memory's rate.
#include "cyfa_internal.h"
#include "cyfa_rows.h"

namespace cyfa {

namespace {

constexpr int AJ_NT = 256;
constexpr int AJ_NV = 4;            // vectors of a thread in flight
constexpr int AJ_COLS = 8192;       // most columns of a slice: 48 KiB of LDS, half as many where it holds the tokens' biases too
constexpr uint32_t AJ_SEEN = 0x80000000u, AJ_BIASED = 0x40000000u, AJ_MADE = 0x3fffffffu;

// A slice's columns that the history or the tokens' biases name: counts [cols],
// their list and its length.
struct Touched {
    uint32_t* counts;
    uint16_t* list;
    int* n;
    __device__ __forceinline__ void met(uint32_t before, int c) const {
        if (before == 0) list[atomicAdd(n, 1)] = (uint16_t)c;
    }
};

template <class I>
__device__ void count_tokens(const I* ids, long long n, long long prompt, int c0, int cols, const Touched& touched) {
    constexpr int U = 8;
    for (long long i0 = threadIdx.x; i0 < n; i0 += AJ_NT * U) {
        I t[U];
#pragma unroll
        for (int u = 0; u < U; u++) t[u] = ids[min(i0 + u * AJ_NT, n - 1)];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const long long i = i0 + u * AJ_NT, c = (long long)t[u] - c0;
            if (i < n && c >= 0 && c < cols)  // (AJ_SEEN and a one: the count of what is behind the prompt, too)
                touched.met(i < prompt ? atomicOr(&touched.counts[c], AJ_SEEN) : atomicAdd(&touched.counts[c], 1u), (int)c);
        }
    }
}

template <class E, bool GRAD, bool TOKENS>
__global__ __launch_bounds__(AJ_NT) void adjust_kernel(AdjustParams p) {
#pragma clang fp contract(off)
    typedef typename RowVec<E>::type Vec;
    constexpr int N = RowVec<E>::N;
    extern __shared__ __align__(16) uint32_t lds[];
    __shared__ int ids_s[TOKENS ? ADJUST_MAX_TOKENS : 1];
    __shared__ float values_s[TOKENS ? ADJUST_MAX_TOKENS : 1];
    __shared__ int listed_s;
    const int tid = threadIdx.x;
    const bool history = p.L > 0, touches = history || TOKENS;
    const Touched touched = {lds, reinterpret_cast<uint16_t*>(lds + p.cols * (TOKENS ? 2 : 1)), &listed_s};
    float* values = reinterpret_cast<float*>(lds + p.cols);  // TOKENS: [cols], the tokens' biases
    const long long slices = (p.V + p.cols - 1) / p.cols;
    const long long job = p.first + blockIdx.x;
    // The slices of a row, which read the same history, go to one XCD's L2
    // (consecutive workgroups run on the eight XCDs in turn).
    long long r, s;
    if (p.rows >= 8) {
        r = job / (8 * slices) * 8 + job % 8;
        s = job / 8 % slices;
        if (r >= p.rows) return;
    } else {
        r = job / slices;
        s = job % slices;
    }
    const long long ro = r / p.inner, ri = r % p.inner;
    const int c0 = (int)s * p.cols, cols = min(p.cols, p.V - c0);
    const E* x = static_cast<const E*>(p.x) + ro * p.x_outer + ri * p.x_row + c0;
    const E* from = GRAD ? static_cast<const E*>(p.dy) + r * p.V + c0 : x;
    E* y = static_cast<E*>(p.y) + ro * p.y_outer + ri * p.y_row + c0;
    const float* bias = !GRAD && p.bias ? p.bias + ro * p.b_outer + ri * p.b_row + c0 : nullptr;
    const unsigned char* allowed =
        p.allowed ? static_cast<const unsigned char*>(p.allowed) + ro * p.a_outer + ri * p.a_row + (p.packed ? c0 / 8 : c0) : nullptr;
    const auto kept = [&](int c) { return !allowed || (p.packed ? (allowed[c >> 3] >> (c & 7) & 1) != 0 : allowed[c] != 0); };
    if (touches) {
        for (int c = tid * 4; c < p.cols; c += AJ_NT * 4) {
            *reinterpret_cast<uint4*>(touched.counts + c) = uint4{0, 0, 0, 0};
            if (TOKENS) *reinterpret_cast<float4*>(values + c) = float4{0.f, 0.f, 0.f, 0.f};
        }
        if (tid == 0) listed_s = 0;
        if (TOKENS) {
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
            const long long n = p.lengths ? max(0ll, min(p.L, p.lengths[r])) : p.L, prompt = p.prompts ? p.prompts[r] : 0;
            const long long at = ro * p.h_outer + ri * p.h_row;
            if (p.wide)
                count_tokens(static_cast<const long long*>(p.history) + at, n, prompt, c0, cols, touched);
            else
                count_tokens(static_cast<const int*>(p.history) + at, n, prompt, c0, cols, touched);
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
                if (first) {
                    values[c] = sum;
                    touched.met(atomicOr(&touched.counts[c], AJ_BIASED), c);
                }
            }
        __syncthreads();
        // the listed columns' results, in place of their counts
        const float repetition = p.repetitions ? p.repetitions[r] : p.repetition;
        const float presence = p.presences ? p.presences[r] : p.presence;
        const float frequency = p.frequencies ? p.frequencies[r] : p.frequency;
        for (int i = tid; i < listed_s; i += AJ_NT) {
            const int c = touched.list[i];
            const uint32_t w = touched.counts[c], made = w & AJ_MADE;
            const float xc = (float)x[c];
            float e;
            if (GRAD) {
                e = (float)from[c];
                if (e != 0.f) e *= xc > 0.f ? 1.f / repetition : repetition;
                e = kept(c) ? e : 0.f;
            } else {
                e = xc;
                if (made || (w & AJ_SEEN)) e = e > 0.f ? e / repetition : e * repetition;
                if (made) e = e - ((float)made * frequency + presence);
                if (bias) e = e + bias[c];
                if (TOKENS && (w & AJ_BIASED)) e = e + values[c];
                e = kept(c) ? e : -INFINITY;
            }
            touched.counts[c] = __builtin_bit_cast(uint32_t, e);
        }
        __syncthreads();  // (y may be x)
    }
    const int nvec = cols / N, tail = cols - nvec * N;
    const float out = GRAD ? 0.f : -INFINITY;
    for (int i0 = 0; i0 < nvec; i0 += AJ_NT * AJ_NV) {
        Vec v[AJ_NV];
        uint32_t keep[AJ_NV][N / 4];  // bytes or bits of the mask
#pragma unroll
        for (int j = 0; j < AJ_NV; j++) v[j] = load_row(from + (size_t)min(i0 + j * AJ_NT + tid, nvec - 1) * N);
        if (allowed)
#pragma unroll
            for (int j = 0; j < AJ_NV; j++) {
                const int c = min(i0 + j * AJ_NT + tid, nvec - 1) * N;
                if (p.packed)
                    keep[j][0] = allowed[c >> 3] >> (c & 7);
                else
                    __builtin_memcpy(keep[j], allowed + c, N);
            }
#pragma unroll
        for (int j = 0; j < AJ_NV; j++) {
            const int i = i0 + j * AJ_NT + tid;
            if (i >= nvec) continue;
            if (bias) {
                float b[N];
                __builtin_memcpy(b, bias + (size_t)i * N, sizeof b);
#pragma unroll
                for (int c = 0; c < N; c++) v[j][c] = (E)((float)v[j][c] + b[c]);
            }
            if (allowed) {
#pragma unroll
                for (int c = 0; c < N; c++) {
                    const bool k = p.packed ? (keep[j][0] >> c & 1) != 0 : (keep[j][c / 4] >> (c % 4 * 8) & 0xff) != 0;
                    v[j][c] = k ? v[j][c] : (E)out;
                }
            }
            store_row(y + (size_t)i * N, v[j]);
        }
    }
    if (tid < tail) {
        const int c = nvec * N + tid;
        float e = (float)from[c];
        if (bias) e = e + bias[c];
        y[c] = (E)(kept(c) ? e : out);
    }
    if (touches) {
        __syncthreads();  // the listed columns are stored again
        for (int i = tid; i < listed_s; i += AJ_NT) {
            const int c = touched.list[i];
            y[c] = (E)__builtin_bit_cast(float, touched.counts[c]);
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
    const long long jobs = (p.rows >= 8 ? (p.rows + 7) / 8 * 8 : p.rows) * slices;
    const size_t lds = p.L > 0 || tokens ? (size_t)p.cols * (tokens ? 10 : 6) : 0;
    for (p.first = 0; p.first < jobs; p.first += LOGPROBS_MAX_GRID) {
        const dim3 grid((unsigned)min(jobs - p.first, (long long)LOGPROBS_MAX_GRID));
        if (grad)
            hipLaunchKernelGGL((adjust_kernel<E, true, false>), grid, dim3(AJ_NT), lds, stream, p);
        else if (tokens)
            hipLaunchKernelGGL((adjust_kernel<E, false, true>), grid, dim3(AJ_NT), lds, stream, p);
        else
            hipLaunchKernelGGL((adjust_kernel<E, false, false>), grid, dim3(AJ_NT), lds, stream, p);
    }
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
