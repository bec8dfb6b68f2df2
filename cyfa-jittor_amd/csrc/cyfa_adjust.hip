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
// fall into the slice in LDS (16 bits a column where the history is no longer than
// they count, else 32: the top bit for any occurrence, the low ones count those
// behind the prompt; integers, so that their order does not matter) and lists the
// columns that it meets; the slice is passed over as where nothing is repeated,
// and the listed columns are formed and stored a second time. So the pass reads no
// counts and does not wait for them. Where many columns are met, or many workgroups
// take turns anyway, it does read them, and nothing is stored twice. (In place a
// listed column's logit is gone after the pass, which is made for what it has met.)
//
// Bound by memory where rows are many. On MI355X 4096 x 32000 bf16 with histories of
// up to 1280 tokens, each shared by 1024 rows, take 110 us (0.52 GB: 4.8 TB/s, where
// a copy of 1 GiB moves 5.0 to 5.2) and their gradient 125, which reads the logits of
// the vectors with a column that was met besides (0.09 GB more); 256 x 50001 fp16
// with a bias, a mask of bytes and 8191 tokens a row 29 to 31 (81 MB, 2.7 TB/s: two slices
// of a row each read its tokens and mark them one by one before their pass). Few rows
// are bound by the steps of a workgroup, the tokens' load, the marks, the list and a
// second load and store: 64 x 32000 with 2048 tokens, 16 token biases and a bit mask
// 9 us, one row 5. The 4096 rows and their gradient took 502 when every vector of
// 8192-column slices read 32-bit counts, 262 with 16 bits, larger slices and the list
// in both, 235 where their pass reads 16-bit counts. The 1024-thread forms need 64
// (bf16) to 69 registers a thread; past 64 one workgroup is on a compute unit at a
// time, in fp16 and in the gradients. In place 4096 x 32000 with 1024 tokens take 95, 380 to 480
// with a bias or a mask, an element at a time (apart 131 to 158); 64 x 32000 8 and 13
// to 14 (apart 9 to 10).

#include <type_traits>

#include "cyfa_internal.h"
#include "cyfa_rows.h"

namespace cyfa {

namespace {

constexpr int AJ_NV = 4;            // vectors of a thread in flight

// What a slice's columns have met, in BITS a column: seen at all, named by the
// tokens' biases, the number behind the prompt.
template <int BITS>
struct Counts {
    static constexpr uint32_t SEEN = 1u << (BITS - 1), BIASED = SEEN >> 1, MADE = BIASED - 1;
    uint32_t* words;
    static __device__ __forceinline__ int shift(int c) { return BITS == 16 ? (c & 1) * 16 : 0; }
    __device__ __forceinline__ uint32_t* word(int c) const { return words + (BITS == 16 ? c >> 1 : c); }
    static __device__ __forceinline__ uint32_t of(uint32_t word, int c) { return BITS == 16 ? word >> shift(c) & 0xffff : word; }
    // each gives what was there before
    __device__ __forceinline__ uint32_t mark(int c, uint32_t bit) const { return of(atomicOr(word(c), bit << shift(c)), c); }
    __device__ __forceinline__ uint32_t count(int c) const { return of(atomicAdd(word(c), 1u << shift(c)), c); }
    __device__ __forceinline__ uint32_t operator[](int c) const { return of(*word(c), c); }
};

template <class E, int NT, int BITS, bool GRAD>
__global__ __launch_bounds__(NT) void adjust_kernel(AdjustParams p) {
#pragma clang fp contract(off)
    typedef typename RowVec<E>::type Vec;
    typedef Counts<BITS> C;
    constexpr int N = RowVec<E>::N, U = 4;
    extern __shared__ __align__(16) uint32_t lds[];
    __shared__ int listed_s;
    const C counts = {lds};                                                              // [cols]
    int* const ids_s = reinterpret_cast<int*>(lds + p.cols / (32 / BITS));               // [n_tokens]
    float* const values_s = reinterpret_cast<float*>(ids_s) + (GRAD ? 0 : p.n_tokens);   // [n_tokens]
    uint16_t* const list = reinterpret_cast<uint16_t*>(values_s + (GRAD ? 0 : p.n_tokens));  // [min(cols, L)]
    const int tid = threadIdx.x;
    const bool tokens = !GRAD && p.n_tokens > 0, touches = p.L > 0 || tokens;
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
    // ---- a row's history, NT * U tokens at a time
    const long long n = p.L == 0 ? 0 : p.lengths ? max(0ll, min(p.L, p.lengths[r])) : p.L, prompt = p.prompts ? p.prompts[r] : 0;
    const long long h0 = ro * p.h_outer + ri * p.h_row;
    long long t[U];
    const auto load_tokens = [&](long long i0) {
        if (i0 < n)
#pragma unroll
            for (int u = 0; u < U; u++) {
                const long long i = h0 + min(i0 + u * NT + tid, n - 1);
                t[u] = p.wide ? static_cast<const long long*>(p.history)[i] : static_cast<const int*>(p.history)[i];
            }
    };
    // The result of a column that has met w, with its tokens' bias.
    const float repetition = p.repetitions ? p.repetitions[r] : p.repetition;
    const float presence = p.presences ? p.presences[r] : p.presence;
    const float frequency = p.frequencies ? p.frequencies[r] : p.frequency;
    const auto penalised = [&](uint32_t w, float e) {
        const uint32_t made = w & C::MADE;
        if (w & (C::SEEN | C::MADE)) e = e > 0.f ? e / repetition : e * repetition;
        if (made) e = e - ((float)made * frequency + presence);
        return e;
    };
    const auto sloped = [&](float e, float xc) {
        if (e != 0.f) e *= xc > 0.f ? 1.f / repetition : repetition;
        return e;
    };
    const auto result = [&](int c, uint32_t w, float xc, float value) {
        if (GRAD) {
            const float e = sloped((float)from[c], xc);
            return kept(c) ? e : 0.f;
        }
        float e = penalised(w, xc);
        if (bias) e = e + bias[c];
        if (w & C::BIASED) e = e + value;
        return kept(c) ? e : -INFINITY;
    };
    const bool apart = GRAD || y != x, dense = apart && p.dense;  // (the pass reads the counts)
    // ---- the slice as where nothing is repeated, or (COUNTED) with what its columns have met
    const float out = GRAD ? 0.f : -INFINITY;
    const auto pass = [&](auto with_counts) {
        constexpr bool COUNTED = decltype(with_counts)::value;
        const int nvec = cols / N, tail = cols - nvec * N;
        for (int i0 = 0; i0 < nvec; i0 += NT * AJ_NV) {
            Vec v[AJ_NV];
            uint32_t keep[AJ_NV][N / 4];  // bytes or bits of the mask
#pragma unroll
            for (int j = 0; j < AJ_NV; j++) v[j] = load_row(from + (size_t)min(i0 + j * NT + tid, nvec - 1) * N);
            if (allowed)
#pragma unroll
                for (int j = 0; j < AJ_NV; j++) {
                    const int c = min(i0 + j * NT + tid, nvec - 1) * N;
                    if (p.packed)
                        keep[j][0] = allowed[c >> 3] >> (c & 7);
                    else
                        __builtin_memcpy(keep[j], allowed + c, N);
                }
            constexpr int M = N * BITS / 32;
            uint32_t met[COUNTED ? AJ_NV : 1][M], any[COUNTED ? AJ_NV : 1];
            Vec own[COUNTED && GRAD ? AJ_NV : 1];  // the logits of vectors with a column that was met
            if (COUNTED)
#pragma unroll
                for (int j = 0; j < AJ_NV; j++) {
                    const int i = min(i0 + j * NT + tid, nvec - 1);
                    __builtin_memcpy(met[j], lds + (size_t)i * M, sizeof met[j]);
                    any[j] = 0;
#pragma unroll
                    for (int c = 0; c < M; c++) any[j] |= met[j][c];
                    if (GRAD && any[j]) own[j] = load_row(x + (size_t)i * N);
                }
#pragma unroll
            for (int j = 0; j < AJ_NV; j++) {
                const int i = i0 + j * NT + tid;
                if (i >= nvec) continue;
                if (COUNTED && GRAD) {
                    if (any[j])
#pragma unroll
                        for (int c = 0; c < N; c++)
                            if (C::of(met[j][c * BITS / 32], c)) v[j][c] = (E)sloped((float)v[j][c], (float)own[j][c]);
                } else if (COUNTED) {
                    if (any[j] || bias) {
                        float e[N];
#pragma unroll
                        for (int c = 0; c < N; c++) e[c] = (float)v[j][c];
                        if (any[j])
#pragma unroll
                            for (int c = 0; c < N; c++) e[c] = penalised(C::of(met[j][c * BITS / 32], c), e[c]);
                        if (bias) {
                            float b[N];
                            __builtin_memcpy(b, bias + (size_t)i * N, sizeof b);
#pragma unroll
                            for (int c = 0; c < N; c++) e[c] = e[c] + b[c];
                        }
#pragma unroll
                        for (int c = 0; c < N; c++) v[j][c] = (E)e[c];
                    }
                } else if (bias) {
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
            if (COUNTED && !GRAD) e = penalised(counts[c], e);
            if (COUNTED && GRAD && counts[c]) e = sloped(e, (float)x[c]);
            if (bias) e = e + bias[c];
            y[c] = (E)(kept(c) ? e : out);
        }
    };
    if (!touches) {
        pass(std::false_type{});
        return;
    }
    // The first store of an output that is apart is on its way while the row's tokens are counted.
    load_tokens(0);
    for (int i = tid * 4; i < p.cols / (32 / BITS); i += NT * 4) *reinterpret_cast<uint4*>(lds + i) = uint4{0, 0, 0, 0};
    if (tid == 0) listed_s = 0;
    if (tokens) {
        const long long* ids = p.token_ids + ro * p.ti_outer + ri * p.ti_row;
        const float* v = p.token_values + ro * p.tv_outer + ri * p.tv_row;
        for (int i = tid; i < p.n_tokens; i += NT) {
            const long long c = ids[i] - c0;
            ids_s[i] = c >= 0 && c < cols ? (int)c : -1;
            values_s[i] = v[i];
        }
    }
    if (apart && !dense) pass(std::false_type{});
    __syncthreads();
    for (long long i0 = 0; i0 < n; i0 += NT * U) {
        if (i0 > 0) load_tokens(i0);
#pragma unroll
        for (int u = 0; u < U; u++) {
            const long long i = i0 + u * NT + tid, c = t[u] - c0;
            if (i < n && c >= 0 && c < cols) {
                const uint32_t before = i < prompt ? counts.mark((int)c, C::SEEN) : counts.count((int)c);
                if (before == 0 && !dense) list[atomicAdd(&listed_s, 1)] = (uint16_t)c;
            }
        }
    }
    __syncthreads();
    // The tokens' biases: the first entry of a token adds all of its entries, in
    // their order, to the column that it takes over from the list.
    float value[ADJUST_MAX_TOKENS / NT > 0 ? ADJUST_MAX_TOKENS / NT : 1];
    uint32_t firsts = 0;
    if (tokens) {
#pragma unroll
        for (int k = 0; k < ADJUST_MAX_TOKENS / NT; k++) {
            const int i = tid + k * NT, c = i < p.n_tokens ? ids_s[i] : -1;
            if (c < 0) continue;
            bool first = true;
            float sum = 0.f;
            for (int j = 0; j < p.n_tokens; j++)
                if (ids_s[j] == c) {
                    if (j < i) first = false;
                    sum += values_s[j];
                }
            value[k] = sum;
            if (first) {
                counts.mark(c, C::BIASED);
                firsts |= 1u << k;
            }
        }
        __syncthreads();
    }
    // ---- the touched columns
    if (apart) {
        if (dense) {
            pass(std::true_type{});
            __syncthreads();
        }
        for (int i = tid; i < listed_s; i += NT) {
            const int c = list[i];
            const uint32_t w = counts[c];
            if (!(w & C::BIASED)) y[c] = (E)result(c, w, (float)x[c], 0.f);
        }
        if (tokens)
#pragma unroll
            for (int k = 0; k < ADJUST_MAX_TOKENS / NT; k++)
                if (firsts >> k & 1) {
                    const int c = ids_s[tid + k * NT];
                    y[c] = (E)result(c, counts[c], (float)x[c], value[k]);
                }
        return;
    }
    // In place: those of the tokens' biases first, whose marks keep the others off them.
    float kept_back[ADJUST_MAX_TOKENS / NT > 0 ? ADJUST_MAX_TOKENS / NT : 1];
    if (tokens)
#pragma unroll
        for (int k = 0; k < ADJUST_MAX_TOKENS / NT; k++)
            if (firsts >> k & 1) {
                const int c = ids_s[tid + k * NT];
                kept_back[k] = result(c, counts[c], (float)x[c], value[k]);
            }
    if (bias || allowed) {
        __syncthreads();
        for (int c = tid; c < cols; c += NT) y[c] = (E)result(c, counts[c] & ~C::BIASED, (float)x[c], 0.f);
        __syncthreads();
    } else {
        for (int i = tid; i < listed_s; i += NT) {
            const int c = list[i];
            const uint32_t w = counts[c];
            if (!(w & C::BIASED)) y[c] = (E)result(c, w, (float)x[c], 0.f);
        }
    }
    if (tokens)
#pragma unroll
        for (int k = 0; k < ADJUST_MAX_TOKENS / NT; k++)
            if (firsts >> k & 1) y[ids_s[tid + k * NT]] = (E)kept_back[k];
}

template <class E, int NT, int BITS, bool GRAD>
void launch_slices(AdjustParams p, long long cols, hipStream_t stream) {
    p.cols = (int)cols;
    const long long slices = (p.V + p.cols - 1) / p.cols, jobs = (p.rows >= 8 ? (p.rows + 7) / 8 * 8 : p.rows) * slices;
    const int tokens = GRAD ? 0 : p.n_tokens;
    const size_t lds = p.L > 0 || tokens > 0 ? (size_t)cols * BITS / 8 + (size_t)tokens * 8 + (size_t)min(cols, p.L) * 2 : 0;
    for (p.first = 0; p.first < jobs; p.first += LOGPROBS_MAX_GRID) {
        const dim3 grid((unsigned)min(jobs - p.first, (long long)LOGPROBS_MAX_GRID));
        hipLaunchKernelGGL((adjust_kernel<E, NT, BITS, GRAD>), grid, dim3(NT), lds, stream, p);
    }
}

// Whether the pass over the logits reads the counts, after them, for a list of the
// touched columns and a second store of each, beside which the pass is on its way
// while the counting goes on. us on MI355X, list / counts, bf16:
//   4096 x 32000, 64 tokens 105 / 101, 500 131 / 110, 1000 141 / 114, 4000 262 / 141; 1024 rows, 200 27 / 29, 500 30.5 / 30, 2000 44 / 35
//   512 x 32000, 500 17 / 19, 1000 20 / 20, 2000 25 / 21; 64 rows, 1000 7.0 / 7.6, 2000 7.6 / 7.9, 4000 9.7 / 8.8, 16000 19 / 13
//   256 x 50001 fp16, 1000 18 / 19, 2000 22 / 21, 4000 28 / 23, 8000 33 / 26, with a bias 39 / 28
//   16384 x 4096, 200 69 / 71, 500 85 / 75; 1024 rows, 500 9.1 / 9.9, 1000 10.4 / 10.1, 4000 20 / 14; 4096 x 1000 fp32, 200 15.7 / 15.5, 1000 20 / 17
// The gradient, which reads the logits of the vectors with counts: 4096 x 32000, 200
// tokens 129 / 120, 1000 182 / 142, 4000 403 / 170; 1024 rows, 500 35 / 31; 256 x 50001, 500 17.9 / 18.5, 2000 25 / 21; 64 x 32000, 1000
// 7.0 / 7.1, 4000 9.7 / 8.2; 16384 x 4096, 200 82 / 77, 2000 308 / 127; 1024 x 4096, 500 9.0 / 9.0, 4000 23 / 14.
bool reads_counts(const AdjustParams& p) {
    return (p.L >= 500 && p.rows * p.V >= 1ll << 24) || (p.L * 4 >= min(p.V, 4096) && p.L * 14 >= p.V);
}

template <class E, bool GRAD>
void launch(AdjustParams p, hipStream_t stream) {
    p.dense = reads_counts(p);
    // Columns of a slice and threads that take it, by us on MI355X. Each slice reads
    // the history; few large ones leave compute units idle:
    //   4096 x 32000 bf16, 1000 tokens: 512 threads, 8192 columns 153, 16384 114; 1024, 32000 158
    //   256 x 50001 fp16: 512, 16384: 2000 tokens 20, 8000 26, 16000 36; 1024, 25024 22, 26, 30
    //   64 x 32000 with a mask, 1500 tokens: 512, 8192 8.7, 16384 9.2; 1024, 25024 10.2
    //   1024 x 4096, 380 tokens: 256, 4096 7.3; 512 9.4
    const long long whole = (p.V + 31ll) / 32 * 32, slices = (whole + 32767) / 32768;
    const bool many = p.rows * p.V >= 16384ll * 512;
    if (p.L > Counts<16>::MADE)
        launch_slices<E, 512, 32, GRAD>(p, min(whole, 8192ll), stream);
    else if (p.V <= 4096)
        launch_slices<E, 256, 16, GRAD>(p, whole, stream);
    else if (many && p.L >= 4096)
        launch_slices<E, 1024, 16, GRAD>(p, (whole / slices + 31) / 32 * 32, stream);
    else
        launch_slices<E, 512, 16, GRAD>(p, min(whole, many ? 16384ll : 8192ll), stream);
}

}  // namespace

void launch_adjust(const AdjustParams& p, int dtype, bool grad, hipStream_t stream) {
    if (dtype == 0)
        grad ? launch<bf16_t, true>(p, stream) : launch<bf16_t, false>(p, stream);
    else if (dtype == 1)
        grad ? launch<float, true>(p, stream) : launch<float, false>(p, stream);
    else
        grad ? launch<f16_t, true>(p, stream) : launch<f16_t, false>(p, stream);
}

}  // namespace cyfa
