// cyfa_logprobs.hip -- log probabilities of given tokens with the entropy and
// the most probable alternatives of each row of logits, their mean as a
// training loss, and the gradients. For a row x [V], t its token:
//   m = max x, S = sum e^(x - m), S1 = sum (x - m) e^(x - m)
//   logprob = x_t - m - log S,  entropy = log S - S1 / S
//   dx_i = p_i (A - dH (log p_i + entropy)) + sum of the cotangents of the
//          outputs that read x_i itself,  p_i = e^(x_i - m) / S,
//          A = -(sum of the cotangents of logprob and of the alternatives)
// One pass over the row each way: the forward keeps m, log S and the entropy of
// each row for the gradient, in fp32 as every sum here. (lse = m + log S alone
// would round away the low bits of log S beside a large m, and p with them.)
//
// Bound by the memory's rate where rows are many: an element costs ten VALU
// instructions and one exponential at a quarter of their rate, two thirds of the
// time of its bytes. On MI355X 16384 x 32000 bf16 rows (1.05 GB) take 156 us
// forward (6.7 TB/s; a copy of 1 GiB moves 5.1), their loss with three labels of
// ten ignored 128 us (those rows are not read), its gradient 312 us (5.7 TB/s of
// 0.73 GB read and 1.05 written). The plain chain of fp32 operations took 7.35 ms
// and, with the gradient, 5.2 ms. Few rows are bound by the latency of a row's
// own steps: one row of 32000 with five alternatives 8 us, 64 rows with twenty 10.
// Alternatives of many rows take a second pass over the row's tiles and a ranking
// by one wave: 8192 x 32000 bf16 rows 96 us with none, 144 with one to five, 150
// with twenty, 155 with 32 (3.5 TB/s of one read); 32768 x 2048 26 and, with twenty,
// 58. Their gradient: 2048 x 32000 rows 42 us (6.3 TB/s both ways) through logprob,
// 43 through the entropy too, 50 through twenty alternatives as well.
#include "cyfa_internal.h"
#include "cyfa_rows.h"

namespace cyfa {

namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kLowest = -3.402823466e38f;
constexpr float kNothing = -200.f;  // the exponent (of 2) of what counts nothing: 0 times minus infinity would be a NaN
constexpr int LP_CAP = 1024;        // candidates for the alternatives held in LDS
constexpr int LP_PARTS = 16;        // most parts of a row
constexpr int LP_NV = 4;            // vectors of a thread in a tile of a row: 64 bytes in flight

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
    a.s1 = f * (a.s1 + fmaxf(d, kNothing) * a.s);
    a.s *= f;
    a.m = m;
}

template <class E>
__device__ __forceinline__ const E* row_of(const LogprobParams& p, long long r) {
    return static_cast<const E*>(p.x) + (r / p.inner) * p.outer_stride + (r % p.inner) * p.row_stride;
}

// The k-th largest of the 64 lanes' values x (no NaN), but for an order of the
// last 6 bits: ranked as integers in the values' order with the lane in place
// of those bits, so that all differ; the smallest of the first k. In every lane.
__device__ __forceinline__ float kth_largest(float x, int k) {
    const uint32_t mine = (value_key(x) & ~63u) | (uint32_t)(threadIdx.x & 63);
    int rank = 0;
#pragma unroll 8
    for (int i = 0; i < 64; i++) rank += (uint32_t)__builtin_amdgcn_readlane((int)mine, i) > mine;
    return -wave_max(rank < k ? -x : -INFINITY);
}

// a += b of another set of elements.
__device__ __forceinline__ void join(RowSums& a, RowSums b) {
    const float m = fmaxf(a.m, b.m);
    rescale(a, m);
    rescale(b, m);
    a.s += b.s;
    a.s1 += b.s1;
}

// Row r's results but its alternatives.
__device__ __forceinline__ void put_row(const LogprobParams& p, long long r, const RowSums& a, float ls, float xt, bool ignored) {
    p.logprob[r] = ignored ? 0.f : (xt - a.m) - ls;
    if (p.entropy) p.entropy[r] = ls - kLn2 * (a.s1 / a.s);
    if (p.stats) {
        p.stats[2 * r] = a.m;
        p.stats[2 * r + 1] = ls * kLog2e;
    }
}

__device__ __forceinline__ void put_top(const LogprobParams& p, long long r, int rank, uint64_t key, const RowSums& a, float ls) {
    p.top_ids[r * p.k + rank] = 0xffffffffu - (uint32_t)key;
    p.top_logprobs[r * p.k + rank] = (key_value(key) - a.m) - ls;
}

// Rows of a workgroup whose rows take NT threads each: a wave's rows share one.
constexpr int rows_of(int NT) { return NT == 64 ? 4 : 1; }

// What the threads of a row wrote to LDS or memory, its other threads see.
template <int NT>
__device__ __forceinline__ void row_sync() {
    if (NT == 64) {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    } else {
        __syncthreads();
    }
}

// NT threads to a row (rows beyond the grid in turn), tiles of NT * LP_NV
// vectors of it in registers: a row of one tile is read from memory
// once, also for its alternatives. With PARTS, to part blockIdx.y of a row, whose
// sums and alternatives go to the workspace for logprobs_join_kernel.
template <class E, int NT, bool TOP, bool PARTS, bool STREAM>
__global__ __launch_bounds__(NT * rows_of(NT)) void logprobs_kernel(LogprobParams p) {
    constexpr int N = RowVec<E>::N, W = NT / 64, RW = rows_of(NT), CAP = LP_CAP / RW;
    __shared__ RowSums red[W];
    __shared__ float best_s[TOP ? W : 1][64];
    __shared__ uint64_t cand_s[RW][TOP ? CAP : 1];
    __shared__ uint64_t next_s[TOP ? W : 1];
    __shared__ float thr_s[RW];
    __shared__ int count_s[RW];
    const int tid = threadIdx.x % NT, lane = tid & 63, wv = tid >> 6, sub = threadIdx.x / NT;
    uint64_t* cand = cand_s[sub];
    const int c0 = PARTS ? blockIdx.y * p.part : 0, cols = PARTS ? min(p.part, p.V - c0) : p.V;
    const int nvec = cols / N, tail = cols - nvec * N;
    for (long long r = (long long)blockIdx.x * RW + sub; r < p.rows; r += (long long)gridDim.x * RW) {
        const E* x = row_of<E>(p, r) + c0;
        const long long t = p.tokens[r];
        const bool ignored = t == p.ignore;
        if (ignored && !TOP && !p.entropy) {  // (the loss: nothing of this row counts)
            if (!PARTS && tid == 0) p.logprob[r] = 0.f;
            continue;
        }
        const float xt = !PARTS && t >= 0 && t < p.V ? (float)x[t] : __builtin_nanf("");
        const float last = tid < tail ? (float)x[nvec * N + tid] : -INFINITY;
        typename RowVec<E>::type v[LP_NV];
        float top[LP_NV];  // the largest element of each
        // Vectors past the end are read as the last one and dropped: no branch
        // among the loads, at which the compiler would wait for those in flight.
        const auto load_tile = [&](int v0) {
#pragma unroll
            for (int j = 0; j < LP_NV; j++) v[j] = load_row<E, STREAM>(x + (size_t)min(v0 + j * NT + tid, nvec - 1) * N);
        };
        const auto largest = [&](int v0) {
#pragma unroll
            for (int j = 0; j < LP_NV; j++) {
                top[j] = -INFINITY;
                if (v0 + j * NT + tid < nvec)
#pragma unroll
                    for (int c = 0; c < N; c++) top[j] = fmaxf(top[j], (float)v[j][c]);
            }
        };
        RowSums a = {kLowest, 0.f, 0.f};
        float best = last;
        const auto add = [&](float e) {
            const float u = (e - a.m) * kLog2e, q = fast_exp2(u);
            a.s += q;
            a.s1 = fmaf(fmaxf(u, kNothing), q, a.s1);
        };
        for (int v0 = 0; v0 < nvec; v0 += NT * LP_NV) {
            load_tile(v0);
            largest(v0);
#pragma unroll
            for (int j = 0; j < LP_NV; j++) best = fmaxf(best, top[j]);
            rescale(a, fmaxf(a.m, best));
#pragma unroll
            for (int j = 0; j < LP_NV; j++)
                if (v0 + j * NT + tid < nvec)
#pragma unroll
                    for (int c = 0; c < N; c++) add((float)v[j][c]);
        }
        rescale(a, fmaxf(a.m, best));
        if (tid < tail) add(last);
        const float m = wave_max(a.m);
        rescale(a, m);
        a.s = wave_sum(a.s);
        a.s1 = wave_sum(a.s1);
        if (W > 1) {
            if (lane == 0) red[wv] = a;
            if (TOP) best_s[wv][lane] = best;
            __syncthreads();
            a = red[0];
#pragma unroll 3
            for (int w = 1; w < W; w++) join(a, red[w]);
        }
        const float ls = logf(a.s);
        const long long at = r * gridDim.y + blockIdx.y;
        if (tid == 0) {
            if (PARTS)
                reinterpret_cast<RowSums*>(p.parts)[at] = a;
            else
                put_row(p, r, a, ls, xt, ignored);
        }
        if (TOP) {
            const auto put = [&](int rank, uint64_t key) {
                if (PARTS)
                    p.part_keys[at * p.k + rank] = key;
                else
                    put_top(p, r, rank, key, a, ls);
            };
            // f(element, column) of this thread's elements that reach ``from`` (and NaN, with from -inf)
            const bool one_tile = nvec <= NT * LP_NV;
            const auto each = [&](float from, auto&& f) {
                for (int v0 = 0; v0 < nvec; v0 += NT * LP_NV) {
                    if (!one_tile) {
                        load_tile(v0);
                        largest(v0);
                    }
#pragma unroll
                    for (int j = 0; j < LP_NV; j++) {
                        const int i = v0 + j * NT + tid;
                        if (i < nvec && top[j] >= from) {
#pragma unroll
                            for (int c = 0; c < N; c++) f((float)v[j][c], c0 + i * N + c);
                        }
                    }
                }
                if (tid < tail) f(last, c0 + nvec * N + tid);
            };
            // A threshold that k elements reach and seldom many more (about
            // 64 ln(64 / (64 - k)) where they lie at random: 24 for 20, 44 for
            // 32): the k-th largest of the largest elements of 64 sets of
            // threads. The candidates' ranks among themselves are those in the row.
            int n = -1;
            if (a.s == a.s) {  // no NaN, no +inf
                if (wv == 0) {
                    for (int w = 1; w < W; w++) best = fmaxf(best, best_s[w][lane]);
                    const float thr = kth_largest(best, p.k);
                    if (lane == 0) {
                        thr_s[sub] = thr;
                        count_s[sub] = 0;
                    }
                }
                row_sync<NT>();
                const float thr = thr_s[sub];
                const auto hold = [&](float e, int i) {
                    const int at = atomicAdd(&count_s[sub], 1);
                    if (at < CAP) cand[at] = order_key(e, i);
                };
                each(thr, [&](float e, int i) {
                    if (e >= thr) hold(e, i);
                });
                row_sync<NT>();
                n = count_s[sub];
                if (n > CAP) {  // many equal elements: all above them, and those of the lowest columns
                    row_sync<NT>();
                    if (tid == 0) count_s[sub] = 0;
                    row_sync<NT>();
                    each(thr, [&](float e, int i) {
                        if (e > thr || (e == thr && i < c0 + CAP / 2)) hold(e, i);
                    });
                    row_sync<NT>();
                    n = count_s[sub];
                    if (n < p.k || n > CAP) n = -1;
                }
            }
            if (n >= 0) {
                for (int c = tid; c < n; c += NT) {
                    const uint64_t key = cand[c];
                    int rank = 0;
#pragma unroll 8
                    for (int i = 0; i < n; i++) rank += cand[i] > key;
                    if (rank < p.k) put(rank, key);
                }
            } else {  // k rounds, each the largest key below the one before
                uint64_t below = ~0ull;
                for (int rank = 0; rank < p.k; rank++) {
                    uint64_t next = 0;
                    each(-INFINITY, [&](float e, int i) {
                        const uint64_t key = order_key(e, i);
                        if (key < below && key > next) next = key;
                    });
                    for (int d = 32; d > 0; d >>= 1) {
                        const uint64_t o = __shfl_xor(next, d);
                        next = o > next ? o : next;
                    }
                    if (W > 1) {
                        __syncthreads();
                        if (lane == 0) next_s[wv] = next;
                        __syncthreads();
                        for (int w = 0; w < W; w++) next = next_s[w] > next ? next_s[w] : next;
                    }
                    if (tid == 0) put(rank, next);
                    below = next;
                }
            }
        }
        if (W > 1 || TOP) row_sync<NT>();  // the shared arrays are free for the next row
    }
}

// A row's results from those of its ``parts`` parts, a workgroup to a row.
template <class E>
__global__ __launch_bounds__(256) void logprobs_join_kernel(LogprobParams p, int parts) {
    __shared__ uint64_t keys[LP_PARTS * LOGPROBS_MAX_TOP];
    for (long long r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const long long t = p.tokens[r];
        const bool ignored = t == p.ignore;
        if (ignored && p.k == 0 && !p.entropy) {
            if (threadIdx.x == 0) p.logprob[r] = 0.f;
            continue;
        }
        const RowSums* part = reinterpret_cast<const RowSums*>(p.parts) + r * parts;
        RowSums a = part[0];
        for (int i = 1; i < parts; i++) join(a, part[i]);
        const float ls = logf(a.s);
        if (threadIdx.x == 0) put_row(p, r, a, ls, t >= 0 && t < p.V ? (float)row_of<E>(p, r)[t] : __builtin_nanf(""), ignored);
        if (p.k == 0) continue;
        const int n = parts * p.k;
        for (int i = threadIdx.x; i < n; i += 256) keys[i] = p.part_keys[r * n + i];
        __syncthreads();
        for (int c = threadIdx.x; c < n; c += 256) {
            const uint64_t key = keys[c];
            int rank = 0;
#pragma unroll 8
            for (int i = 0; i < n; i++) rank += keys[i] > key;
            if (rank < p.k) put_top(p, r, rank, key, a, ls);
        }
        __syncthreads();
    }
}

// loss = -(sum of logprob over the rows whose token counts) / their number, one
// workgroup, in double and in a fixed order; no rows: 0 / 0.
__global__ __launch_bounds__(1024) void loss_mean_kernel(LogprobParams p) {
    __shared__ double sums[16];
    __shared__ double counts[16];
    constexpr int U = 8;  // rows of a thread whose loads are in flight together
    double s = 0., n = 0.;
    for (long long r0 = threadIdx.x; r0 < p.rows; r0 += 1024 * U) {
        long long t[U];
        float lp[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const long long r = min(r0 + 1024 * u, p.rows - 1);
            t[u] = p.tokens[r];
            lp[u] = p.logprob[r];
        }
#pragma unroll
        for (int u = 0; u < U; u++)
            if (r0 + 1024 * u < p.rows && t[u] != p.ignore) {
                s += (double)lp[u];
                n += 1.;
            }
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

constexpr int LG_NV = 4;  // vectors of a thread in flight

// The gradient of the columns [c0, c1) of a row by NT threads: blockIdx.y's
// share of the row, whole vectors. Rows up to 2048 bf16 columns take a wave each
// (2^28 logits in rows of 2048: 185 us on MI355X, 285 with a workgroup to a row;
// in rows of 256, 510 and 1790). The elements that outputs read themselves are
// stored a second time, by one thread each, rather than looked for at every element.
//
// The rows are taken from the last to the first: those that the forward read last
// are in the caches still. A gradient of 128 MiB or more in whole lines goes past
// them (STREAM). us on MI355X for the loss of 8 x 2048 x 32000 bf16 logits, both
// ways: 503 with neither, 486 in that order, 460 past the caches, 438 with both;
// 4 x 1024 rows 140, 137, 142 and 113; 8 x 2048 x 50001, whose rows begin within
// lines, 971, 938, 963 and 937.
template <class E, int NT, bool ENTROPY, bool STREAM>
__global__ __launch_bounds__(256) void logprobs_grad_kernel(LogprobParams p, int share) {
    constexpr int N = RowVec<E>::N, RW = 256 / NT;
    const int tid = threadIdx.x % NT;
    const int c0 = blockIdx.y * share, c1 = min(c0 + share, p.V);
    const int nvec = (c1 - c0) / N, tail = c1 - c0 - nvec * N;
    for (long long i = (long long)blockIdx.x * RW + threadIdx.x / NT; i < p.rows; i += (long long)gridDim.x * RW) {
        const long long r = p.rows - 1 - i;
        const E* x = row_of<E>(p, r) + c0;
        E* dx = static_cast<E*>(p.dx) + r * p.V + c0;
        const long long t = p.tokens[r];
        const float m = p.stats[2 * r], ls = p.stats[2 * r + 1];
        float dlp = 0.f;
        if (t != p.ignore) dlp = p.d_loss ? -*p.d_loss / *p.count : p.d_logprob ? p.d_logprob[r] : 0.f;
        if (dlp != 0.f && (t < 0 || t >= p.V)) dlp = __builtin_nanf("");
        const float dh = ENTROPY ? p.d_entropy[r] : 0.f;
        float total = dlp;
        bool any = dlp != 0.f || dh != 0.f;
        const int k = p.d_top ? p.k : 0;
        for (int j = 0; j < k; j++) {
            const float d = p.d_top[r * p.k + j];
            total += d;
            any |= d != 0.f;
        }
        typename RowVec<E>::type o;
        if (!any) {
#pragma unroll
            for (int c = 0; c < N; c++) o[c] = (E)0.f;
            for (int i = tid; i < nvec; i += NT) store_row<E, STREAM>(dx + (size_t)i * N, o);
            if (tid < tail) dx[nvec * N + tid] = (E)0.f;
            continue;
        }
        // dx = p (a + b log2 p) for the elements that no output reads by itself
        const float a = -total - (ENTROPY && dh != 0.f ? dh * p.entropy[r] : 0.f), b = -dh * kLn2;
        const auto grad = [&](float e) {
            const float l = (e - m) * kLog2e - ls;
            const float q = fast_exp2(l);
            return ENTROPY ? q * fmaf(fmaxf(l, kNothing), b, a) : q * a;
        };
        for (int i0 = 0; i0 < nvec; i0 += NT * LG_NV) {
            typename RowVec<E>::type v[LG_NV];
#pragma unroll
            for (int j = 0; j < LG_NV; j++) v[j] = load_row(x + (size_t)min(i0 + j * NT + tid, nvec - 1) * N);
#pragma unroll
            for (int j = 0; j < LG_NV; j++) {
                const int i = i0 + j * NT + tid;
                if (i < nvec) {
#pragma unroll
                    for (int c = 0; c < N; c++) o[c] = (E)grad((float)v[j][c]);
                    store_row<E, STREAM>(dx + (size_t)i * N, o);
                }
            }
        }
        if (tid < tail) dx[nvec * N + tid] = (E)grad((float)x[nvec * N + tid]);
        row_sync<NT>();  // the elements that outputs read themselves are written again
        if (tid <= k) {
            const auto index = [&](int j) { return j == 0 ? t : p.top_ids[r * p.k + j - 1]; };
            const auto cot = [&](int j) { return j == 0 ? dlp : p.d_top[r * p.k + j - 1]; };
            const long long i = index(tid);
            float sum = 0.f;
            bool first = i >= c0 && i < c1;
            if (first)
                for (int j = 0; j <= k; j++)
                    if (index(j) == i) {
                        if (j < tid) first = false;
                        sum += cot(j);
                    }
            if (first) dx[i - c0] = (E)(grad((float)x[i - c0]) + sum);
        }
    }
}

// Whether rows at ``rows`` go past the caches: 128 MiB or more, half of the last
// of them, in rows of whole 128-byte lines. Logits read for no gradient (16384 x
// 32000 bf16) take 155 us so on MI355X, 177 through the caches; with a gradient
// to follow, which finds the last of them there, they stay.
template <class E>
bool past_caches(const LogprobParams& p, const void* rows) {
    const bool lines = p.V * sizeof(E) % 128 == 0 && (uintptr_t)rows % 128 == 0 &&
                       (rows == p.dx || (p.row_stride * sizeof(E) % 128 == 0 && p.outer_stride * sizeof(E) % 128 == 0));
    return lines && (size_t)p.rows * p.V * sizeof(E) >= (size_t)128 << 20;
}

// Parts of a row, a workgroup each: those of its tiles, where the rows leave
// compute units idle and have four tiles or more. us on MI355X for rows of
// 131072 bf16 logits, with no and with 20 alternatives, in four parts with their
// join, and as one: 1 row 9.9 / 12.3, 11.9 / 17.7; 64 rows 11.3 / 14.2, 13.5 /
// 18.5; 128 rows 15.3 / 22.8, 13.5 / 19.2. Two tiles gain less than their join's launch costs.
int row_parts(long long rows, int V, int size) {
    const long long tile = 1024 * LP_NV * (16 / size), tiles = (V + tile - 1) / tile;
    return tiles < 4 || rows > 64 ? 1 : (int)min(min(tiles, 256 / rows), (long long)LP_PARTS);
}

template <class E, int NT, bool TOP, bool STREAM = false>
void launch_rows(const LogprobParams& p, hipStream_t stream) {
    const dim3 grid((unsigned)min((p.rows + rows_of(NT) - 1) / rows_of(NT), (long long)LOGPROBS_MAX_GRID));
    hipLaunchKernelGGL((logprobs_kernel<E, NT, TOP, false, STREAM>), grid, dim3(NT * rows_of(NT)), 0, stream, p);
}

template <class E, int NT>
void launch_grad(const LogprobParams& p, int shares, hipStream_t stream) {
    constexpr int N = RowVec<E>::N, RW = 256 / NT;
    const int share = ((p.V + shares - 1) / shares + N - 1) / N * N;
    const dim3 grid((unsigned)min((p.rows + RW - 1) / RW, (long long)LOGPROBS_MAX_GRID), (unsigned)((p.V + share - 1) / share));
    const auto run = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, stream, p, share); };
    if (past_caches<E>(p, p.dx))
        p.d_entropy ? run(logprobs_grad_kernel<E, NT, true, true>) : run(logprobs_grad_kernel<E, NT, false, true>);
    else
        p.d_entropy ? run(logprobs_grad_kernel<E, NT, true, false>) : run(logprobs_grad_kernel<E, NT, false, false>);
}

template <class E>
void launch_parts(LogprobParams p, int parts, hipStream_t stream) {
    constexpr int N = RowVec<E>::N;
    p.part = ((p.V + parts - 1) / parts + N - 1) / N * N;
    parts = (p.V + p.part - 1) / p.part;
    p.part_keys = (unsigned long long*)(p.parts + ((p.rows * parts * 3 + 1) / 2 * 2));
    const dim3 grid((unsigned)p.rows, parts);
    if (p.k > 0)
        hipLaunchKernelGGL((logprobs_kernel<E, 1024, true, true, false>), grid, dim3(1024), 0, stream, p);
    else
        hipLaunchKernelGGL((logprobs_kernel<E, 1024, false, true, false>), grid, dim3(1024), 0, stream, p);
    hipLaunchKernelGGL(logprobs_join_kernel<E>, dim3((unsigned)p.rows), dim3(256), 0, stream, p, parts);
}

template <class E>
void launch(const LogprobParams& p, bool grad, hipStream_t stream) {
    constexpr int N = RowVec<E>::N;
    if (grad) {
        if (p.V <= 64 * LG_NV * N)
            launch_grad<E, 64>(p, 1, stream);
        else  // few rows shared out to about four workgroups of a compute unit
            launch_grad<E, 256>(p, (int)min((1024 + p.rows - 1) / p.rows, (long long)(p.V + 256 * N - 1) / (256 * N)), stream);
        return;
    }
    // Threads of a row, by us on MI355X (bf16; no / 20 alternatives):
    //   2048 columns   32768 rows: 64 threads 27 / 61, 256 57 / 171;  1024 rows: 3.7 / 8.3, 4.4 / 8.2
    //   4096           16384 rows: 25 / 50, 34 / 94;                   1024 rows: 4.3 / 10.7, 4.8 / 9.0
    //   8192           1024 rows: 6.4 / 15.1, 5.6 / 10.3
    //   32000          1 row: 256 threads 5.0 / 10.4, 1024 5.7 / 7.9;  256 rows: 6.3 / 12.6, 7.2 / 10.1;
    //                  512 rows: 8.8 / 15.9, 11.2 / 18.6;              8192 rows: 94 / 154, 137 / 279
    // A row's own steps (its reductions, the search for alternatives) take the
    // time where rows are short or few: few threads a row share a workgroup, or
    // many, one row to a compute unit, search its columns.
    const int parts = row_parts(p.rows, p.V, sizeof(E));
    if (parts > 1)
        launch_parts<E>(p, parts, stream);
    else if (p.V <= 128 * LP_NV * N)
        p.k > 0 ? launch_rows<E, 64, true>(p, stream) : launch_rows<E, 64, false>(p, stream);
    else if (p.k > 0 && p.rows <= 256 && p.V > 256 * LP_NV * N)
        launch_rows<E, 1024, true>(p, stream);
    else if (p.k > 0)
        launch_rows<E, 256, true>(p, stream);
    else if (!p.stats && past_caches<E>(p, p.x))
        launch_rows<E, 256, false, true>(p, stream);
    else
        launch_rows<E, 256, false>(p, stream);
}

}  // namespace

// Bytes of the parts' sums and keys, 0 where rows are not shared out.
size_t logprobs_workspace_bytes(long long rows, int V, int k, int size) {
    if (rows <= 0) return 0;
    const int parts = row_parts(rows, V, size);
    return parts > 1 ? (size_t)((rows * parts * 3 + 1) / 2 * 2) * 4 + (size_t)rows * parts * k * 8 : 0;
}

void launch_logprobs(const LogprobParams& p, int dtype, bool grad, hipStream_t stream) {
    if (p.rows > 0) {
        if (dtype == 0)
            launch<bf16_t>(p, grad, stream);
        else if (dtype == 1)
            launch<float>(p, grad, stream);
        else
            launch<f16_t>(p, grad, stream);
    }
    if (!grad && p.loss) hipLaunchKernelGGL(loss_mean_kernel, dim3(1), dim3(1024), 0, stream, p);
}

}  // namespace cyfa
