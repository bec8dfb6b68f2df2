// cyfa_distill.hip -- the divergence of a student's distribution from a teacher's
// that is known at its k most probable tokens, and the gradient. For a row x [V]
// of the student's logits, q = softmax(x / T), the teacher's entries (id_i, t_i),
// those with an id outside [0, V) or t_i = -inf left out:
//   p_i = softmax(t / T)_i over the row's entries          loss = sum p_i (log p_i - log q_id)
//   dx_j = (q_j - sum of p_i over id_i = j) / T
// or, with the tail, T = 1, p_i = e^t_i and the rest of either mass as one more
// outcome, p_r = 1 - sum p_i, q_r = sum of q_j over the columns of no entry:
//   loss = sum p_i (log p_i - log q_id) + p_r (log p_r - log q_r)
//   dx_j = q_j P - sum of p_i over id_i = j, P = sum p_i + p_r,  at the entries' columns
//   dx_j = (q_j / q_r) (q_r P - p_r)                             elsewhere
// The loss is over the entries: where an id is there several times it is less than
// with one entry of their whole mass, by a constant; the gradient is the same.
// One pass over the row each way, sums in fp32; what the teacher's few entries
// give is formed in double (1 - sum p_i cancels), by a wave a row in a launch of
// its own: at the end of the row's pass three waves of four would wait for it. The
// columns of no entry keep a maximum and a sum of their own with the tail: taken
// as the difference of the row's sum and the entries', a small rest would be lost.
//
// Bound by memory. On MI355X 16384 x 32000 bf16 rows with 20 entries, of which 78 %
// count (0.82 GB of logits read, 1.05 of gradient written), take 139 us for the sums
// (5.9 TB/s), 11 for the entries, 5 for the mean and 344 for the gradient (5.4 TB/s
// both ways; a copy of 1 GiB moves 5.0 to 5.2); 1021 x 50001 fp16 rows with a tail and
// 64 entries, 65 % of them counting, 22, 7, 3 and 34. A few rows of 256 columns take 4,
// 4, 2 and 5, the latency of each launch's loads.
#include "cyfa_internal.h"
#include "cyfa_rows.h"

namespace cyfa {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr double kLn2 = 0.6931471805599453;
constexpr float kLowest = -3.402823466e38f;
constexpr int DS_NV = 4;  // vectors of a thread in flight

// What the forward keeps of a row for the gradient.
struct DistillRow {
    float m, ls;        // of all columns: the maximum, log2 of the sum of 2^((x - m) c)
    float rm, rls;      // of the columns of no entry (with the tail; else of all)
    float rest, entry;  // what multiplies the softmax of the columns of no entry, of the entries
    float top, norm;    // p_i = 2^((t_i - top) c - norm)
    float weight;       // of the row in the mean, 0 without entries
    float loss;
};
static_assert(sizeof(DistillRow) == DISTILL_ROW_FLOATS * 4, "DISTILL_ROW_FLOATS");

// Whether an entry counts.
__device__ __forceinline__ bool counts(long long id, float t, int V) { return id >= 0 && id < V && t != -INFINITY; }

template <int NT>
__device__ __forceinline__ void row_sync() {
    if (NT == 64) {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    } else {
        __syncthreads();
    }
}

constexpr int rows_of(int NT) { return NT == 64 ? 4 : 1; }

// A maximum and a sum of 2^((x - m) c) of a set of elements.
struct Sum {
    float m, s;
};

__device__ __forceinline__ void rescale(Sum& a, float m, float c) {
    a.s *= fast_exp2((a.m - m) * c);
    a.m = m;
}

__device__ __forceinline__ void join(Sum& a, Sum b, float c) {
    const float m = fmaxf(a.m, b.m);
    rescale(a, m, c);
    rescale(b, m, c);
    a.s += b.s;
}

__device__ __forceinline__ const void* row_at(const DistillParams& p, long long r, int size) {
    return static_cast<const char*>(p.x) + ((r / p.inner) * p.outer_stride + (r % p.inner) * p.row_stride) * size;
}

// A row's weight in the mean, the same in every lane: 0 where nothing of it counts.
__device__ __forceinline__ float row_weight(const DistillParams& p, long long r) {
    bool any = false;
    for (int i = threadIdx.x & 63; i < p.k; i += 64) any |= counts(p.ids[r * p.k + i], p.values[r * p.k + i], p.V);
    return __any(any) ? (p.weights ? p.weights[r] : 1.f) : 0.f;
}

// The maximum and the sum of a row's columns (TAIL: of those of no entry), by NT threads.
template <class E, int NT, bool TAIL>
__global__ __launch_bounds__(NT * rows_of(NT)) void distill_sums_kernel(DistillParams p) {
    constexpr int N = RowVec<E>::N, W = NT / 64, RW = rows_of(NT);
    extern __shared__ uint32_t entries_s[];  // TAIL: a bit for each column of an entry, p.words words a row
    __shared__ Sum red[RW][W];
    const int tid = threadIdx.x % NT, lane = tid & 63, wv = tid >> 6, sub = threadIdx.x / NT;
    uint32_t* bits = entries_s + (size_t)sub * p.words;
    const float c = kLog2e / p.temperature;
    const long long r = p.first + (long long)blockIdx.x * RW + sub;
    if (r >= p.rows) return;  // (rows of a wave each share no barrier)
    const E* x = static_cast<const E*>(row_at(p, r, sizeof(E)));
    if (row_weight(p, r) == 0.f) return;
    if (TAIL) {
        for (int i = tid; i < p.words; i += NT) bits[i] = 0;
        row_sync<NT>();
        for (int i = tid; i < p.k; i += NT) {
            const long long id = p.ids[r * p.k + i];
            if (counts(id, p.values[r * p.k + i], p.V)) atomicOr(&bits[id >> 5], 1u << (id & 31));
        }
        row_sync<NT>();
    }
    const auto entry_bits = [&](int col) { return TAIL ? bits[col >> 5] >> (col & 31) : 0u; };
    const int nvec = p.V / N, tail = p.V - nvec * N;
    Sum a = {kLowest, 0.f};
    float best = -INFINITY;
    const float last = tid < tail && !(entry_bits(nvec * N + tid) & 1) ? wide(x[nvec * N + tid]) : -INFINITY;
    for (int v0 = 0; v0 < nvec; v0 += NT * DS_NV) {
        typename RowVec<E>::type v[DS_NV];
        uint32_t skip[DS_NV];  // elements of entries, or past the end
#pragma unroll
        for (int j = 0; j < DS_NV; j++) v[j] = load_row(x + (size_t)min(v0 + j * NT + tid, nvec - 1) * N);
#pragma unroll
        for (int j = 0; j < DS_NV; j++) {
            const int i = v0 + j * NT + tid;
            skip[j] = i >= nvec ? ~0u : entry_bits(i * N);
            if (TAIL) {
#pragma unroll
                for (int k = 0; k < N; k++) best = fmaxf(best, skip[j] >> k & 1 ? -INFINITY : wide(v[j][k]));
            } else if (i < nvec) {
#pragma unroll
                for (int k = 0; k < N; k++) best = fmaxf(best, wide(v[j][k]));
            }
        }
        rescale(a, fmaxf(a.m, best), c);
#pragma unroll
        for (int j = 0; j < DS_NV; j++) {
            if (!TAIL && skip[j]) continue;
#pragma unroll
            for (int k = 0; k < N; k++) a.s += fast_exp2((TAIL && (skip[j] >> k & 1) ? -INFINITY : wide(v[j][k]) - a.m) * c);
        }
    }
    rescale(a, fmaxf(a.m, fmaxf(best, last)), c);
    a.s += fast_exp2((last - a.m) * c);
    const float m = wave_max(a.m);
    rescale(a, m, c);
    a.s = wave_sum(a.s);
    if (W > 1) {
        if (lane == 0) red[sub][wv] = a;
        __syncthreads();
        a = red[sub][0];
#pragma unroll 3
        for (int w = 1; w < W; w++) join(a, red[sub][w], c);
    }
    if (tid == 0) {
        DistillRow* keep = reinterpret_cast<DistillRow*>(p.kept) + r;
        keep->rm = a.m;
        keep->rls = a.s;
    }
}

// The rows' losses and what the gradient needs, from those sums and the entries: a
// wave to a row, rows beyond the grid in turn, and the workgroup's part of the mean.
template <class E, bool TAIL, int Q>  // Q: most entries of a lane
__global__ __launch_bounds__(256) void distill_rows_kernel(DistillParams p) {
    __shared__ double part_s[2][4];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const float c = kLog2e / p.temperature;
    const double T = p.temperature;
    double part = 0., parts = 0.;
    for (long long r = (long long)blockIdx.x * 4 + wv; r < p.rows; r += (long long)gridDim.x * 4) {
        const E* x = static_cast<const E*>(row_at(p, r, sizeof(E)));
        DistillRow* keep = reinterpret_cast<DistillRow*>(p.kept) + r;
        const Sum a = {keep->rm, keep->rls};  // (nothing yet in rows that do not count)
        int id[Q];  // -1: none
        float t[Q], e[Q];
        float tmax = -INFINITY;
        bool any = false;
#pragma unroll
        for (int q = 0; q < Q; q++) {
            const int i = q * 64 + lane;
            id[q] = -1;
            t[q] = e[q] = 0.f;
            if (i < p.k) {
                const long long at = p.ids[r * p.k + i];
                t[q] = p.values[r * p.k + i];
                if (counts(at, t[q], p.V)) {
                    id[q] = (int)at;
                    e[q] = wide(x[at]);
                    tmax = fmaxf(tmax, t[q]);
                    any = true;
                }
            }
        }
        const float weight = __any(any) ? (p.weights ? p.weights[r] : 1.f) : 0.f;
        if (weight == 0.f) {
            if (lane == 0) {
                keep->weight = 0.f;
                keep->loss = 0.f;
            }
            continue;
        }
        Sum all = a;
        if (TAIL) {  // the entries' columns, each once
            bool again[Q] = {};
#pragma unroll
            for (int q = 0; q < Q; q++)
                for (int j = 0; j < min(64, p.k - q * 64); j++) {
                    const int other = __builtin_amdgcn_readlane(id[q], j);
#pragma unroll
                    for (int o = 0; o < Q; o++) again[o] |= other == id[o] && q * 64 + j < o * 64 + lane;
                }
            Sum b = {kLowest, 0.f};
#pragma unroll
            for (int q = 0; q < Q; q++)
                if (id[q] >= 0 && !again[q]) {
                    rescale(b, fmaxf(b.m, e[q]), c);
                    b.s += fast_exp2((e[q] - b.m) * c);
                }
            const float bm = wave_max(b.m);
            rescale(b, bm, c);
            b.s = wave_sum(b.s);
            join(all, b, c);
        }
        const float ls = log2f(all.s), rls = log2f(a.s);
        tmax = wave_max(tmax);
        // masses (TAIL: in double, since 1 - their sum cancels) over their norm
        double p_[Q], mass = 0.;
#pragma unroll
        for (int q = 0; q < Q; q++) {
            p_[q] = id[q] < 0 ? 0. : TAIL ? exp((double)t[q]) : (double)fast_exp2((t[q] - tmax) * c);
            mass += p_[q];
        }
        mass = wave_sum(mass);
        const double top = TAIL ? 0. : (double)tmax, lognorm = TAIL ? 0. : (double)logf((float)mass), scale = TAIL ? 1. : 1. / mass;
        double loss = 0.;
#pragma unroll
        for (int q = 0; q < Q; q++)
            if (id[q] >= 0 && p_[q] != 0.) {  // (in double: a mask's lowest value over T, or a row's sum, passes fp32)
                const double lq = ((double)e[q] - (double)all.m) / T - kLn2 * (double)ls;
                loss += p_[q] * scale * ((((double)t[q] - top) / T - lognorm) - lq);
            }
        loss = wave_sum(loss);
        DistillRow row;
        row.m = all.m;
        row.ls = ls;
        row.rm = TAIL && a.s == 0.f ? 0.f : a.m;  // (no column of no entry but -inf: a softmax of zeros)
        row.rls = TAIL && a.s == 0.f ? 0.f : rls;
        row.rest = row.entry = 1.f;
        row.top = (float)top;
        row.norm = (float)(lognorm * 1.4426950408889634);
        row.weight = weight;
        if (TAIL) {
            // the rest, where the student has any
            const double pr = a.s > 0.f ? fmax(0., 1. - mass) : 0.;
            const double lqr = ((double)a.m - (double)all.m) + kLn2 * ((double)rls - (double)ls);
            if (pr > 0.) loss += pr * (log(pr) - lqr);
            row.entry = (float)(mass + pr);
            row.rest = (float)(exp(lqr) * (mass + pr) - pr);
        }
        row.loss = (float)loss;
        if (lane == 0) *keep = row;
        part += (double)weight * loss;
        parts += (double)weight;
    }
    if (lane == 0) {
        part_s[0][wv] = part;
        part_s[1][wv] = parts;
    }
    __syncthreads();
    if (threadIdx.x < 2) {
        const double* s = part_s[threadIdx.x];
        p.parts[2 * blockIdx.x + threadIdx.x] = ((s[0] + s[1]) + s[2]) + s[3];
    }
}

// The weighted mean over the rows from the workgroups' parts, in a fixed order.
__global__ __launch_bounds__(1024) void distill_mean_kernel(DistillParams p, int parts) {
    __shared__ double sums[2][16];
    double s = 0., n = 0.;
#pragma unroll
    for (int i = 0; i < DISTILL_PARTS / 1024; i++) {
        const int at = i * 1024 + threadIdx.x;
        if (at < parts) {
            s += p.parts[2 * at];
            n += p.parts[2 * at + 1];
        }
    }
    s = wave_sum(s);
    n = wave_sum(n);
    if ((threadIdx.x & 63) == 0) {
        sums[0][threadIdx.x >> 6] = s;
        sums[1][threadIdx.x >> 6] = n;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        s = n = 0.;
        for (int w = 0; w < 16; w++) {
            s += sums[0][w];
            n += sums[1][w];
        }
        *p.loss = (float)(s / n);
        *p.total = (float)n;
    }
}

// The gradient of the columns [c0, c1) of a row by NT threads: blockIdx.y's
// share of the row, whole vectors. The entries' columns are stored a second
// time, by one thread each. (Vectors that look for the entries among theirs
// instead took 345 us for 347 with 20 of them, and 65 for 34 with 64.) The rows
// are taken from the last to the first: those that the forward read last are in
// the caches still; a large gradient in whole lines goes past them (STREAM).
template <class E, int NT, bool STREAM>
__global__ __launch_bounds__(256) void distill_grad_kernel(DistillParams p, int share) {
    constexpr int N = RowVec<E>::N, RW = 256 / NT;
    __shared__ int id_s[RW][DISTILL_MAX_K];  // column in the share; -1: none
    __shared__ float mass_s[RW][DISTILL_MAX_K];
    const int tid = threadIdx.x % NT, sub = threadIdx.x / NT;
    int* const id = id_s[sub];
    float* const mass = mass_s[sub];
    const int c0 = blockIdx.y * share, c1 = min(c0 + share, p.V);
    const int nvec = (c1 - c0) / N, tail = c1 - c0 - nvec * N;
    const float c = kLog2e / p.temperature;
    for (long long i = (long long)blockIdx.x * RW + sub; i < p.rows; i += (long long)gridDim.x * RW) {
        const long long r = p.rows - 1 - i;
        const E* x = static_cast<const E*>(row_at(p, r, sizeof(E))) + c0;
        E* dx = static_cast<E*>(p.dx) + r * p.V + c0;
        const DistillRow row = reinterpret_cast<const DistillRow*>(p.kept)[r];
        const float g = row.weight == 0.f ? 0.f : *p.d_loss * row.weight / *p.total / p.temperature;
        typename RowVec<E>::type o;
        if (g == 0.f) {
#pragma unroll
            for (int k = 0; k < N; k++) o[k] = (E)0.f;
            for (int j = tid; j < nvec; j += NT) store_row<E, STREAM>(dx + (size_t)j * N, o);
            if (tid < tail) dx[nvec * N + tid] = (E)0.f;
            continue;
        }
        for (int j = tid; j < p.k; j += NT) {
            const long long at = p.ids[r * p.k + j];
            const float t = p.values[r * p.k + j];
            id[j] = at >= c0 && at < c1 && t != -INFINITY ? (int)at - c0 : -1;
            mass[j] = fast_exp2((t - row.top) * c - row.norm);
        }
        const float a = g * row.rest;
        const auto grad = [&](float e) { return a * fast_exp2((e - row.rm) * c - row.rls); };
        for (int i0 = 0; i0 < nvec; i0 += NT * DS_NV) {
            typename RowVec<E>::type v[DS_NV];
#pragma unroll
            for (int j = 0; j < DS_NV; j++) v[j] = load_row(x + (size_t)min(i0 + j * NT + tid, nvec - 1) * N);
#pragma unroll
            for (int j = 0; j < DS_NV; j++) {
                const int at = i0 + j * NT + tid;
                if (at < nvec) {
#pragma unroll
                    for (int k = 0; k < N; k++) o[k] = (E)grad(wide(v[j][k]));
                    store_row<E, STREAM>(dx + (size_t)at * N, o);
                }
            }
        }
        if (tid < tail) dx[nvec * N + tid] = (E)grad(wide(x[nvec * N + tid]));
        row_sync<NT>();  // the entries' columns are written again, by the first entry of each
        for (int j = tid; j < p.k; j += NT) {
            const int at = id[j];
            if (at < 0) continue;
            bool first = true;
            float sum = 0.f;
            for (int l = 0; l < p.k; l++)
                if (id[l] == at) {
                    if (l < j) first = false;
                    sum += mass[l];
                }
            if (first) dx[at] = (E)(g * (fast_exp2((wide(x[at]) - row.m) * c - row.ls) * row.entry - sum));
        }
        row_sync<NT>();
    }
}

template <class E, int NT>
void launch_sums(DistillParams p, hipStream_t stream) {
    constexpr int RW = rows_of(NT);
    p.words = (p.V + 31) / 32;
    for (p.first = 0; p.first < p.rows; p.first += (long long)LOGPROBS_MAX_GRID * RW) {
        const dim3 grid((unsigned)min((p.rows - p.first + RW - 1) / RW, (long long)LOGPROBS_MAX_GRID)), block(NT * RW);
        if (p.tail)
            hipLaunchKernelGGL((distill_sums_kernel<E, NT, true>), grid, block, (size_t)p.words * 4 * RW, stream, p);
        else
            hipLaunchKernelGGL((distill_sums_kernel<E, NT, false>), grid, block, 0, stream, p);
    }
}

// Whether the gradient goes past the caches: 128 MiB or more, in rows of whole
// 128-byte lines.
template <class E>
bool past_caches(const DistillParams& p) {
    return p.V * sizeof(E) % 128 == 0 && (uintptr_t)p.dx % 128 == 0 && (size_t)p.rows * p.V * sizeof(E) >= (size_t)128 << 20;
}

template <class E, int NT>
void launch_grad(const DistillParams& p, int shares, hipStream_t stream) {
    constexpr int N = RowVec<E>::N, RW = 256 / NT;
    const int share = ((p.V + shares - 1) / shares + N - 1) / N * N;
    const dim3 grid((unsigned)min((p.rows + RW - 1) / RW, (long long)LOGPROBS_MAX_GRID), (unsigned)((p.V + share - 1) / share));
    if (past_caches<E>(p))
        hipLaunchKernelGGL((distill_grad_kernel<E, NT, true>), grid, dim3(256), 0, stream, p, share);
    else
        hipLaunchKernelGGL((distill_grad_kernel<E, NT, false>), grid, dim3(256), 0, stream, p, share);
}

// Workgroups that the rows' losses are formed by.
int parts_of(long long rows) { return (int)min((rows + 3) / 4, (long long)DISTILL_PARTS); }

template <class E>
void launch(const DistillParams& p, bool grad, hipStream_t stream) {
    constexpr int N = RowVec<E>::N;
    const bool narrow = p.V <= 64 * DS_NV * N;
    if (grad) {
        if (narrow)
            launch_grad<E, 64>(p, 1, stream);
        else  // few rows shared out to about four workgroups of a compute unit
            launch_grad<E, 256>(p, (int)min((1024 + p.rows - 1) / p.rows, (long long)(p.V + 256 * N - 1) / (256 * N)), stream);
        return;
    }
    narrow ? launch_sums<E, 64>(p, stream) : launch_sums<E, 256>(p, stream);
    const dim3 grid((unsigned)parts_of(p.rows));
    const auto run = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, stream, p); };
    if (p.k <= 64)
        p.tail ? run(distill_rows_kernel<E, true, 1>) : run(distill_rows_kernel<E, false, 1>);
    else
        p.tail ? run(distill_rows_kernel<E, true, DISTILL_MAX_K / 64>) : run(distill_rows_kernel<E, false, DISTILL_MAX_K / 64>);
}

}  // namespace

void launch_distill(const DistillParams& p, int dtype, bool grad, hipStream_t stream) {
    if (p.rows > 0) {
        if (dtype == 0)
            launch<bf16_t>(p, grad, stream);
        else if (dtype == 1)
            launch<float>(p, grad, stream);
        else
            launch<f16_t>(p, grad, stream);
    }
    if (!grad) hipLaunchKernelGGL(distill_mean_kernel, dim3(1), dim3(1024), 0, stream, p, parts_of(p.rows));
}

}  // namespace cyfa
