// cyfa_sample.hip -- the choice of a token from each row of logits, by
// temperature T, top-k, top-p and min-p and a number u in [0, 1). Weights
// w_j = e^((x_j - max) / T); the order is by falling x, the lower index first.
// Kept are the first top_k; of those, the ones before which less than top_p of
// their mass lies; of those, the ones with w >= min_p: each a prefix of the
// order, so that one key (value, index) tells what is kept. The token is the
// first kept one in the order of the indexes at which the running mass of the
// kept passes u times their mass.
//
// Which token that is must not depend on the order of a sum: weights are formed
// in double and held as integers, multiples of 2^-46 of the largest (fewer bits
// past 2^16 columns, so that a row's sum fits 64), and integers add up the same
// in any order. Weights below half of that step count nothing.
//
// Whole distributions (and what min_p leaves of them) take two passes over a row,
// the maximum and the weights (sample_draw_kernel). Where top_k or top_p cut them
// (sample_kernel), a workgroup to a row, whose passes find it in the L2 (rows held
// in LDS took as long: 13.6 us against 14.0 for 256 rows of 32000 bf16). A prefix
// is found by counting: the elements, or their mass, by bins of their distance to
// the maximum; the bin in which the prefix ends gives its elements to a list, whose
// keys are binned again until few enough are left to rank each against each.
// Masses are counted for runs of the row apart, so that the run that holds the
// token is known from the bins and its weights alone are formed again. A top_k of
// at most 128, the usual one, needs no bins: a value that at least k elements reach
// and seldom many more is the k-th largest of the largest elements of 64 (128) sets
// of threads, and the few that reach it are ranked, cut and drawn from by one wave.
//
// Few wide rows are shared out: a workgroup to each part of a row finds its
// maximum, a second launch counts the parts' bins, and a third, a workgroup to a
// row, goes on from there with the parts as runs.
//
// An element's weight costs 17 operations in double, of 4.3 to 5 cycles of a SIMD
// each, and 6 others, some 95 cycles a wave: 0.6 ps on 256 compute units, where two
// bytes take 0.4 from memory and four 0.8. What bounds a call is that a row's steps
// follow one another (its maximum from memory, its weights, and where it is cut a
// 64-bit LDS atomic an element, the border's list and the draw) in few workgroups a
// compute unit: 80 to 124 vector registers leave room for two or three of 512 threads.
// Rows of a single compute unit each wait besides at their dozen barriers. us, bf16:
// 1024 x 32000 whole 49, top_k 50 37, top_p 0.9 69; 1021 x 50001 fp32 80 to 84, 72, 140.
#include <type_traits>

#include "cyfa_internal.h"
#include "cyfa_rows.h"

namespace cyfa {

namespace {

typedef unsigned long long u64;

constexpr double kLog2eD = 1.4426950408889634;
constexpr int SM_FEW = 512;   // elements ranked each against each, by eight threads each
constexpr int SM_PIECE = 4;  // elements of a row's piece
constexpr int SM_TOP = 128;   // largest top_k that one wave handles

__device__ __forceinline__ uint32_t value_key(float x) {
    x += 0.f;  // -0 equals +0
    const uint32_t b = __builtin_bit_cast(uint32_t, x);
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}

__device__ __forceinline__ u64 order_key(float x, int i) { return (u64)value_key(x) << 32 | (0xffffffffu - (uint32_t)i); }

__device__ __forceinline__ float key_value(u64 key) {
    const uint32_t k = (uint32_t)(key >> 32);
    return __builtin_bit_cast(float, (k & 0x80000000u) ? k ^ 0x80000000u : ~k);
}

__device__ __forceinline__ int key_index(u64 key) { return (int)(0xffffffffu - (uint32_t)key); }

// The value of another lane: 0 where the pattern reads none or MASK leaves the row out.
template <int CTRL, int MASK = 0xF>
__device__ __forceinline__ u64 dpp_or_zero(u64 x) {
    const i32x2 v = __builtin_bit_cast(i32x2, x);
    return __builtin_bit_cast(u64, i32x2{__builtin_amdgcn_update_dpp(0, v[0], CTRL, MASK, 0xF, false),
                                         __builtin_amdgcn_update_dpp(0, v[1], CTRL, MASK, 0xF, false)});
}

// The sum over this lane and those below it: within rows of 16 by shifts, then
// the last lane of each row to the row after, of each half to the half after.
__device__ __forceinline__ u64 wave_scan(u64 x) {
    x += dpp_or_zero<0x111>(x);
    x += dpp_or_zero<0x112>(x);
    x += dpp_or_zero<0x114>(x);
    x += dpp_or_zero<0x118>(x);
    x += dpp_or_zero<0x142, 0xA>(x);
    x += dpp_or_zero<0x143, 0xC>(x);
    return x;
}

__device__ __forceinline__ u64 lane_u64(u64 x, int lane) {
    return (u64)(uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), lane) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)x, lane);
}

// The sum over the lanes, in every lane.
__device__ __forceinline__ u64 wave_add(u64 x) { return lane_u64(wave_scan(x), 63); }

// The sum over eight lanes (8 i .. 8 i + 7), in each of them.
__device__ __forceinline__ unsigned eight_add(unsigned x) {
    x += (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0xB1, 0xF, 0xF, false);
    x += (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x4E, 0xF, 0xF, false);
    return x + (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x141, 0xF, 0xF, false);
}

__device__ __forceinline__ u64 eight_add(u64 x) {
    x += dpp_or_zero<0xB1>(x);
    x += dpp_or_zero<0x4E>(x);
    return x + dpp_or_zero<0x141>(x);
}

// The largest of the lanes, in every lane: as wave_max.
__device__ __forceinline__ u64 wave_most(u64 x) {
    const auto most = [](u64 a, u64 b) { return a > b ? a : b; };
    const auto moved = [](u64 x, auto step) {
        return __builtin_bit_cast(u64, dpp_mov<decltype(step)::value>(__builtin_bit_cast(double, x)));
    };
    x = most(x, moved(x, std::integral_constant<int, 0xB1>{}));
    x = most(x, moved(x, std::integral_constant<int, 0x4E>{}));
    x = most(x, moved(x, std::integral_constant<int, 0x141>{}));
    x = most(x, moved(x, std::integral_constant<int, 0x140>{}));
    return most(most(lane_u64(x, 0), lane_u64(x, 16)), most(lane_u64(x, 32), lane_u64(x, 48)));
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

// The same of 128 values, two of each lane.
__device__ __forceinline__ float kth_largest(float x, float y, int k) {
    const uint32_t a = (value_key(x) & ~127u) | (uint32_t)(threadIdx.x & 63), b = (value_key(y) & ~127u) | 64u | (uint32_t)(threadIdx.x & 63);
    int ra = 0, rb = 0;
#pragma unroll 8
    for (int i = 0; i < 64; i++) {
        const uint32_t oa = (uint32_t)__builtin_amdgcn_readlane((int)a, i), ob = (uint32_t)__builtin_amdgcn_readlane((int)b, i);
        ra += (oa > a) + (ob > a);
        rb += (oa > b) + (ob > b);
    }
    return -wave_max(fmaxf(ra < k ? -x : -INFINITY, rb < k ? -y : -INFINITY));
}

// A row's settings.
struct Choice {
    double m;       // the maximum
    double c;       // log2 e / T
    double least;   // a distance to the maximum whose weight is nothing
    double unit;    // 2^(52 - bits): weights are multiples of 2^-bits
    double k[10];   // kExp2, in scalar registers
};

// The coefficients of the polynomial of degree 10 that meets 2^f at the Chebyshev
// points of [-1/2, 1/2] (off by at most 3.2e-16 of it), but for the first, 1.
constexpr int SM_DEGREE = 10;
__device__ constexpr double kExp2[SM_DEGREE] = {0.69314718055995,       0.24022650695910097,   0.05550410866444772,    0.009618129107606888,
                                                0.0013333558230164974,  0.0001540353044173605, 1.5252657260200837e-05, 1.321544258792169e-06,
                                                1.0208690299958306e-07, 7.072585949269223e-09};

// 2^((x - m) c) as an integer multiple of 2^-bits, without a branch: adding 1.5
// 2^52 leaves the exponent's whole part n in the low bits; 2^n is put into the
// exponent of the polynomial of the rest; adding 2^(52 - bits) rounds to an integer
// in the low bits.
__device__ __forceinline__ u64 weight(const Choice& ch, float x) {
    const double d = fmax((double)x - ch.m, ch.least);
    const double shifted = fma(d, ch.c, 0x1.8p52), f = fma(d, ch.c, 0x1.8p52 - shifted);
    double y = ch.k[SM_DEGREE - 1];
#pragma unroll
    for (int i = SM_DEGREE - 2; i >= 0; i--) y = fma(y, f, ch.k[i]);
    y = fma(y, f, 1.0);
    i32x2 bits = __builtin_bit_cast(i32x2, y);
    bits[1] += __builtin_bit_cast(i32x2, shifted)[0] << 20;
    return __builtin_bit_cast(u64, __builtin_bit_cast(double, bits) + ch.unit) & 0xfffffffffffffull;
}

// What one launch finds of a part of a row for the next.
struct PartStats {
    float best, least;  // the maximum, the least element
    int bad;            // a NaN is there
    int pad;
};

constexpr int SM_BINS = 512;  // bins of a part

// The bins: of the distance to the maximum, over that of the least element or
// what the temperature leaves of it, whichever is less.
struct Bins {
    float m, inv, last;
    __device__ __forceinline__ Bins(float m, float least, double T, int bins) : m(m), last((float)(bins - 1)) {
        const float span = fminf(m - least, 40.f * fmaxf((float)T, 1.f));
        inv = span > 0.f ? (float)bins / span : 0.f;
    }
    __device__ __forceinline__ int of(float e) const { return (int)fminf((m - e) * inv, last); }
};

template <class E>
__device__ __forceinline__ const E* row_of(const SampleParams& p, long long r) {
    return static_cast<const E*>(p.x) + (r / p.inner) * p.outer_stride + (r % p.inner) * p.row_stride;
}

__device__ __forceinline__ void set_choice(Choice& ch, float m, double T) {
    ch.m = m;
    ch.c = fmax(fmin(kLog2eD / T, 1e300), 1e-300);  // (0 times it stays 0, -inf times it -inf)
    ch.least = -60. / ch.c;
}

__device__ __forceinline__ Choice choice_of(const SampleParams& p, float m, double T) {
    Choice ch;
    set_choice(ch, m, T);
    ch.unit = p.unit;
#pragma unroll
    for (int i = 0; i < SM_DEGREE; i++) {
        ch.k[i] = kExp2[i];
        asm("" : "+s"(ch.k[i]));  // (as literals each would be moved to the sum's registers before its product)
    }
    return ch;
}

// The least fp32 value that min_p keeps of a row; the largest is always kept. (An
// infinite temperature gives all finite ones the weight 1.)
__device__ __forceinline__ float lowest_of(double min_p, double m, double T) {
    float lowest = -INFINITY;
    if (min_p > 0. && T < INFINITY) {
        const double border = fmin(m, m + T * log(min_p));
        lowest = (float)border;
        if ((double)lowest < border) lowest = nextafterf(lowest, INFINITY);
    }
    return lowest;
}

// What the running mass has to pass.
__device__ __forceinline__ u64 mass_at(double u, u64 total) {
    const u64 target = u > 0. ? (u64)fmin(u * (double)total, 0x1p63) : 0;
    return target >= total ? total - 1 : target;
}

// f(piece, its index) of the whole pieces begin, begin + STEP, ... below end of a
// row, each on its way while the one before is worked on.
template <int STEP, class E, class F>
__device__ __forceinline__ void each_piece(const E* x, int begin, int end, F&& f) {
    typedef E Piece __attribute__((ext_vector_type(SM_PIECE)));
    if (begin >= end) return;
    const auto load = [&](int i) {
        Piece v;
        __builtin_memcpy(&v, x + (size_t)i * SM_PIECE, sizeof v);
        return v;
    };
    Piece next = load(begin);
    asm volatile("" : "+v"(next));  // (else the compiler takes this load for the loop's, and waits for each where it is used)
#pragma unroll 1
    for (int i = begin; i < end; i += STEP) {
        const Piece v = next;
        next = load(min(i + STEP, end - 1));
        f(v, i);
    }
}

// This part of a row: maximum, least element, NaN. Parts are whole vectors.
template <class E>
__global__ __launch_bounds__(256) void sample_stats_kernel(SampleParams p) {
    constexpr int N = RowVec<E>::N;
    __shared__ float red[2][4];
    __shared__ int bad_s[4];
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const long long r = blockIdx.x;
    const int c0 = blockIdx.y * p.part, cols = min(p.part, p.V - c0), nvec = cols / N, tail = cols - nvec * N;
    const E* x = row_of<E>(p, r) + c0;
    float best = -INFINITY, least = INFINITY;
    bool bad = false;
    const auto add = [&](E v) {
        best = __builtin_elementwise_maximum(best, wide(v));  // (a NaN stays)
        least = __builtin_elementwise_minimum(least, wide(v));
    };
#pragma unroll 2
    for (int i = tid; i < nvec; i += 256) {
        const typename RowVec<E>::type v = load_row(x + (size_t)i * N);
#pragma unroll
        for (int c = 0; c < N; c++) add(v[c]);
    }
    if (tid < tail) add(x[nvec * N + tid]);
    bad = __any(best != best);
    best = wave_max(best);
    least = -wave_max(-least);
    if (lane == 0) {
        red[0][wv] = best;
        red[1][wv] = least;
        bad_s[wv] = bad;
    }
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < 4; w++) {
            best = fmaxf(best, red[0][w]);
            least = fminf(least, red[1][w]);
            bad |= bad_s[w] != 0;
        }
        static_cast<PartStats*>(p.stats)[r * gridDim.y + blockIdx.y] = {best, least, bad, 0};
    }
}

// A row's maximum, least element and NaN from those of its parts, in every lane.
__device__ __forceinline__ PartStats join_parts(const SampleParams& p, long long r, int parts) {
    PartStats a = {-INFINITY, INFINITY, 0, 0};
    for (int i = threadIdx.x & 63; i < parts; i += 64) {
        const PartStats b = static_cast<const PartStats*>(p.stats)[r * parts + i];
        a.best = fmaxf(a.best, b.best);
        a.least = fminf(a.least, b.least);
        a.bad |= b.bad;
    }
    a.best = wave_max(a.best);
    a.least = -wave_max(-a.least);
    a.bad = __any(a.bad);
    return a;
}

// The counts and masses of a part's bins (16 rows of 131072 bf16, a part of 4096 to
// a workgroup: the statistics 3 us, the bins 6, the rows themselves 25).
template <class E>
__global__ __launch_bounds__(256) void sample_bins_kernel(SampleParams p) {
    constexpr int P = SM_PIECE;
    __shared__ u64 mass_s[SM_BINS];
    __shared__ unsigned count_s[SM_BINS];
    const int tid = threadIdx.x;
    const long long r = blockIdx.x;
    const int c0 = blockIdx.y * p.part, cols = min(p.part, p.V - c0), npiece = cols / P, tail = cols - npiece * P;
    const double T = p.temperatures ? (double)p.temperatures[r] : p.temperature;
    const PartStats a = join_parts(p, r, gridDim.y);
    if (a.bad || a.best == INFINITY || a.best == -INFINITY || !(T > 0.)) return;  // (no bins are read)
    const E* x = row_of<E>(p, r) + c0;
    const Choice ch = choice_of(p, a.best, T);
    const Bins bins(a.best, a.least, T, SM_BINS);
    for (int b = tid; b < SM_BINS; b += 256) {
        mass_s[b] = 0;
        count_s[b] = 0;
    }
    __syncthreads();
    const auto add = [&](E v) {
        const int b = bins.of(wide(v));
        atomicAdd(&count_s[b], 1u);
        atomicAdd(&mass_s[b], weight(ch, wide(v)));
    };
    each_piece<256>(x, tid, npiece, [&](const auto& v, int) {
#pragma unroll
        for (int c = 0; c < P; c++) add(v[c]);
    });
    if (tid < tail) add(x[npiece * P + tid]);
    __syncthreads();
    const long long at = (r * gridDim.y + blockIdx.y) * SM_BINS;
    for (int b = tid; b < SM_BINS; b += 256) {
        p.part_mass[at + b] = mass_s[b];
        p.part_count[at + b] = count_s[b];
    }
}

// The rows of a launch, a workgroup each. PARTS: with what the two launches before
// found of the row's p.parts parts.
// Passes that form weights take the row in pieces of four elements: of eight the
// compiler holds all exponentials' operands at a time, and spills them.
template <class E, int NT, bool PARTS>
__global__ __launch_bounds__(NT) void sample_kernel(SampleParams p) {
    typedef typename RowVec<E>::type Vec;
    constexpr int N = RowVec<E>::N, P = SM_PIECE, W = NT / 64, BINS = NT > SM_BINS ? SM_BINS : NT;
    constexpr int RUNS = W > 8 ? 8 : W;
    typedef E Piece __attribute__((ext_vector_type(P)));
    __shared__ u64 run_s[PARTS ? 1 : RUNS][BINS];  // masses of the runs' bins
    __shared__ u64 mass_s[BINS];
    __shared__ unsigned count_s[BINS];
    __shared__ u64 list_s[NT], all_s[NT];
    __shared__ u64 list_w[SM_FEW < NT ? SM_FEW : NT];
    __shared__ u64 red_s[2][W];
    __shared__ u64 runs_s[PARTS ? SAMPLE_PARTS : W];  // masses of the kept in the runs
    __shared__ float redf_s[2][W], thr_s;
    __shared__ unsigned redu_s[W];
    __shared__ u64 found_mass, found_key, found_kept;
    __shared__ unsigned found_count, found_n;
    __shared__ int found_bin, held_s, vecs_s;
    float* const sets_s = reinterpret_cast<float*>(all_s);  // [W][64], until the list is used
    int* const near_s = reinterpret_cast<int*>(mass_s);     // [2 BINS], while no bins are counted
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const int full = p.V / N, nvec = (p.V + N - 1) / N, npiece = (p.V + P - 1) / P;
    const long long r = p.first + blockIdx.x;
    const E* x = row_of<E>(p, r);
    const double T = p.temperatures ? (double)p.temperatures[r] : p.temperature;
    const double top_p = p.top_ps ? (double)p.top_ps[r] : p.top_p;
    const double min_p = p.min_ps ? (double)p.min_ps[r] : p.min_p;
    const long long top_k = p.top_ks ? p.top_ks[r] : p.top_k;
    const double u = p.uniform64 ? p.uniform64[r] : (double)p.uniform[r];
    // Vector i of the row; the columns past the last are -inf.
    const auto from_memory = [&](int i) {
        Vec v;
        if (i < full) {
            v = load_row(x + (size_t)i * N);
        } else {
#pragma unroll
            for (int c = 0; c < N; c++) v[c] = i * N + c < p.V ? x[(size_t)i * N + c] : (E)-INFINITY;
        }
        return v;
    };
    const auto piece = [&](int i) {
        Piece v;
        if ((i + 1) * P <= p.V) {
            __builtin_memcpy(&v, x + (size_t)i * P, sizeof v);
        } else {
#pragma unroll
            for (int c = 0; c < P; c++) v[c] = i * P + c < p.V ? x[(size_t)i * P + c] : (E)-INFINITY;
        }
        return v;
    };
    // f(element, column) of this thread's elements in vectors that reach ``from``
    const auto each = [&](float from, auto&& f) {
#pragma unroll 1
        for (int i = tid; i < nvec; i += NT) {
            const Vec v = from_memory(i);
            float top = wide(v[0]);
#pragma unroll
            for (int c = 1; c < N; c++) top = fmaxf(top, wide(v[c]));
            if (top >= from)
#pragma unroll
                for (int c = 0; c < N; c++) f(wide(v[c]), i * N + c);
        }
    };
    // ---- the maximum, the least element, what no distribution holds
    float best = -INFINITY, least = INFINITY;
    bool bad = false;
    const bool cut_k = top_k > 0 && top_k < p.V, cut_p = top_p < 1., few = cut_k && top_k <= SM_TOP;
    if (tid == 0) held_s = 0;
    if (PARTS && !few) {
        const PartStats a = join_parts(p, r, p.parts);
        best = a.best;
        least = a.least;
        bad = a.bad;
    } else {
        constexpr int U = 4;  // vectors of a thread in flight
        for (int i0 = tid; i0 < nvec; i0 += NT * U) {
            Vec v[U];
#pragma unroll
            for (int j = 0; j < U; j++)
                if (i0 + j * NT < full) v[j] = load_row(x + (size_t)(i0 + j * NT) * N);
#pragma unroll
            for (int j = 0; j < U; j++) {
                const int i = i0 + j * NT;
                if (i >= nvec) continue;
                if (i == full) v[j] = from_memory(i);
#pragma unroll
                for (int c = 0; c < N; c++) {
                    best = __builtin_elementwise_maximum(best, wide(v[j][c]));  // (a NaN stays)
                    least = __builtin_elementwise_minimum(least, wide(v[j][c]));
                }
            }
        }
        sets_s[wv * 64 + lane] = best;
        bad = __any(best != best);
        best = wave_max(best);
        least = -wave_max(-least);
        if (lane == 0) {
            redf_s[0][wv] = best;
            redf_s[1][wv] = least;
            redu_s[wv] = bad;
        }
    }
    __syncthreads();
    if (!PARTS || few)
        for (int w = 0; w < W; w++) {
            best = fmaxf(best, redf_s[0][w]);
            least = fminf(least, redf_s[1][w]);
            bad |= redu_s[w] != 0;
        }
    const bool none = bad || best == INFINITY || best == -INFINITY;
    if (none || !(T > 0.)) {  // the first of the largest, a NaN before all
        unsigned at = 0xffffffffu;
        for (int i = tid; i < npiece; i += NT) {
            const Piece v = piece(i);
#pragma unroll
            for (int c = 0; c < P; c++)
                if (bad ? wide(v[c]) != wide(v[c]) : wide(v[c]) == best) at = min(at, (unsigned)(i * P + c));
        }
        for (int d = 32; d > 0; d >>= 1) at = min(at, (unsigned)__shfl_xor((int)at, d));
        __syncthreads();
        if (lane == 0) redu_s[wv] = at;
        __syncthreads();
        if (tid == 0) {
            for (int w = 1; w < W; w++) at = min(at, redu_s[w]);
            p.ids[r] = at;
            p.logprob[r] = none ? __builtin_nanf("") : 0.f;
        }
        return;
    }
    const Choice ch = choice_of(p, best, T);
    const float lowest = lowest_of(min_p, ch.m, T);
    const auto put = [&](int i, u64 w, u64 total) {
        p.ids[r] = i;
        p.logprob[r] = (float)log((double)w / (double)total);
    };
    u64 base = 0;          // kept so far: keys from here on
    float from = -INFINITY;  // its value
    if (few) {
        const int k = (int)top_k;
        if (wv == 0) {  // (of one set of threads a lane, or, past 64, of two)
            float most[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int w = 0; w < W; w += 2) {
                most[0] = fmaxf(most[0], sets_s[w * 64 + lane]);
                most[1] = fmaxf(most[1], sets_s[(w + 1) * 64 + lane]);
            }
            const float thr = k <= 64 ? kth_largest(fmaxf(most[0], most[1]), k) : kth_largest(most[0], most[1], k);
            if (lane == 0) thr_s = thr;
        }
        __syncthreads();
        const float thr = thr_s;
        each(thr, [&](float e, int i) {
            if (e >= thr) {
                const int at = atomicAdd(&held_s, 1);
                if (at < NT) list_s[at] = order_key(e, i);
            }
        });
        __syncthreads();
        const int n = held_s;
        if (n <= min(SM_FEW, NT)) {
            for (int at = tid / 8; at < n; at += NT / 8) {  // eight threads to one
                const u64 key = list_s[at];
                int rank = 0;
#pragma unroll 4
                for (int i = tid & 7; i < n; i += 8) rank += list_s[i] > key;
#pragma unroll
                for (int d = 4; d > 0; d >>= 1) rank += __shfl_xor(rank, d);
                if ((tid & 7) == 0 && rank < k) all_s[rank] = key;
            }
            __syncthreads();
            const auto draw = [&](auto halves) {  // a lane to each of the first 64 and (2) to each of the second
                constexpr int H = decltype(halves)::value;
                u64 keys[H], w[H], sum[H], before = 0;
                float e[H];
#pragma unroll
                for (int h = 0; h < H; h++) {
                    keys[h] = lane + 64 * h < k ? all_s[lane + 64 * h] : 0;
                    e[h] = key_value(keys[h]);
                    w[h] = lane + 64 * h < k ? weight(ch, e[h]) : 0;
                    sum[h] = before + wave_scan(w[h]);
                    before = lane_u64(sum[h], 63);
                }
                int kept = 0;
#pragma unroll
                for (int h = 0; h < H; h++)
                    kept += __popcll(__ballot((lane == 0 && h == 0) || (lane + 64 * h < k && e[h] >= lowest &&
                                                                        !(cut_p && (double)(sum[h] - w[h]) >= top_p * (double)before))));
                const u64 total = H > 1 && kept > 64 ? lane_u64(sum[H - 1], kept - 65) : lane_u64(sum[0], kept - 1), target = mass_at(u, total);
                u64 upto[H] = {};  // the mass of the kept up to these by index
                const auto pass = [&](u64 other, u64 ow) {
#pragma unroll
                    for (int h = 0; h < H; h++) upto[h] += (uint32_t)other >= (uint32_t)keys[h] ? ow : 0;
                };
                for (int i = 0; i < min(kept, 64); i++) pass(lane_u64(keys[0], i), lane_u64(w[0], i));
                if (H > 1)
                    for (int i = 64; i < kept; i++) pass(lane_u64(keys[H - 1], i - 64), lane_u64(w[H - 1], i - 64));
#pragma unroll
                for (int h = 0; h < H; h++)
                    if (lane + 64 * h < kept && upto[h] > target && upto[h] - w[h] <= target) put(key_index(keys[h]), w[h], total);
            };
            if (wv == 0) k <= 64 ? draw(std::integral_constant<int, 1>{}) : draw(std::integral_constant<int, 2>{});
            return;
        }
        from = thr;  // many equal elements: the bins tell
        base = order_key(thr, 0x7fffffff);
        if (PARTS) least = join_parts(p, r, p.parts).least;  // (without the -inf past the row's end: the parts' bins)
        __syncthreads();
    }
    const Bins bins(best, least, T, BINS);
    // The runs of the row: their masses by bins, whether they have been counted.
    int runs = PARTS ? p.parts : RUNS;
    int run_len = PARTS ? p.part / P : (npiece + RUNS - 1) / RUNS;  // pieces of a run
    bool counted = PARTS;
    const auto run_mass = [&](int run, int b) -> u64 { return PARTS ? p.part_mass[(r * runs + run) * BINS + b] : run_s[PARTS ? 0 : run][b]; };
    u64 total = 0;      // the mass of what the last search looked at
    int k_bin = BINS;   // PARTS: the bin in which top_k ends,
    u64 k_mass = 0;     // and the mass of its kept elements
    int in_all = -1;    // elements of the last border's bin in all_s, where it holds them
    // The values of a bin, but for their rounding: those within half of mid.
    const auto near_bin = [&](int bin, float& mid, float& half) {
        mid = 0.f;
        half = INFINITY;
        if (bin < BINS - 1 && bins.inv > 0.f) {
            const float width = 1.f / bins.inv, low = best - (float)(bin + 1) * width * (1.f + 0x1p-20f);
            const float high = best - (float)bin * width * (1.f - 0x1p-20f);
            mid = 0.5f * low + 0.5f * high;
            half = fmaxf(high - mid, mid - low);  // (roundings keep the order of differences from mid)
        }
    };
    // Lowers what is kept to the longest prefix that ``dropped`` (elements
    // before, mass before, all mass) does not end. MASS: it asks for the mass.
    const auto search = [&](auto with_mass, auto&& dropped) {
        constexpr bool MASS = decltype(with_mass)::value, BOTH = MASS || PARTS;
        // a bin's count and mass to those before it
        unsigned c, cb;
        u64 w, wb;
        const auto scan_bins = [&]() {
            const u64 cs = wave_scan(c), ws = BOTH ? wave_scan(w) : 0;
            if (lane == 63) {
                red_s[0][wv] = cs;
                red_s[1][wv] = ws;
            }
            __syncthreads();
            u64 cbase = 0, wbase = 0, all = 0;
            for (int i = 0; i < BINS / 64; i++) {
                if (i < wv) cbase += red_s[0][i];
                if (BOTH && i < wv) wbase += red_s[1][i];
                if (BOTH) all += red_s[1][i];
            }
            cb = (unsigned)(cbase + cs - c);
            wb = wbase + ws - w;
            return all;
        };
        const auto clear = [&]() {
            if (tid < BINS) {
                count_s[tid] = 0;
                if (BOTH) mass_s[tid] = 0;
            }
            if (tid == 0) {
                held_s = 0;
                vecs_s = 0;
                found_bin = -1;
            }
            __syncthreads();
        };
        const auto hit = [&](int b, float e) {
            atomicAdd(&count_s[b], 1u);
            if (BOTH) atomicAdd(&mass_s[b], weight(ch, e));
        };
        const auto read_bins = [&]() {
            c = tid < BINS ? count_s[tid] : 0;
            w = BOTH && tid < BINS ? mass_s[tid] : 0;
        };
        // the bin in which the prefix ends, known to all
        const auto find_border = [&](unsigned ca, u64 wa) {
            if (tid < BINS && !dropped(ca + cb, wa + wb, total) && dropped(ca + cb + c, wa + wb + w, total)) {
                found_bin = tid;
                found_count = ca + cb;
                found_mass = wa + wb;
                found_n = c;
            }
            __syncthreads();
        };
        if (!PARTS && MASS)
            for (int b = tid; b < RUNS * BINS; b += NT) run_s[0][b] = 0;
        clear();
        if (PARTS) {
            c = 0;
            w = 0;
            if (tid < BINS)
#pragma unroll 4
                for (int i = 0; i < runs; i++) {
                    c += p.part_count[(r * runs + i) * BINS + tid];
                    w += run_mass(i, tid);
                }
            if (tid >= k_bin) {  // past the first top_k
                c = 0;
                w = tid == k_bin ? k_mass : 0;
            }
        } else if (MASS) {  // (the count of the bin that matters is that of the list)
            counted = true;
            constexpr int STEP = NT / RUNS;
            const int run = wv * RUNS / W, begin = run * run_len, end = min(begin + run_len, p.V / P);
            const auto add = [&](float e, int i, int run) {
                if (base == 0 || (e >= from && order_key(e, i) >= base)) atomicAdd(&run_s[PARTS ? 0 : run][bins.of(e)], weight(ch, e));
            };
            if (base == 0) {
                each_piece<STEP>(x, begin + tid % STEP, end, [&](const auto& v, int) {
#pragma unroll
                    for (int c = 0; c < P; c++) atomicAdd(&run_s[PARTS ? 0 : run][bins.of(wide(v[c]))], weight(ch, wide(v[c])));
                });
            } else {
                each_piece<STEP>(x, begin + tid % STEP, end, [&](const auto& v, int i) {
#pragma unroll
                    for (int c = 0; c < P; c++) add(wide(v[c]), i * P + c, run);
                });
            }
            if (tid < p.V % P) {  // (columns behind the last whole piece)
                const int i = p.V / P * P + tid;
                add(wide(x[i]), i, i / P / run_len);
            }
            __syncthreads();
            c = 0;
            w = 0;
            if (tid < BINS)
#pragma unroll
                for (int i = 0; i < RUNS; i++) w += run_s[PARTS ? 0 : i][tid];
        } else {
            each(from, [&](float e, int i) {
                if (e >= from && order_key(e, i) >= base) atomicAdd(&count_s[bins.of(e)], 1u);
            });
            __syncthreads();
            read_bins();
        }
        total = scan_bins();
        find_border(0, 0);
        const int bin = found_bin;
        if (bin < 0) return;  // nothing is dropped
        unsigned ca = found_count, n;
        u64 wa = found_mass;
        const u64 above = wa;
        u64 lo = 0, hi = 0;  // the keys of the undecided, once they are known
        const auto range = [&](u64 low, u64 high) {
            low = ~wave_most(~low);
            high = wave_most(high);
            __syncthreads();
            if (lane == 0) {
                red_s[0][wv] = low;
                red_s[1][wv] = high;
            }
            __syncthreads();
            for (int i = 0; i < W; i++) {
                low = red_s[0][i] < low ? red_s[0][i] : low;
                high = red_s[1][i] > high ? red_s[1][i] : high;
            }
            lo = low;
            hi = high;
            __syncthreads();
        };
        const auto shift_of = [&]() {
            const u64 d = (hi - lo) / BINS;
            return d ? 64 - __builtin_clzll(d) : 0;
        };
        // narrows lo and hi to the bin found in them
        const auto narrow = [&](int shift) {
            const u64 high = hi - ((u64)found_bin << shift), size = ((u64)1 << shift) - 1;
            lo = high - lo > size ? high - size : lo;
            hi = high;
            ca = found_count;
            wa = found_mass;
            n = found_n;
        };
        // f(key) of the bin's elements
        const auto in_bin = [&](auto&& f) {
            each(from, [&](float e, int i) {
                if (e >= from && bins.of(e) == bin) {
                    const u64 key = order_key(e, i);
                    if (key >= base) f(key);
                }
            });
        };
        const auto hold = [&](u64 key) {
            const int at = atomicAdd(&held_s, 1);
            if (at < NT) all_s[at] = key;
        };
        // The vectors that hold some of them first: a wave's next 512 elements hold
        // one or two, and would all be looked at by themselves for those.
        float mid, half;
        near_bin(bin, mid, half);
#pragma unroll 2
        for (int i = tid; i < nvec; i += NT) {
            const Vec v = from_memory(i);
            float near = INFINITY;
#pragma unroll
            for (int c = 0; c < N; c++) near = fminf(near, fabsf(wide(v[c]) - mid));
            if (near <= half) {
                const int at = atomicAdd(&vecs_s, 1);
                if (at < 2 * BINS) near_s[at] = i;
            }
        }
        __syncthreads();
        const int vecs = vecs_s;
        if (vecs <= 2 * BINS) {
            for (int at = tid; at < vecs; at += NT) {
                const int i = near_s[at];
                const Vec v = from_memory(i);
#pragma unroll
                for (int c = 0; c < N; c++) {
                    const float e = wide(v[c]);
                    if (e >= from && bins.of(e) == bin) {
                        const u64 key = order_key(e, i * N + c);
                        if (key >= base) hold(key);
                    }
                }
            }
        } else {
            in_bin(hold);
        }
        __syncthreads();
        n = (unsigned)held_s;
        in_all = n > NT ? -1 : (int)n;
        if (n <= NT) {
            if (tid < (int)n) list_s[tid] = all_s[tid];
            __syncthreads();
        }
        if (n > NT) {  // too many for the list: bins of their keys
            u64 low = ~0ull, high = 0;
            in_bin([&](u64 key) {
                low = key < low ? key : low;
                high = key > high ? key : high;
            });
            range(low, high);
            while (n > NT) {
                const int shift = shift_of();
                clear();
                each(key_value(lo), [&](float e, int i) {
                    const u64 key = order_key(e, i);
                    if (key >= lo && key <= hi) hit((int)((hi - key) >> shift), e);
                });
                __syncthreads();
                read_bins();
                scan_bins();
                find_border(ca, wa);
                if (found_bin < 0) return;  // (never: the bins add up to what was undecided)
                narrow(shift);
                __syncthreads();
            }
            if (tid == 0) held_s = 0;
            __syncthreads();
            each(key_value(lo), [&](float e, int i) {
                const u64 key = order_key(e, i);
                if (key >= lo && key <= hi) list_s[atomicAdd(&held_s, 1)] = key;
            });
            __syncthreads();
        }
        while (n > SM_FEW) {  // (a thread to each of the list)
            const u64 key = tid < (int)n ? list_s[tid] : 0;
            range(tid < (int)n ? key : ~0ull, key);
            const int shift = shift_of();
            clear();
            const int b = (int)((hi - key) >> shift);
            if (tid < (int)n) hit(b, key_value(key));
            __syncthreads();
            read_bins();
            scan_bins();
            find_border(ca, wa);
            if (found_bin < 0) return;
            if (tid < (int)n && b == found_bin) list_s[atomicAdd(&held_s, 1)] = key;
            narrow(shift);
            __syncthreads();
        }
        if (tid == 0) {
            found_key = ~0ull;
            found_kept = wa - above;
        }
        if (BOTH && tid < (int)n) list_w[tid] = weight(ch, key_value(list_s[tid]));
        __syncthreads();
        // each against each, eight threads to one
        u64 lowest_key = ~0ull, kept_mass = 0;
        for (int at0 = 0; at0 < (int)n; at0 += NT / 8) {
            const int at = min(at0 + tid / 8, (int)n - 1);
            const u64 key = list_s[at];
            unsigned before = 0;
            u64 mass = 0;
#pragma unroll 4
            for (int i = tid & 7; i < (int)n; i += 8) {
                const bool first = list_s[i] > key;
                before += first;
                if (BOTH) mass += first ? list_w[i] : 0;
            }
            before = eight_add(before);
            if (BOTH) mass = eight_add(mass);
            if ((tid & 7) == 0 && at0 + tid / 8 < (int)n && !dropped(ca + before, wa + mass, total)) {
                lowest_key = key < lowest_key ? key : lowest_key;
                if (BOTH) kept_mass += list_w[at];
            }
        }
        lowest_key = ~wave_most(~lowest_key);
        if (BOTH) kept_mass = wave_add(kept_mass);
        if (lane == 0) {
            atomicMin(&found_key, lowest_key);
            if (BOTH) atomicAdd(&found_kept, kept_mass);
        }
        __syncthreads();
        base = found_key;
        from = key_value(base);
        if (PARTS) {
            k_bin = bin;
            k_mass = found_kept;
        }
        __syncthreads();
    };
    if (cut_k) search(std::false_type{}, [&](unsigned before, u64, u64) { return before >= top_k; });
    if (cut_p) search(std::true_type{}, [&](unsigned, u64 mass, u64 all) { return mass > 0 && (double)mass >= top_p * (double)all; });
    if (lowest > from) {
        in_all = -1;
        from = lowest;
        base = order_key(lowest, 0x7fffffff);
    }
    // ---- the draw: the runs' masses, those of a wave each of the run of the token, that wave
    const bool every = base == 0;
    const auto kept = [&](float e, int i) { return every || e > from || (e == from && order_key(e, i) >= base); };
    const auto mass_of = [&](const Piece& v, int i) {
        float top = wide(v[0]);
#pragma unroll
        for (int c = 1; c < P; c++) top = fmaxf(top, wide(v[c]));
        u64 s = 0;
        if (top >= from)
#pragma unroll
            for (int c = 0; c < P; c++) {
                const u64 w = weight(ch, wide(v[c]));
                s += kept(wide(v[c]), i * P + c) ? w : 0;
            }
        return s;
    };
    if (counted) {  // by bins
        const int border = every ? BINS : bins.of(from);
        for (int run = wv; run < runs; run += W) {
            u64 s = 0;
            for (int b = lane; b < border; b += 64) s += run_mass(run, b);
            s = wave_add(s);
            if (lane == 0) runs_s[run] = s;
        }
        __syncthreads();
        if (!every) {  // the kept ones of the border's bin
            const auto add = [&](u64 key) {
                if (key >= base && key_index(key) < p.V) atomicAdd(&runs_s[key_index(key) / P / run_len], weight(ch, key_value(key)));
            };
            if (in_all >= 0) {
                if (tid < in_all) add(all_s[tid]);
            } else {
                each(from, [&](float e, int i) {
                    if (e >= from && bins.of(e) == border) add(order_key(e, i));
                });
            }
            __syncthreads();
        }
    } else {
        runs = W;
        run_len = (npiece + W - 1) / W;
        const int begin = min(wv * run_len, npiece), end = min(begin + run_len, npiece);
        u64 s = 0;
#pragma unroll 1
        for (int i = begin + lane; i < end; i += 64) s += mass_of(piece(i), i);
        s = wave_add(s);
        if (lane == 0) runs_s[wv] = s;
        __syncthreads();
    }
    const u64 upto_run = wave_scan(lane < runs ? runs_s[lane] : 0);
    total = lane_u64(upto_run, 63);
    const u64 target = mass_at(u, total);
    const int run = min(__popcll(__ballot(upto_run <= target)), runs - 1);
    u64 passed = run > 0 ? lane_u64(upto_run, run - 1) : 0;
    int begin = min(run * run_len, npiece), end = min(begin + run_len, npiece);
    const int len = (end - begin + W - 1) / W;
    begin = min(begin + wv * len, end);
    end = min(begin + len, end);
    u64 sum = 0, last_mass = 0;
    Piece last;  // this lane's last piece, and its mass
#pragma unroll 1
    for (int i = begin + lane; i < end; i += 64) {
        last = piece(i);
        last_mass = mass_of(last, i);
        sum += last_mass;
    }
    sum = wave_add(sum);
    if (lane == 0) red_s[0][wv] = sum;
    __syncthreads();
    const u64 upto_part = wave_scan(lane < W ? red_s[0][lane] : 0);
    if (wv > 0) passed += lane_u64(upto_part, wv - 1);
    if (passed <= target && target < passed + sum) {  // (one wave)
#pragma unroll 1
        for (int i0 = begin; i0 < end; i0 += 64) {
            const int i = i0 + lane;
            if (len > 64) {
                if (i < end) last = piece(i);
                last_mass = i < end ? mass_of(last, i) : 0;
            }
            const u64 upto = wave_scan(last_mass), all = lane_u64(upto, 63);
            if (passed + all > target) {
                u64 mass = passed + upto - last_mass;
                if (mass <= target && target < mass + last_mass) {  // (one lane)
                    int at = -1;
                    u64 taken = 0;
#pragma unroll
                    for (int c = 0; c < P; c++) {
                        const float e = wide(last[c]);
                        const u64 w = kept(e, i * P + c) ? weight(ch, e) : 0;
                        mass += w;
                        if (at < 0 && mass > target) {
                            at = i * P + c;
                            taken = w;
                        }
                    }
                    put(at, taken, total);
                }
                break;
            }
            passed += all;
        }
    }
}

// Rows whose whole distribution is drawn from, or (KEEP) what min_p leaves of it.
// A workgroup takes rows in turn: while it forms a row's weights it finds the next
// row's maximum, so that one row is on its way from memory while the exponentials
// of the one before, which come from the caches a second time, keep the VALU busy.
// (Past 1024 rows, 2048 of at most 8192 columns: up to there every row has a
// workgroup of its own, and its maximum and its weights follow one another.)
// A wave to each run of the row; the run that holds the token is formed again.
// us on MI355X, by sample_kernel / by this one: 1021 x 50001 fp32 88 / 80 (2.6 TB/s
// of one read; 58 with every row in the L2, where the operations of the weights take
// 31 to 35 and one read of the rows from memory 40), with min_p 0.05 76 /
// 67; bf16, 4096 x 32000 156 / 149, with min_p 119 / 112; 256 x 32000 27 / 13; 1 x
// 32000 16 / 12; 1024 x 4096 13 / 10.5; 16384 x 1000 81 / 79. Threads of a row, 256 /
// 512 / 1024: 1021 x 50001 fp32 90 / 79 / 82, 4096 x 32000 154 / 148 / 170, 1024 x 4096
// 10.4 / 14 / 25.
template <class E, int NT, bool KEEP>
__global__ __launch_bounds__(NT) void sample_draw_kernel(SampleParams p) {
    constexpr int P = SM_PIECE, W = NT / 64;
    constexpr int U = NT > 256 && sizeof(E) == 2 ? 2 : 1;  // pieces of a row that a thread forms at a time
    typedef E Piece __attribute__((ext_vector_type(P)));
    __shared__ u64 sums_s[2][W];
    __shared__ float best_s[W];
    __shared__ unsigned first_s[W];
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const int full = p.V / P, npiece = (p.V + P - 1) / P, len = (npiece + W - 1) / W;
    const int begin = min(wv * len, npiece), end = min(begin + len, npiece), whole = min(end, full);
    const int rest = end > full && begin <= full ? p.V - full * P : 0;  // columns behind the last whole piece, if they are this wave's
    const auto load = [](const E* x, int i) {
        Piece v;
        __builtin_memcpy(&v, x + (size_t)i * P, sizeof v);
        return v;
    };
    const auto top = [](float best, const Piece& v) {
#pragma unroll
        for (int c = 0; c < P; c++) best = __builtin_elementwise_maximum(best, wide(v[c]));  // (a NaN stays)
        return best;
    };
    // The maximum of a wave's runs to that of the row, a NaN where there is one.
    const auto put_best = [&](float best) {
        const bool bad = __any(best != best);
        best = wave_max(best);
        if (lane == 0) best_s[wv] = bad ? __builtin_nanf("") : best;
    };
    const auto get_best = [&]() {
        float best = best_s[0];
#pragma unroll
        for (int w = 1; w < W; w++) best = __builtin_elementwise_maximum(best, best_s[w]);
        return best;
    };
    const auto find_best = [&](const E* x) {  // of this wave's run
        float best = lane < rest ? wide(x[full * P + lane]) : -INFINITY;
        for (int i0 = begin + lane; i0 < whole; i0 += 64 * 4) {
            Piece v[4];
#pragma unroll
            for (int j = 0; j < 4; j++) v[j] = load(x, min(i0 + j * 64, whole - 1));
#pragma unroll
            for (int j = 0; j < 4; j++) best = top(best, v[j]);
        }
        return best;
    };
    long long r = blockIdx.x;
    const E* x = row_of<E>(p, r);
    put_best(find_best(x));
    __syncthreads();
    float best = get_best();
    Choice ch = choice_of(p, best, 1.);
    for (;;) {
        const long long next = r + gridDim.x;
        const bool more = next < p.rows;
        const E* xn = more ? row_of<E>(p, next) : x;
        const double T = p.temperatures ? (double)p.temperatures[r] : p.temperature;
        const double u = p.uniform64 ? p.uniform64[r] : (double)p.uniform[r];
        const bool none = !(fabsf(best) < INFINITY);
        __syncthreads();  // (all have read best_s)
        if (none || !(T > 0.)) {  // the first of the largest, a NaN before all
            unsigned at = 0xffffffffu;
            for (int c = tid; c < p.V; c += NT) {
                const float e = wide(x[c]);
                if (best != best ? e != e : e == best) at = min(at, (unsigned)c);
            }
            for (int d = 32; d > 0; d >>= 1) at = min(at, (unsigned)__shfl_xor((int)at, d));
            if (lane == 0) first_s[wv] = at;
            if (more) put_best(find_best(xn));
            __syncthreads();
            if (tid == 0) {
                for (int w = 1; w < W; w++) at = min(at, first_s[w]);
                p.ids[r] = at;
                p.logprob[r] = none ? __builtin_nanf("") : 0.f;
            }
        } else {
            set_choice(ch, best, T);
            float lowest = -INFINITY;
            if (KEEP) lowest = lowest_of(p.min_ps ? (double)p.min_ps[r] : p.min_p, ch.m, T);
            const auto weight_of = [&](float e) { return weight(ch, KEEP && e < lowest ? -INFINITY : e); };
            const auto sum_of = [&](const Piece& v) {
                u64 s = 0;
                if (!KEEP || top(-INFINITY, v) >= lowest)
#pragma unroll
                    for (int c = 0; c < P; c++) s += weight_of(wide(v[c]));
                return s;
            };
            u64 sum = lane < rest ? weight_of(wide(x[full * P + lane])) : 0;
            float nbest = more && lane < rest ? wide(xn[full * P + lane]) : -INFINITY;
            const auto pass = [&](auto with_next) {
                constexpr bool NEXT = decltype(with_next)::value;
                if (begin >= whole) return;
                Piece a[U], b[NEXT ? U : 1];
                const auto fetch = [&](int i0) {
#pragma unroll
                    for (int j = 0; j < U; j++) {
                        const int i = min(i0 + j * 64, whole - 1);
                        a[j] = load(x, i);
                        if (NEXT) b[j] = load(xn, i);
                    }
                };
                fetch(begin + lane);
#pragma unroll
                for (int j = 0; j < U; j++) {  // (else the compiler takes these loads for the loop's, and waits for each where it is used)
                    asm volatile("" : "+v"(a[j]));
                    if (NEXT) asm volatile("" : "+v"(b[j]));
                }
#pragma unroll 1
                for (int i0 = begin + lane; i0 - lane < whole; i0 += 64 * U) {
                    Piece now[U];
#pragma unroll
                    for (int j = 0; j < U; j++) {
                        now[j] = a[j];
                        if (NEXT) nbest = top(nbest, b[j]);
                    }
                    fetch(i0 + 64 * U);
#pragma unroll
                    for (int j = 0; j < U; j++) {
                        const u64 s = sum_of(now[j]);
                        sum += i0 + j * 64 < whole ? s : 0;
                    }
                }
            };
            more ? pass(std::true_type{}) : pass(std::false_type{});
            sum = wave_add(sum);
            if (lane == 0) sums_s[0][wv] = sum;
            if (more) put_best(nbest);
            __syncthreads();
            // of W sums the one that holds the target, and the mass before it (in every lane)
            u64 total, passed = 0, target = 0;
            const auto find = [&](const u64* sums) {
                const u64 mine = lane < W ? sums[lane] : 0, upto = wave_scan(mine);
                total = lane_u64(upto, 63);
                return upto;
            };
            const u64 runs = find(sums_s[0]), mass = total;
            target = mass_at(u, mass);
            const int run = min(__popcll(__ballot(runs <= target)), W - 1);
            if (run > 0) passed = lane_u64(runs, run - 1);
            // the run again, a wave to each part of it
            const auto piece_of = [&](int i) {
                Piece v;
                if (i < full)
                    v = load(x, i);
                else
#pragma unroll
                    for (int c = 0; c < P; c++) v[c] = i * P + c < p.V ? x[(size_t)i * P + c] : (E)-INFINITY;
                return v;
            };
            int from = min(run * len, npiece), to = min(from + len, npiece);
            const int share = (to - from + W - 1) / W;
            from = min(from + wv * share, to);
            to = min(from + share, to);
            u64 part = 0;
            Piece last;  // this lane's last piece, and its mass
            u64 last_mass = 0;
#pragma unroll 1
            for (int i = from + lane; i < to; i += 64) {
                last = piece_of(i);
                last_mass = sum_of(last);
                part += last_mass;
            }
            part = wave_add(part);
            if (lane == 0) sums_s[1][wv] = part;
            __syncthreads();
            const u64 parts = find(sums_s[1]);
            if (wv > 0) passed += lane_u64(parts, wv - 1);
            if (passed <= target && target < passed + part) {  // (one wave)
#pragma unroll 1
                for (int i0 = from; i0 < to; i0 += 64) {
                    const int i = i0 + lane;
                    if (share > 64) {
                        if (i < to) last = piece_of(i);
                        last_mass = i < to ? sum_of(last) : 0;
                    }
                    const u64 upto = wave_scan(last_mass), all = lane_u64(upto, 63);
                    if (passed + all > target) {
                        u64 before = passed + upto - last_mass;
                        if (before <= target && target < before + last_mass) {  // (one lane)
                            int at = -1;
                            u64 taken = 0;
#pragma unroll
                            for (int c = 0; c < P; c++) {
                                const u64 w = weight_of(wide(last[c]));
                                before += w;
                                if (at < 0 && before > target) {
                                    at = i * P + c;
                                    taken = w;
                                }
                            }
                            p.ids[r] = at;
                            p.logprob[r] = (float)log((double)taken / (double)mass);
                        }
                        break;
                    }
                    passed += all;
                }
            }
        }
        if (!more) return;
        best = get_best();
        r = next;
        x = xn;
    }
}

template <class E, int NT>
void launch_rows(SampleParams p, hipStream_t stream) {
    for (p.first = 0; p.first < p.rows; p.first += LOGPROBS_MAX_GRID) {
        const dim3 grid((unsigned)min(p.rows - p.first, (long long)LOGPROBS_MAX_GRID));
        hipLaunchKernelGGL((sample_kernel<E, NT, false>), grid, dim3(NT), 0, stream, p);
    }
}

// Workgroups of a compute unit that the rows of sample_draw_kernel are shared out to,
// of which (83 to 124 vector registers) two of 512 threads, or four or five of 256,
// are resident.
template <class E, int NT, bool KEEP>
void launch_draw(const SampleParams& p, int per_unit, hipStream_t stream) {
    const long long slots = 256ll * per_unit, turns = (p.rows + slots - 1) / slots;
    const dim3 grid((unsigned)((p.rows + turns - 1) / turns));
    hipLaunchKernelGGL((sample_draw_kernel<E, NT, KEEP>), grid, dim3(NT), 0, stream, p);
}

template <class E, int NT>
void launch_draws(const SampleParams& p, int per_unit, hipStream_t stream) {
    p.min_ps || p.min_p > 0. ? launch_draw<E, NT, true>(p, per_unit, stream) : launch_draw<E, NT, false>(p, per_unit, stream);
}

// Whether nothing but min_p cuts the rows.
bool draws(const SampleParams& p) { return !p.top_ks && !p.top_ps && (p.top_k <= 0 || p.top_k >= p.V) && !(p.top_p < 1.); }

// Parts of a row, 1 where it is not shared out: few wide rows, but for a top_k that
// one wave handles (of which a call with a top_k for each row may hold some). us
// on MI355X, bf16, one workgroup a row against parts of 4096 columns and more:
//   top_p 0.9: 16 rows of 32000 21 / 22, of 50001 32 / 24, of 131072 54 / 33; 64 rows 21 / 24, 32 / 27, 55 / 45; 128 22 / 27, 32 / 32, 57 / 57
//   whole distributions: 16 rows of 50001 19 / 16, of 131072 36 / 16; 64 rows 19 / 18, 37 / 28; 128 20 / 23, 37 / 38
//   the same with min_p 0.05: 16 rows 16 / 17, 22 / 21; 64 rows 17 / 21, 26 / 30
//   top_k 1000: 64 rows of 32000 25 / 24, of 50001 36 / 26, of 131072 66 / 36; top_k 50: 16 rows 11 / 18, 14 / 21, 18 / 25
// Parts of 8192 columns: top_p 0.95, 4 rows of 50001 30 for 27, as long at 131072.
int row_parts(const SampleParams& p) {
    if (p.V < (draws(p) ? 2 * SAMPLE_MIN_V : SAMPLE_MIN_V) || p.rows > SAMPLE_MAX_ROWS || p.rows <= 0 || (!p.top_ks && p.top_k > 0 && p.top_k <= SM_TOP)) return 1;
    return min(p.V / SAMPLE_PART_COLS, SAMPLE_PARTS);
}

template <class E>
void launch(SampleParams p, hipStream_t stream) {
    constexpr int N = RowVec<E>::N;
    const int parts = row_parts(p);
    if (parts > 1) {
        p.part = ((p.V + parts - 1) / parts + N - 1) / N * N;
        p.parts = (p.V + p.part - 1) / p.part;
        const size_t all = (size_t)p.rows * parts;
        p.part_mass = (u64*)((char*)p.stats + all * sizeof(PartStats));
        p.part_count = (unsigned*)(p.part_mass + all * SM_BINS);
        p.first = 0;
        const dim3 grid((unsigned)p.rows, (unsigned)p.parts);
        hipLaunchKernelGGL(sample_stats_kernel<E>, grid, dim3(256), 0, stream, p);
        hipLaunchKernelGGL(sample_bins_kernel<E>, grid, dim3(256), 0, stream, p);
        hipLaunchKernelGGL((sample_kernel<E, 1024, true>), dim3((unsigned)p.rows), dim3(1024), 0, stream, p);
    } else if (p.rows > 0 && draws(p)) {
        p.V <= 8192 ? launch_draws<E, 256>(p, 8, stream) : launch_draws<E, 512>(p, 4, stream);
    } else if (p.V <= 8192) {
        launch_rows<E, 256>(p, stream);
    } else if (p.rows <= 256) {
        launch_rows<E, 1024>(p, stream);
    } else {
        launch_rows<E, 512>(p, stream);
    }
    // Threads of a row by us on MI355X, bf16, 256 / 512 / 1024 threads:
    //   4096 columns, 1024 rows: top_k 50 15 / 18 / 32, top_p 0.9 18 / 24 / 47; 1 row: 11 / 9 / 9, 11 / 11 / 12
    //   16384, 1024 rows: 20 / 23 / 37, 40 / 36 / 62; 1 row: 14 / 11 / 10, 18 / 15 / 16
    //   32000, 1024 rows: 32 / 34 / 45, 72 / 60 / 82; 64 rows: 20 / 14 / 12, 37 / 23 / 21
    //   50001 fp32, 1021 rows: 65 / 69 / 71, 248 / 114 / 135
}

}  // namespace

// Bytes of the parts' statistics and bins, 0 where rows are not shared out.
size_t sample_workspace_bytes(long long rows, int V) {
    SampleParams p{};
    p.rows = rows;
    p.V = V;
    const int parts = row_parts(p);
    return parts > 1 ? (size_t)rows * parts * (sizeof(PartStats) + SM_BINS * 12) : 0;
}

void launch_sample(SampleParams p, int dtype, hipStream_t stream) {
    int bits = 0;  // of the number of columns
    while ((1ll << bits) < p.V) bits++;
    p.unit = (double)(1ull << (52 - (bits > 16 ? 62 - bits : 46)));
    if (dtype == 0)
        launch<bf16_t>(p, stream);
    else if (dtype == 1)
        launch<float>(p, stream);
    else
        launch<f16_t>(p, stream);
}

}  // namespace cyfa
