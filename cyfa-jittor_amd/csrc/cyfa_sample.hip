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
// A workgroup to a row, which it keeps in LDS where it fits. A prefix is found by
// counting: the elements, or their mass, by bins of their distance to the
// maximum; the bin in which the prefix ends gives its elements to a list, whose
// keys are binned again until few enough are left to rank each against each. A
// top_k of at most 64, the usual one, needs no bins: a value that at least k
// elements reach and seldom many more is the k-th largest of the largest elements
// of 64 sets of threads, and the few that reach it are ranked, cut and drawn from
// by one wave.
#include <type_traits>

#include "cyfa_internal.h"
#include "cyfa_rows.h"

namespace cyfa {

namespace {

typedef unsigned long long u64;

constexpr double kLog2eD = 1.4426950408889634;
constexpr int SM_FEW = 128;   // elements ranked each against each by a thread each
constexpr int SM_TOP = 64;    // largest top_k that one wave handles

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

// An element in fp32. (Of a bf16 by its bits: the compiler takes the largest of
// converted bf16 as a bf16, with a rounding and another conversion for each.)
__device__ __forceinline__ float wide(float x) { return x; }
__device__ __forceinline__ float wide(f16_t x) { return (float)x; }
__device__ __forceinline__ float wide(bf16_t x) {
    return __builtin_bit_cast(float, (uint32_t)__builtin_bit_cast(uint16_t, x) << 16);
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

// Rows of up to ROW bytes in LDS; ROW = 0: of any length, read anew for each pass.
// Passes over the row take it in pieces of 8 bytes: of whole vectors the compiler
// holds eight exponentials' operands at a time, and spills them.
template <class E, int NT, int ROW>
__global__ __launch_bounds__(NT) void sample_kernel(SampleParams p) {
    typedef typename RowVec<E>::type Vec;
    constexpr int N = RowVec<E>::N, P = N / 2, W = NT / 64, BINS = NT > 512 ? 512 : NT;
    typedef E Piece __attribute__((ext_vector_type(P)));
    __shared__ Vec row_s[ROW ? ROW / 16 : 1];
    __shared__ u64 mass_s[BINS];
    __shared__ unsigned count_s[BINS];
    __shared__ u64 list_s[NT];
    __shared__ u64 list_w[SM_FEW];
    __shared__ u64 red_s[2][W];
    __shared__ float redf_s[2][W], thr_s;
    __shared__ unsigned redu_s[W];
    __shared__ u64 found_mass, found_key;
    __shared__ unsigned found_count, found_n;
    __shared__ int found_bin, held_s;
    float* const sets_s = reinterpret_cast<float*>(list_s);  // [W][64], until the list is used
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const int full = p.V / N, nvec = (p.V + N - 1) / N, npiece = (p.V + P - 1) / P;
    const long long r = p.first + blockIdx.x;
    const E* x = static_cast<const E*>(p.x) + (r / p.inner) * p.outer_stride + (r % p.inner) * p.row_stride;
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
        if (ROW) return reinterpret_cast<const Piece*>(row_s)[i];
        if ((i + 1) * P <= p.V) {
            __builtin_memcpy(&v, x + (size_t)i * P, 8);
        } else {
#pragma unroll
            for (int c = 0; c < P; c++) v[c] = i * P + c < p.V ? x[(size_t)i * P + c] : (E)-INFINITY;
        }
        return v;
    };
    const auto largest = [&](const Piece& v) {
        float top = wide(v[0]);
#pragma unroll
        for (int c = 1; c < P; c++) top = fmaxf(top, wide(v[c]));
        return top;
    };
    // f(element, column) of this thread's elements in pieces that reach ``from``
    const auto each = [&](float from, auto&& f) {
#pragma unroll 1
        for (int i = tid; i < npiece; i += NT) {
            const Piece v = piece(i);
            if (largest(v) >= from)
#pragma unroll
                for (int c = 0; c < P; c++) f(wide(v[c]), i * P + c);
        }
    };
    // ---- the maximum, the least finite element, what no distribution holds
    float best = -INFINITY, least = INFINITY;
    bool bad = false;
    {
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
                if (ROW) row_s[i] = v[j];
#pragma unroll
                for (int c = 0; c < N; c++) {
                    const float e = wide(v[j][c]);
                    bad |= e != e;
                    best = fmaxf(best, e);
                    least = fminf(least, e > -INFINITY ? e : INFINITY);
                }
            }
        }
    }
    const float own_best = best;
    best = wave_max(best);
    least = -wave_max(-least);
    bad = __any(bad);
    sets_s[wv * 64 + lane] = own_best;
    if (lane == 0) {
        redf_s[0][wv] = best;
        redf_s[1][wv] = least;
        redu_s[wv] = bad;
    }
    if (tid == 0) held_s = 0;
    __syncthreads();
    for (int w = 0; w < W; w++) {
        best = fmaxf(best, redf_s[0][w]);
        least = fminf(least, redf_s[1][w]);
        bad |= redu_s[w] != 0;
    }
    const bool none = bad || best == INFINITY || best == -INFINITY;
    if (none || !(T > 0.)) {  // the first of the largest, a NaN before all
        unsigned at = 0xffffffffu;
        each(-INFINITY, [&](float e, int i) {
            if (e == best && !bad) at = min(at, (unsigned)i);
        });
        if (bad)
            for (int i = tid; i < npiece; i += NT) {
                const Piece v = piece(i);
#pragma unroll
                for (int c = 0; c < P; c++)
                    if (wide(v[c]) != wide(v[c])) at = min(at, (unsigned)(i * P + c));
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
    Choice ch;
    ch.m = best;
    ch.c = fmax(fmin(kLog2eD / T, 1e300), 1e-300);  // (0 times it stays 0, -inf times it -inf)
    ch.least = -60. / ch.c;
    ch.unit = p.unit;
#pragma unroll
    for (int i = 0; i < SM_DEGREE; i++) {
        ch.k[i] = kExp2[i];
        asm("" : "+s"(ch.k[i]));  // (as literals each would be moved to the sum's registers before its product)
    }
    float lowest = -INFINITY;  // the least fp32 value that min_p keeps; the largest is always kept
    if (min_p > 0.) {
        const double border = fmin(ch.m, ch.m + T * log(min_p));
        lowest = (float)border;
        if ((double)lowest < border) lowest = nextafterf(lowest, INFINITY);
    }
    const auto mass_at = [&](u64 total) {  // what the running mass has to pass
        u64 target = u > 0. ? (u64)fmin(u * (double)total, 0x1p63) : 0;
        return target >= total ? total - 1 : target;
    };
    const auto put = [&](int i, u64 w, u64 total) {
        p.ids[r] = i;
        p.logprob[r] = (float)log((double)w / (double)total);
    };
    u64 base = 0;          // kept so far: keys from here on
    float from = -INFINITY;  // its value
    const bool cut_k = top_k > 0 && top_k < p.V, cut_p = top_p < 1.;
    if (cut_k && top_k <= SM_TOP) {
        const int k = (int)top_k;
        if (wv == 0) {
            float most = sets_s[lane];
            for (int w = 1; w < W; w++) most = fmaxf(most, sets_s[w * 64 + lane]);
            const float thr = kth_largest(most, k);
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
        if (n <= 2 * SM_FEW && n <= NT) {
            u64 key = 0;
            int rank = SM_TOP;
            if (tid < n) {
                key = list_s[tid];
                rank = 0;
#pragma unroll 8
                for (int i = 0; i < n; i++) rank += list_s[i] > key;
            }
            __syncthreads();
            if (rank < k) list_s[rank] = key;
            __syncthreads();
            if (wv == 0) {  // a lane to each of the k, in their order
                key = lane < k ? list_s[lane] : 0;
                const float e = key_value(key);
                u64 w = lane < k ? weight(ch, e) : 0;
                const u64 sum = wave_scan(w), all = lane_u64(sum, 63);
                const bool keep = lane == 0 || (lane < k && e >= lowest && !(cut_p && (double)(sum - w) >= top_p * (double)all));
                const int kept = __popcll(__ballot(keep));
                const u64 total = lane_u64(sum, kept - 1), target = mass_at(total);
                u64 upto = 0;  // the mass of the kept up to this one by index
                for (int i = 0; i < kept; i++) {
                    const u64 other = lane_u64(key, i), ow = lane_u64(w, i);
                    if ((uint32_t)other >= (uint32_t)key) upto += ow;
                }
                if (lane < kept && upto > target && upto - w <= target) put(key_index(key), w, total);
            }
            return;
        }
        from = thr;  // many equal elements: the bins tell
        base = order_key(thr, 0x7fffffff);
        __syncthreads();
    }
    // Lowers what is kept to the longest prefix that ``dropped`` (elements
    // before, mass before, all mass) does not end; MASS: it asks for the mass.
    const auto search = [&](auto with_mass, auto&& dropped) {
        constexpr bool MASS = decltype(with_mass)::value;
        // a bin's count and mass to those before it; the total mass
        unsigned c, cb;
        u64 w, wb, total;
        const auto scan_bins = [&]() {
            c = tid < BINS ? count_s[tid] : 0;
            w = MASS && tid < BINS ? mass_s[tid] : 0;
            const u64 cs = wave_scan(c), ws = MASS ? wave_scan(w) : 0;
            if (lane == 63) {
                red_s[0][wv] = cs;
                red_s[1][wv] = ws;
            }
            __syncthreads();
            u64 cbase = 0, wbase = 0, wt = 0;
            for (int i = 0; i < BINS / 64; i++) {
                if (i < wv) cbase += red_s[0][i];
                if (MASS && i < wv) wbase += red_s[1][i];
                if (MASS) wt += red_s[1][i];
            }
            cb = (unsigned)(cbase + cs - c);
            wb = wbase + ws - w;
            return wt;
        };
        const auto clear = [&]() {
            if (tid < BINS) {
                count_s[tid] = 0;
                if (MASS) mass_s[tid] = 0;
            }
            if (tid == 0) {
                held_s = 0;
                found_bin = -1;
            }
            __syncthreads();
        };
        const auto hit = [&](int b, float e) {
            atomicAdd(&count_s[b], 1u);
            if (MASS) atomicAdd(&mass_s[b], weight(ch, e));
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
        // bins of the distance to the maximum, over the least element's or what the temperature leaves of it
        const float m = (float)ch.m, span = fminf(m - fmaxf(least, from), 40.f * fmaxf((float)T, 1.f));
        const float inv = span > 0.f ? (float)BINS / span : 0.f;
        const auto bin_of = [&](float e) { return (int)fminf((m - e) * inv, (float)(BINS - 1)); };
        clear();
        if (MASS && base == 0) {  // (the count of the bin that matters is that of the list)
#pragma unroll 1
            for (int i = tid; i < npiece; i += NT) {
                const Piece v = piece(i);
#pragma unroll
                for (int c = 0; c < P; c++) atomicAdd(&mass_s[bin_of(wide(v[c]))], weight(ch, wide(v[c])));
            }
        } else {
            each(from, [&](float e, int i) {
                if (e >= from && order_key(e, i) >= base) {
                    if (MASS)
                        atomicAdd(&mass_s[bin_of(e)], weight(ch, e));
                    else
                        atomicAdd(&count_s[bin_of(e)], 1u);
                }
            });
        }
        __syncthreads();
        total = scan_bins();
        find_border(0, 0);
        const int bin = found_bin;
        if (bin < 0) return;  // nothing is dropped
        unsigned ca = found_count, n;
        u64 wa = found_mass;
        u64 lo = 0, hi = 0;  // the keys of the undecided, once they are known
        const auto range = [&](u64 low, u64 high) {
            for (int d = 32; d > 0; d >>= 1) {
                const u64 a = __shfl_xor(low, d), b = __shfl_xor(high, d);
                low = a < low ? a : low;
                high = b > high ? b : high;
            }
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
        // (no element of the bin lies more than its lower end and a bin for the roundings below the maximum)
        const float low = bin == BINS - 1 || !(inv > 0.f) ? from : fmaxf(from, m - (float)(bin + 2) / inv);
        each(low, [&](float e, int i) {
            if (e >= low && bin_of(e) == bin) {
                const u64 key = order_key(e, i);
                if (key >= base) {
                    const int at = atomicAdd(&held_s, 1);
                    if (at < NT) list_s[at] = key;
                }
            }
        });
        __syncthreads();
        n = (unsigned)held_s;
        if (n > NT) {  // too many for the list: bins of their keys
            u64 low = ~0ull, high = 0;
            each(from, [&](float e, int i) {
                if (e >= from && bin_of(e) == bin) {
                    const u64 key = order_key(e, i);
                    if (key >= base) {
                        low = key < low ? key : low;
                        high = key > high ? key : high;
                    }
                }
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
        while (n > SM_FEW) {  // a thread to each of the list
            const u64 key = tid < (int)n ? list_s[tid] : 0;
            range(tid < (int)n ? key : ~0ull, key);
            const int shift = shift_of();
            clear();
            const int b = (int)((hi - key) >> shift);
            if (tid < (int)n) hit(b, key_value(key));
            __syncthreads();
            scan_bins();
            find_border(ca, wa);
            if (found_bin < 0) return;
            if (tid < (int)n && b == found_bin) list_s[atomicAdd(&held_s, 1)] = key;
            narrow(shift);
            __syncthreads();
        }
        if (tid == 0) found_key = ~0ull;
        if (MASS && tid < (int)n) list_w[tid] = weight(ch, key_value(list_s[tid]));
        __syncthreads();
        if (tid < (int)n) {
            const u64 key = list_s[tid];
            unsigned before = ca;
            u64 mass = wa;
#pragma unroll 8
            for (int i = 0; i < (int)n; i++) {
                const bool first = list_s[i] > key;
                before += first;
                if (MASS) mass += first ? list_w[i] : 0;
            }
            if (!dropped(before, mass, total)) atomicMin(&found_key, key);
        }
        __syncthreads();
        base = found_key;
        from = key_value(base);
        __syncthreads();
    };
    if (cut_k) search(std::false_type{}, [&](unsigned before, u64, u64) { return before >= top_k; });
    if (cut_p) search(std::true_type{}, [&](unsigned, u64 mass, u64 total) { return mass > 0 && (double)mass >= top_p * (double)total; });
    if (lowest > from) {
        from = lowest;
        base = order_key(lowest, 0x7fffffff);
    }
    // ---- the draw: a wave to a run of the row's pieces
    const int run = (npiece + W - 1) / W, begin = min(wv * run, npiece), end = min(begin + run, npiece);
    const bool every = base == 0;
    const auto kept = [&](float e, int i) { return every || (e >= from && order_key(e, i) >= base); };
    const auto piece_weight = [&](const Piece& v, int i) {
        u64 s = 0;
        if (largest(v) >= from)
#pragma unroll
            for (int c = 0; c < P; c++) {
                const u64 w = weight(ch, wide(v[c]));
                s += kept(wide(v[c]), i * P + c) ? w : 0;
            }
        return s;
    };
    u64 sum = 0;
#pragma unroll 1
    for (int i = begin + lane; i < end; i += 64) sum += piece_weight(piece(i), i);
    sum = wave_add(sum);
    if (lane == 0) red_s[0][wv] = sum;
    __syncthreads();
    u64 total = 0, passed = 0;
    for (int w = 0; w < W; w++) {
        total += red_s[0][w];
        if (w < wv) passed += red_s[0][w];
    }
    const u64 target = mass_at(total);
    if (passed <= target && target < passed + sum) {  // (one wave)
#pragma unroll 1
        for (int i0 = begin; i0 < end; i0 += 64) {
            const int i = i0 + lane;
            const u64 s = i < end ? piece_weight(piece(i), i) : 0;
            const u64 upto = wave_scan(s), all = lane_u64(upto, 63);
            if (passed + all > target) {
                u64 mass = passed + upto - s;
                if (mass <= target && target < mass + s) {  // (one lane)
#pragma unroll 1
                    for (int c = 0; c < P; c++) {
                        const float e = wide(ROW ? reinterpret_cast<const E*>(row_s)[i * P + c] : x[(size_t)i * P + c]);
                        const u64 w = kept(e, i * P + c) ? weight(ch, e) : 0;
                        mass += w;
                        if (mass > target) {
                            put(i * P + c, w, total);
                            break;
                        }
                    }
                }
                break;
            }
            passed += all;
        }
    }
}

template <class E, int NT, int ROW>
void launch_rows(SampleParams p, hipStream_t stream) {
    for (p.first = 0; p.first < p.rows; p.first += LOGPROBS_MAX_GRID) {
        const dim3 grid((unsigned)min(p.rows - p.first, (long long)LOGPROBS_MAX_GRID));
        hipLaunchKernelGGL((sample_kernel<E, NT, ROW>), grid, dim3(NT), 0, stream, p);
    }
}

template <class E>
void launch(const SampleParams& p, hipStream_t stream) {
    const size_t bytes = ((size_t)p.V * sizeof(E) + 15) / 16 * 16;
    if (bytes <= 16384)
        launch_rows<E, 256, 16384>(p, stream);
    else if (bytes <= 65536)
        launch_rows<E, 1024, 65536>(p, stream);
    else if (bytes <= 131072)
        launch_rows<E, 1024, 131072>(p, stream);
    else
        launch_rows<E, 1024, 0>(p, stream);
}

}  // namespace

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
