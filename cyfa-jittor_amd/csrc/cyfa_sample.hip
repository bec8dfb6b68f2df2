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
// A prefix is found by counting: elements, and their mass, by bins of their
// distance to the maximum; the bin in which the prefix ends gives its elements
// to a list, whose keys are binned again until few enough are left to rank each
// against each. A workgroup to a row, which stays in its registers where it fits.
#include <type_traits>

#include "cyfa_internal.h"
#include "cyfa_rows.h"

namespace cyfa {

namespace {

typedef unsigned long long u64;

constexpr double kLog2eD = 1.4426950408889634;
constexpr int SM_FEW = 128;  // elements ranked each against each

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

// The sum over the lanes, in every lane.
__device__ __forceinline__ u64 wave_add(u64 x) {
    for (int d = 32; d > 0; d >>= 1) x += __shfl_xor(x, d);
    return x;
}

// The sum over this lane and those below it.
__device__ __forceinline__ u64 wave_scan(u64 x) {
    for (int d = 1; d < 64; d <<= 1) {
        const u64 y = __shfl_up(x, d);
        if ((int)(threadIdx.x & 63) >= d) x += y;
    }
    return x;
}

// A row's settings.
struct Choice {
    float m;        // the maximum
    double c;       // log2 e / T
    double one;     // the integer of weight 1
};

__device__ __forceinline__ u64 weight(const Choice& ch, float x) {
    if (x == ch.m) return (u64)ch.one;  // (also where log2 e / T is infinite)
    const double t = ((double)x - (double)ch.m) * ch.c;
    if (!(t > -60.)) return 0;
    return (u64)(exp2(t) * ch.one + 0.5);
}

template <class E, int NT, int NV>
__global__ __launch_bounds__(NT) void sample_kernel(SampleParams p) {
    constexpr int N = RowVec<E>::N, W = NT / 64, TILE = NT * NV;
    __shared__ unsigned count_s[NT];
    __shared__ u64 mass_s[NT], list_s[NT], list_w[SM_FEW];
    __shared__ u64 red_s[2][W];
    __shared__ float redf_s[2][W];
    __shared__ unsigned redu_s[W];
    __shared__ u64 found_mass, found_key, found_total;
    __shared__ unsigned found_count, found_n;
    __shared__ int found_bin, held_s;
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const int full = p.V / N, nvec = (p.V + N - 1) / N;
    for (long long r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const E* x = static_cast<const E*>(p.x) + (r / p.inner) * p.outer_stride + (r % p.inner) * p.row_stride;
        const double T = p.temperatures ? (double)p.temperatures[r] : p.temperature;
        const double top_p = p.top_ps ? (double)p.top_ps[r] : p.top_p;
        const double min_p = p.min_ps ? (double)p.min_ps[r] : p.min_p;
        const long long top_k = p.top_ks ? p.top_ks[r] : p.top_k;
        typename RowVec<E>::type v[NV];
        float top[NV];  // the largest element of each
        bool bad = false;
        // A tile is shared out to the waves in whole runs of vectors, so that the
        // order (tile, wave, vector, lane, element) is that of the columns.
        int v0 = 0, per = 0;  // the tile's first vector, vectors of a thread in it
        const auto vec_of = [&](int j) { return v0 + (wv * per + j) * 64 + lane; };
        const auto load_tile = [&](int first) {
            v0 = first;
            per = min(NV, (nvec - first + NT - 1) / NT);
            if (full > 0)
#pragma unroll
                for (int j = 0; j < NV; j++)
                    if (j < per) v[j] = load_row(x + (size_t)min(vec_of(j), full - 1) * N);
#pragma unroll
            for (int j = 0; j < NV; j++) {
                top[j] = -INFINITY;
                const int i = vec_of(j);
                if (j >= per || i >= nvec) continue;
                if (i == full) {  // the columns past whole vectors
#pragma unroll
                    for (int c = 0; c < N; c++) v[j][c] = full * N + c < p.V ? x[full * N + c] : (E)-INFINITY;
                }
#pragma unroll
                for (int c = 0; c < N; c++) top[j] = fmaxf(top[j], (float)v[j][c]);
            }
        };
        const bool one_tile = nvec <= TILE;
        // f(element, column) of this thread's elements in vectors that reach ``from``
        const auto each_in_tile = [&](float from, auto&& f) {
#pragma unroll
            for (int j = 0; j < NV; j++) {
                const int i = vec_of(j);
                if (j < per && i < nvec && top[j] >= from)
#pragma unroll
                    for (int c = 0; c < N; c++) f((float)v[j][c], i * N + c);
            }
        };
        const auto each = [&](float from, auto&& f) {
            for (int first = 0; first < nvec; first += TILE) {
                if (!one_tile) load_tile(first);
                each_in_tile(from, f);
            }
        };
        // ---- the maximum, the least finite element, what no distribution holds
        float best = -INFINITY, least = INFINITY;
        for (int first = 0; first < nvec; first += TILE) {
            load_tile(first);
            each_in_tile(-INFINITY, [&](float e, int) {
                bad |= e != e;
                if (e > -INFINITY) least = fminf(least, e);
            });
#pragma unroll
            for (int j = 0; j < NV; j++) best = fmaxf(best, top[j]);
        }
        best = wave_max(best);
        least = -wave_max(-least);
        bad = __any(bad);
        __syncthreads();  // the row before is done with the shared arrays
        if (lane == 0) {
            redf_s[0][wv] = best;
            redf_s[1][wv] = least;
            redu_s[wv] = bad;
        }
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
                if (bad ? e != e : e == best) at = min(at, (unsigned)i);
            });
            for (int d = 32; d > 0; d >>= 1) at = min(at, (unsigned)__shfl_xor((int)at, d));
            __syncthreads();
            if (lane == 0) redu_s[wv] = at;
            __syncthreads();
            if (tid == 0) {
                for (int w = 1; w < W; w++) at = min(at, redu_s[w]);
                p.ids[r] = at;
                p.logprob[r] = none ? __builtin_nanf("") : 0.f;
            }
            continue;
        }
        Choice ch;
        ch.m = best;
        ch.c = kLog2eD / T;
        ch.one = p.one;
        u64 base = 0;          // kept so far: keys from here on
        float from = -INFINITY;  // its value
        // Lowers what is kept to the longest prefix that ``dropped`` (elements
        // before, mass before) does not end; MASS: it asks for the mass.
        const auto search = [&](auto with_mass, auto&& dropped) {
            constexpr bool MASS = decltype(with_mass)::value;
            // this thread's bin's count and mass to those before it; the totals
            const auto scan_bins = [&](unsigned& c, u64& w, unsigned& cb, u64& wb, u64& wt) {
                c = count_s[tid];
                w = MASS ? mass_s[tid] : 0;
                u64 cs = wave_scan(c), ws = MASS ? wave_scan(w) : 0;
                if (lane == 63) {
                    red_s[0][wv] = cs;
                    red_s[1][wv] = ws;
                }
                __syncthreads();
                u64 cbase = 0, wbase = 0;
                wt = 0;
                for (int i = 0; i < W; i++) {
                    if (i < wv) cbase += red_s[0][i];
                    if (MASS && i < wv) wbase += red_s[1][i];
                    if (MASS) wt += red_s[1][i];
                }
                cb = (unsigned)(cbase + cs - c);
                wb = wbase + ws - w;
            };
            const auto clear = [&]() {
                count_s[tid] = 0;
                if (MASS) mass_s[tid] = 0;
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
            // bins of the distance to the maximum, over the least element's or what the temperature leaves of it
            const float span = fminf(ch.m - fmaxf(least, from), 40.f * fmaxf((float)T, 1.f));
            const float inv = span > 0.f ? (float)NT / span : 0.f;
            const auto bin_of = [&](float e) { return (int)fminf((ch.m - e) * inv, (float)(NT - 1)); };
            clear();
            each(from, [&](float e, int i) {
                if (e >= from && order_key(e, i) >= base) hit(bin_of(e), e);
            });
            __syncthreads();
            unsigned c, cb;
            u64 w, wb, total;
            scan_bins(c, w, cb, wb, total);
            // the bin in which the prefix ends, known to all
            const auto find_border = [&](unsigned ca, u64 wa, u64 t) {
                if (c > 0 && !dropped(ca + cb, wa + wb, t) && dropped(ca + cb + c, wa + wb + w, t)) {
                    found_bin = tid;
                    found_count = ca + cb;
                    found_mass = wa + wb;
                    found_n = c;
                }
                __syncthreads();
            };
            find_border(0, 0, total);
            int bin = found_bin;
            if (bin < 0) return;  // nothing is dropped
            unsigned ca = found_count, n = found_n;
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
                const u64 d = (hi - lo) / NT;
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
                    u64 unused;
                    scan_bins(c, w, cb, wb, unused);
                    find_border(ca, wa, total);
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
            } else {
                each(from, [&](float e, int i) {
                    if (e >= from && bin_of(e) == bin) {
                        const u64 key = order_key(e, i);
                        if (key >= base) list_s[atomicAdd(&held_s, 1)] = key;
                    }
                });
            }
            __syncthreads();
            while (n > SM_FEW) {  // a thread to each of the list
                const u64 key = tid < (int)n ? list_s[tid] : 0;
                range(tid < (int)n ? key : ~0ull, key);
                const int shift = shift_of();
                clear();
                const int b = (int)((hi - key) >> shift);
                if (tid < (int)n) hit(b, key_value(key));
                __syncthreads();
                u64 unused;
                scan_bins(c, w, cb, wb, unused);
                find_border(ca, wa, total);
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
                for (int i = 0; i < (int)n; i++)
                    if (list_s[i] > key) {
                        before++;
                        if (MASS) mass += list_w[i];
                    }
                if (!dropped(before, mass, total)) atomicMin(&found_key, key);
            }
            __syncthreads();
            base = found_key;
            from = key_value(base);
            __syncthreads();
        };
        if (top_k > 0 && top_k < p.V) search(std::false_type{}, [&](unsigned before, u64, u64) { return before >= top_k; });
        if (top_p < 1.)
            search(std::true_type{}, [&](unsigned before, u64 mass, u64 total) { return before > 0 && (double)mass >= top_p * (double)total; });
        if (min_p > 0.) {
            // the least fp32 value that min_p keeps; the largest is always kept
            const double border = fmin((double)ch.m, (double)ch.m + T * log(min_p));
            float f = (float)border;
            if ((double)f < border) f = nextafterf(f, INFINITY);
            const u64 key = order_key(f, 0x7fffffff);
            if (key > base) {
                base = key;
                from = key_value(base);
            }
        }
        // ---- the draw
        const auto kept_weight = [&](float e, int i) { return e >= from && order_key(e, i) >= base ? weight(ch, e) : 0; };
        const auto wave_masses = [&]() {  // of the tile in registers: into red_s[0]
            u64 s = 0;
            each_in_tile(from, [&](float e, int i) { s += kept_weight(e, i); });
            s = wave_add(s);
            __syncthreads();
            if (lane == 0) red_s[0][wv] = s;
            __syncthreads();
        };
        u64 total = 0;
        for (int first = 0; first < nvec; first += TILE) {
            if (!one_tile) load_tile(first);
            wave_masses();
            for (int w = 0; w < W; w++) total += red_s[0][w];
        }
        const double u = p.uniform64 ? p.uniform64[r] : (double)p.uniform[r];
        u64 target = u > 0. ? (u64)fmin(u * (double)total, 0x1p63) : 0;
        if (target >= total) target = total - 1;
        u64 passed = 0;
        for (int first = 0; first < nvec; first += TILE) {
            if (!one_tile) {
                load_tile(first);
                wave_masses();
            }
            int at = -1;
            for (int w = 0; w < W && at < 0; w++) {
                if (passed + red_s[0][w] > target)
                    at = w;
                else
                    passed += red_s[0][w];
            }
            if (at < 0) continue;
            if (wv == at) {
                bool done = false;
#pragma unroll
                for (int j = 0; j < NV; j++) {
                    const int i = vec_of(j);
                    u64 s = 0;
                    if (!done && j < per && i < nvec && top[j] >= from)
#pragma unroll
                        for (int c = 0; c < N; c++) s += kept_weight((float)v[j][c], i * N + c);
                    const u64 sum = wave_scan(s), all = __shfl(sum, 63);
                    if (!done && passed + all > target) {
                        done = true;
                        const u64 mine = passed + sum - s;
                        if (mine <= target && target < mine + s) {
                            u64 run = mine;
                            bool taken = false;
#pragma unroll
                            for (int c = 0; c < N; c++) {
                                const u64 k = kept_weight((float)v[j][c], i * N + c);
                                run += k;
                                if (!taken && run > target) {
                                    taken = true;
                                    p.ids[r] = i * N + c;
                                    p.logprob[r] = (float)(log((double)k / (double)total));
                                }
                            }
                        }
                    } else if (!done) {
                        passed += all;
                    }
                }
            }
            break;
        }
    }
}

template <class E>
void launch(const SampleParams& p, hipStream_t stream) {
    const dim3 grid((unsigned)min(p.rows, (long long)LOGPROBS_MAX_GRID));
    hipLaunchKernelGGL((sample_kernel<E, 1024, 8>), grid, dim3(1024), 0, stream, p);
}

}  // namespace

void launch_sample(SampleParams p, int dtype, hipStream_t stream) {
    int bits = 0;  // of the number of columns
    while ((1ll << bits) < p.V) bits++;
    p.one = (double)(1ull << (bits > 16 ? 62 - bits : 46));
    if (dtype == 0)
        launch<bf16_t>(p, stream);
    else if (dtype == 1)
        launch<float>(p, stream);
    else
        launch<f16_t>(p, stream);
}

}  // namespace cyfa
