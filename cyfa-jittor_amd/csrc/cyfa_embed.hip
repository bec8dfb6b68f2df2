// cyfa_embed.hip -- the scaled embedding lookup out[i] = scale weight[ids[i]]
// and its gradient dweight[v] = scale sum_{i: ids[i] = v} dy[i].
//
// The gradient sorts the positions by id, each id's positions in their order,
// and adds each id's rows of dy in that order in fp32: no atomics on sums, so
// two backward passes give the same bits, and the result is rounded once.
#include "cyfa_internal.h"
#include "cyfa_rows.h"

namespace cyfa {

namespace {

template <class E>
__global__ __launch_bounds__(256) void embed_kernel(EmbedParams p) {
    constexpr int N = RowVec<E>::N;
    const int lane = threadIdx.x & 63;
    const int nvec = p.D / N, tail = p.D - nvec * N;
    const long long waves = (long long)gridDim.x * 4;
    for (long long i = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); i < p.n; i += waves) {
        const long long id = p.ids[i];
        const bool valid = id >= 0 && id < p.V;
        const E* w = static_cast<const E*>(p.weight) + (valid ? id : 0) * p.D;
        E* out = static_cast<E*>(p.out) + i * p.D;
        const float scale = valid ? p.scale : __builtin_nanf("");
        for (int v = lane; v < nvec; v += 64) {
            typename RowVec<E>::type e = load_row(w + v * N);
#pragma unroll
            for (int c = 0; c < N; c++) e[c] = (E)((float)e[c] * scale);
            store_row(out + v * N, e);
        }
        if (lane < tail) out[nvec * N + lane] = (E)((float)w[nvec * N + lane] * scale);
    }
}

// Positions sorted by id. A workgroup owns the ids [v0, v0 + range) and reads
// every id twice: it counts, wave by wave, how often each of its ids comes up
// and how many ids lie below v0, then each wave places its stretch of the
// positions behind those of the waves before it. Ids outside [0, V) and the
// padding id count nowhere.
//   offsets[v] .. offsets[v + 1]: where v's positions lie in order
constexpr int ES_NT = 1024, ES_WAVES = ES_NT / 64;
constexpr int ES_RANGE = 512;  // most ids of a workgroup: 35 KB of LDS

__global__ __launch_bounds__(ES_NT) void embed_sort_kernel(EmbedParams p, int range) {
    extern __shared__ int lds[];
    int* cursor = lds;                      // [ES_WAVES][range]
    int* start = lds + ES_WAVES * range;    // [range]
    int* misc = start + range;              // [2 * ES_WAVES]
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const long long v0 = (long long)blockIdx.x * range;
    const int mine = (int)min((long long)range, p.V - v0);
    const long long stretch = ((p.n + ES_NT - 1) / ES_NT) * 64;
    const long long first = wv * stretch, last = min(first + stretch, p.n);
    for (int i = tid; i < ES_WAVES * range; i += ES_NT) cursor[i] = 0;
    __syncthreads();
    int below = 0;
    for (long long i = first + lane; i < last; i += 64) {
        const long long id = p.ids[i];
        if (id < 0 || id >= p.V || id == p.padding) continue;
        if (id < v0) below++;
        else if (id < v0 + mine) atomicAdd(&cursor[wv * range + (int)(id - v0)], 1);
    }
    for (int d = 32; d > 0; d >>= 1) below += __shfl_xor(below, d);
    if (lane == 0) misc[wv] = below;
    __syncthreads();
    below = 0;
    for (int w = 0; w < ES_WAVES; w++) below += misc[w];
    // this id's positions of the waves before, and of the ids before (range <= ES_RANGE)
    int total = 0;
    if (tid < mine)
        for (int w = 0; w < ES_WAVES; w++) {
            const int c = cursor[w * range + tid];
            cursor[w * range + tid] = total;
            total += c;
        }
    int scan = total;
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(scan, d);
        if (lane >= d) scan += o;
    }
    if (lane == 63) misc[ES_WAVES + wv] = scan;
    __syncthreads();
    for (int w = 0; w < wv; w++) scan += misc[ES_WAVES + w];
    if (tid < mine) {
        start[tid] = below + scan - total;
        p.offsets[v0 + tid] = below + scan - total;
        if (v0 + tid == p.V - 1) p.offsets[p.V] = below + scan;
    }
    __syncthreads();
    for (long long i0 = first; i0 < last; i0 += 64) {
        const long long i = i0 + lane;
        int local = -1;
        if (i < last) {
            const long long id = p.ids[i];
            if (id >= v0 && id < v0 + mine && id != p.padding) local = (int)(id - v0);
        }
        uint64_t todo = __ballot(local >= 0);
        while (todo) {  // one id of these 64 positions after another
            const int id = __builtin_amdgcn_readlane(local, __builtin_ctzll(todo));
            const uint64_t same = __ballot(local == id);
            int* at = &cursor[wv * range + id];
            const int c = *at;
            if (local == id) p.order[start[id] + c + __popcll(same & ((1ull << lane) - 1))] = (int)i;
            *at = c + __popcll(same);  // (every lane, the same value)
            todo &= ~same;
        }
    }
}

// The sum of dy's rows of sorted positions [s, e), columns of one vector of this lane.
template <class E, int U>
__device__ __forceinline__ void add_rows(const EmbedParams& p, const E* dy, int s, int e, float (&acc)[RowVec<E>::N]) {
    constexpr int N = RowVec<E>::N;
    for (int i = s; i < e; i += U) {
        typename RowVec<E>::type v[U];
#pragma unroll
        for (int u = 0; u < U; u++) v[u] = load_row(dy + (long long)p.order[i + u < e ? i + u : e - 1] * p.D);
#pragma unroll
        for (int u = 0; u < U; u++)
            if (i + u < e)
#pragma unroll
                for (int c = 0; c < N; c++) acc[c] += (float)v[u][c];
    }
}

// Columns of a wave: 64 vectors; the last, ragged vector of a row is read and
// written ending at the row's end, so that it overlaps the one before it
// (the same values are stored twice), and rows below one vector go column by column.
template <class E>
__global__ __launch_bounds__(256) void embed_part_kernel(EmbedParams p) {
    constexpr int N = RowVec<E>::N;
    const int lane = threadIdx.x & 63;
    const int cols = (p.D + 64 * N - 1) / (64 * N), n = p.offsets[p.V];
    const long long units = (long long)(n / p.chunk) * cols, waves = (long long)gridDim.x * 4;
    for (long long unit = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); unit < units; unit += waves) {
        const long long c = unit / cols;
        const int s = (int)(c * p.chunk), e = s + p.chunk;
        const int d = (int)(unit % cols) * 64 * N + lane * N;
        if (p.ids[p.order[s]] != p.ids[p.order[e - 1]] || d >= p.D) continue;  // not one id's whole chunk
        float* out = p.part + c * p.D;
        if (p.D >= N) {
            const int at = min(d, p.D - N);
            float acc[N];
#pragma unroll
            for (int i = 0; i < N; i++) acc[i] = 0.f;
            add_rows<E, 8>(p, static_cast<const E*>(p.dy) + at, s, e, acc);
#pragma unroll
            for (int i = 0; i < N; i++) out[at + i] = acc[i];
        } else {
            for (int i = 0; i < p.D; i++) {
                float a = 0.f;
                for (int j = s; j < e; j++) a += (float)static_cast<const E*>(p.dy)[(long long)p.order[j] * p.D + i];
                out[i] = a;
            }
        }
    }
}

template <class E>
__global__ __launch_bounds__(256) void embed_grad_kernel(EmbedParams p) {
    constexpr int N = RowVec<E>::N;
    const int lane = threadIdx.x & 63;
    const int cols = (p.D + 64 * N - 1) / (64 * N);
    const long long units = p.V * cols, waves = (long long)gridDim.x * 4;
    for (long long unit = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); unit < units; unit += waves) {
        const long long v = unit / cols;
        const int d = (int)(unit % cols) * 64 * N + lane * N;
        const int s = p.offsets[v], e = p.offsets[v + 1];
        if (d >= p.D) continue;
        // whole chunks [c0, c1) of this id were added by embed_part_kernel
        const int c0 = (s + p.chunk - 1) / p.chunk, c1 = e / p.chunk;
        const bool parts = c0 < c1;
        E* out = static_cast<E*>(p.dweight) + v * p.D;
        if (p.D >= N) {
            const int at = min(d, p.D - N);
            const E* dy = static_cast<const E*>(p.dy) + at;
            float acc[N];
#pragma unroll
            for (int i = 0; i < N; i++) acc[i] = 0.f;
            add_rows<E, 8>(p, dy, s, parts ? c0 * p.chunk : e, acc);
            if (parts) {
                for (int c = c0; c < c1; c++)
#pragma unroll
                    for (int i = 0; i < N; i++) acc[i] += p.part[(long long)c * p.D + at + i];
                add_rows<E, 8>(p, dy, c1 * p.chunk, e, acc);
            }
            typename RowVec<E>::type o;
#pragma unroll
            for (int i = 0; i < N; i++) o[i] = (E)(acc[i] * p.scale);
            store_row(out + at, o);
        } else {
            for (int i = 0; i < p.D; i++) {
                float a = 0.f;
                const E* dy = static_cast<const E*>(p.dy) + i;
                for (int j = s; j < (parts ? c0 * p.chunk : e); j++) a += (float)dy[(long long)p.order[j] * p.D];
                if (parts) {
                    for (int c = c0; c < c1; c++) a += p.part[(long long)c * p.D + i];
                    for (int j = c1 * p.chunk; j < e; j++) a += (float)dy[(long long)p.order[j] * p.D];
                }
                out[i] = (E)(a * p.scale);
            }
        }
    }
}

constexpr int EMBED_CHUNK = 64;

template <class E>
void launch(EmbedParams p, bool grad, hipStream_t stream) {
    if (!grad) {
        hipLaunchKernelGGL(embed_kernel<E>, dim3((unsigned)min((p.n + 3) / 4, 1ll << 20)), dim3(256), 0, stream, p);
        return;
    }
    p.chunk = EMBED_CHUNK;
    const int range = (int)min((p.V + 255) / 256, (long long)ES_RANGE);
    hipLaunchKernelGGL(embed_sort_kernel, dim3((unsigned)((p.V + range - 1) / range)), dim3(ES_NT),
                       ((ES_WAVES + 1) * range + 2 * ES_WAVES) * sizeof(int), stream, p, range);
    const int cols = (p.D + 64 * RowVec<E>::N - 1) / (64 * RowVec<E>::N);
    const long long chunks = p.n / p.chunk;
    if (chunks)
        hipLaunchKernelGGL(embed_part_kernel<E>, dim3((unsigned)min((chunks * cols + 3) / 4, 1ll << 20)), dim3(256), 0, stream, p);
    hipLaunchKernelGGL(embed_grad_kernel<E>, dim3((unsigned)min((p.V * cols + 3) / 4, 1ll << 20)), dim3(256), 0, stream, p);
}

}  // namespace

// offsets int [V + 1], order int [n], part fp32 [n / chunk, D], each 256-byte aligned
size_t embed_workspace(EmbedParams* p, long long n, long long V, int D, void* base) {
    const auto up = [](size_t b) { return (b + 255) / 256 * 256; };
    const size_t offsets = up((size_t)(V + 1) * 4), order = up((size_t)n * 4);
    if (p) {
        p->offsets = (int*)base;
        p->order = (int*)((char*)base + offsets);
        p->part = (float*)((char*)base + offsets + order);
    }
    return offsets + order + up((size_t)(n / EMBED_CHUNK) * D * 4);
}

void launch_embed(const EmbedParams& p, int dtype, bool grad, hipStream_t stream) {
    if (dtype == 0)
        launch<bf16_t>(p, grad, stream);
    else if (dtype == 1)
        launch<float>(p, grad, stream);
    else
        launch<f16_t>(p, grad, stream);
}

}  // namespace cyfa
