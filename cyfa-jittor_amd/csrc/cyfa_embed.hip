// cyfa_embed.hip -- the scaled embedding lookup out[i] = scale weight[ids[i]]
// and its gradient dweight[v] = scale sum_{i: ids[i] = v} dy[i].
//
// The gradient sorts the positions by id, each id's positions in their order,
// and adds each id's rows of dy in fp32 by a rule that the ids alone fix (in that
// order, chunks of 32 by themselves; below): no atomics on sums, so two backward
// passes give the same bits, and the result is rounded once.
//
// us on MI355X for 16384 positions of natural frequencies, 1024 bf16 columns and
// 32000 ids: the lookup 10.4 (33.5 MB written, the 10 MB of different rows read),
// the gradient 37 in three launches for 33.5 MB read and 65.5 written: the sort
// 14, the shared ids' chunks 5, the rows 18 (5.5 TB/s). Adding the positions by
// atomics, zeroing and rounding an fp32 table took 200.
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

// Positions sorted by id, in the order of id mod G, then of id / G (G a power
// of two, a workgroup for each remainder: the most frequent ids, which most
// vocabularies number together, come to different workgroups). A workgroup reads
// every id: it counts, wave by wave, how often each of its ids comes up and how
// many ids belong to the workgroups before it, then each wave places its stretch
// of the positions behind those of the waves before it. Ids outside [0, V) count
// nowhere.
//   slot(v) = (v mod G) range + v / G;  offsets[slot] .. offsets[slot + 1]: where v's positions lie in order
// Every workgroup reading every id costs less than passes of a radix sort would
// in launches: on MI355X 300 positions take 6.5 us, 4096 8, 16384 11 (14 where one
// workgroup's ids are a fifteenth of them, 24 where all are one id: that
// workgroup's placing takes the time; with the ids of a wave's positions always
// told apart bit by bit 12, 16 and 27), 32768 19 (25, 47), 131072 of natural
// frequencies 81, nearly half of that gradient's 176: every workgroup reads them
// all. Up to 16384 positions stay in registers between counting and placing.
constexpr int ES_NT = 1024, ES_WAVES = ES_NT / 64, ES_U = 16;
constexpr int ES_FEW = 8;      // different ids of 64 positions that are matched one after another
constexpr int ES_RANGE = 512;  // most ids of a workgroup: 33 KB of LDS

__global__ __launch_bounds__(ES_NT) void embed_sort_kernel(EmbedParams p) {
    extern __shared__ int lds[];
    const int range = p.range, shift = p.shift;
    int* cursor = lds;                   // [ES_WAVES][range]: how many, then where the next goes
    int* misc = lds + ES_WAVES * range;  // [2 * ES_WAVES]
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const unsigned mine = blockIdx.x, groups = gridDim.x;
    const long long stretch = ((p.n + ES_NT - 1) / ES_NT) * 64;
    const long long first = wv * stretch, last = min(first + stretch, p.n);
    int* own = cursor + wv * range;
    for (int i = tid; i < ES_WAVES * range; i += ES_NT) cursor[i] = 0;
    __syncthreads();
    int below = 0;
    unsigned ids[ES_U];  // of 64 ES_U positions, ~0 where one counts nowhere
#pragma unroll 1
    for (int pass = 0; pass < 2; pass++) {
#pragma unroll 1
        for (long long i0 = first; i0 < last; i0 += 64 * ES_U) {
            const int left = (int)min(last - i0, (long long)64 * ES_U);  // at least 1
            if (pass == 0 || stretch > 64 * ES_U) {  // (else the ids are still here)
                const unsigned long long* from = reinterpret_cast<const unsigned long long*>(p.ids) + i0;
                unsigned long long id[ES_U];  // all loads in flight at once, those past the end of the last position
#pragma unroll
                for (int u = 0; u < ES_U; u++) id[u] = from[min(64 * u + lane, left - 1)];
#pragma unroll
                for (int u = 0; u < ES_U; u++) ids[u] = id[u] < (unsigned long long)p.V ? (unsigned)id[u] : ~0u;
                if (left < 64 * ES_U)
#pragma unroll
                    for (int u = 0; u < ES_U; u++) ids[u] = 64 * u + lane < left ? ids[u] : ~0u;
            }
#pragma unroll
            for (int u = 0; u < ES_U; u++) {
                if (64 * u >= left) break;
                const unsigned group = ids[u] & (groups - 1);
                const int id = (int)(ids[u] >> shift);  // (~0: past every range, in the last group)
                const bool here = group == mine && id < range;
                if (pass == 0) {
                    below += __popcll(__ballot(group < mine));
                    if (here) atomicAdd(&own[id], 1);
                    continue;
                }
                const uint64_t all = __ballot(here);
                if (!all) continue;
                uint64_t same = all, todo = range > 1 ? all : 0;  // same: the lanes with this lane's id
                for (int i = 0; todo && i < ES_FEW; i++) {        // one id after another, while they are few
                    const uint64_t m = __ballot(here && id == __builtin_amdgcn_readlane(id, __builtin_ctzll(todo)));
                    if ((m >> lane) & 1) same = m;
                    todo &= ~m;
                }
                if (todo) {  // many: bit by bit
                    same = all;
                    for (int b = 1; b < range; b <<= 1) {
                        const uint64_t bit = __ballot((id & b) != 0);
                        same &= (id & b) ? bit : ~bit;
                    }
                }
                // (LDS serves a wave's accesses in order: the next step reads what this one wrote)
                if (here) {
                    const int c = own[id], rank = __popcll(same & ((1ull << lane) - 1)), count = __popcll(same);
                    p.order[c + rank] = (int)(i0 + 64 * u + lane);
                    if (rank == count - 1) own[id] = c + count;
                }
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
            }
        }
        if (pass == 1) break;
        if (lane == 0) misc[wv] = below;
        __syncthreads();
        below = 0;
#pragma unroll
        for (int w = 0; w < ES_WAVES; w++) below += misc[w];
        // how many of this thread's id, and of the ids before it (range <= ES_NT)
        int c[ES_WAVES], total = 0;
        if (tid < range)
#pragma unroll
            for (int w = 0; w < ES_WAVES; w++) {
                c[w] = cursor[w * range + tid];
                total += c[w];
            }
        int scan = total;
        for (int d = 1; d < 64; d <<= 1) {
            const int o = __shfl_up(scan, d);
            if (lane >= d) scan += o;
        }
        if (lane == 63) misc[ES_WAVES + wv] = scan;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < ES_WAVES; w++) scan += w < wv ? misc[ES_WAVES + w] : 0;
        if (tid < range) {
            int at = below + scan - total;
            p.offsets[(long long)mine * range + tid] = at;
            if (mine == groups - 1 && tid == range - 1) p.offsets[(long long)groups * range] = below + scan;
#pragma unroll
            for (int w = 0; w < ES_WAVES; w++) {
                cursor[w * range + tid] = at;
                at += c[w];
            }
        }
        __syncthreads();
    }
}

// Adds dy's rows of the sorted positions [s, e) (the same in every lane) in
// order, the columns of one vector of this lane, EG_U rows' loads in flight (the
// 16384 positions above: the chunks 11.5 us with 4, 5.3 with 8 and 16; the rows,
// by a first form of their kernel, 24.8, 21.4 and 24.8).
constexpr int EG_U = 8;

template <class E>
__device__ __forceinline__ void add_rows(const EmbedParams& p, const E* dy, int s, int e, float (&acc)[RowVec<E>::N]) {
    constexpr int N = RowVec<E>::N;
    for (int i = s; i < e; i += EG_U) {
        typename RowVec<E>::type v[EG_U];
#pragma unroll
        for (int u = 0; u < EG_U; u++) v[u] = load_row(dy + (long long)p.order[min(i + u, e - 1)] * p.D);
#pragma unroll
        for (int u = 0; u < EG_U; u++)
            if (i + u < e)
#pragma unroll
                for (int c = 0; c < N; c++) acc[c] += (float)v[u][c];
    }
}

// An id with many positions is shared out: every EMBED_CHUNK sorted positions
// that all hold one id are added by a wave of embed_part_kernel, and
// embed_grad_kernel adds the rows before them, the chunks and the rows after them
// (chunks of 64 took 13.6 us for the 5 of 32: a wave's rows come eight at a time).
// The cuts are those of all sorted positions, so that an id's last bits also
// depend on how many positions the ids before it hold.
//
// Columns of a wave: 64 vectors; the last, ragged vector of a row is read and
// written ending at the row's end, so that it overlaps the one before it
// (the same values are stored twice), and rows below one vector go column by column.
constexpr int EMBED_CHUNK = 32;
constexpr int EMBED_FEW = 64;  // positions that a wave's lanes hold
constexpr size_t EMBED_STREAM = 128 << 20;
constexpr int EMBED_WAVES = 16384;  // 16 to a SIMD, where rows are taken in turn

template <class E>
__global__ __launch_bounds__(256) void embed_part_kernel(EmbedParams p) {
    constexpr int N = RowVec<E>::N;
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int chunks = p.offsets[(long long)p.range << p.shift] / EMBED_CHUNK;
    const int cols = (p.D + 64 * N - 1) / (64 * N), wave = blockIdx.x * 4 + wv, lines = gridDim.x * 4 / cols;
    const int d = wave % cols * 64 * N + lane * N;
    if (wave >= lines * cols) return;
    for (int c = wave / cols; c < chunks; c += lines) {
        const int s = c * EMBED_CHUNK, e = s + EMBED_CHUNK;
        const long long id = p.ids[p.order[s]];
        if (id != p.ids[p.order[e - 1]] || id == p.padding || d >= p.D) continue;  // not one id's whole chunk
        float* out = p.part + (long long)c * p.D;
        if (p.D >= N) {
            const int at = min(d, p.D - N);
            float acc[N];
#pragma unroll
            for (int i = 0; i < N; i++) acc[i] = 0.f;
            add_rows<E>(p, static_cast<const E*>(p.dy) + at, s, e, acc);
            __builtin_memcpy(out + at, acc, sizeof(acc));
        } else {
            for (int i = 0; i < p.D; i++) {
                float a = 0.f;
                for (int j = s; j < e; j++) a += (float)static_cast<const E*>(p.dy)[(long long)p.order[j] * p.D + i];
                out[i] = a;
            }
        }
    }
}

// Columns [d, d + N) of the gradient's row v from its sorted positions [s, e).
// STREAM: its lines, each written whole by one wave, go past the caches.
template <class E, bool STREAM>
__device__ __forceinline__ void embed_row(const EmbedParams& p, int v, int d, int s, int e) {
    constexpr int N = RowVec<E>::N;
    if (v == p.padding) e = s;
    const int c0 = (s + EMBED_CHUNK - 1) / EMBED_CHUNK, c1 = e / EMBED_CHUNK;
    const bool parts = c0 < c1;  // whole chunks [c0, c1) of this id
    E* out = static_cast<E*>(p.dweight) + (long long)v * p.D;
    if (p.D >= N) {
        const int at = min(d, p.D - N);
        const E* dy = static_cast<const E*>(p.dy) + at;
        float acc[N];
#pragma unroll
        for (int i = 0; i < N; i++) acc[i] = 0.f;
        add_rows<E>(p, dy, s, parts ? c0 * EMBED_CHUNK : e, acc);
        if (parts) {
            for (int c = c0; c < c1; c += EG_U) {
                float part[EG_U][N];
#pragma unroll
                for (int u = 0; u < EG_U; u++)
                    __builtin_memcpy(part[u], p.part + (long long)min(c + u, c1 - 1) * p.D + at, sizeof(part[u]));
#pragma unroll
                for (int u = 0; u < EG_U; u++)
                    if (c + u < c1)
#pragma unroll
                        for (int i = 0; i < N; i++) acc[i] += part[u][i];
            }
            add_rows<E>(p, dy, c1 * EMBED_CHUNK, e, acc);
        }
        typename RowVec<E>::type o;
#pragma unroll
        for (int i = 0; i < N; i++) o[i] = (E)(acc[i] * p.scale);
        store_row<E, STREAM>(out + at, o);
    } else {
        for (int i = 0; i < p.D; i++) {
            float a = 0.f;
            const E* dy = static_cast<const E*>(p.dy) + i;
            for (int j = s; j < (parts ? c0 * EMBED_CHUNK : e); j++) a += (float)dy[(long long)p.order[j] * p.D];
            if (parts) {
                for (int c = c0; c < c1; c++) a += p.part[(long long)c * p.D + i];
                for (int j = c1 * EMBED_CHUNK; j < e; j++) a += (float)dy[(long long)p.order[j] * p.D];
            }
            out[i] = (E)(a * p.scale);
        }
    }
}

__device__ __forceinline__ const int* embed_slot(const EmbedParams& p, int v) {
    return p.offsets + ((long long)(v & ((1 << p.shift) - 1)) * p.range + (v >> p.shift));
}

// A wave for one piece of 64 vectors of a row, the waves along the rows and then
// row after row, each with rows that lie the grid apart, or (ONCE) one row each.
template <class E, bool ONCE, bool STREAM>
__global__ __launch_bounds__(256) void embed_grad_kernel(EmbedParams p) {
    constexpr int N = RowVec<E>::N;
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int cols = (p.D + 64 * N - 1) / (64 * N), V = (int)p.V;
    const long long wave = (long long)blockIdx.x * 4 + wv;
    int v = (int)(wave / cols);
    const int d = (int)(wave % cols) * 64 * N + lane * N, lines = gridDim.x * 4 / cols;
    if (v >= (ONCE ? V : min(V, lines))) return;
    int s = embed_slot(p, v)[0], e = embed_slot(p, v)[1];
    if (ONCE) {
        if (d < p.D) embed_row<E, STREAM>(p, v, d, s, e);
        return;
    }
    while (v < V) {  // (the next row's positions are on their way while this one is added)
        const int next = min(v + lines, V - 1);
        const int next_s = embed_slot(p, next)[0], next_e = embed_slot(p, next)[1];
        if (d < p.D) embed_row<E, STREAM>(p, v, d, s, e);
        v += lines;
        s = next_s;
        e = next_e;
    }
}

// The gradient from at most EMBED_FEW positions, unsorted, in one launch: a wave
// holds every id, one in each lane, and finds the positions of a row by comparing.
// us on MI355X so and sorted: 64 positions, 32000 x 1024 bf16 10.6 and 21 (all of one
// id 14 and 21.5), 512 x 256 2.6 and 12.5; 30, 131072 x 1001 35 and 42.
template <class E, bool STREAM>
__global__ __launch_bounds__(256) void embed_few_kernel(EmbedParams p) {
    constexpr int N = RowVec<E>::N;
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = (int)p.n;
    const int cols = (p.D + 64 * N - 1) / (64 * N), V = (int)p.V;
    const int wave = blockIdx.x * 4 + wv, lines = gridDim.x * 4 / cols, d = wave % cols * 64 * N + lane * N;
    if (wave >= lines * cols) return;
    const long long id = lane < n ? p.ids[lane] : -1;
    for (int v = wave / cols; v < V; v += lines) {
        uint64_t at = __ballot(id == v && v != p.padding);  // the row's positions
        if (d >= p.D) continue;
        E* out = static_cast<E*>(p.dweight) + (long long)v * p.D;
        if (p.D >= N) {
            const int col = min(d, p.D - N);
            float acc[N];
#pragma unroll
            for (int i = 0; i < N; i++) acc[i] = 0.f;
            for (int left = __popcll(at); left > 0; left -= EG_U) {
                typename RowVec<E>::type y[EG_U];
#pragma unroll
                for (int u = 0; u < EG_U; u++) {  // (the last position again where there are fewer)
                    y[u] = load_row(static_cast<const E*>(p.dy) + (long long)__builtin_ctzll(at) * p.D + col);
                    if (u + 1 < left) at &= at - 1;
                }
#pragma unroll
                for (int u = 0; u < EG_U; u++)
                    if (u < left)
#pragma unroll
                        for (int i = 0; i < N; i++) acc[i] += (float)y[u][i];
            }
            typename RowVec<E>::type o;
#pragma unroll
            for (int i = 0; i < N; i++) o[i] = (E)(acc[i] * p.scale);
            store_row<E, STREAM>(out + col, o);
        } else {
            for (int i = 0; i < p.D; i++) {
                float a = 0.f;
                for (uint64_t m = at; m; m &= m - 1) a += (float)static_cast<const E*>(p.dy)[(long long)__builtin_ctzll(m) * p.D + i];
                out[i] = (E)(a * p.scale);
            }
        }
    }
}

template <class E>
void launch(const EmbedParams& p, bool grad, hipStream_t stream) {
    if (!grad) {
        hipLaunchKernelGGL(embed_kernel<E>, dim3((unsigned)min((p.n + 3) / 4, 1ll << 20)), dim3(256), 0, stream, p);
        return;
    }
    const int cols = (p.D + 64 * RowVec<E>::N - 1) / (64 * RowVec<E>::N);  // pieces of 64 vectors of a row
    const auto grid = [&](long long rows, long long most) {
        return dim3((unsigned)((min(rows * cols, max(most, (long long)cols)) + 3) / 4));
    };
    // A gradient in whole lines that the last-level cache cannot keep is written in
    // the order of memory, a wave for every piece, past the caches (fewer than 2^32
    // threads); others by waves in turn. us on MI355X so, by a wave for every piece
    // through the caches, and in turn: 86274 x 2048 fp32 with 2 positions 102, 119,
    // 154 (a fill of it takes 103); 32000 x 2048 fp32 with 2999 42, 50, 54; 32000 x 1024
    // bf16 with 16384 (66 MB) 17.6, 19.7, 18; 32000 x 1536 fp16 with 9 18.5, 20, 16;
    // rows off the lines, 131072 x 1001 bf16 with 4000 52, 57, 47.
    const bool lines = p.D * sizeof(E) % 128 == 0 && (uintptr_t)p.dweight % 128 == 0;
    const bool streamed = (size_t)p.V * p.D * sizeof(E) >= EMBED_STREAM && lines && p.V * cols < 1 << 26;
    const dim3 rows = grid(p.V, streamed ? p.V * cols : EMBED_WAVES);
    if (p.n <= EMBED_FEW) {
        if (streamed)
            hipLaunchKernelGGL((embed_few_kernel<E, true>), rows, dim3(256), 0, stream, p);
        else
            hipLaunchKernelGGL((embed_few_kernel<E, false>), rows, dim3(256), 0, stream, p);
        return;
    }
    hipLaunchKernelGGL(embed_sort_kernel, dim3(1u << p.shift), dim3(ES_NT), (ES_WAVES * p.range + 2 * ES_WAVES) * sizeof(int),
                       stream, p);
    hipLaunchKernelGGL(embed_part_kernel<E>, grid(p.n / EMBED_CHUNK, EMBED_WAVES), dim3(256), 0, stream, p);
    if (streamed)
        hipLaunchKernelGGL((embed_grad_kernel<E, true, true>), rows, dim3(256), 0, stream, p);
    else
        hipLaunchKernelGGL((embed_grad_kernel<E, false, false>), rows, dim3(256), 0, stream, p);
}

}  // namespace

// offsets int [slots + 1], order int [n], part fp32 [n / chunk, D], each 256-byte aligned
// (nothing for the few positions that are not sorted)
size_t embed_workspace(EmbedParams* p, long long n, long long V, int D, void* base) {
    if (n <= EMBED_FEW) return 0;
    const auto up = [](size_t b) { return (b + 255) / 256 * 256; };
    int shift = 8;  // a workgroup of the sort for each of 256 compute units, more for many ids
    while ((V + (1ll << shift) - 1) >> shift > ES_RANGE) shift++;
    const int range = (int)((V + (1ll << shift) - 1) >> shift);
    const size_t offsets = up((((size_t)range << shift) + 1) * 4), order = up((size_t)n * 4);
    if (p) {
        p->shift = shift;
        p->range = range;
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
