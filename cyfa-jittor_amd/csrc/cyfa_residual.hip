// cyfa_residual.hip -- the join between two blocks: a block's output norm and
// gate, the scaled residual add and the next block's norm, and the gradients.
// For a row x, y [, gate] of D columns:
//   n = y r1, r1 = (mean y^2 + eps)^-1/2          (with post; else u = y)
//   u = n post,  b = u [sigmoid(gate)]
//   s = x + scale b
//   h = s r2 weight, r2 = (mean s^2 + eps)^-1/2   (of s before its rounding)
// and from the cotangents ds, dh of s and h, with m = s r2 and e = dh weight:
//   dx      = ds + r2 (e - m mean(e m))
//   db      = scale dx,  du = db [sigmoid(gate)],  dgate = db u sigmoid(gate) (1 - sigmoid(gate))
//   dy      = r1 (du post - n mean(du post n))    (du without post)
//   dweight = sum over rows of dh m,  dpost = sum over rows of du n
// mean(du post n) follows from sums over ds, e and m, so that one reduction
// over the row serves both means. Everything in fp32; s, m and h are formed from
// x and y again in the gradient, so that its sums over rows (dweight, dpost, in
// fp32) do not see the rounding of s.
//
// Bound by the memory's rate. us on MI355X: 16384 x 1024 bf16 rows with output
// norm and gate forward 28 (168 MB, 6.0 TB/s), the gradient 47.5 (268 MB, 5.6 TB/s)
// with 4 for the sums over workgroups; 2999 x 1536 fp32 plain rows 13.5 and 20 + 4
// (5.5 TB/s both); the plain chains of fp32 operations took 1040 and 155 for both
// ways. 64 rows take 3.5 us, a launch's latency. Stores past the caches shorten
// these launches by a tenth (28 -> 27, 47.5 -> 44) and the products and adds that
// read the results after them grow by as much: with those, 116 us and 116 us the
// gradient of 16384 x 1024, 268 and 274 of 16384 x 2048. They stay in the caches.
#include "cyfa_internal.h"
#include "cyfa_rows.h"

namespace cyfa {

namespace {

// Lane t of the T threads of a row holds the vectors t + j T (j < J) of VN
// elements. The last vector of a row of no whole number of vectors is read
// ending at the row's end, and its elements that the vector before it holds
// count as zero and are not stored; so are all elements of vectors past it.
template <class E, int VN, int T, int J>
struct Row {
    typedef E vec __attribute__((ext_vector_type(VN)));

    int at[J], skip[J];  // column of the vector's first element; elements that do not count
    bool full;           // all count, in every thread

    __device__ __forceinline__ Row(int D, int t) : full(D == J * T * VN) {
#pragma unroll
        for (int j = 0; j < J; j++) {
            const int c = (t + j * T) * VN;
            at[j] = min(c, D - VN);
            skip[j] = min(c - at[j], VN);
        }
    }

    template <class X>
    __device__ __forceinline__ void load(const X* row, float (&v)[J][VN]) const {
#pragma unroll
        for (int j = 0; j < J; j++) {
            typedef X xvec __attribute__((ext_vector_type(VN)));
            xvec e;
            __builtin_memcpy(&e, row + at[j], sizeof(e));
#pragma unroll
            for (int c = 0; c < VN; c++) v[j][c] = (float)e[c];
        }
        mask(v);
    }

    __device__ __forceinline__ void mask(float (&v)[J][VN]) const {
        if (full) return;
#pragma unroll
        for (int j = 0; j < J; j++)
#pragma unroll
            for (int c = 0; c < VN; c++) v[j][c] = c < skip[j] ? 0.f : v[j][c];
    }

    // The same in two steps: the vectors, in flight while other work runs, then their elements.
    __device__ __forceinline__ void fetch(const void* rows, long long offset, vec (&v)[J]) const {
#pragma unroll
        for (int j = 0; j < J; j++) __builtin_memcpy(&v[j], static_cast<const E*>(rows) + offset + at[j], sizeof(vec));
    }

    __device__ __forceinline__ void widen(const vec (&v)[J], float (&f)[J][VN]) const {
#pragma unroll
        for (int j = 0; j < J; j++)
#pragma unroll
            for (int c = 0; c < VN; c++) f[j][c] = (float)v[j][c];
        mask(f);
    }

    template <class X>
    __device__ __forceinline__ void store(X* row, const float (&v)[J][VN]) const {
#pragma unroll
        for (int j = 0; j < J; j++) {
            typedef X xvec __attribute__((ext_vector_type(VN)));
            if (skip[j] == 0) {
                xvec e;
#pragma unroll
                for (int c = 0; c < VN; c++) e[c] = (X)v[j][c];
                __builtin_memcpy(row + at[j], &e, sizeof(e));
            } else if (skip[j] < VN) {
#pragma unroll
                for (int c = 1; c < VN; c++)
                    if (c >= skip[j]) row[at[j] + c] = (X)v[j][c];
            }
        }
    }
};

// Sums over the T threads of a row, in a fixed order, in every thread of it.
template <int T, int K>
__device__ __forceinline__ void row_sums(float (&v)[K], float (*red)[K]) {
#pragma unroll
    for (int k = 0; k < K; k++) v[k] = wave_sum(v[k]);
    if (T == 64) return;
    const int wv = threadIdx.x >> 6;
    __syncthreads();  // red is free
    if ((threadIdx.x & 63) == 0)
#pragma unroll
        for (int k = 0; k < K; k++) red[wv][k] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; k++) {
        v[k] = 0.f;
#pragma unroll
        for (int w = 0; w < T / 64; w += 4) v[k] += (red[w][k] + red[w + 1][k]) + (red[w + 2][k] + red[w + 3][k]);
    }
}

// Threads of a workgroup whose rows take T each.
constexpr int block_of(int T) { return T > 256 ? T : 256; }

template <class E, int VN, int T, int J>
__global__ __launch_bounds__(block_of(T)) void residual_norm_kernel(ResidualParams p) {
    constexpr int RW = block_of(T) / T;
    __shared__ float red[block_of(T) / 64][1];
    const Row<E, VN, T, J> cols(p.D, threadIdx.x % T);
    for (long long r = (long long)blockIdx.x * RW + threadIdx.x / T; r < p.rows; r += (long long)gridDim.x * RW) {
        const long long o = r * p.D;
        float s[J][VN], b[J][VN];
        cols.load(static_cast<const E*>(p.x) + o, s);
        cols.load(static_cast<const E*>(p.y) + o, b);
        float ss[1] = {0.f};
        if (p.post) {
            float w[J][VN];
            cols.load(p.post, w);
#pragma unroll
            for (int j = 0; j < J; j++)
#pragma unroll
                for (int c = 0; c < VN; c++) ss[0] = fmaf(b[j][c], b[j][c], ss[0]);
            row_sums<T>(ss, red);
            const float r1 = rsqrtf(ss[0] * p.inverse_d + p.eps);
            if (p.stats && threadIdx.x % T == 0) p.stats[2 * r] = r1;
#pragma unroll
            for (int j = 0; j < J; j++)
#pragma unroll
                for (int c = 0; c < VN; c++) b[j][c] *= r1 * w[j][c];
        }
        if (p.gate) {
            float g[J][VN];
            cols.load(static_cast<const E*>(p.gate) + o, g);
#pragma unroll
            for (int j = 0; j < J; j++)
#pragma unroll
                for (int c = 0; c < VN; c++) b[j][c] *= sigmoidf(g[j][c]);
        }
        ss[0] = 0.f;
#pragma unroll
        for (int j = 0; j < J; j++)
#pragma unroll
            for (int c = 0; c < VN; c++) {
                s[j][c] = fmaf(p.scale, b[j][c], s[j][c]);
                ss[0] = fmaf(s[j][c], s[j][c], ss[0]);
            }
        cols.store(static_cast<E*>(p.s) + o, s);
        row_sums<T>(ss, red);
        const float r2 = rsqrtf(ss[0] * p.inverse_d + p.eps);
        if (p.stats && threadIdx.x % T == 0) p.stats[2 * r + 1] = r2;
        cols.load(p.weight, b);
#pragma unroll
        for (int j = 0; j < J; j++)
#pragma unroll
            for (int c = 0; c < VN; c++) s[j][c] *= r2 * b[j][c];
        cols.store(static_cast<E*>(p.h) + o, s);
    }
}

// Workgroups of p.rows_wg rows; each leaves its sums for dweight and dpost in
// part [workgroup][2][D], which residual_sum_kernel adds (one workgroup alone, as
// the gradients). The weights stay in LDS (rows of a wave) or in registers; two
// waves per SIMD have to fit, so that one's loads cover the other's arithmetic.
template <class E, int VN, int T, int J, bool POST, bool GATE>
__global__ __launch_bounds__(block_of(T), 2) void residual_grad_kernel(ResidualParams p) {
    constexpr int RW = block_of(T) / T, C = J * T * VN;
    __shared__ float red[block_of(T) / 64][3];
    __shared__ __align__(16) float sums[RW > 1 ? RW : 1][RW > 1 ? C : 1];
    __shared__ __align__(16) float weights[2][RW > 1 ? C : 1];
    const int t = threadIdx.x % T;
    const Row<E, VN, T, J> cols(p.D, t);
    float dw[J][VN], dp[J][VN], kept[2][J][VN];
#pragma unroll
    for (int j = 0; j < J; j++)
#pragma unroll
        for (int c = 0; c < VN; c++) dw[j][c] = dp[j][c] = 0.f;
    cols.load(p.weight, kept[0]);
    if (POST) cols.load(p.post, kept[1]);
    if (RW > 1) {
        if (threadIdx.x < T)
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int j = 0; j < J; j++)
#pragma unroll
                    for (int c = 0; c < VN; c++) weights[i][(t + j * T) * VN + c] = kept[i][j][c];
        __syncthreads();
    }
    const auto weight = [&](int which, float (&w)[J][VN]) {
#pragma unroll
        for (int j = 0; j < J; j++)
#pragma unroll
            for (int c = 0; c < VN; c++) w[j][c] = RW > 1 ? weights[which][(t + j * T) * VN + c] : kept[which][j][c];
    };
    const long long end = min((long long)(blockIdx.x + 1) * p.rows_wg, p.rows);
    const long long first = (long long)blockIdx.x * p.rows_wg + threadIdx.x / T;
    // the next row's operands are in flight while this one's are worked on
    typename Row<E, VN, T, J>::vec xv[J], yv[J], gv[J], ev[J], dv[J];
    float r1n, r2n;
    const auto fetch = [&](long long r) {
        const long long o = r * p.D;
        cols.fetch(p.x, o, xv);
        cols.fetch(p.y, o, yv);
        if (GATE) cols.fetch(p.gate, o, gv);
        if (p.d_h) cols.fetch(p.d_h, o, ev);
        if (p.d_s) cols.fetch(p.d_s, o, dv);
        r1n = p.stats[2 * r];
        r2n = p.stats[2 * r + 1];
    };
    fetch(min(first, end - 1));
    for (long long r = first; r < end; r += RW) {
        const long long o = r * p.D;
        float s[J][VN], y[J][VN], g[J][VN], e[J][VN], d[J][VN];
        cols.widen(xv, s);
        cols.widen(yv, y);
        if (GATE) cols.widen(gv, g);
        if (p.d_h) cols.widen(ev, e);
        if (p.d_s) cols.widen(dv, d);
        const float r1 = POST ? r1n : 1.f, r2 = r2n;
        fetch(min(r + RW, end - 1));  // (the last time a row that the caches hold)
        float sum[3] = {0.f, 0.f, 0.f}, w[J][VN], pw[J][VN];
        weight(0, w);
        if (POST) weight(1, pw);
#pragma unroll
        for (int j = 0; j < J; j++)
#pragma unroll
            for (int c = 0; c < VN; c++) {
                float q = p.scale;
                if (GATE) {
                    g[j][c] = sigmoidf(g[j][c]);
                    q *= g[j][c];
                }
                float u = y[j][c];
                if (POST) {
                    y[j][c] *= r1;
                    u = y[j][c] * pw[j][c];
                }
                const float m = fmaf(q, u, s[j][c]) * r2;
                s[j][c] = m;
                if (!p.d_h) e[j][c] = 0.f;
                if (!p.d_s) d[j][c] = 0.f;
                dw[j][c] = fmaf(e[j][c], m, dw[j][c]);
                e[j][c] *= w[j][c];
                sum[0] = fmaf(e[j][c], m, sum[0]);
                d[j][c] = fmaf(r2, e[j][c], d[j][c]);  // ds + r2 e, dx without its mean
                if (POST) {  // q u: scale sigmoid(gate) post n
                    sum[1] = fmaf(q * u, d[j][c], sum[1]);
                    sum[2] = fmaf(q * u, m, sum[2]);
                }
            }
        if (POST) {
            row_sums<T>(sum, red);
        } else {
            float one[1] = {sum[0]};
            row_sums<T>(one, reinterpret_cast<float(*)[1]>(red));
            sum[0] = one[0];
        }
        const float a = sum[0] * p.inverse_d * r2;
        const float mean = (sum[1] - a * sum[2]) * p.inverse_d;
#pragma unroll
        for (int j = 0; j < J; j++)
#pragma unroll
            for (int c = 0; c < VN; c++) d[j][c] = fmaf(-a, s[j][c], d[j][c]);
        if (p.dx) cols.store(static_cast<E*>(p.dx) + o, d);
        if (POST) weight(1, pw);
        if (GATE && p.dgate) {
#pragma unroll
            for (int j = 0; j < J; j++)
#pragma unroll
                for (int c = 0; c < VN; c++) {
                    const float u = POST ? y[j][c] * pw[j][c] : y[j][c];
                    e[j][c] = p.scale * d[j][c] * u * g[j][c] * (1.f - g[j][c]);
                }
            cols.store(static_cast<E*>(p.dgate) + o, e);
        }
#pragma unroll
        for (int j = 0; j < J; j++)
#pragma unroll
            for (int c = 0; c < VN; c++) {
                float du = p.scale * d[j][c];
                if (GATE) du *= g[j][c];
                if (POST) {
                    dp[j][c] = fmaf(du, y[j][c], dp[j][c]);
                    du = r1 * (du * pw[j][c] - y[j][c] * mean);
                }
                d[j][c] = du;
            }
        if (p.dy) cols.store(static_cast<E*>(p.dy) + o, d);
    }
    const auto leave = [&](float (&v)[J][VN], int which) {
        float* out = gridDim.x == 1 ? (which ? p.dpost : p.dweight) : p.part + ((long long)blockIdx.x * 2 + which) * p.D;
        if (RW == 1) {
            cols.store(out, v);
            return;
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < J; j++)
#pragma unroll
            for (int c = 0; c < VN; c++) sums[threadIdx.x / T][(t + j * T) * VN + c] = v[j][c];
        __syncthreads();
        for (int c = threadIdx.x; c < p.D; c += block_of(T)) {
            // column c of the vector that counts it: the last vector ends at D
            const int whole = p.D / VN * VN, at = c < whole ? c : c + VN - (p.D - whole);
            float v = 0.f;
#pragma unroll
            for (int i = 0; i < RW; i++) v += sums[i][at];
            out[c] = v;
        }
    };
    if (p.dweight) leave(dw, 0);
    if (POST && p.dpost) leave(dp, 1);
}

// dweight and dpost: the sums of part's rows, 32 threads per column each every
// 32nd row in order (RS_U loads in flight), then the 32 in order.
constexpr int RS_U = 8;

__global__ __launch_bounds__(1024) void residual_sum_kernel(ResidualParams p, int rows) {
    __shared__ float red[32][33];
    float* out = blockIdx.y ? p.dpost : p.dweight;
    if (!out) return;
    const int col = threadIdx.x & 31, c = min((int)blockIdx.x * 32 + col, p.D - 1), k = threadIdx.x >> 5;
    float s = 0.f;
    for (int i = k; i < rows; i += 32 * RS_U) {
        float v[RS_U];
#pragma unroll
        for (int u = 0; u < RS_U; u++) v[u] = p.part[((long long)min(i + 32 * u, rows - 1) * 2 + blockIdx.y) * p.D + c];
#pragma unroll
        for (int u = 0; u < RS_U; u++)
            if (i + 32 * u < rows) s += v[u];
    }
    red[k][col] = s;
    __syncthreads();
    if (k == 0 && (int)blockIdx.x * 32 + col < p.D) {
        for (int i = 1; i < 32; i++) s += red[i][col];
        out[c] = s;
    }
}

// Rows of a workgroup of the gradient, a multiple of 4: about 512 workgroups, two
// to a compute unit. With 256 / 512 / 1024 / 2048, us on MI355X for the gradient and
// its sums: 16384 x 1024 bf16 with output norm and gate 56 / 52 / 55 / 62, plain 31 /
// 31 / 34 / 37, 2999 x 1536 fp32 22 / 20 / 21 / 21, 16384 x 2048 bf16 143 / 110 / 119 / 120.
long long grad_rows(long long rows) {
    const long long n = (rows + 511) / 512;
    return n < 4 ? 4 : (n + 3) / 4 * 4;
}

template <class E, int VN, int T, int J>
void launch(ResidualParams p, bool grad, hipStream_t stream) {
    p.inverse_d = 1.f / (float)p.D;
    const dim3 block(block_of(T));
    if (!grad) {
        constexpr int RW = block_of(T) / T;
        const long long groups = (p.rows + RW - 1) / RW;
        hipLaunchKernelGGL((residual_norm_kernel<E, VN, T, J>), dim3((unsigned)min(groups, 1ll << 20)), block, 0, stream, p);
        return;
    }
    // Up to four rows for every T threads of a workgroup: one workgroup alone, whose
    // sums are the gradients. us on MI355X so and by several workgroups and
    // their sums: 1024 bf16 columns, 4 rows 5.0 and 9.0, 16 rows 10.2 and 9.5 (13.3
    // and 15.6 with the host's work for the launches), 64 rows 30 and 10; 4096
    // columns, 4 rows 10.5 and 14.5, 16 rows 35 and 14.7.
    constexpr int few = 4 * block_of(T) / T;
    p.rows_wg = p.rows <= few ? few : grad_rows(p.rows);
    const int n = (int)((p.rows + p.rows_wg - 1) / p.rows_wg);
    if (n && p.post && p.gate)
        hipLaunchKernelGGL((residual_grad_kernel<E, VN, T, J, true, true>), dim3(n), block, 0, stream, p);
    else if (n && p.post)
        hipLaunchKernelGGL((residual_grad_kernel<E, VN, T, J, true, false>), dim3(n), block, 0, stream, p);
    else if (n && p.gate)
        hipLaunchKernelGGL((residual_grad_kernel<E, VN, T, J, false, true>), dim3(n), block, 0, stream, p);
    else if (n)
        hipLaunchKernelGGL((residual_grad_kernel<E, VN, T, J, false, false>), dim3(n), block, 0, stream, p);
    if (n != 1 && (p.dweight || p.dpost))
        hipLaunchKernelGGL(residual_sum_kernel, dim3((p.D + 31) / 32, 2), dim3(1024), 0, stream, p, n);
}

// Threads of a row and vectors of each: up to 16 elements a thread, and a wave to
// a row as far as that goes (16384 x 1024 bf16 with output norm and gate, a wave
// against a workgroup to a row: forward 28 and 37 us, gradient 52 and 81). The
// gradient keeps them in registers with two waves per SIMD up to 4096 columns.
// Past those, where the threads of a workgroup hold a row and its weights, it does
// not: with output norm and gate 36 bytes a lane of 16-bit rows go to scratch,
// 292 of fp32 rows (24 with the output norm alone, 36 with the gate alone). us on
// MI355X with both, forward and gradient: 2^24 bf16 elements in rows of 1024 28.5
// and 52.5, of 4096 28.4 and 53.5, of 8192 28.9 and 68.8; 2^23 fp32 elements in
// rows of 4096 26.9 and 55.4, of 8192 27.3 and 106.5.
template <class E>
void launch_type(const ResidualParams& p, bool grad, hipStream_t stream) {
    constexpr int N = 16 / sizeof(E);
    if (p.D < N) return launch<E, 1, 64, 1>(p, grad, stream);
    if (p.D <= 64 * N) return launch<E, N, 64, 1>(p, grad, stream);
    if (p.D <= 128 * N) return launch<E, N, 64, 2>(p, grad, stream);
    if (p.D <= 256 * N) return launch<E, N, 256, 1>(p, grad, stream);
    if (p.D <= 512 * N) return launch<E, N, 256, 2>(p, grad, stream);
    if (p.D <= 1024 * N) return launch<E, N, 512, 2>(p, grad, stream);
    if constexpr (N == 4) launch<E, N, 512, 4>(p, grad, stream);
}

}  // namespace

size_t residual_workspace_bytes(long long rows, int D) {
    const long long w = grad_rows(rows);
    return rows > 0 ? (size_t)((rows + w - 1) / w) * 2 * D * 4 : 16;
}

void launch_residual_norm(const ResidualParams& p, int dtype, bool grad, hipStream_t stream) {
    if (dtype == 0)
        launch_type<bf16_t>(p, grad, stream);
    else if (dtype == 1)
        launch_type<float>(p, grad, stream);
    else
        launch_type<f16_t>(p, grad, stream);
}

}  // namespace cyfa
