// Layer norm over the last axis of [rows, C], forward and backward (with the weights' gradients), for fp32 / fp16 / bf16 rows of any pitch.
//     y = (x - mean) rstd gamma + beta                       stats[row] = (mean, rstd)
//     dx = rstd (g - mean(g) - xhat mean(g xhat)) (+ addend), g = dy gamma, xhat = (x - mean) rstd
//     dgamma = sum_rows dy xhat        dbeta = sum_rows dy
// Both passes read every tensor once: a row lives in the registers of TPR threads (TPR * NC vectors of 16 bytes), the variance is the mean
// of squared deviations from the mean (no cancellation between E[x^2] and mean^2).  All sums are fp32.
//
// Weight gradients without atomics: a persistent grid, every thread owns the same columns in all its rows and keeps their sums in registers;
// a workgroup joins its rows' threads through LDS in a fixed order and leaves ONE partial row in the workspace, which a second launch sums.
// Rows need element alignment only: the 16-byte accesses of this hardware take any address.
//
// Bound by memory: each row's loads are issued one row ahead of their use.  MI355X (a 1 GiB copy runs at 5.2 TB/s): forward 50 432 x 768 bf16
// 29.3 us = 5.3 TB/s; backward with weight gradients and addend 60.4 us = 5.1 TB/s; backward 5 003 x 1001 fp32 16.3 us = 3.7 TB/s (two launches);
// forward 64 x 768 7 us, the time of a launch.  The variant of plan() goes by the row's width only.  Backward above 8192 columns the 512-thread forms spill
// 108 to 197 registers: 4096 x 16384 239 us in bf16 and 415 in fp32, where their bytes take 77 and 154 (8192 x 8192 bf16: 94 us).
#include "dp_common.h"
#include "dp_region.h"

namespace {

template <typename X, int N> struct __attribute__((packed, aligned(sizeof(X)))) Pack { X e[N]; };
template <typename X, int N> __device__ __forceinline__ Pack<X, N> ld(const X* p) { return *reinterpret_cast<const Pack<X, N>*>(p); }
template <typename X, int N> __device__ __forceinline__ void st(X* p, const float* f) {
    Pack<X, N> v;
#pragma unroll
    for (int j = 0; j < N; ++j) v.e[j] = (X)f[j];
    *reinterpret_cast<Pack<X, N>*>(p) = v;
}

// Columns of a thread's vector: the vector that would reach behind the row's end is moved back to end with it (C >= N), so every access is a whole
// vector and nothing branches.  Its first `skip` columns then belong to the vector before it: both threads compute and store the same values
// there; only the sums over the row leave them out.  A thread without columns repeats the last vector and skips all of it.
template <int N> struct Cols {
    int at, skip;
    __device__ __forceinline__ Cols(int vec, int C) {
        const int want = vec * N;
        at = want + N <= C ? want : C - N;
        skip = want - at;
    }
};

// sum over the TPR threads of a row; every thread gets it.  red: one slot per wave (TPR > 64 only: two barriers)
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* red) {
#pragma unroll
    for (int o = (TPR < 64 ? TPR : 64) / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    if constexpr (TPR > 64) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        v = 0.f;
#pragma unroll
        for (int w = 0; w < TPR / 64; ++w) v += red[w];
    }
    return v;
}

template <typename X, typename W, int N, int TPR, int NC>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void layer_norm_kernel(const X* x, long long rows, int C, long long xs, const W* gamma, const W* beta, float eps, X* y,
                                                                           long long ys, float* stats) {
    constexpr int WGT = TPR > 256 ? TPR : 256, RPB = WGT / TPR;
    __shared__ float red[WGT / 64];
    const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR;
    const float inv_c = 1.f / (float)C;
    float ga[NC][N], be[NC][N];
    int at[NC], skip[NC];
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        const Cols<N> c(i * TPR + t, C);
        at[i] = c.at;
        skip[i] = c.skip;
#pragma unroll
        for (int j = 0; j < N; ++j) { ga[i][j] = 1.f; be[i][j] = 0.f; }
        if (gamma) {
            const Pack<W, N> w = ld<W, N>(gamma + c.at);
#pragma unroll
            for (int j = 0; j < N; ++j) ga[i][j] = (float)w.e[j];
        }
        if (beta) {
            const Pack<W, N> w = ld<W, N>(beta + c.at);
#pragma unroll
            for (int j = 0; j < N; ++j) be[i][j] = (float)w.e[j];
        }
    }
    const long long step = (long long)gridDim.x * RPB;
    long long row = (long long)blockIdx.x * RPB + sub;
    Pack<X, N> raw[NC];                                  // a row ahead: the next row's loads are under way while this one is reduced
#pragma unroll
    for (int i = 0; i < NC; ++i) raw[i] = ld<X, N>(x + (row < rows ? row : rows - 1) * xs + at[i]);
    for (long long r0 = (long long)blockIdx.x * RPB; r0 < rows; r0 += step, row += step) {
        float v[NC][N], s = 0.f;
#pragma unroll
        for (int i = 0; i < NC; ++i)
#pragma unroll
            for (int j = 0; j < N; ++j) {
                v[i][j] = (float)raw[i].e[j];
                s += j >= skip[i] ? v[i][j] : 0.f;
            }
        const long long next = row + step < rows ? row + step : rows - 1;
#pragma unroll
        for (int i = 0; i < NC; ++i) raw[i] = ld<X, N>(x + next * xs + at[i]);
        const float mean = row_sum<TPR>(s, red) * inv_c;
        float q = 0.f;
#pragma unroll
        for (int i = 0; i < NC; ++i)
#pragma unroll
            for (int j = 0; j < N; ++j) {
                v[i][j] -= mean;
                q += j >= skip[i] ? v[i][j] * v[i][j] : 0.f;
            }
        const float rstd = 1.f / sqrtf(row_sum<TPR>(q, red) * inv_c + eps);
        if (row >= rows) continue;
        X* yr = y + row * ys;
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            float o[N];
#pragma unroll
            for (int j = 0; j < N; ++j) o[j] = fmaf(v[i][j] * rstd, ga[i][j], be[i][j]);
            if (skip[i] < N) st<X, N>(yr + at[i], o);
        }
        if (stats && t == 0) {
            stats[row * 2] = mean;
            stats[row * 2 + 1] = rstd;
        }
    }
}

template <typename X, typename W, int N, int TPR, int NC>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void layer_norm_bwd_kernel(const X* dy, long long dys, const X* x, long long xs, long long rows, int C, const W* gamma,
                                                                               const float* stats, const X* addend, long long as, X* dx, long long dxs, float* partial) {
    constexpr int WGT = TPR > 256 ? TPR : 256, RPB = WGT / TPR;
    __shared__ float red[2][WGT / 64];
    __shared__ float join[TPR <= 64 ? 2 * TPR * NC * N : 1];
    const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR;
    const float inv_c = 1.f / (float)C;
    float ga[NC][N], dg[NC][N], db[NC][N];
    int at[NC], skip[NC];
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        const Cols<N> c(i * TPR + t, C);
        at[i] = c.at;
        skip[i] = c.skip;
#pragma unroll
        for (int j = 0; j < N; ++j) { ga[i][j] = 1.f; dg[i][j] = 0.f; db[i][j] = 0.f; }
        if (gamma) {
            const Pack<W, N> w = ld<W, N>(gamma + c.at);
#pragma unroll
            for (int j = 0; j < N; ++j) ga[i][j] = (float)w.e[j];
        }
    }
    const long long step = (long long)gridDim.x * RPB;
    long long row = (long long)blockIdx.x * RPB + sub;
    Pack<X, N> rx[NC], rd[NC], ra[NC];                   // a row ahead
    float rmean, rrstd;
    auto fetch = [&](long long r) {
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            rx[i] = ld<X, N>(x + r * xs + at[i]);
            rd[i] = ld<X, N>(dy + r * dys + at[i]);
        }
        rmean = stats[r * 2];
        rrstd = stats[r * 2 + 1];
    };
    fetch(row < rows ? row : rows - 1);
    for (long long r0 = (long long)blockIdx.x * RPB; r0 < rows; r0 += step, row += step) {
        const bool live = row < rows;
        const float mean = rmean, rstd = rrstd;
        float xh[NC][N], d[NC][N], s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int i = 0; i < NC; ++i)
#pragma unroll
            for (int j = 0; j < N; ++j) {
                xh[i][j] = (float)rx[i].e[j];
                d[i][j] = (float)rd[i].e[j];
            }
        if (addend) {
#pragma unroll
            for (int i = 0; i < NC; ++i) ra[i] = ld<X, N>(addend + (live ? row : rows - 1) * as + at[i]);
        }
        fetch(row + step < rows ? row + step : rows - 1);
#pragma unroll
        for (int i = 0; i < NC; ++i)
#pragma unroll
            for (int j = 0; j < N; ++j) {
                xh[i][j] = (xh[i][j] - mean) * rstd;
                const float v = live ? d[i][j] : 0.f;
                dg[i][j] = fmaf(v, xh[i][j], dg[i][j]);
                db[i][j] += v;
                d[i][j] *= ga[i][j];
                const float g = j >= skip[i] ? d[i][j] : 0.f;
                s1 += g;
                s2 = fmaf(g, xh[i][j], s2);
            }
        s1 = row_sum<TPR>(s1, red[0]) * inv_c;
        s2 = row_sum<TPR>(s2, red[1]) * inv_c;
        if (!live) continue;
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            float o[N];
#pragma unroll
            for (int j = 0; j < N; ++j) {
                o[j] = (d[i][j] - s1 - xh[i][j] * s2) * rstd;
                if (addend) o[j] += (float)ra[i].e[j];
            }
            if (skip[i] < N) st<X, N>(dx + row * dxs + at[i], o);
        }
    }
    if (!partial) return;
    float* out = partial + (long long)blockIdx.x * 2 * C;
    if constexpr (TPR <= 64) {
        constexpr int P = TPR * NC * N;                  // by vector, not by column: no two threads of a row share a place
        for (int s = 0; s < RPB; ++s) {
            if (sub == s) {
#pragma unroll
                for (int i = 0; i < NC; ++i)
#pragma unroll
                    for (int j = 0; j < N; ++j) {
                        const int k = (i * N + j) * TPR + t;
                        join[k] = s ? join[k] + dg[i][j] : dg[i][j];
                        join[P + k] = s ? join[P + k] + db[i][j] : db[i][j];
                    }
            }
            __syncthreads();
        }
        if (sub == 0) {
#pragma unroll
            for (int i = 0; i < NC; ++i)
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    dg[i][j] = join[(i * N + j) * TPR + t];
                    db[i][j] = join[P + (i * N + j) * TPR + t];
                }
        }
    }
    if (sub == 0) {
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            if (skip[i] >= N) continue;
            st<float, N>(out + at[i], dg[i]);
            st<float, N>(out + C + at[i], db[i]);
        }
    }
}

// sums of the partial rows: 16 columns per workgroup, 64 groups of threads share the rows (fixed assignment, fixed order of the join)
template <typename W>
__global__ __launch_bounds__(1024) void layer_norm_wsum_kernel(const float* partial, int parts, int C, W* dgamma, W* dbeta) {
    __shared__ float part[64][17];
    const int lane = threadIdx.x & 15, group = threadIdx.x >> 4;
    const int col = blockIdx.x * 16 + lane;
    float s = 0.f;
    if (col < 2 * C) {
        const float* p = partial + col;
        int r = group;
        for (; r + 7 * 64 < parts; r += 8 * 64) {          // eight loads under way at a time: this is a latency, not a bandwidth, problem
            float v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = p[(long long)(r + k * 64) * 2 * C];
#pragma unroll
            for (int k = 0; k < 8; ++k) s += v[k];
        }
        for (; r < parts; r += 64) s += p[(long long)r * 2 * C];
    }
    part[group][lane] = s;
    __syncthreads();
    if (group >= 4) return;
    s = 0.f;
#pragma unroll
    for (int w = 0; w < 16; ++w) s += part[group * 16 + w][lane];
    s += __shfl_xor(s, 16, 64);                            // the four groups left are one wave
    s += __shfl_xor(s, 32, 64);
    W* out = col < C ? dgamma : dbeta;
    if (group == 0 && col < 2 * C && out) out[col < C ? col : col - C] = (W)s;
}

constexpr int MAX_C = 16384;
// Persistent grids: 8 / 2 workgroups of 256 threads per CU.  Backward, 50 432 x 768 bf16 with an addend: 512 blocks 60.4 us, 768 64.3, 1024 73.4, 1536
// 68.7 (5 003 x 1001 fp32: 16.3 / 20.4 / 21.5 / 25.1): every block leaves a partial row, and more than the registers hold at once run as a second, ragged wave of blocks.
constexpr int FWD_BLOCKS = 2048, BWD_BLOCKS = 512;

struct Plan { int tpr, nc; };
// a row on as few threads as hold it in 32 floats each: one wave up to 2048 columns (narrow rows share a wave), 256 threads up to 8192, else 512
Plan plan(int C, int n) {
    const int vecs = C < n ? C : (C + n - 1) / n;        // rows shorter than a vector: element by element
    if (vecs <= 16) return {16, 1};
    if (vecs <= 32) return {32, 1};
    if (vecs <= 64) return {64, 1};
    if (vecs <= 128) return {64, 2};
    if (vecs <= 192) return {64, 3};
    if (vecs <= 256) return {64, 4};
    if (n == 4 && vecs <= 512) return {64, 8};
    if (vecs <= 512) return {256, 2};
    if (vecs <= 1024) return {256, 4};
    if (n == 4 && vecs <= 2048) return {256, 8};
    return {512, n == 4 ? 8 : 4};
}
int blocks_of(long long rows, const Plan& p, int most) {
    const int rpb = p.tpr >= 256 ? 1 : 256 / p.tpr;
    const long long need = (rows + rpb - 1) / rpb;
    return (int)(need < most ? need : most);
}

struct FwdCall {
    const void* x; long long rows; int C; long long xs; const void *gamma, *beta; float eps; void* y; long long ys; float* stats; hipStream_t s;
    template <typename X, typename W, int N, int TPR, int NC> void go() const {
        hipLaunchKernelGGL((layer_norm_kernel<X, W, N, TPR, NC>), dim3(blocks_of(rows, {TPR, NC}, FWD_BLOCKS)), dim3(TPR > 256 ? TPR : 256), 0, s, (const X*)x, rows, C, xs,
                           (const W*)gamma, (const W*)beta, eps, (X*)y, ys, stats);
    }
};
struct BwdCall {
    const void* dy; long long dys; const void* x; long long xs, rows; int C; const void* gamma; const float* stats; const void* addend; long long as; void* dx; long long dxs;
    float* partial; hipStream_t s;
    template <typename X, typename W, int N, int TPR, int NC> void go() const {
        hipLaunchKernelGGL((layer_norm_bwd_kernel<X, W, N, TPR, NC>), dim3(blocks_of(rows, {TPR, NC}, BWD_BLOCKS)), dim3(TPR > 256 ? TPR : 256), 0, s, (const X*)dy, dys,
                           (const X*)x, xs, rows, C, (const W*)gamma, stats, (const X*)addend, as, (X*)dx, dxs, partial);
    }
};
template <typename X, typename W, typename Call>
void dispatch(const Call& c, const Plan& p) {
    constexpr int N = 16 / sizeof(X);
    if (c.C < N) c.template go<X, W, 1, 16, 1>();
    else if (p.tpr == 16) c.template go<X, W, N, 16, 1>();
    else if (p.tpr == 32) c.template go<X, W, N, 32, 1>();
    else if (p.tpr == 64 && p.nc == 1) c.template go<X, W, N, 64, 1>();
    else if (p.tpr == 64 && p.nc == 2) c.template go<X, W, N, 64, 2>();
    else if (p.tpr == 64 && p.nc == 3) c.template go<X, W, N, 64, 3>();
    else if (p.tpr == 64 && p.nc == 4) c.template go<X, W, N, 64, 4>();
    else if (p.tpr == 256 && p.nc == 4) c.template go<X, W, N, 256, 4>();
    else if constexpr (sizeof(X) == 4) {
        if (p.tpr == 64) c.template go<X, W, N, 64, 8>();
        else if (p.tpr == 256) c.template go<X, W, N, 256, 8>();
        else c.template go<X, W, N, 512, 8>();
    } else {
        if (p.tpr == 256) c.template go<X, W, N, 256, 2>();
        else c.template go<X, W, N, 512, 4>();
    }
}
template <typename Call>
void dispatch(const Call& c, int x_dtype, int w_dtype, const Plan& p) {
    if (x_dtype == 0) dispatch<float, float>(c, p);
    else if (x_dtype == 1 && w_dtype == 0) dispatch<_Float16, float>(c, p);
    else if (x_dtype == 1) dispatch<_Float16, _Float16>(c, p);
    else if (w_dtype == 0) dispatch<__bf16, float>(c, p);
    else dispatch<__bf16, __bf16>(c, p);
}

int check(const char* fn, int x_dtype, int w_dtype, long long rows, int C) {
    DP_REQUIRE(x_dtype >= 0 && x_dtype <= 2, "%s: dtype %d (0 = fp32, 1 = fp16, 2 = bf16)", fn, x_dtype);
    DP_REQUIRE(w_dtype == 0 || w_dtype == x_dtype, "%s: the weights are fp32 or of the rows' type (got dtype %d)", fn, w_dtype);
    DP_REQUIRE(rows > 0 && C > 0 && C <= MAX_C, "%s: rows of 1 to %d columns, at least one (got %lld x %d)", fn, MAX_C, rows, C);
    return 0;
}

constexpr long long MAX_PITCH = 1LL << 40;

dp::Region row_region(const char* name, const void* p, long long rows, int C, long long pitch, int es) {
    return dp::Region{name, (intptr_t)p, {rows, 1, 1}, {pitch * es, 0, 0}, p ? (long long)C * es : 0};
}

}  // namespace

extern "C" int dp_layer_norm(const void* x, int x_dtype, long long rows, int C, long long x_stride, const void* gamma, const void* beta, int w_dtype, float eps, void* y,
                             long long y_stride, float* stats, void* stream) {
    const char* fn = "dp_layer_norm";
    if (int rc = check(fn, x_dtype, w_dtype, rows, C)) return rc;
    DP_REQUIRE(x && y, "%s: tensor missing", fn);
    DP_REQUIRE(eps >= 0.f && eps - eps == 0.f, "%s: eps must be finite and not negative", fn);
    DP_REQUIRE(x_stride >= 0 && x_stride <= MAX_PITCH && y_stride <= MAX_PITCH && (y_stride >= C || rows == 1), "%s: row pitch (x %lld, y %lld; y's rows must not overlap)", fn, x_stride, y_stride);
    const int es = x_dtype == 0 ? 4 : 2, wes = w_dtype == 0 ? 4 : 2;
    const dp::Region written[] = {row_region("y", y, rows, C, y_stride, es), dp::flat("stats", stats, rows * 8)},
                     read[] = {row_region("x", x, rows, C, x_stride, es), dp::flat("gamma", gamma, (long long)C * wes), dp::flat("beta", beta, (long long)C * wes)};
    if (dp::check_apart(fn, written, 2, read, 3)) return 1;
    const FwdCall c{x, rows, C, x_stride, gamma, beta, eps, y, y_stride, stats, (hipStream_t)stream};
    dispatch(c, x_dtype, w_dtype, plan(C, x_dtype == 0 ? 4 : 8));
    DP_LAUNCH_CHECK("layer_norm");
    return 0;
}

extern "C" long long dp_layer_norm_bwd_workspace(long long rows, int C, int x_dtype) {
    if (rows <= 0 || C <= 0 || C > MAX_C) return 0;
    return (long long)blocks_of(rows, plan(C, x_dtype == 0 ? 4 : 8), BWD_BLOCKS) * 2 * C * 4;
}

extern "C" int dp_layer_norm_bwd(const void* dy, long long dy_stride, const void* x, long long x_stride, int x_dtype, long long rows, int C, const void* gamma, int w_dtype,
                                 const float* stats, const void* addend, long long addend_stride, void* dx, long long dx_stride, void* dgamma, void* dbeta, void* work,
                                 long long work_bytes, void* stream) {
    const char* fn = "dp_layer_norm_bwd";
    if (int rc = check(fn, x_dtype, w_dtype, rows, C)) return rc;
    DP_REQUIRE(dy && x && stats && dx, "%s: tensor missing", fn);
    DP_REQUIRE(dy_stride >= 0 && x_stride >= 0 && addend_stride >= 0 && dy_stride <= MAX_PITCH && x_stride <= MAX_PITCH && addend_stride <= MAX_PITCH && dx_stride <= MAX_PITCH &&
                   (dx_stride >= C || rows == 1), "%s: row pitch (dx's rows must not overlap)", fn);
    const bool weights = dgamma || dbeta;
    DP_REQUIRE(!weights || (work && (reinterpret_cast<uintptr_t>(work) & 3) == 0 && work_bytes >= dp_layer_norm_bwd_workspace(rows, C, x_dtype)),
               "%s: workspace of %lld bytes needed for the weight gradients (got %lld)", fn, dp_layer_norm_bwd_workspace(rows, C, x_dtype), work_bytes);
    const int es = x_dtype == 0 ? 4 : 2, wes = w_dtype == 0 ? 4 : 2;
    const dp::Region written[] = {row_region("dx", dx, rows, C, dx_stride, es), dp::flat("dgamma", dgamma, (long long)C * wes), dp::flat("dbeta", dbeta, (long long)C * wes),
                                  dp::flat("work", weights ? work : nullptr, dp_layer_norm_bwd_workspace(rows, C, x_dtype))},
                     read[] = {row_region("dy", dy, rows, C, dy_stride, es), row_region("x", x, rows, C, x_stride, es), dp::flat("gamma", gamma, (long long)C * wes),
                               dp::flat("stats", stats, rows * 8), row_region("addend", addend, rows, C, addend_stride, es)};
    if (dp::check_apart(fn, written, 4, read, 5)) return 1;
    hipStream_t s = (hipStream_t)stream;
    const Plan p = plan(C, x_dtype == 0 ? 4 : 8);
    const BwdCall c{dy, dy_stride, x, x_stride, rows, C, gamma, stats, addend, addend_stride, dx, dx_stride, weights ? (float*)work : nullptr, s};
    dispatch(c, x_dtype, w_dtype, p);
    DP_LAUNCH_CHECK("layer_norm_bwd");
    if (weights) {
        const int parts = blocks_of(rows, p, BWD_BLOCKS);
        const dim3 grid((2 * C + 15) / 16);
        if (w_dtype == 0) hipLaunchKernelGGL(layer_norm_wsum_kernel<float>, grid, dim3(1024), 0, s, (const float*)work, parts, C, (float*)dgamma, (float*)dbeta);
        else if (w_dtype == 1) hipLaunchKernelGGL(layer_norm_wsum_kernel<_Float16>, grid, dim3(1024), 0, s, (const float*)work, parts, C, (_Float16*)dgamma, (_Float16*)dbeta);
        else hipLaunchKernelGGL(layer_norm_wsum_kernel<__bf16>, grid, dim3(1024), 0, s, (const float*)work, parts, C, (__bf16*)dgamma, (__bf16*)dbeta);
        DP_LAUNCH_CHECK("layer_norm_wsum");
    }
    return 0;
}
