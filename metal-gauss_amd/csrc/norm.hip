// Layer norm over the last dimension, forward and backward.
//
//   m = mean(x), s = 1 / sqrt(mean((x - m)^2) + eps), u = (x - m) s
//   y = u w + b
//   dx = s (g - mean(g) - u mean(g u)),  g = dy w
//   dw = sum over rows of dy u,  db = sum over rows of dy
//
// Memory bounds every kernel here: a row is read once, held in registers
// between its two reductions (the mean, then the squares about it: a row far
// from zero keeps its variance's digits), and written once. All arithmetic is
// in float32 whatever the type of x; a row's mean and s are kept as float32 for
// the backward pass.
//
// 65280 rows of 1024 bfloat16, float32 weights: forward 45 us (5.9 TB/s), backward
// 66 (6.1 TB/s) and 4 to join the weights' gradients; 64 rows of 256 float32: 3 us,
// the launch. Few or wide rows: 2048 of 8192 take 16 us forward, and 40 and 12 to
// join backward, where the workgroups' sums of columns (67 MB written, then read)
// move more bytes than the rows (101 MB).
#include "mg_types.h"

namespace mg {

// A row is held by kWaves waves, C accesses of V elements a thread: thread t
// has elements (t + i * 64 kWaves) V .. + V - 1 for i < C. Rows longer than the
// widest form are read once per pass instead (norm_loop_*). A workgroup keeps the
// weights in registers over all its rows (from memory for each row they would be
// twice a bfloat16 row's own bytes).

// Sum over the threads that hold a row, in all of them. `slot` alternates so
// that one barrier a reduction suffices: a slot is written again only after
// the barrier of the reduction between.
template <int kWaves>
__device__ __forceinline__ float row_sum(float v, float (*red)[16], int slot) {
    v = wave_sum_all(v);
    if constexpr (kWaves > 1) {
        const int wave = threadIdx.x / 64;
        if (lane_id() == 0) red[slot][wave] = v;
        __syncthreads();
        v = 0.f;
#pragma unroll
        for (int i = 0; i < kWaves; ++i) v += red[slot][i];
        lds_reads_done();
    }
    return v;
}

// Rows handled by one workgroup at a time.
template <int kWaves>
constexpr int kRowsAtOnce = kWaves == 1 ? 4 : 1;
template <int kWaves>
constexpr int kNormThreads = 64 * kWaves * kRowsAtOnce<kWaves>;

template <typename T, typename W, int C, int kWaves>
__global__ __launch_bounds__(kNormThreads<kWaves>) void norm_fwd_kernel(
    int64_t rows, int n, const T *__restrict__ x, int64_t x_stride, const W *__restrict__ weight,
    const W *__restrict__ bias, float eps, T *__restrict__ y, float *__restrict__ mean,
    float *__restrict__ rstd) {
    constexpr int V = kVec<T>;
    __shared__ float red[2][16];
    const int t = threadIdx.x % (64 * kWaves);
    float w[C][V], b[C][V];
#pragma unroll
    for (int i = 0; i < C; ++i) {
        const int at = (t + i * 64 * kWaves) * V;
        if (weight) {
            load_row<W, V>(weight, at, n, w[i]);
        } else {
            for (int k = 0; k < V; ++k) w[i][k] = 1.f;
        }
        if (bias) {
            load_row<W, V>(bias, at, n, b[i]);
        } else {
            for (int k = 0; k < V; ++k) b[i][k] = 0.f;
        }
    }
    const int64_t step = (int64_t)gridDim.x * kRowsAtOnce<kWaves>;
    int64_t row = (int64_t)blockIdx.x * kRowsAtOnce<kWaves> + threadIdx.x / (64 * kWaves);
    for (; row < rows; row += step) {
        const T *xr = x + row * x_stride;
        float v[C][V], sum = 0.f, sq = 0.f;
#pragma unroll
        for (int i = 0; i < C; ++i) {
            load_row<T, V>(xr, (t + i * 64 * kWaves) * V, n, v[i]);
#pragma unroll
            for (int k = 0; k < V; ++k) sum += v[i][k];
        }
        const float m = row_sum<kWaves>(sum, red, 0) / (float)n;
#pragma unroll
        for (int i = 0; i < C; ++i) {
            const int at = (t + i * 64 * kWaves) * V;
#pragma unroll
            for (int k = 0; k < V; ++k) {
                v[i][k] = at + k < n ? v[i][k] - m : 0.f;
                sq = fmaf(v[i][k], v[i][k], sq);
            }
        }
        const float s = 1.f / sqrtf(row_sum<kWaves>(sq, red, 1) / (float)n + eps);
        T *yr = y + row * n;
#pragma unroll
        for (int i = 0; i < C; ++i) {
#pragma unroll
            for (int k = 0; k < V; ++k) v[i][k] = fmaf(v[i][k] * s, w[i][k], b[i][k]);
            store_row<T, V>(yr, (t + i * 64 * kWaves) * V, n, v[i]);
        }
        if (t == 0 && mean) {
            mean[row] = m;
            rstd[row] = s;
        }
    }
}

// Each workgroup adds up dy u and dy over the rows it takes; the column sums of
// all workgroups (partial: (gridDim.x, 2, n)) are joined by norm_join_kernel,
// in a fixed order, so that a gradient is the same from call to call.
//
// kStream: arrays larger than the L2 caches pass by them (65280 rows of 1024
// bfloat16: 77 us, with streaming accesses 67; the forward is the same either
// way).
template <typename T, typename W, int C, int kWaves, bool kStream>
__global__ __launch_bounds__(kNormThreads<kWaves>) void norm_bwd_kernel(
    int64_t rows, int n, const T *__restrict__ x, int64_t x_stride, const T *__restrict__ dy,
    int64_t dy_stride, const W *__restrict__ weight, const float *__restrict__ mean,
    const float *__restrict__ rstd, T *__restrict__ dx, float *__restrict__ partial) {
    constexpr int V = kVec<T>;
    constexpr int kRows = kRowsAtOnce<kWaves>;
    __shared__ float red[4][16];
    __shared__ float s_col[kRows > 1 ? C * V * 64 : 1];
    const int t = threadIdx.x % (64 * kWaves);
    float w[C][V], dw[C][V] = {}, db[C][V] = {};
#pragma unroll
    for (int i = 0; i < C; ++i) {
        if (weight) {
            load_row<W, V>(weight, (t + i * 64 * kWaves) * V, n, w[i]);
        } else {
            for (int k = 0; k < V; ++k) w[i][k] = 1.f;
        }
    }
    const int64_t step = (int64_t)gridDim.x * kRows;
    int64_t row = (int64_t)blockIdx.x * kRows + threadIdx.x / (64 * kWaves);
    int slot = 0;
    for (; row < rows; row += step) {
        const T *xr = x + row * x_stride, *dyr = dy + row * dy_stride;
        const float m = mean[row], s = rstd[row];
        float u[C][V], g[C][V], sg = 0.f, sgu = 0.f;
#pragma unroll
        for (int i = 0; i < C; ++i) {
            const int at = (t + i * 64 * kWaves) * V;
            load_row<T, V, kStream>(xr, at, n, u[i]);
            load_row<T, V, kStream>(dyr, at, n, g[i]);
        }
#pragma unroll
        for (int i = 0; i < C; ++i) {
#pragma unroll
            for (int k = 0; k < V; ++k) {
                // Past the row's end g is 0, and so is all that u enters.
                u[i][k] = (u[i][k] - m) * s;
                dw[i][k] = fmaf(g[i][k], u[i][k], dw[i][k]);
                db[i][k] += g[i][k];
                g[i][k] *= w[i][k];
                sg += g[i][k];
                sgu = fmaf(g[i][k], u[i][k], sgu);
            }
        }
        sg = row_sum<kWaves>(sg, red, slot) / (float)n;
        sgu = row_sum<kWaves>(sgu, red, slot + 1) / (float)n;
        slot ^= 2;
        if (dx) {
#pragma unroll
            for (int i = 0; i < C; ++i) {
#pragma unroll
                for (int k = 0; k < V; ++k) g[i][k] = s * (g[i][k] - sg - u[i][k] * sgu);
                store_row<T, V, kStream>(dx + row * n, (t + i * 64 * kWaves) * V, n, g[i]);
            }
        }
    }
    if (!partial) return;
    float *out = partial + (int64_t)blockIdx.x * 2 * n;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        float(&acc)[C][V] = which ? db : dw;
        if constexpr (kRows > 1) {
            // The four waves' sums, one wave after the other.
            const int wave = threadIdx.x / 64;
            for (int from = 1; from < kRows; ++from) {
                __syncthreads();
                if (wave == from) {
#pragma unroll
                    for (int i = 0; i < C; ++i)
#pragma unroll
                        for (int k = 0; k < V; ++k) s_col[(i * V + k) * 64 + t] = acc[i][k];
                }
                __syncthreads();
                if (wave == 0) {
#pragma unroll
                    for (int i = 0; i < C; ++i)
#pragma unroll
                        for (int k = 0; k < V; ++k) acc[i][k] += s_col[(i * V + k) * 64 + t];
                }
                lds_reads_done();
            }
            if (wave != 0) continue;
        }
#pragma unroll
        for (int i = 0; i < C; ++i)
            store_row<float, V>(out + which * n, (t + i * 64 * kWaves) * V, n, acc[i]);
    }
}

// dw (blockIdx.y 0) and db (1) of 32 columns: 32 threads a column, each over
// every 32nd workgroup's sums.
constexpr int kJoinCols = 32, kJoinThreads = 1024;
template <typename W>
__global__ __launch_bounds__(kJoinThreads) void norm_join_kernel(const float *__restrict__ partial,
                                                                int parts, int n,
                                                                W *__restrict__ dw,
                                                                W *__restrict__ db) {
    constexpr int kGroups = kJoinThreads / kJoinCols;
    __shared__ float s[kGroups][kJoinCols + 1];
    const int col = threadIdx.x % kJoinCols, group = threadIdx.x / kJoinCols;
    const int at = blockIdx.x * kJoinCols + col, which = blockIdx.y;
    float sum = 0.f;
    if (at < n) {
        const float *p = partial + which * (int64_t)n + at;
#pragma unroll 8
        for (int i = group; i < parts; i += kGroups) sum += p[(int64_t)i * 2 * n];
    }
    s[group][col] = sum;
    __syncthreads();
    W *out = which ? db : dw;
    if (group == 0 && at < n && out) {
        float total = 0.f;
#pragma unroll
        for (int i = 0; i < kGroups; ++i) total += s[i][col];
        out[at] = (W)total;
    }
}

// ------------------------------------------------------------- longest rows
// Rows past 16 waves' registers: one workgroup a row, the row read again for
// each of its three passes (from L2 where it fits), an element a lane. 1024 rows of
// 20000 bfloat16: forward 48 us (1.7 TB/s), backward 46 and 20 for the weights' sums.
constexpr int kLoopThreads = 1024;

template <typename T, typename W>
__global__ __launch_bounds__(kLoopThreads) void norm_loop_fwd_kernel(
    int n, const T *__restrict__ x, int64_t x_stride, const W *__restrict__ weight,
    const W *__restrict__ bias, float eps, T *__restrict__ y, float *__restrict__ mean,
    float *__restrict__ rstd) {
    __shared__ float red[2][16];
    const int64_t row = blockIdx.x;
    const T *xr = x + row * x_stride;
    float sum = 0.f, sq = 0.f;
    for (int i = threadIdx.x; i < n; i += kLoopThreads) sum += (float)xr[i];
    const float m = row_sum<16>(sum, red, 0) / (float)n;
    for (int i = threadIdx.x; i < n; i += kLoopThreads) {
        const float d = (float)xr[i] - m;
        sq = fmaf(d, d, sq);
    }
    const float s = 1.f / sqrtf(row_sum<16>(sq, red, 1) / (float)n + eps);
    for (int i = threadIdx.x; i < n; i += kLoopThreads) {
        const float u = ((float)xr[i] - m) * s;
        y[row * n + i] =
            (T)fmaf(u, weight ? (float)weight[i] : 1.f, bias ? (float)bias[i] : 0.f);
    }
    if (threadIdx.x == 0 && mean) {
        mean[row] = m;
        rstd[row] = s;
    }
}

template <typename T, typename W>
__global__ __launch_bounds__(kLoopThreads) void norm_loop_dx_kernel(
    int n, const T *__restrict__ x, int64_t x_stride, const T *__restrict__ dy, int64_t dy_stride,
    const W *__restrict__ weight, const float *__restrict__ mean, const float *__restrict__ rstd,
    T *__restrict__ dx) {
    __shared__ float red[2][16];
    const int64_t row = blockIdx.x;
    const T *xr = x + row * x_stride, *dyr = dy + row * dy_stride;
    const float m = mean[row], s = rstd[row];
    float sg = 0.f, sgu = 0.f;
    for (int i = threadIdx.x; i < n; i += kLoopThreads) {
        const float g = (float)dyr[i] * (weight ? (float)weight[i] : 1.f);
        sg += g;
        sgu = fmaf(g, ((float)xr[i] - m) * s, sgu);
    }
    sg = row_sum<16>(sg, red, 0) / (float)n;
    sgu = row_sum<16>(sgu, red, 1) / (float)n;
    for (int i = threadIdx.x; i < n; i += kLoopThreads) {
        const float g = (float)dyr[i] * (weight ? (float)weight[i] : 1.f);
        dx[row * n + i] = (T)(s * (g - sg - ((float)xr[i] - m) * s * sgu));
    }
}

// Column sums of 256 columns over every gridDim.y-th row.
template <typename T>
__global__ __launch_bounds__(256) void norm_loop_cols_kernel(
    int64_t rows, int n, const T *__restrict__ x, int64_t x_stride, const T *__restrict__ dy,
    int64_t dy_stride, const float *__restrict__ mean, const float *__restrict__ rstd,
    float *__restrict__ partial) {
    const int at = blockIdx.x * 256 + threadIdx.x;
    if (at >= n) return;
    float dw = 0.f, db = 0.f;
    for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) {
        const float g = (float)dy[row * dy_stride + at];
        dw = fmaf(g, ((float)x[row * x_stride + at] - mean[row]) * rstd[row], dw);
        db += g;
    }
    float *out = partial + (int64_t)blockIdx.y * 2 * n;
    out[at] = dw;
    out[n + at] = db;
}

// -------------------------------------------------------------------- host
constexpr int kNormRegElems = 32;                      // elements a thread holds, at most
constexpr int64_t kNormLoopWidth = 16 * 64 * 16;       // 16 waves of 16 elements a thread
// As many as run at once: with more, the last ones run in a half empty GPU
// (forward of 65280 rows of 1024 bfloat16: 45 us with 1024, 51 with 2048).
constexpr int64_t kNormGroups = 1024;
constexpr int64_t kNormStreamBytes = 32 << 20;         // the L2 caches' together

// Workgroups of the forward and backward: rows are dealt round robin.
static int64_t norm_rows_at_once(int64_t n) { return n <= 64 * kNormRegElems ? 4 : 1; }
static int64_t norm_groups(int64_t rows, int64_t n) {
    const int64_t g = ceil_div(rows, norm_rows_at_once(n));
    return g < kNormGroups ? g : kNormGroups;
}
// Column sums held at once: one (2, n) set a workgroup.
static int64_t norm_parts(int64_t rows, int64_t n) {
    if (n > kNormLoopWidth) return rows < 64 ? rows : 64;
    return norm_groups(rows, n);
}

// Calls f<C, kWaves>() for the narrowest form that holds a row of n.
template <typename T, typename F>
static void norm_form(int64_t n, F f) {
    constexpr int V = kVec<T>;
    if (n <= 64 * 8) {
        f(std::integral_constant<int, 8 / V>{}, std::integral_constant<int, 1>{});
    } else if (n <= 64 * 16) {
        f(std::integral_constant<int, 16 / V>{}, std::integral_constant<int, 1>{});
    } else if (n <= 64 * 32) {
        f(std::integral_constant<int, 32 / V>{}, std::integral_constant<int, 1>{});
    } else if (n <= 4 * 64 * 16) {
        f(std::integral_constant<int, 16 / V>{}, std::integral_constant<int, 4>{});
    } else if (n <= 4 * 64 * 32) {
        f(std::integral_constant<int, 32 / V>{}, std::integral_constant<int, 4>{});
    } else {
        f(std::integral_constant<int, 16 / V>{}, std::integral_constant<int, 16>{});
    }
}

struct NormFwd {
    int64_t rows, n, x_stride;
    const void *x, *weight, *bias;
    float eps;
    void *y;
    float *mean, *rstd;
};

template <typename T, typename W>
static int32_t norm_forward(const NormFwd &a, hipStream_t st) {
    const T *x = static_cast<const T *>(a.x);
    const W *w = static_cast<const W *>(a.weight), *b = static_cast<const W *>(a.bias);
    T *y = static_cast<T *>(a.y);
    TimedScope ts("layer_norm_fwd", st);
    if (a.n > kNormLoopWidth) {
        norm_loop_fwd_kernel<T, W><<<(unsigned)a.rows, kLoopThreads, 0, st>>>(
            (int)a.n, x, a.x_stride, w, b, a.eps, y, a.mean, a.rstd);
    } else {
        const int64_t groups = norm_groups(a.rows, a.n);
        norm_form<T>(a.n, [&](auto c, auto waves) {
            constexpr int C = decltype(c)::value, kWaves = decltype(waves)::value;
            norm_fwd_kernel<T, W, C, kWaves><<<(unsigned)groups, kNormThreads<kWaves>, 0, st>>>(
                a.rows, (int)a.n, x, a.x_stride, w, b, a.eps, y, a.mean, a.rstd);
        });
    }
    MG_LAUNCHED("norm_fwd_kernel");
    return MG_OK;
}

struct NormBwd {
    int64_t rows, n, x_stride, dy_stride;
    const void *x, *dy, *weight;
    const float *mean, *rstd;
    void *dx, *dweight, *dbias;
    float *partial;
};

template <typename T, typename W>
static int32_t norm_backward(const NormBwd &a, hipStream_t st) {
    const T *x = static_cast<const T *>(a.x), *dy = static_cast<const T *>(a.dy);
    const W *w = static_cast<const W *>(a.weight);
    T *dx = static_cast<T *>(a.dx);
    const int64_t parts = norm_parts(a.rows, a.n);
    {
        TimedScope ts("layer_norm_bwd", st);
        if (a.n > kNormLoopWidth) {
            if (dx)
                norm_loop_dx_kernel<T, W><<<(unsigned)a.rows, kLoopThreads, 0, st>>>(
                    (int)a.n, x, a.x_stride, dy, a.dy_stride, w, a.mean, a.rstd, dx);
            if (a.partial)
                norm_loop_cols_kernel<T>
                    <<<dim3((unsigned)ceil_div(a.n, 256), (unsigned)parts), 256, 0, st>>>(
                        a.rows, (int)a.n, x, a.x_stride, dy, a.dy_stride, a.mean, a.rstd,
                        a.partial);
        } else {
            norm_form<T>(a.n, [&](auto c, auto waves) {
                constexpr int C = decltype(c)::value, kWaves = decltype(waves)::value;
                const auto go = [&](auto kernel) {
                    kernel<<<(unsigned)parts, kNormThreads<kWaves>, 0, st>>>(
                        a.rows, (int)a.n, x, a.x_stride, dy, a.dy_stride, w, a.mean, a.rstd, dx,
                        a.partial);
                };
                if (a.rows * a.n * (int64_t)sizeof(T) > kNormStreamBytes)
                    go(norm_bwd_kernel<T, W, C, kWaves, true>);
                else
                    go(norm_bwd_kernel<T, W, C, kWaves, false>);
            });
        }
        MG_LAUNCHED("norm_bwd_kernel");
    }
    if (a.partial) {
        TimedScope ts("layer_norm_join", st);
        norm_join_kernel<W><<<dim3((unsigned)ceil_div(a.n, kJoinCols), 2), kJoinThreads, 0, st>>>(
            a.partial, (int)parts, (int)a.n, static_cast<W *>(a.dweight),
            static_cast<W *>(a.dbias));
        MG_LAUNCHED("norm_join_kernel");
    }
    return MG_OK;
}

// f<T, W>() for the types of x and of the weights.
template <typename F>
static int32_t norm_types(int32_t dtype, int32_t wtype, F f) {
    if (dtype == MG_F32) return f(float{}, float{});
    if (dtype == MG_BF16) return wtype == MG_F32 ? f(bf16_t{}, float{}) : f(bf16_t{}, bf16_t{});
    return wtype == MG_F32 ? f(f16_t{}, float{}) : f(f16_t{}, f16_t{});
}

static int32_t norm_check(const char *who, int64_t rows, int64_t n, int32_t dtype, int32_t wtype) {
    MG_REQUIRE(rows >= 0 && rows < (int64_t(1) << 31), "%s: %lld rows", who, (long long)rows);
    MG_REQUIRE(n >= 1 && n <= (int64_t(1) << 24), "%s: rows of %lld elements; 1 to 2^24 are taken",
               who, (long long)n);
    MG_REQUIRE(n <= kNormLoopWidth || grid_fits(rows, kLoopThreads),
               "%s: %lld rows of %lld elements are too many for one call", who, (long long)rows,
               (long long)n);
    MG_REQUIRE(type_known(dtype), "%s: type code %d", who, dtype);
    MG_REQUIRE(wtype == MG_F32 || wtype == dtype,
               "%s: the weights must be float32 or of the input's type", who);
    return MG_OK;
}

}  // namespace mg

extern "C" {

int32_t mg_layer_norm_forward(int64_t rows, int64_t width, int32_t dtype, const void *x,
                              int64_t x_stride, int32_t weight_dtype, const void *weight,
                              const void *bias, float eps, void *y, float *mean, float *rstd,
                              mg_stream_t stream) {
    using namespace mg;
    int32_t rc = norm_check("mg_layer_norm_forward", rows, width, dtype, weight_dtype);
    if (rc != MG_OK) return rc;
    if (rows == 0) return MG_OK;
    MG_REQUIRE(x && y, "mg_layer_norm_forward: x and y are needed");
    MG_REQUIRE((mean == nullptr) == (rstd == nullptr),
               "mg_layer_norm_forward: mean and rstd go together");
    const NormFwd a{rows, width, x_stride, x, weight, bias, eps, y, mean, rstd};
    hipStream_t st = as_stream(stream);
    return norm_types(dtype, weight_dtype, [&](auto t, auto w) {
        return norm_forward<decltype(t), decltype(w)>(a, st);
    });
}

int64_t mg_layer_norm_backward_workspace_bytes(int64_t rows, int64_t width) {
    if (rows <= 0 || width <= 0) return 0;
    return mg::norm_parts(rows, width) * 2 * width * 4;
}

int32_t mg_layer_norm_backward(int64_t rows, int64_t width, int32_t dtype, const void *x,
                               int64_t x_stride, const void *dy, int64_t dy_stride,
                               int32_t weight_dtype, const void *weight, const float *mean,
                               const float *rstd, void *dx, void *dweight, void *dbias,
                               void *workspace, int64_t workspace_bytes, mg_stream_t stream) {
    using namespace mg;
    int32_t rc = norm_check("mg_layer_norm_backward", rows, width, dtype, weight_dtype);
    if (rc != MG_OK) return rc;
    const bool cols = dweight || dbias;
    MG_REQUIRE(rows > 0 || !cols,
               "mg_layer_norm_backward: the weights' gradients of no rows are zeros");
    if (rows == 0) return MG_OK;
    MG_REQUIRE(x && dy && mean && rstd, "mg_layer_norm_backward: x, dy, mean and rstd are needed");
    MG_REQUIRE(!cols || (workspace && workspace_bytes >=
                                          mg_layer_norm_backward_workspace_bytes(rows, width)),
               "mg_layer_norm_backward: workspace of %lld bytes, %lld needed",
               (long long)workspace_bytes,
               (long long)mg_layer_norm_backward_workspace_bytes(rows, width));
    if (!dx && !cols) return MG_OK;
    const NormBwd a{rows, width,  x_stride, dy_stride, x,       dy,   weight,
                    mean, rstd,   dx,       dweight,   dbias,   cols ? static_cast<float *>(workspace) : nullptr};
    hipStream_t st = as_stream(stream);
    return norm_types(dtype, weight_dtype, [&](auto t, auto w) {
        return norm_backward<decltype(t), decltype(w)>(a, st);
    });
}

}  // extern "C"
