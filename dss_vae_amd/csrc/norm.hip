// Layer norm, forward and backward (HBM-bound: forward reads x and writes y, backward reads x and dy and writes dx).
//
// A row lives in registers between its one read and its one write: TPR threads hold E elements each, in granules of 16 bytes
// (granule i of thread t covers columns (i * TPR + t) * VEC ..).  Rows may start anywhere and end inside a granule: loads take
// any alignment, the last granule goes by elements (27513 x 1581 bf16: 50 us forward, 85 us backward; with element loads 69 and
// 136 us).  Mean first, then the deviations and their squares, no cancellation as in E[x^2] - E[x]^2.  Partial sums of values with a
// common offset are rounded to the offset's bits, and the mean of a row of 99999.9 comes out 0.01 off: the deviations from it are exact, and
// their mean corrects it to half a step.  The squares are corrected by it too, or, where it is not small beside them (equal values), taken
// again about the new mean (32768 x 2048 bf16: 56 us, 50 with the first mean, 58 with the squares always taken again).
// Forward, up to 1024 columns a row belongs to one wave or a quarter of one (shuffles only); wider rows take 256 threads.
// Backward keeps E at 8 up to 4096 columns (its column sums cost 2 E registers more) and gives a row up to 512 threads.  Rows
// wider than 8192 columns are walked four times (backward twice) by a block of 1024 (the repeats hit L2).
//   xh = (x - mean) rstd ; y = xh w + b
//   dx = rstd (w dy - mean(w dy) - xh mean(w dy xh)) ; dw = sum_rows dy xh ; db = sum_rows dy
// The column sums: a block walks rows blockIdx, + gridDim, ... and keeps dw / db of its columns in registers; its row groups
// meet in LDS, one [2, D] partial per block goes to the workspace and a second launch adds the partials in order
// (no atomics: the same bits every time).
// Measured: 32768 x 2048 bf16 forward 56 us (4.8 TB/s), backward 78 us (5.2 TB/s) and 6 us for the partials.
#include "elem.h"

namespace {

constexpr int FWD_THREADS = 256;
constexpr int BWD_THREADS = 512;
constexpr int LOOP_THREADS = 1024;

// f(x - mean) for the granule's columns in front of D
template <bool WHOLE, typename T, int VEC, typename F>
__device__ __forceinline__ void deviations(const GranU<T, VEC>& g, int c, int D, float mean, F f) {
    if (WHOLE ? c < D : c + VEC <= D) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) f(g.get(j) - mean);
    } else if (!WHOLE) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) f(c + j < D ? g.get(j) - mean : 0.f);
    }
}

template <typename T, int TPR, int E, bool WHOLE>
__global__ __launch_bounds__(FWD_THREADS) void layer_norm_fwd_kernel(const T* __restrict__ x, int64_t ldx,
                                                                      const void* __restrict__ w,
                                                                      const void* __restrict__ b, int param_f32,
                                                                      int64_t rows, int D, float eps, T* __restrict__ y,
                                                                      int64_t ldy, float* __restrict__ stats) {
    constexpr int VEC = 16 / (int)sizeof(T), NV = E / VEC, RPB = FWD_THREADS / TPR;
    __shared__ float red[2 * FWD_THREADS / 64];
    const int t = threadIdx.x % TPR, g = threadIdx.x / TPR;
    float wv[NV][VEC], bv[NV][VEC];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        load_param<WHOLE, T, VEC>(wv[i], w, param_f32, (i * TPR + t) * VEC, D, 1.f);
        load_param<WHOLE, T, VEC>(bv[i], b, param_f32, (i * TPR + t) * VEC, D, 0.f);
    }
    const float n = (float)D;
    // (every row group of the block makes the same number of trips: the row sums may hold barriers)
    for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < rows; r0 += (int64_t)gridDim.x * RPB) {
        const int64_t r = r0 + g;
        const bool live = r < rows;
        const T* xr = x + (live ? r : 0) * ldx;
        GranU<T, VEC> v[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) load_cols<WHOLE, T, VEC>(v[i], xr, (i * TPR + t) * VEC, D);
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < VEC; ++j) s += v[i].get(j);
        float mean = row_sum<TPR>(s, red) / n, q = 0.f;
        s = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
            deviations<WHOLE, T, VEC>(v[i], (i * TPR + t) * VEC, D, mean, [&](float d) {
                s += d;
                q += d * d;
            });
        row_sums<TPR>(s, q, red);
        const float off = s / n;
        mean += off;
        float var = q / n - off * off;
        if (!(off * off <= 0.01f * var)) {  // (the row alike) hardly any spread beside the first mean's error: squares about the new one
            q = 0.f;
#pragma unroll
            for (int i = 0; i < NV; ++i)
                deviations<WHOLE, T, VEC>(v[i], (i * TPR + t) * VEC, D, mean, [&](float d) { q += d * d; });
            var = row_sum<TPR>(q, red) / n;
        }
        const float rstd = 1.f / sqrtf(var + eps);
        if (!live) continue;
        T* yr = y + r * ldy;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            GranU<T, VEC> o;
#pragma unroll
            for (int j = 0; j < VEC; ++j) o.set(j, (v[i].get(j) - mean) * rstd * wv[i][j] + bv[i][j]);
            store_cols<WHOLE, T, VEC>(o, yr, (i * TPR + t) * VEC, D);
        }
        if (stats && t == 0) {
            stats[2 * r] = mean;
            stats[2 * r + 1] = rstd;
        }
    }
}

// rows too wide for the registers: one block per row, four walks
template <typename T>
__global__ __launch_bounds__(LOOP_THREADS) void layer_norm_fwd_wide_kernel(const T* __restrict__ x, int64_t ldx,
                                                                            const void* __restrict__ w,
                                                                            const void* __restrict__ b, int param_f32,
                                                                            int64_t rows, int D, float eps,
                                                                            T* __restrict__ y, int64_t ldy,
                                                                            float* __restrict__ stats) {
    __shared__ float red[LOOP_THREADS / 64];
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const T* xr = x + r * ldx;
        T* yr = y + r * ldy;
        float s = 0.f;
        for (int64_t c = threadIdx.x; c < D; c += LOOP_THREADS) s += (float)xr[c];
        float mean = row_sum<LOOP_THREADS>(s, red) / (float)D, q = 0.f;
        s = 0.f;
        for (int64_t c = threadIdx.x; c < D; c += LOOP_THREADS) s += (float)xr[c] - mean;
        mean += row_sum<LOOP_THREADS>(s, red) / (float)D;
        for (int64_t c = threadIdx.x; c < D; c += LOOP_THREADS) {
            const float d = (float)xr[c] - mean;
            q += d * d;
        }
        const float rstd = 1.f / sqrtf(row_sum<LOOP_THREADS>(q, red) / (float)D + eps);
        for (int64_t c = threadIdx.x; c < D; c += LOOP_THREADS) {
            float a[1], d[1];
            load_param<true, T, 1>(a, w, param_f32, (int)c, D, 1.f);
            load_param<true, T, 1>(d, b, param_f32, (int)c, D, 0.f);
            yr[c] = (T)(((float)xr[c] - mean) * rstd * a[0] + d[0]);
        }
        if (stats && threadIdx.x == 0) {
            stats[2 * r] = mean;
            stats[2 * r + 1] = rstd;
        }
    }
}

// BWD_THREADS / TPR rows per trip; `part` [gridDim][2][D] (NULL: dx only)
template <typename T, int TPR, int E, bool WHOLE>
__global__ __launch_bounds__(BWD_THREADS, E > 8 ? 2 : 4) void layer_norm_bwd_kernel(const T* __restrict__ x, int64_t ldx,
                                                                        const T* __restrict__ dy, int64_t lddy,
                                                                        const void* __restrict__ w, int param_f32,
                                                                        const float* __restrict__ stats, int64_t rows, int D,
                                                                        T* __restrict__ dx, int64_t lddx,
                                                                        float* __restrict__ part) {
    constexpr int VEC = 16 / (int)sizeof(T), NV = E / VEC, RPB = BWD_THREADS / TPR;
    __shared__ float red[2 * BWD_THREADS / 64];
    __shared__ float sums[RPB > 1 ? (RPB - 1) * 2 * TPR * E : 1];  // [RPB - 1][2][E][TPR]
    const int t = threadIdx.x % TPR, g = threadIdx.x / TPR;
    float wv[NV][VEC], dwa[E], dba[E];
#pragma unroll
    for (int i = 0; i < NV; ++i) load_param<WHOLE, T, VEC>(wv[i], w, param_f32, (i * TPR + t) * VEC, D, 1.f);
#pragma unroll
    for (int e = 0; e < E; ++e) dwa[e] = dba[e] = 0.f;
    const float inv = 1.f / (float)D;
    for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < rows; r0 += (int64_t)gridDim.x * RPB) {
        const int64_t r = r0 + g;
        const bool live = r < rows;
        const T* xr = x + (live ? r : 0) * ldx;
        const T* gr = dy + (live ? r : 0) * lddy;
        GranU<T, VEC> xv[NV], gv[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * TPR + t) * VEC;
            if (WHOLE) {
                load_cols<true, T, VEC>(xv[i], xr, c, live ? D : 0);
                load_cols<true, T, VEC>(gv[i], gr, c, live ? D : 0);
            } else {
                load_near<T, VEC>(xv[i], xr, c, D);
                load_near<T, VEC>(gv[i], gr, c, D);
            }
        }
        // (columns behind D and rows behind the last: dy = 0, and x - mean that of a real column or dropped below)
        if (!WHOLE) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                trim<false, T, VEC>(xv[i], (i * TPR + t) * VEC, D);
                trim<true, T, VEC>(gv[i], (i * TPR + t) * VEC, D);
                if (!live) {
                    xv[i].zero();
                    gv[i].zero();
                }
            }
        }
        const float mean = live ? stats[2 * r] : 0.f, rstd = live ? stats[2 * r + 1] : 0.f;
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const bool in = !WHOLE || (i * TPR + t) * VEC < D;
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const int e = i * VEC + j;
                const float xh = in ? (xv[i].get(j) - mean) * rstd : 0.f, d = gv[i].get(j);
                dwa[e] += d * xh;
                dba[e] += d;
                s1 += d * wv[i][j];
                s2 += d * wv[i][j] * xh;
            }
        }
        row_sums<TPR>(s1, s2, red);
        s1 *= inv;
        s2 *= inv;
        if (!live || !dx) continue;
        T* o = dx + r * lddx;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            GranU<T, VEC> ov;
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const float xh = (xv[i].get(j) - mean) * rstd;
                ov.set(j, rstd * (gv[i].get(j) * wv[i][j] - s1 - xh * s2));
            }
            store_cols<WHOLE, T, VEC>(ov, o, (i * TPR + t) * VEC, D);
        }
    }
    if (!part) return;
    // the block's row groups, added in order by group 0
    if constexpr (RPB > 1) {
        if (g > 0) {
            float* q = sums + (g - 1) * 2 * TPR * E;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                q[e * TPR + t] = dwa[e];
                q[(E + e) * TPR + t] = dba[e];
            }
        }
        __syncthreads();
        if (g > 0) return;
#pragma unroll 1
        for (int k = 0; k < RPB - 1; ++k) {
            const float* q = sums + k * 2 * TPR * E;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                dwa[e] += q[e * TPR + t];
                dba[e] += q[(E + e) * TPR + t];
            }
        }
    }
    float* pw = part + (int64_t)blockIdx.x * 2 * D;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * TPR + t) * VEC;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            if (c + j >= D) continue;
            pw[c + j] = dwa[i * VEC + j];
            pw[D + c + j] = dba[i * VEC + j];
        }
    }
}

template <typename T>
__global__ __launch_bounds__(LOOP_THREADS) void layer_norm_bwd_wide_kernel(const T* __restrict__ x, int64_t ldx,
                                                                            const T* __restrict__ dy, int64_t lddy,
                                                                            const void* __restrict__ w, int param_f32,
                                                                            const float* __restrict__ stats,
                                                                            int64_t rows, int D, T* __restrict__ dx,
                                                                            int64_t lddx) {
    __shared__ float red[LOOP_THREADS / 64];
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const T* xr = x + r * ldx;
        const T* gr = dy + r * lddy;
        const float mean = stats[2 * r], rstd = stats[2 * r + 1];
        float s1 = 0.f, s2 = 0.f;
        for (int64_t c = threadIdx.x; c < D; c += LOOP_THREADS) {
            float a[1];
            load_param<true, T, 1>(a, w, param_f32, (int)c, D, 1.f);
            const float gw = (float)gr[c] * a[0];
            s1 += gw;
            s2 += gw * ((float)xr[c] - mean) * rstd;
        }
        s1 = row_sum<LOOP_THREADS>(s1, red) / (float)D;
        s2 = row_sum<LOOP_THREADS>(s2, red) / (float)D;
        for (int64_t c = threadIdx.x; c < D; c += LOOP_THREADS) {
            float a[1];
            load_param<true, T, 1>(a, w, param_f32, (int)c, D, 1.f);
            dx[r * lddx + c] = (T)(rstd * ((float)gr[c] * a[0] - s1 - ((float)xr[c] - mean) * rstd * s2));
        }
    }
}

// column sums of the wide form: grid (column tiles of 256, row slices); part [gridDim.y][2][D]
template <typename T>
__global__ __launch_bounds__(256) void layer_norm_cols_kernel(const T* __restrict__ x, int64_t ldx,
                                                              const T* __restrict__ dy, int64_t lddy,
                                                              const float* __restrict__ stats, int64_t rows, int D,
                                                              float* __restrict__ part) {
    const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (c >= D) return;
    float dw = 0.f, db = 0.f;
    for (int64_t r = blockIdx.y; r < rows; r += gridDim.y) {
        const float d = (float)dy[r * lddy + c];
        dw += d * ((float)x[r * ldx + c] - stats[2 * r]) * stats[2 * r + 1];
        db += d;
    }
    part[(int64_t)blockIdx.y * 2 * D + c] = dw;
    part[(int64_t)blockIdx.y * 2 * D + D + c] = db;
}

// dw / db [D] = sum over n partials [2, D]: 32 columns per block (and the next 32 a grid behind them), 32 threads share a column
template <typename T>
__global__ __launch_bounds__(1024) void layer_norm_sum_kernel(const float* __restrict__ part, int n, int D, void* dw,
                                                              void* db, int param_f32) {
    __shared__ float red[32][33];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    for (int64_t c0 = (int64_t)blockIdx.x * 32; c0 < 2 * (int64_t)D; c0 += (int64_t)gridDim.x * 32) {
        const int64_t c = c0 + tx;  // column of [dw | db]
        float s = 0.f;
        if (c < 2 * (int64_t)D)
            for (int i = ty; i < n; i += 32) s += part[(int64_t)i * 2 * D + c];
        __syncthreads();  // the sums of the columns before have been read
        red[ty][tx] = s;
        __syncthreads();
        void* o = c < D ? dw : db;
        if (ty != 0 || c >= 2 * (int64_t)D || !o) continue;
#pragma unroll
        for (int i = 1; i < 32; ++i) s += red[i][tx];
        const int64_t k = c < D ? c : c - D;
        if (param_f32) reinterpret_cast<float*>(o)[k] = s;
        else reinterpret_cast<T*>(o)[k] = (T)s;
    }
}

// Which kernel a width takes: the first shape that covers D columns; {0, 0}: the wide form.
struct Shape { int tpr, e; };
template <int N>
inline Shape shape_of(const Shape (&all)[N], int D) {
    for (const Shape& s : all)
        if ((int64_t)s.tpr * s.e >= D) return s;
    return {0, 0};
}
constexpr Shape FWD_SHAPES[] = {{16, 8}, {64, 8}, {64, 16}, {256, 8}, {256, 16}, {256, 32}};
constexpr Shape BWD_SHAPES[] = {{16, 8}, {64, 8}, {128, 8}, {256, 8}, {512, 8}, {512, 16}};

// blocks of the backward kernel: two a CU
inline int64_t bwd_blocks(int64_t rows, int D) {
    const Shape s = shape_of(BWD_SHAPES, D);
    if (s.tpr == 0) return rows < 256 ? (rows < 1 ? 1 : rows) : 256;  // row slices of the column sums
    const int rpb = BWD_THREADS / s.tpr;
    const int64_t need = (rows + rpb - 1) / rpb, most = 2 * (int64_t)device_cus();
    return need < 1 ? 1 : need < most ? need : most;
}

template <typename T, bool WHOLE>
int fwd_launch(const T* x, int64_t ldx, const void* w, const void* b, int pf, int64_t rows, int D, float eps, T* y,
               int64_t ldy, float* stats, hipStream_t s) {
    const Shape sh = shape_of(FWD_SHAPES, D);
    const int64_t most = 8 * (int64_t)device_cus();
    if (sh.tpr == 0) {
        const int64_t grid = rows < most ? rows : most;
        hipLaunchKernelGGL((layer_norm_fwd_wide_kernel<T>), dim3((unsigned)grid), dim3(LOOP_THREADS), 0, s, x, ldx, w, b, pf,
                           rows, D, eps, y, ldy, stats);
        DSSVAE_CHECK_LAUNCH();
        return DSSVAE_OK;
    }
    const int rpb = FWD_THREADS / sh.tpr;
    const int64_t need = (rows + rpb - 1) / rpb;
    const dim3 grid((unsigned)(need < most ? need : most));
#define GO(TPR, E)                                                                                                  \
    if (sh.tpr == TPR && sh.e == E)                                                                                 \
    hipLaunchKernelGGL((layer_norm_fwd_kernel<T, TPR, E, WHOLE>), grid, dim3(FWD_THREADS), 0, s, x, ldx, w, b, pf, rows, D, eps, \
                       y, ldy, stats)
    GO(16, 8); GO(64, 8); GO(64, 16); GO(256, 8); GO(256, 16); GO(256, 32);
#undef GO
    DSSVAE_CHECK_LAUNCH();
    return DSSVAE_OK;
}

template <typename T, bool WHOLE>
int bwd_launch(const T* x, int64_t ldx, const T* dy, int64_t lddy, const void* w, int pf, const float* stats, int64_t rows,
               int D, T* dx, int64_t lddx, void* dw, void* db, float* part, hipStream_t s) {
    const Shape sh = shape_of(BWD_SHAPES, D);
    const int64_t blocks = bwd_blocks(rows, D);
    if (sh.tpr == 0) {
        const int64_t most = 4 * (int64_t)device_cus();
        if (dx && rows > 0) {
            hipLaunchKernelGGL((layer_norm_bwd_wide_kernel<T>), dim3((unsigned)(rows < most ? rows : most)), dim3(LOOP_THREADS), 0,
                               s, x, ldx, dy, lddy, w, pf, stats, rows, D, dx, lddx);
            DSSVAE_CHECK_LAUNCH();
        }
        if (part) {
            hipLaunchKernelGGL((layer_norm_cols_kernel<T>), dim3((unsigned)((D + 255) / 256), (unsigned)blocks), dim3(256), 0, s, x, ldx,
                               dy, lddy, stats, rows, D, part);
            DSSVAE_CHECK_LAUNCH();
        }
    } else {
#define GO(TPR, E)                                                                                                  \
    if (sh.tpr == TPR && sh.e == E)                                                                                 \
    hipLaunchKernelGGL((layer_norm_bwd_kernel<T, TPR, E, WHOLE>), dim3((unsigned)blocks), dim3(BWD_THREADS), 0, s, x, ldx, dy, lddy, w, pf, \
                       stats, rows, D, dx, lddx, part)
        GO(16, 8); GO(64, 8); GO(128, 8); GO(256, 8); GO(512, 8); GO(512, 16);
#undef GO
        DSSVAE_CHECK_LAUNCH();
    }
    if (part) {
        // (a launch holds fewer than 2^32 threads, 64 to a column here: rows of 2^26 and more columns take several trips)
        const int64_t groups = (2 * (int64_t)D + 31) / 32, most = 1 << 20;
        hipLaunchKernelGGL((layer_norm_sum_kernel<T>), dim3((unsigned)(groups < most ? groups : most)), dim3(1024), 0, s, part,
                           (int)blocks, D, dw, db, pf);
        DSSVAE_CHECK_LAUNCH();
    }
    return DSSVAE_OK;
}

}  // namespace

extern "C" int dssvae_layer_norm_fwd(const void* x, int64_t ldx, int dtype, const void* w, const void* b, int param_f32,
                                     int64_t rows, int D, float eps, void* y, int64_t ldy, float* stats, void* stream) {
    if (!dtype_ok(dtype) || rows < 0 || D < 1 || D > (1 << 30) || ldx < D || ldy < D || !(eps >= 0.f)) return DSSVAE_EINVAL;
    if (rows == 0) return DSSVAE_OK;
    if (!x || !y) return DSSVAE_EINVAL;
    hipStream_t s = (hipStream_t)stream;
    const int pf = param_f32 || dtype == DSSVAE_F32;
#define GO(T)                                                                                                       \
    return D % (16 / (int)sizeof(T)) == 0                                                                           \
               ? fwd_launch<T, true>((const T*)x, ldx, w, b, pf, rows, D, eps, (T*)y, ldy, stats, s)                \
               : fwd_launch<T, false>((const T*)x, ldx, w, b, pf, rows, D, eps, (T*)y, ldy, stats, s)
    if (dtype == DSSVAE_F32) GO(float);
    if (dtype == DSSVAE_BF16) GO(bf16_t);
    GO(f16_t);
#undef GO
}

extern "C" int64_t dssvae_layer_norm_bwd_workspace_bytes(int64_t rows, int D) {
    if (rows < 0 || D < 1) return DSSVAE_EINVAL;
    return bwd_blocks(rows, D) * 2 * (int64_t)D * 4;
}

extern "C" int dssvae_layer_norm_bwd(const void* x, int64_t ldx, int dtype, const void* dy, int64_t lddy, const void* w,
                                     int param_f32, const float* stats, int64_t rows, int D, void* dx, int64_t lddx,
                                     void* dw, void* db, void* workspace, int64_t workspace_bytes, void* stream) {
    if (!dtype_ok(dtype) || rows < 0 || D < 1 || D > (1 << 30) || ldx < D || lddy < D || (dx && lddx < D)) return DSSVAE_EINVAL;
    if (rows > 0 && (!x || !dy || !stats)) return DSSVAE_EINVAL;
    const bool cols = dw || db;
    if (cols && (!workspace || workspace_bytes < dssvae_layer_norm_bwd_workspace_bytes(rows, D))) return DSSVAE_EINVAL;
    if (!cols && (!dx || rows == 0)) return DSSVAE_OK;
    hipStream_t s = (hipStream_t)stream;
    const int pf = param_f32 || dtype == DSSVAE_F32;
    float* part = cols ? (float*)workspace : nullptr;
#define GO(T)                                                                                                       \
    return D % (16 / (int)sizeof(T)) == 0                                                                           \
               ? bwd_launch<T, true>((const T*)x, ldx, (const T*)dy, lddy, w, pf, stats, rows, D, (T*)dx, lddx, dw, db, part, s) \
               : bwd_launch<T, false>((const T*)x, ldx, (const T*)dy, lddy, w, pf, stats, rows, D, (T*)dx, lddx, dw, db, part, s)
    if (dtype == DSSVAE_F32) GO(float);
    if (dtype == DSSVAE_BF16) GO(bf16_t);
    GO(f16_t);
#undef GO
}
