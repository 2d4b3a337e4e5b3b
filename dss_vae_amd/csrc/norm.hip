// Layer norm, forward and backward (HBM-bound: forward reads x and writes y, backward reads x and dy and writes dx).
//
// A row lives in registers between its one read and its one write: TPR threads hold E elements each, in granules of VEC
// (granule i of thread t covers columns (i * TPR + t) * VEC ..).  Mean first, then the centred squares: two reductions over
// registers, no cancellation as in E[x^2] - E[x]^2.  Up to 64 x 16 columns a row belongs to ONE wave (shuffles only); wider
// rows take 256 threads, rows beyond 256 x 32 columns (or unaligned ones that need more than 32 elements a thread) are
// walked three times by a block of 1024 (the repeats hit L2).
//   xh = (x - mean) rstd ; y = xh w + b
//   dx = rstd (w dy - mean(w dy) - xh mean(w dy xh)) ; dw = sum_rows dy xh ; db = sum_rows dy
// The column sums: a block walks rows blockIdx, + gridDim, ... and keeps dw / db of its columns in registers; its row groups
// meet in LDS, one [2, D] partial per block goes to the workspace and a second launch adds the partials in order
// (no atomics: the same bits every time).
#include "elem.h"

namespace {

constexpr int FWD_THREADS = 256;
constexpr int BWD_THREADS = 512;
constexpr int LOOP_THREADS = 1024;

template <typename T, int VEC, int TPR, int E>
__global__ __launch_bounds__(FWD_THREADS) void layer_norm_fwd_kernel(const T* __restrict__ x, int64_t ldx,
                                                                      const void* __restrict__ w,
                                                                      const void* __restrict__ b, int param_f32,
                                                                      int64_t rows, int D, float eps, T* __restrict__ y,
                                                                      int64_t ldy, float* __restrict__ stats) {
    constexpr int NV = E / VEC, RPB = FWD_THREADS / TPR;
    __shared__ float red[FWD_THREADS / 64];
    const int t = threadIdx.x % TPR, g = threadIdx.x / TPR;
    float wv[E], bv[E];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * TPR + t) * VEC;
        float a[VEC], d[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) { a[j] = 1.f; d[j] = 0.f; }
        if (c < D) {
            if (w) load_param<T, VEC>(a, w, param_f32, c);
            if (b) load_param<T, VEC>(d, b, param_f32, c);
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) { wv[i * VEC + j] = a[j]; bv[i * VEC + j] = d[j]; }
    }
    const float n = (float)D;  // (divided by, not multiplied with 1 / n: the mean of equal values is that value)
    // (every row group of the block makes the same number of trips: the row sums may hold barriers)
    for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < rows; r0 += (int64_t)gridDim.x * RPB) {
        const int64_t r = r0 + g;
        const bool live = r < rows;
        const T* xr = x + (live ? r : 0) * ldx;
        Gran<T, VEC> v[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * TPR + t) * VEC;
            if (c < D) v[i].load(xr + c);
            else v[i].zero();
        }
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < VEC; ++j) s += v[i].get(j);
        const float mean = row_sum<TPR>(s, red) / n;
        float q = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const bool in = (i * TPR + t) * VEC < D;
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const float d = v[i].get(j) - mean;
                q += in ? d * d : 0.f;
            }
        }
        const float rstd = 1.f / sqrtf(row_sum<TPR>(q, red) / n + eps);
        if (!live) continue;
        T* yr = y + r * ldy;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * TPR + t) * VEC;
            if (c >= D) continue;
            Gran<T, VEC> o;
#pragma unroll
            for (int j = 0; j < VEC; ++j) o.set(j, (v[i].get(j) - mean) * rstd * wv[i * VEC + j] + bv[i * VEC + j]);
            o.store(yr + c);
        }
        if (stats && t == 0) {
            stats[2 * r] = mean;
            stats[2 * r + 1] = rstd;
        }
    }
}

// rows too wide for the registers: one block per row, three walks
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
        const float mean = row_sum<LOOP_THREADS>(s, red) / (float)D;
        float q = 0.f;
        for (int64_t c = threadIdx.x; c < D; c += LOOP_THREADS) {
            const float d = (float)xr[c] - mean;
            q += d * d;
        }
        const float rstd = 1.f / sqrtf(row_sum<LOOP_THREADS>(q, red) / (float)D + eps);
        for (int64_t c = threadIdx.x; c < D; c += LOOP_THREADS) {
            float a[1] = {1.f}, d[1] = {0.f};
            if (w) load_param<T, 1>(a, w, param_f32, c);
            if (b) load_param<T, 1>(d, b, param_f32, c);
            yr[c] = (T)(((float)xr[c] - mean) * rstd * a[0] + d[0]);
        }
        if (stats && threadIdx.x == 0) {
            stats[2 * r] = mean;
            stats[2 * r + 1] = rstd;
        }
    }
}

// BWD_THREADS / TPR rows per trip; `part` [gridDim][2][D] (NULL: dx only)
template <typename T, int VEC, int TPR, int E>
__global__ __launch_bounds__(BWD_THREADS, E == 32 ? 2 : 4) void layer_norm_bwd_kernel(const T* __restrict__ x, int64_t ldx,
                                                            const T* __restrict__ dy, int64_t lddy,
                                                            const void* __restrict__ w, int param_f32,
                                                            const float* __restrict__ stats, int64_t rows, int D,
                                                            T* __restrict__ dx, int64_t lddx,
                                                            float* __restrict__ part) {
    constexpr int NV = E / VEC, RPB = BWD_THREADS / TPR;
    __shared__ float red[2 * BWD_THREADS / 64];
    extern __shared__ float sums[];  // [RPB - 1][2][TPR * E]
    const int t = threadIdx.x % TPR, g = threadIdx.x / TPR;
    float wv[E], dwa[E], dba[E];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * TPR + t) * VEC;
        float a[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) a[j] = 1.f;
        if (w && c < D) load_param<T, VEC>(a, w, param_f32, c);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            wv[i * VEC + j] = a[j];
            dwa[i * VEC + j] = dba[i * VEC + j] = 0.f;
        }
    }
    const float inv = 1.f / (float)D;
    for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < rows; r0 += (int64_t)gridDim.x * RPB) {
        const int64_t r = r0 + g;
        const bool live = r < rows;
        const T* xr = x + (live ? r : 0) * ldx;
        const T* gr = dy + (live ? r : 0) * lddy;
        Gran<T, VEC> xv[NV], gv[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * TPR + t) * VEC;
            if (live && c < D) {
                xv[i].load(xr + c);
                gv[i].load(gr + c);
            } else {
                xv[i].zero();
                gv[i].zero();
            }
        }
        // a dead row group (or column) adds zeros: dy = 0 and, with x = 0 and finite statistics, a finite xh
        const float mean = live ? stats[2 * r] : 0.f, rstd = live ? stats[2 * r + 1] : 0.f;
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const bool in = live && (i * TPR + t) * VEC < D;
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const int e = i * VEC + j;
                const float xh = in ? (xv[i].get(j) - mean) * rstd : 0.f, d = gv[i].get(j);
                dwa[e] += d * xh;
                dba[e] += d;
                s1 += d * wv[e];
                s2 += d * wv[e] * xh;
            }
        }
        if constexpr (TPR <= 64) {
            s1 = row_sum<TPR>(s1, red) * inv;
            s2 = row_sum<TPR>(s2, red) * inv;
        } else {  // both sums behind one pair of barriers
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) {
                s1 += __shfl_xor(s1, o, 64);
                s2 += __shfl_xor(s2, o, 64);
            }
            constexpr int NW = TPR / 64;
            const int wave = threadIdx.x >> 6, w0 = wave / NW * NW;
            __syncthreads();
            if ((threadIdx.x & 63) == 0) {
                red[2 * wave] = s1;
                red[2 * wave + 1] = s2;
            }
            __syncthreads();
            s1 = s2 = 0.f;
#pragma unroll
            for (int i = 0; i < NW; ++i) {
                s1 += red[2 * (w0 + i)];
                s2 += red[2 * (w0 + i) + 1];
            }
            s1 *= inv;
            s2 *= inv;
        }
        if (!live || !dx) continue;
        T* o = dx + r * lddx;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * TPR + t) * VEC;
            if (c >= D) continue;
            Gran<T, VEC> ov;
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const int e = i * VEC + j;
                const float xh = (xv[i].get(j) - mean) * rstd;
                ov.set(j, rstd * (gv[i].get(j) * wv[e] - s1 - xh * s2));
            }
            ov.store(o + c);
        }
    }
    if (!part) return;
    // the block's row groups, added in order by group 0
    if constexpr (RPB > 1) {
        if (g > 0) {
            float* q = sums + (int64_t)(g - 1) * 2 * TPR * E;
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
            const float* q = sums + (int64_t)k * 2 * TPR * E;
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
        if (c >= D) continue;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
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
            float a[1] = {1.f};
            if (w) load_param<T, 1>(a, w, param_f32, c);
            const float gw = (float)gr[c] * a[0];
            s1 += gw;
            s2 += gw * ((float)xr[c] - mean) * rstd;
        }
        s1 = row_sum<LOOP_THREADS>(s1, red) / (float)D;
        s2 = row_sum<LOOP_THREADS>(s2, red) / (float)D;
        for (int64_t c = threadIdx.x; c < D; c += LOOP_THREADS) {
            float a[1] = {1.f};
            if (w) load_param<T, 1>(a, w, param_f32, c);
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

// dw / db [D] = sum over n partials [2, D]: 32 columns per block, 32 threads share a column
template <typename T>
__global__ __launch_bounds__(1024) void layer_norm_sum_kernel(const float* __restrict__ part, int n, int D, void* dw,
                                                              void* db, int param_f32) {
    __shared__ float red[32][33];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const int64_t c = (int64_t)blockIdx.x * 32 + tx;  // column of [dw | db]
    float s = 0.f;
    if (c < 2 * (int64_t)D)
        for (int i = ty; i < n; i += 32) s += part[(int64_t)i * 2 * D + c];
    red[ty][tx] = s;
    __syncthreads();
    if (ty != 0 || c >= 2 * (int64_t)D) return;
#pragma unroll
    for (int i = 1; i < 32; ++i) s += red[i][tx];
    void* o = c < D ? dw : db;
    const int64_t k = c < D ? c : c - D;
    if (!o) return;
    if (param_f32) reinterpret_cast<float*>(o)[k] = s;
    else reinterpret_cast<T*>(o)[k] = (T)s;
}

// Which kernel a width takes: the smallest of the shapes below that covers D columns (its granules tile TPR x E exactly).
struct Shape { int tpr, e; };
inline Shape shape_of(int D) {
    static const Shape all[] = {{64, 8}, {64, 16}, {256, 8}, {256, 16}, {256, 32}};
    for (const Shape& s : all)
        if ((int64_t)s.tpr * s.e >= D) return s;
    return {0, 0};  // the wide form
}

// blocks of the backward kernel: two a CU
inline int64_t bwd_blocks(int64_t rows, int D) {
    const Shape s = shape_of(D);
    if (s.tpr == 0) return rows < 256 ? (rows < 1 ? 1 : rows) : 256;  // row slices of the column sums
    const int rpb = BWD_THREADS / s.tpr;
    const int64_t need = (rows + rpb - 1) / rpb, most = 2 * (int64_t)device_cus();
    return need < 1 ? 1 : need < most ? need : most;
}

// elements per granule: 16 or 8 bytes where every row and parameter starts on that boundary and D divides, else one
inline int pick_vec(int es, int D, bool param_f32, const void* const* ptrs, const int64_t* lds, int n,
                    const void* const* params, int np) {
    for (int bytes = 16; bytes >= 8; bytes /= 2) {
        const int vec = bytes / es;
        if (vec == 1 || D % vec) continue;
        bool ok = true;
        for (int i = 0; i < n; ++i) ok = ok && (!ptrs[i] || (aligned_to(ptrs[i], bytes) && lds[i] % vec == 0));
        for (int i = 0; i < np; ++i) ok = ok && (!params[i] || aligned_to(params[i], param_f32 ? 4 : bytes));
        if (ok) return vec;
    }
    return 1;
}

template <typename T, int VEC>
int fwd_launch(const T* x, int64_t ldx, const void* w, const void* b, int pf, int64_t rows, int D, float eps, T* y,
               int64_t ldy, float* stats, hipStream_t s) {
    const Shape sh = shape_of(D);
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
    hipLaunchKernelGGL((layer_norm_fwd_kernel<T, VEC, TPR, E>), grid, dim3(FWD_THREADS), 0, s, x, ldx, w, b, pf, rows, D, eps, \
                       y, ldy, stats)
    GO(64, 8); GO(64, 16); GO(256, 8); GO(256, 16); GO(256, 32);
#undef GO
    DSSVAE_CHECK_LAUNCH();
    return DSSVAE_OK;
}

template <typename T, int VEC>
int bwd_launch(const T* x, int64_t ldx, const T* dy, int64_t lddy, const void* w, int pf, const float* stats, int64_t rows,
               int D, T* dx, int64_t lddx, void* dw, void* db, float* part, hipStream_t s) {
    const Shape sh = shape_of(D);
    const int64_t blocks = bwd_blocks(rows, D);
    if (sh.tpr == 0) {
        const int64_t most = 4 * (int64_t)device_cus();
        if (dx) {
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
#define GO(TPR, E)                                                                                              \
    if (sh.tpr == TPR && sh.e == E) {                                                                               \
        constexpr int lds = (BWD_THREADS / TPR - 1) * 2 * TPR * E * 4;                                                       \
        auto kern = layer_norm_bwd_kernel<T, VEC, TPR, E>;                                                      \
        static const hipError_t allowed = hipFuncSetAttribute(                                                      \
            reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, lds);                  \
        if (allowed != hipSuccess) return (int)allowed;                                                             \
        hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(BWD_THREADS), part ? lds : 0, s, x, ldx, dy, lddy, w, pf, stats, rows, D, \
                           dx, lddx, part);                                                                         \
    }
        GO(64, 8) GO(64, 16) GO(256, 8) GO(256, 16) GO(256, 32)
#undef GO
        DSSVAE_CHECK_LAUNCH();
    }
    if (part) {
        hipLaunchKernelGGL((layer_norm_sum_kernel<T>), dim3((unsigned)((2 * (int64_t)D + 31) / 32)), dim3(1024), 0, s, part,
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
    const void* ptrs[] = {x, y};
    const int64_t lds[] = {ldx, ldy};
    const void* params[] = {w, b};
    const int es = elem_size(dtype);
    const int pf = param_f32 || dtype == DSSVAE_F32;
    const int vec = pick_vec(es, D, pf, ptrs, lds, 2, params, 2);
#define GO(T, V)                                                                                                    \
    if (vec == V) return fwd_launch<T, V>((const T*)x, ldx, w, b, pf, rows, D, eps, (T*)y, ldy, stats, s)
    if (dtype == DSSVAE_F32) { GO(float, 4); GO(float, 2); GO(float, 1); }
    else if (dtype == DSSVAE_BF16) { GO(bf16_t, 8); GO(bf16_t, 4); GO(bf16_t, 1); }
    else { GO(f16_t, 8); GO(f16_t, 4); GO(f16_t, 1); }
#undef GO
    return DSSVAE_EINVAL;
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
    const void* ptrs[] = {x, dy, dx};
    const int64_t lds[] = {ldx, lddy, lddx};
    const void* params[] = {w};
    const int es = elem_size(dtype);
    const int pf = param_f32 || dtype == DSSVAE_F32;
    const int vec = pick_vec(es, D, pf, ptrs, lds, 3, params, 1);
    float* part = cols ? (float*)workspace : nullptr;
#define GO(T, V)                                                                                                    \
    if (vec == V)                                                                                                   \
    return bwd_launch<T, V>((const T*)x, ldx, (const T*)dy, lddy, w, pf, stats, rows, D, (T*)dx, lddx, dw, db, part, s)
    if (dtype == DSSVAE_F32) { GO(float, 4); GO(float, 2); GO(float, 1); }
    else if (dtype == DSSVAE_BF16) { GO(bf16_t, 8); GO(bf16_t, 4); GO(bf16_t, 1); }
    else { GO(f16_t, 8); GO(f16_t, 4); GO(f16_t, 1); }
#undef GO
    return DSSVAE_EINVAL;
}
