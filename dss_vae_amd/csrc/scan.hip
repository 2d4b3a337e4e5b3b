// Gated linear recurrence over time, forward and backward (HBM-bound).
//
//   a_t = sigmoid(z_t), n_t = tanh(v_t) or v_t          x[b, t] = (z_t | v_t), 2H wide
//   h_t = a_t h_{t-1} + (1 - a_t) n_t                   the GRU's update without its reset gate and its W_hh
//   E_t = a_t (dout_t + E_{t+1})                        gradient that reaches h_{t-1}; E_T = dh_last, dh0 = E_0
//   D_t = dout_t + E_{t+1}: dz = D (1 - a)(h_t - n), dv = D (1 - a)(1 - n^2 | 1)      (a (h_{t-1} - n) = h_t - n)
//
// Both recurrences are affine maps y -> A y + B per channel and compose: (A2, B2) after (A1, B1) = (A1 A2, A2 B1 + B2).
// A block owns LPR * VEC neighbouring channels of one sequence and walks time in chunks of 128 steps: thread (g, l)
// holds KT consecutive steps of VEC channels in registers, the block's groups are joined by a shuffle scan inside each
// wave and through LDS across the waves, the chunk's state is carried in registers.  One read of x (and
// dout), one write.  The forward pass leaves the state at each chunk's start ("checkpoint", 1/128 of out); backward rebuilds
// h inside the chunk from it, in fp32, and never reads out.
// Few sequences and channels, many steps: the time axis is cut into segments; a first launch reads the segment's inputs
// for its (A, B) per channel, the second starts each segment from the composition of those before it (backward: behind it).
// Steps at or behind a sequence's length are the identity (A = 1, B = 0): the state is kept, out and dx are zero there.
#include "elem.h"

namespace {

constexpr int CHUNK = 128;
// threads of a block: a thread's share of a chunk is 16 values of a 16-byte granule in either width
template <typename T> constexpr int NT = sizeof(T) == 4 ? 256 : 512;
constexpr int STEP_THREADS = 256;

__device__ __forceinline__ float sigmoid_f(float x) {
    return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.4426950408889634f * x));
}
// (absolute error ~2e-7: hardware exp2 and rcp)
__device__ __forceinline__ float tanh_f(float x) {
    return 1.f - 2.f * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(2.8853900817779268f * x));
}

struct Dims {
    const int32_t* lengths;
    int64_t xb, xt;      // strides of x [B, T, 2H]
    int64_t ob, ot;      // strides of out / dout [B, T, H]
    int64_t gb, gt;      // strides of dx [B, T, 2H]
    int B, T, H, reverse;
    int tiles, nchunk, segs, seg_chunks;  // channel tiles, chunks of the time axis, its segments and their chunks
};

// what a block works on: channel tile, sequence, segment
struct Where { int c0, b, seg, len; };
template <int LPR, int VEC>
__device__ __forceinline__ Where where(const Dims& d) {
    const int wid = xcd_remap(blockIdx.x, gridDim.x);  // neighbouring tiles, which may share cache lines, on one XCD
    Where w;
    w.c0 = (wid % d.tiles) * LPR * VEC;
    const int rest = wid / d.tiles;
    w.b = rest % d.B;
    w.seg = rest / d.B;
    int len = d.lengths ? d.lengths[w.b] : d.T;
    w.len = len < 0 ? 0 : len > d.T ? d.T : len;
    return w;
}

// An affine map per channel, applied through a whole block.  In: each thread's own map (its KT steps) and `carry`, the state
// that enters the chunk, held by the lanes as one value per channel (channel lane % (LPR * VEC), the same in every wave).
// Out: y, the state that enters this thread's steps, and the carry behind the chunk.  FWD: earlier steps first, else later
// ones.  Lanes scan their wave's groups by shuffles, the waves' totals meet in LDS (one barrier), and every wave runs the NW
// totals over the carry by itself: 2 NW floats read per lane, where reading them per thread and channel cost VEC times that.
// prod (or NULL): the product of the chunk's A, per channel.
template <int NW, int LPR, int VEC, bool FWD>
__device__ __forceinline__ void block_scan(float (&A)[VEC], float (&B)[VEC], float& carry, float (&y)[VEC],
                                           float2* lds /* [NW][LPR * VEC] */, float* prod = nullptr) {
    constexpr int GW = 64 / LPR, CH = LPR * VEC;  // groups per wave, channels
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l = lane % LPR, g = lane / LPR;
    const int pos = FWD ? g : GW - 1 - g, wpos = FWD ? wave : NW - 1 - wave;
#pragma unroll
    for (int o = 1; o < GW; o <<= 1) {
        const int src = FWD ? lane - o * LPR : lane + o * LPR;
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            const float pA = __shfl(A[v], src & 63, 64), pB = __shfl(B[v], src & 63, 64);
            if (pos >= o) {
                B[v] = A[v] * pB + B[v];
                A[v] = A[v] * pA;
            }
        }
    }
    if (pos == GW - 1) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) lds[wpos * CH + l * VEC + v] = make_float2(A[v], B[v]);
    }
    __syncthreads();
    float mine = carry, run = carry, pa = 1.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
        const float2 q = lds[w * CH + lane % CH];
        if (w == wpos) mine = run;
        run = q.x * run + q.y;
        pa *= q.x;
    }
    carry = run;
    if (prod) *prod *= pa;
    const int src = FWD ? lane - LPR : lane + LPR;
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
        const float pA = __shfl(A[v], src & 63, 64), pB = __shfl(B[v], src & 63, 64), m = __shfl(mine, l * VEC + v, 64);
        y[v] = pos > 0 ? pA * m + pB : m;
    }
}

// state entering segment `seg` of channel c: y0 through the maps of the segments before it (fwd) or behind it
__device__ __forceinline__ float enter(float y, const float* __restrict__ maps, const Dims& d, int b, int seg, int c, bool fwd) {
    for (int j = fwd ? 0 : d.segs - 1; j != seg; j += fwd ? 1 : -1) {
        const float* m = maps + ((int64_t)b * d.segs + j) * 2 * d.H + c;
        y = m[0] * y + m[d.H];
    }
    return y;
}

// One chunk's loads for this thread: granules of (z | v) of its KT steps; steps that are not live are not read.
template <typename T, int VEC, int LPR, int KT, bool HALF>
struct Steps {
    Gran<T, VEC> z[KT], v[HALF ? 1 : KT], g[KT];
    unsigned live;   // bit k: step k is live
    __device__ __forceinline__ void load(const T* x, const T* dout, const Dims& d, const Where& w, int chunk, int c, bool on) {
        live = 0;
        const int s0 = chunk * CHUNK + (int)(threadIdx.x / LPR) * KT;
#pragma unroll
        for (int k = 0; k < KT; ++k) {
            const int s = s0 + k, t = d.reverse ? d.T - 1 - s : s;
            const bool ok = on && s < d.T && t < w.len;
            live |= ok ? 1u << k : 0u;
            if (ok) {
                const T* p = x + t * d.xt + c;
                z[k].load(p);
                if constexpr (!HALF) v[k].load(p + d.H);
                if (dout) g[k].load(dout + t * d.ot + c);
                else g[k].zero();
            } else {
                z[k].zero();
                if constexpr (!HALF) v[k].zero();
                g[k].zero();
            }
        }
    }
};

// ---- segment maps: (A, B) of the forward recurrence, or of E (BWD) ------------------------------------------------
template <typename T, int VEC, int LPR, bool TANH, bool BWD>
__global__ __launch_bounds__(NT<T>) void gated_scan_maps_kernel(const T* __restrict__ x, const T* __restrict__ dout, Dims d,
                                                                  float* __restrict__ maps) {
    constexpr int NW = NT<T> / 64, KT = CHUNK * LPR / NT<T>;
    __shared__ float2 lds[2][NW * LPR * VEC];
    const Where w = where<LPR, VEC>(d);
    if (w.seg == (BWD ? 0 : d.segs - 1)) return;  // nobody starts behind the last one
    const int l = threadIdx.x % LPR, c = w.c0 + l * VEC;
    const bool on = c < d.H;
    const T* xb = x + w.b * d.xb;
    const T* gb = dout ? dout + w.b * d.ob : nullptr;
    const int cc = w.c0 + (int)(threadIdx.x & 63) % (LPR * VEC);  // the channel whose carry this lane holds
    const bool writer = cc < d.H && threadIdx.x < LPR * VEC;
    float SA = 1.f, SB = 0.f;
    const int first = w.seg * d.seg_chunks, last = min(d.nchunk, first + d.seg_chunks);
    for (int i = 0; i < last - first; ++i) {
        const int chunk = BWD ? last - 1 - i : first + i;
        Steps<T, VEC, LPR, KT, BWD> s;
        s.load(xb, BWD ? gb : nullptr, d, w, chunk, c, on);
        float A[VEC], B[VEC], y[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) { A[v] = 1.f; B[v] = 0.f; }
#pragma unroll
        for (int kk = 0; kk < KT; ++kk) {
            const int k = BWD ? KT - 1 - kk : kk;
            const bool ok = (s.live >> k) & 1;
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                const float a = sigmoid_f(s.z[k].get(v));
                if (ok) {
                    if constexpr (BWD) {
                        B[v] = a * (s.g[k].get(v) + B[v]);
                    } else {
                        const float n = TANH ? tanh_f(s.v[k].get(v)) : s.v[k].get(v);
                        B[v] = a * B[v] + (1.f - a) * n;
                    }
                    A[v] *= a;
                }
            }
        }
        block_scan<NW, LPR, VEC, !BWD>(A, B, SB, y, lds[i & 1], &SA);
    }
    if (writer) {
        float* m = maps + ((int64_t)w.b * d.segs + w.seg) * 2 * d.H + cc;
        m[0] = SA;
        m[d.H] = SB;
    }
}

// ---- forward ---------------------------------------------------------------------------------------------------------
template <typename T, int VEC, int LPR, bool TANH>
__global__ __launch_bounds__(NT<T>) void gated_scan_fwd_kernel(const T* __restrict__ x, Dims d, const float* __restrict__ h0,
                                                                 const float* __restrict__ maps, T* __restrict__ out,
                                                                 float* __restrict__ h_last, float* __restrict__ ckpt) {
    constexpr int NW = NT<T> / 64, KT = CHUNK * LPR / NT<T>;
    __shared__ float2 lds[2][NW * LPR * VEC];
    const Where w = where<LPR, VEC>(d);
    const int l = threadIdx.x % LPR, c = w.c0 + l * VEC;
    const bool on = c < d.H;
    const T* xb = x + w.b * d.xb;
    T* ob = out + w.b * d.ob;
    const int cc = w.c0 + (int)(threadIdx.x & 63) % (LPR * VEC);  // the channel whose carry this lane holds
    const bool con = cc < d.H, writer = con && threadIdx.x < LPR * VEC;
    float h = h0 && con ? h0[(int64_t)w.b * d.H + cc] : 0.f;
    if (d.segs > 1 && con) h = enter(h, maps, d, w.b, w.seg, cc, true);
    const int first = w.seg * d.seg_chunks, last = min(d.nchunk, first + d.seg_chunks);
    Steps<T, VEC, LPR, KT, false> s, next;
    next.load(xb, nullptr, d, w, first, c, on);
    for (int chunk = first; chunk < last; ++chunk) {
        s = next;
        if (chunk + 1 < last) next.load(xb, nullptr, d, w, chunk + 1, c, on);
        float a[KT][VEC], bn[KT][VEC], A[VEC], B[VEC], y[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) { A[v] = 1.f; B[v] = 0.f; }
#pragma unroll
        for (int k = 0; k < KT; ++k) {
            const bool ok = (s.live >> k) & 1;
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                const float ak = sigmoid_f(s.z[k].get(v)), n = TANH ? tanh_f(s.v[k].get(v)) : s.v[k].get(v);
                a[k][v] = ok ? ak : 1.f;
                bn[k][v] = ok ? (1.f - ak) * n : 0.f;
                B[v] = a[k][v] * B[v] + bn[k][v];
                A[v] *= a[k][v];
            }
        }
        if (ckpt && writer) ckpt[((int64_t)w.b * d.nchunk + chunk) * d.H + cc] = h;
        block_scan<NW, LPR, VEC, true>(A, B, h, y, lds[chunk & 1]);
        const int s0 = chunk * CHUNK + (int)(threadIdx.x / LPR) * KT;
#pragma unroll
        for (int k = 0; k < KT; ++k) {
            const bool ok = (s.live >> k) & 1;
            Gran<T, VEC> o;
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                y[v] = a[k][v] * y[v] + bn[k][v];
                o.set(v, ok ? y[v] : 0.f);
            }
            const int st = s0 + k, t = d.reverse ? d.T - 1 - st : st;
            if (on && st < d.T) o.store(ob + t * d.ot + c);
        }
    }
    if (w.seg == d.segs - 1 && h_last && writer) h_last[(int64_t)w.b * d.H + cc] = h;
}

// ---- backward --------------------------------------------------------------------------------------------------------
template <typename T, int VEC, int LPR, bool TANH>
__global__ __launch_bounds__(NT<T>) void gated_scan_bwd_kernel(const T* __restrict__ x, const T* __restrict__ dout, Dims d,
                                                                 const float* __restrict__ ckpt,
                                                                 const float* __restrict__ dh_last,
                                                                 const float* __restrict__ maps, T* __restrict__ dx,
                                                                 float* __restrict__ dh0) {
    constexpr int NW = NT<T> / 64, KT = CHUNK * LPR / NT<T>;
    __shared__ float2 lds[2][2][NW * LPR * VEC];
    const Where w = where<LPR, VEC>(d);
    const int l = threadIdx.x % LPR, c = w.c0 + l * VEC;
    const bool on = c < d.H;
    const T* xb = x + w.b * d.xb;
    const T* gb = dout ? dout + w.b * d.ob : nullptr;
    T* db = dx + w.b * d.gb;
    const int cc = w.c0 + (int)(threadIdx.x & 63) % (LPR * VEC);  // the channel whose carry this lane holds
    const bool con = cc < d.H, writer = con && threadIdx.x < LPR * VEC;
    float E = dh_last && con ? dh_last[(int64_t)w.b * d.H + cc] : 0.f;
    if (d.segs > 1 && con) E = enter(E, maps, d, w.b, w.seg, cc, false);
    const int first = w.seg * d.seg_chunks, last = min(d.nchunk, first + d.seg_chunks);
    for (int chunk = last - 1; chunk >= first; --chunk) {
        Steps<T, VEC, LPR, KT, false> s;
        s.load(xb, gb, d, w, chunk, c, on);
        float hc = con ? ckpt[((int64_t)w.b * d.nchunk + chunk) * d.H + cc] : 0.f;
        float a[KT][VEC], n[KT][VEC], A[VEC], B[VEC], F[VEC], G[VEC], y[VEC], e[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) { A[v] = 1.f; B[v] = 0.f; G[v] = 0.f; }
#pragma unroll
        for (int k = 0; k < KT; ++k) {
            const bool ok = (s.live >> k) & 1;
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                const float ak = sigmoid_f(s.z[k].get(v));
                n[k][v] = TANH ? tanh_f(s.v[k].get(v)) : s.v[k].get(v);
                a[k][v] = ok ? ak : 1.f;
                B[v] = a[k][v] * B[v] + (ok ? (1.f - ak) * n[k][v] : 0.f);
                A[v] *= a[k][v];
            }
        }
#pragma unroll
        for (int k = KT - 1; k >= 0; --k) {
            const bool ok = (s.live >> k) & 1;
#pragma unroll
            for (int v = 0; v < VEC; ++v) G[v] = ok ? a[k][v] * (s.g[k].get(v) + G[v]) : G[v];
        }
#pragma unroll
        for (int v = 0; v < VEC; ++v) F[v] = A[v];
        block_scan<NW, LPR, VEC, true>(A, B, hc, y, lds[chunk & 1][0]);
        block_scan<NW, LPR, VEC, false>(F, G, E, e, lds[chunk & 1][1]);
        float h[KT][VEC];  // h_t
#pragma unroll
        for (int k = 0; k < KT; ++k) {
            const bool ok = (s.live >> k) & 1;
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                y[v] = ok ? a[k][v] * y[v] + (1.f - a[k][v]) * n[k][v] : y[v];
                h[k][v] = y[v];
            }
        }
        const int s0 = chunk * CHUNK + (int)(threadIdx.x / LPR) * KT;
#pragma unroll
        for (int k = KT - 1; k >= 0; --k) {
            const bool ok = (s.live >> k) & 1;
            Gran<T, VEC> oz, on_;
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                const float D = s.g[k].get(v) + e[v], q = D * (1.f - a[k][v]);
                oz.set(v, ok ? q * (h[k][v] - n[k][v]) : 0.f);
                on_.set(v, ok ? (TANH ? q * (1.f - n[k][v] * n[k][v]) : q) : 0.f);
                e[v] = ok ? a[k][v] * D : e[v];
            }
            const int st = s0 + k, t = d.reverse ? d.T - 1 - st : st;
            if (on && st < d.T) {
                oz.store(db + t * d.gt + c);
                on_.store(db + t * d.gt + d.H + c);
            }
        }
    }
    if (w.seg == 0 && dh0 && writer) dh0[(int64_t)w.b * d.H + cc] = E;
}

// ---- one token: h' = a h + (1 - a) n, out = h' rounded to T; h_out may be h -------------------------------------------
template <typename T, int VEC, bool TANH>
__global__ __launch_bounds__(STEP_THREADS) void gated_step_kernel(const T* __restrict__ x, int64_t xb, const float* h, int B, int H,
                                                             T* __restrict__ out, int64_t ob, float* h_out) {
    const int per = H / VEC;
    const int64_t i = (int64_t)blockIdx.x * STEP_THREADS + threadIdx.x;
    if (i >= (int64_t)B * per) return;
    const int64_t b = i / per;
    const int c = (int)(i % per) * VEC;
    Gran<T, VEC> z, v, o;
    z.load(x + b * xb + c);
    v.load(x + b * xb + H + c);
    float hv[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) hv[j] = h ? h[b * H + c + j] : 0.f;
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
        const float a = sigmoid_f(z.get(j)), n = TANH ? tanh_f(v.get(j)) : v.get(j);
        hv[j] = a * hv[j] + (1.f - a) * n;
        o.set(j, hv[j]);
    }
    o.store(out + b * ob + c);
#pragma unroll
    for (int j = 0; j < VEC; ++j) h_out[b * H + c + j] = hv[j];
}

// Segments of the time axis.  One while the tiles (128 bytes of channels each) alone give two blocks a CU: the segment maps
// cost a second read of the inputs.
inline int plan_segs(int B, int T, int H, int es) {
    const int64_t blocks = (int64_t)B * (((int64_t)H * es + 127) / 128), nchunk = ((int64_t)T + CHUNK - 1) / CHUNK;
    const int64_t cus = device_cus();
    if (blocks >= 2 * cus || nchunk <= 2) return 1;
    int64_t segs = (4 * cus + blocks - 1) / blocks;
    if (segs > nchunk) segs = nchunk;
    const int64_t per = (nchunk + segs - 1) / segs;
    return (int)((nchunk + per - 1) / per);
}

inline int pick_vec(int es, int H, const void* const* ptrs, const int64_t* strides, int n) {
    for (int bytes = 16; bytes >= 8; bytes /= 2) {
        const int vec = bytes / es;
        if (H % vec) continue;
        bool ok = true;
        for (int i = 0; i < n; ++i)
            ok = ok && (!ptrs[i] || (aligned_to(ptrs[i], bytes) && strides[2 * i] % vec == 0 && strides[2 * i + 1] % vec == 0));
        if (ok) return vec;
    }
    return 1;
}

template <typename T, int VEC, int LPR, bool TANH>
int fwd_launch(const T* x, Dims d, const float* h0, T* out, float* h_last, float* ckpt, float* maps, hipStream_t s) {
    d.tiles = (d.H + LPR * VEC - 1) / (LPR * VEC);
    const int64_t grid = (int64_t)d.tiles * d.B * d.segs;
    if (grid > 0x7fffffff) return DSSVAE_ETOOBIG;
    if (d.segs > 1) {
        hipLaunchKernelGGL((gated_scan_maps_kernel<T, VEC, LPR, TANH, false>), dim3((unsigned)grid), dim3(NT<T>), 0, s, x,
                           (const T*)nullptr, d, maps);
        DSSVAE_CHECK_LAUNCH();
    }
    hipLaunchKernelGGL((gated_scan_fwd_kernel<T, VEC, LPR, TANH>), dim3((unsigned)grid), dim3(NT<T>), 0, s, x, d, h0, maps, out,
                       h_last, ckpt);
    DSSVAE_CHECK_LAUNCH();
    return DSSVAE_OK;
}

template <typename T, int VEC, int LPR, bool TANH>
int bwd_launch(const T* x, const T* dout, Dims d, const float* ckpt, const float* dh_last, T* dx, float* dh0, float* maps,
               hipStream_t s) {
    d.tiles = (d.H + LPR * VEC - 1) / (LPR * VEC);
    const int64_t grid = (int64_t)d.tiles * d.B * d.segs;
    if (grid > 0x7fffffff) return DSSVAE_ETOOBIG;
    if (d.segs > 1) {
        hipLaunchKernelGGL((gated_scan_maps_kernel<T, VEC, LPR, false, true>), dim3((unsigned)grid), dim3(NT<T>), 0, s, x, dout, d,
                           maps);
        DSSVAE_CHECK_LAUNCH();
    }
    hipLaunchKernelGGL((gated_scan_bwd_kernel<T, VEC, LPR, TANH>), dim3((unsigned)grid), dim3(NT<T>), 0, s, x, dout, d, ckpt,
                       dh_last, maps, dx, dh0);
    DSSVAE_CHECK_LAUNCH();
    return DSSVAE_OK;
}

// a granule of 16 bytes: 8 lanes cover 128 bytes of channels; 8 bytes or one element: 16 lanes
#define DSSVAE_SCAN_VECS(CALL, T, V16, V8)                       \
    do {                                                         \
        if (vec == V16) { if (tanh) return CALL(T, V16, 8, true); return CALL(T, V16, 8, false); }   \
        if (vec == V8) { if (tanh) return CALL(T, V8, 16, true); return CALL(T, V8, 16, false); }    \
        if (tanh) return CALL(T, 1, 16, true);                   \
        return CALL(T, 1, 16, false);                            \
    } while (0)
#define DSSVAE_SCAN_TYPES(CALL)                                  \
    do {                                                         \
        if (dtype == DSSVAE_F32) DSSVAE_SCAN_VECS(CALL, float, 4, 2);    \
        if (dtype == DSSVAE_BF16) DSSVAE_SCAN_VECS(CALL, bf16_t, 8, 4);  \
        DSSVAE_SCAN_VECS(CALL, f16_t, 8, 4);                     \
    } while (0)

int bad_dims(int dtype, int B, int T, int H, int64_t xb, int64_t xt) {
    if (!dtype_ok(dtype) || B < 0 || T < 0 || H < 1 || H > (1 << 29)) return 1;
    if (T > 1 && xt < 2 * (int64_t)H) return 1;
    return B > 1 && xb < 2 * (int64_t)H;
}

Dims make_dims(const int32_t* lengths, int B, int T, int H, int reverse, int es) {
    Dims d{};
    d.lengths = lengths;
    d.B = B; d.T = T; d.H = H; d.reverse = reverse != 0;
    d.nchunk = (T + CHUNK - 1) / CHUNK;
    d.segs = plan_segs(B, T, H, es);
    d.seg_chunks = (d.nchunk + d.segs - 1) / d.segs;
    return d;
}

}  // namespace

extern "C" int dssvae_gated_scan_chunks(int T) { return T < 0 ? DSSVAE_EINVAL : (T + CHUNK - 1) / CHUNK; }

extern "C" int64_t dssvae_gated_scan_workspace_bytes(int B, int T, int H, int dtype) {
    if (!dtype_ok(dtype) || B < 0 || T < 0 || H < 1) return DSSVAE_EINVAL;
    const int segs = plan_segs(B, T, H, elem_size(dtype));
    return segs > 1 ? (int64_t)B * segs * 2 * H * 4 : 0;
}

extern "C" int dssvae_gated_scan_fwd(const void* x, int64_t xb, int64_t xt, int dtype, const float* h0,
                                     const int32_t* lengths, int reverse, int tanh_candidate, int B, int T, int H, void* out,
                                     int64_t ob, int64_t ot, float* h_last, float* checkpoints, void* workspace,
                                     int64_t workspace_bytes, void* stream) {
    if (bad_dims(dtype, B, T, H, xb, xt) || (T > 1 && ot < H) || (B > 1 && ob < H)) return DSSVAE_EINVAL;
    if (B == 0 || T == 0) return DSSVAE_OK;  // (no step: the caller's h_last is its h0)
    if (!x || !out || workspace_bytes < dssvae_gated_scan_workspace_bytes(B, T, H, dtype)) return DSSVAE_EINVAL;
    const int es = elem_size(dtype);
    Dims d = make_dims(lengths, B, T, H, reverse, es);
    if (d.segs > 1 && !workspace) return DSSVAE_EINVAL;
    d.xb = xb; d.xt = xt; d.ob = ob; d.ot = ot;
    const void* ptrs[] = {x, out};
    const int64_t strides[] = {B > 1 ? xb : 0, T > 1 ? xt : 0, B > 1 ? ob : 0, T > 1 ? ot : 0};
    const int vec = pick_vec(es, H, ptrs, strides, 2), tanh = tanh_candidate != 0;
    hipStream_t s = (hipStream_t)stream;
#define CALL(T_, V, L, TH) fwd_launch<T_, V, L, TH>((const T_*)x, d, h0, (T_*)out, h_last, checkpoints, (float*)workspace, s)
    DSSVAE_SCAN_TYPES(CALL);
#undef CALL
}

extern "C" int dssvae_gated_scan_bwd(const void* x, int64_t xb, int64_t xt, int dtype, const int32_t* lengths, int reverse,
                                     int tanh_candidate, const float* checkpoints, const void* dout, int64_t ob, int64_t ot,
                                     const float* dh_last, int B, int T, int H, void* dx, int64_t gb, int64_t gt, float* dh0,
                                     void* workspace, int64_t workspace_bytes, void* stream) {
    if (bad_dims(dtype, B, T, H, xb, xt) || bad_dims(dtype, B, T, H, gb, gt)) return DSSVAE_EINVAL;
    if (dout && ((T > 1 && ot < H) || (B > 1 && ob < H))) return DSSVAE_EINVAL;
    if (B == 0 || T == 0) return DSSVAE_OK;
    if (!x || !dx || !checkpoints || workspace_bytes < dssvae_gated_scan_workspace_bytes(B, T, H, dtype)) return DSSVAE_EINVAL;
    const int es = elem_size(dtype);
    Dims d = make_dims(lengths, B, T, H, reverse, es);
    if (d.segs > 1 && !workspace) return DSSVAE_EINVAL;
    d.xb = xb; d.xt = xt; d.ob = ob; d.ot = ot; d.gb = gb; d.gt = gt;
    const void* ptrs[] = {x, dout, dx};
    const int64_t strides[] = {B > 1 ? xb : 0, T > 1 ? xt : 0, B > 1 ? ob : 0, T > 1 ? ot : 0, B > 1 ? gb : 0, T > 1 ? gt : 0};
    const int vec = pick_vec(es, H, ptrs, strides, 3), tanh = tanh_candidate != 0;
    hipStream_t s = (hipStream_t)stream;
#define CALL(T_, V, L, TH)                                                                                             \
    bwd_launch<T_, V, L, TH>((const T_*)x, (const T_*)dout, d, checkpoints, dh_last, (T_*)dx, dh0, (float*)workspace, s)
    DSSVAE_SCAN_TYPES(CALL);
#undef CALL
}

namespace {

template <typename T, int VEC, bool TANH>
int step_launch(const T* x, int64_t xb, const float* h, int B, int H, T* out, int64_t ob, float* h_out, hipStream_t s) {
    const int64_t n = (int64_t)B * (H / VEC), grid = (n + STEP_THREADS - 1) / STEP_THREADS;
    if (grid > 0x7fffffff) return DSSVAE_ETOOBIG;
    hipLaunchKernelGGL((gated_step_kernel<T, VEC, TANH>), dim3((unsigned)grid), dim3(STEP_THREADS), 0, s, x, xb, h, B, H, out, ob, h_out);
    DSSVAE_CHECK_LAUNCH();
    return DSSVAE_OK;
}

}  // namespace

extern "C" int dssvae_gated_step(const void* x, int64_t xb, int dtype, const float* h, int tanh_candidate, int B, int H,
                                 void* out, int64_t ob, float* h_out, void* stream) {
    if (bad_dims(dtype, B, 1, H, xb, 2 * (int64_t)H) || (B > 1 && ob < H)) return DSSVAE_EINVAL;
    if (B == 0) return DSSVAE_OK;
    if (!x || !out || !h_out) return DSSVAE_EINVAL;
    const void* ptrs[] = {x, out};
    const int64_t strides[] = {B > 1 ? xb : 0, 0, B > 1 ? ob : 0, 0};
    const int vec = pick_vec(elem_size(dtype), H, ptrs, strides, 2), tanh = tanh_candidate != 0;
    hipStream_t s = (hipStream_t)stream;
#define CALL(T_, V, L, TH) step_launch<T_, V, TH>((const T_*)x, xb, h, B, H, (T_*)out, ob, h_out, s)
    DSSVAE_SCAN_TYPES(CALL);
#undef CALL
}
