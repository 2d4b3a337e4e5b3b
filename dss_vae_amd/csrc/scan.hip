// Gated linear recurrence over time, forward and backward (HBM-bound).
//
//   a_t = sigmoid(z_t), n_t = tanh(v_t) or v_t          x[b, t] = (z_t | v_t), 2H wide
//   h_t = a_t h_{t-1} + (1 - a_t) n_t                   the GRU's update without its reset gate and its W_hh
//   E_t = a_t (dout_t + E_{t+1})                        gradient that reaches h_{t-1}; E_T = dh_last, dh0 = E_0
//   D_t = dout_t + E_{t+1}: dz = D (1 - a)(h_t - n), dv = D (1 - a)(1 - n^2 | 1)      (a (h_{t-1} - n) = h_t - n)
//
// Both recurrences are affine maps y -> A y + B per channel and compose: (A2, B2) after (A1, B1) = (A1 A2, A2 B1 + B2).
// A block owns LPR * VEC neighbouring channels of one sequence and walks time in chunks: thread (g, l) holds KT consecutive
// steps of VEC channels in registers (16 values), the block's groups are joined by a shuffle scan inside each wave and
// through LDS across the waves, the chunk's state is carried in registers; the next chunk's loads are in flight meanwhile.
// One read of x (and dout), one write.  The forward pass leaves the state at each chunk's start ("checkpoint"); backward
// rebuilds h inside the chunk from it, in fp32, and never reads out.
// A granule is only 4 bytes: the scan costs log2(64 / LPR) shuffled compositions per channel and thread, so many steps per
// thread (KT = 8, fp32 16) beat wide granules (16-byte ones leave 2: 265 us for backward over 2 x 16384 x 2048 bf16, 8-byte
// ones 213 us, this form 153 us = 4.4 TB/s; forward 109 / 97 / 87 us = 4.6 TB/s).
// Too few tiles (128 bytes of channels each) to fill the chip: the time axis is cut into segments; a first launch reads the
// segment's inputs for its (A, B) per channel, the second starts each segment from the composition of those before it
// (backward: behind it).  Narrower tiles instead (32 bytes: no second read, but four blocks per cache line) took 192 us
// forward where the two launches take 158 us.
// Steps at or behind a sequence's length are the identity (A = 1, B = 0): the state is kept, out and dx are zero there.
#include "elem.h"

namespace {

// lanes per row; threads of a block and steps per thread: 128 steps a chunk in either width
constexpr int LPR = 32, CHUNK = 128;
template <typename T> constexpr int KT = sizeof(T) == 4 ? 16 : 8;
// Threads of a block: 256 or 512, and half or a quarter of that where the sequence ends in that part of its only chunk
// (512 x 30 x 2048 bf16, forward / backward: 128 / 230 us with the whole chunk, 36 / 66 us with a quarter of it)
template <typename T, int DIV> constexpr int NT = CHUNK / DIV * LPR / KT<T>;
constexpr int STEP_THREADS = 256;

// a = sigmoid(z) and b = 1 - a, each to its own accuracy: long memories are gates whose 1 - a is small, and the update and both
// gradients are proportional to it.  With w = exp(-|z|) the smaller of the two is w / (1 + w) and the larger one 1 minus it, rounded to
// nearest; 1 - a from a rounded a keeps a few bits (off by 1e-3 at z = 10, by all of it at 17), and what 1 + w and the reciprocal lose in
// an a close to 1 would add up over thousands of steps.  z = +-inf gives 1 and 0 exactly; NaN stays.
__device__ __forceinline__ void gate_f(float z, float& a, float& b) {
    const float w = __builtin_amdgcn_exp2f(-1.4426950408889634f * fabsf(z)), less = w * __builtin_amdgcn_rcpf(1.f + w), more = 1.f - less;
    a = z < 0.f ? less : more;
    b = z < 0.f ? more : less;
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
template <int VEC>
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
template <int NW, int VEC, bool FWD>
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

// This thread's steps of a chunk.  Pointers walk: one 64-bit add per row instead of a multiplication (which cost more than
// the recurrence).  Bit k of `live`: step k is inside [lo, hi).  Steps that are not are never read: z = +inf, v = 0 and dout = 0
// stand in their place, which makes a = 1 and (1 - a) n = 0 exactly, the identity, without a select in the arithmetic (these
// kernels are bound by the vector ALUs as much as by memory); only what is stored there is chosen.
template <typename T, int VEC, bool HALF, bool GRAD>
struct Steps {
    Gran<T, VEC> z[KT<T>], v[HALF ? 1 : KT<T>], g[GRAD ? KT<T> : 1];
    unsigned live;
    __device__ __forceinline__ void load(const T* px, int64_t dx, const T* pg, int64_t dg, int H, int s0, int lo, int hi) {
        live = 0;
#pragma unroll
        for (int k = 0; k < KT<T>; ++k) {
            const bool ok = s0 + k >= lo && s0 + k < hi;
            live |= ok ? 1u << k : 0u;
            if (ok) {
                z[k].load(px);
                if constexpr (!HALF) v[k].load(px + H);
                if constexpr (GRAD) {
                    if (pg) g[k].load(pg);
                    else g[k].zero();
                }
            } else {
#pragma unroll
                for (int j = 0; j < VEC; ++j) z[k].set(j, __builtin_huge_valf());
                if constexpr (!HALF) v[k].zero();
                if constexpr (GRAD) g[k].zero();
            }
            px += dx;
            if constexpr (GRAD) pg += pg ? dg : 0;
        }
    }
};

// Where a thread stands: channels c.. (clamped for loads), first step s0 of chunk `first`, live steps [lo, hi) of the
// sequence in walking order, and the carry's channel cc of its lane.
template <typename T, int VEC>
struct Thread {
    Where w;
    int c, cc, s0, lo, hi, first, last;
    bool on, con, writer;
    __device__ __forceinline__ explicit Thread(const Dims& d) {
        w = where<VEC>(d);
        c = w.c0 + (int)(threadIdx.x % LPR) * VEC;
        on = c < d.H;
        cc = w.c0 + (int)(threadIdx.x & 63) % (LPR * VEC);
        con = cc < d.H;
        writer = con && threadIdx.x < LPR * VEC;
        s0 = (int)(threadIdx.x / LPR) * KT<T>;
        lo = d.reverse ? d.T - w.len : 0;
        hi = d.reverse ? d.T : w.len;
        first = w.seg * d.seg_chunks;
        last = min(d.nchunk, first + d.seg_chunks);
    }
    // row of this thread's first step of a chunk, for strides (sb, st) of a tensor; `step` = the walk's stride
    __device__ __forceinline__ int64_t at(const Dims& d, int64_t sb, int64_t st, int chunk) const {
        const int s = chunk * CHUNK + s0;
        return w.b * sb + (int64_t)(d.reverse ? d.T - 1 - s : s) * st + (on ? c : 0);
    }
};
#define DSSVAE_SCAN_LOAD(steps, chunk_, pg)                                                                               \
    do {                                                                                                                  \
        const T* px_ = x + th.at(d, d.xb, d.xt, chunk_);                                                                  \
        const T* pg_ = (pg) ? (pg) + th.at(d, d.ob, d.ot, chunk_) : nullptr;                                              \
        steps.load(px_, dxs, pg_, dgs, d.H, (chunk_) * CHUNK + th.s0, th.lo, th.hi);                                       \
    } while (0)

// ---- segment maps: (A, B) of the forward recurrence, or of E (BWD) ------------------------------------------------
template <typename T, int VEC, bool TANH, bool BWD>
__global__ __launch_bounds__((NT<T, 1>)) void gated_scan_maps_kernel(const T* __restrict__ x, const T* __restrict__ dout, Dims d,
                                                                float* __restrict__ maps) {
    constexpr int NW = NT<T, 1> / 64, K = KT<T>;
    __shared__ float2 lds[2][NW * LPR * VEC];
    const Thread<T, VEC> th(d);
    if (th.w.seg == (BWD ? 0 : d.segs - 1)) return;  // nobody starts behind the last one
    const int64_t dxs = d.reverse ? -d.xt : d.xt, dgs = d.reverse ? -d.ot : d.ot;
    float SA = 1.f, SB = 0.f;
    Steps<T, VEC, BWD, BWD> s, next;
    const int n = th.last - th.first;
    DSSVAE_SCAN_LOAD(next, (BWD ? th.last - 1 : th.first), dout);
    for (int i = 0; i < n; ++i) {
        s = next;
        if (i + 1 < n) {
            const int chunk = BWD ? th.last - 2 - i : th.first + 1 + i;
            DSSVAE_SCAN_LOAD(next, chunk, dout);
        }
        float A[VEC], B[VEC], y[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) { A[v] = 1.f; B[v] = 0.f; }
#pragma unroll
        for (int kk = 0; kk < K; ++kk) {
            const int k = BWD ? K - 1 - kk : kk;
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                float a, b;
                gate_f(s.z[k].get(v), a, b);
                if constexpr (BWD) {
                    B[v] = a * (s.g[k].get(v) + B[v]);
                } else {
                    const float n = TANH ? tanh_f(s.v[k].get(v)) : s.v[k].get(v);
                    B[v] = a * B[v] + b * n;
                }
                A[v] *= a;
            }
        }
        block_scan<NW, VEC, !BWD>(A, B, SB, y, lds[i & 1], &SA);
    }
    if (th.writer) {
        float* m = maps + ((int64_t)th.w.b * d.segs + th.w.seg) * 2 * d.H + th.cc;
        m[0] = SA;
        m[d.H] = SB;
    }
}

// ---- forward ---------------------------------------------------------------------------------------------------------
template <typename T, int VEC, bool TANH, int DIV>
__device__ __forceinline__ void fwd_chunk(const Steps<T, VEC, false, false>& s, const Thread<T, VEC>& th,
                                          const Dims& d, int chunk, float& h, float2* lds, T* out) {
    constexpr int NW = NT<T, DIV> / 64, K = KT<T>;
    float a[K][VEC], bn[K][VEC], A[VEC], B[VEC], y[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) { A[v] = 1.f; B[v] = 0.f; }
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            const float n = TANH ? tanh_f(s.v[k].get(v)) : s.v[k].get(v);
            float b;
            gate_f(s.z[k].get(v), a[k][v], b);
            bn[k][v] = b * n;
            B[v] = a[k][v] * B[v] + bn[k][v];
            A[v] *= a[k][v];
        }
    }
    block_scan<NW, VEC, true>(A, B, h, y, lds);
    const int64_t dos = d.reverse ? -d.ot : d.ot;
    const int s0 = chunk * CHUNK + th.s0;
    T* po = out + th.at(d, d.ob, d.ot, chunk);
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const bool ok = (s.live >> k) & 1;
        Gran<T, VEC> o;
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            y[v] = a[k][v] * y[v] + bn[k][v];
            o.set(v, y[v]);
        }
        if (!ok) o.zero();
        if (th.on && s0 + k < d.T) o.store(po);
        po += dos;
    }
}

template <typename T, int VEC, bool TANH, int DIV>
__global__ __launch_bounds__((NT<T, DIV>)) void gated_scan_fwd_kernel(const T* __restrict__ x, Dims d, const float* __restrict__ h0,
                                                               const float* __restrict__ maps, T* __restrict__ out,
                                                               float* __restrict__ h_last, float* __restrict__ ckpt) {
    constexpr int NW = NT<T, DIV> / 64;
    __shared__ float2 lds[2][NW * LPR * VEC];
    const Thread<T, VEC> th(d);
    const int64_t dxs = d.reverse ? -d.xt : d.xt, dgs = 0, row = (int64_t)th.w.b * d.H + th.cc;
    float h = h0 && th.con ? h0[row] : 0.f;
    if (d.segs > 1 && th.con) h = enter(h, maps, d, th.w.b, th.w.seg, th.cc, true);
    Steps<T, VEC, false, false> s, next;
    const T* none = nullptr;
    DSSVAE_SCAN_LOAD(next, th.first, none);
    for (int chunk = th.first; chunk < th.last; ++chunk) {
        s = next;
        if (chunk + 1 < th.last) DSSVAE_SCAN_LOAD(next, (chunk + 1), none);
        if (ckpt && th.writer) ckpt[((int64_t)th.w.b * d.nchunk + chunk) * d.H + th.cc] = h;
        fwd_chunk<T, VEC, TANH, DIV>(s, th, d, chunk, h, lds[chunk & 1], out);
    }
    if (th.w.seg == d.segs - 1 && h_last && th.writer) h_last[row] = h;
}

// ---- backward --------------------------------------------------------------------------------------------------------
template <typename T, int VEC, bool TANH, int DIV>
__device__ __forceinline__ void bwd_chunk(const Steps<T, VEC, false, true>& s, const Thread<T, VEC>& th,
                                          const Dims& d, int chunk, float hc, float& E, float2* lds0, float2* lds1, T* dx) {
    constexpr int NW = NT<T, DIV> / 64, K = KT<T>;
    float a[K][VEC], b[K][VEC], n[K][VEC], dn[TANH ? K : 1][VEC], A[VEC], B[VEC], F[VEC], G[VEC], y[VEC], e[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) { A[v] = 1.f; B[v] = 0.f; G[v] = 0.f; }
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            gate_f(s.z[k].get(v), a[k][v], b[k][v]);
            if constexpr (TANH) n[k][v] = tanh_f(s.v[k].get(v), dn[k][v]);
            else n[k][v] = s.v[k].get(v);
            B[v] = a[k][v] * B[v] + b[k][v] * n[k][v];
            A[v] *= a[k][v];
        }
    }
#pragma unroll
    for (int k = K - 1; k >= 0; --k) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) G[v] = a[k][v] * (s.g[k].get(v) + G[v]);
    }
#pragma unroll
    for (int v = 0; v < VEC; ++v) F[v] = A[v];
    block_scan<NW, VEC, true>(A, B, hc, y, lds0);
    block_scan<NW, VEC, false>(F, G, E, e, lds1);
    float h[K][VEC];  // h_t - n_t = a_t (h_{t-1} - n_t)
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            h[k][v] = a[k][v] * (y[v] - n[k][v]);
            y[v] = a[k][v] * y[v] + b[k][v] * n[k][v];  // (h[k] + n would carry n's roundings into a small state)
        }
    }
    const int64_t dgs = d.reverse ? -d.gt : d.gt;
    const int s0 = chunk * CHUNK + th.s0;
    T* pd = dx + th.at(d, d.gb, d.gt, chunk) + (K - 1) * dgs;
#pragma unroll
    for (int k = K - 1; k >= 0; --k) {
        const bool ok = (s.live >> k) & 1;
        Gran<T, VEC> oz, on_;
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            const float D = s.g[k].get(v) + e[v], q = D * b[k][v];
            oz.set(v, q * h[k][v]);
            on_.set(v, TANH ? q * dn[TANH ? k : 0][v] : q);
            e[v] = a[k][v] * D;
        }
        if (!ok) {
            oz.zero();
            on_.zero();
        }
        if (th.on && s0 + k < d.T) {
            oz.store(pd);
            on_.store(pd + d.H);
        }
        pd -= dgs;
    }
}

template <typename T, int VEC, bool TANH, int DIV>
__global__ __launch_bounds__((NT<T, DIV>)) void gated_scan_bwd_kernel(const T* __restrict__ x, const T* __restrict__ dout, Dims d,
                                                               const float* __restrict__ ckpt,
                                                               const float* __restrict__ dh_last,
                                                               const float* __restrict__ maps, T* __restrict__ dx,
                                                               float* __restrict__ dh0) {
    constexpr int NW = NT<T, DIV> / 64;
    __shared__ float2 lds[2][2][NW * LPR * VEC];
    const Thread<T, VEC> th(d);
    const int64_t dxs = d.reverse ? -d.xt : d.xt, dgs = d.reverse ? -d.ot : d.ot, row = (int64_t)th.w.b * d.H + th.cc;
    float E = dh_last && th.con ? dh_last[row] : 0.f;
    if (d.segs > 1 && th.con) E = enter(E, maps, d, th.w.b, th.w.seg, th.cc, false);
    Steps<T, VEC, false, true> s, next;
    DSSVAE_SCAN_LOAD(next, (th.last - 1), dout);
    for (int chunk = th.last - 1; chunk >= th.first; --chunk) {
        s = next;
        if (chunk > th.first) DSSVAE_SCAN_LOAD(next, (chunk - 1), dout);
        const float hc = th.con ? ckpt[((int64_t)th.w.b * d.nchunk + chunk) * d.H + th.cc] : 0.f;
        float2 *l0 = lds[chunk & 1][0], *l1 = lds[chunk & 1][1];
        bwd_chunk<T, VEC, TANH, DIV>(s, th, d, chunk, hc, E, l0, l1, dx);
    }
    if (th.w.seg == 0 && dh0 && th.writer) dh0[row] = E;
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
        const float n = TANH ? tanh_f(v.get(j)) : v.get(j);
        float a, b;
        gate_f(z.get(j), a, b);
        hv[j] = a * hv[j] + b * n;
        o.set(j, hv[j]);
    }
    o.store(out + b * ob + c);
#pragma unroll
    for (int j = 0; j < VEC; ++j) h_out[b * H + c + j] = hv[j];
}

// Segments of the time axis: one while the tiles alone give more than half the CUs a block (the segment maps cost a second
// read of the inputs).  Measured, forward, T = 4096, bf16: 256 tiles 100 us whole, 147 us in segments; 128 tiles 82 / 76 us;
// 5 tiles x 16384 steps 304 / 33 us.
inline int plan_segs(int B, int T, int H, int es) {
    const int64_t cus = device_cus(), blocks = (int64_t)B * (((int64_t)H * es + 127) / 128);
    const int64_t nchunk = ((int64_t)T + CHUNK - 1) / CHUNK;
    if (blocks < 1 || 2 * blocks > cus || nchunk <= 2) return 1;
    int64_t segs = 2 * cus / blocks;
    if (segs > nchunk) segs = nchunk;
    const int64_t per = (nchunk + segs - 1) / segs;
    return (int)((nchunk + per - 1) / per);
}

// 16-bit channels move in pairs where every row starts on 4 bytes
inline int pick_vec(int es, int H, const void* const* ptrs, const int64_t* strides, int n) {
    if (es == 4 || H % 2) return 1;
    for (int i = 0; i < n; ++i)
        if (ptrs[i] && (!aligned_to(ptrs[i], 4) || strides[2 * i] % 2 || strides[2 * i + 1] % 2)) return 1;
    return 2;
}

template <typename T, int VEC, bool TANH>
int fwd_launch(const T* x, Dims d, const float* h0, T* out, float* h_last, float* ckpt, float* maps, hipStream_t s) {
    d.tiles = (d.H + LPR * VEC - 1) / (LPR * VEC);
    const int64_t grid = (int64_t)d.tiles * d.B * d.segs;
    if (!grid_fits(grid, NT<T, 1>)) return DSSVAE_ETOOBIG;
    if (d.segs > 1) {
        hipLaunchKernelGGL((gated_scan_maps_kernel<T, VEC, TANH, false>), dim3((unsigned)grid), dim3((NT<T, 1>)), 0, s, x,
                           (const T*)nullptr, d, maps);
        DSSVAE_CHECK_LAUNCH();
    }
#define GO(DIV)                                                                                                     \
    hipLaunchKernelGGL((gated_scan_fwd_kernel<T, VEC, TANH, DIV>), dim3((unsigned)grid), dim3((NT<T, DIV>)), 0, s, x, d, h0, maps, \
                       out, h_last, ckpt)
    if (d.T <= CHUNK / 4) GO(4);
    else if (d.T <= CHUNK / 2) GO(2);
    else GO(1);
#undef GO
    DSSVAE_CHECK_LAUNCH();
    return DSSVAE_OK;
}

template <typename T, int VEC, bool TANH>
int bwd_launch(const T* x, const T* dout, Dims d, const float* ckpt, const float* dh_last, T* dx, float* dh0, float* maps,
               hipStream_t s) {
    d.tiles = (d.H + LPR * VEC - 1) / (LPR * VEC);
    const int64_t grid = (int64_t)d.tiles * d.B * d.segs;
    if (!grid_fits(grid, NT<T, 1>)) return DSSVAE_ETOOBIG;
    if (d.segs > 1) {
        hipLaunchKernelGGL((gated_scan_maps_kernel<T, VEC, false, true>), dim3((unsigned)grid), dim3((NT<T, 1>)), 0, s, x, dout, d,
                           maps);
        DSSVAE_CHECK_LAUNCH();
    }
#define GO(DIV)                                                                                                     \
    hipLaunchKernelGGL((gated_scan_bwd_kernel<T, VEC, TANH, DIV>), dim3((unsigned)grid), dim3((NT<T, DIV>)), 0, s, x, dout, d, ckpt, \
                       dh_last, maps, dx, dh0)
    if (d.T <= CHUNK / 4) GO(4);
    else if (d.T <= CHUNK / 2) GO(2);
    else GO(1);
#undef GO
    DSSVAE_CHECK_LAUNCH();
    return DSSVAE_OK;
}

#define DSSVAE_SCAN_TYPES(CALL)                                          \
    do {                                                                 \
        if (dtype == DSSVAE_F32) {                                       \
            if (tanh) return CALL(float, 1, true);                       \
            return CALL(float, 1, false);                                \
        }                                                                \
        if (dtype == DSSVAE_BF16) {                                      \
            if (vec == 2 && tanh) return CALL(bf16_t, 2, true);          \
            if (vec == 2) return CALL(bf16_t, 2, false);                 \
            if (tanh) return CALL(bf16_t, 1, true);                      \
            return CALL(bf16_t, 1, false);                               \
        }                                                                \
        if (vec == 2 && tanh) return CALL(f16_t, 2, true);               \
        if (vec == 2) return CALL(f16_t, 2, false);                      \
        if (tanh) return CALL(f16_t, 1, true);                           \
        return CALL(f16_t, 1, false);                                    \
    } while (0)

int bad_dims(int dtype, int B, int T, int H, int64_t xb, int64_t xt) {
    if (!dtype_ok(dtype) || B < 0 || T < 0 || T > (1 << 30) || H < 1 || H > (1 << 29)) return 1;
    if (T > 1 && xt < 2 * (int64_t)H) return 1;
    return B > 1 && xb < 2 * (int64_t)H;
}

Dims make_dims(const int32_t* lengths, int B, int T, int H, int reverse, int es) {
    Dims d{};
    d.lengths = lengths;
    d.B = B; d.T = T; d.H = H; d.reverse = reverse != 0;
    d.nchunk = (int)(((int64_t)T + CHUNK - 1) / CHUNK);
    d.segs = plan_segs(B, T, H, es);
    d.seg_chunks = (d.nchunk + d.segs - 1) / d.segs;
    return d;
}

}  // namespace

extern "C" int dssvae_gated_scan_chunks(int T) { return T < 0 ? DSSVAE_EINVAL : (int)(((int64_t)T + CHUNK - 1) / CHUNK); }

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
#define CALL(T_, V, TH) fwd_launch<T_, V, TH>((const T_*)x, d, h0, (T_*)out, h_last, checkpoints, (float*)workspace, s)
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
#define CALL(T_, V, TH)                                                                                             \
    bwd_launch<T_, V, TH>((const T_*)x, (const T_*)dout, d, checkpoints, dh_last, (T_*)dx, dh0, (float*)workspace, s)
    DSSVAE_SCAN_TYPES(CALL);
#undef CALL
}

namespace {

template <typename T, int VEC, bool TANH>
int step_launch(const T* x, int64_t xb, const float* h, int B, int H, T* out, int64_t ob, float* h_out, hipStream_t s) {
    const int64_t n = (int64_t)B * (H / VEC), grid = (n + STEP_THREADS - 1) / STEP_THREADS;
    if (!grid_fits(grid, STEP_THREADS)) return DSSVAE_ETOOBIG;
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
    const int es = elem_size(dtype), wide = 16 / es;
    // 16-byte granules where rows allow them, else single elements
    const bool ok = H % wide == 0 && aligned_to(x, 16) && aligned_to(out, 16) && (B == 1 || (xb % wide == 0 && ob % wide == 0));
    hipStream_t s = (hipStream_t)stream;
#define GO(T, V)                                                                                                       \
    do {                                                                                                               \
        if (tanh_candidate) return step_launch<T, V, true>((const T*)x, xb, h, B, H, (T*)out, ob, h_out, s);           \
        return step_launch<T, V, false>((const T*)x, xb, h, B, H, (T*)out, ob, h_out, s);                              \
    } while (0)
    if (dtype == DSSVAE_F32) { if (ok) GO(float, 4); GO(float, 1); }
    if (dtype == DSSVAE_BF16) { if (ok) GO(bf16_t, 8); GO(bf16_t, 1); }
    if (ok) GO(f16_t, 8);
    GO(f16_t, 1);
#undef GO
}
