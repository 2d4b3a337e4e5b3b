// Element types of the sequence-block kernels (layer norm, gated scan, linear_act, distillation): fp32, bf16, fp16 in
// memory, fp32 in registers.  A granule is VEC consecutive elements moved by one load / store instruction.
#pragma once
#include "common.h"

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

template <typename T, int N> struct VecOf { typedef T type __attribute__((ext_vector_type(N))); };
template <typename T> struct VecOf<T, 1> { typedef T type; };

// raw granule -> floats (exact) and floats -> raw granule (one rounding to nearest even; bf16 on v_cvt_pk_bf16_f32)
template <typename T, int VEC>
struct Gran {
    typedef typename VecOf<T, VEC>::type V;
    V v;
    __device__ __forceinline__ void load(const T* p) { v = *reinterpret_cast<const V*>(p); }
    __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<V*>(p) = v; }
    __device__ __forceinline__ float get(int i) const {
        if constexpr (VEC == 1) return (float)v;
        else return (float)v[i];
    }
    __device__ __forceinline__ void set(int i, float f) {
        if constexpr (VEC == 1) v = (T)f;
        else v[i] = (T)f;
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < VEC; ++i) set(i, 0.f);
    }
};

// The same without alignment beyond the element's: still one 16-byte instruction (global memory takes any address), a little
// dearer where it crosses a cache line
template <typename T, int VEC>
struct GranU : Gran<T, VEC> {
    typedef typename Gran<T, VEC>::V U __attribute__((aligned(sizeof(T))));
    __device__ __forceinline__ void load(const T* p) { this->v = *reinterpret_cast<const U*>(p); }
    __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<U*>(p) = this->v; }
    __device__ __forceinline__ void store_nt(T* p) const { __builtin_nontemporal_store(this->v, reinterpret_cast<U*>(p)); }
};

// The granule at column c of a row of D elements: what lies behind D reads as zero and is not stored.  WHOLE: D is a multiple
// of VEC, a granule is inside or outside.
template <bool WHOLE, typename T, int VEC>
__device__ __forceinline__ void load_cols(GranU<T, VEC>& g, const T* row, int c, int D) {
    if (WHOLE ? c < D : c + VEC <= D) {
        g.load(row + c);
    } else {
        g.zero();
        if (!WHOLE) {
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                if (c + j < D) g.set(j, (float)row[c + j]);
        }
    }
}
template <bool WHOLE, typename T, int VEC>
__device__ __forceinline__ void store_cols(const GranU<T, VEC>& g, T* row, int c, int D) {
    if (WHOLE ? c < D : c + VEC <= D) {
        g.store(row + c);
    } else if (!WHOLE) {
#pragma unroll
        for (int j = 0; j < VEC; ++j)
            if (c + j < D) row[c + j] = (T)g.get(j);
    }
}

// The same in two steps, so that nothing waits between the loads of a row: load_near takes a granule that is always whole,
// trim puts its columns in place (columns behind D: zero, or with ZERO false the value of some column of the row).
// Rows narrower than a granule go by elements.
template <typename T, int VEC>
__device__ __forceinline__ void load_near(GranU<T, VEC>& g, const T* row, int c, int D) {
    if (D >= VEC) {
        g.load(row + (c + VEC <= D ? c : D - VEC));
    } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) g.set(j, (float)row[c + j < D ? c + j : D - 1]);
    }
}
template <bool ZERO, typename T, int VEC>
__device__ __forceinline__ void trim(GranU<T, VEC>& g, int c, int D) {
    static_assert(VEC * sizeof(T) == 16, "16-byte granules");
    if (c + VEC <= D) return;
    const int out = c + VEC - D;  // columns behind the row's end
    if (D >= VEC && out < VEC) {
        const unsigned __int128 raw = __builtin_bit_cast(unsigned __int128, g.v);
        const int bits = out * 8 * (int)sizeof(T);
        g.v = __builtin_bit_cast(typename Gran<T, VEC>::V, ZERO ? raw >> bits : raw >> bits | raw << (128 - bits));
    } else if (ZERO) {
#pragma unroll
        for (int j = 0; j < VEC; ++j)
            if (c + j >= D) g.set(j, 0.f);
    }
}

// A parameter vector [D] (norm weight, bias) whose type is the activations' T or fp32, `none` where it is NULL: elements
// [c, c + VEC) as floats, zero behind D
template <bool WHOLE, typename T, int VEC>
__device__ __forceinline__ void load_param(float (&o)[VEC], const void* p, bool f32, int c, int D, float none) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) o[j] = c + j < D ? none : 0.f;
    if (!p || c >= D) return;
    if (f32) {
        GranU<float, VEC> g;
        load_cols<WHOLE, float, VEC>(g, reinterpret_cast<const float*>(p), c, D);
#pragma unroll
        for (int j = 0; j < VEC; ++j) o[j] = g.get(j);
    } else {
        GranU<T, VEC> g;
        load_cols<WHOLE, T, VEC>(g, reinterpret_cast<const T*>(p), c, D);
#pragma unroll
        for (int j = 0; j < VEC; ++j) o[j] = g.get(j);
    }
}

// Sum over the TPR neighbouring threads that share a row: within a wave by shuffles, over several waves through `red`
// (one float per wave of the block).  Every thread of the block calls it; all threads of a row get the same sum.
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* red) {
    constexpr int W = TPR < 64 ? TPR : 64;
#pragma unroll
    for (int o = W / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    if constexpr (TPR > 64) {
        constexpr int NW = TPR / 64;
        const int wave = threadIdx.x >> 6;
        __syncthreads();  // the previous use of `red` has been read
        if ((threadIdx.x & 63) == 0) red[wave] = v;
        __syncthreads();
        const int w0 = wave / NW * NW;
        v = 0.f;
#pragma unroll
        for (int i = 0; i < NW; ++i) v += red[w0 + i];
    }
    return v;
}

// The same of two values behind one pair of barriers; `red` holds two floats per wave
template <int TPR>
__device__ __forceinline__ void row_sums(float& a, float& b, float* red) {
    constexpr int W = TPR < 64 ? TPR : 64;
#pragma unroll
    for (int o = W / 2; o > 0; o >>= 1) {
        a += __shfl_xor(a, o, 64);
        b += __shfl_xor(b, o, 64);
    }
    if constexpr (TPR > 64) {
        constexpr int NW = TPR / 64;
        const int wave = threadIdx.x >> 6, w0 = wave / NW * NW;
        __syncthreads();
        if ((threadIdx.x & 63) == 0) {
            red[2 * wave] = a;
            red[2 * wave + 1] = b;
        }
        __syncthreads();
        a = b = 0.f;
#pragma unroll
        for (int i = 0; i < NW; ++i) {
            a += red[2 * (w0 + i)];
            b += red[2 * (w0 + i) + 1];
        }
    }
}

// tanh and its slope from u = exp(-2 |x|), both to their own accuracy: tanh = (1 - u) / (1 + u), which cancels near 0 (1 - 2 / (1 + exp(2 x))
// is off by 1e-3 of itself at 1e-4): below 0.3 an odd polynomial takes its place (x^3 (c0 + c1 x^2 + c2 x^4), fitted for the least
// relative error, 1.2e-8); slope = 4 u / (1 + u)^2, which 1 - tanh^2 loses where tanh saturates (6 % off at 8).
__device__ __forceinline__ float tanh_f(float x, float& slope) {
    const float m = fabsf(x), u = __builtin_amdgcn_exp2f(-2.8853900817779268f * m), r = __builtin_amdgcn_rcpf(1.f + u), s = x * x;
    slope = 4.f * u * r * r;
    const float p = x + x * s * (-0.33333060f + s * (0.13314833f + s * -0.050366241f));
    return m < 0.3f ? p : copysignf((1.f - u) * r, x);
}
__device__ __forceinline__ float tanh_f(float x) {
    float slope;
    return tanh_f(x, slope);
}

// A launch holds fewer than 2^32 threads.
static inline bool grid_fits(int64_t blocks, int threads) { return blocks >= 0 && blocks <= 0xffffffffLL / threads; }

static inline bool aligned_to(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) % bytes) == 0; }

// Compute units (one kind of device per process; 256 without one: the host-side plans are tested there).
static inline int device_cus() {
    static const int cus = [] {
        int n = 0;
        return dssvae_device_cus(&n) == DSSVAE_OK && n > 0 ? n : 256;
    }();
    return cus;
}

static inline int elem_size(int dtype) { return dtype == DSSVAE_F32 ? 4 : 2; }
static inline bool dtype_ok(int dtype) { return dtype >= DSSVAE_F32 && dtype <= DSSVAE_F16; }
