// Distillation from a teacher's top logits (HBM-bound: one read of the student's logits, one write of their gradient).
//
//   p = softmax(teacher / tau) over the row's valid slots, q = softmax(logits / tau) over the vocabulary
//   row = tau^2 sum_j p_j (log p_j - log q[id_j]) ; total = sum_i w_i row_i ; dlogits = w tau (q - scatter(p))
//
// One block per row.  The weight of a row is known at the call, so the gradient leaves in the SAME pass: a row stays in
// registers (NV granules of 16 bytes per thread) between its read and the store; of rows wider than 16 granules x 1024 threads,
// 8 granules a thread more stay in LDS, and what is behind those is read twice (2048 x
// 100003 fp32: 346 us = 4.7 TB/s, 454 us with the whole row read twice).  Without a gradient nothing is kept of them.
// Maximum and sum are one walk, granule by granule as they arrive: two walks left the memory idle for the second where only
// one block fits a CU (2048 x 100003 bf16, NV = 16: 222 us, now 185 us = 4.4 TB/s).  Up to NV = 8 two blocks share a CU (64
// registers) and fill each other's gaps: 7936 x 30000 fp32 in 350 us = 5.4 TB/s.  Rows may start at any element: up to VEC - 1
// elements in front of the first 16-byte boundary and behind the last granule are "edge" elements, one per thread.
// The k teacher slots are wave 0's: softmax by shuffles while the block loads.  The k gradient entries are written over the
// dense store behind a barrier, by the first slot of each distinct id with the sum of its probabilities: no atomics, and
// repeated ids add up in slot order.
// An upstream gradient f other than 1 (a loss scale, a mixing weight) is only known in backward.  It has to come before the rounding to
// 16 bits: at 7936 rows and 30000 words the unit gradient of a word is about 1e-8, zero in fp16, and 65536 times it is not.  So
// backward forms the rows again with w f in place of w, from the logits (read and write: what multiplying the stored gradient
// would move, too: 7936 x 30000 fp32 366 us a step with f = 1, 739 with 0.3; 2048 x 100003 bf16 187 and 389).  Where f is 1 its blocks
// end at once.
#include "elem.h"

namespace {

constexpr int MAX_TOP = DSSVAE_DISTILL_MAX_TOP;
constexpr float LOG2E = 1.4426950408889634f, NINF = -__builtin_huge_valf();

__device__ __forceinline__ float exp2_f(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    return v;
}

// Running maximum m and sum s of exp((x - m) / tau): one more granule
template <typename T, int VEC>
__device__ __forceinline__ void online(const Gran<T, VEC>& v, float c, float& m, float& s) {
    float top = m;
#pragma unroll
    for (int j = 0; j < VEC; ++j) top = fmaxf(top, v.get(j));
    const float ref = top == NINF ? 0.f : top;  // (all -inf so far: every term is 0; a NaN stays one)
    s *= exp2_f((m - ref) * c);
#pragma unroll
    for (int j = 0; j < VEC; ++j) s += exp2_f((v.get(j) - ref) * c);
    m = top;
}

// The granules stay in their 16 bytes between the walks over them: the compiler may not keep them as floats as well, which
// would double a 16-bit row's registers (and spill).
template <typename T, int VEC>
__device__ __forceinline__ void keep_raw(Gran<T, VEC>& v) {
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    u32x4 r = __builtin_bit_cast(u32x4, v.v);
    asm volatile("" : "+v"(r));
    v.v = __builtin_bit_cast(typename Gran<T, VEC>::V, r);
}

// One row by a block.  NV granules per thread in registers; HOLD > 0: any width, the next HOLD granules per thread stay in LDS and
// what is still left is read twice; NV = 0: any width, no gradient.  f: the gradient's factor; rows NULL: the loss is not wanted.
template <typename T, int NT, int NV, int HOLD>
__device__ __forceinline__ void distill_row(const T* __restrict__ z, int64_t ldz, int V, const int64_t* __restrict__ ids,
                                            const float* __restrict__ teacher, int k, float tau, const float* __restrict__ weight,
                                            float w_all, T* __restrict__ dz, int64_t lddz, float* __restrict__ rows, int64_t row, float f) {
    constexpr int VEC = 16 / (int)sizeof(T);
    constexpr int NR = NV > 0 ? NV : 1, AHEAD = 4;  // loads in flight in the walk over what the registers do not hold
    static_assert(HOLD % AHEAD == 0, "whole steps of the walk are held");
    __shared__ float2 red[NT / 64];  // (maximum, sum) of each wave
    __shared__ uint4 held[HOLD > 0 ? HOLD * NT : 1];
    extern __shared__ int s_id[];  // [k], and behind it the probabilities [k]
    float* s_p = reinterpret_cast<float*>(s_id + k);
    __shared__ float s_mass;  // 1, 0 (no valid slot) or NaN (an id outside the vocabulary, a NaN or +inf among the teacher's logits)
    const int tid = threadIdx.x;
    const float w = weight ? weight[row] : w_all, c = LOG2E / tau;
    const T* zr = z + row * ldz;
    T* dr = dz ? dz + row * lddz : nullptr;
    const int mis = (int)((reinterpret_cast<uintptr_t>(zr) & 15u) / sizeof(T));
    const int head = min((VEC - mis) % VEC, V), nvec = (V - head) / VEC, tail = V - head - nvec * VEC;
    const int edge = tid < head ? tid : tid - head < tail ? V - tail + (tid - head) : -1;
    const T* zb = zr + head;

    bool dead = w == 0.f;  // nothing is read, nothing but zeros is written
    Gran<T, VEC> v[NR];
    float ev = NINF;
    if (!dead) {
        if constexpr (NV > 0) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int g = i * NT + tid;
                if (g < nvec) {
                    v[i].load(zb + (unsigned)(g * VEC));
                } else {
#pragma unroll
                    for (int j = 0; j < VEC; ++j) v[i].set(j, NINF);
                }
            }
        }
        if (edge >= 0) ev = (float)zr[edge];
        if (tid < 64) {
            float top = NINF;
            bool bad = false;
            for (int j = tid; j < k; j += 64) {
                const int64_t id = ids[row * k + j];
                const float t = id >= 0 ? teacher[row * k + j] : NINF;
                bad |= id >= V || !(t < -NINF);
                s_id[j] = id >= 0 && id < V ? (int)id : -1;
                s_p[j] = t;
                top = fmaxf(top, t);
            }
            top = wave_max(top);
            float sum = 0.f;
            for (int j = tid; j < k; j += 64) sum += exp2_f((s_p[j] - top) * c);
            sum = wave_sum(sum);
            const bool any_bad = __any(bad), none = top == NINF;
            for (int j = tid; j < k; j += 64) s_p[j] = none ? 0.f : exp2_f((s_p[j] - top) * c) / sum;
            if (tid == 0) s_mass = any_bad ? __builtin_nanf("") : none ? 0.f : 1.f;
        }
    }
    // maximum and sum in ONE walk that consumes the granules in the order they arrive, the later ones still in flight
    float m = ev, s = ev == NINF ? 0.f : 1.f;
    if (!dead) {
        if constexpr (NV > 0) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                online(v[i], c, m, s);
                keep_raw(v[i]);
            }
        }
        if constexpr (NV == 0 || HOLD > 0) {
            for (int i = 0, g = NV * NT + tid; g < nvec; i += AHEAD, g += AHEAD * NT) {
                Gran<T, VEC> r[AHEAD];
#pragma unroll
                for (int j = 0; j < AHEAD; ++j) {
                    if (g + j * NT < nvec) {
                        r[j].load(zb + (unsigned)((g + j * NT) * VEC));
                    } else {
#pragma unroll
                        for (int e = 0; e < VEC; ++e) r[j].set(e, NINF);
                    }
                }
#pragma unroll
                for (int j = 0; j < AHEAD; ++j) {
                    online(r[j], c, m, s);
                    if (HOLD > 0 && i < HOLD) held[(i + j) * NT + tid] = __builtin_bit_cast(uint4, r[j].v);
                }
            }
        }
    }
    const float mw = wave_max(m);
    s *= exp2_f((m - (mw == NINF ? 0.f : mw)) * c);
    s = wave_sum(s);
    if ((tid & 63) == 0) red[tid >> 6] = make_float2(mw, s);
    __syncthreads();
    const float mass = dead ? 0.f : s_mass;
    if (mass == 0.f) {  // (the whole block alike)
        if (rows && tid == 0) rows[row] = 0.f;
        if (!dr) return;
        Gran<T, VEC> o;
        o.zero();
        T* db = dr + head;
        for (int64_t g = tid; g < nvec; g += NT) o.store(db + g * VEC);
        if (edge >= 0) dr[edge] = (T)0.f;
        return;
    }
    const float2 r = red[tid % (NT / 64)];  // every NT / 64 neighbouring lanes hold all the waves' pairs
    float M = r.x;
#pragma unroll
    for (int o = NT / 128; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor(M, o, 64));
    float S = r.y * exp2_f((r.x - M) * c);
#pragma unroll
    for (int o = NT / 128; o > 0; o >>= 1) S += __shfl_xor(S, o, 64);
    if (rows && tid < 64) {
        float part = 0.f;
        for (int j = tid; j < k; j += 64) {
            const float p = s_p[j];
            if (p > 0.f && s_id[j] >= 0) part += p * (logf(p) - ((float)zr[s_id[j]] - M) / tau);
        }
        part = wave_sum(part);
        if (tid == 0) rows[row] = tau * tau * (part + logf(S)) * mass;
    }
    if (NV == 0 || !dr) return;
    const float wt = w * tau * f, a = wt * mass / S;
    T* db = dr + head;
    {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int g = i * NT + tid;
            if (g >= nvec) continue;
            Gran<T, VEC> o;
#pragma unroll
            for (int j = 0; j < VEC; ++j) o.set(j, a * exp2_f((v[i].get(j) - M) * c));
            o.store(db + (unsigned)(g * VEC));
        }
    }
    if constexpr (HOLD > 0) {
        for (int i = 0, g = NV * NT + tid; g < nvec; ++i, g += NT) {
            Gran<T, VEC> r, o;
            if (i < HOLD) r.v = __builtin_bit_cast(typename Gran<T, VEC>::V, held[i * NT + tid]);
            else r.load(zb + (unsigned)(g * VEC));
#pragma unroll
            for (int j = 0; j < VEC; ++j) o.set(j, a * exp2_f((r.get(j) - M) * c));
            o.store(db + (unsigned)(g * VEC));
        }
    }
    if (edge >= 0) dr[edge] = (T)(a * exp2_f((ev - M) * c));
    __syncthreads();  // the dense stores come before the k entries written over them
    for (int j = tid; j < k; j += NT) {
        const int id = s_id[j];
        if (id < 0) continue;
        float p = 0.f;
        bool first = true;
#pragma unroll 4
        for (int i = 0; i < k; ++i) {
            const bool same = s_id[i] == id;
            first = first && !(same && i < j);
            p += same ? s_p[i] : 0.f;
        }
        if (first) dr[id] = (T)(a * exp2_f(((float)zr[id] - M) * c) - wt * p * mass);
    }
}

template <typename T, int NT, int NV, int HOLD>
__global__ __launch_bounds__(NT, NV == 8 ? 8 : 4) void distill_kernel(
    const T* __restrict__ z, int64_t ldz, int V, const int64_t* __restrict__ ids, const float* __restrict__ teacher, int k,
    float tau, const float* __restrict__ weight, float w_all, T* __restrict__ dz, int64_t lddz, float* __restrict__ rows) {
    distill_row<T, NT, NV, HOLD>(z, ldz, V, ids, teacher, k, tau, weight, w_all, dz, lddz, rows, blockIdx.x, 1.f);
}

// the gradient again, times *factor, unless that is 1: as many blocks as the chip holds, row after row
template <typename T, int NT, int NV, int HOLD>
__global__ __launch_bounds__(NT, NV == 8 ? 8 : 4) void distill_again_kernel(
    const T* __restrict__ z, int64_t ldz, int64_t N, int V, const int64_t* __restrict__ ids, const float* __restrict__ teacher, int k,
    float tau, const float* __restrict__ weight, float w_all, const float* __restrict__ factor, T* __restrict__ dz, int64_t lddz) {
    const float f = *factor;
    if (f == 1.f) return;
    for (int64_t row = blockIdx.x; row < N; row += gridDim.x) {
        distill_row<T, NT, NV, HOLD>(z, ldz, V, ids, teacher, k, tau, weight, w_all, dz, lddz, nullptr, row, f);
        __syncthreads();  // the row's slots and sums have been read
    }
}

// total = sum of w_i row_i in a fixed order (64-bit sums)
__global__ __launch_bounds__(1024) void distill_total_kernel(const float* __restrict__ rows, const float* __restrict__ weight,
                                                             float w_all, int64_t n, float* __restrict__ total) {
    __shared__ double red[16];
    double s = 0.0;
    // (eight rows' loads at a time; a row of weight 0 holds 0)
    for (int64_t i0 = threadIdx.x; i0 < n; i0 += 8 * 1024) {
        float w[8], r[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int64_t i = i0 + j * 1024;
            w[j] = i >= n ? 0.f : weight ? weight[i] : w_all;
            r[j] = i >= n ? 0.f : rows[i];
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) s += (double)w[j] * r[j];
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < 16; ++i) s += red[i];
        *total = (float)s;
    }
}

// x *= *g; *g = 1 (the usual upstream gradient of a loss) costs one scalar read
template <typename T>
__global__ __launch_bounds__(256) void scale_kernel(T* __restrict__ x, int64_t ld, int64_t rows, int V,
                                                    const float* __restrict__ g) {
    const float f = *g;
    if (f == 1.f) return;
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x)
        for (int64_t c = threadIdx.x; c < V; c += 256) x[r * ld + c] = (T)((float)x[r * ld + c] * f);
}

// (factor: the gradient alone, again)
template <typename T>
int launch(const T* z, int64_t ldz, int64_t N, int V, const int64_t* ids, const float* teacher, int k, float tau,
           const float* weight, float w_all, const float* factor, T* dz, int64_t lddz, float* rows, hipStream_t s) {
    constexpr int VEC = 16 / (int)sizeof(T);
    const int64_t gran = ((int64_t)V + VEC - 1) / VEC;
#define GO(NT, NV, HOLD)                                                                                                   \
    do {                                                                                                               \
        if constexpr ((NV) > 0) {                                                                                      \
            if (factor) {                                                                                              \
                const int64_t most = (int64_t)device_cus() * (2048 / NT);                                              \
                hipLaunchKernelGGL((distill_again_kernel<T, NT, NV, HOLD>), dim3((unsigned)(N < most ? N : most)), dim3(NT), k * 8, s, z, ldz, \
                                   N, V, ids, teacher, k, tau, weight, w_all, factor, dz, lddz);                       \
                DSSVAE_CHECK_LAUNCH();                                                                                 \
                return DSSVAE_OK;                                                                                      \
            }                                                                                                          \
        }                                                                                                              \
        hipLaunchKernelGGL((distill_kernel<T, NT, NV, HOLD>), dim3((unsigned)N), dim3(NT), k * 8, s, z, ldz, V, ids, teacher, k, tau, weight, \
                           w_all, dz, lddz, rows);                                                                     \
        DSSVAE_CHECK_LAUNCH();                                                                                         \
        return DSSVAE_OK;                                                                                              \
    } while (0)
    // the fewest threads that hold a row in 8 granules each: more rows in flight where a row is short (60000 x 300 bf16: 54 us, with
    // 256 threads a row 117 us; 8000 x 5000 fp32: 35 us, with 1024 threads a row 67 us)
    if (gran <= 64) GO(64, 1, 0);
    if (gran <= 64 * 4) GO(64, 4, 0);
    if (gran <= 64 * 8) GO(64, 8, 0);
    if (gran <= 128 * 8) GO(128, 8, 0);
    if (gran <= 256 * 8) GO(256, 8, 0);
    if (gran <= 512 * 8) GO(512, 8, 0);
    if (gran <= 1024 * 8) GO(1024, 8, 0);
    if (!dz) GO(1024, 0, 0);
    if (gran <= 1024 * 16) GO(1024, 16, 0);
    GO(1024, 16, 8);
#undef GO
}

}  // namespace

namespace {

bool bad_args(const void* logits, int64_t ldz, int dtype, int64_t N, int V, const int64_t* ids, const float* teacher, int k, float tau,
              const void* dlogits, int64_t lddz) {
    if (!dtype_ok(dtype) || N < 0 || N > 0x7fffffff || V < 1 || V > (1 << 30) || k < 1 || k > MAX_TOP || ldz < V ||
        !(tau > 0.f) || !(tau < __builtin_huge_valf()) || (dlogits && lddz < V))
        return true;
    if (N > 0 && (!logits || !ids || !teacher)) return true;
    const int es = elem_size(dtype);
    if (!aligned_to(logits, es) || !aligned_to(dlogits, es)) return true;
    // a granule of the gradient is stored where its logits were loaded: same offset from the 16-byte boundary in every row
    return dlogits && N > 0 && ((reinterpret_cast<uintptr_t>(logits) - reinterpret_cast<uintptr_t>(dlogits)) % 16 != 0 ||
                                (N > 1 && (ldz - lddz) % (16 / es) != 0));
}

int all_rows(const void* logits, int64_t ldz, int dtype, int64_t N, int V, const int64_t* ids, const float* teacher, int k, float tau,
             const float* weight, float weight_all, const float* factor, void* dlogits, int64_t lddz, float* rows, hipStream_t s) {
    constexpr int64_t PART = 1 << 21;  // rows of a launch: 1024 threads each stay below 2^32
    for (int64_t r = 0; r < N; r += PART) {
        const int64_t n = N - r < PART ? N - r : PART;
        int e;
#define GO(T)                                                                                                          \
    launch<T>((const T*)logits + r * ldz, ldz, n, V, ids + r * k, teacher + r * k, k, tau, weight ? weight + r : nullptr, weight_all, factor, \
              dlogits ? (T*)dlogits + r * lddz : nullptr, lddz, rows ? rows + r : nullptr, s)
        if (dtype == DSSVAE_F32) e = GO(float);
        else if (dtype == DSSVAE_BF16) e = GO(bf16_t);
        else e = GO(f16_t);
#undef GO
        if (e != DSSVAE_OK) return e;
    }
    return DSSVAE_OK;
}

}  // namespace

extern "C" int dssvae_distill(const void* logits, int64_t ldz, int dtype, int64_t N, int V, const int64_t* ids,
                              const float* teacher, int k, float tau, const float* weight, float weight_all, void* dlogits,
                              int64_t lddz, float* rows, float* total, void* stream) {
    if (bad_args(logits, ldz, dtype, N, V, ids, teacher, k, tau, dlogits, lddz) || !total || (N > 0 && !rows)) return DSSVAE_EINVAL;
    hipStream_t s = (hipStream_t)stream;
    const int e = all_rows(logits, ldz, dtype, N, V, ids, teacher, k, tau, weight, weight_all, nullptr, dlogits, lddz, rows, s);
    if (e != DSSVAE_OK) return e;
    hipLaunchKernelGGL(distill_total_kernel, dim3(1), dim3(1024), 0, s, rows, weight, weight_all, N, total);
    DSSVAE_CHECK_LAUNCH();
    return DSSVAE_OK;
}

extern "C" int dssvae_distill_again(const void* logits, int64_t ldz, int dtype, int64_t N, int V, const int64_t* ids,
                                    const float* teacher, int k, float tau, const float* weight, float weight_all, const float* factor,
                                    void* dlogits, int64_t lddz, void* stream) {
    if (bad_args(logits, ldz, dtype, N, V, ids, teacher, k, tau, dlogits, lddz) || !factor || (N > 0 && !dlogits)) return DSSVAE_EINVAL;
    return all_rows(logits, ldz, dtype, N, V, ids, teacher, k, tau, weight, weight_all, factor, dlogits, lddz, nullptr, (hipStream_t)stream);
}

extern "C" int dssvae_scale_rows(void* x, int64_t ld, int dtype, int64_t rows, int V, const float* factor, void* stream) {
    if (!dtype_ok(dtype) || rows < 0 || V < 1 || ld < V || !factor) return DSSVAE_EINVAL;
    if (rows == 0) return DSSVAE_OK;
    if (!x) return DSSVAE_EINVAL;
    const int64_t most = 16 * (int64_t)device_cus();
    const dim3 grid((unsigned)(rows < most ? rows : most));
    hipStream_t s = (hipStream_t)stream;
    if (dtype == DSSVAE_F32) hipLaunchKernelGGL((scale_kernel<float>), grid, dim3(256), 0, s, (float*)x, ld, rows, V, factor);
    else if (dtype == DSSVAE_BF16) hipLaunchKernelGGL((scale_kernel<bf16_t>), grid, dim3(256), 0, s, (bf16_t*)x, ld, rows, V, factor);
    else hipLaunchKernelGGL((scale_kernel<f16_t>), grid, dim3(256), 0, s, (f16_t*)x, ld, rows, V, factor);
    DSSVAE_CHECK_LAUNCH();
    return DSSVAE_OK;
}
