// Linear layer with its epilogue:  z = x w^T + b,  y = act(z) + residual,  and its backward pass
//   dz = dy act'(z),  dx = dz w,  dw = dz^T x,  db = sum_rows dz,  dresidual = dy.
//
// Products run on one tile kernel: v_mfma_f32_32x32x16 for bf16 / fp16, fp32 accumulation, one rounding per output.
// fp32 operands are taken apart into three bf16 each (24 bits, exact) as they come out of LDS, and six of the nine products of
// the parts are added: what is left out is below 2^-22 of a product, and on the mean of random inputs the sums are closer to
// the exact ones than v_mfma_f32_32x32x2_f32's order gives (K = 7936: 7e-7 of the norm; the library's fp32 product 1.6e-6).  Sums of
// at most 32 products, where that would show (a single product came out up to four times as far off as one fp32 rounding), take the
// fp32 instruction, which does a sixteenth of the bf16 one's work: a library product of 4096^3 takes 0.91 ms, this one 0.70 ms (the six
// run at 1170 TFLOP/s; a library product of bf16 operands reaches 1326).  Taking operands apart once per block, on their way
// into LDS through registers, halves the vector instructions but measured the same: 0.73 ms.
//
// The tile kernel: C[M, N] = A[M, K] . B[N, K]^T, both operands contiguous along K.  A BM x BN block walks K in steps of
// 128 bytes (64 or 32 elements); operand tiles go global -> LDS directly (16 bytes a lane, no registers), double buffered.  LDS row r keeps its
// 16-byte chunk c at place c ^ (r & 7): the eight rows a quarter wave reads at one chunk then cover all banks (rows are 128
// bytes apart, unswizzled they would share one).  The pipeline is rotated: fragments of the step's first half are already in
// registers when it begins; one barrier per step, passed between the halves: by then the next tile has landed and every
// wave has read all of this one, so its buffer takes the tile after next while the second half multiplies.
// The backward operands that are contiguous the other way (w and x along the summed axis, dz for dw) are transposed into the
// workspace first: dz in both orders by the pass that forms it, which also leaves the column sums for db.
// 16-bit types: that pass leaves dz in two parts of the type (dy act'(z) is not a number of the type: rounded once, its error is as
// large as that of the results' own rounding), and the products run over both: low parts first, then high ones, into the same
// accumulators.  The low parts cost the matrix work again (16384 x 2048 -> 8192 bf16 and fp16, gelu, forward and backward: 2.75 ms,
// products of backward 1.8 and transposes 0.39 of it; with a rounded dz 1.76 ms, 0.9 and 0.29): DSSVAE_ACT_ROUND_DZ does without
// them.  None and relu need none: their dz is dy, or zero.
// Few output tiles: K is split over blocks, fp32 partials go to the workspace and a second launch adds them in order and
// applies the epilogue (no atomics: same bits every time).  Backward is three launches: the transposes, both products, and
// the partials with db's column sums.
#include "elem.h"

namespace {

// elements of a k-tile's row (128 bytes) and of a 16-byte granule
template <typename T> constexpr int BK = 128 / (int)sizeof(T);
template <typename T> constexpr int GR = 16 / (int)sizeof(T);

typedef float f32x8 __attribute__((ext_vector_type(8)));

// ---- activations --------------------------------------------------------------------------------------------------
__device__ __forceinline__ float sigmoid_f(float x) {
    return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.4426950408889634f * x));
}
// Phi(z) of the normal distribution, given e = exp(-z^2 / 2).  fp32: from the complementary error function.  16-bit types, whose epilogue is
// bound by the vector ALUs: Phi(-|z|) = e P(t) with t = 1 / (1 + 0.2652 |z|), P of degree 7 fitted for the least RELATIVE error over
// |z| <= 13.3 (6.4e-7, in fp32 9.4e-7: a 200th of fp16's half step; a form with a small absolute error is 2 to 7 half steps off in the tail).
template <typename T>
__device__ __forceinline__ float normal_cdf(float z, float e) {
    if constexpr (sizeof(T) == 4) return 0.5f * erfcf(-0.70710678118654752f * z);
    const float t = __builtin_amdgcn_rcpf(1.f + 0.265165043f * fabsf(z));
    const float p = 0.14153056f + t * (-0.064798355f + t * (0.19396870f + t * -0.067547888f));
    const float q = e * (t * (0.10566972f + t * (0.10784458f + t * (0.083332367f + t * p))));
    return z < 0.f ? q : 1.f - q;
}
__device__ __forceinline__ float normal_exp(float z) { return __builtin_amdgcn_exp2f(-0.72134752044448170f * z * z); }
template <typename T>
__device__ __forceinline__ float act_f(int act, float z) {
    switch (act) {
        case DSSVAE_ACT_RELU: return z > 0.f ? z : (z != z ? z : 0.f);
        case DSSVAE_ACT_GELU: return z * normal_cdf<T>(z, normal_exp(z));
        case DSSVAE_ACT_SILU: return z * sigmoid_f(z);
        case DSSVAE_ACT_TANH: return tanh_f(z);
        default: return z;
    }
}
// (an infinite z has the slope it tends to, not inf * 0; what NaN turns into here meets a NaN)
__device__ __forceinline__ float finite(float z) { return __builtin_amdgcn_fmed3f(z, -1000.f, 1000.f); }
template <typename T>
__device__ __forceinline__ float act_slope(int act, float z) {
    switch (act) {
        case DSSVAE_ACT_RELU: return z > 0.f ? 1.f : (z != z ? z : 0.f);
        case DSSVAE_ACT_GELU: {
            const float e = normal_exp(z);
            return normal_cdf<T>(z, e) + finite(z) * 0.3989422804014327f * e;
        }
        case DSSVAE_ACT_SILU: {
            const float s = sigmoid_f(z);
            return s * (1.f + finite(z) * (1.f - s));
        }
        case DSSVAE_ACT_TANH: {
            float slope;
            tanh_f(z, slope);
            return slope;
        }
        default: return 1.f;
    }
}

// What backward needs of the pre-activation z.  fp32: z.  16-bit types: a 16-bit code of act'(z), its signed fourth root in steps of
// 1 / 31744 (the largest slope, gelu's 1.129, fits; 0 and 1 are exact): a slope s is off by at most 6.3e-5 |s|^(3/4), that is 6e-5 of
// itself at 1, 2e-4 at 0.01, 2e-3 at 1e-6 (fp16's half step: 2.4e-4 to 4.9e-4).  Even steps of z (8 / 32767) were off by 1e-4 in s wherever it bends, more than
// the type's rounding where s is below 0.2; z rounded to the type loses 4e-3 (bf16).  Forward has the slope's exponential at hand
// and backward decodes with four multiplications.  relu keeps z > 0 only.  NaN has a code of its own.
constexpr int16_t CODE_NAN = -32768;
constexpr float CODE_ONE = 31744.f;
template <typename T, int ACT>
__device__ __forceinline__ void encode8(const float (&z)[8], int16_t (&q)[8]) {
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        sum += z[j] + z[j + 1];
        if constexpr (ACT == DSSVAE_ACT_RELU) {
            q[j] = z[j] > 0.f;
            q[j + 1] = z[j + 1] > 0.f;
        } else {
            typedef short s16x2 __attribute__((ext_vector_type(2)));
            float c[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float s = act_slope<T>(ACT, z[j + i]);
                c[i] = copysignf(__builtin_amdgcn_sqrtf(__builtin_amdgcn_sqrtf(fabsf(s))) * (CODE_ONE / 32767.f), s);
            }
            const s16x2 p = __builtin_bit_cast(s16x2, __builtin_amdgcn_cvt_pknorm_i16(c[0], c[1]));
            q[j] = p.x;
            q[j + 1] = p.y;
        }
    }
    if (sum != sum) {  // a NaN (or infinities of both signs) among them
#pragma unroll
        for (int j = 0; j < 8; ++j) q[j] = z[j] != z[j] ? CODE_NAN : q[j];
    }
}
template <int ACT>
__device__ __forceinline__ float decode(int16_t q) {
    if (q == CODE_NAN) return __builtin_nanf("");
    if constexpr (ACT == DSSVAE_ACT_RELU) return q ? 1.f : 0.f;
    const float c = (float)q * (1.f / CODE_ONE);
    return c * c * (c * fabsf(c));
}
// act'(z) from what forward kept
template <typename T, int ACT>
__device__ __forceinline__ float slope_kept(const T* z, int64_t i) {
    if constexpr (sizeof(T) == 4) return act_slope<T>(ACT, (float)z[i]);
    else return decode<ACT>(reinterpret_cast<const int16_t*>(z)[i]);
}

// What happens to an accumulated element on its way out
struct Epilogue {
    const void* bias; int bias_f32;   // [N] or NULL
    const void* res; int64_t ldr;     // [M, N] or NULL
    void* z; int64_t ldz;             // pre-activation as backward needs it, or NULL
    void* y; int64_t ldy;
    int act;
};

template <typename T>
__device__ __forceinline__ float bias_at(const Epilogue& e, int64_t n) {
    if (!e.bias) return 0.f;
    return e.bias_f32 ? reinterpret_cast<const float*>(e.bias)[n] : (float)reinterpret_cast<const T*>(e.bias)[n];
}

template <typename T>
__device__ __forceinline__ f32x8 bias8(const Epilogue& e, int n, int N) {
    f32x8 b;
#pragma unroll
    for (int j = 0; j < 8; ++j) b[j] = n + j < N ? bias_at<T>(e, n + j) : 0.f;
    return b;
}

// eight consecutive columns n .. of row m (those below N): a without the bias b
template <typename T, int ACT>
__device__ __forceinline__ void finish8_act(const Epilogue& e, f32x8 a, f32x8 b, int64_t m, int n, int N) {
    T* y = reinterpret_cast<T*>(e.y) + m * e.ldy + n;
    T* z = e.z ? reinterpret_cast<T*>(e.z) + m * e.ldz + n : nullptr;
    const T* r = e.res ? reinterpret_cast<const T*>(e.res) + m * e.ldr + n : nullptr;
    if (n + 8 <= N) {
        GranU<T, 8> g, gy;
        if (r) g.load(r);
        else g.zero();
        float zz[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            zz[j] = a[j] + b[j];
            gy.set(j, act_f<T>(ACT, zz[j]) + g.get(j));
        }
        if (z) {
            if constexpr (sizeof(T) == 4) {
#pragma unroll
                for (int j = 0; j < 8; ++j) g.set(j, zz[j]);
                g.store(z);
            } else {
                int16_t q[8];
                encode8<T, ACT>(zz, q);
                GranU<int16_t, 8> gq;
#pragma unroll
                for (int j = 0; j < 8; ++j) gq.v[j] = q[j];
                gq.store(reinterpret_cast<int16_t*>(z));
            }
        }
        gy.store(y);
    } else {
        float zz[8];
        int16_t q[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) zz[j] = a[j] + b[j];
        if constexpr (sizeof(T) == 2) encode8<T, ACT>(zz, q);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (n + j >= N) continue;
            if (z) {
                if constexpr (sizeof(T) == 4) z[j] = zz[j];
                else reinterpret_cast<int16_t*>(z)[j] = q[j];
            }
            y[j] = (T)(act_f<T>(ACT, zz[j]) + (r ? (float)r[j] : 0.f));
        }
    }
}
// (one branch on the activation per eight elements, not one per element)
template <typename T>
__device__ __forceinline__ void finish8(const Epilogue& e, f32x8 a, f32x8 b, int64_t m, int n, int N) {
    switch (e.act) {
        case DSSVAE_ACT_RELU: finish8_act<T, DSSVAE_ACT_RELU>(e, a, b, m, n, N); break;
        case DSSVAE_ACT_GELU: finish8_act<T, DSSVAE_ACT_GELU>(e, a, b, m, n, N); break;
        case DSSVAE_ACT_SILU: finish8_act<T, DSSVAE_ACT_SILU>(e, a, b, m, n, N); break;
        case DSSVAE_ACT_TANH: finish8_act<T, DSSVAE_ACT_TANH>(e, a, b, m, n, N); break;
        default: finish8_act<T, DSSVAE_ACT_NONE>(e, a, b, m, n, N);
    }
}

// A number v as two of a 16-bit type, v = (lo LOW + hi) HIGH to 2^-16 of v (bf16) or 2^-22 (fp16).  bf16: hi the number cut off.
// fp16: of v / 2, which stays in the range (|dy act'| < 1.13 * 65504), and the rest times 1024, which lifts the rest of a number
// among the smallest.  hi is always below v in magnitude, so that lo is not zero and has its sign: an infinity on the other side of the
// product stays one.  What is not finite is itself in both.
template <typename T> struct Apart { static constexpr float LOW = 1.f, HIGH = 1.f; };  // (fp32 stays whole)
template <> struct Apart<bf16_t> {
    static constexpr float LOW = 1.f, HIGH = 1.f;
    static __device__ __forceinline__ void of(float v, bf16_t& lo, bf16_t& hi) {
        const bool odd = v == 0.f || !(fabsf(v) < __builtin_huge_valf());
        const float h = odd ? v : __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, v) - 1) & 0xffff0000u);
        hi = (bf16_t)h;
        lo = (bf16_t)(odd ? v : v - h);
    }
};
template <> struct Apart<f16_t> {
    static constexpr float LOW = 1.f / 1024.f, HIGH = 2.f;
    static __device__ __forceinline__ void of(float v, f16_t& lo, f16_t& hi) {
        v *= 0.5f;
        const bool odd = v == 0.f || !(fabsf(v) < __builtin_huge_valf());
        const auto cut = __builtin_amdgcn_cvt_pkrtz(__builtin_bit_cast(float, __builtin_bit_cast(uint32_t, v) - 1), 0.f);
        const float h = odd ? v : (float)cut[0];
        hi = (f16_t)h;
        lo = (f16_t)(odd ? v : (v - h) * 1024.f);
    }
};

// ---- the tile kernel -----------------------------------------------------------------------------------------
typedef __attribute__((address_space(1))) const void* gptr_t;
typedef __attribute__((address_space(3))) void* lptr_t;

__device__ const uint4 zero_granule = {0, 0, 0, 0};

// V: what a lane holds of a 32-row block's granule pair (16 bytes of its row, lanes 32.. the second granule); go: the product
// over both granules.  fp32 takes one float per lane and instruction: which k a (step, lane half) pair multiplies is free as
// long as A and B agree, so four steps use up the 16 bytes.
template <typename T> struct Mfma;
template <> struct Mfma<float> {
    typedef f32x4 V;
    static constexpr int N = 4;  // instructions
    static __device__ __forceinline__ f32x16 go(V a, V b, f32x16 c) {
#pragma unroll
        for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
        return c;
    }
};
template <> struct Mfma<bf16_t> {
    typedef bf16_t V __attribute__((ext_vector_type(8)));
    static constexpr int N = 1;
    static __device__ __forceinline__ f32x16 go(V a, V b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};
template <> struct Mfma<f16_t> {
    typedef f16_t V __attribute__((ext_vector_type(8)));
    static constexpr int N = 1;
    static __device__ __forceinline__ f32x16 go(V a, V b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};

// One operand's share of a tile load: R rows x 128 bytes, TH threads, 16 bytes a lane.  A thread's granules all lie in the same
// place of their rows (rows TH / 8 apart, a multiple of 8: the swizzle is the same).  Rows behind the last are loaded from
// it and never stored.  `base` is uniform: row r0 of the operand at the tile's first k.
template <typename T, int R, int TH>
struct Loader {
    static constexpr int NR = R * 8 / TH;
    unsigned off[NR];  // bytes behind base
    __device__ __forceinline__ static int k_of() {
        const int row = threadIdx.x >> 3;
        return (int)((threadIdx.x & 7) ^ (row & 7)) * GR<T>;
    }
    __device__ __forceinline__ void init(int64_t ld, int64_t rows_left) {
        const int row = threadIdx.x >> 3;
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            int64_t r = row + i * (TH / 8);
            r = r < rows_left ? r : rows_left - 1;
            off[i] = (unsigned)((r * ld + k_of()) * (int64_t)sizeof(T));
        }
    }
    __device__ __forceinline__ void load(T* lds, const T* base) const {
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            unsigned o = off[i];
            asm("" : "+v"(o));  // (extended to 64 bits here, which the load does by itself: extended ahead of the loop it took twice the registers)
            put(lds, i, reinterpret_cast<const char*>(base) + o);
        }
    }
    // a tile that may reach behind K: granules there come from a granule of zeros
    __device__ __forceinline__ void load_last(T* lds, const T* base, int64_t left) const {
        const bool in = k_of() < left;
#pragma unroll
        for (int i = 0; i < NR; ++i)
            put(lds, i, in ? reinterpret_cast<const char*>(base) + off[i] : reinterpret_cast<const char*>(&zero_granule));
    }
    static __device__ __forceinline__ void put(T* lds, int i, const char* src) {
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);  // (places in LDS in scalar registers)
        __builtin_amdgcn_global_load_lds((gptr_t)src, (lptr_t)(lds + (i * TH + wave * 64) * GR<T>), 16, 0, 0);
    }
};

// Eight fp32 values as sums of three bf16 each, x = p0 + p1 + p2 exactly (the first rounded to nearest, so that the rest has
// either sign, the others cut off; p2 runs out of exponent below 2^-110: what is smaller than 2^-133 is dropped).  Infinities, and
// the last 0.4 % below the largest finite value, become NaN.
struct Split {
    Mfma<bf16_t>::V p[3];
    __device__ __forceinline__ void of(f32x4 lo, f32x4 hi) {
        typedef float f32x2 __attribute__((ext_vector_type(2)));
        typedef bf16_t bf16x2 __attribute__((ext_vector_type(2)));
        typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
        u32x4 q[3];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float x = j < 2 ? lo[2 * j] : hi[2 * j - 4], y = j < 2 ? lo[2 * j + 1] : hi[2 * j - 3];
            q[0][j] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{x, y}, bf16x2));
            x -= __builtin_bit_cast(float, q[0][j] << 16);
            y -= __builtin_bit_cast(float, q[0][j] & 0xffff0000u);
#pragma unroll
            for (int t = 1; t < 3; ++t) {
                const uint32_t bx = __builtin_bit_cast(uint32_t, x), by = __builtin_bit_cast(uint32_t, y);
                q[t][j] = __builtin_amdgcn_perm(by, bx, 0x07060302u);  // the upper halves
                x -= __builtin_bit_cast(float, bx & 0xffff0000u);
                y -= __builtin_bit_cast(float, by & 0xffff0000u);
            }
        }
#pragma unroll
        for (int t = 0; t < 3; ++t) p[t] = __builtin_bit_cast(Mfma<bf16_t>::V, q[t]);
    }
};

// MI x NI blocks of 32 x 32 of this wave's tile: the operands of K half `h` (two granule pairs)
template <typename T, int MI, int NI>
struct Frags {
    typename Mfma<T>::V a[2][MI], b[2][NI];
    __device__ __forceinline__ void read(const T* __restrict__ sa, int b_at, int ra, int rb, int h) {
        const T* sb = sa + b_at;
        const int lane = threadIdx.x & 63, r = lane & 31;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const int c = ((h * 4 + s * 2 + (lane >> 5)) ^ (r & 7)) * GR<T>;  // (tile rows start at multiples of 8)
#pragma unroll
            for (int i = 0; i < MI; ++i) a[s][i] = *reinterpret_cast<const typename Mfma<T>::V*>(sa + (ra + i * 32 + r) * BK<T> + c);
#pragma unroll
            for (int j = 0; j < NI; ++j) b[s][j] = *reinterpret_cast<const typename Mfma<T>::V*>(sb + (rb + j * 32 + r) * BK<T> + c);
        }
    }
    __device__ __forceinline__ void multiply(f32x16 (&acc)[MI][NI]) const {
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int j = 0; j < NI; ++j) acc[i][j] = Mfma<T>::go(a[s][i], b[s][j], acc[i][j]);
    }
};

// A K half of fp32 operands (16 elements a row) as bf16 triples
template <int MI, int NI>
struct Planes {
    Split a[MI], b[NI];
    __device__ __forceinline__ void of(const Frags<float, MI, NI>& f) {
#pragma unroll
        for (int i = 0; i < MI; ++i) a[i].of(f.a[0][i], f.a[1][i]);
#pragma unroll
        for (int j = 0; j < NI; ++j) b[j].of(f.b[0][j], f.b[1][j]);
    }
    // smallest terms first; p1 p2, p2 p1 and p2 p2 are left out: |p1| <= 2^-8 |x|, |p2| < 2^-15 |x|, both signs: below 2^-22 of x y together
    __device__ __forceinline__ void multiply(f32x16 (&acc)[MI][NI]) const {
        constexpr int TERMS[6][2] = {{0, 2}, {2, 0}, {1, 1}, {0, 1}, {1, 0}, {0, 0}};
#pragma unroll
        for (int t = 0; t < 6; ++t)
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int j = 0; j < NI; ++j)
                    acc[i][j] = Mfma<bf16_t>::go(a[i].p[TERMS[t][0]], b[j].p[TERMS[t][1]], acc[i][j]);
    }
};

struct Shape {
    const void* A; int64_t lda;
    const void* B; int64_t ldb;
    int64_t M; int N; int64_t K;
    int tiles_m, tiles_n, ksplit;
    int parts;           // of A, `part_at` elements apart: the sum over both, B the same for each; K is then whole k-tiles
    int64_t part_at;
    int64_t ktiles;      // k-tiles per split (of those of all parts, one part behind the other)
    float* part;         // [ksplit][M][N] where ksplit > 1
};

// A launch makes one or two products (dx and dw of a backward call: one fills the CUs that the other leaves idle): blocks
// 0 .. first - 1 are the first one's.
struct Job { Shape s; Epilogue e; int blocks; };
struct Jobs { Job job[2]; int first; };

// output tile of work item `wid`: groups of 8 tile rows, column by column inside a group, so that the blocks of an XCD that run
// together share operand panels in its L2
__device__ __forceinline__ void tile_of(const Shape& s, int t, int& tm, int& tn) {
    constexpr int G = 8;
    const int per = G * s.tiles_n, g = t / per, first = g * G, rows = min(G, s.tiles_m - first), in = t - g * per;
    tm = first + in % rows;
    tn = in / rows;
}

// Loads the tile at (a, b) into the buffer `lds`: BM rows of A, then BN rows of B.  (One restrict pointer per buffer: the
// compiler's bookkeeping of loads that write LDS distinguishes few destinations; past those it waits for all of them in
// front of every LDS read.)
template <typename T, int BM, int BN, int TH>
__device__ __forceinline__ void tile_load(T* __restrict__ lds, const Loader<T, BM, TH>& la, const Loader<T, BN, TH>& lb, const T* a,
                                          const T* b) {
    la.load(lds, a);
    lb.load(lds + BM * BK<T>, b);
}

// Barrier that also waits for this wave's loads into LDS (a workgroup fence alone does not order them).
__device__ __forceinline__ void tile_barrier() {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
}

// The k-tile in `cur`, whose first half is in f0: multiplies it, starts the load of the tile after next (at a, b) into its
// place and leaves the first half of the next tile in f0.  The instruction groups keep the matrix pipe fed: an LDS read (or
// a load) between two MFMAs, all of them issued half a step before their data is needed.
template <typename T, int BM, int BN, int TH, int MI, int NI>
__device__ __forceinline__ void k_step(Frags<T, MI, NI>& f0, Frags<T, MI, NI>& f1, f32x16 (&acc)[MI][NI], const Loader<T, BM, TH>& la,
                                       const Loader<T, BN, TH>& lb, T* cur, const T* next, int ra, int rb, const T* a, const T* b) {
    constexpr int READS = 2 * (MI + NI), MULS = 2 * MI * NI * Mfma<T>::N, LOADS = Loader<T, BM, TH>::NR + Loader<T, BN, TH>::NR;
    f1.read(cur, BM * BK<T>, ra, rb, 1);
    f0.multiply(acc);
#pragma unroll
    for (int i = 0; i < MULS; ++i) {
        if (i < READS) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    }
    tile_barrier();  // this tile has been read by every wave, the next one has landed
    tile_load<T, BM, BN, TH>(cur, la, lb, a, b);
    f0.read(next, BM * BK<T>, ra, rb, 0);
    f1.multiply(acc);
#pragma unroll
    for (int i = 0; i < MULS; ++i) {
        if (i < LOADS) __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);
        if (i < READS) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    }
}

// The same for fp32 operands as bf16 triples.  On entry p0 holds the first half of the tile in `cur` and f1 the second as it is,
// and so of the next tile when it ends: a half is taken apart (11 vector instructions for two elements) behind the MFMAs of
// the half before it, about 7 to an MFMA (4096^3: 0.77 ms with the two one after the other, 0.71 ms so).
template <int BM, int BN, int TH, int MI, int NI>
__device__ __forceinline__ void k_step_split(Planes<MI, NI>& p0, Frags<float, MI, NI>& f1, f32x16 (&acc)[MI][NI],
                                             const Loader<float, BM, TH>& la, const Loader<float, BN, TH>& lb, float* cur, const float* next,
                                             int ra, int rb, const float* a, const float* b) {
    constexpr int READS = 2 * (MI + NI), MULS = 6 * MI * NI, OPS = 44 * (MI + NI), LOADS = Loader<float, BM, TH>::NR + Loader<float, BN, TH>::NR;
    Planes<MI, NI> p1;
    p1.of(f1);
    p0.multiply(acc);
#pragma unroll
    for (int i = 0; i < MULS; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, (OPS + MULS - 1) / MULS, 0);
    }
    tile_barrier();  // this tile has been read by every wave, the next one has landed
    Frags<float, MI, NI> f0;
    f0.read(next, BM * BK<float>, ra, rb, 0);
    tile_load<float, BM, BN, TH>(cur, la, lb, a, b);
    f1.read(next, BM * BK<float>, ra, rb, 1);
    p0.of(f0);
    p1.multiply(acc);
    constexpr int AHEAD = MULS / 6;  // MFMAs that cover the first reads
    __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
#pragma unroll
    for (int i = 0; i < MULS; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        if (i < LOADS) __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);
        if (i < READS) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        if (i >= AHEAD) __builtin_amdgcn_sched_group_barrier(0x002, (OPS + MULS - AHEAD - 1) / (MULS - AHEAD), 0);
    }
}

template <int MI, int NI>
__device__ __forceinline__ void fill(f32x16 (&acc)[MI][NI], float f) {
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = f;
}

template <int MI, int NI>
__device__ __forceinline__ void times(f32x16 (&acc)[MI][NI], float f) {
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] *= f;
}

// acc = this wave's part of the output tile at (m0, n0), over the k-tiles kt0 .. kt1 - 1 of A's parts
template <typename T, int BM, int BN, int WR, int WC, bool SPLIT>
__device__ __forceinline__ void tile_product(const Shape& s, int64_t m0, int n0, int64_t kt0, int64_t kt1, T* __restrict__ buf0,
                                             T* __restrict__ buf1, f32x16 (&acc)[BM / WR / 32][BN / WC / 32]) {
    constexpr int TH = 64 * WR * WC, MI = BM / WR / 32, NI = BN / WC / 32;
    constexpr bool PARTS = sizeof(T) == 2, LIFTED = PARTS && Apart<T>::LOW != 1.f;
    const int wave = threadIdx.x >> 6;
    const int ra = wave / WC * (BM / WR), rb = wave % WC * (BN / WC);
    fill(acc, 0.f);
    if (kt0 >= kt1) return;
    Loader<T, BM, TH> la;
    Loader<T, BN, TH> lb;
    la.init(s.lda, s.M - m0);
    lb.init(s.ldb, s.N - n0);
    const T* A = (const T*)s.A + m0 * s.lda;
    const T* B = (const T*)s.B + (int64_t)n0 * s.ldb;
    const int64_t nk = (s.K + BK<T> - 1) / BK<T>, n = kt1 - kt0;
    const auto at = [&](int64_t t, const T*& a, const T*& b) {  // k-tile t of all parts
        const bool second = PARTS && t >= nk;
        const int64_t k = (second ? t - nk : t) * BK<T>;
        a = A + (second ? s.part_at : 0) + k;
        b = B + k;
    };
    // The order of the tiles of one part is free: the last one, which alone may reach behind K, goes first, then kt0 .. kt1 - 2, so
    // that the loop's loads need no test.  Two parts: in order.  A tile behind the end is the one before it again (loaded, never
    // multiplied).
    const int ordered = PARTS && s.parts > 1;
    const T *a, *b;
    const int64_t t0 = ordered ? kt0 : kt1 - 1, left = s.K - (t0 >= nk ? t0 - nk : t0) * BK<T>;
    at(t0, a, b);
    la.load_last(buf0, a, left);
    lb.load_last(buf0 + BM * BK<T>, b, left);
    const int64_t most = n > 1 ? kt1 - 2 + ordered : kt0;
    at(min(kt0 + ordered, most), a, b);
    if (n > 1) tile_load<T, BM, BN, TH>(buf1, la, lb, a, b);
    tile_barrier();
    // step i multiplies the i-th tile in that order and loads the (i + 2)-th: kt0 + i + 1 (+ 1 in order).  The low part's sums are
    // brought to the high one's scale behind its last tile.
    const int64_t next = kt0 + 1 + ordered, edge = LIFTED && ordered && kt0 < nk ? min(nk, kt1) - kt0 : -1;  // (tiles of the low part)
    int64_t i = 0;
    if constexpr (SPLIT) {
        Frags<T, MI, NI> f0, f1;
        Planes<MI, NI> p0, p1;
        f0.read(buf0, BM * BK<T>, ra, rb, 0);
        f1.read(buf0, BM * BK<T>, ra, rb, 1);
        p0.of(f0);
        if (n > 1) {
            for (; i + 1 < n; i += 2) {
                at(min(next + i, most), a, b);
                k_step_split<BM, BN, TH, MI, NI>(p0, f1, acc, la, lb, buf0, buf1, ra, rb, a, b);
                at(min(next + i + 1, most), a, b);
                k_step_split<BM, BN, TH, MI, NI>(p0, f1, acc, la, lb, buf1, buf0, ra, rb, a, b);
            }
        }
        if (i < n) {
            p1.of(f1);
            p0.multiply(acc);
            p1.multiply(acc);
        }
    } else {
        Frags<T, MI, NI> f0, f1;
        f0.read(buf0, BM * BK<T>, ra, rb, 0);
        if (n > 1) {
            for (; i + 1 < n; i += 2) {
                at(min(next + i, most), a, b);
                k_step<T, BM, BN, TH, MI, NI>(f0, f1, acc, la, lb, buf0, buf1, ra, rb, a, b);
                if constexpr (LIFTED) {
                    if (i + 1 == edge) times(acc, Apart<T>::LOW);
                }
                __builtin_amdgcn_sched_barrier(0);  // (both steps' operands at once do not fit the registers)
                at(min(next + i + 1, most), a, b);
                k_step<T, BM, BN, TH, MI, NI>(f0, f1, acc, la, lb, buf1, buf0, ra, rb, a, b);
                if constexpr (LIFTED) {
                    if (i + 2 == edge) times(acc, Apart<T>::LOW);
                }
            }
        }
        if (i < n) {  // an odd tile is left: nothing behind it
            f1.read(buf0, BM * BK<T>, ra, rb, 1);
            f0.multiply(acc);
            f1.multiply(acc);
            if constexpr (LIFTED) {
                if (i + 1 == edge) times(acc, Apart<T>::LOW);
            }
        }
        if constexpr (LIFTED) {
            if (ordered) times(acc, Apart<T>::HIGH);
        }
    }
    tile_barrier();  // operand buffers are free (and no load is in flight)
}

template <typename T, int BM, int BN, int WR, int WC>
__global__ __launch_bounds__(64 * WR * WC, 2) void linear_tile_kernel(Jobs jobs) {
    constexpr int MI = BM / WR / 32, NI = BN / WC / 32;
    __shared__ __attribute__((aligned(16))) T buf0[(BM + BN) * BK<T>], buf1[(BM + BN) * BK<T>];
    const int which = (int)blockIdx.x >= jobs.first;
    const Shape& s = jobs.job[which].s;
    const Epilogue& e = jobs.job[which].e;
    const int wid = xcd_remap(blockIdx.x - (which ? jobs.first : 0), jobs.job[which].blocks), tiles = s.tiles_m * s.tiles_n;
    const int split = wid / tiles;
    int tm, tn;
    tile_of(s, wid - split * tiles, tm, tn);
    const int64_t m0 = (int64_t)tm * BM;
    const int n0 = tn * BN;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int ra = wave / WC * (BM / WR), rb = wave % WC * (BN / WC);
    const int64_t nk = (s.K + BK<T> - 1) / BK<T>, kt0 = split * s.ktiles, kt1 = min(nk * s.parts, kt0 + s.ktiles);

    f32x16 acc[MI][NI];
    if constexpr (sizeof(T) == 4) {
        int redo = 1;
        if (s.K > BK<T>) {
            tile_product<T, BM, BN, WR, WC, true>(s, m0, n0, kt0, kt1, buf0, buf1, acc);
            float odd = 0.f;  // NaN once a sum is not finite
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int j = 0; j < NI; ++j)
#pragma unroll
                    for (int r = 0; r < 16; ++r) odd += 0.f * acc[i][j][r];
            redo = __syncthreads_or(odd != odd);  // infinities have no triple: those sums, and no others, from fp32 products
        } else {  // sums of one k-tile: too few terms for what the triples leave out to be lost among their roundings
            fill(acc, __builtin_huge_valf());
        }
        if (redo) {
            f32x16 whole[MI][NI];
            tile_product<T, BM, BN, WR, WC, false>(s, m0, n0, kt0, kt1, buf0, buf1, whole);
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int j = 0; j < NI; ++j)
#pragma unroll
                    for (int r = 0; r < 16; ++r) acc[i][j][r] = fabsf(acc[i][j][r]) < __builtin_huge_valf() ? acc[i][j][r] : whole[i][j][r];
        }
    } else {
        tile_product<T, BM, BN, WR, WC, false>(s, m0, n0, kt0, kt1, buf0, buf1, acc);
    }

    // 32 rows x CW columns of this wave at a time through LDS of its own, read back along rows
    constexpr int CW = 32 * NI, LR = CW / 8, RP = 64 / LR;  // columns, lanes per row, rows per pass
    float* stage = reinterpret_cast<float*>(buf0) + wave * 32 * CW;
    static_assert(WR * WC * 32 * CW * 4 <= (int)sizeof(buf0), "the waves' staging rows fit an operand buffer");
    const int col = (lane % LR) * 8, n = n0 + rb + col;  // the lane's columns in every row
    const f32x8 bias = bias8<T>(e, n, s.N);
#pragma unroll 1
    for (int i = 0; i < MI; ++i) {
#pragma unroll
        for (int ii = 0; ii < MI; ++ii) {  // (accumulators are only ever named by constants: else they go to memory)
            if (ii != i) continue;
#pragma unroll
            for (int j = 0; j < NI; ++j)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    stage[((r & 3) + 8 * (r >> 2) + 4 * (lane >> 5)) * CW + j * 32 + (lane & 31)] = acc[ii][j][r];
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int q = 0; q < 32 / RP; ++q) {
            const int row = q * RP + lane / LR;
            const f32x8 v = *reinterpret_cast<const f32x8*>(stage + row * CW + col);
            const int64_t m = m0 + ra + i * 32 + row;
            if (m >= s.M || n >= s.N) continue;
            if (s.ksplit > 1) {
                float* o = s.part + ((int64_t)split * s.M + m) * s.N + n;
                if (n + 8 <= s.N && s.N % 4 == 0) {
                    reinterpret_cast<float4*>(o)[0] = make_float4(v[0], v[1], v[2], v[3]);
                    reinterpret_cast<float4*>(o)[1] = make_float4(v[4], v[5], v[6], v[7]);
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (n + j < s.N) o[j] = v[j];
                }
            } else {
                finish8<T>(e, v, bias, m, n, s.N);
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
}

// Few rows (a token or a small batch of them): the time is one read of w.  A block computes 16 columns of y: its eight waves
// take K in turns of 64 bytes a row, operands straight from memory into the MFMA's registers (16 x 16 x 32, fp32 16 x 16 x 4; rows at
// any alignment, four turns' loads in flight), and their sums meet in LDS, added in order, where the epilogue follows.  No
// workspace, one launch.
template <typename T> struct Mfma16;
template <> struct Mfma16<float> {
    static __device__ __forceinline__ f32x4 go(f32x4 a, f32x4 b, f32x4 c) {
#pragma unroll
        for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
        return c;
    }
};
template <> struct Mfma16<bf16_t> {
    typedef Mfma<bf16_t>::V V;
    static __device__ __forceinline__ f32x4 go(V a, V b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <> struct Mfma16<f16_t> {
    typedef Mfma<f16_t>::V V;
    static __device__ __forceinline__ f32x4 go(V a, V b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};

template <typename T, int MI>
__global__ __launch_bounds__(512) void linear_rows_kernel(const T* __restrict__ x, int64_t ldx, const T* __restrict__ w, int64_t ldw, int M,
                                                          int N, int K, Epilogue e) {
    constexpr int W = 8, VEC = GR<T>, KS = 4 * VEC, U = 4;
    typedef typename Mfma<T>::V V;
    __shared__ __attribute__((aligned(16))) float part[W][MI * 16][16];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int n0 = (int)blockIdx.x * 16;
    // (rows behind the last are that one, and never stored)
    const T* wr = w + (int64_t)min(n0 + r, N - 1) * ldw;
    const T* xr[MI];
#pragma unroll
    for (int i = 0; i < MI; ++i) xr[i] = x + (int64_t)min(i * 16 + r, M - 1) * ldx;
    f32x4 acc[MI];
#pragma unroll
    for (int i = 0; i < MI; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int turns = K / KS;
    GranU<T, VEC> wv[U], xv[U][MI];
    // (two turns in a row to a wave: a cache line of every row)
    const auto turn = [](int s, int u) { return s + u / 2 * (2 * W) + u % 2; };
    for (int s = 2 * wave; s < turns; s += W * U) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = min(turn(s, u), turns - 1) * KS + g * VEC;
            wv[u].load(wr + k);
#pragma unroll
            for (int i = 0; i < MI; ++i) xv[u][i].load(xr[i] + k);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (turn(s, u) >= turns) break;
#pragma unroll
            for (int i = 0; i < MI; ++i) acc[i] = Mfma16<T>::go(__builtin_bit_cast(V, wv[u].v), __builtin_bit_cast(V, xv[u][i].v), acc[i]);
        }
    }
    if (K % KS != 0 && wave == turns / 2 % W) {  // the turn that K ends in
        load_cols<false, T, VEC>(wv[0], wr, turns * KS + g * VEC, K);
#pragma unroll
        for (int i = 0; i < MI; ++i) {
            load_cols<false, T, VEC>(xv[0][i], xr[i], turns * KS + g * VEC, K);
            acc[i] = Mfma16<T>::go(__builtin_bit_cast(V, wv[0].v), __builtin_bit_cast(V, xv[0][i].v), acc[i]);
        }
    }
    // a lane holds columns 4 g .. 4 g + 3 of row r of each 16
#pragma unroll
    for (int i = 0; i < MI; ++i) *reinterpret_cast<f32x4*>(&part[wave][i * 16 + r][g * 4]) = acc[i];
    __syncthreads();
    const int m = threadIdx.x >> 1, c = (threadIdx.x & 1) * 8;
    if (m >= M || n0 + c >= N) return;
    f32x8 v;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = part[0][m][c + j];
#pragma unroll
    for (int k = 1; k < W; ++k)
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] += part[k][m][c + j];
    finish8<T>(e, v, bias8<T>(e, n0 + c, N), m, n0 + c, N);
}

// What is left behind the tile kernel, in one launch: blocks begin[i] .. begin[i + 1] add the partials of product i's K splits in
// order and apply its epilogue, 8 columns a thread; the last ones add the rows of db's partial sums in a fixed order, 8 columns a
// block, 32 threads to a column.
struct Rest {
    const float* part[2]; int ksplit[2]; int64_t M[2]; int N[2]; Epilogue e[2];
    const float* sums; int n; int64_t C; void* db; int db_f32;
    int begin[3];
};

template <typename T>
__global__ __launch_bounds__(256) void linear_rest_kernel(Rest a) {
    __shared__ float red[32][9];
    const int block = (int)blockIdx.x;
    if (block >= a.begin[2]) {
        const int tx = threadIdx.x & 7, ty = threadIdx.x >> 3;
        const int64_t c = (int64_t)(block - a.begin[2]) * 8 + tx;
        float s = 0.f;
        if (c < a.C)
            for (int i = ty; i < a.n; i += 32) s += a.sums[(int64_t)i * a.C + c];
        red[ty][tx] = s;
        __syncthreads();
        if (ty != 0 || c >= a.C) return;
#pragma unroll
        for (int i = 1; i < 32; ++i) s += red[i][tx];
        if (a.db_f32) reinterpret_cast<float*>(a.db)[c] = s;
        else reinterpret_cast<T*>(a.db)[c] = (T)s;
        return;
    }
    const int which = block >= a.begin[1];
    const Epilogue& e = a.e[which];
    const float* part = a.part[which];
    const int64_t M = a.M[which];
    const int N = a.N[which], ksplit = a.ksplit[which], per = (N + 7) / 8;
    const int64_t i = (int64_t)(block - a.begin[which]) * 256 + threadIdx.x;
    if (i >= M * per) return;
    const int64_t m = i / per;
    const int n = (int)(i % per) * 8;
    f32x8 v;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = 0.f;
    for (int k = 0; k < ksplit; ++k) {
        const float* p = part + ((int64_t)k * M + m) * N + n;
        if (n + 8 <= N && N % 4 == 0) {
            const float4 f = reinterpret_cast<const float4*>(p)[0], g = reinterpret_cast<const float4*>(p)[1];
            v[0] += f.x; v[1] += f.y; v[2] += f.z; v[3] += f.w;
            v[4] += g.x; v[5] += g.y; v[6] += g.z; v[7] += g.w;
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (n + j < N) v[j] += p[j];
        }
    }
    finish8<T>(e, v, bias8<T>(e, n, N), m, n, N);
}

// ---- operands into the form the tile kernel takes -----------------------------------------------------------------
// dst [R, ldd] = src [R, C], columns C .. ldd zero; ldd is a multiple of a granule, src starts and ends anywhere.  A launch
// copies one or two matrices: blocks 0 .. first - 1 are the first one's.
struct Pack { const void* src; int64_t ld, R, C; void* dst; int64_t ldd; };
struct Packs { Pack job[2]; int first; };

template <typename T>
__global__ __launch_bounds__(256) void linear_pack_kernel(Packs p) {
    const int which = (int)blockIdx.x >= p.first;
    const Pack& j = p.job[which];
    const T* __restrict__ src = (const T*)j.src;
    T* __restrict__ dst = (T*)j.dst;
    const int64_t per = j.ldd / GR<T>, n = j.R * per;
    const int block = (int)blockIdx.x - (which ? p.first : 0), blocks = which ? (int)gridDim.x - p.first : p.first;
    for (int64_t i = (int64_t)block * 256 + threadIdx.x; i < n; i += (int64_t)blocks * 256) {
        const int64_t r = i / per;
        const int c = (int)(i - r * per) * GR<T>;
        GranU<T, GR<T>> g;
        load_cols<false, T, GR<T>>(g, src + r * j.ld, c, (int)j.C);
        g.store(dst + r * j.ldd + c);
    }
}

// One pass over a [R, C] matrix in 64 x 64 tiles (a block walks the row tiles first, + stride, .. of one column tile):
//   v = src                      (z NULL)
//   v = src * act'(z)            else (z as linear_tile_kernel's epilogue kept it)
// out [R, ldo] (NULL: not wanted) gets v, columns C .. ldo zero; outT [C, ldt] (NULL) its transpose, columns R .. ldt zero;
// sums [stride][C] (NULL) the block's column sums of the unrounded v.  parts = 2 (16-bit types): out and outT get v's low parts, and
// its high ones `out_part` / `outT_part` elements behind.
// A thread moves eight neighbouring elements of a row.  The tile keeps its eight (r, chunk) at chunk ^ (r / 8): the eight lanes
// that gather one column's 64 rows then read eight different banks.
// A launch makes several such passes (dy, w and x of one backward call): blocks begin[i] .. begin[i + 1] belong to the i-th.
struct Turn {
    const void* src; int64_t ld;
    const void* z; int64_t ldz;
    int64_t R, C;
    void* out; int64_t ldo;
    void* outT; int64_t ldt;
    int parts; int64_t out_part, outT_part;
    float* sums;
    int stride;  // blocks along the rows
    int stream;  // the outputs are larger than what the caches keep until the products read them: streaming stores
};
struct Turns { Turn job[3]; int begin[4]; };

// columns c .. c + 7 of a row of ld elements
template <typename T>
__device__ __forceinline__ void turn_row(const GranU<T, 8>& g, T* row, int64_t c, int64_t ld, int stream) {
    if (c + 8 <= ld) {
        if (stream) g.store_nt(row + c);
        else g.store(row + c);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (c + j < ld) row[c + j] = g.v[j];
    }
}

template <typename T, int ACT>
__global__ __launch_bounds__(256) void linear_turn_kernel(Turns jobs) {
    constexpr bool APART = sizeof(T) == 2 && (ACT == DSSVAE_ACT_GELU || ACT == DSSVAE_ACT_SILU || ACT == DSSVAE_ACT_TANH);
    __shared__ __attribute__((aligned(16))) T tile[APART ? 2 : 1][64 * 64];
    __shared__ float red[32][64];
    int which = 0;
    while ((int)blockIdx.x >= jobs.begin[which + 1]) ++which;
    const Turn& t = jobs.job[which];
    const T *__restrict__ src = (const T*)t.src, *__restrict__ z = (const T*)t.z;
    T *__restrict__ out = (T*)t.out, *__restrict__ outT = (T*)t.outT;
    float* __restrict__ sums = t.sums;
    const int64_t ld = t.ld, ldz = t.ldz, R = t.R, C = t.C, ldo = t.ldo, ldt = t.ldt;
    const int block = (int)blockIdx.x - jobs.begin[which], stride = t.stride, first = block % stride;
    const int64_t c0 = (int64_t)(block / stride) * 64;
    const int ch = threadIdx.x & 7, rr = threadIdx.x >> 3;
    const int64_t rtiles = (R + 63) / 64, c = c0 + ch * 8;
    float sum[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) sum[j] = 0.f;
    for (int64_t rt = first; rt < rtiles; rt += stride) {
        const int64_t r0 = rt * 64;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int tr = i * 32 + rr;
            const int64_t r = r0 + tr;
            float v[8];
            GranU<T, 8> g;
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = 0.f;
            if (r < R && c < C) {
                if (c + 8 <= C) {
                    g.load(src + r * ld + c);
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[j] = g.get(j);
                    if (z) {
                        if constexpr (sizeof(T) == 4) {
                            g.load(z + r * ldz + c);
#pragma unroll
                            for (int j = 0; j < 8; ++j) v[j] *= act_slope<T>(ACT, g.get(j));
                        } else {
                            GranU<int16_t, 8> gq;
                            gq.load(reinterpret_cast<const int16_t*>(z) + r * ldz + c);
#pragma unroll
                            for (int j = 0; j < 8; ++j) v[j] *= decode<ACT>(gq.v[j]);
                        }
                    }
                } else {
                    for (int j = 0; j < 8 && c + j < C; ++j) {
                        float u = (float)src[r * ld + c + j];
                        if (z) u *= slope_kept<T, ACT>(z, r * ldz + c + j);
#pragma unroll
                        for (int jj = 0; jj < 8; ++jj) v[jj] = jj == j ? u : v[jj];
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                sum[j] += v[j];
                g.set(j, v[j]);
            }
            if constexpr (APART) {
                if (t.parts == 2) {
                    GranU<T, 8> hi;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        T l, h;
                        Apart<T>::of(v[j], l, h);
                        g.v[j] = l;
                        hi.v[j] = h;
                    }
                    if (out && r < R) turn_row(hi, out + t.out_part + r * ldo, c, ldo, t.stream);
                    if (outT) hi.store(tile[1] + tr * 64 + (ch ^ (tr >> 3)) * 8);
                }
            }
            if (out && r < R) turn_row(g, out + r * ldo, c, ldo, t.stream);
            if (outT) g.store(tile[0] + tr * 64 + (ch ^ (tr >> 3)) * 8);
        }
        if (outT) {
            __syncthreads();
#pragma unroll
            for (int q = 0; q < (APART ? 2 : 1); ++q) {
                if (q > 0 && t.parts < 2) break;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    // lane ch gathers rows 8 ch .. of column i * 32 + rr
                    const int tc = i * 32 + rr;
                    GranU<T, 8> g;
#pragma unroll
                    for (int j = 0; j < 8; ++j) g.v[j] = tile[q][(ch * 8 + j) * 64 + ((tc >> 3) ^ ch) * 8 + (tc & 7)];
                    if (c0 + tc < C) turn_row(g, outT + q * t.outT_part + (c0 + tc) * ldt, r0 + ch * 8, ldt, t.stream);
                }
            }
            __syncthreads();
        }
    }
    if (!sums) return;
#pragma unroll
    for (int j = 0; j < 8; ++j) red[rr][ch * 8 + j] = sum[j];
    __syncthreads();
    if (threadIdx.x < 64 && c0 + threadIdx.x < C) {
        float s = 0.f;
        for (int i = 0; i < 32; ++i) s += red[i][threadIdx.x];
        sums[(int64_t)first * C + c0 + threadIdx.x] = s;
    }
}

// ---- host ---------------------------------------------------------------------------------------------------------
inline int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

// Tile width and K splits of a launch's products: the smallest of a modelled time in microseconds,
//   max(work of all blocks over the CUs, the longest block's steps) + prologue and epilogue + partials' traffic,
// with `per` the time of a step at a CU's full rate and `least` what a step takes a block alone (the latency of its loads).  The
// work counts as if every CU took as many blocks as the fullest.  (Every width and split of 46 forward
// shapes: within 13 % of the best choice but for four with few tiles and a long K, bf16 300 x 7936 -> 600 22.6 us
// against 16.7 and 256 x 16384 -> 256 19.4 against 16.2, fp32 512 x 4096 -> 4096 134 against 105 and 300 x 7936 -> 600 44 against 37.)
struct Plan { int tile, ksplit; };
struct Extent { int64_t M, N, K; };
template <typename T> constexpr int MAX_TILE = sizeof(T) == 4 ? 128 : 256;
template <typename T, int COUNT>
inline double plan_products(const Extent (&x)[COUNT], Plan (&best)[COUNT]) {
    static const int splits[] = {1, 2, 3, 4, 6, 8, 12, 16, 24, 32};
    const bool f32 = sizeof(T) == 4;
    const double cus = device_cus();
    double lowest = -1;
    for (int tile = MAX_TILE<T>; tile >= 64; tile /= 2) {
        const double per = f32 ? (tile == 128 ? 1.33 : 0.5) : tile == 256 ? 1.68 : tile == 128 ? 0.57 : 0.3;
        const double least = f32 ? (tile == 128 ? 1.45 : 0.5) : tile == 256 ? 1.7 : tile == 128 ? 0.8 : 0.35;
        const double wait = tile == 256 ? 8 : tile == 128 ? 5 : 3;
        double work = 0;
        for (const Extent& e : x) work += (double)(up(e.M, tile) / tile) * (double)(up(e.N, tile) / tile) * (double)(up(e.K, BK<T>) / BK<T>);
        work *= per / cus;
        double blocks = 0, chain = 0, join = 0;
        Plan p[COUNT];
        for (int i = 0; i < COUNT; ++i) {
            const Extent& e = x[i];
            const int64_t nk = up(e.K, BK<T>) / BK<T>;
            double low = -1, chain_i = 0, join_i = 0;
            for (int ks : splits) {
                if (ks > 1 && nk / ks < 4) break;
                const double steps = (double)((nk + ks - 1) / ks) * least;
                const double more = ks > 1 ? 6 + (double)(2 * ks + 1) * (double)e.M * (double)e.N * 4 / 6e6 : 0;
                const double cost = (steps > work ? steps : work) + more;
                if (low < 0 || cost < low) {
                    low = cost;
                    chain_i = steps;
                    join_i = more;
                    p[i] = Plan{tile, ks};
                }
            }
            blocks += (double)(up(e.M, tile) / tile) * (double)(up(e.N, tile) / tile) * p[i].ksplit / cus;
            chain = chain_i > chain ? chain_i : chain;
            join += join_i;
        }
        const double full = blocks > 1 ? work * (double)((int64_t)blocks + (blocks > (double)(int64_t)blocks)) / blocks : work;
        const double cost = (full > chain ? full : chain) + wait + join;
        if (lowest < 0 || cost < lowest) {
            lowest = cost;
            for (int i = 0; i < COUNT; ++i) best[i] = p[i];
        }
    }
    return lowest;
}
// tile 0: linear_rows_kernel, where its modelled time is the smaller: 3.5 us and 45 GB/s a CU for what its blocks load, 16 rows of
// w and up to 64 of x each.  Measured against the tiles, bf16, M x K -> N: 1 x 1024 -> 1024 4.1 / 7.3 us, 50 x 600 -> 300 5.4 / 7.2, 50 x 2048
// -> 2048 10.8 / 10.1, 50 x 4096 -> 4096 21 / 15 (taken by the tiles); fp32: 1 x 2048 -> 8192 14.6 / 24.7, 50 x 8192 -> 2048 67 / 29 (tiles).
constexpr int64_t FEW_ROWS = 64;
inline int row_blocks(int64_t M) { return M <= 16 ? 1 : M <= 32 ? 2 : 4; }  // of 16 rows
template <typename T>
inline Plan plan(int64_t M, int64_t N, int64_t K) {
    const Extent x[1] = {{M, N, K}};
    Plan p[1];
    const double tiles = plan_products<T, 1>(x, p);
    if (M <= FEW_ROWS) {
        const int64_t cus = device_cus(), turns = (up(N, 16) / 16 + cus - 1) / cus;
        if (3.5 + (double)turns * (double)(K * (int64_t)sizeof(T)) * 16 * (1 + row_blocks(M)) / 45e3 < tiles) return Plan{0, 1};
    }
    return p[0];
}
// dx [M, K] over N and dw [N, K] over M, whichever of them a call wants (its bits do not depend on that); dz in one or two parts
struct Plans { Plan x, w; };
template <typename T>
inline Plans plan_bwd(int64_t M, int64_t N, int64_t K, int parts) {
    const Extent x[2] = {{M, K, parts * up(N, parts > 1 ? BK<T> : GR<T>)}, {N, K, parts * up(M, parts > 1 ? BK<T> : GR<T>)}};
    Plan p[2];
    plan_products<T, 2>(x, p);
    return Plans{p[0], p[1]};
}
inline int64_t part_bytes(const Plan& p, int64_t M, int64_t N) { return p.ksplit > 1 ? up((int64_t)p.ksplit * M * N * 4, 256) : 0; }

// operand rows usable as they are: 16-byte granules, and the 256 rows of a tile within 32-bit byte offsets
constexpr int64_t MAX_LD = 1 << 21;
template <typename T>
inline bool direct(const void* p, int64_t ld, int64_t K) {
    return aligned_to(p, 16) && ld % GR<T> == 0 && K % GR<T> == 0 && ld <= MAX_LD;
}

// C [M, N] = A [M, K] . B [N, K]^T and its epilogue, as a list of up to two for one launch
template <typename T>
struct Products {
    Jobs jobs{};
    Rest rest{};
    int n = 0, tile = 0;
    int add(const Plan& p, const void* A, int64_t lda, const void* B, int64_t ldb, int64_t M, int64_t N, int64_t K, const Epilogue& e,
            void* part, int parts = 1) {
        if (M == 0 || N == 0) return DSSVAE_OK;
        Shape s;
        s.A = A; s.lda = lda; s.B = B; s.ldb = ldb; s.M = M; s.N = (int)N; s.K = K;
        s.parts = parts; s.part_at = M * lda;
        const int64_t tm = up(M, p.tile) / p.tile, tn = up(N, p.tile) / p.tile, blocks = tm * tn * p.ksplit;
        const int64_t join = p.ksplit > 1 ? (M * ((N + 7) / 8) + 255) / 256 : 0;
        if (!grid_fits(2 * blocks, 512) || !grid_fits(2 * join, 512)) return DSSVAE_ETOOBIG;  // (two products to a launch)
        s.tiles_m = (int)tm; s.tiles_n = (int)tn; s.ksplit = p.ksplit;
        const int64_t nk = parts * (up(K, BK<T>) / BK<T>);
        s.ktiles = (nk + p.ksplit - 1) / p.ksplit;
        s.part = (float*)part;
        jobs.job[n] = Job{s, e, (int)blocks};
        if (n == 0) jobs.first = (int)blocks;
        rest.part[n] = s.part; rest.ksplit[n] = p.ksplit; rest.M[n] = M; rest.N[n] = (int)N; rest.e[n] = e;
        rest.begin[n + 1] = rest.begin[n] + (int)join;
        tile = p.tile;
        ++n;
        return DSSVAE_OK;
    }
    int run(hipStream_t st) {
        if (n == 0) return DSSVAE_OK;
        if (n > 1 && jobs.job[1].s.ktiles > jobs.job[0].s.ktiles) {  // the blocks with more steps start first
            const Job j = jobs.job[0];
            jobs.job[0] = jobs.job[1];
            jobs.job[1] = j;
            jobs.first = jobs.job[0].blocks;
        }
        const dim3 grid((unsigned)(jobs.first + (n > 1 ? jobs.job[1].blocks : 0)));
        if (tile == 256) {
            if constexpr (sizeof(T) == 2) hipLaunchKernelGGL((linear_tile_kernel<T, 256, 256, 2, 4>), grid, dim3(512), 0, st, jobs);
        } else if (tile == 128) {
            hipLaunchKernelGGL((linear_tile_kernel<T, 128, 128, 2, 2>), grid, dim3(256), 0, st, jobs);
        } else {
            hipLaunchKernelGGL((linear_tile_kernel<T, 64, 64, 2, 2>), grid, dim3(256), 0, st, jobs);
        }
        DSSVAE_CHECK_LAUNCH();
        return DSSVAE_OK;
    }
    // the splits' partials and, with db, its column sums from n_sums rows of partial ones
    int finish(hipStream_t st, const float* sums = nullptr, int n_sums = 0, int64_t C = 0, void* db = nullptr, int db_f32 = 0) {
        for (int i = n; i < 2; ++i) rest.begin[i + 1] = rest.begin[i];
        rest.sums = sums; rest.n = n_sums; rest.C = C; rest.db = db; rest.db_f32 = db_f32;
        const int64_t blocks = rest.begin[2] + (db ? (C + 7) / 8 : 0);
        if (!grid_fits(blocks, 256)) return DSSVAE_ETOOBIG;
        if (blocks == 0) return DSSVAE_OK;
        hipLaunchKernelGGL((linear_rest_kernel<T>), dim3((unsigned)blocks), dim3(256), 0, st, rest);
        DSSVAE_CHECK_LAUNCH();
        return DSSVAE_OK;
    }
};

struct PackList {
    Packs p{};
    int n = 0, blocks = 0;
    void add(const void* src, int64_t ld, int64_t R, int64_t C, void* dst, int64_t ldd, int granule) {
        const int64_t need = (R * (ldd / granule) + 255) / 256, most = 16 * (int64_t)device_cus();
        p.job[n] = Pack{src, ld, R, C, dst, ldd};
        if (n == 0) p.first = (int)(need < most ? need : most);
        blocks += (int)(need < most ? need : most);
        ++n;
    }
};
template <typename T>
int pack(const PackList& l, hipStream_t st) {
    if (l.blocks == 0) return DSSVAE_OK;
    hipLaunchKernelGGL((linear_pack_kernel<T>), dim3((unsigned)l.blocks), dim3(256), 0, st, l.p);
    DSSVAE_CHECK_LAUNCH();
    return DSSVAE_OK;
}

// blocks along the rows of linear_turn_kernel: enough to fill the chip
inline int64_t turn_rows(int64_t R, int64_t C) {
    const int64_t ct = (C + 63) / 64, rt = (R + 63) / 64, want = (8 * (int64_t)device_cus() + ct - 1) / ct;
    return rt < 1 ? 1 : rt < want ? rt : want;  // (at most 8 blocks a CU and one per column tile: begin[] stays small)
}
struct TurnList {
    int64_t es;
    Turns t{};
    int n = 0;
    void add(const void* src, int64_t ld, const void* z, int64_t ldz, int64_t R, int64_t C, void* out, int64_t ldo, void* outT, int64_t ldt,
             float* sums, int parts = 1) {
        const int64_t rows = turn_rows(R, C);
        // (streaming stores: 8192 x 16384 bf16, two outputs, 302 -> 268 us; at 10-20 MB they cost the product behind it 13 us of 43)
        const int stream = R * C * es * parts * ((out != nullptr) + (outT != nullptr)) > (int64_t)128 << 20;
        t.job[n] = Turn{src, ld, z, ldz, R, C, out, ldo, outT, ldt, parts, R * ldo, C * ldt, sums, (int)rows, stream};
        t.begin[n + 1] = t.begin[n] + (int)(rows * ((C + 63) / 64));
        ++n;
    }
};
template <typename T>
int turn(const TurnList& l, int act, hipStream_t st) {
    if (l.n == 0) return DSSVAE_OK;
    Turns t = l.t;
    for (int i = l.n; i < 3; ++i) t.begin[i + 1] = t.begin[l.n];
    const dim3 grid((unsigned)t.begin[l.n]);
#define GO(ACT)                                                                                                        \
    if (act == ACT) hipLaunchKernelGGL((linear_turn_kernel<T, ACT>), grid, dim3(256), 0, st, t)
    GO(DSSVAE_ACT_NONE); GO(DSSVAE_ACT_RELU); GO(DSSVAE_ACT_GELU); GO(DSSVAE_ACT_SILU); GO(DSSVAE_ACT_TANH);
#undef GO
    DSSVAE_CHECK_LAUNCH();
    return DSSVAE_OK;
}

// workspace pieces, each on a 256-byte boundary
struct Space {
    char* p; int64_t used, size;
    void* take(int64_t bytes) {
        void* r = p ? p + used : nullptr;
        used += up(bytes, 256);
        return r;
    }
};

bool bad_args(int dtype, int act, int64_t M, int N, int K) {
    return !dtype_ok(dtype) || act < DSSVAE_ACT_NONE || act > DSSVAE_ACT_TANH || M < 0 || M > 0x7fffffff || N < 1 || K < 1 ||
           N > (1 << 30) || K > (1 << 30);
}

template <typename T>
int few_rows(const void* x, int64_t ldx, const void* w, int64_t ldw, int M, int N, int K, const Epilogue& e, hipStream_t st) {
    const int64_t blocks = ((int64_t)N + 15) / 16;
    if (!grid_fits(blocks, 512)) return DSSVAE_ETOOBIG;
#define GO(MI)                                                                                                      \
    hipLaunchKernelGGL((linear_rows_kernel<T, MI>), dim3((unsigned)blocks), dim3(512), 0, st, (const T*)x, ldx, (const T*)w, ldw, M, N, K, e)
    if (row_blocks(M) == 1) GO(1);
    else if (row_blocks(M) == 2) GO(2);
    else GO(4);
#undef GO
    DSSVAE_CHECK_LAUNCH();
    return DSSVAE_OK;
}

// (`p`: plan of the product, made where the call's workspace is added up and used where it is launched)
template <typename T>
int forward(const void* x, int64_t ldx, const void* w, int64_t ldw, int64_t M, int N, int K, const Epilogue& e, Space& sp, hipStream_t st,
            bool dry, Plan& p) {
    const int64_t ldk = up(K, GR<T>), es = sizeof(T);
    if (dry) p = plan<T>(M, N, ldk);
    if (p.tile == 0) return dry ? DSSVAE_OK : few_rows<T>(x, ldx, w, ldw, (int)M, N, K, e, st);
    PackList packs;
    if (!direct<T>(x, ldx, K)) {
        void* d = sp.take(M * ldk * es);
        packs.add(x, ldx, M, K, d, ldk, GR<T>);
        x = d; ldx = ldk;
    }
    if (!direct<T>(w, ldw, K)) {
        void* d = sp.take((int64_t)N * ldk * es);
        packs.add(w, ldw, N, K, d, ldk, GR<T>);
        w = d; ldw = ldk;
    }
    void* part = sp.take(part_bytes(p, M, N));
    if (dry) return DSSVAE_OK;
    int rc = pack<T>(packs, st);
    if (rc) return rc;
    Products<T> l;
    rc = l.add(p, x, ldx, w, ldw, M, N, ldk, e, part);
    if (!rc) rc = l.run(st);
    return rc ? rc : l.finish(st);
}

struct BwdArgs {
    const void *dy, *z, *x, *w;
    int64_t lddy, ldz, ldx, ldw, lddx, lddw;
    void *dx, *dw, *db;
    int db_f32, act;
    int64_t M; int N, K;
    int parts;    // of dz: 2 where dy act'(z) is no number of the type
    Plans plans;  // made by the pass that adds up the workspace
};

template <typename T>
int backward(BwdArgs& a, Space& sp, hipStream_t st, bool dry) {
    const int64_t M = a.M, N = a.N, K = a.K, es = sizeof(T), whole = a.parts > 1 ? BK<T> : GR<T>, ldn = up(N, whole), ldm = up(M, whole);
    int rc = DSSVAE_OK;
    // dz: a copy where it differs from dy or dy's rows cannot be loaded as they are
    const bool copy = a.dx && (a.z || !direct<T>(a.dy, a.lddy, N));
    const void* dz = a.dy;
    int64_t lddz = a.lddy;
    void *dzc = nullptr, *dzt = nullptr;
    if (copy) { dzc = sp.take(a.parts * M * ldn * es); dz = dzc; lddz = ldn; }
    if (a.dw) dzt = sp.take(a.parts * N * ldm * es);
    float* sums = a.db ? (float*)sp.take(turn_rows(M, N) * N * 4) : nullptr;
    void* wt = a.dx ? sp.take(K * ldn * es) : nullptr;
    void* xt = a.dw ? sp.take(K * ldm * es) : nullptr;
    if (dry) a.plans = plan_bwd<T>(M, N, K, a.parts);
    const Plans& p = a.plans;
    void* part_x = a.dx ? sp.take(part_bytes(p.x, M, K)) : nullptr;
    void* part_w = a.dw ? sp.take(part_bytes(p.w, N, K)) : nullptr;
    if (dry) return rc;
    TurnList l{es};
    if (copy || a.dw || a.db) l.add(a.dy, a.lddy, a.z, a.ldz, M, N, dzc, ldn, dzt, ldm, sums, a.parts);
    if (a.dx) l.add(a.w, a.ldw, nullptr, 0, N, K, nullptr, 0, wt, ldn, nullptr);
    if (a.dw) l.add(a.x, a.ldx, nullptr, 0, M, K, nullptr, 0, xt, ldm, nullptr);
    if ((rc = turn<T>(l, a.act, st))) return rc;
    Products<T> q;
    if (a.dx) {
        Epilogue e{};
        e.y = a.dx; e.ldy = a.lddx;
        if ((rc = q.add(p.x, dz, lddz, wt, ldn, M, K, ldn, e, part_x, a.parts))) return rc;
    }
    if (a.dw) {
        Epilogue e{};
        e.y = a.dw; e.ldy = a.lddw;
        if ((rc = q.add(p.w, dzt, ldm, xt, ldm, N, K, ldm, e, part_w, a.parts))) return rc;
    }
    if ((rc = q.run(st))) return rc;
    return q.finish(st, sums, a.db ? (int)turn_rows(M, N) : 0, N, a.db, a.db_f32);
}

int bwd_any(int dtype, BwdArgs& a, Space& sp, hipStream_t st, bool dry) {
    if (dtype == DSSVAE_F32) return backward<float>(a, sp, st, dry);
    return dtype == DSSVAE_BF16 ? backward<bf16_t>(a, sp, st, dry) : backward<f16_t>(a, sp, st, dry);
}

}  // namespace

namespace {
int64_t fwd_space(const void* x, int64_t ldx, const void* w, int64_t ldw, int dtype, int64_t M, int N, int K, Plan& p) {
    Space sp{nullptr, 0, 0};
    if (dtype == DSSVAE_F32) forward<float>(x, ldx, w, ldw, M, N, K, Epilogue{}, sp, nullptr, true, p);
    else forward<bf16_t>(x, ldx, w, ldw, M, N, K, Epilogue{}, sp, nullptr, true, p);  // (fp16: the same sizes)
    return sp.used;
}
}  // namespace

extern "C" int64_t dssvae_linear_act_fwd_workspace_bytes(const void* x, int64_t ldx, const void* w, int64_t ldw, int dtype,
                                                         int64_t M, int N, int K) {
    if (bad_args(dtype, DSSVAE_ACT_NONE, M, N, K)) return DSSVAE_EINVAL;
    Plan p;
    return fwd_space(x, ldx, w, ldw, dtype, M, N, K, p);
}

extern "C" int dssvae_linear_act_fwd(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias, int bias_f32,
                                     const void* res, int64_t ldr, int dtype, int act, int64_t M, int N, int K, void* y,
                                     int64_t ldy, void* z, int64_t ldz, void* workspace, int64_t workspace_bytes,
                                     void* stream) {
    if (bad_args(dtype, act, M, N, K) || ldx < K || ldw < K || ldy < N || (res && ldr < N) || (z && ldz < N)) return DSSVAE_EINVAL;
    if (M == 0) return DSSVAE_OK;
    if (K > MAX_LD) return DSSVAE_ETOOBIG;
    if (!x || !w || !y || (z && z == y)) return DSSVAE_EINVAL;
    Plan p;
    const int64_t need = fwd_space(x, ldx, w, ldw, dtype, M, N, K, p);
    if (need > 0 && (!workspace || workspace_bytes < need || !aligned_to(workspace, 16))) return DSSVAE_EINVAL;
    hipStream_t st = (hipStream_t)stream;
    Epilogue e{};
    e.bias = bias; e.bias_f32 = bias_f32 || dtype == DSSVAE_F32; e.res = res; e.ldr = ldr; e.z = z; e.ldz = ldz; e.y = y; e.ldy = ldy; e.act = act;
    Space sp{(char*)workspace, 0, workspace_bytes};
    if (dtype == DSSVAE_F32) return forward<float>(x, ldx, w, ldw, M, N, K, e, sp, st, false, p);
    if (dtype == DSSVAE_BF16) return forward<bf16_t>(x, ldx, w, ldw, M, N, K, e, sp, st, false, p);
    return forward<f16_t>(x, ldx, w, ldw, M, N, K, e, sp, st, false, p);
}

extern "C" int64_t dssvae_linear_act_bwd_workspace_bytes(const void* dy, int64_t lddy, int has_z, int dtype, int64_t M, int N, int K,
                                                         int want_dx, int want_dw, int want_db) {
    if (bad_args(dtype, DSSVAE_ACT_NONE, M, N, K)) return DSSVAE_EINVAL;
    static char some;
    BwdArgs a{};
    a.dy = dy; a.lddy = lddy; a.z = has_z ? &some : nullptr; a.M = M; a.N = N; a.K = K;
    a.dx = want_dx ? &some : nullptr; a.dw = want_dw ? &some : nullptr; a.db = want_db ? &some : nullptr;
    int64_t most = 0;
    for (a.parts = 1; a.parts <= (has_z && dtype != DSSVAE_F32 ? 2 : 1); ++a.parts) {  // (whatever the activation)
        Space sp{nullptr, 0, 0};
        bwd_any(dtype, a, sp, nullptr, true);
        most = sp.used > most ? sp.used : most;
    }
    return most;
}

extern "C" int dssvae_linear_act_bwd(const void* dy, int64_t lddy, const void* z, int64_t ldz, const void* x, int64_t ldx,
                                     const void* w, int64_t ldw, int dtype, int act, int64_t M, int N, int K, void* dx,
                                     int64_t lddx, void* dw, int64_t lddw, void* db, int db_f32, void* workspace,
                                     int64_t workspace_bytes, void* stream) {
    const bool round_dz = act & DSSVAE_ACT_ROUND_DZ;
    act &= ~DSSVAE_ACT_ROUND_DZ;
    if (bad_args(dtype, act, M, N, K) || lddy < N || (z && ldz < N) || (dw && (ldx < K || lddw < K)) || (dx && (ldw < K || lddx < K)))
        return DSSVAE_EINVAL;
    if (act != DSSVAE_ACT_NONE && !z && M > 0) return DSSVAE_EINVAL;
    if ((M > 0 && (!dy || (dw && !x))) || (dx && !w)) return DSSVAE_EINVAL;
    if ((dx && N > MAX_LD) || (dw && M > MAX_LD)) return DSSVAE_ETOOBIG;
    BwdArgs a{};
    a.dy = dy; a.lddy = lddy; a.z = act == DSSVAE_ACT_NONE ? nullptr : z; a.ldz = ldz; a.x = x; a.ldx = ldx; a.w = w; a.ldw = ldw;
    a.dx = M > 0 ? dx : nullptr; a.lddx = lddx; a.dw = dw; a.lddw = lddw; a.db = db; a.db_f32 = db_f32 || dtype == DSSVAE_F32;
    a.act = act; a.M = M; a.N = N; a.K = K;
    a.parts = dtype != DSSVAE_F32 && act > DSSVAE_ACT_RELU && !round_dz ? 2 : 1;
    Space need{nullptr, 0, 0};
    bwd_any(dtype, a, need, nullptr, true);
    if (need.used > 0 && (!workspace || workspace_bytes < need.used || !aligned_to(workspace, 16))) return DSSVAE_EINVAL;
    Space sp{(char*)workspace, 0, workspace_bytes};
    return bwd_any(dtype, a, sp, (hipStream_t)stream, false);
}
