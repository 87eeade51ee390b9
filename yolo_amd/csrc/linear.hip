// Matrix product with bias, activation and residual in its epilogue, and its gradients, for gfx950.
//
//   P = x W^T + b          x [M][K], W [N][K], bf16 or fp16, fp32 accumulation on the matrix units
//   Y = act(P) + r
//   dP = dY * act'(P);  dX = dP W;  dW = dP^T x;  db = sum over rows of dP;  dr = dY
//
// The matrix units take 16-bit operands and dP is an fp32 value: where the operands' type does not hold it, it goes in as
// two parts of that type, dP = hi + lo up to its rounding squared (2^-16 relative in bf16, 2^-22 in fp16), and the products sum
// hi and lo of 64 reduction indices in turn into the same accumulators.  fp16 lacks fp32's range as well: there dP is
// multiplied by the power of two that brings its largest finite value to 2^14 .. 2^15, and the products' sums by its inverse.
//
// All three products are D[m][n] = sum_k A(m, k) B(n, k) with operands that are contiguous either along k
// (x and W in the forward product) or along their own rows' index (W in dX, dP and x in dW): one tile kernel
// takes both, the second kind through the transposing LDS read (ds_read_b64_tr_b16).
#include <algorithm>

#include "common.h"
#include "lds_dma.h"
#include "../../include/yolo_amd.h"

namespace yolo_amd {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
template <typename T> struct Vec;
template <> struct Vec<__bf16> { typedef __bf16 v8 __attribute__((ext_vector_type(8))); };
template <> struct Vec<_Float16> { typedef _Float16 v8 __attribute__((ext_vector_type(8))); };
template <typename T> using v8 = typename Vec<T>::v8;

__device__ __forceinline__ f32x4 mfma(v8<__bf16> a, v8<__bf16> b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma(v8<_Float16> a, v8<_Float16> b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// The same in place on accumulators held in accumulation registers: with 64 of them (all 256 registers) the
// compiler's own allocation rotates them through copies at every turn of a loop.  The compiler does not see that a
// matrix instruction is in flight: a kernel waits (mfma_drain) before it reads its accumulators otherwise.
__device__ __forceinline__ void mfma_in_place(v8<__bf16> a, v8<__bf16> b, f32x4& c) {
    asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
}
__device__ __forceinline__ void mfma_in_place(v8<_Float16> a, v8<_Float16> b, f32x4& c) {
    asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
}
// The same with a load of 16 bytes per lane to lds_dst + 16 * lane (lds_dma16_buf) behind it, in one statement: between the
// write of m0 and the load that reads it another instruction must lie and the compiler must not (8192^3: with s_nop there
// 745 us, with the matrix instruction 722).
#define YA_MFMA_LOAD(T, NAME)                                                                                              \
    __device__ __forceinline__ void mfma_in_place_load(v8<T> a, v8<T> b, f32x4& c, __amdgpu_buffer_rsrc_t rsrc, uint32_t voff, \
                                                       char* lds_dst) {                                                    \
        const uint32_t to = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds_dst;                         \
        asm volatile("s_mov_b32 m0, %5\n\t" NAME " %0, %1, %2, %0\n\tbuffer_load_dwordx4 %3, %4, 0 offen lds"              \
                     : "+a"(c) : "v"(a), "v"(b), "v"(voff), "s"(rsrc), "s"(to) : "memory", "m0");                          \
    }
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
YA_MFMA_LOAD(__bf16, "v_mfma_f32_16x16x32_bf16")
YA_MFMA_LOAD(_Float16, "v_mfma_f32_16x16x32_f16")
#pragma clang diagnostic pop
#undef YA_MFMA_LOAD
// more wait states than any matrix instruction's result takes (16 passes at most)
__device__ __forceinline__ void mfma_drain() { asm volatile("s_nop 15\n\ts_nop 15" ::: "memory"); }

// ---------------------------------------------------------------- activations
// exp2, reciprocal: the hardware's (1 ulp each).  erfc(x) for x >= 0 is t exp(-x^2) times a polynomial in t = 1 / (1 + 0.36 x),
// the form of Abramowitz and Stegun, Handbook of Mathematical Functions, 7.1.26, with a degree and coefficients of its own:
// fitted to erfc(x) exp(x^2) / t over x = 0 .. 9.5 so that the largest error is least, counted in units of 2e-8 of GELU and its slope
// or 4e-6 of erfc, whichever is larger there (it is 1.3 of them).  GELU in fp32 is off by at most 7.1e-8 (the sum
// 1 + erf loses 8.3e-8) and keeps five digits in its negative tail.  An epilogue of one activation per matrix-unit column is
// bound by the instructions of this: two terms fewer take 886 us instead of 900 at 8192 x 16384 x 4096 and leave 2.1e-7.
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kErfcT = 0.36f * 0.70710678118654752f;            // of |p|, x = |p| / sqrt 2
constexpr float kErfc[7] = {0.202154681f, 0.217184246f, 0.105075903f, 0.434264660f, -0.362271845f, 0.568214238f, -0.164621860f};
constexpr float kGeluC = 0.7978845608028654f, kGeluA = 0.044715f;

// erfc(|p| / sqrt 2) and exp(-p^2 / 2); NaN for NaN, 0 and 0 for infinities
__device__ __forceinline__ float erfc_scaled(float p, float& e) {
    const float t = __builtin_amdgcn_rcpf(fmaf(fabsf(p), kErfcT, 1.f));
    e = __builtin_amdgcn_exp2f(p * p * (-0.5f * kLog2e));
    float q = fmaf(t, kErfc[6], kErfc[5]);
#pragma unroll
    for (int k = 4; k >= 0; --k) q = fmaf(q, t, kErfc[k]);
    return q * t * e;
}

// max(p, 0) in one instruction (fmaxf would canonicalise p first); 0 for NaN
__device__ __forceinline__ float max0(float p) {
    float r;
    asm("v_max_f32 %0, %1, 0" : "=v"(r) : "v"(p));
    return r;
}

template <int ACT>
__device__ __forceinline__ float act_value(float p) {
    if constexpr (ACT == YOLO_AMD_ACT_LEAKY) return p > 0.f ? p : 0.1f * p;
    if constexpr (ACT == YOLO_AMD_ACT_RELU) return p < 0.f ? 0.f : p;
    if constexpr (ACT == YOLO_AMD_ACT_GELU) {
        // max(p, 0) - |p| erfc(|p| / sqrt 2) / 2; the clamp keeps inf * 0 out (erfc is 0 from 15 on), NaN comes through q
        float e;
        const float q = erfc_scaled(p, e);
        return fmaf(fabsf(__builtin_amdgcn_fmed3f(p, -100.f, 100.f)) * q, -0.5f, max0(p));
    }
    // (1 + tanh z) / 2 = 1 / (1 + exp(-2 z))
    if constexpr (ACT == YOLO_AMD_ACT_GELU_TANH)
        return p * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(p * fmaf(p * p, -2.f * kLog2e * kGeluC * kGeluA, -2.f * kLog2e * kGeluC)));
    if constexpr (ACT == YOLO_AMD_ACT_SILU) return p * sigmoid_fast(p);
    return p;
}
// Eight of them, stage by stage: one after the other, as the compiler likes to order them, every element waits for its
// own exponential and reciprocal, and an epilogue with one wave per SIMD has nothing else to run meanwhile.
template <int ACT>
__device__ __forceinline__ void act_values(float (&v)[2][4]) {
#define YA_EACH _Pragma("unroll") for (int i = 0; i < 8; ++i)
#define YA_STAGE() __builtin_amdgcn_sched_barrier(0)
    float* p = &v[0][0];
    if constexpr (ACT == YOLO_AMD_ACT_GELU) {
        float t[8], e[8], q[8];
        YA_EACH t[i] = fmaf(fabsf(p[i]), kErfcT, 1.f);
        YA_STAGE();
        YA_EACH t[i] = __builtin_amdgcn_rcpf(t[i]);
        YA_EACH e[i] = p[i] * p[i] * (-0.5f * kLog2e);
        YA_STAGE();
        YA_EACH e[i] = __builtin_amdgcn_exp2f(e[i]);
        YA_EACH q[i] = fmaf(t[i], kErfc[6], kErfc[5]);
        YA_STAGE();
#pragma unroll
        for (int k = 4; k >= 0; --k) {
            YA_EACH q[i] = fmaf(q[i], t[i], kErfc[k]);
            YA_STAGE();
        }
        YA_EACH q[i] = q[i] * t[i] * e[i];
        YA_STAGE();
        YA_EACH p[i] = fmaf(fabsf(__builtin_amdgcn_fmed3f(p[i], -100.f, 100.f)) * q[i], -0.5f, max0(p[i]));
    } else if constexpr (ACT == YOLO_AMD_ACT_GELU_TANH || ACT == YOLO_AMD_ACT_SILU) {
        float z[8];
        if constexpr (ACT == YOLO_AMD_ACT_SILU) {
            YA_EACH z[i] = p[i] * -kLog2e;
        } else {
            YA_EACH z[i] = p[i] * fmaf(p[i] * p[i], -2.f * kLog2e * kGeluC * kGeluA, -2.f * kLog2e * kGeluC);
        }
        YA_STAGE();
        YA_EACH z[i] = 1.f + __builtin_amdgcn_exp2f(z[i]);
        YA_STAGE();
        YA_EACH z[i] = __builtin_amdgcn_rcpf(z[i]);
        YA_STAGE();
        YA_EACH p[i] *= z[i];
    } else {
        YA_EACH p[i] = act_value<ACT>(p[i]);
    }
#undef YA_EACH
#undef YA_STAGE
}
__device__ __forceinline__ float act_value(float p, int act) {
    switch (act) {
        case YOLO_AMD_ACT_LEAKY: return act_value<YOLO_AMD_ACT_LEAKY>(p);
        case YOLO_AMD_ACT_RELU: return act_value<YOLO_AMD_ACT_RELU>(p);
        case YOLO_AMD_ACT_GELU: return act_value<YOLO_AMD_ACT_GELU>(p);
        case YOLO_AMD_ACT_GELU_TANH: return act_value<YOLO_AMD_ACT_GELU_TANH>(p);
        case YOLO_AMD_ACT_SILU: return act_value<YOLO_AMD_ACT_SILU>(p);
        default: return p;
    }
}

// act'(p).  From 100 on the curved ones have slope 1 and below -100 slope 0 in fp32: p is held there, so that no product
// of an infinity (of the sum itself, or of one past fp16's range kept in that type) and a zero arises.  NaN stays NaN.
template <int ACT>
__device__ __forceinline__ float act_slope(float p) {
    if constexpr (ACT == YOLO_AMD_ACT_LEAKY) return p > 0.f ? 1.f : 0.1f;
    if constexpr (ACT == YOLO_AMD_ACT_RELU) return p > 0.f ? 1.f : 0.f;
    if constexpr (ACT != YOLO_AMD_ACT_NONE) p = fabsf(p) > 100.f ? copysignf(100.f, p) : p;
    if constexpr (ACT == YOLO_AMD_ACT_GELU) {
        float e;
        const float q = 0.5f * erfc_scaled(p, e);
        return fmaf(p * 0.3989422804014327f, e, p < 0.f ? q : 1.f - q);
    }
    if constexpr (ACT == YOLO_AMD_ACT_GELU_TANH) {
        const float z = sigmoid_fast(2.f * kGeluC * (p + kGeluA * p * p * p));
        return z + p * z * (1.f - z) * 2.f * kGeluC * (1.f + 3.f * kGeluA * p * p);
    }
    if constexpr (ACT == YOLO_AMD_ACT_SILU) {
        const float z = sigmoid_fast(p);
        return z * (1.f + p * (1.f - z));
    }
    return 1.f;
}
// d *= act'(p)
template <int V>
__device__ __forceinline__ void times_slopes(float (&d)[V], const float (&p)[V], int act) {
#define YA_SLOPES(ACT)                                                   \
    case ACT:                                                            \
        _Pragma("unroll") for (int i = 0; i < V; ++i) d[i] *= act_slope<ACT>(p[i]); \
        break;
    switch (act) {
        YA_SLOPES(YOLO_AMD_ACT_LEAKY)
        YA_SLOPES(YOLO_AMD_ACT_RELU)
        YA_SLOPES(YOLO_AMD_ACT_GELU)
        YA_SLOPES(YOLO_AMD_ACT_GELU_TANH)
        YA_SLOPES(YOLO_AMD_ACT_SILU)
        default: break;
    }
#undef YA_SLOPES
}

// ---------------------------------------------------------------- epilogue
struct Epilogue {
    const void* bias;      // [N] or null
    const void* res;       // [M][ldr] or null
    void* y;               // [M][ldy]
    void* pre;             // [M][ldp] or null: P for the backward pass
    long long ldr, ldy, ldp;
    int bias_f32, res_f32, y_f32, pre_f32, act;
    const float* unscale;  // not null: the sums are multiplied by this first (products of the backward pass)
    float* part;           // not null: the raw sums of one K slice go to [slice][M][ld_part] instead
    long long ld_part, slice_stride;
};

// Rows of a user's tensor may start anywhere: 16-byte accesses at the elements' own alignment (the machine takes them;
// a wave that runs along a row touches one more line for it).
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x4u __attribute__((ext_vector_type(4), aligned(2)));
template <typename T>
__device__ __forceinline__ void load8(const void* p, long long at, int f32, float (&v)[8]) {
    if (f32) {
        const f32x4u a = *reinterpret_cast<const f32x4u*>((const float*)p + at);
        const f32x4u b = *reinterpret_cast<const f32x4u*>((const float*)p + at + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) { v[i] = a[i]; v[4 + i] = b[i]; }
    } else {
        const v8<T> a = __builtin_bit_cast(v8<T>, *reinterpret_cast<const u32x4u*>((const T*)p + at));
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (float)a[i];
    }
}
template <typename T>
__device__ __forceinline__ void store8(void* p, long long at, int f32, const float (&v)[8]) {
    if (f32) {
        f32x4u a, b;
#pragma unroll
        for (int i = 0; i < 4; ++i) { a[i] = v[i]; b[i] = v[4 + i]; }
        *reinterpret_cast<f32x4u*>((float*)p + at) = a;
        *reinterpret_cast<f32x4u*>((float*)p + at + 4) = b;
    } else {
        v8<T> a;
#pragma unroll
        for (int i = 0; i < 8; ++i) a[i] = (T)v[i];
        *reinterpret_cast<u32x4u*>((T*)p + at) = __builtin_bit_cast(u32x4u, a);
    }
}
template <typename T>
__device__ __forceinline__ float load1(const void* p, long long at, int f32) {
    return f32 ? ((const float*)p)[at] : (float)((const T*)p)[at];
}
template <typename T>
__device__ __forceinline__ void store1(void* p, long long at, int f32, float v) {
    if (f32) ((float*)p)[at] = v;
    else ((T*)p)[at] = (T)v;
}

// One sum of row m, column n: bias, activation, residual, one rounding, store.
template <typename T>
__device__ __forceinline__ void finish1(const Epilogue& e, long long m, int n, float s) {
    if (e.bias) s += load1<T>(e.bias, n, e.bias_f32);
    if (e.pre) store1<T>(e.pre, m * e.ldp + n, e.pre_f32, s);
    s = act_value(s, e.act);
    if (e.res) s += load1<T>(e.res, m * e.ldr + n, e.res_f32);
    store1<T>(e.y, m * e.ldy + n, e.y_f32, s);
}

// Eight sums of row m, columns n .. n + 7 (n a multiple of 8, n < N): bias, activation, residual, one
// rounding, store.
template <typename T>
__device__ __forceinline__ void finish8(const Epilogue& e, long long m, int n, int N, float (&v)[8]) {
    if (n + 8 <= N) {
        if (e.bias) {
            float b[8];
            load8<T>(e.bias, n, e.bias_f32, b);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] += b[i];
        }
        if (e.pre) store8<T>(e.pre, m * e.ldp + n, e.pre_f32, v);
        if (e.act) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = act_value(v[i], e.act);
        }
        if (e.res) {
            float r[8];
            load8<T>(e.res, m * e.ldr + n, e.res_f32, r);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] += r[i];
        }
        store8<T>(e.y, m * e.ldy + n, e.y_f32, v);
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (n + i < N) finish1<T>(e, m, n + i, v[i]);
}

// ---- from the accumulators of a wave, without LDS
// A wave's accumulator tile has lane l's row l & 15 and four columns (l >> 4) * 4 ..  Two neighbouring tiles, rounded
// and packed to two registers each, change lanes so that a lane holds eight consecutive columns: a 16-byte store of
// each lane then fills 64 contiguous bytes of 16 rows.  Swapping lane halves, then odd and even rows of 16 lanes, does
// it; the two swaps in the other order undo it.
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ void swap32(uint32_t& x, uint32_t& y) {
    const auto r = __builtin_amdgcn_permlane32_swap(x, y, false, false);
    x = r[0];
    y = r[1];
}
__device__ __forceinline__ void swap16(uint32_t& x, uint32_t& y) {
    const auto r = __builtin_amdgcn_permlane16_swap(x, y, false, false);
    x = r[0];
    y = r[1];
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    typedef T t2 __attribute__((ext_vector_type(2)));
    const t2 v = {(T)a, (T)b};
    return __builtin_bit_cast(uint32_t, v);
}
template <typename T>
__device__ __forceinline__ void unpack2(uint32_t u, float& a, float& b) {
    typedef T t2 __attribute__((ext_vector_type(2)));
    const t2 v = __builtin_bit_cast(t2, u);
    a = (float)v[0];
    b = (float)v[1];
}
// v: columns of two tiles -> the lane's 16 bytes
template <typename T>
__device__ __forceinline__ u32x4 pair_out(const float (&v)[2][4]) {
    uint32_t a0 = pack2<T>(v[0][0], v[0][1]), a1 = pack2<T>(v[0][2], v[0][3]);
    uint32_t b0 = pack2<T>(v[1][0], v[1][1]), b1 = pack2<T>(v[1][2], v[1][3]);
    swap32(a0, b0);
    swap32(a1, b1);
    swap16(a0, b0);
    swap16(a1, b1);
    return u32x4{a0, a1, b0, b1};
}
template <typename T>
__device__ __forceinline__ void pair_in(u32x4 u, float (&v)[2][4]) {
    uint32_t a0 = u[0], a1 = u[1], b0 = u[2], b1 = u[3];
    swap16(a0, b0);
    swap16(a1, b1);
    swap32(a0, b0);
    swap32(a1, b1);
    unpack2<T>(a0, v[0][0], v[0][1]);
    unpack2<T>(a1, v[0][2], v[0][3]);
    unpack2<T>(b0, v[1][0], v[1][1]);
    unpack2<T>(b1, v[1][2], v[1][3]);
}

// Four accumulators, read where they are used (IN_PLACE: see mfma_in_place; the compiler would fetch all 256 at once)
template <bool IN_PLACE>
__device__ __forceinline__ void acc_read(f32x4& c, float (&v)[4]) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if constexpr (IN_PLACE) asm volatile("v_accvgpr_read_b32 %0, %1" : "=v"(v[k]) : "a"(c[k]));
        else v[k] = c[k];
    }
}

// The wave's rows m0 .. and columns n0 ...  Whole eights of columns (below NV = N rounded down) are stored from here; the
// last one to seven columns of a row go, with bias and activation, through `tail` (LDS of this wave, [2][16 TM][8]:
// outputs, pre-activations) and are finished by element behind the loop, in code that is short because it is cold.
template <typename T, int ACT, bool IN_PLACE, bool SCALED, int TM, int TN>
__device__ __forceinline__ void finish_direct(const Epilogue& e, f32x4 (&acc)[TM][TN], int m0, int n0, int M, int N, int NV,
                                              int lane, float* tail) {
    const float factor = SCALED && e.unscale ? *e.unscale : 1.f;
    const int row = lane & 15, c4 = (lane >> 4) * 4, c8 = (lane >> 4) * 8;
    float bias[TN][4];
#pragma unroll
    for (int j = 0; j < TN; ++j) {
        const int n = n0 + j * 16 + c4;
#pragma unroll
        for (int k = 0; k < 4; ++k) bias[j][k] = 0.f;
        if (e.bias) {
#pragma unroll
            for (int k = 0; k < 4; ++k) bias[j][k] = load1<T>(e.bias, min(n + k, N - 1), e.bias_f32);
        }
    }
    u32x4 ahead[TN / 2];                               // the next rows' residual, if it has T's size
    auto fetch = [&](int i) {
        const long long m = (long long)m0 + i * 16 + row;
#pragma unroll
        for (int p = 0; p < TN / 2; ++p) {
            const int n = n0 + p * 32 + c8;
            if (m < M && n < NV) ahead[p] = *reinterpret_cast<const u32x4u*>((const T*)e.res + m * e.ldr + n);
        }
    };
    const bool res_t = e.res && !e.res_f32;
    if (res_t) fetch(0);
#pragma unroll
    for (int i = 0; i < TM; ++i) {
        const long long m = (long long)m0 + i * 16 + row;
        u32x4 now[TN / 2];
#pragma unroll
        for (int p = 0; p < TN / 2; ++p) now[p] = ahead[p];
        if (res_t && i + 1 < TM) fetch(i + 1);
#pragma unroll
        for (int p = 0; p < TN / 2; ++p) {
            const int n = n0 + p * 32;
            const bool in8 = m < M && n + c8 < NV;
            const bool ends = tail && n <= NV && NV < n + 32;          // the last columns are among these (wave-uniform)
            float v[2][4];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                acc_read<IN_PLACE>(acc[i][p * 2 + h], v[h]);
#pragma unroll
                for (int k = 0; k < 4; ++k) v[h][k] = (SCALED ? v[h][k] * factor : v[h][k]) + bias[p * 2 + h][k];
            }
            auto to_tail = [&](float* t) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int c = n + h * 16 + c4 - NV;
                    if (c >= 0 && c < 8) *reinterpret_cast<f32x4*>(t + (i * 16 + row) * 8 + c) = f32x4{v[h][0], v[h][1], v[h][2], v[h][3]};
                }
            };
            auto out = [&](void* p, long long ld, int f32) {
                if (f32) {
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        if (m < M && n + h * 16 + c4 < NV)
                            *reinterpret_cast<f32x4u*>((float*)p + m * ld + n + h * 16 + c4) = f32x4{v[h][0], v[h][1], v[h][2], v[h][3]};
                } else {
                    const u32x4 o = pair_out<T>(v);
                    if (in8) *reinterpret_cast<u32x4u*>((T*)p + m * ld + n + c8) = o;
                }
            };
            if (e.pre) {
                if (ends) to_tail(tail + TM * 16 * 8);
                out(e.pre, e.ldp, e.pre_f32);
            }
            act_values<ACT>(v);
            if (ends) to_tail(tail);
            if (res_t) {
                float r[2][4];
                pair_in<T>(now[p], r);
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int k = 0; k < 4; ++k) v[h][k] += r[h][k];
            } else if (e.res) {
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    if (m < M && n + h * 16 + c4 < NV) {
                        const f32x4 r = *reinterpret_cast<const f32x4u*>((const float*)e.res + m * e.ldr + n + h * 16 + c4);
#pragma unroll
                        for (int k = 0; k < 4; ++k) v[h][k] += r[k];
                    }
            }
            out(e.y, e.ldy, e.y_f32);
        }
    }
    if (!tail || n0 > NV || NV >= n0 + TN * 16) return;
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");                 // this wave's own writes
    const int c = lane & 7;
    if (c >= N - NV) return;
#pragma unroll 4
    for (int r = lane >> 3; r < TM * 16; r += 8) {
        const long long m = (long long)m0 + r;
        if (m < M) {
            float s = tail[r * 8 + c];
            if (e.res) s += load1<T>(e.res, m * e.ldr + NV + c, e.res_f32);
            if (e.pre) store1<T>(e.pre, m * e.ldp + NV + c, e.pre_f32, tail[TM * 16 * 8 + r * 8 + c]);
            store1<T>(e.y, m * e.ldy + NV + c, e.y_f32, s);
        }
    }
}

// ---------------------------------------------------------------- tile kernel
struct TileArgs {
    const void *A, *B;
    long long lda, ldb;     // elements
    int M, N, K;
    int tiles_m, tiles_n;
    int ksteps;             // units of 64 reduction indices per slice (blockIdx.y = slice)
    long long lo;           // bytes from A to its second part (AT or BT only), 0: it has one
    Epilogue e;
};

constexpr int kBK = 64;         // reduction indices per step: whole 128-byte lines of a row
constexpr uint32_t kBufferBytes = 0x80000000u;   // descriptor size: offsets built below stay under it

// One operand's tile of R rows (its own index) x 64 reduction indices in LDS, filled by W waves.
//   TR = false: contiguous along k in memory.  Image: R rows of 128 bytes, 16-byte chunk c of row r at
//     position c ^ (r & 7): the 16 lanes of a fragment read then hit 8 different bank groups.
//   TR = true: contiguous along R.  Image: 64 rows (k) of 2R bytes, 16-byte chunk c of row k at position
//     c ^ 2 f(k), f(k) = (k & 3) | (k >> 3 & 1) << 2 for R >= 128, (k >> 1 & 1) | (k >> 3 & 1) << 1 for R = 64: the
//     32 lanes that one transposing read serves at a time (4 k-rows x 2 groups of 8 k apart, 32 bytes each) then
//     cover all 64 banks once.
// Rows past the operand's end and reduction indices past K are read as zero through the buffer
// descriptor's range check, so no tile reads outside its matrix.
template <int R>
__device__ __forceinline__ int k_swizzle(int k) {
    static_assert(R == 64 || R % 128 == 0, "rows of half or whole bank widths");
    return R == 64 ? (k >> 1 & 1) | (k >> 3 & 1) << 1 : (k & 3) | (k >> 3 & 1) << 2;
}

template <int R, int W, bool TR>
struct Operand {
    static constexpr int NI = R / 8 / W;          // LDS-DMA instructions (1 KiB each) per wave and step
    static constexpr int BYTES = R * kBK * 2;
    uint32_t voff[NI];
    int kfirst, kstride;                          // reduction index of this lane's first chunk, and per instruction
    const char* base;                             // wave-uniform: this tile at the current step
    long long step;                               // bytes from one step to the next

    __device__ __forceinline__ void init(const void* p, long long ld, int row0, int extent, int kbeg, int lane, int w) {
        if constexpr (!TR) {
            const int r = lane >> 3, c = (lane & 7) ^ r;
            kfirst = c * 8;
            kstride = 0;
#pragma unroll
            for (int j = 0; j < NI; ++j) {
                const int row = (j * W + w) * 8 + r;
                voff[j] = row0 + row < extent ? (uint32_t)(row * (uint32_t)ld * 2u) + c * 16u : kBufferNowhere;
            }
            base = (const char*)p + ((long long)row0 * ld + kbeg) * 2;
            step = kBK * 2;
        } else {
            constexpr int CPR = R / 8, RPI = 64 / CPR;     // chunks per row, rows per instruction
            const int k = w * RPI + lane / CPR;
            kfirst = k;
            kstride = W * RPI;
#pragma unroll
            for (int j = 0; j < NI; ++j) {
                const int kj = k + j * W * RPI;
                const int c = (lane % CPR) ^ (k_swizzle<R>(kj) << 1);
                voff[j] = row0 + c * 8 < extent ? (uint32_t)(kj * (uint32_t)ld * 2u) + c * 16u : kBufferNowhere;
            }
            base = (const char*)p + ((long long)kbeg * ld + row0) * 2;
            step = kBK * ld * 2;
        }
    }
    // from here on only reduction indices below `left` of the step at `base` are valid (left <= 0: none; the loads
    // then write zeros and touch no memory)
    __device__ __forceinline__ void limit(int left) {
#pragma unroll
        for (int j = 0; j < NI; ++j) voff[j] = kfirst + j * kstride < left ? voff[j] : kBufferNowhere;
    }
    // instruction j of the step at `base`: source and destination
    __device__ __forceinline__ __amdgpu_buffer_rsrc_t source() const {
        return __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, (int)kBufferBytes, (int)kRawBufferWord3);
    }
    __device__ __forceinline__ static char* target(int j, char* buf, int w) { return buf + (j * W + w) * 1024; }
    __device__ __forceinline__ void issue(int j, char* buf, int w) const { lds_dma16_buf(source(), voff[j], 0, target(j, buf, w)); }
};

// fragment reads: 16 rows x 32 reduction indices; lane l holds row (l & 15), indices (l >> 4) * 8 ..
template <typename T, int R, bool TR>
struct Fragments {
    uint32_t at0;
    __device__ __forceinline__ void init(int row0, int lane) {
        if constexpr (!TR) {
            at0 = (row0 + (lane & 15)) * 128 + (((lane >> 4) ^ (lane & 7)) << 4);
        } else {
            const int g = lane >> 4, j = lane & 15;
            const int f = k_swizzle<R>(g * 8 + (j >> 2));
            at0 = (uint32_t)((g * 8 + (j >> 2)) * (R * 2) + (((row0 >> 4) ^ f) << 5) + ((j & 3) << 3));
        }
    }
    __device__ __forceinline__ v8<T> get(const char* buf, int i, int s) const {
        if constexpr (!TR) {
            return *reinterpret_cast<const v8<T>*>(buf + ((at0 ^ (s << 6)) + i * 2048));
        } else {
            const char* p = buf + ((at0 ^ (i << 5)) + s * (32 * R * 2));
            typedef __attribute__((address_space(3))) s16x4* lds_p;
            union { s16x4 h[2]; v8<T> v; } u;
            u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_p)p);
            u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_p)(p + 4 * R * 2));
            return u.v;
        }
    }
};

// Workgroups (of one wave per SIMD) that a CU's 160 KB of LDS hold.
constexpr int tile_occupancy(int b, int ahead) { return 163840 / ((2 * ahead + 1) * b * kBK * 2); }

// The product of a BM x BN tile over one slice of K, and its epilogue.  Bound by the matrix units where K is long and tiles
// are many: an operand element read from LDS into a wave's fragments feeds TM or TN matrix instructions, so the largest
// tile whose accumulators fit (256 x 256: half of a SIMD's registers, one wave per SIMD) needs the fewest LDS reads and
// the fewest bytes from L2, and with no second wave to fill gaps the instruction stream is laid by hand.  Smaller tiles
// give every CU work in smaller products, with two workgroups to a CU or a deeper ring against memory's latency.
// bf16: 8192^3 in 721 to 749 us, 1.47 to 1.52 PFLOP/s; 8192 x 16384 x 4096 with gelu_tanh 812 to 842 us, 1.31 to 1.35;
// 86528 x 128 x 256 with residual 22 us, 4.1 TB/s.  dX of 4096 x 1024 with 4096 terms: in two parts 77 us, in one 39.
template <typename T, int BM, int BN, int AHEAD, bool AT, bool BT>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(tile_occupancy(BM, AHEAD), tile_occupancy(BM, AHEAD))))
linear_tile_kernel(const TileArgs a) {
    constexpr int WM = 2, WN = 2, W = WM * WN;
    constexpr int WTM = BM / WM, WTN = BN / WN, TM = WTM / 16, TN = WTN / 16;
    typedef Operand<BM, W, AT> OpA;
    typedef Operand<BN, W, BT> OpB;
    constexpr int SLOTS = 2 * AHEAD + 1, RING = SLOTS * OpA::BYTES;
    constexpr bool IN_PLACE = tile_occupancy(BM, AHEAD) == 1;
    constexpr int PER = OpA::NI + OpB::NI;             // loads per wave and step
    static_assert(RING >= W * 2 * WTM * 8 * 4, "the epilogue's last columns fit into the ring");
    __shared__ __attribute__((aligned(1024))) char lds[RING];

    const int lane = threadIdx.x & 63;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = w % WM, wn = w / WM;
    // XCD-aware order: the blocks of one XCD (blockIdx % 8) take a contiguous run of tiles, and a run walks
    // groups of 8 tile rows column by column, so that the tiles an XCD works on at a time share rows and columns.
    int tile_m, tile_n;
    {
        const int T_ = a.tiles_m * a.tiles_n, q = T_ >> 3, r = T_ & 7;
        const int xcd = blockIdx.x & 7, loc = blockIdx.x >> 3;
        const int t = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + loc;
        const int per = 8 * a.tiles_n, g = t / per, in = t - g * per;
        const int gm = min(8, a.tiles_m - g * 8);
        tile_n = in / gm;
        tile_m = g * 8 + (in - tile_n * gm);
    }
    const int m0 = tile_m * BM, n0 = tile_n * BN;
    const int kbeg = (int)blockIdx.y * a.ksteps * kBK;
    const int kend = min(a.K, kbeg + a.ksteps * kBK);
    // steps of 64 reduction indices; A's two parts take one each
    const bool two = (AT || BT) && a.lo != 0;
    const int nt = kend > kbeg ? (kend - kbeg + kBK - 1) / kBK << (two ? 1 : 0) : 0;

    OpA opa;
    OpB opb;
    opa.init(a.A, a.lda, m0, a.M, kbeg, lane, w);
    opb.init(a.B, a.ldb, n0, a.N, kbeg, lane, w);
    Fragments<T, BM, AT> fa;
    Fragments<T, BN, BT> fb;
    fa.init(wm * WTM, lane);
    fb.init(wn * WTN, lane);

    f32x4 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    // A ring of 2 AHEAD + 1 operand tiles in LDS -- A(t), B(t), A(t+1), B(t+1), .. in turn -- and two sets of fragments
    // in registers.  The matrix instructions of half a step (32 reduction indices) run while the fragments of the next
    // half are read; in the middle of step t a barrier says that every wave has read its last fragments of A(t) and
    // B(t), whose places B(t + AHEAD) and A(t + 1 + AHEAD) take over the next two halves, one load (1 KiB) after every
    // eighth matrix instruction of the 256-wide tile: with one wave per SIMD a load that finds the memory pipe busy holds
    // up the matrix unit, and evenly spaced loads do that least (8192^3, before the loop was laid as it is: all of a step's
    // loads in one eighth of it 872 us, in a quarter 836, in a half 813).  The instruction stream is held in the order
    // written by scheduling fences, the reads and loads spread one by one between the matrix instructions: a wave issues an
    // instruction every four cycles and a matrix instruction occupies its unit for sixteen, so three others fit behind each
    // and no more.
    constexpr int PRODUCTS = TM * TN, READS = TM + TN;
    constexpr int TILE = OpA::BYTES;
    static_assert(OpA::BYTES == OpB::BYTES && PRODUCTS % OpA::NI == 0, "slots of one size, loads evenly spaced");
    constexpr int SPACE = PRODUCTS / OpA::NI, ISSUE_AT = SPACE > 2 ? SPACE - 2 : SPACE - 1;
    int left_a = kend - kbeg, left_b = left_a;
    auto limit_a = [&]() {
        if (left_a < kBK) opa.limit(left_a);
    };
    auto limit_b = [&]() {
        if (left_b < kBK) opb.limit(left_b);
    };
    bool lo_a = false, lo_b = false;                   // at A's second part; B's tile for it is the same again
    auto next_a = [&]() {
        const bool stay = two && !lo_a;
        opa.base += stay ? a.lo : two ? opa.step - a.lo : opa.step;
        left_a -= stay ? 0 : kBK;
        lo_a = stay;
        limit_a();
    };
    auto next_b = [&]() {
        const bool stay = two && !lo_b;
        opb.base += stay ? 0 : opb.step;
        left_b -= stay ? 0 : kBK;
        lo_b = stay;
        limit_b();
    };
    // the slot two on (one step), as byte offsets
    auto two_on = [](int slot) { return slot >= (SLOTS - 2) * TILE ? slot - (SLOTS - 2) * TILE : slot + 2 * TILE; };
    auto fetch = [&](v8<T> (&fr)[READS], int q, const char* ta, const char* tb, int s) {     // B's fragments, then A's
        fr[q] = q < TN ? fb.get(tb, q, s) : fa.get(ta, q - TN, s);
    };
    auto product = [&](const v8<T> (&fr)[READS], int e) {
        const int i = e / TN, j = e % TN;
        if constexpr (IN_PLACE) mfma_in_place(fr[j], fr[TN + i], acc[i][j]);
        else acc[i][j] = mfma(fr[j], fr[TN + i], acc[i][j]);
    };
    // the same and load q of an operand
    auto product_load = [&](const v8<T> (&fr)[READS], int e, const auto& op, int q, char* buf) {
        const int i = e / TN, j = e % TN;
        if constexpr (IN_PLACE) {
            mfma_in_place_load(fr[j], fr[TN + i], acc[i][j], op.source(), op.voff[q], op.target(q, buf, w));
        } else {
            product(fr, e);
            op.issue(q, buf, w);
        }
    };
#define YA_FENCE() __builtin_amdgcn_sched_barrier(0)
    v8<T> f0[READS], f1[READS];
    limit_a();
    limit_b();
#pragma unroll
    for (int t = 0; t < AHEAD; ++t) {
#pragma unroll
        for (int q = 0; q < OpA::NI; ++q) opa.issue(q, lds + t * 2 * TILE, w);
#pragma unroll
        for (int q = 0; q < OpB::NI; ++q) opb.issue(q, lds + t * 2 * TILE + TILE, w);
        next_a();
        next_b();
    }
    wait_vmcnt<(AHEAD - 1) * PER>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
#pragma unroll
    for (int q = 0; q < READS; ++q) fetch(f0, q, lds, lds + TILE, 0);
    int sa = 0, sb = TILE, fill = (SLOTS - 1) * TILE;  // slots of A(t), B(t), A(t + AHEAD)
    for (int t = 0; t < nt; ++t) {
        // first half: the second half's fragments in the first three quarters of it
#pragma unroll
        for (int e = 0; e < PRODUCTS; ++e) {
            if (e % SPACE == ISSUE_AT) product_load(f0, e, opa, e / SPACE, lds + fill);
            else product(f0, e);
#pragma unroll
            for (int q = 0; q < READS; ++q)
                if (q * PRODUCTS / (READS * 2) == e) fetch(f1, q, lds + sa, lds + sb, 1);
            YA_FENCE();
        }
        next_a();
        // this wave's reads of A(t) and B(t) have returned and its loads of A(t+1) and B(t+1) landed (those of
        // A(t+2 .. t + AHEAD) and B(t+2 .. t + AHEAD - 1) may be on their way); then everybody's
        wait_vmcnt<(AHEAD - 1) * OpA::NI + (AHEAD - 2) * OpB::NI>();
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        YA_FENCE();
        // second half: the next step's first fragments
        const int na = two_on(sa), nb = two_on(sb);
#pragma unroll
        for (int e = 0; e < PRODUCTS; ++e) {
            if (e % SPACE == ISSUE_AT) product_load(f1, e, opb, e / SPACE, lds + sa);
            else product(f1, e);
#pragma unroll
            for (int q = 0; q < READS; ++q)
                if (q * PRODUCTS / READS == e) fetch(f0, q, lds + na, lds + nb, 0);
            YA_FENCE();
        }
        next_b();
        fill = sb;
        sa = na;
        sb = nb;
    }
#undef YA_FENCE
    if constexpr (IN_PLACE) mfma_drain();
    wait_vmcnt<0>();                                   // no load may land in the epilogue's LDS

    const int mw = m0 + wm * WTM, nw = n0 + wn * WTN;
    Epilogue e = a.e;
    int nv = a.N & ~7;
    if (e.part) {                                      // a K slice: raw sums, rows of whole eights
        e.y = e.part + blockIdx.y * e.slice_stride;
        e.ldy = e.ld_part;
        e.y_f32 = 1;
        nv = (a.N + 7) & ~7;
    }
    float* tail = nullptr;
    if (nv < a.N && n0 + BN > nv) {
        __syncthreads();                               // every wave is done with the ring
        tail = reinterpret_cast<float*>(lds) + w * (2 * WTM * 8);
    }
#define YA_FINISH(ACT) finish_direct<T, ACT, IN_PLACE, AT || BT>(e, acc, mw, nw, a.M, a.N, nv, lane, tail)
    if constexpr (AT || BT) {
        YA_FINISH(YOLO_AMD_ACT_NONE);
    } else {
        switch (e.act) {
            case YOLO_AMD_ACT_LEAKY: YA_FINISH(YOLO_AMD_ACT_LEAKY); break;
            case YOLO_AMD_ACT_RELU: YA_FINISH(YOLO_AMD_ACT_RELU); break;
            case YOLO_AMD_ACT_GELU: YA_FINISH(YOLO_AMD_ACT_GELU); break;
            case YOLO_AMD_ACT_GELU_TANH: YA_FINISH(YOLO_AMD_ACT_GELU_TANH); break;
            case YOLO_AMD_ACT_SILU: YA_FINISH(YOLO_AMD_ACT_SILU); break;
            default: YA_FINISH(YOLO_AMD_ACT_NONE); break;
        }
    }
#undef YA_FINISH
}

// Adds the K slices in ascending order and finishes, eight columns per thread.  A read of the slices at 4 TB/s (they were
// just written) behind a launch of 3.4 us: what plan_product charges a split.
template <typename T>
__global__ void __launch_bounds__(256)
linear_finish_kernel(const Epilogue e, const float* part, int slices, int M, int N) {
    const int n = (blockIdx.x * 64 + (threadIdx.x & 63)) * 8;
    const int step = gridDim.y * 4;
    if (n >= N) return;
    for (int m = blockIdx.y * 4 + (threadIdx.x >> 6); m < M; m += step) {
        const float* p = part + (long long)m * e.ld_part + n;
        float v[8];
        load8<T>(p, 0, 1, v);
#pragma unroll 4
        for (int s = 1; s < slices; ++s) {
            float u[8];
            load8<T>(p, s * e.slice_stride, 1, u);
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] += u[k];
        }
        if (e.unscale) {
            const float factor = *e.unscale;
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] *= factor;
        }
        finish8<T>(e, m, n, N, v);
    }
}

// ---------------------------------------------------------------- few rows
// M <= 16 * MT rows of x: the product is a read of W.  A workgroup owns 16 * NT rows of W (columns of Y) and
// its eight waves take 64 reduction indices each in turn, straight from memory into matrix-instruction fragments;
// the eight partial sums meet in LDS in a fixed order.  Every workgroup reads all of x (from L2): more rows of W per
// workgroup save that, fewer fill the chip (one row, N 16384, K 4096: NT 1 25.5 us, 5.3 TB/s, NT 2 30.2; sixteen rows:
// NT 1 40.6, NT 2 36.7, and the 64-wide tile 33.4).  Where even 16 columns each leave CUs without a workgroup, K is cut into slices (blockIdx.y).
// U steps' loads are issued before the first product: what bounds this kernel is how much of W is on its way.
template <typename T, int MT, int NT, int U>
__global__ void __launch_bounds__(512)
linear_rows_kernel(const TileArgs a) {
    __shared__ __attribute__((aligned(16))) f32x4 red[8][MT][NT][64];
    const int lane = threadIdx.x & 63;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n0 = blockIdx.x * (16 * NT);
    const int kl = (lane >> 4) * 8;
    const T* xp[MT];
    const T* wp[NT];
#pragma unroll
    for (int i = 0; i < MT; ++i) xp[i] = (const T*)a.A + (long long)min(i * 16 + (lane & 15), a.M - 1) * a.lda;
#pragma unroll
    for (int j = 0; j < NT; ++j) wp[j] = (const T*)a.B + (long long)min(n0 + j * 16 + (lane & 15), a.N - 1) * a.ldb;
    f32x4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int k1 = min(a.K, ((int)blockIdx.y + 1) * a.ksteps * kBK);
    for (int k = (int)blockIdx.y * a.ksteps * kBK + w * 64; k < k1; k += 512 * U) {
        v8<T> xv[U][2][MT], wv[U][2][NT];
        bool in[U][2];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                // past the slice (whole chunks: K is a multiple of 8): the row's start, taken as zeros below
                const int at = k + u * 512 + s * 32 + kl;
                in[u][s] = at < k1;
                const int from = in[u][s] ? at : 0;
#pragma unroll
                for (int j = 0; j < NT; ++j) wv[u][s][j] = *reinterpret_cast<const v8<T>*>(wp[j] + from);
#pragma unroll
                for (int i = 0; i < MT; ++i) xv[u][s][i] = *reinterpret_cast<const v8<T>*>(xp[i] + from);
            }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                if (!in[u][s]) {
#pragma unroll
                    for (int j = 0; j < NT; ++j) wv[u][s][j] = v8<T>{};
#pragma unroll
                    for (int i = 0; i < MT; ++i) xv[u][s][i] = v8<T>{};
                }
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int j = 0; j < NT; ++j) acc[i][j] = mfma(wv[u][s][j], xv[u][s][i], acc[i][j]);
            }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) red[w][i][j][lane] = acc[i][j];
    __syncthreads();
    for (int it = threadIdx.x; it < MT * 16 * NT * 2; it += 512) {
        const int mr = it / (NT * 2), n8 = it % (NT * 2);
        const int n = n0 + n8 * 8;
        if (mr < a.M && n < a.N) {
            const int l0 = (n8 & 1) * 32 + (mr & 15);
            f32x4 lo = f32x4{0.f, 0.f, 0.f, 0.f}, hi = lo;
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                lo += red[q][mr >> 4][n8 >> 1][l0];
                hi += red[q][mr >> 4][n8 >> 1][l0 + 16];
            }
            float v[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) { v[i] = lo[i]; v[4 + i] = hi[i]; }
            if (a.e.part) store8<T>(a.e.part, blockIdx.y * a.e.slice_stride + mr * a.e.ld_part + n, 1, v);
            else finish8<T>(a.e, mr, n, a.N, v);
        }
    }
}

// ---------------------------------------------------------------- operand copies
// Rows of C elements at any stride and alignment -> rows of C rounded up to 8, zero filled: what the kernels
// above need (16-byte chunks that never straddle a row's end).  One thread per chunk, both operands in one launch: a
// launch's own time at the sizes that come without alignment (333 + 755 rows of 1021: 4.8 us for 4.4 MB).
struct PackArgs {
    const void* src[2];
    void* dst[2];
    long long ld[2], chunks[2];
    int cols[2], c8[2];
};
template <typename T>
__global__ void __launch_bounds__(256)
linear_pack_kernel(const PackArgs a) {
    const int w = blockIdx.y;
    const T* src = (const T*)a.src[w];
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < a.chunks[w]; i += (long long)gridDim.x * 256) {
        const long long r = i / a.c8[w];
        const int c = (int)(i - r * a.c8[w]) * 8;
        v8<T> v;
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = c + k < a.cols[w] ? src[r * a.ld[w] + c + k] : (T)0.f;
        *reinterpret_cast<v8<T>*>((T*)a.dst[w] + i * 8) = v;
    }
}

// ---------------------------------------------------------------- backward: dP and the bias gradient
struct DpreArgs {
    const void *dy, *pre;
    long long lddy, ldpre;
    int dy_f32, pre_f32, act;
    void* dp;               // [M][ldp], zero filled past N; null: only the column sums are wanted
    void* dp_lo;            // dP - dp, the same way; null: dp holds dP as it is
    long long ldp;
    const float* scale;     // null: 1; else what dP is multiplied by where it is stored
    float* peaks;           // [row block][column block] largest finite |dP|, or null
    float* part;            // [row block][N] column sums, or null
    int M, N, rows;         // rows per block
};

// Thread = eight columns of a run of rows (the last ones by element); column sums in fp32 over that run, added over the
// runs by linear_dbias_kernel.  4096 x 4096 with GELU, fp32 pre-activation, two parts: 36 us, 168 MB, 4.7 TB/s.  One row at a
// time: more rows in flight cost registers that hide more of memory's latency as further waves (the same with a 16-bit
// pre-activation and one part, 100 MB: 1 row 20.8 us, 2 rows 23.9, 4 rows 28.2).
// fp16 in two parts wants the largest value first: this kernel runs twice, dY and P are read twice (1531 x 1030: 8.1 + 8.2 us
// and 1.7 between them).  Keeping fp32 dP for the second run instead would move as much.
template <typename T>
__global__ void __launch_bounds__(256)
linear_dpre_kernel(const DpreArgs a) {
    constexpr int CL = 32, RL = 8;                     // column lanes x rows
    const int lane_c = threadIdx.x % CL, lane_r = threadIdx.x / CL;
    const int n = (blockIdx.x * CL + lane_c) * 8;
    __shared__ float red[RL][CL * 8 + 1];
    const long long r0 = (long long)blockIdx.y * a.rows;
    const long long r1 = min((long long)a.M, r0 + a.rows);
    const bool whole = n + 8 <= a.N;
    float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    float peak = 0.f;
    const float scale = a.scale ? *a.scale : 1.f;
    auto fetch = [&](const void* p, long long at, int f32, float (&v)[8]) {
        if (whole) {
            load8<T>(p, at, f32, v);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = n + i < a.N ? load1<T>(p, at + i, f32) : 0.f;
        }
    };
    if (n < a.N) {
        for (long long m = r0 + lane_r; m < r1; m += RL) {
            float d[8], p[8];
            fetch(a.dy, m * a.lddy + n, a.dy_f32, d);
            if (a.pre) {
                fetch(a.pre, m * a.ldpre + n, a.pre_f32, p);
                times_slopes<8>(d, p, a.act);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) sum[i] += d[i];
            if (a.peaks) {
#pragma unroll
                for (int i = 0; i < 8; ++i) peak = fabsf(d[i]) < __builtin_inff() ? fmaxf(peak, fabsf(d[i])) : peak;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) d[i] *= scale;
            if (a.dp) store8<T>(a.dp, m * a.ldp + n, 0, d);          // padded rows: zeros behind the last column
            if (a.dp_lo) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float r = d[i] - (float)(T)d[i];           // exact; no part of a value past the type's range
                    d[i] = fabsf(r) < __builtin_inff() ? r : 0.f;
                }
                store8<T>(a.dp_lo, m * a.ldp + n, 0, d);
            }
        }
    }
    if (a.peaks) {
        red[0][threadIdx.x] = peak;
        __syncthreads();
        if (threadIdx.x < 64) {
            peak = fmaxf(fmaxf(red[0][threadIdx.x], red[0][threadIdx.x + 64]), fmaxf(red[0][threadIdx.x + 128], red[0][threadIdx.x + 192]));
#pragma unroll
            for (int i = 32; i; i >>= 1) peak = fmaxf(peak, __shfl_xor(peak, i));
            if (threadIdx.x == 0) a.peaks[(long long)blockIdx.y * gridDim.x + blockIdx.x] = peak;
        }
        __syncthreads();
    }
    if (!a.part) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) red[lane_r][lane_c * 8 + i] = sum[i];
    __syncthreads();
    const int c = blockIdx.x * (CL * 8) + threadIdx.x;
    if (c < a.N) {
        float s = 0.f;
#pragma unroll
        for (int r = 0; r < RL; ++r) s += red[r][threadIdx.x];
        a.part[(long long)blockIdx.y * a.N + c] = s;
    }
}

// scale[0]: the power of two that brings the largest of the peaks to 2^14 .. 2^15 (1 if there is none); scale[1]: its inverse.
// Both are normal numbers: values below 2^-112, which come out lower than that, are zeros in any result of type fp16.
__global__ void __launch_bounds__(1024)
linear_scale_kernel(const float* peaks, int n, float* scale) {
    __shared__ float red[16];
    float peak = 0.f;
    for (int i = threadIdx.x; i < n; i += 1024) peak = fmaxf(peak, peaks[i]);
#pragma unroll
    for (int i = 32; i; i >>= 1) peak = fmaxf(peak, __shfl_xor(peak, i));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = peak;
    __syncthreads();
    if (threadIdx.x == 0) {
#pragma unroll
        for (int i = 1; i < 16; ++i) peak = fmaxf(peak, red[i]);
        int e = 0;
        if (peak > 0.f) {
            frexpf(peak, &e);                          // peak = 0.5 .. 1 times 2^e
            e = min(15 - e, 126);
        }
        scale[0] = ldexpf(1.f, e);
        scale[1] = ldexpf(1.f, -e);
    }
}

// 64 columns per workgroup; wave w adds runs w, w + 16, .. in ascending order, the waves are added in order.  Latency of
// one launch (128 runs of 4096 columns: 4 to 5 us).
template <typename T>
__global__ void __launch_bounds__(1024)
linear_dbias_kernel(const float* part, int blocks, int N, void* db, int db_f32) {
    __shared__ float red[16][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int n = blockIdx.x * 64 + lane;
    float s = 0.f;
    if (n < N) {
#pragma unroll 8
        for (int b = w; b < blocks; b += 16) s += part[(long long)b * N + n];
    }
    red[w][lane] = s;
    __syncthreads();
    if (w == 0 && n < N) {
#pragma unroll
        for (int i = 1; i < 16; ++i) s += red[i][lane];
        store1<T>(db, n, db_f32, s);
    }
}

// ---------------------------------------------------------------- host side
struct Matrix {
    const void* p;
    long long ld;
    long long rows;
    int cols;
};

// Tiles address their rows with 32-bit byte offsets: 256 rows of this many elements.
constexpr long long kMaxLd = (1ll << 22) - 1, kMaxRows = 1ll << 30;
// A launch holds fewer than 2^32 threads: so many workgroups of 256.
constexpr long long kMaxTiles = (1ll << 24) - 1;

// can be read in place: whole 16-byte chunks, no row's last one reaching into the next
static bool packed_ok(const Matrix& m) {
    return ((uintptr_t)m.p & 15) == 0 && m.cols % 8 == 0 && ((m.ld % 8 == 0 && m.ld <= kMaxLd) || m.rows <= 1);
}
static size_t packed_bytes(const Matrix& m) {
    return packed_ok(m) ? 0 : align_up((size_t)m.rows * align_up(m.cols, 8) * 2, 256);
}

// Which kernel a product D[M][N] over K runs on.
struct TilePlan {
    int kernel, bm, bn, slices, ksteps, ahead;
};

// The tile kernels, with what a full round of workgroups takes (microseconds: start, prologue and epilogue; then each
// step of 64 reduction indices), and a round that leaves at most one workgroup to a CU.  Fitted to bf16 products y in
// captured graphs, every kernel and split on 70 sizes from 33 x 64 x 64 to 8192^3: the choice they make is 1.0 % slower
// than the fastest of each size (geometric mean; 22 % at the worst).  On 30 other sizes, geometric mean and worst: y in bf16
// 0.9 and 17 %, in fp16 0.7 and 10; dX 0.2 and 2, 0.3 and 3; dW 0.5 and 6, 0.5 and 7.  The 256-wide tile moves the fewest bytes per
// product but wants a tile for every CU; 128 four steps ahead hides memory's latency where a CU has one workgroup
// (4096 x 1024 x 4096: 38.8 against 46.1 us), two ahead lets two workgroups do that for each other (2048 x 4096 x 4096:
// 69.5 against 76.6); 64 is for what has fewer than 256 tiles of 128 (1024^3: 7.4 against 12.8).
struct TileConfig {
    int b, ahead;
    double start, step, start_1, step_1;
};
static const TileConfig kTileConfigs[] = {
    {256, 2, 10.9, 1.44, 10.5, 1.04},
    {128, 2, 4.0, 1.02, 4.4, 0.59},
    {128, 4, 4.1, 0.54, 4.9, 0.52},
    {64, 4, 3.2, 0.436, 3.1, 0.274},
};

// `parts` of the first operand: each step of 64 reduction indices is so many.  kernel 0: more tiles than a launch holds.
static TilePlan plan_product(long long M, int N, long long K, bool kc_operands, int act, int parts = 1) {
    TilePlan p{};
    const long long steps = std::max<long long>(1, (K + kBK - 1) / kBK);
    // An activation's instructions lengthen an epilogue that nothing overlaps (256: 12 to 13 us a round for erf, 3 to 5 for the
    // two with an exponential and a reciprocal) more than one that another workgroup's products run beside (128: 2.3 and 1).
    const double slow = act == YOLO_AMD_ACT_GELU ? 1.0 : act == YOLO_AMD_ACT_GELU_TANH || act == YOLO_AMD_ACT_SILU ? 0.4 : 0.0;
    double best = 0;
    // Few rows: one workgroup streams 22.5 bytes a nanosecond, many 6000 (80 of them half as fast); x from L2 costs two
    // thirds of a byte of W.  K is cut only where sixteen columns to a workgroup leave CUs without one.
    for (int nt = 1; kc_operands && M <= 32 && nt <= 4; nt *= 2) {
        const long long wgs = (N + 16 * nt - 1) / (16 * nt);
        for (int s = 1; s <= 16 && s * 8 <= steps + 7; s *= 2) {
            const long long per = (steps + s - 1) / s;
            if ((steps + per - 1) / per != s) continue;
            if (s > 1 && (nt > 1 || wgs * s > 512)) break;
            const double w = (double)wgs * s, rate = std::min(22.5 * w, 6000.0 * w / (w + 80.0));
            double t = 1.8 + 2.0 * K * (N + 0.65 * wgs * M) * 1e-3 / rate;
            if (s > 1) t += 3.4 + 0.08 * s + (double)s * M * N * 2e-6;
            if (p.kernel == 0 || t < best) {
                best = t;
                p.kernel = YOLO_AMD_LINEAR_ROWS;
                p.bm = M <= 16 ? 16 : 32;
                p.bn = 16 * nt;
                p.ahead = 0;
                p.slices = s;
                p.ksteps = (int)per;
            }
        }
    }
    for (const TileConfig& c : kTileConfigs) {
        const long long tiles = ((M + c.b - 1) / c.b) * ((N + c.b - 1) / c.b);
        if (tiles > kMaxTiles) continue;
        const int slots = 256 * tile_occupancy(c.b, c.ahead);
        for (int s = 1; s <= 64 && s <= steps; ++s) {
            const long long per = (steps + s - 1) / s, wgs = tiles * s, rest = wgs % slots;
            if ((steps + per - 1) / per != s) continue;
            if (s > 1 && wgs > slots) break;           // a split only fills a round that is not full
            double t = (double)(wgs / slots) * (c.start + parts * per * c.step);
            if (s == 1) t += (double)((wgs + slots - 1) / slots) * slow * (c.b == 256 ? 12.0 : c.b == 128 ? 2.5 : 0.7);
            if (rest > 0) t += rest <= 256 ? c.start_1 + parts * per * c.step_1 : c.start + parts * per * c.step;
            t = std::max(t, 2.0 + 2.0 * ((double)parts * M * K + (double)N * K + (double)M * N) * 2e-7);   // at 5 TB/s
            if (s > 1) t += 3.4 + 0.08 * s + (double)s * M * N * 2e-6;     // one more launch; partial sums out and in at 4 TB/s
            if (p.kernel == 0 || t < best) {
                best = t;
                p.kernel = YOLO_AMD_LINEAR_TILE;
                p.bm = p.bn = c.b;
                p.ahead = c.ahead;
                p.slices = s;
                p.ksteps = (int)per;
            }
        }
    }
    return p;
}

static size_t partial_bytes(const TilePlan& p, long long M, int N) {
    return p.slices > 1 ? align_up((size_t)p.slices * M * align_up(N, 8) * 4, 256) : 0;
}

// Scratch of a call, handed out front to back.
struct Scratch {
    char* p;
    void* take(size_t bytes) {
        void* r = p;
        p += bytes;
        return r;
    }
};

// Copies of the operands that want one (bytes > 0), in one launch.
template <typename T>
static void launch_pack(Matrix (&m)[2], const size_t (&bytes)[2], Scratch& sc, hipStream_t s) {
    PackArgs a{};
    int n = 0;
    for (int i = 0; i < 2; ++i) {
        if (bytes[i] == 0) continue;
        const int c8 = (int)(align_up(m[i].cols, 8) / 8);
        a.src[n] = m[i].p;
        a.dst[n] = sc.take(bytes[i]);
        a.ld[n] = m[i].ld;
        a.cols[n] = m[i].cols;
        a.c8[n] = c8;
        a.chunks[n] = m[i].rows * c8;
        m[i] = Matrix{a.dst[n], c8 * 8, m[i].rows, c8 * 8};
        ++n;
    }
    if (n == 0) return;
    const long long most = std::max(a.chunks[0], a.chunks[1]);
    hipLaunchKernelGGL((linear_pack_kernel<T>), dim3((unsigned)std::min<long long>((most + 255) / 256, 1 << 14), n), dim3(256), 0, s, a);
}

template <typename T, bool AT, bool BT>
static int launch_product(const TilePlan& p, TileArgs a, void* partial, hipStream_t s) {
    a.ksteps = p.ksteps;
    const Epilogue e = a.e;
    if (p.slices > 1) {
        a.e = Epilogue{};
        a.e.part = (float*)partial;
        a.e.ld_part = (long long)align_up(a.N, 8);
        a.e.slice_stride = a.e.ld_part * a.M;
    }
    const int kernel = p.kernel == YOLO_AMD_LINEAR_ROWS ? 0 : p.bm * 10 + p.ahead;
    if (kernel == 0) {
        if constexpr (!AT && !BT) {
            const dim3 grid((a.N + p.bn - 1) / p.bn, p.slices);
            const bool deep = p.ksteps > 16;           // four steps of 512 in flight
#define YA_ROWS(MT, NT)                                                                                              \
    do {                                                                                                             \
        if (deep) hipLaunchKernelGGL((linear_rows_kernel<T, MT, NT, 4>), grid, dim3(512), 0, s, a);                  \
        else hipLaunchKernelGGL((linear_rows_kernel<T, MT, NT, 2>), grid, dim3(512), 0, s, a);                       \
    } while (0)
            if (p.bm == 16 && p.bn == 16) YA_ROWS(1, 1);
            else if (p.bm == 16 && p.bn == 32) YA_ROWS(1, 2);
            else if (p.bm == 16) hipLaunchKernelGGL((linear_rows_kernel<T, 1, 4, 2>), grid, dim3(512), 0, s, a);
            else if (p.bn == 16) YA_ROWS(2, 1);
            else if (p.bn == 32) YA_ROWS(2, 2);
            else hipLaunchKernelGGL((linear_rows_kernel<T, 2, 4, 2>), grid, dim3(512), 0, s, a);
#undef YA_ROWS
        }
    }
    a.tiles_m = (a.M + p.bm - 1) / p.bm;
    a.tiles_n = (a.N + p.bn - 1) / p.bn;
    const dim3 grid((unsigned)((long long)a.tiles_m * a.tiles_n), (unsigned)p.slices);
    if (kernel == 2562) hipLaunchKernelGGL((linear_tile_kernel<T, 256, 256, 2, AT, BT>), grid, dim3(256), 0, s, a);
    else if (kernel == 1282) hipLaunchKernelGGL((linear_tile_kernel<T, 128, 128, 2, AT, BT>), grid, dim3(256), 0, s, a);
    else if (kernel == 1284) hipLaunchKernelGGL((linear_tile_kernel<T, 128, 128, 4, AT, BT>), grid, dim3(256), 0, s, a);
    else if (kernel == 644) hipLaunchKernelGGL((linear_tile_kernel<T, 64, 64, 4, AT, BT>), grid, dim3(256), 0, s, a);
    if (p.slices > 1) {
        Epilogue f = e;
        f.ld_part = a.e.ld_part;
        f.slice_stride = a.e.slice_stride;
        const dim3 fgrid((a.N + 511) / 512, (unsigned)std::min<long long>((a.M + 3) / 4, 4096));
        hipLaunchKernelGGL((linear_finish_kernel<T>), fgrid, dim3(256), 0, s, f, (const float*)partial, p.slices, a.M, a.N);
    }
    YA_CHECK_HIP(hipGetLastError());
    return YA_OK;
}


static int check_common(const char* what, int64_t m, int64_t n, int64_t k, int type, int act) {
    YA_REQUIRE(m >= 0 && n >= 0 && k >= 0 && m <= kMaxRows && n <= kMaxLd && k <= kMaxLd,
               "%s: m=%lld n=%lld k=%lld (m up to %lld, n and k up to %lld)", what, (long long)m, (long long)n, (long long)k,
               kMaxRows, kMaxLd);
    YA_REQUIRE(type == YOLO_AMD_TYPE_BF16 || type == YOLO_AMD_TYPE_F16, "%s: type %d (bf16 or fp16)", what, type);
    YA_REQUIRE(act >= YOLO_AMD_ACT_NONE && act <= YOLO_AMD_ACT_SILU, "%s: activation %d", what, act);
    return YA_OK;
}

static int check_matrix(const char* what, const char* name, const void* p, long long ld, long long rows, int cols, int esize) {
    if (rows == 0 || cols == 0) return YA_OK;
    YA_REQUIRE(p, "%s: %s is null", what, name);
    YA_REQUIRE(((uintptr_t)p & (esize - 1)) == 0, "%s: %s is not aligned to its elements", what, name);
    YA_REQUIRE(rows <= 1 || ld >= cols, "%s: %s has row stride %lld for %d columns", what, name, ld, cols);
    return YA_OK;
}
static int check_forward(const yolo_amd_linear_desc* d) {
    YA_REQUIRE(d, "linear_forward: null descriptor");
    YA_TRY(check_common("linear_forward", d->m, d->n, d->k, d->type, d->activation));
    YA_TRY(check_matrix("linear_forward", "x", d->x, d->ldx, d->m, (int)d->k, 2));
    YA_TRY(check_matrix("linear_forward", "weight", d->weight, d->ldw, d->n, (int)d->k, 2));
    YA_TRY(check_matrix("linear_forward", "y", d->y, d->ldy, d->m, (int)d->n, d->y_f32 ? 4 : 2));
    if (d->residual) YA_TRY(check_matrix("linear_forward", "residual", d->residual, d->ldr, d->m, (int)d->n, d->residual_f32 ? 4 : 2));
    if (d->bias) YA_TRY(check_matrix("linear_forward", "bias", d->bias, d->n, 1, (int)d->n, d->bias_f32 ? 4 : 2));
    if (d->pre) YA_TRY(check_matrix("linear_forward", "pre", d->pre, d->n, d->m, (int)d->n, d->pre_f32 ? 4 : 2));
    return YA_OK;
}

struct ForwardPlan {
    TilePlan tile;
    Matrix x, w;
    size_t x_bytes, w_bytes, part_bytes;
    size_t bytes() const { return x_bytes + w_bytes + part_bytes; }
};

static ForwardPlan plan_forward(const yolo_amd_linear_desc* d) {
    ForwardPlan f{};
    f.x = Matrix{d->x, d->ldx, d->m, (int)d->k};
    f.w = Matrix{d->weight, d->ldw, d->n, (int)d->k};
    if (d->m == 0 || d->n == 0) return f;
    f.tile = plan_product(d->m, (int)d->n, d->k, true, d->activation);
    f.x_bytes = packed_bytes(f.x);
    f.w_bytes = packed_bytes(f.w);
    f.part_bytes = partial_bytes(f.tile, d->m, (int)d->n);
    return f;
}

static int check_plan(const char* what, const TilePlan& p, long long m, long long n) {
    YA_REQUIRE(p.kernel, "%s: a product of %lld x %lld takes more tiles than a launch holds (%lld of 256 x 256)", what, m, n, kMaxTiles);
    return YA_OK;
}
static int check_plan(const yolo_amd_linear_desc* d, const ForwardPlan& f) {
    return d->m == 0 || d->n == 0 ? YA_OK : check_plan("linear_forward", f.tile, d->m, d->n);
}

static int check_workspace(const char* what, const void* ws, size_t have, size_t need) {
    if (need == 0) return YA_OK;
    YA_REQUIRE(ws && ((uintptr_t)ws & 255) == 0, "%s: the workspace is null or not 256-byte aligned", what);
    if (have < need) {
        set_error("%s: workspace of %zu bytes, %zu needed", what, have, need);
        return YA_ERR_WORKSPACE;
    }
    return YA_OK;
}

template <typename T>
static int forward(const yolo_amd_linear_desc* d, const ForwardPlan& f, hipStream_t s) {
    Scratch sc{(char*)d->workspace};
    Matrix in[2] = {f.x, f.w};
    launch_pack<T>(in, {f.x_bytes, f.w_bytes}, sc, s);
    const Matrix &x = in[0], &w = in[1];
    TileArgs a{};
    a.A = x.p; a.lda = x.ld;
    a.B = w.p; a.ldb = w.ld;
    a.M = (int)d->m; a.N = (int)d->n; a.K = std::min(x.cols, w.cols);
    Epilogue& e = a.e;
    e.bias = d->bias; e.res = d->residual; e.y = d->y; e.pre = d->pre;
    e.ldr = d->ldr; e.ldy = d->ldy; e.ldp = d->n;
    e.bias_f32 = d->bias_f32; e.res_f32 = d->residual_f32; e.y_f32 = d->y_f32; e.pre_f32 = d->pre_f32;
    e.act = d->activation;
    return launch_product<T, false, false>(f.tile, a, sc.take(f.part_bytes), s);
}

// ---- backward
static int check_backward(const yolo_amd_linear_backward_desc* d) {
    const char* me = "linear_backward";
    YA_REQUIRE(d, "%s: null descriptor", me);
    YA_TRY(check_common(me, d->m, d->n, d->k, d->type, d->activation));
    YA_TRY(check_matrix(me, "dy", d->dy, d->lddy, d->m, (int)d->n, d->dy_f32 ? 4 : 2));
    if (d->dweight) YA_TRY(check_matrix(me, "x", d->x, d->ldx, d->m, (int)d->k, 2));
    if (d->dx) YA_TRY(check_matrix(me, "weight", d->weight, d->ldw, d->n, (int)d->k, 2));
    if (d->activation != YOLO_AMD_ACT_NONE) YA_TRY(check_matrix(me, "pre", d->pre, d->n, d->m, (int)d->n, d->pre_f32 ? 4 : 2));
    if (d->dx) YA_TRY(check_matrix(me, "dx", d->dx, d->k, d->m, (int)d->k, 2));
    if (d->dweight) YA_TRY(check_matrix(me, "dweight", d->dweight, d->k, d->n, (int)d->k, 2));
    if (d->dbias) YA_TRY(check_matrix(me, "dbias", d->dbias, d->n, 1, (int)d->n, d->dbias_f32 ? 4 : 2));
    return YA_OK;
}

struct LinearBackwardPlan {
    TilePlan dx, dw;
    Matrix x, w;
    bool own_dp;            // dP is a tensor of its own (else dY is dP)
    int parts;              // of dP
    bool scaled;            // by a power of two
    int blocks, rows;       // row blocks of the column sums
    size_t dp_bytes, db_bytes, scale_bytes, x_bytes, w_bytes, part_bytes;
    size_t bytes() const { return dp_bytes + db_bytes + scale_bytes + x_bytes + w_bytes + part_bytes; }
};

static LinearBackwardPlan plan_backward(const yolo_amd_linear_backward_desc* d) {
    LinearBackwardPlan b{};
    const bool empty = d->m == 0 || d->n == 0;
    const Matrix dy{d->dy, d->lddy, d->m, (int)d->n};
    b.x = Matrix{d->x, d->ldx, d->m, (int)d->k};
    b.w = Matrix{d->weight, d->ldw, d->n, (int)d->k};
    const bool products = (d->dx || d->dweight) && d->k > 0 && !empty;
    b.own_dp = products && (d->activation != YOLO_AMD_ACT_NONE || d->dy_f32 || !packed_ok(dy));
    // dY in the operands' type times 1 or 0 is a value of that type
    b.parts = !d->dy_f32 && (d->activation == YOLO_AMD_ACT_NONE || d->activation == YOLO_AMD_ACT_RELU) ? 1 : 2;
    if (b.own_dp) b.dp_bytes = b.parts * align_up((size_t)d->m * align_up(d->n, 8) * 2, 256);
    // enough blocks of rows to fill the chip, at least 16 rows each
    const long long cols = std::max<long long>(1, (d->n + 255) / 256), want = std::max<long long>(1, 2048 / cols);
    b.rows = (int)std::max<long long>(16, (d->m + want - 1) / want);
    if (d->dbias && !empty) b.db_bytes = align_up((size_t)((d->m + b.rows - 1) / b.rows) * d->n * 4, 256);
    b.blocks = (int)((d->m + b.rows - 1) / b.rows);
    b.scaled = b.own_dp && b.parts == 2 && d->type == YOLO_AMD_TYPE_F16;
    if (b.scaled) b.scale_bytes = align_up(((size_t)b.blocks * cols + 2) * 4, 256);
    if (!products) return b;
    if (d->dx) {
        b.dx = plan_product(d->m, (int)d->k, d->n, false, YOLO_AMD_ACT_NONE, b.parts);
        b.w_bytes = packed_bytes(b.w);
        b.part_bytes = partial_bytes(b.dx, d->m, (int)d->k);
    }
    if (d->dweight) {
        b.dw = plan_product(d->n, (int)d->k, d->m, false, YOLO_AMD_ACT_NONE, b.parts);
        b.x_bytes = packed_bytes(b.x);
        b.part_bytes = std::max(b.part_bytes, partial_bytes(b.dw, d->n, (int)d->k));
    }
    return b;
}

static int check_plan(const yolo_amd_linear_backward_desc* d, const LinearBackwardPlan& b) {
    if (d->m == 0 || d->n == 0 || d->k == 0) return YA_OK;
    if (d->dx) YA_TRY(check_plan("linear_backward", b.dx, d->m, d->k));
    if (d->dweight) YA_TRY(check_plan("linear_backward", b.dw, d->n, d->k));
    return YA_OK;
}

template <typename T>
__global__ void __launch_bounds__(256) linear_zero_kernel(T* p, long long n) {
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) p[i] = (T)0.f;
}
template <typename T>
static void launch_zero(T* p, long long n, hipStream_t s) {
    if (n > 0) hipLaunchKernelGGL((linear_zero_kernel<T>), dim3((unsigned)std::min<long long>((n + 255) / 256, 4096)), dim3(256), 0, s, p, n);
}

template <typename T>
static int backward(const yolo_amd_linear_backward_desc* d, const LinearBackwardPlan& b, hipStream_t s) {
    const int M = (int)d->m, N = (int)d->n, K = (int)d->k;
    if (M == 0 || N == 0) {                       // sums over nothing are zero
        if (d->dx) launch_zero((T*)d->dx, (long long)M * K, s);
        if (d->dweight) launch_zero((T*)d->dweight, (long long)N * K, s);
        if (d->dbias && d->dbias_f32) launch_zero((float*)d->dbias, N, s);
        else if (d->dbias) launch_zero((T*)d->dbias, N, s);
        YA_CHECK_HIP(hipGetLastError());
        return YA_OK;
    }
    Scratch sc{(char*)d->workspace};
    void* dp = sc.take(b.dp_bytes);
    float* db = (float*)sc.take(b.db_bytes);
    float* scale = b.scaled ? (float*)sc.take(b.scale_bytes) : nullptr;    // the two of them, then the peaks
    if (b.own_dp || d->dbias) {
        DpreArgs g{};
        g.dy = d->dy; g.lddy = d->lddy; g.dy_f32 = d->dy_f32;
        g.act = d->activation; g.pre_f32 = d->pre_f32;
        g.pre = g.act == YOLO_AMD_ACT_NONE ? nullptr : d->pre;
        g.ldpre = N;
        g.dp = b.own_dp ? dp : nullptr;
        g.dp_lo = b.own_dp && b.parts == 2 ? (char*)dp + b.dp_bytes / 2 : nullptr;
        g.ldp = (long long)align_up(N, 8);
        g.part = d->dbias ? db : nullptr;
        g.M = M; g.N = N; g.rows = b.rows;
        const dim3 grid((N + 255) / 256, b.blocks);
        if (b.scaled) {                           // the largest value first: dY and P are read twice
            DpreArgs first = g;
            first.dp = first.dp_lo = nullptr;
            first.peaks = scale + 2;
            g.part = nullptr;
            g.scale = scale;
            hipLaunchKernelGGL((linear_dpre_kernel<T>), grid, dim3(256), 0, s, first);
            hipLaunchKernelGGL(linear_scale_kernel, dim3(1), dim3(1024), 0, s, scale + 2, (int)(grid.x * grid.y), scale);
        }
        hipLaunchKernelGGL((linear_dpre_kernel<T>), grid, dim3(256), 0, s, g);
        if (d->dbias)
            hipLaunchKernelGGL((linear_dbias_kernel<T>), dim3((N + 63) / 64), dim3(1024), 0, s, db, b.blocks, N, d->dbias, d->dbias_f32);
    }
    const void* P = b.own_dp ? dp : d->dy;
    const long long ldP = b.own_dp ? (long long)align_up(N, 8) : d->lddy;
    if (K > 0) {
        TileArgs a{};
        a.e.act = YOLO_AMD_ACT_NONE;
        a.e.ldy = K;
        a.e.unscale = b.scaled ? scale + 1 : nullptr;
        a.lo = b.own_dp && b.parts == 2 ? (long long)(b.dp_bytes / 2) : 0;
        Matrix in[2] = {b.x, b.w};
        launch_pack<T>(in, {b.x_bytes, b.w_bytes}, sc, s);
        const Matrix &x = in[0], &w = in[1];
        void* part = sc.take(b.part_bytes);
        if (d->dx) {
            a.A = P; a.lda = ldP;
            a.B = w.p; a.ldb = w.ld;
            a.M = M; a.N = K; a.K = N;
            a.e.y = d->dx;
            YA_TRY((launch_product<T, false, true>(b.dx, a, part, s)));
        }
        if (d->dweight) {
            a.A = P; a.lda = ldP;
            a.B = x.p; a.ldb = x.ld;
            a.M = N; a.N = K; a.K = M;
            a.e.y = d->dweight;
            YA_TRY((launch_product<T, true, true>(b.dw, a, part, s)));
        }
    }
    YA_CHECK_HIP(hipGetLastError());
    return YA_OK;
}

}  // namespace yolo_amd

using namespace yolo_amd;

extern "C" size_t yolo_amd_linear_workspace_bytes(const yolo_amd_linear_desc* d) {
    if (check_forward(d) != YA_OK) return 0;
    const ForwardPlan f = plan_forward(d);
    return check_plan(d, f) == YA_OK ? f.bytes() : 0;
}

extern "C" int yolo_amd_linear_query(const yolo_amd_linear_desc* d, yolo_amd_linear_choice* out) {
    YA_REQUIRE(out, "linear_query: null output");
    YA_TRY(check_forward(d));
    const ForwardPlan f = plan_forward(d);
    YA_TRY(check_plan(d, f));
    *out = yolo_amd_linear_choice{f.tile.kernel, f.tile.bm, f.tile.bn, f.tile.slices, f.x_bytes != 0, f.w_bytes != 0, f.tile.ahead};
    return YA_OK;
}

extern "C" int yolo_amd_linear_forward(const yolo_amd_linear_desc* d, void* stream) {
    YA_TRY(check_forward(d));
    const ForwardPlan f = plan_forward(d);
    if (d->m == 0 || d->n == 0) return YA_OK;
    YA_TRY(check_plan(d, f));
    YA_TRY(check_workspace("linear_forward", d->workspace, d->workspace_bytes, f.bytes()));
    return d->type == YOLO_AMD_TYPE_BF16 ? forward<__bf16>(d, f, (hipStream_t)stream) : forward<_Float16>(d, f, (hipStream_t)stream);
}

extern "C" size_t yolo_amd_linear_backward_workspace_bytes(const yolo_amd_linear_backward_desc* d) {
    if (check_backward(d) != YA_OK) return 0;
    const LinearBackwardPlan b = plan_backward(d);
    return check_plan(d, b) == YA_OK ? b.bytes() : 0;
}

extern "C" int yolo_amd_linear_backward_query(const yolo_amd_linear_backward_desc* d, yolo_amd_linear_choice* dx,
                                              yolo_amd_linear_choice* dweight) {
    YA_REQUIRE(dx && dweight, "linear_backward_query: null output");
    YA_TRY(check_backward(d));
    const LinearBackwardPlan b = plan_backward(d);
    YA_TRY(check_plan(d, b));
    *dx = yolo_amd_linear_choice{b.dx.kernel, b.dx.bm, b.dx.bn, b.dx.slices, 0, b.w_bytes != 0, b.dx.ahead};
    *dweight = yolo_amd_linear_choice{b.dw.kernel, b.dw.bm, b.dw.bn, b.dw.slices, b.x_bytes != 0, 0, b.dw.ahead};
    return YA_OK;
}

extern "C" int yolo_amd_linear_backward(const yolo_amd_linear_backward_desc* d, void* stream) {
    YA_TRY(check_backward(d));
    const LinearBackwardPlan b = plan_backward(d);
    YA_TRY(check_plan(d, b));
    YA_TRY(check_workspace("linear_backward", d->workspace, d->workspace_bytes, b.bytes()));
    return d->type == YOLO_AMD_TYPE_BF16 ? backward<__bf16>(d, b, (hipStream_t)stream) : backward<_Float16>(d, b, (hipStream_t)stream);
}
