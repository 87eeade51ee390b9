// Norms after and before a block, fused with the block's gate, residual scale and residual add; forward and
// backward, for gfx950.  Per row of D values:
//
//   p = after ? norm(u) * wa + ba : u        norm(v) = v / sqrt(mean(v^2) + eps)                  (rms)
//   h = r + s * g * p                                  (v - mean(v)) / sqrt(var(v) + eps)         (layer)
//   y = norm(h) * wb + bb
//
//   q  = dy * wb;  dH = dh + f_h (q - [mean(q)] - h^ mean(q h^))       h^ = norm(h), f_h its factor
//   dr = dH;  dg = s p dH (summed over the rows that share the gate);  dp = s g dH
//   q' = dp * wa;  du = after ? f_u (q' - [mean(q')] - u^ mean(q' u^)) : dp
//   dwb = sum dy h^;  dbb = sum dy;  dwa = sum dp u^;  dba = sum dp    over all rows
//
// Memory bound: a row is read once, held in registers (a group of TPR threads, 8 * CH values each) through
// every statistic, and written once.  The backward kernel recomputes p and h from u and r instead of reading a
// stored h: the same bytes, and no rounding of h enters the gradients.  Statistics and sums are fp32; a variance
// is taken around its mean in a second sweep over the registers.
//   forward: 16384 x 4096 bf16 with an fp32 stream 150 to 164 us, 4.9 to 5.4 TB/s (a copy of that size reaches 5.5);
//     8192 x 2048 bf16 33 to 35 us, 3.9 to 4.1 TB/s
//   backward: 8192 x 2048 bf16 46 us, 4.4 TB/s, and 6 for the partial sums
// (kernel times under rocprofv3; called again and again on the same inputs, partly in the caches, they are lower.)
#pragma once
#include <algorithm>

#include "common.h"
#include "../../include/yolo_amd.h"

namespace yolo_amd {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

struct NormArgs {
    const void *x, *res, *gate, *aw, *ab, *bw, *bb;
    long long ldx, ldr;
    void *h, *y;
    long long rows;
    int D;
    int gate_f32, after_f32, before_f32;
    long long rows_per_gate;       // rows that share a row of the gate
    int gate_shared;               // all of them do
    int after, before, layer;
    float eps, scale, inv_d;
    // backward
    const void *dy, *dh;
    void *dx, *dres, *dgate;       // dgate here: a gate row per token, written directly
    float* part;                   // [block][vector][D] column sums of this launch's blocks
    int vectors;                   // vectors per block, in the order wb, wa, gate, bb, ba (those that are wanted)
    int at_wb, at_wa, at_g, at_bb, at_ba;   // position among them, or -1
    // rows are walked as `sequences` runs of `length` rows; block (i, c): runs i * seq_per_block .., chunk c of `chunks`
    long long sequences, length, chunk_rows;
    int seq_per_block, chunks;
    float* gate_part;              // [sequence][chunk][D]: gate sums where a run of rows shares a gate row
};

// Eight consecutive values at the elements' own alignment (the machine takes 16-byte accesses anywhere).
template <typename S>
struct Eight {
    typedef S vec __attribute__((ext_vector_type(8)));
    typedef S vecu __attribute__((ext_vector_type(8), aligned(sizeof(S))));
};

// The columns thread t of a group owns: CH runs of eight, TPR * 8 apart.  D may be any number: a run that would pass the
// row's end holds the row's last eight values instead, and those of them that are not its own (the run before it owns
// them, or it owns none) are left out of sums and stores.
//   FULL: the threads there are hold exactly D columns and none needs a check.
//   EIGHTS: D is a multiple of 8: a run is the row's or it is not.
//   ANY: element by element, in the waves that hold a row's end.
// (rms, bf16, forward, 67 MB in and out: rows of 1536, FULL, 25 us; of 1528, EIGHTS, 30; of 1500, ANY, 38, with
// every other row starting between 16-byte boundaries.)
enum { ANY, EIGHTS, FULL };
template <int TPR, int CH, int MODE>
struct Cols {
    static constexpr int E = CH * 8;
    // run c's first column as counted, and as held
    __device__ static __forceinline__ int run(int t, int c) { return (c * TPR + t) * 8; }
    __device__ static __forceinline__ int held(int t, int c, int D) { return MODE == FULL ? run(t, c) : min(run(t, c), max(D - 8, 0)); }
    __device__ static __forceinline__ int col(int t, int e, int D) { return held(t, e >> 3, D) + (e & 7); }
    // is element e a column of its own
    __device__ static __forceinline__ bool in(int t, int e, int D) {
        const int c = col(t, e, D);
        return MODE == FULL || (MODE == EIGHTS ? run(t, e >> 3) < D : c >= run(t, e >> 3) && c < D);
    }
    // has this wave (ANY) a run that is not whole
    __device__ static __forceinline__ bool edge(int t, int c, int D) { return __builtin_amdgcn_ballot_w64(run(t, c) + 8 > D) != 0; }
    // sum over the thread's columns; add(e, s): s and element e's share
    template <typename F>
    __device__ static __forceinline__ float total(int t, int D, F add) {
        float s = 0.f;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            float r = 0.f;
            if (MODE == ANY && edge(t, c, D)) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float n = add(c * 8 + i, r);
                    r = in(t, c * 8 + i, D) ? n : r;
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) r = add(c * 8 + i, r);
            }
            if (MODE == EIGHTS) r = in(t, c * 8, D) ? r : 0.f;
            s = c ? s + r : r;
        }
        return s;
    }

    // a row's values as they are in memory, so that a row can be on its way while another is worked on
    template <typename S>
    struct Raw {
        typename Eight<S>::vec v[CH];
        __device__ __forceinline__ void load(const S* row, int D, int t) {
            if (MODE != ANY || D >= 8) {
#pragma unroll
                for (int c = 0; c < CH; ++c) {
                    const typename Eight<S>::vecu x = *reinterpret_cast<const typename Eight<S>::vecu*>(row + held(t, c, D));
                    v[c] = x;
                }
            } else {                                   // a row shorter than eight: by element
#pragma unroll
                for (int i = 0; i < 8; ++i) v[0][i] = row[min(i, D - 1)];
            }
        }
        __device__ __forceinline__ void get(float (&f)[E]) const {
#pragma unroll
            for (int e = 0; e < E; ++e) f[e] = (float)v[e >> 3][e & 7];
        }
    };
    template <typename S>
    __device__ static __forceinline__ void store(S* row, int D, int t, const float (&v)[E]) {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int at = run(t, c);
            if (MODE == FULL || at + 8 <= D) {
                typename Eight<S>::vecu x;
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = (S)v[c * 8 + i];
                *reinterpret_cast<typename Eight<S>::vecu*>(row + at) = x;
            } else if (MODE == ANY && at < D) {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (in(t, c * 8 + i, D)) row[col(t, c * 8 + i, D)] = (S)v[c * 8 + i];
            }
        }
    }
    // a parameter row, fp32 or T, in two steps: the same registers for either
    template <typename T>
    struct Param {
        u32x4 w[CH][2];
        __device__ __forceinline__ void load(const void* p, int f32, long long at, int D, int t) {
            if (f32) {
                Raw<float> r;
                r.load((const float*)p + at, D, t);
#pragma unroll
                for (int c = 0; c < CH; ++c) {
                    w[c][0] = __builtin_bit_cast(u32x4, __builtin_shufflevector(r.v[c], r.v[c], 0, 1, 2, 3));
                    w[c][1] = __builtin_bit_cast(u32x4, __builtin_shufflevector(r.v[c], r.v[c], 4, 5, 6, 7));
                }
            } else if constexpr (sizeof(T) == 2) {
                Raw<T> r;
                r.load((const T*)p + at, D, t);
#pragma unroll
                for (int c = 0; c < CH; ++c) w[c][0] = __builtin_bit_cast(u32x4, r.v[c]);
            }
        }
        __device__ __forceinline__ void get(int f32, float (&f)[E]) const {
            if (f32) {
#pragma unroll
                for (int e = 0; e < E; ++e) f[e] = __uint_as_float(w[e >> 3][(e >> 2) & 1][e & 3]);
            } else if constexpr (sizeof(T) == 2) {
#pragma unroll
                for (int c = 0; c < CH; ++c) {
                    const typename Eight<T>::vec v = __builtin_bit_cast(typename Eight<T>::vec, w[c][0]);
#pragma unroll
                    for (int i = 0; i < 8; ++i) f[c * 8 + i] = (float)v[i];
                }
            }
        }
    };
    template <typename T>
    __device__ static __forceinline__ void param(const void* p, int f32, long long at, int D, int t, float (&v)[E]) {
        Param<T> r;
        r.load(p, f32, at, D, t);
        r.get(f32, v);
    }
};

// sum over the 64 lanes, the same bits in every lane
__device__ __forceinline__ float wave_sum(float v) {
    // lanes 1, 2 (quad_perm), 4 (row_half_mirror) and 8 (row_mirror) apart, then the four rows of 16
#define YA_DPP_ADD(ctrl) v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), ctrl, 0xF, 0xF, true))
    YA_DPP_ADD(0xB1);
    YA_DPP_ADD(0x4E);
    YA_DPP_ADD(0x141);
    YA_DPP_ADD(0x140);
#undef YA_DPP_ADD
    const int b = __float_as_int(v);
    return (__int_as_float(__builtin_amdgcn_readlane(b, 0)) + __int_as_float(__builtin_amdgcn_readlane(b, 16))) +
           (__int_as_float(__builtin_amdgcn_readlane(b, 32)) + __int_as_float(__builtin_amdgcn_readlane(b, 48)));
}

// Sums over a group of TPR threads (or of the first so many waves of them: see threads_of); every thread of the
// workgroup makes the same calls.  Two slot sets in turn: a set is written again only after the barrier of the call in
// between, which its readers reach after reading.
template <int TPR, int NT>
struct GroupSum {
    float (*slots)[2][NT / 64];
    int parity;
    // waves that are not there add zeros (their slots are written here alone, ahead of the first call's barrier)
    __device__ __forceinline__ void init() {
        parity = 0;
        const int w = threadIdx.x % (NT / 64);
        if (threadIdx.x < 4 * (NT / 64) && w >= (int)(blockDim.x >> 6)) (&slots[0][0][0])[threadIdx.x] = 0.f;
    }
    __device__ __forceinline__ void two(float& a, float& b) {
        a = wave_sum(a);
        b = wave_sum(b);
        if constexpr (TPR > 64) {
            const int w = threadIdx.x >> 6;
            if ((threadIdx.x & 63) == 0) {
                slots[parity][0][w] = a;
                slots[parity][1][w] = b;
            }
            __syncthreads();
            const int w0 = w / (TPR / 64) * (TPR / 64);
            a = slots[parity][0][w0];
            b = slots[parity][1][w0];
#pragma unroll
            for (int i = 1; i < TPR / 64; ++i) {
                a += slots[parity][0][w0 + i];
                b += slots[parity][1][w0 + i];
            }
            parity ^= 1;
        }
    }
    __device__ __forceinline__ float one(float a) {
        a = wave_sum(a);
        if constexpr (TPR > 64) {
            const int w = threadIdx.x >> 6;
            if ((threadIdx.x & 63) == 0) slots[parity][0][w] = a;
            __syncthreads();
            const int w0 = w / (TPR / 64) * (TPR / 64);
            a = slots[parity][0][w0];
#pragma unroll
            for (int i = 1; i < TPR / 64; ++i) a += slots[parity][0][w0 + i];
            parity ^= 1;
        }
        return a;
    }
};

__device__ __forceinline__ long long gate_row(const NormArgs& a, long long row) {
    return a.gate_shared ? 0 : (long long)((uint32_t)row / (uint32_t)a.rows_per_gate);
}

// mean (0 for rms) and factor of a row
template <typename C, typename G>
__device__ __forceinline__ void row_stats(const float (&v)[C::E], const NormArgs& a, int t, G& sum, float& mean, float& f) {
    mean = 0.f;
    if (a.layer) {
        const float s = C::total(t, a.D, [&](int e, float r) { return r + v[e]; });
        mean = sum.one(s) * a.inv_d;
    }
    const float q = C::total(t, a.D, [&](int e, float r) {
        const float d = v[e] - mean;
        return fmaf(d, d, r);
    });
    f = rsqrtf(sum.one(q) * a.inv_d + a.eps);
}

template <typename T, typename R, int TPR, int CH, int MODE>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR)
block_norm_forward_kernel(const NormArgs a) {
    constexpr int NT = TPR < 256 ? 256 : TPR, GROUPS = NT / TPR, E = CH * 8;
    typedef Cols<TPR, CH, MODE> C;
    __shared__ float slots[2][2][NT / 64];
    GroupSum<TPR, NT> sum{slots};
    sum.init();
    const int t = threadIdx.x % TPR, group = threadIdx.x / TPR;
    for (long long base = (long long)blockIdx.x * GROUPS; base < a.rows; base += (long long)gridDim.x * GROUPS) {
        const bool valid = base + group < a.rows;
        const long long row = valid ? base + group : a.rows - 1;
        float u[E], h[E], w[E];
        typename C::template Raw<T> ru;
        typename C::template Raw<R> rh;
        typename C::template Param<T> rg, rw;
        ru.load((const T*)a.x + row * a.ldx, a.D, t);
        if (a.res) rh.load((const R*)a.res + row * a.ldr, a.D, t);
        if (a.gate) rg.load(a.gate, a.gate_f32, gate_row(a, row) * a.D, a.D, t);
        if (a.aw) rw.load(a.aw, a.after_f32, 0, a.D, t);
        ru.get(u);
        if (a.after) {
            float mean, f;
            row_stats<C>(u, a, t, sum, mean, f);
#pragma unroll
            for (int e = 0; e < E; ++e) u[e] = (u[e] - mean) * f;
            if (a.aw) {
                rw.get(a.after_f32, w);
#pragma unroll
                for (int e = 0; e < E; ++e) u[e] *= w[e];
            }
            if (a.ab) {
                C::template param<T>(a.ab, a.after_f32, 0, a.D, t, w);
#pragma unroll
                for (int e = 0; e < E; ++e) u[e] += w[e];
            }
        }
        if (a.bw) rw.load(a.bw, a.before_f32, 0, a.D, t);
        if (a.gate) {
            rg.get(a.gate_f32, w);
#pragma unroll
            for (int e = 0; e < E; ++e) u[e] *= w[e];
        }
        if (a.res) {
            rh.get(h);
#pragma unroll
            for (int e = 0; e < E; ++e) h[e] = fmaf(a.scale, u[e], h[e]);
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) h[e] = a.scale * u[e];
        }
        if (a.h && valid) C::store((R*)a.h + row * a.D, a.D, t, h);
        if (a.before) {
            float mean, f;
            row_stats<C>(h, a, t, sum, mean, f);
#pragma unroll
            for (int e = 0; e < E; ++e) h[e] = (h[e] - mean) * f;
            if (a.bw) {
                rw.get(a.before_f32, w);
#pragma unroll
                for (int e = 0; e < E; ++e) h[e] *= w[e];
            }
            if (a.bb) {
                C::template param<T>(a.bb, a.before_f32, 0, a.D, t, w);
#pragma unroll
                for (int e = 0; e < E; ++e) h[e] += w[e];
            }
            if (valid) C::store((T*)a.y + row * a.D, a.D, t, h);
        }
    }
}

// The column sums of a workgroup: N vectors, each thread's columns of each.  As many of them in LDS as fit (a thread only
// ever touches its own words, in order): the registers they would take hide more of memory's latency as further waves,
// and with sixteen columns to a thread there are none to spare (2048 rows of 8192, layer, bf16 with an fp32 stream: in
// registers 150 us, in LDS 90).
template <typename C, int TPR, int GROUPS, int N>
struct Sums {
    static constexpr int NT = TPR * GROUPS, Q = C::E / 4;
    static constexpr int FIT = ((C::E == 8 ? 80 : 160) * 1024 - 1024) / (C::E * NT * 4), IN_LDS = FIT < N ? FIT : N;
    static constexpr int WORDS = IN_LDS * Q * NT;
    static_assert(IN_LDS == N || GROUPS == 1, "rows this long have a workgroup each");
    f32x4* lds;                                        // WORDS of them
    float v[IN_LDS < N ? N - IN_LDS : 1][C::E];

    __device__ __forceinline__ void clear(int k) {
        if (k < IN_LDS) {
#pragma unroll
            for (int q = 0; q < Q; ++q) lds[(k * Q + q) * NT + threadIdx.x] = f32x4{0.f, 0.f, 0.f, 0.f};
        } else {
#pragma unroll
            for (int e = 0; e < C::E; ++e) v[k - IN_LDS][e] = 0.f;
        }
    }
    // sums[k] += x * y
    __device__ __forceinline__ void add(int k, const float (&x)[C::E], const float (&y)[C::E]) {
        if (k < IN_LDS) {
#pragma unroll
            for (int q = 0; q < Q; ++q) {
                f32x4 s = lds[(k * Q + q) * NT + threadIdx.x];
#pragma unroll
                for (int i = 0; i < 4; ++i) s[i] = fmaf(x[q * 4 + i], y[q * 4 + i], s[i]);
                lds[(k * Q + q) * NT + threadIdx.x] = s;
            }
        } else {
#pragma unroll
            for (int e = 0; e < C::E; ++e) v[k - IN_LDS][e] = fmaf(x[e], y[e], v[k - IN_LDS][e]);
        }
    }
    __device__ __forceinline__ void add(int k, const float (&x)[C::E]) {
        float one[C::E];
#pragma unroll
        for (int e = 0; e < C::E; ++e) one[e] = 1.f;
        add(k, x, one);
    }
    // the groups' sums in group order -> out[0 .. D); every thread calls it
    __device__ __forceinline__ void write(int k, int t, int group, int D, float* out) {
        if (k < IN_LDS) {
            __syncthreads();
            if (group == 0) {
#pragma unroll
                for (int q = 0; q < Q; ++q) {
                    f32x4 s = lds[(k * Q + q) * NT + t];
#pragma unroll
                    for (int g = 1; g < GROUPS; ++g) s += lds[(k * Q + q) * NT + g * TPR + t];
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (C::in(t, q * 4 + i, D)) out[C::col(t, q * 4 + i, D)] = s[i];
                }
            }
            __syncthreads();
        } else {
#pragma unroll
            for (int e = 0; e < C::E; ++e)
                if (C::in(t, e, D)) out[C::col(t, e, D)] = v[k - IN_LDS][e];
        }
    }
};

// The next row of each group is on its way (as it is in memory) while one is worked on; parameters that all rows share
// stay in registers.  1024 threads of sixteen columns have 128 registers each, too few for either: they read a row where
// it is used, and the parameters (from L2) again with every row (2048 bf16 rows of 16384, rms: 149 us, otherwise 331).
template <typename T, typename R, int TPR, int CH, int MODE, bool LAYER>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR)
block_norm_backward_kernel(const NormArgs a) {
    constexpr int NT = TPR < 256 ? 256 : TPR, GROUPS = NT / TPR, E = CH * 8;
    constexpr bool AHEAD = TPR * CH < 2048;
    typedef Cols<TPR, CH, MODE> C;
    __shared__ float slots[2][2][NT / 64];
    enum { WB, WA, WG, BB, BA };
    typedef Sums<C, TPR, GROUPS, LAYER ? 5 : 3> S;
    __shared__ f32x4 words[S::WORDS];
    S sums;
    sums.lds = words;
    GroupSum<TPR, NT> sum{slots};
    sum.init();
    const int t = threadIdx.x % TPR, group = threadIdx.x / TPR;
    const int chunk = blockIdx.x % a.chunks;
    const long long s0 = (long long)(blockIdx.x / a.chunks) * a.seq_per_block;
    const long long s1 = min(a.sequences, s0 + a.seq_per_block);
#pragma unroll
    for (int k = 0; k < (LAYER ? 5 : 3); ++k) sums.clear(k);
    const bool row_gate = a.gate && !a.gate_shared;
    float pa[E], pb[E], pg[E];
    auto parameter = [&](const void* p, int f32, long long at, float (&v)[E]) {
        if constexpr (!AHEAD) asm volatile("" : "+s"(at));     // not to be read ahead of the loop and kept after all
        if (p) {
            C::template param<T>(p, f32, at, a.D, t, v);
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = 1.f;
        }
    };
    auto after_weight = [&] { parameter(a.aw, a.after_f32, 0, pa); };
    auto before_weight = [&] { parameter(a.bw, a.before_f32, 0, pb); };
    auto gate_of = [&](long long row) { parameter(a.gate, a.gate_f32, a.gate ? gate_row(a, row) * a.D : 0, pg); };
    if constexpr (AHEAD) {
        after_weight();
        before_weight();
        gate_of(0);                                    // of all rows, or none
    }
    typename C::template Raw<T> ru, ry;
    typename C::template Raw<R> rh, rd;
    typename C::template Param<T> rg;
    auto fetch_values = [&](long long row) {
        ru.load((const T*)a.x + row * a.ldx, a.D, t);
        if (a.res) rh.load((const R*)a.res + row * a.ldr, a.D, t);
        if (AHEAD && row_gate) rg.load(a.gate, a.gate_f32, gate_row(a, row) * a.D, a.D, t);
    };
    auto fetch_gradients = [&](long long row) {
        if (a.dy) ry.load((const T*)a.dy + row * a.D, a.D, t);
        if (a.dh) rd.load((const R*)a.dh + row * a.D, a.D, t);
    };
    for (long long seq = s0; seq < s1; ++seq) {
        const long long r0 = seq * a.length + chunk * a.chunk_rows;
        const long long r1 = min(seq * a.length + a.length, r0 + a.chunk_rows);
        if constexpr (AHEAD) {
            fetch_values(min(r0 + group, r1 - 1));
            fetch_gradients(min(r0 + group, r1 - 1));
        }
        for (long long base = r0; base < r1; base += GROUPS) {
            const bool valid = base + group < r1;
            const long long row = valid ? base + group : r1 - 1;
            const long long next = min(base + GROUPS + group, r1 - 1);
            const bool more = AHEAD && base + GROUPS < r1;
            float u[E], h[E], d[E], dy[E], p[E];
            if constexpr (!AHEAD) fetch_values(row);
            ru.get(u);
#pragma unroll
            for (int e = 0; e < E; ++e) h[e] = d[e] = 0.f;
            if (a.res) rh.get(h);
            if (AHEAD && row_gate) rg.get(a.gate_f32, pg);
            auto gradients = [&] {
                if constexpr (!AHEAD) fetch_gradients(row);
                if (a.dy) ry.get(dy);
                if (a.dh) rd.get(d);
            };
            // sixteen columns to a thread: the gradients later, when fewer registers are taken
            if constexpr (CH == 1) gradients();
            if (more) fetch_values(next);
            if (CH == 1 && more) fetch_gradients(next);
            // forward again: u becomes u^ (its norm without weights), h the stream
            float fu = 1.f;
            if (a.after) {
                float mean;
                row_stats<C>(u, a, t, sum, mean, fu);
#pragma unroll
                for (int e = 0; e < E; ++e) u[e] = (u[e] - mean) * fu;
            }
            if constexpr (!AHEAD) after_weight();
#pragma unroll
            for (int e = 0; e < E; ++e) p[e] = u[e] * pa[e];
            if (LAYER && a.ab) {
                float w[E];
                C::template param<T>(a.ab, a.after_f32, 0, a.D, t, w);
#pragma unroll
                for (int e = 0; e < E; ++e) p[e] += w[e];
            }
            float mean_h = 0.f, fh = 0.f;
            if (a.dy) {
                if constexpr (!AHEAD) gate_of(row);
#pragma unroll
                for (int e = 0; e < E; ++e) h[e] = fmaf(a.scale, pg[e] * p[e], h[e]);
                row_stats<C>(h, a, t, sum, mean_h, fh);
            }
            if constexpr (CH > 1) gradients();
            if (CH > 1 && more) fetch_gradients(next);
            if (a.dy) {
#pragma unroll
                for (int e = 0; e < E; ++e) h[e] = (h[e] - mean_h) * fh;
                if (valid) {
                    if (a.at_wb >= 0) sums.add(WB, dy, h);
                    if (LAYER && a.at_bb >= 0) sums.add(BB, dy);
                }
                if constexpr (!AHEAD) before_weight();
#pragma unroll
                for (int e = 0; e < E; ++e) dy[e] *= pb[e];
                float c0 = C::total(t, a.D, [&](int e, float r) { return r + dy[e]; });
                float c1 = C::total(t, a.D, [&](int e, float r) { return fmaf(dy[e], h[e], r); });
                if (LAYER) sum.two(c0, c1);
                else { c1 = sum.one(c1); c0 = 0.f; }
                c0 *= a.inv_d;
                c1 *= a.inv_d;
#pragma unroll
                for (int e = 0; e < E; ++e) d[e] = d[e] + fh * (dy[e] - c0 - h[e] * c1);
            }
            if (a.dres && valid) C::store((R*)a.dres + row * a.D, a.D, t, d);
            // gate
            if constexpr (!AHEAD) gate_of(row);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                p[e] *= a.scale * d[e];
                d[e] *= a.scale * pg[e];
            }
            if (a.dgate && valid) {
                if (a.gate_f32) C::store((float*)a.dgate + row * a.D, a.D, t, p);
                else C::store((T*)a.dgate + row * a.D, a.D, t, p);
            }
            if (valid) {
                if (a.gate_part || a.at_g >= 0) sums.add(WG, p);
                if (a.at_wa >= 0) sums.add(WA, d, u);
                if (LAYER && a.at_ba >= 0) sums.add(BA, d);
            }
            if (a.after && a.dx) {
                if constexpr (!AHEAD) after_weight();
#pragma unroll
                for (int e = 0; e < E; ++e) d[e] *= pa[e];
                float c0 = C::total(t, a.D, [&](int e, float r) { return r + d[e]; });
                float c1 = C::total(t, a.D, [&](int e, float r) { return fmaf(d[e], u[e], r); });
                if (LAYER) sum.two(c0, c1);
                else { c1 = sum.one(c1); c0 = 0.f; }
                c0 *= a.inv_d;
                c1 *= a.inv_d;
#pragma unroll
                for (int e = 0; e < E; ++e) d[e] = fu * (d[e] - c0 - u[e] * c1);
            }
            if (a.dx && valid) C::store((T*)a.dx + row * a.D, a.D, t, d);
        }
        if (a.gate_part) {
            sums.write(WG, t, group, a.D, a.gate_part + (seq * a.chunks + chunk) * a.D);
            sums.clear(WG);
        }
    }
    float* out = a.part + (long long)blockIdx.x * a.vectors * a.D;
    if (a.at_wb >= 0) sums.write(WB, t, group, a.D, out + (long long)a.at_wb * a.D);
    if (a.at_wa >= 0) sums.write(WA, t, group, a.D, out + (long long)a.at_wa * a.D);
    if (a.at_g >= 0) sums.write(WG, t, group, a.D, out + (long long)a.at_g * a.D);
    if (LAYER && a.at_bb >= 0) sums.write(BB, t, group, a.D, out + (long long)a.at_bb * a.D);
    if (LAYER && a.at_ba >= 0) sums.write(BA, t, group, a.D, out + (long long)a.at_ba * a.D);
}

// ---------------------------------------------------------------- launch, one translation unit per element type
// Threads per row by its length: eight values each; sixteen where twelve waves of eight (forward: two rows to a CU;
// 2048 bf16 rows of 8192, rms: 16 waves 29.9 us, 8 of sixteen 26.5) or 512 threads (backward, whose row, parameters and
// column sums share the registers) do not hold it.
// A row with a workgroup of its own has as many waves as it fills: the registers of those that would only wait hold
// another row's (forward, 3048 rows of 5504: 16 waves 61 us, 11 waves 47, and 30 with EIGHTS).
template <int TPR, int CH>
static inline int threads_of(int D) {
    return TPR < 256 ? 256 : CH > 1 ? TPR : (D + 511) / 512 * 64;
}
template <int TPR, int CH>
static inline int mode_of(int D) {
    return (TPR < 256 || CH > 1 ? D == TPR * CH * 8 : D % 512 == 0) ? FULL : D % 8 == 0 ? EIGHTS : ANY;
}
template <typename T, typename R, int TPR, int CH>
static void norm_launch_forward(const NormArgs& a, int blocks, hipStream_t s) {
    const dim3 threads(threads_of<TPR, CH>(a.D));
    switch (mode_of<TPR, CH>(a.D)) {
        case FULL: hipLaunchKernelGGL((block_norm_forward_kernel<T, R, TPR, CH, FULL>), dim3(blocks), threads, 0, s, a); break;
        case EIGHTS: hipLaunchKernelGGL((block_norm_forward_kernel<T, R, TPR, CH, EIGHTS>), dim3(blocks), threads, 0, s, a); break;
        default: hipLaunchKernelGGL((block_norm_forward_kernel<T, R, TPR, CH, ANY>), dim3(blocks), threads, 0, s, a);
    }
}
template <typename T, typename R, int TPR, int CH, int MODE>
static void norm_launch_backward(const NormArgs& a, int blocks, hipStream_t s) {
    const dim3 threads(threads_of<TPR, CH>(a.D));
    if (a.layer) hipLaunchKernelGGL((block_norm_backward_kernel<T, R, TPR, CH, MODE, true>), dim3(blocks), threads, 0, s, a);
    else hipLaunchKernelGGL((block_norm_backward_kernel<T, R, TPR, CH, MODE, false>), dim3(blocks), threads, 0, s, a);
}
template <typename T, typename R, int TPR, int CH>
static void norm_launch_backward(const NormArgs& a, int blocks, hipStream_t s) {
    switch (mode_of<TPR, CH>(a.D)) {
        case FULL: norm_launch_backward<T, R, TPR, CH, FULL>(a, blocks, s); break;
        case EIGHTS: norm_launch_backward<T, R, TPR, CH, EIGHTS>(a, blocks, s); break;
        default: norm_launch_backward<T, R, TPR, CH, ANY>(a, blocks, s);
    }
}

// rows a workgroup has in hand at a time
static inline int norm_forward_groups(int D) { return D <= 512 ? 4 : D <= 1024 ? 2 : 1; }
static inline int norm_backward_groups(int D) { return D <= 512 ? 4 : D <= 1024 ? 2 : 1; }
template <typename T, typename R>
static void norm_launch(const NormArgs& a, int blocks, bool backward, hipStream_t s) {
    if (!backward) {
        if (a.D <= 512) norm_launch_forward<T, R, 64, 1>(a, blocks, s);
        else if (a.D <= 1024) norm_launch_forward<T, R, 128, 1>(a, blocks, s);
        else if (a.D <= 2048) norm_launch_forward<T, R, 256, 1>(a, blocks, s);
        else if (a.D <= 4096) norm_launch_forward<T, R, 512, 1>(a, blocks, s);
        else if (a.D <= 6144) norm_launch_forward<T, R, 1024, 1>(a, blocks, s);
        else if (a.D <= 8192) norm_launch_forward<T, R, 512, 2>(a, blocks, s);
        else norm_launch_forward<T, R, 1024, 2>(a, blocks, s);
    } else {
        if (a.D <= 512) norm_launch_backward<T, R, 64, 1>(a, blocks, s);
        else if (a.D <= 1024) norm_launch_backward<T, R, 128, 1>(a, blocks, s);
        else if (a.D <= 2048) norm_launch_backward<T, R, 256, 1>(a, blocks, s);
        else if (a.D <= 4096) norm_launch_backward<T, R, 512, 1>(a, blocks, s);
        else if (a.D <= 8192) norm_launch_backward<T, R, 512, 2>(a, blocks, s);
        else norm_launch_backward<T, R, 1024, 2>(a, blocks, s);
    }
}

void block_norm_launch_bf16(const NormArgs& a, bool stream_f32, int blocks, bool backward, hipStream_t s);
void block_norm_launch_f16(const NormArgs& a, bool stream_f32, int blocks, bool backward, hipStream_t s);
void block_norm_launch_f32(const NormArgs& a, int blocks, bool backward, hipStream_t s);

}  // namespace yolo_amd
