// The kernels of block_norm.h for fp32 rows, and the entry points of the operator.
#include "block_norm.h"

namespace yolo_amd {

void block_norm_launch_f32(const NormArgs& a, int blocks, bool backward, hipStream_t s) {
    norm_launch<float, float>(a, blocks, backward, s);
}

// Sums of partial column sums: out[o][c] = sum over b of part[(o * blocks + b) * stride + c], b ascending within
// each of the workgroup's 16 waves, the waves in order.  745 blocks x 3 vectors of 2048: 6.0 us, 18 MB; else latency.
struct SumArgs {
    const float* part[5];
    void* out[5];
    int f32[5];
    int n, blocks, D, type;
    long long stride, outer_stride, out_stride;
};
__global__ void __launch_bounds__(1024)
block_norm_sum_kernel(const SumArgs a) {
    __shared__ float red[16][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int c = blockIdx.x * 64 + lane, v = blockIdx.y;
    float s = 0.f;
    if (c < a.D) {
        const float* p = a.part[v] + blockIdx.z * a.outer_stride + c;
#pragma unroll 8
        for (int b = w; b < a.blocks; b += 16) s += p[b * a.stride];
    }
    red[w][lane] = s;
    __syncthreads();
    if (w == 0 && c < a.D) {
#pragma unroll
        for (int i = 1; i < 16; ++i) s += red[i][lane];
        const long long at = blockIdx.z * a.out_stride + c;
        if (a.f32[v]) ((float*)a.out[v])[at] = s;
        else if (a.type == YOLO_AMD_TYPE_BF16) ((__bf16*)a.out[v])[at] = (__bf16)s;
        else ((_Float16*)a.out[v])[at] = (_Float16)s;
    }
}

constexpr int kMaxWidth = 16384;

static int check(const char* me, const yolo_amd_block_norm_desc* d) {
    YA_REQUIRE(d, "%s: null descriptor", me);
    YA_REQUIRE(d->type >= YOLO_AMD_TYPE_F32 && d->type <= YOLO_AMD_TYPE_F16, "%s: type %d", me, d->type);
    YA_REQUIRE(d->norm == YOLO_AMD_NORM_RMS || d->norm == YOLO_AMD_NORM_LAYER, "%s: norm %d", me, d->norm);
    YA_REQUIRE(d->rows >= 0 && d->rows < (1ll << 31) && d->d >= 1 && d->d <= kMaxWidth,
               "%s: %lld rows of %lld values (rows of 1 to %d values)", me, (long long)d->rows, (long long)d->d, kMaxWidth);
    YA_REQUIRE(d->eps >= 0.f, "%s: eps=%g", me, (double)d->eps);
    YA_REQUIRE(!d->gate || d->rows_per_gate >= 1, "%s: rows_per_gate=%lld", me, (long long)d->rows_per_gate);
    YA_REQUIRE(d->after || (!d->after_weight && !d->after_bias), "%s: after_weight or after_bias without the norm they belong to", me);
    YA_REQUIRE(d->before || (!d->before_weight && !d->before_bias), "%s: before_weight or before_bias without the norm they belong to", me);
    YA_REQUIRE(d->norm == YOLO_AMD_NORM_LAYER || (!d->after_bias && !d->before_bias), "%s: an rms norm has no bias", me);
    if (d->rows == 0) return YA_OK;
    const int e = d->type == YOLO_AMD_TYPE_F32 ? 4 : 2, r = d->stream_f32 ? 4 : e;
    YA_REQUIRE(d->x && ((uintptr_t)d->x & (e - 1)) == 0, "%s: x is null or not aligned to its elements", me);
    YA_REQUIRE(((uintptr_t)d->residual & (r - 1)) == 0, "%s: residual is not aligned to its elements", me);
    YA_REQUIRE(d->rows == 1 || d->ldx >= d->d, "%s: x has row stride %lld for rows of %lld", me, (long long)d->ldx, (long long)d->d);
    YA_REQUIRE(d->rows == 1 || !d->residual || d->ldr >= d->d, "%s: residual has row stride %lld for rows of %lld", me,
               (long long)d->ldr, (long long)d->d);
    const void* par[5] = {d->gate, d->after_weight, d->after_bias, d->before_weight, d->before_bias};
    const int f32[5] = {d->gate_f32, d->after_f32, d->after_f32, d->before_f32, d->before_f32};
    for (int i = 0; i < 5; ++i)
        YA_REQUIRE(((uintptr_t)par[i] & ((f32[i] ? 4 : e) - 1)) == 0, "%s: a parameter is not aligned to its elements", me);
    return YA_OK;
}

static NormArgs arguments(const yolo_amd_block_norm_desc* d) {
    NormArgs a{};
    const bool f32 = d->type == YOLO_AMD_TYPE_F32;
    a.x = d->x; a.res = d->residual; a.gate = d->gate;
    a.aw = d->after_weight; a.ab = d->after_bias; a.bw = d->before_weight; a.bb = d->before_bias;
    a.ldx = d->ldx; a.ldr = d->ldr;
    a.rows = d->rows; a.D = (int)d->d;
    a.gate_f32 = d->gate_f32 || f32; a.after_f32 = d->after_f32 || f32; a.before_f32 = d->before_f32 || f32;
    a.rows_per_gate = d->gate ? d->rows_per_gate : 1;
    a.gate_shared = d->gate && d->rows_per_gate >= d->rows;
    a.after = d->after != 0; a.before = d->before != 0; a.layer = d->norm == YOLO_AMD_NORM_LAYER;
    a.eps = d->eps; a.scale = d->scale; a.inv_d = 1.f / (float)d->d;
    return a;
}

static int launch(const yolo_amd_block_norm_desc* d, const NormArgs& a, int blocks, bool backward, hipStream_t s) {
    if (d->type == YOLO_AMD_TYPE_BF16) block_norm_launch_bf16(a, d->stream_f32 != 0, blocks, backward, s);
    else if (d->type == YOLO_AMD_TYPE_F16) block_norm_launch_f16(a, d->stream_f32 != 0, blocks, backward, s);
    else block_norm_launch_f32(a, blocks, backward, s);
    YA_CHECK_HIP(hipGetLastError());
    return YA_OK;
}

// How the backward pass cuts its rows: runs that share a gate row (one run where none does), each run in chunks or
// several runs to a block.  A block for every CU, and up to three (what the registers of rows to 2048 allow) where each
// still has four rows or more for each of its groups: every block adds a row of partial sums per parameter.  All kernels of
// the pass, bf16 rms: 24000 rows of 2048 256 blocks 264 us, 512 155, 768 137; 1500 of 4096 33, 38, 44; 300 of 1500 17, 19, 19;
// fp32 layer: 6000 of 1500 101, 68, 62; 1500 of 8192 100, 114, 134.  On 60 sizes from 300 x 256 to 6000 x 8192 the rule is 0.9 %
// behind the best of 256, 384, 512 and 768 (geometric mean; 7 % at the worst).  Runs are not cut and joined across their
// ends: with few rows over the target's count of runs, or between half of it and all, some CUs have none.
struct NormBackwardPlan {
    bool sequence_gate, channel_gate, token_gate;
    long long sequences, length, chunk_rows;
    int seq_per_block, chunks, blocks, vectors;
    size_t part_bytes, gate_bytes;
};

static NormBackwardPlan plan(const yolo_amd_block_norm_backward_desc* b) {
    const yolo_amd_block_norm_desc* d = &b->forward;
    NormBackwardPlan p{};
    if (d->rows == 0) return p;
    const bool want_gate = d->gate && b->dgate;
    p.token_gate = want_gate && d->rows_per_gate == 1;
    p.channel_gate = want_gate && d->rows_per_gate >= d->rows;
    if (p.channel_gate) p.token_gate = false;
    p.sequence_gate = want_gate && !p.token_gate && !p.channel_gate;
    p.length = p.sequence_gate ? d->rows_per_gate : d->rows;
    p.sequences = (d->rows + p.length - 1) / p.length;
    const int groups = norm_backward_groups((int)d->d);
    const long long target = std::min<long long>(d->d <= 2048 ? 768 : 256, std::max<long long>(256, d->rows / (4 * groups)));
    if (p.sequences >= target) {
        p.chunks = 1;
        p.chunk_rows = p.length;
        p.seq_per_block = (int)((p.sequences + target - 1) / target);
    } else {
        p.seq_per_block = 1;
        const long long want = target / p.sequences;
        p.chunk_rows = (p.length + want - 1) / want;
        p.chunk_rows = (p.chunk_rows + groups - 1) / groups * groups;
        p.chunks = (int)((p.length + p.chunk_rows - 1) / p.chunk_rows);
    }
    p.blocks = (int)((p.sequences + p.seq_per_block - 1) / p.seq_per_block) * p.chunks;
    p.vectors = (b->dbefore_weight != nullptr) + (b->dafter_weight != nullptr) + p.channel_gate + (b->dbefore_bias != nullptr) +
                (b->dafter_bias != nullptr);
    p.part_bytes = align_up((size_t)p.blocks * p.vectors * d->d * 4, 256);
    if (p.sequence_gate) p.gate_bytes = align_up((size_t)p.sequences * p.chunks * d->d * 4, 256);
    return p;
}

static int check_backward(const yolo_amd_block_norm_backward_desc* b) {
    const char* me = "block_norm_backward";
    YA_REQUIRE(b, "%s: null descriptor", me);
    const yolo_amd_block_norm_desc* d = &b->forward;
    YA_TRY(check(me, d));
    YA_REQUIRE(!b->dgate || d->gate, "%s: dgate without a gate", me);
    YA_REQUIRE((!b->dafter_weight && !b->dafter_bias) || d->after, "%s: gradients of a norm that is not there (after)", me);
    YA_REQUIRE((!b->dbefore_weight && !b->dbefore_bias) || d->before, "%s: gradients of a norm that is not there (before)", me);
    YA_REQUIRE((!b->dafter_bias && !b->dbefore_bias) || d->norm == YOLO_AMD_NORM_LAYER, "%s: an rms norm has no bias", me);
    YA_REQUIRE(!b->dnormed || d->before, "%s: dnormed without the norm before", me);
    YA_REQUIRE(!d->gate || d->rows % d->rows_per_gate == 0 || d->rows_per_gate >= d->rows,
               "%s: %lld rows are not whole runs of %lld rows that share a gate", me, (long long)d->rows, (long long)d->rows_per_gate);
    const int e = d->type == YOLO_AMD_TYPE_F32 ? 4 : 2, r = d->stream_f32 ? 4 : e;
    YA_REQUIRE((((uintptr_t)b->dnormed | (uintptr_t)b->dx) & (e - 1)) == 0 &&
                   (((uintptr_t)b->dstream | (uintptr_t)b->dresidual) & (r - 1)) == 0 &&
                   ((uintptr_t)b->dgate & ((d->gate_f32 ? 4 : e) - 1)) == 0 &&
                   (((uintptr_t)b->dafter_weight | (uintptr_t)b->dafter_bias) & ((d->after_f32 ? 4 : e) - 1)) == 0 &&
                   (((uintptr_t)b->dbefore_weight | (uintptr_t)b->dbefore_bias) & ((d->before_f32 ? 4 : e) - 1)) == 0,
               "%s: a gradient is not aligned to its elements", me);
    return YA_OK;
}

__global__ void __launch_bounds__(256) block_norm_zero_kernel(char* p, long long n) {
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) p[i] = 0;
}

}  // namespace yolo_amd

using namespace yolo_amd;

extern "C" int yolo_amd_block_norm_forward(const yolo_amd_block_norm_desc* d, void* stream) {
    const char* me = "block_norm_forward";
    YA_TRY(check(me, d));
    if (d->rows == 0) return YA_OK;
    const int e = d->type == YOLO_AMD_TYPE_F32 ? 4 : 2, r = d->stream_f32 ? 4 : e;
    YA_REQUIRE((d->before != 0) == (d->normed != nullptr), "%s: normed goes with the norm before", me);
    YA_REQUIRE(((uintptr_t)d->normed & (e - 1)) == 0 && ((uintptr_t)d->stream & (r - 1)) == 0,
               "%s: an output is not aligned to its elements", me);
    NormArgs a = arguments(d);
    a.h = d->stream;
    a.y = d->normed;
    const int groups = norm_forward_groups(a.D);
    const long long blocks = std::min<long long>((d->rows + groups - 1) / groups, 1 << 20);
    return launch(d, a, (int)blocks, false, (hipStream_t)stream);
}

extern "C" size_t yolo_amd_block_norm_backward_workspace_bytes(const yolo_amd_block_norm_backward_desc* b) {
    if (check_backward(b) != YA_OK) return 0;
    const NormBackwardPlan p = plan(b);
    return p.part_bytes + p.gate_bytes;
}

extern "C" int yolo_amd_block_norm_backward(const yolo_amd_block_norm_backward_desc* b, void* stream) {
    const char* me = "block_norm_backward";
    YA_TRY(check_backward(b));
    const yolo_amd_block_norm_desc* d = &b->forward;
    hipStream_t s = (hipStream_t)stream;
    NormArgs a = arguments(d);
    if (d->rows == 0) {                          // sums over no rows are zero
        void* out[5] = {b->dafter_weight, b->dafter_bias, b->dbefore_weight, b->dbefore_bias, nullptr};
        const int f32[5] = {a.after_f32, a.after_f32, a.before_f32, a.before_f32, 0};
        for (int i = 0; i < 4; ++i)
            if (out[i]) hipLaunchKernelGGL(block_norm_zero_kernel, dim3((a.D + 63) / 64), dim3(256), 0, s, (char*)out[i], (long long)a.D * (f32[i] ? 4 : 2));
        YA_CHECK_HIP(hipGetLastError());
        return YA_OK;
    }
    const NormBackwardPlan p = plan(b);
    const size_t need = p.part_bytes + p.gate_bytes;
    if (need) {
        YA_REQUIRE(b->workspace && ((uintptr_t)b->workspace & 255) == 0, "%s: the workspace is null or not 256-byte aligned", me);
        if (b->workspace_bytes < need) {
            set_error("%s: workspace of %zu bytes, %zu needed", me, b->workspace_bytes, need);
            return YA_ERR_WORKSPACE;
        }
    }
    a.dy = b->dnormed; a.dh = b->dstream;
    a.dx = b->dx; a.dres = b->dresidual;
    a.dgate = p.token_gate ? b->dgate : nullptr;
    a.part = (float*)b->workspace;
    a.gate_part = p.sequence_gate ? (float*)((char*)b->workspace + p.part_bytes) : nullptr;
    a.vectors = p.vectors;
    int at = 0;
    a.at_wb = b->dbefore_weight ? at++ : -1;
    a.at_wa = b->dafter_weight ? at++ : -1;
    a.at_g = p.channel_gate ? at++ : -1;
    a.at_bb = b->dbefore_bias ? at++ : -1;
    a.at_ba = b->dafter_bias ? at++ : -1;
    a.sequences = p.sequences; a.length = p.length; a.chunk_rows = p.chunk_rows;
    a.seq_per_block = p.seq_per_block; a.chunks = p.chunks;
    YA_TRY(launch(d, a, p.blocks, true, s));
    SumArgs g{};
    g.D = a.D;
    g.type = d->type;
    if (at) {
        const int pos[5] = {a.at_wb, a.at_wa, a.at_g, a.at_bb, a.at_ba};
        void* out[5] = {b->dbefore_weight, b->dafter_weight, b->dgate, b->dbefore_bias, b->dafter_bias};
        const int f32[5] = {a.before_f32, a.after_f32, a.gate_f32, a.before_f32, a.after_f32};
        for (int i = 0; i < 5; ++i)
            if (pos[i] >= 0) {
                g.part[g.n] = a.part + (long long)pos[i] * a.D;
                g.out[g.n] = out[i];
                g.f32[g.n++] = f32[i];
            }
        g.blocks = p.blocks;
        g.stride = (long long)p.vectors * a.D;
        hipLaunchKernelGGL(block_norm_sum_kernel, dim3((a.D + 63) / 64, g.n, 1), dim3(1024), 0, s, g);
    }
    if (p.sequence_gate) {
        for (long long z = 0; z < p.sequences; z += 32768) {
            g.n = 1;
            g.part[0] = a.gate_part + z * p.chunks * a.D;
            g.out[0] = (char*)b->dgate + z * a.D * (a.gate_f32 ? 4 : 2);
            g.f32[0] = a.gate_f32;
            g.blocks = p.chunks;
            g.stride = a.D;
            g.outer_stride = (long long)p.chunks * a.D;
            g.out_stride = a.D;
            const unsigned n = (unsigned)std::min<long long>(32768, p.sequences - z);
            hipLaunchKernelGGL(block_norm_sum_kernel, dim3((a.D + 63) / 64, 1, n), dim3(1024), 0, s, g);
        }
    }
    YA_CHECK_HIP(hipGetLastError());
    return YA_OK;
}
