// The norm behind a block, its gate, the residual sum and the norm before the next block, in one pass over the rows:
//     n = post(x),   s = residual_scale r + gate n,   h = pre(s) (1 + mod) + shift,
// post and pre each a layer norm (x - mean) / sqrt(var + eps) w + b, an RMS norm x / sqrt(mean(x^2) + eps) w + b, or nothing.
//
// A row stays in registers between its sums and its outputs: a wavefront a row up to 1024 columns, workgroups of 4 to 16
// wavefronts beyond.  Means and variances are fp32 sums over the registers; the variance is that of the differences from the mean, a
// second pass over registers that costs no memory.
// Bound: memory, 16 bytes a number (x, r, s, h).  12544 x 2048 with two RMS norms, gate, shift and scale: 91 us, 4.5 TB/s; 50000 x 1000 with two layer
// norms 159 us, 5.0 TB/s; 12544 x 512 17.5 us, 5.9 TB/s (partly from the last-level cache).  Rows that are no multiple of four columns (or not
// aligned) are read 4 bytes at a time: 50000 x 1001 351 us.  Rows of 64 columns use 16 of a wavefront's lanes: 400000 x 64 223 us, 1.8 TB/s.
#include <math.h>

#include <algorithm>

#include "common.h"

using namespace eddlhip;

namespace {

typedef float floatx4 __attribute__((ext_vector_type(4)));

struct Norm {
    int kind;
    float eps;
    const float *w, *b;
};
struct NormParams {
    const float *X, *R, *gate, *mod, *shift;
    float *S, *H;
    long long ldx, ldr, lds, ldh;
    long long gate_stride;  // cols where a group of rows has a gate of its own, 0 where all share one
    int rows, cols, group_rows;
    float residual_scale;
    Norm post, pre;
};

template <int THREADS>
__device__ __forceinline__ float row_sum(float x, float *red) {
#pragma unroll
    for (int step = 32; step > 0; step >>= 1) x += __shfl_xor(x, step);
    if constexpr (THREADS > 64) {
        constexpr int WAVES = THREADS / 64;
        __syncthreads();
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
        __syncthreads();
        x = red[0];
#pragma unroll
        for (int w = 1; w < WAVES; w++) x += red[w];
    }
    return x;
}

template <bool VEC>
__device__ __forceinline__ floatx4 get4(const float *p, int c, int cols) {
    if (VEC) return *reinterpret_cast<const floatx4 *>(p + c);
    floatx4 v;
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = c + i < cols ? p[c + i] : 0.0f;
    return v;
}
template <bool VEC>
__device__ __forceinline__ void set4(float *p, int c, int cols, floatx4 v) {
    if (VEC) {
        __builtin_nontemporal_store(v, reinterpret_cast<floatx4 *>(p + c));  // (written once, in whole lines: 12544 x 512 21.8 -> 17.4 us)
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (c + i < cols) p[c + i] = v[i];
    }
}

// x[i] holds the columns 4 (i THREADS + t) ..; zeros behind the last column
template <int THREADS, int NV, bool VEC>
__device__ __forceinline__ void normed(const Norm &n, floatx4 (&x)[NV], int t, int cols, float *red) {
    if (n.kind == EDDLHIP_NORM_NONE) return;
    // (short rows: weight and bias are on their way while the sums are formed)
    constexpr bool AHEAD = THREADS == 64 && NV <= 2;
    floatx4 w[AHEAD ? NV : 1], b[AHEAD ? NV : 1];
    if constexpr (AHEAD) {
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int c = 4 * (i * THREADS + t);
            if (c < cols && n.w) w[i] = get4<VEC>(n.w, c, cols);
            if (c < cols && n.b) b[i] = get4<VEC>(n.b, c, cols);
        }
    }
    float mean = 0.0f;
    if (n.kind == EDDLHIP_NORM_LAYER) {
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; i++) sum += (x[i][0] + x[i][1]) + (x[i][2] + x[i][3]);
        mean = row_sum<THREADS>(sum, red) / (float)cols;
    }
    float squares = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const int c = 4 * (i * THREADS + t);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            x[i][j] = c + j < cols ? x[i][j] - mean : 0.0f;
            squares += x[i][j] * x[i][j];
        }
    }
    const float scale = 1.0f / sqrtf(row_sum<THREADS>(squares, red) / (float)cols + n.eps);
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const int c = 4 * (i * THREADS + t);
        if (c < cols) {
            x[i] *= scale;
            if constexpr (AHEAD) {
                if (n.w) x[i] *= w[i];
                if (n.b) x[i] += b[i];
            } else {
                if (n.w) x[i] *= get4<VEC>(n.w, c, cols);
                if (n.b) x[i] += get4<VEC>(n.b, c, cols);
            }
        }
    }
}

template <int THREADS, int NV, bool VEC>
__global__ __launch_bounds__(THREADS < 256 ? 256 : THREADS) void norm_residual_kernel(const NormParams p) {
    constexpr int PER = THREADS < 256 ? 256 / THREADS : 1;  // rows of a workgroup
    __shared__ float red[16];
    const int t = threadIdx.x % THREADS;
    for (long long row = (long long)blockIdx.x * PER + threadIdx.x / THREADS; row < p.rows; row += (long long)gridDim.x * PER) {
        const long long group = row / p.group_rows;
        floatx4 x[NV];
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int c = 4 * (i * THREADS + t);
            x[i] = c < p.cols ? get4<VEC>(p.X + row * p.ldx, c, p.cols) : floatx4{0.0f, 0.0f, 0.0f, 0.0f};
        }
        // The residual is asked for before the sums that it would wait behind (50000 x 1000, two norms, 217 -> 159 us; 3000 x 8192 91 -> 83;
        // without a norm before it a wavefront's short row is better off with the registers, 12544 x 512 17.5 against 19.4).
        const bool early = p.R && (THREADS > 64 || p.post.kind != EDDLHIP_NORM_NONE);
        floatx4 r[NV];
        if (early) {
#pragma unroll
            for (int i = 0; i < NV; i++) {
                const int c = 4 * (i * THREADS + t);
                r[i] = c < p.cols ? get4<VEC>(p.R + row * p.ldr, c, p.cols) : floatx4{0.0f, 0.0f, 0.0f, 0.0f};
            }
        }
        normed<THREADS, NV, VEC>(p.post, x, t, p.cols, red);
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int c = 4 * (i * THREADS + t);
            if (c < p.cols) {
                if (p.gate) x[i] *= get4<VEC>(p.gate + group * p.gate_stride, c, p.cols);
                if (early) x[i] = r[i] * p.residual_scale + x[i];
                else if (p.R) x[i] = get4<VEC>(p.R + row * p.ldr, c, p.cols) * p.residual_scale + x[i];
                if (p.S) set4<VEC>(p.S + row * p.lds, c, p.cols, x[i]);
            }
        }
        if (p.H) {
            normed<THREADS, NV, VEC>(p.pre, x, t, p.cols, red);
#pragma unroll
            for (int i = 0; i < NV; i++) {
                const int c = 4 * (i * THREADS + t);
                if (c < p.cols) {
                    if (p.mod) x[i] *= 1.0f + get4<VEC>(p.mod + group * p.cols, c, p.cols);
                    if (p.shift) x[i] += get4<VEC>(p.shift + group * p.cols, c, p.cols);
                    set4<VEC>(p.H + row * p.ldh, c, p.cols, x[i]);
                }
            }
        }
    }
}

template <bool VEC>
void launch(const NormParams &p, hipStream_t st) {
    typedef void (*kernel)(NormParams);
    static const struct {
        int threads, nv;
        kernel fn;
    } sizes[] = {{64, 1, norm_residual_kernel<64, 1, VEC>},     {64, 2, norm_residual_kernel<64, 2, VEC>},     {64, 4, norm_residual_kernel<64, 4, VEC>},
                 {256, 2, norm_residual_kernel<256, 2, VEC>},   {512, 2, norm_residual_kernel<512, 2, VEC>},   {1024, 2, norm_residual_kernel<1024, 2, VEC>},
                 {1024, 4, norm_residual_kernel<1024, 4, VEC>}, {1024, 8, norm_residual_kernel<1024, 8, VEC>}};
    int k = 0;
    while (4 * sizes[k].threads * sizes[k].nv < p.cols) k++;
    const int per = sizes[k].threads < 256 ? 256 / sizes[k].threads : 1, threads = std::max(256, sizes[k].threads);
    hipLaunchKernelGGL(sizes[k].fn, dim3(eh_blocks(p.rows, per)), dim3(threads), 0, st, p);
}

constexpr int MAX_COLS = 32768;

}  // namespace

extern "C" int eddlhip_norm_residual(int dev, const float *X, long long ldx, const float *R, long long ldr, float residual_scale, float *S, long long lds, float *H,
                                     long long ldh, int rows, int cols, int post_kind, const float *post_w, const float *post_b, float post_eps,
                                     const float *gate, int gate_groups, int pre_kind, const float *pre_w, const float *pre_b, float pre_eps, const float *mod,
                                     const float *shift, int group_rows) {
    EH_REQUIRE(rows >= 0 && cols > 0 && cols <= MAX_COLS, "norm_residual: %d rows of %d columns (1 to %d)", rows, cols, MAX_COLS);
    for (int kind : {post_kind, pre_kind})
        EH_REQUIRE(kind == EDDLHIP_NORM_NONE || kind == EDDLHIP_NORM_LAYER || kind == EDDLHIP_NORM_RMS, "norm_residual: unknown norm %d", kind);
    EH_REQUIRE(group_rows > 0, "norm_residual: groups of %d rows", group_rows);
    const int groups = rows > 0 ? (rows - 1) / group_rows + 1 : 0;
    EH_REQUIRE(gate == nullptr || gate_groups == 1 || gate_groups >= groups, "norm_residual: gates of %d groups for %d", gate_groups, groups);
    EH_REQUIRE(ldx >= cols && (!R || ldr >= cols) && (!S || lds >= cols) && (!H || ldh >= cols), "norm_residual: rows shorter than %d columns", cols);
    if (rows == 0) return 0;
    EH_REQUIRE(X && (S || H), "norm_residual: NULL tensor");
    EH_REQUIRE(H || (pre_kind == EDDLHIP_NORM_NONE && !mod && !shift), "norm_residual: the norm before the next block has no output");
    for (const float *out : {S, H}) {
        EH_REQUIRE(out != X || (out == S ? lds : ldh) == ldx, "norm_residual: in place, but with rows of another length");
        EH_REQUIRE(!out || out != R || (out == S ? lds : ldh) == ldr, "norm_residual: in place, but with rows of another length");
    }
    for (const float *out : {S, H})
        for (const float *in : {X, R})
            EH_REQUIRE(out == in || !eh_rows_overlap(out, out == S ? lds : ldh, cols, in, in == X ? ldx : ldr, cols, rows), "norm_residual: an output lies on a part of an input");
    EH_REQUIRE(!eh_rows_overlap(S, lds, cols, H, ldh, cols, rows), "norm_residual: the sum and the norm of it share their rows");
    const struct {
        const float *at;
        size_t floats;
    } read[] = {{post_w, (size_t)cols}, {post_b, (size_t)cols},  {pre_w, (size_t)cols}, {pre_b, (size_t)cols},
                {gate, (size_t)(gate_groups == 1 ? 1 : groups) * cols}, {mod, (size_t)groups * cols}, {shift, (size_t)groups * cols}};
    for (const auto &r : read)
        EH_REQUIRE(!eh_rows_meet(S, lds, cols, rows, r.at, r.floats * sizeof(float)) && !eh_rows_meet(H, ldh, cols, rows, r.at, r.floats * sizeof(float)),
                   "norm_residual: an output lies on a weight, bias, gate, mod or shift");
    EH_TRY(use_device(dev));
    NormParams p;
    p.X = X;
    p.R = R;
    p.gate = gate;
    p.mod = mod;
    p.shift = shift;
    p.S = S;
    p.H = H;
    p.ldx = ldx;
    p.ldr = ldr;
    p.lds = lds;
    p.ldh = ldh;
    p.gate_stride = gate_groups == 1 ? 0 : cols;
    p.rows = rows;
    p.cols = cols;
    p.group_rows = group_rows;
    p.residual_scale = residual_scale;
    p.post = Norm{post_kind, post_eps, post_w, post_b};
    p.pre = Norm{pre_kind, pre_eps, pre_w, pre_b};
    uintptr_t bits = 0;
    for (const void *q : {(const void *)X, (const void *)R, (const void *)S, (const void *)H, (const void *)gate, (const void *)mod, (const void *)shift, (const void *)post_w,
                          (const void *)post_b, (const void *)pre_w, (const void *)pre_b})
        bits |= (uintptr_t)q;
    const bool vec = (bits & 15) == 0 && cols % 4 == 0 && ldx % 4 == 0 && (!R || ldr % 4 == 0) && (!S || lds % 4 == 0) && (!H || ldh % 4 == 0);
    if (vec) launch<true>(p, state(dev).stream);
    else launch<false>(p, state(dev).stream);
    EH_CHECK_LAUNCH();
    return 0;
}
