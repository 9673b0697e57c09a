// Group norm with its activation: the mean and variance of the channels of a group over all pixels of an image,
//     n = (x - mean) / sqrt(variance + eps) w + b,   y = act(n (1 + mod) + shift).
// Maps [images][channels][pixels], where a group is one stretch of memory, or rows of tokens [images * pixels][channels], where it is a
// piece of every row.
#include <math.h>

#include <algorithm>

#include "common.h"
#include "activation.h"

using namespace eddlhip;

namespace {

struct GroupNormParams {
    const float *X, *w, *b, *mod, *shift;
    float *Y;
    long long ldx, ldy;
    int images, channels, pixels, groups, activation;
    bool rows;
    float eps;
};

template <int THREADS>
__device__ __forceinline__ float block_sum(float x, float *red) {
#pragma unroll
    for (int step = 32; step > 0; step >>= 1) x += __shfl_xor(x, step);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
    __syncthreads();
    x = red[0];
#pragma unroll
    for (int w = 1; w < THREADS / 64; w++) x += red[w];
    return x;
}

// A workgroup a group of an image, three passes over memory.
__global__ __launch_bounds__(256) void group_norm_kernel(const GroupNormParams p) {
    __shared__ float red[4];
    const int per = p.channels / p.groups;
    const long long count = (long long)per * p.pixels;
    for (long long job = blockIdx.x; job < (long long)p.images * p.groups; job += gridDim.x) {
        const int image = (int)(job / p.groups), group = (int)(job % p.groups), c0 = group * per;
        const long long row0 = (long long)image * p.pixels;
        auto at = [&](long long e, long long ld, int &c) -> long long {
            if (p.rows) {
                c = c0 + (int)(e % per);
                return (row0 + e / per) * ld + c;
            }
            c = c0 + (int)(e / p.pixels);
            return ((long long)image * p.channels + c0) * p.pixels + e;
        };
        int c;
        float sum = 0.0f, squares = 0.0f;
        for (long long e = threadIdx.x; e < count; e += 256) sum += p.X[at(e, p.ldx, c)];
        const float mean = block_sum<256>(sum, red) / (float)count;
        for (long long e = threadIdx.x; e < count; e += 256) {
            const float d = p.X[at(e, p.ldx, c)] - mean;
            squares += d * d;
        }
        const float scale = 1.0f / sqrtf(block_sum<256>(squares, red) / (float)count + p.eps);
        for (long long e = threadIdx.x; e < count; e += 256) {
            float v = (p.X[at(e, p.ldx, c)] - mean) * scale;
            if (p.w) v *= p.w[c];
            if (p.b) v += p.b[c];
            if (p.mod) v *= 1.0f + p.mod[(long long)image * p.channels + c];
            if (p.shift) v += p.shift[(long long)image * p.channels + c];
            p.Y[at(e, p.ldy, c)] = activated(v, p.activation);
        }
    }
}

}  // namespace

extern "C" int eddlhip_group_norm(int dev, const float *X, long long ldx, float *Y, long long ldy, int images, int channels, int pixels, int channels_last, int groups,
                                  const float *w, const float *b, float eps, const float *mod, const float *shift, int activation) {
    EH_REQUIRE(images >= 0 && channels > 0 && pixels > 0, "group_norm: %d images of %d channels of %d pixels", images, channels, pixels);
    EH_REQUIRE(groups > 0 && channels % groups == 0, "group_norm: %d channels in %d groups", channels, groups);
    EH_REQUIRE((long long)images * pixels <= 0x7fffffffLL && (long long)images * channels <= 0x7fffffffLL, "group_norm: %d images of %d channels of %d pixels are out of range", images, channels, pixels);
    EH_REQUIRE(activation == EDDLHIP_ACT_NONE || activation == EDDLHIP_ACT_RELU || activation == EDDLHIP_ACT_SILU, "group_norm: unknown activation %d", activation);
    EH_REQUIRE(!channels_last || (ldx >= channels && ldy >= channels), "group_norm: rows shorter than %d channels", channels);
    if (images == 0) return 0;
    EH_REQUIRE(X && Y, "group_norm: NULL tensor");
    // (maps are taken as one row)
    const long long rows = channels_last ? (long long)images * pixels : 1, width = channels_last ? channels : (long long)images * channels * pixels;
    const long long sx = channels_last ? ldx : width, sy = channels_last ? ldy : width;
    EH_REQUIRE(X != Y || sx == sy, "group_norm: in place, but with rows of another length");
    EH_REQUIRE(X == Y || !eh_rows_overlap(X, sx, width, Y, sy, width, rows), "group_norm: the output lies on a part of the input");
    for (const float *read : {w, b})
        EH_REQUIRE(!eh_rows_meet(Y, sy, width, rows, read, (size_t)channels * sizeof(float)), "group_norm: the output lies on a weight, bias, mod or shift");
    for (const float *read : {mod, shift})
        EH_REQUIRE(!eh_rows_meet(Y, sy, width, rows, read, (size_t)images * channels * sizeof(float)), "group_norm: the output lies on a weight, bias, mod or shift");
    EH_TRY(use_device(dev));
    GroupNormParams p;
    p.X = X;
    p.w = w;
    p.b = b;
    p.mod = mod;
    p.shift = shift;
    p.Y = Y;
    p.ldx = ldx;
    p.ldy = ldy;
    p.images = images;
    p.channels = channels;
    p.pixels = pixels;
    p.groups = groups;
    p.activation = activation;
    p.rows = channels_last != 0;
    p.eps = eps;
    hipLaunchKernelGGL(group_norm_kernel, dim3(eh_blocks((size_t)images * groups, 1)), dim3(256), 0, state(dev).stream, p);
    EH_CHECK_LAUNCH();
    return 0;
}
