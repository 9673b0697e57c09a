// The short causal convolution of every channel along the tokens of a ragged batch of sequences, whose last inputs lie in slots of a pool.
#include <algorithm>

#include "common.h"
#include "activation.h"
#include "state_batch.h"

using namespace eddlhip;

namespace {

struct ConvParams {
    const float *X, *W, *bias;
    float *Y, *states;
    long long ldx, ldy;
    int channels, chunks, activation;
    StateBatch batch;
};
constexpr int CONV_TOKENS = 16;  // of a thread

// A thread a channel and 16 tokens; the first tokens' thread also reads and writes the state, so that no other thread meets it.
template <int WIDTH>
__global__ __launch_bounds__(256) void causal_conv_kernel(const ConvParams p) {
    const Sequence q = sequence(p.batch, blockIdx.y);
    const int c = blockIdx.x / p.chunks * 256 + threadIdx.x;
    if (c >= p.channels) return;
    float w[WIDTH];
#pragma unroll
    for (int k = 0; k < WIDTH; k++) w[k] = p.W[(long long)c * WIDTH + k];
    const float bias = p.bias ? p.bias[c] : 0.0f;
    for (long long from = blockIdx.x % p.chunks * CONV_TOKENS; from < q.fresh; from += (long long)p.chunks * CONV_TOKENS) {
        const int t0 = (int)from;
        float x[WIDTH];  // the last inputs, the newest behind
#pragma unroll
        for (int k = 0; k < WIDTH - 1; k++) {
            const int t = t0 - (WIDTH - 1) + k;
            x[k + 1] = 0.0f;
            if (t >= 0) x[k + 1] = p.X[q.row(t) * p.ldx + c];
            else if (q.read >= 0) x[k + 1] = p.states[((long long)q.read * (WIDTH - 1) + k) * p.channels + c];
            else if (q.read == -2) x[k + 1] = __builtin_nanf("");
        }
        if (t0 == 0 && q.write >= 0) {
#pragma unroll
            for (int k = 0; k < WIDTH - 1; k++) {
                const int t = q.fresh - (WIDTH - 1) + k;  // of an input that is kept
                float kept = 0.0f;
                if (t >= 0) kept = p.X[q.row(t) * p.ldx + c];
#pragma unroll
                for (int j = 0; j < WIDTH - 1; j++)
                    if (t == j - (WIDTH - 1)) kept = x[j + 1];
                p.states[((long long)q.write * (WIDTH - 1) + k) * p.channels + c] = kept;
            }
        }
        const int end = min(t0 + CONV_TOKENS, q.fresh);
        for (int t = t0; t < end; t++) {
            const long long row = q.row(t);
#pragma unroll
            for (int k = 0; k < WIDTH - 1; k++) x[k] = x[k + 1];
            x[WIDTH - 1] = p.X[row * p.ldx + c];
            float y = bias;
#pragma unroll
            for (int k = 0; k < WIDTH; k++) y = __builtin_fmaf(w[k], x[k], y);
            p.Y[row * p.ldy + c] = activated(y, p.activation);
        }
    }
}

constexpr int MOST_WIDTH = 8;

}  // namespace

extern "C" int eddlhip_causal_conv(int dev, const float *X, long long ldx, const float *W, const float *bias, float *Y, long long ldy, int rows, int channels, int width,
                                   int activation, int reverse, float *states, int pool, const int *offsets, const int *lengths, const int *slots, const int *out_slots,
                                   int seqs, int max_new) {
    EH_REQUIRE(channels > 0 && channels <= MOST_CHANNELS && width >= 2 && width <= MOST_WIDTH, "causal_conv: %d channels (up to %d), a width of %d (2 to %d)", channels, MOST_CHANNELS, width, MOST_WIDTH);
    EH_REQUIRE(activation == EDDLHIP_ACT_NONE || activation == EDDLHIP_ACT_RELU || activation == EDDLHIP_ACT_SILU, "causal_conv: unknown activation %d", activation);
    EH_REQUIRE(ldx >= channels && ldy >= channels, "causal_conv: rows shorter than %d channels", channels);
    EH_TRY(check_batch("causal_conv", rows, seqs, max_new, states, pool, offsets, lengths, slots, out_slots));
    if (rows == 0 || seqs == 0) return 0;
    EH_REQUIRE(X && W && Y, "causal_conv: NULL tensor");
    const struct {
        const void *at;
        size_t bytes;
    } others[] = {{states, (size_t)pool * (width - 1) * channels * 4}, {W, (size_t)channels * width * 4}, {bias, (size_t)channels * 4},
                  {offsets, ((size_t)seqs + 1) * 4}, {lengths, (size_t)seqs * 4}, {slots, (size_t)seqs * 4}, {out_slots, (size_t)seqs * 4}};
    EH_REQUIRE(!eh_rows_overlap(X, ldx, channels, Y, ldy, channels, rows), "causal_conv: the output lies on the input");
    for (const auto &o : others) {
        EH_REQUIRE(!eh_rows_meet(Y, ldy, channels, rows, o.at, o.bytes), "causal_conv: the output lies on the states, weights or the batch");
        EH_REQUIRE(&o == others || !eh_rows_meet((const float *)o.at, o.bytes / 4, o.bytes / 4, 1, states, others[0].bytes), "causal_conv: the states lie on the weights or the batch");
    }
    EH_REQUIRE(!eh_rows_meet(X, ldx, channels, rows, states, others[0].bytes), "causal_conv: the states lie on the input");
    EH_TRY(use_device(dev));
    ConvParams p;
    p.X = X;
    p.W = W;
    p.bias = bias;
    p.Y = Y;
    p.states = states;
    p.ldx = ldx;
    p.ldy = ldy;
    p.channels = channels;
    p.activation = activation;
    p.batch = StateBatch{offsets, lengths, slots, out_slots, rows, pool, reverse != 0};
    typedef void (*kernel)(ConvParams);
    static const kernel kernels[] = {causal_conv_kernel<2>, causal_conv_kernel<3>, causal_conv_kernel<4>, causal_conv_kernel<5>,
                                     causal_conv_kernel<6>, causal_conv_kernel<7>, causal_conv_kernel<8>};
    const int blocks = (channels + 255) / 256;
    p.chunks = std::min((std::max(1, std::min(max_new, rows)) + CONV_TOKENS - 1) / CONV_TOKENS, std::max(1, (1 << 23) / blocks));  // (a grid holds less than 2^32 threads)
    hipLaunchKernelGGL(kernels[width - 2], dim3(blocks * p.chunks, seqs), dim3(256), 0, state(dev).stream, p);
    EH_CHECK_LAUNCH();
    return 0;
}
