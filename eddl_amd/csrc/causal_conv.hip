// The short causal convolution of every channel along the tokens of a ragged batch of sequences, whose last inputs lie in slots of a pool:
//     Y[t][c] = act(bias[c] + sum_k W[c][k] x[t - width + 1 + k][c]).
// Bound: memory, 8 bytes a number.  A thread keeps its channels' weights and walks along the tokens, so that an input is read from memory once and the width - 1 rows
// that two threads share come from the L2.  Eight ragged sequences of up to 2048 tokens of 2048 channels: 20 us for 86 MB, 4.3 TB/s; 32 single tokens 4.6 us in
// the kernel, a chain of the batch's numbers, weights and states.
#include <algorithm>

#include "common.h"
#include "activation.h"
#include "state_batch.h"
#include "xcd.h"

using namespace eddlhip;

namespace {

typedef float floatx4 __attribute__((ext_vector_type(4), aligned(4)));  // (the hardware reads and writes 16 bytes at any multiple of four)

struct ConvParams {
    const float *X, *W, *bias;
    float *Y, *states;
    long long ldx, ldy;
    long long jobs;
    int channels, activation;
    unsigned blocks, chunks;
    StateBatch batch;
};
constexpr int CONV_TOKENS = 8;  // of a thread (us at 4, 8, 16, 32: 4096 tokens of 4096 channels 36, 38, 39, 35; 64 x 196 of 768 18, 20, 25, 25; 16 x 2048 of 2048 120, 114, 120, 135)

template <int UNIT>
struct Unit {
    float v[UNIT];
};
template <int UNIT>
__device__ __forceinline__ Unit<UNIT> get(const float *from) {
    Unit<UNIT> u;
    if constexpr (UNIT == 4) {
        const floatx4 v = *reinterpret_cast<const floatx4 *>(from);
#pragma unroll
        for (int i = 0; i < 4; i++) u.v[i] = v[i];
    } else {
        u.v[0] = *from;
    }
    return u;
}
// Outputs are written past the caches (4096 tokens of 4096 channels 38 -> 30 us; rows that begin inside a line too: 16 x 2048 of 2044 channels 114 -> 109).
template <int UNIT>
__device__ __forceinline__ void set(float *to, const Unit<UNIT> &u) {
    if constexpr (UNIT == 4) __builtin_nontemporal_store(floatx4{u.v[0], u.v[1], u.v[2], u.v[3]}, reinterpret_cast<floatx4 *>(to));
    else *to = u.v[0];
}

// UNIT channels of a sequence from c on, of eight tokens, all of whose inputs are asked for at once; the first tokens' thread also reads and writes the
// state, so that no other thread meets it.
template <int WIDTH, int UNIT>
__device__ __forceinline__ void convolve(const ConvParams &p, const Sequence &q, int c, long long from) {
    static_assert(CONV_TOKENS >= WIDTH - 1, "inputs of the state reach the first chunk only");
    Unit<UNIT> w[WIDTH], bias;  // w[k].v[i]: number i * WIDTH + k of the channels' weights
    {
        Unit<UNIT> in[WIDTH];
#pragma unroll
        for (int k = 0; k < WIDTH; k++) in[k] = get<UNIT>(p.W + (long long)c * WIDTH + k * UNIT);
#pragma unroll
        for (int k = 0; k < WIDTH; k++)
#pragma unroll
            for (int i = 0; i < UNIT; i++) w[k].v[i] = in[(i * WIDTH + k) / UNIT].v[(i * WIDTH + k) % UNIT];
#pragma unroll
        for (int i = 0; i < UNIT; i++) bias.v[i] = 0.0f;
        if (p.bias) bias = get<UNIT>(p.bias + c);
    }
    for (; from < q.fresh; from += (long long)p.chunks * CONV_TOKENS) {
        const int t0 = (int)from;
        Unit<UNIT> x[WIDTH - 1 + CONV_TOKENS];  // x[k]: the input of token t0 - (WIDTH - 1) + k
#pragma unroll
        for (int k = 0; k < WIDTH - 1 + CONV_TOKENS; k++) {
            const int t = t0 - (WIDTH - 1) + k;
#pragma unroll
            for (int i = 0; i < UNIT; i++) x[k].v[i] = k < WIDTH - 1 && t < 0 && q.read == -2 ? __builtin_nanf("") : 0.0f;
            if (k >= WIDTH - 1 ? t < q.fresh : t >= 0) x[k] = get<UNIT>(p.X + q.row(t) * p.ldx + c);
            else if (k < WIDTH - 1 && q.read >= 0) x[k] = get<UNIT>(p.states + ((long long)q.read * (WIDTH - 1) + k) * p.channels + c);
        }
        if (t0 == 0 && q.write >= 0) {
#pragma unroll
            for (int k = 0; k < WIDTH - 1; k++) {
                const int t = q.fresh - (WIDTH - 1) + k;  // of an input that is kept
                Unit<UNIT> kept;
                if (t >= 0) {
                    kept = get<UNIT>(p.X + q.row(t) * p.ldx + c);
                } else {
#pragma unroll
                    for (int j = 0; j < WIDTH - 1; j++)
                        if (t == j - (WIDTH - 1)) kept = x[j];
                }
                set<UNIT>(p.states + ((long long)q.write * (WIDTH - 1) + k) * p.channels + c, kept);
            }
        }
#pragma unroll
        for (int j = 0; j < CONV_TOKENS; j++) {
            if (t0 + j < q.fresh) {
                Unit<UNIT> y = bias;
#pragma unroll
                for (int i = 0; i < UNIT; i++) {
#pragma unroll
                    for (int k = 0; k < WIDTH; k++) y.v[i] = __builtin_fmaf(w[k].v[i], x[j + k].v[i], y.v[i]);
                    y.v[i] = activated(y.v[i], p.activation);
                }
                set<UNIT>(p.Y + q.row(t0 + j) * p.ldy + c, y);
            }
        }
    }
}

// Four channels a thread; those behind the last four one a thread (16 sequences of 2048 tokens of 2046 channels, us: all one a thread 151, so 117).
template <int WIDTH>
__global__ __launch_bounds__(256) void causal_conv_kernel(const ConvParams p) {
    // (neighbours in time share width - 1 rows)
    for (long long id = blockIdx.x; id < xcd_padded(p.jobs); id += gridDim.x) {
        const long long job = xcd_job<true>(id);
        if (job >= p.jobs) continue;
        const unsigned chunk = (unsigned)job % p.chunks, rest = (unsigned)job / p.chunks;  // (fewer than 2^31 jobs)
        const Sequence q = sequence(p.batch, rest / p.blocks);
        const int unit = rest % p.blocks * 256 + threadIdx.x, units = p.channels / 4, single = unit - (units + 63) / 64 * 64;  // (those one a thread are in a wavefront of their own)
        const long long from = (long long)chunk * CONV_TOKENS;
        if (from >= q.fresh) continue;
        if (unit < units) convolve<WIDTH, 4>(p, q, unit * 4, from);
        else if (single >= 0 && single < p.channels % 4) convolve<WIDTH, 1>(p, q, units * 4 + single, from);
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
    static const kernel kernels[MOST_WIDTH - 1] = {causal_conv_kernel<2>, causal_conv_kernel<3>, causal_conv_kernel<4>, causal_conv_kernel<5>,
                                                   causal_conv_kernel<6>, causal_conv_kernel<7>, causal_conv_kernel<8>};
    p.blocks = ((channels / 4 + 63) / 64 * 64 + channels % 4 + 255) / 256;
    // Chunks of the longest sequence that the host allows, as far as the rows are worth it: a thread walks the chunks beyond, and workgroups without tokens cost time too
    // (2048 sequences of 3 tokens of 1024 channels, 8192 allowed: all chunks 1325 us, so 57).
    const long long each = (long long)p.blocks * seqs, chunks = (std::max(1, std::min(max_new, rows)) + CONV_TOKENS - 1) / CONV_TOKENS;
    p.chunks = (unsigned)std::min(chunks, std::max(1LL, std::max(32768LL, (long long)rows * p.blocks) / each));
    p.jobs = (long long)p.blocks * p.chunks * seqs;
    hipLaunchKernelGGL(kernels[width - 2], dim3(xcd_grid(p.jobs, 256)), dim3(256), 0, state(dev).stream, p);
    EH_CHECK_LAUNCH();
    return 0;
}
