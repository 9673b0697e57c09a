// Blocks that mix the tokens of a sequence by a state instead of attention: the short causal convolution of every channel and the selective scan
//     d = softplus(dt + dt_bias),   h[c][n] = e^(d A[c][n]) h[c][n] + d x B[n],   y = (sum_n C[n] h[c][n] + skip x) silu(gate),
// token by token, over ragged batches of sequences whose states lie in slots of a pool.
#include <math.h>

#include <algorithm>

#include "common.h"
#include "activation.h"
#include "sequence_rows.h"

using namespace eddlhip;

namespace {

typedef float floatx4 __attribute__((ext_vector_type(4)));

struct Batch {
    const int *offsets, *lengths, *slots, *out_slots;  // the last three where there are states
    int rows, pool;
    bool reverse;
};
// What a workgroup does with its sequence: the rows of its new tokens, the slot that it continues (-1: none, -2: one outside the pool) and the one
// that its state goes to (-1: none).
struct Sequence {
    int row0, fresh, read, write;
    int step;  // from a token's row to the next one's

    __device__ __forceinline__ int row(int token) const { return step > 0 ? row0 + token : row0 + fresh - 1 - token; }
};
__device__ __forceinline__ Sequence sequence(const Batch &b, int s) {
    const SequenceRows r = sequence_rows(b.offsets[s], b.offsets[s + 1], b.rows);
    Sequence q{r.row0, r.fresh, -1, -1, b.reverse ? -1 : 1};
    if (b.pool > 0) {
        const int read = b.slots[s], write = b.out_slots[s];
        if (b.lengths[s] > r.fresh) q.read = (unsigned)read < (unsigned)b.pool ? read : -2;
        if ((unsigned)write < (unsigned)b.pool) q.write = write;
    }
    return q;
}

// ------------------------------------------------------------------------------------------------- the convolution
struct ConvParams {
    const float *X, *W, *bias;
    float *Y, *states;
    long long ldx, ldy;
    int channels, chunks, activation;
    Batch batch;
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
    for (int t0 = blockIdx.x % p.chunks * CONV_TOKENS; t0 < q.fresh; t0 += p.chunks * CONV_TOKENS) {
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

// ------------------------------------------------------------------------------------------------- the scan
struct ScanParams {
    const float *X, *dt, *gate, *B, *C, *A, *skip, *dt_bias;
    float *Y, *states;
    long long ldx, lddt, ldg, ldb, ldc, ldy;
    int channels, n, per;  // channels that share B and C
    bool softplus;
    Batch batch;
};

// LANES lanes a channel, NL states each; token after token from memory.
template <int LANES, int NL>
__global__ __launch_bounds__(256) void scan_tokens_kernel(const ScanParams p) {
    const Sequence q = sequence(p.batch, blockIdx.y);
    const int c = blockIdx.x * (256 / LANES) + threadIdx.x / LANES, lane = threadIdx.x % LANES, n0 = lane * NL;
    if (q.fresh == 0 || c >= p.channels) return;
    float a[NL], h[NL];
    bool has[NL];
#pragma unroll
    for (int i = 0; i < NL; i++) {
        has[i] = n0 + i < p.n;
        a[i] = has[i] ? p.A[(long long)c * p.n + n0 + i] * LOG2_E : 0.0f;
        h[i] = 0.0f;
        if (q.read >= 0 && has[i]) h[i] = p.states[((long long)q.read * p.channels + c) * p.n + n0 + i];
        if (q.read == -2) h[i] = __builtin_nanf("");
    }
    const float bias = p.dt_bias ? p.dt_bias[c] : 0.0f, skip = p.skip ? p.skip[c] : 0.0f;
    const int v0 = c / p.per * p.n + n0;
    for (int t = 0; t < q.fresh; t++) {
        const long long row = q.row(t);
        const float raw = p.dt[row * p.lddt + c] + bias, d = p.softplus ? softplus(raw) : raw, x = p.X[row * p.ldx + c], dx = d * x;
        float y = 0.0f;
#pragma unroll
        for (int i = 0; i < NL; i++) {
            const float b = has[i] ? p.B[row * p.ldb + v0 + i] : 0.0f, cc = has[i] ? p.C[row * p.ldc + v0 + i] : 0.0f;
            h[i] = __builtin_fmaf(__builtin_amdgcn_exp2f(d * a[i]), h[i], dx * b);
            y = __builtin_fmaf(cc, h[i], y);
        }
#pragma unroll
        for (int step = 1; step < LANES; step <<= 1) y += __shfl_xor(y, step);
        if (lane == 0) {
            if (p.skip) y = __builtin_fmaf(skip, x, y);
            if (p.gate) y *= silu(p.gate[row * p.ldg + c]);
            p.Y[row * p.ldy + c] = y;
        }
    }
    if (q.write >= 0) {
#pragma unroll
        for (int i = 0; i < NL; i++)
            if (has[i]) p.states[((long long)q.write * p.channels + c) * p.n + n0 + i] = h[i];
    }
}

constexpr int MOST_STATES = 64, MOST_WIDTH = 8;

// What both entry points ask of a batch; `name` opens the error's text.
int check_batch(const char *name, int rows, int seqs, int max_new, const float *states, int pool, const int *offsets, const int *lengths, const int *slots, const int *out_slots) {
    EH_REQUIRE(rows >= 0 && seqs >= 0 && seqs <= 65535, "%s: %d rows of %d sequences (at most 65535)", name, rows, seqs);
    EH_REQUIRE(max_new >= 0 && pool >= 0 && (states != nullptr) == (pool > 0), "%s: max_new %d, a pool of %d states%s", name, max_new, pool, states ? "" : " at NULL");
    if (rows == 0 || seqs == 0) return 0;
    EH_REQUIRE(offsets && (!states || (lengths && slots && out_slots)), "%s: NULL offsets, lengths or slots", name);
    return 0;
}

}  // namespace

extern "C" int eddlhip_causal_conv(int dev, const float *X, long long ldx, const float *W, const float *bias, float *Y, long long ldy, int rows, int channels, int width,
                                   int activation, int reverse, float *states, int pool, const int *offsets, const int *lengths, const int *slots, const int *out_slots,
                                   int seqs, int max_new) {
    EH_REQUIRE(channels > 0 && width >= 2 && width <= MOST_WIDTH, "causal_conv: %d channels, a width of %d (2 to %d)", channels, width, MOST_WIDTH);
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
    p.batch = Batch{offsets, lengths, slots, out_slots, rows, pool, reverse != 0};
    typedef void (*kernel)(ConvParams);
    static const kernel kernels[] = {causal_conv_kernel<2>, causal_conv_kernel<3>, causal_conv_kernel<4>, causal_conv_kernel<5>,
                                     causal_conv_kernel<6>, causal_conv_kernel<7>, causal_conv_kernel<8>};
    const int blocks = (channels + 255) / 256;
    p.chunks = std::min((std::max(1, std::min(max_new, rows)) + CONV_TOKENS - 1) / CONV_TOKENS, 0x7fffffff / blocks);
    hipLaunchKernelGGL(kernels[width - 2], dim3(blocks * p.chunks, seqs), dim3(256), 0, state(dev).stream, p);
    EH_CHECK_LAUNCH();
    return 0;
}

extern "C" int eddlhip_selective_scan(int dev, const float *X, long long ldx, const float *dt, long long lddt, const float *A, const float *B, long long ldb,
                                      const float *C, long long ldc, const float *skip, const float *gate, long long ldg, const float *dt_bias, float *Y, long long ldy,
                                      int rows, int channels, int n, int groups, int softplus, int reverse, float *states, int pool, const int *offsets,
                                      const int *lengths, const int *slots, const int *out_slots, int seqs, int max_new) {
    EH_REQUIRE(channels > 0 && n > 0 && n <= MOST_STATES, "selective_scan: %d channels of %d states (1 to %d)", channels, n, MOST_STATES);
    EH_REQUIRE(groups > 0 && channels % groups == 0, "selective_scan: %d channels in %d groups", channels, groups);
    EH_REQUIRE(ldx >= channels && lddt >= channels && ldy >= channels && (!gate || ldg >= channels), "selective_scan: rows shorter than %d channels", channels);
    EH_REQUIRE(ldb >= (long long)groups * n && ldc >= (long long)groups * n, "selective_scan: rows shorter than %d vectors of %d", groups, n);
    EH_TRY(check_batch("selective_scan", rows, seqs, max_new, states, pool, offsets, lengths, slots, out_slots));
    if (rows == 0 || seqs == 0) return 0;
    EH_REQUIRE(X && dt && A && B && C && Y, "selective_scan: NULL tensor");
    const size_t state_bytes = (size_t)pool * channels * n * 4;
    const struct {
        const float *at;
        long long ld, width;
    } inputs[] = {{X, ldx, channels}, {dt, lddt, channels}, {gate, ldg, channels}, {B, ldb, (long long)groups * n}, {C, ldc, (long long)groups * n}};
    for (const auto &i : inputs) {
        EH_REQUIRE(!eh_rows_overlap(i.at, i.ld, i.width, Y, ldy, channels, rows), "selective_scan: the output lies on an input");
        EH_REQUIRE(!eh_rows_meet(i.at, i.ld, i.width, rows, states, state_bytes), "selective_scan: the states lie on an input");
    }
    const struct {
        const void *at;
        size_t bytes;
    } others[] = {{states, state_bytes}, {A, (size_t)channels * n * 4}, {skip, (size_t)channels * 4}, {dt_bias, (size_t)channels * 4},
                  {offsets, ((size_t)seqs + 1) * 4}, {lengths, (size_t)seqs * 4}, {slots, (size_t)seqs * 4}, {out_slots, (size_t)seqs * 4}};
    for (const auto &o : others) {
        EH_REQUIRE(!eh_rows_meet(Y, ldy, channels, rows, o.at, o.bytes), "selective_scan: the output lies on the states, weights or the batch");
        EH_REQUIRE(&o == others || !eh_rows_meet((const float *)o.at, o.bytes / 4, o.bytes / 4, 1, states, state_bytes), "selective_scan: the states lie on the weights or the batch");
    }
    EH_TRY(use_device(dev));
    ScanParams p;
    p.X = X;
    p.dt = dt;
    p.gate = gate;
    p.B = B;
    p.C = C;
    p.A = A;
    p.skip = skip;
    p.dt_bias = dt_bias;
    p.Y = Y;
    p.states = states;
    p.ldx = ldx;
    p.lddt = lddt;
    p.ldg = ldg;
    p.ldb = ldb;
    p.ldc = ldc;
    p.ldy = ldy;
    p.channels = channels;
    p.n = n;
    p.per = channels / groups;
    p.softplus = softplus != 0;
    p.batch = Batch{offsets, lengths, slots, out_slots, rows, pool, reverse != 0};
    typedef void (*kernel)(ScanParams);
    static const struct {
        int lanes, nl;
        kernel fn;
    } sizes[] = {{1, 1, scan_tokens_kernel<1, 1>}, {1, 4, scan_tokens_kernel<1, 4>}, {2, 4, scan_tokens_kernel<2, 4>}, {4, 4, scan_tokens_kernel<4, 4>},
                 {8, 4, scan_tokens_kernel<8, 4>}, {16, 4, scan_tokens_kernel<16, 4>}};
    int k = 0;
    while (sizes[k].lanes * sizes[k].nl < n) k++;
    hipLaunchKernelGGL(sizes[k].fn, dim3((unsigned)(((long long)channels * sizes[k].lanes + 255) / 256), seqs), dim3(256), 0, state(dev).stream, p);
    EH_CHECK_LAUNCH();
    return 0;
}
