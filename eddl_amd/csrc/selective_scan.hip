// The selective scan
//     d = softplus(dt + dt_bias),   h[c][n] = e^(d A[c][n]) h[c][n] + d x B[n],   y = (sum_n C[n] h[c][n] + skip x) silu(gate),
// token by token, over ragged batches of sequences whose states lie in slots of a pool.
//
// A token after the other is a chain of one multiplication and addition a state, so what a device can do at once are sequences, channels and states; tokens only
// because runs of them compose: a run takes h to F h + H, F the product of its factors (one exponential of the summed steps), H its state from zeros.  Where channels
// and sequences do not fill the device, wavefronts take runs of tokens and pass states on, and long sequences take two launches.
//
// Bound: memory where the tokens are few (a single token reads and writes its channel's state: 128 sequences of 4096 channels of 16 states 15 us, 4.5 TB/s).  Along
// many tokens 16 bytes of memory stand beside n exponentials and four more instructions a state: with 16 states the vector instructions bind (cycles of a SIMD
// an instruction, measured: exponential 8.3; other fp32 ones 2.5 to 3 with eight wavefronts of a SIMD, 3 to 4 with four; 4.8 with a DPP operand).  64 sequences of 196 tokens of 768
// channels: 53 us (2.9 TB/s); a vector instruction is at work in 70 % of the cycles, 22 of 35 of them for the states, the others for softplus, silu and places in LDS.
// Rounding: fp32 throughout; 1e-7 of the outputs against 64 bits (2-norm), where the products of a long run take the rounding of one exponential instead of hundreds.
#include <limits.h>

#include <algorithm>

#include "common.h"
#include "activation.h"
#include "state_batch.h"
#include "xcd.h"

using namespace eddlhip;

namespace {

typedef float floatx4 __attribute__((ext_vector_type(4)));

struct ScanParams {
    const float *X, *dt, *gate, *B, *C, *A, *skip, *dt_bias;
    float *Y, *states;
    float *part_states, *part_exponents;  // [sequence][the state that it continues, parts, pieces of them][channel][NP], [sequence][parts, pieces][channel][NP]: half the exponents
    long long ldx, lddt, ldg, ldb, ldc, ldy;
    int channels, n, per;  // channels that share B and C
    unsigned blocks, group_blocks, parts;
    long long jobs;
    const int *list;  // tiles: the sequences that are meant (-1: none), or NULL: all of up to `most` new tokens
    int most;
    bool softplus;
    StateBatch batch;
};

// Sums over LANES lanes side by side, in all of them.
template <int CTRL>
__device__ __forceinline__ float swapped(float x) {
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}
template <int LANES>
__device__ __forceinline__ float lane_sum(float x) {
    if constexpr (LANES >= 2) x += swapped<0xB1>(x);    // the neighbour
    if constexpr (LANES >= 4) x += swapped<0x4E>(x);    // the other pair of four
    if constexpr (LANES >= 8) x += swapped<0x141>(x);   // the other four of eight, mirrored
    if constexpr (LANES >= 16) x += swapped<0x140>(x);  // the other eight of sixteen, mirrored
    return x;
}

// NL numbers from n0 of n on; 0 behind the last.  The hardware reads 16 bytes from any multiple of four.  WHOLE: n is a multiple of NL.
template <int NL, bool WHOLE>
__device__ __forceinline__ void get(const float *from, int n0, int n, float (&v)[NL]) {
    typedef float vec __attribute__((ext_vector_type(NL), aligned(4)));
    if (WHOLE || n0 + NL <= n) {
        vec u;
#pragma unroll
        for (int i = 0; i < NL; i++) u[i] = 0.0f;
        if (!WHOLE || n0 < n) u = *reinterpret_cast<const vec *>(from + n0);
#pragma unroll
        for (int i = 0; i < NL; i++) v[i] = u[i];
    } else {
#pragma unroll
        for (int i = 0; i < NL; i++) v[i] = n0 + i < n ? from[n0 + i] : 0.0f;
    }
}
// The NL states of channel c from n0 on: as the sequence finds them, and on their way to the pool; the factors of the steps in powers of two.
template <int NL, bool WHOLE>
__device__ __forceinline__ void first_state(const ScanParams &p, const Sequence &q, int c, int n0, float (&h)[NL]) {
#pragma unroll
    for (int i = 0; i < NL; i++) h[i] = q.read == -2 ? __builtin_nanf("") : 0.0f;
    if (q.read >= 0) get<NL, WHOLE>(p.states + ((long long)q.read * p.channels + c) * p.n, n0, p.n, h);
}
template <int NL>
__device__ __forceinline__ void keep_state(const ScanParams &p, const Sequence &q, int c, int n0, const float (&h)[NL]) {
    typedef float vec __attribute__((ext_vector_type(NL), aligned(4)));
    if (q.write < 0) return;
    float *to = p.states + ((long long)q.write * p.channels + c) * p.n + n0;
    if (n0 + NL <= p.n) {
        vec u;
#pragma unroll
        for (int i = 0; i < NL; i++) u[i] = h[i];
        *reinterpret_cast<vec *>(to) = u;
    } else {
#pragma unroll
        for (int i = 0; i < NL; i++)
            if (n0 + i < p.n) to[i] = h[i];
    }
}
template <int NL, bool WHOLE>
__device__ __forceinline__ void exponents(const ScanParams &p, int c, int n0, float (&a)[NL]) {
    constexpr float MOST = 3.40282347e38f;
    get<NL, WHOLE>(p.A + (long long)c * p.n, n0, p.n, a);
#pragma unroll
    for (int i = 0; i < NL; i++) {
        a[i] *= LOG2_E;
        a[i] = a[i] > MOST ? MOST : a[i] < -MOST ? -MOST : a[i];  // (an infinite one would make NaN of the steps of 0 behind the last token)
    }
}

// A run of tokens is joined to a state by its factor 2^l, which passes the largest number where the run's steps grow, though no token's does: times a state of zeros it would be NaN,
// and whether a batch's tokens are joined in runs is not the formula's.  So the state is multiplied by the root 2^(l/2) twice: 0 stays 0, and past 2^254 any other is
// infinite (those below the normal numbers aside).  Sums of steps stay finite, so that A of 0 has l = 0.  (The factor itself would be cheaper: 8192 tokens of 4096 channels
// 215 us, by roots 221; 4102 tokens of 128 channels 24.7 and 25.0.)
__device__ __forceinline__ float within(float steps) { return __builtin_amdgcn_fmed3f(steps, -3.40282347e38f, 3.40282347e38f); }
__device__ __forceinline__ float run_root(float half_exponent) { return __builtin_amdgcn_exp2f(__builtin_amdgcn_fmed3f(half_exponent, -150.0f, 127.0f)); }
__device__ __forceinline__ float behind_run(float root, float h, float brought) { return __builtin_fmaf(root * h, root, brought); }

// Few tokens a sequence: LANES lanes a channel, NL states each; token after token from memory.  WHOLE: loads that no branch
// parts (128 sequences of 4096 channels 17.3 -> 16.1 us).
template <int LANES, int NL, bool WHOLE>
__global__ __launch_bounds__(256) void scan_tokens_kernel(const ScanParams p) {
    const Sequence q = sequence(p.batch, blockIdx.y);
    const int c = blockIdx.x * (256 / LANES) + threadIdx.x / LANES, lane = threadIdx.x % LANES, n0 = lane * NL;
    if (q.fresh == 0 || c >= p.channels) return;
    float a[NL], h[NL];
    first_state<NL, WHOLE>(p, q, c, n0, h);
    exponents<NL, WHOLE>(p, c, n0, a);
    const float bias = p.dt_bias ? p.dt_bias[c] : 0.0f, skip = p.skip ? p.skip[c] : 0.0f;
    const int v0 = c / p.per * p.n;
    for (int t = 0; t < q.fresh; t++) {
        const long long row = q.row(t);
        float b[NL], cc[NL];
        get<NL, WHOLE>(p.B + row * p.ldb + v0, n0, p.n, b);
        get<NL, WHOLE>(p.C + row * p.ldc + v0, n0, p.n, cc);
        const float raw = p.dt[row * p.lddt + c] + bias, x = p.X[row * p.ldx + c], g = p.gate ? p.gate[row * p.ldg + c] : 0.0f;
        const float d = p.softplus ? softplus(raw) : raw, dx = d * x;
        float y = 0.0f;
#pragma unroll
        for (int i = 0; i < NL; i++) {
            h[i] = __builtin_fmaf(__builtin_amdgcn_exp2f(d * a[i]), h[i], dx * b[i]);
            y = __builtin_fmaf(cc[i], h[i], y);
        }
        y = lane_sum<LANES>(y);
        if (lane == 0) {
            y = __builtin_fmaf(skip, x, y);
            if (p.gate) y *= silu(g);
            p.Y[row * p.ldy + c] = y;
        }
    }
    keep_state<NL>(p, q, c, n0, h);
}

// Many tokens.  A wavefront lays a tile of its tokens and channels out in LDS of its own - steps d, products d x, vectors B and C - and walks it with LANES
// lanes a channel, NL states each; nothing but a wavefront's own order of instructions stands between the two.  WT of a workgroup's WAVES wavefronts divide
// the tokens of the same channels: each first brings its tokens' state from zeros, keeping factors e^(d A) and products d x B in registers, then takes
// in what the wavefronts before it brought, and walks its tokens again with the state that they begin with.  The others have channels of their own.
template <int LANES, int NL, int WAVES, int WT>
struct ScanTile {
    static constexpr int THREADS = 64 * WAVES;
    static constexpr int TT = LANES >= 4 ? 16 : 8;         // tokens of a wavefront
    static constexpr int TOKENS = TT * WT;                 // of a workgroup at a time
    static constexpr int CH = 64 / LANES;                  // channels of a wavefront
    static constexpr int CHANNELS = CH * (WAVES / WT);     // of a workgroup
    static constexpr int NP = LANES * NL;                  // states, with those behind the last
    static constexpr int STRIDE = TT + 4;                  // floats from a channel's steps to the next one's (16 bytes of neighbours lie in banks of their own)
    static constexpr int U = TT / LANES < 4 ? TT / LANES : 4;  // a lane brings numbers of U channels side by side
    static constexpr int CQ = CH / U;
    static constexpr int PER = TT * CQ / 64;
    static constexpr int VECTORS = TT * LANES;             // pieces of NL numbers of B or C
    static constexpr int VPER = (VECTORS + 63) / 64;
};
// What a wavefront's lanes wrote to LDS before is what they read behind: the hardware keeps the order, the compiler has to.
__device__ __forceinline__ void in_order() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// The sequences of `least` new tokens or more, one after another, and -1 behind them, `count` numbers in all.
constexpr int LIST_THREADS = 1024;
__global__ __launch_bounds__(LIST_THREADS) void list_sequences_kernel(const StateBatch batch, int seqs, int least, int *list, int count) {
    __shared__ int found[LIST_THREADS / 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int before = 0;
    for (int first = 0; first < seqs; first += LIST_THREADS) {
        const int s = first + (int)threadIdx.x;
        const bool is = s < seqs && sequence_rows(batch.offsets[s], batch.offsets[s + 1], batch.rows).fresh >= least;
        const unsigned long long all = __ballot(is);
        __syncthreads();
        if (lane == 0) found[wave] = __popcll(all);
        __syncthreads();
        int at = before + __popcll(all & ((1ull << lane) - 1));
        for (int w = 0; w < LIST_THREADS / 64; w++) {
            if (w < wave) at += found[w];
            before += found[w];
        }
        if (is && at < count) list[at] = s;
    }
    for (int k = before + (int)threadIdx.x; k < count; k += LIST_THREADS) list[k] = -1;
}

// PART 0: the whole scan of a sequence.  A long one that would leave the device empty is divided over workgroups, and a workgroup's part over its wavefronts, which
// walk their pieces on their own: PART 1 brings the state of every piece and part from zeros and the factor of what comes before it, PART 2 takes in what lies
// before its own and brings the outputs.
template <int LANES, int NL, int WAVES, int WT, int PART>
__global__ __launch_bounds__(64 * WAVES, WT > 1 || LANES == 1 || (PART == 2 && LANES == 16) ? 2 : 4) void scan_tile_kernel(const ScanParams p) {
    using T = ScanTile<LANES, NL, WAVES, WT>;
    constexpr int U = T::U;
    typedef float vec __attribute__((ext_vector_type(NL)));
    typedef float unit __attribute__((ext_vector_type(U)));
    typedef float loose_unit __attribute__((ext_vector_type(U), aligned(4)));
    typedef float loose_vec __attribute__((ext_vector_type(NL), aligned(4)));
    static_assert(PART == 0 || WT == 1, "pieces of a part are walked on their own");
    constexpr int SETS = 64 * (WAVES / WT);  // lanes that walk the same tokens
    constexpr int PIECES = PART ? WAVES : 1;
    __shared__ __attribute__((aligned(16))) float all_steps[WAVES][T::CH * T::STRIDE], all_inputs[WAVES][T::CH * T::STRIDE];  // d and d x, whose place the outputs take
    __shared__ __attribute__((aligned(16))) vec all_b[WAVES][T::VECTORS], all_c[WAVES][PART == 1 ? 1 : T::VECTORS];
    // (two of each: a wavefront may be a tile ahead of the slowest one)
    __shared__ __attribute__((aligned(16))) vec brought[WT > 1 || PART == 2 ? 2 * T::THREADS : PART ? T::THREADS : 1],
        factor[WT > 1 || PART == 2 ? 2 * T::THREADS : PART ? T::THREADS : 1], begin[WT > 1 ? 2 * SETS : 1];
    __shared__ float halves[PART == 1 ? T::THREADS : 1];

    // (workgroups side by side in channels share lines of memory, and B and C)
    for (long long id = blockIdx.x; id < xcd_padded(p.jobs); id += gridDim.x) {
        const long long job = xcd_job(id);
        if (job >= p.jobs) continue;
        const unsigned rest = (unsigned)job / p.blocks;  // (fewer than 2^31 jobs)
        const int block = (unsigned)job % p.blocks, group = block / p.group_blocks, part = rest % p.parts, place = rest / p.parts;
        const int s = p.list ? p.list[place] : place;
        if (s < 0) continue;
        const Sequence q = sequence(p.batch, s);
        const int tiles = (int)(((long long)q.fresh + T::TOKENS - 1) / T::TOKENS), share = (tiles + (int)p.parts * PIECES - 1) / ((int)p.parts * PIECES);  // (of a piece)
        if (part * PIECES * share >= tiles || q.fresh > p.most) continue;

        const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), wt = wave % WT, wc = PART ? 0 : wave / WT, set = wc * 64 + lane;
        const int tile0 = PART ? min(tiles, (part * PIECES + wave) * share) : 0, tile1 = PART ? min(tiles, tile0 + share) : tiles;
        const int c0 = group * p.per + (int)(block % p.group_blocks) * (PART ? T::CH : T::CHANNELS) + wc * T::CH, cend = (group + 1) * p.per;  // the wavefront's first channel
        const int ch = lane / LANES, c = c0 + ch, ln = lane % LANES, n0 = ln * NL;
        const bool mine = c < cend;

        float a[NL], h[NL], through = 0.0f, through_low = 0.0f;  // (through: the steps of all tokens of a piece, and what their sum lost to rounding)
#pragma unroll
        for (int i = 0; i < NL; i++) a[i] = h[i] = 0.0f;
        if (mine) exponents<NL, false>(p, c, n0, a);
        // What a lane brings of a tile, one tile ahead.  Its places are pointers that go on by a tile's rows.
        unit x[T::PER], d[T::PER], g[T::PER];
        vec b[T::VPER], cc[T::VPER];
        const int tq = lane / T::CQ, at = lane % T::CQ * U, tv = lane / LANES, av = lane % LANES * NL;  // token and first channel, or state
        const int dir = p.batch.reverse ? -1 : 1, t0 = wt * T::TT;
        const long long row = q.row(tile0 * T::TOKENS + t0 + tq), vrow = q.row(tile0 * T::TOKENS + t0 + tv);
        const float *px = p.X + row * p.ldx + c0 + at, *pd = p.dt + row * p.lddt + c0 + at, *pg = p.gate + row * p.ldg + c0 + at;
        const float *pb = p.B + vrow * p.ldb + (long long)group * p.n + av, *pc = p.C + vrow * p.ldc + (long long)group * p.n + av;
        float *py = p.Y + row * p.ldy + c0 + at;
        const long long mx = dir * p.ldx, md = dir * p.lddt, mg = dir * p.ldg, my = dir * p.ldy, mb = dir * p.ldb, mc = dir * p.ldc;
        constexpr int APART = 64 / T::CQ, VAPART = 64 / LANES;  // tokens between a lane's pieces
        const bool has = c0 + at < cend, hasv = av < p.n, wholev = av + NL <= p.n;
        const bool whole = c0 + at + U <= cend;  // (wherever rows begin, since 16 bytes are read from any multiple of four: 7 ragged sequences of 1002 channels 26.1 -> 22.2 us)
        auto get_unit = [&](const float *from) {
            unit v;
            if (whole) {
                v = *reinterpret_cast<const loose_unit *>(from);
                return v;
            }
#pragma unroll
            for (int i = 0; i < U; i++) v[i] = c0 + at + i < cend ? from[i] : 0.0f;
            return v;
        };
        unit zeros, bias, skip;
#pragma unroll
        for (int i = 0; i < U; i++) zeros[i] = 0.0f;
        bias = p.dt_bias && has ? get_unit(p.dt_bias + c0 + at) : zeros;
        skip = p.skip && has ? get_unit(p.skip + c0 + at) : zeros;
        auto fetch = [&](int tile) {
            const int left = q.fresh - tile * T::TOKENS - t0;  // tokens from the wavefront's first one on
#pragma unroll
            for (int k = 0; k < T::PER; k++) {
                x[k] = d[k] = g[k] = zeros;
                if (has && tq + k * APART < left) {
                    x[k] = get_unit(px + k * APART * mx);
                    d[k] = get_unit(pd + k * APART * md);
                    if (PART != 1 && p.gate) g[k] = get_unit(pg + k * APART * mg);
                }
            }
#pragma unroll
            for (int k = 0; k < T::VPER; k++) {
#pragma unroll
                for (int i = 0; i < NL; i++) b[k][i] = cc[k][i] = 0.0f;
                if (hasv && (T::VECTORS >= 64 || lane < T::VECTORS) && tv + k * VAPART < left) {
                    const float *fb = pb + k * VAPART * mb, *fc = pc + k * VAPART * mc;
                    if (wholev) {
                        b[k] = *reinterpret_cast<const loose_vec *>(fb);
                        if (PART != 1) cc[k] = *reinterpret_cast<const loose_vec *>(fc);
                    } else {
#pragma unroll
                        for (int i = 0; i < NL; i++)
                            if (av + i < p.n) {
                                b[k][i] = fb[i];
                                if (PART != 1) cc[k][i] = fc[i];
                            }
                    }
                }
            }
            px += T::TOKENS * mx;
            pd += T::TOKENS * md;
            pg += T::TOKENS * mg;
            pb += T::TOKENS * mb;
            pc += T::TOKENS * mc;
        };
        float *steps = all_steps[wave], *inputs = all_inputs[wave];
        vec *vb = all_b[wave], *vc = all_c[wave];
        // steps and inputs are 0 behind the sequence's last token and the last channel: the state stays
        auto stage = [&](int tile) {
            const int left = q.fresh - tile * T::TOKENS - t0;
#pragma unroll
            for (int k = 0; k < T::PER; k++) {
                const bool in = tq + k * APART < left;
                unit step = d[k] + bias;
                if (p.softplus) {  // (side by side: each is a chain of dependent instructions)
#pragma unroll
                    for (int i = 0; i < U; i++) step[i] = softplus(step[i]);
                }
#pragma unroll
                for (int i = 0; i < U; i++) {
                    step[i] = in && c0 + at + i < cend ? step[i] : 0.0f;
                    steps[(at + i) * T::STRIDE + tq + k * APART] = step[i];
                    inputs[(at + i) * T::STRIDE + tq + k * APART] = step[i] * x[k][i];
                }
            }
#pragma unroll
            for (int k = 0; k < T::VPER; k++)
                if (T::VECTORS >= 64 || lane < T::VECTORS) {
                    vb[lane + k * 64] = b[k];
                    if (PART != 1) vc[lane + k * 64] = cc[k];
                }
        };

        const float *my_steps = steps + ch * T::STRIDE;
        float *my_inputs = inputs + ch * T::STRIDE;
        const vec *my_b = vb + ln, *my_c = vc + (PART == 1 ? 0 : ln);

        if (tile0 < tile1) fetch(tile0);

        // Workspace of a sequence: the state that it continues, the states of its parts, those of its pieces; half the exponents of both (runs side by side have the sum of theirs).
        const long long step = (long long)p.channels * T::NP, at0 = (long long)c * T::NP + n0;
        const int all = (int)p.parts * (PIECES + 1);
        float *states = PART ? p.part_states + (long long)place * (all + 1) * step + at0 : nullptr, *halves_of = PART ? p.part_exponents + (long long)place * all * step + at0 : nullptr;
        auto take_in = [&](vec &f, vec &b, int which) {  // a part or piece behind what f and b hold
            const vec pf = *reinterpret_cast<const vec *>(halves_of + which * step), pb = *reinterpret_cast<const vec *>(states + (which + 1) * step);
#pragma unroll
            for (int i = 0; i < NL; i++) {
                b[i] = behind_run(run_root(pf[i]), b[i], pb[i]);
                f[i] += pf[i];
            }
        };
        if constexpr (PART == 0) {
            if (mine && wt == 0) first_state<NL, false>(p, q, c, n0, h);
            if (WT > 1 && wt == 0) {
                vec v;
#pragma unroll
                for (int i = 0; i < NL; i++) v[i] = h[i];
                begin[set] = v;
            }
        } else if constexpr (PART == 1) {
            if (mine && part == 0 && wave == 0) {  // kept for the second launch, in which the slot may be written already
                float kept[NL];
                first_state<NL, false>(p, q, c, n0, kept);
#pragma unroll
                for (int i = 0; i < NL; i++) states[i] = kept[i];
            }
        } else {  // a stretch of the parts before this one and a piece of its own by every wavefront, joined by all of them
            vec f, b, v, pf, pb;
#pragma unroll
            for (int i = 0; i < NL; i++) f[i] = pf[i] = b[i] = v[i] = pb[i] = 0.0f;
            const int each = (part + WAVES - 1) / WAVES, end = min(part, (wave + 1) * each);
            if (mine) {
                v = *reinterpret_cast<const vec *>(states);
                take_in(pf, pb, (int)p.parts + part * PIECES + wave);
#pragma unroll 4
                for (int j = wave * each; j < end; j++) take_in(f, b, j);
            }
#pragma unroll
            for (int i = 0; i < NL; i++) {
                f[i] = run_root(f[i]);
                pf[i] = run_root(pf[i]);
            }
            factor[tid] = f;
            brought[tid] = b;
            factor[T::THREADS + tid] = pf;
            brought[T::THREADS + tid] = pb;
            __syncthreads();
            for (int w = 0; w < WAVES + wave; w++) {
                const vec wf = factor[w * 64 + lane], wb = brought[w * 64 + lane];
#pragma unroll
                for (int i = 0; i < NL; i++) v[i] = behind_run(wf[i], v[i], wb[i]);
            }
#pragma unroll
            for (int i = 0; i < NL; i++) h[i] = v[i];
        }

        for (int tile = tile0; tile < tile1; tile++) {
            in_order();
            stage(tile);
            unit x0[T::PER], g0[T::PER];
#pragma unroll
            for (int k = 0; k < T::PER; k++) {
                x0[k] = x[k];
                g0[k] = g[k];
            }
            if (tile + 1 < tile1) fetch(tile + 1);
            in_order();
            float kept[WT > 1 ? T::TT : 1][NL], put[WT > 1 ? T::TT : 1][NL];  // factors and products of the tokens
            if constexpr (WT > 1) {
                float local[NL], sum = 0.0f;
#pragma unroll
                for (int i = 0; i < NL; i++) local[i] = 0.0f;
#pragma unroll
                for (int t = 0; t < T::TT; t += 4) {
                    const floatx4 dv = *reinterpret_cast<const floatx4 *>(my_steps + t), xv = *reinterpret_cast<const floatx4 *>(my_inputs + t);
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const vec bv = my_b[(t + j) * LANES];
                        sum += dv[j];
#pragma unroll
                        for (int i = 0; i < NL; i++) {
                            const float f = __builtin_amdgcn_exp2f(dv[j] * a[i]), u = xv[j] * bv[i];
                            local[i] = __builtin_fmaf(f, local[i], u);
                            kept[t + j][i] = f;
                            put[t + j][i] = u;
                        }
                    }
                }
                const float half_sum = 0.5f * within(sum);
                vec v, f;
#pragma unroll
                for (int i = 0; i < NL; i++) {
                    v[i] = local[i];
                    f[i] = run_root(half_sum * a[i]);
                }
                const int half = tile - tile0 & 1;
                vec *all = brought + half * T::THREADS + set, *all_f = factor + half * T::THREADS + set;
                all[wt * SETS] = v;
                all_f[wt * SETS] = f;
                __syncthreads();
                const vec v0 = begin[half * SETS + set];
#pragma unroll
                for (int i = 0; i < NL; i++) h[i] = v0[i];
                auto take = [&](int w, auto count) {  // (reads in flight together)
                    constexpr int N = decltype(count)::value;
                    vec wf[N], wb[N];
#pragma unroll
                    for (int k = 0; k < N; k++) {
                        wf[k] = all_f[(w + k) * SETS];
                        wb[k] = all[(w + k) * SETS];
                    }
#pragma unroll
                    for (int k = 0; k < N; k++)
#pragma unroll
                        for (int i = 0; i < NL; i++) h[i] = behind_run(wf[k][i], h[i], wb[k][i]);
                };
                int w = 0;
                for (; w + 4 <= wt; w += 4) take(w, std::integral_constant<int, 4>());
                if (wt & 2) take(w, std::integral_constant<int, 2>()), w += 2;
                if (wt & 1) take(w, std::integral_constant<int, 1>());
            }
            float sum_d = 0.0f;
#pragma unroll
            for (int t = 0; t < T::TT; t += 4) {
                // The exponentials of four tokens first: one after another, each would be waited for (32 sequences of 512 tokens of 2048 channels
                // 175 -> 165 us).
                float f[4][NL], u[4][NL];
                if constexpr (WT == 1) {
                    const floatx4 dv = *reinterpret_cast<const floatx4 *>(my_steps + t), xv = *reinterpret_cast<const floatx4 *>(my_inputs + t);
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const vec bv = my_b[(t + j) * LANES];
                        if (PART == 1) sum_d += dv[j];
#pragma unroll
                        for (int i = 0; i < NL; i++) {
                            f[j][i] = __builtin_amdgcn_exp2f(dv[j] * a[i]);
                            u[j][i] = xv[j] * bv[i];
                        }
                    }
                    __builtin_amdgcn_sched_barrier(0);
                } else {
#pragma unroll
                    for (int j = 0; j < 4; j++)
#pragma unroll
                        for (int i = 0; i < NL; i++) {
                            f[j][i] = kept[t + j][i];
                            u[j][i] = put[t + j][i];
                        }
                }
                if constexpr (PART == 1) {
#pragma unroll
                    for (int j = 0; j < 4; j++)
#pragma unroll
                        for (int i = 0; i < NL; i++) h[i] = __builtin_fmaf(f[j][i], h[i], u[j][i]);
                } else {
                    floatx4 y;
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const vec cv = my_c[(t + j) * LANES];
                        float sum = 0.0f;
#pragma unroll
                        for (int i = 0; i < NL; i++) {
                            h[i] = __builtin_fmaf(f[j][i], h[i], u[j][i]);
                            sum = i ? __builtin_fmaf(cv[i], h[i], sum) : cv[i] * h[i];
                        }
                        y[j] = sum;
                    }
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        y[j] = lane_sum<LANES>(y[j]);
                        asm volatile("" : "+v"(y[j]));  // (or the last addition goes into the branch below, apart from its swap)
                    }
                    if (ln == 0) *reinterpret_cast<floatx4 *>(my_inputs + t) = y;
                }
            }
            if constexpr (PART == 1) {
                const float sum = within(through + sum_d), of_tile = sum - through;
                through_low += (through - (sum - of_tile)) + (sum_d - of_tile);
                through = sum;
            } else {
                if (WT > 1 && wt == WT - 1) {
                    vec v;
#pragma unroll
                    for (int i = 0; i < NL; i++) v[i] = h[i];
                    begin[(tile - tile0 + 1 & 1) * SETS + set] = v;
                }
                in_order();
                const int left = q.fresh - tile * T::TOKENS - t0;
#pragma unroll
                for (int k = 0; k < T::PER; k++) {
                    if (has && tq + k * APART < left) {
                        unit y;
#pragma unroll
                        for (int i = 0; i < U; i++) {
                            y[i] = inputs[(at + i) * T::STRIDE + tq + k * APART];
                            y[i] = __builtin_fmaf(skip[i], x0[k][i], y[i]);
                        }
                        if (p.gate) {
#pragma unroll
                            for (int i = 0; i < U; i++) y[i] *= silu(g0[k][i]);
                        }
                        float *to = py + k * APART * my;
                        if (whole) {
                            *reinterpret_cast<loose_unit *>(to) = y;
                        } else {
#pragma unroll
                            for (int i = 0; i < U; i++)
                                if (c0 + at + i < cend) to[i] = y[i];
                        }
                    }
                }
                py += T::TOKENS * my;
            }
        }
        if constexpr (PART == 1) {  // the piece's, and by the first wavefront all pieces' together
            float half = 0.5f * within(through + through_low);
            vec f, b;
#pragma unroll
            for (int i = 0; i < NL; i++) {
                f[i] = half * a[i];
                b[i] = h[i];
            }
            auto keep = [&](int which) {
                *reinterpret_cast<vec *>(halves_of + which * step) = f;
                *reinterpret_cast<vec *>(states + (which + 1) * step) = b;
            };
            if (mine) keep((int)p.parts + part * PIECES + wave);
#pragma unroll
            for (int i = 0; i < NL; i++) f[i] = run_root(f[i]);
            factor[tid] = f;
            brought[tid] = b;
            halves[tid] = half;
            __syncthreads();
            if (mine && wave == 0) {
#pragma unroll
                for (int w = 1; w < WAVES; w++) {
                    const vec wf = factor[w * 64 + lane], wb = brought[w * 64 + lane];
                    half += halves[w * 64 + lane];
#pragma unroll
                    for (int i = 0; i < NL; i++) b[i] = behind_run(wf[i], b[i], wb[i]);
                }
                half = within(half);
#pragma unroll
                for (int i = 0; i < NL; i++) f[i] = half * a[i];
                keep(part);
            }
        } else if (mine && wt == WT - 1 && tile0 < tile1 && tile1 == tiles) {
            keep_state<NL>(p, q, c, n0, h);
        }
        __syncthreads();  // (the next job's states)
    }
}

constexpr int MOST_STATES = 64;
constexpr int FEW_TOKENS = 3;  // up to here token after token from memory (32 sequences of 2 tokens of 2048 channels 8.8 us, as tiles 10.9; of 8 19.0 and 12.1)

constexpr int MIXED_TOKENS = 128;  // of the longest sequence, from which on long and short sequences are taken apart

template <int LANES, int NL>
int launch_scan(int dev, ScanParams &p, int seqs, int rows, int tokens) {
    const hipStream_t st = state(dev).stream;
    if (tokens <= FEW_TOKENS) {
        hipLaunchKernelGGL((p.n % NL == 0 ? scan_tokens_kernel<LANES, NL, true> : scan_tokens_kernel<LANES, NL, false>), dim3((unsigned)(((long long)p.channels * LANES + 255) / 256), seqs), dim3(256), 0, st, p);
        EH_CHECK_LAUNCH();
        return 0;
    }
    const int groups = p.channels / p.per;
    const long long num_cu = state(dev).num_cu;
    auto launch = [&](auto fn, int threads, long long count) {
        p.jobs = (long long)p.blocks * p.parts * (p.list ? count : seqs);
        EH_REQUIRE(p.jobs < (1LL << 31), "selective_scan: %d sequences of %d channels in %d groups are out of range", seqs, p.channels, groups);
        hipLaunchKernelGGL(fn, dim3(xcd_grid(p.jobs, threads)), dim3(threads), 0, st, p);
        EH_CHECK_LAUNCH();
        return 0;
    };
    // By the workgroups that there are, in multiples of the compute units: four wavefronts of different channels do the least work a token; where that leaves
    // the device half empty, they divide the tokens of a quarter of the channels (512 tokens of 2048 channels, us: 16 sequences 107 against 128, 12 105 and 95, 4 84 and
    // 36); where that would, too, eight do (2 sequences 28 and 22); and where those do not meet every unit, sequences are divided over workgroups (1000 tokens of
    // 1024 channels: not divided 39 us, divided 20; 8192 of 4096, as many workgroups as units: 221 and 276, since all exponentials are formed twice).
    using Alone = ScanTile<LANES, NL, 4, 1>;
    using Four = ScanTile<LANES, NL, 4, 4>;
    using Eight = ScanTile<LANES, NL, 8, 8>;
    auto blocks = [&](auto tile) { return (p.per + decltype(tile)::CHANNELS - 1) / decltype(tile)::CHANNELS; };  // of a group
    const long long wide = (long long)groups * blocks(Alone()), narrow = (long long)groups * blocks(Four());     // workgroups a sequence (eight wavefronts have as many channels as four)
    auto wavefronts = [&](long long seqs, int tokens) { return wide * seqs >= 2 * num_cu || tokens <= Alone::TOKENS ? 1 : 2 * narrow * seqs >= 3 * num_cu ? 4 : 8; };
    // The sequences of least to most tokens, `count` of them at most, of up to `tokens`; least 0: all up to most.
    auto run = [&](long long count, int tokens, int least, int most) {
        const int kind = wavefronts(count, tokens);
        p.group_blocks = kind == 1 ? blocks(Alone()) : blocks(Four());
        p.blocks = groups * p.group_blocks;
        const long long parts = num_cu / (narrow * count), tiles = (tokens + Eight::TOKENS - 1) / Eight::TOKENS;
        const bool divided = kind == 8 && parts >= 2 && tiles >= 4;
        // Eight wavefronts a part; two parts a unit where they are long (a workgroup and two a unit, us: 65536 tokens of 256 channels 164 and 140, 4096 of 1024 49 and 45,
        // 1000 of 1024 20.5 and 21.8).
        p.parts = (unsigned)(!divided ? 1 : tiles >= 8 * parts ? 2 * parts : std::min(parts, tiles));
        const size_t all = (size_t)p.parts * 9, each = (size_t)p.channels * Eight::NP * sizeof(float) * count;  // (parts and their pieces)
        const size_t part_bytes = divided ? each * (2 * all + 1) : 0, list_bytes = least > 0 ? (size_t)count * sizeof(int) : 0;
        void *ws = nullptr;
        if (part_bytes + list_bytes > 0) EH_TRY(get_workspace(dev, part_bytes + list_bytes, &ws));
        p.part_states = (float *)ws;
        p.part_exponents = (float *)((char *)ws + each * (all + 1));
        p.most = most;
        p.list = nullptr;
        if (least > 0) {
            int *list = (int *)((char *)ws + part_bytes);
            hipLaunchKernelGGL(list_sequences_kernel, dim3(1), dim3(LIST_THREADS), 0, st, p.batch, seqs, least, list, (int)count);
            EH_CHECK_LAUNCH();
            p.list = list;
        }
        if (kind == 1) return launch(scan_tile_kernel<LANES, NL, 4, 1, 0>, Alone::THREADS, count);
        if (kind == 4) return launch(scan_tile_kernel<LANES, NL, 4, 4, 0>, Four::THREADS, count);
        if (!divided) return launch(scan_tile_kernel<LANES, NL, 8, 8, 0>, Eight::THREADS, count);
        EH_TRY(launch(scan_tile_kernel<LANES, NL, 8, 1, 1>, Eight::THREADS, count));
        return launch(scan_tile_kernel<LANES, NL, 8, 1, 2>, Eight::THREADS, count);
    };
    // A few long sequences among many short ones would be walked as if there were many long ones.  Of more than half the longest's tokens there are no more than the rows
    // hold: where they are few, and would be walked by more wavefronts, they are taken by themselves (31
    // single tokens and a prompt of 2048 of 2048 channels 255 us, so 61; 255 of 3 tokens and one of 8192 of 1024 channels 998 and 110; 60 of 20 and 4 of 500 of 768 71 and 37).
    const int half = tokens / 2;
    const long long few = std::max(1, std::min(seqs, rows / (half + 1)));
    const bool mixed = tokens >= MIXED_TOKENS && 4 * few <= seqs && wavefronts(few, tokens) != wavefronts(seqs, tokens);
    if (mixed) EH_TRY(run(seqs, half, 0, half));
    return mixed ? run(few, tokens, half + 1, INT_MAX) : run(seqs, tokens, 0, INT_MAX);
}

}  // namespace

extern "C" int eddlhip_selective_scan(int dev, const float *X, long long ldx, const float *dt, long long lddt, const float *A, const float *B, long long ldb,
                                      const float *C, long long ldc, const float *skip, const float *gate, long long ldg, const float *dt_bias, float *Y, long long ldy,
                                      int rows, int channels, int n, int groups, int softplus, int reverse, float *states, int pool, const int *offsets,
                                      const int *lengths, const int *slots, const int *out_slots, int seqs, int max_new) {
    EH_REQUIRE(channels > 0 && channels <= MOST_CHANNELS && n > 0 && n <= MOST_STATES, "selective_scan: %d channels (up to %d) of %d states (1 to %d)", channels, MOST_CHANNELS, n, MOST_STATES);
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
    p.batch = StateBatch{offsets, lengths, slots, out_slots, rows, pool, reverse != 0};
    const int tokens = std::max(1, std::min(max_new, rows));
    if (n == 1) return launch_scan<1, 1>(dev, p, seqs, rows, tokens);
    if (n <= 4) return launch_scan<1, 4>(dev, p, seqs, rows, tokens);
    if (n <= 8) return launch_scan<2, 4>(dev, p, seqs, rows, tokens);
    if (n <= 16) return launch_scan<4, 4>(dev, p, seqs, rows, tokens);
    if (n <= 32) return launch_scan<8, 4>(dev, p, seqs, rows, tokens);
    return launch_scan<16, 4>(dev, p, seqs, rows, tokens);
}
