// The selective scan
//     d = softplus(dt + dt_bias),   h[c][n] = e^(d A[c][n]) h[c][n] + d x B[n],   y = (sum_n C[n] h[c][n] + skip x) silu(gate),
// token by token, over ragged batches of sequences whose states lie in slots of a pool.
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
    float *part_states, *part_factors;  // [sequence][part + 1][channel][NP], [sequence][part][channel][NP]
    long long ldx, lddt, ldg, ldb, ldc, ldy;
    int channels, n, per;  // channels that share B and C
    unsigned blocks, group_blocks, parts;
    long long jobs;
    bool softplus, vectors;  // B and C are read 16 bytes at a time
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

// NL numbers from n0 of n on; 0 behind the last.  VEC: n is a multiple of NL and the place one of their size.
template <int NL, bool VEC>
__device__ __forceinline__ void get(const float *from, int n0, int n, float (&v)[NL]) {
    typedef float vec __attribute__((ext_vector_type(NL)));
    if constexpr (VEC) {
        vec u;
#pragma unroll
        for (int i = 0; i < NL; i++) u[i] = 0.0f;
        if (n0 < n) u = *reinterpret_cast<const vec *>(from + n0);
#pragma unroll
        for (int i = 0; i < NL; i++) v[i] = u[i];
    } else {
#pragma unroll
        for (int i = 0; i < NL; i++) v[i] = n0 + i < n ? from[n0 + i] : 0.0f;
    }
}
// The NL states of channel c from n0 on: as the sequence finds them, and on their way to the pool; the factors of the steps in powers of two.
template <int NL, bool VEC>
__device__ __forceinline__ void first_state(const ScanParams &p, const Sequence &q, int c, int n0, float (&h)[NL]) {
#pragma unroll
    for (int i = 0; i < NL; i++) h[i] = q.read == -2 ? __builtin_nanf("") : 0.0f;
    if (q.read >= 0) get<NL, VEC>(p.states + ((long long)q.read * p.channels + c) * p.n, n0, p.n, h);
}
template <int NL, bool VEC>
__device__ __forceinline__ void keep_state(const ScanParams &p, const Sequence &q, int c, int n0, const float (&h)[NL]) {
    typedef float vec __attribute__((ext_vector_type(NL)));
    if (q.write < 0) return;
    float *to = p.states + ((long long)q.write * p.channels + c) * p.n + n0;
    if constexpr (VEC) {
        vec u;
#pragma unroll
        for (int i = 0; i < NL; i++) u[i] = h[i];
        if (n0 < p.n) *reinterpret_cast<vec *>(to) = u;
    } else {
#pragma unroll
        for (int i = 0; i < NL; i++)
            if (n0 + i < p.n) to[i] = h[i];
    }
}
template <int NL, bool VEC>
__device__ __forceinline__ void exponents(const ScanParams &p, int c, int n0, float (&a)[NL]) {
    constexpr float MOST = 3.40282347e38f;
    get<NL, VEC>(p.A + (long long)c * p.n, n0, p.n, a);
#pragma unroll
    for (int i = 0; i < NL; i++) {
        a[i] *= LOG2_E;
        a[i] = a[i] > MOST ? MOST : a[i] < -MOST ? -MOST : a[i];  // (an infinite one would make NaN of the steps of 0 behind the last token)
    }
}

// Few tokens a sequence: LANES lanes a channel, NL states each; token after token from memory.  VEC: vectors, states and A are read 16 bytes at a time.
template <int LANES, int NL, bool VEC>
__global__ __launch_bounds__(256) void scan_tokens_kernel(const ScanParams p) {
    const Sequence q = sequence(p.batch, blockIdx.y);
    const int c = blockIdx.x * (256 / LANES) + threadIdx.x / LANES, lane = threadIdx.x % LANES, n0 = lane * NL;
    if (q.fresh == 0 || c >= p.channels) return;
    float a[NL], h[NL];
    first_state<NL, VEC>(p, q, c, n0, h);
    exponents<NL, VEC>(p, c, n0, a);
    const float bias = p.dt_bias ? p.dt_bias[c] : 0.0f, skip = p.skip ? p.skip[c] : 0.0f;
    const int v0 = c / p.per * p.n;
    for (int t = 0; t < q.fresh; t++) {
        const long long row = q.row(t);
        float b[NL], cc[NL];
        get<NL, VEC>(p.B + row * p.ldb + v0, n0, p.n, b);
        get<NL, VEC>(p.C + row * p.ldc + v0, n0, p.n, cc);
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
    keep_state<NL, VEC>(p, q, c, n0, h);
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

// PART 0: the whole scan of a sequence.  A long one that would leave the device empty is divided over workgroups: PART 1 brings the state of every part from
// zeros and the factor of what comes before it, PART 2 takes in the parts before its own and brings the outputs.
template <int LANES, int NL, int WAVES, int WT, bool VEC, int PART>
__global__ __launch_bounds__(64 * WAVES, WT > 1 || LANES == 1 ? 2 : 4) void scan_tile_kernel(const ScanParams p) {
    using T = ScanTile<LANES, NL, WAVES, WT>;
    constexpr int U = T::U;
    typedef float vec __attribute__((ext_vector_type(NL)));
    typedef float unit __attribute__((ext_vector_type(U)));
    constexpr int SETS = 64 * (WAVES / WT);  // lanes that walk the same tokens
    __shared__ __attribute__((aligned(16))) float all_steps[WAVES][T::CH * T::STRIDE], all_inputs[WAVES][T::CH * T::STRIDE];  // d and d x, whose place the outputs take
    __shared__ __attribute__((aligned(16))) vec all_b[WAVES][T::VECTORS], all_c[WAVES][PART == 1 ? 1 : T::VECTORS];
    // (two of each: a wavefront may be a tile ahead of the slowest one)
    __shared__ __attribute__((aligned(16))) vec brought[WT > 1 ? 2 * T::THREADS : 1], factor[WT > 1 ? 2 * T::THREADS : 1], begin[WT > 1 ? 2 * SETS : 1];

    // (workgroups side by side in channels share lines of memory, and B and C)
    for (long long id = blockIdx.x; id < xcd_padded(p.jobs); id += gridDim.x) {
        const long long job = xcd_job(id);
        if (job >= p.jobs) continue;
        const unsigned rest = (unsigned)job / p.blocks;  // (fewer than 2^31 jobs)
        const int block = (unsigned)job % p.blocks, group = block / p.group_blocks, part = rest % p.parts, s = rest / p.parts;
        const Sequence q = sequence(p.batch, s);
        const int tiles = (int)(((long long)q.fresh + T::TOKENS - 1) / T::TOKENS), share = (tiles + (int)p.parts - 1) / (int)p.parts;  // (of a part)
        const int tile0 = min(tiles, part * share), tile1 = min(tiles, tile0 + share);
        if (tile0 == tile1) continue;

        const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), wt = wave % WT, wc = wave / WT, set = wc * 64 + lane;
        const int c0 = group * p.per + (int)(block % p.group_blocks) * T::CHANNELS + wc * T::CH, cend = (group + 1) * p.per;  // the wavefront's first channel
        const int ch = lane / LANES, c = c0 + ch, ln = lane % LANES, n0 = ln * NL;
        const bool mine = c < cend;

        float a[NL], h[NL], through[NL];  // (through: the factor of all tokens of a part)
#pragma unroll
        for (int i = 0; i < NL; i++) {
            a[i] = h[i] = 0.0f;
            through[i] = 1.0f;
        }
        if (mine) exponents<NL, false>(p, c, n0, a);
        if constexpr (PART == 2) {  // the parts before this one: a stretch of them by every wavefront, joined by the first (the second half is free until the second tile)
            vec f, b;
#pragma unroll
            for (int i = 0; i < NL; i++) {
                f[i] = 1.0f;
                b[i] = 0.0f;
            }
            const int each = (part + WT - 1) / WT, end = min(part, (wt + 1) * each);
            const long long step = (long long)p.channels * T::NP;
            const float *factors = p.part_factors + ((long long)s * (int)p.parts * p.channels + c) * T::NP + n0;
            const float *states = p.part_states + ((long long)s * ((int)p.parts + 1) * p.channels + c) * T::NP + n0;
            if (mine)
#pragma unroll 4
                for (int j = wt * each; j < end; j++) {
                    const vec pf = *reinterpret_cast<const vec *>(factors + j * step), pb = *reinterpret_cast<const vec *>(states + (j + 1) * step);
#pragma unroll
                    for (int i = 0; i < NL; i++) {
                        b[i] = __builtin_fmaf(pf[i], b[i], pb[i]);
                        f[i] *= pf[i];
                    }
                }
            factor[T::THREADS + wt * SETS + set] = f;
            brought[T::THREADS + wt * SETS + set] = b;
            __syncthreads();
        }
        if (mine && wt == 0) {
            float *states = PART ? p.part_states + ((long long)s * ((int)p.parts + 1) * p.channels + c) * T::NP + n0 : nullptr;
            if (PART == 0) {
                first_state<NL, false>(p, q, c, n0, h);
            } else if (PART == 1) {
                if (part == 0) {  // kept for the second launch, in which the slot may be written already
                    float kept[NL];
                    first_state<NL, false>(p, q, c, n0, kept);
#pragma unroll
                    for (int i = 0; i < NL; i++) states[i] = kept[i];
                }
            } else {
                const vec v = *reinterpret_cast<const vec *>(states);
#pragma unroll
                for (int i = 0; i < NL; i++) h[i] = v[i];
#pragma unroll 1
                for (int w = 0; w < WT; w++) {
                    const vec f = factor[T::THREADS + w * SETS + set], b = brought[T::THREADS + w * SETS + set];
#pragma unroll
                    for (int i = 0; i < NL; i++) h[i] = __builtin_fmaf(f[i], h[i], b[i]);
                }
            }
            if (WT > 1 && PART != 1) {
                vec v;
#pragma unroll
                for (int i = 0; i < NL; i++) v[i] = h[i];
                begin[set] = v;
            }
        }

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
        const bool has = c0 + at < cend, hasv = av < p.n;
        auto get_unit = [&](const float *from) {
            if (VEC) return *reinterpret_cast<const unit *>(from);
            unit v;
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
                    if (p.vectors) {
                        b[k] = *reinterpret_cast<const vec *>(fb);
                        if (PART != 1) cc[k] = *reinterpret_cast<const vec *>(fc);
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

        fetch(tile0);
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
            float kept[WT > 1 ? T::TT : 1][NL], put[WT > 1 && PART != 1 ? T::TT : 1][NL];  // factors and products of the tokens
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
                            if (PART != 1) put[t + j][i] = u;
                        }
                    }
                }
                vec v, f;
#pragma unroll
                for (int i = 0; i < NL; i++) {
                    v[i] = local[i];
                    f[i] = __builtin_amdgcn_exp2f(sum * a[i]);
                }
                const int half = tile - tile0 & 1;
                vec *all = brought + half * T::THREADS + set, *all_f = factor + half * T::THREADS + set;
                all[wt * SETS] = v;
                all_f[wt * SETS] = f;
                __syncthreads();
                const int before = PART == 1 ? (wt == 0 ? WT : 0) : wt;
                if (PART != 1) {
                    const vec v0 = begin[half * SETS + set];
#pragma unroll
                    for (int i = 0; i < NL; i++) h[i] = v0[i];
                }
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
                        for (int i = 0; i < NL; i++) {
                            h[i] = __builtin_fmaf(wf[k][i], h[i], wb[k][i]);
                            if (PART == 1) through[i] *= wf[k][i];
                        }
                };
                int w = 0;
                for (; w + 4 <= before; w += 4) take(w, std::integral_constant<int, 4>());
                if (before & 2) take(w, std::integral_constant<int, 2>()), w += 2;
                if (before & 1) take(w, std::integral_constant<int, 1>());
            }
            if constexpr (PART != 1) {
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
                        if (VEC) {
                            *reinterpret_cast<unit *>(to) = y;
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
        if (PART == 1) {
            if (mine && wt == 0) {
                float *states = p.part_states + (((long long)s * ((int)p.parts + 1) + part + 1) * p.channels + c) * T::NP + n0;
                float *factors = p.part_factors + (((long long)s * (int)p.parts + part) * p.channels + c) * T::NP + n0;
#pragma unroll
                for (int i = 0; i < NL; i++) {
                    states[i] = h[i];
                    factors[i] = through[i];
                }
            }
        } else if (mine && wt == WT - 1 && tile1 == tiles) {
            keep_state<NL, false>(p, q, c, n0, h);
        }
        __syncthreads();  // (the next job's states)
    }
}

constexpr int MOST_STATES = 64;
constexpr int FEW_TOKENS = 3;  // up to here token after token from memory (32 sequences of 2 tokens of 2048 channels 8.8 us, as tiles 10.9; of 8 19.0 and 12.1)

template <int LANES, int NL>
int launch_scan(int dev, ScanParams &p, int seqs, int tokens, bool vec) {
    const hipStream_t st = state(dev).stream;
    if (tokens <= FEW_TOKENS) {
        const bool whole = p.vectors && (((uintptr_t)p.states | (uintptr_t)p.A) & 15) == 0;
        hipLaunchKernelGGL((whole ? scan_tokens_kernel<LANES, NL, true> : scan_tokens_kernel<LANES, NL, false>), dim3((unsigned)(((long long)p.channels * LANES + 255) / 256), seqs), dim3(256), 0, st, p);
        EH_CHECK_LAUNCH();
        return 0;
    }
    const int groups = p.channels / p.per;
    const long long num_cu = state(dev).num_cu;
    auto launch = [&](auto fn, int threads) {
        p.jobs = (long long)p.blocks * p.parts * seqs;
        EH_REQUIRE(p.jobs < (1LL << 31), "selective_scan: %d sequences of %d channels in %d groups are out of range", seqs, p.channels, groups);
        hipLaunchKernelGGL(fn, dim3(xcd_grid(p.jobs, threads)), dim3(threads), 0, st, p);
        EH_CHECK_LAUNCH();
        return 0;
    };
    // (workgroups of a call without parts)
    auto sized = [&](auto tile) {
        using T = decltype(tile);
        p.parts = 1;
        p.group_blocks = (p.per + T::CHANNELS - 1) / T::CHANNELS;
        p.blocks = groups * p.group_blocks;
        return (long long)p.blocks * seqs;
    };
    auto divided = [&](auto tile, auto first, auto second, int parts) {
        using T = decltype(tile);
        p.parts = parts;
        const size_t each = (size_t)p.channels * T::NP * sizeof(float);
        void *ws = nullptr;
        EH_TRY(get_workspace(dev, each * seqs * (2 * (size_t)parts + 1), &ws));
        p.part_states = (float *)ws;
        p.part_factors = (float *)((char *)ws + each * seqs * (parts + 1));
        EH_TRY(launch(first, T::THREADS));
        return launch(second, T::THREADS);
    };
    // By the workgroups that there are, in multiples of the compute units: four wavefronts of different channels do the least work a token; where that leaves
    // the device half empty, they divide the tokens of a quarter of the channels (512 tokens of 2048 channels, us: 16 sequences 107 against 128, 12 105 and 95, 4 84 and
    // 36); where that would, too, eight do (2 sequences 28 and 22); and where those do not meet every unit, sequences are divided over workgroups.
    using Alone = ScanTile<LANES, NL, 4, 1>;
    using Four = ScanTile<LANES, NL, 4, 4>;
    using Eight = ScanTile<LANES, NL, 8, 8>;
    if (sized(Alone()) >= 2 * num_cu || tokens <= Alone::TOKENS)
        return launch(vec ? scan_tile_kernel<LANES, NL, 4, 1, true, 0> : scan_tile_kernel<LANES, NL, 4, 1, false, 0>, Alone::THREADS);
    const long long workgroups = sized(Four());  // (as many as of eight wavefronts, which have as many channels)
    if (2 * workgroups >= 3 * num_cu) return launch(vec ? scan_tile_kernel<LANES, NL, 4, 4, true, 0> : scan_tile_kernel<LANES, NL, 4, 4, false, 0>, Four::THREADS);
    const long long parts = num_cu / workgroups, tiles = (tokens + Eight::TOKENS - 1) / Eight::TOKENS;
    if (parts < 2 || tiles < 4)
        return launch(vec ? scan_tile_kernel<LANES, NL, 8, 8, true, 0> : scan_tile_kernel<LANES, NL, 8, 8, false, 0>, Eight::THREADS);
    // (4096 tokens of 1024 channels: not divided 125 us, 4 parts of eight wavefronts 63, 8 of four 57; 1000 tokens 39, 24 and 25)
    if (tiles >= 8 * parts)
        return vec ? divided(Four(), scan_tile_kernel<LANES, NL, 4, 4, true, 1>, scan_tile_kernel<LANES, NL, 4, 4, true, 2>, (int)(2 * parts))
                   : divided(Four(), scan_tile_kernel<LANES, NL, 4, 4, false, 1>, scan_tile_kernel<LANES, NL, 4, 4, false, 2>, (int)(2 * parts));
    const int n = (int)std::min(parts, tiles);
    return vec ? divided(Eight(), scan_tile_kernel<LANES, NL, 8, 8, true, 1>, scan_tile_kernel<LANES, NL, 8, 8, true, 2>, n)
               : divided(Eight(), scan_tile_kernel<LANES, NL, 8, 8, false, 1>, scan_tile_kernel<LANES, NL, 8, 8, false, 2>, n);
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
    // (a group's first channel, too, has to be aligned)
    uintptr_t rows16 = 0, vectors16 = (uintptr_t)B | (uintptr_t)C;
    for (const void *at : {(const void *)X, (const void *)dt, (const void *)gate, (const void *)Y, (const void *)skip, (const void *)dt_bias}) rows16 |= (uintptr_t)at;
    const bool vec = (rows16 & 15) == 0 && p.per % 4 == 0 && ldx % 4 == 0 && lddt % 4 == 0 && ldy % 4 == 0 && (!gate || ldg % 4 == 0);
    p.vectors = n == 1 || ((vectors16 & 15) == 0 && n % 4 == 0 && ldb % 4 == 0 && ldc % 4 == 0);
    const int tokens = std::max(1, std::min(max_new, rows));
    if (n == 1) return launch_scan<1, 1>(dev, p, seqs, tokens, vec);
    if (n <= 4) return launch_scan<1, 4>(dev, p, seqs, tokens, vec);
    if (n <= 8) return launch_scan<2, 4>(dev, p, seqs, tokens, vec);
    if (n <= 16) return launch_scan<4, 4>(dev, p, seqs, tokens, vec);
    if (n <= 32) return launch_scan<8, 4>(dev, p, seqs, tokens, vec);
    return launch_scan<16, 4>(dev, p, seqs, tokens, vec);
}
