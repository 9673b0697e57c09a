// Group norm with its activation: the mean and variance of the channels of a group over all pixels of an image,
//     n = (x - mean) / sqrt(variance + eps) w + b,   y = act(n (1 + mod) + shift).
// Maps [images][channels][pixels], where a group is one stretch of memory, or rows of tokens [images * pixels][channels], where it is a
// piece of every row.
//
// Bound: memory, 8 bytes a number, if a group is read once.  A group of up to 32768 numbers (in rows about 32000, where threads stay in their columns; of groups of
// few channels all that are taken together) stays in the registers of a workgroup between its sums and its outputs (WHOLE).  A larger one is divided: the first launch
// brings mean and variance of every part, the second joins them and reads the numbers again, from the last one to the first: what was read last may still be in the
// last-level cache.  The variance is that of differences from a mean, never a difference of squares.
//
// Measured: rows of 64 images of 196 tokens of 768 channels, modulated, 17.2 us (4.5 TB/s); maps of 4 x 64 x 512 x 512, groups of 524288 numbers, 126 us (sums 39 and
// outputs 80, both 6.7 TB/s); rows of 3 x 1369 x 330, groups of 41070, 10.4 us, two launches of 4.4 and 6.6; 1 x 512 x 7 x 7 4.9 us, the host's call.
#include <math.h>

#include <algorithm>

#include "common.h"
#include "activation.h"
#include "xcd.h"

using namespace eddlhip;

namespace {

enum { WHOLE, SUMS, APPLY };  // what a launch does

struct GroupNormParams {
    const float *X, *w, *b, *mod, *shift;
    float *Y;
    float2 *parts;  // mean and variance of every part
    long long ldx, ldy;
    int images, channels, pixels, activation;
    unsigned groups;
    int per;              // channels of a group
    unsigned split;       // parts of a group
    unsigned blocks;      // groups taken together, of an image (short rows)
    long long part;       // numbers of a part, or rows of one (short rows)
    long long jobs;       // of the launch
    int together;         // groups of a workgroup (short rows)
    bool lines;           // a workgroup writes whole lines of memory
    float eps, of_nan;    // what a ReLU makes of NaN
};

// A ReLU that keeps NaN and one that does not differ in a number, not in a branch (which every number would take: 17.3 -> 18.1 us, 6.0 -> 6.4).
__device__ __forceinline__ float activated(float x, const GroupNormParams &p) {
    if (p.activation == EDDLHIP_ACT_SILU) return silu(x);
    return p.activation == EDDLHIP_ACT_RELU ? (x != x ? p.of_nan : x > 0.0f ? x : 0.0f) : x;
}

// The sum over a wavefront, in all lanes: across the 16 lanes of a row by operands of other lanes, the four rows one after another.
template <int CTRL>
__device__ __forceinline__ float swapped(float x) {
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float wave_sum(float x) {
    x += swapped<0xB1>(x);   // the neighbour
    x += swapped<0x4E>(x);   // the other pair of four
    x += swapped<0x141>(x);  // the other four of eight, mirrored
    x += swapped<0x140>(x);  // the other eight of sixteen, mirrored
    float row[4];
#pragma unroll
    for (int r = 0; r < 4; r++) row[r] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), 16 * r));
    return (row[0] + row[1]) + (row[2] + row[3]);
}
__device__ __forceinline__ float2 wave_sum(float2 x) { return float2{wave_sum(x.x), wave_sum(x.y)}; }
__device__ __forceinline__ void add(float &x, float y) { x += y; }
__device__ __forceinline__ void add(float2 &x, float2 y) {
    x.x += y.x;
    x.y += y.y;
}
template <int THREADS, typename T>
__device__ __forceinline__ T block_sum(T x, float2 *place) {
    T *red = reinterpret_cast<T *>(place);
    x = wave_sum(x);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
    __syncthreads();
    x = red[0];
#pragma unroll
    for (int w = 1; w < THREADS / 64; w++) add(x, red[w]);
    return x;
}

// Of n numbers, nth = 1 / n, whose sum gave `mean`: `off` holds the sum of their differences from it and that of the differences' squares.  The first is what the mean lost to rounding, so
// that equal numbers have their own value as their mean, and nothing but the bias is left of them (of 1234.567, 32768 times, the mean's last bits made 0.04).
__device__ __forceinline__ void settle(float &mean, float &variance, float nth, float2 off) {
    const float more = off.x * nth, left = off.y - more * off.x;
    mean += more;
    variance = left < 0.0f ? 0.0f : left * nth;
}

template <int UNIT>
struct Unit {
    float v[UNIT];
};
template <int UNIT>
__device__ __forceinline__ Unit<UNIT> get(const float *from) {
    typedef float vec __attribute__((ext_vector_type(UNIT), aligned(4)));  // (the hardware reads and writes 16 bytes at any multiple of four)
    const vec v = *reinterpret_cast<const vec *>(from);
    Unit<UNIT> u;
#pragma unroll
    for (int i = 0; i < UNIT; i++) u.v[i] = v[i];
    return u;
}
// Whole lines of memory are written past the caches (rows of 32 channels a group 29 -> 24 us); of a piece of a line the L2 makes a whole one
// (24 channels a group 27 -> 21).
template <int UNIT>
__device__ __forceinline__ void set(float *to, const Unit<UNIT> &u, bool lines) {
    typedef float vec __attribute__((ext_vector_type(UNIT), aligned(4)));
    vec v;
#pragma unroll
    for (int i = 0; i < UNIT; i++) v[i] = u.v[i];
    if (UNIT == 4 && lines) {
        asm volatile("");  // (or the compiler makes one store of the two, without the hint)
        __builtin_nontemporal_store(v, reinterpret_cast<vec *>(to));
        asm volatile("");
    } else {
        *reinterpret_cast<vec *>(to) = v;
    }
}

// y = act((x - mean) slope + lift) for UNIT channels of an image.  What they are made of is asked for before the sums, behind which it would be waited for.
template <int UNIT>
struct Coefficients {
    Unit<UNIT> w, b, mod, shift;

    __device__ __forceinline__ void ask(const GroupNormParams &p, int image, int c) {
        const long long at = (long long)image * p.channels + c;
#pragma unroll
        for (int i = 0; i < UNIT; i++) {
            w.v[i] = 1.0f;
            b.v[i] = mod.v[i] = shift.v[i] = 0.0f;
        }
        if (p.w) w = get<UNIT>(p.w + c);
        if (p.b) b = get<UNIT>(p.b + c);
        if (p.mod) mod = get<UNIT>(p.mod + at);
        if (p.shift) shift = get<UNIT>(p.shift + at);
    }
    __device__ __forceinline__ void make(float scale, float *slope, float *lift) const {
#pragma unroll
        for (int i = 0; i < UNIT; i++) {
            const float more = 1.0f + mod.v[i];
            slope[i] = scale * w.v[i] * more;
            lift[i] = b.v[i] * more + shift.v[i];
        }
    }
};

// Mean and variance of n more numbers taken into those of `count`: no sum of squares, which passes the largest number before the variance does.
__device__ __forceinline__ void join(double &count, float &mean, float &variance, double n, float mean_n, float variance_n) {
    const float delta = mean_n - mean, share = (float)(n / (count + n));
    mean = __builtin_fmaf(delta, share, mean);
    variance = variance * (1.0f - share) + variance_n * share + delta * (share * (1.0f - share)) * delta;  // (of the first n numbers nothing but their own, also of 1e20, whose square is infinite)
    count += n;
}
constexpr int MOST_PARTS = 256;  // of a group

// Those of all parts of a group of `total` numbers, parts of `part` each, by a wavefront; in all of its lanes.
struct Parts {
    float2 v[MOST_PARTS / 64];

    __device__ __forceinline__ void ask(const float2 *parts, int split) {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int k = 0; k < MOST_PARTS / 64; k++) {
            v[k] = float2{0.0f, 0.0f};
            if (lane + k * 64 < split) v[k] = parts[lane + k * 64];
        }
    }
    __device__ __forceinline__ void join(int split, long long part, long long total, float &mean, float &variance) const {
        const int lane = threadIdx.x & 63;
        const float first = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, v[0].x)));  // (differences from it: equal means are the mean)
        float sum = 0.0f, share[MOST_PARTS / 64];
#pragma unroll
        for (int k = 0; k < MOST_PARTS / 64; k++) {
            share[k] = lane + k * 64 < split ? (float)min(part, total - (lane + k * 64) * part) / (float)total : 0.0f;
            sum += (v[k].x - first) * share[k];
        }
        mean = first + wave_sum(sum);
        sum = 0.0f;
#pragma unroll
        for (int k = 0; k < MOST_PARTS / 64; k++) sum += v[k].y * share[k] + (v[k].x - mean) * share[k] * (v[k].x - mean);
        variance = wave_sum(sum);
    }
};

constexpr int SHORT = 16;  // channels of a group in rows: of smaller ones as many are taken together as make 2 * SHORT channels, 128 bytes of a row

constexpr int MOST_CHANNELS = 4096;  // of a group: their slopes and lifts lie in LDS

// A workgroup a group of an image or a part of one.  UNIT numbers are read at a time; ROWS: the numbers are counted along the group's pieces of the rows.
template <int THREADS, int NV, int UNIT, bool ROWS, int WHAT>
__global__ __launch_bounds__(THREADS) void group_norm_kernel(const GroupNormParams p) {
    __shared__ float2 red[THREADS / 64];
    extern __shared__ float slopes[];  // of the group's channels, and their lifts
    float *lifts = slopes + p.per;
    constexpr int STEP = THREADS * UNIT, TILE = STEP * NV;
    const long long count = (long long)p.per * p.pixels;
    const unsigned inner = ROWS ? p.per : p.pixels, step_hi = STEP / inner, step_lo = STEP % inner;  // (a number's row and channel, or channel and pixel)
    const bool whole_units = p.pixels % UNIT == 0;
    for (long long id = blockIdx.x; id < xcd_padded(p.jobs); id += gridDim.x) {
        long long job = xcd_job(id);  // (groups side by side share lines of memory where they are pieces of rows)
        if (job >= p.jobs) continue;
        if (WHAT == APPLY) job = p.jobs - 1 - job;  // (what the sums read last is still in the last-level cache)
        // (fewer than 2^31 jobs; in rows the groups of a piece come one after another, since they share lines)
        const unsigned piece = ROWS ? (unsigned)job / p.groups % p.split : (unsigned)job % p.split;
        const unsigned which = ROWS ? (unsigned)job / p.groups / p.split * p.groups + (unsigned)job % p.groups : (unsigned)job / p.split;
        const long long first = piece * p.part, last = min(count, first + p.part);
        const int image = which / p.groups, c0 = (int)(which % p.groups) * p.per;
        const float *X = p.X + (ROWS ? (long long)image * p.pixels * p.ldx + c0 : ((long long)image * p.channels + c0) * p.pixels);
        float *Y = p.Y + (ROWS ? (long long)image * p.pixels * p.ldy + c0 : ((long long)image * p.channels + c0) * p.pixels);
        float mean = 0.0f, variance = 0.0f;
        double seen = 0.0;
        Coefficients<1> own;
        auto ask = [&](int c) {
            if (WHAT != SUMS && c < p.per) own.ask(p, image, c0 + c);
        };
        ask(threadIdx.x);
        Parts parts;  // (what comes back first is asked for first)
        if (WHAT == APPLY) parts.ask(p.parts + (long long)which * (int)p.split, (int)p.split);
        auto prepare = [&]() {  // slopes and lifts of the group's channels
            const float scale = 1.0f / sqrtf(variance + p.eps);
            if (WHAT == APPLY) __syncthreads();  // (the job before may still read them)
            for (int c = threadIdx.x; c < p.per; c += THREADS) {
                own.make(scale, slopes + c, lifts + c);
                ask(c + THREADS);
            }
            __syncthreads();
        };
        for (long long at = first; at < last; at += TILE) {
            const long long e0 = at + threadIdx.x * UNIT;
            const int left = (int)(min((long long)TILE, last - at) - threadIdx.x * UNIT);  // (numbers of the tile from the thread's first one on)
            const float *x = X + e0;
            float *y = Y + e0;
            // (the tile's first number by the workgroup, the thread's in 32 bits)
            const unsigned hi_at = WHAT == WHOLE ? 0 : (unsigned)(at / inner), lo_at = (WHAT == WHOLE ? 0 : (unsigned)(at % inner)) + threadIdx.x * UNIT;
            const int hi0 = hi_at + lo_at / inner, lo0 = lo_at % inner;
            Unit<UNIT> v[NV];
            int hi = hi0, lo = lo0;
            float sum = 0.0f;
            auto advance = [&]() {
                hi += step_hi;
                lo += step_lo;
                if ((unsigned)lo >= inner) {
                    lo -= inner;
                    hi++;
                }
            };
#pragma unroll
            for (int k = 0; k < NV; k++) {
#pragma unroll
                for (int i = 0; i < UNIT; i++) v[k].v[i] = 0.0f;
                if (k * STEP < left) v[k] = get<UNIT>(ROWS ? X + hi * p.ldx + lo : x + k * STEP);
                if (ROWS) {
                    advance();
                    asm volatile("" : "+v"(hi), "+v"(lo));  // (one place that goes on: all of them at once take registers)
                }
            }
            if (WHAT == APPLY && at == first) {  // (while the first numbers are on their way)
                parts.join((int)p.split, p.part, count, mean, variance);
                prepare();
            }
            if (WHAT != APPLY) {
#pragma unroll
                for (int k = 0; k < NV; k++) {
                    if constexpr (UNIT == 4) sum += (v[k].v[0] + v[k].v[1]) + (v[k].v[2] + v[k].v[3]);
                    else if constexpr (UNIT == 2) sum += v[k].v[0] + v[k].v[1];
                    else sum += v[k].v[0];
                }
                const float n = (float)min((long long)TILE, last - at), nth = 1.0f / n;
                float mean_n = block_sum<THREADS>(sum, red) * nth, variance_n;
                float2 off = {0.0f, 0.0f};
#pragma unroll
                for (int k = 0; k < NV; k++)
                    if (k * STEP < left) {
#pragma unroll
                        for (int i = 0; i < UNIT; i++) {
                            const float d = v[k].v[i] - mean_n;
                            off.x += d;
                            off.y = __builtin_fmaf(d, d, off.y);
                        }
                    }
                settle(mean_n, variance_n, nth, block_sum<THREADS>(off, red));
                if (WHAT == SUMS) {
                    join(seen, mean, variance, n, mean_n, variance_n);
                } else {
                    mean = mean_n;
                    variance = variance_n;
                    prepare();
                }
            }
            if (WHAT != SUMS) {
                hi = hi0;
                lo = lo0;
#pragma unroll
                for (int k = 0; k < NV; k++) {
                    if (k * STEP < left) {
                        // (numbers read together lie in one channel of a map where its pixels are a multiple of them)
                        const bool alike = !ROWS && whole_units;
                        float slope = slopes[ROWS ? lo : hi], lift = lifts[ROWS ? lo : hi];
#pragma unroll
                        for (int i = 0; i < UNIT; i++) {
                            if (i && !alike) {
                                const int c = ROWS ? lo + i : hi + ((unsigned)(lo + i) >= inner ? 1 : 0);
                                slope = slopes[c];
                                lift = lifts[c];
                            }
                            v[k].v[i] = activated(__builtin_fmaf(v[k].v[i] - mean, slope, lift), p);
                        }
                        set<UNIT>(ROWS ? Y + hi * p.ldy + lo : y + k * STEP, v[k], p.lines);
                    }
                    advance();
                    asm volatile("" : "+v"(hi), "+v"(lo));
                }
            }
        }
        if (WHAT == SUMS && threadIdx.x == 0) p.parts[(long long)which * (int)p.split + (int)piece] = float2{mean, variance};
    }
}

// Rows of tokens whose groups are not wide: a thread stays in its columns.  ONE: a workgroup a group; otherwise several groups side by side, whose
// pieces of a row would be short.
template <int THREADS, int NV, int UNIT, bool ONE, int WHAT>
__global__ __launch_bounds__(THREADS) void group_norm_rows_kernel(const GroupNormParams p) {
    __shared__ float2 red[ONE ? THREADS / 64 : THREADS], stat[ONE ? 1 : 2 * SHORT];
    for (long long id = blockIdx.x; id < xcd_padded(p.jobs); id += gridDim.x) {
        long long job = xcd_job(id);
        if (job >= p.jobs) continue;
        if (WHAT == APPLY) job = p.jobs - 1 - job;
        const unsigned which = (unsigned)job / p.blocks, piece = which % p.split;  // (fewer than 2^31 jobs; pieces of the same rows one after another)
        const int image = which / p.split, g0 = (int)((unsigned)job % p.blocks) * p.together, here = ONE ? 1 : min(p.together, (int)p.groups - g0);
        const int units = p.per / UNIT, wide = here * units, rows_at_once = THREADS / wide;  // (of a group, of a row, rows of a step)
        const int tr = threadIdx.x / wide, cu = threadIdx.x % wide, g = ONE ? 0 : cu / units, c = g0 * p.per + cu * UNIT;
        const bool mine = tr < rows_at_once;
        const long long first = piece * p.part, last = min((long long)p.pixels, first + p.part), total = (long long)p.per * p.pixels;
        const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
        // the sums of the groups over all threads; of several groups by the wavefronts in turn
        auto group_sum = [&](auto x) {
            using T = decltype(x);
            if constexpr (ONE) {
                return block_sum<THREADS>(x, red);
            } else {
                T *all = reinterpret_cast<T *>(red), *sums = reinterpret_cast<T *>(stat);
                __syncthreads();
                all[threadIdx.x] = x;
                __syncthreads();
                for (int j = wave; j < here; j += THREADS / 64) {
                    T s = T();
                    for (int k = lane; k < rows_at_once * units; k += 64) add(s, all[k / units * wide + j * units + k % units]);
                    s = wave_sum(s);
                    if (lane == 0) sums[j] = s;
                }
                __syncthreads();
                return sums[mine ? g : 0];
            }
        };
        float mean = 0.0f, variance = 0.0f, slope[UNIT], lift[UNIT];
        double seen = 0.0;
        Coefficients<UNIT> own;
        if (WHAT != SUMS && mine) own.ask(p, image, c);
        const float2 *all_parts = p.parts + ((long long)image * (int)p.groups + g0) * (int)p.split;
        Parts parts;  // (what comes back first is asked for first)
        if (WHAT == APPLY && ONE) parts.ask(all_parts, (int)p.split);
        auto prepare = [&]() {
            if (mine) own.make(1.0f / sqrtf(variance + p.eps), slope, lift);
        };
        for (long long at = first; at < last; at += (long long)rows_at_once * NV) {
            const long long step_x = rows_at_once * p.ldx, step_y = rows_at_once * p.ldy;
            const long long row0 = (long long)image * p.pixels + at + tr;
            const int left = mine ? (int)min((long long)rows_at_once * NV, last - at) - tr : 0;  // (rows of the tile from the thread's first one on)
            const float *x = p.X + row0 * p.ldx + c;
            float *y = p.Y + row0 * p.ldy + c;
            Unit<UNIT> v[NV];
            float sum = 0.0f;
#pragma unroll
            for (int k = 0; k < NV; k++) {
#pragma unroll
                for (int i = 0; i < UNIT; i++) v[k].v[i] = 0.0f;
                if (k * rows_at_once < left) v[k] = get<UNIT>(x);
                x += step_x;
                asm volatile("" : "+v"(x));  // (one place that goes on: all of them at once take two registers each)
            }
            if (WHAT == APPLY && at == first) {  // (while the first numbers are on their way)
                if constexpr (ONE) {
                    parts.join((int)p.split, p.part * p.per, total, mean, variance);
                } else {
                    __syncthreads();
                    for (int j = wave; j < here; j += THREADS / 64) {
                        parts.ask(all_parts + j * (int)p.split, (int)p.split);
                        parts.join((int)p.split, p.part * p.per, total, mean, variance);
                        if (lane == 0) stat[j] = float2{mean, variance};
                    }
                    __syncthreads();
                    mean = stat[mine ? g : 0].x;
                    variance = stat[mine ? g : 0].y;
                }
                prepare();
            }
#pragma unroll
            for (int k = 0; k < NV; k++) {
                if constexpr (UNIT == 4) sum += (v[k].v[0] + v[k].v[1]) + (v[k].v[2] + v[k].v[3]);
                else if constexpr (UNIT == 2) sum += v[k].v[0] + v[k].v[1];
                else sum += v[k].v[0];
            }
            if (WHAT != APPLY) {
                const double n = (double)min((long long)rows_at_once * NV, last - at) * p.per;
                const float nth = 1.0f / (float)n;
                float mean_n = group_sum(sum) * nth, variance_n;
                float2 off = {0.0f, 0.0f};
#pragma unroll
                for (int k = 0; k < NV; k++)
                    if (k * rows_at_once < left) {
#pragma unroll
                        for (int i = 0; i < UNIT; i++) {
                            const float d = v[k].v[i] - mean_n;
                            off.x += d;
                            off.y = __builtin_fmaf(d, d, off.y);
                        }
                    }
                settle(mean_n, variance_n, nth, group_sum(off));
                if (WHAT == SUMS) {
                    join(seen, mean, variance, n, mean_n, variance_n);
                } else {
                    mean = mean_n;
                    variance = variance_n;
                    prepare();
                }
            }
            if (WHAT != SUMS) {
#pragma unroll
                for (int k = 0; k < NV; k++) {
                    if (k * rows_at_once < left) {
#pragma unroll
                        for (int i = 0; i < UNIT; i++) v[k].v[i] = activated(__builtin_fmaf(v[k].v[i] - mean, slope[i], lift[i]), p);
                        set<UNIT>(y, v[k], p.lines);
                    }
                    y += step_y;
                    asm volatile("" : "+v"(y));
                }
            }
        }
        if (WHAT == SUMS && tr == 0 && cu % units == 0) p.parts[((long long)image * (int)p.groups + g0 + g) * (int)p.split + (int)piece] = float2{mean, variance};
    }
}

typedef void (*Kernel)(GroupNormParams);

// A workgroup for every part of `groups` groups (or of groups taken together).
int launch(int dev, GroupNormParams &p, Kernel fn, int threads, long long groups, size_t lds) {
    p.jobs = groups * p.split;
    hipLaunchKernelGGL(fn, dim3(xcd_grid(p.jobs, threads)), dim3(threads), lds, state(dev).stream, p);
    EH_CHECK_LAUNCH();
    return 0;
}

// Sums and outputs of divided groups.
int launch_divided(int dev, GroupNormParams &p, Kernel sums, Kernel apply, long long groups, size_t lds) {
    void *ws = nullptr;
    EH_TRY(get_workspace(dev, (size_t)p.images * p.groups * p.split * sizeof(float2), &ws));
    p.parts = (float2 *)ws;
    EH_TRY(launch(dev, p, sums, 256, groups, 0));
    return launch(dev, p, apply, 256, groups, lds);
}

constexpr int WORKGROUPS = 4096;  // after which groups are not divided further

// The kernels of a group of `count` numbers: the smallest workgroup that holds it in registers, up to 32 numbers a thread.
struct Size {
    int threads, numbers;  // of a thread
    Kernel fn;
};
template <int UNIT, bool ROWS>
int launch_groups(int dev, GroupNormParams &p) {
    constexpr int NV = 32 / UNIT;
    static const Size sizes[] = {{256, 4, group_norm_kernel<256, 4 / UNIT, UNIT, ROWS, WHOLE>},   {256, 8, group_norm_kernel<256, 8 / UNIT, UNIT, ROWS, WHOLE>},
                                 {256, 16, group_norm_kernel<256, 16 / UNIT, UNIT, ROWS, WHOLE>}, {256, 32, group_norm_kernel<256, NV, UNIT, ROWS, WHOLE>},
                                 {512, 32, group_norm_kernel<512, NV, UNIT, ROWS, WHOLE>},        {1024, 32, group_norm_kernel<1024, NV, UNIT, ROWS, WHOLE>}};
    const long long count = (long long)p.per * p.pixels, groups = (long long)p.images * p.groups;
    const size_t lds = 2 * p.per * sizeof(float);
    p.split = 1;
    p.part = count;
    for (const Size &s : sizes)
        if (count <= (long long)s.threads * s.numbers) return launch(dev, p, s.fn, s.threads, groups, lds);
    constexpr int TILE = 256 * 16;  // parts of half of what a workgroup's registers hold (maps of 2 x 256 x 64 x 64, 32 channels a group: 13.0 -> 12.1 us; of a quarter 1 x 64 x 256 x 256 15 -> 17)
    const long long tiles = (count + TILE - 1) / TILE, parts = std::max(1LL, std::min<long long>({tiles, MOST_PARTS, WORKGROUPS / groups}));
    p.part = (tiles + parts - 1) / parts * TILE;
    p.split = (unsigned)((count + p.part - 1) / p.part);
    return launch_divided(dev, p, group_norm_kernel<256, NV, UNIT, ROWS, SUMS>, group_norm_kernel<256, NV, UNIT, ROWS, APPLY>, groups, lds);
}

template <int UNIT, bool ONE>
int launch_rows(int dev, GroupNormParams &p) {
    constexpr int NV = 32 / UNIT;
    static const Size sizes[] = {{256, 4, group_norm_rows_kernel<256, 4 / UNIT, UNIT, ONE, WHOLE>},   {256, 8, group_norm_rows_kernel<256, 8 / UNIT, UNIT, ONE, WHOLE>},
                                 {256, 16, group_norm_rows_kernel<256, 16 / UNIT, UNIT, ONE, WHOLE>}, {256, 24, group_norm_rows_kernel<256, 24 / UNIT, UNIT, ONE, WHOLE>},
                                 {256, 32, group_norm_rows_kernel<256, NV, UNIT, ONE, WHOLE>},        {512, 32, group_norm_rows_kernel<512, NV, UNIT, ONE, WHOLE>},
                                 {1024, 32, group_norm_rows_kernel<1024, NV, UNIT, ONE, WHOLE>}};
    p.together = ONE ? 1 : std::min((int)p.groups, (2 * SHORT + p.per - 1) / p.per);
    p.blocks = (p.groups + p.together - 1) / p.together;
    const int wide = p.together * p.per / UNIT;  // units of a row
    const long long groups = (long long)p.images * p.blocks;
    p.split = 1;
    p.part = p.pixels;
    for (const Size &s : sizes)
        if (p.pixels <= (long long)(s.threads / wide) * (s.numbers / UNIT)) return launch(dev, p, s.fn, s.threads, groups, 0);
    const int tile = 256 / wide * NV / 2;  // rows: parts of half of what a workgroup's registers hold (1 and 4 x 4096 x 640, 20 channels a group: 15.6 -> 14.3 us and 32 -> 29)
    const long long tiles = (p.pixels + tile - 1) / tile, parts = std::max(1LL, std::min<long long>({tiles, MOST_PARTS, WORKGROUPS / groups}));
    p.part = (tiles + parts - 1) / parts * tile;
    p.split = (unsigned)((p.pixels + p.part - 1) / p.part);
    return launch_divided(dev, p, group_norm_rows_kernel<256, NV, UNIT, ONE, SUMS>, group_norm_rows_kernel<256, NV, UNIT, ONE, APPLY>, groups, 0);
}

// Maps: a group is a number of UNITs, which meet two channels at most.
int launch_maps(int dev, GroupNormParams &p) {
    const long long count = (long long)p.per * p.pixels;
    if (count % 4 == 0 && p.pixels >= 4) return launch_groups<4, false>(dev, p);
    if (count % 2 == 0 && p.pixels >= 2) return launch_groups<2, false>(dev, p);
    return launch_groups<1, false>(dev, p);
}
template <int UNIT>
int launch_tokens(int dev, GroupNormParams &p) {
    if (p.per < SHORT && p.groups > 1) return launch_rows<UNIT, false>(dev, p);
    return p.per / UNIT <= 32 ? launch_rows<UNIT, true>(dev, p) : launch_groups<UNIT, true>(dev, p);  // (an eighth of the threads idle at most)
}

}  // namespace

extern "C" int eddlhip_group_norm(int dev, const float *X, long long ldx, float *Y, long long ldy, int images, int channels, int pixels, int channels_last, int groups,
                                  const float *w, const float *b, float eps, const float *mod, const float *shift, int activation) {
    EH_REQUIRE(images >= 0 && channels > 0 && pixels > 0, "group_norm: %d images of %d channels of %d pixels", images, channels, pixels);
    EH_REQUIRE(groups > 0 && channels % groups == 0 && channels / groups <= MOST_CHANNELS, "group_norm: %d channels in %d groups (of up to %d)", channels, groups, MOST_CHANNELS);
    EH_REQUIRE((long long)images * pixels <= 0x7fffffffLL && (long long)images * channels <= 0x7fffffffLL, "group_norm: %d images of %d channels of %d pixels are out of range", images, channels, pixels);
    EH_REQUIRE(activation == EDDLHIP_ACT_NONE || activation == EDDLHIP_ACT_RELU || activation == EDDLHIP_ACT_SILU || activation == EDDLHIP_ACT_RELU_LAYER, "group_norm: unknown activation %d", activation);
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
    p.activation = activation == EDDLHIP_ACT_RELU_LAYER ? EDDLHIP_ACT_RELU : activation;
    p.of_nan = activation == EDDLHIP_ACT_RELU_LAYER ? 0.0f : NAN;
    p.per = channels / groups;
    p.parts = nullptr;
    p.together = 1;
    p.blocks = groups;
    p.eps = eps;
    p.lines = !channels_last || (p.per % 32 == 0 && ldy % 32 == 0 && (uintptr_t)Y % 128 == 0);
    if (!channels_last) return launch_maps(dev, p);
    return p.per % 4 == 0 ? launch_tokens<4>(dev, p) : p.per % 2 == 0 ? launch_tokens<2>(dev, p) : launch_tokens<1>(dev, p);
}
