// Attention of new tokens over a paged cache, in fp32 accuracy on the 16-bit matrix instructions.
//
// Row i of a sequence's `new` query rows stands at position p = length - new + i.  With the visible tokens j (j < length; causal:
// j <= p; window: j > p - window)
//     s_j = scale q . k_j,   o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),   m = max_j s_j,   and o = 0 where nothing is visible.
// One pass over the tokens with running maximum, sum and output; all three in fp32.  The exponentials are powers of two: log2(e)
// goes into the scores together with the scale.
//
// Two kernels: attend_few_kernel for up to 32 rows (a token's query heads of one key head are rows side by side), which is bound by the
// cache's bytes, and attend_chunk_kernel for more, which is bound by the matrix instruction.  A long sequence with few rows is
// divided over workgroups, whose parts are joined.
//
// Both products are formed transposed, S^T = K Q^T and O^T = V^T P^T, so that a query is a column: a lane holds scores of one query in
// registers, the maximum of a query is that of two or four lanes, the rescaling of the output is one factor a lane.  And S^T is the
// second product's operand as it stands: a lane needs eight consecutive tokens of its query, which it has when the rows of K are read
// in the right order (with 32 rows, row 8a + 4h + i of the product is token 16 (a / 2) + 8h + 4 (a % 2) + i; with 16, row 4g + i of
// tile t is token 8g + 4t + i).  No score ever moves between lanes.
//
// The cache is kept in the order in which these operands are read (eddlhip.h): a lane's operand is 16 (32) bytes side by side, and
// the lanes' operands are side by side too.
//
// What is not visible has no influence beyond fp32 rounding.  Masked scores are replaced, values that no row of a tile sees are
// replaced by zeros.  Other numbers share exponents with their neighbours in the kernel of many rows: rows that lose bits by that are computed
// again in fp32 (attend_rows_fp32).  A NaN or infinity in a visible or masked place of a tile otherwise reaches the sums as NaN (0 * inf, or the
// parts of an infinity), and rows whose sums are not finite are computed again one token at a time (attend_row_again), with
// what the formula gives - in the kernel of many rows only those that fp32 leaves with a finite sum of weights (2048 tokens over 8192
// that all see a NaN: among the keys 3.7 ms, among the values 259).
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "common.h"
#include "sequence_rows.h"
#include "split_parts.h"

using namespace eddlhip;

namespace {

typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef unsigned short ushortx2 __attribute__((ext_vector_type(2)));

constexpr int TILE_KV = 32;  // tokens of a step
constexpr int MAX_TOKENS = 1 << 30;
constexpr float NEG_INF = -__builtin_inff();

struct AttendParams {
    const float *Q;
    float *O;
    const void *K, *V;
    const int *table, *offsets, *lengths;
    float *part_o;   // [splits][part_rows][D]
    float2 *part_s;  // [splits][part_rows] maximum and sum
    long long ldq, ldo, part_rows;  // part_rows: rows * q_heads, or the rows of the launch's tiles where the last workgroup joins
    int rows, q_heads, kv_heads, group, D, pages, page_shift, width, seqs, causal, window, splits, q_tiles, vec, grouped;
    float scale;  // with log2(e)
};

// A sequence's part of the batch, from the device's arrays, kept within the buffers whatever those hold.
struct Sequence {
    int row0, fresh, length;
    bool bad;  // longer than its row of the table, or negative
};
__device__ __forceinline__ Sequence sequence_of(const AttendParams &p, int s) {
    Sequence q;
    const int begin = p.offsets[s], end = p.offsets[s + 1];
    int length = p.lengths[s];
    asm volatile("" : "+s"(length));  // (asked for together with the offsets, not behind a branch on them: 1 token over 50 6.1 -> 5.9 us)
    const SequenceRows r = sequence_rows(begin, end, p.rows);
    q.row0 = r.row0;
    q.fresh = r.fresh;
    q.length = length;
    q.bad = q.length < 0 || (long long)q.length > ((long long)p.width << p.page_shift);
    if (q.bad) q.length = 0;
    return q;
}

// Element offset of 16 tokens of a key head; a page that is not in the pool gives `bad` and the place of page 0.  (16 tokens that a tile's rows have
// behind their windows are asked for there too, whatever the table holds: a program may have released their page.  Their numbers do not count.)
__device__ __forceinline__ size_t block_base(const AttendParams &p, int page, int block16, int head, bool &bad) {
    if ((unsigned)page >= (unsigned)p.pages) {
        bad = true;
        page = 0;
    }
    const int in_page = block16 & ((1 << (p.page_shift - 4)) - 1);
    return ((((size_t)page * p.kv_heads + head) << (p.page_shift - 4)) + in_page) * (16 * p.D);
}

template <bool F32>
struct Raw;
template <>
struct Raw<false> {
    uintx4 v;
    // ONCE: with the streaming hint, where no other wavefront reads the number
    template <bool ONCE = false>
    __device__ __forceinline__ void load(const void *base, size_t at) {
        const uintx4 *src = reinterpret_cast<const uintx4 *>((const unsigned short *)base + at);
        v = ONCE ? __builtin_nontemporal_load(src) : *src;
    }
    // tokens from `count` of the eight on are zeros
    __device__ __forceinline__ void keep(int count) {
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = 2 * i + 1 < count ? v[i] : 2 * i < count ? v[i] & 0xffffu : 0u;
    }
    __device__ __forceinline__ void numbers(float (&x)[8]) const {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            x[2 * i] = __builtin_bit_cast(float, v[i] << 16);
            x[2 * i + 1] = __builtin_bit_cast(float, v[i] & 0xffff0000u);
        }
    }
    __device__ __forceinline__ unsigned largest() const {  // the bits of the largest magnitude (of a NaN, if there is one)
        ushortx2 m = __builtin_bit_cast(ushortx2, v[0] & 0x7fff7fffu);
#pragma unroll
        for (int i = 1; i < 4; i++) m = __builtin_elementwise_max(m, __builtin_bit_cast(ushortx2, v[i] & 0x7fff7fffu));
        return (unsigned)max(m[0], m[1]) << 16;
    }
};
template <>
struct Raw<true> {
    floatx4 lo, hi;
    template <bool ONCE = false>
    __device__ __forceinline__ void load(const void *base, size_t at) {
        const floatx4 *src = reinterpret_cast<const floatx4 *>((const float *)base + at);
        lo = ONCE ? __builtin_nontemporal_load(src) : src[0];
        hi = ONCE ? __builtin_nontemporal_load(src + 1) : src[1];
    }
    __device__ __forceinline__ void keep(int count) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            lo[i] = i < count ? lo[i] : 0.0f;
            hi[i] = 4 + i < count ? hi[i] : 0.0f;
        }
    }
    __device__ __forceinline__ void numbers(float (&x)[8]) const {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            x[i] = lo[i];
            x[4 + i] = hi[i];
        }
    }
    __device__ __forceinline__ unsigned largest() const {  // the bits of the largest magnitude, NaN left out
        float m = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; i++) m = fmaxf(fmaxf(m, fabsf(lo[i])), fabsf(hi[i]));
        return __builtin_bit_cast(unsigned, m);
    }
};

struct Parts {
    uintx4 p[3];
};
__device__ __forceinline__ Parts split8(const float (&x)[8]) {
    Parts s;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        unsigned h, m, l;
        split_pair(x[2 * i], x[2 * i + 1], h, m, l);
        s.p[0][i] = h;
        s.p[1][i] = m;
        s.p[2][i] = l;
    }
    return s;
}
__device__ __forceinline__ float power2(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float element(const AttendParams &p, const void *base, size_t at, bool f32) {
    return f32 ? ((const float *)base)[at] : __builtin_bit_cast(float, (unsigned)((const unsigned short *)base)[at] << 16);
}

// Parts of a divided length are written past the caches of an XCD and read so by the workgroup that joins them.
__device__ __forceinline__ void put_part(float *dst, float a, float b) {
    const float2 x = make_float2(a, b);
    __hip_atomic_store((unsigned long long *)dst, __builtin_bit_cast(unsigned long long, x), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 get_part(const float *src) {
    return __builtin_bit_cast(float2, __hip_atomic_load((const unsigned long long *)src, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
}

// Where a row's result goes: the output, or its partial result.
__device__ __forceinline__ void store_scale(const AttendParams &p, float m, float l, float &factor) {
    // (no visible token: m = -inf, l = 0, o = 0; visible ones that are all -inf: l > 0 and o = NaN, as the formula)
    factor = m == NEG_INF && l == 0.0f ? 0.0f : 1.0f / l;
}

// One row over the tokens [lo, hi), a wavefront together, one token at a time: lanes hold the dimensions lane, lane + 64, ...
template <bool F32>
__device__ void attend_row_again(const AttendParams &p, const Sequence &q, int seq, int kv_head, int token, int head, int lo, int hi, size_t slot, int splits, bool bad) {
    const int lane = threadIdx.x & 63, pos = q.length - q.fresh + token;
    if (p.causal) hi = min(hi, pos + 1);
    if (p.window > 0) lo = max(lo, pos - p.window + 1);
    const float *qrow = p.Q + (size_t)(q.row0 + token) * p.ldq + (size_t)head * p.D;
    float x[4], o[4] = {0.0f, 0.0f, 0.0f, 0.0f}, m = NEG_INF, l = 0.0f;
    for (int i = 0; i < 4; i++) x[i] = lane + 64 * i < p.D ? qrow[lane + 64 * i] * p.scale : 0.0f;
    for (int j = lo; j < hi; j++) {
        const size_t base = block_base(p, p.table[(size_t)seq * p.width + (j >> p.page_shift)], j >> 4, kv_head, bad);
        float s = 0.0f;
        for (int i = 0; i < 4; i++) {
            const int d = lane + 64 * i;
            if (d < p.D) s += x[i] * element(p, p.K, base + (d >> 3) * 128 + (j & 15) * 8 + (d & 7), F32);
        }
        for (int step = 32; step > 0; step >>= 1) s += __shfl_xor(s, step);
        const float top = s > m || s != s ? s : m;  // a NaN stays
        const float keep = top == NEG_INF ? 1.0f : power2(m - top), w = top == NEG_INF ? 0.0f : power2(s - top);
        l = l * keep + (top == NEG_INF ? 1.0f : w);
        if (top != NEG_INF && m == NEG_INF) l = w;
        for (int i = 0; i < 4; i++) {
            const int d = lane + 64 * i;
            if (d < p.D) o[i] = (m == NEG_INF ? 0.0f : o[i] * keep) + w * element(p, p.V, base + ((j >> 3) & 1) * 8 * p.D + d * 8 + (j & 7), F32);
        }
        m = top;
        if (bad || m != m) break;  // (the row is NaN, whatever comes)
    }
    if (bad) l = __builtin_nanf("");
    if (splits > 1) {
        if (lane == 0) put_part((float *)(p.part_s + slot), m, l);
        for (int i = 0; i < 4; i++)
            if (lane + 64 * i < p.D) __hip_atomic_store(p.part_o + slot * p.D + lane + 64 * i, o[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    } else {
        float factor;
        store_scale(p, m, l, factor);
        if (m == NEG_INF && l > 0.0f) factor = __builtin_nanf("");
        for (int i = 0; i < 4; i++)
            if (lane + 64 * i < p.D) p.O[(size_t)(q.row0 + token) * p.ldo + (size_t)head * p.D + lane + 64 * i] = o[i] * factor;
    }
}

// The tokens that any row of a tile sees, and the bounds that all of them share.
struct Range {
    int lo, hi;            // tokens of the tile's rows (lo on a boundary of TILE_KV)
    int first;             // the first of them, where it is
    int all_lo, all_hi;    // every row sees [all_lo, all_hi)
};
__device__ __forceinline__ Range range_of(const AttendParams &p, const Sequence &q, int row_lo, int row_hi) {
    const int first = q.length - q.fresh + row_lo / p.group, last = q.length - q.fresh + (row_hi - 1) / p.group;
    Range r;
    r.hi = p.causal ? min(q.length, last + 1) : q.length;
    r.all_hi = p.causal ? min(q.length, first + 1) : q.length;
    r.first = p.window > 0 ? max(0, first - p.window + 1) : 0;
    r.all_lo = p.window > 0 ? max(0, last - p.window + 1) : 0;
    r.lo = r.first & ~(TILE_KV - 1);
    return r;
}

// Step at which part `n` of `parts` begins: parts differ by at most one step.
__device__ __forceinline__ int part_at(int steps, int n, int parts) {
    const int each = (int)((unsigned)steps / (unsigned)parts), more = steps - each * parts;
    return n * each + min(n, more);
}

// ------------------------------------------------------------------------------------------------ divided lengths
// Few rows in up to 64 parts: workgroups that share rows count themselves in when their parts have reached the memory that all XCDs see;
// the one that completes the count joins the parts, in groups that the shape alone fixes.  Nobody waits for another, and the
// bits do not depend on who comes last.  A launch less: one token over 4096 28.6 -> 20.7 us.
// Many rows, or more parts, are joined by a launch of their own, which the whole device works on (4 x 196 rows of 8 heads in 6 parts: 9 us
// where the last workgroups took 19).  Where the last workgroup joins, rows that the launch did not count on (beyond q_tiles) are not divided.
// (One array for all launches on the device, zeros between them: they come one after another, on one stream, and eddlhip_set_stream
// waits for the old one's.)
constexpr int MAX_COUNTS = 1024;  // divided launches have no more row tiles: two workgroups a tile fill the device
static __device__ unsigned part_counts[MAX_COUNTS];

constexpr int JOIN_HERE = 64;  // most parts that are joined so
constexpr size_t MOST_PARTS = (size_t)1 << 30;  // bytes of the parts that a launch joins
// `sums`: LDS of rows x parts; `red`: LDS of THREADS.
template <int THREADS>
__device__ __forceinline__ void join_parts(const AttendParams &p, const Sequence &q, int kv_head, int row_lo, int row_hi, float2 *sums, floatx4 *red, unsigned count,
                                           size_t slot, int *last) {  // slot: the tile's first in a part
    const int tid = threadIdx.x, n = row_hi - row_lo, parts = p.splits, quads = p.D >> 2;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (tid == 0) {
        const unsigned before = __hip_atomic_fetch_add(&part_counts[count], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        *last = before == (unsigned)parts - 1;
        if (before == (unsigned)parts - 1) __hip_atomic_store(&part_counts[count], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // as the next launch expects it
    }
    __syncthreads();
    if (!*last) return;
    const size_t total = p.part_rows;
    for (int i = tid; i < n * parts; i += THREADS) {
        const int r = i / parts, s = i - r * parts;
        sums[i] = get_part((const float *)(p.part_s + s * total + slot + r));
    }
    __syncthreads();
    // four dimensions of a row a thread, or several threads where there are few
    const int items = n * quads, lanes = items > THREADS / 2 ? 1 : THREADS / items;
    for (int i0 = 0; i0 < items; i0 += THREADS) {
        const int i = lanes > 1 ? tid % items : i0 + tid, lane = lanes > 1 ? tid / items : 0, r = i / quads, d = 4 * (i - r * quads);
        const bool works = i < items && lane < lanes;
        float m = NEG_INF, l = 0.0f;
        floatx4 o = {0.0f, 0.0f, 0.0f, 0.0f};
        if (works) {
            const float2 *ms = sums + r * parts;
#pragma unroll 8
            for (int s = 0; s < parts; s++) m = fmaxf(m, ms[s].x);
            const float *src = p.part_o + (slot + r) * p.D + d;
            constexpr int AHEAD = 16;
            for (int s0 = lane; s0 < parts; s0 += AHEAD * lanes) {
                float2 a[AHEAD], b[AHEAD];
#pragma unroll
                for (int k = 0; k < AHEAD; k++) {
                    const int s = min(s0 + k * lanes, parts - 1);
                    a[k] = get_part(src + s * total * p.D);
                    b[k] = get_part(src + s * total * p.D + 2);
                }
#pragma unroll
                for (int k = 0; k < AHEAD; k++) {
                    const int s = s0 + k * lanes;
                    if (s < parts) {
                        const float2 x = ms[s];
                        const float w = x.x == NEG_INF && x.y == 0.0f ? 0.0f : m == NEG_INF ? 1.0f : power2(x.x - m);
                        l += w * x.y;
                        o += floatx4{a[k].x, a[k].y, b[k].x, b[k].y} * w;
                    }
                }
            }
        }
        if (lanes > 1) {
            __syncthreads();  // (all have read the sums)
            red[tid] = o;
            ((float *)sums)[tid] = l;
            __syncthreads();
            if (works && lane == 0)
                for (int k = 1; k < lanes; k++) {
                    o += red[k * items + i];
                    l += ((float *)sums)[k * items + i];
                }
        }
        if (works && lane == 0) {
            float factor;
            store_scale(p, m, l, factor);
            if (m == NEG_INF && l != 0.0f) factor = __builtin_nanf("");
            const int row = row_lo + r, token = row / p.group;
            float *dst = p.O + (size_t)(q.row0 + token) * p.ldo + (size_t)(kv_head * p.group + row % p.group) * p.D + d;
            o *= factor;
            if (p.vec) {
                *reinterpret_cast<floatx4 *>(dst) = o;
            } else {
#pragma unroll
                for (int k = 0; k < 4; k++) dst[k] = o[k];
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------ few rows
// Up to 16 NQ rows of a sequence and key head (single tokens, short drafts): bound by the cache's bytes.  A workgroup takes a part of the
// tokens, its four or eight wavefronts take steps of 32 tokens in turn, operands straight from the cache into registers: every byte is read
// once, by one wavefront, so LDS would only add a trip.  Keys of the next step are asked for as soon as the products have
// used this step's, values likewise, into the same registers: a step's loads are on their way while the other half of a step is
// computed, 16 (32) KB a wavefront.  The 16x16x32 instruction keeps the queries that are not there at 15 of 16 columns
// instead of 31 of 32, and the registers at half.  The wavefronts' sums meet in LDS once.
// The matrix instruction has time to spare, so every fp32 operand (queries, weights, an fp32 cache) is the sum of three bf16 numbers
// (split_parts.h), six products for an fp32 cache and three for a bf16 one, whose sum has no rounding but the accumulator's; no
// exponents are kept.  (Parts of numbers below 2^-110 lose bits: absolute errors of 2^-133.)
// Measured: 1 token over 131072, 8 key heads of 128 in bf16 (537 MB): 94 us, 5.7 TB/s, where a plain read stream reaches 6.9 - 7.1;
// 32 over 4096 (fp32, 1.07 GB) 186 us, 5.8 TB/s.  Without the streaming hint 104 us; a second step in flight gains nothing, more
// workgroups than the device holds at a time lose 4 to 15 %.
// Rows of the product K Q^T: row 4g + i of tile t is token 8g + 4t + i of the step, so that lane group g holds tokens 8g .. 8g + 7.
// Wavefronts of a SIMD, as the registers of a step's keys, values and outputs allow without spills, and wavefronts of a workgroup: all that a
// CU holds where that is 8 (fewer parts to join, and a part lasts as long as possible: 1 token over 131072, heads of 128 in bf16, 95 us,
// with two workgroups of 4 100 us).
constexpr int few_per_simd(int dp, bool f32, int nq) { return dp > 128 || (f32 && dp > 96) || (f32 && dp > 64 && nq > 1) ? 1 : !f32 && dp <= 64 && nq == 1 ? 3 : 2; }
constexpr int few_waves(int dp, bool f32, int nq) { return few_per_simd(dp, f32, nq) == 2 && !f32 ? 8 : 4; }
constexpr int few_groups(int dp, bool f32, int nq) { return 4 * few_per_simd(dp, f32, nq) / few_waves(dp, f32, nq); }  // workgroups of a CU
constexpr int FEW_SPLITS = 512;  // most parts of a length for up to 16 rows, half of it for up to 32

__device__ __forceinline__ floatx4 mfma16(uintx4 a, uintx4 b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <bool F32>
struct Operand;
template <>
struct Operand<false> {
    uintx4 v;
    __device__ __forceinline__ explicit Operand(const Raw<false> &r) : v(r.v) {}
    __device__ __forceinline__ void multiply(const uintx4 &b0, const uintx4 &b1, const uintx4 &b2, floatx4 &large, floatx4 &small) const {
        small = mfma16(v, b2, small);
        small = mfma16(v, b1, small);
        large = mfma16(v, b0, large);
    }
};
template <>
struct Operand<true> {
    Parts s;
    __device__ __forceinline__ explicit Operand(const Raw<true> &r) {
        const float x[8] = {r.lo[0], r.lo[1], r.lo[2], r.lo[3], r.hi[0], r.hi[1], r.hi[2], r.hi[3]};
        s = split8(x);
    }
    __device__ __forceinline__ void multiply(const uintx4 &b0, const uintx4 &b1, const uintx4 &b2, floatx4 &large, floatx4 &small) const {
        small = mfma16(s.p[0], b2, small);
        small = mfma16(s.p[1], b1, small);
        small = mfma16(s.p[2], b0, small);
        small = mfma16(s.p[0], b1, small);
        small = mfma16(s.p[1], b0, small);
        large = mfma16(s.p[0], b0, large);
    }
};

// The rows of a tile of keys: a load's or, in the odd lane groups of a bf16 cache, the other's.
__device__ __forceinline__ Raw<false> tile_rows(const Raw<false> &a, const Raw<false> &b, bool exchanged) {
    Raw<false> r;
#pragma unroll
    for (int i = 0; i < 4; i++) r.v[i] = exchanged ? b.v[i] : a.v[i];
    return r;
}
__device__ __forceinline__ const Raw<true> &tile_rows(const Raw<true> &a, const Raw<true> &, bool) { return a; }

// FULL: head_dim is DP; otherwise DP - 64 < head_dim < DP: dimensions past the last are zeros of the queries, which meet the last 8
// dimensions of the keys again, and outputs that nobody reads.  grid (q_tiles * splits, kv_heads, seqs)
template <int DP, bool F32, int NQ, bool FULL>
__global__ __launch_bounds__(64 * few_waves(DP, F32, NQ), few_per_simd(DP, F32, NQ)) void attend_few_kernel(const AttendParams p) {
    constexpr int KS = DP / 32, DT = DP / 16, W = few_waves(DP, F32, NQ), COLS = 16 * NQ, PITCH = DP + 4;
    constexpr int Q_BYTES = 3 * KS * NQ * 64 * 16, O_BYTES = W * COLS * PITCH * 4;
    constexpr int S_BYTES = COLS * JOIN_HERE * 8, MOST = Q_BYTES > O_BYTES ? Q_BYTES : O_BYTES;
    __shared__ __attribute__((aligned(16))) char lds[S_BYTES > MOST ? S_BYTES : MOST];
    __shared__ floatx4 red[64 * W];
    __shared__ int last;
    __shared__ float sums[W][COLS][2];
    __shared__ unsigned redo_columns;
    uintx4(*q_parts)[KS][NQ][64] = reinterpret_cast<uintx4(*)[KS][NQ][64]>(lds);
    float(*o_lds)[COLS][PITCH] = reinterpret_cast<float(*)[COLS][PITCH]>(lds);

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 15, g = lane >> 4;
    const int D = FULL ? DP : p.D;
    const int own_split = blockIdx.x % p.splits, kv_head = blockIdx.y, seq = blockIdx.z;
    const Sequence q = sequence_of(p, seq);
    const int rows = q.fresh * p.group;
    const int *pages = p.table + (size_t)seq * p.width;

    for (int tile = blockIdx.x / p.splits; tile * COLS < rows; tile += p.q_tiles) {
        const bool counted = tile < p.q_tiles || p.splits > JOIN_HERE;  // (a launch joins the parts of all rows)
        if (!counted && own_split != 0) break;
        const int split = counted ? own_split : 0, splits = counted ? p.splits : 1;
        const int row_lo = tile * COLS, row_hi = min(rows, row_lo + COLS);
        const Range range = range_of(p, q, row_lo, row_hi);
        const int steps_all = max(0, (range.hi - range.lo + TILE_KV - 1) / TILE_KV);
        const int step_lo = part_at(steps_all, split, splits), step_hi = part_at(steps_all, split + 1, splits);
        const int lo = range.lo + step_lo * TILE_KV, hi = min(range.hi, range.lo + step_hi * TILE_KV);
        __syncthreads();  // (the tile before has been stored)

        // ---- the cache's operands of a step
        bool bad = q.bad;
        int page_lane = 0, page_it = -64;
        Raw<F32> k[2][KS], v[DT];
        size_t base[2];
        auto find = [&](int it) __attribute__((always_inline)) {  // the wavefront's step `it`: 16 tokens' places, twice
            if (it >= page_it + 32) {
                page_it = it;
                const int j = lo + ((wave + W * (it + (lane >> 1))) * 2 + (lane & 1)) * 16;
                page_lane = pages[min(j, hi - 1) >> p.page_shift];  // (behind the last token: its page again, whose values do not count)
            }
            const int b = (lo >> 4) + (wave + W * it) * 2, at = 2 * (it - page_it);
            base[0] = block_base(p, 16 * b + 16 <= range.first ? 0 : __builtin_amdgcn_readlane(page_lane, at), b, kv_head, bad);
            base[1] = block_base(p, __builtin_amdgcn_readlane(page_lane, at + 1), b + 1, kv_head, bad);
        };
        // (bf16: lanes g and g ^ 1 read the same 8 dimensions, one the rows of tile 0 and one those of tile 1, so that a load covers whole lines;
        // the next load brings the other 8 dimensions with the tiles exchanged.  fp32 rows fill their lines by themselves.)
        auto load_keys = [&]() __attribute__((always_inline)) {
            const size_t from = (col >> 3 ? base[1] : base[0]);
#pragma unroll
            for (int n = 0; n < 2; n++) {
                const int token = (8 * (col >> 2) + 4 * (F32 ? n : (g ^ n) & 1) + (col & 3)) & 15;
#pragma unroll
                for (int ks = 0; ks < KS; ks++) {
                    const int chunk = 4 * ks + (F32 ? g : (g & 2) + n);
                    k[n][ks].template load<true>(p.K, from + token * 8 + (FULL ? chunk : min(chunk, (D >> 3) - 1)) * 128);
                }
            }
        };
        auto load_values = [&]() __attribute__((always_inline)) {
            const size_t from = (g & 2 ? base[1] : base[0]) + (size_t)(g & 1) * 8 * D;
#pragma unroll
            for (int dt = 0; dt < DT; dt++) v[dt].template load<true>(p.V, from + (FULL ? 16 * dt + col : min(16 * dt + col, D - 1)) * 8);
        };
        const int its = (step_hi - step_lo - wave + W - 1) / W;  // steps of this wavefront
        if (its > 0 && hi > lo) {
            find(0);
            load_keys();
            load_values();
        }

        // ---- queries: parts of 8 dimensions of a row a lane, in LDS, made by all wavefronts together
        for (int i = wave; i < KS * NQ; i += W) {
            const int ks = i / NQ, nq = i % NQ, row = min(row_lo + 16 * nq + col, row_hi - 1), token = row / p.group, head = kv_head * p.group + row % p.group;
            const int d = 32 * ks + 8 * g;
            float x[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
            if (d < D) {
                const float *src = p.Q + (size_t)(q.row0 + token) * p.ldq + (size_t)head * D + d;
                if (p.vec) {
                    const floatx4 a = *reinterpret_cast<const floatx4 *>(src), b = *reinterpret_cast<const floatx4 *>(src + 4);
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        x[j] = a[j] * p.scale;
                        x[4 + j] = b[j] * p.scale;
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 8; j++) x[j] = src[j] * p.scale;
                }
            }
            const Parts s = split8(x);
#pragma unroll
            for (int n = 0; n < 3; n++) q_parts[n][ks][nq][lane] = s.p[n];
        }
        if (tid == 0) redo_columns = 0;
        int see_lo[NQ], see_hi[NQ];
#pragma unroll
        for (int nq = 0; nq < NQ; nq++) {
            const int pos = q.length - q.fresh + min(row_lo + 16 * nq + col, row_hi - 1) / p.group;
            see_lo[nq] = p.window > 0 ? pos - p.window + 1 : 0;
            see_hi[nq] = p.causal ? min(q.length, pos + 1) : q.length;
        }
        __syncthreads();

        floatx4 o[NQ][DT];
        float m[NQ], l[NQ];
#pragma unroll
        for (int nq = 0; nq < NQ; nq++) {
            m[nq] = NEG_INF;
            l[nq] = 0.0f;
#pragma unroll
            for (int dt = 0; dt < DT; dt++) o[nq][dt] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
        }
        for (int it = 0; it < its; it++) {
            const int j0 = lo + (wave + W * it) * TILE_KV;
            const bool more = it + 1 < its;
            floatx4 large[NQ][2], small[NQ][2];
#pragma unroll
            for (int nq = 0; nq < NQ; nq++)
#pragma unroll
                for (int t = 0; t < 2; t++) large[nq][t] = small[nq][t] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                // rows of tile 0 with dimensions 8 (4 ks + g) .., rows of tile 1 with the same or (bf16) those of lane g ^ 1
                const Operand<F32> a0(tile_rows(k[0][ks], k[1][ks], g & 1)), a1(tile_rows(k[1][ks], k[0][ks], g & 1));
                const int other = F32 ? lane : lane ^ 16;
#pragma unroll
                for (int nq = 0; nq < NQ; nq++) {
                    a0.multiply(q_parts[0][ks][nq][lane], q_parts[1][ks][nq][lane], q_parts[2][ks][nq][lane], large[nq][0], small[nq][0]);
                    a1.multiply(q_parts[0][ks][nq][other], q_parts[1][ks][nq][other], q_parts[2][ks][nq][other], large[nq][1], small[nq][1]);
                }
                __builtin_amdgcn_sched_barrier(0);  // (one operand's parts at a time: registers)
            }
            if (more) {
                find(it + 1);
                load_keys();
            }
            __builtin_amdgcn_sched_barrier(0);
            const bool early = j0 + 16 <= range.first;  // (nobody sees the first 16: page 0 stands in for theirs)
            if (j0 + TILE_KV > q.length || early) {
#pragma unroll
                for (int dt = 0; dt < DT; dt++) v[dt].keep(early && g < 2 ? 0 : q.length - (j0 + 8 * g));
            }
            Parts ws[NQ];
#pragma unroll
            for (int nq = 0; nq < NQ; nq++) {
                float s[8];
#pragma unroll
                for (int r = 0; r < 8; r++) s[r] = large[nq][r >> 2][r & 3] + small[nq][r >> 2][r & 3];
                if (j0 < range.all_lo || j0 + TILE_KV > range.all_hi) {
#pragma unroll
                    for (int r = 0; r < 8; r++) {
                        const int j = j0 + 8 * g + r;
                        s[r] = j >= see_lo[nq] && j < see_hi[nq] ? s[r] : NEG_INF;
                    }
                }
                float top = fmaxf(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])), fmaxf(fmaxf(s[4], s[5]), fmaxf(s[6], s[7])));
                top = fmaxf(top, __shfl_xor(top, 16));
                top = fmaxf(top, __shfl_xor(top, 32));
                top = fmaxf(top, m[nq]);
                if (__any(top > m[nq])) {
                    const float keep = m[nq] == NEG_INF ? 0.0f : power2(m[nq] - top);
                    l[nq] *= keep;
#pragma unroll
                    for (int dt = 0; dt < DT; dt++) o[nq][dt] *= keep;
                    m[nq] = top;
                }
                const float from = m[nq] == NEG_INF ? 0.0f : m[nq];
#pragma unroll
                for (int r = 0; r < 8; r++) {
                    s[r] = power2(s[r] - from);
                    l[nq] += s[r];
                }
                ws[nq] = split8(s);
            }
#pragma unroll
            for (int dt = 0; dt < DT; dt++) {
                const Operand<F32> a(v[dt]);
#pragma unroll
                for (int nq = 0; nq < NQ; nq++) a.multiply(ws[nq].p[0], ws[nq].p[1], ws[nq].p[2], o[nq][dt], o[nq][dt]);
                if (F32) __builtin_amdgcn_sched_barrier(0);
            }
            if (more) load_values();
        }
        __syncthreads();  // (the queries have been read: their place takes the outputs)
#pragma unroll
        for (int nq = 0; nq < NQ; nq++) {
            l[nq] += __shfl_xor(l[nq], 16);
            l[nq] += __shfl_xor(l[nq], 32);
            if (bad) l[nq] = __builtin_nanf("");
            if (g == 0) {
                sums[wave][16 * nq + col][0] = m[nq];
                sums[wave][16 * nq + col][1] = l[nq];
            }
#pragma unroll
            for (int dt = 0; dt < DT; dt++) *reinterpret_cast<floatx4 *>(&o_lds[wave][16 * nq + col][16 * dt + 4 * g]) = o[nq][dt];
        }
        __syncthreads();

        const size_t first_slot = (size_t)((seq * p.kv_heads + kv_head) * p.q_tiles + tile) * COLS;  // (of a part that the last workgroup joins)
        auto slot_of = [&](int c) __attribute__((always_inline)) {
            const int row = row_lo + c, token = row / p.group;
            return (size_t)split * p.part_rows + (splits > JOIN_HERE ? (size_t)(q.row0 + token) * p.q_heads + kv_head * p.group + row % p.group : first_slot + c);
        };

        // ---- the wavefronts' sums together, four dimensions of a row a thread
        const int quads = D >> 2, items = (row_hi - row_lo) * quads;
        for (int i0 = 0; i0 < items; i0 += 64 * W) {
            const int i = i0 + tid, c = i / quads, d = 4 * (i - c * quads);
            if (i < items) {
                float top = sums[0][c][0];
#pragma unroll
                for (int w = 1; w < W; w++) top = fmaxf(top, sums[w][c][0]);
                float sum = 0.0f;
                floatx4 x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int w = 0; w < W; w++) {
                    const float f = sums[w][c][0] == NEG_INF ? (sums[w][c][1] == 0.0f ? 0.0f : sums[w][c][1]) : power2(sums[w][c][0] - top);
                    sum += f * sums[w][c][1];
                    x += *reinterpret_cast<const floatx4 *>(&o_lds[w][c][d]) * f;
                }
                const int row = row_lo + c, token = row / p.group, head = kv_head * p.group + row % p.group;
                const int pos = q.length - q.fresh + token, from = p.window > 0 ? max(lo, pos - p.window + 1) : lo, to = p.causal ? min(hi, pos + 1) : hi;
                const float worst = (sum - sum) + ((x[0] - x[0]) + (x[1] - x[1])) + ((x[2] - x[2]) + (x[3] - x[3]));
                if (worst != 0.0f || (top == NEG_INF && from < to)) {
                    atomicOr(&redo_columns, 1u << c);
                }
                const size_t slot = slot_of(c);
                if (splits > JOIN_HERE) {
                    if (d == 0) p.part_s[slot] = make_float2(top, sum);
                    *reinterpret_cast<floatx4 *>(p.part_o + slot * D + d) = x;
                } else if (splits > 1) {
                    if (d == 0) put_part((float *)(p.part_s + slot), top, sum);
                    put_part(p.part_o + slot * D + d, x[0], x[1]);
                    put_part(p.part_o + slot * D + d + 2, x[2], x[3]);
                } else {
                    float factor;
                    store_scale(p, top, sum, factor);
                    float *dst = p.O + (size_t)(q.row0 + token) * p.ldo + (size_t)head * D + d;
                    x *= factor;
                    if (p.vec) {
                        *reinterpret_cast<floatx4 *>(dst) = x;
                    } else {
#pragma unroll
                        for (int j = 0; j < 4; j++) dst[j] = x[j];
                    }
                }
            }
        }
        // ---- rows whose sums are not finite, and rows that see tokens but no score above -inf, one by one (behind the stores above)
        __syncthreads();
        const bool any_bad = q.bad;
        for (unsigned todo = redo_columns; todo != 0; todo &= todo - 1) {
            const int c = __builtin_ctz(todo), r = row_lo + c;
            if (c % W == wave) attend_row_again<F32>(p, q, seq, kv_head, r / p.group, kv_head * p.group + r % p.group, lo, hi, slot_of(c), splits, any_bad);
        }
        if (splits > 1 && splits <= JOIN_HERE)
            join_parts<64 * W>(p, q, kv_head, row_lo, row_hi, reinterpret_cast<float2 *>(lds), red, (seq * p.kv_heads + kv_head) * p.q_tiles + tile, first_slot, &last);
    }
}

// ------------------------------------------------------------------------------------------------ many rows
// A workgroup takes 128 or 256 rows, 32 a wavefront, and walks through its part of the tokens 32 at a time, which all its wavefronts read
// from LDS.  Bound by the matrix instruction, so its operands are pairs of fp16 numbers here and not three bf16 numbers:
// x 2^e = hi + lo, hi = fp16(x 2^e), lo = fp16(x 2^e - hi), with e such that the largest number of a row of queries, or of 16 tokens'
// keys or values of a head, lies in 2^14 .. 2^15.  Each half brings 11 bits and its sign: a pair is off by at most 2^-23 of x, or, where
// lo runs out of fp16's range, by 2^-25 of 2^-14 of the largest number, 2^-39.  A bf16 number is its own hi down to 2^-31 of the largest.
// Two pairs take three products (lo lo is left out), a pair and a bf16 number two, where the bf16 parts take six and
// three; and a pair costs 4 instructions for two numbers where three parts cost 11.  The rows' and blocks' exponents go into the scores as
// factors, and the blocks' exponents of values into the weights: a weight is exp2(s - m + c) with c = 14 + (the block's exponent) - (the largest so
// far), the output carries the largest, a whole number of doublings like m.  (14: weights of 2^-28 still have eleven bits in hi.)
// A block whose largest number is infinite takes a NaN as its factor, so that its rows are computed again.  (lo lo: each lo is 2^-11 of its number at
// most, their product 2^-22 of the whole; of numbers whose bits are even by chance 2^-25, with either sign.)
// Tiles: each of the first four wavefronts brings the keys or the values of 16 tokens, their numbers go through its registers (the largest, the pairs) into LDS;
// two tiles, one filled while the other is used, one barrier a tile.  The cache's order is the operands' order: every LDS
// access is 16 bytes a lane of 16 lanes side by side.  The queries' pairs stay in registers.
// Eight wavefronts (two on each SIMD, one of which brings tiles) halve that work for a row: 2048 tokens over 8192, 32 and 8 heads of 128, bf16
// 561 -> 516 us, 4 x 1000 over 2000, heads of 64 102 -> 86; but a ragged batch has more empty rows in tiles of 256 (35 -> 44 us).
// Measured: 2048 tokens over 8192, 32 and 8 heads of 128, bf16 cache: 508 us, 473 TFLOP/s, 950 on the matrix instructions (48 % of the
// cycles busy; the vector instructions fill 53 % and the two do not overlap: a version that computed the next tile's scores beside the
// weights in one block, with the scheduler's groups, spilled and took 890).  As three bf16 parts with tiles loaded straight into LDS 621 us.
constexpr int CHUNK_SPLITS = 64;  // most parts of a length

typedef _Float16 halfx2 __attribute__((ext_vector_type(2)));
typedef _Float16 halfx8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ floatx16 mfma(uintx4 a, uintx4 b, floatx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(halfx8, a), __builtin_bit_cast(halfx8, b), c, 0, 0, 0);
}
__device__ __forceinline__ unsigned round_half(float a, float b) {  // two fp16, rounded to nearest even
    return __builtin_bit_cast(unsigned, __builtin_convertvector((floatx2){a, b}, halfx2));
}
// Two numbers as pairs; the differences are exact, one instruction each.
__device__ __forceinline__ void pair_up(float a, float b, unsigned &hi, unsigned &lo) {
    float ra, rb;
    hi = round_half(a, b);
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(ra) : "v"(hi), "v"(a));
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(rb) : "v"(hi), "v"(b));
    lo = round_half(ra, rb);
}
struct Pair {
    uintx4 hi, lo;
};
__device__ __forceinline__ Pair pair8(const float (&x)[8]) {
    Pair r;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        unsigned h, l;
        pair_up(x[2 * i], x[2 * i + 1], h, l);
        r.hi[i] = h;
        r.lo[i] = l;
    }
    return r;
}
// Factor 2^(14 - exponent) of numbers whose largest magnitude is given by its bits, its inverse, and that as a power of two.  Numbers below 2^-112
// take the exponent of 2^-112, and so do blocks of zeros (tokens behind the last one among them): their power is the lowest and never raises another's.
struct Scale {
    float up, down, power;
};
__device__ __forceinline__ Scale scale_of(unsigned bits) {
    unsigned e = bits >> 23;
    const bool whole = e < 255u;
    e = max(e, 15u);
    Scale s;
    s.up = whole ? __builtin_bit_cast(float, (268u - e) << 23) : 1.0f;
    s.down = whole ? __builtin_bit_cast(float, (e - 14u) << 23) : __builtin_nanf("");
    s.power = whole ? (float)((int)e - 141) : __builtin_nanf("");
    return s;
}
__device__ __forceinline__ unsigned wave_max(unsigned v) {  // in lane 63, read from there
    v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xf, 0xf, false));  // row_shr:1, 2, 4, 8
    v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xf, 0xf, false));
    v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xf, 0xf, false));
    v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xf, 0xf, false));
    v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xf, 0xf, false));  // row_bcast:15, 31
    v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xf, 0xf, false));
    return (unsigned)__builtin_amdgcn_readlane((int)v, 63);
}
// The larger of a lane's and that of lane ^ 32.  (As assembly: of the builtin's two results with equal operands the compiler keeps one.  The
// instruction wants two wait states behind the operands' last vector instruction.)
__device__ __forceinline__ float larger_half(float x) {
    float y = x;
    asm("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(x), "+v"(y));
    return fmaxf(x, y);
}
template <int NP>
__device__ __forceinline__ floatx16 multiply(const uintx4 (&a)[NP], const Pair &b, floatx16 c) {
    if constexpr (NP == 2) c = mfma(a[1], b.hi, c);
    c = mfma(a[0], b.lo, c);
    return mfma(a[0], b.hi, c);
}

// Where shared exponents end.  A number that is small beside the largest of its row or block is off by 2^-39 of that largest one:
//   scores  by D f 2^-9 doublings at most, f their factor.  Up to f D = 2^-10 (products of the largest numbers of 2^20) that is 2^-19, and 2^-24 as
//           the errors of many numbers add up;
//   values  by 2^-39 of the largest value that the wavefront met, for every token (weights below 2^-28 have no more bits than that).  Where the
//           largest sum of the row is 2^-12 of it or more, that is 2^-27 of the sum a token and, as errors add up, 2^-23 for thousands.
// Rows beyond (a hidden token, or one without weight, is thousands of times larger than what the row's result consists of) are computed
// again by attend_rows_fp32, 32 together.
constexpr float SCORES_SPREAD = 0x1p-10f, LEAST_POWER = -126.0f;
constexpr int VALUES_SPREAD = 12;

// The rows of a wavefront over [lo, hi) on the fp32 matrix instruction, operands straight from memory: no exponents are shared and nothing is split, so a
// row has the errors of the formula in fp32 whatever stands beside it.  The instruction takes two dimensions (tokens) where the fp16
// one takes sixteen, and nothing is asked for ahead: 2048 tokens over 8192 (bf16) with all rows again 3550 us, without 506.
template <int DT, bool F32, bool FULL>
__device__ __forceinline__ void attend_rows_fp32(const AttendParams &p, const Sequence &q, const int *pages, int kv_head, const float *q_row, const Range &range, int lo, int hi,
                                                 int see_lo, int see_hi, int k_token, floatx16 (&o)[DT], float &m, float &l) {
    const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5, D = FULL ? 32 * DT : p.D;
#pragma unroll
    for (int dt = 0; dt < DT; dt++)
#pragma unroll
        for (int r = 0; r < 16; r++) o[dt][r] = 0.0f;
    m = NEG_INF;
    l = 0.0f;
    const int to = min(hi, range.hi);
#pragma unroll 1
    for (int j0 = max(lo, range.lo); j0 < to; j0 += TILE_KV) {
        bool bad[2] = {false, false};
        size_t base[2];
#pragma unroll
        for (int b = 0; b < 2; b++)
            base[b] = block_base(p, j0 + 16 * b + 16 <= range.first ? 0 : pages[min(j0 + 16 * b, to - 1) >> p.page_shift], (j0 >> 4) + b, kv_head, bad[b]);
        floatx16 s;
#pragma unroll
        for (int r = 0; r < 16; r++) s[r] = 0.0f;
        const size_t k_from = (k_token >> 4 ? base[1] : base[0]) + (k_token & 15) * 8 + half * 128;
#pragma unroll 1
        for (int ks = 0; 16 * ks < D; ks++) {
            Raw<F32> raw;
            float k[8], x[8];
            raw.load(p.K, k_from + ks * 256);
            raw.numbers(k);
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] = q_row[16 * ks + 8 * half + i] * p.scale;
#pragma unroll
            for (int i = 0; i < 8; i++) s = __builtin_amdgcn_mfma_f32_32x32x2f32(k[i], x[i], s, 0, 0, 0);
        }
        float top = m;
#pragma unroll
        for (int r = 0; r < 16; r++) {
            const int j = j0 + 16 * (r >> 3) + 8 * half + (r & 7);
            s[r] = j >= see_lo && j < see_hi && j < to ? (bad[r >> 3] ? __builtin_nanf("") : s[r]) : NEG_INF;
            top = fmaxf(top, s[r]);
        }
        top = larger_half(top);
        const float keep = m == NEG_INF ? 0.0f : power2(m - top), from = top == NEG_INF ? 0.0f : top;
        l *= keep;
        m = top;
#pragma unroll
        for (int r = 0; r < 16; r++) {
            s[r] = power2(s[r] - from);
            l += s[r];
        }
#pragma unroll
        for (int dt = 0; dt < DT; dt++) {
            o[dt] *= keep;
#pragma unroll
            for (int b = 0; b < 2; b++) {
                Raw<F32> raw;
                float v[8];
                raw.load(p.V, base[b] + (size_t)half * 8 * D + (FULL ? 32 * dt + col : min(32 * dt + col, D - 1)) * 8);
                raw.keep(j0 + 16 * b + 16 <= range.first ? 0 : to - (j0 + 16 * b + 8 * half));
                raw.numbers(v);
#pragma unroll
                for (int i = 0; i < 8; i++) o[dt] = __builtin_amdgcn_mfma_f32_32x32x2f32(v[i], s[8 * b + i], o[dt], 0, 0, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    l += __shfl_xor(l, 32);
}

// FULL: head_dim is DP; otherwise the dimensions past the last are zeros in LDS.  grid: a multiple of 8 workgroups
template <int DP, bool F32, bool FULL, int W>
__global__ __launch_bounds__(64 * W, W == 8 || DP <= 128 ? 2 : 1) void attend_chunk_kernel(const AttendParams p, const int total) {
    constexpr int KS = DP / 16, DT = DP / 32, NP = F32 ? 2 : 1, UNITS = 4 * DP, EACH = DP / 32, ROWS = 32 * W;  // units: 8 numbers of a tile's keys or values
    __shared__ uintx4 kv[2][2][NP][UNITS];
    __shared__ float scales[2][4];  // of a tile's two blocks: keys' factors, values' powers of two
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 31, half = lane >> 5;
    const int D = FULL ? DP : p.D;
    // Workgroups that share an XCD get consecutive work: tiles and parts of one key head, whose keys and values its L2 keeps (2048 tokens over
    // 8192 549 us, dealt round 595).  Not where sequences are ragged: an XCD would get the long ones (7 of 4 to 301 new tokens 48 us, dealt round 36).
    const int per = (total + EDDLHIP_NUM_XCD - 1) / EDDLHIP_NUM_XCD;
    const int vid = p.grouped ? (blockIdx.x % EDDLHIP_NUM_XCD) * per + blockIdx.x / EDDLHIP_NUM_XCD : blockIdx.x;
    if (vid >= total) return;
    const int split = vid % p.splits, splits = p.splits, rest = vid / p.splits, of_head = rest / p.q_tiles, kv_head = of_head % p.kv_heads, seq = of_head / p.kv_heads;
    const Sequence q = sequence_of(p, seq);
    const int rows = q.fresh * p.group;
    const int *pages = p.table + (size_t)seq * p.width;
    // K's lane order: row col of the product is token `k_token` of the tile
    const int a8 = col >> 3, k_token = 16 * (a8 >> 1) + 8 * ((col >> 2) & 1) + 4 * (a8 & 1) + (col & 3);
    const int k_unit = (k_token >> 4) * 2 * DP + half * 16 + (k_token & 15);
    const int values = wave >> 1 & 1, block = wave & 1;  // what this wavefront brings of a tile (the first four do)

    if constexpr (!FULL) {
        for (int i = tid; i < 2 * 2 * NP * UNITS; i += 64 * W) kv[0][0][0][i] = uintx4{0u, 0u, 0u, 0u};
    }

    for (int tile = p.q_tiles - 1 - rest % p.q_tiles; tile * ROWS < rows; tile += p.q_tiles) {
        const Range all = range_of(p, q, tile * ROWS, min(rows, (tile + 1) * ROWS));
        const int steps_all = max(0, (all.hi - all.lo + TILE_KV - 1) / TILE_KV);
        const int step_lo = part_at(steps_all, split, splits), step_hi = part_at(steps_all, split + 1, splits);
        const int lo = all.lo + step_lo * TILE_KV, hi = min(all.hi, all.lo + step_hi * TILE_KV);
        const int row_lo = min(rows, tile * ROWS + 32 * wave), row_hi = min(rows, row_lo + 32);
        const bool works = row_lo < row_hi;
        const Range range = works ? range_of(p, q, row_lo, row_hi) : Range{0, 0, 0, 0, 0};

        // ---- the tiles' way into LDS
        bool bad = false;  // of the block that is on its way
        int page_lane = 0, page_from = -1;
        Raw<F32> raw[EACH];
        auto fetch = [&](int j0) __attribute__((always_inline)) {
            const int b = (j0 >> 4) + block;
            if (page_from < 0 || b >= page_from + 64) {
                page_from = b;
                page_lane = pages[min((b + lane) << 4, hi - 1) >> p.page_shift];  // (behind the last token: its page again, whose values do not count)
            }
            bad = false;
            const size_t base = block_base(p, 16 * b + 16 <= all.first ? 0 : __builtin_amdgcn_readlane(page_lane, b - page_from), b, kv_head, bad);
            const void *src = values ? p.V : p.K;
#pragma unroll
            for (int i = 0; i < EACH; i++)
                if (FULL || 64 * i + lane < 2 * D) raw[i].load(src, base + (size_t)(64 * i + lane) * 8);
        };
        auto place = [&](int j0, int buf) __attribute__((always_inline)) {
            const int from = j0 + 16 * block, end = from + 16 <= all.first ? 0 : all.hi;
            if (from + 16 > end) {  // what none of the tile's rows sees takes no part in the block's exponent
#pragma unroll
                for (int i = 0; i < EACH; i++) {
                    const int u = 64 * i + lane;
                    if (values) raw[i].keep(end - (from + (u >= D ? 8 : 0)));
                    else raw[i].keep(from + (u & 15) < end ? 8 : 0);
                }
            }
            unsigned top = 0;
#pragma unroll
            for (int i = 0; i < EACH; i++)
                if (FULL || 64 * i + lane < 2 * D) top = max(top, raw[i].largest());
            const Scale scale = scale_of(wave_max(top));
            if (lane == 0) scales[buf][wave] = bad ? __builtin_nanf("") : values ? scale.power : scale.down;
#pragma unroll
            for (int i = 0; i < EACH; i++) {
                const int u = 64 * i + lane, at = block * 2 * DP + u + (!FULL && values && u >= D ? DP - D : 0);
                if (FULL || u < 2 * D) {
                    float x[8];
                    raw[i].numbers(x);
#pragma unroll
                    for (int j = 0; j < 8; j++) x[j] *= scale.up;
                    if constexpr (F32) {
                        const Pair r = pair8(x);
                        kv[buf][values][0][at] = r.hi;
                        kv[buf][values][NP - 1][at] = r.lo;
                    } else {
                        kv[buf][values][0][at] = uintx4{round_half(x[0], x[1]), round_half(x[2], x[3]), round_half(x[4], x[5]), round_half(x[6], x[7])};
                    }
                }
            }
        };
        const int brings_to = W == 4 || wave < 4 ? hi : lo;  // (the first four wavefronts bring tiles; a bound, and no condition, keeps the loop's outputs in one place)
        if (lo < brings_to) fetch(lo);

        // ---- queries
        const int row = works ? min(row_lo + col, row_hi - 1) : 0, token = row / p.group, head = kv_head * p.group + row % p.group;
        const int pos = q.length - q.fresh + token;
        Pair qp[KS];
        float q_down;
        {
            float x[KS][8], top = 0.0f;
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                const float *src = p.Q + (size_t)(q.row0 + token) * p.ldq + (size_t)head * D + 16 * ks + 8 * half;
#pragma unroll
                for (int j = 0; j < 8; j++) x[ks][j] = 0.0f;
                if (FULL || 16 * ks < D) {
                    if (p.vec) {
                        const floatx4 u = *reinterpret_cast<const floatx4 *>(src), v = *reinterpret_cast<const floatx4 *>(src + 4);
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            x[ks][j] = u[j];
                            x[ks][4 + j] = v[j];
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < 8; j++) x[ks][j] = src[j];
                    }
                }
#pragma unroll
                for (int j = 0; j < 8; j++) top = fmaxf(top, fabsf(x[ks][j]));
            }
            const Scale scale = scale_of(__builtin_bit_cast(unsigned, fmaxf(top, __shfl_xor(top, 32))));
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
#pragma unroll
                for (int j = 0; j < 8; j++) x[ks][j] *= p.scale < 0.0f ? -scale.up : scale.up;
                qp[ks] = pair8(x[ks]);
            }
            q_down = scale.down * fabsf(p.scale);  // (factors are positive: a block's largest score is that of its largest product)
        }
        floatx16 o[DT];
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
#pragma unroll
            for (int r = 0; r < 16; r++) o[dt][r] = 0.0f;
        float m = NEG_INF, l = 0.0f, power = NEG_INF;  // power: the outputs' doublings, those of the largest values so far
        float f_most = 0.0f;                           // the largest factor of the row's scores
        const int see_lo = p.window > 0 ? pos - p.window + 1 : 0, see_hi = p.causal ? min(q.length, pos + 1) : q.length;

        __syncthreads();  // (the tile of rows before has read its last operands; zeros are in place)
        if (lo < brings_to) {
            place(lo, 0);
            if (lo + TILE_KV < brings_to) fetch(lo + TILE_KV);
        }
        __syncthreads();
        for (int j0 = lo, buf = 0; j0 < hi; j0 += TILE_KV, buf ^= 1) {
            if (j0 < range.hi && j0 + TILE_KV > range.lo) {  // (some of this wavefront's rows see the tile)
                floatx16 s;
#pragma unroll
                for (int r = 0; r < 16; r++) s[r] = 0.0f;
#pragma unroll
                for (int ks = 0; ks < KS; ks++) {
                    uintx4 k[NP];
#pragma unroll
                    for (int n = 0; n < NP; n++) k[n] = kv[buf][0][n][k_unit + 32 * ks];
                    s = multiply<NP>(k, qp[ks], s);
                }
                // (a factor of 0 would make NaN of what is masked)
                const float f[2] = {fmaxf(scales[buf][0] * q_down, 0x1p-126f), fmaxf(scales[buf][1] * q_down, 0x1p-126f)};
                const float poison = (scales[buf][0] - scales[buf][0]) + (scales[buf][1] - scales[buf][1]);  // 0, or NaN (the maximum above drops it)
                const float powers[2] = {scales[buf][2], scales[buf][3]};
                f_most = fmaxf(f_most, fmaxf(f[0], f[1]));
                if (j0 < range.all_lo || j0 + TILE_KV > range.all_hi) {
#pragma unroll
                    for (int r = 0; r < 16; r++) {
                        const int j = j0 + 16 * (r >> 3) + 8 * half + (r & 7);
                        s[r] = j >= see_lo && j < see_hi ? s[r] : NEG_INF;
                    }
                }
                float top = NEG_INF;
#pragma unroll
                for (int b = 0; b < 2; b++) {
                    float t = s[8 * b];
#pragma unroll
                    for (int r = 1; r < 8; r++) t = fmaxf(t, s[8 * b + r]);
                    top = fmaxf(top, t * f[b]);
                }
                top = fmaxf(larger_half(top), m);
                const float most = fmaxf(fmaxf(powers[0], powers[1]), power);
                if (__any(top > m) || most > power) {
                    const float keep = m == NEG_INF ? 0.0f : power2(m - top), turn = keep * power2(power - most);
                    l *= keep;
#pragma unroll
                    for (int dt = 0; dt < DT; dt++)
#pragma unroll
                        for (int r = 0; r < 16; r++) o[dt][r] *= turn;
                    m = top;
                    power = most;
                }
                const float from = m == NEG_INF ? 0.0f : m;
#pragma unroll
                for (int b = 0; b < 2; b++) {
                    const float c = powers[b] - power + 14.0f, shift = c - from + poison;
                    float w[8], sum = 0.0f;
#pragma unroll
                    for (int r = 0; r < 8; r++) {
                        w[r] = power2(__builtin_fmaf(s[8 * b + r], f[b], shift));
                        sum += w[r];
                    }
                    if (c < -20.0f) {  // (values of another size than those before: their weights leave fp32's range earlier than the sum's)
                        sum = 0.0f;
#pragma unroll
                        for (int r = 0; r < 8; r++) sum += power2(__builtin_fmaf(s[8 * b + r], f[b], -from));
                        l += sum;
                    } else {
                        l = __builtin_fmaf(sum, power2(-c), l);
                    }
                    const Pair ws = pair8(w);
#pragma unroll
                    for (int dt = 0; dt < DT; dt++) {
                        uintx4 v[NP];
#pragma unroll
                        for (int n = 0; n < NP; n++) v[n] = kv[buf][1][n][(b * 2 + half) * DP + 32 * dt + col];
                        o[dt] = multiply<NP>(v, ws, o[dt]);
                    }
                }
            }
            if (j0 + TILE_KV < brings_to) {
                place(j0 + TILE_KV, buf ^ 1);
                if (j0 + 2 * TILE_KV < brings_to) fetch(j0 + 2 * TILE_KV);
            }
            __syncthreads();
        }
        l += __shfl_xor(l, 32);
        const int doublings = power == NEG_INF ? 0 : (int)power - 14;
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
#pragma unroll
            for (int r = 0; r < 16; r++) o[dt][r] = __builtin_amdgcn_ldexpf(o[dt][r], doublings);

        // ---- rows whose numbers differ too much in size for shared exponents, and those that the next step concerns, in fp32
        const bool sees = max(lo, see_lo) < min(hi, see_hi);
        auto not_finite = [&]() __attribute__((always_inline)) {
            float worst = l - l;
#pragma unroll
            for (int dt = 0; dt < DT; dt++)
#pragma unroll
                for (int r = 0; r < 16; r++) worst += o[dt][r] - o[dt][r];
            return worst != 0.0f || (m == NEG_INF && sees);
        };
        bool again = not_finite();
        {
            float most = 0.0f;
#pragma unroll
            for (int dt = 0; dt < DT; dt++)
#pragma unroll
                for (int r = 0; r < 16; r++) most = fmaxf(most, fabsf(o[dt][r]));
            most = fmaxf(most, __shfl_xor(most, 32));
            const bool lost = f_most * (float)D > SCORES_SPREAD || (power > LEAST_POWER && most < __builtin_amdgcn_ldexpf(1.0f, (int)power + 14 - VALUES_SPREAD));
            if (__any((lost && sees) || again) && works && !q.bad) {
                attend_rows_fp32<DT, F32, FULL>(p, q, pages, kv_head, p.Q + (size_t)(q.row0 + token) * p.ldq + (size_t)head * D, range, lo, hi, see_lo, see_hi, k_token, o, m, l);
                again = not_finite() && l == l;  // (a sum that is NaN is that of visible scores: so is the row)
            }
        }

        // ---- rows whose sums are not finite, and rows that see tokens but no score above -inf, one by one
        again = (again || q.bad) && row_lo + col < row_hi;
        unsigned long long todo = __ballot(again);
        todo = (todo | (todo >> 32)) & 0xffffffffull;
        const bool redo = (todo >> col) & 1;
        for (unsigned long long t = todo; t != 0; t &= t - 1) {
            const int r = row_lo + __builtin_ctzll(t);
            const int head_r = kv_head * p.group + r % p.group;
            attend_row_again<F32>(p, q, seq, kv_head, r / p.group, head_r, lo, hi, (size_t)split * p.part_rows + (size_t)(q.row0 + r / p.group) * p.q_heads + head_r, splits, q.bad);
        }

        if (row_lo + col < row_hi && !redo) {
            const size_t at = (size_t)(q.row0 + token) * p.q_heads + head;
            const size_t slot = (size_t)split * p.part_rows + at;
            float factor = 1.0f, *dst;
            if (splits > 1) {
                if (half == 0) p.part_s[slot] = make_float2(m, l);
                dst = p.part_o + slot * D;
            } else {
                store_scale(p, m, l, factor);
                dst = p.O + (size_t)(q.row0 + token) * p.ldo + (size_t)head * D;
            }
#pragma unroll
            for (int dt = 0; dt < DT; dt++)
#pragma unroll
                for (int g = 0; g < 4; g++) {
                    const int d = 32 * dt + 8 * g + 4 * half;
                    if (FULL || d < D) {
                        const floatx4 x = {o[dt][4 * g] * factor, o[dt][4 * g + 1] * factor, o[dt][4 * g + 2] * factor, o[dt][4 * g + 3] * factor};
                        if (splits > 1 || p.vec) {
                            *reinterpret_cast<floatx4 *>(dst + d) = x;
                        } else {
#pragma unroll
                            for (int i = 0; i < 4; i++) dst[d + i] = x[i];
                        }
                    }
                }
        }
    }
}

// Joins parts in a launch of their own, a row in 16, 32 or 64 lanes of a wavefront: all parts' sums first, eight parts' outputs on their way at a
// time; added in the order of the tokens.
template <int LANES>
__global__ __launch_bounds__(256) void attend_join_kernel(const AttendParams p) {
    const int sub = threadIdx.x % LANES, d = 4 * sub;
    const long long total = (long long)p.rows * p.q_heads, at = (long long)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
    if (at >= total) return;
    const int row = (int)((unsigned)at / (unsigned)p.q_heads), head = (int)at - row * p.q_heads;
    if (row < max(p.offsets[0], 0) || row >= p.offsets[p.seqs]) return;
    constexpr int AHEAD = 8;
    float m = NEG_INF, l = 0.0f;
    floatx4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    const float *src = p.part_o + at * p.D + min(d, p.D - 4);
    for (int s0 = 0; s0 < p.splits; s0 += AHEAD) {  // (a running maximum over groups of parts)
        float2 ms[AHEAD];
        floatx4 x[AHEAD];
#pragma unroll
        for (int k = 0; k < AHEAD; k++) ms[k] = p.part_s[min(s0 + k, p.splits - 1) * total + at];
#pragma unroll
        for (int k = 0; k < AHEAD; k++) x[k] = *reinterpret_cast<const floatx4 *>(src + min(s0 + k, p.splits - 1) * total * p.D);
        float top = m;
#pragma unroll
        for (int k = 0; k < AHEAD; k++) top = fmaxf(top, ms[k].x);
        const float keep = m == NEG_INF ? (top == NEG_INF ? 1.0f : 0.0f) : power2(m - top);
        l = m == NEG_INF && top != NEG_INF ? (l == l ? 0.0f : l) : l * keep;
        o *= keep;
        m = top;
#pragma unroll
        for (int k = 0; k < AHEAD; k++)
            if (s0 + k < p.splits) {
                const float w = ms[k].x == NEG_INF && ms[k].y == 0.0f ? 0.0f : m == NEG_INF ? 1.0f : power2(ms[k].x - m);
                l += w * ms[k].y;
                o += x[k] * w;
            }
    }
    float factor;
    store_scale(p, m, l, factor);
    if (m == NEG_INF && l != 0.0f) factor = __builtin_nanf("");
    if (d < p.D) {
        float *dst = p.O + (size_t)row * p.ldo + (size_t)head * p.D + d;
        o *= factor;
        if (p.vec) {
            *reinterpret_cast<floatx4 *>(dst) = o;
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) dst[i] = o[i];
        }
    }
}

template <int DP, bool FULL>
void launch_few(const AttendParams &p, bool f32, int nq, dim3 grid, hipStream_t st) {
    typedef void (*kernel)(AttendParams);
    constexpr int MOST = DP <= 128 ? 2 : 1;
    static const kernel kernels[2][2] = {{attend_few_kernel<DP, false, 1, FULL>, attend_few_kernel<DP, false, MOST, FULL>},
                                         {attend_few_kernel<DP, true, 1, FULL>, attend_few_kernel<DP, true, MOST, FULL>}};
    hipLaunchKernelGGL(kernels[f32][nq - 1], grid, dim3(64 * few_waves(DP, f32, nq)), 0, st, p);
}

template <int DP, bool FULL>
void launch_chunk(const AttendParams &p, bool f32, int waves, int total, hipStream_t st) {
    typedef void (*kernel)(AttendParams, int);
    constexpr int MOST = DP <= 128 ? 8 : 4;
    static const kernel kernels[2][2] = {{attend_chunk_kernel<DP, false, FULL, 4>, attend_chunk_kernel<DP, false, FULL, MOST>},
                                         {attend_chunk_kernel<DP, true, FULL, 4>, attend_chunk_kernel<DP, true, FULL, MOST>}};
    const dim3 grid((total + EDDLHIP_NUM_XCD - 1) / EDDLHIP_NUM_XCD * EDDLHIP_NUM_XCD);
    hipLaunchKernelGGL(kernels[f32][waves == 8], grid, dim3(64 * waves), 0, st, p, total);
}

}  // namespace

namespace eddlhip {

int attention_setup_device(int dev) {
    void *ptr = nullptr;
    EH_TRY_HIP(hipGetSymbolAddress(&ptr, HIP_SYMBOL(part_counts)));
    EH_TRY_HIP(hipMemset(ptr, 0, sizeof(part_counts)));  // (also after a shutdown that cut launches short)
    EH_TRY_HIP(hipDeviceSynchronize());
    (void)dev;
    return 0;
}

}  // namespace eddlhip

extern "C" int eddlhip_paged_attention(int dev, const float *Q, long long ldq, float *O, long long ldo, int rows, const void *k_pages, const void *v_pages,
                                       int cache_type, int pages, int page_size, int q_heads, int kv_heads, int head_dim, const int *table, int table_width,
                                       const int *offsets, const int *lengths, int seqs, int max_new, int max_length, float scale, int causal, int window) {
    EH_REQUIRE(rows >= 0 && seqs >= 0 && seqs <= 65535, "paged_attention: %d rows of %d sequences (at most 65535)", rows, seqs);
    EH_REQUIRE(cache_type == EDDLHIP_CACHE_F32 || cache_type == EDDLHIP_CACHE_BF16, "paged_attention: unknown cache type %d", cache_type);
    EH_REQUIRE(head_dim >= 16 && head_dim <= 256 && head_dim % 16 == 0, "paged_attention: head_dim %d is not a multiple of 16 up to 256", head_dim);
    EH_REQUIRE(kv_heads > 0 && kv_heads <= 65535 && q_heads > 0 && q_heads % kv_heads == 0, "paged_attention: %d query heads do not share %d key heads evenly",
               q_heads, kv_heads);
    EH_REQUIRE(page_size >= 16 && page_size <= (1 << 20) && (page_size & (page_size - 1)) == 0, "paged_attention: page size %d is not a power of two from 16 on",
               page_size);
    EH_REQUIRE(pages > 0 && table_width > 0 && (long long)table_width * page_size <= MAX_TOKENS, "paged_attention: a pool of %d pages, a table of %d columns", pages,
               table_width);
    EH_REQUIRE(rows <= MAX_TOKENS && (long long)rows * q_heads <= 1LL << 30, "paged_attention: %d rows of %d heads are out of range", rows, q_heads);
    EH_REQUIRE(ldq >= (long long)q_heads * head_dim && ldo >= (long long)q_heads * head_dim, "paged_attention: rows of %lld and %lld floats do not hold %d heads of %d",
               ldq, ldo, q_heads, head_dim);
    EH_REQUIRE(std::isfinite(scale), "paged_attention: the scale is not finite");
    EH_REQUIRE(max_new >= 0 && max_length >= 0 && window >= 0, "paged_attention: negative max_new, max_length or window");
    if (rows == 0 || seqs == 0) return 0;
    EH_REQUIRE(Q && O && k_pages && v_pages && table && offsets && lengths, "paged_attention: NULL tensor");
    EH_REQUIRE(!eh_rows_overlap(Q, ldq, (long long)q_heads * head_dim, O, ldo, (long long)q_heads * head_dim, rows), "paged_attention: the output lies on the queries");
    EH_REQUIRE((((uintptr_t)k_pages | (uintptr_t)v_pages) & 15) == 0, "paged_attention: the cache is not aligned to 16 bytes");
    for (const void *cache : {k_pages, v_pages})
        EH_REQUIRE(!eh_rows_meet(O, ldo, (long long)q_heads * head_dim, rows, cache, (size_t)pages * page_size * kv_heads * head_dim * (cache_type == EDDLHIP_CACHE_F32 ? 4 : 2)),
                   "paged_attention: the output shares memory with the cache");
    EH_TRY(use_device(dev));
    AttendParams p;
    p.Q = Q;
    p.O = O;
    p.K = k_pages;
    p.V = v_pages;
    p.table = table;
    p.offsets = offsets;
    p.lengths = lengths;
    p.ldq = ldq;
    p.ldo = ldo;
    p.rows = rows;
    p.q_heads = q_heads;
    p.kv_heads = kv_heads;
    p.group = q_heads / kv_heads;
    p.D = head_dim;
    p.pages = pages;
    p.page_shift = __builtin_ctz((unsigned)page_size);
    p.width = table_width;
    p.seqs = seqs;
    p.causal = causal != 0;
    p.window = std::min(window, MAX_TOKENS);  // (no sequence is longer)
    p.vec = (((uintptr_t)Q | (uintptr_t)O) & 15) == 0 && ldq % 4 == 0 && ldo % 4 == 0;
    p.scale = scale * 1.44269504088896340736f;
    // The launch goes by the bounds max_new and max_length; what is beyond them is still computed, by the same wavefronts.
    const long long fresh = std::min(max_new > 0 ? max_new : 1, rows), tile_rows = fresh * p.group;
    const int nq = tile_rows <= 16 ? 1 : tile_rows <= 32 ? (head_dim <= 128 ? 2 : 1) : 0;
    // (the rows fill the tiles of all sequences, but for one begun tile each)
    const bool even = ((long long)rows * p.group) / 128 + seqs >= (tile_rows + 127) / 128 * seqs;
    const int waves = head_dim <= 128 && tile_rows > 128 && even ? 8 : 4, per_tile = nq ? 16 * nq : 32 * waves;
    const long long tiles = (tile_rows + per_tile - 1) / per_tile;
    p.q_tiles = (int)tiles;
    // (sequences of fewer new tokens than max_new have fewer tiles, all together no more than their rows fill and one begun tile each)
    const long long groups = tiles * kv_heads * seqs, filled = kv_heads * std::min(tiles * seqs, ((long long)rows * p.group) / per_tile + seqs), want = (nq ? few_groups(head_dim, cache_type == EDDLHIP_CACHE_F32, nq) : 8LL / waves) * state(dev).num_cu;
    long long seen = max_length > 0 ? max_length : 1;
    if (window > 0) seen = std::min<long long>(seen, (long long)window + fresh);
    const long long steps = (seen + TILE_KV - 1) / TILE_KV;
    p.splits = (int)std::max(1LL, std::min({want / filled, steps / (nq ? 8 : 4), (long long)(nq ? FEW_SPLITS / nq : CHUNK_SPLITS)}));
    if (nq && groups > MAX_COUNTS) p.splits = 1;
    // Parts that a launch joins have a place for every row of the tensors: with many more rows than the batch has (room for other batches), fewer
    // parts, or those that the last workgroup joins, whose places are those of the launch's tiles.  A full batch takes 100 MB at most.
    p.part_rows = (long long)rows * q_heads;
    const size_t part_bytes = (size_t)p.part_rows * (head_dim + 2) * sizeof(float);
    if (p.splits > (nq ? JOIN_HERE : 1) && p.splits * part_bytes > MOST_PARTS) p.splits = nq ? JOIN_HERE : (int)std::max((size_t)1, MOST_PARTS / part_bytes);
    if (nq && p.splits <= JOIN_HERE) p.part_rows = groups * per_tile;
    p.grouped = even;
    p.part_o = nullptr;
    p.part_s = nullptr;
    if (p.splits > 1) {
        const size_t slots = (size_t)p.splits * p.part_rows;
        void *ws = nullptr;
        EH_TRY(get_workspace(dev, slots * (head_dim + 2) * sizeof(float), &ws));
        p.part_o = (float *)ws;
        p.part_s = (float2 *)((char *)ws + slots * head_dim * sizeof(float));
    }
    EH_REQUIRE(groups * p.splits < (1LL << 30), "paged_attention: shape out of range");
    const dim3 grid((unsigned)(tiles * p.splits), kv_heads, seqs);
    const hipStream_t st = state(dev).stream;
    const bool f32 = cache_type == EDDLHIP_CACHE_F32;
    const int total = (int)(groups * p.splits);
    auto launch = [&](auto size, auto full) {
        if (nq) launch_few<size(), full()>(p, f32, nq, grid, st);
        else launch_chunk<size(), full()>(p, f32, waves, total, st);
    };
    auto sized = [&](auto size) {
        if (head_dim == size()) launch(size, std::true_type());
        else launch(size, std::false_type());
    };
    if (head_dim <= 64) sized(std::integral_constant<int, 64>());
    else if (head_dim <= 96) sized(std::integral_constant<int, 96>());
    else if (head_dim <= 128) sized(std::integral_constant<int, 128>());
    else if (head_dim <= 192) sized(std::integral_constant<int, 192>());
    else sized(std::integral_constant<int, 256>());
    EH_CHECK_LAUNCH();
    if (p.splits > (nq ? JOIN_HERE : 1)) {
        const long long joined = (long long)rows * q_heads;
        if (head_dim <= 64) hipLaunchKernelGGL(attend_join_kernel<16>, dim3((unsigned)((joined + 15) / 16)), dim3(256), 0, st, p);
        else if (head_dim <= 128) hipLaunchKernelGGL(attend_join_kernel<32>, dim3((unsigned)((joined + 7) / 8)), dim3(256), 0, st, p);
        else hipLaunchKernelGGL(attend_join_kernel<64>, dim3((unsigned)((joined + 3) / 4)), dim3(256), 0, st, p);
        EH_CHECK_LAUNCH();
    }
    return 0;
}
