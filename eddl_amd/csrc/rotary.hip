// Rotary positions with several axes (time, row, column of a token of an image or a video), and the write of keys and values into
// the paged cache that goes with them.
//
// Pair n of a head's first rot_dim dimensions turns by the angle a = position[axis[n]] * frequency[n]:
//     y_i = x_i cos a - x_j sin a,   y_j = x_j cos a + x_i sin a,    (i, j) = (n, n + rot_dim / 2) or (2n, 2n + 1);
// the dimensions behind rot_dim are copied.  Axis and frequency of every pair come from the host and travel as the kernel's
// arguments.  Angles of far positions lose their meaning in 32 bits (position 1e5 at frequency 1: steps of 0.008), so the angle is
// formed in 64 bits, in turns, and only its distance from the nearest quarter of a turn, an eighth at most, goes into the fp32 sine and cosine: rounded by
// 2^-28 of a turn at most, 0.4 of the half step of a sine near 1 (the fraction of a whole turn would be rounded by four times that, and
// the error of a turned pair be 1.39 times that of correctly rounded sines where it is 1.03).  They are computed once for a token and pair and
// kept in LDS for all heads.
//
// Bound: memory, 8 bytes a number.  12544 rows of 16 heads of 128: 36 us, 5.7 TB/s (a copy stream reaches 5.7 - 6.3).  Append of 4 x 1568 tokens, 16 heads
// of 64, fp32: 41 us, 3.7 TB/s - the keys' and values' rows are read 64 and 256 bytes at a time, for the order of the pages.
#include <math.h>

#include <algorithm>

#include "common.h"
#include "sequence_rows.h"
#include "split_parts.h"

using namespace eddlhip;

namespace {

typedef float floatx4 __attribute__((ext_vector_type(4)));

constexpr int TPB = 256;
constexpr int MAX_PAIRS = 128;

struct Rotary {
    double turns[MAX_PAIRS];  // frequency / (2 pi)
    unsigned char axis[MAX_PAIRS];
    const float *positions;  // [rows][axes]
    int pairs, axes, adjacent;
};

__device__ __forceinline__ float2 turn(const Rotary &r, int row, int n) {
    const double t = (double)r.positions[(size_t)row * r.axes + r.axis[n]] * r.turns[n];
    const double quarters = rint(4.0 * t);
    const int quarter = (int)(quarters - 4.0 * floor(0.25 * quarters));
    float s, c;
    sincospif(2.0f * (float)(t - 0.25 * quarters), &s, &c);
    const float x = quarter & 1 ? s : c, y = quarter & 1 ? c : s;  // (cos and sin of a quarter more: -sin, cos)
    return make_float2(quarter == 1 || quarter == 2 ? -x : x, quarter & 2 ? -y : y);
}

__device__ __forceinline__ floatx4 load4(const float *p, bool vec) {
    if (vec) return *reinterpret_cast<const floatx4 *>(p);
    return floatx4{p[0], p[1], p[2], p[3]};
}
__device__ __forceinline__ void store4(float *p, floatx4 x, bool vec) {
    if (vec) {
        __builtin_nontemporal_store(x, reinterpret_cast<floatx4 *>(p));  // (written once, in whole lines)
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) p[i] = x[i];
    }
}

// A thread takes four numbers side by side and, where halves are paired, the four that they turn with: its accesses and its
// neighbours' lie side by side.  Pieces of a head: pairs / 4 of eight numbers and the rest of four, or all of four.
__device__ __forceinline__ int pieces_of(const Rotary &r, int D) { return r.adjacent ? D / 4 : r.pairs / 4 + (D - 2 * r.pairs) / 4; }
struct Piece {
    int d0, d1;  // d1 < 0: four numbers only
};
__device__ __forceinline__ Piece piece_at(const Rotary &r, int n) {
    if (r.adjacent) return Piece{4 * n, -1};
    return 4 * n < r.pairs ? Piece{4 * n, 4 * n + r.pairs} : Piece{4 * n + r.pairs, -1};
}
__device__ __forceinline__ void turn_piece(const Rotary &r, int n, const float2 *cs, floatx4 &x, floatx4 &y) {
    if (r.adjacent) {
        if (2 * n >= r.pairs) return;
        const float2 s = cs[2 * n], t = cs[2 * n + 1];
        x = floatx4{x[0] * s.x - x[1] * s.y, x[1] * s.x + x[0] * s.y, x[2] * t.x - x[3] * t.y, x[3] * t.x + x[2] * t.y};
    } else if (4 * n < r.pairs) {
        const floatx4 a = x, b = y;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 t = cs[4 * n + i];
            x[i] = a[i] * t.x - b[i] * t.y;
            y[i] = b[i] * t.x + a[i] * t.y;
        }
    }
}

// grid: groups of ROWS rows, looping
template <int ROWS>
__global__ __launch_bounds__(TPB) void rotary_kernel(const Rotary r, const float *X, float *Y, long long ldx, long long ldy, int rows, int heads, int D, int vec) {
    __shared__ float2 cs[ROWS][MAX_PAIRS];
    const int pieces = pieces_of(r, D), per_row = heads * pieces;
    for (long long first = (long long)blockIdx.x * ROWS; first < rows; first += (long long)gridDim.x * ROWS) {  // (64 bits: the step beyond the last of 2^31 - 1 rows)
        const int row0 = (int)first, n_rows = min(ROWS, rows - row0);
        __syncthreads();
        for (int i = threadIdx.x; i < n_rows * r.pairs; i += TPB) cs[i / r.pairs][i % r.pairs] = turn(r, row0 + i / r.pairs, i % r.pairs);
        __syncthreads();
        for (int i = threadIdx.x; i < n_rows * per_row; i += TPB) {
            const int at = i / per_row, rest = i - at * per_row, head = rest / pieces, n = rest - head * pieces;
            const Piece c = piece_at(r, n);
            const float *src = X + (size_t)(row0 + at) * ldx + (size_t)head * D;
            floatx4 x = load4(src + c.d0, vec), y = x;
            if (c.d1 >= 0) y = load4(src + c.d1, vec);
            turn_piece(r, n, cs[at], x, y);
            float *dst = Y + (size_t)(row0 + at) * ldy + (size_t)head * D;
            store4(dst + c.d0, x, vec);
            if (c.d1 >= 0) store4(dst + c.d1, y, vec);
        }
    }
}

struct AppendParams {
    const float *Q, *K, *V;
    float *Qout;
    void *k_pages, *v_pages;
    const int *table, *offsets, *lengths;
    long long ldq, ldk, ldv, ldo;
    int rows, q_heads, kv_heads, D, pages, page_shift, width, f32, vec, head_groups;
};

__device__ __forceinline__ void put4(void *base, size_t at, floatx4 x, int f32) {
    if (f32) {
        *reinterpret_cast<floatx4 *>((float *)base + at) = x;
    } else {  // (rounded to nearest even: the cache's type)
        *reinterpret_cast<uint2 *>((unsigned short *)base + at) = make_uint2(split_round(x[0], x[1]), split_round(x[2], x[3]));
    }
}

// The new tokens of a sequence that lie in one block of 16 places of the cache, and a part of the heads.
// grid (blocks of 16 places, looping; head_groups; seqs)
__global__ __launch_bounds__(TPB) void paged_append_kernel(const Rotary r, const AppendParams p) {
    __shared__ float2 cs[16][MAX_PAIRS];
    const int seq = blockIdx.z, length = max(p.lengths[seq], 0);
    const SequenceRows own = sequence_rows(p.offsets[seq], p.offsets[seq + 1], p.rows);
    const int row0 = own.row0, fresh = own.fresh;
    const int start = length - fresh;  // place of row row0 (below 0: the first rows have none)
    if (fresh == 0) return;
    const int D = p.D, pieces = pieces_of(r, D);
    // blocks of 16 rows of the sequence, aligned to the places
    const int shift = start & 15;
    for (long long from = 16LL * blockIdx.x - shift; from < fresh; from += 16LL * gridDim.x) {
        const int first = (int)max(0LL, from), n_rows = (int)min((long long)fresh, from + 16) - first;  // of the sequence's rows
        // the block's place in the cache; nothing is written where there is none
        const int place = start + first;
        int page = -1;
        if (place >= 0 && length > 0 && (place >> p.page_shift) < p.width) page = p.table[(size_t)seq * p.width + (place >> p.page_shift)];
        __syncthreads();
        for (int i = threadIdx.x; i < n_rows * r.pairs; i += TPB) cs[i / r.pairs][i % r.pairs] = turn(r, row0 + first + i / r.pairs, i % r.pairs);
        __syncthreads();
        const bool stored = (unsigned)page < (unsigned)p.pages;
        const size_t block = ((size_t)page * p.kv_heads << (p.page_shift - 4)) + ((place >> 4) & ((1 << (p.page_shift - 4)) - 1));
        const size_t head_stride = (size_t)16 * D << (p.page_shift - 4);
        const int t0 = place & 15;
        const int q_items = p.Q ? p.q_heads : 0, head_lo = (int)((long long)(q_items + 2 * p.kv_heads) * blockIdx.y / p.head_groups),
                  head_hi = (int)((long long)(q_items + 2 * p.kv_heads) * (blockIdx.y + 1) / p.head_groups);
        // queries, keys and values of the group's heads, each as one run of work for all threads
        const int q_hi = min(head_hi, q_items), q_work = max(0, q_hi - head_lo) * n_rows * pieces;
        for (int i = threadIdx.x; i < q_work; i += TPB) {
            const int rest = i / pieces, n = i - rest * pieces, h = rest / n_rows, at = rest - h * n_rows;
            const size_t row = row0 + first + at, col = (size_t)(head_lo + h) * D;
            const Piece c = piece_at(r, n);
            const float *src = p.Q + row * p.ldq + col;
            floatx4 x = load4(src + c.d0, p.vec), y = x;
            if (c.d1 >= 0) y = load4(src + c.d1, p.vec);
            turn_piece(r, n, cs[at], x, y);
            float *dst = p.Qout + row * p.ldo + col;
            store4(dst + c.d0, x, p.vec);
            if (c.d1 >= 0) store4(dst + c.d1, y, p.vec);
        }
        if (!stored) continue;
        const int k_lo = max(head_lo - q_items, 0), k_hi = min(head_hi - q_items, p.kv_heads), k_work = max(0, k_hi - k_lo) * n_rows * pieces;
        for (int i = threadIdx.x; i < k_work; i += TPB) {
            const int rest = i / n_rows, at = i - rest * n_rows, h = rest / pieces, n = rest - h * pieces;  // (tokens side by side: theirs are the neighbouring places)
            const int kv = k_lo + h;
            const Piece c = piece_at(r, n);
            const float *src = p.K + (size_t)(row0 + first + at) * p.ldk + (size_t)kv * D;
            floatx4 x = load4(src + c.d0, p.vec), y = x;
            if (c.d1 >= 0) y = load4(src + c.d1, p.vec);
            turn_piece(r, n, cs[at], x, y);
            const size_t t = block * 16 * D + kv * head_stride + (t0 + at) * 8;
            put4(p.k_pages, t + (c.d0 >> 3) * 128 + (c.d0 & 7), x, p.f32);
            if (c.d1 >= 0) put4(p.k_pages, t + (c.d1 >> 3) * 128 + (c.d1 & 7), y, p.f32);
        }
        const int v_lo = max(head_lo - q_items - p.kv_heads, 0), v_hi = head_hi - q_items - p.kv_heads, v_work = max(0, v_hi - v_lo) * 2 * D;
        for (int i = threadIdx.x; i < v_work; i += TPB) {  // eight tokens of a dimension: theirs are the places side by side
            const int rest = i / D, d = i - rest * D, half = rest & 1, kv = v_lo + (rest >> 1), at = 8 * half - t0;  // (row of the half's first token)
            if (at + 8 <= 0 || at >= n_rows) continue;
            const float *src = p.V + (long long)(row0 + first + at) * p.ldv + (long long)kv * D + d;
            float x[8];
            const size_t t = block * 16 * D + kv * head_stride + (size_t)half * 8 * D + d * 8;
            if (at >= 0 && at + 8 <= n_rows) {
#pragma unroll
                for (int k = 0; k < 8; k++) x[k] = src[k * p.ldv];
                put4(p.v_pages, t, floatx4{x[0], x[1], x[2], x[3]}, p.f32);
                put4(p.v_pages, t + 4, floatx4{x[4], x[5], x[6], x[7]}, p.f32);
            } else {
#pragma unroll
                for (int k = 0; k < 8; k++)
                    if (at + k >= 0 && at + k < n_rows) {
                        const float v = src[k * p.ldv];
                        if (p.f32) ((float *)p.v_pages)[t + k] = v;
                        else ((unsigned short *)p.v_pages)[t + k] = (unsigned short)split_round(v, v);
                    }
            }
        }
    }
}

int rotary_plan(Rotary &r, const char *what, const float *positions, int head_dim, int rot_dim, int adjacent, int axes, const int *host_axis,
                const double *host_freq) {
    EH_REQUIRE(head_dim >= 8 && head_dim % 8 == 0, "%s: head_dim %d is not a multiple of 8", what, head_dim);
    EH_REQUIRE(rot_dim >= 0 && rot_dim % 8 == 0 && rot_dim <= head_dim && rot_dim <= 2 * MAX_PAIRS, "%s: rot_dim %d is not a multiple of 8 up to %d of a head of %d",
               what, rot_dim, 2 * MAX_PAIRS, head_dim);
    r.pairs = rot_dim / 2;
    r.adjacent = adjacent != 0;
    r.positions = positions;
    r.axes = axes;
    if (rot_dim == 0) return 0;
    EH_REQUIRE(positions && host_axis && host_freq, "%s: NULL positions, axes or frequencies", what);
    EH_REQUIRE(axes > 0 && axes <= 256, "%s: %d axes", what, axes);
    for (int n = 0; n < r.pairs; n++) {
        EH_REQUIRE(host_axis[n] >= 0 && host_axis[n] < axes, "%s: pair %d turns by axis %d of %d", what, n, host_axis[n], axes);
        r.axis[n] = (unsigned char)host_axis[n];
        r.turns[n] = host_freq[n] * 0.15915494309189533576888;  // 1 / (2 pi)
    }
    return 0;
}

bool aligned16(const void *p, long long ld) { return ((uintptr_t)p & 15) == 0 && ld % 4 == 0; }

}  // namespace

extern "C" {

int eddlhip_rotary_axes(int dev, const float *X, long long ldx, float *Y, long long ldy, int rows, int heads, int head_dim, const float *positions, int rot_dim,
                        int adjacent, int axes, const int *host_axis, const double *host_freq) {
    EH_REQUIRE(rows >= 0 && heads > 0, "rotary_axes: %d rows of %d heads", rows, heads);
    Rotary r;
    EH_TRY(rotary_plan(r, "rotary_axes", positions, head_dim, rot_dim, adjacent, axes, host_axis, host_freq));
    EH_REQUIRE((long long)heads * head_dim <= (1 << 24) && ldx >= (long long)heads * head_dim && ldy >= (long long)heads * head_dim,
               "rotary_axes: rows of %lld and %lld floats do not hold %d heads of %d", ldx, ldy, heads, head_dim);
    if (rows == 0) return 0;
    EH_REQUIRE(X && Y, "rotary_axes: NULL tensor");
    EH_REQUIRE(X == Y || !eh_rows_overlap(X, ldx, (long long)heads * head_dim, Y, ldy, (long long)heads * head_dim, rows), "rotary_axes: the output lies on a part of the input");
    EH_REQUIRE(X != Y || ldx == ldy, "rotary_axes: in place, but rows of %lld and %lld floats", ldx, ldy);
    EH_REQUIRE(rot_dim == 0 || !eh_rows_meet(Y, ldy, (long long)heads * head_dim, rows, positions, (size_t)rows * axes * sizeof(float)), "rotary_axes: the output lies on the positions");
    EH_TRY(use_device(dev));
    const int vec = aligned16(X, ldx) && aligned16(Y, ldy);
    if (rows >= 4 * 4 * state(dev).num_cu)
        hipLaunchKernelGGL(rotary_kernel<4>, dim3(std::min((rows - 1) / 4 + 1, 1 << 20)), dim3(TPB), 0, state(dev).stream, r, X, Y, ldx, ldy, rows, heads, head_dim, vec);
    else
        hipLaunchKernelGGL(rotary_kernel<1>, dim3(std::min(rows, 1 << 20)), dim3(TPB), 0, state(dev).stream, r, X, Y, ldx, ldy, rows, heads, head_dim, vec);
    EH_CHECK_LAUNCH();
    return 0;
}

int eddlhip_paged_append(int dev, const float *Q, long long ldq, float *Qout, long long ldo, const float *K, long long ldk, const float *V, long long ldv, int rows,
                         int q_heads, int kv_heads, int head_dim, const float *positions, int rot_dim, int adjacent, int axes, const int *host_axis,
                         const double *host_freq, void *k_pages, void *v_pages, int cache_type, int pages, int page_size, const int *table, int table_width,
                         const int *offsets, const int *lengths, int seqs, int max_new) {
    EH_REQUIRE(rows >= 0 && seqs >= 0 && seqs <= 65535, "paged_append: %d rows of %d sequences (at most 65535)", rows, seqs);
    EH_REQUIRE(cache_type == EDDLHIP_CACHE_F32 || cache_type == EDDLHIP_CACHE_BF16, "paged_append: unknown cache type %d", cache_type);
    EH_REQUIRE(head_dim >= 16 && head_dim <= 256 && head_dim % 16 == 0, "paged_append: head_dim %d is not a multiple of 16 up to 256", head_dim);
    EH_REQUIRE(kv_heads > 0 && (Q == nullptr || q_heads > 0) && q_heads >= 0 && (long long)q_heads + 2LL * kv_heads <= (1 << 20), "paged_append: %d query and %d key heads",
               q_heads, kv_heads);
    EH_REQUIRE((Q == nullptr) == (Qout == nullptr), "paged_append: queries and their output come together");
    EH_REQUIRE(page_size >= 16 && page_size <= (1 << 20) && (page_size & (page_size - 1)) == 0, "paged_append: page size %d is not a power of two from 16 on", page_size);
    EH_REQUIRE(pages > 0 && table_width > 0 && max_new >= 0, "paged_append: a pool of %d pages, a table of %d columns, max_new %d", pages, table_width, max_new);
    Rotary r;
    EH_TRY(rotary_plan(r, "paged_append", positions, head_dim, rot_dim, adjacent, axes, host_axis, host_freq));
    EH_REQUIRE(ldk >= (long long)kv_heads * head_dim && ldv >= (long long)kv_heads * head_dim &&
                   (Q == nullptr || (ldq >= (long long)q_heads * head_dim && ldo >= (long long)q_heads * head_dim)),
               "paged_append: rows of %lld, %lld, %lld and %lld floats do not hold %d and %d heads of %d", ldq, ldo, ldk, ldv, q_heads, kv_heads, head_dim);
    if (rows == 0 || seqs == 0) return 0;
    EH_REQUIRE(K && V && k_pages && v_pages && table && offsets && lengths, "paged_append: NULL tensor");
    EH_REQUIRE((((uintptr_t)k_pages | (uintptr_t)v_pages) & 15) == 0, "paged_append: the cache is not aligned to 16 bytes");
    const long long q_width = (long long)q_heads * head_dim, kv_width = (long long)kv_heads * head_dim;
    EH_REQUIRE((Q == Qout || !eh_rows_overlap(Q, ldq, q_width, Qout, ldo, q_width, rows)) && !eh_rows_overlap(K, ldk, kv_width, Qout, ldo, q_width, rows) &&
                   !eh_rows_overlap(V, ldv, kv_width, Qout, ldo, q_width, rows), "paged_append: the turned queries lie on a part of what is read");
    EH_REQUIRE(Q != Qout || ldq == ldo, "paged_append: queries in place, but rows of %lld and %lld floats", ldq, ldo);
    EH_REQUIRE(rot_dim == 0 || !eh_rows_meet(Qout, ldo, q_width, rows, positions, (size_t)rows * axes * sizeof(float)), "paged_append: the turned queries lie on the positions");
    const size_t cache_bytes = (size_t)pages * page_size * kv_heads * head_dim * (cache_type == EDDLHIP_CACHE_F32 ? 4 : 2);
    for (const void *cache : {(const void *)k_pages, (const void *)v_pages})
        EH_REQUIRE(!eh_rows_meet(Q, ldq, q_width, rows, cache, cache_bytes) && !eh_rows_meet(Qout, ldo, q_width, rows, cache, cache_bytes) &&
                       !eh_rows_meet(K, ldk, kv_width, rows, cache, cache_bytes) && !eh_rows_meet(V, ldv, kv_width, rows, cache, cache_bytes),
                   "paged_append: rows share memory with the cache");
    EH_TRY(use_device(dev));
    AppendParams p;
    p.Q = Q;
    p.K = K;
    p.V = V;
    p.Qout = Qout;
    p.k_pages = k_pages;
    p.v_pages = v_pages;
    p.table = table;
    p.offsets = offsets;
    p.lengths = lengths;
    p.ldq = ldq;
    p.ldk = ldk;
    p.ldv = ldv;
    p.ldo = ldo;
    p.rows = rows;
    p.q_heads = q_heads;
    p.kv_heads = kv_heads;
    p.D = head_dim;
    p.pages = pages;
    p.page_shift = __builtin_ctz((unsigned)page_size);
    p.width = table_width;
    p.f32 = cache_type == EDDLHIP_CACHE_F32;
    p.vec = aligned16(K, ldk) && aligned16(V, ldv) && (Q == nullptr || (aligned16(Q, ldq) && aligned16(Qout, ldo)));
    // The launch goes by the bound max_new; sequences with more new tokens loop.
    const int fresh = std::min(max_new > 0 ? max_new : 1, rows), blocks = (int)((fresh + 14LL) / 16) + 1;
    const long long items = (Q ? q_heads : 0) + 2LL * kv_heads, there = (long long)blocks * seqs;
    p.head_groups = (int)std::max(1LL, std::min({items, (8LL * state(dev).num_cu + there - 1) / there, 65535LL}));
    hipLaunchKernelGGL(paged_append_kernel, dim3(blocks, p.head_groups, seqs), dim3(TPB), 0, state(dev).stream, r, p);
    EH_CHECK_LAUNCH();
    return 0;
}

}  // extern "C"
