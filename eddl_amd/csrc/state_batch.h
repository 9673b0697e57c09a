// What the operators along the tokens of a ragged batch share: its description on the device, and what a workgroup reads of it for its sequence.
#pragma once
#include "common.h"
#include "sequence_rows.h"

namespace eddlhip {

struct StateBatch {
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
__device__ __forceinline__ Sequence sequence(const StateBatch &b, int s) {
    const SequenceRows r = sequence_rows(b.offsets[s], b.offsets[s + 1], b.rows);
    Sequence q{r.row0, r.fresh, -1, -1, b.reverse ? -1 : 1};
    if (b.pool > 0) {
        const int read = b.slots[s], write = b.out_slots[s];
        if (b.lengths[s] > r.fresh) q.read = (unsigned)read < (unsigned)b.pool ? read : -2;
        if ((unsigned)write < (unsigned)b.pool) q.write = write;
    }
    return q;
}

constexpr int MOST_CHANNELS = 1 << 20, MOST_ROWS = 1 << 30;

// What both entry points ask of a batch; `name` opens the error's text.
inline int check_batch(const char *name, int rows, int seqs, int max_new, const float *states, int pool, const int *offsets, const int *lengths, const int *slots, const int *out_slots) {
    EH_REQUIRE(rows >= 0 && rows <= MOST_ROWS && seqs >= 0 && seqs <= 65535, "%s: %d rows (at most %d) of %d sequences (at most 65535)", name, rows, MOST_ROWS, seqs);
    EH_REQUIRE(max_new >= 0 && pool >= 0 && (states != nullptr) == (pool > 0), "%s: max_new %d, a pool of %d states%s", name, max_new, pool, states ? "" : " at NULL");
    if (rows == 0 || seqs == 0) return 0;
    EH_REQUIRE(offsets && (!states || (lengths && slots && out_slots)), "%s: NULL offsets, lengths or slots", name);
    return 0;
}

}  // namespace eddlhip
