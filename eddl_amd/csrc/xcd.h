// Workgroups are dealt to the XCDs in turn.  Jobs whose neighbours share lines of memory are put on one XCD in runs of EDDLHIP_XCD_RUN, so that its L2 holds what
// they share; longer runs (an eighth of all jobs) would give an XCD whole sequences, of which a ragged batch has long and short ones (the convolution of eight
// ragged sequences: 45 us, in runs 25).
#pragma once
#include "common.h"

#define EDDLHIP_XCD_RUN 8

namespace eddlhip {

// The job of workgroup `id`, which may lie behind the last one.  TURN: the XCDs change places from 64 jobs to the next.  Where only every so many jobs have work - the
// first chunks of sequences shorter than the host's bound - and that is a power of two, it would all meet one of them (the convolution of 255 sequences of 100 tokens and one
// of 4096: 262 us, so 119; of eight ragged ones 22.9 and 21.0).  Where all jobs have work, their own places are better (the scan of 8192 tokens of 4096 channels 3 % less).
template <bool TURN = false>
__device__ __forceinline__ long long xcd_job(long long id) {
    constexpr int RUN = EDDLHIP_XCD_RUN, ALL = EDDLHIP_NUM_XCD * RUN;
    const int r = (int)(id % ALL);
    int turn = 0;
    if (TURN) {  // (the sum of the octal digits)
        static_assert(EDDLHIP_NUM_XCD == 8, "");
        for (long long all = id / ALL; all > 0; all >>= 3) turn += (int)(all & 7);
    }
    return id - r + (r + turn) % EDDLHIP_NUM_XCD * RUN + r / EDDLHIP_NUM_XCD;
}
// Workgroups that have all of `jobs` among their jobs.
constexpr long long xcd_padded(long long jobs) {
    constexpr int ALL = EDDLHIP_NUM_XCD * EDDLHIP_XCD_RUN;
    return (jobs + ALL - 1) / ALL * ALL;
}
// Workgroups of a launch: a grid holds less than 2^32 threads, and its workgroups walk what is beyond.
inline unsigned xcd_grid(long long jobs, int threads) {
    const long long most = ((1LL << 32) / threads - 1) / EDDLHIP_NUM_XCD * EDDLHIP_NUM_XCD, all = xcd_padded(jobs);
    return (unsigned)(all < most ? all : most);
}

}  // namespace eddlhip
