// Workgroups are dealt to the XCDs in turn.  Jobs whose neighbours share lines of memory are put on one XCD in runs of EDDLHIP_XCD_RUN, so that its L2 holds what
// they share; longer runs (an eighth of all jobs) would give an XCD whole sequences, of which a ragged batch has long and short ones (the convolution of eight
// ragged sequences: 45 us, in runs 25).
#pragma once
#include "common.h"

#define EDDLHIP_XCD_RUN 8

namespace eddlhip {

// The job of workgroup `id`, which may lie behind the last one.
__device__ __forceinline__ long long xcd_job(long long id) {
    constexpr int RUN = EDDLHIP_XCD_RUN, ALL = EDDLHIP_NUM_XCD * RUN;
    const int r = (int)(id % ALL);
    return id - r + r % EDDLHIP_NUM_XCD * RUN + r / EDDLHIP_NUM_XCD;
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
