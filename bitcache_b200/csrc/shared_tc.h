// The tensor-memory kernel of shared prefixes (shared_tc.cu): its list and launch.
#pragma once

#include "shared.cuh"

namespace bc {

// Prefixes only; rows of a block: an even division of the group's query rows into blocks of at most 128.
ShList sh_tc_list(int n_seqs, int n_groups, int group);
// head_dim 64 or 128.
int sh_tc_run(const SharedArgs& a, const ShList& L, int head_dim, bool compensated, cudaStream_t st);

}  // namespace bc
