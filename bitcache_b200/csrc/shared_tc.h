// The tensor-memory kernel of shared prefixes (shared_tc.cu): its list and launch.
#pragma once

#include "shared.cuh"

namespace bc {

// Prefixes only; rows of a block: an even division of the group's query rows into blocks of at most 128.
ShList sh_tc_list(int n_seqs, int n_groups, int group);
// Bytes of its operand rows (rows: n_seqs * n_kv * group).
size_t sh_tc_scratch(int64_t rows, int head_dim);
// head_dim 64 or 128.
int sh_tc_run(const SharedArgs& a, const ShList& L, void* scratch, int head_dim, bool compensated, cudaStream_t st);

}  // namespace bc
