// Limits and status bits shared by the tree verification operators.
#pragma once

#include "common.cuh"
#include "tc_common.cuh"

namespace af {

constexpr int64_t AF_TREE_MAX_NODES = 16384;    // nodes per tree (64 KB of parents in shared memory)
constexpr int64_t AF_TABLES_MAX_BATCH = 16384;  // requests per call (three sums each in shared memory)
constexpr int64_t AF_TREE_ATTN_MAX_BATCH = 16384;

}  // namespace af
