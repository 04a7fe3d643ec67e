// The two forms of the 8-bit linear layer: linear_int8_sm100.cu has the entry points and the tensor-memory kernel,
// linear_int8_small.cu the kernel for a few tokens.
#pragma once

#include "internal.h"

namespace fdb {

constexpr int kInt8SmallRows = 32;
constexpr int kInt8SmallSmem = 100 * 1024;  // two CTAs per SM

// Whether a checked call goes to the kernel for a few tokens (which needs no workspace).
bool int8_is_small(const fdb_linear_int8_params& p);
int launch_linear_int8_small(const fdb_linear_int8_params& p, void* stream);

}  // namespace fdb
