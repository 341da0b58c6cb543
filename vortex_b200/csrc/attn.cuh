// What the attention-layer kernels share.
#pragma once

#include "common.cuh"

namespace vtx {

// Device status code of a block-table entry that a call needs and that names no page of the pool.
constexpr int kStatusBadPage = 0x7a6e;

}  // namespace vtx
