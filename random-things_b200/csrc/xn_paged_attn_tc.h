// xn_paged_attn_tc.h - host entry of the tensor-core kernel of the paged attention.
#pragma once

#include "xn_paged_attn.cuh"

namespace xn {
namespace paged {

constexpr int kTcRows = 256, kTcKeys = 128;  // rows of a query tile, keys of a key tile

// Enqueues the kernel (bf16 / f16); XN_OK, or the error recorded.
int launch_tc(const Args &a, int d, int dtype, cudaStream_t st, const char *op);

}  // namespace paged
}  // namespace xn
