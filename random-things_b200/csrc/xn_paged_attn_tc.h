// xn_paged_attn_tc.h - host entries of the paged attention's tensor-core kernels.
#pragma once

#include "xn_paged_attn.cuh"

namespace xn {
namespace paged {

// Rows of a query tile and keys of a key tile: chunks, and single tokens.
constexpr int kTcRows = 256, kTcKeys = 64;
constexpr int kDecRows = 16, kDecKeys = 64;

constexpr long long kWaitClocks = 4000000000ll;  // a wait gives up after 2 s or more

// Enqueue the kernel for chunks / for single tokens (bf16 / f16); XN_OK, or the error recorded.
int launch_tc(const Args &a, int d, int dtype, cudaStream_t st, const char *op);
int launch_dec(const Args &a, int d, int dtype, cudaStream_t st, const char *op);

}  // namespace paged
}  // namespace xn
