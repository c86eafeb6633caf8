// Launchers of the biased attention, one translation unit per kernel family.
#pragma once
#include "attn_rows.cuh"
#include "block_host.cuh"

namespace fxh {

constexpr int64_t kMaxGrid = INT32_MAX;

// ---- launch_attn_tc.cu: tcgen05 kernels
// A.splits parts of the keys, more than one: joined by attn_join_kernel.
int launch_attn_tc_fwd(cudaStream_t s, const AttnArgs& A, bool is_f32, bool aligned);
// Parts of the keys that fill the device.
int attn_tc_splits(const AttnArgs& A, bool is_f32, int sms);
// Backward (float32: dim <= 64). A.delta, A.lut and A.dpart (batch x query blocks of 128 parts a
// head) are workspace.
int launch_attn_tc_bwd(cudaStream_t s, const AttnArgs& A, bool is_f32, bool aligned);

}  // namespace fxh
