// efg_attn_launch.h - the attention kernels' launchers (efg_attn.cu chooses among them).
#pragma once

#include <cuda_runtime.h>

namespace efg {

struct AttnParams;

// Warp-level tensor cores (efg_attn_mma.cu): head sizes up to 128 in whole 16-byte pieces, rows
// and bases 16-byte aligned.
bool attn_mma_takes(int type, const AttnParams& p);
int launch_attn_mma(int type, const AttnParams& p, int sms, cudaStream_t s);

}  // namespace efg
