// efg_attn_launch.h - the attention kernels' launchers (efg_attn.cu chooses among them).
#pragma once

#include <cstddef>

#include <cuda_runtime.h>

namespace efg {

struct AttnParams;

// Warp-level tensor cores (efg_attn_mma.cu): head sizes to 128 in whole 16-byte pieces, rows
// and bases 16-byte aligned.
bool attn_mma_takes(int type, const AttnParams& p);
int launch_attn_mma(int type, const AttnParams& p, int sms, cudaStream_t s);

// At most kDecodeRows rows per key head (efg_attn_decode.cu); the workspace joins the parts of long sequences.
constexpr int kDecodeRows = 16;
bool attn_decode_takes(int type, const AttnParams& p);
size_t attn_decode_workspace(int type, const AttnParams& p, int sms);
int launch_attn_decode(int type, const AttnParams& p, int sms, void* work, cudaStream_t s);

// 5th-generation tensor cores (efg_attn_tc.cu): more than 16 rows per key head, over pages more than 64; F32 head
// sizes to 64.
bool attn_tc_takes(int type, const AttnParams& p);
// With a workspace of attn_tc_workspace bytes the work is cut evenly along the keys; without one (or where
// that is 0) row tiles stay whole.
size_t attn_tc_workspace(const AttnParams& p, int sms);
int launch_attn_tc(int type, const AttnParams& p, int sms, void* work, cudaStream_t s);

}  // namespace efg
