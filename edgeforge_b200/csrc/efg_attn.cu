// efg_attn.cu - softmax attention entry points: packed prompts (efg_attn_prompt) and new tokens
// over a paged cache (efg_attn_paged).
//
//   out[r][h] = sum_j w_j v[j][h / group],  w = softmax_j(scale q[r][h] . k[j][h / group])
//
// over the positions j that row r sees: those of its own sequence up to its own position.
#include <algorithm>
#include <type_traits>

#include <cuda_runtime.h>

#include "../../include/efg.h"
#include "efg_attn.cuh"
#include "efg_attn_launch.h"
#include "efg_host.h"

namespace efg {
namespace {

constexpr int kRowWarps = 4;

// Any head size, stride and alignment: one warp per row and query head.
template <typename T>
__global__ void __launch_bounds__(kRowWarps * 32) attn_rows_kernel(const AttnParams p) {
  const int warp = threadIdx.x >> 5;
  if (blockIdx.x == 0) check_offsets(p);
  const int64_t item = static_cast<int64_t>(blockIdx.x) * kRowWarps + warp;
  const int64_t row = item / p.heads;
  if (row >= p.n_rows) return;
  const int64_t s = find_sequence(p.cu, p.n_seqs, row);
  if (s < 0 || s >= p.n_seqs) return;  // behind the last sequence
  Chunk c;
  if (!chunk_of_seq(p, s, c)) return;
  attend_row<T>(p, c, row, static_cast<int>(item % p.heads));
}

template <typename T>
int launch_rows(const AttnParams& p, cudaStream_t s) {
  const int64_t items = p.n_rows * p.heads, ctas = (items + kRowWarps - 1) / kRowWarps;
  if (ctas > 0x7FFFFFFFll) return fail(EFG_EINVAL, "attention: too many rows");
  attn_rows_kernel<T><<<static_cast<unsigned>(ctas), kRowWarps * 32, 0, s>>>(p);
  EFG_TRY_CUDA(cudaGetLastError(), "attention launch");
  return EFG_OK;
}

int check_workspace(size_t need, const void* work, size_t bytes) {
  if (need > bytes || (need && !work))
    return fail(EFG_EINVAL, "attention: a workspace of %zu bytes is needed, got %zu", need, bytes);
  if (need && reinterpret_cast<uintptr_t>(work) % 16)
    return fail(EFG_EINVAL, "attention: the workspace is not 16-byte aligned");
  return EFG_OK;
}

int launch_attn(int type, const AttnParams& p, int sms, void* work, size_t work_bytes, cudaStream_t s) {
  if (attn_decode_takes(type, p)) {
    const size_t need = attn_decode_workspace(type, p, sms);
    if (int st = check_workspace(need, work, work_bytes)) return st;
    return launch_attn_decode(type, p, sms, work, s);
  }
  if (attn_tc_takes(type, p)) {
    const size_t need = attn_tc_workspace(p, sms);
    if (int st = check_workspace(need, work, work_bytes)) return st;
    return launch_attn_tc(type, p, sms, need ? work : nullptr, s);
  }
  if (attn_mma_takes(type, p)) return launch_attn_mma(type, p, sms, s);
  if (type == EFG_F32) return launch_rows<float>(p, s);
  if (type == EFG_F16) return launch_rows<__half>(p, s);
  return launch_rows<__nv_bfloat16>(p, s);
}

// The checks that both calls make; `who` names the call.
int check_attn(const char* who, int type, size_t n_seqs, size_t n_rows, size_t heads, size_t kv_heads,
               size_t head_dim, size_t q_stride, float scale) {
  if (type < EFG_F32 || type > EFG_BF16) return fail(EFG_EINVAL, "%s: unknown type %d", who, type);
  if (head_dim == 0 || head_dim > 256) return fail(EFG_EINVAL, "%s: head_dim %zu is not in 1..256", who, head_dim);
  if (kv_heads == 0 || heads == 0 || heads > 4096 || heads % kv_heads)
    return fail(EFG_EINVAL, "%s: %zu query heads do not divide into %zu key heads", who, heads, kv_heads);
  if (n_rows > 0x7FFFFF00ull || n_seqs > (1ull << 24)) return fail(EFG_EINVAL, "%s: a size is out of range", who);
  if (q_stride < heads * head_dim) return fail(EFG_EINVAL, "%s: a row stride is shorter than a row", who);
  if (!(scale == scale) || scale - scale != 0.f) return fail(EFG_EINVAL, "%s: scale is not finite", who);
  return EFG_OK;
}

}  // namespace
}  // namespace efg

using efg::fail;

extern "C" {

int efg_attn_prompt(const efg_attn_prompt_args* args, void* stream) {
  if (!args) return fail(EFG_EINVAL, "attn_prompt: null pointer");
  const auto& [type, scale, d_out, d_q, q_stride, d_k, k_stride, d_v, v_stride, d_cu, n_seqs, n_rows, heads, kv_heads,
               head_dim] = *args;
  if (int st = efg::check_attn("attn_prompt", type, n_seqs, n_rows, heads, kv_heads, head_dim, q_stride, scale))
    return st;
  if (k_stride < kv_heads * head_dim || v_stride < kv_heads * head_dim)
    return fail(EFG_EINVAL, "attn_prompt: a row stride is shorter than a row");
  if (n_rows == 0 || n_seqs == 0) return EFG_OK;
  if (!d_out || !d_q || !d_k || !d_v || !d_cu) return fail(EFG_EINVAL, "attn_prompt: null pointer");
  const size_t es = type == EFG_F32 ? 4 : 2, n_out = n_rows * heads * head_dim * es, row = kv_heads * head_dim;
  if (efg::overlap(d_out, n_out, d_q, n_rows, q_stride, heads * head_dim, es) ||
      efg::overlap(d_out, n_out, d_k, n_rows, k_stride, row, es) ||
      efg::overlap(d_out, n_out, d_v, n_rows, v_stride, row, es) || efg::overlap(d_out, n_out, d_cu, 1, 0, n_seqs + 1, 4))
    return fail(EFG_EINVAL, "attn_prompt: out overlaps an input");
  efg::DeviceInfo* dev = efg::current_device();
  if (!dev) return EFG_ECUDA;
  efg::AttnParams p{};
  p.out = d_out;
  p.q = d_q;
  p.k = d_k;
  p.v = d_v;
  p.cu = d_cu;
  p.q_stride = static_cast<int64_t>(q_stride);
  p.k_stride = static_cast<int64_t>(k_stride);
  p.v_stride = static_cast<int64_t>(v_stride);
  p.n_rows = static_cast<int64_t>(n_rows);
  p.n_seqs = static_cast<int64_t>(n_seqs);
  p.heads = static_cast<int>(heads);
  p.kv_heads = static_cast<int>(kv_heads);
  p.group = p.heads / p.kv_heads;
  p.head_dim = static_cast<int>(head_dim);
  p.scale = scale;
  p.err = dev->d_err;
  p.checks = dev->d_checks;
  return efg::launch_attn(type, p, dev->sm_count, nullptr, 0, static_cast<cudaStream_t>(stream));
}

uint64_t efg_attn_paged_workspace(const efg_attn_paged_args* args) {
  if (!args) return 0;
  const size_t n_seqs = args->n_seqs, max_pages = args->max_pages, page_size = args->page_size, heads = args->heads,
               kv_heads = args->kv_heads, head_dim = args->head_dim, max_new = args->max_new, n_rows = args->n_rows;
  efg::AttnParams p{};
  p.kv_len = reinterpret_cast<const int32_t*>(1);  // a paged call; never read
  p.n_seqs = static_cast<int64_t>(n_seqs);
  p.max_pages = static_cast<int64_t>(max_pages);
  p.page_size = static_cast<int64_t>(page_size);
  p.kv_heads = static_cast<int>(kv_heads);
  p.head_dim = static_cast<int>(head_dim);
  p.max_new = static_cast<int64_t>(max_new);
  p.n_rows = static_cast<int64_t>(n_rows);
  if (kv_heads == 0 || n_seqs == 0 || heads < kv_heads || head_dim > 128) return 0;
  p.group = static_cast<int>(heads / kv_heads);
  efg::DeviceInfo* dev = efg::current_device();
  if (!dev) return 0;
  if (std::min(max_new, n_rows) * p.group <= static_cast<size_t>(efg::kDecodeRows))
    return efg::attn_decode_workspace(args->type, p, dev->sm_count);
  return (args->type == EFG_F32 && head_dim > 64) || p.group > 128 ? 0 : efg::attn_tc_workspace(p, dev->sm_count);
}

int efg_attn_paged(const efg_attn_paged_args* args, void* stream) {
  if (!args) return fail(EFG_EINVAL, "attn_paged: null pointer");
  const auto& [type, scale, d_out, d_q, q_stride, d_k_cache, d_v_cache, n_pages, page_size, d_block_table, max_pages,
               d_cu, d_kv_len, n_seqs, n_rows, max_new, heads, kv_heads, head_dim, d_workspace, workspace_bytes] = *args;
  if (int st = efg::check_attn("attn_paged", type, n_seqs, n_rows, heads, kv_heads, head_dim, q_stride, scale))
    return st;
  if (page_size == 0 || page_size > (1u << 30)) return fail(EFG_EINVAL, "attn_paged: page size %zu", page_size);
  if (max_new > 0x7FFFFFFFull) return fail(EFG_EINVAL, "attn_paged: max_new is out of range");
  if (n_pages > 0x7FFFFF00ull / page_size || max_pages > 0x7FFFFF00ull / page_size)
    return fail(EFG_EINVAL, "attn_paged: %zu pages (%zu a sequence) of %zu slots pass the 2^31 slots of a cache",
                n_pages, max_pages, page_size);
  if (n_rows == 0 || n_seqs == 0 || max_new == 0) return EFG_OK;
  if (!d_out || !d_q || !d_cu || !d_kv_len || (n_pages && (!d_k_cache || !d_v_cache)) ||
      (max_pages && !d_block_table))
    return fail(EFG_EINVAL, "attn_paged: null pointer");
  const size_t es = type == EFG_F32 ? 4 : 2, n_out = n_rows * heads * head_dim * es, row = kv_heads * head_dim;
  auto meets = [&](const void* to, size_t n) {
    return efg::overlap(to, n, d_q, n_rows, q_stride, heads * head_dim, es) ||
           efg::overlap(to, n, d_k_cache, n_pages * page_size, row, row, es) ||
           efg::overlap(to, n, d_v_cache, n_pages * page_size, row, row, es) ||
           efg::overlap(to, n, d_block_table, n_seqs, max_pages, max_pages, 4) ||
           efg::overlap(to, n, d_cu, 1, 0, n_seqs + 1, 4) || efg::overlap(to, n, d_kv_len, 1, 0, n_seqs, 4);
  };
  if (meets(d_out, n_out)) return fail(EFG_EINVAL, "attn_paged: out overlaps an input");
  if (meets(d_workspace, workspace_bytes) || efg::overlap(d_workspace, workspace_bytes, d_out, 1, 0, n_out, 1))
    return fail(EFG_EINVAL, "attn_paged: the workspace overlaps out or an input");
  efg::DeviceInfo* dev = efg::current_device();
  if (!dev) return EFG_ECUDA;
  efg::AttnParams p{};
  p.out = d_out;
  p.q = d_q;
  p.k = d_k_cache;
  p.v = d_v_cache;
  p.cu = d_cu;
  p.kv_len = d_kv_len;
  p.table = d_block_table;
  p.q_stride = static_cast<int64_t>(q_stride);
  p.k_stride = p.v_stride = static_cast<int64_t>(kv_heads * head_dim);
  p.n_rows = static_cast<int64_t>(n_rows);
  p.n_seqs = static_cast<int64_t>(n_seqs);
  p.n_pages = static_cast<int64_t>(n_pages);
  p.max_pages = static_cast<int64_t>(max_pages);
  p.page_size = static_cast<int64_t>(page_size);
  p.max_new = static_cast<int64_t>(max_new);
  p.page_shift = (page_size & (page_size - 1)) == 0 ? __builtin_ctzll(page_size) : -1;
  p.heads = static_cast<int>(heads);
  p.kv_heads = static_cast<int>(kv_heads);
  p.group = p.heads / p.kv_heads;
  p.head_dim = static_cast<int>(head_dim);
  p.scale = scale;
  p.err = dev->d_err;
  p.checks = dev->d_checks;
  return efg::launch_attn(type, p, dev->sm_count, d_workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
