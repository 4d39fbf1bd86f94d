// efg_paged.cuh - index arithmetic of the paged key/value cache, shared by the kernels that
// plan a step, store into pages and attend over them. Plain C++ (no CUDA types), so the same
// lines run in a host test with out-of-range lengths and page ids.
//
// A cache is n_pages pages of page_size token slots; slot = page * page_size + offset. The
// block table of a sequence lists its pages in order: position p lies in entry p / page_size.
#pragma once

#include <cstddef>
#include <cstdint>

#if defined(__CUDACC__)
#define EFG_HD __host__ __device__ __forceinline__
#else
#define EFG_HD inline
#endif

namespace efg {

// What one sequence needs for its step.
struct SeqNeed {
  int64_t rows;  // rows of the packed batch that belong to it (its new tokens)
  int64_t have;  // pages that already hold its cached tokens
  int64_t need;  // fresh pages; 0 for a sequence that cannot be served
  bool valid;    // lengths are non-negative and the block table is wide enough
};

EFG_HD int64_t pages_for(uint32_t positions, uint32_t page_size) {
  const uint32_t whole = positions / page_size;
  return static_cast<int64_t>(whole) + (positions != whole * page_size);
}

// `most`: positions that a sequence may have.
EFG_HD SeqNeed seq_need_upto(int32_t cached, int32_t fresh, int64_t page_size, int64_t most) {
  SeqNeed n;
  n.rows = fresh > 0 ? fresh : 0;
  const int64_t end = static_cast<int64_t>(cached) + fresh;
  n.valid = cached >= 0 && fresh >= 0 && end <= most;
  // lengths fit 32 unsigned bits here, and a 32-bit division is a fraction of a 64-bit one
  n.have = n.valid ? pages_for(static_cast<uint32_t>(cached), static_cast<uint32_t>(page_size)) : 0;
  n.need = n.valid ? pages_for(static_cast<uint32_t>(end), static_cast<uint32_t>(page_size)) - n.have : 0;
  return n;
}

EFG_HD SeqNeed seq_need(int32_t cached, int32_t fresh, int64_t page_size, int64_t max_pages) {
  return seq_need_upto(cached, fresh, page_size, max_pages * page_size);
}

// Lengths and positions are held in 32 signed bits by the kernels that read them (with room for a tile).
constexpr int64_t kMaxPositions = 0x7FFFFF00;
EFG_HD int64_t most_positions(int64_t max_pages, int64_t page_size) {
  const int64_t held = max_pages * page_size;
  return held < kMaxPositions ? held : kMaxPositions;
}
EFG_HD SeqNeed seq_need_held(int32_t cached, int32_t fresh, int64_t page_size, int64_t max_pages) {
  return seq_need_upto(cached, fresh, page_size, most_positions(max_pages, page_size));
}

// Fresh pages are handed out in sequence order. A sequence is served when its own pages end
// inside the free list; once one is not, none after it that needs a page is (`first` counts
// the needs of every sequence before it, served or not).
EFG_HD bool seq_served(const SeqNeed& n, int64_t first, int64_t n_free) {
  return n.valid && (n.need == 0 || first + n.need <= n_free);
}

EFG_HD bool page_ok(int32_t page, int64_t n_pages) { return page >= 0 && page < n_pages; }

// The keys that row `row` of the packed batch sees: positions [0, count) of its sequence, whose chunk
// ends before row `end` and whose cache holds kv_len positions with the chunk at the end.
// 0 when the row sees nothing (more rows than positions).
EFG_HD int32_t visible_keys(int32_t row, int32_t end, int32_t kv_len) {
  const int32_t n = kv_len - (end - row) + 1;  // 0 <= kv_len <= 2^31 - 256, row < end
  return n > 0 ? n : 0;
}

// Largest s with cu[s] <= row, over cu[0..n_seqs]; -1 when cu[0] > row. In bounds for any cu.
EFG_HD int64_t find_sequence(const int32_t* cu, int64_t n_seqs, int64_t row) {
  int64_t lo = 0, hi = n_seqs + 1;  // cu[lo - 1] <= row < cu[hi] in sorted input
  while (lo < hi) {
    const int64_t mid = (lo + hi) / 2;
    if (cu[mid] <= row)
      lo = mid + 1;
    else
      hi = mid;
  }
  return lo - 1;
}

// Whether `out` (n_out bytes) and n_rows rows of `in` (`row` of `stride` elements of es bytes each) overlap.
inline bool overlap(const void* out, size_t n_out, const void* in, size_t n_rows, size_t stride, size_t row, size_t es) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(out), b = reinterpret_cast<uintptr_t>(in);
  return out && in && n_out && n_rows && row && a < b + ((n_rows - 1) * stride + row) * es && b < a + n_out;
}

}  // namespace efg
