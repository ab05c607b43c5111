// Paged attention of single next tokens whose requests share a prefix (a system prompt, the beams of one search).
//
// Rows (one token each) come in groups: the rows group_start[g] .. group_start[g + 1] - 1 share the positions
// [0, prefix_len[g]), which lie in the pages of block-table row prefix_slot[g].  A position behind them lies in the
// pages of the row's own request, or, with a history, in those of the member of the group that wrote it: the beams of a search
// keep their keys where they were written, and what a beam inherits is a list of writers (history[slot][n] is the
// member that wrote position prefix_len + n; the row's own position is always its own).  A row at position pos sees
// [max(0, pos - window + 1), pos].
//
// The query heads of all members over one key/value head are the rows of one matrix product over the shared keys, so
// these are read once for the group instead of once for every member: out = sum_j softmax(s)_j v_j is taken apart into the
// part over the shared positions and the part over the others, each with its maximum m, its sum l of 2^(s - m) and its
// unnormalised output o, all in float32, and the parts are added up as sum_i 2^(m_i - m) o_i / sum_i 2^(m_i - m) l_i.
//
// Here: what the kernels of the parts have in common.
#pragma once

#include "mma_utils.cuh"

namespace tk {

struct SharedParams {
  const void* q;                // [rows, n_q_heads, d]
  void* out;                    // [rows, n_q_heads, dv]
  const void* k_cache;          // [num_pages, n_kv_heads, page_size, d]
  const void* v_cache;          // [num_pages, n_kv_heads, page_size, dv]
  const int* group_start;       // [n_groups + 1]
  const int* prefix_slot;       // [n_groups]
  const int* prefix_len;        // [n_groups]
  const int* positions;         // [rows]
  const int* req_slot;          // [rows]
  const int* block_table;       // [max_slots, max_pages]
  const unsigned char* history; // [max_slots, history_ld] or null
  const float* sinks;           // [n_q_heads] or null
  float* part_o;                // [rows, n_q_heads, n_parts, dv]   (the general kernel's)
  float* part_ml;               // [rows, n_q_heads, n_parts, 2]
  float* scratch;               // 32-byte aligned
  int* err;
  int n_rows, n_groups, max_members, n_q_heads, n_kv_heads, d, dv, page_size, max_pages, num_pages, max_slots, history_ld, window;
  int n_shared, n_own, n_parts; // parts of the shared and of the other positions; n_parts = n_shared + n_own (on the tensor cores
                                // n_shared is the number of blocks for the shared ones, 0: nothing is but by a history)
  int wide_k, wide_v;           // rows of queries and keys, of values, can be read four elements at a time
  float scale_log2, cap_log2, inv_cap;
};

// The group that holds a row: the last one that starts at or before it.
__device__ __forceinline__ int group_of_row(const SharedParams& p, int row) {
  int lo = 0, hi = p.n_groups - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (p.group_start[mid] <= row) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// Rows of group g, cut to what exists.
__device__ __forceinline__ int2 group_rows(const SharedParams& p, int g) {
  const int a = max(0, min(p.n_rows, p.group_start[g]));
  const int b = max(a, min(p.n_rows, p.group_start[g + 1]));
  return make_int2(a, min(b, a + p.max_members));
}

__device__ __forceinline__ int checked_slot(const SharedParams& p, int slot, int row) {
  if (slot >= 0 && slot < p.max_slots) return slot;
  set_error(p.err, kErrRequest, row, slot, p.max_slots);
  return -1;
}

// Place of a position in the pools: (page * n_kv_heads + head) * page_size + offset, -1 for one that has no page.
__device__ __forceinline__ long long pool_row(const SharedParams& p, int slot, int pos, int hkv, int row) {
  const int pidx = pos / p.page_size;
  const int page = (slot >= 0 && pidx < p.max_pages) ? p.block_table[(size_t)slot * p.max_pages + pidx] : -1;
  if (page < 0 || page >= p.num_pages) {
    if (slot >= 0) set_error(p.err, kErrPage, row, pidx, page);
    return -1;
  }
  return ((long long)page * p.n_kv_heads + hkv) * p.page_size + pos % p.page_size;
}

// The slot that holds position `pos` (behind the shared ones) of row `row`.
__device__ __forceinline__ int writer_slot(const SharedParams& p, int row, int slot, int pos, int own_pos, int prefix, int2 rows) {
  if (p.history == nullptr || pos == own_pos || slot < 0) return slot;
  const int n = pos - prefix;
  if (n >= p.history_ld) { set_error(p.err, kErrPosition, row, pos, p.history_ld); return -1; }
  const int member = p.history[(size_t)slot * p.history_ld + n];
  if (member >= rows.y - rows.x) { set_error(p.err, kErrRequest, row, member, rows.y - rows.x); return -1; }
  return checked_slot(p, p.req_slot[rows.x + member], row);
}

// Whether the row belongs to a group as it should; where not, its shared parts are marked as empty here (head >= 0: for that
// head), since no block of the shared positions does it, and an error is set.
__device__ __forceinline__ bool row_has_group(const SharedParams& p, int row, int2 rows, int prefix, int head) {
  if (row >= rows.x && row < rows.y && (p.n_shared > 0 || prefix == 0)) return true;
  set_error(p.err, kErrRequest, row, p.max_members, prefix);
  if (head >= 0) {
    float* ml = p.part_ml + 2 * ((size_t)row * p.n_q_heads + head) * p.n_parts;
    for (int i = 0; i < p.n_shared; ++i) { ml[2 * i] = -INFINITY; ml[2 * i + 1] = 0.0f; }
  }
  return false;
}

// What a row sees: [lo, pos]; bad positions see nothing.
struct RowSpan { int pos, lo; };
__device__ __forceinline__ RowSpan row_span(const SharedParams& p, int row) {
  const int pos = p.positions[row];
  if (pos < 0 || pos >= (long long)p.max_pages * p.page_size) {          // none, or one that the block table has no place for
    set_error(p.err, kErrPosition, row, pos, p.max_pages);
    return {-1, 0};
  }
  return {pos, first_visible(pos, p.window, 0)};
}

// ---- attention_shared_tc.cu -------------------------------------------------------------------------------------------
// bfloat16 heads of 64 or 128: the shared positions on tcgen05, the others on mma.sync.
bool shared_tc_takes(const SharedParams& p);
long long shared_tc_scratch(const SharedParams& p, int sms);
int launch_shared_tc(const SharedParams& p, int sms, cudaStream_t stream);

}  // namespace tk
