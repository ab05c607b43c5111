// Search over beams: the best continuations of the beams of every group, and what follows from them for the next step.
//
// Selection.  Beam w of a group has a score s_w (the sum of its tokens' log probabilities) and a row of logits x_w; its
// continuation by token v has the key
//     key(w, v) = s_w + ((x_wv - M_w) - log sum_u exp(x_wu - M_w)),      M_w any reference of the row,
// and the K largest keys of a group's W * V are wanted in order; equal keys of one beam by the larger logit, others by the
// lowest w * V + v.  Keys of neighbouring ranks differ by less than a float's last place often enough to change what a
// search does, so sums and keys are 64-bit: the exponentials are floats (an error of some 1e-7 each that falls away in the
// sum, where the largest terms are exact or nearly so), added four at a time as floats and then as doubles.
//
// One pass over the logits.  Within a row the order of the keys is that of the logits, so the K best of a row's segment can
// be kept without knowing the row's sum: a block streams its segment in tiles, holds a threshold with at least K elements
// at or above it, and sets aside only what is above (the threshold of the first tile is the K-th largest of the threads'
// own maxima; random rows set aside some K ln(n) elements behind it).  A second kernel, started early, has a block per
// group: it adds the segments' sums up in their order, makes the keys of the elements set aside and ranks them.  Two kernels and
// no counter: calls on two streams, or two captured graphs, share nothing.
//
// Beams with a score of -inf (or NaN) are not read: their continuations have the key -inf and count from token 0 on.  A NaN
// logit counts as -inf.  A row with logits of +inf has its mass on these, in equal shares.
#include "common.cuh"

namespace tk {

constexpr int kSelThreads = 512;
constexpr int kSelVecs = 2;                                    // 16-byte loads of a thread in one tile
constexpr int kSelTile = kSelThreads * 4 * kSelVecs;           // logits of a tile
constexpr int kSelBuffer = 2 * kSelTile;                       // elements set aside: a whole tile always fits behind what is kept
constexpr int kSelRanked = kSelThreads;                        // so many are ranked by comparing each with each
constexpr int kSelMaxK = 256;
constexpr int kSelMaxBeams = 64;
constexpr int kSelMaxEntries = 16384;                          // beams * segments * K that a joining block takes
constexpr float kSelRaise = 60.0f;                             // exponents above the reference that the sums hold

struct SelectParams {
  const float* logits;          // [groups * beams, vocab], row stride ld
  const float* scores;          // [groups, beams]
  double* seg_sum;              // [rows, segments, 2]: reference, sum of exponentials
  unsigned long long* seg_key;  // [rows, segments, K]: ordered logit, then ~token; 0 behind the last
  float* out_scores;            // [groups, K]
  int* out_parents;
  int* out_tokens;
  long long ld;
  int beams, vocab, k, segments, seg_len;
};

// Floats in an order that unsigned integers have too; both zeros are one.
__device__ __forceinline__ unsigned int ordered_f32(float v) {
  const unsigned int b = __float_as_uint(v + 0.0f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float from_ordered_f32(unsigned int o) {
  return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}
__device__ __forceinline__ unsigned long long ordered_f64(double v) {
  const unsigned long long b = (unsigned long long)__double_as_longlong(v + 0.0);
  return (b >> 63) ? ~b : (b | 0x8000000000000000ull);
}
__device__ __forceinline__ double from_ordered_f64(unsigned long long o) {
  return __longlong_as_double((long long)((o >> 63) ? (o & 0x7fffffffffffffffull) : ~o));
}

__device__ __forceinline__ bool dead_score(float s) { return !(s > -INFINITY); }        // -inf or NaN

// The largest threshold, bit by bit from the top, with at least k of the block's values at or above it; it stops early at one
// with at most `most`.  count(t) gives this thread's values at or above t.
template <typename U, typename Count>
__device__ __forceinline__ U block_threshold(int k, int most, Count count) {
  U t = 0;
  for (int bit = 8 * (int)sizeof(U) - 1; bit >= 0; --bit) {
    const U trial = t | ((U)1 << bit);
    // a thread's count may exceed one: the warps' sums are added up by the barrier's own reduction, bit by bit
    const int mine = count(trial);
    __shared__ int s_warp[2][kSelThreads / 32];
    const int sum = __reduce_add_sync(0xffffffffu, mine);
    int* w = s_warp[bit & 1];
    if ((threadIdx.x & 31) == 0) w[threadIdx.x >> 5] = sum;
    __syncthreads();
    int total = 0;
#pragma unroll
    for (int i = 0; i < kSelThreads / 32; ++i) total += w[i];
    if (total >= k) {
      t = trial;
      if (total <= most) break;
    }
  }
  __syncthreads();
  return t;
}

// Keeps the k largest (and a few behind them, up to kSelRanked) of the n distinct elements set aside; returns how many.
__device__ __forceinline__ int thin_out(unsigned long long* buf, int* s_count, int n, int k) {
  constexpr int PER = kSelBuffer / kSelThreads;
  unsigned long long mine[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int at = i * kSelThreads + threadIdx.x;
    mine[i] = at < n ? buf[at] : 0ull;
  }
  const unsigned long long t = block_threshold<unsigned long long>(k, kSelRanked, [&](unsigned long long trial) {
    int c = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) c += mine[i] >= trial ? 1 : 0;
    return c;
  });
  if (threadIdx.x == 0) *s_count = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (mine[i] != 0ull && mine[i] >= t) buf[atomicAdd(s_count, 1)] = mine[i];
  }
  __syncthreads();
  return *s_count;
}

__global__ void __launch_bounds__(kSelThreads)
beam_segments_kernel(SelectParams p) {
  pdl_trigger();
  extern __shared__ unsigned long long s_buf[];                // [kSelBuffer]
  __shared__ int s_count;
  __shared__ float s_max[kSelThreads / 32];
  __shared__ double s_sum[kSelThreads / 32];
  const int seg = blockIdx.x;
  const long long row = blockIdx.y;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const size_t at_part = (size_t)row * p.segments + seg;
  unsigned long long* out = p.seg_key + at_part * p.k;
  const int begin = seg * p.seg_len, end = min(p.vocab, begin + p.seg_len);
  pdl_wait();
  if (dead_score(p.scores[row])) {
    // the first tokens stand for a beam that cannot go on
    for (int i = threadIdx.x; i < p.k; i += kSelThreads) {
      out[i] = (seg == 0 && i < p.vocab) ? ((unsigned long long)ordered_f32(-INFINITY) << 32) | (0xffffffffu - (unsigned)i) : 0ull;
    }
    if (threadIdx.x == 0) { p.seg_sum[2 * at_part] = -INFINITY; p.seg_sum[2 * at_part + 1] = 0.0; }
    return;
  }
  const float* x = p.logits + row * p.ld;
  // 16-byte loads on their boundaries, wherever the row begins; what lies outside the segment is not read
  const int shift = (int)(((uintptr_t)x >> 2) & 3);
  const int v_begin = (begin + shift) / 4, v_end = (end + shift + 3) / 4;
  auto load = [&](int v, float (&e)[4]) {
    const int i0 = 4 * v - shift;
    if (i0 >= begin && i0 + 4 <= end) {
      const float4 f = __ldcs(reinterpret_cast<const float4*>(x + i0));
      e[0] = f.x; e[1] = f.y; e[2] = f.z; e[3] = f.w;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) e[j] = (i0 + j >= begin && i0 + j < end) ? x[i0 + j] : -INFINITY;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) e[j] = fmaxf(e[j], -INFINITY);          // a NaN becomes -inf
  };
  float e[kSelVecs][4];
  auto load_tile = [&](int v0) {
#pragma unroll
    for (int u = 0; u < kSelVecs; ++u) {
      const int v = v0 + u * kSelThreads + (int)threadIdx.x;
      if (v < v_end) load(v, e[u]);
      else e[u][0] = e[u][1] = e[u][2] = e[u][3] = -INFINITY;
    }
  };
  auto tile_max = [&]() {
    float m = -INFINITY;
#pragma unroll
    for (int u = 0; u < kSelVecs; ++u) m = fmaxf(m, fmaxf(fmaxf(e[u][0], e[u][1]), fmaxf(e[u][2], e[u][3])));
    return m;
  };
  auto set_aside = [&](int v0, unsigned int least, bool strict) {
#pragma unroll
    for (int u = 0; u < kSelVecs; ++u) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = 4 * (v0 + u * kSelThreads + (int)threadIdx.x) - shift + j;
        const unsigned int o = ordered_f32(e[u][j]);
        if (i >= begin && i < end && (strict ? o > least : o >= least)) {
          s_buf[atomicAdd(&s_count, 1)] = ((unsigned long long)o << 32) | (0xffffffffu - (unsigned)i);
        }
      }
    }
  };

  // ---- the first tile: a reference for the sums, and a threshold -----------------------------------------------
  if (threadIdx.x == 0) s_count = 0;
  load_tile(v_begin);
  float top = tile_max();
  {
    const float w = warp_max(top);
    if (lane == 0) s_max[warp] = w;
  }
  const unsigned int o_top = ordered_f32(top);
  const bool any = 4 * (v_begin + (int)threadIdx.x) - shift < end;
  unsigned int least = block_threshold<unsigned int>(p.k, p.k + 32, [&](unsigned int t) { return any && o_top >= t ? 1 : 0; });
  float ref = -INFINITY;
#pragma unroll
  for (int i = 0; i < kSelThreads / 32; ++i) ref = fmaxf(ref, s_max[i]);
  set_aside(v_begin, least, false);
  double sum = 0.0;
  float least_f = from_ordered_f32(least);        // 0 (fewer than K elements in all) is below every float's place: a NaN
  if (least == 0u) least_f = -INFINITY;

  // The sum of this tile's exponentials.  The reference is the first tile's maximum; it is raised (and what has been
  // summed so far scaled down) only where an exponent would leave the range that the sums hold.
  auto add_tile = [&]() {
    const float m = tile_max();
    if (!(m - ref <= kSelRaise)) {                // also with a reference of -inf or +inf
      if (m == -INFINITY) return;
      if (m == INFINITY || ref == INFINITY) {     // from the first +inf on these are counted, and nothing else
        if (ref != INFINITY) { sum = 0.0; ref = INFINITY; }
#pragma unroll
        for (int u = 0; u < kSelVecs; ++u) {
#pragma unroll
          for (int j = 0; j < 4; ++j) sum += e[u][j] == INFINITY ? 1.0 : 0.0;
        }
        return;
      }
      sum = ref == -INFINITY ? 0.0 : sum * exp((double)ref - (double)m);
      ref = m;
    }
#pragma unroll
    for (int u = 0; u < kSelVecs; ++u) {
      const float a = expf(e[u][0] - ref) + expf(e[u][1] - ref), b = expf(e[u][2] - ref) + expf(e[u][3] - ref);
      sum += (double)(a + b);
    }
  };
  add_tile();
  for (int v0 = v_begin + kSelThreads * kSelVecs; v0 < v_end; v0 += kSelThreads * kSelVecs) {
    load_tile(v0);
    if (tile_max() > least_f) set_aside(v0, least, true);
    add_tile();
    if (__syncthreads_or(s_count > kSelBuffer - kSelTile)) {
      // many elements in rising order: keep the best and raise the threshold
      int n = s_count;
      __syncthreads();
      n = thin_out(s_buf, &s_count, n, p.k);
      unsigned int lowest = threadIdx.x < n ? (unsigned int)(s_buf[threadIdx.x] >> 32) : 0xffffffffu;
      lowest = __reduce_min_sync(0xffffffffu, lowest);
      if (lane == 0) s_max[warp] = __uint_as_float(lowest);
      __syncthreads();
      least = 0xffffffffu;
#pragma unroll
      for (int i = 0; i < kSelThreads / 32; ++i) least = min(least, __float_as_uint(s_max[i]));
      least_f = from_ordered_f32(least);
      __syncthreads();
    }
  }
  __syncthreads();

  // ---- the segment's sum and its K best ---------------------------------------------------------------------------
  {
    const float w = warp_max(ref);
    if (lane == 0) s_max[warp] = w;
  }
  int n = s_count;
  __syncthreads();
  float ref_all = -INFINITY;
#pragma unroll
  for (int i = 0; i < kSelThreads / 32; ++i) ref_all = fmaxf(ref_all, s_max[i]);
  if (ref != ref_all) sum = (ref == -INFINITY || ref_all == INFINITY) ? 0.0 : sum * exp((double)ref - (double)ref_all);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) s_sum[warp] = sum;
  if (n > kSelRanked) n = thin_out(s_buf, &s_count, n, p.k);
  __syncthreads();
  if (threadIdx.x == 0) {
    double total = 0.0;
    for (int i = 0; i < kSelThreads / 32; ++i) total += s_sum[i];
    p.seg_sum[2 * at_part] = (double)ref_all;
    p.seg_sum[2 * at_part + 1] = total;
  }
  if ((int)threadIdx.x < n) {
    const unsigned long long mine = s_buf[threadIdx.x];
    int rank = 0;
    for (int i = 0; i < n; ++i) rank += s_buf[i] > mine ? 1 : 0;
    if (rank < p.k) out[rank] = mine;
  }
  for (int i = n + (int)threadIdx.x; i < p.k; i += kSelThreads) out[i] = 0ull;
}

// One block per group: the sums of its rows, the keys of the elements set aside, the K best of them in order.
__global__ void __launch_bounds__(kSelThreads)
beam_join_kernel(SelectParams p) {
  pdl_trigger();
  extern __shared__ unsigned long long s_key[];                // [beams * segments * K] keys in their order
  __shared__ double s_ref[kSelMaxBeams], s_log[kSelMaxBeams];
  __shared__ unsigned long long s_best[kSelRanked];
  __shared__ unsigned long long s_second[kSelRanked];
  __shared__ int s_count;
  const int group = blockIdx.x;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const size_t row0 = (size_t)group * p.beams;
  const int per_row = p.segments * p.k;
  const int n = p.beams * per_row;
  if (threadIdx.x == 0) s_count = 0;
  pdl_wait();
  for (int b = warp; b < p.beams; b += kSelThreads / 32) {
    const double* seg = p.seg_sum + (row0 + b) * p.segments * 2;
    double ref = -INFINITY;
    for (int s = lane; s < p.segments; s += 32) ref = fmax(ref, __ldcg(seg + 2 * s));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ref = fmax(ref, __shfl_xor_sync(0xffffffffu, ref, o));
    double sum = 0.0;
    for (int s = lane; s < p.segments; s += 32) {
      const double m = __ldcg(seg + 2 * s), part = __ldcg(seg + 2 * s + 1);
      if (m == ref) sum += part;
      else if (m != -INFINITY && ref != INFINITY) sum += part * exp(m - ref);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) { s_ref[b] = ref; s_log[b] = log(sum); }
  }
  __syncthreads();
  auto key_of = [&](int b, unsigned long long elem) {
    const double x = (double)from_ordered_f32((unsigned int)(elem >> 32));
    const double s = (double)p.scores[row0 + b];
    const double ref = s_ref[b];
    double key = s + ((ref == INFINITY ? (x == INFINITY ? 0.0 : -INFINITY) : x - ref) - s_log[b]);
    if (!(key > -INFINITY)) key = -INFINITY;                   // dead beams, -inf logits, rows of -inf alone
    return ordered_f64(key);
  };
  const unsigned long long* elems = p.seg_key + row0 * per_row;
  for (int i = threadIdx.x; i < n; i += kSelThreads) {
    const unsigned long long elem = __ldcg(elems + i);
    s_key[i] = elem == 0ull ? 0ull : key_of(i / per_row, elem);
  }
  __syncthreads();
  // what comes after the key: the logit where it decides, then the place
  auto second_of = [&](int i) {
    const unsigned long long elem = __ldcg(elems + i);
    const unsigned int place = (unsigned int)(i / per_row) * (unsigned int)p.vocab + (0xffffffffu - (unsigned int)elem);
    const unsigned int logit = s_key[i] == ordered_f64(-INFINITY) ? 0u : (unsigned int)(elem >> 32);
    return ((unsigned long long)logit << 32) | (0xffffffffu - place);
  };
  unsigned long long t = 1ull;                                   // everything there is
  if (n > kSelRanked) {
    t = block_threshold<unsigned long long>(p.k, kSelRanked, [&](unsigned long long trial) {
      int c = 0;
      for (int i = threadIdx.x; i < n; i += kSelThreads) c += s_key[i] >= trial ? 1 : 0;
      return c;
    });
    if (t == 0ull) t = 1ull;
  }
  // Where more than can be ranked share the K-th key (beams that all are dead, rows of equal logits), the same search goes on
  // over what comes after the key.
  int mine = 0, above = 0;
  for (int i = threadIdx.x; i < n; i += kSelThreads) { mine += s_key[i] >= t ? 1 : 0; above += s_key[i] > t ? 1 : 0; }
  unsigned long long t2 = 0ull;
  {
    __shared__ int s_sums[2][kSelThreads / 32];
    mine = __reduce_add_sync(0xffffffffu, mine);
    above = __reduce_add_sync(0xffffffffu, above);
    if (lane == 0) { s_sums[0][warp] = mine; s_sums[1][warp] = above; }
    __syncthreads();
    mine = above = 0;
#pragma unroll
    for (int i = 0; i < kSelThreads / 32; ++i) { mine += s_sums[0][i]; above += s_sums[1][i]; }
  }
  if (mine > kSelRanked) {
    t2 = block_threshold<unsigned long long>(p.k - above, kSelRanked - above, [&](unsigned long long trial) {
      int c = 0;
      for (int i = threadIdx.x; i < n; i += kSelThreads) c += (s_key[i] == t && second_of(i) >= trial) ? 1 : 0;
      return c;
    });
  }
  for (int i = threadIdx.x; i < n; i += kSelThreads) {
    if (s_key[i] > t || (s_key[i] == t && (t2 == 0ull || second_of(i) >= t2))) {
      const int at = atomicAdd(&s_count, 1);
      s_best[at] = s_key[i];
      s_second[at] = second_of(i);
    }
  }
  __syncthreads();
  const int m = s_count;
  if ((int)threadIdx.x < m) {
    const unsigned long long a = s_best[threadIdx.x], b = s_second[threadIdx.x];
    int rank = 0;
    for (int i = 0; i < m; ++i) rank += (s_best[i] > a || (s_best[i] == a && s_second[i] > b)) ? 1 : 0;
    if (rank < p.k) {
      const size_t at = (size_t)group * p.k + rank;
      const unsigned int place = 0xffffffffu - (unsigned int)b;
      p.out_scores[at] = (float)from_ordered_f64(a);
      p.out_parents[at] = (int)(place / (unsigned int)p.vocab);
      p.out_tokens[at] = (int)(place % (unsigned int)p.vocab);
    }
  }
}

// ---- the next step's beams ---------------------------------------------------------------------------------------
//
// Of a group's candidates, in order, the first W whose token is no stop token go on.  A beam whose parent has not been
// claimed by a better one stays in its parent's seat; the others take the seats that are left, in order.  So a seat that
// goes on is never written, and what has to move is one record for every beam that ends.  A seat that is left without a
// candidate (a vocabulary of stop tokens) keeps its parent with a score of -inf.
struct AdvanceParams {
  const float* cand_scores;     // [groups, K], best first
  const int* cand_parents;
  const int* cand_tokens;
  const int* stop_tokens;       // [n_stop]
  const int* slots;             // [groups, beams]
  float* scores;                // [groups, beams], rewritten
  int* parents;                 // [groups, beams]: the seat that each seat goes on from
  int* tokens;                  // [groups, beams]
  int* records;                 // [max_slots, words] or null: word `token_word` receives the token
  unsigned char* history;       // [max_slots, history_ld] or null
  const int* positions;         // [groups * beams]: the position that this step wrote
  const int* prefix_len;        // [groups]: positions in front of the history
  int* err;
  int k, beams, n_stop, max_slots, words, token_word, history_ld, from_one;
};

__global__ void __launch_bounds__(64) beam_advance_kernel(AdvanceParams p) {
  pdl_trigger();
  __shared__ int s_cand[kSelMaxBeams];       // candidate of every seat, -1: none yet
  __shared__ int s_late[kSelMaxBeams];
  pdl_wait();
  const int g = blockIdx.x;
  const size_t c0 = (size_t)g * p.k, b0 = (size_t)g * p.beams;
  const int seat = threadIdx.x;
  if (seat < p.beams) s_cand[seat] = -1;
  __syncthreads();
  if (threadIdx.x == 0) {
    int taken = 0, late = 0;
    for (int i = 0; i < p.k && taken < p.beams; ++i) {
      if (!(p.cand_scores[c0 + i] > -INFINITY)) break;          // what comes now cannot go on
      const int tok = p.cand_tokens[c0 + i];
      bool stop = false;
      for (int j = 0; j < p.n_stop; ++j) stop = stop || p.stop_tokens[j] == tok;
      if (stop) continue;
      const int parent = p.cand_parents[c0 + i];
      // out of one row (a search that begins) the beams take the seats in order
      const int want = p.from_one ? taken : parent;
      if (want >= 0 && want < p.beams && s_cand[want] < 0) s_cand[want] = i;
      else s_late[late++] = i;
      ++taken;
    }
    int next = 0;
    for (int i = 0; i < late; ++i) {
      while (s_cand[next] >= 0) ++next;
      s_cand[next] = s_late[i];
    }
  }
  __syncthreads();
  if (seat >= p.beams) return;
  const int c = s_cand[seat];
  const int token = c >= 0 ? p.cand_tokens[c0 + c] : 0;
  int parent = c >= 0 && !p.from_one ? p.cand_parents[c0 + c] : seat;
  if (parent < 0 || parent >= p.beams) { set_error(p.err, kErrRequest, g, parent, p.beams); parent = seat; }
  p.scores[b0 + seat] = c >= 0 ? p.cand_scores[c0 + c] : -INFINITY;
  p.parents[b0 + seat] = parent;
  p.tokens[b0 + seat] = token;
  const int slot = p.slots[b0 + seat];
  if (slot < 0 || slot >= p.max_slots) { set_error(p.err, kErrRequest, g, slot, p.max_slots); return; }
  if (p.records != nullptr) p.records[(size_t)slot * p.words + p.token_word] = token;
  if (p.history != nullptr && !p.from_one) {
    // the position of this step lies in the seat's own pages; the records move afterwards, and this with them
    const int n = p.positions[b0 + seat] - p.prefix_len[g];
    if (n < 0 || n >= p.history_ld) set_error(p.err, kErrPosition, g, n, p.history_ld);
    else p.history[(size_t)slot * p.history_ld + n] = (unsigned char)seat;
  }
}

// ---- records that follow their beams --------------------------------------------------------------------------------
//
// records[key][slots[g, i]] becomes what records[key][slots[g, parents[g, i]]] was, for all seats i of a group at once and in
// place.  A thread owns a column of 16 bytes (less where the records' size or address asks for it) of all records of one
// group: it reads every source that moves, then writes, so no order of the moves can go wrong and no copy is made.  Bound by
// the bytes: sources that move are read, seats that change are written, nothing else is touched.
constexpr int kMoveThreads = 256;
constexpr int kMoveMaxTensors = 24;
constexpr int kMoveMaxSeats = 64;

struct MoveTensor {
  unsigned char* base;          // [keys, max_slots, bytes]
  long long bytes;              // of a record
  long long first_block;        // of the grid's x that belongs to this tensor
  int keys, vec;                // bytes of a thread's column: 16, 8, 4, 2 or 1
};
struct MoveParams {
  MoveTensor t[kMoveMaxTensors];
  const int* slots;             // [groups, seats]
  const int* parents;           // [groups, seats]
  int* err;
  int n_tensors, seats, max_slots;
};

template <typename V, int kSeats>
__device__ __forceinline__ void move_column(const MoveTensor& t, long long at, const int* s_src, const int* s_dst, int n, int max_slots) {
  const long long columns = t.bytes / (long long)sizeof(V);
  if (at >= columns * t.keys) return;
  const long long key = at / columns, col = at % columns;
  V* base = reinterpret_cast<V*>(t.base) + key * max_slots * columns + col;
  V v[kSeats];
#pragma unroll
  for (int i = 0; i < kSeats; ++i) {
    if (i < n) v[i] = base[(long long)s_src[i] * columns];
  }
#pragma unroll
  for (int i = 0; i < kSeats; ++i) {
    if (i < n) base[(long long)s_dst[i] * columns] = v[i];
  }
}

template <int kSeats>
__global__ void __launch_bounds__(kMoveThreads) reorder_slots_kernel(const __grid_constant__ MoveParams p) {
  pdl_trigger();
  __shared__ int s_src[kMoveMaxSeats], s_dst[kMoveMaxSeats];
  __shared__ int s_n;
  pdl_wait();
  const int g = blockIdx.y;
  if (threadIdx.x < 32) {
    // the seats that change, in order
    int n = 0;
    for (int i0 = 0; i0 < p.seats; i0 += 32) {
      const int i = i0 + (int)threadIdx.x;
      bool moves = false;
      int src = 0, dst = 0;
      if (i < p.seats) {
        const int parent = p.parents[(size_t)g * p.seats + i];
        dst = p.slots[(size_t)g * p.seats + i];
        if (parent < 0 || parent >= p.seats) {
          set_error(p.err, kErrRequest, g, parent, p.seats);
        } else if (parent != i) {
          src = p.slots[(size_t)g * p.seats + parent];
          if (src < 0 || src >= p.max_slots || dst < 0 || dst >= p.max_slots) {
            set_error(p.err, kErrRequest, g, src < 0 || src >= p.max_slots ? src : dst, p.max_slots);
          } else {
            moves = src != dst;
          }
        }
      }
      const unsigned mask = __ballot_sync(0xffffffffu, moves);
      if (moves) {
        const int at = n + __popc(mask & ((1u << threadIdx.x) - 1u));
        s_src[at] = src;
        s_dst[at] = dst;
      }
      n += __popc(mask);
    }
    if (threadIdx.x == 0) s_n = n;
  }
  __syncthreads();
  const int n = s_n;
  if (n == 0) return;
  int k = 0;
  while (k + 1 < p.n_tensors && (long long)blockIdx.x >= p.t[k + 1].first_block) ++k;
  const MoveTensor& t = p.t[k];
  const long long at = ((long long)blockIdx.x - t.first_block) * kMoveThreads + threadIdx.x;
  if (kSeats <= 32 && t.vec == 16) move_column<uint4, (kSeats <= 32 ? kSeats : 1)>(t, at, s_src, s_dst, n, p.max_slots);
  else if (t.vec == 8) move_column<uint2, kSeats>(t, at, s_src, s_dst, n, p.max_slots);
  else if (t.vec == 4) move_column<unsigned int, kSeats>(t, at, s_src, s_dst, n, p.max_slots);
  else if (t.vec == 2) move_column<unsigned short, kSeats>(t, at, s_src, s_dst, n, p.max_slots);
  else move_column<unsigned char, kSeats>(t, at, s_src, s_dst, n, p.max_slots);
}

}  // namespace tk

TK_API int tk_beam_select_tile(void) { return tk::kSelTile; }
TK_API int tk_beam_max_beams(void) { return tk::kSelMaxBeams; }
TK_API int tk_beam_max_candidates(void) { return tk::kSelMaxK; }
TK_API int tk_beam_max_entries(void) { return tk::kSelMaxEntries; }
TK_API int tk_reorder_max_tensors(void) { return tk::kMoveMaxTensors; }

// scratch: rows * segments * (16 + 8 k) bytes, on 8 bytes.
TK_API int tk_beam_select(const float* logits, long long ld, const float* scores, void* scratch, float* out_scores,
                          int* out_parents, int* out_tokens, int groups, int beams, int vocab, int k, int segments,
                          cudaStream_t stream) {
  if (groups <= 0) return 0;
  if (beams < 1 || beams > tk::kSelMaxBeams || k < 1 || k > tk::kSelMaxK || vocab < 1 || segments < 1 || ld < vocab ||
      (long long)beams * segments * k > tk::kSelMaxEntries || (long long)beams * vocab > 0x7fffffffLL ||
      (long long)groups * beams > 65535 || (long long)k > (long long)beams * vocab) {
    return (int)cudaErrorInvalidValue;
  }
  tk::SelectParams p;
  p.logits = logits; p.scores = scores; p.ld = ld;
  const long long parts = (long long)groups * beams * segments;
  p.seg_sum = (double*)scratch;
  p.seg_key = (unsigned long long*)scratch + 2 * parts;
  p.out_scores = out_scores; p.out_parents = out_parents; p.out_tokens = out_tokens;
  p.beams = beams; p.vocab = vocab; p.k = k; p.segments = segments;
  p.seg_len = (vocab + segments - 1) / segments;
  constexpr int seg_smem = tk::kSelBuffer * 8;
  const int join_smem = beams * segments * k * 8;
  static bool configured[64] = {false};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return (int)e;
  if (dev < 0 || dev >= 64) return (int)cudaErrorInvalidValue;
  if (!configured[dev]) {
    e = cudaFuncSetAttribute(tk::beam_segments_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, seg_smem);
    if (e != cudaSuccess) return (int)e;
    e = cudaFuncSetAttribute(tk::beam_join_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, tk::kSelMaxEntries * 8);
    if (e != cudaSuccess) return (int)e;
    configured[dev] = true;
  }
  e = tk::launch(tk::beam_segments_kernel, dim3(segments, groups * beams), dim3(tk::kSelThreads), seg_smem, stream, p);
  if (e != cudaSuccess) return (int)e;
  return (int)tk::launch(tk::beam_join_kernel, dim3(groups), dim3(tk::kSelThreads), join_smem, stream, p);
}

TK_API int tk_beam_advance(const float* cand_scores, const int* cand_parents, const int* cand_tokens, const int* stop_tokens,
                           const int* slots, float* scores, int* parents, int* tokens, int* records,
                           unsigned char* history, const int* positions, const int* prefix_len, int* err, int groups, int beams, int k, int n_stop,
                           int max_slots, int words, int token_word, int history_ld, int from_one, cudaStream_t stream) {
  if (groups <= 0) return 0;
  if (beams < 1 || beams > tk::kSelMaxBeams || k < 1 || n_stop < 0) return (int)cudaErrorInvalidValue;
  tk::AdvanceParams p{cand_scores, cand_parents, cand_tokens, stop_tokens, slots, scores, parents, tokens, records, history,
                      positions, prefix_len, err, k, beams, n_stop, max_slots, words, token_word, history_ld, from_one};
  return (int)tk::launch(tk::beam_advance_kernel, dim3(groups), dim3(64), 0, stream, p);
}

// bases, bytes, keys: of every tensor; a record's bytes and its tensor's address decide how wide its columns are.
TK_API int tk_reorder_slots(void* const* bases, const long long* bytes, const int* keys, int n_tensors, const int* slots,
                            const int* parents, int* err, int groups, int seats, int max_slots, cudaStream_t stream) {
  if (groups <= 0 || n_tensors <= 0) return 0;
  if (n_tensors > tk::kMoveMaxTensors || seats < 1 || seats > tk::kMoveMaxSeats || groups > 65535 || max_slots < 1) {
    return (int)cudaErrorInvalidValue;
  }
  tk::MoveParams p;
  p.slots = slots; p.parents = parents; p.err = err; p.n_tensors = 0; p.seats = seats; p.max_slots = max_slots;
  long long blocks = 0;
  for (int i = 0; i < n_tensors; ++i) {
    if (bytes[i] < 0 || keys[i] < 0) return (int)cudaErrorInvalidValue;
    if (bytes[i] == 0 || keys[i] == 0) continue;
    tk::MoveTensor& t = p.t[p.n_tensors++];
    t.base = (unsigned char*)bases[i];
    t.bytes = bytes[i];
    t.keys = keys[i];
    t.vec = 16;
    // 64 seats of 16 bytes would not fit a thread's registers
    if (seats > 32) t.vec = 8;
    while (((uintptr_t)bases[i] | (unsigned long long)bytes[i]) % (unsigned long long)t.vec) t.vec /= 2;
    t.first_block = blocks;
    blocks += (t.bytes / t.vec * t.keys + tk::kMoveThreads - 1) / tk::kMoveThreads;
  }
  if (blocks == 0) return 0;
  if (blocks > 0x7fffffffLL) return (int)cudaErrorInvalidValue;
  const dim3 grid((unsigned)blocks, groups);
  if (seats <= 4) return (int)tk::launch(tk::reorder_slots_kernel<4>, grid, dim3(tk::kMoveThreads), 0, stream, p);
  if (seats <= 8) return (int)tk::launch(tk::reorder_slots_kernel<8>, grid, dim3(tk::kMoveThreads), 0, stream, p);
  if (seats <= 16) return (int)tk::launch(tk::reorder_slots_kernel<16>, grid, dim3(tk::kMoveThreads), 0, stream, p);
  if (seats <= 32) return (int)tk::launch(tk::reorder_slots_kernel<32>, grid, dim3(tk::kMoveThreads), 0, stream, p);
  return (int)tk::launch(tk::reorder_slots_kernel<64>, grid, dim3(tk::kMoveThreads), 0, stream, p);
}
