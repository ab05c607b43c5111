// Search over beams: the best continuations of the beams of every group, and what follows from them for the next step.
//
// Selection.  Beam w of a group has a score s_w (the sum of its tokens' log probabilities) and a row of logits x_w; its
// continuation by token v has the key
//     key(w, v) = s_w + ((x_wv - M_w) - log sum_u exp(x_wu - M_w)),      M_w any reference of the row,
// and the K largest keys of a group's W * V are wanted in order; equal keys: the lower beam, of one beam the larger logit, then
// the lower token.  Keys of neighbouring ranks differ by less than a float's last place often enough to change what a
// search does, so sums and keys are 64-bit.  The exponentials are floats, added four at a time as floats and then as doubles, and the
// largest, those of the candidates, are put right in 64 bits: a row's logarithm is off by some 1e-8 to 1e-7, each row's by its own,
// and two rows' by no more than order_bound() says.  Where continuations of different beams are closer than that and it matters, the
// joining kernel forms the sums of their rows again, with every exponential in 64 bits, and ranks once more: in one call of
// forty of 32 groups of 16 beams, which then takes 60 us more.  (With all exponentials in 64 bits each of these calls takes 103 us
// instead of 56.)
//
// One pass over the logits.  Within a row the order of the keys is that of the logits, so the K best of a row's segment can
// be kept without knowing the row's sum: a block streams its segment in tiles, holds a threshold with at least K elements
// at or above it, and sets aside only what is above (the threshold of the first tile is the K-th largest of the threads'
// own maxima; it rises when four and sixteen times as many logits have been seen).  A second kernel, started early, has a block per
// group: it adds the segments' sums up in their order, makes the keys of the elements set aside and ranks them.  Two kernels and
// no counter: calls on two streams, or two captured graphs, share nothing.
//
// Bound by the logits' bytes where there are many: 205 MB (512 rows of 100,003) in 56 us, 3.7 TB/s; what is left are the
// instructions beside the loads, an exponential and a comparison a logit (44 us without either).  Few rows are bound by
// latency: 10 us for one row of 151,936, 16 for 32.
//
// Beams with a score of -inf (or NaN) are not read: their continuations have the key -inf and count from token 0 on.  A NaN
// logit counts as -inf.  A row with logits of +inf has its mass on these, in equal shares.
#include "common.cuh"

#include <type_traits>

namespace tk {

constexpr int kSelThreads = 256;
constexpr int kSelEach = 14;                                   // logits of a thread in one tile (16: 60 us for 512 rows of 100,003 instead
                                                               // of 54, more than the registers hold; 10: 58)
constexpr int kSelTile = kSelThreads * kSelEach;               // logits of a tile
constexpr int kSelCheck = 4;                                   // tiles between two looks at how many were set aside
constexpr int kSelKept = 512;                                  // elements set aside that are left when they are thinned out
constexpr int kSelBuffer = 2048;                               // elements set aside
constexpr int kJoinThreads = 512;                              // and so many are ranked by comparing each with each
constexpr int kSelMaxK = 256;
constexpr int kSelMaxBeams = 64;
constexpr int kSelTokenBits = 26;                              // of a token in what ranks behind a key
constexpr int kSelMaxEntries = 16384;                          // beams * segments * K that a joining block takes
constexpr float kSelRaise = 12.0f;                             // exponents above the reference that the sums hold

struct SelectParams {
  const float* logits;          // [groups * beams, vocab], row stride ld
  const void* scores;           // [groups, beams], of the type that the kernels are made for
  double* seg_sum;              // [rows, segments, 2]: reference, sum of exponentials
  unsigned long long* seg_key;  // [rows, segments, K]: ordered logit, then ~token; 0 behind the last
  void* out_scores;             // [groups, K]
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

__device__ __forceinline__ bool dead_score(double s) { return !(s > -INFINITY); }       // -inf or NaN

// The largest threshold, bit by bit from the top, with at least k of the block's values at or above it; it stops early at one
// with at most `most`.  count(t) gives this thread's values at or above t.
template <int kThreads, typename U, typename Count>
__device__ __forceinline__ U block_threshold(int k, int most, Count count) {
  __shared__ int s_warp[2][kThreads / 32];
  U t = 0;
  for (int bit = 8 * (int)sizeof(U) - 1; bit >= 0; --bit) {
    const U trial = t | ((U)1 << bit);
    const int sum = __reduce_add_sync(0xffffffffu, count(trial));
    int* w = s_warp[bit & 1];
    if ((threadIdx.x & 31) == 0) w[threadIdx.x >> 5] = sum;
    __syncthreads();
    int total = 0;
#pragma unroll
    for (int i = 0; i < kThreads / 32; ++i) total += w[i];
    if (total >= k) {
      t = trial;
      if (total <= most) break;
    }
  }
  __syncthreads();
  return t;
}

// The same with one value a thread, which the barrier itself counts.
template <typename U>
__device__ __forceinline__ U block_threshold_of(int k, int most, bool any, U value) {
  U t = 0;
  for (int bit = 8 * (int)sizeof(U) - 1; bit >= 0; --bit) {
    const U trial = t | ((U)1 << bit);
    const int total = __syncthreads_count(any && value >= trial);
    if (total >= k) {
      t = trial;
      if (total <= most) break;
    }
  }
  return t;
}

// Those of the n elements set aside that are at or above t are kept.  Returns how many.
__device__ __noinline__ int keep_from(unsigned long long* buf, int* s_count, int n, unsigned long long t) {
  constexpr int PER = kSelBuffer / kSelThreads;
  unsigned long long mine[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int at = i * kSelThreads + threadIdx.x;
    mine[i] = at < n ? buf[at] : 0ull;
  }
  __syncthreads();
  if (threadIdx.x == 0) *s_count = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (mine[i] != 0ull && mine[i] >= t) buf[atomicAdd(s_count, 1)] = mine[i];
  }
  __syncthreads();
  return *s_count;
}

// Of the n elements set aside those of tokens before `limit` are kept, and of these, where they are more than kSelKept, the k
// largest (and a few behind them, up to kSelKept).  Returns how many.  (Elements are distinct.)
__device__ __noinline__ int thin_out(unsigned long long* buf, int* s_count, int n, int k, unsigned int limit) {
  constexpr int PER = kSelBuffer / kSelThreads;
  unsigned long long mine[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int at = i * kSelThreads + threadIdx.x;
    mine[i] = at < n ? buf[at] : 0ull;
    if (0xffffffffu - (unsigned int)mine[i] >= limit) mine[i] = 0ull;
  }
  const unsigned long long t = block_threshold<kSelThreads, unsigned long long>(k, kSelKept, [&](unsigned long long trial) {
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

// The smallest logit of the n elements set aside (at most kSelKept), as a float.
__device__ __forceinline__ float lowest_of(const unsigned long long* buf, int n) {
  __shared__ unsigned int s_low[kSelThreads / 32];
  unsigned int low = 0xffffffffu;
  for (int i = threadIdx.x; i < n; i += kSelThreads) low = min(low, (unsigned int)(buf[i] >> 32));
  low = __reduce_min_sync(0xffffffffu, low);
  if ((threadIdx.x & 31) == 0) s_low[threadIdx.x >> 5] = low;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kSelThreads / 32; ++i) low = min(low, s_low[i]);
  __syncthreads();
  return from_ordered_f32(low);
}

// s_rank[j] (zero before) becomes the number of the n elements that come before element j: as many threads as there are work on
// each of up to a block's threads, or a thread on several.
template <int kThreads, typename Before>
__device__ __forceinline__ void rank_by_slices(int n, int* s_rank, Before before) {
  const int slices = max(1, kThreads / max(1, n));
  const int slice = (int)threadIdx.x / max(1, n);
  if (slice < slices) {
    for (int j = slice == 0 ? (int)threadIdx.x : (int)threadIdx.x % n; j < n; j += kThreads) {
      int c = 0;
      for (int i = slice; i < n; i += slices) c += before(i, j) ? 1 : 0;
      if (slices > 1) atomicAdd(&s_rank[j], c);
      else s_rank[j] = c;
    }
  }
  __syncthreads();
}

// Exponentials as the sums take them: a subtraction that is exact for the terms that matter, a product, and the fast power of two.
__device__ __forceinline__ float2 terms_f32(float x, float y, float ref) {
  float2 d = mul2(add2(make_float2(x, y), make_float2(-ref, -ref)), make_float2(1.4426950408889634f, 1.4426950408889634f));
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(d.x));
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(d.y));
  return d;
}

// How far apart the logarithms of two rows' sums may be from what they are by the float exponentials.  A term e^d is off by 2^-24 |d|
// each for the roundings of d and of d log2(e), 1.4e-8 |d| for the constant's, 2^-22 for the power of two and 2^-23 for two additions,
// relative to itself.  Weighed by the terms themselves, |d| is no more than kSelRaise where d > 0, and, since the reference is a term,
// no more than ln(vocab) where d < 0; both kinds together no more than the larger of the two and 1 / e.
__device__ __forceinline__ double order_bound(int vocab) {
  return 2.0 * (1.34e-7 * ((double)fmaxf(kSelRaise, logf((float)vocab)) + 0.4) + 3.7e-7);
}

// Exponentials in 64 bits, added to one of two sums in turn, of d = x - ref in (-87, 87): 2^(k / 16) from a table, times the series of e^r up to r^5 / 120,
// r = d - k ln(2) / 16 (table-driven, after P. T. P. Tang, 1989).  |r| <= ln(2) / 32, so the terms left out are less than 1.5e-13
// of it.
__constant__ double kPowers[16] = {           // 2^(j / 16)
    0x1.0000000000000p+0, 0x1.0b5586cf9890fp+0, 0x1.172b83c7d517bp+0, 0x1.2387a6e756238p+0,
    0x1.306fe0a31b715p+0, 0x1.3dea64c123422p+0, 0x1.4bfdad5362a27p+0, 0x1.5ab07dd485429p+0,
    0x1.6a09e667f3bcdp+0, 0x1.7a11473eb0187p+0, 0x1.8ace5422aa0dbp+0, 0x1.9c49182a3f090p+0,
    0x1.ae89f995ad3adp+0, 0x1.c199bdd85529cp+0, 0x1.d5818dcfba487p+0, 0x1.ea4afa2a490dap+0};
template <int N>
__device__ __forceinline__ void add_terms(double (&sum)[2], const float* x, float ref, double ref64, const double* powers) {
  const double whole = 6755399441055744.0;             // 1.5 * 2^52: what is added to it is rounded to a whole number
  double r[N], scaled[N], e[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const double d = (double)x[i] - ref64, shifted = fma(d, 0x1.71547652b82fep+4, whole);
    const int k = __double2loint(shifted);
    r[i] = fma(shifted - whole, -0x1.62e42fefa39efp-5, d);
    const double t = powers[k & 15];
    scaled[i] = __hiloint2double(__double2hiint(t) + ((k & ~15) << 16), __double2loint(t));
  }
#pragma unroll
  for (int i = 0; i < N; ++i) e[i] = fma(r[i], 1.0 / 120.0, 1.0 / 24.0);
#pragma unroll
  for (int i = 0; i < N; ++i) e[i] = fma(r[i], e[i], 1.0 / 6.0);
#pragma unroll
  for (int i = 0; i < N; ++i) e[i] = fma(r[i], e[i], 0.5);
#pragma unroll
  for (int i = 0; i < N; ++i) e[i] = fma(r[i], e[i], 1.0);
#pragma unroll
  for (int i = 0; i < N; ++i) e[i] = fma(r[i], e[i], 1.0);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (x[i] - ref > -87.0f) sum[i & 1] = fma(scaled[i], e[i], sum[i & 1]);          // e^-87 is nothing beside the reference's own term
  }
}

// kPerSm: blocks on an SM at a time.  Four leave a thread 64 registers, and it keeps some of its values in memory; where there are
// no more blocks than three an SM take, they are faster by themselves: 8 groups of 4 beams over 151,936 tokens in 13 segments, 416 blocks,
// 19.9 us against 21.8 (and 22.4 in 15 segments, 480 blocks, with four; inputs not in L2).  512 rows of 100,003 logits, more than that:
// 68 us with three, 55 with four.  With 64-bit exponentials 20.0 against 24.0.
template <int kPerSm, typename Score>
__global__ void __launch_bounds__(kSelThreads, kPerSm)
beam_segments_kernel(SelectParams p) {
  constexpr bool kWide = sizeof(Score) == 8;      // exponentials in 64 bits
  pdl_trigger();
  __shared__ unsigned long long s_buf[kSelBuffer];
  __shared__ int s_count, s_rank[kSelKept];
  __shared__ float s_max[kSelThreads / 32];
  __shared__ double s_sum[kSelThreads / 32], s_late[kWide ? 1 : kSelMaxK], s_powers[16];
  const int seg = blockIdx.x;
  const long long row = blockIdx.y;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const size_t at_part = (size_t)row * p.segments + seg;
  unsigned long long* out = p.seg_key + at_part * p.k;
  const int begin = min(p.vocab, seg * p.seg_len), end = min(p.vocab, begin + p.seg_len);
  if (kWide && threadIdx.x < 16) s_powers[threadIdx.x] = kPowers[threadIdx.x];
  pdl_wait();
  if (dead_score(((const Score*)p.scores)[row])) {
    // the first tokens stand for a beam that cannot go on
    for (int i = threadIdx.x; i < p.k; i += kSelThreads) {
      out[i] = (seg == 0 && i < p.vocab) ? ((unsigned long long)ordered_f32(-INFINITY) << 32) | (0xffffffffu - (unsigned)i) : 0ull;
    }
    if (threadIdx.x == 0) { p.seg_sum[2 * at_part] = -INFINITY; p.seg_sum[2 * at_part + 1] = 0.0; }
    return;
  }
  const float* x = p.logits + row * p.ld;
  // A thread takes every kSelThreads-th logit of a tile, wherever the row begins: two rows with the same logits have the same
  // sum to the last bit then, whatever their addresses, and their continuations are ties.
  auto load_tile = [&](int t0, float (&e)[kSelEach]) {
    const float* src = x + t0 + threadIdx.x;
    if (t0 + kSelTile <= end) {
#pragma unroll
      for (int j = 0; j < kSelEach; ++j) e[j] = __ldcs(src + j * kSelThreads);
    } else {
#pragma unroll
      for (int j = 0; j < kSelEach; ++j) e[j] = t0 + j * kSelThreads + (int)threadIdx.x < end ? src[j * kSelThreads] : -INFINITY;
    }
  };
  auto clean = [&](float (&e)[kSelEach]) {                        // a NaN becomes -inf
#pragma unroll
    for (int j = 0; j < kSelEach; ++j) e[j] = fmaxf(e[j], -INFINITY);
  };
  auto tile_max = [&](const float (&e)[kSelEach]) {
    float m = fmaxf(e[0], e[1]);
#pragma unroll
    for (int j = 2; j < kSelEach; j += 2) m = fmaxf(m, fmaxf(e[j], e[j + 1]));
    return m;
  };
  auto set_aside = [&](int i, float v) {
    const int at = atomicAdd(&s_count, 1);
    if (at < kSelBuffer) s_buf[at] = ((unsigned long long)ordered_f32(v) << 32) | (0xffffffffu - (unsigned)i);
  };

  // ---- the first tile: a reference for the sums, and a threshold -----------------------------------------------
  if (threadIdx.x == 0) s_count = 0;
  float cur[kSelEach], nxt[kSelEach];
  load_tile(begin, cur);
  if (begin + kSelTile < end) load_tile(begin + kSelTile, nxt);
  clean(cur);
  const float top = tile_max(cur);
  {
    const float w = warp_max(top);
    if (lane == 0) s_max[warp] = w;
  }
  const unsigned int o_least = block_threshold_of<unsigned int>(p.k, p.k, begin + (int)threadIdx.x < end, ordered_f32(top));
  float ref = -INFINITY;
#pragma unroll
  for (int i = 0; i < kSelThreads / 32; ++i) ref = fmaxf(ref, s_max[i]);
  // elements at or above this are set aside in the first tile, those above it in later ones: what is equal and comes later
  // loses.  (At or below -inf's place: fewer than K threads have an element that is more.)
  float least = o_least <= ordered_f32(-INFINITY) ? -INFINITY : from_ordered_f32(o_least);
  double sum = 0.0;

  // More elements than the buffer holds: those of the tiles from t0 to t1, before which all were held, are set aside again, a row
  // of a block's threads at a time, with the threshold raised in between.  (Logits in rising order, or many equal ones.)
  auto crowded = [&](int t0, int t1, bool first) {
    int n = thin_out(s_buf, &s_count, min(s_count, kSelBuffer), p.k, (unsigned int)t0);
    bool reached = first;                         // whether an element equal to the threshold still counts
    if (n >= p.k) { least = lowest_of(s_buf, n); reached = false; }
    for (int i0 = t0; i0 < min(t1, end); i0 += kSelThreads) {
      const int i = i0 + (int)threadIdx.x;
      const float v = i < end ? x[i] : -INFINITY;
      if (i < end && (reached ? fmaxf(v, -INFINITY) >= least : v > least)) set_aside(i, fmaxf(v, -INFINITY));
      __syncthreads();
      n = s_count;
      __syncthreads();
      if (n > kSelBuffer - kSelThreads) {
        n = thin_out(s_buf, &s_count, n, p.k, 0xffffffffu);
        least = lowest_of(s_buf, n);
        reached = false;
      }
    }
  };
#pragma unroll
  for (int j = 0; j < kSelEach; ++j) {
    if (cur[j] >= least && begin + j * kSelThreads + (int)threadIdx.x < end) set_aside(begin + j * kSelThreads + (int)threadIdx.x, cur[j]);
  }
  if (__syncthreads_or(s_count > kSelBuffer)) crowded(begin, begin + kSelTile, true);

  // The sum of a tile's exponentials.  The reference is the first tile's maximum; it is raised (and what has been
  // summed so far scaled down) only where an exponent would leave the range that the sums hold.
  auto add_tile = [&](const float (&e)[kSelEach], float m) {
    if (!(m - ref <= kSelRaise)) {                // also with a reference of -inf or +inf
      if (m == -INFINITY) return;
      if (m == INFINITY || ref == INFINITY) {     // from the first +inf on these are counted, and nothing else
        if (ref != INFINITY) { sum = 0.0; ref = INFINITY; }
#pragma unroll
        for (int j = 0; j < kSelEach; ++j) sum += e[j] == INFINITY ? 1.0 : 0.0;
        return;
      }
      sum = ref == -INFINITY ? 0.0 : sum * exp((double)ref - (double)m);
      ref = m;
    }
    if constexpr (kWide) {
      double two[2] = {sum, 0.0};
#pragma unroll
      for (int j = 0; j < kSelEach; j += 2) add_terms<2>(two, e + j, ref, (double)ref, s_powers);
      sum = two[0] + two[1];
    } else {
#pragma unroll
      for (int j = 0; j + 3 < kSelEach; j += 4) {
        const float2 a = terms_f32(e[j], e[j + 1], ref), b = terms_f32(e[j + 2], e[j + 3], ref);
        const float2 c = add2(a, b);
        sum += (double)(c.x + c.y);
      }
      if (kSelEach % 4 == 2) {
        const float2 a = terms_f32(e[kSelEach - 2], e[kSelEach - 1], ref);
        sum += (double)(a.x + a.y);
      }
    }
  };
  add_tile(cur, top);
  float best = top;                               // of the thread, so far
  for (int t0 = begin + kSelTile; t0 < end; t0 += kSelTile) {
#pragma unroll
    for (int j = 0; j < kSelEach; ++j) cur[j] = nxt[j];
    if (t0 + kSelTile < end) load_tile(t0 + kSelTile, nxt);
    clean(cur);
    const float m = tile_max(cur);
    if (m > least) {                              // -inf behind the segment's end is never more
      unsigned int bits = 0u;
#pragma unroll
      for (int j = 0; j < kSelEach; ++j) bits |= cur[j] > least ? 1u << j : 0u;
      if ((bits & (bits - 1u)) == 0u) {
        set_aside(t0 + (__ffs(bits) - 1) * kSelThreads + (int)threadIdx.x, m);
      } else {
        for (; bits != 0u; bits &= bits - 1u) {   // read again: a register cannot be picked at run time
          const int i = t0 + (__ffs(bits) - 1) * kSelThreads + (int)threadIdx.x;
          set_aside(i, x[i]);
        }
      }
    }
    add_tile(cur, m);
    best = fmaxf(best, m);
    const int seen = t0 + kSelTile - begin;       // a number of tiles, but for the last
    if (seen % (kSelCheck * kSelTile) != 0 && t0 + kSelTile < end) continue;
    if (__syncthreads_or(s_count > kSelBuffer)) {
      crowded(begin + max(kSelTile, (seen / kSelTile - 1) / kSelCheck * (kSelCheck * kSelTile)), t0 + kSelTile, false);
    }
    // The threshold that the first tile gave lets one logit in kSelTile / K pass, and whatever passes costs its whole warp.  Once
    // four times (or sixteen times) as many have been seen, K of the threads' best so far are at or above a higher one.
    if ((seen == 4 * kSelTile || seen == 16 * kSelTile) && end - t0 > 4 * kSelTile) {
      const unsigned int o = block_threshold_of<unsigned int>(p.k, p.k + p.k / 2, begin + (int)threadIdx.x < end, ordered_f32(best));
      if (o > ordered_f32(-INFINITY)) least = fmaxf(least, from_ordered_f32(o));
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
  if (n > 2 * p.k && n > 64) {                    // ranking them all would compare each with each
    const unsigned int o = block_threshold_of<unsigned int>(p.k, p.k + p.k / 2, begin + (int)threadIdx.x < end, ordered_f32(best));
    n = keep_from(s_buf, &s_count, n, (unsigned long long)o << 32);
  }
  if (n > kSelKept) n = thin_out(s_buf, &s_count, n, p.k, 0xffffffffu);
  float ref_all = -INFINITY;
#pragma unroll
  for (int i = 0; i < kSelThreads / 32; ++i) ref_all = fmaxf(ref_all, s_max[i]);
  const bool same = ref == ref_all;
  if (!same) sum = (ref == -INFINITY || ref_all == INFINITY) ? 0.0 : sum * exp((double)ref - (double)ref_all);
  // Where no thread raised its reference, the K best, which the sum is mostly made of, are summed in 64 bits after all: what their
  // fast exponentials were off by is added.
  const bool one_ref = !kWide && __syncthreads_and(same) && ref_all > -INFINITY && ref_all < INFINITY;
  if (!kWide && (int)threadIdx.x < p.k) s_late[threadIdx.x] = 0.0;
  for (int i = threadIdx.x; i < kSelKept; i += kSelThreads) s_rank[i] = 0;
  __syncthreads();
  rank_by_slices<kSelThreads>(n, s_rank, [&](int i, int j) { return s_buf[i] > s_buf[j]; });
  for (int i = threadIdx.x; i < n; i += kSelThreads) {
    const unsigned long long mine = s_buf[i];
    const int rank = s_rank[i];
    if (rank < p.k) {
      out[rank] = mine;
      const float v = from_ordered_f32((unsigned int)(mine >> 32));
      if (one_ref && v > -INFINITY) s_late[rank] = exp((double)v - (double)ref_all) - (double)terms_f32(v, v, ref_all).x;
    }
  }
  for (int i = n + (int)threadIdx.x; i < p.k; i += kSelThreads) out[i] = 0ull;
  __syncthreads();
  if (!kWide && (int)threadIdx.x < p.k) sum += s_late[threadIdx.x];        // by rank: the order of the additions is always the same
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) s_sum[warp] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    double total = 0.0;
    for (int i = 0; i < kSelThreads / 32; ++i) total += s_sum[i];
    p.seg_sum[2 * at_part] = (double)ref_all;
    p.seg_sum[2 * at_part + 1] = total;
  }
}

// A row's sum with every exponential in 64 bits; `parts` is for a value of each of the block's warps.  28 us for a row of 100,003.
// (Shared out over a cluster of eight blocks a group 9 us, but then every call takes 2 us more.)
__device__ __noinline__ double sum_again(const float* x, int vocab, double ref, const double* powers, double* parts) {
  constexpr int AHEAD = 16;
  double two[2] = {0.0, 0.0};
  for (int i0 = threadIdx.x; i0 < vocab; i0 += AHEAD * kJoinThreads) {
    float v[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) v[j] = i0 + j * kJoinThreads < vocab ? fmaxf(x[i0 + j * kJoinThreads], -INFINITY) : -INFINITY;
#pragma unroll
    for (int j = 0; j < AHEAD; j += 4) add_terms<4>(two, v + j, (float)ref, ref, powers);
  }
  double sum = two[0] + two[1];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) parts[threadIdx.x >> 5] = sum;
  __syncthreads();
  sum = 0.0;
#pragma unroll
  for (int i = 0; i < kJoinThreads / 32; ++i) sum += parts[i];
  return sum;
}

// One block per group: the sums of its rows, the keys of the elements set aside, the K best of them in order.  A segment's elements
// come best first, so where there are more segments than K only those whose first is among the K best firsts matter.
template <typename Score>
__global__ void __launch_bounds__(kJoinThreads, 2)
beam_join_kernel(SelectParams p) {
  pdl_trigger();
  extern __shared__ unsigned long long s_key[];                // [beams * segments * K] keys in their order
  __shared__ double s_ref[kSelMaxBeams], s_log[kSelMaxBeams];
  __shared__ unsigned long long s_best[kJoinThreads];
  __shared__ unsigned long long s_second[kJoinThreads];
  __shared__ unsigned long long s_top[kSelMaxK], s_top_second[kSelMaxK], s_doubt;
  __shared__ double s_powers[16], s_part[kJoinThreads / 32];
  __shared__ int s_count, s_rank[kJoinThreads];
  const int group = blockIdx.x;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const size_t row0 = (size_t)group * p.beams;
  const int per_row = p.segments * p.k;
  const int n = p.beams * per_row, lists = p.beams * p.segments;
  if (threadIdx.x == 0) s_doubt = 0ull;
  if (threadIdx.x < 16) s_powers[threadIdx.x] = kPowers[threadIdx.x];
  pdl_wait();
  const unsigned long long* elems = p.seg_key + row0 * per_row;
  const bool one_each = n <= kJoinThreads;                     // a thread has one element: it stays in a register
  const unsigned long long my_elem = one_each && (int)threadIdx.x < n ? __ldcg(elems + threadIdx.x) : 0ull;
  for (int b = warp; b < p.beams; b += kJoinThreads / 32) {
    const double2* seg = reinterpret_cast<const double2*>(p.seg_sum) + (row0 + b) * p.segments;
    const double2 first = lane < p.segments ? __ldcg(seg + lane) : make_double2(-INFINITY, 0.0);
    double ref = first.x;
    for (int s = lane + 32; s < p.segments; s += 32) ref = fmax(ref, __ldcg(seg + s).x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ref = fmax(ref, __shfl_xor_sync(0xffffffffu, ref, o));
    double sum = 0.0;
    for (int s = lane; s < p.segments; s += 32) {
      const double2 part = s == lane ? first : __ldcg(seg + s);
      if (part.x == ref) sum += part.y;
      else if (part.x != -INFINITY && ref != INFINITY) sum += part.y * exp(part.x - ref);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) { s_ref[b] = ref; s_log[b] = log(sum); }
  }
  __syncthreads();
  auto key_of = [&](int b, unsigned long long elem) {
    const double x = (double)from_ordered_f32((unsigned int)(elem >> 32));
    const double s = (double)((const Score*)p.scores)[row0 + b];
    const double ref = s_ref[b];
    double key = s + ((ref == INFINITY ? (x == INFINITY ? 0.0 : -INFINITY) : x - ref) - s_log[b]);
    if (!(key > -INFINITY)) key = -INFINITY;                   // dead beams, -inf logits, rows of -inf alone
    return ordered_f64(key);
  };
  auto any_key = [&](int i) {
    const unsigned long long elem = __ldcg(elems + i);
    return elem == 0ull ? 0ull : key_of(i / per_row, elem);
  };
  // Keys as floats, rounded down, are in the keys' order but for what they round away, and half the bits to look at.
  auto as_float = [&](unsigned long long key) { return key == 0ull ? 0u : ordered_f32(__double2float_rd(from_ordered_f64(key))); };
  auto from_float = [&](unsigned int t32) { return t32 <= ordered_f32(-INFINITY) ? 1ull : ordered_f64((double)from_ordered_f32(t32)); };
  // what comes after the key: the beam, the logit where there is one, the token (logits of different beams cannot be compared)
  constexpr unsigned int kTokens = 1u << kSelTokenBits;
  static_assert(kSelMaxBeams == 1 << (64 - 32 - kSelTokenBits), "a beam, a logit and a token in 64 bits");
  auto second_of = [&](int i, unsigned long long key, unsigned long long elem) {
    const unsigned int token = 0xffffffffu - (unsigned int)elem;
    const unsigned int logit = key == ordered_f64(-INFINITY) ? 0u : (unsigned int)(elem >> 32);
    return ((unsigned long long)(kSelMaxBeams - 1 - i / per_row) << (32 + kSelTokenBits)) |
           ((unsigned long long)logit << kSelTokenBits) | (kTokens - 1u - token);
  };
  // The K best in order, by the sums as they are.  Returns how many there are.
  unsigned long long my_key = 0ull;
  auto rank_all = [&]() -> int {
    s_rank[threadIdx.x] = 0;
    if (threadIdx.x == 0) s_count = 0;
    __syncthreads();
    my_key = my_elem == 0ull ? 0ull : key_of((int)threadIdx.x / per_row, my_elem);
    int m = 0;
    if (!one_each) {
      unsigned long long t = 1ull;                                   // everything there is
      if (lists > p.k) {
        for (int i = threadIdx.x; i < lists; i += kJoinThreads) s_key[i * p.k] = any_key(i * p.k);
        __syncthreads();
        if (lists <= kJoinThreads) {
          const unsigned long long key = (int)threadIdx.x < lists ? s_key[threadIdx.x * p.k] : 0ull;
          t = from_float(block_threshold_of<unsigned int>(p.k, p.k, key != 0ull, as_float(key)));
        } else {
          t = from_float(block_threshold<kJoinThreads, unsigned int>(p.k, p.k + p.k / 4, [&](unsigned int trial) {
            int c = 0;
            for (int i = threadIdx.x; i < lists; i += kJoinThreads) c += as_float(s_key[i * p.k]) >= trial ? 1 : 0;
            return c;
          }));
        }
        __syncthreads();
        for (int i = threadIdx.x; i < n; i += kJoinThreads) {
          const int list = i / p.k, first = list * p.k;
          if (i != first) s_key[i] = s_key[first] >= t ? any_key(i) : 0ull;
        }
      } else {
        for (int i = threadIdx.x; i < n; i += kJoinThreads) s_key[i] = any_key(i);
      }
      __syncthreads();
      auto gather = [&](unsigned long long t, unsigned long long t2) {
        __syncthreads();
        if (threadIdx.x == 0) s_count = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < n; i += kJoinThreads) {
          const unsigned long long key = s_key[i];
          if (key < t) continue;
          const unsigned long long second = second_of(i, s_key[i], __ldcg(elems + i));
          if (key > t || second >= t2) {
            const int at = atomicAdd(&s_count, 1);
            if (at < kJoinThreads) { s_best[at] = key; s_second[at] = second; }
          }
        }
        __syncthreads();
        return s_count;
      };
      m = gather(t, 0ull);
      if (m > kJoinThreads) {
        // more than can be ranked: a threshold over all of them
        t = max(t, from_float(block_threshold<kJoinThreads, unsigned int>(p.k, kJoinThreads, [&](unsigned int trial) {
          int c = 0;
          for (int i = threadIdx.x; i < n; i += kJoinThreads) c += as_float(s_key[i]) >= trial ? 1 : 0;
          return c;
        })));
        m = gather(t, 0ull);
      }
      if (m > kJoinThreads) {
        // Where more than can be ranked share the K-th key (beams that all are dead, rows of equal logits), the same search goes on
        // over all bits of the keys, and then over what comes after the key.
        auto at_least = [&](unsigned long long trial) {
          int c = 0;
          for (int i = threadIdx.x; i < n; i += kJoinThreads) c += s_key[i] >= trial ? 1 : 0;
          return c;
        };
        t = max(1ull, block_threshold<kJoinThreads, unsigned long long>(p.k, kJoinThreads, at_least));
        unsigned long long t2 = 0ull;
        __shared__ int s_above;
        if (threadIdx.x == 0) s_above = 0;
        __syncthreads();
        const int above_here = at_least(t + 1ull);
        if (above_here > 0) atomicAdd(&s_above, above_here);
        __syncthreads();
        const int above = s_above;
        if (above < p.k) {
          t2 = block_threshold<kJoinThreads, unsigned long long>(p.k - above, kJoinThreads - above, [&](unsigned long long trial) {
            int c = 0;
            for (int i = threadIdx.x; i < n; i += kJoinThreads) c += (s_key[i] == t && second_of(i, s_key[i], __ldcg(elems + i)) >= trial) ? 1 : 0;
            return c;
          });
        }
        m = gather(t, t2);
      }
    }
    if (one_each || (m > 64 && m > 2 * p.k)) {
      // ranking compares each with each: a threshold over them first
      const bool there = (int)threadIdx.x < m;
      const unsigned long long key = one_each ? my_key : there ? s_best[threadIdx.x] : 0ull;
      const unsigned long long second = one_each ? second_of(threadIdx.x, my_key, my_elem) : there ? s_second[threadIdx.x] : 0ull;
      const bool any = key != 0ull;
      const unsigned long long least = from_float(block_threshold_of<unsigned int>(p.k, p.k + p.k / 4, any, as_float(key)));
      __syncthreads();
      if (threadIdx.x == 0) s_count = 0;
      __syncthreads();
      if (any && key >= least) {
        const int at = atomicAdd(&s_count, 1);
        s_best[at] = key;
        s_second[at] = second;
      }
      __syncthreads();
      m = s_count;
    }
    rank_by_slices<kJoinThreads>(m, s_rank, [&](int i, int j) {
      const unsigned long long a = s_best[i], b = s_best[j];
      return a > b || (a == b && s_second[i] > s_second[j]);
    });
    if ((int)threadIdx.x < m && s_rank[threadIdx.x] < p.k) {
      s_top[s_rank[threadIdx.x]] = s_best[threadIdx.x];
      s_top_second[s_rank[threadIdx.x]] = s_second[threadIdx.x];
    }
    __syncthreads();
    return min(m, p.k);
  };

  // ---- beams whose order the float exponentials may have wrong: a bit each -------------------------------------------
  auto in_doubt = [&](int last) -> unsigned long long {
    const double bound = order_bound(p.vocab);
    auto top = [&](int i) { return from_ordered_f64(s_top[i]); };
    const unsigned long long all = ~0ull >> (kSelMaxBeams - p.beams);
    auto beam_of = [&](unsigned long long second) { return kSelMaxBeams - 1 - (int)(second >> (32 + kSelTokenBits)); };
    unsigned long long rows = 0ull;                                   // a bit a beam
    for (int i = threadIdx.x; i < last; i += kJoinThreads) {         // of those that are wanted, two that are neighbours
      const int a = beam_of(s_top_second[i]), b = beam_of(s_top_second[i + 1]);
      if (a != b && top(i + 1) > -INFINITY && top(i) - top(i + 1) < bound) rows |= 1ull << a | 1ull << b;
    }
    if (top(last) > -INFINITY) {                                      // and those behind the last that is
      const unsigned long long edge = ordered_f64(top(last) - bound);
      // returns whether the element is one of them
      auto look = [&](int i, unsigned long long key, unsigned long long elem) {
        if (key < edge) return false;
        const unsigned long long second = second_of(i, key, elem);
        if (key > s_top[last] || (key == s_top[last] && second >= s_top_second[last])) return true;
        const int b = beam_of(second);
        for (int j = last; j >= 0 && rows != all && top(j) - from_ordered_f64(key) < bound; --j) {
          const int a = beam_of(s_top_second[j]);
          if (a != b) rows |= 1ull << a | 1ull << b;
        }
        return false;
      };
      if (one_each) {
        look(threadIdx.x, my_key, my_elem);
      } else {
        // of every list, best first, the first that is none of them: whoever is close to a later one is close to it
        for (int l = threadIdx.x; l < lists; l += kJoinThreads) {
          const unsigned long long* list = s_key + l * p.k;
          if (list[0] < edge) continue;
          int lo = 0;
          for (int hi = p.k; lo < hi;) {
            const int mid = (lo + hi) >> 1;
            if (list[mid] > s_top[last]) lo = mid + 1; else hi = mid;
          }
          for (; lo < p.k; ++lo) {
            const int i = l * p.k + lo;
            if (!look(i, list[lo] != 0ull ? list[lo] : any_key(i), __ldcg(elems + i))) break;
          }
        }
      }
    }
    if (rows != 0ull) atomicOr(&s_doubt, rows);
    __syncthreads();
    return s_doubt;
  };

  // (One copy of this code for both rankings: two take every call a microsecond more.)
#pragma unroll 1
  for (int pass = 0;; ++pass) {
    const int found = rank_all();
    if (pass > 0 || p.beams == 1 || sizeof(Score) == 8) break;
    const unsigned long long rows = in_doubt(found - 1);
    if (rows == 0ull) break;
    for (int b = 0; b < p.beams; ++b) {
      const double ref = s_ref[b];
      if (!(rows >> b & 1ull) || ref == INFINITY) continue;           // (the sum of a row of +inf is exact)
      const double sum = sum_again(p.logits + (long long)(row0 + b) * p.ld, p.vocab, ref, s_powers, s_part);
      if (threadIdx.x == 0) s_log[b] = log(sum);
    }
    __syncthreads();
  }
  for (int i = threadIdx.x; i < p.k; i += kJoinThreads) {
    const size_t at = (size_t)group * p.k + i;
    const unsigned long long second = s_top_second[i];
    ((Score*)p.out_scores)[at] = (Score)from_ordered_f64(s_top[i]);
    p.out_parents[at] = kSelMaxBeams - 1 - (int)(second >> (32 + kSelTokenBits));
    p.out_tokens[at] = (int)(kTokens - 1u - ((unsigned int)second & (kTokens - 1u)));
  }
}

// ---- the next step's beams ---------------------------------------------------------------------------------------
//
// Of a group's candidates, in order, the first W whose token is no stop token go on.  A beam whose parent has not been
// claimed by a better one stays in its parent's seat; the others take the seats that are left, in order.  So a seat that
// goes on is never written, and what has to move is one record for every beam that ends.  A seat that is left without a
// candidate (a vocabulary of stop tokens) keeps its parent with a score of -inf.
struct AdvanceParams {
  const void* cand_scores;      // [groups, K], best first, of the type that the kernel is made for
  const int* cand_parents;
  const int* cand_tokens;
  const int* stop_tokens;       // [n_stop]
  const int* slots;             // [groups, beams]
  void* scores;                 // [groups, beams], rewritten
  int* parents;                 // [groups, beams]: the seat that each seat goes on from
  int* tokens;                  // [groups, beams]
  int* records;                 // [max_slots, words] or null: word `token_word` receives the token
  unsigned char* history;       // [max_slots, history_ld] or null
  const int* positions;         // [groups * beams]: the position that this step wrote
  const int* prefix_len;        // [groups]: positions in front of the history
  int* err;
  int k, beams, n_stop, max_slots, words, token_word, history_ld, from_one;
};

template <typename Score>
__global__ void __launch_bounds__(64) beam_advance_kernel(AdvanceParams p) {
  pdl_trigger();
  const Score* cand_scores = (const Score*)p.cand_scores;
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
      if (!(cand_scores[c0 + i] > -INFINITY)) break;          // what comes now cannot go on
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
  ((Score*)p.scores)[b0 + seat] = c >= 0 ? cand_scores[c0 + c] : (Score)-INFINITY;
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
// Before its first load a block has to know which seats change, which costs it as long as a column's loads: where there are more
// columns than threads at a time on the device, a thread takes up to four, one after the other.  12 groups of 8 beams with 8
// layers of 1 MB states, three in ten of which change, 313 MB to read and write: 53 us (5.9 TB/s).  (With
// twice the registers 60, 65 with two columns, 59 with eight, which cost a call of 60 MB 9.8 us instead of 9.0.)  One to
// four seats that change have code of their own (66 us for all of them with a question for each of eight), and a kernel is held
// to the registers that leave room for six blocks on an SM up to 8 seats, four up to 32 (8 seats: 60 us with four; 12 groups of 16:
// 46 us with four, 62 with the two that columns of 16 bytes of all seats would leave; there more than 8 seats that change move in
// columns of 8 bytes, more than 16 in columns of 4).  Where every seat changes that costs something: 144 us for 805 MB of 8 seats
// instead of 128, 262 instead of 250 for 1.6 GB of 16, 331 instead of 255 of 32.
constexpr int kMoveThreads = 256;
constexpr int kMoveColumns = 4;
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
  int per_thread;               // columns of a thread
};

// s_src, s_dst: of the n seats that change, in bytes from slot 0's record.  kExact: n is kSeats, so that nothing is asked seat by seat.
template <typename V, int kSeats, bool kExact>
__device__ __forceinline__ void move_columns(const MoveTensor& t, long long first, int count, const long long* s_src, const long long* s_dst,
                                             int n, int max_slots) {
  const long long columns = t.bytes / (long long)sizeof(V), all = columns * t.keys;
#pragma unroll 1
  for (int c = 0; c < count; ++c, first += kMoveThreads) {
    const long long at = first + threadIdx.x;
    if (at >= all) return;
    const long long key = all <= 0x7fffffffLL ? (long long)((unsigned)at / (unsigned)columns) : at / columns;
    unsigned char* base = t.base + (key * (max_slots - 1) * columns + at) * (long long)sizeof(V);          // column at % columns of the key's records
    V v[kSeats];
#pragma unroll
    for (int i = 0; i < kSeats; ++i) {
      if (kExact || i < n) v[i] = *reinterpret_cast<const V*>(base + s_src[i]);
    }
#pragma unroll
    for (int i = 0; i < kSeats; ++i) {
      if (kExact || i < n) *reinterpret_cast<V*>(base + s_dst[i]) = v[i];
    }
  }
}

template <int kSeats>
__global__ void __launch_bounds__(kMoveThreads, kSeats <= 8 ? 6 : kSeats <= 32 ? 4 : 2) reorder_slots_kernel(const __grid_constant__ MoveParams p) {
  pdl_trigger();
  __shared__ long long s_src[kMoveMaxSeats], s_dst[kMoveMaxSeats];
  __shared__ int s_n;
  int k = 0;
  while (k + 1 < p.n_tensors && (long long)blockIdx.x >= p.t[k + 1].first_block) ++k;
  const MoveTensor& t = p.t[k];
  pdl_wait();
  const int g = blockIdx.y;
  if (threadIdx.x < 32) {
    // the seats that change, in order
    const int lane = threadIdx.x;
    const int* slots = p.slots + (size_t)g * p.seats;
    const int* parents = p.parents + (size_t)g * p.seats;
    const int slot0 = lane < p.seats ? slots[lane] : -1, slot1 = lane + 32 < p.seats ? slots[lane + 32] : -1;
    const int parent0 = lane < p.seats ? parents[lane] : 0, parent1 = lane + 32 < p.seats ? parents[lane + 32] : 0;
    int n = 0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int i = lane + 32 * h;
      const int parent = h == 0 ? parent0 : parent1, dst = h == 0 ? slot0 : slot1;
      const int low = __shfl_sync(0xffffffffu, slot0, parent & 31), high = __shfl_sync(0xffffffffu, slot1, parent & 31);
      const int src = parent < 32 ? low : high;
      bool moves = false;
      if (i < p.seats) {
        if (parent < 0 || parent >= p.seats) {
          set_error(p.err, kErrRequest, g, parent, p.seats);
        } else if (parent != i) {
          if (src < 0 || src >= p.max_slots || dst < 0 || dst >= p.max_slots) {
            set_error(p.err, kErrRequest, g, src < 0 || src >= p.max_slots ? src : dst, p.max_slots);
          } else {
            moves = src != dst;
          }
        }
      }
      const unsigned mask = __ballot_sync(0xffffffffu, moves);
      if (moves) {
        const int at = n + __popc(mask & ((1u << lane) - 1u));
        s_src[at] = src * t.bytes;
        s_dst[at] = dst * t.bytes;
      }
      n += __popc(mask);
    }
    if (lane == 0) s_n = n;
  }
  __syncthreads();
  const int n = s_n;
  if (n == 0) return;
  const long long at = ((long long)blockIdx.x - t.first_block) * kMoveThreads * p.per_thread;
  // columns of the tensor's width, or of a part of it where so many seats change that a thread's registers would not hold them
  auto move = [&](auto seats, auto exact, auto type) {
    const int parts = t.vec / (int)sizeof(type);
    move_columns<decltype(type), decltype(seats)::value, decltype(exact)::value>(t, at * parts, p.per_thread * parts, s_src, s_dst, n, p.max_slots);
  };
  using std::integral_constant;
  using Any = integral_constant<bool, false>;
  using Exact = integral_constant<bool, true>;
  constexpr int kEight = kSeats < 8 ? kSeats : 8, kSixteen = kSeats < 16 ? kSeats : 16;
  if (t.vec == 16 && n == 1) move(integral_constant<int, 1>(), Exact(), uint4());
  else if (t.vec == 16 && n == 2) move(integral_constant<int, 2>(), Exact(), uint4());
  else if (t.vec == 16 && n == 3) move(integral_constant<int, 3>(), Exact(), uint4());
  else if (t.vec == 16 && n == 4) move(integral_constant<int, 4>(), Exact(), uint4());
  else if (t.vec == 16 && n <= kEight) move(integral_constant<int, kEight>(), Any(), uint4());
  else if (t.vec >= 8 && n <= kSixteen) move(integral_constant<int, kSixteen>(), Any(), uint2());
  else if (t.vec >= 4) move(integral_constant<int, kSeats>(), Any(), (unsigned int)0);
  else if (t.vec == 2) move(integral_constant<int, kSeats>(), Any(), (unsigned short)0);
  else move(integral_constant<int, kSeats>(), Any(), (unsigned char)0);
}

}  // namespace tk

// scratch: rows * segments * (16 + 8 k) bytes, on 8 bytes.
// wide: scores and out_scores are doubles.
TK_API int tk_beam_select(const float* logits, long long ld, const void* scores, void* scratch, void* out_scores,
                          int* out_parents, int* out_tokens, int groups, int beams, int vocab, int k, int segments, int wide,
                          cudaStream_t stream) {
  if (groups <= 0) return 0;
  if (beams < 1 || beams > tk::kSelMaxBeams || k < 1 || k > tk::kSelMaxK || vocab < 1 || segments < 1 || ld < vocab ||
      (long long)beams * segments * k > tk::kSelMaxEntries || vocab > 1 << tk::kSelTokenBits ||
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
  const int join_smem = beams * segments * k * 8;
  static bool configured[64] = {false};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return (int)e;
  if (dev < 0 || dev >= 64) return (int)cudaErrorInvalidValue;
  if (!configured[dev]) {
    e = cudaFuncSetAttribute(tk::beam_join_kernel<float>, cudaFuncAttributeMaxDynamicSharedMemorySize, tk::kSelMaxEntries * 8);
    if (e != cudaSuccess) return (int)e;
    e = cudaFuncSetAttribute(tk::beam_join_kernel<double>, cudaFuncAttributeMaxDynamicSharedMemorySize, tk::kSelMaxEntries * 8);
    if (e != cudaSuccess) return (int)e;
    configured[dev] = true;
  }
  const bool few = (long long)segments * groups * beams <= 3LL * tk::device_sm_count();
  auto* first = wide ? (few ? tk::beam_segments_kernel<3, double> : tk::beam_segments_kernel<4, double>)
                     : (few ? tk::beam_segments_kernel<3, float> : tk::beam_segments_kernel<4, float>);
  e = tk::launch(first, dim3(segments, groups * beams), dim3(tk::kSelThreads), 0, stream, p);
  if (e != cudaSuccess) return (int)e;
  return (int)tk::launch(wide ? tk::beam_join_kernel<double> : tk::beam_join_kernel<float>, dim3(groups), dim3(tk::kJoinThreads), join_smem,
                         stream, p);
}

// wide: the scores are doubles.
TK_API int tk_beam_advance(const void* cand_scores, const int* cand_parents, const int* cand_tokens, const int* stop_tokens,
                           const int* slots, void* scores, int* parents, int* tokens, int* records,
                           unsigned char* history, const int* positions, const int* prefix_len, int* err, int groups, int beams, int k, int n_stop,
                           int max_slots, int words, int token_word, int history_ld, int from_one, int wide, cudaStream_t stream) {
  if (groups <= 0) return 0;
  if (beams < 1 || beams > tk::kSelMaxBeams || k < 1 || n_stop < 0) return (int)cudaErrorInvalidValue;
  tk::AdvanceParams p{cand_scores, cand_parents, cand_tokens, stop_tokens, slots, scores, parents, tokens, records, history,
                      positions, prefix_len, err, k, beams, n_stop, max_slots, words, token_word, history_ld, from_one};
  return (int)tk::launch(wide ? tk::beam_advance_kernel<double> : tk::beam_advance_kernel<float>, dim3(groups), dim3(64), 0, stream, p);
}

// tensors: address, bytes of a record and keys of each; a record's bytes and its tensor's address decide how wide its columns are.
TK_API int tk_reorder_slots(const long long* tensors, int n_tensors, const int* slots, const int* parents, int* err, int groups,
                            int seats, int max_slots, cudaStream_t stream) {
  if (groups <= 0 || n_tensors <= 0) return 0;
  if (n_tensors > tk::kMoveMaxTensors || seats < 1 || seats > tk::kMoveMaxSeats || groups > 65535 || max_slots < 1) {
    return (int)cudaErrorInvalidValue;
  }
  tk::MoveParams p;
  p.slots = slots; p.parents = parents; p.err = err; p.n_tensors = 0; p.seats = seats; p.max_slots = max_slots;
  long long columns = 0;
  for (int i = 0; i < n_tensors; ++i) {
    const long long base = tensors[3 * i], bytes = tensors[3 * i + 1], keys = tensors[3 * i + 2];
    if (bytes < 0 || keys < 0 || keys > 0x7fffffffLL) return (int)cudaErrorInvalidValue;
    if (bytes == 0 || keys == 0) continue;
    tk::MoveTensor& t = p.t[p.n_tensors++];
    t.base = (unsigned char*)base;
    t.bytes = bytes;
    t.keys = (int)keys;
    t.vec = 16;
    while (((unsigned long long)base | (unsigned long long)bytes) % (unsigned long long)t.vec) t.vec /= 2;
    columns += t.bytes / t.vec * t.keys;
  }
  p.per_thread = 1;
  while (p.per_thread < tk::kMoveColumns && columns * groups > 8LL * tk::device_sm_count() * tk::kMoveThreads * p.per_thread) p.per_thread *= 2;
  long long blocks = 0;
  for (int i = 0; i < p.n_tensors; ++i) {
    tk::MoveTensor& t = p.t[i];
    const long long per_block = (long long)tk::kMoveThreads * p.per_thread;
    t.first_block = blocks;
    blocks += (t.bytes / t.vec * t.keys + per_block - 1) / per_block;
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
