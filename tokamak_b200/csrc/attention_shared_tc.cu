// Attention over shared prefixes in bfloat16 with heads of 64 or 128 elements (attention_shared.cuh has the definition).
//
// Plan (a block of its own): what every group shares.  Beside the prefix these are, with a history, the positions behind it that
// all members inherited from the same writers: the beams of a search differ in their last few tokens only, so nearly all of
// what they generated is read once for the group too.  The key tiles (64 keys) of all (group, tile of rows, key/value head)
// triples form one sequence.
//
// Shared positions: tcgen05, one block per SM; block b of G takes the tiles [T b / G, T (b + 1) / G) of the sequence, so the
// SMs end together whatever the groups' sizes are: the end of one triple, whole ones, the beginning of another.  The
// query heads of a group's members over one key/value head are the rows of Q, up to two tiles of 128.  Roles of a block:
//   warps 0, 10  load keys (and the query tiles) and values: the prefix's with TMA, page by page; positions behind the prefix, whose
//                neighbours lie in different members' pages, row by row with cp.async.  Block-table entries are fetched 32 at a
//                time and a batch ahead, the chain from a position to its place (writer, slot, page) a tile ahead a link: looked up
//                as they are needed they alone took 1.5 us a tile;
//   warps 1, 11  a thread each issues tcgen05.mma for one group of softmax warps: S = Q K^T (M 128, N 64) into one of its two score
//                buffers in tensor memory, and, a tile behind, O += P V with P from tensor memory and V as an MN-major operand
//                straight from its page layout.  (A product costs the thread that issues it 77 clocks whatever its N up to 128:
//                one thread for both groups needed 1,820 clocks a tile.)
//   warps 2..5, 6..9   softmax, two groups with an output accumulator each, thread i owns row i of its tile: scores with
//                tcgen05.ld, mask, running reference and sum in float32, probabilities over the scores.  The output is rescaled
//                in tensor memory only when a row's maximum grew by more than 2^8 since its reference was set.  With more than 128 rows the two groups have a tile of rows each and every key tile; with fewer they
//                take turns at the key tiles, so that the softmax of two of them is under way at a time.
// A probability is two bfloat16 here, its rounded value and what the rounding left, and P V a product of either, in both kernels:
// the sum that divides the output has the probabilities as floats, so that one rounding of each would stay in the result (2.1e-3 of it
// where the result's own is 1.66e-3).  It costs 4 to 10 %: 65 us instead of 61 for 16 groups of 4, 126 instead of 114 for 4 of 16.
// Bound: the keys' bytes.  A tile of 64 keys of 128 elements is 32 KB, 0.74 us of an SM's share of the memory bandwidth, against
// 0.5 us of tensor time; a softmax group needs more than a microsecond for it, the two together half of that.  A call of 4 groups of
// 16 rows, 32 query heads over 8 of 128, 32,768 shared and 1,024 further positions (456 MB) takes 126 us, one of 16 groups of 4 over up
// to 4,093 + 129 (216 MB) 65: the plan is 3 to 6 us of that, the first tile's way 4, a change of group 3, the rows' own positions and the
// parts 10 behind it all.
//
// Rows of V that no row may see (behind the prefix in its last page, in front of a window) are zeroed in shared memory
// before they are used: their probabilities are zero, and what lies there may be anything.
//
// Other positions: mma.sync, a block per (range of keys, key/value head, row), the query heads over the key/value head as
// the rows of a 16-row tile.  Four warps walk 16-key tiles with cp.async, each key's address looked up once, ahead of the
// loop, for the block.  Where the shared positions get all SMs and a row is one range, the block adds the shared parts up itself;
// otherwise the two kinds of positions run side by side and a third kernel does.
#include "attention_shared.cuh"
#include "tcgen05_utils.cuh"

namespace tk {

constexpr int kSpBM = 128;            // rows of a query tile
constexpr int kSpBN = 64;             // keys of a tile
constexpr int kSpStages = 4;
constexpr int kSpThreads = 384;       // loads of keys, products, eight warps of softmax, loads of values, products
constexpr int kSpValueWarp = 10, kSpSecondIssuer = 11;
constexpr float kSpRescale = 8.0f;    // log2 units
constexpr int kSpMinTiles = 3;        // tiles of a block, where there are so many
constexpr int kSpSegments = 32;       // pieces of triples that a block lists at a time

// ---- plan ------------------------------------------------------------------------------------------------------------------
constexpr int kPlanHead = 8, kPlanRecord = 8, kPlanThreads = 1024, kPlanGroups = 64, kPlanMembers = 64;
// head: 0 tiles in all, 1 blocks that take part.  A group's record: 0 first row, 1 members, 2 lowest visible position, 3 last visible
// position of the prefix (< 2: none), 4 key tiles of the prefix, 5 first position of the common ones behind it, 6 one past their
// last (where each member's own begin), 7 tiles of all groups before this one
struct SharedPlan {
  int* ints;
  int blocks;              // of the shared positions' kernel
  int members_per_tile;
  bool apart;              // rows' own parts go to own_o and the parts are added up by a kernel of their own
  float* slot_o;           // [blocks][2 pieces][2 softmax groups][128 rows][D]
  float* slot_ml;          // [blocks][2][2][128][2]
  float* whole_o;          // [rows][n_q_heads][2][D]: triples that one block holds whole
  float* whole_ml;         // [rows][n_q_heads][2][2]
  float* own_o;            // [rows][n_q_heads][n_own][D]
  float* own_ml;           // [rows][n_q_heads][n_own][2]
};
struct GroupPlan { int row0, members, lo, hi, prefix_tiles, common0, common1, first; };

__device__ __forceinline__ GroupPlan group_plan(const SharedPlan& s, int g) {
  const int4* r = reinterpret_cast<const int4*>(s.ints + kPlanHead + g * kPlanRecord);
  const int4 a = __ldcg(r), b = __ldcg(r + 1);
  return {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
}
__device__ __forceinline__ int plan_tiles(const GroupPlan& g) {          // key tiles of one of its triples
  return g.prefix_tiles + max(0, g.common1 - g.common0 + kSpBN - 1) / kSpBN;
}
__device__ __forceinline__ int plan_row_tiles(const GroupPlan& g, int members_per_tile) {
  return (g.members + 2 * members_per_tile - 1) / (2 * members_per_tile);
}

__global__ void __launch_bounds__(kPlanThreads) shared_plan_kernel(const __grid_constant__ SharedParams p, const __grid_constant__ SharedPlan s) {
  pdl_trigger();
  // what is looked up once stays here: the kernels behind this one wait for it, and a load after another is most of its time
  __shared__ int s_common[kPlanGroups], s_first[kPlanGroups], s_lo[kPlanGroups], s_hi[kPlanGroups], s_prefix[kPlanGroups];
  __shared__ int2 s_rows[kPlanGroups];
  __shared__ int s_slot[kPlanGroups][kPlanMembers];          // of the first members
  constexpr int WARPS = kPlanThreads / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int carry = 0;                                             // warp 0: tiles of the groups so far
  pdl_wait();
  for (int g0 = 0; g0 < p.n_groups; g0 += kPlanGroups) {
    const int n_here = min(kPlanGroups, p.n_groups - g0);
    // what the members see
    for (int k = warp; k < n_here; k += WARPS) {
      const int g = g0 + k;
      const int2 rows = group_rows(p, g);
      const int prefix = max(0, p.prefix_len[g]), prefix_slot = p.prefix_slot[g];
      int lo = 0x7fffffff, last = -1, first = 0x7fffffff, bad = 0;
      for (int i = rows.x + lane; i < rows.y; i += 32) {
        const int slot = p.req_slot[i];
        if (slot < 0 || slot >= p.max_slots) bad = 1;
        if (i - rows.x < kPlanMembers) s_slot[k][i - rows.x] = slot;
        const RowSpan sp = row_span(p, i);
        if (sp.pos < 0) { bad = 1; continue; }
        lo = min(lo, sp.lo); last = max(last, sp.pos); first = min(first, sp.pos);
      }
      lo = __reduce_min_sync(0xffffffffu, lo);
      last = __reduce_max_sync(0xffffffffu, last);
      first = __reduce_min_sync(0xffffffffu, first);
      bad = __reduce_or_sync(0xffffffffu, (unsigned)bad);
      if (lane == 0) {
        int hi = min(prefix - 1, last);
        if (hi >= lo && checked_slot(p, prefix_slot, rows.x) < 0) hi = -1;
        s_lo[k] = lo; s_hi[k] = hi; s_prefix[k] = prefix; s_rows[k] = rows;
        // positions behind the prefix and in front of every member's own, for which there are writers
        s_first[k] = p.history != nullptr && rows.y > rows.x && !bad ? max(0, min(first - prefix, p.history_ld)) : 0;
        s_common[k] = s_first[k];
      }
    }
    __syncthreads();
    // of those the first that not all members inherited from the same writer (or from one that is none: each member reports it)
    if (p.history != nullptr) {
      const bool wide = p.history_ld % 16 == 0 && ((uintptr_t)p.history & 15) == 0;
      for (int pair = warp; pair < n_here * p.max_members; pair += WARPS) {
        const int k = pair / p.max_members, i = pair % p.max_members;
        const int2 rows = s_rows[k];
        const int n = rows.y - rows.x, most = s_first[k];
        if (i >= n || most == 0) continue;
        const unsigned char* h0 = p.history + (size_t)s_slot[k][0] * p.history_ld;
        const unsigned char* h = p.history + (size_t)(i < kPlanMembers ? s_slot[k][i] : p.req_slot[rows.x + i]) * p.history_ld;
        int common = most;
        if (wide) {
#pragma unroll 2
          for (int c = lane; 16 * c < most; c += 32) {
            const uint4 x = *reinterpret_cast<const uint4*>(h0 + 16 * c), y = *reinterpret_cast<const uint4*>(h + 16 * c);
            // a byte of the first member's row is looked at for its value, the others' for being the same
            const unsigned int limit = (unsigned int)min(n, 255) * 0x01010101u;
            const unsigned int w[4] = {x.x, x.y, x.z, x.w}, v[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
            for (int q = 3; q >= 0; --q) {
              const unsigned int off = i > 0 ? w[q] ^ v[q] : n <= 255 ? __vcmpgeu4(w[q], limit) : 0u;
              if (off != 0u) common = min(common, 16 * c + 4 * q + ((__ffs((int)off) - 1) >> 3));
            }
          }
        } else {
          for (int c = lane; c < most; c += 32) {
            if (h[c] != h0[c] || h0[c] >= n) common = min(common, c);
          }
        }
        common = __reduce_min_sync(0xffffffffu, common);
        if (lane == 0) atomicMin(&s_common[k], common);
      }
    }
    __syncthreads();
    if (warp == 0) {
      for (int k0 = 0; k0 < n_here; k0 += 32) {
        const int k = k0 + lane, g = g0 + k;
        int v = 0;
        GroupPlan gp = {};
        if (k < n_here) {
          const int2 rows = s_rows[k];
          const int prefix = s_prefix[k], lo = s_lo[k], hi = s_hi[k], end = prefix + s_common[k];
          gp = {rows.x, rows.y - rows.x, lo, hi, hi >= lo ? hi / kSpBN - lo / kSpBN + 1 : 0, max(prefix, min(lo, end)), end, 0};
          v = plan_tiles(gp) * plan_row_tiles(gp, s.members_per_tile) * p.n_kv_heads;
        }
        int sum = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int x = __shfl_up_sync(0xffffffffu, sum, o);
          if (lane >= o) sum += x;
        }
        if (k < n_here) {
          int4* r = reinterpret_cast<int4*>(s.ints + kPlanHead + g * kPlanRecord);
          r[0] = make_int4(gp.row0, gp.members, gp.lo, gp.hi);
          r[1] = make_int4(gp.prefix_tiles, gp.common0, gp.common1, carry + sum - v);
        }
        carry += __shfl_sync(0xffffffffu, sum, 31);
      }
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    s.ints[0] = carry;
    s.ints[1] = max(1, min(s.blocks, carry / kSpMinTiles));
  }
}

// Where block c of G begins in the sequence of T tiles, and the block that holds tile t: the largest c that begins at or before it.
__device__ __forceinline__ int block_start(int T, int G, int c) {
  return T < (1 << 24) ? (int)((unsigned)T * (unsigned)c / (unsigned)G) : (int)((long long)T * c / G);
}
__device__ __forceinline__ int tile_owner(int T, int G, int t) {
  if (T < (1 << 24)) return (int)(((unsigned)(t + 1) * (unsigned)G + (unsigned)T - 1u) / (unsigned)T) - 1;
  return (int)((((long long)t + 1) * G + T - 1) / T) - 1;
}

// ---- shared positions ----------------------------------------------------------------------------------------------------
struct Segment {          // what a block does of one triple
  int row0, members;      // rows of its query tiles
  int hkv, slot;          // key/value head, block-table row of the prefix
  int lo, hi, common0, common1, prefix_tiles, lo_tile;
  int tile0, n_tiles;     // its key tiles
  int piece;              // 0, 1: the block's first or last, a part of a triple; 2: the whole of one
  int writers;            // a member's slot whose history names the common positions' writers
  int group_row0, prefix;
};

__device__ __forceinline__ void st_global_32(float* dst, const uint32_t* r) {          // 32 bytes, on 32
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};\n"
               ::"l"(dst), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
}

__device__ __forceinline__ float sp_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float sp_rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}

// What is left of a and b behind their roundings in `hi`, as bfloat16.
__device__ __forceinline__ uint32_t rest_bf16(float a, float b, uint32_t hi) {
  return pack_bf16(a - __uint_as_float(hi << 16), b - __uint_as_float(hi & 0xffff0000u));
}

template <int D>
__global__ void __launch_bounds__(kSpThreads, 1)
shared_prefix_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                     const __grid_constant__ CUtensorMap map_v, const __grid_constant__ SharedParams p, const __grid_constant__ SharedPlan s) {
  constexpr int SUB = D / 64;
  constexpr uint32_t Q_BYTES = kSpBM * D * 2;
  constexpr uint32_t KSUB_BYTES = kSpBN * 64 * 2;
  constexpr uint32_t KV_BYTES = kSpBN * D * 2;
  constexpr uint32_t V_RING = kSpStages * KV_BYTES;
  constexpr uint32_t DATA_BYTES = 2 * Q_BYTES + 2 * kSpStages * KV_BYTES;
  constexpr uint32_t TMEM_COLS = 512;                      // group t: scores at t * 128 + {0, 64}, output at 256 + t * 128

  extern __shared__ __align__(1024) unsigned char smem_raw[];
  const uint32_t raw = gt_smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  unsigned char* smem = smem_raw + (base - raw);
  const uint32_t q_smem = base, kv_smem = base + 2 * Q_BYTES;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + DATA_BYTES);
  uint64_t* k_full = bars;
  uint64_t* k_empty = k_full + kSpStages;
  uint64_t* v_full = k_empty + kSpStages;
  uint64_t* v_empty = v_full + kSpStages;
  uint64_t* group_bars = v_empty + kSpStages;              // per softmax group: s_full[2] p_full[2] pv_done[2] o_full o_empty
  auto s_full = [&](int t, int b) { return gt_smem_u32(group_bars + t * 8 + b); };
  auto p_full = [&](int t, int b) { return gt_smem_u32(group_bars + t * 8 + 2 + b); };
  auto pv_done = [&](int t, int b) { return gt_smem_u32(group_bars + t * 8 + 4 + b); };
  auto o_full = [&](int t) { return gt_smem_u32(group_bars + t * 8 + 6); };
  auto o_empty = [&](int t) { return gt_smem_u32(group_bars + t * 8 + 7); };
  const uint32_t q_full = gt_smem_u32(group_bars + 16), q_empty = gt_smem_u32(group_bars + 17);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(group_bars + 18);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  __shared__ Segment s_seg[kSpSegments];
  __shared__ int s_n_seg, s_more;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per = p.n_q_heads / p.n_kv_heads, mpt = s.members_per_tile;
  if (threadIdx.x >= 32 && threadIdx.x < 35) {
    const CUtensorMap* m = threadIdx.x == 32 ? &map_k : threadIdx.x == 33 ? &map_v : &map_q;
    asm volatile("prefetch.tensormap [%0];\n" ::"l"(m) : "memory");
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < kSpStages; ++i) {
      mbar_init(gt_smem_u32(&k_full[i]), 32);       // the lanes of its loads' warp, and what TMA brings
      mbar_init(gt_smem_u32(&k_empty[i]), 2);       // both issuers
      mbar_init(gt_smem_u32(&v_full[i]), 32);
      mbar_init(gt_smem_u32(&v_empty[i]), 2);       // both issuers
    }
    for (int t = 0; t < 2; ++t) {
      for (int i = 0; i < 2; ++i) {
        mbar_init(s_full(t, i), 1);
        mbar_init(p_full(t, i), 4);
        mbar_init(pv_done(t, i), 1);
      }
      mbar_init(o_full(t), 1);
      mbar_init(o_empty(t), 4);
    }
    mbar_init(q_full, 1);
    mbar_init(q_empty, 2);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  pdl_wait();
  const int T = __ldcg(s.ints), G = __ldcg(s.ints + 1);
  const int t_begin = (int)blockIdx.x < G ? block_start(T, G, blockIdx.x) : 0, t_end = (int)blockIdx.x < G ? block_start(T, G, blockIdx.x + 1) : 0;
  if (t_begin >= t_end) return;                            // the whole block
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n"
                 ::"r"(gt_smem_u32(tmem_slot)), "r"(TMEM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  // from here on the next kernel may begin: tensor memory is this block's own, and what came before this kernel is complete
  pdl_trigger();

  // positions of the roles, which run on across segments
  int st = 0, st_v = 0;                   // loads: stage to fill (st); issuer: stages of the next S and of the next P V; softmax: stage (st)
  uint32_t ph = 0, ph_v = 0;              // and their phases
  uint32_t n_seg_done = 0;                // segments so far
  uint32_t units0 = 0;                    // issuers and softmax: score tiles of their group so far
  uint32_t outs0 = 0;                     // and the segments in which it had any
  bool ok = true;

  int t_list = t_begin;
  while (true) {
    // ---- the next pieces of the block's range ------------------------------------------------------------------------
    if (threadIdx.x == 0) {
      int n = 0;
      // the group that holds the tile: the last that begins at or before it and is not empty
      int lo_g = 0, hi_g = p.n_groups - 1;
      while (lo_g < hi_g) {
        const int mid = (lo_g + hi_g + 1) >> 1;
        if (__ldcg(s.ints + kPlanHead + mid * kPlanRecord + 7) <= t_list) lo_g = mid; else hi_g = mid - 1;
      }
      int g = lo_g;
      int t = t_list;
      while (t < t_end && n < kSpSegments && g < p.n_groups) {
        const GroupPlan gp = group_plan(s, g);
        const int tiles = plan_tiles(gp), row_tiles = plan_row_tiles(gp, mpt);
        const int end = gp.first + tiles * row_tiles * p.n_kv_heads;
        if (t >= end) { ++g; continue; }
        const int triple = (t - gp.first) / tiles, tile0 = (t - gp.first) % tiles;
        const int n_tiles = min(tiles - tile0, t_end - t);
        const int rt = triple % row_tiles, hkv = triple / row_tiles;
        Segment x;
        x.row0 = gp.row0 + rt * 2 * mpt;
        x.members = min(2 * mpt, gp.members - rt * 2 * mpt);
        x.hkv = hkv;
        x.slot = p.prefix_slot[g];
        x.lo = gp.lo; x.hi = gp.hi; x.common0 = gp.common0; x.common1 = gp.common1; x.prefix_tiles = gp.prefix_tiles;
        x.lo_tile = gp.lo / kSpBN;
        x.tile0 = tile0; x.n_tiles = n_tiles;
        x.piece = n_tiles == tiles ? 2 : t == t_begin ? 0 : 1;
        x.writers = p.req_slot[gp.row0];
        x.group_row0 = gp.row0;
        x.prefix = max(0, p.prefix_len[g]);
        s_seg[n++] = x;
        t += n_tiles;
      }
      s_n_seg = n;
      s_more = t < t_end && n > 0;
    }
    __syncthreads();
    const int n_seg = s_n_seg;
    const bool more = s_more;
    for (int i = 0; i < n_seg; ++i) t_list += s_seg[i].n_tiles;

    if (warp == 0 || warp == kSpValueWarp) {
      // ---- loads of keys, or of values ------------------------------------------------------------------------------------
      const bool values = warp == kSpValueWarp;
      uint64_t* full = values ? v_full : k_full;
      uint64_t* empty = values ? v_empty : k_empty;
      const CUtensorMap* map = values ? &map_v : &map_k;
      const __nv_bfloat16* cache = (const __nv_bfloat16*)(values ? p.v_cache : p.k_cache);
      const uint32_t ring = kv_smem + (values ? V_RING : 0u);
      const int kpl = p.page_size < kSpBN ? p.page_size : kSpBN;     // keys per load
      const int ppt = kSpBN / kpl;                                   // loads of a tile (times SUB halves): at most 8
      const bool loader = lane < ppt * SUB;
      const int c = lane % SUB, u = lane / SUB;
      auto load_queries = [&](const Segment& x) {
        const int n_q = x.members > mpt ? 2 : 1;
        mbar_expect_tx(q_full, (uint32_t)(n_q * SUB * mpt * per * 128));
        for (int t = 0; t < n_q; ++t) {
#pragma unroll
          for (int cc = 0; cc < SUB; ++cc) {
            tma_load_3d(q_smem + t * Q_BYTES + cc * (kSpBM * 128), &map_q, cc * 64, x.hkv * per, x.row0 + t * mpt, q_full);
          }
        }
      };
      for (int i = 0; i < n_seg && ok; ++i, ++n_seg_done) {
        const Segment x = s_seg[i];
        const int n_prefix = min(x.n_tiles, max(0, x.prefix_tiles - x.tile0));       // tiles of the prefix come first
        if (values && n_seg_done == 0) {                             // a block's first queries, while the other warp loads keys
          if (lane == 0) load_queries(x);
          __syncwarp();
        }
        // ---- pages of the prefix's tiles: lane l of a batch has load number 32 * batch + l of the segment ----
        const int* table = p.block_table + (size_t)x.slot * p.max_pages;
        auto batch_of = [&](int batch) {
          const int w = 32 * batch + lane;
          if (w >= n_prefix * ppt) return 0;
          int key0 = (x.lo_tile + x.tile0) * kSpBN + w * kpl;
          if (key0 + kpl - 1 < x.lo || key0 > x.hi) key0 = x.hi / kpl * kpl;          // nothing visible there: any page does
          const int pidx = key0 / p.page_size;
          int page = pidx < p.max_pages ? table[pidx] : -1;
          if (page < 0 || page >= p.num_pages) {
            if (!values) set_error(p.err, kErrPage, x.row0, pidx, page);
            page = 0;
          }
          return (page * p.n_kv_heads + x.hkv) * p.page_size + key0 % p.page_size;    // row of the pools
        };
        int batch_now = 0, rows_now = batch_of(0), rows_next = batch_of(1);
        // ---- places of the common positions behind the prefix: the keys lane and lane + 32 of a tile ----
        int writer0 = 0, writer1 = 0, from0 = -1, from1 = -1, at0 = -1, at1 = -1;
        auto key_of = [&](int j) { return x.common0 + (x.tile0 + j - x.prefix_tiles) * kSpBN + lane; };
        auto follow = [&](int j) {                                   // tile j + 1's pages, tile j + 2's slots, tile j + 3's writers
          if (j + 3 < n_prefix || n_prefix == x.n_tiles) return;
          at0 = at1 = -1;
          if (j + 1 >= n_prefix && j + 1 < x.n_tiles) {
            const int key = key_of(j + 1);
            if (from0 >= 0) at0 = (int)pool_row(p, from0, key, x.hkv, x.group_row0);
            if (from1 >= 0) at1 = (int)pool_row(p, from1, key + 32, x.hkv, x.group_row0);
          }
          from0 = from1 = -1;
          if (j + 2 >= n_prefix && j + 2 < x.n_tiles) {
            const int key = key_of(j + 2);
            if (key < x.common1) from0 = p.req_slot[x.group_row0 + writer0];
            if (key + 32 < x.common1) from1 = p.req_slot[x.group_row0 + writer1];
          }
          if (j + 3 >= n_prefix && j + 3 < x.n_tiles) {
            const unsigned char* h = p.history + (size_t)x.writers * p.history_ld + (key_of(j + 3) - x.prefix);
            if (key_of(j + 3) < x.common1) writer0 = h[0];
            if (key_of(j + 3) + 32 < x.common1) writer1 = h[32];
          }
        };
        follow(-3);
        follow(-2);
        for (int j = 0; j < x.n_tiles && ok; ++j) {
          follow(j - 1);
          ok = __all_sync(0xffffffffu, mbar_wait(gt_smem_u32(&empty[st]), ph ^ 1u, abort_flag));
          if (!ok) { if (lane == 0) { set_error(p.err, kErrWait, 40, values, st); *abort_flag = 1; } break; }
          const uint32_t bar = gt_smem_u32(&full[st]), dst0 = ring + st * KV_BYTES;
          if (j < n_prefix) {
            const int w = j * ppt + u;
            if ((j * ppt) / 32 != batch_now) {                       // a tile's loads are in one batch: ppt divides 32
              ++batch_now;
              rows_now = rows_next;
              rows_next = batch_of(batch_now + 1);
            }
            const int row = __shfl_sync(0xffffffffu, rows_now, w & 31);
            if (lane == 0) {
              mbar_expect_tx(bar, KV_BYTES);
              asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0], 31;\n" ::"r"(bar) : "memory");
            }
            __syncwarp();
            if (loader) tma_load_2d(dst0 + c * KSUB_BYTES + u * kpl * 128, map, c * 64, row, bar);
          } else {
            // rows of 128 bytes in the layout of the 128-byte swizzle: 16-byte chunk ch of row r at (ch ^ (r & 7))
            constexpr int CH = D / 8, ROWS = 32 / CH;                // rows of one pass of the warp
#pragma unroll 8
            for (int r0 = 0; r0 < kSpBN; r0 += ROWS) {
              const int r = r0 + lane / CH, ch = lane % CH;
              const int a = __shfl_sync(0xffffffffu, at0, r & 31), b = __shfl_sync(0xffffffffu, at1, r & 31);
              const int from = r < 32 ? a : b;
              cp_async16(dst0 + (ch / 8) * KSUB_BYTES + r * 128 + (((ch % 8) ^ (r & 7)) * 16), cache + (size_t)(from < 0 ? 0 : from) * D + ch * 8,
                         from >= 0);
            }
            // a lane arrives when its copies have: nobody waits for them here
            asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];\n" ::"r"(bar) : "memory");
          }
          if (++st == kSpStages) { st = 0; ph ^= 1u; }
          if (!values && n_seg_done > 0 && j == min(1, x.n_tiles - 1)) {
            // the queries, behind the first keys, once those of the segment before are done with
            ok = __all_sync(0xffffffffu, mbar_wait(q_empty, (n_seg_done - 1u) & 1u, abort_flag));
            if (!ok) { if (lane == 0) { set_error(p.err, kErrWait, 46, i, 0); *abort_flag = 1; } break; }
            if (lane == 0) load_queries(x);
            __syncwarp();
          }
        }
      }
      cp_async_wait<0>();
    } else if (warp == 1 || warp == kSpSecondIssuer) {
      // ---- products of softmax group t --------------------------------------------------------------------------------------
      // The whole warp walks and waits; one thread issues.  Both issuers give every stage back; one that is not theirs once they
      // have seen it filled.
      const int t = warp == 1 ? 0 : 1;
      const uint32_t idesc_s = umma_idesc(kSpBN, false), idesc_o = umma_idesc(D, true);
      const uint64_t desc_q = umma_desc_sw128(q_smem), desc_k = umma_desc_sw128(kv_smem);
      const uint64_t desc_v = umma_desc_sw128_mn(kv_smem + V_RING, KSUB_BYTES);
      const uint32_t tmem_s = tmem_base + (uint32_t)(t * 128), tmem_o = tmem_base + (uint32_t)(256 + t * 128);
      int where = 0;
      auto wait = [&](uint32_t bar, uint32_t parity, int at) {
        if (ok && !__all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag))) { ok = false; where = at; }
        return ok;
      };
      auto pass_keys = [&]() {             // a key tile of the other group's
        if (!wait(gt_smem_u32(&k_full[st]), ph, 1)) return;
        if (lane == 0) mbar_arrive(gt_smem_u32(&k_empty[st]));
        if (++st == kSpStages) { st = 0; ph ^= 1u; }
      };
      auto pass_values = [&]() {
        if (!wait(gt_smem_u32(&v_full[st_v]), ph_v, 2)) return;
        if (lane == 0) mbar_arrive(gt_smem_u32(&v_empty[st_v]));
        if (++st_v == kSpStages) { st_v = 0; ph_v ^= 1u; }
      };
      for (int i = 0; i < n_seg && ok; ++i, ++n_seg_done) {
        const int n_tiles = s_seg[i].n_tiles, n_prefix = s_seg[i].prefix_tiles - s_seg[i].tile0;
        const bool both = s_seg[i].members > mpt;          // two tiles of rows; otherwise the groups take turns at the key tiles
        const int n_mine = both ? n_tiles : (n_tiles + 1 - t) / 2;
        if (!wait(q_full, n_seg_done & 1u, 4)) break;
        const uint64_t da0 = desc_q + (uint64_t)((both ? t : 0) * (Q_BYTES >> 4));
        if (n_mine == 0 && lane == 0) mbar_arrive(q_empty);
        // scores of tile n, then the second product of tile n - 1
        for (int n = 0; ok && n <= n_mine; ++n) {
          if (n < n_mine) {
            if (!both && (t == 1 || n > 0)) pass_keys();
            if (!wait(gt_smem_u32(&k_full[st]), ph, 1)) break;
            if ((both ? n : 2 * n + t) >= n_prefix) fence_async_shared();          // rows that cp.async brought
            tc_fence_after();
            const int bf = (int)((units0 + (uint32_t)n) & 1u);
            if (elect_one()) {
              const uint64_t db0 = desc_k + (uint64_t)(st * (KV_BYTES >> 4));
#pragma unroll
              for (int ks = 0; ks < D / 16; ++ks) {
                umma_bf16(tmem_s + (uint32_t)(bf * kSpBN), da0 + (uint64_t)((ks / 4) * ((kSpBM * 128) >> 4) + 2 * (ks % 4)),
                          db0 + (uint64_t)((ks / 4) * (KSUB_BYTES >> 4) + 2 * (ks % 4)), idesc_s, ks > 0 ? 1u : 0u);
              }
              umma_commit(s_full(t, bf));
              umma_commit(gt_smem_u32(&k_empty[st]));
              if (n == n_mine - 1) umma_commit(q_empty);
            }
            __syncwarp();
            if (++st == kSpStages) { st = 0; ph ^= 1u; }
          }
          if (n > 0) {
            const uint32_t mine = units0 + (uint32_t)(n - 1);
            const int bf = (int)(mine & 1u);
            if (!both && (t == 1 || n > 1)) pass_values();
            if (!wait(gt_smem_u32(&v_full[st_v]), ph_v, 2)) break;
            if (!wait(p_full(t, bf), (mine >> 1) & 1u, 3)) break;
            if (n == 1 && outs0 > 0 && !wait(o_empty(t), (outs0 - 1u) & 1u, 5)) break;          // the segment before has been read
            if ((both ? n - 1 : 2 * n - 2 + t) >= n_prefix) fence_async_shared();
            tc_fence_after();
            if (elect_one()) {
              const uint64_t db0 = desc_v + (uint64_t)(st_v * (KV_BYTES >> 4));
#pragma unroll
              for (int kk = 0; kk < kSpBN / 16; ++kk) {
                const uint64_t db = db0 + (uint64_t)(kk * ((16 * 128) >> 4));
                const uint32_t a = tmem_s + (uint32_t)(bf * kSpBN + (kk / 2) * 32 + (kk % 2) * 8);
                umma_bf16_ts(tmem_o, a, db, idesc_o, (n > 1 || kk > 0) ? 1u : 0u);
                umma_bf16_ts(tmem_o, a + 16u, db, idesc_o, 1u);
              }
              umma_commit(pv_done(t, bf));
              if (n == n_mine) umma_commit(o_full(t));
              umma_commit(gt_smem_u32(&v_empty[st_v]));
            }
            __syncwarp();
            if (++st_v == kSpStages) { st_v = 0; ph_v ^= 1u; }
          }
        }
        if (!ok) break;
        units0 += (uint32_t)n_mine;
        if (n_mine > 0) ++outs0;
        if (!both && (n_tiles & 1) == t) {                 // the last key tile is the other group's
          pass_keys();
          pass_values();
        }
      }
      if (!ok && lane == 0) { if (!*abort_flag) set_error(p.err, kErrWait, 41, where, (int)n_seg_done); *abort_flag = 1; }
      __syncwarp();
    } else {
      // ---- softmax: row = tensor-memory lane --------------------------------------------------------------------------------
      const int t = (warp - 2) >> 2;
      const int quarter = warp & 3;
      const int row = quarter * 32 + lane;
      const uint32_t lane_addr = (uint32_t)(quarter * 32) << 16;
      const uint32_t tmem_s = tmem_base + lane_addr + (uint32_t)(t * 128);
      const uint32_t tmem_o = tmem_base + lane_addr + (uint32_t)(256 + t * 128);
      uint32_t g = units0, n_out = outs0;
      for (int i = 0; i < n_seg && ok; ++i) {
        const Segment& x = s_seg[i];
        const bool both = x.members > mpt;
        const int n_rows = both ? min(mpt, x.members - t * mpt) * per : x.members * per;
        const bool active = quarter * 32 < n_rows;         // warps without rows keep the barriers' count and do nothing else
        const int tok = x.row0 + (both ? t * mpt : 0) + row / per, head = x.hkv * per + row % per;
        RowSpan sp = {0x7fffffff, 0};                      // a lane without a row masks nothing: nobody reads what comes of it
        if (row < n_rows) sp = row_span(p, tok);
        const int j0 = both ? 0 : t, step = both ? 1 : 2;
        const int n_mine = both ? x.n_tiles : (x.n_tiles - t + 1) / 2;
        float m_ref = -INFINITY, l_sum = 0.0f;
        int j_stage = 0;                                   // key tiles of the segment that `st` has moved on by
        for (int n = 0; n < n_mine && ok; ++n, ++g) {
          const int j = j0 + n * step;
          while (j_stage < j) { if (++st == kSpStages) { st = 0; ph ^= 1u; } ++j_stage; }
          const int bf = (int)(g & 1u);
          const bool prefix = x.tile0 + j < x.prefix_tiles;
          const int key_first = prefix ? (x.lo_tile + x.tile0 + j) * kSpBN : x.common0 + (x.tile0 + j - x.prefix_tiles) * kSpBN;
          const int last = prefix ? x.hi : x.common1 - 1;
          const int hi_r = min(last, sp.pos), lo_r = sp.lo;          // a row without a position sees nothing
          ok = __all_sync(0xffffffffu, mbar_wait(s_full(t, bf), (g >> 1) & 1u, abort_flag));
          if (!ok) { if (lane == 0) { set_error(p.err, kErrWait, 43, j, t); *abort_flag = 1; } break; }
          if (prefix && quarter == 0 && (key_first < x.lo || key_first + kSpBN - 1 > x.hi)) {
            // Values that nobody sees (each group for itself, where both read them: their products are not ordered).  Not before
            // the scores: they say that the values this stage held before have been seen by the group's issuer, without which
            // the wait below could take an older filling, that has yet to arrive, for this one.
            ok = __all_sync(0xffffffffu, mbar_wait(gt_smem_u32(&v_full[st]), ph, abort_flag));
            if (!ok) { if (lane == 0) { set_error(p.err, kErrWait, 42, j, t); *abort_flag = 1; } break; }
            unsigned char* v = smem + 2 * Q_BYTES + V_RING + st * KV_BYTES;
            for (int e = lane; e < kSpBN * D / 8; e += 32) {
              const int k = e / (D / 8), ch = e % (D / 8);
              if (key_first + k < x.lo || key_first + k > x.hi) {
                *reinterpret_cast<uint4*>(v + (ch / 8) * KSUB_BYTES + k * 128 + (ch % 8) * 16) = make_uint4(0u, 0u, 0u, 0u);
              }
            }
            fence_async_shared();
          }
          if (active) {
            tc_fence_after();
            uint32_t sraw[kSpBN];
            {
              uint32_t(&a)[32] = *reinterpret_cast<uint32_t(*)[32]>(&sraw[0]);
              uint32_t(&c)[32] = *reinterpret_cast<uint32_t(*)[32]>(&sraw[32]);
              tmem_ld32(tmem_s + (uint32_t)(bf * kSpBN), a);
              tmem_ld32(tmem_s + (uint32_t)(bf * kSpBN) + 32, c);
              tmem_wait_ld();
            }
            const bool interior = __all_sync(0xffffffffu, key_first >= lo_r && key_first + kSpBN - 1 <= hi_r);
            float sv[kSpBN];
            float mx = -INFINITY;
            if (interior) {
              float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};          // four chains: there is one warp to a scheduler or two
#pragma unroll
              for (int c = 0; c < kSpBN; ++c) { sv[c] = __uint_as_float(sraw[c]); m4[c & 3] = fmaxf(m4[c & 3], sv[c]); }
              mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
            } else {
#pragma unroll
              for (int c = 0; c < kSpBN; ++c) {
                const int key = key_first + c;
                sv[c] = (key >= lo_r && key <= hi_r) ? __uint_as_float(sraw[c]) : -INFINITY;
                mx = fmaxf(mx, sv[c]);
              }
            }
            const bool capped = p.cap_log2 != 0.0f;
            const float eff_scale = capped ? 1.0f : p.scale_log2;
            if (capped) {
              const float cap_in = 2.0f * 1.4426950408889634f * p.inv_cap;
#pragma unroll
              for (int c = 0; c < kSpBN; c += 2) {
                // cap tanh(x / cap) = cap - 2 cap / (2^(2 x log2(e) / cap) + 1), two at a time and on the special functions' own
                // instructions.  (A branch around it, to skip what is masked, would let no two of them overlap: 160 clocks an element.)
                const float2 z = mul2(make_float2(sv[c], sv[c + 1]), make_float2(cap_in, cap_in));
                const float2 e = add2(make_float2(sp_ex2(z.x), sp_ex2(z.y)), make_float2(1.0f, 1.0f));
                const float2 y = fma2(make_float2(sp_rcp(e.x), sp_rcp(e.y)), make_float2(-2.0f * p.cap_log2, -2.0f * p.cap_log2),
                                      make_float2(p.cap_log2, p.cap_log2));
                sv[c] = sv[c] == -INFINITY ? -INFINITY : y.x;
                sv[c + 1] = sv[c + 1] == -INFINITY ? -INFINITY : y.y;
              }
              if (mx != -INFINITY) mx = capped_score_log2(mx, p.scale_log2, p.cap_log2, p.inv_cap);
            }
            mx *= eff_scale;
            const float m_new = fmaxf(m_ref, mx);
            const bool need = m_new > m_ref + kSpRescale;      // also when the first visible key arrives
            if (__any_sync(0xffffffffu, need)) {
              const float corr = need ? exp2f(m_ref - m_new) : 1.0f;
              if (need) { l_sum *= corr; m_ref = m_new; }
              if (n > 0) {
                ok = __all_sync(0xffffffffu, mbar_wait(pv_done(t, (int)((g - 1u) & 1u)), ((g - 1u) >> 1) & 1u, abort_flag));
                if (!ok) { if (lane == 0) { set_error(p.err, kErrWait, 44, j, t); *abort_flag = 1; } break; }
                tc_fence_after();
#pragma unroll
                for (int c = 0; c < D / 32; ++c) {
                  uint32_t o[32];
                  tmem_ld32(tmem_o + c * 32, o);
                  tmem_wait_ld();
#pragma unroll
                  for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * corr);
                  tmem_st32(tmem_o + c * 32, o);
                }
                tmem_wait_st();
                tc_fence_before();
              }
            }
            const float m_use = (m_ref == -INFINITY) ? 0.0f : m_ref;
            float2 psum = make_float2(0.0f, 0.0f);
            const float2 scale2 = make_float2(eff_scale, eff_scale), shift2 = make_float2(-m_use, -m_use);
#pragma unroll
            for (int half = 0; half < kSpBN; half += 32) {
              uint32_t packed[32];         // 32 keys' rounded probabilities, then what the rounding left of each
#pragma unroll
              for (int c = 0; c < 32; c += 2) {
                const float2 y = fma2(make_float2(sv[half + c], sv[half + c + 1]), scale2, shift2);
                const float2 e = make_float2(sp_ex2(y.x), sp_ex2(y.y));
                psum = add2(psum, e);
                packed[c / 2] = pack_bf16(e.x, e.y);
                packed[16 + c / 2] = rest_bf16(e.x, e.y, packed[c / 2]);
              }
              tmem_st32(tmem_s + (uint32_t)(bf * kSpBN + half), packed);
            }
            l_sum += psum.x + psum.y;
            tmem_wait_st();
            tc_fence_before();
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(p_full(t, bf));
        }
        while (j_stage < x.n_tiles) { if (++st == kSpStages) { st = 0; ph ^= 1u; } ++j_stage; }
        if (!ok) break;
        // ---- the rows' part ---------------------------------------------------------------------------------------------
        const size_t at_row = ((size_t)tok * p.n_q_heads + head) * 2 + (both ? 0 : t);
        const size_t at_slot = ((size_t)(blockIdx.x * 2 + (x.piece & 1)) * 2 + t) * kSpBM + row;
        float* ml = x.piece == 2 ? s.whole_ml + 2 * at_row : s.slot_ml + 2 * at_slot;
        float* po = x.piece == 2 ? s.whole_o + at_row * D : s.slot_o + at_slot * D;
        if (n_mine > 0) {
          ok = __all_sync(0xffffffffu, mbar_wait(o_full(t), n_out & 1u, abort_flag));
          if (!ok) { if (lane == 0) { set_error(p.err, kErrWait, 45, i, t); *abort_flag = 1; } break; }
          ++n_out;
          if (active) {
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
              uint32_t o[32];
              tmem_ld32(tmem_o + c * 32, o);
              tmem_wait_ld();
              if (row < n_rows && l_sum > 0.0f) {
#pragma unroll
                for (int q = 0; q < 4; ++q) st_global_32(po + c * 32 + 8 * q, &o[8 * q]);          // (16 bytes at a time: twice the time)
              }
            }
            tc_fence_before();
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(o_empty(t));
        }
        if (row < n_rows) *reinterpret_cast<float2*>(ml) = make_float2(m_ref, l_sum);
      }
      units0 = g;
      outs0 = n_out;
    }
    __syncthreads();
    if (!more || *abort_flag) break;
  }
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) __nanosleep(1000000);       // a block that gave up: its copies in flight land before its memory is another's
  if (warp == 2) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem_base), "r"(TMEM_COLS) : "memory");
  }
}

// ---- parts added up -----------------------------------------------------------------------------------------------------
constexpr int kSpMaxBlocks = 160, kSpMaxOwn = 16;
constexpr int kSpMaxParts = 2 * kSpMaxBlocks + kSpMaxOwn;

struct PartWeight { float m, l; int at; };
struct OwnParts { const float* ml; const float* o; int n, ml_stride, o_stride; };       // strides in floats, from part to part

// One (row, query head) by one warp: the shared positions' parts, wherever the blocks left them, and its own.  `w` is a warp's
// memory for kSpMaxParts weights.
template <int D>
__device__ __forceinline__ void add_parts(const SharedParams& p, const SharedPlan& s, const GroupPlan& gp, bool shared, int row, int hkv,
                                          int j, const OwnParts& own, PartWeight* w, int lane) {
  const int per = p.n_q_heads / p.n_kv_heads, mpt = s.members_per_tile;
  const int head = hkv * per + j;
  const int tiles = shared ? plan_tiles(gp) : 0;
  int n_parts = 0, subs = 1, c0 = 0, t_row = 0, r_in = 0;
  int T = 1, G = 1, a = 0;
  bool whole = false, both = false;
  if (tiles > 0) {
    T = __ldcg(s.ints);
    G = __ldcg(s.ints + 1);
    const int row_tiles = plan_row_tiles(gp, mpt);
    const int rel = row - gp.row0, rt = rel / (2 * mpt), in = rel - rt * 2 * mpt;
    both = min(2 * mpt, gp.members - rt * 2 * mpt) > mpt;
    subs = both ? 1 : 2;
    t_row = both ? in / mpt : 0;
    r_in = (both ? in % mpt : in) * per + j;
    a = gp.first + (hkv * row_tiles + rt) * tiles;
    c0 = tile_owner(T, G, a);
    const int c1 = tile_owner(T, G, a + tiles - 1);
    whole = c0 == c1;
    n_parts = (c1 - c0 + 1) * subs;
  }
  auto place = [&](int i) -> int {             // of part i among its kind
    if (whole) return (row * p.n_q_heads + head) * 2 + i;
    const int c = c0 + (subs == 2 ? i >> 1 : i);
    const int piece = block_start(T, G, c) >= a ? 0 : 1;
    return ((c * 2 + piece) * 2 + (both ? t_row : i & 1)) * kSpBM + r_in;
  };
  const float* shared_ml = whole ? s.whole_ml : s.slot_ml;
  const float* shared_o = whole ? s.whole_o : s.slot_o;
  const int n = n_parts + own.n;
  // w: a part's weight, and its place (of the row's own parts: -1 - index)
  float m_all = -INFINITY;
  for (int i = lane; i < n; i += 32) {
    const int at = i < n_parts ? place(i) : -1 - (i - n_parts);
    const float2 v = at >= 0 ? __ldcg(reinterpret_cast<const float2*>(shared_ml) + at)
                             : *reinterpret_cast<const float2*>(own.ml + (-1 - at) * own.ml_stride);
    w[i] = {v.x, v.y, at};
    if (v.y > 0.0f) m_all = fmaxf(m_all, v.x);
  }
  m_all = warp_max(m_all);
  float l_all = 0.0f;
  for (int i = lane; i < n; i += 32) {
    const PartWeight v = w[i];
    const float f = v.l > 0.0f ? exp2f(v.m - m_all) : 0.0f;
    l_all += v.l * f;
    w[i].m = f;
  }
  l_all = warp_sum(l_all);
  __syncwarp();
  const float inv = l_all > 0.0f ? 1.0f / (l_all + sink_term_log2(p.sinks, head, m_all)) : 0.0f;
  // a lane has four columns; with heads of 64 the two halves of the warp take every second part
  constexpr int LANES = D / 4, STEP = 32 / LANES, AHEAD = 8;
  const int c4 = lane % LANES, part0 = lane / LANES;
  float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int i0 = part0; i0 < n; i0 += STEP * AHEAD) {
    float4 v[AHEAD];
    float f[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int i = i0 + k * STEP;
      f[k] = i < n ? w[i].m : 0.0f;
      v[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (f[k] != 0.0f) {                      // an empty part has no output that is anything
        const int at = w[i].at;
        v[k] = at >= 0 ? __ldcg(reinterpret_cast<const float4*>(shared_o + (size_t)at * D) + c4)
                       : *(reinterpret_cast<const float4*>(own.o + (-1 - at) * own.o_stride) + c4);
      }
    }
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      acc.x += v[k].x * f[k]; acc.y += v[k].y * f[k]; acc.z += v[k].z * f[k]; acc.w += v[k].w * f[k];
    }
  }
  if (STEP == 2) {
    acc.x += __shfl_xor_sync(0xffffffffu, acc.x, 16); acc.y += __shfl_xor_sync(0xffffffffu, acc.y, 16);
    acc.z += __shfl_xor_sync(0xffffffffu, acc.z, 16); acc.w += __shfl_xor_sync(0xffffffffu, acc.w, 16);
  }
  if (part0 == 0) {
    uint2 out;
    out.x = pack_bf16(acc.x * inv, acc.y * inv);
    out.y = pack_bf16(acc.z * inv, acc.w * inv);
    reinterpret_cast<uint2*>((__nv_bfloat16*)p.out + ((size_t)row * p.n_q_heads + head) * D)[c4] = out;
  }
  __syncwarp();
}

// A row's group as the plan has it, or an error and false where the row is in none (or in more members than planned for).
__device__ __forceinline__ bool row_group(const SharedParams& p, const SharedPlan& s, int row, GroupPlan& gp, int2& rows, int& prefix) {
  const int g = group_of_row(p, row);
  rows = group_rows(p, g);
  prefix = max(0, p.prefix_len[g]);
  const bool shared = s.ints != nullptr;
  if (shared) gp = group_plan(s, g);
  if (row >= rows.x && row < rows.y && (shared || prefix == 0) && (p.n_shared > 0 || prefix == 0)) return true;
  set_error(p.err, kErrRequest, row, p.max_members, prefix);
  return false;
}

// ---- the positions behind the shared ones -------------------------------------------------------------------------------
constexpr int kSoWarps = 4;
constexpr int kSoTile = 16;           // keys of a warp's tile
constexpr int kSoChunk = 1024;        // keys whose places are looked up at a time

template <int D, int STAGES>
constexpr int own_smem(int per) {
  const int tiles = kSoWarps * STAGES * 2 * kSoTile * D * 2, parts = kSoWarps * (per * (D + 2) * 4 + kSpMaxParts * (int)sizeof(PartWeight));
  return tiles > parts ? tiles : parts;
}

// STAGES: tiles of a warp on their way or in use.  With a history most positions behind the prefix are common to a group, few are
// left to a row, and what counts is how many rows are under way: one stage, four blocks on an SM (62 us against 67 for 16 groups of 4,
// 113 against 119 for 4 of 16, measured, as all in these comments but the times of whole calls, before probabilities were two bfloat16).
// Without one all of them are the rows' own: two stages, three blocks (58 us against 73 for 48 rows
// with up to 700).
template <int D, int STAGES>
__global__ void __launch_bounds__(kSoWarps * 32, STAGES == 1 ? 4 : 3)
shared_own_kernel(const __grid_constant__ SharedParams p, const __grid_constant__ SharedPlan s) {
  constexpr int CH = D / 8;                       // 16-byte chunks per row
  constexpr int TILE_BYTES = kSoTile * D * 2;
  constexpr int STAGE_BYTES = 2 * TILE_BYTES;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ int s_row[kSoChunk];                 // row of the pools, -1: none
  const int split = blockIdx.x, hkv = blockIdx.y, row = blockIdx.z;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int gi = lane >> 2, t4 = lane & 3;
  const int per = p.n_q_heads / p.n_kv_heads;
  const bool shared = s.ints != nullptr;
  const __nv_bfloat16* kc = (const __nv_bfloat16*)p.k_cache;
  const __nv_bfloat16* vc = (const __nv_bfloat16*)p.v_cache;
  // The kernel in front of this one (the shared positions') writes nothing that is read here, and lets this one begin only when
  // all before it, the plan too, was complete; where there is none, this waits for what is.
  if (!shared) pdl_wait();
  pdl_trigger();

  GroupPlan gp = {};
  int2 rows;
  int prefix;
  int slot = checked_slot(p, p.req_slot[row], row);
  const bool in_group = row_group(p, s, row, gp, rows, prefix);
  if (!in_group) slot = -1;
  const RowSpan sp = row_span(p, row);
  const int lo = max(sp.lo, shared && in_group ? gp.common1 : prefix), pos = slot < 0 ? -1 : sp.pos;
  const int n_tiles = pos >= lo ? (pos - lo) / kSoTile + 1 : 0;
  const int per_split = (n_tiles + p.n_own - 1) / p.n_own;
  const int t_begin = split * per_split, t_end = min(n_tiles, t_begin + per_split);

  const uint32_t my_smem = smem_u32(smem + warp * STAGES * STAGE_BYTES);
  float o[D / 8][4];
#pragma unroll
  for (int i = 0; i < D / 8; ++i) { o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f; }
  float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.0f, 0.0f};
  uint32_t qa[D / 16][4];
  if (t_begin < t_end) {
    const __nv_bfloat16* qbase = (const __nv_bfloat16*)p.q + ((size_t)row * p.n_q_heads + (size_t)hkv * per) * D;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      const int c0 = ks * 16 + 2 * t4;
      qa[ks][0] = (gi < per) ? *reinterpret_cast<const uint32_t*>(qbase + (size_t)gi * D + c0) : 0u;
      qa[ks][2] = (gi < per) ? *reinterpret_cast<const uint32_t*>(qbase + (size_t)gi * D + c0 + 8) : 0u;
      qa[ks][1] = (gi + 8 < per) ? *reinterpret_cast<const uint32_t*>(qbase + (size_t)(gi + 8) * D + c0) : 0u;
      qa[ks][3] = (gi + 8 < per) ? *reinterpret_cast<const uint32_t*>(qbase + (size_t)(gi + 8) * D + c0 + 8) : 0u;
    }
  }
  for (int c0 = t_begin; c0 < t_end; c0 += kSoChunk / kSoTile) {
    const int c1 = min(t_end, c0 + kSoChunk / kSoTile);
    const int key_base = lo + c0 * kSoTile;
    if (c0 > t_begin) __syncthreads();            // the places of the chunk before are not read any more
    for (int i = threadIdx.x; i < (c1 - c0) * kSoTile; i += kSoWarps * 32) {
      const int key = key_base + i;
      s_row[i] = key <= pos ? (int)pool_row(p, writer_slot(p, row, slot, key, pos, prefix, rows), key, hkv, row) : -1;
    }
    __syncthreads();
    auto issue_load = [&](int tile, int stage) {
      const uint32_t kdst = my_smem + stage * STAGE_BYTES, vdst = kdst + TILE_BYTES;
#pragma unroll
      for (int i = 0; i < (kSoTile * CH) / 32; ++i) {
        const int idx = i * 32 + lane;
        const int r = idx / CH, chunk = idx % CH;
        const int at = s_row[(tile - c0) * kSoTile + r];
        const int off = swizzled_offset(r, chunk, CH);
        const size_t src = (size_t)(at < 0 ? 0 : at) * D + chunk * 8;
        cp_async16(kdst + off, kc + src, at >= 0);
        cp_async16(vdst + off, vc + src, at >= 0);
      }
    };
    const int n_mine = (c1 - c0 - warp + kSoWarps - 1) / kSoWarps;
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) {
      if (s < n_mine) issue_load(c0 + warp + s * kSoWarps, s);
      cp_async_commit();
    }
    for (int i = 0; i < n_mine; ++i) {
      const int tile = c0 + warp + i * kSoWarps;
      if (i + STAGES - 1 < n_mine) issue_load(tile + (STAGES - 1) * kSoWarps, (i + STAGES - 1) % STAGES);
      cp_async_commit();
      cp_async_wait<STAGES - 1>();
      __syncwarp();
      const uint32_t kbase = my_smem + (i % STAGES) * STAGE_BYTES, vbase = kbase + TILE_BYTES;
      float s[2][4];
#pragma unroll
      for (int nt = 0; nt < 2; ++nt) { s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.0f; }
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        const int r = ((lane >> 4) << 3) + (lane & 7);
        const int chunk = 2 * ks + ((lane >> 3) & 1);
        uint32_t b0, b1, b2, b3;
        ldmatrix_x4(kbase + swizzled_offset(r, chunk, CH), b0, b1, b2, b3);
        mma_bf16_16816(s[0], qa[ks][0], qa[ks][1], qa[ks][2], qa[ks][3], b0, b1);
        mma_bf16_16816(s[1], qa[ks][0], qa[ks][1], qa[ks][2], qa[ks][3], b2, b3);
      }
      float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int nt = 0; nt < 2; ++nt) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const bool valid = s_row[(tile - c0) * kSoTile + nt * 8 + 2 * t4 + (e & 1)] >= 0;
          s[nt][e] = valid ? capped_score_log2(s[nt][e], p.scale_log2, p.cap_log2, p.inv_cap) : -INFINITY;
          mx[e >> 1] = fmaxf(mx[e >> 1], s[nt][e]);
        }
      }
      float corr[2], m_use[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
        mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
        const float m_new = fmaxf(m_run[h], mx[h]);
        m_use[h] = (m_new == -INFINITY) ? 0.0f : m_new;
        corr[h] = exp2f(m_run[h] - m_use[h]);
        m_run[h] = m_new;
      }
      float psum[2] = {0.0f, 0.0f};
#pragma unroll
      for (int nt = 0; nt < 2; ++nt) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[nt][e] = exp2f(s[nt][e] - m_use[e >> 1]);
          psum[e >> 1] += s[nt][e];
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) l_run[h] = l_run[h] * corr[h] + psum[h];
#pragma unroll
      for (int i2 = 0; i2 < D / 8; ++i2) {
        o[i2][0] *= corr[0]; o[i2][1] *= corr[0];
        o[i2][2] *= corr[1]; o[i2][3] *= corr[1];
      }
      const uint32_t pa0 = pack_bf16(s[0][0], s[0][1]), pa1 = pack_bf16(s[0][2], s[0][3]);
      const uint32_t pa2 = pack_bf16(s[1][0], s[1][1]), pa3 = pack_bf16(s[1][2], s[1][3]);
      const uint32_t pr0 = rest_bf16(s[0][0], s[0][1], pa0), pr1 = rest_bf16(s[0][2], s[0][3], pa1);
      const uint32_t pr2 = rest_bf16(s[1][0], s[1][1], pa2), pr3 = rest_bf16(s[1][2], s[1][3], pa3);
#pragma unroll
      for (int c = 0; c < D / 8; c += 2) {
        const int r = (((lane >> 3) & 1) << 3) + (lane & 7);
        const int chunk = c + (lane >> 4);
        uint32_t b0, b1, b2, b3;
        ldmatrix_x4_trans(vbase + swizzled_offset(r, chunk, CH), b0, b1, b2, b3);
        mma_bf16_16816(o[c], pa0, pa1, pa2, pa3, b0, b1);
        mma_bf16_16816(o[c + 1], pa0, pa1, pa2, pa3, b2, b3);
        mma_bf16_16816(o[c], pr0, pr1, pr2, pr3, b0, b1);
        mma_bf16_16816(o[c + 1], pr0, pr1, pr2, pr3, b2, b3);
      }
      __syncwarp();
    }
    cp_async_wait<0>();
  }

  // ---- the warps' parts ----------------------------------------------------------------------------------------------------
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    l_run[h] += __shfl_xor_sync(0xffffffffu, l_run[h], 1);
    l_run[h] += __shfl_xor_sync(0xffffffffu, l_run[h], 2);
  }
  __syncthreads();
  float* so = reinterpret_cast<float*>(smem);                  // [warps][query heads][D]
  float* sml = so + kSoWarps * per * D;                        // [warps][query heads][2]
#pragma unroll
  for (int i2 = 0; i2 < D / 8; ++i2) {
    const int col = i2 * 8 + 2 * t4;
    if (gi < per) *reinterpret_cast<float2*>(so + (warp * per + gi) * D + col) = make_float2(o[i2][0], o[i2][1]);
    if (gi + 8 < per) *reinterpret_cast<float2*>(so + (warp * per + gi + 8) * D + col) = make_float2(o[i2][2], o[i2][3]);
  }
  if (t4 == 0) {
    if (gi < per) *reinterpret_cast<float2*>(sml + (warp * per + gi) * 2) = make_float2(m_run[0], l_run[0]);
    if (gi + 8 < per) *reinterpret_cast<float2*>(sml + (warp * per + gi + 8) * 2) = make_float2(m_run[1], l_run[1]);
  }
  __syncthreads();
  if (!s.apart) {
    if (shared) pdl_wait();           // the shared positions' parts are there; and whoever waits for this kernel waits for that one
    PartWeight* w = reinterpret_cast<PartWeight*>(sml + kSoWarps * per * 2) + warp * kSpMaxParts;
    for (int j = warp; j < per; j += kSoWarps) {
      const OwnParts own = {sml + j * 2, so + j * D, kSoWarps, per * 2, per * D};
      add_parts<D>(p, s, gp, shared && in_group, row, hkv, j, own, w, lane);
    }
    return;
  }
  for (int idx = threadIdx.x; idx < per * D; idx += kSoWarps * 32) {
    const int r = idx / D, col = idx % D;
    float m_all = -INFINITY;
#pragma unroll
    for (int w = 0; w < kSoWarps; ++w) m_all = fmaxf(m_all, sml[(w * per + r) * 2]);
    float acc = 0.0f, l_all = 0.0f;
#pragma unroll
    for (int w = 0; w < kSoWarps; ++w) {
      const float mw = sml[(w * per + r) * 2];
      const float f = (mw == -INFINITY) ? 0.0f : exp2f(mw - m_all);
      acc += so[(w * per + r) * D + col] * f;
      l_all += sml[(w * per + r) * 2 + 1] * f;
    }
    const size_t at = ((size_t)row * p.n_q_heads + (size_t)hkv * per + r) * p.n_own + split;
    if (l_all > 0.0f) s.own_o[at * D + col] = acc;
    if (col == 0) { s.own_ml[2 * at] = m_all; s.own_ml[2 * at + 1] = l_all; }
  }
  // whoever waits for this kernel waits for the shared positions' one, for which one block that does is enough
  if (shared && blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0) pdl_wait();
}

// The parts of rows whose own ones were left apart: a warp per (row, query head).
constexpr int kSmWarps = 8;
template <int D>
__global__ void __launch_bounds__(kSmWarps * 32) shared_add_kernel(const __grid_constant__ SharedParams p, const __grid_constant__ SharedPlan s) {
  __shared__ PartWeight s_w[kSmWarps][kSpMaxParts];
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long pair = (long long)blockIdx.x * kSmWarps + warp;
  if (pair >= (long long)p.n_rows * p.n_q_heads) return;
  const int row = (int)(pair / p.n_q_heads), head = (int)(pair % p.n_q_heads), per = p.n_q_heads / p.n_kv_heads;
  GroupPlan gp = {};
  int2 rows;
  int prefix;
  const bool in_group = row_group(p, s, row, gp, rows, prefix);
  const OwnParts own = {s.own_ml + 2 * pair * p.n_own, s.own_o + pair * p.n_own * D, p.n_own, 2, D};
  add_parts<D>(p, s, gp, s.ints != nullptr && in_group, row, head / per, head % per, own, s_w[warp], lane);
}

// ---- host ------------------------------------------------------------------------------------------------------------------
bool shared_tc_takes(const SharedParams& p) {
  const int per = p.n_kv_heads > 0 ? p.n_q_heads / p.n_kv_heads : 0;
  const bool pages = p.page_size >= 8 && p.page_size % 8 == 0 && (kSpBN % p.page_size == 0 || p.page_size % kSpBN == 0);
  return (p.d == 64 || p.d == 128) && p.dv == p.d && p.n_kv_heads <= 65535 && p.n_rows <= 65535 && per >= 1 && per <= 16 && pages &&
         p.n_own <= kSpMaxOwn && (((uintptr_t)p.q | (uintptr_t)p.k_cache | (uintptr_t)p.v_cache) & 15) == 0 && ((uintptr_t)p.out & 7) == 0 &&
         (long long)p.num_pages * p.n_kv_heads * p.page_size <= 0x7fffffffLL;
}

static bool has_shared(const SharedParams& p) { return p.n_shared > 0 || p.history != nullptr; }

static SharedPlan layout(const SharedParams& p, int sms, long long* floats) {
  SharedPlan s = {};
  long long at = 0;
  auto take = [&](long long n) { float* q = p.scratch + at; at += (n + 7) / 8 * 8; return q; };
  const long long pairs = (long long)p.n_rows * p.n_q_heads;
  if (has_shared(p)) {
    s.ints = reinterpret_cast<int*>(take(kPlanHead + (long long)p.n_groups * kPlanRecord));
    s.blocks = sms < kSpMaxBlocks ? sms : kSpMaxBlocks;
    if (p.n_shared > 0 && p.n_shared < s.blocks) { s.blocks = p.n_shared; s.apart = true; }
    s.members_per_tile = kSpBM / (p.n_q_heads / p.n_kv_heads);
    s.slot_ml = take(4LL * s.blocks * kSpBM * 2);
    s.whole_ml = take(pairs * 2 * 2);
    s.slot_o = take(4LL * s.blocks * kSpBM * p.d);
    s.whole_o = take(pairs * 2 * p.d);
  }
  s.apart = s.apart || p.n_own > 1;
  if (s.apart) {
    s.own_ml = take(pairs * p.n_own * 2);
    s.own_o = take(pairs * p.n_own * p.d);
  }
  *floats = at;
  return s;
}

long long shared_tc_scratch(const SharedParams& p, int sms) {
  long long floats = 0;
  layout(p, sms, &floats);
  return floats;
}

template <int D>
static int launch_tc(const SharedParams& p, int sms, cudaStream_t stream) {
  long long floats = 0;
  const SharedPlan s = layout(p, sms, &floats);
  // the key tiles of all triples are counted in 32 bits
  const long long triples = (long long)p.n_kv_heads * (p.n_groups + (has_shared(p) ? p.n_rows / (2 * s.members_per_tile) : 0));
  if (triples * ((long long)p.max_pages * p.page_size / kSpBN + 3) > 0x7fffffffLL) return (int)cudaErrorInvalidValue;
  const int stages = p.history != nullptr ? 1 : 2;
  constexpr int smem_shared = 2 * kSpBM * D * 2 + 2 * kSpStages * kSpBN * D * 2 + 1024 + 512;
  static_assert(smem_shared + kSpSegments * sizeof(Segment) + 64 <= 232448, "shared memory of one block");
  static_assert((4 * kSpStages + 18) * 8 + 16 <= 512, "barriers");
  const int per = p.n_q_heads / p.n_kv_heads, smem_own = stages == 1 ? own_smem<D, 1>(per) : own_smem<D, 2>(per);
  static bool configured[64] = {false};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return (int)e;
  if (dev < 0 || dev >= 64) return (int)cudaErrorInvalidValue;
  if (!configured[dev]) {
    e = cudaFuncSetAttribute(shared_prefix_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_shared);
    if (e != cudaSuccess) return (int)e;
    e = cudaFuncSetAttribute(shared_own_kernel<D, 1>, cudaFuncAttributeMaxDynamicSharedMemorySize, own_smem<D, 1>(16));
    if (e != cudaSuccess) return (int)e;
    e = cudaFuncSetAttribute(shared_own_kernel<D, 2>, cudaFuncAttributeMaxDynamicSharedMemorySize, own_smem<D, 2>(16));
    if (e != cudaSuccess) return (int)e;
    configured[dev] = true;
  }
  if (has_shared(p)) {
    CUtensorMap mq, mk, mv;
    {
      cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)p.n_q_heads, (cuuint64_t)p.n_rows};
      cuuint64_t strides[2] = {(cuuint64_t)D * 2, (cuuint64_t)p.n_q_heads * D * 2};
      cuuint32_t box[3] = {64, (cuuint32_t)(p.n_q_heads / p.n_kv_heads), (cuuint32_t)s.members_per_tile};
      const int rc = make_bf16_map(&mq, p.q, 3, dims, strides, box);
      if (rc != 0) return rc;
    }
    {
      cuuint64_t dims[2] = {(cuuint64_t)D, (cuuint64_t)p.num_pages * p.n_kv_heads * p.page_size};
      cuuint64_t strides[1] = {(cuuint64_t)D * 2};
      cuuint32_t box[2] = {64, (cuuint32_t)(p.page_size < kSpBN ? p.page_size : kSpBN)};
      int rc = make_bf16_map(&mk, p.k_cache, 2, dims, strides, box);
      if (rc != 0) return rc;
      rc = make_bf16_map(&mv, p.v_cache, 2, dims, strides, box);
      if (rc != 0) return rc;
    }
    e = launch(shared_plan_kernel, dim3(1), dim3(kPlanThreads), 0, stream, p, s);
    if (e != cudaSuccess) return (int)e;
    e = launch(shared_prefix_kernel<D>, dim3(s.blocks), dim3(kSpThreads), smem_shared, stream, mq, mk, mv, p, s);
    if (e != cudaSuccess) return (int)e;
  }
  e = launch(stages == 1 ? shared_own_kernel<D, 1> : shared_own_kernel<D, 2>, dim3(p.n_own, p.n_kv_heads, p.n_rows), dim3(kSoWarps * 32), smem_own, stream, p, s);
  if (e != cudaSuccess || !s.apart) return (int)e;
  const long long pairs = (long long)p.n_rows * p.n_q_heads;
  return (int)launch(shared_add_kernel<D>, dim3((unsigned)((pairs + kSmWarps - 1) / kSmWarps)), dim3(kSmWarps * 32), 0, stream, p, s);
}

int launch_shared_tc(const SharedParams& p, int sms, cudaStream_t stream) {
  return p.d == 128 ? launch_tc<128>(p, sms, stream) : launch_tc<64>(p, sms, stream);
}

}  // namespace tk
