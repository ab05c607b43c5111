// Attention over shared prefixes in bfloat16 with heads of 64 or 128 elements (attention_shared.cuh has the definition).
//
// Shared positions: tcgen05.  The query heads of a group's members over one key/value head are up to 128 (two tiles: 256)
// rows of Q; a block takes a range of 64-key tiles of one (group, key/value head), so the keys are read from memory once for
// all of these rows.  Roles of a block:
//   warp 0       loads with TMA: the query tiles, then key and value tiles, page by page, into rings of their own;
//   warp 1       one thread issues tcgen05.mma: S = Q K^T (M 128, N 64) into one of a query tile's two score buffers in tensor
//                memory, then, for the key tile before, O += P V (N head size) with P from tensor memory and V as an
//                MN-major operand straight from its page layout, so S of a tile is under way while the softmax of
//                the one before runs;
//   warps 2..    four per query tile, thread i owns row i: scores with tcgen05.ld, mask, running reference and sum in float32,
//                probabilities as bfloat16 pairs over the scores.  The output is rescaled in tensor memory only when a
//                row's maximum grew by more than 2^8 since its reference was set.  Warps without rows do nothing.
// Bound: the keys' bytes.  A 64-key tile of 128 elements is 32 KB (0.74 us of an SM's share of the memory bandwidth) against
// 0.38 us of tensor time a query tile, which 32 or 128 rows cost alike.
//
// Rows of V that no row may see (behind the prefix in its last page, in front of a window) are zeroed in shared memory
// before they are used: their probabilities are zero, and what lies there may be anything.
//
// Other positions: mma.sync, a block per (range of keys, key/value head, row), the query heads over the key/value head as
// the rows of a 16-row tile.  Four warps walk 16-key tiles with cp.async, each key's address looked up once, ahead of the
// loop, for the block: with a history neighbouring keys lie in different members' pages.
#include "attention_shared.cuh"
#include "tcgen05_utils.cuh"

namespace tk {

constexpr int kSpBM = 128;            // rows of a query tile
constexpr int kSpBN = 64;             // keys of a tile
constexpr int kSpStages = 4;
constexpr float kSpRescale = 8.0f;    // log2 units

__device__ __forceinline__ float sp_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}

template <int D, int QT>
__global__ void __launch_bounds__(64 + 128 * QT, 1)
shared_prefix_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                     const __grid_constant__ CUtensorMap map_v, const __grid_constant__ SharedParams p, int row_tiles, int members_per_tile) {
  constexpr int SUB = D / 64;
  constexpr uint32_t Q_BYTES = kSpBM * D * 2;
  constexpr uint32_t KSUB_BYTES = kSpBN * 64 * 2;
  constexpr uint32_t KV_BYTES = kSpBN * D * 2;
  constexpr uint32_t V_RING = kSpStages * KV_BYTES;
  constexpr uint32_t DATA_BYTES = QT * Q_BYTES + 2 * kSpStages * KV_BYTES;
  constexpr uint32_t TMEM_COLS = QT == 1 ? 256 : 512;      // scores of tile t at t * 128, outputs at QT * 128 + t * 128

  extern __shared__ __align__(1024) unsigned char smem_raw[];
  const uint32_t raw = gt_smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  unsigned char* smem = smem_raw + (base - raw);
  const uint32_t q_smem = base, kv_smem = base + QT * Q_BYTES;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + DATA_BYTES);
  uint64_t* k_full = bars;
  uint64_t* k_empty = k_full + kSpStages;
  uint64_t* v_full = k_empty + kSpStages;
  uint64_t* v_empty = v_full + kSpStages;
  uint64_t* tile_bars = v_empty + kSpStages;               // per query tile: s_full[2] p_full[2] pv_done[2] o_full; then q_full
  auto s_full = [&](int t, int b) { return gt_smem_u32(tile_bars + t * 7 + b); };
  auto p_full = [&](int t, int b) { return gt_smem_u32(tile_bars + t * 7 + 2 + b); };
  auto pv_done = [&](int t, int b) { return gt_smem_u32(tile_bars + t * 7 + 4 + b); };
  auto o_full = [&](int t) { return gt_smem_u32(tile_bars + t * 7 + 6); };
  const uint32_t q_full = gt_smem_u32(tile_bars + QT * 7);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tile_bars + QT * 7 + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* s_range = const_cast<int*>(abort_flag) + 1;         // lowest visible key, highest position

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per = p.n_q_heads / p.n_kv_heads;
  int b = blockIdx.x;
  const int rt = b % row_tiles; b /= row_tiles;
  const int split = b % p.n_shared; b /= p.n_shared;
  const int hkv = b % p.n_kv_heads;
  const int g = b / p.n_kv_heads;
  if (threadIdx.x == 0) { s_range[0] = 0x7fffffff; s_range[1] = -1; *abort_flag = 0; }
  __syncthreads();
  pdl_wait();

  // ---- what this block's rows see ------------------------------------------------------------------------------------
  const int2 rows = group_rows(p, g);
  const int row0 = rows.x + rt * members_per_tile * QT;
  const int n_members = min(members_per_tile * QT, rows.y - row0);
  if (n_members <= 0) return;
  const int prefix = max(0, p.prefix_len[g]);
  const int slot = prefix > 0 ? checked_slot(p, p.prefix_slot[g], row0) : -1;
  for (int i = threadIdx.x; i < n_members; i += blockDim.x) {
    const RowSpan sp = row_span(p, row0 + i);
    if (sp.pos >= 0) { atomicMin(&s_range[0], sp.lo); atomicMax(&s_range[1], sp.pos); }
  }
  __syncthreads();
  const int lo = s_range[0], hi = slot < 0 ? -1 : min(prefix - 1, s_range[1]);
  int first = 0, n_kt = 0;
  if (hi >= lo) {
    const int t_lo = lo / kSpBN, n_tiles = hi / kSpBN - t_lo + 1;
    const int per_split = (n_tiles + p.n_shared - 1) / p.n_shared;
    first = t_lo + split * per_split;
    n_kt = max(0, min(per_split, t_lo + n_tiles - first));
  }
  auto tile_members = [&](int t) { return min(members_per_tile, n_members - t * members_per_tile); };
  auto part_of = [&](int row, int head) { return ((size_t)row * p.n_q_heads + head) * p.n_parts + split; };
  if (n_kt == 0) {
    for (int i = threadIdx.x; i < n_members * per; i += blockDim.x) {
      float* ml = p.part_ml + 2 * part_of(row0 + i / per, hkv * per + i % per);
      ml[0] = -INFINITY; ml[1] = 0.0f;
    }
    return;
  }
  const int n_q = n_members > members_per_tile ? 2 : 1;    // query tiles that have rows
  if (threadIdx.x == 0) {
    for (int s = 0; s < kSpStages; ++s) {
      mbar_init(gt_smem_u32(&k_full[s]), 1);
      mbar_init(gt_smem_u32(&k_empty[s]), 1);
      mbar_init(gt_smem_u32(&v_full[s]), 1);
      mbar_init(gt_smem_u32(&v_empty[s]), 1);
    }
    for (int t = 0; t < n_q; ++t) {
      for (int i = 0; i < 2; ++i) {
        mbar_init(s_full(t, i), 1);
        mbar_init(p_full(t, i), (tile_members(t) * per + 31) / 32);        // an arrival per warp with rows
        mbar_init(pv_done(t, i), 1);
      }
      mbar_init(o_full(t), 1);
    }
    mbar_init(q_full, 1);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
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

  if (warp == 0) {
    // ---- producer -----------------------------------------------------------------------------------------------------
    if (lane == 0) {
      mbar_expect_tx(q_full, (uint32_t)(n_q * SUB * members_per_tile * per * 128));
      for (int t = 0; t < n_q; ++t) {
#pragma unroll
        for (int c = 0; c < SUB; ++c) {
          tma_load_3d(q_smem + t * Q_BYTES + c * (kSpBM * 128), &map_q, c * 64, hkv * per, row0 + t * members_per_tile, q_full);
        }
      }
    }
    __syncwarp();
    const int kpl = p.page_size < kSpBN ? p.page_size : kSpBN;     // keys per load
    const int n_loads = (kSpBN / kpl) * SUB * 2;                   // at most 32: page sizes from 8
    const bool loader = lane < n_loads;
    const int is_v = lane & 1, c = (lane >> 1) % SUB, u = lane / (2 * SUB);
    const int* table = p.block_table + (size_t)slot * p.max_pages;
    auto key0_of = [&](int j) {
      const int key0 = (first + j) * kSpBN + u * kpl;
      return (key0 + kpl - 1 < lo || key0 > hi) ? hi / kpl * kpl : key0;          // nothing visible there: any page does
    };
    auto lookup = [&](int j) {
      const int pidx = key0_of(j) / p.page_size;
      return (loader && j < n_kt && pidx < p.max_pages) ? table[pidx] : -1;
    };
    int page = lookup(0), st = 0;
    uint32_t ph = 0;
    for (int j = 0; j < n_kt; ++j) {
      const int next = lookup(j + 1);
      const int key0 = key0_of(j);
      if (loader && (page < 0 || page >= p.num_pages)) {
        set_error(p.err, kErrPage, row0, key0 / p.page_size, page);
        page = 0;
      }
      const int row = (page * p.n_kv_heads + hkv) * p.page_size + key0 % p.page_size;
      const uint32_t dst = kv_smem + st * KV_BYTES + c * KSUB_BYTES + u * kpl * 128;
      bool ok = __all_sync(0xffffffffu, mbar_wait(gt_smem_u32(&k_empty[st]), ph ^ 1u, abort_flag));
      if (ok) {
        if (lane == 0) mbar_expect_tx(gt_smem_u32(&k_full[st]), KV_BYTES);
        __syncwarp();
        if (loader && !is_v) tma_load_2d(dst, &map_k, c * 64, row, gt_smem_u32(&k_full[st]));
        ok = __all_sync(0xffffffffu, mbar_wait(gt_smem_u32(&v_empty[st]), ph ^ 1u, abort_flag));
      }
      if (!ok) { if (lane == 0) { set_error(p.err, kErrWait, 40, j, st); *abort_flag = 1; } break; }
      if (lane == 0) mbar_expect_tx(gt_smem_u32(&v_full[st]), KV_BYTES);
      __syncwarp();
      if (loader && is_v) tma_load_2d(dst + V_RING, &map_v, c * 64, row, gt_smem_u32(&v_full[st]));
      if (++st == kSpStages) { st = 0; ph ^= 1u; }
      page = next;
    }
  } else if (warp == 1) {
    // ---- products -------------------------------------------------------------------------------------------------------
    if (elect_one()) {
      const uint32_t idesc_s = umma_idesc(kSpBN, false), idesc_o = umma_idesc(D, true);
      const uint64_t desc_q = umma_desc_sw128(q_smem), desc_k = umma_desc_sw128(kv_smem);
      const uint64_t desc_v = umma_desc_sw128_mn(kv_smem + V_RING, KSUB_BYTES);
      int st = 0, st_v = 0;
      uint32_t ph = 0, ph_v = 0;
      bool ok = mbar_wait(q_full, 0, abort_flag);
      int where = 0;
      for (int j = 0; ok && j <= n_kt; ++j) {
        if (j < n_kt) {
          // scores of key tile j; their buffer held the probabilities of tile j - 2, whose product this thread has issued
          ok = mbar_wait(gt_smem_u32(&k_full[st]), ph, abort_flag);
          if (!ok) { where = 1; break; }
          tc_fence_after();
          for (int t = 0; t < n_q; ++t) {
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks) {
              const uint64_t da = desc_q + (uint64_t)(t * (Q_BYTES >> 4) + (ks / 4) * ((kSpBM * 128) >> 4) + 2 * (ks % 4));
              const uint64_t db = desc_k + (uint64_t)(st * (KV_BYTES >> 4) + (ks / 4) * (KSUB_BYTES >> 4) + 2 * (ks % 4));
              umma_bf16(tmem_base + (uint32_t)(t * 128 + (j & 1) * kSpBN), da, db, idesc_s, ks > 0 ? 1u : 0u);
            }
            umma_commit(s_full(t, j & 1));
          }
          umma_commit(gt_smem_u32(&k_empty[st]));
          if (++st == kSpStages) { st = 0; ph ^= 1u; }
        }
        if (j > 0) {
          const int i = j - 1;
          ok = mbar_wait(gt_smem_u32(&v_full[st_v]), ph_v, abort_flag);
          if (!ok) { where = 2; break; }
          for (int t = 0; t < n_q; ++t) {
            ok = mbar_wait(p_full(t, i & 1), (uint32_t)(i >> 1) & 1u, abort_flag);
            if (!ok) { where = 3; break; }
            tc_fence_after();
#pragma unroll
            for (int kk = 0; kk < kSpBN / 16; ++kk) {
              const uint64_t db = desc_v + (uint64_t)(st_v * (KV_BYTES >> 4) + kk * ((16 * 128) >> 4));
              umma_bf16_ts(tmem_base + (uint32_t)(QT * 128 + t * 128), tmem_base + (uint32_t)(t * 128 + (i & 1) * kSpBN + 8 * kk), db, idesc_o,
                           (i > 0 || kk > 0) ? 1u : 0u);
            }
            umma_commit(pv_done(t, i & 1));
            if (i == n_kt - 1) umma_commit(o_full(t));
          }
          if (!ok) break;
          umma_commit(gt_smem_u32(&v_empty[st_v]));
          if (++st_v == kSpStages) { st_v = 0; ph_v ^= 1u; }
        }
      }
      if (!ok) { set_error(p.err, kErrWait, 41, where, n_kt); *abort_flag = 1; }
    }
  } else {
    // ---- softmax of query tile t: row = tensor-memory lane ----------------------------------------------------------------
    const int t = (warp - 2) >> 2;
    const int quarter = warp & 3;
    const int n_rows = t < n_q ? tile_members(t) * per : 0;
    if (quarter * 32 < n_rows) {
      const int row = quarter * 32 + lane;
      const uint32_t lane_addr = (uint32_t)(quarter * 32) << 16;
      const uint32_t tmem_s = tmem_base + lane_addr + (uint32_t)(t * 128);
      const uint32_t tmem_o = tmem_base + lane_addr + (uint32_t)(QT * 128 + t * 128);
      const int tok = row0 + t * members_per_tile + row / per, head = hkv * per + row % per;
      RowSpan sp = {-1, 0};
      if (row < n_rows) sp = row_span(p, tok);
      const int hi_r = min(hi, sp.pos), lo_r = sp.lo;      // a row without a position sees nothing: hi_r < 0
      float m_ref = -INFINITY, l_sum = 0.0f;
      bool ok = true;
      int st = 0;
      uint32_t ph = 0;
      for (int j = 0; j < n_kt; ++j) {
        const int bf = j & 1;
        const int key_first = (first + j) * kSpBN;
        if (t == 0 && quarter == 0 && (key_first < lo || key_first + kSpBN - 1 > hi)) {
          // values that nobody sees
          ok = __all_sync(0xffffffffu, mbar_wait(gt_smem_u32(&v_full[st]), ph, abort_flag));
          if (!ok) { if (lane == 0) { set_error(p.err, kErrWait, 42, j, t); *abort_flag = 1; } break; }
          unsigned char* v = smem + QT * Q_BYTES + V_RING + st * KV_BYTES;
          for (int i = lane; i < kSpBN * D / 8; i += 32) {
            const int k = i / (D / 8), ch = i % (D / 8);
            if (key_first + k < lo || key_first + k > hi) {
              *reinterpret_cast<uint4*>(v + (ch / 8) * KSUB_BYTES + k * 128 + (ch % 8) * 16) = make_uint4(0u, 0u, 0u, 0u);
            }
          }
          fence_async_shared();
        }
        if (++st == kSpStages) { st = 0; ph ^= 1u; }
        ok = __all_sync(0xffffffffu, mbar_wait(s_full(t, bf), (uint32_t)(j >> 1) & 1u, abort_flag));
        if (!ok) { if (lane == 0) { set_error(p.err, kErrWait, 43, j, t); *abort_flag = 1; } break; }
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
#pragma unroll
          for (int c = 0; c < kSpBN; ++c) { sv[c] = __uint_as_float(sraw[c]); mx = fmaxf(mx, sv[c]); }
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
#pragma unroll
          for (int c = 0; c < kSpBN; ++c) {
            if (sv[c] != -INFINITY) sv[c] = capped_score_log2(sv[c], p.scale_log2, p.cap_log2, p.inv_cap);
          }
          if (mx != -INFINITY) mx = capped_score_log2(mx, p.scale_log2, p.cap_log2, p.inv_cap);
        }
        mx *= eff_scale;
        const float m_new = fmaxf(m_ref, mx);
        const bool need = m_new > m_ref + kSpRescale;      // also when the first visible key arrives
        if (__any_sync(0xffffffffu, need)) {
          const float corr = need ? exp2f(m_ref - m_new) : 1.0f;
          if (need) { l_sum *= corr; m_ref = m_new; }
          if (j > 0) {
            ok = __all_sync(0xffffffffu, mbar_wait(pv_done(t, (j - 1) & 1), (uint32_t)((j - 1) >> 1) & 1u, abort_flag));
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
        for (int c = 0; c < kSpBN; c += 2) {
          const float2 x = fma2(make_float2(sv[c], sv[c + 1]), scale2, shift2);
          sv[c] = sp_ex2(x.x);
          sv[c + 1] = sp_ex2(x.y);
          psum = add2(psum, make_float2(sv[c], sv[c + 1]));
        }
        l_sum += psum.x + psum.y;
        {
          uint32_t packed[kSpBN / 2];
#pragma unroll
          for (int c = 0; c < kSpBN / 2; ++c) packed[c] = pack_bf16(sv[2 * c], sv[2 * c + 1]);
          tmem_st32(tmem_s + (uint32_t)(bf * kSpBN), packed);
          tmem_wait_st();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full(t, bf));
      }
      if (ok) {
        ok = __all_sync(0xffffffffu, mbar_wait(o_full(t), 0, abort_flag));
        if (!ok && lane == 0) { set_error(p.err, kErrWait, 45, n_kt, t); *abort_flag = 1; }
      }
      if (ok) {
        tc_fence_after();
        const size_t at = part_of(row < n_rows ? tok : row0, head);
        if (row < n_rows) { p.part_ml[2 * at] = m_ref; p.part_ml[2 * at + 1] = l_sum; }
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          tmem_ld32(tmem_o + c * 32, o);
          tmem_wait_ld();
          if (row < n_rows && l_sum > 0.0f) {
#pragma unroll
            for (int q = 0; q < 8; ++q) {
              reinterpret_cast<uint4*>(p.part_o + at * D + c * 32)[q] = make_uint4(o[4 * q], o[4 * q + 1], o[4 * q + 2], o[4 * q + 3]);
            }
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) __nanosleep(1000000);       // a block that gave up: its copies in flight land before its memory is another's
  if (warp == 2) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem_base), "r"(TMEM_COLS) : "memory");
  }
}

// ---- the positions behind the prefix -----------------------------------------------------------------------------------
constexpr int kSoWarps = 4;
constexpr int kSoTile = 16;           // keys of a warp's tile
constexpr int kSoChunk = 1024;        // keys whose places are looked up at a time

template <int D, int STAGES>
__global__ void __launch_bounds__(kSoWarps * 32)
shared_own_kernel(const __grid_constant__ SharedParams p) {
  constexpr int CH = D / 8;                       // 16-byte chunks per row
  constexpr int TILE_BYTES = kSoTile * D * 2;
  constexpr int STAGE_BYTES = 2 * TILE_BYTES;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ int s_row[kSoChunk];                 // row of the pools, -1: none
  const int split = blockIdx.x, hkv = blockIdx.y, row = blockIdx.z;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int gi = lane >> 2, t4 = lane & 3;
  const int per = p.n_q_heads / p.n_kv_heads;
  const __nv_bfloat16* kc = (const __nv_bfloat16*)p.k_cache;
  const __nv_bfloat16* vc = (const __nv_bfloat16*)p.v_cache;
  // The kernel in front of this one (the shared positions') writes nothing that is read here, and began only when all
  // before it was complete; where there is none, this waits for what is.
  if (p.n_shared == 0) pdl_wait();
  pdl_trigger();

  const int g = group_of_row(p, row);
  const int2 rows = group_rows(p, g);
  const int prefix = max(0, p.prefix_len[g]);
  int slot = checked_slot(p, p.req_slot[row], row);
  if (!row_has_group(p, row, rows, prefix, split == 0 && (int)threadIdx.x < per ? hkv * per + (int)threadIdx.x : -1)) slot = -1;
  const RowSpan sp = row_span(p, row);
  const int lo = max(sp.lo, prefix), pos = slot < 0 ? -1 : sp.pos;
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
#pragma unroll
      for (int c = 0; c < D / 8; c += 2) {
        const int r = (((lane >> 3) & 1) << 3) + (lane & 7);
        const int chunk = c + (lane >> 4);
        uint32_t b0, b1, b2, b3;
        ldmatrix_x4_trans(vbase + swizzled_offset(r, chunk, CH), b0, b1, b2, b3);
        mma_bf16_16816(o[c], pa0, pa1, pa2, pa3, b0, b1);
        mma_bf16_16816(o[c + 1], pa0, pa1, pa2, pa3, b2, b3);
      }
      __syncwarp();
    }
    cp_async_wait<0>();
  }

  // ---- the warps' parts become the block's -------------------------------------------------------------------------------
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    l_run[h] += __shfl_xor_sync(0xffffffffu, l_run[h], 1);
    l_run[h] += __shfl_xor_sync(0xffffffffu, l_run[h], 2);
  }
  __syncthreads();
  float* so = reinterpret_cast<float*>(smem);                  // [warps][16][D]
  float* sml = so + kSoWarps * 16 * D;                         // [warps][16][2]
#pragma unroll
  for (int i2 = 0; i2 < D / 8; ++i2) {
    const int col = i2 * 8 + 2 * t4;
    float* row0 = so + ((size_t)warp * 16 + gi) * D + col;
    float* row1 = so + ((size_t)warp * 16 + gi + 8) * D + col;
    row0[0] = o[i2][0]; row0[1] = o[i2][1];
    row1[0] = o[i2][2]; row1[1] = o[i2][3];
  }
  if (t4 == 0) {
    sml[(warp * 16 + gi) * 2 + 0] = m_run[0];     sml[(warp * 16 + gi) * 2 + 1] = l_run[0];
    sml[(warp * 16 + gi + 8) * 2 + 0] = m_run[1]; sml[(warp * 16 + gi + 8) * 2 + 1] = l_run[1];
  }
  __syncthreads();
  if (p.n_shared > 0) pdl_wait();      // the scratch memory may have belonged to the kernel before; and whoever waits for this one waits for it too
  for (int idx = threadIdx.x; idx < per * D; idx += kSoWarps * 32) {
    const int r = idx / D, col = idx % D;
    float m_all = -INFINITY;
#pragma unroll
    for (int w = 0; w < kSoWarps; ++w) m_all = fmaxf(m_all, sml[(w * 16 + r) * 2]);
    float acc = 0.0f, l_all = 0.0f;
#pragma unroll
    for (int w = 0; w < kSoWarps; ++w) {
      const float mw = sml[(w * 16 + r) * 2];
      const float f = (mw == -INFINITY) ? 0.0f : exp2f(mw - m_all);
      acc += so[((size_t)w * 16 + r) * D + col] * f;
      l_all += sml[(w * 16 + r) * 2 + 1] * f;
    }
    const size_t at = ((size_t)row * p.n_q_heads + (size_t)hkv * per + r) * p.n_parts + p.n_shared + split;
    if (l_all > 0.0f) p.part_o[at * D + col] = acc;
    if (col == 0) { p.part_ml[2 * at] = m_all; p.part_ml[2 * at + 1] = l_all; }
  }
}

bool shared_tc_takes(const SharedParams& p) {
  const int per = p.n_kv_heads > 0 ? p.n_q_heads / p.n_kv_heads : 0;
  const bool pages = p.page_size >= 8 && p.page_size % 8 == 0 && (kSpBN % p.page_size == 0 || p.page_size % kSpBN == 0);
  return (p.d == 64 || p.d == 128) && p.dv == p.d && p.n_kv_heads <= 65535 && p.n_rows <= 65535 && per >= 1 && per <= 16 && pages &&
         (((uintptr_t)p.q | (uintptr_t)p.k_cache | (uintptr_t)p.v_cache) & 15) == 0 &&
         (long long)p.num_pages * p.n_kv_heads * p.page_size <= 0x7fffffffLL;
}

template <int D, int QT>
static int launch_prefix(const SharedParams& p, int members_per_tile, cudaStream_t stream) {
  const int per = p.n_q_heads / p.n_kv_heads;
  CUtensorMap mq, mk, mv;
  {
    cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)p.n_q_heads, (cuuint64_t)p.n_rows};
    cuuint64_t strides[2] = {(cuuint64_t)D * 2, (cuuint64_t)p.n_q_heads * D * 2};
    cuuint32_t box[3] = {64, (cuuint32_t)per, (cuuint32_t)members_per_tile};
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
  constexpr int smem = QT * kSpBM * D * 2 + 2 * kSpStages * kSpBN * D * 2 + 1024 + 512;
  static_assert(smem <= 232448, "shared memory of one block");
  static_assert((4 * kSpStages + QT * 7 + 1) * 8 + 16 <= 512, "barriers");
  cudaError_t e = cudaFuncSetAttribute(shared_prefix_kernel<D, QT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return (int)e;
  const int row_tiles = (p.max_members + members_per_tile * QT - 1) / (members_per_tile * QT);
  const long long blocks = (long long)p.n_groups * p.n_kv_heads * p.n_shared * row_tiles;
  if (blocks > 0x7fffffffLL) return (int)cudaErrorInvalidValue;
  return (int)launch(shared_prefix_kernel<D, QT>, dim3((unsigned)blocks), dim3(64 + 128 * QT), smem, stream, mq, mk, mv, p, row_tiles,
                     members_per_tile);
}

template <int D>
static int launch_tc(const SharedParams& p, cudaStream_t stream) {
  if (p.n_shared > 0) {
    const int members_per_tile = kSpBM / (p.n_q_heads / p.n_kv_heads);
    const int e = p.max_members > members_per_tile ? launch_prefix<D, 2>(p, members_per_tile, stream)
                                                    : launch_prefix<D, 1>(p, members_per_tile, stream);
    if (e != 0) return e;
  }
  constexpr int STAGES = 2;
  constexpr int stages = kSoWarps * STAGES * 2 * kSoTile * D * 2, merge = kSoWarps * 16 * (D + 2) * 4;
  constexpr int smem = stages > merge ? stages : merge;
  cudaError_t e = cudaFuncSetAttribute(shared_own_kernel<D, STAGES>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return (int)e;
  return (int)launch(shared_own_kernel<D, STAGES>, dim3(p.n_own, p.n_kv_heads, p.n_rows), dim3(kSoWarps * 32), smem, stream, p);
}

int launch_shared_tc(const SharedParams& p, cudaStream_t stream) {
  return p.d == 128 ? launch_tc<128>(p, stream) : launch_tc<64>(p, stream);
}

}  // namespace tk
