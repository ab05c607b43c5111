// Attention over shared prefixes: the general kernel (float32 or bfloat16, any head size up to 256) for both parts, the
// one that adds parts up, and the entry point.  attention_shared.cuh has the definition.
#include "attention_shared.cuh"

namespace tk {

// ---- general kernel -----------------------------------------------------------------------------------------------
//
// A block takes up to 32 (row, query head) pairs over one key/value head and a range of keys: of the shared positions, where
// the pairs are those of a tile of the group's members, or of one row's others.  Tiles of 32 keys go through shared memory as
// float32; warp w holds four pairs: a lane computes the four scores of its key, then owns four (or eight) columns of the output.
// Bound by latency where it is used (float32, and shapes the tensor-core kernels refuse): 4 rows of 16 query heads over 8 of
// 64, 1,021 shared and 61 further positions in float32 take 19 us, of which the keys' 4.5 MB would need one.  So the
// keys are cut down to 32 a block, both kinds of positions go into one launch (64 a block and two launches: 37 us, 23 without
// them), and a warp's loads of a tile are on their way together.
constexpr int kShRows = 32;
constexpr int kShKeys = 32;
constexpr int kShThreads = 256;

// Four elements as floats.
template <typename T>
__device__ __forceinline__ float4 load4(const T* src) {
  if constexpr (sizeof(T) == 4) return *reinterpret_cast<const float4*>(src);
  const uint2 u = *reinterpret_cast<const uint2*>(src);
  const __nv_bfloat162 a = *reinterpret_cast<const __nv_bfloat162*>(&u.x), b = *reinterpret_cast<const __nv_bfloat162*>(&u.y);
  return make_float4(__bfloat162float(a.x), __bfloat162float(a.y), __bfloat162float(b.x), __bfloat162float(b.y));
}

// N rows of len(r) elements, `longest` at most, to shared memory by a warp, padded with zeros to a multiple of four; src(r) is null
// for a row of zeros, dst(r) null for none.  The rows' loads are under way together.
template <typename T, int N, typename Len, typename Src, typename Dst>
__device__ __forceinline__ void load_rows(int longest, bool wide, int lane, Len len, Src src, Dst dst) {
  for (int c = 4 * lane; c < longest; c += 128) {
    float4 f[N];
#pragma unroll
    for (int r = 0; r < N; ++r) {
      const T* from = src(r);
      f[r] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (from == nullptr || c >= len(r)) continue;
      if (wide) {
        f[r] = load4<T>(from + c);
      } else {
        float* e = &f[r].x;
#pragma unroll
        for (int k = 0; k < 4; ++k) if (c + k < len(r)) e[k] = to_f32<T>(from[c + k]);
      }
    }
#pragma unroll
    for (int r = 0; r < N; ++r) {
      float* to = dst(r);
      if (to != nullptr && c < len(r)) *reinterpret_cast<float4*>(to + c) = f[r];
    }
  }
}

// A score in units of log2(e), capped by cap tanh(x / cap).  In float32 with tanhf: what capped_score_log2's fast exponential and division
// leave, a few 1e-7 of the cap, is 1e-6 of a result, where float32 products and sums alone leave 3e-7.
template <typename T>
__device__ __forceinline__ float shared_score_log2(const SharedParams& p, float dot) {
  if (sizeof(T) == 4 && p.cap_log2 != 0.0f) return p.cap_log2 * tanhf(dot * p.inv_cap);
  return capped_score_log2(dot, p.scale_log2, p.cap_log2, p.inv_cap);
}

template <typename T, int kChunks>       // kChunks: 128-column chunks of a value row
__global__ void __launch_bounds__(kShThreads) shared_parts_kernel(SharedParams p, int shared_tiles, int own_tiles, int n_shared_blocks) {
  pdl_trigger();
  extern __shared__ __align__(16) float s_mem[];
  __shared__ long long s_row[kShKeys];
  __shared__ int s_pos[kShRows], s_lo[kShRows], s_tok[kShRows], s_head[kShRows];
  __shared__ float s_p[kShRows / 4][kShKeys][4];
  const int dp = (p.d + 3) / 4 * 4, dvp = (p.dv + 3) / 4 * 4;
  const int ldk = dp + 4;
  float* s_q = s_mem;                          // [kShRows][dp]
  float* s_k = s_q + kShRows * dp;             // [kShKeys][ldk]
  float* s_v = s_k + kShKeys * ldk;            // [kShKeys][dvp]
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = p.n_q_heads / p.n_kv_heads;
  pdl_wait();

  // ---- what this block does ------------------------------------------------------------------------------------
  const bool shared = (int)blockIdx.x < n_shared_blocks;
  int b = shared ? (int)blockIdx.x : (int)blockIdx.x - n_shared_blocks;
  const int splits = shared ? p.n_shared : p.n_own;
  const int split = b % splits; b /= splits;
  const int hkv = b % p.n_kv_heads; b /= p.n_kv_heads;
  const int row_tiles = shared ? shared_tiles : own_tiles;
  const int tile = b % row_tiles; b /= row_tiles;
  int g, first_pair, n_pairs, prefix, slot = -1, own_row = -1;
  int2 rows;
  if (shared) {
    g = b;
    rows = group_rows(p, g);
    first_pair = tile * kShRows;
    n_pairs = min(kShRows, (rows.y - rows.x) * per - first_pair);
    prefix = max(0, p.prefix_len[g]);
    slot = prefix > 0 && n_pairs > 0 ? checked_slot(p, p.prefix_slot[g], rows.x) : -1;
  } else {
    own_row = b;
    g = group_of_row(p, own_row);
    rows = group_rows(p, g);
    first_pair = tile * kShRows;
    n_pairs = min(kShRows, per - first_pair);
    prefix = max(0, p.prefix_len[g]);
    slot = checked_slot(p, p.req_slot[own_row], own_row);
  }
  if (n_pairs <= 0) return;
  if (!shared && !row_has_group(p, own_row, rows, prefix, split == 0 && tid < n_pairs ? hkv * per + first_pair + tid : -1)) slot = -1;
  if (tid < kShRows) {
    const int pair = first_pair + tid;
    const int row = shared ? rows.x + pair / per : own_row;
    s_tok[tid] = row;
    s_head[tid] = hkv * per + pair % per;
    RowSpan sp = {-1, 0};
    if (tid < n_pairs) sp = row_span(p, row);
    s_pos[tid] = sp.pos;
    s_lo[tid] = sp.lo;
  }
  __syncthreads();
  int lo = 0x7fffffff, hi = -1;                // keys that any of the pairs sees
  for (int i = 0; i < n_pairs; ++i) {
    if (s_pos[i] >= 0) { lo = min(lo, s_lo[i]); hi = max(hi, s_pos[i]); }
  }
  if (shared) hi = min(hi, prefix - 1); else lo = max(lo, prefix);
  if (slot < 0) hi = -1;
  const int n_keys = hi >= lo ? hi - lo + 1 : 0;
  const int n_tiles = (n_keys + kShKeys - 1) / kShKeys;
  const int per_split = (n_tiles + splits - 1) / splits;
  const int t0 = split * per_split, t1 = min(n_tiles, t0 + per_split);

  const bool wide_k = p.wide_k, wide_v = p.wide_v;
  if (t0 < t1) {
    constexpr int WARPS = kShThreads / 32;
    load_rows<T, kShRows / WARPS>(p.d, wide_k, lane, [&](int) { return p.d; }, [&](int r) -> const T* {
      const int i = warp + r * WARPS;
      return i < n_pairs ? (const T*)p.q + ((size_t)s_tok[i] * p.n_q_heads + s_head[i]) * p.d : nullptr;
    }, [&](int r) -> float* { return warp + r * WARPS < n_pairs ? s_q + (warp + r * WARPS) * dp : nullptr; });
  }
  float m[4], l[4], acc[4][4 * kChunks];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    m[r] = -INFINITY; l[r] = 0.0f;
#pragma unroll
    for (int c = 0; c < 4 * kChunks; ++c) acc[r][c] = 0.0f;
  }
  const bool active = 4 * warp < n_pairs;
  for (int t = t0; t < t1; ++t) {
    const int key0 = lo + t * kShKeys;
    __syncthreads();                           // the tile before is done with
    if (tid < kShKeys) {
      const int key = key0 + tid;
      long long at = -1;
      if (key <= hi) {
        const int from = shared ? slot : writer_slot(p, own_row, slot, key, s_pos[0], prefix, rows);
        at = pool_row(p, from, key, hkv, s_tok[0]);
      }
      s_row[tid] = at;
    }
    __syncthreads();
    {
      // (a key that is not there is zeros: nothing that lies in its place may reach the result)
      constexpr int WARPS = kShThreads / 32, N = kShKeys / WARPS;
      load_rows<T, 2 * N>(max(p.d, p.dv), wide_k && wide_v, lane, [&](int r) { return r < N ? p.d : p.dv; }, [&](int r) -> const T* {
        const long long at = s_row[warp + r % N * WARPS];
        return at < 0 ? nullptr : r < N ? (const T*)p.k_cache + at * p.d : (const T*)p.v_cache + at * p.dv;
      }, [&](int r) { return r < N ? s_k + (warp + r * WARPS) * ldk : s_v + (warp + (r - N) * WARPS) * dvp; });
    }
    __syncthreads();
    if (active) {
      float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      const float* kr = s_k + lane * ldk;
      const float* qr = s_q + 4 * warp * dp;
#pragma unroll 4
      for (int c = 0; c < dp; c += 4) {
        const float4 kv = *reinterpret_cast<const float4*>(kr + c);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float4 qv = *reinterpret_cast<const float4*>(qr + r * dp + c);
          s[r] = fmaf(qv.x, kv.x, s[r]); s[r] = fmaf(qv.y, kv.y, s[r]);
          s[r] = fmaf(qv.z, kv.z, s[r]); s[r] = fmaf(qv.w, kv.w, s[r]);
        }
      }
      const int key = key0 + lane;
      float4 prob;
      float* pr = &prob.x;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = 4 * warp + r;
        const bool seen = i < n_pairs && s_row[lane] >= 0 && key <= s_pos[i] && key >= s_lo[i];
        const float x = seen ? shared_score_log2<T>(p, s[r]) : -INFINITY;
        const float m_new = fmaxf(m[r], warp_max(x));
        const float m_use = m_new == -INFINITY ? 0.0f : m_new;
        const float corr = exp2f(m[r] - m_use);
        m[r] = m_new;
        pr[r] = exp2f(x - m_use);
        l[r] = l[r] * corr + warp_sum(pr[r]);
#pragma unroll
        for (int c = 0; c < 4 * kChunks; ++c) acc[r][c] *= corr;
      }
      *reinterpret_cast<float4*>(&s_p[warp][lane][0]) = prob;
      __syncwarp();
#pragma unroll
      for (int ch = 0; ch < kChunks; ++ch) {
        const int col = ch * 128 + lane * 4;
        if (col < dvp) {
#pragma unroll 8
          for (int j = 0; j < kShKeys; ++j) {
            const float4 w = *reinterpret_cast<const float4*>(&s_p[warp][j][0]);
            const float4 vv = *reinterpret_cast<const float4*>(s_v + j * dvp + col);
            const float wr[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              acc[r][4 * ch] = fmaf(wr[r], vv.x, acc[r][4 * ch]);
              acc[r][4 * ch + 1] = fmaf(wr[r], vv.y, acc[r][4 * ch + 1]);
              acc[r][4 * ch + 2] = fmaf(wr[r], vv.z, acc[r][4 * ch + 2]);
              acc[r][4 * ch + 3] = fmaf(wr[r], vv.w, acc[r][4 * ch + 3]);
            }
          }
        }
      }
      __syncwarp();
    }
  }
  if (!active) return;
  const int part = shared ? split : p.n_shared + split;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int i = 4 * warp + r;
    if (i >= n_pairs) break;
    const size_t at = ((size_t)s_tok[i] * p.n_q_heads + s_head[i]) * p.n_parts + part;
    if (lane == 0) { p.part_ml[2 * at] = m[r]; p.part_ml[2 * at + 1] = l[r]; }
    if (l[r] > 0.0f) {                         // a part without keys has no output that anybody reads
#pragma unroll
      for (int ch = 0; ch < kChunks; ++ch) {
        const int col = ch * 128 + lane * 4;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          if (col + c < p.dv) p.part_o[at * p.dv + col + c] = acc[r][4 * ch + c];
        }
      }
    }
  }
}

// ---- parts added up -------------------------------------------------------------------------------------------------
// A warp per (row, query head); a row that sees nothing is zero.
constexpr int kMergeWarps = 8;

template <typename T>
__global__ void __launch_bounds__(kMergeWarps * 32) shared_merge_kernel(SharedParams p) {
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const long long pair = (long long)blockIdx.x * kMergeWarps + (threadIdx.x >> 5);
  if (pair >= (long long)p.n_rows * p.n_q_heads) return;
  const int head = (int)(pair % p.n_q_heads);
  const float2* ml = reinterpret_cast<const float2*>(p.part_ml) + pair * p.n_parts;
  const float* o = p.part_o + (size_t)pair * p.n_parts * p.dv;
  float2 mine = lane < p.n_parts ? __ldcg(ml + lane) : make_float2(-INFINITY, 0.0f);
  float m_all = mine.x;
  for (int i = lane + 32; i < p.n_parts; i += 32) m_all = fmaxf(m_all, __ldcg(ml + i).x);
  m_all = warp_max(m_all);
  const bool wide = p.dv % 4 == 0;
  T* out = (T*)p.out + pair * p.dv;
  for (int c0 = 0; c0 < p.dv; c0 += 128) {
    const int c = c0 + 4 * lane;
    float l_all = 0.0f;
    float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int i0 = 0; i0 < p.n_parts; i0 += 32) {
      if (i0 > 0 || c0 > 0) mine = i0 + lane < p.n_parts ? __ldcg(ml + i0 + lane) : make_float2(-INFINITY, 0.0f);
      const float f = mine.y > 0.0f ? exp2f(mine.x - m_all) : 0.0f;
      l_all += f * mine.y;
      const int n = min(32, p.n_parts - i0);
      // eight parts' loads at a time: they have nothing to wait for but each other's latency
      for (int j = 0; j < n; j += 8) {
        float v[8][4], w[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          w[k] = j + k < n ? __shfl_sync(0xffffffffu, f, j + k) : 0.0f;
          v[k][0] = v[k][1] = v[k][2] = v[k][3] = 0.0f;
          if (w[k] == 0.0f || c >= p.dv) continue;        // an empty part has no output that is anything
          const float* src = o + (size_t)(i0 + j + k) * p.dv + c;
          if (wide) {
            const float4 x = __ldcg(reinterpret_cast<const float4*>(src));
            v[k][0] = x.x; v[k][1] = x.y; v[k][2] = x.z; v[k][3] = x.w;
          } else {
            for (int e = 0; e < 4 && c + e < p.dv; ++e) v[k][e] = __ldcg(src + e);
          }
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[e] += v[k][e] * w[k];
        }
      }
    }
    l_all = warp_sum(l_all);
    const float inv = l_all > 0.0f ? 1.0f / (l_all + sink_term_log2(p.sinks, head, m_all)) : 0.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (c + e < p.dv) out[c + e] = from_f32<T>(acc[e] * inv);
    }
  }
}

template <typename T>
static int launch_general(const SharedParams& p, cudaStream_t stream) {
  const int per = p.n_q_heads / p.n_kv_heads;
  const int dp = (p.d + 3) / 4 * 4, dvp = (p.dv + 3) / 4 * 4;
  const size_t smem = sizeof(float) * ((size_t)kShRows * dp + (size_t)kShKeys * (dp + 4) + (size_t)kShKeys * dvp);
  const int shared_tiles = (p.max_members * per + kShRows - 1) / kShRows, own_tiles = (per + kShRows - 1) / kShRows;
  const long long n_shared = (long long)p.n_groups * shared_tiles * p.n_kv_heads * p.n_shared;
  const long long n_own = (long long)p.n_rows * own_tiles * p.n_kv_heads * p.n_own;
  if (n_shared + n_own > 0x7fffffffLL) return (int)cudaErrorInvalidValue;
  auto run = [&](auto kernel) -> int {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return (int)e;
    return (int)launch(kernel, dim3((unsigned)(n_shared + n_own)), dim3(kShThreads), smem, stream, p, shared_tiles, own_tiles, (int)n_shared);
  };
  return p.dv <= 128 ? run(shared_parts_kernel<T, 1>) : run(shared_parts_kernel<T, 2>);
}

template <typename T>
static int launch_merge(const SharedParams& p, cudaStream_t stream) {
  const long long pairs = (long long)p.n_rows * p.n_q_heads;
  return (int)launch(shared_merge_kernel<T>, dim3((unsigned)((pairs + kMergeWarps - 1) / kMergeWarps)), dim3(kMergeWarps * 32), 0,
                     stream, p);
}

}  // namespace tk

// Whether the kernels of attention_shared_tc.cu take a shape (addresses on 16 bytes besides).
TK_API int tk_attention_shared_tc_takes(int n_q_heads, int n_kv_heads, int head_dim, int v_dim, int page_size) {
  tk::SharedParams p = {};
  p.n_q_heads = n_q_heads; p.n_kv_heads = n_kv_heads; p.d = head_dim; p.dv = v_dim; p.page_size = page_size; p.n_own = 1;
  return tk::shared_tc_takes(p);
}

// scratch: 32-byte aligned, as many floats as tk_attention_shared_scratch says for the same arguments.
static int shared_params(tk::SharedParams& p, const void* q, void* out, const void* k_cache, const void* v_cache, int n_rows, int n_groups,
                         int max_members, int n_q_heads, int n_kv_heads, int head_dim, int v_dim, int page_size, int num_pages, int n_shared,
                         int n_own, const unsigned char* history, int dtype) {
  const long long parts = (long long)n_rows * n_q_heads * ((long long)n_shared + n_own);
  if (n_kv_heads < 1 || n_q_heads < 1 || n_q_heads % n_kv_heads != 0 || head_dim < 1 || head_dim > 256 || v_dim < 1 || v_dim > 256 ||
      page_size < 1 || max_members < 1 || n_shared < 0 || n_own < 1 || parts > 0x7fffffffLL || (dtype != tk::kF32 && dtype != tk::kBF16)) {
    return (int)cudaErrorInvalidValue;
  }
  p = {};
  p.q = q; p.out = out; p.k_cache = k_cache; p.v_cache = v_cache; p.history = history;
  p.n_rows = n_rows; p.n_groups = n_groups; p.max_members = max_members; p.n_q_heads = n_q_heads; p.n_kv_heads = n_kv_heads;
  p.d = head_dim; p.dv = v_dim; p.page_size = page_size; p.num_pages = num_pages;
  p.n_shared = n_shared; p.n_own = n_own; p.n_parts = n_shared + n_own;
  return 0;
}

static bool on_tensor_cores(const tk::SharedParams& p, int dtype) { return dtype == tk::kBF16 && tk::shared_tc_takes(p); }

TK_API long long tk_attention_shared_scratch(const void* q, void* out, const void* k_cache, const void* v_cache, const unsigned char* history,
                                             int n_rows, int n_groups, int max_members, int n_q_heads, int n_kv_heads, int head_dim, int v_dim,
                                             int page_size, int num_pages, int n_shared, int n_own, int dtype) {
  tk::SharedParams p;
  if (shared_params(p, q, out, k_cache, v_cache, n_rows, n_groups, max_members, n_q_heads, n_kv_heads, head_dim, v_dim, page_size, num_pages,
                    n_shared, n_own, history, dtype) != 0) {
    return -1;
  }
  if (on_tensor_cores(p, dtype)) return tk::shared_tc_scratch(p, tk::device_sm_count());
  const long long parts = (long long)n_rows * n_q_heads * p.n_parts;
  return (parts * v_dim + 1) / 2 * 2 + 2 * parts;
}

TK_API int tk_attention_shared(const void* q, void* out, const void* k_cache, const void* v_cache, const int* group_start,
                               const int* prefix_slot, const int* prefix_len, const int* positions, const int* req_slot,
                               const int* block_table, const unsigned char* history, const float* sinks, float* scratch,
                               int* err, int n_rows, int n_groups, int max_members, int n_q_heads, int n_kv_heads, int head_dim,
                               int v_dim, int page_size, int max_pages, int num_pages, int max_slots, int history_ld,
                               int window, int n_shared, int n_own, float scale, float softcap, int dtype,
                               cudaStream_t stream) {
  if (n_rows <= 0 || n_groups <= 0) return 0;
  tk::SharedParams p;
  const int bad = shared_params(p, q, out, k_cache, v_cache, n_rows, n_groups, max_members, n_q_heads, n_kv_heads, head_dim, v_dim, page_size,
                                num_pages, n_shared, n_own, history, dtype);
  if (bad != 0) return bad;
  if (max_slots < 1 || max_pages < 1 || (history != nullptr && history_ld < 1) || ((uintptr_t)scratch & 31) != 0) return (int)cudaErrorInvalidValue;
  p.group_start = group_start; p.prefix_slot = prefix_slot; p.prefix_len = prefix_len; p.positions = positions; p.req_slot = req_slot;
  p.block_table = block_table; p.sinks = sinks; p.err = err; p.scratch = scratch;
  p.max_pages = max_pages; p.max_slots = max_slots; p.history_ld = history_ld; p.window = window;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.cap_log2 = softcap > 0.0f ? softcap * 1.4426950408889634f : 0.0f;
  p.inv_cap = softcap > 0.0f ? scale / softcap : 0.0f;
  if (on_tensor_cores(p, dtype)) return tk::launch_shared_tc(p, tk::device_sm_count(), stream);
  const long long parts = (long long)n_rows * n_q_heads * p.n_parts;
  p.part_o = scratch;
  p.part_ml = scratch + (parts * v_dim + 1) / 2 * 2;
  const uintptr_t mask = dtype == tk::kF32 ? 15 : 7;
  p.wide_k = head_dim % 4 == 0 && (((uintptr_t)q | (uintptr_t)k_cache) & mask) == 0;
  p.wide_v = v_dim % 4 == 0 && ((uintptr_t)v_cache & mask) == 0;
  const int e = dtype == tk::kF32 ? tk::launch_general<float>(p, stream) : tk::launch_general<__nv_bfloat16>(p, stream);
  if (e != 0) return e;
  return dtype == tk::kF32 ? tk::launch_merge<float>(p, stream) : tk::launch_merge<__nv_bfloat16>(p, stream);
}
