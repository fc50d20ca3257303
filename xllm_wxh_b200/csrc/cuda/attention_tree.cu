// Attention of a tree of drafted tokens over a paged cache: o_i = sum_j softmax_j(scale q_i . k_j) v_j over the cached keys ahead of the
// tree and over those of the sequence's own rows whose bit is set in row i's words (its ancestors and itself).
//
// Both kernels make one pass over the keys with a running maximum and sum.
#include <atomic>
#include <type_traits>

#include "attention_tc.cuh"
#include "tree_api.h"
#include "vec8.cuh"

namespace xl_at {
using namespace xl;

struct Params {
  const void* q;                  // [T, n_q, D], pitches in elements
  const void* k_cache;            // [slots, n_kv, D]
  const void* v_cache;
  void* out;                      // [T, n_q * D]
  const int *q_cu, *kv_lens, *block_tables, *token_seq, *positions;
  const unsigned long long* tree; // [T, words]
  int T, B, max_blocks, block_size, n_q, n_kv, D, words;
  long q_row, q_head, num_slots;
  float scale;
  int window;                     // > 0: keys at positions above (row's position - window)
};

constexpr int BKV = 64;          // keys of a tile of the tensor-core kernel; the first tile starts at a multiple
struct Seq {
  int q_start, n, kv_len, base, kv_begin, row_tiles, key_tiles;
};
__device__ __forceinline__ Seq load_seq(const Params& p, int s, int per_item) {
  Seq q;
  q.q_start = max(p.q_cu[s], 0);
  q.n = min(p.q_cu[s + 1], p.T) - q.q_start;
  q.kv_len = int(min(long(p.kv_lens[s]), long(p.max_blocks) * p.block_size));
  q.base = max(q.kv_len - q.n, 0);
  q.kv_begin = p.window > 0 ? max(0, q.base - p.window + 1) / BKV * BKV : 0;
  q.row_tiles = q.n > 0 && q.kv_len > 0 ? (q.n + per_item - 1) / per_item : 0;
  q.key_tiles = (q.kv_len - q.kv_begin + BKV - 1) / BKV;
  return q;
}

// Position of row t of the sequence for the window.  It counts as one of the sequence's rows', the nearest: which tiles the window opens,
// cuts and leaves out goes by base and n alone, so a position outside would open or lose keys by the tile that they lie in.
__device__ __forceinline__ int row_position(const Params& p, const Seq& q, int t) {
  return min(max(p.positions[t], q.base), q.base + q.n - 1);
}

// whether row t belongs to no sequence, or to one without keys: its output is zero
__device__ __forceinline__ bool row_is_idle(const Params& p, int t) {
  const int s = p.token_seq[t];
  return s < 0 || s >= p.B || t < p.q_cu[s] || t >= p.q_cu[s + 1] || p.kv_lens[s] <= 0 || p.max_blocks == 0;
}

// keys of the tile at kv0 that row t (at position pos) sees
__device__ __forceinline__ uint64_t seen_keys(const Params& p, const Seq& q, int t, int pos, int kv0) {
  const int c = q.base - kv0;
  uint64_t see = c >= 64 ? ~0ull : c > 0 ? (1ull << c) - 1 : 0;
  if (p.window > 0) {
    const int lo = pos - p.window + 1 - kv0;
    see = lo >= 64 ? 0 : lo > 0 ? see >> lo << lo : see;
  }
  if (c < 64) {
    const unsigned long long* words = p.tree + size_t(t) * p.words;
    uint64_t bits;
    if (c >= 0) {
      bits = words[0] << c;
    } else {
      const int i = (-c) >> 6, sh = (-c) & 63;
      bits = i < p.words ? words[i] >> sh : 0;
      if (sh && i + 1 < p.words) bits |= words[i + 1] << (64 - sh);
    }
    const int end = q.kv_len - kv0;
    if (end < 64) bits = end > 0 ? bits & ((1ull << end) - 1) : 0;
    if (p.window > 0 && pos - p.window >= q.base)
      for (uint64_t todo = bits; todo; todo &= todo - 1) {
        const int k = __ffsll(todo) - 1;
        // (as `row_position` would say: the border lies between the first and the last row's)
        if (p.positions[q.q_start + kv0 + k - q.base] <= pos - p.window) bits &= ~(1ull << k);
      }
    see |= bits;
  }
  return see;
}

// ---------------------------------------------------------------- fp32-pipe kernel
// fp32, and bf16 of the sizes that the tensor-core kernel does not take.  One CTA = (sequence, 32 rows of a key head's query heads times
// nodes, key head, part of the keys): 32 keys at a time go through shared memory as fp32, a thread computes 4 rows x 2 keys of the
// scores and 4 rows x 4 NC columns of the sums, so that the multiply-adds bound it rather than shared memory; parts of the keys
// keep the SMs busy when there are few rows, and are joined by a second kernel.  Scores, weights and sums stay fp32; only the result is
// rounded.  8 trees of 3 to 12 rows, 14 query heads for 2 key heads of 64 columns, up to 2000 keys in fp32: 28 us (floor of the bytes 1.4),
// four tiles of keys a CTA (parts of 128 keys), of which loads through the table, latency of 4 x 2 products and the join (4 us) are all of it;
// of the 768 CTAs that the bounds ask for, about 270 have rows and keys.
constexpr int SR = 32, SK = 32, kSimtThreads = 128, kMaxParts = 64;
template <int NC> struct SimtSmem {
  static constexpr int DP = 64 * NC, PITCH = DP + 4;         // 16 rows apart lie in 16 banks
  float q[SR][PITCH], k[SK][PITCH], v[SK][DP], p[SR][SK + 4];
  long slot[2][SK];                                          // of this tile and the next; -1: behind the last key
};

template <typename T, int NC>
__global__ void __launch_bounds__(kSimtThreads) attention_tree_simt_kernel(const Params p, int row_tiles, int splits, int part_keys, float* ws_o,
                                                                           float2* ws_ml) {
  extern __shared__ __align__(16) uint8_t smem[];
  grid_dep_launch();
  using S = SimtSmem<NC>;
  S& sm = *reinterpret_cast<S*>(smem);
  const int tid = threadIdx.x, ty = tid >> 4, tx = tid & 15, D = p.D;
  const int seq = blockIdx.x / row_tiles, row0 = (blockIdx.x - seq * row_tiles) * SR, kvh = blockIdx.y, G = p.n_q / p.n_kv;
  const Seq q = load_seq(p, seq, 1);
  if (splits == 1 && kvh == 0) {                             // a row at a time: a vote of the warp costs the rest registers and 3 us
    for (long i = blockIdx.x; i < p.T; i += gridDim.x)
      if (row_is_idle(p, int(i)))
        for (int c = tid; c < p.n_q * D; c += kSimtThreads) from_f32(static_cast<T*>(p.out) + i * p.n_q * D + c, 0.f);
  }
  if (row0 >= q.n * G || q.kv_len <= 0) return;
  const int first = q.kv_begin + int(blockIdx.z) * part_keys, last = int(blockIdx.z) == splits - 1 ? q.kv_len : min(q.kv_len, first + part_keys);
  if (first >= last) return;
  // rows of this thread: 4 ty + i
  int t[4], pos[4];
  bool valid[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int node = (row0 + 4 * ty + i) / G;
    valid[i] = node < q.n;
    t[i] = q.q_start + (valid[i] ? node : 0);
    pos[i] = p.window > 0 ? row_position(p, q, t[i]) : 0;
  }
  const bool vectors = D % 8 == 0 && (reinterpret_cast<uintptr_t>(p.k_cache) | reinterpret_cast<uintptr_t>(p.v_cache)) % 16 == 0;
  const float scale = p.scale * 1.4426950408889634f;         // scores in the log2 domain
  if (D < S::DP) {                                           // columns past D stay zero
    for (int i = tid; i < 32 * S::DP; i += kSimtThreads) {
      const int r = i / S::DP, c = i % S::DP;
      if (c >= D) sm.q[r][c] = sm.k[r][c] = sm.v[r][c] = 0.f;
    }
  }
  const bool q_vectors = D % 8 == 0 && reinterpret_cast<uintptr_t>(p.q) % 16 == 0 && (p.q_row | p.q_head) % 8 == 0;
  const int q_step = q_vectors ? 8 : 1, q_per = D / q_step;
#pragma unroll 2
  for (int i = tid; i < SR * q_per; i += kSimtThreads) {
    const int r = i / q_per, c = (i - r * q_per) * q_step, node = (row0 + r) / G, h = kvh * G + row0 + r - node * G;
    const T* from = static_cast<const T*>(p.q) + (q.q_start + (node < q.n ? node : 0)) * p.q_row + h * p.q_head + c;
    if (q_vectors) {
      float f[8];
      load8(from, f);
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = node < q.n ? f[e] * scale : 0.f;
      store8(&sm.q[r][c], f);
    } else {
      sm.q[r][c] = node < q.n ? to_f32(*from) * scale : 0.f;
    }
  }
  const int* bt = p.block_tables + size_t(seq) * p.max_blocks;
  float m[4], l[4], o[4][4 * NC];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int c = 0; c < 4 * NC; ++c) o[i][c] = 0.f;
  }
  auto find_slots = [&](int tile) {
    const int key = first + tile * SK + tid;
    if (tid >= SK) return;
    const int blk = key / p.block_size;
    const long slot = key < last && blk < p.max_blocks ? long(bt[blk]) * p.block_size + key % p.block_size : -1;
    sm.slot[tile & 1][tid] = slot < p.num_slots ? slot : -1;
  };
  // Eight columns of a key and its values at a time.  Small heads: the next tile's wait in registers while this one is computed.
  constexpr bool kAhead = NC <= 2;
  constexpr int kItems = kAhead ? SK * S::DP / 8 / kSimtThreads : 1;
  const int per = D / 8;
  float ka[kItems][8], va[kItems][8];
  auto fetch = [&](int tile, int i, float (&a)[8], float (&b)[8]) {
    const int j = i / per, c = (i - j * per) * 8;
#pragma unroll
    for (int e = 0; e < 8; ++e) a[e] = b[e] = 0.f;
    if (j < SK && sm.slot[tile & 1][j] >= 0) {
      const size_t at = (size_t(sm.slot[tile & 1][j]) * p.n_kv + kvh) * D + c;
      load8(static_cast<const T*>(p.k_cache) + at, a);
      load8(static_cast<const T*>(p.v_cache) + at, b);
    }
  };
  auto keep = [&](int i, const float (&a)[8], const float (&b)[8]) {
    const int j = i / per, c = (i - j * per) * 8;
    if (j >= SK) return;
    store8(&sm.k[j][c], a);
    store8(&sm.v[j][c], b);
  };
  find_slots(0);
  find_slots(1);
  __syncthreads();
  if (kAhead && vectors)
#pragma unroll
    for (int n = 0; n < kItems; ++n) fetch(0, tid + n * kSimtThreads, ka[n], va[n]);
  int tile = 0;
  for (int kv0 = first; kv0 < last; kv0 += SK, ++tile) {
    __syncthreads();
    if (kAhead && vectors) {
#pragma unroll
      for (int n = 0; n < kItems; ++n) keep(tid + n * kSimtThreads, ka[n], va[n]);
    } else if (vectors) {
      for (int i = tid; i < SK * per; i += kSimtThreads) {
        fetch(tile, i, ka[0], va[0]);
        keep(i, ka[0], va[0]);
      }
    } else {
      for (int i = tid; i < SK * D; i += kSimtThreads) {
        const int j = i / D, c = i - j * D;
        const long slot = sm.slot[tile & 1][j];
        const size_t at = (size_t(max(slot, 0l)) * p.n_kv + kvh) * D + c;
        sm.k[j][c] = slot >= 0 ? to_f32(static_cast<const T*>(p.k_cache)[at]) : 0.f;
        sm.v[j][c] = slot >= 0 ? to_f32(static_cast<const T*>(p.v_cache)[at]) : 0.f;
      }
    }
    __syncthreads();
    find_slots(tile + 2);                                    // (in the place of this tile's, which is loaded)
    if (kAhead && vectors && kv0 + SK < last)
#pragma unroll
      for (int n = 0; n < kItems; ++n) fetch(tile + 1, tid + n * kSimtThreads, ka[n], va[n]);
    // scores of rows 4 ty + i and keys tx, tx + 16
    float s[4][2] = {};
#pragma unroll 8
    for (int c = 0; c < S::DP; c += 4) {
      const float4 k0 = *reinterpret_cast<const float4*>(&sm.k[tx][c]), k1 = *reinterpret_cast<const float4*>(&sm.k[tx + 16][c]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 w = *reinterpret_cast<const float4*>(&sm.q[4 * ty + i][c]);
        s[i][0] = fmaf(w.x, k0.x, fmaf(w.y, k0.y, fmaf(w.z, k0.z, fmaf(w.w, k0.w, s[i][0]))));
        s[i][1] = fmaf(w.x, k1.x, fmaf(w.y, k1.y, fmaf(w.z, k1.z, fmaf(w.w, k1.w, s[i][1]))));
      }
    }
    const bool partly = kv0 + SK > min(q.base, last) || (p.window > 0 && kv0 < q.base + q.n - p.window);
    uint32_t see[4] = {~0u, ~0u, ~0u, ~0u};
    if (partly) {
      const uint32_t there = last - kv0 >= SK ? ~0u : (1u << (last - kv0)) - 1;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        see[i] = valid[i] ? uint32_t(seen_keys(p, q, t[i], pos[i], kv0)) & there : 0u;
        if (!(see[i] >> tx & 1u)) s[i][0] = -INFINITY;
        if (!(see[i] >> (tx + 16) & 1u)) s[i][1] = -INFINITY;
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float mx = fmaxf(s[i][0], s[i][1]);
#pragma unroll
      for (int off = 8; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
      const float m_new = fmaxf(m[i], mx), ref = m_new == -INFINITY ? 0.f : m_new;
      const float alpha = m[i] == -INFINITY ? 1.f : fast_exp2(m[i] - ref);
      const float e0 = see[i] >> tx & 1u ? fast_exp2(s[i][0] - ref) : 0.f, e1 = see[i] >> (tx + 16) & 1u ? fast_exp2(s[i][1] - ref) : 0.f;
      float sum = e0 + e1;
#pragma unroll
      for (int off = 8; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
      m[i] = m_new;
      l[i] = l[i] * alpha + sum;
#pragma unroll
      for (int c = 0; c < 4 * NC; ++c) o[i][c] *= alpha;
      sm.p[4 * ty + i][tx] = e0;
      sm.p[4 * ty + i][tx + 16] = e1;
    }
    __syncwarp();                                            // a half-warp's weights are its own
    auto sums = [&](auto masked) {
#pragma unroll 2
      for (int j = 0; j < SK; j += 4) {
        float w[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) *reinterpret_cast<float4*>(w[i]) = *reinterpret_cast<const float4*>(&sm.p[4 * ty + i][j]);
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int c = 0; c < NC; ++c) {
            const float4 v = *reinterpret_cast<const float4*>(&sm.v[j + k][64 * c + 4 * tx]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              if (decltype(masked)::value && !(see[i] >> (j + k) & 1u)) continue;       // whatever stands there
              o[i][4 * c] = fmaf(w[i][k], v.x, o[i][4 * c]);
              o[i][4 * c + 1] = fmaf(w[i][k], v.y, o[i][4 * c + 1]);
              o[i][4 * c + 2] = fmaf(w[i][k], v.z, o[i][4 * c + 2]);
              o[i][4 * c + 3] = fmaf(w[i][k], v.w, o[i][4 * c + 3]);
            }
          }
      }
    };
    if (partly) sums(std::true_type{});
    else sums(std::false_type{});
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (!valid[i]) continue;
    const size_t row = size_t(t[i]) * p.n_q + kvh * G + (row0 + 4 * ty + i) % G;
    if (splits > 1) {
      const size_t at = size_t(blockIdx.z) * p.T * p.n_q + row;
      if (tx == 0) ws_ml[at] = make_float2(m[i], l[i]);
#pragma unroll
      for (int c = 0; c < 4 * NC; ++c) {
        const int col = 64 * (c >> 2) + 4 * tx + (c & 3);
        if (col < D) ws_o[at * D + col] = o[i][c];
      }
    } else {
      const float inv = l[i] != 0.f ? 1.f / l[i] : 0.f;      // a row that sees nothing: zeros
#pragma unroll
      for (int c = 0; c < 4 * NC; ++c) {
        const int col = 64 * (c >> 2) + 4 * tx + (c & 3);
        if (col < D) from_f32(static_cast<T*>(p.out) + row * D + col, o[i][c] * inv);
      }
    }
  }
}

// One warp per (row, query head): joins the parts of its keys, and clears rows of no sequence.
template <typename T>
__global__ void __launch_bounds__(128) attention_tree_join_kernel(const Params p, int splits, int part_keys, const float* ws_o, const float2* ws_ml) {
  grid_dep_wait();
  const long row = blockIdx.x * 4l + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= long(p.T) * p.n_q) return;
  const int t = int(row / p.n_q), seq = p.token_seq[t];
  T* out = static_cast<T*>(p.out) + size_t(row) * p.D;
  int parts = 0;
  if (seq >= 0 && seq < p.B) {
    const Seq q = load_seq(p, seq, 1);
    if (t >= q.q_start && t < q.q_start + q.n && q.kv_len > 0) parts = min(splits, (q.kv_len - q.kv_begin + part_keys - 1) / part_keys);
  }
  // a lane's share of the (at most kMaxParts) parts
  const size_t pitch = size_t(p.T) * p.n_q;
  float2 ml[kMaxParts / 32];
  float m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < kMaxParts / 32; ++i) {
    ml[i] = lane + 32 * i < parts ? ws_ml[(lane + 32 * i) * pitch + row] : make_float2(-INFINITY, 0.f);
    m = fmaxf(m, ml[i].x);
  }
  m = warp_max(m);
#pragma unroll
  for (int i = 0; i < kMaxParts / 32; ++i) {
    // a part whose row saw nothing has no weight, unless its scores were not numbers; one far below the others still makes the sums
    // NaN if its own are no numbers, as within a part
    const float w = ml[i].x == -INFINITY ? (ml[i].y != 0.f ? 1.f : 0.f) : fast_exp2(ml[i].x - m);
    l += w * ml[i].y;
    ml[i].x = w;
  }
  l = warp_sum(l);
  const float inv = l != 0.f ? 1.f / l : 0.f;
  // four columns a lane; the two halves of the warp take the parts in turn, eight loads at a time
  for (int c0 = 0; c0 < p.D; c0 += 64) {
    const int c = c0 + 4 * (lane & 15);
    float o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
    for (int k = 0; k < parts; k += 2) {
      const int mine = k + (lane >> 4);
      float w = __shfl_sync(0xffffffffu, ml[0].x, mine & 31);
#pragma unroll
      for (int i = 1; i < kMaxParts / 32; ++i) {
        const float v = __shfl_sync(0xffffffffu, ml[i].x, mine & 31);
        if (mine >> 5 == i) w = v;
      }
      const float* from = ws_o + (mine * pitch + row) * p.D + c;
      float x[4] = {0.f, 0.f, 0.f, 0.f};
      if (mine < parts && p.D % 4 == 0 && c < p.D) {
        *reinterpret_cast<float4*>(x) = *reinterpret_cast<const float4*>(from);
      } else if (mine < parts) {
        for (int e = 0; e < 4; ++e)
          if (c + e < p.D) x[e] = from[e];
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (mine < parts) o[e] = fmaf(w, x[e], o[e]);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      o[e] += __shfl_xor_sync(0xffffffffu, o[e], 16);
      if (lane < 16 && c + e < p.D) from_f32(out + c + e, o[e] * inv);
    }
  }
}

// floats of the parts' maxima and sums, so that what follows lies on 16 bytes
inline long ml_floats(int splits, int T, int n_q) { return (2l * splits * T * n_q + 3) / 4 * 4; }

template <typename T, int NC>
int launch_simt(const Params& p, int row_tiles, int splits, int part_keys, float* ws, cudaStream_t s) {
  auto* kernel = attention_tree_simt_kernel<T, NC>;
  static std::atomic<bool> ready[64];                        // per device
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -1;
  if (!ready[dev].load(std::memory_order_acquire)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(sizeof(SimtSmem<NC>))) != cudaSuccess) return -1;
    ready[dev].store(true, std::memory_order_release);
  }
  float2* ml = reinterpret_cast<float2*>(ws);
  float* o = ws + ml_floats(splits, p.T, p.n_q);
  if (p.B > 0) {
    kernel<<<dim3(p.B * row_tiles, p.n_kv, splits), kSimtThreads, sizeof(SimtSmem<NC>), s>>>(p, row_tiles, splits, part_keys, o, ml);
    if (cudaGetLastError() != cudaSuccess) return -1;
  }
  if (p.B > 0 && splits == 1) return 0;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned((long(p.T) * p.n_q + 3) / 4));
  cfg.blockDim = dim3(128);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.B > 0 ? 1 : 0;
  const float* from = o;
  const float2* from_ml = ml;
  return cudaLaunchKernelEx(&cfg, attention_tree_join_kernel<T>, p, splits, part_keys, from, from_ml) == cudaSuccess ? 0 : -1;
}
template <typename T>
int launch_simt(const Params& p, int row_tiles, int splits, int part_keys, float* ws, cudaStream_t s) {
  if (p.D <= 64) return launch_simt<T, 1>(p, row_tiles, splits, part_keys, ws, s);
  if (p.D <= 128) return launch_simt<T, 2>(p, row_tiles, splits, part_keys, ws, s);
  if (p.D <= 256) return launch_simt<T, 4>(p, row_tiles, splits, part_keys, ws, s);
  return launch_simt<T, 8>(p, row_tiles, splits, part_keys, ws, s);
}

// ---------------------------------------------------------------- tensor-core kernel
// bf16, up to 128 columns a head.  A key head's query heads times a tree's nodes are the rows of one product: 128 rows (TMEM lanes) take in
// 128 / G nodes of G heads each, so that a key is read once for all of them (two row tiles: for 256 rows).  Reading K and V bounds the
// kernel up to about 256 rows; above, exponentials and products do.
//
//   work      : the key tiles (64 keys) of every item (rows, key head, sequence) one behind the other, each item with kItemCost tiles'
//               worth of work ahead of it, cut into equal stretches, one per CTA (one CTA per SM): ragged lengths leave no SM idle.
//               Sequences run fastest, so that the CTAs of a sequence's further rows go through the same keys at the same time and
//               find them in L2.  A stretch begins and ends anywhere; the at most two pieces of it that are not whole items leave fp32 partials (sums,
//               maximum, denominator) that the merge kernel joins.
//   warp 0    : TMA producer - says what the next piece is, fetches its query rows (box: 64 columns x G heads x nodes), then a ring of units
//               in the order of use, each 64 tokens of K or of V through the block table;
//   warps 1, 2: MMA issuers  - each for one softmax group: S = Q K^T (128 x 64 x D, fp32 in TMEM, two buffers a group), O += P V with P
//               from TMEM (one issuer's waits would leave the tensor pipe idle);
//   warps 3-6 and 7-10: two softmax groups, one row per thread: running maximum and sum in the log2 domain, P as bf16 over the
//               scores it comes from, O rescaled only when the maximum grew by more than 2^8.
//               An item of two row tiles gives each group one; otherwise the groups take the key tiles in turn for the same rows, each
//               with its own O, and join at the end of a piece: a single group could not keep up with memory.
// A warp's products run in the order of their issue, so S of a tile may overwrite P of the tile two before as soon as that one's P V is issued.
//
// Measured (single calls on two GPUs; in a long row of calls the power cap lowers the clocks: 238 and 981 us for the first two):
//   64 trees of 9 to 32 rows, 32 query heads for 8 of 128 columns, contexts of 300 to 8192: 196 and 205 us, 1.14 GB at 5.8 TB/s, 0.88 of a copy's
//   bandwidth; 16 trees of 64 rows, 64 heads for 8, contexts of 16000 to 32704: 830 and 855 us, 985 TFLOP/s, 0.60 of cuBLAS:
//   per 64 keys of 256 rows the products take 1280 cycles (S is issued at 48 cycles a step of 16, where N = 128 would take 64 for twice
//   the columns), the exponentials 1024, a softmax thread's own chain for a tile about 2200, in which code that is rarely run (masks,
//   values that are not finite, rescaling) is kept out of the way and the piece's numbers in registers (8 % more otherwise);
//   one tree of 16 rows over 1000 keys: 13.9 us, of which launch, first loads and the join are 9.
//   Earlier forms at 64 x 32 rows: fp32 pipe 97 ms, P through shared memory 273 us, without pieces published by the producer 215 us.
//   Tried without gain: the next tile's scores fetched while a tile's weights are stored (8 to 28 % slower, with registers moved from the
//   other warps to the softmax warps or without), two threads a row, every eighth exponential as a polynomial, turns between the groups,
//   144 CTAs by head.
//
// Roundings to bf16: P (2^-8 of each weight at most, with the sum taken of the unrounded ones in fp32) because the products take bf16, and the result.
//
// Masks: keys ahead of the tree are seen by all rows (within the window), the tree's by the row's words; only tiles that hold either
// border look at them.  There, values behind the last row are cleared, and values that are not finite are taken out of the tile and
// added to the rows that do see them, so that whatever stands in a masked place reaches no other row.
// Every wait on an mbarrier is bounded; on expiry the kernel records a status code and leaves once its copies and products in flight have ended.
// The softmax warps meet at named barriers, which know no bound: they decide together whether to leave, and go on without waiting until then.
constexpr int BQ = 128;
constexpr int kTcThreads = 352;
constexpr int Q_SLAB = BQ * 128, KV_SLAB = BKV * 128;
constexpr int kMaxUnits = 20, kPieces = 8;
constexpr int kItemCost = 3;     // (16 rows, 1000 keys: 13.8 us; 2: 14.3, 5: 14.0; long contexts alike)

__device__ __forceinline__ int item_work(const Seq& q) { return q.key_tiles + kItemCost; }
// of a key head's items of row tile `plane`
__device__ __forceinline__ int plane_work(const Seq& q, int plane) { return q.row_tiles > plane ? item_work(q) : 0; }
struct Piece {
  Seq q;
  int seq, head, node0, j0, nt;            // node0: first node of the piece's rows; its key tiles j0 .. j0 + nt - 1 (0: no more pieces)
  int pair, whole, slot;                   // pair: two row tiles; slot: of its partials
  __device__ __forceinline__ int key0(int j) const { return q.kv_begin + (j0 + j) * BKV; }
  __device__ __forceinline__ int tile_number(int kv0) const {        // of such a tile among its item's
    return kv0 + BKV > q.base ? min(8 + (kv0 - q.base / BKV * BKV) / BKV, 15) : min((kv0 - q.kv_begin) / BKV, 7);
  }
};
struct TcBarriers {
  uint64_t full[kMaxUnits], empty[kMaxUnits];
  uint64_t q_full, q_empty, info[kPieces], drained[2];
  // [group][buffer]: softmax may be two tiles ahead of the products and need not look at each one's end, so that a barrier a group
  // would be a phase off
  uint64_t s_full[2][2], p_full[2][2], pv_done[2][2];
  uint32_t tmem_base;
  int work[kTcThreads], most[kTcThreads];                    // of a thread's sequences: work of the first row tiles, row tiles at most
  int any_bad[4][2];                                         // [piece & 3][group]
  uint32_t bad[4][2][16][2];                                 // [piece & 3][group][tile][key]: keys whose values are not all finite
  float2 ml[2][BQ];
  Piece piece[kPieces];
};
template <int QS, int NQ> struct Cfg {                       // NQ: row tiles of an item at most
  static constexpr int DV = 64 * QS;                         // padded columns
  static constexpr int Q_BYTES = QS * Q_SLAB, UNIT = QS * KV_SLAB;
  static constexpr int kFit = (227 * 1024 - int(sizeof(TcBarriers)) - NQ * Q_BYTES) / UNIT;
  static constexpr int U = kFit < kMaxUnits ? kFit : kMaxUnits;
  static constexpr int kSmem = NQ * Q_BYTES + U * UNIT + int(sizeof(TcBarriers));
  static constexpr int kRows = NQ * BQ;
  static_assert(U >= 6 && kSmem <= 227 * 1024, "the units up to a tile's values fit the ring");
};

struct TcParams {
  Params a;
  int group, nodes;             // query heads per key head, nodes of one row tile
  int box_tokens, block_shift, min_work;   // block_shift: -1 where the block size is no power of two
  float scale_log2;
  float4* ws_o;                 // [2 * CTA + which][D / 4][rows]
  float2* ws_ml;                // [2 * CTA + which][rows]: (maximum in the log2 domain, sum)
  int* ws_desc;                 // [CTA][8]
  int* status;
};
enum { DESC_MERGE, DESC_FIRST, DESC_SLOT, DESC_START, DESC_NODES, DESC_HEAD };   // of the item that ends in a CTA's first piece

// S of a tile is issued `lag` tiles ahead of P V: by one tile of the same group.  Unit (within its piece) of the keys and values of tile j.
__device__ __forceinline__ int k_unit(int j, int lag) { return j < lag ? j : 2 * j - lag; }
__device__ __forceinline__ int v_unit(int j, int lag, int nt) { return j + lag < nt ? 2 * j + lag + 1 : nt + j; }

__device__ __forceinline__ bool not_finite(uint32_t pair) {
  return (pair & 0x7F800000u) == 0x7F800000u || (pair & 0x7F80u) == 0x7F80u;
}
__device__ __forceinline__ uint32_t finite_part(uint32_t pair) {
  return ((pair & 0x7F800000u) == 0x7F800000u ? 0 : pair & 0xFFFF0000u) | ((pair & 0x7F80u) == 0x7F80u ? 0 : pair & 0xFFFFu);
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
// D[tmem] (+)= A[tmem] * B[smem desc]: row i of A in lane i, two bf16 per column
__device__ __forceinline__ void tc_mma_f16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(tmem_d), "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
      : "memory");
}

template <int QS, int NQ>
__global__ void __launch_bounds__(kTcThreads, 1)
attention_tree_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                         const TcParams p) {
  using C = Cfg<QS, NQ>;
  constexpr int U = C::U, UNIT = C::UNIT, DV = C::DV;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* sQ = smem;
  uint8_t* ring = sQ + NQ * C::Q_BYTES;
  TcBarriers* bars = reinterpret_cast<TcBarriers*>(ring + U * UNIT);
  const Params& a = p.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  grid_dep_launch();                                         // the merge kernel may take its place; it waits for this one's end
  if (smem_u32(smem) & 1023u) {
    if (tid == 0) {
      atomicExch(p.status, XL_ERR_BOUNDS);
      p.ws_desc[blockIdx.x * 8 + DESC_MERGE] = 0;
    }
    return;
  }
  // ------------------------------------------------------------ this CTA's stretch of the work
  const int per_item = NQ * p.nodes;
  const int share = (a.B + kTcThreads - 1) / kTcThreads;
  const int s0 = min(tid * share, a.B), s1 = min(s0 + share, a.B);
  int mine = 0, most = 1;
  for (int s = s0; s < s1; ++s) {
    const Seq q = load_seq(a, s, per_item);
    mine += plane_work(q, 0);
    most = max(most, q.row_tiles);
  }
  bars->work[tid] = mine;
  bars->most[tid] = most;
  if (warp == 0 && lane < 3) prefetch_tmap(lane == 0 ? &tmQ : lane == 1 ? &tmK : &tmV);
  if (tid == 64) {
    for (int u = 0; u < U; ++u) {
      mbar_init(&bars->full[u], 1);
      mbar_init(&bars->empty[u], 2);
    }
    mbar_init(&bars->q_full, 1);
    mbar_init(&bars->q_empty, 2);
    for (int i = 0; i < kPieces; ++i) mbar_init(&bars->info[i], 1);
    for (int g = 0; g < 2; ++g) {
      mbar_init(&bars->drained[g], 1);
      for (int b = 0; b < 2; ++b) {
        mbar_init(&bars->s_full[g][b], 1);
        mbar_init(&bars->p_full[g][b], 4);
        mbar_init(&bars->pv_done[g][b], 1);
      }
    }
    mbar_fence_init();
  }
  if (tid < 4 * 2 * 16 * 2) (&bars->bad[0][0][0][0])[tid] = 0;
  if (tid < 8) bars->any_bad[tid >> 1][tid & 1] = 0;
  if (warp == 1) {
    tmem_alloc(&bars->tmem_base, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem_base;                     // group g: S / P buffers at g * 256 + {0, 64}, O at g * 256 + 128

  if (warp == 0) {
    // ---------------------------------------------------------- TMA producer (whole warp: lanes share the boxes)
    const int boxes = BKV / p.box_tokens, per_unit = boxes * QS;       // boxes of a 64-column slab; at most 8 x 2
    const int slab = lane / boxes, bx = lane % boxes;
    // the sum of the work; this CTA's stretch [w0, w1) of it; the item that it begins in.  (Only this warp needs them.)
    auto inclusive = [&](int v) {
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int w = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += w;
      }
      return v;
    };
    constexpr int kEach = kTcThreads / 32;
    int sum = 0, planes = 1;
#pragma unroll 1
    for (int i = 0; i < kEach; ++i) {
      sum += bars->work[lane * kEach + i];
      planes = max(planes, bars->most[lane * kEach + i]);
    }
    planes = __reduce_max_sync(0xffffffffu, planes);
    int upto = inclusive(sum), per_head = __shfl_sync(0xffffffffu, upto, 31), total = per_head * a.n_kv;
    auto plane_sum = [&](int plane) {
      int v = 0;
      for (int s = lane; s < a.B; s += 32) v += plane_work(load_seq(a, s, per_item), plane);
      return __reduce_add_sync(0xffffffffu, v);
    };
    for (int i = 1; i < planes; ++i) total += plane_sum(i) * a.n_kv;
    int ctas = max(1, min(int(gridDim.x), total / p.min_work));
    // row tiles side by side, if that leaves no more than a thirtieth of the SMs idle
    const int lanes = a.n_kv * planes;
    if (planes > 1 && ctas % lanes * 30 <= ctas && ctas >= lanes) ctas -= ctas % lanes;
    const int per_cta = total / ctas, longer = total - per_cta * ctas;   // the first `longer` stretches have one more
    auto begin = [&](int c) { return c * per_cta + min(c, longer); };
    const int w0 = begin(min(int(blockIdx.x), ctas)), w1 = begin(min(int(blockIdx.x) + 1, ctas));
    const bool busy = w0 < w1;
    Piece x;
    int w = 0, plane = 0;                                              // w: work ahead of the current item
    if (busy) {
      while (w0 >= w + per_head * a.n_kv) {                            // the row tile
        w += per_head * a.n_kv;
        per_head = plane_sum(++plane);
      }
      x.head = (w0 - w) / per_head;
      w += x.head * per_head;
      int s = 0, at = 0;                                               // a sequence at or ahead of the one, the work ahead of it
      if (plane == 0) {                                                // by the threads' sums
        const uint32_t here = __ballot_sync(0xffffffffu, upto - sum <= w0 - w && w0 - w < upto);
        const int l = __ffs(here) - 1;
        at = __shfl_sync(0xffffffffu, upto - sum, l);
        int t = l * kEach;
        while (at + bars->work[t] <= w0 - w) at += bars->work[t++];
        s = t * share;
      }
      while (true) {
        x.seq = s;
        x.q = load_seq(a, s, per_item);
        const int n = plane_work(x.q, plane);
        if (w0 - w < at + n) break;
        at += n;
        ++s;
      }
      w += at;
    }
    bool ok = true;
    int st = 0, phase = 0, count = 0, units = 0, q_sent = 0;           // (q_sent: of lane 0)
    while (ok && busy && w < w1) {
      // the part of the item that lies in the stretch
      x.j0 = max(w0 - w - kItemCost, 0);
      x.nt = min(w1 - w - kItemCost, x.q.key_tiles) - x.j0;
      if (x.nt > 0) {
        x.node0 = plane * per_item;
        x.pair = NQ == 2 && x.q.n - x.node0 > p.nodes;
        x.whole = x.nt == x.q.key_tiles;
        x.slot = 2 * blockIdx.x + (count > 0);
        // a lane's place in tile j; the values of a tile are fetched `lag` tiles after its keys, from the same places
        const int* bt = a.block_tables + size_t(x.seq) * a.max_blocks;
        auto block_of = [&](int j) {
          const int tok = x.key0(j) + bx * p.box_tokens;
          return min(p.block_shift >= 0 ? tok >> p.block_shift : tok / a.block_size, a.max_blocks - 1);
        };
        auto place = [&](int j, int entry) {
          const int tok = x.key0(j) + bx * p.box_tokens;
          const long slot = long(entry) * a.block_size + (p.block_shift >= 0 ? tok & (a.block_size - 1) : tok % a.block_size);
          return slot < 0 || slot + p.box_tokens > a.num_slots ? 0 : int(slot);  // places behind the last row
        };
        int next = lane < per_unit ? bt[block_of(0)] : 0, held0 = 0, held1 = 0;  // (looked up one tile ahead)
        const int info = count % kPieces;
        if (lane == 0) {
          ok = mbar_wait(&bars->q_empty, (count & 1) ^ 1);
          if (ok) {
            bars->piece[info] = x;
            mbar_arrive(&bars->info[info]);
            const int tiles = x.pair ? 2 : 1;
            ++q_sent;
            mbar_arrive_expect_tx(&bars->q_full, uint32_t(tiles * QS * 128 * p.group * p.nodes));
            for (int h = 0; h < tiles; ++h)
#pragma unroll
              for (int sl = 0; sl < QS; ++sl)
                tma_load_3d(sQ + h * C::Q_BYTES + sl * Q_SLAB, &tmQ, &bars->q_full, sl * 64, x.head * p.group, x.q.q_start + x.node0 + h * p.nodes);
          }
        }
        ok = __shfl_sync(0xffffffffu, ok, 0);
        auto unit = [&](const CUtensorMap* map, int slot) {
          if (lane == 0) {
            ok = mbar_wait(&bars->empty[st], phase ^ 1);
            if (ok) mbar_arrive_expect_tx(&bars->full[st], UNIT);
          }
          ok = __shfl_sync(0xffffffffu, ok, 0);
          units += ok;
          if (ok && lane < per_unit)
            tma_load_3d(ring + st * UNIT + slab * KV_SLAB + bx * p.box_tokens * 128, map, &bars->full[st], slab * 64, x.head, slot);
          if (++st == U) {
            st = 0;
            phase ^= 1;
          }
        };
        const int lag = x.pair ? 1 : 2;
        for (int j = 0; ok && j < x.nt + lag; ++j) {
          const int slot = place(j, next);
          if (j < x.nt) {
            if (lane < per_unit && j + 1 < x.nt) next = bt[block_of(j + 1)];
            unit(&tmK, slot);
          }
          if (ok && j >= lag && j - lag < x.nt) unit(&tmV, lag == 1 ? held0 : held1);
          held1 = held0;
          held0 = slot;
        }
        if (count == 0 && lane == 0) {
          int* d = p.ws_desc + blockIdx.x * 8;
          const bool merge = x.j0 > 0 && x.j0 + x.nt == x.q.key_tiles;
          d[DESC_MERGE] = merge;
          if (merge) {
            const int tile0 = w + kItemCost, even = (per_cta + 1) * longer;     // the item's first tile; work of the longer stretches
            const int first = tile0 < even ? tile0 / (per_cta + 1) : longer + (tile0 - even) / per_cta;
            d[DESC_FIRST] = first;
            d[DESC_SLOT] = 2 * first + (begin(first) < w ? 1 : 0);
            d[DESC_START] = x.q.q_start + x.node0;
            d[DESC_NODES] = min(per_item, x.q.n - x.node0);
            d[DESC_HEAD] = x.head;
          }
        }
        ++count;
      }
      w += item_work(x.q);
      if (w < w1) {
        do {
          if (++x.seq == a.B) {
            x.seq = 0;
            if (++x.head == a.n_kv) {
              x.head = 0;
              ++plane;
            }
          }
          x.q = load_seq(a, x.seq, per_item);
        } while (x.q.row_tiles <= plane);
      }
    }
    if (lane == 0) {
      bars->piece[count % kPieces].nt = 0;
      mbar_arrive(&bars->info[count % kPieces]);
      if (count == 0) p.ws_desc[blockIdx.x * 8 + DESC_MERGE] = 0;
      if (!ok) atomicExch(p.status, XL_ERR_WAIT_EMPTY);
      // no copy may land behind the CTA's end (all have, unless a wait ran out)
      ok = q_sent == 0 || mbar_wait(&bars->q_full, (q_sent - 1) & 1);
      for (int u = max(units - U, 0); ok && u < units; ++u) ok = mbar_wait(&bars->full[u % U], (u / U) & 1);
    }
  } else if (warp <= 2) {
    // ---------------------------------------------------------- MMA issuer of group g
    if (elect_one_sync()) {
      const int g = warp - 1;
      const uint32_t idesc_s = umma_idesc_f16(BQ, BKV, 1), idesc_o = umma_idesc_f16(BQ, DV, 1) | (1u << 16);   // V is MN-major
      // descriptors count in units of 16 bytes: a step along a tile is an addition
      const uint64_t q_desc = umma_desc_sw128(smem_u32(sQ), 0), k_desc = umma_desc_sw128(smem_u32(ring), 0);
      const uint64_t v_desc = umma_desc_sw128_mn(smem_u32(ring), KV_SLAB, 1024);
      const uint32_t t_s = tmem + g * 256, t_o = t_s + 128;
      bool ok = true;
      int st = 0, phase = 0, s_count = 0, p_count = 0;
      // both issuers go through all units; one that has no use for a unit lets go of it as soon as it is there
      auto next = [&] {
        if (++st == U) {
          st = 0;
          phase ^= 1;
        }
      };
      for (int count = 0; ok; ++count) {
        const int info = count % kPieces;
        if (!(ok = mbar_wait(&bars->info[info], (count / kPieces) & 1))) break;
        const int nt = bars->piece[info].nt;
        if (nt == 0) break;
        const bool pair = NQ == 2 && bars->piece[info].pair;
        const int lag = pair ? 1 : 2;
        const uint64_t q0 = q_desc + (pair ? g * C::Q_BYTES / 16 : 0);
        if (!(ok = mbar_wait(&bars->q_full, count & 1))) break;
        for (int j = 0; j < nt + lag; ++j) {
          if (j < nt) {
            if (!(ok = mbar_wait(&bars->full[st], phase))) break;
            if (pair || (j & 1) == g) {
              tc_fence_after();
              const uint64_t k0 = k_desc + st * (UNIT / 16);
              const int b = s_count++ & 1;
#pragma unroll
              for (int k = 0; k < DV / 16; ++k)
                tc_mma_f16(t_s + b * 64, q0 + (k >> 2) * (Q_SLAB / 16) + (k & 3) * 2, k0 + (k >> 2) * (KV_SLAB / 16) + (k & 3) * 2, idesc_s, k != 0);
              tc_commit(&bars->s_full[g][b]);
              tc_commit(&bars->empty[st]);
            } else {
              mbar_arrive(&bars->empty[st]);
            }
            if (j == nt - 1) tc_commit(&bars->q_empty);
            next();
          }
          if (j >= lag && j - lag < nt) {
            const int i = j - lag;
            if (!(ok = mbar_wait(&bars->full[st], phase))) break;
            if (pair || (i & 1) == g) {
              const uint64_t v0 = v_desc + st * (UNIT / 16);
              const int b = p_count & 1;
              if (!(ok = mbar_wait(&bars->p_full[g][b], (p_count >> 1) & 1))) break;
              ++p_count;
              tc_fence_after();
#pragma unroll
              for (int k = 0; k < BKV / 16; ++k)
                tc_mma_f16_ts(t_o, t_s + b * 64 + k * 8, v0 + k * (2048 / 16), idesc_o, ((pair ? i : i >> 1) | k) != 0);
              tc_commit(&bars->pv_done[g][b]);
              tc_commit(&bars->empty[st]);
            } else {
              mbar_arrive(&bars->empty[st]);
            }
            next();
          }
        }
      }
      if (!ok) atomicExch(p.status, XL_ERR_WAIT_FULL);
      tc_commit(&bars->drained[g]);                                    // nor a product run on memory that has been given back
      mbar_wait(&bars->drained[g], 0);
    }
  } else {
    // ---------------------------------------------------------- softmax, one row per thread
    const int g = (warp - 3) >> 2, quarter = warp & 3, r = quarter * 32 + lane;
    const int gt = (warp - 3 - 4 * g) * 32 + lane;                     // thread of the group
    const uint32_t t_lane = tmem + (uint32_t(quarter * 32) << 16), t_s = t_lane + g * 256, t_o = t_s + 128;
    const int node = r / p.group, head_in = r - node * p.group;
    const float sc = p.scale_log2;
    auto group_sync = [&] { asm volatile("bar.sync %0, 128;" ::"r"(2 + g) : "memory"); };
    auto both_sync = [] { asm volatile("bar.sync 1, 256;" ::: "memory"); };
    auto both_agree = [](bool mine) {                                  // whether it is true of all threads of the two groups
      uint32_t all;
      asm volatile(
          "{\n\t.reg .pred P, Q;\n\t"
          "setp.ne.u32 P, %1, 0;\n\t"
          "barrier.cta.red.and.pred Q, 1, 256, P;\n\t"
          "selp.u32 %0, 1, 0, Q;\n\t}"
          : "=r"(all)
          : "r"(uint32_t(mine))
          : "memory");
      return all != 0;
    };
    // idle rows: every thread looks at one of this CTA's share, a warp clears what its lanes found
    for (long t0 = blockIdx.x; t0 < a.T; t0 += 256l * gridDim.x) {
      const long t = t0 + (tid - 96l) * gridDim.x;
      for (uint32_t todo = __ballot_sync(0xffffffffu, t < a.T && row_is_idle(a, int(t))); todo; todo &= todo - 1) {
        const long idle = __shfl_sync(0xffffffffu, t, __ffs(todo) - 1);
        for (int c = tid & 31; c < a.n_q * a.D / 8; c += 32)
          reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(a.out) + idle * a.n_q * a.D)[c] = make_uint4(0, 0, 0, 0);
      }
    }
    bool ok = true;
    int u0 = 0, count = 0;                                             // units ahead of the piece; tiles of this group so far
    for (int piece = 0;; ++piece) {
      // Both groups have read the last piece's O and maxima.  (And a warp that left alone would be missed at the barriers by those that saw
      // the piece.)
      if (!both_agree(mbar_wait(&bars->info[piece % kPieces], (piece / kPieces) & 1))) {
        ok = false;
        break;
      }
      tc_fence_after();
      const Piece& x = bars->piece[piece % kPieces];
      const int nt = x.nt;
      if (nt == 0) break;
      const bool pair = NQ == 2 && x.pair;
      const int lag = pair ? 1 : 2, owner = pair ? 0 : g;              // owner: whose flags hold for this group's keys
      const int my_node = x.node0 + (pair ? g * p.nodes : 0) + node;
      const bool valid = node < p.nodes && my_node < x.q.n;
      const bool warp_valid = __any_sync(0xffffffffu, valid);
      const int t = x.q.q_start + (valid ? my_node : 0);
      const int pos = valid && a.window > 0 ? row_position(a, x.q, t) : 0;
      float m_ref = -INFINITY, l_run = 0.f;
      int done = 0;                                                    // tiles of this group in this piece
      // tiles up to the window's border and from the tree's first on are seen in part (in registers: the piece itself is read again each time)
      const int first_key = x.key0(0);
      const int ahead = a.window > 0 ? (x.q.base + x.q.n - a.window - first_key + BKV - 1) / BKV : 0, behind = (x.q.base - first_key) / BKV;
      // (a group whose wait ran out goes on without waiting, so that the others still meet it at the barriers)
      for (int j = pair ? 0 : g; j < nt; j += pair ? 1 : 2, ++done, ++count) {
        const int b = count & 1, kv0 = first_key + j * BKV;
        if (ok && !__all_sync(0xffffffffu, mbar_wait(&bars->s_full[g][b], (count >> 1) & 1))) ok = false;
        tc_fence_after();
        const bool partly = j < ahead || j >= behind;
        if (warp_valid) {
          uint32_t s0[32], s1[32];
          tmem_ld_32x32(t_s + b * 64, s0);
          tmem_ld_32x32(t_s + b * 64 + 32, s1);
          tc_wait_ld();
          float v[64];
#pragma unroll
          for (int c = 0; c < 32; ++c) {
            v[c] = __uint_as_float(s0[c]);
            v[32 + c] = __uint_as_float(s1[c]);
          }
          if (__builtin_expect(partly, 0)) {
            const uint64_t see = valid ? seen_keys(a, x.q, t, pos, kv0) : 0;
            const uint32_t lo = uint32_t(see), hi = uint32_t(see >> 32);
#pragma unroll
            for (int c = 0; c < 32; ++c) {
              if (!(lo >> c & 1u)) v[c] = -INFINITY;
              if (!(hi >> c & 1u)) v[32 + c] = -INFINITY;
            }
          }
          float mx4[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) mx4[i] = fmaxf(v[i], v[i + 4]);
#pragma unroll
          for (int c = 8; c < 64; c += 8)
#pragma unroll
            for (int i = 0; i < 4; ++i) mx4[i] = max3(mx4[i], v[c + i], v[c + 4 + i]);
          const float mx = fmaxf(max3(mx4[0], mx4[1], mx4[2]), mx4[3]);
          // the reference stays unless the scaled maximum grew by more than 8: P stays below 2^8
          const bool had = m_ref != -INFINITY;
          const bool grow = (mx - m_ref) * sc > 8.f || (!had && mx != -INFINITY);
          const float m_new = grow ? mx : m_ref;
          const bool rescale = grow && had;
          const float alpha = rescale ? fast_exp2((m_ref - m_new) * sc) : 1.f;
          m_ref = m_new;
          const float mneg = m_ref == -INFINITY ? 0.f : -m_ref * sc;
          const uint64_t sc2 = pack2(sc, sc), mneg2 = pack2(mneg, mneg);
          uint64_t sum2[4] = {0, 0, 0, 0};
          uint32_t pk[32];
#pragma unroll
          for (int c = 0; c < 64; c += 2) {
            const float2 z = unpack2(fma2(pack2(v[c], v[c + 1]), sc2, mneg2));
            const float e0 = fast_exp2(z.x), e1 = fast_exp2(z.y);
            sum2[(c >> 1) & 3] = add2(sum2[(c >> 1) & 3], pack2(e0, e1));
            pk[c >> 1] = pack_bf16x2(e0, e1);
          }
          const float2 sum = unpack2(add2(add2(sum2[0], sum2[1]), add2(sum2[2], sum2[3])));
          l_run = l_run * alpha + (sum.x + sum.y);
          tmem_st_32x32(t_s + b * 64, pk);
          if (__builtin_expect(done > 0 && __any_sync(0xffffffffu, rescale), 0)) {
            // O is at rest once P V of this group's tile before has run
            if (ok && !__all_sync(0xffffffffu, mbar_wait(&bars->pv_done[g][(count - 1) & 1], ((count - 1) >> 1) & 1))) ok = false;
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < DV; c += 32) {
              uint32_t o[32];
              tmem_ld_32x32(t_o + c, o);
              tc_wait_ld();
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
              tmem_st_32x32(t_o + c, o);
            }
          }
          tc_wait_st();
        }
        if (__builtin_expect(partly && owner == g, 0)) {
          // two threads look at the values of one key
          const int u = u0 + v_unit(j, lag, nt), st = u % U, key = gt >> 1;
          if (ok && !__all_sync(0xffffffffu, mbar_wait(&bars->full[st], (u / U) & 1))) ok = false;
          uint4* row = reinterpret_cast<uint4*>(ring + st * UNIT + key * 128 + (gt & 1) * 64);
          bool bad = false;
#pragma unroll
          for (int i = 0; i < 4 * QS; ++i) {
            uint4* at = row + (i >> 2) * (KV_SLAB / 16) + (i & 3);
            if (kv0 + key >= x.q.kv_len) {
              *at = make_uint4(0, 0, 0, 0);
            } else {
              const uint4 v = *at;
              if (not_finite(v.x) || not_finite(v.y) || not_finite(v.z) || not_finite(v.w)) {
                *at = make_uint4(finite_part(v.x), finite_part(v.y), finite_part(v.z), finite_part(v.w));
                bad = true;
              }
            }
          }
          if (bad) {
            atomicOr(&bars->bad[piece & 3][g][x.tile_number(kv0)][key >> 5], 1u << (key & 31));
            bars->any_bad[piece & 3][g] = 1;
          }
          fence_proxy_async_smem();
          if (!pair) group_sync();
        }
        if (__builtin_expect(partly && pair, 0)) both_sync();                               // the other group's products wait for the values too
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->p_full[g][b]);
      }
      if (ok && done > 0 && !__all_sync(0xffffffffu, mbar_wait(&bars->pv_done[g][(count - 1) & 1], ((count - 1) >> 1) & 1))) ok = false;
      tc_fence_after();
      u0 += 2 * nt;
      // ------------------------------------------------ end of a piece
      if (ok && done > 0 && warp_valid && bars->any_bad[piece & 3][owner]) {
        // values that are not finite join the rows that see them
        for (int i = 0; i < 16 * 64; ++i) {
          const int tile = i >> 6, k = i & 63;
          if (!(bars->bad[piece & 3][owner][tile][k >> 5] >> (k & 31) & 1u)) continue;
          const int kv0 = tile >= 8 ? x.q.base / BKV * BKV + (tile - 8) * BKV : x.q.kv_begin + tile * BKV, key = kv0 + k;
          const bool see = valid && (seen_keys(a, x.q, t, pos, kv0) >> k & 1ull);
          const long slot = long(a.block_tables[size_t(x.seq) * a.max_blocks + key / a.block_size]) * a.block_size + key % a.block_size;
          if (slot < 0 || slot >= a.num_slots) continue;
          const __nv_bfloat16* from = static_cast<const __nv_bfloat16*>(a.v_cache) + (size_t(slot) * a.n_kv + x.head) * a.D;
          for (int c = 0; c < DV; c += 32) {
            uint32_t o[32];
            tmem_ld_32x32(t_o + c, o);
            tc_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              const float f = c + e < a.D ? __bfloat162float(from[c + e]) : 0.f;
              if (see && !(fabsf(f) <= 3.4e38f)) o[e] = __float_as_uint(__uint_as_float(o[e]) + f);
            }
            tmem_st_32x32(t_o + c, o);
          }
          tc_wait_st();
        }
      }
      const float m_log2 = m_ref == -INFINITY ? -INFINITY : m_ref * sc;
      // weights of the two groups' sums (two row tiles: its own alone), and the columns that this group stores
      float wa = 1.f, wb = 0.f, m_all = m_log2, l_all = l_run;
      int c_lo = 0, c_hi = DV;
      uint32_t t_oa = t_o;
      if (!pair) {
        bars->ml[g][r] = make_float2(m_log2, l_run);
        tc_fence_before();
        both_sync();
        tc_fence_after();
        const float2 fa = bars->ml[0][r], fb = bars->ml[1][r];
        m_all = fmaxf(fa.x, fb.x);
        // a group whose row saw nothing has nothing to add, unless its scores were not numbers
        wa = fa.x == -INFINITY ? (fa.y != fa.y ? fa.y : 0.f) : fast_exp2(fa.x - m_all);
        wb = fb.x == -INFINITY ? (fb.y != fb.y ? fb.y : 0.f) : fast_exp2(fb.x - m_all);
        l_all = fa.y * wa + fb.y * wb;
        t_oa = t_lane + 128;
        c_lo = g * (DV / 2);
        c_hi = c_lo + DV / 2;
      }
      if (ok && warp_valid) {
        const bool whole = x.whole, two = !pair && nt > 1;
        const int ws_row = pair ? g * BQ + r : r;
        const float inv = l_all != 0.f ? 1.f / l_all : 0.f;            // a row that sees nothing: zeros
        __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(a.out) + size_t(t) * (size_t(a.n_q) * a.D) + (x.head * p.group + head_in) * a.D;
        float4* wo = p.ws_o + size_t(x.slot) * (DV / 4) * C::kRows + ws_row;
        const float fa = whole ? wa * inv : wa, fb = whole ? wb * inv : wb;
#pragma unroll 1
        for (int c = c_lo; c < c_hi; c += 32) {
          uint32_t oa[32], ob[32];
          tmem_ld_32x32(t_oa + c, oa);
          if (two) tmem_ld_32x32(t_lane + 256 + 128 + c, ob);
          tc_wait_ld();
          float f[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) f[i] = __uint_as_float(oa[i]) * fa;
          if (two) {
#pragma unroll
            for (int i = 0; i < 32; ++i) f[i] = fmaf(__uint_as_float(ob[i]), fb, f[i]);
          }
          if (valid && whole) {
#pragma unroll
            for (int i = 0; i < 32; i += 8)
              if (c + i < a.D)
                *reinterpret_cast<uint4*>(dst + c + i) = make_uint4(pack_bf16x2(f[i], f[i + 1]), pack_bf16x2(f[i + 2], f[i + 3]),
                                                                    pack_bf16x2(f[i + 4], f[i + 5]), pack_bf16x2(f[i + 6], f[i + 7]));
          } else if (valid) {
#pragma unroll
            for (int i = 0; i < 32; i += 4) wo[size_t((c + i) / 4) * C::kRows] = make_float4(f[i], f[i + 1], f[i + 2], f[i + 3]);
          }
        }
        if (valid && !whole && (pair || g == 0)) p.ws_ml[size_t(x.slot) * C::kRows + ws_row] = make_float2(m_all, l_all);
      }
      // the next piece's flags were last read three pieces ago
      if (bars->any_bad[(piece + 1) & 3][g]) {
        if (gt < 32) (&bars->bad[(piece + 1) & 3][g][0][0])[gt] = 0;
        group_sync();
        if (gt == 0) bars->any_bad[(piece + 1) & 3][g] = 0;
        group_sync();
      }
      tc_fence_before();
    }
    if (!ok && lane == 0) atomicExch(p.status, XL_ERR_WAIT_TMEM_FULL);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, 512);
}

// Joins the partials of the item that ends in CTA blockIdx.x's first piece: o = sum 2^(m_i - m) o_i / sum 2^(m_i - m) l_i.
// Bound by the latency of the loads (from L2), so four parts at a time are fetched together and 16 CTAs share an item: behind a step of 16
// rows and 1000 keys it takes 3.4 us, 1.3 of them the launch (4.3 with 8 CTAs an item; eight parts at a time or 32 CTAs gain nothing more).
template <int QS, int NQ>
__global__ void __launch_bounds__(128) attention_tree_merge_kernel(const TcParams p) {
  using C = Cfg<QS, NQ>;
  const Params& a = p.a;
  grid_dep_wait();
  const int4 d0 = __ldcg(reinterpret_cast<const int4*>(p.ws_desc) + blockIdx.x * 2), d1 = __ldcg(reinterpret_cast<const int4*>(p.ws_desc) + blockIdx.x * 2 + 1);
  if (!d0.x) return;
  const int first = d0.y, slot0 = d0.z, start = d0.w, rows = d1.x * p.group, head = d1.y;
  const int parts = int(blockIdx.x) - first + 1, items = rows * (a.D / 4);
  for (int i = blockIdx.y * 128 + threadIdx.x; i < items; i += gridDim.y * 128) {
    const int row = i % rows, c = i / rows;                            // neighbours share a column group: partials are read side by side
    const int node = row / p.group, h = row - node * p.group;
    const int tile = NQ == 2 && node >= p.nodes ? 1 : 0;
    const int ws_row = tile * BQ + (node - tile * p.nodes) * p.group + h;
    float m = -INFINITY, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k0 = 0; k0 < parts; k0 += 4) {
      float2 ml[4];
      float4 v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const size_t slot = k0 + k == 0 ? slot0 : 2 * (first + k0 + k);
        ml[k] = make_float2(-INFINITY, 0.f);
        if (k0 + k < parts) {
          ml[k] = __ldcg(&p.ws_ml[slot * C::kRows + ws_row]);
          v[k] = __ldcg(&p.ws_o[(slot * (C::DV / 4) + c) * C::kRows + ws_row]);
        }
      }
      const float m_new = fmaxf(fmaxf(m, fmaxf(ml[0].x, ml[1].x)), fmaxf(ml[2].x, ml[3].x));
      const float w0 = m == -INFINITY ? 1.f : fast_exp2(m - m_new);
      l *= w0;
      o.x *= w0; o.y *= w0; o.z *= w0; o.w *= w0;
      m = m_new;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (ml[k].x == -INFINITY && ml[k].y == 0.f) continue;          // sees no key of that part
        const float w = ml[k].x == -INFINITY ? 1.f : fast_exp2(ml[k].x - m);
        l += w * ml[k].y;
        o.x += w * v[k].x; o.y += w * v[k].y; o.z += w * v[k].z; o.w += w * v[k].w;
      }
    }
    const float inv = l != 0.f ? 1.f / l : 0.f;
    __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(a.out) + size_t(start + node) * (size_t(a.n_q) * a.D) + (head * p.group + h) * a.D + 4 * c;
    *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16x2(o.x * inv, o.y * inv), pack_bf16x2(o.z * inv, o.w * inv));
  }
}

template <int QS, int NQ>
int launch_tc(const TcParams& p, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, int ctas, cudaStream_t s) {
  using C = Cfg<QS, NQ>;
  auto* kernel = attention_tree_tc_kernel<QS, NQ>;
  static std::atomic<bool> ready[64];                                  // per device
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -1;
  if (!ready[dev].load(std::memory_order_acquire)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem) != cudaSuccess) return -1;
    ready[dev].store(true, std::memory_order_release);
  }
  kernel<<<ctas, kTcThreads, C::kSmem, s>>>(q, k, v, p);
  if (cudaGetLastError() != cudaSuccess) return -1;
  if (ctas == 1) return 0;                                             // nothing was split
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(ctas, 16);                                        // an item over 16 CTAs: short chains of loads
  cfg.blockDim = dim3(128);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, attention_tree_merge_kernel<QS, NQ>, p) == cudaSuccess ? 0 : -1;
}

}  // namespace xl_at

static bool tc_serves(const void* q, const void* k, const void* v, int block_size, int n_q, int n_kv, int D, long q_row, long q_head,
                      float scale, int f32) {
  const int box = block_size & -block_size;                 // largest power of two that divides it
  return !f32 && D % 8 == 0 && D <= 128 && n_q / n_kv <= xl_at::BQ && box >= 8 && scale > 0.f && q_row % 8 == 0 && q_head % 8 == 0 && q_head > 0 &&
         q_row % q_head == 0 && (reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) % 16 == 0;
}

// Whether the places of the caches and the work of a step (key tiles of all its items) count in 32 bits, and there are any.
static bool tc_counts(int T, int B, int max_blocks, int block_size, int num_blocks, int n_q, int n_kv) {
  const long places = long(num_blocks) * block_size;
  const double items = (double(B) + double(T) / (xl_at::BQ / (n_q / n_kv))) * n_kv;       // row tiles at most, of as many nodes as fit 128 rows
  return B > 0 && max_blocks > 0 && places > 0 && places <= 0x7fffffffl &&
         items * (double(max_blocks) * block_size / xl_at::BKV + 2 + xl_at::kItemCost) <= double(0x7fffffff);
}

// How the fp32-pipe kernel is launched: row tiles of a sequence, parts of the keys, keys of a part.  max_q, max_kv: bounds of a sequence's rows
// and keys.
struct SimtPlan { int row_tiles, splits, part_keys; };
static SimtPlan simt_plan(int B, int n_q, int n_kv, int max_q, int max_kv, int sms) {
  SimtPlan s{};
  s.row_tiles = max(1, int((long(max_q) * (n_q / n_kv) + xl_at::SR - 1) / xl_at::SR));
  const long units = long(s.row_tiles) * n_kv * max(B, 1);
  // parts of a multiple of 64 keys, up to eight CTAs an SM (its registers hold two or three at a time) by the bounds, as if every
  // sequence had max_q rows and max_kv keys
  s.splits = int(max(1l, min(min(long(max_kv + 63) / 64, long(xl_at::kMaxParts)), 8l * sms / units)));
  max_kv = min(max(max_kv, 1), 0x7fffffff - 4096);
  s.part_keys = (max_kv + s.splits - 1) / s.splits;
  s.part_keys = (s.part_keys + 63) / 64 * 64;
  s.splits = (max_kv + s.part_keys - 1) / s.part_keys;
  return s;
}

// CTAs of the tensor-core kernel: one per SM, fewer where there are fewer key tiles (of 64 keys for up to 128 rows).
static int tc_ctas(int T, int B, int n_q, int n_kv, int max_kv, int sms) {
  return int(max(1l, min(long(sms), (long(max_kv) / 64 + 1) * n_kv * (B + long(T) * (n_q / n_kv) / xl_at::BQ))));
}

XL_API long xl_attention_tree_workspace(int T, int B, int max_blocks, int block_size, int num_blocks, int n_q, int n_kv, int D, int plain, int max_q,
                                        int max_kv, int* tc) {
  *tc = tc_serves(nullptr, nullptr, nullptr, block_size, n_q, n_kv, D, 8, 8, 1.f, plain) &&
        tc_counts(T, B, max_blocks, block_size, num_blocks, n_q, n_kv);
  const int sms = xl_host::sm_count();
  if (*tc) {
    const long rows = long(max_q) * (n_q / n_kv) > xl_at::BQ ? 256 : 128, DV = (D + 63) / 64 * 64, ctas = tc_ctas(T, B, n_q, n_kv, max_kv, sms);
    return 2l * ctas * rows * (DV * 4 + 8) + 32l * ctas;
  }
  const SimtPlan s = simt_plan(B, n_q, n_kv, max_q, max_kv, sms);
  return s.splits > 1 ? 4 * (xl_at::ml_floats(s.splits, T, n_q) + long(s.splits) * T * n_q * D) : 0;
}

XL_API int xl_attention_tree(const void* q, const void* k_cache, const void* v_cache, void* out, const void* q_cu, const void* kv_lens,
                             const void* block_tables, const void* token_seq, const void* positions, const void* tree, int T, int B,
                             int max_blocks, int block_size, int num_blocks, int n_q, int n_kv, int D, int words, long q_row, long q_head,
                             float scale, int window, int f32, int max_q, int max_kv, int tc, void* workspace, long workspace_bytes, void* stream) {
  using namespace xl_at;
  if (T < 0 || B < 0 || n_kv < 1 || n_q < 1 || n_q % n_kv || D < 1 || D > 512 || words < 1 || block_size < 1 || max_blocks < 0) return -2;
  if (T == 0) return 0;
  int served = 0;
  if (workspace_bytes < xl_attention_tree_workspace(T, B, max_blocks, block_size, num_blocks, n_q, n_kv, D, f32 || !tc, max_q, max_kv, &served)) return -2;
  const int sms = xl_host::sm_count();
  Params p{};
  p.q = q; p.k_cache = k_cache; p.v_cache = v_cache; p.out = out;
  p.q_cu = static_cast<const int*>(q_cu);
  p.kv_lens = static_cast<const int*>(kv_lens);
  p.block_tables = static_cast<const int*>(block_tables);
  p.token_seq = static_cast<const int*>(token_seq);
  p.positions = static_cast<const int*>(positions);
  p.tree = static_cast<const unsigned long long*>(tree);
  p.T = T; p.B = B; p.max_blocks = max_blocks; p.block_size = block_size; p.n_q = n_q; p.n_kv = n_kv; p.D = D; p.words = words;
  p.q_row = q_row; p.q_head = q_head;
  p.num_slots = long(num_blocks) * block_size;
  p.scale = scale; p.window = window;
  auto s = static_cast<cudaStream_t>(stream);
  if (tc) {
    if (!workspace || !tc_counts(T, B, max_blocks, block_size, num_blocks, n_q, n_kv) || !tc_serves(q, k_cache, v_cache, block_size, n_q, n_kv, D, q_row, q_head, scale, f32)) return -2;
    const bool pair = long(max_q) * (n_q / n_kv) > BQ;
    const int ctas = tc_ctas(T, B, n_q, n_kv, max_kv, sms);
    TcParams t{};
    t.a = p;
    t.group = n_q / n_kv;
    t.nodes = BQ / t.group;
    t.box_tokens = min(block_size & -block_size, BKV);
    t.block_shift = (block_size & (block_size - 1)) == 0 ? __builtin_ctz(block_size) : -1;
    t.min_work = 3;                                         // (16 rows, 1000 keys: 13.8 us; 2: 13.9, 5: 14.7)
    t.scale_log2 = scale * 1.4426950408889634f;
    const int rows = pair ? 256 : 128, DV = (D + 63) / 64 * 64;
    t.ws_o = static_cast<float4*>(workspace);
    t.ws_ml = reinterpret_cast<float2*>(t.ws_o + size_t(2) * ctas * rows * (DV / 4));
    t.ws_desc = reinterpret_cast<int*>(t.ws_ml + size_t(2) * ctas * rows);          // on 16 bytes: rows is even
    t.status = xl_host::status_word();
    CUtensorMap mq, mk, mv;
    const uint64_t q_dims[3] = {uint64_t(D), uint64_t(n_q), uint64_t(T)}, q_strides[2] = {uint64_t(q_head) * 2, uint64_t(q_row) * 2};
    const uint32_t q_box[3] = {64, uint32_t(t.group), uint32_t(t.nodes)};
    const uint64_t kv_dims[3] = {uint64_t(D), uint64_t(n_kv), uint64_t(p.num_slots)}, kv_strides[2] = {uint64_t(D) * 2, uint64_t(n_kv) * D * 2};
    const uint32_t kv_box[3] = {64, 1, uint32_t(t.box_tokens)};
    const auto bf16 = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    const auto swz = CU_TENSOR_MAP_SWIZZLE_128B;
    if (xl_host::encode_tiled(&mq, bf16, 3, q, q_dims, q_strides, q_box, swz) != CUDA_SUCCESS ||
        xl_host::encode_tiled(&mk, bf16, 3, k_cache, kv_dims, kv_strides, kv_box, swz) != CUDA_SUCCESS ||
        xl_host::encode_tiled(&mv, bf16, 3, v_cache, kv_dims, kv_strides, kv_box, swz) != CUDA_SUCCESS)
      return -4;
    if (D <= 64) return pair ? launch_tc<1, 2>(t, mq, mk, mv, ctas, s) : launch_tc<1, 1>(t, mq, mk, mv, ctas, s);
    return pair ? launch_tc<2, 2>(t, mq, mk, mv, ctas, s) : launch_tc<2, 1>(t, mq, mk, mv, ctas, s);
  }
  const SimtPlan plan = simt_plan(B, n_q, n_kv, max_q, max_kv, sms);
  if (long(B) * plan.row_tiles > 0x7fffffffl || n_kv > 65535 || long(T) * n_q > 0x7fffffffl) return -2;
  auto* ws = static_cast<float*>(workspace);
  return f32 ? launch_simt<float>(p, plan.row_tiles, plan.splits, plan.part_keys, ws, s)
             : launch_simt<__nv_bfloat16>(p, plan.row_tiles, plan.splits, plan.part_keys, ws, s);
}
