// Attention of a tree of drafted tokens over a paged cache: o_i = sum_j softmax_j(scale q_i . k_j) v_j over the cached keys ahead of the
// tree and over those of the sequence's own rows whose bit is set in row i's words (its ancestors and itself).
//
// The fp32-pipe kernel serves every type and size: one warp per (row, query head), 32 keys at a time, one key per lane for the scores, then
// one slice of the value columns per lane for the weighted sum, with a running maximum and sum.
#include "vec8.cuh"

namespace xl_at {
using namespace xl;

constexpr int kMaxCols = 16;      // value columns per lane: up to 512 columns

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

template <typename T>
__global__ void __launch_bounds__(128) attention_tree_simt_kernel(const Params p) {
  extern __shared__ float s_q[];                 // one query vector per warp
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long item = blockIdx.x * 4l + warp;
  if (item >= long(p.T) * p.n_q) return;
  const int t = int(item / p.n_q), h = int(item % p.n_q);
  T* out = static_cast<T*>(p.out) + (size_t(t) * p.n_q + h) * p.D;
  const int seq = p.token_seq[t];
  const int start = seq >= 0 && seq < p.B ? p.q_cu[seq] : 0, n = seq >= 0 && seq < p.B ? p.q_cu[seq + 1] - start : 0;
  if (t < start || t >= start + n) {             // a row of no sequence
    for (int c = lane; c < p.D; c += 32) from_f32(out + c, 0.f);
    return;
  }
  const int kv_len = p.kv_lens[seq], base = max(kv_len - n, 0), pos = p.positions[t];
  const int kvh = h / (p.n_q / p.n_kv);
  const int* bt = p.block_tables + size_t(seq) * p.max_blocks;
  const unsigned long long* words = p.tree + size_t(t) * p.words;
  const T* qrow = static_cast<const T*>(p.q) + t * p.q_row + h * p.q_head;
  float* q = s_q + warp * p.D;
  for (int i = lane; i < p.D; i += 32) q[i] = to_f32(qrow[i]) * p.scale;
  __syncwarp();
  float m = -INFINITY, l = 0.f;
  float acc[kMaxCols];
#pragma unroll
  for (int c = 0; c < kMaxCols; ++c) acc[c] = 0.f;
  const int lo = p.window > 0 ? max(0, pos - p.window + 1) : 0;
  for (int first = min(lo, base) / 32 * 32; first < kv_len; first += 32) {
    const int key = first + lane;
    bool see = key >= lo && key < base;
    if (key >= base && key < kv_len) {
      const int node = key - base;
      see = node < n && (node >> 6) < p.words && (words[node >> 6] >> (node & 63) & 1ull);
      if (see && p.window > 0) see = p.positions[start + node] > pos - p.window;
    }
    float s = -INFINITY;
    long slot = 0;
    if (see) {
      const int blk = key / p.block_size;
      slot = blk < p.max_blocks ? long(bt[blk]) * p.block_size + key % p.block_size : 0;
      if (slot < 0 || slot >= p.num_slots) slot = 0;
      const T* k = static_cast<const T*>(p.k_cache) + (size_t(slot) * p.n_kv + kvh) * p.D;
      float d = 0.f;
      for (int i = 0; i < p.D; ++i) d = fmaf(q[i], to_f32(k[i]), d);
      s = d;
    }
    unsigned todo = __ballot_sync(0xffffffffu, see);
    if (!todo) continue;
    const float m_new = fmaxf(m, warp_max(s));
    const float ref = m_new == -INFINITY ? 0.f : m_new;
    const float alpha = m == -INFINITY ? 0.f : expf(m - ref);
    const float w = see ? expf(s - ref) : 0.f;
    l = l * alpha + warp_sum(w);
    m = m_new;
#pragma unroll
    for (int c = 0; c < kMaxCols; ++c) acc[c] *= alpha;
    for (; todo; todo &= todo - 1) {
      const int j = __ffs(todo) - 1;
      const float wj = __shfl_sync(0xffffffffu, w, j);
      const long sj = __shfl_sync(0xffffffffu, slot, j);
      const T* v = static_cast<const T*>(p.v_cache) + (size_t(sj) * p.n_kv + kvh) * p.D;
#pragma unroll
      for (int c = 0; c < kMaxCols; ++c)
        if (c * 32 + lane < p.D) acc[c] = fmaf(wj, to_f32(v[c * 32 + lane]), acc[c]);
    }
  }
  const float inv = l != 0.f ? 1.f / l : 0.f;   // a row that sees nothing: zeros
#pragma unroll
  for (int c = 0; c < kMaxCols; ++c)
    if (c * 32 + lane < p.D) from_f32(out + c * 32 + lane, acc[c] * inv);
}

}  // namespace xl_at

XL_API int xl_attention_tree(const void* q, const void* k_cache, const void* v_cache, void* out, const void* q_cu, const void* kv_lens,
                             const void* block_tables, const void* token_seq, const void* positions, const void* tree, int T, int B,
                             int max_blocks, int block_size, int num_blocks, int n_q, int n_kv, int D, int words, long q_row, long q_head,
                             float scale, int window, int f32, void* stream) {
  using namespace xl_at;
  if (T < 0 || B < 0 || n_kv < 1 || n_q % n_kv || D < 1 || D > 32 * kMaxCols || words < 1 || block_size < 1 || max_blocks < 1) return -2;
  if (T == 0) return 0;
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
  const long items = long(T) * n_q, ctas = (items + 3) / 4;
  if (ctas > 0x7fffffffl) return -2;
  auto s = static_cast<cudaStream_t>(stream);
  if (f32) attention_tree_simt_kernel<float><<<unsigned(ctas), 128, 4 * D * sizeof(float), s>>>(p);
  else attention_tree_simt_kernel<__nv_bfloat16><<<unsigned(ctas), 128, 4 * D * sizeof(float), s>>>(p);
  return cudaGetLastError() == cudaSuccess ? 0 : -1;
}
