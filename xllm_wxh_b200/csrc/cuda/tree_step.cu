// The two ends of a step whose sequences carry trees of drafted tokens: the step's maps from the lengths on the device
// (step_rows), and the choice of the path that the target model agrees with together with the cache rows it leaves (accept_tree).
//
// Both are bound by latency for small steps and by copying for large ones (block tables; kept cache rows), so each is one launch:
// every CTA finds the little it needs of the other sequences by itself instead of waiting for a kernel that prepares it.
#include "common.cuh"
#include "tree_api.h"

namespace xl_ts {
using namespace xl;

constexpr int kTreeRows = 256;                  // rows of a sequence that can form a tree: four 64-bit words of ancestors
constexpr int kThreads = 256;

__device__ __forceinline__ long block_sum(long v, long* s) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0;
#pragma unroll
  for (int i = 0; i < kThreads / 32; ++i) v += s[i];
  return v;
}

// ---------------------------------------------------------------- step_rows
struct RowsParams {
  const int* tables;            // [pool, columns], rows table_ld apart
  const int* lens;              // [pool]
  const int* seqs;              // [B] rows of the pool (outside: no sequence)
  const int* counts;            // [B]
  const int* parents;           // [n_rows] or null
  int *positions, *slots, *token_seq, *q_cu, *kv_lens, *block_tables;
  unsigned long long* tree;     // [n_rows, words] or null
  int pool, columns, B, n_rows, max_q, max_blocks, block_size, words, per_cta, table_parts, vectors;
  long table_ld;
};

// blockIdx.y = sequence (B: the rows behind the last one); blockIdx.x = a part of `per_cta` entries of its table, or behind those a part of
// as many rows.  The table does not wait for the sum of the sequences ahead, which only the rows need.
//
// A row's slot is table[(len + i) / block] * block + (len + i) % block, its position len + its ancestors' number; its set of ancestors is
// its own bit and its parent's set, which doubling finds in log2(depth) steps.  Copying the tables' used entries bounds large steps: 1024
// trees of 32 rows with tables of 8192 columns take 12.1 us, 51 MB at 4.2 TB/s (0.64 of a copy's bandwidth; most of it stays in L2,
// and launch and first loads are 3 us of it).  Small steps are those 3 us: one tree of 8 rows 3.1 us, 256 single rows 3.2 us.
__global__ void __launch_bounds__(kThreads) step_rows_kernel(const RowsParams p) {
  __shared__ long s_sum[kThreads / 32];
  __shared__ unsigned long long s_anc[kTreeRows * 4];
  __shared__ int s_up[kTreeRows];
  const int b = blockIdx.y, tid = threadIdx.x;
  auto rows_of = [&](int i) { return unsigned(p.seqs[i]) < unsigned(p.pool) ? min(max(p.counts[i], 0), p.max_q) : 0; };

  int src = -1, mine = 0, len = 0;
  if (b < p.B) {
    src = p.seqs[b];
    mine = p.counts[b];
    if (unsigned(src) >= unsigned(p.pool)) src = -1;
    mine = src >= 0 ? min(max(mine, 0), p.max_q) : 0;
    len = src >= 0 ? max(p.lens[src], 0) : 0;
  }
  const int* from = p.tables + size_t(max(src, 0)) * p.table_ld;
  if (int(blockIdx.x) < p.table_parts) {
    if (b == p.B) return;
    const int used = int(min(long(p.max_blocks), (long(len) + mine + p.block_size - 1) / p.block_size));
    const int lo = blockIdx.x * p.per_cta, hi = min(lo + p.per_cta, p.max_blocks);
    int* to = p.block_tables + size_t(b) * p.max_blocks;
    if (p.vectors) {                                                   // rows on 16-byte boundaries: four entries at a time, four times
      for (int i0 = lo + 4 * tid; i0 < hi; i0 += 16 * kThreads) {
        int4 v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int i = i0 + k * 4 * kThreads;
          v[k] = i < min(used, hi) ? *reinterpret_cast<const int4*>(from + i) : make_int4(0, 0, 0, 0);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int i = i0 + k * 4 * kThreads;
          if (i + 1 >= used) v[k].y = 0;
          if (i + 2 >= used) v[k].z = 0;
          if (i + 3 >= used) v[k].w = 0;
          if (i < hi) *reinterpret_cast<int4*>(to + i) = v[k];
        }
      }
    } else {
      for (int i = lo + tid; i < hi; i += kThreads) to[i] = i < used ? from[i] : 0;
    }
    return;
  }
  const int part = blockIdx.x - p.table_parts, lo = part * p.per_cta;
  if (part > 0 && lo >= mine && b < p.B) return;
  long ahead = 0;
  for (int i = tid; i < b; i += kThreads) ahead += rows_of(i);
  const long sum = block_sum(ahead, s_sum);
  const int start = int(min(sum, long(p.n_rows)));
  if (part == 0 && tid == 0) p.q_cu[b] = start;
  if (b == p.B) {
    for (long t = start + long(part) * kThreads + tid; t < p.n_rows; t += long(gridDim.x - p.table_parts) * kThreads) {
      p.positions[t] = 0;
      p.slots[t] = int(t % p.block_size);
      p.token_seq[t] = -1;
      for (int w = 0; w < p.words; ++w) p.tree[size_t(t) * p.words + w] = 0;
    }
    return;
  }
  const int n = min(mine, p.n_rows - start);
  if (part == 0 && tid == 0) p.kv_lens[b] = len + n;
  auto slot_of = [&](long at, int t) {
    const long blk = at / p.block_size;
    return blk < p.columns ? from[blk] * p.block_size + int(at % p.block_size) : t % p.block_size;   // past the table: the reserved block
  };
  if (!p.parents) {
    const int hi = min(lo + p.per_cta, n);
    for (int i = lo + tid; i < hi; i += kThreads) {
      const int t = start + i;
      p.positions[t] = len + i;
      p.slots[t] = slot_of(long(len) + i, t);
      p.token_seq[t] = b;
    }
    return;
  }
  // Ancestors by doubling: a row's set takes in the set of the row it points to, then points where that one points.
  const int W = p.words;
  unsigned long long a[4] = {0, 0, 0, 0};
  int up = -1;
  if (tid < n) {
    up = p.parents[start + tid];
    if (up < 0 || up >= tid) up = -1;            // only an earlier row can be followed
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      if (w == (tid >> 6)) a[w] = 1ull << (tid & 63);
      s_anc[tid * 4 + w] = a[w];
    }
    s_up[tid] = up;
  }
  while (__syncthreads_or(tid < n && up >= 0)) {
    int next = -1;
    if (tid < n && up >= 0) {
#pragma unroll
      for (int w = 0; w < 4; ++w) a[w] |= s_anc[up * 4 + w];
      next = s_up[up];
    }
    __syncthreads();
    if (tid < n) {
#pragma unroll
      for (int w = 0; w < 4; ++w) s_anc[tid * 4 + w] = a[w];
      s_up[tid] = up = next;
    }
  }
  if (tid < n) {
    const int t = start + tid;
    int depth = -1;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      depth += __popcll(a[w]);
      if (w < W) p.tree[size_t(t) * W + w] = a[w];
    }
    p.positions[t] = len + depth;
    p.slots[t] = slot_of(long(len) + tid, t);
    p.token_seq[t] = b;
  }
}

// ---------------------------------------------------------------- accept_tree
constexpr int kCaches = 128;                    // caches of one launch (their addresses travel as kernel arguments)

struct AcceptParams {
  const int* target;            // [T] the target model's token at every row
  const int* tokens;            // [T] the rows' own tokens
  const int* parents;           // [T]
  const int *q_cu, *kv_lens, *block_tables;
  int* out;                     // [B, depth + 1]
  int* accepted;                // [B]
  int* path;                    // [B, depth + 1]
  int T, max_blocks, block_size, depth, n_caches, write;
  void* cache[kCaches];
  int units[kCaches];           // of sizeof(U) bytes per cache row
  int blocks[kCaches];
};

// blockIdx.y = sequence, blockIdx.x = a share of the caches.  next[i] is the first row that follows row i with the token that the
// target has there; the path is the chain from row 0.  Its rows move to the places of its numbers: the i-th row of the path has a
// number of at least i, so no source is a place that an earlier move has written, and a thread that takes the moves of its
// columns in order needs no other thread.
//
// Every CTA walks its sequence's tree again (a few hundred cycles in shared memory), which is cheaper than a launch between walk and
// moves.  The moved rows bound large steps: 64 trees of 9 to 32 rows over the 72 caches of 36 layers (8 x 128 bf16 a row) take 10.0 us, 57 MB
// read and written at 5.7 TB/s (0.86 of a copy's bandwidth); one tree of 8 rows and 4 caches takes 3.1 us, launch and three dependent loads.
template <typename U>
__global__ void __launch_bounds__(kThreads) accept_tree_kernel(const __grid_constant__ AcceptParams p) {
  __shared__ int s_next[kTreeRows], s_path[kTreeRows], s_target[kTreeRows];
  __shared__ long s_src[kTreeRows], s_dst[kTreeRows];
  __shared__ int s_len;
  const int b = blockIdx.y, tid = threadIdx.x;
  const int start = max(p.q_cu[b], 0), n = max(0, min(min(p.q_cu[b + 1], p.T) - start, kTreeRows));
  int up = -1, token = 0;
  if (tid < n) {
    up = p.parents[start + tid];
    token = p.tokens[start + tid];
    s_target[tid] = p.target[start + tid];
    s_next[tid] = kTreeRows;
  }
  __syncthreads();
  if (tid < n && up >= 0 && up < tid && token == s_target[up]) atomicMin(&s_next[up], tid);
  __syncthreads();
  if (tid == 0) {
    int len = 0;
    if (n > 0)
      for (int at = 0; at < kTreeRows && len <= p.depth; at = s_next[at]) s_path[len++] = at;
    s_len = len;
  }
  __syncthreads();
  const int len = s_len;
  if (p.write && blockIdx.x == 0) {
    if (tid == 0) p.accepted[b] = max(len - 1, 0);
    for (int i = tid; i <= p.depth; i += kThreads) {
      p.out[size_t(b) * (p.depth + 1) + i] = i < len ? s_target[s_path[i]] : -1;
      p.path[size_t(b) * (p.depth + 1) + i] = i < len ? s_path[i] : -1;
    }
  }
  if (len < 2 || p.n_caches == 0) return;
  const int base = p.kv_lens[b] - n;
  const int* bt = p.block_tables + size_t(b) * p.max_blocks;
  for (int i = tid; i < len; i += kThreads) {
    auto slot = [&](int at) {
      const int blk = at / p.block_size;
      return at >= 0 && blk < p.max_blocks ? long(bt[blk]) * p.block_size + at % p.block_size : -1l;
    };
    s_src[i] = slot(base + s_path[i]);
    s_dst[i] = slot(base + i);
  }
  __syncthreads();
  for (int c = blockIdx.x; c < p.n_caches; c += gridDim.x) {
    U* rows = static_cast<U*>(p.cache[c]);
    const int units = p.units[c];
    const long most = long(p.blocks[c]) * p.block_size;
    for (int u = tid; u < units; u += kThreads)
      for (int i = 1; i < len; ++i) {
        const long s = s_src[i], d = s_dst[i];
        if (s != d && s >= 0 && d >= 0 && s < most && d < most) rows[d * units + u] = rows[s * units + u];
      }
  }
}

}  // namespace xl_ts

XL_API int xl_step_rows(const void* tables, const void* lens, const void* seqs, const void* counts, const void* parents, void* positions,
                        void* slots, void* token_seq, void* q_cu, void* kv_lens, void* block_tables, void* tree, int pool, int columns, long table_ld, int B,
                        int n_rows, int max_q, int max_blocks, int block_size, int words, void* stream) {
  using namespace xl_ts;
  if (B < 0 || B > 65534 || n_rows < 0 || max_q < 1 || max_blocks < 0 || max_blocks > columns || table_ld < 0 || block_size < 1 || pool < 0) return -2;
  if (parents && (max_q > kTreeRows || words != (max_q + 63) / 64)) return -2;
  RowsParams p{};
  p.tables = static_cast<const int*>(tables);
  p.lens = static_cast<const int*>(lens);
  p.seqs = static_cast<const int*>(seqs);
  p.counts = static_cast<const int*>(counts);
  p.parents = static_cast<const int*>(parents);
  p.positions = static_cast<int*>(positions);
  p.slots = static_cast<int*>(slots);
  p.token_seq = static_cast<int*>(token_seq);
  p.q_cu = static_cast<int*>(q_cu);
  p.kv_lens = static_cast<int*>(kv_lens);
  p.block_tables = static_cast<int*>(block_tables);
  p.tree = static_cast<unsigned long long*>(tree);
  p.pool = pool; p.columns = columns; p.table_ld = table_ld; p.B = B; p.n_rows = n_rows; p.max_q = max_q; p.max_blocks = max_blocks;
  p.block_size = block_size; p.words = parents ? words : 0;
  p.vectors = max_blocks % 4 == 0 && table_ld % 4 == 0 && (reinterpret_cast<uintptr_t>(tables) | reinterpret_cast<uintptr_t>(block_tables)) % 16 == 0;
  // table entries of a CTA: as many as keep all CTAs resident, from two rounds of scalars to four of vectors
  const long resident = 8l * xl_host::sm_count();
  p.per_cta = 2048;
  while (p.per_cta < 16384 && long(max_blocks + p.per_cta - 1) / p.per_cta * B > resident) p.per_cta *= 2;
  p.table_parts = (max_blocks + p.per_cta - 1) / p.per_cta;
  const int row_parts = parents ? 1 : (min(max_q, n_rows) + p.per_cta - 1) / p.per_cta;
  step_rows_kernel<<<dim3(p.table_parts + max(row_parts, 1), B + 1), kThreads, 0, static_cast<cudaStream_t>(stream)>>>(p);
  return cudaGetLastError() == cudaSuccess ? 0 : -1;
}

XL_API int xl_accept_tree(const void* target, const void* tokens, const void* parents, const void* q_cu, const void* kv_lens,
                          const void* block_tables, void* out, void* accepted, void* path, int T, int B, int max_blocks, int block_size, int depth,
                          void** caches, const int* units, const int* blocks, int n, int unit, void* stream) {
  using namespace xl_ts;
  if (B < 0 || B > 65535 || T < 0 || depth < 0 || depth >= kTreeRows || block_size < 1 || n < 0) return -2;
  if (B == 0) return 0;
  AcceptParams p{};
  p.target = static_cast<const int*>(target);
  p.tokens = static_cast<const int*>(tokens);
  p.parents = static_cast<const int*>(parents);
  p.q_cu = static_cast<const int*>(q_cu);
  p.kv_lens = static_cast<const int*>(kv_lens);
  p.block_tables = static_cast<const int*>(block_tables);
  p.out = static_cast<int*>(out);
  p.accepted = static_cast<int*>(accepted);
  p.path = static_cast<int*>(path);
  p.T = T; p.max_blocks = max_blocks; p.block_size = block_size; p.depth = depth;
  for (int first = 0; first == 0 || first < n; first += kCaches) {
    p.n_caches = max(0, min(kCaches, n - first));
    p.write = first == 0;
    for (int i = 0; i < p.n_caches; ++i) {
      p.cache[i] = caches[first + i];
      p.units[i] = units[first + i];
      p.blocks[i] = blocks[first + i];
    }
    const dim3 grid(max(p.n_caches, 1), B);
    auto s = static_cast<cudaStream_t>(stream);
    if (unit == 16) accept_tree_kernel<uint4><<<grid, kThreads, 0, s>>>(p);
    else if (unit == 4) accept_tree_kernel<uint32_t><<<grid, kThreads, 0, s>>>(p);
    else if (unit == 2) accept_tree_kernel<uint16_t><<<grid, kThreads, 0, s>>>(p);
    else if (unit == 1) accept_tree_kernel<uint8_t><<<grid, kThreads, 0, s>>>(p);
    else return -2;
    if (cudaGetLastError() != cudaSuccess) return -1;
  }
  return 0;
}
