// Penalties for repeated tokens, biases and grammar masks on the logits of a step's rows, in place and in one launch.
//
// For an id that the row has behind it (its sequence's history, or the tokens on the row's way from the root of its drafted tree),
// made of them generated ones: x -= made freq + (made > 0) pres, then x *= rep below zero and x /= rep above.  Biases are
// added; ids that the row's mask forbids become -inf.  Everything is computed in fp32 and rounded once.
//
// The kernel reads the history itself, so that nothing of it has to be counted and sent by the host.  Two kinds of CTAs share the launch
// and never write the same logit:
//   penalties: (sequence, part, rows) - counts the history's ids in a table in shared memory, which the sequence's rows share, and
//              touches only the logits whose ids are in it; forbidden ids are left to the other kind;
//   masks:     (row, columns) - writes -inf where the mask forbids and reads no logit.
// The table is a hash table when the history, the path and the biases fit three quarters of it, otherwise it holds a slice of the
// vocabulary at a time, so that any length works.  Counts are whole numbers and the last bias of an id wins by its index: the
// order in which threads arrive changes nothing.
#include "vec8.cuh"

namespace xl_lr {
using namespace xl;

constexpr int kThreads = 512;
constexpr int kPathRows = 256;
constexpr uint32_t kPrompt = 0x80000000u, kOnPath = 0x40000000u, kMade = 0x3FFFFFFFu;

struct Params {
  void* logits;
  long ld;
  int V, S, B, pool, max_q;
  const int* q_cu;              // [B + 1] rows of each sequence
  const int* seqs;              // [B] pool rows (null: the sequence's own number)
  const int* text;              // [pool, text_ld] (null: no histories)
  long text_ld;
  int text_cap;
  const int *lens, *prompts;    // [pool]
  const float *rep, *freq, *pres;
  const int* tokens;            // [S] (null: rows have no tokens of their own)
  const int* parents;           // [S] (null: every row follows the one before)
  const int *bias_cu, *bias_ids;
  const float* bias_values;
  int n_bias;
  const int* words;             // [n_masks, words_ld], bit 1: allowed (null: no masks)
  const int* mask_of;           // [S]
  int words_ld, n_masks;
  int slots;                    // entries of the table
  int parts, row_parts;
  int penalty_ctas;             // parts * row_parts * B
  int columns, mask_parts;      // columns of a mask CTA, such CTAs of a row
};

__device__ __forceinline__ float adjusted(float x, uint32_t word, float bias, bool biased, float rep, float freq, float pres) {
  if (word != 0) {
    const float made = float(word & kMade);
    x -= made * freq + (made > 0.f ? pres : 0.f);
    x = x < 0.f ? x * rep : __fdiv_rn(x, rep);
  }
  return biased ? x + bias : x;
}

template <typename T>
__device__ void mask_columns(const Params& p, int row, int c0) {
  const int m = p.mask_of[row];
  if (m < 0 || m >= p.n_masks) return;
  constexpr int kPer16 = 16 / sizeof(T);
  T* x = static_cast<T*>(p.logits) + size_t(row) * p.ld;
  const uint32_t* w = reinterpret_cast<const uint32_t*>(p.words) + size_t(m) * p.words_ld;
  const int n_words = (p.V + 31) / 32;
  // groups of eight columns start on 16-byte boundaries of the row's address
  const int shift = int((reinterpret_cast<uintptr_t>(x) / sizeof(T)) % kPer16);
  T low;
  from_f32(&low, -INFINITY);
  const int hi = min(c0 + p.columns, p.V + shift);
  for (int g = c0 + 8 * int(threadIdx.x); g < hi; g += 8 * kThreads) {
    const int t = g - shift, at = t >> 5;                          // may start below 0
    const uint32_t a = at >= 0 && at < n_words ? w[at] : ~0u, b = at + 1 < n_words ? w[at + 1] : ~0u;
    const uint32_t bits = __funnelshift_r(a, b, t & 31) & 0xFFu;
    if (bits == 0xFFu) continue;
    if (bits == 0 && t >= 0 && t + 8 <= p.V) {
      const uint32_t pair = sizeof(T) == 2 ? 0xFF80FF80u : 0xFF800000u;
      uint4* to = reinterpret_cast<uint4*>(x + t);
      to[0] = make_uint4(pair, pair, pair, pair);
      if (sizeof(T) == 4) to[1] = make_uint4(pair, pair, pair, pair);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (!(bits >> e & 1u) && t + e >= 0 && t + e < p.V) x[t + e] = low;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) adjust_logits_kernel(const Params p) {
  extern __shared__ __align__(16) uint32_t smem[];
  if (int(blockIdx.x) >= p.penalty_ctas) {
    const int i = blockIdx.x - p.penalty_ctas;
    mask_columns<T>(p, i / p.mask_parts, i % p.mask_parts * p.columns);
    return;
  }
  const int tid = threadIdx.x, C = p.slots;
  int* s_id = reinterpret_cast<int*>(smem);                        // [C]
  uint32_t* s_word = smem + C;                                     // [C]
  int* s_bias = reinterpret_cast<int*>(smem + 2 * C);              // [C] index of the bias, then its value's bits
  __shared__ unsigned long long s_anc[kPathRows][4], s_same[kPathRows][4];
  __shared__ int s_up[kPathRows], s_tok[kPathRows], s_first[kPathRows];
  __shared__ uint32_t s_pword[kPathRows];
  __shared__ float s_pbias[kPathRows];
  __shared__ int s_pbiased[kPathRows];
  __shared__ unsigned long long s_made[4];                          // rows whose tokens lie behind the prompt
  __shared__ int s_count, s_firsts;

  const int part = blockIdx.x % p.parts, rp = blockIdx.x / p.parts % p.row_parts, b = blockIdx.x / p.parts / p.row_parts;
  const int src = p.seqs ? p.seqs[b] : b;
  if (unsigned(src) >= unsigned(p.pool)) return;
  const int start = max(p.q_cu[b], 0), n = min(min(p.q_cu[b + 1], p.S) - start, p.max_q);
  const int share = (max(n, 0) + p.row_parts - 1) / p.row_parts;
  const int r0 = rp * share, r1 = min(n, r0 + share);
  if (r0 >= r1) return;
  float rep = 1.f, freq = 0.f, pres = 0.f;
  int len = 0, prompt = 0;
  if (p.text) {
    rep = p.rep[src]; freq = p.freq[src]; pres = p.pres[src];
    if (rep != 1.f || freq != 0.f || pres != 0.f) {                // otherwise the history changes nothing
      len = min(max(p.lens[src], 0), p.text_cap);
      prompt = p.prompts[src];
    }
  }
  const bool penal = p.text && (rep != 1.f || freq != 0.f || pres != 0.f);
  int e0 = 0, e1 = 0;
  if (p.bias_cu) {
    e0 = max(p.bias_cu[src], 0);
    e1 = min(p.bias_cu[src + 1], p.n_bias);
  }
  const int path = penal && p.tokens ? r1 : 0;                     // rows whose tokens can be on a way to the rows r0 .. r1 - 1
  if (len == 0 && path == 0 && e1 <= e0) return;
  const int* text = p.text + size_t(src) * p.text_ld;

  // ancestors of the rows, as sets of rows (by doubling), and the rows with the same token as each
  if (path > 0) {
    unsigned long long a[4] = {0, 0, 0, 0};
    int up = -1;
    if (tid < 4) s_made[tid] = 0;
    if (tid < path) {
      up = p.parents ? p.parents[start + tid] : tid - 1;
      if (up < 0 || up >= tid) up = -1;
      s_up[tid] = up;
      s_tok[tid] = p.tokens[start + tid];
#pragma unroll
      for (int w = 0; w < 4; ++w) s_anc[tid][w] = a[w] = w == (tid >> 6) ? 1ull << (tid & 63) : 0;
    }
    while (__syncthreads_or(tid < path && up >= 0)) {
      int next = -1;
      if (tid < path && up >= 0) {
#pragma unroll
        for (int w = 0; w < 4; ++w) a[w] |= s_anc[up][w];
        next = s_up[up];
      }
      __syncthreads();
      if (tid < path) {
#pragma unroll
        for (int w = 0; w < 4; ++w) s_anc[tid][w] = a[w];
        s_up[tid] = up = next;
      }
    }
    if (tid < path) {
      const int depth = __popcll(a[0]) + __popcll(a[1]) + __popcll(a[2]) + __popcll(a[3]) - 1;
      if (long(max(p.lens[src], 0)) + depth >= prompt) atomicOr(&s_made[tid >> 6], 1ull << (tid & 63));
    }
  }

  const bool hashed = long(len) + max(e1 - e0, 0) <= C / 4 * 3;
  const int slices = hashed ? 1 : (p.V + C - 1) / C;
  for (int slice = part; slice < slices; slice += p.parts) {
    const int v0 = hashed ? 0 : slice * C, v1 = hashed ? p.V : min(p.V, v0 + C);
    __syncthreads();
    for (int i = tid; i < C; i += kThreads) {
      s_id[i] = hashed ? -1 : v0 + i;
      s_word[i] = 0;
      s_bias[i] = -1;
    }
    if (tid == 0) s_count = s_firsts = 0;
    __syncthreads();
    auto first_slot = [&](int id) { return int((uint32_t(id) * 2654435761u) >> 16) & (C - 1); };
    // the table has free entries (it is at most three quarters full), so the search ends
    auto entry = [&](int id) {
      if (!hashed) return id - v0;
      int at = first_slot(id);
      while (true) {
        const int was = atomicCAS(&s_id[at], -1, id);
        if (was == -1 || was == id) return at;
        at = (at + 1) & (C - 1);
      }
    };
    auto find = [&](int id) {
      if (!hashed) return id - v0;
      int at = first_slot(id);
      while (s_id[at] != id) {
        if (s_id[at] == -1) return -1;
        at = (at + 1) & (C - 1);
      }
      return at;
    };
    for (int i = tid; i < len; i += kThreads) {
      const int id = text[i];
      if (id < v0 || id >= v1) continue;
      uint32_t* w = &s_word[entry(id)];
      if (i < prompt) atomicOr(w, kPrompt);
      else atomicAdd(w, 1u);
    }
    for (int e = e0 + tid; e < e1; e += kThreads) {
      const int id = p.bias_ids[e];
      if (id >= v0 && id < v1) atomicMax(&s_bias[entry(id)], e);
    }
    __syncthreads();
    // ids on the path: one entry for each distinct one, with the set of the rows that hold it; their counts differ from row to row
    if (tid < path) {
      const int id = s_tok[tid];
      bool first = id >= v0 && id < v1;
      unsigned long long same[4] = {0, 0, 0, 0};
      for (int i = 0; i < path; ++i) {
        const bool eq = s_tok[i] == id;
        first = first && !(eq && i < tid);
#pragma unroll
        for (int w = 0; w < 4; ++w)
          if (eq && w == (i >> 6)) same[w] |= 1ull << (i & 63);
      }
      if (first) {
        const int at = find(id);
        uint32_t word = 0;
        int e = -1;
        if (at >= 0) {
          word = s_word[at];
          e = s_bias[at];
          s_word[at] = word | kOnPath;
        }
        s_pword[tid] = word;
        s_pbiased[tid] = e >= 0;
        s_pbias[tid] = e >= 0 ? p.bias_values[e] : 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) s_same[tid][w] = same[w];
        s_first[atomicAdd(&s_firsts, 1)] = tid;
      }
    }
    __syncthreads();
    // the other entries that change something move to the front of the table
    for (int base = 0; base < C; base += kThreads) {
      const int i = base + tid;
      int id = -1, e = -1;
      uint32_t word = 0;
      if (i < C) {
        id = s_id[i];
        word = s_word[i];
        e = s_bias[i];
      }
      const bool keep = id >= 0 && !(word & kOnPath) && (word != 0 || e >= 0);
      const uint32_t votes = __ballot_sync(0xffffffffu, keep);
      int at = 0;
      if ((tid & 31) == 0) at = atomicAdd(&s_count, __popc(votes));
      at = __shfl_sync(0xffffffffu, at, 0) + __popc(votes & ((1u << (tid & 31)) - 1));
      const float value = keep && e >= 0 ? p.bias_values[e] : 0.f;
      __syncthreads();                                             // everything below base + kThreads has been read
      if (keep) {
        s_id[at] = e >= 0 ? ~id : id;                              // ids with a bias are stored complemented
        s_word[at] = word;
        s_bias[at] = __float_as_int(value);
      }
    }
    __syncthreads();
    const int count = s_count, firsts = s_firsts, rows = r1 - r0;
    T* x0 = static_cast<T*>(p.logits);
    auto allowed = [&](int row, int id) {
      if (!p.words) return true;
      const int m = p.mask_of[row];
      return m < 0 || m >= p.n_masks || (p.words[size_t(m) * p.words_ld + (id >> 5)] >> (id & 31) & 1);
    };
    for (int i = tid; i < count * rows; i += kThreads) {
      const int r = i / count, e = i - r * count, row = start + r0 + r;
      const int raw = s_id[e], id = raw < 0 ? ~raw : raw;
      if (!allowed(row, id)) continue;
      T* x = x0 + size_t(row) * p.ld + id;
      from_f32(x, adjusted(to_f32(*x), s_word[e], __int_as_float(s_bias[e]), raw < 0, rep, freq, pres));
    }
    for (int i = tid; i < firsts * rows; i += kThreads) {
      const int r = i / firsts, f = s_first[i - r * firsts], row = start + r0 + r, id = s_tok[f];
      int more = 0;
      bool given = false;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const unsigned long long mine = s_anc[r0 + r][w] & s_same[f][w];
        more += __popcll(mine & s_made[w]);
        given = given || (mine & ~s_made[w]);
      }
      const uint32_t word = (s_pword[f] + uint32_t(more)) | (given ? kPrompt : 0u);
      if ((word == 0 && !s_pbiased[f]) || !allowed(row, id)) continue;
      T* x = x0 + size_t(row) * p.ld + id;
      from_f32(x, adjusted(to_f32(*x), word, s_pbias[f], s_pbiased[f], rep, freq, pres));
    }
  }
}

}  // namespace xl_lr

XL_API int xl_adjust_logits(void* logits, int f32, int S, int V, long ld, const void* q_cu, const void* seqs, int B, int pool, int max_q,
                            const void* text, long text_ld, int text_cap, const void* lens, const void* prompts, const void* rep,
                            const void* freq, const void* pres, const void* tokens, const void* parents, const void* bias_cu,
                            const void* bias_ids, const void* bias_values, int n_bias, const void* words, int words_ld, int n_masks,
                            const void* mask_of, void* stream) {
  using namespace xl_lr;
  if (S < 0 || V < 1 || B < 0 || max_q < 1 || (tokens && max_q > kPathRows) || (words && words_ld < (V + 31) / 32)) return -2;
  if (S == 0 || B == 0) return 0;
  Params p{};
  p.logits = logits;
  p.ld = ld;
  p.V = V; p.S = S; p.B = B; p.pool = pool; p.max_q = max_q;
  p.q_cu = static_cast<const int*>(q_cu);
  p.seqs = static_cast<const int*>(seqs);
  p.text = static_cast<const int*>(text);
  p.text_ld = text_ld; p.text_cap = text_cap;
  p.lens = static_cast<const int*>(lens);
  p.prompts = static_cast<const int*>(prompts);
  p.rep = static_cast<const float*>(rep);
  p.freq = static_cast<const float*>(freq);
  p.pres = static_cast<const float*>(pres);
  p.tokens = static_cast<const int*>(tokens);
  p.parents = static_cast<const int*>(parents);
  p.bias_cu = static_cast<const int*>(bias_cu);
  p.bias_ids = static_cast<const int*>(bias_ids);
  p.bias_values = static_cast<const float*>(bias_values);
  p.n_bias = n_bias;
  p.words = static_cast<const int*>(words);
  p.mask_of = static_cast<const int*>(mask_of);
  p.words_ld = words_ld; p.n_masks = n_masks;
  p.slots = 8192;
  p.parts = 1;
  p.row_parts = 1;
  const bool penalties = text || bias_cu;
  const long ctas = penalties ? long(B) * p.parts * p.row_parts : 0;
  p.columns = 16384;
  p.mask_parts = (V + 16 + p.columns - 1) / p.columns;
  const long grid = ctas + (words ? long(S) * p.mask_parts : 0);
  if (grid == 0) return 0;
  if (grid > 0x7fffffffl) return -2;
  p.penalty_ctas = int(ctas);
  const int smem = penalties ? 12 * p.slots : 0;
  auto* kernel = f32 ? adjust_logits_kernel<float> : adjust_logits_kernel<__nv_bfloat16>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 12 * 8192);
  if (e != cudaSuccess) return -1;
  kernel<<<unsigned(grid), kThreads, smem, static_cast<cudaStream_t>(stream)>>>(p);
  return cudaGetLastError() == cudaSuccess ? 0 : -1;
}
