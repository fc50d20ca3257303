// Penalties for repeated tokens, biases and grammar masks on the logits of a step's rows, in place.
//
// For an id that the row has behind it (its sequence's history, or the tokens on the row's way from the root of its drafted tree),
// made of them generated ones: x -= made freq + (made > 0) pres, then x *= rep below zero and x /= rep above.  Biases are
// added; ids that the row's mask forbids become -inf.  Everything is computed in fp32 and rounded once.
//
// Two kernels that never write the same logit, so that they may run side by side:
//   masks    : (row, columns) - writes -inf where the mask forbids and reads no logit; bound by the bytes written.  1024 rows of 152064 fp32
//              logits, seven of ten forbidden: 100 us alone, about 440 MB (67 us at a copy's rate).  Single open ids among forbidden
//              ones leave sectors that are written in part, which the 43 MB that it reads come from; that does not account for
//              all of the distance;
//   penalties: (sequence, part, rows) - counts the history's ids in a table in shared memory, so that nothing of the history has to be
//              counted and sent by the host, and touches only the logits whose ids are in it (one sector each); forbidden ids are left
//              to the other kernel.  Bound by the latency of a few dependent loads and of the shared-memory counts when there are few rows:
//              256 rows with histories of 50 to 3100 ids take 18.5 us, where the bytes alone would take 2.6.
// Both together, for 64 sequences of 16 rows with histories of 200 to 8000 ids: 131 us (masks 100; penalties 49 alone, of which 31 do not
// hide behind the masks), and 7.6 ms written as a row's torch calls.
// The ids that a CTA has to do with (history, path, biases) are marked in a bitmap of the vocabulary; an id's rank in it is its place in
// the table of counts, so that the table is as long as there are distinct ids, nothing is probed for, and the logits are visited in
// the order of their addresses.  More ids than the table holds are taken window by window, larger vocabularies slice by slice.  Counts
// are whole numbers and the last bias of an id wins by its index: the order in which threads arrive changes nothing.
#include <atomic>

#include "tree_api.h"
#include "vec8.cuh"

namespace xl_lr {
using namespace xl;

constexpr int kThreads = 512, kWarps = kThreads / 32, kMaskThreads = 256;
constexpr int kPathRows = 256, kMaxWords = 8192, kMaxSlots = 4608;   // ids of a bitmap / 32; entries of the table
constexpr uint32_t kPrompt = 0x80000000u, kOnPath = 0x40000000u, kMade = 0x3FFFFFFFu;

struct Params {
  void* logits;
  long ld;
  int V, S, B, pool, max_q;
  const int* q_cu;              // [B + 1] rows of each sequence
  const int* seqs;              // [B] pool rows (null: the sequence's own number)
  const int* text;              // [pool, text_ld] (null where text_cap is 0)
  long text_ld;
  int text_cap;
  const int *lens, *prompts;    // [pool] (null: no histories)
  const float *rep, *freq, *pres;
  const int* tokens;            // [S] (null: rows have no tokens of their own)
  const int* parents;           // [S] (null: every row follows the one before)
  const int *bias_cu, *bias_ids;
  const float* bias_values;
  int n_bias;
  const int* words;             // [n_masks, words_ld], bit 1: allowed (null: no masks)
  const int* mask_of;           // [S]
  int words_ld, n_masks;
  int slots, bitmap_words;      // entries of the table, words of the bitmap
  int parts, row_parts;         // CTAs that share a sequence's windows, and its rows
};

// ---------------------------------------------------------------- masks
// A warp takes 32 words of the mask at a time, one a lane, and writes their columns in pieces of 512 bytes, 16 a lane, on 16-byte
// boundaries of the row's address (so that a lane's columns may straddle two words).
template <typename T>
__global__ void __launch_bounds__(kMaskThreads) mask_logits_kernel(const Params p, int parts) {
  const int row = blockIdx.x / parts;
  const int m = p.mask_of[row];
  // what follows on the stream waits for this kernel only, so its last CTA stays until the penalties are done
  const bool last = blockIdx.x == gridDim.x - 1;
  if (m < 0 || m >= p.n_masks) {
    if (last) grid_dep_wait();
    return;
  }
  constexpr int G = 16 / sizeof(T), kPer = 32 / G;                 // columns of a lane, and words of a piece; lanes of a word
  constexpr uint32_t kAll = (1u << G) - 1, kLow = sizeof(T) == 2 ? 0xFF80FF80u : 0xFF800000u;
  T* x = static_cast<T*>(p.logits) + size_t(row) * p.ld;
  const uint32_t* words = reinterpret_cast<const uint32_t*>(p.words) + size_t(m) * p.words_ld;
  const int n_words = (p.V + 31) / 32, lane = threadIdx.x & 31;
  const int shift = int((reinterpret_cast<uintptr_t>(x) / sizeof(T)) % G);       // the lanes' columns start `shift` ahead of the words'
  T low;
  from_f32(&low, -INFINITY);
  const int warp = (blockIdx.x % parts) * (kMaskThreads / 32) + (threadIdx.x >> 5), warps = parts * (kMaskThreads / 32);
  auto word = [&](int w) {                                         // columns past the vocabulary count as allowed
    if (w < 0 || w >= n_words) return ~0u;
    const uint32_t v = words[w];
    return w == n_words - 1 && (p.V & 31) ? v | (~0u << (p.V & 31)) : v;
  };
  auto put = [&](uint32_t bits, int t) {
    if (bits == 0) {
      *reinterpret_cast<uint4*>(x + t) = make_uint4(kLow, kLow, kLow, kLow);
    } else if (bits != kAll) {
#pragma unroll
      for (int e = 0; e < G; ++e)
        if (!(bits >> e & 1u)) x[t + e] = low;
    }
  };
  const int bit = lane % kPer * G - shift;
  uint32_t next = word(warp * 32 + lane), next_before = word(warp * 32 - 1);
  for (int w0 = warp * 32; w0 < n_words + 1; w0 += warps * 32) {   // (the last columns may need a word's worth of lanes more)
    const uint32_t mine = next, before = next_before;
    next = word(w0 + warps * 32 + lane);
    next_before = word(w0 + warps * 32 - 1);
    if (__all_sync(0xffffffffu, mine == ~0u) && before == ~0u) continue;
    const int t0 = (w0 + lane / kPer) * 32 + bit;
    if (shift == 0) {                                              // (of the whole row)
#pragma unroll
      for (int k = 0; k < kPer; ++k) {
        const uint32_t bits = __shfl_sync(0xffffffffu, mine, k * G + lane / kPer) >> bit & kAll;
        if (__any_sync(0xffffffffu, bits != 0 && bits != kAll)) {  // column by column, a word at a time
#pragma unroll
          for (int e = 0; e < G; ++e)
            if (!(__shfl_sync(0xffffffffu, mine, k * G + e) >> lane & 1u)) x[(w0 + k * G + e) * 32 + lane] = low;
        } else if (bits == 0) {
          *reinterpret_cast<uint4*>(x + t0 + k * G * 32) = make_uint4(kLow, kLow, kLow, kLow);
        }
      }
    } else {
#pragma unroll
      for (int k = 0; k < kPer; ++k) {
        const int at = k * G + lane / kPer;
        const uint32_t hi = __shfl_sync(0xffffffffu, mine, at), up = __shfl_sync(0xffffffffu, mine, (at + 31) & 31);
        put((bit >= 0 ? hi >> bit : __funnelshift_r(at == 0 ? before : up, hi, bit & 31)) & kAll, t0 + k * G * 32);
      }
    }
  }
  if (last) grid_dep_wait();
}

// ---------------------------------------------------------------- penalties and biases
__device__ __forceinline__ float adjusted(float x, uint32_t word, float bias, bool biased, float rep, float freq, float pres) {
  if (word != 0) {
    const float made = float(word & kMade);
    x -= made * freq + (made > 0.f ? pres : 0.f);
    x = x < 0.f ? x * rep : __fdiv_rn(x, rep);
  }
  return biased ? x + bias : x;
}

struct PathSmem {                // of a row of the sequence (only where rows have tokens)
  unsigned long long anc[4];     // the row and its ancestors
  unsigned long long same[4];    // rows with the same token
  int up, token, first;          // first: list of the rows that are the first with their token
  uint32_t word;                 // what the table had for the token
  int bias;
  int pad;
};

template <typename T>
__global__ void __launch_bounds__(kThreads, 2) penalise_logits_kernel(const Params p) {
  extern __shared__ __align__(16) uint8_t smem[];
  grid_dep_launch();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, C = p.slots, W = p.bitmap_words;
  uint32_t* s_bits = reinterpret_cast<uint32_t*>(smem);            // [W] ids of the slice that are there
  int* s_rank = reinterpret_cast<int*>(s_bits + W);                // [W] how many ahead of the word
  int* s_id = s_rank + W;                                          // [C]
  uint32_t* s_word = reinterpret_cast<uint32_t*>(s_id + C);        // [C]
  int* s_bias = reinterpret_cast<int*>(s_word + C);                // [C] index of the bias
  PathSmem* path_of = reinterpret_cast<PathSmem*>(s_bias + C);     // [max_q]
  __shared__ unsigned long long s_made[4];                         // rows whose tokens lie behind the prompt
  __shared__ int s_firsts, s_total[kWarps];

  const int part = blockIdx.x % p.parts, rp = blockIdx.x / p.parts % p.row_parts, b = blockIdx.x / p.parts / p.row_parts;
  const int src = p.seqs ? p.seqs[b] : b;
  const int start = max(p.q_cu[b], 0), n = min(min(p.q_cu[b + 1], p.S) - start, p.max_q);
  const int share = (max(n, 0) + p.row_parts - 1) / p.row_parts;
  const int r0 = rp * share, r1 = min(n, r0 + share);
  if (unsigned(src) >= unsigned(p.pool) || r0 >= r1) return;
  float rep = 1.f, freq = 0.f, pres = 0.f;
  int given = 0, prompt = 0, e0 = 0, e1 = 0;
  if (p.lens) {
    rep = p.rep[src]; freq = p.freq[src]; pres = p.pres[src];
    given = max(p.lens[src], 0);
    prompt = p.prompts[src];
  }
  if (p.bias_cu) {
    e0 = max(p.bias_cu[src], 0);
    e1 = max(e0, min(p.bias_cu[src + 1], p.n_bias));
  }
  const bool penal = rep != 1.f || freq != 0.f || pres != 0.f;     // otherwise the history changes nothing
  const int len = penal ? min(given, p.text_cap) : 0;
  const int path = penal && p.tokens ? r1 : 0;                     // rows whose tokens can be on a way to the rows r0 .. r1 - 1
  if (len == 0 && path == 0 && e1 == e0) return;
  const int* text = p.text + size_t(src) * p.text_ld;

  // ancestors of the rows, as sets of rows (by doubling)
  if (path > 0) {
    unsigned long long a[4] = {0, 0, 0, 0};
    int up = -1;
    if (tid < 4) s_made[tid] = 0;
    if (tid < path) {
      up = p.parents ? p.parents[start + tid] : tid - 1;
      if (up < 0 || up >= tid) up = -1;
      path_of[tid].up = up;
      path_of[tid].token = p.tokens[start + tid];
#pragma unroll
      for (int w = 0; w < 4; ++w) path_of[tid].anc[w] = a[w] = w == (tid >> 6) ? 1ull << (tid & 63) : 0;
    }
    while (__syncthreads_or(tid < path && up >= 0)) {
      int next = -1;
      if (tid < path && up >= 0) {
#pragma unroll
        for (int w = 0; w < 4; ++w) a[w] |= path_of[up].anc[w];
        next = path_of[up].up;
      }
      __syncthreads();
      if (tid < path) {
#pragma unroll
        for (int w = 0; w < 4; ++w) path_of[tid].anc[w] = a[w];
        path_of[tid].up = up = next;
      }
    }
    if (tid < path) {
      const int depth = __popcll(a[0]) + __popcll(a[1]) + __popcll(a[2]) + __popcll(a[3]) - 1;
      if (long(given) + depth >= prompt) atomicOr(&s_made[tid >> 6], 1ull << (tid & 63));
    }
  }

  int window = 0;                                                  // of all slices
  for (int v0 = 0; v0 < p.V; v0 += 32 * W) {
    const int v1 = min(p.V, v0 + 32 * W);
    __syncthreads();
    for (int i = tid; i < W; i += kThreads) s_bits[i] = 0;
    __syncthreads();
    auto mark = [&](int id) {
      if (id < v0 || id >= v1) return;
      uint32_t* w = &s_bits[(id - v0) >> 5];
      const uint32_t bit = 1u << ((id - v0) & 31);
      if (!(*reinterpret_cast<volatile uint32_t*>(w) & bit)) atomicOr(w, bit);   // frequent ids are there already
    };
    auto each_of_text = [&](auto&& f) {                            // eight loads at a time
      for (int i0 = tid; i0 < len; i0 += 8 * kThreads) {
        int id[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) id[k] = i0 + k * kThreads < len ? text[i0 + k * kThreads] : -1;
#pragma unroll
        for (int k = 0; k < 8; ++k) f(id[k], i0 + k * kThreads);
      }
    };
    each_of_text([&](int id, int) { mark(id); });
    for (int e = e0 + tid; e < e1; e += kThreads) mark(p.bias_ids[e]);
    if (tid < path) mark(path_of[tid].token);
    __syncthreads();
    // ranks: every thread sums its stretch of the words.  (Short loops: code that runs once per launch costs its fetch.)
    const int each = (W + kThreads - 1) / kThreads, b0 = min(W, tid * each), b1 = min(W, b0 + each);
    int sum = 0;
#pragma unroll 1
    for (int w = b0; w < b1; ++w) sum += __popc(s_bits[w]);
    int incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) s_total[warp] = incl;
    __syncthreads();
    int run = incl - sum, distinct = 0;
#pragma unroll 4
    for (int i = 0; i < kWarps; ++i) {
      if (i < warp) run += s_total[i];
      distinct += s_total[i];
    }
#pragma unroll 1
    for (int w = b0; w < b1; ++w) {
      s_rank[w] = run;
      run += __popc(s_bits[w]);
    }
    __syncthreads();
    auto rank = [&](int id) { return s_rank[(id - v0) >> 5] + __popc(s_bits[(id - v0) >> 5] & ((1u << ((id - v0) & 31)) - 1)); };

    for (int k0 = 0; k0 < distinct; k0 += C, ++window) {
      if (window % p.parts != part) continue;
      const int count = min(C, distinct - k0);
      __syncthreads();
      for (int i = tid; i < count; i += kThreads) {
        s_word[i] = 0;
        s_bias[i] = -1;
      }
      if (tid == 0) s_firsts = 0;
      __syncthreads();
      each_of_text([&](int id, int i) {
        if (id < v0 || id >= v1) return;
        const int k = rank(id) - k0;
        if (k < 0 || k >= count) return;
        s_id[k] = id;
        if (i >= prompt) atomicAdd(&s_word[k], 1u);
        else if (!(*reinterpret_cast<volatile uint32_t*>(&s_word[k]) & kPrompt)) atomicOr(&s_word[k], kPrompt);
      });
      for (int e = e0 + tid; e < e1; e += kThreads) {
        const int id = p.bias_ids[e];
        if (id < v0 || id >= v1) continue;
        const int k = rank(id) - k0;
        if (k < 0 || k >= count) continue;
        s_id[k] = id;
        atomicMax(&s_bias[k], e);
      }
      __syncthreads();
      // ids on the path: one entry for each distinct one, with the set of the rows that hold it; their counts differ from row to row
      if (tid < path) {
        const int id = path_of[tid].token;
        const int k = id >= v0 && id < v1 ? rank(id) - k0 : -1;
        if (k >= 0 && k < count) {
          bool first = true;
          unsigned long long same[4] = {0, 0, 0, 0};
          for (int i = 0; i < path; ++i) {
            const bool eq = path_of[i].token == id;
            first = first && !(eq && i < tid);
#pragma unroll
            for (int w = 0; w < 4; ++w)
              if (eq && w == (i >> 6)) same[w] |= 1ull << (i & 63);
          }
          if (first) {
            const uint32_t word = s_word[k];
            path_of[tid].word = word;
            path_of[tid].bias = s_bias[k];
            s_word[k] = word | kOnPath;
#pragma unroll
            for (int w = 0; w < 4; ++w) path_of[tid].same[w] = same[w];
            path_of[atomicAdd(&s_firsts, 1)].first = tid;
          }
        }
      }
      __syncthreads();
      const int firsts = s_firsts, rows = r1 - r0;
      T* x0 = static_cast<T*>(p.logits);
      // what a row's mask says of an id: word and bit, looked up ahead of the logit, which a forbidden id leaves alone
      auto mask_word = [&](int row, int id) {
        if (!p.words) return ~0u;
        const int m = p.mask_of[row];
        return m < 0 || m >= p.n_masks ? ~0u : uint32_t(p.words[size_t(m) * p.words_ld + (id >> 5)]);
      };
      // four logits at a time, so that their loads are under way together
      for (int i0 = tid; i0 < count * rows; i0 += 4 * kThreads) {
        T* at[4];
        float x[4];
        int entry[4];
        uint32_t open[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int i = min(i0 + k * kThreads, count * rows - 1), r = i / count, row = start + r0 + r;
          entry[k] = i - r * count;
          const int id = s_id[entry[k]];
          at[k] = x0 + size_t(row) * p.ld + id;
          open[k] = i0 + k * kThreads < count * rows && !(s_word[entry[k]] & kOnPath) ? mask_word(row, id) >> (id & 31) & 1u : 0u;
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = open[k] ? to_f32(*at[k]) : 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (open[k]) {
            const int e = s_bias[entry[k]];
            from_f32(at[k], adjusted(x[k], s_word[entry[k]], e >= 0 ? p.bias_values[e] : 0.f, e >= 0, rep, freq, pres));
          }
      }
      for (int i = tid; i < firsts * rows; i += kThreads) {
        const int r = i / firsts, f = path_of[i - r * firsts].first, row = start + r0 + r, id = path_of[f].token;
        int more = 0;
        bool before = false;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const unsigned long long mine = path_of[r0 + r].anc[w] & path_of[f].same[w];
          more += __popcll(mine & s_made[w]);
          before = before || (mine & ~s_made[w]);
        }
        const uint32_t word = (path_of[f].word + uint32_t(more)) | (before ? kPrompt : 0u);
        const int e = path_of[f].bias;
        if ((word == 0 && e < 0) || !(mask_word(row, id) >> (id & 31) & 1u)) continue;
        T* x = x0 + size_t(row) * p.ld + id;
        from_f32(x, adjusted(to_f32(*x), word, e >= 0 ? p.bias_values[e] : 0.f, e >= 0, rep, freq, pres));
      }
    }
  }
}

// The penalties come first: they are latency, and leave room for the masks' CTAs, which start as soon as all of theirs run.
template <typename T>
int launch(const Params& p, bool penalties, int mask_parts, cudaStream_t s) {
  const long grid = long(p.B) * p.parts * p.row_parts, mask_grid = long(p.S) * mask_parts;
  if (grid > 0x7fffffffl || mask_grid > 0x7fffffffl) return -2;
  if (penalties) {
    auto* kernel = penalise_logits_kernel<T>;
    static std::atomic<bool> ready[64];                            // per device
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -1;
    if (!ready[dev].load(std::memory_order_acquire)) {
      if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 8 * kMaxWords + 12 * kMaxSlots + int(sizeof(PathSmem)) * kPathRows) != cudaSuccess)
        return -1;
      ready[dev].store(true, std::memory_order_release);
    }
    kernel<<<unsigned(grid), kThreads, 8 * p.bitmap_words + 12 * p.slots + (p.tokens ? sizeof(PathSmem) * p.max_q : 0), s>>>(p);
    if (cudaGetLastError() != cudaSuccess) return -1;
  }
  if (!p.words) return 0;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(mask_grid));
  cfg.blockDim = dim3(kMaskThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = penalties ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, mask_logits_kernel<T>, p, mask_parts) == cudaSuccess ? 0 : -1;
}

}  // namespace xl_lr

XL_API int xl_adjust_logits(void* logits, int f32, int S, int V, long ld, const void* q_cu, const void* seqs, int B, int pool, int max_q,
                            const void* text, long text_ld, int text_cap, const void* lens, const void* prompts, const void* rep,
                            const void* freq, const void* pres, const void* tokens, const void* parents, const void* bias_cu,
                            const void* bias_ids, const void* bias_values, int n_bias, const void* words, int words_ld, int n_masks,
                            const void* mask_of, void* stream) {
  using namespace xl_lr;
  if (S < 0 || V < 1 || B < 0 || max_q < 1 || (tokens && max_q > kPathRows) || V > (1 << 30) || words_ld < 0) return -2;
  if (text_cap < 0 || (lens && text_cap > 0 && !text)) return -2;
  if (S == 0) return 0;
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
  const int sms = xl_host::sm_count();
  // a table that holds any history of the given length; of long ones their distinct ids, which text has far fewer of, at a time
  p.bitmap_words = (min((V + 31) / 32, kMaxWords) + 1) & ~1;
  p.slots = int(min(long(kMaxSlots), (text_cap + long(n_bias) + max_q + 31) / 32 * 32));
  // rows of a sequence over several CTAs (each counts the history again), as long as an SM has fewer than two (64 sequences of 16 rows
  // beside their masks: 131 us, with one CTA an SM 146, with three 137); windows, where
  // histories are long enough to need several
  p.row_parts = B > 0 ? max(1, min(min(max_q, S), 2 * sms / B)) : 1;
  p.row_parts = max(p.row_parts, (min(max_q, S) >> 18) + 1);                       // rows of a CTA times its table's entries count in 32 bits
  p.parts = B > 0 && text_cap > 4l * p.slots ? max(1, min(text_cap / p.slots + 1, 2 * sms / (B * p.row_parts))) : 1;
  // a row's mask over CTAs of eight warps, two times 32 words a warp: in more CTAs their start costs open rows more, in fewer what is
  // written at a time lies further apart (1024 rows of 152064 fp32: 99 us with one, 102 with two, 107 with four, 122 with nineteen)
  const int mask_parts = ((V + 31) / 32 + 1 + 2 * kMaskThreads - 1) / (2 * kMaskThreads);
  auto s = static_cast<cudaStream_t>(stream);
  const bool penalties = B > 0 && (lens || bias_cu);
  return f32 ? launch<float>(p, penalties, mask_parts, s) : launch<__nv_bfloat16>(p, penalties, mask_parts, s);
}
