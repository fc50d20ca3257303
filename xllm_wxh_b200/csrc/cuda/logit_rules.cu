// Penalties for repeated tokens, biases and grammar masks on the logits of a step's rows, in place.
//
// For an id that the row has behind it (its sequence's history, or the tokens on the row's way from the root of its drafted tree),
// made of them generated ones: x -= made freq + (made > 0) pres, then x *= rep below zero and x /= rep above.  Biases are
// added; ids that the row's mask forbids become -inf.  Everything is computed in fp32 and rounded once.
//
// Two kernels that never write the same logit, so that they may run side by side:
//   masks    : (row, columns) - writes -inf where the mask forbids and reads no logit; bound by the bytes written;
//   penalties: (sequence, part, rows) - counts the history's ids in a table in shared memory, so that nothing of the history has to be
//              counted and sent by the host, and touches only the logits whose ids are in it (one sector each); forbidden ids are left
//              to the other kernel.  Bound by the latency of a few dependent loads when there are few rows.
// The table is a hash table (linear probing) where history and biases are sure to fit.  Longer ones are tried, since text has far fewer
// distinct ids than tokens; where an id finds no place within kProbes, or the history is longer still, the CTA goes through the
// vocabulary slice by slice with the table as a plain array, so that any history works.  Counts are whole
// numbers and the last bias of an id wins by its index: the order in which threads arrive changes nothing.
#include <atomic>

#include "vec8.cuh"

namespace xl_lr {
using namespace xl;

constexpr int kThreads = 512, kMaskThreads = 256;
constexpr int kPathRows = 256, kProbes = 64, kMaxSlots = 7680;   // two such tables fit an SM
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
  int parts, row_parts;         // CTAs that share a sequence's vocabulary slices, and its rows
};

// ---------------------------------------------------------------- masks
// Groups of 16 bytes start on 16-byte boundaries of the row's address.  A group's bits straddle two words of the mask.
template <typename T>
__global__ void __launch_bounds__(kMaskThreads) mask_logits_kernel(const Params p, int parts) {
  grid_dep_launch();
  const int row = blockIdx.x / parts;
  const int m = p.mask_of[row];
  if (m < 0 || m >= p.n_masks) return;
  constexpr int G = 16 / sizeof(T);
  constexpr uint32_t kAll = (1u << G) - 1, kLow = sizeof(T) == 2 ? 0xFF80FF80u : 0xFF800000u;
  T* x = static_cast<T*>(p.logits) + size_t(row) * p.ld;
  const uint32_t* w = reinterpret_cast<const uint32_t*>(p.words) + size_t(m) * p.words_ld;
  const int n_words = (p.V + 31) / 32;
  const int shift = int((reinterpret_cast<uintptr_t>(x) / sizeof(T)) % G), groups = (p.V + shift + G - 1) / G;
  T low;
  from_f32(&low, -INFINITY);
  const int share = (groups + parts - 1) / parts, g1 = min(groups, int(blockIdx.x % parts + 1) * share);
  for (int g0 = blockIdx.x % parts * share + threadIdx.x; g0 < g1; g0 += 4 * kMaskThreads) {
    uint32_t bits[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int g = g0 + i * kMaskThreads, t = g * G - shift, at = t >> 5;        // t may start below 0
      bits[i] = kAll;
      if (g < g1) {
        const uint32_t lo = at >= 0 ? w[at] : ~0u, hi = at + 1 < n_words && (t & 31) > 32 - G ? w[at + 1] : ~0u;
        bits[i] = __funnelshift_r(lo, hi, t & 31) & kAll;
        if (t < 0) bits[i] |= (1u << -t) - 1;
        if (t + G > p.V) bits[i] |= kAll & ~((1u << (p.V - t)) - 1);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int t = (g0 + i * kMaskThreads) * G - shift;
      if (bits[i] == 0) {
        *reinterpret_cast<uint4*>(x + t) = make_uint4(kLow, kLow, kLow, kLow);
      } else if (bits[i] != kAll) {
#pragma unroll
        for (int e = 0; e < G; ++e)
          if (!(bits[i] >> e & 1u)) x[t + e] = low;
      }
    }
  }
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
__global__ void __launch_bounds__(kThreads) penalise_logits_kernel(const Params p) {
  extern __shared__ __align__(16) uint8_t smem[];
  const int tid = threadIdx.x, C = p.slots;
  int* s_id = reinterpret_cast<int*>(smem);                        // [C]
  uint32_t* s_word = reinterpret_cast<uint32_t*>(s_id + C);        // [C]
  int* s_bias = reinterpret_cast<int*>(s_word + C);                // [C] index of the bias
  uint16_t* s_list = reinterpret_cast<uint16_t*>(s_bias + C);      // [C] entries that change something
  PathSmem* path_of = reinterpret_cast<PathSmem*>(s_list + C);     // [max_q]
  __shared__ unsigned long long s_made[4];                         // rows whose tokens lie behind the prompt
  __shared__ int s_count, s_firsts, s_full;

  const int part = blockIdx.x % p.parts, rp = blockIdx.x / p.parts % p.row_parts, b = blockIdx.x / p.parts / p.row_parts;
  const int src = p.seqs ? p.seqs[b] : b;
  const int start = max(p.q_cu[b], 0), n = min(min(p.q_cu[b + 1], p.S) - start, p.max_q);
  const int share = (max(n, 0) + p.row_parts - 1) / p.row_parts;
  const int r0 = rp * share, r1 = min(n, r0 + share);
  if (unsigned(src) >= unsigned(p.pool) || r0 >= r1) {
    grid_dep_wait();
    return;
  }
  float rep = 1.f, freq = 0.f, pres = 0.f;
  int given = 0, prompt = 0, e0 = 0, e1 = 0;
  if (p.text) {
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
  if (len == 0 && path == 0 && e1 == e0) {
    grid_dep_wait();
    return;
  }
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

  // Attempt 0 hashes, attempt 1 goes through slices.  Parts that share a sequence's slices must not differ on it: they hash only what
  // is sure to fit, and leave that to the first of them.
  const long most = long(len) + (e1 - e0);
  const bool sure = most <= C / 8 * 7;
  const int probes = sure ? C : kProbes;
  for (int attempt = sure || (p.parts == 1 && most <= 4l * C) ? 0 : 1; attempt < 2; ++attempt) {
    const bool hashed = attempt == 0;
    if (hashed && part > 0) break;
    const int slices = hashed ? 1 : (p.V + C - 1) / C;
    bool full = false;
    for (int slice = hashed ? 0 : part; slice < slices; slice += p.parts) {
      const int v0 = hashed ? 0 : slice * C, v1 = hashed ? p.V : min(p.V, v0 + C);
      __syncthreads();
      for (int i = 4 * tid; i < C; i += 4 * kThreads) {
        *reinterpret_cast<int4*>(s_id + i) = hashed ? make_int4(-1, -1, -1, -1) : make_int4(v0 + i, v0 + i + 1, v0 + i + 2, v0 + i + 3);
        *reinterpret_cast<int4*>(s_word + i) = make_int4(0, 0, 0, 0);
        *reinterpret_cast<int4*>(s_bias + i) = make_int4(-1, -1, -1, -1);
      }
      if (tid == 0) s_count = s_firsts = s_full = 0;
      __syncthreads();
      auto first_slot = [&](int id) { return int(__umulhi(uint32_t(id) * 2654435761u, uint32_t(C))); };
      auto entry = [&](int id) {                                   // -1: no place
        if (!hashed) return id - v0;
        int at = first_slot(id);
        for (int k = 0; k < probes; ++k) {
          const int was = atomicCAS(&s_id[at], -1, id);
          if (was == -1 || was == id) return at;
          at = at + 1 < C ? at + 1 : 0;
        }
        s_full = 1;
        return -1;
      };
      auto find = [&](int id) {
        if (!hashed) return id - v0;
        int at = first_slot(id);
        for (int k = 0; k < probes && s_id[at] != -1; ++k) {
          if (s_id[at] == id) return at;
          at = at + 1 < C ? at + 1 : 0;
        }
        return -1;
      };
      for (int i0 = tid; i0 < len; i0 += 8 * kThreads) {
        int id[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) id[k] = i0 + k * kThreads < len ? text[i0 + k * kThreads] : -1;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          if (id[k] < v0 || id[k] >= v1) continue;
          const int at = entry(id[k]);
          if (at < 0) continue;
          if (i0 + k * kThreads < prompt) atomicOr(&s_word[at], kPrompt);
          else atomicAdd(&s_word[at], 1u);
        }
      }
      for (int e = e0 + tid; e < e1; e += kThreads) {
        const int id = p.bias_ids[e];
        if (id < v0 || id >= v1) continue;
        const int at = entry(id);
        if (at >= 0) atomicMax(&s_bias[at], e);
      }
      __syncthreads();
      full = s_full;
      if (full) break;                                             // (only a hash table fills up)
      // ids on the path: one entry for each distinct one, with the set of the rows that hold it; their counts differ from row to row
      if (tid < path) {
        const int id = path_of[tid].token;
        bool first = id >= v0 && id < v1;
        unsigned long long same[4] = {0, 0, 0, 0};
        for (int i = 0; i < path; ++i) {
          const bool eq = path_of[i].token == id;
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
          path_of[tid].word = word;
          path_of[tid].bias = e;
#pragma unroll
          for (int w = 0; w < 4; ++w) path_of[tid].same[w] = same[w];
          path_of[atomicAdd(&s_firsts, 1)].first = tid;
        }
      }
      __syncthreads();
      for (int i = tid; i < C; i += kThreads) {
        const uint32_t word = s_word[i];
        const bool keep = !(word & kOnPath) && (word != 0 || s_bias[i] >= 0);
        const uint32_t votes = __ballot_sync(0xffffffffu, keep);
        int at = 0;
        if ((tid & 31) == 0 && votes) at = atomicAdd(&s_count, __popc(votes));
        at = __shfl_sync(0xffffffffu, at, 0) + __popc(votes & ((1u << (tid & 31)) - 1));
        if (keep) s_list[at] = uint16_t(i);
      }
      __syncthreads();
      const int count = s_count, firsts = s_firsts, rows = r1 - r0;
      T* x0 = static_cast<T*>(p.logits);
      auto allowed = [&](int row, int id) {
        if (!p.words) return true;
        const int m = p.mask_of[row];
        return m < 0 || m >= p.n_masks || (p.words[size_t(m) * p.words_ld + (id >> 5)] >> (id & 31) & 1);
      };
      // four logits at a time, so that their loads are under way together
      for (int i0 = tid; i0 < count * rows; i0 += 4 * kThreads) {
        T* at[4];
        float x[4];
        int slot[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int i = i0 + k * kThreads;
          at[k] = nullptr;
          x[k] = 0.f;
          slot[k] = 0;
          if (i < count * rows) {
            const int r = i / count, row = start + r0 + r;
            slot[k] = s_list[i - r * count];
            const int id = s_id[slot[k]];
            T* to = x0 + size_t(row) * p.ld + id;
            x[k] = to_f32(*to);
            if (allowed(row, id)) at[k] = to;
          }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (at[k]) {
            const int e = s_bias[slot[k]];
            from_f32(at[k], adjusted(x[k], s_word[slot[k]], e >= 0 ? p.bias_values[e] : 0.f, e >= 0, rep, freq, pres));
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
        if ((word == 0 && e < 0) || !allowed(row, id)) continue;
        T* x = x0 + size_t(row) * p.ld + id;
        from_f32(x, adjusted(to_f32(*x), word, e >= 0 ? p.bias_values[e] : 0.f, e >= 0, rep, freq, pres));
      }
    }
    if (hashed && !full) break;
  }
  grid_dep_wait();                                                 // what follows on the stream waits for this kernel only
}

template <typename T>
int launch(const Params& p, bool penalties, int mask_parts, cudaStream_t s) {
  if (p.words) {
    const long grid = long(p.S) * mask_parts;
    if (grid > 0x7fffffffl) return -2;
    mask_logits_kernel<T><<<unsigned(grid), kMaskThreads, 0, s>>>(p, mask_parts);
    if (cudaGetLastError() != cudaSuccess) return -1;
  }
  if (!penalties) return 0;
  const long grid = long(p.B) * p.parts * p.row_parts;
  if (grid > 0x7fffffffl) return -2;
  auto* kernel = penalise_logits_kernel<T>;
  static std::atomic<bool> ready[64];                              // per device
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -1;
  if (!ready[dev].load(std::memory_order_acquire)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 14 * kMaxSlots + int(sizeof(PathSmem)) * kPathRows) != cudaSuccess) return -1;
    ready[dev].store(true, std::memory_order_release);
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(grid));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = 14 * p.slots + (p.tokens ? sizeof(PathSmem) * p.max_q : 0);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.words ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, p) == cudaSuccess ? 0 : -1;
}

}  // namespace xl_lr

XL_API int xl_adjust_logits(void* logits, int f32, int S, int V, long ld, const void* q_cu, const void* seqs, int B, int pool, int max_q,
                            const void* text, long text_ld, int text_cap, const void* lens, const void* prompts, const void* rep,
                            const void* freq, const void* pres, const void* tokens, const void* parents, const void* bias_cu,
                            const void* bias_ids, const void* bias_values, int n_bias, const void* words, int words_ld, int n_masks,
                            const void* mask_of, void* stream) {
  using namespace xl_lr;
  if (S < 0 || V < 1 || B < 0 || max_q < 1 || (tokens && max_q > kPathRows) || (words && words_ld < (V + 31) / 32)) return -2;
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
  // a table that holds any history of the given length; long ones go by their distinct ids, which text has far fewer of
  p.slots = int(min(long(kMaxSlots), (long(text ? text_cap : 0) + 64) / 448 * 512 + 512));
  // rows of a sequence over several CTAs (each counts the history again), as long as there are SMs without one; slices of the
  // vocabulary, where histories are too long to be hashed
  p.row_parts = B > 0 ? max(1, min(min(max_q, S), 2 * sms / B)) : 1;
  p.parts = B > 0 && text && text_cap > 4l * p.slots ? max(1, min((V + p.slots - 1) / p.slots, 2 * sms / (B * p.row_parts))) : 1;
  // 16-byte groups of a row over CTAs of up to 4 x 4 groups a thread, smaller ones where there are few rows
  const int groups = V * (f32 ? 4 : 2) / 16 + 2;
  const int mask_parts = max(1, min((groups + 4 * kMaskThreads - 1) / (4 * kMaskThreads),
                                    max((groups + 16 * kMaskThreads - 1) / (16 * kMaskThreads), 4 * sms / S)));
  auto s = static_cast<cudaStream_t>(stream);
  const bool penalties = B > 0 && (text || bias_cu);
  return f32 ? launch<float>(p, penalties, mask_parts, s) : launch<__nv_bfloat16>(p, penalties, mask_parts, s);
}
