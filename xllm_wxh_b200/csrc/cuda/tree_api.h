// Entry points of the kernels of a step with trees of drafted tokens, for the files that define them and for the host side that calls them
// through addresses: an argument list that changes in one place only does not compile.
#pragma once

#ifndef XL_API
#define XL_API extern "C" __attribute__((visibility("default")))
#endif

XL_API int xl_step_rows(const void* tables, const void* lens, const void* seqs, const void* counts, const void* parents, void* positions,
                        void* slots, void* token_seq, void* q_cu, void* kv_lens, void* block_tables, void* tree, int pool, int columns,
                        long table_ld, int B, int n_rows, int max_q, int max_blocks, int block_size, int words, void* stream);

// `caches`, `units`, `blocks`: host arrays of n entries.  unit: bytes that move at once (16, 4, 2 or 1).
XL_API int xl_accept_tree(const void* target, const void* tokens, const void* parents, const void* q_cu, const void* kv_lens,
                          const void* block_tables, void* out, void* accepted, void* path, int T, int B, int max_blocks, int block_size,
                          int depth, void** caches, const int* units, const int* blocks, int n, int unit, void* stream);

// Bytes of the workspace.  max_q, max_kv: bounds of a sequence's rows and keys; plain: fp32, or scores or caches that the tensor-core kernel
// does not take.  *tc: whether that kernel serves these sizes (for query rows on 16-byte boundaries).
XL_API long xl_attention_tree_workspace(int T, int B, int max_blocks, int block_size, int num_blocks, int n_q, int n_kv, int D, int plain,
                                        int max_q, int max_kv, int* tc);
XL_API int xl_attention_tree(const void* q, const void* k_cache, const void* v_cache, void* out, const void* q_cu, const void* kv_lens,
                             const void* block_tables, const void* token_seq, const void* positions, const void* tree, int T, int B,
                             int max_blocks, int block_size, int num_blocks, int n_q, int n_kv, int D, int words, long q_row, long q_head,
                             float scale, int window, int f32, int max_q, int max_kv, int tc, void* workspace, long workspace_bytes,
                             void* stream);

XL_API int xl_adjust_logits(void* logits, int f32, int S, int V, long ld, const void* q_cu, const void* seqs, int B, int pool, int max_q,
                            const void* text, long text_ld, int text_cap, const void* lens, const void* prompts, const void* rep,
                            const void* freq, const void* pres, const void* tokens, const void* parents, const void* bias_cu,
                            const void* bias_ids, const void* bias_values, int n_bias, const void* words, int words_ld, int n_masks,
                            const void* mask_of, void* stream);
