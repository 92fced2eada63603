// What the entry points of the 8-bit cache take, in structures whose fields a caller can lay down in one go (fields of 8 bytes in
// front of those of 4, no padding but at the rules' bias).
#pragma once

#include "attention_rules.h"

// A layer's cache in 8 bits and a step's block table.  Codes [num_pages][n_kv_heads][page_size][head_dim] of `code` (0: e4m3, 1: int8),
// keys and values with one page pitch (bytes); scales float32 [num_pages][n_kv_heads], row pitch scale_stride.
typedef struct SandyCache8 {
    void *k, *v;
    float *k_scale, *v_scale;
    long long page_stride, scale_stride;
    const int* block_table;        // int32 [n_seqs][max_blocks]
    int* status;                   // device int or null
    int max_blocks, n_seqs, n_kv_heads, head_dim, page_size, num_pages, code;
    int dtype;                     // of rows, queries and results: 0 = float32, 1 = bfloat16
} SandyCache8;

// Rows of keys and values beside the cache: [n_rows, n_kv_heads * head_dim], row pitches in elements.  Request s's are rows start[s] ..
// start[s + 1] - 1, for its positions first[s] on; max_len: the most that one request has.
typedef struct SandyRows8 {
    SandyCache8 cache;
    void *k_rows, *v_rows;
    long long ld_k, ld_v;
    const int *start, *first;
    int n_rows, max_len;
} SandyRows8;

// Attention over the cache.  q and out [n_rows, n_heads * head_dim], row pitches in elements.  Prompt portions: q_start [n_z + 1], positions =
// kv_before [n_z], token_seq null, request z = row z of the block table (n_z = n_seqs), max_n the most tokens of one.  Single tokens:
// q_start null, token z of request token_seq[z] at positions[z], max_n 1.
typedef struct SandyAttend8 {
    SandyCache8 cache;
    const void* q;
    void* out;
    long long ld_q, ld_out;
    const int *token_seq, *positions, *q_start;
    float* scratch;
    SandyAttentionRules rules;
    int n_rows, n_z, max_n, n_heads;
    int num_splits, max_keys;
    float scale;
    int unused;
} SandyAttend8;
