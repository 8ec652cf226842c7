// The 8-bit token cache: int8 codes [pages][kv head][32 tokens][head size] of keys and of values, and an f32 scale for each token and key/value head
// [pages][kv head][32].  A value is code * scale, scale = f32(amax / 127) of the token's line, code = rint(x * f32(127 / amax)).
//
// Why a scale per token and head: one that several tokens share would have to grow while its page fills, and what the page holds would be rounded
// again, so that a cache would depend on how a prompt was cut into batches.  It costs 4 bytes beside head-size codes (3 % at 128).
#pragma once
#include "common.cuh"
#include "../../../include/dllama_b200.h"

#define KV8_PAGE 32                  // tokens per page (fixed)
#define KV8_TINY 0x1p-100f           // a line whose largest magnitude is below is held as zeros: 127 / amax stays finite, the scale normal

// rows of a batch and the tables that lead to their pages
struct Kv8Rows {
    const int* pos;
    const int* slot;
    const int* block_table;          // [n_slots][max_pages]
    int M, n_slots, max_pages, n_pages;
};
// tokens that row m sees (position + 1); 0: the row has none (a negative position); -1: its sequence or position is not in the table
DL_DEVINL int kv8_tokens(const Kv8Rows& r, int pos, int slot) {
    if (pos < 0) return 0;
    return (unsigned)slot < (unsigned)r.n_slots && pos < r.max_pages * KV8_PAGE ? pos + 1 : -1;
}
