// Prompt attention whose items leave SMs idle: the steps of an item go to several CTAs (shares).  What a warp has of its 32 rows lies here until the last of
// the item's shares comes, whose warp joins them, in the order of the shares.
#pragma once

#define PT_SHARE_SLOTS 160             // CTAs of such a launch at most, each with one share
#define PT_LEAST_STEPS 4               // of 128 tokens, of a share; of an item that goes to two CTAs: 32
#define PT_SHARE_TOKENS (3 * 128 * PT_LEAST_STEPS)      // no sequence below that has shares
#define PT_SHARE_WARPS 8               // of a CTA, 32 rows each

struct PtShares {
    unsigned* arrived;                 // [slot][warp], 0 between launches; null: no shares
    float2* norms;                     // [slot][warp][32] reference maximum (in the log2 domain) and sum of weights, < 0: no steps of that tile
    float4* sums;                      // [slot][warp][head size / 4][32]: weights times values, four columns of a row
};
static long long pt_share_bytes(int head_size) { return (long long)PT_SHARE_SLOTS * PT_SHARE_WARPS * (sizeof(unsigned) + 32 * (sizeof(float2) + head_size * sizeof(float))); }
