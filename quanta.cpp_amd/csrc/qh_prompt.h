// Attention of packed prompts over their own keys and values (qh_prompt.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "qh_internal.h"

namespace qh {

// Rows ld elements apart, on their type's alignment. Entry b: query rows [start[b], start[b + 1]), keys [kstart[b],
// kstart[b + 1]).
struct PromptArgs {
    const void *q, *k, *v;
    void* out;
    int64_t ldq, ldk, ldv, ldo;
    const int32_t *start, *kstart;
    int n, n_tok, n_keys, n_kv, group, causal;
    // |scale| log2(e), 1 for 0; sign: what queries are multiplied by, -1, 0 or 1, so that a hidden score of -infinity stays one
    float scale_log2e, sign;
    // the rest belongs to the launch
    int items, splits;      // row tiles; workgroups that may share one's keys
    float *part_o, *part_ml;  // their results, [items][n_kv][splits][rows of a tile]: [head_dim], and base and sum
};
size_t prompt_workspace_bytes(int dtype, int n_heads, int n_kv, int hd, int n, int n_tok, int n_keys);
hipError_t launch_prompt(PromptArgs a, int dtype, int hd, void* ws, hipStream_t s);

}  // namespace qh
