// Operators on the rows of a step of many sequences: norm with residual, rotary positions, and beam search's selection.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "qh_internal.h"

namespace qh {

// Rows ld elements apart; what a call does not use is null. Any alignment of the type's own size.
struct NormArgs {
    const void *x, *res;  // [n_tok][n]
    const float* w;
    void *sum, *y;
    int8_t* q;  // [n_tok][n], d [n_tok][n / 32]
    float* d;
    int64_t ldx, ldr, lds, ldy;
    int n_tok, n;
    double eps;
};
constexpr int kMaxNorm = 32768;  // elements of a row: what a workgroup of 1,024 threads holds in registers
hipError_t launch_rmsnorm(const NormArgs& a, int dtype, hipStream_t s);

struct RopeRows {
    const void* x;
    void* out;
    int64_t ld, ldo;
    int heads;
};
struct RopeArgs {
    const double* turns;  // [rot / 2] turns per position
    const int32_t* pos;   // [n_tok]
    RopeRows q, k;        // k.heads 0: none
    float magnitude;
    int hd, rot, n_tok;
};
hipError_t launch_rope(const RopeArgs& a, int dtype, bool interleaved, hipStream_t s);

// Beam search's selection (qh_beam.hip): logits [prompts * beams][n_valid], rows ld apart, on their type's alignment; the k
// best candidates of each prompt, best first.
struct BeamArgs {
    const void* logits;
    const float* scores;  // [prompts * beams], or null: 0
    int32_t *parent, *token;
    float* best;
    void* ws;
    int64_t ld;
    int prompts, beams, n_valid, k;
};
size_t beam_workspace_bytes(int dtype, int prompts, int beams, int n_valid);
hipError_t launch_beam_select(const BeamArgs& a, int dtype, hipStream_t s);

}  // namespace qh
