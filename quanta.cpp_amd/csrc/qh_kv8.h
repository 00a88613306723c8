// The 8-bit paged key / value cache: its layout, and what the kernels that read and write it share.
//
// A block is 16 tokens of one KV head, keys and values apart: 16 * head_dim codes (int8) and one f32 scale. A page holds
// page_tokens / 16 blocks of every KV head: the key blocks [n_kv][page_tokens / 16], the value blocks likewise, then the
// scales f32 [key, value][n_kv][page_tokens / 16]; pages are padded to 128 bytes. A code is stored as code + 128 (the
// attention makes f16 of it with one instruction less a word). Within a block the codes lie in the order in
// which a wave's 64 lanes take them as matrix operands, 16 bytes to a lane, so that every load of a block is one
// contiguous KB per 64 dimensions, without a transposition of the values:
//   keys    [head_dim / 64][4 groups][16 tokens][16 dims]: lane 16 g + t holds dims 64 c + 16 g .. + 15 of token t
//   values  [head_dim / 64][4 groups][16][4 dims][4 tokens]: lane 16 g + j holds dims 64 c + 4 j .. + 3 of tokens
//           4 g .. 4 g + 3, the tokens whose weights the same lane holds after the product of keys and queries
// A value block's scale has its sign set where some of its tokens have only zeros for codes though the scale is not 0: next to
// the token that gave the scale theirs were too small. Attention counts such tokens in the sum of weights alone, so that they
// do not bring that scale to rows which give the large token no weight.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "qh_internal.h"

namespace qh {

constexpr int kBlk = QH_KV8_BLOCK;
constexpr uint32_t kBias = 0x80808080u;  // the 128 that stored codes carry, in each byte of a word

// What the kernels need of a qh_kv8_cache for one layer.
struct Kv8View {
    uint8_t* pages;  // the layer's first page
    int32_t *table, *lens, *refs, *status;
    size_t page_bytes;
    int n_pages, n_kv, hd, n_seqs, seq_pages;
    int page_shift;  // log2(page_tokens)
};

__host__ __device__ __forceinline__ size_t kv8_page_bytes(int page_tokens, int n_kv, int hd) {
    const size_t raw = 2 * (size_t)n_kv * page_tokens * hd + 8 * (size_t)n_kv * (page_tokens / kBlk);
    return (raw + 127) / 128 * 128;
}

#if defined(__HIPCC__)
// A load of what is read once: it does not displace what others keep in the caches.
__device__ __forceinline__ uint4 load_once(const uint4* p) {
    typedef uint32_t u4 __attribute__((ext_vector_type(4)));
    return __builtin_bit_cast(uint4, __builtin_nontemporal_load(reinterpret_cast<const u4*>(p)));
}

// Tokens of a sequence, never more than its table row can hold.
__device__ __forceinline__ int kv8_len(const Kv8View& c, int seq) {
    return min(max(c.lens[seq], 0), c.seq_pages << c.page_shift);
}

// x combined by or over the 16 lanes of each row of the wave.
__device__ __forceinline__ uint32_t or_row16(uint32_t x) {
    x |= (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x128, 0xF, 0xF, false);
    x |= (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x124, 0xF, 0xF, false);
    x |= (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x122, 0xF, 0xF, false);
    return x | (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x121, 0xF, 0xF, false);
}

// The codes of block `blk` (of the page) of KV head h, which = 0 keys, 1 values.
__device__ __forceinline__ uint8_t* kv8_codes(const Kv8View& c, int page, int which, int h, int blk) {
    const int per = 1 << (c.page_shift - 4);
    return c.pages + (size_t)page * c.page_bytes + ((size_t)((which * c.n_kv + h) * per + blk) * (kBlk * c.hd));
}
__device__ __forceinline__ float* kv8_scale(const Kv8View& c, int page, int which, int h, int blk) {
    const int per = 1 << (c.page_shift - 4);
    uint8_t* s = c.pages + (size_t)page * c.page_bytes + 2 * ((size_t)c.n_kv * c.hd << c.page_shift);
    return reinterpret_cast<float*>(s) + (which * c.n_kv + h) * per + blk;
}

// A ragged batch: entry b is the last rows [start[b], start[b + 1]) of sequence seqs[b] (null: seq0 + b); start null: one
// row each. Whatever the arrays hold, rows stay in [0, n_tok) and sequences outside the cache have none.
struct Kv8Batch {
    const int32_t *start, *seqs;
    int n, n_tok, seq0;
    __device__ __forceinline__ int at(int b) const {
        return start ? min(max(start[b], 0), n_tok) : min(b, n_tok);
    }
    __device__ __forceinline__ int seq(int b) const { return seqs ? seqs[b] : seq0 + b; }
};

// Work items of a ragged batch without a prefix sum: entry b's items begin at floor(start[b] * mul / unit) + pad * b,
// which leaves every entry floor(rows * mul / unit) + pad of them at least. The entry of `item` (a wave calls it, all
// lanes with one item): the last one that begins at or before it, found 64 entries at a time, each round in the stretch
// that the one before has left.
__device__ __forceinline__ int kv8_entry_of(const Kv8Batch& q, int item, int mul, int unit, int pad, int* first) {
    const int lane = (int)threadIdx.x & 63;
    for (int lo = 0, n = q.n;;) {
        const int stride = (n + 63) >> 6, at = lane * stride, i = lo + at;
        const int key = at < n ? (int)((long)q.at(i) * mul / unit) + pad * i : 0x7fffffff;
        const uint64_t m = __ballot(key <= item);
        if (m == 0) return -1;
        const int l = 63 - __builtin_clzll(m);
        *first = __builtin_amdgcn_readlane(key, l);
        if (stride <= 1) return lo + l;
        lo += l * stride;
        n = min(stride, n - l * stride);
    }
}
#endif

// qh_kv8.hip
hipError_t launch_kv8_append(const Kv8View& c, const void* k, const void* v, int dtype, int64_t ldk, int64_t ldv,
                             const int32_t* start, const int32_t* seqs, int n, int n_tok, hipStream_t s);
hipError_t launch_kv8_read(const Kv8View& c, void* k, void* v, int dtype, int64_t ldk, int64_t ldv, const int32_t* start,
                           const int32_t* seqs, int n, int n_tok, hipStream_t s);
// A decode step's token, one f32 row of q, k and v as projected: bias and RoPE at position *pos (in q in place), and k and v
// stored as the last token of sequence *seq. cs: [ctx][head_dim / 2] cosines and sines; biases may be null.
struct Kv8Token {
    float* q;
    const float *k, *v, *bq, *bk, *bv, *cs;
    const int* pos;
    int ctx, n_heads;
};
hipError_t launch_kv8_append_token(const Kv8View& c, const Kv8Token& t, const int32_t* seq, hipStream_t s);
size_t kv8_pages_workspace_bytes(int n_pages, int n_seqs);
// pages: the first layer's; n_layers of them lie layer_bytes apart.
hipError_t launch_kv8_reset(const Kv8View& c, hipStream_t s);
hipError_t launch_kv8_resize(const Kv8View& c, int n_layers, const int32_t* seqs, const int32_t* lens, int n, void* ws,
                             hipStream_t s);
hipError_t launch_kv8_fork(const Kv8View& c, int n_layers, const int32_t* src, const int32_t* dst, int n, bool copy,
                           void* ws, hipStream_t s);
hipError_t launch_kv8_compact(const Kv8View& c, int n_layers, int32_t* live, void* ws, hipStream_t s);
// qh_kv8_attn.hip
// capacity: positions that a sequence can have. oq, od (one entry): the f32 rows of out (without gaps) in 8 bits too, as
// launch_quantize_q8 makes them.
size_t kv8_attention_workspace_bytes(int n_heads, int n_kv, int hd, int capacity, int n, int n_tok);
qh_kv8_plan kv8_attention_plan(int n_heads, int n_kv, int hd, int capacity, int n, int n_tok, bool single);
hipError_t launch_kv8_attention(const Kv8View& c, const void* q, void* out, int dtype, int n_heads, int64_t ldq,
                                int64_t ldo, const int32_t* start, const int32_t* seqs, int n, int n_tok, bool causal,
                                float scale, void* ws, hipStream_t s, int8_t* oq = nullptr, float* od = nullptr);

// The decoder over a bound cache (qh_decoder.hip): c is its layer 0, null to unbind.
struct Decoder;
const qh_model_desc& decoder_desc(const Decoder* d);
hipError_t decoder_bind_kv8(Decoder* d, const Kv8View* c, int seq);

}  // namespace qh
