// The 8-bit paged key / value cache (layout in qh_kv8.h): rows quantized into it, rows read back, and its pages (resize,
// fork, compact).
#include "qh_device.h"
#include "qh_kv8.h"

namespace qh {
namespace {

// ------------------------------------------------------------------------------------------- append and read back

__device__ __forceinline__ void load_row4(const float* p, float* x) {
    typedef float f4 __attribute__((ext_vector_type(4)));
    const f4 a = __builtin_nontemporal_load(reinterpret_cast<const f4*>(p));
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w;
}
__device__ __forceinline__ void load_row4(const _Float16* p, float* x) {
    typedef _Float16 h4 __attribute__((ext_vector_type(4)));
    const h4 a = __builtin_nontemporal_load(reinterpret_cast<const h4*>(p));
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = (float)a[j];
}
__device__ __forceinline__ void store_row4(float* p, const float* x) {
    *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
}
__device__ __forceinline__ void store_row4(_Float16* p, const float* x) {
    typedef _Float16 h4 __attribute__((ext_vector_type(4)));
    h4 a;
#pragma unroll
    for (int j = 0; j < 4; ++j) a[j] = (_Float16)x[j];
    *reinterpret_cast<h4*>(p) = a;
}

// Lane q of each aligned group of four takes word q of the four lanes: w[j] becomes lane j's w[q].
__device__ __forceinline__ void transpose_quad(uint32_t (&w)[4]) {
    const bool odd = (threadIdx.x & 1) != 0, high = (threadIdx.x & 2) != 0;
#pragma unroll
    for (int k = 0; k < 4; k += 2) {
        const uint32_t got = (uint32_t)__builtin_amdgcn_mov_dpp((int)(odd ? w[k] : w[k + 1]), 0xB1, 0xF, 0xF, false);
        w[k] = odd ? got : w[k];
        w[k + 1] = odd ? w[k + 1] : got;
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const uint32_t got = (uint32_t)__builtin_amdgcn_mov_dpp((int)(high ? w[k] : w[k + 2]), 0x4E, 0xF, 0xF, false);
        w[k] = high ? got : w[k];
        w[k + 2] = high ? w[k + 2] : got;
    }
}

// The integer nearest to (a + e) / d, halves upwards, for 0 <= (a + e) / d < 127.6 and |e| at most half an ulp of a: the
// candidate from the rounded reciprocal is at most one off, and the signs of the exact remainders at its two borders
// settle it. Each border product is exact inside the FMA; where the remainder is within d of zero it has at most 24 bits,
// so it is exact too and e joins it without loss, and where it is larger e cannot change its sign.
__device__ __forceinline__ float nearest_code(float a, float e, float d, float inv) {
    float k = __builtin_floorf(a * inv + 0.5f);
    const float up = __builtin_fmaf(-(k + 0.5f), d, a) + e;
    const float dn = __builtin_fmaf(-(k - 0.5f), d, a) + e;
    k = up >= 0.0f ? k + 1.0f : dn < 0.0f ? k - 1.0f : k;
    return __builtin_fminf(k, 127.0f);  // a scale that underflowed to few bits
}

__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
    return wave_reduce32x2(v, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
}

// One wave stores the new tokens of one block: the positions [first, len) of a sequence are new, the one at position p in
// row row0 + p. Bound by the memory traffic of long batches (each value read once, its code written once) and by the
// dependent loads (entry, length, page, scale, codes) of single tokens.
// Lane 16 g + j reads dims 4 j .. 4 j + 3 of tokens 4 g .. 4 g + 3, 16 lanes to a row, so that rows are read in one piece;
// the values' codes are in place then, the keys' cross four lanes. 24,001 x 8 heads of 128, f32: 62.6 us; with the rows read
// by the lanes that store them, 16 dims of one token, 71. Codes from the rounded quotient (below) 60.8, and rows loaded past
// the caches, which nothing reads again, 46.
// The block's scale is max|x| / 127 over every token it has been given since its first one: a block that already holds
// tokens (held > 0) keeps the larger of its scale and the new tokens', and its codes are rounded to the new scale where
// that grew. Only the block's own wave touches it, so the update needs no atomics.
template <typename T, int kC>
__device__ __forceinline__ void load_block(const T* __restrict__ x, int64_t ld, int pos0, int first, int len, int row0,
                                           float (&v)[kC][4][4]) {
    const int lane = (int)threadIdx.x & 63, g = lane >> 4, j = lane & 15;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int p = pos0 + 4 * g + r;
        const bool there = p >= first && p < len;
        const T* row = x + (int64_t)(row0 + (there ? p : first)) * ld + 4 * j;
#pragma unroll
        for (int k = 0; k < kC; ++k) load_row4(row + 64 * k, v[k][r]);
    }
}

template <int kC, bool kValues>
__device__ __forceinline__ void append_block(const Kv8View& c, float (&v)[kC][4][4], int h, int page, int blk_in_page, int pos0,
                                             int first, int len) {
    const int lane = (int)threadIdx.x & 63, g = lane >> 4, j = lane & 15;
    const int held = min(max(first - pos0, 0), kBlk);
    // the 16 bytes that this lane stores: values where it reads them, keys of token 4 g + j % 4 and dims 16 (j / 4) ..
    const int unit = kValues ? lane : 16 * (j >> 2) + 4 * g + (j & 3);
    uint4* codes = reinterpret_cast<uint4*>(kv8_codes(c, page, kValues ? 1 : 0, h, blk_in_page)) + unit;
    float* scale = kv8_scale(c, page, kValues ? 1 : 0, h, blk_in_page);
    const float before = held ? __builtin_fabsf(*scale) : 0.0f;
    uint4 old[kC];
    if (held) {
#pragma unroll
        for (int k = 0; k < kC; ++k) old[k] = codes[64 * k];
    }
    uint32_t top = 0;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int p = pos0 + 4 * g + r;
        const bool there = p >= first && p < len;
#pragma unroll
        for (int k = 0; k < kC; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (!there) v[k][r][i] = 0.0f;
                top = max(top, __builtin_bit_cast(uint32_t, v[k][r][i]) & 0x7fffffffu);
            }
    }
    top = wave_max_u32(top);  // on the bits, so that a NaN is not lost
    float d = __builtin_bit_cast(float, top) / 127.0f;
    // an infinity or a NaN leaves no scale for the other tokens: the block reads as NaN, never as something plausible
    if (top >= 0x7f800000u || before != before) d = __builtin_nanf("");
    else d = __builtin_fmaxf(d, before);
    // scales near the end of the range are moved up by an exact power of two, so that the reciprocal and remainders are
    // normal numbers
    const float lift = d < 0x1p-100f ? 0x1p64f : 1.0f;
    const float ds = d * lift, inv = d > 0.0f ? 1.0f / ds : 0.0f;  // 0 for d = 0 and for NaN: every code 0
    const float db = before * lift;
    // Codes from the rounded quotient, stored with their bias by the conversion itself. The quotient is off by at most
    // 127 * 2^-23 < 2^-16, so a code is certain unless the quotient is that close to a half; a wave with such a value (one
    // in twenty at 2,048 values) or a lifted scale takes every code again by the exact remainders.
    uint32_t w[kC][4] = {};
    float worst = 0.0f;
#pragma unroll
    for (int k = 0; k < kC; ++k)
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float t = v[k][r][i] * inv, q = __builtin_truncf(t + __builtin_copysignf(0.5f, t));
                worst = __builtin_fmaxf(worst, __builtin_fabsf(t - q));
                w[k][kValues ? i : r] = __builtin_amdgcn_cvt_pk_u8_f32(q + 128.0f, kValues ? r : i, w[k][kValues ? i : r]);
            }
    if (__any(!(worst <= 0.5f - 0x1p-16f)) || lift != 1.0f || !(inv > 0.0f)) {
#pragma unroll
        for (int k = 0; k < kC; ++k)
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float q = 0.0f;
                    if (inv > 0.0f) q = nearest_code(__builtin_fabsf(v[k][r][i] * lift), 0.0f, ds, inv);
                    w[k][kValues ? i : r] = __builtin_amdgcn_cvt_pk_u8_f32(__builtin_copysignf(q, v[k][r][i]) + 128.0f,
                                                                          kValues ? r : i, w[k][kValues ? i : r]);
                }
    }
#pragma unroll
    for (int k = 0; k < kC; ++k) {
        if (!kValues) transpose_quad(w[k]);
        if (held) {
            const uint32_t o[4] = {old[k].x ^ kBias, old[k].y ^ kBias, old[k].z ^ kBias, old[k].w ^ kBias};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint32_t keep = o[i];
                if (d != before) {
                    keep = 0;
                    if (inv > 0.0f) {
#pragma unroll
                        for (int b = 0; b < 4; ++b) {
                            const float f = (float)(int8_t)(o[i] >> (8 * b)), m = __builtin_fabsf(f);
                            const float a = m * db, e = __builtin_fmaf(m, db, -a);
                            keep |= ((uint32_t)(int)__builtin_copysignf(nearest_code(a, e, ds, inv), f) & 0xffu) << (8 * b);
                        }
                    }
                }
                uint32_t mask = 0;  // the bytes of tokens the block held: byte b of values is token 4 g + b
#pragma unroll
                for (int b = 0; b < 4; ++b) mask |= 4 * g + (kValues ? b : j & 3) < held ? 0xffu << (8 * b) : 0u;
                w[k][i] = ((keep ^ kBias) & mask) | (w[k][i] & ~mask);
            }
        }
        codes[64 * k] = make_uint4(w[k][0], w[k][1], w[k][2], w[k][3]);
    }
    if constexpr (kValues) {  // the sign: a token of the block has only zeros
        uint32_t any = 0;     // byte b: of token 4 g + b
#pragma unroll
        for (int k = 0; k < kC; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i) any |= w[k][i] ^ kBias;
        any = or_row16(any);
        bool none = false;
#pragma unroll
        for (int b = 0; b < 4; ++b) none |= pos0 + 4 * g + b < len && ((any >> (8 * b)) & 0xffu) == 0;
        if (__any(none) && d > 0.0f) d = -d;
    }
    if (lane == 0) *scale = d;
}

// An entry's share of the cache: row0 + p is the row of position p, the positions [first, len) are its own.
struct Span {
    int seq, first, len, row0;
};
__device__ __forceinline__ Span span_of(const Kv8View& c, const Kv8Batch& q, int b) {
    const int seq = q.seq(b), s0 = q.at(b), s1 = max(s0, q.at(b + 1));
    if (seq < 0 || seq >= c.n_seqs) return {0, 0, 0, 0};
    const int len = kv8_len(c, seq), p0 = len - (s1 - s0);  // p0 < 0: rows before the first position have no place
    return {seq, max(p0, 0), len, s0 - p0};
}

// One wave per block of 16 positions, KV head, keys or values; the workgroups (4 waves) of one block follow each other, so
// that a row's heads are read at about the same time.
template <typename T, int kC>
__global__ __launch_bounds__(256) void kv8_append_kernel(Kv8View c, const T* __restrict__ k, const T* __restrict__ v,
                                                         int64_t ldk, int64_t ldv, Kv8Batch q) {
    const unsigned groups = (unsigned)(2 * c.n_kv + 3) / 4;
    const int item = (int)(blockIdx.x / groups), hw = (int)(blockIdx.x % groups) * 4 + (int)(threadIdx.x >> 6);
    int b = item, from = item;
    if (q.start) b = kv8_entry_of(q, item, 1, kBlk, 2, &from);
    if (b < 0 || hw >= 2 * c.n_kv) return;
    const Span sp = span_of(c, q, b);
    const int blk = sp.first / kBlk + (item - from), pos0 = blk * kBlk;
    if (max(pos0, sp.first) >= sp.len) return;
    const int h = hw >> 1;
    const bool values = (hw & 1) != 0;
    float x[kC][4][4];  // [.][token][dim]; in flight while the page is looked up
    load_block<T, kC>((values ? v : k) + (int64_t)h * c.hd, values ? ldv : ldk, pos0, sp.first, sp.len, sp.row0, x);
    const int page = c.table[(size_t)sp.seq * c.seq_pages + (pos0 >> c.page_shift)];
    if (page < 0 || page >= c.n_pages) return;
    if (c.refs[page] > 1) {  // other sequences read this page
        if ((threadIdx.x & 63) == 0) atomicOr(c.status, QH_KV8_SHARED);
        return;
    }
    const int bp = blk & ((1 << (c.page_shift - 4)) - 1);
    if (values)
        append_block<kC, true>(c, x, h, page, bp, pos0, sp.first, sp.len);
    else
        append_block<kC, false>(c, x, h, page, bp, pos0, sp.first, sp.len);
}

// A decode step's token: the waves of append, which first add the bias and rotate their key row, and behind them workgroups
// that do so to the query heads in place: the decoder's rotation of many tokens in its order, with a launch less to a layer.
template <int kC>
__global__ __launch_bounds__(256) void kv8_append_token_kernel(Kv8View c, Kv8Token t, const int32_t* __restrict__ seqs) {
    constexpr int kHd = 64 * kC, kHalf = kHd / 2;
    const unsigned groups = (unsigned)(2 * c.n_kv + 3) / 4;
    const int pos = *t.pos;
    if (pos < 0 || pos >= t.ctx) return;
    const float* cs = t.cs + (size_t)pos * kHd;
    if (blockIdx.x >= groups) {
        const int e = (int)(blockIdx.x - groups) * 256 + (int)threadIdx.x, h = e / kHalf, i = e % kHalf;
        if (h >= t.n_heads) return;
        float *row = t.q + (size_t)h * kHd, a = row[i], b = row[i + kHalf];
        if (t.bq) {
            a = a + t.bq[h * kHd + i];
            b = b + t.bq[h * kHd + i + kHalf];
        }
        const float co = cs[2 * i], sn = cs[2 * i + 1];
        row[i] = __builtin_fmaf(a, co, -(b * sn));
        row[i + kHalf] = __builtin_fmaf(b, co, a * sn);
        return;
    }
    const int hw = (int)blockIdx.x * 4 + (int)(threadIdx.x >> 6), h = hw >> 1, j = (int)threadIdx.x & 15;
    if (hw >= 2 * c.n_kv) return;
    const bool values = (hw & 1) != 0;
    const float *row = (values ? t.v : t.k) + h * kHd + 4 * j, *bias = values ? t.bv : t.bk;
    float x[kC][4];
#pragma unroll
    for (int k = 0; k < kC; ++k) {
        const float4 r = *reinterpret_cast<const float4*>(row + 64 * k);
        x[k][0] = r.x, x[k][1] = r.y, x[k][2] = r.z, x[k][3] = r.w;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (bias) x[k][i] = x[k][i] + bias[h * kHd + 64 * k + 4 * j + i];
    }
    if (!values) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int d = (4 * j + i) % kHalf;
            const float co = cs[2 * d], sn = cs[2 * d + 1];
            if constexpr (kC == 2) {
                const float a = x[0][i], b = x[1][i];
                x[0][i] = __builtin_fmaf(a, co, -(b * sn));
                x[1][i] = __builtin_fmaf(b, co, a * sn);
            } else {  // the other half is eight lanes away
                const float mine = x[0][i], other = __shfl_xor(mine, 8);
                x[0][i] = j < 8 ? __builtin_fmaf(mine, co, -(other * sn)) : __builtin_fmaf(mine, co, other * sn);
            }
        }
    }
    const Span sp = span_of(c, Kv8Batch{nullptr, seqs, 1, 1, 0}, 0);
    const int blk = sp.first / kBlk, pos0 = blk * kBlk;
    if (sp.first >= sp.len) return;
    const int page = c.table[(size_t)sp.seq * c.seq_pages + (pos0 >> c.page_shift)];
    if (page < 0 || page >= c.n_pages) return;
    if (c.refs[page] > 1) {
        if ((threadIdx.x & 63) == 0) atomicOr(c.status, QH_KV8_SHARED);
        return;
    }
    float rows[kC][4][4];  // append_block takes the one that is the new token's
#pragma unroll
    for (int k = 0; k < kC; ++k)
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int i = 0; i < 4; ++i) rows[k][r][i] = x[k][i];
    const int bp = blk & ((1 << (c.page_shift - 4)) - 1);
    if (values)
        append_block<kC, true>(c, rows, h, page, bp, pos0, sp.first, sp.len);
    else
        append_block<kC, false>(c, rows, h, page, bp, pos0, sp.first, sp.len);
}

// The same items: one wave writes the values of one block's tokens, code * scale rounded to f32, then to T. Lanes as in
// append_block.
template <typename T, int kC>
__global__ __launch_bounds__(256) void kv8_read_kernel(Kv8View c, T* __restrict__ k, T* __restrict__ v, int64_t ldk,
                                                       int64_t ldv, Kv8Batch q) {
    const unsigned groups = (unsigned)(2 * c.n_kv + 3) / 4;
    const int item = (int)(blockIdx.x / groups), hw = (int)(blockIdx.x % groups) * 4 + (int)(threadIdx.x >> 6);
    const int lane = (int)threadIdx.x & 63, g = lane >> 4, j = lane & 15;
    int b = item, from = item;
    if (q.start) b = kv8_entry_of(q, item, 1, kBlk, 2, &from);
    if (b < 0 || hw >= 2 * c.n_kv) return;
    const Span sp = span_of(c, q, b);
    const int blk = sp.first / kBlk + (item - from), pos0 = blk * kBlk, h = hw >> 1;
    if (max(pos0, sp.first) >= sp.len) return;
    const int page = c.table[(size_t)sp.seq * c.seq_pages + (pos0 >> c.page_shift)];
    const bool ok = page >= 0 && page < c.n_pages, values = (hw & 1) != 0;  // a missing page reads as zeros
    const int bp = blk & ((1 << (c.page_shift - 4)) - 1);
    const float d = ok ? __builtin_fabsf(*kv8_scale(c, page, hw & 1, h, bp)) : 0.0f;
    const uint4* codes = reinterpret_cast<const uint4*>(kv8_codes(c, ok ? page : 0, hw & 1, h, bp)) +
                         (values ? lane : 16 * (j >> 2) + 4 * g + (j & 3));
    T* out = values ? v : k;
    const int64_t ld = values ? ldv : ldk;
#pragma unroll
    for (int kk = 0; kk < kC; ++kk) {
        const uint4 w4 = ok ? codes[64 * kk] : make_uint4(kBias, kBias, kBias, kBias);
        uint32_t w[4] = {w4.x ^ kBias, w4.y ^ kBias, w4.z ^ kBias, w4.w ^ kBias};
        if (!values) transpose_quad(w);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int p = pos0 + 4 * g + r;
            float x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = (float)(int8_t)(values ? w[i] >> (8 * r) : w[r] >> (8 * i)) * d;
            if (p >= sp.first && p < sp.len)
                store_row4(out + (int64_t)(sp.row0 + p) * ld + (int64_t)h * c.hd + 64 * kk + 4 * j, x);
        }
    }
}

// ------------------------------------------------------------------------------------------------------- pages

constexpr int kWg = 1024;  // the planning kernels: one workgroup, so that page numbers come out in one order

// The planning kernels' results for the kernels that follow, in the caller's workspace.
struct PagesWs {
    int* n_copy;     // pages to copy
    int* ok;         // 0: the call was refused and nothing is to be done
    int2* copies;    // [n_pages] (from, to)
    int* goes;       // [n_pages] a page's new number (compact)
    int* free_list;  // [n_pages] free pages in order (resize, fork); the page numbers that move (compact)
    int* first;      // [n_seqs + 1] pages the list entries before this one take
    int* split;      // [n_seqs] 1: the entry's last page is to be replaced by a copy
};
__host__ __device__ __forceinline__ PagesWs pages_ws(void* ws, int n_pages, int n_seqs) {
    int* p = static_cast<int*>(ws);
    PagesWs w;
    w.n_copy = p;
    w.ok = p + 1;
    w.copies = reinterpret_cast<int2*>(p + 4);
    w.goes = p + 4 + 2 * (size_t)n_pages;
    w.free_list = w.goes + n_pages;
    w.first = w.free_list + n_pages;
    w.split = w.first + n_seqs + 1;
    return w;
}

__device__ __forceinline__ int load_ref(const int32_t* refs, int i) {  // after atomics of this launch: from the L2
    return __hip_atomic_load(refs + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Exclusive prefix sum of v over the workgroup's kWg threads; *total their sum. Every thread calls it.
__device__ __forceinline__ int scan_wg(int v, int* total) {
    __shared__ int sums[kWg / 64];
    const int lane = (int)threadIdx.x & 63, w = (int)threadIdx.x >> 6;
    int x = v;
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
        const int y = __shfl_up(x, s);
        x += lane >= s ? y : 0;
    }
    __syncthreads();  // the sums of an earlier call have been read
    if (lane == 63) sums[w] = x;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int i = 0; i < kWg / 64; ++i) {
        before += i < w ? sums[i] : 0;
        all += sums[i];
    }
    *total = all;
    return before + x - v;
}

// The first `want` free pages in order into list; returns how many there are (fewer where the pool has fewer).
__device__ int find_free(const int32_t* refs, int n_pages, int want, int* list) {
    int have = 0;
    for (int base = 0; base < n_pages && have < want; base += 4 * kWg) {
        const int i = base + 4 * (int)threadIdx.x;
        bool f[4];
        int c = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            f[j] = i + j < n_pages && load_ref(refs, i + j) == 0;
            c += f[j];
        }
        int total, at = have + scan_wg(c, &total);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (f[j] && at < want) list[at] = i + j;
            at += f[j];
        }
        have += total;
    }
    return have;
}

// The list entry that takes page t of the pages the entries take together: the last i with first[i] <= t among n.
__device__ __forceinline__ int taker(const int* first, int n, int t) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (first[mid] <= t) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

__device__ __forceinline__ int pages_of(const Kv8View& c, int tokens) {
    return (int)(((long)tokens + (1 << c.page_shift) - 1) >> c.page_shift);
}

// One reference less for the pages [from, to) of a sequence's table row, by one wave.
__device__ __forceinline__ void drop_pages(const Kv8View& c, int seq, int from, int to) {
    int32_t* row = c.table + (size_t)seq * c.seq_pages;
    for (int j = from + ((int)threadIdx.x & 63); j < to; j += 64) {
        const int page = row[j];
        if (page >= 0 && page < c.n_pages) atomicSub(&c.refs[page], 1);
        row[j] = -1;
    }
}

// A sequence number once in a list: sets its bit in seen (LDS, zeroed), false when it was set or is out of range.
__device__ __forceinline__ bool first_seen(uint32_t* seen, int seq, int n_seqs) {
    if (seq < 0 || seq >= n_seqs) return false;
    const uint32_t bit = 1u << (seq & 31);
    return (atomicOr(&seen[seq >> 5], bit) & bit) == 0;
}

__global__ __launch_bounds__(256) void kv8_reset_kernel(Kv8View c) {
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (i < (size_t)c.n_seqs * c.seq_pages) c.table[i] = -1;
    if (i < (size_t)c.n_pages) c.refs[i] = 0;
    if (i < (size_t)c.n_seqs) c.lens[i] = 0;
    if (i == 0) *c.status = 0;
}

// New lengths: first the pages that shorter sequences give back, then the pages that longer ones need, all of them or
// none: the lowest free numbers, in the list's order, a sequence's replaced last page first. One workgroup: the work is a
// pass over the counts (4 bytes a page) and over the table entries that change, and its order is the result.
__global__ __launch_bounds__(kWg) void kv8_resize_kernel(Kv8View c, const int32_t* __restrict__ seqs,
                                                         const int32_t* __restrict__ want, int n, void* ws) {
    __shared__ uint32_t seen[QH_KV8_MAX_SEQS / 32];
    __shared__ int n_split;
    const PagesWs w = pages_ws(ws, c.n_pages, c.n_seqs);
    const int tid = (int)threadIdx.x, cap = c.seq_pages << c.page_shift;
    for (int i = tid; i < (c.n_seqs + 31) / 32; i += kWg) seen[i] = 0;
    if (tid == 0) {
        *w.n_copy = 0;
        n_split = 0;
    }
    __syncthreads();
    int bad = 0;
    for (int i = tid; i < n; i += kWg) bad |= !first_seen(seen, seqs[i], c.n_seqs) || want[i] < 0 || want[i] > cap;
    if (__syncthreads_or(bad)) {
        if (tid == 0) atomicOr(c.status, QH_KV8_BAD_LIST);
        return;
    }
    for (int i = tid >> 6; i < n; i += kWg / 64) {
        const int s = seqs[i], before = pages_of(c, kv8_len(c, s)), after = pages_of(c, want[i]);
        drop_pages(c, s, after, before);
    }
    __syncthreads();
    int need_all = 0;
    for (int base = 0; base < n; base += kWg) {
        const int i = base + tid;
        int need = 0, split = 0;
        if (i < n) {
            const int s = seqs[i], len = kv8_len(c, s), before = pages_of(c, len);
            if (want[i] > len) {
                if (len & ((1 << c.page_shift) - 1)) {
                    const int page = c.table[(size_t)s * c.seq_pages + before - 1];
                    split = page >= 0 && page < c.n_pages && load_ref(c.refs, page) > 1;
                }
                need = pages_of(c, want[i]) - before + split;
            } else {
                c.lens[s] = want[i];  // no later step reads this sequence's old length
            }
        }
        int total;
        const int at = need_all + scan_wg(need, &total);
        if (i < n) {
            w.first[i] = at;
            w.split[i] = split;
        }
        need_all += total;
    }
    __syncthreads();
    if (need_all > 0) {
        if (find_free(c.refs, c.n_pages, need_all, w.free_list) < need_all) {  // the same for every thread
            if (tid == 0) atomicOr(c.status, QH_KV8_NO_PAGES);
            return;
        }
        __syncthreads();
        for (int t = tid; t < need_all; t += kWg) {
            const int i = taker(w.first, n, t), s = seqs[i], k = t - w.first[i], split = w.split[i], page = w.free_list[t];
            const int before = pages_of(c, kv8_len(c, s));
            int32_t* slot = c.table + (size_t)s * c.seq_pages + before - split + k;
            if (k == 0 && split) {
                const int old = *slot;
                w.copies[atomicAdd(&n_split, 1)] = make_int2(old, page);
                atomicSub(&c.refs[old], 1);
            }
            *slot = page;
            c.refs[page] = 1;
        }
        __syncthreads();
    }
    for (int i = tid; i < n; i += kWg) c.lens[seqs[i]] = want[i];
    if (tid == 0) *w.n_copy = n_split;
}

// dst[i] becomes a fork of src[i]: dst's pages are given back, then (copy) it takes as many pages as src has, to be
// filled by kv8_move_kernel, or shares src's: entry by entry here (mode kShareHere), or in kv8_share_kernel on the whole GPU
// where the table rows are many.
enum { kShareLater, kShareHere, kCopy };
__device__ __forceinline__ void share_page(const Kv8View& c, int src, int dst, int j);
__global__ __launch_bounds__(kWg) void kv8_fork_kernel(Kv8View c, const int32_t* __restrict__ src,
                                                       const int32_t* __restrict__ dst, int n, int mode, void* ws) {
    __shared__ uint32_t seen[QH_KV8_MAX_SEQS / 32];
    const PagesWs w = pages_ws(ws, c.n_pages, c.n_seqs);
    const int tid = (int)threadIdx.x;
    for (int i = tid; i < (c.n_seqs + 31) / 32; i += kWg) seen[i] = 0;
    if (tid == 0) {
        *w.n_copy = 0;
        *w.ok = 0;
    }
    __syncthreads();
    int bad = 0;
    for (int i = tid; i < n; i += kWg) bad |= !first_seen(seen, dst[i], c.n_seqs);
    __syncthreads();
    for (int i = tid; i < n; i += kWg) {
        const int s = src[i];
        bad |= s < 0 || s >= c.n_seqs || ((seen[s >> 5] >> (s & 31)) & 1u) != 0;
    }
    if (__syncthreads_or(bad)) {
        if (tid == 0) atomicOr(c.status, QH_KV8_BAD_LIST);
        return;
    }
    for (int i = tid >> 6; i < n; i += kWg / 64) drop_pages(c, dst[i], 0, pages_of(c, kv8_len(c, dst[i])));
    __syncthreads();
    if (mode != kCopy) {
        if (mode == kShareHere)
            for (int t = tid; t < n * c.seq_pages; t += kWg) share_page(c, src[t / c.seq_pages], dst[t / c.seq_pages], t % c.seq_pages);
        for (int i = tid; i < n; i += kWg) c.lens[dst[i]] = kv8_len(c, src[i]);
        if (tid == 0) *w.ok = 1;
        return;
    }
    int need_all = 0;
    for (int base = 0; base < n; base += kWg) {
        const int i = base + tid;
        int total;
        const int at = need_all + scan_wg(i < n ? pages_of(c, kv8_len(c, src[i])) : 0, &total);
        if (i < n) w.first[i] = at;
        need_all += total;
    }
    __syncthreads();
    const int have = need_all > 0 ? find_free(c.refs, c.n_pages, need_all, w.free_list) : 0;
    const bool ok = have >= need_all;
    __syncthreads();
    for (int t = tid; ok && t < need_all; t += kWg) {
        const int i = taker(w.first, n, t), j = t - w.first[i], page = w.free_list[t];
        const int from = c.table[(size_t)src[i] * c.seq_pages + j];
        w.copies[t] = make_int2(from, page);
        c.table[(size_t)dst[i] * c.seq_pages + j] = page;
        c.refs[page] = 1;
    }
    for (int i = tid; i < n; i += kWg) c.lens[dst[i]] = ok ? kv8_len(c, src[i]) : 0;
    if (tid == 0) {
        *w.n_copy = ok ? need_all : 0;
        if (!ok) atomicOr(c.status, QH_KV8_NO_PAGES);
    }
}

// Table entry j of a shared fork: src's page, which has one reference more then.
__device__ __forceinline__ void share_page(const Kv8View& c, int src, int dst, int j) {
    if (j >= pages_of(c, kv8_len(c, src))) return;
    const int page = c.table[(size_t)src * c.seq_pages + j];
    c.table[(size_t)dst * c.seq_pages + j] = page;
    if (page >= 0 && page < c.n_pages) atomicAdd(&c.refs[page], 1);
}
__global__ __launch_bounds__(256) void kv8_share_kernel(Kv8View c, const int32_t* __restrict__ src,
                                                        const int32_t* __restrict__ dst, int n, void* ws) {
    if (*pages_ws(ws, c.n_pages, c.n_seqs).ok == 0) return;
    share_page(c, src[blockIdx.y], dst[blockIdx.y], (int)(blockIdx.x * 256 + threadIdx.x));
}

// Which pages move: of L live pages those numbered L and above go, in order, to the free numbers below L, so sources and
// destinations never meet.
__global__ __launch_bounds__(kWg) void kv8_compact_kernel(Kv8View c, int32_t* __restrict__ live, void* ws) {
    const PagesWs w = pages_ws(ws, c.n_pages, c.n_seqs);
    const int tid = (int)threadIdx.x;
    int mine = 0, n_live;
    for (int i = tid; i < c.n_pages; i += kWg) mine += c.refs[i] > 0;
    scan_wg(mine, &n_live);
    // free numbers below n_live into free_list, live pages from it on into `goes` (by rank; the copies pair them)
    int holes = 0, high = 0;
    for (int base = 0; base < c.n_pages; base += kWg) {
        const int i = base + tid;
        const bool is_live = i < c.n_pages && c.refs[i] > 0;
        const bool hole = i < n_live && !is_live, up = i >= n_live && is_live;
        int total;
        const int at = scan_wg((int)hole | ((int)up << 16), &total);
        if (hole) w.free_list[holes + (at & 0xffff)] = i;
        if (up) w.copies[high + (at >> 16)].x = i;
        holes += total & 0xffff;
        high += total >> 16;
    }
    __syncthreads();
    for (int i = n_live + tid; i < c.n_pages; i += kWg) w.goes[i] = i;
    __syncthreads();
    for (int r = tid; r < high; r += kWg) {
        const int from = w.copies[r].x, to = w.free_list[r];
        w.copies[r].y = to;
        w.goes[from] = to;
        c.refs[to] = c.refs[from];
        c.refs[from] = 0;
    }
    if (tid == 0) {
        *w.n_copy = high;
        if (live) *live = n_live;
    }
}

// Copies the listed pages in every layer. All pages of all layers lie end to end as 16-byte words, and a workgroup takes
// kPer of 256 of them at a time, wherever pages end, so that every lane has kPer loads in flight whatever a page's size
// is; remap (compact): first the table entries take the pages' new numbers. Bound by memory (large lists) and by the two
// dependent reads of the list (a page or two).
template <int kPer>
__global__ __launch_bounds__(256) void kv8_move_kernel(Kv8View c, int n_layers, int remap, void* ws) {
    const PagesWs w = pages_ws(ws, c.n_pages, c.n_seqs);
    const int n = *w.n_copy;
    if (n == 0) return;
    if (remap) {
        // the first copy's source is the lowest number that moves; `goes` holds every number from it on
        const int first = w.copies[0].x;
        for (size_t e = (size_t)blockIdx.x * 256 + threadIdx.x; e < (size_t)c.n_seqs * c.seq_pages;
             e += (size_t)gridDim.x * 256) {
            const int page = c.table[e];
            if (page >= first && page < c.n_pages) c.table[e] = w.goes[page];
        }
    }
    const uint32_t words = (uint32_t)(c.page_bytes / 16);
    const uint64_t total = (uint64_t)n * n_layers * words;
    for (uint64_t base = (uint64_t)blockIdx.x * (256 * kPer); base < total; base += (uint64_t)gridDim.x * (256 * kPer)) {
        // the page of the first word, copy by copy with the layers in turn
        const uint64_t item = base / words;
        const uint32_t copy0 = (uint32_t)(item / (uint32_t)n_layers), layer0 = (uint32_t)(item % (uint32_t)n_layers);
        const uint32_t off0 = (uint32_t)(base - item * words);
        uint4 r[kPer];
        uint4* to[kPer];
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            uint32_t off = off0 + threadIdx.x + 256 * j, copy = copy0, layer = layer0;
            while (off >= words) {
                off -= words;
                if (++layer == (uint32_t)n_layers) {
                    layer = 0;
                    ++copy;
                }
            }
            to[j] = nullptr;
            if (copy < (uint32_t)n) {
                const int2 p = w.copies[copy];
                if (p.x >= 0 && p.x < c.n_pages) {
                    uint8_t* at = c.pages + (size_t)layer * c.n_pages * c.page_bytes;
                    r[j] = load_once(reinterpret_cast<const uint4*>(at + (size_t)p.x * c.page_bytes) + off);
                    to[j] = reinterpret_cast<uint4*>(at + (size_t)p.y * c.page_bytes) + off;
                }
            }
        }
#pragma unroll
        for (int j = 0; j < kPer; ++j)
            if (to[j]) *to[j] = r[j];
    }
}

hipError_t launch_move(const Kv8View& c, int n_layers, long most_copies, bool remap, void* ws, hipStream_t s) {
    // one word to a lane up to 2,048 workgroups of them, else four
    const uint64_t words = (uint64_t)most_copies * n_layers * (c.page_bytes / 16);
    const bool few = words <= (uint64_t)2048 * 256;
    uint64_t grid = (words + (few ? 255 : 1023)) / (few ? 256 : 1024);
    if (remap && grid < 64) grid = 64;
    if (grid > 2048) grid = 2048;
    if (few)
        qh_launch((kv8_move_kernel<1>), dim3((unsigned)grid), dim3(256), 0, s, c, n_layers, remap ? 1 : 0, ws);
    else
        qh_launch((kv8_move_kernel<4>), dim3((unsigned)grid), dim3(256), 0, s, c, n_layers, remap ? 1 : 0, ws);
    return hipGetLastError();
}

// Calls f with the element type and head_dim / 64 of a call.
template <typename F>
hipError_t by_type(int dtype, int hd, F&& f) {
    using std::integral_constant;
    if (dtype == QH_F32 && hd == 64) f((float*)nullptr, integral_constant<int, 1>{});
    else if (dtype == QH_F32 && hd == 128) f((float*)nullptr, integral_constant<int, 2>{});
    else if (dtype == QH_F16 && hd == 64) f((_Float16*)nullptr, integral_constant<int, 1>{});
    else if (dtype == QH_F16 && hd == 128) f((_Float16*)nullptr, integral_constant<int, 2>{});
    else return hipErrorInvalidValue;
    return hipGetLastError();
}

// Blocks that a batch's entries can touch: an entry of m rows at any offset touches at most floor(m / 16) + 2.
unsigned block_items(const int32_t* start, int n, int n_tok) {
    return start ? (unsigned)(n_tok / kBlk + 2 * n) : (unsigned)n;
}

}  // namespace

hipError_t launch_kv8_append(const Kv8View& c, const void* k, const void* v, int dtype, int64_t ldk, int64_t ldv,
                             const int32_t* start, const int32_t* seqs, int n, int n_tok, hipStream_t s) {
    const dim3 grid(block_items(start, n, n_tok) * (unsigned)((2 * c.n_kv + 3) / 4));
    return by_type(dtype, c.hd, [&](auto* t, auto kc) {
        using T = std::remove_pointer_t<decltype(t)>;
        qh_launch((kv8_append_kernel<T, decltype(kc)::value>), grid, dim3(256), 0, s, c, (const T*)k, (const T*)v, ldk,
                  ldv, Kv8Batch{start, seqs, n, n_tok, 0});
    });
}

hipError_t launch_kv8_append_token(const Kv8View& c, const Kv8Token& t, const int32_t* seq, hipStream_t s) {
    const dim3 grid((unsigned)(2 * c.n_kv + 3) / 4 + (unsigned)(t.n_heads * (c.hd / 2) + 255) / 256);
    if (c.hd == 64) qh_launch((kv8_append_token_kernel<1>), grid, dim3(256), 0, s, c, t, seq);
    else qh_launch((kv8_append_token_kernel<2>), grid, dim3(256), 0, s, c, t, seq);
    return hipGetLastError();
}

hipError_t launch_kv8_read(const Kv8View& c, void* k, void* v, int dtype, int64_t ldk, int64_t ldv, const int32_t* start,
                           const int32_t* seqs, int n, int n_tok, hipStream_t s) {
    const dim3 grid(block_items(start, n, n_tok) * (unsigned)((2 * c.n_kv + 3) / 4));
    return by_type(dtype, c.hd, [&](auto* t, auto kc) {
        using T = std::remove_pointer_t<decltype(t)>;
        qh_launch((kv8_read_kernel<T, decltype(kc)::value>), grid, dim3(256), 0, s, c, (T*)k, (T*)v, ldk, ldv,
                  Kv8Batch{start, seqs, n, n_tok, 0});
    });
}

size_t kv8_pages_workspace_bytes(int n_pages, int n_seqs) {
    return sizeof(int) * (4 + 4 * (size_t)n_pages + 2 * (size_t)n_seqs + 1);
}

hipError_t launch_kv8_reset(const Kv8View& c, hipStream_t s) {
    size_t most = (size_t)c.n_seqs * c.seq_pages;
    most = most > (size_t)c.n_pages ? most : (size_t)c.n_pages;
    qh_launch(kv8_reset_kernel, dim3((unsigned)((most + 255) / 256)), dim3(256), 0, s, c);
    return hipGetLastError();
}

hipError_t launch_kv8_resize(const Kv8View& c, int n_layers, const int32_t* seqs, const int32_t* lens, int n, void* ws,
                             hipStream_t s) {
    qh_launch(kv8_resize_kernel, dim3(1), dim3(kWg), 0, s, c, seqs, lens, n, ws);
    if (hipError_t e = hipGetLastError()) return e;
    return launch_move(c, n_layers, n, false, ws, s);
}

hipError_t launch_kv8_fork(const Kv8View& c, int n_layers, const int32_t* src, const int32_t* dst, int n, bool copy,
                           void* ws, hipStream_t s) {
    // up to 2,048 table entries in the planning workgroup (16 forks of 128 pages: 5.9 us, with a second launch 6.8; of 256
    // pages 8.8 and 7.5; 4 of 16: 3.5 and 5.4)
    const int mode = copy ? kCopy : (int64_t)n * c.seq_pages <= 2048 ? kShareHere : kShareLater;
    qh_launch(kv8_fork_kernel, dim3(1), dim3(kWg), 0, s, c, src, dst, n, mode, ws);
    if (hipError_t e = hipGetLastError()) return e;
    if (copy) return launch_move(c, n_layers, c.n_pages, false, ws, s);
    if (mode == kShareHere) return hipSuccess;
    qh_launch(kv8_share_kernel, dim3((unsigned)((c.seq_pages + 255) / 256), (unsigned)n), dim3(256), 0, s, c, src, dst, n,
              ws);
    return hipGetLastError();
}

hipError_t launch_kv8_compact(const Kv8View& c, int n_layers, int32_t* live, void* ws, hipStream_t s) {
    qh_launch(kv8_compact_kernel, dim3(1), dim3(kWg), 0, s, c, live, ws);
    if (hipError_t e = hipGetLastError()) return e;
    return launch_move(c, n_layers, c.n_pages, true, ws, s);
}

}  // namespace qh
