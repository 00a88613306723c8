// Attention over the 8-bit paged key / value cache (layout in qh_kv8.h).
//
// For query row q of a head and the positions j it sees:  o = sum_j e_j d_j v_j / sum_j e_j,  e_j = 2^(x_j - base),
// x_j = (q . k_j) c_j scale log2(e), with k_j, v_j the integer codes and c_j, d_j the scales of their blocks. One pass
// over the cache with a running base (the same in both sums) and sum: 64 positions (a tile) at a time, in f32.
//
// Both products run on the f16 matrix instructions (16 x 16 x 32): a code in [-127, 127] is exact in f16, so a tile's
// codes become f16 operands (four instructions for four of them) and the block scales are applied to the scores and to
// the weights, whose tokens a lane holds next to each other. Scores are computed transposed (codes . queries), so that a
// lane's weights are already the operand of the second product (values . weights, transposed too): no weight passes
// through shared memory, and a row's maximum and sum belong to one lane column.
//   f32 queries are split into two f16 (22 bits), scaled by a power of two so that the row's largest value has exponent
//   13: what the split drops is at most 2^-22 of a value or, in f16's subnormals, 2^-38 of the row's largest, about what f32
//   sums round off. Weights are split too, but for prompts in f16 calls, which round each weight to f16 once: half an ulp of
//   the result's own type, for half of the second product (4 x 2,000 tokens over 8,000, 32 heads of 128 over 8: 392 us, with
//   two halves 521; error against 64 bits 2.9e-4 and 2.1e-4, which is the result's own rounding). Few rows wait for memory,
//   and two halves cost them little (48 conversations of those heads 52.2 and 53.3 us).
//   A weight carries the value scale of its block over a unit, a power of two above all value scales so far, and the base
//   that a row's exponentials are relative to follows the largest product of exponential and value scale that the row has
//   seen, not the largest exponential: so the weights of every row reach 2^6, clear of f16's subnormals and of its infinity,
//   whatever the scales of blocks are that the row does not see or gives no weight to.
#include <algorithm>
#include <type_traits>

#include "qh_device.h"
#include "qh_kv8.h"

namespace qh {
namespace {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));

constexpr int kTile = 64;            // positions of one step
constexpr int kRowTile = 16;         // query rows of a workgroup of the row kernel
constexpr int kMaxItems = 1024;      // row tiles of one launch of the row kernel
constexpr int kWhole = 1024;         // positions up to which a workgroup takes a row tile's sequence whole
constexpr int kSplitTiles = 5;       // positions of a split of the tile kernel, in tiles, at least
constexpr int kMaxParts = 512;       // shares of the row kernel: partial results of a row
constexpr long kMaxTiles = 1l << 30; // tiles of all items of one of its launches, so that counts and sums of them are ints

// Four codes as f16: the stored bytes, code + 128, under the high byte 0x64 are the numbers 1024 + 128 + code.
__device__ __forceinline__ void codes_to_f16(uint32_t x, uint32_t* out) {
    const h2 bias = {(_Float16)1152.0f, (_Float16)1152.0f};
    out[0] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, x, 0x04010400u)) - bias);
    out[1] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, x, 0x04030402u)) - bias);
}
__device__ __forceinline__ h8 codes8_to_f16(uint32_t a, uint32_t b) {
    uint32_t r[4];
    codes_to_f16(a, r);
    codes_to_f16(b, r + 2);
    return __builtin_bit_cast(h8, make_uint4(r[0], r[1], r[2], r[3]));
}

// v combined over the four lanes that hold one query column (lane, lane ^ 16, lane ^ 32, lane ^ 48).
template <typename Op>
__device__ __forceinline__ float over_groups(float v, Op op) {
    uint32_t u = __builtin_bit_cast(uint32_t, v);
    const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    v = op(__builtin_bit_cast(float, (uint32_t)a[0]), __builtin_bit_cast(float, (uint32_t)a[1]));
    u = __builtin_bit_cast(uint32_t, v);
    const auto b = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return op(__builtin_bit_cast(float, (uint32_t)b[0]), __builtin_bit_cast(float, (uint32_t)b[1]));
}
__device__ __forceinline__ float fmax2(float a, float b) { return __builtin_fmaxf(a, b); }

// 16 query rows as the operand of the score product: lane 16 g + r holds dims 64 c + 16 g .. + 15 of row r.
template <typename T, int kC>
struct Query {
    static constexpr bool kSplit = std::is_same<T, float>::value;
    h8 hi[kC][2], lo[kSplit ? kC : 1][2];
    float unit;  // x = product * unit * key scale, positive: a negative scale's sign goes into the operands

    // The row's values as loaded; convert() makes the operands of them, so that other loads can be issued in between.
    using Raw = std::conditional_t<kSplit, float4, h8>;
    static constexpr int kRaw = kSplit ? 4 : 2;
    __device__ __forceinline__ static void fetch(Raw (&r)[kC][kRaw], const T* p) {
#pragma unroll
        for (int c = 0; c < kC; ++c)
#pragma unroll
            for (int i = 0; i < kRaw; ++i) r[c][i] = reinterpret_cast<const Raw*>(p + 64 * c)[i];
    }

    __device__ __forceinline__ void convert(const Raw (&r)[kC][kRaw], bool valid, float scale_log2e) {
        if constexpr (kSplit) {
            float v[kC][16], top = 0.0f;
#pragma unroll
            for (int c = 0; c < kC; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    v[c][4 * i] = r[c][i].x, v[c][4 * i + 1] = r[c][i].y, v[c][4 * i + 2] = r[c][i].z,
                              v[c][4 * i + 3] = r[c][i].w;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        if (!valid) v[c][4 * i + j] = 0.0f;
                        top = __builtin_fmaxf(top, __builtin_fabsf(v[c][4 * i + j]));
                    }
                }
            top = over_groups(top, fmax2);
            // the power of two that takes the largest value to [2^13, 2^14); an infinite row becomes NaN
            const int e = max((int)(__builtin_bit_cast(uint32_t, top) >> 23) - 127, -100);
            const float up = top < __builtin_inff() ? __builtin_copysignf(__builtin_ldexpf(1.0f, 13 - e), scale_log2e)
                                                    : __builtin_nanf("");
            unit = __builtin_ldexpf(__builtin_fabsf(scale_log2e), e - 13);
#pragma unroll
            for (int c = 0; c < kC; ++c)
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float x = v[c][8 * h + j] * up;
                        hi[c][h][j] = (_Float16)x;
                        lo[c][h][j] = (_Float16)(x - (float)hi[c][h][j]);
                    }
        } else {
            unit = __builtin_fabsf(scale_log2e);
            float z = 0.0f;  // NaN for a row that is not finite, and then all of it becomes NaN
#pragma unroll
            for (int c = 0; c < kC; ++c)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    hi[c][h] = valid ? (scale_log2e < 0.0f ? -r[c][h] : r[c][h]) : h8{};
#pragma unroll
                    for (int j = 0; j < 8; ++j) z = __builtin_fmaf((float)hi[c][h][j], 0.0f, z);
                }
            z = over_groups(z, [](float p, float q) { return p + q; });
            if (z != z) {
#pragma unroll
                for (int c = 0; c < kC; ++c) hi[c][0] = hi[c][1] = h8{} + (_Float16)__builtin_nanf("");
            }
        }
    }

    __device__ __forceinline__ f4 dot(h8 k, int c, int h, f4 acc) const {
        acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, hi[c][h], acc, 0, 0, 0);
        if constexpr (kSplit) acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, lo[c][h], acc, 0, 0, 0);
        return acc;
    }
};

// The page and scales of 64 blocks, one to a lane: 16 tiles, lane 4 j + b block b of the j-th.
struct Blocks {
    int page;
    float ck, cv;
    uint64_t ok;     // lanes whose block exists
    uint64_t blank;  // lanes whose block has tokens with values of zero alone (the sign of its value scale)

    // tile: this lane's; blocks at or past len, or without a page, are left out.
    __device__ __forceinline__ void load(const Kv8View& c, int seq, int h, int tile, bool in_range, int len) {
        const int pos = tile * kTile + ((int)threadIdx.x & 3) * kBlk;
        page = -1;
        if (in_range && pos < len) page = c.table[(size_t)seq * c.seq_pages + (pos >> c.page_shift)];
        const bool good = page >= 0 && page < c.n_pages;
        ok = __ballot(good);
        ck = cv = 0.0f;
        const int blk = (pos >> 4) & ((1 << (c.page_shift - 4)) - 1);
        if (good) {
            ck = *kv8_scale(c, page, 0, h, blk);
            cv = *kv8_scale(c, page, 1, h, blk);
        }
        blank = __ballot(cv < 0.0f);
        cv = __builtin_fabsf(cv);
        page = good ? page : 0;
    }
    __device__ __forceinline__ int page_of(int i) const { return __builtin_amdgcn_readlane(page, i); }
};

// The running state of 16 query rows: the base that exponents are relative to, this lane's share of the sum, and the
// output, transposed: lane 16 g + r holds row r, register [4 c + i][s] dimension 64 c + 16 g + 4 s + i.
// The base is the largest x + level that the row has had, x a score (log2) and level the exponent of its block's value scale
// over the unit (see Unit; below 0, and -kDepth at least), and no later one exceeds it by more than kSlack: only then does
// it move and the output with it (16 registers per 64 dimensions and row tile), so that most tiles need neither that nor the
// maximum over the row's four lanes. The weight at the base, with the value scale, is in [2^kRoom, 2^(kRoom + 1)), so that
// weights stay below 2^15 and the smallest step of an f16, 2^-24, is 2^-30 of it. Without the value scale it is at most
// 2^(kDepth + kSlack), far enough from f32's end for sums of them. A row whose value scales, weighted, are more than
// 2^kDepth below the unit loses a bit of its weights for each power of two beyond.
constexpr float kSlack = 8.0f;
constexpr int kRoom = 6, kDepth = 80;
constexpr float kMostWeight = 0x1p15f;                          // of a lane's weights of a tile together
constexpr float kMostBare = kMostWeight / 0x1p88f;              // and of those without the value scale, 2^(kDepth + kSlack)

// A tile's scales, the same for every lane.
struct Scales {
    float key[4], weight[4];
    float level[4];  // exponents of the value scales over the unit
    int grown;       // powers of two by which the unit grew
    uint32_t ok;     // bits of the blocks that exist
    uint32_t nan;    // and of those with a NaN scale: they count as zeros here, see Rows::poison
    uint32_t blank;  // and of those with tokens whose values are all zero, see Rows::set_apart
};

// The value scales' running unit, a power of two above all of them so far and at least 2^-110, as its biased exponent (0:
// none yet). Weights are value scales over it, times 2^kRoom.
struct Unit {
    int e = 0;
    // The scales of the tile whose first block is lane i0 of bl; the unit grows where it has to.
    __device__ __forceinline__ Scales next(const Blocks& bl, int i0) {
        Scales t;
        int v[4], top = 17 << 23;
        t.ok = (uint32_t)(bl.ok >> i0) & 15u;
        t.blank = (uint32_t)(bl.blank >> i0) & 15u;
        t.nan = 0;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            int k = __builtin_amdgcn_readlane(__builtin_bit_cast(int, bl.ck), i0 + b);
            v[b] = __builtin_amdgcn_readlane(__builtin_bit_cast(int, bl.cv), i0 + b);
            const bool bad = max(k, v[b]) >= 0x7f800000;  // scales of keys are never negative
            t.nan |= bad ? 1u << b : 0u;
            k = bad ? 0 : k;
            v[b] = bad ? 0 : v[b];
            t.key[b] = __builtin_bit_cast(float, k);
            top = max(top, v[b]);
        }
        const int unit = max(e, min((top >> 23) + 1, 253));
        t.grown = e ? unit - e : 0;  // no row has an output before the first tile
        e = unit;
        const float inv = __builtin_bit_cast(float, (127 + kRoom + 127 - unit) << 23);
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            t.weight[b] = __builtin_bit_cast(float, v[b]) * inv;
            t.level[b] = (float)max((v[b] >> 23) - unit, -kDepth);
        }
        return t;
    }
    // What the output is multiplied by at the end.
    __device__ __forceinline__ float back() const { return e ? __builtin_bit_cast(float, (e - kRoom) << 23) : 0.0f; }
};

// kTwo: weights as two f16 each, else one.
template <int kC, bool kTwo>
struct Rows {
    float m = -__builtin_inff(), l = 0.0f;
    f4 o[4 * kC];

    __device__ __forceinline__ void clear() {
        m = -__builtin_inff();
        l = 0.0f;
#pragma unroll
        for (int i = 0; i < 4 * kC; ++i) o[i] = f4{0, 0, 0, 0};
    }

    // A step over a tile: x its products of codes and queries, [block][token 4 g + s]; x * f[b] is the score (log2).
    // The row sees the positions below vis; pos: this lane's first position in the tile, ok: bit b for a block that
    // exists. A masked position gets the score -inf, and so the weight 0: f may not be 0 for that (scores that a larger f
    // changes are below 2^-80).
    __device__ __forceinline__ static void mask(f4 (&x)[4], float (&f)[4], int pos, int vis, uint32_t ok) {
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            f[b] = __builtin_fmaxf(f[b], 0x1p-126f);
            const int end = (ok >> b) & 1u ? vis : 0;
#pragma unroll
            for (int s = 0; s < 4; ++s) x[b][s] = pos + 16 * b + s >= end ? -__builtin_inff() : x[b][s];
        }
    }
    // Blocks of a tile whose scales are NaN (bits of nan) make NaN of the rows that see any of their tokens.
    __device__ __forceinline__ void poison(uint32_t nan, int pos0, int vis) {
#pragma unroll
        for (int b = 0; b < 4; ++b)
            if ((nan >> b) & 1u) l = pos0 + 16 * b < vis ? __builtin_nanf("") : l;
    }

    // Tokens whose values are all zero (bit 4 b + s of blank for the scores x[b][s]) join the sum alone and are masked then:
    // at the lowest level, as a block of zeros. The base moves where it has to for that. Selections by masks of whole words:
    // conditions would take sixteen pairs of scalar registers from the loop around this.
    __device__ __forceinline__ void set_apart(f4 (&x)[4], const float (&f)[4], uint32_t blank) {
        const auto mask_of = [&](int n) { return (int)(blank << (31 - n)) >> 31; };
        const auto pick = [](int mask, float a, float b) {
            return __builtin_bit_cast(float, (__builtin_bit_cast(int, a) & mask) | (__builtin_bit_cast(int, b) & ~mask));
        };
        const float none = -__builtin_inff();
        float top = none;
        asm volatile("" : "+v"(blank));  // the masks are made here, not with those of the other row tiles
#pragma unroll
        for (int b = 0; b < 4; ++b) {
#pragma unroll
            for (int s = 0; s < 4; ++s)
                top = fmax2(top, pick(mask_of(4 * b + s), __builtin_fmaf(x[b][s], f[b], (float)-kDepth), none));
            __builtin_amdgcn_sched_barrier(0);
        }
        const float was = m;
        m = __builtin_fmaxf(m, over_groups(top, fmax2));
        const float alpha = m == was ? 1.0f : __builtin_amdgcn_exp2f(was - m), base = m == none ? 0.0f : m;
        l *= alpha;
#pragma unroll
        for (int i = 0; i < 4 * kC; ++i) o[i] *= alpha;
        asm volatile("" : "+v"(blank));  // and made again, not kept
#pragma unroll
        for (int b = 0; b < 4; ++b) {
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const int mask = mask_of(4 * b + s);
                l += pick(mask, __builtin_amdgcn_exp2f(__builtin_fmaf(x[b][s], f[b], -base)), 0.0f);
                x[b][s] = pick(mask, none, x[b][s]);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    }

    // Moves the base where a score passes it by too much, and the output with it. Where the unit grew, the levels of the
    // scores so far fall: the base falls with them, so that later weights reach 2^kRoom again, as far as the sum has room.
    __device__ __forceinline__ void settle(const f4 (&x)[4], const float (&f)[4], const Scales& sc, float slack) {
        float top = -__builtin_inff();
#pragma unroll
        for (int b = 0; b < 4; ++b)
            top = fmax2(top, __builtin_fmaf(fmax2(fmax2(x[b][0], x[b][1]), fmax2(x[b][2], x[b][3])), f[b], sc.level[b]));
        if (__any(top > m + slack) || sc.grown) {
            const float was = m;
            if (sc.grown) {
                const int most = (int)(__builtin_bit_cast(uint32_t, over_groups(l, fmax2)) >> 23) - 127;
                m -= (float)min(sc.grown, max(kDepth - max(most, 0), 0));
            }
            m = __builtin_fmaxf(m, over_groups(top, fmax2));
            const float alpha = m == was ? 1.0f : __builtin_amdgcn_exp2f(was - m);
            l *= alpha;
            const float a = __builtin_ldexpf(alpha, -sc.grown);
#pragma unroll
            for (int i = 0; i < 4 * kC; ++i) o[i] *= a;
        }
    }

    // The weights as operands w, two blocks to each (and their low halves lo); their sum, without the value scales, joins
    // `sum`, and with them `load`.
    __device__ __forceinline__ void weigh(const f4 (&x)[4], const float (&f)[4], const Scales& sc, h8 (&w)[2], h8 (&lo)[2],
                                          float& sum, float& load) const {
        // a row that has seen nothing yet: subtract 0, so that its weights are 2^-inf = 0 and not NaN
        const float base = m == -__builtin_inff() ? 0.0f : m;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            float p[4];
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                p[s] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[b][s], f[b], -base));
                float v = p[s] * sc.weight[b];
                // the halves are of one number: without this the compiler may round the product straight to f16 for one
                // use of hi and the f32 product for the other, which differ where the product is close to a tie
                if constexpr (kTwo) asm("" : "+v"(v));
                const _Float16 hi = (_Float16)v;
                w[b >> 1][4 * (b & 1) + s] = hi;
                if constexpr (kTwo) lo[b >> 1][4 * (b & 1) + s] = (_Float16)(v - (float)hi);
            }
            const float of_block = (p[0] + p[1]) + (p[2] + p[3]);
            sum += of_block;
            load = __builtin_fmaf(of_block, sc.weight[b], load);
        }
    }
};

// What a launch needs besides the cache.
struct AttnArgs {
    const void* q;
    void* out;
    int64_t ldq, ldo;
    Kv8Batch batch;
    int group;  // query heads to a KV head; the rows of an entry are (token, head of the group)
    int causal;
    float scale_log2e;
    float* part_o;   // partial outputs, means [slot][n_kv][rows][hd], with their base and sum [slot][n_kv][rows][2]
    float* part_ml;
    int4* rec;       // [items] where an item's partials are: first slot, how many (0: none), first row, rows
    int items, splits;
    int8_t* oq;  // the output in 8 bits as well, and its scales (f32 calls; null: not)
    float* od;
};

// Entry b's rows: global rows (token * group + head) from first on, and the positions its tokens see.
struct Entry {
    int seq, len, tokens, row0, rows;
};
__device__ __forceinline__ Entry entry_of(const Kv8View& c, const AttnArgs& a, int b) {
    const int s0 = a.batch.at(b), s1 = max(s0, a.batch.at(b + 1)), seq = a.batch.seq(b);
    const bool known = seq >= 0 && seq < c.n_seqs;
    return {known ? seq : 0, known ? kv8_len(c, seq) : 0, s1 - s0, s0 * a.group, (s1 - s0) * a.group};
}
// The same in scalar registers (every lane has the same entry).
__device__ __forceinline__ Entry uniform(const Entry& e) {
    return {__builtin_amdgcn_readfirstlane(e.seq), __builtin_amdgcn_readfirstlane(e.len),
            __builtin_amdgcn_readfirstlane(e.tokens), __builtin_amdgcn_readfirstlane(e.row0),
            __builtin_amdgcn_readfirstlane(e.rows)};
}
// Positions that row r of the entry sees.
__device__ __forceinline__ int visible(const Entry& e, const AttnArgs& a, int r) {
    return a.causal ? min(max(e.len - e.tokens + r / a.group + 1, 0), e.len) : e.len;
}

// a over a row's sum of weights, zero where it saw nothing. Outputs are weighted means before they meet, never sums of values,
// which may be past f32's largest number where no value is.
__device__ __forceinline__ float over_sum(float a, float l) { return l == 0.0f ? 0.0f : a / l; }

// 4 values of the output. kX8: 8 lanes in a row hold 32 values of a row, and write them in 8 bits too where the call asks for
// that.
template <typename T, bool kX8>
__device__ __forceinline__ void store_out(const AttnArgs& a, T* out, float4 v) {
    if constexpr (std::is_same<T, float>::value) {
        *reinterpret_cast<float4*>(out) = v;
        if (kX8 && a.oq) {
            const int64_t at = (out - static_cast<float*>(a.out)) & ~31ll;
            quant_block_x8(v, a.oq + at, a.od + at / 32);
        }
    } else {
        typedef _Float16 h4 __attribute__((ext_vector_type(4)));
        *reinterpret_cast<h4*>(out) = h4{(_Float16)v.x, (_Float16)v.y, (_Float16)v.z, (_Float16)v.w};
    }
}
template <typename T>
__device__ __forceinline__ T* out_row(const AttnArgs& a, const Kv8View& c, int grow, int kvh) {
    const int tok = grow / a.group, head = kvh * a.group + (grow - tok * a.group);
    return static_cast<T*>(a.out) + (int64_t)tok * a.ldo + (int64_t)head * c.hd;
}
template <typename T>
__device__ __forceinline__ const T* q_row(const AttnArgs& a, const Kv8View& c, int grow, int kvh) {
    const int tok = grow / a.group, head = kvh * a.group + (grow - tok * a.group);
    return static_cast<const T*>(a.q) + (int64_t)tok * a.ldq + (int64_t)head * c.hd;
}

// ------------------------------------------------------------------------------------------------ few rows

// The waves of a workgroup meet here.
template <int kC, int kW>
struct RowsLds {
    __align__(16) float so[kW][kRowTile][64 * kC + 4];
    float sm[kW][kRowTile], sl[kW][kRowTile];
};

// The tiles [t0, t1) of one row tile, from row r0 of entry e, by a workgroup of kW waves: they take every kW-th tile, each
// with a base and sum of its own, straight from global memory into registers (one contiguous KB a load, the next tile's
// loads in flight while one is computed), and meet in shared memory at the end. whole: those are all tiles of the rows, and
// the result goes to out, else into partial result `slot`.
template <typename T, int kC, int kW>
__device__ __forceinline__ void rows_tiles(const Kv8View& c, const AttnArgs& a, RowsLds<kC, kW>& sh, int kvh, const Entry& e,
                                           int r0, int t0, int t1, bool whole, int slot) {
    constexpr int kHd = 64 * kC;
    const int tid = (int)threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, g = lane >> 4,
              col = lane & 15;
    const int r = r0 + col;
    const bool valid = r < e.rows;
    const int n_mine = t1 - t0 > wave ? (t1 - t0 - wave + kW - 1) / kW : 0;  // tiles t0 + wave + kW j
    Blocks bl;
    auto blocks = [&](int j) {
        const int jl = j + (lane >> 2);
        bl.load(c, e.seq, kvh, t0 + wave + kW * jl, jl < n_mine, e.len);
    };
    uint4 kr[4][kC], vr[4][kC];
    auto fetch = [&](uint4 (&to)[4][kC], int which, int j) {
        const int tile = t0 + wave + kW * j;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int page = bl.page_of(4 * (j & 15) + k), blk = (tile * 4 + k) & ((1 << (c.page_shift - 4)) - 1);
            const uint4* p = reinterpret_cast<const uint4*>(kv8_codes(c, page, which, kvh, blk)) + lane;
#pragma unroll
            for (int cc = 0; cc < kC; ++cc) to[k][cc] = load_once(p + 64 * cc);
        }
    };
    typename Query<T, kC>::Raw raw[kC][Query<T, kC>::kRaw];
    blocks(0);
    Query<T, kC>::fetch(raw, q_row<T>(a, c, e.row0 + (valid ? r : r0), kvh) + 16 * g);
    if (n_mine > 0) {
        fetch(kr, 0, 0);
        fetch(vr, 1, 0);
    }
    const int vis = valid ? visible(e, a, r) : 0;
    const int all_see = visible(e, a, r0);  // positions that every row sees: the first row's
    Query<T, kC> q;
    q.convert(raw, valid, a.scale_log2e);
    Rows<kC, true> st;
    st.clear();
    Unit unit;

    for (int j = 0; j < n_mine; ++j) {
        const int pos0 = (t0 + wave + kW * j) * kTile, i0 = 4 * (j & 15);
        const Scales sc = unit.next(bl, i0);
        f4 x[4];
        float f[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            f4 acc = {0, 0, 0, 0};
#pragma unroll
            for (int cc = 0; cc < kC; ++cc) {
                acc = q.dot(codes8_to_f16(kr[k][cc].x, kr[k][cc].y), cc, 0, acc);
                acc = q.dot(codes8_to_f16(kr[k][cc].z, kr[k][cc].w), cc, 1, acc);
            }
            x[k] = acc;
            f[k] = sc.key[k] * q.unit;
        }
        // the next tile's keys are in flight from here on, its values from the end of the step
        __builtin_amdgcn_sched_barrier(0);
        const bool more = j + 1 < n_mine;
        if (more) {
            if (((j + 1) & 15) == 0) blocks(j + 1);
            fetch(kr, 0, j + 1);
        }
        __builtin_amdgcn_sched_barrier(0);
        h8 w[2], lo[2];
        if (pos0 + kTile > all_see || sc.ok != 15u || sc.blank) {
            st.mask(x, f, pos0 + 4 * g, vis, sc.ok);
            if (sc.blank) {
                uint32_t blank = 0;
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    uint32_t any = 0;  // byte s: of token 4 g + s
#pragma unroll
                    for (int cc = 0; cc < kC; ++cc)
                        any |= (vr[b][cc].x ^ kBias) | (vr[b][cc].y ^ kBias) | (vr[b][cc].z ^ kBias) | (vr[b][cc].w ^ kBias);
                    any = or_row16(any);
                    any = ~(any | ((any & 0x7f7f7f7fu) + 0x7f7f7f7fu)) & 0x80808080u;  // the top bits of bytes that are 0
                    any = ((any >> 7) | (any >> 14) | (any >> 21) | (any >> 28)) & 15u;
                    blank |= (sc.blank >> b) & 1u ? any << (4 * b) : 0u;
                }
                st.set_apart(x, f, blank);
            }
        }
        if (sc.nan) st.poison(sc.nan, pos0, vis);
        st.settle(x, f, sc, kSlack);
        float load = 0.0f;
        st.weigh(x, f, sc, w, lo, st.l, load);
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int cc = 0; cc < kC; ++cc) {
                const uint4 v0 = vr[2 * u][cc], v1 = vr[2 * u + 1][cc];
                const uint32_t a0[4] = {v0.x, v0.y, v0.z, v0.w}, a1[4] = {v1.x, v1.y, v1.z, v1.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const h8 v = codes8_to_f16(a0[i], a1[i]);
                    f4& o = st.o[4 * cc + i];
                    o = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, w[u], o, 0, 0, 0);
                    o = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, lo[u], o, 0, 0, 0);
                }
            }
        __builtin_amdgcn_sched_barrier(0);
        if (more) fetch(vr, 1, j + 1);
    }

    // the waves' results of this item together
    const float l = over_groups(st.l, [](float p, float q2) { return p + q2; });
    const float mean = over_sum(unit.back(), l);
    if (g == 0) {
        sh.sm[wave][col] = st.m;
        sh.sl[wave][col] = l;
    }
#pragma unroll
    for (int cc = 0; cc < kC; ++cc)
#pragma unroll
        for (int s = 0; s < 4; ++s)
            *reinterpret_cast<float4*>(&sh.so[wave][col][64 * cc + 16 * g + 4 * s]) =
                make_float4(st.o[4 * cc][s] * mean, st.o[4 * cc + 1][s] * mean, st.o[4 * cc + 2][s] * mean,
                            st.o[4 * cc + 3][s] * mean);
    __syncthreads();
    const int rr = (tid >> 4) & 15, d0 = 4 * (tid & 15);
    if (r0 + rr < e.rows) {
        float top = sh.sm[0][rr];
#pragma unroll
        for (int w2 = 1; w2 < kW; ++w2) top = __builtin_fmaxf(top, sh.sm[w2][rr]);
        const float base = top == -__builtin_inff() ? 0.0f : top;
        float f[kW], lsum = 0.0f;
#pragma unroll
        for (int w2 = 0; w2 < kW; ++w2) {
            f[w2] = __builtin_amdgcn_exp2f(sh.sm[w2][rr] - base) * sh.sl[w2][rr];
            lsum += f[w2];
        }
        const float inv = over_sum(1.0f, lsum);
#pragma unroll
        for (int w2 = 0; w2 < kW; ++w2) f[w2] *= inv;
        const size_t pr = ((size_t)slot * c.n_kv + kvh) * kRowTile + rr;
        for (int cc = tid >> 8; cc < kC; cc += kW / 4) {
            float4 o = make_float4(0, 0, 0, 0);
#pragma unroll
            for (int w2 = 0; w2 < kW; ++w2) {
                const float4 v = *reinterpret_cast<const float4*>(&sh.so[w2][rr][64 * cc + d0]);
                o.x = __builtin_fmaf(f[w2], v.x, o.x);
                o.y = __builtin_fmaf(f[w2], v.y, o.y);
                o.z = __builtin_fmaf(f[w2], v.z, o.z);
                o.w = __builtin_fmaf(f[w2], v.w, o.w);
            }
            if (whole)
                store_out<T, true>(a, out_row<T>(a, c, e.row0 + r0 + rr, kvh) + 64 * cc + d0, o);
            else
                *reinterpret_cast<float4*>(a.part_o + pr * kHd + 64 * cc + d0) = o;
        }
        if (!whole && tid < 256 && (tid & 15) == 0) {
            a.part_ml[2 * pr] = top;
            a.part_ml[2 * pr + 1] = lsum;
        }
    }
}

// Row tiles of 16 (single tokens: the query heads of one KV head) over long caches, bound by reading the codes. The
// tiles of all items lie end to end, and each of the gridDim.x workgroups of a KV head takes an equal share of them,
// whatever the lengths are: a share may end inside an item (the parts are joined by kv8_join_kernel) or span several.
// Every workgroup finds its share from the lengths itself.
template <typename T, int kC, int kW>
__global__ __launch_bounds__(64 * kW, 2) void kv8_rows_kernel(Kv8View c, AttnArgs a) {
    __shared__ int pre_all[kMaxItems + 1];
    __shared__ uint16_t ent_all[kMaxItems];
    __shared__ Entry entries_all[kMaxItems];
    __shared__ int wave_sum[3 * kW];
    __shared__ RowsLds<kC, kW> sh;
    const int tid = (int)threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int kvh = (int)blockIdx.y, tiles_per_token = (a.group + kRowTile - 1) / kRowTile, shares = (int)gridDim.x;
    auto first_item = [&](const Entry& e, int b) {
        return a.batch.start ? (int)((long)e.row0 / kRowTile) + b : b * tiles_per_token;
    };
    // up to 64 items each wave works the shares out for itself, without a barrier (one token over 100,000 positions, 12
    // heads of 128 over 2, f32: 24.3 us, by the workgroup 25.3)
    const bool alone = a.items <= 64;
    int* pre = pre_all + (alone ? 65 * wave : 0);
    uint16_t* ent = ent_all + (alone ? 64 * wave : 0);
    Entry* entries = entries_all + (alone ? 64 * wave : 0);
    const int me = alone ? lane : tid, width = alone ? 64 : 64 * kW;
    auto meet = [&] {
        if (alone) __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        else __syncthreads();
    };

    // the items' tile counts, then their prefix sums
    for (int i = me; i < a.items; i += width) pre[i] = 0;
    meet();
    for (int b = me; b < a.batch.n; b += width) {
        const Entry e = entry_of(c, a, b);
        entries[b] = e;
        const int at = first_item(e, b);
        for (int t = 0; t * kRowTile < e.rows && at + t < a.items; ++t) {
            const int last = min((t + 1) * kRowTile, e.rows) - 1;
            pre[at + t] = max(1, (visible(e, a, last) + kTile - 1) / kTile);
            ent[at + t] = (uint16_t)b;
        }
    }
    meet();
    constexpr int kPer = kMaxItems / (64 * kW);
    const int per = alone ? 1 : kPer;
    int mine[kPer], sum = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        mine[j] = j < per && me * per + j < a.items ? pre[me * per + j] : 0;
        sum += mine[j];
    }
    auto all_of = [&](int v, int* s) {  // the sum over the workgroup, or the wave that is alone
        v = wave_sum_i32(v);
        if (alone) return v;
        if (lane == 0) s[wave] = v;
        __syncthreads();
        v = 0;
#pragma unroll
        for (int i = 0; i < kW; ++i) v += s[i];
        return v;
    };
    // a tile to each wave at least, but no whole rounds of them (48 conversations of 2,500, 32 heads of 128 over 8, f16:
    // 46.8 us, in whole rounds 48.2)
    const int share = max(kW, (all_of(sum, wave_sum) + shares - 1) / shares);
    // items that begin on a share of their own where the shares suffice for that: no workgroup then has two items in turn
    // (counted in shares: in tiles, many short items would pass an int)
    int own[kPer];
    sum = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        own[j] = (mine[j] + share - 1) / share;
        sum += own[j];
    }
    const bool apart = all_of(sum, wave_sum + kW) <= shares;
    sum = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        mine[j] = apart ? own[j] * share : mine[j];
        sum += mine[j];
    }
    int incl = sum;
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
        const int y = __shfl_up(incl, s);
        incl += lane >= s ? y : 0;
    }
    int at = incl - sum, total = __builtin_amdgcn_readlane(incl, 63);
    if (!alone) {
        if (lane == 63) wave_sum[2 * kW + wave] = incl;
        __syncthreads();
        total = 0;
#pragma unroll
        for (int i = 0; i < kW; ++i) {
            at += i < wave ? wave_sum[2 * kW + i] : 0;
            total += wave_sum[2 * kW + i];
        }
    }
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        if (j < per && me * per + j < a.items) pre[me * per + j] = at;
        at += mine[j];
    }
    if (me == 0) pre[a.items] = total;
    meet();

    // tiles of an item: its own, without what pads it
    auto tiles_of = [&](int i) {
        const Entry e = entries[ent[i]];
        const int r1 = min((i - first_item(e, ent[i]) + 1) * kRowTile, e.rows) - 1;
        return max(1, (visible(e, a, r1) + kTile - 1) / kTile);
    };
    if (blockIdx.x == 0 && kvh == 0) {
        for (int i = tid; i < a.items; i += 64 * kW) {
            int4 r = make_int4(0, 0, 0, 0);
            if (pre[i + 1] > pre[i]) {
                const int b = ent[i];
                const Entry e = entries[b];
                const int t = i - first_item(e, b), end = min(pre[i] + tiles_of(i), pre[i + 1]);
                const int w0 = pre[i] / share, w1 = (end - 1) / share;
                r = make_int4(2 * w0 + (pre[i] > w0 * share ? 1 : 0), w1 > w0 ? w1 - w0 + 1 : 0, e.row0 + t * kRowTile,
                              min(kRowTile, e.rows - t * kRowTile));
            }
            a.rec[i] = r;
        }
    }
    const int from = (int)blockIdx.x * share, to = min(total, from + share);
    if (from >= to) return;

    // the item that holds tile `from`: the last one whose prefix is at or below it (items without tiles have the
    // following item's prefix)
    int item = 0;
    {
        int lo = 0, hi = a.items - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (pre[mid] <= from) lo = mid;
            else hi = mid - 1;
        }
        item = __builtin_amdgcn_readfirstlane(lo);
    }

    for (int done = from; done < to; ++item) {
        const int p0 = pre[item], p1 = pre[item + 1];
        if (p1 <= done) continue;
        const int n_tiles = __builtin_amdgcn_readfirstlane(tiles_of(item));
        const int t0 = done - p0, t1 = min(min(to, p1) - p0, n_tiles);  // this item's tiles of the share
        done = min(to, p1);
        if (t0 >= t1) continue;  // only what pads the item
        const int b = __builtin_amdgcn_readfirstlane((int)ent[item]);
        const Entry e = uniform(entries[b]);
        rows_tiles<T, kC, kW>(c, a, sh, kvh, e, (item - first_item(e, b)) * kRowTile, t0, t1, t0 == 0 && t1 == n_tiles,
                              2 * (int)blockIdx.x + (p0 + t0 > from ? 1 : 0));
        __syncthreads();
    }
}

// Row tiles over sequences of a few tiles: a workgroup each, with nothing to share out or to join. Bound by its dependent
// loads: the entry, the length, pages, scales and then two or three tiles' codes (one token over 64 positions 4.5 us).
template <typename T, int kC, int kW>
__global__ __launch_bounds__(64 * kW, 2) void kv8_whole_kernel(Kv8View c, AttnArgs a) {
    __shared__ RowsLds<kC, kW> sh;
    const int kvh = (int)blockIdx.y, item = (int)blockIdx.x, tiles_per_token = (a.group + kRowTile - 1) / kRowTile;
    int b = item / tiles_per_token, from = b * tiles_per_token;
    if (a.batch.start) b = kv8_entry_of(a.batch, item, a.group, kRowTile, 1, &from);
    if (b < 0) return;
    const Entry e = uniform(entry_of(c, a, b));
    const int r0 = (item - __builtin_amdgcn_readfirstlane(from)) * kRowTile;
    if (r0 >= e.rows) return;
    const int tiles = (visible(e, a, min(r0 + kRowTile, e.rows) - 1) + kTile - 1) / kTile;
    rows_tiles<T, kC, kW>(c, a, sh, kvh, e, r0, 0, tiles, true, 0);
}

// Joins an item's partial results: one workgroup per item, KV head and row. First the partials' bases, a thread to each,
// and from them every partial's share; then hd / 4 threads to a partial's row, the workgroup's groups of them taking
// turns, so that the loads are independent of each other. Partial k is slot first (k = 0) or the k-th even one after.
template <typename T, int kC>
__global__ __launch_bounds__(256) void kv8_join_kernel(Kv8View c, AttnArgs a) {
    constexpr int kHd = 64 * kC, kThr = kHd / 4, kGroups = 256 / kThr;
    __shared__ __align__(16) float so[kGroups][kHd];
    __shared__ float share[kMaxParts], wave_top[4], wave_sum[4];
    const int4 rec = a.rec[blockIdx.x];
    const int row = (int)blockIdx.z, kvh = (int)blockIdx.y, tid = (int)threadIdx.x, grp = tid / kThr, d = 4 * (tid % kThr);
    if (rec.y == 0 || row >= rec.w) return;
    auto at = [&](int k) {
        const int slot = k == 0 ? rec.x : (rec.x & ~1) + 2 * k;
        return ((size_t)slot * c.n_kv + kvh) * kRowTile + row;
    };
    float m[kMaxParts / 256], top = -__builtin_inff();
#pragma unroll
    for (int j = 0; j < kMaxParts / 256; ++j) {
        const int k = tid + 256 * j;
        m[j] = k < rec.y ? a.part_ml[2 * at(k)] : -__builtin_inff();
        top = __builtin_fmaxf(top, m[j]);
    }
    top = wave_reduce32x2(top, fmax2);
    if ((tid & 63) == 0) wave_top[tid >> 6] = top;
    __syncthreads();
    top = __builtin_fmaxf(__builtin_fmaxf(wave_top[0], wave_top[1]), __builtin_fmaxf(wave_top[2], wave_top[3]));
    const float base = top == -__builtin_inff() ? 0.0f : top;
    float l = 0.0f;
#pragma unroll
    for (int j = 0; j < kMaxParts / 256; ++j) {
        const int k = tid + 256 * j;
        if (k < rec.y) {
            const float f = __builtin_amdgcn_exp2f(m[j] - base) * a.part_ml[2 * at(k) + 1];
            share[k] = f;
            l += f;
        }
    }
    l = wave_reduce32x2(l, [](float p, float q) { return p + q; });
    if ((tid & 63) == 0) wave_sum[tid >> 6] = l;
    __syncthreads();
    const float inv = over_sum(1.0f, (wave_sum[0] + wave_sum[1]) + (wave_sum[2] + wave_sum[3]));
    float4 o = make_float4(0, 0, 0, 0);
#pragma unroll 4
    for (int k = grp; k < rec.y; k += kGroups) {
        const float4 v = *reinterpret_cast<const float4*>(a.part_o + at(k) * kHd + d);
        const float f = share[k] * inv;
        o.x = __builtin_fmaf(f, v.x, o.x);
        o.y = __builtin_fmaf(f, v.y, o.y);
        o.z = __builtin_fmaf(f, v.z, o.z);
        o.w = __builtin_fmaf(f, v.w, o.w);
    }
    *reinterpret_cast<float4*>(&so[grp][d]) = o;
    __syncthreads();
    if (grp != 0) return;
#pragma unroll
    for (int k = 1; k < kGroups; ++k) {
        const float4 v = *reinterpret_cast<const float4*>(&so[k][d]);
        o.x += v.x, o.y += v.y, o.z += v.z, o.w += v.w;
    }
    store_out<T, true>(a, out_row<T>(a, c, rec.z + row, kvh) + d, o);
}

// The same for few partials (the splits of the tile kernel): every group of hd / 4 threads joins a row of its own.
template <typename T, int kC>
__global__ __launch_bounds__(256) void kv8_join_splits_kernel(Kv8View c, AttnArgs a, int rows) {
    constexpr int kHd = 64 * kC, kThr = kHd / 4, kGroups = 256 / kThr;
    const int4 rec = a.rec[blockIdx.x];
    const int row = (int)blockIdx.z * kGroups + (int)threadIdx.x / kThr, kvh = (int)blockIdx.y;
    const int d = 4 * ((int)threadIdx.x % kThr);
    if (rec.y == 0 || row >= rec.w) return;
    const size_t first = ((size_t)rec.x * c.n_kv + kvh) * rows + row, next = (size_t)c.n_kv * rows;
    float top = -__builtin_inff();
    for (int k = 0; k < rec.y; ++k) top = __builtin_fmaxf(top, a.part_ml[2 * (first + k * next)]);
    const float base = top == -__builtin_inff() ? 0.0f : top;
    float l = 0.0f;
    for (int k = 0; k < rec.y; ++k) {
        const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + 2 * (first + k * next));
        l = __builtin_fmaf(__builtin_amdgcn_exp2f(ml.x - base), ml.y, l);
    }
    const float inv = over_sum(1.0f, l);
    float4 o = make_float4(0, 0, 0, 0);
#pragma unroll 4
    for (int k = 0; k < rec.y; ++k) {
        const size_t p = first + k * next;
        const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + 2 * p);
        const float f = __builtin_amdgcn_exp2f(ml.x - base) * ml.y * inv;
        const float4 v = *reinterpret_cast<const float4*>(a.part_o + p * kHd + d);
        o.x = __builtin_fmaf(f, v.x, o.x);
        o.y = __builtin_fmaf(f, v.y, o.y);
        o.z = __builtin_fmaf(f, v.z, o.z);
        o.w = __builtin_fmaf(f, v.w, o.w);
    }
    store_out<T, false>(a, out_row<T>(a, c, rec.z + row, kvh) + d, o);
}

// ------------------------------------------------------------------------------------------------ many rows

// Row tiles of 16 kW kCt (a prompt's tokens times the query heads of a KV head), bound by instruction issue: the matrix
// instructions and, next to them, the exponentials. Each of the kW waves holds 16 kCt rows; a tile's codes become f16 once
// per workgroup, into shared memory, in the order in which the waves read them as operands (1 KB a read, no bank
// conflicts), in two buffers: one barrier a tile, the next tile's codes converted between the matrix instructions of this
// one and the one after that in flight. The KV head is the fastest grid index, so that the workgroups of one head share an
// XCD's L2 where there are eight heads, and the last row tiles (which see the most positions) start first. splits > 1:
// up to that many workgroups share a row tile's positions and leave partials. kG groups of four waves share a workgroup's
// positions, each with buffers of its own, and meet in shared memory at the end.
template <typename T, int kC, int kCt, int kG>
__global__ __launch_bounds__(256 * kG, 2) void kv8_tile_kernel(Kv8View c, AttnArgs a) {
    constexpr int kHd = 64 * kC, kW = 4, kRows = 16 * kW * kCt;
    constexpr int kUnits = 4 * kC * 2 * 64;  // 16-byte units of a tile's keys (and values) in f16
    extern __shared__ __align__(16) uint4 lds_all[];  // [group][buffer][keys, values][kUnits]
    const int tid = (int)threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6) & 3,
              grp = __builtin_amdgcn_readfirstlane(tid >> 8), lane = tid & 63, g = lane >> 4, col = lane & 15;
    uint4* lds = lds_all + grp * 4 * kUnits;
    const int kvh = (int)(blockIdx.x % (unsigned)c.n_kv), split = (int)blockIdx.y;
    const int item = a.items - 1 - (int)(blockIdx.x / (unsigned)c.n_kv);
    int from = 0, b = item;
    b = kv8_entry_of(a.batch, item, a.group, kRows, 1, &from);
    Entry e{0, 0, 0, 0, 0};
    if (b >= 0) e = uniform(entry_of(c, a, b));
    const int r0 = b < 0 ? 0 : (item - __builtin_amdgcn_readfirstlane(from)) * kRows;
    const int last = min(r0 + kRows, e.rows) - 1;
    const int tiles = r0 < e.rows ? (visible(e, a, last) + kTile - 1) / kTile : 0;
    // The splits that this item takes, of at least five tiles: the join moves the rows' outputs twice in f32 (14 heads of
    // 64 over 2, f32: a prompt of 512 whole 17.3 us, in two splits 17.8; 4 x 120 behind 580 21.7 and 18.3; 256 tokens of
    // 32 heads of 128 over 8, f16, whole 12.1, a tile to a split 21.2)
    const int splits = min(a.splits, max(tiles / kSplitTiles, 1));
    if (a.splits > 1 && split == 0 && kvh == 0 && tid == 0)
        a.rec[item] = splits > 1 ? make_int4(item * a.splits, splits, e.row0 + r0, last + 1 - r0) : make_int4(0, 0, 0, 0);
    if (r0 >= e.rows || split >= splits) return;
    const int first = tiles * split / splits, end = tiles * (split + 1) / splits;  // the workgroup's tiles
    const int steps = (end - first + kG - 1) / kG, t0 = first + grp * steps, t1 = min(t0 + steps, end);  // the group's

    Query<T, kC> q[kCt];
    Rows<kC, Query<T, kC>::kSplit> st[kCt];
    int vis[kCt];
#pragma unroll
    for (int ct = 0; ct < kCt; ++ct) {
        const int r = r0 + wave * (16 * kCt) + ct * 16 + col;
        const bool valid = r < e.rows;
        vis[ct] = valid ? visible(e, a, r) : 0;
        typename Query<T, kC>::Raw raw[kC][Query<T, kC>::kRaw];
        Query<T, kC>::fetch(raw, q_row<T>(a, c, e.row0 + (valid ? r : r0), kvh) + 16 * g);
        q[ct].convert(raw, valid, a.scale_log2e);
        st[ct].clear();
        if (!valid) st[ct].m = 0.0f;  // a row that is not there asks for no base
    }
    const int w0 = r0 + wave * (16 * kCt);
    const int all_see = w0 <= last ? visible(e, a, w0) : 0;  // positions that each row of the wave sees
    Unit unit;

    // Each wave stages kPer operands of the keys and of the values, of one block of keys and one pair of blocks of values.
    constexpr int kPer = 8 * kC / kW;
    static_assert(kPer == 2 || kPer == 4, "loads of whole uint4 of keys, uint2 or uint4 of values");
    const int k_op = wave * kPer, k_blk = k_op / (2 * kC), v_pair = k_op / (4 * kC), v_c = k_op / 4 % kC, v_i = k_op % 4;
    Blocks bl, ahead;
    uint32_t kr[2 * kPer], vr[2][kPer];
    const int per = (1 << (c.page_shift - 4)) - 1;
    auto fetch = [&](int t) {
        const int j = (t - t0) & 15;
        if (j == 0) {
            const int tl = t + (lane >> 2);
            ahead.load(c, e.seq, kvh, tl, tl < t1, e.len);
        }
        const uint8_t* kp = kv8_codes(c, ahead.page_of(4 * j + k_blk), 0, kvh, (t * 4 + k_blk) & per);
#pragma unroll
        for (int n = 0; n < kPer / 2; ++n) {
            const uint4 x = reinterpret_cast<const uint4*>(kp)[64 * ((k_op / 2 + n) % kC) + lane];
            kr[4 * n] = x.x, kr[4 * n + 1] = x.y, kr[4 * n + 2] = x.z, kr[4 * n + 3] = x.w;
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int blk = 2 * v_pair + k;
            const uint32_t* vp = reinterpret_cast<const uint32_t*>(
                                     kv8_codes(c, ahead.page_of(4 * j + blk), 1, kvh, (t * 4 + blk) & per)) +
                                 4 * (64 * v_c + lane) + v_i;
            if constexpr (kPer == 4) {
                const uint4 x = *reinterpret_cast<const uint4*>(vp);
                vr[k][0] = x.x, vr[k][1] = x.y, vr[k][2] = x.z, vr[k][3] = x.w;
            } else {
                const uint2 x = *reinterpret_cast<const uint2*>(vp);
                vr[k][0] = x.x, vr[k][1] = x.y;
            }
        }
    };
    auto stage = [&](int buf) {
        uint4* ks = lds + (size_t)buf * 2 * kUnits + (size_t)k_op * 64 + lane;
        uint4* vs = ks + kUnits;
#pragma unroll
        for (int n = 0; n < kPer; ++n) {
            ks[n * 64] = __builtin_bit_cast(uint4, codes8_to_f16(kr[2 * n], kr[2 * n + 1]));
            vs[n * 64] = __builtin_bit_cast(uint4, codes8_to_f16(vr[0][n], vr[1][n]));
        }
    };

    // One tile from buffer buf, while the next tile's codes go into the other one. The matrix instructions run in the
    // background of a wave, four issue slots each: the conversion of the next tile fills them in the first product, and
    // each operand is read from shared memory kDeep reads before its use. A wave in one of its products goes before the
    // other wave of its SIMD, which has exponentials to fill the slots that are left (4 x 2,000 tokens over 8,000, 32
    // heads of 128 over 8, f16: 1,047 -> 996 us).
    constexpr int kMm = kCt * (Query<T, kC>::kSplit ? 2 : 1);  // matrix instructions to an operand read
    constexpr int kOps = 8 * kC, kDeep = 4;
    auto compute = [&](int buf, int t) {
        const int pos0 = t * kTile, i0 = 4 * ((t - t0) & 15);
        const uint4* ks = lds + (size_t)buf * 2 * kUnits + lane;
        const uint4* vs = ks + kUnits;
        h8 kk[kDeep], vv[kDeep];
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int r = 0; r < kDeep; ++r) kk[r] = __builtin_bit_cast(h8, ks[r * 64]);
        f4 x[kCt][4];
#pragma unroll
        for (int r = 0; r < kOps; ++r) {  // operand r: key block r / (2 kC), dimensions by r % (2 kC)
            const int k = r / (2 * kC), cc = r / 2 % kC, h = r & 1;
#pragma unroll
            for (int ct = 0; ct < kCt; ++ct) {
                if (r % (2 * kC) == 0) x[ct][k] = f4{0, 0, 0, 0};
                x[ct][k] = q[ct].dot(kk[r % kDeep], cc, h, x[ct][k]);
            }
            if (r + kDeep < kOps) kk[r % kDeep] = __builtin_bit_cast(h8, ks[(r + kDeep) * 64]);
        }
        stage(buf ^ 1);
        __builtin_amdgcn_sched_group_barrier(0x100, kDeep, 0);
#pragma unroll
        for (int r = 0; r < kOps; ++r) {
            __builtin_amdgcn_sched_group_barrier(0x008, kMm, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x002, 5, 0);
            if (r & 1) __builtin_amdgcn_sched_group_barrier(0x200, 1, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_setprio(0);
        if (t + 2 < t1) fetch(t + 2);
        // (before the scales; with two f32 row tiles behind the masks, where fewer registers are in use: 843 and 890 us)
        const auto values_ahead = [&] {
#pragma unroll
            for (int r = 0; r < kDeep; ++r) vv[r] = __builtin_bit_cast(h8, vs[r * 64]);
            __builtin_amdgcn_sched_barrier(0);
        };
        if constexpr (kMm < 4) values_ahead();
        const Scales sc = unit.next(bl, i0);
        float f[kCt][4];
#pragma unroll
        for (int ct = 0; ct < kCt; ++ct)
#pragma unroll
            for (int k = 0; k < 4; ++k) f[ct][k] = sc.key[k] * q[ct].unit;
        if (pos0 + kTile > all_see || sc.ok != 15u || sc.blank) {
#pragma unroll
            for (int ct = 0; ct < kCt; ++ct) st[ct].mask(x[ct], f[ct], pos0 + 4 * g, vis[ct], sc.ok);
            if (sc.blank) {
                uint32_t blank = 0;
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    uint32_t any[4] = {};  // tokens 0 1 and 2 3 of blocks 2 u and 2 u + 1, as the operands' f16
#pragma unroll
                    for (int i = 0; i < 4 * kC; ++i) {
                        const uint4 v = vs[(u * 4 * kC + i) * 64];
                        any[0] |= v.x, any[1] |= v.y, any[2] |= v.z, any[3] |= v.w;
                    }
#pragma unroll
                    for (int n = 0; n < 4; ++n) {
                        const int b = 2 * u + (n >> 1), s = 2 * (n & 1);
                        uint32_t w = or_row16(any[n]);
                        w = ~((w & 0x7fff7fffu) + 0x7fff7fffu) & 0x80008000u;  // the top bits of halves that are 0 or -0
                        w = ((w >> 15) | (w >> 30)) & 3u;
                        blank |= (sc.blank >> b) & 1u ? w << (4 * b + s) : 0u;
                    }
                }
#pragma unroll
                for (int ct = 0; ct < kCt; ++ct) st[ct].set_apart(x[ct], f[ct], blank);
            }
        }
        if (sc.nan) {
#pragma unroll
            for (int ct = 0; ct < kCt; ++ct) st[ct].poison(sc.nan, pos0, vis[ct]);
        }
        if constexpr (kMm == 4) values_ahead();
        h8 w[kCt][2], lo[kCt][2];
        if constexpr (Query<T, kC>::kSplit) {
#pragma unroll
            for (int ct = 0; ct < kCt; ++ct) st[ct].settle(x[ct], f[ct], sc, kSlack);
            float load = 0.0f;
#pragma unroll
            for (int ct = 0; ct < kCt; ++ct) st[ct].weigh(x[ct], f[ct], sc, w[ct], lo[ct], st[ct].l, load);
        } else {
            // No maximum over the scores: the weights from the base as it is, and again from a new one where their sums, with
            // and without the value scales, say that one may be too large (2,000 of 8,000 tokens, f16: 14 heads of 64 over 2
            // 398 -> 361 us, 32 of 128 over 8 1,030 -> 1,001; f32, with more registers to keep, 32 of 128 over 8 1,402 and
            // 1,543).
            float sum[kCt];
            bool move = sc.grown != 0;
#pragma unroll
            for (int ct = 0; ct < kCt; ++ct) {
                sum[ct] = 0.0f;
                float load = 0.0f;
                st[ct].weigh(x[ct], f[ct], sc, w[ct], lo[ct], sum[ct], load);
                move |= !(__builtin_fmaf(sum[ct], kMostBare, load) <= kMostWeight) || st[ct].m == -__builtin_inff();
            }
            if (__any(move)) {
#pragma unroll
                for (int ct = 0; ct < kCt; ++ct) {
                    st[ct].settle(x[ct], f[ct], sc, 0.0f);
                    sum[ct] = 0.0f;
                    float load = 0.0f;
                    st[ct].weigh(x[ct], f[ct], sc, w[ct], lo[ct], sum[ct], load);
                }
            }
#pragma unroll
            for (int ct = 0; ct < kCt; ++ct) st[ct].l += sum[ct];
        }
        __builtin_amdgcn_s_setprio(1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int r = 0; r < kOps; ++r) {  // operand r: token pair of blocks r / (4 kC), dimensions by r % (4 kC)
            const int u = r / (4 * kC), i = r % (4 * kC);
#pragma unroll
            for (int ct = 0; ct < kCt; ++ct) {
                f4& o = st[ct].o[i];
                o = __builtin_amdgcn_mfma_f32_16x16x32_f16(vv[r % kDeep], w[ct][u], o, 0, 0, 0);
                if constexpr (Query<T, kC>::kSplit)
                    o = __builtin_amdgcn_mfma_f32_16x16x32_f16(vv[r % kDeep], lo[ct][u], o, 0, 0, 0);
            }
            if (r + kDeep < kOps) vv[r % kDeep] = __builtin_bit_cast(h8, vs[(r + kDeep) * 64]);
        }
#pragma unroll
        for (int r = 0; r < kOps; ++r) {
            __builtin_amdgcn_sched_group_barrier(0x008, kMm, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
    };

    if (t0 < t1) {
        fetch(t0);
        bl = ahead;
        stage(0);
        if (t0 + 1 < t1) fetch(t0 + 1);
    }
    for (int t = t0; t < t0 + steps; ++t) {
        __syncthreads();  // tile t is staged, and tile t - 1 (whose buffer comes next) has been read
        if (kG > 1 && t >= t1) continue;
        if (t > t0 && ((t - t0) & 15) == 0) bl = ahead;
        compute((t - t0) & 1, t);  // past the last tile it stages what it has once more, for nobody
    }
    __builtin_amdgcn_s_setprio(0);

    float mean[kCt];  // what makes the output of a row its weighted mean
#pragma unroll
    for (int ct = 0; ct < kCt; ++ct) {
        st[ct].l = over_groups(st[ct].l, [](float p, float q2) { return p + q2; });
        mean[ct] = over_sum(unit.back(), st[ct].l);
    }
    if constexpr (kG == 2) {
        // the second group's results to the first
        f4* so = reinterpret_cast<f4*>(lds_all) + (tid & 255);
        float* ml = reinterpret_cast<float*>(lds_all + kCt * 4 * kC * 256) + (tid & 255);
        __syncthreads();
        if (grp == 1) {
#pragma unroll
            for (int ct = 0; ct < kCt; ++ct) {
#pragma unroll
                for (int n = 0; n < 4 * kC; ++n) so[(ct * 4 * kC + n) * 256] = st[ct].o[n] * mean[ct];
                ml[512 * ct] = st[ct].m;
                ml[512 * ct + 256] = st[ct].l;
            }
        }
        __syncthreads();
        if (grp == 1) return;
#pragma unroll
        for (int ct = 0; ct < kCt; ++ct) {
            const float m1 = ml[512 * ct], top = __builtin_fmaxf(st[ct].m, m1);
            const float base = top == -__builtin_inff() ? 0.0f : top;
            const float l0 = __builtin_amdgcn_exp2f(st[ct].m - base) * st[ct].l,
                        l1 = __builtin_amdgcn_exp2f(m1 - base) * ml[512 * ct + 256];
            st[ct].m = top;
            st[ct].l = l0 + l1;
            const float f0 = over_sum(l0, st[ct].l), f1 = over_sum(l1, st[ct].l);
#pragma unroll
            for (int n = 0; n < 4 * kC; ++n)
                st[ct].o[n] = st[ct].o[n] * mean[ct] * f0 + so[(ct * 4 * kC + n) * 256] * f1;
            mean[ct] = 1.0f;
        }
    }
#pragma unroll
    for (int ct = 0; ct < kCt; ++ct) {
        const int rr = wave * (16 * kCt) + ct * 16 + col, r = r0 + rr;
        if (r >= e.rows) continue;
        const size_t pr = ((size_t)(item * a.splits + split) * c.n_kv + kvh) * kRows + rr;
        T* out = out_row<T>(a, c, e.row0 + r, kvh);
#pragma unroll
        for (int cc = 0; cc < kC; ++cc)
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const float4 o = make_float4(st[ct].o[4 * cc][s] * mean[ct], st[ct].o[4 * cc + 1][s] * mean[ct],
                                             st[ct].o[4 * cc + 2][s] * mean[ct], st[ct].o[4 * cc + 3][s] * mean[ct]);
                const int d = 64 * cc + 16 * g + 4 * s;
                if (splits == 1)
                    store_out<T, false>(a, out + d, o);
                else
                    *reinterpret_cast<float4*>(a.part_o + pr * kHd + d) = o;
            }
        if (splits > 1 && g == 0) {
            a.part_ml[2 * pr] = st[ct].m;
            a.part_ml[2 * pr + 1] = st[ct].l;
        }
    }
}

// ------------------------------------------------------------------------------------------------ launches

// How a call is split: few rows to an entry take the row kernel (shares over all lengths), many the tile kernel.
struct Plan {
    bool rows;
    int entries;  // of a launch (single tokens)
    int items, shares, splits;
    bool whole;        // a workgroup to a row tile, else shares
    int waves;         // of a workgroup of the row kernels
    int tile;          // rows of an item
    int groups;        // of four waves to a workgroup of the tile kernel
    int join_rows;     // rows of an item that can have partial results; 0: none, and no workspace
    size_t part_rows;  // rows of partial results (per KV head)
    size_t bytes(int n_kv, int hd) const {
        return join_rows ? sizeof(int4) * (size_t)items + sizeof(float) * part_rows * n_kv * (hd + 2) : 0;
    }
};
// capacity: positions that a sequence can have.
Plan plan_of(int group, int n_kv, int hd, int capacity, int n, int n_tok, bool single) {
    const long rows = (long)n_tok * group;
    const int tiles = (group + kRowTile - 1) / kRowTile;  // of a single token
    const long few = single ? (long)n * tiles : rows / kRowTile + n;
    const int cus = device_cus();
    // sequences whole up to 1,024 positions (one token, 14 heads of 64 over 2, f32: over 300 positions 6.1 us, in shares and
    // joined 9.2; 1,024 8.0 and 10.7; 2,048 12.1 and 10.7; 32 heads of 128 over 8: 900 10.9 and 13.0, 2,048 16.5 and
    // 12.8), and where their row tiles fill the GPU up to 2,048 (32 tokens of the latter, f16, over 2,048: 22.0 and 25.8; a
    // batch of unlike lengths lasts as long as its longest, and that no longer than the single one)
    const bool whole = capacity <= kWhole || (capacity <= 2 * kWhole && few * n_kv >= cus);
    // row tiles of a launch
    const long most = whole ? (1 << 23) / n_kv : std::min<long>(kMaxItems, kMaxTiles / ((capacity + kTile - 1) / kTile));
    Plan p{};
    if ((single || few <= most) && rows <= 32l * n) {
        // single tokens in launches of as many entries as make that many row tiles (shares: 2,048 sequences of 2,000, 32
        // heads of 128 over 8, f16: 1,328 us, by the tile kernel 2,803; 14 heads of 64 over 2: 221 and 335)
        p.rows = true;
        p.entries = single && few > most ? (int)(most / tiles) : n;
        p.items = single ? p.entries * tiles : (int)few;
        p.splits = 1;
        p.tile = kRowTile;
        // 8 waves to a workgroup while there is a compute unit for each row tile and KV head. Whole: 32 tokens as above over
        // 1,024 11.8 us, by 4 waves 13.9; 64 tokens 24.6 and 21.9; 2,000 over 100 275 and 120. Shares (one workgroup to a
        // compute unit, half the partial results): 32 over 4,096 46.8 and 51.4; 48 over 2,500 45.3 and 46.8; but 40 over up
        // to 300 23.5 and 12.0, 500 over 100 75 and 53
        p.waves = (long)p.items * n_kv <= cus ? 8 : 4;
        p.whole = whole;
        if (whole) return p;
        p.shares = ((p.waves == 8 ? 1 : 2) * cus + n_kv - 1) / n_kv;
        if (p.shares > kMaxParts) p.shares = kMaxParts;
        p.join_rows = single && group < kRowTile ? group : kRowTile;
        p.part_rows = 2 * (size_t)p.shares * kRowTile;
        return p;
    }
    // 128 rows to a workgroup at head_dim 128 (4 x 2,000 tokens behind 6,000, 32 heads over 8: f16 1,002 us, with 64 rows
    // 1,372; f32 1,404 and 1,648), but 64 where 128 would leave compute units idle, and at head_dim 64, where the longer
    // loop is no faster (14 heads over 2: f32 505 us, with 128 rows 541; f16 361 and 369)
    p.tile = hd == 128 && rows / 128 * n_kv >= cus ? 128 : 64;
    p.items = (int)(rows / p.tile + n);
    const long wgs = (long)p.items * n_kv;
    // Splits for two workgroups of four waves to a compute unit, or one of eight, and no more, which would run after the
    // others (100 tokens behind 8,000, 32 heads of 128 over 8, f16: 43.5 us, rounded up 57.9). Eight waves, whose halves
    // share the positions without a join, where there is a compute unit to each workgroup (14 heads of 64 over 2, f32: a
    // prompt of 512 13.7 us, by four waves 15.9; 64 tokens behind 30,000 45.7 and 55.6), but not where their splits leave
    // a third of the GPU empty (620 tokens behind 4,380 76.2 and 57.2).
    const long room = capacity / (kSplitTiles * kTile);
    auto splits = [&](long places) {
        const long k = std::min({places / wgs, room, 16l});
        return (int)(k > 1 ? k : 1);
    };
    p.groups = wgs <= cus && 5 * 2 * splits(cus) >= 4 * splits(2 * cus) ? 2 : 1;
    p.splits = wgs < cus ? splits(p.groups == 2 ? cus : 2 * cus) : 1;
    p.join_rows = p.splits > 1 ? p.tile : 0;
    p.part_rows = p.splits > 1 ? (size_t)p.items * p.splits * p.tile : 0;
    return p;
}

}  // namespace

size_t kv8_attention_workspace_bytes(int n_heads, int n_kv, int hd, int capacity, int n, int n_tok) {
    const int group = n_heads / n_kv;
    size_t b = plan_of(group, n_kv, hd, capacity, n, n_tok, false).bytes(n_kv, hd);
    if (n == n_tok) {
        const size_t single = plan_of(group, n_kv, hd, capacity, n, n_tok, true).bytes(n_kv, hd);
        b = b > single ? b : single;
    }
    return b;
}

qh_kv8_plan kv8_attention_plan(int n_heads, int n_kv, int hd, int capacity, int n, int n_tok, bool single) {
    const Plan p = plan_of(n_heads / n_kv, n_kv, hd, capacity, n, n_tok, single);
    if (!p.rows) return {QH_KV8_TILES, p.tile, 4 * (p.tile == 64 ? p.groups : 1), p.splits, 1};
    return {p.whole ? QH_KV8_WHOLE : QH_KV8_SHARES, p.tile, p.waves, p.whole ? 1 : p.shares, (n + p.entries - 1) / p.entries};
}

hipError_t launch_kv8_attention(const Kv8View& c, const void* q, void* out, int dtype, int n_heads, int64_t ldq,
                                int64_t ldo, const int32_t* start, const int32_t* seqs, int n, int n_tok, bool causal,
                                float scale, void* ws, hipStream_t s, int8_t* oq, float* od) {
    AttnArgs a{};
    a.q = q;
    a.out = out;
    a.oq = oq;
    a.od = od;
    a.ldq = ldq;
    a.ldo = ldo;
    a.batch = Kv8Batch{start, seqs, n, n_tok, 0};
    a.group = n_heads / c.n_kv;
    a.causal = causal ? 1 : 0;
    a.scale_log2e = scale * 1.44269504088896340736f;
    const Plan p = plan_of(a.group, c.n_kv, c.hd, c.seq_pages << c.page_shift, n, n_tok, start == nullptr);
    a.items = p.items;
    a.splits = p.splits;
    a.rec = static_cast<int4*>(ws);
    a.part_o = reinterpret_cast<float*>(a.rec + p.items);
    a.part_ml = a.part_o + p.part_rows * c.n_kv * c.hd;
    auto go = [&](auto* t, auto kc) {
        using T = std::remove_pointer_t<decltype(t)>;
        constexpr int kC = decltype(kc)::value;
        if (p.rows) {
            const int tiles = (a.group + kRowTile - 1) / kRowTile;
            for (int b = 0; b < n; b += p.entries) {
                a.q = static_cast<const T*>(q) + (int64_t)b * ldq;  // only single tokens take more than one launch
                a.out = static_cast<T*>(out) + (int64_t)b * ldo;
                if (start == nullptr) {
                    const int m = n - b < p.entries ? n - b : p.entries;
                    a.batch = Kv8Batch{nullptr, seqs ? seqs + b : nullptr, m, m, b};
                    a.items = m * tiles;
                }
                const dim3 grid((unsigned)(p.whole ? a.items : p.shares), (unsigned)c.n_kv);
                if (p.whole && p.waves == 8) qh_launch((kv8_whole_kernel<T, kC, 8>), grid, dim3(512), 0, s, c, a);
                else if (p.whole) qh_launch((kv8_whole_kernel<T, kC, 4>), grid, dim3(256), 0, s, c, a);
                else if (p.waves == 8) qh_launch((kv8_rows_kernel<T, kC, 8>), grid, dim3(512), 0, s, c, a);
                else qh_launch((kv8_rows_kernel<T, kC, 4>), grid, dim3(256), 0, s, c, a);
                if (p.join_rows)
                    qh_launch((kv8_join_kernel<T, kC>), dim3((unsigned)a.items, (unsigned)c.n_kv, (unsigned)p.join_rows),
                              dim3(256), 0, s, c, a);
            }
        } else {
            constexpr size_t lds = 2 * 2 * (size_t)kTile * 64 * kC * 2;
            const dim3 grid((unsigned)c.n_kv * (unsigned)p.items, (unsigned)p.splits);
            if constexpr (kC == 2) {
                if (p.tile == 128) qh_launch((kv8_tile_kernel<T, kC, 2, 1>), grid, dim3(256), lds, s, c, a);
            }
            if (p.tile == 64 && p.groups == 2) qh_launch((kv8_tile_kernel<T, kC, 1, 2>), grid, dim3(512), 2 * lds, s, c, a);
            else if (p.tile == 64) qh_launch((kv8_tile_kernel<T, kC, 1, 1>), grid, dim3(256), lds, s, c, a);
            if (p.join_rows)
                qh_launch((kv8_join_splits_kernel<T, kC>),
                          dim3((unsigned)p.items, (unsigned)c.n_kv, (unsigned)(p.join_rows * kC / 16)), dim3(256), 0, s, c,
                          a, p.tile);
        }
    };
    using std::integral_constant;
    if (dtype == QH_F32 && c.hd == 64) go((float*)nullptr, integral_constant<int, 1>{});
    else if (dtype == QH_F32 && c.hd == 128) go((float*)nullptr, integral_constant<int, 2>{});
    else if (dtype == QH_F16 && c.hd == 64) go((_Float16*)nullptr, integral_constant<int, 1>{});
    else if (dtype == QH_F16 && c.hd == 128) go((_Float16*)nullptr, integral_constant<int, 2>{});
    else return hipErrorInvalidValue;
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || !oq || p.rows) return e;
    return launch_quantize_q8(static_cast<const float*>(out), n_tok, n_heads * c.hd, oq, od, s);
}

}  // namespace qh
