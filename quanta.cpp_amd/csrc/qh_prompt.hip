// Attention of packed prompts over their own keys and values: out = sum_j softmax_j(scale q . k_j) v_j, in one pass over the
// keys with a running base and sum, a tile of them at a time.
//
// Rows are a sequence's tokens times the query heads of a KV head (row = token * group + head), so that those heads share
// the tile. A wave holds 32 of them; the tile's keys and values lie in shared memory. Scores are computed transposed (keys .
// queries, 32 x 32 x 16): a lane then holds weights of one row alone, next to each other in the order in which the second
// product (values transposed . weights) takes them as its operand, so no weight leaves its lane. That product sums over
// positions, and any order of them does as long as both operands have the same: the operand's element e of lane half h stands
// for position 4 h + e of the first 8 of its 16 positions (e < 4) or of the second (e - 4).
//   Values come out of shared memory transposed (ds_read_b64_tr_b16: 16 lanes read 4 rows of 16 and get 4 positions of a dim
//   each). Rows of shared memory are cut in 16-byte chunks whose places are permuted by the row (swizzle), so that neither the
//   16 rows of a key operand nor the 4 rows of a value operand meet in a bank.
//   f16: the operands as they are; weights rounded to f16 once, and their sum taken of the rounded ones. (With two f16 of each weight
//   the error against 64 bits is 2.05e-4, which the rounding of the result alone is, in place of 2.3e-4 to 2.9e-4; but 12,001 tokens
//   of 32 heads of 128 take 1,599 us in place of 1,176, 16 prompts of up to 2,000 of 14 heads of 64 135 in place of 110, and a token
//   behind 4,000 15.4 in place of 14.4.)
//   f32: every value as three bf16 (8 bits each: the first cut off, the others rounded, the last exact down to bf16's smallest,
//   2^-133), and of the nine products the six above 2^-22 of the whole: no scale is needed, and a hidden value takes nothing from
//   others.
// A row's base only moves when a tile's sum of weights asks for it (f16: over 2^15, before they leave f16's range), so that
// tiles after the first have no maximum to find. In f16 a new base puts the largest weight at 2^6, clear of the subnormals.
#include <type_traits>

#include "qh_device.h"
#include "qh_kv8.h"
#include "qh_prompt.h"

namespace qh {
namespace {

// Key tiles of a split, at least (300 tokens of 32 heads of 128 f32: 23.9 us, with one or four 32; 4 x 64 behind 3,000 of 14 heads
// of 64 f16 18.4, with one 21.1).
constexpr int kSplitTiles = 2;
constexpr int kMaxSplits = 64;

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b2 __attribute__((ext_vector_type(2)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

// Eight values as matrix operands: f16 itself, or three bf16 that add up to the f32.
template <typename T>
struct Parts;
template <>
struct Parts<_Float16> {
    static constexpr int kN = 1, kLong = 20;  // (plan_of)
    typedef h8 Op;
    u4 p[1];
};
template <>
struct Parts<float> {
    static constexpr int kN = 3, kLong = 12;
    typedef b8 Op;
    u4 p[3];
};

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2){a, b}, b2));
}
__device__ __forceinline__ float bf16_lo(uint32_t w) { return __builtin_bit_cast(float, w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __builtin_bit_cast(float, w & 0xffff0000u); }
__device__ __forceinline__ bool infinite(float x) { return __builtin_fabsf(x) == __builtin_inff(); }

// Two f32 as three pairs of bf16. kFinite: no infinities among them, whose rest would be NaN.
template <bool kFinite>
__device__ __forceinline__ void split2(float a, float b, uint32_t& p0, uint32_t& p1, uint32_t& p2) {
    const uint32_t ua = __builtin_bit_cast(uint32_t, a), ub = __builtin_bit_cast(uint32_t, b);
    p0 = __builtin_amdgcn_perm(ub, ua, 0x07060302u);
    float ra = a - __builtin_bit_cast(float, ua & 0xffff0000u), rb = b - __builtin_bit_cast(float, ub & 0xffff0000u);
    if (!kFinite) {
        ra = infinite(a) ? 0.0f : ra;
        rb = infinite(b) ? 0.0f : rb;
    }
    p1 = pack_bf16(ra, rb);
    p2 = pack_bf16(ra - bf16_lo(p1), rb - bf16_hi(p1));
}

template <typename T>
struct Raw;  // eight values as they are in memory, at any address of their type's alignment
template <>
struct Raw<_Float16> {
    typedef uint32_t v __attribute__((ext_vector_type(4), aligned(2)));
    u4 w;
    __device__ __forceinline__ void load(const _Float16* p) { w = *reinterpret_cast<const v*>(p); }
    __device__ __forceinline__ Parts<_Float16> parts() const { return {{w}}; }
    // (a bit cast of a vector's element itself would be one of the vector's first)
    __device__ __forceinline__ h2 pair(int i) const {
        const uint32_t x = w[i];
        return __builtin_bit_cast(h2, x);
    }
    __device__ __forceinline__ bool finite() const {
        h2 z = {0, 0};
#pragma unroll
        for (int i = 0; i < 4; ++i) z += pair(i) * (h2){0, 0};
        return z[0] == (_Float16)0 && z[1] == (_Float16)0;
    }
    __device__ __forceinline__ float value(int i) const { return (float)pair(i >> 1)[i & 1]; }
    __device__ __forceinline__ void clean() {  // values that are not finite become 0
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if ((w[i] & 0x7c00u) == 0x7c00u) w[i] &= 0xffff0000u;
            if ((w[i] & 0x7c000000u) == 0x7c000000u) w[i] &= 0xffffu;
        }
    }
    __device__ __forceinline__ void scale(float f) {
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = __builtin_bit_cast(uint32_t, pair(i) * (h2){(_Float16)f, (_Float16)f});
    }
};
template <>
struct Raw<float> {
    typedef float v __attribute__((ext_vector_type(4), aligned(4)));
    float x[8];
    __device__ __forceinline__ void load(const float* p) {
        const v a = reinterpret_cast<const v*>(p)[0], b = reinterpret_cast<const v*>(p)[1];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = a[i], x[4 + i] = b[i];
    }
    __device__ __forceinline__ Parts<float> parts() const {
        Parts<float> r;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t a, b, c;
            split2<false>(x[2 * i], x[2 * i + 1], a, b, c);
            r.p[0][i] = a, r.p[1][i] = b, r.p[2][i] = c;
        }
        return r;
    }
    __device__ __forceinline__ float value(int i) const { return x[i]; }
    __device__ __forceinline__ void clean() {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = __builtin_fabsf(x[i]) < __builtin_inff() ? x[i] : 0.0f;
    }
    __device__ __forceinline__ void scale(float f) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] *= f;
    }
    __device__ __forceinline__ bool finite() const {
        float z = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) z = __builtin_fmaf(x[i], 0.0f, z);
        return z == 0.0f;
    }
};

__device__ __forceinline__ f16v mma(h8 a, h8 b, f16v c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f16v mma(b8 a, b8 b, f16v c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }

// acc += a . b, the products of the parts that count.
template <typename T>
__device__ __forceinline__ f16v product(const Parts<T>& a, const Parts<T>& b, f16v acc) {
    typedef typename Parts<T>::Op Op;
    auto op = [](u4 w) { return __builtin_bit_cast(Op, w); };
    if constexpr (Parts<T>::kN == 3) {
        acc = mma(op(a.p[0]), op(b.p[2]), acc);
        acc = mma(op(a.p[2]), op(b.p[0]), acc);
        acc = mma(op(a.p[1]), op(b.p[1]), acc);
        acc = mma(op(a.p[0]), op(b.p[1]), acc);
        acc = mma(op(a.p[1]), op(b.p[0]), acc);
    }
    return mma(op(a.p[0]), op(b.p[0]), acc);
}

// The other half wave's value of the same row.
__device__ __forceinline__ float other_half(float v) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return __builtin_bit_cast(float, (uint32_t)((threadIdx.x & 32) ? r[0] : r[1]));
}

// The place of 16-byte chunk c of row r among the row's: rows 4 i .. 4 i + 3 put the four chunks of 32 dims in different
// quarters of 256 bytes, and 16 rows in a row put one chunk in different places.
template <int kHd>
__device__ __forceinline__ int swizzle(int r, int c) {
    if constexpr (kHd == 128) return c ^ (((r & 3) << 2) | ((r >> 2) & 3));
    else return c ^ ((((r >> 1) & 1) << 2) | ((r >> 2) & 3));
}

// Entry b: its first query row (token) and rows, its first key and keys, whatever the starts hold inside the arrays.
struct Entry {
    int row0, rows, key0, keys;
    // keys that row r (token * group + head) sees: its token's own position is keys - rows + token
    __device__ __forceinline__ int visible(const PromptArgs& a, int r) const {
        return a.causal ? min(max(keys - rows + (int)((unsigned)r / (unsigned)a.group) + 1, 0), keys) : keys;
    }
};
// The entry of row tile `item`, false where there is none; *r0: the tile's first row. Up to 63 entries come with one load of
// each list, a lane to a start; more are searched for.
__device__ __forceinline__ bool entry_of(const PromptArgs& a, int item, int tile_rows, Entry* e, int* r0) {
    const int lane = (int)threadIdx.x & 63;
    int b, first, q0, q1, k0, k1;
    if (a.n < 64) {
        const int i = min(lane, a.n), q = min(max(a.start[i], 0), a.n_tok), k = min(max(a.kstart[i], 0), a.n_keys);
        const int key = lane < a.n ? (int)((int64_t)q * a.group / tile_rows) + lane : 0x7fffffff;
        const uint64_t at = __ballot(key <= item);
        if (at == 0) return false;
        b = 63 - __builtin_clzll(at);
        first = __builtin_amdgcn_readlane(key, b);
        q0 = __builtin_amdgcn_readlane(q, b), q1 = __builtin_amdgcn_readlane(q, b + 1);
        k0 = __builtin_amdgcn_readlane(k, b), k1 = __builtin_amdgcn_readlane(k, b + 1);
    } else {
        b = kv8_entry_of(Kv8Batch{a.start, nullptr, a.n, a.n_tok, 0}, item, a.group, tile_rows, 1, &first);
        if (b < 0) return false;
        b = __builtin_amdgcn_readfirstlane(b);
        q0 = min(max(a.start[b], 0), a.n_tok), q1 = min(max(a.start[b + 1], 0), a.n_tok);
        k0 = min(max(a.kstart[b], 0), a.n_keys), k1 = min(max(a.kstart[b + 1], 0), a.n_keys);
    }
    *e = {q0, max(q1 - q0, 0), k0, max(k1 - k0, 0)};
    *r0 = (item - first) * tile_rows;
    return *r0 < e->rows * a.group;
}
// The workgroups that share a row tile's key tiles.
__device__ __forceinline__ int splits_of(const PromptArgs& a, int tiles) { return min(a.splits, max(tiles / kSplitTiles, 1)); }

template <typename T, int kHd, int kTile, int kW>
struct Prompt {
    static constexpr int kN = Parts<T>::kN, kRowBytes = 2 * kHd, kPlane = kTile * kRowBytes, kBuffer = 2 * kN * kPlane;
    static constexpr int kRows = 32 * kW, kThreads = 64 * kW, kChunks = kHd / 8;
    static constexpr int kPer = kTile * kChunks / kThreads;  // chunks of keys, and of values, that a thread stages
    static constexpr int kKt = kTile / 32, kDt = kHd / 32, kKs = kHd / 16;
    static constexpr int kSimdWaves = kThreads / 256 * (160 * 1024 / (2 * kBuffer)) < 2 ? 1 : 2;  // by shared memory, or registers
    static_assert(kPer >= 1 && kTile * kChunks % kThreads == 0, "whole chunks to a thread");
};

// 16 bytes to each lane from its address g (a multiple of 16) into shared memory at `to` (the wave's) + 16 * lane, without a
// register in between. Counted in vmcnt: what reads them is behind wait_loads and a barrier.
__device__ __forceinline__ void load_to_lds(const void* g, uint32_t to) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(g), "s"(to) : "memory", "m0");
}
__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// kDirect: f16 keys and values on multiples of 16 bytes, which go into shared memory as they are, past the registers (12,001
// tokens of 32 heads of 128 over 8: 1,198 us, by registers 1,267).
// Bound by the issue of instructions: that call takes 1,145 to 1,237 us with eight waves on several cards, 1,031 to 954 TFLOP/s, its
// matrix instructions busy for 49% of the cycles and vector instructions issued in 31%; 16 f32 prompts of up to 2,000 tokens of 14
// heads of 64 over 2 take 309 to 329, 47% and 39%; the same prompts in f16 110, 467 TFLOP/s, 19% and 27%. A call of few rows is bound
// by the tiles that a workgroup takes one after the other (512 of those tokens: 14.5 us).
template <typename T, int kHd, int kTile, int kW, bool kDirect>
__global__ __launch_bounds__(64 * kW, (Prompt<T, kHd, kTile, kW>::kSimdWaves)) void prompt_kernel(PromptArgs a) {
    typedef Prompt<T, kHd, kTile, kW> P;
    constexpr int kN = P::kN, kKt = P::kKt, kDt = P::kDt, kKs = P::kKs, kDeep = kN == 1 ? 4 : kHd == 64 ? 2 : 1;
    __shared__ __align__(16) uint8_t lds[2 * P::kBuffer];
    __shared__ int odd;  // a value of a tile that is looked at is not finite
    const int tid = (int)threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, half = lane >> 5,
              col = lane & 31;
    const int kvh = (int)(blockIdx.x % (unsigned)a.n_kv), item = a.items - 1 - (int)(blockIdx.x / (unsigned)a.n_kv);
    Entry e;
    int r0;
    if (!entry_of(a, item, P::kRows, &e, &r0)) return;
    const int rows = e.rows * a.group;
    auto visible = [&](int r) { return e.visible(a, r); };
    const int last = min(r0 + P::kRows, rows) - 1, seen = visible(last), all_tiles = (seen + kTile - 1) / kTile;
    // this workgroup's share of the tiles, where a row tile's are shared out
    const int splits = splits_of(a, all_tiles), split = (int)blockIdx.y;
    if (split >= splits) return;
    const int tile0 = all_tiles * split / splits, tiles = all_tiles * (split + 1) / splits;
    const int first_sees = visible(r0);  // every row of the workgroup sees these
    const int w0 = r0 + 32 * wave, r = w0 + col;
    const bool valid = r < rows;
    const int vis = valid ? visible(r) : 0, token = (int)((unsigned)(valid ? r : r0) / (unsigned)a.group);
    const int head = kvh * a.group + ((valid ? r : r0) - token * a.group);
    const int all_see = w0 < rows ? visible(w0) : e.keys;

    f16v o[kDt];
#pragma unroll
    for (int d = 0; d < kDt; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] = 0.0f;
    // A new base puts the largest weight at 2^-lift, and a tile's sum asks for one above `limit`. f32: at most 1 / 2 for all
    // weights of a row together, so that no sum of weighted values overflows before it is divided (the lift shows in a base up to
    // 2^28; beyond, weights are at most 1 each).
    const int shift = kN == 1 ? 0 : 33 - __builtin_clz((unsigned)max(e.keys, 1));
    const float lift = kN == 1 ? -6.0f : (float)(shift + 8);
    const float limit = kN == 1 ? 32768.0f : __builtin_ldexpf((float)(kTile / 2), -shift);
    float base = vis > 0 ? -__builtin_inff() : 0.0f, sum = 0.0f;  // a row that sees nothing asks for no base
    // A weight is 2^(s * times - base) by one fused step, whose s * times is exact where the base was rounded: they are up to 2^-24 of
    // the base apart, which is nothing up to some 2^20, and from 2^26 on would make weights of 0 or infinity. Rows with such a base have
    // their scores multiplied and rounded first, as the base was, and `times` 1.
    constexpr float kFar = 0x1p20f;
    float times = a.scale_log2e;
    bool any_far = false;

    Raw<T> kr[kDirect ? 1 : P::kPer], vr[kDirect ? 1 : P::kPer];
    const T* const kp = static_cast<const T*>(a.k) + (int64_t)kvh * kHd;
    const T* const vp = static_cast<const T*>(a.v) + (int64_t)kvh * kHd;
    // A thread's chunks: row tid / kChunks and every kStep-th after it; kDirect: the one whose place is the thread's
    constexpr int kStep = P::kThreads / P::kChunks;
    static_assert(kStep % 16 == 0, "the same swizzle for all chunks of a thread");
    const int c_row = tid / P::kChunks, c_at = kDirect ? swizzle<kHd>(c_row, tid % P::kChunks) : tid % P::kChunks;
    const T* k_at = kp + (int64_t)(e.key0 + tile0 * kTile + c_row) * a.ldk + 8 * c_at;  // of the next tile to fetch
    const T* v_at = vp + (int64_t)(e.key0 + tile0 * kTile + c_row) * a.ldv + 8 * c_at;
    auto load_direct = [&](int t, int buf) {
        const uint32_t to = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds + buf * P::kBuffer + 1024 * wave;
        const bool whole = (t + 1) * kTile <= e.keys;
#pragma unroll
        for (int i = 0; i < P::kPer; ++i) {
            const T *k = k_at + i * (kStep * a.ldk), *v = v_at + i * (kStep * a.ldv);
            if (!whole) {  // the last tile: rows that are not there are the last one's
                const int64_t row = e.key0 + min(t * kTile + i * kStep + c_row, e.keys - 1);
                k = kp + row * a.ldk + 8 * c_at;
                v = vp + row * a.ldv + 8 * c_at;
            }
            load_to_lds(k, to + i * (16 * P::kThreads));
            load_to_lds(v, to + P::kPlane + i * (16 * P::kThreads));
        }
        k_at += kTile * a.ldk;
        v_at += kTile * a.ldv;
    };
    // the values of a tile in shared memory that are not finite become 0
    auto clean_direct = [&](int buf) {
#pragma unroll
        for (int i = 0; i < P::kPer; ++i) {
            u4* at = reinterpret_cast<u4*>(lds + buf * P::kBuffer + P::kPlane) + i * P::kThreads + tid;
            Raw<T> v;
            if constexpr (kDirect) v.w = *at;
            if (!v.finite()) {
                v.clean();
                if constexpr (kDirect) *at = v.w;
                odd = 1;
            }
        }
    };
    auto fetch = [&](int t) {
        if ((t + 1) * kTile <= e.keys) {
#pragma unroll
            for (int i = 0; i < P::kPer; ++i) {
                kr[i].load(k_at + i * (kStep * a.ldk));
                vr[i].load(v_at + i * (kStep * a.ldv));
            }
            k_at += kTile * a.ldk;
            v_at += kTile * a.ldv;
        } else {  // the last tile: rows that are not there are the last one's
#pragma unroll
            for (int i = 0; i < P::kPer; ++i) {
                const int64_t row = e.key0 + min(t * kTile + i * kStep + c_row, e.keys - 1);
                kr[i].load(kp + row * a.ldk + 8 * c_at);
                vr[i].load(vp + row * a.ldv + 8 * c_at);
            }
        }
    };
    // f32 heads of 128: the next tile is staged between the products of scores (1,500 tokens of 32 heads over 8: 138.6 us, before
    // them 153.8; heads of 64, whose two workgroups to a compute unit do so by themselves, 316 and 312 for 16 prompts of up to
    // 2,000 tokens). A tile's values that are not finite become 0; then chunk p / 2 of its keys (p even) or values, in parts
    // (behind the last tile the registers hold one that was staged before, and what it writes is not read).
    constexpr bool kWoven = kN == 3 && kHd == 128;
    constexpr int kStaging = 2;
    auto clean = [&]() {
        bool fine = true;
#pragma unroll
        for (int i = 0; i < P::kPer; ++i) fine = fine && vr[kDirect ? 0 : i].finite();
        if (!fine) {
#pragma unroll
            for (int i = 0; i < P::kPer; ++i) vr[kDirect ? 0 : i].clean();
            odd = 1;
        }
    };
    auto stage_piece = [&](int p, int buf) {
        if constexpr (kWoven) {
            const int c = (p >> 1) * P::kThreads + tid, row = c / P::kChunks;
            uint8_t* at = lds + buf * P::kBuffer + row * P::kRowBytes + 16 * swizzle<kHd>(row, c % P::kChunks) + (p & 1) * kN * P::kPlane;
            const Parts<T> x = (p & 1) ? vr[p >> 1].parts() : kr[p >> 1].parts();
#pragma unroll
            for (int i = 0; i < kN; ++i) *reinterpret_cast<u4*>(at + i * P::kPlane) = x.p[i];
        }
    };
    auto stage = [&](int t, int buf) {
        bool fine = true;
#pragma unroll
        for (int i = 0; i < P::kPer; ++i) {
            const int c = i * P::kThreads + tid, row = c / P::kChunks;
            uint8_t* at = lds + buf * P::kBuffer + row * P::kRowBytes + 16 * swizzle<kHd>(row, c % P::kChunks);
            if ((kN == 3 || (t + 1) * kTile > first_sees) && !vr[i].finite()) {
                vr[i].clean();
                fine = false;
            }
            const Parts<T> k = kr[i].parts(), v = vr[i].parts();
#pragma unroll
            for (int p = 0; p < kN; ++p) {
                *reinterpret_cast<u4*>(at + p * P::kPlane) = k.p[p];
                *reinterpret_cast<u4*>(at + (kN + p) * P::kPlane) = v.p[p];
            }
        }
        if (!fine) odd = 1;
    };

    if (tid == 0) odd = 0;
    if constexpr (kDirect) {
        if (tiles > tile0) load_direct(tile0, 0);
    } else {
        if (tiles > tile0) fetch(tile0);
    }
    Parts<T> q[kKs];
    {
        const T* p = static_cast<const T*>(a.q) + (int64_t)(e.row0 + token) * a.ldq + (int64_t)head * kHd + 8 * half;
#pragma unroll
        for (int s = 0; s < kKs; ++s) {
            Raw<T> raw;
            raw.load(p + 16 * s);
            if (a.sign != 1.0f) raw.scale(a.sign);
            q[s] = raw.parts();
            if (!valid) q[s] = Parts<T>{};
        }
    }
    __syncthreads();
    if constexpr (kDirect) {
        wait_loads();
    } else {
        if (tiles > tile0) stage(tile0, 0);
        if (tiles > tile0 + 1) fetch(tile0 + 1);
    }
    __syncthreads();

    // This lane's places in a buffer: row `col` of a key operand, chunk 2 s + half; rows 4 half + lane / 4 % 4 (and 8 more) of
    // a value operand, dims 32 d + 16 (lane / 16 % 2) + 4 (lane % 4)
    const int v_row = 4 * half + ((lane & 15) >> 2), v_chunk = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
    auto key_op = [&](const uint8_t* buf, int kt, int s) {
        Parts<T> r;
        const uint8_t* at = buf + (32 * kt + col) * P::kRowBytes + 16 * swizzle<kHd>(col, 2 * s + half);
#pragma unroll
        for (int p = 0; p < kN; ++p) r.p[p] = *reinterpret_cast<const u4*>(at + p * P::kPlane);
        return r;
    };
    auto value_op = [&](const uint8_t* buf, int u, int d) {
        Parts<T> r;
#pragma unroll
        for (int p = 0; p < kN; ++p) {
            s4 x[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int row = 16 * u + v_row + 8 * j;
                const uint8_t* at = buf + (kN + p) * P::kPlane + row * P::kRowBytes +
                                    16 * swizzle<kHd>(row & 15, 4 * d + v_chunk) + 8 * (lane & 1);
                x[j] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)at);
            }
            typedef short s8 __attribute__((ext_vector_type(8)));
            r.p[p] = __builtin_bit_cast(u4, (s8)__builtin_shufflevector(x[0], x[1], 0, 1, 2, 3, 4, 5, 6, 7));
        }
        return r;
    };

    for (int t = tile0; t < tiles; ++t) {
        const int cur = (t - tile0) & 1;
        const uint8_t* buf = lds + cur * P::kBuffer;
        if constexpr (kDirect) {
            if ((t + 1) * kTile > first_sees) {  // the same for the whole workgroup
                clean_direct(cur);
                __syncthreads();
            }
            if (t + 1 < tiles) load_direct(t + 1, cur ^ 1);
        } else if constexpr (!kWoven) {
            if (t + 1 < tiles) stage(t + 1, cur ^ 1);
            if (t + 2 < tiles) fetch(t + 2);
        } else {
            clean();
        }
        // The tile in blocks of 32 keys. Matrix instructions run in the background of a wave, eight issue slots each, so a block's
        // weights are computed between the products of the next block's scores, and the last block's between the first products
        // with values; operands are read kDeep products before their use, and a wave in its products goes before the others of
        // its SIMD.
        const int pos0 = t * kTile;
        const bool masked = pos0 + kTile > all_see;
        f16v s[kKt];
        Parts<T> w[kKt][2];  // weights 2^(scale s - base) of a block, two operands of 16 keys
        float l[kKt];
        auto mask = [&](int kt) {
            if (masked || any_far) {
                const float before = times == 1.0f ? a.scale_log2e : 1.0f;
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    s[kt][i] = pos0 + 32 * kt + 8 * (i >> 2) + 4 * half + (i & 3) < vis ? s[kt][i] * before : -__builtin_inff();
            }
        };
        auto weights2 = [&](int kt, int n, float from) {  // values 2 n and 2 n + 1 of the block's 16
            const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kt][2 * n], times, -from));
            const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kt][2 * n + 1], times, -from));
            Parts<T>& to = w[kt][n >> 2];
            if (n == 0) l[kt] = 0.0f;
            if constexpr (kN == 1) {
                const h2 h = __builtin_convertvector((f2){x, y}, h2);
                to.p[0][n & 3] = __builtin_bit_cast(uint32_t, h);
                l[kt] = __builtin_amdgcn_fdot2(h, (h2){1, 1}, l[kt], false);
            } else {
                uint32_t p0, p1, p2;
                split2<true>(x, y, p0, p1, p2);
                to.p[0][n & 3] = p0, to.p[1][n & 3] = p1, to.p[2][n & 3] = p2;
                l[kt] += x + y;
            }
        };
        // Products n of the block's (scores kKs, values 2 kDt) with a share of the eight pairs of weights of block `of` (-1: none;
        // kStaging: of the next tile's chunks in their place) after each.
        auto between = [&](int n, int all, int of) {
            if (of == kStaging) {
#pragma unroll
                for (int p = 0; p < 2 * P::kPer; ++p)
                    if (p * all / (2 * P::kPer) == n) stage_piece(p, cur ^ 1);
            } else if (of >= 0) {
#pragma unroll
                for (int p = 0; p < 8; ++p)
                    if (p * all / 8 == n) weights2(of, p, base);
            }
            __builtin_amdgcn_sched_barrier(0);
        };
        auto scores = [&](int kt, int of) {
            Parts<T> ring[kDeep];
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int r = 0; r < kDeep; ++r) ring[r] = key_op(buf, kt, r);
#pragma unroll
            for (int i = 0; i < 16; ++i) s[kt][i] = 0.0f;
#pragma unroll
            for (int r = 0; r < kKs; ++r) {
                s[kt] = product<T>(ring[r % kDeep], q[r], s[kt]);
                if (r + kDeep < kKs) ring[r % kDeep] = key_op(buf, kt, r + kDeep);
                between(r, kKs, of);
            }
            __builtin_amdgcn_s_setprio(0);
        };
        auto values = [&](int kt, int of) {
            constexpr int kOps = 2 * kDt;
            Parts<T> ring[kDeep];
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int r = 0; r < kDeep; ++r) ring[r] = value_op(buf, 2 * kt + r / kDt, r % kDt);
#pragma unroll
            for (int r = 0; r < kOps; ++r) {
                o[r % kDt] = product<T>(ring[r % kDeep], w[kt][r / kDt], o[r % kDt]);
                if (r + kDeep < kOps) ring[r % kDeep] = value_op(buf, 2 * kt + (r + kDeep) / kDt, (r + kDeep) % kDt);
                between(r, kOps, of);
            }
            __builtin_amdgcn_s_setprio(0);
        };
        // a block's weights stand, or its rows get a new base
        auto settle = [&](int kt) {
            if (__any(!(l[kt] <= limit))) {
                float top = -__builtin_inff();
#pragma unroll
                for (int i = 0; i < 16; ++i) top = __builtin_fmaxf(top, s[kt][i] * times);
                top = __builtin_fmaxf(top, other_half(top));
                // only rows that ask for it (either half of one), so that no row depends on its neighbours
                const float both = other_half(l[kt]);
                const bool asks = !(l[kt] <= limit) || !(both <= limit);
                const float now = asks ? __builtin_fmaxf(base, top + lift) : base;
                const float f = now == base ? 1.0f : __builtin_amdgcn_exp2f(base - now);
                base = now;
                const bool far = times != 1.0f && __builtin_fabsf(base) >= kFar && base != -__builtin_inff();
                if (__any(far)) {
                    any_far = true;
                    if (far) {
                        times = 1.0f;
#pragma unroll
                        for (int b = 0; b < kKt; ++b)  // the blocks whose scores stand (a later one is multiplied by its mask)
                            if (b >= kt)
#pragma unroll
                                for (int i = 0; i < 16; ++i) s[b][i] *= a.scale_log2e;
                    }
                }
                sum *= f;
#pragma unroll
                for (int d = 0; d < kDt; ++d)
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[d][i] *= f;
                const float from = base == -__builtin_inff() ? 0.0f : base;
#pragma unroll
                for (int n = 0; n < 8; ++n) weights2(kt, n, from);
            }
            sum += l[kt];
        };
        scores(0, kWoven ? kStaging : -1);
        if constexpr (kWoven) {
            if (t + 2 < tiles) fetch(t + 2);
        }
        mask(0);
        if constexpr (kKt == 1) {
            between(0, 1, 0);
            settle(0);
            values(0, -1);
        } else {
            static_assert(kKt <= 2, "a tile of one or two blocks");
            scores(1, 0);
            mask(1);
            settle(0);
            values(0, 1);
            settle(1);
            values(1, -1);
        }
        if constexpr (kDirect) wait_loads();
        __syncthreads();
    }

    sum += other_half(sum);
    if (w0 >= rows) return;
    // Values that are not finite. Weights of hidden positions are 0, but 0 times such a value is NaN, and so are an infinity's
    // products with the parts of a weight: in f16 of the tiles with hidden positions, in f32 of all, they went into the product as
    // zeros. f16: of a tile that every row sees they went in as they are, and an infinity is NaN where its weight rounds to 0 or a
    // later base scales it by 0 (a NaN without one in the sum comes from values alone; of parts the join looks for such).
    bool lost = false;
    if (kN == 1 && splits == 1) {
#pragma unroll
        for (int d = 0; d < kDt; ++d)
#pragma unroll
            for (int i = 0; i < 16; i += 2) lost = lost || __builtin_isunordered(o[d][i], o[d][i + 1]);
        lost = lost && sum == sum;
    }
    const bool any_lost = __any(lost);
    if (odd || any_lost) {
        // The wave looks for the first position of each dim with a NaN, an infinity and a negative one; a row whose keys reach it
        // has that in the dim, whatever the weight. The values once more for each wave: 12,001 tokens of 32 heads of 128 over 8 with a
        // NaN that all rows see, f16, 2,210 us, without 1,190; 16 f32 prompts 405 and 339 (by each row for itself 60,900 and 1,018).
        // (The buffers are behind their last barrier; a part of one to each wave.)
        int* first = reinterpret_cast<int*>(lds) + wave * 3 * kHd;
        for (int i = lane; i < 3 * kHd; i += 64) first[i] = 0x7fffffff;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
        const int end = min(visible(min(w0 + 31, rows - 1)), tiles * kTile);
        constexpr int kAhead = 4, kStride = 64 / P::kChunks;  // keys of a load
        for (int j = max(tile0, kN == 3 || any_lost ? 0 : first_sees / kTile) * kTile; j < end; j += kAhead * kStride) {
            Raw<T> x[kAhead];
#pragma unroll
            for (int n = 0; n < kAhead; ++n)
                x[n].load(vp + (int64_t)(e.key0 + min(j + n * kStride + lane / P::kChunks, end - 1)) * a.ldv + 8 * (lane % P::kChunks));
#pragma unroll
            for (int n = 0; n < kAhead; ++n) {
                if (x[n].finite()) continue;
                const int at = min(j + n * kStride + lane / P::kChunks, end - 1);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float v = x[n].value(i);
                    if (__builtin_fabsf(v) < __builtin_inff()) continue;
                    int* to = first + (v != v ? 0 : v > 0.0f ? kHd : 2 * kHd) + 8 * (lane % P::kChunks) + i;
                    if (*to > at) atomicMin(to, at);
                }
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
#pragma unroll
        for (int d = 0; d < kDt; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int* at = first + 32 * d + 8 * i + 4 * half;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float is = o[d][4 * i + k];  // an infinity that came through the product
                    const bool nan = at[k] < vis, up = at[kHd + k] < vis || is == __builtin_inff(),
                               down = at[2 * kHd + k] < vis || is == -__builtin_inff();
                    const float strange = nan || (up && down) ? __builtin_nanf("") : up ? __builtin_inff() : -__builtin_inff();
                    o[d][4 * i + k] = nan || up || down ? strange : is;
                }
            }
    }
    if (!valid) return;
    typedef T t4 __attribute__((ext_vector_type(4), aligned(sizeof(T))));
    if (splits > 1) {  // as they are: the join divides
        const size_t row = (((size_t)item * a.n_kv + kvh) * a.splits + split) * P::kRows + (r - r0);
        if (half == 0) reinterpret_cast<float2*>(a.part_ml)[row] = make_float2(base, sum);
        float* part = a.part_o + row * kHd + 4 * half;
#pragma unroll
        for (int d = 0; d < kDt; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<float4*>(part + 32 * d + 8 * i) =
                    make_float4(o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]);
        return;
    }
    const float inv = vis > 0 ? 1.0f / sum : 0.0f;
    T* out = static_cast<T*>(a.out) + (int64_t)(e.row0 + token) * a.ldo + (int64_t)head * kHd + 4 * half;
#pragma unroll
    for (int d = 0; d < kDt; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            t4 x;
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = (T)(o[d][4 * i + j] * inv);
            *reinterpret_cast<t4*>(out + 32 * d + 8 * i) = x;
        }
}

// Joins the parts of the row tiles that were shared out: hd / 4 threads to a row. Bound by latency (512 tokens of 14 heads of 64:
// 4.1 us).
template <typename T, int kHd, int kRows, int kTile>
__global__ __launch_bounds__(256) void prompt_join_kernel(PromptArgs a) {
    constexpr int kThr = kHd / 4, kPer = 256 / kThr;
    const int kvh = (int)(blockIdx.x % (unsigned)a.n_kv), item = (int)(blockIdx.x / (unsigned)a.n_kv);
    Entry e;
    int r0;
    if (!entry_of(a, item, kRows, &e, &r0)) return;
    const int rows = e.rows * a.group;
    const int splits = splits_of(a, (e.visible(a, min(r0 + kRows, rows) - 1) + kTile - 1) / kTile);
    const int r = r0 + (int)blockIdx.y * kPer + (int)threadIdx.x / kThr, d = 4 * ((int)threadIdx.x % kThr);
    if (splits == 1 || r >= rows) return;
    const size_t first = (((size_t)item * a.n_kv + kvh) * a.splits) * kRows + (r - r0);
    const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + first;
    float top = -__builtin_inff(), sum = 0.0f;
    float4 o = make_float4(0, 0, 0, 0);
    constexpr int kAhead = 8;  // parts in flight
    for (int k = 0; k < splits; k += kAhead) {
        float2 m[kAhead];
        float4 v[kAhead];
        float now = top;
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            m[j] = make_float2(-__builtin_inff(), 0.0f);
            v[j] = make_float4(0, 0, 0, 0);
            if (k + j < splits) {
                m[j] = ml[(size_t)(k + j) * kRows];
                v[j] = *reinterpret_cast<const float4*>(a.part_o + (first + (size_t)(k + j) * kRows) * kHd + d);
            }
        }
#pragma unroll
        for (int j = 0; j < kAhead; ++j) now = __builtin_fmaxf(now, m[j].x);
        const float base = now == -__builtin_inff() ? 0.0f : now, f = k > 0 ? __builtin_amdgcn_exp2f(top - base) : 1.0f;
        top = now;
        sum *= f;
        o = make_float4(o.x * f, o.y * f, o.z * f, o.w * f);
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            if (k + j >= splits) break;
            const float w = __builtin_amdgcn_exp2f(m[j].x - base);
            sum = __builtin_fmaf(w, m[j].y, sum);
            o.x = __builtin_fmaf(w, v[j].x, o.x);
            o.y = __builtin_fmaf(w, v[j].y, o.y);
            o.z = __builtin_fmaf(w, v[j].z, o.z);
            o.w = __builtin_fmaf(w, v[j].w, o.w);
        }
    }
    typedef T t4 __attribute__((ext_vector_type(4), aligned(sizeof(T))));
    if ((__builtin_isunordered(o.x, o.y) || __builtin_isunordered(o.z, o.w)) && sum == sum) {
        // a value that is not finite, in a part or by a weight of 0 (lost, above): what the row sees of such is all that counts
        const float was[4] = {o.x, o.y, o.z, o.w};
        float f[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = was[i] == was[i] ? was[i] : 0.0f;
        const T* v = static_cast<const T*>(a.v) + (int64_t)e.key0 * a.ldv + (int64_t)kvh * kHd + d;
        const int vis = e.visible(a, r);
        constexpr int kLook = 16;
        for (int j = 0; j < vis; j += kLook) {
            t4 x[kLook];
#pragma unroll
            for (int n = 0; n < kLook; ++n) x[n] = *reinterpret_cast<const t4*>(v + (int64_t)min(j + n, vis - 1) * a.ldv);
#pragma unroll
            for (int n = 0; n < kLook; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (!(__builtin_fabsf((float)x[n][i]) < __builtin_inff())) f[i] += (float)x[n][i];
            bool found = true;  // a NaN, or both infinities, in all that were NaN
#pragma unroll
            for (int i = 0; i < 4; ++i) found = found && (was[i] == was[i] || f[i] != f[i]);
            if (found) break;
        }
        o = make_float4(f[0], f[1], f[2], f[3]);
    }
    const int token = (int)((unsigned)r / (unsigned)a.group), head = kvh * a.group + (r - token * a.group);
    const float inv = e.visible(a, r) > 0 ? 1.0f / sum : 0.0f;
    *reinterpret_cast<t4*>(static_cast<T*>(a.out) + (int64_t)(e.row0 + token) * a.ldo + (int64_t)head * kHd + d) =
        (t4){(T)(o.x * inv), (T)(o.y * inv), (T)(o.z * inv), (T)(o.w * inv)};
}

// Calls f with the element type and, as constants, head_dim, keys of a tile and waves: eight where that leaves a row tile to
// every compute unit, else four (12,001 tokens of 32 heads of 128 over 8, f16, timed in turn: 1,149 us and, with four, 1,186; on
// another card 1,237 and 1,284; with fewer row tiles, f16, 1,500 tokens of 14 heads of 64 over 2: 26.7 and, with four, 24.3; f32, 300
// of 32 of 128: 28.7 and 24.0). f32 heads of 64 stay with four, whose workgroups do not wait for each other (16 prompts of up to 2,000 tokens: 322 us, eight waves over 64 keys
// 340).
template <typename F>
void by_shape(int dtype, int hd, int group, int n_kv, int n_tok, F&& f) {
    using std::integral_constant;
    typedef integral_constant<int, 32> K32;
    typedef integral_constant<int, 64> K64;
    typedef integral_constant<int, 128> K128;
    typedef integral_constant<int, 4> W4;
    typedef integral_constant<int, 8> W8;
    const bool many = (int64_t)n_tok * group / 256 * n_kv >= device_cus();
    if (dtype == QH_F16 && hd == 128 && many) f((_Float16*)nullptr, K128{}, K64{}, W8{});
    else if (dtype == QH_F16 && hd == 128) f((_Float16*)nullptr, K128{}, K64{}, W4{});
    else if (dtype == QH_F16 && many) f((_Float16*)nullptr, K64{}, K64{}, W8{});
    else if (dtype == QH_F16) f((_Float16*)nullptr, K64{}, K64{}, W4{});
    else if (hd == 128 && many) f((float*)nullptr, K128{}, K32{}, W8{});
    else if (hd == 128) f((float*)nullptr, K128{}, K32{}, W4{});
    else f((float*)nullptr, K64{}, K32{}, W4{});
}

// Row tiles of a call, and how many workgroups may share one where the row tiles are fewer than the compute units: a workgroup to
// a compute unit, or two where one would still have more than `long_way` key tiles one after the other (f32 12: 512 tokens of 14
// heads of 64 18.1 us, with two 20.5, 1,000 36.8 and 30.6; f16 20: 8 prompts of up to 300 behind 500 17.3 and 21.4, 1,500 tokens
// 25.3 and 24.5), by the entries' mean length, which is all that the host knows of them.
struct Plan {
    int items, splits;
};
Plan plan_of(int rows, int tile, int long_way, int group, int n_kv, int n, int n_tok, int n_keys) {
    Plan p;
    p.items = (int)((int64_t)n_tok * group / rows) + n;
    const int64_t tiles = ((int64_t)n_tok * group + rows - 1) / rows, wgs = (tiles > n ? tiles : n) * n_kv;
    const int64_t keys = n_keys / n / tile, most = keys / kSplitTiles;
    int64_t s = device_cus() / (wgs > 0 ? wgs : 1);
    if (keys > long_way * (s > 1 ? s : 1)) s = 2 * device_cus() / (wgs > 0 ? wgs : 1);
    s = s < most ? s : most;
    p.splits = (int)(s < 1 ? 1 : s < kMaxSplits ? s : kMaxSplits);
    return p;
}

}  // namespace

size_t prompt_workspace_bytes(int dtype, int n_heads, int n_kv, int hd, int n, int n_tok, int n_keys) {
    size_t bytes = 0;
    by_shape(dtype, hd, n_heads / n_kv, n_kv, n_tok, [&](auto* type, auto, auto tile, auto waves) {
        constexpr int kRows = 32 * decltype(waves)::value, kLong = Parts<std::remove_pointer_t<decltype(type)>>::kLong;
        const Plan p = plan_of(kRows, decltype(tile)::value, kLong, n_heads / n_kv, n_kv, n, n_tok, n_keys);
        if (p.splits > 1) bytes = (size_t)p.items * n_kv * p.splits * kRows * (hd + 2) * sizeof(float);
    });
    return bytes;
}

hipError_t launch_prompt(PromptArgs a, int dtype, int hd, void* ws, hipStream_t s) {
    hipError_t rc = hipSuccess;
    by_shape(dtype, hd, a.group, a.n_kv, a.n_tok, [&](auto* type, auto head, auto tile, auto waves) {
        using T = std::remove_pointer_t<decltype(type)>;
        constexpr int kHd = decltype(head)::value, kTile = decltype(tile)::value, kW = decltype(waves)::value, kRows = 32 * kW;
        const Plan p = plan_of(kRows, kTile, Parts<T>::kLong, a.group, a.n_kv, a.n, a.n_tok, a.n_keys);
        a.items = p.items, a.splits = p.splits;
        a.part_o = static_cast<float*>(ws);
        a.part_ml = a.part_o + (size_t)p.items * a.n_kv * p.splits * kRows * hd;
        const unsigned wgs = (unsigned)p.items * (unsigned)a.n_kv;
        const dim3 grid(wgs, (unsigned)p.splits);
        bool direct = false;
        if constexpr (std::is_same<T, _Float16>::value) {
            direct = ((reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v)) & 15) == 0 && a.ldk % 8 == 0 && a.ldv % 8 == 0;
            if (direct) qh_launch((prompt_kernel<T, kHd, kTile, kW, true>), grid, dim3(64 * kW), 0, s, a);
        }
        if (!direct) qh_launch((prompt_kernel<T, kHd, kTile, kW, false>), grid, dim3(64 * kW), 0, s, a);
        if ((rc = hipGetLastError()) != hipSuccess || p.splits == 1) return;
        qh_launch((prompt_join_kernel<T, kHd, kRows, kTile>), dim3(wgs, (unsigned)(kRows * kHd / 1024)), dim3(256), 0, s, a);
        rc = hipGetLastError();
    });
    return rc;
}

}  // namespace qh
