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
//   f16: the operands as they are; weights rounded to f16 once, and their sum taken of the rounded ones.
//   f32: every value as three bf16 (8 bits each: the first cut off, the others rounded, the last exact), and of the nine
//   products the six above 2^-22 of the whole: no scale is needed for any range, and a hidden value takes nothing from others.
// A row's base only moves when a tile's sum of weights asks for it (f16: over 2^15, before they leave f16's range), so that
// tiles after the first have no maximum to find. In f16 a new base puts the largest weight at 2^6, clear of the subnormals.
#include <type_traits>

#include "qh_device.h"
#include "qh_kv8.h"
#include "qh_prompt.h"

namespace qh {
namespace {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
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
    static constexpr int kN = 1;
    typedef h8 Op;
    u4 p[1];
};
template <>
struct Parts<float> {
    static constexpr int kN = 3;
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

struct Entry {
    int row0, rows, key0, keys;  // first query row (token) and rows, first key and keys
};

template <typename T, int kHd, int kTile, int kW>
struct Prompt {
    static constexpr int kN = Parts<T>::kN, kRowBytes = 2 * kHd, kPlane = kTile * kRowBytes, kBuffer = 2 * kN * kPlane;
    static constexpr int kRows = 32 * kW, kThreads = 64 * kW, kChunks = kHd / 8;
    static constexpr int kPer = kTile * kChunks / kThreads;  // chunks of keys, and of values, that a thread stages
    static constexpr int kKt = kTile / 32, kDt = kHd / 32, kKs = kHd / 16;
    static_assert(kPer >= 1 && kTile * kChunks % kThreads == 0, "whole chunks to a thread");
};

template <typename T, int kHd, int kTile, int kW>
__global__ __launch_bounds__(64 * kW, 2) void prompt_kernel(PromptArgs a) {
    typedef Prompt<T, kHd, kTile, kW> P;
    constexpr int kN = P::kN, kKt = P::kKt, kDt = P::kDt, kKs = P::kKs, kDeep = 4 / (kN == 3 ? 2 : 1);
    __shared__ __align__(16) uint8_t lds[2 * P::kBuffer];
    __shared__ int odd;  // a value of a tile that is looked at is not finite
    const int tid = (int)threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, half = lane >> 5,
              col = lane & 31;
    const int kvh = (int)(blockIdx.x % (unsigned)a.n_kv), item = a.items - 1 - (int)(blockIdx.x / (unsigned)a.n_kv);
    int from = 0;
    const int b = kv8_entry_of(Kv8Batch{a.start, nullptr, a.n, a.n_tok, 0}, item, a.group, P::kRows, 1, &from);
    if (b < 0) return;
    Entry e;
    {
        auto span = [&](const int32_t* start, int most, int& first, int& n) {
            first = min(max(start[b], 0), most);
            n = max(min(max(start[b + 1], 0), most) - first, 0);
        };
        span(a.start, a.n_tok, e.row0, e.rows);
        span(a.kstart, a.n_keys, e.key0, e.keys);
        e = {__builtin_amdgcn_readfirstlane(e.row0), __builtin_amdgcn_readfirstlane(e.rows),
             __builtin_amdgcn_readfirstlane(e.key0), __builtin_amdgcn_readfirstlane(e.keys)};
    }
    const int rows = e.rows * a.group, r0 = (item - __builtin_amdgcn_readfirstlane(from)) * P::kRows;
    if (r0 >= rows) return;
    // keys that row r sees: its token's own position is keys - rows + token
    auto visible = [&](int r) {
        return a.causal ? min(max(e.keys - e.rows + (int)((unsigned)r / (unsigned)a.group) + 1, 0), e.keys) : e.keys;
    };
    const int last = min(r0 + P::kRows, rows) - 1, seen = visible(last), tiles = (seen + kTile - 1) / kTile;
    const int first_sees = visible(r0);  // every row of the workgroup sees these
    const int w0 = r0 + 32 * wave, r = w0 + col;
    const bool valid = r < rows;
    const int vis = valid ? visible(r) : 0, token = (int)((unsigned)(valid ? r : r0) / (unsigned)a.group);
    const int head = kvh * a.group + ((valid ? r : r0) - token * a.group);
    const int all_see = w0 < rows ? visible(w0) : e.keys;

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
    f16v o[kDt];
#pragma unroll
    for (int d = 0; d < kDt; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] = 0.0f;
    // A new base puts the largest weight at 2^-lift, and a tile's sum asks for one above `limit`. f32: at most 1 / 2 for all
    // weights of a row together, so that no sum of weighted values overflows before it is divided.
    const int shift = kN == 1 ? 0 : 33 - __builtin_clz((unsigned)max(e.keys, 1));
    const float lift = kN == 1 ? -6.0f : (float)(shift + 8);
    const float limit = kN == 1 ? 32768.0f : __builtin_ldexpf((float)(kTile / 2), -shift);
    float base = vis > 0 ? -__builtin_inff() : 0.0f, sum = 0.0f;  // a row that sees nothing asks for no base

    Raw<T> kr[P::kPer], vr[P::kPer];
    const T* const kp = static_cast<const T*>(a.k) + (int64_t)kvh * kHd;
    const T* const vp = static_cast<const T*>(a.v) + (int64_t)kvh * kHd;
    constexpr int kStep = P::kThreads / P::kChunks;  // rows from a thread's chunk to its next
    const T* k_at = kp + (int64_t)(e.key0 + tid / P::kChunks) * a.ldk + 8 * (tid % P::kChunks);  // of the next tile to fetch
    const T* v_at = vp + (int64_t)(e.key0 + tid / P::kChunks) * a.ldv + 8 * (tid % P::kChunks);
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
                const int64_t row = e.key0 + min(t * kTile + i * kStep + tid / P::kChunks, e.keys - 1);
                kr[i].load(kp + row * a.ldk + 8 * (tid % P::kChunks));
                vr[i].load(vp + row * a.ldv + 8 * (tid % P::kChunks));
            }
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
    if (tiles > 0) fetch(0);
    __syncthreads();
    if (tiles > 0) stage(0, 0);
    if (tiles > 1) fetch(1);
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

    for (int t = 0; t < tiles; ++t) {
        const int cur = t & 1;
        const uint8_t* buf = lds + cur * P::kBuffer;
        if (t + 1 < tiles) stage(t + 1, cur ^ 1);
        if (t + 2 < tiles) fetch(t + 2);
        // operands are read kDeep products before their use, and a wave in its products goes before the others of its SIMD
        f16v s[kKt];
        __builtin_amdgcn_s_setprio(1);
        {
            constexpr int kOps = kKt * kKs;
            Parts<T> ring[kDeep];
#pragma unroll
            for (int r = 0; r < kDeep; ++r) ring[r] = key_op(buf, r % kKt, r / kKt);
#pragma unroll
            for (int r = 0; r < kOps; ++r) {  // the tiles in turn, so that a product does not wait for the one before
                const int kt = r % kKt, k = r / kKt;
                if (k == 0) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[kt][i] = 0.0f;
                }
                s[kt] = product<T>(ring[r % kDeep], q[k], s[kt]);
                if (r + kDeep < kOps) ring[r % kDeep] = key_op(buf, (r + kDeep) % kKt, (r + kDeep) / kKt);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        __builtin_amdgcn_s_setprio(0);
        const int pos0 = t * kTile;
        const bool masked = pos0 + kTile > all_see;
        if (masked) {
#pragma unroll
            for (int kt = 0; kt < kKt; ++kt)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    s[kt][i] = pos0 + 32 * kt + 8 * (i >> 2) + 4 * half + (i & 3) < vis ? s[kt][i] : -__builtin_inff();
        }
        // weights 2^(scale s - base) as operands, and their sum
        Parts<T> w[2 * kKt];
        auto weights = [&](float from_base) {
            float l = 0.0f;
#pragma unroll
            for (int u = 0; u < 2 * kKt; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u >> 1][8 * (u & 1) + 2 * i], a.scale_log2e, -from_base));
                    const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u >> 1][8 * (u & 1) + 2 * i + 1], a.scale_log2e, -from_base));
                    if constexpr (kN == 1) {
                        const h2 h = __builtin_convertvector((f2){x, y}, h2);
                        w[u].p[0][i] = __builtin_bit_cast(uint32_t, h);
                        l = __builtin_amdgcn_fdot2(h, (h2){1, 1}, l, false);
                    } else {
                        uint32_t p0, p1, p2;
                        split2<true>(x, y, p0, p1, p2);
                        w[u].p[0][i] = p0, w[u].p[1][i] = p1, w[u].p[2][i] = p2;
                        l += x + y;
                    }
                }
            return l;
        };
        float l = weights(base);
        if (__any(!(l <= limit))) {
            float top = -__builtin_inff();
#pragma unroll
            for (int kt = 0; kt < kKt; ++kt)
#pragma unroll
                for (int i = 0; i < 16; ++i) top = __builtin_fmaxf(top, s[kt][i] * a.scale_log2e);
            top = __builtin_fmaxf(top, other_half(top));
            // only rows that ask for it (either half of one), so that no row depends on its neighbours
            const bool asks = !(__builtin_fmaxf(l, other_half(l)) <= limit) || l != l || other_half(l) != other_half(l);
            const float now = asks ? __builtin_fmaxf(base, top + lift) : base;
            const float f = now == base ? 1.0f : __builtin_amdgcn_exp2f(base - now);
            base = now;
            sum *= f;
#pragma unroll
            for (int d = 0; d < kDt; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[d][i] *= f;
            l = weights(base == -__builtin_inff() ? 0.0f : base);
        }
        sum += l;
        __builtin_amdgcn_s_setprio(1);
        {
            constexpr int kOps = 2 * kKt * kDt;
            Parts<T> ring[kDeep];
#pragma unroll
            for (int r = 0; r < kDeep; ++r) ring[r] = value_op(buf, r / kDt, r % kDt);
#pragma unroll
            for (int r = 0; r < kOps; ++r) {
                o[r % kDt] = product<T>(ring[r % kDeep], w[r / kDt], o[r % kDt]);
                if (r + kDeep < kOps) ring[r % kDeep] = value_op(buf, (r + kDeep) / kDt, (r + kDeep) % kDt);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        __builtin_amdgcn_s_setprio(0);
        __syncthreads();
    }

    sum += other_half(sum);
    if (!valid) return;
    typedef T t4 __attribute__((ext_vector_type(4), aligned(sizeof(T))));
    if (odd) {
        // weights of hidden positions are 0, but 0 times a value that is not finite is NaN, and so are an infinity's products
        // with the parts of a weight: such values, in f16 of the tiles with hidden positions alone, went into the product as
        // zeros, and are added here to the rows that see them
        for (int j = kN == 3 ? 0 : first_sees / kTile * kTile; j < vis; ++j) {
            const T* v = vp + (int64_t)(e.key0 + j) * a.ldv + 4 * half;
#pragma unroll
            for (int d = 0; d < kDt; ++d)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const t4 x = *reinterpret_cast<const t4*>(v + 32 * d + 8 * i);
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (!(__builtin_fabsf((float)x[k]) < __builtin_inff())) o[d][4 * i + k] += (float)x[k];
                }
        }
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

}  // namespace

size_t prompt_workspace_bytes(int, int, int, int, int, int, int) { return 0; }

hipError_t launch_prompt(PromptArgs a, int dtype, int hd, void*, hipStream_t s) {
    auto go = [&](auto* type, auto head, auto tile, auto waves) {
        using T = std::remove_pointer_t<decltype(type)>;
        typedef Prompt<T, decltype(head)::value, decltype(tile)::value, decltype(waves)::value> P;
        a.items = (int)((int64_t)a.n_tok * a.group / P::kRows) + a.n;
        qh_launch((prompt_kernel<T, decltype(head)::value, decltype(tile)::value, decltype(waves)::value>),
                  dim3((unsigned)a.items * (unsigned)a.n_kv), dim3(P::kThreads), 0, s, a);
    };
    using std::integral_constant;
    if (dtype == QH_F16 && hd == 128) go((_Float16*)nullptr, integral_constant<int, 128>{}, integral_constant<int, 64>{}, integral_constant<int, 4>{});
    else if (dtype == QH_F16) go((_Float16*)nullptr, integral_constant<int, 64>{}, integral_constant<int, 64>{}, integral_constant<int, 4>{});
    else if (hd == 128) go((float*)nullptr, integral_constant<int, 128>{}, integral_constant<int, 32>{}, integral_constant<int, 8>{});
    else go((float*)nullptr, integral_constant<int, 64>{}, integral_constant<int, 32>{}, integral_constant<int, 4>{});
    return hipGetLastError();
}

}  // namespace qh
