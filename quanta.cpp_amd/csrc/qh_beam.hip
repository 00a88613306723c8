// Beam search's selection: of each prompt's beams b and ids v, the k candidates with the largest
//     score_b + logit_bv - log sum_u exp(logit_bu),
// ties to the lower (b, v). Two launches:
//   1. over the whole GPU (beam_rows_kernel): every logit once, for the largest of each group of ids and, wave by wave, the
//      sum of exponentials. Bound by memory (192 x 151,936 f32: 26.9 us, 4.3 TB/s with start and end).
//   2. a workgroup to a prompt (beam_pick_kernel): the rows' sums, then the k best groups by their largest candidate (a
//      group that is not among them holds none of the k best candidates, for k others have one before its own best), and
//      the k best of what those groups hold. Bound by latency: sums, groups, their logits and ranks wait for each other, and
//      what sixteen waves all compute costs each SIMD four times (4 beams 5.3 us, 24 prompts of 8 8.7).
// Candidates of different rows meet in the order of their scores, so sums, exponentials and scores are 64-bit: rounded to
// f32, scores that are 2^-20 apart would tie. (A 64-bit multiply-add takes no longer than a 32-bit one here.)
#include "qh_device.h"
#include "qh_rows.h"

namespace qh {
namespace {

constexpr int kPickThreads = 1024;
constexpr int kPool = kPickThreads;  // candidates that are held, one to a thread
constexpr int kList = QH_BEAM_MAX_K + 16;  // groups that are read again, at most

template <typename T>
constexpr int kE = 16 / (int)sizeof(T);
// Loads of a wave in flight, or a group's (192 x 151,936 f32, groups of 4: 26.8 us, with 8 28.2, with 16 32.2; 512 x 50,257 f16
// 24.2, with 4 38).
constexpr int kMostVecs = 2;
template <typename T>
struct Vec {  // at any address of the type's alignment
    typedef T type __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
};

// How the rows are cut: a workgroup's part of a row is four waves' `vecs` vectors of 64 * E ids, a group `group` of them: one
// where that leaves a group to a thread of the picking workgroup, or four and the k best may take most of a row's larger ones
// (64 of 16 beams of 50,257 f16, 8 prompts: 25.5 us, with groups of 1,024 ids 44.9), else 1,024 ids (24 prompts of 4 beams of
// 151,936 f32: 22.2 us, of 256 28.2), or 2,048 where a thread had more than 32.
struct BeamCut {
    int vecs, group;
    int parts, groups;  // of a row
};

template <typename T>
BeamCut beam_cut(int rows, int beams, int n_valid, int k) {
    const int v = (n_valid + 64 * kE<T> - 1) / (64 * kE<T>), wide = 1024 / (64 * kE<T>);
    BeamCut c{};
    const bool small = beams * v <= kPickThreads || (beams * v <= 4 * kPickThreads && 2 * k > (v + wide - 1) / wide);
    c.group = small ? 1 : wide;
    if ((int64_t)beams * ((v + c.group - 1) / c.group) > 32 * kPickThreads) c.group *= 2;
    c.vecs = kMostVecs > c.group ? kMostVecs : c.group;  // fewer where there are not workgroups enough
    while (c.vecs > c.group && (int64_t)rows * ((v + 4 * c.vecs - 1) / (4 * c.vecs)) < 1024) c.vecs /= 2;
    c.parts = (v + 4 * c.vecs - 1) / (4 * c.vecs);
    c.groups = (v + c.group - 1) / c.group;
    return c;
}

// 2^(n + f) for a polynomial of f, |f| <= 1/2, off by 2^-38 of it at most: it interpolates (2^f - 1) / f at the Chebyshev
// nodes, and 2^0 is 1. n is the low word of `k`, a number beside 1.5 * 2^52, and goes into the exponent as an integer.
constexpr double kLog2e = 0x1.71547652b82fep+0, kShift = 0x1.8p+52;
__device__ __forceinline__ double exp2_parts(double f, double k) {
    double p = 0x1.63b2d7971923fp-20;
    p = __builtin_fma(p, f, 0x1.00c0e4e15189cp-16);
    p = __builtin_fma(p, f, 0x1.4308c7183d6a2p-13);
    p = __builtin_fma(p, f, 0x1.5d877598350dep-10);
    p = __builtin_fma(p, f, 0x1.3b2ab70ad2565p-7);
    p = __builtin_fma(p, f, 0x1.c6b08da70cce3p-5);
    p = __builtin_fma(p, f, 0x1.ebfbdff82a734p-3);
    p = __builtin_fma(p, f, 0x1.62e42fef9cc69p-1);
    p = __builtin_fma(p, f, 1.0);
    typedef uint32_t u2 __attribute__((ext_vector_type(2)));
    const u2 w = __builtin_bit_cast(u2, p), n = __builtin_bit_cast(u2, k);
    return __builtin_bit_cast(double, (u2){w.x, w.y + (n.x << 20)});
}
// exp(d) for d <= 1. From -700 down the result stays at 2^-1010, which no sum of logits notices.
__device__ __forceinline__ double exp_below(double d) {
    d = __builtin_fmax(d, -700.0);
    const double k = __builtin_fma(d, kLog2e, kShift);
    return exp2_parts(__builtin_fma(d, kLog2e, kShift - k), k);
}

template <typename T, int kVecs>
__global__ __launch_bounds__(256) void beam_rows_kernel(const T* __restrict__ logits, int64_t ld, int n_valid,
                                                        BeamCut cut, uint32_t part_magic, float* __restrict__ gmax,
                                                        float* __restrict__ pmax, double* __restrict__ psum) {
    constexpr int E = kE<T>;
    __shared__ float wave_max[4];
    __shared__ double wave_sum[4];
    const int row = (int)(part_magic ? div_magic(blockIdx.x, part_magic) : blockIdx.x), part = (int)blockIdx.x - row * cut.parts;
    const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6, first = (4 * part + wave) * kVecs;
    const T* x = logits + (int64_t)row * ld;
    typename Vec<T>::type raw[kVecs];
    if ((first + kVecs) * 64 * E <= n_valid) {  // (a branch of single lanes would have every load waited for by itself)
#pragma unroll
        for (int j = 0; j < kVecs; ++j)
            raw[j] = *reinterpret_cast<const typename Vec<T>::type*>(x + ((first + j) * 64 + lane) * E);
    } else {
#pragma unroll
        for (int j = 0; j < kVecs; ++j) {
            const int i = ((first + j) * 64 + lane) * E;
            if (i + E <= n_valid) {
                raw[j] = *reinterpret_cast<const typename Vec<T>::type*>(x + i);
            } else {
#pragma unroll
                for (int e = 0; e < E; ++e) raw[j][e] = i + e < n_valid ? x[i + e] : (T)-__builtin_inff();
            }
        }
    }
    float m = -__builtin_inff(), g = m;  // maxima pass over a NaN, which the sum does not
    bool nan = false;
#pragma unroll
    for (int j = 0; j < kVecs; ++j) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float v = (float)raw[j][e];
            g = __builtin_fmaxf(g, v);
            nan |= v != v;
        }
        if (((j + 1) & (cut.group - 1)) == 0) {  // uniform: groups begin at multiples of their size, and so do parts
            g = wave_reduce32x2(g, [](float a, float b) { return __builtin_fmaxf(a, b); });
            const int at = (first + j) / cut.group;
            if (lane == 0 && at < cut.groups) gmax[(size_t)row * cut.groups + at] = g;
            m = __builtin_fmaxf(m, g);
            g = -__builtin_inff();
        }
    }
    double s = 0.0;
    if (__builtin_fabsf(m) <= 4096.0f) {
        // relative to 2^at, the power of two next to exp(m), which n takes up: a logit's product with log2(e) rounds to an integer
        // beside kShift - at, and the rest of it is exact before its own rounding
        const double at = __builtin_rint((double)m * kLog2e), a = kShift - at;
        const float low = m - 690.0f;
#pragma unroll
        for (int j = 0; j < kVecs; ++j)
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const double x = (double)__builtin_amdgcn_fmed3f((float)raw[j][e], low, __builtin_inff());
                const double k = __builtin_fma(x, kLog2e, a);
                s += exp2_parts(__builtin_fma(x, kLog2e, a - k), k);
            }
        s = wave_reduce32x2(s, [](double p, double q) { return p + q; });
        s *= exp_below(at * 0x1.62e42fefa39efp-1 - (double)m);  // relative to exp(m)
    } else {
        const double base = (double)__builtin_fmaxf(m, -0x1.fffffep127f);  // a part without a finite logit sums to 0 or so
        for (int j = 0; j < kVecs; ++j)
            for (int e = 0; e < E; ++e) s += exp_below((double)(float)raw[j][e] - base);
        s = wave_reduce32x2(s, [](double p, double q) { return p + q; });
    }
    if (__any(nan) || m == __builtin_inff()) s = __builtin_nan("");
    if (lane == 0) {
        wave_max[wave] = m;
        wave_sum[wave] = s;
    }
    __syncthreads();
    if (threadIdx.x < 64) {  // lane w takes wave w's
        const float mine = wave_max[lane & 3];
        const float top = __builtin_fmaxf(__builtin_fmaxf(wave_max[0], wave_max[1]), __builtin_fmaxf(wave_max[2], wave_max[3]));
        double all = wave_sum[lane & 3] * exp_below((double)mine - (double)__builtin_fmaxf(top, -0x1.fffffep127f));
        all += __shfl_xor(all, 1);
        all += __shfl_xor(all, 2);
        if (lane == 0) {
            pmax[(size_t)row * cut.parts + part] = top;
            psum[(size_t)row * cut.parts + part] = all;
        }
    }
}

// Monotone map of a finite f64 onto uint64, above 0 (which stands for "no candidate").
__device__ __forceinline__ uint64_t ordered_f64(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    return (u >> 63) ? ~u : (u | ((uint64_t)1 << 63));
}
constexpr uint64_t kLeastKey = (uint64_t)1 << 52;  // of the lowest finite f64: those below stand for no number
__device__ __forceinline__ double from_ordered_f64(uint64_t k) {
    return __builtin_bit_cast(double, (k >> 63) ? (k & ~((uint64_t)1 << 63)) : ~k);
}

// A value that is the same in all lanes, in scalar registers.
__device__ __forceinline__ uint64_t scalar(uint64_t v) {
    return (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32 |
           (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)v);
}

// A candidate's place in the order: a larger key first, then a lower index. Those up to a limit are taken.
struct Limit {
    uint64_t key;
    uint32_t index;
    __device__ __forceinline__ bool takes(uint64_t k, uint32_t i) const { return k > key || (k == key && i <= index); }
};

// Sum over the 16 lanes of each row of the wave.
__device__ __forceinline__ uint32_t sum_row16(uint32_t x) {
    x += (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x128, 0xF, 0xF, false);
    x += (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x124, 0xF, 0xF, false);
    x += (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x122, 0xF, 0xF, false);
    return x + (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x121, 0xF, 0xF, false);
}
// The largest of the 16 lanes of each row of the wave.
__device__ __forceinline__ uint64_t max_row16(uint64_t v) {
    auto step = [&](auto ror) {
        const uint32_t lo = (uint32_t)__builtin_amdgcn_mov_dpp((int)(uint32_t)v, decltype(ror)::value, 0xF, 0xF, false),
                       hi = (uint32_t)__builtin_amdgcn_mov_dpp((int)(v >> 32), decltype(ror)::value, 0xF, 0xF, false);
        const uint64_t u = (uint64_t)hi << 32 | lo;
        v = u > v ? u : v;
    };
    step(std::integral_constant<int, 0x128>{});
    step(std::integral_constant<int, 0x124>{});
    step(std::integral_constant<int, 0x122>{});
    step(std::integral_constant<int, 0x121>{});
    return v;
}

// Sum over the workgroup of what its waves count (the same in a wave's lanes), for every thread. `red` holds 16 values for each
// parity of `turn`, so that a call needs one barrier.
__device__ __forceinline__ int wg_sum(int v, int (*red)[16], int& turn) {
    int* r = red[turn & 1];
    ++turn;
    if ((threadIdx.x & 63) == 0) r[threadIdx.x >> 6] = v;
    __syncthreads();
    return __builtin_amdgcn_readfirstlane((int)sum_row16((uint32_t)r[threadIdx.x & 15]));
}

// A limit that takes at least k and at most `most` of the candidates that count(limit) counts (the workgroup's, the same for
// every thread), or all where there are fewer; top: a key that none is above. Steps down from the top, four times as far
// each time, halves the keys between the last two steps, and then, where more than `most` share one key, the indexes.
template <typename Count>
__device__ __forceinline__ Limit find_limit(uint64_t top, int k, int most, Count&& count) {
    constexpr uint32_t kAny = 0xffffffffu;
    uint64_t lo = 1, hi = top + 1;  // at least k at lo and above, fewer than k at hi and above
    for (uint64_t step = (uint64_t)1 << 49;;) {  // 2^49: 2 of a score between 16 and 32
        const uint64_t at = hi - 1 > step ? hi - step : 1;
        const int n = count(Limit{at, kAny});
        if (n <= most && (n >= k || at == 1)) return Limit{at, kAny};
        if (n >= k) {
            lo = at;
            break;
        }
        hi = at;
        step = step < (uint64_t)1 << 60 ? 4 * step : ~(uint64_t)0;
    }
    while (hi - lo > 1) {
        const uint64_t mid = lo + (hi - lo) / 2;
        const int n = count(Limit{mid, kAny});
        if (n < k) hi = mid;
        else if (n <= most) return Limit{mid, kAny};
        else lo = mid;
    }
    uint32_t a = 0, b = kAny;  // fewer than k up to index a - 1, at least k up to b
    while (a < b) {
        const uint32_t mid = a + (b - a) / 2;
        const int n = count(Limit{lo, mid});
        if (n < k) a = mid + 1;
        else if (n <= most) return Limit{lo, mid};
        else b = mid;
    }
    return Limit{lo, b};
}

// kKeys: groups to a thread, at most; kGroup: vectors of a group.
template <typename T, int kKeys, int kGroup>
__global__ __launch_bounds__(kPickThreads) void beam_pick_kernel(const T* __restrict__ logits, int64_t ld,
                                                                 const float* __restrict__ scores, int beams, int n_valid,
                                                                 int k, BeamCut cut, uint32_t group_magic,
                                                                 const float* __restrict__ gmax,
                                                                 const float* __restrict__ pmax,
                                                                 const double* __restrict__ psum, int32_t* __restrict__ parent,
                                                                 int32_t* __restrict__ token, float* __restrict__ best) {
    constexpr int E = kE<T>;
    __shared__ double row_max[QH_BEAM_MAX_BEAMS], row_add[QH_BEAM_MAX_BEAMS];  // a NaN sum: a row without candidates
    __shared__ uint64_t pool_key[kPool];
    __shared__ uint32_t pool_at[kPool];
    __shared__ int list[kList];
    __shared__ int red[2][16];
    __shared__ uint64_t cell[64], least_key;
    __shared__ int n_list, n_pool;
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int prompt = (int)blockIdx.x, row0 = prompt * beams;
    if (tid == 0) least_key = 0, n_list = n_pool = 0;
    const int n_groups = beams * cut.groups;
    // groups of 16 lanes take every 64th group, so that those of one row, which may hold all the best, are with all of them
    const int mine = (tid & 15) * 64 + (tid >> 4);
    float best_of[kKeys];  // in flight while the rows are summed
#pragma unroll
    for (int j = 0; j < kKeys; ++j) {
        const int i = j * kPickThreads + mine;
        best_of[j] = i < n_groups ? gmax[(size_t)row0 * cut.groups + i] : -__builtin_inff();
    }
    for (int b = wave; b < beams; b += 16) {
        const float* pm = pmax + (size_t)(row0 + b) * cut.parts;
        const double* ps = psum + (size_t)(row0 + b) * cut.parts;
        constexpr int kHeld = 4;  // parts of a lane: a row has 64 at most, or 256 where a group is one vector
        float m[kHeld], top = -__builtin_inff();
        double p[kHeld];
#pragma unroll
        for (int j = 0; j < kHeld; ++j) {
            const int i = 64 * j + lane;
            m[j] = i < cut.parts ? pm[i] : -__builtin_inff();
            p[j] = i < cut.parts ? ps[i] : 0.0;
        }
        const double score = scores ? (double)scores[row0 + b] : 0.0;
#pragma unroll
        for (int j = 0; j < kHeld; ++j) top = __builtin_fmaxf(top, m[j]);
        top = wave_reduce32x2(top, [](float x, float y) { return __builtin_fmaxf(x, y); });
        const double base = (double)__builtin_fmaxf(top, -0x1.fffffep127f);
        double s = 0.0;
#pragma unroll
        for (int j = 0; j < kHeld; ++j) s += p[j] * exp_below((double)m[j] - base);
        s = wave_reduce32x2(s, [](double x, double y) { return x + y; });
        if (lane == 0) {
            const bool fine = s > 0.0 && s < __builtin_inf() && __builtin_fabs(score) < __builtin_inf();
            row_max[b] = base;
            row_add[b] = fine ? score - ::log(s) : __builtin_nan("");
        }
    }
    __syncthreads();
    // the order of candidates: by the score in 64 bits; a logit of -inf (or NaN) is none
    auto key_of = [&](float x, int b) {
        const double v = ((double)x - row_max[b]) + row_add[b];
        return __builtin_fabs(v) < __builtin_inf() ? ordered_f64(v) : (uint64_t)0;
    };
    static_assert((int64_t)QH_BEAM_MAX_BEAMS * QH_SAMPLE_MAX_VOCAB <= (int64_t)1 << 32, "an id and its beam in 32 bits");
    auto index_of = [](int b, int id) { return (uint32_t)b * QH_SAMPLE_MAX_VOCAB + (uint32_t)id; };
    // 1. the groups
    uint64_t key[kKeys], top = 0;  // the largest key is that of a row's largest logit, which is row_add
    {
        double t = -__builtin_inff();
        for (int b = lane; b < beams; b += 64) t = __builtin_fmax(t, row_add[b]);
        t = wave_reduce32x2(t, [](double x, double y) { return __builtin_fmax(x, y); });
        if (t > -__builtin_inff()) top = ordered_f64(t);
        top = scalar(top);
    }
#pragma unroll
    for (int j = 0; j < kKeys; ++j) {
        const int i = j * kPickThreads + mine;
        key[j] = 0;
        if (i < n_groups) key[j] = key_of(best_of[j], (int)(group_magic ? div_magic((uint32_t)i, group_magic) : (uint32_t)i));
    }
    auto to_list = [&](const Limit& l) {
#pragma unroll
        for (int j = 0; j < kKeys; ++j) {
            const int i = j * kPickThreads + mine;
            if (l.takes(key[j], (uint32_t)i)) {
                const int at = atomicAdd(&n_list, 1);
                if (at < kList) list[at] = i;
            }
        }
        __syncthreads();
    };
    int turn = 0;
    Limit groups{1, 0xffffffffu};
    if (k <= 32) {
        // the k-th largest of the 64 maxima of 16 lanes: k groups or more are at or above it, and rarely more than k + 16
        uint64_t m = key[0];
#pragma unroll
        for (int j = 1; j < kKeys; ++j) m = key[j] > m ? key[j] : m;
        m = max_row16(m);
        if ((lane & 15) == 0) cell[tid >> 4] = m;
        __syncthreads();
        m = cell[lane];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const uint64_t c = scalar(cell[4 * wave + q]);
            const int above = __builtin_popcountll(__ballot(m > c)), up_to = __builtin_popcountll(__ballot(m >= c));
            if (lane == 0 && above < k && up_to >= k) least_key = c;
        }
        __syncthreads();
        const uint64_t least = scalar(least_key);
        if (least > 1) groups.key = least;
        to_list(groups);
    }
    if (k > 32 || __builtin_amdgcn_readfirstlane(n_list) > k + 16) {
        groups = find_limit(top, k, k + 16, [&](const Limit& l) {
            int n = 0;
#pragma unroll
            for (int j = 0; j < kKeys; ++j) n += __builtin_popcountll(__ballot(l.takes(key[j], (uint32_t)(j * kPickThreads + mine))));
            return wg_sum(n, red, turn);
        });
        if (tid == 0) n_list = 0;
        __syncthreads();
        to_list(groups);
    }
    // 2. their candidates: where k groups are listed, k of their best are at the limit's key or above, so only such ones count
    const int listed = __builtin_amdgcn_readfirstlane(n_list);
    // f(logit, row, id) of every id of the listed groups whose logit can reach the limit, a wave to a group. A logit x is left out
    // only where its key lies below the limit's, so that counts by f are the counts of the keys themselves (else the search for a
    // limit below need not end). A key's score (x - u) + row_add reaches `goal` only where x - u >= (goal - row_add), less the
    // roundings of the sum, at most 2^-53 of goal, and of t, u and x - u, 2^-53 of each and of row_add; 2^-51 and 2^-22 are more.
    // (The rounding to f32 leaves out nothing: x is an f32.)
    constexpr int kAhead = kKeys <= 4 ? 2 : 1;  // groups of a wave in flight (as many as its registers hold)
    auto each = [&](uint64_t limit_key, auto&& f) {
        const double goal = limit_key >= kLeastKey ? from_ordered_f64(limit_key) : -__builtin_inff();
        for (int w = wave; w < listed; w += 16 * kAhead) {
            typename Vec<T>::type v[kAhead][kGroup];
            int row[kAhead], id0[kAhead];
#pragma unroll
            for (int h = 0; h < kAhead; ++h) {
                if (w + 16 * h >= listed) break;
                const int i = __builtin_amdgcn_readfirstlane(list[w + 16 * h]);
                row[h] = (int)(group_magic ? div_magic((uint32_t)i, group_magic) : (uint32_t)i);
                id0[h] = (i - row[h] * cut.groups) * kGroup * 64 * E;
                const T* x = logits + (int64_t)(row0 + row[h]) * ld;
                if (id0[h] + kGroup * 64 * E <= n_valid) {
#pragma unroll
                    for (int g = 0; g < kGroup; ++g)
                        v[h][g] = *reinterpret_cast<const typename Vec<T>::type*>(x + id0[h] + (64 * g + lane) * E);
                } else {
#pragma unroll
                    for (int g = 0; g < kGroup; ++g)
#pragma unroll
                        for (int e = 0; e < E; ++e) {
                            const int id = id0[h] + (64 * g + lane) * E + e;
                            v[h][g][e] = id < n_valid ? x[id] : (T)-__builtin_inff();
                        }
                }
            }
#pragma unroll
            for (int h = 0; h < kAhead; ++h) {
                if (w + 16 * h >= listed) break;
                const double add = row_add[row[h]], t = goal - add, u = row_max[row[h]];
                const float least = (float)(t + u - (0x1p-22 * (__builtin_fabs(t) + __builtin_fabs(u)) +
                                                     0x1p-51 * (__builtin_fabs(goal) + __builtin_fabs(add))));
#pragma unroll
                for (int g = 0; g < kGroup; ++g) {
                    float m = (float)v[h][g][0];
#pragma unroll
                    for (int e = 1; e < E; ++e) m = __builtin_fmaxf(m, (float)v[h][g][e]);
                    if (!__any(m >= least)) continue;  // most vectors of a group hold none
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        const float l = (float)v[h][g][e];
                        if (l >= least) f(l, row[h], id0[h] + (64 * g + lane) * E + e);
                    }
                }
            }
        }
    };
    Limit limit{listed < k ? (uint64_t)1 : groups.key, 0xffffffffu};  // fewer groups: all that they hold
    auto collect = [&]() {
        each(limit.key, [&](float l, int b, int id) {
            const uint64_t c = key_of(l, b);
            const uint32_t at = index_of(b, id);
            if (limit.takes(c, at)) {
                const int i = atomicAdd(&n_pool, 1);
                if (i < kPool) {
                    pool_key[i] = c;
                    pool_at[i] = at;
                }
            }
        });
        __syncthreads();
    };
    collect();
    // More than the ranks are for: a limit near the k best of those that the pool holds, and where it does not hold all, another
    // look at the groups. Two such looks suffice but where the pool gets the worst of many first: then the limit comes from
    // counts of all and takes no more than the pool holds, so that the look after it is the last (64 of 16 beams of 50,257 f16, 8
    // prompts, where one beam's groups are fewer than 64: 44.9 us, by counts of all at once 56.2).
    for (int look = 0; n_pool > k + 64; ++look) {
        const int held = n_pool;
        const uint64_t c = tid < held ? pool_key[tid] : 0;
        const uint32_t at = tid < held ? pool_at[tid] : 0;
        if (held <= kPool || look < 2) {
            limit = find_limit(top, k, k + 32, [&](const Limit& l) {
                return wg_sum((int)__builtin_popcountll(__ballot(l.takes(c, at))), red, turn);
            });
        } else {
            limit = find_limit(top, k, kPool, [&](const Limit& l) {
                int n = 0;
                each(l.key, [&](float x, int b, int id) { n += l.takes(key_of(x, b), index_of(b, id)); });
                return wg_sum(wave_sum_i32(n), red, turn);
            });
        }
        __syncthreads();
        if (tid == 0) n_pool = 0;
        __syncthreads();
        if (held > kPool) {
            collect();
        } else {
            if (limit.takes(c, at)) {
                const int i = atomicAdd(&n_pool, 1);
                pool_key[i] = c;
                pool_at[i] = at;
            }
            __syncthreads();
        }
    }
    // 3. their ranks: a wave to a candidate, how many come before it. They are k + 64 at most, five to a lane.
    const int n = __builtin_amdgcn_readfirstlane(n_pool);
    constexpr int kEach = (QH_BEAM_MAX_K + 64) / 64;
    uint64_t held[kEach];
    uint32_t held_at[kEach];
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
        const int i = 64 * j + lane;
        held[j] = i < n ? pool_key[i] : 0;
        held_at[j] = i < n ? pool_at[i] : 0;
    }
    for (int i = wave; i < n; i += 16) {
        const uint64_t c = scalar(pool_key[i]);
        const uint32_t at = (uint32_t)__builtin_amdgcn_readfirstlane((int)pool_at[i]);
        int rank = 0;
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            if (64 * j >= n) break;
            rank += __builtin_popcountll(__ballot(held[j] > c || (held[j] == c && held_at[j] < at)));
        }
        if (lane == 0 && rank < k) {
            parent[(size_t)prompt * k + rank] = row0 + (int)(at / QH_SAMPLE_MAX_VOCAB);
            token[(size_t)prompt * k + rank] = (int)(at % QH_SAMPLE_MAX_VOCAB);
            best[(size_t)prompt * k + rank] = (float)from_ordered_f64(c);
        }
    }
    for (int i = n + tid; i < k; i += kPickThreads) {  // fewer candidates than k
        parent[(size_t)prompt * k + i] = -1;
        token[(size_t)prompt * k + i] = -1;
        best[(size_t)prompt * k + i] = -__builtin_inff();
    }
}

// Exact floor(g / d) by div_magic with this number (0: d is 1), for g * d < 2^32.
uint32_t magic_of(int d) { return d == 1 ? 0u : (uint32_t)((((uint64_t)1 << 32) + (uint32_t)d - 1) / (uint32_t)d); }

template <typename T>
hipError_t beam_select_of(const BeamArgs& a, hipStream_t s) {
    const int rows = a.prompts * a.beams;
    const BeamCut c = beam_cut<T>(rows, a.beams, a.n_valid, a.k);
    double* psum = static_cast<double*>(a.ws);
    float* pmax = reinterpret_cast<float*>(psum + (size_t)rows * c.parts);
    float* gmax = pmax + (size_t)rows * c.parts;
    const T* logits = static_cast<const T*>(a.logits);
    const dim3 grid((unsigned)(rows * c.parts));
    auto go = [&](auto vecs) {
        qh_launch((beam_rows_kernel<T, decltype(vecs)::value>), grid, dim3(256), 0, s, logits, a.ld, a.n_valid, c,
                  magic_of(c.parts), gmax, pmax, psum);
    };
    using std::integral_constant;
    if (c.vecs == 1) go(integral_constant<int, 1>{});
    else if (c.vecs == 2) go(integral_constant<int, 2>{});
    else if (c.vecs == 4) go(integral_constant<int, 4>{});
    else go(integral_constant<int, 8>{});
    if (hipError_t e = hipGetLastError()) return e;
    constexpr int kGroup = 1024 / (64 * kE<T>);
    auto pick = [&](auto keys, auto group) {
        qh_launch((beam_pick_kernel<T, decltype(keys)::value, decltype(group)::value>), dim3((unsigned)a.prompts),
                  dim3(kPickThreads), 0, s, logits, a.ld, a.scores, a.beams, a.n_valid, a.k, c, magic_of(c.groups), gmax, pmax,
                  psum, a.parent, a.token, a.best);
    };
    const int groups = a.beams * c.groups;
    if (c.group == 1 && groups <= kPickThreads) pick(integral_constant<int, 1>{}, integral_constant<int, 1>{});
    else if (c.group == 1) pick(integral_constant<int, 4>{}, integral_constant<int, 1>{});
    else if (c.group != kGroup) pick(integral_constant<int, 32>{}, integral_constant<int, 2 * kGroup>{});
    else if (groups <= kPickThreads) pick(integral_constant<int, 1>{}, integral_constant<int, kGroup>{});
    else if (groups <= 4 * kPickThreads) pick(integral_constant<int, 4>{}, integral_constant<int, kGroup>{});
    else pick(integral_constant<int, 32>{}, integral_constant<int, kGroup>{});
    return hipGetLastError();
}

}  // namespace

// For any k: the cut of few and of many.
size_t beam_workspace_bytes(int dtype, int prompts, int beams, int n_valid) {
    const int rows = prompts * beams;
    size_t bytes = 0;
    for (int k : {1, QH_BEAM_MAX_K}) {
        const BeamCut c = dtype == QH_F32 ? beam_cut<float>(rows, beams, n_valid, k) : beam_cut<_Float16>(rows, beams, n_valid, k);
        const size_t need = (size_t)rows * ((size_t)c.parts * 12 + (size_t)c.groups * 4);
        bytes = need > bytes ? need : bytes;
    }
    return bytes;
}

hipError_t launch_beam_select(const BeamArgs& a, int dtype, hipStream_t s) {
    return dtype == QH_F32 ? beam_select_of<float>(a, s) : beam_select_of<_Float16>(a, s);
}

}  // namespace qh
