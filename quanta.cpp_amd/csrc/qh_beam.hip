// Beam search's selection: of each prompt's beams b and ids v, the k candidates with the largest
//     score_b + logit_bv - log sum_u exp(logit_bu),
// ties to the lower (b, v). Two launches:
//   1. over the whole GPU (beam_rows_kernel): every logit once, for the largest of each group of ids and, wave by wave, the
//      sum of exponentials. Bound by memory: 192 x 151,936 f32.
//   2. a workgroup to a prompt (beam_pick_kernel): the rows' sums, then the k best groups by their largest candidate (a
//      group that is not among them holds none of the k best candidates, for k others have one before its own best), and
//      the k best of what those groups hold.
// Candidates of different rows meet in the order of their scores, so sums, exponentials and scores are 64-bit: rounded to
// f32, scores that are 2^-20 apart would tie. (A 64-bit multiply-add takes no longer than a 32-bit one here.)
#include "qh_device.h"
#include "qh_rows.h"

namespace qh {
namespace {

constexpr int kPickThreads = 1024;
constexpr int kPool = 1024;       // candidates that are ranked
constexpr int kList = 2 * QH_BEAM_MAX_K + 32;  // groups that are read again, at most

template <typename T>
constexpr int kE = 16 / (int)sizeof(T);
template <typename T>
struct Vec {  // at any address of the type's alignment
    typedef T type __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
};

// How the rows are cut: a wave's part of a row is `vecs` vectors of 64 * E ids, a group `group` of them.
struct BeamCut {
    int vecs, group;
    int parts, groups;  // of a row
};

template <typename T>
BeamCut beam_cut(int rows, int beams, int n_valid) {
    const int v = (n_valid + 64 * kE<T> - 1) / (64 * kE<T>);
    BeamCut c{};
    c.group = 1;  // groups of a prompt: 8 keys to a thread of the picking workgroup, or 32 where groups cannot be larger
    while (c.group < 8 && (int64_t)beams * ((v + c.group - 1) / c.group) > 8 * kPickThreads) c.group *= 2;
    c.vecs = 8;  // the loads that a wave has in flight, fewer where there are not waves enough
    while (c.vecs > c.group && (int64_t)rows * ((v + c.vecs - 1) / c.vecs) < 4096) c.vecs /= 2;
    c.parts = (v + c.vecs - 1) / c.vecs;
    c.groups = (v + c.group - 1) / c.group;
    return c;
}

// exp(d) for d <= 0, off by 2^-38 of it at most: d log2(e) = n + f, and a polynomial for 2^f, |f| <= 1/2, that interpolates
// (2^f - 1) / f at the Chebyshev nodes; exp(0) is 1. 0 from -800 down.
__device__ __forceinline__ double exp_below(double d) {
    const double t = __builtin_fmax(d, -800.0) * 0x1.71547652b82fep+0;
    const double n = __builtin_rint(t), f = t - n;
    double p = 0x1.63b2d7971923fp-20;
    p = __builtin_fma(p, f, 0x1.00c0e4e15189cp-16);
    p = __builtin_fma(p, f, 0x1.4308c7183d6a2p-13);
    p = __builtin_fma(p, f, 0x1.5d877598350dep-10);
    p = __builtin_fma(p, f, 0x1.3b2ab70ad2565p-7);
    p = __builtin_fma(p, f, 0x1.c6b08da70cce3p-5);
    p = __builtin_fma(p, f, 0x1.ebfbdff82a734p-3);
    p = __builtin_fma(p, f, 0x1.62e42fef9cc69p-1);
    p = __builtin_fma(p, f, 1.0);
    return __builtin_ldexp(p, (int)n);
}

template <typename T, int kVecs>
__global__ __launch_bounds__(256) void beam_rows_kernel(const T* __restrict__ logits, int64_t ld, int rows, int n_valid,
                                                        BeamCut cut, uint32_t part_magic, float* __restrict__ gmax,
                                                        float* __restrict__ pmax, double* __restrict__ psum) {
    constexpr int E = kE<T>;
    const uint32_t item = blockIdx.x * 4 + (threadIdx.x >> 6);
    const int row = (int)(part_magic ? div_magic(item, part_magic) : item), part = (int)item - row * cut.parts;
    if (row >= rows) return;
    const int lane = (int)threadIdx.x & 63, first = part * kVecs;
    const T* x = logits + (int64_t)row * ld;
    typename Vec<T>::type raw[kVecs];
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
    const double base = (double)__builtin_fmaxf(m, -3.402823466e38f);  // a part without a finite logit sums to 0
    double s = 0.0;
#pragma unroll
    for (int j = 0; j < kVecs; ++j)
#pragma unroll
        for (int e = 0; e < E; ++e) s += exp_below((double)(float)raw[j][e] - base);
    s = wave_reduce32x2(s, [](double a, double b) { return a + b; });
    if (__any(nan) || m == __builtin_inff()) s = __builtin_nan("");
    if (lane == 0) {
        pmax[(size_t)row * cut.parts + part] = m;
        psum[(size_t)row * cut.parts + part] = s;
    }
}

// Monotone map of a finite f64 onto uint64, above 0 (which stands for "no candidate").
__device__ __forceinline__ uint64_t ordered_f64(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    return (u >> 63) ? ~u : (u | ((uint64_t)1 << 63));
}
__device__ __forceinline__ double from_ordered_f64(uint64_t k) {
    return __builtin_bit_cast(double, (k >> 63) ? (k & ~((uint64_t)1 << 63)) : ~k);
}

// A candidate's place in the order: a larger key first, then a lower index. Those up to a limit are taken.
struct Limit {
    uint64_t key;
    uint32_t index;
    __device__ __forceinline__ bool takes(uint64_t k, uint32_t i) const { return k > key || (k == key && i <= index); }
};

// Sum of v over the workgroup, for every thread. `red` holds 16 values for each parity of `turn`, so that a call needs one
// barrier.
__device__ __forceinline__ int wg_sum(int v, int (*red)[16], int& turn) {
    v = wave_sum_i32(v);
    int* r = red[turn & 1];
    ++turn;
    if ((threadIdx.x & 63) == 0) r[threadIdx.x >> 6] = v;
    __syncthreads();
    int all = 0;
#pragma unroll
    for (int w = 0; w < 16; ++w) all += r[w];
    return all;
}

// A limit that takes at least k and at most `most` of the candidates that count(limit) counts (the workgroup's, the same for
// every thread), or all where there are fewer; top: a key that none is above. Steps down from the top, four times as far
// each time, halves the keys between the last two steps, and then, where more than `most` share one key, the indexes.
template <typename Count>
__device__ __forceinline__ Limit find_limit(uint64_t low, uint64_t top, int k, int most, Count&& count) {
    Limit all{low, 0xffffffffu};
    if (count(all) <= most) return all;
    uint64_t lo = low, hi = top + 1;  // at least k at lo and above, fewer than k at hi and above
    for (uint64_t step = (uint64_t)1 << 49; hi - lo > step; step = step < (uint64_t)1 << 60 ? 4 * step : ~(uint64_t)0) {
        const uint64_t at = hi - step;  // 2^49: 2 of a score between 16 and 32
        const int n = count(Limit{at, 0xffffffffu});
        if (n < k) {
            hi = at;
        } else {
            if (n <= most) return Limit{at, 0xffffffffu};
            lo = at;
            break;
        }
    }
    while (hi - lo > 1) {
        const uint64_t mid = lo + (hi - lo) / 2;
        const int n = count(Limit{mid, 0xffffffffu});
        if (n < k) hi = mid;
        else if (n <= most) return Limit{mid, 0xffffffffu};
        else lo = mid;
    }
    uint32_t a = 0, b = 0xffffffffu;  // fewer than k up to index a - 1, at least k up to b
    while (a < b) {
        const uint32_t mid = a + (b - a) / 2;
        const int n = count(Limit{lo, mid});
        if (n < k) a = mid + 1;
        else if (n <= most) return Limit{lo, mid};
        else b = mid;
    }
    return Limit{lo, b};
}

template <typename T, int kKeys>
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
    __shared__ uint64_t ends[2][16];
    __shared__ int n_list, n_pool;
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6, prompt = (int)blockIdx.x, row0 = prompt * beams;
    if (tid == 0) n_list = n_pool = 0;
    for (int b = wave; b < beams; b += 16) {
        const float* pm = pmax + (size_t)(row0 + b) * cut.parts;
        const double* ps = psum + (size_t)(row0 + b) * cut.parts;
        float m = -__builtin_inff();
        for (int i = lane; i < cut.parts; i += 64) m = __builtin_fmaxf(m, pm[i]);
        m = wave_reduce32x2(m, [](float a, float c) { return __builtin_fmaxf(a, c); });
        const double base = (double)__builtin_fmaxf(m, -3.402823466e38f);
        double s = 0.0;
        for (int i = lane; i < cut.parts; i += 64) {
            const double p = ps[i];
            if (p != 0.0) s += p * exp_below((double)pm[i] - base);
        }
        s = wave_reduce32x2(s, [](double a, double c) { return a + c; });
        if (lane == 0) {
            const double score = scores ? (double)scores[row0 + b] : 0.0;
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
    // 1. the groups
    const int n_groups = beams * cut.groups;
    uint64_t key[kKeys];
    uint64_t low = ~(uint64_t)0, top = 0;
#pragma unroll
    for (int j = 0; j < kKeys; ++j) {
        const int i = j * kPickThreads + tid;
        key[j] = 0;
        if (i < n_groups) {
            const int b = (int)(group_magic ? div_magic((uint32_t)i, group_magic) : (uint32_t)i);
            key[j] = key_of(gmax[(size_t)row0 * cut.groups + i], b);
        }
        if (key[j]) {
            low = key[j] < low ? key[j] : low;
            top = key[j] > top ? key[j] : top;
        }
    }
    low = ~wave_max_u64(~low);
    top = wave_max_u64(top);
    if (lane == 0) {
        ends[0][wave] = low;
        ends[1][wave] = top;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 16; ++w) {
        low = ends[0][w] < low ? ends[0][w] : low;
        top = ends[1][w] > top ? ends[1][w] : top;
    }
    if (top == 0) low = 1;  // no candidate at all
    int turn = 0;
    const Limit groups = find_limit(low, top, k, 2 * k + 32, [&](const Limit& l) {
        int n = 0;
#pragma unroll
        for (int j = 0; j < kKeys; ++j) n += l.takes(key[j], (uint32_t)(j * kPickThreads + tid));
        return wg_sum(n, red, turn);
    });
#pragma unroll
    for (int j = 0; j < kKeys; ++j) {
        const int i = j * kPickThreads + tid;
        if (groups.takes(key[j], (uint32_t)i)) list[atomicAdd(&n_list, 1)] = i;
    }
    __syncthreads();
    // 2. their candidates: where k groups are listed, k of their best are at the limit's key or above, so only such ones count
    const int listed = n_list, per = 64 * E;
    auto each = [&](auto&& f) {  // f(key, row * n_valid + id) of every candidate of the listed groups, a wave to a vector of ids
        for (int w = wave; w < listed * cut.group; w += 16) {
            const int i = list[w / cut.group], b = (int)(group_magic ? div_magic((uint32_t)i, group_magic) : (uint32_t)i);
            const int id = ((i - b * cut.groups) * cut.group + w % cut.group) * per + lane * E;
            const T* x = logits + (int64_t)(row0 + b) * ld + id;
            if (id + E <= n_valid) {
                const auto v = *reinterpret_cast<const typename Vec<T>::type*>(x);
#pragma unroll
                for (int e = 0; e < E; ++e) f(key_of((float)v[e], b), (uint32_t)(b * n_valid + id + e));
            } else {
                for (int e = 0; e < E; ++e)
                    if (id + e < n_valid) f(key_of((float)x[e], b), (uint32_t)(b * n_valid + id + e));
            }
        }
    };
    Limit limit{listed < k ? (uint64_t)1 : groups.key, 0xffffffffu};  // fewer groups: all that they hold
    auto collect = [&]() {
        each([&](uint64_t c, uint32_t at) {
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
    if (n_pool > kPool) {  // many of them next to each other, or equal: the limit from counts of them all
        limit = find_limit(limit.key, top, k, kPool, [&](const Limit& l) {
            int n = 0;
            each([&](uint64_t c, uint32_t at) { n += l.takes(c, at); });
            return wg_sum(n, red, turn);
        });
        __syncthreads();
        if (tid == 0) n_pool = 0;
        __syncthreads();
        collect();
    }
    // 3. their ranks, each from a look at all of them
    const int n = n_pool;
    if (tid < n) {
        const uint64_t c = pool_key[tid];
        const uint32_t at = pool_at[tid];
        int rank = 0;
        for (int j = 0; j < n; ++j) rank += pool_key[j] > c || (pool_key[j] == c && pool_at[j] < at);
        if (rank < k) {
            const int b = (int)(at / (uint32_t)n_valid);
            parent[(size_t)prompt * k + rank] = row0 + b;
            token[(size_t)prompt * k + rank] = (int)(at - (uint32_t)b * (uint32_t)n_valid);
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
    const BeamCut c = beam_cut<T>(rows, a.beams, a.n_valid);
    double* psum = static_cast<double*>(a.ws);
    float* pmax = reinterpret_cast<float*>(psum + (size_t)rows * c.parts);
    float* gmax = pmax + (size_t)rows * c.parts;
    const T* logits = static_cast<const T*>(a.logits);
    const dim3 grid((unsigned)(((int64_t)rows * c.parts + 3) / 4));
    auto go = [&](auto vecs) {
        qh_launch((beam_rows_kernel<T, decltype(vecs)::value>), grid, dim3(256), 0, s, logits, a.ld, rows, a.n_valid, c,
                  magic_of(c.parts), gmax, pmax, psum);
    };
    using std::integral_constant;
    if (c.vecs == 1) go(integral_constant<int, 1>{});
    else if (c.vecs == 2) go(integral_constant<int, 2>{});
    else if (c.vecs == 4) go(integral_constant<int, 4>{});
    else go(integral_constant<int, 8>{});
    if (hipError_t e = hipGetLastError()) return e;
    auto pick = [&](auto keys) {
        qh_launch((beam_pick_kernel<T, decltype(keys)::value>), dim3((unsigned)a.prompts), dim3(kPickThreads), 0, s, logits,
                  a.ld, a.scores, a.beams, a.n_valid, a.k, c, magic_of(c.groups), gmax, pmax, psum, a.parent, a.token, a.best);
    };
    if (a.beams * c.groups <= 8 * kPickThreads) pick(integral_constant<int, 8>{});
    else pick(integral_constant<int, 32>{});
    return hipGetLastError();
}

}  // namespace

size_t beam_workspace_bytes(int dtype, int prompts, int beams, int n_valid) {
    const int rows = prompts * beams;
    const BeamCut c = dtype == QH_F32 ? beam_cut<float>(rows, beams, n_valid) : beam_cut<_Float16>(rows, beams, n_valid);
    return (size_t)rows * ((size_t)c.parts * 12 + (size_t)c.groups * 4);
}

hipError_t launch_beam_select(const BeamArgs& a, int dtype, hipStream_t s) {
    return dtype == QH_F32 ? beam_select_of<float>(a, s) : beam_select_of<_Float16>(a, s);
}

}  // namespace qh
