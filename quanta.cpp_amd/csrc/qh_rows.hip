// Rows between the matmuls of a step of many sequences: root-mean-square norm with the residual's addition (into rows or
// into the matmuls' 8-bit blocks), and rotary positions. Both read and write every element once and are bound by memory;
// calls of a few rows by the launch and one round of loads.
#include "qh_device.h"
#include "qh_rows.h"

namespace qh {
namespace {

// E elements at any address of the type's alignment: the hardware takes 16-byte accesses at any of them, so odd widths and
// strides need no second kernel.
template <typename T>
constexpr int kE = 16 / (int)sizeof(T);
template <typename T>
struct Vec {
    typedef T type __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
};

// Elements [0, n) of the E at p into f32 (the others 0), n uniform over most lanes.
template <typename T>
__device__ __forceinline__ void load_e(const T* p, int n, float (&x)[kE<T>]) {
    if (n >= kE<T>) {
        const auto v = *reinterpret_cast<const typename Vec<T>::type*>(p);
#pragma unroll
        for (int i = 0; i < kE<T>; ++i) x[i] = (float)v[i];
    } else {
#pragma unroll
        for (int i = 0; i < kE<T>; ++i) x[i] = i < n ? (float)p[i] : 0.0f;
    }
}
// Stores pass by the caches, whose lines the loads of rows to come take: 16,000 x 4,096 f16 norms with residual 84.0 us replayed
// one after the other, by plain stores 99.3, and 161.9 and 166.2 with an addition that reads both results next; 512 x 4,096 5.4 and
// 6.1, 10.9 and 11.1; 8,000 tokens of 40 heads of 128 f16 turned 26.5 and 28.2. (8-bit codes, a quarter of the bytes, do not: 8,000 x
// 5,120 with their reading back 173, past the caches 200.)
template <typename T>
__device__ __forceinline__ void store_e(T* p, int n, const float (&x)[kE<T>]) {
    if (n >= kE<T>) {
        typename Vec<T>::type v;
#pragma unroll
        for (int i = 0; i < kE<T>; ++i) v[i] = (T)x[i];
        __builtin_nontemporal_store(v, reinterpret_cast<typename Vec<T>::type*>(p));
    } else {
#pragma unroll
        for (int i = 0; i < kE<T>; ++i)
            if (i < n) p[i] = (T)x[i];
    }
}

// ------------------------------------------------------------------------------------------------------- norm

// The 8-bit block of which this lane holds E consecutive values and the 32 / E lanes of its aligned group the others:
// quantize_q8's codes and scale.
__device__ __forceinline__ void quant_lanes(const float (&v)[4], int8_t* q, float* d) {
    quant_block_x8(make_float4(v[0], v[1], v[2], v[3]), q, d);
}
__device__ __forceinline__ void quant_lanes(const float (&v)[8], int8_t* q, float* d) {
    float a = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) a = __builtin_fmaxf(a, __builtin_fabsf(v[i]));
    a = dpp_max<0xB1>(a);
    a = dpp_max<0x4E>(a);
    const float sc = a / 127.0f, inv = sc > 0.0f ? 1.0f / sc : 0.0f;
    uint32_t c[2] = {};
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i >> 2] |= (uint32_t)(uint8_t)(int8_t)(int)round_half_away(v[i] * inv) << (8 * (i & 3));
    const int j = (int)threadIdx.x & 3;
    *reinterpret_cast<uint2*>(q + 8 * j) = make_uint2(c[0], c[1]);
    if (j == 0) *d = sc;
}

// kWaves waves to a row, kVec vectors of E elements to a lane, 4 / kWaves rows to a workgroup of at least 4 waves. The sum
// of squares and the scaled products are 64-bit (as fast as 32-bit ones here, and far from the memory's time): no square
// overflows, the order of the sum does not show, and y is rounded to f32 once (f16 rows from there, so by 2^-11 and 2^-24: a
// single rounding from 64 bits has no instruction). Bound by memory: 4,001 x 5,120 f32 with residual into blocks 49.3 us, 16,000 x
// 4,096 f16 with residual 91.6 among calls into new rows (84 replayed), 5.5 and 5.7 TB/s; 1 x 896 2.4.
template <typename T, int kWaves, int kVec>
__global__ __launch_bounds__(kWaves < 4 ? 256 : 64 * kWaves) void rmsnorm_kernel(NormArgs a) {
    constexpr int E = kE<T>, kRows = kWaves < 4 ? 4 / kWaves : 1, kPass = 64 * kWaves * E;
    const int tid = (int)threadIdx.x % (64 * kWaves);
    const int row = (int)blockIdx.x * kRows + (int)threadIdx.x / (64 * kWaves);
    __shared__ double part[kWaves < 4 ? 4 : kWaves];
    if (kWaves == 1 && row >= a.n_tok) return;
    const bool there = row < a.n_tok;
    float h[kVec][E];
    double ss = 0.0;
    if (there) {
        const T* x = static_cast<const T*>(a.x) + (int64_t)row * a.ldx;
        const T* res = static_cast<const T*>(a.res) + (int64_t)row * a.ldr;
        T* sum = static_cast<T*>(a.sum) + (int64_t)row * a.lds;
        float r[kVec][E];
        // whole passes of the row without a branch of single lanes, which would have every load waited for by itself
        auto load = [&](const T* p, float (&v)[kVec][E]) {
#pragma unroll
            for (int c = 0; c < kVec; ++c) {
                const int i = (c * 64 * kWaves + tid) * E;
                if ((c + 1) * kPass <= a.n) load_e(p + i, E, v[c]);
                else load_e(p + i, a.n - i, v[c]);
            }
        };
        load(x, h);
        if (a.res) load(res, r);
#pragma unroll
        for (int c = 0; c < kVec; ++c) {
            const int i = (c * 64 * kWaves + tid) * E;
            if (a.res) {
#pragma unroll
                for (int e = 0; e < E; ++e) h[c][e] = (float)(T)(h[c][e] + r[c][e]);
            }
            if (a.sum) store_e(sum + i, (c + 1) * kPass <= a.n ? E : a.n - i, h[c]);
#pragma unroll
            for (int e = 0; e < E; ++e) ss = __builtin_fma((double)h[c][e], (double)h[c][e], ss);
        }
    }
    ss = wave_reduce32x2(ss, [](double p, double q) { return p + q; });
    if (kWaves > 1) {
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = ss;
        __syncthreads();
        const int first = (int)threadIdx.x / (64 * kWaves) * kWaves;
        ss = 0.0;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) ss += part[first + w];
    }
    if (!there) return;
    const double scale = 1.0 / __builtin_sqrt(ss / (double)a.n + a.eps);
#pragma unroll
    for (int c = 0; c < kVec; ++c) {
        const int i = (c * 64 * kWaves + tid) * E;
        if (i >= a.n) break;
        float w[kE<T>];
#pragma unroll
        for (int v = 0; v < E / 4; ++v) {
            float w4[4];
            load_e(a.w + i + 4 * v, a.n - i - 4 * v, w4);
#pragma unroll
            for (int e = 0; e < 4; ++e) w[4 * v + e] = w4[e];
        }
        float y[E];
#pragma unroll
        for (int e = 0; e < E; ++e) y[e] = (float)((double)h[c][e] * scale * (double)w[e]);
        if (a.y) store_e(static_cast<T*>(a.y) + (int64_t)row * a.ldy + i, a.n - i, y);
        if (a.q) quant_lanes(y, a.q + (int64_t)row * a.n + i / 32 * 32, a.d + (int64_t)row * (a.n / 32) + i / 32);
    }
}

template <typename T>
hipError_t rmsnorm_of(const NormArgs& a, hipStream_t s) {
    const int vecs = (a.n + kE<T> - 1) / kE<T>;
    auto run = [&](auto waves, auto vec) {
        constexpr int kWaves = decltype(waves)::value, kRows = kWaves < 4 ? 4 / kWaves : 1;
        qh_launch((rmsnorm_kernel<T, kWaves, decltype(vec)::value>), dim3((unsigned)((a.n_tok + kRows - 1) / kRows)),
                  dim3(kWaves < 4 ? 256 : 64 * kWaves), 0, s, a);
    };
    using std::integral_constant;
    // Loads in flight for waves enough, and one row's lanes not far apart (all by plain stores: 16,000 x 4,096 f16 98.5 us, a wave to a
    // row with 8 vectors 162, eight with one 104; 16,000 x 256 f32 with a wave 27.9, with four 33.5; 16,000 x 8,192 f16 197.7, four
    // waves with four vectors 201.5; 64 x 8,192 f32 5.7 with eight waves, four 6.7; 2,000 x 16,384 f32 176, four waves with 16 vectors
    // 183)
    if (vecs <= 64) run(integral_constant<int, 1>{}, integral_constant<int, 1>{});
    else if (vecs <= 256) run(integral_constant<int, 4>{}, integral_constant<int, 1>{});
    else if (vecs <= 512) run(integral_constant<int, 4>{}, integral_constant<int, 2>{});
    else if (vecs <= 1024) run(integral_constant<int, 8>{}, integral_constant<int, 2>{});
    else if (vecs <= 2048) run(integral_constant<int, 8>{}, integral_constant<int, 4>{});
    else if (vecs <= 4096) run(integral_constant<int, 16>{}, integral_constant<int, 4>{});  // f16: kMaxNorm elements
    else if constexpr (kE<T> == 4) run(integral_constant<int, 16>{}, integral_constant<int, 8>{});
    return hipGetLastError();
}

// ------------------------------------------------------------------------------------------------------- rope

// cos and sin of 2 pi t, |t| <= 1/2. t is brought within an eighth of a turn of a multiple of a quarter, exactly; there the
// power series to x^9 and x^10 end less than 2^-29 short.
__device__ __forceinline__ float2 turn(double t) {
    const double k = __builtin_rint(4.0 * t);
    const float x = (float)((4.0 * t - k) * 1.5707963267948966), z = x * x;
    float s = __builtin_fmaf(z, 1.0f / 362880, -1.0f / 5040);
    s = __builtin_fmaf(z, s, 1.0f / 120);
    s = __builtin_fmaf(z, s, -1.0f / 6);
    s = __builtin_fmaf(z * x, s, x);
    float c = __builtin_fmaf(z, -1.0f / 3628800, 1.0f / 40320);
    c = __builtin_fmaf(z, c, -1.0f / 720);
    c = __builtin_fmaf(z, c, 1.0f / 24);
    c = __builtin_fmaf(z, c, -0.5f);
    c = __builtin_fmaf(z, c, 1.0f);
    const int quarter = (int)k & 3;
    const float co = (quarter & 1) ? s : c, si = (quarter & 1) ? c : s;
    return make_float2(quarter == 1 || quarter == 2 ? -co : co, quarter >= 2 ? -si : si);
}

// floor(g / d) with d's number from magic_of.
__device__ __forceinline__ uint32_t div_below(uint32_t g, uint32_t magic) { return magic ? div_magic(g, magic) : g; }

constexpr int kRopeThreads = 256;
constexpr int kRopePairs = 512;  // cosines and sines that a workgroup keeps

// A workgroup takes `per` tokens: their cosines and sines once into LDS (angles in 64 bits: position times turns per
// position, less its whole turns), then every head's pairs, E of them to an item, and after them the dims past rot, E to an
// item, where the result is not written in place. Consecutive lanes take consecutive items of a head, so rows move in one
// piece. Bound by memory: 8,000 tokens of 40 heads of 128 f16 25.9 us, 6.3 TB/s; 48 of 16 heads of 64 f32 2.8.
// kWhole: no item is cut off by the end of the pairs or of the head.
template <typename T, bool kInterleaved, bool kWhole>
__global__ __launch_bounds__(kRopeThreads) void rope_kernel(RopeArgs a, int per, int units, int rest, uint32_t unit_magic,
                                                            uint32_t head_magic) {
    constexpr int E = kE<T>;
    __shared__ float2 cs[kRopePairs];
    const int half = a.rot >> 1, t0 = (int)blockIdx.x * per, n = min(per, a.n_tok - t0), tid = (int)threadIdx.x;
    for (int i = tid; i < n * half; i += kRopeThreads) {
        const int t = i / half;
        const double turns = (double)a.pos[t0 + t] * a.turns[i - t * half];
        const float2 v = turn(turns - __builtin_rint(turns));
        cs[i] = make_float2(v.x * a.magnitude, v.y * a.magnitude);
    }
    __syncthreads();
    const int each = units + rest, heads = a.q.heads + a.k.heads;
    for (int item = tid; item < n * heads * each; item += kRopeThreads) {
        const int th = (int)div_below((uint32_t)item, unit_magic), u = item - th * each;
        const int t = (int)div_below((uint32_t)th, head_magic), h = th - t * heads;
        const bool of_q = h < a.q.heads;
        const int at = (of_q ? h : h - a.q.heads) * a.hd;
        const T* x = static_cast<const T*>(of_q ? a.q.x : a.k.x) + (int64_t)(t0 + t) * (of_q ? a.q.ld : a.k.ld) + at;
        T* out = static_cast<T*>(of_q ? a.q.out : a.k.out) + (int64_t)(t0 + t) * (of_q ? a.q.ldo : a.k.ldo) + at;
        if (u >= units) {
            const int i = a.rot + (u - units) * E;
            float v[E];
            const int m = kWhole ? E : a.hd - i;
            load_e(x + i, m, v);
            store_e(out + i, m, v);
            continue;
        }
        const int p = u * E, m = kWhole ? E : half - p;
        const float2* c = cs + t * half + p;
        float f[E], g[E];  // firsts and seconds of the pairs (half), or the pairs in order (interleaved)
        if (kInterleaved) {
            load_e(x + 2 * p, 2 * m, f);
            load_e(x + 2 * p + E, 2 * m - E, g);
            float o[2][E];
#pragma unroll
            for (int i = 0; i < E; ++i) {
                const float2 w = c[i < m ? i : 0];
                const float lo = 2 * i < E ? f[2 * i % E] : g[2 * i % E], hi = 2 * i < E ? f[2 * i % E + 1] : g[2 * i % E + 1];
                o[2 * i / E][2 * i % E] = __builtin_fmaf(lo, w.x, -(hi * w.y));
                o[2 * i / E][2 * i % E + 1] = __builtin_fmaf(hi, w.x, lo * w.y);
            }
            store_e(out + 2 * p, 2 * m, o[0]);
            store_e(out + 2 * p + E, 2 * m - E, o[1]);
        } else {
            load_e(x + p, m, f);
            load_e(x + half + p, m, g);
#pragma unroll
            for (int i = 0; i < E; ++i) {
                const float2 w = c[i < m ? i : 0];
                const float lo = f[i], hi = g[i];
                f[i] = __builtin_fmaf(lo, w.x, -(hi * w.y));
                g[i] = __builtin_fmaf(hi, w.x, lo * w.y);
            }
            store_e(out + p, m, f);
            store_e(out + half + p, m, g);
        }
    }
}

// Exact floor(g / d) by div_below with this number, for g * d < 2^32.
uint32_t magic_of(int d) { return d == 1 ? 0u : (uint32_t)((((uint64_t)1 << 32) + (uint32_t)d - 1) / (uint32_t)d); }

template <typename T>
hipError_t rope_of(const RopeArgs& a, bool interleaved, hipStream_t s) {
    constexpr int E = kE<T>;
    const int half = a.rot / 2, units = (half + E - 1) / E, heads = a.q.heads + a.k.heads;
    const bool copies = a.q.x != a.q.out || (a.k.heads > 0 && a.k.x != a.k.out);
    const int rest = copies ? (a.hd - a.rot + E - 1) / E : 0;
    // 8,192 workgroups, fewer where a token would leave threads of one without an item and 2,048 are left (8,000 tokens of 40
    // heads of 128 f16: 28.3 us, by 2,048 workgroups 29.4; 4,096 of 16 heads of 64 f32: 6.8, a token to a workgroup 7.5)
    const int64_t items = (int64_t)heads * (units + rest), fill = kRopeThreads / items, few = a.n_tok / 2048;
    int64_t per = a.n_tok / 8192;
    per = per > (fill < few ? fill : few) ? per : (fill < few ? fill : few);
    per = per < kRopePairs / half ? per : kRopePairs / half;
    // items of a workgroup times what they are divided by stay in 32 bits (at one token: 4,096 heads in all of 65 items)
    const int64_t most = ((int64_t)1 << 31) / (items * (heads > units + rest ? heads : units + rest));
    per = per < most ? per : most;
    per = per < 1 ? 1 : per;
    const dim3 grid((unsigned)((a.n_tok + per - 1) / per));
    const uint32_t um = magic_of(units + rest), hm = magic_of(heads);
    const bool whole = half % E == 0 && (rest == 0 || (a.hd - a.rot) % E == 0);
    auto go = [&](auto inter, auto all) {
        qh_launch((rope_kernel<T, decltype(inter)::value, decltype(all)::value>), grid, dim3(kRopeThreads), 0, s, a, (int)per, units,
                  rest, um, hm);
    };
    if (interleaved && whole) go(std::true_type{}, std::true_type{});
    else if (interleaved) go(std::true_type{}, std::false_type{});
    else if (whole) go(std::false_type{}, std::true_type{});
    else go(std::false_type{}, std::false_type{});
    return hipGetLastError();
}

}  // namespace

hipError_t launch_rmsnorm(const NormArgs& a, int dtype, hipStream_t s) {
    return dtype == QH_F32 ? rmsnorm_of<float>(a, s) : rmsnorm_of<_Float16>(a, s);
}

hipError_t launch_rope(const RopeArgs& a, int dtype, bool interleaved, hipStream_t s) {
    return dtype == QH_F32 ? rope_of<float>(a, interleaved, s) : rope_of<_Float16>(a, interleaved, s);
}

}  // namespace qh
