// gdn_logits.hip -- from a batch of logits to tokens on the caller's device
// buffers: gdn_logits_process (penalties, biases, masks) and
// gdn_sample_tokens (the draw).
#include <hip/hip_runtime.h>

#include <cstdio>
#include <type_traits>

#include "gdn_amd.h"
#include "gdn_device.h"
#include "gdn_internal.h"

namespace gdn {
namespace lg {

constexpr float kInf = __builtin_inff();

// Sixteen bytes of logits of a type, at any element's address.
struct Bf16 {
    static constexpr int kVec = 8;
    typedef uint16_t E;
    __device__ static float get(E e) { return u2f((uint32_t)e << 16); }
    __device__ static E put(float x) { return (E)cvt_pk(x, 0.0f); }
};
struct Fp16 {
    static constexpr int kVec = 8;
    typedef _Float16 E;
    __device__ static float get(E e) { return (float)e; }
    __device__ static E put(float x) { return (E)x; }
};
struct Fp32 {
    static constexpr int kVec = 4;
    typedef float E;
    __device__ static float get(E e) { return e; }
    __device__ static E put(float x) { return x; }
};
template <class T>
struct Vec {
    typename T::E e[T::kVec];
};

// Elements at .. at + kVec - 1 of a row of n; `rest` past its end.
template <class T>
__device__ __forceinline__ void load_vec(const typename T::E *row, int at, int n, float rest, float (&x)[T::kVec]) {
    if (at + T::kVec <= n) {
        Vec<T> v;
        __builtin_memcpy(&v, row + at, sizeof(v));
#pragma unroll
        for (int i = 0; i < T::kVec; ++i) x[i] = T::get(v.e[i]);
    } else {
#pragma unroll
        for (int i = 0; i < T::kVec; ++i) x[i] = at + i < n ? T::get(row[at + i]) : rest;
    }
}
template <class T>
__device__ __forceinline__ void store_vec(typename T::E *row, int at, int n, const float (&x)[T::kVec]) {
    if (at + T::kVec <= n) {
        Vec<T> v;
#pragma unroll
        for (int i = 0; i < T::kVec; ++i) v.e[i] = T::put(x[i]);
        __builtin_memcpy(row + at, &v, sizeof(v));
    } else {
#pragma unroll
        for (int i = 0; i < T::kVec; ++i)
            if (at + i < n) row[at + i] = T::put(x[i]);
    }
}

// ------------------------------------------------------------ processing

// kTile tokens of a row: grid (tiles, rows).  The tile's share of the row's
// history is counted in LDS (whole-number atomics, so no order shows): the
// output's occurrences, and a bit for any occurrence.  A bias' entry number
// goes in by maximum, so the last of equal ids holds.
constexpr int kTile = 8192, kPT = 512;
constexpr uint32_t kSeen = 0x80000000u;

template <class T>
__global__ __launch_bounds__(kPT) void k_process(GDNLogits p) {
    extern __shared__ __attribute__((aligned(16))) uint32_t mem[];
    uint32_t *count = mem, *entry = mem + (p.history ? kTile : 0);
    const int r = blockIdx.y, t0 = blockIdx.x * kTile, t = threadIdx.x;
    const int n = min((int)p.vocab - t0, kTile);
    int len = 0, prompt = 0, b0 = 0, b1 = 0;
    if (p.history) {
        len = min(max(p.history_len[r], 0), (int)p.history_width);
        prompt = p.prompt_len ? p.prompt_len[r] : 0;
        for (int i = t; i < kTile / 4; i += kPT) reinterpret_cast<u32x4 *>(count)[i] = (u32x4){0u, 0u, 0u, 0u};
    }
    if (p.bias_offsets) {
        b0 = min(max(p.bias_offsets[r], 0), (int)p.n_bias);
        b1 = min(max(p.bias_offsets[r + 1], b0), (int)p.n_bias);
        for (int i = t; i < kTile / 4; i += kPT) reinterpret_cast<u32x4 *>(entry)[i] = (u32x4){0u, 0u, 0u, 0u};
    }
    __syncthreads();
    const int32_t *hist = p.history + (size_t)r * p.history_stride;
    for (int i = t; i < len; i += kPT) {
        const uint32_t id = (uint32_t)hist[i] - (uint32_t)t0;
        if (id < (uint32_t)n) {
            if (i >= prompt) atomicAdd(&count[id], 1u);
            atomicOr(&count[id], kSeen);
        }
    }
    for (int i = b0 + t; i < b1; i += kPT) {
        const uint32_t id = (uint32_t)p.bias_ids[i] - (uint32_t)t0;
        if (id < (uint32_t)n) atomicMax(&entry[id], (uint32_t)(i - b0) + 1u);
    }
    __syncthreads();
    const float rep = p.repetition ? p.repetition[r] : 1.0f, pres = p.presence ? p.presence[r] : 0.0f,
                freq = p.frequency ? p.frequency[r] : 0.0f;
    const int mi = p.mask ? (p.mask_index ? p.mask_index[r] : r) : -1;
    const uint32_t *mask = mi >= 0 && mi < (int)p.n_masks ? p.mask + (size_t)mi * p.mask_stride + t0 / 32 : nullptr;
    const typename T::E *in = static_cast<const typename T::E *>(p.logits) + (size_t)r * p.logits_stride + t0;
    typename T::E *out = static_cast<typename T::E *>(p.out) + (size_t)r * p.out_stride + t0;
    constexpr int V = T::kVec;
    for (int at = t * V; at < n; at += kPT * V) {
        float x[V];
        load_vec<T>(in, at, n, 0.0f, x);
        const uint32_t allowed = mask ? mask[at / 32] >> (at & 31) : ~0u;
        uint32_t c[V] = {}, b[V] = {};
        if (p.history) {
#pragma unroll
            for (int i = 0; i < V; ++i) c[i] = count[at + i];
        }
        if (p.bias_offsets) {
#pragma unroll
            for (int i = 0; i < V; ++i) b[i] = entry[at + i];
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
            if (c[i]) {
                x[i] = x[i] > 0.0f ? x[i] / rep : x[i] * rep;
                const uint32_t said = c[i] & ~kSeen;
                if (said) x[i] = (x[i] - freq * (float)said) - pres;
            }
            if (b[i]) x[i] = x[i] + p.bias_values[b0 + (int)b[i] - 1];
            if (!((allowed >> i) & 1u)) x[i] = -kInf;
        }
        store_vec<T>(out, at, n, x);
    }
}

// ------------------------------------------------------------ the draw

// A workgroup a row.  Weights are whole numbers of 2^-shift, so counts and
// sums over the row are the same in any order.  The kept tokens are the first
// ones of the ranking up to a border (key, index): one histogram over kBins
// steps of 1 / 32 in (max - x) / temperature -- what lies past them has no
// weight -- gives the step the border is in, and the step's tokens, usually
// some tens, are ranked against each other in LDS.  More than fit there go
// through histograms of 11, 11 and 10 bits of their keys.
constexpr int kST = 1024, kBins = kST, kWaves = kST / 64;
constexpr int kList = 1024;           // tokens of a step that are ranked directly
constexpr int kRadix = 2048;          // bins of a key histogram
constexpr int kCells = (1 << 20) / 256;  // pieces of the longest row

// The 32-bit key of x that grows as x falls (x not NaN; the zeros are equal).
__device__ __forceinline__ uint32_t fall_key(float x) {
    const uint32_t u = f2u(x + 0.0f);
    return u & 0x80000000u ? u : ~u & 0x7fffffffu;
}

// exp(-x), x >= 0, to 2 units of 2^-24 (0 for infinity and NaN): the base-2
// exponential with the rounding error of its argument made good.
__device__ __forceinline__ float exp_neg(float x) {
    constexpr float kL = 1.44269502f, kLo = 1.92596299e-8f;  // log2(e)
    const float y = x * kL, e = __builtin_fmaf(x, kLo, __builtin_fmaf(x, kL, -y));
    const float p = __builtin_amdgcn_exp2f(-y);
    return y < 126.0f ? __builtin_fmaf(p, -0.693147181f * e, p) : 0.0f;
}

__device__ __forceinline__ uint64_t shfl_up64(uint64_t v, int d) {
    return ((uint64_t)(uint32_t)__shfl_up((int)(v >> 32), d) << 32) | (uint32_t)__shfl_up((int)v, d);
}
__device__ __forceinline__ uint64_t wave_scan(uint64_t v, int lane) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint64_t o = shfl_up64(v, d);
        if (lane >= d) v += o;
    }
    return v;
}

struct Ranked {
    uint32_t key;
    int at;
    uint64_t w;
};
struct SampleLds {
    double power[kBins];  // exp(-b / 32) 2^shift
    union {
        struct {
            unsigned long long mass[kRadix];
            uint32_t count[kRadix];
        };
        Ranked list[kList];
        uint64_t cell[kCells];
    };
    uint64_t wsum[kWaves];
    float wmax[kWaves];
    int warg[kWaves];
    double wexp[kWaves];
    uint64_t base;    // weight ranked before a bin found
    double left;      // of the goal, in it
    uint32_t key;     // a border
    int at;
    uint32_t bin, n;
};

// The sum over the workgroup before each thread, and the whole sum.
__device__ __forceinline__ uint64_t block_scan(uint64_t v, uint64_t *wsum, uint64_t &total) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const uint64_t s = wave_scan(v, lane);
    __syncthreads();
    if (lane == 63) wsum[w] = s;
    __syncthreads();
    uint64_t at = 0, all = 0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
        at += i < w ? wsum[i] : 0;
        all += wsum[i];
    }
    total = all;
    return at + s - v;
}

// A row and how its tokens fall and weigh.
template <class T>
struct Row {
    static constexpr int V = T::kVec;
    const typename T::E *row;
    const double *power;
    int n;
    float top;
    double top_d, inv_temp, step;  // step: 32 / temperature

    // f(value, index), a wave's 64 V tokens consecutive
    template <class F>
    __device__ __forceinline__ void each(F &&f) const {
#pragma unroll 2
        for (int at = (int)threadIdx.x * V; at < n; at += kST * V) {
            float x[V];
            load_vec<T>(row, at, n, __builtin_nanf(""), x);
#pragma unroll
            for (int j = 0; j < V; ++j) f(x[j], at + j);
        }
    }
    // how far below the highest; NaN for NaN, whose bin and exponential are
    // those of infinity
    __device__ __forceinline__ double fall(float v) const { return v == top ? 0.0 : top_d - (double)v; }
    // kBins where the weight is 0: exp(-32) is half a unit of 2^-45
    __device__ __forceinline__ int bin(double d) const { return (int)__builtin_fmin(d * step, (double)kBins); }
    // exp(-d / temperature) 2^shift, rounded to a whole number: from the
    // step's power and the Taylor series of what is left (1 / 32 at most: the
    // first term left out is 6e-15)
    __device__ __forceinline__ uint64_t weight(double d, int b) const {
        if (b >= kBins) return 0;
        const double t = __builtin_fma(-d, inv_temp, (double)b * (1.0 / 32.0));
        double y = 1.0 / 720.0;
        y = __builtin_fma(y, t, 1.0 / 120.0);
        y = __builtin_fma(y, t, 1.0 / 24.0);
        y = __builtin_fma(y, t, 1.0 / 6.0);
        y = __builtin_fma(y, t, 0.5);
        y = __builtin_fma(y, t, 1.0);
        y = __builtin_fma(y, t, 1.0);
        // the sum's low bits are the rounded number
        return __builtin_bit_cast(uint64_t, __builtin_fma(power[b], y, 0x1p52)) & 0xfffffffffffffull;
    }
    __device__ __forceinline__ uint64_t weight(double d) const { return weight(d, bin(d)); }
};

// The border of the tokens of step `b` whose ranked counts (by_mass: weights)
// first reach `left`, into lds.key and lds.at; their weight is the result.
template <class T>
__device__ uint64_t border_in(const Row<T> &r, SampleLds &lds, int b, bool by_mass, double left) {
    const int t = threadIdx.x;
    __syncthreads();
    if (t == 0) lds.n = 0;
    __syncthreads();
    r.each([&](float v, int at) __attribute__((always_inline)) {
        const double d = r.fall(v);
        if (r.bin(d) == b) {
            const uint32_t i = atomicAdd(&lds.n, 1u);
            if (i < (uint32_t)kList) lds.list[i] = Ranked{fall_key(v), at, r.weight(d, b)};
        }
    });
    __syncthreads();
    const int n = (int)lds.n;
    if (n <= kList) {
        // the tokens' own ranks
        if (t < n) {
            const Ranked me = lds.list[t];
            int rank = 0;
            uint64_t before = 0;
            for (int i = 0; i < n; ++i) {
                const Ranked o = lds.list[i];
                if (o.key < me.key || (o.key == me.key && o.at < me.at)) {
                    ++rank;
                    before += o.w;
                }
            }
            const double from = by_mass ? (double)before : (double)rank,
                         to = by_mass ? (double)(before + me.w) : (double)(rank + 1);
            // rounding in `left` past the step's end: its last token
            if ((from < left && to >= left) || (rank == n - 1 && to < left)) {
                lds.key = me.key;
                lds.at = me.at;
                lds.base = before + me.w;
            }
        }
        __syncthreads();
        return lds.base;
    }
    uint64_t base = 0;
    uint32_t prefix = 0, have = 0;
    uint64_t each_w = 0;
    for (int level = 0; level < 3; ++level) {
        const int sh = level == 0 ? 21 : level == 1 ? 10 : 0;
        const uint32_t bits = level == 2 ? 0x3ffu : 0x7ffu;
        const uint32_t above = level == 0 ? 0u : ~0u << (level == 1 ? 21 : 10);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kRadix / kST; ++i) {
            lds.count[t + i * kST] = 0;
            lds.mass[t + i * kST] = 0;
        }
        __syncthreads();
        r.each([&](float v, int) __attribute__((always_inline)) {
            const double d = r.fall(v);
            const uint32_t key = fall_key(v);
            if (r.bin(d) == b && (key & above) == prefix) {
                atomicAdd(&lds.count[(key >> sh) & bits], 1u);
                atomicAdd(&lds.mass[(key >> sh) & bits], (unsigned long long)r.weight(d, b));
            }
        });
        __syncthreads();
        const int at = 2 * t;
        const uint64_t m0 = lds.mass[at], m1 = lds.mass[at + 1], c0 = lds.count[at], c1 = lds.count[at + 1];
        uint64_t all_m, all_c;
        const uint64_t mb = block_scan(m0 + m1, lds.wsum, all_m), cb = block_scan(c0 + c1, lds.wsum, all_c);
        const uint64_t v0 = by_mass ? m0 : c0, v1 = by_mass ? m1 : c1, vb = by_mass ? mb : cb;
        // what the bin above holds is all here: rounding past it ends there
        const double goal = __builtin_fmin(left, (double)(by_mass ? all_m : all_c));
        if (v0 + v1 != 0 && (double)vb < goal && (double)(vb + v0 + v1) >= goal) {
            const bool second = !((double)(vb + v0) >= goal);
            lds.bin = at + second;
            lds.left = goal - (double)(vb + (second ? v0 : 0));
            lds.base = mb + (second ? m0 : 0);
        }
        __syncthreads();
        prefix |= lds.bin << sh;
        left = lds.left;
        base += lds.base;
        have = lds.count[lds.bin];
        each_w = lds.mass[lds.bin] / have;
    }
    // of the border key's tokens (one weight all), the first `need` are kept
    uint64_t need = by_mass ? (uint64_t)__builtin_ceil(left / (double)each_w) : (uint64_t)left;
    need = need < 1 ? 1 : (need < have ? need : have);
    // the place of the last of these: the pieces' counts, then the piece's own
    constexpr int V = T::kVec;
    const int n_cells = (r.n + 64 * V - 1) / (64 * V), lane = t & 63, w = t >> 6;
    __syncthreads();
    for (int c = w; c < n_cells; c += kWaves) {
        float x[V];
        load_vec<T>(r.row, (c * 64 + lane) * V, r.n, __builtin_nanf(""), x);
        uint64_t k = 0;
#pragma unroll
        for (int j = 0; j < V; ++j) k += x[j] == x[j] && fall_key(x[j]) == prefix;
        k = wave_scan(k, lane);
        if (lane == 63) lds.cell[c] = k;
    }
    __syncthreads();
    const int per = (n_cells + kST - 1) / kST;
    uint64_t mine = 0, all;
    for (int i = 0; i < per; ++i) mine += t * per + i < n_cells ? lds.cell[t * per + i] : 0;
    uint64_t at = block_scan(mine, lds.wsum, all);
    if (at < need && at + mine >= need) {
        int c = t * per;
        while (at + lds.cell[c] < need) at += lds.cell[c++];
        for (int i = c * 64 * V; i < r.n; ++i) {
            const float v = T::get(r.row[i]);
            if (v == v && fall_key(v) == prefix && ++at == need) {
                lds.key = prefix;
                lds.at = i;
                break;
            }
        }
    }
    __syncthreads();
    return base + need * each_w;
}

template <class T>
__global__ __launch_bounds__(kST) void k_sample(GDNSample p, int shift) {
    constexpr int V = T::kVec;
    __shared__ SampleLds lds;
    const int ri = blockIdx.x, t = threadIdx.x, lane = t & 63, w = t >> 6;
    Row<T> r;
    r.row = static_cast<const typename T::E *>(p.logits) + (size_t)ri * p.logits_stride;
    r.n = (int)p.vocab;
    r.power = lds.power;

    // the highest logit, and its first place
    float top = -kInf;
    int arg = 0x7fffffff;
    r.each([&](float v, int at) __attribute__((always_inline)) {
        if (v > top) {
            top = v;
            arg = at;
        }
    });
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
        const float ov = __shfl_xor(top, s);
        const int oi = __shfl_xor(arg, s);
        if (ov > top || (ov == top && oi < arg)) {
            top = ov;
            arg = oi;
        }
    }
    if (lane == 0) {
        lds.wmax[w] = top;
        lds.warg[w] = arg;
    }
    const float temp = p.temperature ? p.temperature[ri] : 0.0f;
    const bool greedy = !(temp > 0.0f);
    const int k = p.top_k ? p.top_k[ri] : 0;
    const float tp = p.top_p ? p.top_p[ri] : 1.0f;
    const bool first_only = tp <= 0.0f;
    const bool by_k = !greedy && !first_only && k > 0 && k < r.n, by_p = !greedy && !first_only && tp < 1.0f;
    lds.power[t] = __builtin_ldexp(exp(-(double)t / 32.0), shift);
    lds.count[t] = 0;
    lds.mass[t] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kWaves; ++i)
        if (lds.wmax[i] > top || (lds.wmax[i] == top && lds.warg[i] < arg)) {
            top = lds.wmax[i];
            arg = lds.warg[i];
        }
    if (arg == 0x7fffffff) {  // nothing above -infinity
        if (t == 0) {
            p.tokens[ri] = -1;
            if (p.logprobs) p.logprobs[ri] = -kInf;
        }
        return;
    }
    r.top = top;
    r.top_d = (double)top;
    r.inv_temp = 1.0 / (double)temp;
    r.step = 32.0 * r.inv_temp;

    // the sum of exponentials, and the steps' counts and weights
    double sum = 0.0;
    auto pass = [&](auto sum_on, auto count_on, auto mass_on) __attribute__((always_inline)) {
        r.each([&](float v, int) __attribute__((always_inline)) {
            const double d = r.fall(v);
            if (sum_on) sum += (double)exp_neg((float)d);
            if (count_on || mass_on) {
                const int b = r.bin(d);
                if (b < kBins) {
                    if (count_on) atomicAdd(&lds.count[b], 1u);
                    if (mass_on) atomicAdd(&lds.mass[b], (unsigned long long)r.weight(d, b));
                }
            }
        });
    };
    constexpr std::true_type on;
    constexpr std::false_type off;
    if (by_k && by_p) pass(on, on, on);
    else if (by_k) pass(on, on, off);
    else if (by_p) pass(on, off, on);
    else if (p.logprobs) pass(on, off, off);
    double log_sum = 0.0;
    if (p.logprobs) {
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d);
        if (lane == 0) lds.wexp[w] = sum;
        __syncthreads();
        sum = 0.0;
#pragma unroll
        for (int i = 0; i < kWaves; ++i) sum += lds.wexp[i];
        log_sum = log(sum);
    }
    if (greedy) {
        if (t == 0) {
            p.tokens[ri] = arg;
            if (p.logprobs) p.logprobs[ri] = (float)-log_sum;
        }
        return;
    }

    // the border: tokens of a key below it are kept, of its key those up to
    // place edge_at
    uint32_t edge = 0xffffffffu;
    int edge_at = 0x7fffffff;
    if (by_k || by_p) {
        __syncthreads();
        const uint64_t count = lds.count[t], mass = lds.mass[t];
        uint64_t n_all = 0, kept = 0, n_before = 0, m_before = 0;
        if (by_k) n_before = block_scan(count, lds.wsum, n_all);
        if (by_p) m_before = block_scan(mass, lds.wsum, kept);
        if (by_k && (uint64_t)k <= n_all) {
            if (n_before < (uint64_t)k && n_before + count >= (uint64_t)k) {
                lds.bin = t;
                lds.left = (double)((uint64_t)k - n_before);
                lds.base = m_before;
            }
            __syncthreads();
            const uint64_t base = lds.base;
            kept = base + border_in(r, lds, (int)lds.bin, false, lds.left);
            edge = lds.key;
            edge_at = lds.at;
        }
        if (by_p) {
            const double goal = (double)tp * (double)kept;
            __syncthreads();
            // a goal that rounds past the last step's end ends there
            if (mass != 0 && (double)m_before < goal && (double)(m_before + mass) >= goal) {
                lds.bin = t;
                lds.left = goal - (double)m_before;
            }
            __syncthreads();
            // tokens past the first border rank behind all that reach the goal
            border_in(r, lds, (int)lds.bin, true, lds.left);
            if (lds.key < edge || (lds.key == edge && lds.at < edge_at)) {
                edge = lds.key;
                edge_at = lds.at;
            }
        }
    } else if (first_only) {
        edge = fall_key(top);
        edge_at = arg;
    }
    const float mp = p.min_p ? p.min_p[ri] : 0.0f;
    const double least = mp > 0.0f ? __builtin_ldexp((double)__builtin_fminf(mp, 1.0f), shift) : 0.0;
    auto weight = [&](float v, int at) __attribute__((always_inline)) -> uint64_t {
        const uint32_t key = fall_key(v);
        if (!(key < edge || (key == edge && at <= edge_at))) return 0;
        const uint64_t s = r.weight(r.fall(v));
        return (double)s >= least ? s : 0;
    };

    // the kept weights by pieces of 64 V tokens, the piece the draw falls in,
    // the token in it
    const int cells = (r.n + 64 * V - 1) / (64 * V);
    __syncthreads();
    for (int c = w; c < cells; c += kWaves) {
        const int at = (c * 64 + lane) * V;
        float x[V];
        load_vec<T>(r.row, at, r.n, __builtin_nanf(""), x);
        uint64_t s = 0;
#pragma unroll
        for (int j = 0; j < V; ++j) s += weight(x[j], at + j);
        if (__ballot(s != 0) != 0) s = wave_scan(s, lane);
        if (lane == 63) lds.cell[c] = s;
    }
    __syncthreads();
    uint64_t mine = 0, all;
    const int per = (cells + kST - 1) / kST;
    for (int i = 0; i < per; ++i) mine += t * per + i < cells ? lds.cell[t * per + i] : 0;
    uint64_t at = block_scan(mine, lds.wsum, all);
    const double u = (double)p.uniform[ri];
    uint64_t goal = u > 0.0 ? (uint64_t)__builtin_fmin(u * (double)all, 9.2e18) : 0;
    goal = goal < all ? goal : all - 1;
    if (at <= goal && at + mine > goal) {
        int c = t * per;
        while (at + lds.cell[c] <= goal) at += lds.cell[c++];
        lds.bin = (uint32_t)c;
        lds.base = at;
    }
    __syncthreads();
    if (w == 0) {
        const int c0 = (int)lds.bin * 64 * V + lane * V;
        float y[V];
        load_vec<T>(r.row, c0, r.n, __builtin_nanf(""), y);
        uint64_t s[V], own = 0;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            s[j] = weight(y[j], c0 + j);
            own += s[j];
        }
        uint64_t run = lds.base + wave_scan(own, lane) - own;
        if (run <= goal && run + own > goal) {
            int j = 0;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                if (run + s[i] <= goal) {
                    run += s[i];
                    j = i + 1;
                } else {
                    break;
                }
            }
            p.tokens[ri] = c0 + j;
            if (p.logprobs) p.logprobs[ri] = (float)(-r.fall(T::get(r.row[c0 + j])) - log_sum);
        }
    }
}

int refuse(const char *who, const char *why) {
    std::fprintf(stderr, "%s: %s\n", who, why);
    return -1;
}
int launched(const char *who) {
    const hipError_t rc = hipGetLastError();
    if (rc != hipSuccess) {
        std::fprintf(stderr, "%s: launch failed: %s\n", who, hipGetErrorString(rc));
        return -1;
    }
    return 0;
}
bool misaligned(const void *p, int32_t dtype) {
    return (reinterpret_cast<uintptr_t>(p) & (dtype == GDN_DTYPE_FP32 ? 3 : 1)) != 0;
}

}  // namespace lg
}  // namespace gdn

extern "C" int gdn_logits_process(const GDNLogits *args, void *stream) {
    using namespace gdn::lg;
    constexpr const char *who = "gdn_logits_process";
    if (args == nullptr) return refuse(who, "args is NULL");
    const GDNLogits &a = *args;
    if (a.dtype < GDN_DTYPE_BF16 || a.dtype > GDN_DTYPE_FP32) return refuse(who, "unknown dtype");
    if (a.vocab > (1u << 24)) return refuse(who, "the vocabulary is larger than 2^24");
    if (a.rows > 65535) return refuse(who, "at most 65535 rows");
    if (a.rows == 0 || a.vocab == 0) return 0;
    if (!a.logits || !a.out || (a.history && !a.history_len) || (a.bias_offsets && a.n_bias && (!a.bias_ids || !a.bias_values)))
        return refuse(who, "a buffer pointer is NULL");
    if (misaligned(a.logits, a.dtype) || misaligned(a.out, a.dtype)) return refuse(who, "logits or out is misaligned");
    if (a.rows > 1 && (a.logits_stride < (int64_t)a.vocab || a.out_stride < (int64_t)a.vocab ||
                       (a.history && a.history_stride < (int64_t)a.history_width)))
        return refuse(who, "a row stride is smaller than the row");
    if (a.history_width > 0x7fffffffu || a.n_bias > 0x7fffffffu || a.n_masks > 0x7fffffffu)
        return refuse(who, "a size passes 2^31 - 1");
    if (a.mask && a.mask_stride < (int64_t)((a.vocab + 31) / 32)) return refuse(who, "mask rows are shorter than the vocabulary");
    if (a.mask && !a.mask_index && a.n_masks < a.rows) return refuse(who, "fewer masks than rows, and no mask_index");
    const dim3 grid((a.vocab + kTile - 1) / kTile, a.rows);
    const size_t lds = sizeof(uint32_t) * kTile * ((a.history != nullptr) + (a.bias_offsets != nullptr));
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (a.dtype == GDN_DTYPE_BF16) hipLaunchKernelGGL(k_process<Bf16>, grid, dim3(kPT), lds, s, a);
    else if (a.dtype == GDN_DTYPE_FP16) hipLaunchKernelGGL(k_process<Fp16>, grid, dim3(kPT), lds, s, a);
    else hipLaunchKernelGGL(k_process<Fp32>, grid, dim3(kPT), lds, s, a);
    return launched(who);
}

extern "C" int gdn_sample_tokens(const GDNSample *args, void *stream) {
    using namespace gdn::lg;
    constexpr const char *who = "gdn_sample_tokens";
    if (args == nullptr) return refuse(who, "args is NULL");
    const GDNSample &a = *args;
    if (a.dtype < GDN_DTYPE_BF16 || a.dtype > GDN_DTYPE_FP32) return refuse(who, "unknown dtype");
    if (a.vocab > (1u << 20)) return refuse(who, "the vocabulary is larger than 2^20");
    if (a.rows > 0x7fffffffu) return refuse(who, "at most 2^31 - 1 rows");
    if (a.rows == 0) return 0;
    if (a.vocab == 0) return refuse(who, "the vocabulary is empty");
    if (!a.logits || !a.tokens || (a.temperature && !a.uniform)) return refuse(who, "a buffer pointer is NULL");
    if (misaligned(a.logits, a.dtype)) return refuse(who, "logits is misaligned");
    if (a.rows > 1 && a.logits_stride < (int64_t)a.vocab) return refuse(who, "the row stride is smaller than the row");
    // 2^shift times the vocabulary stays below 2^63
    const int shift = a.vocab <= (1u << 18) ? 45 : 43;
    const dim3 grid(a.rows), block(kST);
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (a.dtype == GDN_DTYPE_BF16) hipLaunchKernelGGL(k_sample<Bf16>, grid, block, 0, s, a, shift);
    else if (a.dtype == GDN_DTYPE_FP16) hipLaunchKernelGGL(k_sample<Fp16>, grid, block, 0, s, a, shift);
    else hipLaunchKernelGGL(k_sample<Fp32>, grid, block, 0, s, a, shift);
    return launched(who);
}
