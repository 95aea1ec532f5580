// gdn_logits.hip -- from a batch of logits to tokens on the caller's device
// buffers: gdn_logits_process (penalties, biases, masks) and
// gdn_sample_tokens (the draw).
#include <hip/hip_runtime.h>

#include <cstdio>

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
// ones of the ranking up to a border (key, index), found by histograms: first
// over 2048 equal steps of (max - x) / temperature up to 32 -- what lies past
// them has no weight -- then over 11, 11 and 10 bits of the border step's keys.
constexpr int kST = 1024, kVals = 32, kBins = 2048;
constexpr int kCells = (1 << 20) / 256;  // waves' pieces of the longest row

// The 32-bit key of x that grows as x falls (x not NaN; the zeros are equal).
__device__ __forceinline__ uint32_t fall_key(float x) {
    const uint32_t u = f2u(x + 0.0f);
    return u & 0x80000000u ? u : ~u & 0x7fffffffu;
}

// exp(-d k ln 2) in steps of 2^-shift, d >= 0 (infinity: 0), from the Taylor
// series of the exponential about the nearest power of two (12 terms:
// 2e-16), k = log2(e) / temperature.
struct Weights {
    double k, unit, half;  // 2^shift
    __device__ __forceinline__ uint64_t of(float d) const {
        const double z = (double)d * k;
        if (!(z < 64.0)) return 0;
        const double e = __builtin_rint(z), t = (e - z) * 0.69314718055994530942;
        double y = 1.0 / 479001600.0;
        y = __builtin_fma(y, t, 1.0 / 39916800.0);
        y = __builtin_fma(y, t, 1.0 / 3628800.0);
        y = __builtin_fma(y, t, 1.0 / 362880.0);
        y = __builtin_fma(y, t, 1.0 / 40320.0);
        y = __builtin_fma(y, t, 1.0 / 5040.0);
        y = __builtin_fma(y, t, 1.0 / 720.0);
        y = __builtin_fma(y, t, 1.0 / 120.0);
        y = __builtin_fma(y, t, 1.0 / 24.0);
        y = __builtin_fma(y, t, 1.0 / 6.0);
        y = __builtin_fma(y, t, 0.5);
        y = __builtin_fma(y, t, 1.0);
        y = __builtin_fma(y, t, 1.0);
        // the sum's low bits are the rounded number of steps
        const double s = __builtin_fma(__builtin_ldexp(y, -(int)e), unit, 0x1p52);
        return __builtin_bit_cast(uint64_t, s) & 0xfffffffffffffull;
    }
};

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

struct SampleLds {
    uint32_t count[kBins];
    unsigned long long mass[kBins];
    uint64_t cell[kCells];
    uint64_t wsum[kST / 64];
    float wmax[kST / 64];
    uint32_t warg[kST / 64];
    double wexp[kST / 64];
    uint64_t before, inside;  // of the bin found: weight (or count) ranked before it, and in it
    uint64_t base;            // weight before it where counts decide
    uint32_t bin;
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
    for (int i = 0; i < kST / 64; ++i) {
        at += i < w ? wsum[i] : 0;
        all += wsum[i];
    }
    total = all;
    return at + s - v;
}

template <class T, bool ONE>
__global__ __launch_bounds__(kST) void k_sample(GDNSample p, int shift) {
    constexpr int V = T::kVec, NV = kVals / V, kPage = kST * kVals;
    __shared__ SampleLds lds;
    const int r = blockIdx.x, t = threadIdx.x, lane = t & 63, w = t >> 6, n = (int)p.vocab;
    const typename T::E *row = static_cast<const typename T::E *>(p.logits) + (size_t)r * p.logits_stride;
    const float nan = __builtin_nanf("");
    float x[NV][V];
    // f(value, index) over the row, a page of it in registers at a time; index
    // = page + (i kST + thread) V + j, so a wave's 64 V are consecutive
    auto load = [&](int page) {
#pragma unroll
        for (int i = 0; i < NV; ++i) load_vec<T>(row, page + (i * kST + t) * V, n, nan, x[i]);
    };
    if (ONE) load(0);
    auto each = [&](auto &&f) __attribute__((always_inline)) {
        for (int page = 0; page < (ONE ? 1 : n); page += kPage) {
            if (!ONE) load(page);
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    // a value of its own in every pass: what the passes form
                    // from it is cheaper again than kept (32 values a thread)
                    float v = x[i][j];
                    asm volatile("" : "+v"(v));
                    f(v, page + (i * kST + t) * V + j);
                }
        }
    };

    // the highest logit, and its first place
    float top = -kInf;
    int arg = 0x7fffffff;
    each([&](float v, int at) __attribute__((always_inline)) {
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
        lds.warg[w] = (uint32_t)arg;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kST / 64; ++i)
        if (lds.wmax[i] > top || (lds.wmax[i] == top && (int)lds.warg[i] < arg)) {
            top = lds.wmax[i];
            arg = (int)lds.warg[i];
        }
    if (arg == 0x7fffffff) {  // nothing above -infinity
        if (t == 0) {
            p.tokens[r] = -1;
            if (p.logprobs) p.logprobs[r] = -kInf;
        }
        return;
    }
    // how far below the highest, infinity for what carries no weight
    auto fall = [&](float v) __attribute__((always_inline)) {
        const float d = top - v;
        return v == top ? 0.0f : (d >= 0.0f ? d : kInf);
    };
    double log_sum = 0.0;
    if (p.logprobs) {
        double s = 0.0;
        each([&](float v, int) __attribute__((always_inline)) { s += (double)expf(-fall(v)); });
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) s += __shfl_xor(s, d);
        if (lane == 0) lds.wexp[w] = s;
        __syncthreads();
        s = 0.0;
#pragma unroll
        for (int i = 0; i < kST / 64; ++i) s += lds.wexp[i];
        log_sum = log(s);
    }
    const float temp = p.temperature ? p.temperature[r] : 0.0f;
    if (!(temp > 0.0f)) {
        if (t == 0) {
            p.tokens[r] = arg;
            if (p.logprobs) p.logprobs[r] = (float)-log_sum;
        }
        return;
    }
    Weights wt;
    wt.k = 1.44269504088896340736 / (double)temp;
    wt.unit = __builtin_ldexp(1.0, shift);
    const float step = __builtin_fminf((float)(kBins - 1) / (32.0f * temp), 3.0e38f);
    auto bin_of = [&](float d) __attribute__((always_inline)) {
        return (int)__builtin_fminf(d * step, (float)(kBins - 1));
    };
    const int k = p.top_k ? p.top_k[r] : 0;
    const float tp = p.top_p ? p.top_p[r] : 1.0f;
    // the border: tokens of a key below it are kept, of its key those up to
    // place edge_at
    uint32_t edge = 0xffffffffu;
    int edge_at = 0x7fffffff;

    // the first bin up to which the counts (by_mass: the weights) reach `goal`;
    // false if they never do
    auto find = [&](bool by_mass, double goal) __attribute__((always_inline)) {
        __syncthreads();
        const int b = 2 * t;
        const uint64_t m0 = lds.mass[b], m1 = lds.mass[b + 1], c0 = lds.count[b], c1 = lds.count[b + 1];
        uint64_t all;
        const uint64_t mb = block_scan(m0 + m1, lds.wsum, all), cb = block_scan(c0 + c1, lds.wsum, all);
        const uint64_t v0 = by_mass ? m0 : c0, v1 = by_mass ? m1 : c1, vb = by_mass ? mb : cb;
        if (t == 0) lds.bin = kBins;
        __syncthreads();
        if (v0 + v1 != 0 && (double)vb < goal && (double)(vb + v0 + v1) >= goal) {
            const bool second = !((double)(vb + v0) >= goal);
            lds.bin = b + second;
            lds.before = vb + (second ? v0 : 0);
            lds.inside = second ? v1 : v0;
            lds.base = mb + (second ? m0 : 0);
        }
        __syncthreads();
        return lds.bin;
    };
    // moves the border to where the ranking's counts or weights reach `goal`,
    // and gives the weight up to it (~0: it stays)
    auto cut = [&](bool by_mass, double goal) -> uint64_t {
        auto clear = [&]() __attribute__((always_inline)) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < kBins / kST; ++i) {
                lds.count[t + i * kST] = 0;
                lds.mass[t + i * kST] = 0;
            }
            __syncthreads();
        };
        auto put = [&](int bin, float d) __attribute__((always_inline)) {
            atomicAdd(&lds.count[bin], 1u);
            atomicAdd(&lds.mass[bin], (unsigned long long)wt.of(d));
        };
        clear();
        each([&](float v, int at) __attribute__((always_inline)) {
            const float d = fall(v);
            const int b = bin_of(d);
            const uint32_t key = fall_key(v);
            if (b < kBins - 1 && (key < edge || (key == edge && at <= edge_at))) put(b, d);
        });
        const uint32_t b0 = find(by_mass, goal);
        if (b0 >= kBins) return ~0ull;  // past the weights' end
        uint64_t base = lds.base;
        double left = goal - (double)lds.before;
        uint32_t prefix = 0;
        for (int level = 0; level < 3; ++level) {
            const int sh = level == 0 ? 21 : level == 1 ? 10 : 0;
            const uint32_t bits = level == 2 ? 0x3ffu : 0x7ffu;
            const uint32_t above = level == 0 ? 0u : ~0u << (level == 1 ? 21 : 10);
            clear();
            each([&](float v, int at) __attribute__((always_inline)) {
                const float d = fall(v);
                const uint32_t key = fall_key(v);
                if (bin_of(d) == (int)b0 && d < kInf && (key & above) == prefix &&
                    (key < edge || (key == edge && at <= edge_at)))
                    put((int)((key >> sh) & bits), d);
            });
            // what the bin above holds is all here: rounding past it ends there
            left = __builtin_fmin(left, (double)lds.inside);
            const uint32_t b = find(by_mass, left);
            prefix |= b << sh;
            left -= (double)lds.before;
            base += lds.base;
        }
        // of the border key's tokens (one weight all), the first `need` are kept
        const uint32_t have = lds.count[prefix & 0x3ffu];
        const uint64_t each_w = lds.mass[prefix & 0x3ffu] / have;
        uint64_t need;
        if (by_mass) {
            need = each_w ? (uint64_t)__builtin_ceil(left / (double)each_w) : have;
        } else {
            need = (uint64_t)left;
        }
        need = need < 1 ? 1 : need;
        if (need < have) {
            // its place: the pieces' counts, then the piece's own tokens
            __syncthreads();
            const int cells = (n + 64 * V - 1) / (64 * V);
            for (int page = 0; page < n; page += kPage) {
                if (!ONE) load(page);
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    uint32_t c = 0;
#pragma unroll
                    for (int j = 0; j < V; ++j) c += fall_key(x[i][j]) == prefix && x[i][j] == x[i][j];
#pragma unroll
                    for (int d = 1; d < 64; d <<= 1) c += __shfl_xor((int)c, d);
                    const int at = page / (64 * V) + i * (kST / 64) + w;
                    if (lane == 0 && at < cells) lds.cell[at] = c;
                }
            }
            __syncthreads();
            uint64_t mine = 0, all;
            const int per = (cells + kST - 1) / kST;
            for (int i = 0; i < per; ++i) mine += t * per + i < cells ? lds.cell[t * per + i] : 0;
            uint64_t at = block_scan(mine, lds.wsum, all);
            if (at < need && at + mine >= need) {
                int c = t * per;
                while (at + lds.cell[c] < need) at += lds.cell[c++];
                for (int i = c * 64 * V; i < n; ++i) {
                    const float v = T::get(row[i]);
                    if (v == v && fall_key(v) == prefix && ++at == need) {
                        lds.bin = (uint32_t)i;
                        break;
                    }
                }
            }
            __syncthreads();
            edge_at = (int)lds.bin;
        } else {
            need = have;
            if (prefix != edge) edge_at = 0x7fffffff;
        }
        edge = prefix;
        return base + need * each_w;
    };

    uint64_t kept_mass = ~0ull;
    if (k > 0 && k < n) kept_mass = cut(false, (double)k);
    if (tp < 1.0f) {
        if (!(tp > 0.0f)) {
            edge = fall_key(top);
            edge_at = arg;
        } else {
            if (kept_mass == ~0ull) {
                uint64_t s = 0;
                each([&](float v, int) __attribute__((always_inline)) { s += wt.of(fall(v)); });
                block_scan(s, lds.wsum, kept_mass);
            }
            cut(true, (double)tp * (double)kept_mass);
        }
    }
    const float mp = p.min_p ? p.min_p[r] : 0.0f;
    const double least = mp > 0.0f ? (double)__builtin_fminf(mp, 1.0f) * wt.unit : 0.0;
    auto weight = [&](float v, int at) __attribute__((always_inline)) -> uint64_t {
        const uint32_t key = fall_key(v);
        if (!(key < edge || (key == edge && at <= edge_at))) return 0;
        const uint64_t s = wt.of(fall(v));
        return (double)s >= least ? s : 0;
    };

    // the kept weights by pieces of 64 V tokens, the piece the draw falls in,
    // the token in it
    const int cells = (n + 64 * V - 1) / (64 * V);
    __syncthreads();
    for (int page = 0; page < n; page += kPage) {
        if (!ONE) load(page);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            uint64_t s = 0;
#pragma unroll
            for (int j = 0; j < V; ++j) s += weight(x[i][j], page + (i * kST + t) * V + j);
            s = wave_scan(s, lane);
            const int at = page / (64 * V) + i * (kST / 64) + w;
            if (lane == 63 && at < cells) lds.cell[at] = s;
        }
    }
    __syncthreads();
    uint64_t mine = 0, all;
    const int per = (cells + kST - 1) / kST;
    for (int i = 0; i < per; ++i) mine += t * per + i < cells ? lds.cell[t * per + i] : 0;
    uint64_t at = block_scan(mine, lds.wsum, all);
    const double u = (double)p.uniform[r];
    uint64_t goal = u > 0.0 ? (uint64_t)__builtin_fmin(u * (double)all, 9.2e18) : 0;
    goal = goal < all ? goal : all - 1;
    if (at <= goal && at + mine > goal) {
        int c = t * per;
        while (at + lds.cell[c] <= goal) at += lds.cell[c++];
        lds.bin = (uint32_t)c;
        lds.before = at;
    }
    __syncthreads();
    if (w == 0) {
        const int c0 = (int)lds.bin * 64 * V + lane * V;
        float y[V];
        load_vec<T>(row, c0, n, nan, y);
        uint64_t s[V], sum = 0;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            s[j] = weight(y[j], c0 + j);
            sum += s[j];
        }
        uint64_t run = lds.before + wave_scan(sum, lane) - sum;
        if (run <= goal && run + sum > goal) {
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
            p.tokens[r] = c0 + j;
            if (p.logprobs) p.logprobs[r] = (float)(-(double)fall(T::get(row[c0 + j])) - log_sum);
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
    const bool one = a.vocab <= (uint32_t)(kST * kVals);
    hipStream_t s = static_cast<hipStream_t>(stream);
#define GDN_LAUNCH_SAMPLE(T)                                                                  \
    if (one) hipLaunchKernelGGL((k_sample<T, true>), grid, block, 0, s, a, shift);            \
    else hipLaunchKernelGGL((k_sample<T, false>), grid, block, 0, s, a, shift)
    if (a.dtype == GDN_DTYPE_BF16) {
        GDN_LAUNCH_SAMPLE(Bf16);
    } else if (a.dtype == GDN_DTYPE_FP16) {
        GDN_LAUNCH_SAMPLE(Fp16);
    } else {
        GDN_LAUNCH_SAMPLE(Fp32);
    }
#undef GDN_LAUNCH_SAMPLE
    return launched(who);
}
