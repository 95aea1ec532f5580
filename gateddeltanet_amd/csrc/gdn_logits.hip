// gdn_logits.hip -- from a batch of logits to tokens on the caller's device
// buffers: gdn_logits_process (penalties, biases, masks) and
// gdn_sample_tokens (the draw).
#include <hip/hip_runtime.h>

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

// Sixteen bytes in one load (copied element by element they take four).
template <class T>
__device__ __forceinline__ Vec<T> load16(const typename T::E *p) {
    u32x4 w;
    __builtin_memcpy(&w, p, sizeof(w));
    return __builtin_bit_cast(Vec<T>, w);
}
// Elements at .. at + kVec - 1 of a row of n; `rest` past its end.
template <class T>
__device__ __forceinline__ void load_vec(const typename T::E *row, int at, int n, float rest, float (&x)[T::kVec]) {
    if (at + T::kVec <= n) {
        const Vec<T> v = load16<T>(row + at);
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
// goes in by maximum, so the last of equal ids holds.  The tile's logits are on
// their way meanwhile.
// 64 rows of 32000 FP32 logits, histories of 2500 tokens, biases and masks: 7.1 us
// (17 MB, 2.4 TB/s; one row 4.1 us), bound by the steps' latencies: clearing, the
// ids, the atomics, the row.  256 rows of 99991 BF16 logits: 36 us (2.9 TB/s), 30
// without histories.  Tiles of 4096 on 512 threads: 35 and 27 us there, but 16.2
// against 15.0 at 256 x 32000 and 11.6 against 8.7 for histories of 20000, which
// every tile reads; the ids ahead of the clearing 2 to 4 % slower.
constexpr int kTile = 8192, kPT = 1024;
constexpr uint32_t kSeen = 0x80000000u;

template <class T>
__global__ __launch_bounds__(kPT) void k_process(GDNLogits p) {
    constexpr int V = T::kVec, NV = kTile / (V * kPT), kAhead = 4;
    extern __shared__ __attribute__((aligned(16))) uint32_t mem[];
    uint32_t *count = mem, *entry = mem + (p.history ? kTile : 0);
    const int r = blockIdx.y, t0 = blockIdx.x * kTile, t = threadIdx.x;
    const int n = min((int)p.vocab - t0, kTile);
    const typename T::E *in = static_cast<const typename T::E *>(p.logits) + (size_t)r * p.logits_stride + t0;
    typename T::E *out = static_cast<typename T::E *>(p.out) + (size_t)r * p.out_stride + t0;
    float x[NV][V];
#pragma unroll
    for (int i = 0; i < NV; ++i)
        if ((i * kPT + t) * V < n) load_vec<T>(in, (i * kPT + t) * V, n, 0.0f, x[i]);
    int len = 0, prompt = 0, b0 = 0, b1 = 0;
    const u32x4 none = {0u, 0u, 0u, 0u};
    if (p.history) {
        len = min(max(p.history_len[r], 0), (int)p.history_width);
        prompt = p.prompt_len ? p.prompt_len[r] : 0;
        for (int i = t; i < kTile / 4; i += kPT) reinterpret_cast<u32x4 *>(count)[i] = none;
    }
    if (p.bias_offsets) {
        b0 = min(max(p.bias_offsets[r], 0), (int)p.n_bias);
        b1 = min(max(p.bias_offsets[r + 1], b0), (int)p.n_bias);
        for (int i = t; i < kTile / 4; i += kPT) reinterpret_cast<u32x4 *>(entry)[i] = none;
    }
    const float rep = p.repetition ? p.repetition[r] : 1.0f, pres = p.presence ? p.presence[r] : 0.0f,
                freq = p.frequency ? p.frequency[r] : 0.0f;
    const int mi = p.mask ? (p.mask_index ? p.mask_index[r] : r) : -1;
    const uint32_t *mask = mi >= 0 && mi < (int)p.n_masks ? p.mask + (size_t)mi * p.mask_stride + t0 / 32 : nullptr;
    uint32_t allowed[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int at = (i * kPT + t) * V;
        allowed[i] = mask && at < n ? mask[at / 32] >> (at & 31) : ~0u;
    }
    __syncthreads();
    const int32_t *hist = p.history + (size_t)r * p.history_stride;
    for (int i0 = t; i0 < len; i0 += kAhead * kPT) {
        uint32_t id[kAhead];
#pragma unroll
        for (int a = 0; a < kAhead; ++a) id[a] = (uint32_t)hist[min(i0 + a * kPT, len - 1)] - (uint32_t)t0;
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            const int i = i0 + a * kPT;
            if (i < len && id[a] < (uint32_t)n) {
                if (i >= prompt) atomicAdd(&count[id[a]], 1u);
                atomicOr(&count[id[a]], kSeen);
            }
        }
    }
    for (int i = b0 + t; i < b1; i += kPT) {
        const uint32_t id = (uint32_t)p.bias_ids[i] - (uint32_t)t0;
        if (id < (uint32_t)n) atomicMax(&entry[id], (uint32_t)(i - b0) + 1u);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int at = (i * kPT + t) * V;
        if (at >= n) break;
        uint32_t c[V] = {}, b[V] = {};
        if (p.history) {
#pragma unroll
            for (int j = 0; j < V; ++j) c[j] = count[at + j];
        }
        if (p.bias_offsets) {
#pragma unroll
            for (int j = 0; j < V; ++j) b[j] = entry[at + j];
        }
#pragma unroll
        for (int j = 0; j < V; ++j) {
            if (c[j]) {
                x[i][j] = x[i][j] > 0.0f ? x[i][j] / rep : x[i][j] * rep;
                const uint32_t said = c[j] & ~kSeen;
                if (said) x[i][j] = (x[i][j] - freq * (float)said) - pres;
            }
            if (b[j]) x[i][j] = x[i][j] + p.bias_values[b0 + (int)b[j] - 1];
            if (!((allowed[i] >> j) & 1u)) x[i][j] = -kInf;
        }
        store_vec<T>(out, at, n, x[i]);
    }
}

// ------------------------------------------------------------ the draw

// A workgroup a row.  Weights are whole numbers of 2^-shift, so counts and
// sums over the row are the same in any order.  The kept tokens are the first
// ones of the ranking up to a border (logit, index): one histogram over kBins
// steps of 1 / 32 in (max - x) / temperature -- what lies past them has no
// weight -- gives the step the border is in, and the step's tokens, usually
// some tens, are ranked against each other in LDS.  More than fit there go
// through histograms of 10 bits of their keys at a time.  A row that fits stays
// in LDS from its one reading on (HELD); what each pass then costs is its
// instructions, so the FP64 weights are formed only for the tokens that need
// them: a token's bounds are compared in FP32 first.
// 64 rows of 32000 FP32 logits: 18 us for top-k 50, 20 us for a top-p whose border
// lies among the threads' highest tokens; 37 us for one that lies among hundreds,
// of which 13 are the FP64 weights of the whole row; 24 us with neither.  Held rows
// against slices (below), 64 x 32000: 18 against 30 us for top-k, 37 against 36 for
// the flat top-p; 1024 x 32000: 76 against 137, 146 against 182.  Few long rows are
// the rule's cost: one BF16 row of 65536 takes 40 us with neither and 87 with a top-p
// of 0.99, one of 131072 in slices 19 and 46.  A thread's 128 registers spill 18 for
// the 16-bit types, 2 for FP32 (in k_wide_border 8 to 14).
constexpr int kST = 1024, kBins = kST, kWaves = kST / 64;
constexpr int kList = 512;             // tokens that are ranked against each other
// A step of more tokens is cut in parts first, 2.4 us; ranking 65 takes 1.9 us, 111
// 2.8, 196 6.7, 276 16.  512 here: 8 x 131072 54 to 58 us for 46 to 50; 64: equal.
constexpr int kFew = 128;
constexpr int kHeldBytes = 128 << 10;  // of a row in LDS
constexpr int kMostVocab = 1 << 20;
constexpr int kNowhere = 0x7fffffff;

// The 32-bit key of x that grows as x falls (x not NaN; the zeros are equal).
__device__ __forceinline__ uint32_t fall_key(float x) {
    const uint32_t u = f2u(x + 0.0f);
    return u & 0x80000000u ? u : ~u & 0x7fffffffu;
}
__device__ __forceinline__ float of_key(uint32_t k) { return u2f(k & 0x80000000u ? k : ~k & 0x7fffffffu); }

struct Ranked {
    float x;
    int at;
    uint64_t w;
};
template <class T, bool HELD>
struct SampleLds {
    static constexpr int kHeld = HELD ? kHeldBytes / (int)sizeof(typename T::E) : T::kVec;
    // pieces of 64 vectors
    static constexpr int kCells = (HELD ? kHeld : kMostVocab) / (64 * T::kVec);
    typename T::E held[kHeld] __attribute__((aligned(16)));
    union {
        struct {
            unsigned long long mass[kBins];
            uint32_t count[kBins];
        };
        Ranked list[kList];
        uint64_t cell[kCells];
    };
    // tokens gathered from the row, and their places
    static constexpr int kSome = HELD ? 3 * kST / 2 : 8 * kST;
    float some[kSome];
    int some_at[kSome];
    uint64_t before[kList];
    uint64_t wsum[2][kWaves];
    float wmax[kWaves];
    int warg[kWaves];
    double wexp[kWaves], guess[2][kWaves];
    uint64_t base;    // weight ranked before a bin found
    double left;      // of the goal, in it
    float x;          // a border
    int at;
    uint32_t bin, n, ahead, n_some, all_above, crowded;
};

__device__ __forceinline__ uint64_t lane_of(uint64_t v, int lane) {
    return ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32) |
           (uint32_t)__builtin_amdgcn_readlane((int)v, lane);
}
// The sum over the workgroup before each thread, and the whole sum.  Between
// two uses of one `wsum` stands a barrier.
__device__ __forceinline__ uint64_t block_scan(uint64_t v, uint64_t (&wsum)[kWaves], uint64_t &total) {
    static_assert(kWaves <= 64, "a lane a wave");
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint64_t s = wave_scan64(v);
    if (lane == 63) wsum[w] = s;
    __syncthreads();
    const uint64_t waves = wave_scan64(lane < kWaves ? wsum[lane] : 0);
    total = lane_of(waves, kWaves - 1);
    return (w ? lane_of(waves, w - 1) : 0) + s - v;
}

// A row and how its tokens fall and weigh.
template <class T, bool HELD>
struct Row {
    static constexpr int V = T::kVec;
    typedef SampleLds<T, HELD> Lds;
    const typename T::E *row;
    Lds *lds;
    int n;
    float top;
    bool endless;  // the highest is infinity
    int shift;
    double top_d, rate, step, width;  // log2(e) / temperature, 32 / temperature, temperature / 32

    __device__ __forceinline__ void set(float highest, float temp, int to) {
        top = highest;
        top_d = (double)highest;
        endless = highest == kInf;
        shift = to;
        rate = 1.44269504088896340736 / (double)temp;
        step = 32.0 / (double)temp;
        width = (double)temp * (1.0 / 32.0);
    }
    __device__ __forceinline__ void load(int at, float (&x)[V]) const {
        if constexpr (HELD) {
            const Vec<T> v = *reinterpret_cast<const Vec<T> *>(__builtin_assume_aligned(&lds->held[at], 16));
#pragma unroll
            for (int j = 0; j < V; ++j) x[j] = T::get(v.e[j]);
        } else {
            load_vec<T>(row, at, n, __builtin_nanf(""), x);
        }
    }
    // f(values, index of the first), a wave's 64 V tokens consecutive; from
    // memory eight vectors of a thread on their way at a time
    template <class F>
    __device__ __forceinline__ void each(F &&f) const {
        if constexpr (HELD) {
            constexpr int kUnroll = 16 / V;
#pragma unroll kUnroll
            for (int at = (int)threadIdx.x * V; at < n; at += kST * V) {
                float x[V];
                load(at, x);
                f(x, at);
            }
        } else {
            constexpr int kAhead = 8;
            const int whole = n / V;
            for (int first = (int)threadIdx.x; first < whole; first += kAhead * kST) {
                Vec<T> v[kAhead];
#pragma unroll
                for (int a = 0; a < kAhead; ++a)
                    v[a] = load16<T>(row + (size_t)min(first + a * kST, whole - 1) * V);
#pragma unroll
                for (int a = 0; a < kAhead; ++a)
                    if (first + a * kST < whole) {
                        float x[V];
#pragma unroll
                        for (int j = 0; j < V; ++j) x[j] = T::get(v[a].e[j]);
                        f(x, (first + a * kST) * V);
                    }
            }
            if (n % V != 0 && threadIdx.x == kST - 1) {
                float x[V];
                load(whole * V, x);
                f(x, whole * V);
            }
        }
    }
    // how far below the highest; NaN for NaN, whose bin and weight are those of
    // infinity
    __device__ __forceinline__ double fall(float v) const {
        if (endless) return v == top ? 0.0 : (double)kInf;
        return top_d - (double)v;
    }
    // kBins where the weight is 0: exp(-32) is half a unit of 2^-45
    __device__ __forceinline__ int bin(double d) const { return (int)__builtin_fmin(d * step, (double)kBins); }
    // exp(-d / temperature) 2^shift, rounded to a whole number: the Taylor
    // series of the exponential about the nearest power of two (|t| <= ln 2 / 2:
    // the first term left out is 6e-15)
    __device__ __forceinline__ uint64_t weight(double d) const {
        const double z = __builtin_fmin(d * rate, 1000.0), n = __builtin_rint(z), t = (n - z) * 0.69314718055994530942;
        double y = 1.0 / 39916800.0;
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
        // the sum's low bits are the rounded number
        return __builtin_bit_cast(uint64_t, __builtin_ldexp(y, shift - (int)n) + 0x1p52) & 0xfffffffffffffull;
    }
    // FP32 bounds that hold every token of the steps b .. e - 1 (and a few
    // others: rounding)
    __device__ __forceinline__ void bounds(int b, int e, float &lo, float &hi) const {
        const double slack = __builtin_fabs(top_d) * 0x1p-22 + 0x1p-126;
        hi = (float)(top_d - (double)b * width + slack);
        lo = (float)(top_d - (double)e * width - slack);
        if (!(hi < top)) hi = top;
        if (!(lo > -kInf)) lo = -kInf;  // (-infinity - infinity too)
    }
};

// The border of the tokens of step `b` (there are `inside`, and `ahead` above) whose ranked counts
// (by_mass: weights) first reach `left`, into lds.x and lds.at; their weight is
// the result.  listed: they are among the threads' `own` (none: at < 0).
template <class T, bool HELD>
__device__ __forceinline__ uint64_t border_in(const Row<T, HELD> &r, SampleLds<T, HELD> &lds, int b, uint32_t ahead,
                                              uint32_t inside, bool by_mass, double left, bool listed, const Ranked &own) {
    constexpr int V = T::kVec;
    const int t = threadIdx.x;
    float lo, hi;
    r.bounds(b, b + 1, lo, hi);
    // The step's tokens lie among many others, so that nearly every wave would
    // form their weights for a few lanes: they are gathered first where they
    // fit (131072 tokens: 30 us a pass otherwise); with those above them, for
    // the draw, if the row is held and these fit too
    constexpr int kSome = SampleLds<T, HELD>::kSome;
    uint32_t n_some = kSome + 1;
    for (int turn = HELD && ahead + inside <= (uint32_t)kSome ? 0 : 1; turn < 2 && !listed && n_some > (uint32_t)kSome; ++turn) {
        const float most = turn == 0 ? kInf : hi;
        __syncthreads();
        if (t == 0) {
            lds.n_some = 0;
            lds.all_above = turn == 0;
        }
        __syncthreads();
        r.each([&](const float(&x)[V], int at) __attribute__((always_inline)) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const bool in = x[j] >= lo && x[j] <= most;
                const uint64_t who = __ballot(in);
                if (who == 0) continue;
                const int before = (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0u));
                uint32_t i = 0;
                if (in && before == 0) i = atomicAdd(&lds.n_some, (uint32_t)__builtin_popcountll(who));
                i = (uint32_t)__builtin_amdgcn_readlane((int)i, __builtin_ctzll(who)) + before;
                if (in && i < (uint32_t)kSome) {
                    lds.some[i] = x[j];
                    lds.some_at[i] = at + j;
                }
            }
        });
        __syncthreads();
        n_some = lds.n_some;
    }
    // f(token, index, fall) over the step's
    auto each_of = [&](auto &&f) __attribute__((always_inline)) {
        auto one = [&](float x, int at) __attribute__((always_inline)) {
            const double d = r.fall(x);
            if (r.bin(d) == b) f(x, at, d);
        };
        if (listed) {
            if (own.at >= 0) one(own.x, own.at);
        } else if (n_some <= (uint32_t)kSome) {
            for (uint32_t i = t; i < n_some; i += kST) one(lds.some[i], lds.some_at[i]);
        } else {
            r.each([&](const float(&x)[V], int at) __attribute__((always_inline)) {
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (x[j] >= lo && x[j] <= hi) one(x[j], at + j);
            });
        }
    };
    // the bin of a histogram in lds that the goal is in, into lds.bin; moves
    // base and left to it and gives its count
    uint64_t base = 0;
    auto find = [&]() __attribute__((always_inline)) -> uint32_t {
        __syncthreads();
        const uint64_t m = lds.mass[t], c = lds.count[t];
        uint64_t all_m, all_c;
        const uint64_t mb = block_scan(m, lds.wsum[0], all_m), cb = block_scan(c, lds.wsum[1], all_c);
        const uint64_t v = by_mass ? m : c, vb = by_mass ? mb : cb;
        // what the bin above holds is all here: rounding past it ends there
        const double goal = __builtin_fmin(left, (double)(by_mass ? all_m : all_c));
        if (v != 0 && (double)vb < goal && (double)(vb + v) >= goal) {
            lds.bin = (uint32_t)t;
            lds.left = goal - (double)vb;
            lds.base = mb;
        }
        __syncthreads();
        left = lds.left;
        base += lds.base;
        return lds.count[lds.bin];
    };
    auto clear = [&]() __attribute__((always_inline)) {
        __syncthreads();
        lds.count[t] = 0;
        lds.mass[t] = 0;
        __syncthreads();
    };
    auto put = [&](int i, double d) __attribute__((always_inline)) {
        atomicAdd(&lds.count[i], 1u);
        atomicAdd(&lds.mass[i], (unsigned long long)r.weight(d));
    };
    // a crowded step in kBins parts
    auto part_of = [&](double d) __attribute__((always_inline)) {
        return min(max((int)((d * r.step - (double)b) * (double)kBins), 0), kBins - 1);
    };
    int part = -1;
    if (inside > (uint32_t)kFew) {
        clear();
        each_of([&](float, int, double d) __attribute__((always_inline)) { put(part_of(d), d); });
        inside = find();
        part = (int)lds.bin;
    }
    if (inside <= (uint32_t)kList) {
        __syncthreads();
        if (t == 0) lds.n = 0;
        __syncthreads();
        each_of([&](float x, int at, double d) __attribute__((always_inline)) {
            if (part >= 0 && part_of(d) != part) return;
            const uint32_t i = atomicAdd(&lds.n, 1u);
            if (i < (uint32_t)kList) lds.list[i] = Ranked{x, at, r.weight(d)};
        });
        __syncthreads();
        inside = lds.n;
    }
    if (inside <= (uint32_t)kList) {
        // the tokens' own ranks, several threads a token: i % each of them
        // compares with every each-th
        const int n = (int)inside;
        int lanes = kST / kList;
        while (lanes < 64 && 2 * lanes * n <= kST) lanes *= 2;
        static_assert(kList <= kBins, "room for ranks");
        if (t < kList) {
            lds.count[t] = 0;
            lds.before[t] = 0;
        }
        __syncthreads();
        const int who = t / lanes;
        if (who < n) {
            const Ranked me = lds.list[who];
            uint32_t rank = 0;
            uint64_t before = 0;
#pragma unroll 4
            for (int i = t % lanes; i < n; i += lanes) {
                const Ranked o = lds.list[i];
                const bool first = o.x > me.x || (o.x == me.x && o.at < me.at);
                rank += first;
                before += first ? o.w : 0;
            }
            if (rank != 0) {
                atomicAdd(&lds.count[who], rank);
                atomicAdd(reinterpret_cast<unsigned long long *>(&lds.before[who]), (unsigned long long)before);
            }
        }
        __syncthreads();
        if (t < n) {
            const Ranked me = lds.list[t];
            const int rank = (int)lds.count[t];
            const uint64_t before = lds.before[t];
            const double from = by_mass ? (double)before : (double)rank,
                         to = by_mass ? (double)(before + me.w) : (double)(rank + 1);
            // rounding in `left` past the step's end: its last token
            if ((from < left && to >= left) || (rank == n - 1 && to < left)) {
                lds.x = me.x;
                lds.at = me.at;
                lds.base = before + me.w;
            }
        }
        __syncthreads();
        return base + lds.base;
    }
    // by their keys' bits
    uint64_t each_w = 0;
    uint32_t prefix = 0, above = 0, have = 0;
    for (int sh = 22; sh >= 0; sh -= sh > 2 ? 10 : sh == 2 ? 2 : 1) {
        const uint32_t bits = sh == 0 ? 3u : 0x3ffu;
        clear();
        each_of([&](float x, int, double d) __attribute__((always_inline)) {
            const uint32_t key = fall_key(x);
            if ((key & above) == prefix && (part < 0 || part_of(d) == part)) put((int)((key >> sh) & bits), d);
        });
        have = find();
        prefix |= lds.bin << sh;
        above |= bits << sh;
        each_w = lds.mass[lds.bin] / have;
    }
    // of the border key's tokens (one weight all), the first `need` are kept
    uint64_t need = by_mass ? (uint64_t)__builtin_ceil(left / (double)each_w) : (uint64_t)left;
    need = need < 1 ? 1 : (need < have ? need : have);
    const float edge = of_key(prefix);
    // the place of the last of these: the pieces' counts, then the piece's own
    const int n_cells = (r.n + 64 * V - 1) / (64 * V), lane = t & 63, w = t >> 6;
    __syncthreads();
    for (int c = w; c < n_cells; c += kWaves) {
        const int at = (c * 64 + lane) * V;
        float x[V] = {};
        uint32_t k = 0;
        if (at < r.n) {
            r.load(at, x);
#pragma unroll
            for (int j = 0; j < V; ++j) k += x[j] == edge;
        }
        const uint64_t sum = wave_scan64((uint64_t)k);
        if (lane == 63) lds.cell[c] = sum;
    }
    __syncthreads();
    const int per = (n_cells + kST - 1) / kST;
    uint64_t mine = 0, all;
    for (int i = 0; i < per; ++i) mine += t * per + i < n_cells ? lds.cell[t * per + i] : 0;
    uint64_t at = block_scan(mine, lds.wsum[0], all);
    if (at < need && at + mine >= need) {
        int c = t * per;
        while (at + lds.cell[c] < need) at += lds.cell[c++];
        for (int i = c * 64 * V; i < r.n; ++i)
            if (T::get(r.row[i]) == edge && ++at == need) {
                lds.x = edge;
                lds.at = i;
                break;
            }
    }
    __syncthreads();
    return base + need * each_w;
}

// What a row is asked for.
struct Ask {
    float temp, top_p, min_p;
    int k;
    double u;
    bool greedy, first_only, by_k, by_p;
    __device__ __forceinline__ Ask(const GDNSample &p, int r) {
        temp = p.temperature ? p.temperature[r] : 0.0f;
        k = p.top_k ? p.top_k[r] : 0;
        top_p = p.top_p ? p.top_p[r] : 1.0f;
        min_p = p.min_p ? p.min_p[r] : 0.0f;
        u = p.temperature ? (double)p.uniform[r] : 0.0;
        greedy = !(temp > 0.0f);
        first_only = top_p <= 0.0f;
        by_k = !greedy && !first_only && k > 0 && k < (int)p.vocab;
        by_p = !greedy && !first_only && top_p < 1.0f;
    }
};

// The highest of a wave's values and its first place, in every lane.
__device__ __forceinline__ void first_of_highest(float &v, int &at) {
    const float most = u2f(wave_reduce64(f2u(v), [](uint32_t a, uint32_t b) { return f2u(__builtin_fmaxf(u2f(a), u2f(b))); }));
    at = (int)wave_reduce64((uint32_t)(v == most ? at : kNowhere), [](uint32_t a, uint32_t b) { return a < b ? a : b; });
    v = most;
}
template <class T>
__device__ __forceinline__ void higher(const float (&x)[T::kVec], int at, float &top, int &arg) {
#pragma unroll
    for (int j = 0; j < T::kVec; ++j)
        if (x[j] > top) {
            top = x[j];
            arg = at + j;
        }
}

// The sum of exp(x - top), each to (2 + d) 2^-24 of it; 0 for NaN and what is
// too small (of two infinities: with the highest's 1).
template <class R, int V>
__device__ __forceinline__ float exponentials(const R &r, const float (&x)[V]) {
    constexpr float kL = 1.44269502f, kLo = 1.92596299e-8f;  // log2(e)
    float s = 0.0f;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const float d = r.top - x[j];
        s += __builtin_fmaxf(__builtin_amdgcn_exp2f(-__builtin_fmaf(d, kL, d * kLo)), 0.0f);
        if (r.endless) s += x[j] == r.top ? 1.0f : 0.0f;
    }
    return s;
}

// What is kept: tokens above `edge`, of its logit those up to place edge_at, of
// weight `least` and more.
struct Keep {
    float edge = -kInf, from = -kInf;
    int edge_at = kNowhere;
    double least = 0.0;
    template <class R>
    __device__ __forceinline__ void finish(const R &r, const Ask &ask, float lowest) {
        from = edge > lowest ? edge : lowest;
        least = ask.min_p > 0.0f ? __builtin_ldexp((double)__builtin_fminf(ask.min_p, 1.0f), r.shift) : 0.0;
    }
    __device__ __forceinline__ bool has(float x, int at) const { return x > edge || (x == edge && at <= edge_at); }
    template <class R>
    __device__ __forceinline__ uint64_t weight(const R &r, float x, int at) const {
        if (!(x >= from) || (x == edge && at > edge_at)) return 0;
        const uint64_t s = r.weight(r.fall(x));
        return (double)s >= least ? s : 0;
    }
    // of the 64 V tokens from `c`, in lane 63
    template <class R>
    __device__ __forceinline__ uint64_t piece(const R &r, int c, int lane) const {
        const int at = (c * 64 + lane) * R::V;
        uint64_t s = 0;
        if (at < r.n) {
            float x[R::V];
            r.load(at, x);
#pragma unroll
            for (int j = 0; j < R::V; ++j) s += weight(r, x[j], at + j);
        }
        return __ballot(s != 0) != 0 ? wave_scan64(s) : 0;
    }
};

// The borders asked for, from the steps' counts and weights (a thread a step);
// `kept`: the weight that top-p is a share of, unless top-k gives another.
// Returns the weight up to the last.
template <class T, bool HELD>
__device__ __forceinline__ uint64_t borders(const Row<T, HELD> &r, SampleLds<T, HELD> &lds, const Ask &ask, uint64_t count,
                                            uint64_t mass, uint64_t n_before, uint64_t m_before, uint64_t n_all,
                                            uint64_t kept, bool listed, const Ranked &own, Keep &keep) {
    // by counts, then by weights: tokens past the first border rank behind all
    // that reach the second goal, which is less than the whole weight
    for (int turn = 0; turn < 2; ++turn) {
        const bool by_mass = turn == 1;
        if (by_mass ? !ask.by_p : !ask.by_k || (uint64_t)ask.k > n_all) continue;
        const double goal = by_mass ? (double)ask.top_p * (double)kept : (double)ask.k;
        const uint64_t before = by_mass ? m_before : n_before, here = by_mass ? mass : count;
        __syncthreads();
        if (here != 0 && (double)before < goal && (double)(before + here) >= goal) {
            lds.bin = threadIdx.x;
            lds.left = goal - (double)before;
            lds.base = m_before;
            lds.n = (uint32_t)count;
            lds.ahead = (uint32_t)n_before;
        }
        __syncthreads();
        const uint64_t base = lds.base;
        kept = base + border_in(r, lds, (int)lds.bin, lds.ahead, lds.n, by_mass, lds.left, listed, own);
        if (lds.x > keep.edge || (lds.x == keep.edge && lds.at < keep.edge_at)) {
            keep.edge = lds.x;
            keep.edge_at = lds.at;
        }
    }
    return kept;
}

// The token up to which the pieces' kept weights (lds.cell) reach the draw, in
// one lane of wave 0; -1 elsewhere.
template <class T, bool HELD>
__device__ __forceinline__ int drawn(const Row<T, HELD> &r, SampleLds<T, HELD> &lds, const Keep &keep, double u) {
    constexpr int V = T::kVec;
    const int t = threadIdx.x, lane = t & 63, w = t >> 6;
    const int cells = (r.n + 64 * V - 1) / (64 * V), per = (cells + kST - 1) / kST;
    uint64_t mine = 0, all;
    for (int i = 0; i < per; ++i) mine += t * per + i < cells ? lds.cell[t * per + i] : 0;
    uint64_t at = block_scan(mine, lds.wsum[0], all);
    // (u is bounded, not the product: `all` may be 2^63)
    uint64_t goal = u > 0.0 ? (uint64_t)(__builtin_fmin(u, 1.0) * (double)all) : 0;
    goal = goal < all ? goal : all - 1;
    if (at <= goal && at + mine > goal) {
        int c = t * per;
        while (at + lds.cell[c] <= goal) at += lds.cell[c++];
        lds.bin = (uint32_t)c;
        lds.base = at;
    }
    __syncthreads();
    if (w != 0) return -1;
    const int c0 = (int)lds.bin * 64 * V + lane * V;
    float y[V];
    uint64_t s[V], here = 0;
    if (c0 < r.n) r.load(c0, y);
#pragma unroll
    for (int j = 0; j < V; ++j) {
        s[j] = c0 < r.n ? keep.weight(r, y[j], c0 + j) : 0;
        here += s[j];
    }
    uint64_t run = lds.base + wave_scan64(here) - here;
    if (!(run <= goal && run + here > goal)) return -1;
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
    return c0 + j;
}

// Rows that LDS holds.
template <class T>
__global__ __launch_bounds__(kST) void k_sample(GDNSample p, int shift) {
    constexpr int V = T::kVec;
    __shared__ SampleLds<T, true> lds;
    static_assert(sizeof(lds) <= 160 << 10, "the LDS of a CU");
    const int ri = blockIdx.x, t = threadIdx.x, lane = t & 63, w = t >> 6;
    Row<T, true> r;
    r.row = static_cast<const typename T::E *>(p.logits) + (size_t)ri * p.logits_stride;
    r.n = (int)p.vocab;
    r.lds = &lds;
    const Ask ask(p, ri);

    // the highest logit, and its first place; every vector of a thread on its
    // way at a time
    float top = -kInf;
    int arg = kNowhere;
    {
        constexpr int kAhead = SampleLds<T, true>::kHeld / (kST * V);
        const int whole = r.n / V, rest = r.n % V;
        if (whole > 0) {
            Vec<T> v[kAhead];
#pragma unroll
            for (int i = 0; i < kAhead; ++i)
                v[i] = load16<T>(r.row + (size_t)min(i * kST + t, whole - 1) * V);
#pragma unroll
            for (int i = 0; i < kAhead; ++i)
                if (i * kST + t < whole) {
                    float x[V];
#pragma unroll
                    for (int j = 0; j < V; ++j) x[j] = T::get(v[i].e[j]);
                    higher<T>(x, (i * kST + t) * V, top, arg);
                    *reinterpret_cast<Vec<T> *>(__builtin_assume_aligned(&lds.held[(i * kST + t) * V], 16)) = v[i];
                }
        }
        if (rest > 0 && t == kST - 1) {
            float x[V];
            load_vec<T>(r.row, whole * V, r.n, __builtin_nanf(""), x);
            higher<T>(x, whole * V, top, arg);
#pragma unroll
            for (int j = 0; j < V; ++j) lds.held[whole * V + j] = T::put(x[j]);
        }
    }
    const float own_top = top;
    first_of_highest(top, arg);
    if (lane == 0) {
        lds.wmax[w] = top;
        lds.warg[w] = arg;
    }
    lds.count[t] = 0;
    lds.mass[t] = 0;
    __syncthreads();
    top = lane < kWaves ? lds.wmax[lane] : -kInf;
    arg = lane < kWaves ? lds.warg[lane] : kNowhere;
    first_of_highest(top, arg);
    if (arg == kNowhere) {  // nothing above -infinity
        if (t == 0) {
            p.tokens[ri] = -1;
            if (p.logprobs) p.logprobs[ri] = -kInf;
        }
        return;
    }
    r.set(top, ask.temp, shift);
    float lowest, unused;
    r.bounds(0, kBins, lowest, unused);

    // as many tokens as are asked for are no lower than `bound`: every thread's
    // highest, counted by steps, tells (for top-p a guess, made good below)
    float bound = lowest;
    if (ask.by_k || ask.by_p) {
        const int b = r.bin(r.fall(own_top));
        if (b < kBins) atomicAdd(&lds.count[b], 1u);
        if (t == 0) {
            lds.bin = kBins;
            lds.crowded = 0;
            lds.all_above = 0;
        }
        __syncthreads();
        const uint64_t n = lds.count[t], enough = ask.by_k ? (uint64_t)ask.k : 64;
        lds.count[t] = 0;
        uint64_t all;
        const uint64_t before = block_scan(n, lds.wsum[0], all);
        if (before < enough && before + n >= enough) lds.bin = (uint32_t)t;
        __syncthreads();
        if (lds.bin < (uint32_t)kBins) r.bounds((int)lds.bin, (int)lds.bin + 1, bound, unused);
    }

    // the sum of exponentials; where top-p stands alone also an estimate of the
    // weights above the bound and of all, in FP32.  A weight's argument, at most
    // 46.2 powers of two, is rounded three times (difference, rate, product), the
    // exponential to 2^-23 of it, then each of a thread's additions; smaller
    // weights are below 2^-30 of the whole together.  kOff is twice the sum of
    // these (9.7e-6 for 64 tokens a thread)
    constexpr int kTokens = SampleLds<T, true>::kHeld / kST;  // a thread's
    constexpr double kRoundings = 3 * 46.2 * 0.69315 * 0x1p-24 + 0x1p-23 + kTokens * 0x1p-24, kOff = 2e-5;
    static_assert(kOff >= 1.5 * kRoundings, "the border's uncertainty");
    double sum = 0.0;
    const bool alone = ask.by_p && !ask.by_k;
    if (alone) {
        const float rate = (float)r.rate;
        float all = 0.0f, high = 0.0f;
        r.each([&](const float(&x)[V], int) __attribute__((always_inline)) {
            sum += (double)exponentials(r, x);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float q = __builtin_fmaxf(__builtin_amdgcn_exp2f((x[j] - top) * rate), 0.0f);
                all += q;
                high += x[j] >= bound ? q : 0.0f;
            }
        });
        const double d = wave_scan64((double)all), h = wave_scan64((double)high);
        if (lane == 63) {
            lds.guess[0][w] = d;
            lds.guess[1][w] = h;
        }
    } else if (p.logprobs) {
        r.each([&](const float(&x)[V], int) __attribute__((always_inline)) { sum += (double)exponentials(r, x); });
    }
    auto count_in = [&](float v) __attribute__((always_inline)) -> uint64_t {
        const double d = r.fall(v);
        const int b = r.bin(d);
        const uint64_t s = r.weight(d);
        if (b < kBins) {
            atomicAdd(&lds.count[b], 1u);
            if (ask.by_p) atomicAdd(&lds.mass[b], (unsigned long long)s);
        }
        return s;
    };
    auto steps = [&](float from) __attribute__((always_inline)) {
        r.each([&](const float(&x)[V], int) __attribute__((always_inline)) {
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (x[j] >= from) count_in(x[j]);
        });
    };
    // the tokens above the bound, a thread each: few lie among many, so the
    // waves gather theirs before anything is formed from them.  False if one
    // met more than it has lanes
    Ranked own = {0.0f, -1, 0};
    auto gather = [&]() __attribute__((always_inline)) {
        int n = 0;  // the wave's
        r.each([&](const float(&x)[V], int at) __attribute__((always_inline)) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const uint64_t who = __ballot(x[j] >= bound);
                if (who == 0) continue;
                const int i = n + (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0u));
                if (x[j] >= bound && i < 64) {
                    lds.some[64 * w + i] = x[j];
                    lds.some_at[64 * w + i] = at + j;
                }
                n += __builtin_popcountll(who);
            }
        });
        n = __builtin_amdgcn_readfirstlane(n);
        if (n > 64 && lane == 0) lds.crowded = 1;
        __syncthreads();
        if (lds.crowded) return false;
        if (lane < n) {
            own.x = lds.some[t];
            own.at = lds.some_at[t];
            own.w = count_in(own.x);
        }
        return true;
    };
    sum = wave_scan64(sum);
    if (lane == 63) lds.wexp[w] = sum;
    __syncthreads();
    // (the thread that writes a result finishes it)
    auto log_sum = [&]() __attribute__((always_inline)) {
        double s = 0.0;
#pragma unroll
        for (int i = 0; i < kWaves; ++i) s += lds.wexp[i];
        return log(s);
    };
    if (ask.greedy) {
        if (t == 0) {
            p.tokens[ri] = arg;
            if (p.logprobs) p.logprobs[ri] = (float)-log_sum();
        }
        return;
    }

    Keep keep;
    bool listed = false;    // what is kept is among the threads' own
    bool gathered = false;  // or among lds.some
    if (ask.by_k || ask.by_p) {
        double all = 0.0, high = 0.0;
        if (alone)
#pragma unroll
            for (int i = 0; i < kWaves; ++i) {
                all += lds.guess[0][i];
                high += lds.guess[1][i];
            }
        // Top-p alone: if the estimates place its border above the bound, from
        // the tokens there, and it holds if the goal's whole uncertainty lies
        // inside the border's token.  Else from all tokens
        for (int turn = 0; turn < 2; ++turn) {
            const bool guess = alone && turn == 0;
            listed = bound > lowest && (alone ? guess && !r.endless && high > (double)ask.top_p * all * (1.0 + 4.0 * kOff) : true) &&
                     gather();
            if (!listed) {
                if (guess) continue;
                own.at = -1;
                if (alone) {
                    __syncthreads();
                    lds.count[t] = 0;
                    lds.mass[t] = 0;
                    __syncthreads();
                }
                steps(alone ? lowest : bound);
            }
            __syncthreads();
            const uint64_t count = lds.count[t], mass = lds.mass[t];
            uint64_t n_all, m_all;
            const uint64_t m_before = block_scan(mass, lds.wsum[0], m_all), n_before = block_scan(count, lds.wsum[1], n_all);
            const double whole = __builtin_ldexp(all, shift);
            const uint64_t kept = borders(r, lds, ask, count, mass, n_before, m_before, n_all,
                                          guess ? (uint64_t)(whole * (1.0 - kOff)) : m_all, listed, own, keep);
            gathered = !listed && lds.all_above && lds.n_some <= (uint32_t)SampleLds<T, true>::kSome;
            if (!guess || (double)ask.top_p * whole * (1.0 + kOff) <= (double)kept) break;
            keep = Keep();
        }
    } else if (ask.first_only) {
        keep.edge = top;
        keep.edge_at = arg;
    }
    keep.finish(r, ask, lowest);

    // the kept weights by pieces of 64 V tokens
    const int cells = (r.n + 64 * V - 1) / (64 * V);
    __syncthreads();
    if (listed || gathered) {
        for (int c = t; c < cells; c += kST) lds.cell[c] = 0;
        __syncthreads();
        auto add = [&](int at, uint64_t s) __attribute__((always_inline)) {
            if ((double)s >= keep.least)
                atomicAdd(reinterpret_cast<unsigned long long *>(&lds.cell[at / (64 * V)]), (unsigned long long)s);
        };
        if (listed) {
            if (own.at >= 0 && keep.has(own.x, own.at)) add(own.at, own.w);
        } else {
            for (uint32_t i = t; i < lds.n_some; i += kST)
                if (keep.has(lds.some[i], lds.some_at[i])) add(lds.some_at[i], r.weight(r.fall(lds.some[i])));
        }
    } else {
        for (int c = w; c < cells; c += kWaves) {
            const uint64_t s = keep.piece(r, c, lane);
            if (lane == 63) lds.cell[c] = s;
        }
    }
    __syncthreads();
    const int token = drawn(r, lds, keep, ask.u);
    if (token >= 0) {
        p.tokens[ri] = token;
        if (p.logprobs) p.logprobs[ri] = (float)(-r.fall(T::get(r.row[token])) - log_sum());
    }
}

// Longer rows, a row's slices by workgroups of their own: the highest logit;
// sums and the steps' counts and weights; the borders (a workgroup a row, which
// reads the row once for each); the kept weights of the pieces; the token.  8 rows
// of 131072 BF16 logits, top-p 0.9: 37 us (top-k 50: 32, neither: 21); one
// workgroup a row for all of it took twice the slices' time when both were built
// alike (305 against 163 us).
constexpr int kSlices = 32;
struct WideRow {
    float top[kSlices];
    int arg[kSlices];
    double sum[kSlices];
    unsigned long long mass[kBins];
    uint32_t count[kBins];
    Keep keep;
    double log_sum;
    int done;
    uint64_t cell[];
};
template <class T>
__host__ __device__ constexpr size_t wide_bytes(uint32_t vocab) {
    return (sizeof(WideRow) + (vocab + 64 * T::kVec - 1) / (64 * T::kVec) * sizeof(uint64_t) + 15) / 16 * 16;
}
template <class T>
__device__ __forceinline__ WideRow &wide_row(void *ws, const GDNSample &p, int r) {
    return *reinterpret_cast<WideRow *>(static_cast<char *>(ws) + (size_t)r * wide_bytes<T>(p.vocab));
}
// The tokens of slice i of n: whole pieces.
template <class T>
__device__ __forceinline__ void slice_of(const GDNSample &p, int i, int n, int &c0, int &c1) {
    const int cells = ((int)p.vocab + 64 * T::kVec - 1) / (64 * T::kVec);
    c0 = (int)((int64_t)cells * i / n);
    c1 = (int)((int64_t)cells * (i + 1) / n);
}
template <class T>
__device__ __forceinline__ void wide_set(Row<T, false> &r, const GDNSample &p, int ri, int shift, const WideRow &row,
                                         int slices, float temp, int &arg) {
    const int lane = threadIdx.x & 63;
    float top = lane < slices ? row.top[lane] : -kInf;
    arg = lane < slices ? row.arg[lane] : kNowhere;
    first_of_highest(top, arg);
    r.row = static_cast<const typename T::E *>(p.logits) + (size_t)ri * p.logits_stride;
    r.n = (int)p.vocab;
    r.set(top, temp, shift);
}

// f(values, index of the first) over the tokens of pieces c0 .. c1 - 1
template <class R, class F>
__device__ __forceinline__ void each_in(const R &r, int c0, int c1, F &&f) {
    const int end = min(c1 * 64 * R::V, r.n);
    for (int at = (c0 * 64 + (int)threadIdx.x) * R::V; at < end; at += kST * R::V) {
        float x[R::V];
        r.load(at, x);
        f(x, at);
    }
}

template <class T>
__global__ __launch_bounds__(kST) void k_wide_top(GDNSample p, void *ws) {
    __shared__ float wmax[kWaves];
    __shared__ int warg[kWaves];
    const int ri = blockIdx.y, t = threadIdx.x, lane = t & 63, w = t >> 6;
    WideRow &row = wide_row<T>(ws, p, ri);
    Row<T, false> r;
    r.row = static_cast<const typename T::E *>(p.logits) + (size_t)ri * p.logits_stride;
    r.n = (int)p.vocab;
    int c0, c1;
    slice_of<T>(p, blockIdx.x, gridDim.x, c0, c1);
    float top = -kInf;
    int arg = kNowhere;
    each_in(r, c0, c1, [&](const float(&x)[T::kVec], int at) __attribute__((always_inline)) { higher<T>(x, at, top, arg); });
    for (int i = blockIdx.x * kST + t; i < kBins; i += gridDim.x * kST) {
        row.mass[i] = 0;
        row.count[i] = 0;
    }
    first_of_highest(top, arg);
    if (lane == 0) {
        wmax[w] = top;
        warg[w] = arg;
    }
    __syncthreads();
    top = lane < kWaves ? wmax[lane] : -kInf;
    arg = lane < kWaves ? warg[lane] : kNowhere;
    first_of_highest(top, arg);
    if (t == 0) {
        row.top[blockIdx.x] = top;
        row.arg[blockIdx.x] = arg;
    }
}

template <class T>
__global__ __launch_bounds__(kST) void k_wide_steps(GDNSample p, int shift, void *ws) {
    constexpr int V = T::kVec;
    __shared__ unsigned long long mass[kBins];
    __shared__ uint32_t count[kBins];
    __shared__ double wexp[kWaves];
    const int ri = blockIdx.y, t = threadIdx.x, lane = t & 63, w = t >> 6;
    WideRow &row = wide_row<T>(ws, p, ri);
    const Ask ask(p, ri);
    Row<T, false> r;
    int arg;
    wide_set(r, p, ri, shift, row, gridDim.x, ask.temp, arg);
    if (arg == kNowhere) return;
    count[t] = 0;
    mass[t] = 0;
    __syncthreads();
    int c0, c1;
    slice_of<T>(p, blockIdx.x, gridDim.x, c0, c1);
    double sum = 0.0;
    each_in(r, c0, c1, [&](const float(&x)[V], int) __attribute__((always_inline)) {
        sum += (double)exponentials(r, x);
        if (ask.by_k || ask.by_p) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const double d = r.fall(x[j]);
                const int b = r.bin(d);
                if (b < kBins) {
                    atomicAdd(&count[b], 1u);
                    if (ask.by_p) atomicAdd(&mass[b], (unsigned long long)r.weight(d));
                }
            }
        }
    });
    sum = wave_scan64(sum);
    if (lane == 63) wexp[w] = sum;
    __syncthreads();
    if (count[t]) atomicAdd(&row.count[t], count[t]);
    if (mass[t]) atomicAdd(&row.mass[t], mass[t]);
    if (t == 0) {
        double s = 0.0;
#pragma unroll
        for (int i = 0; i < kWaves; ++i) s += wexp[i];
        row.sum[blockIdx.x] = s;
    }
}

template <class T>
__global__ __launch_bounds__(kST) void k_wide_border(GDNSample p, int shift, void *ws, int slices) {
    __shared__ SampleLds<T, false> lds;
    const int ri = blockIdx.x, t = threadIdx.x;
    WideRow &row = wide_row<T>(ws, p, ri);
    const Ask ask(p, ri);
    Row<T, false> r;
    int arg;
    wide_set(r, p, ri, shift, row, slices, ask.temp, arg);
    const bool none = arg == kNowhere;
    const int lane = t & 63;
    const uint64_t sums = __builtin_bit_cast(uint64_t, wave_scan64(lane < slices && !none ? row.sum[lane] : 0.0));
    const double log_sum = log(__builtin_bit_cast(double, lane_of(sums, 63)));
    if (t == 0) {
        row.log_sum = log_sum;
        row.done = none || ask.greedy;
    }
    if (none || ask.greedy) {  // nothing above -infinity, or the highest
        if (t == 0) {
            p.tokens[ri] = none ? -1 : arg;
            if (p.logprobs) p.logprobs[ri] = none ? -kInf : (float)-log_sum;
        }
        return;
    }
    float lowest, unused;
    r.bounds(0, kBins, lowest, unused);
    Keep keep;
    if (ask.by_k || ask.by_p) {
        const uint64_t count = row.count[t], mass = row.mass[t];
        uint64_t n_all, m_all;
        const uint64_t n_before = block_scan(count, lds.wsum[0], n_all), m_before = block_scan(mass, lds.wsum[1], m_all);
        borders(r, lds, ask, count, mass, n_before, m_before, n_all, m_all, false, Ranked{0.0f, -1, 0}, keep);
    } else if (ask.first_only) {
        keep.edge = r.top;
        keep.edge_at = arg;
    }
    keep.finish(r, ask, lowest);
    if (t == 0) row.keep = keep;
}

template <class T>
__global__ __launch_bounds__(kST) void k_wide_pieces(GDNSample p, int shift, void *ws) {
    const int ri = blockIdx.y, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    WideRow &row = wide_row<T>(ws, p, ri);
    if (row.done) return;
    const Ask ask(p, ri);
    Row<T, false> r;
    int arg, c0, c1;
    wide_set(r, p, ri, shift, row, gridDim.x, ask.temp, arg);
    const Keep keep = row.keep;
    slice_of<T>(p, blockIdx.x, gridDim.x, c0, c1);
    for (int c = c0 + w; c < c1; c += kWaves) {
        const uint64_t s = keep.piece(r, c, lane);
        if (lane == 63) row.cell[c] = s;
    }
}

template <class T>
__global__ __launch_bounds__(kST) void k_wide_draw(GDNSample p, int shift, void *ws, int slices) {
    __shared__ SampleLds<T, false> lds;
    const int ri = blockIdx.x, t = threadIdx.x;
    WideRow &row = wide_row<T>(ws, p, ri);
    if (row.done) return;
    const Ask ask(p, ri);
    Row<T, false> r;
    int arg;
    wide_set(r, p, ri, shift, row, slices, ask.temp, arg);
    const Keep keep = row.keep;
    const int cells = (r.n + 64 * T::kVec - 1) / (64 * T::kVec);
    for (int c = t; c < cells; c += kST) lds.cell[c] = row.cell[c];
    __syncthreads();
    const int token = drawn(r, lds, keep, ask.u);
    if (token >= 0) {
        p.tokens[ri] = token;
        if (p.logprobs) p.logprobs[ri] = (float)(-r.fall(T::get(r.row[token])) - row.log_sum);
    }
}

bool misaligned(const void *p, int32_t dtype) {
    return (reinterpret_cast<uintptr_t>(p) & (dtype == GDN_DTYPE_FP32 ? 3 : 1)) != 0;
}

}  // namespace lg
}  // namespace gdn

extern "C" int gdn_logits_process(const GDNLogits *args, void *stream) {
    using namespace gdn::lg;
    using gdn::refuse;
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
    // (the kernel's steps past an end stay in 32 bits)
    if (a.history_width > (1u << 30) || a.n_bias > (1u << 30) || a.n_masks > (1u << 30))
        return refuse(who, "a width or count is larger than 2^30");
    if (a.mask && a.mask_stride < (int64_t)((a.vocab + 31) / 32)) return refuse(who, "mask rows are shorter than the vocabulary");
    if (a.mask && !a.mask_index && a.n_masks < a.rows) return refuse(who, "fewer masks than rows, and no mask_index");
    const int64_t size = a.dtype == GDN_DTYPE_FP32 ? 4 : 2;
    if (!(a.logits == a.out && (a.rows == 1 || a.logits_stride == a.out_stride)) &&
        gdn::rows_overlap(a.logits, a.vocab * size, a.logits_stride * size, a.out, a.vocab * size, a.out_stride * size, a.rows))
        return refuse(who, "out overlaps logits, and is not the same rows");
    const dim3 grid((a.vocab + kTile - 1) / kTile, a.rows);
    const size_t lds = sizeof(uint32_t) * kTile * ((a.history != nullptr) + (a.bias_offsets != nullptr));
    hipStream_t s = static_cast<hipStream_t>(stream);
    const auto kernel = a.dtype == GDN_DTYPE_BF16 ? k_process<Bf16> : a.dtype == GDN_DTYPE_FP16 ? k_process<Fp16> : k_process<Fp32>;
    return gdn::launched(who, gdn::launch(kernel, grid, dim3(kPT), lds, s, a));
}

namespace gdn {
namespace lg {
template <class T>
bool held(const GDNSample &a) {
    return a.vocab <= (uint32_t)SampleLds<T, true>::kHeld;
}
template <class T>
hipError_t launch_sample(const GDNSample &a, void *ws, hipStream_t s) {
    // 2^shift times the vocabulary is at most 2^63
    const int shift = a.vocab <= (1u << 18) ? 45 : 43;
    const dim3 rows(a.rows), block(kST);
    if (held<T>(a)) return launch(k_sample<T>, rows, block, 0, s, a, shift);
    // slices for two workgroups a CU (131072 tokens, against one and four: 32 rows
    // 47.6, 47.4 and 54.9 us, 128 rows 87.6, 90.6 and 90.0)
    const int slices = a.rows >= 512 ? 1 : a.rows * kSlices <= 512 ? kSlices : 512 / (int)a.rows;
    const dim3 parts(slices, a.rows);
    hipError_t rc = launch(k_wide_top<T>, parts, block, 0, s, a, ws);
    if (rc == hipSuccess) rc = launch(k_wide_steps<T>, parts, block, 0, s, a, shift, ws);
    if (rc == hipSuccess) rc = launch(k_wide_border<T>, rows, block, 0, s, a, shift, ws, slices);
    if (rc == hipSuccess) rc = launch(k_wide_pieces<T>, parts, block, 0, s, a, shift, ws);
    if (rc == hipSuccess) rc = launch(k_wide_draw<T>, rows, block, 0, s, a, shift, ws, slices);
    return rc;
}
}  // namespace lg
}  // namespace gdn

extern "C" size_t gdn_sample_workspace(const GDNSample *args) {
    using namespace gdn::lg;
    if (args == nullptr || args->vocab > (uint32_t)kMostVocab) return 0;
    const GDNSample &a = *args;
    if (a.dtype == GDN_DTYPE_BF16) return held<Bf16>(a) ? 0 : a.rows * wide_bytes<Bf16>(a.vocab);
    if (a.dtype == GDN_DTYPE_FP16) return held<Fp16>(a) ? 0 : a.rows * wide_bytes<Fp16>(a.vocab);
    if (a.dtype == GDN_DTYPE_FP32) return held<Fp32>(a) ? 0 : a.rows * wide_bytes<Fp32>(a.vocab);
    return 0;
}

extern "C" int gdn_sample_tokens(const GDNSample *args, void *workspace, size_t workspace_bytes, void *stream) {
    using namespace gdn::lg;
    using gdn::refuse;
    constexpr const char *who = "gdn_sample_tokens";
    if (args == nullptr) return refuse(who, "args is NULL");
    const GDNSample &a = *args;
    if (a.dtype < GDN_DTYPE_BF16 || a.dtype > GDN_DTYPE_FP32) return refuse(who, "unknown dtype");
    if (a.vocab > (uint32_t)kMostVocab) return refuse(who, "the vocabulary is larger than 2^20");
    if (a.rows > 65535) return refuse(who, "at most 65535 rows");
    if (a.rows == 0) return 0;
    if (a.vocab == 0) return refuse(who, "the vocabulary is empty");
    if (!a.logits || !a.tokens || (a.temperature && !a.uniform)) return refuse(who, "a buffer pointer is NULL");
    if (misaligned(a.logits, a.dtype)) return refuse(who, "logits is misaligned");
    if (a.rows > 1 && a.logits_stride < (int64_t)a.vocab) return refuse(who, "the row stride is smaller than the row");
    const size_t need = gdn_sample_workspace(args);
    if (need != 0 && (workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 15) != 0 || workspace_bytes < need))
        return refuse(who, "the workspace is missing, misaligned or too small");
    hipStream_t s = static_cast<hipStream_t>(stream);
    return gdn::launched(who, a.dtype == GDN_DTYPE_BF16   ? launch_sample<Bf16>(a, workspace, s)
                              : a.dtype == GDN_DTYPE_FP16 ? launch_sample<Fp16>(a, workspace, s)
                                                          : launch_sample<Fp32>(a, workspace, s));
}
