// gdn_conv.hip -- the short causal convolution over a batch on the caller's
// device buffers: gdn_conv_prefill (packed sequences) and gdn_conv_step (one token
// of every sequence).
#include <hip/hip_runtime.h>

#include "gdn_amd.h"
#include "gdn_device.h"
#include "gdn_internal.h"
#include "gdn_packed.h"

namespace gdn {
namespace conv {

using namespace packed;

// Channels of a thread: sixteen bytes of a row.
template <class T>
constexpr int kVec = T::kTerms == 1 || T::kTerms == 2 ? 8 : 4;

// Sixteen bytes of a row's channels at any element's address, `n` of them the
// row's (the others zero), and back.
template <class T>
struct Vec {
    u32x4 w;
    __device__ __forceinline__ void load(const void *p, size_t at, int n) {
        constexpr int kSize = 16 / kVec<T>;
        const char *from = static_cast<const char *>(p) + at * kSize;
        if (n >= kVec<T>) {
            __builtin_memcpy(&w, from, 16);
        } else {
            w = (u32x4){0u, 0u, 0u, 0u};
#pragma unroll
            for (int i = 0; i < kVec<T>; ++i)
                if (i < n) {
                    if constexpr (kSize == 4) w[i] = reinterpret_cast<const uint32_t *>(from)[i];
                    else w[i / 2] |= (uint32_t) reinterpret_cast<const uint16_t *>(from)[i] << (16 * (i % 2));
                }
        }
    }
    __device__ __forceinline__ void store(void *p, size_t at, int n) const {
        constexpr int kSize = 16 / kVec<T>;
        char *to = static_cast<char *>(p) + at * kSize;
        if (n >= kVec<T>) {
            __builtin_memcpy(to, &w, 16);
        } else {
#pragma unroll
            for (int i = 0; i < kVec<T>; ++i)
                if (i < n) {
                    if constexpr (kSize == 4) reinterpret_cast<uint32_t *>(to)[i] = w[i];
                    else reinterpret_cast<uint16_t *>(to)[i] = (uint16_t)(w[i / 2] >> (16 * (i % 2)));
                }
        }
    }
    __device__ __forceinline__ void get(float (&x)[kVec<T>]) const {
        if constexpr (kVec<T> == 8) {
            T::get8(&w, x);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = u2f(w[i]);
        }
    }
    __device__ __forceinline__ void put(const float (&x)[kVec<T>]) {
        if constexpr (kVec<T> == 4) {
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = f2u(x[i]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = T::pack(x[2 * i], x[2 * i + 1]);
        }
    }
};

// A thread's channels: their taps and bias, and the window's sum.
template <class T, int W>
struct Taps {
    float w[W][kVec<T>], b[kVec<T>];
    __device__ __forceinline__ void load(const GDNConv &p, int ch, int n) {
        float flat[kVec<T> * W];
        if (n >= kVec<T>) {
            __builtin_memcpy(flat, p.weight + (size_t)ch * W, sizeof(flat));
        } else {
#pragma unroll
            for (int i = 0; i < kVec<T> * W; ++i) flat[i] = i < n * W ? p.weight[(size_t)ch * W + i] : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < kVec<T>; ++i) {
#pragma unroll
            for (int j = 0; j < W; ++j) w[j][i] = flat[i * W + j];
            b[i] = p.bias && i < n ? p.bias[ch + i] : 0.0f;
        }
    }
    // of z[0 .. W - 1], oldest first
    template <class Z>
    __device__ __forceinline__ Vec<T> of(const GDNConv &p, Z &&z) const {
        float y[kVec<T>], x[kVec<T>];
#pragma unroll
        for (int i = 0; i < kVec<T>; ++i) y[i] = b[i];
#pragma unroll
        for (int j = 0; j < W; ++j) {
            z(j).get(x);
#pragma unroll
            for (int i = 0; i < kVec<T>; ++i) y[i] = __builtin_fmaf(w[j][i], x[i], y[i]);
        }
        if (p.silu) {
#pragma unroll
            for (int i = 0; i < kVec<T>; ++i) y[i] = silu_of(y[i]);
        }
        Vec<T> out;
        out.put(y);
        return out;
    }
};

// The workgroups are of two kinds, groups of 256 threads' channels each.  The
// first `tiles` tiles of `rows` rows: the tokens with a whole window of their
// sequence's inputs before them, a window that slides down the rows in registers,
// kAhead rows loaded at a time.  Behind them one for each sequence: its first width
// - 1 tokens and its tail, so that whatever reads or writes a slot is one thread,
// and the tails may be updated in place.  Memory-bound: 8111 tokens of 6144 BF16 channels
// in 24 sequences, 201 MB, in 44.5 us (4.5 TB/s); 70 tokens 5.2 us, the lookup, a row's
// loads and the store one behind the other.
constexpr int kAhead = 4;
template <class T, int W>
__global__ __launch_bounds__(kT) void k_conv_prefill(GDNConv p, int groups, int tiles, int rows) {
    constexpr int H = W - 1;
    const int tile = blockIdx.x / groups, ch = ((blockIdx.x % groups) * kT + (int)threadIdx.x) * kVec<T>;
    const int n = (int)p.channels - ch;  // (a wave's other threads go on: they search too)
    Taps<T, W> taps;
    if (tile >= tiles) {
        const int seq = tile - tiles, slot = slot_of(p, seq);
        if (slot < 0 || n <= 0) return;
        const Span sp = span_of(p, seq);
        taps.load(p, ch, n);
        const size_t at = (size_t)slot * H * p.channels + ch;
        Vec<T> z[2 * H], last[H];
#pragma unroll
        for (int j = 0; j < H; ++j) {
            if (p.state_in) z[j].load(p.state_in, at + (size_t)j * p.channels, n);
            else z[j].w = (u32x4){0u, 0u, 0u, 0u};
            z[H + j].w = last[j].w = (u32x4){0u, 0u, 0u, 0u};
            if (j < sp.n) z[H + j].load(p.x, (size_t)(sp.first + j) * p.x_stride + ch, n);
            if (sp.n - H + j >= 0) last[j].load(p.x, (size_t)(sp.first + sp.n - H + j) * p.x_stride + ch, n);
        }
#pragma unroll
        for (int j = 0; j < H; ++j)
            if (j < sp.n)
                taps.of(p, [&](int k) { return z[j + k]; }).store(p.out, (size_t)(sp.first + j) * p.out_stride + ch, n);
        if (p.state_out) {
            // fewer tokens than the tail has rows: the rest is the old tail's
            Vec<T> keep[H];
#pragma unroll
            for (int j = 0; j < H; ++j) {
                keep[j] = last[j];
#pragma unroll
                for (int m = 0; m < H; ++m)
                    if (sp.n == m && j + m < H) keep[j] = z[j + m];
            }
#pragma unroll
            for (int j = 0; j < H; ++j) keep[j].store(p.state_out, at + (size_t)j * p.channels, n);
        }
        return;
    }
    const int end = min((tile + 1) * rows, (int)p.n_tokens);
    if (n > 0) taps.load(p, ch, n);
    for (int r = tile * rows; r < end;) {
        const Found found = find(p, r, [](int first, int) { return first; });
        const int from = found.rows.first, to = min(end, from + found.rows.n);
        if (r >= to) break;  // behind the last sequence
        if (r < from) {      // before the first
            r = min(end, from);
            continue;
        }
        int at = max(r, from + H);
        r = to;
        if (found.slot < 0 || n <= 0 || at >= to) continue;
        Vec<T> z[H + kAhead];
#pragma unroll
        for (int j = 0; j < H; ++j) z[j].load(p.x, (size_t)(at - H + j) * p.x_stride + ch, n);
        for (; at < to; at += kAhead) {
#pragma unroll
            for (int j = 0; j < kAhead; ++j) z[H + j].load(p.x, (size_t)min(at + j, to - 1) * p.x_stride + ch, n);
#pragma unroll
            for (int j = 0; j < kAhead; ++j)
                if (at + j < to)
                    taps.of(p, [&](int k) { return z[j + k]; }).store(p.out, (size_t)(at + j) * p.out_stride + ch, n);
#pragma unroll
            for (int j = 0; j < H; ++j) z[j] = z[kAhead + j];
        }
    }
}

// A token of every sequence: grid (channel groups, sequences).  201 sequences of 4352
// FP32 channels, 27 MB, in 7.7 us (3.5 TB/s); one of 6144 BF16 channels in 3.3, two
// memory latencies.
template <class T, int W>
__global__ __launch_bounds__(kT) void k_conv_step(GDNConv p) {
    constexpr int H = W - 1;
    const int ch = (blockIdx.x * kT + (int)threadIdx.x) * kVec<T>, n = (int)p.channels - ch, seq = blockIdx.y;
    const int slot = slot_of(p, seq);
    if (slot < 0 || n <= 0) return;
    const size_t at = (size_t)slot * H * p.channels + ch;
    Vec<T> z[W];
#pragma unroll
    for (int j = 0; j < H; ++j) {
        if (p.state_in) z[j].load(p.state_in, at + (size_t)j * p.channels, n);
        else z[j].w = (u32x4){0u, 0u, 0u, 0u};
    }
    z[H].load(p.x, (size_t)seq * p.x_stride + ch, n);
    Taps<T, W> taps;
    taps.load(p, ch, n);
    taps.of(p, [&](int k) { return z[k]; }).store(p.out, (size_t)seq * p.out_stride + ch, n);
    if (p.state_out) {
#pragma unroll
        for (int j = 0; j < H; ++j) z[1 + j].store(p.state_out, at + (size_t)j * p.channels, n);
    }
}

// ------------------------------------------------------------ host

int elem_size(const GDNConv *a) { return a->dtype == GDN_DTYPE_FP32 ? 4 : 2; }
int groups_of(const GDNConv *a) {
    const int per = kT * (16 / elem_size(a));
    return (int)((a->channels + per - 1) / per);
}

// What the host can see of a call; 1: nothing to do.
int check(const char *who, const GDNConv *a, bool packed) {
    if (a == nullptr) return refuse(who, "args is NULL");
    if (a->dtype < GDN_DTYPE_BF16 || a->dtype > GDN_DTYPE_FP32) return refuse(who, "unknown dtype");
    if (a->width < 2 || a->width > 4) return refuse(who, "the width is 2, 3 or 4");
    if (a->channels == 0 || a->channels > (1u << 20)) return refuse(who, "1 to 2^20 channels");
    if (a->n_seqs > 65535) return refuse(who, "at most 65535 sequences");
    if (a->n_tokens > 0x7fffff00u) return refuse(who, "at most 2^31 - 256 tokens");
    if (a->n_slots > 0x7fffffffu) return refuse(who, "at most 2^31 - 1 slots");
    if (a->n_seqs == 0) return 1;
    if (!packed && a->n_tokens != a->n_seqs) return refuse(who, "a step has one token a sequence");
    if (!a->slots && a->n_slots < a->n_seqs) return refuse(who, "n_slots is smaller than n_seqs, and there are no slots");
    if ((packed && !a->cu_seqlens) || !a->weight || (a->n_tokens != 0 && (!a->x || !a->out)))
        return refuse(who, "a buffer pointer is NULL");
    const int size = elem_size(a);
    const uintptr_t at = reinterpret_cast<uintptr_t>(a->x) | reinterpret_cast<uintptr_t>(a->out) |
                         reinterpret_cast<uintptr_t>(a->state_in) | reinterpret_cast<uintptr_t>(a->state_out);
    if (at % size != 0) return refuse(who, "x, out or the tails are not aligned to an element");
    constexpr int64_t most = (int64_t)1 << 40;
    if (a->n_tokens > 1 && (a->x_stride < (int64_t)a->channels || a->out_stride < (int64_t)a->channels ||
                            a->x_stride > most || a->out_stride > most))
        return refuse(who, "a row stride is smaller than the row, or above 2^40");
    const uint64_t row = (uint64_t)a->channels * size;
    if (!(a->x == a->out && (a->n_tokens == 1 || a->x_stride == a->out_stride) && !packed) &&
        rows_overlap(a->out, row, a->out_stride * size, a->x, row, a->x_stride * size, a->n_tokens))
        return refuse(who, "out overlaps x");
    if (a->state_in && a->state_out && a->state_in != a->state_out) {
        const uint64_t in = reinterpret_cast<uintptr_t>(a->state_in), out = reinterpret_cast<uintptr_t>(a->state_out);
        if ((in < out ? out - in : in - out) / (row * (a->width - 1)) < a->n_slots)
            return refuse(who, "state_out overlaps a part of state_in");
    }
    return 0;
}

// Rows a tile: two workgroups of tiles a CU before the tiles grow, since each loads
// its taps (128 bytes a thread) and looks its sequence up, and 16 at most.  6144 BF16
// channels, tiles of 4, 8, 16, 32 rows: 1000 tokens 11.5 us with 4, 19.4 with 32; 2000
// 19.5, 16.3; 4000 32.5 with 8, 23.6 with 16; 8111 in 24 sequences 48.3 with 16, 50.5
// with 32 (46.6 with 8 and 41.2 with 32 where the last-level cache holds what the calls
// before wrote).  Stores past the caches: 44.6, but the call that reads the rows next is
// as much slower and more (a copy behind 4000 tokens: 43.5 against 40.0 together).
int rows_of(const GDNConv *a) {
    const uint64_t want = (uint64_t)a->n_tokens * groups_of(a) / 512;
    return want >= 16 ? 16 : want >= 8 ? 8 : 4;
}

template <class T, int W>
hipError_t launch_prefill(const GDNConv &a, hipStream_t s) {
    const int groups = groups_of(&a), rows = rows_of(&a), tiles = (int)(((uint64_t)a.n_tokens + rows - 1) / rows);
    return launch(k_conv_prefill<T, W>, dim3((unsigned)(((uint64_t)tiles + a.n_seqs) * groups)), dim3(kT), 0, s, a, groups,
                  tiles, rows);
}
template <class T, int W>
hipError_t launch_step(const GDNConv &a, hipStream_t s) {
    return launch(k_conv_step<T, W>, dim3((unsigned)groups_of(&a), a.n_seqs), dim3(kT), 0, s, a);
}
template <class T>
hipError_t launch_width(const GDNConv &a, bool packed, hipStream_t s) {
    if (packed)
        return a.width == 4 ? launch_prefill<T, 4>(a, s) : a.width == 3 ? launch_prefill<T, 3>(a, s) : launch_prefill<T, 2>(a, s);
    return a.width == 4 ? launch_step<T, 4>(a, s) : a.width == 3 ? launch_step<T, 3>(a, s) : launch_step<T, 2>(a, s);
}

int run(const char *who, const GDNConv *args, bool packed, void *stream) {
    const int rc = check(who, args, packed);
    if (rc != 0) return rc < 0 ? -1 : 0;
    // a grid has fewer than 2^32 threads along an axis
    if (packed && (((uint64_t)args->n_tokens + rows_of(args) - 1) / rows_of(args) + args->n_seqs) * groups_of(args) >=
                      (1ull << 32) / kT)
        return refuse(who, "too many rows for one launch");
    hipStream_t s = static_cast<hipStream_t>(stream);
    return launched(who, args->dtype == GDN_DTYPE_BF16   ? launch_width<Bf16>(*args, packed, s)
                         : args->dtype == GDN_DTYPE_FP16 ? launch_width<Fp16>(*args, packed, s)
                                                         : launch_width<Fp32>(*args, packed, s));
}

}  // namespace conv
}  // namespace gdn

extern "C" int gdn_conv_prefill(const GDNConv *args, void *stream) {
    return gdn::conv::run("gdn_conv_prefill", args, true, stream);
}

extern "C" int gdn_conv_step(const GDNConv *args, void *stream) {
    return gdn::conv::run("gdn_conv_step", args, false, stream);
}
