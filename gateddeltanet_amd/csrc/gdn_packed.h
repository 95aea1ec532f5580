// gdn_packed.h -- what the operators over packed sequences share (gdn_delta.hip,
// gdn_conv.hip, gdn_scan.hip): input types, their BF16 terms, sequences and slots.
// Not part of the ABI.
#ifndef GDN_PACKED_H
#define GDN_PACKED_H

#include "gdn_device.h"
#include "gdn_wy.h"

namespace gdn {
namespace packed {

// An input type and the BF16 terms its values split into without loss.
struct Bf16 {
    static constexpr int kTerms = 1, kWords = 4;  // words of eight values
    __device__ static void get8(const u32x4 *p, float (&x)[8]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = u2f(p[0][i] << 16);
            x[2 * i + 1] = u2f(p[0][i] & 0xffff0000u);
        }
    }
    __device__ static float get(const void *p, size_t i) { return u2f((uint32_t) static_cast<const uint16_t *>(p)[i] << 16); }
    __device__ static void put(void *p, size_t i, float x) {
        static_cast<uint16_t *>(p)[i] = (uint16_t)cvt_pk(x, 0.0f);
    }
    __device__ static uint32_t pack(float x, float y) { return cvt_pk(x, y); }
};
struct Fp16 {
    static constexpr int kTerms = 2, kWords = 4;
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    __device__ static void get8(const u32x4 *p, float (&x)[8]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const h2 v = __builtin_bit_cast(h2, (uint32_t)p[0][i]);
            x[2 * i] = (float)v.x;
            x[2 * i + 1] = (float)v.y;
        }
    }
    __device__ static float get(const void *p, size_t i) { return (float)static_cast<const _Float16 *>(p)[i]; }
    __device__ static void put(void *p, size_t i, float x) { static_cast<_Float16 *>(p)[i] = (_Float16)x; }
    __device__ static uint32_t pack(float x, float y) { return __builtin_bit_cast(uint32_t, (h2){(_Float16)x, (_Float16)y}); }
};
struct Fp32 {
    static constexpr int kTerms = 3, kWords = 8;
    __device__ static void get8(const u32x4 *p, float (&x)[8]) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = u2f(p[i / 4][i % 4]);
    }
    __device__ static float get(const void *p, size_t i) { return static_cast<const float *>(p)[i]; }
    __device__ static void put(void *p, size_t i, float x) { static_cast<float *>(p)[i] = x; }
};

// Eight consecutive values as raw words.
template <class T>
struct Raw8 {
    u32x4 w[T::kWords / 4];
    __device__ __forceinline__ void load(const void *p, size_t i) {
#pragma unroll
        for (int j = 0; j < T::kWords / 4; ++j)
            w[j] = reinterpret_cast<const u32x4 *>(static_cast<const char *>(p) + i * (T::kWords / 2))[j];
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int j = 0; j < T::kWords / 4; ++j) w[j] = (u32x4){0u, 0u, 0u, 0u};
    }
    // the values' BF16 terms, packed pairs
    __device__ __forceinline__ void terms(u32x4 (&t)[T::kTerms]) const {
        if constexpr (T::kTerms == 1) {
            t[0] = w[0];
        } else {
            float x[8];
            T::get8(w, x);
            u32x2 a[3], b[3];
            split3((f32x4){x[0], x[1], x[2], x[3]}, a);
            split3((f32x4){x[4], x[5], x[6], x[7]}, b);
#pragma unroll
            for (int j = 0; j < T::kTerms; ++j) t[j] = (u32x4){a[j].x, a[j].y, b[j].x, b[j].y};
        }
    }
};

// f(a, b) for the terms a, b of two operands, of NA and NB terms, whose
// products count, smallest first.  Left out are products of 2^-24 of the whole at
// most where both operands' terms are rounded, of 2^-23 where one's first is cut.
template <int NA, int NB, class F>
__device__ __forceinline__ void for_terms(F &&f) {
#pragma unroll
    for (int s = 2; s >= 0; --s)
#pragma unroll
        for (int i = NA - 1; i >= 0; --i)
            if (s - i >= 0 && s - i < NB) f(i, s - i);
}

// Four values of 16-bit columns l % 16: of each 16 lanes, lane l names the
// 8 bytes of row l / 4, columns 4 (l % 4) .. + 3, and gets its column's four rows.
__device__ __forceinline__ u32x2 read_transposed(const u32x2 *lds) {
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s16x4 *Ptr;
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Ptr)(const_cast<u32x2 *>(lds))));
}

// One sequence's rows, its ends held to the rows there are, and its slot (-1:
// left out).  A: a call's arguments (GDNDelta, GDNConv, GDNScan).
struct Span {
    int first, n;
};
template <class A>
__device__ __forceinline__ Span span_of(const A &p, int i) {
    const int end = (int)p.n_tokens;
    const int a = min(max(p.cu_seqlens[i], 0), end), b = min(max(p.cu_seqlens[i + 1], a), end);
    return {a, b - a};
}
template <class A>
__device__ __forceinline__ int slot_of(const A &p, int i) {
    const int s = p.slots ? p.slots[i] : i;
    return s >= 0 && s < (int)p.n_slots ? s : -1;
}
// The last number in 0 .. n - 1 whose key is at most `most`, keys that grow with
// the number (0 where none is): the wave's lanes look at 64 of them at a time, a
// memory latency for 64 numbers and one more for every further factor of 64.
template <class Key>
__device__ __forceinline__ int last_at_most(int n, int most, Key &&key) {
    const int lane = threadIdx.x & 63;
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int step = (hi - lo + 63) / 64, at = lo + step * (lane + 1);
        const bool below = at <= hi && key(at) <= most;
        lo += step * __builtin_popcountll(__ballot(below));
        hi = min(hi, lo + step - 1);
    }
    return __builtin_amdgcn_readfirstlane(lo);
}

// The sequence that last_at_most finds by key(its first row, its number), its rows
// and its slot.  Of up to 64 every lane holds one's, so that they take one memory
// latency and not three in a row.
struct Found {
    int seq, slot;
    Span rows;
};
template <class A, class Key>
__device__ __forceinline__ Found find(const A &p, int most, Key &&key) {
    const int n = (int)p.n_seqs, lane = threadIdx.x & 63;
    Found f;
    if (n <= 64) {
        const int i = min(lane, n - 1), slot = slot_of(p, i);
        const Span sp = span_of(p, i);
        f.seq = max(__builtin_popcountll(__ballot(lane < n && key(sp.first, i) <= most)) - 1, 0);
        f.slot = __builtin_amdgcn_readlane(slot, f.seq);
        f.rows = {__builtin_amdgcn_readlane(sp.first, f.seq), __builtin_amdgcn_readlane(sp.n, f.seq)};
    } else {
        f.seq = last_at_most(n, most, [&](int i) { return key(span_of(p, i).first, i); });
        const Span sp = span_of(p, f.seq);
        f.slot = __builtin_amdgcn_readfirstlane(slot_of(p, f.seq));
        f.rows = {__builtin_amdgcn_readfirstlane(sp.first), __builtin_amdgcn_readfirstlane(sp.n)};
    }
    return f;
}

// The sequence of this rank by size(its rows), the largest first and equal ones in
// turn, where the wave's lanes hold them all; else of this number.
template <class A, class Size>
__device__ __forceinline__ Found ranked(const A &p, int rank, Size &&size) {
    const int n = (int)p.n_seqs, lane = threadIdx.x & 63, i = n <= 64 ? min(lane, n - 1) : rank;
    const int slot = slot_of(p, i);
    const Span sp = span_of(p, i);
    int of = 0;
    if (n <= 64) {
        const int own = size(sp);
        int before = 0;
        for (int j = 0; j < n; ++j) {
            const int other = __builtin_amdgcn_readlane(own, j);
            before += other > own || (other == own && j < lane);
        }
        of = __builtin_ctzll(__ballot(lane < n && before == rank) | (1ull << 63));
    }
    return {n <= 64 ? of : rank, __builtin_amdgcn_readlane(slot, of),
            {__builtin_amdgcn_readlane(sp.first, of), __builtin_amdgcn_readlane(sp.n, of)}};
}

// 2^y, to about 2^-23 of it: the whole powers apart from the rest, which is
// small enough for FP32.
__device__ __forceinline__ float exp2_of(double y) {
    const double n = __builtin_rint(y);
    return __builtin_ldexpf(__builtin_amdgcn_exp2f((float)(y - n)), (int)n);
}

// x / (1 + exp(-x)), to a few 2^-24 of it (0 below -88): the exponential's whole
// powers of two apart from the rest, which is small enough for FP32, with log2(e) in two
// parts for it (Cody and Waite's reduction).
__device__ __forceinline__ float silu_of(float x) {
    const float y = __builtin_amdgcn_fmed3f(-x, -200.0f, 200.0f), n = __builtin_rintf(y * 1.44269504f);
    const float f = __builtin_fmaf(y, 1.925963033e-8f, __builtin_fmaf(y, 1.44269502f, -n));  // log2(e) in two parts
    const float e = __builtin_ldexpf(__builtin_amdgcn_exp2f(f), (int)n);
    return x * __builtin_amdgcn_rcpf(1.0f + e);
}

}  // namespace packed
}  // namespace gdn

#endif
