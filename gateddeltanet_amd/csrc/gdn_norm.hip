// gdn_norm.hip -- gdn_rms_norm: the root-mean-square norm of a batch's rows on the
// caller's device buffers, with the residual's addition, a gate, and an output in
// the rows' type or in 8 bits with scales.
#include <hip/hip_runtime.h>

#include "gdn_amd.h"
#include "gdn_device.h"
#include "gdn_internal.h"
#include "gdn_packed.h"

namespace gdn {
namespace norm {

using namespace packed;

// Eight values at any element's address, `n` of them there (the others zero).
template <class T>
__device__ __forceinline__ void load8(const void *p, size_t at, int n, float (&x)[8]) {
    if (n >= 8) {
        u32x4 w[T::kWords / 4];
        __builtin_memcpy(w, static_cast<const char *>(p) + at * (T::kWords / 2), sizeof(w));
        T::get8(w, x);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = i < n ? T::get(p, at + i) : 0.0f;
    }
}
template <class T>
__device__ __forceinline__ void store8(void *p, size_t at, int n, const float (&x)[8]) {
    if (n >= 8) {
        uint32_t w[T::kWords];
#pragma unroll
        for (int i = 0; i < T::kWords; ++i) {
            if constexpr (T::kWords == 8) w[i] = f2u(x[i]);
            else w[i] = T::pack(x[2 * i], x[2 * i + 1]);
        }
        __builtin_memcpy(static_cast<char *>(p) + at * (T::kWords / 2), w, sizeof(w));
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) T::put(p, at + i, x[i]);
    }
}
// Eight values in E4M3, rounded to nearest even.
__device__ __forceinline__ void store8_fp8(void *p, size_t at, int n, const float (&x)[8]) {
    int w[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        w[i] = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i], x[4 * i + 1], w[i], false);
        w[i] = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i + 2], x[4 * i + 3], w[i], true);
    }
    char *to = static_cast<char *>(p) + at;
    if (n >= 8) {
        __builtin_memcpy(to, w, 8);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) to[i] = (char)(w[i / 4] >> (8 * (i % 4)));
    }
}

// Reduction over groups of n lanes (a power of two, 4 to 64), left in every lane.
template <class Op>
__device__ __forceinline__ uint32_t lanes(uint32_t v, int n, Op op) {
    v = op(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xf, 0xf, false));                // [1,0,3,2]
    v = op(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xf, 0xf, false));                // [2,3,0,1]
    if (n >= 8) v = op(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x141, 0xf, 0xf, false));   // row_half_mirror
    if (n >= 16) v = op(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x140, 0xf, 0xf, false));  // row_mirror
    const int lane = threadIdx.x & 63;
    if (n >= 32) {
        const auto s = __builtin_amdgcn_permlane16_swap((int)v, (int)v, false, false);
        v = op(v, (uint32_t)(((lane >> 4) & 1) ? s[0] : s[1]));
    }
    if (n >= 64) {
        const auto s = __builtin_amdgcn_permlane32_swap((int)v, (int)v, false, false);
        v = op(v, (uint32_t)((lane >> 5) ? s[0] : s[1]));
    }
    return v;
}
__device__ __forceinline__ float lanes_sum(float v, int n) {
    return u2f(lanes(f2u(v), n, [](uint32_t a, uint32_t b) { return f2u(u2f(a) + u2f(b)); }));
}
// of magnitudes as bits, in which NaN is above infinity
__device__ __forceinline__ uint32_t lanes_max(uint32_t v, int n) {
    return lanes(v, n, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
}
// (0 of no values: behind a row's heads there is no root, with an eps of 0 a NaN)
__device__ __forceinline__ uint32_t largest(const float (&y)[8], int n) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, f2u(y[i]) & 0x7fffffffu);
    return n > 0 ? m : 0;
}
// 1 for a block whose largest magnitude is too small to be divided by
__device__ __forceinline__ float scale_of(uint32_t magnitude) {
    const float m = u2f(magnitude);
    return m < 0x1p-100f ? 1.0f : m / 448.0f;
}
// y / scale: the product with the reciprocal, corrected by what it leaves of y, so that a
// quotient that FP32 holds, as one halfway between two E4M3 values, is exact, and others
// are a division's but within 2^-23 of a step of halfway between two FP32 values.  (4096
// x 8192 BF16 with a residual 42.8 us, with divisions 47.)  Of an infinite scale 0, or NaN
// of an infinity.
struct Quotient {
    float inv, by;
    __device__ __forceinline__ explicit Quotient(float scale) : inv(1.0f / scale), by(inv == 0.0f ? 0.0f : scale) {}
    __device__ __forceinline__ float operator()(float y) const {
        const float q = y * inv;
        return __builtin_fmaf(__builtin_fmaf(-q, by, y), inv, q);
    }
};

// u (and h) of eight values at `at` of row `row`; s(gate) where it comes behind.
template <class T>
__device__ __forceinline__ void inputs(const GDNNorm &p, size_t row, int at, int n, float (&h)[8], float (&u)[8], float (&g)[8]) {
    load8<T>(p.x, row * p.x_stride + at, n, h);
    if (p.gate) load8<T>(p.gate, row * p.gate_stride + at, n, g);
    if (p.residual) {
        float r[8];
        load8<T>(p.residual, row * p.residual_stride + at, n, r);
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] += r[i];
    }
    if (p.gate) {
#pragma unroll
        for (int i = 0; i < 8; ++i) g[i] = silu_of(g[i]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) u[i] = p.gate && p.gate_first ? h[i] * g[i] : h[i];
}
__device__ __forceinline__ float squares(const float (&u)[8]) {
    float a = 0.0f, b = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        a = __builtin_fmaf(u[i], u[i], a);
        b = __builtin_fmaf(u[i + 1], u[i + 1], b);
    }
    return a + b;
}
__device__ __forceinline__ float root_of(const GDNNorm &p, float sum) {
    return 1.0f / __builtin_sqrtf(sum / (float)p.dim + p.eps);
}
// y in u's place
__device__ __forceinline__ void normed(const GDNNorm &p, float root, int w_at, int n, float (&u)[8], const float (&g)[8]) {
    float w[8];
    if (p.weight) load8<Fp32>(p.weight, w_at, n, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        float y = u[i] * root;
        if (p.weight) y *= w[i];
        if (p.gate && !p.gate_first) y *= g[i];
        u[i] = y;
    }
}

// Units, a head or a row of several, whose values stay in registers: L lanes of V
// vectors of eight a unit.  `head_lanes`: the lanes of each of a unit's heads (a power of
// two; those behind its values idle), 0 where the unit is a head.  Memory-bound, each
// value read and written once: 4096 x 2048 BF16 with a residual into 8 bits, 59 MB, in
// 14.3 us (4.1 TB/s); 64 x 8 heads of 256 with a gate 3.2 us, two memory latencies and a
// reduction.
template <class T, int L, int V, bool kFp8>
__global__ __launch_bounds__((L > kT ? L : kT)) void k_norm(GDNNorm p, int units, int head_lanes) {
    constexpr int W = L > 64 ? L / 64 : 1, LW = L > 64 ? 64 : L;  // waves a unit, lanes of each
    constexpr int kUnits = L > kT ? 1 : kT / L;  // of a workgroup
    __shared__ float sums[W];
    __shared__ uint32_t tops[W];
    const int t = threadIdx.x, l = t % L, w = t >> 6, per_row = head_lanes ? 1 : (int)p.heads, dim = (int)p.dim;
    const int unit = min((int)(blockIdx.x * kUnits) + t / L, units - 1), own_head = unit % per_row;
    const bool own = (int)(blockIdx.x * kUnits) + t / L < units;
    const size_t row = unit / per_row;
    const int turn = head_lanes ? __builtin_ctz(head_lanes) : 0;
    // of vector v: its head, its place in it, its values that there are
    auto head_of = [&](int v) { return head_lanes ? (v * L + l) >> turn : own_head; };
    auto place_of = [&](int v) { return head_lanes ? 8 * (l & (head_lanes - 1)) : 8 * (v * L + l); };
    auto left_of = [&](int v) { return head_of(v) < (int)p.heads ? dim - place_of(v) : 0; };
    float h[V][8], u[V][8], g[V][8], sum[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        inputs<T>(p, row, head_of(v) * dim + place_of(v), left_of(v), h[v], u[v], g[v]);
        sum[v] = squares(u[v]);
    }
    // (at once: 4096 rows of 8192 BF16 values into 8 bits 42.4 us, with the outputs 6 more)
    if (own && p.sum) {
#pragma unroll
        for (int v = 0; v < V; ++v)
            store8<T>(p.sum, row * p.sum_stride + head_of(v) * dim + place_of(v), left_of(v), h[v]);
    }
    if (head_lanes) {
#pragma unroll
        for (int v = 0; v < V; ++v) sum[v] = lanes_sum(sum[v], head_lanes);
    } else {
#pragma unroll
        for (int v = 1; v < V; ++v) sum[0] += sum[v];
        sum[0] = lanes_sum(sum[0], LW);
        if constexpr (W > 1) {
            if ((t & 63) == 0) sums[w] = sum[0];
            __syncthreads();
            sum[0] = 0.0f;
#pragma unroll
            for (int i = 0; i < W; i += 4) sum[0] += (sums[i] + sums[i + 1]) + (sums[i + 2] + sums[i + 3]);
        }
    }
    float root = root_of(p, sum[0]);
    uint32_t top = 0;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int place = place_of(v), at = head_of(v) * dim + place, n = left_of(v);
        if (head_lanes && v > 0) root = root_of(p, sum[v]);
        normed(p, root, p.weight_heads ? at : place, n, u[v], g[v]);
        if constexpr (!kFp8) {
            if (own) store8<T>(p.out, row * p.out_stride + at, n, u[v]);
        }
        if constexpr (kFp8) {
            uint32_t m = largest(u[v], n);
            if (p.block == 0) {
                top = max(top, m);
            } else {
                const float scale = scale_of(lanes_max(m, (int)p.block / 8));
                const Quotient over(scale);
#pragma unroll
                for (int i = 0; i < 8; ++i) u[v][i] = over(u[v][i]);
                if (own && n > 0) {
                    store8_fp8(p.out, row * p.out_stride + at, n, u[v]);
                    if (place % (int)p.block == 0) p.scales[(row * p.heads * dim + at) / p.block] = scale;
                }
            }
        }
    }
    if constexpr (kFp8) {
        if (p.block == 0) {
            top = lanes_max(top, LW);
            if constexpr (W > 1) {
                if ((t & 63) == 0) tops[w] = top;
                __syncthreads();
#pragma unroll
                for (int i = 0; i < W; ++i) top = max(top, tops[i]);
            }
            const float scale = scale_of(top);
            const Quotient over(scale);
#pragma unroll
            for (int v = 0; v < V; ++v) {
#pragma unroll
                for (int i = 0; i < 8; ++i) u[v][i] = over(u[v][i]);
                if (own) store8_fp8(p.out, row * p.out_stride + head_of(v) * dim + place_of(v), left_of(v), u[v]);
            }
            if (own && l == 0) p.scales[row] = scale;
        }
    }
}

// Rows of any length and number of heads, a workgroup each, read again for every
// pass: the squares, the largest magnitude of the row's y where it has one scale,
// the outputs.  Heads of `head_lanes` lanes (a power of two up to 64) side by side, or of
// all 256 in turn.  A value is read and written by one thread throughout.
template <class T, bool kFp8>
__global__ __launch_bounds__(kT) void k_norm_long(GDNNorm p, int head_lanes) {
    __shared__ float sums[2][4];
    __shared__ uint32_t tops[4];
    const int t = threadIdx.x, w = t >> 6, l = t & (head_lanes - 1), own = t / head_lanes, per = kT / head_lanes;
    const int dim = (int)p.dim, heads = (int)p.heads, steps = (dim + 8 * head_lanes - 1) / (8 * head_lanes);
    const size_t row = blockIdx.x;
    float h[8], u[8], g[8];
    int turn = 0;
    auto place_of = [&](int s) { return 8 * (s * head_lanes + l); };
    auto left_of = [&](int head, int s) { return head < heads ? dim - place_of(s) : 0; };
    auto read = [&](int head, int s) { inputs<T>(p, row, head * dim + place_of(s), left_of(head, s), h, u, g); };
    auto root_at = [&](int head) {
        float sum = 0.0f;
        for (int s = 0; s < steps; ++s) {
            read(head, s);
            sum += squares(u);
        }
        sum = lanes_sum(sum, min(head_lanes, 64));
        if (head_lanes > 64) {
            turn ^= 1;  // (a turn's readers are done before the one after next)
            if ((t & 63) == 0) sums[turn][w] = sum;
            __syncthreads();
            sum = (sums[turn][0] + sums[turn][1]) + (sums[turn][2] + sums[turn][3]);
        }
        return root_of(p, sum);
    };
    auto finish = [&](int head, int s, float root) {
        read(head, s);
        normed(p, root, (p.weight_heads ? head * dim : 0) + place_of(s), left_of(head, s), u, g);
    };
    float scale = 1.0f;
    if (kFp8 && p.block == 0) {
        uint32_t top = 0;
        for (int from = 0; from < heads; from += per) {
            const int head = from + own;
            const float root = root_at(head);
            for (int s = 0; s < steps; ++s) {
                finish(head, s, root);
                top = max(top, largest(u, left_of(head, s)));
            }
        }
        top = lanes_max(top, 64);
        if ((t & 63) == 0) tops[w] = top;
        __syncthreads();
        scale = scale_of(max(max(tops[0], tops[1]), max(tops[2], tops[3])));
        if (t == 0) p.scales[row] = scale;
    }
    for (int from = 0; from < heads; from += per) {
        const int head = from + own;
        const float root = root_at(head);
        for (int s = 0; s < steps; ++s) {
            const int place = place_of(s), at = head * dim + place, n = left_of(head, s);
            finish(head, s, root);
            if (p.sum) store8<T>(p.sum, row * p.sum_stride + at, n, h);
            if constexpr (kFp8) {
                if (p.block != 0) {
                    scale = scale_of(lanes_max(largest(u, n), (int)p.block / 8));
                    if (n > 0 && place % (int)p.block == 0) p.scales[(row * heads * dim + at) / p.block] = scale;
                }
                const Quotient over(scale);
#pragma unroll
                for (int i = 0; i < 8; ++i) u[i] = over(u[i]);
                store8_fp8(p.out, row * p.out_stride + at, n, u);
            } else {
                store8<T>(p.out, row * p.out_stride + at, n, u);
            }
        }
    }
}

// ------------------------------------------------------------ host

// A row with one scale for several heads is a unit, each head in lanes of its own (all
// of k_norm_long's above 2048 values), else a head is.  Lanes of a unit, 0: k_norm_long's.
bool joint(const GDNNorm *a) { return a->fp8 && a->block == 0 && a->heads > 1; }
uint64_t units_of(const GDNNorm *a) { return joint(a) ? a->rows : (uint64_t)a->rows * a->heads; }
int head_lanes_of(const GDNNorm *a) {
    int n = 4;
    while (n < 64 && 8u * n < a->dim) n *= 2;
    return a->dim > 2048 ? kT : n;
}
uint64_t length_of(const GDNNorm *a) { return joint(a) ? (uint64_t)a->heads * head_lanes_of(a) * 8 : a->dim; }
int lanes_of(const GDNNorm *a) {
    const uint64_t len = length_of(a);
    if (len > 16384 || (joint(a) && a->dim > 512)) return 0;
    return len <= 64 ? 8 : len <= 128 ? 16 : len <= 256 ? 32 : len <= 512 ? 64 : len <= 8192 ? 256 : a->fp8 ? 512 : 1024;
}

template <class T, int L, int V, bool kFp8>
hipError_t launch_units(const GDNNorm &a, int units, int head_lanes, hipStream_t s) {
    return launch(k_norm<T, L, V, kFp8>, dim3((unsigned)(L > kT ? units : (units + kT / L - 1) / (kT / L))), dim3(L > kT ? L : kT),
                  0, s, a, units, head_lanes);
}
template <class T, bool kFp8>
hipError_t launch_norm(const GDNNorm &a, hipStream_t s) {
    const int units = (int)units_of(&a), head_lanes = joint(&a) ? head_lanes_of(&a) : 0;
    const uint64_t len = length_of(&a);
    switch (lanes_of(&a)) {
        case 8: return launch_units<T, 8, 1, kFp8>(a, units, head_lanes, s);
        case 16: return launch_units<T, 16, 1, kFp8>(a, units, head_lanes, s);
        case 32: return launch_units<T, 32, 1, kFp8>(a, units, head_lanes, s);
        case 64: return launch_units<T, 64, 1, kFp8>(a, units, head_lanes, s);
        // 256 threads a row, not a wave with more vectors: 4096 x 2048 BF16 with a
        // residual 12.6 and 15.0 us, 16384 rows 44.5 and 64, 512 equal.  Above 8192 values
        // more threads: with 256, 512, 1024 of them and in k_norm_long, 4096 x 12288 BF16
        // with a residual take 138, 92, 80 and 99 us, into 8 bits, which holds the values
        // across a second barrier, 135, 90, 102 and 133 (512 now 91, its quotients exact)
        case 256:
            return len <= 2048   ? launch_units<T, 256, 1, kFp8>(a, units, head_lanes, s)
                   : len <= 4096 ? launch_units<T, 256, 2, kFp8>(a, units, head_lanes, s)
                                 : launch_units<T, 256, 4, kFp8>(a, units, head_lanes, s);
        case 512:
        case 1024: return launch_units<T, kFp8 ? 512 : 1024, kFp8 ? 4 : 2, kFp8>(a, units, head_lanes, s);
        default: return launch(k_norm_long<T, kFp8>, dim3(a.rows), dim3(kT), 0, s, a, joint(&a) ? head_lanes_of(&a) : kT);
    }
}
template <class T>
hipError_t launch_out(const GDNNorm &a, hipStream_t s) {
    return a.fp8 ? launch_norm<T, true>(a, s) : launch_norm<T, false>(a, s);
}

}  // namespace norm
}  // namespace gdn

extern "C" int gdn_rms_norm(const GDNNorm *args, void *stream) {
    using namespace gdn::norm;
    using gdn::refuse;
    constexpr const char *who = "gdn_rms_norm";
    const GDNNorm *a = args;
    if (a == nullptr) return refuse(who, "args is NULL");
    if (a->dtype < GDN_DTYPE_BF16 || a->dtype > GDN_DTYPE_FP32) return refuse(who, "unknown dtype");
    const uint64_t len = (uint64_t)a->heads * a->dim;
    if (len == 0 || len > (1u << 20)) return refuse(who, "rows have 1 to 2^20 values");
    // a grid has fewer than 2^32 threads along an axis
    const uint64_t each = lanes_of(a) ? lanes_of(a) : gdn::kT;
    if (units_of(a) >= 0x7fffff00u || units_of(a) * each >= (1ull << 32) - gdn::kT)
        return refuse(who, "too many rows for one launch");
    if (a->fp8 && a->block != 0 && ((a->block != 32 && a->block != 64 && a->block != 128) || a->dim % a->block != 0))
        return refuse(who, "a block is 0, 32, 64 or 128 and divides dim");
    if (!(a->eps >= 0.0f) || a->eps > 3.4e38f) return refuse(who, "eps is a finite number from 0 up");
    if (a->rows == 0) return 0;
    if (!a->x || !a->out || (a->fp8 && !a->scales)) return refuse(who, "a buffer pointer is NULL");
    const uint64_t size = a->dtype == GDN_DTYPE_FP32 ? 4 : 2, width = len * size;
    const uint64_t out_size = a->fp8 ? 1 : size;
    const uintptr_t at = reinterpret_cast<uintptr_t>(a->x) | reinterpret_cast<uintptr_t>(a->residual) |
                         reinterpret_cast<uintptr_t>(a->gate) | reinterpret_cast<uintptr_t>(a->sum);
    if (at % size != 0 || reinterpret_cast<uintptr_t>(a->out) % out_size != 0)
        return refuse(who, "a buffer is not aligned to an element");
    const struct {
        const void *at;
        int64_t stride;
    } in[3] = {{a->x, a->x_stride}, {a->residual, a->residual_stride}, {a->gate, a->gate_stride}},
      to[2] = {{a->out, a->out_stride}, {a->sum, a->sum_stride}};
    auto bad_stride = [&](int64_t s) { return a->rows > 1 && (s < (int64_t)len || s > (int64_t)1 << 40); };
    for (const auto &x : in)
        if (x.at && bad_stride(x.stride)) return refuse(who, "a row stride is smaller than the row, or above 2^40");
    for (const auto &x : to)
        if (x.at && bad_stride(x.stride)) return refuse(who, "a row stride is smaller than the row, or above 2^40");
    for (int o = 0; o < 2; ++o) {
        if (!to[o].at) continue;
        const uint64_t each = o == 0 ? out_size : size;
        for (int i = 0; i < 3; ++i) {
            // in place, but the sum not over the gate
            if (!in[i].at || (each == size && !(o == 1 && i == 2) && to[o].at == in[i].at &&
                              (a->rows == 1 || to[o].stride == in[i].stride)))
                continue;
            if (gdn::rows_overlap(to[o].at, len * each, to[o].stride * (int64_t)each, in[i].at, width,
                                  in[i].stride * (int64_t)size, a->rows))
                return refuse(who, "an output overlaps an input that it is not in the place of");
        }
    }
    if (a->sum && gdn::rows_overlap(a->out, len * out_size, a->out_stride * (int64_t)out_size, a->sum, width,
                                    a->sum_stride * (int64_t)size, a->rows))
        return refuse(who, "out overlaps sum");
    hipStream_t s = static_cast<hipStream_t>(stream);
    return gdn::launched(who, a->dtype == GDN_DTYPE_BF16   ? launch_out<gdn::packed::Bf16>(*a, s)
                              : a->dtype == GDN_DTYPE_FP16 ? launch_out<gdn::packed::Fp16>(*a, s)
                                                           : launch_out<gdn::packed::Fp32>(*a, s));
}
