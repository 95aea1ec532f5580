// gdn_delta.hip -- the gated delta rule over a batch on the caller's device
// buffers: gdn_delta_prefill (packed sequences, chunk-parallel form) and
// gdn_delta_step (one token of every sequence).
#include <hip/hip_runtime.h>

#include <type_traits>
#include <utility>

#include "gdn_amd.h"
#include "gdn_device.h"
#include "gdn_internal.h"
#include "gdn_wy.h"

namespace gdn {
namespace delta {

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
// products count, smallest first; products below 2^-24 of the whole are left
// out.
template <int NA, int NB, class F>
__device__ __forceinline__ void for_terms(F &&f) {
#pragma unroll
    for (int s = 2; s >= 0; --s)
#pragma unroll
        for (int i = NA - 1; i >= 0; --i)
            if (s - i >= 0 && s - i < NB) f(i, s - i);
}

// Tokens of a chunk.
template <class T>
constexpr int kChunk = T::kTerms == 1 ? 64 : 32;

// Four values of 16-bit columns l % 16: of each 16 lanes, lane l names the
// 8 bytes of row l / 4, columns 4 (l % 4) .. + 3, and gets its column's four rows.
__device__ __forceinline__ u32x2 read_transposed(const u32x2 *lds) {
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s16x4 *Ptr;
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Ptr)(const_cast<u32x2 *>(lds))));
}

// Where a 16 x 32 tile (row tile i, column step j) of a chunk's lower
// triangular matrix is kept: tiles above the diagonal are zero and left out.
template <int C>
constexpr int kTriTiles = C == 64 ? 6 : 2;
__device__ __forceinline__ constexpr int tri_tile(int i, int j) { return i < 2 ? i : 2 * i - 2 + j; }

// What k_delta_seq needs of one (chunk, value head).  Matrices as MFMA A
// fragments of the three BF16 terms: lane l carries row 16 i + l % 16 and
// columns 32 j + 4 (l / 16) + {0..3, 16..19}, the tokens that lane holds of a
// 32-token step in the accumulator layout.
//   sc[m]  exp(G_m) |k_m|^-1, beta_m, scale exp(G_m) |q_m|^-1,
//          exp(G_{n-1} - G_m) |k_m|^-1; zeros past the chunk's n tokens
//   dn     exp(G_{n-1})
template <int C>
struct ChunkOps {
    u32x4 tf[kTriTiles<C>][3][64], mf[kTriTiles<C>][3][64];
    f32x4 sc[C];
    f32x4 dn;
};

// k and q of one (chunk, query/key head) as BF16 terms, rows past the chunk's
// end zero: for the types that do not enter the products as they are.
template <class T, int DK>
struct Planes {
    uint16_t k[T::kTerms][kChunk<T>][DK], q[T::kTerms][kChunk<T>][DK];
};

// One sequence's rows.
struct Span {
    int first, n;
};
__device__ __forceinline__ Span span_of(const GDNDelta &p, int i) {
    const int end = (int)p.n_tokens;
    const int a = min(max(p.cu_seqlens[i], 0), end), b = min(max(p.cu_seqlens[i + 1], a), end);
    return {a, b - a};
}
__device__ __forceinline__ int slot_of(const GDNDelta &p, int i) {
    const int s = p.slots ? p.slots[i] : i;
    return s >= 0 && s < (int)p.n_slots ? s : -1;
}
// Chunk c of the sequence that starts at row `first` as number i has place
// first / C + i + c: places grow with (i, c), none is shared, and there are
// at most n_tokens / C + n_seqs, so nothing has to be counted first.
template <int C>
__device__ __forceinline__ int place_of(int first, int i) {
    return first / C + i;
}
// The sequence whose chunk a place is, where starts do not fall.
template <int C>
__device__ __forceinline__ int seq_at(const GDNDelta &p, int place) {
    int lo = 0, hi = (int)p.n_seqs - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (place_of<C>(span_of(p, mid).first, mid) <= place) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// ------------------------------------------------------------ chunk operands

// 2^y, to about 2^-23 of it: the whole powers apart from the rest, which is
// small enough for FP32.
__device__ __forceinline__ float exp2_of(double y) {
    const double n = __builtin_rint(y);
    return __builtin_ldexpf(__builtin_amdgcn_exp2f((float)(y - n)), (int)n);
}

// Column `col` of the inverse of a unit lower triangular 16 x 16 block whose
// row r is lane r's `row`: forward substitution, row M's values broadcast
// over its 16 lanes (row_newbcast).
template <int M, int... S>
__device__ __forceinline__ float subst_row(const float (&row)[16], const float (&col)[16], float unit,
                                           std::integer_sequence<int, S...>) {
    float acc[2] = {unit, 0.0f};
    ((acc[S & 1] = __builtin_fmaf(
          -__builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, row[S]), 0x150 + M, 0xf, 0xf, true)),
          col[S], acc[S & 1])),
     ...);
    return acc[0] + acc[1];
}
template <int... M>
__device__ __forceinline__ void subst(const float (&row)[16], int li, float (&col)[16], std::integer_sequence<int, M...>) {
    ((col[M] = subst_row<M>(row, col, li == M ? 1.0f : 0.0f, std::make_integer_sequence<int, M>())), ...);
}

// The matrices of one (chunk, value head): grid (places + 1, value heads), a
// wave for every 16 tokens.  With G the cumulative log decay inside the chunk
// and k, q normalised:
//   L[m][s] = beta_m exp(G_m - G_s) (k_m . k_s), s < m;  T = (I + L)^-1
//   M[m][s] = scale exp(G_m - G_s) (q_m . k_s), s <= m
// G is summed in 64 bits: the weights are exponentials of its differences.
// Wave w forms the products of k's 16-token tile w and of q's tile NW - 1 - w
// with the tiles before them, five each of four waves' twenty.  T by 16 x 16
// blocks: the diagonal ones by substitution, all in wave 0 (a lane a column)
// while the others write M; then T_21 = -T_22 L_21 T_11 for the 32 x 32 blocks'
// and for the whole's halves on FP32 MFMAs.
// The last place's workgroup orders the sequences for k_delta_seq, longest
// first, by counting their chunks in 256 steps, and tells it behind them whether
// a start falls: then places may be shared, and a sequence's searched in vain.
// Bound by latency: loads, the products, 16 steps of substitution, four stages
// of the inverse.  BF16, 8 heads of 256: 10.1 us for 70 tokens, 18.9 for 4096 (36
// MB, 1.9 TB/s), 32.6 for 8111 in 24 sequences; FP32, 2005 tokens, 8 heads of 128:
// 15.7 us.
template <class T, int DK>
__global__ __launch_bounds__(4 * kChunk<T>) void k_delta_prep(GDNDelta p, int *__restrict__ order,
                                                              ChunkOps<kChunk<T>> *__restrict__ ops_all,
                                                              Planes<T, DK> *__restrict__ planes) {
    constexpr int C = kChunk<T>, NW = C / 16, NT = T::kTerms, KS = DK / 32, LD = C + 4;
    struct Mats {
        float t[C][LD], m[C][LD];
    };
    __shared__ __attribute__((aligned(16))) union {
        u32x4 kb[NW][KS][NT][64];
        Mats mat;  // once the products are formed
        uint32_t bucket[256];
    } mem;
    __shared__ __attribute__((aligned(16))) float lm[C][LD];
    __shared__ double glog[C];
    __shared__ float ikn[C], iqn[C], bet[C];
    __shared__ int falls;
    const int t = threadIdx.x, w = __builtin_amdgcn_readfirstlane(t >> 6), lane = t & 63, li = lane & 15, kk = lane >> 4;
    const int place = blockIdx.x, hv = blockIdx.y, hk = hv / (int)(p.n_v_heads / p.n_qk_heads);
    if (place == (int)gridDim.x - 1) {
        if (hv != 0) return;
        for (int i = t; i < 256; i += 64 * NW) mem.bucket[i] = 0;
        if (t == 0) falls = 0;
        __syncthreads();
        auto step = [&](int i) { return 255 - min((span_of(p, i).n + C - 1) / C, 255); };
        for (int i = t; i < (int)p.n_seqs; i += 64 * NW) {
            atomicAdd(&mem.bucket[step(i)], 1u);
            if (i > 0 && span_of(p, i).first < span_of(p, i - 1).first) falls = 1;
        }
        __syncthreads();
        if (t == 0) order[p.n_seqs] = falls;
        if (w == 0) {
            u32x4 &own = *reinterpret_cast<u32x4 *>(&mem.bucket[4 * lane]);
            const u32x4 n = own;
            uint32_t at = n.x + n.y + n.z + n.w;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const uint32_t o = (uint32_t)__shfl_up((int)at, d);
                if (lane >= d) at += o;
            }
            at -= n.x + n.y + n.z + n.w;
            own = (u32x4){at, at + n.x, at + n.x + n.y, at + n.x + n.y + n.z};
        }
        __syncthreads();
        for (int i = t; i < (int)p.n_seqs; i += 64 * NW) order[atomicAdd(&mem.bucket[step(i)], 1u)] = i;
        return;
    }
    const int seq = seq_at<C>(p, place);
    const Span sp = span_of(p, seq);
    const int m0 = (place - place_of<C>(sp.first, seq)) * C;
    if (m0 < 0 || m0 >= sp.n || slot_of(p, seq) < 0) return;
    const int n = min(C, sp.n - m0), row0 = sp.first + m0;
    ChunkOps<C> &ops = ops_all[(size_t)place * p.n_v_heads + hv];

    // the wave's 16 tokens of k and of q, as A and as B fragments the same
    const int wq = NW - 1 - w, km = 16 * w + li, qm = 16 * wq + li;
    Raw8<T> kr[KS], qr[KS];
    float gv, bv;
    {
        // (loads return in order: the gates first)
        const size_t r = (size_t)(row0 + min(t, n - 1)) * p.g_stride + hv;
        gv = p.g[r];
        bv = p.beta[r];
        const size_t rk = (size_t)(row0 + min(km, n - 1)), rq = (size_t)(row0 + min(qm, n - 1));
#pragma unroll
        for (int s = 0; s < KS; ++s) kr[s].load(p.k, rk * p.k_stride + hk * DK + 32 * s + 8 * kk);
#pragma unroll
        for (int s = 0; s < KS; ++s) qr[s].load(p.q, rq * p.q_stride + hk * DK + 32 * s + 8 * kk);
    }
    if (w == 0) {
        // a decay of zero is one too small for FP32, so that differences of G
        // stay numbers; G in powers of two
        gv = gv < -1e5f ? -1e5f : gv;
        const double sum = wave_scan64(t < n ? (double)gv * 1.44269504088896340736 : 0.0);
        if (t < C) {
            glog[t] = sum;
            bet[t] = t < n ? bv : 0.0f;
        }
    }
    u32x4 qa[KS][NT], ka[KS][NT];
    float kn[2] = {0.0f, 0.0f}, qn[2] = {0.0f, 0.0f};
#pragma unroll
    for (int s = 0; s < KS; ++s) {
        if (km >= n) kr[s].zero();
        float x[8];
        T::get8(kr[s].w, x);
#pragma unroll
        for (int e = 0; e < 8; ++e) kn[e & 1] = __builtin_fmaf(x[e], x[e], kn[e & 1]);
        kr[s].terms(ka[s]);
#pragma unroll
        for (int j = 0; j < NT; ++j) mem.kb[w][s][j][lane] = ka[s][j];
    }
#pragma unroll
    for (int s = 0; s < KS; ++s) {
        if (qm >= n) qr[s].zero();
        float x[8];
        T::get8(qr[s].w, x);
#pragma unroll
        for (int e = 0; e < 8; ++e) qn[e & 1] = __builtin_fmaf(x[e], x[e], qn[e & 1]);
        qr[s].terms(qa[s]);
    }
    if constexpr (NT > 1) {
        if (hv % (int)(p.n_v_heads / p.n_qk_heads) == 0) {
            Planes<T, DK> &pl = planes[(size_t)place * p.n_qk_heads + hk];
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    *reinterpret_cast<u32x4 *>(&pl.k[j][km][32 * s + 8 * kk]) = ka[s][j];
                    *reinterpret_cast<u32x4 *>(&pl.q[j][qm][32 * s + 8 * kk]) = qa[s][j];
                }
        }
    }
    auto norm = [&](const float(&x)[2]) __attribute__((always_inline)) {
        float v = x[0] + x[1];
        v += __shfl_xor(v, 16);
        v += __shfl_xor(v, 32);
        return p.l2norm ? 1.0f / __builtin_sqrtf(v + 1e-6f) : 1.0f;
    };
    const float kv = norm(kn), qv = norm(qn);
    if (kk == 0) {
        ikn[km] = kv;
        iqn[qm] = qv;
    }
    __syncthreads();
    if (t < C) {
        const float eg = exp2_of(glog[t]);
        const bool in = t < n;
        ops.sc[t] = (f32x4){in ? eg * ikn[t] : 0.0f, bet[t], in ? p.scale * (eg * iqn[t]) : 0.0f,
                            in ? exp2_of(glog[n - 1] - glog[t]) * ikn[t] : 0.0f};
        if (t == 0) ops.dn = (f32x4){exp2_of(glog[n - 1]), 0.0f, 0.0f, 0.0f};
    }
    // products of the wave's tiles with those before them, then the weights;
    // W: the wave, known where it is compiled
    auto products = [&](auto W) __attribute__((always_inline)) {
        constexpr int kW = decltype(W)::value, kQ = NW - 1 - kW, kMost = kW > kQ ? kW : kQ;
        f32x4 gk[kW + 1], gq[kQ + 1];
#pragma unroll
        for (int c = 0; c <= kW; ++c) gk[c] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int c = 0; c <= kQ; ++c) gq[c] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            u32x4 b[kMost + 1][NT];
#pragma unroll
            for (int c = 0; c <= kMost; ++c)
#pragma unroll
                for (int j = 0; j < NT; ++j) b[c][j] = mem.kb[c][s][j][lane];
            for_terms<NT, NT>([&](int x, int y) __attribute__((always_inline)) {
#pragma unroll
                for (int c = 0; c <= kMost; ++c) {
                    if (c <= kW) gk[c] = mfma_bf16(ka[s][x], b[c][y], gk[c]);
                    if (c <= kQ) gq[c] = mfma_bf16(qa[s][x], b[c][y], gq[c]);
                }
            });
        }
        __syncthreads();  // k's fragments are read; T and M take their place
        double gm[2][4];
        float fk[4], fq[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int mk = 16 * kW + 4 * kk + r, mq = 16 * kQ + 4 * kk + r;
            gm[0][r] = glog[mk];
            gm[1][r] = glog[mq];
            fk[r] = mk < n ? bet[mk] * ikn[mk] : 0.0f;
            fq[r] = mq < n ? p.scale * iqn[mq] : 0.0f;
        }
#pragma unroll
        for (int c = 0; c <= kMost; ++c) {
            const int col = 16 * c + li;
            const double gc = glog[col];
            const float ic = ikn[col];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                if (c <= kW) {
                    const float e = exp2_of(gm[0][r] - gc) * ic;
                    lm[16 * kW + 4 * kk + r][col] = c < kW || li < 4 * kk + r ? (e * fk[r]) * gk[c][r] : 0.0f;
                }
                if (c <= kQ) {
                    const float e = exp2_of(gm[1][r] - gc) * ic;
                    mem.mat.m[16 * kQ + 4 * kk + r][col] = c < kQ || li <= 4 * kk + r ? (e * fq[r]) * gq[c][r] : 0.0f;
                }
            }
        }
        // above the diagonal, the other half of a 32-column step
        if constexpr (kW % 2 == 0) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                mem.mat.t[16 * kW + 4 * kk + r][16 * (kW + 1) + li] = 0.0f;
                mem.mat.m[16 * kW + 4 * kk + r][16 * (kW + 1) + li] = 0.0f;
            }
        }
    };
    if (w == 0) products(std::integral_constant<int, 0>());
    else if (w == 1) products(std::integral_constant<int, 1>());
    if constexpr (NW == 4) {
        if (w == 2) products(std::integral_constant<int, 2>());
        else if (w == 3) products(std::integral_constant<int, 3>());
    }
    __syncthreads();
    float(&tm)[C][LD] = mem.mat.t;
    auto write_terms = [&](const float(&src)[C][LD], u32x4(&dst)[kTriTiles<C>][3][64], int f) __attribute__((always_inline)) {
        const int i = f < 2 ? f : 2 + (f - 2) / 2, j = f < 2 ? 0 : f & 1;
        u32x2 a[3], b[3];
        split3(*reinterpret_cast<const f32x4 *>(&src[16 * i + li][32 * j + 4 * kk]), a);
        split3(*reinterpret_cast<const f32x4 *>(&src[16 * i + li][32 * j + 16 + 4 * kk]), b);
#pragma unroll
        for (int q = 0; q < 3; ++q) dst[f][q][lane] = (u32x4){a[q].x, a[q].y, b[q].x, b[q].y};
    };
    if (w == 0) {
        const int b0 = 16 * (kk < NW ? kk : 0);
        float row[16], tc[16];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const f32x4 v = *reinterpret_cast<const f32x4 *>(&lm[b0 + li][b0 + 4 * q]);
#pragma unroll
            for (int e = 0; e < 4; ++e) row[4 * q + e] = v[e];
        }
        subst(row, li, tc, std::make_integer_sequence<int, 16>());
        if (kk < NW) {
#pragma unroll
            for (int m = 0; m < 16; ++m) tm[b0 + m][b0 + li] = tc[m];
        }
    } else {
        for (int f = w - 1; f < kTriTiles<C>; f += NW - 1) write_terms(mem.mat.m, ops.mf, f);
    }
    __syncthreads();
    // a tile's product A B over 16 columns, A from LDS, B's rows 4 kk + q of
    // column l % 16 in registers (as a product's result lies)
    auto times = [&](const float(&A)[C][LD], int i, int k, const f32x4 b, f32x4 c) __attribute__((always_inline)) {
        const f32x4 a = *reinterpret_cast<const f32x4 *>(&A[16 * i + li][16 * k + 4 * kk]);
#pragma unroll
        for (int q = 0; q < 4; ++q) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[q], b[q], c, 0, 0, 0);
        return c;
    };
    auto tile = [&](int k, int j) __attribute__((always_inline)) {
        f32x4 b;
#pragma unroll
        for (int q = 0; q < 4; ++q) b[q] = tm[16 * k + 4 * kk + q][16 * j + li];
        return b;
    };
    auto put = [&](int i, int j, const f32x4 z) __attribute__((always_inline)) {
#pragma unroll
        for (int r = 0; r < 4; ++r) tm[16 * i + 4 * kk + r][16 * j + li] = -z[r];
    };
    const f32x4 none = {0.0f, 0.0f, 0.0f, 0.0f};
    if (w % 2 == 0) put(w + 1, w, times(tm, w + 1, w + 1, times(lm, w + 1, w, tile(w, w), none), none));
    __syncthreads();
    if constexpr (NW == 4) {
        // wave w: tile (2 + w / 2, w % 2) of the lower left half
        const int j = w % 2;
        const f32x4 b0 = tile(0, 0), b1 = j ? tile(1, 1) : tile(1, 0);
        f32x4 y2 = none, y3 = none, z;
        if (j == 0) y2 = times(lm, 2, 0, b0, none);
        y2 = times(lm, 2, 1, b1, y2);
        if (w < 2) {
            z = times(tm, 2, 2, y2, none);
        } else {
            if (j == 0) y3 = times(lm, 3, 0, b0, none);
            y3 = times(lm, 3, 1, b1, y3);
            z = times(tm, 3, 3, y3, times(tm, 3, 2, y2, none));
        }
        put(2 + w / 2, j, z);
        __syncthreads();
    }
    for (int f = w; f < kTriTiles<C>; f += NW) write_terms(tm, ops.tf, f);
}

// ------------------------------------------------------------ the sequences

// One (sequence, value head)'s chunks in order:
//   d = T (beta (v - exp(G) K S));  o = exp(G) Q S + M d;
//   S' = exp(G_{n-1}) S + K^T (exp(G_{n-1} - G) d)
// A workgroup has CT tiles of 16 value columns, its KP waves a KP-th of the keys
// each.  A wave's state is the accumulator tiles of its updates, and lies
// so that it is also the B operand of its K S and Q S: of a 32-key step, lane l
// holds keys 8 (l / 16) .. + 7 of column l % 16, the first four in one tile, the
// others in the next.  A wave's K and Q go through LDS areas of its own, which
// turn whole lines of memory into A fragments (16-byte units XORed with the
// row's low bits); the update reads K transposed (ds_read_b64_tr_b16).  The KP
// waves' shares of K S and Q S meet in LDS where the wave that owns a 16-token
// tile adds them; it forms b, its rows of d and of o, and leaves the BF16 terms
// of b, d and the scaled d in LDS as the B operands that the tile's waves read.
// Three barriers a chunk; every operand of the next chunk is on its way into
// registers meanwhile, in the order of its use.
// Bound, with few sequences, by a chunk's chain of dependent products: 64 chunks
// of 8 heads of 256 x 256 in 194 us, 3.0 us each, the matrix unit busy for 1536
// of 7200 cycles; with many, by the operands that a head's 16 column tiles read
// through L2 (8111 tokens in 24 sequences: 199 us, 9 TB/s).  FP32, 2005 tokens in
// 5 sequences, 8 heads of 128 x 128: 60 us.  Measured against it at 4096 tokens:
// all keys in one wave 656 us (the products of a tile in a row); two waves and
// 64 columns 432 (registers spill); 32 columns with K and Q shared by eight waves
// 259; fragments read from memory 269; two workgroups a CU by force 415 (spills).
// Two workgroups a CU leave a thread 256 registers: <Bf16, 256, 4, 1> spills 2,
// <Bf16, 64, 2, 1> 6.
// A wave takes 32 keys or more, so KP is 2 for 64 keys, else 4.
template <class T, int DK, int KP, int CT>
struct SeqLds {
    static constexpr int C = kChunk<T>, NT = T::kTerms, MT = C / 16, JT = C / 32, UR = DK / KP / 8;
    // tiles a wave does not own, blocks of b that its area holds
    static constexpr int kFor = KP <= MT ? MT - MT / KP : MT, kB = (3 * CT * JT + KP - 1) / KP;
    // q's area takes the shares for other waves and b once Q S is formed
    union Area {
        u32x4 q[NT][C][UR];
        struct {
            f32x4 part[kFor][CT][2][64];  // [tile][column tile][K S, Q S]
            u32x4 b[kB][64];              // the column tiles' blocks 3 step + term, a KP-th of them
        };
    };
    u32x4 k[KP][NT][C][UR];
    Area area[KP];
    u32x4 df[2][CT][JT][3][64];  // d and the scaled d, B operands: [which][column tile][step][term]
};

// Workgroups that a CU's LDS holds (its registers hold one where two tiles of
// columns meet two of tokens).
template <class T, int DK, int KP, int CT>
constexpr int kSeqPerCu = sizeof(SeqLds<T, DK, KP, CT>) <= (80 << 10) ? 2 : 1;

template <class T, int DK, int KP, int CT>
__global__ __launch_bounds__(64 * KP, (kSeqPerCu<T, DK, KP, CT> == 2 && (CT == 1 || KP == 4 || kChunk<T> == 32)) ? 2 : 1) void k_delta_seq(
    GDNDelta p, const int *__restrict__ order, const ChunkOps<kChunk<T>> *__restrict__ ops_all,
    const Planes<T, DK> *__restrict__ planes, int pairs) {
    using Lds = SeqLds<T, DK, KP, CT>;
    constexpr int C = Lds::C, NT = Lds::NT, MT = Lds::MT, JT = Lds::JT;
    constexpr int KS = DK / 32 / KP;              // 32-key steps of a wave
    constexpr int OT = MT >= KP ? MT / KP : 1;    // token tiles a wave owns (with KP > MT, the first MT waves)
    constexpr int UR = Lds::UR;                   // 16-byte units of a row's keys
    constexpr int kStage = NT * C * UR / 64;      // a lane's units of a chunk's K
    static_assert(KS >= 1 && (UR == 4 || UR == 8) && (KP == 2 || KP == 4), "the layouts below");
    __shared__ Lds lds;
    const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
    const int t = threadIdx.x, ks = __builtin_amdgcn_readfirstlane(t >> 6), lane = t & 63, li = lane & 15, kk = lane >> 4;
    // the column groups of a (sequence, head) share its operands: one XCD's
    // (workgroups go to the eight in turn)
    const int groups = (int)p.value_dim / (16 * CT), x = blockIdx.x >> 3;
    const int pair = (x / groups) * 8 + (blockIdx.x & 7), cg = x % groups;
    if (pair >= pairs) return;
    const int seq = order[pair / (int)p.n_v_heads], hv = pair % (int)p.n_v_heads;
    const int hk = hv / (int)(p.n_v_heads / p.n_qk_heads);
    const int slot = __builtin_amdgcn_readfirstlane(slot_of(p, seq));
    if (slot < 0) return;
    Span sp = span_of(p, seq);
    sp.first = __builtin_amdgcn_readfirstlane(sp.first);
    sp.n = __builtin_amdgcn_readfirstlane(sp.n);
    const int chunks = (sp.n + C - 1) / C, col = 16 * CT * cg + li;
    const size_t place = (size_t)place_of<C>(sp.first, seq);
    // left out unless all its matrices were formed
    if (order[p.n_seqs])
        for (int c = 0; c < chunks; ++c)
            if (seq_at<C>(p, (int)place + c) != seq) return;
    const ChunkOps<C> *ops = ops_all + place * p.n_v_heads + hv;
    // the state's key of tile a, register r of step s: key0 + 32 s + 4 a + r
    const int key0 = ks * (DK / KP) + 8 * kk;
    const size_t state_at = (((size_t)slot * p.n_v_heads + hv) * DK + key0) * p.value_dim + col;

    f32x4 S[CT][KS][2];
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int ct = 0; ct < CT; ++ct)
                    S[ct][s][a][r] =
                        p.state_in ? p.state_in[state_at + (size_t)(32 * s + 4 * a + r) * p.value_dim + 16 * ct] : 0.0f;

    // the token tiles this wave owns; tile i's matrix rows have steps 0 .. i / 2
    const bool owns = KP <= MT || ks < MT;
    auto owner = [&](int i) { return i < KP ? i : MT - 1 - i; };
    auto tile_of = [&](int o) { return o == 0 ? (owns ? ks : 0) : MT - 1 - ks; };
    constexpr int kTri = C == 32 ? 1 : KP == 4 ? 2 : 3;  // their matrix tiles
    // rows at a chunk's uniform address, their offsets in 32 bits
    constexpr uint32_t kSize = T::kWords / 2;
    const uint32_t k_row = (uint32_t)p.k_stride * kSize, q_row = (uint32_t)p.q_stride * kSize,
                   v_row = (uint32_t)p.v_stride * kSize, o_row = (uint32_t)p.o_stride * kSize;
    auto rows_at = [&](const void *x, int64_t stride, int row, int head) __attribute__((always_inline)) {
        return static_cast<const char *>(x) + ((size_t)row * stride + head) * kSize;
    };
    u32x4 kreg[kStage], qreg[kStage], tri[kTri][3];
    f32x4 sc[OT][4];
    float vv[OT][CT][4], dn;
    // rows past the sequence's end: its last one, whose products meet zero
    // factors (the planes hold zeros there)
    auto fetch_rows = [&](int c) __attribute__((always_inline)) {
        const int n = sp.n - C * c;
        if constexpr (NT == 1) {
            const char *kp = rows_at(p.k, p.k_stride, sp.first + C * c, hk * DK),
                       *qp = rows_at(p.q, p.q_stride, sp.first + C * c, hk * DK);
#pragma unroll
            for (int i = 0; i < kStage; ++i) {
                const int row = min((64 * i + lane) / UR, n - 1), at = 2 * ks * (DK / KP) + 16 * (lane % UR);
                kreg[i] = *reinterpret_cast<const u32x4 *>(kp + (__umul24(row, k_row) + at));
                qreg[i] = *reinterpret_cast<const u32x4 *>(qp + (__umul24(row, q_row) + at));
            }
        } else {
            const Planes<T, DK> &pl = planes[(place + c) * p.n_qk_heads + hk];
            const int row = lane / UR, at = ks * (DK / KP) + 8 * (lane % UR);
#pragma unroll
            for (int i = 0; i < kStage; ++i) {
                constexpr int kRows = 64 / UR;
                const int j = i * kRows / C, r = i * kRows % C;
                kreg[i] = *reinterpret_cast<const u32x4 *>(&pl.k[j][r + row][at]);
                qreg[i] = *reinterpret_cast<const u32x4 *>(&pl.q[j][r + row][at]);
            }
        }
    };
    auto fetch_own = [&](int c) __attribute__((always_inline)) {
        const ChunkOps<C> &o = ops[(size_t)c * p.n_v_heads];
        const char *vp = rows_at(p.v, p.v_stride, sp.first + C * c, hv * (int)p.value_dim);
        const int n = sp.n - C * c;
#pragma unroll
        for (int i = 0; i < OT; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int m = 16 * tile_of(i) + 4 * kk + r;
                sc[i][r] = o.sc[m];
#pragma unroll
                for (int ct = 0; ct < CT; ++ct)
                    vv[i][ct][r] = T::get(vp + (__umul24(min(m, n - 1), v_row) + (col + 16 * ct) * kSize), 0);
            }
    };
    auto fetch_tri = [&](const u32x4(&m)[kTriTiles<C>][3][64]) __attribute__((always_inline)) {
#pragma unroll
        for (int q = 0; q < 3; ++q) {
            if constexpr (C == 32) {
                tri[0][q] = m[tile_of(0)][q][lane];
            } else if constexpr (KP == 4) {
                // tile ks: one step or two (else the first's again, unused)
                tri[0][q] = m[tri_tile(ks, 0)][q][lane];
                tri[1][q] = m[tri_tile(ks, ks / 2)][q][lane];
            } else {
                tri[0][q] = m[ks][q][lane];
                tri[1][q] = m[tri_tile(3 - ks, 0)][q][lane];
                tri[2][q] = m[tri_tile(3 - ks, 1)][q][lane];
            }
        }
    };
    // this wave's rows of the matrix in `tri` times the terms in LDS, in a
    // chain for each order of the terms' products
    auto tri_product = [&](const u32x4(&bo)[JT][3], f32x4(&y)[OT]) __attribute__((always_inline)) {
        f32x4 acc[kTri][3];
#pragma unroll
        for (int i = 0; i < kTri; ++i)
#pragma unroll
            for (int q = 0; q < 3; ++q) acc[i][q] = zero;
        for_terms<3, 3>([&](int m, int q) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < kTri; ++i) {
                const int j = kTri == 2 ? i : i == 2;
                acc[i][m + q] = mfma_bf16(tri[i][m], bo[j][q], acc[i][m + q]);
            }
        });
        f32x4 sum[kTri];
#pragma unroll
        for (int i = 0; i < kTri; ++i) sum[i] = (acc[i][2] + acc[i][1]) + acc[i][0];
        y[0] = sum[0];
        if constexpr (kTri == 2) {
            if (ks >= 2) y[0] += sum[1];
        }
        if constexpr (kTri == 3) y[1] = sum[1] + sum[2];
    };
    // the terms of a tile's values, as half a B operand
    auto put_terms = [&](auto &&block, int ct, int tile, const f32x4 v) __attribute__((always_inline)) {
        u32x2 e[3];
        split3(v, e);
#pragma unroll
        for (int q = 0; q < 3; ++q) reinterpret_cast<u32x2 *>(&block(ct, 3 * (tile >> 1) + q)[lane])[tile & 1] = e[q];
    };
    auto b_block = [&](int ct, int i) -> u32x4(&)[64] {
        i += 3 * JT * ct;
        return lds.area[i / Lds::kB].b[i % Lds::kB];
    };
    auto d_block = [&](int ct, int i) -> u32x4(&)[64] { return lds.df[0][ct][i / 3][i % 3]; };
    auto f_block = [&](int ct, int i) -> u32x4(&)[64] { return lds.df[1][ct][i / 3][i % 3]; };
    auto get_operand = [&](auto &&block, int ct, u32x4(&b)[JT][3]) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < JT; ++j)
#pragma unroll
            for (int q = 0; q < 3; ++q) b[j][q] = block(ct, 3 * j + q)[lane];
    };
    // the place in wave a's area of its share of a tile
    auto slot_in = [&](int a, int tile) {
        int n = 0;
#pragma unroll
        for (int i = 0; i < MT; ++i) n += i < tile && owner(i) != a;
        return n;
    };
    u32x4(&kl)[NT][C][UR] = lds.k[ks], (&ql)[NT][C][UR] = lds.area[ks].q;
    auto put_rows = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < kStage; ++i) {
            constexpr int kRows = 64 / UR;
            const int j = i * kRows / C, r = i * kRows % C + lane / UR;
            const int u = (lane % UR) ^ (UR == 8 ? r & 7 : (r >> 1) & 3);
            kl[j][r][u] = kreg[i];
            ql[j][r][u] = qreg[i];
        }
    };
    auto unit = [&](int row, int u) { return u ^ (UR == 8 ? row & 7 : (row >> 1) & 3); };

    if (chunks > 0) {
        fetch_rows(0);
        if (owns) {
            fetch_own(0);
            fetch_tri(ops[0].tf);
        }
        dn = ops[0].dn.x;
        put_rows();
    }
    for (int c = 0; c < chunks; ++c) {
        const int n = min(C, sp.n - C * c), cn = min(c + 1, chunks - 1);  // (the last chunk is fetched again, unused)
        const ChunkOps<C> &next_ops = ops[(size_t)cn * p.n_v_heads];
        fetch_rows(cn);
        // this wave's share of K S and Q S
        f32x4 y[MT][CT][2];
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) y[i][ct][0] = y[i][ct][1] = zero;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            u32x4 sb[CT][3];
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) {
                u32x2 lo[3], hi[3];
                split3(S[ct][s][0], lo);
                split3(S[ct][s][1], hi);
#pragma unroll
                for (int q = 0; q < 3; ++q) sb[ct][q] = (u32x4){lo[q].x, lo[q].y, hi[q].x, hi[q].y};
            }
            u32x4 ka[MT][NT], qa[MT][NT];
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    const int m = 16 * i + li;
                    ka[i][j] = kl[j][m][unit(m, 4 * s + kk)];
                    qa[i][j] = ql[j][m][unit(m, 4 * s + kk)];
                }
            // chains in turn: a product that waits for the one before it takes
            // twice its time
            for_terms<NT, 3>([&](int a, int b) __attribute__((always_inline)) {
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int ct = 0; ct < CT; ++ct) {
                        y[i][ct][0] = mfma_bf16(ka[i][a], sb[ct][b], y[i][ct][0]);
                        y[i][ct][1] = mfma_bf16(qa[i][a], sb[ct][b], y[i][ct][1]);
                    }
            });
        }
        // a load between two products each: issued in a row they hold the wave
        // for 900 cycles
#pragma unroll
        for (int i = 0; i < 2 * kStage; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x008, 2 * CT, 0);
        }
#pragma unroll
        for (int i = 0; i < MT; ++i)
            if (owner(i) != ks) {
                f32x4(&part)[CT][2][64] = lds.area[ks].part[slot_in(ks, i)];
#pragma unroll
                for (int ct = 0; ct < CT; ++ct) {
                    part[ct][0][lane] = y[i][ct][0];
                    part[ct][1][lane] = y[i][ct][1];
                }
            }
        __syncthreads();
        f32x4 qs[OT][CT], sw[OT];
        if (owns) {
            // b, and what stands of o
#pragma unroll
            for (int o = 0; o < OT; ++o) {
                const int tile = tile_of(o);
#pragma unroll
                for (int ct = 0; ct < CT; ++ct) {
                    f32x4 kv = zero, qv = zero;
#pragma unroll
                    for (int i = 0; i < MT; ++i)
                        if (i == tile) {
                            kv = y[i][ct][0];
                            qv = y[i][ct][1];
                        }
#pragma unroll
                    for (int a = 1; a < KP; ++a) {
                        const int from = (ks + a) % KP;
                        const f32x4(&part)[CT][2][64] = lds.area[from].part[slot_in(from, tile)];
                        kv += part[ct][0][lane];
                        qv += part[ct][1][lane];
                    }
                    f32x4 b;
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const f32x4 e = sc[o][r];
                        b[r] = e.y * (vv[o][ct][r] - e.x * kv[r]);
                        qs[o][ct][r] = e.z * qv[r];
                        sw[o][r] = e.w;
                    }
                    put_terms(b_block, ct, tile, b);
                }
            }
            fetch_own(cn);
        }
        __syncthreads();
        if (owns) {
            f32x4 d[CT][OT];
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) {
                u32x4 bo[JT][3];
                get_operand(b_block, ct, bo);
                tri_product(bo, d[ct]);
            }
            fetch_tri(ops[(size_t)c * p.n_v_heads].mf);
#pragma unroll
            for (int ct = 0; ct < CT; ++ct)
#pragma unroll
                for (int o = 0; o < OT; ++o) {
                    put_terms(f_block, ct, tile_of(o), d[ct][o] * sw[o]);
                    put_terms(d_block, ct, tile_of(o), d[ct][o]);
                }
        }
        __syncthreads();
        // the update, and the rows of o
        u32x4 fo[CT][JT][3];
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) get_operand(f_block, ct, fo[ct]);
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            u32x4 a[2][JT][NT];
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int j = 0; j < JT; ++j)
#pragma unroll
                    for (int q = 0; q < NT; ++q) {
                        // this lane's address: token + l % 16 / 4 of each group
                        // of four, keys of group l % 4
                        const int m = 32 * j + 4 * kk + (li >> 2), u = unit(m, 4 * s + (li & 3));
                        const u32x2 lo = read_transposed(reinterpret_cast<const u32x2 *>(&kl[q][m][u]) + h);
                        const u32x2 hi = read_transposed(
                            reinterpret_cast<const u32x2 *>(&kl[q][m + 16][unit(m + 16, 4 * s + (li & 3))]) + h);
                        a[h][j][q] = (u32x4){lo.x, lo.y, hi.x, hi.y};
                    }
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) {
                S[ct][s][0] *= dn;
                S[ct][s][1] *= dn;
            }
            for_terms<NT, 3>([&](int e, int f) __attribute__((always_inline)) {
#pragma unroll
                for (int j = 0; j < JT; ++j)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int ct = 0; ct < CT; ++ct) S[ct][s][h] = mfma_bf16(a[h][j][e], fo[ct][j][f], S[ct][s][h]);
            });
        }
        dn = next_ops.dn.x;
        // (q's area, the shares' and b's until here, is free)
        put_rows();
        if (owns) {
            f32x4 om[CT][OT];
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) {
                u32x4 bo[JT][3];
                get_operand(d_block, ct, bo);
                tri_product(bo, om[ct]);
            }
            fetch_tri(next_ops.tf);
            char *op = const_cast<char *>(rows_at(p.o, p.o_stride, sp.first + C * c, hv * (int)p.value_dim));
            auto put_o = [&](int o, int r) __attribute__((always_inline)) {
                const int m = 16 * tile_of(o) + 4 * kk + r;
#pragma unroll
                for (int ct = 0; ct < CT; ++ct)
                    T::put(op + (__umul24(m, o_row) + (col + 16 * ct) * kSize), 0, qs[o][ct][r] + om[ct][o][r]);
            };
            if (n == C) {
#pragma unroll
                for (int o = 0; o < OT; ++o)
#pragma unroll
                    for (int r = 0; r < 4; ++r) put_o(o, r);
            } else {
#pragma unroll
                for (int o = 0; o < OT; ++o)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (16 * tile_of(o) + 4 * kk + r < n) put_o(o, r);
            }
        }
    }
    if (p.state_out) {
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int a = 0; a < 2; ++a)
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int ct = 0; ct < CT; ++ct)
                        p.state_out[state_at + (size_t)(32 * s + 4 * a + r) * p.value_dim + 16 * ct] = S[ct][s][a][r];
    }
}

// ------------------------------------------------------------ a single token

// A (sequence, value head)'s token for 64 value columns: grid (value_dim / 64,
// value heads, sequences).  The state tile goes through registers once: with
// a = exp(g), the sums S^T k and S^T q are formed from the state as it is read,
//   d = beta (v - a S^T k);  o = scale (a S^T q + (k . q) d);  S' = a S + k d^T
// so its bytes, in and out, are what bounds the kernel: 64 sequences of 8 heads of
// 256 x 256, 268 MB, in 57 us (4.7 TB/s; 41 us where the last-level cache still
// holds part of them), one in 5.7 us, two memory latencies and two reductions.
// 64 columns: whole 256-byte pieces of a row.  16 columns fill more CUs in small
// batches and lose there too (4 heads: 9.5 against 6.3 us at 8 sequences, 14.0
// against 7.7 at 15; 4.9 against 5.1 at one).
constexpr int kStepCols = 64;
template <class T, int DK>
__global__ __launch_bounds__(kT) void k_delta_step(GDNDelta p) {
    constexpr int NC = kStepCols, L = NC / 4, RP = kT / L, NR = (DK + RP - 1) / RP;  // lanes a row, rows a pass, passes
    static_assert(DK % RP == 0, "whole passes");
    __shared__ __attribute__((aligned(16))) float kq[2][DK];
    __shared__ float part[3][4];
    __shared__ __attribute__((aligned(16))) f32x4 sums[4][2][L];
    const int seq = blockIdx.z, hv = blockIdx.y, hk = hv / (int)(p.n_v_heads / p.n_qk_heads);
    const int slot = slot_of(p, seq);
    if (slot < 0) return;
    const int t = threadIdx.x, w = t >> 6, lane = t & 63, c4 = t % L, row = t / L, col = blockIdx.x * NC + 4 * c4;
    const size_t at = ((size_t)slot * p.n_v_heads + hv) * DK * p.value_dim + (size_t)row * p.value_dim + col;
    f32x4 S[NR];
#pragma unroll
    for (int i = 0; i < NR; ++i)
        S[i] = p.state_in ? *reinterpret_cast<const f32x4 *>(p.state_in + at + (size_t)(RP * i) * p.value_dim)
                          : (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
    const float q0 = t < DK ? T::get(p.q, (size_t)seq * p.q_stride + hk * DK + t) : 0.0f;
    const float k0 = t < DK ? T::get(p.k, (size_t)seq * p.k_stride + hk * DK + t) : 0.0f;
    const size_t sc = (size_t)seq * p.g_stride + hv, va = (size_t)seq * p.v_stride + (size_t)hv * p.value_dim + col;
    const float a = expf(p.g[sc]), beta = p.beta[sc];
    f32x4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = T::get(p.v, va + e);
    if (t < DK) {
        kq[0][t] = k0;
        kq[1][t] = q0;
    }
    {
        const float kk = wave_tree64(k0 * k0), qq = wave_tree64(q0 * q0), x = wave_tree64(k0 * q0);
        if (lane == 0) {
            part[0][w] = kk;
            part[1][w] = qq;
            part[2][w] = x;
        }
    }
    __syncthreads();
    const float kk = (part[0][0] + part[0][1]) + (part[0][2] + part[0][3]);
    const float qq = (part[1][0] + part[1][1]) + (part[1][2] + part[1][3]);
    const float ikn = p.l2norm ? 1.0f / __builtin_sqrtf(kk + 1e-6f) : 1.0f;
    const float iqn = p.l2norm ? 1.0f / __builtin_sqrtf(qq + 1e-6f) : 1.0f;
    const float qk = ((part[2][0] + part[2][1]) + (part[2][2] + part[2][3])) * ikn * iqn;
    f32x4 sk = {0.0f, 0.0f, 0.0f, 0.0f}, sq = sk;
    float kv[NR];
#pragma unroll
    for (int i = 0; i < NR; ++i) {
        kv[i] = kq[0][row + RP * i] * ikn;
        const float qv = kq[1][row + RP * i] * iqn;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            sk[e] = __builtin_fmaf(S[i][e], kv[i], sk[e]);
            sq[e] = __builtin_fmaf(S[i][e], qv, sq[e]);
        }
    }
    // the rows of a wave, then the waves
#pragma unroll
    for (int m = L; m < 64; m <<= 1)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            sk[e] += __shfl_xor(sk[e], m);
            sq[e] += __shfl_xor(sq[e], m);
        }
    if (lane < L) {
        sums[w][0][lane] = sk;
        sums[w][1][lane] = sq;
    }
    __syncthreads();
    sk = (sums[0][0][c4] + sums[1][0][c4]) + (sums[2][0][c4] + sums[3][0][c4]);
    sq = (sums[0][1][c4] + sums[1][1][c4]) + (sums[2][1][c4] + sums[3][1][c4]);
    f32x4 d;
#pragma unroll
    for (int e = 0; e < 4; ++e) d[e] = beta * (v[e] - a * sk[e]);
    if (t < L) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            T::put(p.o, (size_t)seq * p.o_stride + (size_t)hv * p.value_dim + col + e,
                   p.scale * (a * sq[e] + qk * d[e]));
    }
    if (p.state_out) {
#pragma unroll
        for (int i = 0; i < NR; ++i) {
#pragma unroll
            for (int e = 0; e < 4; ++e) S[i][e] = __builtin_fmaf(kv[i], d[e], a * S[i][e]);
            *reinterpret_cast<f32x4 *>(p.state_out + at + (size_t)(RP * i) * p.value_dim) = S[i];
        }
    }
}

// ------------------------------------------------------------ host

int chunk_of(const GDNDelta *a) { return a->dtype == GDN_DTYPE_BF16 ? kChunk<Bf16> : kChunk<Fp32>; }
size_t places(const GDNDelta *a) { return (size_t)a->n_tokens / chunk_of(a) + a->n_seqs; }
// The workspace: the sequences' order and whether a start falls, the chunks'
// matrices, k and q in terms.
size_t order_bytes(const GDNDelta *a) { return (((size_t)a->n_seqs + 1) * sizeof(int) + 255) / 256 * 256; }
size_t ops_bytes(const GDNDelta *a) {
    return places(a) * a->n_v_heads *
           (a->dtype == GDN_DTYPE_BF16 ? sizeof(ChunkOps<kChunk<Bf16>>) : sizeof(ChunkOps<kChunk<Fp32>>));
}
size_t plane_bytes(const GDNDelta *a) {
    if (a->dtype == GDN_DTYPE_BF16) return 0;
    const int terms = a->dtype == GDN_DTYPE_FP16 ? Fp16::kTerms : Fp32::kTerms;
    return places(a) * a->n_qk_heads * 2 * terms * kChunk<Fp32> * a->key_dim * sizeof(uint16_t);
}

bool dim_ok(uint32_t d) { return d == 64 || d == 128 || d == 256; }

// What the host can see of a call; 1: nothing to do.
int check(const char *who, const GDNDelta *a, bool packed) {
    if (a == nullptr) return refuse(who, "args is NULL");
    if (a->dtype < GDN_DTYPE_BF16 || a->dtype > GDN_DTYPE_FP32) return refuse(who, "unknown dtype");
    if (!dim_ok(a->key_dim) || !dim_ok(a->value_dim)) return refuse(who, "head dimensions are 64, 128 or 256");
    if (a->n_qk_heads == 0 || a->n_v_heads == 0 || a->n_v_heads % a->n_qk_heads != 0 || a->n_v_heads > 65535)
        return refuse(who, "n_v_heads must be a multiple of n_qk_heads, at most 65535");
    if (a->n_seqs > 65535) return refuse(who, "at most 65535 sequences");
    if (a->n_tokens > 0x7fffffffu) return refuse(who, "at most 2^31 - 1 tokens");
    if (a->n_slots > 0x7fffffffu) return refuse(who, "at most 2^31 - 1 slots");
    if (a->n_seqs == 0 || (!packed && a->n_tokens == 0)) return 1;
    if (!packed && a->n_tokens != a->n_seqs) return refuse(who, "a step has one token a sequence");
    if (!a->slots && a->n_slots < a->n_seqs) return refuse(who, "n_slots is smaller than n_seqs, and there are no slots");
    if ((packed && !a->cu_seqlens) || (a->n_tokens != 0 && (!a->q || !a->k || !a->v || !a->o || !a->g || !a->beta)))
        return refuse(who, "a buffer pointer is NULL");
    const int64_t size = a->dtype == GDN_DTYPE_FP32 ? 4 : 2, per16 = 16 / size;
    const uintptr_t at = reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->k) |
                         reinterpret_cast<uintptr_t>(a->v) | reinterpret_cast<uintptr_t>(a->o) |
                         reinterpret_cast<uintptr_t>(a->state_in) | reinterpret_cast<uintptr_t>(a->state_out);
    const int64_t strides = a->n_tokens > 1 ? a->q_stride | a->k_stride | a->v_stride | a->o_stride : 0;
    if ((at & 15) != 0 || strides % per16 != 0)
        return refuse(who, "rows of q, k, v and o and the states start at multiples of 16 bytes");
    // rows' offsets inside a chunk are formed in 24 x 24 bits
    if (strides < 0 || strides >= (1 << 24) / size) return refuse(who, "a row stride is negative, or 16 MB or more");
    const int64_t dq = (int64_t)a->n_qk_heads * a->key_dim, dv = (int64_t)a->n_v_heads * a->value_dim;
    if (a->n_tokens > 1 && (a->q_stride < dq || a->k_stride < dq || a->v_stride < dv || a->o_stride < dv ||
                            a->g_stride < (int64_t)a->n_v_heads))
        return refuse(who, "a row stride is smaller than the row");
    return 0;
}

// Whether o shares memory with q, k or v, or one of two pools of states with the other.
bool overlaps(const GDNDelta &a) {
    const int size = a.dtype == GDN_DTYPE_FP32 ? 4 : 2;
    const uint64_t q = (uint64_t)a.n_qk_heads * a.key_dim * size, v = (uint64_t)a.n_v_heads * a.value_dim * size;
    if (gdn::rows_overlap(a.o, v, a.o_stride * size, a.q, q, a.q_stride * size, a.n_tokens) ||
        gdn::rows_overlap(a.o, v, a.o_stride * size, a.k, q, a.k_stride * size, a.n_tokens) ||
        gdn::rows_overlap(a.o, v, a.o_stride * size, a.v, v, a.v_stride * size, a.n_tokens))
        return true;
    if (!a.state_in || !a.state_out || a.state_in == a.state_out) return false;
    const uint64_t in = reinterpret_cast<uintptr_t>(a.state_in), out = reinterpret_cast<uintptr_t>(a.state_out);
    return (in < out ? out - in : in - out) / (4ull * a.n_v_heads * a.key_dim * a.value_dim) < a.n_slots;
}

template <class T, int DK, int KP, int CT>
hipError_t launch_seq(const GDNDelta &a, const int *order, const ChunkOps<kChunk<T>> *ops, const Planes<T, DK> *planes,
                      hipStream_t s) {
    const int pairs = (int)(a.n_seqs * a.n_v_heads), groups = (int)a.value_dim / (16 * CT);
    return launch(k_delta_seq<T, DK, KP, CT>, dim3((unsigned)((pairs + 7) / 8 * 8 * groups)), dim3(64 * KP), 0, s, a, order,
                  ops, planes, pairs);
}
template <class T, int DK>
hipError_t launch_prefill(const GDNDelta &a, void *ws, hipStream_t s) {
    constexpr int C = kChunk<T>, KP = DK == 64 ? 2 : 4;
    char *mem = static_cast<char *>(ws);
    int *order = reinterpret_cast<int *>(mem);
    auto *ops = reinterpret_cast<ChunkOps<C> *>(mem + order_bytes(&a));
    auto *planes = reinterpret_cast<Planes<T, DK> *>(mem + order_bytes(&a) + ops_bytes(&a));
    const hipError_t rc = launch(k_delta_prep<T, DK>, dim3((unsigned)places(&a) + 1, a.n_v_heads), dim3(4 * C), 0, s, a,
                                 order, ops, planes);
    if (rc != hipSuccess) return rc;
    // 32 columns a workgroup where as many workgroups of them fit a CU and fill
    // all.  1024 tokens a sequence, 8 heads, 16 against 32 columns: FP32, 128 x 128,
    // 16 sequences 293 and 235 us, 8 (half the CUs' places) 125 and 131; FP32, 256 x
    // 256, 4 sequences 218 and 178; FP16, 128 x 128, 16 sequences 208 and 181; BF16,
    // 64 x 64, 64 sequences 332 and 278, 32 equal.  Where a CU holds one of them for
    // two of the others: BF16, 256 x 256, 8 sequences 182 and 194.
    constexpr int kPerCu = kSeqPerCu<T, DK, KP, 1>;
    if constexpr (kSeqPerCu<T, DK, KP, 2> == kPerCu) {
        if ((size_t)a.n_seqs * a.n_v_heads * (a.value_dim / 32) >= 256 * kPerCu)
            return launch_seq<T, DK, KP, 2>(a, order, ops, planes, s);
    }
    return launch_seq<T, DK, KP, 1>(a, order, ops, planes, s);
}
template <class T>
hipError_t launch_prefill_dk(const GDNDelta &a, void *ws, hipStream_t s) {
    return a.key_dim == 256   ? launch_prefill<T, 256>(a, ws, s)
           : a.key_dim == 128 ? launch_prefill<T, 128>(a, ws, s)
                              : launch_prefill<T, 64>(a, ws, s);
}

template <class T, int DK>
hipError_t launch_step(const GDNDelta &a, hipStream_t s) {
    return launch(k_delta_step<T, DK>, dim3(a.value_dim / kStepCols, a.n_v_heads, a.n_seqs), dim3(kT), 0, s, a);
}
template <class T>
hipError_t launch_step_dk(const GDNDelta &a, hipStream_t s) {
    return a.key_dim == 256 ? launch_step<T, 256>(a, s) : a.key_dim == 128 ? launch_step<T, 128>(a, s) : launch_step<T, 64>(a, s);
}

}  // namespace delta
}  // namespace gdn

extern "C" size_t gdn_delta_prefill_workspace(const GDNDelta *args) {
    using namespace gdn::delta;
    if (args == nullptr || args->dtype < GDN_DTYPE_BF16 || args->dtype > GDN_DTYPE_FP32) return 0;
    return order_bytes(args) + ops_bytes(args) + plane_bytes(args);
}

extern "C" int gdn_delta_prefill(const GDNDelta *args, void *workspace, size_t workspace_bytes, void *stream) {
    using namespace gdn::delta;
    constexpr const char *who = "gdn_delta_prefill";
    const int rc = check(who, args, true);
    if (rc != 0) return rc < 0 ? -1 : 0;
    // a grid has fewer than 2^32 threads along an axis
    constexpr uint64_t most = (1ull << 32) / (64 * 4) - 8;
    if (places(args) >= most || (uint64_t)args->n_seqs * args->n_v_heads > most / (args->value_dim / 16) - 8)
        return gdn::refuse(who, "too many chunks or heads for one launch");
    if (workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 15) != 0 ||
        workspace_bytes < gdn_delta_prefill_workspace(args))
        return gdn::refuse(who, "the workspace is missing, misaligned or too small");
    if (overlaps(*args)) return gdn::refuse(who, "o overlaps q, k or v, or state_out a part of state_in");
    hipStream_t s = static_cast<hipStream_t>(stream);
    return gdn::launched(who, args->dtype == GDN_DTYPE_BF16   ? launch_prefill_dk<Bf16>(*args, workspace, s)
                              : args->dtype == GDN_DTYPE_FP16 ? launch_prefill_dk<Fp16>(*args, workspace, s)
                                                              : launch_prefill_dk<Fp32>(*args, workspace, s));
}

extern "C" int gdn_delta_step(const GDNDelta *args, void *stream) {
    using namespace gdn::delta;
    constexpr const char *who = "gdn_delta_step";
    const int rc = check(who, args, false);
    if (rc != 0) return rc < 0 ? -1 : 0;
    if (overlaps(*args)) return gdn::refuse(who, "o overlaps q, k or v, or state_out a part of state_in");
    hipStream_t s = static_cast<hipStream_t>(stream);
    return gdn::launched(who, args->dtype == GDN_DTYPE_BF16   ? launch_step_dk<Bf16>(*args, s)
                              : args->dtype == GDN_DTYPE_FP16 ? launch_step_dk<Fp16>(*args, s)
                                                              : launch_step_dk<Fp32>(*args, s));
}
