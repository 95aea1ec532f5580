// gdn_delta.hip -- the gated delta rule over a batch on the caller's device
// buffers: gdn_delta_prefill (packed sequences, chunk-parallel form) and
// gdn_delta_step (one token of every sequence).
#include <hip/hip_runtime.h>

#include <cstdio>
#include <mutex>

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
template <int NA, int NB>
__device__ __forceinline__ f32x4 mfma_terms(const u32x4 (&a)[NA], const u32x4 (&b)[NB], f32x4 c) {
    for_terms<NA, NB>([&](int i, int j) __attribute__((always_inline)) { c = mfma_bf16(a[i], b[j], c); });
    return c;
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

// ------------------------------------------------------------ chunk operands

// The matrices of one (chunk, value head): grid (places, value heads), a wave
// for every 16 tokens.  With G the cumulative log decay inside the chunk and
// k, q normalised:
//   L[m][s] = beta_m exp(G_m - G_s) (k_m . k_s), s < m;  T = (I + L)^-1
//   M[m][s] = scale exp(G_m - G_s) (q_m . k_s), s <= m
// T by 16 x 16 blocks: the diagonal ones by forward substitution (a lane a
// column), then T[I][J] = -T[I][I] sum_{J <= K < I} L[I][K] T[K][J] by distance
// from the diagonal on FP32 MFMAs.  G is summed in 64 bits: the weights are
// exponentials of its differences.
template <class T, int DK>
__global__ __launch_bounds__(4 * kChunk<T>) void k_delta_prep(GDNDelta p, ChunkOps<kChunk<T>> *__restrict__ ops_all,
                                                                Planes<T, DK> *__restrict__ planes) {
    constexpr int C = kChunk<T>, NW = C / 16, NT = T::kTerms, KS = DK / 32, LD = C + 4;
    constexpr int kFrag = NW * KS * NT * 64 * 16, kMat = C * LD * 4;
    __shared__ __attribute__((aligned(16))) unsigned char mem[kFrag > kMat ? kFrag : kMat];
    __shared__ __attribute__((aligned(16))) float lm[C][LD], mm[C][LD];
    __shared__ double glog[C];
    __shared__ float ikn[C], iqn[C], bet[C];
    u32x4(*kb)[KS][NT][64] = reinterpret_cast<u32x4(*)[KS][NT][64]>(mem);
    float(*tm)[LD] = reinterpret_cast<float(*)[LD]>(mem);  // once the products are formed
    const int t = threadIdx.x, w = t >> 6, lane = t & 63, li = lane & 15, kk = lane >> 4;
    const int place = blockIdx.x, hv = blockIdx.y, hk = hv / (int)(p.n_v_heads / p.n_qk_heads);
    int lo = 0, hi = (int)p.n_seqs - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (place_of<C>(span_of(p, mid).first, mid) <= place) lo = mid;
        else hi = mid - 1;
    }
    const Span sp = span_of(p, lo);
    const int m0 = (place - place_of<C>(sp.first, lo)) * C;
    if (m0 < 0 || m0 >= sp.n || slot_of(p, lo) < 0) return;
    const int n = min(C, sp.n - m0), row0 = sp.first + m0;
    ChunkOps<C> &ops = ops_all[(size_t)place * p.n_v_heads + hv];

    // wave w's 16 tokens, as A and as B fragments the same
    Raw8<T> kr[KS], qr[KS];
    const int mine = 16 * w + li;
    {
        const size_t r = (size_t)(row0 + min(mine, n - 1));
#pragma unroll
        for (int s = 0; s < KS; ++s) kr[s].load(p.k, r * p.k_stride + hk * DK + 32 * s + 8 * kk);
#pragma unroll
        for (int s = 0; s < KS; ++s) qr[s].load(p.q, r * p.q_stride + hk * DK + 32 * s + 8 * kk);
    }
    if (t < 64) {
        const size_t r = (size_t)(row0 + min(t, n - 1)) * p.g_stride + hv;
        // a decay of zero is one too small for FP32, so that differences of G
        // stay numbers
        float gv = p.g[r];
        gv = gv < -1e5f ? -1e5f : gv;
        double v = t < n ? (double)gv : 0.0;
#pragma unroll
        for (int d = 1; d < C; d <<= 1) {
            const double o = __shfl_up(v, d);
            if (lane >= d) v += o;
        }
        if (t < C) {
            glog[t] = v;
            bet[t] = t < n ? p.beta[r] : 0.0f;
        }
    }
    u32x4 qa[KS][NT];
    float kn = 0.0f, qn = 0.0f;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
        if (mine >= n) {
            kr[s].zero();
            qr[s].zero();
        }
        float x[8];
        T::get8(kr[s].w, x);
#pragma unroll
        for (int e = 0; e < 8; ++e) kn = __builtin_fmaf(x[e], x[e], kn);
        T::get8(qr[s].w, x);
#pragma unroll
        for (int e = 0; e < 8; ++e) qn = __builtin_fmaf(x[e], x[e], qn);
        u32x4 ka[NT];
        kr[s].terms(ka);
        qr[s].terms(qa[s]);
#pragma unroll
        for (int j = 0; j < NT; ++j) kb[w][s][j][lane] = ka[j];
        if constexpr (NT > 1) {
            if (hv % (int)(p.n_v_heads / p.n_qk_heads) == 0) {
                Planes<T, DK> &pl = planes[(size_t)place * p.n_qk_heads + hk];
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    *reinterpret_cast<u32x4 *>(&pl.k[j][mine][32 * s + 8 * kk]) = ka[j];
                    *reinterpret_cast<u32x4 *>(&pl.q[j][mine][32 * s + 8 * kk]) = qa[s][j];
                }
            }
        }
    }
    kn += __shfl_xor(kn, 16);
    qn += __shfl_xor(qn, 16);
    kn += __shfl_xor(kn, 32);
    qn += __shfl_xor(qn, 32);
    if (kk == 0) {
        ikn[mine] = p.l2norm ? 1.0f / __builtin_sqrtf(kn + 1e-6f) : 1.0f;
        iqn[mine] = p.l2norm ? 1.0f / __builtin_sqrtf(qn + 1e-6f) : 1.0f;
    }
    __syncthreads();
    if (t < C) {
        const float eg = expf((float)glog[t]);
        const bool in = t < n;
        ops.sc[t] = (f32x4){in ? eg * ikn[t] : 0.0f, bet[t], in ? p.scale * (eg * iqn[t]) : 0.0f,
                            in ? expf((float)(glog[n - 1] - glog[t])) * ikn[t] : 0.0f};
        if (t == 0) ops.dn = (f32x4){expf((float)glog[n - 1]), 0.0f, 0.0f, 0.0f};
    }
    f32x4 gk[NW], gq[NW];
#pragma unroll
    for (int s = 0; s < NW; ++s) gk[s] = gq[s] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int s = 0; s < KS; ++s) {
        u32x4 ka[NT];
#pragma unroll
        for (int j = 0; j < NT; ++j) ka[j] = kb[w][s][j][lane];
#pragma unroll
        for (int c = 0; c < NW; ++c)
            if (c <= w) {
                u32x4 b[NT];
#pragma unroll
                for (int j = 0; j < NT; ++j) b[j] = kb[c][s][j][lane];
                gk[c] = mfma_terms<NT, NT>(ka, b, gk[c]);
                gq[c] = mfma_terms<NT, NT>(qa[s], b, gq[c]);
            }
    }
    __syncthreads();  // k's fragments are read; T takes their place
#pragma unroll
    for (int s = 0; s < NW; ++s) {
        const int c = 16 * s + li;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int m = 16 * w + 4 * kk + r;
            float lv = 0.0f, mv = 0.0f;
            if (m < n && c <= m) {
                const float ratio = expf((float)(glog[m] - glog[c])) * ikn[c];
                if (c < m) lv = bet[m] * (ratio * ikn[m]) * gk[s][r];
                mv = p.scale * ((ratio * iqn[m]) * gq[s][r]);
            }
            lm[m][c] = lv;
            mm[m][c] = mv;
            tm[m][c] = 0.0f;
        }
    }
    __syncthreads();
    auto write_terms = [&](const float(*src)[LD], u32x4(&dst)[kTriTiles<C>][3][64], int i, int j) {
        u32x2 a[3], b[3];
        split3(*reinterpret_cast<const f32x4 *>(&src[16 * i + li][32 * j + 4 * kk]), a);
        split3(*reinterpret_cast<const f32x4 *>(&src[16 * i + li][32 * j + 16 + 4 * kk]), b);
#pragma unroll
        for (int q = 0; q < 3; ++q) dst[tri_tile(i, j)][q][lane] = (u32x4){a[q].x, a[q].y, b[q].x, b[q].y};
    };
    if (w == 0) {
        // lane 16 B + j: column j of the inverse of diagonal block B
        const int b0 = 16 * (kk < NW ? kk : 0);
        float tc[16];
#pragma unroll
        for (int m = 0; m < 16; ++m) {
            float acc = m == li ? 1.0f : 0.0f;
#pragma unroll
            for (int s4 = 0; s4 < (m + 3) / 4; ++s4) {
                const f32x4 lv = *reinterpret_cast<const f32x4 *>(&lm[b0 + m][b0 + 4 * s4]);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (4 * s4 + e < m) acc = __builtin_fmaf(lv[e], -tc[4 * s4 + e], acc);
            }
            tc[m] = acc;
        }
        if (kk < NW) {
#pragma unroll
            for (int m = 0; m < 16; ++m) tm[b0 + m][b0 + li] = tc[m];
        }
    } else {
        for (int f = w - 1; f < kTriTiles<C>; f += NW - 1) {
            const int i = f < 2 ? f : 2 + (f - 2) / 2, j = f < 2 ? 0 : f & 1;
            write_terms(mm, ops.mf, i, j);
        }
    }
    __syncthreads();
#pragma unroll
    for (int d = 1; d < NW; ++d) {
        if (w + d < NW) {
            const int I = w + d, J = w;
            f32x4 y = {0.0f, 0.0f, 0.0f, 0.0f}, z = y;
            for (int K = J; K < I; ++K) {
                const f32x4 a = *reinterpret_cast<const f32x4 *>(&lm[16 * I + li][16 * K + 4 * kk]);
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    y = __builtin_amdgcn_mfma_f32_16x16x4f32(a[q], tm[16 * K + 4 * kk + q][16 * J + li], y, 0, 0, 0);
            }
            // y's rows 4 kk + r are the B operand's k = 4 kk + q as they lie
            const f32x4 a = *reinterpret_cast<const f32x4 *>(&tm[16 * I + li][16 * I + 4 * kk]);
#pragma unroll
            for (int q = 0; q < 4; ++q) z = __builtin_amdgcn_mfma_f32_16x16x4f32(a[q], y[q], z, 0, 0, 0);
#pragma unroll
            for (int r = 0; r < 4; ++r) tm[16 * I + 4 * kk + r][16 * J + li] = -z[r];
        }
        __syncthreads();
    }
    for (int f = w; f < kTriTiles<C>; f += NW) {
        const int i = f < 2 ? f : 2 + (f - 2) / 2, j = f < 2 ? 0 : f & 1;
        write_terms(tm, ops.tf, i, j);
    }
}

// ------------------------------------------------------------ the sequences

// One (sequence, value head)'s chunks in order:
//   d = T (beta (v - exp(G) K S));  o = exp(G) Q S + M d;
//   S' = exp(G_{n-1}) S + K^T (exp(G_{n-1} - G) d)
// A workgroup of eight waves has CT = 8 / KP tiles of 16 value columns, KP waves
// a tile, a KP-th of the keys each.  A wave's state is the accumulator tiles of
// its updates, and lies so that it is also the B operand of its K S and Q S: of
// a 32-key step, lane l holds keys 8 (l / 16) .. + 7 of column l % 16, the first
// four in one tile, the others in the next.  The KP waves' shares of K S and Q S
// meet in LDS where the wave that owns a 16-token tile adds them; it forms b, its
// rows of d and of o, and leaves the BF16 terms of b, d and the scaled d in LDS
// as the B operands that the tile's waves read.  K and Q lie in LDS by rows, the
// 16-byte units XORed with the row's low bits (no two of eight rows on one
// bank); the update reads K transposed (ds_read_b64_tr_b16).  The next chunk's
// operands are loaded into registers meanwhile.
template <class T, int DK, int KP, int NW>
struct SeqLds {
    static constexpr int C = kChunk<T>, NT = T::kTerms, CT = NW / KP, MT = C / 16, JT = C / 32;
    // K of two chunks where the LDS holds it: the next one's is written while
    // this one's is read, a barrier less
    static constexpr int kBuf = NT * C * DK >= 3 * 32 * 256 ? 1 : 2;
    u32x4 k[kBuf][NT][C][DK / 8];
    // b's terms take q's place once Q S is formed
    union {
        u32x4 q[NT][C][DK / 8];
        u32x4 b[CT][JT][3][64];
    };
    union {
        f32x4 part[CT][MT][2][KP - 1][64];  // K S and Q S: [tile][token tile][which][wave but the owner]
        u32x4 df[CT][2][JT][3][64];         // d and the scaled d: [tile][which][step][term]
    };
    f32x4 sc[2][C + 1];  // a chunk's sc and, last, dn
};

template <class T, int DK, int KP, int NW>
__global__ __launch_bounds__(64 * NW) void k_delta_seq(GDNDelta p, const ChunkOps<kChunk<T>> *__restrict__ ops_all,
                                                        const Planes<T, DK> *__restrict__ planes, int pairs) {
    using Lds = SeqLds<T, DK, KP, NW>;
    constexpr int kSeqT = 64 * NW;
    constexpr int C = Lds::C, NT = Lds::NT, CT = Lds::CT, MT = Lds::MT, JT = Lds::JT, kBuf = Lds::kBuf;
    constexpr int KS = DK / 32 / KP;              // 32-key steps of a wave
    constexpr int OT = MT >= KP ? MT / KP : 1;    // token tiles a wave owns
    constexpr int kUnits = NT * C * DK / 8, PU = (kUnits + kSeqT - 1) / kSeqT;
    constexpr int kSc = C + 1;
    static_assert(KS >= 1 && MT >= KP, "whole steps and tiles");
    __shared__ Lds lds;
    const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
    const int t = threadIdx.x, w = __builtin_amdgcn_readfirstlane(t >> 6), lane = t & 63, li = lane & 15, kk = lane >> 4;
    const int ks = w % KP, ct = w / KP;
    // the column groups of a (sequence, head) share its operands: one XCD's
    // (workgroups go to the eight in turn)
    const int groups = (int)p.value_dim / (16 * CT), x = blockIdx.x >> 3;
    const int pair = (x / groups) * 8 + (blockIdx.x & 7), cg = x % groups;
    if (pair >= pairs) return;
    const int seq = pair / (int)p.n_v_heads, hv = pair % (int)p.n_v_heads;
    const int hk = hv / (int)(p.n_v_heads / p.n_qk_heads);
    const int slot = __builtin_amdgcn_readfirstlane(slot_of(p, seq));
    if (slot < 0) return;
    Span sp = span_of(p, seq);
    sp.first = __builtin_amdgcn_readfirstlane(sp.first);
    sp.n = __builtin_amdgcn_readfirstlane(sp.n);
    const int chunks = (sp.n + C - 1) / C, col = 16 * (CT * cg + ct) + li;
    const size_t place = (size_t)place_of<C>(sp.first, seq);
    const ChunkOps<C> *ops = ops_all + place * p.n_v_heads + hv;
    // the state's key of tile a, register r of step s: key0 + 32 s + 4 a + r
    const int key0 = ks * (DK / KP) + 8 * kk;
    const size_t state_at = (((size_t)slot * p.n_v_heads + hv) * DK + key0) * p.value_dim + col;

    f32x4 S[KS][2];
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                S[s][a][r] = p.state_in ? p.state_in[state_at + (size_t)(32 * s + 4 * a + r) * p.value_dim] : 0.0f;

    // the tiles this wave owns; tile i has column steps 0 .. i / 2
    auto tile_of = [&](int o) { return o == 0 ? ks : MT - 1 - ks; };
    constexpr int kTri = KP == 4 ? 2 : OT == 2 ? 3 : 1;  // their matrix tiles
    // rows at a chunk's uniform address, their offsets in 32 bits
    constexpr uint32_t kSize = T::kWords / 2;
    const uint32_t k_row = (uint32_t)p.k_stride * kSize, q_row = (uint32_t)p.q_stride * kSize,
                   v_row = (uint32_t)p.v_stride * kSize, o_row = (uint32_t)p.o_stride * kSize;
    auto rows_at = [&](const void *x, int64_t stride, int row, int head) __attribute__((always_inline)) {
        return static_cast<const char *>(x) + ((size_t)row * stride + head) * kSize;
    };
    u32x4 kreg[PU], qreg[PU], tri[kTri][3];
    f32x4 sreg;
    auto fetch_rows = [&](int c) __attribute__((always_inline)) {
        if constexpr (NT == 1) {
            // rows past the sequence's end: its last one, whose products meet
            // zero factors
            const int n = sp.n - C * c;
            const char *kp = rows_at(p.k, p.k_stride, sp.first + C * c, hk * DK),
                       *qp = rows_at(p.q, p.q_stride, sp.first + C * c, hk * DK);
#pragma unroll
            for (int i = 0; i < PU; ++i) {
                static_assert(kUnits % kSeqT == 0, "whole units a thread");
                const int u = t + i * kSeqT, row = min(u / (DK / 8), n - 1), at = 16 * (u % (DK / 8));
                kreg[i] = *reinterpret_cast<const u32x4 *>(kp + (__umul24(row, k_row) + at));
                qreg[i] = *reinterpret_cast<const u32x4 *>(qp + (__umul24(row, q_row) + at));
            }
        } else {
            const Planes<T, DK> &pl = planes[(place + c) * p.n_qk_heads + hk];
#pragma unroll
            for (int i = 0; i < PU; ++i) {
                const int u = min(t + i * kSeqT, kUnits - 1);
                kreg[i] = reinterpret_cast<const u32x4 *>(pl.k)[u];
                qreg[i] = reinterpret_cast<const u32x4 *>(pl.q)[u];
            }
        }
        const ChunkOps<C> &o = ops[(size_t)c * p.n_v_heads];
        sreg = t < C ? o.sc[min(t, C - 1)] : o.dn;
    };
    auto fetch_tri = [&](const u32x4(&m)[kTriTiles<C>][3][64]) __attribute__((always_inline)) {
        auto &f = tri;
#pragma unroll
        for (int q = 0; q < 3; ++q) {
            if constexpr (KP == 4) {
                // tile ks: one step or two (a second load of the first, unused)
                f[0][q] = m[tri_tile(ks, 0)][q][lane];
                f[1][q] = m[tri_tile(ks, ks / 2)][q][lane];
            } else {
                f[0][q] = m[ks][q][lane];
                if constexpr (OT == 2) {
                    f[1][q] = m[tri_tile(3 - ks, 0)][q][lane];
                    f[2][q] = m[tri_tile(3 - ks, 1)][q][lane];
                }
            }
        }
    };
    auto put_units = [&](u32x4 *dst, const u32x4(&src)[PU]) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < PU; ++i) {
            const int u = t + i * kSeqT;
            if (kUnits % kSeqT == 0 || u < kUnits) dst[u ^ ((u / (DK / 8)) & 7)] = src[i];
        }
    };
    auto put_sc = [&](int c) __attribute__((always_inline)) {
        if (t < kSc) lds.sc[c & 1][t] = sreg;
    };
    // this wave's rows of the matrix in `tri` times the terms in LDS, in a
    // chain for each order of the terms' products
    auto tri_product = [&](const u32x4(&b)[JT][3][64], f32x4(&y)[OT]) __attribute__((always_inline)) {
        u32x4 bo[JT][3];
#pragma unroll
        for (int j = 0; j < JT; ++j)
#pragma unroll
            for (int q = 0; q < 3; ++q) bo[j][q] = b[j][q][lane];
        f32x4 acc[kTri][3];
#pragma unroll
        for (int i = 0; i < kTri; ++i)
#pragma unroll
            for (int q = 0; q < 3; ++q) acc[i][q] = zero;
        for_terms<3, 3>([&](int m, int q) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < kTri; ++i) {
                const int j = KP == 4 ? i : i == 2;
                acc[i][m + q] = mfma_bf16(tri[i][m], bo[j][q], acc[i][m + q]);
            }
        });
        f32x4 sum[kTri];
#pragma unroll
        for (int i = 0; i < kTri; ++i) sum[i] = (acc[i][2] + acc[i][1]) + acc[i][0];
        if constexpr (KP == 4) {
            y[0] = ks < 2 ? sum[0] : sum[0] + sum[1];
        } else {
            y[0] = sum[0];
            if constexpr (OT == 2) y[1] = sum[1] + sum[2];
        }
    };
    // the terms of a tile's values, as half a B operand
    auto put_terms = [&](u32x4(&dst)[JT][3][64], int tile, const f32x4 v) __attribute__((always_inline)) {
        u32x2 e[3];
        split3(v, e);
#pragma unroll
        for (int q = 0; q < 3; ++q) reinterpret_cast<u32x2 *>(&dst[tile >> 1][q][lane])[tile & 1] = e[q];
    };

    if (chunks > 0) {
        fetch_rows(0);
        fetch_tri(ops[0].tf);
        put_units(&lds.k[0][0][0][0], kreg);
        put_units(&lds.q[0][0][0], qreg);
        put_sc(0);
    }
    for (int c = 0; c < chunks; ++c) {
        const int n = min(C, sp.n - C * c), cn = min(c + 1, chunks - 1);
        const char *vp = rows_at(p.v, p.v_stride, sp.first + C * c, hv * (int)p.value_dim);
        const auto &kc = lds.k[kBuf == 2 ? c & 1 : 0];
        const f32x4 *sc = lds.sc[c & 1];
        __syncthreads();  // this chunk's K, Q and scalars
        float v[OT][4];
#pragma unroll
        for (int o = 0; o < OT; ++o)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int m = min(16 * tile_of(o) + 4 * kk + r, n - 1);
                v[o][r] = T::get(vp + (__umul24(m, v_row) + col * kSize), 0);
            }
        fetch_rows(cn);  // (the last chunk's again, unused)
        {
            // this wave's share of K S and Q S
            f32x4 y[MT][2];
#pragma unroll
            for (int i = 0; i < MT; ++i) y[i][0] = y[i][1] = zero;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                u32x2 lo[3], hi[3];
                split3(S[s][0], lo);
                split3(S[s][1], hi);
                u32x4 sb[3];
#pragma unroll
                for (int q = 0; q < 3; ++q) sb[q] = (u32x4){lo[q].x, lo[q].y, hi[q].x, hi[q].y};
                u32x4 ka[MT][NT], qa[MT][NT];
                const int u = (key0 / 8 + 4 * s) ^ (li & 7);
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        ka[i][j] = kc[j][16 * i + li][u];
                        qa[i][j] = lds.q[j][16 * i + li][u];
                    }
                // eight chains in turn: a product that waits for the one
                // before it takes twice its time
                for_terms<NT, 3>([&](int a, int b) __attribute__((always_inline)) {
#pragma unroll
                    for (int i = 0; i < MT; ++i) {
                        y[i][0] = mfma_bf16(ka[i][a], sb[b], y[i][0]);
                        y[i][1] = mfma_bf16(qa[i][a], sb[b], y[i][1]);
                    }
                });
            }
            auto owner = [&](int i) { return i < KP ? i : MT - 1 - i; };
#pragma unroll
            for (int i = 0; i < MT; ++i)
                if (owner(i) != ks) {
                    const int at = ks < owner(i) ? ks : ks - 1;
                    lds.part[ct][i][0][at][lane] = y[i][0];
                    lds.part[ct][i][1][at][lane] = y[i][1];
                }
            __syncthreads();
            // b, and what stands of o, of the owned tiles
            f32x4 qs[OT], sw[OT];
#pragma unroll
            for (int o = 0; o < OT; ++o) {
                const int tile = tile_of(o);
                f32x4 kv = zero, qv = zero;
#pragma unroll
                for (int i = 0; i < MT; ++i)
                    if (i == tile) {
                        kv = y[i][0];
                        qv = y[i][1];
                    }
#pragma unroll
                for (int a = 0; a < KP - 1; ++a) {
                    kv += lds.part[ct][tile][0][a][lane];
                    qv += lds.part[ct][tile][1][a][lane];
                }
                f32x4 b;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const f32x4 e = sc[16 * tile + 4 * kk + r];
                    b[r] = e.y * (v[o][r] - e.x * kv[r]);
                    qs[o][r] = e.z * qv[r];
                    sw[o][r] = e.w;
                }
                put_terms(lds.b[ct], tile, b);
            }
            __syncthreads();
            f32x4 d[OT];
            tri_product(lds.b[ct], d);
            fetch_tri(ops[(size_t)c * p.n_v_heads].mf);
#pragma unroll
            for (int o = 0; o < OT; ++o) {
                put_terms(lds.df[ct][1], tile_of(o), d[o] * sw[o]);
                put_terms(lds.df[ct][0], tile_of(o), d[o]);
            }
            __syncthreads();
            // the update, and the rows of o
            u32x4 fo[JT][3];
#pragma unroll
            for (int j = 0; j < JT; ++j)
#pragma unroll
                for (int q = 0; q < 3; ++q) fo[j][q] = lds.df[ct][1][j][q][lane];
            // the next chunk's rows (q's place, b's until here, is free)
            if (kBuf == 2) put_units(&lds.k[(c + 1) & 1][0][0][0], kreg);
            put_units(&lds.q[0][0][0], qreg);
            put_sc(c + 1);
            const float dn = sc[C].x;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                u32x4 a[2][JT][NT];
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int j = 0; j < JT; ++j)
#pragma unroll
                        for (int q = 0; q < NT; ++q) {
                            // this lane's address: token + l % 16 / 4 of each
                            // group of four, keys of group l % 4
                            const int m = 32 * j + 4 * kk + (li >> 2);
                            const int u = (ks * (DK / KP) / 8 + 4 * s + (li & 3)) ^ (m & 7);
                            const u32x2 lo = read_transposed(reinterpret_cast<const u32x2 *>(&kc[q][m][u]) + h);
                            const u32x2 hi = read_transposed(reinterpret_cast<const u32x2 *>(&kc[q][m + 16][u]) + h);
                            a[h][j][q] = (u32x4){lo.x, lo.y, hi.x, hi.y};
                        }
                S[s][0] *= dn;
                S[s][1] *= dn;
                for_terms<NT, 3>([&](int e, int f) __attribute__((always_inline)) {
#pragma unroll
                    for (int j = 0; j < JT; ++j)
#pragma unroll
                        for (int h = 0; h < 2; ++h) S[s][h] = mfma_bf16(a[h][j][e], fo[j][f], S[s][h]);
                });
            }
            f32x4 om[OT];
            tri_product(lds.df[ct][0], om);
            fetch_tri(ops[(size_t)cn * p.n_v_heads].tf);
            char *op = const_cast<char *>(rows_at(p.o, p.o_stride, sp.first + C * c, hv * (int)p.value_dim));
            auto put_o = [&](int o, int r) __attribute__((always_inline)) {
                const int m = 16 * tile_of(o) + 4 * kk + r;
                T::put(op + (__umul24(m, o_row) + col * kSize), 0, qs[o][r] + om[o][r]);
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
        if (kBuf == 1) {
            __syncthreads();
            put_units(&lds.k[0][0][0][0], kreg);
        }
    }
    if (p.state_out) {
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int a = 0; a < 2; ++a)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    p.state_out[state_at + (size_t)(32 * s + 4 * a + r) * p.value_dim] = S[s][a][r];
    }
}

// ------------------------------------------------------------ a single token

// A (sequence, value head)'s token for NC value columns: grid (value_dim / NC,
// value heads, sequences).  The state tile goes through registers once: with
// a = exp(g), the sums S^T k and S^T q are formed from the state as it is read,
//   d = beta (v - a S^T k);  o = scale (a S^T q + (k . q) d);  S' = a S + k d^T
// so its bytes, in and out, are what bounds the kernel.
template <class T, int DK, int NC>
__global__ __launch_bounds__(kT) void k_delta_step(GDNDelta p) {
    constexpr int L = NC / 4, RP = kT / L, NR = (DK + RP - 1) / RP;  // lanes a row, rows a pass, passes
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

#ifndef SEQ_ONE
#define SEQ_ONE 256
#define SEQ_TWO 1000000
#endif
int chunk_of(const GDNDelta *a) { return a->dtype == GDN_DTYPE_BF16 ? kChunk<Bf16> : kChunk<Fp32>; }
size_t places(const GDNDelta *a) { return (size_t)a->n_tokens / chunk_of(a) + a->n_seqs; }
// The chunks' matrices, then k and q in terms.
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

int refuse(const char *who, const char *why) {
    std::fprintf(stderr, "%s: %s\n", who, why);
    return -1;
}

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
    if ((packed && !a->cu_seqlens) || (a->n_tokens != 0 && (!a->q || !a->k || !a->v || !a->o || !a->g || !a->beta)))
        return refuse(who, "a buffer pointer is NULL");
    const int64_t size = a->dtype == GDN_DTYPE_FP32 ? 4 : 2, per16 = 16 / size;
    const uintptr_t at = reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->k) |
                         reinterpret_cast<uintptr_t>(a->v) | reinterpret_cast<uintptr_t>(a->o) |
                         reinterpret_cast<uintptr_t>(a->state_in) | reinterpret_cast<uintptr_t>(a->state_out);
    if ((at & 15) != 0 || ((a->q_stride | a->k_stride | a->v_stride | a->o_stride) % per16) != 0)
        return refuse(who, "rows of q, k, v and o and the states start at multiples of 16 bytes");
    // rows' offsets inside a chunk are formed in 24 x 24 bits
    if (((a->q_stride | a->k_stride | a->v_stride | a->o_stride) * size) >> 24 != 0)
        return refuse(who, "a row stride is negative or larger than 16 MB");
    const int64_t dq = (int64_t)a->n_qk_heads * a->key_dim, dv = (int64_t)a->n_v_heads * a->value_dim;
    if (a->n_tokens > 1 && (a->q_stride < dq || a->k_stride < dq || a->v_stride < dv || a->o_stride < dv ||
                            a->g_stride < (int64_t)a->n_v_heads))
        return refuse(who, "a row stride is smaller than the row");
    return 0;
}

int launched(const char *who) {
    const hipError_t rc = hipGetLastError();
    if (rc != hipSuccess) {
        std::fprintf(stderr, "%s: launch failed: %s\n", who, hipGetErrorString(rc));
        return -1;
    }
    return 0;
}

template <class T, int DK, int KP, int NW>
void launch_seq(const GDNDelta &a, const ChunkOps<kChunk<T>> *ops, const Planes<T, DK> *planes, hipStream_t s) {
    const int pairs = (int)(a.n_seqs * a.n_v_heads), groups = (int)a.value_dim / (16 * (NW / KP));
    hipLaunchKernelGGL((k_delta_seq<T, DK, KP, NW>), dim3((unsigned)((pairs + 7) / 8 * 8 * groups)), dim3(64 * NW), 0, s,
                       a, ops, planes, pairs);
}
template <class T, int DK>
void launch_prefill(const GDNDelta &a, void *ws, hipStream_t s) {
    constexpr int C = kChunk<T>;
    auto *ops = static_cast<ChunkOps<C> *>(ws);
    auto *planes = reinterpret_cast<Planes<T, DK> *>(static_cast<char *>(ws) + ops_bytes(&a));
    if (a.n_tokens != 0)
        hipLaunchKernelGGL((k_delta_prep<T, DK>), dim3((unsigned)places(&a), a.n_v_heads), dim3(4 * C), 0, s, a, ops,
                           planes);
    const size_t tiles = (size_t)a.n_seqs * a.n_v_heads * (a.value_dim / 16);
    if constexpr (C == 64 && DK >= 128) {
        if (tiles <= SEQ_ONE) launch_seq<T, DK, 4, 4>(a, ops, planes, s);
        else if (tiles <= SEQ_TWO) launch_seq<T, DK, 4, 8>(a, ops, planes, s);
        else launch_seq<T, DK, 2, 8>(a, ops, planes, s);
    } else {
        if (tiles <= SEQ_ONE) launch_seq<T, DK, 2, 4>(a, ops, planes, s);
        else launch_seq<T, DK, 2, 8>(a, ops, planes, s);
    }
}
template <class T>
void launch_prefill_dk(const GDNDelta &a, void *ws, hipStream_t s) {
    if (a.key_dim == 256) launch_prefill<T, 256>(a, ws, s);
    else if (a.key_dim == 128) launch_prefill<T, 128>(a, ws, s);
    else launch_prefill<T, 64>(a, ws, s);
}

template <class T, int DK>
void launch_step(const GDNDelta &a, hipStream_t s) {
    // columns a workgroup: whole 256-byte row pieces, or 64-byte ones where
    // the former would leave CUs idle
    const size_t wide = (size_t)a.n_seqs * a.n_v_heads * (a.value_dim / 64);
    if (wide >= 256)
        hipLaunchKernelGGL((k_delta_step<T, DK, 64>), dim3(a.value_dim / 64, a.n_v_heads, a.n_seqs), dim3(kT), 0, s, a);
    else
        hipLaunchKernelGGL((k_delta_step<T, DK, 16>), dim3(a.value_dim / 16, a.n_v_heads, a.n_seqs), dim3(kT), 0, s, a);
}
template <class T>
void launch_step_dk(const GDNDelta &a, hipStream_t s) {
    if (a.key_dim == 256) launch_step<T, 256>(a, s);
    else if (a.key_dim == 128) launch_step<T, 128>(a, s);
    else launch_step<T, 64>(a, s);
}

}  // namespace delta
}  // namespace gdn

extern "C" size_t gdn_delta_prefill_workspace(const GDNDelta *args) {
    using namespace gdn::delta;
    if (args == nullptr || args->dtype < GDN_DTYPE_BF16 || args->dtype > GDN_DTYPE_FP32) return 0;
    return ops_bytes(args) + plane_bytes(args);
}

extern "C" int gdn_delta_prefill(const GDNDelta *args, void *workspace, size_t workspace_bytes, void *stream) {
    using namespace gdn::delta;
    constexpr const char *who = "gdn_delta_prefill";
    const int rc = check(who, args, true);
    if (rc != 0) return rc < 0 ? -1 : 0;
    if (places(args) > 0x7fffffffu / 4 || (uint64_t)args->n_seqs * args->n_v_heads > (1u << 24))
        return refuse(who, "too many chunks or heads for one launch");
    if (workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 15) != 0 ||
        workspace_bytes < gdn_delta_prefill_workspace(args))
        return refuse(who, "the workspace is missing, misaligned or too small");
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (args->dtype == GDN_DTYPE_BF16) launch_prefill_dk<Bf16>(*args, workspace, s);
    else if (args->dtype == GDN_DTYPE_FP16) launch_prefill_dk<Fp16>(*args, workspace, s);
    else launch_prefill_dk<Fp32>(*args, workspace, s);
    return launched(who);
}

extern "C" int gdn_delta_step(const GDNDelta *args, void *stream) {
    using namespace gdn::delta;
    constexpr const char *who = "gdn_delta_step";
    const int rc = check(who, args, false);
    if (rc != 0) return rc < 0 ? -1 : 0;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (args->dtype == GDN_DTYPE_BF16) launch_step_dk<Bf16>(*args, s);
    else if (args->dtype == GDN_DTYPE_FP16) launch_step_dk<Fp16>(*args, s);
    else launch_step_dk<Fp32>(*args, s);
    return launched(who);
}
