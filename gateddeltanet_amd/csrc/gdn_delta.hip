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

// A product of operands of NA and NB terms over one 32-wide k step, smallest
// terms first; terms below 2^-24 of the product are left out.
template <int NA, int NB>
__device__ __forceinline__ f32x4 mfma_terms(const u32x4 (&a)[NA], const u32x4 (&b)[NB], f32x4 c) {
#pragma unroll
    for (int s = 2; s >= 0; --s)
#pragma unroll
        for (int i = NA - 1; i >= 0; --i)
            if (s - i >= 0 && s - i < NB) c = mfma_bf16(a[i], b[s - i], c);
    return c;
}

// Tokens of a chunk.
template <class T>
constexpr int kChunk = T::kTerms == 1 ? 64 : 32;

// Where a 16 x 32 tile (row tile i, column step j) of a chunk's lower
// triangular matrix is kept: tiles above the diagonal are zero and left out.
template <int C>
constexpr int kTriTiles = C == 64 ? 6 : 2;
__device__ __forceinline__ constexpr int tri_tile(int i, int j) { return i < 2 ? i : 2 * i - 2 + j; }

// What k_delta_seq needs of one (chunk, value head), as it lies in its LDS.
// Matrices as MFMA A fragments of the three BF16 terms: lane l carries row
// 16 i + l % 16 and columns 32 j + 4 (l / 16) + {0..3, 16..19}, the tokens that
// lane holds of a 32-token step in the accumulator layout, so that results
// become the next product's B operand where they lie.
//   sc[m]  exp(G_m) |k_m|^-1, beta_m, scale exp(G_m) |q_m|^-1,
//          exp(G_{n-1} - G_m) |k_m|^-1; zeros past the chunk's n tokens
//   dn     exp(G_{n-1})
template <int C>
struct ChunkOps {
    u32x4 tf[kTriTiles<C>][3][64], mf[kTriTiles<C>][3][64];
    f32x4 sc[C];
    f32x4 dn;
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
__global__ __launch_bounds__(4 * kChunk<T>) void k_delta_prep(GDNDelta p, ChunkOps<kChunk<T>> *__restrict__ ops_all) {
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

// One (sequence, value head)'s chunks in order for 16 NW value columns, a wave
// 16 of them with all keys: its state is the accumulator tiles of its updates
// (lane l: key 16 tile + 4 (l / 16) + r, column l % 16), and every product of a
// chunk has its B operand in the wave's own registers:
//   d = T (beta (v - exp(G) K S));  o = exp(G) Q S + M d;
//   S' = exp(G_{n-1}) S + K^T (exp(G_{n-1} - G) d)
// so the waves meet only where the chunk's A operands change in LDS: K and Q by
// rows, K by keys, T and M.  The next chunk's are on their way in registers
// meanwhile.  16-byte units of a row are XORed with the row's low bits, which
// spreads both the fragments' reads and the transposed writes over the banks.
template <class T, int DK>
struct SeqLds {
    static constexpr int C = kChunk<T>, NT = T::kTerms;
    u32x4 kr[NT][C][DK / 8], qr[NT][C][DK / 8], kt[NT][DK][C / 8];
    ChunkOps<C> ops;
};

template <class T, int DK, int NW>
__global__ __launch_bounds__(64 * NW) void k_delta_seq(GDNDelta p, const ChunkOps<kChunk<T>> *__restrict__ ops_all,
                                                       int pairs) {
    constexpr int C = kChunk<T>, NT = T::kTerms, TPB = 64 * NW, MT = C / 16, JT = C / 32, KS = DK / 32;
    constexpr int kTasks = (C / 4) * (DK / 8), PT = (kTasks + TPB - 1) / TPB;
    constexpr int kOps = sizeof(ChunkOps<C>) / 16, PO = (kOps + TPB - 1) / TPB;
    __shared__ SeqLds<T, DK> lds;
    const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
    const int t = threadIdx.x, w = t >> 6, lane = t & 63, li = lane & 15, kk = lane >> 4;
    // the column groups of a (sequence, head) share its operands: one XCD's
    // (workgroups go to the eight in turn)
    const int groups = (int)p.value_dim / (16 * NW), x = blockIdx.x >> 3;
    const int pair = (x / groups) * 8 + (blockIdx.x & 7), cg = x % groups;
    if (pair >= pairs) return;
    const int seq = pair / (int)p.n_v_heads, hv = pair % (int)p.n_v_heads;
    const int hk = hv / (int)(p.n_v_heads / p.n_qk_heads);
    const int slot = slot_of(p, seq);
    if (slot < 0) return;
    const Span sp = span_of(p, seq);
    const int chunks = (sp.n + C - 1) / C, col = 16 * (NW * cg + w) + li;
    const size_t state_at = ((size_t)slot * p.n_v_heads + hv) * DK * p.value_dim + col;
    const ChunkOps<C> *ops = ops_all + (size_t)place_of<C>(sp.first, seq) * p.n_v_heads + hv;

    f32x4 S[DK / 16];
#pragma unroll
    for (int i = 0; i < DK / 16; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r)
            S[i][r] = p.state_in ? p.state_in[state_at + (size_t)(16 * i + 4 * kk + r) * p.value_dim] : 0.0f;

    Raw8<T> kreg[PT][4], qreg[PT][4];
    u32x4 oreg[PO];
    auto fetch = [&](int c) __attribute__((always_inline)) {
        const int n = min(C, sp.n - C * c);
#pragma unroll
        for (int i = 0; i < PT; ++i) {
            const int task = min(t + i * TPB, kTasks - 1), g8 = task % (DK / 8), quad = task / (DK / 8);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const size_t row = (size_t)(sp.first + C * c + min(4 * quad + e, n - 1));
                kreg[i][e].load(p.k, row * p.k_stride + hk * DK + 8 * g8);
                qreg[i][e].load(p.q, row * p.q_stride + hk * DK + 8 * g8);
            }
        }
        const u32x4 *src = reinterpret_cast<const u32x4 *>(ops + (size_t)c * p.n_v_heads);
#pragma unroll
        for (int i = 0; i < PO; ++i) oreg[i] = src[min(t + i * TPB, kOps - 1)];
    };
    auto place = [&](int c) __attribute__((always_inline)) {
        const int n = min(C, sp.n - C * c);
#pragma unroll
        for (int i = 0; i < PT; ++i) {
            const int task = t + i * TPB, g8 = task % (DK / 8), quad = task / (DK / 8);
            if (kTasks % TPB != 0 && task >= kTasks) break;
            // keys 8 g8 .. + 7: two groups of four of the 32-key step g8 / 4
            const int u0 = 4 * (g8 / 4) + 2 * (g8 & 1), half = (g8 >> 1) & 1;
            u32x4 kt[4][NT], qt[NT];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int m = 4 * quad + e;
                if (m >= n) {
                    kreg[i][e].zero();
                    qreg[i][e].zero();
                }
                kreg[i][e].terms(kt[e]);
                qreg[i][e].terms(qt);
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int u = (u0 + h) ^ (m & 7);
                        reinterpret_cast<u32x2 *>(&lds.kr[j][m][u])[half] = (u32x2){kt[e][j][2 * h], kt[e][j][2 * h + 1]};
                        reinterpret_cast<u32x2 *>(&lds.qr[j][m][u])[half] = (u32x2){qt[j][2 * h], qt[j][2 * h + 1]};
                    }
            }
            // tokens 4 quad .. + 3 of each key
            const int ut = 4 * (quad / 8) + (quad & 3), th = (quad >> 2) & 1;
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const uint32_t sel = e & 1 ? 0x07060302u : 0x05040100u;
                    u32x2 v;
                    v.x = __builtin_amdgcn_perm(kt[1][j][e / 2], kt[0][j][e / 2], sel);
                    v.y = __builtin_amdgcn_perm(kt[3][j][e / 2], kt[2][j][e / 2], sel);
                    const int key = 8 * g8 + e;
                    const int u = ut ^ (C == 64 ? (key ^ (key >> 3)) & 7 : ((key >> 1) ^ (key >> 3)) & 3);
                    reinterpret_cast<u32x2 *>(&lds.kt[j][key][u])[th] = v;
                }
        }
        u32x4 *dst = reinterpret_cast<u32x4 *>(&lds.ops);
#pragma unroll
        for (int i = 0; i < PO; ++i)
            if (t + i * TPB < kOps) dst[t + i * TPB] = oreg[i];
    };

    if (chunks > 0) fetch(0);
    for (int c = 0; c < chunks; ++c) {
        const int n = min(C, sp.n - C * c);
        const size_t row0 = (size_t)sp.first + (size_t)C * c;
        if (c > 0) __syncthreads();
        place(c);
        __syncthreads();
        f32x4 v[MT];
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int m = 16 * i + 4 * kk + r;
                const float x = T::get(p.v, (row0 + min(m, n - 1)) * p.v_stride + (size_t)hv * p.value_dim + col);
                v[i][r] = m < n ? x : 0.0f;
            }
        if (c + 1 < chunks) fetch(c + 1);
        // K S and Q S
        f32x4 ks[MT], qs[MT];
#pragma unroll
        for (int i = 0; i < MT; ++i) ks[i] = qs[i] = zero;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            u32x2 a[3], b[3];
            split3(S[2 * s], a);
            split3(S[2 * s + 1], b);
            u32x4 sb[3];
#pragma unroll
            for (int q = 0; q < 3; ++q) sb[q] = (u32x4){a[q].x, a[q].y, b[q].x, b[q].y};
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const int u = (4 * s + kk) ^ (li & 7);
                u32x4 ka[NT], qa[NT];
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    ka[j] = lds.kr[j][16 * i + li][u];
                    qa[j] = lds.qr[j][16 * i + li][u];
                }
                ks[i] = mfma_terms<NT, 3>(ka, sb, ks[i]);
                qs[i] = mfma_terms<NT, 3>(qa, sb, qs[i]);
            }
        }
        // a step's 32 tokens as a B operand's terms, from accumulator tiles
        auto as_operand = [&](const f32x4 *x, u32x4(&b)[JT][3]) __attribute__((always_inline)) {
#pragma unroll
            for (int j = 0; j < JT; ++j) {
                u32x2 lo[3], hi[3];
                split3(x[2 * j], lo);
                split3(x[2 * j + 1], hi);
#pragma unroll
                for (int q = 0; q < 3; ++q) b[j][q] = (u32x4){lo[q].x, lo[q].y, hi[q].x, hi[q].y};
            }
        };
        f32x4 fs[MT], d[MT];
        u32x4 ob[JT][3];
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            f32x4 b;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const f32x4 sc = lds.ops.sc[16 * i + 4 * kk + r];
                b[r] = sc.y * (v[i][r] - sc.x * ks[i][r]);
                qs[i][r] *= sc.z;
                fs[i][r] = sc.w;
            }
            ks[i] = b;
        }
        as_operand(ks, ob);
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            d[i] = zero;
#pragma unroll
            for (int j = 0; j <= i / 2; ++j) {
                u32x4 a[3];
#pragma unroll
                for (int q = 0; q < 3; ++q) a[q] = lds.ops.tf[tri_tile(i, j)][q][lane];
                d[i] = mfma_split(a, ob[j], d[i]);
            }
        }
        as_operand(d, ob);
#pragma unroll
        for (int i = 0; i < MT; ++i) {
#pragma unroll
            for (int j = 0; j <= i / 2; ++j) {
                u32x4 a[3];
#pragma unroll
                for (int q = 0; q < 3; ++q) a[q] = lds.ops.mf[tri_tile(i, j)][q][lane];
                qs[i] = mfma_split(a, ob[j], qs[i]);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int m = 16 * i + 4 * kk + r;
                if (m < n) T::put(p.o, (row0 + m) * p.o_stride + (size_t)hv * p.value_dim + col, qs[i][r]);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) d[i][r] *= fs[i][r];
        }
        as_operand(d, ob);
        const float dn = lds.ops.dn.x;
#pragma unroll
        for (int i = 0; i < DK / 16; ++i) {
            const int key = 16 * i + li;
            const int sw = C == 64 ? (key ^ (key >> 3)) & 7 : ((key >> 1) ^ (key >> 3)) & 3;
            f32x4 s = S[i];
#pragma unroll
            for (int r = 0; r < 4; ++r) s[r] *= dn;
#pragma unroll
            for (int j = 0; j < JT; ++j) {
                u32x4 a[NT];
#pragma unroll
                for (int q = 0; q < NT; ++q) a[q] = lds.kt[q][key][(4 * j + kk) ^ sw];
                s = mfma_terms<NT, 3>(a, ob[j], s);
            }
            S[i] = s;
        }
    }
    if (p.state_out) {
#pragma unroll
        for (int i = 0; i < DK / 16; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) p.state_out[state_at + (size_t)(16 * i + 4 * kk + r) * p.value_dim] = S[i][r];
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

int chunk_of(const GDNDelta *a) { return a->dtype == GDN_DTYPE_BF16 ? kChunk<Bf16> : kChunk<Fp32>; }
size_t ops_bytes(const GDNDelta *a) {
    return a->dtype == GDN_DTYPE_BF16 ? sizeof(ChunkOps<64>) : sizeof(ChunkOps<32>);
}
size_t places(const GDNDelta *a) { return (size_t)a->n_tokens / chunk_of(a) + a->n_seqs; }

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

template <class T, int DK>
void launch_prefill(const GDNDelta &a, void *ws, hipStream_t s) {
    constexpr int C = kChunk<T>, NW = 4;
    auto *ops = static_cast<ChunkOps<C> *>(ws);
    if (a.n_tokens != 0)
        hipLaunchKernelGGL((k_delta_prep<T, DK>), dim3((unsigned)places(&a), a.n_v_heads), dim3(4 * C), 0, s, a, ops);
    const int pairs = (int)(a.n_seqs * a.n_v_heads), groups = (int)a.value_dim / (16 * NW);
    hipLaunchKernelGGL((k_delta_seq<T, DK, NW>), dim3((unsigned)((pairs + 7) / 8 * 8 * groups)), dim3(64 * NW), 0, s,
                       a, ops, pairs);
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
    return places(args) * args->n_v_heads * ops_bytes(args);
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
