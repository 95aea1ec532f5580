// gdn_scan.hip -- the selective state space scan over a batch on the caller's
// device buffers: gdn_scan_prefill (packed sequences, chunk-parallel form) and
// gdn_scan_step (one token of every sequence).
#include <hip/hip_runtime.h>

#include "gdn_amd.h"
#include "gdn_device.h"
#include "gdn_internal.h"
#include "gdn_packed.h"
#include "gdn_wy.h"

namespace gdn {
namespace scan {

using namespace packed;

// Tokens of a chunk.
template <class T>
constexpr int kChunk = T::kTerms == 1 ? 64 : 32;
// BF16 terms of the FP32 operands that only y is formed from: two leave 2^-17 of a
// product out, which a y of 8 or 11 significand bits does not show; the state's
// have three throughout.
template <class T>
constexpr int kOutTerms = T::kTerms == 3 ? 3 : 2;

// A token's step: dt + dt_bias, softplus of it where asked for.
template <class T>
__device__ __forceinline__ float step_of(const GDNScan &p, size_t row, int head) {
    const size_t at = row * p.dt_stride + head;
    return (p.dt_dtype == GDN_DTYPE_FP32 ? static_cast<const float *>(p.dt)[at] : T::get(p.dt, at)) +
           (p.dt_bias ? p.dt_bias[head] : 0.0f);
}
__device__ __forceinline__ float step_size(const GDNScan &p, float h) {
    return p.softplus ? fmaxf(h, 0.0f) + log1pf(expf(-fabsf(h))) : h;
}

// Sequences are cut in segments of `seg` tokens, so that one long sequence fills
// the chip.  A sequence of m + 1 segments (m = 0 for an empty one) has m states in
// the workspace, behind all its segments but the last, at places first / seg + 0 ..
// m - 1: none is shared, as a sequence of n tokens has m <= n / seg, and there are at
// most n_tokens / seg.
__device__ __forceinline__ int cuts_of(const Span &sp, int seg) { return sp.n > 0 ? (sp.n - 1) / seg : 0; }

template <class T, int N, int NW>
struct Lds {
    static constexpr int C = kChunk<T>, NT = T::kTerms, kTri = C == 64 ? 6 : 2;
    // 16-byte units of a row, the last of them padding: rows four banks apart
    static constexpr int kRow = N / 8 + 1, kXRow = 2 * NW + 1;
    u32x4 b[NT][C][kRow], c[NT][C][kRow], x[NT][C][kXRow];
    u32x4 m[kTri][kOutTerms<T>][64];
    f32x4 sc[NW][C];
    float eg[NW][C];
};
// Where a 16 x 32 tile of a chunk's lower triangular matrix is kept: row tile j,
// column step i.
__device__ __forceinline__ constexpr int tri_tile(int j, int i) { return j < 2 ? j : 2 * j - 2 + i; }

// A segment's chunks in order, for a head's 16 NW columns, 16 a wave.  With G the
// running log decay of a chunk (sums in 64 bits) and h the steps:
//   y = exp(G) C S + M x + D x,  M[m][s] = exp(G_m - G_s) h_s (C_m . B_s), s <= m
//   S' = exp(G_last) S + B^T (exp(G_last - G) h x)
// Products are BF16 matrix instructions on the terms that the operands split into.
// A wave's state is the accumulator tiles of its update, and lies so that it is
// also the B operand of C S: of a 32-row step, lane l holds rows 8 (l / 16) .. + 7 of
// column l % 16, the first four in one tile, the others in the next.  M's tiles are
// formed transposed, B C^T, spread over the waves: an accumulator is then half an A
// operand of M x as it is.  x and B^T are read transposed (ds_read_b64_tr_b16).  The
// steps and decays of NW chunks are formed at a time, a chunk a wave.  The next
// chunk's rows are on their way into registers meanwhile.
//   pass 0   the segments with a later one: the first whole, of the others the
//            state they add to zero and their decay
//   pass 1   the others whole, from the states behind the segments before them
// so the slot of a sequence is read before pass 1 writes it, or by the workgroup
// that does.
template <class T, int N, int NW>
__global__ __launch_bounds__(64 * NW, 2) void k_scan_segment(GDNScan p, float *__restrict__ states,
                                                             float *__restrict__ decays, int seg, int pass, int units) {
    using L = Lds<T, N, NW>;
    constexpr int C = L::C, NT = L::NT, MT = C / 16, JT = C / 32, KS = N / 32, OT = kOutTerms<T>, kThreads = 64 * NW;
    constexpr int kB = C * (N / 8), kX = C * 2 * NW;  // 16-byte units (of 16-bit values) of a chunk's rows
    constexpr int kBr = (kB + kThreads - 1) / kThreads, kXr = (kX + kThreads - 1) / kThreads;
    __shared__ L lds;
    const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
    const int t = threadIdx.x, w = __builtin_amdgcn_readfirstlane(t >> 6), lane = t & 63, li = lane & 15, kk = lane >> 4;
    // the column groups of a (segment, head) share its rows of B and C: one XCD's
    // (workgroups go to the eight in turn)
    const int groups = (int)p.head_dim / (16 * NW), bx = blockIdx.x >> 3;
    const int unit = (bx / groups) * 8 + (blockIdx.x & 7), cg = bx % groups;
    if (unit >= units) return;
    const int head = unit % (int)p.n_heads, place = unit / (int)p.n_heads, group = head / (int)(p.n_heads / p.n_groups);
    const int seq = last_at_most((int)p.n_seqs, place,
                                 [&](int i) { return span_of(p, i).first / seg + (pass ? i : 0); });
    Span sp = span_of(p, seq);
    sp.first = __builtin_amdgcn_readfirstlane(sp.first);
    sp.n = __builtin_amdgcn_readfirstlane(sp.n);
    const int slot = __builtin_amdgcn_readfirstlane(slot_of(p, seq));
    const int cuts = cuts_of(sp, seg), base = sp.first / seg, c0 = place - base - (pass ? seq : 0);
    if (slot < 0 || c0 < 0 || (pass ? c0 > cuts || (c0 == 0 && cuts > 0) : c0 >= cuts)) return;
    const bool whole = pass || c0 == 0;
    const int row0 = sp.first + c0 * seg, n_rows = min(seg, sp.n - c0 * seg), chunks = (n_rows + C - 1) / C;
    const int col = 16 * (NW * cg + w) + li;
    const size_t head_at = (size_t)8 * kk * p.head_dim + col, tile = (size_t)N * p.head_dim;
    auto at_of = [&](int s, int a, int r) { return head_at + (size_t)(32 * s + 4 * a + r) * p.head_dim; };
    f32x4 S[KS][2];
    {
        const float *from = c0 > 0 ? (pass ? states + ((size_t)(base + c0 - 1) * p.n_heads + head) * tile : nullptr)
                            : p.state_in ? p.state_in + ((size_t)slot * p.n_heads + head) * tile
                                         : nullptr;
#pragma unroll
        for (int s = 0; s < KS; ++s) S[s][0] = S[s][1] = zero;
        if (from) {
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int a = 0; a < 2; ++a)
#pragma unroll
                    for (int r = 0; r < 4; ++r) S[s][a][r] = from[at_of(s, a, r)];
        }
    }

    constexpr uint32_t kSize = T::kWords / 2;  // bytes of a value
    Raw8<T> breg[kBr], creg[kBr], xreg[kXr];
    auto rows_at = [&](const void *x, int64_t stride, int row, int first) __attribute__((always_inline)) {
        return static_cast<const char *>(x) + ((size_t)row * stride + first) * kSize;
    };
    // rows past the segment's end: its last one, in bounds, put as zeros
    auto fetch = [&](int c) __attribute__((always_inline)) {
        const int n = n_rows - C * c, row = row0 + C * c;
        const char *bp = rows_at(p.b, p.b_stride, row, group * N), *cp = rows_at(p.c, p.c_stride, row, group * N),
                   *xp = rows_at(p.x, p.x_stride, row, head * (int)p.head_dim + 16 * NW * cg);
        const uint32_t bs = (uint32_t)p.b_stride * kSize, cs = (uint32_t)p.c_stride * kSize, xs = (uint32_t)p.x_stride * kSize;
#pragma unroll
        for (int i = 0; i < kBr; ++i) {
            const int u = i * kThreads + t, r = min(u / (N / 8), n - 1), at = 8 * kSize * (u % (N / 8));
            if (kB % kThreads == 0 || u < kB) {
                breg[i].load(bp + (__umul24(r, bs) + at), 0);
                if (whole) creg[i].load(cp + (__umul24(r, cs) + at), 0);
            }
        }
#pragma unroll
        for (int i = 0; i < kXr; ++i) {
            const int u = i * kThreads + t, r = min(u / (2 * NW), n - 1), at = 8 * kSize * (u % (2 * NW));
            if (kX % kThreads == 0 || u < kX) xreg[i].load(xp + (__umul24(r, xs) + at), 0);
        }
    };
    auto put_rows = [&](int c) __attribute__((always_inline)) {
        const int n = n_rows - C * c;
        u32x4 e[NT];
#pragma unroll
        for (int i = 0; i < kBr; ++i) {
            const int u = i * kThreads + t, r = u / (N / 8);
            if (kB % kThreads != 0 && u >= kB) break;
            if (r >= n) {
                breg[i].zero();
                creg[i].zero();
            }
            breg[i].terms(e);
#pragma unroll
            for (int q = 0; q < NT; ++q) lds.b[q][r][u % (N / 8)] = e[q];
            if (whole) {
                creg[i].terms(e);
#pragma unroll
                for (int q = 0; q < NT; ++q) lds.c[q][r][u % (N / 8)] = e[q];
            }
        }
#pragma unroll
        for (int i = 0; i < kXr; ++i) {
            const int u = i * kThreads + t, r = u / (2 * NW);
            if (kX % kThreads != 0 && u >= kX) break;
            if (r >= n) xreg[i].zero();
            xreg[i].terms(e);
#pragma unroll
            for (int q = 0; q < NT; ++q) lds.x[q][r][u % (2 * NW)] = e[q];
        }
    };
    // wave w's chunk of a block of NW: steps, decays
    const double rate = (double)p.A[head] * 1.44269504088896340736;
    const float skip = p.D ? p.D[head] : 0.0f;
    float dt = 0.0f;
    auto fetch_dt = [&](int c) __attribute__((always_inline)) {
        const int m = C * (c + w) + lane;
        if (lane < C && m < n_rows) dt = step_of<T>(p, (size_t)(row0 + m), head);
    };
    auto put_steps = [&](int c) __attribute__((always_inline)) {
        const bool in = lane < C && C * (c + w) + lane < n_rows;
        const float h = in ? step_size(p, dt) : 0.0f;
        // held to a size whose differences stay numbers, far beyond FP32's powers
        double g = (double)h * rate;
        g = g < -1e5 ? -1e5 : g > 1e5 ? 1e5 : g;
        const double sum = wave_scan64(in ? g : 0.0), last = __shfl(sum, 63), n = __builtin_rint(sum);
        if (lane < C) {
            lds.sc[w][lane] = (f32x4){(float)(sum - n), u2f((uint32_t)(int)n), h, exp2_of(last - sum) * h};
            lds.eg[w][lane] = exp2_of(sum);
        }
    };

    if (chunks > 0) {
        fetch(0);
        fetch_dt(0);
    }
    // of M's tiles on the diagonal, the half above it
    if (w == 0) {
#pragma unroll
        for (int j = 0; j < MT; j += 2)
#pragma unroll
            for (int q = 0; q < OT; ++q)
                reinterpret_cast<u32x2 *>(&lds.m[tri_tile(j, j / 2)][q][lane])[1] = (u32x2){0u, 0u};
    }
    float decay = 1.0f;
    for (int c = 0; c < chunks; ++c) {
        const int n = min(C, n_rows - C * c), cb = c % NW;
        put_rows(c);
        if (cb == 0) {
            put_steps(c);
            fetch_dt(c + NW);
        }
        __syncthreads();
        if (c + 1 < chunks) fetch(c + 1);
        const f32x4(&sc)[C] = lds.sc[cb];
        const float(&eg)[C] = lds.eg[cb];
        f32x4 y[MT];
        if (whole) {
            // M's tiles, two halves of a step
            for (int q = w; q < MT * (MT + 1) / 2; q += NW) {
                const int j = q < 1 ? 0 : q < 3 ? 1 : q < 6 ? 2 : 3, i = q - j * (j + 1) / 2;
                f32x4 z[2] = {zero, zero};
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    u32x4 a[NT], b[NT];
#pragma unroll
                    for (int k = 0; k < NT; ++k) {
                        a[k] = lds.b[k][16 * i + li][4 * s + kk];
                        b[k] = lds.c[k][16 * j + li][4 * s + kk];
                    }
                    for_terms<NT, NT>([&](int k, int l) __attribute__((always_inline)) { z[s & 1] = mfma_bf16(a[k], b[l], z[s & 1]); });
                }
                const f32x4 to = sc[16 * j + li];
                f32x4 v;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const f32x4 of = sc[16 * i + 4 * kk + r];
                    // (above the diagonal a power that makes it zero, not a branch)
                    const int n2 = i < j || 4 * kk + r <= li ? (int)f2u(to.y) - (int)f2u(of.y) : -1000;
                    const float e = __builtin_ldexpf(__builtin_amdgcn_exp2f(to.x - of.x), n2) * of.z;
                    v[r] = e * (z[0][r] + z[1][r]);
                }
                u32x2 e[3];
                split3(v, e);
#pragma unroll
                for (int k = 0; k < OT; ++k) reinterpret_cast<u32x2 *>(&lds.m[tri_tile(j, i / 2)][k][lane])[i & 1] = e[k];
            }
#pragma unroll
            for (int i = 0; i < MT; ++i) y[i] = zero;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                u32x2 lo[3], hi[3];
                split3(S[s][0], lo);
                split3(S[s][1], hi);
                u32x4 sb[OT], ca[MT][NT];
#pragma unroll
                for (int q = 0; q < OT; ++q) sb[q] = (u32x4){lo[q].x, lo[q].y, hi[q].x, hi[q].y};
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int q = 0; q < NT; ++q) ca[i][q] = lds.c[q][16 * i + li][4 * s + kk];
                for_terms<NT, OT>([&](int a, int b) __attribute__((always_inline)) {
#pragma unroll
                    for (int i = 0; i < MT; ++i) y[i] = mfma_bf16(ca[i][a], sb[b], y[i]);
                });
            }
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) y[i][r] *= eg[16 * i + 4 * kk + r];
            __syncthreads();
        }
        // x as a B operand: of a 32-token step, tokens 4 (l / 16) .. + 3 and those 16 on
        u32x4 xb[JT][NT], xo[JT][3];
        f32x4 xv[MT];
#pragma unroll
        for (int j = 0; j < JT; ++j)
#pragma unroll
            for (int q = 0; q < NT; ++q) {
                const int m = 32 * j + 4 * kk + (li >> 2);
                const u32x2 lo = read_transposed(reinterpret_cast<const u32x2 *>(&lds.x[q][m][0]) + 4 * w + (li & 3));
                const u32x2 hi = read_transposed(reinterpret_cast<const u32x2 *>(&lds.x[q][m + 16][0]) + 4 * w + (li & 3));
                xb[j][q] = (u32x4){lo.x, lo.y, hi.x, hi.y};
            }
#pragma unroll
        for (int j = 0; j < JT; ++j) {
            u32x2 e[2][3];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                f32x4 v = zero;
#pragma unroll
                for (int q = NT - 1; q >= 0; --q)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const uint32_t u = xb[j][q][2 * h + r / 2];
                        v[r] += u2f(r % 2 ? u & 0xffff0000u : u << 16);
                    }
                xv[2 * j + h] = v;
#pragma unroll
                for (int r = 0; r < 4; ++r) v[r] *= sc[32 * j + 16 * h + 4 * kk + r].w;
                split3(v, e[h]);
            }
#pragma unroll
            for (int q = 0; q < 3; ++q) xo[j][q] = (u32x4){e[0][q].x, e[0][q].y, e[1][q].x, e[1][q].y};
        }
        const float dn = eg[C - 1];
        decay *= dn;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            u32x4 a[2][JT][NT];
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int j = 0; j < JT; ++j)
#pragma unroll
                    for (int q = 0; q < NT; ++q) {
                        const int m = 32 * j + 4 * kk + (li >> 2), u = 2 * (4 * s + (li & 3)) + h;
                        const u32x2 lo = read_transposed(reinterpret_cast<const u32x2 *>(&lds.b[q][m][0]) + u);
                        const u32x2 hi = read_transposed(reinterpret_cast<const u32x2 *>(&lds.b[q][m + 16][0]) + u);
                        a[h][j][q] = (u32x4){lo.x, lo.y, hi.x, hi.y};
                    }
            S[s][0] *= dn;
            S[s][1] *= dn;
            for_terms<NT, 3>([&](int e, int f) __attribute__((always_inline)) {
#pragma unroll
                for (int j = 0; j < JT; ++j)
#pragma unroll
                    for (int h = 0; h < 2; ++h) S[s][h] = mfma_bf16(a[h][j][e], xo[j][f], S[s][h]);
            });
        }
        if (whole) {
            for_terms<OT, NT>([&](int a, int b) __attribute__((always_inline)) {
#pragma unroll
                for (int j = 0; j < MT; ++j)
#pragma unroll
                    for (int i = 0; i <= j / 2; ++i) y[j] = mfma_bf16(lds.m[tri_tile(j, i)][a][lane], xb[i][b], y[j]);
            });
            char *yp = const_cast<char *>(rows_at(p.y, p.y_stride, row0 + C * c, head * (int)p.head_dim));
            const uint32_t ys = (uint32_t)p.y_stride * kSize;
#pragma unroll
            for (int j = 0; j < MT; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int m = 16 * j + 4 * kk + r;
                    if (m < n) T::put(yp + (__umul24(m, ys) + col * kSize), 0, __builtin_fmaf(skip, xv[j][r], y[j][r]));
                }
        }
        __syncthreads();
    }
    float *to = nullptr;
    if (pass) {
        if (c0 == cuts && p.state_out) to = p.state_out + ((size_t)slot * p.n_heads + head) * tile;
    } else {
        to = states + ((size_t)place * p.n_heads + head) * tile;
        if (cg == 0 && t == 0) decays[(size_t)place * p.n_heads + head] = decay;
    }
    if (to) {
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int a = 0; a < 2; ++a)
#pragma unroll
                for (int r = 0; r < 4; ++r) to[at_of(s, a, r)] = S[s][a][r];
    }
}

// Between the passes: a sequence's states behind its segments from what each of
// them adds.  Grid (state values / 1024, heads, sequences in turn).
__global__ __launch_bounds__(kT) void k_scan_join(GDNScan p, float *__restrict__ states, const float *__restrict__ decays,
                                                  int seg) {
    const size_t tile = (size_t)p.state_dim * p.head_dim;
    const int head = blockIdx.y, at = (blockIdx.x * kT + (int)threadIdx.x) * 4;
    for (int seq = blockIdx.z; seq < (int)p.n_seqs; seq += gridDim.z) {
        const Span sp = span_of(p, seq);
        const int cuts = cuts_of(sp, seg);
        if (cuts < 2 || slot_of(p, seq) < 0) continue;
        const size_t unit = (size_t)(sp.first / seg) * p.n_heads + head;
        float *s = states + unit * tile + at;
        const float *d = decays + unit;
        const size_t step = p.n_heads * tile;
        f32x4 v = *reinterpret_cast<const f32x4 *>(s);
        constexpr int kAhead = 8;  // segments on their way at once
        for (int c = 1; c < cuts; c += kAhead) {
            f32x4 u[kAhead];
            float a[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                const int i = min(c + k, cuts - 1);
                u[k] = *reinterpret_cast<const f32x4 *>(s + i * step);
                a[k] = d[(size_t)i * p.n_heads];
            }
#pragma unroll
            for (int k = 0; k < kAhead; ++k)
                if (c + k < cuts) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = __builtin_fmaf(a[k], v[e], u[k][e]);
                    *reinterpret_cast<f32x4 *>(s + (c + k) * step) = v;
                }
        }
    }
}

// ------------------------------------------------------------ a single token

// A (sequence, head)'s token for 64 columns: grid (head_dim / 64, heads,
// sequences).  The state's tile goes through registers once.
template <class T, int N>
__global__ __launch_bounds__(kT) void k_scan_step(GDNScan p) {
    constexpr int L = 16, RP = kT / L, NR = N / RP;  // lanes a row, rows a pass, passes
    __shared__ __attribute__((aligned(16))) f32x4 sums[4][L];
    const int seq = blockIdx.z, head = blockIdx.y, group = head / (int)(p.n_heads / p.n_groups);
    const int slot = slot_of(p, seq);
    if (slot < 0) return;
    const int t = threadIdx.x, w = t >> 6, lane = t & 63, c4 = t % L, row = t / L, col = blockIdx.x * 64 + 4 * c4;
    const size_t at = ((size_t)slot * p.n_heads + head) * N * p.head_dim + (size_t)row * p.head_dim + col;
    f32x4 S[NR];
#pragma unroll
    for (int i = 0; i < NR; ++i)
        S[i] = p.state_in ? *reinterpret_cast<const f32x4 *>(p.state_in + at + (size_t)(RP * i) * p.head_dim)
                          : (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
    float b[NR], c[NR];
    const size_t b_at = (size_t)seq * p.b_stride + group * N + row, c_at = (size_t)seq * p.c_stride + group * N + row;
#pragma unroll
    for (int i = 0; i < NR; ++i) {
        b[i] = T::get(p.b, b_at + RP * i);
        c[i] = T::get(p.c, c_at + RP * i);
    }
    const size_t x_at = (size_t)seq * p.x_stride + (size_t)head * p.head_dim + col;
    f32x4 x, y = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = T::get(p.x, x_at + e);
    const float h = step_size(p, step_of<T>(p, seq, head)), a = expf(h * p.A[head]);
#pragma unroll
    for (int i = 0; i < NR; ++i) {
        const float hb = h * b[i];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            S[i][e] = __builtin_fmaf(hb, x[e], a * S[i][e]);
            y[e] = __builtin_fmaf(c[i], S[i][e], y[e]);
        }
        if (p.state_out) *reinterpret_cast<f32x4 *>(p.state_out + at + (size_t)(RP * i) * p.head_dim) = S[i];
    }
    // the rows of a wave, then the waves
#pragma unroll
    for (int m = L; m < 64; m <<= 1)
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] += __shfl_xor(y[e], m);
    if (lane < L) sums[w][lane] = y;
    __syncthreads();
    if (t < L) {
        y = (sums[0][t] + sums[1][t]) + (sums[2][t] + sums[3][t]);
        const float skip = p.D ? p.D[head] : 0.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            T::put(p.y, (size_t)seq * p.y_stride + (size_t)head * p.head_dim + col + e, __builtin_fmaf(skip, x[e], y[e]));
    }
}

// ------------------------------------------------------------ host

bool dim_ok(uint32_t d) { return d == 64 || d == 128 || d == 256; }
constexpr int kWaves = 4;

// Tokens of a segment: see k_scan_segment.
int segment_of(const GDNScan *a) {
    const uint64_t per = (uint64_t)a->n_heads * (a->head_dim / (16 * kWaves));
    uint64_t seg = (a->n_tokens * per / 768 + 63) / 64 * 64;
    const uint64_t least = 2 * a->state_dim;
    seg = seg < least ? least : seg;
    return (int)(seg > 1024 ? 1024 : seg);
}
size_t places(const GDNScan *a) { return a->n_tokens / (uint32_t)segment_of(a); }
bool cut(const GDNScan *a) { return a->n_tokens > (uint32_t)segment_of(a); }
size_t decay_bytes(const GDNScan *a) { return (places(a) * a->n_heads * sizeof(float) + 255) / 256 * 256; }

// What the host can see of a call; 1: nothing to do.
int check(const char *who, const GDNScan *a, bool packed) {
    if (a == nullptr) return refuse(who, "args is NULL");
    if (a->dtype < GDN_DTYPE_BF16 || a->dtype > GDN_DTYPE_FP32) return refuse(who, "unknown dtype");
    if (a->dt_dtype != a->dtype && a->dt_dtype != GDN_DTYPE_FP32) return refuse(who, "dt_dtype is dtype or FP32");
    if (!dim_ok(a->state_dim) || !dim_ok(a->head_dim)) return refuse(who, "state_dim and head_dim are 64, 128 or 256");
    if (a->n_groups == 0 || a->n_heads == 0 || a->n_heads % a->n_groups != 0 || a->n_heads > 65535)
        return refuse(who, "n_heads must be a multiple of n_groups, at most 65535");
    if (a->n_seqs > 65535) return refuse(who, "at most 65535 sequences");
    if (a->n_tokens > 0x7fffff00u) return refuse(who, "at most 2^31 - 256 tokens");
    if (a->n_slots > 0x7fffffffu) return refuse(who, "at most 2^31 - 1 slots");
    if (a->n_seqs == 0) return 1;
    if (!packed && a->n_tokens != a->n_seqs) return refuse(who, "a step has one token a sequence");
    if (!a->slots && a->n_slots < a->n_seqs) return refuse(who, "n_slots is smaller than n_seqs, and there are no slots");
    if ((packed && !a->cu_seqlens) || !a->A || (a->n_tokens != 0 && (!a->x || !a->b || !a->c || !a->dt || !a->y)))
        return refuse(who, "a buffer pointer is NULL");
    const int64_t size = a->dtype == GDN_DTYPE_FP32 ? 4 : 2, per16 = 16 / size;
    const uintptr_t at = reinterpret_cast<uintptr_t>(a->x) | reinterpret_cast<uintptr_t>(a->b) |
                         reinterpret_cast<uintptr_t>(a->c) | reinterpret_cast<uintptr_t>(a->y) |
                         reinterpret_cast<uintptr_t>(a->state_in) | reinterpret_cast<uintptr_t>(a->state_out);
    const int64_t strides = a->n_tokens > 1 ? a->x_stride | a->b_stride | a->c_stride | a->y_stride : 0;
    if ((at & 15) != 0 || strides % per16 != 0)
        return refuse(who, "rows of x, b, c and y and the states start at multiples of 16 bytes");
    // rows' offsets inside a chunk are formed in 24 x 24 bits
    if (strides < 0 || strides >= (1 << 24) / size) return refuse(who, "a row stride is negative, or 16 MB or more");
    const int64_t dx = (int64_t)a->n_heads * a->head_dim, db = (int64_t)a->n_groups * a->state_dim;
    if (a->n_tokens > 1 && (a->x_stride < dx || a->y_stride < dx || a->b_stride < db || a->c_stride < db ||
                            a->dt_stride < (int64_t)a->n_heads || a->dt_stride > (int64_t)1 << 40))
        return refuse(who, "a row stride is smaller than the row, or dt's above 2^40");
    const uint64_t rx = dx * size, rb = db * size, rd = a->n_heads * (a->dt_dtype == GDN_DTYPE_FP32 ? 4ull : 2ull);
    const int64_t ys = a->y_stride * size;
    if (rows_overlap(a->y, rx, ys, a->x, rx, a->x_stride * size, a->n_tokens) ||
        rows_overlap(a->y, rx, ys, a->b, rb, a->b_stride * size, a->n_tokens) ||
        rows_overlap(a->y, rx, ys, a->c, rb, a->c_stride * size, a->n_tokens) ||
        rows_overlap(a->y, rx, ys, a->dt, rd, a->dt_stride * (int64_t)(rd / a->n_heads), a->n_tokens))
        return refuse(who, "y overlaps x, b, c or dt");
    if (a->state_in && a->state_out && a->state_in != a->state_out) {
        const uint64_t in = reinterpret_cast<uintptr_t>(a->state_in), out = reinterpret_cast<uintptr_t>(a->state_out);
        if ((in < out ? out - in : in - out) / (4ull * a->n_heads * a->state_dim * a->head_dim) < a->n_slots)
            return refuse(who, "state_out overlaps a part of state_in");
    }
    return 0;
}

template <class T, int N>
hipError_t launch_prefill(const GDNScan &a, void *ws, hipStream_t s) {
    const int seg = segment_of(&a), groups = (int)a.head_dim / (16 * kWaves);
    float *decays = static_cast<float *>(ws), *states = reinterpret_cast<float *>(static_cast<char *>(ws) + decay_bytes(&a));
    auto pass = [&](int number, size_t n_places) {
        const int units = (int)(n_places * a.n_heads);
        return launch(k_scan_segment<T, N, kWaves>, dim3((unsigned)((units + 7) / 8 * 8 * groups)), dim3(64 * kWaves), 0, s, a,
                      states, decays, seg, number, units);
    };
    if (cut(&a)) {
        hipError_t rc = pass(0, places(&a));
        if (rc != hipSuccess) return rc;
        if (a.n_tokens > 2u * (uint32_t)seg) {
            rc = launch(k_scan_join, dim3(a.state_dim * a.head_dim / 1024, a.n_heads, a.n_seqs < 1024 ? a.n_seqs : 1024),
                        dim3(kT), 0, s, a, states, static_cast<const float *>(decays), seg);
            if (rc != hipSuccess) return rc;
        }
    }
    return pass(1, places(&a) + a.n_seqs);
}
template <class T>
hipError_t launch_prefill_n(const GDNScan &a, void *ws, hipStream_t s) {
    return a.state_dim == 256   ? launch_prefill<T, 256>(a, ws, s)
           : a.state_dim == 128 ? launch_prefill<T, 128>(a, ws, s)
                                : launch_prefill<T, 64>(a, ws, s);
}
template <class T, int N>
hipError_t launch_step(const GDNScan &a, hipStream_t s) {
    return launch(k_scan_step<T, N>, dim3(a.head_dim / 64, a.n_heads, a.n_seqs), dim3(kT), 0, s, a);
}
template <class T>
hipError_t launch_step_n(const GDNScan &a, hipStream_t s) {
    return a.state_dim == 256 ? launch_step<T, 256>(a, s) : a.state_dim == 128 ? launch_step<T, 128>(a, s) : launch_step<T, 64>(a, s);
}

}  // namespace scan
}  // namespace gdn

extern "C" size_t gdn_scan_prefill_workspace(const GDNScan *args) {
    using namespace gdn::scan;
    if (args == nullptr || !dim_ok(args->state_dim) || !dim_ok(args->head_dim) || !cut(args)) return 0;
    return decay_bytes(args) + places(args) * args->n_heads * args->state_dim * args->head_dim * sizeof(float);
}

extern "C" int gdn_scan_prefill(const GDNScan *args, void *workspace, size_t workspace_bytes, void *stream) {
    using namespace gdn::scan;
    constexpr const char *who = "gdn_scan_prefill";
    const int rc = check(who, args, true);
    if (rc != 0) return rc < 0 ? -1 : 0;
    // a grid has fewer than 2^32 threads along an axis
    if (((uint64_t)places(args) + args->n_seqs + 8) * args->n_heads * (args->head_dim / (16 * kWaves)) >=
        (1ull << 32) / (64 * kWaves))
        return gdn::refuse(who, "too many segments or heads for one launch");
    const size_t need = gdn_scan_prefill_workspace(args);
    if (need != 0 && (workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 15) != 0 || workspace_bytes < need))
        return gdn::refuse(who, "the workspace is missing, misaligned or too small");
    hipStream_t s = static_cast<hipStream_t>(stream);
    return gdn::launched(who, args->dtype == GDN_DTYPE_BF16   ? launch_prefill_n<Bf16>(*args, workspace, s)
                              : args->dtype == GDN_DTYPE_FP16 ? launch_prefill_n<Fp16>(*args, workspace, s)
                                                              : launch_prefill_n<Fp32>(*args, workspace, s));
}

extern "C" int gdn_scan_step(const GDNScan *args, void *stream) {
    using namespace gdn::scan;
    constexpr const char *who = "gdn_scan_step";
    const int rc = check(who, args, false);
    if (rc != 0) return rc < 0 ? -1 : 0;
    hipStream_t s = static_cast<hipStream_t>(stream);
    return gdn::launched(who, args->dtype == GDN_DTYPE_BF16   ? launch_step_n<Bf16>(*args, s)
                              : args->dtype == GDN_DTYPE_FP16 ? launch_step_n<Fp16>(*args, s)
                                                              : launch_step_n<Fp32>(*args, s));
}
