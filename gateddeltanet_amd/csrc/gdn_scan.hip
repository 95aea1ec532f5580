// gdn_scan.hip -- the selective state space scan over a batch on the caller's
// device buffers: gdn_scan_prefill (packed sequences, chunk-parallel form) and
// gdn_scan_step (one token of every sequence).
#include <hip/hip_runtime.h>

#include <type_traits>

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

template <class T, int N, int NW, bool kY>
struct Lds {
    static constexpr int C = kChunk<T>, NT = T::kTerms, kTri = C == 64 ? 6 : 2;
    // 16-byte units of a row with its padding: B's and C's rows eight banks apart,
    // which keeps their rows' reads apart and halves the conflicts of B's transposed ones
    static constexpr int kRow = N / 8 + 2, kXRow = 2 * NW + 1;
    u32x4 b[NT][C][kRow], c[kY ? NT : 0][C][kRow], x[NT][C][kXRow];
    u32x4 m[kY ? kTri : 0][3][64];
    // of a block of NW chunks, by token: G's whole powers of two and the rest, the
    // step h, exp(G), exp(G_last - G) h; with E_j the G in front of 16-token tile j,
    // exp(G - E) of the token's own tile and exp(E_j - G) h for the tiles behind it
    struct Steps {
        int whole[C];
        float rest[C], step[C], eg[C], left[C], in[C], to[C / 16 - 1][C];
    } s[NW];
};
// Where a 16 x 32 tile of a chunk's lower triangular matrix is kept: row tile j,
// column step i.
__device__ __forceinline__ constexpr int tri_tile(int j, int i) { return j < 2 ? j : 2 * j - 2 + i; }

// The workspace: by place, the states behind cut segments, the starts of cut
// sequences at their first place (NULL where their slots are not written), decays.
struct Pools {
    float *states, *starts, *decays;
};

// Four values as three BF16 terms, which are exact: the first cut, so that none is
// rounded up to an infinity, the second rounded.  (An infinity or NaN has a NaN term.)
__device__ __forceinline__ void split(const f32x4 x, u32x2 (&p)[3]) {
    uint32_t u[4];
    float r[4] = {x.x, x.y, x.z, x.w};
    auto cut = [&](u32x2 &to) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = f2u(r[i]);
        to.x = __builtin_amdgcn_perm(u[1], u[0], 0x07060302u);
        to.y = __builtin_amdgcn_perm(u[3], u[2], 0x07060302u);
    };
    cut(p[0]);
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] -= u2f(u[i] & 0xffff0000u);
    p[1].x = cvt_pk(r[0], r[1]);
    p[1].y = cvt_pk(r[2], r[3]);
    r[0] -= u2f(p[1].x << 16);
    r[1] -= u2f(p[1].x & 0xffff0000u);
    r[2] -= u2f(p[1].y << 16);
    r[3] -= u2f(p[1].y & 0xffff0000u);
    cut(p[2]);
}

// Waves a SIMD that the LDS leaves room for, at most two.
template <class T, int N, int NW, bool kY>
constexpr int kPerSimd = NW == 8 || sizeof(Lds<T, N, NW, kY>) <= (80 << 10) ? 2 : 1;

// A segment's chunks in order, for a head's 16 NW columns, 16 a wave.  With G the
// running log decay of a chunk (sums in 64 bits) and h the steps:
//   y = exp(G) C S + M x,  M[m][s] = exp(G_m - G_s) h_s (C_m . B_s), s <= m, and D on
//   the diagonal;  S' = exp(G_last) S + B^T (exp(G_last - G) h x)
// Products are BF16 matrix instructions on the terms that the operands split into.
// A wave's state is the accumulator tiles of its update, and lies so that it is
// also an operand of C S: of a 32-row step, lane l holds rows 8 (l / 16) .. + 7 of
// column l % 16, the first four in one tile, the others in the next.  y is formed
// transposed, a lane's token with four columns in a row.  M's tiles are formed
// transposed too, B C^T, spread over the waves: an accumulator is then half an
// operand of M x as it is.  x and B^T are read transposed (ds_read_b64_tr_b16).  The
// steps and decays of NW chunks are formed at a time, a chunk a wave.  Two barriers a
// chunk.  A step's operands are read a step ahead, the next chunk's rows loaded one by
// one between the products of the update, and the splitting of the state and of x goes
// between those of C S.
// Two kernels of it:
//   kY false  the segments with a later one: the state that each leaves, the first
//             of a sequence from its start, the others from zero; their decays; and
//             the start itself where the sequence's slot is written
//   kY true   all segments, from the states behind the ones before them
// Bound by the instructions that a wave can issue: two waves a SIMD, each with 650
// vector instructions a chunk of 64 tokens, 126 products and 130 LDS instructions, one in
// seven cycles or so.  512 workgroups of one to four chunks, two on a CU, from zero states
// 12.3, 18.6, 24.5, 29.7 us: 5.8 a chunk, 6.5 for launch, lookup and first loads; with
// states in and out 2.5 to 3 more.  4096 tokens, 32 heads of 128 x 64: kY 29.8 us, not kY
// 14.1; matrix unit 29 % busy, vector units 45, LDS 34.  8111 tokens in 24 sequences, 8
// heads of 256 x 256, 100 MB of states: 105 and 28.8 us.  Measured at 4096 tokens against
// 26.6, when y's operands of a 16-bit type had two terms: M's weights as exponentials for
// each value, loads in one piece, three barriers 28.8; two column tiles in each of four
// waves (one wave a SIMD) 34.5; two heads a workgroup of eight waves equal; chunks of 32
// tokens 49 against 45 in all.  Conflict-free reads of B^T (the state's rows in another
// order, C read by 8 bytes) halve the LDS's busy cycles and change no time.
template <class T, int N, int NW, bool kY>
__global__ __launch_bounds__(64 * NW, (kPerSimd<T, N, NW, kY>)) void k_scan_segment(GDNScan p, Pools ws, int seg, int n_places, int units) {
    using L = Lds<T, N, NW, kY>;
    constexpr int C = L::C, NT = L::NT, MT = C / 16, JT = C / 32, KS = N / 32, kThreads = 64 * NW;
    constexpr int kCols = 16 * NW, kB = C * (N / 8), kX = C * (kCols / 8);  // 16-byte units (of 16-bit values) of a chunk's rows
    constexpr int kBr = (kB + kThreads - 1) / kThreads, kXr = (kX + kThreads - 1) / kThreads;
    __shared__ L lds;
    const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
    const int t = threadIdx.x, w = __builtin_amdgcn_readfirstlane(t >> 6), lane = t & 63, li = lane & 15, kk = lane >> 4;
    // the column groups of a (segment, head) share its rows of B and C: one XCD's
    // (workgroups go to the eight in turn)
    const int groups = (int)p.head_dim / kCols, bx = blockIdx.x >> 3;
    const int unit = (bx / groups) * 8 + (blockIdx.x & 7), cg = bx % groups;
    if (unit >= units) return;
    const int head = unit % (int)p.n_heads, place = unit / (int)p.n_heads, group = head / (int)(p.n_heads / p.n_groups);
    // cut segments by place; behind them, shorter, the sequences' last ones
    const bool last = kY && place >= n_places;
    const Found at = last ? ranked(p, place - n_places, [&](const Span &sp) { return sp.n - cuts_of(sp, seg) * seg; })
                          : find(p, place, [&](int first, int) { return first / seg; });
    const int slot = at.slot;
    const Span sp = at.rows;
    const int cuts = cuts_of(sp, seg), base = sp.first / seg, c0 = last ? cuts : place - base;
    if (slot < 0 || c0 < 0 || (!last && c0 >= cuts)) return;
    const int row0 = sp.first + c0 * seg, n_rows = min(seg, sp.n - c0 * seg), chunks = (n_rows + C - 1) / C;
    const int col0 = kCols * cg + 16 * w;  // the wave's first column
    const size_t head_at = (size_t)8 * kk * p.head_dim + col0 + li, tile = (size_t)N * p.head_dim;
    auto at_of = [&](int s, int a, int r) { return head_at + (size_t)(32 * s + 4 * a + r) * p.head_dim; };

    constexpr uint32_t kSize = T::kWords / 2;  // bytes of a value
    Raw8<T> breg[kBr], creg[kBr], xreg[kXr];
    auto rows_at = [&](const void *x, int64_t stride, int row, int first) __attribute__((always_inline)) {
        return static_cast<const char *>(x) + ((size_t)row * stride + first) * kSize;
    };
    // The part'th of `parts` parts of a chunk's loads.  Rows past the segment's end: its
    // last one, in bounds, put as zeros.
    constexpr int kLoads = kBr + kXr + (kY ? kBr : 0);
    auto fetch = [&](int c, int part, int parts) __attribute__((always_inline)) {
        const int last_row = min(n_rows - C * c, C) - 1, row = row0 + C * c;  // (its offset stays in 32 bits)
        auto load = [&](Raw8<T> &to, const char *from, int64_t stride, int i, int per) __attribute__((always_inline)) {
            const uint32_t step = (uint32_t)stride * kSize, at = 8 * kSize * (t % per);
            const uint32_t r = (uint32_t)(i * kThreads + t) / per;
            to.load(from + min((uint32_t)__umul24(r, step) + at, (uint32_t)__umul24((uint32_t)last_row, step) + at), 0);
        };
        const char *bp = rows_at(p.b, p.b_stride, row, group * N), *cp = rows_at(p.c, p.c_stride, row, group * N),
                   *xp = rows_at(p.x, p.x_stride, row, head * (int)p.head_dim + kCols * cg);
#pragma unroll
        for (int i = 0; i < kLoads; ++i)
            if (i * parts / kLoads == part) {
                if (i < kBr) load(breg[i], bp, p.b_stride, i, N / 8);
                else if (i < kBr + kXr) load(xreg[i - kBr], xp, p.x_stride, i - kBr, kCols / 8);
                else if constexpr (kY) load(creg[i - kBr - kXr], cp, p.c_stride, i - kBr - kXr, N / 8);
            }
    };
    auto put_rows = [&](int c) __attribute__((always_inline)) {
        const int n = n_rows - C * c;
        if (n < C) {
#pragma unroll
            for (int i = 0; i < kBr; ++i)
                if ((i * kThreads + t) / (N / 8) >= n) {
                    breg[i].zero();
                    if constexpr (kY) creg[i].zero();
                }
#pragma unroll
            for (int i = 0; i < kXr; ++i)
                if ((i * kThreads + t) / (kCols / 8) >= n) xreg[i].zero();
        }
        auto put = [&](auto &to, const Raw8<T> &from, int i, int per, int total) __attribute__((always_inline)) {
            const int u = i * kThreads + t;
            if (total % kThreads != 0 && u >= total) return;
            u32x4 e[NT];
            from.terms(e);
#pragma unroll
            for (int q = 0; q < NT; ++q) to[q][u / per][u % per] = e[q];
        };
#pragma unroll
        for (int i = 0; i < kBr; ++i) put(lds.b, breg[i], i, N / 8, kB);
#pragma unroll
        for (int i = 0; i < kXr; ++i) put(lds.x, xreg[i], i, kCols / 8, kX);
        if constexpr (kY) {
#pragma unroll
            for (int i = 0; i < kBr; ++i) put(lds.c, creg[i], i, N / 8, kB);
        }
    };
    // wave w's chunk of a block of NW: steps, decays
    const double rate = (double)p.A[head] * 1.44269504088896340736;
    const float skip = kY && p.D ? p.D[head] : 0.0f;
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
        const double sum = wave_scan64(in ? g : 0.0), n = __builtin_rint(sum);
        auto of_lane = [&](int l) {
            const uint64_t u = __builtin_bit_cast(uint64_t, sum);
            const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)u, l),
                           hi = (uint32_t)__builtin_amdgcn_readlane((int)(u >> 32), l);
            return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
        };
        const double last = of_lane(C - 1);
        double front = 0.0;
        if constexpr (kY) {
#pragma unroll
            for (int j = 1; j < MT; ++j) {
                const double e = of_lane(16 * j - 1);
                if (lane >= 16 * j) front = e;
                else lds.s[w].to[j - 1][lane] = exp2_of(e - sum) * h;
            }
            if (lane < C) lds.s[w].in[lane] = exp2_of(sum - front);
        }
        if (lane < C) {
            lds.s[w].whole[lane] = (int)n;
            lds.s[w].rest[lane] = (float)(sum - n);
            lds.s[w].step[lane] = h;
            lds.s[w].eg[lane] = exp2_of(sum);
            lds.s[w].left[lane] = exp2_of(last - sum) * h;
        }
    };

    if (chunks > 0) {
        fetch_dt(0);
        fetch(0, 0, 1);
    }
    f32x4 S[KS][2];
    auto each_state = [&](auto &&f) __attribute__((always_inline)) {
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int a = 0; a < 2; ++a)
#pragma unroll
                for (int r = 0; r < 4; ++r) f(s, a, r);
    };
    auto put_state = [&](float *to) __attribute__((always_inline)) {
        each_state([&](int s, int a, int r) __attribute__((always_inline)) { to[at_of(s, a, r)] = S[s][a][r]; });
    };
    // the workspace's states lie as the registers do, a wave's together
    const size_t kept = (size_t)(col0 / 16) * (16 * N) + 4 * lane;
    auto keep = [&](float *to) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 2 * KS; ++i) *reinterpret_cast<f32x4 *>(to + kept + 256 * i) = S[i / 2][i % 2];
    };
    {
        const size_t first = ((size_t)base * p.n_heads + head) * tile;  // in the pools of places
        const float *ours = !kY          ? nullptr
                            : c0 > 0     ? ws.states + first + (size_t)(c0 - 1) * p.n_heads * tile
                            : cuts > 0   ? ws.starts ? ws.starts + first : nullptr
                                         : nullptr;
        each_state([&](int s, int a, int r) __attribute__((always_inline)) { S[s][a][r] = 0.0f; });
        if (ours) {
#pragma unroll
            for (int i = 0; i < 2 * KS; ++i) S[i / 2][i % 2] = *reinterpret_cast<const f32x4 *>(ours + kept + 256 * i);
        } else if (c0 == 0 && p.state_in) {
            const float *from = p.state_in + ((size_t)slot * p.n_heads + head) * tile;
            each_state([&](int s, int a, int r) __attribute__((always_inline)) { S[s][a][r] = from[at_of(s, a, r)]; });
            if (!kY && ws.starts) keep(ws.starts + first);
        }
    }
    // of M's tiles on the diagonal, the half above it
    if (kY && w == 0) {
#pragma unroll
        for (int j = 0; j < MT; j += 2)
#pragma unroll
            for (int q = 0; q < 3; ++q)
                reinterpret_cast<u32x2 *>(&lds.m[tri_tile(j, j / 2)][q][lane])[1] = (u32x2){0u, 0u};
    }
    float decay = 1.0f;
    if (chunks > 0) {
        put_steps(0);
        put_rows(0);
        fetch_dt(NW);
        __syncthreads();
    }
    for (int c = 0; c < chunks; ++c) {
        const int n = min(C, n_rows - C * c), cb = c % NW;
        const int next = min(c + 1, chunks - 1);  // (the last chunk's rows are loaded again, unused)
        const typename L::Steps &sc = lds.s[cb];
        f32x4 y[MT];
        u32x4 xb[JT][NT], xo[JT][3];
        // the value of a 16-bit operand's terms
        auto value = [&](const uint32_t(&u)[NT], int r) __attribute__((always_inline)) {
            auto term = [&](int q) { return u2f(r % 2 ? u[q] & 0xffff0000u : u[q] << 16); };
            float v = term(NT - 1);
#pragma unroll
            for (int q = NT - 2; q >= 0; --q) v += term(q);
            return v;
        };
        // x as an operand: of a 32-token step, tokens 4 (l / 16) .. + 3 and those 16 on
        auto read_x = [&]() __attribute__((always_inline)) {
#pragma unroll
            for (int j = 0; j < JT; ++j)
#pragma unroll
                for (int q = 0; q < NT; ++q) {
                    const int m = 32 * j + 4 * kk + (li >> 2), u = 4 * w + (li & 3);
                    const u32x2 lo = read_transposed(reinterpret_cast<const u32x2 *>(&lds.x[q][m][0]) + u);
                    const u32x2 hi = read_transposed(reinterpret_cast<const u32x2 *>(&lds.x[q][m + 16][0]) + u);
                    xb[j][q] = (u32x4){lo.x, lo.y, hi.x, hi.y};
                }
        };
        // the terms of its values times exp(G_last - G) h, the k'th four
        auto weigh = [&](int k) __attribute__((always_inline)) {
            const int j = k / 2, h = k % 2;
            f32x4 v;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                uint32_t u[NT];
#pragma unroll
                for (int q = 0; q < NT; ++q) u[q] = xb[j][q][2 * h + r / 2];
                v[r] = value(u, r) * sc.left[32 * j + 16 * h + 4 * kk + r];
            }
            u32x2 e[3];
            split(v, e);
#pragma unroll
            for (int q = 0; q < 3; ++q) {
                xo[j][q][2 * h] = e[q].x;
                xo[j][q][2 * h + 1] = e[q].y;
            }
        };
        // operands of a 32-row step: C's rows, B^T's, the state's terms
        auto read_c = [&](int s, u32x4(&ca)[MT][NT]) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int q = 0; q < NT; ++q) ca[i][q] = lds.c[q][16 * i + li][4 * s + kk];
        };
        auto read_b = [&](int s, u32x4(&a)[2][JT][NT]) __attribute__((always_inline)) {
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
        };
        auto terms_of = [&](int s, u32x4(&sb)[3]) __attribute__((always_inline)) {
            u32x2 lo[3], hi[3];
            split(S[s][0], lo);
            split(S[s][1], hi);
#pragma unroll
            for (int q = 0; q < 3; ++q) sb[q] = (u32x4){lo[q].x, lo[q].y, hi[q].x, hi[q].y};
        };
        // what stands between two of these: the loads first, then products with some
        // of the rest behind each
        auto mix = [&](auto products, auto others) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < decltype(products)::value; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x002, decltype(others)::value, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
        };
        using std::integral_constant;
        u32x4 ab[2][2][JT][NT];
        if constexpr (kY) {
            // C_m . B_s of row tile j (a lane's token m), column tile i (its four s)
            struct Operands {
                u32x4 a[NT], b[NT];
            };
            auto read_step = [&](int j, int i, int s, Operands &o) __attribute__((always_inline)) {
#pragma unroll
                for (int k = 0; k < NT; ++k) {
                    o.a[k] = lds.b[k][16 * i + li][4 * s + kk];
                    o.b[k] = lds.c[k][16 * j + li][4 * s + kk];
                }
            };
            auto multiply = [&](const Operands &o, f32x4 z) __attribute__((always_inline)) {
                for_terms<NT, NT>([&](int k, int l) __attribute__((always_inline)) { z = mfma_bf16(o.a[k], o.b[l], z); });
                return z;
            };
            auto read_tile = [&](int j, int i, Operands(&o)[KS]) __attribute__((always_inline)) {
#pragma unroll
                for (int s = 0; s < KS; ++s) read_step(j, i, s, o[s]);
            };
            auto products = [&](const Operands(&o)[KS]) __attribute__((always_inline)) {
                f32x4 z[2] = {zero, zero};
#pragma unroll
                for (int s = 0; s < KS; ++s) z[s & 1] = multiply(o[s], z[s & 1]);
                return z[0] + z[1];
            };
            auto products_at = [&](int j, int i) __attribute__((always_inline)) {
                f32x4 z[2] = {zero, zero};
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    Operands o;
                    read_step(j, i, s, o);
                    z[s & 1] = multiply(o, z[s & 1]);
                }
                return z[0] + z[1];
            };
            auto put_tile = [&](int j, int i, const f32x4 v) __attribute__((always_inline)) {
                u32x2 e[3];
                split(v, e);
#pragma unroll
                for (int k = 0; k < 3; ++k) reinterpret_cast<u32x2 *>(&lds.m[tri_tile(j, i / 2)][k][lane])[i & 1] = e[k];
            };
            // M's tiles: on the diagonal a power for each value, above it zeros whatever the
            // tokens hold
            auto diagonal = [&](int j, const f32x4 z) __attribute__((always_inline)) {
                const int to = 16 * j + li, of = 16 * j + 4 * kk;
                const int n_to = sc.whole[to];
                const float f_to = sc.rest[to];
                f32x4 e;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int n2 = n_to - sc.whole[of + r];
                    e[r] = __builtin_ldexpf(__builtin_amdgcn_exp2f(f_to - sc.rest[of + r]), n2) * sc.step[of + r];
                }
                f32x4 v = z * e;
#pragma unroll
                for (int r = 0; r < 4; ++r) v[r] = 4 * kk + r <= li ? v[r] + (4 * kk + r == li ? skip : 0.0f) : 0.0f;
                put_tile(j, j, v);
            };
            // below it what falls in front of the row tile and inside it
            auto row_of = [](int q) { return q < 1 ? 1 : q < 3 ? 2 : 3; };
            auto column_of = [&](int q) { return q - row_of(q) * (row_of(q) - 1) / 2; };
            auto below = [&](int q, const f32x4 z) __attribute__((always_inline)) {
                const int j = row_of(q), i = column_of(q);
                const float in = sc.in[16 * j + li];
                f32x4 e;
#pragma unroll
                for (int r = 0; r < 4; ++r) e[r] = in * sc.to[j - 1][16 * i + 4 * kk + r];
                put_tile(j, i, z * e);
            };
            // spread over the waves
            constexpr int kBelow = MT * (MT - 1) / 2;
            if constexpr (MT == NW && KS * NT <= 4) {
                // ten tiles, three a wave (two waves have one of theirs twice), the next
                // one's operands read ahead
                const int q = w < kBelow - NW ? NW + w : w;
                Operands o[2][KS];
                read_tile(row_of(q), column_of(q), o[0]);
                read_tile(row_of(w), column_of(w), o[1]);
                below(q, products(o[0]));
                read_tile(w, w, o[0]);
                below(w, products(o[1]));
                diagonal(w, products(o[0]));
            } else {
                constexpr int kFirst = MT >= NW ? 0 : MT, kEach = NW - kFirst;
                if (w < MT) diagonal(w, products_at(w, w));
#pragma unroll
                for (int from = 0; from < kBelow; from += kEach) {
                    const int q = from + w - kFirst;
                    if (q >= from && q < kBelow) below(q, products_at(row_of(q), column_of(q)));
                }
            }
            __builtin_amdgcn_sched_barrier(0);

            // C S (y's lane l: token l % 16, columns 4 (l / 16) .. + 3) and x's terms
            u32x4 ca[2][MT][NT], sb[2][3];
            read_c(0, ca[0]);
            read_x();
            terms_of(0, sb[0]);
#pragma unroll
            for (int i = 0; i < MT; ++i) y[i] = zero;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                if (s + 1 < KS) read_c(s + 1, ca[(s + 1) & 1]);
                else read_b(0, ab[0]);
                if (s + 1 < KS) terms_of(s + 1, sb[(s + 1) & 1]);
#pragma unroll
                for (int k = 0; k < 2 * JT; ++k)
                    if (k * KS / (2 * JT) == s) weigh(k);
                for_terms<3, NT>([&](int a, int b) __attribute__((always_inline)) {
#pragma unroll
                    for (int i = 0; i < MT; ++i) y[i] = mfma_bf16(sb[s & 1][a], ca[s & 1][i][b], y[i]);
                });
                mix(integral_constant<int, MT * (NT == 3 ? 6 : NT == 2 ? 5 : 3)>(), integral_constant<int, 5>());
            }
        } else {
            read_x();
            read_b(0, ab[0]);
#pragma unroll
            for (int k = 0; k < 2 * JT; ++k) weigh(k);
        }
        const float dn = sc.eg[C - 1];
        decay *= dn;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            if (s + 1 < KS) read_b(s + 1, ab[(s + 1) & 1]);
            fetch(next, s, KS);
            S[s][0] *= dn;
            S[s][1] *= dn;
            for_terms<NT, 3>([&](int e, int f) __attribute__((always_inline)) {
#pragma unroll
                for (int j = 0; j < JT; ++j)
#pragma unroll
                    for (int h = 0; h < 2; ++h) S[s][h] = mfma_bf16(ab[s & 1][h][j][e], xo[j][f], S[s][h]);
            });
            __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (kY) {
#pragma unroll
            for (int i = 0; i < MT; ++i) y[i] *= sc.eg[16 * i + li];
        }
        __syncthreads();
        // (B's, C's and x's rows and the steps are free from here, M's tiles from the
        // next barrier; the rows before the stores, which would be waited for too)
        if (c + 1 < chunks) {
            put_rows(c + 1);
            if (cb == NW - 1) {
                put_steps(c + 1);
                fetch_dt(c + 1 + NW);
            }
        }
        if constexpr (kY) {
            // a value of x that is not finite, times M's zeros, would reach the tokens before it:
            // its column's outputs from it on are made NaN instead, and it 0
            auto word = [&](int j, int i) __attribute__((always_inline)) { return xb[j][NT == 1 ? 0 : 1][i] & 0x7fff7fffu; };
            typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
            u16x2 top = {0, 0};
#pragma unroll
            for (int j = 0; j < JT; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, word(j, i)));
            if (__ballot(top.x >= 0x7f80 || top.y >= 0x7f80) != 0) {
                int first = C;  // (the terms behind the first show it, of values of several)
#pragma unroll
                for (int j = 0; j < JT; ++j)
#pragma unroll
                    for (int r = 7; r >= 0; --r) {
                        const uint32_t half = r % 2 ? 0xffff0000u : 0xffffu;
                        if ((word(j, r / 2) & half) >= (0x7f807f80u & half)) {
                            first = min(first, 32 * j + 16 * (r / 4) + 4 * kk + r % 4);
#pragma unroll
                            for (int q = 0; q < NT; ++q) xb[j][q][r / 2] &= ~half;
                        }
                    }
                first = min(first, __shfl_xor(first, 16));
                first = min(first, __shfl_xor(first, 32));
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int from = __shfl(first, 4 * kk + r);
#pragma unroll
                    for (int j = 0; j < MT; ++j)
                        if (16 * j + li >= from) y[j][r] = __builtin_nanf("");
                }
            }
            for_terms<NT, 3>([&](int a, int b) __attribute__((always_inline)) {
#pragma unroll
                for (int i = 0; i < JT; ++i)
#pragma unroll
                    for (int j = 2 * i; j < MT; ++j) y[j] = mfma_bf16(xb[i][a], lds.m[tri_tile(j, i)][b][lane], y[j]);
            });
            char *yp = const_cast<char *>(rows_at(p.y, p.y_stride, row0 + C * c, head * (int)p.head_dim + col0));
#pragma unroll
            for (int j = 0; j < MT; ++j) {
                const int m = 16 * j + li;
                char *to = yp + ((uint32_t)__umul24((uint32_t)m, (uint32_t)p.y_stride * kSize) + 4 * kSize * kk);
                if (m < n) {
                    if constexpr (kSize == 4) *reinterpret_cast<f32x4 *>(to) = y[j];
                    else *reinterpret_cast<u32x2 *>(to) = (u32x2){T::pack(y[j].x, y[j].y), T::pack(y[j].z, y[j].w)};
                }
            }
        }
        __syncthreads();
    }
    if constexpr (kY) {
        if (c0 == cuts && p.state_out) put_state(p.state_out + ((size_t)slot * p.n_heads + head) * tile);
    } else {
        keep(ws.states + ((size_t)place * p.n_heads + head) * tile);
        if (cg == 0 && t == 0) ws.decays[(size_t)place * p.n_heads + head] = decay;
    }
}

// Between the two: a sequence's states behind its segments from what each of them
// adds, their bytes once in and out (4096 tokens, 32 heads of 128 x 64, 15 states of 1 MB:
// 7.3 us, 4.3 TB/s), of 1024 values a workgroup: grid (state values / 1024, heads, sequences of two
// cuts and more, which up to 64 sequences' lanes tell; of more, the sequences in turn, or the
// places where they are fewer, a sequence's first one for it).  500 sequences of one token, 32
// heads of 128 x 64, have 7 places: 4.8 us, by sequence 67; 70 of 3000 tokens, 4 heads of 64 x 64,
// by sequence 165 us in all, by their 205 places 169.
__global__ __launch_bounds__(kT) void k_scan_join(GDNScan p, Pools ws, int seg, int n_places) {
    const size_t tile = (size_t)p.state_dim * p.head_dim;
    const int head = blockIdx.y, at = (blockIdx.x * kT + (int)threadIdx.x) * 4;
    auto join = [&](int first, int cuts) __attribute__((always_inline)) {
        const size_t unit = (size_t)(first / seg) * p.n_heads + head;
        float *s = ws.states + unit * tile + at;
        const float *d = ws.decays + unit;
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
    };
    const int n = (int)p.n_seqs, lane = threadIdx.x & 63;
    if (n <= 64) {
        const int i = min(lane, n - 1);
        const Span sp = span_of(p, i);
        uint64_t mask = __ballot(lane < n && cuts_of(sp, seg) >= 2 && slot_of(p, i) >= 0);
        for (int z = blockIdx.z; z > 0; --z) mask &= mask - 1;
        if (mask == 0) return;
        const int of = __builtin_ctzll(mask), first = __builtin_amdgcn_readlane(sp.first, of);
        join(first, cuts_of({first, __builtin_amdgcn_readlane(sp.n, of)}, seg));
    } else if (n <= n_places) {
        for (int i = blockIdx.z; i < n; i += gridDim.z) {
            const Span sp = span_of(p, i);
            if (cuts_of(sp, seg) >= 2 && slot_of(p, i) >= 0) join(sp.first, cuts_of(sp, seg));
        }
    } else {
        for (int place = blockIdx.z; place < n_places; place += gridDim.z) {
            const Found at = find(p, place, [&](int first, int) { return first / seg; });
            const int cuts = cuts_of(at.rows, seg);
            if (at.rows.first / seg == place && cuts >= 2 && at.slot >= 0) join(at.rows.first, cuts);
        }
    }
}

// ------------------------------------------------------------ a single token

// A (sequence, head)'s token for 64 columns: grid (head_dim / 64, heads,
// sequences).  The state's tile goes through registers once, y's sums formed as it is
// written, so its bytes bound the kernel: 64 sequences of 32 heads of 128 x 64, 134 MB, in
// 21 us (6.3 TB/s, partly from the last-level cache), one of 16 heads of 128 x 128 in 4.3.
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
// Waves of a workgroup, 16 columns each, and workgroups of a segment: the eight share
// their rows of B and C, which four would stage twice as often (not measured).
int waves_of(const GDNScan *a) { return a->head_dim == 64 ? 4 : 8; }
uint64_t groups_of(const GDNScan *a) { return (uint64_t)a->n_heads * a->head_dim / (16 * waves_of(a)); }

// Tokens of a segment: as many as give eleven waves a CU, in 128s, of which eight run
// at a time (sequences end inside them; of BF16 256 x 64 only four run, which the rule
// does not look at), at most 1024.  Measured when y's operands of a 16-bit type had two
// terms: 4096 tokens in one sequence, 32
// heads of 128 x 64, segments of 192, 256, 384, 512, 1024: 52, 43, 52, 49, 80 us; 8111 in
// 24, 8 heads of 256 x 256, of 256, 320, 384, 512, 768: 146, 143, 126, 138, 158; 512 in
// one, of 128, 256: 36, 42.  64 tokens where that leaves half of the eight or so idle, for
// the chunks that follow each other are what takes the time: 300 tokens of 8 heads of 128
// x 128, segments of 128 and 64, BF16 22.6, 18.9, FP32 33.9, 24.3; 1000 25.2, 25.2 and
// 36.6, 30.8; (more: the states' traffic, 4 x 500 of 256 x 128 38, 48).  Up to 256
// tokens are not cut (one launch in place of two or three): 150 of 32 heads of 128 x 64
// 13.3 us, 16.9 in two segments; 256, 16.4 and 17.1.
int segment_of(const GDNScan *a) {
    if (a->n_tokens <= 256) return 256;
    const uint64_t waves = a->n_tokens * groups_of(a) * waves_of(a);  // times tokens of a segment
    const uint64_t even = (waves / (11 * 256) + 127) / 128 * 128;
    return waves <= 32 * 11 * 256 ? 64 : even > 1024 ? 1024 : (int)even;
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

// The first segments' starts are kept where the slots that they come from are written.
bool keeps_starts(const GDNScan *a) { return a->state_in && a->state_in == a->state_out; }
size_t pool_bytes(const GDNScan *a) { return places(a) * a->n_heads * a->state_dim * a->head_dim * sizeof(float); }

template <class T, int N, int NW, bool kY>
hipError_t launch_segments(const GDNScan &a, const Pools &ws, int seg, int n_places, hipStream_t s) {
    const int units = (int)((n_places + (kY ? a.n_seqs : 0)) * a.n_heads), groups = (int)a.head_dim / (16 * NW);
    return launch(k_scan_segment<T, N, NW, kY>, dim3((unsigned)((units + 7) / 8 * 8 * groups)), dim3(64 * NW), 0, s, a, ws, seg,
                  n_places, units);
}
template <class T, int N, int NW>
hipError_t launch_prefill(const GDNScan &a, void *mem, hipStream_t s) {
    const int seg = segment_of(&a);
    char *at = static_cast<char *>(mem);
    Pools ws = {nullptr, nullptr, nullptr};
    if (cut(&a)) {
        ws.decays = reinterpret_cast<float *>(at);
        ws.states = reinterpret_cast<float *>(at + decay_bytes(&a));
        if (keeps_starts(&a)) ws.starts = reinterpret_cast<float *>(at + decay_bytes(&a) + pool_bytes(&a));
        hipError_t rc = launch_segments<T, N, NW, false>(a, ws, seg, (int)places(&a), s);
        if (rc != hipSuccess) return rc;
        if (a.n_tokens > 2u * (uint32_t)seg) {
            // a sequence of two cuts has two places
            const unsigned n = (unsigned)places(&a), most = a.n_seqs <= 64 ? n / 2 : n < 1024 ? n : 1024;
            rc = launch(k_scan_join, dim3(a.state_dim * a.head_dim / 1024, a.n_heads, a.n_seqs < most ? a.n_seqs : most), dim3(kT),
                        0, s, a, ws, seg, (int)n);
            if (rc != hipSuccess) return rc;
        }
    }
    return launch_segments<T, N, NW, true>(a, ws, seg, cut(&a) ? (int)places(&a) : 0, s);
}
template <class T, int N>
hipError_t launch_prefill_w(const GDNScan &a, void *ws, hipStream_t s) {
    return waves_of(&a) == 4 ? launch_prefill<T, N, 4>(a, ws, s) : launch_prefill<T, N, 8>(a, ws, s);
}
template <class T>
hipError_t launch_prefill_n(const GDNScan &a, void *ws, hipStream_t s) {
    return a.state_dim == 256   ? launch_prefill_w<T, 256>(a, ws, s)
           : a.state_dim == 128 ? launch_prefill_w<T, 128>(a, ws, s)
                                : launch_prefill_w<T, 64>(a, ws, s);
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
    return decay_bytes(args) + pool_bytes(args) * (keeps_starts(args) ? 2 : 1);
}

extern "C" int gdn_scan_prefill(const GDNScan *args, void *workspace, size_t workspace_bytes, void *stream) {
    using namespace gdn::scan;
    constexpr const char *who = "gdn_scan_prefill";
    const int rc = check(who, args, true);
    if (rc != 0) return rc < 0 ? -1 : 0;
    // a grid has fewer than 2^32 threads along an axis
    if (((uint64_t)places(args) + args->n_seqs + 8) * groups_of(args) >= (1ull << 32) / (64 * (uint64_t)waves_of(args)))
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
